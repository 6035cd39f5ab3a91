// The selective scan of whole sequences (selective_scan.h has the formulas and the split).
#include "selective_scan.h"

#include <algorithm>

namespace rka {
namespace scan {
namespace {

// One block of channels through one chunk.  STATES_ONLY: from nothing to the chunk's own state
// and the sum of its steps; else from the state at its start to the outputs.  16384 tokens of 2048
// channels, 16 states, bf16: 101 and 156 us.  Bound by vector instructions: a token takes 20 for
// its four states of a lane (and the exponentials twice an instruction's time), 2.5 for its sum
// and a share of some 10 of what the tile makes of its inputs; they issue in three quarters of the
// clocks.  Memory alone would take 56.  Four wavefronts to a SIMD hold the registers; five with
// some of them spilled take 7% longer; one channel to a lane with all its states is no faster.
template <typename T, int NB, bool STATES_ONLY>
__global__ __launch_bounds__(64) void chunk_kernel(Dims d, float* states, float* sums, const float* initial, T* y,
                                                   float* final_state, float* kept) {
    __shared__ __attribute__((aligned(16))) float steps[16][2 * kTile + 4];  // of a channel: s; s x
    __shared__ __attribute__((aligned(16))) float bt[kTile][NB * 16], ct[STATES_ONLY ? 1 : kTile][NB * 16];
    const int lane = threadIdx.x, c = lane % 16, nl = lane / 16;
    const int Dg = d.D / d.G, per_group = (Dg - 1) / 16 + 1, blocks = d.G * per_group;
    const int chunks = STATES_ONLY ? d.chunks - 1 : d.chunks;
    const long long id = in_order();
    const int block = (int)(id % blocks), chunk = (int)(id / blocks % chunks), b = (int)(id / blocks / chunks);
    const int g = block / per_group, in = block % per_group * 16 + c;
    const bool on = in < Dg;
    const int ch = g * Dg + min(in, Dg - 1);
    const int len = row_length(d.lengths, b, d.T);
    const int t0 = chunk * d.chunk, t_end = min(d.T, t0 + d.chunk), t1 = min(len, t_end);
    const size_t at = (size_t)b * d.chunks + chunk;

    f32x4 a2[NB], h[NB];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        const int n0 = 16 * k + 4 * nl;
        a2[k] = finite_rates(load_states_of(d.A + (size_t)ch * d.N, n0, d.N));
        if (STATES_ONLY)
            h[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        else if (d.chunks > 1)
            h[k] = load_states(states + at * d.N * d.D, n0, d.N, d.D, ch);
        else
            h[k] = initial ? load_states_of(initial + ((size_t)b * d.D + ch) * d.N, n0, d.N) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float bias = d.bias ? d.bias[ch] : 0.f, skip = !STATES_ONLY && d.skip ? d.skip[ch] : 0.f;
    const T* px = static_cast<const T*>(d.x) + b * d.xs[0];
    const T* pt = static_cast<const T*>(d.dt) + b * d.ts[0];
    const T* pz = static_cast<const T*>(d.gate) + b * d.zs[0];
    const T* gb = static_cast<const T*>(d.Bm) + b * d.bs[0] + g * d.bs[2];
    const T* gc = static_cast<const T*>(d.C) + b * d.cs[0] + g * d.cs[2];
    T* py = STATES_ONLY ? nullptr : y + (size_t)b * d.T * d.D;
    Rows<T> x, dt, gate, bv[NB], cv[NB];
    Offsets ox, ot, oz, ob[NB], oc[NB], oy;
    auto set = [&](int rows) {
        ox.set(d.xs[1], ch, rows, sizeof(T));
        ot.set(d.ts[1], ch, rows, sizeof(T));
        if (!STATES_ONLY && d.gate) oz.set(d.zs[1], ch, rows, sizeof(T));
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const int n = min(16 * k + c, d.N - 1);
            ob[k].set(d.bs[1], n, rows, sizeof(T));
            if (!STATES_ONLY) oc[k].set(d.cs[1], n, rows, sizeof(T));
        }
    };
    auto load = [&](int t) {
        if (t1 - t < kTile) set(t1 - t);
        x.load(px + t * d.xs[1], ox);
        dt.load(pt + t * d.ts[1], ot);
        if (!STATES_ONLY && d.gate) gate.load(pz + t * d.zs[1], oz);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            bv[k].load(gb + t * d.bs[1], ob[k]);
            if (!STATES_ONLY) cv[k].load(gc + t * d.cs[1], oc[k]);
        }
    };
    float sum = 0.f;
    set(kTile);
    oy.set(d.D, ch, kTile, sizeof(T));
    if (t0 < t1) load(t0);
    for (int t = t0; t < t1; t += kTile) {
        if (!STATES_ONLY && kept) {
            float* to = kept + ((size_t)b * ((d.T - 1) / kTile + 1) + t / kTile) * d.N * d.D;
#pragma unroll
            for (int k = 0; k < NB; ++k)
                if (on) store_states(to, 16 * k + 4 * nl, d.N, d.D, ch, h[k]);
        }
        // (a token behind the last has a step of 0, which changes nothing, and is no output)
        const int rows = t1 - t - 4 * nl;
        float xf[4], zf[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float slope, s = to_f32(dt.v[r]) + bias;
            if (d.softplus) s = softplus<T>(s, &slope);
            s = r < rows ? s : 0.f;
            xf[r] = r < rows ? to_f32(x.v[r]) : 0.f;
            zf[r] = !STATES_ONLY && d.gate ? to_f32(gate.v[r]) : 0.f;
            sum += s;
            steps[c][4 * nl + r] = s;
            steps[c][kTile + 4 * nl + r] = s * xf[r];
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                const bool is = r < rows && 16 * k + c < d.N;
                bt[4 * nl + r][16 * k + c] = is ? to_f32(bv[k].v[r]) : 0.f;
                if (!STATES_ONLY) ct[4 * nl + r][16 * k + c] = is ? to_f32(cv[k].v[r]) : 0.f;
            }
        }
        __syncthreads();
        if (t + kTile < t1) load(t + kTile);
        f32x4 acc{0.f, 0.f, 0.f, 0.f};
        // (addresses from one place for four tokens: each array's own would cost an addition a token)
        const float *ps = &steps[c][0], *pb = &bt[0][4 * nl], *pc = &ct[0][4 * nl];
#pragma unroll 1
        for (int q = 0; q < 4; ++q, ps += 4, pb += 64 * NB, pc += 64 * NB) {
            const f32x4 s4 = load4(ps), i4 = load4(ps + kTile);
            float parts[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float part = 0.f;
#pragma unroll
                for (int k = 0; k < NB; ++k) {
                    const f32x4 bq = load4(pb + 16 * (NB * i + k));
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[k][j] = fmaf(__builtin_amdgcn_exp2f(s4[i] * a2[k][j]), h[k][j], i4[i] * bq[j]);
                    if (!STATES_ONLY) {
                        const f32x4 cq = load4(pc + 16 * (NB * i + k));
#pragma unroll
                        for (int j = 0; j < 4; ++j) part = fmaf(cq[j], h[k][j], part);
                    }
                }
                parts[i] = part;
            }
            if (!STATES_ONLY) acc = f32x4{acc[1], acc[2], acc[3], token_sums(parts[0], parts[1], parts[2], parts[3])};
        }
        if (!STATES_ONLY) {
            own_tokens(&acc);
            const Memory to(py + (size_t)t * d.D);
            const int room = t_end - t - 4 * nl;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v = fmaf(skip, xf[r], acc[r]);
                if (d.gate) v *= zf[r] * sigmoid_of<T>(zf[r]);
                if (on && r < room) to.store(from_f32<T>(r < rows ? v : 0.f), oy.at[r]);
            }
        }
        __syncthreads();
    }
    if (STATES_ONLY) {
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (on && nl == 0) sums[at * d.D + ch] = sum;
    } else {
        // tiles behind the row's end
        const int rest = t1 <= t0 ? t0 : t0 + ((t1 - t0 - 1) / kTile + 1) * kTile;
        for (int t = rest + nl; t < t_end; t += 4)
            if (on) py[(size_t)t * d.D + ch] = from_f32<T>(0.f);
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        const int n0 = 16 * k + 4 * nl;
        if (!on) continue;
        if (STATES_ONLY)
            store_states(states + at * d.N * d.D, n0, d.N, d.D, ch, h[k]);
        else if (chunk == d.chunks - 1)
            store_states_of(final_state + ((size_t)b * d.D + ch) * d.N, n0, d.N, h[k]);
    }
}

__global__ __launch_bounds__(256) void join_kernel(Dims d, float* own, const float* sums, const float* first, int backward) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, per = (long long)d.N * d.D;
    if (i >= per * d.B) return;
    const int b = (int)(i / per), n = (int)(i % per / d.D), ch = (int)(i % d.D);
    const float a2 = finite_rate(d.A[(size_t)ch * d.N + n], 0.5f * kLog2e);
    float h = first ? first[((size_t)b * d.D + ch) * d.N + n] : 0.f;
    const long long start = backward ? d.chunks - 1 : 0, step = backward ? -1 : 1;
    float* p = own + ((size_t)b * d.chunks + start) * per + (size_t)n * d.D + ch;
    const float* ps = sums + ((size_t)b * d.chunks + start) * d.D + ch;
    constexpr int kDeep = 8;
    for (int c0 = 0; c0 < d.chunks; c0 += kDeep) {
        float mine[kDeep], sum[kDeep];
        const int left = d.chunks - c0;
#pragma unroll
        for (int j = 0; j < kDeep; ++j) {
            // (the last chunk's own is not made: where it alone is left, what is loaded is not used)
            const long long of = step * min(j, max(0, left - 2));
            mine[j] = p[of * per];
            sum[j] = ps[of * d.D];
        }
#pragma unroll
        for (int j = 0; j < kDeep; ++j) {
            if (j >= left) break;
            p[step * j * per] = h;
            // (by its root twice, which stays finite: a growing chunk's factor may be infinite where what it
            // makes of h, which may be 0, is not; where a sum is NaN so is the chunk's own state)
            const float root = fminf(__builtin_amdgcn_exp2f(sum[j] * a2), 3e38f);
            h = fmaf(root, root * h, mine[j]);
        }
        p += step * kDeep * per;
        ps += step * kDeep * d.D;
    }
}

struct Layout {
    size_t states, sums, total;
};
Layout forward_layout(const Dims& d) {
    Layout l{};
    if (d.chunks > 1) {
        l.sums = align_up((size_t)d.B * d.chunks * d.N * d.D * sizeof(float), 256);
        l.total = l.sums + align_up((size_t)d.B * d.chunks * d.D * sizeof(float), 256);
    }
    return l;
}

template <typename T, int NB>
int forward(const Dims& d, const float* initial, T* y, float* final_state, float* kept, char* ws, hipStream_t s) {
    const Layout l = forward_layout(d);
    float *states = reinterpret_cast<float*>(ws + l.states), *sums = reinterpret_cast<float*>(ws + l.sums);
    const long long blocks = channel_blocks(d, 16) * d.B;
    if (d.chunks > 1) {
        hipLaunchKernelGGL((chunk_kernel<T, NB, true>), dim3((unsigned)(blocks * (d.chunks - 1))), dim3(64), 0, s, d, states,
                           sums, nullptr, nullptr, nullptr, nullptr);
        RKA_RETURN_IF_HIP(hipGetLastError());
        RKA_RETURN_IF_ERR(launch_join(d, states, sums, initial, false, s));
    }
    hipLaunchKernelGGL((chunk_kernel<T, NB, false>), dim3((unsigned)(blocks * d.chunks)), dim3(64), 0, s, d, states, nullptr,
                       initial, y, final_state, kept);
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}

template <typename T>
int forward(const Dims& d, const float* initial, void* y, float* final_state, float* kept, char* ws, hipStream_t s) {
    T* out = static_cast<T*>(y);
    switch (state_blocks(d.N)) {
        case 1: return forward<T, 1>(d, initial, out, final_state, kept, ws, s);
        case 2: return forward<T, 2>(d, initial, out, final_state, kept, ws, s);
        default: return forward<T, 4>(d, initial, out, final_state, kept, ws, s);
    }
}

}  // namespace

// Chunks for some eight wavefronts to a SIMD: 16384 tokens of 2048 channels take 475, 297, 252,
// 246 and 249 us with one, two, four, eight and sixteen, 16 x 1000 of 520 in float32 255, 168, 140,
// 128 and 121, training on 4 x 2048 of 2048 750, 511, 466, 466 and 482.  At least four tiles: what
// a chunk's state costs in memory is then a third of its tokens' at most.
int chunk_tokens(int tokens, long long waves) {
    constexpr long long kWant = 8192;
    const long long chunks = std::max(1LL, kWant / std::max(1LL, waves));
    if (chunks == 1) return std::max(1, tiles_of(tokens)) * kTile;
    const int tiles = std::max(4, (int)((tiles_of(tokens) + chunks - 1) / chunks));
    return tiles * kTile;
}

int check_launches(const char* what, const Dims& d, bool training) {
    const long long chunks = (long long)d.B * d.chunks;
    RKA_RETURN_IF_ERR(check_grid(channel_blocks(d, 16) * chunks, 64, what));
    if (d.chunks > 1) RKA_RETURN_IF_ERR(check_grid(((long long)d.B * d.N * d.D + 255) / 256, 256, what));
    return training ? check_grid(channel_blocks(d, kChannels) * chunks, kWaves * 64, what) : 0;
}

int launch_join(const Dims& d, float* own, const float* sums, const float* first, bool backward, hipStream_t s) {
    const long long blocks = ((long long)d.B * d.N * d.D + 255) / 256;
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)blocks), dim3(256), 0, s, d, own, sums, first, backward ? 1 : 0);
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}

int make_dims(const char* what, int batch, int tokens, int channels, int states, int groups, Dims* d) {
    const std::string name(what);
    if (batch < 0 || tokens < 0) return fail(RKA_ERR_INVALID_ARGUMENT, name + ": batch and tokens must be >= 0");
    if (channels < 1 || states < 1 || groups < 1 || channels % groups != 0)
        return fail(RKA_ERR_INVALID_ARGUMENT, name + ": channels and states must be >= 1, channels a multiple of groups");
    if (states > kMaxStates) return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": more than 64 states per channel");
    // (what a kernel counts in 32 bits)
    if (tokens > (1 << 30)) return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": more than 2^30 tokens");
    *d = Dims{};
    d->B = batch;
    d->T = tokens;
    d->D = channels;
    d->N = states;
    d->G = groups;
    d->chunk = chunk_tokens(tokens, channel_blocks(*d, 16) * std::max(batch, 1));
    d->chunks = tokens > 0 ? (tokens - 1) / d->chunk + 1 : 1;
    return 0;
}

int set_call(const char* what, Dims* d, const void* x, const void* dt, const float* A, const void* Bm, const void* C,
             const float* skip, const void* gate, const float* bias, const int* lengths, const long long* strides, int softplus,
             int dtype) {
    RKA_RETURN_IF_ERR(check_dtype(dtype, what));
    if (!strides) return fail(RKA_ERR_INVALID_ARGUMENT, std::string(what) + ": null strides");
    if (!A || (d->B > 0 && d->T > 0 && (!x || !dt || !Bm || !C)))
        return fail(RKA_ERR_INVALID_ARGUMENT, std::string(what) + ": null tensor pointer");
    d->x = x;
    d->dt = dt;
    d->A = A;
    d->Bm = Bm;
    d->C = C;
    d->skip = skip;
    d->gate = gate;
    d->bias = bias;
    d->lengths = lengths;
    d->softplus = softplus;
    for (int i = 0; i < 2; ++i) {
        d->xs[i] = strides[i];
        d->ts[i] = strides[2 + i];
        d->zs[i] = strides[4 + i];
    }
    for (int i = 0; i < 3; ++i) {
        d->bs[i] = strides[6 + i];
        d->cs[i] = strides[9 + i];
    }
    if (d->D > kMaxStride) return fail(RKA_ERR_UNSUPPORTED_SHAPE, std::string(what) + ": more than 2^21 channels");
    for (const long long of_token : {d->xs[1], d->ts[1], d->zs[1], d->bs[1], d->cs[1]})
        if (d->T > 1 && (of_token < 0 || of_token > kMaxStride))
            return fail(RKA_ERR_UNSUPPORTED_SHAPE, std::string(what) + ": the strides of a token must be in [0, 2^21]");
    return 0;
}

}  // namespace scan
}  // namespace rka

using namespace rka;
using namespace rka::scan;

extern "C" {

size_t rka_selective_scan_forward_workspace_bytes(int batch, int tokens, int channels, int states, int groups) {
    Dims d;
    if (make_dims("selective_scan", batch, tokens, channels, states, groups, &d) != 0) return 0;
    return forward_layout(d).total;
}

size_t rka_selective_scan_reserve_bytes(int batch, int tokens, int channels, int states, int groups) {
    Dims d;
    if (make_dims("selective_scan", batch, tokens, channels, states, groups, &d) != 0) return 0;
    return (size_t)batch * tiles_of(tokens) * states * channels * sizeof(float);
}

int rka_selective_scan_forward(const void* x, const void* dt, const float* A, const void* B, const void* C, const float* skip,
                               const void* gate, const float* dt_bias, const float* initial_state, const int* lengths, void* y,
                               float* final_state, void* reserve, void* workspace, size_t workspace_bytes, int batch, int tokens,
                               int channels, int states, int groups, const long long* strides, int softplus, int dtype,
                               void* stream) {
    clear_error();
    Dims d;
    RKA_RETURN_IF_ERR(make_dims("selective_scan_forward", batch, tokens, channels, states, groups, &d));
    RKA_RETURN_IF_ERR(set_call("selective_scan_forward", &d, x, dt, A, B, C, skip, gate, dt_bias, lengths, strides, softplus, dtype));
    if (batch == 0) return 0;
    if ((tokens > 0 && !y) || !final_state) return fail(RKA_ERR_INVALID_ARGUMENT, "selective_scan_forward: null tensor pointer");
    RKA_RETURN_IF_ERR(check_launches("selective_scan_forward", d, reserve != nullptr));
    RKA_RETURN_IF_ERR(check_workspace(workspace, workspace_bytes, forward_layout(d).total, "selective_scan_forward"));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    float* kept = static_cast<float*>(reserve);
    return dtype == RKA_DTYPE_F32 ? forward<float>(d, initial_state, y, final_state, kept, ws, s)
                                  : forward<bf16>(d, initial_state, y, final_state, kept, ws, s);
}

}  // extern "C"
