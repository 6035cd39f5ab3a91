// The gradients of the selective scan (selective_scan.h has the formulas and the split).
//
// Each tile's start state was kept by the forward: a tile's states are made again from it, on
// their way into LDS, and met from there backwards.  Sums over channels (dB, dC) go through
// the lanes of a channel block, then over a workgroup's four blocks in LDS, then over the
// workgroups by a launch of their own, always in the same order.
//
// 4 x 2048 tokens of 2048 channels, 16 states, bf16: chunks' ends 60 us, gradients 270, the sums
// behind them 12.  Bound by vector instructions, some 105 a token and lane (16 of them the sums
// over channels), at two wavefronts to a SIMD, which is what the states in LDS leave.  From 33 states
// on LDS and registers leave one: 4 x 2048 tokens of 1024 channels 177 us backward with 16 states, 304 with
// 32, 803 with 48, 818 with 64.
#include "selective_scan.h"

#include <algorithm>

namespace rka {
namespace scan {
namespace {

// Where a workgroup stands.
struct Place {
    int g, ch, b, chunk, len, t0, t1, t_end, block;
    bool on;
    size_t at;
};
__device__ __forceinline__ Place place(const Dims& d, int width, int skipped) {
    Place p;
    const int Dg = d.D / d.G, per_group = (Dg - 1) / width + 1, blocks = d.G * per_group, chunks = d.chunks - skipped;
    const long long id = in_order();
    p.block = (int)(id % blocks);
    p.chunk = (int)(id / blocks % chunks) + skipped;
    p.b = (int)(id / blocks / chunks);
    p.g = p.block / per_group;
    const int in = p.block % per_group * width + threadIdx.x / 64 * 16 + threadIdx.x % 16;
    p.on = in < Dg;
    p.ch = p.g * Dg + min(in, Dg - 1);
    p.len = row_length(d.lengths, p.b, d.T);
    p.t0 = p.chunk * d.chunk;
    p.t_end = min(d.T, p.t0 + d.chunk);
    p.t1 = min(p.len, p.t_end);
    p.at = (size_t)p.b * d.chunks + p.chunk;
    return p;
}

// A chunk's own part of the gradient of the state at its start, and the sum of its steps.
template <typename T, int NB>
__global__ __launch_bounds__(64) void ends_kernel(Dims d, const T* dy, float* own, float* sums) {
    __shared__ __attribute__((aligned(16))) float steps[16][2 * kTile + 4];  // of a channel: s; r
    __shared__ __attribute__((aligned(16))) float ct[kTile][NB * 16];
    const int lane = threadIdx.x, c = lane % 16, nl = lane / 16;
    const Place p = place(d, 16, 1);
    f32x4 a2[NB], dh[NB];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        a2[k] = finite_rates(load_states_of(d.A + (size_t)p.ch * d.N, 16 * k + 4 * nl, d.N));
        dh[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float bias = d.bias ? d.bias[p.ch] : 0.f;
    const T* pt = static_cast<const T*>(d.dt) + p.b * d.ts[0];
    const T* pz = static_cast<const T*>(d.gate) + p.b * d.zs[0];
    const T* pd = dy ? dy + (size_t)p.b * d.T * d.D : nullptr;
    const T* pc = static_cast<const T*>(d.C) + p.b * d.cs[0] + p.g * d.cs[2];
    float sum = 0.f;
    Rows<T> dt, gate, up, cv[NB];
    Offsets ot, oz, od, oc[NB];
    auto set = [&](int rows) {
        ot.set(d.ts[1], p.ch, rows, sizeof(T));
        if (d.gate) oz.set(d.zs[1], p.ch, rows, sizeof(T));
        od.set(d.D, p.ch, rows, sizeof(T));
#pragma unroll
        for (int k = 0; k < NB; ++k) oc[k].set(d.cs[1], min(16 * k + c, d.N - 1), rows, sizeof(T));
    };
    auto load = [&](int t) {
        dt.load(pt + t * d.ts[1], ot);
        if (d.gate) gate.load(pz + t * d.zs[1], oz);
        if (pd) up.load(pd + (size_t)t * d.D, od);
#pragma unroll
        for (int k = 0; k < NB; ++k) cv[k].load(pc + t * d.cs[1], oc[k]);
    };
    const int last = p.t0 + (p.t1 - 1 - p.t0) / kTile * kTile;
    if (p.t0 < p.t1) {
        set(p.t1 - last);
        load(last);
        set(kTile);
    }
    for (int t = p.t0 < p.t1 ? last : p.t0 - 1; t >= p.t0; t -= kTile) {
        const int rows = p.t1 - t - 4 * nl;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 4 * nl + r;
            const bool live = r < rows;
            float slope, s = to_f32(dt.v[r]) + bias;
            if (d.softplus) s = softplus<T>(s, &slope);
            s = live ? s : 0.f;
            float dr = pd ? to_f32(up.v[r]) : 0.f;
            if (d.gate) dr *= to_f32(gate.v[r]) * sigmoid_of<T>(to_f32(gate.v[r]));
            sum += s;
            steps[c][row] = s;
            steps[c][kTile + row] = live ? dr : 0.f;
#pragma unroll
            for (int k = 0; k < NB; ++k) ct[row][16 * k + c] = live && 16 * k + c < d.N ? to_f32(cv[k].v[r]) : 0.f;
        }
        __syncthreads();
        if (t > p.t0) load(t - kTile);
        const float *ps = &steps[c][kTile - 4], *pq = &ct[kTile - 4][4 * nl];
#pragma unroll 1
        for (int q = 0; q < 4; ++q, ps -= 4, pq -= 64 * NB) {
            const f32x4 s4 = load4(ps), r4 = load4(ps + kTile);
#pragma unroll
            for (int i = 3; i >= 0; --i)
#pragma unroll
                for (int k = 0; k < NB; ++k) {
                    const f32x4 cq = load4(pq + 16 * (NB * i + k));
#pragma unroll
                    for (int j = 0; j < 4; ++j) dh[k][j] = fmaf(r4[i], cq[j], dh[k][j]) * __builtin_amdgcn_exp2f(s4[i] * a2[k][j]);
                }
        }
        __syncthreads();
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (!p.on) return;
    if (nl == 0) sums[p.at * d.D + p.ch] = sum;
#pragma unroll
    for (int k = 0; k < NB; ++k) store_states(own + p.at * d.N * d.D, 16 * k + 4 * nl, d.N, d.D, p.ch, dh[k]);
}

template <int CTRL>
__device__ __forceinline__ float from_lane(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
// Sums of eight values over the 16 lanes of a row: lane c ends with the one numbered c / 2.
// At each step a lane passes on the half that its partner keeps.  The first two steps' partners,
// c ^ 8 and c ^ 7, have them in other groups of four lanes: an addition for all lanes and one for
// the groups that keep the other value, where selects would take a third instruction.  (Written
// out, as the compiler has no masked addition.  Its inputs are read from other lanes two states
// after they are there, and so is what the first step leaves for the second.)
__device__ __forceinline__ float row_sums(const float (&v)[8]) {
    const int c = threadIdx.x % 16;
    float a0, a1, a2, a3, b0, b1;
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %6, %6 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %1, %7, %7 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %2, %8, %8 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %3, %9, %9 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %0, %10, %10 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %1, %11, %11 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %2, %12, %12 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %3, %13, %13 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %4, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %5, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %4, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
        "v_add_f32_dpp %5, %3, %3 row_half_mirror row_mask:0xf bank_mask:0xa"
        : "=&v"(a0), "=&v"(a1), "=&v"(a2), "=&v"(a3), "=&v"(b0), "=&v"(b1)
        : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[4]), "v"(v[5]), "v"(v[6]), "v"(v[7]));
    const float s = (c & 2 ? b1 : b0) + from_lane<0x4e>(c & 2 ? b0 : b1);  // c ^ 2
    return s + from_lane<0xb1>(s);  // c ^ 1
}

template <typename T>
struct Grads {
    T *x, *dt, *gate;
    float* bc;       // [channel blocks][B][T][dB, dC][N]
    float* a;        // [B][chunks][N][D]
    float* vec;      // [B][chunks][skip, bias][D]
    float* initial;  // [B][D][N] or null
};

template <typename T, int NB>
__global__ __launch_bounds__(kWaves * 64) void grads_kernel(Dims d, const float* kept, const float* ends, const float* dfinal,
                                                            const T* dy, Grads<T> out) {
    // The states before each token; then, in each token's first 32 numbers, its dB and dC
    // over the wavefront's channels.
    __shared__ __attribute__((aligned(16))) f32x4 before[kWaves][kTile][64];
    __shared__ __attribute__((aligned(16))) float steps[kWaves][16][3 * kTile + (NB == 1 ? 8 : 0)];  // of a channel: s; r; s x (two workgroups to a CU up to NB 2)
    __shared__ __attribute__((aligned(16))) float bt[kTile][NB * 16], ct[kTile][NB * 16];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = lane % 16, nl = lane / 16;
    const Place p = place(d, kChannels, 0);
    const int tiles = (d.T - 1) / kTile + 1;
    f32x4 a2[NB], dh[NB], da[NB], h[NB];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        const int n0 = 16 * k + 4 * nl;
        a2[k] = finite_rates(load_states_of(d.A + (size_t)p.ch * d.N, n0, d.N));
        dh[k] = da[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (d.chunks > 1)
            dh[k] = load_states(ends + p.at * d.N * d.D, n0, d.N, d.D, p.ch);
        else if (dfinal)
            dh[k] = load_states_of(dfinal + ((size_t)p.b * d.D + p.ch) * d.N, n0, d.N);
    }
    const float bias = d.bias ? d.bias[p.ch] : 0.f, skip = d.skip ? d.skip[p.ch] : 0.f;
    const T* px = static_cast<const T*>(d.x) + p.b * d.xs[0];
    const T* pt = static_cast<const T*>(d.dt) + p.b * d.ts[0];
    const T* pz = static_cast<const T*>(d.gate) + p.b * d.zs[0];
    const T* pd = dy ? dy + (size_t)p.b * d.T * d.D : nullptr;
    const T* pb = static_cast<const T*>(d.Bm) + p.b * d.bs[0] + p.g * d.bs[2];
    const T* pc = static_cast<const T*>(d.C) + p.b * d.cs[0] + p.g * d.cs[2];
    Rows<T> xv, dt, gate, up;
    Offsets ox, ot, oz, od, oy;
    T bv[NB], cv[NB];
    unsigned ob[NB], oc[NB], oh[4];
    const int btoken = threadIdx.x / 16;  // B and C are staged by all wavefronts
    auto set = [&](int rows) {
        ox.set(d.xs[1], p.ch, rows, sizeof(T));
        ot.set(d.ts[1], p.ch, rows, sizeof(T));
        if (d.gate) oz.set(d.zs[1], p.ch, rows, sizeof(T));
        od.set(d.D, p.ch, rows, sizeof(T));
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const unsigned n = min(16 * k + c, d.N - 1), row = min(btoken, rows - 1);
            ob[k] = (row * (unsigned)d.bs[1] + n) * (unsigned)sizeof(T);
            oc[k] = (row * (unsigned)d.cs[1] + n) * (unsigned)sizeof(T);
        }
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) oh[j] = ((unsigned)(4 * nl + j) * (unsigned)d.D + (unsigned)p.ch) * 4u;
    auto load = [&](int t) {
        xv.load(px + t * d.xs[1], ox);
        dt.load(pt + t * d.ts[1], ot);
        if (d.gate) gate.load(pz + t * d.zs[1], oz);
        if (pd) up.load(pd + (size_t)t * d.D, od);
        const float* from = kept + ((size_t)p.b * tiles + t / kTile) * d.N * d.D;
        const Memory fb(pb + t * d.bs[1]), fc(pc + t * d.cs[1]);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            fb.load(&bv[k], ob[k]);
            fc.load(&cv[k], oc[k]);
            const Memory fh(from + (size_t)16 * k * d.D);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v = 0.f;
                if (16 * k + 4 * nl + j < d.N) fh.load(&v, oh[j]);
                h[k][j] = v;
            }
        }
    };
    float dskip = 0.f, dbias = 0.f;
    const int last = p.t0 + (p.t1 - 1 - p.t0) / kTile * kTile;
    oy.set(d.D, p.ch, kTile, sizeof(T));
    if (p.t0 < p.t1) {
        set(p.t1 - last);
        load(last);
        set(kTile);
    }
    for (int t = p.t0 < p.t1 ? last : p.t0 - 1; t >= p.t0; t -= kTile) {
        const int rows = p.t1 - t - 4 * nl;
        // (a token behind the last has a step, an upper gradient, B and C of 0: it adds nothing)
        float x[4], s[4], slope[4], z[4], u[4], dr[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 4 * nl + r;
            const bool live = r < rows && p.on;
            s[r] = to_f32(dt.v[r]) + bias;
            slope[r] = 1.f;
            if (d.softplus) s[r] = softplus<T>(s[r], &slope[r]);
            s[r] = r < rows ? s[r] : 0.f;
            x[r] = live ? to_f32(xv.v[r]) : 0.f;
            z[r] = d.gate ? to_f32(gate.v[r]) : 0.f;
            u[r] = live && pd ? to_f32(up.v[r]) : 0.f;
            dr[r] = d.gate && live ? u[r] * z[r] * sigmoid_of<T>(z[r]) : u[r];
            steps[wave][c][row] = s[r];
            steps[wave][c][kTile + row] = dr[r];
            steps[wave][c][2 * kTile + row] = s[r] * x[r];
        }
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const bool is = t + btoken < p.t1 && 16 * k + c < d.N;
            bt[btoken][16 * k + c] = is ? to_f32(bv[k]) : 0.f;
            ct[btoken][16 * k + c] = is ? to_f32(cv[k]) : 0.f;
        }
        f32x4 start[NB];
#pragma unroll
        for (int k = 0; k < NB; ++k) start[k] = h[k];
        __syncthreads();
        if (t > p.t0) load(t - kTile);
        f32x4 read{0.f, 0.f, 0.f, 0.f}, q1 = read, q2 = read;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            if (k > 0) __syncthreads();  // the sums of the block before are out
            f32x4 hk = start[k];
            const int n0 = 16 * k + 4 * nl;
            // (addresses from one place for four tokens: each array's own would cost an addition a token)
            const float *ps = &steps[wave][c][0], *pbt = &bt[0][n0], *pct = &ct[0][n0];
            f32x4* ph = &before[wave][0][lane];
            float* sums = reinterpret_cast<float*>(&before[wave][0][0]) + nl * 8 + c / 2;
            f32x4 reads, q1s, q2s;
#pragma unroll 1
            for (int q = 0; q < 4; ++q, ps += 4, pbt += 64 * NB, pct += 64 * NB, ph += 4 * 64) {
                const f32x4 s4 = load4(ps), i4 = load4(ps + 2 * kTile);
                float parts[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 bq = load4(pbt + 16 * NB * i), cq = load4(pct + 16 * NB * i);
                    ph[64 * i] = hk;
                    float part = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        hk[j] = fmaf(__builtin_amdgcn_exp2f(s4[i] * a2[k][j]), hk[j], i4[i] * bq[j]);
                        part = fmaf(cq[j], hk[j], part);
                    }
                    parts[i] = part;
                }
                reads = f32x4{reads[1], reads[2], reads[3], token_sums(parts[0], parts[1], parts[2], parts[3])};
            }
            sums += kTile * 256;
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
                ps -= 4, pbt -= 64 * NB, pct -= 64 * NB, ph -= 4 * 64, sums -= 4 * 256;
                float of_b[4], of_a[4];
                const f32x4 s4 = load4(ps), r4 = load4(ps + kTile), i4 = load4(ps + 2 * kTile);
#pragma unroll
                for (int i = 3; i >= 0; --i) {
                    const f32x4 bq = load4(pbt + 16 * NB * i), cq = load4(pct + 16 * NB * i), hp = ph[64 * i];
                    float v[8];
                    of_b[i] = of_a[i] = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float full = fmaf(r4[i], cq[j], dh[k][j]);
                        v[j] = i4[i] * full;
                        v[4 + j] = r4[i] * hk[j];
                        of_b[i] = fmaf(full, bq[j], of_b[i]);
                        dh[k][j] = full * __builtin_amdgcn_exp2f(s4[i] * a2[k][j]);
                        const float w = dh[k][j] * hp[j];
                        of_a[i] = fmaf(w, a2[k][j], of_a[i]);
                        da[k][j] = fmaf(w, s4[i], da[k][j]);
                    }
                    hk = hp;
                    sums[256 * i] = row_sums(v);  // (two lanes write the same)
                }
                q1s = f32x4{token_sums(of_b[0], of_b[1], of_b[2], of_b[3]), q1s[0], q1s[1], q1s[2]};
                q2s = f32x4{token_sums(of_a[0], of_a[1], of_a[2], of_a[3]), q2s[0], q2s[1], q2s[2]};
            }
            own_tokens(&reads);
            own_tokens(&q1s);
            own_tokens(&q2s);
            read += reads, q1 += q1s, q2 += q2s;
            __syncthreads();
            // 32 sums of 16 tokens, two to a thread
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int token = threadIdx.x / 32 + 8 * j, i = threadIdx.x % 32, n = 16 * k + i / 8 * 4 + i % 4;
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) sum += reinterpret_cast<const float*>(&before[w][token][0])[i];
                if (t + token < p.t1 && n < d.N)
                    out.bc[(((size_t)p.block * d.B + p.b) * d.T + t + token) * 2 * d.N + (i / 4 % 2 ? d.N : 0) + n] = sum;
            }
        }
        const size_t first = ((size_t)p.b * d.T + t) * d.D;
        const int room = p.t_end - t - 4 * nl;
        const Memory to_x(out.x + first), to_dt(out.dt + first), to_gate(out.gate + first);
        auto put = [&](const Memory& to, int r, float v) {
            if (p.on && r < room) to.store(from_f32<T>(r < rows ? v : 0.f), oy.at[r]);
        };
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float dx = fmaf(s[r], q1[r], skip * dr[r]);
            // (a2 is A log2(e))
            const float ddt = slope[r] * fmaf(x[r], q1[r], 0.6931471805599453f * q2[r]);
            if (r < rows) {
                dskip = fmaf(dr[r], x[r], dskip);
                dbias += ddt;
            }
            put(to_x, r, dx);
            put(to_dt, r, ddt);
            if (d.gate) {
                const float sig = sigmoid_of<T>(z[r]);
                put(to_gate, r, u[r] * fmaf(skip, x[r], read[r]) * sig * (1.f + z[r] * (1.f - sig)));
            }
        }
    }
    // tokens behind the row's end
    const int rest = p.t1 <= p.t0 ? p.t0 : last + kTile;
    if (p.on) {
        for (int t = rest + nl; t < p.t_end; t += 4) {
            const size_t i = ((size_t)p.b * d.T + t) * d.D + p.ch;
            out.x[i] = out.dt[i] = from_f32<T>(0.f);
            if (d.gate) out.gate[i] = from_f32<T>(0.f);
        }
    }
    dskip += __shfl_xor(dskip, 16);
    dskip += __shfl_xor(dskip, 32);
    dbias += __shfl_xor(dbias, 16);
    dbias += __shfl_xor(dbias, 32);
    if (!p.on) return;
    if (nl == 0) {
        out.vec[(p.at * 2) * d.D + p.ch] = dskip;
        out.vec[(p.at * 2 + 1) * d.D + p.ch] = dbias;
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        const int n0 = 16 * k + 4 * nl;
        store_states(out.a + p.at * d.N * d.D, n0, d.N, d.D, p.ch, da[k]);
        if (out.initial && p.chunk == 0) store_states_of(out.initial + ((size_t)p.b * d.D + p.ch) * d.N, n0, d.N, dh[k]);
    }
}

// dB and dC [B][T][G][N] over a group's channel blocks.
template <typename T>
__global__ __launch_bounds__(256) void inputs_kernel(Dims d, const float* bc, int per_group, T* dB, T* dC) {
    const long long width = 2LL * d.N, total = (long long)d.B * d.T * d.G * width;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int in = (int)(i % width), g = (int)(i / width % d.G);
        const long long row = i / width / d.G;
        const int b = (int)(row / d.T), t = (int)(row % d.T);
        float sum = 0.f;
        if (t < row_length(d.lengths, b, d.T)) {
            const float* p = bc + ((size_t)g * per_group * d.B * d.T + row) * width + in;
#pragma unroll 8
            for (int k = 0; k < per_group; ++k) sum += p[(size_t)k * d.B * d.T * width];
        }
        (in < d.N ? dB : dC)[(row * d.G + g) * d.N + in % d.N] = from_f32<T>(sum);
    }
}

// dA, dskip and dbias over batch rows and chunks.
__global__ __launch_bounds__(256) void weights_kernel(Dims d, const float* a, const float* vec, float* dA, float* dskip,
                                                      float* dbias) {
    const int ch = blockIdx.x * 64 + threadIdx.x % 64, n = blockIdx.y, part = threadIdx.x / 64, count = d.B * d.chunks;
    __shared__ float sums[3][64];
    float sum = 0.f;
    if (ch < d.D) {
        const float* p = n < d.N ? a + (size_t)n * d.D + ch : vec + (size_t)(n - d.N) * d.D + ch;
        const size_t step = (size_t)(n < d.N ? d.N : 2) * d.D;
#pragma unroll 8
        for (int i = part; i < count; i += 4) sum += p[i * step];
    }
    if (part > 0) sums[part - 1][threadIdx.x % 64] = sum;
    __syncthreads();
    if (part > 0 || ch >= d.D) return;
    for (int k = 0; k < 3; ++k) sum += sums[k][threadIdx.x];
    if (n < d.N) {
        if (dA) dA[(size_t)ch * d.N + n] = sum;
    } else {
        float* to = n == d.N ? dskip : dbias;
        if (to) to[ch] = sum;
    }
}

struct Layout {
    size_t ends, sums, bc, a, vec, total;
};
Layout backward_layout(const Dims& d) {
    Layout l{};
    const size_t chunks = (size_t)d.B * d.chunks;
    l.sums = l.ends + (d.chunks > 1 ? align_up(chunks * d.N * d.D * sizeof(float), 256) : 0);
    l.bc = l.sums + (d.chunks > 1 ? align_up(chunks * d.D * sizeof(float), 256) : 0);
    l.a = l.bc + align_up((size_t)channel_blocks(d, kChannels) * d.B * d.T * 2 * d.N * sizeof(float), 256);
    l.vec = l.a + align_up(chunks * d.N * d.D * sizeof(float), 256);
    l.total = l.vec + align_up(chunks * 2 * d.D * sizeof(float), 256);
    return l;
}

template <typename T, int NB>
int backward(const Dims& d, const float* kept, const T* dy, const float* dfinal, Grads<T> out, T* dB, T* dC, float* dA,
             float* dskip, float* dbias, char* ws, hipStream_t s) {
    const Layout l = backward_layout(d);
    float *ends = reinterpret_cast<float*>(ws + l.ends), *sums = reinterpret_cast<float*>(ws + l.sums);
    out.bc = reinterpret_cast<float*>(ws + l.bc);
    out.a = reinterpret_cast<float*>(ws + l.a);
    out.vec = reinterpret_cast<float*>(ws + l.vec);
    const long long small = channel_blocks(d, 16) * d.B * d.chunks, large = channel_blocks(d, kChannels) * d.B * d.chunks;
    if (d.chunks > 1) {
        hipLaunchKernelGGL((ends_kernel<T, NB>), dim3((unsigned)(small / d.chunks * (d.chunks - 1))), dim3(64), 0, s, d, dy, ends,
                           sums);
        RKA_RETURN_IF_HIP(hipGetLastError());
        RKA_RETURN_IF_ERR(launch_join(d, ends, sums, dfinal, true, s));
    }
    hipLaunchKernelGGL((grads_kernel<T, NB>), dim3((unsigned)large), dim3(kWaves * 64), 0, s, d, kept, ends, dfinal, dy, out);
    RKA_RETURN_IF_HIP(hipGetLastError());
    const long long items = std::min(((long long)d.B * d.T * d.G * 2 * d.N + 255) / 256, 1LL << 23);
    if (items > 0) {
        hipLaunchKernelGGL((inputs_kernel<T>), dim3((unsigned)items), dim3(256), 0, s, d, out.bc,
                           (int)(channel_blocks(d, kChannels) / d.G), dB, dC);
        RKA_RETURN_IF_HIP(hipGetLastError());
    }
    hipLaunchKernelGGL(weights_kernel, dim3((unsigned)((d.D - 1) / 64 + 1), (unsigned)(d.N + 2)), dim3(256), 0, s, d, out.a,
                       out.vec, dA, dskip, dbias);
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}

template <typename T>
int backward(const Dims& d, const float* kept, const void* dy, const float* dfinal, void* dx, void* ddt, void* dgate, void* dB,
             void* dC, float* dA, float* dskip, float* dbias, float* dinitial, char* ws, hipStream_t s) {
    const Grads<T> out{static_cast<T*>(dx), static_cast<T*>(ddt), static_cast<T*>(dgate), nullptr, nullptr, nullptr, dinitial};
    T *tB = static_cast<T*>(dB), *tC = static_cast<T*>(dC);
    const T* up = static_cast<const T*>(dy);
    switch (state_blocks(d.N)) {
        case 1: return backward<T, 1>(d, kept, up, dfinal, out, tB, tC, dA, dskip, dbias, ws, s);
        case 2: return backward<T, 2>(d, kept, up, dfinal, out, tB, tC, dA, dskip, dbias, ws, s);
        default: return backward<T, 4>(d, kept, up, dfinal, out, tB, tC, dA, dskip, dbias, ws, s);
    }
}

}  // namespace
}  // namespace scan
}  // namespace rka

using namespace rka;
using namespace rka::scan;

extern "C" {

size_t rka_selective_scan_backward_workspace_bytes(int batch, int tokens, int channels, int states, int groups) {
    Dims d;
    if (make_dims("selective_scan", batch, tokens, channels, states, groups, &d) != 0) return 0;
    return backward_layout(d).total;
}

int rka_selective_scan_backward(const void* x, const void* dt, const float* A, const void* B, const void* C, const float* skip,
                                const void* gate, const float* dt_bias, const int* lengths, const void* reserve,
                                const void* grad_y, const float* grad_final_state, void* grad_x, void* grad_dt, float* grad_A,
                                void* grad_B, void* grad_C, float* grad_skip, void* grad_gate, float* grad_dt_bias,
                                float* grad_initial_state, void* workspace, size_t workspace_bytes, int batch, int tokens,
                                int channels, int states, int groups, const long long* strides, int softplus, int dtype,
                                void* stream) {
    clear_error();
    Dims d;
    RKA_RETURN_IF_ERR(make_dims("selective_scan_backward", batch, tokens, channels, states, groups, &d));
    RKA_RETURN_IF_ERR(set_call("selective_scan_backward", &d, x, dt, A, B, C, skip, gate, dt_bias, lengths, strides, softplus, dtype));
    if (batch < 1) return fail(RKA_ERR_INVALID_ARGUMENT, "selective_scan_backward: batch must be >= 1");
    if (!reserve || (tokens > 0 && (!grad_x || !grad_dt || !grad_B || !grad_C || (gate && !grad_gate))))
        return fail(RKA_ERR_INVALID_ARGUMENT, "selective_scan_backward: null tensor pointer");
    RKA_RETURN_IF_ERR(check_launches("selective_scan_backward", d, true));
    RKA_RETURN_IF_ERR(check_workspace(workspace, workspace_bytes, backward_layout(d).total, "selective_scan_backward"));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const float* kept = static_cast<const float*>(reserve);
    char* ws = static_cast<char*>(workspace);
    return dtype == RKA_DTYPE_F32
               ? backward<float>(d, kept, grad_y, grad_final_state, grad_x, grad_dt, grad_gate, grad_B, grad_C, grad_A, grad_skip,
                                 grad_dt_bias, grad_initial_state, ws, s)
               : backward<bf16>(d, kept, grad_y, grad_final_state, grad_x, grad_dt, grad_gate, grad_B, grad_C, grad_A, grad_skip,
                                grad_dt_bias, grad_initial_state, ws, s);
}

}  // extern "C"
