// The gradients of the gated delta rule that are made for all chunks at once after the
// backward's chain (gated_delta.h has the formulas).
//
// A workgroup of eight wavefronts takes a chunk of a key head through its value heads
// and keeps the sums of dq and dk in registers: they are rounded once, in a fixed
// order, and nothing of a value head goes through memory.  A wavefront has 16 tokens'
// rows and half of Dk.  Over Dv, 32 columns at a time: the rows of dO and dX come from
// memory to the operand registers, the blocks of S, dS' and E are split into bf16 pieces
// once and shared through LDS, loaded a step ahead.
//
// Bound by latency, with one workgroup to a CU, whose registers and LDS the sums and the
// operands more than fill: 8192 tokens of 16 heads of 128x128 bf16 282 us, in which the matrix
// instructions are busy for 16% of the clocks.  624 MB are read and 99 written, 150 us of a
// copy; 65 of the MB written are registers spilled to memory (1024 workgroups of 512 lanes, 124
// bytes each), dq, dk, dg and dbeta are 35.  Bytes that a lane spills, with 16-byte loads
// and without: bf16 none at Dk up to 64, 124 and 188 to 128, 716 and 784 to 192, 1076 and
// 1176 to 256; float32 160 and 256, 504 and 548, 1068 and 1148, 1464 and 1512.  Holding the
// next head's first loads through what follows a head's last step spills more and took
// 347 us.
#include "gated_delta.h"

namespace rka {
namespace delta {
namespace {

constexpr int kThreads = 512;
constexpr int kLd = 68;  // row of a 64-wide LDS tile: 16 bytes past a multiple of all banks

// An element of q and one of k.
template <typename T>
struct Pair;
template <>
struct Pair<float> {
    float x, y;
    __device__ __forceinline__ void set(float a, float b) {
        x = a;
        y = b;
    }
    __device__ __forceinline__ float q() const { return made(x); }
    __device__ __forceinline__ float k() const { return made(y); }
};
template <>
struct Pair<bf16> {
    unsigned x;
    __device__ __forceinline__ void set(bf16 a, bf16 b) { x = (unsigned)b.bits << 16 | a.bits; }
    // (unpacked where it is used, not ahead of the loop into twice the registers)
    __device__ __forceinline__ unsigned here() const {
        unsigned y = x;
        asm volatile("" : "+v"(y));
        return y;
    }
    __device__ __forceinline__ float q() const { return __uint_as_float(here() << 16); }
    __device__ __forceinline__ float k() const { return __uint_as_float(here() & 0xffff0000u); }
};

// Sum over the 16 lanes that hold a row of a 16x16 block, by rotations within them (which
// pass no LDS, as shuffles do).
template <int N>
__device__ __forceinline__ float rotate(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x120 + N, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_sum(float x) {
    x += rotate<8>(x);
    x += rotate<4>(x);
    x += rotate<2>(x);
    x += rotate<1>(x);
    return x;
}

// Where four neighbouring columns (c of 32) of row `row` go among the fragments of a
// 32-wide step: 8 bytes per piece.
__device__ __forceinline__ void put_columns(u32x4* frags, int row, int c, f32x4 x) {
    u32x2 p[3];
    split<3>(x, p);
    u32x2* at = reinterpret_cast<u32x2*>(frags + (size_t)(row / 16) * 3 * kFragLanes + c / 8 * 16 + row % 16) + c / 4 % 2;
#pragma unroll
    for (int i = 0; i < 3; ++i) at[i * kFragLanes * 2] = p[i];
}

// KU: 32-wide steps over Dk (even).  VEC: Dv is a multiple of eight.
template <typename T, int KU, bool VEC>
__global__ __launch_bounds__(kThreads, 1) void gradients_kernel(Dims d, const T* q, const T* k, const T* dout, const void* g,
                                                                const int* lengths, ChunkData in, BackwardData bd, T* dq,
                                                                T* dk, void* dg, void* dbeta) {
    constexpr int NP = kPieces<T>, TB = 2 * KU, TH = KU;  // blocks of 16 rows of the state; a wavefront's
    constexpr int kRows = TB * 16, kN = kRows * 8 / kThreads;  // float4 of S (and dS') per thread and step
    constexpr int kFrags = (2 * TB + 4) * 3;                   // of a step: S, dS', E
    constexpr int kShared = kFrags * kFragLanes * 16 > 2 * kChunk * kLd * 4 ? kFrags * kFragLanes * 16 : 2 * kChunk * kLd * 4;
    __shared__ __attribute__((aligned(16))) char shared[kShared];
    // sums of dq and dk over the value heads, a lane's own: in LDS where they fit
    constexpr bool kSumsInLds = KU <= 4;
    __shared__ f32x4 lds_sums[kSumsInLds ? 2 * TH * kThreads : 1];
    f32x4 reg_sums[kSumsInLds ? 1 : 2 * TH];
    auto sum = [&](int which, int t) -> f32x4& {
        if constexpr (kSumsInLds)
            return lds_sums[(which * TH + t) * kThreads + threadIdx.x];
        else
            return reg_sums[which * TH + t];
    };
    __shared__ double gsum[kChunk];
    __shared__ float bet[kChunk], sums[2][4][kChunk], dots[8];
    u32x4* fs = reinterpret_cast<u32x4*>(shared);
    u32x4* fd = fs + TB * 3 * kFragLanes;
    u32x4* fe = fd + TB * 3 * kFragLanes;
    float* f1 = reinterpret_cast<float*>(shared);  // (after the steps)
    float* f2 = f1 + kChunk * kLd;
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 16, hi = lane / 16;
    const int w4 = wave % 4, half = wave / 4;
    const int c = blockIdx.x % d.chunks, bk = blockIdx.x / d.chunks, b = bk / d.Hk, hk = bk % d.Hk, rep = d.Hv / d.Hk;
    const int t0 = c * kChunk, live = min(kChunk, row_length(lengths, b, d.T) - t0), here = min(kChunk, d.T - t0);
    const size_t kch = blockIdx.x;
    if (live <= 0) {
        for (int i = tid; i < here * rep; i += kThreads) {
            const size_t at = ((size_t)b * d.T + t0 + i / rep) * d.Hv + hk * rep + i % rep;
            store_gate(dg, at, 0.f, d.gate_bf16);
            store_gate(dbeta, at, 0.f, d.gate_bf16);
        }
        for (int i = tid; i < here * d.Dk; i += kThreads) {
            const size_t at = (((size_t)b * d.T + t0 + i / d.Dk) * d.Hk + hk) * d.Dk + i % d.Dk;
            dq[at] = from_f32<T>(0.f);
            dk[at] = from_f32<T>(0.f);
        }
        return;
    }
    const float* norm = in.norm + kch * 2 * kChunk;
    const size_t turned = kch * row_frags<T>(d.Dk) * kFragLanes + lane;
    const long long vrow = (long long)d.Hv * d.Dv;
    const int first = 16 * w4 + 4 * hi;
    const f32x4 ck = *reinterpret_cast<const f32x4*>(norm + first), cq = *reinterpret_cast<const f32x4*>(norm + kChunk + first);
    // the rows of q and k, as a product leaves its blocks
    Pair<T> qk[TH][4];
#pragma unroll
    for (int t = 0; t < TH; ++t) {
        const int dim = min(16 * (half * TH + t) + n, d.Dk - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int tok = t0 + min(first + i, live - 1);
            const T none = from_f32<T>(0.f);
            const bool real = first + i < live && 16 * (half * TH + t) + n < d.Dk;
            const T x = q[b * d.q_s[0] + tok * d.q_s[1] + hk * d.q_s[2] + dim];
            const T y = k[b * d.k_s[0] + tok * d.k_s[1] + hk * d.k_s[2] + dim];
            qk[t][i].set(real ? x : none, real ? y : none);
        }
    }
    auto values = [&](int which, int t) {
        f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = which ? qk[t][i].k() * ck[i] : qk[t][i].q() * cq[i];
        return y;
    };
    f32x4 dot_q{}, dot_k{};
#pragma unroll
    for (int t = 0; t < TH; ++t) sum(0, t) = sum(1, t) = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int r = 0; r < rep; ++r) {
        const int h = hk * rep + r;
        const size_t ch = ((size_t)b * d.Hv + h) * d.chunks + c;
        const size_t row0 = ((size_t)b * d.T + t0) * d.Hv + h;  // token row of the [B, T, Hv] tensors
        const float* coef = in.coef + ch * kCoefFloats;
        // (a zero that the compiler does not know: what hangs on it stays in the loop,
        // where the addresses of every block of Dk would fill the registers)
        size_t zero = 0;
        asm volatile("" : "+s"(zero));
        // of the lane's rows as operands
        const bool on = 16 * w4 + n < live;
        const int token = min(16 * w4 + n, live - 1);
        const T* pdo = dout ? dout + row0 * d.Dv + token * vrow : nullptr;
        const float* pdx = bd.dx + row0 * d.Dv + token * vrow;
        const float* pe = bd.e + row0 * d.Dv;
        const float* ps = bd.states + ch * d.Dk * d.Dv;
        const float* pd = bd.dstates + ch * d.Dk * d.Dv;
        // of the next step: S, dS' and E as they will go to LDS, dO and dX
        f32x4 ns[kN], nd[kN], ne;
        Eight<T> no{};
        Eight<float> nx;
        auto load = [&](int v0) {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int x = tid + i * kThreads, row = min(x / 8, d.Dk - 1);
                ns[i] = load4<VEC>(ps + (size_t)row * d.Dv, v0 + x % 8 * 4, d.Dv);
                nd[i] = load4<VEC>(pd + (size_t)row * d.Dv, v0 + x % 8 * 4, d.Dv);
            }
            ne = load4<VEC>(pe + min(tid / 8, live - 1) * vrow, v0 + tid % 8 * 4, d.Dv);
            if (dout) no.template load<VEC>(pdo, v0 + 8 * hi, d.Dv);
            nx.template load<VEC>(pdx, v0 + 8 * hi, d.Dv);
        };
        f32x4 aq[TH] = {}, ar[TH] = {}, az[TH] = {}, af[4] = {};
        float dot = 0.f, gate = 0.f;
        load(0);
        if (wave == 0)
            gate = load_gate(g, b * d.g_s[0] + (t0 + min(lane, live - 1)) * d.g_s[1] + h * d.g_s[2], d.gate_bf16);
        for (int v0 = 0; v0 < d.Dv; v0 += 32) {
            u32x4 xo[NP], xx[3], xe[3];
            no.pieces(on && dout, xo);
            nx.pieces(on, xx);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int x = tid + i * kThreads;
                if (x / 8 >= d.Dk || v0 + x % 8 * 4 >= d.Dv) ns[i] = nd[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < 4; ++j) dot += ns[i][j] * nd[i][j];
                put_columns(fs, x / 8, x % 8 * 4, ns[i]);
                put_columns(fd, x / 8, x % 8 * 4, nd[i]);
            }
            put_columns(fe, tid / 8, tid % 8 * 4, tid / 8 < live && v0 + tid % 8 * 4 < d.Dv ? ne : f32x4{0.f, 0.f, 0.f, 0.f});
            __syncthreads();
            if (v0 + 32 < d.Dv) load(v0 + 32);
#pragma unroll
            for (int i = 0; i < 3; ++i) xe[i] = fe[(w4 * 3 + i) * kFragLanes + lane];
            // dO E^T by the one half of the wavefronts, dX E^T by the other
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j > w4) break;
                u32x4 y[3];
#pragma unroll
                for (int i = 0; i < 3; ++i) y[i] = fe[(j * 3 + i) * kFragLanes + lane];
                af[j] = half ? mul(xx, y, af[j]) : mul(xo, y, af[j]);
                settle(af[j]);
            }
#pragma unroll
            for (int t = 0; t < TH; ++t) {
                u32x4 ys[3], yd[3];
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    ys[i] = fs[((half * TH + t) * 3 + i) * kFragLanes + lane];
                    yd[i] = fd[((half * TH + t) * 3 + i) * kFragLanes + lane];
                }
                aq[t] = mul(xo, ys, aq[t]);
                ar[t] = mul(xx, ys, ar[t]);
                az[t] = mul(xe, yd, az[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int t = 0; t < TH; ++t) {
                settle(aq[t]);
                settle(ar[t]);
                settle(az[t]);
            }
        }
        if (wave == 0) {
            gsum[lane] = chunk_sum(lane < live ? gate : 0.f, lane);
            bet[lane] = coef[BETA * kChunk + lane];
        }
        __syncthreads();
        {
            float* f = half ? f2 : f1;
            const float by = half ? -1.f : d.scale;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = first + i, col = 16 * j + n;
                    const bool in_f = half ? row > col : row >= col;
                    const float w = made(expf((float)(gsum[row] - gsum[col])));
                    f[row * kLd + col] = in_f ? by * af[j][i] * w : 0.f;
                }
        }
        f32x4 eg, el, beta;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            eg[i] = expf((float)gsum[first + i]);
            el[i] = expf((float)(gsum[kChunk - 1] - gsum[first + i]));
            beta[i] = bet[first + i];
        }
        __syncthreads();
        // Rows of F1 B and F2 B (of the normalised keys), then of F1^T and F2^T (of the
        // normalised queries and keys): two at a time, and a block of Dk at a time, for
        // the registers' sake.  (The half of a triangle that is zero is multiplied too:
        // no branch between the products.)
        f32x4 rq{}, rk{}, rz{}, rw{};
        u32x4 x[2][2][3];
        auto operands = [&](auto value) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    f32x4 a[2];
#pragma unroll
                    for (int i = 0; i < 8; ++i) a[i / 4][i % 4] = value(m, 32 * w + 8 * hi + i);
                    split8<3>(a[0], a[1], x[m][w]);
                }
        };
        auto turned_frags = [&](const u32x4* from, int t, u32x4 (&y)[2][NP]) {
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < NP; ++i)
                    y[w][i] = from[zero + turned + ((size_t)((half * TH + t) * 2 + w) * NP + i) * kFragLanes];
        };
        // (loaded a block ahead)
        u32x4 yk[2][2][NP], yq[2][2][NP];
        turned_frags(in.kt, 0, yk[0]);
        operands([&](int m, int t) { return (m ? f2 : f1)[(16 * w4 + n) * kLd + t] * (bet[t] * norm[t]); });
#pragma unroll
        for (int t = 0; t < TH; ++t) {
            turned_frags(in.kt, (t + 1) % TH, yk[(t + 1) % 2]);
            if (t + 1 == TH) turned_frags(in.qt, 0, yq[0]);
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            aq[t] *= d.scale * eg;
            ar[t] *= -eg;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                aq[t] = mul(x[0][w], yk[t % 2][w], aq[t]);
                ar[t] = mul(x[1][w], yk[t % 2][w], ar[t]);
            }
            settle(aq[t]);
            settle(ar[t]);
            sum(0, t) += aq[t];
            sum(1, t) += ar[t];
            rq += aq[t] * values(0, t);
            rk += ar[t] * values(1, t);
        }
        operands([&](int m, int t) { return (m ? f2 : f1)[t * kLd + 16 * w4 + n] * norm[m ? t : kChunk + t]; });
#pragma unroll
        for (int t = 0; t < TH; ++t) {
            if (t + 1 < TH) {
                turned_frags(in.kt, t + 1, yk[(t + 1) % 2]);
                turned_frags(in.qt, t + 1, yq[(t + 1) % 2]);
            }
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            const f32x4 y = values(1, t);
            az[t] *= el;
            rw += az[t] * y;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                az[t] = mul(x[0][w], yq[t % 2][w], az[t]);
                az[t] = mul(x[1][w], yk[t % 2][w], az[t]);
            }
            settle(az[t]);
            rz += az[t] * y;
            sum(1, t) += beta * az[t];
        }
        dot_q += rq;
        dot_k += rk + beta * rz;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = row_sum(rq[i]), bb = row_sum(rk[i]), z = row_sum(rz[i]), w = row_sum(rw[i]);
            if (n == 0) {
                sums[half][0][first + i] = a;
                sums[half][1][first + i] = bb;
                sums[half][2][first + i] = z;
                sums[half][3][first + i] = w * beta[i];
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o *= 2) dot += __shfl_xor(dot, o);
        if (lane == 0) dots[wave] = dot;
        __syncthreads();
        if (wave == 0) {
            float w = sums[0][3][lane] + sums[1][3][lane];
#pragma unroll
            for (int o = 1; o < 64; o *= 2) w += __shfl_xor(w, o);
            const float db = sums[0][2][lane] + sums[1][2][lane];
            float v = (sums[0][0][lane] + sums[1][0][lane]) + (sums[0][1][lane] + sums[1][1][lane]) - bet[lane] * db;
            if (lane == 63) {
                float all = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) all += dots[i];
                v += w + expf((float)gsum[kChunk - 1]) * all;
            }
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                const float down = __shfl_down(v, o);
                if (lane + o < 64) v += down;
            }
            if (lane < here) {
                store_gate(dg, row0 + (size_t)lane * d.Hv, lane < live ? v : 0.f, d.gate_bf16);
                store_gate(dbeta, row0 + (size_t)lane * d.Hv, lane < live ? db : 0.f, d.gate_bf16);
            }
        }
        __syncthreads();
    }
    // The normalisation's gradient, dx = c (dy - y (y . dy)) with y = c x.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = row_sum(dot_q[i]), bb = row_sum(dot_k[i]);
        if (n == 0) {
            sums[half][0][first + i] = a;
            sums[half][1][first + i] = bb;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int tok = first + i;
        if (tok >= here) continue;
        const float yq = sums[0][0][tok] + sums[1][0][tok], yk = sums[0][1][tok] + sums[1][1][tok];
        const size_t to = (((size_t)b * d.T + t0 + tok) * d.Hk + hk) * d.Dk;
#pragma unroll
        for (int t = 0; t < TH; ++t) {
            const int dim = 16 * (half * TH + t) + n;
            if (dim >= d.Dk) continue;
            float vq = sum(0, t)[i], vk = sum(1, t)[i];
            if (d.normalize && tok < live) {
                vq = cq[i] * (vq - cq[i] * qk[t][i].q() * yq);
                vk = ck[i] * (vk - ck[i] * qk[t][i].k() * yk);
            }
            dq[to + dim] = from_f32<T>(tok < live ? vq : 0.f);
            dk[to + dim] = from_f32<T>(tok < live ? vk : 0.f);
        }
    }
}

}  // namespace

template <typename T>
int launch_gradients(const Dims& d, const T* q, const T* k, const T* dout, const void* g, const int* lengths,
                     const ChunkData& in, const BackwardData& bd, T* dq, T* dk, void* dg, void* dbeta,
                     hipStream_t stream) {
    const long long blocks = (long long)d.B * d.Hk * d.chunks;
    if (blocks == 0) return 0;
    RKA_RETURN_IF_ERR(check_grid(blocks, kThreads, "gated_delta_backward"));
    auto go = [&](auto ku) {
        constexpr int KU = decltype(ku)::value;
        if (d.Dv % 8 == 0)
            hipLaunchKernelGGL((gradients_kernel<T, KU, true>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, d, q, k,
                               dout, g, lengths, in, bd, dq, dk, dg, dbeta);
        else
            hipLaunchKernelGGL((gradients_kernel<T, KU, false>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, d, q, k,
                               dout, g, lengths, in, bd, dq, dk, dg, dbeta);
    };
    switch (chain_steps(d.Dk)) {
        case 2: go(std::integral_constant<int, 2>{}); break;
        case 4: go(std::integral_constant<int, 4>{}); break;
        case 6: go(std::integral_constant<int, 6>{}); break;
        default: go(std::integral_constant<int, 8>{}); break;
    }
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}
template int launch_gradients<float>(const Dims&, const float*, const float*, const float*, const void*, const int*,
                                     const ChunkData&, const BackwardData&, float*, float*, void*, void*, hipStream_t);
template int launch_gradients<bf16>(const Dims&, const bf16*, const bf16*, const bf16*, const void*, const int*,
                                    const ChunkData&, const BackwardData&, bf16*, bf16*, void*, void*, hipStream_t);

}  // namespace delta
}  // namespace rka
