// The gated delta rule (gated_delta.h has the formulas): entry points, and what is made
// for all chunks at once before the chains.
#include "gated_delta.h"

#include <algorithm>

namespace rka {
namespace delta {
namespace {

constexpr int kThreads = 256;

// A chunk's q (which = 1) or k (0) as fragments, by rows and transposed, and what
// normalises its rows.  The chunk is staged in LDS once, as it is.  VEC: Dk is a multiple
// of eight.  Bound by memory and the launch's ends: 16384 tokens of 8 heads of 128 bf16
// (67 MB read, 102 written) 40 us, 4.2 TB/s.  (In bf16 the fragments by rows are
// q's and k's own 16 bytes, two thirds of what is written.)
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void rows_kernel(Dims d, const T* q, const T* k, const int* lengths, ChunkData out) {
    constexpr int NP = kPieces<T>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    T* rows = reinterpret_cast<T*>(lds);
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, n = lane % 16, hi = lane / 16;
    const int which = blockIdx.x % 2, kch = blockIdx.x / 2, c = kch % d.chunks, bk = kch / d.chunks;
    const int b = bk / d.Hk, hk = bk % d.Hk, t0 = c * kChunk;
    const int live = min(kChunk, row_length(lengths, b, d.T) - t0);
    if (live <= 0) return;
    const int steps = chain_steps(d.Dk), width = steps * 32, ld = width + 8;
    const long long* st = which ? d.q_s : d.k_s;
    const T* src = (which ? q : k) + b * st[0] + t0 * st[1] + hk * st[2];
    // (four loads at a time)
    for (int i = tid; i < kChunk * width / 8; i += 4 * kThreads) {
        Eight<T> x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = min(i + j * kThreads, kChunk * width / 8 - 1), r = min(at / (width / 8), live - 1);
            x[j].template load<VEC>(src + r * st[1], at % (width / 8) * 8, d.Dk);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = i + j * kThreads, r = at / (width / 8);
            if (at < kChunk * width / 8) x[j].store(r < live, rows + r * ld + at % (width / 8) * 8);
        }
    }
    __syncthreads();
    {
        float x2 = 0.f;
        for (int e = tid % 4; e < d.Dk; e += 4) {
            const float x = to_f32(rows[tid / 4 * ld + e]);
            x2 += x * x;
        }
        x2 += __shfl_xor(x2, 1);
        x2 += __shfl_xor(x2, 2);
        if (tid % 4 == 0)
            out.norm[((size_t)kch * 2 + which) * kChunk + tid / 4] = d.normalize ? 1.f / sqrtf(x2 + kNormEps) : 1.f;
    }
    const size_t at = (size_t)kch * row_frags<T>(d.Dk) * kFragLanes;
    u32x4* byrow = (which ? out.q : out.k) + at;
    for (int f = wave; f < 4 * steps; f += kThreads / 64) {
        const T* p = rows + (f / steps * 16 + n) * ld + f % steps * 32 + 8 * hi;
        u32x4 x[NP];
        split8<NP>(f32x4{to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3])},
                   f32x4{to_f32(p[4]), to_f32(p[5]), to_f32(p[6]), to_f32(p[7])}, x);
#pragma unroll
        for (int i = 0; i < NP; ++i) byrow[(f * NP + i) * kFragLanes + lane] = x[i];
    }
    u32x4* turned = which ? out.qt : out.kt;
    if (!turned) return;
    turned += at;
    for (int f = wave; f < 4 * steps; f += kThreads / 64) {  // 2 steps blocks of Dk x 2 steps of tokens
        const T* p = rows + (f % 2 * 32 + 8 * hi) * ld + f / 2 * 16 + n;
        u32x4 x[NP];
        split8<NP>(f32x4{to_f32(p[0]), to_f32(p[ld]), to_f32(p[2 * ld]), to_f32(p[3 * ld])},
                   f32x4{to_f32(p[4 * ld]), to_f32(p[5 * ld]), to_f32(p[6 * ld]), to_f32(p[7 * ld])}, x);
#pragma unroll
        for (int i = 0; i < NP; ++i) turned[(f * NP + i) * kFragLanes + lane] = x[i];
    }
}

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

constexpr int kLd = 68;  // row of a 64-wide LDS tile: 16 bytes past a multiple of all banks

// c += A B of 16x16 blocks in LDS in float32: rows of A at a, rows of B at b.
__device__ __forceinline__ f32x4 block_product(const float* a, const float* b, int n, int hi, f32x4 c) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(a + n * kLd + 4 * hi);
#pragma unroll
    for (int r = 0; r < 4; ++r) c = mfma4(x[r], b[(4 * hi + r) * kLd + n], c);
    return c;
}
// The same with B as a result block in registers.
__device__ __forceinline__ f32x4 block_product(const float* a, f32x4 b, int n, int hi, f32x4 c) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(a + n * kLd + 4 * hi);
#pragma unroll
    for (int r = 0; r < 4; ++r) c = mfma4(x[r], b[r], c);
    return c;
}
__device__ __forceinline__ void put_result(float* to, f32x4 x, int n, int hi) {
#pragma unroll
    for (int r = 0; r < 4; ++r) to[(4 * hi + r) * kLd + n] = x[r];
}

// What the chains read of a chunk and value head.  The inverse of I + N diag(beta) in
// float32: its 16x16 diagonal blocks by forward substitution (a column per lane), then
// the blocks below from theirs, [A 0; B C]^-1 = [A^-1 0; -C^-1 B A^-1 C^-1], for 32 and 64
// rows.  (Backward stable; a series of powers of N is not where keys are alike.)
// `x`: v, or (backward) dO, which may be null.  VEC: Dv is a multiple of eight.
//
// Bound by what it writes: of a chunk and head of 128x128 bf16 32 KB of `own` (float32, as
// the chain adds it), 48 KB of `read` and 18 KB of `p` in three pieces, of which the bf16
// chain reads two; 16384 tokens of 16 heads (418 MB written, 225 read) 160 us, 4.0 TB/s; the
// inverse, a chain of its own, is hidden by the other workgroups of the CU.  Written in the form that the chain's
// registers take, since the chain, which is serial, would pay for every conversion.
template <typename T, bool BACKWARD, bool VEC>
__global__ __launch_bounds__(kThreads) void prepare_kernel(Dims d, const T* x, const void* g, const void* beta,
                                                           const int* lengths, ChunkData out) {
    constexpr int NP = kPieces<T>;
    constexpr int kLdX = sizeof(T) == 4 ? 68 : 72;  // row of 64 columns of x
    __shared__ __attribute__((aligned(16))) float nb[kChunk * kLd], ti[kChunk * kLd];
    __shared__ double gsum[kChunk];
    __shared__ float bet[kChunk], ck[kChunk], cq[kChunk], scaled[kChunk];
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 16, hi = lane / 16;
    const int c = blockIdx.x % d.chunks, bh = blockIdx.x / d.chunks;
    const int b = bh / d.Hv, h = bh % d.Hv, hk = h / (d.Hv / d.Hk);
    const int t0 = c * kChunk, live = min(kChunk, row_length(lengths, b, d.T) - t0);
    if (live <= 0) return;
    const size_t ch = blockIdx.x, kch = ((size_t)b * d.Hk + hk) * d.chunks + c;
    // the rows of x, 64 columns at a time, the first loaded now
    const T* px = x;
    long long stride = 0;
    if constexpr (BACKWARD) {
        stride = (long long)d.Hv * d.Dv;
        if (px) px += (((size_t)b * d.T + t0) * d.Hv + h) * d.Dv;
    } else {
        stride = d.v_s[1];
        px += b * d.v_s[0] + t0 * d.v_s[1] + h * d.v_s[2];
    }
    Eight<T> next[2] = {};
    auto load_x = [&](int v0) {
        if (!px) return;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            next[i].template load<VEC>(px + min(tid / 8 + 32 * i, live - 1) * stride, v0 + tid % 8 * 8, d.Dv);
    };
    load_x(0);
    if (wave == 0) {
        float gv = load_gate(g, b * d.g_s[0] + (t0 + min(lane, live - 1)) * d.g_s[1] + h * d.g_s[2], d.gate_bf16);
        float bv = load_gate(beta, b * d.b_s[0] + (t0 + min(lane, live - 1)) * d.b_s[1] + h * d.b_s[2], d.gate_bf16);
        gsum[lane] = chunk_sum(lane < live ? gv : 0.f, lane);
        bet[lane] = lane < live ? bv : 0.f;
    } else if (wave == 1) {
        ck[lane] = out.norm[kch * 2 * kChunk + lane];
        cq[lane] = out.norm[(kch * 2 + 1) * kChunk + lane];
    }
    const int steps = chain_steps(d.Dk);
    const u32x4* fk = out.k + kch * row_frags<T>(d.Dk) * kFragLanes + lane;
    const u32x4* fq = out.q + kch * row_frags<T>(d.Dk) * kFragLanes + lane;
    f32x4 kk[4] = {}, qk[4] = {};
    for (int u = 0; u < steps; ++u) {
        u32x4 a[NP], aq[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            a[i] = fk[((wave * steps + u) * NP + i) * kFragLanes];
            aq[i] = fq[((wave * steps + u) * NP + i) * kFragLanes];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > wave) break;
            u32x4 y[NP];
#pragma unroll
            for (int i = 0; i < NP; ++i) y[i] = fk[((j * steps + u) * NP + i) * kFragLanes];
            kk[j] = mul(a, y, kk[j]);
            qk[j] = mul(aq, y, qk[j]);
            settle_all();
        }
    }
    __syncthreads();
    f32x4 p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * wave + 4 * hi + r, col = 16 * j + n;
            const float w = made(expf((float)(gsum[row] - gsum[col]))) * ck[col] * bet[col];
            const float nv = row > col ? kk[j][r] * ck[row] * w : 0.f;
            const float pv = row >= col ? d.scale * qk[j][r] * cq[row] * w : 0.f;
            nb[row * kLd + col] = nv;
            ti[row * kLd + col] = 0.f;
            p[j][r] = pv;
        }
    if (tid < kChunk) {
        float* coef = out.coef + ch * kCoefFloats;
        const float eg = expf((float)gsum[tid]), el = expf((float)(gsum[kChunk - 1] - gsum[tid]));
        const bool on = tid < live;
        const float rk = on ? eg * ck[tid] : 0.f, wk = on ? el * ck[tid] * bet[tid] : 0.f;
        coef[RK * kChunk + tid] = rk;
        coef[WK * kChunk + tid] = wk;
        coef[RQ * kChunk + tid] = on ? d.scale * eg * cq[tid] : 0.f;
        coef[BETA * kChunk + tid] = bet[tid];
        coef[CK * kChunk + tid] = ck[tid];
        coef[CQ * kChunk + tid] = cq[tid];
        if (tid == 0) coef[NCOEF * kChunk] = expf((float)gsum[kChunk - 1]);
        scaled[tid] = BACKWARD ? wk : rk;
    }
    __syncthreads();
    {
        // the wavefront's own diagonal block (the four 16-lane groups alike)
        const float* a = nb + 16 * wave * kLd + 16 * wave;
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v = i == n ? 1.f : 0.f;
#pragma unroll
            for (int m = 0; m < i; ++m) v = fmaf(-a[i * kLd + m], y[m], v);
            y[i] = v;
        }
        if (hi == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) ti[(16 * wave + i) * kLd + 16 * wave + n] = y[i];
        }
    }
    __syncthreads();
    auto at = [&](float* m, int i, int j) { return m + 16 * i * kLd + 16 * j; };
    if (wave == 1 || wave == 3) {
        const f32x4 y = block_product(at(nb, wave, wave - 1), at(ti, wave - 1, wave - 1), n, hi, f32x4{});
        put_result(at(ti, wave, wave - 1), -block_product(at(ti, wave, wave), y, n, hi, f32x4{}), n, hi);
    }
    __syncthreads();
    {
        // block (2 + i, j) of the lower left quarter
        const int i = wave / 2, j = wave % 2;
        f32x4 sum{};
        for (int m = 0; m <= i; ++m) {
            f32x4 y{};
            for (int l = j; l < 2; ++l) {
                y = block_product(at(nb, 2 + m, l), at(ti, l, j), n, hi, y);
                settle_all();
            }
            sum = block_product(at(ti, 2 + i, 2 + m), y, n, hi, sum);
            settle_all();
        }
        put_result(at(ti, 2 + i, j), -sum, n, hi);
    }
    __syncthreads();
    // P where N was (which nobody reads any more)
#pragma unroll
    for (int j = 0; j < 4; ++j) put_result(at(nb, wave, j), p[j], n, hi);
    __syncthreads();
    // Operands of the wavefront's 16 rows: of T with its columns (backward: of T^T with
    // them) scaled for the keys, and of what x is multiplied by: T (backward: (P T)^T).
    // T and T^T differ in which 32-wide steps are not all zero.
    u32x4 tk[2][3], tx[2][3];
    auto operand = [&](const float* m, int w, bool scale, u32x4 (&f)[3]) {
        f32x4 y[2];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = 32 * w + 8 * hi + e;
            const float v = BACKWARD ? m[i * kLd + 16 * wave + n] : m[(16 * wave + n) * kLd + i];
            y[e / 4][e % 4] = scale ? v * scaled[i] : v;
        }
        split8<3>(y[0], y[1], f);
    };
    auto live_step = [&](int w) { return BACKWARD ? w >= wave / 2 : w <= wave / 2; };
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if (!live_step(w)) continue;
        operand(ti, w, true, tk[w]);
        if constexpr (!BACKWARD) {
            operand(ti, w, false, tx[w]);
            u32x4 f[3];
            operand(nb, w, false, f);
#pragma unroll
            for (int i = 0; i < 3; ++i)
                out.p[(ch * kTriFrags * 3 + lower_frag(wave, w) * 3 + i) * kFragLanes + lane] = f[i];
        }
    }
    if constexpr (BACKWARD) {
        f32x4 m[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int l = j; l <= wave; ++l) {
                m[j] = block_product(at(nb, wave, l), at(ti, l, j), n, hi, m[j]);
                settle_all();
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) put_result(at(nb, wave, j), m[j], n, hi);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 2; ++w)
            if (live_step(w)) operand(nb, w, false, tx[w]);
    }
    // transposed: rows of Dk, columns the wavefront's tokens
    u32x4* read = out.read + (ch * read_frags(d.Dk) + (size_t)wave * steps * 3) * kFragLanes;
    const u32x4* fkt = out.kt + kch * row_frags<T>(d.Dk) * kFragLanes + lane;
    for (int b0 = 0; b0 < 2 * steps; b0 += 4) {  // (a multiple of four; their loads at once)
        u32x4 a[4][2][NP];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < NP; ++i) a[j][w][i] = fkt[(((b0 + j) * 2 + w) * NP + i) * kFragLanes];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4 y{};
            if (live_step(0)) {
                y = mul(a[j][0], tk[0], y);
                settle(y);
            }
            if (live_step(1)) {
                y = mul(a[j][1], tk[1], y);
                settle(y);
            }
            u32x2 pieces[3];
            split<3>(y, pieces);
            put_block(read, 3, b0 + j, hi, n, pieces);
        }
    }
    // the products with x, 64 columns of it at a time in LDS
    T* xs = reinterpret_cast<T*>(ti);
    const int blocks = column_blocks(d.Dv);
    for (int v0 = 0; v0 < d.Dv; v0 += 64) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
            next[i].store(px && tid / 8 + 32 * i < live, xs + (tid / 8 + 32 * i) * kLdX + tid % 8 * 8);
        if (v0 + 64 < d.Dv) load_x(v0 + 64);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (v0 + 16 * j >= d.Dv) break;
            f32x4 y{};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (!live_step(w)) continue;
                const T* q = xs + (32 * w + 8 * hi) * kLdX + 16 * j + n;
                u32x4 f[NP];
                split8<NP>(f32x4{to_f32(q[0]), to_f32(q[kLdX]), to_f32(q[2 * kLdX]), to_f32(q[3 * kLdX])},
                           f32x4{to_f32(q[4 * kLdX]), to_f32(q[5 * kLdX]), to_f32(q[6 * kLdX]), to_f32(q[7 * kLdX])}, f);
                y = mul(tx[w], f, y);
                settle(y);
            }
            out.own[((ch * blocks + v0 / 16 + j) * 4 + wave) * kFragLanes + lane] = y;
        }
    }
}

// ---------------------------------------------------------- workspaces ---
struct ChunkLayout {
    size_t coef, norm, k, q, kt, qt, read, p, own, total;
};
// Of the backward (with qt, without p) or the forward.  Sized for float32 pieces
// where `wide`.
ChunkLayout chunk_layout(const Dims& d, bool wide, bool backward) {
    ChunkLayout l{};
    const size_t ch = (size_t)d.B * d.Hv * d.chunks, kch = (size_t)d.B * d.Hk * d.chunks;
    const size_t rows = kch * (wide ? row_frags<float>(d.Dk) : row_frags<bf16>(d.Dk)) * kFragLanes * 16;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t was = at;
        at += align_up(bytes, 256);
        return was;
    };
    l.coef = take(ch * kCoefFloats * sizeof(float));
    l.norm = take(kch * 2 * kChunk * sizeof(float));
    l.k = take(rows);
    l.q = take(rows);
    l.kt = take(rows);
    l.qt = backward ? take(rows) : 0;
    l.read = take(ch * read_frags(d.Dk) * kFragLanes * 16);
    l.p = backward ? 0 : take(ch * kTriFrags * 3 * kFragLanes * 16);
    l.own = take(ch * column_blocks(d.Dv) * 4 * kFragLanes * 16);
    l.total = at;
    return l;
}
struct ReserveLayout {
    size_t states, e, total;
};
ReserveLayout reserve_layout(const Dims& d) {
    ReserveLayout l{};
    l.states = 0;
    l.e = align_up((size_t)d.B * d.Hv * d.chunks * d.Dk * d.Dv * sizeof(float), 256);
    l.total = l.e + align_up((size_t)d.B * d.T * d.Hv * d.Dv * sizeof(float), 256);
    return l;
}
struct BackwardLayout {
    ChunkLayout f;
    size_t dstates, dx, total;
};
BackwardLayout backward_layout(const Dims& d, bool wide) {
    BackwardLayout l{};
    l.f = chunk_layout(d, wide, true);
    l.dstates = l.f.total;
    l.dx = l.dstates + align_up((size_t)d.B * d.Hv * d.chunks * d.Dk * d.Dv * sizeof(float), 256);
    l.total = l.dx + align_up((size_t)d.B * d.T * d.Hv * d.Dv * sizeof(float), 256);
    return l;
}

ChunkData chunk_data(char* ws, const ChunkLayout& l) {
    ChunkData c{};
    c.coef = reinterpret_cast<float*>(ws + l.coef);
    c.norm = reinterpret_cast<float*>(ws + l.norm);
    c.k = reinterpret_cast<u32x4*>(ws + l.k);
    c.q = reinterpret_cast<u32x4*>(ws + l.q);
    c.kt = reinterpret_cast<u32x4*>(ws + l.kt);
    c.qt = l.qt ? reinterpret_cast<u32x4*>(ws + l.qt) : nullptr;
    c.read = reinterpret_cast<u32x4*>(ws + l.read);
    c.p = l.p ? reinterpret_cast<u32x4*>(ws + l.p) : nullptr;
    c.own = reinterpret_cast<f32x4*>(ws + l.own);
    return c;
}

// x: v, or (backward) dO.
template <typename T, bool BACKWARD>
int prepare(const Dims& d, const T* q, const T* k, const T* x, const void* g, const void* beta, const int* lengths,
            const ChunkData& out, hipStream_t stream) {
    const long long blocks = (long long)d.B * d.Hv * d.chunks, rows = (long long)d.B * d.Hk * d.chunks * 2;
    if (blocks == 0) return 0;
    RKA_RETURN_IF_ERR(check_grid(std::max(blocks, rows), kThreads, "gated_delta"));
    const size_t lds = (size_t)kChunk * (chain_steps(d.Dk) * 32 + 8) * sizeof(T);
    auto by_rows = [&](auto kernel) {
        RKA_RETURN_IF_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(kThreads), lds, stream, d, q, k, lengths, out);
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    };
    RKA_RETURN_IF_ERR(d.Dk % 8 == 0 ? by_rows(&rows_kernel<T, true>) : by_rows(&rows_kernel<T, false>));
    if (d.Dv % 8 == 0)
        hipLaunchKernelGGL((prepare_kernel<T, BACKWARD, true>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, d, x, g,
                           beta, lengths, out);
    else
        hipLaunchKernelGGL((prepare_kernel<T, BACKWARD, false>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, d, x, g,
                           beta, lengths, out);
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}

template <typename T>
int forward(const Dims& d, const void* q, const void* k, const void* v, const void* g, const void* beta, const float* s0,
            const int* lengths, void* o, float* state_out, char* reserve, char* ws, hipStream_t s) {
    const ChunkData cd = chunk_data(ws, chunk_layout(d, sizeof(T) == 4, false));
    RKA_RETURN_IF_ERR((prepare<T, false>(d, static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), g,
                                         beta, lengths, cd, s)));
    const ReserveLayout r = reserve_layout(d);
    return launch_chain_forward<T>(d, s0, lengths, cd, static_cast<T*>(o), state_out,
                                   reserve ? reinterpret_cast<float*>(reserve + r.states) : nullptr,
                                   reserve ? reinterpret_cast<float*>(reserve + r.e) : nullptr, s);
}

template <typename T>
int backward(const Dims& d, const void* q, const void* k, const void* g, const void* beta, const int* lengths,
             const char* reserve, const void* dout, const float* dstate_out, void* dq, void* dk, void* dv, void* dg,
             void* dbeta, float* ds0, char* ws, hipStream_t s) {
    const BackwardLayout l = backward_layout(d, sizeof(T) == 4);
    const ReserveLayout r = reserve_layout(d);
    const ChunkData cd = chunk_data(ws, l.f);
    const T *tq = static_cast<const T*>(q), *tk = static_cast<const T*>(k), *tdo = static_cast<const T*>(dout);
    const BackwardData bd{reinterpret_cast<const float*>(reserve + r.states), reinterpret_cast<const float*>(reserve + r.e),
                          reinterpret_cast<float*>(ws + l.dstates), reinterpret_cast<float*>(ws + l.dx)};
    RKA_RETURN_IF_ERR((prepare<T, true>(d, tq, tk, tdo, g, beta, lengths, cd, s)));
    RKA_RETURN_IF_ERR(launch_chain_backward<T>(d, tdo, dstate_out, lengths, cd, static_cast<T*>(dv), ds0, bd, s));
    return launch_gradients<T>(d, tq, tk, tdo, g, lengths, cd, bd, static_cast<T*>(dq), static_cast<T*>(dk), dg, dbeta, s);
}

}  // namespace

int make_dims(const char* what, int B, int T, int Hk, int Hv, int Dk, int Dv, Dims* d) {
    const std::string name(what);
    if (B < 0 || T < 0 || Hk < 1 || Hv < 1 || Dk < 1 || Dv < 1)
        return fail(RKA_ERR_INVALID_ARGUMENT, name + ": batch and tokens must be >= 0, heads and head sizes >= 1");
    if (Hv % Hk != 0)
        return fail(RKA_ERR_INVALID_ARGUMENT, name + ": value heads must be a multiple of key heads");
    if (Dk > kMaxKeyDim)
        return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": key head size exceeds " + std::to_string(kMaxKeyDim));
    if ((long long)B * Hv > 0x7fffffffLL || (long long)Hv * Dv > 0x7fffffffLL || (long long)Hk * Dk > 0x7fffffffLL)
        return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": batch x heads or heads x head size exceeds 2^31 - 1");
    *d = Dims{};
    d->B = B;
    d->T = T;
    d->Hk = Hk;
    d->Hv = Hv;
    d->Dk = Dk;
    d->Dv = Dv;
    d->chunks = (int)(((long long)T + kChunk - 1) / kChunk);
    return 0;
}

int set_call(const char* what, Dims* d, int dtype, int gate_dtype, int normalize, double scale, const long long* strides) {
    const std::string name(what);
    if ((dtype != RKA_DTYPE_F32 && dtype != RKA_DTYPE_BF16) || (gate_dtype != RKA_DTYPE_F32 && gate_dtype != RKA_DTYPE_BF16))
        return fail(RKA_ERR_INVALID_ARGUMENT, name + ": dtype must be RKA_DTYPE_F32 or RKA_DTYPE_BF16");
    if (!strides) return fail(RKA_ERR_INVALID_ARGUMENT, name + ": strides must be non-NULL");
    d->scale = (float)scale;
    d->normalize = normalize != 0;
    d->gate_bf16 = gate_dtype == RKA_DTYPE_BF16;
    for (int i = 0; i < 3; ++i) {
        d->q_s[i] = strides[i];
        d->k_s[i] = strides[3 + i];
        d->v_s[i] = strides[6 + i];
        d->g_s[i] = strides[9 + i];
        d->b_s[i] = strides[12 + i];
    }
    return 0;
}

int check_grid(long long blocks, int threads, const char* what) {
    if (blocks * threads >= (1LL << 32))
        return fail(RKA_ERR_UNSUPPORTED_SHAPE, std::string(what) + ": more workgroups than a launch may have");
    return 0;
}

}  // namespace delta
}  // namespace rka

using namespace rka;
using namespace rka::delta;

extern "C" {

size_t rka_gated_delta_forward_workspace_bytes(int batch, int tokens, int key_heads, int value_heads, int key_dim,
                                               int value_dim, int dtype) {
    Dims d;
    if (make_dims("gated_delta", batch, tokens, key_heads, value_heads, key_dim, value_dim, &d) != 0) return 0;
    return chunk_layout(d, dtype == RKA_DTYPE_F32, false).total;
}

size_t rka_gated_delta_reserve_bytes(int batch, int tokens, int key_heads, int value_heads, int key_dim, int value_dim) {
    Dims d;
    if (make_dims("gated_delta", batch, tokens, key_heads, value_heads, key_dim, value_dim, &d) != 0) return 0;
    return reserve_layout(d).total;
}

size_t rka_gated_delta_backward_workspace_bytes(int batch, int tokens, int key_heads, int value_heads, int key_dim,
                                                int value_dim, int dtype) {
    Dims d;
    if (make_dims("gated_delta", batch, tokens, key_heads, value_heads, key_dim, value_dim, &d) != 0) return 0;
    return backward_layout(d, dtype == RKA_DTYPE_F32).total;
}

int rka_describe_gated_delta(int batch, int value_heads, int key_dim, int value_dim, int dtype, int* out, int n_out) {
    clear_error();
    if (!out || n_out < 1) return fail(RKA_ERR_INVALID_ARGUMENT, "describe_gated_delta: out must be non-NULL and n_out >= 1");
    if (dtype != RKA_DTYPE_F32 && dtype != RKA_DTYPE_BF16)
        return fail(RKA_ERR_INVALID_ARGUMENT, "describe_gated_delta: dtype must be RKA_DTYPE_F32 or RKA_DTYPE_BF16");
    Dims d;
    RKA_RETURN_IF_ERR(make_dims("describe_gated_delta", batch, 0, 1, value_heads, key_dim, value_dim, &d));
    const int columns = chain_columns(d, dtype == RKA_DTYPE_F32 ? kPieces<float> : kPieces<bf16>);
    const int v[3] = {chain_steps(d.Dk), columns, (int)std::min<long long>(chain_blocks(d, columns), 0x7fffffff)};
    for (int i = 0; i < 3 && i < n_out; ++i) out[i] = v[i];
    return 0;
}

int rka_gated_delta_forward(const void* q, const void* k, const void* v, const void* g, const void* beta,
                            const float* initial_state, const int* lengths, void* o, float* final_state, void* reserve,
                            void* workspace, size_t workspace_bytes, int batch, int tokens, int key_heads,
                            int value_heads, int key_dim, int value_dim, const long long* strides, int dtype,
                            int gate_dtype, int normalize, double scale, void* stream) {
    clear_error();
    Dims d;
    RKA_RETURN_IF_ERR(make_dims("gated_delta_forward", batch, tokens, key_heads, value_heads, key_dim, value_dim, &d));
    RKA_RETURN_IF_ERR(set_call("gated_delta_forward", &d, dtype, gate_dtype, normalize, scale, strides));
    if (d.B == 0) return 0;
    if (!final_state || (d.T > 0 && (!q || !k || !v || !g || !beta || !o)))
        return fail(RKA_ERR_INVALID_ARGUMENT, "gated_delta_forward: null tensor pointer");
    const size_t need = chunk_layout(d, dtype == RKA_DTYPE_F32, false).total;
    if (workspace_bytes < need || (need > 0 && !workspace))
        return fail(RKA_ERR_WORKSPACE_TOO_SMALL, "gated_delta_forward: workspace needs " + std::to_string(need) +
                                                     " bytes, got " + std::to_string(workspace_bytes));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    char *ws = static_cast<char*>(workspace), *rs = static_cast<char*>(reserve);
    return dtype == RKA_DTYPE_F32 ? forward<float>(d, q, k, v, g, beta, initial_state, lengths, o, final_state, rs, ws, s)
                                  : forward<bf16>(d, q, k, v, g, beta, initial_state, lengths, o, final_state, rs, ws, s);
}

int rka_gated_delta_backward(const void* q, const void* k, const void* g, const void* beta, const int* lengths,
                             const void* reserve, const void* grad_o, const float* grad_final_state, void* grad_q,
                             void* grad_k, void* grad_v, void* grad_g, void* grad_beta, float* grad_initial_state,
                             void* workspace, size_t workspace_bytes, int batch, int tokens, int key_heads,
                             int value_heads, int key_dim, int value_dim, const long long* strides, int dtype,
                             int gate_dtype, int normalize, double scale, void* stream) {
    clear_error();
    Dims d;
    RKA_RETURN_IF_ERR(make_dims("gated_delta_backward", batch, tokens, key_heads, value_heads, key_dim, value_dim, &d));
    RKA_RETURN_IF_ERR(set_call("gated_delta_backward", &d, dtype, gate_dtype, normalize, scale, strides));
    if (d.B == 0) return 0;
    if (d.T > 0 && (!q || !k || !g || !beta || !reserve || !grad_q || !grad_k || !grad_v || !grad_g || !grad_beta))
        return fail(RKA_ERR_INVALID_ARGUMENT, "gated_delta_backward: null tensor pointer");
    const size_t need = backward_layout(d, dtype == RKA_DTYPE_F32).total;
    if (workspace_bytes < need || (need > 0 && !workspace))
        return fail(RKA_ERR_WORKSPACE_TOO_SMALL, "gated_delta_backward: workspace needs " + std::to_string(need) +
                                                     " bytes, got " + std::to_string(workspace_bytes));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    const char* rs = static_cast<const char*>(reserve);
    return dtype == RKA_DTYPE_F32
               ? backward<float>(d, q, k, g, beta, lengths, rs, grad_o, grad_final_state, grad_q, grad_k, grad_v, grad_g,
                                 grad_beta, grad_initial_state, ws, s)
               : backward<bf16>(d, q, k, g, beta, lengths, rs, grad_o, grad_final_state, grad_q, grad_k, grad_v, grad_g,
                                grad_beta, grad_initial_state, ws, s);
}

}  // extern "C"
