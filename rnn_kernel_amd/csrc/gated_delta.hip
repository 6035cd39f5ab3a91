// The gated delta rule (gated_delta.h has the formulas): entry points, what is made
// for all chunks at once before the chains (prepare) and the gradients made after
// the backward's chain.
#include "gated_delta.h"

#include <algorithm>

namespace rka {
namespace delta {
namespace {

constexpr int kThreads = 256;
constexpr int kLd = 68;  // row of a 64-wide LDS tile: 16 bytes past a multiple of all banks

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// rows x 64 elements (from column d0 of `width`) of a strided matrix as float32 in
// LDS; zero past `live` rows and the width.
template <typename T>
__device__ __forceinline__ void stage64(float* lds, const T* src, long long stride, int live, int d0, int width,
                                        int tid) {
#pragma unroll
    for (int i = 0; i < kChunk * 16 / kThreads; ++i) {
        const int r = (tid + i * kThreads) / 16, c = (tid + i * kThreads) % 16 * 4;
        f32x4 x{0.f, 0.f, 0.f, 0.f};
        if (r < live) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d0 + c + j < width) x[j] = to_f32(src[r * stride + d0 + c + j]);
        }
        *reinterpret_cast<f32x4*>(lds + r * kLd + c) = x;
    }
}

// Running sums of the floored gates of a chunk (by one wavefront; lane = token).
// In 64 bits: a difference of sums is as exact after a closed gate as before it.
__device__ __forceinline__ double chunk_sum(float g, int lane) {
    double s = floor_gate(g);
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const double up = __shfl_up(s, o);
        if (lane >= o) s += up;
    }
    return s;
}

// T and P of a chunk.  K K^T and Q K^T on fp32 matrix instructions, then the inverse of the
// unit lower triangular I + N diag(beta) by forward substitution, one column per
// lane (backward stable, which a series of powers of N is not).
template <typename T, bool TRANSPOSE>
__global__ __launch_bounds__(kThreads) void prepare_kernel(Dims d, const T* q, const T* k, const void* g,
                                                           const void* beta, const int* lengths, ChunkData out) {
    __shared__ float ks[kChunk * kLd], qs[kChunk * kLd], nb[kChunk * kLd], ps[kChunk * kLd];
    __shared__ double gsum[kChunk];
    __shared__ float bet[kChunk], ck[kChunk], cq[kChunk];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, n = lane % 16, hi = lane / 16;
    const int c = blockIdx.x % d.chunks, bh = blockIdx.x / d.chunks;
    const int b = bh / d.Hv, h = bh % d.Hv, hk = h / (d.Hv / d.Hk);
    const int t0 = c * kChunk, live = min(kChunk, row_length(lengths, b, d.T) - t0);
    if (live <= 0) return;
    const T* kb = k + b * d.k_s[0] + t0 * d.k_s[1] + hk * d.k_s[2];
    const T* qb = q + b * d.q_s[0] + t0 * d.q_s[1] + hk * d.q_s[2];
    if (wave == 0) {
        float gv = 0.f, bv = 0.f;
        if (lane < live) {
            gv = load_gate(g, b * d.g_s[0] + (t0 + lane) * d.g_s[1] + h * d.g_s[2], d.gate_bf16);
            bv = load_gate(beta, b * d.b_s[0] + (t0 + lane) * d.b_s[1] + h * d.b_s[2], d.gate_bf16);
        }
        gsum[lane] = chunk_sum(gv, lane);
        bet[lane] = bv;
    }
    f32x4 kk[4] = {}, qk[4] = {};
    float k2 = 0.f, q2 = 0.f;
    for (int d0 = 0; d0 < d.Dk; d0 += 64) {
        __syncthreads();
        stage64(ks, kb, d.k_s[1], live, d0, d.Dk, tid);
        stage64(qs, qb, d.q_s[1], live, d0, d.Dk, tid);
        __syncthreads();
        // a quarter of a row's squares per thread
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float x = ks[tid / 4 * kLd + tid % 4 * 16 + j], y = qs[tid / 4 * kLd + tid % 4 * 16 + j];
            k2 += x * x;
            q2 += y * y;
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const f32x4 ak = *reinterpret_cast<const f32x4*>(ks + (16 * wave + n) * kLd + s * 16 + hi * 4);
            const f32x4 aq = *reinterpret_cast<const f32x4*>(qs + (16 * wave + n) * kLd + s * 16 + hi * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j > wave) break;
                const f32x4 x = *reinterpret_cast<const f32x4*>(ks + (16 * j + n) * kLd + s * 16 + hi * 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    kk[j] = mfma4(ak[r], x[r], kk[j]);
                    qk[j] = mfma4(aq[r], x[r], qk[j]);
                }
            }
        }
    }
    k2 += __shfl_xor(k2, 1);
    q2 += __shfl_xor(q2, 1);
    k2 += __shfl_xor(k2, 2);
    q2 += __shfl_xor(q2, 2);
    if (tid % 4 == 0) {
        ck[tid / 4] = d.normalize ? 1.f / sqrtf(k2 + kNormEps) : 1.f;
        cq[tid / 4] = d.normalize ? 1.f / sqrtf(q2 + kNormEps) : 1.f;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * wave + 4 * hi + r, col = 16 * j + n;
            float nv = 0.f, pv = 0.f;
            if (row >= col) {
                const float w = expf((float)(gsum[row] - gsum[col])) * ck[col] * bet[col];
                if (row > col) nv = kk[j][r] * ck[row] * w;
                pv = d.scale * qk[j][r] * cq[row] * w;
            }
            nb[row * kLd + col] = nv;
            ps[row * kLd + col] = pv;
        }
    const size_t ch = blockIdx.x;
    if (tid < kChunk) {
        float* coef = out.coef + ch * kCoefFloats;
        const float eg = expf((float)gsum[tid]), el = expf((float)(gsum[kChunk - 1] - gsum[tid]));
        const bool on = tid < live;
        coef[RK * kChunk + tid] = on ? eg * ck[tid] : 0.f;
        coef[WK * kChunk + tid] = on ? el * ck[tid] * bet[tid] : 0.f;
        coef[RQ * kChunk + tid] = on ? d.scale * eg * cq[tid] : 0.f;
        coef[BETA * kChunk + tid] = bet[tid];
        coef[CK * kChunk + tid] = ck[tid];
        coef[CQ * kChunk + tid] = cq[tid];
        if (tid == 0) coef[NCOEF * kChunk] = expf((float)gsum[kChunk - 1]);
    }
    __syncthreads();
    if (wave == 0) {
        float x[kChunk];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            float v = i == lane ? 1.f : 0.f;
#pragma unroll
            for (int m = 0; m < i; ++m) v = fmaf(-nb[i * kLd + m], x[m], v);
            x[i] = v;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < kChunk; ++i) nb[i * kLd + lane] = x[i];
    }
    __syncthreads();
    float* tt = out.t + ch * kTriFloats;
    float* pp = out.p + ch * kTriFloats;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j > wave) break;
        const int blk = (wave * (wave + 1) / 2 + j) * 256 + lane * 4;
        f32x4 tv, pv;
        if constexpr (TRANSPOSE) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                tv[r] = nb[(16 * wave + 4 * hi + r) * kLd + 16 * j + n];
                pv[r] = ps[(16 * wave + 4 * hi + r) * kLd + 16 * j + n];
            }
        } else {
            tv = *reinterpret_cast<const f32x4*>(nb + (16 * wave + n) * kLd + 16 * j + 4 * hi);
            pv = *reinterpret_cast<const f32x4*>(ps + (16 * wave + n) * kLd + 16 * j + 4 * hi);
        }
        *reinterpret_cast<f32x4*>(tt + blk) = tv;
        *reinterpret_cast<f32x4*>(pp + blk) = pv;
    }
}


constexpr int kLdV = 36;  // row of a 32-wide LDS tile

// 64 rows x 32 columns (from v0 of Dv) of a dense matrix of row stride `stride` as
// float32 in LDS, zero past `rows` rows and Dv.
template <typename T>
__device__ __forceinline__ void stage32(float* lds, const T* src, long long stride, int rows, int v0, int Dv, int tid) {
#pragma unroll
    for (int i = 0; i < kChunk * 8 / kThreads; ++i) {
        const int r = (tid + i * kThreads) / 8, c = (tid + i * kThreads) % 8 * 4;
        f32x4 x{0.f, 0.f, 0.f, 0.f};
        if (src && r < rows) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v0 + c + j < Dv) x[j] = to_f32(src[r * stride + v0 + c + j]);
        }
        *reinterpret_cast<f32x4*>(lds + r * kLdV + c) = x;
    }
}

// Sum over the 16 lanes that hold a row of a 16x16 block.
__device__ __forceinline__ float row_sum(float x) {
    x += __shfl_xor(x, 1);
    x += __shfl_xor(x, 2);
    x += __shfl_xor(x, 4);
    x += __shfl_xor(x, 8);
    return x;
}

// The gradients of q, k, g and beta of a chunk and value head.
template <typename T>
__global__ __launch_bounds__(kThreads) void gradients_kernel(Dims d, const T* q, const T* k, const T* dout, const void* g,
                                                             const int* lengths, ChunkData in, BackwardData bd, void* dg,
                                                             void* dbeta) {
    __shared__ float f1[kChunk * kLd], f2[kChunk * kLd], ks[kChunk * kLd], qs[kChunk * kLd];
    __shared__ float sdo[kChunk * kLdV], sdx[kChunk * kLdV], se[kChunk * kLdV], ss[kChunk * kLdV], sds[kChunk * kLdV];
    __shared__ double gsum[kChunk];
    __shared__ float sums[4][kChunk], dots[4];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, n = lane % 16, hi = lane / 16;
    const int c = blockIdx.x % d.chunks, bh = blockIdx.x / d.chunks;
    const int b = bh / d.Hv, h = bh % d.Hv, hk = h / (d.Hv / d.Hk);
    const int t0 = c * kChunk, live = min(kChunk, row_length(lengths, b, d.T) - t0);
    const size_t ch = blockIdx.x;
    const size_t row0 = ((size_t)b * d.T + t0) * d.Hv + h;  // token row of the [B, T, Hv] tensors
    if (live <= 0) {
        if (tid < min(kChunk, d.T - t0)) {
            store_gate(dg, row0 + (size_t)tid * d.Hv, 0.f, d.gate_bf16);
            store_gate(dbeta, row0 + (size_t)tid * d.Hv, 0.f, d.gate_bf16);
        }
        return;
    }
    const float* coef = in.coef + ch * kCoefFloats;
    if (wave == 0)
        gsum[lane] = chunk_sum(
            lane < live ? load_gate(g, b * d.g_s[0] + (t0 + lane) * d.g_s[1] + h * d.g_s[2], d.gate_bf16) : 0.f, lane);
    const T* pdo = dout ? dout + row0 * d.Dv : nullptr;
    const float* pdx = bd.dx + row0 * d.Dv;
    const float* pe = bd.e + row0 * d.Dv;
    const float* ps = bd.states + ch * d.Dk * d.Dv;
    const float* pds = bd.dstates + ch * d.Dk * d.Dv;
    const long long vrow = (long long)d.Hv * d.Dv;
    {
        f32x4 a1[4] = {}, a2[4] = {};
        for (int v0 = 0; v0 < d.Dv; v0 += 32) {
            __syncthreads();
            stage32(sdo, pdo, vrow, live, v0, d.Dv, tid);
            stage32(sdx, pdx, vrow, live, v0, d.Dv, tid);
            stage32(se, pe, vrow, live, v0, d.Dv, tid);
            __syncthreads();
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const f32x4 x1 = *reinterpret_cast<const f32x4*>(sdo + (16 * wave + n) * kLdV + s * 16 + hi * 4);
                const f32x4 x2 = *reinterpret_cast<const f32x4*>(sdx + (16 * wave + n) * kLdV + s * 16 + hi * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j > wave) break;
                    const f32x4 y = *reinterpret_cast<const f32x4*>(se + (16 * j + n) * kLdV + s * 16 + hi * 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        a1[j] = mfma4(x1[r], y[r], a1[j]);
                        a2[j] = mfma4(x2[r], y[r], a2[j]);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * wave + 4 * hi + r, col = 16 * j + n;
                const float w = row >= col ? expf((float)(gsum[row] - gsum[col])) : 0.f;
                f1[row * kLd + col] = row >= col ? d.scale * a1[j][r] * w : 0.f;
                f2[row * kLd + col] = row > col ? -a2[j][r] * w : 0.f;
            }
    }
    const T* kb = k + b * d.k_s[0] + t0 * d.k_s[1] + hk * d.k_s[2];
    const T* qb = q + b * d.q_s[0] + t0 * d.q_s[1] + hk * d.q_s[2];
    // exp(G) and exp(G_C - G) of the thread's rows
    float eg[4], el[4], cki[4], cqi[4], bi[4], rq[4] = {}, rk[4] = {}, rz[4] = {}, rw[4] = {}, dot = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = 16 * wave + 4 * hi + r;
        eg[r] = expf((float)gsum[row]);
        el[r] = expf((float)(gsum[kChunk - 1] - gsum[row]));
        cki[r] = coef[CK * kChunk + row];
        cqi[r] = coef[CQ * kChunk + row];
        bi[r] = coef[BETA * kChunk + row];
    }
    for (int d0 = 0; d0 < d.Dk; d0 += 64) {
        f32x4 aq[4] = {}, ar[4] = {}, az[4] = {};
        for (int v0 = 0; v0 < d.Dv; v0 += 32) {
            __syncthreads();
            if (v0 == 0) {
                stage64(ks, kb, d.k_s[1], live, d0, d.Dk, tid);
                stage64(qs, qb, d.q_s[1], live, d0, d.Dk, tid);
            }
            stage32(sdo, pdo, vrow, live, v0, d.Dv, tid);
            stage32(sdx, pdx, vrow, live, v0, d.Dv, tid);
            stage32(se, pe, vrow, live, v0, d.Dv, tid);
            stage32(ss, ps + (size_t)d0 * d.Dv, d.Dv, d.Dk - d0, v0, d.Dv, tid);
            stage32(sds, pds + (size_t)d0 * d.Dv, d.Dv, d.Dk - d0, v0, d.Dv, tid);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kChunk * 32 / kThreads; ++i) {
                const int r = (tid + i * kThreads) / 32, cc = (tid + i * kThreads) % 32;
                dot += ss[r * kLdV + cc] * sds[r * kLdV + cc];
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int at = (16 * wave + n) * kLdV + s * 16 + hi * 4;
                const f32x4 xo = *reinterpret_cast<const f32x4*>(sdo + at);
                const f32x4 xx = *reinterpret_cast<const f32x4*>(sdx + at);
                const f32x4 xe = *reinterpret_cast<const f32x4*>(se + at);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 ys = *reinterpret_cast<const f32x4*>(ss + (16 * j + n) * kLdV + s * 16 + hi * 4);
                    const f32x4 yd = *reinterpret_cast<const f32x4*>(sds + (16 * j + n) * kLdV + s * 16 + hi * 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        aq[j] = mfma4(xo[r], ys[r], aq[j]);
                        ar[j] = mfma4(xx[r], ys[r], ar[j]);
                        az[j] = mfma4(xe[r], yd[r], az[j]);
                    }
                }
            }
        }
        // now in terms of the normalised keys and queries
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * wave + 4 * hi + r, col = 16 * j + n;
                aq[j][r] *= d.scale * eg[r];
                ar[j][r] *= -eg[r];
                az[j][r] *= el[r];
                rw[r] += az[j][r] * ks[row * kLd + col] * cki[r];
            }
#pragma unroll
        for (int m = 0; m < 4; ++m) {  // 16 tokens of the sum
            const f32x4 ckm = *reinterpret_cast<const f32x4*>(coef + CK * kChunk + 16 * m + 4 * hi);
            const f32x4 cqm = *reinterpret_cast<const f32x4*>(coef + CQ * kChunk + 16 * m + 4 * hi);
            const f32x4 bm = *reinterpret_cast<const f32x4*>(coef + BETA * kChunk + 16 * m + 4 * hi);
            const f32x4 x1 = *reinterpret_cast<const f32x4*>(f1 + (16 * wave + n) * kLd + 16 * m + 4 * hi);
            const f32x4 x2 = *reinterpret_cast<const f32x4*>(f2 + (16 * wave + n) * kLd + 16 * m + 4 * hi);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int tok = 16 * m + 4 * hi + r;
                const float xt1 = f1[tok * kLd + 16 * wave + n], xt2 = f2[tok * kLd + 16 * wave + n];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float kv = ks[tok * kLd + 16 * j + n] * ckm[r], qv = qs[tok * kLd + 16 * j + n] * cqm[r];
                    aq[j] = mfma4(x1[r] * bm[r], kv, aq[j]);
                    ar[j] = mfma4(x2[r] * bm[r], kv, ar[j]);
                    az[j] = mfma4(xt1, qv, az[j]);
                    az[j] = mfma4(xt2, kv, az[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * wave + 4 * hi + r, col = 16 * j + n;
                const float kv = ks[row * kLd + col] * cki[r], qv = qs[row * kLd + col] * cqi[r];
                rq[r] += aq[j][r] * qv;
                rk[r] += ar[j][r] * kv;
                rz[r] += az[j][r] * kv;
                if (row < live && d0 + col < d.Dk) {
                    const size_t at = (row0 + (size_t)row * d.Hv) * d.Dk + d0 + col;
                    bd.dq[at] = aq[j][r];
                    bd.dk[at] = ar[j][r] + bi[r] * az[j][r];
                }
            }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = 16 * wave + 4 * hi + r;
        const float a = row_sum(rq[r]), bb = row_sum(rk[r]), z = row_sum(rz[r]), w = row_sum(rw[r]);
        if (n == 0) {
            sums[0][row] = a;
            sums[1][row] = bb;
            sums[2][row] = z;
            sums[3][row] = w * bi[r];
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) dot += __shfl_xor(dot, o);
    if (lane == 0) dots[wave] = dot;
    __syncthreads();
    if (wave != 0) return;
    float w = sums[3][lane];
#pragma unroll
    for (int o = 1; o < 64; o *= 2) w += __shfl_xor(w, o);
    const float db = sums[2][lane];
    float dgv = sums[0][lane] + sums[1][lane] - coef[BETA * kChunk + lane] * db;
    if (lane == 63) dgv += w + expf((float)gsum[kChunk - 1]) * (dots[0] + dots[1] + dots[2] + dots[3]);
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const float down = __shfl_down(dgv, o);
        if (lane + o < 64) dgv += down;
    }
    if (lane < min(kChunk, d.T - t0)) {
        store_gate(dg, row0 + (size_t)lane * d.Hv, lane < live ? dgv : 0.f, d.gate_bf16);
        store_gate(dbeta, row0 + (size_t)lane * d.Hv, lane < live ? db : 0.f, d.gate_bf16);
    }
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) x += __shfl_xor(x, o);
    return x;
}

// dq and dk of the key heads: the sum over the value heads that share one, then
// the normalisation's gradient, dx = c (dy - y (y . dy)) with y = c x.  A wavefront
// per token and key head.
template <typename T>
__global__ __launch_bounds__(kThreads) void finish_kernel(Dims d, const T* q, const T* k, const int* lengths,
                                                          BackwardData bd, T* dq, T* dk) {
    constexpr int M = kMaxKeyDim / 64;
    const long long row = (long long)blockIdx.x * (kThreads / 64) + threadIdx.x / 64;
    if (row >= (long long)d.B * d.T * d.Hk) return;
    const int lane = threadIdx.x % 64, hk = (int)(row % d.Hk), rep = d.Hv / d.Hk;
    const long long bt = row / d.Hk;
    const int b = (int)(bt / d.T), t = (int)(bt % d.T);
    const bool on = t < row_length(lengths, b, d.T);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const float* part = (which ? bd.dk : bd.dq) + (bt * d.Hv + (long long)hk * rep) * d.Dk;
        const T* x = which ? k + b * d.k_s[0] + t * d.k_s[1] + hk * d.k_s[2] : q + b * d.q_s[0] + t * d.q_s[1] + hk * d.q_s[2];
        T* out = (which ? dk : dq) + row * d.Dk;
        float v[M], xv[M], x2 = 0.f, xd = 0.f;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const int i = lane + 64 * m;
            v[m] = xv[m] = 0.f;
            if (!on || i >= d.Dk) continue;
            for (int r = 0; r < rep; ++r) v[m] += part[(long long)r * d.Dk + i];
            xv[m] = to_f32(x[i]);
            x2 += xv[m] * xv[m];
            xd += xv[m] * v[m];
        }
        if (d.normalize) {
            x2 = wave_sum(x2);
            xd = wave_sum(xd);
            const float c = 1.f / sqrtf(x2 + kNormEps);
#pragma unroll
            for (int m = 0; m < M; ++m) v[m] = c * (v[m] - c * c * xd * xv[m]);
        }
#pragma unroll
        for (int m = 0; m < M; ++m)
            if (lane + 64 * m < d.Dk) out[lane + 64 * m] = from_f32<T>(v[m]);
    }
}

struct ForwardLayout {
    size_t coef, t, p, total;
};
ForwardLayout forward_layout(long long chunk_heads) {
    ForwardLayout l{};
    l.coef = 0;
    l.t = align_up((size_t)chunk_heads * kCoefFloats * sizeof(float), 256);
    l.p = l.t + align_up((size_t)chunk_heads * kTriFloats * sizeof(float), 256);
    l.total = l.p + align_up((size_t)chunk_heads * kTriFloats * sizeof(float), 256);
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
    ForwardLayout f;
    size_t dstates, dx, dq, dk, total;
};
BackwardLayout backward_layout(const Dims& d) {
    BackwardLayout l{};
    l.f = forward_layout((long long)d.B * d.Hv * d.chunks);
    l.dstates = l.f.total;
    l.dx = l.dstates + align_up((size_t)d.B * d.Hv * d.chunks * d.Dk * d.Dv * sizeof(float), 256);
    l.dq = l.dx + align_up((size_t)d.B * d.T * d.Hv * d.Dv * sizeof(float), 256);
    l.dk = l.dq + align_up((size_t)d.B * d.T * d.Hv * d.Dk * sizeof(float), 256);
    l.total = l.dk + align_up((size_t)d.B * d.T * d.Hv * d.Dk * sizeof(float), 256);
    return l;
}

ChunkData chunk_data(char* ws, const ForwardLayout& l) {
    return ChunkData{reinterpret_cast<float*>(ws + l.coef), reinterpret_cast<float*>(ws + l.t),
                     reinterpret_cast<float*>(ws + l.p)};
}

template <typename T>
int forward(const Dims& d, const void* q, const void* k, const void* v, const void* g, const void* beta, const float* s0,
            const int* lengths, void* o, float* state_out, char* reserve, char* ws, hipStream_t s) {
    const ChunkData cd = chunk_data(ws, forward_layout((long long)d.B * d.Hv * d.chunks));
    const T *tq = static_cast<const T*>(q), *tk = static_cast<const T*>(k), *tv = static_cast<const T*>(v);
    RKA_RETURN_IF_ERR(launch_prepare<T>(d, tq, tk, g, beta, lengths, cd, false, s));
    const ReserveLayout r = reserve_layout(d);
    return launch_chain_forward<T>(d, tq, tk, tv, s0, lengths, cd, static_cast<T*>(o), state_out,
                                   reserve ? reinterpret_cast<float*>(reserve + r.states) : nullptr,
                                   reserve ? reinterpret_cast<float*>(reserve + r.e) : nullptr, s);
}

template <typename T>
int backward(const Dims& d, const void* q, const void* k, const void* g, const void* beta, const int* lengths,
             const char* reserve, const void* dout, const float* dstate_out, void* dq, void* dk, void* dv, void* dg,
             void* dbeta, float* ds0, char* ws, hipStream_t s) {
    const BackwardLayout l = backward_layout(d);
    const ReserveLayout r = reserve_layout(d);
    const ChunkData cd = chunk_data(ws, l.f);
    const T *tq = static_cast<const T*>(q), *tk = static_cast<const T*>(k), *tdo = static_cast<const T*>(dout);
    const BackwardData bd{reinterpret_cast<const float*>(reserve + r.states), reinterpret_cast<const float*>(reserve + r.e),
                          reinterpret_cast<float*>(ws + l.dstates), reinterpret_cast<float*>(ws + l.dx),
                          reinterpret_cast<float*>(ws + l.dq), reinterpret_cast<float*>(ws + l.dk)};
    RKA_RETURN_IF_ERR(launch_prepare<T>(d, tq, tk, g, beta, lengths, cd, true, s));
    RKA_RETURN_IF_ERR(
        launch_chain_backward<T>(d, tq, tk, tdo, dstate_out, lengths, cd, static_cast<T*>(dv), ds0, bd, s));
    const long long blocks = (long long)d.B * d.Hv * d.chunks;
    if (blocks == 0) return 0;
    RKA_RETURN_IF_ERR(check_grid(blocks, kThreads, "gated_delta_backward"));
    hipLaunchKernelGGL((gradients_kernel<T>), dim3((unsigned)blocks), dim3(kThreads), 0, s, d, tq, tk, tdo, g, lengths, cd,
                       bd, dg, dbeta);
    RKA_RETURN_IF_HIP(hipGetLastError());
    const long long rows = (long long)d.B * d.T * d.Hk, fin = (rows + kThreads / 64 - 1) / (kThreads / 64);
    RKA_RETURN_IF_ERR(check_grid(fin, kThreads, "gated_delta_backward"));
    hipLaunchKernelGGL((finish_kernel<T>), dim3((unsigned)fin), dim3(kThreads), 0, s, d, tq, tk, lengths, bd,
                       static_cast<T*>(dq), static_cast<T*>(dk));
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
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

template <typename T>
int launch_prepare(const Dims& d, const T* q, const T* k, const void* g, const void* beta, const int* lengths,
                   const ChunkData& out, bool transpose, hipStream_t stream) {
    const long long blocks = (long long)d.B * d.Hv * d.chunks;
    if (blocks == 0) return 0;
    RKA_RETURN_IF_ERR(check_grid(blocks, kThreads, "gated_delta"));
    if (transpose)
        hipLaunchKernelGGL((prepare_kernel<T, true>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, d, q, k, g, beta,
                           lengths, out);
    else
        hipLaunchKernelGGL((prepare_kernel<T, false>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, d, q, k, g, beta,
                           lengths, out);
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}

}  // namespace delta
}  // namespace rka

using namespace rka;
using namespace rka::delta;

extern "C" {

size_t rka_gated_delta_forward_workspace_bytes(int batch, int tokens, int key_heads, int value_heads, int key_dim,
                                               int value_dim) {
    Dims d;
    if (make_dims("gated_delta", batch, tokens, key_heads, value_heads, key_dim, value_dim, &d) != 0) return 0;
    return forward_layout((long long)d.B * d.Hv * d.chunks).total;
}

size_t rka_gated_delta_reserve_bytes(int batch, int tokens, int key_heads, int value_heads, int key_dim, int value_dim) {
    Dims d;
    if (make_dims("gated_delta", batch, tokens, key_heads, value_heads, key_dim, value_dim, &d) != 0) return 0;
    return reserve_layout(d).total;
}

size_t rka_gated_delta_backward_workspace_bytes(int batch, int tokens, int key_heads, int value_heads, int key_dim,
                                                int value_dim) {
    Dims d;
    if (make_dims("gated_delta", batch, tokens, key_heads, value_heads, key_dim, value_dim, &d) != 0) return 0;
    return backward_layout(d).total;
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
    const size_t need = forward_layout((long long)d.B * d.Hv * d.chunks).total;
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
    const size_t need = backward_layout(d).total;
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
