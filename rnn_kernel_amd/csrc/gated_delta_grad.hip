// The gradients of the gated delta rule that are made for all chunks at once after the
// backward's chain (gated_delta.h has the formulas).
#include "gated_delta.h"

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

}  // namespace

template <typename T>
int launch_gradients(const Dims& d, const T* q, const T* k, const T* dout, const void* g, const int* lengths,
                     const ChunkData& in, const BackwardData& bd, T* dq, T* dk, void* dg, void* dbeta,
                     hipStream_t stream) {
    const long long blocks = (long long)d.B * d.Hv * d.chunks;
    if (blocks == 0) return 0;
    RKA_RETURN_IF_ERR(check_grid(blocks, kThreads, "gated_delta_backward"));
    hipLaunchKernelGGL((gradients_kernel<T>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, d, q, k, dout, g, lengths,
                       in, bd, dg, dbeta);
    RKA_RETURN_IF_HIP(hipGetLastError());
    const long long rows = (long long)d.B * d.T * d.Hk, fin = (rows + kThreads / 64 - 1) / (kThreads / 64);
    RKA_RETURN_IF_ERR(check_grid(fin, kThreads, "gated_delta_backward"));
    hipLaunchKernelGGL((finish_kernel<T>), dim3((unsigned)fin), dim3(kThreads), 0, stream, d, q, k, lengths, bd, dq, dk);
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}
template int launch_gradients<float>(const Dims&, const float*, const float*, const float*, const void*, const int*,
                                     const ChunkData&, const BackwardData&, float*, float*, void*, void*, hipStream_t);
template int launch_gradients<bf16>(const Dims&, const bf16*, const bf16*, const bf16*, const void*, const int*,
                                    const ChunkData&, const BackwardData&, bf16*, bf16*, void*, void*, hipStream_t);

}  // namespace delta
}  // namespace rka
