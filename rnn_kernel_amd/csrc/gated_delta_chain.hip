// The gated delta rule's chains over chunks, forward and backward (gated_delta.h has
// the formulas).  A wavefront takes 16 columns of the state through all chunks of its
// sequence; the state stays in its registers as the result of the matrix
// instructions that update it, and that layout (lane: column lane % 16, rows 4
// (lane / 16) .. + 3 of each 16x16 block) is also the one in which the next
// instruction takes its second operand, so nothing of the chain passes through LDS.
#include "gated_delta.h"

namespace rka {
namespace delta {
namespace {

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// 64 rows of a chunk's q or k as float32 in LDS, zero past `live` rows and Dk.
template <typename T, int KT>
__device__ __forceinline__ void stage_rows(float* lds, const T* src, long long stride, int live, int Dk, int tid,
                                           int threads) {
    constexpr int LD = KT * 16 + 4, Q = KT * 4;
    for (int i = tid; i < kChunk * Q; i += threads) {
        const int r = i / Q, d = i % Q * 4;
        f32x4 x{0.f, 0.f, 0.f, 0.f};
        if (r < live) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d + j < Dk) x[j] = to_f32(src[r * stride + d + j]);
        }
        *reinterpret_cast<f32x4*>(lds + r * LD + d) = x;
    }
}

template <typename T, int KT>
__global__ __launch_bounds__(256) void chain_forward_kernel(Dims d, const T* q, const T* k, const T* v, const float* s0,
                                                            const int* lengths, ChunkData in, T* o, float* state_out,
                                                            float* states, float* e_out) {
    extern __shared__ float lds[];
    constexpr int LD = KT * 16 + 4;
    float* ks = lds;
    float* qs = lds + kChunk * LD;
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid % 64, n = lane % 16, hi = lane / 16;
    const int cols = threads / 64 * 16, nblk = (d.Dv - 1) / cols + 1;
    const int bh = blockIdx.x / nblk, b = bh / d.Hv, h = bh % d.Hv, hk = h / (d.Hv / d.Hk);
    const int col = blockIdx.x % nblk * cols + tid / 64 * 16 + n;
    const bool ok = col < d.Dv;
    const int len = row_length(lengths, b, d.T);
    const size_t head = (size_t)bh * d.Dk * d.Dv;

    f32x4 s[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int dk = t * 16 + hi * 4 + r;
            s[t][r] = s0 && ok && dk < d.Dk ? s0[head + (size_t)dk * d.Dv + col] : 0.f;
        }
    const int live_chunks = (len + kChunk - 1) / kChunk;
    for (int c = 0; c < live_chunks; ++c) {
        const int t0 = c * kChunk, live = min(kChunk, len - t0);
        const size_t ch = (size_t)bh * d.chunks + c;
        __syncthreads();
        stage_rows<T, KT>(ks, k + b * d.k_s[0] + t0 * d.k_s[1] + hk * d.k_s[2], d.k_s[1], live, d.Dk, tid, threads);
        stage_rows<T, KT>(qs, q + b * d.q_s[0] + t0 * d.q_s[1] + hk * d.q_s[2], d.q_s[1], live, d.Dk, tid, threads);
        const float* coef = in.coef + ch * kCoefFloats;
        const float* tt = in.t + ch * kTriFloats;
        const float* pp = in.p + ch * kTriFloats;
        f32x4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * i + 4 * hi + r;
                x[i][r] = ok && row < live ? to_f32(v[b * d.v_s[0] + (long long)(t0 + row) * d.v_s[1] + h * d.v_s[2] + col]) : 0.f;
            }
        if (states && ok) {
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int dk = t * 16 + hi * 4 + r;
                    if (dk < d.Dk) states[(ch * d.Dk + dk) * d.Dv + col] = s[t][r];
                }
        }
        __syncthreads();
        f32x4 y[4] = {}, out[4] = {};
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(ks + (16 * i + n) * LD + t * 16 + hi * 4);
                const f32x4 aq = *reinterpret_cast<const f32x4*>(qs + (16 * i + n) * LD + t * 16 + hi * 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    y[i] = mfma4(a[r], s[t][r], y[i]);
                    out[i] = mfma4(aq[r], s[t][r], out[i]);
                }
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 rk = *reinterpret_cast<const f32x4*>(coef + RK * kChunk + 16 * i + 4 * hi);
            const f32x4 rq = *reinterpret_cast<const f32x4*>(coef + RQ * kChunk + 16 * i + 4 * hi);
            x[i] -= rk * y[i];
            out[i] *= rq;
        }
        f32x4 e[4] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(tt + (i * (i + 1) / 2 + j) * 256 + lane * 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) e[i] = mfma4(a[r], x[j][r], e[i]);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(pp + (i * (i + 1) / 2 + j) * 256 + lane * 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) out[i] = mfma4(a[r], e[j][r], out[i]);
            }
        const float last = coef[NCOEF * kChunk];
#pragma unroll
        for (int t = 0; t < KT; ++t) s[t] *= last;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(coef + WK * kChunk + 16 * i + 4 * hi) * e[i];
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    s[t] = mfma4(ks[(16 * i + 4 * hi + r) * LD + t * 16 + n], w[r], s[t]);
        }
        if (ok) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * i + 4 * hi + r;
                    if (row < live) {
                        const size_t at = (((size_t)b * d.T + t0 + row) * d.Hv + h) * d.Dv + col;
                        o[at] = from_f32<T>(out[i][r]);
                        if (e_out) e_out[at] = e[i][r];
                    }
                }
        }
    }
    if (!ok) return;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int dk = t * 16 + hi * 4 + r;
            if (dk < d.Dk) state_out[head + (size_t)dk * d.Dv + col] = s[t][r];
        }
    for (int t = len + hi; t < d.T; t += 4) o[(((size_t)b * d.T + t) * d.Hv + h) * d.Dv + col] = from_f32<T>(0.f);
}

template <typename T, int KT>
__global__ __launch_bounds__(256) void chain_backward_kernel(Dims d, const T* q, const T* k, const T* dout,
                                                             const float* dstate_out, const int* lengths, ChunkData in,
                                                             T* dv, float* ds0, BackwardData bd) {
    extern __shared__ float lds[];
    constexpr int LD = KT * 16 + 4;
    float* ks = lds;
    float* qs = lds + kChunk * LD;
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid % 64, n = lane % 16, hi = lane / 16;
    const int cols = threads / 64 * 16, nblk = (d.Dv - 1) / cols + 1;
    const int bh = blockIdx.x / nblk, b = bh / d.Hv, h = bh % d.Hv, hk = h / (d.Hv / d.Hk);
    const int col = blockIdx.x % nblk * cols + tid / 64 * 16 + n;
    const bool ok = col < d.Dv;
    const int len = row_length(lengths, b, d.T);
    const size_t head = (size_t)bh * d.Dk * d.Dv;

    f32x4 s[KT];  // dS'
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int dk = t * 16 + hi * 4 + r;
            s[t][r] = dstate_out && ok && dk < d.Dk ? dstate_out[head + (size_t)dk * d.Dv + col] : 0.f;
        }
    const int live_chunks = (len + kChunk - 1) / kChunk;
    for (int c = live_chunks - 1; c >= 0; --c) {
        const int t0 = c * kChunk, live = min(kChunk, len - t0);
        const size_t ch = (size_t)bh * d.chunks + c;
        __syncthreads();
        stage_rows<T, KT>(ks, k + b * d.k_s[0] + t0 * d.k_s[1] + hk * d.k_s[2], d.k_s[1], live, d.Dk, tid, threads);
        stage_rows<T, KT>(qs, q + b * d.q_s[0] + t0 * d.q_s[1] + hk * d.q_s[2], d.q_s[1], live, d.Dk, tid, threads);
        const float* coef = in.coef + ch * kCoefFloats;
        const float* tt = in.t + ch * kTriFloats;
        const float* pp = in.p + ch * kTriFloats;
        f32x4 go[4];  // dO
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * i + 4 * hi + r;
                const size_t at = (((size_t)b * d.T + t0 + row) * d.Hv + h) * d.Dv + col;
                go[i][r] = dout && ok && row < live ? to_f32(dout[at]) : 0.f;
            }
        if (ok) {
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int dk = t * 16 + hi * 4 + r;
                    if (dk < d.Dk) bd.dstates[(ch * d.Dk + dk) * d.Dv + col] = s[t][r];
                }
        }
        __syncthreads();
        f32x4 u[4] = {};
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(ks + (16 * i + n) * LD + t * 16 + hi * 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) u[i] = mfma4(a[r], s[t][r], u[i]);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] *= *reinterpret_cast<const f32x4*>(coef + WK * kChunk + 16 * i + 4 * hi);
        // block (i, j) transposed: rows j of the result from rows i of the operand
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(pp + (i * (i + 1) / 2 + j) * 256 + lane * 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) u[j] = mfma4(a[r], go[i][r], u[j]);
            }
        f32x4 x[4] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(tt + (i * (i + 1) / 2 + j) * 256 + lane * 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[j] = mfma4(a[r], u[i][r], x[j]);
            }
        const float last = coef[NCOEF * kChunk];
#pragma unroll
        for (int t = 0; t < KT; ++t) s[t] *= last;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 wo = *reinterpret_cast<const f32x4*>(coef + RQ * kChunk + 16 * i + 4 * hi) * go[i];
            const f32x4 wx = *reinterpret_cast<const f32x4*>(coef + RK * kChunk + 16 * i + 4 * hi) * x[i];
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[t] = mfma4(qs[(16 * i + 4 * hi + r) * LD + t * 16 + n], wo[r], s[t]);
                    s[t] = mfma4(-ks[(16 * i + 4 * hi + r) * LD + t * 16 + n], wx[r], s[t]);
                }
        }
        if (ok) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * i + 4 * hi + r;
                    if (row < live) {
                        const size_t at = (((size_t)b * d.T + t0 + row) * d.Hv + h) * d.Dv + col;
                        dv[at] = from_f32<T>(x[i][r]);
                        bd.dx[at] = x[i][r];
                    }
                }
        }
    }
    if (!ok) return;
    if (ds0) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int dk = t * 16 + hi * 4 + r;
                if (dk < d.Dk) ds0[head + (size_t)dk * d.Dv + col] = s[t][r];
            }
    }
    for (int t = len + hi; t < d.T; t += 4) dv[(((size_t)b * d.T + t) * d.Hv + h) * d.Dv + col] = from_f32<T>(0.f);
}

int waves_of(int Dv) { return std::min(4, (Dv + 15) / 16); }

// Calls f with the number of 16-row blocks that hold Dk, as an integral constant.
template <typename F>
int with_key_blocks(int Dk, F f) {
    if (Dk <= 64) return f(std::integral_constant<int, 4>{});
    if (Dk <= 128) return f(std::integral_constant<int, 8>{});
    if (Dk <= 192) return f(std::integral_constant<int, 12>{});
    return f(std::integral_constant<int, 16>{});
}

}  // namespace

template <typename T>
int launch_chain_forward(const Dims& d, const T* q, const T* k, const T* v, const float* s0, const int* lengths,
                         const ChunkData& in, T* o, float* state_out, float* states, float* e, hipStream_t stream) {
    const int waves = waves_of(d.Dv);
    const long long blocks = (long long)d.B * d.Hv * ((d.Dv - 1) / (16 * waves) + 1);
    RKA_RETURN_IF_ERR(check_grid(blocks, waves * 64, "gated_delta_forward"));
    return with_key_blocks(d.Dk, [&](auto kt) {
        constexpr int KT = decltype(kt)::value;
        const size_t lds = 2 * kChunk * (KT * 16 + 4) * sizeof(float);
        RKA_RETURN_IF_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&chain_forward_kernel<T, KT>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL((chain_forward_kernel<T, KT>), dim3((unsigned)blocks), dim3(waves * 64), lds, stream, d, q, k,
                           v, s0, lengths, in, o, state_out, states, e);
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    });
}

template <typename T>
int launch_chain_backward(const Dims& d, const T* q, const T* k, const T* dout, const float* dstate_out,
                          const int* lengths, const ChunkData& in, T* dv, float* ds0, const BackwardData& bd,
                          hipStream_t stream) {
    const int waves = waves_of(d.Dv);
    const long long blocks = (long long)d.B * d.Hv * ((d.Dv - 1) / (16 * waves) + 1);
    RKA_RETURN_IF_ERR(check_grid(blocks, waves * 64, "gated_delta_backward"));
    return with_key_blocks(d.Dk, [&](auto kt) {
        constexpr int KT = decltype(kt)::value;
        const size_t lds = 2 * kChunk * (KT * 16 + 4) * sizeof(float);
        RKA_RETURN_IF_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&chain_backward_kernel<T, KT>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL((chain_backward_kernel<T, KT>), dim3((unsigned)blocks), dim3(waves * 64), lds, stream, d, q,
                           k, dout, dstate_out, lengths, in, dv, ds0, bd);
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    });
}

#define RKA_DELTA_CHAIN(T)                                                                                         \
    template int launch_chain_forward<T>(const Dims&, const T*, const T*, const T*, const float*, const int*,     \
                                         const ChunkData&, T*, float*, float*, float*, hipStream_t);              \
    template int launch_chain_backward<T>(const Dims&, const T*, const T*, const T*, const float*, const int*,    \
                                          const ChunkData&, T*, float*, const BackwardData&, hipStream_t);
RKA_DELTA_CHAIN(float)
RKA_DELTA_CHAIN(bf16)

}  // namespace delta
}  // namespace rka
