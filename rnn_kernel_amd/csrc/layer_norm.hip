// Layer norm over rows and its gradients:
//   u = (x - mean) rstd, rstd = 1 / sqrt(var + eps);  y = u w + b
//   g = dy w;  dx = rstd (g - mean(g) - u mean(g u));  dw = sum over rows of dy u;  db = of dy
//
// A row is in registers between its one read and its one write: mean first, then the
// squares of what is left, so that a large mean takes nothing from the variance.  Bound by
// memory: 65536 rows of 2048 bf16 take 96 us forward (5.6 TB/s of x and y; a copy of 4 GiB 4.8)
// and 162 us backward (5.0 TB/s of dy, x and dx, the columns' sums 5 us of it); 1000 rows of 385
// float32 4 and 5 us, a launch's latency.  Backwards wide rows are slower, bound by barriers and, with
// sixteen wavefronts, spills: 2^26 elements of float32 in rows of 8192 take 109 and 197 us, of bf16 in
// rows of 16384 47 and 148; and rows that fill few lanes of their wavefront: of 64 bf16 308 and 627.
#include "elementwise.h"

#include <algorithm>

namespace rka {
namespace norm {
namespace {

using namespace elem;

constexpr int kMaxSize = 16384;

// Sum over the WAVES wavefronts that share a row, always in the same order.
template <int WAVES>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
    v = wave_sum(v);
    if constexpr (WAVES > 1) {
        __syncthreads();
        if (threadIdx.x % 64 == 0) scratch[threadIdx.x / 64] = v;
        __syncthreads();
        v = scratch[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v += scratch[i];
    }
    return v;
}

// WAVES wavefronts to a row (1: the four of a workgroup have a row each), P pieces of 16
// bytes to a lane.
template <int WAVES>
constexpr int kThreads = WAVES == 1 ? 256 : WAVES * 64;

template <typename T, int WAVES, int P>
__global__ __launch_bounds__(kThreads<WAVES>) void forward_kernel(const T* x, long long ldx, const T* weight, const T* bias,
                                                                  T* y, float* mean, float* rstd, int rows, int size,
                                                                  float eps) {
    constexpr int V = kVec<T>, kRows = kThreads<WAVES> / 64 / WAVES, kLanes = 64 * WAVES;
    __shared__ float scratch[WAVES];
    const int lane = threadIdx.x % kLanes;
    const long long row = (long long)blockIdx.x * kRows + threadIdx.x / kLanes;
    if (row >= rows) return;
    const T* px = x + row * ldx;
    Piece<T> p[P];
    float v[P][V], sum = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) p[i] = load_piece(px + (i * kLanes + lane) * V, size - (i * kLanes + lane) * V);
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            v[i][j] = to_f32(p[i].e[j]);
            sum += v[i][j];
        }
    const float m = row_sum<WAVES>(sum, scratch) / size;
    float squares = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            v[i][j] = (i * kLanes + lane) * V + j < size ? v[i][j] - m : 0.f;
            squares += v[i][j] * v[i][j];
        }
    const float r = 1.f / sqrtf(row_sum<WAVES>(squares, scratch) / size + eps);
    if (mean && lane == 0) {
        mean[row] = m;
        rstd[row] = r;
    }
    T* py = y + row * size;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int at = (i * kLanes + lane) * V, left = size - at;
        if (left <= 0) break;
        Piece<T> w, b, out;
        if (weight) w = load_piece(weight + at, left);
        if (bias) b = load_piece(bias + at, left);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float z = v[i][j] * r;
            if (weight) z *= to_f32(w.e[j]);
            if (bias) z += to_f32(b.e[j]);
            out.e[j] = from_f32<T>(z);
        }
        store_piece(py + at, out, left);
    }
}

// The rows of a workgroup, one after another: their columns' sums stay in registers, in
// `sums` as [workgroup][dw, db][size] in the end.
template <typename T, int WAVES, int P>
__global__ __launch_bounds__(kThreads<WAVES>) void backward_kernel(const T* dy, long long lddy, const T* x, long long ldx,
                                                                   const T* weight, const float* mean, const float* rstd,
                                                                   T* dx, float* sums, int rows, int size) {
    constexpr int V = kVec<T>, kRows = kThreads<WAVES> / 64 / WAVES, kLanes = 64 * WAVES;
    __shared__ float scratch[WAVES];
    __shared__ float part[kRows > 1 ? kRows - 1 : 1][kRows > 1 ? 64 * V : 1];
    const int lane = threadIdx.x % kLanes;
    float dw[P][V] = {}, db[P][V] = {}, w[P][V];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int at = (i * kLanes + lane) * V;
        Piece<T> q;
        if (weight) q = load_piece(weight + at, size - at);
#pragma unroll
        for (int j = 0; j < V; ++j) w[i][j] = weight ? to_f32(q.e[j]) : 1.f;
    }
    for (long long row = (long long)blockIdx.x * kRows + threadIdx.x / kLanes; row < rows; row += (long long)gridDim.x * kRows) {
        Piece<T> px[P], pd[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int at = (i * kLanes + lane) * V;
            px[i] = load_piece(x + row * ldx + at, size - at);
            pd[i] = load_piece(dy + row * lddy + at, size - at);
        }
        const float m = mean[row], r = rstd[row];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = to_f32(pd[i].e[j]), u = (to_f32(px[i].e[j]) - m) * r, g = d * w[i][j];
                s1 += g;
                s2 += g * u;
                db[i][j] += d;
                dw[i][j] += d * u;
            }
        if (!dx) continue;
        s1 = row_sum<WAVES>(s1, scratch) / size;
        s2 = row_sum<WAVES>(s2, scratch) / size;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int at = (i * kLanes + lane) * V, left = size - at;
            if (left <= 0) break;
            Piece<T> out;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = to_f32(pd[i].e[j]), u = (to_f32(px[i].e[j]) - m) * r;
                out.e[j] = from_f32<T>(r * (d * w[i][j] - s1 - u * s2));
            }
            store_piece(dx + row * size + at, out, left);
        }
    }
    if (!sums) return;
    float* to = sums + (size_t)blockIdx.x * 2 * size;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float* own = which ? db[i] : dw[i];
            if constexpr (kRows > 1) {
                const int of = threadIdx.x / 64;
                __syncthreads();
                if (of > 0) {
#pragma unroll
                    for (int j = 0; j < V; ++j) part[of - 1][j * 64 + lane] = own[j];
                }
                __syncthreads();
                if (of > 0) continue;
#pragma unroll
                for (int k = 0; k < kRows - 1; ++k)
#pragma unroll
                    for (int j = 0; j < V; ++j) own[j] += part[k][j * 64 + lane];
            }
            const int at = (i * kLanes + lane) * V;
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (at + j < size) to[which * size + at + j] = own[j];
        }
}

// dw and db from the workgroups' sums, always in their order: 32 columns and 8 ranges of
// workgroups to a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void columns_kernel(const float* sums, int count, int size, T* dweight, T* dbias) {
    __shared__ float part[8][33];
    const int c = threadIdx.x % 32, p = threadIdx.x / 32, col = blockIdx.x * 32 + c, which = blockIdx.y;
    T* out = which ? dbias : dweight;
    if (!out) return;
    float s = 0.f;
    if (col < size) {
#pragma unroll 8
        for (int r = p; r < count; r += 8) s += sums[((size_t)r * 2 + which) * size + col];
    }
    part[p][c] = s;
    __syncthreads();
    if (p != 0 || col >= size) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) s += part[k][c];
    out[col] = from_f32<T>(s);
}

// Calls f with the wavefronts of a row and the pieces of a lane as constants: as few wavefronts
// as hold a row in 64 registers or so, as sums between them wait at barriers.  2^27 elements of
// bf16, forward and backward, in rows of 1024: one wavefront 98 and 152 us, four 185 and 416; of 2048
// 96 and 162, 124 and 232; of 4096: four 112 and 203, sixteen 196 and 292.
template <typename T, typename F>
int with_form(int size, F f) {
    const int pieces = (size - 1) / kVec<T> + 1;
    const auto form = [&](auto waves, auto p) { return f(waves, p); };
    if (pieces <= 64) return form(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
    if (pieces <= 128) return form(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
    if (pieces <= 256) return form(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
    if (pieces <= 1024) return form(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
    return form(std::integral_constant<int, 16>{}, std::integral_constant<int, kMaxSize / 1024 / kVec<T>>{});
}

// Workgroups of the backward, each with sums of its own: 2^27 elements in rows of 2048 take 170,
// 162 and 171 us with at most 256, 512 and 1024, in rows of 4096 304, 203 and 221.
int backward_blocks(int rows, int size, int esize) {
    const int a_block = (size - 1) / (16 / esize) + 1 <= 256 ? 4 : 1;
    return (int)std::min<long long>(((long long)rows - 1) / a_block + 1, 512);
}

template <typename T>
int forward(const void* x, long long ldx, const void* weight, const void* bias, void* y, float* mean, float* rstd, int rows,
            int size, double eps, hipStream_t s) {
    return with_form<T>(size, [&](auto waves, auto p) {
        constexpr int W = decltype(waves)::value, P = decltype(p)::value, kRows = W == 1 ? 4 : 1;
        // (as many rows to a launch as it may have threads for)
        constexpr int kMost = (int)(((1LL << 32) - 1) / kThreads<W>) * kRows;
        for (long long row = 0; row < rows; row += kMost) {
            const int some = (int)std::min<long long>(kMost, rows - row);
            hipLaunchKernelGGL((forward_kernel<T, W, P>), dim3((unsigned)((some - 1) / kRows + 1)), dim3(kThreads<W>), 0, s,
                               static_cast<const T*>(x) + row * ldx, ldx, static_cast<const T*>(weight), static_cast<const T*>(bias),
                               static_cast<T*>(y) + row * size, mean ? mean + row : nullptr, rstd ? rstd + row : nullptr, some, size,
                               (float)eps);
            RKA_RETURN_IF_HIP(hipGetLastError());
        }
        return 0;
    });
}

template <typename T>
int backward(const void* dy, long long lddy, const void* x, long long ldx, const void* weight, const float* mean,
             const float* rstd, void* dx, void* dweight, void* dbias, float* sums, int rows, int size, hipStream_t s) {
    const int blocks = backward_blocks(rows, size, sizeof(T));
    if (!dweight && !dbias) sums = nullptr;
    RKA_RETURN_IF_ERR(with_form<T>(size, [&](auto waves, auto p) {
        constexpr int W = decltype(waves)::value, P = decltype(p)::value;
        hipLaunchKernelGGL((backward_kernel<T, W, P>), dim3(blocks), dim3(kThreads<W>), 0, s, static_cast<const T*>(dy), lddy,
                           static_cast<const T*>(x), ldx, static_cast<const T*>(weight), mean, rstd, static_cast<T*>(dx),
                           sums, rows, size);
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    }));
    if (sums) {
        hipLaunchKernelGGL((columns_kernel<T>), dim3((size - 1) / 32 + 1, 2), dim3(256), 0, s, sums, blocks, size,
                           static_cast<T*>(dweight), static_cast<T*>(dbias));
        RKA_RETURN_IF_HIP(hipGetLastError());
    }
    return 0;
}

int check(const char* what, int rows, int size, long long ld0, long long ld1, int dtype) {
    if (rows < 0 || size < 1) return fail(RKA_ERR_INVALID_ARGUMENT, std::string(what) + ": rows must be >= 0 and size >= 1");
    if (size > kMaxSize) return fail(RKA_ERR_UNSUPPORTED_SHAPE, std::string(what) + ": size exceeds " + std::to_string(kMaxSize));
    if (ld0 < 0 || ld1 < 0) return fail(RKA_ERR_INVALID_ARGUMENT, std::string(what) + ": row strides must be >= 0");
    return check_dtype(dtype, what);
}

}  // namespace
}  // namespace norm
}  // namespace rka

using namespace rka;
using namespace rka::norm;

extern "C" {

int rka_layer_norm_forward(const void* x, long long ldx, const void* weight, const void* bias, void* y, float* mean,
                           float* rstd, int rows, int size, double eps, int dtype, void* stream) {
    clear_error();
    RKA_RETURN_IF_ERR(check("layer_norm_forward", rows, size, ldx, 0, dtype));
    if (rows == 0) return 0;
    if (!x || !y || !mean != !rstd) return fail(RKA_ERR_INVALID_ARGUMENT, "layer_norm_forward: null tensor pointer");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return dtype == RKA_DTYPE_F32 ? forward<float>(x, ldx, weight, bias, y, mean, rstd, rows, size, eps, s)
                                  : forward<bf16>(x, ldx, weight, bias, y, mean, rstd, rows, size, eps, s);
}

size_t rka_layer_norm_backward_workspace_bytes(int rows, int size, int dtype) {
    if (rows < 1 || size < 1 || size > kMaxSize) return 0;
    return (size_t)backward_blocks(rows, size, dtype == RKA_DTYPE_F32 ? 4 : 2) * 2 * size * sizeof(float);
}

int rka_layer_norm_backward(const void* grad_y, long long ldy, const void* x, long long ldx, const void* weight,
                            const float* mean, const float* rstd, void* grad_x, void* grad_weight, void* grad_bias,
                            void* workspace, size_t workspace_bytes, int rows, int size, int dtype, void* stream) {
    clear_error();
    RKA_RETURN_IF_ERR(check("layer_norm_backward", rows, size, ldx, ldy, dtype));
    if (rows < 1) return fail(RKA_ERR_INVALID_ARGUMENT, "layer_norm_backward: rows must be >= 1");
    if (!grad_y || !x || !mean || !rstd) return fail(RKA_ERR_INVALID_ARGUMENT, "layer_norm_backward: null tensor pointer");
    if (grad_weight || grad_bias)
        RKA_RETURN_IF_ERR(check_workspace(workspace, workspace_bytes, rka_layer_norm_backward_workspace_bytes(rows, size, dtype),
                                          "layer_norm_backward"));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    float* sums = static_cast<float*>(workspace);
    return dtype == RKA_DTYPE_F32
               ? backward<float>(grad_y, ldy, x, ldx, weight, mean, rstd, grad_x, grad_weight, grad_bias, sums, rows, size, s)
               : backward<bf16>(grad_y, ldy, x, ldx, weight, mean, rstd, grad_x, grad_weight, grad_bias, sums, rows, size, s);
}

}  // extern "C"
