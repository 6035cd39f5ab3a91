// The causal convolution of each channel over few tokens, its gradients, and its form for
// single tokens:
//   z_t = b + sum_j w_j x_{t-W+1+j},  y = act(z);  x_{-W+1} .. x_{-1} are the initial state
//   dz = dy act'(z);  dx_s = sum_j w_j dz_{s+W-1-j};  dw_j = sum_t dz_t x_{t-W+1+j};  db = sum dz
// The final state is a row's last W - 1 inputs; its gradient adds to theirs.
//
// A thread takes 16 bytes of channels through a run of tokens, the last W - 1 inputs (and
// in the backward the last dz) in registers.  Bound by memory.
#include "elementwise.h"

#include <algorithm>

namespace rka {
namespace conv {
namespace {

using namespace elem;

constexpr int kMaxWidth = 8;
constexpr int kLanes = 64, kRuns = 4;  // channel groups and runs of a workgroup
constexpr int kForwardRun = 32, kBackwardRun = 32;

struct Dims {
    int B, T, D, act;
    long long xb, xt;  // x's strides: batch row, token
    const int* lengths;
};

__device__ __forceinline__ float activate(float z, int act) { return act == RKA_ACT_SILU ? z * sigmoid_fast(z) : z; }
__device__ __forceinline__ float slope(float z, int act) {
    const float s = sigmoid_fast(z);
    return act == RKA_ACT_SILU ? s * (1.f + z * (1.f - s)) : 1.f;
}

template <typename T, int W>
struct Weights {
    float w[W][kVec<T>], b[kVec<T>];

    __device__ __forceinline__ void load(const T* weight, const T* bias, int d0, int left) {
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e) {
            const int d = d0 + min(e, left - 1);
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][e] = to_f32(weight[(long long)d * W + j]);
            b[e] = bias ? to_f32(bias[d]) : 0.f;
        }
    }
    __device__ __forceinline__ float z(const float (&x)[W][kVec<T>], int e) const {
        float sum = b[e];
#pragma unroll
        for (int j = 0; j < W; ++j) sum = fmaf(w[j][e], x[j][e], sum);
        return sum;
    }
};

// Input t of a row with `len` tokens: from the initial state before the first, 0 behind the
// last.
template <typename T, int W>
__device__ __forceinline__ Piece<T> input(const Dims& d, const T* x, const T* initial, int b, int t, int len, int d0, int left) {
    if (t >= 0 && t < len) return load_piece(x + b * d.xb + t * d.xt + d0, left);
    if (t >= -(W - 1) && t < 0 && initial) return load_piece(initial + ((long long)b * (W - 1) + t + W - 1) * d.D + d0, left);
    Piece<T> none;
    none.u = u32x4{0, 0, 0, 0};
    return none;
}

template <typename T, int W>
__global__ __launch_bounds__(kLanes* kRuns) void forward_kernel(Dims d, const T* x, const T* weight, const T* bias,
                                                                const T* initial, T* y, T* final_state) {
    constexpr int V = kVec<T>;
    const int b = blockIdx.z, d0 = (blockIdx.x * kLanes + threadIdx.x) * V, left = d.D - d0;
    const int run = blockIdx.y * kRuns + threadIdx.y;
    const long long first = (long long)run * kForwardRun;
    if (left <= 0 || first > d.T) return;
    const int t0 = (int)first, t1 = min(d.T, t0 + min(kForwardRun, d.T - t0)), len = row_length(d.lengths, b, d.T);
    if (run == 0) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
            store_piece(final_state + ((long long)b * (W - 1) + j) * d.D + d0,
                        input<T, W>(d, x, initial, b, len - (W - 1) + j, len, d0, left), left);
    }
    if (t0 >= d.T) return;
    Weights<T, W> wt;
    wt.load(weight, bias, d0, left);
    float win[W][V];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        const Piece<T> p = input<T, W>(d, x, initial, b, t0 - (W - 1) + j, len, d0, left);
#pragma unroll
        for (int e = 0; e < V; ++e) win[j][e] = to_f32(p.e[e]);
    }
    T* py = y + ((long long)b * d.T + t0) * d.D + d0;
#pragma unroll 4
    for (int t = t0; t < t1; ++t, py += d.D) {
        const Piece<T> p = input<T, W>(d, x, initial, b, t, len, d0, left);
        Piece<T> out;
#pragma unroll
        for (int e = 0; e < V; ++e) win[W - 1][e] = to_f32(p.e[e]);
#pragma unroll
        for (int e = 0; e < V; ++e) out.e[e] = from_f32<T>(t < len ? activate(wt.z(win, e), d.act) : 0.f);
        store_piece(py, out, left);
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) win[j][e] = win[j + 1][e];
    }
}

// Run r takes the dz of tokens [r R, r R + R) of [0, T + W - 1) (those from the length on
// are 0) and the dx that the last of them completes, those of tokens [r R - W + 1,
// r R + R - W + 1), where tokens before 0 are the initial state's; the dz before its first
// it makes again.  Sums of dw and db: [batch row][workgroup's runs][W + 1][channels].
template <typename T, int W>
__global__ __launch_bounds__(kLanes* kRuns) void backward_kernel(Dims d, const T* dy, const T* dstate, const T* x,
                                                                 const T* weight, const T* bias, const T* initial, T* dx,
                                                                 T* dinitial, float* sums) {
    constexpr int V = kVec<T>;
    __shared__ float part[kRuns - 1][V][kLanes];
    const int b = blockIdx.z, d0 = (blockIdx.x * kLanes + threadIdx.x) * V, left = d.D - d0;
    const int len = row_length(d.lengths, b, d.T);
    const long long first = (long long)(blockIdx.y * kRuns + threadIdx.y) * kBackwardRun;
    float dw[W][V] = {}, db[V] = {};
    if (left > 0 && first < (long long)d.T + W - 1) {
        const int t0 = (int)first, t1 = (int)min(first + kBackwardRun, (long long)d.T + W - 1);
        Weights<T, W> wt;
        wt.load(weight, bias, d0, left);
        float win[W][V], dz[W][V] = {};  // inputs up to t; dz up to t
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            const Piece<T> p = input<T, W>(d, x, initial, b, t0 - 2 * (W - 1) + j, len, d0, left);
#pragma unroll
            for (int e = 0; e < V; ++e) win[j][e] = to_f32(p.e[e]);
        }
#pragma unroll 2
        for (int t = t0 - (W - 1); t < t1; ++t) {
            const Piece<T> p = input<T, W>(d, x, initial, b, t, len, d0, left);
#pragma unroll
            for (int e = 0; e < V; ++e) win[W - 1][e] = to_f32(p.e[e]);
            const bool on = t >= 0 && t < len && dy;
            if (on) {
                const Piece<T> g = load_piece(dy + ((long long)b * d.T + t) * d.D + d0, left);
#pragma unroll
                for (int e = 0; e < V; ++e) dz[W - 1][e] = to_f32(g.e[e]) * slope(wt.z(win, e), d.act);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) dz[W - 1][e] = 0.f;
            }
            if (t >= t0) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    db[e] += dz[W - 1][e];
#pragma unroll
                    for (int j = 0; j < W; ++j) dw[j][e] = fmaf(dz[W - 1][e], win[j][e], dw[j][e]);
                }
                const int s = t - (W - 1);
                T* to = s >= 0 ? dx : dinitial;
                if (to && s < d.T) {
                    float sum[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        sum[e] = 0.f;
#pragma unroll
                        for (int j = 0; j < W; ++j) sum[e] = fmaf(wt.w[j][e], dz[W - 1 - j][e], sum[e]);
                    }
                    const int kept = s - (len - (W - 1));  // its place in the final state
                    if (dstate && kept >= 0 && kept < W - 1) {
                        const Piece<T> g = load_piece(dstate + ((long long)b * (W - 1) + kept) * d.D + d0, left);
#pragma unroll
                        for (int e = 0; e < V; ++e) sum[e] += to_f32(g.e[e]);
                    }
                    Piece<T> out;
#pragma unroll
                    for (int e = 0; e < V; ++e) out.e[e] = from_f32<T>(sum[e]);
                    to += s >= 0 ? ((long long)b * d.T + s) * d.D : ((long long)b * (W - 1) + s + W - 1) * d.D;
                    store_piece(to + d0, out, left);
                }
            }
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    win[j][e] = win[j + 1][e];
                    dz[j][e] = dz[j + 1][e];
                }
        }
    }
    if (!sums) return;
    float* to = sums + ((long long)b * gridDim.y + blockIdx.y) * (W + 1) * d.D + d0;
#pragma unroll
    for (int j = 0; j <= W; ++j) {
        float* own = j < W ? dw[j < W ? j : 0] : db;
        __syncthreads();
        if (threadIdx.y > 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) part[threadIdx.y - 1][e][threadIdx.x] = own[e];
        }
        __syncthreads();
        if (threadIdx.y == 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float s = own[e];
#pragma unroll
                for (int k = 0; k < kRuns - 1; ++k) s += part[k][e][threadIdx.x];
                if (e < left) to[(long long)j * d.D + e] = s;
            }
        }
    }
}

// dw and db from the sums, always in their order.
template <typename T>
__global__ __launch_bounds__(256) void sums_kernel(const float* sums, int count, int D, int W, T* dweight, T* dbias) {
    __shared__ float part[8][33];
    const int c = threadIdx.x % 32, p = threadIdx.x / 32, col = blockIdx.x * 32 + c, j = blockIdx.y;
    float s = 0.f;
    if (col < D) {
#pragma unroll 8
        for (int r = p; r < count; r += 8) s += sums[((size_t)r * (W + 1) + j) * D + col];
    }
    part[p][c] = s;
    __syncthreads();
    if (p != 0 || col >= D) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) s += part[k][c];
    if (j < W) {
        if (dweight) dweight[(long long)col * W + j] = from_f32<T>(s);
    } else if (dbias) {
        dbias[col] = from_f32<T>(s);
    }
}

template <typename T, int W>
__global__ __launch_bounds__(kLanes) void step_kernel(int B, int D, int act, const T* x, long long ldx, const T* weight,
                                                      const T* bias, T* state, const int* slots, int num_slots, T* y) {
    constexpr int V = kVec<T>;
    const int groups = (D - 1) / (kLanes * V) + 1;
    const int b = blockIdx.x / groups, d0 = (blockIdx.x % groups * kLanes + threadIdx.x) * V, left = D - d0;
    if (left <= 0) return;
    const int slot = slots ? slots[b] : b;
    Piece<T> out;
    T* py = y + (long long)b * D + d0;
    if (slot < 0 || slot >= num_slots) {
        // a request without a state: nothing is read or written but its output
#pragma unroll
        for (int e = 0; e < V; ++e) out.e[e] = from_f32<T>(slot < 0 ? 0.f : __builtin_nanf(""));
        store_piece(py, out, left);
        return;
    }
    T* ps = state + (long long)slot * (W - 1) * D + d0;
    Piece<T> p[W];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) p[j] = load_piece(ps + (long long)j * D, left);
    p[W - 1] = load_piece(x + b * ldx + d0, left);
    Weights<T, W> wt;
    wt.load(weight, bias, d0, left);
    float win[W][V];
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) win[j][e] = to_f32(p[j].e[e]);
#pragma unroll
    for (int e = 0; e < V; ++e) out.e[e] = from_f32<T>(activate(wt.z(win, e), act));
    store_piece(py, out, left);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_piece(ps + (long long)j * D, p[j + 1], left);
}

template <typename F>
int with_width(int width, F f) {
    switch (width) {
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 5: return f(std::integral_constant<int, 5>{});
        case 6: return f(std::integral_constant<int, 6>{});
        case 7: return f(std::integral_constant<int, 7>{});
        default: return f(std::integral_constant<int, 8>{});
    }
}

int blocks_of_runs(long long tokens, int run) { return (int)((std::max(tokens, 1LL) - 1) / ((long long)run * kRuns) + 1); }
dim3 grid(const Dims& d, int esize, int run_blocks) {
    return dim3((unsigned)((d.D - 1) / (kLanes * (16 / esize)) + 1), (unsigned)run_blocks, (unsigned)d.B);
}
// (65535 is the most of a grid's second and third size)
int check_sizes(const char* what, const Dims& d, int width, int dtype) {
    const std::string name(what);
    if (d.B < 0 || d.T < 0 || d.D < 1) return fail(RKA_ERR_INVALID_ARGUMENT, name + ": batch and tokens must be >= 0, channels >= 1");
    if (width < 2 || width > kMaxWidth) return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": width must be in [2, 8]");
    if (d.act != RKA_ACT_NONE && d.act != RKA_ACT_SILU) return fail(RKA_ERR_INVALID_ARGUMENT, name + ": activation must be none or silu");
    if (d.B > 65535 || d.T > 65535 * 64) return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": batch exceeds 65535 or tokens 2^22 - 64");
    return check_dtype(dtype, what);
}

template <typename T>
int forward(const Dims& d, const void* x, const void* weight, const void* bias, const void* initial, void* y,
            void* final_state, int width, hipStream_t s) {
    const dim3 blocks = grid(d, sizeof(T), blocks_of_runs(d.T, kForwardRun));
    RKA_RETURN_IF_ERR(check_grid((long long)blocks.x * blocks.y * blocks.z, kLanes * kRuns, "causal_conv_forward"));
    return with_width(width, [&](auto w) {
        hipLaunchKernelGGL((forward_kernel<T, decltype(w)::value>), blocks, dim3(kLanes, kRuns), 0, s, d, static_cast<const T*>(x), static_cast<const T*>(weight),
                           static_cast<const T*>(bias), static_cast<const T*>(initial), static_cast<T*>(y),
                           static_cast<T*>(final_state));
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    });
}

template <typename T>
int backward(const Dims& d, const void* dy, const void* dstate, const void* x, const void* weight, const void* bias,
             const void* initial, void* dx, void* dweight, void* dbias, void* dinitial, float* sums, int width,
             hipStream_t s) {
    const int runs = blocks_of_runs((long long)d.T + width - 1, kBackwardRun);
    if (!dweight && !dbias) sums = nullptr;
    const dim3 blocks = grid(d, sizeof(T), runs);
    RKA_RETURN_IF_ERR(check_grid((long long)blocks.x * blocks.y * blocks.z, kLanes * kRuns, "causal_conv_backward"));
    RKA_RETURN_IF_ERR(with_width(width, [&](auto w) {
        hipLaunchKernelGGL((backward_kernel<T, decltype(w)::value>), blocks, dim3(kLanes, kRuns), 0, s, d,
                           static_cast<const T*>(dy), static_cast<const T*>(dstate), static_cast<const T*>(x),
                           static_cast<const T*>(weight), static_cast<const T*>(bias), static_cast<const T*>(initial),
                           static_cast<T*>(dx), static_cast<T*>(dinitial), sums);
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    }));
    if (sums) {
        hipLaunchKernelGGL((sums_kernel<T>), dim3((d.D - 1) / 32 + 1, width + 1), dim3(256), 0, s, sums, runs * d.B, d.D, width,
                           static_cast<T*>(dweight), static_cast<T*>(dbias));
        RKA_RETURN_IF_HIP(hipGetLastError());
    }
    return 0;
}

template <typename T>
int step(int B, int D, int act, const void* x, long long ldx, const void* weight, const void* bias, void* state,
         const int* slots, int num_slots, void* y, int width, hipStream_t s) {
    const long long blocks = (long long)B * ((D - 1) / (kLanes * kVec<T>) + 1);
    RKA_RETURN_IF_ERR(check_grid(blocks, kLanes, "causal_conv_step"));
    return with_width(width, [&](auto w) {
        hipLaunchKernelGGL((step_kernel<T, decltype(w)::value>), dim3((unsigned)blocks), dim3(kLanes), 0, s, B, D, act,
                           static_cast<const T*>(x), ldx, static_cast<const T*>(weight), static_cast<const T*>(bias),
                           static_cast<T*>(state), slots, num_slots, static_cast<T*>(y));
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    });
}

}  // namespace
}  // namespace conv
}  // namespace rka

using namespace rka;
using namespace rka::conv;

extern "C" {

int rka_causal_conv_forward(const void* x, long long x_batch_stride, long long x_token_stride, const void* weight,
                            const void* bias, const void* initial_state, const int* lengths, void* y, void* final_state,
                            int batch, int tokens, int channels, int width, int act, int dtype, void* stream) {
    clear_error();
    const Dims d{batch, tokens, channels, act, x_batch_stride, x_token_stride, lengths};
    RKA_RETURN_IF_ERR(check_sizes("causal_conv_forward", d, width, dtype));
    if (batch == 0) return 0;
    if ((tokens > 0 && (!x || !y)) || !weight || !final_state)
        return fail(RKA_ERR_INVALID_ARGUMENT, "causal_conv_forward: null tensor pointer");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return dtype == RKA_DTYPE_F32 ? forward<float>(d, x, weight, bias, initial_state, y, final_state, width, s)
                                  : forward<bf16>(d, x, weight, bias, initial_state, y, final_state, width, s);
}

size_t rka_causal_conv_backward_workspace_bytes(int batch, int tokens, int channels, int width) {
    if (batch < 1 || tokens < 0 || channels < 1 || width < 2 || width > kMaxWidth) return 0;
    return (size_t)batch * blocks_of_runs((long long)tokens + width - 1, kBackwardRun) * (width + 1) * channels * sizeof(float);
}

int rka_causal_conv_backward(const void* grad_y, const void* grad_final_state, const void* x, long long x_batch_stride,
                             long long x_token_stride, const void* weight, const void* bias, const void* initial_state,
                             const int* lengths, void* grad_x, void* grad_weight, void* grad_bias, void* grad_initial_state,
                             void* workspace, size_t workspace_bytes, int batch, int tokens, int channels, int width, int act,
                             int dtype, void* stream) {
    clear_error();
    const Dims d{batch, tokens, channels, act, x_batch_stride, x_token_stride, lengths};
    RKA_RETURN_IF_ERR(check_sizes("causal_conv_backward", d, width, dtype));
    if (batch < 1) return fail(RKA_ERR_INVALID_ARGUMENT, "causal_conv_backward: batch must be >= 1");
    if ((tokens > 0 && !x) || !weight) return fail(RKA_ERR_INVALID_ARGUMENT, "causal_conv_backward: null tensor pointer");
    if (grad_weight || grad_bias)
        RKA_RETURN_IF_ERR(check_workspace(workspace, workspace_bytes,
                                          rka_causal_conv_backward_workspace_bytes(batch, tokens, channels, width),
                                          "causal_conv_backward"));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    float* sums = static_cast<float*>(workspace);
    return dtype == RKA_DTYPE_F32
               ? backward<float>(d, grad_y, grad_final_state, x, weight, bias, initial_state, grad_x, grad_weight, grad_bias,
                                 grad_initial_state, sums, width, s)
               : backward<bf16>(d, grad_y, grad_final_state, x, weight, bias, initial_state, grad_x, grad_weight, grad_bias,
                                grad_initial_state, sums, width, s);
}

int rka_causal_conv_step(const void* x, long long ldx, const void* weight, const void* bias, void* state, const int* slots,
                         int num_slots, void* y, int batch, int channels, int width, int act, int dtype, void* stream) {
    clear_error();
    const Dims d{batch < 0 ? -1 : 0, 1, channels, act, 0, 0, nullptr};
    RKA_RETURN_IF_ERR(check_sizes("causal_conv_step", d, width, dtype));
    if (num_slots < 0 || (!slots && num_slots < batch))
        return fail(RKA_ERR_INVALID_ARGUMENT, "causal_conv_step: fewer states than requests");
    if (batch == 0) return 0;
    if (!x || !weight || !state || !y) return fail(RKA_ERR_INVALID_ARGUMENT, "causal_conv_step: null tensor pointer");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return dtype == RKA_DTYPE_F32 ? step<float>(batch, channels, act, x, ldx, weight, bias, state, slots, num_slots, y, width, s)
                                  : step<bf16>(batch, channels, act, x, ldx, weight, bias, state, slots, num_slots, y, width, s);
}

}  // extern "C"
