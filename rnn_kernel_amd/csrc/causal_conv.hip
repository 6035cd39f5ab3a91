// The causal convolution of each channel over few tokens, its gradients, and its form for
// single tokens:
//   z_t = b + sum_j w_j x_{t-W+1+j},  y = act(z);  x_{-W+1} .. x_{-1} are the initial state
//   dz = dy act'(z);  dx_s = sum_j w_j dz_{s+W-1-j};  dw_j = sum_t dz_t x_{t-W+1+j};  db = sum dz
// The final state is a row's last W - 1 inputs; its gradient adds to theirs.
//
// A thread takes four channels through a run of tokens, whose inputs it loads at once: what it
// needs of its neighbours' tokens it loads and makes again (from L2).  Bound by memory: 16 x 2048
// tokens of 2048 channels, width 4, bf16 take 51 us forward (5.3 TB/s of x and y) and 100 backward
// (4.0 TB/s of dy, x and dx), float32 103 and 170; a quarter of them, which caches hold, 19 and 28 us, a third of it
// the exponentials.  Token by token with one channel to a thread 98 us instead of the last two and
// the sums.
#include "elementwise.h"

#include <algorithm>
#include <type_traits>

namespace rka {
namespace conv {
namespace {

using namespace elem;

constexpr int kMaxWidth = 8;
constexpr int kLanes = 64, kRuns = 4;  // groups of channels and runs of a workgroup
constexpr int kGroup = 4;              // channels of a thread
// Tokens of a run, of the forward and of the backward with those before it whose dz it makes
// again: 4 x 2048 tokens of 2048 channels are then some 4000 wavefronts.  16 x 2048 tokens take 56,
// 51 and 58 us forward with 8, 16 and 32, and 142, 100 and 124 backward.
constexpr int kForwardRun = 16, kBackwardSpan = 16;

struct Dims {
    int B, T, D, act;
    long long xb, xt;  // x's strides: batch row, token
    const int* lengths;
};

template <typename T>
__device__ __forceinline__ float activate(float z, int act) {
    return act == RKA_ACT_SILU ? z * sigmoid_of<T>(z) : z;
}
template <typename T>
__device__ __forceinline__ float slope(float z, int act) {
    const float s = sigmoid_of<T>(z);
    return act == RKA_ACT_SILU ? s * (1.f + z * (1.f - s)) : 1.f;
}

// Four channels of a token.
template <typename T>
struct Quad {
    T e[kGroup];
};
// SMALL: there are fewer than four channels, `left`.
template <bool SMALL, typename T>
__device__ __forceinline__ Quad<T> load_quad(const T* p, int left) {
    struct __attribute__((packed, aligned(2))) Bytes {
        unsigned w[sizeof(T)];
    };
    Quad<T> q;
    if constexpr (SMALL) {
#pragma unroll
        for (int e = 0; e < kGroup; ++e) q.e[e] = p[min(e, left - 1)];
    } else {
        const Bytes b = *reinterpret_cast<const Bytes*>(p);
        q = __builtin_bit_cast(Quad<T>, b);
    }
    return q;
}
template <bool SMALL, typename T>
__device__ __forceinline__ void store_quad(T* p, const Quad<T>& q, int left) {
    struct __attribute__((packed, aligned(2))) Bytes {
        unsigned w[sizeof(T)];
    };
    if constexpr (SMALL) {
#pragma unroll
        for (int e = 0; e < kGroup; ++e)
            if (e < left) p[e] = q.e[e];
    } else {
        *reinterpret_cast<Bytes*>(p) = __builtin_bit_cast(Bytes, q);
    }
}

template <bool SMALL, typename T, int W>
struct Weights {
    float w[W][kGroup], b[kGroup];

    __device__ __forceinline__ void load(const T* weight, const T* bias, int d0, int left) {
#pragma unroll
        for (int e = 0; e < kGroup; ++e) {
            const int d = d0 + (SMALL ? min(e, left - 1) : e);
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][e] = to_f32(weight[(long long)d * W + j]);
            b[e] = bias ? to_f32(bias[d]) : 0.f;
        }
    }
    // x: the token's input and the W - 1 before it
    __device__ __forceinline__ float z(const Quad<T>* x, int e) const {
        float sum = b[e];
#pragma unroll
        for (int j = 0; j < W; ++j) sum = fmaf(w[j][e], to_f32(x[j].e[e]), sum);
        return sum;
    }
};

// A thread's channels: the last four again where fewer are left (two threads then make, and
// write, the same).
__device__ __forceinline__ int first_channel(int D) { return min((int)(blockIdx.x * kLanes + threadIdx.x) * kGroup, max(0, D - kGroup)); }
__device__ __forceinline__ bool has_channels(int D) { return (long long)(blockIdx.x * kLanes + threadIdx.x) * kGroup < D; }

// Input t of a row with `len` tokens, those behind the last as the last; before the first, from
// the initial state, and before that 0.
template <bool SMALL, typename T, int W>
__device__ __forceinline__ Quad<T> input(const Dims& d, const T* x, const T* initial, int b, int t, int len, int d0) {
    if (t >= 0 && len > 0) return load_quad<SMALL>(x + b * d.xb + min(t, len - 1) * d.xt + d0, d.D);
    if (t < 0 && t >= -(W - 1) && initial) return load_quad<SMALL>(initial + ((long long)b * (W - 1) + t + W - 1) * d.D + d0, d.D);
    return Quad<T>{};
}

template <bool SMALL, typename T, int W>
__global__ __launch_bounds__(kLanes* kRuns) void forward_kernel(Dims d, const T* x, const T* weight, const T* bias,
                                                                const T* initial, T* y, T* final_state) {
    const int b = blockIdx.z, d0 = first_channel(d.D), run = blockIdx.y * kRuns + __builtin_amdgcn_readfirstlane(threadIdx.y);
    if (!has_channels(d.D) || (long long)run * kForwardRun > d.T) return;
    const int t0 = run * kForwardRun, len = row_length(d.lengths, b, d.T);
    if (run == 0) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
            store_quad<SMALL>(final_state + ((long long)b * (W - 1) + j) * d.D + d0,
                              input<SMALL, T, W>(d, x, initial, b, len - (W - 1) + j, len, d0), d.D);
    }
    if (t0 >= d.T) return;
    Weights<SMALL, T, W> wt;
    wt.load(weight, bias, d0, d.D);
    Quad<T> in[kForwardRun + W - 1];
#pragma unroll
    for (int i = 0; i < kForwardRun + W - 1; ++i) in[i] = input<SMALL, T, W>(d, x, initial, b, t0 - (W - 1) + i, len, d0);
    T* py = y + ((long long)b * d.T + t0) * d.D + d0;
#pragma unroll
    for (int i = 0; i < kForwardRun; ++i, py += d.D) {
        if (t0 + i >= d.T) break;
        Quad<T> out;
#pragma unroll
        for (int e = 0; e < kGroup; ++e) out.e[e] = from_f32<T>(t0 + i < len ? activate<T>(wt.z(in + i, e), d.act) : 0.f);
        store_quad<SMALL>(py, out, d.D);
    }
}

// Run r takes the dz of R = kBackwardSpan - W + 1 tokens of [0, T + W - 1) (those from the
// length on are 0) and the dx that they complete, of the tokens W - 1 before, where tokens before
// 0 are the initial state's.  Sums of dw and db: [batch row][workgroup's runs][W + 1][channels].
template <bool SMALL, typename T, int W>
__global__ __launch_bounds__(kLanes* kRuns) void backward_kernel(Dims d, const T* dy, const T* dstate, const T* x,
                                                                 const T* weight, const T* bias, const T* initial, T* dx,
                                                                 T* dinitial, float* sums) {
    constexpr int R = kBackwardSpan - W + 1;
    __shared__ float part[kRuns - 1][kGroup][kLanes];
    const int b = blockIdx.z, d0 = first_channel(d.D), wave = __builtin_amdgcn_readfirstlane(threadIdx.y);
    const bool on = has_channels(d.D);
    const int len = row_length(d.lengths, b, d.T);
    const long long first = (long long)(blockIdx.y * kRuns + wave) * R;
    float dw[W][kGroup] = {}, db[kGroup] = {};
    if (on && first < (long long)d.T + W - 1) {
        const int t0 = (int)first - (W - 1);  // the first whose dz is made
        Weights<SMALL, T, W> wt;
        wt.load(weight, bias, d0, d.D);
        Quad<T> in[kBackwardSpan + W - 1], up[kBackwardSpan];
#pragma unroll
        for (int i = 0; i < kBackwardSpan + W - 1; ++i) in[i] = input<SMALL, T, W>(d, x, initial, b, t0 - (W - 1) + i, len, d0);
        const bool given = dy && len > 0;
        if (given) {
#pragma unroll
            for (int i = 0; i < kBackwardSpan; ++i)
                up[i] = load_quad<SMALL>(dy + ((long long)b * d.T + max(0, min(t0 + i, len - 1))) * d.D + d0, d.D);
        }
        float dz[kBackwardSpan][kGroup];
#pragma unroll
        for (int i = 0; i < kBackwardSpan; ++i) {
            const int t = t0 + i;
            const bool live = given && t >= 0 && t < len;
#pragma unroll
            for (int e = 0; e < kGroup; ++e) dz[i][e] = live ? to_f32(up[i].e[e]) * slope<T>(wt.z(in + i, e), d.act) : 0.f;
            if (i < W - 1) continue;
            if (live) {
#pragma unroll
                for (int e = 0; e < kGroup; ++e) {
                    db[e] += dz[i][e];
#pragma unroll
                    for (int j = 0; j < W; ++j) dw[j][e] = fmaf(dz[i][e], to_f32(in[i + j].e[e]), dw[j][e]);
                }
            }
            const int s = t - (W - 1);
            T* to = s >= 0 ? dx : dinitial;
            if (!to || s >= d.T) continue;
            float sum[kGroup] = {};
            if (given && s < len) {  // (else it is 0 whatever the weights)
#pragma unroll
                for (int e = 0; e < kGroup; ++e)
#pragma unroll
                    for (int j = 0; j < W; ++j) sum[e] = fmaf(wt.w[j][e], dz[i - j][e], sum[e]);
            }
            const int kept = s - (len - (W - 1));  // its place in the final state
            if (dstate && kept >= 0 && kept < W - 1) {
                const Quad<T> g = load_quad<SMALL>(dstate + ((long long)b * (W - 1) + kept) * d.D + d0, d.D);
#pragma unroll
                for (int e = 0; e < kGroup; ++e) sum[e] += to_f32(g.e[e]);
            }
            Quad<T> out;
#pragma unroll
            for (int e = 0; e < kGroup; ++e) out.e[e] = from_f32<T>(sum[e]);
            to += s >= 0 ? ((long long)b * d.T + s) * d.D : ((long long)b * (W - 1) + s + W - 1) * d.D;
            store_quad<SMALL>(to + d0, out, d.D);
        }
    }
    if (!sums) return;
    float* to = sums + ((long long)b * gridDim.y + blockIdx.y) * (W + 1) * d.D + d0;
#pragma unroll
    for (int j = 0; j <= W; ++j) {
        float* own = j < W ? dw[j < W ? j : 0] : db;
        __syncthreads();
        if (wave > 0) {
#pragma unroll
            for (int e = 0; e < kGroup; ++e) part[wave - 1][e][threadIdx.x] = own[e];
        }
        __syncthreads();
        if (wave == 0 && on) {
#pragma unroll
            for (int e = 0; e < kGroup; ++e) {
                float s = own[e];
#pragma unroll
                for (int k = 0; k < kRuns - 1; ++k) s += part[k][e][threadIdx.x];
                if (!SMALL || e < d.D) to[(long long)j * d.D + e] = s;
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

// (in place, so that no channel has two threads: element by element where the last of them would
// have fewer than four)
template <bool SMALL, typename T, int W>
__global__ __launch_bounds__(kLanes) void step_kernel(int B, int D, int act, const T* x, long long ldx, const T* weight,
                                                      const T* bias, T* state, const int* slots, int num_slots, T* y) {
    const int groups = (D - 1) / (kLanes * kGroup) + 1;
    const int b = blockIdx.x / groups, d0 = (blockIdx.x % groups * kLanes + threadIdx.x) * kGroup, left = D - d0;
    if (left <= 0) return;
    const int slot = slots ? slots[b] : b;
    Quad<T> out;
    T* py = y + (long long)b * D + d0;
    if (slot < 0 || slot >= num_slots) {
        // a request without a state: nothing is read or written but its output
#pragma unroll
        for (int e = 0; e < kGroup; ++e) out.e[e] = from_f32<T>(slot < 0 ? 0.f : __builtin_nanf(""));
        store_quad<SMALL>(py, out, left);
        return;
    }
    T* ps = state + (long long)slot * (W - 1) * D + d0;
    Quad<T> p[W];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) p[j] = load_quad<SMALL>(ps + (long long)j * D, left);
    p[W - 1] = load_quad<SMALL>(x + b * ldx + d0, left);
    Weights<SMALL, T, W> wt;
    wt.load(weight, bias, d0, left);
#pragma unroll
    for (int e = 0; e < kGroup; ++e) out.e[e] = from_f32<T>(activate<T>(wt.z(p, e), act));
    store_quad<SMALL>(py, out, left);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_quad<SMALL>(ps + (long long)j * D, p[j + 1], left);
}

// Calls f with `small` and the width as constants.
template <typename F>
int with_form(bool small, int width, F f) {
    const auto go = [&](auto w) { return small ? f(std::true_type{}, w) : f(std::false_type{}, w); };
    switch (width) {
        case 2: return go(std::integral_constant<int, 2>{});
        case 3: return go(std::integral_constant<int, 3>{});
        case 4: return go(std::integral_constant<int, 4>{});
        case 5: return go(std::integral_constant<int, 5>{});
        case 6: return go(std::integral_constant<int, 6>{});
        case 7: return go(std::integral_constant<int, 7>{});
        default: return go(std::integral_constant<int, 8>{});
    }
}

int blocks_of_runs(long long tokens, int run) { return (int)((std::max(tokens, 1LL) - 1) / ((long long)run * kRuns) + 1); }
dim3 grid(const Dims& d, int run_blocks) {
    return dim3((unsigned)((d.D - 1) / (kLanes * kGroup) + 1), (unsigned)run_blocks, (unsigned)d.B);
}
// (65535 is the most of a grid's second and third size)
int check_sizes(const char* what, const Dims& d, int width, int dtype) {
    const std::string name(what);
    if (d.B < 0 || d.T < 0 || d.D < 1) return fail(RKA_ERR_INVALID_ARGUMENT, name + ": batch and tokens must be >= 0, channels >= 1");
    if (width < 2 || width > kMaxWidth) return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": width must be in [2, 8]");
    if (d.act != RKA_ACT_NONE && d.act != RKA_ACT_SILU) return fail(RKA_ERR_INVALID_ARGUMENT, name + ": activation must be none or silu");
    if (d.B > 65535 || d.T > (1 << 20)) return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": batch exceeds 65535 or tokens 2^20");
    return check_dtype(dtype, what);
}

// Batch rows of a launch, of as many as it may have threads for.
int rows_of(const dim3& blocks) {
    return (int)std::max(1LL, std::min<long long>(blocks.z, ((1LL << 32) - 1) / (kLanes * kRuns) / ((long long)blocks.x * blocks.y)));
}
// `d`, and a tensor of `row` elements to a batch row, from row b on.
Dims rows_from(const Dims& d, int b, int rows) {
    Dims e = d;
    e.B = std::min(rows, d.B - b);
    if (d.lengths) e.lengths = d.lengths + b;
    return e;
}
template <typename T>
T* from(const void* p, long long b, long long row) {
    return p ? static_cast<T*>(const_cast<void*>(p)) + b * row : nullptr;
}

template <typename T>
int forward(const Dims& d, const void* x, const void* weight, const void* bias, const void* initial, void* y,
            void* final_state, int width, hipStream_t s) {
    const int runs = blocks_of_runs(d.T, kForwardRun), rows = rows_of(grid(d, runs));
    const long long all = (long long)d.T * d.D, kept = (long long)(width - 1) * d.D;
    return with_form(d.D < kGroup, width, [&](auto small, auto w) {
        for (int b = 0; b < d.B; b += rows) {
            const Dims e = rows_from(d, b, rows);
            const dim3 blocks = grid(e, runs);
            RKA_RETURN_IF_ERR(check_grid((long long)blocks.x * blocks.y * blocks.z, kLanes * kRuns, "causal_conv_forward"));
            hipLaunchKernelGGL((forward_kernel<decltype(small)::value, T, decltype(w)::value>), blocks, dim3(kLanes, kRuns), 0, s, e,
                               from<T>(x, b, d.xb), from<T>(weight, 0, 0), from<T>(bias, 0, 0), from<T>(initial, b, kept),
                               from<T>(y, b, all), from<T>(final_state, b, kept));
            RKA_RETURN_IF_HIP(hipGetLastError());
        }
        return 0;
    });
}

template <typename T>
int backward(const Dims& d, const void* dy, const void* dstate, const void* x, const void* weight, const void* bias,
             const void* initial, void* dx, void* dweight, void* dbias, void* dinitial, float* sums, int width,
             hipStream_t s) {
    const int runs = blocks_of_runs((long long)d.T + width - 1, kBackwardSpan - width + 1), rows = rows_of(grid(d, runs));
    const long long all = (long long)d.T * d.D, kept = (long long)(width - 1) * d.D, of_sums = (long long)runs * (width + 1) * d.D;
    if (!dweight && !dbias) sums = nullptr;
    RKA_RETURN_IF_ERR(with_form(d.D < kGroup, width, [&](auto small, auto w) {
        for (int b = 0; b < d.B; b += rows) {
            const Dims e = rows_from(d, b, rows);
            const dim3 blocks = grid(e, runs);
            RKA_RETURN_IF_ERR(check_grid((long long)blocks.x * blocks.y * blocks.z, kLanes * kRuns, "causal_conv_backward"));
            hipLaunchKernelGGL((backward_kernel<decltype(small)::value, T, decltype(w)::value>), blocks, dim3(kLanes, kRuns), 0, s, e,
                               from<T>(dy, b, all), from<T>(dstate, b, kept), from<T>(x, b, d.xb), from<T>(weight, 0, 0),
                               from<T>(bias, 0, 0), from<T>(initial, b, kept), from<T>(dx, b, all), from<T>(dinitial, b, kept),
                               from<float>(sums, b, of_sums));
            RKA_RETURN_IF_HIP(hipGetLastError());
        }
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
    const long long blocks = (long long)B * ((D - 1) / (kLanes * kGroup) + 1);
    RKA_RETURN_IF_ERR(check_grid(blocks, kLanes, "causal_conv_step"));
    return with_form(D % kGroup != 0, width, [&](auto small, auto w) {
        hipLaunchKernelGGL((step_kernel<decltype(small)::value, T, decltype(w)::value>), dim3((unsigned)blocks), dim3(kLanes), 0, s, B, D, act,
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
    return (size_t)batch * blocks_of_runs((long long)tokens + width - 1, kBackwardSpan - width + 1) * (width + 1) * channels * sizeof(float);
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
