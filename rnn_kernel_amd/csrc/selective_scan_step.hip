// The selective scan for one token of each of many requests (selective_scan.h has the
// formulas): every state is read and written once, in place.
//
// A lane takes four states of a channel (16 bytes), as many neighbouring lanes as they need a
// channel's; their sum over the states passes through those lanes.  Bound by memory: 256 requests
// of 4096 channels with 16 states take 31 us, 4.5 TB/s (a copy of 4 GiB 4.8), 62 with states that
// are not on 16 bytes; one request of 256 channels 3 us.
#include "selective_scan.h"

namespace rka {
namespace scan {
namespace {

constexpr int kThreads = 256;

// LANES to a channel.  VEC: its states are aligned float4.
template <typename T, int LANES, bool VEC>
__global__ __launch_bounds__(kThreads) void step_kernel(Dims d, float* state, const int* slots, int num_slots, T* y) {
    constexpr int kChannels = kThreads / LANES;
    const int blocks = (d.D - 1) / kChannels + 1;
    const int b = blockIdx.x / blocks, in = blockIdx.x % blocks * kChannels + threadIdx.x / LANES, n0 = threadIdx.x % LANES * 4;
    const int ch = min(in, d.D - 1), g = ch / (d.D / d.G);
    const int slot = slots ? slots[b] : b;
    if (slot < 0 || slot >= num_slots) {
        // a request without a state: nothing is read or written but its output
        if (n0 == 0 && in < d.D) y[(size_t)b * d.D + ch] = from_f32<T>(slot < 0 ? 0.f : __builtin_nanf(""));
        return;
    }
    float* p = state + ((size_t)slot * d.D + ch) * d.N;
    const float* pa = d.A + (size_t)ch * d.N;
    const T* pb = static_cast<const T*>(d.Bm) + b * d.bs[0] + g * d.bs[2];
    const T* pc = static_cast<const T*>(d.C) + b * d.cs[0] + g * d.cs[2];
    f32x4 h, a;
    T bv[4], cv[4];
    // Everything is loaded at once, from clamped addresses: a load under a branch would be
    // waited for there.
    if constexpr (VEC) {
        const int at = min(n0, d.N - 4);
        h = *reinterpret_cast<const f32x4*>(p + at);
        a = *reinterpret_cast<const f32x4*>(pa + at);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = p[min(n0 + j, d.N - 1)];
            a[j] = pa[min(n0 + j, d.N - 1)];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        bv[j] = pb[min(n0 + j, d.N - 1)];
        cv[j] = pc[min(n0 + j, d.N - 1)];
    }
    const float x = to_f32(static_cast<const T*>(d.x)[b * d.xs[0] + ch]);
    const float gate = d.gate ? to_f32(static_cast<const T*>(d.gate)[b * d.zs[0] + ch]) : 0.f;
    float slope, s = to_f32(static_cast<const T*>(d.dt)[b * d.ts[0] + ch]) + (d.bias ? d.bias[ch] : 0.f);
    const float skip = d.skip ? d.skip[ch] : 0.f;
    if (d.softplus) s = softplus<T>(s, &slope);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h[j] = fmaf(__builtin_amdgcn_exp2f(s * finite_rate(a[j])), h[j], s * x * to_f32(bv[j]));
        if (n0 + j < d.N) sum = fmaf(to_f32(cv[j]), h[j], sum);
    }
#pragma unroll
    for (int o = 1; o < LANES; o *= 2) sum += __shfl_xor(sum, o);
    if (in >= d.D) return;
    if (n0 == 0) {
        float v = fmaf(skip, x, sum);
        if (d.gate) v *= gate * sigmoid_of<T>(gate);
        y[(size_t)b * d.D + ch] = from_f32<T>(v);
    }
    if constexpr (VEC) {
        if (n0 < d.N) *reinterpret_cast<f32x4*>(p + n0) = h;
    } else {
        store_states_of(p, n0, d.N, h);
    }
}

template <typename T>
int step(const Dims& d, float* state, const int* slots, int num_slots, void* y, hipStream_t s) {
    const bool vec = d.N % 4 == 0 && ((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(d.A)) & 15u) == 0;
    auto go = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        const long long blocks = (long long)d.B * ((d.D - 1) / (kThreads / L) + 1);
        RKA_RETURN_IF_ERR(check_grid(blocks, kThreads, "selective_step"));
        if (vec)
            hipLaunchKernelGGL((step_kernel<T, L, true>), dim3((unsigned)blocks), dim3(kThreads), 0, s, d, state, slots, num_slots,
                               static_cast<T*>(y));
        else
            hipLaunchKernelGGL((step_kernel<T, L, false>), dim3((unsigned)blocks), dim3(kThreads), 0, s, d, state, slots, num_slots,
                               static_cast<T*>(y));
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    };
    if (d.N <= 4) return go(std::integral_constant<int, 1>{});
    if (d.N <= 8) return go(std::integral_constant<int, 2>{});
    if (d.N <= 16) return go(std::integral_constant<int, 4>{});
    if (d.N <= 32) return go(std::integral_constant<int, 8>{});
    return go(std::integral_constant<int, 16>{});
}

}  // namespace
}  // namespace scan
}  // namespace rka

using namespace rka;
using namespace rka::scan;

extern "C" int rka_selective_step(const void* x, const void* dt, const float* A, const void* B, const void* C, const float* skip,
                                  const void* gate, const float* dt_bias, float* state, const int* slots, int num_slots, void* y,
                                  int batch, int channels, int states, int groups, const long long* strides, int softplus,
                                  int dtype, void* stream) {
    clear_error();
    Dims d;
    RKA_RETURN_IF_ERR(make_dims("selective_step", batch, 1, channels, states, groups, &d));
    RKA_RETURN_IF_ERR(set_call("selective_step", &d, x, dt, A, B, C, skip, gate, dt_bias, nullptr, strides, softplus, dtype));
    if (num_slots < 0 || (!slots && num_slots < batch))
        return fail(RKA_ERR_INVALID_ARGUMENT, "selective_step: fewer states than requests");
    if (batch == 0) return 0;
    if (!state || !y) return fail(RKA_ERR_INVALID_ARGUMENT, "selective_step: null tensor pointer");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return dtype == RKA_DTYPE_F32 ? step<float>(d, state, slots, num_slots, y, s) : step<bf16>(d, state, slots, num_slots, y, s);
}
