// What the operators that go through memory once share: element types, 16 bytes of
// elements at any address, sums over lanes, exp and its like.
#pragma once

#include "rka_internal.h"

namespace rka {
namespace elem {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct bf16 {
    unsigned short bits;
};
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __uint_as_float((unsigned)x.bits << 16); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
    return x;
}
// round to nearest even
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) {
    return bf16{__builtin_bit_cast(unsigned short, (__bf16)x)};
}

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);  // elements of 16 bytes

// 16 bytes from or to any element's address (the hardware's loads and stores of four
// dwords ask for no alignment beyond the element's).
struct __attribute__((packed, aligned(2))) Bytes16 {
    unsigned w[4];
};
template <typename T>
union Piece {
    u32x4 u;
    T e[kVec<T>];
};
// The first `left` (kVec or fewer) elements at p; the others are 0.
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* p, int left) {
    Piece<T> q;
    if (left >= kVec<T>) {
        const Bytes16 v = *reinterpret_cast<const Bytes16*>(p);
        q.u = u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
    } else {
        q.u = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < kVec<T>; ++j)
            if (j < left) q.e[j] = p[j];
    }
    return q;
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, const Piece<T>& q, int left) {
    if (left >= kVec<T>) {
        *reinterpret_cast<Bytes16*>(p) = Bytes16{{q.u[0], q.u[1], q.u[2], q.u[3]}};
    } else {
#pragma unroll
        for (int j = 0; j < kVec<T>; ++j)
            if (j < left) p[j] = q.e[j];
    }
}

// Over all 64 lanes, always in the same order.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

constexpr float kLog2e = 1.4426950408889634f;
// exp(x) for results of type T (those under 2^-126 are 0).  The hardware's exponential takes a
// product, whose rounding is worth |x| 2^-24 of the result: nothing beside bf16's last bit.  float32
// puts it back: e^x = 2^hi (1 + (x - ln(2) hi)), unless 2^hi is 0 or infinite, which it then is.  (expf
// and a division cost the float32 scan 8% and the convolution's gradients 17%, this 5% either.)
template <typename T>
__device__ __forceinline__ float exp_of(float x) {
    const float hi = kLog2e * x, e = __builtin_amdgcn_exp2f(hi);
    if constexpr (sizeof(T) == 2) {
        return e;
    } else {
        // (ln(2) in two parts)
        const float rest = fmaf(hi, 1.9046542e-9f, fmaf(hi, -0.6931471824645996f, x));
        return fabsf(hi) < 128.f ? fmaf(e, rest, e) : e;
    }
}
// 1 / (1 + exp(-z)), in float32 with a step of Newton's for the reciprocal's last bit.
template <typename T>
__device__ __forceinline__ float sigmoid_of(float z) {
    const float w = 1.f + exp_of<T>(-z), r = __builtin_amdgcn_rcpf(w);
    if constexpr (sizeof(T) == 2)
        return r;
    else
        return fmaf(fminf(fmaf(-w, r, 1.f), 1.f), r, r);  // (w infinite: r is 0)
}

__device__ __forceinline__ int row_length(const int* lengths, int b, int tokens) {
    return lengths ? max(0, min(tokens, lengths[b])) : tokens;
}

// A launch has fewer than 2^32 threads.
inline int check_grid(long long blocks, int threads, const char* what) {
    if (blocks * threads >= (1LL << 32))
        return fail(RKA_ERR_UNSUPPORTED_SHAPE, std::string(what) + ": more workgroups than a launch may have");
    return 0;
}
inline int check_dtype(int dtype, const char* what) {
    if (dtype != RKA_DTYPE_F32 && dtype != RKA_DTYPE_BF16)
        return fail(RKA_ERR_INVALID_ARGUMENT, std::string(what) + ": dtype must be RKA_DTYPE_F32 or RKA_DTYPE_BF16");
    return 0;
}
inline int check_workspace(const void* workspace, size_t bytes, size_t need, const char* what) {
    if (bytes < need || (need > 0 && !workspace))
        return fail(RKA_ERR_WORKSPACE_TOO_SMALL, std::string(what) + ": workspace needs " + std::to_string(need) +
                                                     " bytes, got " + std::to_string(bytes));
    if (need > 0 && reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(RKA_ERR_INVALID_ARGUMENT, std::string(what) + ": the workspace must begin at a multiple of 16 bytes");
    return 0;
}

}  // namespace elem
}  // namespace rka
