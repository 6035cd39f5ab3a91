// Declarations shared by the gated delta rule's translation units
// (gated_delta.hip: entry points, per-chunk products and gradients;
// gated_delta_chain.hip: the chains over chunks; gated_delta_step.hip: one token).
//
// Per batch row and value head, with S [Dk, Dv] in float32:
//   S~ = exp(g_t) S_{t-1};  e_t = v_t - S~^T k_t;  S_t = S~ + k_t (beta_t e_t)^T;
//   o_t = scale S_t^T q_t.
//
// Over a chunk of C = 64 tokens that starts from the state S, with G the running
// sum of g in the chunk, L_ij = exp(G_i - G_j) for i >= j, and K, Q, V, E the
// tokens' rows:
//   N = strictly lower part of (K K^T * L),   T = (I + N diag(beta))^-1
//   E = T (V - diag(exp G) K S)
//   O = scale diag(exp G) Q S + P E,          P = lower part of scale (Q K^T * L) diag(beta)
//   S' = exp(G_C) S + K^T diag(exp(G_C - G) beta) E
// T and P hang on no state, so they are made for all chunks at once ("prepare");
// only E, O and S' go from chunk to chunk ("chain").  Columns of S, V, E and O do
// not mix, so a wavefront takes 16 of them through all chunks on its own.
//
// With dS' the gradient of S' and dO that of O:
//   B dU = P^T dO + diag(exp(G_C - G) beta) K dS'          (B = diag(beta))
//   dX = T^T (B dU)                                        (= dV)
//   dS = exp(G_C) dS' + scale Q^T diag(exp G) dO - K^T diag(exp G) dX
// goes through the chunks backwards; the rest of the gradients is again made for
// all chunks at once, from S, dS', E and dX of each:
//   F1 = scale dO E^T * L,  F2 = -(dX E^T * L) strictly lower,  W = diag(exp(G_C - G)) E dS'^T
//   dQ = scale diag(exp G) dO S^T + F1 B K
//   Z  = W + F1^T Q + F2^T K;  dK (as a written key) = B Z;  dbeta_j = k_j . Z_j
//   dK (as a read key) = -diag(exp G) dX S^T + F2 B K
//   dG_i = q_i . dq_i + k_i . dk_i(read) - beta_i dbeta_i, and for the chunk's last
//   token also sum_j beta_j k_j . W_j + exp(G_C) <S, dS'>;  dg = dG summed from the end.
// beta is never divided by: it may be zero.
#pragma once

#include "rka_internal.h"

namespace rka {
namespace delta {

constexpr int kChunk = 64;
constexpr int kMaxKeyDim = 256;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Element types of q, k, v, o and their gradients.
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
    const __bf16 y = (__bf16)x;
    return bf16{__builtin_bit_cast(unsigned short, y)};
}

// A call's sizes and where its tensors lie (strides in elements: batch row,
// token, head; the head's elements are contiguous).
struct Dims {
    int B, T, Hk, Hv, Dk, Dv;
    int chunks;  // of T
    float scale;
    int normalize;  // q and k are divided by sqrt(|.|^2 + kNormEps)
    int gate_bf16;  // g and beta are bf16 (else float32)
    long long q_s[3], k_s[3], v_s[3], g_s[3], b_s[3];
};
constexpr float kNormEps = 1e-6f;

__device__ __forceinline__ float load_gate(const void* p, long long i, int is_bf16) {
    return is_bf16 ? to_f32(static_cast<const bf16*>(p)[i]) : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_gate(void* p, long long i, float v, int is_bf16) {
    if (is_bf16)
        static_cast<bf16*>(p)[i] = from_f32<bf16>(v);
    else
        static_cast<float*>(p)[i] = v;
}

// A decay below exp(-200) is zero in float32 however it is summed, and a finite
// floor keeps exp(G_i - G_j) free of inf - inf where a gate closes fully (g = -inf).
// NaN stays NaN.
__device__ __forceinline__ float floor_gate(float g) { return g < -200.f ? -200.f : g; }

__device__ __forceinline__ int row_length(const int* lengths, int b, int T) {
    return lengths ? max(0, min(T, lengths[b])) : T;
}

// Per chunk and head, made by `prepare` (a chunk past the row's length has none):
// kCoefs rows of 64 floats, then exp(G_C).
enum Coef { RK = 0, WK, RQ, BETA, CK, CQ, NCOEF };
//   RK: exp(G) ck;  WK: exp(G_C - G) ck beta;  RQ: scale exp(G) cq;  CK, CQ: what
//   normalises k and q (1 if nothing does)
constexpr int kCoefFloats = NCOEF * kChunk + 4;
// T and P as 16x16 blocks of the lower triangle, block (i, j) at i (i + 1) / 2 + j,
// each 256 floats in the order that a matrix instruction's operand takes them.
constexpr int kBlocks = 10;
constexpr int kTriFloats = kBlocks * 256;

struct ChunkData {
    float* coef;  // [chunk-head][kCoefFloats]
    float* t;     // [chunk-head][kTriFloats]
    float* p;
};

// Gradients' inputs and outputs that pass between the backward's launches.
struct BackwardData {
    const float* states;  // [chunk-head][Dk][Dv]: S of each chunk
    const float* e;       // [B][T][Hv][Dv]
    float* dstates;       // [chunk-head][Dk][Dv]: dS' of each chunk
    float* dx;            // [B][T][Hv][Dv]
    float* dq;            // [B][T][Hv][Dk]: of each value head
    float* dk;
};

// The launches below take lengths == nullptr for rows of T tokens each.
// Forward operands (transpose false) or the backward's transposed ones (true).
template <typename T>
int launch_prepare(const Dims& d, const T* q, const T* k, const void* g, const void* beta, const int* lengths,
                   const ChunkData& out, bool transpose, hipStream_t stream);
// states, e: saved for the backward, or both null.
template <typename T>
int launch_chain_forward(const Dims& d, const T* q, const T* k, const T* v, const float* s0, const int* lengths,
                         const ChunkData& in, T* o, float* state_out, float* states, float* e, hipStream_t stream);
// dstate_out (of the final state), dO: either may be null (zeros).
template <typename T>
int launch_chain_backward(const Dims& d, const T* q, const T* k, const T* dout, const float* dstate_out,
                          const int* lengths, const ChunkData& in, T* dv, float* ds0, const BackwardData& bd,
                          hipStream_t stream);

// A call's sizes and its other arguments, checked (the errors of the C entries).
int make_dims(const char* what, int B, int T, int Hk, int Hv, int Dk, int Dv, Dims* d);
int set_call(const char* what, Dims* d, int dtype, int gate_dtype, int normalize, double scale,
             const long long* strides);
// Blocks of a launch, checked against the grid's limit of 2^32 threads.
int check_grid(long long blocks, int threads, const char* what);

}  // namespace delta
}  // namespace rka
