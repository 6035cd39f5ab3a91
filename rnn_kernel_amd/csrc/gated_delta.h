// Declarations shared by the gated delta rule's translation units: gated_delta.hip
// (entry points, what is made for all chunks at once before the chains),
// gated_delta_chain.h (the chains over chunks), gated_delta_grad.hip (the gradients
// made for all chunks at once after the backward's chain), gated_delta_step.hip (one
// token).
//
// Per batch row and value head, with S [Dk, Dv] in float32:
//   S~ = exp(g_t) S_{t-1};  e_t = v_t - S~^T k_t;  S_t = S~ + k_t (beta_t e_t)^T;
//   o_t = scale S_t^T q_t.
//
// Over a chunk of C = 64 tokens that starts from the state S, with G the running
// sum of g in the chunk, L_ij = exp(G_i - G_j) for i >= j, and K, Q, V, E the
// tokens' rows:
//   N = strictly lower part of (K K^T * L),   T = (I + N diag(beta))^-1
//   E = T (V - diag(exp G) K S) = T V - (T diag(exp G) K) S
//   O = scale diag(exp G) Q S + P E,          P = lower part of scale (Q K^T * L) diag(beta)
//   S' = exp(G_C) S + K^T diag(exp(G_C - G) beta) E
// T V, T diag(exp G) K and P hang on no state, so they are made for all chunks at once
// ("prepare"); E, O and S' go from chunk to chunk ("chain"): two products that wait for
// one another.  Columns of S, V, E and O do not mix.
//
// With dS' the gradient of S' and dO that of O (B = diag(beta)):
//   B dU = P^T dO + diag(exp(G_C - G) beta) K dS'
//   dX = T^T (B dU) = (P T)^T dO + (T^T diag(exp(G_C - G) beta) K) dS'       (= dV)
//   dS = exp(G_C) dS' + scale Q^T diag(exp G) dO - K^T diag(exp G) dX
// goes through the chunks backwards, again with the factors of dO and dS' made before;
// the rest of the gradients is made for all chunks at once, from S, dS', E and dX of
// each:
//   F1 = scale dO E^T * L,  F2 = -(dX E^T * L) strictly lower,  W = diag(exp(G_C - G)) E dS'^T
//   dQ = scale diag(exp G) dO S^T + F1 B K
//   Z  = W + F1^T Q + F2^T K;  dK (as a written key) = B Z;  dbeta_j = k_j . Z_j
//   dK (as a read key) = -diag(exp G) dX S^T + F2 B K
//   dG_i = q_i . dq_i + k_i . dk_i(read) - beta_i dbeta_i, and for the chunk's last
//   token also sum_j beta_j k_j . W_j + exp(G_C) <S, dS'>;  dg = dG summed from the end.
// beta is never divided by: it may be zero.
//
// All products run on the bf16 matrix cores.  A float32 is the sum of three bf16 values
// (24 bits in three rounded pieces of 8), a bf16 is one; of the products of pieces
// those up to 2^-16 of the largest are taken, smallest first, each exact and summed in
// float32: three where one operand is bf16, six where neither is.  The error is that
// of a float32 product (lower pieces of numbers under some 2^-110 are lost; a number past
// bf16's largest, 3.39e38, has no first piece and becomes NaN, as an infinity does).  What
// only reaches a bf16 o is taken in two pieces of S, E and P: 16 bits, of which o keeps 8.
// One 16x16x32 bf16 instruction takes 16 clocks, the eight 16x16x4 float32 ones for the
// same block 256.
#pragma once

#include "rka_internal.h"

namespace rka {
namespace delta {

constexpr int kChunk = 64;
constexpr int kMaxKeyDim = 256;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

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
// bf16 pieces of a value of type T
template <typename T>
constexpr int kPieces = sizeof(T) == 4 ? 3 : 1;

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

__device__ __forceinline__ int row_length(const int* lengths, int b, int T) {
    return lengths ? max(0, min(T, lengths[b])) : T;
}

// ------------------------------------------------- pieces and products ---
// Four values as N pieces of four bf16 each.
template <int N>
__device__ __forceinline__ void split(f32x4 x, u32x2 (&p)[N]) {
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bf16x2 v = {(__bf16)x[2 * h], (__bf16)x[2 * h + 1]};
            p[c][h] = __builtin_bit_cast(unsigned, v);
            if (c + 1 < N) {
                x[2 * h] -= __uint_as_float(p[c][h] << 16);
                x[2 * h + 1] -= __uint_as_float(p[c][h] & 0xffff0000u);
            }
        }
}
// Eight values as N fragments of a lane.
template <int N>
__device__ __forceinline__ void split8(f32x4 lo, f32x4 hi, u32x4 (&p)[N]) {
    u32x2 a[N], b[N];
    split<N>(lo, a);
    split<N>(hi, b);
#pragma unroll
    for (int c = 0; c < N; ++c) p[c] = u32x4{a[c][0], a[c][1], b[c][0], b[c][1]};
}

// c += A B for a 16x16x32 block in NA and NB pieces.  Lane l holds row (A) or column
// (B) l % 16 at the sum's indices 8 (l / 16) .. + 7; of the result column l % 16, rows 4
// (l / 16) .. + 3.
template <int NA, int NB>
__device__ __forceinline__ f32x4 mul(const u32x4 (&a)[NA], const u32x4 (&b)[NB], f32x4 c) {
    constexpr int most = (NA < NB ? NB : NA) - 1;
#pragma unroll
    for (int s = most; s >= 0; --s)
#pragma unroll
        for (int i = NA - 1; i >= 0; --i) {
            const int j = s - i;
            if (j < 0 || j >= NB) continue;
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[i]), __builtin_bit_cast(bf16x8, b[j]),
                                                        c, 0, 0, 0);
        }
    return c;
}

// Waits until the last product of a sum is in its registers.  Between a matrix
// instruction and the reader of its result the compiler (clang 22 of ROCm 7.2) counts the
// wait states on most paths, but has missed some that pass a branch: there the reader
// came after one state instead of eight and saw the old value now and then.  So every sum
// that is read in another basic block than its last product's ends with this.
__device__ __forceinline__ void settle(f32x4& c) { asm volatile("s_nop 9" : "+v"(c)); }
// The same, right behind the product, for sums that may be in accumulation registers: an
// operand of it would be copied out of them before the wait, and behind a branch they may
// have been copied already.
__device__ __forceinline__ void settle_all() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 9" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// A value that is made whether or not it is used: without this the compiler puts loads
// and exponentials whose result is then selected away under branches, one each.
__device__ __forceinline__ float made(float x) {
    asm volatile("" : "+v"(x));
    return x;
}

// --------------------------------------------------------------- loads ---
struct __attribute__((packed, aligned(4))) Float4U {
    float x, y, z, w;
};
struct __attribute__((packed, aligned(2))) Bytes16 {
    unsigned w[4];
};

// Loads of neighbouring columns, from column c of a row of `width` in memory, without
// branches (clamped addresses).  For the widths that are multiples of eight (VEC) in
// 16-byte loads, and as they come: what lies past the width is made zero where it is
// used, since a select beside the load would wait for it.
template <bool VEC>
__device__ __forceinline__ f32x4 load4(const float* row, int c, int width) {
    f32x4 x;
    if constexpr (VEC) {
        const Float4U v = *reinterpret_cast<const Float4U*>(row + min(c, width - 4));
        x = f32x4{v.x, v.y, v.z, v.w};
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float v = row[min(c + j, width - 1)];
            x[j] = c + j < width ? v : 0.f;
        }
    }
    return x;
}

// Eight columns of a row: a lane's part of an operand, as loaded, in pieces, or put
// where rows are kept (zero where the row is not `on`, or past the width).
template <typename T>
struct Eight;
template <>
struct Eight<float> {
    f32x4 a, b;
    bool in;
    template <bool VEC>
    __device__ __forceinline__ void load(const float* row, int c, int width) {
        in = c < width;
        a = load4<VEC>(row, c, width);
        b = load4<VEC>(row, c + 4, width);
    }
    __device__ __forceinline__ void pieces(bool on, u32x4 (&p)[3]) {
        if (!on || !in) a = b = f32x4{0.f, 0.f, 0.f, 0.f};
        split8<3>(a, b, p);
    }
    __device__ __forceinline__ void store(bool on, float* to) const {
        const f32x4 none{0.f, 0.f, 0.f, 0.f};
        *reinterpret_cast<f32x4*>(to) = on && in ? a : none;
        *reinterpret_cast<f32x4*>(to + 4) = on && in ? b : none;
    }
};
template <>
struct Eight<bf16> {
    u32x4 x;
    bool in;
    template <bool VEC>
    __device__ __forceinline__ void load(const bf16* row, int c, int width) {
        in = c < width;
        if constexpr (VEC) {
            const Bytes16 v = *reinterpret_cast<const Bytes16*>(row + min(c, width - 8));
            x = u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
        } else {
            x = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const unsigned v = row[min(c + j, width - 1)].bits;
                x[j / 2] |= (c + j < width ? v : 0u) << (j % 2 * 16);
            }
        }
    }
    __device__ __forceinline__ void pieces(bool on, u32x4 (&p)[1]) { p[0] = on && in ? x : u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void store(bool on, bf16* to) const {
        *reinterpret_cast<u32x4*>(to) = on && in ? x : u32x4{0, 0, 0, 0};
    }
};

// ------------------------------------------------------- chunk operands ---
// A "fragment" is what one matrix instruction takes of an operand: 64 lanes x 16 bytes.
constexpr int kFragLanes = 64;

// 32-wide steps over Dk.
inline __host__ __device__ int key_steps(int Dk) { return (Dk + 31) / 32; }
// The steps that the chains' instances are made for: 2, 4, 6 or 8.
inline __host__ __device__ int chain_steps(int Dk) { return (Dk + 63) / 64 * 2; }

// Of a chunk's q or k, per key head, in kPieces<T> pieces: rows for the products over
// Dk, [16-token block][step][piece], and transposed for those over tokens,
// [16-wide block of Dk][32-token step][piece].  Each 4 steps (8 blocks x 2) fragments.
template <typename T>
inline __host__ __device__ size_t row_frags(int Dk) {
    return (size_t)4 * chain_steps(Dk) * kPieces<T>;
}

// The fragments of a lower triangular 64x64 matrix (or, transposed, of an upper one)
// that are not all zero, of 16 rows x 32 of the sum: six.
//   lower: rows 0, 1: step 0; rows 2, 3: steps 0, 1.   (i, w) at i + w * 2 (w = 1: i >= 2)
//   upper: rows 0, 1: steps 0, 1; rows 2, 3: step 1.
constexpr int kTriFrags = 6;
inline __host__ __device__ constexpr int lower_frag(int i, int w) { return w == 0 ? i : i + 2; }
inline __host__ __device__ constexpr int upper_frag(int i, int w) { return w == 0 ? i : i + 2; }

// Per chunk and value head (a chunk past the row's length has none): rows of 64
// floats, then exp(G_C).
//   RK: exp(G) ck;  WK: exp(G_C - G) ck beta;  RQ: scale exp(G) cq;  CK, CQ: what
//   normalises k and q (1 if nothing does)
enum Coef { RK = 0, WK, RQ, BETA, CK, CQ, NCOEF };
constexpr int kCoefFloats = NCOEF * kChunk + 4;

struct ChunkData {
    float* coef;      // [value chunk-head][kCoefFloats]
    float* norm;      // [key chunk-head][2][64]: CK, CQ
    u32x4 *k, *q;     // [key chunk-head] row fragments
    u32x4 *kt, *qt;   // [key chunk-head] transposed (qt: backward only)
    u32x4* read;      // [value chunk-head][16-token block][step][3]: T diag(exp G) K, or (backward)
                      // T^T diag(exp(G_C - G) beta) K
    u32x4* p;         // [value chunk-head][kTriFrags][3]: P (forward only)
    f32x4* own;       // [value chunk-head][16-column block][16-token block][lane], as a product leaves it: T V, or
                      // (backward) (P T)^T dO
};
inline __host__ __device__ size_t read_frags(int Dk) { return (size_t)4 * chain_steps(Dk) * 3; }
inline __host__ __device__ int column_blocks(int Dv) { return (Dv + 15) / 16; }

// Where a 16x16 result block goes among the fragments over its rows: block x of 16
// rows, lane (hi, n): eight bytes of step x / 2 at lane (2 (x % 2) + hi / 2, n).
__device__ __forceinline__ void put_block(u32x4* frags, int pieces, int x, int hi, int n, const u32x2* p) {
    u32x2* at = reinterpret_cast<u32x2*>(frags + (size_t)(x / 2) * pieces * kFragLanes) +
                ((2 * (x % 2) + hi / 2) * 16 + n) * 2 + hi % 2;
    for (int c = 0; c < pieces; ++c) at[c * kFragLanes * 2] = p[c];
}

// Gradients' inputs and outputs that pass between the backward's launches.
struct BackwardData {
    const float* states;  // [chunk-head][Dk][Dv]: S of each chunk
    const float* e;       // [B][T][Hv][Dv]
    float* dstates;       // [chunk-head][Dk][Dv]: dS' of each chunk
    float* dx;            // [B][T][Hv][Dv]
};

// Blocks of 16 columns that a chain's workgroup takes, one or two.  Two halve what is read
// of K, Q, T and P per column, one has the shorter chain: two where one to a workgroup would
// not have a CU for each.  Measured, the whole forward in us with one and two (bf16,
// 128x128): 256 workgroups of one (2048 tokens) 107 and 122, 320 160 and 138, 512 262 and
// 226, 1024 (1024 tokens) 307 and 229; 128 (16384 tokens) 733 and 847.  float32 (512
// tokens): 256 57 and 61, 320 81 and 68, 512 91 and 80.  (Float32 operands of the largest
// Dk leave no registers for two.)
inline int chain_columns(const Dims& d, int pieces) {
    constexpr int kCus = 256;
    if (pieces > 1 && chain_steps(d.Dk) == 8) return 1;
    return d.Dv > 16 && (long long)d.B * d.Hv * column_blocks(d.Dv) > kCus ? 2 : 1;
}
// A chain's workgroups with that many blocks each (grid: 8 x heads per XCD x blocks).
inline long long chain_blocks(const Dims& d, int columns) {
    return (((long long)d.B * d.Hv + 7) / 8) * 8 * ((d.Dv - 1) / (16 * columns) + 1);
}

// The launches below take lengths == nullptr for rows of T tokens each.
// states, e: saved for the backward, or both null.
template <typename T>
int launch_chain_forward(const Dims& d, const float* s0, const int* lengths, const ChunkData& in, T* o, float* state_out,
                         float* states, float* e, hipStream_t stream);
// dstate_out (of the final state), dO: either may be null (zeros).
template <typename T>
int launch_chain_backward(const Dims& d, const T* dout, const float* dstate_out, const int* lengths, const ChunkData& in,
                          T* dv, float* ds0, const BackwardData& bd, hipStream_t stream);
// dq, dk, dg, dbeta after the chain.
template <typename T>
int launch_gradients(const Dims& d, const T* q, const T* k, const T* dout, const void* g, const int* lengths,
                     const ChunkData& in, const BackwardData& bd, T* dq, T* dk, void* dg, void* dbeta,
                     hipStream_t stream);

// A call's sizes and its other arguments, checked (the errors of the C entries).
int make_dims(const char* what, int B, int T, int Hk, int Hv, int Dk, int Dv, Dims* d);
int set_call(const char* what, Dims* d, int dtype, int gate_dtype, int normalize, double scale,
             const long long* strides);
// Blocks of a launch, checked against the grid's limit of 2^32 threads.
int check_grid(long long blocks, int threads, const char* what);

}  // namespace delta
}  // namespace rka
