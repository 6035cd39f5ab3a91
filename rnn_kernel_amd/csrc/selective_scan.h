// The selective scan: a recurrence of N numbers per channel whose decay and input are made
// of the token.  Per batch row, channel d (of group g) and state n, with the step size
// s = softplus(dt + bias) or dt + bias:
//
//   h_t = exp(s A[d, n]) h_{t-1} + s x_t B_t[g, n]
//   y_t = (sum_n C_t[g, n] h_t + skip[d] x_t) silu(gate_t)
//
// and, with r_t = dy_t silu(gate_t) and H_t the gradient of h_t,
//
//   H_t = C_t r_t + a_{t+1} H_{t+1},  a_t = exp(s_t A)
//   dC_t = sum_d r_t h_t;  dB_t = sum_d s x_t H_t;  q_t = sum_n H_t B_t
//   dx_t = s q_t + skip r_t;  ds_t = x_t q_t + sum_n H_t a_t h_{t-1} A;  dA = sum_t H_t a_t h_{t-1} s
//   dskip = sum_t r_t x_t;  dgate_t = dy_t (sum_n C h + skip x) silu'(gate_t)
//
// Tokens are split over chunks that run at once.  A chunk's state from nothing and the sum of
// its s (its decay is exp(A sum s)) come first, then the states at the chunks' starts one
// after another, then the chunks themselves; the gradients the same backwards.  With enough
// channels there is one chunk and only the last of the three.
//
// A wavefront takes 16 channels through tiles of 16 tokens: lane l has channel l % 16 and of
// every 16 states the four from 4 (l / 16) on.  What a tile needs of its tokens is loaded and
// made by all lanes at once, a lane four tokens of its channel, and handed round through LDS.
// A token's sums over n are added up between the four lanes of a channel for four tokens at a
// time, by exchanges of half of the lanes after which each lane holds one token's: 2.5
// instructions a token, and the tile's sums end where its x and gate are.
#pragma once

#include "elementwise.h"

namespace rka {
namespace scan {

using namespace elem;

constexpr int kTile = 16;       // tokens of a tile, channels of a wavefront's block, states of a block
constexpr int kMaxStates = 64;  // N
constexpr int kWaves = 4, kChannels = 16 * kWaves;  // of a workgroup of the gradients
constexpr long long kMaxStride = 1 << 21;  // of a token, in elements: a tile's offsets are 32-bit

struct Dims {
    int B, T, D, N, G;
    int softplus;
    int chunk, chunks;  // tokens of a chunk, a multiple of kTile; chunks of T, at least one
    const int* lengths;
    const float *A, *skip, *bias;
    const void *x, *dt, *gate, *Bm, *C;
    long long xs[2], ts[2], zs[2], bs[3], cs[3];  // element strides: batch row, token (, group)
};

inline int tiles_of(int tokens) { return tokens <= 0 ? 1 : (tokens - 1) / kTile + 1; }
inline int state_blocks(int n) { return n <= 16 ? 1 : n <= 32 ? 2 : 4; }
// Blocks of `width` channels, each within a group.
inline long long channel_blocks(const Dims& d, int width) { return (long long)d.G * ((d.D / d.G - 1) / width + 1); }

// Workgroups of the same tokens follow one another on one XCD (consecutive workgroups go to
// the eight in turn): neighbouring channels share lines of memory, all channels of a group B
// and C.
__device__ __forceinline__ long long in_order() {
    const unsigned total = gridDim.x, per = total / 8, rest = total % 8, xcd = blockIdx.x % 8, i = blockIdx.x / 8;
    return (long long)xcd * per + min(xcd, rest) + i;
}

// log(1 + exp(r)) as max(r, 0) + log(1 + u), u = exp(-|r|).  1 + u is rounded; what it lost,
// (u - (w - 1)) / w, is added to log(w), without the division, as it matters where w is next to
// 1: small steps keep their 24 bits.  slope: its derivative.
template <typename T>
__device__ __forceinline__ float softplus(float r, float* slope) {
    const float u = exp_of<T>(-fabsf(r)), w = 1.f + u;
    *slope = (r < 0.f ? u : 1.f) * __builtin_amdgcn_rcpf(w);
    // (NaN stays)
    return (r < 0.f ? 0.f : r) + fmaf(__builtin_amdgcn_logf(w), 0.6931471805599453f, u - (w - 1.f));
}

// Offsets in bytes of the values of a tile that a lane holds: tokens 4 (lane / 16) + r of one
// column, rows from `rows` on as the last.  (Strides are at most kMaxStride elements: they fit.)
struct Offsets {
    unsigned at[4];
    __device__ __forceinline__ void set(long long stride, int column, int rows, int esize) {
        const int first = threadIdx.x % 64 / 16 * 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) at[r] = ((unsigned)min(first + r, rows - 1) * (unsigned)stride + (unsigned)column) * (unsigned)esize;
    }
};
// Memory from an address that is the same for all lanes on, which a lane addresses by 32 bits:
// with pointers the compiler keeps a 64-bit address of each load's from tile to tile.
struct Memory {
    __amdgpu_buffer_rsrc_t of;
    __device__ __forceinline__ explicit Memory(const void* p)
        : of(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)0xffffffffu, 0x27000)) {}
    __device__ __forceinline__ void load(float* v, unsigned at) const {
        *v = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(of, (int)at, 0, 0));
    }
    __device__ __forceinline__ void load(bf16* v, unsigned at) const { v->bits = __builtin_amdgcn_raw_buffer_load_b16(of, (int)at, 0, 0); }
    __device__ __forceinline__ void store(float v, unsigned at) const {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), of, (int)at, 0, 0);
    }
    __device__ __forceinline__ void store(bf16 v, unsigned at) const { __builtin_amdgcn_raw_buffer_store_b16(v.bits, of, (int)at, 0, 0); }
};
// The values themselves; `p` is the tile's first token's row.
template <typename T>
struct Rows {
    T v[4];
    __device__ __forceinline__ void load(const T* p, const Offsets& o) {
        const Memory m(p);
#pragma unroll
        for (int r = 0; r < 4; ++r) m.load(&v[r], o.at[r]);
    }
};

// Two values to a lane become others: of `a` the second half of the lanes (or the second of each
// two rows of 16 lanes) changes places with the first half (or the first) of `b`.
__device__ __forceinline__ void swap_halves(float* a, float* b) {
    const auto v = __builtin_amdgcn_permlane32_swap(__float_as_uint(*a), __float_as_uint(*b), false, false);
    *a = __uint_as_float(v[0]), *b = __uint_as_float(v[1]);
}
__device__ __forceinline__ void swap_rows(float* a, float* b) {
    const auto v = __builtin_amdgcn_permlane16_swap(__float_as_uint(*a), __float_as_uint(*b), false, false);
    *a = __uint_as_float(v[0]), *b = __uint_as_float(v[1]);
}
// Sums of four tokens' parts over a channel's four lanes: lanes of row i end with token i's.
// (Matrix instructions would take a token's sum times 0 into the others': not where it is infinite.)
__device__ __forceinline__ float token_sums(float v0, float v1, float v2, float v3) {
    swap_halves(&v0, &v2);
    swap_halves(&v1, &v3);
    float a = v0 + v2, b = v1 + v3;
    swap_rows(&a, &b);
    return a + b;
}
// Of a tile's four such (w[q]: lanes of row i have token 4 q + i) the lane's own tokens, 4 (lane / 16) + r.
__device__ __forceinline__ void own_tokens(f32x4* w) {
    float v0 = (*w)[0], v1 = (*w)[1], v2 = (*w)[2], v3 = (*w)[3];
    swap_halves(&v0, &v2);
    swap_halves(&v1, &v3);
    swap_rows(&v0, &v1);
    swap_rows(&v2, &v3);
    *w = f32x4{v0, v1, v2, v3};
}
__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }

// A lane's states of a block: rows 4 (lane / 16) .. + 3 of [states][channels].
__device__ __forceinline__ f32x4 load_states(const float* p, int n0, int N, long long D, int ch) {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = n0 + i < N ? p[(n0 + i) * D + ch] : 0.f;
    return v;
}
__device__ __forceinline__ void store_states(float* p, int n0, int N, long long D, int ch, f32x4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n0 + i < N) p[(n0 + i) * D + ch] = v[i];
}
// The same of [channels][states].
__device__ __forceinline__ f32x4 load_states_of(const float* p, int n0, int N) {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = n0 + i < N ? p[n0 + i] : 0.f;
    return v;
}
__device__ __forceinline__ void store_states_of(float* p, int n0, int N, f32x4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n0 + i < N) p[n0 + i] = v[i];
}

// A log2(e) as a finite number (NaN stays): the step of a token behind a row's end is 0, and its
// decay has to be 1 where A is -infinity, or next to it, too.
__device__ __forceinline__ float finite_rate(float a, float log2e = kLog2e) {
    const float v = log2e * a;
    return fabsf(v) == INFINITY ? copysignf(3.4e38f, v) : v;
}
__device__ __forceinline__ f32x4 finite_rates(f32x4 a) {
    return f32x4{finite_rate(a[0]), finite_rate(a[1]), finite_rate(a[2]), finite_rate(a[3])};
}

// Tokens of a chunk for channel blocks that give `waves` wavefronts per chunk.
int chunk_tokens(int tokens, long long waves);
int make_dims(const char* what, int batch, int tokens, int channels, int states, int groups, Dims* d);
int set_call(const char* what, Dims* d, const void* x, const void* dt, const float* A, const void* Bm, const void* C,
             const float* skip, const void* gate, const float* bias, const int* lengths, const long long* strides, int softplus,
             int dtype);
// Whether every launch of a forward takes its size, and of the backward that it saves for: a call is
// refused whole, and where it is for training.
int check_launches(const char* what, const Dims& d, bool training);
// States at the chunks' starts (forward) or the gradients at their ends (backward), in place
// of the chunks' own: h_{c+1} = exp(A sum_c) h_c + own_c, from `first` ([batch, D, N] or null).
int launch_join(const Dims& d, float* own, const float* sums, const float* first, bool backward, hipStream_t s);

}  // namespace scan
}  // namespace rka
