// The matrix product with its epilogue, y = act(x W^T + b) + r, and its gradients:
//   dz = dy act'(z), z = x W^T + b;  dx = dz W;  dW = dz^T x;  db = sum of dz's rows.
//
// One tile kernel serves the three products; they differ in how an operand's rows lie
// in memory (along the sum, or across it).  Both kinds end up in LDS as rows of 128
// bytes along the sum (64 bf16 or 32 float32), in 16-byte pieces whose order within
// a row is permuted by the row's number, so that neither the stores of transposed
// pieces nor the reads of 32 rows at once meet in a bank.
#include "rka_internal.h"

#include <algorithm>
#include <cmath>

namespace rka {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
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

// 16 bytes from or to any element's address (the hardware's loads and stores of
// four dwords ask for no alignment beyond the element's).
struct __attribute__((packed, aligned(2))) Bytes16 {
    unsigned w[4];
};
__device__ __forceinline__ u32x4 load16(const void* p) {
    const Bytes16 v = *static_cast<const Bytes16*>(p);
    return u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
}
__device__ __forceinline__ void store16(void* p, u32x4 v) {
    *static_cast<Bytes16*>(p) = Bytes16{{v[0], v[1], v[2], v[3]}};
}
__device__ __forceinline__ f32x4 load4(const float* p) { return __builtin_bit_cast(f32x4, load16(p)); }
__device__ __forceinline__ void store4(float* p, f32x4 v) { store16(p, __builtin_bit_cast(u32x4, v)); }
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);  // elements of 16 bytes

template <typename T>
union Piece {
    u32x4 u;
    T e[kVec<T>];
};

// ---------------------------------------------------------- activations ---
// exp and 1/x for results of type T: for bf16 the hardware's own, whose relative error (1e-6
// at |z| = 20) is far below its last bit.
template <typename T>
__device__ __forceinline__ float exp_for(float x) {
    if constexpr (sizeof(T) == 2)
        return __builtin_amdgcn_exp2f(1.4426950408889634f * x);
    else
        return expf(x);
}
template <typename T>
__device__ __forceinline__ float inverse_for(float x) {
    if constexpr (sizeof(T) == 2)
        return __builtin_amdgcn_rcpf(x);
    else
        return 1.f / x;
}
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
    return inverse_for<T>(1.f + exp_for<T>(-z));
}
// The normal distribution's function, half of erfc(x) at x = -z / sqrt(2).  For x >= 0,
// erfc(x) = exp(-x^2) t P(t) with t = 1 / (1 + 0.4 x) and P fitted over all of t in (0, 1]
// for the least relative error, 1.3e-7: no branch on z, where the library's erfc has three.
template <typename T>
__device__ __forceinline__ float normal(float z, float gauss) {  // gauss: exp(-z^2 / 2)
    const float t = inverse_for<T>(1.f + (0.4f * 0.70710678118654752f) * fabsf(z));
    float p = 0.05026539f;
    p = fmaf(p, t, -0.18291503f);
    p = fmaf(p, t, 0.16910847f);
    p = fmaf(p, t, -0.00562818f);
    p = fmaf(p, t, 0.14144189f);
    p = fmaf(p, t, 0.168539f);
    p = fmaf(p, t, 0.20784314f);
    p = fmaf(p, t, 0.22566957f);
    p = fmaf(p, t, 0.22567586f);
    const float tail = 0.5f * gauss * (p * t);
    return z < 0.f ? tail : 1.f - tail;
}
template <typename T>
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case RKA_ACT_RELU: return z < 0.f ? 0.f : z;  // NaN stays
        case RKA_ACT_GELU: return z * normal<T>(z, exp_for<T>(-0.5f * z * z));
        case RKA_ACT_SILU: return z * sigmoid<T>(z);
        case RKA_ACT_SIGMOID: return sigmoid<T>(z);
        case RKA_ACT_LOGSIGMOID: return (z < 0.f ? z : z != z ? z : 0.f) - log1pf(expf(-fabsf(z)));
        default: return z;
    }
}
// dy act'(z)
template <typename T>
__device__ __forceinline__ float slope(float dy, float z, int act) {
    switch (act) {
        case RKA_ACT_RELU: return z <= 0.f ? 0.f : dy;
        case RKA_ACT_GELU: {
            const float gauss = exp_for<T>(-0.5f * z * z);
            return dy * (normal<T>(z, gauss) + z * 0.3989422804014327f * gauss);
        }
        case RKA_ACT_SILU: return dy * sigmoid<T>(z) * (1.f + z * sigmoid<T>(-z));
        case RKA_ACT_SIGMOID: return dy * sigmoid<T>(z) * sigmoid<T>(-z);
        case RKA_ACT_LOGSIGMOID: return dy * sigmoid<T>(-z);
        default: return dy;
    }
}

// ------------------------------------------------------------- operands ---
// Rows of an operand are what the output's rows (or columns) are; the sum runs
// along k.  Element (row, k) at ptr[row * ld + k] (along) or ptr[k * ld + row] (across).
struct Operand {
    const void* ptr;
    long long ld;
};

struct Epilogue {
    const void* bias;      // [n] or null
    const void* residual;  // [m][ldr] or null
    long long ldr;
    void* z;  // [m][n] or null: the sum before the activation, for the backward
    int act;
};

struct Args {
    int m, n, k;
    Operand a, b;       // m rows, n rows
    void* c;            // [m][n]
    float* partial;     // [slice][m][n] where slices > 1
    int slices, stages; // stages of a slice
    Epilogue ep;
};

constexpr int kRowBytes = 128;  // of a stage's row

__device__ __forceinline__ int piece_at(int row, int piece) {
    return row * kRowBytes + (((piece ^ row ^ (row >> 3)) & 7) << 4);
}

// One operand's share of a stage in registers, on its way to LDS.
template <typename T, int ROWS, int NT, bool ACROSS>
struct Stage;

template <typename T, int ROWS, int NT>
struct Stage<T, ROWS, NT, false> {
    static constexpr int kV = kVec<T>, kK = 8 * kV, N = ROWS * 8 / NT;
    u32x4 v[N];

    __device__ __forceinline__ void load(const Operand& op, int row0, int rows, int k0, int k1, int tid) {
        const char* base = static_cast<const char*>(op.ptr) + ((long long)row0 * op.ld + k0) * (long long)sizeof(T);
        if (k0 + kK <= k1) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int x = tid + i * NT, r = min(x / 8, rows - 1 - row0);
                v[i] = load16(base + (unsigned)(r * (int)op.ld + x % 8 * kV) * (unsigned)sizeof(T));
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = tid + i * NT, r = min(x / 8, rows - 1 - row0), k = k0 + x % 8 * kV;
            const T* p = reinterpret_cast<const T*>(base) + (unsigned)(r * (int)op.ld + x % 8 * kV);
            Piece<T> q;
            q.u = u32x4{0, 0, 0, 0};
            if (k + kV <= k1) {
                q.u = load16(p);
            } else {
#pragma unroll
                for (int j = 0; j < kV; ++j)
                    if (k + j < k1) q.e[j] = p[j];
            }
            v[i] = q.u;
        }
    }
    __device__ __forceinline__ void store(char* lds, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = tid + i * NT;
            *reinterpret_cast<u32x4*>(lds + piece_at(x / 8, x % 8)) = v[i];
        }
    }
};

// Four k of kVec rows per unit, turned on their way.
template <typename T, int ROWS, int NT>
struct Stage<T, ROWS, NT, true> {
    static constexpr int kV = kVec<T>, kK = 8 * kV, kGroups = ROWS / kV, kUnits = kGroups * (kK / 4);
    static constexpr int N = (kUnits + NT - 1) / NT;
    u32x4 v[N][4];

    __device__ __forceinline__ void load(const Operand& op, int row0, int rows, int k0, int k1, int tid) {
        const char* base = static_cast<const char*>(op.ptr) + ((long long)k0 * op.ld + row0) * (long long)sizeof(T);
        const bool whole = k0 + kK <= k1 && row0 + ROWS <= rows;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = tid + i * NT;
            if (kUnits % NT != 0 && x >= kUnits) break;
            const int r = x % kGroups * kV, kk = x / kGroups * 4;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const T* p = reinterpret_cast<const T*>(base) + (unsigned)((kk + j) * (int)op.ld + r);
                if (whole) {
                    v[i][j] = load16(p);
                    continue;
                }
                Piece<T> q;
                q.u = u32x4{0, 0, 0, 0};
                if (k0 + kk + j < k1) {
                    if (row0 + r + kV <= rows) {
                        q.u = load16(p);
                    } else {
#pragma unroll
                        for (int e = 0; e < kV; ++e)
                            if (row0 + r + e < rows) q.e[e] = p[e];
                    }
                }
                v[i][j] = q.u;
            }
        }
    }
    __device__ __forceinline__ void store(char* lds, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = tid + i * NT;
            if (kUnits % NT != 0 && x >= kUnits) break;
            const int r = x % kGroups * kV, kk = x / kGroups;  // kk: quadruple of k
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<u32x4*>(lds + piece_at(r + e, kk)) =
                        u32x4{v[i][0][e], v[i][1][e], v[i][2][e], v[i][3][e]};
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    // bytes of the rows e of two k side by side
                    const unsigned sel = e % 2 ? 0x07060302u : 0x05040100u;
                    const u32x2 w{__builtin_amdgcn_perm(v[i][1][e / 2], v[i][0][e / 2], sel),
                                  __builtin_amdgcn_perm(v[i][3][e / 2], v[i][2][e / 2], sel)};
                    *reinterpret_cast<u32x2*>(lds + piece_at(r + e, kk / 2) + kk % 2 * 8) = w;
                }
            }
        }
    }
};

// 16 bytes of 32 rows each: 16 (bf16) or 8 (float32) k of a 32x32 block.
template <typename T>
__device__ __forceinline__ f32x16 multiply(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                       0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    }
}

// Waits until the last products of a wavefront's sums are in their registers, before sums
// are stored in another basic block than their last product's: between a matrix instruction
// and the reader of its result the compiler has missed wait states on paths that pass a
// branch.  18 states, what 32x32x2 float32 asks for, the most of those here.  (The sums are
// no operands of it: that copies them out of accumulation registers, before the wait.)
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 1" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Results of V neighbouring columns, with the epilogue.
template <typename T, int V>
__device__ __forceinline__ void finish(const Args& p, long long row, int col, const float (&sum)[V]) {
    const int left = p.n - col;  // columns that are the output's
    if (left <= 0) return;
    const size_t at = (size_t)row * p.n + col;
    const T* bias = p.ep.bias ? static_cast<const T*>(p.ep.bias) + col : nullptr;
    const T* res = p.ep.residual ? static_cast<const T*>(p.ep.residual) + row * p.ep.ldr + col : nullptr;
    T* c = static_cast<T*>(p.c) + at;
    T* z = p.ep.z ? static_cast<T*>(p.ep.z) + at : nullptr;
    if (V == kVec<T> && left >= V) {
        Piece<T> pb, pr, pz, pc;
        if (bias) pb.u = load16(bias);
        if (res) pr.u = load16(res);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float x = sum[j];
            if (bias) x += to_f32(pb.e[j]);
            pz.e[j] = from_f32<T>(x);
            x = activate<T>(x, p.ep.act);
            if (res) x += to_f32(pr.e[j]);
            pc.e[j] = from_f32<T>(x);
        }
        if (z) store16(z, pz.u);
        store16(c, pc.u);
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (j >= left) continue;
        float x = sum[j];
        if (bias) x += to_f32(bias[j]);
        if (z) z[j] = from_f32<T>(x);
        x = activate<T>(x, p.ep.act);
        if (res) x += to_f32(res[j]);
        c[j] = from_f32<T>(x);
    }
}

// The tile and slice of a workgroup: consecutive workgroups go to the eight XCDs in
// turn, so each XCD takes a run of tiles, in groups of eight tile rows whose operands
// then stay in its L2.
__device__ __forceinline__ void tile_of(int tiles_m, int tiles_n, int slices, int* tm, int* tn, int* slice) {
    const int total = tiles_m * tiles_n * slices, per = total / 8, rest = total % 8;
    const int xcd = blockIdx.x % 8, i = blockIdx.x / 8;
    int t = xcd * per + min(xcd, rest) + i;
    *slice = t / (tiles_m * tiles_n);
    t -= *slice * tiles_m * tiles_n;
    constexpr int G = 8;
    const int group = t / (G * tiles_n), first = group * G, rows = min(G, tiles_m - first), in = t - group * G * tiles_n;
    *tm = first + in % rows;
    *tn = in / rows;
}

// A wavefront's WM x WN of the output, from row0 and col0.  Through LDS (`out`), 32 rows
// at a time: a lane holds four neighbouring columns of one row, memory wants whole rows.
template <int WN>
constexpr int kOutBytes = 32 * (WN + 4) * 4;
template <typename T, int WM, int WN>
__device__ __forceinline__ void put_out(const Args& p, const f32x16 (&acc)[WM / 32][WN / 32], float* out, int row0, int col0,
                                        int slice) {
    constexpr int kLd = WN + 4, kV = kVec<T>, kLanes = WN / kV, kRows = 64 / kLanes, MB = WM / 32, NB = WN / 32;
    const int lane = threadIdx.x % 64, i32 = lane % 32, hi = lane / 32;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<f32x4*>(out + i32 * kLd + 32 * j + 8 * r + 4 * hi) =
                    f32x4{acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]};
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int x = 0; x < 32 / kRows; ++x) {
            const int r = x * kRows + lane / kLanes, c = lane % kLanes * kV;
            const int row = row0 + 32 * i + r, col = col0 + c;
            float sum[kV];
#pragma unroll
            for (int e = 0; e < kV; e += 4) {
                const f32x4 q = *reinterpret_cast<const f32x4*>(out + r * kLd + c + e);
#pragma unroll
                for (int y = 0; y < 4; ++y) sum[e + y] = q[y];
            }
            if (row >= p.m) continue;
            if (p.slices > 1) {
                float* part = p.partial + ((size_t)slice * p.m + row) * p.n + col;
                if (col + kV <= p.n) {
#pragma unroll
                    for (int e = 0; e < kV; e += 4) store4(part + e, f32x4{sum[e], sum[e + 1], sum[e + 2], sum[e + 3]});
                    continue;
                }
#pragma unroll
                for (int e = 0; e < kV; ++e)
                    if (col + e < p.n) part[e] = sum[e];
            } else {
                finish<T, kV>(p, row, col, sum);
            }
        }
    }
}

// BM x BN tiles, WM x WN of them per wavefront: through registers, for operands that are
// turned on their way and for rows of any address and length.  Bound by its waits: the
// registers that hold the next stage leave those of one k step's fragments, so that
// LDS's latency shows between the products.  8192 x 2048 over 2048 bf16, one operand
// turned: 87 us, 790 TFLOP/s; direct_kernel: 69 us.
template <typename T, int BM, int BN, int WM, int WN, bool A_ACROSS, bool B_ACROSS>
__global__ __launch_bounds__(BM / WM * BN / WN * 64) void tile_kernel(Args p) {
    constexpr int NT = BM / WM * BN / WN * 64, kK = 8 * kVec<T>, MB = WM / 32, NB = WN / 32;
    constexpr int kStage = (BM + BN) * kRowBytes;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, i32 = lane % 32, hi = lane / 32;
    int tm, tn, slice;
    tile_of((p.m - 1) / BM + 1, (p.n - 1) / BN + 1, p.slices, &tm, &tn, &slice);
    const int m0 = tm * BM, n0 = tn * BN, wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
    const int kbeg = min(p.k, slice * p.stages * kK), kend = min(p.k, kbeg + p.stages * kK);
    Stage<T, BM, NT, A_ACROSS> sa;
    Stage<T, BN, NT, B_ACROSS> sb;
    f32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x16{};
    const int stages = (kend - kbeg + kK - 1) / kK;
    if (stages > 0) {
        sa.load(p.a, m0, p.m, kbeg, kend, tid);
        sb.load(p.b, n0, p.n, kbeg, kend, tid);
        sa.store(lds, tid);
        sb.store(lds + BM * kRowBytes, tid);
        __syncthreads();
    }
    for (int s = 0; s < stages; ++s) {
        const char* cur = lds + s % 2 * kStage;
        if (s + 1 < stages) {
            sa.load(p.a, m0, p.m, kbeg + (s + 1) * kK, kend, tid);
            sb.load(p.b, n0, p.n, kbeg + (s + 1) * kK, kend, tid);
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            u32x4 fa[MB], fb[NB];
#pragma unroll
            for (int i = 0; i < MB; ++i)
                fa[i] = *reinterpret_cast<const u32x4*>(cur + piece_at(wm + 32 * i + i32, kk * 2 + hi));
#pragma unroll
            for (int j = 0; j < NB; ++j)
                fb[j] = *reinterpret_cast<const u32x4*>(cur + BM * kRowBytes + piece_at(wn + 32 * j + i32, kk * 2 + hi));
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j) acc[i][j] = multiply<T>(fb[j], fa[i], acc[i][j]);
        }
        if (s + 1 < stages) {
            char* next = lds + (s + 1) % 2 * kStage;
            sa.store(next, tid);
            sb.store(next + BM * kRowBytes, tid);
        }
        __syncthreads();
    }
    settle();
    put_out<T, WM, WN>(p, acc, reinterpret_cast<float*>(lds + wave * kOutBytes<WN>), m0 + wm, n0 + wn, slice);
}

// Order of the 16-byte pieces of a row: sixteen rows' pieces of one number are on
// different banks, and 32 rows further the order is the same.
__device__ __forceinline__ int direct_turn(int row) { return (row ^ (row >> 3 & 3)) & 7; }

// The same for operands that both lie along the sum, in whole stages and on 16 bytes:
// they go from memory to LDS without registers between, which leaves those for the
// fragments of the next products.  16384 x 4096 over 4096 bf16: 458 us, 1200 TFLOP/s (576
// through registers).  Bound by how the loads and their arrival interleave with the products:
// the matrix instructions are busy for 52% of the clocks, LDS for 21%; without the loads (a
// copy, with wrong results) 344 us, with all of them from L2 461; half stages in a ring of four,
// whose next fragments are read before the barrier, 494 (rows of 64 bytes); 128 x 128 to a
// wavefront, with one wavefront to a SIMD, 565.
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(BM / WM * BN / WN * 64) void direct_kernel(Args p) {
    constexpr int W = BM / WM * BN / WN, kK = 8 * kVec<T>, MB = WM / 32, NB = WN / 32;
    constexpr int kStage = (BM + BN) * kRowBytes, kLoads = (BM + BN) / 8 / W;  // a wavefront's, 8 rows each
    constexpr int kBuffer = kStage > W / 2 * kOutBytes<WN> ? kStage : W / 2 * kOutBytes<WN>;
    // (two variables, by which the compiler knows that reads of the one need not wait for
    // loads into the other)
    __shared__ __attribute__((aligned(16))) char even[kBuffer];
    __shared__ __attribute__((aligned(16))) char odd[kBuffer];
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), i32 = lane % 32, hi = lane / 32;
    int tm, tn, slice;
    tile_of((p.m - 1) / BM + 1, (p.n - 1) / BN + 1, p.slices, &tm, &tn, &slice);
    const int m0 = tm * BM, n0 = tn * BN, wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
    const int kbeg = min(p.k, slice * p.stages * kK), kend = min(p.k, kbeg + p.stages * kK);
    const int stages = (kend - kbeg) / kK;
    // What lane l loads goes to LDS's l-th 16 bytes of 8 rows: it is the piece that
    // belongs there.  A wavefront loads rows of one operand.
    const bool of_a = wave < W / 2;
    const Operand& op = of_a ? p.a : p.b;
    const int row0 = of_a ? m0 : n0, rows = of_a ? p.m : p.n, first = wave % (W / 2) * kLoads * 8;
    const auto memory = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(static_cast<const char*>(op.ptr)) + ((long long)row0 * op.ld + kbeg) * (long long)sizeof(T), 0,
        (int)0xffffffffu, 0x27000);
    unsigned from[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int row = first + i * 8 + lane / 8;
        from[i] = (unsigned)min(row, rows - 1 - row0) * ((unsigned)op.ld * (unsigned)sizeof(T)) + (lane % 8 ^ direct_turn(row)) * 16;
    }
    auto load = [&](char* to, int stage, int i0, int i1) {
#pragma unroll
        for (int i = i0; i < i1; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                memory, (__attribute__((address_space(3))) void*)(to + (wave * kLoads + i) * 8 * kRowBytes), 16, (int)from[i],
                stage * kRowBytes, 0, 0);
    };
    f32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x16{};
    // (the next stage's loads are issued in two lots, 1.5% faster than in one)
    auto compute = [&](const char* cur, char* next, int stage) {
        u32x4 fa[2][MB], fb[2][NB];
        // (made here each time: the addresses of all stages would fill the registers)
        unsigned at = i32 * kRowBytes + ((hi ^ direct_turn(i32)) << 4);
        asm volatile("" : "+v"(at));
        auto read = [&](int kk) {
            const char* of = cur + (at ^ (unsigned)kk << 5);
#pragma unroll
            for (int j = 0; j < NB; ++j)
                fb[kk % 2][j] = *reinterpret_cast<const u32x4*>(of + (BM + wn + 32 * j) * kRowBytes);
#pragma unroll
            for (int i = 0; i < MB; ++i) fa[kk % 2][i] = *reinterpret_cast<const u32x4*>(of + (wm + 32 * i) * kRowBytes);
        };
        read(0);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            if (kk < 3) read(kk + 1);
            if (next && kk < 2) load(next, stage, kk * kLoads / 2, (kk + 1) * kLoads / 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j) acc[i][j] = multiply<T>(fb[kk % 2][j], fa[kk % 2][i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // all of the wavefront's loads are in LDS, then everyone's
    auto arrive = [&] {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    load(even, 0, 0, kLoads);
    arrive();
    int s = 0;
    for (; s + 2 < stages; s += 2) {
        compute(even, odd, s + 1);
        arrive();
        compute(odd, even, s + 2);
        arrive();
    }
    if (s + 1 < stages) load(odd, s + 1, 0, kLoads);
    compute(even, nullptr, 0);
    settle();
    arrive();
    if (s + 1 < stages) {
        compute(odd, nullptr, 0);
        settle();
    }
    __syncthreads();
    float* out = reinterpret_cast<float*>((wave < W / 2 ? even : odd) + wave % (W / 2) * kOutBytes<WN>);
    put_out<T, WM, WN>(p, acc, out, m0 + wm, n0 + wn, slice);
}

// The slices' sums, always in their order, and the epilogue.
template <typename T>
__global__ __launch_bounds__(256) void slices_kernel(Args p) {
    constexpr int kV = kVec<T>;
    const int groups = (p.n + kV - 1) / kV;
    const long long total = (long long)p.m * groups;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long row = i / groups;
        const int col = (int)(i % groups) * kV;
        float sum[kV] = {};
        const float* part = p.partial + (size_t)row * p.n + col;
        if (col + kV <= p.n) {
#pragma unroll 4
            for (int s = 0; s < p.slices; ++s, part += (size_t)p.m * p.n) {
#pragma unroll
                for (int e = 0; e < kV; e += 4) {
                    const f32x4 q = load4(part + e);
#pragma unroll
                    for (int y = 0; y < 4; ++y) sum[e + y] += q[y];
                }
            }
        } else {
            for (int s = 0; s < p.slices; ++s, part += (size_t)p.m * p.n) {
#pragma unroll
                for (int e = 0; e < kV; ++e)
                    if (col + e < p.n) sum[e] += part[e];
            }
        }
        finish<T, kV>(p, row, col, sum);
    }
}

// Few rows: 16 columns of the output per workgroup, whose wavefronts share the sum.
// The weight goes from memory to the matrix instructions' operands directly, every
// element once.  4 rows of 4096 over 2048 bf16 (16.8 MB, which the chip's caches hold
// between calls): 5.7 us.
// SWAP: few columns instead, 16 rows of x per workgroup: a is the weight, b is x, and the
// output is written the other way round.
constexpr int kRowsThreads = 512;
template <typename T, int MT, bool SWAP>
__global__ __launch_bounds__(kRowsThreads) void rows_kernel(Args p) {
    constexpr int kV = kVec<T>, kK = 4 * kV, kWaves = kRowsThreads / 64, kDeep = 4;
    __shared__ float sums[kWaves][MT][16][17];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, i16 = lane % 16, hi = lane / 16;
    const int n0 = blockIdx.x * 16;
    const T* w = static_cast<const T*>(p.b.ptr) + (long long)min(n0 + i16, p.n - 1) * p.b.ld;
    const T* x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = static_cast<const T*>(p.a.ptr) + (long long)min(16 * t + i16, p.m - 1) * p.a.ld;
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto fetch = [&](const T* q, int k) {
        Piece<T> v;
        v.u = u32x4{0, 0, 0, 0};
        if (k + kV <= p.k) {
            v.u = load16(q + k);
        } else {
#pragma unroll
            for (int j = 0; j < kV; ++j)
                if (k + j < p.k) v.e[j] = q[k + j];
        }
        return v.u;
    };
    for (int k0 = wave * kK * kDeep; k0 < p.k; k0 += kWaves * kK * kDeep) {
        u32x4 fw[kDeep], fx[kDeep][MT];
#pragma unroll
        for (int s = 0; s < kDeep; ++s) fw[s] = fetch(w, k0 + s * kK + hi * kV);
#pragma unroll
        for (int s = 0; s < kDeep; ++s)
#pragma unroll
            for (int t = 0; t < MT; ++t) fx[s][t] = fetch(x[t], k0 + s * kK + hi * kV);
#pragma unroll
        for (int s = 0; s < kDeep; ++s)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if constexpr (sizeof(T) == 2) {
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fx[s][t]),
                                                                     __builtin_bit_cast(bf16x8, fw[s]), acc[t], 0, 0, 0);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(fx[s][t][j]),
                                                                      __uint_as_float(fw[s][j]), acc[t], 0, 0, 0);
                }
            }
    }
    settle();
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[wave][t][4 * hi + r][i16] = acc[t][r];
    __syncthreads();
    Args out = p;
    if (SWAP) out.n = p.m;
    for (int i = threadIdx.x; i < MT * 256; i += kRowsThreads) {
        const int t = SWAP ? i / 16 % MT : i / 256, r = SWAP ? i % 16 : i / 16 % 16, c = SWAP ? i / (16 * MT) : i % 16;
        if (16 * t + r >= p.m || n0 + c >= p.n) continue;
        float sum[1] = {0.f};
#pragma unroll
        for (int k = 0; k < kWaves; ++k) sum[0] += sums[k][t][r][c];
        if (SWAP)
            finish<T, 1>(out, n0 + c, 16 * t + r, sum);
        else
            finish<T, 1>(out, 16 * t + r, n0 + c, sum);
    }
}

// dz = dy act'(z) and the sums of its columns over a range of rows: 8 rows of 32
// threads per workgroup, kVec columns each.  z comes, and dz goes, as T: the products that
// take dz are products of T, and in bf16 z is half of what the forward keeps; dx and dW
// are then off by 0.0024 instead of 0.0017 (db, summed before the rounding, by less).
// Bound by memory: 8192 x 2048 bf16 (100 MB) 20 us, 5 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void slope_kernel(const T* dy, long long lddy, const T* z, T* dz, float* sums, int m,
                                                    int n, int rows_per_block, int act) {
    constexpr int kV = kVec<T>;
    __shared__ float part[8][32 * kV + 1];
    const int c = threadIdx.x % 32 * kV, col = blockIdx.x * 32 * kV + c, r0 = threadIdx.x / 32;
    const long long first = (long long)blockIdx.y * rows_per_block, last = min((long long)m, first + rows_per_block);
    float sum[kV] = {};
    if (col < n) {
        const int left = min(kV, n - col);
        for (long long row = first + r0; row < last; row += 8) {
            Piece<T> a, b, o;
            const T* pa = dy + row * lddy + col;
            const T* pb = z ? z + row * n + col : nullptr;
            T* po = dz ? dz + row * n + col : nullptr;
            if (left == kV) {
                a.u = load16(pa);
                if (pb) b.u = load16(pb);
            } else {
#pragma unroll
                for (int j = 0; j < kV; ++j)
                    if (j < left) {
                        a.e[j] = pa[j];
                        if (pb) b.e[j] = pb[j];
                    }
            }
#pragma unroll
            for (int j = 0; j < kV; ++j) {
                const float g = slope<T>(to_f32(a.e[j]), pb ? to_f32(b.e[j]) : 0.f, act);
                o.e[j] = from_f32<T>(g);
                if (j < left) sum[j] += g;
            }
            if (po) {
                if (left == kV) {
                    store16(po, o.u);
                } else {
#pragma unroll
                    for (int j = 0; j < kV; ++j)
                        if (j < left) po[j] = o.e[j];
                }
            }
        }
    }
    if (!sums) return;
#pragma unroll
    for (int j = 0; j < kV; ++j) part[r0][c + j] = sum[j];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * kV; i += 256) {
        const int at = blockIdx.x * 32 * kV + i;
        if (at >= n) break;
        float s = part[0][i];
#pragma unroll
        for (int r = 1; r < 8; ++r) s += part[r][i];
        sums[(size_t)blockIdx.y * n + at] = s;
    }
}

// db from the ranges' sums, always in their order.
template <typename T>
__global__ __launch_bounds__(256) void bias_kernel(const float* sums, int ranges, int n, T* db) {
    __shared__ float part[16][17];
    const int c = threadIdx.x % 16, p = threadIdx.x / 16, col = blockIdx.x * 16 + c;
    float s = 0.f;
    if (col < n)
        for (int r = p; r < ranges; r += 16) s += sums[(size_t)r * n + col];
    part[p][c] = s;
    __syncthreads();
    if (p != 0 || col >= n) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) s += part[k][c];
    db[col] = from_f32<T>(s);
}

// ------------------------------------------------------------- choices ---
enum Tile { TILE_256, TILE_128, TILE_64 };
constexpr long long kLaunchThreads = 1LL << 32;  // a launch has fewer
struct Plan {
    Tile tile;
    int slices, stages;
    double cost;
};

// Tile and slices of a product: the least of a model of the time in us.  A stage of a
// tile takes a CU `work` of its time and, alone there, `least` (the loads' latency);
// measured with 1, 2 and 4 workgroups to a CU, bf16: 256: 1.8; 128: 0.7, 1.1; 64: 0.25-0.5,
// 0.4, 0.73.  `across`: an operand is turned on its way.  Slices write and read float32 sums.
// Of 24 products measured with every choice, the one taken costs at most a tenth more than
// the best for 23: 8192 x 2048 x 2048's gradient of the weight 91 us with 256 tiles in 4
// slices, 148 and 234 with 64 and 256 tiles unsliced; 8192 x 32 over 2048 12 and 19 us with 64
// tiles in 4 slices and one.  The 24th: float32's gradient of a 1024 x 1024 weight over 4096
// rows, 118 us with 64 tiles in 2 slices, 85 with 128 tiles in 8.
Plan plan_product(int m, int n, int k, int esize, bool across) {
    const int kk = kRowBytes / esize, all = std::max(1, (k + kk - 1) / kk);
    struct Cost {
        Tile tile;
        int edge, threads;
        double share, least, work, turn, f32;
    };
    // (float32: four 128 tiles, two to a CU, are faster than a 256 tile at any count)
    static const Cost costs[] = {{TILE_256, 256, 512, 1, 1.8, 1.8, 1.2, 0},
                                 {TILE_128, 128, 256, 2, 0.7, 0.55, 1.2, 3.1},
                                 {TILE_64, 64, 256, 4, 0.35, 0.165, 1.25, 2.95}};
    Plan best{TILE_64, 1, all, 1e30};
    for (const Cost& c : costs) {
        if (esize == 4 && c.tile == TILE_256) continue;
        const double tiles = (double)((m - 1) / c.edge + 1) * ((n - 1) / c.edge + 1);
        for (int want = 1; want <= 64 && want <= all; want *= 2) {
            const int stages = (all + want - 1) / want, slices = (all + stages - 1) / stages;
            if (tiles * slices * c.threads >= kLaunchThreads) continue;
            const double to_a_cu = std::ceil(tiles * slices / 256), rounds = std::floor(to_a_cu / c.share), rest = to_a_cu - rounds * c.share;
            double stage = rounds * std::max(c.least, c.share * c.work) + (rest > 0 ? std::max(c.least, rest * c.work) : 0);
            if (across) stage *= c.turn;
            if (esize == 4) stage *= c.f32;
            double cost = (stages + 3) * stage;
            if (slices > 1) cost += 3 + 0.15 * slices + (double)slices * m * n * 8 / 6e6;
            if (cost < best.cost) best = Plan{c.tile, slices, stages, cost};
        }
    }
    return best;
}
size_t partial_bytes(int m, int n, const Plan& p) {
    return p.slices > 1 ? align_up((size_t)p.slices * m * n * sizeof(float), 256) : 0;
}
// The rows' kernel, whose workgroup goes through the whole sum, for few rows or few columns
// (with a workgroup for 16 of the others), or tiles, in slices where those are few: models of
// the measured times in us.  Rows and tiles, bf16, 4096 columns over 2048: 1 row 4.6 and 8.6, 16
// 5.7 and 9.7, 32 7.6 and 10.7; 256 columns over 4096: 8 rows 7.4 and 9.9, 32 12.3 and 10.7.
// float32, 64 columns over 4096: 1 row 11.5 and 8.7.  Columns and tiles, bf16, over 2048: 16
// columns of 2048 rows 5.5 and 9.1, of 8192 9.2 and 11.2, of 65536 65 and 40; 32 of 8192 13.9
// and 11.8.  float32: 16 of 8192 18.9 and 25.0, 32 29.5 and 25.0.
enum Few { FEW_NONE, FEW_ROWS, FEW_COLUMNS };
// (tiles also where a launch may not have a workgroup for 16 of the others)
Few few_of(int m, int n, int k, int esize) {
    if ((long long)((m <= 32 ? n : m) - 1) / 16 + 1 >= kLaunchThreads / kRowsThreads) return FEW_NONE;
    const double row = (double)k * esize, kb = row / 1024;
    if (m <= 32) return 4 + kb * (m <= 16 ? 0.5 : 1.15) < 9.3 + n * row / 6e6 ? FEW_ROWS : FEW_NONE;
    if (n > 32) return FEW_NONE;
    const double rounds = ((m - 1) / 16 + 1) / 512.0, at_once = n <= 16 ? std::max(0.5, 1.5 * rounds) : std::max(1.15, 2.5 * rounds);
    return 4 + kb * at_once * (esize == 4 ? 1.4 : 1) < 2.5 + plan_product(m, n, k, esize, false).cost ? FEW_COLUMNS : FEW_NONE;
}

// Whether a sum is whole stages, which direct_kernel takes.
bool whole_stages(int k, int esize) { return k % (kRowBytes / esize) == 0; }

template <int N>
using Int = std::integral_constant<int, N>;

template <typename T, bool A, bool B>
int launch_tiles(const Args& p, Tile tile, hipStream_t s) {
    auto go = [&](auto kernel, bool direct, int edge, int wm, int wn) {
        const int threads = edge / wm * edge / wn * 64;
        const long long blocks = (long long)((p.m - 1) / edge + 1) * ((p.n - 1) / edge + 1) * p.slices;
        if (blocks * threads >= kLaunchThreads) return fail(RKA_ERR_UNSUPPORTED_SHAPE, "linear: more workgroups than a launch may have");
        const size_t lds = direct ? 0 : std::max<size_t>((size_t)4 * edge * kRowBytes, (size_t)threads / 64 * 32 * (wn + 4) * 4);
        if (lds > (64 << 10))
            RKA_RETURN_IF_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, s, p);
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    };
    auto either = [&](auto direct) {
        constexpr bool D = decltype(direct)::value;
        const auto kernel = [](auto bm, auto wm, auto wn) {
            constexpr int BM = decltype(bm)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
            if constexpr (D)
                return &direct_kernel<T, BM, BM, WM, WN>;
            else
                return &tile_kernel<T, BM, BM, WM, WN, A, B>;
        };
        if constexpr (sizeof(T) == 2)
            if (tile == TILE_256) return go(kernel(Int<256>{}, Int<128>{}, Int<64>{}), D, 256, 128, 64);
        if (tile == TILE_128) return go(kernel(Int<128>{}, Int<64>{}, Int<64>{}), D, 128, 64, 64);
        return go(kernel(Int<64>{}, Int<32>{}, Int<32>{}), D, 64, 32, 32);
    };
    bool done = false;
    if constexpr (!A && !B) {
        const auto on16 = [](const Operand& o) { return (reinterpret_cast<uintptr_t>(o.ptr) | (size_t)o.ld * sizeof(T)) % 16 == 0; };
        if (whole_stages(p.k, sizeof(T)) && on16(p.a) && on16(p.b)) {
            RKA_RETURN_IF_ERR(either(std::true_type{}));
            done = true;
        }
    }
    if (!done) RKA_RETURN_IF_ERR(either(std::false_type{}));
    if (p.slices > 1) {
        const long long items = (long long)p.m * ((p.n + kVec<T> - 1) / kVec<T>);
        hipLaunchKernelGGL((slices_kernel<T>), dim3((unsigned)std::min<long long>((items + 255) / 256, 2048)), dim3(256), 0, s, p);
        RKA_RETURN_IF_HIP(hipGetLastError());
    }
    return 0;
}

// C = A B^T (+ epilogue); `partial` holds partial_bytes of the plan.
template <typename T, bool A, bool B>
int product(int m, int n, int k, const Operand& a, const Operand& b, void* c, const Epilogue& ep, float* partial,
            hipStream_t s) {
    const Plan plan = plan_product(m, n, k, sizeof(T), A || B);
    return launch_tiles<T, A, B>(Args{m, n, k, a, b, c, partial, plan.slices, plan.stages, ep}, plan.tile, s);
}

template <typename T>
int forward(int m, int n, int k, const Operand& x, const Operand& w, void* y, const Epilogue& ep, float* partial,
            hipStream_t s) {
    const Few few = few_of(m, n, k, sizeof(T));
    if (few == FEW_NONE) return product<T, false, false>(m, n, k, x, w, y, ep, partial, s);
    const bool swap = few == FEW_COLUMNS;
    const Args p = swap ? Args{n, m, k, w, x, y, nullptr, 1, 0, ep} : Args{m, n, k, x, w, y, nullptr, 1, 0, ep};
    const auto kernel = p.m <= 16 ? (swap ? &rows_kernel<T, 1, true> : &rows_kernel<T, 1, false>)
                                  : (swap ? &rows_kernel<T, 2, true> : &rows_kernel<T, 2, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)((p.n - 1) / 16 + 1)), dim3(kRowsThreads), 0, s, p);
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}

// Row ranges of the slope kernel: enough workgroups for the GPU, at least two rows to a thread
// (with eight, 1000 rows of 385 float32 took 18 us).
int slope_ranges(int m, int n, int esize, int* rows) {
    const int cols = (n - 1) / (32 * (16 / esize)) + 1;
    const int want = std::max(1, 2048 / cols);
    *rows = std::max(16, ((m - 1) / want + 8) / 8 * 8);
    return (m - 1) / *rows + 1;
}

struct BackwardLayout {
    size_t dz, sums, partial, total;
};
BackwardLayout backward_layout(int m, int n, int k, int esize) {
    BackwardLayout l{};
    int rows = 0;
    l.dz = 0;
    l.sums = align_up((size_t)m * n * esize, 256);
    l.partial = l.sums + align_up((size_t)slope_ranges(m, n, esize, &rows) * n * sizeof(float), 256);
    // one after the other on the stream
    l.total = l.partial + std::max(partial_bytes(m, k, plan_product(m, k, n, esize, true)), partial_bytes(n, k, plan_product(n, k, m, esize, true)));
    return l;
}

template <typename T>
int backward(int m, int n, int k, const Operand& dy, const Operand& x, const Operand& w, const void* z, void* dx, void* dw,
             void* db, int act, char* ws, hipStream_t s) {
    const BackwardLayout l = backward_layout(m, n, k, sizeof(T));
    Operand dz = dy;
    if (act != RKA_ACT_NONE || db) {
        int rows = 0;
        const int ranges = slope_ranges(m, n, sizeof(T), &rows);
        T* out = act != RKA_ACT_NONE ? reinterpret_cast<T*>(ws + l.dz) : nullptr;
        float* sums = db ? reinterpret_cast<float*>(ws + l.sums) : nullptr;
        hipLaunchKernelGGL((slope_kernel<T>), dim3((unsigned)((n - 1) / (32 * kVec<T>) + 1), (unsigned)ranges), dim3(256), 0,
                           s, static_cast<const T*>(dy.ptr), dy.ld, static_cast<const T*>(z), out, sums, m, n, rows, act);
        RKA_RETURN_IF_HIP(hipGetLastError());
        if (db) {
            hipLaunchKernelGGL((bias_kernel<T>), dim3((unsigned)((n - 1) / 16 + 1)), dim3(256), 0, s, sums, ranges, n,
                               static_cast<T*>(db));
            RKA_RETURN_IF_HIP(hipGetLastError());
        }
        if (out) dz = Operand{out, n};
    }
    float* partial = reinterpret_cast<float*>(ws + l.partial);
    if (dx) RKA_RETURN_IF_ERR((product<T, false, true>(m, k, n, dz, w, dx, Epilogue{}, partial, s)));
    if (dw) RKA_RETURN_IF_ERR((product<T, true, true>(n, k, m, dz, x, dw, Epilogue{}, partial, s)));
    return 0;
}

int check(const char* what, int m, int n, int k, long long ld0, long long ld1, long long ld2, int act, int dtype) {
    const std::string name(what);
    if (m < 1 || n < 1 || k < 1) return fail(RKA_ERR_INVALID_ARGUMENT, name + ": sizes must be >= 1");
    if (act < RKA_ACT_NONE || act > RKA_ACT_LOGSIGMOID) return fail(RKA_ERR_INVALID_ARGUMENT, name + ": unknown activation");
    if (dtype != RKA_DTYPE_F32 && dtype != RKA_DTYPE_BF16)
        return fail(RKA_ERR_INVALID_ARGUMENT, name + ": dtype must be RKA_DTYPE_F32 or RKA_DTYPE_BF16");
    // a tile's 32-bit offsets: 256 rows of a leading dimension
    constexpr long long kMost = 1LL << 21;
    for (const long long ld : {ld0, ld1, ld2, (long long)n, (long long)k})
        if (ld < 0 || ld > kMost) return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": row strides, inputs and outputs must be at most 2^21 elements");
    return 0;
}

}  // namespace
}  // namespace rka

using namespace rka;

extern "C" {

size_t rka_linear_forward_workspace_bytes(int rows, int outputs, int inputs, int dtype) {
    const int esize = dtype == RKA_DTYPE_F32 ? 4 : 2;
    if (rows < 1 || outputs < 1 || inputs < 1 || few_of(rows, outputs, inputs, esize) != FEW_NONE) return 0;
    return partial_bytes(rows, outputs, plan_product(rows, outputs, inputs, esize, false));
}

size_t rka_linear_backward_workspace_bytes(int rows, int outputs, int inputs, int dtype) {
    if (rows < 1 || outputs < 1 || inputs < 1) return 0;
    return backward_layout(rows, outputs, inputs, dtype == RKA_DTYPE_F32 ? 4 : 2).total;
}

int rka_describe_linear(int product, int rows, int outputs, int inputs, int dtype, int aligned, int* out, int n_out) {
    clear_error();
    if (product < 0 || product > 2 || !out || n_out < 1)
        return fail(RKA_ERR_INVALID_ARGUMENT, "describe_linear: product must be 0, 1 or 2, out non-NULL and n_out >= 1");
    RKA_RETURN_IF_ERR(check("describe_linear", rows, outputs, inputs, 0, 0, 0, RKA_ACT_NONE, dtype));
    const int esize = dtype == RKA_DTYPE_F32 ? 4 : 2;
    const int m = product == 2 ? outputs : rows, n = product == 0 ? outputs : inputs;
    const int k = product == 0 ? inputs : product == 1 ? outputs : rows;
    const Few few = product == 0 ? few_of(m, n, k, esize) : FEW_NONE;
    int v[4] = {few == FEW_ROWS ? RKA_LINEAR_FORM_ROWS : RKA_LINEAR_FORM_COLUMNS, 16, 1,
                ((few == FEW_ROWS ? n : m) - 1) / 16 + 1};
    if (few == FEW_NONE) {
        const Plan p = plan_product(m, n, k, esize, product != 0);
        const int edge = p.tile == TILE_256 ? 256 : p.tile == TILE_128 ? 128 : 64;
        const long long blocks = (long long)((m - 1) / edge + 1) * ((n - 1) / edge + 1) * p.slices;
        v[0] = product == 0 && aligned && whole_stages(k, esize) ? RKA_LINEAR_FORM_DIRECT : RKA_LINEAR_FORM_TILES;
        v[1] = edge;
        v[2] = p.slices;
        v[3] = (int)std::min<long long>(blocks, 0x7fffffff);
    }
    for (int i = 0; i < 4 && i < n_out; ++i) out[i] = v[i];
    return 0;
}

int rka_linear_forward(const void* x, long long ldx, const void* weight, long long ldw, const void* bias,
                       const void* residual, long long ldr, void* y, void* z, void* workspace, size_t workspace_bytes,
                       int rows, int outputs, int inputs, int act, int dtype, void* stream) {
    clear_error();
    if (rows == 0 && outputs > 0 && inputs > 0) return 0;
    RKA_RETURN_IF_ERR(check("linear_forward", rows, outputs, inputs, ldx, ldw, residual ? ldr : 0, act, dtype));
    if (!x || !weight || !y) return fail(RKA_ERR_INVALID_ARGUMENT, "linear_forward: null tensor pointer");
    const size_t need = rka_linear_forward_workspace_bytes(rows, outputs, inputs, dtype);
    if (workspace_bytes < need || (need > 0 && !workspace))
        return fail(RKA_ERR_WORKSPACE_TOO_SMALL, "linear_forward: workspace needs " + std::to_string(need) + " bytes, got " +
                                                     std::to_string(workspace_bytes));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const Epilogue ep{bias, residual, ldr, z, act};
    float* partial = static_cast<float*>(workspace);
    return dtype == RKA_DTYPE_F32
               ? forward<float>(rows, outputs, inputs, Operand{x, ldx}, Operand{weight, ldw}, y, ep, partial, s)
               : forward<bf16>(rows, outputs, inputs, Operand{x, ldx}, Operand{weight, ldw}, y, ep, partial, s);
}

int rka_linear_backward(const void* grad_y, long long ldy, const void* x, long long ldx, const void* weight, long long ldw,
                        const void* z, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                        size_t workspace_bytes, int rows, int outputs, int inputs, int act, int dtype, void* stream) {
    clear_error();
    RKA_RETURN_IF_ERR(check("linear_backward", rows, outputs, inputs, ldy, ldx, ldw, act, dtype));
    if (!grad_y || (grad_weight && !x) || (grad_x && !weight) || (act != RKA_ACT_NONE && !z))
        return fail(RKA_ERR_INVALID_ARGUMENT, "linear_backward: null tensor pointer");
    const size_t need = rka_linear_backward_workspace_bytes(rows, outputs, inputs, dtype);
    if (workspace_bytes < need || !workspace)
        return fail(RKA_ERR_WORKSPACE_TOO_SMALL, "linear_backward: workspace needs " + std::to_string(need) +
                                                     " bytes, got " + std::to_string(workspace_bytes));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    const Operand dy{grad_y, ldy}, xo{x, ldx}, wo{weight, ldw};
    return dtype == RKA_DTYPE_F32
               ? backward<float>(rows, outputs, inputs, dy, xo, wo, z, grad_x, grad_weight, grad_bias, act, ws, s)
               : backward<bf16>(rows, outputs, inputs, dy, xo, wo, z, grad_x, grad_weight, grad_bias, act, ws, s);
}

}  // extern "C"
