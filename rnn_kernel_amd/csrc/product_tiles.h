// Tiles of a matrix product on the matrix cores, for the operators that are products: C =
// A B^T, with operands whose rows lie along the sum in memory, or across it.  Both kinds end up
// in LDS as rows of 128 bytes along the sum (64 bf16 or 32 float32), in 16-byte pieces whose
// order within a row is permuted by the row's number, so that neither the stores of transposed
// pieces nor the reads of 32 rows at once meet in a bank.
//
// A kernel's argument P is a Product with what becomes of the sums: put<T, WM, WN>(acc, lds,
// row0, col0, slice) takes a wavefront's.  live_rows() and depth() are how many rows of C, and
// how long a sum, the call has: kDynamic says that only the GPU knows.
#pragma once

#include "elementwise.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace rka {
namespace tiles {

using namespace elem;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ u32x4 load16(const void* p) {
    const Bytes16 v = *static_cast<const Bytes16*>(p);
    return u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
}
__device__ __forceinline__ void store16(void* p, u32x4 v) {
    *static_cast<Bytes16*>(p) = Bytes16{{v[0], v[1], v[2], v[3]}};
}
__device__ __forceinline__ f32x4 load4(const float* p) { return __builtin_bit_cast(f32x4, load16(p)); }
__device__ __forceinline__ void store4(float* p, f32x4 v) { store16(p, __builtin_bit_cast(u32x4, v)); }

// ------------------------------------------------------------- operands ---
// Rows of an operand are what the output's rows (or columns) are; the sum runs
// along k.  Element (row, k) at ptr[row * ld + k] (along) or ptr[k * ld + row] (across).
struct Operand {
    const void* ptr;
    long long ld;
};

// m x n sums over k, in `slices` of `stages` stages.
struct Product {
    static constexpr bool kDynamic = false;
    // Whether long float32 sums are added up in parts of kPart stages, 512 terms, for sums whose
    // absolute error is what counts: gradients of the loss of 17 rows of 2518 and 657 tokens are off by
    // 2e-7, by 8e-7 without.  1 to 4% of a product's time (3000 x 1024 over 20000 tokens 980 us, 943).
    static constexpr bool kParts = false;
    int m, n, k;
    Operand a, b;       // m rows, n rows
    int slices, stages; // stages of a slice
    __device__ __forceinline__ int live_rows() const { return m; }
    __device__ __forceinline__ int depth() const { return k; }
};

constexpr int kRowBytes = 128;  // of a stage's row
constexpr int kPart = 16;

// The parts of a wavefront's sums.
template <bool ON, int MB, int NB>
struct Parts {
    f32x16 total[MB][NB] = {};
    // (sums are read and set in another block than their products: states between, settle())
    __device__ __forceinline__ void end_part(f32x16 (&acc)[MB][NB]);
    __device__ __forceinline__ void end(f32x16 (&acc)[MB][NB]) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] += total[i][j];
    }
};
template <int MB, int NB>
struct Parts<false, MB, NB> {
    __device__ __forceinline__ void end_part(f32x16 (&)[MB][NB]) {}
    __device__ __forceinline__ void end(f32x16 (&)[MB][NB]) {}
};

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

template <bool ON, int MB, int NB>
__device__ __forceinline__ void Parts<ON, MB, NB>::end_part(f32x16 (&acc)[MB][NB]) {
    settle();
    end(acc);
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            total[i][j] = acc[i][j];
            acc[i][j] = f32x16{};
        }
    settle();
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

// Of a wavefront's sums on their way out: 32 rows, padded.
template <int WN>
constexpr int kOutBytes = 32 * (WN + 4) * 4;
// BM x BN tiles, WM x WN of them per wavefront: through registers, for operands that are
// turned on their way and for rows of any address and length.  Bound by its waits: the
// registers that hold the next stage leave those of one k step's fragments, so that
// LDS's latency shows between the products.  8192 x 2048 over 2048 bf16, one operand
// turned: 87 us, 790 TFLOP/s; direct_kernel: 69 us.  (Two wavefronts to a SIMD where parts are
// held too: with one to a SIMD the 128 tile takes 38% longer.)
template <typename T, int BM, int BN, int WM, int WN, bool A_ACROSS, bool B_ACROSS, typename P>
__global__ __launch_bounds__(BM / WM * BN / WN * 64, P::kParts && sizeof(T) == 4 ? 2 : 1) void tile_kernel(P p) {
    constexpr int NT = BM / WM * BN / WN * 64, kK = 8 * kVec<T>, MB = WM / 32, NB = WN / 32;
    constexpr int kStage = (BM + BN) * kRowBytes;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, i32 = lane % 32, hi = lane / 32;
    int tm, tn, slice;
    tile_of((p.m - 1) / BM + 1, (p.n - 1) / BN + 1, p.slices, &tm, &tn, &slice);
    const int m0 = tm * BM, n0 = tn * BN, wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
    if (P::kDynamic && m0 >= p.live_rows()) return;
    const int depth = p.depth(), kbeg = min(depth, slice * p.stages * kK), kend = min(depth, kbeg + p.stages * kK);
    Stage<T, BM, NT, A_ACROSS> sa;
    Stage<T, BN, NT, B_ACROSS> sb;
    f32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x16{};
    constexpr bool kInParts = P::kParts && sizeof(T) == 4;
    Parts<kInParts, MB, NB> parts;
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
        if (kInParts && (s + 1) % kPart == 0) parts.end_part(acc);
    }
    settle();
    parts.end(acc);
    p.template put<T, WM, WN>(acc, reinterpret_cast<float*>(lds + wave * kOutBytes<WN>), m0 + wm, n0 + wn, slice);
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
// wavefront, with one wavefront to a SIMD, 565.  Loads issued between the products of a quarter
// of a stage, the next stage's fragments read in its last quarter, as written-out instructions that
// the compiler does not wait for: 473 beside 470 in one run, 545 at 128 x 128.  A good part is power: the
// same product of zeros takes 377 (a library's 255, and 355 of random numbers).
template <typename T, int BM, int BN, int WM, int WN, typename P>
__global__ __launch_bounds__(BM / WM * BN / WN * 64) void direct_kernel(P p) {
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
    if (P::kDynamic && m0 >= p.live_rows()) return;
    const int depth = p.depth(), kbeg = min(depth, slice * p.stages * kK), kend = min(depth, kbeg + p.stages * kK);
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
    constexpr bool kInParts = P::kParts && sizeof(T) == 4;
    Parts<kInParts, MB, NB> parts;
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
    // (a slice may lie behind the sum's end where only the GPU knows that)
    if (!P::kDynamic || stages > 0) {
        load(even, 0, 0, kLoads);
        arrive();
        int s = 0;
        for (; s + 2 < stages; s += 2) {
            compute(even, odd, s + 1);
            arrive();
            compute(odd, even, s + 2);
            arrive();
            if (kInParts && (s + 2) % kPart == 0) parts.end_part(acc);
        }
        if (s + 1 < stages) load(odd, s + 1, 0, kLoads);
        compute(even, nullptr, 0);
        settle();
        arrive();
        if (s + 1 < stages) {
            compute(odd, nullptr, 0);
            settle();
        }
    }
    parts.end(acc);
    __syncthreads();
    float* out = reinterpret_cast<float*>((wave < W / 2 ? even : odd) + wave % (W / 2) * kOutBytes<WN>);
    p.template put<T, WM, WN>(acc, out, m0 + wm, n0 + wn, slice);
}

// ------------------------------------------------------------- choices ---
enum Tile { TILE_256, TILE_128, TILE_64 };
constexpr long long kLaunchThreads = 1LL << 32;  // a launch has fewer
constexpr double kNoPlan = 1e30;
struct Plan {
    Tile tile;
    int slices, stages;
    double cost;  // kNoPlan: every tile would take more threads than a launch may have
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
inline Plan plan_product(int m, int n, int k, int esize, bool across, int most_slices = 64) {
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
    Plan best{TILE_64, 1, all, kNoPlan};
    for (const Cost& c : costs) {
        if (esize == 4 && c.tile == TILE_256) continue;
        const double tiles = (double)((m - 1) / c.edge + 1) * ((n - 1) / c.edge + 1);
        for (int want = 1; want <= most_slices && want <= all; want *= 2) {
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
// Whether a sum is whole stages, which direct_kernel takes.
inline bool whole_stages(int k, int esize) { return k % (kRowBytes / esize) == 0; }

template <int N>
using Int = std::integral_constant<int, N>;

// A launch of the kernel that a product's tile and operands ask for.  A, B: whether an
// operand's rows lie across the sum.
template <bool DIRECT, typename T, bool A, bool B, typename P>
int launch_form(const P& p, Tile tile, const char* what, hipStream_t s) {
    auto go = [&](auto kernel, int edge, int wm, int wn) {
        const int threads = edge / wm * edge / wn * 64;
        const long long blocks = (long long)((p.m - 1) / edge + 1) * ((p.n - 1) / edge + 1) * p.slices;
        if (blocks * threads >= kLaunchThreads) return fail(RKA_ERR_UNSUPPORTED_SHAPE, std::string(what) + ": more workgroups than a launch may have");
        const size_t lds = DIRECT ? 0 : std::max<size_t>((size_t)4 * edge * kRowBytes, (size_t)threads / 64 * 32 * (wn + 4) * 4);
        if (lds > (64 << 10))
            RKA_RETURN_IF_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, s, p);
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    };
    const auto kernel = [](auto bm, auto wm, auto wn) {
        constexpr int BM = decltype(bm)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
        if constexpr (DIRECT)
            return &direct_kernel<T, BM, BM, WM, WN, P>;
        else
            return &tile_kernel<T, BM, BM, WM, WN, A, B, P>;
    };
    if constexpr (sizeof(T) == 2)
        if (tile == TILE_256) return go(kernel(Int<256>{}, Int<128>{}, Int<64>{}), 256, 128, 64);
    if (tile == TILE_128) return go(kernel(Int<128>{}, Int<64>{}, Int<64>{}), 128, 64, 64);
    return go(kernel(Int<64>{}, Int<32>{}, Int<32>{}), 64, 32, 32);
}
// Whole stages and operands on 16 bytes, both along the sum.
template <typename T, typename P>
int launch_direct(const P& p, Tile tile, const char* what, hipStream_t s) {
    return launch_form<true, T, false, false>(p, tile, what, s);
}
template <typename T, bool A, bool B, typename P>
int launch(const P& p, Tile tile, const char* what, hipStream_t s) {
    if constexpr (!A && !B) {
        const auto on16 = [](const Operand& o) { return (reinterpret_cast<uintptr_t>(o.ptr) | (size_t)o.ld * sizeof(T)) % 16 == 0; };
        if (whole_stages(p.k, sizeof(T)) && on16(p.a) && on16(p.b)) return launch_direct<T>(p, tile, what, s);
    }
    return launch_form<false, T, A, B>(p, tile, what, s);
}

}  // namespace tiles
}  // namespace rka
