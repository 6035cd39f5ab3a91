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
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);  // elements of 16 bytes

template <typename T>
union Piece {
    u32x4 u;
    T e[kVec<T>];
};

// ---------------------------------------------------------- activations ---
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case RKA_ACT_RELU: return z < 0.f ? 0.f : z;  // NaN stays
        case RKA_ACT_GELU: return 0.5f * z * erfcf(-0.70710678118654752f * z);
        case RKA_ACT_SILU: return z / (1.f + expf(-z));
        case RKA_ACT_SIGMOID: return 1.f / (1.f + expf(-z));
        case RKA_ACT_LOGSIGMOID: return (z < 0.f ? z : z != z ? z : 0.f) - log1pf(expf(-fabsf(z)));
        default: return z;
    }
}
// dy act'(z)
__device__ __forceinline__ float slope(float dy, float z, int act) {
    switch (act) {
        case RKA_ACT_RELU: return z <= 0.f ? 0.f : dy;
        case RKA_ACT_GELU:
            return dy * (0.5f * erfcf(-0.70710678118654752f * z) + z * 0.3989422804014327f * expf(-0.5f * z * z));
        case RKA_ACT_SILU: {
            const float s = 1.f / (1.f + expf(-z));
            return dy * s * (1.f + z * (1.f / (1.f + expf(z))));
        }
        case RKA_ACT_SIGMOID: return dy * (1.f / (1.f + expf(-z))) * (1.f / (1.f + expf(z)));
        case RKA_ACT_LOGSIGMOID: return dy * (1.f / (1.f + expf(z)));
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
            x = activate(x, p.ep.act);
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
        x = activate(x, p.ep.act);
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

// BM x BN tiles, WM x WN of them per wavefront.
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
    // Through LDS, 32 rows of the wavefront at a time: a lane holds four
    // neighbouring columns of one row, memory wants whole rows.
    constexpr int kLd = WN + 4, kV = kVec<T>, kLanes = WN / kV, kRows = 64 / kLanes;
    float* out = reinterpret_cast<float*>(lds) + wave * 32 * kLd;
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
            const int row = m0 + wm + 32 * i + r, col = n0 + wn + c;
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
#pragma unroll
                for (int e = 0; e < kV; ++e)
                    if (col + e < p.n) part[e] = sum[e];
            } else {
                finish<T, kV>(p, row, col, sum);
            }
        }
    }
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
        for (int s = 0; s < p.slices; ++s, part += (size_t)p.m * p.n) {
#pragma unroll
            for (int e = 0; e < kV; ++e)
                if (col + e < p.n) sum[e] += part[e];
        }
        finish<T, kV>(p, row, col, sum);
    }
}

// Few rows: 16 columns of the output per workgroup, whose wavefronts share the sum.
// The weight goes from memory to the matrix instructions' operands directly, every
// element once.
template <typename T, int MT>
__global__ __launch_bounds__(512) void rows_kernel(Args p) {
    constexpr int kV = kVec<T>, kK = 4 * kV, kWaves = 8, kDeep = 4;
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
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[wave][t][4 * hi + r][i16] = acc[t][r];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 256; i += 512) {
        const int t = i / 256, r = i / 16 % 16, c = i % 16;
        if (16 * t + r >= p.m) continue;
        float sum[1] = {0.f};
#pragma unroll
        for (int k = 0; k < kWaves; ++k) sum[0] += sums[k][t][r][c];
        finish<T, 1>(p, 16 * t + r, n0 + c, sum);
    }
}

// dz = dy act'(z) and the sums of its columns over a range of rows: 8 rows of 32
// threads per workgroup, kVec columns each.
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
                const float g = slope(to_f32(a.e[j]), pb ? to_f32(b.e[j]) : 0.f, act);
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
struct Plan {
    Tile tile;
    int slices, stages;
};

// Tile and slices of a product.
Plan plan_product(int m, int n, int k, int esize) {
    const int kk = kRowBytes / esize, all = std::max(1, (k + kk - 1) / kk);
    Plan best{TILE_64, 1, all};
    double least = 1e30;
    for (const Tile tile : {TILE_256, TILE_128, TILE_64}) {
        const int edge = tile == TILE_256 ? 256 : tile == TILE_128 ? 128 : 64;
        const double per_cu = tile == TILE_256 ? 1 : tile == TILE_128 ? 2 : 4;
        // a stage of as many workgroups as share a CU, in us
        const double stage = (tile == TILE_256 ? 1.25 : tile == TILE_128 ? 0.75 : 0.5) * (esize == 4 ? 8 : 1);
        const double tiles = (double)((m - 1) / edge + 1) * ((n - 1) / edge + 1);
        for (int want = 1; want <= 64 && want <= all; want *= 2) {
            const int stages = (all + want - 1) / want, slices = (all + stages - 1) / stages;
            const double rounds = std::ceil(tiles * slices / (256 * per_cu));
            double cost = rounds * (stages + 3) * stage;
            if (slices > 1) cost += 4 + (double)slices * m * n * 8 / 4e6;
            if (cost < least) {
                least = cost;
                best = Plan{tile, slices, stages};
            }
        }
    }
    return best;
}
size_t partial_bytes(int m, int n, const Plan& p) {
    return p.slices > 1 ? align_up((size_t)p.slices * m * n * sizeof(float), 256) : 0;
}
constexpr int kFewRows = 64;  // up to here the rows' kernel

template <typename T, bool A, bool B>
int launch_tiles(const Args& p, Tile tile, hipStream_t s) {
    auto go = [&](auto kernel, int edge, int wm, int wn) {
        const int threads = edge / wm * edge / wn * 64;
        const long long blocks = (long long)((p.m - 1) / edge + 1) * ((p.n - 1) / edge + 1) * p.slices;
        if (blocks * threads >= (1LL << 32)) return fail(RKA_ERR_UNSUPPORTED_SHAPE, "linear: more workgroups than a launch may have");
        const size_t lds = std::max<size_t>((size_t)4 * edge * kRowBytes, (size_t)threads / 64 * 32 * (wn + 4) * 4);
        RKA_RETURN_IF_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, s, p);
        RKA_RETURN_IF_HIP(hipGetLastError());
        return 0;
    };
    if (tile == TILE_256) {
        RKA_RETURN_IF_ERR(go(&tile_kernel<T, 256, 256, 128, 64, A, B>, 256, 128, 64));
    } else if (tile == TILE_128) {
        RKA_RETURN_IF_ERR(go(&tile_kernel<T, 128, 128, 64, 64, A, B>, 128, 64, 64));
    } else {
        RKA_RETURN_IF_ERR(go(&tile_kernel<T, 64, 64, 32, 32, A, B>, 64, 32, 32));
    }
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
    const Plan plan = plan_product(m, n, k, sizeof(T));
    return launch_tiles<T, A, B>(Args{m, n, k, a, b, c, partial, plan.slices, plan.stages, ep}, plan.tile, s);
}

template <typename T>
int forward(int m, int n, int k, const Operand& x, const Operand& w, void* y, const Epilogue& ep, float* partial,
            hipStream_t s) {
    if (m > kFewRows) return product<T, false, false>(m, n, k, x, w, y, ep, partial, s);
    const Args p{m, n, k, x, w, y, nullptr, 1, 0, ep};
    const dim3 grid((unsigned)((n - 1) / 16 + 1));
    if (m <= 16)
        hipLaunchKernelGGL((rows_kernel<T, 1>), grid, dim3(512), 0, s, p);
    else if (m <= 32)
        hipLaunchKernelGGL((rows_kernel<T, 2>), grid, dim3(512), 0, s, p);
    else
        hipLaunchKernelGGL((rows_kernel<T, 4>), grid, dim3(512), 0, s, p);
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}

// Row ranges of the slope kernel: enough workgroups for the GPU, at least 64 rows each.
int slope_ranges(int m, int n, int esize, int* rows) {
    const int cols = (n - 1) / (32 * (16 / esize)) + 1;
    const int want = std::max(1, 2048 / cols);
    *rows = std::max(64, ((m - 1) / want + 8) / 8 * 8);
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
    l.total = l.partial + std::max(partial_bytes(m, k, plan_product(m, k, n, esize)), partial_bytes(n, k, plan_product(n, k, m, esize)));
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
        if (ld < 0 || ld > kMost) return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": row strides must be at most 2^21 elements");
    return 0;
}

}  // namespace
}  // namespace rka

using namespace rka;

extern "C" {

size_t rka_linear_forward_workspace_bytes(int rows, int outputs, int inputs, int dtype) {
    if (rows < 1 || outputs < 1 || inputs < 1 || rows <= kFewRows) return 0;
    return partial_bytes(rows, outputs, plan_product(rows, outputs, inputs, dtype == RKA_DTYPE_F32 ? 4 : 2));
}

size_t rka_linear_backward_workspace_bytes(int rows, int outputs, int inputs, int dtype) {
    if (rows < 1 || outputs < 1 || inputs < 1) return 0;
    return backward_layout(rows, outputs, inputs, dtype == RKA_DTYPE_F32 ? 4 : 2).total;
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
