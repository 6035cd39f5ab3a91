// The cross entropy of a product with a vocabulary, and its gradients, without the logits in
// memory:
//   l = x W^T + b;  loss = log sum exp(l) - l[target]
//   dl = (exp(l - lse) - onehot(target)) scale;  dx = dl W;  dW = dl^T x;  db = sum of dl's rows
// (a scale that all rows share is put in at the end).
//
// Rows without a target are left out before anything is multiplied: the others are numbered
// in their order, and the products' tiles end where those do, which only the GPU knows.
//
// Forward: a tile's logits stay in registers; what leaves is, of each row and 64 (or 32)
// columns, the largest and the sum of the exponentials over it, and the target's logit.
// Backward: the logits are made again for one piece of the vocabulary after another, dl goes to
// memory as it is and turned, and dx and dW are products whose operands all lie along their sums
// (W's piece and x are turned for that).  dx is summed over the pieces in float32.  Four
// products in all, which bound it; logarithms are of base 2 throughout.
//
// 8192 rows, 7373 of them with a target, 2048 inputs, 64000 tokens, bf16: forward 1.7 to 1.8 ms,
// backward 5.6; logits 1.71 ms (1130 TFLOP/s, a library's product of the sizes 1.40), dl 0.52 for
// each of four pieces, dx 0.43, dW 0.44 (1100 to 1150).  What keeps the products from the library's rate is
// in product_tiles.h; of the first three pieces' 0.52, 0.05 are an eighth round of tiles, 35 for 256 CUs.
// 1000 x 1024 over 10007 in float32: 0.19 and 0.53 ms (110 and 117 TFLOP/s); 1 x 1024 over 100000 85 us.
#include "product_tiles.h"

namespace rka {
namespace loss {
namespace {

using namespace tiles;

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMost = 1 << 21;  // rows, inputs, outputs: tiles' offsets are 32-bit
// Bytes of a piece's dl and its turned copy: pieces so large that dx's sums are long and its
// float32 rows pass through memory a few times only.  Training on 8192 rows of 64000 tokens: 7.95, 7.39,
// 7.33 and 7.34 ms with 128, 256, 512 and 1024 MiB.
constexpr size_t kPieceBytes = (size_t)512 << 20;
constexpr int kLeastPiece = 1024;

// What a forward leaves for its backward, by the rows' new numbers except `place`.
struct Rows {
    float* lse;   // log2 of the sum of exp
    int* from;    // old number
    int* target;  // -1: outside the vocabulary
    int* place;   // of an old number its new one, or -1
    int* count;   // of rows with a target
};
size_t rows_bytes(int rows) { return 4 * align_up((size_t)rows * 4, 256) + 256; }
Rows rows_of(void* p, int rows) {
    char* c = static_cast<char*>(p);
    const size_t step = align_up((size_t)rows * 4, 256);
    return Rows{reinterpret_cast<float*>(c), reinterpret_cast<int*>(c + step), reinterpret_cast<int*>(c + 2 * step),
                reinterpret_cast<int*>(c + 3 * step), reinterpret_cast<int*>(c + 4 * step)};
}

// Numbers the rows with a target; one workgroup, 1024 rows at a time.
template <typename I>
__global__ __launch_bounds__(1024) void number_kernel(const I* target, long long ignore, int rows, int outputs, Rows r,
                                                      float* target_logit, float* losses) {
    __shared__ int before[16];
    __shared__ int total;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    int base = 0;
    for (int first = 0; first < rows; first += 1024) {
        const int i = first + tid;
        const long long t = i < rows ? (long long)target[i] : ignore;
        const bool on = t != ignore;
        const unsigned long long votes = __ballot(on);
        if (lane == 0) before[wave] = __popcll(votes);
        __syncthreads();
        if (tid == 0) {
            int sum = 0;
            for (int w = 0; w < 16; ++w) {
                const int n = before[w];
                before[w] = sum;
                sum += n;
            }
            total = sum;
        }
        __syncthreads();
        if (i < rows) {
            const int n = base + before[wave] + __popcll(votes & ((1ULL << lane) - 1));
            r.place[i] = on ? n : -1;
            if (on) {
                r.from[n] = i;
                r.target[n] = t >= 0 && t < outputs ? (int)t : -1;
                target_logit[n] = __builtin_nanf("");  // until its tile comes by
            } else {
                losses[i] = 0.f;
            }
        }
        base += total;
        __syncthreads();
    }
    if (tid == 0) *r.count = base;
}

// The numbered rows of x, padded with zeros to `width`, and rows of zeros behind them to the end
// of the largest tile: their logits are numbers.
template <typename T>
__global__ __launch_bounds__(256) void gather_kernel(const T* x, long long ldx, int inputs, int width, int rows, Rows r, T* out) {
    const int n = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x % 64;
    const int live = *r.count;
    if (n >= min(rows, (live + 255) / 256 * 256)) return;
    const T* p = x + (n < live ? r.from[n] : 0) * ldx;
    for (int k = lane * kVec<T>; k < width; k += 64 * kVec<T>)
        store_piece(out + (size_t)n * width + k, load_piece(p + k, n < live ? inputs - k : 0), kVec<T>);
}

// Rows (numbered ones where `r.from` is set, else `first` on) as columns: out[k][row], zeros
// from the last row to `width`, a multiple of 64.
template <typename T>
__global__ __launch_bounds__(256) void turn_kernel(const T* x, long long ldx, int inputs, int first, int rows, int width, Rows r,
                                                   T* out) {
    constexpr int V = kVec<T>, kPieces = 64 / V;
    __shared__ T tile[64][64 + 2];
    const int live = r.from ? *r.count : rows, row0 = blockIdx.x * 64, k0 = blockIdx.y * 64;
    // (behind the last row only the rest of its 64 is ever read)
    if (row0 >= max(live, 1)) return;
    for (int i = threadIdx.x; i < 64 * kPieces; i += 256) {
        const int row = row0 + i / kPieces, k = k0 + i % kPieces * V;
        Piece<T> p;
        p.u = u32x4{0, 0, 0, 0};
        if (row < live && k < inputs) p = load_piece(x + (long long)(r.from ? r.from[row] : first + row) * ldx + k, inputs - k);
#pragma unroll
        for (int j = 0; j < V; ++j) tile[i / kPieces][i % kPieces * V + j] = p.e[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * kPieces; i += 256) {
        const int k = i / kPieces, row = i % kPieces * V;
        if (k0 + k >= inputs) break;
        Piece<T> p;
#pragma unroll
        for (int j = 0; j < V; ++j) p.e[j] = tile[row + j][k];
        store_piece(out + (size_t)(k0 + k) * width + row0 + row, p, V);
    }
}

// ------------------------------------------------------------- products ---
// Column of a lane's sum acc[..][j][4 r + e] in its wavefront's.
__device__ __forceinline__ int column(int j, int r, int e) { return 32 * j + 8 * r + 4 * (threadIdx.x % 64 / 32) + e; }

// Logits of a wavefront's columns from the sums: the bias, and -infinity past the last column.
template <typename T, int NB>
struct Bias {
    float b[NB][16];
    __device__ __forceinline__ void load(const void* bias, int col0, int n) {
        const T* p = static_cast<const T*>(bias);
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const int col = col0 + column(j, x / 4, x % 4);
                b[j][x] = col >= n ? -INFINITY : p ? to_f32(p[col]) : 0.f;
            }
    }
};

struct Logits : Product {
    static constexpr bool kParts = true;  // (an exponential's relative error is its logit's absolute one)
    static constexpr bool kDynamic = true;
    Rows r;
    const void* bias;
    float2* stats;  // [blocks of columns][m]: log2 of the largest exp, and the sum over it
    float* target_logit;
    __device__ __forceinline__ int live_rows() const { return *r.count; }

    template <typename T, int WM, int WN>
    __device__ __forceinline__ void put(const f32x16 (&acc)[WM / 32][WN / 32], float*, int row0, int col0, int) const {
        if (col0 >= n) return;
        if (!bias && col0 + WN <= n)
            of_tile<true, T, WM, WN>(acc, row0, col0);
        else
            of_tile<false, T, WM, WN>(acc, row0, col0);
    }
    // PLAIN: no bias, and every column is the vocabulary's.
    template <bool PLAIN, typename T, int WM, int WN>
    __device__ __forceinline__ void of_tile(const f32x16 (&acc)[WM / 32][WN / 32], int row0, int col0) const {
        constexpr int MB = WM / 32, NB = WN / 32;
        const int live = live_rows(), i32 = threadIdx.x % 32;
        Bias<T, NB> b;
        if (!PLAIN) b.load(bias, col0, n);
        int target[MB];  // (at once, ahead of what it is needed for)
#pragma unroll
        for (int i = 0; i < MB; ++i) target[i] = r.target[min(row0 + 32 * i + i32, live - 1)];
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const int row = row0 + 32 * i + i32;
            float l[NB][16], top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    // (a sum past the last column is another column's again: finite or not, it is not one;
                    // a masked column's, whose bias is -infinity, is: NaN stays)
                    l[j][x] = PLAIN ? acc[i][j][x] : col0 + column(j, x / 4, x % 4) >= n ? -INFINITY : acc[i][j][x] + b.b[j][x];
                    top = fmaxf(top, l[j][x]);  // (NaN comes back in the sum)
                }
            top *= kLog2e;
            const float base = top == -INFINITY ? 0.f : top;  // (of nothing but -infinity, or NaN, the sum is 0, or NaN)
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int x = 0; x < 16; ++x) sum += __builtin_amdgcn_exp2f(fmaf(l[j][x], kLog2e, -base));
            // the row's other half of columns
            const float other = __shfl_xor(top, 32), both = fmaxf(top, other);
            sum = top == -INFINITY ? sum : sum * __builtin_amdgcn_exp2f(top - both);
            sum += __shfl_xor(sum, 32);
            if (row >= live) continue;
            if (threadIdx.x % 64 < 32) stats[(size_t)(col0 / WN) * m + row] = float2{both, sum};
            const int t = target[i] - col0;
            if (t >= 0 && t < WN) {
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        if (t == column(j, x / 4, x % 4)) target_logit[row] = l[j][x];
            }
        }
    }
};

// What all rows' gradients are multiplied with, in float32 at the end: in dl it would decide how
// -(1 - p), a row's largest element, is rounded to bf16, in all rows alike (the error of dW over 192
// rows and 1000 tokens, as 2-norms: 0.0027; 0.0018 without).
struct Scale {
    const float* grad;  // null: dl has each row's own
    const int* count;
    int mean;
    __device__ __forceinline__ float of() const {
        if (!grad || *count < 1) return 1.f;
        return mean ? grad[0] / (float)*count : grad[0];
    }
};

// dl for a piece of the vocabulary, from column `first` of it on.
struct Slopes : Product {
    static constexpr bool kParts = true;
    static constexpr bool kDynamic = true;
    Rows r;
    const void* bias;
    const float* grad;  // of each row's loss by old numbers, or null
    int first;
    void *dl, *turned;       // [m][ld], [n][ldt]; zeros from n to ld and from the last row to a multiple of 64
    long long ld, ldt;
    float* sums;             // [m / WM][n] column sums, or null
    __device__ __forceinline__ int live_rows() const { return *r.count; }

    template <typename T, int WM, int WN>
    __device__ __forceinline__ void put(const f32x16 (&acc)[WM / 32][WN / 32], float* out, int row0, int col0, int) const {
        if (row0 >= ldt || col0 >= ld) return;
        if (!bias && col0 + WN <= n && row0 + WM <= live_rows())
            of_tile<true, T, WM, WN>(acc, out, row0, col0);
        else
            of_tile<false, T, WM, WN>(acc, out, row0, col0);
    }
    // PLAIN: no bias, every column is the vocabulary's, and every row one of the call's (dl behind
    // the last is a 0 for dW: the exponential of a logit of no row is not always one).
    template <bool PLAIN, typename T, int WM, int WN>
    __device__ __forceinline__ void of_tile(const f32x16 (&acc)[WM / 32][WN / 32], float* out, int row0, int col0) const {
        constexpr int MB = WM / 32, NB = WN / 32, kLd = WN + 4, kV = kVec<T>, kLanes = WN / kV, kRows = 64 / kLanes;
        const int live = live_rows(), lane = threadIdx.x % 64, i32 = lane % 32;
        Bias<T, NB> b;
        if (!PLAIN) b.load(bias, col0, n);
        float total[kV] = {}, scales[MB], lses[MB];
        int targets[MB];
        // (ahead of all that goes through LDS: their latency is waited for once)
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const int row = row0 + 32 * i + i32, at = min(row, live - 1);
            targets[i] = r.target[at];
            lses[i] = r.lse[at];
            scales[i] = grad ? grad[r.from[at]] : 1.f;
        }
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const int row = row0 + 32 * i + i32, t = targets[i] - first - col0;
            float scale = scales[i];
            if (targets[i] < 0 && row < live) scale = __builtin_nanf("");
            const float lse = lses[i];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float l = PLAIN ? acc[i][j][4 * q + e] : acc[i][j][4 * q + e] + b.b[j][4 * q + e];
                        v[e] = __builtin_amdgcn_exp2f(fmaf(l, kLog2e, -lse)) * scale;
                        if (!PLAIN && (row >= live || col0 + column(j, q, e) >= n)) v[e] = 0.f;
                    }
                    *reinterpret_cast<f32x4*>(out + i32 * kLd + column(j, q, 0)) = v;
                }
            __builtin_amdgcn_wave_barrier();
            if (row < live && t >= 0 && t < WN && lane < 32) out[i32 * kLd + t] -= scale;
            __builtin_amdgcn_wave_barrier();
#pragma unroll 2
            for (int x = 0; x < 32 / kRows; ++x) {
                const int y = x * kRows + lane / kLanes, c = lane % kLanes * kV;
                Piece<T> p;
#pragma unroll
                for (int e = 0; e < kV; ++e) {
                    const float v = out[y * kLd + c + e];
                    total[e] += v;
                    p.e[e] = from_f32<T>(v);
                }
                if (row0 + 32 * i + y < live && col0 + c < ld)
                    store16(static_cast<T*>(dl) + (row0 + 32 * i + y) * ld + col0 + c, p.u);
            }
#pragma unroll 2
            for (int z = 0; z < WN * 32 / kV / 64; ++z) {
                // (neighbouring lanes along a column's 32 rows)
                const int x = z * 64 + lane, c = x / (32 / kV), y = x % (32 / kV) * kV;
                Piece<T> p;
#pragma unroll
                for (int e = 0; e < kV; ++e) p.e[e] = from_f32<T>(out[(y + e) * kLd + c]);
                if (col0 + c < n && row0 + 32 * i + y < ldt)
                    store16(static_cast<T*>(turned) + (col0 + c) * ldt + row0 + 32 * i + y, p.u);
            }
        }
        if (!sums) return;
#pragma unroll
        for (int e = 0; e < kV; ++e) {
#pragma unroll
            for (int o = kLanes; o < 64; o *= 2) total[e] += __shfl_xor(total[e], o);
            const int col = col0 + lane * kV + e;
            if (lane < kLanes && col < n) sums[(size_t)(row0 / WM) * n + col] = total[e];
        }
    }
};

// dx and dW.  By their count the rows end (dx), or the sum (dW).
struct Gradient : Product {
    static constexpr bool kDynamic = true;
    const int* count;
    int of_sum;       // the sum ends with the count
    float* partial;   // [slice][m][n], where it is set
    int add;          // to what is there
    void* c;          // [m][n], else, times `scale`
    Scale scale;
    __device__ __forceinline__ int live_rows() const { return of_sum ? m : *count; }
    __device__ __forceinline__ int depth() const { return of_sum ? min(k, (*count + 63) / 64 * 64) : k; }

    template <typename T, int WM, int WN>
    __device__ __forceinline__ void put(const f32x16 (&acc)[WM / 32][WN / 32], float* out, int row0, int col0, int slice) const {
        constexpr int MB = WM / 32, NB = WN / 32, kLd = WN + 4, kV = kVec<T>, kLanes = WN / kV, kRows = 64 / kLanes;
        const int rows = live_rows(), lane = threadIdx.x % 64, i32 = lane % 32;
        const float factor = partial ? 1.f : scale.of();
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<f32x4*>(out + i32 * kLd + column(j, q, 0)) =
                        f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            __builtin_amdgcn_wave_barrier();
#pragma unroll 2
            for (int x = 0; x < 32 / kRows; ++x) {
                const int y = x * kRows + lane / kLanes, at = lane % kLanes * kV, row = row0 + 32 * i + y, col = col0 + at;
                if (row >= rows || col >= n) continue;
                const int left = min(kV, n - col);
                const float* from = out + y * kLd + at;
                if (partial) {
                    float* to = partial + ((size_t)slice * m + row) * n + col;
#pragma unroll
                    for (int e = 0; e < kV; e += 4) {
                        f32x4 v = *reinterpret_cast<const f32x4*>(from + e);
                        if (e + 4 <= left) {
                            if (add) v += load4(to + e);
                            store4(to + e, v);
                        } else {
#pragma unroll
                            for (int y4 = 0; y4 < 4; ++y4)
                                if (e + y4 < left) to[e + y4] = add ? to[e + y4] + v[y4] : v[y4];
                        }
                    }
                } else {
                    Piece<T> p;
#pragma unroll
                    for (int e = 0; e < kV; ++e) p.e[e] = from_f32<T>(from[e] * factor);
                    store_piece(static_cast<T*>(c) + (size_t)row * n + col, p, left);
                }
            }
        }
    }
};

// ------------------------------------------------------- rows and sums ---
// log2 sum exp and loss of each numbered row, over the blocks of columns in their order: 32
// rows and eight ranges of blocks to a workgroup.
__global__ __launch_bounds__(256) void rows_kernel(const float2* stats, int blocks, int rows, Rows r, const float* target_logit,
                                                   float* losses) {
    __shared__ float2 part[8][32];
    const int x = threadIdx.x % 32, p = threadIdx.x / 32, n = blockIdx.x * 32 + x;
    const bool on = n < *r.count;
    float top = -INFINITY, sum = 0.f;
    const auto join = [&](float2 s) {
        const float both = fmaxf(top, s.x);
        // (a part of nothing but -infinity is 0 and has no exponent)
        const float mine = top == -INFINITY ? sum : sum * __builtin_amdgcn_exp2f(top - both);
        const float other = s.x == -INFINITY ? s.y : s.y * __builtin_amdgcn_exp2f(s.x - both);
        top = both;
        sum = mine + other;
    };
    if (on) {
#pragma unroll 8
        for (int b = p; b < blocks; b += 8) join(stats[(size_t)b * rows + n]);
    }
    part[p][x] = float2{top, sum};
    __syncthreads();
    if (p != 0 || !on) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) join(part[k][x]);
    const float lse = top + log2f(sum);
    r.lse[n] = lse;
    losses[r.from[n]] = lse * kLn2 - target_logit[n];
}

// The rows' sum or mean (0 of no rows).
__global__ __launch_bounds__(1024) void total_kernel(const float* losses, int rows, const int* count, int mean, float* loss) {
    __shared__ double part[16];
    double sum = 0.0;
    for (int i = threadIdx.x; i < rows; i += 1024) sum += losses[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int k = 1; k < 16; ++k) sum += part[k];
    *loss = (float)(mean ? sum / max(*count, 1) : sum);
}

// dx by old numbers, over the slices in their order; 0 without a target.
template <typename T>
__global__ __launch_bounds__(256) void scatter_kernel(const float* partial, int slices, int rows, int n, const int* place, Scale scale, T* dx) {
    constexpr int V = kVec<T>;
    const int groups = (n - 1) / V + 1;
    const long long total = (long long)rows * groups;
    const float factor = scale.of();
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long row = i / groups;
        const int col = (int)(i % groups) * V, left = min(V, n - col), from = place ? place[row] : (int)row;
        float sum[V] = {};
        if (from >= 0) {
            const float* p = partial + (size_t)from * n + col;
            for (int s = 0; s < slices; ++s, p += (size_t)rows * n) {
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    if (e + 4 <= left) {
                        const f32x4 q = load4(p + e);
#pragma unroll
                        for (int y = 0; y < 4; ++y) sum[e + y] += q[y];
                    } else {
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            if (e + y < left) sum[e + y] += p[e + y];
                    }
                }
            }
        }
        Piece<T> q;
#pragma unroll
        for (int e = 0; e < V; ++e) q.e[e] = from_f32<T>(from >= 0 ? sum[e] * factor : 0.f);
        store_piece(dx + row * n + col, q, left);
    }
}

// db of a piece over the row blocks in their order.
template <typename T>
__global__ __launch_bounds__(256) void bias_kernel(const float* sums, const int* count, int rows_per_block, int n, Scale scale, T* db) {
    __shared__ float part[8][33];
    const int c = threadIdx.x % 32, p = threadIdx.x / 32, col = blockIdx.x * 32 + c, blocks = (*count + rows_per_block - 1) / rows_per_block;
    float s = 0.f;
    if (col < n)
        for (int b = p; b < blocks; b += 8) s += sums[(size_t)b * n + col];
    part[p][c] = s;
    __syncthreads();
    if (p != 0 || col >= n) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) s += part[k][c];
    db[col] = from_f32<T>(s * scale.of());
}

// -------------------------------------------------------------- choices ---
int up64(int v) { return (v + 63) / 64 * 64; }
// Columns of a wavefront's sums and rows of them.
int columns_of(Tile t) { return t == TILE_64 ? 32 : 64; }
int rows_of(Tile t) { return t == TILE_256 ? 128 : t == TILE_128 ? 64 : 32; }

struct Sizes {
    int m, k, v, esize;
    int width;  // of x's copy
    Tile tile;  // of the logits
};
Sizes sizes_of(int rows, int inputs, int outputs, int dtype) {
    Sizes s{rows, inputs, outputs, dtype == RKA_DTYPE_F32 ? 4 : 2, up64(inputs), TILE_64};
    s.tile = plan_product(rows, outputs, inputs, s.esize, false, 1).tile;
    return s;
}

struct Forward {
    size_t x, stats, target_logit, losses, total;
};
Forward forward_layout(const Sizes& z) {
    Forward l{};
    l.stats = align_up((size_t)z.m * z.width * z.esize, 256);
    l.target_logit = l.stats + align_up((size_t)((z.v - 1) / columns_of(z.tile) + 1) * z.m * sizeof(float2), 256);
    l.losses = l.target_logit + align_up((size_t)z.m * 4, 256);
    l.total = l.losses + align_up((size_t)z.m * 4, 256);
    return l;
}

struct Backward {
    int piece;           // columns of a piece, at most
    Tile tile;           // of its logits
    Plan of_x, of_w;     // plans of dx and dW
    int mp;              // rows, a multiple of 64
    size_t x, turned_x, dl, turned_dl, turned_w, dx, dw, sums, total;
};
Backward backward_layout(const Sizes& z) {
    Backward l{};
    l.mp = up64(z.m);
    const int most = (int)std::min<size_t>(z.v, std::max<size_t>(kLeastPiece, kPieceBytes / (2 * (size_t)z.esize * l.mp) / 256 * 256));
    const int pieces = (z.v - 1) / most + 1;
    l.piece = std::min(z.v, ((z.v - 1) / pieces + 256) / 256 * 256);
    l.tile = plan_product(z.m, l.piece, z.k, z.esize, false, 1).tile;
    l.of_x = plan_product(z.m, z.k, up64(l.piece), z.esize, false);
    l.of_w = plan_product(l.piece, z.k, l.mp, z.esize, false);
    const size_t e = z.esize, wide = up64(l.piece);
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align_up(bytes, 256);
        return here;
    };
    l.x = take(z.m * (size_t)z.width * e);
    l.turned_x = take((size_t)z.k * l.mp * e);
    l.dl = take(z.m * wide * e);
    l.turned_dl = take((size_t)l.piece * l.mp * e);
    l.turned_w = take(z.k * wide * e);
    l.dx = take((size_t)l.of_x.slices * z.m * z.k * 4);
    l.dw = take(l.of_w.slices > 1 ? (size_t)l.of_w.slices * l.piece * z.k * 4 : 0);
    l.sums = take((size_t)((l.mp - 1) / rows_of(l.tile) + 1) * l.piece * 4);
    l.total = at;
    return l;
}

int blocks_of(long long items) { return (int)std::max(1LL, std::min((items + 255) / 256, 4096LL)); }

template <typename T>
int gather(const Sizes& z, const Rows& r, const T* x, long long ldx, T* out, hipStream_t s) {
    hipLaunchKernelGGL((gather_kernel<T>), dim3((z.m - 1) / 4 + 1), dim3(256), 0, s, x, ldx, z.k, z.width, z.m, r, out);
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}

template <typename T>
int forward(const Sizes& z, const T* x, long long ldx, const T* w, long long ldw, const T* bias, const void* target,
            int target64, long long ignore, int reduction, float* loss, void* reserve, char* ws, hipStream_t s) {
    const Forward l = forward_layout(z);
    const Rows r = rows_of(reserve, z.m);
    float *zt = reinterpret_cast<float*>(ws + l.target_logit), *losses = reduction ? reinterpret_cast<float*>(ws + l.losses) : loss;
    float2* stats = reinterpret_cast<float2*>(ws + l.stats);
    T* xc = reinterpret_cast<T*>(ws + l.x);
    if (target64)
        hipLaunchKernelGGL((number_kernel<long long>), dim3(1), dim3(1024), 0, s, static_cast<const long long*>(target), ignore,
                           z.m, z.v, r, zt, losses);
    else
        hipLaunchKernelGGL((number_kernel<int>), dim3(1), dim3(1024), 0, s, static_cast<const int*>(target), ignore, z.m, z.v, r,
                           zt, losses);
    RKA_RETURN_IF_HIP(hipGetLastError());
    RKA_RETURN_IF_ERR(gather(z, r, x, ldx, xc, s));
    const int stages = (z.k * z.esize - 1) / kRowBytes + 1;
    Logits p{{z.m, z.v, z.k, Operand{xc, z.width}, Operand{w, ldw}, 1, stages}, r, bias, stats, zt};
    RKA_RETURN_IF_ERR((launch<T, false, false>(p, z.tile, "cross_entropy", s)));
    hipLaunchKernelGGL(rows_kernel, dim3((z.m - 1) / 32 + 1), dim3(256), 0, s, stats, (z.v - 1) / columns_of(z.tile) + 1, z.m, r, zt,
                       losses);
    RKA_RETURN_IF_HIP(hipGetLastError());
    if (reduction) {
        hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, s, losses, z.m, r.count, reduction == RKA_REDUCE_MEAN ? 1 : 0, loss);
        RKA_RETURN_IF_HIP(hipGetLastError());
    }
    return 0;
}

template <typename T>
int backward(const Sizes& z, const float* grad, const T* x, long long ldx, const T* w, long long ldw, const T* bias,
             int reduction, const void* reserve, T* dx, T* dw, T* db, char* ws, hipStream_t s) {
    const Backward l = backward_layout(z);
    const Rows r = rows_of(const_cast<void*>(reserve), z.m);
    const Rows all{};
    const Scale scale{reduction == RKA_REDUCE_NONE ? nullptr : grad, r.count, reduction == RKA_REDUCE_MEAN};
    T *xc = reinterpret_cast<T*>(ws + l.x), *xt = reinterpret_cast<T*>(ws + l.turned_x), *dl = reinterpret_cast<T*>(ws + l.dl);
    T *dlt = reinterpret_cast<T*>(ws + l.turned_dl), *wt = reinterpret_cast<T*>(ws + l.turned_w);
    float *px = reinterpret_cast<float*>(ws + l.dx), *pw = reinterpret_cast<float*>(ws + l.dw), *sums = reinterpret_cast<float*>(ws + l.sums);
    RKA_RETURN_IF_ERR(gather(z, r, x, ldx, xc, s));
    const unsigned ktiles = (unsigned)((z.k - 1) / 64 + 1);
    if (dw) {
        hipLaunchKernelGGL((turn_kernel<T>), dim3((unsigned)(l.mp / 64), ktiles), dim3(256), 0, s, x, ldx, z.k, 0, z.m, l.mp, r, xt);
        RKA_RETURN_IF_HIP(hipGetLastError());
    }
    const int kk = kRowBytes / z.esize;
    for (int first = 0; first < z.v; first += l.piece) {
        const int n = std::min(l.piece, z.v - first), wide = up64(n);
        const T* wp = w + (long long)first * ldw;
        Slopes q{{z.m, n, z.k, Operand{xc, z.width}, Operand{wp, ldw}, 1, (z.k - 1) / kk + 1}, r, bias ? bias + first : nullptr, scale.grad ? nullptr : grad,
                 first, dl, dlt, wide, l.mp, db ? sums : nullptr};
        RKA_RETURN_IF_ERR((launch<T, false, false>(q, l.tile, "cross_entropy", s)));
        if (db) {
            hipLaunchKernelGGL((bias_kernel<T>), dim3((n - 1) / 32 + 1), dim3(256), 0, s, sums, r.count, rows_of(l.tile), n, scale, db + first);
            RKA_RETURN_IF_HIP(hipGetLastError());
        }
        if (dx) {
            hipLaunchKernelGGL((turn_kernel<T>), dim3((unsigned)(wide / 64), ktiles), dim3(256), 0, s, wp, ldw, z.k, 0, n, wide, all, wt);
            RKA_RETURN_IF_HIP(hipGetLastError());
            const int stages = (wide / kk - 1) / l.of_x.slices + 1;
            Gradient g{{z.m, z.k, wide, Operand{dl, wide}, Operand{wt, wide}, l.of_x.slices, stages}, r.count, 0, px, first > 0, nullptr, scale};
            RKA_RETURN_IF_ERR((launch_direct<T>(g, l.of_x.tile, "cross_entropy", s)));
        }
        if (dw) {
            T* to = dw + (size_t)first * z.k;
            const int slices = l.of_w.slices, stages = (l.mp / kk - 1) / slices + 1;
            Gradient g{{n, z.k, l.mp, Operand{dlt, l.mp}, Operand{xt, l.mp}, slices, stages}, r.count, 1, slices > 1 ? pw : nullptr, 0, to, scale};
            RKA_RETURN_IF_ERR((launch_direct<T>(g, l.of_w.tile, "cross_entropy", s)));
            if (slices > 1) {
                hipLaunchKernelGGL((scatter_kernel<T>), dim3(blocks_of((long long)n * ((z.k - 1) / kVec<T> + 1))), dim3(256), 0, s, pw,
                                   slices, n, z.k, nullptr, scale, to);
                RKA_RETURN_IF_HIP(hipGetLastError());
            }
        }
    }
    if (dx) {
        hipLaunchKernelGGL((scatter_kernel<T>), dim3(blocks_of((long long)z.m * ((z.k - 1) / kVec<T> + 1))), dim3(256), 0, s, px,
                           l.of_x.slices, z.m, z.k, r.place, scale, dx);
        RKA_RETURN_IF_HIP(hipGetLastError());
    }
    return 0;
}

// Whether a launch takes all logits, of the forward, or of the backward's pieces, whose turned
// operands are launches of a thread to 16 elements.
bool launches(const Sizes& z, bool backward) {
    if (!backward) return plan_product(z.m, z.v, z.k, z.esize, false, 1).cost < kNoPlan;
    const Backward l = backward_layout(z);
    for (const int rows : {z.m, l.piece})
        if ((long long)up64(rows) * up64(z.k) / 16 >= kLaunchThreads) return false;
    return plan_product(z.m, l.piece, z.k, z.esize, false, 1).cost < kNoPlan && l.of_x.cost < kNoPlan && l.of_w.cost < kNoPlan;
}
int check_launches(const char* what, const Sizes& z, bool backward) {
    if (launches(z, backward)) return 0;
    return fail(RKA_ERR_UNSUPPORTED_SHAPE, std::string(what) + ": more logits than a launch may have (2^38 or so in float32, 2^39 in bfloat16)");
}

int check(const char* what, int rows, int inputs, int outputs, long long ldx, long long ldw, int reduction, int dtype) {
    const std::string name(what);
    if (rows < 1 || inputs < 1 || outputs < 1) return fail(RKA_ERR_INVALID_ARGUMENT, name + ": sizes must be >= 1");
    if (rows > kMost || inputs > kMost || outputs > kMost || ldw < 0 || ldw > kMost)
        return fail(RKA_ERR_UNSUPPORTED_SHAPE, name + ": rows, inputs, outputs and the weight's row stride must be at most 2^21");
    if (ldx < 0) return fail(RKA_ERR_INVALID_ARGUMENT, name + ": row strides must be >= 0");
    if (reduction != RKA_REDUCE_NONE && reduction != RKA_REDUCE_MEAN && reduction != RKA_REDUCE_SUM)
        return fail(RKA_ERR_INVALID_ARGUMENT, name + ": unknown reduction");
    return check_dtype(dtype, what);
}
bool fits(int rows, int inputs, int outputs, int dtype, bool backward) {
    return rows >= 1 && inputs >= 1 && outputs >= 1 && rows <= kMost && inputs <= kMost && outputs <= kMost &&
           launches(sizes_of(rows, inputs, outputs, dtype), backward);
}

}  // namespace
}  // namespace loss
}  // namespace rka

using namespace rka;
using namespace rka::loss;

extern "C" {

size_t rka_cross_entropy_reserve_bytes(int rows) { return rows < 1 || rows > kMost ? 0 : rows_bytes(rows); }

size_t rka_cross_entropy_forward_workspace_bytes(int rows, int inputs, int outputs, int dtype) {
    return fits(rows, inputs, outputs, dtype, false) ? forward_layout(sizes_of(rows, inputs, outputs, dtype)).total : 0;
}

size_t rka_cross_entropy_backward_workspace_bytes(int rows, int inputs, int outputs, int dtype) {
    return fits(rows, inputs, outputs, dtype, true) ? backward_layout(sizes_of(rows, inputs, outputs, dtype)).total : 0;
}

int rka_describe_cross_entropy(int rows, int inputs, int outputs, int dtype, int aligned, int* out, int n_out) {
    clear_error();
    if (!out || n_out < 1) return fail(RKA_ERR_INVALID_ARGUMENT, "describe_cross_entropy: out must be non-NULL and n_out >= 1");
    RKA_RETURN_IF_ERR(check("describe_cross_entropy", rows, inputs, outputs, 0, 0, RKA_REDUCE_MEAN, dtype));
    const Sizes z = sizes_of(rows, inputs, outputs, dtype);
    const Backward l = backward_layout(z);
    const auto edge = [](Tile t) { return t == TILE_256 ? 256 : t == TILE_128 ? 128 : 64; };
    const int v[9] = {aligned && whole_stages(inputs, z.esize) ? RKA_LINEAR_FORM_DIRECT : RKA_LINEAR_FORM_TILES,
                      edge(z.tile),
                      (outputs - 1) / l.piece + 1,
                      l.piece,
                      edge(l.tile),
                      edge(l.of_x.tile),
                      l.of_x.slices,
                      edge(l.of_w.tile),
                      l.of_w.slices};
    for (int i = 0; i < 9 && i < n_out; ++i) out[i] = v[i];
    return 0;
}

int rka_cross_entropy_forward(const void* x, long long ldx, const void* weight, long long ldw, const void* bias,
                              const void* target, int target_is_64bit, long long ignore_index, float* loss, void* reserve,
                              void* workspace, size_t workspace_bytes, int rows, int inputs, int outputs, int reduction, int dtype,
                              void* stream) {
    clear_error();
    RKA_RETURN_IF_ERR(check("cross_entropy_forward", rows, inputs, outputs, ldx, ldw, reduction, dtype));
    if (!x || !weight || !target || !loss || !reserve) return fail(RKA_ERR_INVALID_ARGUMENT, "cross_entropy_forward: null tensor pointer");
    const Sizes z = sizes_of(rows, inputs, outputs, dtype);
    RKA_RETURN_IF_ERR(check_launches("cross_entropy_forward", z, false));
    RKA_RETURN_IF_ERR(check_workspace(workspace, workspace_bytes, forward_layout(z).total, "cross_entropy_forward"));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    const auto go = [&](auto zero) {
        using T = decltype(zero);
        return forward<T>(z, static_cast<const T*>(x), ldx, static_cast<const T*>(weight), ldw, static_cast<const T*>(bias), target,
                          target_is_64bit, ignore_index, reduction, loss, reserve, ws, s);
    };
    return dtype == RKA_DTYPE_F32 ? go(float{}) : go(bf16{});
}

int rka_cross_entropy_backward(const float* grad_loss, const void* x, long long ldx, const void* weight, long long ldw,
                               const void* bias, const void* reserve, void* grad_x, void* grad_weight, void* grad_bias,
                               void* workspace, size_t workspace_bytes, int rows, int inputs, int outputs, int reduction, int dtype,
                               void* stream) {
    clear_error();
    RKA_RETURN_IF_ERR(check("cross_entropy_backward", rows, inputs, outputs, ldx, ldw, reduction, dtype));
    if (!grad_loss || !x || !weight || !reserve) return fail(RKA_ERR_INVALID_ARGUMENT, "cross_entropy_backward: null tensor pointer");
    const Sizes z = sizes_of(rows, inputs, outputs, dtype);
    RKA_RETURN_IF_ERR(check_launches("cross_entropy_backward", z, true));
    RKA_RETURN_IF_ERR(check_workspace(workspace, workspace_bytes, backward_layout(z).total, "cross_entropy_backward"));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    const auto go = [&](auto zero) {
        using T = decltype(zero);
        return backward<T>(z, grad_loss, static_cast<const T*>(x), ldx, static_cast<const T*>(weight), ldw,
                           static_cast<const T*>(bias), reduction, reserve, static_cast<T*>(grad_x), static_cast<T*>(grad_weight),
                           static_cast<T*>(grad_bias), ws, s);
    };
    return dtype == RKA_DTYPE_F32 ? go(float{}) : go(bf16{});
}

}  // extern "C"
