// The gated delta rule's chains over chunks, forward and backward (gated_delta.h has
// the formulas), instantiated per element type and direction in the
// gated_delta_chain_*.hip files.
//
// A workgroup of eight wavefronts takes NC blocks of 16 columns of one head's state
// through all chunks.  A step has two products that wait for one another: that of S
// (or dS') which gives E (or dX), and that which updates the state.  Four wavefronts make
// the first, 16 tokens' rows each; the other four make what the step does not wait for
// (forward: Q S and, a step later, P E and o; backward: the pieces of scale exp(G) dO);
// the second is shared by all eight, a part of Dk's rows each.  The rows of the prepared
// factors come straight from memory into the operand registers of the wavefront that
// uses them, each loaded again for a later chunk as soon as it has been used, one by one
// between the products: a load takes 16 clocks to issue, and a step's hundred in one go
// hold up the wavefronts longer than its products; what the
// products hand on (S, E, each split into bf16 pieces by the wavefront that made it)
// passes through LDS in operand order, one barrier apiece.  The workgroups of a head are
// eight apart, on one XCD, whose L2 then answers all but the first of them.
//
// Bound by the latency of the chain.  bf16, 128x128, one column block to a workgroup,
// 16384 tokens of 16 heads: 481 us, 4400 clocks per chunk, of which the wavefronts that
// make E spend 1500 on its products with the loads between them, 250 on handing it on, 600
// on the state's update and 1300 at the two barriers, where the other four arrive last.
// Without its loads of rows (a copy, with wrong results) the same takes 280 us.
// 64 heads of 2048 tokens with two blocks: 151 us forward and 155 backward.  In float32 the
// operands of a Dk above 128 do not fit the registers: 48 to 236 bytes of a lane are spilled
// to memory in the forward, 236 to 352 in the backward (bf16: 52 in the backward of a Dk
// above 192 with two blocks, else none).
#pragma once

#include <algorithm>

#include "gated_delta.h"

namespace rka {
namespace delta {
namespace {

constexpr int kChainThreads = 512;

template <int N>
__device__ __forceinline__ void get_frag(const u32x4* frags, int step, int stride, int lane, u32x4 (&f)[N]) {
#pragma unroll
    for (int c = 0; c < N; ++c) f[c] = frags[((size_t)step * stride + c) * kFragLanes + lane];
}

// Sums of KU steps for NC column blocks, from the blocks' fragments in LDS (NF pieces of
// them, three apart): the reads run two products ahead, pinned there, as the compiler
// would put each right before its use and wait for it.  `use(u, j, f)` makes a product,
// `done(u)` follows the last of a step.
template <int KU, int NC, int NF, int FRAGS, typename Use, typename Done>
__device__ __forceinline__ void steps_ahead(const u32x4 (&from)[NC][FRAGS], int lane, Use use, Done done) {
    constexpr int kAhead = 2, kAll = KU * NC;
    u32x4 f[kAhead + 1][NF];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (i < kAll) get_frag(from[i % NC], i / NC, 3, lane, f[i % (kAhead + 1)]);
#pragma unroll
    for (int i = 0; i < kAll; ++i) {
        if (i + kAhead < kAll)
            get_frag(from[(i + kAhead) % NC], (i + kAhead) / NC, 3, lane, f[(i + kAhead) % (kAhead + 1)]);
        __builtin_amdgcn_sched_barrier(0);
        use(i / NC, i % NC, f[i % (kAhead + 1)]);
        if (i % NC == NC - 1) done(i / NC);
        __builtin_amdgcn_sched_barrier(0);
    }
}

__device__ __forceinline__ f32x4 coef4(const float* coef, int which, int block, int hi) {
    return *reinterpret_cast<const f32x4*>(coef + which * kChunk + 16 * block + 4 * hi);
}

// Head and column block of a workgroup (grid: 8 x heads per XCD x blocks); false:
// none.
__device__ __forceinline__ bool head_and_block(int heads, int* bh, int* blk) {
    const int xcd = blockIdx.x % 8, i = blockIdx.x / 8, per = (heads + 7) / 8;
    *bh = i % per * 8 + xcd;
    *blk = i / per;
    return *bh < heads;
}

// What both directions share of a workgroup's place.
template <int KU, int NC>
struct Place {
    static constexpr int TW = (2 * KU + 7) / 8;  // blocks of 16 rows of the state per wavefront, at most
    int lane, wave, n, hi, w4, bh, blk, b, h, hk, col0, len, live_chunks;
    bool chain;  // of the wavefronts that the step waits for
    size_t head;
    __device__ __forceinline__ bool init(const Dims& d, const int* lengths) {
        lane = threadIdx.x % 64;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        n = lane % 16;
        hi = lane / 16;
        w4 = wave % 4;
        chain = wave < 4;
        if (!head_and_block(d.B * d.Hv, &bh, &blk)) return false;
        b = bh / d.Hv;
        h = bh % d.Hv;
        hk = h / (d.Hv / d.Hk);
        col0 = blk * 16 * NC + n;
        len = row_length(lengths, b, d.T);
        live_chunks = (len + kChunk - 1) / kChunk;
        head = (size_t)bh * d.Dk * d.Dv;
        return true;
    }
    // The wavefront's block t of the state's rows; whether there is one.
    __device__ __forceinline__ int block(int t) const { return wave + 8 * t; }
    __device__ __forceinline__ bool has(int t) const { return 8 * t + 8 <= 2 * KU || block(t) < 2 * KU; }
    // That block, or the last one in its place (whose result is not used).
    __device__ __forceinline__ int near(int t) const { return min(block(t), 2 * KU - 1); }

    // The state, from and to [Dk][Dv] in memory.
    __device__ __forceinline__ void load_state(const Dims& d, const float* from, f32x4 (&s)[NC][TW]) const {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int t = 0; t < TW; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int dk = block(t) * 16 + hi * 4 + r, col = col0 + 16 * j;
                    s[j][t][r] = from && col < d.Dv && dk < d.Dk ? from[(size_t)dk * d.Dv + col] : 0.f;
                }
    }
    __device__ __forceinline__ void store_state(const Dims& d, float* to, const f32x4 (&s)[NC][TW]) const {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int col = col0 + 16 * j;
            if (col >= d.Dv) continue;
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                if (!has(t)) continue;
                float* p = to + (size_t)(block(t) * 16 + hi * 4) * d.Dv + col;
                if (block(t) * 16 + 16 <= d.Dk) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[(size_t)r * d.Dv] = s[j][t][r];
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (block(t) * 16 + hi * 4 + r < d.Dk) p[(size_t)r * d.Dv] = s[j][t][r];
                }
            }
        }
    }
};

// A lane's four tokens (of the wavefront's 16) x NC columns of chunk c; rows `stride`
// elements apart, `p` at the lane's first token of chunk 0 and its first column.
// Loads past the row's end or the columns take the last ones (a load under a branch
// would be waited for there).
template <typename T, int NC>
__device__ __forceinline__ void load_tokens(const T* p, long long stride, int c, int first, int len, int col0, int Dv,
                                            T (&x)[NC][4]) {
    const T* base = p + (long long)c * kChunk * stride;
    if ((c + 1) * kChunk <= len) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int back = min(0, Dv - 1 - (col0 + 16 * j));
#pragma unroll
            for (int r = 0; r < 4; ++r) x[j][r] = base[r * stride + 16 * j + back];
        }
    } else {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int back = min(0, Dv - 1 - (col0 + 16 * j));
#pragma unroll
            for (int r = 0; r < 4; ++r)
                x[j][r] = base[min(r, len - 1 - c * kChunk - first) * stride + 16 * j + back];
        }
    }
}
// Their stores, of one column.
template <typename T>
__device__ __forceinline__ void store_tokens(T* p, long long stride, int c, int first, int len, f32x4 x) {
    p += (long long)c * kChunk * stride;
    if ((c + 1) * kChunk <= len) {
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r * stride] = from_f32<T>(x[r]);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (c * kChunk + first + r < len) p[r * stride] = from_f32<T>(x[r]);
    }
}
// As float32, zero past the row's end.
template <typename T>
__device__ __forceinline__ f32x4 token_values(const T (&x)[4], int c, int first, int len) {
    f32x4 y{to_f32(x[0]), to_f32(x[1]), to_f32(x[2]), to_f32(x[3])};
    if ((c + 1) * kChunk > len) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (c * kChunk + first + r >= len) y[r] = 0.f;
    }
    return y;
}

// Sets of row registers, which take the chunks in turn: with two, a load has a whole
// step more to arrive.  Where the operands leave room for two.
template <typename T, int KU>
constexpr int kRowSets = kPieces<T> == 1 && KU <= 4 ? 2 : 1;

// KU: 32-wide steps over Dk (even).
template <typename T, int KU, int NC>
__global__ __launch_bounds__(kChainThreads, 1) void chain_forward_kernel(Dims d, const float* s0, const int* lengths,
                                                                         ChunkData in, T* o, float* state_out,
                                                                         float* states, float* e_out) {
    constexpr int NP = kPieces<T>, TW = Place<KU, NC>::TW;
    constexpr int PO = NP == 1 ? 2 : 3;  // pieces for what only reaches o: bf16 keeps 8 bits, two pieces 16
    __shared__ u32x4 fs[NC][KU * 3 * kFragLanes], fe[2][NC][2 * PO * kFragLanes], fw[NC][2 * 3 * kFragLanes];
    Place<KU, NC> at;
    if (!at.init(d, lengths)) return;
    const int lane = at.lane, n = at.n, hi = at.hi, w4 = at.w4, len = at.len, col0 = at.col0;
    const bool chain = at.chain;
    const int first = 16 * w4 + 4 * hi;  // the lane's tokens of a chunk

    f32x4 s[NC][TW];
    auto put_state = [&]() {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                if (!at.has(t)) continue;
                u32x2 p[3];
                split<3>(s[j][t], p);
                put_block(fs[j], 3, at.block(t), hi, n, p);
            }
    };
    at.load_state(d, s0 ? s0 + at.head : nullptr, s);
    put_state();

    // chain: rows of T diag(exp G) K; others: of Q (kPieces<T>) and P
    const size_t kch0 = ((size_t)at.b * d.Hk + at.hk) * d.chunks, ch0 = (size_t)at.bh * d.chunks;
    const size_t rows = row_frags<T>(d.Dk) * kFragLanes, reads = read_frags(d.Dk) * kFragLanes;
    const int blocks = column_blocks(d.Dv), block0 = at.blk * NC, final = at.live_chunks - 1;
    const size_t orow = (size_t)d.Hv * d.Dv;
    constexpr int NS = kRowSets<T, KU>;

    // of K^T, and exp(G_C)
    struct Turned {
        u32x4 frag[TW][2][NP];
        float last;
    };
    auto load_turned = [&](Turned& x, int c) {
        const u32x4* p = in.kt + (kch0 + c) * rows + lane;
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < NP; ++i) x.frag[t][w][i] = p[((at.near(t) * 2 + w) * NP + i) * kFragLanes];
        x.last = in.coef[(ch0 + c) * kCoefFloats + NCOEF * kChunk];
    };
    // the second product, all wavefronts' part of a step
    auto update = [&](Turned& x, int c) {
        u32x4 f[NC][2][3];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            get_frag(fw[j], 0, 3, lane, f[j][0]);
            get_frag(fw[j], 1, 3, lane, f[j][1]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                s[j][t] = mul(x.frag[t][0], f[j][0], s[j][t] * x.last);
                s[j][t] = mul(x.frag[t][1], f[j][1], s[j][t]);
                settle(s[j][t]);
            }
        load_turned(x, min(c + NS, final));
        put_state();
    };

    // The two kinds of wavefront in loops of their own: the compiler waits for what may
    // have been loaded on either side of a branch.
    if (chain) {
        struct Rows {
            u32x4 row[KU][3];  // of T diag(exp G) K
            f32x4 own[NC];     // of T V
            f32x4 wk;
            Turned turned;
        } sets[NS];
        const u32x4* pread = in.read + ch0 * reads + (size_t)w4 * KU * 3 * kFragLanes + lane;
        float* pe = e_out ? e_out + (((size_t)at.b * d.T + first) * d.Hv + at.h) * d.Dv + col0 : nullptr;
        auto load_rows = [&](Rows& x, int c) {
            const u32x4* p = pread + c * reads;
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int i = 0; i < 3; ++i) x.row[u][i] = p[(u * 3 + i) * kFragLanes];
        };
        auto load_rest = [&](Rows& x, int c) {
#pragma unroll
            for (int j = 0; j < NC; ++j)
                x.own[j] = in.own[(((ch0 + c) * blocks + min(block0 + j, blocks - 1)) * 4 + w4) * kFragLanes + lane];
            x.wk = coef4(in.coef + (ch0 + c) * kCoefFloats, WK, w4, hi);
        };
        auto step = [&](Rows& x, int c) {
            if (states) at.store_state(d, states + (ch0 + c) * d.Dk * d.Dv, s);
            __syncthreads();
            const u32x4* p = pread + min(c + NS, final) * reads;
            f32x4 part[NC][2] = {};
            steps_ahead<KU, NC, 3>(
                fs, lane, [&](int u, int j, const u32x4(&f)[3]) { part[j][u % 2] = mul(x.row[u], f, part[j][u % 2]); },
                [&](int u) {
#pragma unroll
                    for (int i = 0; i < 3; ++i) x.row[u][i] = p[(u * 3 + i) * kFragLanes];
                });
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                settle(part[j][0]);
                settle(part[j][1]);
                const f32x4 e = x.own[j] - (part[j][0] + part[j][1]);
                u32x2 pw[3], pp[PO];
                split<3>(x.wk * e, pw);
                put_block(fw[j], 3, w4, hi, n, pw);
                split<PO>(e, pp);
                put_block(fe[c % 2][j], PO, w4, hi, n, pp);
                if (pe && col0 + 16 * j < d.Dv) store_tokens(pe + 16 * j, orow, c, first, len, e);
            }
            load_rest(x, min(c + NS, final));
            __syncthreads();
            update(x.turned, c);
        };
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (final >= 0) {
                load_rows(sets[i], min(i, final));
                load_rest(sets[i], min(i, final));
                load_turned(sets[i].turned, min(i, final));
            }
        for (int c = 0; c <= final; c += NS) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (c + i <= final) step(sets[i], c + i);
        }
    } else {
        struct Rows {
            u32x4 row[KU][NP];  // of Q
            f32x4 rq;
            Turned turned;
        } sets[NS];
        u32x4 tri[2][PO];
        f32x4 out[NC];
        const u32x4* pq = in.q + kch0 * rows + (size_t)w4 * KU * NP * kFragLanes + lane;
        const u32x4* ptri = in.p + ch0 * (kTriFrags * 3 * kFragLanes) + lane;
        T* po = o + (((size_t)at.b * d.T + first) * d.Hv + at.h) * d.Dv + col0;
        auto load = [&](Rows& x, int c) {
            const u32x4* p = pq + c * rows;
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int i = 0; i < NP; ++i) x.row[u][i] = p[(u * NP + i) * kFragLanes];
            x.rq = coef4(in.coef + (ch0 + c) * kCoefFloats, RQ, w4, hi);
        };
        // rows w4 of P; their second step is zero for the first two (and not taken)
        auto load_tri = [&](int c) {
            const u32x4* p = ptri + (size_t)c * (kTriFrags * 3 * kFragLanes);
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < PO; ++i) tri[w][i] = p[(lower_frag(w4, w4 / 2 < w ? 0 : w) * 3 + i) * kFragLanes];
        };
        // P E of chunk c, whose E is in fe[c % 2], and its outputs
        auto finish = [&](int c) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                u32x4 f[2][PO];
                get_frag(fe[c % 2][j], 0, PO, lane, f[0]);
                get_frag(fe[c % 2][j], 1, PO, lane, f[1]);
                __builtin_amdgcn_sched_barrier(0);
                out[j] = mul(tri[0], f[0], out[j]);
                settle(out[j]);
                if (w4 >= 2) {
                    out[j] = mul(tri[1], f[1], out[j]);
                    settle(out[j]);
                }
                if (col0 + 16 * j < d.Dv) store_tokens(po + 16 * j, orow, c, first, len, out[j]);
            }
        };
        auto step = [&](Rows& x, int c) {
            if (states) at.store_state(d, states + (ch0 + c) * d.Dk * d.Dv, s);
            __syncthreads();
            const int then = min(c + NS, final);
            f32x4 part[NC][2] = {}, y[NC];
            steps_ahead<KU, NC, PO>(
                fs, lane, [&](int u, int j, const u32x4(&f)[PO]) { part[j][u % 2] = mul(x.row[u], f, part[j][u % 2]); },
                [&](int u) {
#pragma unroll
                    for (int i = 0; i < NP; ++i) x.row[u][i] = pq[then * rows + (u * NP + i) * kFragLanes];
                });
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                settle(part[j][0]);
                settle(part[j][1]);
                y[j] = x.rq * (part[j][0] + part[j][1]);
            }
            x.rq = coef4(in.coef + (ch0 + then) * kCoefFloats, RQ, w4, hi);
            if (c > 0) finish(c - 1);
            load_tri(c);
#pragma unroll
            for (int j = 0; j < NC; ++j) out[j] = y[j];
            __syncthreads();
            update(x.turned, c);
        };
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (final >= 0) {
                load(sets[i], min(i, final));
                load_turned(sets[i].turned, min(i, final));
            }
        for (int c = 0; c <= final; c += NS) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (c + i <= final) step(sets[i], c + i);
        }
        if (final >= 0) finish(final);
#pragma unroll
        for (int j = 0; j < NC; ++j)
            if (col0 + 16 * j < d.Dv)
                for (int t = len + w4 * 4 + hi; t < d.T; t += 16)
                    o[((size_t)at.b * d.T + t) * orow + (size_t)at.h * d.Dv + col0 + 16 * j] = from_f32<T>(0.f);
    }
    at.store_state(d, state_out + at.head, s);
}

template <typename T, int KU, int NC>
__global__ __launch_bounds__(kChainThreads, 1) void chain_backward_kernel(Dims d, const T* dout, const float* dstate_out,
                                                                          const int* lengths, ChunkData in, T* dv,
                                                                          float* ds0, BackwardData bd) {
    constexpr int NP = kPieces<T>, TW = Place<KU, NC>::TW;
    __shared__ u32x4 fs[NC][KU * 3 * kFragLanes], fw[NC][2 * 3 * kFragLanes], fq[NC][2 * 3 * kFragLanes];
    Place<KU, NC> at;
    if (!at.init(d, lengths)) return;
    const int lane = at.lane, n = at.n, hi = at.hi, w4 = at.w4, len = at.len, col0 = at.col0;
    const bool chain = at.chain;
    const int first = 16 * w4 + 4 * hi;

    f32x4 s[NC][TW];  // dS'
    auto put_state = [&]() {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                if (!at.has(t)) continue;
                u32x2 p[3];
                split<3>(s[j][t], p);
                put_block(fs[j], 3, at.block(t), hi, n, p);
            }
    };
    at.load_state(d, dstate_out ? dstate_out + at.head : nullptr, s);
    put_state();

    const size_t kch0 = ((size_t)at.b * d.Hk + at.hk) * d.chunks, ch0 = (size_t)at.bh * d.chunks;
    const size_t rows = row_frags<T>(d.Dk) * kFragLanes, reads = read_frags(d.Dk) * kFragLanes;
    const int blocks = column_blocks(d.Dv), block0 = at.blk * NC, final = at.live_chunks - 1;
    const size_t token = (((size_t)at.b * d.T + first) * d.Hv + at.h) * d.Dv + col0;
    const size_t orow = (size_t)d.Hv * d.Dv;
    constexpr int NS = kRowSets<T, KU>;

    // of K^T and Q^T, and exp(G_C)
    struct Turned {
        u32x4 kt[TW][2][NP], qt[TW][2][NP];
        float last;
    };
    auto load_turned = [&](Turned& x, int c) {
        const u32x4 *pk = in.kt + (kch0 + c) * rows + lane, *pq = in.qt + (kch0 + c) * rows + lane;
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const int f = ((at.near(t) * 2 + w) * NP + i) * kFragLanes;
                    x.kt[t][w][i] = pk[f];
                    x.qt[t][w][i] = pq[f];
                }
        x.last = in.coef[(ch0 + c) * kCoefFloats + NCOEF * kChunk];
    };
    auto update = [&](Turned& x, int c) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            u32x4 f[2][3], g[2][3];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                get_frag(fq[j], w, 3, lane, g[w]);
                get_frag(fw[j], w, 3, lane, f[w]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                f32x4 other{0.f, 0.f, 0.f, 0.f};
                s[j][t] *= x.last;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    other = mul(x.qt[t][w], g[w], other);
                    s[j][t] = mul(x.kt[t][w], f[w], s[j][t]);
                }
                settle(other);
                settle(s[j][t]);
                s[j][t] += other;
            }
        }
        load_turned(x, max(c - NS, 0));
        put_state();
    };

    // (loops of their own, as in the forward)
    if (chain) {
        struct Rows {
            u32x4 row[KU][3];  // of T^T diag(exp(G_C - G) beta) K
            f32x4 own[NC];     // of (P T)^T dO
            f32x4 rk;
            Turned turned;
        } sets[NS];
        const u32x4* pread = in.read + ch0 * reads + (size_t)w4 * KU * 3 * kFragLanes + lane;
        auto load_rows = [&](Rows& x, int c) {
            const u32x4* p = pread + c * reads;
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int i = 0; i < 3; ++i) x.row[u][i] = p[(u * 3 + i) * kFragLanes];
        };
        auto load_rest = [&](Rows& x, int c) {
#pragma unroll
            for (int j = 0; j < NC; ++j)
                x.own[j] = in.own[(((ch0 + c) * blocks + min(block0 + j, blocks - 1)) * 4 + w4) * kFragLanes + lane];
            x.rk = coef4(in.coef + (ch0 + c) * kCoefFloats, RK, w4, hi);
        };
        auto step = [&](Rows& x, int c) {
            at.store_state(d, bd.dstates + (ch0 + c) * d.Dk * d.Dv, s);
            __syncthreads();
            const u32x4* p = pread + max(c - NS, 0) * reads;
            f32x4 y[NC][2];
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                y[j][0] = x.own[j];
                y[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            steps_ahead<KU, NC, 3>(
                fs, lane, [&](int u, int j, const u32x4(&f)[3]) { y[j][u % 2] = mul(x.row[u], f, y[j][u % 2]); },
                [&](int u) {
#pragma unroll
                    for (int i = 0; i < 3; ++i) x.row[u][i] = p[(u * 3 + i) * kFragLanes];
                });
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                settle(y[j][0]);
                settle(y[j][1]);
                const f32x4 dx = y[j][0] + y[j][1];
                u32x2 pw[3];
                split<3>(-x.rk * dx, pw);
                put_block(fw[j], 3, w4, hi, n, pw);
                if (col0 + 16 * j < d.Dv) {
                    store_tokens(dv + token + 16 * j, orow, c, first, len, dx);
                    store_tokens(bd.dx + token + 16 * j, orow, c, first, len, dx);
                }
            }
            load_rest(x, max(c - NS, 0));
            __syncthreads();
            update(x.turned, c);
        };
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (final >= 0) {
                load_rows(sets[i], max(final - i, 0));
                load_rest(sets[i], max(final - i, 0));
                load_turned(sets[i].turned, max(final - i, 0));
            }
        for (int c = final; c >= 0; c -= NS) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (c - i >= 0) step(sets[i], c - i);
        }
    } else {
        struct Rows {
            T go[NC][4];  // dO
            f32x4 rq;
            Turned turned;
        } sets[NS];
        auto load = [&](Rows& x, int c) {
            if (dout) load_tokens<T, NC>(dout + token, orow, c, first, len, col0, d.Dv, x.go);
            x.rq = coef4(in.coef + (ch0 + c) * kCoefFloats, RQ, w4, hi);
        };
        auto step = [&](Rows& x, int c) {
            at.store_state(d, bd.dstates + (ch0 + c) * d.Dk * d.Dv, s);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                u32x2 p[3];
                split<3>(x.rq * (dout ? token_values(x.go[j], c, first, len) : f32x4{0.f, 0.f, 0.f, 0.f}), p);
                put_block(fq[j], 3, w4, hi, n, p);
            }
            load(x, max(c - NS, 0));
            __syncthreads();
            update(x.turned, c);
        };
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (final >= 0) {
                load(sets[i], max(final - i, 0));
                load_turned(sets[i].turned, max(final - i, 0));
            }
        for (int c = final; c >= 0; c -= NS) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (c - i >= 0) step(sets[i], c - i);
        }
#pragma unroll
        for (int j = 0; j < NC; ++j)
            if (col0 + 16 * j < d.Dv)
                for (int t = len + w4 * 4 + hi; t < d.T; t += 16)
                    dv[((size_t)at.b * d.T + t) * orow + (size_t)at.h * d.Dv + col0 + 16 * j] = from_f32<T>(0.f);
    }
    if (ds0) at.store_state(d, ds0 + at.head, s);
}

// Calls f with the chain's steps over Dk and its column blocks as integral constants.
template <typename T, typename F>
int with_chain(const Dims& d, F f) {
    const bool two = chain_columns(d, kPieces<T>) == 2;
    auto pick = [&](auto ku) {
        if constexpr (kPieces<T> == 1 || decltype(ku)::value < 8)  // (as chain_columns has it)
            if (two) return f(ku, std::integral_constant<int, 2>{});
        return f(ku, std::integral_constant<int, 1>{});
    };
    switch (chain_steps(d.Dk)) {
        case 2: return pick(std::integral_constant<int, 2>{});
        case 4: return pick(std::integral_constant<int, 4>{});
        case 6: return pick(std::integral_constant<int, 6>{});
        default: return pick(std::integral_constant<int, 8>{});
    }
}

}  // namespace
}  // namespace delta
}  // namespace rka
