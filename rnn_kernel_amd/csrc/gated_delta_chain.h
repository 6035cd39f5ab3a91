// The gated delta rule's chains over chunks, forward and backward (gated_delta.h has
// the formulas), instantiated per element type and direction in the
// gated_delta_chain_*.hip files.
//
// A workgroup of eight wavefronts takes NC blocks of 16 columns of one head's state
// through all chunks.  A step has three products that wait for one another: K S, T X
// and K^T (..) E.  Four wavefronts make the first two, 16 tokens' rows each; the other
// four make what the step does not wait for (forward: Q S and, a step later, P E and o;
// backward: P^T dO a step ahead, and the pieces of dO); the third is shared by all
// eight, a part of Dk's rows each.  The rows of K, Q, T, P and K^T come straight from
// memory into the operand registers of the wavefront that uses them, each loaded again
// for a later chunk as soon as it has been used; what the products hand on (S, X, E,
// each split into bf16 pieces by the wavefront that made it) passes through LDS in
// operand order, one barrier apiece.  The workgroups of a head are eight apart, on one
// XCD, whose L2 then answers all but the first of them.
//
#pragma once

#include <algorithm>

#include "gated_delta.h"

namespace rka {
namespace delta {
namespace {

constexpr int kChainThreads = 512;

// Where a 16x16 result block goes among the fragments over its rows: block x of 16
// rows, lane (hi, n): eight bytes of step x / 2 at lane (2 (x % 2) + hi / 2, n).
__device__ __forceinline__ void put_block(u32x4* frags, int pieces, int x, int hi, int n, const u32x2* p) {
    u32x2* at = reinterpret_cast<u32x2*>(frags + (size_t)(x / 2) * pieces * kFragLanes) +
                ((2 * (x % 2) + hi / 2) * 16 + n) * 2 + hi % 2;
    for (int c = 0; c < pieces; ++c) at[c * kFragLanes * 2] = p[c];
}

template <int N>
__device__ __forceinline__ void get_frag(const u32x4* frags, int step, int stride, int lane, u32x4 (&f)[N]) {
#pragma unroll
    for (int c = 0; c < N; ++c) f[c] = frags[((size_t)step * stride + c) * kFragLanes + lane];
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
inline long long chain_blocks(const Dims& d, int nc) {
    return (((long long)d.B * d.Hv + 7) / 8) * 8 * ((d.Dv - 1) / (16 * nc) + 1);
}

// What both directions share of a workgroup's place.
template <int KU, int NC>
struct Place {
    static constexpr int TW = (2 * KU + 7) / 8;  // blocks of 16 rows of the state per wavefront, at most
    int lane, wave, n, hi, w4, bh, b, h, hk, col0, len, live_chunks;
    bool chain;  // of the wavefronts that the step waits for
    size_t head;
    __device__ __forceinline__ bool init(const Dims& d, const int* lengths) {
        lane = threadIdx.x % 64;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        n = lane % 16;
        hi = lane / 16;
        w4 = wave % 4;
        chain = wave < 4;
        int blk;
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

// KU: 32-wide steps over Dk (even).
template <typename T, int KU, int NC>
__global__ __launch_bounds__(kChainThreads, 1) void chain_forward_kernel(Dims d, const T* v, const float* s0,
                                                                         const int* lengths, ChunkData in, T* o,
                                                                         float* state_out, float* states, float* e_out) {
    constexpr int NP = kPieces<T>, TW = Place<KU, NC>::TW;
    constexpr int PO = NP == 1 ? 2 : 3;  // pieces for what only reaches o: bf16 keeps 8 bits, two pieces 16
    __shared__ u32x4 fs[NC][KU * 3 * kFragLanes], fx[NC][2 * 3 * kFragLanes], fe[2][NC][2 * PO * kFragLanes],
        fw[NC][2 * 3 * kFragLanes];
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

    // rows: of K and T (chain), of Q and P (others)
    u32x4 row[KU][NP], tri[2][3], turned[TW][2][NP];
    T vv[NC][4];
    f32x4 rc, wk;  // RK (chain) or RQ (others); WK
    float last;
    const size_t kch0 = ((size_t)at.b * d.Hk + at.hk) * d.chunks, ch0 = (size_t)at.bh * d.chunks;
    const size_t rows = row_frags<T>(d.Dk) * kFragLanes;
    const u32x4* prow = (chain ? in.k : in.q) + kch0 * rows + (size_t)w4 * KU * NP * kFragLanes + lane;
    const u32x4* ptri = (chain ? in.t : in.p) + ch0 * (kTriFrags * 3 * kFragLanes) + lane;
    const u32x4* pturned = in.kt + kch0 * rows + lane;
    const T* pv = v + at.b * d.v_s[0] + first * d.v_s[1] + at.h * d.v_s[2] + col0;
    T* po = o + (((size_t)at.b * d.T + first) * d.Hv + at.h) * d.Dv + col0;
    const size_t orow = (size_t)d.Hv * d.Dv;
    auto load_rows = [&](int c) {
        const u32x4* p = prow + c * rows;
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int i = 0; i < NP; ++i) row[u][i] = p[(u * NP + i) * kFragLanes];
    };
    auto load_tri = [&](int c) {
        const u32x4* p = ptri + (size_t)c * (kTriFrags * 3 * kFragLanes);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if (w > w4 / 2) break;
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (PO == 3 || i < 2 || chain) tri[w][i] = p[(lower_frag(w4, w) * 3 + i) * kFragLanes];
        }
    };
    auto load_turned = [&](int c) {
        const u32x4* p = pturned + c * rows;
#pragma unroll
        for (int t = 0; t < TW; ++t) {
            if (!at.has(t)) continue;
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < NP; ++i) turned[t][w][i] = p[((at.block(t) * 2 + w) * NP + i) * kFragLanes];
        }
    };
    auto load_coef = [&](int c) {
        const float* coef = in.coef + (ch0 + c) * kCoefFloats;
        rc = coef4(coef, chain ? RK : RQ, w4, hi);
        if (chain) wk = coef4(coef, WK, w4, hi);
        last = coef[NCOEF * kChunk];
    };
    // P E of chunk c, whose E is in fe[c % 2], and its outputs
    auto finish = [&](int c, f32x4 (&out)[NC]) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (w > w4 / 2) break;
                u32x4 f[PO], a[PO];
                get_frag(fe[c % 2][j], w, PO, lane, f);
#pragma unroll
                for (int i = 0; i < PO; ++i) a[i] = tri[w][i];
                out[j] = mul(a, f, out[j]);
            }
            if (col0 + 16 * j >= d.Dv) continue;
            T* p = po + (size_t)c * kChunk * orow + 16 * j;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if ((c + 1) * kChunk <= len || c * kChunk + first + r < len) p[r * orow] = from_f32<T>(out[j][r]);
        }
    };
    const int final = at.live_chunks - 1;
    if (final >= 0) {
        load_rows(0);
        load_tri(0);
        load_turned(0);
        load_coef(0);
        if (chain) load_tokens<T, NC>(pv, d.v_s[1], 0, first, len, col0, d.Dv, vv);
    }
    f32x4 out[NC];
    for (int c = 0; c <= final; ++c) {
        const int next = min(c + 1, final);
        if (states) at.store_state(d, states + (ch0 + c) * d.Dk * d.Dv, s);
        __syncthreads();
        f32x4 y[NC];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            f32x4 part[2] = {};
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                if (chain || PO == 3) {
                    u32x4 f[3];
                    get_frag(fs[j], u, 3, lane, f);
                    part[u % 2] = mul(row[u], f, part[u % 2]);
                } else {
                    u32x4 f[2];
                    get_frag(fs[j], u, 3, lane, f);
                    part[u % 2] = mul(row[u], f, part[u % 2]);
                }
            }
            y[j] = rc * (part[0] + part[1]);
            if (chain) {
                u32x2 p[3];
                split<3>(token_values(vv[j], c, first, len) - y[j], p);
                put_block(fx[j], 3, w4, hi, n, p);
            }
        }
        load_rows(next);
        if (chain) load_tokens<T, NC>(pv, d.v_s[1], next, first, len, col0, d.Dv, vv);
        __syncthreads();
        if (chain) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                f32x4 a[2] = {};
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (w > w4 / 2) break;
                    u32x4 f[3];
                    get_frag(fx[j], w, 3, lane, f);
                    a[w] = mul(tri[w], f, a[w]);
                }
                const f32x4 e = a[0] + a[1];
                u32x2 pw[3], pe[PO];
                split<3>(wk * e, pw);
                put_block(fw[j], 3, w4, hi, n, pw);
                split<PO>(e, pe);
                put_block(fe[c % 2][j], PO, w4, hi, n, pe);
                if (e_out && col0 + 16 * j < d.Dv) {
                    float* p = e_out + (((size_t)at.b * d.T + c * kChunk + first) * d.Hv + at.h) * d.Dv + col0 + 16 * j;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if ((c + 1) * kChunk <= len || c * kChunk + first + r < len) p[r * orow] = e[r];
                }
            }
            load_tri(next);
        } else if (c > 0) {
            finish(c - 1, out);
            load_tri(c);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            u32x4 f[2][3];
            get_frag(fw[j], 0, 3, lane, f[0]);
            get_frag(fw[j], 1, 3, lane, f[1]);
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                if (!at.has(t)) continue;
                s[j][t] = mul(turned[t][0], f[0], s[j][t] * last);
                s[j][t] = mul(turned[t][1], f[1], s[j][t]);
            }
            out[j] = y[j];
        }
        put_state();
        load_turned(next);
        load_coef(next);
    }
    if (final >= 0 && !chain) finish(final, out);
    at.store_state(d, state_out + at.head, s);
    if (!chain) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
            if (col0 + 16 * j < d.Dv)
                for (int t = len + w4 * 4 + hi; t < d.T; t += 16)
                    o[((size_t)at.b * d.T + t) * orow + (size_t)at.h * d.Dv + col0 + 16 * j] = from_f32<T>(0.f);
    }
}

template <typename T, int KU, int NC>
__global__ __launch_bounds__(kChainThreads, 1) void chain_backward_kernel(Dims d, const T* dout, const float* dstate_out,
                                                                          const int* lengths, ChunkData in, T* dv,
                                                                          float* ds0, BackwardData bd) {
    constexpr int NP = kPieces<T>, TW = Place<KU, NC>::TW;
    __shared__ u32x4 fs[NC][KU * 3 * kFragLanes], fx[NC][2 * 3 * kFragLanes], fo[NC][2 * NP * kFragLanes],
        fw[NC][2 * 3 * kFragLanes], fq[NC][2 * 3 * kFragLanes];
    __shared__ f32x4 pd[NC][4][kFragLanes];  // P^T dO, as its makers hold it
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

    u32x4 row[KU][NP], tri[2][3], kt[TW][2][NP], qt[TW][2][NP];  // row: chain only; tri: T^T (chain), P^T (others)
    T go[NC][4], go1[NC][4];                                      // dO of this chunk and the next (others)
    f32x4 rc, wk;                                                 // RK (chain) or RQ (others); WK
    float last;
    const size_t kch0 = ((size_t)at.b * d.Hk + at.hk) * d.chunks, ch0 = (size_t)at.bh * d.chunks;
    const size_t rows = row_frags<T>(d.Dk) * kFragLanes;
    const u32x4* prow = in.k + kch0 * rows + (size_t)w4 * KU * NP * kFragLanes + lane;
    const u32x4* ptri = (chain ? in.t : in.p) + ch0 * (kTriFrags * 3 * kFragLanes) + lane;
    const size_t token = (((size_t)at.b * d.T + first) * d.Hv + at.h) * d.Dv + col0;
    const size_t orow = (size_t)d.Hv * d.Dv;
    auto load_rows = [&](int c) {
        const u32x4* p = prow + c * rows;
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int i = 0; i < NP; ++i) row[u][i] = p[(u * NP + i) * kFragLanes];
    };
    // rows `w4` of the transposes, steps w4 / 2 and up
    auto load_tri = [&](int c) {
        const u32x4* p = ptri + (size_t)c * (kTriFrags * 3 * kFragLanes);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if (w < w4 / 2) continue;
#pragma unroll
            for (int i = 0; i < 3; ++i) tri[w][i] = p[(upper_frag(w4, w) * 3 + i) * kFragLanes];
        }
    };
    auto load_turned = [&](int c) {
        const u32x4 *pk = in.kt + (kch0 + c) * rows + lane, *pq = in.qt + (kch0 + c) * rows + lane;
#pragma unroll
        for (int t = 0; t < TW; ++t) {
            if (!at.has(t)) continue;
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const int f = ((at.block(t) * 2 + w) * NP + i) * kFragLanes;
                    kt[t][w][i] = pk[f];
                    qt[t][w][i] = pq[f];
                }
        }
    };
    auto load_do = [&](int c, T (&x)[NC][4]) {
        if (dout) load_tokens<T, NC>(dout + token, orow, c, first, len, col0, d.Dv, x);
    };
    // the pieces of dO of chunk c (exact in its type), and those of scale exp(G) dO
    auto put_do = [&](int c, const T (&x)[NC][4]) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            u32x2 p[NP];
            split<NP>(dout ? token_values(x[j], c, first, len) : f32x4{0.f, 0.f, 0.f, 0.f}, p);
            put_block(fo[j], NP, w4, hi, n, p);
        }
    };
    auto put_query = [&](int c) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            u32x2 p[3];
            split<3>(rc * (dout ? token_values(go[j], c, first, len) : f32x4{0.f, 0.f, 0.f, 0.f}), p);
            put_block(fq[j], 3, w4, hi, n, p);
        }
    };
    auto put_pd = [&]() {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            f32x4 u{};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (w < w4 / 2) continue;
                u32x4 f[NP];
                get_frag(fo[j], w, NP, lane, f);
                u = mul(tri[w], f, u);
            }
            pd[j][w4][lane] = u;
        }
    };
    auto load_coef = [&](int c) {
        const float* coef = in.coef + (ch0 + c) * kCoefFloats;
        rc = coef4(coef, chain ? RK : RQ, w4, hi);
        if (chain) wk = coef4(coef, WK, w4, hi);
        last = coef[NCOEF * kChunk];
    };
    const int final = at.live_chunks - 1;
    if (final >= 0) {
        load_coef(final);
        load_turned(final);
        load_tri(final);
        if (chain) {
            load_rows(final);
        } else {
            load_do(final, go);
            load_do(max(final - 1, 0), go1);
            put_do(final, go);
        }
        __syncthreads();
        if (!chain) {
            put_pd();
            load_tri(max(final - 1, 0));
        }
    }
    for (int c = final; c >= 0; --c) {
        const int next = max(c - 1, 0);
        at.store_state(d, bd.dstates + (ch0 + c) * d.Dk * d.Dv, s);
        __syncthreads();
        if (chain) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                f32x4 y[2] = {};
#pragma unroll
                for (int u = 0; u < KU; ++u) {
                    u32x4 f[3];
                    get_frag(fs[j], u, 3, lane, f);
                    y[u % 2] = mul(row[u], f, y[u % 2]);
                }
                u32x2 p[3];
                split<3>(pd[j][w4][lane] + wk * (y[0] + y[1]), p);
                put_block(fx[j], 3, w4, hi, n, p);
            }
            load_rows(next);
        } else {
            put_query(c);
            put_do(next, go1);
#pragma unroll
            for (int j = 0; j < NC; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) go[j][r] = go1[j][r];
            load_do(max(c - 2, 0), go1);
        }
        __syncthreads();
        if (chain) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                f32x4 a[2] = {};
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (w < w4 / 2) continue;
                    u32x4 f[3];
                    get_frag(fx[j], w, 3, lane, f);
                    a[w] = mul(tri[w], f, a[w]);
                }
                const f32x4 x = a[0] + a[1];
                u32x2 p[3];
                split<3>(-rc * x, p);
                put_block(fw[j], 3, w4, hi, n, p);
                if (col0 + 16 * j < d.Dv) {
                    const size_t to = token + (size_t)c * kChunk * orow + 16 * j;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if ((c + 1) * kChunk <= len || c * kChunk + first + r < len) {
                            dv[to + r * orow] = from_f32<T>(x[r]);
                            bd.dx[to + r * orow] = x[r];
                        }
                }
            }
            load_tri(next);
        } else {
            put_pd();
            load_tri(max(c - 2, 0));
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            u32x4 f[2][3], g[2][3];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                get_frag(fq[j], w, 3, lane, g[w]);
                get_frag(fw[j], w, 3, lane, f[w]);
            }
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                if (!at.has(t)) continue;
                s[j][t] *= last;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    s[j][t] = mul(qt[t][w], g[w], s[j][t]);
                    s[j][t] = mul(kt[t][w], f[w], s[j][t]);
                }
            }
        }
        put_state();
        load_turned(next);
        load_coef(next);
    }
    if (ds0) at.store_state(d, ds0 + at.head, s);
    if (!chain) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
            if (col0 + 16 * j < d.Dv)
                for (int t = len + w4 * 4 + hi; t < d.T; t += 16)
                    dv[((size_t)at.b * d.T + t) * orow + (size_t)at.h * d.Dv + col0 + 16 * j] = from_f32<T>(0.f);
    }
}

// Calls f with the chain's steps over Dk and its column blocks as integral constants.
// Two blocks halve what is read of K, Q, T and P per column, one has the shorter
// chain: two once every CU has a workgroup anyway.  (Float32 operands of the largest
// Dk leave no registers for two.)
template <typename T, typename F>
int with_chain(const Dims& d, F f) {
    const bool two = d.Dv > 16 && (long long)d.B * d.Hv * ((d.Dv + 31) / 32) >= 256;
    auto pick = [&](auto ku) {
        if constexpr (kPieces<T> == 1 || decltype(ku)::value < 8)
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
