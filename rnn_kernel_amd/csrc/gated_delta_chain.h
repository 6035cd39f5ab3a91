// The gated delta rule's chains over chunks, forward and backward (gated_delta.h has
// the formulas), instantiated per element type and direction in the
// gated_delta_chain_*.hip files.
//
// A workgroup of four wavefronts takes NC blocks of 16 columns of one head's state
// through all chunks.  A step has three products that wait for one another: K S, T X
// and K^T (..) E.  Each wavefront makes a quarter of the rows of each (16 tokens, 16
// tokens, a quarter of Dk), with its own rows of K, Q, T, P and K^T straight from memory
// into its operand registers, each loaded again for the next chunk as soon as it has
// been used, so a load has most of a step to arrive; what the products hand on
// (S, X, E, each split into bf16 pieces by the wavefront that made it) passes through LDS
// in operand order, one barrier apiece.
//
// Bound by the latency of that chain: per chunk some 50 matrix instructions of 16
// clocks per wavefront and column block, three LDS round trips, three barriers.
#pragma once

#include <algorithm>

#include "gated_delta.h"

namespace rka {
namespace delta {
namespace {

constexpr int kChainThreads = 256;

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

// KU: 32-wide steps over Dk (even).
template <typename T, int KU, int NC>
__global__ __launch_bounds__(kChainThreads, 1) void chain_forward_kernel(Dims d, const T* v, const float* s0,
                                                                         const int* lengths, ChunkData in, T* o,
                                                                         float* state_out, float* states, float* e_out) {
    constexpr int NP = kPieces<T>, TW = KU / 2;  // blocks of 16 rows of the state per wavefront
    constexpr int PO = NP == 1 ? 2 : 3;          // pieces for what only reaches o: bf16 keeps 8 bits, two pieces 16
    __shared__ u32x4 fs[NC][KU * 3 * kFragLanes], fx[NC][2 * 3 * kFragLanes], fe[NC][2 * PO * kFragLanes],
        fw[NC][2 * 3 * kFragLanes];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), n = lane % 16, hi = lane / 16;
    const int nblk = (d.Dv - 1) / (16 * NC) + 1;
    const int bh = blockIdx.x / nblk, b = bh / d.Hv, h = bh % d.Hv, hk = h / (d.Hv / d.Hk);
    const int col0 = blockIdx.x % nblk * 16 * NC + n;
    const int len = row_length(lengths, b, d.T);
    const size_t head = (size_t)bh * d.Dk * d.Dv;
    const int live_chunks = (len + kChunk - 1) / kChunk;

    f32x4 s[NC][TW];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int t = 0; t < TW; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int dk = (wave * TW + t) * 16 + hi * 4 + r, col = col0 + 16 * c;
                s[c][t][r] = s0 && col < d.Dv && dk < d.Dk ? s0[head + (size_t)dk * d.Dv + col] : 0.f;
            }
            u32x2 p[3];
            split<3>(s[c][t], p);
            put_block(fs[c], 3, wave * TW + t, hi, n, p);
        }

    // the operands' registers and what fills them
    u32x4 kf[KU][NP], qf[KU][NP], tf[2][3], pf[2][PO], ktf[TW][2][NP];
    T vv[NC][4];
    const size_t kch0 = ((size_t)b * d.Hk + hk) * d.chunks, ch0 = (size_t)bh * d.chunks;
    const size_t rows = row_frags<T>(d.Dk) * kFragLanes;
    auto load_rows = [&](int c) {
        const u32x4* pk = in.k + (kch0 + c) * rows + (size_t)wave * KU * NP * kFragLanes + lane;
        const u32x4* pq = in.q + (kch0 + c) * rows + (size_t)wave * KU * NP * kFragLanes + lane;
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                kf[u][i] = pk[(u * NP + i) * kFragLanes];
                qf[u][i] = pq[(u * NP + i) * kFragLanes];
            }
    };
    auto load_v = [&](int c) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                // (clamped, not guarded: a load under a branch is waited for there)
                const int t = min(c * kChunk + 16 * wave + 4 * hi + r, len - 1), col = min(col0 + 16 * j, d.Dv - 1);
                vv[j][r] = v[b * d.v_s[0] + t * d.v_s[1] + h * d.v_s[2] + col];
            }
    };
    auto load_tri = [&](int c) {
        const u32x4* pt = in.t + (ch0 + c) * (size_t)(kTriFrags * 3 * kFragLanes) + lane;
        const u32x4* pp = in.p + (ch0 + c) * (size_t)(kTriFrags * 3 * kFragLanes) + lane;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if (w > wave / 2) break;
#pragma unroll
            for (int i = 0; i < 3; ++i) tf[w][i] = pt[(lower_frag(wave, w) * 3 + i) * kFragLanes];
#pragma unroll
            for (int i = 0; i < PO; ++i) pf[w][i] = pp[(lower_frag(wave, w) * 3 + i) * kFragLanes];
        }
    };
    auto load_kt = [&](int c) {
        const u32x4* p = in.kt + (kch0 + c) * rows + (size_t)wave * TW * 2 * NP * kFragLanes + lane;
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < NP; ++i) ktf[t][w][i] = p[((t * 2 + w) * NP + i) * kFragLanes];
    };
    if (live_chunks > 0) {
        load_rows(0);
        load_v(0);
        load_tri(0);
        load_kt(0);
    }
    for (int c = 0; c < live_chunks; ++c) {
        const int t0 = c * kChunk, next = min(c + 1, live_chunks - 1);
        const float* coef = in.coef + (ch0 + c) * kCoefFloats;
        const f32x4 rk = coef4(coef, RK, wave, hi), rq = coef4(coef, RQ, wave, hi), wk = coef4(coef, WK, wave, hi);
        const float last = coef[NCOEF * kChunk];
        if (states) {
#pragma unroll
            for (int j = 0; j < NC; ++j)
#pragma unroll
                for (int t = 0; t < TW; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int dk = (wave * TW + t) * 16 + hi * 4 + r, col = col0 + 16 * j;
                        if (dk < d.Dk && col < d.Dv) states[((ch0 + c) * d.Dk + dk) * d.Dv + col] = s[j][t][r];
                    }
        }
        __syncthreads();
        f32x4 out[NC];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            f32x4 y[2] = {};
            out[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                u32x4 f[3];
                get_frag(fs[j], u, 3, lane, f);
                y[u % 2] = mul(kf[u], f, y[u % 2]);
                if constexpr (PO == 2) {
                    const u32x4 g[2] = {f[0], f[1]};
                    out[j] = mul(qf[u], g, out[j]);
                } else {
                    out[j] = mul(qf[u], f, out[j]);
                }
            }
            f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                x[r] = t0 + 16 * wave + 4 * hi + r < len && col0 + 16 * j < d.Dv ? to_f32(vv[j][r]) : 0.f;
            x -= rk * (y[0] + y[1]);
            out[j] *= rq;
            u32x2 p[3];
            split<3>(x, p);
            put_block(fx[j], 3, wave, hi, n, p);
        }
        load_rows(next);
        load_v(next);
        __syncthreads();
        f32x4 e[NC];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            f32x4 a[2] = {};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (w > wave / 2) break;
                u32x4 f[3];
                get_frag(fx[j], w, 3, lane, f);
                a[w] = mul(tf[w], f, a[w]);
            }
            e[j] = a[0] + a[1];
            u32x2 pe[PO], pw[3];
            split<PO>(e[j], pe);
            put_block(fe[j], PO, wave, hi, n, pe);
            split<3>(wk * e[j], pw);
            put_block(fw[j], 3, wave, hi, n, pw);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            u32x4 f[2][3];
            get_frag(fw[j], 0, 3, lane, f[0]);
            get_frag(fw[j], 1, 3, lane, f[1]);
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                s[j][t] = mul(ktf[t][0], f[0], s[j][t] * last);
                s[j][t] = mul(ktf[t][1], f[1], s[j][t]);
                u32x2 p[3];
                split<3>(s[j][t], p);
                put_block(fs[j], 3, wave * TW + t, hi, n, p);
            }
        }
        load_kt(next);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (w > wave / 2) break;
                u32x4 f[PO];
                get_frag(fe[j], w, PO, lane, f);
                out[j] = mul(pf[w], f, out[j]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = t0 + 16 * wave + 4 * hi + r, col = col0 + 16 * j;
                if (t < len && col < d.Dv) {
                    const size_t at = (((size_t)b * d.T + t) * d.Hv + h) * d.Dv + col;
                    o[at] = from_f32<T>(out[j][r]);
                    if (e_out) e_out[at] = e[j][r];
                }
            }
        }
        load_tri(next);
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int col = col0 + 16 * j;
        if (col >= d.Dv) continue;
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int dk = (wave * TW + t) * 16 + hi * 4 + r;
                if (dk < d.Dk) state_out[head + (size_t)dk * d.Dv + col] = s[j][t][r];
            }
        for (int t = len + wave * 4 + hi; t < d.T; t += 16)
            o[(((size_t)b * d.T + t) * d.Hv + h) * d.Dv + col] = from_f32<T>(0.f);
    }
}

template <typename T, int KU, int NC>
__global__ __launch_bounds__(kChainThreads, 1) void chain_backward_kernel(Dims d, const T* dout, const float* dstate_out,
                                                                          const int* lengths, ChunkData in, T* dv,
                                                                          float* ds0, BackwardData bd) {
    constexpr int NP = kPieces<T>, TW = KU / 2;
    __shared__ u32x4 fs[NC][KU * 3 * kFragLanes], fx[NC][2 * 3 * kFragLanes], fo[NC][2 * NP * kFragLanes],
        fw[NC][2 * 3 * kFragLanes], fq[NC][2 * 3 * kFragLanes];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), n = lane % 16, hi = lane / 16;
    const int nblk = (d.Dv - 1) / (16 * NC) + 1;
    const int bh = blockIdx.x / nblk, b = bh / d.Hv, h = bh % d.Hv, hk = h / (d.Hv / d.Hk);
    const int col0 = blockIdx.x % nblk * 16 * NC + n;
    const int len = row_length(lengths, b, d.T);
    const size_t head = (size_t)bh * d.Dk * d.Dv;
    const int live_chunks = (len + kChunk - 1) / kChunk;

    f32x4 s[NC][TW];  // dS'
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int t = 0; t < TW; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int dk = (wave * TW + t) * 16 + hi * 4 + r, col = col0 + 16 * c;
                s[c][t][r] = dstate_out && col < d.Dv && dk < d.Dk ? dstate_out[head + (size_t)dk * d.Dv + col] : 0.f;
            }
            u32x2 p[3];
            split<3>(s[c][t], p);
            put_block(fs[c], 3, wave * TW + t, hi, n, p);
        }

    u32x4 kf[KU][NP], tf[2][3], pf[2][3], ktf[TW][2][NP], qtf[TW][2][NP];
    T go[NC][4] = {};  // dO of the wavefront's rows
    const size_t kch0 = ((size_t)b * d.Hk + hk) * d.chunks, ch0 = (size_t)bh * d.chunks;
    const size_t rows = row_frags<T>(d.Dk) * kFragLanes;
    auto load_rows = [&](int c) {
        const u32x4* pk = in.k + (kch0 + c) * rows + (size_t)wave * KU * NP * kFragLanes + lane;
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int i = 0; i < NP; ++i) kf[u][i] = pk[(u * NP + i) * kFragLanes];
    };
    auto load_do = [&](int c) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = min(c * kChunk + 16 * wave + 4 * hi + r, len - 1), col = min(col0 + 16 * j, d.Dv - 1);
                if (dout) go[j][r] = dout[(((size_t)b * d.T + t) * d.Hv + h) * d.Dv + col];
            }
    };
    auto masked_do = [&](int c, int j) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            x[r] = c * kChunk + 16 * wave + 4 * hi + r < len && col0 + 16 * j < d.Dv ? to_f32(go[j][r]) : 0.f;
        return x;
    };
    // (exact in the pieces of its type)
    auto put_do = [&](int c) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            u32x2 p[NP];
            split<NP>(masked_do(c, j), p);
            put_block(fo[j], NP, wave, hi, n, p);
        }
    };
    // the transposes: rows `wave`, steps wave / 2 and up
    auto load_tri = [&](const u32x4* from, int c, u32x4 (&f)[2][3]) {
        const u32x4* p = from + (ch0 + c) * (size_t)(kTriFrags * 3 * kFragLanes) + lane;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if (w < wave / 2) continue;
#pragma unroll
            for (int i = 0; i < 3; ++i) f[w][i] = p[(upper_frag(wave, w) * 3 + i) * kFragLanes];
        }
    };
    auto load_transposed = [&](int c) {
        const u32x4* pk = in.kt + (kch0 + c) * rows + (size_t)wave * TW * 2 * NP * kFragLanes + lane;
        const u32x4* pq = in.qt + (kch0 + c) * rows + (size_t)wave * TW * 2 * NP * kFragLanes + lane;
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    ktf[t][w][i] = pk[((t * 2 + w) * NP + i) * kFragLanes];
                    qtf[t][w][i] = pq[((t * 2 + w) * NP + i) * kFragLanes];
                }
    };
    if (live_chunks > 0) {
        const int c = live_chunks - 1;
        load_rows(c);
        load_do(c);
        load_tri(in.t, c, tf);
        load_tri(in.p, c, pf);
        load_transposed(c);
        put_do(c);
    }
    for (int c = live_chunks - 1; c >= 0; --c) {
        const int t0 = c * kChunk, next = max(c - 1, 0);
        const float* coef = in.coef + (ch0 + c) * kCoefFloats;
        const f32x4 rk = coef4(coef, RK, wave, hi), rq = coef4(coef, RQ, wave, hi), wk = coef4(coef, WK, wave, hi);
        const float last = coef[NCOEF * kChunk];
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int t = 0; t < TW; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int dk = (wave * TW + t) * 16 + hi * 4 + r, col = col0 + 16 * j;
                    if (dk < d.Dk && col < d.Dv) bd.dstates[((ch0 + c) * d.Dk + dk) * d.Dv + col] = s[j][t][r];
                }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            f32x4 y[2] = {}, u = {};
#pragma unroll
            for (int k = 0; k < KU; ++k) {
                u32x4 f[3];
                get_frag(fs[j], k, 3, lane, f);
                y[k % 2] = mul(kf[k], f, y[k % 2]);
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (w < wave / 2) continue;
                u32x4 f[NP];
                get_frag(fo[j], w, NP, lane, f);
                u = mul(pf[w], f, u);
            }
            u32x2 p[3];
            split<3>(u + wk * (y[0] + y[1]), p);
            put_block(fx[j], 3, wave, hi, n, p);
            split<3>(rq * masked_do(c, j), p);
            put_block(fq[j], 3, wave, hi, n, p);
        }
        load_rows(next);
        load_do(next);
        load_tri(in.p, next, pf);
        __syncthreads();
        f32x4 x[NC];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            f32x4 a[2] = {};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (w < wave / 2) continue;
                u32x4 f[3];
                get_frag(fx[j], w, 3, lane, f);
                a[w] = mul(tf[w], f, a[w]);
            }
            x[j] = a[0] + a[1];
            u32x2 p[3];
            split<3>(-rk * x[j], p);
            put_block(fw[j], 3, wave, hi, n, p);
        }
        load_tri(in.t, next, tf);
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
                s[j][t] *= last;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    s[j][t] = mul(qtf[t][w], g[w], s[j][t]);
                    s[j][t] = mul(ktf[t][w], f[w], s[j][t]);
                }
                u32x2 p[3];
                split<3>(s[j][t], p);
                put_block(fs[j], 3, wave * TW + t, hi, n, p);
            }
        }
        load_transposed(next);
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = t0 + 16 * wave + 4 * hi + r, col = col0 + 16 * j;
                if (t < len && col < d.Dv) {
                    const size_t at = (((size_t)b * d.T + t) * d.Hv + h) * d.Dv + col;
                    dv[at] = from_f32<T>(x[j][r]);
                    bd.dx[at] = x[j][r];
                }
            }
        put_do(next);
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int col = col0 + 16 * j;
        if (col >= d.Dv) continue;
        if (ds0) {
#pragma unroll
            for (int t = 0; t < TW; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int dk = (wave * TW + t) * 16 + hi * 4 + r;
                    if (dk < d.Dk) ds0[head + (size_t)dk * d.Dv + col] = s[j][t][r];
                }
        }
        for (int t = len + wave * 4 + hi; t < d.T; t += 16)
            dv[(((size_t)b * d.T + t) * d.Hv + h) * d.Dv + col] = from_f32<T>(0.f);
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
