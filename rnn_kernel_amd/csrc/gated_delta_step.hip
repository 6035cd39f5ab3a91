// The gated delta rule for one token of each of many requests (gated_delta.h has the
// formulas): every state is read and written once, in place.
//
// A workgroup takes a block of columns of one state, in registers; k^T S~ and
// q^T S~ come out of one reduction over the rows, since o = q^T S' needs only
// q^T S~ and q . k besides the error e:  o = scale (q^T S~ + (q . k) beta e).
//
// Bound by memory: 256 requests on 32 heads of 128x128 (1.07 GB) 225 us, 4.8 TB/s, the rate of
// a large copy.  Blocks of 32 columns give one request on 8 heads of 64x64 16 workgroups;
// that call is 13 us, 12 of them the host's.
#include "gated_delta.h"

namespace rka {
namespace delta {
namespace {

constexpr int kThreads = 256;
constexpr int kColThreads = 8;                       // threads of a row, four columns each
constexpr int kCols = 4 * kColThreads;
constexpr int kRowGroups = kThreads / kColThreads;   // rows in flight

// VEC: the state's rows are aligned float4.  kRows: rows of a thread, at most.
template <typename T, bool VEC, int kRows>
__global__ __launch_bounds__(kThreads) void step_kernel(Dims d, const T* q, const T* k, const T* v, const void* g,
                                                        const void* beta, float* state, const int* slots, int num_slots,
                                                        T* o) {
    __shared__ float part[2][4][kCols], ck_q[3][4];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int nblk = (d.Dv - 1) / kCols + 1;
    const int bh = blockIdx.x / nblk, b = bh / d.Hv, h = bh % d.Hv, hk = h / (d.Hv / d.Hk);
    const int col = blockIdx.x % nblk * kCols + tid % kColThreads * 4, row = tid / kColThreads;
    const int slot = slots ? slots[b] : b;
    T* ob = o + ((size_t)b * d.Hv + h) * d.Dv;
    if (slot < 0 || slot >= num_slots) {
        // a request without a state: nothing is read or written but its output
        const float none = slot < 0 ? 0.f : __builtin_nanf("");
        if (tid < kColThreads) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < d.Dv) ob[col + j] = from_f32<T>(none);
        }
        return;
    }
    float* sb = state + ((size_t)slot * d.Hv + h) * d.Dk * d.Dv;
    const T* qb = q + b * d.q_s[0] + hk * d.q_s[2];
    const T* kb = k + b * d.k_s[0] + hk * d.k_s[2];
    // Everything is loaded at once, from clamped addresses: a load under a branch would
    // be waited for there.
    f32x4 s[kRows];
    T kr[kRows], qr[kRows], vr[4];
    const float gate = load_gate(g, b * d.g_s[0] + h * d.g_s[2], d.gate_bf16);
    const float bt = load_gate(beta, b * d.b_s[0] + h * d.b_s[2], d.gate_bf16);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = min(row + i * kRowGroups, d.Dk - 1);
        const float* p = sb + (size_t)r * d.Dv;
        if constexpr (VEC) {
            s[i] = *reinterpret_cast<const f32x4*>(p + min(col, d.Dv - 4));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = p[min(col + j, d.Dv - 1)];
        }
        kr[i] = kb[r];
        qr[i] = qb[r];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) vr[j] = v[b * d.v_s[0] + h * d.v_s[2] + min(col + j, d.Dv - 1)];
    const float decay = expf(floor_gate(gate));
    float kv[kRows], qv[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const bool on = row + i * kRowGroups < d.Dk;
        kv[i] = on ? to_f32(kr[i]) : 0.f;
        qv[i] = on ? to_f32(qr[i]) : 0.f;
        if (!on) s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    f32x4 ak{0.f, 0.f, 0.f, 0.f}, aq{0.f, 0.f, 0.f, 0.f};
    float k2 = 0.f, q2 = 0.f, qk = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        s[i] *= decay;
        ak += kv[i] * s[i];
        aq += qv[i] * s[i];
        k2 += kv[i] * kv[i];
        q2 += qv[i] * qv[i];
        qk += qv[i] * kv[i];
    }
    // over the rows of the wavefront, then over the wavefronts, always in this order
#pragma unroll
    for (int off = kColThreads; off < 64; off *= 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            ak[j] += __shfl_xor(ak[j], off);
            aq[j] += __shfl_xor(aq[j], off);
        }
        k2 += __shfl_xor(k2, off);
        q2 += __shfl_xor(q2, off);
        qk += __shfl_xor(qk, off);
    }
    if (lane < kColThreads) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            part[0][wave][lane * 4 + j] = ak[j];
            part[1][wave][lane * 4 + j] = aq[j];
        }
        if (lane == 0) {
            ck_q[0][wave] = k2;
            ck_q[1][wave] = q2;
            ck_q[2][wave] = qk;
        }
    }
    __syncthreads();
    const float ck = d.normalize ? 1.f / sqrtf(ck_q[0][0] + ck_q[0][1] + ck_q[0][2] + ck_q[0][3] + kNormEps) : 1.f;
    const float cq = d.normalize ? 1.f / sqrtf(ck_q[1][0] + ck_q[1][1] + ck_q[1][2] + ck_q[1][3] + kNormEps) : 1.f;
    qk = (ck_q[2][0] + ck_q[2][1] + ck_q[2][2] + ck_q[2][3]) * ck;
    f32x4 u{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = tid % kColThreads * 4 + j;
        if (col + j >= d.Dv) continue;
        const float ks = part[0][0][c] + part[0][1][c] + part[0][2][c] + part[0][3][c];
        u[j] = bt * (to_f32(vr[j]) - ck * ks);
        if (row == 0) {
            const float qs = part[1][0][c] + part[1][1][c] + part[1][2][c] + part[1][3][c];
            ob[col + j] = from_f32<T>(d.scale * cq * (qs + qk * u[j]));
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = row + i * kRowGroups;
        if (r >= d.Dk) continue;
        s[i] += (ck * kv[i]) * u;
        float* p = sb + (size_t)r * d.Dv + col;
        if constexpr (VEC) {
            if (col < d.Dv) *reinterpret_cast<f32x4*>(p) = s[i];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < d.Dv) p[j] = s[i][j];
        }
    }
}

template <typename T>
int launch_step(const Dims& d, const void* q, const void* k, const void* v, const void* g, const void* beta, float* state,
                const int* slots, int num_slots, void* o, hipStream_t stream) {
    const long long blocks = (long long)d.B * d.Hv * ((d.Dv - 1) / kCols + 1);
    RKA_RETURN_IF_ERR(check_grid(blocks, kThreads, "gated_delta_step"));
    const bool vec = d.Dv % 4 == 0 && (reinterpret_cast<uintptr_t>(state) & 15u) == 0;
    const T *tq = static_cast<const T*>(q), *tk = static_cast<const T*>(k), *tv = static_cast<const T*>(v);
    T* to = static_cast<T*>(o);
    auto go = [&](auto rows) {
        constexpr int R = decltype(rows)::value;
        if (vec)
            hipLaunchKernelGGL((step_kernel<T, true, R>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, d, tq, tk, tv,
                               g, beta, state, slots, num_slots, to);
        else
            hipLaunchKernelGGL((step_kernel<T, false, R>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, d, tq, tk, tv,
                               g, beta, state, slots, num_slots, to);
    };
    if (d.Dk <= kRowGroups)
        go(std::integral_constant<int, 1>{});
    else if (d.Dk <= 2 * kRowGroups)
        go(std::integral_constant<int, 2>{});
    else if (d.Dk <= 4 * kRowGroups)
        go(std::integral_constant<int, 4>{});
    else
        go(std::integral_constant<int, kMaxKeyDim / kRowGroups>{});
    RKA_RETURN_IF_HIP(hipGetLastError());
    return 0;
}

}  // namespace
}  // namespace delta
}  // namespace rka

using namespace rka;
using namespace rka::delta;

extern "C" int rka_gated_delta_step(const void* q, const void* k, const void* v, const void* g, const void* beta,
                                    float* state, const int* slots, int num_slots, void* o, int batch, int key_heads,
                                    int value_heads, int key_dim, int value_dim, const long long* strides, int dtype,
                                    int gate_dtype, int normalize, double scale, void* stream) {
    clear_error();
    Dims d;
    RKA_RETURN_IF_ERR(make_dims("gated_delta_step", batch, 1, key_heads, value_heads, key_dim, value_dim, &d));
    RKA_RETURN_IF_ERR(set_call("gated_delta_step", &d, dtype, gate_dtype, normalize, scale, strides));
    if (num_slots < 0 || (!slots && num_slots < batch))
        return fail(RKA_ERR_INVALID_ARGUMENT, "gated_delta_step: fewer states than requests");
    if (d.B == 0) return 0;
    if (!q || !k || !v || !g || !beta || !state || !o)
        return fail(RKA_ERR_INVALID_ARGUMENT, "gated_delta_step: null tensor pointer");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return dtype == RKA_DTYPE_F32 ? launch_step<float>(d, q, k, v, g, beta, state, slots, num_slots, o, s)
                                  : launch_step<bf16>(d, q, k, v, g, beta, state, slots, num_slots, o, s);
}
