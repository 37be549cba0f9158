// delta.hip -- the gated delta rule (the recurrence of K3's linear attention
// layers) over ragged sequences with their states in HBM.
//
//   S = exp(g) S,  u = beta (v - S^T k),  S = S + k u^T,  o = scale S^T q
//
// for each value head, S [K][V] in fp32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "k3x_ops.hpp"

using namespace k3x_dev;
using namespace k3x_ops;

namespace {

struct DeltaArgs {
    const void *q, *k, *v;
    const float *gate, *beta;
    const uint32_t *offsets, *limits, *slot_index;
    const float* state_in;
    float* state_out;
    void* out;
    uint32_t N, T, Hk, H, K, V;
    uint32_t slots;
    float scale, eps;
    uint64_t qs, ks, vs, os;  // elements from token to token
    uint32_t* status;
};

// Sequence n's rows and state, checked; returns 0 or the status to latch.
struct Sequence {
    uint32_t begin, len;
    uint32_t slot;
};

__device__ inline uint32_t find_sequence(const DeltaArgs& a, uint32_t n, Sequence* s) {
    uint32_t b, e;
    if (a.offsets) {
        b = a.offsets[n];
        e = a.offsets[n + 1];
    } else {
        const uint32_t len = a.T / a.N;
        b = n * len;
        e = b + len;
    }
    s->slot = a.slot_index ? a.slot_index[n] : n;
    if (e < b || e > a.T) return K3X_ERR_INVALID_STATE;
    if ((a.state_in || a.state_out) && s->slot >= a.slots) return K3X_ERR_INVALID_STATE;
    s->begin = b;
    s->len = a.limits ? min(e - b, a.limits[n]) : e - b;
    return 0;
}

// Whether another sequence has sequence n's state (by the whole workgroup).
__device__ inline bool slot_taken(const DeltaArgs& a, uint32_t n, uint32_t slot) {
    if (!a.slot_index || !a.state_out || a.N == 1) return false;
    bool taken = false;
    for (uint32_t m = threadIdx.x; m < a.N; m += blockDim.x)
        taken |= m != n && a.slot_index[m] == slot;
    return __syncthreads_or(taken);
}

// Sum over the lanes that share a lane's column: lanes of equal lane % 4.
__device__ inline float sum_rows(float v) {
#pragma unroll
    for (int d = 4; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// R values from x (element r0 on; those past n are 0) as fp32.  z takes a NaN
// where one of them is not finite.
template <uint32_t DT, int R>
__device__ inline void load_rows(const typename Elem<DT>::type* x, uint32_t r0, uint32_t n,
                                 float (&y)[R], float& z) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
        y[i] = r0 + i < n ? Elem<DT>::load(x[r0 + i]) : 0.0f;
        z = __builtin_fmaf(y[i], 0.0f, z);
    }
}

__device__ inline float exp_decay(float g) {
    return __builtin_amdgcn_exp2f(g * 1.44269504088896341f);
}

// Token by token.  A wave holds 16 columns of one head's state: lane l has
// columns 4 (l % 4) .. + 3 and the R rows from R (l / 4), all in registers.
// The two products over the rows, S^T k and S^T q, are taken of the decayed
// state before its update (S_new^T q = S^T q + (k . q) u), so that a token
// costs one pass over the registers for both, one for the update, and one
// round of sums over the 16 row groups.  A workgroup's waves are neighbours
// in the columns of one head and share nothing else.
constexpr int kStepWaves = 4;
constexpr uint32_t kStepCols = 16 * kStepWaves;

template <uint32_t DT, int R, uint32_t GATE>
__global__ __launch_bounds__(64 * kStepWaves) void delta_step_kernel(DeltaArgs a) {
    typedef typename Elem<DT>::type E;
    const uint32_t blocks = (a.V + kStepCols - 1) / kStepCols;
    const uint32_t cb = blockIdx.x % blocks, h = blockIdx.x / blocks % a.H;
    const uint32_t n = blockIdx.x / blocks / a.H;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sequence sq;
    uint32_t bad = find_sequence(a, n, &sq);
    if (!bad && slot_taken(a, n, sq.slot)) bad = K3X_ERR_INVALID_STATE;
    if (bad) {
        if (threadIdx.x == 0) latch(a.status, bad);
        return;
    }
    // From here on the waves of the workgroup do not wait for one another.
    if (*(volatile uint32_t*)a.status) return;
    const uint32_t c0 = cb * kStepCols + wave * 16 + 4 * (lane % 4), r0 = R * (lane / 4);
    const uint32_t hk = h / (a.H / a.Hk);
    const size_t base = ((size_t)sq.slot * a.H + h) * a.K * a.V;
    float S[R][4];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            S[i][j] = a.state_in && r0 + i < a.K && c0 + j < a.V
                          ? a.state_in[base + (size_t)(r0 + i) * a.V + c0 + j]
                          : 0.0f;
    float z = 0.0f;  // NaN once an input is not finite
    bool wrong = false;
    for (uint32_t t = 0; t < sq.len; ++t) {
        const size_t row = (size_t)sq.begin + t;
        float q[R], k[R], v[4];
        load_rows<DT>(static_cast<const E*>(a.q) + row * a.qs + (size_t)hk * a.K, r0, a.K, q, z);
        load_rows<DT>(static_cast<const E*>(a.k) + row * a.ks + (size_t)hk * a.K, r0, a.K, k, z);
        load_rows<DT>(static_cast<const E*>(a.v) + row * a.vs + (size_t)h * a.V, c0, a.V, v, z);
        const float beta = a.beta[row * a.H + h];
        z = __builtin_fmaf(beta, 0.0f, z);
        float rq = a.scale, rk = 1.0f;
        if (a.eps > 0.0f) {
            float qq = 0.0f, kk = 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                qq = __builtin_fmaf(q[i], q[i], qq);
                kk = __builtin_fmaf(k[i], k[i], kk);
            }
            rq = a.scale / sqrtf(sum_rows(qq) + a.eps);
            rk = 1.0f / sqrtf(sum_rows(kk) + a.eps);
        }
        if (GATE != K3X_GATE_NONE) {
            const float* g = a.gate + (row * a.H + h) * (GATE == K3X_GATE_CHANNEL ? a.K : 1);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const float gi = GATE == K3X_GATE_HEAD ? g[0] : r0 + i < a.K ? g[r0 + i] : 0.0f;
                wrong |= !(gi <= 0.0f);
                const float d = exp_decay(gi);
#pragma unroll
                for (int j = 0; j < 4; ++j) S[i][j] *= d;
            }
        }
        float p[4] = {}, o[4] = {}, kq = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            k[i] *= rk;
            kq = __builtin_fmaf(k[i], q[i], kq);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                p[j] = __builtin_fmaf(S[i][j], k[i], p[j]);
                o[j] = __builtin_fmaf(S[i][j], q[i], o[j]);
            }
        }
        kq = sum_rows(kq);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float u = beta * (v[j] - sum_rows(p[j]));
            o[j] = rq * __builtin_fmaf(kq, u, sum_rows(o[j]));
#pragma unroll
            for (int i = 0; i < R; ++i) S[i][j] = __builtin_fmaf(k[i], u, S[i][j]);
        }
        if (lane < 4) {
            E* out = static_cast<E*>(a.out) + row * a.os + (size_t)h * a.V;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c0 + j < a.V) out[c0 + j] = Elem<DT>::store(o[j]);
        }
    }
    if (wrong || z != z) latch(a.status, K3X_ERR_INVALID_MXFP4);
    if (!a.state_out || (!sq.len && a.state_in == a.state_out)) return;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (r0 + i < a.K && c0 + j < a.V)
                a.state_out[base + (size_t)(r0 + i) * a.V + c0 + j] = S[i][j];
}

template <uint32_t DT, int R>
void launch_step(const DeltaArgs& a, uint32_t gate, uint32_t grid, hipStream_t stream) {
    const dim3 b(64 * kStepWaves);
    if (gate == K3X_GATE_NONE)
        hipLaunchKernelGGL((delta_step_kernel<DT, R, K3X_GATE_NONE>), dim3(grid), b, 0, stream, a);
    else if (gate == K3X_GATE_HEAD)
        hipLaunchKernelGGL((delta_step_kernel<DT, R, K3X_GATE_HEAD>), dim3(grid), b, 0, stream, a);
    else
        hipLaunchKernelGGL((delta_step_kernel<DT, R, K3X_GATE_CHANNEL>), dim3(grid), b, 0, stream,
                           a);
}

template <uint32_t DT>
void launch_step_rows(const DeltaArgs& a, uint32_t gate, uint32_t grid, hipStream_t stream) {
    if (a.K <= 64) launch_step<DT, 4>(a, gate, grid, stream);
    else if (a.K <= 128) launch_step<DT, 8>(a, gate, grid, stream);
    else launch_step<DT, 16>(a, gate, grid, stream);
}

bool delta_ok(const k3x_hip_delta_params* p) {
    if (!p->sequences || p->sequences > 65535 || p->tokens > (1u << 24) || !p->value_heads ||
        p->value_heads > 1024 || !p->key_heads || p->value_heads % p->key_heads || !p->key_dim ||
        p->key_dim > 256 || !p->value_dim || p->value_dim > 1024 || p->dtype > K3X_DTYPE_F16 ||
        p->gate > K3X_GATE_CHANNEL || !std::isfinite(p->scale) ||
        !std::isfinite(p->norm_epsilon) || p->norm_epsilon < 0.0f)
        return false;
    const uint64_t kw = (uint64_t)p->key_heads * p->key_dim;
    const uint64_t vw = (uint64_t)p->value_heads * p->value_dim, most = 1ull << 32;
    return (!p->q_stride || (p->q_stride >= kw && p->q_stride < most)) &&
           (!p->k_stride || (p->k_stride >= kw && p->k_stride < most)) &&
           (!p->v_stride || (p->v_stride >= vw && p->v_stride < most)) &&
           (!p->out_stride || (p->out_stride >= vw && p->out_stride < most)) &&
           (uint64_t)p->sequences * p->value_heads * 16 < (1ull << 31);  // workgroups of a launch
}

}  // namespace

extern "C" {

size_t k3x_hip_delta_workspace(const k3x_hip_delta_params* p) {
    (void)p;
    return 0;
}

int k3x_hip_delta_rule(k3x_hip_ctx* ctx, const k3x_hip_delta_params* p, const void* q,
                       const void* k, const void* v, const float* gate, const float* beta,
                       const uint32_t* offsets, const uint32_t* limits,
                       const uint32_t* slot_index, const float* state_in, float* state_out,
                       void* out, void* workspace, size_t workspace_bytes) {
    if (!ctx || !p || !delta_ok(p)) return K3X_ERR_INVALID_EXTENT;
    const uintptr_t es = p->dtype == K3X_DTYPE_F32 ? 4 : 2;
    if (p->tokens && (!q || !k || !v || !beta || !out)) return K3X_ERR_INVALID_EXTENT;
    if ((p->gate == K3X_GATE_NONE) != !gate && p->tokens) return K3X_ERR_INVALID_EXTENT;
    if (!offsets && p->tokens % p->sequences) return K3X_ERR_INVALID_EXTENT;
    if (!aligned(q, es) || !aligned(k, es) || !aligned(v, es) || !aligned(out, es) ||
        !aligned(gate, 4) || !aligned(beta, 4) || !aligned(offsets, 4) || !aligned(limits, 4) ||
        !aligned(slot_index, 4) || !aligned(state_in, 16) || !aligned(state_out, 16))
        return K3X_ERR_INVALID_EXTENT;
    if ((state_in || state_out) && (!p->slots || (!slot_index && p->slots < p->sequences)))
        return K3X_ERR_INVALID_EXTENT;
    if (state_in && state_out && state_in != state_out) {  // apart, or the same
        const size_t n = (size_t)p->slots * p->value_heads * p->key_dim * p->value_dim;
        const uintptr_t x = reinterpret_cast<uintptr_t>(state_in);
        const uintptr_t y = reinterpret_cast<uintptr_t>(state_out);
        if (x < y + n * 4 && y < x + n * 4) return K3X_ERR_INVALID_EXTENT;
    }
    const size_t need = k3x_hip_delta_workspace(p);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 256)))
        return K3X_ERR_INVALID_EXTENT;
    if (hipSetDevice(ctx->device) != hipSuccess) return K3X_ERR_BACKEND_UNAVAILABLE;
    const uint64_t kw = (uint64_t)p->key_heads * p->key_dim;
    const uint64_t vw = (uint64_t)p->value_heads * p->value_dim;
    DeltaArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.gate = gate;
    a.beta = beta;
    a.offsets = offsets;
    a.limits = limits;
    a.slot_index = slot_index;
    a.state_in = state_in;
    a.state_out = state_out;
    a.out = out;
    a.N = p->sequences;
    a.T = p->tokens;
    a.Hk = p->key_heads;
    a.H = p->value_heads;
    a.K = p->key_dim;
    a.V = p->value_dim;
    a.slots = p->slots;
    a.scale = p->scale;
    a.eps = p->norm_epsilon;
    a.qs = p->q_stride ? p->q_stride : kw;
    a.ks = p->k_stride ? p->k_stride : kw;
    a.vs = p->v_stride ? p->v_stride : vw;
    a.os = p->out_stride ? p->out_stride : vw;
    a.status = ctx->status;
    const uint32_t grid = a.N * a.H * ((a.V + kStepCols - 1) / kStepCols);
    if (p->dtype == K3X_DTYPE_F32)
        launch_step_rows<K3X_DTYPE_F32>(a, p->gate, grid, ctx->stream);
    else if (p->dtype == K3X_DTYPE_BF16)
        launch_step_rows<K3X_DTYPE_BF16>(a, p->gate, grid, ctx->stream);
    else
        launch_step_rows<K3X_DTYPE_F16>(a, p->gate, grid, ctx->stream);
    return launched(ctx, 1);
}

}  // extern "C"
