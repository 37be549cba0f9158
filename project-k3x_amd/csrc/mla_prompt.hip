// mla_prompt.hip -- attention of prompts over expanded keys and values, with a
// part of the key that all heads share.
#include <hip/hip_runtime.h>

#include "k3x_mla.hpp"

using namespace k3x_dev;
using namespace k3x_ops;

namespace {

constexpr uint32_t kThreads = 256;

struct PromptArgs {
    const void *q, *k, *v, *rotary;
    const uint32_t *offsets, *key_offsets;
    void* out;
    float* lse;
    uint32_t N, T, S, H, Dn, R, Dv, causal;
    uint64_t qs, ks, vs, rs, os, kh, vh;
    float scale;
    uint32_t* status;
};

// Sequence n's queries and keys; false: offsets that are not fit.
struct Ranges {
    uint32_t q, m, k, n;
};
__device__ inline bool ranges_of(const PromptArgs& a, uint32_t n, Ranges* r) {
    uint32_t b, e, f, g;
    if (a.offsets) {
        b = a.offsets[n];
        e = a.offsets[n + 1];
    } else {
        b = n * (a.T / a.N);
        e = b + a.T / a.N;
    }
    if (a.key_offsets) {
        f = a.key_offsets[n];
        g = a.key_offsets[n + 1];
    } else {
        f = n * (a.S / a.N);
        g = f + a.S / a.N;
    }
    *r = Ranges{b, e - b, f, g - f};
    return e >= b && e <= a.T && g >= f && g <= a.S;
}

// A workgroup a query and head: 256 keys at a time.
template <uint32_t DT>
__global__ __launch_bounds__(kThreads) void mla_prompt_kernel(PromptArgs a) {
    typedef typename Elem<DT>::type E;
    __shared__ float q[192], w[kThreads], red[kThreads];
    __shared__ uint32_t owner;
    const uint32_t tid = threadIdx.x, t = blockIdx.x / a.H, h = blockIdx.x % a.H;
    if (*(volatile uint32_t*)a.status) return;
    if (tid == 0) owner = a.N;
    __syncthreads();
    for (uint32_t n = tid; n < a.N; n += kThreads) {
        Ranges r;
        if (!ranges_of(a, n, &r)) latch(a.status, K3X_ERR_INVALID_STATE);
        else if (t >= r.q && t - r.q < r.m) atomicMin(&owner, n);
    }
    __syncthreads();
    if (owner >= a.N) return;
    Ranges s;
    ranges_of(a, owner, &s);
    const int64_t p = a.causal ? (int64_t)s.n - s.m + (t - s.q) + 1 : s.n;
    const uint32_t sees = p < 0 ? 0 : (uint32_t)p;
    const uint32_t D = a.Dn + a.R;
    const E* qr = static_cast<const E*>(a.q) + t * a.qs + (size_t)h * D;
    for (uint32_t d = tid; d < D; d += kThreads) q[d] = Elem<DT>::load(qr[d]);
    float m = -3.4e38f, l = 0.0f, o = 0.0f;
    for (uint32_t at = 0; at < sees; at += kThreads) {
        __syncthreads();
        float x = -__builtin_inff();
        if (at + tid < sees) {
            const size_t row = s.k + at + tid;
            const E* k = static_cast<const E*>(a.k) + row * a.ks + h * a.kh;
            const E* r = static_cast<const E*>(a.rotary) + row * a.rs;
            x = 0.0f;
            for (uint32_t d = 0; d < D; ++d)
                x = __builtin_fmaf(q[d], Elem<DT>::load(d < a.Dn ? k[d] : r[d - a.Dn]), x);
            x *= a.scale;
        }
        red[tid] = x;
        __syncthreads();
        float top = m;
        for (uint32_t i = 0; i < kThreads; ++i) top = fmaxf(top, red[i]);
        w[tid] = expf(x - top);
        __syncthreads();
        const float keep = expf(m - top);
        m = top;
        l *= keep;
        o *= keep;
        for (uint32_t i = 0; i < min(kThreads, sees - at); ++i) {
            l += w[i];
            if (tid < a.Dv)
                o = __builtin_fmaf(w[i], Elem<DT>::load((static_cast<const E*>(a.v) + (size_t)(s.k + at + i) * a.vs + h * a.vh)[tid]), o);
        }
    }
    if (tid < a.Dv) {
        const float v = sees ? o / l : 0.0f;
        if (!(fabsf(v) < __builtin_inff())) latch(a.status, K3X_ERR_INVALID_MXFP4);
        (static_cast<E*>(a.out) + t * a.os + (size_t)h * a.Dv)[tid] = Elem<DT>::store(v);
    }
    if (a.lse && tid == 0)
        a.lse[(size_t)t * a.H + h] = sees ? m + logf(l) : -__builtin_inff();
}

bool prompt_ok(const k3x_hip_mla_prompt_params* p) {
    const uint64_t most = 1ull << 32, H = p->heads, kh = p->k_head_stride, vh = p->v_head_stride;
    auto fits = [&](uint64_t stride, uint64_t least) {
        return !stride || (stride >= least && stride % 8 == 0 && stride <= most);
    };
    return p->sequences && p->sequences <= 65535 && p->tokens <= (1u << 22) &&
           p->keys <= (1u << 22) && p->heads && p->heads <= 1024 && p->key_dim &&
           p->key_dim <= 128 && p->key_dim % 8 == 0 && p->rotary <= 64 && p->rotary % 8 == 0 &&
           p->value_dim && p->value_dim <= 128 && p->value_dim % 8 == 0 &&
           (p->dtype == K3X_DTYPE_BF16 || p->dtype == K3X_DTYPE_F16) && p->causal <= 1 &&
           std::isfinite(p->scale) && p->scale > 0.0f && fits(kh, p->key_dim) &&
           fits(vh, p->value_dim) && fits(p->q_stride, H * (p->key_dim + p->rotary)) &&
           fits(p->k_stride, p->key_dim) && fits(p->v_stride, p->value_dim) &&
           fits(p->rotary_stride, p->rotary) && fits(p->out_stride, H * p->value_dim);
}

}  // namespace

extern "C" {

int k3x_hip_mla_prompt(k3x_hip_ctx* ctx, const k3x_hip_mla_prompt_params* p, const void* q,
                       const void* k, const void* v, const void* rotary, const uint32_t* offsets,
                       const uint32_t* key_offsets, void* out, float* lse) {
    if (!ctx || !p || !prompt_ok(p) || !q || !k || !v || (p->rotary && !rotary) || !out)
        return K3X_ERR_INVALID_EXTENT;
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(rotary, 16) ||
        !aligned(out, 16) || !aligned(offsets, 4) || !aligned(key_offsets, 4) || !aligned(lse, 4))
        return K3X_ERR_INVALID_EXTENT;
    if (hipSetDevice(ctx->device) != hipSuccess) return K3X_ERR_BACKEND_UNAVAILABLE;
    PromptArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.rotary = rotary;
    a.offsets = offsets;
    a.key_offsets = key_offsets;
    a.out = out;
    a.lse = lse;
    a.N = p->sequences;
    a.T = p->tokens;
    a.S = p->keys;
    a.H = p->heads;
    a.Dn = p->key_dim;
    a.R = p->rotary;
    a.Dv = p->value_dim;
    a.causal = p->causal;
    a.kh = p->k_head_stride ? p->k_head_stride : p->key_dim;
    a.vh = p->v_head_stride ? p->v_head_stride : p->value_dim;
    a.qs = p->q_stride ? p->q_stride : (uint64_t)a.H * (a.Dn + a.R);
    a.ks = p->k_stride ? p->k_stride : a.H * a.kh;
    a.vs = p->v_stride ? p->v_stride : a.H * a.vh;
    a.rs = p->rotary_stride ? p->rotary_stride : a.R;
    a.os = p->out_stride ? p->out_stride : (uint64_t)a.H * a.Dv;
    a.scale = p->scale;
    a.status = ctx->status;
    if (!a.T) return K3X_OK;
    const dim3 grid(a.T * a.H), block(kThreads);
    if (p->dtype == K3X_DTYPE_F16)
        hipLaunchKernelGGL(mla_prompt_kernel<K3X_DTYPE_F16>, grid, block, 0, ctx->stream, a);
    else
        hipLaunchKernelGGL(mla_prompt_kernel<K3X_DTYPE_BF16>, grid, block, 0, ctx->stream, a);
    return launched(ctx, 1);
}

}  // extern "C"
