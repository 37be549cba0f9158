// mla_attention.hip -- attention over the cached latents, the up-projections
// absorbed into queries and outputs.
#include <hip/hip_runtime.h>

#include "k3x_mla.hpp"

using namespace k3x_dev;
using namespace k3x_ops;
using namespace k3x_mla;

namespace {

constexpr uint32_t kThreads = 256;

struct AttentionArgs {
    Pages pages;
    const void* q;
    const uint8_t* pool;
    void* out;
    float* lse;
    uint32_t H, L, R, F;
    uint64_t qs, os;
    float scale;
    uint32_t* status;
};

template <uint32_t DT>
__device__ inline float cached(const AttentionArgs& a, const uint8_t* row, uint32_t d) {
    typedef typename Elem<DT>::type E;
    if (d >= a.L) return Elem<DT>::load(reinterpret_cast<const E*>(row + a.pages.row.codes)[d - a.L]);
    if (a.F == K3X_CACHE_16BIT) return Elem<DT>::load(reinterpret_cast<const E*>(row)[d]);
    const float s = e8m0_to_f32(row[a.pages.row.scales + d / 32]);
    if (a.F == K3X_CACHE_MXFP8)
        return (float)mxfp8_8(uint2{row[d], 0u}, s)[0];
    return (float)dequant8(row[d / 2] >> (d & 1 ? 4 : 0), s)[0];
}

// A workgroup a token and head: 256 keys at a time.
template <uint32_t DT>
__global__ __launch_bounds__(kThreads) void mla_attention_kernel(AttentionArgs a) {
    typedef typename Elem<DT>::type E;
    __shared__ float q[576], w[kThreads], red[kThreads];
    const uint32_t tid = threadIdx.x, t = blockIdx.x / a.H, h = blockIdx.x % a.H;
    if (*(volatile uint32_t*)a.status) return;
    if (blockIdx.x == 0) check_sequences(a.pages, a.status);
    const uint32_t n = sequence_of(a.pages, t);
    Tokens s;
    if (n >= a.pages.N || !tokens_of(a.pages, n, &s) || t < s.begin || t - s.begin >= s.count)
        return;
    const int64_t p = (int64_t)s.len - s.count + (t - s.begin);
    const uint32_t sees = p < 0 ? 0 : (uint32_t)p + 1;
    const E* qr = static_cast<const E*>(a.q) + t * a.qs + (size_t)h * (a.L + a.R);
    for (uint32_t d = tid; d < a.L + a.R; d += kThreads) q[d] = Elem<DT>::load(qr[d]);
    float m = -3.4e38f, l = 0.0f, o[2] = {0.0f, 0.0f};
    for (uint32_t at = 0; at < sees; at += kThreads) {
        const uint32_t k = at + tid;
        __syncthreads();
        float x = -__builtin_inff();
        if (k < sees) {
            const uint8_t* row = cached_row(a.pages, const_cast<uint8_t*>(a.pool), n, k);
            if (row) {
                x = 0.0f;
                for (uint32_t d = 0; d < a.L + a.R; ++d)
                    x = __builtin_fmaf(q[d], cached<DT>(a, row, d), x);
                x *= a.scale;
            } else {
                latch(a.status, K3X_ERR_INVALID_STATE);
            }
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
        o[0] *= keep;
        o[1] *= keep;
        for (uint32_t i = 0; i < min(kThreads, sees - at); ++i) {
            l += w[i];
            const uint8_t* row = cached_row(a.pages, const_cast<uint8_t*>(a.pool), n, at + i);
            if (!row) continue;
            for (uint32_t j = 0; j < 2; ++j)
                if (tid + j * kThreads < a.L)
                    o[j] = __builtin_fmaf(w[i], cached<DT>(a, row, tid + j * kThreads), o[j]);
        }
    }
    E* out = static_cast<E*>(a.out) + t * a.os + (size_t)h * a.L;
    for (uint32_t j = 0; j < 2; ++j)
        if (tid + j * kThreads < a.L) {
            const float v = sees ? o[j] / l : 0.0f;
            if (!(fabsf(v) < __builtin_inff())) latch(a.status, K3X_ERR_INVALID_MXFP4);
            out[tid + j * kThreads] = Elem<DT>::store(v);
        }
    if (a.lse && tid == 0)
        a.lse[(size_t)t * a.H + h] = sees ? m + logf(l) : -__builtin_inff();
}

}  // namespace

extern "C" {

size_t k3x_hip_mla_attention_workspace(const k3x_hip_mla_params* p) { return 0; }

int k3x_hip_mla_attention(k3x_hip_ctx* ctx, const k3x_hip_mla_params* p, const void* q,
                          const void* pool, const uint32_t* table, const uint32_t* offsets,
                          const uint32_t* lens, void* out, float* lse, void* workspace,
                          size_t workspace_bytes) {
    if (!ctx || !p || !mla_ok(p) || !q || !pool || !table || !lens || !out ||
        p->q_stride % 8 || p->out_stride % 8)
        return K3X_ERR_INVALID_EXTENT;
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(pool, 256) || !aligned(table, 4) ||
        !aligned(offsets, 4) || !aligned(lens, 4) || !aligned(lse, 4))
        return K3X_ERR_INVALID_EXTENT;
    if (hipSetDevice(ctx->device) != hipSuccess) return K3X_ERR_BACKEND_UNAVAILABLE;
    AttentionArgs a{};
    a.pages = pages_of(p, table, offsets, lens);
    a.q = q;
    a.pool = static_cast<const uint8_t*>(pool);
    a.out = out;
    a.lse = lse;
    a.H = p->heads;
    a.L = p->latent;
    a.R = p->rotary;
    a.F = p->cache_format;
    a.qs = p->q_stride ? p->q_stride : (uint64_t)p->heads * (p->latent + p->rotary);
    a.os = p->out_stride ? p->out_stride : (uint64_t)p->heads * p->latent;
    a.scale = p->scale;
    a.status = ctx->status;
    if (!p->tokens) return K3X_OK;
    const dim3 grid(p->tokens * p->heads), block(kThreads);
    if (p->dtype == K3X_DTYPE_F16)
        hipLaunchKernelGGL(mla_attention_kernel<K3X_DTYPE_F16>, grid, block, 0, ctx->stream, a);
    else
        hipLaunchKernelGGL(mla_attention_kernel<K3X_DTYPE_BF16>, grid, block, 0, ctx->stream, a);
    return launched(ctx, 1);
}

}  // extern "C"
