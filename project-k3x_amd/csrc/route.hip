// route.hip -- routing from given logits: scores, groups, Top-K, weights.
//
// Scores, the sort key and the renormalisation are those of the layer's own
// router (sigmoid_cr, topk_key, sums in slot order), so that both route the
// same logits alike, bit for bit; softmax scores, expert groups and plain
// weights are this operator's own.
#include <hip/hip_runtime.h>

#include <cmath>

#include "k3x_ops.hpp"

using namespace k3x_dev;
using namespace k3x_ops;

namespace {

struct RouteArgs {
    const void* logits;
    const float* bias;
    uint32_t T, E, K;
    uint32_t scoring, renorm;
    float scale;
    uint32_t G, top_groups, group_score;
    uint32_t stride;
    uint32_t* ids;
    float* weights;
    uint32_t* status;
};

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

__device__ inline uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_xor(v, d);
        v = v > o ? v : o;
    }
    return v;
}

// The adjusted score of a sort key (topk_key).
__device__ inline float key_score(uint64_t key) {
    const uint32_t ord = (uint32_t)(key >> 32);
    return __uint_as_float((ord & 0x80000000u) ? (ord & 0x7fffffffu) : ~ord);
}

// Renormalised weight of slot `lane` of K whose scores the lanes hold;
// *err = 0 or the status to latch (the same on every lane).
__device__ inline float route_weight(const RouteArgs& a, float selsc, uint32_t* err) {
    *err = 0;
    if (a.renorm == K3X_RENORM_NONE) return __fmul_rn(selsc, a.scale);
    if (a.renorm == K3X_RENORM_DOUBLE) {
        double den = 0.0;
        for (uint32_t s = 0; s < a.K; ++s)
            den = __dadd_rn(den, (double)__int_as_float(__builtin_amdgcn_readlane(
                                     __float_as_int(selsc), s)));
        if (!__builtin_isfinite(den) || !(den > 0.0))
            *err = a.scoring == K3X_SCORE_SIGMOID ? K3X_ERR_INVALID_EXTENT : K3X_ERR_INVALID_STATE;
        return __fmul_rn((float)__ddiv_rn((double)selsc, den), a.scale);
    }
    float den = 0.0f;
    for (uint32_t s = 0; s < a.K; ++s)
        den = __fadd_rn(den, __int_as_float(__builtin_amdgcn_readlane(__float_as_int(selsc), s)));
    if (!__builtin_isfinite(den) || !(den > 0.0f)) *err = K3X_ERR_INVALID_STATE;
    return __fmul_rn(__fdiv_rn(selsc, den), a.scale);
}

// Whether one expert's values are fit to route by; 0 or the status to latch.
__device__ inline uint32_t route_check(const RouteArgs& a, float logit, float s, float b,
                                       float adj) {
    if (a.renorm == K3X_RENORM_DOUBLE && a.scoring == K3X_SCORE_SIGMOID)
        return __builtin_isfinite(logit) && __builtin_isfinite(b) ? 0 : K3X_ERR_INVALID_EXTENT;
    return __builtin_isfinite(s) && __builtin_isfinite(b) && __builtin_isfinite(adj)
               ? 0
               : K3X_ERR_INVALID_STATE;
}

// Any E: one wave a token, keys and scores in LDS, K passes over the keys.
template <uint32_t DT>
__global__ __launch_bounds__(64) void route_lds_kernel(RouteArgs a) {
    extern __shared__ uint64_t keys[];  // [E], then the scores [E]
    float* sc = reinterpret_cast<float*>(keys + a.E);
    __shared__ uint64_t gkey[64];
    typedef typename Elem<DT>::type T;
    const uint32_t t = blockIdx.x, lane = threadIdx.x, E = a.E;
    if (*(volatile uint32_t*)a.status) return;
    const T* row = static_cast<const T*>(a.logits) + (size_t)t * a.stride;
    double mx = 0.0, den = 1.0;
    if (a.scoring == K3X_SCORE_SOFTMAX) {
        float m = -__builtin_inff();
        bool nan = false;
        for (uint32_t e = lane; e < E; e += 64) {
            const float l = Elem<DT>::load(row[e]);
            nan |= l != l;
            m = fmaxf(m, l);
        }
        for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
        mx = __any(nan) ? (double)__builtin_nanf("") : (double)m;
        den = 0.0;
        for (uint32_t e = lane; e < E; e += 64) den += exp((double)Elem<DT>::load(row[e]) - mx);
        den = wave_sum_f64(den);
    }
    uint32_t bad = 0;
    for (uint32_t e = lane; e < E; e += 64) {
        const float l = Elem<DT>::load(row[e]);
        const float b = a.bias ? a.bias[e] : 0.0f;
        const float s = a.scoring == K3X_SCORE_SOFTMAX ? (float)(exp((double)l - mx) / den)
                                                       : sigmoid_cr(l);
        const float adj = __fadd_rn(s, b);
        bad = max(bad, route_check(a, l, s, b, adj));
        sc[e] = s;
        keys[e] = topk_key(adj, e);
    }
    for (int d = 1; d < 64; d <<= 1) bad = max(bad, (uint32_t)__shfl_xor((int)bad, d));
    if (bad) {
        if (lane == 0) latch(a.status, bad);
        return;
    }
    __syncthreads();
    if (a.G > 1) {
        // Lane g ranks group g; the experts of the groups left out lose their keys.
        const uint32_t n = E / a.G;
        uint64_t gk = 0;
        if (lane < a.G) {
            uint64_t k1 = 0, k2 = 0;
            for (uint32_t i = 0; i < n; ++i) {
                const uint64_t k = keys[lane * n + i];
                if (k > k1) {
                    k2 = k1;
                    k1 = k;
                } else if (k > k2) {
                    k2 = k;
                }
            }
            float gs = key_score(k1);
            if (a.group_score == K3X_GROUP_TOP2 && n > 1) gs = __fadd_rn(gs, key_score(k2));
            gk = topk_key(gs, lane);
        }
        gkey[lane] = gk;
        __syncthreads();
        uint32_t rank = 0;
        for (uint32_t g = 0; g < a.G; ++g) rank += gkey[g] > gk;
        const uint64_t kept = __ballot(lane < a.G && rank < a.top_groups);
        for (uint32_t e = lane; e < E; e += 64)
            if (!(kept >> (e / n) & 1)) keys[e] = 0;
        __syncthreads();
    }
    float selsc = 0.0f;
    uint32_t selid = 0;
    for (uint32_t slot = 0; slot < a.K; ++slot) {
        uint64_t best = 0;
        for (uint32_t e = lane; e < E; e += 64) best = keys[e] > best ? keys[e] : best;
        best = wave_max_u64(best);
        const uint32_t win = 0xffffffffu - (uint32_t)best;
        if (lane == slot) {
            selid = win;
            selsc = sc[win];
        }
        __syncthreads();
        if (lane == 0) keys[win] = 0;
        __syncthreads();
    }
    uint32_t err;
    const float w = route_weight(a, selsc, &err);
    if (err) {
        if (lane == 0) latch(a.status, err);
        return;
    }
    if (lane < a.K) {
        a.ids[(size_t)t * a.K + lane] = selid;
        a.weights[(size_t)t * a.K + lane] = w;
    }
}

bool route_ok(const k3x_hip_route_params* p) {
    if (!p->tokens || p->tokens > (1u << 20) || !p->experts || p->experts > 4096 || !p->top_k ||
        p->top_k > 64 || p->dtype > K3X_DTYPE_BF16 || p->scoring > K3X_SCORE_SOFTMAX ||
        p->renorm > K3X_RENORM_NONE || !std::isfinite(p->routed_scale) ||
        p->group_score > K3X_GROUP_TOP2)
        return false;
    if (!p->groups || p->groups > 64 || p->experts % p->groups || !p->top_groups ||
        p->top_groups > p->groups || p->top_k > p->top_groups * (p->experts / p->groups))
        return false;
    return !p->logits_stride || p->logits_stride >= p->experts;
}

}  // namespace

extern "C" {

int k3x_hip_route(k3x_hip_ctx* ctx, const k3x_hip_route_params* p, const void* logits,
                  const float* bias, uint32_t* ids, float* weights) {
    if (!ctx || !p || !logits || !ids || !weights || !route_ok(p)) return K3X_ERR_INVALID_EXTENT;
    if (!aligned(logits, p->dtype == K3X_DTYPE_F32 ? 4 : 2) || !aligned(bias, 4) ||
        !aligned(ids, 4) || !aligned(weights, 4))
        return K3X_ERR_INVALID_EXTENT;
    if (hipSetDevice(ctx->device) != hipSuccess) return K3X_ERR_BACKEND_UNAVAILABLE;
    RouteArgs a{};
    a.logits = logits;
    a.bias = bias;
    a.T = p->tokens;
    a.E = p->experts;
    a.K = p->top_k;
    a.scoring = p->scoring;
    a.renorm = p->renorm;
    a.scale = p->routed_scale;
    a.G = p->top_groups == p->groups ? 1 : p->groups;  // every group stays: no groups
    a.top_groups = p->top_groups;
    a.group_score = p->group_score;
    a.stride = p->logits_stride ? p->logits_stride : p->experts;
    a.ids = ids;
    a.weights = weights;
    a.status = ctx->status;
    if (p->dtype == K3X_DTYPE_F32)
        hipLaunchKernelGGL(route_lds_kernel<K3X_DTYPE_F32>, dim3(a.T), dim3(64),
                           (size_t)a.E * 12, ctx->stream, a);
    else
        hipLaunchKernelGGL(route_lds_kernel<K3X_DTYPE_BF16>, dim3(a.T), dim3(64),
                           (size_t)a.E * 12, ctx->stream, a);
    return launched(ctx, 1);
}

}  // extern "C"
