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
    uint32_t group, group_by;  // experts a group; 2^20 / group + 1
    uint32_t stride;
    uint32_t* ids;
    float* weights;
    uint32_t* status;
};

__device__ inline uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_xor(v, d);
        v = v > o ? v : o;
    }
    return v;
}

// The adjusted score of a sort key (topk_key).
__device__ inline float key_score(uint64_t key) { return unordered((uint32_t)(key >> 32)); }

// sigmoid_cr without its branches: past +-200 the exponential is infinite or 0
// in fp32 already, so the argument may stop there.
__device__ inline float sigmoid_flat(float v) {
    const float x = fminf(fmaxf(-v, -200.0f), 200.0f);
    const double xd = (double)x;
    const double k = __builtin_rint(xd * 1.4426950408889634);
    const float t = __fadd_rn(1.0f, (float)__builtin_ldexp(exp_series(xd, k), (int)k));
    return v == v ? __fdiv_rn(1.0f, t) : v;
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

// x or, if that is larger, its neighbour's by the DPP control; the same for
// the smaller one.
template <int Ctrl>
__device__ inline uint32_t dpp_max(uint32_t x) {
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, Ctrl, 0xf, 0xf, true));
}
template <int Ctrl>
__device__ inline uint32_t dpp_min(uint32_t x) {
    return min(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, Ctrl, 0xf, 0xf, true));
}
template <bool MAX>
__device__ inline uint32_t across_rows(uint32_t x, bool halves) {
    const auto r = halves ? __builtin_amdgcn_permlane32_swap(x, x, false, false)
                          : __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return MAX ? max(r[0], r[1]) : min(r[0], r[1]);
}

// A bound that at least K keys reach: the smallest of the largest keys of the
// 64 / n groups of n neighbouring lanes, n the largest with 64 / n >= K (head:
// the lane's largest key).  Few others reach it, about 64 / n times its log.
__device__ inline uint32_t reached_by(uint32_t head, uint32_t K) {
    uint32_t x = head;
    const uint32_t steps = K > 32 ? 0 : K > 16 ? 1 : K > 8 ? 2 : K > 4 ? 3 : K > 2 ? 4 : K > 1 ? 5 : 6;
    x = steps > 0 ? dpp_max<0xb1>(x) : dpp_min<0xb1>(x);    // quad_perm [1,0,3,2]
    x = steps > 1 ? dpp_max<0x4e>(x) : dpp_min<0x4e>(x);    // quad_perm [2,3,0,1]
    x = steps > 2 ? dpp_max<0x141>(x) : dpp_min<0x141>(x);  // row_half_mirror
    x = steps > 3 ? dpp_max<0x140>(x) : dpp_min<0x140>(x);  // row_mirror
    x = steps > 4 ? across_rows<true>(x, false) : across_rows<false>(x, false);
    return steps > 5 ? across_rows<true>(x, true) : across_rows<false>(x, true);
}

// More than 1024 experts, for which a wave has no registers: one wave a token,
// keys and scores in LDS, K passes over the keys.  8192 tokens of 1024 experts,
// Top-8 of sigmoid scores: 59 us, and 23 in registers.
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
        for (uint32_t e = lane; e < E; e += 64) den += exp_f64((double)Elem<DT>::load(row[e]) - mx);
        den = 1.0 / wave_sum(den);
    }
    uint32_t bad = 0;
    for (uint32_t e = lane; e < E; e += 64) {
        const float l = Elem<DT>::load(row[e]);
        const float b = a.bias ? a.bias[e] : 0.0f;
        const float s = a.scoring == K3X_SCORE_SOFTMAX ? (float)(exp_f64((double)l - mx) * den)
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
        const uint32_t n = a.group;
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

// E <= 64 KPL: a wave a token, lane l with experts l + 64 i in registers.  The
// keys that reach a bound which K of them reach are written to LDS in the
// experts' order, and each is ranked by counting those above it: a pass over a
// few dozen keys in place of K passes over all.
//
// Bound by the instructions: 30011 tokens of 256 experts (bf16, softmax, Top-8
// in 4 of 8 groups) take 33 us, some 600 vector instructions a token, where
// the logits' 15 MB take 4 us; 2048 tokens of 896 experts (sigmoid) 13 us.
// The fewest registers that hold the experts (Top-8 of sigmoid scores, 30011
// tokens): 256 experts 23 us with 4 a lane, 33 with 8, 61 with 16; 512 experts
// 36 with 8 and 64 with 16.
constexpr int kRouteWaves = 4;

template <uint32_t DT, int KPL>
__global__ __launch_bounds__(64 * kRouteWaves) void route_wave_kernel(RouteArgs a) {
    typedef typename Elem<DT>::type T;
    struct Wave {
        __attribute__((aligned(16))) uint64_t key[64 * KPL + 8];
        float score[64 * KPL];
        uint32_t id[64];
        float sel[64];
    };
    __shared__ Wave waves[kRouteWaves];
    const uint32_t lane = threadIdx.x & 63, E = a.E;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t t = blockIdx.x * kRouteWaves + w;
    if (t >= a.T) return;
    Wave& s = waves[w];
    const T* row = static_cast<const T*>(a.logits) + (size_t)t * a.stride;
    float l[KPL], b[KPL], sc[KPL];
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        const uint32_t e = min(lane + 64u * i, E - 1);
        l[i] = Elem<DT>::load(row[e]);
        b[i] = a.bias ? a.bias[e] : 0.0f;
    }
    if (*(volatile uint32_t*)a.status) return;
    if (a.scoring == K3X_SCORE_SOFTMAX) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < KPL; ++i) top = max(top, ordered(l[i]));
        const double mx = (double)unordered(wave_max_u32(top));
        double e[KPL], den = 0.0;
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
            // Past E the last expert's once more, and left out after: no branch.
            const double y = exp_f64((double)l[i] - mx);
            e[i] = lane + 64u * i < E ? y : 0.0;
            den += e[i];
        }
        const double inv = 1.0 / wave_sum(den);
#pragma unroll
        for (int i = 0; i < KPL; ++i) sc[i] = (float)(e[i] * inv);
    } else {
#pragma unroll
        for (int i = 0; i < KPL; ++i) sc[i] = sigmoid_flat(l[i]);
    }
    uint32_t bad = 0, ord[KPL];
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        const float adj = __fadd_rn(sc[i], b[i]);
        const bool in = lane + 64u * i < E;
        if (in) bad = max(bad, route_check(a, l[i], sc[i], b[i], adj));
        ord[i] = in ? (uint32_t)(topk_key(adj, 0) >> 32) : 0u;
    }
    if (__any(bad)) {
        bad = wave_max_u32(bad);
        if (lane == 0) latch(a.status, bad);
        return;
    }
    if (a.G > 1) {
        // Several lanes a group: each takes every so many-th of its experts'
        // keys, then they join their two largest.
        uint32_t* keys = reinterpret_cast<uint32_t*>(s.key);
#pragma unroll
        for (int i = 0; i < KPL; ++i)
            if (lane + 64u * i < E) keys[lane + 64u * i] = ord[i];
        wave_sync();
        const uint32_t n = a.group, width = 64u >> (32 - __clz(a.G - 1));  // lanes a group
        const uint32_t g = lane / width;
        uint32_t k1 = 0, k2 = 0;
        if (g < a.G)
            for (uint32_t i = lane % width; i < n; i += width) {
                const uint32_t k = keys[g * n + i];
                k2 = max(k2, min(k1, k));
                k1 = max(k1, k);
            }
        for (uint32_t d = 1; d < width; d <<= 1) {
            const uint32_t o1 = (uint32_t)__shfl_xor((int)k1, d);
            const uint32_t o2 = (uint32_t)__shfl_xor((int)k2, d);
            k2 = max(max(k2, o2), min(k1, o1));
            k1 = max(k1, o1);
        }
        float gs = key_score((uint64_t)k1 << 32);
        if (a.group_score == K3X_GROUP_TOP2 && n > 1)
            gs = __fadd_rn(gs, key_score((uint64_t)k2 << 32));
        // A group's lanes compare it with every width-th group each.
        const uint32_t gk = (uint32_t)(topk_key(gs, 0) >> 32);
        uint32_t rank = 0;
        for (uint32_t i = 0; i < a.G; i += width) {
            const uint32_t o = i + lane % width;
            const uint32_t ok = (uint32_t)__shfl((int)gk, (int)(o * width & 63));
            const uint64_t above = __ballot(o < a.G && (ok > gk || (ok == gk && o < g)));
            rank += (uint32_t)__popcll(above >> (g * width & 63) & (~0ull >> (64 - width)));
        }
        const uint64_t kept = __ballot(g < a.G && rank < a.top_groups);
        // e / n by a factor: e (2^20 / n + 1) 2^-20 is over it by 2^-10 <= 1 / n at most.
#pragma unroll
        for (int i = 0; i < KPL; ++i)
            if (!(kept >> (((lane + 64u * i) * a.group_by >> 20) * width & 63) & 1)) ord[i] = 0;
        wave_sync();
    }
    uint32_t head = 0;
#pragma unroll
    for (int i = 0; i < KPL; ++i) head = max(head, ord[i]);
    const uint32_t bound = max(reached_by(head, a.K), 1u);
    uint32_t count = 0;
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        const bool up = ord[i] >= bound;
        const uint64_t mask = __ballot(up);
        if (up) {
            const uint32_t at = count + __builtin_amdgcn_mbcnt_hi(
                                            (uint32_t)(mask >> 32),
                                            __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
            s.key[at] = (uint64_t)ord[i] << 32 | (0xffffffffu - (lane + 64u * i));
            s.score[at] = sc[i];
        }
        count += (uint32_t)__popcll(mask);
    }
    // Eight keys at a time are counted; 0 is below every key.
    if (lane < 8) s.key[count + lane] = 0;
    wave_sync();
    for (uint32_t c0 = 0; c0 < count; c0 += 64) {
        const uint32_t c = c0 + lane;
        const uint64_t key = s.key[min(c, count - 1)];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < count; j += 8) {
            typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
            const u64x2* p = reinterpret_cast<const u64x2*>(&s.key[j]);
            const u64x2 o[4] = {p[0], p[1], p[2], p[3]};
#pragma unroll
            for (int x = 0; x < 8; ++x) rank += o[x / 2][x % 2] > key;
        }
        if (c < count && rank < a.K) {
            s.id[rank] = 0xffffffffu - (uint32_t)key;
            s.sel[rank] = s.score[c];
        }
    }
    wave_sync();
    const float selsc = lane < a.K ? s.sel[lane] : 0.0f;
    uint32_t err;
    const float weight = route_weight(a, selsc, &err);
    if (err) {
        if (lane == 0) latch(a.status, err);
        return;
    }
    if (lane < a.K) {
        a.ids[(size_t)t * a.K + lane] = s.id[lane];
        a.weights[(size_t)t * a.K + lane] = weight;
    }
}

template <uint32_t DT>
void launch_route(const RouteArgs& a, hipStream_t stream) {
    const dim3 grid((a.T + kRouteWaves - 1) / kRouteWaves), block(64 * kRouteWaves);
    if (a.E <= 256) hipLaunchKernelGGL((route_wave_kernel<DT, 4>), grid, block, 0, stream, a);
    else if (a.E <= 512) hipLaunchKernelGGL((route_wave_kernel<DT, 8>), grid, block, 0, stream, a);
    else if (a.E <= 1024)
        hipLaunchKernelGGL((route_wave_kernel<DT, 16>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL(route_lds_kernel<DT>, dim3(a.T), dim3(64), (size_t)a.E * 12, stream, a);
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
    a.group = a.E / a.G;
    a.group_by = (1u << 20) / a.group + 1;
    a.top_groups = p->top_groups;
    a.group_score = p->group_score;
    a.stride = p->logits_stride ? p->logits_stride : p->experts;
    a.ids = ids;
    a.weights = weights;
    a.status = ctx->status;
    if (p->dtype == K3X_DTYPE_F32) launch_route<K3X_DTYPE_F32>(a, ctx->stream);
    else launch_route<K3X_DTYPE_BF16>(a, ctx->stream);
    return launched(ctx, 1);
}

}  // extern "C"
