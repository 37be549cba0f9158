// mla_cache.hip -- the paged cache of latent attention: rows written with their
// norm and quantisation, and read back.
//
// A wave a token at a time: eight neighbours of the latent a lane, so that a block
// of 32 is four lanes, its largest two exchanges within them, and a row one load and
// one store a lane.  Of many tokens a wave takes eight, looked up together, with
// their loads on their way together.
//
// Bound: memory, and with few tokens the chain of a token's sequence, page and row.
// Kernels at a latent of 512 and a rotary part of 64: 64 decode tokens in E4M3 4.4 us
// written and 3.8 read; 8192 tokens with their norm in E2M1 8.7 (13 MB) and 6.3; six
// prefixes of 131072 tokens together read in 57 us, 237 MB at 4.1 TB/s, where a large
// copy reaches 5.1 (38 us where the last cache holds the rows).
#include <hip/hip_runtime.h>

#include "k3x_mla.hpp"

using namespace k3x_dev;
using namespace k3x_ops;
using namespace k3x_mla;

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kLowestScale = 17;  // 2^-110: what codes stand for stays a normal bf16 number

struct CacheArgs {
    Pages pages;
    void *latent, *rotary;
    const float* gamma;
    uint8_t* pool;
    uint32_t L, R;
    uint64_t ls, rs;  // elements from token to token
    double eps;
    uint32_t vec;     // rows of latent and rotary by 16 bytes
    uint32_t* status;
};

typedef __attribute__((ext_vector_type(8))) uint16_t u16x8;

__device__ inline u16x8 load8(const uint16_t* p, uint32_t vec) {
    if (vec) return *reinterpret_cast<const u16x8*>(p);
    u16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j];
    return v;
}
__device__ inline void store8(uint16_t* p, u16x8 v, uint32_t vec) {
    if (vec) {
        *reinterpret_cast<u16x8*>(p) = v;
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = v[j];
}

template <uint32_t DT>
__device__ inline float value(uint16_t v) {
    return Elem<DT>::load(__builtin_bit_cast(typename Elem<DT>::type, v));
}
template <uint32_t DT>
__device__ inline uint16_t bits(float v) {
    return __builtin_bit_cast(uint16_t, Elem<DT>::store(v));
}

// Cached rows of the call's tokens t0 .. t0 + TP - 1, token i's in lane i; null: it
// has none (or its page is none of the pool, which is latched).  By a wave.
template <int TP>
__device__ inline uint8_t* find_rows(const CacheArgs& a, uint32_t t0) {
    const Pages& p = a.pages;
    const uint32_t lane = threadIdx.x & 63;
    uint32_t n = sequence_of(p, t0);
    if (TP > 1) {
        if (p.offsets) {
            // Of the 64 sequences from the first token's on (the first ones, where it lies
            // before them all); another search past them.
            const uint32_t from = n < p.N ? n : 0, o = p.offsets[min(from + lane, p.N)];
#pragma unroll
            for (int i = 1; i < TP; ++i) {
                const uint32_t k = __popcll(__ballot(from + lane < p.N && o <= t0 + i));
                uint32_t m = from + max(k, 1u) - 1;
                if (k == 64) m = sequence_of(p, t0 + i);
                if (lane == (uint32_t)i) n = m;
            }
        } else if (n < p.N) {
            n = (t0 + min(lane, (uint32_t)TP - 1)) / (p.T / p.N);
        }
    }
    const uint32_t t = t0 + lane;
    Tokens s;
    if (lane >= TP || t >= p.T || n >= p.N || !tokens_of(p, n, &s) || t < s.begin ||
        t - s.begin >= s.count)
        return nullptr;
    const int64_t pos = (int64_t)s.len - s.count + (t - s.begin);
    if (pos < 0) return nullptr;
    uint8_t* row = cached_row(p, a.pool, n, (uint32_t)pos);
    if (!row) latch(a.status, K3X_ERR_INVALID_STATE);
    return row;
}
// Lane i's pointer, in every lane.
__device__ inline uint8_t* row_of(uint8_t* mine, int i) {
    const uint64_t v = reinterpret_cast<uint64_t>(mine);
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, i);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), i);
    return reinterpret_cast<uint8_t*>((uint64_t)hi << 32 | lo);
}

// 1 / sqrt(x) in double: an estimate of 24 bits or so, and Newton's step twice.
__device__ inline double rsqrt_f64(double x) {
    double y = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; ++i) y = y * __builtin_fma(-0.5 * x * y, y, 1.5);
    return y;
}

template <uint32_t DT, uint32_t F>
__device__ inline void store_row(const CacheArgs& a, uint8_t* row, u16x8 v, u16x8 r,
                                 const float (&gamma)[8]) {
    const uint32_t lane = threadIdx.x & 63;
    const bool mine = 8 * lane < a.L, turns = 8 * lane < a.R;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = value<DT>(v[j]);
    if (a.gamma) {
        // In double, so that a value next to a border of the codes falls on the
        // side that the formula says.
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) s = __builtin_fma((double)x[j], (double)x[j], s);
        s = wave_sum(s);
        const double inv = rsqrt_f64(s / a.L + a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = bits<DT>((float)((double)x[j] * inv * (double)gamma[j]));
            x[j] = value<DT>(v[j]);
        }
    }
    bool wrong = false;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        wrong |= !(fabsf(x[j]) < __builtin_inff()) || !(fabsf(value<DT>(r[j])) < __builtin_inff());
    if (__any(wrong)) {
        if (lane == 0) latch(a.status, K3X_ERR_INVALID_MXFP4);
        return;
    }
    const RowLayout& at = a.pages.row;
    if (turns) *reinterpret_cast<u16x8*>(row + at.codes + 16 * lane) = r;
    if constexpr (F == K3X_CACHE_16BIT) {
        if (mine) *reinterpret_cast<u16x8*>(row + 16 * lane) = v;
    } else {
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(x[j]));
        m = fmaxf(m, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(m), 0xb1, 0xf, 0xf, false)));
        m = fmaxf(m, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(m), 0x4e, 0xf, 0xf, false)));
        // The largest is f 2^e, f in 1 .. 2; the codes' largest 1.75 2^8 or 1.5 2^2.
        const uint32_t b = __float_as_uint(m), f = b & 0x7fffffu;
        int scale = (int)(b >> 23);
        if constexpr (F == K3X_CACHE_MXFP8) scale += (f > 0x600000u) - 8;
        else scale += (f > 0x400000u) - 2;
        scale = max(scale, (int)kLowestScale);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __builtin_ldexpf(x[j], 127 - scale);
        if constexpr (F == K3X_CACHE_MXFP8) {
            typedef __attribute__((ext_vector_type(2))) short s16x2;
            s16x2 lo{}, hi{};
            lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[0], x[1], 1.0f, false);
            lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[2], x[3], 1.0f, true);
            hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[4], x[5], 1.0f, false);
            hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[6], x[7], 1.0f, true);
            const uint2 c{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
            if (mine) *reinterpret_cast<uint2*>(row + 8 * lane) = c;
        } else {
            uint32_t c = 0;
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], 1.0f, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], 1.0f, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], 1.0f, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], 1.0f, 3);
            if (mine) *reinterpret_cast<uint32_t*>(row + 4 * lane) = c;
        }
        const int s = __shfl(scale, (int)(4 * lane & 63));
        if (lane < 16) row[at.scales + lane] = lane < a.L / 32 ? (uint8_t)s : (uint8_t)0;
    }
}

template <uint32_t DT, uint32_t F, int TP>
__global__ __launch_bounds__(kThreads) void mla_store_kernel(CacheArgs a) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t t0 = (blockIdx.x * (kThreads / 64) +
                         __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * TP;
    const uint32_t status = *(volatile uint32_t*)a.status;
    if (blockIdx.x == 0) check_sequences(a.pages, a.status);
    if (t0 >= a.pages.T) return;
    u16x8 v[TP]{}, r[TP]{};
#pragma unroll
    for (int i = 0; i < TP; ++i) {
        const size_t t = min(t0 + i, a.pages.T - 1);
        if (8 * lane < a.L)
            v[i] = load8(static_cast<const uint16_t*>(a.latent) + t * a.ls + 8 * lane, a.vec);
        if (8 * lane < a.R)
            r[i] = load8(static_cast<const uint16_t*>(a.rotary) + t * a.rs + 8 * lane, a.vec);
    }
    float gamma[8] = {};
    if (a.gamma && 8 * lane < a.L)
#pragma unroll
        for (int j = 0; j < 8; ++j) gamma[j] = a.gamma[8 * lane + j];
    uint8_t* const rows = find_rows<TP>(a, t0);
    if (status) return;
#pragma unroll
    for (int i = 0; i < TP; ++i)
        if (uint8_t* row = row_of(rows, i)) store_row<DT, F>(a, row, v[i], r[i], gamma);
}

template <uint32_t F, int TP>
__global__ __launch_bounds__(kThreads) void mla_load_kernel(CacheArgs a) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t t0 = (blockIdx.x * (kThreads / 64) +
                         __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * TP;
    const uint32_t status = *(volatile uint32_t*)a.status;
    if (blockIdx.x == 0) check_sequences(a.pages, a.status);
    if (t0 >= a.pages.T) return;
    uint8_t* const rows = find_rows<TP>(a, t0);
    if (status) return;
    const RowLayout& at = a.pages.row;
    const bool mine = 8 * lane < a.L, turns = a.rotary && 8 * lane < a.R;
    u16x8 v[TP], r[TP];
    uint2 codes[TP];
    uint32_t scale[TP];
#pragma unroll
    for (int i = 0; i < TP; ++i) {
        const uint8_t* row = row_of(rows, i);
        if (!row) continue;
        if (turns) r[i] = *reinterpret_cast<const u16x8*>(row + at.codes + 16 * lane);
        if (!mine) continue;
        if constexpr (F == K3X_CACHE_16BIT) {
            v[i] = *reinterpret_cast<const u16x8*>(row + 16 * lane);
        } else {
            scale[i] = row[at.scales + lane / 4];
            if constexpr (F == K3X_CACHE_MXFP8)
                codes[i] = *reinterpret_cast<const uint2*>(row + 8 * lane);
            else
                codes[i].x = *reinterpret_cast<const uint32_t*>(row + 4 * lane);
        }
    }
#pragma unroll
    for (int i = 0; i < TP; ++i) {
        if (!row_of(rows, i)) continue;
        const size_t t = t0 + i;
        if (turns) store8(static_cast<uint16_t*>(a.rotary) + t * a.rs + 8 * lane, r[i], a.vec);
        if (!mine) continue;
        if constexpr (F == K3X_CACHE_MXFP8)
            v[i] = __builtin_bit_cast(u16x8, mxfp8_8(codes[i], e8m0_to_f32(scale[i])));
        else if constexpr (F == K3X_CACHE_MXFP4)
            v[i] = __builtin_bit_cast(u16x8, dequant8(codes[i].x, e8m0_to_f32(scale[i])));
        store8(static_cast<uint16_t*>(a.latent) + t * a.ls + 8 * lane, v[i], a.vec);
    }
}

// What both calls share; 0 or the status to return.
int cache_args(k3x_hip_ctx* ctx, const k3x_hip_mla_params* p, const void* latent,
               const void* rotary, const uint32_t* table, const uint32_t* offsets,
               const uint32_t* lens, const void* pool, CacheArgs* a) {
    if (!ctx || !p || !mla_ok(p) || (p->tokens && !latent) || !table || !lens || !pool)
        return K3X_ERR_INVALID_EXTENT;
    if (!aligned(latent, 2) || !aligned(rotary, 2) || !aligned(table, 4) ||
        !aligned(offsets, 4) || !aligned(lens, 4) || !aligned(pool, 256))
        return K3X_ERR_INVALID_EXTENT;
    if (hipSetDevice(ctx->device) != hipSuccess) return K3X_ERR_BACKEND_UNAVAILABLE;
    a->pages = pages_of(p, table, offsets, lens);
    a->latent = const_cast<void*>(latent);
    a->rotary = const_cast<void*>(rotary);
    a->pool = static_cast<uint8_t*>(const_cast<void*>(pool));
    a->L = p->latent;
    a->R = p->rotary;
    a->ls = p->latent_stride ? p->latent_stride : p->latent;
    a->rs = p->rotary_stride ? p->rotary_stride : p->rotary;
    a->vec = aligned(latent, 16) && a->ls % 8 == 0 &&
             (!rotary || (aligned(rotary, 16) && a->rs % 8 == 0));
    a->status = ctx->status;
    return K3X_OK;
}

// One token a wave, or eight past twice the waves that are held at once: with fewer, waves
// that wait hide each other's time better.  Kernels over eight inputs in turn, E2M1 with the
// norm, one and eight: 8192 tokens stored 9.2 and 10.5 us, 16384 16.8 and 16.6, 32768 28.0 and
// 26.4; read 6.4 and 7.8, 9.0 and 8.6, 14.7 and 11.1.
constexpr uint32_t kByEights = 16384;
template <uint32_t DT, uint32_t F>
int launch_store(k3x_hip_ctx* ctx, const CacheArgs& a) {
    const uint32_t T = a.pages.T;
    if (T > kByEights)
        hipLaunchKernelGGL((mla_store_kernel<DT, F, 8>), dim3((T + 31) / 32), dim3(kThreads), 0, ctx->stream, a);
    else
        hipLaunchKernelGGL((mla_store_kernel<DT, F, 1>), dim3((T + 3) / 4 + !T), dim3(kThreads), 0, ctx->stream, a);
    return launched(ctx, 1);
}
template <uint32_t F>
int launch_load(k3x_hip_ctx* ctx, const CacheArgs& a) {
    const uint32_t T = a.pages.T;
    if (T > kByEights)
        hipLaunchKernelGGL((mla_load_kernel<F, 8>), dim3((T + 31) / 32), dim3(kThreads), 0, ctx->stream, a);
    else
        hipLaunchKernelGGL((mla_load_kernel<F, 1>), dim3((T + 3) / 4 + !T), dim3(kThreads), 0, ctx->stream, a);
    return launched(ctx, 1);
}

}  // namespace

extern "C" {

size_t k3x_hip_mla_row_bytes(const k3x_hip_mla_params* p) {
    return p && mla_ok(p) ? row_layout(p->cache_format, p->latent, p->rotary).bytes : 0;
}

int k3x_hip_mla_store(k3x_hip_ctx* ctx, const k3x_hip_mla_params* p, const void* latent,
                      const void* rotary, const float* gamma, const uint32_t* table,
                      const uint32_t* offsets, const uint32_t* lens, void* pool) {
    if (!p || (p->tokens && p->rotary && !rotary) || !aligned(gamma, 4)) return K3X_ERR_INVALID_EXTENT;
    CacheArgs a{};
    const int st = cache_args(ctx, p, latent, rotary, table, offsets, lens, pool, &a);
    if (st != K3X_OK) return st;
    a.gamma = gamma;
    a.eps = p->norm_epsilon;
    if (p->dtype == K3X_DTYPE_F16) return launch_store<K3X_DTYPE_F16, K3X_CACHE_16BIT>(ctx, a);
    switch (p->cache_format) {
        case K3X_CACHE_16BIT: return launch_store<K3X_DTYPE_BF16, K3X_CACHE_16BIT>(ctx, a);
        case K3X_CACHE_MXFP8: return launch_store<K3X_DTYPE_BF16, K3X_CACHE_MXFP8>(ctx, a);
        default: return launch_store<K3X_DTYPE_BF16, K3X_CACHE_MXFP4>(ctx, a);
    }
}

int k3x_hip_mla_load(k3x_hip_ctx* ctx, const k3x_hip_mla_params* p, const void* pool,
                     const uint32_t* table, const uint32_t* offsets, const uint32_t* lens,
                     void* latent, void* rotary) {
    CacheArgs a{};
    const int st = cache_args(ctx, p, latent, rotary, table, offsets, lens, pool, &a);
    if (st != K3X_OK) return st;
    switch (p->cache_format) {
        case K3X_CACHE_16BIT: return launch_load<K3X_CACHE_16BIT>(ctx, a);  // bits as they are
        case K3X_CACHE_MXFP8: return launch_load<K3X_CACHE_MXFP8>(ctx, a);
        default: return launch_load<K3X_CACHE_MXFP4>(ctx, a);
    }
}

}  // extern "C"
