// mla_cache.hip -- the paged cache of latent attention: rows written with their
// norm and quantisation, and read back.
//
// A wave a token: eight neighbours of the latent a lane, so that a block of 32
// is four lanes, its largest two exchanges within them, and a row one load and
// one store a lane.
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

// Row t's sequence and position; false: it has none that is cached.
__device__ inline bool locate(const Pages& a, uint32_t t, uint32_t* n, uint32_t* pos) {
    *n = sequence_of(a, t);
    Tokens s;
    if (*n >= a.N || !tokens_of(a, *n, &s) || t < s.begin || t - s.begin >= s.count) return false;
    const int64_t p = (int64_t)s.len - s.count + (t - s.begin);
    *pos = (uint32_t)p;
    return p >= 0;
}

template <uint32_t DT, uint32_t F>
__global__ __launch_bounds__(kThreads) void mla_store_kernel(CacheArgs a) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t t = blockIdx.x * (kThreads / 64) +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (*(volatile uint32_t*)a.status) return;
    if (blockIdx.x == 0) check_sequences(a.pages, a.status);
    uint32_t n, pos;
    if (t >= a.pages.T || !locate(a.pages, t, &n, &pos)) return;
    uint8_t* row = cached_row(a.pages, a.pool, n, pos);
    if (!row) {
        if (lane == 0) latch(a.status, K3X_ERR_INVALID_STATE);
        return;
    }
    const bool mine = 8 * lane < a.L, turns = 8 * lane < a.R;
    u16x8 v{}, r{};
    if (mine) v = load8(static_cast<const uint16_t*>(a.latent) + t * a.ls + 8 * lane, a.vec);
    if (turns) r = load8(static_cast<const uint16_t*>(a.rotary) + t * a.rs + 8 * lane, a.vec);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = value<DT>(v[j]);
    if (a.gamma) {
        // In double, so that a value next to a border of the codes falls on the
        // side that the formula says.
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += (double)x[j] * (double)x[j];
        s = wave_sum(s);
        const double inv = 1.0 / sqrt(s / a.L + a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float g = mine ? a.gamma[8 * lane + j] : 0.0f;
            v[j] = bits<DT>((float)((double)x[j] * inv * (double)g));
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

template <uint32_t DT, uint32_t F>
__global__ __launch_bounds__(kThreads) void mla_load_kernel(CacheArgs a) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t t = blockIdx.x * (kThreads / 64) +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (*(volatile uint32_t*)a.status) return;
    if (blockIdx.x == 0) check_sequences(a.pages, a.status);
    uint32_t n, pos;
    if (t >= a.pages.T || !locate(a.pages, t, &n, &pos)) return;
    const uint8_t* row = cached_row(a.pages, a.pool, n, pos);
    if (!row) {
        if (lane == 0) latch(a.status, K3X_ERR_INVALID_STATE);
        return;
    }
    const RowLayout& at = a.pages.row;
    if (a.rotary && 8 * lane < a.R)
        store8(static_cast<uint16_t*>(a.rotary) + t * a.rs + 8 * lane,
               *reinterpret_cast<const u16x8*>(row + at.codes + 16 * lane), a.vec);
    if (8 * lane >= a.L) return;
    u16x8 v;
    if constexpr (F == K3X_CACHE_16BIT) {
        v = *reinterpret_cast<const u16x8*>(row + 16 * lane);
    } else {
        const float scale = e8m0_to_f32(row[at.scales + lane / 4]);
        bf16x8 w;
        if constexpr (F == K3X_CACHE_MXFP8) w = mxfp8_8(*reinterpret_cast<const uint2*>(row + 8 * lane), scale);
        else w = dequant8(*reinterpret_cast<const uint32_t*>(row + 4 * lane), scale);
        v = __builtin_bit_cast(u16x8, w);
    }
    store8(static_cast<uint16_t*>(a.latent) + t * a.ls + 8 * lane, v, a.vec);
}

// What both calls share; 0 or the status to return.
int cache_args(k3x_hip_ctx* ctx, const k3x_hip_mla_params* p, const void* latent,
               const void* rotary, const uint32_t* table, const uint32_t* offsets,
               const uint32_t* lens, const void* pool, CacheArgs* a) {
    if (!ctx || !p || !mla_ok(p) || !latent || !table || !lens || !pool)
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

dim3 grid_of(const CacheArgs& a) { return dim3(a.pages.T ? (a.pages.T + 3) / 4 : 1); }

}  // namespace

extern "C" {

size_t k3x_hip_mla_row_bytes(const k3x_hip_mla_params* p) {
    return p && mla_ok(p) ? row_layout(p->cache_format, p->latent, p->rotary).bytes : 0;
}

int k3x_hip_mla_store(k3x_hip_ctx* ctx, const k3x_hip_mla_params* p, const void* latent,
                      const void* rotary, const float* gamma, const uint32_t* table,
                      const uint32_t* offsets, const uint32_t* lens, void* pool) {
    if (!p || (p->rotary && !rotary) || !aligned(gamma, 4)) return K3X_ERR_INVALID_EXTENT;
    CacheArgs a{};
    const int st = cache_args(ctx, p, latent, rotary, table, offsets, lens, pool, &a);
    if (st != K3X_OK) return st;
    a.gamma = gamma;
    a.eps = p->norm_epsilon;
    const dim3 grid = grid_of(a), block(kThreads);
    if (p->dtype == K3X_DTYPE_F16)
        hipLaunchKernelGGL((mla_store_kernel<K3X_DTYPE_F16, K3X_CACHE_16BIT>), grid, block, 0, ctx->stream, a);
    else if (p->cache_format == K3X_CACHE_16BIT)
        hipLaunchKernelGGL((mla_store_kernel<K3X_DTYPE_BF16, K3X_CACHE_16BIT>), grid, block, 0, ctx->stream, a);
    else if (p->cache_format == K3X_CACHE_MXFP8)
        hipLaunchKernelGGL((mla_store_kernel<K3X_DTYPE_BF16, K3X_CACHE_MXFP8>), grid, block, 0, ctx->stream, a);
    else
        hipLaunchKernelGGL((mla_store_kernel<K3X_DTYPE_BF16, K3X_CACHE_MXFP4>), grid, block, 0, ctx->stream, a);
    return launched(ctx, 1);
}

int k3x_hip_mla_load(k3x_hip_ctx* ctx, const k3x_hip_mla_params* p, const void* pool,
                     const uint32_t* table, const uint32_t* offsets, const uint32_t* lens,
                     void* latent, void* rotary) {
    CacheArgs a{};
    const int st = cache_args(ctx, p, latent, rotary, table, offsets, lens, pool, &a);
    if (st != K3X_OK) return st;
    const dim3 grid = grid_of(a), block(kThreads);
    if (p->cache_format == K3X_CACHE_16BIT)  // bits as they are, of either type
        hipLaunchKernelGGL((mla_load_kernel<K3X_DTYPE_BF16, K3X_CACHE_16BIT>), grid, block, 0, ctx->stream, a);
    else if (p->cache_format == K3X_CACHE_MXFP8)
        hipLaunchKernelGGL((mla_load_kernel<K3X_DTYPE_BF16, K3X_CACHE_MXFP8>), grid, block, 0, ctx->stream, a);
    else
        hipLaunchKernelGGL((mla_load_kernel<K3X_DTYPE_BF16, K3X_CACHE_MXFP4>), grid, block, 0, ctx->stream, a);
    return launched(ctx, 1);
}

}  // extern "C"
