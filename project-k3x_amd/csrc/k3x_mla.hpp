// k3x_mla.hpp -- what the latent attention operators (mla_cache.hip,
// mla_attention.hip, mla_prompt.hip) share: the tokens of a call, the pages of a
// cache and the rows in them.
#pragma once

#include <algorithm>
#include <cmath>

#include "k3x_ops.hpp"

namespace k3x_mla {

// The rows of a cache: codes, rotary part, then (with codes) 16 bytes of scales.
struct RowLayout {
    uint32_t codes;   // bytes of the latent
    uint32_t scales;  // where they begin; 0: none
    uint32_t bytes;
};

inline __host__ __device__ RowLayout row_layout(uint32_t format, uint32_t L, uint32_t R) {
    RowLayout r;
    r.codes = format == K3X_CACHE_16BIT ? 2 * L : format == K3X_CACHE_MXFP8 ? L : L / 2;
    r.scales = format == K3X_CACHE_16BIT ? 0 : r.codes + 2 * R;
    r.bytes = r.codes + 2 * R + (format == K3X_CACHE_16BIT ? 0 : 16);
    return r;
}

// The sequences of a call and their pages.
struct Pages {
    const uint32_t *table, *offsets, *lens;
    uint32_t N, T, page, pages, width, longest, most;  // most: positions of a sequence
    uint32_t page_by, page_shift;  // page_of
    RowLayout row;
    // p / page for p < 2^31: page_by = ceil(2^page_shift / page) with 2^(page_shift - 31)
    // >= page, so that its product is off by less than p / 2^page_shift <= 1 / page.
    __device__ inline uint32_t page_of(uint32_t p) const {
        return (uint32_t)((uint64_t)p * page_by >> page_shift);
    }
};

// Sequence n's rows of the call; false: offsets or length are not fit (latched
// by check_sequences).
struct Tokens {
    uint32_t begin, count, len;
};
__device__ inline bool tokens_of(const Pages& a, uint32_t n, Tokens* s) {
    uint32_t b, e;
    if (a.offsets) {
        b = a.offsets[n];
        e = a.offsets[n + 1];
    } else {
        const uint32_t each = a.T / a.N;
        b = n * each;
        e = b + each;
    }
    s->begin = b;
    s->count = e - b;
    s->len = a.lens[n];
    return e >= b && e <= a.T && e - b <= a.longest && s->len <= a.most;
}

// Latches what tokens_of refuses, by the whole workgroup, which is one of the
// grid's.
__device__ inline void check_sequences(const Pages& a, uint32_t* status) {
    bool bad = false;
    for (uint32_t n = threadIdx.x; n < a.N; n += blockDim.x) {
        Tokens s;
        bad |= !tokens_of(a, n, &s);
    }
    if (bad) k3x_ops::latch(status, K3X_ERR_INVALID_STATE);
}

// The sequence that row t of the call belongs to, by a wave: a 64-ary search for
// the last n with offsets[n] <= t.  N: none.
__device__ inline uint32_t sequence_of(const Pages& a, uint32_t t) {
    if (!a.offsets) {
        const uint32_t each = a.T / a.N;
        return each ? min(t / each, a.N) : a.N;
    }
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, count = a.N;
    for (;;) {
        const uint32_t step = (count + 63) / 64, at = lane * step;
        const uint64_t m = __ballot(at < count && a.offsets[lo + min(at, count - 1)] <= t);
        if (!m) return a.N;
        const uint32_t k = (__popcll(m) - 1) * step;
        lo += k;
        count = min(step, count - k);
        if (step == 1) return lo;
    }
}

// Row of position p (below the sequence's length) of a sequence's pages; null
// where the page is not one of the pool.
__device__ inline uint8_t* cached_row(const Pages& a, uint8_t* pool, uint32_t n, uint32_t p) {
    const uint32_t page = a.page_of(p), id = a.table[(size_t)n * a.width + page];
    if (id >= a.pages) return nullptr;
    return pool + ((size_t)id * a.page + (p - page * a.page)) * a.row.bytes;
}

// Eight E4M3 codes times a power of two as bf16, exact (four significant bits).
__device__ inline k3x_dev::bf16x8 mxfp8_8(uint2 c, float scale) {
    const k3x_dev::bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, scale, false);
    const k3x_dev::bf16x2 q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, scale, true);
    const k3x_dev::bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, scale, false);
    const k3x_dev::bf16x2 s = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, scale, true);
    return k3x_dev::bf16x8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}

inline bool mla_ok(const k3x_hip_mla_params* p) {
    return p->sequences && p->sequences <= 65535 && p->tokens <= (1u << 22) && p->heads &&
           p->heads <= 1024 && p->latent && p->latent <= 512 && p->latent % 32 == 0 &&
           p->rotary <= 64 && p->rotary % 8 == 0 && p->cache_format <= K3X_CACHE_MXFP4 &&
           (p->dtype == K3X_DTYPE_BF16 ||
            (p->dtype == K3X_DTYPE_F16 && p->cache_format == K3X_CACHE_16BIT)) &&
           p->page_size && p->page_size <= 65536 && p->pages &&
           (uint64_t)p->pages * p->page_size <= (1ull << 31) && p->table_width &&
           p->table_width <= (1u << 20) && std::isfinite(p->scale) && p->scale > 0.0f &&
           std::isfinite(p->norm_epsilon) && p->norm_epsilon >= 0.0f &&
           (!p->latent_stride || p->latent_stride >= p->latent) &&
           (!p->rotary_stride || p->rotary_stride >= p->rotary) &&
           (!p->q_stride || p->q_stride >= (uint64_t)p->heads * (p->latent + p->rotary)) &&
           (!p->out_stride || p->out_stride >= (uint64_t)p->heads * p->latent) &&
           p->latent_stride <= (1ull << 32) && p->rotary_stride <= (1ull << 32) &&
           p->q_stride <= (1ull << 32) && p->out_stride <= (1ull << 32);
}

inline Pages pages_of(const k3x_hip_mla_params* p, const uint32_t* table, const uint32_t* offsets,
                      const uint32_t* lens) {
    Pages a{};
    a.table = table;
    a.offsets = offsets;
    a.lens = lens;
    a.N = p->sequences;
    a.T = p->tokens;
    a.page = p->page_size;
    a.page_shift = 31;
    while (1ull << (a.page_shift - 31) < a.page) ++a.page_shift;
    a.page_by = (uint32_t)(((1ull << a.page_shift) + a.page - 1) / a.page);
    a.pages = p->pages;
    a.width = p->table_width;
    a.longest = p->longest ? p->longest : p->tokens;
    a.most = (uint32_t)std::min<uint64_t>((uint64_t)a.width * a.page, 1u << 29);
    a.row = row_layout(p->cache_format, p->latent, p->rotary);
    return a;
}

}  // namespace k3x_mla
