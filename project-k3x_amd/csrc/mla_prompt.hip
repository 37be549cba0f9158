// mla_prompt.hip -- attention of prompts over expanded keys and values, with a
// part of the key that all heads share.
//
// S^T = K Q^T and O^T = V^T P^T on the matrix cores, as in mla_attention.hip: the
// result of the first product is, lane for lane, the second one's operand.  A
// wave holds 32 queries of one head and their outputs; the tiles of K and V of a
// workgroup's head lie in LDS, brought straight from memory a tile ahead.
//
// Bound: the matrix cores (busy for 53% of the cycles) and LDS: the two workgroups of a
// compute unit take 3900 cycles for a tile of 64 keys each, 2560 of them products; reads of
// LDS take about as long, and weights, 420 a wave, stand between.  One prompt of 2048
// tokens, 32 heads of 128 + 64 and 128: 56 us, 765 TFLOP/s of products that count (a large
// matrix product reaches 1218); seven ragged ones of 8192 tokens together 305 to 315 us,
// 788 to 813 TFLOP/s.  Two tiles of 32 queries a wave, one wave a SIMD, read LDS half as
// often, but take 547: then every cycle of weights is one without products.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "k3x_mla.hpp"
#include "k3x_mla_mma.hpp"

using namespace k3x_dev;
using namespace k3x_ops;
using namespace k3x_mla;

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kRows = 128;  // queries a workgroup

struct PromptArgs {
    const void *q, *k, *v, *rotary;
    const uint32_t *offsets, *key_offsets;
    void* out;
    float* lse;
    uint32_t N, T, S, H, Dn, R, Dv, causal, blocks, flip;
    uint64_t qs, ks, vs, rs, os, kh, vh;
    float rate;  // scale * log2(e)
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

// KD columns of a key and VD of a value at most, in groups of 64 in LDS; TILE keys a
// step.  OWN > 0: Dn is OWN whole groups, R the others and Dv is VD, so that nothing is
// left out.
template <uint32_t DT, int KD, int VD, int TILE, int OWN>
__global__ __launch_bounds__(kThreads, 2) void mla_prompt_kernel(PromptArgs a) {
    constexpr bool FULL = OWN > 0;
    constexpr int KG = KD / 64, VG = VD / 64, ST = TILE / 32, OT = VD / 32;
    constexpr uint32_t kGroup = TILE * 128;      // bytes of a group
    constexpr uint32_t kBuffer = (KG + VG) * kGroup;
    typedef Mma<DT, 32> M;
    typedef typename M::Acc Acc;
    // One array: see mla_attention.hip.
    __shared__ __attribute__((aligned(256))) uint8_t smem[2 * kBuffer];
    uint32_t* const scan = reinterpret_cast<uint32_t*>(smem);  // before the first tile
    uint32_t* const found = scan + 4;
    lds_byte* const lds = (lds_byte*)smem;
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t h = blockIdx.x % a.H;
    // All waves or none: another workgroup may latch between their looks.
    if (tid == 0) scan[0] = *(volatile uint32_t*)a.status;
    __syncthreads();
    const uint32_t status = scan[0];
    __syncthreads();
    if (status) return;

    // The workgroup's block of queries.  Blocks of up to 64 sequences are taken from those
    // with the most keys to those with the fewest, in 64 classes, so that no long one begins
    // last; of one sequence, and of more than 64, from the last to the first.
    // blocks_of(r, k): the blocks of a sequence with at least k keys, which are its last ones.
    auto blocks_of = [&](const Ranges& r, uint32_t k) -> uint32_t {
        const uint32_t all = (r.m + kRows - 1) / kRows;
        if (k == 0) return all;
        if (r.n < k) return 0;
        // The i-th block's last query sees n - m + min(m, kRows (i + 1)) keys.
        const uint32_t more = r.n - k;
        return a.causal && r.m > more ? all + 1 - (r.m - more + kRows - 1) / kRows : all;
    };
    uint32_t at = blockIdx.x / a.H, n = a.N, i0 = 0;
    bool bad = false;
    Ranges s{};
    auto load = [&](uint32_t x) {
        s = Ranges{};
        if (x < a.N && !ranges_of(a, x, &s)) {
            bad = true;
            s = Ranges{};
        }
    };
    auto scan_lanes = [&](uint32_t c) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(c, d);
            if (lane >= (uint32_t)d) c += o;
        }
        return c;
    };
    if (a.N <= 64) {  // every wave for itself
        load(lane);
        const uint32_t unit = a.N == 1 ? a.S + 1 : a.S / 64 + 1;
        uint32_t count = 0;  // blocks with at least lane * unit keys
        for (uint32_t x = 0; x < a.N; ++x) {
            Ranges r{};
            r.m = __builtin_amdgcn_readlane(s.m, x);
            r.n = __builtin_amdgcn_readlane(s.n, x);
            count += blocks_of(r, lane * unit);
        }
        const uint32_t blocks = __builtin_amdgcn_readfirstlane(count);
        // Blocks mostly of one sequence, up to two a compute unit, all begin at once: then the
        // second half goes the other way, so that a long and a short one share a unit.  2048
        // tokens, 32 heads: 60.5 us, 62.4 without; 4096 tokens, in two rounds: 201, 184
        // without; 1000, 700 and 300 tokens: 38.5, 34.2 without.
        if (a.flip && at < blocks && at >= blocks - blocks / 2)
            at = 2 * blocks - 1 - blocks / 2 - at;
        const uint64_t above = __ballot(count > at);
        if (above) {
            // A class falls with its number of keys: the last one that `at` is below.
            const uint32_t c = 63 - __builtin_clzll(above);
            const uint32_t before = c < 63 ? __builtin_amdgcn_readlane(count, c + 1 & 63) : 0;
            const uint32_t more = c < 63 ? blocks_of(s, (c + 1) * unit) : 0;
            const uint32_t own = blocks_of(s, c * unit) - more, end = before + scan_lanes(own);
            const uint64_t mine = __ballot(at < end && at >= end - own);
            if (mine) {
                const uint32_t x = __builtin_ctzll(mine);
                const uint32_t i = (s.m + kRows - 1) / kRows - 1 - more - (at - (end - own));
                n = x;
                i0 = __builtin_amdgcn_readlane(i, x) * kRows;
            }
        }
    } else {
        if (tid == 0) found[0] = a.N;
        at = a.blocks - 1 - at;
        uint32_t carry = 0;
        for (uint32_t base = 0; base < a.N; base += kThreads) {
            load(base + tid);
            const uint32_t own = blocks_of(s, 0);
            uint32_t c = scan_lanes(own);
            __syncthreads();
            if (lane == 63) scan[wave] = c;
            __syncthreads();
            for (uint32_t i = 0; i < wave; ++i) c += scan[i];
            c += carry;  // with the thread's own
            if (own && at >= c - own && at < c) {
                found[0] = base + tid;
                found[1] = at - (c - own);
            }
            carry += scan[0] + scan[1] + scan[2] + scan[3];
        }
        __syncthreads();
        n = __builtin_amdgcn_readfirstlane(found[0]);
        i0 = __builtin_amdgcn_readfirstlane(found[1]) * kRows;
    }
    if (blockIdx.x == 0 && bad) latch(a.status, K3X_ERR_INVALID_STATE);
    if (n >= a.N) return;
    ranges_of(a, n, &s);
    __syncthreads();
    if (!FULL) {  // columns that are not brought stay zero
        for (uint32_t i = tid * 16; i < 2 * kBuffer; i += kThreads * 16)
            *reinterpret_cast<u32x4*>(smem + i) = u32x4{};
        __syncthreads();
    }

    const uint32_t col = lane & 31, g = lane >> 5;
    const uint32_t w0 = i0 + 32 * wave;                        // the wave's first query
    const int32_t hidden = a.causal ? (int32_t)(s.m - 1) : 0;  // keys of the first query's future
    const uint32_t query = min(w0 + col, s.m - 1);             // the lane's
    auto sees_of = [&](uint32_t x) {
        return a.causal ? (int32_t)s.n - hidden + (int32_t)x : (int32_t)s.n;
    };
    const int32_t least = sees_of(min(w0, s.m - 1));             // of the wave
    const int32_t most = sees_of(min(i0 + kRows - 1, s.m - 1));  // of the workgroup
    const uint32_t tiles = most > 0 ? ((uint32_t)most + TILE - 1) / TILE : 0;

    const uint32_t kat0 = col * 128 + (g ^ swizzle(col)) * 16;
    const uint32_t i16 = lane & 15, vrow = 4 * g + i16 / 4;
    const uint32_t vat0 = vrow * 128 + ((2 * (lane >> 4 & 1) + (i16 & 3) / 2) ^ swizzle(vrow)) * 16 +
                          (i16 & 1) * 8;
    // What the lane brings: token 8 (wave + 4 x) + lane / 8 of a tile, 16 bytes a group.
    const uint32_t btok = 8 * wave + lane / 8, bput = lane % 8 ^ swizzle(btok);
    const uint32_t own = FULL ? OWN : (a.Dn + 63) / 64;  // groups of a head's own columns, then the rotary part's

    // A tile's loads in pieces, each 128 bytes of eight tokens a wave: they take long to
    // be issued, so they are spread over the products.
    struct Source {
        __amdgpu_buffer_rsrc_t k, v, r;
        uint32_t kf, vf, rf;
        u32x4* dst;
    };
    auto source = [&](uint32_t t, uint32_t b, int x) {
        const uint32_t p = min(t * TILE + 32 * x + 8 * wave, s.n - 1);
        const uint32_t to = min(t * TILE + 32 * x + btok, s.n - 1) - p;
        const uint64_t row = s.k + p;
        auto from = [&](const void* base, uint64_t stride, uint64_t at) {
            return __builtin_amdgcn_make_buffer_rsrc(
                static_cast<uint8_t*>(const_cast<void*>(base)) + 2 * (row * stride + at), 0,
                0xffffffffu, 0x00020000);
        };
        return Source{from(a.k, a.ks, h * a.kh), from(a.v, a.vs, h * a.vh),
                      from(a.rotary, a.rs, 0), to * (uint32_t)(2 * a.ks) + bput * 16,
                      to * (uint32_t)(2 * a.vs) + bput * 16, to * (uint32_t)(2 * a.rs) + bput * 16,
                      reinterpret_cast<u32x4*>(smem + b * kBuffer + x * 4096 + wave * 1024)};
    };
    constexpr int kPieces = KG + VG;
    auto bring = [&](const Source& f, int c) {
        if (c >= KG) {
            if (FULL || (c - KG) * 8 + bput < a.Dv / 8)
                load_lds16(f.v, f.dst + c * (kGroup / 16), f.vf, (c - KG) * 128);
        } else if ((uint32_t)c < own) {
            if (FULL || c * 8 + bput < a.Dn / 8)
                load_lds16(f.k, f.dst + c * (kGroup / 16), f.kf, c * 128);
        } else if ((uint32_t)c == own && (FULL || bput < a.R / 8)) {
            load_lds16(f.r, f.dst + c * (kGroup / 16), f.rf, 0);
        }
    };

    u32x4 qf[KG * 4];
    {
        const uint8_t* q = static_cast<const uint8_t*>(a.q) +
                           2 * ((uint64_t)(s.q + query) * a.qs + (uint64_t)h * (a.Dn + a.R));
#pragma unroll
        for (int c = 0; c < KG; ++c)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const bool mine = (uint32_t)c < own;
                const uint32_t d = (mine ? c * 64 : (c - own) * 64) + y * 16 + g * 8;
                const bool in = FULL || d < (mine ? a.Dn : a.R);
                const u32x4 z = *reinterpret_cast<const u32x4*>(
                    q + (in ? 2 * (mine ? d : a.Dn + d) : 0));
                qf[c * 4 + y] = z & (in ? 0xffffffffu : 0u);
            }
    }
    Acc o[OT];
#pragma unroll
    for (int x = 0; x < OT; ++x) o[x] = Acc{};
    float m = -3.4028235e38f, l = 0.0f;
    const int32_t sees = sees_of(query);

    // Tile t in buffer b; the next one's loads (the last one's again) to the other.
    auto tile = [&](uint32_t t, uint32_t b) {
        const lds_byte* kb = lds + b * kBuffer;
        Source next[ST];
#pragma unroll
        for (int x = 0; x < ST; ++x) next[x] = source(min(t + 1, tiles - 1), b ^ 1, x);
        Acc sc[ST];
#pragma unroll
        for (int x = 0; x < ST; ++x) sc[x] = Acc{};
        // Operands are read a few products ahead: LDS takes some 200 cycles, four waves
        // at once, a product 32.
        constexpr int NK = KG * 4 * ST, kAhead = 8;
        u32x4 kf[kAhead];
        auto keys = [&](int i) {
            const int y = i / ST, x = i % ST;
            kf[i % kAhead] = lds16(kb + y / 4 * kGroup + x * 4096 + (kat0 ^ y % 4 * 32));
        };
#pragma unroll
        for (int i = 0; i < kAhead - 1; ++i) keys(i);
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            if (i + kAhead - 1 < NK) keys(i + kAhead - 1);
            if (i % 2 == 0 && i / 2 < ST * kPieces) bring(next[i / 2 % ST], i / 2 / ST);
            __builtin_amdgcn_sched_barrier(0);
            sc[i % ST] = M::run(kf[i % kAhead], qf[i / ST], sc[i % ST]);
            __builtin_amdgcn_sched_barrier(0);
        }
        static_assert(2 * ST * kPieces <= NK + 1, "pieces within the products");
        // The first values are on their way while weights are formed.
        constexpr int NF = ST * OT * 2;
        u32x4 vf[kAhead];
        auto values = [&](int i) {  // i: 32 keys, 32 columns, 16 of the keys
            const int x = i / (2 * OT), y = i / 2 % OT, z = i % 2;
            const lds_byte* vb = kb + (KG + y / 2) * kGroup + x * 4096 + z * 2048;
            const uint32_t c = vat0 ^ y % 2 * 64;
            const uint2 v0 = lds_transposed(vb + c), v1 = lds_transposed(vb + 1024 + (c ^ 16));
            vf[i % kAhead] = u32x4{v0.x, v0.y, v1.x, v1.y};
        };
#pragma unroll
        for (int i = 0; i < kAhead - 1; ++i) values(i);
        if ((int32_t)((t + 1) * TILE) > least) {
            // Past what the query sees.
#pragma unroll
            for (int x = 0; x < ST; ++x)
#pragma unroll
                for (int y = 0; y < 16; ++y)
                    if ((int32_t)(t * TILE + 32 * x + 8 * (y / 4) + 4 * g + y % 4) >= sees)
                        sc[x][y] = -__builtin_inff();
        }
        float top = sc[0][0];
#pragma unroll
        for (int x = 0; x < ST; ++x)
#pragma unroll
            for (int y = 0; y < 16; ++y) top = fmaxf(top, sc[x][y]);
        top = across<32>(top, [](float u, float v) { return fmaxf(u, v); }) * a.rate;
        if (__any(Weights<DT>::over(top, m))) {
            const float up = Weights<DT>::reference(top, m);
            const float keep = __builtin_amdgcn_exp2f(m - up);
            m = up;
            l *= keep;
            scale_tiles<false, 0, OT>(o, keep);
        }
        uint32_t p[ST][8];
        float sum = 0.0f;
#pragma unroll
        for (int x = 0; x < ST; ++x)
#pragma unroll
            for (int y = 0; y < 16; y += 2) {
                const float u = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x][y], a.rate, -m));
                const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x][y + 1], a.rate, -m));
                sum += u + v;
                p[x][y / 2] = pack2<DT>(u, v);
            }
        l += sum;
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            if (i + kAhead - 1 < NF) values(i + kAhead - 1);
            __builtin_amdgcn_sched_barrier(0);
            const int x = i / (2 * OT), y = i / 2 % OT, z = i % 2;
            o[y] = M::run(vf[i % kAhead],
                          u32x4{p[x][4 * z], p[x][4 * z + 1], p[x][4 * z + 2], p[x][4 * z + 3]},
                          o[y]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if (tiles) {
#pragma unroll
        for (int x = 0; x < ST; ++x) {
            const Source f = source(0, 0, x);
#pragma unroll
            for (int c = 0; c < kPieces; ++c) bring(f, c);
        }
        for (uint32_t t = 0; t < tiles; ++t) {
            wait_loads<0>();
            barrier();
            tile(t, t & 1);
        }
        wait_loads<0>();
    }
    l = across<32>(l, [](float u, float v) { return u + v; });
    const bool live = w0 + col < s.m;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const uint64_t row = s.q + query;
    uint16_t* out = static_cast<uint16_t*>(a.out) + row * a.os + (uint64_t)h * a.Dv;
    float check = l * 0.0f;  // NaN once something is not finite
#pragma unroll
    for (int y = 0; y < OT; ++y)
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            const uint32_t d = y * 32 + 8 * z + 4 * g;
            const float4 v{o[y][4 * z] * inv, o[y][4 * z + 1] * inv, o[y][4 * z + 2] * inv,
                           o[y][4 * z + 3] * inv};
            if (FULL || d < a.Dv) {
                check = __builtin_fmaf(v.x, 0.0f, check);
                check = __builtin_fmaf(v.y, 0.0f, check);
                check = __builtin_fmaf(v.z, 0.0f, check);
                check = __builtin_fmaf(v.w, 0.0f, check);
                if (live) *reinterpret_cast<uint2*>(out + d) = outputs4<DT>(v);
            }
        }
    if (live && (!(check == 0.0f) || no_softmax<DT>(sees, l, m))) latch(a.status, K3X_ERR_INVALID_MXFP4);
    if (a.lse && live && g == 0)
        a.lse[row * a.H + h] = l > 0.0f ? (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f
                                        : -__builtin_inff();
}

// A call of no queries: its offsets are looked at all the same.
__global__ __launch_bounds__(kThreads) void prompt_check_kernel(PromptArgs a) {
    bool bad = false;
    for (uint32_t n = threadIdx.x; n < a.N; n += kThreads) {
        Ranges r;
        bad |= !ranges_of(a, n, &r);
    }
    if (bad) latch(a.status, K3X_ERR_INVALID_STATE);
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

template <uint32_t DT>
int launch(k3x_hip_ctx* ctx, const PromptArgs& a) {
    const dim3 grid(a.blocks * a.H), block(kThreads);
    if (a.Dn == 128 && a.R == 64 && a.Dv == 128)
        hipLaunchKernelGGL((mla_prompt_kernel<DT, 192, 128, 64, 2>), grid, block, 0, ctx->stream, a);
    else if (a.Dn == 128 && a.R == 0 && a.Dv == 128)
        hipLaunchKernelGGL((mla_prompt_kernel<DT, 128, 128, 64, 2>), grid, block, 0, ctx->stream, a);
    else
        hipLaunchKernelGGL((mla_prompt_kernel<DT, 192, 128, 32, 0>), grid, block, 0, ctx->stream, a);
    return launched(ctx, 1);
}

}  // namespace

extern "C" {

int k3x_hip_mla_prompt(k3x_hip_ctx* ctx, const k3x_hip_mla_prompt_params* p, const void* q,
                       const void* k, const void* v, const void* rotary, const uint32_t* offsets,
                       const uint32_t* key_offsets, void* out, float* lse) {
    if (!ctx || !p || !prompt_ok(p) || (p->tokens && (!q || !out)) ||
        (p->keys && (!k || !v || (p->rotary && !rotary))))
        return K3X_ERR_INVALID_EXTENT;
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(rotary, 16) ||
        !aligned(out, 16) || !aligned(offsets, 4) || !aligned(key_offsets, 4) || !aligned(lse, 4))
        return K3X_ERR_INVALID_EXTENT;
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
    if (a.S <= 1) a.ks = a.vs = a.rs = 0;  // no row lies behind another
    a.os = p->out_stride ? p->out_stride : (uint64_t)a.H * a.Dv;
    a.rate = p->scale * 1.4426950408889634f;
    a.status = ctx->status;
    // Blocks of all sequences at most, each with one that is not full; the threads of a
    // launch, and eight rows apart within 32 bits.
    a.blocks = a.T / kRows + std::min(a.N, a.T);
    const uint32_t longest = p->longest ? p->longest : a.T / a.N;
    a.flip = longest > a.T / 2 && a.T / kRows * a.H <= 512;
    if ((uint64_t)a.blocks * a.H * kThreads >= (1ull << 32) ||
        a.ks > (1u << 27) || a.vs > (1u << 27) || a.rs > (1u << 27))
        return K3X_ERR_INVALID_EXTENT;
    if (hipSetDevice(ctx->device) != hipSuccess) return K3X_ERR_BACKEND_UNAVAILABLE;
    if (!a.T) {
        hipLaunchKernelGGL(prompt_check_kernel, dim3(1), dim3(kThreads), 0, ctx->stream, a);
        return launched(ctx, 1);
    }
    return p->dtype == K3X_DTYPE_F16 ? launch<K3X_DTYPE_F16>(ctx, a)
                                     : launch<K3X_DTYPE_BF16>(ctx, a);
}

}  // extern "C"
