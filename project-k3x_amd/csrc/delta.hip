// delta.hip -- the gated delta rule (the recurrence of K3's linear attention
// layers) over ragged sequences with their states in HBM.
//
//   S = exp(g) S,  u = beta (v - S^T k),  S = S + k u^T,  o = scale S^T q
//
// for each value head, S [K][V] in fp32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <type_traits>

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
    const uint32_t* status;   // set: nothing is done
    uint32_t* errors;         // the call's own: status, or apart from it (report_kernel)
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

__device__ inline float exp_decay(float g) {
    return __builtin_amdgcn_exp2f(g * 1.44269504088896341f);
}

// Registers exchanged between rows of 16 lanes, or halves of the wave: a gets
// [x row 0, y row 0, x row 2, y row 2] and b the odd rows (or a the lower
// halves, b the upper ones).
__device__ inline void swap_rows(float x, float y, float* a, float* b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false,
                                                    false);
    *a = __uint_as_float(r[0]);
    *b = __uint_as_float(r[1]);
}
__device__ inline void swap_halves(float x, float y, float* a, float* b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false,
                                                    false);
    *a = __uint_as_float(r[0]);
    *b = __uint_as_float(r[1]);
}
// x summed over both halves in the lower one and y in the upper one; the same
// with even and odd rows.
__device__ inline float fold_halves(float x, float y) {
    float a, b;
    swap_halves(x, y, &a, &b);
    return a + b;
}
__device__ inline float fold_rows(float x, float y) {
    float a, b;
    swap_rows(x, y, &a, &b);
    return a + b;
}

template <int Ctrl>
__device__ inline float dpp(float x, float old = 0.0f) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(x), Ctrl,
                                                      0xf, 0xf, false));
}

// x of lane i of the lane's four.
__device__ inline float of_four(float x, int i) {
    const int v = __float_as_int(x);
    return __int_as_float(i == 0   ? __builtin_amdgcn_update_dpp(0, v, 0x00, 0xf, 0xf, true)
                          : i == 1 ? __builtin_amdgcn_update_dpp(0, v, 0x55, 0xf, 0xf, true)
                          : i == 2 ? __builtin_amdgcn_update_dpp(0, v, 0xaa, 0xf, 0xf, true)
                                   : __builtin_amdgcn_update_dpp(0, v, 0xff, 0xf, 0xf, true));
}

// Four elements as they lie.
template <typename E>
using Vec4 = E __attribute__((ext_vector_type(4)));

// Four elements from c on of a row of n; those past it are some others of the
// row.  vec (n a multiple of 4, the row aligned to four): one load.  Nothing
// here branches by lane, so that many loads are in flight at once.
template <typename E>
__device__ inline Vec4<E> load4(const E* row, uint32_t c, uint32_t n, bool vec) {
    if (vec) return *reinterpret_cast<const Vec4<E>*>(row + min(c, n - 4));
    Vec4<E> y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = row[min(c + j, n - 1)];
    return y;
}

// Token by token.  A wave holds 16 columns of one head's state: lane l has
// columns 4 (l % 4) .. + 3 and the R rows from R (l / 4), all in registers.
// The two products over the rows, S^T k and S^T q, are taken of the decayed
// state before its update (S_new^T q = S^T q + (k . q) u) and of q and k as
// they are (norms scale the sums), so that a token is one pass over the
// registers for all of its sums, one for the update, and one round of sums
// over the 16 row groups, in which each exchange folds two sums into one
// register.  The next token's rows are loaded meanwhile.  A workgroup's waves
// are neighbours in the columns of one head and share nothing else.
//
// One token a sequence is the state's read and write: 64 sequences of 32 heads
// of 128 x 128 take 48 us, 5.6 TB/s.  More tokens are bound by the vector
// instructions of a token and the sums' chain: 16 tokens a sequence (8 sequences,
// limits) 24 us, 1.2 us a token.
constexpr int kStepWaves = 4;
constexpr uint32_t kStepCols = 16 * kStepWaves;

// vec: bit 0, q, k and gate by several elements (of the calls above 48 and 24 us;
// by one 55 and 33); bit 1, v (by one 49 and 26); bit 2, states.
template <uint32_t DT, int R, uint32_t GATE>
__global__ __launch_bounds__(64 * kStepWaves) void delta_step_kernel(DeltaArgs a, uint32_t vec) {
    typedef typename Elem<DT>::type E;
    const uint32_t blocks = (a.V + kStepCols - 1) / kStepCols;
    const uint32_t cb = blockIdx.x % blocks, h = blockIdx.x / blocks % a.H;
    const uint32_t n = blockIdx.x / blocks / a.H;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t status = *(volatile const uint32_t*)a.status;  // with the offsets, not after
    Sequence sq;
    uint32_t bad = find_sequence(a, n, &sq);
    if (!bad && slot_taken(a, n, sq.slot)) bad = K3X_ERR_INVALID_STATE;
    if (bad) {
        if (threadIdx.x == 0) latch(a.errors, bad);
        return;
    }
    // From here on the waves of the workgroup do not wait for one another.
    if (status) return;
    const uint32_t c0 = cb * kStepCols + wave * 16 + 4 * (lane % 4), r0 = R * (lane / 4);
    if (cb * kStepCols + wave * 16 >= a.V) return;
    const uint32_t hk = h / (a.H / a.Hk);
    const size_t base = ((size_t)sq.slot * a.H + h) * a.K * a.V;
    f32x4 S[R] = {};
    if (a.state_in) {
#pragma unroll
        for (int i = 0; i < R; ++i)
            S[i] = load4(a.state_in + base + (size_t)min(r0 + i, a.K - 1) * a.V, c0, a.V, vec & 4);
    }
    // Four lanes share their rows' gates, a quarter each.
    constexpr int kGates = R / 4;
    const uint32_t g0 = r0 + kGates * (lane % 4);
    struct Row {
        Vec4<E> q[R / 4], k[R / 4], v;
        float gate[GATE == K3X_GATE_CHANNEL ? kGates : 1];
        float beta;
    } next, now;
    auto fetch = [&](uint32_t t) {
        const size_t row = (size_t)sq.begin + t;
        const E* q = static_cast<const E*>(a.q) + row * a.qs + (size_t)hk * a.K;
        const E* k = static_cast<const E*>(a.k) + row * a.ks + (size_t)hk * a.K;
        const float* g = a.gate + (row * a.H + h) * (GATE == K3X_GATE_CHANNEL ? a.K : 1);
#pragma unroll
        for (int i = 0; i < R / 4; ++i) {
            next.q[i] = load4(q, r0 + 4 * i, a.K, vec & 1);
            next.k[i] = load4(k, r0 + 4 * i, a.K, vec & 1);
        }
        if constexpr (GATE == K3X_GATE_CHANNEL) {
            typedef float Gates __attribute__((ext_vector_type(kGates)));
            if (kGates > 1 && (vec & 1)) {
                const Gates x = *reinterpret_cast<const Gates*>(g + min(g0, a.K - kGates));
#pragma unroll
                for (int i = 0; i < kGates; ++i) next.gate[i] = x[i];
            } else {
#pragma unroll
                for (int i = 0; i < kGates; ++i) next.gate[i] = g[min(g0 + i, a.K - 1)];
            }
        }
        if (GATE == K3X_GATE_HEAD) next.gate[0] = g[0];
        next.v = load4(static_cast<const E*>(a.v) + row * a.vs + (size_t)h * a.V, c0, a.V, vec & 2);
        next.beta = a.beta[row * a.H + h];
    };
    if (sq.len) fetch(0);
    // Rows past the head's end hold another's: they are 0, and stay so.
    if (r0 + R > a.K) {
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (r0 + i >= a.K) S[i] = f32x4{};
    }
    float z = 0.0f;  // NaN once an input is not finite
    float longest = 0.0f;  // of the squared norms, by rows of lanes
    bool wrong = false;
    for (uint32_t t = 0; t < sq.len; ++t) {
        now = next;
        fetch(min(t + 1, sq.len - 1));
        float q[R], k[R], v[4], d[kGates];
        float qq = 0.0f, kk = 0.0f, kq = 0.0f;
        f32x4 p = {}, o = {};
#pragma unroll
        for (int i = 0; i < R; ++i) {
            q[i] = Elem<DT>::load(now.q[i / 4][i % 4]);
            k[i] = Elem<DT>::load(now.k[i / 4][i % 4]);
        }
        if (r0 + R > a.K) {
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (r0 + i >= a.K) q[i] = k[i] = 0.0f;
        }
        z = __builtin_fmaf(now.beta, 0.0f, z);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = Elem<DT>::load(now.v[j]);
            z = __builtin_fmaf(v[j], 0.0f, z);
        }
        if (GATE != K3X_GATE_NONE) {
#pragma unroll
            for (int i = 0; i < (GATE == K3X_GATE_CHANNEL ? kGates : 1); ++i) {
                wrong |= !(now.gate[i] <= 0.0f);
                d[i] = exp_decay(now.gate[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            z = __builtin_fmaf(q[i], 0.0f, z);
            z = __builtin_fmaf(k[i], 0.0f, z);
            const float decay = GATE == K3X_GATE_CHANNEL ? of_four(d[i % kGates], i / kGates) : d[0];
            qq = __builtin_fmaf(q[i], q[i], qq);
            kk = __builtin_fmaf(k[i], k[i], kk);
            kq = __builtin_fmaf(k[i], q[i], kq);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (GATE != K3X_GATE_NONE) S[i][j] *= decay;
                p[j] = __builtin_fmaf(S[i][j], k[i], p[j]);
                o[j] = __builtin_fmaf(S[i][j], q[i], o[j]);
            }
        }
        // Rows of 16 lanes then hold: x the sums of p0, p1, o0, o1, y those of
        // p2, p3, o2, o3, w those of kk, kq, qq, kq.
        float x = fold_rows(fold_halves(p[0], o[0]), fold_halves(p[1], o[1]));
        float y = fold_rows(fold_halves(p[2], o[2]), fold_halves(p[3], o[3]));
        float w = fold_rows(fold_halves(kk, qq), fold_halves(kq, kq));
        x += dpp<0x124>(x);  // row_ror:4
        y += dpp<0x124>(y);
        w += dpp<0x124>(w);
        x += dpp<0x128>(x);  // row_ror:8
        y += dpp<0x128>(y);
        w += dpp<0x128>(w);
        longest = fmaxf(longest, w);
        const float sk = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), 0));
        const float skq = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), 16));
        const float sq2 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), 32));
        const float rk = a.eps > 0.0f ? rsqrtf(sk + a.eps) : 1.0f;
        const float rq = a.eps > 0.0f ? a.scale * rsqrtf(sq2 + a.eps) : a.scale;
        const bool odd = lane & 16;
        // u of rows 0 and 1, then of every row.
        float ux = now.beta * __builtin_fmaf(-rk, x, odd ? v[1] : v[0]);
        float uy = now.beta * __builtin_fmaf(-rk, y, odd ? v[3] : v[2]);
        z = __builtin_fmaf(ux, 0.0f, z);  // of a state that is not finite, too
        z = __builtin_fmaf(uy, 0.0f, z);
        float any, u[4];
        swap_halves(ux, ux, &ux, &any);
        swap_halves(uy, uy, &uy, &any);
        const float kqr = rk * skq;
        const float ox = rq * __builtin_fmaf(kqr, ux, x), oy = rq * __builtin_fmaf(kqr, uy, y);
        swap_rows(ux, ux, &u[0], &u[1]);
        swap_rows(uy, uy, &u[2], &u[3]);
        if ((lane & 44) == 32) {  // rows 2 and 3, one lane a column group
            E* out = static_cast<E*>(a.out) + ((size_t)sq.begin + t) * a.os + (size_t)h * a.V;
            const uint32_t c = c0 + (odd ? 1 : 0);
            if (c < a.V) out[c] = Elem<DT>::store(ox);
            if (c + 2 < a.V) out[c + 2] = Elem<DT>::store(oy);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] *= rk;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = __builtin_fmaf(k[i], u[j], S[i][j]);
    }
    if (a.eps > 0.0f) wrong |= longest == __builtin_inff();
    if (wrong || z != z) latch(a.errors, K3X_ERR_INVALID_MXFP4);
    if (!a.state_out || (!sq.len && a.state_in == a.state_out)) return;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (r0 + i >= a.K) continue;
        float* row = a.state_out + base + (size_t)(r0 + i) * a.V;
        if (vec & 4) {
            if (c0 < a.V) *reinterpret_cast<f32x4*>(row + c0) = S[i];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c0 + j < a.V) row[c0 + j] = S[i][j];
        }
    }
}

template <uint32_t DT, int R>
void launch_step(const DeltaArgs& a, uint32_t gate, uint32_t vec, hipStream_t stream) {
    const dim3 b(64 * kStepWaves), grid(a.N * a.H * ((a.V + kStepCols - 1) / kStepCols));
    if (gate == K3X_GATE_NONE)
        hipLaunchKernelGGL((delta_step_kernel<DT, R, K3X_GATE_NONE>), grid, b, 0, stream, a, vec);
    else if (gate == K3X_GATE_HEAD)
        hipLaunchKernelGGL((delta_step_kernel<DT, R, K3X_GATE_HEAD>), grid, b, 0, stream, a, vec);
    else
        hipLaunchKernelGGL((delta_step_kernel<DT, R, K3X_GATE_CHANNEL>), grid, b, 0, stream, a,
                           vec);
}

template <uint32_t DT>
void launch_step_rows(const DeltaArgs& a, uint32_t gate, uint32_t vec, hipStream_t stream) {
    if (a.K <= 64) launch_step<DT, 4>(a, gate, vec, stream);
    else if (a.K <= 128) launch_step<DT, 8>(a, gate, vec, stream);
    else launch_step<DT, 16>(a, gate, vec, stream);
}

// ---------------------------------------------------------------------------
// Chunks of 32 tokens.  With P_i the decay from the chunk's start to token i,
// D_ij that after token j up to token i, S the state at its start and c_i k_i
// the keys (k_i their operands of size 1 at most, c_i a power of two, 1 for
// normalised keys), the chunk's writes and outputs are
//
//   L_ij = beta_i c_i c_j sum_c k_ic D_ijc k_jc   (i > j)
//   U    = c (I + L)^-1 beta (V - c (P k) S)
//   O    = scale ((P q) S + Pq U),   Pq_ij = sum_c q_ic D_ijc k_jc   (i >= j)
//   S    = P_31 S + sum_j (D_31,j k_j) U_j^T
//
// all of them products of 16 x 16 tiles on the matrix cores.  Two launches:
// delta_prep_channel_kernel or delta_prep_head_kernel makes (I + L)^-1 and Pq of
// every chunk and its keys and queries as operands, all chunks at once;
// delta_scan_kernel walks a sequence's chunks with the state in registers.  The
// operands are made once and not by each of the scan's workgroups (a head's
// columns lie in several), whose chain of chunks is what a long prompt waits for.
//
// Operands are f16 pairs hi + lo (22 bits: what is left out of a product of two
// pairs, lo lo, is 2^-22 of it), sums fp32.  f16 ends at 65504 and 2^-24, so
// keys and queries are scaled to 64 at most, rows of the inverse by a power of
// two each, and a column of the state and its values by one power of two that
// follows their size.
// ---------------------------------------------------------------------------
constexpr uint32_t kChunk = 32;
constexpr float kOperand = 64.0f;  // keys, queries and Pq are held times this

// Eight values of a lane as a vector and not an array: what the loops over them
// index stays in registers whatever is unrolled when.
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

struct Pair8 {
    f16x8 hi, lo;
};

// hi = f16(x), lo = f16(x - hi).  The factor -1 is kept from the compiler so
// that difference and rounding are one fused instruction on the packed halves.
__device__ __forceinline__ Pair8 split8(f32x8 x) {
    typedef __attribute__((ext_vector_type(2))) float f32x2;
    float minus = -1.0f;
    asm("" : "+s"(minus));
    u32x4 hi, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f32x2 v = {x[2 * j], x[2 * j + 1]};
        uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
        asm("" : "+v"(u));
        const f16x2 h = __builtin_bit_cast(f16x2, u);
        const f16x2 r = {(_Float16)__builtin_fmaf((float)h[0], minus, v[0]),
                         (_Float16)__builtin_fmaf((float)h[1], minus, v[1])};
        hi[j] = u;
        lo[j] = __builtin_bit_cast(uint32_t, r);
    }
    return Pair8{__builtin_bit_cast(f16x8, hi), __builtin_bit_cast(f16x8, lo)};
}

__device__ inline f32x4 mfma_f16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ inline f32x4 mfma_pairs(const Pair8& a, const Pair8& b, f32x4 c) {
    c = mfma_f16(a.lo, b.hi, c);
    c = mfma_f16(a.hi, b.lo, c);
    return mfma_f16(a.hi, b.hi, c);
}

// What the scan needs of one chunk of one value head.  T and Pq in the order
// of the matrix operand: lane l, element j of tile r is row 16 r + l % 16,
// column token_of(l / 16, j); the columns' order is that in which a lane holds
// the rows of a product's result, so that results feed the next product as
// they are.
struct ChunkRecord {
    f16x8 T[2][2][64];           // [tile][hi, lo]; a row times row_t is c (I + L)^-1 beta
    f16x8 P[2][2][64];           // Pq times kOperand
    float row_r[kChunk];         // of (k S) in V - c (P k) S
    float row_o[kChunk];         // of (q S) and
    float row_p[kChunk];         //   (Pq U) in O
    float row_t[kChunk];
    float row_u[kChunk];         // head gates: of U in the state's update
    float unused[3 * kChunk];
    float decay[128];            // of the state over the chunk, by channel
    float unused2[128];
};
static_assert(sizeof(ChunkRecord) == 10240, "ten loads of a wave");

// Its keys and queries as operands, times kOperand: hi and, where they need
// one, lo.  With a decay a channel they carry it (P k, P q and D_31 k, of a
// value head); with one a head they are the elements times a power of two (of a
// key head), 8 or 11 bits, which need no lo.
template <bool LO, int KB>
struct ChunkOperands {
    static constexpr int kParts = LO ? 2 : 1;
    f16x8 K[kParts][2][KB][64];    // [tile of tokens][channels by 32]
    f16x8 Q[kParts][2][KB][64];
    f16x8 Kt[kParts][2 * KB][64];  // [channels by 16][tokens]
};

__device__ inline uint32_t token_of(uint32_t q, uint32_t j) { return 4 * q + (j & 3) + 4 * (j & 4); }

// Sum and maximum over the lanes of equal lane % 16.
__device__ inline float sum_groups(float v) {
    v = fold_rows(v, v);
    return fold_halves(v, v);
}
// Of v >= 0, whose order is that of its bits.
__device__ inline float max_groups(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t x = max(r[0], r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __uint_as_float(max(h[0], h[1]));
}

__device__ inline int max_groups(int v) {
    const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    const int x = max((int)r[0], (int)r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
    return max((int)h[0], (int)h[1]);
}

// 2^-e and 2^e for the least e with |x| < 2^e (x finite), as far as both are
// numbers of fp32: what is below 2^-100 stays below 1/2, what is above 2^127
// below 2.  1 and 1 for x = 0.
__device__ inline void unit_scale(float x, float* down, float* up) {
    int e = x > 0.0f ? __builtin_amdgcn_frexp_expf(x) : 0;
    e = e < -100 ? -100 : e > 127 ? 127 : e;
    *down = __builtin_ldexpf(1.0f, -e);
    *up = __builtin_ldexpf(1.0f, e);
}

// Which sequence and chunk of it has record slot x: sequence n's chunks begin at
// slot offsets[n] / 32 + n, which leaves room for each one's last part.
__device__ inline uint32_t first_slot(const DeltaArgs& a, uint32_t n) {
    const uint32_t b = a.offsets ? a.offsets[n] : n * (a.T / a.N);
    return b / kChunk + n;
}

__device__ inline uint32_t sequence_of_slot(const DeltaArgs& a, uint32_t x) {
    uint32_t lo = 0, hi = a.N;  // first_slot(lo) <= x
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (first_slot(a, mid) <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A chunk's place: its sequence, first token and slot.
struct ChunkPlace {
    Sequence sq;
    uint32_t first;
};

__device__ inline bool find_chunk(const DeltaArgs& a, uint32_t slot, ChunkPlace* c) {
    const uint32_t n = sequence_of_slot(a, slot), slot0 = first_slot(a, n);
    if (find_sequence(a, n, &c->sq)) return false;  // latched by the scan
    if (slot < slot0 || slot - slot0 >= (c->sq.len + kChunk - 1) / kChunk) return false;
    c->first = (slot - slot0) * kChunk;
    return true;
}

// LDS written before is seen after, by the whole workgroup; loads from and
// stores to global memory stay in flight across it.
__device__ inline void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

typedef float Tile32[kChunk][36];  // rows of 16-byte alignment that spread over the banks

// T of a chunk from L (strictly lower triangular; overwritten), by one wave in
// fp32: the inverses of the two diagonal tiles by forward substitution, a
// column a lane, and -T22 L21 T11 below them.
__device__ __forceinline__ void write_inverse(Tile32& L, const float* c, const float* beta,
                                     ChunkRecord* rec) {
    const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const uint32_t half = 16 * (g & 1);
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float s = (uint32_t)i == m ? 1.0f : 0.0f;
#pragma unroll
        for (int j = 0; j < i; ++j) s = __builtin_fmaf(-L[half + i][half + j], x[j], s);
        x[i] = s;
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // not every row of L at once
    }
    wave_sync();
    if (g < 2) {
#pragma unroll
        for (int i = 0; i < 16; ++i) L[half + i][half + m] = x[i];
    }
    wave_sync();
    // Rows 4 g + i of a result are rows k = 4 g + s of the next product's right
    // operand; its left operand takes the columns in the same order.
    f32x4 y = {}, z = {};
    const f32x4 l21 = *reinterpret_cast<const f32x4*>(&L[16 + m][4 * g]);
    const f32x4 t22 = *reinterpret_cast<const f32x4*>(&L[16 + m][16 + 4 * g]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y = __builtin_amdgcn_mfma_f32_16x16x4f32(l21[i], L[4 * g + i][m], y, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        z = __builtin_amdgcn_mfma_f32_16x16x4f32(t22[i], y[i], z, 0, 0, 0);
    wave_sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        L[16 + 4 * g + i][m] = -z[i];
        L[4 * g + i][16 + m] = 0.0f;
    }
    wave_sync();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        f32x8 e;
        float most = 0.0f, down, up;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t t = token_of(g, j);
            e[j] = L[16 * r + m][t] * c[16 * r + m] * beta[t];
            most = fmaxf(most, fabsf(e[j]));
        }
        unit_scale(max_groups(most), &down, &up);
        const Pair8 p = split8(e * (down * kOperand));
        rec->T[r][0][lane] = p.hi;
        rec->T[r][1][lane] = p.lo;
        if (g == 0) rec->row_t[16 * r + m] = up / kOperand;
    }
}

__device__ __forceinline__ void write_scores(const Tile32& P, ChunkRecord* rec) {
    const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        f32x8 e;
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = P[16 * r + m][token_of(g, j)];
        const Pair8 p = split8(e);
        rec->P[r][0][lane] = p.hi;
        rec->P[r][1][lane] = p.lo;
    }
}

// Eight channels of a lane's token in the operand's order: element j of part b is
// channel 32 b + token_of(l / 16, j).  WHOLE: the head fills its parts and its
// rows are loaded by four; else elements past the head's end are 0.
template <uint32_t DT, bool WHOLE>
struct TokenPart {
    typedef typename Elem<DT>::type E;
    Vec4<E> q[2], k[2];
    __device__ __forceinline__ void load(const DeltaArgs& a, const E* qr, const E* kr, int b,
                                         uint32_t g) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t c = 32 * b + 16 * x + 4 * g;
            if constexpr (WHOLE) {
                q[x] = *reinterpret_cast<const Vec4<E>*>(qr + c);
                k[x] = *reinterpret_cast<const Vec4<E>*>(kr + c);
            } else {
                q[x] = load4(qr, c, a.K, false);
                k[x] = load4(kr, c, a.K, false);
            }
        }
    }
    __device__ __forceinline__ void values(const DeltaArgs& a, int b, uint32_t g, f32x8& x,
                                           f32x8& y) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in = WHOLE || 32 * b + token_of(g, j) < a.K;
            x[j] = in ? Elem<DT>::load(q[j / 4][j % 4]) : 0.0f;
            y[j] = in ? Elem<DT>::load(k[j / 4][j % 4]) : 0.0f;
        }
    }
};

// What a token's key and query are scaled by.
struct TokenScales {
    float qd, qu, kd, ku;  // 2^-e and 2^e of the largest element
    float qn, kn;          // 1 / norm
    // By the whole wave; latches an element, or a norm in use, that is not finite
    // (here and now: a check at the end would hold every element until then).
    template <uint32_t DT, int KB, bool WHOLE>
    __device__ __forceinline__ void find(const DeltaArgs& a, const typename Elem<DT>::type* qr,
                                         const typename Elem<DT>::type* kr, uint32_t g) {
        TokenPart<DT, WHOLE> part[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) part[b].load(a, qr, kr, b, g);
        float qm = 0.0f, km = 0.0f, qq = 0.0f, kk = 0.0f, z = 0.0f;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            __builtin_amdgcn_sched_barrier(0);  // one part's values at a time
            f32x8 x, y;
            part[b].values(a, b, g, x, y);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                z = __builtin_fmaf(x[j], 0.0f, z);
                z = __builtin_fmaf(y[j], 0.0f, z);
                qm = fmaxf(qm, fabsf(x[j]));
                km = fmaxf(km, fabsf(y[j]));
                qq = __builtin_fmaf(x[j], x[j], qq);
                kk = __builtin_fmaf(y[j], y[j], kk);
            }
        }
        qq = sum_groups(qq);
        kk = sum_groups(kk);
        if (a.eps > 0.0f) z = __builtin_fmaf(fmaxf(qq, kk), 0.0f, z);  // too long for a norm
        if (z != z) latch(a.errors, K3X_ERR_INVALID_MXFP4);
        unit_scale(max_groups(qm), &qd, &qu);
        unit_scale(max_groups(km), &kd, &ku);
        qn = 1.0f / sqrtf(qq + a.eps);
        kn = 1.0f / sqrtf(kk + a.eps);
    }
};

// A part's keys by channel, for the state's update: a wave's tokens into `tr` (a
// row a channel), and from there, once all are in, as operands.
typedef _Float16 ByChannel[32][kChunk + 8];

__device__ inline void put_by_channel(ByChannel& tr, uint32_t g, uint32_t token, const f16x8& x) {
#pragma unroll
    for (int j = 0; j < 8; ++j) tr[token_of(g, j)][token] = x[j];
}

__device__ inline f16x8 by_channel(const ByChannel& tr, uint32_t tile) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const f16x4 lo = *reinterpret_cast<const f16x4*>(&tr[16 * tile + m][4 * g]);
    const f16x4 hi = *reinterpret_cast<const f16x4*>(&tr[16 * tile + m][16 + 4 * g]);
    return f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// One chunk of one head under a decay a channel, by two waves of 16 tokens.
//
// Such a decay does not factor over (i, j) without overflow, so a tile's lower
// triangle is made level by level: pairs (i, j) whose highest differing bit is
// b have D_ij = pre_b(i) suf_b(j), the decays up to the border between i's and
// j's blocks of 2^b tokens and from there on, both at most 1.  Each level is
// one product of the whole tile, of which its own pairs are kept.  pre, suf and
// a block's total come from the level before by one exchange over the lanes of
// a row; after the last they are those of the tile.
//
// 2048 tokens of 32 heads of 128: 50 us for 66 MB read and 119 MB written, 3.7
// TB/s; one 32-channel part in registers at a time, two workgroups a SIMD pair
// (three or four do not fit without spills).
// WHOLE: K = 32 KB and rows by four elements, so that no load is guarded (rows
// off by one element: 191 us in place of 165 with the scan, on warm inputs).
template <uint32_t DT, int KB, bool WHOLE>
__global__ __launch_bounds__(128, 2) void delta_prep_channel_kernel(
    DeltaArgs a, ChunkRecord* records, ChunkOperands<true, KB>* operands) {
    typedef typename Elem<DT>::type E;
    __shared__ Tile32 Ls, Ps;
    __shared__ Pair8 cross[64];
    __shared__ float total[2][32];
    __shared__ __attribute__((aligned(16))) ByChannel tr[2];
    __shared__ float beta_s[kChunk], c_s[kChunk];
    const uint32_t h = blockIdx.x % a.H, slot = blockIdx.x / a.H;
    const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (__syncthreads_or(*(volatile const uint32_t*)a.status)) return;
    ChunkPlace place;
    if (!find_chunk(a, slot, &place)) return;
    ChunkRecord* rec = records + (size_t)slot * a.H + h;
    ChunkOperands<true, KB>* ops = operands + (size_t)slot * a.H + h;
    const uint32_t t = 16 * w + m, hk = h / (a.H / a.Hk);
    const bool live = place.first + t < place.sq.len;
    const size_t row = (size_t)place.sq.begin + place.first + (live ? t : 0);
    float z = 0.0f;  // NaN once an input is not finite
    bool wrong = false;
    const E* qr = static_cast<const E*>(a.q) + row * a.qs + (size_t)hk * a.K;
    const E* kr = static_cast<const E*>(a.k) + row * a.ks + (size_t)hk * a.K;
    const float* gr = a.gate + (row * a.H + h) * a.K;
    TokenScales rows;
    rows.find<DT, KB, WHOLE>(a, qr, kr, g);
    const float beta = live ? a.beta[row * a.H + h] : 0.0f;
    z = __builtin_fmaf(beta, 0.0f, z);
    const bool norm = a.eps > 0.0f;
    // A row past the sequence's end (read as the chunk's first) counts as 0.
    const float kmul = live ? (norm ? rows.kn : rows.kd) * kOperand : 0.0f;
    const float qmul = live ? (norm ? rows.qn : rows.qd) * kOperand : 0.0f;
    const float c_up = norm ? 1.0f : rows.ku, o_up = a.scale * (norm ? 1.0f : rows.qu);
    if (lane < 16) {
        beta_s[t] = beta;
        c_s[t] = c_up;
        rec->row_r[t] = c_up / (kOperand * kOperand);
        rec->row_o[t] = o_up / (kOperand * kOperand);
        rec->row_p[t] = o_up / kOperand;
    }
    f32x4 accL[4] = {}, accP[4] = {}, l21 = {}, p21 = {};
    float diag = 0.0f;
    // The parts one after another, the next one's loads on their way (the first
    // pass has them in the cache).
    TokenPart<DT, WHOLE> next;
    next.load(a, qr, kr, 0, g);
    auto gates = [&](uint32_t c) {
        if constexpr (WHOLE) return *reinterpret_cast<const f32x4*>(gr + c);
        else return load4(gr, c, a.K, false);
    };
    f32x4 gate[2] = {gates(4 * g), gates(16 + 4 * g)};
#pragma unroll 1
    for (int b = 0; b < KB; ++b) {
        f32x8 kk, qq, pre, suf, tot;
        next.values(a, b, g, qq, kk);
        qq *= qmul;
        kk *= kmul;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t c = 32 * b + token_of(g, j);
            const float e = live && (WHOLE || c < a.K) ? gate[j / 4][j % 4] : 0.0f;
            wrong |= !(e <= 0.0f);
            tot[j] = exp_decay(e);
            suf[j] = 1.0f;
            diag = __builtin_fmaf(kk[j], qq[j], diag);
        }
        pre = tot;
        if (b + 1 < KB) {
            next.load(a, qr, kr, b + 1, g);
            gate[0] = gates(32 * (b + 1) + 4 * g);
            gate[1] = gates(32 * (b + 1) + 16 + 4 * g);
        }
#pragma unroll
        for (int level = 0; level < 4; ++level) {
            const bool bit = m >> level & 1;
            const f32x8 f = bit ? pre : suf;
            const Pair8 kp = split8(kk * f), qp = split8(qq * f);
            accL[level] = mfma_pairs(kp, kp, accL[level]);
            accP[level] = mfma_pairs(qp, kp, accP[level]);
            // The other block's total: from across bit `level` (a total is the
            // same on every lane of its block, so that mirrors do).
            f32x8 o;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                o[j] = level == 0   ? dpp<0xb1>(tot[j])
                       : level == 1 ? dpp<0x4e>(tot[j])
                       : level == 2 ? dpp<0x141>(tot[j])
                                    : dpp<0x140>(tot[j]);
            const f32x8 one = 1.0f;
            pre *= bit ? o : one;
            suf *= bit ? one : o;
            tot *= o;
        }
        // Tile 0's keys up to the border of the tiles, for tile 1.
        suf *= kk;
        if (w == 0) cross[lane] = split8(suf);
        if (m == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) total[w][token_of(g, j)] = tot[j];
        }
        lds_barrier();
        f32x8 other;
#pragma unroll
        for (int j = 0; j < 8; ++j) other[j] = total[1 - w][token_of(g, j)];
        kk *= pre;
        qq *= pre;
        Pair8 kp = split8(kk), qp = split8(qq);
        if (w == 1) {
            const Pair8 before = cross[lane];
            l21 = mfma_pairs(kp, before, l21);
            p21 = mfma_pairs(qp, before, p21);
            kp = split8(kk * other);
            qp = split8(qq * other);
        } else {
            suf *= other;
        }
        ops->K[0][w][b][lane] = kp.hi;
        ops->K[1][w][b][lane] = kp.lo;
        ops->Q[0][w][b][lane] = qp.hi;
        ops->Q[1][w][b][lane] = qp.lo;
        const Pair8 sp = split8(suf);
        put_by_channel(tr[0], g, t, sp.hi);
        put_by_channel(tr[1], g, t, sp.lo);
        if (w == 0 && m == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) rec->decay[32 * b + token_of(g, j)] = tot[j] * other[j];
        }
        lds_barrier();
        ops->Kt[0][2 * b + w][lane] = by_channel(tr[0], w);
        ops->Kt[1][2 * b + w][lane] = by_channel(tr[1], w);
    }
    diag = sum_groups(diag);
    if (wrong || z != z) latch(a.errors, K3X_ERR_INVALID_MXFP4);
    // Row 4 g + i and column m of the wave's tile on the diagonal.
    const float un = 1.0f / (kOperand * kOperand);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t r = 4 * g + i, ti = 16 * w + r, differ = r ^ m;
        float l = accL[0][i], p = accP[0][i];
#pragma unroll
        for (int level = 1; level < 4; ++level)
            if (differ >= 1u << level) {
                l = accL[level][i];
                p = accP[level][i];
            }
        Ls[ti][t] = r > m ? l * un * beta_s[ti] * c_s[ti] * c_s[t] : 0.0f;
        Ps[ti][t] = (r > m ? p : r == m ? diag : 0.0f) / kOperand;
        if (w == 0) {
            Ps[r][16 + m] = 0.0f;
        } else {
            Ls[ti][m] = l21[i] * un * beta_s[ti] * c_s[ti] * c_s[m];
            Ps[ti][m] = p21[i] / kOperand;
        }
    }
    lds_barrier();
    if (w == 0) write_inverse(Ls, c_s, beta_s, rec);
    else write_scores(Ps, rec);
}

// One chunk of one key head under a decay a value head, by two waves of 16
// tokens: the products of keys and queries once, and for each value head (a
// wave every other one) its factors exp(G_i - G_j), G the log decays summed in
// double.  8192 tokens of 16 key and 32 value heads of 128: 77 us for 67 MB read
// and 185 MB written, 3.3 TB/s.  WHOLE as above (242 in place of 203 us).
template <uint32_t DT, int KB, bool WHOLE>
__global__ __launch_bounds__(128, 2) void delta_prep_head_kernel(
    DeltaArgs a, ChunkRecord* records, ChunkOperands<DT == K3X_DTYPE_F32, KB>* operands) {
    typedef typename Elem<DT>::type E;
    constexpr bool LO = DT == K3X_DTYPE_F32;
    __shared__ Tile32 Gk, Gq, work[2];
    __shared__ Pair8 cross[64];
    __shared__ __attribute__((aligned(16))) ByChannel tr[LO ? 2 : 1];
    __shared__ float c_s[kChunk], rk_s[kChunk], rq_s[kChunk], o_s[kChunk], beta_s[2][kChunk];
    __shared__ double G_s[2][kChunk];
    const uint32_t hk = blockIdx.x % a.Hk, slot = blockIdx.x / a.Hk, per = a.H / a.Hk;
    const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (__syncthreads_or(*(volatile const uint32_t*)a.status)) return;
    ChunkPlace place;
    if (!find_chunk(a, slot, &place)) return;
    ChunkOperands<LO, KB>* ops = operands + (size_t)slot * a.Hk + hk;
    const uint32_t t = 16 * w + m;
    const bool live = place.first + t < place.sq.len;
    const size_t row0 = (size_t)place.sq.begin + place.first, row = row0 + (live ? t : 0);
    float z = 0.0f;  // NaN once an input is not finite
    bool wrong = false;
    const E* qr = static_cast<const E*>(a.q) + row * a.qs + (size_t)hk * a.K;
    const E* kr = static_cast<const E*>(a.k) + row * a.ks + (size_t)hk * a.K;
    TokenScales rows;
    rows.find<DT, KB, WHOLE>(a, qr, kr, g);
    const bool norm = a.eps > 0.0f;
    if (lane < 16) {
        c_s[t] = norm ? 1.0f : rows.ku;
        rk_s[t] = norm ? rows.kn * rows.ku : 1.0f;
        rq_s[t] = norm ? rows.qn * rows.qu : 1.0f;
        o_s[t] = a.scale * (norm ? 1.0f : rows.qu);
    }
    const float qmul = live ? rows.qd * kOperand : 0.0f, kmul = live ? rows.kd * kOperand : 0.0f;
    f32x4 accK = {}, accQ = {}, k21 = {}, q21 = {};
    float diag = 0.0f;
    // The parts one after another, the next one's loads on their way (the first
    // pass has them in the cache).
    TokenPart<DT, WHOLE> next;
    next.load(a, qr, kr, 0, g);
#pragma unroll 1
    for (int b = 0; b < KB; ++b) {
        f32x8 kk, qq;
        next.values(a, b, g, qq, kk);
        if (b + 1 < KB) next.load(a, qr, kr, b + 1, g);
        qq *= qmul;
        kk *= kmul;
#pragma unroll
        for (int j = 0; j < 8; ++j) diag = __builtin_fmaf(kk[j], qq[j], diag);
        const Pair8 kp = split8(kk), qp = split8(qq);
        accK = mfma_pairs(kp, kp, accK);
        accQ = mfma_pairs(qp, kp, accQ);
        if (w == 0) cross[lane] = kp;
        ops->K[0][w][b][lane] = kp.hi;
        ops->Q[0][w][b][lane] = qp.hi;
        put_by_channel(tr[0], g, t, kp.hi);
        if (LO) {
            ops->K[LO ? 1 : 0][w][b][lane] = kp.lo;
            ops->Q[LO ? 1 : 0][w][b][lane] = qp.lo;
            put_by_channel(tr[LO ? 1 : 0], g, t, kp.lo);
        }
        lds_barrier();
        if (w == 1) {
            const Pair8 before = cross[lane];
            k21 = mfma_pairs(kp, before, k21);
            q21 = mfma_pairs(qp, before, q21);
        }
#pragma unroll
        for (int y = 0; y < (LO ? 2 : 1); ++y) ops->Kt[y][2 * b + w][lane] = by_channel(tr[y], w);
        lds_barrier();
    }
    diag = sum_groups(diag);
    const float un = 1.0f / (kOperand * kOperand);
    // Products of the normalised rows: row 4 g + i, column m.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t r = 4 * g + i, ti = 16 * w + r;
        Gk[ti][t] = accK[i] * un * rk_s[ti] * rk_s[t];
        Gq[ti][t] = (r == m ? diag : accQ[i]) * un * rq_s[ti] * rk_s[t];
        if (w == 1) {
            Gk[ti][m] = k21[i] * un * rk_s[ti] * rk_s[m];
            Gq[ti][m] = q21[i] * un * rq_s[ti] * rk_s[m];
        }
    }
    lds_barrier();
    for (uint32_t v = w; v < per; v += 2) {
        const uint32_t h = hk * per + v;
        ChunkRecord* rec = records + (size_t)slot * a.H + h;
        const uint32_t tok = lane & 31;
        const bool in = place.first + tok < place.sq.len;
        const size_t at = (row0 + (in ? tok : 0)) * a.H + h;
        const float beta = in ? a.beta[at] : 0.0f, gate = in && a.gate ? a.gate[at] : 0.0f;
        z = __builtin_fmaf(beta, 0.0f, z);
        wrong |= !(gate <= 0.0f);
        double G = (double)fmaxf(gate, -128.0f);  // exp of less is 0 in fp32
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const double o = __shfl_up(G, d, 32);
            if (tok >= (uint32_t)d) G += o;
        }
        const double all = __shfl(G, 31, 32);
        wave_sync();  // the head before is done with its LDS
        if (lane < 32) {
            beta_s[w][tok] = beta;
            G_s[w][tok] = G;
            const float p = exp_decay((float)G), s = exp_decay((float)(all - G));
            rec->row_r[tok] = c_s[tok] * un * p * rk_s[tok];
            rec->row_o[tok] = o_s[tok] * un * p * rq_s[tok];
            rec->row_p[tok] = o_s[tok] / kOperand;
            rec->row_u[tok] = s * rk_s[tok];
        }
        const float whole = exp_decay((float)all);
        rec->decay[lane] = whole;
        rec->decay[64 + lane] = whole;
        wave_sync();
        auto factor = [&](uint32_t i, uint32_t j) {
            return i >= j ? exp_decay((float)(G_s[w][i] - G_s[w][j])) : 0.0f;
        };
        // Pq first, through the same tile.
        Tile32& tile = work[w];
        float f[3][4];
#pragma unroll
        for (int x = 0; x < 3; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t ri = 4 * g + i + (x ? 16 : 0), cj = m + (x == 2 ? 16 : 0);
                f[x][i] = factor(ri, cj);
                tile[ri][cj] = Gq[ri][cj] * f[x][i] * kOperand;
                if (x == 0) tile[ri][16 + m] = 0.0f;
            }
        wave_sync();
        write_scores(tile, rec);
        wave_sync();
#pragma unroll
        for (int x = 0; x < 3; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t ri = 4 * g + i + (x ? 16 : 0), cj = m + (x == 2 ? 16 : 0);
                tile[ri][cj] = ri > cj ? Gk[ri][cj] * f[x][i] * beta_s[w][ri] * c_s[ri] * c_s[cj]
                                       : 0.0f;
            }
        wave_sync();
        write_inverse(tile, c_s, beta_s[w], rec);
    }
    if (wrong || z != z) latch(a.errors, K3X_ERR_INVALID_MXFP4);
}

// Rows of a tensor from `base` on as a buffer: 32 at most, of `width` bytes
// every `stride` bytes.  Reads past the last row give 0 and writes are dropped,
// so that a sequence's end needs no care; kOutside is past every row.
constexpr uint32_t kOutside = 0xf0000000u;

__device__ inline __amdgpu_buffer_rsrc_t rows_buffer(const void* base, uint32_t rows,
                                                     uint32_t stride, uint32_t width) {
    // The extent stays scalar (the borrow of rows - 1 would take it to the
    // vector unit, and each load into a loop over its lanes).
    const uint32_t bytes =
        __builtin_amdgcn_readfirstlane(rows ? (rows - 1) * stride + width : 0u);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, 0x00020000);
}

template <typename E>
__device__ inline E load_one(__amdgpu_buffer_rsrc_t r, uint32_t voffset, uint32_t soffset) {
    if constexpr (sizeof(E) == 4)
        return __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b32(r, voffset, soffset, 0));
    else
        return __builtin_bit_cast(
            E, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, voffset, soffset, 0));
}

template <typename E>
__device__ inline void store_one(E x, __amdgpu_buffer_rsrc_t r, uint32_t voffset,
                                 uint32_t soffset) {
    if constexpr (sizeof(E) == 4)
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), r, voffset, soffset,
                                              0);
    else
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, x), r, voffset, soffset,
                                              0);
}

// load_lds16 at an offset of the instruction, from both addresses.
template <int Offset>
__device__ inline void load_lds16_at(__amdgpu_buffer_rsrc_t r, u32x4* dst, uint32_t voffset,
                                     uint32_t soffset) {
    typedef __attribute__((address_space(3))) void* lds_ptr_t;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 16, voffset, soffset, Offset, 0);
}

// Walks one sequence's chunks for 64 value columns of one head.  Each of the four
// waves holds 16 columns of the state as the results of 2 KB products (rows by
// 16): row 16 t + 4 (l / 16) + i and column l % 16 in register i of tile t of
// lane l, and splits it into the next products' operands where it is.  While a
// chunk is multiplied, the next one's record, operands and values come to LDS
// as they lie, the loads spread over the products.
//
// A chunk takes 1.9 us: (P k) S, U, its operand, T U and the update follow one
// another, and one wave a SIMD issues all of them, some 580 instructions of
// which 84 are products (1344 of 4400 cycles).  So a sequence of 2048 tokens
// takes 124 us, and seven of 8192 together (448 workgroups, two a CU) 150 us.
// Neither fewer columns a workgroup (two waves as long on the first, one 15%
// longer), nor more (eight waves 11% longer on the second), nor two waves to 16
// columns, each with half of the channels (15%), shorten that.
template <bool LO, int KB>
struct ScanChunk {
    ChunkRecord r;
    ChunkOperands<LO, KB> o;
};
// A wave's values of a chunk, [32][16].
template <uint32_t DT>
using ScanTile = typename Elem<DT>::type[kChunk][16];

// A column's largest is brought below 2^kHeld, as the state is held, once it is
// out of 2^(kHeld - 4) .. 2^(kHeld + 1).  As large as f16 allows: parts of an
// operand end at 2^-24, so that a value is held to 2^-25 / 2^(kHeld - 10) of the
// column's largest at worst, also of a later token of its chunk.
constexpr int kHeld = 14;

constexpr int kScanWaves = 4;
constexpr uint32_t kScanCols = 16 * kScanWaves;

template <uint32_t DT, bool LO, int KB>
constexpr size_t scan_lds() {
    return 2 * sizeof(ScanChunk<LO, KB>) + 2 * kScanWaves * sizeof(ScanTile<DT>);
}

// VEC: rows of v by 16 bytes (165 us with the operands' kernel, by one element
// 177, of the first call above on warm inputs).
template <uint32_t DT, bool CHANNEL, int KB, bool VEC>
__global__ __launch_bounds__(64 * kScanWaves, 2) void delta_scan_kernel(
    DeltaArgs a, const ChunkRecord* records,
    const ChunkOperands<CHANNEL || DT == K3X_DTYPE_F32, KB>* operands) {
    typedef typename Elem<DT>::type E;
    constexpr bool LO = CHANNEL || DT == K3X_DTYPE_F32;
    typedef ScanChunk<LO, KB> Chunk;
    // Sized at the launch: were the extent known here, the compiler would count
    // on one wave a SIMD and move results through the accumulation registers.
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    Chunk* buf = reinterpret_cast<Chunk*>(lds);
    const uint32_t blocks = (a.V + kScanCols - 1) / kScanCols;
    // Quotients come from the vector unit: kept scalar, as buffers want them.
    const uint32_t cb = __builtin_amdgcn_readfirstlane(blockIdx.x % blocks);
    const uint32_t h = __builtin_amdgcn_readfirstlane(blockIdx.x / blocks % a.H);
    const uint32_t n = __builtin_amdgcn_readfirstlane(blockIdx.x / blocks / a.H);
    const uint32_t lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Sequence sq;
    uint32_t bad = find_sequence(a, n, &sq);
    if (!bad && slot_taken(a, n, sq.slot)) bad = K3X_ERR_INVALID_STATE;
    if (bad) {
        if (threadIdx.x == 0) latch(a.errors, bad);
        return;
    }
    // Where offsets fall, their sequence latches it, and nothing is done: chunks are
    // searched for by the offsets, so that others' may not have been made.
    uint32_t stop = *(volatile const uint32_t*)a.status;
    if (a.offsets)
        for (uint32_t x = threadIdx.x; x < a.N; x += blockDim.x)
            stop |= a.offsets[x + 1] < a.offsets[x];
    if (__syncthreads_or(stop)) return;
    const uint32_t begin = __builtin_amdgcn_readfirstlane(sq.begin);
    const uint32_t len = __builtin_amdgcn_readfirstlane(sq.len);
    const uint32_t chunks = (len + kChunk - 1) / kChunk;
    const uint32_t hk = __builtin_amdgcn_readfirstlane(h / (a.H / a.Hk));
    const size_t slot0 = __builtin_amdgcn_readfirstlane(first_slot(a, n));
    constexpr uint32_t es = sizeof(E);
    constexpr int kTileLoads = sizeof(ScanTile<DT>) / 1024;
    ScanTile<DT>* tiles = reinterpret_cast<ScanTile<DT>*>(lds + 2 * sizeof(Chunk)) + 2 * wave;
    const uint32_t vst = (uint32_t)a.vs * es, ost = (uint32_t)a.os * es;
    const uint32_t col0 = (cb * kScanWaves + wave) * 16, col = col0 + m;
    const bool in = col < a.V;
    // Sixteen bytes of a row of the tile: lane's row (of each load's) and column.
    constexpr uint32_t kRowLanes = 16 * es / 16;
    const uint32_t trow = lane / kRowLanes, tcol = col0 + lane % kRowLanes * (16 / es);
    auto left = [&](uint32_t i) { return i < chunks ? min(len - i * kChunk, kChunk) : 0; };
    auto value_rows = [&](uint32_t i) {
        return rows_buffer(static_cast<const E*>(a.v) + (begin + (size_t)i * kChunk) * a.vs +
                               (size_t)h * a.V,
                           left(i), vst, a.V * es);
    };
    E direct[8];  // a chunk's values where rows are not by 16 bytes
    auto bring_values = [&](uint32_t i) {
        const auto r = value_rows(i);
        if (VEC) {
            // What lies past the last row or column is not used, but finite.
            const uint32_t c = tcol < a.V ? tcol * es : 0, last = left(i) - 1;
#pragma unroll
            for (int x = 0; x < kTileLoads; ++x)
                load_lds16(r, reinterpret_cast<u32x4*>(tiles[i & 1]) + 64 * x,
                           min(trow + x * (64 / kRowLanes), last) * vst + c, 0);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                direct[j] = load_one<E>(r, in ? (4 * g + 16 * (j / 4) + j % 4) * vst + col * es
                                              : kOutside, 0);
        }
    };
    auto put_values = [&](uint32_t i) {
        if (VEC) return;
#pragma unroll
        for (int j = 0; j < 8; ++j) tiles[i & 1][4 * g + 16 * (j / 4) + j % 4][m] = direct[j];
    };
    // The wave's share of a chunk, 1 KiB a load: the parts x of `of`.
    const ChunkRecord* rec = records + slot0 * a.H + h;
    const ChunkOperands<LO, KB>* ops = operands + (CHANNEL ? slot0 * a.H + h : slot0 * a.Hk + hk);
    const uint32_t heads = CHANNEL ? a.H : a.Hk;
    struct Source {
        __amdgpu_buffer_rsrc_t rec, ops;
    };
    auto source = [&]() {
        return Source{__builtin_amdgcn_make_buffer_rsrc(const_cast<ChunkRecord*>(rec), (short)0,
                                                        sizeof(ChunkRecord), 0x00020000),
                      __builtin_amdgcn_make_buffer_rsrc(
                          const_cast<ChunkOperands<LO, KB>*>(ops), (short)0,
                          sizeof(ChunkOperands<LO, KB>), 0x00020000)};
    };
    auto bring = [&](const Source& from, uint32_t i, uint32_t x, uint32_t of) {
        constexpr uint32_t kRec = sizeof(ChunkRecord) / 1024;
        constexpr uint32_t kOps = sizeof(ChunkOperands<LO, KB>) / 1024 / kScanWaves;
        constexpr uint32_t kRecLoads = (kRec + kScanWaves - 1) / kScanWaves;
        u32x4* dst = reinterpret_cast<u32x4*>(&buf[i & 1]);
        // Neighbouring loads go by the instruction's offset, four from one base.
        auto four = [&](__amdgpu_buffer_rsrc_t r, uint32_t first, uint32_t skip, uint32_t y) {
            u32x4* to = dst + 64 * (skip + first);
            if (y == 0) load_lds16_at<0>(r, to, lane * 16, first * 1024);
            if (y == 1) load_lds16_at<1024>(r, to, lane * 16, first * 1024);
            if (y == 2) load_lds16_at<2048>(r, to, lane * 16, first * 1024);
            if (y == 3) load_lds16_at<3 * 1024>(r, to, lane * 16, first * 1024);
        };
#pragma unroll
        for (uint32_t y = 0; y < kRecLoads + kOps; ++y) {
            if (y * of / (kRecLoads + kOps) != x) continue;
            if (y < kRecLoads) {
                if (kRecLoads * wave + y < kRec) four(from.rec, kRecLoads * wave, 0, y);
            } else {
                const uint32_t z = y - kRecLoads;
                four(from.ops, kOps * wave + z / 4 * 4, kRec, z % 4);
            }
        }
    };
    const size_t base = ((size_t)sq.slot * a.H + h) * a.K * a.V;
    if (!chunks) {  // the state as it is, which a column's scale need not hold
        if (!a.state_out || !in || a.state_in == a.state_out) return;
        for (uint32_t r = g; r < a.K; r += 4)
            a.state_out[base + (size_t)r * a.V + col] =
                a.state_in ? a.state_in[base + (size_t)r * a.V + col] : 0.0f;
        return;
    }
    // A column is held times 2^-shift, the state times kOperand besides.
    f32x4 S[2 * KB];
    int shift = 0;
    {
        float most = 0.0f;
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t r = 16 * t + 4 * g + i;
                S[t][i] = a.state_in && in && r < a.K ? a.state_in[base + (size_t)r * a.V + col]
                                                      : 0.0f;
                most = fmaxf(most, fabsf(S[t][i]));
            }
        most = max_groups(most);
        if (most > 0.0f) shift = __builtin_amdgcn_frexp_expf(most) + 6 - kHeld;
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[t][i] = kOperand * __builtin_ldexpf(S[t][i], -shift);
    }
    bring_values(0);
    bring(source(), 0, 0, 1);
    put_values(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    for (uint32_t ci = 0; ci < chunks; ++ci) {
        const ChunkRecord& rc = buf[ci & 1].r;
        const ChunkOperands<LO, KB>& o = buf[ci & 1].o;
        const bool more = ci + 1 < chunks;
        rec += a.H;
        ops += heads;
        const Source from = source();  // the next chunk
        f32x4 v[2], aq[2] = {}, ak[2] = {};
        // Operands of 32 channels, the next ones on their way while these are
        // multiplied.
        constexpr int kParts = LO ? 2 : 1;
        f16x8 kf[2][kParts][2], qf[2][kParts][2];
        auto frags = [&](int b) {
#pragma unroll
            for (int p = 0; p < kParts; ++p)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    kf[b & 1][p][t] = o.K[p][t][b][lane];
                    qf[b & 1][p][t] = o.Q[p][t][b][lane];
                }
        };
        auto factors = [&](const float* f, int t) {
            return *reinterpret_cast<const f32x4*>(f + 16 * t + 4 * g);
        };
        float most = 0.0f, vmost = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[t][j] = Elem<DT>::load(tiles[ci & 1][16 * t + 4 * g + j][m]);
        frags(0);
        if (more) bring_values(ci + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(S[t][i]));
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) vmost = fmaxf(vmost, fabsf(v[t][j]));
        // A column's size is an exponent of 2, that of the values as they came (times
        // kOperand, as the state is held): by the shift that a state next to nothing
        // has left behind they need not be numbers of fp32.
        constexpr int kEmpty = -(1 << 30);
        const int size =
            max_groups(max(most > 0.0f ? __builtin_amdgcn_frexp_expf(most) + shift : kEmpty,
                           vmost > 0.0f ? __builtin_amdgcn_frexp_expf(vmost) + 6 : kEmpty));
        int d = size - shift - kHeld;
        const bool off = ((d > 1) | (d < -3)) & (size > kEmpty);
        if (__builtin_amdgcn_ballot_w64(off)) {
            d = off ? d : 0;
            shift += d;
#pragma unroll
            for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[t][i] = __builtin_ldexpf(S[t][i], -d);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[t][j] = __builtin_ldexpf(v[t][j], -shift);
        // (P k) S and (P q) S; the products of one sum lie apart.
        f16x8 tf[2][2];
        f32x4 rt[2], rr[2];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            if (b + 1 < KB) {
                frags(b + 1);
            } else {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    tf[0][t] = rc.T[t][0][lane];
                    tf[1][t] = rc.T[t][1][lane];
                    rr[t] = factors(rc.row_r, t);
                    rt[t] = factors(rc.row_t, t);
                }
            }
            if (more) bring(from, ci + 1, b, KB);
            __builtin_amdgcn_sched_barrier(0);
            const f32x4 &l = S[2 * b], &u = S[2 * b + 1];
            const Pair8 s = split8(f32x8{l[0], l[1], l[2], l[3], u[0], u[1], u[2], u[3]});
            const auto& kp = kf[b & 1];
            const auto& qp = qf[b & 1];
            if (LO) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    ak[t] = mfma_f16(kp[kParts - 1][t], s.hi, ak[t]);
                    aq[t] = mfma_f16(qp[kParts - 1][t], s.hi, aq[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                ak[t] = mfma_f16(kp[0][t], s.lo, ak[t]);
                aq[t] = mfma_f16(qp[0][t], s.lo, aq[t]);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                ak[t] = mfma_f16(kp[0][t], s.hi, ak[t]);
                aq[t] = mfma_f16(qp[0][t], s.hi, aq[t]);
            }
            // The state's decay, for the update.
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const f32x4 f = factors(rc.decay, 2 * b + y);
#pragma unroll
                for (int i = 0; i < 4; ++i) S[2 * b + y][i] *= f[i];
            }
        }
        // A column that a product would take past f16 is made smaller.
        auto fit = [&](f32x4 (&y)[2]) {
            float big = 0.0f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) big = fmaxf(big, fabsf(y[t][j]));
            if (!__builtin_amdgcn_ballot_w64(big > 16384.0f)) return;
            big = max_groups(big);
            const int d = big > 16384.0f ? __builtin_amdgcn_frexp_expf(big) - 12 : 0;
            shift += d;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[t][j] = __builtin_ldexpf(y[t][j], -d);
                    aq[t][j] = __builtin_ldexpf(aq[t][j], -d);
                }
#pragma unroll
            for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[t][i] = __builtin_ldexpf(S[t][i], -d);
        };
        auto operand = [&](const f32x4 (&x)[2]) {
            return split8(f32x8{x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2],
                                x[1][3]});
        };
        f32x4 u[2], ap[2] = {};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) u[t][j] = __builtin_fmaf(-rr[t][j], ak[t][j], v[t][j]);
        fit(u);
        Pair8 up = operand(u);
        u[0] = u[1] = f32x4{};
        f16x8 pf[2][2], tk[2][kParts][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            pf[0][t] = rc.P[t][0][lane];
            pf[1][t] = rc.P[t][1][lane];
        }
        // Two tiles of channels of the keys for the update.
        auto channels = [&](int y) {
#pragma unroll
            for (int p = 0; p < kParts; ++p)
#pragma unroll
                for (int t = 0; t < 2; ++t) tk[y & 1][p][t] = o.Kt[p][2 * y + t][lane];
        };
        channels(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int y = 0; y < 3; ++y)
#pragma unroll
            for (int t = 0; t < 2; ++t)
                u[t] = mfma_f16(tf[y == 0][t], y == 1 ? up.lo : up.hi, u[t]);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) u[t][j] *= rt[t][j];
        fit(u);
        up = operand(u);
        f32x4 fo[2], fp[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            fo[t] = factors(rc.row_o, t);
            fp[t] = factors(rc.row_p, t);
        }
#pragma unroll
        for (int y = 0; y < 3; ++y)
#pragma unroll
            for (int t = 0; t < 2; ++t)
                ap[t] = mfma_f16(pf[y == 0][t], y == 1 ? up.lo : up.hi, ap[t]);
        if (!CHANNEL) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const f32x4 f = factors(rc.row_u, t);
#pragma unroll
                for (int j = 0; j < 4; ++j) u[t][j] *= f[j];
            }
            up = operand(u);
        }
        // The state's update.
#pragma unroll
        for (int y = 0; y < KB; ++y) {
            if (y + 1 < KB) channels(y + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (LO) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    S[2 * y + t] = mfma_f16(tk[y & 1][kParts - 1][t], up.hi, S[2 * y + t]);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
                S[2 * y + t] = mfma_f16(tk[y & 1][0][t], up.lo, S[2 * y + t]);
#pragma unroll
            for (int t = 0; t < 2; ++t)
                S[2 * y + t] = mfma_f16(tk[y & 1][0][t], up.hi, S[2 * y + t]);
        }
        const auto outs = rows_buffer(static_cast<E*>(a.out) +
                                          (begin + (size_t)ci * kChunk) * a.os + (size_t)h * a.V,
                                      left(ci), ost, a.V * es);
        // Outputs of 32 bytes a row and wave, as they lie in the registers.  Nothing above
        // is moved down here (without this the compiler does, and it takes 12% longer).
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int t = j / 4, i = j % 4;
            const float y = __builtin_fmaf(fp[t][i], ap[t][i], fo[t][i] * aq[t][i]);
            store_one<E>(Elem<DT>::store(__builtin_ldexpf(y, shift)), outs,
                         in ? (4 * g + 16 * t + i) * ost + col * es : kOutside, 0);
        }
        if (more) put_values(ci + 1);
        __builtin_amdgcn_sched_barrier(0);
        // The next chunk is in LDS (only these eight stores may still be on their
        // way) and every wave is done with this one.
        asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    // A value that is not finite has made every row of its column NaN (the
    // products' operands hold no infinity that is not NaN in a sum).
    if (!(S[0][0] - S[0][0] == 0.0f)) latch(a.errors, K3X_ERR_INVALID_MXFP4);
    if (!a.state_out || !in) return;
#pragma unroll
    for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = 16 * t + 4 * g + i;
            if (r < a.K)
                a.state_out[base + (size_t)r * a.V + col] = __builtin_ldexpf(S[t][i], shift - 6);
        }
}

// Chunks for heads that the products' tiles take, from the length on where one
// chunk costs no more than its tokens one by one.  Measured over 32 heads of
// 128 x 128, us in chunks and token by token:
//   gates by channel, 1 / 8 / 64 sequences of 20 tokens  22, 24 | 43, 35 | 196, 187
//                                             24 tokens  22, 28 | 43, 43 | 198, 214
//   gates by head (16 key heads),              8 tokens  17, 13 | 27, 17 | 106, 91
//                                             16 tokens  17, 19 | 27, 27 | 113, 147
bool runs_in_chunks(const k3x_hip_delta_params* p) {
    const uint32_t longest =
        p->longest ? p->longest : (p->tokens + p->sequences - 1) / p->sequences;
    return p->key_dim <= 128 && longest >= (p->gate == K3X_GATE_CHANNEL ? 24u : 16u);
}

// Where a call's records and operands lie in its workspace.
struct ChunkSpace {
    uint64_t slots;
    size_t operands_at, bytes;
};

ChunkSpace chunk_space(const k3x_hip_delta_params* p) {
    const bool channel = p->gate == K3X_GATE_CHANNEL;
    const uint64_t slots = p->tokens / kChunk + p->sequences;
    const size_t part = p->key_dim <= 64 ? sizeof(ChunkOperands<false, 2>)
                                         : sizeof(ChunkOperands<false, 4>);
    const size_t one = channel || p->dtype == K3X_DTYPE_F32 ? 2 * part : part;
    const size_t at = slots * p->value_heads * sizeof(ChunkRecord);
    return {slots, at, at + slots * (channel ? p->value_heads : p->key_heads) * one};
}

template <uint32_t DT, bool CHANNEL, int KB>
void launch_chunks(const DeltaArgs& a, void* workspace, const ChunkSpace& space, bool vec,
                   hipStream_t stream) {
    typedef ChunkOperands<CHANNEL || DT == K3X_DTYPE_F32, KB> Operands;
    ChunkRecord* records = static_cast<ChunkRecord*>(workspace);
    Operands* ops = reinterpret_cast<Operands*>(static_cast<uint8_t*>(workspace) +
                                                space.operands_at);
    const uint32_t slots = (uint32_t)space.slots;
    auto prepare = [&](auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        if constexpr (CHANNEL)
            hipLaunchKernelGGL((delta_prep_channel_kernel<DT, KB, kWhole>), dim3(slots * a.H),
                               dim3(128), 0, stream, a, records, ops);
        else
            hipLaunchKernelGGL((delta_prep_head_kernel<DT, KB, kWhole>), dim3(slots * a.Hk),
                               dim3(128), 0, stream, a, records, ops);
    };
    if (vec && a.K == 32 * KB) prepare(std::true_type{});
    else prepare(std::false_type{});
    constexpr bool LO = CHANNEL || DT == K3X_DTYPE_F32;
    const uint32_t es = sizeof(typename Elem<DT>::type);
    auto scan = [&](auto by16) {
        hipLaunchKernelGGL((delta_scan_kernel<DT, CHANNEL, KB, decltype(by16)::value>),
                           dim3(a.N * a.H * ((a.V + kScanCols - 1) / kScanCols)),
                           dim3(64 * kScanWaves), (scan_lds<DT, LO, KB>()), stream, a,
                           records, ops);
    };
    if (a.V * es % 16 == 0 && a.vs * es % 16 == 0 && aligned(a.v, 16)) scan(std::true_type{});
    else scan(std::false_type{});
}

template <uint32_t DT>
void launch_chunks_of(const DeltaArgs& a, void* workspace, const ChunkSpace& space, bool channel,
                      bool vec, hipStream_t stream) {
    if (a.K <= 64)
        channel ? launch_chunks<DT, true, 2>(a, workspace, space, vec, stream)
                : launch_chunks<DT, false, 2>(a, workspace, space, vec, stream);
    else
        channel ? launch_chunks<DT, true, 4>(a, workspace, space, vec, stream)
                : launch_chunks<DT, false, 4>(a, workspace, space, vec, stream);
}

bool delta_ok(const k3x_hip_delta_params* p) {
    if (!p->sequences || p->sequences > 65535 || p->tokens > (1u << 24) || !p->value_heads ||
        p->value_heads > 1024 || !p->key_heads || p->value_heads % p->key_heads || !p->key_dim ||
        p->key_dim > 256 || !p->value_dim || p->value_dim > 1024 || p->dtype > K3X_DTYPE_F16 ||
        p->gate > K3X_GATE_CHANNEL || !std::isfinite(p->scale) ||
        !std::isfinite(p->norm_epsilon) || p->norm_epsilon < 0.0f)
        return false;
    const uint64_t kw = (uint64_t)p->key_heads * p->key_dim;
    const uint64_t vw = (uint64_t)p->value_heads * p->value_dim, most = 1ull << 24;
    return (!p->q_stride || (p->q_stride >= kw && p->q_stride <= most)) &&
           (!p->k_stride || (p->k_stride >= kw && p->k_stride <= most)) &&
           (!p->v_stride || (p->v_stride >= vw && p->v_stride <= most)) &&
           (!p->out_stride || (p->out_stride >= vw && p->out_stride <= most)) &&
           // threads of a launch
           (uint64_t)p->sequences * p->value_heads * ((p->value_dim + 63) / 64) * 256 <
               (1ull << 32) &&
           ((uint64_t)p->tokens / kChunk + p->sequences) * p->value_heads * 128 < (1ull << 32);
}

}  // namespace

extern "C" {

size_t k3x_hip_delta_workspace(const k3x_hip_delta_params* p) {
    if (!p || !delta_ok(p) || !runs_in_chunks(p)) return 0;
    return chunk_space(p).bytes;
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
    // 64 sequences of 1 token of 32 heads, warm: 45.0 us a call, without report_kernel 43.6.
    const bool apart = state_out && state_in == state_out && a.N > 1;
    a.errors = apart ? ctx->status + 1 : ctx->status;
    // Four elements a load: rows and heads that keep the alignment.
    const bool vec = a.K % 4 == 0 && a.qs % 4 == 0 && a.ks % 4 == 0 && aligned(q, 4 * es) &&
                     aligned(k, 4 * es) && aligned(gate, 16);
    unsigned launches = apart ? 1 : 0;
    if (need) {
        const ChunkSpace space = chunk_space(p);
        const bool channel = p->gate == K3X_GATE_CHANNEL;
        if (p->dtype == K3X_DTYPE_F32)
            launch_chunks_of<K3X_DTYPE_F32>(a, workspace, space, channel, vec, ctx->stream);
        else if (p->dtype == K3X_DTYPE_BF16)
            launch_chunks_of<K3X_DTYPE_BF16>(a, workspace, space, channel, vec, ctx->stream);
        else launch_chunks_of<K3X_DTYPE_F16>(a, workspace, space, channel, vec, ctx->stream);
        launches += 2;
    } else {
        const uint32_t by_four = (vec ? 1 : 0) |
                                 (a.V % 4 == 0 && a.vs % 4 == 0 && aligned(v, 4 * es) ? 2 : 0) |
                                 (a.V % 4 == 0 ? 4 : 0);
        if (p->dtype == K3X_DTYPE_F32)
            launch_step_rows<K3X_DTYPE_F32>(a, p->gate, by_four, ctx->stream);
        else if (p->dtype == K3X_DTYPE_BF16)
            launch_step_rows<K3X_DTYPE_BF16>(a, p->gate, by_four, ctx->stream);
        else launch_step_rows<K3X_DTYPE_F16>(a, p->gate, by_four, ctx->stream);
        launches += 1;
    }
    if (apart)
        hipLaunchKernelGGL(report_kernel, dim3(1), dim3(1), 0, ctx->stream, a.errors, ctx->status);
    return launched(ctx, launches);
}

}  // extern "C"
