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
// delta_prep_kernel makes (I + L)^-1 and Pq of every chunk, all at once;
// delta_scan_kernel walks a sequence's chunks with the state in registers.
//
// Operands are f16 pairs hi + lo (22 bits: what is left out of a product of two
// pairs, lo lo, is 2^-22 of it), sums fp32.  f16 ends at 65504 and 2^-24, so
// keys and queries are scaled to 64 at most, rows of the inverse by a power of
// two each, and a column of the state and its values by one power of two that
// follows their size.
// ---------------------------------------------------------------------------
constexpr uint32_t kChunk = 32;
constexpr float kOperand = 64.0f;  // keys, queries and Pq are held times this

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

struct Pair8 {
    f16x8 hi, lo;
};

// hi = f16(x), lo = f16(x - hi).  The factor -1 is kept from the compiler so
// that the difference is one fused instruction on the packed halves.
__device__ inline Pair8 split8(const float (&x)[8]) {
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
        const f32x2 r = {__builtin_fmaf((float)h[0], minus, v[0]),
                         __builtin_fmaf((float)h[1], minus, v[1])};
        hi[j] = u;
        lo[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, f16x2));
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

// What the scan needs of one chunk of one head.  T and Pq in the order of the
// matrix operand: lane l, element j of tile r is row 16 r + l % 16, column
// token_of(l / 16, j); the columns' order is that in which a lane holds the
// rows of a product's result, so that results feed the next product as they
// are.
struct ChunkRecord {
    f16x8 T[2][2][64];   // [tile][hi, lo]; a row times row_t is c (I + L)^-1 beta
    f16x8 P[2][2][64];   // Pq times kOperand
    float key_mul[kChunk], query_mul[kChunk];  // element -> operand / kOperand
    float row_r[kChunk];                       // of (k S) in V - c (P k) S
    float row_o[kChunk], row_p[kChunk];        // of (q S) and (Pq U) in O
    float row_t[kChunk];
    float row_u[kChunk];                       // head gates: of U in the state's update
    float unused[kChunk];
    float total[2][128];  // decay over tokens 0 .. 15 and 16 .. 31, by channel
};
static_assert(sizeof(ChunkRecord) == 10240, "chunk record");

__device__ inline uint32_t token_of(uint32_t q, uint32_t j) { return 4 * q + (j & 3) + 4 * (j & 4); }

template <int Ctrl>
__device__ inline float dpp(float x, float old = 0.0f) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(x), Ctrl,
                                                      0xf, 0xf, false));
}

// Sum and maximum over the lanes of equal lane % 16: rows of 16 lanes, then
// halves of the wave, exchanged in registers.
__device__ inline void swap_rows(float x, float* a, float* b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    *a = __uint_as_float(r[0]);
    *b = __uint_as_float(r[1]);
}
__device__ inline void swap_halves(float x, float* a, float* b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    *a = __uint_as_float(r[0]);
    *b = __uint_as_float(r[1]);
}
__device__ inline float sum_groups(float v) {
    float a, b;
    swap_rows(v, &a, &b);
    swap_halves(a + b, &a, &b);
    return a + b;
}
__device__ inline float max_groups(float v) {
    float a, b;
    swap_rows(v, &a, &b);
    swap_halves(fmaxf(a, b), &a, &b);
    return fmaxf(a, b);
}

// 2^-e and 2^e for the least e with |x| < 2^e (x finite); 1 and 1 for x = 0.
__device__ inline void unit_scale(float x, float* down, float* up) {
    int e = x > 0.0f ? __builtin_amdgcn_frexp_expf(x) : 0;
    e = e < -100 ? -100 : e > 100 ? 100 : e;
    *down = __builtin_ldexpf(1.0f, -e);
    *up = __builtin_ldexpf(1.0f, e);
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

// Eight elements from c on in fp32, 0 past the row's end or where it is not
// live; z takes a NaN where one is not finite.
template <uint32_t DT>
__device__ inline void load8(const typename Elem<DT>::type* row, uint32_t c, uint32_t n, bool live,
                             bool vec, float (&y)[8], float& z) {
    const auto a = load4(row, c, n, vec), b = load4(row, c + 4, n, vec);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = Elem<DT>::load(j < 4 ? a[j & 3] : b[j & 3]);
        y[j] = live && c + j < n ? x : 0.0f;
        z = __builtin_fmaf(y[j], 0.0f, z);
    }
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

// LDS written before is seen after, by the whole workgroup; loads from global
// memory stay in flight across it.
__device__ inline void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// (I + L)^-1 and Pq of one chunk of one head, by two waves: wave w has tokens
// 16 w .. + 15, lane l token l % 16 and the channels 32 b + 8 (l / 16) .. + 7.
//
// A decay a channel does not factor over (i, j) without overflow, so a tile's
// lower triangle is made level by level: pairs (i, j) whose highest differing
// bit is b have D_ij = pre_b(i) suf_b(j), the decays up to the border between
// i's and j's blocks of 2^b tokens and from there on, both at most 1.  Each
// level is one product of the whole tile, of which its own pairs are kept.
// pre, suf and a block's total come from the level before by one exchange over
// the lanes of a row.  A decay a head is one factor exp(G_i - G_j) a pair, G
// summed in double.
template <uint32_t DT, bool CHANNEL, int KB>
__global__ __launch_bounds__(128) void delta_prep_kernel(DeltaArgs a, ChunkRecord* records,
                                                         bool vec) {
    typedef typename Elem<DT>::type E;
    constexpr int kLevels = CHANNEL ? 4 : 1;
    __shared__ float Ls[kChunk][36], Ps[kChunk][36];
    __shared__ Pair8 cross[KB][64];
    __shared__ float beta_s[kChunk], c_s[kChunk];
    __shared__ double G_s[kChunk];  // head gates: log decay from the tile's start
    const uint32_t h = blockIdx.x % a.H, slot = blockIdx.x / a.H;
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    if (__syncthreads_or(*(volatile uint32_t*)a.status)) return;
    const uint32_t n = sequence_of_slot(a, slot);
    Sequence sq;
    if (find_sequence(a, n, &sq)) return;  // latched by the scan
    const uint32_t slot0 = first_slot(a, n);
    if (slot < slot0 || slot - slot0 >= (sq.len + kChunk - 1) / kChunk) return;
    const uint32_t first = (slot - slot0) * kChunk;
    ChunkRecord* rec = records + (size_t)slot * a.H + h;
    const uint32_t t = 16 * w + m, hk = h / (a.H / a.Hk);
    const bool live = first + t < sq.len;
    const size_t row = (size_t)sq.begin + first + (live ? t : 0);
    float z = 0.0f;  // NaN once an input is not finite
    bool wrong = false;
    float q[KB][8], k[KB][8];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
        const uint32_t c = 32 * b + 8 * g;
        load8<DT>(static_cast<const E*>(a.q) + row * a.qs + (size_t)hk * a.K, c, a.K, live, vec,
                  q[b], z);
        load8<DT>(static_cast<const E*>(a.k) + row * a.ks + (size_t)hk * a.K, c, a.K, live, vec,
                  k[b], z);
    }
    const float beta = live ? a.beta[row * a.H + h] : 0.0f;
    z = __builtin_fmaf(beta, 0.0f, z);
    // Operands' scales: the norm, or a power of two.
    float qd, qu, kd, ku, qn = 1.0f, kn = 1.0f;
    {
        float qm = 0.0f, km = 0.0f, qq = 0.0f, kk = 0.0f;
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                qm = fmaxf(qm, fabsf(q[b][j]));
                km = fmaxf(km, fabsf(k[b][j]));
                qq = __builtin_fmaf(q[b][j], q[b][j], qq);
                kk = __builtin_fmaf(k[b][j], k[b][j], kk);
            }
        unit_scale(max_groups(qm), &qd, &qu);
        unit_scale(max_groups(km), &kd, &ku);
        qn = 1.0f / sqrtf(sum_groups(qq) + a.eps);
        kn = 1.0f / sqrtf(sum_groups(kk) + a.eps);
    }
    const bool norm = a.eps > 0.0f;
    const float kmul = norm ? kn : kd, qmul = norm ? qn : qd;
    const float c_up = norm ? 1.0f : ku, o_up = a.scale * (norm ? 1.0f : qu);
    if (lane < 16) {
        beta_s[t] = beta;
        c_s[t] = c_up;
    }
    if (!CHANNEL) {
        const float gate = live && a.gate ? a.gate[row * a.H + h] : 0.0f;
        wrong |= !(gate <= 0.0f);
        double G = (double)fmaxf(gate, -128.0f);  // exp of less is 0 in fp32
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            const double o = __shfl_up(G, d, 16);
            if (m >= (uint32_t)d) G += o;
        }
        if (lane < 16) G_s[t] = G;
    }
    f32x4 accL[kLevels] = {}, accP[kLevels] = {};
    Pair8 krow[KB], qrow[KB];  // wave 1: rows of the tile below the diagonal
    float diag = 0.0f;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
        float kk[8], qq[8], x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            kk[j] = k[b][j] * kmul * kOperand;
            qq[j] = q[b][j] * qmul * kOperand;
            diag = __builtin_fmaf(kk[j], qq[j], diag);
        }
        if (!CHANNEL) {
            krow[b] = split8(kk);
            qrow[b] = split8(qq);
            accL[0] = mfma_pairs(krow[b], krow[b], accL[0]);
            accP[0] = mfma_pairs(qrow[b], krow[b], accP[0]);
            if (w == 0) cross[b][lane] = krow[b];
            continue;
        }
        float pre[8], suf[8], tot[8], gate[8], any = 0.0f;
        const uint32_t c = 32 * b + 8 * g;
        load8<K3X_DTYPE_F32>(a.gate + (row * a.H + h) * a.K, c, a.K, live, vec, gate, any);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            wrong |= !(gate[j] <= 0.0f);
            pre[j] = tot[j] = exp_decay(gate[j]);
            suf[j] = 1.0f;
        }
#pragma unroll
        for (int level = 0; level < kLevels; ++level) {
            const bool bit = m >> level & 1;
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f[j] = bit ? pre[j] : suf[j];
                x[j] = kk[j] * f[j];
            }
            const Pair8 kp = split8(x);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = qq[j] * f[j];
            const Pair8 qp = split8(x);
            accL[level] = mfma_pairs(kp, kp, accL[level]);
            accP[level] = mfma_pairs(qp, kp, accP[level]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // The other block's total: from across bit `level` (a total is
                // the same on every lane of its block, so that mirrors do).
                const float o = level == 0   ? dpp<0xb1>(tot[j])
                                : level == 1 ? dpp<0x4e>(tot[j])
                                : level == 2 ? dpp<0x141>(tot[j])
                                             : dpp<0x140>(tot[j]);
                pre[j] *= bit ? o : 1.0f;
                suf[j] *= bit ? 1.0f : o;
                tot[j] *= o;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = kk[j] * (w ? pre[j] : suf[j]);
        krow[b] = split8(x);
        if (w == 0) {
            cross[b][lane] = krow[b];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = qq[j] * pre[j];
            qrow[b] = split8(x);
        }
        if (m == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) rec->total[w][c + j] = tot[j];
        }
    }
    diag = sum_groups(diag);
    if (wrong || z != z) latch(a.status, K3X_ERR_INVALID_MXFP4);
    __syncthreads();
    const float un = 1.0f / (kOperand * kOperand);
    if (lane < 16) {
        const float rk = CHANNEL || !norm ? 1.0f : kn * ku, rq = CHANNEL || !norm ? 1.0f : qn * qu;
        float p = 1.0f, s = 1.0f;
        if (!CHANNEL) {
            const double G = G_s[t] + (w ? G_s[15] : 0.0), all = G_s[15] + G_s[31];
            p = (float)exp(G);
            s = (float)exp(all - G);
            if (t == 31) rec->total[0][0] = p;
        }
        // 0 past the sequence's end, where the scan reads another row.
        rec->key_mul[t] = !live ? 0.0f : CHANNEL ? kmul : kd;
        rec->query_mul[t] = !live ? 0.0f : CHANNEL ? qmul : qd;
        rec->row_r[t] = c_up * un * p * rk;
        rec->row_o[t] = o_up * un * p * rq;
        rec->row_p[t] = o_up / kOperand;
        rec->row_u[t] = s * rk;
    }
    // Row 4 g + i and column m of the wave's tile on the diagonal.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t r = 4 * g + i, ti = 16 * w + r;
        float l = accL[0][i], p = accP[0][i];
        if (CHANNEL) {
            const uint32_t differ = r ^ m;
#pragma unroll
            for (int level = 1; level < kLevels; ++level)
                if (differ >= 1u << level) {
                    l = accL[level][i];
                    p = accP[level][i];
                }
        } else {
            const float f = r > m ? (float)exp(G_s[ti] - G_s[t]) : 1.0f;
            l *= f;
            p *= f;
        }
        Ls[ti][t] = r > m ? l * un * beta_s[ti] * c_s[ti] * c_s[t] : 0.0f;
        Ps[ti][t] = (r > m ? p : r == m ? diag : 0.0f) / kOperand;
        if (w == 0) Ps[r][16 + m] = 0.0f;
    }
    if (w == 1) {  // rows 16 .. 31, columns 0 .. 15
        f32x4 l = {}, p = {};
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const Pair8 kp = cross[b][lane];
            l = mfma_pairs(krow[b], kp, l);
            p = mfma_pairs(qrow[b], kp, p);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t ti = 16 + 4 * g + i;
            const float f = CHANNEL ? 1.0f : (float)exp(G_s[ti] + (G_s[15] - G_s[m]));
            Ls[ti][m] = l[i] * f * un * beta_s[ti] * c_s[ti] * c_s[m];
            Ps[ti][m] = p[i] * f / kOperand;
        }
    }
    __syncthreads();
    if (w == 1) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = Ps[16 * r + m][token_of(g, j)];
            const Pair8 s = split8(x);
            rec->P[r][0][lane] = s.hi;
            rec->P[r][1][lane] = s.lo;
        }
        return;
    }
    // Column lane % 32 of (I + L)^-1 by forward substitution, in fp32.
    const uint32_t col = lane & 31;
    float x[kChunk];
#pragma unroll
    for (int i = 0; i < (int)kChunk; ++i) {
        float s = (uint32_t)i == col ? 1.0f : 0.0f;
#pragma unroll
        for (int j = 0; j < i; ++j) s = __builtin_fmaf(-Ls[i][j], x[j], s);
        x[i] = s;
    }
    if (lane < 32) {
        const float right = beta_s[col];
#pragma unroll
        for (int i = 0; i < (int)kChunk; ++i) Ls[i][col] = x[i] * c_s[i] * right;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        float y[8], most = 0.0f, down, up;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            y[j] = Ls[16 * r + m][token_of(g, j)];
            most = fmaxf(most, fabsf(y[j]));
        }
        unit_scale(max_groups(most), &down, &up);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] *= down * kOperand;
        const Pair8 s = split8(y);
        rec->T[r][0][lane] = s.hi;
        rec->T[r][1][lane] = s.lo;
        if (g == 0) rec->row_t[16 * r + m] = up / kOperand;
    }
}

// One chunk's operands in LDS, in the order of the matrix operand: hi and,
// where the terms need it, lo.
template <uint32_t DT, bool CHANNEL, int KB>
struct ScanTerms {
    // Keys and queries under a head's decay are the elements themselves times a
    // power of two: 8 and 11 bits are f16 without rest.
    static constexpr bool kKeyLo = CHANNEL || DT == K3X_DTYPE_F32;
    struct Chunk {
        f16x8 K[kKeyLo ? 2 : 1][2][KB][64];    // [tile of tokens][channels]: decayed keys
        f16x8 Q[kKeyLo ? 2 : 1][2][KB][64];
        f16x8 Kt[kKeyLo ? 2 : 1][2 * KB][64];  // [tile of channels][tokens]: keys for the state
        f16x8 T[2][2][64], P[2][2][64];        // as in the chunk's record
        float row_r[kChunk], row_o[kChunk], row_p[kChunk], row_t[kChunk], row_u[kChunk];
        float decay[32 * KB];
    };
};

// Product over the lanes of a row up to and with the lane's own.
__device__ inline float scan_row(float x) {
    x *= dpp<0x111>(x, 1.0f);  // row_shr
    x *= dpp<0x112>(x, 1.0f);
    x *= dpp<0x114>(x, 1.0f);
    return x * dpp<0x118>(x, 1.0f);
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
__device__ inline Vec4<E> load_four(__amdgpu_buffer_rsrc_t r, uint32_t voffset, uint32_t soffset) {
    if constexpr (sizeof(E) == 4)
        return __builtin_bit_cast(Vec4<E>,
                                  __builtin_amdgcn_raw_buffer_load_b128(r, voffset, soffset, 0));
    else
        return __builtin_bit_cast(Vec4<E>,
                                  __builtin_amdgcn_raw_buffer_load_b64(r, voffset, soffset, 0));
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

// Walks one sequence's chunks for 64 value columns of one head.  Waves 0 .. 3
// hold 16 columns of the state each, as the results of eight products (rows by
// 16): row 16 t + 4 (l / 16) + i and column l % 16 in register i of tile t of
// lane l, and split it into the next products' operands where it is.  Waves 4
// .. 7 make the next chunk's key and query operands meanwhile: two of them a
// tile of 16 tokens each, lane = token, decays by a product along the lanes;
// two the keys by channel, lane = channel, decays by a walk back over the
// tokens.
template <uint32_t DT, bool CHANNEL, int KB, int NT>
__global__ __launch_bounds__(512) void delta_scan_kernel(DeltaArgs a, const ChunkRecord* records,
                                                         bool vec) {
    typedef typename Elem<DT>::type E;
    typedef ScanTerms<DT, CHANNEL, KB> Terms;
    typedef typename Terms::Chunk Chunk;
    __shared__ Chunk buf[2];
    const uint32_t blocks = (a.V + 64 * NT - 1) / (64 * NT);
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
        if (threadIdx.x == 0) latch(a.status, bad);
        return;
    }
    if (__syncthreads_or(*(volatile uint32_t*)a.status)) return;
    const uint32_t begin = __builtin_amdgcn_readfirstlane(sq.begin);
    const uint32_t len = __builtin_amdgcn_readfirstlane(sq.len);
    const uint32_t chunks = (len + kChunk - 1) / kChunk, hk = __builtin_amdgcn_readfirstlane(h / (a.H / a.Hk));
    // The record of chunk i is i a.H on.
    const ChunkRecord* rec =
        records + (size_t)__builtin_amdgcn_readfirstlane(first_slot(a, n)) * a.H + h;

    constexpr uint32_t es = sizeof(E);
    const uint32_t kst = (uint32_t)a.ks * es, qst = (uint32_t)a.qs * es, gst = a.H * a.K * 4;
    auto left = [&](uint32_t i) { return i < chunks ? min(len - i * kChunk, kChunk) : 0; };
    // Chunk i's rows of this head (none past the last chunk).
    auto key_rows = [&](uint32_t i) {
        return rows_buffer(static_cast<const E*>(a.k) + (begin + (size_t)i * kChunk) * a.ks +
                               (size_t)hk * a.K,
                           left(i), kst, a.K * es);
    };
    auto query_rows = [&](uint32_t i) {
        return rows_buffer(static_cast<const E*>(a.q) + (begin + (size_t)i * kChunk) * a.qs +
                               (size_t)hk * a.K,
                           left(i), qst, a.K * es);
    };
    auto gate_rows = [&](uint32_t i) {
        return rows_buffer(a.gate + ((begin + (size_t)i * kChunk) * a.H + h) * a.K, left(i), gst,
                           a.K * 4);
    };
    auto record = [&](uint32_t i) { return rec + (size_t)min(i, chunks - 1) * a.H; };
    // Each of waves 4 .. 7 also copies two of the eight operands T and P.
    auto copied = [&](const ChunkRecord* r, uint32_t x) {
        return (&r->T[0][0][0])[64 * (2 * (wave - 4) + x) + lane];
    };
    static_assert(offsetof(ChunkRecord, P) == sizeof(ChunkRecord::T), "T, then P");
    static_assert(offsetof(Chunk, P) - offsetof(Chunk, T) == sizeof(ChunkRecord::T), "T, then P");
    auto paste = [&](Chunk& o, const f16x8 (&x)[2]) {
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) (&o.T[0][0][0])[64 * (2 * (wave - 4) + j) + lane] = x[j];
    };
    // The makers hold one chunk's elements and, as they use them up, load the
    // next one's in their place, so that loads have a chunk's time to arrive.
    if (wave >= 6) {  // keys by channel, and the rows' factors
        const uint32_t c = 64 * (wave - 6) + lane;
        const uint32_t koff = c < a.K ? c * es : kOutside, goff = c < a.K ? c * 4 : kOutside;
        E k[kChunk];
        float gate[CHANNEL ? kChunk : 1], mul = 0.0f, total = 0.0f, factor[3] = {};
        f16x8 copy[2] = {};
        auto scalars = [&](uint32_t i) {
            const ChunkRecord* r = record(i);
            copy[0] = copied(r, 0);
            copy[1] = copied(r, 1);
            mul = r->key_mul[lane & 31];
            if (!CHANNEL) total = r->total[0][0];
            if (wave == 6) {
                factor[0] = (&r->row_r[0])[lane];
                factor[1] = (&r->row_r[0])[64 + lane];
                factor[2] = (&r->row_r[0])[128 + (lane & 31)];
            }
        };
        auto make = [&](uint32_t i, Chunk& o) {
            const auto kr = key_rows(i + 1), gr = gate_rows(i + 1);
            const float own = mul;
            // Row offsets are formed anew: held over the loop they would not fit.
            uint32_t ks = kst, gs = gst;
            asm volatile("" : "+s"(ks), "+s"(gs));
            paste(o, copy);
            if (wave == 6) {
                (&o.row_r[0])[lane] = factor[0];
                (&o.row_r[0])[64 + lane] = factor[1];
                if (lane < 32) (&o.row_r[0])[128 + lane] = factor[2];
            }
            if (!CHANNEL && c < 32 * KB) o.decay[c] = total;
            scalars(i + 1);
            float s = kOperand, late[kChunk / 2];
            auto next = [&](int t) {
                const float one =
                    __int_as_float(__builtin_amdgcn_readlane(__float_as_int(own), t));
                const float x = Elem<DT>::load(k[t]) * one * s;
                k[t] = load_one<E>(kr, koff, t * ks);
                if (CHANNEL) {
                    s *= exp_decay(gate[t]);
                    gate[t] = load_one<float>(gr, goff, t * gs);
                }
                return x;
            };
#pragma unroll
            for (int t = kChunk - 1; t >= (int)kChunk / 2; --t) late[t - kChunk / 2] = next(t);
#pragma unroll
            for (int q = 3; q >= 0; --q) {
                float y[8];
#pragma unroll
                for (int j = 3; j >= 0; --j) {
                    y[j] = next(4 * q + j);
                    y[4 + j] = late[4 * q + j];
                }
                const Pair8 p = split8(y);
                if (c >= 32 * KB) continue;
                o.Kt[0][c / 16][q * 16 + c % 16] = p.hi;
                if (Terms::kKeyLo) o.Kt[Terms::kKeyLo ? 1 : 0][c / 16][q * 16 + c % 16] = p.lo;
            }
            if (CHANNEL && c < 32 * KB) o.decay[c] = s * (1.0f / kOperand);
        };
        if (chunks) {
            const auto kr = key_rows(0), gr = gate_rows(0);
            scalars(0);
#pragma unroll
            for (int t = kChunk - 1; t >= 0; --t) {
                k[t] = load_one<E>(kr, koff, t * kst);
                if (CHANNEL) gate[t] = load_one<float>(gr, goff, t * gst);
            }
            make(0, buf[0]);
        }
        lds_barrier();
        for (uint32_t i = 1; i <= chunks; ++i) {
            if (i < chunks) make(i, buf[i & 1]);
            lds_barrier();
        }
        return;
    }
    if (wave >= 4) {  // keys and queries by token
        const uint32_t r = wave - 4;
        Vec4<E> k[KB][2], q[KB][2];
        f32x4 gate[CHANNEL ? KB : 1][2], before[CHANNEL ? KB : 1][2];
        float kmul = 0.0f, qmul = 0.0f;
        f16x8 copy[2] = {};
        const uint32_t t = 16 * r + m;
        const bool whole = vec && a.K == 32 * KB;
        auto scalars = [&](uint32_t i) {
            const ChunkRecord* rc = record(i);
            copy[0] = copied(rc, 0);
            copy[1] = copied(rc, 1);
            kmul = rc->key_mul[t] * kOperand;
            qmul = rc->query_mul[t] * kOperand;
        };
        auto total_row = [&](uint32_t i) { return rows_buffer(record(i)->total[0], 1, 0, 512); };
        auto load = [&](int b, __amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t qr,
                        __amdgpu_buffer_rsrc_t gr, __amdgpu_buffer_rsrc_t tr) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t c = 32 * b + 16 * j + 4 * g;
                if (whole) {
                    k[b][j] = load_four<E>(kr, t * kst + c * es, 0);
                    q[b][j] = load_four<E>(qr, t * qst + c * es, 0);
                    if (CHANNEL) gate[b][j] = load_four<float>(gr, t * gst + c * 4, 0);
                } else {
                    uint32_t row = t, first = c;  // offsets formed anew, as above
                    asm volatile("" : "+v"(row), "+v"(first));
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t at = first + x;
                        const bool in = at < a.K;
                        k[b][j][x] = load_one<E>(kr, in ? row * kst + at * es : kOutside, 0);
                        q[b][j][x] = load_one<E>(qr, in ? row * qst + at * es : kOutside, 0);
                        if (CHANNEL)
                            gate[b][j][x] =
                                load_one<float>(gr, in ? row * gst + at * 4 : kOutside, 0);
                    }
                }
                if (CHANNEL && r) before[b][j] = load_four<float>(tr, c * 4, 0);
            }
        };
        auto make = [&](uint32_t i, Chunk& o) {
            const auto kr = key_rows(i + 1), qr = query_rows(i + 1), gr = gate_rows(i + 1);
            const auto tr = total_row(i + 1);
            const float km = kmul, qm = qmul;
            paste(o, copy);
            scalars(i + 1);
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                float kx[8], qx[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    kx[j] = Elem<DT>::load(k[b][j / 4][j % 4]) * km;
                    qx[j] = Elem<DT>::load(q[b][j / 4][j % 4]) * qm;
                    if (CHANNEL) {
                        float p = scan_row(exp_decay(gate[b][j / 4][j % 4]));
                        if (r) p *= before[b][j / 4][j % 4];
                        kx[j] *= p;
                        qx[j] *= p;
                    }
                }
                load(b, kr, qr, gr, tr);
                const Pair8 kp = split8(kx), qp = split8(qx);
                o.K[0][r][b][lane] = kp.hi;
                if (Terms::kKeyLo) o.K[Terms::kKeyLo ? 1 : 0][r][b][lane] = kp.lo;
                o.Q[0][r][b][lane] = qp.hi;
                if (Terms::kKeyLo) o.Q[Terms::kKeyLo ? 1 : 0][r][b][lane] = qp.lo;
            }
        };
        if (chunks) {
            const auto kr = key_rows(0), qr = query_rows(0), gr = gate_rows(0);
            const auto tr = total_row(0);
            scalars(0);
#pragma unroll
            for (int b = 0; b < KB; ++b) load(b, kr, qr, gr, tr);
            make(0, buf[0]);
        }
        lds_barrier();
        for (uint32_t i = 1; i <= chunks; ++i) {
            if (i < chunks) make(i, buf[i & 1]);
            lds_barrier();
        }
        return;
    }

    const size_t base = ((size_t)sq.slot * a.H + h) * a.K * a.V;
    const uint32_t vst = (uint32_t)a.vs * es, ost = (uint32_t)a.os * es;
    uint32_t col[NT], voff[NT], ooff[NT];
    // A column is held times 2^-shift, the state times kOperand besides.
    f32x4 S[NT][2 * KB];
    int shift[NT];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
        col[x] = (cb * 4 + wave) * 16 * NT + 16 * x + m;
        const bool in = col[x] < a.V;
        voff[x] = in ? 4 * g * vst + col[x] * es : kOutside;
        ooff[x] = in ? 4 * g * ost + col[x] * es : kOutside;
        float most = 0.0f;
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t r = 16 * t + 4 * g + i;
                S[x][t][i] = a.state_in && in && r < a.K
                                 ? a.state_in[base + (size_t)r * a.V + col[x]]
                                 : 0.0f;
                most = fmaxf(most, fabsf(S[x][t][i]));
            }
        most = max_groups(most);
        shift[x] = most > 0.0f ? __builtin_amdgcn_frexp_expf(most) - 3 : 0;
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                S[x][t][i] = kOperand * __builtin_ldexpf(S[x][t][i], -shift[x]);
    }
    E next[NT][2][4];
    auto fetch = [&](uint32_t i) {
        const auto r = rows_buffer(static_cast<const E*>(a.v) +
                                       (begin + (size_t)i * kChunk) * a.vs + (size_t)h * a.V,
                                   left(i), vst, a.V * es);
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    next[x][t][j] = load_one<E>(r, voff[x], (16 * t + j) * vst);
    };
    float z = 0.0f;
    if (chunks) fetch(0);
    lds_barrier();
    for (uint32_t ci = 0; ci < chunks; ++ci) {
        const Chunk& o = buf[ci & 1];
        f32x4 v[NT][2], aq[NT][2] = {}, ak[NT][2] = {};
        // Operands of 32 channels, the next ones on their way while these are
        // multiplied.
        constexpr int kParts = Terms::kKeyLo ? 2 : 1;
        f16x8 kf[2][kParts][2], qf[2][kParts][2];
        auto operands = [&](int b) {
#pragma unroll
            for (int p = 0; p < kParts; ++p)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    kf[b & 1][p][t] = o.K[p][t][b][lane];
                    qf[b & 1][p][t] = o.Q[p][t][b][lane];
                }
        };
        operands(0);
        float most[NT];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            most[x] = 0.0f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float y = Elem<DT>::load(next[x][t][j]);
                    z = __builtin_fmaf(y, 0.0f, z);
                    v[x][t][j] = __builtin_ldexpf(y, -shift[x]);
                    most[x] = fmaxf(most[x], fabsf(v[x][t][j]) * kOperand);
                }
#pragma unroll
            for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) most[x] = fmaxf(most[x], fabsf(S[x][t][i]));
        }
        fetch(ci + 1);
        // Column sizes near 1 leave both the products' growth and the parts
        // below hi their room.
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            const float all = max_groups(most[x]);
            const bool off = all > 32.0f * kOperand || (all < 0.5f * kOperand && all > 0.0f);
            if (__any(off)) {
                const int d = off ? __builtin_amdgcn_frexp_expf(all) - 3 - 6 : 0;
                shift[x] += d;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[x][t][j] = __builtin_ldexpf(v[x][t][j], -d);
#pragma unroll
                for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[x][t][i] = __builtin_ldexpf(S[x][t][i], -d);
            }
        }
        // (P k) S and (P q) S; the products of one sum lie apart.
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            if (b + 1 < KB) operands(b + 1);
            __builtin_amdgcn_sched_barrier(0);
            Pair8 s[NT];
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                const f32x4 &l = S[x][2 * b], &u = S[x][2 * b + 1];
                const float y[8] = {l[0], l[1], l[2], l[3], u[0], u[1], u[2], u[3]};
                s[x] = split8(y);
            }
            const auto& kp = kf[b & 1];
            const auto& qp = qf[b & 1];
            if (Terms::kKeyLo) {
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        ak[x][t] = mfma_f16(kp[kParts - 1][t], s[x].hi, ak[x][t]);
                        aq[x][t] = mfma_f16(qp[kParts - 1][t], s[x].hi, aq[x][t]);
                    }
            }
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    ak[x][t] = mfma_f16(kp[0][t], s[x].lo, ak[x][t]);
                    aq[x][t] = mfma_f16(qp[0][t], s[x].lo, aq[x][t]);
                }
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    ak[x][t] = mfma_f16(kp[0][t], s[x].hi, ak[x][t]);
                    aq[x][t] = mfma_f16(qp[0][t], s[x].hi, aq[x][t]);
                }
            // The state's decay, for the update.
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const f32x4 f =
                    *reinterpret_cast<const f32x4*>(&o.decay[16 * (2 * b + y) + 4 * g]);
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[x][2 * b + y][i] *= f[i];
            }
        }
        // A column that a product would take past f16 is made smaller.
        auto fit = [&](f32x4 (&y)[2], int x) {
            float big = 0.0f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) big = fmaxf(big, fabsf(y[t][j]));
            if (!__any(big > 16384.0f)) return;
            big = max_groups(big);
            const int d = big > 16384.0f ? __builtin_amdgcn_frexp_expf(big) - 5 : 0;
            shift[x] += d;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[t][j] = __builtin_ldexpf(y[t][j], -d);
                    aq[x][t][j] = __builtin_ldexpf(aq[x][t][j], -d);
                }
#pragma unroll
            for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[x][t][i] = __builtin_ldexpf(S[x][t][i], -d);
        };
        auto operand = [&](const f32x4 (&x)[2]) {
            const float y[8] = {x[0][0], x[0][1], x[0][2], x[0][3],
                                x[1][0], x[1][1], x[1][2], x[1][3]};
            return split8(y);
        };
        auto factors = [&](const float* f, int t) {
            return *reinterpret_cast<const f32x4*>(f + 16 * t + 4 * g);
        };
        f32x4 u[NT][2];
        Pair8 up[NT];
        {
            f16x8 tf[2][2];
            f32x4 rt[2], rr[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                tf[0][t] = o.T[t][0][lane];
                tf[1][t] = o.T[t][1][lane];
                rr[t] = factors(o.row_r, t);
                rt[t] = factors(o.row_t, t);
            }
#pragma unroll
            for (int x = 0; x < NT; ++x) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        u[x][t][j] = __builtin_fmaf(-rr[t][j], ak[x][t][j], v[x][t][j]);
                fit(u[x], x);
                up[x] = operand(u[x]);
                u[x][0] = u[x][1] = f32x4{};
            }
#pragma unroll
            for (int y = 0; y < 3; ++y)
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        u[x][t] = mfma_f16(tf[y == 0][t], y == 1 ? up[x].lo : up[x].hi, u[x][t]);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) u[x][t][j] *= rt[t][j];
                fit(u[x], x);
                up[x] = operand(u[x]);
            }
        }
        f32x4 ap[NT][2] = {};
        {
            f16x8 pf[2][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                pf[0][t] = o.P[t][0][lane];
                pf[1][t] = o.P[t][1][lane];
            }
#pragma unroll
            for (int y = 0; y < 3; ++y)
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        ap[x][t] = mfma_f16(pf[y == 0][t], y == 1 ? up[x].lo : up[x].hi, ap[x][t]);
        }
        if (!CHANNEL) {
#pragma unroll
            for (int x = 0; x < NT; ++x) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const f32x4 f = factors(o.row_u, t);
#pragma unroll
                    for (int j = 0; j < 4; ++j) u[x][t][j] *= f[j];
                }
                up[x] = operand(u[x]);
            }
        }
        // The state's update, two tiles of channels at a time.
        f16x8 tk[2][kParts][2];
        auto channels = [&](int y) {
#pragma unroll
            for (int p = 0; p < kParts; ++p)
#pragma unroll
                for (int t = 0; t < 2; ++t) tk[y & 1][p][t] = o.Kt[p][2 * y + t][lane];
        };
        channels(0);
#pragma unroll
        for (int y = 0; y < KB; ++y) {
            if (y + 1 < KB) channels(y + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (Terms::kKeyLo) {
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        S[x][2 * y + t] =
                            mfma_f16(tk[y & 1][kParts - 1][t], up[x].hi, S[x][2 * y + t]);
            }
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    S[x][2 * y + t] = mfma_f16(tk[y & 1][0][t], up[x].lo, S[x][2 * y + t]);
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    S[x][2 * y + t] = mfma_f16(tk[y & 1][0][t], up[x].hi, S[x][2 * y + t]);
        }
        const auto outs = rows_buffer(static_cast<E*>(a.out) +
                                          (begin + (size_t)ci * kChunk) * a.os + (size_t)h * a.V,
                                      left(ci), ost, a.V * es);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const f32x4 fo = factors(o.row_o, t), fp = factors(o.row_p, t);
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float y = __builtin_fmaf(fp[j], ap[x][t][j], fo[j] * aq[x][t][j]);
                    store_one<E>(Elem<DT>::store(__builtin_ldexpf(y, shift[x])), outs, ooff[x],
                                 (16 * t + j) * ost);
                }
        }
        lds_barrier();
    }
    if (z != z) latch(a.status, K3X_ERR_INVALID_MXFP4);
    if (!a.state_out || (!chunks && a.state_in == a.state_out)) return;
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t r = 16 * t + 4 * g + i;
                if (r < a.K && col[x] < a.V)
                    a.state_out[base + (size_t)r * a.V + col[x]] =
                        __builtin_ldexpf(S[x][t][i], shift[x] - 6);
            }
}

// Chunks for sequences that fill one and heads that the products' tiles take.
constexpr uint32_t kChunkMinTokens = 24;

bool runs_in_chunks(const k3x_hip_delta_params* p) {
    const uint32_t longest =
        p->longest ? p->longest : (p->tokens + p->sequences - 1) / p->sequences;
    return p->key_dim <= 128 && longest >= kChunkMinTokens;
}

uint64_t chunk_slots(const k3x_hip_delta_params* p) { return p->tokens / kChunk + p->sequences; }

template <uint32_t DT, bool CHANNEL, int KB>
int launch_chunks(k3x_hip_ctx* ctx, const DeltaArgs& a, ChunkRecord* records, uint32_t slots,
                  bool vec) {
    hipLaunchKernelGGL((delta_prep_kernel<DT, CHANNEL, KB>), dim3(slots * a.H), dim3(128), 0,
                       ctx->stream, a, records, vec);
    const uint32_t heads = a.N * a.H;
    if (a.V > 64 && heads >= ctx->cu_count / 2)
        hipLaunchKernelGGL((delta_scan_kernel<DT, CHANNEL, KB, 2>),
                           dim3(heads * ((a.V + 127) / 128)), dim3(512), 0, ctx->stream, a, records,
                           vec);
    else
        hipLaunchKernelGGL((delta_scan_kernel<DT, CHANNEL, KB, 1>),
                           dim3(heads * ((a.V + 63) / 64)), dim3(512), 0, ctx->stream, a, records,
                           vec);
    return launched(ctx, 2);
}

template <uint32_t DT>
int launch_chunks_of(k3x_hip_ctx* ctx, const DeltaArgs& a, ChunkRecord* records, uint32_t slots,
                     bool channel, bool vec) {
    if (a.K <= 64)
        return channel ? launch_chunks<DT, true, 2>(ctx, a, records, slots, vec)
                       : launch_chunks<DT, false, 2>(ctx, a, records, slots, vec);
    return channel ? launch_chunks<DT, true, 4>(ctx, a, records, slots, vec)
                   : launch_chunks<DT, false, 4>(ctx, a, records, slots, vec);
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
           // workgroups of a launch
           (uint64_t)p->sequences * p->value_heads * 16 < (1ull << 31) &&
           ((uint64_t)p->tokens / 32 + p->sequences) * p->value_heads < (1ull << 31);
}

}  // namespace

extern "C" {

size_t k3x_hip_delta_workspace(const k3x_hip_delta_params* p) {
    if (!p || !delta_ok(p) || !runs_in_chunks(p)) return 0;
    return chunk_slots(p) * p->value_heads * sizeof(ChunkRecord);
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
    if (need) {
        // Four elements a load: rows and heads that keep the alignment.
        const bool vec = a.K % 4 == 0 && a.qs % 4 == 0 && a.ks % 4 == 0 && aligned(q, 4 * es) &&
                         aligned(k, 4 * es) && aligned(gate, 16);
        ChunkRecord* records = static_cast<ChunkRecord*>(workspace);
        const uint32_t slots = (uint32_t)chunk_slots(p);
        const bool channel = p->gate == K3X_GATE_CHANNEL;
        return p->dtype == K3X_DTYPE_F32
                   ? launch_chunks_of<K3X_DTYPE_F32>(ctx, a, records, slots, channel, vec)
               : p->dtype == K3X_DTYPE_BF16
                   ? launch_chunks_of<K3X_DTYPE_BF16>(ctx, a, records, slots, channel, vec)
                   : launch_chunks_of<K3X_DTYPE_F16>(ctx, a, records, slots, channel, vec);
    }
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
