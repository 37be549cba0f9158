// verify.hip -- verification of drafted tokens against the target's rows.
//
// Four launches: each row's parts (largest entry, sum of exponentials), the
// accepted count of each sequence, the parts' sums of the distribution that
// its next token is drawn from, and the draw.  Everything that a choice
// rests on is formed in double: the sums run over a whole vocabulary, and
// the drawn token sits next to a border of the cumulative sum.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "k3x_ops.hpp"

using namespace k3x_dev;
using namespace k3x_ops;

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxParts = 64;  // parts of a row
constexpr uint32_t kPartEntries = 4096;

// A row's entries [part * len, ...) by workgroup.  max NaN: the part holds an
// entry that no row may.
struct RowPart {
    double sum;        // sum of exp((l - max) / temperature)
    float max;
    uint32_t arg;      // first entry that is max
};

// What the draw needs of sequence n.
struct Drawn {
    uint32_t accepted, rows;  // rows: drafts of this sequence
    uint32_t bad;             // status to latch, 0
    uint32_t next;            // greedy: the next token
    double pmax, pinv, qmax, qinv;
};

struct VerifyArgs {
    const void *target, *draft;
    const uint32_t *tokens, *draft_counts;
    const float *accept_u, *sample_u;
    uint32_t *accepted, *out_tokens;
    uint32_t N, D, V, stride;
    uint32_t parts, part_len;
    uint32_t form, greedy;
    double temperature;
    RowPart* row_parts;   // [N (2 D + 1)][parts]: a sequence's target rows, then its draft's
    Drawn* drawn;         // [N]
    double* sums;         // [N][parts]
    uint32_t* status;
};

__device__ inline uint32_t drafts_of(const VerifyArgs& a, uint32_t n) {
    return a.draft_counts ? a.draft_counts[n] : a.D;
}

template <uint32_t DT>
__device__ inline const typename Elem<DT>::type* row_of(const VerifyArgs& a, uint32_t n,
                                                        uint32_t r) {
    typedef const typename Elem<DT>::type* P;
    return r <= a.D ? static_cast<P>(a.target) + ((size_t)n * (a.D + 1) + r) * a.stride
                    : static_cast<P>(a.draft) + ((size_t)n * a.D + (r - a.D - 1)) * a.stride;
}

__device__ inline size_t part_index(const VerifyArgs& a, uint32_t n, uint32_t r) {
    return ((size_t)n * (2 * a.D + 1) + r) * a.parts;
}

// The larger of two (entry, index) pairs, the lower index on a tie.
__device__ inline void take_max(float& m, uint32_t& i, float om, uint32_t oi) {
    if (om > m || (om == m && oi < i)) {
        m = om;
        i = oi;
    }
}

template <uint32_t DT>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyArgs a) {
    __shared__ float sm[kThreads / 64];
    __shared__ uint32_t si[kThreads / 64];
    __shared__ double sd[kThreads / 64];
    const uint32_t part = blockIdx.x % a.parts, rr = blockIdx.x / a.parts;
    const uint32_t rows = a.draft ? 2 * a.D + 1 : a.D + 1;
    const uint32_t n = rr / rows, r = rr % rows, tid = threadIdx.x, wave = tid >> 6;
    const uint32_t count = drafts_of(a, n);
    if (__syncthreads_or(*(volatile uint32_t*)a.status)) return;
    if (count > a.D || (r <= a.D ? r > count : r - a.D - 1 >= count)) return;
    const auto* x = row_of<DT>(a, n, r);
    const uint32_t lo = part * a.part_len, hi = min(a.V, lo + a.part_len);
    float m = -__builtin_inff();
    uint32_t arg = 0xffffffffu;
    bool wrong = false;
    for (uint32_t i = lo + tid; i < hi; i += kThreads) {
        const float l = Elem<DT>::load(x[i]);
        wrong |= !(l < __builtin_inff()) || (a.form == K3X_DIST_PROBS && l < 0.0f);
        take_max(m, arg, l, i);
    }
    for (int d = 1; d < 64; d <<= 1)
        take_max(m, arg, __shfl_xor(m, d), (uint32_t)__shfl_xor((int)arg, d));
    if ((tid & 63) == 0) {
        sm[wave] = m;
        si[wave] = arg;
    }
    wrong = __syncthreads_or(wrong);
    for (uint32_t w = 0; w < kThreads / 64; ++w) take_max(m, arg, sm[w], si[w]);
    double s = 0.0;
    if (!a.greedy && m > -__builtin_inff())
        for (uint32_t i = lo + tid; i < hi; i += kThreads)
            s += exp(((double)Elem<DT>::load(x[i]) - (double)m) / a.temperature);
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if ((tid & 63) == 0) sd[wave] = s;
    __syncthreads();
    if (tid) return;
    s = 0.0;
    for (uint32_t w = 0; w < kThreads / 64; ++w) s += sd[w];
    a.row_parts[part_index(a, n, r) + part] =
        RowPart{s, wrong ? __builtin_nanf("") : m, arg};
}

// A row's largest entry and 1 / sum from its parts, by a wave (lane = part);
// false: the row is unfit.
__device__ inline bool row_total(const VerifyArgs& a, uint32_t n, uint32_t r, double* mx,
                                 double* inv, uint32_t* arg) {
    const uint32_t lane = threadIdx.x & 63;
    RowPart p{0.0, -__builtin_inff(), 0xffffffffu};
    if (lane < a.parts) p = a.row_parts[part_index(a, n, r) + lane];
    if (__any(p.max != p.max)) return false;
    float m = p.max;
    uint32_t at = p.arg;
    for (int d = 1; d < 64; d <<= 1)
        take_max(m, at, __shfl_xor(m, d), (uint32_t)__shfl_xor((int)at, d));
    if (m == -__builtin_inff() || (a.form == K3X_DIST_PROBS && m == 0.0f)) return false;
    double s = p.sum > 0.0 ? p.sum * exp(((double)p.max - (double)m) / a.temperature) : 0.0;
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    *mx = m;
    *inv = 1.0 / s;
    *arg = at;
    return true;
}

__device__ inline double prob(const VerifyArgs& a, float l, double mx, double inv) {
    return a.form == K3X_DIST_PROBS ? (double)l : exp(((double)l - mx) / a.temperature) * inv;
}

// One wave a sequence walks its drafts (every lane the same).
template <uint32_t DT>
__global__ __launch_bounds__(64) void verify_accept_kernel(VerifyArgs a) {
    if (*(volatile uint32_t*)a.status) return;
    const uint32_t n = blockIdx.x;
    const uint32_t count = drafts_of(a, n);
    Drawn d{};
    d.rows = count;
    d.pinv = d.qinv = 1.0;
    const bool totals = a.form == K3X_DIST_LOGITS || a.greedy;
    uint32_t arg = 0, i = 0;
    if (count > a.D && count != K3X_VERIFY_SKIP) d.bad = K3X_ERR_INVALID_STATE;
    for (; !d.bad && count != K3X_VERIFY_SKIP; ++i) {
        if (totals && !row_total(a, n, i, &d.pmax, &d.pinv, &arg)) d.bad = K3X_ERR_INVALID_STATE;
        if (d.bad || i == count) break;
        const uint32_t x = a.tokens[(size_t)n * a.D + i];
        if (x >= a.V) {
            d.bad = K3X_ERR_INVALID_STATE;
            break;
        }
        if (a.greedy) {
            if (arg != x) break;
            continue;
        }
        const float u = a.accept_u[(size_t)n * a.D + i];
        const double p = prob(a, Elem<DT>::load(row_of<DT>(a, n, i)[x]), d.pmax, d.pinv);
        double q = 1.0;
        if (a.draft) {
            if (totals && !row_total(a, n, a.D + 1 + i, &d.qmax, &d.qinv, &arg)) {
                d.bad = K3X_ERR_INVALID_STATE;
                break;
            }
            q = prob(a, Elem<DT>::load(row_of<DT>(a, n, a.D + 1 + i)[x]), d.qmax, d.qinv);
        }
        if (!(u >= 0.0f && u < 1.0f) || !(p >= 0.0 && p < __builtin_inf()) ||
            !(q >= 0.0 && q < __builtin_inf())) {
            d.bad = K3X_ERR_INVALID_STATE;
            break;
        }
        if (!((double)u * q < p)) break;
    }
    d.accepted = count == K3X_VERIFY_SKIP ? 0 : i;
    d.next = arg;
    if (threadIdx.x == 0) a.drawn[n] = d;
}

// The distribution that sequence n's next token is drawn from: entry i is
// max(p_i - q_i, 0) at a draft that was not accepted (p_i without the drafted
// token where there is no q), else p_i.  NaN: an entry that no row may hold.
template <uint32_t DT>
struct Rest {
    typedef typename Elem<DT>::type E;
    const E *p, *q;
    double pmax, pinv, qmax, qinv;
    uint32_t token;  // 0xffffffff: none
    __device__ Rest(const VerifyArgs& a, const Drawn& d, uint32_t n) {
        const bool reject = d.accepted < d.rows;
        p = row_of<DT>(a, n, d.accepted);
        q = reject && a.draft ? row_of<DT>(a, n, a.D + 1 + d.accepted) : nullptr;
        token = reject && !q ? a.tokens[(size_t)n * a.D + d.accepted] : 0xffffffffu;
        pmax = d.pmax;
        pinv = d.pinv;
        qmax = d.qmax;
        qinv = d.qinv;
    }
    __device__ inline double at(const VerifyArgs& a, uint32_t i) const {
        const double r = prob(a, Elem<DT>::load(p[i]), pmax, pinv);
        const double o = q ? prob(a, Elem<DT>::load(q[i]), qmax, qinv) : 0.0;
        if (!(r >= 0.0 && o >= 0.0 && o < __builtin_inf())) return __builtin_nan("");
        return i == token || r <= o ? 0.0 : r - o;
    }
    // Only the target's probabilities.
    __device__ inline void whole() {
        q = nullptr;
        token = 0xffffffffu;
    }
};

__device__ inline double block_sum(double s, double* sd) {
    for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sd[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
    for (uint32_t w = 0; w < kThreads / 64; ++w) s += sd[w];
    return s;
}

template <uint32_t DT>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a) {
    __shared__ double sd[kThreads / 64];
    const uint32_t part = blockIdx.x % a.parts, n = blockIdx.x / a.parts, tid = threadIdx.x;
    if (__syncthreads_or(*(volatile uint32_t*)a.status)) return;
    const Drawn d = a.drawn[n];
    if (d.bad || d.rows == K3X_VERIFY_SKIP) return;
    const Rest<DT> rest(a, d, n);
    const uint32_t lo = part * a.part_len, hi = min(a.V, lo + a.part_len);
    double s = 0.0;
    for (uint32_t i = lo + tid; i < hi; i += kThreads) s += rest.at(a, i);
    s = block_sum(s, sd);
    if (tid == 0) a.sums[(size_t)n * a.parts + part] = s;
}

// The token of [lo, hi) that the border falls in: the last entry over 0 that
// the cumulative sum (start before lo) has not passed the border before.
// By the whole workgroup; the range holds an entry over 0 and start <= border.
template <uint32_t DT>
__device__ inline uint32_t draw_token(const VerifyArgs& a, const Rest<DT>& rest, uint32_t lo,
                                      uint32_t hi, double start, double border, double* sd,
                                      uint32_t* found) {
    const uint32_t tid = threadIdx.x, per = (hi - lo + kThreads - 1) / kThreads;
    const uint32_t b = min(hi, lo + tid * per), e = min(hi, b + per);
    double s = 0.0;
    for (uint32_t i = b; i < e; ++i) s += rest.at(a, i);
    __syncthreads();
    sd[tid] = s;
    if (tid == 0) *found = 0;
    __syncthreads();
    double c = start;
    for (uint32_t w = 0; w < tid; ++w) c += sd[w];
    uint32_t hit = 0;
    for (uint32_t i = b; i < e && c <= border; ++i) {
        const double r = rest.at(a, i);
        c += r;
        if (r > 0.0) hit = i + 1;
    }
    if (hit) atomicMax(found, hit);
    __syncthreads();
    return *found - 1;
}

// One workgroup a sequence: the part that the drawn border falls in, then the
// entry, then the sequence's outputs.
template <uint32_t DT>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a) {
    __shared__ double sd[kThreads];
    __shared__ uint32_t found;
    const uint32_t n = blockIdx.x, tid = threadIdx.x;
    if (__syncthreads_or(*(volatile uint32_t*)a.status)) return;
    const Drawn d = a.drawn[n];
    uint32_t* out = a.out_tokens + (size_t)n * (a.D + 1);
    if (d.rows == K3X_VERIFY_SKIP) {
        if (tid == 0) a.accepted[n] = 0;
        if (tid <= a.D) out[tid] = 0xffffffffu;
        return;
    }
    uint32_t bad = d.bad, next = d.next;
    if (!bad && !a.greedy) {
        const float u = a.sample_u[n];
        double total = 0.0;
        for (uint32_t i = 0; i < a.parts; ++i) total += a.sums[(size_t)n * a.parts + i];
        if (!(u >= 0.0f && u < 1.0f) || !(total >= 0.0 && total < __builtin_inf())) {
            bad = K3X_ERR_INVALID_STATE;
        } else {
            Rest<DT> rest(a, d, n);
            uint32_t lo = 0, hi = a.V;
            double start = 0.0, border = (double)u * total;
            if (total > 0.0) {
                double before = 0.0;
                uint32_t part = 0;
                for (uint32_t i = 0; i < a.parts; ++i) {
                    const double s = a.sums[(size_t)n * a.parts + i];
                    if (s > 0.0 && before <= border) {
                        part = i;
                        start = before;
                    }
                    before += s;
                }
                lo = part * a.part_len;
                hi = min(a.V, lo + a.part_len);
            } else {
                // Nothing is left over q (or of a row without its drafted
                // token): the target's own probabilities.
                rest.whole();
                double s = 0.0;
                for (uint32_t i = tid; i < a.V; i += kThreads) s += rest.at(a, i);
                total = block_sum(s, sd);
                border = (double)u * total;
                if (!(total > 0.0 && total < __builtin_inf())) bad = K3X_ERR_INVALID_STATE;
            }
            if (!bad) next = draw_token<DT>(a, rest, lo, hi, start, border, sd, &found);
        }
    }
    if (bad) {
        if (tid == 0) latch(a.status, bad);
        return;
    }
    if (tid == 0) a.accepted[n] = d.accepted;
    if (tid <= a.D)
        out[tid] = tid < d.accepted    ? a.tokens[(size_t)n * a.D + tid]
                   : tid == d.accepted ? next
                                       : 0xffffffffu;
}

template <uint32_t DT>
int launch_verify(k3x_hip_ctx* ctx, const VerifyArgs& a) {
    unsigned launches = 2;
    if (a.form == K3X_DIST_LOGITS || a.greedy) {
        const uint32_t rows = a.draft ? 2 * a.D + 1 : a.D + 1;
        hipLaunchKernelGGL(verify_rows_kernel<DT>, dim3(a.N * rows * a.parts), dim3(kThreads), 0,
                           ctx->stream, a);
        ++launches;
    }
    hipLaunchKernelGGL(verify_accept_kernel<DT>, dim3(a.N), dim3(64), 0, ctx->stream, a);
    if (!a.greedy) {
        hipLaunchKernelGGL(verify_sums_kernel<DT>, dim3(a.N * a.parts), dim3(kThreads), 0,
                           ctx->stream, a);
        ++launches;
    }
    hipLaunchKernelGGL(verify_draw_kernel<DT>, dim3(a.N), dim3(kThreads), 0, ctx->stream, a);
    return launched(ctx, launches);
}

bool verify_ok(const k3x_hip_verify_params* p) {
    return p->sequences && p->sequences <= 65535 && p->drafts <= 64 && p->vocab &&
           p->vocab <= (1u << 20) && p->dtype <= K3X_DTYPE_BF16 && p->form <= K3X_DIST_PROBS &&
           p->greedy <= 1 && std::isfinite(p->temperature) && p->temperature > 0.0f &&
           (!p->row_stride || p->row_stride >= p->vocab) &&
           (uint64_t)p->sequences * (2 * p->drafts + 1) * kMaxParts < (1ull << 31);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

uint32_t parts_of(const k3x_hip_verify_params* p) {
    return std::min((p->vocab + kPartEntries - 1) / kPartEntries, kMaxParts);
}

}  // namespace

extern "C" {

size_t k3x_hip_verify_workspace(const k3x_hip_verify_params* p) {
    if (!p || !verify_ok(p)) return 0;
    const size_t n = p->sequences, parts = parts_of(p);
    return up256(n * (2 * p->drafts + 1) * parts * sizeof(RowPart)) + up256(n * sizeof(Drawn)) +
           up256(n * parts * sizeof(double));
}

int k3x_hip_verify_draft(k3x_hip_ctx* ctx, const k3x_hip_verify_params* p, const void* target,
                         const void* draft, const uint32_t* tokens, const uint32_t* draft_counts,
                         const float* accept_u, const float* sample_u, uint32_t* accepted,
                         uint32_t* out_tokens, void* workspace, size_t workspace_bytes) {
    if (!ctx || !p || !verify_ok(p) || !target || !accepted || !out_tokens)
        return K3X_ERR_INVALID_EXTENT;
    if (p->drafts && !tokens) return K3X_ERR_INVALID_EXTENT;
    if (!p->greedy && (!sample_u || (p->drafts && !accept_u))) return K3X_ERR_INVALID_EXTENT;
    const uintptr_t es = p->dtype == K3X_DTYPE_F32 ? 4 : 2;
    if (!aligned(target, es) || !aligned(draft, es) || !aligned(tokens, 4) ||
        !aligned(draft_counts, 4) || !aligned(accept_u, 4) || !aligned(sample_u, 4) ||
        !aligned(accepted, 4) || !aligned(out_tokens, 4))
        return K3X_ERR_INVALID_EXTENT;
    const size_t need = k3x_hip_verify_workspace(p);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 256))
        return K3X_ERR_INVALID_EXTENT;
    if (hipSetDevice(ctx->device) != hipSuccess) return K3X_ERR_BACKEND_UNAVAILABLE;
    VerifyArgs a{};
    a.target = target;
    a.draft = p->greedy ? nullptr : draft;
    a.tokens = tokens;
    a.draft_counts = draft_counts;
    a.accept_u = accept_u;
    a.sample_u = sample_u;
    a.accepted = accepted;
    a.out_tokens = out_tokens;
    a.N = p->sequences;
    a.D = p->drafts;
    a.V = p->vocab;
    a.stride = p->row_stride ? p->row_stride : p->vocab;
    a.parts = parts_of(p);
    a.part_len = (a.V + a.parts - 1) / a.parts;
    a.form = p->form;
    a.greedy = p->greedy;
    a.temperature = p->temperature;
    uint8_t* w = static_cast<uint8_t*>(workspace);
    a.row_parts = reinterpret_cast<RowPart*>(w);
    w += up256((size_t)a.N * (2 * a.D + 1) * a.parts * sizeof(RowPart));
    a.drawn = reinterpret_cast<Drawn*>(w);
    w += up256((size_t)a.N * sizeof(Drawn));
    a.sums = reinterpret_cast<double*>(w);
    a.status = ctx->status;
    return p->dtype == K3X_DTYPE_F32 ? launch_verify<K3X_DTYPE_F32>(ctx, a)
                                     : launch_verify<K3X_DTYPE_BF16>(ctx, a);
}

}  // extern "C"
