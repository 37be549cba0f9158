// verify.hip -- verification of drafted tokens against the target's rows.
//
//   rows     each row by parts of 1024 entries, a wave each: the largest entry and
//            the sum of exponentials over it (logits, and greedy choices);
//   accept   one workgroup a sequence: every row's totals and drafted token's
//            probabilities at once, then the walk over the drafts;
//   draw     the row that the next token is drawn from, by the same parts: their
//            sums, and by the sequence's last workgroup the part and the entry
//            that the border falls in.
//
// Everything that a choice rests on is formed in double: the sums run over a
// whole vocabulary, and a drawn token lies next to a border of the cumulative
// sum (at 10^5 entries a sum off by 10^-9 moves one draw in 10^4).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "k3x_ops.hpp"

using namespace k3x_dev;
using namespace k3x_ops;

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kEntries = 16;  // of a part, a lane
constexpr uint32_t kPart = 64 * kEntries;  // a wave's
constexpr uint32_t kWaves = kThreads / 64;
constexpr uint32_t kMaxDrafts = 64;

// One part of a row; max NaN: it holds an entry that no row may.
struct RowPart {
    double sum;    // of exp((l - max) / temperature)
    float max;
    uint32_t arg;  // first entry that is max
};

// What the draw needs of a sequence.
struct Drawn {
    uint32_t accepted, rows;  // rows: drafts of this sequence, or K3X_VERIFY_SKIP
    uint32_t done;            // its result is out (or it is unfit)
    uint32_t arrived;         // workgroups of the draw that have written their sum
    double pmax, pinv, qmax, qinv;
};

struct VerifyArgs {
    const void *target, *draft;
    const uint32_t *tokens, *draft_counts;
    const float *accept_u, *sample_u;
    uint32_t *accepted, *out_tokens;
    uint32_t N, D, V, stride;
    uint32_t parts;     // of a row
    uint32_t form, greedy;
    uint32_t vec;       // rows by 16 bytes
    double rate;        // log2(e) / temperature
    RowPart* row_parts; // [N (2 D + 1)][parts]: a sequence's target rows, then its draft's
    Drawn* drawn;       // [N]
    double* sums;       // [N][parts]
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

// 2^y in double, y <= 0 (a NaN gives 0: a row that holds one is unfit): the series
// (ln2 f)^n / n! to n = 11 on |f| <= 1 / 2, 9e-15 of it at most before roundings.
__device__ inline double exp2_f64(double y) {
    y = __builtin_fmax(y, -1080.0);  // 2^y is 0 from there on
    const double k = __builtin_rint(y), f = y - k;
    double p = 4.4455382718708116e-10;
    p = __builtin_fma(p, f, 7.054911620801123e-09);
    p = __builtin_fma(p, f, 1.01780860092397e-07);
    p = __builtin_fma(p, f, 1.321548679014431e-06);
    p = __builtin_fma(p, f, 1.5252733804059841e-05);
    p = __builtin_fma(p, f, 0.0001540353039338161);
    p = __builtin_fma(p, f, 0.0013333558146428443);
    p = __builtin_fma(p, f, 0.009618129107628477);
    p = __builtin_fma(p, f, 0.05550410866482158);
    p = __builtin_fma(p, f, 0.24022650695910072);
    p = __builtin_fma(p, f, 0.6931471805599453);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)k);
}

// A lane's sixteen entries of a part, neighbours by 16 bytes where rows are, so
// that a wave's loads are whole lines; where() rises with j.  By 16 bytes against
// by one entry, all launches: 131072 and 131073 probabilities of 64 sequences 26
// and 28 us, logits of 16 sequences of 4 drafts 43 and 47.
template <uint32_t DT>
struct Entries {
    typedef typename Elem<DT>::type E;
    static constexpr uint32_t kWide = 16 / sizeof(E);
    static __device__ inline uint32_t where(const VerifyArgs& a, uint32_t lo, uint32_t lane,
                                            int j) {
        return a.vec ? lo + j / kWide * (64 * kWide) + lane * kWide + j % kWide
                     : lo + j * 64 + lane;
    }
    // Past hi: `past`.
    static __device__ inline void load(const VerifyArgs& a, const E* x, uint32_t lo, uint32_t hi,
                                       uint32_t lane, float past, float (&l)[kEntries]) {
        typedef E Vec __attribute__((ext_vector_type(kWide)));
        if (a.vec && lo + kPart <= hi) {
#pragma unroll
            for (int j = 0; j < (int)kEntries; j += kWide) {
                const Vec v = *reinterpret_cast<const Vec*>(x + where(a, lo, lane, j));
#pragma unroll
                for (int y = 0; y < (int)kWide; ++y) l[j + y] = Elem<DT>::load(v[y]);
            }
        } else if (lo + kPart <= hi) {
#pragma unroll
            for (int j = 0; j < (int)kEntries; ++j) l[j] = Elem<DT>::load(x[lo + lane + j * 64]);
        } else {
#pragma unroll
            for (int j = 0; j < (int)kEntries; ++j) {
                const uint32_t i = where(a, lo, lane, j);
                l[j] = Elem<DT>::load(x[min(i, hi - 1)]);
                if (i >= hi) l[j] = past;
            }
        }
    }
};

// Parts of a row by waves, which do not wait for one another.  16 sequences of 4
// drafts and 100003 fp32 logits (58 MB): 17 us, 3.4 TB/s; the exponentials in
// double, some 18 operations each, take 7 us of it at the unit's rate.
template <uint32_t DT>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyArgs a) {
    const uint32_t rows = a.draft ? 2 * a.D + 1 : a.D + 1;
    const uint32_t blocks = (a.parts + kWaves - 1) / kWaves;
    const uint32_t rr = blockIdx.x / blocks, n = rr / rows, r = rr % rows, lane = threadIdx.x & 63;
    const uint32_t part = blockIdx.x % blocks * kWaves +
                          __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t count = drafts_of(a, n);
    if (part >= a.parts || count > a.D || (r <= a.D ? r > count : r - a.D - 1 >= count))
        return;
    typedef Entries<DT> Mine;
    const uint32_t lo = part * kPart, hi = min(a.V, lo + kPart);
    float l[kEntries];
    Mine::load(a, row_of<DT>(a, n, r), lo, hi, lane, -__builtin_inff(), l);
    if (*(volatile uint32_t*)a.status) return;
    float m = -__builtin_inff();
    uint32_t arg = 0xffffffffu;
    bool wrong = false;
#pragma unroll
    for (int j = 0; j < (int)kEntries; ++j) wrong |= !(l[j] < __builtin_inff());
    if (!a.greedy) {
#pragma unroll
        for (int j = 0; j < (int)kEntries; ++j) m = fmaxf(m, l[j]);
    } else {
#pragma unroll
        for (int j = 0; j < (int)kEntries; ++j)
            if (l[j] > m) {
                m = l[j];
                arg = Mine::where(a, lo, lane, j);
            }
        // Past the row's end minus infinity: no entry of a row of
        // probabilities, but not one that is looked at either.
        if (a.form == K3X_DIST_PROBS)
#pragma unroll
            for (int j = 0; j < (int)kEntries; ++j)
                wrong |= l[j] < 0.0f && Mine::where(a, lo, lane, j) < hi;
    }
    const float top = unordered(wave_max_u32(ordered(m)));
    if (a.greedy) arg = ~wave_max_u32(m == top ? ~arg : 0u);
    double s = 0.0;
    if (!a.greedy && top > -__builtin_inff()) {
#pragma unroll
        for (int j = 0; j < (int)kEntries; ++j)
            s += exp2_f64(((double)l[j] - (double)top) * a.rate);
        s = wave_sum(s);
    }
    wrong = __any(wrong);
    if (lane == 0)
        a.row_parts[part_index(a, n, r) + part] = RowPart{s, wrong ? __builtin_nanf("") : top, arg};
}

// A row's largest entry and 1 / sum from its parts, by a wave; false: the row
// is unfit.
__device__ inline bool row_total(const VerifyArgs& a, uint32_t n, uint32_t r, double* mx,
                                 double* inv, uint32_t* arg) {
    const uint32_t lane = threadIdx.x & 63;
    const RowPart* parts = a.row_parts + part_index(a, n, r);
    float m = -__builtin_inff();
    uint32_t at = 0xffffffffu;
    bool nan = false;
    for (uint32_t i = lane; i < a.parts; i += 64) {
        nan |= parts[i].max != parts[i].max;
        take_max(m, at, parts[i].max, parts[i].arg);
    }
    if (__any(nan)) return false;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
        take_max(m, at, __shfl_xor(m, d), (uint32_t)__shfl_xor((int)at, d));
    if (m == -__builtin_inff() || (a.form == K3X_DIST_PROBS && m == 0.0f)) return false;
    double s = 0.0;
    if (!a.greedy)
        for (uint32_t i = lane; i < a.parts; i += 64)
            if (parts[i].sum > 0.0)
                s += parts[i].sum *
                     exp2_f64(((double)parts[i].max - (double)m) * a.rate);
    *mx = m;
    *inv = 1.0 / wave_sum(s);
    *arg = at;
    return true;
}

__device__ inline double prob(const VerifyArgs& a, float l, double mx, double inv) {
    return a.form == K3X_DIST_PROBS ? (double)l
                                    : exp2_f64(((double)l - mx) * a.rate) * inv;
}

// One workgroup a sequence: a wave a row, the drafts' rows together.  What it
// reads is a few KB a sequence: 5 to 7 us of loads that wait for one another.
template <uint32_t DT>
__global__ __launch_bounds__(1024) void verify_accept_kernel(VerifyArgs a) {
    struct Row {
        double max, inv, prob;  // prob: of the drafted token
        uint32_t arg, fit;
        uint32_t token;  // drafted after it
        float u;
    };
    __shared__ Row rows[2 * kMaxDrafts + 1];
    __shared__ uint32_t verdict;
    const uint32_t n = blockIdx.x, tid = threadIdx.x;
    const uint32_t status = *(volatile uint32_t*)a.status;  // looked at with the rows
    const uint32_t count = drafts_of(a, n);
    uint32_t* out = a.out_tokens + (size_t)n * (a.D + 1);
    if (count > a.D) {  // left out, or out of range
        if (__syncthreads_or(status)) return;
        if (count == K3X_VERIFY_SKIP) {
            for (uint32_t i = tid; i <= a.D; i += blockDim.x) out[i] = 0xffffffffu;
            if (tid == 0) a.accepted[n] = 0;
        } else if (tid == 0) {
            latch(a.status, K3X_ERR_INVALID_STATE);
        }
        if (tid == 0) a.drawn[n].done = 1;
        return;
    }
    const bool totals = a.form == K3X_DIST_LOGITS || a.greedy;
    // Target rows 0 .. count, then the draft's.
    const uint32_t all = count + 1 + (a.draft ? count : 0);
    for (uint32_t i = tid >> 6; i < all; i += blockDim.x >> 6) {
        const bool target = i <= count;
        const uint32_t d = target ? i : i - count - 1, r = target ? i : a.D + 1 + d;
        const uint32_t x = d < count ? a.tokens[(size_t)n * a.D + d] : 0;
        const float l = x < a.V && !a.greedy ? Elem<DT>::load(row_of<DT>(a, n, r)[x]) : 0.0f;
        Row row{0.0, 1.0, 0.0, 0, 1, x, 0.0f};
        if (target && d < count && !a.greedy) row.u = a.accept_u[(size_t)n * a.D + d];
        if (totals) row.fit = row_total(a, n, r, &row.max, &row.inv, &row.arg);
        if (row.fit && !a.greedy) row.prob = prob(a, l, row.max, row.inv);
        if ((tid & 63) == 0) rows[i] = row;
    }
    if (__syncthreads_or(status)) return;
    if (tid == 0) {
        uint32_t bad = 0, i = 0;
        for (;; ++i) {
            const Row& p = rows[i];
            if (!p.fit) bad = 1;
            if (bad || i == count) break;
            if (p.token >= a.V) {
                bad = 1;
                break;
            }
            if (a.greedy) {
                if (p.arg != p.token) break;
                continue;
            }
            const float u = p.u;
            const Row one{0.0, 1.0, 1.0, 0, 1, 0, 0.0f};
            const Row& q = a.draft ? rows[count + 1 + i] : one;
            if (!q.fit || !(u >= 0.0f && u < 1.0f) ||
                !(p.prob >= 0.0 && p.prob < __builtin_inf()) ||
                !(q.prob >= 0.0 && q.prob < __builtin_inf())) {
                bad = 1;
                break;
            }
            if (!((double)u * q.prob < p.prob)) break;
        }
        if (bad) latch(a.status, K3X_ERR_INVALID_STATE);
        Drawn d{};
        d.accepted = i;
        d.rows = count;
        d.done = bad || a.greedy;
        d.pmax = rows[i].max;
        d.pinv = rows[i].inv;
        if (a.draft && i < count) {
            d.qmax = rows[count + 1 + i].max;
            d.qinv = rows[count + 1 + i].inv;
        }
        a.drawn[n] = d;
        if (!bad && a.greedy) a.accepted[n] = i;
        verdict = bad ? 0xffffffffu : i;
    }
    __syncthreads();
    if (!a.greedy || verdict == 0xffffffffu) return;
    for (uint32_t i = tid; i <= a.D; i += blockDim.x)
        out[i] = i < verdict    ? rows[i].token
                 : i == verdict ? rows[verdict].arg
                                : 0xffffffffu;
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
    __device__ inline double of(const VerifyArgs& a, uint32_t i, float pl, float ql) const {
        const double r = prob(a, pl, pmax, pinv);
        const double o = q ? prob(a, ql, qmax, qinv) : 0.0;
        if (!(r >= 0.0 && o >= 0.0 && o < __builtin_inf())) return __builtin_nan("");
        return i == token || r <= o ? 0.0 : r - o;
    }
    __device__ inline double at(const VerifyArgs& a, uint32_t i) const {
        return of(a, i, Elem<DT>::load(p[i]), q ? Elem<DT>::load(q[i]) : 0.0f);
    }
    // Only the target's probabilities.
    __device__ inline void whole() {
        q = nullptr;
        token = 0xffffffffu;
    }
};

__device__ inline double block_sum(double s, double* sd) {
    s = wave_sum(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sd[threadIdx.x >> 6] = s;
    __syncthreads();
    return sd[0] + sd[1] + sd[2] + sd[3];
}

// Where a cumulative sum over [lo, ...), a run of `per` entries a thread, passes
// the border: start lies before lo, s is the thread's sum; returns what lies
// before the thread's run.  By the whole workgroup.
__device__ inline double run_start(double s, double start, double* sd) {
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    double c = s;  // of this and the wave's threads before
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(c, d);
        if (lane >= (uint32_t)d) c += o;
    }
    __syncthreads();
    if (lane == 63) sd[tid >> 6] = c;
    __syncthreads();
    c = __shfl_up(c, 1);
    c = start + (lane ? c : 0.0);
    for (uint32_t w = 0; w < tid >> 6; ++w) c += sd[w];
    return c;
}

// Sum over the lanes before and the lane itself.
__device__ inline double lanes_sum(double c) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(c, d);
        if (lane >= (uint32_t)d) c += o;
    }
    return c;
}

// The token of a part that the border falls in: the last entry over 0 that the
// cumulative sum (start before the part) has not passed the border before.  By
// a wave; the part holds an entry over 0 and start <= border.  The part's
// chunks of W neighbours a lane, then the lanes, then the neighbours: at each
// level the last one over 0 that starts at the border or before, and the first
// over 0 is one, so that something is found whatever the sums' roundings.
template <uint32_t DT, int W>
__device__ inline uint32_t draw_token(const VerifyArgs& a, uint32_t lo,
                                      const double (&r)[kEntries], double start, double border) {
    const uint32_t lane = threadIdx.x & 63;
    double mine[W] = {}, sum = 0.0, at = start;
    uint32_t chunk = 0;
#pragma unroll
    for (int c = 0; c < (int)kEntries / W; ++c) {
        double l = 0.0;
#pragma unroll
        for (int y = 0; y < W; ++y) l += r[c * W + y];
        const double all = wave_sum(l);
        if (all > 0.0 && at <= border) {
            chunk = c;
            start = at;
            sum = l;
#pragma unroll
            for (int y = 0; y < W; ++y) mine[y] = r[c * W + y];
        }
        at += all;
    }
    double c = __shfl_up(lanes_sum(sum), 1);
    c = lane ? start + c : start;
    const int from = 63 - __clzll((unsigned long long)__ballot(sum > 0.0 && c <= border));
    uint32_t hit = 0;
#pragma unroll
    for (int y = 0; y < W; ++y) {
        if (mine[y] > 0.0 && c <= border) hit = y;
        c += mine[y];
    }
    return lo + (chunk * 64 + from) * W + (uint32_t)__shfl((int)hit, from);
}

// The same over the whole row, by the workgroup.
template <uint32_t DT>
__device__ inline uint32_t draw_whole(const VerifyArgs& a, const Rest<DT>& rest, double border,
                                      double* sd, uint32_t* found) {
    const uint32_t per = (a.V + kThreads - 1) / kThreads;
    const uint32_t b = min(a.V, threadIdx.x * per), e = min(a.V, b + per);
    double s = 0.0;
    for (uint32_t i = b; i < e; ++i) s += rest.at(a, i);
    double c = run_start(s, 0.0, sd);
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

// The row that the next token is drawn from: sums of all parts, and the entry by
// the last workgroup that arrives, so that no launch waits between.  64 sequences
// of 131072 probabilities (67 MB): 20 us, 13 of them the sums (5.2 TB/s) and the
// others the last workgroup's loads that wait for one another, for which one
// wave holds the part in registers (by the workgroup, runs of sixteen neighbours
// a thread: 20 us in place of 8).
template <uint32_t DT>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a) {
    __shared__ double sd[kThreads / 64];
    __shared__ uint32_t found, last;
    const uint32_t blocks = (a.parts + kWaves - 1) / kWaves;
    const uint32_t n = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 63;
    const uint32_t part = blockIdx.x % blocks * kWaves + (tid >> 6);
    const uint32_t status = *(volatile uint32_t*)a.status;
    const Drawn d = a.drawn[n];
    if (__syncthreads_or(status)) return;
    if (d.done) return;
    Rest<DT> rest(a, d, n);
    const float past = a.form == K3X_DIST_PROBS ? 0.0f : -__builtin_inff();
    typedef Entries<DT> Mine;
    // The wave's entries of the part at lo of what is drawn from.
    auto entries = [&](uint32_t lo, double (&r)[kEntries]) {
        const uint32_t hi = min(a.V, lo + kPart);
        float pl[kEntries], ql[kEntries] = {};
        Mine::load(a, rest.p, lo, hi, lane, past, pl);
        if (rest.q) Mine::load(a, rest.q, lo, hi, lane, past, ql);
#pragma unroll
        for (int j = 0; j < (int)kEntries; ++j)
            r[j] = rest.of(a, Mine::where(a, lo, lane, j), pl[j], ql[j]);
    };
    if (part < a.parts) {
        double r[kEntries], s = 0.0;
        entries(part * kPart, r);
#pragma unroll
        for (int j = 0; j < (int)kEntries; ++j) s += r[j];
        s = wave_sum(s);
        // The sums, then the arrival, all past the caches of one die: the last
        // workgroup sees every sum.  (A releasing add would write back the
        // die's whole cache for each workgroup: it made 91 us of 31.)
        if (lane == 0) {
            __hip_atomic_store(a.sums + (size_t)n * a.parts + part, s, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
    }
    __syncthreads();
    if (tid == 0) {
        found = 0;
        last = __hip_atomic_fetch_add(&a.drawn[n].arrived, 1u, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) == blocks - 1;
    }
    __syncthreads();
    if (!last) return;
    // A run of parts a lane, in order: their sums and what lies before each.
    constexpr uint32_t kRun = (1u << 20) / kPart / 64;
    const uint32_t run = (a.parts + 63) / 64;
    const float u = a.sample_u[n];
    uint32_t* out = a.out_tokens + (size_t)n * (a.D + 1);
    double own[kRun], all = 0.0;
#pragma unroll
    for (uint32_t x = 0; x < kRun; ++x) {
        const uint32_t i = lane * run + x;
        own[x] = x < run && i < a.parts
                     ? __hip_atomic_load(a.sums + (size_t)n * a.parts + i, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT)
                     : 0.0;
    }
#pragma unroll
    for (uint32_t x = 0; x < kRun; ++x) all += own[x];
    double c = lanes_sum(all);
    double total = __shfl(c, 63);
    c = __shfl_up(c, 1);
    if (lane == 0) c = 0.0;
    uint32_t bad = 0, next = 0;
    if (!(u >= 0.0f && u < 1.0f) || !(total >= 0.0 && total < __builtin_inf())) bad = 1;
    if (!bad) {
        double border = (double)u * total;
        if (total > 0.0) {
            if (tid >= 64) return;
            // The last part over 0 that starts at the border or before.
            const uint64_t mask = __ballot(all > 0.0 && c <= border);
            const int from = 63 - __clzll((unsigned long long)mask);
            uint32_t in = 0;
            double start = 0.0;
#pragma unroll
            for (uint32_t x = 0; x < kRun; ++x) {
                if (own[x] > 0.0 && c <= border) {
                    in = x;
                    start = c;
                }
                c += own[x];
            }
            const uint32_t lo = ((uint32_t)from * run + (uint32_t)__shfl((int)in, from)) * kPart;
            start = __shfl(start, from);
            double r[kEntries];
            entries(lo, r);
            next = a.vec ? draw_token<DT, Mine::kWide>(a, lo, r, start, border)
                         : draw_token<DT, 1>(a, lo, r, start, border);
        } else {
            // Nothing is left over q (or of a row without its drafted token):
            // the target's own probabilities.
            rest.whole();
            double s = 0.0;
            for (uint32_t i = tid; i < a.V; i += kThreads) s += rest.at(a, i);
            total = block_sum(s, sd);
            border = (double)u * total;
            if (!(total > 0.0 && total < __builtin_inf())) bad = 1;
            if (!bad) next = draw_whole<DT>(a, rest, border, sd, &found);
        }
    }
    if (bad) {
        if (tid == 0) latch(a.status, K3X_ERR_INVALID_STATE);
        return;
    }
    if (tid == 0) a.accepted[n] = d.accepted;
    if (tid >= 64) return;
    for (uint32_t i = tid; i <= a.D; i += 64)
        out[i] = i < d.accepted    ? a.tokens[(size_t)n * a.D + i]
                 : i == d.accepted ? next
                                   : 0xffffffffu;
}

template <uint32_t DT>
int launch_verify(k3x_hip_ctx* ctx, const VerifyArgs& a) {
    unsigned launches = 1;
    const uint32_t rows = a.draft ? 2 * a.D + 1 : a.D + 1;
    if (a.form == K3X_DIST_LOGITS || a.greedy) {
        hipLaunchKernelGGL(verify_rows_kernel<DT>,
                           dim3(a.N * rows * ((a.parts + kWaves - 1) / kWaves)),
                           dim3(kThreads), 0, ctx->stream, a);
        ++launches;
    }
    hipLaunchKernelGGL(verify_accept_kernel<DT>, dim3(a.N), dim3(64 * std::min(rows, 16u)), 0,
                       ctx->stream, a);
    if (!a.greedy) {
        hipLaunchKernelGGL(verify_draw_kernel<DT>, dim3(a.N * ((a.parts + kWaves - 1) / kWaves)),
                           dim3(kThreads), 0, ctx->stream, a);
        ++launches;
    }
    return launched(ctx, launches);
}

uint32_t parts_of(const k3x_hip_verify_params* p) { return (p->vocab + kPart - 1) / kPart; }
bool verify_ok(const k3x_hip_verify_params* p) {
    return p->sequences && p->sequences <= 65535 && p->drafts <= kMaxDrafts && p->vocab &&
           p->vocab <= (1u << 20) && p->dtype <= K3X_DTYPE_BF16 && p->form <= K3X_DIST_PROBS &&
           p->greedy <= 1 && std::isfinite(p->temperature) && p->temperature > 0.0f &&
           (!p->row_stride || p->row_stride >= p->vocab) &&
           // threads of a launch
           (uint64_t)p->sequences * (2 * p->drafts + 1) * ((parts_of(p) + kWaves - 1) / kWaves) *
                   kThreads < (1ull << 32);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

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
    a.vec = a.stride * es % 16 == 0 && aligned(target, 16) && aligned(draft, 16);
    a.form = p->form;
    a.greedy = p->greedy;
    a.rate = 1.4426950408889634 / p->temperature;
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
