// logits.hip -- penalties, biases and masks on the rows of a draft window.
//
// A workgroup takes a part of the vocabulary for all rows of a sequence: it
// counts the history's tokens of that part in LDS once, keeps each one's bias
// beside them, and walks the rows, the drafted token after each added to the
// counts.  So nothing of a vocabulary's size is kept between calls or cleared.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "k3x_ops.hpp"

using namespace k3x_dev;
using namespace k3x_ops;

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kPart = 2048;  // tokens of the vocabulary a workgroup
constexpr uint32_t kInPrompt = 1u << 31;

// 16 bytes of elements at any element's address: rows of an odd vocabulary are not
// aligned, and memory takes such accesses as they are.
template <uint32_t DT>
struct Wide {
    typedef typename Elem<DT>::type E;
    static constexpr int W = 16 / sizeof(E);
    typedef E Vec __attribute__((ext_vector_type(W), aligned(sizeof(E))));
};
typedef uint32_t Tokens4 __attribute__((ext_vector_type(4), aligned(4)));

struct LogitsArgs {
    const void* logits;
    void* out;
    const uint32_t *history, *history_lens, *prompt_lens, *drafts, *draft_counts;
    const float *repetition, *frequency, *presence;
    const uint32_t *bias_offsets, *bias_tokens;
    const float* bias_values;
    const uint32_t *masks, *mask_index;
    uint32_t N, D, V, stride, out_stride, width, biases, mask_rows, mask_stride;
    const uint32_t* status;  // set: nothing is done
    uint32_t* errors;        // the call's own: status, or apart from it (report_kernel)
};

// KE tokens a thread, by 16 bytes.  A row's loads are on their way while the one
// before it is adjusted; counts and biases of the thread's tokens stay in registers.
// Bound: memory, and in small calls the part's history.  64 sequences of 4 drafts and
// 100003 fp32 logits with histories of 8000 (259 MB): 70 us, 3.7 TB/s, from memory, 54
// where half of it lies in the last cache; one sequence of 163840 bf16 logits 10.6 us.
// Parts of 4096 read each history half as often, but fill the chip worse: 18.6 for 12.0 us
// with one sequence (fp32), 26.8 for 22.2 with 16, 55.5 for 51.0 with 64.
template <uint32_t DT>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(LogitsArgs a) {
    typedef typename Wide<DT>::E E;
    typedef typename Wide<DT>::Vec Vec;
    constexpr int W = Wide<DT>::W, KE = kPart / kThreads, NV = KE / W;
    __shared__ uint32_t count[kPart], entry[kPart], stop;
    const uint32_t n = blockIdx.y, lo = blockIdx.x * kPart;
    const uint32_t tid = threadIdx.x, hi = min(a.V, lo + kPart);
    if (tid == 0) stop = *(volatile const uint32_t*)a.status;
    const uint32_t drafts = a.draft_counts ? a.draft_counts[n] : a.D;
    const uint32_t length = a.history ? a.history_lens[n] : 0;
    const uint32_t prompt = a.history && a.prompt_lens ? a.prompt_lens[n] : 0;
    const uint32_t b0 = a.bias_offsets ? a.bias_offsets[n] : 0;
    const uint32_t b1 = a.bias_offsets ? a.bias_offsets[n + 1] : 0;
    const float rep = a.repetition ? a.repetition[n] : 1.0f;
    const float freq = a.frequency ? a.frequency[n] : 0.0f;
    const float pres = a.presence ? a.presence[n] : 0.0f;
    // All waves or none: another workgroup may latch between their looks.
    __syncthreads();
    if (stop || drafts == K3X_VERIFY_SKIP) return;
    if (drafts > a.D || length > a.width || prompt > length || b1 < b0 || b1 > a.biases ||
        !(rep > 0.0f && rep < __builtin_inff()) || !(fabsf(freq) < __builtin_inff()) ||
        !(fabsf(pres) < __builtin_inff())) {
        if (tid == 0) latch(a.errors, K3X_ERR_INVALID_STATE);
        return;
    }
    bool bad = false;
    // The thread's tokens: W from lo + (v kThreads + tid) W on, for each v.
    auto first = [&](int v) { return lo + (v * kThreads + tid) * W; };
    struct Row {
        Vec x[NV];
        uint32_t allowed[NV];  // bits of the W tokens
    };
    auto load = [&](uint32_t r, Row& row) {
        const size_t at = (size_t)n * (a.D + 1) + r;
        const E* x = static_cast<const E*>(a.logits) + at * a.stride;
        const uint32_t mask = a.masks ? a.mask_index[at] : K3X_NO_MASK;
        const bool has = mask < a.mask_rows;
        bad |= mask != K3X_NO_MASK && !has;
        const uint32_t* words = a.masks + (size_t)(has ? mask : 0) * a.mask_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const uint32_t t = first(v);
            if (t + W <= hi) {
                row.x[v] = *reinterpret_cast<const Vec*>(x + t);
            } else {
#pragma unroll
                for (int y = 0; y < W; ++y)
                    if (t + y < hi) row.x[v][y] = x[t + y];
            }
            row.allowed[v] = has && t < hi ? words[t / 32] >> (t % 32) : 0xffffffffu;
        }
    };
    Row next;
    load(0, next);

#pragma unroll
    for (int i = 0; i < KE; ++i) count[i * kThreads + tid] = entry[i * kThreads + tid] = 0;
    __syncthreads();
    {
        const uint32_t* h = a.history + (size_t)n * a.width;
        auto take = [&](uint32_t t, uint32_t i) {
            bad |= t >= a.V;
            if (t >= lo && t < hi) {
                if (i < prompt) atomicOr(&count[t - lo], kInPrompt);
                else atomicAdd(&count[t - lo], 1u);
            }
        };
        const uint32_t whole = length / 4;
        constexpr int kAhead = 4;
        for (uint32_t i = tid; i < whole; i += kThreads * kAhead) {
            Tokens4 t[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                t[j] = *reinterpret_cast<const Tokens4*>(h + 4 * min(i + j * kThreads, whole - 1));
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (i + j * kThreads < whole)
#pragma unroll
                    for (int y = 0; y < 4; ++y) take(t[j][y], 4 * (i + j * kThreads) + y);
        }
        if (tid < length % 4) take(h[4 * whole + tid], 4 * whole + tid);
    }
    for (uint32_t i = b0 + tid; i < b1; i += kThreads) {
        const uint32_t t = a.bias_tokens[i];
        bad |= t >= a.V;
        if (t >= lo && t < hi) atomicMax(&entry[t - lo], i - b0 + 1);
    }
    __syncthreads();
    uint32_t c[KE], biased = 0;
    float bias[KE];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int y = 0; y < W; ++y) {
            const int i = v * W + y;
            c[i] = count[first(v) - lo + y];
            const uint32_t e = entry[first(v) - lo + y];
            bias[i] = 0.0f;
            if (e) {
                bias[i] = a.bias_values[b0 + e - 1];
                biased |= 1u << i;
            }
        }

    for (uint32_t r = 0; r <= drafts; ++r) {
        const Row row = next;
        if (r < drafts) load(r + 1, next);
        E* out = static_cast<E*>(a.out) + ((size_t)n * (a.D + 1) + r) * a.out_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            Vec z;
#pragma unroll
            for (int y = 0; y < W; ++y) {
                const int i = v * W + y;
                float l = Elem<DT>::load(row.x[v][y]);
                if (c[i]) {
                    if (a.repetition) l = l > 0.0f ? l / rep : l * rep;
                    const uint32_t times = c[i] & ~kInPrompt;
                    if (times) {
                        if (a.frequency) l = l - freq * (float)times;
                        if (a.presence) l = l - pres;
                    }
                }
                if (biased >> i & 1) l = l + bias[i];
                if (!(row.allowed[v] >> y & 1)) l = -__builtin_inff();
                z[y] = Elem<DT>::store(l);
            }
            const uint32_t t = first(v);
            if (t + W <= hi) {
                *reinterpret_cast<Vec*>(out + t) = z;
            } else {
#pragma unroll
                for (int y = 0; y < W; ++y)
                    if (t + y < hi) out[t + y] = z[y];
            }
        }
        if (r < drafts) {
            const uint32_t t = a.drafts[(size_t)n * a.D + r];
            bad |= t >= a.V;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int y = 0; y < W; ++y) c[v * W + y] += t == first(v) + y;
        }
    }
    if (bad) latch(a.errors, K3X_ERR_INVALID_STATE);
}

template <uint32_t DT>
int launch_logits(k3x_hip_ctx* ctx, const LogitsArgs& a) {
    hipLaunchKernelGGL((adjust_logits_kernel<DT>), dim3((a.V + kPart - 1) / kPart, a.N), dim3(kThreads),
                       0, ctx->stream, a);
    if (a.errors == a.status) return launched(ctx, 1);
    hipLaunchKernelGGL(report_kernel, dim3(1), dim3(1), 0, ctx->stream, a.errors, ctx->status);
    return launched(ctx, 2);
}

bool logits_ok(const k3x_hip_logits_params* p) {
    const uint32_t words = (p->vocab + 31) / 32;
    return p->sequences && p->sequences <= 65535 && p->drafts <= 64 && p->vocab &&
           p->vocab <= (1u << 20) && p->dtype <= K3X_DTYPE_BF16 &&
           (!p->row_stride || p->row_stride >= p->vocab) &&
           (!p->out_stride || p->out_stride >= p->vocab) &&
           (!p->mask_stride || p->mask_stride >= words);
}

}  // namespace

extern "C" {

int k3x_hip_adjust_logits(k3x_hip_ctx* ctx, const k3x_hip_logits_params* p, const void* logits,
                          const uint32_t* history, const uint32_t* history_lens,
                          const uint32_t* prompt_lens, const uint32_t* drafts,
                          const uint32_t* draft_counts, const float* repetition,
                          const float* frequency, const float* presence,
                          const uint32_t* bias_offsets, const uint32_t* bias_tokens,
                          const float* bias_values, const uint32_t* masks,
                          const uint32_t* mask_index, void* out) {
    if (!ctx || !p || !logits_ok(p) || !logits || !out) return K3X_ERR_INVALID_EXTENT;
    if ((p->drafts && !drafts) || (history && !history_lens) ||
        (bias_offsets && p->biases && (!bias_tokens || !bias_values)) || (masks && !mask_index))
        return K3X_ERR_INVALID_EXTENT;
    const uintptr_t es = p->dtype == K3X_DTYPE_F32 ? 4 : 2;
    if (!aligned(logits, es) || !aligned(out, es)) return K3X_ERR_INVALID_EXTENT;
    for (const void* x : {(const void*)history, (const void*)history_lens,
                          (const void*)prompt_lens, (const void*)drafts,
                          (const void*)draft_counts, (const void*)repetition,
                          (const void*)frequency, (const void*)presence,
                          (const void*)bias_offsets, (const void*)bias_tokens,
                          (const void*)bias_values, (const void*)masks, (const void*)mask_index})
        if (!aligned(x, 4)) return K3X_ERR_INVALID_EXTENT;
    if (hipSetDevice(ctx->device) != hipSuccess) return K3X_ERR_BACKEND_UNAVAILABLE;
    LogitsArgs a{};
    a.logits = logits;
    a.out = out;
    a.history = history;
    a.history_lens = history_lens;
    a.prompt_lens = prompt_lens;
    a.drafts = drafts;
    a.draft_counts = draft_counts;
    a.repetition = repetition;
    a.frequency = frequency;
    a.presence = presence;
    a.bias_offsets = bias_offsets;
    a.bias_tokens = bias_tokens;
    a.bias_values = bias_values;
    a.masks = masks;
    a.mask_index = mask_index;
    a.N = p->sequences;
    a.D = p->drafts;
    a.V = p->vocab;
    a.stride = p->row_stride ? p->row_stride : p->vocab;
    a.out_stride = p->out_stride ? p->out_stride : p->vocab;
    a.width = p->history_width;
    a.biases = p->biases;
    a.mask_rows = p->masks;
    a.mask_stride = p->mask_stride ? p->mask_stride : (p->vocab + 31) / 32;
    a.status = ctx->status;
    // 64 sequences in place, inputs warm: 50.4 us a call, without report_kernel 48.6.
    a.errors = out == logits && a.N > 1 ? ctx->status + 1 : ctx->status;
    return p->dtype == K3X_DTYPE_F32 ? launch_logits<K3X_DTYPE_F32>(ctx, a)
                                     : launch_logits<K3X_DTYPE_BF16>(ctx, a);
}

}  // extern "C"
