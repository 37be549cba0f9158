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
constexpr uint32_t kPart = 4096;  // tokens a workgroup
constexpr uint32_t kInPrompt = 1u << 31;

struct LogitsArgs {
    const void* logits;
    void* out;
    const uint32_t *history, *history_lens, *prompt_lens, *drafts, *draft_counts;
    const float *repetition, *frequency, *presence;
    const uint32_t *bias_offsets, *bias_tokens;
    const float* bias_values;
    const uint32_t *masks, *mask_index;
    uint32_t N, D, V, stride, out_stride, width, biases, mask_rows, mask_stride, parts;
    uint32_t* status;
};

template <uint32_t DT>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(LogitsArgs a) {
    typedef typename Elem<DT>::type E;
    __shared__ uint32_t count[kPart], entry[kPart];
    const uint32_t n = blockIdx.x / a.parts, lo = blockIdx.x % a.parts * kPart;
    const uint32_t tid = threadIdx.x, hi = min(a.V, lo + kPart);
    if (*(volatile uint32_t*)a.status) return;
    const uint32_t drafts = a.draft_counts ? a.draft_counts[n] : a.D;
    if (drafts == K3X_VERIFY_SKIP) return;
    const uint32_t length = a.history ? a.history_lens[n] : 0;
    const uint32_t prompt = a.history && a.prompt_lens ? a.prompt_lens[n] : 0;
    const uint32_t b0 = a.bias_offsets ? a.bias_offsets[n] : 0;
    const uint32_t b1 = a.bias_offsets ? a.bias_offsets[n + 1] : 0;
    const float rep = a.repetition ? a.repetition[n] : 1.0f;
    const float freq = a.frequency ? a.frequency[n] : 0.0f;
    const float pres = a.presence ? a.presence[n] : 0.0f;
    if (drafts > a.D || length > a.width || prompt > length || b1 < b0 || b1 > a.biases ||
        !(rep > 0.0f && rep < __builtin_inff()) || !(fabsf(freq) < __builtin_inff()) ||
        !(fabsf(pres) < __builtin_inff())) {
        if (tid == 0) latch(a.status, K3X_ERR_INVALID_STATE);
        return;
    }
    bool bad = false;
    for (uint32_t i = tid; i < kPart; i += kThreads) count[i] = entry[i] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < length; i += kThreads) {
        const uint32_t t = a.history[(size_t)n * a.width + i];
        bad |= t >= a.V;
        if (t >= lo && t < hi) {
            if (i < prompt) atomicOr(&count[t - lo], kInPrompt);
            else atomicAdd(&count[t - lo], 1u);
        }
    }
    for (uint32_t i = b0 + tid; i < b1; i += kThreads) {
        const uint32_t t = a.bias_tokens[i];
        bad |= t >= a.V;
        if (t >= lo && t < hi) atomicMax(&entry[t - lo], i - b0 + 1);
    }
    for (uint32_t r = 0; r <= drafts; ++r) {
        __syncthreads();
        const uint32_t mask = a.masks ? a.mask_index[(size_t)n * (a.D + 1) + r] : K3X_NO_MASK;
        const uint32_t* words = nullptr;
        if (mask != K3X_NO_MASK) {
            bad |= mask >= a.mask_rows;
            if (mask < a.mask_rows) words = a.masks + (size_t)mask * a.mask_stride;
        }
        const size_t row = (size_t)n * (a.D + 1) + r;
        const E* x = static_cast<const E*>(a.logits) + row * a.stride;
        E* y = static_cast<E*>(a.out) + row * a.out_stride;
        for (uint32_t t = lo + tid; t < hi; t += kThreads) {
            float l = Elem<DT>::load(x[t]);
            const uint32_t c = count[t - lo], times = c & ~kInPrompt, e = entry[t - lo];
            if (a.repetition && c) l = l > 0.0f ? l / rep : l * rep;
            if (times) {
                if (a.frequency) l = l - freq * (float)times;
                if (a.presence) l = l - pres;
            }
            if (e) l = l + a.bias_values[b0 + e - 1];
            if (words && !(words[t / 32] >> (t % 32) & 1)) l = -__builtin_inff();
            y[t] = Elem<DT>::store(l);
        }
        __syncthreads();
        if (r < drafts && tid == 0) {
            const uint32_t t = a.drafts[(size_t)n * a.D + r];
            bad |= t >= a.V;
            if (t >= lo && t < hi) ++count[t - lo];
        }
    }
    if (bad) latch(a.status, K3X_ERR_INVALID_STATE);
}

bool logits_ok(const k3x_hip_logits_params* p) {
    const uint32_t words = (p->vocab + 31) / 32, parts = (p->vocab + kPart - 1) / kPart;
    return p->sequences && p->sequences <= 65535 && p->drafts <= 64 && p->vocab &&
           p->vocab <= (1u << 20) && p->dtype <= K3X_DTYPE_BF16 &&
           (!p->row_stride || p->row_stride >= p->vocab) &&
           (!p->out_stride || p->out_stride >= p->vocab) &&
           (!p->mask_stride || p->mask_stride >= words) &&
           (uint64_t)p->sequences * parts * kThreads < (1ull << 32);  // threads of a launch
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
    a.parts = (p->vocab + kPart - 1) / kPart;
    a.status = ctx->status;
    const dim3 grid(a.N * a.parts), block(kThreads);
    if (p->dtype == K3X_DTYPE_F32)
        hipLaunchKernelGGL(adjust_logits_kernel<K3X_DTYPE_F32>, grid, block, 0, ctx->stream, a);
    else
        hipLaunchKernelGGL(adjust_logits_kernel<K3X_DTYPE_BF16>, grid, block, 0, ctx->stream, a);
    return launched(ctx, 1);
}

}  // extern "C"
