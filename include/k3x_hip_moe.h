/*
 * k3x_hip_moe.h -- C ABI of the MI355X (gfx950) routed-expert MoE layer.
 *
 * Plain C: opaque handles, plain pointers and sizes, int status codes.  No
 * exception crosses this boundary and no torch type appears in it.  Every
 * entry point validates its arguments before it touches device state
 * (fail-closed), and returns one of the k3x_status values, which are the
 * numeric values of k3x::ErrorCode (runtime/include/k3x/status.hpp:9-31).
 *
 * Pointer conventions: parameters documented "host" are CPU memory, "device"
 * are HIP device memory of the context's device.  All device work is
 * enqueued on the context's stream; entry points return after enqueueing
 * unless documented otherwise.  Errors detected by kernels (non-finite input,
 * invalid router scores) are latched in a per-context status word that
 * k3x_hip_ctx_synchronize() returns and clears; a latched error makes every
 * later kernel of the context skip its work until it is read.
 *
 * Each declaration names the reference interface it replaces (file:line in
 * the rsb1813/project-k3x tree).
 */
#ifndef K3X_HIP_MOE_H
#define K3X_HIP_MOE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define K3X_HIP_ABI_VERSION 1

/* k3x::ErrorCode values (runtime/include/k3x/status.hpp:9-31). */
enum k3x_status {
    K3X_OK = 0,
    K3X_ERR_IO = 1,
    K3X_ERR_BAD_MAGIC = 2,
    K3X_ERR_UNSUPPORTED_VERSION = 3,
    K3X_ERR_UNSUPPORTED_REQUIRED_FEATURE = 4,
    K3X_ERR_SUPERBLOCK_CRC_MISMATCH = 6,
    K3X_ERR_TRUNCATED_FILE = 7,
    K3X_ERR_INVALID_DIRECTORY = 8,
    K3X_ERR_INVALID_EXTENT = 9,
    K3X_ERR_DATA_CRC_MISMATCH = 10,
    K3X_ERR_AUXILIARY_CRC_MISMATCH = 11,
    K3X_ERR_DIRECTORY_SHA256_MISMATCH = 12,
    K3X_ERR_ROOT_SHA256_MISMATCH = 13,
    K3X_ERR_TENSOR_NOT_FOUND = 14,
    K3X_ERR_INVALID_MXFP4 = 15,
    K3X_ERR_INVALID_STATE = 16,
    K3X_ERR_BACKEND_UNAVAILABLE = 17,
};

/* GLU activation policy.  SiTU: runtime/src/ops.cpp:20-30.
 * SwiGLU: silu(g) * u with silu from runtime/src/model.cpp:60-61. */
enum k3x_glu { K3X_GLU_SWIGLU = 0, K3X_GLU_SITU = 1 };

/* Renormalisation of the selected router scores.
 * FLOAT:  runtime/src/routing_policy.cpp:146-157 (synthetic/resident path).
 * DOUBLE: runtime/src/official_moe.cpp:235-242 (official path). */
enum k3x_renorm { K3X_RENORM_FLOAT = 0, K3X_RENORM_DOUBLE = 1 };
/* k3x_hip_route only: the selected scores as they are. */
#define K3X_RENORM_NONE 2u

/* Matrices of one expert, as addressed by the debug/read-back entry points. */
enum k3x_matrix { K3X_MATRIX_GATE = 0, K3X_MATRIX_UP = 1, K3X_MATRIX_DOWN = 2 };

/* Streams of the portable synthetic generator (k3x_hip_bank_fill_synthetic):
 * stream id = (kind << 32) | expert index. */
enum k3x_synth_stream {
    K3X_STREAM_GATE_CODES = 1,
    K3X_STREAM_GATE_SCALES = 2,
    K3X_STREAM_UP_CODES = 3,
    K3X_STREAM_UP_SCALES = 4,
    K3X_STREAM_DOWN_CODES = 5,
    K3X_STREAM_DOWN_SCALES = 6,
    K3X_STREAM_ROUTER = 7,
    K3X_STREAM_BIAS = 8,
    K3X_STREAM_SHARED_GATE = 9,
    K3X_STREAM_SHARED_UP = 10,
    K3X_STREAM_SHARED_DOWN = 11,
    K3X_STREAM_INPUT = 12,
};

typedef struct k3x_hip_ctx k3x_hip_ctx;
typedef struct k3x_hip_bank k3x_hip_bank;

/* Shape of one MoE layer.  hidden and inter must be multiples of 128,
 * group_size must be 32 (the CUDA backend's contract,
 * runtime/cuda/backend_cuda.cu:1865-1867), shared_inter is 0 (no shared
 * expert) or a multiple of 128. */
typedef struct k3x_hip_layer_desc {
    uint32_t hidden;
    uint32_t inter;
    uint32_t experts;
    uint32_t group_size;
    uint32_t shared_inter;
} k3x_hip_layer_desc;

/* Per-call parameters of the layer.  Mirrors the scalar arguments of
 * ComputeBackend::resident_mxfp4_moe_layer (runtime/include/k3x/
 * backend.hpp:369-375) plus the router controls that runtime/src/
 * model.cpp:917-1010 applies on the host. */
typedef struct k3x_hip_moe_params {
    uint32_t tokens;          /* T, rows of x */
    uint32_t top_k;           /* natural Top-K, 1..64 and <= experts */
    float routed_scale;       /* multiplies renormalised weights */
    float rms_epsilon;        /* > 0 */
    uint32_t glu;             /* enum k3x_glu */
    float situ_beta;          /* > 0, SiTU only */
    uint32_t has_situ_linear; /* SiTU only */
    float situ_linear_beta;   /* > 0 when has_situ_linear */
    uint32_t renorm;          /* enum k3x_renorm */
    uint32_t flags;           /* K3X_FLAG_* */
} k3x_hip_moe_params;

/* k3x_hip_moe_params.flags */
enum k3x_flags {
    /* Use the general multi-launch path even where the decode path
     * (tokens <= 4) applies; both compute the same layer. */
    K3X_FLAG_GENERAL_PATH = 1u,
    /* Round each expert output to bf16 before the slot-ordered mix, as the
     * official layer does (runtime/src/official_moe.cpp:99-101, :318-326);
     * runs the general path. */
    K3X_FLAG_ROUND_EXPERT_OUT = 2u,
    /* Keep the routed GLU activation at fp32 precision into the down
     * projection (stored as a bf16 hi + lo pair per element, the down
     * projection run over both halves), as the official layer does
     * (runtime/src/official_moe.cpp:82-101); runs the general path. */
    K3X_FLAG_SPLIT_ACT = 4u,
    /* k3x_hip_moe_forward_routed only: the input rows are fp32 values held
     * as bf16 hi + lo halves, [T][2 H] (hi = bf16(v), lo = bf16(v - hi)),
     * and the gate/up projections run over both halves; the latent layer's
     * fp32 experts (runtime/src/backend_cpu.cpp:317-318).  Runs the
     * general path's streaming GEMM. */
    K3X_FLAG_SPLIT_INPUT = 8u,
    /* Multiply the routed experts of the wide GEMM (prefill chunks, many
     * rows per expert) on the scaled FP4 MFMA: the bf16 activation rows are
     * re-encoded as two FP8 E4M3 terms with one power-of-two scale per 32
     * values each (exact for bf16 values down to 2^-13 of their block's
     * largest, within 2^-21 of it below), the MXFP4 weights go in as they
     * are stored.  Ignored with K3X_FLAG_SPLIT_ACT and below 128 tokens
     * (the decode kernels and the streaming GEMM). */
    K3X_FLAG_SCALED_FP4 = 16u,
};

/* Optional device buffers that receive intermediates of k3x_hip_moe_forward;
 * any member may be NULL.  Shapes use T = tokens, K = top_k, E = experts,
 * H = hidden, I = inter, S = shared_inter. */
typedef struct k3x_hip_moe_taps {
    uint16_t* normed_x;          /* [T][H] bf16 bits, RMSNorm output */
    float* logits;               /* [T][E] */
    uint32_t* ids;               /* [T][K] router order */
    float* weights;              /* [T][K] contributions */
    uint32_t* counts;            /* [E] pairs per expert */
    uint32_t* offsets;           /* [E+1] expert-major CSR offsets */
    uint32_t* pair_token;        /* [T*K] CSR rows -> token */
    uint32_t* pair_slot;         /* [T*K] CSR rows -> router slot */
    uint32_t* first_use;         /* [E] min(token*K+slot), 0xffffffff unused */
    uint32_t* n_active;          /* [1] experts with at least one pair */
    uint32_t* active_first_use;  /* [E] active experts in first-use order */
    uint16_t* act;               /* [T*K][I] bf16 bits, CSR row order */
    float* expert_out;           /* [T][K][H] per-pair down projections */
    float* shared_out;           /* [T][H] shared expert output */
    float* out_f32;              /* [T][H] output before the bf16 cast */
    uint16_t* shared_act;        /* [T][S] bf16 bits, shared-expert GLU output */
} k3x_hip_moe_taps;

/* Descriptor of the seeded synthetic bank (no reference counterpart: the
 * reference's benches read converted checkpoints).  Codes are uniform over
 * the 16 E2M1 codes, scale bytes uniform over [scale_lo, scale_hi], normal
 * tensors are Irwin-Hall(12) approximations of N(0, sigma^2). */
typedef struct k3x_hip_synth_desc {
    uint64_t seed;
    uint32_t scale_lo;
    uint32_t scale_hi;
    float router_sigma;
    float bias_sigma;
    float shared_sigma;
    float gamma_value;
} k3x_hip_synth_desc;

/* Stages of k3x_hip_moe_forward timed by k3x_hip_ctx_set_profiling. */
enum k3x_stage {
    K3X_STAGE_ROUTE = 0,        /* RMSNorm, router logits, Top-K */
    K3X_STAGE_GROUP = 1,        /* expert-major grouping */
    K3X_STAGE_GATE_UP = 2,      /* routed MXFP4 gate/up + GLU */
    K3X_STAGE_SHARED_GATE_UP = 3,
    K3X_STAGE_DOWN = 4,         /* routed MXFP4 down projection */
    K3X_STAGE_SHARED_DOWN = 5,
    K3X_STAGE_COMBINE = 6,      /* slot-ordered mix + shared add + bf16 cast */
    /* Decode path (T <= 4); its combine is part of K3X_STAGE_DECODE_DOWN. */
    K3X_STAGE_DECODE_FRONT = 7,   /* RMSNorm, router logits, shared gate/up */
    K3X_STAGE_DECODE_SELECT = 8,  /* Top-K, grouping, shared down */
    K3X_STAGE_DECODE_GATE_UP = 9, /* routed gate/up + GLU */
    K3X_STAGE_DECODE_DOWN = 10,   /* routed down, then the slot-ordered mix */
    K3X_STAGE_COUNT = 11,
};

/* Counters, after BackendRuntimeStats (runtime/include/k3x/backend.hpp:50-129). */
typedef struct k3x_hip_stats {
    uint64_t forward_calls;
    uint64_t kernel_launches;
    uint64_t scratch_bytes;
    uint64_t resident_weight_bytes;
    uint64_t weight_h2d_bytes;
    uint64_t experts_resident;
} k3x_hip_stats;

/* ---- context ------------------------------------------------------------ */

/* Replaces make_cuda_backend (runtime/include/k3x/backend.hpp:465-466;
 * runtime/cuda/backend_cuda.cu:5264-5367): one device, one stream. */
int k3x_hip_ctx_create(int device, k3x_hip_ctx** out);
/* Fails with K3X_ERR_INVALID_STATE while banks created on the context are
 * alive: destroy them first. */
int k3x_hip_ctx_destroy(k3x_hip_ctx* ctx);
/* Enqueue on a caller-owned hipStream_t (NULL = the device's null stream). */
int k3x_hip_ctx_set_stream(k3x_hip_ctx* ctx, void* hip_stream);
/* Back to the context's own non-blocking stream (the default). */
int k3x_hip_ctx_use_own_stream(k3x_hip_ctx* ctx);
void* k3x_hip_ctx_stream(k3x_hip_ctx* ctx);
/* Waits for the stream, returns and clears the latched kernel status.
 * Replaces the cudaStreamSynchronize at the end of each backend call
 * (e.g. runtime/cuda/backend_cuda.cu:2421). */
int k3x_hip_ctx_synchronize(k3x_hip_ctx* ctx);
/* Replaces ComputeBackend::runtime_stats (backend.hpp:331). */
int k3x_hip_ctx_stats(k3x_hip_ctx* ctx, k3x_hip_stats* out);
const char* k3x_hip_status_name(int status); /* error_code_name, status.hpp:33-56 */
/* Per-stage device timing: when enabled, every stage that a forward call
 * enqueues is bracketed by a hipEvent pair on the context stream (the
 * reference brackets each launch with cudaEvent pairs and records
 * ProfileEvent::device_nanoseconds, runtime/cuda/backend_cuda.cu:2251-2298,
 * runtime/include/k3x/profile.hpp:32-42). */
int k3x_hip_ctx_set_profiling(k3x_hip_ctx* ctx, int enabled);
/* Waits for the stream, then adds the elapsed milliseconds and the number of
 * timed launches of each stage since the last reset into ms[K3X_STAGE_COUNT]
 * and launches[K3X_STAGE_COUNT] (host arrays, overwritten); reset != 0
 * clears the totals afterwards. */
int k3x_hip_ctx_stage_times(k3x_hip_ctx* ctx, double* ms, uint64_t* launches,
                            int reset);

/* ---- resident expert bank ------------------------------------------------ */

/* Replaces ResidentWeightTable (runtime/cuda/resident_weights.cuh:19-25,
 * resident_weights.cu:107-166): the whole layer's bank is allocated once in
 * HBM in the gfx950 tile layout and admitted expert by expert. */
int k3x_hip_bank_create(k3x_hip_ctx* ctx, const k3x_hip_layer_desc* desc,
                        k3x_hip_bank** out);
int k3x_hip_bank_destroy(k3x_hip_bank* bank);
/* Admits one expert from host memory in the K3X reference layout (packed
 * [rows][cols/2], low nibble = even column; scales [rows][cols/32] E8M0),
 * gate/up [inter x hidden], down [hidden x inter].  tensor_ids are the
 * residency identities (non-zero, unique within the bank), as in
 * Mxfp4WeightView::tensor_id (backend.hpp:150-157).  Scale byte 0xFF is
 * rejected with K3X_ERR_INVALID_MXFP4 (runtime/src/ops.cpp:46-49).
 * Synchronous. */
int k3x_hip_bank_upload_expert(k3x_hip_bank* bank, uint32_t expert,
                               const uint64_t tensor_ids[3],
                               const uint8_t* gate_packed,
                               const uint8_t* gate_scales,
                               const uint8_t* up_packed,
                               const uint8_t* up_scales,
                               const uint8_t* down_packed,
                               const uint8_t* down_scales);
/* Finds the expert/matrix admitted under tensor_id (host). */
int k3x_hip_bank_find(k3x_hip_bank* bank, uint64_t tensor_id,
                      uint32_t* expert, uint32_t* matrix);
/* Shared expert, host bf16 bits: gate/up [shared_inter x hidden],
 * down [hidden x shared_inter] (Bf16MlpView, backend.hpp:165-169). */
int k3x_hip_bank_upload_shared(k3x_hip_bank* bank, const uint16_t* gate,
                               const uint16_t* up, const uint16_t* down);
/* Router weight fp32 [experts x hidden], correction bias fp32 [experts],
 * RMSNorm weight fp32 [hidden]; host memory (router_weight /
 * correction_bias of runtime/src/model.cpp:918-922). */
int k3x_hip_bank_upload_router(k3x_hip_bank* bank, const float* weight,
                               const float* bias, const float* gamma);
/* Same, from device memory (no host round trip). */
int k3x_hip_bank_set_router_device(k3x_hip_bank* bank, const float* weight,
                                   const float* bias, const float* gamma);
/* Fills every expert, the router, the bias, gamma and the shared expert
 * from the seeded generator on the device (identical to the oracle's
 * generator, so the CPU checker can regenerate any expert). */
int k3x_hip_bank_fill_synthetic(k3x_hip_bank* bank,
                                const k3x_hip_synth_desc* desc);
/* Fills a device bf16 tensor of n elements with the seeded normal generator
 * (stream K3X_STREAM_INPUT). */
int k3x_hip_synth_normal_bf16(k3x_hip_ctx* ctx, uint64_t seed,
                              uint64_t stream, float sigma, size_t n,
                              uint16_t* out);
/* Debug read-back: rows [row0, row0+nrows) of one matrix, dequantised to
 * fp32 by the same conversion the GEMM kernels use, into device memory
 * out [nrows][cols].  Replaces decode_mxfp4 (runtime/src/ops.cpp:32-55)
 * for the bit-exact weight check. */
int k3x_hip_bank_dequant_rows(k3x_hip_bank* bank, uint32_t expert,
                              uint32_t matrix, uint32_t row0, uint32_t nrows,
                              float* out);
uint64_t k3x_hip_bank_bytes(const k3x_hip_bank* bank);

/* ---- the layer ----------------------------------------------------------- */

/* One routed-expert MoE layer over T tokens with device routing:
 *   xn  = bf16(RMSNorm(x) * gamma)                        (ops.cpp:10-18)
 *   ids, w = natural Top-K of sigmoid(W_r xn) + bias,
 *            renormalised, * routed_scale    (model.cpp:917-1009,
 *            routing_policy.cpp:31-160 / official_moe.cpp:211-245)
 *   expert-major grouping                          (expert_major.cpp:10-54)
 *   y[t][k] = down(bf16(GLU(gate xn, up xn)))   (backend_cpu.cpp:124-154)
 *   out = bf16(sum_k w[t][k] y[t][k] + shared(xn))  (backend_cpu.cpp:295-301,
 *                                                    model.cpp:1145)
 * x: device bf16 [T][hidden]; out: device bf16 [T][hidden]; taps optional.
 * Replaces ComputeBackend::resident_mxfp4_moe_layer (backend.hpp:369-375,
 * runtime/cuda/backend_cuda.cu:1789-2545) for a latent-free layer with
 * routing on the device.  Asynchronous. */
int k3x_hip_moe_forward(k3x_hip_ctx* ctx, k3x_hip_bank* bank,
                        const k3x_hip_moe_params* params, const uint16_t* x,
                        uint16_t* out, const k3x_hip_moe_taps* taps);

/* Bytes of the fixed device scratch behind k3x_hip_moe_forward_noalloc. */
#define K3X_HIP_NOALLOC_SCRATCH_BYTES (32u << 20)

/* k3x_hip_moe_forward that allocates nothing: no reference counterpart.  It
 * is for callers that cannot allocate device memory -- code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc.  The
 * per-call buffers (normalised input, logits, routes, grouping, activations,
 * per-pair outputs, shared expert) come from a fixed device array of
 * K3X_HIP_NOALLOC_SCRATCH_BYTES per device (32 MiB, held until the process
 * ends) instead of the context's grow-only scratch; a call whose buffers do
 * not fit in it less its last 16 KiB returns K3X_ERR_INVALID_EXTENT before
 * anything is enqueued (the config-3 decode layer needs about 1.1 MiB, T=16
 * of it about 9 MiB).  The array is shared by every call on the device,
 * whatever the context or stream: calls that overlap on one GPU race, so a
 * caller serialises them (one stream, or events).  Its last 16 KiB hold the
 * decode path's combine counters, zero when the process loads the library
 * and left zero by every call that completes; nothing else in it needs to
 * start at zero (every other buffer a call reads was written earlier in the
 * same call).  Stage timing
 * (k3x_hip_ctx_set_profiling) is not recorded for these calls.  Results are
 * bit-identical to k3x_hip_moe_forward's.  Asynchronous. */
int k3x_hip_moe_forward_noalloc(k3x_hip_ctx* ctx, k3x_hip_bank* bank,
                                const k3x_hip_moe_params* params, const uint16_t* x,
                                uint16_t* out, const k3x_hip_moe_taps* taps);

/* The same layer with host-decided routes (the reference's own contract:
 * routing on the host, model.cpp:917-1010): xn is the already-normalised
 * bf16 input [T][hidden], ids/weights device [T][K] in router order.  Routes
 * must not repeat an expert within a token and weights must be finite
 * (checked on the host copy passed in host_ids/host_weights, which may be
 * NULL to skip the host check).  Only the routed slots must hold admitted
 * experts: with host_ids the call returns K3X_ERR_INVALID_STATE otherwise;
 * without, the grouping latches K3X_ERR_INVALID_STATE for a route to an
 * empty slot, an expert id out of range or an expert repeated within a
 * token.  Replaces ComputeBackend::mxfp4_situ_moe
 * (backend.hpp:364-368) batched over tokens.  Asynchronous. */
int k3x_hip_moe_forward_routed(k3x_hip_ctx* ctx, k3x_hip_bank* bank,
                               const k3x_hip_moe_params* params,
                               const uint16_t* xn, const uint32_t* ids,
                               const float* weights, const uint32_t* host_ids,
                               const float* host_weights, uint16_t* out,
                               const k3x_hip_moe_taps* taps);

/* Expert-major grouping of device ids [T][K] into the CSR taps (counts,
 * offsets, pair_token, pair_slot, first_use, n_active, active_first_use must
 * be non-NULL).  Replaces build_expert_major_plan
 * (runtime/include/k3x/expert_major.hpp:33-34, expert_major.cpp:10-54).
 * Asynchronous. */
int k3x_hip_expert_major_plan(k3x_hip_ctx* ctx, const uint32_t* ids,
                              uint32_t tokens, uint32_t top_k,
                              uint32_t experts, const k3x_hip_moe_taps* taps);

/* ---- routing from given logits -------------------------------------------- */

/* Element types of the operators that take more than one. */
enum k3x_dtype { K3X_DTYPE_F32 = 0, K3X_DTYPE_BF16 = 1, K3X_DTYPE_F16 = 2 };

/* Score of expert e from its logit l: SIGMOID 1 / (1 + exp(-l)) with the
 * roundings of k3x_hip_moe_forward's router; SOFTMAX exp(l - max) / sum over
 * all experts of the token, formed in double and rounded to fp32 once. */
enum k3x_score { K3X_SCORE_SIGMOID = 0, K3X_SCORE_SOFTMAX = 1 };
/* Score of a group of experts: its largest score + bias, or the sum of its
 * two largest (one, where a group has one expert). */
enum k3x_group_score { K3X_GROUP_MAX = 0, K3X_GROUP_TOP2 = 1 };

typedef struct k3x_hip_route_params {
    uint32_t tokens;        /* T, 1 .. 2^20 */
    uint32_t experts;       /* E, 1 .. 4096 */
    uint32_t top_k;         /* K, 1 .. 64, at most top_groups * E / groups */
    uint32_t dtype;         /* of the logits: K3X_DTYPE_F32 or K3X_DTYPE_BF16 */
    uint32_t scoring;       /* enum k3x_score */
    uint32_t renorm;        /* enum k3x_renorm or K3X_RENORM_NONE */
    float routed_scale;     /* multiplies the weights */
    uint32_t groups;        /* G equal groups of consecutive experts, 1 .. 64, divides E */
    uint32_t top_groups;    /* groups that experts are taken from, 1 .. G */
    uint32_t group_score;   /* enum k3x_group_score */
    uint32_t logits_stride; /* elements from token to token, >= E; 0: E */
} k3x_hip_route_params;

/* Routes T tokens by their router logits (device [T][E]): s = score, a = s +
 * bias in fp32 (bias device fp32 [E], or NULL); with G > 1 only the experts
 * of the top_groups groups of the largest group scores stay; the K largest a
 * in descending order, every tie to the lower index -> ids device u32 [T][K];
 * weights device fp32 [T][K] = s / (sum of the selected s) * routed_scale, or
 * s * routed_scale.  With sigmoid scores and G = 1 the route is that of
 * k3x_hip_moe_forward for the same logits, bit for bit.  ids and weights are
 * what k3x_hip_moe_forward_routed and k3x_hip_expert_major_plan take.
 * A logit of minus infinity has the score 0.  Latched, the token's outputs
 * left as they were: a score, bias or sum that is not finite, with renormalised
 * weights a sum of 0 (K3X_ERR_INVALID_STATE; with K3X_RENORM_DOUBLE and sigmoid
 * scores a logit or bias that is not finite, or the sum, as
 * K3X_ERR_INVALID_EXTENT); other tokens' outputs may then be missing.  The
 * reference routes on the host (runtime/src/routing_policy.cpp:31-160;
 * official_moe.cpp:211-245).
 * Asynchronous. */
int k3x_hip_route(k3x_hip_ctx* ctx, const k3x_hip_route_params* params, const void* logits,
                  const float* bias, uint32_t* ids, float* weights);

/* ---- gated delta rule ------------------------------------------------------ */

/* Decay of the state: none, one a value head, one a key channel. */
enum k3x_gate { K3X_GATE_NONE = 0, K3X_GATE_HEAD = 1, K3X_GATE_CHANNEL = 2 };

typedef struct k3x_hip_delta_params {
    uint32_t sequences;   /* N, 1 .. 65535 */
    uint32_t tokens;      /* T rows of q, k, v, gate, beta and out, 0 .. 2^24 */
    uint32_t key_heads;   /* Hk, divides Hv */
    uint32_t value_heads; /* Hv, 1 .. 1024; value head h has key head h / (Hv / Hk) */
    uint32_t key_dim;     /* K, 1 .. 256 */
    uint32_t value_dim;   /* V, 1 .. 1024 */
    uint32_t dtype;       /* enum k3x_dtype, of q, k, v and out */
    uint32_t gate;        /* enum k3x_gate */
    float scale;          /* of the queries */
    float norm_epsilon;   /* > 0: q and k each over sqrt(sum of squares + epsilon); 0: as given */
    uint32_t longest;     /* tokens of the longest sequence if known, 0: not (then the
                             average).  Chooses the kernels only, token by token or in
                             chunks: results hold whatever it says. */
    uint32_t slots;       /* states in state_in and state_out */
    /* Elements from token to token of q, k, v and out (q, k and v may be
     * parts of one projection's rows), 2^24 at most; 0: packed. */
    uint64_t q_stride, k_stride, v_stride, out_stride;
} k3x_hip_delta_params;

/* The gated delta rule over N sequences, for each value head a state S
 * [K][V] in fp32 and for each of its tokens in order
 *   S = exp(gate) S            (row c times exp(gate_c), or all by one)
 *   u = beta (v - S^T k)
 *   S = S + k u^T
 *   out = scale S^T q
 * q, k device [T][Hk][K], v, out [T][Hv][V], out apart from the inputs; gate
 * fp32 [T][Hv][K] or [T][Hv], <= 0 (minus infinity empties the state; NULL with
 * K3X_GATE_NONE); beta fp32 [T][Hv].  Sequence n has the rows offsets[n] ..
 * offsets[n + 1] - 1 (device u32 [N + 1]; NULL: T / N rows each), of which the
 * first limits[n] only are taken where limits (device u32 [N]) is given: rows of
 * out past them are left as they were.  So a window of the last token and the
 * drafted ones is run with state_out NULL, and run again with it up to the last
 * accepted token.
 * state_in: device fp32 [slots][Hv][K][V], 16-byte aligned, or NULL (zeros);
 * state_out: the same, state_in itself or apart from it, or NULL (not
 * written).  Sequence n has the state slot_index[n] (device u32 [N]), or n
 * without slot_index (then slots >= N).  A sequence of no tokens has its state
 * copied.
 * One token a sequence and short sequences run token by token; longer ones in
 * chunks of 32 whose writes are solved for at once; there an output is also off
 * by up to 2^-28 |q| scale times the largest value that its column takes in the
 * chunk, later tokens' too, for each of the chunk's tokens up to its own.
 * workspace: device, 256-byte aligned, k3x_hip_delta_workspace(params) bytes
 * (NULL where that is 0), the call's own until it is done: calls that may
 * overlap, and captured graphs that may, have one each.
 * Latched: offsets that fall or pass T, a slot past slots, two sequences of
 * one state with state_out (K3X_ERR_INVALID_STATE; nothing of those sequences
 * is read or written); a q, k, v, gate or beta or a state in use that is not
 * finite, with norm_epsilon > 0 a q or k whose sum of squares is not (in fp32),
 * or a gate above 0 (K3X_ERR_INVALID_MXFP4, as for the layer's input); token by
 * token also a product of the state with a k or q as given past fp32.
 * The outputs of a sequence with such values are then not defined.  With states
 * in place (state_out = state_in) the other sequences' outputs and states are
 * those of a call without it (such a call cannot be repeated), but where offsets
 * fall a call in chunks writes nothing.  Of any other call they may be missing,
 * and its state_in is what it was.  Calls of one context that overlap share its
 * status, so that an error of one may leave out parts of the other.  Replaces
 * the recurrence of ComputeBackend::official_kda
 * (runtime/cuda/official_kda.cuh:11-37), batched.
 * Asynchronous. */
int k3x_hip_delta_rule(k3x_hip_ctx* ctx, const k3x_hip_delta_params* params, const void* q,
                       const void* k, const void* v, const float* gate, const float* beta,
                       const uint32_t* offsets, const uint32_t* limits,
                       const uint32_t* slot_index, const float* state_in, float* state_out,
                       void* out, void* workspace, size_t workspace_bytes);
/* Bytes of workspace of such a call; 0 also for parameters that it refuses. */
size_t k3x_hip_delta_workspace(const k3x_hip_delta_params* params);

/* ---- verification of drafted tokens ---------------------------------------- */

/* What a row holds: logits, or probabilities (>= 0; used as they are). */
enum k3x_dist { K3X_DIST_LOGITS = 0, K3X_DIST_PROBS = 1 };

/* draft_counts[n] of a sequence that is left out. */
#define K3X_VERIFY_SKIP 0xffffffffu

typedef struct k3x_hip_verify_params {
    uint32_t sequences;   /* N, 1 .. 65535 */
    uint32_t drafts;      /* D, drafted tokens a sequence, 0 .. 64 */
    uint32_t vocab;       /* V, 1 .. 2^20 */
    uint32_t dtype;       /* of target and draft: K3X_DTYPE_F32 or K3X_DTYPE_BF16 */
    uint32_t form;        /* enum k3x_dist, of target and draft */
    uint32_t greedy;      /* 1: the target's largest entry, ties to the lower token */
    float temperature;    /* > 0; divides logits */
    uint32_t row_stride;  /* elements from row to row of target and draft, >= V; 0: V */
} k3x_hip_verify_params;

/* Verifies N sequences' drafted tokens x (device u32 [N][D]) against the
 * target model's rows (device [N][D + 1][V]; row i follows i drafted tokens).
 * With p and q the target's and the draft's probabilities (softmax(logits /
 * temperature), or the rows themselves), draft i is accepted while
 *   accept_u[n][i] q_i(x_i) < p_i(x_i)
 * and the next token is drawn from max(p_i - q_i, 0) at the first draft i that
 * is not (p_i itself where that is 0 everywhere), or from p_D: the first token
 * whose cumulative sum is over sample_u[n] times the whole.  draft (device
 * [N][D][V]) NULL: q_i is 1 at x_i.
 * accept_u fp32 [N][D], sample_u fp32 [N], in [0, 1).  greedy: accepted while
 * x_i is the largest entry of the target's row i, and the next token is the
 * largest of its row (draft, accept_u and sample_u are not read).
 * Probabilities and their sums are formed in double.
 * accepted u32 [N]; out_tokens u32 [N][D + 1]: the accepted tokens, the next
 * token, then 0xffffffff.  draft_counts (device u32 [N], or NULL) gives
 * sequences fewer drafts than D (the next row is then the last), or
 * K3X_VERIFY_SKIP: accepted 0, no tokens, nothing read.  So a sequence's tokens
 * to commit (limits of k3x_hip_delta_rule) are accepted + 1, and none where
 * out_tokens[n][0] is 0xffffffff.
 * workspace as k3x_hip_delta_rule's, k3x_hip_verify_workspace(params) bytes.
 * Latched as K3X_ERR_INVALID_STATE, the sequence's outputs left as they were: a
 * drafted token past V that is reached, a used row that holds NaN, plus
 * infinity (logits) or a negative or infinite entry (probabilities) or nothing
 * but minus infinity or zeros, a uniform outside [0, 1), a draft count past D;
 * other sequences' outputs may then be missing.  Rows past the first draft that
 * is not accepted are not used; of probabilities, unless greedy, the rows before
 * it only at the drafted token.
 * The reference verifies on the host (generate_speculative,
 * runtime/src/model.cpp:1507).  Asynchronous. */
int k3x_hip_verify_draft(k3x_hip_ctx* ctx, const k3x_hip_verify_params* params,
                         const void* target, const void* draft, const uint32_t* tokens,
                         const uint32_t* draft_counts, const float* accept_u,
                         const float* sample_u, uint32_t* accepted, uint32_t* out_tokens,
                         void* workspace, size_t workspace_bytes);
size_t k3x_hip_verify_workspace(const k3x_hip_verify_params* params);

/* ---- adjustment of logits --------------------------------------------------- */

/* mask_index of a row that no mask applies to. */
#define K3X_NO_MASK 0xffffffffu

typedef struct k3x_hip_logits_params {
    uint32_t sequences;     /* N, 1 .. 65535 */
    uint32_t drafts;        /* D, drafted tokens a sequence, 0 .. 64 */
    uint32_t vocab;         /* V, 1 .. 2^20 */
    uint32_t dtype;         /* of logits and out: K3X_DTYPE_F32 or K3X_DTYPE_BF16 */
    uint32_t row_stride;    /* elements from row to row of logits, >= V; 0: V */
    uint32_t out_stride;    /* the same of out */
    uint32_t history_width; /* tokens from row to row of history */
    uint32_t biases;        /* entries of bias_tokens and bias_values */
    uint32_t masks;         /* rows of masks */
    uint32_t mask_stride;   /* words from row to row of masks, >= ceil(V / 32); 0: that */
} k3x_hip_logits_params;

/* Adjusts the rows that k3x_hip_verify_draft takes (device [N][D + 1][V]; row i
 * follows i drafted tokens) before anything is drawn from them.  With c the
 * number of times that a token stands in the sequence's answer, the history past
 * its prompt and the drafted tokens before the row, each logit l becomes, in fp32
 * and in this order,
 *   l > 0 ? l / repetition : l * repetition   where the token stands in the
 *                                             prompt or the answer
 *   l - frequency c, then l - presence        where c > 0
 *   l + its bias
 *   minus infinity                            where the row's mask bit is 0
 * and is rounded to its type once.  out (device [N][D + 1][V]) is logits or apart
 * from it.
 * history: device u32 [N][history_width], of which sequence n has
 * history_lens[n] tokens and of those prompt_lens[n] (NULL: 0) in its prompt;
 * drafts as k3x_hip_verify_draft's tokens, u32 [N][D], and draft_counts: rows of
 * sequences that are left out and rows past a sequence's drafts are left as they
 * were.  repetition, frequency, presence: fp32 [N]; NULL leaves a step out.
 * Biases: entries bias_offsets[n] .. bias_offsets[n + 1] - 1 (device u32 [N + 1])
 * of bias_tokens (u32) and bias_values (fp32) are sequence n's; of several for one
 * token the last holds.  masks: device u32 [masks][mask_stride], bit t % 32 of word
 * t / 32 set where token t is allowed; row i of sequence n has the mask
 * mask_index[n][i] (u32 [N][D + 1]) or K3X_NO_MASK.  history, bias_offsets and
 * masks may each be NULL, with what belongs to them; without a history drafted
 * tokens count all the same.
 * Latched as K3X_ERR_INVALID_STATE: a history longer than its row, a prompt longer
 * than its history, a token of the history, a draft or a bias past V, bias offsets
 * that fall or pass `biases`, a mask past `masks`, a draft count past D, a
 * repetition that is not a number above 0, a frequency or presence that is not
 * finite; rows of that sequence may then be missing or hold some of the steps.  With
 * out = logits all rows of the other sequences are adjusted (such a call cannot be
 * repeated); of any other call they may be missing.  Calls that overlap on one
 * context: as for k3x_hip_delta_rule.
 * Logits and biases may hold anything and go through the arithmetic as they are.
 * Asynchronous. */
int k3x_hip_adjust_logits(k3x_hip_ctx* ctx, const k3x_hip_logits_params* params,
                          const void* logits, const uint32_t* history,
                          const uint32_t* history_lens, const uint32_t* prompt_lens,
                          const uint32_t* drafts, const uint32_t* draft_counts,
                          const float* repetition, const float* frequency,
                          const float* presence, const uint32_t* bias_offsets,
                          const uint32_t* bias_tokens, const float* bias_values,
                          const uint32_t* masks, const uint32_t* mask_index, void* out);

/* ---- latent attention -------------------------------------------------------- */

/* How a cached token's latent is held: 16-bit values of the call's type, or E4M3
 * or E2M1 codes with one E8M0 scale for 32 of them. */
enum k3x_cache_format { K3X_CACHE_16BIT = 0, K3X_CACHE_MXFP8 = 1, K3X_CACHE_MXFP4 = 2 };

/* A cache of latents in pages, and the tokens of a call.
 *
 * pool: device, 256-byte aligned, [pages][page_size] rows of
 * k3x_hip_mla_row_bytes() bytes, each
 *   the latent: L 16-bit values, L E4M3 codes, or L / 2 bytes of E2M1 codes, low
 *   nibble first;
 *   the rotary part: R 16-bit values;
 *   with codes: L / 32 scale bytes (2^(b - 127)) and zeros up to 16.
 * table: device u32 [N][table_width]: position p of sequence n is row p %
 * page_size of page table[n][p / page_size].  Pages may be shared between
 * sequences; entries past the last used one are not read.
 * lens: device u32 [N], the positions of each sequence with the call's own
 * tokens: sequence n has the rows offsets[n] .. offsets[n + 1] - 1 of the call's
 * tensors (device u32 [N + 1]; NULL: T / N rows each), and they are its last
 * positions, lens[n] - (offsets[n + 1] - offsets[n]) .. lens[n] - 1.  Rows at
 * positions below 0 (a padded sequence has lens[n] = 0) are not written, read or
 * seen.  Rows past offsets[N] are left as they were.
 * Tensors of a call without tokens may be NULL.
 * Latched as K3X_ERR_INVALID_STATE by every call, which then reads and writes
 * nothing outside its tensors and the pool, and leaves outputs undefined: offsets
 * that fall or pass T, a length past table_width * page_size or 2^29, a page in use
 * that is not below `pages`, more tokens in a sequence than `longest`.  Attention
 * may also latch more work than one call takes: a sequence whose rows (tokens x
 * heads) times positions pass 2^36, or sequences for which these products together
 * pass 2^40 or whose positions together pass 2^34. */
typedef struct k3x_hip_mla_params {
    uint32_t sequences;    /* N, 1 .. 65535 */
    uint32_t tokens;       /* T, 0 .. 2^22 */
    uint32_t heads;        /* H, 1 .. 1024 (k3x_hip_mla_attention) */
    uint32_t latent;       /* L, a multiple of 32, 32 .. 512 */
    uint32_t rotary;       /* R, a multiple of 8, 0 .. 64 */
    uint32_t dtype;        /* K3X_DTYPE_BF16, or K3X_DTYPE_F16 with K3X_CACHE_16BIT */
    uint32_t cache_format; /* enum k3x_cache_format */
    uint32_t page_size;    /* 1 .. 65536 */
    uint32_t pages;        /* of the pool, pages * page_size at most 2^31 */
    uint32_t table_width;  /* 1 .. 2^20 */
    uint32_t longest;      /* tokens of the call in a sequence at most; 0: T.  Times heads
                              below 2^31 (k3x_hip_mla_attention). */
    float scale;           /* of the scores, > 0 (k3x_hip_mla_attention) */
    float norm_epsilon;    /* >= 0, with gamma (k3x_hip_mla_store) */
    /* Elements from token to token of latent, rotary, q and out; 0: packed. */
    uint64_t latent_stride, rotary_stride, q_stride, out_stride;
} k3x_hip_mla_params;

/* Bytes of a cached row; 0 for parameters that the calls refuse. */
size_t k3x_hip_mla_row_bytes(const k3x_hip_mla_params* params);

/* Writes the call's tokens to their pages: latent device [T][L], rotary [T][R]
 * (NULL with R = 0), both of the call's type.  gamma (device fp32 [L], or NULL):
 * the latent is normalised first, x / sqrt(mean(x^2) + norm_epsilon) * gamma,
 * formed in double, rounded to fp32 and then to the call's type.  Codes are rounded
 * to nearest, ties to even, with the least scale (2^-110 at least) by which the
 * largest of its 32 is at most 448 (E4M3) or 6 (E2M1), so that nothing saturates.
 * Tokens of sequences that share the page of their last positions overwrite one
 * another.
 * Also latched, as K3X_ERR_INVALID_MXFP4, the token's row left as it was: a latent
 * or rotary part that is not finite as it is written; other tokens' rows may then
 * be missing (repeated, such a call writes what it wrote again).  Asynchronous. */
int k3x_hip_mla_store(k3x_hip_ctx* ctx, const k3x_hip_mla_params* params, const void* latent,
                      const void* rotary, const float* gamma, const uint32_t* table,
                      const uint32_t* offsets, const uint32_t* lens, void* pool);

/* Reads the call's tokens back from their pages, as the values that they stand
 * for: latent device [T][L], rotary [T][R] (NULL: not read), of the call's type
 * (codes times their scales are bf16 numbers).  A whole prefix of n tokens is a
 * call with n rows and lens n.  Asynchronous. */
int k3x_hip_mla_load(k3x_hip_ctx* ctx, const k3x_hip_mla_params* params, const void* pool,
                     const uint32_t* table, const uint32_t* offsets, const uint32_t* lens,
                     void* latent, void* rotary);

/* Attention over the cached latents with the up-projections absorbed: q device
 * [T][H][L + R], the latent part of each query multiplied by its head's key
 * projection already; a token's key is its row of L + R values for every head and
 * its value the first L of them.  A token at position p sees positions 0 .. p:
 *   out = sum softmax(scale q . key) latent    (device [T][H][L], of the call's type)
 * and lse (device fp32 [T][H], or NULL) is the logarithm of the softmax's sum.  A
 * token that sees nothing has zeros and minus infinity.  Sums are held in fp32;
 * a key's weight is rounded to the call's type before it multiplies the latent.
 * q, out and pool 16-byte aligned, strides of q and out multiples of 8 elements.
 * workspace as k3x_hip_delta_rule's, k3x_hip_mla_attention_workspace(params)
 * bytes, also for a call without tokens (0: parameters that it refuses).
 * Also latched, as K3X_ERR_INVALID_MXFP4: an output that is not finite (for a query
 * or a cached row that is not, or sums of weighted latents past fp32), scores of a
 * token that are all minus infinity (past fp32, or for such a query), and with fp16
 * scores (times scale) of 2^24 and more, which its weights may not hold.  Replaces
 * the attention of reference/k3x_ref/mla.py, batched.  Asynchronous. */
int k3x_hip_mla_attention(k3x_hip_ctx* ctx, const k3x_hip_mla_params* params, const void* q,
                          const void* pool, const uint32_t* table, const uint32_t* offsets,
                          const uint32_t* lens, void* out, float* lse, void* workspace,
                          size_t workspace_bytes);
size_t k3x_hip_mla_attention_workspace(const k3x_hip_mla_params* params);

typedef struct k3x_hip_mla_prompt_params {
    uint32_t sequences; /* N, 1 .. 65535 */
    uint32_t tokens;    /* T rows of q and out, 0 .. 2^22 */
    uint32_t keys;      /* S rows of k, v and rotary, 0 .. 2^22 */
    uint32_t heads;     /* H, 1 .. 1024 */
    uint32_t key_dim;   /* Dn of a head of its own, a multiple of 8, 8 .. 128 */
    uint32_t rotary;    /* R, a multiple of 8, 0 .. 64 */
    uint32_t value_dim; /* Dv, a multiple of 8, 8 .. 128 */
    uint32_t dtype;     /* K3X_DTYPE_BF16 or K3X_DTYPE_F16 */
    uint32_t causal;    /* 1: the last query sees every key, each before it one less */
    uint32_t longest;   /* queries of the longest sequence if known, 0: not (then T).  Only
                           how the work is laid out: results hold whatever it says. */
    float scale;        /* of the scores, > 0 */
    /* Elements from row to row (of k, v and rotary 2^27 at most; with one key not
     * used), and of k and v from head to head (k and v may be parts of one
     * projection's rows); multiples of 8; 0: packed. */
    uint64_t q_stride, k_stride, v_stride, rotary_stride, out_stride;
    uint64_t k_head_stride, v_head_stride;
} k3x_hip_mla_prompt_params;

/* Attention of prompts over expanded keys and values: q device [T][H][Dn + R], k
 * [S][H][Dn], v [S][H][Dv], rotary [S][R] (the part of a key that all heads share;
 * NULL with R = 0):
 *   out = sum softmax(scale q . (k, rotary)) v    (device [T][H][Dv])
 * Sequence n has the queries offsets[n] .. offsets[n + 1] - 1 and the keys
 * key_offsets[n] .. key_offsets[n + 1] - 1 (device u32 [N + 1] each; NULL: T / N and
 * S / N rows each), a cached prefix's first.  causal: query i of m sees the first
 * n - m + i + 1 of n keys.  lse, empty rows, sums and weights as for
 * k3x_hip_mla_attention.  q, k, v, rotary and out 16-byte aligned, those without rows
 * may be NULL.  Heads times (T / 128 + min(N, T)) are below 2^24.
 * Latched: offsets that fall, pass T or S (K3X_ERR_INVALID_STATE; nothing of such
 * a sequence is read), and as for k3x_hip_mla_attention outputs that are not finite
 * and scores (K3X_ERR_INVALID_MXFP4).
 * Asynchronous. */
int k3x_hip_mla_prompt(k3x_hip_ctx* ctx, const k3x_hip_mla_prompt_params* params, const void* q,
                       const void* k, const void* v, const void* rotary, const uint32_t* offsets,
                       const uint32_t* key_offsets, void* out, float* lse);

/* ---- official K3 MoE FFN (Stable LatentMoE) ------------------------------ */

/* The official layer wraps a bank of experts that run at the latent width L
 * (the bank's hidden): routed_down [L][H] bf16 -> experts -> slot-ordered
 * mix -> routed_norm RMSNorm -> routed_up [H][L] bf16, plus a bf16 shared
 * FFN at H (shared_inter Is, the reference's two shared experts side by
 * side) and the prefix add (runtime/src/official_moe.cpp:271-344;
 * OfficialMoeFfnView, runtime/include/k3x/backend.hpp:171-176). */
typedef struct k3x_hip_official k3x_hip_official;

typedef struct k3x_hip_official_desc {
    uint32_t hidden;          /* H, multiple of 128 */
    uint32_t shared_inter;    /* Is, 0 (none) or a multiple of 128 */
    uint32_t router_experts;  /* rows of the router: 0 (the bank's experts) with
                                 a bank; without one (a route-only object:
                                 uploads of the route and prepare only;
                                 shared_inter 0), the router's row count */
} k3x_hip_official_desc;

/* Optional device buffers for intermediates of k3x_hip_official_ffn (any may
 * be NULL).  T tokens, K top_k, E experts, L latent, H hidden. */
typedef struct k3x_hip_official_taps {
    float* logits;         /* [T][E] (device routing only) */
    uint32_t* ids;         /* [T][K] route order */
    float* contributions;  /* [T][K] */
    uint16_t* latent;      /* [T][L] bf16 bits, routed_down output */
    float* expert_out;     /* [T][K][L] expert outputs before their bf16 rounding */
    uint16_t* mixed;       /* [T][L] bf16 bits, slot-ordered mix */
    float* routed;         /* [T][H] routed_up output before rounding */
    float* shared;         /* [T][H] shared FFN output before rounding */
} k3x_hip_official_taps;

/* experts: a bank of hidden L (its own shared expert unused); the official
 * layer keeps a reference to it and must be destroyed first.  experts NULL
 * makes a route-only object (desc->router_experts rows): upload_route,
 * fill_synthetic and prepare work on it, upload_ffn and ffn return
 * K3X_ERR_INVALID_STATE -- route preparation needs no experts, as
 * prepare_official_moe_route (backend.hpp:384-389) takes none. */
int k3x_hip_official_create(k3x_hip_ctx* ctx, k3x_hip_bank* experts,
                            const k3x_hip_official_desc* desc,
                            k3x_hip_official** out);
int k3x_hip_official_destroy(k3x_hip_official* official);

/* Host bf16 words: routed_down [L][H], routed_norm [L], routed_up [H][L];
 * shared gate, up [Is][H] and down [H][Is] (NULL when Is = 0).
 * OfficialMoeFfnView (backend.hpp:171-176).  Synchronous. */
int k3x_hip_official_upload_ffn(k3x_hip_official* official, const uint16_t* routed_down,
                                const uint16_t* routed_norm, const uint16_t* routed_up,
                                const uint16_t* shared_gate, const uint16_t* shared_up,
                                const uint16_t* shared_down);

/* Host: bf16 words residual_norm [H], residual_proj [H], post_norm [H],
 * router [E][H]; fp32 correction [E].  OfficialMoeRoutePrepareView
 * (backend.hpp:184-189) plus the router correction.  Synchronous. */
int k3x_hip_official_upload_route(k3x_hip_official* official, const uint16_t* residual_norm,
                                  const uint16_t* residual_proj, const uint16_t* post_norm,
                                  const uint16_t* router, const float* correction);

/* Seeded synthetic weights for both uploads (no reference counterpart):
 * dense matrices and the router ~ N(0, sigma^2) in bf16, the three norm
 * vectors 1, residual_proj ~ N(0, proj_sigma^2), correction ~
 * N(0, correction_sigma^2).  Synchronous. */
int k3x_hip_official_fill_synthetic(k3x_hip_official* official, uint64_t seed, float sigma,
                                    float router_sigma, float proj_sigma,
                                    float correction_sigma);

/* Route preparation for T tokens: the two-source attention-residual mix and
 * post-norm (official_moe.cpp:156-209) -> hidden bf16 [T][H], and, when
 * logits is non-NULL, the router logits [T][E] over it (official_moe.cpp:
 * 247-269).  prefix and block_residual device fp32 [T][H].  Replaces
 * ComputeBackend::prepare_official_moe_route (backend.hpp:384-389) with the
 * hidden kept on the device.  Asynchronous. */
int k3x_hip_official_prepare(k3x_hip_ctx* ctx, k3x_hip_official* official, uint32_t tokens,
                             float rms_epsilon, const float* prefix,
                             const float* block_residual, uint16_t* hidden, float* logits);

/* The FFN for T tokens: hidden bf16 [T][H] (prepared), prefix fp32 [T][H];
 * the route as device ids [T][K] + contributions [T][K], or ids ==
 * contributions == NULL to route on the device (router logits over hidden,
 * sigmoid + correction, natural Top-K, contributions s / sum s in double:
 * official_moe.cpp:211-245; every slot of the bank must then hold an
 * admitted expert, while a given route needs only its own slots).  out bf16 [T][H] = bf16(bf16(prefix) +
 * bf16(routed + shared)).  params: tokens, top_k, rms_epsilon and the GLU
 * (SiTU for the reference's layer); routed_scale, renorm and flags are not
 * used.  Replaces ComputeBackend::official_mxfp4_moe_ffn
 * (backend.hpp:376-383) batched over tokens.  Asynchronous. */
int k3x_hip_official_ffn(k3x_hip_ctx* ctx, k3x_hip_official* official,
                         const k3x_hip_moe_params* params, const uint16_t* hidden,
                         const float* prefix, const uint32_t* ids,
                         const float* contributions, uint16_t* out,
                         const k3x_hip_official_taps* taps);

/* ---- fp32 products and the resident latent layer ------------------------ */

/* The fp32 operations of ComputeBackend: each product is formed exactly in
 * double and summed in double, one rounding to fp32 at the end (the
 * reference sums sequentially; only the order differs).  All pointers are
 * device memory; every call is asynchronous on the context stream.  Inputs
 * x are [tokens][cols] fp32, outputs [tokens][rows] fp32. */

/* y = W x, W fp32 [rows][cols] row-major.  Replaces
 * ComputeBackend::dense_matvec (runtime/include/k3x/backend.hpp:333-335;
 * runtime/src/backend_cpu.cpp:22-45). */
int k3x_hip_dense_f32_matvec(k3x_hip_ctx* ctx, const float* W, uint32_t rows, uint32_t cols,
                             const float* x, uint32_t tokens, float* y);

/* y = W x for an MXFP4 matrix in the K3X layout: packed [rows][cols / 2]
 * (low nibble = even column, 16-byte aligned), E8M0 scales
 * [rows][cols / 32], group size 32.  Replaces ComputeBackend::mxfp4_matvec
 * (backend.hpp:336-338; backend_cpu.cpp:47-59, runtime/src/ops.cpp:57-76);
 * scale bytes must be checked for 0xFF by the caller (the reference's
 * decode_mxfp4 rejects them). */
int k3x_hip_mxfp4_matvec(k3x_hip_ctx* ctx, const uint8_t* packed, const uint8_t* scales,
                         uint32_t rows, uint32_t cols, const float* x, uint32_t tokens, float* y);

/* The fp32 SiTU MLP: act [tokens][inter] = situ_glu(gate x, up x) (gate and
 * up [inter][hidden]), y [tokens][out_rows] = down act (down
 * [out_rows][inter]).  Replaces ComputeBackend::dense_situ_mlp
 * (backend.hpp:345-348; backend_cpu.cpp:108-122). */
int k3x_hip_dense_situ_mlp(k3x_hip_ctx* ctx, const float* gate, const float* up,
                           const float* down, uint32_t hidden, uint32_t inter, uint32_t out_rows,
                           float situ_beta, int has_situ_linear, float situ_linear_beta,
                           const float* x, uint32_t tokens, float* act, float* y);

/* fp32 dense weights of the resident latent MoE layer, device row-major
 * (ResidentMoeLayerView, backend.hpp:302-307). */
typedef struct k3x_hip_latent_weights {
    const float* routed_down;  /* [latent][hidden] */
    const float* routed_norm;  /* [latent] */
    const float* routed_up;    /* [hidden][latent] */
    const float* shared_gate;  /* [shared_inter][hidden] */
    const float* shared_up;    /* [shared_inter][hidden] */
    const float* shared_down;  /* [hidden][shared_inter] */
    uint32_t hidden, latent, shared_inter;
    /* The width routed_norm's RMSNorm divides the sum of squares by: 0 means
     * latent.  A caller that pads the latent to the bank's width with zeros
     * (zero routed_down rows, zero expert codes in the padded rows and
     * columns, zero routed_norm entries and routed_up columns) passes the
     * unpadded width, so the padded layer computes the unpadded one. */
    uint32_t latent_norm;
} k3x_hip_latent_weights;

/* The resident latent MoE layer for T tokens: latent = routed_down x; the
 * routed experts of `bank` (hidden = latent, no shared expert) on the fp32
 * latent, slots ids [T][K] (device) mixed in slot order with contributions
 * [T][K] in fp32; normalized = RMSNorm(mixed, routed_norm); out [T][hidden]
 * = routed_up normalized + the fp32 SiTU MLP of x.  x, out device fp32;
 * mixed_out (optional) receives the mix [T][latent].  params: tokens,
 * top_k, rms_epsilon, glu = SiTU and its betas; flags must be 0 (the call
 * sets its own).  host_ids / host_contributions as
 * k3x_hip_moe_forward_routed.  Replaces
 * ComputeBackend::resident_mxfp4_moe_layer (backend.hpp:369-375;
 * runtime/src/backend_cpu.cpp:305-339, runtime/cuda/backend_cuda.cu:
 * 1789-2545). */
int k3x_hip_resident_moe_layer(k3x_hip_ctx* ctx, k3x_hip_bank* bank,
                               const k3x_hip_latent_weights* weights,
                               const k3x_hip_moe_params* params, const float* x,
                               const uint32_t* ids, const float* contributions,
                               const uint32_t* host_ids, const float* host_contributions,
                               float* out, float* mixed_out);

/* ---- Measurement --------------------------------------------------------- */

/* Streams `bytes` device bytes at `data` (16-byte aligned, a multiple of 16)
 * through the vector memory path once, on the context stream, and XORs
 * every 32-bit word of them into *fold (device memory, left as is
 * otherwise): the device's plain streaming-read rate, the practical ceiling
 * that a streaming kernel's HBM rate is read against beside the nominal
 * 8 TB/s.  No counterpart in the reference (measurement only).
 * Asynchronous. */
int k3x_hip_stream_read(k3x_hip_ctx* ctx, const void* data, size_t bytes, uint32_t* fold);

/* ---- K3X storage records -------------------------------------------------- */

/* CRC32C (Castagnoli, reflected, preset and final inversion 0xFFFFFFFF) of
 * `bytes` device bytes at `data` (16-byte aligned), computed on the device:
 * the value runtime/src/crc32c.cpp:22-28 computes on the host, for data
 * already in HBM.  Synchronous (the context stream is drained). */
int k3x_hip_crc32c(k3x_hip_ctx* ctx, const void* data, size_t bytes, uint32_t* crc);

/* Uploads expert `expert` of the bank from six device extents in the K3X
 * storage order -- gate codes, gate scales, up codes, up scales, down codes,
 * down scales (runtime/src/storage_slice.cpp:56-73), each 16-byte aligned
 * and of the bank's sizes -- after checking each against its CRC32C
 * (crc32c[6] as the tensor records hold them, runtime/src/reader.cpp:98-99;
 * NULL skips the check): K3X_ERR_DATA_CRC_MISMATCH or
 * K3X_ERR_AUXILIARY_CRC_MISMATCH, slot untouched, on a mismatch; a scale
 * byte 0xFF is K3X_ERR_INVALID_MXFP4.  Identities as
 * k3x_hip_bank_upload_expert.  Synchronous. */
int k3x_hip_bank_upload_expert_device(k3x_hip_bank* bank, uint32_t expert,
                                      const uint64_t tensor_ids[3],
                                      const uint8_t* const extents[6],
                                      const uint32_t crc32c[6]);

/* A K3X checkpoint opened for expert loads (K3X_FORMAT.md).  Opening reads
 * and checks the superblock and the directories as Reader::open does
 * (runtime/src/reader.cpp:414-560): magic, version, superblock CRC32C,
 * required features, reserved bytes, finalized state and length, directory
 * ranges and headers, model-config invariants, tensor record fields,
 * distinct tensor ids; every tensor extent in range, 4 KiB aligned and
 * disjoint from the others.  Status codes are the reader's (K3X_ERR_IO ..
 * K3X_ERR_INVALID_EXTENT).  Host work only. */
typedef struct k3x_hip_storage k3x_hip_storage;
int k3x_hip_storage_open(const char* path, k3x_hip_storage** out);
int k3x_hip_storage_close(k3x_hip_storage* storage);
/* The checks Reader::open adds with VerifyMode::checksums
 * (runtime/src/reader.cpp:672-721), in its order: every tensor's data and
 * auxiliary CRC32C (K3X_ERR_DATA_CRC_MISMATCH, K3X_ERR_AUXILIARY_CRC_MISMATCH),
 * the SHA-256 of the tensor, layer and expert directories and the model
 * config concatenated against superblock bytes 168..199
 * (K3X_ERR_DIRECTORY_SHA256_MISMATCH), the SHA-256 of the whole file with
 * bytes 200..231 and 4092..4095 read as zeros against bytes 200..231
 * (K3X_ERR_ROOT_SHA256_MISMATCH).  Host work only (SHA-256 is sequential). */
int k3x_hip_storage_verify(k3x_hip_storage* storage);

/* load_storage_expert (runtime/src/storage_slice.cpp:42-92) into bank slot
 * `expert`: the tensors model.layers.<layer>.feed_forward.experts.<id>.
 * {gate,up,down}, found by the FNV-1a 64 hash of their names, must be
 * native MXFP4 matrices of the bank's shape (gate/up [inter][hidden], down
 * [hidden][inter]; K3X_ERR_INVALID_MXFP4) of that layer and expert; the
 * artifact must carry the STORAGE_FIXTURE optional feature
 * (K3X_ERR_INVALID_EXTENT otherwise).  The six extents are read in one batch
 * into pinned host memory, copied to the device once, checked against their
 * records' CRC32C on the device and uploaded with
 * k3x_hip_bank_upload_expert_device; the slot's tensor ids are the records'.
 * *bytes_read (may be NULL): the six extents' total.  ordered_sha256 (may be
 * NULL; 32 bytes): the SHA-256 of the six extents in their order (gate data,
 * gate scales, up data, up scales, down data, down scales), the digest
 * load_storage_expert returns (storage_slice.cpp:80-90), formed on the host
 * from the bytes read.  Synchronous. */
int k3x_hip_storage_upload_expert(k3x_hip_storage* storage, k3x_hip_bank* bank, uint32_t expert,
                                  uint32_t layer_id, uint32_t expert_id, uint64_t* bytes_read,
                                  uint8_t* ordered_sha256);

#ifdef __cplusplus
}
#endif
#endif
