// k3x_mla_mma.hpp -- what the kernels of latent attention on the matrix cores
// (mla_attention.hip, mla_prompt.hip) share: products of 32 (or 16) rows, tiles
// in LDS and how their reads are kept apart.
#pragma once

#include "k3x_ops.hpp"

namespace k3x_mla {

using namespace k3x_dev;

// Which columns of 16 bytes are exchanged in token t of a tile's 64-column group
// (128 bytes a token), so that reads do not meet in a bank: 64 banks hold two
// tokens, keys are read sixteen tokens at a time at one column, values four or
// eight tokens at four or two columns.  So the bits of t / 2, reversed.
__device__ inline uint32_t swizzle(uint32_t t) {
    return (t << 1 & 4) | (t >> 1 & 2) | (t >> 3 & 1);
}

template <uint32_t DT, int HT>
struct Mma;
template <uint32_t DT>
struct Mma<DT, 32> {
    typedef __attribute__((ext_vector_type(16))) float Acc;
    static __device__ inline Acc run(u32x4 a, u32x4 b, Acc c) {
        typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
        if constexpr (DT == K3X_DTYPE_BF16)
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                           __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                          __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <uint32_t DT>
struct Mma<DT, 16> {
    typedef f32x4 Acc;
    static __device__ inline Acc run(u32x4 a, u32x4 b, Acc c) {
        typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
        if constexpr (DT == K3X_DTYPE_BF16)
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                           __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                          __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// Two values as the type's bits, the first in the low half.
template <uint32_t DT>
__device__ inline uint32_t pack2(float a, float b) {
    typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
    if constexpr (DT == K3X_DTYPE_BF16)
        return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
    else
        return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}

// Four outputs as the type's bits.  An output lies between the values that it is a mean of, but
// rounded weights and their unrounded sum may put it past them by 2^-11 of itself: not past
// fp16's largest number.  (Values of bf16 so large have sums past fp32 first.)
template <uint32_t DT>
__device__ inline uint2 outputs4(float4 v) {
    auto within = [](float x) {
        return DT == K3X_DTYPE_F16 ? __builtin_amdgcn_fmed3f(x, -65504.0f, 65504.0f) : x;
    };
    return uint2{pack2<DT>(within(v.x), within(v.y)), pack2<DT>(within(v.z), within(v.w))};
}

// Over the lanes that hold one row's scores: the halves, and for 16 rows the
// 16-lane rows too.
template <int HT, typename Op>
__device__ inline float across(float x, Op op) {
    const uint32_t u = __float_as_uint(x);
    const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    x = op(__uint_as_float(h[0]), __uint_as_float(h[1]));
    if constexpr (HT == 16) {
        const uint32_t w = __float_as_uint(x);
        const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
        x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return x;
}

// Weights are powers of two of the scores past a row's reference, which is its largest score so
// far less kLift, and may lag behind it: by kLag in all, so that sums and outputs are seldom
// multiplied again.  They are rounded to the call's type for the second product, as the matrix
// cores take operands of 16 bits; sums are of the unrounded ones.  Outputs of bf16 are off by
// 0.0017 to 0.0021 of themselves so, with fp32 weights by the 0.0016 to 0.0017 of their own
// rounding.  bf16 has fp32's exponents.
// Of fp16 the range is spent above: with the largest at 2^0 weights below 2^-25 would vanish,
// 0.3% of the output where 10^5 are of about that size; at 2^7 (2^15 at most of its 2^16) they
// are rounded by 2^-32 of the largest.
template <uint32_t DT>
struct Weights {
    static constexpr float kLift = DT == K3X_DTYPE_F16 ? 7.0f : 0.0f;
    static constexpr float kLag = DT == K3X_DTYPE_F16 ? 15.0f : 8.0f;
    static __device__ inline bool over(float top, float m) { return top > m + kLag; }
    static __device__ inline float reference(float top, float m) { return fmaxf(m, top - kLift); }
};

// A row that sees tokens has a sum: its largest weight is 1 or more.  None (or NaN) is that of scores
// that are all minus infinity, or no numbers.  And of scores of 2^28 and more a weight's power
// of two is off by the rounding of its reference m, more than 2^4 either way: in fp16 even the
// largest weight may vanish while the sum, in fp32, is there.
template <uint32_t DT>
__device__ inline bool no_softmax(int32_t sees, float sum, float m) {
    return sees > 0 && (!(sum > 0.0f) || (DT == K3X_DTYPE_F16 && fabsf(m) > 0x1p28f));
}

// x, as a value that is not computed ahead of the place and held until then.
__device__ inline uint32_t opaque(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

typedef __attribute__((address_space(3))) uint8_t lds_byte;

__device__ inline u32x4 lds16(const lds_byte* p) {
    return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(p);
}
// Of a 16-lane row's four tokens by 16 columns, its lane's column.  __restrict__: read
// without it the compiler waits for every direct load to LDS before, those of later
// tiles too; what may be read is settled by the tile's own wait and barrier.
__device__ inline uint2 lds_transposed(const lds_byte* __restrict__ p) {
    typedef __attribute__((ext_vector_type(4))) short s16x4;
    return __builtin_bit_cast(
        uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (__attribute__((address_space(3))) s16x4*)const_cast<lds_byte*>(p)));
}

template <int N>
__device__ inline void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ inline void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// o[FROM .. FROM + N - 1] *= k.  HELD: the kernel's results fill so much of the
// register file that they stay in its accumulators, which no other instruction
// multiplies: each goes through one register in between.  (Left to the compiler, the
// branch around this makes it hold them twice: in mla_attention.hip 700 registers go to
// memory.)  The products that wrote them have ended: those of the next tile's scores lie
// between, and the waits here cover what the compiler does not see.
template <bool HELD, int FROM, int N, int OT, typename Acc>
__device__ __forceinline__ void scale_tiles(Acc (&o)[OT], float k) {
    constexpr int W = sizeof(Acc) / 4;
    if constexpr (!HELD) {
#pragma unroll
        for (int i = FROM; i < FROM + N; ++i) o[i] *= k;
    } else {
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
        for (int i = FROM; i < FROM + N; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                float x = o[i][j], t;
                asm volatile(
                    "v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %2, %1\n\t"
                    "v_accvgpr_write_b32 %0, %1"
                    : "+a"(x), "=&v"(t) : "v"(k));
                o[i][j] = x;
            }
        asm volatile("s_nop 15" ::: "memory");
    }
}

}  // namespace k3x_mla
