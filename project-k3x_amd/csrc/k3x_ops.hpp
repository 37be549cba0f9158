// k3x_ops.hpp -- what the operators on caller tensors (route.hip, delta.hip,
// verify.hip) share: element types and the error latch.
#pragma once

#include "k3x_device.hpp"
#include "k3x_internal.hpp"

namespace k3x_ops {

__device__ inline void latch(uint32_t* status, uint32_t code) { atomicCAS(status, 0u, code); }

// One element type of a caller's tensor: its storage, and fp32 in and out
// (out rounds to nearest even).
template <uint32_t DT>
struct Elem;
template <>
struct Elem<K3X_DTYPE_F32> {
    typedef float type;
    static __device__ inline float load(type v) { return v; }
    static __device__ inline type store(float v) { return v; }
};
template <>
struct Elem<K3X_DTYPE_BF16> {
    typedef uint16_t type;
    static __device__ inline float load(type v) { return k3x_dev::bf16_to_f32(v); }
    static __device__ inline type store(float v) {
        return __builtin_bit_cast(uint16_t, (__bf16)v);
    }
};
template <>
struct Elem<K3X_DTYPE_F16> {
    typedef _Float16 type;
    static __device__ inline float load(type v) { return (float)v; }
    static __device__ inline type store(float v) { return (_Float16)v; }
};

// exp(x - k ln2) for k = rint(x / ln2), by the series to r^13 on |r| <= ln2 / 2:
// the steps of expf_cr.
__device__ inline double exp_series(double x, double k) {
    double r = __builtin_fma(-k, 6.93147180369123816490e-01, x);
    r = __builtin_fma(-k, 1.90821492927058770002e-10, r);
    double p = 1.6059043836821614599e-10;
    p = __builtin_fma(p, r, 2.0876756987868098979e-09);
    p = __builtin_fma(p, r, 2.5052108385441718775e-08);
    p = __builtin_fma(p, r, 2.7557319223985890653e-07);
    p = __builtin_fma(p, r, 2.7557319223985890653e-06);
    p = __builtin_fma(p, r, 2.4801587301587301587e-05);
    p = __builtin_fma(p, r, 1.9841269841269841270e-04);
    p = __builtin_fma(p, r, 1.3888888888888888889e-03);
    p = __builtin_fma(p, r, 8.3333333333333333333e-03);
    p = __builtin_fma(p, r, 4.1666666666666666667e-02);
    p = __builtin_fma(p, r, 1.6666666666666666667e-01);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_fma(p, r, 1.0);
}

// exp(x), x <= 0, in double.  Minus infinity gives 0, NaN itself.
__device__ inline double exp_f64(double x) {
    const double y = x < -746.0 ? -746.0 : x;  // exp is 0 from there on; keeps a NaN
    const double k = __builtin_rint(y * 1.4426950408889634);
    return __builtin_ldexp(exp_series(y, k), (int)k);
}

// A wave's LDS writes are seen by its other lanes, in order.
__device__ inline void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// One double by a DPP control or a lane exchange of its halves.
template <int Ctrl>
__device__ inline double dpp_f64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, Ctrl, 0xf, 0xf,
                                                              false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), Ctrl,
                                                              0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Sum over the wave, the same on every lane: a tree over pairs, quads, halves
// of rows, rows, row pairs and halves, in registers.
__device__ inline double wave_sum(double x) {
    x += dpp_f64<0xb1>(x);   // quad_perm [1,0,3,2]
    x += dpp_f64<0x4e>(x);   // quad_perm [2,3,0,1]
    x += dpp_f64<0x141>(x);  // row_half_mirror
    x += dpp_f64<0x140>(x);  // row_mirror
#pragma unroll
    for (int halves = 0; halves < 2; ++halves) {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        const uint32_t l = (uint32_t)u, h = (uint32_t)(u >> 32);
        const auto lo = halves ? __builtin_amdgcn_permlane32_swap(l, l, false, false)
                               : __builtin_amdgcn_permlane16_swap(l, l, false, false);
        const auto hi = halves ? __builtin_amdgcn_permlane32_swap(h, h, false, false)
                               : __builtin_amdgcn_permlane16_swap(h, h, false, false);
        x = __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) +
            __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
    }
    return x;
}

// fp32 values in the order of their numbers as unsigned ones, and back.
__device__ inline uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ inline float unordered(uint32_t u) {
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

inline bool aligned(const void* p, uintptr_t n) {
    return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

inline int launched(k3x_hip_ctx* ctx, unsigned n) {
    ctx->kernel_launches += n;
    return hipGetLastError() == hipSuccess ? K3X_OK : K3X_ERR_BACKEND_UNAVAILABLE;
}

}  // namespace k3x_ops
