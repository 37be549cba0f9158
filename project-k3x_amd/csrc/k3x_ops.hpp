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

// exp(x), x <= 0, in double: x = k ln2 + r, the series to r^13 on |r| <= ln2 / 2
// (expf_cr without its last rounding).  Minus infinity gives 0, NaN itself.
__device__ inline double exp_f64(double x) {
    if (x < -745.0) return 0.0;
    const double k = __builtin_rint(x * 1.4426950408889634);
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
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)k);
}

// A wave's LDS writes are seen by its other lanes, in order.
__device__ inline void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

inline bool aligned(const void* p, uintptr_t n) {
    return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

inline int launched(k3x_hip_ctx* ctx, unsigned n) {
    ctx->kernel_launches += n;
    return hipGetLastError() == hipSuccess ? K3X_OK : K3X_ERR_BACKEND_UNAVAILABLE;
}

}  // namespace k3x_ops
