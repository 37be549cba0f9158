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

inline bool aligned(const void* p, uintptr_t n) {
    return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

inline int launched(k3x_hip_ctx* ctx, unsigned n) {
    ctx->kernel_launches += n;
    return hipGetLastError() == hipSuccess ? K3X_OK : K3X_ERR_BACKEND_UNAVAILABLE;
}

}  // namespace k3x_ops
