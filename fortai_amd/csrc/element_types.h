// Element types of the serving operators (rotary positions, the 8-bit cache and
// its attention, draft verification): fp32, fp16 and bf16 arrays, computed on in
// fp32 and rounded once, to nearest even, when stored.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fortai_hip {

// FORTAI_HIP_DTYPE_* of the C ABI
enum class Dtype : int { F32 = 0, F16 = 1, BF16 = 2 };

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

template <Dtype DT> struct Element;
template <> struct Element<Dtype::F32> {
    typedef float type;
    typedef f32x4_t vec4;
};
template <> struct Element<Dtype::F16> {
    typedef _Float16 type;
    typedef f16x4_t vec4;
};
template <> struct Element<Dtype::BF16> {
    typedef __bf16 type;
    typedef bf16x4_t vec4;
};

// Four consecutive elements.  VEC: the address is aligned to all four.
template <Dtype DT, bool VEC>
__device__ __forceinline__ f32x4_t load4(const typename Element<DT>::type *p) {
    if constexpr (VEC) {
        const typename Element<DT>::vec4 v = *reinterpret_cast<const typename Element<DT>::vec4 *>(p);
        return f32x4_t{static_cast<float>(v[0]), static_cast<float>(v[1]), static_cast<float>(v[2]), static_cast<float>(v[3])};
    } else {
        return f32x4_t{static_cast<float>(p[0]), static_cast<float>(p[1]), static_cast<float>(p[2]), static_cast<float>(p[3])};
    }
}

template <Dtype DT, bool VEC>
__device__ __forceinline__ void store4(typename Element<DT>::type *p, f32x4_t v) {
    typedef typename Element<DT>::type E;
    if constexpr (VEC) {
        *reinterpret_cast<typename Element<DT>::vec4 *>(p) =
            typename Element<DT>::vec4{static_cast<E>(v[0]), static_cast<E>(v[1]), static_cast<E>(v[2]), static_cast<E>(v[3])};
    } else {
        p[0] = static_cast<E>(v[0]);
        p[1] = static_cast<E>(v[1]);
        p[2] = static_cast<E>(v[2]);
        p[3] = static_cast<E>(v[3]);
    }
}

// A workgroup barrier that orders LDS accesses only: loads from memory that are in
// flight stay so (__syncthreads waits for them).
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

}  // namespace fortai_hip
