// op_device.h -- element types, unaligned vector access and lane-group reductions shared by layer_norm.hip, embedding.hip,
// row_sort.hip, gate.hip and int8_product.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mnr_api.h"

namespace mnr {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

inline bool type_ok(int t) { return t == MNR_F32 || t == MNR_F16 || t == MNR_BF16; }

// One element of a vector of runtime type (norm weights, biases: read once per wave, so the switch costs nothing)
__device__ __forceinline__ float load_any(const void *p, int64_t i, int type) {
    if (type == MNR_F32) return reinterpret_cast<const float *>(p)[i];
    if (type == MNR_F16) return (float)reinterpret_cast<const f16_t *>(p)[i];
    return (float)reinterpret_cast<const bf16_t *>(p)[i];
}
__device__ __forceinline__ void store_any(void *p, int64_t i, float v, int type) {
    if (type == MNR_F32) reinterpret_cast<float *>(p)[i] = v;
    else if (type == MNR_F16) reinterpret_cast<f16_t *>(p)[i] = (f16_t)v;
    else reinterpret_cast<bf16_t *>(p)[i] = (bf16_t)v;
}

// 16 bytes of T, at any element's address: gfx950 takes global accesses of every alignment, so a row of odd width needs no scalar
// path (aligned(sizeof(T)) tells the compiler; it still emits one dwordx4 access).
template <class T> struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    typedef T raw __attribute__((ext_vector_type(N)));
    typedef raw type __attribute__((aligned(sizeof(T))));
};

// V elements from p, of which the first n exist (n <= 0: none); the rest become 0
template <class T>
__device__ __forceinline__ void load_part(float (&v)[Vec<T>::N], const T *p, int n) {
    if (n >= Vec<T>::N) {
        const typename Vec<T>::type x = *reinterpret_cast<const typename Vec<T>::type *>(p);
#pragma unroll
        for (int i = 0; i < Vec<T>::N; ++i) v[i] = (float)x[i];
    } else {
#pragma unroll
        for (int i = 0; i < Vec<T>::N; ++i) v[i] = i < n ? (float)p[i] : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store_part(T *p, const float (&v)[Vec<T>::N], int n) {
    if (n >= Vec<T>::N) {
        typename Vec<T>::type x;
#pragma unroll
        for (int i = 0; i < Vec<T>::N; ++i) x[i] = (T)v[i];
        *reinterpret_cast<typename Vec<T>::type *>(p) = x;
    } else {
#pragma unroll
        for (int i = 0; i < Vec<T>::N; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// load_part's 16 bytes as they are: four registers until they are needed
template <class T>
__device__ __forceinline__ typename Vec<T>::raw load_raw(const T *p, int n) {
    if (n >= Vec<T>::N) return *reinterpret_cast<const typename Vec<T>::type *>(p);
    typename Vec<T>::raw x;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) x[i] = i < n ? p[i] : (T)0.f;
    return x;
}

// V elements of a vector of runtime type from element i on, of which the first n exist; the rest become 0
template <int V>
__device__ __forceinline__ void load_any_part(float (&v)[V], const void *p, int64_t i, int n, int type) {
    if (type == MNR_F32) {
#pragma unroll
        for (int k = 0; k < V; k += 4) load_part<float>(reinterpret_cast<float (&)[4]>(v[k]), reinterpret_cast<const float *>(p) + i + k, n - k);
    } else if (n >= V) {
        if (type == MNR_F16) {
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = (float)reinterpret_cast<const f16_t *>(p)[i + k];
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = (float)reinterpret_cast<const bf16_t *>(p)[i + k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = k < n ? load_any(p, i + k, type) : 0.f;
    }
}

// orders LDS accesses between the lanes of one wave (its LDS operations run in order; this keeps the compiler's order too)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---- reductions over groups of LANES (power of two) consecutive lanes; every lane gets the result -------------------------------
// Steps 1, 2, 4, 8 are DPP moves inside a row of 16 lanes (quad permutes, half mirror, mirror: after each step the lanes of a
// sub-group agree, so a mirror is as good as an exchange); 16 and 32 are gfx950's permlane swaps.  No LDS traffic.
template <int CTRL> __device__ __forceinline__ uint32_t dpp_u32(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
}
template <int STEP> __device__ __forceinline__ uint32_t lane_other(uint32_t x) {
    if constexpr (STEP == 1) return dpp_u32<0xB1>(x);          // quad_perm [1,0,3,2]
    else if constexpr (STEP == 2) return dpp_u32<0x4E>(x);     // quad_perm [2,3,0,1]
    else if constexpr (STEP == 4) return dpp_u32<0x141>(x);    // row_half_mirror
    else return dpp_u32<0x140>(x);                             // row_mirror
}
// the two halves of step 16 / 32 as (lower lanes' value, upper lanes' value): the same pair on both sides, so sums round alike
template <int STEP> __device__ __forceinline__ void lane_halves(uint32_t x, uint32_t &lo, uint32_t &hi) {
    if constexpr (STEP == 16) {
        auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        lo = r[0]; hi = r[1];
    } else {
        auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        lo = r[0]; hi = r[1];
    }
}
template <int STEP, class F> __device__ __forceinline__ float lane_step(float x, F f) {
    if constexpr (STEP >= 16) {
        uint32_t lo, hi;
        lane_halves<STEP>(__float_as_uint(x), lo, hi);
        return f(__uint_as_float(lo), __uint_as_float(hi));
    } else {
        return f(x, __uint_as_float(lane_other<STEP>(__float_as_uint(x))));
    }
}
template <int LANES, class F> __device__ __forceinline__ float lane_reduce(float x, F f) {
    if constexpr (LANES >= 2) x = lane_step<1>(x, f);
    if constexpr (LANES >= 4) x = lane_step<2>(x, f);
    if constexpr (LANES >= 8) x = lane_step<4>(x, f);
    if constexpr (LANES >= 16) x = lane_step<8>(x, f);
    if constexpr (LANES >= 32) x = lane_step<16>(x, f);
    if constexpr (LANES >= 64) x = lane_step<32>(x, f);
    return x;
}
template <int LANES> __device__ __forceinline__ float lane_sum(float x) { return lane_reduce<LANES>(x, [](float a, float b) { return a + b; }); }
template <int LANES> __device__ __forceinline__ float lane_max(float x) { return lane_reduce<LANES>(x, [](float a, float b) { return fmaxf(a, b); }); }

}  // namespace mnr
