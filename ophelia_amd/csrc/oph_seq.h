// libophelia_seq.so -- what its sources share: element types, vector access, matrix-instruction fragments, error text.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#pragma GCC visibility push(default)      // the library is built with -fvisibility=hidden: only the C ABI is exported
#include "../../include/ophelia_seq.h"
#pragma GCC visibility pop

#pragma GCC visibility push(hidden)
namespace ophseq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16_t;
typedef _Float16 f16_t;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// Elements of a 16-byte piece, and the operand of the 32x32 matrix instruction: 8 elements of the contracted axis per lane, lanes
// 0..31 the first 8 of 16, lanes 32..63 the others.  fp32 has no such instruction: eight 32x32x2 steps contract element j of both
// halves each, so that the same 16 elements meet and the layout of operand and result is that of the 16-bit types.
template <class T> struct El;
template <> struct El<float> {
    static constexpr int PER16 = 4;
    typedef f32x8 frag;
    static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, f32x16 c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};
template <> struct El<bf16_t> {
    static constexpr int PER16 = 8;
    typedef bf16_t frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct El<f16_t> {
    static constexpr int PER16 = 8;
    typedef f16_t frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <class T> using frag_t = typename El<T>::frag;

// 16 bytes at an address that is only aligned to the element: global memory takes it as one dwordx4 load or store all the same
struct __attribute__((packed, aligned(2))) Any16 { uint32_t w[4]; };
__device__ __forceinline__ u32x4 load16(const void* p) {
    const Any16 v = *(const Any16*)p;
    return u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
}
__device__ __forceinline__ void store16(void* p, u32x4 v) { *(Any16*)p = Any16{{v[0], v[1], v[2], v[3]}}; }

template <class T> __device__ __forceinline__ frag_t<T> bits_to_frag(u32x4 lo, u32x4 hi);
template <> __device__ __forceinline__ f32x8 bits_to_frag<float>(u32x4 lo, u32x4 hi) {
    const f32x4 a = __builtin_bit_cast(f32x4, lo), b = __builtin_bit_cast(f32x4, hi);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <> __device__ __forceinline__ frag_t<bf16_t> bits_to_frag<bf16_t>(u32x4 lo, u32x4) { return __builtin_bit_cast(frag_t<bf16_t>, lo); }
template <> __device__ __forceinline__ frag_t<f16_t> bits_to_frag<f16_t>(u32x4 lo, u32x4) { return __builtin_bit_cast(frag_t<f16_t>, lo); }

// four consecutive results to memory, rounded to nearest even
template <class T> __device__ __forceinline__ void store4(T* p, f32x4 v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    struct __attribute__((packed, aligned(2))) Any { t4 v; };
    ((Any*)p)->v = __builtin_convertvector(v, t4);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// ---- host side ---------------------------------------------------------------------------------------------------------------
int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int device_fail(hipError_t e, const char* what);
int type_bytes(int dtype);        // 0: not a type

// makes `device` current for the life of the object
struct OnDevice {
    int before = -1, status = 0;
    explicit OnDevice(int device);
    ~OnDevice();
};

template <class P> int launch(void (*kernel)(P), dim3 grid, int threads, const P& p, size_t lds, void* stream) {
    P arg = p;
    void* args[] = {&arg};
    const hipError_t e = hipLaunchKernel((const void*)kernel, grid, dim3((unsigned)threads), args, lds, (hipStream_t)stream);
    return e == hipSuccess ? 0 : device_fail(e, "kernel launch");
}

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace ophseq
#pragma GCC visibility pop
