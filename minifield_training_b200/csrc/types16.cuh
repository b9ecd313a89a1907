// The two 16-bit element types of the rotary and paged-cache kernels: packing,
// unpacking and the warp-level MMA, for bf16 and fp16 alike.
#pragma once

#include "common.cuh"

namespace mfb {

template <typename T>
struct Num16;

template <>
struct Num16<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack2(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_bf16(lo, hi); }
  static __device__ __forceinline__ void mma(float* d, const uint32_t* a, const uint32_t* b) {
    mma_bf16_16816(d, a, b);
  }
};

template <>
struct Num16<__half> {
  static __device__ __forceinline__ float2 unpack2(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float* d, const uint32_t* a, const uint32_t* b) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  }
};

template <typename T>
__device__ __forceinline__ void unpack16x8(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Num16<T>::unpack2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack16x8(const float* x) {
  return make_uint4(Num16<T>::pack2(x[0], x[1]), Num16<T>::pack2(x[2], x[3]), Num16<T>::pack2(x[4], x[5]),
                    Num16<T>::pack2(x[6], x[7]));
}

// Two FP32 lanes per instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Four 16-bit values as two FP32 pairs, and back.
template <typename T>
__device__ __forceinline__ void unpack16x4(const uint2& v, uint64_t* x) {
  const float2 a = Num16<T>::unpack2(v.x), b = Num16<T>::unpack2(v.y);
  x[0] = pair(a.x, a.y);
  x[1] = pair(b.x, b.y);
}
template <typename T>
__device__ __forceinline__ uint2 pack16x4(const uint64_t* x) {
  const float2 a = unpair(x[0]), b = unpair(x[1]);
  return make_uint2(Num16<T>::pack2(a.x, a.y), Num16<T>::pack2(b.x, b.y));
}

}  // namespace mfb
