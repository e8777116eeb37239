// Loads and stores of VEC consecutive elements of a 32- or 16-bit type as fp32 values (one
// 16-byte access when VEC fills it), for the kernels whose tensors come in several types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace tsb {

// element types of the C ABI's `dtype` arguments
enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };
inline int dtype_size(int t) { return t == kF32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

template <int BYTES>
struct Bits;
template <>
struct Bits<2> { using type = uint16_t; };
template <>
struct Bits<4> { using type = uint32_t; };
template <>
struct Bits<8> { using type = uint2; };
template <>
struct Bits<16> { using type = uint4; };

__device__ __forceinline__ uint32_t word(uint16_t b, int) { return b; }
__device__ __forceinline__ uint32_t word(uint32_t b, int) { return b; }
__device__ __forceinline__ uint32_t word(uint2 b, int i) { return i == 0 ? b.x : b.y; }
__device__ __forceinline__ uint32_t word(uint4 b, int i) { return i == 0 ? b.x : (i == 1 ? b.y : (i == 2 ? b.z : b.w)); }

// VEC consecutive elements as they lie in memory, moved by one access of VEC * sizeof(T) = 2, 4, 8 or 16
// bytes (aligned to it).  What is fetched ahead stays in this form until it is used: elements of a 16-bit
// type held one by one would be taken apart, and so waited for, where they are loaded (backward norm of
// 6000 x 2048 in bf16: 102 us that way).
template <class T, int VEC>
struct Raw {
  typename Bits<sizeof(T) * VEC>::type b;
  __device__ __forceinline__ void load(const T* p) { b = *reinterpret_cast<const decltype(b)*>(p); }
  __device__ __forceinline__ float operator[](int i) const;
  // Elements [0, n) alone, word by word (n odd in a 16-bit type: the last is the low half of its word, so it too
  // lands in its register as it is); the rest keeps its bits.
  __device__ __forceinline__ void load_first(const T* p, int n) {
    constexpr int PER = 4 / sizeof(T), WORDS = VEC / PER;
    static_assert(WORDS >= 1, "whole words");
    uint32_t w[WORDS];
    memcpy(w, &b, sizeof(w));
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if ((i + 1) * PER <= n) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
      else if (i * PER < n) w[i] = *reinterpret_cast<const uint16_t*>(p + i * PER);
    }
    memcpy(&b, w, sizeof(w));
  }
  // the bits of the elements [from, to) set
  __device__ __forceinline__ void mask(int from, int to) {
    constexpr int PER = 4 / sizeof(T), WORDS = VEC / PER;
    uint32_t w[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (i * PER + e >= from && i * PER + e < to) w[i] |= (PER == 1 ? 0xffffffffu : 0xffffu) << (16 * e);
    }
    memcpy(&b, w, sizeof(w));
  }
  __device__ __forceinline__ Raw operator&(const Raw& m) const {
    constexpr int WORDS = VEC * sizeof(T) / 4;
    uint32_t x[WORDS], y[WORDS];
    memcpy(x, &b, sizeof(x));
    memcpy(y, &m.b, sizeof(y));
#pragma unroll
    for (int i = 0; i < WORDS; ++i) x[i] &= y[i];
    Raw r;
    memcpy(&r.b, x, sizeof(x));
    return r;
  }
};
template <int VEC>
__device__ __forceinline__ float raw_get(const Raw<float, VEC>& r, int i) { return __uint_as_float(word(r.b, i)); }
template <int VEC>
__device__ __forceinline__ float raw_get(const Raw<__nv_bfloat16, VEC>& r, int i) {
  const uint32_t w = word(r.b, i / 2);
  return __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
}
template <int VEC>
__device__ __forceinline__ float raw_get(const Raw<__half, VEC>& r, int i) {
  return __half2float(__ushort_as_half((unsigned short)(word(r.b, i / 2) >> (i % 2 * 16))));
}
template <class T, int VEC>
__device__ __forceinline__ float Raw<T, VEC>::operator[](int i) const { return raw_get(*this, i); }

// two values of a 16-bit type in a word
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// VEC values as one access's bits
template <class T, int VEC>
__device__ __forceinline__ typename Bits<sizeof(T) * VEC>::type bits_of(const float (&in)[VEC]) {
  typename Bits<sizeof(T) * VEC>::type b;
  if constexpr (sizeof(T) == 4) {
    memcpy(&b, in, sizeof(b));
  } else if constexpr (VEC == 1) {
    const T v = from_f32<T>(in[0]);
    memcpy(&b, &v, sizeof(b));
  } else {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = pack2<T>(in[2 * i], in[2 * i + 1]);
    memcpy(&b, w, sizeof(b));
  }
  return b;
}
template <class T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[VEC]) {
  Raw<T, VEC> r;
  r.load(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = r[i];
}

template <class T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[VEC]) {
  *reinterpret_cast<typename Bits<sizeof(T) * VEC>::type*>(p) = bits_of<T, VEC>(in);
}

}  // namespace tsb
