// Rows in chunks of eight entries: 16-byte loads and stores of each storage type, and its entries as floats.
#pragma once
#include "common.cuh"

namespace b200 {
namespace {

template <typename T> struct Chunk {
  static constexpr int kLoads = sizeof(T) / 2;
  uint4 raw[kLoads];
};
template <typename T> __device__ __forceinline__ float2 pair_f(uint32_t p);
template <> __device__ __forceinline__ float2 pair_f<__half>(uint32_t p) { return __half22float2(*reinterpret_cast<const __half2*>(&p)); }
template <> __device__ __forceinline__ float2 pair_f<__nv_bfloat16>(uint32_t p) {
  return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ Chunk<T> load8(const T* p) {
  Chunk<T> c;
#pragma unroll
  for (int i = 0; i < Chunk<T>::kLoads; ++i) c.raw[i] = reinterpret_cast<const uint4*>(p)[i];
  return c;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Chunk<T>& c) {
#pragma unroll
  for (int i = 0; i < Chunk<T>::kLoads; ++i) reinterpret_cast<uint4*>(p)[i] = c.raw[i];
}
template <typename T> __device__ __forceinline__ void unpack8(const Chunk<T>& c, float (&v)[8]) {
  const uint32_t w[4] = {c.raw[0].x, c.raw[0].y, c.raw[0].z, c.raw[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = pair_f<T>(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <> __device__ __forceinline__ void unpack8<float>(const Chunk<float>& c, float (&v)[8]) {
  const uint32_t w[8] = {c.raw[0].x, c.raw[0].y, c.raw[0].z, c.raw[0].w, c.raw[1].x, c.raw[1].y, c.raw[1].z, c.raw[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}

// Two floats as a pair of T, one rounding each; fp16 saturates to its largest finite value, NaN stays NaN.
template <typename T> __device__ __forceinline__ uint32_t two_of(float lo, float hi);
template <> __device__ __forceinline__ uint32_t two_of<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));  // first source -> upper half
  return r;
}
template <> __device__ __forceinline__ uint32_t two_of<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ T one_of(float v) {
  const uint32_t p = two_of<T>(v, 0.f);
  const unsigned short h = (unsigned short)p;
  return *reinterpret_cast<const T*>(&h);
}
template <> __device__ __forceinline__ float one_of<float>(float v) { return v; }
template <typename T> __device__ __forceinline__ Chunk<T> pack8(const float (&v)[8]) {
  Chunk<T> c;
  c.raw[0] = make_uint4(two_of<T>(v[0], v[1]), two_of<T>(v[2], v[3]), two_of<T>(v[4], v[5]), two_of<T>(v[6], v[7]));
  return c;
}
template <> __device__ __forceinline__ Chunk<float> pack8<float>(const float (&v)[8]) {
  Chunk<float> c;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    c.raw[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
  return c;
}

}  // namespace
}  // namespace b200
