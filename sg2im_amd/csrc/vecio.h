// 16-byte pieces of rows whose start has only the alignment of one element.  gfx950 runs with unaligned access on for
// global memory, so a dwordx4 load or store of a 2-byte aligned address is one instruction; odd widths then need no
// scalar path, only their last piece of a row does.
#pragma once
#include <hip/hip_runtime.h>

namespace sg2im {

typedef __bf16 bf16_s;

template <typename T> struct VecOf { static constexpr int n = 16 / sizeof(T); };

__device__ __forceinline__ float bf16_bits_to_f32(unsigned short b) { return __uint_as_float((unsigned)b << 16); }
// (round to nearest even; v_cvt_pk_bf16_f32)
__device__ __forceinline__ unsigned short f32_to_bf16_bits(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }

template <typename T> __device__ __forceinline__ float load1(const T* p);
template <> __device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float load1<bf16_s>(const bf16_s* p) {
  return bf16_bits_to_f32(*reinterpret_cast<const unsigned short*>(p));
}
template <typename T> __device__ __forceinline__ void store1(T* p, float v);
template <> __device__ __forceinline__ void store1<float>(float* p, float v) { *p = v; }
template <> __device__ __forceinline__ void store1<bf16_s>(bf16_s* p, float v) {
  *reinterpret_cast<unsigned short*>(p) = f32_to_bf16_bits(v);
}

// NV elements of T <-> registers, any element alignment
template <typename T, int NV> struct RawVec { unsigned short h[NV]; };
template <int NV> struct RawVec<float, NV> { float h[NV]; };

typedef unsigned u32x4_u __attribute__((ext_vector_type(4), aligned(1)));
typedef unsigned u32x2_u __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned u32_u __attribute__((aligned(1)));
template <int BYTES> __device__ __forceinline__ void store_bytes_nt(void* p, const void* from) {
  static_assert(BYTES == 16 || BYTES == 8 || BYTES == 4, "one store");
  if constexpr (BYTES == 16) { u32x4_u w; __builtin_memcpy(&w, from, 16); __builtin_nontemporal_store(w, reinterpret_cast<u32x4_u*>(p)); }
  else if constexpr (BYTES == 8) { u32x2_u w; __builtin_memcpy(&w, from, 8); __builtin_nontemporal_store(w, reinterpret_cast<u32x2_u*>(p)); }
  else { u32_u w; __builtin_memcpy(&w, from, 4); __builtin_nontemporal_store(w, reinterpret_cast<u32_u*>(p)); }
}
template <int BYTES> __device__ __forceinline__ void load_bytes_nt(void* to, const void* p) {
  static_assert(BYTES == 16 || BYTES == 8, "one load");
  if constexpr (BYTES == 16) { const u32x4_u w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_u*>(p)); __builtin_memcpy(to, &w, 16); }
  else { const u32x2_u w = __builtin_nontemporal_load(reinterpret_cast<const u32x2_u*>(p)); __builtin_memcpy(to, &w, 8); }
}

template <typename T, int NV> __device__ __forceinline__ RawVec<T, NV> load_raw(const T* p) {
  RawVec<T, NV> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <int NV> __device__ __forceinline__ void widen(const RawVec<float, NV>& r, float (&v)[NV]) {
  #pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = r.h[j];
}
template <int NV> __device__ __forceinline__ void widen(const RawVec<bf16_s, NV>& r, float (&v)[NV]) {
  #pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = bf16_bits_to_f32(r.h[j]);
}
template <typename T, int NV> __device__ __forceinline__ void load_vec(const T* p, float (&v)[NV]) {
  widen(load_raw<T, NV>(p), v);
}
template <typename T, int NV> __device__ __forceinline__ void store_vec(T* p, const float (&v)[NV]) {
  RawVec<T, NV> r;
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    if constexpr (sizeof(T) == 4) r.h[j] = v[j]; else r.h[j] = f32_to_bf16_bits(v[j]);
  }
  __builtin_memcpy(p, &r, sizeof(r));
}

// the same past the caches: for what is larger than they are, or not read again soon
template <typename T, int NV> __device__ __forceinline__ void store_vec_nt(T* p, const float (&v)[NV]) {
  RawVec<T, NV> r;
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    if constexpr (sizeof(T) == 4) r.h[j] = v[j]; else r.h[j] = f32_to_bf16_bits(v[j]);
  }
  store_bytes_nt<sizeof(r)>(p, &r);
}

// the parameters (affine, bias) are float32 or bfloat16: a wave-uniform choice
__device__ __forceinline__ float load_param(const void* p, int is_bf16, long long i) {
  return is_bf16 ? load1(reinterpret_cast<const bf16_s*>(p) + i) : reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_param(void* p, int is_bf16, long long i, float v, int accumulate) {
  if (is_bf16) {
    bf16_s* q = reinterpret_cast<bf16_s*>(p) + i;
    store1(q, accumulate ? load1(q) + v : v);
  } else {
    float* q = reinterpret_cast<float*>(p) + i;
    *q = accumulate ? *q + v : v;
  }
}

}  // namespace sg2im
