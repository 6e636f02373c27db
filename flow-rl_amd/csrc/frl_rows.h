// Device helpers of the kernels that work on rows of logits (logits.hip, distill.hip): element types, vector access at any
// alignment, reductions over the group of threads that shares a row.  Not part of the public ABI.
#pragma once

#include "frl_device.h"

namespace frl {

void clear_kernels();      // capi.hip: frl_last_kernels starts anew

typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// gfx950 takes global vector accesses at any byte alignment (the runtime turns unaligned mode on), so odd vocabularies and
// odd row strides need no peeling; the copies below become one global_load / global_store each.
template <typename V>
__device__ __forceinline__ V ldu(const void* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}
template <typename V>
__device__ __forceinline__ void stu(void* p, V v) {
  __builtin_memcpy(p, &v, sizeof(V));
}

struct Bf16 { unsigned short u; };
struct F16 { unsigned short u; };

template <typename T> struct Elt;
template <> struct Elt<float> {
  static constexpr int id = FRL_ELT_F32;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
  static __device__ __forceinline__ f32x4 load4(const float* p) { return ldu<f32x4>(p); }
  static __device__ __forceinline__ void store4(float* p, f32x4 v) { stu(p, v); }
};
template <> struct Elt<Bf16> {
  static constexpr int id = FRL_ELT_BF16;
  static __device__ __forceinline__ float get(Bf16 v) { return __uint_as_float((unsigned)v.u << 16); }
  static __device__ __forceinline__ Bf16 put(float v) { return Bf16{__builtin_bit_cast(unsigned short, (__bf16)v)}; }
  static __device__ __forceinline__ f32x4 load4(const Bf16* p) {
    const u32x2 r = ldu<u32x2>(p);
    return f32x4{__uint_as_float(r[0] << 16), __uint_as_float(r[0] & 0xffff0000u), __uint_as_float(r[1] << 16), __uint_as_float(r[1] & 0xffff0000u)};
  }
  static __device__ __forceinline__ void store4(Bf16* p, f32x4 v) { stu(p, u16x4{put(v[0]).u, put(v[1]).u, put(v[2]).u, put(v[3]).u}); }
};
template <> struct Elt<F16> {
  static constexpr int id = FRL_ELT_F16;
  static __device__ __forceinline__ float get(F16 v) { return (float)__builtin_bit_cast(_Float16, v.u); }
  static __device__ __forceinline__ F16 put(float v) { return F16{__builtin_bit_cast(unsigned short, (_Float16)v)}; }
  static __device__ __forceinline__ f32x4 load4(const F16* p) {
    const u16x4 r = ldu<u16x4>(p);
    return f32x4{get(F16{r[0]}), get(F16{r[1]}), get(F16{r[2]}), get(F16{r[3]})};
  }
  static __device__ __forceinline__ void store4(F16* p, f32x4 v) { stu(p, u16x4{put(v[0]).u, put(v[1]).u, put(v[2]).u, put(v[3]).u}); }
};

__device__ __forceinline__ long long ld_id(const void* p, long long i, int ids64) {
  return ids64 ? ((const long long*)p)[i] : (long long)((const int*)p)[i];
}

// A group of G threads shares a row: one wave (four groups to a workgroup of 256) or a whole workgroup.  A wave's LDS
// accesses execute in order, so a one-wave group needs the compiler kept from reordering them and no barrier.
template <int G>
__device__ __forceinline__ void group_sync() {
  if constexpr (G == 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

__device__ __forceinline__ unsigned long long shfl_xor64(unsigned long long v, int off) {
  const unsigned lo = __shfl_xor((unsigned)v, off), hi = __shfl_xor((unsigned)(v >> 32), off);
  return ((unsigned long long)hi << 32) | lo;
}

struct MaxOp {
  static __device__ __forceinline__ float f(float a, float b) { return fmaxf(a, b); }
  static __device__ __forceinline__ unsigned long long f(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
};
struct SumOp {
  template <typename V>
  static __device__ __forceinline__ V f(V a, V b) { return a + b; }
};
__device__ __forceinline__ float shfl_x(float v, int off) { return __shfl_xor(v, off); }
__device__ __forceinline__ double shfl_x(double v, int off) { return __shfl_xor(v, off); }
__device__ __forceinline__ unsigned long long shfl_x(unsigned long long v, int off) { return shfl_xor64(v, off); }

template <typename Op, typename V>
__device__ __forceinline__ V wave_reduce(V v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = Op::f(v, shfl_x(v, off));
  return v;
}

// Every thread of the group gets the result; the order of the operations is fixed.  `red` holds one V per wave of the group
// and is free again after the next group_sync the caller makes (callers alternate between two arrays).
template <typename Op, int G, typename V>
__device__ __forceinline__ V group_reduce(V v, V* red) {
  v = wave_reduce<Op>(v);
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < G / 64; ++w) v = Op::f(v, red[w]);
  }
  return v;
}

}  // namespace frl
