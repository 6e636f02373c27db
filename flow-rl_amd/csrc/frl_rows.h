// Device helpers of the kernels that work on rows of logits (logits.hip, distill.hip): element types, vector access at any
// alignment, reductions over the group of threads that shares a row.  Not part of the public ABI.
#pragma once

#include <type_traits>

#include "frl_device.h"

// No product is fused into a sum but where the code says so (also for what follows in the including file): results do not depend on
// which products the compiler fuses in which kernel.
#pragma clang fp contract(off)

namespace frl {

void clear_kernels();      // capi.hip: frl_last_kernels starts anew

typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// gfx950 takes global vector accesses at any byte alignment (the runtime turns unaligned mode on), so odd vocabularies and
// odd row strides are right without peeling (distill.hip peels for speed); the copies below become one global_load / global_store each.
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

// The same with the non-temporal hint, for what is read once or written once: it leaves the caches first, and what is read again stays
template <typename V>
__device__ __forceinline__ void stu_nt(void* p, V v) {
  typedef V VU __attribute__((aligned(2)));
  __builtin_nontemporal_store(v, (VU*)p);
}
template <typename V>
__device__ __forceinline__ V ldu_nt(const void* p) {
  typedef V VU __attribute__((aligned(2)));
  return __builtin_nontemporal_load((const VU*)p);
}

struct Bf16 { unsigned short u; };
struct F16 { unsigned short u; };

template <typename T> struct Elt;
template <> struct Elt<float> {
  static constexpr int id = FRL_ELT_F32;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
  static __device__ __forceinline__ f32x4 load4(const float* p) { return ldu<f32x4>(p); }
  static __device__ __forceinline__ void store4(float* p, f32x4 v) { stu_nt(p, v); }
};
template <> struct Elt<Bf16> {
  static constexpr int id = FRL_ELT_BF16;
  static __device__ __forceinline__ float get(Bf16 v) { return __uint_as_float((unsigned)v.u << 16); }
  static __device__ __forceinline__ Bf16 put(float v) { return Bf16{__builtin_bit_cast(unsigned short, (__bf16)v)}; }
  static __device__ __forceinline__ f32x4 load4(const Bf16* p) {
    const u32x2 r = ldu<u32x2>(p);
    return f32x4{__uint_as_float(r[0] << 16), __uint_as_float(r[0] & 0xffff0000u), __uint_as_float(r[1] << 16), __uint_as_float(r[1] & 0xffff0000u)};
  }
  static __device__ __forceinline__ void store4(Bf16* p, f32x4 v) { stu_nt(p, u16x4{put(v[0]).u, put(v[1]).u, put(v[2]).u, put(v[3]).u}); }
};
template <> struct Elt<F16> {
  static constexpr int id = FRL_ELT_F16;
  static __device__ __forceinline__ float get(F16 v) { return (float)__builtin_bit_cast(_Float16, v.u); }
  static __device__ __forceinline__ F16 put(float v) { return F16{__builtin_bit_cast(unsigned short, (_Float16)v)}; }
  static __device__ __forceinline__ f32x4 load4(const F16* p) {
    const u16x4 r = ldu<u16x4>(p);
    return f32x4{get(F16{r[0]}), get(F16{r[1]}), get(F16{r[2]}), get(F16{r[3]})};
  }
  static __device__ __forceinline__ void store4(F16* p, f32x4 v) { stu_nt(p, u16x4{put(v[0]).u, put(v[1]).u, put(v[2]).u, put(v[3]).u}); }
};

// 16 bytes of a row at a time: VEC elements, kept packed until they are used
template <typename T>
struct Vec16 {
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void unpack(u32x4 r, float* x) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
    } else if constexpr (Elt<T>::id == FRL_ELT_BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(r[i] << 16); x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u); }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = Elt<T>::get(T{(unsigned short)r[i]});
        x[2 * i + 1] = Elt<T>::get(T{(unsigned short)(r[i] >> 16)});
      }
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float* x) {
    u32x4 r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (Elt<T>::id == FRL_ELT_BF16) {
          typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
          r[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{x[2 * i], x[2 * i + 1]}, bf2));     // v_cvt_pk_bf16_f32
        } else {
          r[i] = (unsigned)Elt<T>::put(x[2 * i]).u | (unsigned)Elt<T>::put(x[2 * i + 1]).u << 16;
        }
      }
    }
    return r;
  }
  static __device__ __forceinline__ u32x4 fill_minus_inf() {
    const unsigned w = sizeof(T) == 4 ? 0xff800000u : Elt<T>::id == FRL_ELT_BF16 ? 0xff80ff80u : 0xfc00fc00u;
    return u32x4{w, w, w, w};
  }
};

__device__ __forceinline__ long long ld_id(const void* p, long long i, int ids64) {
  return ids64 ? ((const long long*)p)[i] : (long long)((const int*)p)[i];
}

// A group of G threads shares a row: 16 lanes or one wave (16 or four groups to a workgroup of 256), or a whole workgroup.  A wave's LDS
// accesses execute in order, so a group within one needs the compiler kept from reordering them and no barrier.
template <int G>
__device__ __forceinline__ void group_sync() {
  if constexpr (G <= 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

// The thread's number as a value of its own: what is derived from it, an index and an address per vector, is then computed where it is used and not
// kept in registers across the passes and rows.
__device__ __forceinline__ int fresh(int tid) {
  asm volatile("" : "+v"(tid));
  return tid;
}

// 2^(x c - R) about a reference R, m c or what stands for it.  Where |m c| is below LIMIT, R is the rounded product M and an exponential is one
// fma: M is off by at most 2^-9, every exponent of the sum is shifted alike, and whoever takes the sum's logarithm adds residue() back.  Beyond
// (masked rows of -1e9 or the type's lowest value, forced tokens, tiny temperatures) the rounding of M would be whole powers of two, or more than
// an exponential can hold from 2^31 on: there R is m c itself and the difference from m is taken first.
struct Shift {
  static constexpr float LIMIT = 65536.0f;
  float m, M, c;
  bool fast;
  __device__ __forceinline__ Shift(float m_, float c_) : m(m_), M(m_ * c_), c(c_) { fast = fabsf(M) < LIMIT; }
  // R - m c, exact but for the last rounding
  __device__ __forceinline__ float residue() const { return fabsf(M) < LIMIT ? -__builtin_fmaf(m, c, -M) : 0.0f; }
  // `fast` may be taken back (so that a wave branches as one): the difference's form has the same reference
  template <int N>
  __device__ __forceinline__ void exps(float* x) const {
    if (fast) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c, -M));
    } else {
      const float back = residue();
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i] - m, c, -back));
    }
  }
  // the factor that turns a sum about another, lower reference into one about this
  __device__ __forceinline__ float from(const Shift& o) const {
    return __builtin_amdgcn_exp2f(fast && o.fast ? o.M - M : __builtin_fmaf(o.m - m, c, o.residue() - residue()));
  }
  // the same for a sum about lower c itself
  __device__ __forceinline__ float from_exact(float lower) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(lower - m, c, -residue())); }
};

template <int N>
__device__ __forceinline__ float max_of(const float* x, float m) {
#pragma unroll
  for (int i = 0; i < N; i += 2) m = fmaxf(fmaxf(x[i], x[i + 1]), m);      // v_max3_f32
  return m;
}

// A grid of any number of workgroups: the second dimension takes over where the first times the workgroup would pass 2^32 threads.
inline dim3 grid_of(long long blocks) {
  const long long x = blocks < (1 << 20) ? blocks : (1 << 20);
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
__device__ __forceinline__ long long block_index() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }

// Whether rows of wa bytes, sa bytes apart from a on, share a byte with rows of wb bytes, sb apart from b on (a distance is no less than its rows).  Rows
// at one distance may lie between one another, as the column blocks of one buffer do; of different distances only ranges that do not meet are
// taken to be apart.
inline bool rows_overlap(uintptr_t a, long long wa, long long sa, uintptr_t b, long long wb, long long sb, long long rows) {
  if (a >= b + (uintptr_t)((rows - 1) * sb + wb) || b >= a + (uintptr_t)((rows - 1) * sa + wa)) return false;
  if (rows == 1 || sa != sb) return true;
  const long long apart = (long long)(b - a) % sa, d = apart < 0 ? apart + sa : apart;      // where a row of b begins behind the last row of a
  return d < wa || d + wb > sa;
}

struct MaxOp {
  static __device__ __forceinline__ float f(float a, float b) { return fmaxf(a, b); }
  static __device__ __forceinline__ unsigned long long f(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
};
struct SumOp {
  template <typename V>
  static __device__ __forceinline__ V f(V a, V b) { return a + b; }
};
// v from another lane of the same row of 16 lanes, by the data-parallel-primitive control CTRL (no LDS traffic)
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
template <int CTRL>
__device__ __forceinline__ float dpp(float v) { return __uint_as_float(dpp<CTRL>(__float_as_uint(v))); }
template <int CTRL>
__device__ __forceinline__ unsigned long long dpp(unsigned long long v) {
  return ((unsigned long long)dpp<CTRL>((unsigned)(v >> 32)) << 32) | dpp<CTRL>((unsigned)v);
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) { return __builtin_bit_cast(double, dpp<CTRL>(__builtin_bit_cast(unsigned long long, v))); }

__device__ __forceinline__ unsigned lane_of(unsigned v, int l) { return (unsigned)__builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ float lane_of(float v, int l) { return __uint_as_float(lane_of(__float_as_uint(v), l)); }
__device__ __forceinline__ unsigned long long lane_of(unsigned long long v, int l) {
  return ((unsigned long long)lane_of((unsigned)(v >> 32), l) << 32) | lane_of((unsigned)v, l);
}
__device__ __forceinline__ double lane_of(double v, int l) { return __builtin_bit_cast(double, lane_of(__builtin_bit_cast(unsigned long long, v), l)); }

// Over W lanes, all of which have to be active: neighbours, quads and halves of a row of 16 by DPP, then the four rows by lane reads.
// Every lane gets the result; the order of the operations is fixed.
template <typename Op, int W, typename V>
__device__ __forceinline__ V lanes_reduce(V v) {
  static_assert(W == 16 || W == 64, "a row of lanes or a wave");
  v = Op::f(v, dpp<0xB1>(v));      // quad_perm 1 0 3 2
  v = Op::f(v, dpp<0x4E>(v));      // quad_perm 2 3 0 1
  v = Op::f(v, dpp<0x141>(v));     // row_half_mirror: the other quad of eight
  v = Op::f(v, dpp<0x140>(v));     // row_mirror: the other eight of the row
  if constexpr (W == 16) return v;
  else return Op::f(Op::f(lane_of(v, 0), lane_of(v, 16)), Op::f(lane_of(v, 32), lane_of(v, 48)));
}
template <typename Op, typename V>
__device__ __forceinline__ V wave_reduce(V v) { return lanes_reduce<Op, 64>(v); }

// Every thread of the group gets the result; the order of the operations is fixed.  `red` holds one V per wave of the group
// and is free again after the next group_sync the caller makes (callers alternate between two arrays).
template <typename Op, int G, typename V>
__device__ __forceinline__ V group_reduce(V v, V* red) {
  v = lanes_reduce<Op, G < 64 ? G : 64>(v);
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
