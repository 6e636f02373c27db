// KL divergence of a student's softmax from a teacher's top entries, and its gradient: frl_distill_fwd / frl_distill_bwd.
//
// Mathematics (include/flowrl_hip.h).  With c = log2(e) / T, a row needs m = max z, s = sum 2^((z - m) c) and, where the
// teacher's unnamed mass is a class of its own, r = the same sum without the named entries.  Then q = 2^((z - m) c) / s and
//     L      = sum p (log p - z / T) + sum p * (m / T + log s)   [+ P (log P - log (r / s))]
//     dL/dz  = (q - p) / T        named entries   (FRL_DISTILL_TOP: sum p = 1)
//     dL/dz  = k q / T            the others, k = 1 (FRL_DISTILL_TOP) or 1 - P s / r (FRL_DISTILL_REST with P > 0)
// The gradient is therefore one scaled exponential per element plus a correction of `top` elements.
//
// HBM-bound for long rows: the logits once, the gradient once.  A group of threads (a wave or a workgroup) takes a whole row:
// maximum and sum in one pass, the teacher's entries beside it, then the gradient in a second pass whose reads come from the cache.
// Few rows are split over their length, joined by a second kernel, and differentiated by a third.
#include "frl_rows.h"

// The value-and-gradient kernels and the backward kernel share the code below and agree bit for bit: no product is fused into a sum
// in one of them and not in the other.
#pragma clang fp contract(off)

namespace frl {

struct DistillArgs {
  const void* logits; const void* ids; const void* teacher; const float* weights;
  float* rowloss;             // (rows,) weight * L
  float* stats;               // (rows + 1, 4) or NULL: m, 1 / s, factor of the named entries, factor of the others; last row: 1 / denominator
  const float* inv_denom;     // device 1 / sum of weights, or NULL: `denom_scale`
  const float* g_loss;        // backward: cotangent, `g_stride` apart per row (0: one scalar); NULL: 1
  void* grad;
  float* part;                // split rows: (rows, segs, 3) m, s, r
  long long rows, logits_stride, grad_stride, ids_stride, teacher_stride;
  float inv_temp, scale2, denom_scale;   // 1 / T, log2(e) / T
  int vocab, top, ids64, teacher_dtype, segs, seg_len, g_stride;
};

constexpr int DSEG_MAX = 1 << 18;      // entries whose named bits one workgroup keeps in LDS (32 KB)

template <typename T>
__device__ __forceinline__ f32x4 quad(const T* p, int left) {
  if (left >= 4) return Elt<T>::load4(p);
  f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if (left > 0) v[0] = Elt<T>::get(p[0]);
  if (left > 1) v[1] = Elt<T>::get(p[1]);
  if (left > 2) v[2] = Elt<T>::get(p[2]);
  return v;
}

__device__ __forceinline__ float teacher_at(const void* p, long long i, int dtype) {
  if (dtype == FRL_ELT_F32) return ((const float*)p)[i];
  if (dtype == FRL_ELT_BF16) return Elt<Bf16>::get(((const Bf16*)p)[i]);
  return Elt<F16>::get(((const F16*)p)[i]);
}

// the named tokens of [v0, v0 + n) as bits; `words` covers n rounded up to 32
template <int G>
__device__ __forceinline__ void mark_named(const DistillArgs& a, long long row, int tid, int v0, int n, unsigned* words) {
  for (int w = tid; w < (n + 31) / 32; w += G) words[w] = 0u;
  group_sync<G>();
  for (int k = tid; k < a.top; k += G) {
    const long long loc = ld_id(a.ids, row * a.ids_stride + k, a.ids64) - v0;
    if (loc >= 0 && loc < n) atomicOr(&words[loc >> 5], 1u << (loc & 31));
  }
  group_sync<G>();
}

// m, s, r of entries [v0, v0 + n) of a row over the group's threads.  Each thread keeps its own running maximum and rescales
// its sums when a batch of 16 entries raises it.
template <typename T, int G, bool REST>
__device__ __forceinline__ void row_sums(const T* z, int n, float c, const unsigned* words, int tid, float* red0, float* red1, float& m, float& s, float& r) {
  constexpr int U = 4;
  float mt = -INFINITY, st = 0.0f, rt = 0.0f;
  for (int v = 4 * tid; v < n; v += 4 * U * G) {
    f32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = v + 4 * G * u;
      x[u] = quad(z + at, n - at);
    }
    float bm = mt;
#pragma unroll
    for (int u = 0; u < U; ++u) bm = fmaxf(bm, fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3])));
    const float m0 = bm == -INFINITY ? 0.0f : bm;
    const float f = __builtin_amdgcn_exp2f((mt - m0) * c);
    st *= f;
    rt *= f;
    mt = bm;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = v + 4 * G * u;
      unsigned named = 0;
      if (REST && at < n) named = words[at >> 5] >> (at & 31);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f((x[u][i] - m0) * c);
        st += e;
        if (REST) rt += (named >> i & 1u) ? 0.0f : e;
      }
    }
  }
  m = group_reduce<MaxOp, G>(mt, red0);
  const float f = __builtin_amdgcn_exp2f((mt - (m == -INFINITY ? 0.0f : m)) * c);
  s = group_reduce<SumOp, G>(st * f, red1);
  r = 0.0f;
  if constexpr (REST) {                                      // red0 is free: every thread has read it before the barrier in the sum
    r = group_reduce<SumOp, G>(rt * f, red0);
  }
}

// What one wave makes of a row's teacher entries: p (into sp, 0 for padding), the tokens (into sid, -1 for padding), sum p and
// sum p (log p - z / T).  FRL_DISTILL_REST needs 1 - sum p, which float32 exponentials would leave without digits: float64.
template <typename T, bool REST>
__device__ __forceinline__ void teacher_part(const DistillArgs& a, long long row, const T* z, int lane, int* sid, float* sp, double& sum_p, double& cross) {
  sum_p = cross = 0.0;
  float tm = -INFINITY, tot = 0.0f;
  if constexpr (!REST) {
    for (int k = lane; k < a.top; k += 64) {
      const long long id = ld_id(a.ids, row * a.ids_stride + k, a.ids64);
      if (id >= 0 && id < a.vocab) tm = fmaxf(tm, teacher_at(a.teacher, row * a.teacher_stride + k, a.teacher_dtype));
    }
    tm = wave_reduce<MaxOp>(tm);
    const float t0 = tm == -INFINITY ? 0.0f : tm;
    for (int k = lane; k < a.top; k += 64) {
      const long long id = ld_id(a.ids, row * a.ids_stride + k, a.ids64);
      if (id >= 0 && id < a.vocab) tot += expf((teacher_at(a.teacher, row * a.teacher_stride + k, a.teacher_dtype) - t0) * a.inv_temp);
    }
    tot = wave_reduce<SumOp>(tot);
  }
  const float log_tot = REST ? 0.0f : logf(tot);
  for (int k = lane; k < a.top; k += 64) {
    const long long id = ld_id(a.ids, row * a.ids_stride + k, a.ids64);
    const bool valid = id >= 0 && id < a.vocab;
    float p = 0.0f;
    if (valid) {
      const float t = teacher_at(a.teacher, row * a.teacher_stride + k, a.teacher_dtype);
      const float y = Elt<T>::get(z[id]) * a.inv_temp;
      float lp;
      if constexpr (REST) {
        const double pd = exp((double)t);
        p = (float)pd;
        lp = t;
        sum_p += pd;
      } else {
        const float d = (t - tm) * a.inv_temp;
        p = expf(d) / tot;
        lp = d - log_tot;
        sum_p += (double)p;
      }
      if (p != 0.0f) cross += (double)p * ((double)lp - (double)y);
    }
    sid[k] = valid ? (int)id : -1;
    sp[k] = p;
  }
  sum_p = wave_reduce<SumOp>(sum_p);
  cross = wave_reduce<SumOp>(cross);
}

struct RowResult { float loss, inv_s, k_named, k_rest; };

template <bool REST>
__device__ __forceinline__ RowResult row_result(const DistillArgs& a, float m, float s, float r, double sum_p, double cross) {
  RowResult o;
  o.inv_s = 1.0f / s;
  double loss = cross + sum_p * ((double)m * (double)a.inv_temp + (double)logf(s));
  o.k_named = o.k_rest = (float)sum_p;
  if constexpr (REST) {
    const double P = 1.0 - sum_p;
    if (P > 0.0) {
      loss += P * (log(P) - (double)(logf(r) - logf(s)));
      o.k_named = 1.0f;
      o.k_rest = 1.0f - (float)P * s / r;
    }
  } else {
    // softmax over the named entries sums to one; a row that names nothing has neither loss nor gradient
    o.k_named = o.k_rest = sum_p != 0.0 ? 1.0f : 0.0f;
    if (sum_p != sum_p) o.k_named = o.k_rest = (float)sum_p;
    else if (sum_p == 0.0) loss = 0.0;
  }
  o.loss = (float)loss;
  return o;
}

template <typename T, int G>
__device__ __forceinline__ void zero_row(T* g, int n, int tid) {
  for (int v = 4 * tid; v < n; v += 4 * G) {
    if (n - v >= 4) Elt<T>::store4(g + v, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
    else for (int i = 0; i < n - v; ++i) g[v + i] = Elt<T>::put(0.0f);
  }
}

// Gradient of entries [v0, v0 + n): the scaled exponential everywhere, then the named entries over it.  Both are plain stores of one
// workgroup with a barrier between them, so the second is what stays.
template <typename T, int G>
__device__ __forceinline__ void row_gradient(const DistillArgs& a, const T* z, T* g, int v0, int n, float m, float inv_s, float k_named, float k_rest,
                                             float f, const int* sid, const float* sp, int tid) {
  constexpr int U = 4;
  if (k_named == 0.0f && k_rest == 0.0f) {                   // the row names nothing: no gradient, whatever stands in the logits
    zero_row<T, G>(g + v0, n, tid);
    return;
  }
  const float c = a.scale2, f_rest = f * k_rest * inv_s, f_named = f * k_named * inv_s;
  for (int v = 4 * tid; v < n; v += 4 * U * G) {
    f32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = v + 4 * G * u;
      x[u] = quad(z + v0 + at, n - at);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = v + 4 * G * u, left = n - at;
      f32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = f_rest * __builtin_amdgcn_exp2f((x[u][i] - m) * c);
      T* to = g + v0 + at;
      if (left >= 4) Elt<T>::store4(to, o);
      else {
        if (left > 0) to[0] = Elt<T>::put(o[0]);
        if (left > 1) to[1] = Elt<T>::put(o[1]);
        if (left > 2) to[2] = Elt<T>::put(o[2]);
      }
    }
  }
  group_sync<G>();
  for (int k = tid; k < a.top; k += G) {
    const int id = sid[k];
    if (id < v0 || id >= v0 + n) continue;
    float p = 0.0f;
    bool first = true;
    for (int j = 0; j < a.top; ++j)
      if (sid[j] == id) { p += sp[j]; first = first && j >= k; }
    if (first) g[id] = Elt<T>::put(f_named * __builtin_amdgcn_exp2f((Elt<T>::get(z[id]) - m) * c) - f * p);
  }
}

// A row to a group: value, what the backward needs, and (GRAD) the gradient.
template <typename T, int G, bool REST, bool GRAD>
__global__ void __launch_bounds__(G == 64 ? 256 : G) frl_distill_row_kernel(const DistillArgs a) {
  extern __shared__ __align__(16) unsigned lds[];
  constexpr int GPB = G == 64 ? 4 : 1;
  __shared__ float red0[G / 64], red1[G / 64];
  __shared__ double row_p[GPB], row_x[GPB];
  const int tid = threadIdx.x % G, grp = threadIdx.x / G;
  const int nwords = REST ? (a.vocab + 31) / 32 : 0;
  unsigned* words = lds + (size_t)grp * (nwords + 2 * a.top);
  int* sid = (int*)(words + nwords);
  float* sp = (float*)(sid + a.top);
  const float inv = a.inv_denom != nullptr ? *a.inv_denom : a.denom_scale;
  for (long long row = (long long)blockIdx.x * GPB + grp; row < a.rows; row += (long long)gridDim.x * GPB) {
    const T* z = (const T*)a.logits + row * a.logits_stride;
    T* g = GRAD ? (T*)a.grad + row * a.grad_stride : nullptr;
    const float w = a.weights != nullptr ? a.weights[row] : 1.0f;
    if (w == 0.0f) {                                       // uniform over the group
      if (tid == 0) {
        a.rowloss[row] = 0.0f;
        if (a.stats != nullptr) *(f32x4*)(a.stats + 4 * row) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
      if constexpr (GRAD) zero_row<T, G>(g, a.vocab, tid);
      continue;
    }
    if constexpr (REST) mark_named<G>(a, row, tid, 0, a.vocab, words);
    if (tid < 64) {
      double sum_p, cross;
      teacher_part<T, REST>(a, row, z, tid, sid, sp, sum_p, cross);
      if (tid == 0) { row_p[grp] = sum_p; row_x[grp] = cross; }
    }
    float m, s, r;
    row_sums<T, G, REST>(z, a.vocab, a.scale2, words, tid, red0, red1, m, s, r);
    group_sync<G>();                                       // the teacher's part is visible (and red1 free)
    const RowResult o = row_result<REST>(a, m, s, r, row_p[grp], row_x[grp]);
    if (tid == 0) {
      a.rowloss[row] = w * o.loss;
      if (a.stats != nullptr) *(f32x4*)(a.stats + 4 * row) = f32x4{m, o.inv_s, o.k_named, o.k_rest};
    }
    if constexpr (GRAD) row_gradient<T, G>(a, z, g, 0, a.vocab, m, o.inv_s, o.k_named, o.k_rest, w * inv * a.inv_temp, sid, sp, tid);
    group_sync<G>();                                       // the next row writes the shared arrays again
  }
}

// ---- rows split over their length ---------------------------------------------------------------------------------------

template <typename T, int G, bool REST>
__global__ void __launch_bounds__(G) frl_distill_part_kernel(const DistillArgs a) {
  extern __shared__ __align__(16) unsigned lds[];
  __shared__ float red0[G / 64], red1[G / 64];
  const long long row = blockIdx.x / a.segs;
  const int seg = blockIdx.x % a.segs, v0 = seg * a.seg_len, n = min(a.vocab - v0, a.seg_len);
  if (a.weights != nullptr && a.weights[row] == 0.0f) return;
  if constexpr (REST) mark_named<G>(a, row, threadIdx.x, v0, n, lds);
  float m, s, r;
  row_sums<T, G, REST>((const T*)a.logits + row * a.logits_stride + v0, n, a.scale2, lds, threadIdx.x, red0, red1, m, s, r);
  if (threadIdx.x == 0) {
    float* p = a.part + 3 * (row * a.segs + seg);
    p[0] = m; p[1] = s; p[2] = r;
  }
}

// one wave per row: the segments joined in order, then the teacher's entries
template <typename T, bool REST>
__global__ void __launch_bounds__(64) frl_distill_join_kernel(const DistillArgs a) {
  extern __shared__ __align__(16) unsigned lds[];
  int* sid = (int*)lds;
  float* sp = (float*)(sid + a.top);
  const long long row = blockIdx.x;
  const int lane = threadIdx.x;
  const float w = a.weights != nullptr ? a.weights[row] : 1.0f;
  if (w == 0.0f) {
    if (lane == 0) {
      a.rowloss[row] = 0.0f;
      if (a.stats != nullptr) *(f32x4*)(a.stats + 4 * row) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    return;
  }
  double sum_p, cross;
  teacher_part<T, REST>(a, row, (const T*)a.logits + row * a.logits_stride, lane, sid, sp, sum_p, cross);
  float m = -INFINITY, s = 0.0f, r = 0.0f;
  const float* p = a.part + 3 * row * a.segs;
  for (int i = lane; i < a.segs; i += 64) m = fmaxf(m, p[3 * i]);
  m = wave_reduce<MaxOp>(m);
  const float m0 = m == -INFINITY ? 0.0f : m;
  for (int i = lane; i < a.segs; i += 64) {
    const float f = __builtin_amdgcn_exp2f((p[3 * i] - m0) * a.scale2);
    s += p[3 * i + 1] * f;
    r += p[3 * i + 2] * f;
  }
  s = wave_reduce<SumOp>(s);
  r = wave_reduce<SumOp>(r);
  const RowResult o = row_result<REST>(a, m, s, r, sum_p, cross);
  if (lane == 0) {
    a.rowloss[row] = w * o.loss;
    if (a.stats != nullptr) *(f32x4*)(a.stats + 4 * row) = f32x4{m, o.inv_s, o.k_named, o.k_rest};
  }
}

// gradient of one segment of a row from the row's statistics
template <typename T, int G, bool REST>
__global__ void __launch_bounds__(G == 64 ? 256 : G) frl_distill_grad_kernel(const DistillArgs a) {
  extern __shared__ __align__(16) unsigned lds[];
  constexpr int GPB = G == 64 ? 4 : 1;
  const int tid = threadIdx.x % G, grp = threadIdx.x / G;
  int* sid = (int*)lds + (size_t)grp * 2 * a.top;
  float* sp = (float*)(sid + a.top);
  const float inv = a.inv_denom != nullptr ? *a.inv_denom : a.denom_scale;
  const long long items = a.rows * a.segs;
  for (long long item = (long long)blockIdx.x * GPB + grp; item < items; item += (long long)gridDim.x * GPB) {
    const long long row = item / a.segs;
    const int v0 = (int)(item - row * a.segs) * a.seg_len, n = min(a.vocab - v0, a.seg_len);
    const T* z = (const T*)a.logits + row * a.logits_stride;
    T* g = (T*)a.grad + row * a.grad_stride;
    const float w = a.weights != nullptr ? a.weights[row] : 1.0f;
    if (w == 0.0f) {
      zero_row<T, G>(g + v0, n, tid);
      continue;
    }
    if (tid < 64) {
      double sum_p, cross;
      teacher_part<T, REST>(a, row, z, tid, sid, sp, sum_p, cross);
    }
    const f32x4 st = *(const f32x4*)(a.stats + 4 * row);
    const float cot = a.g_loss != nullptr ? a.g_loss[row * a.g_stride] : 1.0f;
    group_sync<G>();
    row_gradient<T, G>(a, z, g, v0, n, st[0], st[1], st[2], st[3], cot * w * inv * a.inv_temp, sid, sp, tid);
    group_sync<G>();
  }
}

// ---- over the rows ------------------------------------------------------------------------------------------------------

__device__ __forceinline__ double block_sum(double v, double* red) {
  v = wave_reduce<SumOp>(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v += red[w];
  __syncthreads();
  return v;
}

// 1 / sum of the weights (0 where the sum is 0), or 1 / rows
__global__ void __launch_bounds__(1024) frl_distill_denom_kernel(const float* __restrict__ w, long long rows, float* __restrict__ inv) {
  __shared__ double red[16];
  double s = 0.0;
  for (long long i = threadIdx.x; i < rows; i += 1024) s += (double)w[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) *inv = s != 0.0 ? (float)(1.0 / s) : 0.0f;
}

__global__ void __launch_bounds__(1024) frl_distill_sum_kernel(const float* __restrict__ rowloss, long long rows, const float* __restrict__ inv, float scale,
                                                               float* __restrict__ loss) {
  __shared__ double red[16];
  double s = 0.0;
  for (long long i = threadIdx.x; i < rows; i += 1024) s += (double)rowloss[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) *loss = (float)(s * (double)(inv != nullptr ? *inv : scale));
}

// ---- host ---------------------------------------------------------------------------------------------------------------

struct DistillPlan { int G, segs, seg_len; };

static DistillPlan distill_plan(long long rows, int vocab) {
  DistillPlan p;
  p.G = vocab <= 1024 ? 64 : vocab <= 8192 ? 256 : 1024;
  p.segs = 1;
  p.seg_len = vocab;
  if (p.G == 1024 && rows > 0 && (rows < 256 || vocab > DSEG_MAX)) {
    // enough segments for two workgroups per CU, of at least 4096 entries
    long long want = (512 + rows - 1) / rows;
    const long long most = (vocab + 4095) / 4096, least = ((long long)vocab + DSEG_MAX - 1) / DSEG_MAX;
    if (want > most) want = most;
    if (want < least) want = least;
    p.seg_len = (int)(((vocab + want - 1) / want + 31) / 32 * 32);
    p.segs = (vocab + p.seg_len - 1) / p.seg_len;
    if (p.segs > 1) p.G = 256;
  }
  return p;
}

static int distill_validate(const FrlDistillDesc* d) {
  if (d == nullptr) { set_error("distill: desc is NULL"); return FRL_EINVAL; }
  if (d->abi_version != FRL_ABI_VERSION) { set_error("desc.abi_version %d != library %d", d->abi_version, FRL_ABI_VERSION); return FRL_EINVAL; }
  if (d->dtype < FRL_ELT_F32 || d->dtype > FRL_ELT_F16) { set_error("distill: dtype %d invalid", d->dtype); return FRL_EINVAL; }
  if (d->teacher_dtype < FRL_ELT_F32 || d->teacher_dtype > FRL_ELT_F16) { set_error("distill: teacher_dtype %d invalid", d->teacher_dtype); return FRL_EINVAL; }
  if (d->kind < FRL_DISTILL_TOP || d->kind > FRL_DISTILL_REST) { set_error("distill: kind %d invalid", d->kind); return FRL_EINVAL; }
  if (d->reduction < FRL_REDUCE_NONE || d->reduction > FRL_REDUCE_MEAN) { set_error("distill: reduction %d invalid", d->reduction); return FRL_EINVAL; }
  if (d->rows < 0 || d->vocab < 1 || d->top < 1) { set_error("distill: rows %lld / vocab %d / top %d invalid", (long long)d->rows, d->vocab, d->top); return FRL_EINVAL; }
  if (!(d->temperature > 0.0f)) { set_error("distill: temperature %g must be > 0", d->temperature); return FRL_EINVAL; }
  if (d->top > FRL_DISTILL_MAX_TOP) { set_error("distill: top %d > %d", d->top, FRL_DISTILL_MAX_TOP); return FRL_EUNSUPPORTED; }
  if (d->vocab > (1 << 30)) { set_error("distill: vocab %d > 2^30", d->vocab); return FRL_EUNSUPPORTED; }
  if (d->rows > (1LL << 30)) { set_error("distill: %lld rows > 2^30", (long long)d->rows); return FRL_EUNSUPPORTED; }
  const DistillPlan p = distill_plan(d->rows, d->vocab);
  if (p.segs > 1 && d->rows * p.segs > (1LL << 22)) { set_error("distill: %lld rows of %d entries are more than 2^22 segments in one call", (long long)d->rows, d->vocab); return FRL_EUNSUPPORTED; }
  if (d->rows > 1 && d->logits_stride < d->vocab) { set_error("distill: row stride %lld < vocab %d", (long long)d->logits_stride, d->vocab); return FRL_EINVAL; }
  return FRL_OK;
}

static bool distill_overlap(const FrlDistillDesc* d, const FrlDistillBufs* b) {
  const size_t elt = d->dtype == FRL_ELT_F32 ? 4 : 2;
  const uintptr_t i0 = (uintptr_t)b->logits, i1 = i0 + ((size_t)(d->rows - 1) * d->logits_stride + d->vocab) * elt;
  const uintptr_t o0 = (uintptr_t)b->grad, o1 = o0 + ((size_t)(d->rows - 1) * d->grad_stride + d->vocab) * elt;
  return i0 < o1 && o0 < i1;
}

static DistillArgs distill_args(const FrlDistillDesc* d, const FrlDistillBufs* b, const DistillPlan& p) {
  DistillArgs a = {};
  a.logits = b->logits; a.ids = b->ids; a.teacher = b->teacher; a.weights = b->weights; a.grad = b->grad;
  a.rows = d->rows; a.logits_stride = d->logits_stride; a.grad_stride = d->grad_stride; a.ids_stride = d->ids_stride; a.teacher_stride = d->teacher_stride;
  a.inv_temp = (float)(1.0 / (double)d->temperature);
  a.scale2 = (float)(1.4426950408889634 / (double)d->temperature);
  a.denom_scale = d->reduction == FRL_REDUCE_MEAN ? (float)(1.0 / (double)d->rows) : 1.0f;
  a.vocab = d->vocab; a.top = d->top; a.ids64 = d->ids64; a.teacher_dtype = d->teacher_dtype;
  a.segs = p.segs; a.seg_len = p.seg_len;
  return a;
}

// workspace: row losses, the inverse of the denominator (64 floats), row statistics where the caller keeps none, segments
struct DistillWs { size_t rowloss, inv, stats, part, total; };
static DistillWs distill_ws(const FrlDistillDesc* d, const DistillPlan& p) {
  auto up = [](size_t n) { return (n + 63) / 64 * 64; };
  DistillWs w;
  w.rowloss = 0;
  w.inv = up((size_t)d->rows);
  w.stats = w.inv + 64;
  w.part = w.stats + up(4 * (size_t)(d->rows + 1));
  w.total = (w.part + (p.segs > 1 ? up(3 * (size_t)d->rows * p.segs) : 0)) * sizeof(float);
  return w;
}

template <typename T, bool REST>
static hipError_t launch_rows(const DistillArgs& a, int G, bool grad, hipStream_t st) {
  const size_t per = ((size_t)(REST ? (a.vocab + 31) / 32 : 0) + 2 * (size_t)a.top) * 4;
  const size_t lds = G == 64 ? 4 * per : per;
  const long long blocks = G == 64 ? (a.rows + 3) / 4 : a.rows;
  const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
#define FRL_GO(g, gr) hipLaunchKernelGGL((frl_distill_row_kernel<T, g, REST, gr>), dim3(grid), dim3(g == 64 ? 256 : g), lds, st, a)
  if (G == 64) { if (grad) FRL_GO(64, true); else FRL_GO(64, false); }
  else if (G == 256) { if (grad) FRL_GO(256, true); else FRL_GO(256, false); }
  else { if (grad) FRL_GO(1024, true); else FRL_GO(1024, false); }
#undef FRL_GO
  note_kernel("frl_distill_row_kernel<%s, %d threads> [%u]", grad ? "value + gradient" : "value", G, grid);
  return hipGetLastError();
}

template <typename T, bool REST>
static hipError_t launch_parts(const DistillArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)(a.rows * a.segs);
  hipLaunchKernelGGL((frl_distill_part_kernel<T, 256, REST>), dim3(grid), dim3(256), REST ? (size_t)(a.seg_len / 32) * 4 : 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((frl_distill_join_kernel<T, REST>), dim3((unsigned)a.rows), dim3(64), (size_t)a.top * 8, st, a);
  note_kernel("frl_distill_part_kernel [%u] + frl_distill_join_kernel [%lld]", grid, a.rows);
  return hipGetLastError();
}

template <typename T, bool REST>
static hipError_t launch_grad(const DistillArgs& a, int G, hipStream_t st) {
  const long long items = a.rows * a.segs, blocks = G == 64 ? (items + 3) / 4 : items;
  const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
  const size_t lds = (size_t)a.top * 8 * (G == 64 ? 4 : 1);
  if (G == 64) hipLaunchKernelGGL((frl_distill_grad_kernel<T, 64, REST>), dim3(grid), dim3(256), lds, st, a);
  else if (G == 256) hipLaunchKernelGGL((frl_distill_grad_kernel<T, 256, REST>), dim3(grid), dim3(256), lds, st, a);
  else hipLaunchKernelGGL((frl_distill_grad_kernel<T, 1024, REST>), dim3(grid), dim3(1024), lds, st, a);
  note_kernel("frl_distill_grad_kernel<%d threads> [%u]", G, grid);
  return hipGetLastError();
}

#define FRL_BY_TYPE(call)                                                                                                       \
  (dtype == FRL_ELT_F32 ? (rest ? call<float, true> : call<float, false>)                                                      \
   : dtype == FRL_ELT_BF16 ? (rest ? call<Bf16, true> : call<Bf16, false>) : (rest ? call<F16, true> : call<F16, false>))

}  // namespace frl

using namespace frl;

extern "C" {

size_t frl_distill_workspace_bytes(const FrlDistillDesc* desc) {
  if (distill_validate(desc) != FRL_OK) return 0;
  return distill_ws(desc, distill_plan(desc->rows, desc->vocab)).total;
}

int frl_distill_fwd(const FrlDistillDesc* desc, const FrlDistillBufs* bufs, void* workspace, size_t workspace_bytes, void* hip_stream) {
  clear_kernels();
  const int rc = distill_validate(desc);
  if (rc != FRL_OK) return rc;
  if (bufs == nullptr || bufs->loss == nullptr) { set_error("distill: bufs.loss is NULL"); return FRL_EINVAL; }
  if (desc->rows > 0 && (bufs->logits == nullptr || bufs->ids == nullptr || bufs->teacher == nullptr)) { set_error("distill: bufs.logits / ids / teacher is NULL"); return FRL_EINVAL; }
  if (desc->rows == 0 && desc->reduction == FRL_REDUCE_NONE) return FRL_OK;
  if (((uintptr_t)bufs->row_stats & 15) != 0) { set_error("distill: bufs.row_stats must be 16-byte aligned"); return FRL_EINVAL; }
  const bool grad = bufs->grad != nullptr && desc->rows > 0;
  if (grad && desc->rows > 1 && desc->grad_stride < desc->vocab) { set_error("distill: grad row stride %lld < vocab %d", (long long)desc->grad_stride, desc->vocab); return FRL_EINVAL; }
  if (grad && distill_overlap(desc, bufs)) { set_error("distill: grad overlaps logits"); return FRL_EINVAL; }
  const DistillPlan p = distill_plan(desc->rows, desc->vocab);
  const DistillWs w = distill_ws(desc, p);
  if (workspace == nullptr || ((uintptr_t)workspace & 255) != 0) { set_error("workspace must be non-NULL and 256-byte aligned"); return FRL_EWORKSPACE; }
  if (workspace_bytes < w.total) { set_error("workspace %zu B < required %zu B", workspace_bytes, w.total); return FRL_EWORKSPACE; }
  float* ws = (float*)workspace;
  hipStream_t st = (hipStream_t)hip_stream;
  DistillArgs a = distill_args(desc, bufs, p);
  const int dtype = desc->dtype;
  const bool rest = desc->kind == FRL_DISTILL_REST, split = p.segs > 1;
  a.rowloss = desc->reduction == FRL_REDUCE_NONE ? bufs->loss : ws + w.rowloss;
  a.stats = bufs->row_stats != nullptr ? bufs->row_stats : (split && grad) ? ws + w.stats : nullptr;
  a.part = ws + w.part;
  hipError_t e = hipSuccess;
  if (desc->reduction == FRL_REDUCE_MEAN && bufs->weights != nullptr && desc->rows > 0) {
    float* inv = bufs->row_stats != nullptr ? bufs->row_stats + 4 * desc->rows : ws + w.inv;
    a.inv_denom = inv;
    hipLaunchKernelGGL(frl_distill_denom_kernel, dim3(1), dim3(1024), 0, st, bufs->weights, (long long)desc->rows, inv);
    e = hipGetLastError();
    if (e == hipSuccess) note_kernel("frl_distill_denom_kernel");
  }
  if (e == hipSuccess && desc->rows > 0) {
    if (split) {
      e = FRL_BY_TYPE(launch_parts)(a, st);
      if (e == hipSuccess && grad) e = FRL_BY_TYPE(launch_grad)(a, p.G, st);
    } else {
      e = FRL_BY_TYPE(launch_rows)(a, p.G, grad, st);
    }
  }
  if (e == hipSuccess && desc->reduction != FRL_REDUCE_NONE) {
    hipLaunchKernelGGL(frl_distill_sum_kernel, dim3(1), dim3(1024), 0, st, a.rowloss, (long long)desc->rows, a.inv_denom, desc->rows > 0 ? a.denom_scale : 0.0f, bufs->loss);
    e = hipGetLastError();
    if (e == hipSuccess) note_kernel("frl_distill_sum_kernel");
  }
  if (e != hipSuccess) { set_error("distill launch: %s", hipGetErrorString(e)); return FRL_EHIP; }
  return FRL_OK;
}

int frl_distill_bwd(const FrlDistillDesc* desc, const FrlDistillBufs* bufs, void* hip_stream) {
  clear_kernels();
  const int rc = distill_validate(desc);
  if (rc != FRL_OK) return rc;
  if (desc->rows == 0) return FRL_OK;
  if (bufs == nullptr || bufs->logits == nullptr || bufs->ids == nullptr || bufs->teacher == nullptr) { set_error("distill: bufs.logits / ids / teacher is NULL"); return FRL_EINVAL; }
  if (bufs->grad == nullptr || bufs->row_stats == nullptr || bufs->g_loss == nullptr) { set_error("distill: bufs.grad / row_stats / g_loss is NULL"); return FRL_EINVAL; }
  if (((uintptr_t)bufs->row_stats & 15) != 0) { set_error("distill: bufs.row_stats must be 16-byte aligned"); return FRL_EINVAL; }
  if (desc->rows > 1 && desc->grad_stride < desc->vocab) { set_error("distill: grad row stride %lld < vocab %d", (long long)desc->grad_stride, desc->vocab); return FRL_EINVAL; }
  if (distill_overlap(desc, bufs)) { set_error("distill: grad overlaps logits"); return FRL_EINVAL; }
  const DistillPlan p = distill_plan(desc->rows, desc->vocab);
  DistillArgs a = distill_args(desc, bufs, p);
  a.stats = bufs->row_stats;
  a.g_loss = bufs->g_loss;
  a.g_stride = desc->reduction == FRL_REDUCE_NONE ? 1 : 0;
  if (desc->reduction == FRL_REDUCE_MEAN && bufs->weights != nullptr) a.inv_denom = bufs->row_stats + 4 * desc->rows;
  const int dtype = desc->dtype;
  const bool rest = desc->kind == FRL_DISTILL_REST;
  const hipError_t e = FRL_BY_TYPE(launch_grad)(a, p.G, (hipStream_t)hip_stream);
  if (e != hipSuccess) { set_error("distill gradient launch: %s", hipGetErrorString(e)); return FRL_EHIP; }
  return FRL_OK;
}

}  // extern "C"
