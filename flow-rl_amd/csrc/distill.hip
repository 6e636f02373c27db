// KL divergence of a student's softmax from a teacher's top entries, and its gradient: frl_distill_fwd / frl_distill_bwd.
//
// Mathematics (include/flowrl_hip.h).  With c = log2(e) / T, a row needs m = max z and s = sum 2^((z - m) c); where the teacher's unnamed mass is a
// class of its own, its entries ("the rest") have a maximum m' and a sum r = sum 2^((z - m') c) of theirs, and the named entries another pair: the
// rest of a student that is sure of what is named, or of a vocabulary masked beside it, lies further below m than an exponential spans, and
// still has a divergence and a gradient.  Then q = 2^((z - m) c) / s, Q = 2^((m' - m) c) r / s and
//     L      = sum p (log p + (a - z) / T) + sum p * ((m - a) / T + log s)   [+ P (log P - log Q)]
//     dL/dz  = (q - p) / T                              named entries   (FRL_DISTILL_TOP: sum p = 1)
//     dL/dz  = q / T, or                                the others, FRL_DISTILL_TOP
//              2^((z - m') c) (Q - P) / (r T)           the others, FRL_DISTILL_REST with P > 0
// with a the largest named logit, so that rows far from zero (and small T) lose no digits: a - z and m - a are not negative.
// The gradient is therefore one scaled exponential per element plus a correction of `top` elements.
//
// HBM-bound for long rows: the logits once, the gradient once.  For a gradient a row lives in the registers of the threads that share it (16
// lanes up to a workgroup of 512, at most 16 vectors of 16 bytes each: 65536 entries of two bytes) and behind those in LDS (36864 more); only what
// is longer is read a second time.  A value keeps nothing and streams.  An element costs two quarter-rate exponentials (four issue slots each), one
// for the sum and one for the gradient; the rest is kept to four slots per element: the shift by the maximum is one fma, two bytes are packed by one
// convert, and the factor of a two-byte gradient goes into the exponent.  The gradient, and logits that are read for the last time, pass the
// caches by (non-temporal): 8192 x 131072 bf16 with its gradient 963 -> 907 us, 4096 x 32000 126 -> 107.
// Rows beyond 2^18 entries, or too few to fill the chip, are split over their length, joined by a second kernel, and differentiated by a third.
#include "frl_rows.h"

namespace frl {

struct DistillArgs {
  const void* logits; const void* ids; const void* teacher; const float* weights;
  float* rowloss;             // (rows,) weight * L
  float* stats;               // (rows + 1, 4) or NULL: m, factor of 2^((z - m) c) of the named entries, m', factor of 2^((z - m') c) of the others; last
                              // row: 1 / denominator
  const float* inv_denom;     // device 1 / sum of weights, or NULL: `denom_scale`
  const float* g_loss;        // backward: cotangent, `g_stride` apart per row (0: one scalar); NULL: 1
  void* grad;
  float* part;                // split rows: (rows, segs, 4) maximum and sum of the rest (FRL_DISTILL_TOP: of everything), of the named entries
  long long rows, logits_stride, grad_stride, ids_stride, teacher_stride;
  float inv_temp, scale2, denom_scale;   // 1 / T, log2(e) / T
  int vocab, top, ids64, teacher_dtype, segs, seg_len, g_stride;
  int kept, kept_at;          // row kernel: vectors per thread that stay in LDS behind those in registers, and where (in words)
};

constexpr double LN2 = 0.6931471805599453;
constexpr int DSEG_MAX = 1 << 16;      // entries of a segment
constexpr int DROW_MAX = 1 << 18;      // entries of a row that is not split

__device__ __forceinline__ float teacher_at(const void* p, long long i, int dtype) {
  if (dtype == FRL_ELT_F32) return ((const float*)p)[i];
  if (dtype == FRL_ELT_BF16) return Elt<Bf16>::get(((const Bf16*)p)[i]);
  return Elt<F16>::get(((const F16*)p)[i]);
}

// n entries from z, cut where 16-byte vectors lie on 16-byte boundaries (rows of an odd two-byte vocabulary would otherwise read at odd
// words: 171 against 138 us for a value of 2048 x 200001 bf16): `head` single entries, `nvec` vectors, `tail` single ones.  The entries' named bits
// stand `pad` behind their number, so that a vector's bits do not cross a word.
template <typename T>
struct Cut {
  static constexpr int N = Vec16<T>::N;
  int head, nvec, tail, pad;
  __device__ __forceinline__ Cut(const T* z, int n) {
    head = min((N - (int)(((uintptr_t)z & 15) / sizeof(T))) % N, n);
    nvec = (n - head) / N;
    tail = n - head - nvec * N;
    pad = (N - head) % N;
  }
  // the single entry that thread tid sees to, or -1 (G >= 16 threads: N for the head, N for the tail)
  __device__ __forceinline__ int lone(int tid) const { return tid < head ? tid : tid >= N && tid - N < tail ? head + nvec * N + tid - N : -1; }
  __device__ __forceinline__ int bit(int at) const { return head + pad + at * N; }
};

// the named tokens of [v0, v0 + n) as bits, token v0 at bit `pad`; `words` covers n rounded up to 32, and one more
template <int G>
__device__ __forceinline__ void mark_named(const DistillArgs& a, long long row, int tid, int v0, int n, int pad, unsigned* words) {
  for (int w = tid; w < (n + 31) / 32 + 1; w += G) words[w] = 0u;
  group_sync<G>();
  for (int k = tid; k < a.top; k += G) {
    const long long loc = ld_id(a.ids, row * a.ids_stride + k, a.ids64) - v0;
    if (loc >= 0 && loc < n) atomicOr(&words[(loc + pad) >> 5], 1u << ((loc + pad) & 31));
  }
  group_sync<G>();
}

template <int N>
__device__ __forceinline__ float sum_of(const float* e) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) s += e[i];
  return s;
}
// the named bits of the N entries from v (a multiple of N)
template <int N>
__device__ __forceinline__ unsigned named_bits(const unsigned* words, int v) { return (words[v >> 5] >> (v & 31)) & ((1u << N) - 1u); }

// A thread's running maximum, and a sum that it rescales when something raises the maximum.
struct Running {
  float m = -INFINITY, s = 0.0f;
  __device__ __forceinline__ void raise(float to, float c) {
    if (to > m) {
      about(to, c);
      m = to;
    }
  }
  __device__ __forceinline__ void one(float x, float c) {
    raise(x, c);
    Shift(m == -INFINITY ? 0.0f : m, c).exps<1>(&x);
    s += x;
  }
  // the sum with respect to a maximum over more threads; a thread that saw only -inf has a sum of 0 (or NaN) and keeps it
  __device__ __forceinline__ void about(float all, float c) {
    if (m != -INFINITY) s *= Shift(all, c).from(Shift(m, c));
  }
};

// The same for the few named entries of a thread, one at a time and without a branch; the reference is m c itself.
struct Few {
  float m = -INFINITY, s = 0.0f;
  __device__ __forceinline__ void about(float all, float c) {
    const float base = all == -INFINITY ? 0.0f : all;
    s *= __builtin_amdgcn_exp2f((m - base) * c);
    m = all;
  }
  __device__ __forceinline__ void one(float x, float c) {
    about(fmaxf(m, x), c);
    s += __builtin_amdgcn_exp2f((x - (m == -INFINITY ? 0.0f : m)) * c);
  }
};

// Named entries among a vector's N: they go into a sum of their own, and -inf takes their place among the rest.  Few vectors have one.
template <typename T>
__device__ __forceinline__ void take_named(u32x4& raw, unsigned named, float c, Few& of_named) {
  const unsigned ninf = Vec16<T>::fill_minus_inf()[0];
  while (named != 0u) {
    const int i = __builtin_ctz(named), w = sizeof(T) == 4 ? i : i >> 1;
    named &= named - 1u;
    const unsigned word = w == 0 ? raw[0] : w == 1 ? raw[1] : w == 2 ? raw[2] : raw[3];
    unsigned mask = 0xffffffffu;
    float x;
    if constexpr (sizeof(T) == 4) {
      x = __uint_as_float(word);
    } else {
      mask = (i & 1) ? 0xffff0000u : 0x0000ffffu;
      x = Elt<T>::get(T{(unsigned short)((i & 1) ? word >> 16 : word)});
    }
    const unsigned without = (word & ~mask) | (ninf & mask);
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j] = j == w ? without : raw[j];
    of_named.one(x, c);
  }
}

// A thread's share of a row that is streamed
template <bool REST>
struct Share {
  Running run;                                             // without REST everything is in here
  Few of_named;
  // vectors [from, to) of the vectors at z, G threads apart; the first one's named bits begin at bit0.  Those before `keep` stay in LDS (at `kept`) for
  // the same thread's gradient.
  template <typename T, int G>
  __device__ __forceinline__ void stream(const T* z, int from, int to, float c, const unsigned* words, int bit0, int tid, int keep = 0, u32x4* kept = nullptr) {
    constexpr int U = 4, N = Vec16<T>::N;
    for (int at = from + tid; at < to; at += U * G) {
      u32x4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = at + u * G < to ? ldu<u32x4>(z + (size_t)(at + u * G) * N) : Vec16<T>::fill_minus_inf();
      if (keep > 0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (at + u * G < keep) kept[at + u * G - from] = raw[u];
      }
      if constexpr (REST) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (at + u * G < to) take_named<T>(raw[u], named_bits<N>(words, bit0 + (at + u * G) * N), c, of_named);
      }
      float bm = run.m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[N];
        Vec16<T>::unpack(raw[u], x);
        bm = max_of<N>(x, bm);
      }
      run.raise(bm, c);
      const Shift sh(run.m == -INFINITY ? 0.0f : run.m, c);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[N];
        Vec16<T>::unpack(raw[u], x);
        sh.exps<N>(x);
        run.s += sum_of<N>(x);
      }
    }
  }
  __device__ __forceinline__ void one(float x, float c, bool named) {
    if constexpr (REST) of_named.one(named ? x : -INFINITY, c);      // of -inf there is nothing to add; a branch would put both sums into memory
    run.one(named ? -INFINITY : x, c);
  }
};

// A row's maximum and sum, and the rest's (FRL_DISTILL_TOP: the same)
struct Sums {
  float m, s, mr, r, down;                                 // down: the rest's sum times this is about the row's reference
  template <bool REST>
  static __device__ __forceinline__ Sums of(float mr, float r, float mn, float n, float c) {
    Sums o = {mr, r, mr, r, 1.0f};
    if constexpr (REST) {
      o.m = fmaxf(mr, mn);
      const Shift sh(o.m, c);
      o.down = mr == -INFINITY ? 0.0f : sh.from(Shift(mr, c));
      o.s = (mr == -INFINITY ? r : r * o.down) + (mn == -INFINITY ? n : n * sh.from_exact(mn));      // of -inf alone a sum is 0 (or NaN)
    }
    return o;
  }
};

// What W lanes make of a row's teacher entries: the tokens (into sid, -1 for padding), p (into sp, 0 for padding) and their logits (into sz),
// sum p, the largest of their logits and sum p (log p + (largest - z) / T).  The three loads of an entry are under way together; what follows
// works on LDS.  FRL_DISTILL_REST needs 1 - sum p, which float32 exponentials would leave without digits: float64.
template <typename T, int W, bool REST>
__device__ __forceinline__ void teacher_part(const DistillArgs& a, long long row, const T* z, int lane, int* sid, float* sp, float* sz, double& sum_p, double& cross, float& largest) {
  sum_p = cross = 0.0;
  float tm = -INFINITY, tot = 0.0f, zm = -INFINITY;
  const void* ids = (const char*)a.ids + row * a.ids_stride * (a.ids64 ? 8 : 4);
  for (int k = lane; k < a.top; k += W) {
    const long long id = ld_id(ids, k, a.ids64);
    const float t = teacher_at(a.teacher, row * a.teacher_stride + k, a.teacher_dtype);
    const bool valid = id >= 0 && id < a.vocab;
    sid[k] = valid ? (int)id : -1;
    sp[k] = t;
    const float x = valid ? Elt<T>::get(z[id]) : -INFINITY;
    sz[k] = x;
    zm = fmaxf(zm, x);
    if (valid) tm = fmaxf(tm, t);
  }
  zm = lanes_reduce<MaxOp, W>(zm);
  largest = zm == -INFINITY ? 0.0f : zm;                     // only -inf is named: any number will do, what has p > 0 makes the loss infinite
  if constexpr (!REST) {
    tm = lanes_reduce<MaxOp, W>(tm);
    const float t0 = tm == -INFINITY ? 0.0f : tm;
    for (int k = lane; k < a.top; k += W)
      if (sid[k] >= 0) tot += expf((sp[k] - t0) * a.inv_temp);
    tot = lanes_reduce<SumOp, W>(tot);
  }
  const float log_tot = REST ? 0.0f : logf(tot);
  for (int k = lane; k < a.top; k += W) {
    float p = 0.0f;
    if (sid[k] >= 0) {
      const float t = sp[k];
      const double y = ((double)largest - (double)sz[k]) * (double)a.scale2 * LN2;   // with the rounded log2(e) / T of the exponentials: one temperature throughout
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
      if (p != 0.0f) cross += (double)p * ((double)lp + y);
    }
    sp[k] = p;
  }
  sum_p = lanes_reduce<SumOp, W>(sum_p);
  cross = lanes_reduce<SumOp, W>(cross);
}

__device__ __forceinline__ float inverse(double s) { return s != 0.0 ? (float)(1.0 / s) : 0.0f; }

// The gradient is T^-1 times the cotangent times: named 2^((z - m) c) - p, and rest 2^((z - m') c)
struct Factors { float named, rest; };

template <bool REST>
__device__ __forceinline__ Factors row_factors(const Sums& t, double sum_p) {
  const float inv_s = 1.0f / t.s;
  if constexpr (REST) {
    const double P = 1.0 - sum_p;
    if (P > 0.0) return Factors{inv_s, t.r == 0.0f ? 0.0f : t.down * inv_s - (float)P / t.r};      // an empty rest has no gradient
    return Factors{(float)sum_p * inv_s, (float)sum_p * t.down * inv_s};
  } else {
    // a softmax sums to one; a row that names nothing has neither loss nor gradient
    const float k = sum_p != sum_p ? (float)sum_p * inv_s : sum_p != 0.0 ? inv_s : 0.0f;
    return Factors{k, k};
  }
}

template <bool REST>
__device__ __forceinline__ float row_loss(const DistillArgs& a, const Sums& t, double sum_p, double cross, float largest) {
  if (!REST && sum_p == 0.0) return 0.0f;
  const double c = (double)a.scale2, m = (double)t.m;
  const double log_s = (double)Shift(t.m, a.scale2).residue() * LN2 + log((double)t.s);
  double loss = cross + sum_p * ((m - (double)largest) * c * LN2 + log_s);
  if constexpr (REST) {
    const double P = 1.0 - sum_p;
    if (P > 0.0) {
      const double log_r = (double)Shift(t.mr, a.scale2).residue() * LN2 + log((double)t.r);
      loss += P * (log(P) + (m - (double)t.mr) * c * LN2 + log_s - log_r);
    }
  }
  return (float)loss;
}

template <typename T, int G>
__device__ __forceinline__ void zero_row(T* g, int n, int tid) {
  constexpr int N = Vec16<T>::N;
  const int nvec = n / N, tail = n - nvec * N;
  for (int at = tid; at < nvec; at += G) stu(g + (size_t)at * N, u32x4{0u, 0u, 0u, 0u});
  if (tid < tail) g[nvec * N + tid] = Elt<T>::put(0.0f);
}

// f_rest 2^((x - m) c) of a vector.  A two-byte gradient takes |f_rest| into the exponent while |M| < 128 rounds M - log2 |f_rest| by less than 2^-17
// (the gradient's own rounding is 2^-11 or 2^-8).
template <typename T>
struct Scaled {
  Shift sh;
  float f, M;
  unsigned sign;
  __device__ __forceinline__ Scaled(const Shift& s, float f_rest) : sh(s), f(f_rest), M(s.M - __builtin_amdgcn_logf(fabsf(f_rest))), sign(f_rest < 0.0f ? 0x80008000u : 0u) {}
  __device__ __forceinline__ u32x4 of(u32x4 raw) const {
    constexpr int N = Vec16<T>::N;
    float x[N];
    Vec16<T>::unpack(raw, x);
    if (sizeof(T) == 2 && fabsf(sh.M) < 128.0f) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], sh.c, -M));
      u32x4 r = Vec16<T>::pack(x);
      r ^= sign;
      return r;
    }
    sh.exps<N>(x);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= f;
    return Vec16<T>::pack(x);
  }
  __device__ __forceinline__ float one(float x) const {
    sh.exps<1>(&x);
    return f * x;
  }
};

template <typename T, int G>
__device__ __forceinline__ void stream_gradient(const T* z, T* g, int from, int to, const Scaled<T>& sc, int tid, int keep = 0, const u32x4* kept = nullptr) {
  constexpr int U = 4, N = Vec16<T>::N;
  int done = from;
  for (; done < keep; done += G)                           // what the sums left in LDS
    if (done + tid < min(keep, to)) stu_nt(g + (size_t)(done + tid) * N, sc.of(kept[done + tid - from]));
  from = done;
  for (int at = from + tid; at < to; at += U * G) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at + u * G < to) raw[u] = ldu_nt<u32x4>(z + (size_t)(at + u * G) * N);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at + u * G < to) stu_nt(g + (size_t)(at + u * G) * N, sc.of(raw[u]));
  }
}

// The named entries of [v0, v0 + n), over what the scaled exponentials put there.  Both are plain stores of one workgroup with a barrier
// between them, so these are what stays; of a token named twice the first entry writes, with both probabilities.
template <typename T, int G>
__device__ __forceinline__ void named_gradient(const DistillArgs& a, T* g, int v0, int n, const Shift& sh, float f_named, float f, const int* sid, const float* sp,
                                               const float* sz, int tid) {
  for (int k = tid; k < a.top; k += G) {
    const int id = sid[k];
    if (id < v0 || id >= v0 + n) continue;
    float p = 0.0f;
    bool first = true;
    for (int j = 0; j < a.top; ++j)
      if (sid[j] == id) { p += sp[j]; first = first && j >= k; }
    if (!first) continue;
    float x = sz[k];
    sh.exps<1>(&x);
    g[id] = Elt<T>::put(f_named * x - f * p);
  }
}

// Between two passes over the vectors: the compiler may not carry their unpacked elements from one to the other, twice the registers.
template <int NV>
__device__ __forceinline__ void keep_packed(u32x4* raw) {
#pragma unroll
  for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(raw[i]));
}

// A row to a group, its first NV vectors per thread held in registers: value, what the backward needs, and (GRAD) the gradient.
// Bound by HBM: 2048 x 131072 bf16, value with a rest: 94 us, 5.7 TB/s of the 5.9 that reads alone reach; 4096 x 32000 bf16 with its gradient: 100 us,
// 5.2 TB/s; 8192 x 131072 bf16 with a rest and its gradient: 888 us, 5.0 TB/s (a large copy: 4.9 to 5.4).  A row's passes (maximum, sum, gradient) wait for
// one another, so it takes a second workgroup on the CU to keep the memory busy; hence at most 512 threads with what they hold in registers.
template <typename T, int G, int NV, bool REST, bool GRAD>
__global__ void __launch_bounds__(G <= 64 ? 256 : G, 4) frl_distill_row_kernel(const DistillArgs a) {
  extern __shared__ __align__(16) unsigned lds[];
  constexpr int GPB = G <= 64 ? 256 / G : 1, N = Vec16<T>::N;
  constexpr int WAVES = G < 64 ? 1 : G / 64;
  __shared__ float red0[WAVES], red1[WAVES];
  __shared__ double row_p[GPB], row_x[GPB];
  __shared__ float row_z[GPB];
  const int tid = threadIdx.x % G, grp = G < 64 ? threadIdx.x / G : G == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int nwords = REST ? (a.vocab + 31) / 32 + 1 : 0;
  unsigned* words = lds + (size_t)grp * (nwords + 3 * a.top);
  int* sid = (int*)(words + nwords);
  float* sp = (float*)(sid + a.top);
  float* sz = sp + a.top;
  u32x4* kept = (u32x4*)(lds + a.kept_at);
  const float inv = a.inv_denom != nullptr ? *a.inv_denom : a.denom_scale;
  const long long row = block_index() * GPB + grp;
  if (row >= a.rows) return;
  const T* z = (const T*)a.logits + row * a.logits_stride;
  T* g = GRAD ? (T*)a.grad + row * a.grad_stride : nullptr;
  const Cut<T> cut(z, a.vocab);
  const T* zv = z + cut.head;
  const int nvec = cut.nvec, nv = (nvec + G - 1) / G, lone = cut.lone(tid);
  const float w = a.weights != nullptr ? a.weights[row] : 1.0f;
  if (w == 0.0f) {                                       // uniform over the group
    if (tid == 0) {
      a.rowloss[row] = 0.0f;
      if (a.stats != nullptr) *(f32x4*)(a.stats + 4 * row) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if constexpr (GRAD) zero_row<T, G>(g, a.vocab, tid);
    return;
  }
  // what the row holds is asked for before anything else; the teacher's part works meanwhile
  constexpr int R = NV > 0 ? NV : 1;
  u32x4 raw[R];
  const int t0 = fresh(tid);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    raw[i] = Vec16<T>::fill_minus_inf();
    if (i < nv && i * G + t0 < nvec) raw[i] = ldu_nt<u32x4>((const char*)zv + 16u * (unsigned)(i * G + t0));
  }
  if constexpr (REST) mark_named<G>(a, row, tid, 0, a.vocab, cut.pad, words);
  if (tid < 64) {
    double sum_p, cross;
    float largest;
    teacher_part<T, G < 64 ? G : 64, REST>(a, row, z, tid, sid, sp, sz, sum_p, cross, largest);
    if (tid == 0) { row_p[grp] = sum_p; row_x[grp] = cross; row_z[grp] = largest; }
  }
  Share<REST> mine;
  if (nvec > NV * G) mine.template stream<T, G>(zv, NV * G, nvec, a.scale2, words, cut.bit(0), t0, GRAD ? (NV + a.kept) * G : 0, kept);
  if (lone >= 0) mine.one(Elt<T>::get(z[lone]), a.scale2, REST && named_bits<1>(words, lone + cut.pad) != 0u);
  float mr = mine.run.m;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i < nv) {
      if constexpr (REST)
        if (i * G + t0 < nvec) take_named<T>(raw[i], named_bits<N>(words, cut.bit(i * G + t0)), a.scale2, mine.of_named);
      float x[N];
      Vec16<T>::unpack(raw[i], x);
      mr = max_of<N>(x, mr);
      __builtin_amdgcn_sched_barrier(0);
    }
  mr = group_reduce<MaxOp, G>(mr, red0);
  const float mn = REST ? group_reduce<MaxOp, G>(mine.of_named.m, red1) : -INFINITY;
  mine.run.about(mr, a.scale2);
  const Shift sh(mr == -INFINITY ? 0.0f : mr, a.scale2);
  keep_packed<NV>(raw);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i < nv) {
      float x[N];
      Vec16<T>::unpack(raw[i], x);
      sh.exps<N>(x);
      mine.run.s += sum_of<N>(x);
      __builtin_amdgcn_sched_barrier(0);                     // one vector unpacked at a time: eight independent elements are parallel enough
    }
  // two arrays in turn: between a result that is read and the next that is written into the same one lies the other's barrier
  const float r = group_reduce<SumOp, G>(mine.run.s, REST ? red0 : red1);
  float n = 0.0f;
  if constexpr (REST) {
    mine.of_named.about(mn, a.scale2);
    n = group_reduce<SumOp, G>(mine.of_named.s, red1);
  }
  if constexpr (G <= 64) group_sync<G>();                    // the teacher's part is visible (a workgroup has passed barriers since)
  const Sums sums = Sums::of<REST>(mr, r, mn, n, a.scale2);
  const double sum_p = row_p[grp];
  const Factors k = row_factors<REST>(sums, sum_p);
  if constexpr (GRAD) {
    const float f = w * inv * a.inv_temp;
    if (k.named == 0.0f && k.rest == 0.0f) {
      zero_row<T, G>(g, a.vocab, tid);
    } else {
      const Scaled<T> sc(sh, f * k.rest);
      keep_packed<NV>(raw);
      const int t2 = fresh(tid);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i < nv && i * G + t2 < nvec) {
          stu_nt((char*)(g + cut.head) + 16u * (unsigned)(i * G + t2), sc.of(raw[i]));
          __builtin_amdgcn_sched_barrier(0);
        }
      if (nvec > NV * G) stream_gradient<T, G>(zv, g + cut.head, NV * G, nvec, sc, t2, (NV + a.kept) * G, kept);
      if (lone >= 0) g[lone] = Elt<T>::put(sc.one(Elt<T>::get(z[lone])));
      group_sync<G>();
      named_gradient<T, G>(a, g, 0, a.vocab, Shift(sums.m, a.scale2), f * k.named, f, sid, sp, sz, tid);
    }
  }
  if (tid == 0) {
    a.rowloss[row] = w * row_loss<REST>(a, sums, sum_p, row_x[grp], row_z[grp]);
    if (a.stats != nullptr) *(f32x4*)(a.stats + 4 * row) = f32x4{sums.m, k.named, sums.mr, k.rest};
  }
}

// ---- rows split over their length ---------------------------------------------------------------------------------------

// A segment to a workgroup of 256, so that few rows reach many CUs.  3 x 200001 f16: 3.8 us, then 4.0 for the join and 5.6 for the gradient, each
// little more than a launch and one trip to memory; a finished row could only be seen by the other workgroups of the same launch through a counter
// in memory.

template <typename T, int G, bool REST>
__global__ void __launch_bounds__(G) frl_distill_part_kernel(const DistillArgs a) {
  extern __shared__ __align__(16) unsigned lds[];
  __shared__ float red0[G / 64], red1[G / 64];
  const long long item = block_index();
  if (item >= a.rows * a.segs) return;
  const long long row = item / a.segs;
  const int v0 = (int)(item - row * a.segs) * a.seg_len, n = min(a.vocab - v0, a.seg_len);
  if (a.weights != nullptr && a.weights[row] == 0.0f) return;
  const T* z = (const T*)a.logits + row * a.logits_stride + v0;
  const int tid = threadIdx.x;
  const Cut<T> cut(z, n);
  const int lone = cut.lone(tid);
  if constexpr (REST) mark_named<G>(a, row, tid, v0, n, cut.pad, lds);
  Share<REST> mine;
  mine.template stream<T, G>(z + cut.head, 0, cut.nvec, a.scale2, lds, cut.bit(0), tid);
  if (lone >= 0) mine.one(Elt<T>::get(z[lone]), a.scale2, REST && named_bits<1>(lds, lone + cut.pad) != 0u);
  const float mr = group_reduce<MaxOp, G>(mine.run.m, red0), mn = REST ? group_reduce<MaxOp, G>(mine.of_named.m, red1) : -INFINITY;
  mine.run.about(mr, a.scale2);
  const float r = group_reduce<SumOp, G>(mine.run.s, REST ? red0 : red1);                 // the arrays in turn, as in the row kernel
  float named = 0.0f;
  if constexpr (REST) {
    mine.of_named.about(mn, a.scale2);
    named = group_reduce<SumOp, G>(mine.of_named.s, red1);
  }
  if (threadIdx.x == 0) *(f32x4*)(a.part + 4 * item) = f32x4{mr, r, mn, named};
}

// One wave per row: the segments joined in order, then the teacher's entries.  A workgroup of 16 waves that holds every row finishes the loss as well.
template <typename T, bool REST>
__global__ void __launch_bounds__(1024) frl_distill_join_kernel(const DistillArgs a, float* loss, float* inv_out) {
  extern __shared__ __align__(16) unsigned lds[];
  __shared__ float row_w[16], row_l[16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  int* sid = (int*)lds + (size_t)wave * 3 * a.top;
  float* sp = (float*)(sid + a.top);
  float* sz = sp + a.top;
  const long long row = block_index() * waves + wave;
  float w = 0.0f, value = 0.0f;
  if (row < a.rows) {
    w = a.weights != nullptr ? a.weights[row] : 1.0f;
    f32x4 st = {0.0f, 0.0f, 0.0f, 0.0f};
    if (w != 0.0f) {
      double sum_p, cross;
      float largest;
      teacher_part<T, 64, REST>(a, row, (const T*)a.logits + row * a.logits_stride, lane, sid, sp, sz, sum_p, cross, largest);
      float mr = -INFINITY, mn = -INFINITY, r = 0.0f, n = 0.0f;
      const float* p = a.part + 4 * row * a.segs;
      for (int i = lane; i < a.segs; i += 64) {
        mr = fmaxf(mr, p[4 * i]);
        mn = fmaxf(mn, p[4 * i + 2]);
      }
      mr = wave_reduce<MaxOp>(mr);
      mn = wave_reduce<MaxOp>(mn);
      for (int i = lane; i < a.segs; i += 64) {              // a segment of -inf alone has a sum of 0 (or NaN)
        const f32x4 v = *(const f32x4*)(p + 4 * i);
        r += v[0] == -INFINITY ? v[1] : v[1] * Shift(mr, a.scale2).from(Shift(v[0], a.scale2));
        n += v[2] == -INFINITY ? v[3] : v[3] * __builtin_amdgcn_exp2f((v[2] - mn) * a.scale2);
      }
      r = wave_reduce<SumOp>(r);
      n = wave_reduce<SumOp>(n);
      const Sums sums = Sums::of<REST>(mr, r, mn, n, a.scale2);
      const Factors k = row_factors<REST>(sums, sum_p);
      value = w * row_loss<REST>(a, sums, sum_p, cross, largest);
      st = f32x4{sums.m, k.named, sums.mr, k.rest};
    }
    if (lane == 0) {
      a.rowloss[row] = value;
      if (a.stats != nullptr) *(f32x4*)(a.stats + 4 * row) = st;
    }
  }
  if (loss == nullptr) return;
  if (lane == 0) {
    row_w[wave] = w;
    row_l[wave] = value;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double sw = 0.0, sl = 0.0;
    for (int i = 0; i < waves; ++i) {
      sw += (double)row_w[i];
      sl += (double)row_l[i];
    }
    const float f = inv_out != nullptr ? inverse(sw) : a.denom_scale;
    if (inv_out != nullptr) *inv_out = f;
    *loss = (float)(sl * (double)f);
  }
}

// Gradient of one segment of a row from the row's statistics, also autograd's backward.  HBM: 1024 x 50001 f32 70 us, 410 MB read and written at 5.9 TB/s
// (part of the logits still lies in the caches from the forward).
template <typename T, int G, bool REST>
__global__ void __launch_bounds__(G == 64 ? 256 : G) frl_distill_grad_kernel(const DistillArgs a) {
  extern __shared__ __align__(16) unsigned lds[];
  constexpr int GPB = G == 64 ? 4 : 1, N = Vec16<T>::N;
  const int tid = threadIdx.x % G, grp = G == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  int* sid = (int*)lds + (size_t)grp * 3 * a.top;
  float* sp = (float*)(sid + a.top);
  float* sz = sp + a.top;
  const float inv = a.inv_denom != nullptr ? *a.inv_denom : a.denom_scale;
  const long long item = block_index() * GPB + grp;
  if (item >= a.rows * a.segs) return;
  const long long row = item / a.segs;
  const int v0 = (int)(item - row * a.segs) * a.seg_len, n = min(a.vocab - v0, a.seg_len);
  const T* z = (const T*)a.logits + row * a.logits_stride;
  T* g = (T*)a.grad + row * a.grad_stride;
  const float w = a.weights != nullptr ? a.weights[row] : 1.0f;
  const f32x4 st = *(const f32x4*)(a.stats + 4 * row);
  if (w == 0.0f || (st[1] == 0.0f && st[3] == 0.0f)) {
    zero_row<T, G>(g + v0, n, tid);
    return;
  }
  const float cot = a.g_loss != nullptr ? a.g_loss[row * a.g_stride] : 1.0f;
  const float f = cot * w * inv * a.inv_temp;
  const Scaled<T> sc(Shift(st[2] == -INFINITY ? 0.0f : st[2], a.scale2), f * st[3]);
  const Cut<T> cut(z + v0, n);
  const int lone = cut.lone(tid);
  stream_gradient<T, G>(z + v0 + cut.head, g + v0 + cut.head, 0, cut.nvec, sc, tid);
  if (lone >= 0) g[v0 + lone] = Elt<T>::put(sc.one(Elt<T>::get(z[v0 + lone])));
  if (tid < 64) {
    double sum_p, cross;
    float largest;
    teacher_part<T, 64, REST>(a, row, z, tid, sid, sp, sz, sum_p, cross, largest);
  }
  group_sync<G>();
  named_gradient<T, G>(a, g, v0, n, Shift(st[0], a.scale2), f * st[1], f, sid, sp, sz, tid);
}

// ---- over the rows ------------------------------------------------------------------------------------------------------

// The sum of n floats by one workgroup of 1024 in float64, in a fixed order; thread 0 has it.  One workgroup, because a second one would need a second
// launch or a counter; eight loads of four floats are under way per thread before the first is added (32768 rows in one go).
__device__ __forceinline__ double sum_of_rows(const float* __restrict__ x, long long n) {
  __shared__ double red[16];
  double s = 0.0;
  const long long quads = n / 4;
  for (long long i = threadIdx.x; i < quads; i += 8 * 1024) {
    f32x4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i + u * 1024 < quads ? ldu<f32x4>(x + 4 * (i + u * 1024)) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < 8; ++u) s += ((double)v[u][0] + (double)v[u][1]) + ((double)v[u][2] + (double)v[u][3]);
  }
  if (threadIdx.x < n - 4 * quads) s += (double)x[4 * quads + threadIdx.x];
  s = wave_reduce<SumOp>(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return 0.0;
  return wave_reduce<SumOp>(threadIdx.x < 16 ? red[threadIdx.x] : 0.0);
}

// 1 / sum of the weights, 0 where the sum is 0: ahead of a gradient
__global__ void __launch_bounds__(1024) frl_distill_denom_kernel(const float* __restrict__ w, long long rows, float* __restrict__ inv) {
  const double s = sum_of_rows(w, rows);
  if (threadIdx.x == 0) *inv = inverse(s);
}

// loss = the rows' losses summed, times *inv or scale; with weights their inverse sum is the factor, and is left in inv for the backward
__global__ void __launch_bounds__(1024) frl_distill_sum_kernel(const float* __restrict__ rowloss, long long rows, const float* __restrict__ w, float* __restrict__ inv,
                                                               float scale, float* __restrict__ loss) {
  if (w != nullptr) {
    const double s = sum_of_rows(w, rows);
    scale = inverse(s);
    if (threadIdx.x == 0) *inv = scale;
    __syncthreads();
  } else if (inv != nullptr) {
    scale = *inv;
  }
  const double s = sum_of_rows(rowloss, rows);
  if (threadIdx.x == 0) *loss = (float)(s * (double)scale);
}

// ---- host ---------------------------------------------------------------------------------------------------------------

struct DistillPlan { int G, NV, segs, seg_len; bool split; };

// Threads per row: 16 lanes for a row of at most 256 entries and 64 names (65536 x 200 f32 with gradient: 42 us so, 69 by a wave), else as few as hold
// it with 16 vectors of 16 bytes each, more while the rows alone leave the chip's 1024 SIMDs short of four waves.  A value alone keeps nothing and
// streams, up to 1024 threads; a gradient keeps what 512 threads hold (two workgroups to a CU, one loads while the other computes) and reads what
// LDS does not hold of a longer row again.  Measured, bf16, value + gradient: 8192 x 131072 920 us by 512 threads with 16 vectors each, 1145 by 1024
// threads and all of it held, 968 by 512 with nothing held; 4096 x 32000 109 by 256 threads, 133 by 512.  2048 x 131072, value alone: 95 us streamed
// by 1024 threads, 115 held by 512.
// Fewer than 256 rows of more than 8192 entries, and rows whose named bits would take more than 32 KB of LDS, are split: at least 512 segments,
// each of 4096 to 65536 entries.
static DistillPlan distill_plan(const FrlDistillDesc* d, bool grad) {
  const long long rows = d->rows;
  const int vocab = d->vocab, vec = d->dtype == FRL_ELT_F32 ? 4 : 8;
  DistillPlan p = {vocab <= 256 && d->top <= 64 ? 16 : 64, 0, 1, vocab, false};
  if (vocab <= DROW_MAX && !(rows < 256 && vocab > 8192)) {
    const int most = grad ? 512 : 1024;
    auto next = [](int G) { return G < 256 ? 4 * G : 2 * G; };
    while (p.G < most && vocab > p.G * 16 * vec) p.G = next(p.G);
    while (p.G < most && rows * p.G < 4096 * 64 && vocab > 2 * p.G * vec) p.G = next(p.G);
    if (grad) p.NV = vocab <= p.G * 4 * vec ? 4 : 16;
    return p;
  }
  p.G = 256;
  long long want = rows > 0 ? (512 + rows - 1) / rows : 1;
  const long long most = ((long long)vocab + 4095) / 4096, least = ((long long)vocab + DSEG_MAX - 1) / DSEG_MAX;
  if (want > most) want = most;
  if (want < least) want = least;
  p.seg_len = (int)(((vocab + want - 1) / want + 31) / 32 * 32);
  p.segs = (vocab + p.seg_len - 1) / p.seg_len;
  p.split = true;
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
  if (!(d->temperature >= 1e-30f && d->temperature <= 1e30f)) { set_error("distill: temperature %g outside [1e-30, 1e30]", d->temperature); return FRL_EINVAL; }
  if (d->top > FRL_DISTILL_MAX_TOP) { set_error("distill: top %d > %d", d->top, FRL_DISTILL_MAX_TOP); return FRL_EUNSUPPORTED; }
  if (d->vocab > (1 << 30)) { set_error("distill: vocab %d > 2^30", d->vocab); return FRL_EUNSUPPORTED; }
  if (d->rows > (1LL << 30)) { set_error("distill: %lld rows > 2^30", (long long)d->rows); return FRL_EUNSUPPORTED; }
  if (d->rows > 1 && d->logits_stride < d->vocab) { set_error("distill: row stride %lld < vocab %d", (long long)d->logits_stride, d->vocab); return FRL_EINVAL; }
  return FRL_OK;
}

static bool distill_overlap(const FrlDistillDesc* d, const FrlDistillBufs* b) {
  const long long elt = d->dtype == FRL_ELT_F32 ? 4 : 2, width = d->vocab * elt;
  return rows_overlap((uintptr_t)b->logits, width, d->logits_stride * elt, (uintptr_t)b->grad, width, d->grad_stride * elt, d->rows);
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
  w.total = (w.part + (p.split ? up(4 * (size_t)d->rows * p.segs) : 0)) * sizeof(float);
  return w;
}

template <typename T, bool REST>
static hipError_t launch_rows(DistillArgs a, const DistillPlan& p, bool grad, hipStream_t st) {
  const size_t per = ((size_t)(REST ? (a.vocab + 31) / 32 + 1 : 0) + 3 * (size_t)a.top) * 4;
  const int gpb = p.G <= 64 ? 256 / p.G : 1;
  size_t lds = gpb * per;
  if (grad && p.G == 512 && a.vocab > p.G * p.NV * Vec16<T>::N) {
    // Two workgroups to a CU's 160 KB: what is left of a half, 9 vectors a thread and fewer beside named bits, holds more of the row (512 bytes are the
    // kernel's own arrays).  Measured, bf16, against reading that part again: 8192 x 131072 913 -> 896 us, 2048 x 200000 343 -> 334.
    constexpr size_t HALF = 80 * 1024 - 512;
    lds = (lds + 15) / 16 * 16;
    a.kept_at = (int)(lds / 4);
    a.kept = (int)((HALF - lds) / ((size_t)p.G * 16));
    lds += (size_t)a.kept * p.G * 16;
  }
  const long long blocks = (a.rows + gpb - 1) / gpb;
  const dim3 grid = grid_of(blocks);
#define FRL_GO(g, nv, gr) hipLaunchKernelGGL((frl_distill_row_kernel<T, g, nv, REST, gr>), grid, dim3(g <= 64 ? 256 : g), lds, st, a)
  if (!grad) {
    if (p.G == 16) FRL_GO(16, 0, false);
    else if (p.G == 64) FRL_GO(64, 0, false);
    else if (p.G == 256) FRL_GO(256, 0, false);
    else if (p.G == 512) FRL_GO(512, 0, false);
    else FRL_GO(1024, 0, false);
  } else if (p.NV == 4) {
    if (p.G == 16) FRL_GO(16, 4, true);
    else if (p.G == 64) FRL_GO(64, 4, true);
    else if (p.G == 256) FRL_GO(256, 4, true);
    else FRL_GO(512, 4, true);
  } else {
    if (p.G == 64) FRL_GO(64, 16, true);
    else if (p.G == 256) FRL_GO(256, 16, true);
    else FRL_GO(512, 16, true);
  }
#undef FRL_GO
  note_kernel("frl_distill_row_kernel<%s, %d threads, %d vectors> [%lld]", grad ? "value + gradient" : "value", p.G, p.NV, blocks);
  return hipGetLastError();
}

// `loss` and `inv` (mean over weights): where the join is one workgroup, it finishes them
template <typename T, bool REST>
static hipError_t launch_parts(const DistillArgs& a, float* loss, float* inv, hipStream_t st) {
  const long long items = a.rows * a.segs;
  hipLaunchKernelGGL((frl_distill_part_kernel<T, 256, REST>), grid_of(items), dim3(256), REST ? (size_t)((a.seg_len + 31) / 32 + 1) * 4 : 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int waves = loss != nullptr ? (int)a.rows : 1;
  hipLaunchKernelGGL((frl_distill_join_kernel<T, REST>), grid_of((a.rows + waves - 1) / waves), dim3(64 * waves), (size_t)waves * a.top * 12, st, a, loss, inv);
  note_kernel("frl_distill_part_kernel [%lld] + frl_distill_join_kernel<%d rows> [%lld]", items, waves, (a.rows + waves - 1) / waves);
  return hipGetLastError();
}

template <typename T, bool REST>
static hipError_t launch_grad(const DistillArgs& a, const DistillPlan& p, hipStream_t st) {
  const bool wave = p.G <= 64;
  const long long items = a.rows * a.segs, blocks = wave ? (items + 3) / 4 : items;
  const dim3 grid = grid_of(blocks);
  const size_t lds = (size_t)a.top * 12 * (wave ? 4 : 1);
  if (wave) hipLaunchKernelGGL((frl_distill_grad_kernel<T, 64, REST>), grid, dim3(256), lds, st, a);
  else if (p.G == 256) hipLaunchKernelGGL((frl_distill_grad_kernel<T, 256, REST>), grid, dim3(256), lds, st, a);
  else hipLaunchKernelGGL((frl_distill_grad_kernel<T, 1024, REST>), grid, dim3(1024), lds, st, a);
  note_kernel("frl_distill_grad_kernel<%d threads> [%lld]", wave ? 64 : p.G == 256 ? 256 : 1024, blocks);
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
  return distill_ws(desc, distill_plan(desc, true)).total;
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
  const DistillPlan p = distill_plan(desc, grad);
  const DistillWs w = distill_ws(desc, p);
  if (workspace == nullptr || ((uintptr_t)workspace & 255) != 0) { set_error("workspace must be non-NULL and 256-byte aligned"); return FRL_EWORKSPACE; }
  if (workspace_bytes < w.total) { set_error("workspace %zu B < required %zu B", workspace_bytes, w.total); return FRL_EWORKSPACE; }
  float* ws = (float*)workspace;
  hipStream_t st = (hipStream_t)hip_stream;
  DistillArgs a = distill_args(desc, bufs, p);
  const int dtype = desc->dtype;
  const bool rest = desc->kind == FRL_DISTILL_REST, split = p.split;
  a.rowloss = desc->reduction == FRL_REDUCE_NONE ? bufs->loss : ws + w.rowloss;
  a.stats = bufs->row_stats != nullptr ? bufs->row_stats : (split && grad) ? ws + w.stats : nullptr;
  a.part = ws + w.part;
  hipError_t e = hipSuccess;
  const bool reduce = desc->reduction != FRL_REDUCE_NONE, weighted = desc->reduction == FRL_REDUCE_MEAN && bufs->weights != nullptr && desc->rows > 0;
  float* inv = weighted ? (bufs->row_stats != nullptr ? bufs->row_stats + 4 * desc->rows : ws + w.inv) : nullptr;
  const bool finish = split && reduce && desc->rows <= 16 && desc->top * desc->rows * 12 <= 48 * 1024;     // the join is one workgroup and finishes the loss
  const bool have_inv = weighted && grad && !split;          // a gradient needs the weights' sum before it starts; else the last kernel adds them up
  if (have_inv) {
    hipLaunchKernelGGL(frl_distill_denom_kernel, dim3(1), dim3(1024), 0, st, bufs->weights, (long long)desc->rows, inv);
    e = hipGetLastError();
    note_kernel("frl_distill_denom_kernel");
  }
  a.inv_denom = have_inv ? inv : nullptr;
  if (e == hipSuccess && desc->rows > 0) {
    if (split) e = FRL_BY_TYPE(launch_parts)(a, finish ? bufs->loss : nullptr, inv, st);
    else e = FRL_BY_TYPE(launch_rows)(a, p, grad, st);
  }
  if (e == hipSuccess && reduce && !finish) {
    hipLaunchKernelGGL(frl_distill_sum_kernel, dim3(1), dim3(1024), 0, st, a.rowloss, (long long)desc->rows, weighted && !have_inv ? bufs->weights : nullptr, inv,
                       desc->rows > 0 ? a.denom_scale : 0.0f, bufs->loss);
    e = hipGetLastError();
    note_kernel("frl_distill_sum_kernel");
  }
  if (e == hipSuccess && split && grad) {
    a.inv_denom = inv;
    e = FRL_BY_TYPE(launch_grad)(a, p, st);
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
  const DistillPlan p = distill_plan(desc, false);
  DistillArgs a = distill_args(desc, bufs, p);
  a.stats = bufs->row_stats;
  a.g_loss = bufs->g_loss;
  a.g_stride = desc->reduction == FRL_REDUCE_NONE ? 1 : 0;
  if (desc->reduction == FRL_REDUCE_MEAN && bufs->weights != nullptr) a.inv_denom = bufs->row_stats + 4 * desc->rows;
  const int dtype = desc->dtype;
  const bool rest = desc->kind == FRL_DISTILL_REST;
  const hipError_t e = FRL_BY_TYPE(launch_grad)(a, p, (hipStream_t)hip_stream);
  if (e != hipSuccess) { set_error("distill gradient launch: %s", hipGetErrorString(e)); return FRL_EHIP; }
  return FRL_OK;
}

}  // extern "C"
