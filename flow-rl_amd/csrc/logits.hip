// Rules on rows of logits, and the choice of one entry per row: frl_logits_constrain / frl_logits_choose.
//
// Mathematics (include/flowrl_hip.h): each element takes its repetition, frequency and presence penalties from how often
// its token stands in the row's history, then its biases, then the mask; choose adds y = x / T, key = y + gumbel, the first
// argmax of key and y[token] - log sum exp y from a maximum and a sum.
//
// HBM-bound: an element is read once (and, choose, its noise), a result written once.  What must not cost a pass over the
// vocabulary of its own is the history, a list of tokens.  A group of G threads therefore owns a chunk of 8 G entries
// of one row: it counts the tokens of the history that fall into its chunk in LDS (integer adds: any order gives the same counts),
// sums the listed biases there, and applies both to the logits that it loaded into registers before it began.
#include "frl_rows.h"

namespace frl {

struct LogitsArgs {
  const void* logits; void* out; const void* history; const int32_t* lengths; const int32_t* prompt_lengths;
  const float* repetition; const float* frequency; const float* presence;
  const float* bias; const void* bias_tokens; const float* bias_values; const void* allowed;
  const float* temperature; const float* gumbel; int32_t* token; float* logprob;
  unsigned long long* part_key; float* part_m; float* part_s; float* part_y;   // choose over several chunks: one entry per (row, chunk)
  long long logits_stride, out_stride, gumbel_stride, history_stride, bias_stride, sparse_stride, mask_stride;
  float rep, freq, pres, temp;
  unsigned items, chunks;
  int vocab, ids64, L, K, mask;
};

constexpr unsigned SEEN_IN_PROMPT = 0x80000000u;

// key as an unsigned number in argmax's order (a NaN above everything, -0 equal to +0), then the index so that the lower wins
__device__ __forceinline__ unsigned long long key_of(float key, unsigned v) {
  const unsigned u = __float_as_uint(key + 0.0f);
  const unsigned o = (key != key) ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)o << 32) | (unsigned)~v;
}

// the chunk's counts: history entries t of [0, len), the first `plen` of them prompt
template <int G>
__device__ __forceinline__ void count_history(const LogitsArgs& a, long long row, int tid, unsigned v0, unsigned n, unsigned* cnt) {
  int len = a.L, plen = 0;
  if (a.lengths != nullptr) len = min(max(a.lengths[row], 0), a.L);
  if (a.prompt_lengths != nullptr) plen = min(max(a.prompt_lengths[row], 0), len);
  auto count = [&](unsigned long long id, int t) {
    const unsigned long long loc = id - v0;                 // a token below the chunk wraps round and is out of range too
    if (loc < n) {
      if (t < plen) atomicOr(&cnt[loc], SEEN_IN_PROMPT);
      else atomicAdd(&cnt[loc], 1u);
    }
  };
  if (a.ids64) {
    const long long* h = (const long long*)a.history + row * a.history_stride;
#pragma unroll 4
    for (int t = tid; t < len; t += G) count((unsigned long long)h[t], t);
  } else {
    const int* h = (const int*)a.history + row * a.history_stride;
#pragma unroll 4
    for (int t = tid; t < len; t += G) count((unsigned long long)(long long)h[t], t);
  }
}

// Listed biases, summed per token in the order of the list whatever threads hold them: a first pass counts how many entries
// name a token, a lone entry then stores its value, and of several the first one sums them all.
template <int G>
__device__ __forceinline__ void mark_listed(const LogitsArgs& a, long long row, int tid, unsigned v0, unsigned n, int* add) {
  for (int k = tid; k < a.K; k += G) {
    const unsigned long long loc = (unsigned long long)ld_id(a.bias_tokens, row * a.sparse_stride + k, a.ids64) - v0;
    if (loc < n) atomicAdd(&add[loc], 1);
  }
}
template <int G>
__device__ __forceinline__ void sum_listed(const LogitsArgs& a, long long row, int tid, unsigned v0, unsigned n, float* add) {
  const long long at = row * a.sparse_stride;
  unsigned several = 0;                                      // bit i: this thread's entry i shares its token (K <= 2048: at most 32 entries)
  for (int k = tid, i = 0; k < a.K; k += G, ++i) {
    const unsigned long long loc = (unsigned long long)ld_id(a.bias_tokens, at + k, a.ids64) - v0;
    if (loc < n && ((const int*)add)[loc] > 1) several |= 1u << i;
  }
  group_sync<G>();                                           // every count is read before a value takes its place
  for (int k = tid, i = 0; k < a.K; k += G, ++i) {
    const long long id = ld_id(a.bias_tokens, at + k, a.ids64);
    const unsigned long long loc = (unsigned long long)id - v0;
    if (loc >= n) continue;
    float s = a.bias_values[at + k];
    if (several >> i & 1u) {
      bool first = true;
      for (int j = 0; j < k && first; ++j) first = ld_id(a.bias_tokens, at + j, a.ids64) != id;
      if (!first) continue;
      for (int j = k + 1; j < a.K; ++j)
        if (ld_id(a.bias_tokens, at + j, a.ids64) == id) s += a.bias_values[at + j];
    }
    add[loc] = s;
  }
}

// allowed bits of entries v .. v + 3 (v a multiple of 4, v < vocab); bits beyond the vocabulary are unspecified
__device__ __forceinline__ unsigned allowed4(const LogitsArgs& a, long long row, unsigned v) {
  if (a.mask == FRL_MASK_WORDS) {
    const unsigned w = ((const unsigned*)a.allowed)[row * a.mask_stride + (v >> 5)];
    return (w >> (v & 31)) & 15u;
  }
  const unsigned char* b = (const unsigned char*)a.allowed + row * a.mask_stride + v;
  unsigned bits = 0;
  if ((int)v + 4 <= a.vocab) {
    const unsigned w = ldu<unsigned>(b);
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= ((w >> (8 * i) & 255u) != 0u ? 1u : 0u) << i;
  } else {
    for (int i = 0; (int)v + i < a.vocab; ++i) bits |= (b[i] != 0 ? 1u : 0u) << i;
  }
  return bits;
}

template <typename T>
__device__ __forceinline__ f32x4 load_quad(const T* p, int left, float fill) {
  if (left >= 4) return Elt<T>::load4(p);
  f32x4 v = {fill, fill, fill, fill};
  if (left > 0) v[0] = Elt<T>::get(p[0]);
  if (left > 1) v[1] = Elt<T>::get(p[1]);
  if (left > 2) v[2] = Elt<T>::get(p[2]);
  return v;
}

template <typename T, typename O, int G, bool HIST, bool SPARSE, bool CHOOSE>
__global__ void __launch_bounds__(G == 64 ? 256 : G) frl_logits_kernel(const LogitsArgs a) {
#pragma clang fp contract(off)      // each operation rounded on its own: results do not depend on which products the compiler fuses
  constexpr int CH = 8 * G, GPB = G == 64 ? 4 : 1;
  __shared__ __align__(16) unsigned cnt_all[HIST ? GPB * CH : 4];
  __shared__ __align__(16) float add_all[SPARSE ? GPB * CH : 4];
  __shared__ unsigned long long red_k[G / 64];
  __shared__ float red_m[G / 64], red_s[G / 64];
  const int tid = threadIdx.x % G, grp = threadIdx.x / G;
  unsigned* cnt = cnt_all + (HIST ? grp * CH : 0);
  float* add = add_all + (SPARSE ? grp * CH : 0);
  const float NINF = -INFINITY;

  for (unsigned item = blockIdx.x * GPB + grp; item < a.items; item += gridDim.x * GPB) {
    const long long row = item / a.chunks;
    const unsigned v0 = (item - (unsigned)row * a.chunks) * CH;
    const unsigned n = min((unsigned)a.vocab - v0, (unsigned)CH);
    const float temp = !CHOOSE ? 0.0f : a.temperature != nullptr ? a.temperature[row] : a.temp;
    const bool sampled = CHOOSE && a.gumbel != nullptr && temp > 0.0f;
    unsigned bits[2];
    f32x4 x[2], g[2], b[2];
    // everything that streams is asked for first; a quad of which nothing is allowed is not read at all
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const unsigned v = v0 + q * 4 * G + 4 * tid;
      const int left = a.vocab - (int)v;
      bits[q] = left <= 0 ? 0u : a.mask != FRL_MASK_NONE ? allowed4(a, row, v) : 15u;
      if (left < 4 && left > 0) bits[q] &= (1u << left) - 1u;
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const unsigned v = v0 + q * 4 * G + 4 * tid;
      const int left = a.vocab - (int)v;
      x[q] = f32x4{NINF, NINF, NINF, NINF};
      g[q] = b[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (bits[q] != 0u) {
        x[q] = load_quad((const T*)a.logits + row * a.logits_stride + v, left, NINF);
        if (sampled) g[q] = load_quad(a.gumbel + row * a.gumbel_stride + v, left, 0.0f);
        if (a.bias != nullptr) b[q] = load_quad(a.bias + row * a.bias_stride + v, left, 0.0f);
      }
    }
    if constexpr (HIST || SPARSE) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if constexpr (HIST) *(i32x4*)(cnt + q * 4 * G + 4 * tid) = i32x4{0, 0, 0, 0};
        if constexpr (SPARSE) *(f32x4*)(add + q * 4 * G + 4 * tid) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
      group_sync<G>();
      if constexpr (SPARSE) mark_listed<G>(a, row, tid, v0, n, (int*)add);
      if constexpr (HIST) count_history<G>(a, row, tid, v0, n, cnt);
      group_sync<G>();
      if constexpr (SPARSE) {
        sum_listed<G>(a, row, tid, v0, n, add);
        group_sync<G>();
      }
    }
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if constexpr (HIST) {
      rep = a.repetition != nullptr ? a.repetition[row] : a.rep;
      freq = a.frequency != nullptr ? a.frequency[row] : a.freq;
      pres = a.presence != nullptr ? a.presence[row] : a.pres;
    }
    const float inv = sampled ? 1.0f / (1e-6f + temp) : 1.0f;
    unsigned long long best = 0;
    float m = NINF;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const unsigned v = v0 + q * 4 * G + 4 * tid;
      i32x4 c4 = {0, 0, 0, 0};
      f32x4 a4 = {0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (HIST) c4 = *(const i32x4*)(cnt + q * 4 * G + 4 * tid);
      if constexpr (SPARSE) a4 = *(const f32x4*)(add + q * 4 * G + 4 * tid);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float t = x[q][i];
        if constexpr (HIST) {
          const unsigned c = (unsigned)c4[i] & ~SEEN_IN_PROMPT;
          if (c4[i] != 0) t = t > 0.0f ? t / rep : t * rep;
          const float f = freq * (float)c, p = c != 0u ? pres : 0.0f;
          t = t - (f + p);
        }
        if (a.bias != nullptr) t = t + b[q][i];
        if constexpr (SPARSE) t = t + a4[i];
        t = (bits[q] >> i & 1u) ? t : NINF;
        if constexpr (CHOOSE) {
          float key = t;
          if (sampled) { t = t * inv; key = t + g[q][i]; }
          if (!(t == NINF)) {
            const unsigned long long k = key_of(key, v + i);
            best = k > best ? k : best;
          }
          m = fmaxf(m, t);
        }
        x[q][i] = t;
      }
      if constexpr (!CHOOSE) {
        const int left = a.vocab - (int)v;
        O* o = (O*)a.out + row * a.out_stride + v;
        if (left >= 4) Elt<O>::store4(o, x[q]);
        else {
          if (left > 0) o[0] = Elt<O>::put(x[q][0]);
          if (left > 1) o[1] = Elt<O>::put(x[q][1]);
          if (left > 2) o[2] = Elt<O>::put(x[q][2]);
        }
      }
    }
    if constexpr (CHOOSE) {
      constexpr float LOG2E = 1.4426950408889634f;
      m = group_reduce<MaxOp, G>(m, red_m);
      const float m0 = m == NINF ? 0.0f : m;
      float s = 0.0f;
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) s += __builtin_amdgcn_exp2f((x[q][i] - m0) * LOG2E);
      best = group_reduce<MaxOp, G>(best, red_k);
      s = group_reduce<SumOp, G>(s, red_s);
      // the thread that holds the winner answers; thread 0 where there is none
      const unsigned win = ~(unsigned)best;
      bool mine = best == 0 && tid == 0;
      float y = NINF;
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (best != 0 && win == v0 + q * 4 * G + 4 * tid + i) { mine = true; y = x[q][i]; }
      if (mine) {
        if (a.chunks == 1) {
          a.token[row] = best != 0 ? (int32_t)win : -1;
          if (a.logprob != nullptr) a.logprob[row] = best != 0 ? (y - m) - logf(s) : NINF;
        } else {
          a.part_key[item] = best;
          a.part_m[item] = m;
          a.part_s[item] = s;
          a.part_y[item] = y;
        }
      }
      if constexpr (G > 64) __syncthreads();                 // the next item writes red_* again
    }
  }
}

// the chunks of a row joined: one wave per row, a fixed order
__global__ void __launch_bounds__(256) frl_logits_join_kernel(const LogitsArgs a, long long rows) {
  constexpr float LOG2E = 1.4426950408889634f;
  const int lane = threadIdx.x & 63;
  for (long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (long long)gridDim.x * 4) {
    const long long at = row * a.chunks;
    unsigned long long best = 0;
    float m = -INFINITY, y = -INFINITY;
    for (unsigned c = lane; c < a.chunks; c += 64) {
      const unsigned long long k = a.part_key[at + c];
      if (k > best) { best = k; y = a.part_y[at + c]; }
      m = fmaxf(m, a.part_m[at + c]);
    }
    m = wave_reduce<MaxOp>(m);
    const float m0 = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
    for (unsigned c = lane; c < a.chunks; c += 64) s += a.part_s[at + c] * __builtin_amdgcn_exp2f((a.part_m[at + c] - m0) * LOG2E);
    s = wave_reduce<SumOp>(s);
    const unsigned long long all = wave_reduce<MaxOp>(best);
    if (all == 0 ? lane == 0 : best == all) {                // indices differ between chunks, so one lane holds the winner
      a.token[row] = all != 0 ? (int32_t) ~(unsigned)all : -1;
      if (a.logprob != nullptr) a.logprob[row] = all != 0 ? (y - m) - logf(s) : -INFINITY;
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------

// Threads per (row, chunk).
static int logits_group(long long rows, int vocab) {
  if (vocab <= 512) return 64;
  const long long wide = rows * ((vocab + 8191) / 8192);
  return (vocab > 4096 && wide >= 512) ? 1024 : 256;
}

template <typename T, typename O, bool CHOOSE>
static hipError_t launch_logits(const LogitsArgs& a, int G, unsigned grid, hipStream_t stream) {
#define FRL_LAUNCH(g, h, s)                                                                                             \
  hipLaunchKernelGGL((frl_logits_kernel<T, O, g, h, s, CHOOSE>), dim3(grid), dim3(g == 64 ? 256 : g), 0, stream, a)
#define FRL_PICK(g)                                                                                                     \
  do {                                                                                                                  \
    if (a.L > 0 && a.K > 0) FRL_LAUNCH(g, true, true);                                                                  \
    else if (a.L > 0) FRL_LAUNCH(g, true, false);                                                                       \
    else if (a.K > 0) FRL_LAUNCH(g, false, true);                                                                       \
    else FRL_LAUNCH(g, false, false);                                                                                   \
  } while (0)
  if (G == 64) FRL_PICK(64);
  else if (G == 256) FRL_PICK(256);
  else FRL_PICK(1024);
#undef FRL_PICK
#undef FRL_LAUNCH
  return hipGetLastError();
}

static int logits_validate(const FrlLogitsDesc* d, bool choose) {
  if (d == nullptr) { set_error("logits: desc is NULL"); return FRL_EINVAL; }
  if (d->abi_version != FRL_ABI_VERSION) { set_error("desc.abi_version %d != library %d", d->abi_version, FRL_ABI_VERSION); return FRL_EINVAL; }
  if (d->dtype < FRL_ELT_F32 || d->dtype > FRL_ELT_F16) { set_error("logits: dtype %d invalid", d->dtype); return FRL_EINVAL; }
  if (!choose && d->out_dtype != d->dtype && d->out_dtype != FRL_ELT_F32) { set_error("logits: out_dtype %d: the logits' own or FRL_ELT_F32", d->out_dtype); return FRL_EINVAL; }
  if (d->vocab < 1 || d->rows < 0) { set_error("logits: rows %lld / vocab %d invalid", (long long)d->rows, d->vocab); return FRL_EINVAL; }
  if (d->history_len < 0) { set_error("logits: history_len %d invalid", d->history_len); return FRL_EINVAL; }
  if (d->n_sparse < 0) { set_error("logits: n_sparse %d invalid", d->n_sparse); return FRL_EINVAL; }
  if (d->n_sparse > FRL_LOGITS_MAX_SPARSE) { set_error("logits: %d listed biases per row > %d (use the dense bias)", d->n_sparse, FRL_LOGITS_MAX_SPARSE); return FRL_EUNSUPPORTED; }
  if (d->mask < FRL_MASK_NONE || d->mask > FRL_MASK_BYTES) { set_error("logits: mask %d invalid", d->mask); return FRL_EINVAL; }
  if (d->vocab > (1 << 30)) { set_error("logits: vocab %d > 2^30", d->vocab); return FRL_EUNSUPPORTED; }
  const int G = logits_group(d->rows, d->vocab);
  const long long chunks = ((long long)d->vocab + 8 * G - 1) / (8 * G);
  if (d->rows > (1LL << 30) / chunks) { set_error("logits: %lld rows of %d entries are more than 2^30 chunks in one call", (long long)d->rows, d->vocab); return FRL_EUNSUPPORTED; }
  const long long V = d->vocab;
  if (d->rows > 1 && d->logits_stride < V) { set_error("logits: row stride %lld < vocab %lld", (long long)d->logits_stride, V); return FRL_EINVAL; }
  if (d->rows > 1 && !choose && d->out_stride < V) { set_error("logits: out row stride %lld < vocab %lld", (long long)d->out_stride, V); return FRL_EINVAL; }
  return FRL_OK;
}

static int logits_fill(const FrlLogitsDesc* d, const FrlLogitsBufs* b, bool choose, LogitsArgs& a, int& G) {
  if (b == nullptr || b->logits == nullptr) { set_error("logits: bufs.logits is NULL"); return FRL_EINVAL; }
  if (d->history_len > 0 && b->history == nullptr) { set_error("logits: bufs.history is NULL (history_len %d)", d->history_len); return FRL_EINVAL; }
  if (d->n_sparse > 0 && (b->bias_tokens == nullptr || b->bias_values == nullptr)) { set_error("logits: bufs.bias_tokens / bias_values is NULL (n_sparse %d)", d->n_sparse); return FRL_EINVAL; }
  if ((d->mask != FRL_MASK_NONE) != (b->allowed != nullptr)) { set_error("logits: bufs.allowed must be non-NULL exactly when desc.mask is set"); return FRL_EINVAL; }
  if (d->history_len > 0 && b->repetition == nullptr && !(d->repetition > 0.0f)) { set_error("logits: repetition %g must be > 0", d->repetition); return FRL_EINVAL; }
  a = LogitsArgs{b->logits, b->out, b->history, b->lengths, b->prompt_lengths, b->repetition, b->frequency, b->presence,
                 b->bias, b->bias_tokens, b->bias_values, b->allowed, b->temperature, b->gumbel, b->token, b->logprob,
                 nullptr, nullptr, nullptr, nullptr,
                 d->logits_stride, d->out_stride, d->gumbel_stride, d->history_stride, d->bias_stride, d->sparse_stride, d->mask_stride,
                 d->repetition, d->frequency, d->presence, d->temperature, 0, 0, d->vocab, d->ids64, d->history_len, d->n_sparse, d->mask};
  G = logits_group(d->rows, d->vocab);
  a.chunks = (unsigned)((d->vocab + 8LL * G - 1) / (8 * G));
  a.items = (unsigned)(d->rows * a.chunks);
  return FRL_OK;
}

// Enough workgroups for every CU to be full many times over; beyond that a workgroup takes several items.
static unsigned logits_grid(const LogitsArgs& a, int G) {
  const unsigned groups = G == 64 ? (a.items + 3) / 4 : a.items;
  return groups < (1u << 20) ? groups : (1u << 20);
}

static size_t logits_workspace(const FrlLogitsDesc* d) {
  const int G = logits_group(d->rows, d->vocab);
  const size_t chunks = (size_t)((d->vocab + 8LL * G - 1) / (8 * G));
  const size_t items = chunks > 1 ? (size_t)d->rows * chunks : 0;
  return (items * 20 + 511) / 256 * 256;
}

}  // namespace frl

using namespace frl;

extern "C" {

int frl_logits_constrain(const FrlLogitsDesc* desc, const FrlLogitsBufs* bufs, void* hip_stream) {
  clear_kernels();
  int rc = logits_validate(desc, false);
  if (rc != FRL_OK) return rc;
  if (desc->rows == 0) return FRL_OK;
  LogitsArgs a;
  int G;
  if ((rc = logits_fill(desc, bufs, false, a, G)) != FRL_OK) return rc;
  if (a.out == nullptr) { set_error("logits: bufs.out is NULL"); return FRL_EINVAL; }
  // in place is the very same rows; any other overlap would be read after it was written
  const size_t in_elt = desc->dtype == FRL_ELT_F32 ? 4 : 2, out_elt = desc->out_dtype == FRL_ELT_F32 ? 4 : 2;
  const uintptr_t i0 = (uintptr_t)a.logits, i1 = i0 + ((size_t)(desc->rows - 1) * desc->logits_stride + desc->vocab) * in_elt;
  const uintptr_t o0 = (uintptr_t)a.out, o1 = o0 + ((size_t)(desc->rows - 1) * desc->out_stride + desc->vocab) * out_elt;
  const bool same = i0 == o0 && desc->dtype == desc->out_dtype && (desc->logits_stride == desc->out_stride || desc->rows == 1);
  if (!same && i0 < o1 && o0 < i1) { set_error("logits: out overlaps logits without being the same rows"); return FRL_EINVAL; }
  const unsigned grid = logits_grid(a, G);
  const bool f32 = desc->out_dtype == FRL_ELT_F32;
  hipStream_t st = (hipStream_t)hip_stream;
  hipError_t e = hipErrorInvalidValue;
  if (desc->dtype == FRL_ELT_F32) e = launch_logits<float, float, false>(a, G, grid, st);
  else if (desc->dtype == FRL_ELT_BF16) e = f32 ? launch_logits<Bf16, float, false>(a, G, grid, st) : launch_logits<Bf16, Bf16, false>(a, G, grid, st);
  else e = f32 ? launch_logits<F16, float, false>(a, G, grid, st) : launch_logits<F16, F16, false>(a, G, grid, st);
  if (e != hipSuccess) { set_error("logits constrain launch: %s", hipGetErrorString(e)); return FRL_EHIP; }
  note_kernel("frl_logits_kernel<constrain, %d threads> [%u]", G, grid);
  return FRL_OK;
}

size_t frl_logits_workspace_bytes(const FrlLogitsDesc* desc) {
  return logits_validate(desc, true) == FRL_OK ? logits_workspace(desc) : 0;
}

int frl_logits_choose(const FrlLogitsDesc* desc, const FrlLogitsBufs* bufs, void* workspace, size_t workspace_bytes, void* hip_stream) {
  clear_kernels();
  int rc = logits_validate(desc, true);
  if (rc != FRL_OK) return rc;
  if (desc->rows == 0) return FRL_OK;
  LogitsArgs a;
  int G;
  if ((rc = logits_fill(desc, bufs, true, a, G)) != FRL_OK) return rc;
  if (a.token == nullptr) { set_error("logits: bufs.token is NULL"); return FRL_EINVAL; }
  if (a.gumbel != nullptr && desc->rows > 1 && desc->gumbel_stride < desc->vocab) { set_error("logits: gumbel row stride %lld < vocab %d", (long long)desc->gumbel_stride, desc->vocab); return FRL_EINVAL; }
  if (a.gumbel == nullptr && a.temperature == nullptr && desc->temperature > 0.0f) { set_error("logits: temperature %g > 0 draws: bufs.gumbel is NULL", desc->temperature); return FRL_EINVAL; }
  if (a.chunks > 1) {
    if (workspace == nullptr || ((uintptr_t)workspace & 255) != 0) { set_error("workspace must be non-NULL and 256-byte aligned"); return FRL_EWORKSPACE; }
    if (workspace_bytes < logits_workspace(desc)) { set_error("workspace %zu B < required %zu B", workspace_bytes, logits_workspace(desc)); return FRL_EWORKSPACE; }
    a.part_key = (unsigned long long*)workspace;
    a.part_m = (float*)(a.part_key + a.items);
    a.part_s = a.part_m + a.items;
    a.part_y = a.part_s + a.items;
  }
  const unsigned grid = logits_grid(a, G);
  hipStream_t st = (hipStream_t)hip_stream;
  hipError_t e = desc->dtype == FRL_ELT_F32 ? launch_logits<float, float, true>(a, G, grid, st)
               : desc->dtype == FRL_ELT_BF16 ? launch_logits<Bf16, float, true>(a, G, grid, st) : launch_logits<F16, float, true>(a, G, grid, st);
  if (e != hipSuccess) { set_error("logits choose launch: %s", hipGetErrorString(e)); return FRL_EHIP; }
  note_kernel("frl_logits_kernel<choose, %d threads> [%u]", G, grid);
  if (a.chunks > 1) {
    const long long blocks = (desc->rows + 3) / 4;
    const unsigned jg = (unsigned)(blocks < 65536 ? blocks : 65536);
    hipLaunchKernelGGL(frl_logits_join_kernel, dim3(jg), dim3(256), 0, st, a, (long long)desc->rows);
    e = hipGetLastError();
    if (e != hipSuccess) { set_error("logits join launch: %s", hipGetErrorString(e)); return FRL_EHIP; }
    note_kernel("frl_logits_join_kernel [%u]", jg);
  }
  return FRL_OK;
}

}  // extern "C"
