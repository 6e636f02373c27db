// Rules on rows of logits, and the choice of one entry per row: frl_logits_constrain / frl_logits_choose.
//
// Mathematics (include/flowrl_hip.h): each element takes its repetition, frequency and presence penalties from how often
// its token stands in the row's history, then its biases, then the mask; choose adds y = x / T, key = y + gumbel, the first
// argmax of key and y[token] - log sum exp y from a maximum and a sum.
//
// HBM-bound where the lists are short: an element is read once (and, choose, its noise), a result written once.  What must not cost a pass over the
// vocabulary of its own is the lists, a history of tokens and biases by token.  A group of G threads (a wave up to a workgroup of 1024) takes
// consecutive chunks of 8 G entries of one row.  For each it counts the history's tokens that fall into the chunk in one LDS word per entry
// (integer adds: any order gives the same counts), puts the number of a listed bias beside the count, and applies both to the
// logits, which are on their way meanwhile.  Two sets of words take turns, so a chunk costs one barrier; a choice keeps its maximum and sum in
// registers from chunk to chunk and reduces them once.
// Measured: constraining 512 x 131072 f32 with every rule 105 us, 5.2 TB/s of the 5.4 a copy reaches, by HBM; a choice of 256 x 131072 bf16
// with every rule 50 us and 4.6 for the join, 3.5 TB/s, mostly by vector issue (40 instructions an entry, 35 of the 50 us: nearly every wave has a
// listed entry at nearly every place, so it is the lists' arithmetic that counts; a loop over what each lane has listed instead took 60 us);
// greedy and without lists 24 us and 4.6 for the join, by vector issue (22 instructions an entry, 20 of the 24 us; one of them is the
// exponential); a few rows 7 us, by the latency of lists, LDS and logits.
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
  int vocab, ids64, L, K, mask, eager;
  long long items;          // rows x parts
  int chunks, per, parts;   // of a row: chunks of 8 G entries, `per` of them to a part (one group's work)
};

// One LDS word per entry of a chunk: bit 31 the token stands in the prompt; bits 19..30 one more than the slot of its listed bias, 0 for none;
// bits 0..18 how often it was generated.  Without listed biases the count has all 31 bits.
constexpr unsigned SEEN_IN_PROMPT = 0x80000000u;
constexpr int SLOT_SHIFT = 19;
constexpr unsigned COUNT_MASK = (1u << SLOT_SHIFT) - 1u, SLOT_MASK = 0xfffu;
constexpr int MAX_HISTORY_WITH_SLOTS = (1 << SLOT_SHIFT) - 1;
constexpr int HIST_REGS = 4;                               // history entries a thread keeps; longer histories are read again for every chunk
constexpr unsigned NO_TOKEN = 0x7fffffffu;                 // beyond every vocabulary (at most 2^30) from any chunk's first entry

// key as an unsigned number in argmax's order (a NaN above everything, -0 equal to +0), then the index so that the lower wins
__device__ __forceinline__ unsigned long long key_of(float key, unsigned v) {
  const unsigned u = __float_as_uint(key + 0.0f);
  const unsigned o = (key != key) ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)o << 32) | (unsigned)~v;
}

// A seen token's logit: x / d where it is positive, else x * d; r = 1 / d.  The quotient's error is brought back in by one fma (Markstein), which
// leaves the correctly rounded quotient but where it is subnormal; an infinite quotient stays.  Of a subnormal d there may be no reciprocal; it is refused.
__device__ __forceinline__ float pushed_down(float x, float d, float r) {
  const bool above = x > 0.0f;
  const float q = x * (above ? r : d);
  const float q2 = __builtin_fmaf(__builtin_fmaf(-q, d, x), r, q);
  return above && q2 == q2 ? q2 : q;
}

// Entry t of the history: its token (NO_TOKEN for padding), bit 31 set in the prompt
__device__ __forceinline__ unsigned history_entry(const LogitsArgs& a, const void* h, int t, int plen) {
  const long long id = ld_id(h, t, a.ids64);
  return id >= 0 && id < a.vocab ? (unsigned)id | (t < plen ? SEEN_IN_PROMPT : 0u) : NO_TOKEN;
}

__device__ __forceinline__ void count_entry(unsigned e, unsigned v0, unsigned n, unsigned* cnt) {
  const unsigned loc = (e & ~SEEN_IN_PROMPT) - v0;          // tokens below the chunk wrap round and are out of range too
  if (loc < n) {
    if (e & SEEN_IN_PROMPT) atomicOr(&cnt[loc], SEEN_IN_PROMPT);
    else atomicAdd(&cnt[loc], 1u);
  }
}

// The row's listed biases, once: tokens and values into LDS, a token named several times summed in the order of the list into its first
// entry (the others become NO_TOKEN).  Whether any is, a table of the tokens finds out; `table` is the chunks' words, free and zero before and after.
template <int G>
__device__ __forceinline__ void stage_listed(const LogitsArgs& a, long long row, int tid, unsigned* table, unsigned* tok, float* val, int* several) {
  constexpr unsigned SLOTS = 8 * G;                        // a power of two
  const long long at = row * a.sparse_stride;
  if (tid == 0) *several = a.K > (int)SLOTS / 2;
  for (int k = tid; k < a.K; k += G) {
    const long long id = ld_id(a.bias_tokens, at + k, a.ids64);
    tok[k] = id >= 0 && id < a.vocab ? (unsigned)id : NO_TOKEN;
    val[k] = a.bias_values[at + k];
  }
  group_sync<G>();
  if (a.K <= (int)SLOTS / 2) {                             // at most half full: a free slot is always found
    for (int k = tid; k < a.K; k += G) {
      if (tok[k] == NO_TOKEN) continue;
      const unsigned mine = tok[k] + 1u;
      // the product's highest bits: its lowest would be the token's own, the same for tokens a multiple of SLOTS apart
      for (unsigned i = mine * 2654435761u >> (32 - __builtin_ctz(SLOTS)), probe = 0; probe < SLOTS; ++probe, ++i) {
        const unsigned was = atomicCAS(&table[i % SLOTS], 0u, mine);
        if (was == mine) *several = 1;
        if (was == 0u || was == mine) break;
      }
    }
    group_sync<G>();
#pragma unroll
    for (int q = 0; q < 2; ++q) *(i32x4*)(table + q * 4 * G + 4 * tid) = i32x4{0, 0, 0, 0};
  }
  group_sync<G>();
  if (*several != 0) {
    unsigned drop = 0;                                     // bit i: this thread's entry i is not its token's first (K <= 2048: at most 32 entries)
    for (int k = tid, i = 0; k < a.K; k += G, ++i) {
      const unsigned t = tok[k];
      if (t == NO_TOKEN) continue;
      bool first = true;
      for (int j = 0; j < k && first; ++j) first = tok[j] != t;
      if (!first) { drop |= 1u << i; continue; }
      float s = a.bias_values[at + k];
      for (int j = k + 1; j < a.K; ++j)
        if (tok[j] == t) s += a.bias_values[at + j];
      val[k] = s;
    }
    group_sync<G>();
    for (int k = tid, i = 0; k < a.K; k += G, ++i)
      if (drop >> i & 1u) tok[k] = NO_TOKEN;
    group_sync<G>();
  }
}

// allowed bits of entries v .. v + 3 (v a multiple of 4), of which `left` are in the vocabulary
template <bool FULL>
__device__ __forceinline__ unsigned allowed4(const LogitsArgs& a, const void* mask, unsigned v, int left) {
  if (!FULL && left <= 0) return 0u;
  unsigned bits = 15u;
  if (a.mask == FRL_MASK_WORDS) {
    bits = (((const unsigned*)mask)[v >> 5] >> (v & 31)) & 15u;
  } else if (a.mask == FRL_MASK_BYTES) {
    const unsigned char* b = (const unsigned char*)mask + v;
    if (FULL || left >= 4) {
      unsigned w = ldu<unsigned>(b);
      w |= w >> 4;
      w |= w >> 2;
      w |= w >> 1;
      bits = ((w & 0x01010101u) * 0x10204080u) >> 28;       // byte i's lowest bit to bit i
    } else {
      bits = 0u;
      for (int i = 0; i < left; ++i) bits |= (b[i] != 0 ? 1u : 0u) << i;
    }
  }
  return FULL || left >= 4 ? bits : bits & ((1u << left) - 1u);
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

// The running answer of a thread over its entries, in index order: the best key and where, its y, and the sum of exponentials
struct Choice {
  float key = -INFINITY, y = -INFINITY, m = -INFINITY, s = 0.0f;
  unsigned v = 0xffffffffu;
  bool nan = false;         // v is its first NaN
};
constexpr float LOG2E = 1.4426950408889634f;

// what the chunks of a row that one group took come to, in the join's terms
__device__ __forceinline__ void answer(const LogitsArgs& a, long long row, unsigned long long best, float m, float s, float y) {
  a.token[row] = best != 0 ? (int32_t) ~(unsigned)best : -1;
  if (a.logprob == nullptr) return;
  const Shift sh(m, LOG2E);
  const float d = sh.fast ? __builtin_fmaf(y, LOG2E, -sh.M) : (y - m) * LOG2E;
  a.logprob[row] = best != 0 ? (d - __builtin_amdgcn_logf(s)) * 0.69314718f : -INFINITY;
}

// Four elements as they lie in memory: a two-byte type keeps them in two registers until they are used.
template <typename T>
struct Packed4 {
  u32x2 r;
  __device__ __forceinline__ void load(const T* p, int left) {
    if (left >= 4) { r = ldu_nt<u32x2>(p); return; }
    const unsigned ninf = Elt<T>::put(-INFINITY).u;
    const unsigned e0 = left > 0 ? p[0].u : ninf, e1 = left > 1 ? p[1].u : ninf, e2 = left > 2 ? p[2].u : ninf;
    r = u32x2{e0 | e1 << 16, e2 | ninf << 16};
  }
  __device__ __forceinline__ void none() { const unsigned ninf = Elt<T>::put(-INFINITY).u; r = u32x2{ninf | ninf << 16, ninf | ninf << 16}; }
  __device__ __forceinline__ f32x4 get() const {
    return f32x4{Elt<T>::get(T{(unsigned short)r[0]}), Elt<T>::get(T{(unsigned short)(r[0] >> 16)}),
                 Elt<T>::get(T{(unsigned short)r[1]}), Elt<T>::get(T{(unsigned short)(r[1] >> 16)})};
  }
};
template <>
struct Packed4<float> {
  f32x4 r;
  __device__ __forceinline__ void load(const float* p, int left) { r = left >= 4 ? ldu_nt<f32x4>(p) : load_quad(p, left, -INFINITY); }
  __device__ __forceinline__ void none() { r = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY}; }
  __device__ __forceinline__ f32x4 get() const { return r; }
};

template <typename T, typename O, int G, bool HIST, bool SPARSE, bool CHOOSE>
__global__ void __launch_bounds__(G == 64 ? 256 : G, 8) frl_logits_kernel(const LogitsArgs a) {
  constexpr int CH = 8 * G, GPB = G == 64 ? 4 : 1;
  constexpr bool WORDS = HIST || SPARSE;
  __shared__ __align__(16) unsigned cnt_all[WORDS ? GPB * 2 * CH : 4];
  extern __shared__ __align__(16) unsigned lists[];         // tokens, then values, of the listed biases
  __shared__ int several_all[GPB];
  __shared__ unsigned long long red_k[G / 64];
  __shared__ float red_m[G / 64], red_s[G / 64];
  const int tid = threadIdx.x % G, grp = G == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  unsigned* cnt = cnt_all + (WORDS ? grp * 2 * CH : 0);
  unsigned* tok = lists + (SPARSE ? grp * 2 * a.K : 0);
  float* val = (float*)(tok + (SPARSE ? a.K : 0));
  const float NINF = -INFINITY;

  const long long item = block_index() * GPB + grp;
  if (item >= a.items) return;
  const long long row = item / a.parts;
  const int part = (int)(item - row * a.parts);
  const int c0 = part * a.per, c1 = min(c0 + a.per, a.chunks);
  const T* z = (const T*)a.logits + row * a.logits_stride;
  const float temp = !CHOOSE ? 0.0f : a.temperature != nullptr ? a.temperature[row] : a.temp;
  const bool sampled = CHOOSE && a.gumbel != nullptr && temp > 0.0f;
  const float inv = sampled ? fmaxf(1.0f / (1e-6f + temp), 1.17549435e-38f) : 1.0f;      // never 0: an infinite temperature leaves -inf what it is
  const float* noise = sampled ? a.gumbel + row * a.gumbel_stride : nullptr;

  const void* mask = a.mask == FRL_MASK_WORDS ? (const void*)((const unsigned*)a.allowed + row * a.mask_stride) : (const void*)((const unsigned char*)a.allowed + row * a.mask_stride);
  const int whole = a.vocab / CH;                           // chunks before this one lie in the vocabulary altogether
  auto bits_of = [&](int c, int q, int t) -> unsigned {
    const unsigned v = (unsigned)c * CH + q * 4 * G + 4 * t;
    return c >= c1 ? 0u : c < whole ? allowed4<true>(a, mask, v, 4) : allowed4<false>(a, mask, v, a.vocab - (int)v);
  };
  unsigned bits[2] = {bits_of(c0, 0, tid), bits_of(c0, 1, tid)};

  int len = 0, plen = 0;
  unsigned mine[HIST ? HIST_REGS : 1];
  float rep = 1.0f, rrep = 1.0f, freq = 0.0f, pres = 0.0f;
  const void* h = nullptr;
  if constexpr (HIST) {
    h = (const char*)a.history + row * a.history_stride * (a.ids64 ? 8 : 4);
    len = a.lengths != nullptr ? min(max(a.lengths[row], 0), a.L) : a.L;
    plen = a.prompt_lengths != nullptr ? min(max(a.prompt_lengths[row], 0), len) : 0;
#pragma unroll
    for (int i = 0; i < HIST_REGS; ++i) mine[i] = tid + i * G < len ? history_entry(a, h, tid + i * G, plen) : NO_TOKEN;
    rep = a.repetition != nullptr ? a.repetition[row] : a.rep;
    freq = a.frequency != nullptr ? a.frequency[row] : a.freq;
    pres = a.presence != nullptr ? a.presence[row] : a.pres;
    rrep = 1.0f / rep;
  }
  if constexpr (WORDS) {
#pragma unroll
    for (int q = 0; q < 4; ++q) *(i32x4*)(cnt + q * 4 * G + 4 * tid) = i32x4{0, 0, 0, 0};
    if constexpr (SPARSE) stage_listed<G>(a, row, tid, cnt, tok, val, several_all + grp);
    group_sync<G>();
  }

  Choice ch;
  float ahead = NINF;                                       // the best key that any lane of the wave has
  auto chunk = [&](int c, auto full) {
    constexpr bool FULL = decltype(full)::value;
    const int t0 = fresh(tid);
    const unsigned v0 = (unsigned)c * CH, n = FULL ? (unsigned)CH : (unsigned)a.vocab - v0;
    Packed4<T> raw[2];
    f32x4 g[2];
    // everything that streams is asked for first.  In a batch that fills the chip a quad of which nothing is allowed is not read at all; a small one
    // does not wait for its mask
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const unsigned v = v0 + q * 4 * G + 4 * t0;
      const int left = FULL ? 4 : a.vocab - (int)v;
      raw[q].none();
      g[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (a.eager ? left > 0 : bits[q] != 0u) {
        raw[q].load((const T*)((const char*)z + v * (unsigned)sizeof(T)), left);
        if (sampled) g[q] = load_quad((const float*)((const char*)noise + v * 4u), left, 0.0f);
      }
    }
    const unsigned now[2] = {bits[0], bits[1]};
    bits[0] = bits_of(c + 1, 0, t0);
    bits[1] = bits_of(c + 1, 1, t0);
    unsigned* w = cnt + (WORDS ? ((c - c0) & 1) * CH : 0);
    if constexpr (HIST) {
#pragma unroll
      for (int i = 0; i < HIST_REGS; ++i) count_entry(mine[i], v0, n, w);
      for (int t = t0 + HIST_REGS * G; t < len; t += G) count_entry(history_entry(a, h, t, plen), v0, n, w);
    }
    if constexpr (SPARSE) {
      for (int k = t0; k < a.K; k += G) {
        const unsigned loc = tok[k] - v0;
        if (loc < n) atomicAdd(&w[loc], (unsigned)(k + 1) << SLOT_SHIFT);
      }
    }
    float x[2][4], top[2];
    if constexpr (WORDS) group_sync<G>();                   // the words are complete; the other set was cleared by the threads that read it
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const unsigned v = v0 + q * 4 * G + 4 * t0;
      const int left = FULL ? 4 : a.vocab - (int)v;
      const f32x4 in = raw[q].get();
      i32x4 w4 = {0, 0, 0, 0};
      if constexpr (WORDS) {
        w4 = *(const i32x4*)(w + q * 4 * G + 4 * t0);
        *(i32x4*)(w + q * 4 * G + 4 * t0) = i32x4{0, 0, 0, 0};
      }
      f32x4 b = {-0.0f, -0.0f, -0.0f, -0.0f};               // t + -0 is t, whatever t is
      if (a.bias != nullptr && now[q] != 0u) b = load_quad(a.bias + row * a.bias_stride + v, left, 0.0f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float t = in[i];
        const unsigned word = (unsigned)w4[i];
        if (WORDS && word != 0u) {                          // few tokens are listed: often no lane of a wave has one, and the wave skips this
          if constexpr (HIST) {
            const unsigned count = SPARSE ? word & COUNT_MASK : word & ~SEEN_IN_PROMPT;
            const unsigned seen = SPARSE ? word & (SEEN_IN_PROMPT | COUNT_MASK) : word;
            t = seen != 0u ? pushed_down(t, rep, rrep) : t;
            t = t - (freq * (float)count + (count != 0u ? pres : 0.0f));
          }
          t = t + b[i];
          if constexpr (SPARSE) {
            const unsigned slot = word >> SLOT_SHIFT & SLOT_MASK;
            if (slot != 0u) t = t + val[slot - 1u];
          }
        } else {
          t = t + b[i];
        }
        const unsigned keep = (unsigned)((int)(now[q] << (31 - i)) >> 31);
        x[q][i] = __uint_as_float((__float_as_uint(t) & keep) | (0xff800000u & ~keep));
      }
      if constexpr (!CHOOSE) {
        O* o = (O*)((char*)a.out + row * a.out_stride * (long long)sizeof(O) + v * (unsigned)sizeof(O));
        const f32x4 to = {x[q][0], x[q][1], x[q][2], x[q][3]};
        if (left >= 4) Elt<O>::store4(o, to);
        else {
          if (left > 0) o[0] = Elt<O>::put(to[0]);
          if (left > 1) o[1] = Elt<O>::put(to[1]);
          if (left > 2) o[2] = Elt<O>::put(to[2]);
        }
      } else {
        float key[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[q][i] = x[q][i] * inv;                          // a greedy row: times 1, plus 0
          key[i] = x[q][i] + g[q][i];
        }
        top[q] = max_of<4>(x[q], NINF);
        // A later quad of the wave has the greater indices, so only what is ahead of every lane's best counts; that soon becomes rare
        if (__builtin_amdgcn_ballot_w64(max_of<4>(key, NINF) > ahead) != 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool better = key[i] > ch.key;            // the first of equal keys stays; against a NaN nothing is better
            ch.key = better ? key[i] : ch.key;
            ch.y = better ? x[q][i] : ch.y;
            ch.v = better ? v + i : ch.v;
          }
          ahead = wave_reduce<MaxOp>(ch.key);
        }
      }
      __builtin_amdgcn_sched_barrier(0);                    // one quad at a time: 64 registers let two workgroups of 1024 share a CU
    }
    if constexpr (CHOOSE) {
      // The sum's shift need not be the maximum: it follows once that is 30 ahead, where the exponentials (below 2^44) are far from overflowing
      const float bm = fmaxf(top[0], top[1]);
      if (bm > ch.m + 30.0f) {
        if (ch.m != NINF) ch.s *= Shift(bm, LOG2E).from(Shift(ch.m, LOG2E));
        ch.m = bm;
      }
      Shift sh(ch.m == NINF ? 0.0f : ch.m, LOG2E);
      sh.fast = __builtin_amdgcn_ballot_w64(!sh.fast) == 0;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float e[4] = {x[q][0], x[q][1], x[q][2], x[q][3]};
        sh.exps<4>(e);
        const float sum = (e[0] + e[1]) + (e[2] + e[3]);
        ch.s += sum;
        if (sum != sum && !ch.nan) {                        // a NaN among the four, or infinity less infinity
#pragma unroll
          for (int i = 3; i >= 0; --i)
            if (x[q][i] != x[q][i]) { ch.nan = true; ch.v = v0 + q * 4 * G + 4 * t0 + i; ch.key = ch.y = x[q][i]; }
        }
      }
    }
  };
  for (int c = c0; c < min(c1, whole); ++c) chunk(c, std::true_type());
  if (c1 > whole) chunk(whole, std::false_type());

  if constexpr (CHOOSE) {
    const float m = group_reduce<MaxOp, G>(ch.m, red_m);
    if (ch.m != NINF) ch.s *= Shift(m, LOG2E).from(Shift(ch.m, LOG2E));
    unsigned long long best = ch.v != 0xffffffffu ? key_of(ch.key, ch.v) : 0ull;
    best = group_reduce<MaxOp, G>(best, red_k);
    const float s = group_reduce<SumOp, G>(ch.s, red_s);
    const bool none = best == 0;
    if (none ? tid == 0 : ch.v == ~(unsigned)best) {        // the thread that holds the winner answers
      if (a.parts == 1) answer(a, row, best, m, s, ch.y);
      else {
        a.part_key[item] = best;
        a.part_m[item] = m;
        a.part_s[item] = s;
        a.part_y[item] = ch.y;
      }
    }
  }
}

// the parts of a row joined: one wave per row, a fixed order (2 to 5 us, by latency)
__global__ void __launch_bounds__(256) frl_logits_join_kernel(const LogitsArgs a, long long rows) {
  const int lane = threadIdx.x & 63;
  const long long row = block_index() * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const long long at = row * a.parts;
  unsigned long long best = 0;
  float m = -INFINITY, y = -INFINITY;
  for (int c = lane; c < a.parts; c += 64) {
    const unsigned long long k = a.part_key[at + c];
    if (k > best) { best = k; y = a.part_y[at + c]; }
    m = fmaxf(m, a.part_m[at + c]);
  }
  m = wave_reduce<MaxOp>(m);
  const Shift sh(m, LOG2E);
  float s = 0.0f;
  for (int c = lane; c < a.parts; c += 64) {
    const float mc = a.part_m[at + c];
    s += a.part_s[at + c] * (mc == -INFINITY ? 1.0f : sh.from(Shift(mc, LOG2E)));      // a part of -inf alone has a sum of 0 (or NaN)
  }
  s = wave_reduce<SumOp>(s);
  const unsigned long long all = wave_reduce<MaxOp>(best);
  if (all == 0 ? lane == 0 : best == all) answer(a, row, all, m, s, y);                // indices differ between parts, so one lane holds the winner
}

// ---- host ---------------------------------------------------------------------------------------------------------------

struct LogitsPlan { int G, chunks, per, parts; };

// Threads per group and groups per row: a wave for short rows, else what the model below expects to end first.  A group of G threads takes `start` us
// before its first and after its last chunk (its lists are loaded, its answer is reduced) and `chunk` us a chunk of 8 G entries, both longer
// by the lists, which every chunk searches (per 1024 entries of them).  The chip holds 2048 groups of 256 threads, which share its issue slots (one on
// a CU of its own takes ALONE of the time), or 512 of 1024; a choice over several groups of a row pays for the join, its launch and its scratch.
// The constants are fitted to bf16 calls in which either size was forced, us by 256 / by 1024 threads, with a history of
//                               64          1024         4096          16384
//   constrain    1 x  32000    3.8 /  4.5   4.7 /  4.9   7.4 /  5.5   17.8 /  8.4
//   constrain   64 x 131072   11.1 / 10.0  12.6 / 10.5  18.0 / 11.8   46.1 / 21.2
//   constrain 4000 x  12000   39   / 49    45   / 55    79   / 63
//   choose       1 x  32000    7.5 /  9.7   8.4 / 10.3  11.1 / 10.9   22.1 / 13.7
//   choose     300 x 131072   35   / 43    41   / 46    67   / 51    180   / 92
//   choose    4000 x   5000   39   / 61    46   / 65    68   / 70
// Over 25 sizes of each operator with five or six histories the calls it picks are 1.17 times as fast (geometric mean; 0.88 to 3.3 times) as with 1024
// threads wherever lists meet two such workgroups a CU.  The model knows neither the size of an element nor noise: of 512 x 131072 f32 with a history of 4096
// it expects 46 us and not 105.  What it picks is still near the better of the two: over 108 calls (constrain, greedy and drawn choices, f32 and
// bf16, six sizes, histories of 0, 256 and 4096, either size forced) 1.01 times its time (geometric mean), 1.12 at the worst (constrain 4000 x
// 12000 f32, 72 us by 256 and 65 by 1024 threads).  Six candidates for the groups of a row, so that choosing costs well under a microsecond.
struct GroupCost { float start, start_list, chunk, chunk_list; };

static LogitsPlan logits_plan(const FrlLogitsDesc* d, bool choose) {
  static const GroupCost COST[2][2] = {              // constrain, choose; 256, 1024 threads
      {{0.4f, 0.3f, 3.1f, 0.72f}, {1.9f, 0.12f, 2.1f, 0.15f}},
      {{4.2f, 0.2f, 2.3f, 0.78f}, {4.9f, 0.1f, 2.7f, 0.2f}}};
  const float JOIN = 4.0f, ALONE = 0.45f;
  LogitsPlan best;
  best.G = 64;
  best.chunks = (int)((d->vocab + 511LL) / 512);
  best.per = best.parts = 1;
  if (d->vocab <= 512 && d->n_sparse <= 512) return best;
  const float lists = ((float)d->history_len + (float)d->n_sparse) * (1.0f / 1024.0f), rows = (float)d->rows;
  float least = INFINITY;
  for (int w = 0; w < 2; ++w) {
    const GroupCost& g = COST[choose][w];
    const int G = w != 0 ? 1024 : 256, chunks = (int)((d->vocab + 8LL * G - 1) / (8 * G));
    const float slots = w != 0 ? 512.0f : 2048.0f;
    int last = 0;
    for (int rounds = 0; rounds <= 5; ++rounds) {            // one group per row; what fills the chip once to four times; one group per chunk
      const float fill = slots * (float)rounds / fmaxf(rows, 1.0f);
      int parts = rounds == 0 ? 1 : rounds == 5 || fill >= (float)chunks ? chunks : fill < 1.0f ? 1 : (int)fill;
      const int per = (chunks + parts - 1) / parts;
      parts = (chunks + per - 1) / per;
      if (parts == last) continue;
      last = parts;
      const float full = rows * (float)parts / slots, alone = w != 0 ? 1.0f : ALONE + (1.0f - ALONE) * fminf(full, 1.0f);
      const float cost = fmaxf(full, 1.0f) * (alone * (g.start + (float)per * g.chunk) + lists * (g.start_list + (float)per * g.chunk_list)) + (choose && parts > 1 ? JOIN : 0.0f);
      if (cost < least) {
        least = cost;
        best.G = G; best.chunks = chunks; best.per = per; best.parts = parts;
      }
    }
  }
  return best;
}

template <typename T, typename O, bool CHOOSE>
static hipError_t launch_logits(const LogitsArgs& a, int G, hipStream_t stream) {
  const dim3 grid = grid_of(G == 64 ? (a.items + 3) / 4 : a.items);
  const size_t lds = (size_t)(G == 64 ? 4 : 1) * a.K * 8;
#define FRL_LAUNCH(g, h, s)                                                                                             \
  hipLaunchKernelGGL((frl_logits_kernel<T, O, g, h, s, CHOOSE>), grid, dim3(g == 64 ? 256 : g), lds, stream, a)
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
  if (d->n_sparse > 0 && d->history_len > MAX_HISTORY_WITH_SLOTS) { set_error("logits: history_len %d > %d beside listed biases", d->history_len, MAX_HISTORY_WITH_SLOTS); return FRL_EUNSUPPORTED; }
  if (d->rows > (1LL << 35) || d->rows * logits_plan(d, choose).chunks > (1LL << 35)) { set_error("logits: %lld rows of %d entries are more than 2^35 chunks in one call", (long long)d->rows, d->vocab); return FRL_EUNSUPPORTED; }
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
  if (d->history_len > 0 && b->repetition == nullptr && !(d->repetition >= 1.17549435e-38f)) { set_error("logits: repetition %g must be > 0 and no subnormal number", d->repetition); return FRL_EINVAL; }
  a = LogitsArgs{b->logits, b->out, b->history, b->lengths, b->prompt_lengths, b->repetition, b->frequency, b->presence,
                 b->bias, b->bias_tokens, b->bias_values, b->allowed, b->temperature, b->gumbel, b->token, b->logprob,
                 nullptr, nullptr, nullptr, nullptr,
                 d->logits_stride, d->out_stride, d->gumbel_stride, d->history_stride, d->bias_stride, d->sparse_stride, d->mask_stride,
                 d->repetition, d->frequency, d->presence, d->temperature, d->vocab, d->ids64, d->history_len, d->n_sparse, d->mask, 0, 0, 0, 0, 0};
  const LogitsPlan p = logits_plan(d, choose);
  G = p.G;
  a.chunks = p.chunks; a.per = p.per; a.parts = p.parts;
  a.items = (long long)d->rows * p.parts;
  a.eager = a.items * p.G < 2048LL * 1024 || p.G == 64;      // less than two waves for every slot of the chip, or rows shorter than what skipping saves
  return FRL_OK;
}

static size_t logits_workspace(const FrlLogitsDesc* d) {
  const int parts = logits_plan(d, true).parts;
  return parts > 1 ? ((size_t)d->rows * parts * 20 + 511) / 256 * 256 : 256;
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
  const long long in_elt = desc->dtype == FRL_ELT_F32 ? 4 : 2, out_elt = desc->out_dtype == FRL_ELT_F32 ? 4 : 2, V = desc->vocab;
  const bool same = a.logits == a.out && desc->dtype == desc->out_dtype && (desc->logits_stride == desc->out_stride || desc->rows == 1);
  if (!same && rows_overlap((uintptr_t)a.logits, V * in_elt, desc->logits_stride * in_elt, (uintptr_t)a.out, V * out_elt, desc->out_stride * out_elt, desc->rows)) { set_error("logits: out overlaps logits without being the same rows"); return FRL_EINVAL; }
  const bool f32 = desc->out_dtype == FRL_ELT_F32;
  hipStream_t st = (hipStream_t)hip_stream;
  hipError_t e = hipErrorInvalidValue;
  if (desc->dtype == FRL_ELT_F32) e = launch_logits<float, float, false>(a, G, st);
  else if (desc->dtype == FRL_ELT_BF16) e = f32 ? launch_logits<Bf16, float, false>(a, G, st) : launch_logits<Bf16, Bf16, false>(a, G, st);
  else e = f32 ? launch_logits<F16, float, false>(a, G, st) : launch_logits<F16, F16, false>(a, G, st);
  if (e != hipSuccess) { set_error("logits constrain launch: %s", hipGetErrorString(e)); return FRL_EHIP; }
  note_kernel("frl_logits_kernel<constrain, %d threads> [%lld]", G, a.items);
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
  if (a.parts > 1) {
    if (workspace == nullptr || ((uintptr_t)workspace & 255) != 0) { set_error("workspace must be non-NULL and 256-byte aligned"); return FRL_EWORKSPACE; }
    if (workspace_bytes < logits_workspace(desc)) { set_error("workspace %zu B < required %zu B", workspace_bytes, logits_workspace(desc)); return FRL_EWORKSPACE; }
    a.part_key = (unsigned long long*)workspace;
    a.part_m = (float*)(a.part_key + a.items);
    a.part_s = a.part_m + a.items;
    a.part_y = a.part_s + a.items;
  }
  hipStream_t st = (hipStream_t)hip_stream;
  hipError_t e = desc->dtype == FRL_ELT_F32 ? launch_logits<float, float, true>(a, G, st)
               : desc->dtype == FRL_ELT_BF16 ? launch_logits<Bf16, float, true>(a, G, st) : launch_logits<F16, float, true>(a, G, st);
  if (e != hipSuccess) { set_error("logits choose launch: %s", hipGetErrorString(e)); return FRL_EHIP; }
  note_kernel("frl_logits_kernel<choose, %d threads> [%lld]", G, a.items);
  if (a.parts > 1) {
    const long long blocks = (desc->rows + 3) / 4;
    hipLaunchKernelGGL(frl_logits_join_kernel, grid_of(blocks), dim3(256), 0, st, a, (long long)desc->rows);
    e = hipGetLastError();
    if (e != hipSuccess) { set_error("logits join launch: %s", hipGetErrorString(e)); return FRL_EHIP; }
    note_kernel("frl_logits_join_kernel [%lld]", blocks);
  }
  return FRL_OK;
}

}  // extern "C"
