// Log probabilities of given tokens with the distribution's entropy and its largest entries, and the logits' gradient:
//   z = x / T (masked places -inf),  lse = log sum e^z,  p = e^(z - lse)
//   log_prob = z[token] - lse,  H = -sum p log p,  top: the K largest, ties by the lowest index
//   dx_j = (g_lp ([j = token] - p_j) - g_H p_j (log p_j + H)) / T
// One pass over a row: with the running maximum m, the sums s = sum e^(z - m) and u = sum e^(z - m) (x - m) are rescaled when m
// moves, and H = log s - u / (s T).  Differences to m are taken before they are scaled, so large logits lose nothing.  Places
// at -inf add nothing to u either: 0 * -inf is kept out by a bound on x - m, which a thread applies when its sum shows that it
// is needed.  Backward needs m, log s and H of each row.  An entry costs one exponential and, two at a time, about four other
// instructions: less than the bytes take, but not by much (single operations took twice as long as the bytes).
//
// Short rows: a few lanes hold a row in registers.  Longer ones: a warp a row where there are rows for all warps and a block would
// have little of each, blocks that walk the rows where these are long and many, else a block, or, where rows are few, a cluster of
// up to eight blocks, whose sums meet in distributed shared memory.
//
// The largest entries, as keys of (value, index) that are all different: each of 32 groups of a block's threads knows its
// largest key from the one pass; the K-th largest of those bounds the K-th largest of all from below, and only threads whose
// own largest reaches the bound look at their elements again.  What they find (about K log K keys) is ranked by counting.
//
// Bytes bound it, the logits once; backward logits in, gradient out.  8000 rows of 50001 bf16 logits: forward 160 us, 5.0 TB/s (a
// warp a row leaves 18 warps an SM in 2.7 waves, and the pipe of the exponentials is in use half of the time), backward 255 us, 6.3 TB/s;
// in float32 255 and 462 us, 6.3 and 6.9 TB/s.  131072 float32 rows of 1000: 99 and 149 us, 5.3 and 7.0 TB/s.  64 rows of 32768
// with their eight largest: 8.0 us, of which the pass over the row is 4.7 and the search 3.3, chains of barriers and memory
// latency.  131072 rows of 18 with a mask: 9.9 and 10.8, several waves of short blocks.
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "elements.cuh"
#include "packed.cuh"

namespace mxk {
namespace {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kColdest = 1e-30f, kHottest = 1e27f;   // temperatures: a bound on x - m (below) still has the exponential zero
constexpr float kLeastLog = -128.f; // of a probability: one of this logarithm is zero in float32, and so is what it is a factor of
constexpr int kNarrow = 128;        // longest row of the kernels that hold one in registers
constexpr int kShort = 1024;        // and longest that is one where the largest entries are wanted, or else a warp's, however few they are
constexpr int kMaxTop = 32;
constexpr int kFound = 1024;        // keys that the second look may find; more: K rounds of a block-wide maximum

__device__ __forceinline__ float ninf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// x - m, no less than a bound whose exponential is zero; NaN stays
__device__ __forceinline__ float below(float x, float m) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x - m), "f"(-1e30f));
  return y;
}

// In the order of (value, then lowest index); 0 is below every key.
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t index) {
  uint32_t b = __float_as_uint(x + 0.f);         // (-0 and 0 are the same value)
  if (x != x) b = 0xff800000u;                   // NaN: with the lowest, so that every row has its K entries
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(b) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_index(unsigned long long k) { return 0xffffffffu - static_cast<uint32_t>(k); }
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t b = static_cast<uint32_t>(k >> 32);
  return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ unsigned long long larger(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

// How many of `count` keys are larger.  keys: 16-byte aligned, room for an even number.  Several loads at a time: one after the other
// they were most of the time of a search.
__device__ __forceinline__ int larger_ones(const unsigned long long* keys, int count, unsigned long long key) {
  const ulonglong2* const pairs = reinterpret_cast<const ulonglong2*>(keys);
  int n = 0;
#pragma unroll 4
  for (int j = 0; j < count; j += 2) {
    const ulonglong2 two = pairs[j / 2];
    n += two.x > key;
    n += j + 1 < count && two.y > key;
  }
  return n;
}

struct Sums {                        // of a set of entries: their maximum, sum e^(z - m), sum e^(z - m) (x - m)
  float m, s, u;
};
// k: log2(e) / T
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float k) {
  const float m = fmaxf(a.m, b.m);
  if (m == ninf()) return {m, a.s + b.s, a.u + b.u};                    // (zeros, or NaN)
  const float da = below(a.m, m), db = below(b.m, m);
  const float ca = exp2_fast(da * k), cb = exp2_fast(db * k);
  return {m, a.s * ca + b.s * cb, (a.u + a.s * da) * ca + (b.u + b.s * db) * cb};
}
__device__ __forceinline__ Sums join_lanes(const Sums& a, int lanes, float k) {
  float m = a.m;
  for (int off = 1; off < lanes; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  Sums all{m, a.s, a.u};
  if (m != ninf()) {                 // (else zeros, or NaN)
    const float d = below(a.m, m), c = exp2_fast(d * k);
    all.s = a.s * c;
    all.u = (a.u + a.s * d) * c;
  }
  for (int off = 1; off < lanes; off <<= 1) {
    all.s += __shfl_xor_sync(0xffffffffu, all.s, off);
    all.u += __shfl_xor_sync(0xffffffffu, all.u, off);
  }
  return all;
}

struct LogprobArgs {
  const void* x;
  long long ld;                      // elements between rows
  const uint8_t* mask;               // non-zero: allowed
  long long mask_ld;
  const void* tokens;
  int tokens_bytes;
  float *log_prob, *entropy, *top_value;
  long long* top_index;
  float4* stats;                     // of each row: m, log s, H
  long long rows;
  int vocab, top;
  float inv_t;
  int lanes;                         // of a short row
};
struct Row {
  float m, logs, h;
};
__device__ __forceinline__ Row finish(const Sums& s, float inv_t) {
  if (s.s == 0.f) return {0.f, __int_as_float(0x7f800000), 0.f};        // nothing is left of the row: e^(x - 0 - inf) = 0
  const float logs = logf(s.s);
  return {s.m, logs, logs - s.u / s.s * inv_t};
}
__device__ __forceinline__ float log_p(float x, const Row& r, float inv_t) { return (x - r.m) * inv_t - r.logs; }
__device__ __forceinline__ long long token_of(const void* tokens, int bytes, long long n) {
  return bytes == 8 ? static_cast<const long long*>(tokens)[n] : static_cast<const int*>(tokens)[n];
}
// What the row's first thread leaves: a token outside of the vocabulary marks a row that is not there.
__device__ __forceinline__ void leave_row(const LogprobArgs& a, long long n, const Row& r, bool known, float at_token) {
  float h = r.h;
  if (a.tokens) {
    a.log_prob[n] = known ? log_p(at_token, r, a.inv_t) : 0.f;
    if (!known) h = 0.f;
  }
  if (a.entropy) a.entropy[n] = h;
  if (a.stats) a.stats[n] = make_float4(r.m, r.logs, r.h, 0.f);
}
template <typename T>
__device__ __forceinline__ void leave_row(const LogprobArgs& a, long long n, const Row& r) {
  const long long t = a.tokens ? token_of(a.tokens, a.tokens_bytes, n) : -1;
  const bool known = t >= 0 && t < a.vocab, allowed = known && (!a.mask || a.mask[n * a.mask_ld + t]);
  leave_row(a, n, r, known, allowed ? as_float(static_cast<const T*>(a.x)[n * a.ld + t]) : ninf());
}

// ---------------------------------------------------------------------------------------------------------- short rows
// Lane l of a row's `lanes` holds the entries l, l + lanes, ...  A row's time is its loads' latency: none waits for another.
template <typename T, int E, bool kMask>
__global__ void __launch_bounds__(128)
logprob_short_kernel(const LogprobArgs a) {
  enter_kernel();
  const int L = a.lanes, l = threadIdx.x % L;
  const long long n = static_cast<long long>(blockIdx.x) * (128 / L) + threadIdx.x / L;
  const bool live = n < a.rows;
  const T* const row = static_cast<const T*>(a.x) + n * a.ld;
  const uint8_t* const mask = kMask ? a.mask + n * a.mask_ld : nullptr;
  const float k = a.inv_t * kLog2e;
  const long long token = a.tokens && live ? token_of(a.tokens, a.tokens_bytes, n) : -1;
  float x[E];
  uint8_t allowed[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = l + e * L;
    x[e] = ninf();
    if (live && j < a.vocab) {
      x[e] = as_float(row[j]);
      if (kMask) allowed[e] = mask[j];
    }
  }
  float at_token = ninf();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (kMask && live && l + e * L < a.vocab && !allowed[e]) x[e] = ninf();
    if (l + e * L == token) at_token = x[e];
  }
  const bool known = token >= 0 && token < a.vocab;
  at_token = __shfl_sync(0xffffffffu, at_token, known ? static_cast<int>(token) & (L - 1) : 0, L);
  Sums s{ninf(), 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < E; ++e) s.m = fmaxf(s.m, x[e]);
  for (int off = 1; off < L; off <<= 1) s.m = fmaxf(s.m, __shfl_xor_sync(0xffffffffu, s.m, off));
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (x[e] == ninf()) continue;
    const float y = below(x[e], s.m), w = exp2_fast(y * k);
    s.s += w;
    s.u = fmaf(w, y, s.u);
  }
  for (int off = 1; off < L; off <<= 1) {
    s.s += __shfl_xor_sync(0xffffffffu, s.s, off);
    s.u += __shfl_xor_sync(0xffffffffu, s.u, off);
  }
  const Row r = finish(s, a.inv_t);
  if (live && l == 0) leave_row(a, n, r, known, at_token);
  unsigned long long last = ~0ull;
  for (int q = 0; q < a.top; ++q) {           // the largest key below the one before
    unsigned long long best = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = l + e * L;
      if (j < a.vocab) {
        const unsigned long long key = key_of(x[e], j);
        if (key < last) best = larger(best, key);
      }
    }
    for (int off = 1; off < L; off <<= 1) best = larger(best, __shfl_xor_sync(0xffffffffu, best, off));
    last = best;
    if (live && l == 0) {
      a.top_index[n * a.top + q] = key_index(best);
      a.top_value[n * a.top + q] = log_p(key_value(best), r, a.inv_t);
    }
  }
}

struct LogprobGradArgs {
  const void* x;
  long long ld;
  const uint8_t* mask;
  long long mask_ld;
  const void* tokens;
  int tokens_bytes;
  const float4* stats;
  const float *g_lp, *g_h;           // either may be null
  long long g_lp_ld, g_h_ld;
  void* dx;                          // (rows, vocab)
  long long rows;
  int vocab, lanes, chunks;
  float inv_t;
};
struct RowGrad {
  Row r;
  float g1, g2;                      // dx_j = (-p_j (g1 + g2 log p_j), plus `at_token` at the token) times `post`
  float at_token, post;              // post: 1, the division by T being in the others, or 1 / T where it would make them infinite
  int token;                         // -1: none
  bool there;                        // else zeros, whatever the row holds: its token is outside of the vocabulary, or all is -inf
};
__device__ __forceinline__ RowGrad row_grad(const LogprobGradArgs& a, long long n) {
  const float4 st = a.stats[n];
  RowGrad g{{st.x, st.y, st.z}, 0.f, 0.f, 0.f, 1.f, -1, st.y != __int_as_float(0x7f800000)};
  const float gh = a.g_h ? a.g_h[n * a.g_h_ld] : 0.f;
  float glp = a.tokens && a.g_lp ? a.g_lp[n * a.g_lp_ld] : 0.f;
  if (a.tokens) {
    const long long token = token_of(a.tokens, a.tokens_bytes, n);
    g.there = g.there && token >= 0 && token < a.vocab;
    g.token = static_cast<int>(token);
  }
  const float g1 = glp + gh * st.z;
  // (a cold row of one token has no gradient, and infinities would leave NaN of it)
  const bool small = (fabsf(glp) + fabsf(g1) - kLeastLog * fabsf(gh)) * a.inv_t < 3e38f;
  const float scale = small ? a.inv_t : 1.f;
  g.g1 = g1 * scale;
  g.g2 = gh * scale;
  g.at_token = glp * scale;
  g.post = small ? 1.f : a.inv_t;
  return g;
}
__device__ __forceinline__ float entry_grad(float x, const RowGrad& g, float inv_t) {
  float lp = fmaf(x - g.r.m, inv_t, -g.r.logs);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(lp) : "f"(kLeastLog));
  return -exp2_fast(lp * kLog2e) * fmaf(g.g2, lp, g.g1);
}

// Of N entries at once, two in each instruction; where an infinite one shows in the sum, or one so cold that its factor is, one at a time.
template <int N>
__device__ __forceinline__ void entry_grads(float* x, const RowGrad& g, float inv_t) {
  if constexpr (N % 2 == 0) {
    const F2 minus(-g.r.m), scale(inv_t), logs(-g.r.logs), to2(kLog2e), g1(-g.g1), g2(-g.g2);
    F2 d[N / 2], sum(0.f);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const F2 lp = fma(add(F2(x[2 * i], x[2 * i + 1]), minus), scale, logs), z = mul(lp, to2);
      d[i] = mul(F2(exp2_fast(z.lo()), exp2_fast(z.hi())), fma(g2, lp, g1));
      sum = add(sum, d[i]);
    }
    const float all = sum.sum();
    if (all == all) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) x[2 * i] = d[i].lo(), x[2 * i + 1] = d[i].hi();
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = entry_grad(x[i], g, inv_t);
}

template <typename T, int E, bool kMask>
__global__ void __launch_bounds__(128)
logprob_short_bwd_kernel(const LogprobGradArgs a) {
  enter_kernel();
  const int L = a.lanes, l = threadIdx.x % L;
  const long long n = static_cast<long long>(blockIdx.x) * (128 / L) + threadIdx.x / L;
  if (n >= a.rows) return;
  const T* const row = static_cast<const T*>(a.x) + n * a.ld;
  const uint8_t* const mask = kMask ? a.mask + n * a.mask_ld : nullptr;
  T* const out = static_cast<T*>(a.dx) + n * a.vocab;
  float x[E];
  uint8_t allowed[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = l + e * L;
    if (j < a.vocab) {
      x[e] = as_float(row[j]);
      if (kMask) allowed[e] = mask[j];
    }
  }
  const RowGrad g = row_grad(a, n);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = l + e * L;
    if (j >= a.vocab) continue;
    float d = 0.f;
    if (g.there && (!kMask || allowed[e])) {
      d = entry_grad(x[e], g, a.inv_t);
      if (j == g.token) d += g.at_token;
      d *= g.post;
    }
    out[j] = from_float<T>(d);
  }
}

// ----------------------------------------------------------------------------------------------------------- long rows
// A row's entries as aligned vectors with what is in front of and behind them.
template <typename T, int V>
struct Split {
  int lead, vecs;
  __device__ __forceinline__ Split(const T* row, int vocab) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) / sizeof(T) % V);
    lead = off ? V - off : 0;
    if (lead > vocab) lead = vocab;
    vecs = (vocab - lead) / V;
  }
};
// V mask bytes as they are in memory (aligned to V), and what they hide.
template <int V>
struct MaskWord {
  typename Raw<V>::type bits;
  __device__ __forceinline__ void load(const uint8_t* p, bool aligned) {
    if (aligned) {
      bits = *reinterpret_cast<const typename Raw<V>::type*>(p);
    } else {
      uint8_t* const b = reinterpret_cast<uint8_t*>(&bits);
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] = p[i];
    }
  }
  __device__ __forceinline__ bool hides(int i) const {
    if constexpr (V == 1) return !bits;
    else return !(reinterpret_cast<const uint32_t*>(&bits)[i / 4] >> i % 4 * 8 & 0xff);
  }
  __device__ __forceinline__ void apply(float* x, float to) const {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = hides(i) ? to : x[i];
  }
};

// One thread's running sums over entries, N at a time.
template <int N>
__device__ __forceinline__ void take(Sums& s, const float* x, float k) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
  if (top > s.m) {
    const float d = below(s.m, top), c = exp2_fast(d * k);
    s.u = (s.u + s.s * d) * c;
    s.s *= c;
    s.m = top;
  }
  if (s.m == ninf()) {                // so far nothing but -inf, and NaN
#pragma unroll
    for (int i = 0; i < N; ++i) if (x[i] != x[i]) s.s = x[i];
    return;
  }
  if constexpr (N % 2 == 0) {
    const F2 minus(-s.m), scale(k);
    F2 sum(0.f), moment(0.f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const F2 y = add(F2(x[i], x[i + 1]), minus), z = mul(y, scale), w(exp2_fast(z.lo()), exp2_fast(z.hi()));
      sum = add(sum, w);
      moment = fma(w, y, moment);
    }
    const float u = moment.sum();
    if (u == u) {
      s.s += sum.sum();
      s.u += u;
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = below(x[i], s.m), w = exp2_fast(y * k);
    s.s += w;
    s.u = fmaf(w, y, s.u);
  }
}
template <int N>
__device__ __forceinline__ void note(float& best, int& best_at, const float* x, int at) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
  if (top > best || best_at < 0) {
    int where = 0;
#pragma unroll
    for (int i = N - 1; i >= 0; --i) if (x[i] == top) where = i;
    best = top;                       // (NaN alone: index 0 of the vector, and a key that counts as -inf)
    best_at = at + where;
  }
}

// A row, or a block's part of one (`from` .. `to` of its vectors, the first part with what is around them), by kThreads threads:
// each thread's sums, and its largest entry.
template <typename T, int kThreads, bool kTop, bool kMask, int kEach = 16>
struct Scan {
  static constexpr int V = 16 / sizeof(T), kAhead = kTop ? 2 : kEach / V, kStep = kThreads * kAhead;     // (fewer registers where the largest are kept)
  const T* row;
  const uint8_t* mask;
  Split<T, V> split;
  int from, to, vocab, tid;
  bool first, aligned;                // the first part; the mask's words
  Sums s{ninf(), 0.f, 0.f};
  float best = ninf();
  int best_at = -1;

  struct Group {
    Vec<T, V> x[kAhead];
    MaskWord<V> m[kAhead];
  };
  __device__ __forceinline__ Scan(const T* row, const uint8_t* mask, int vocab, int tid, int rank, int parts) : row(row), mask(mask), split(row, vocab), vocab(vocab), tid(tid), first(rank == 0) {
    from = static_cast<int>(static_cast<long long>(split.vecs) * rank / parts);
    to = static_cast<int>(static_cast<long long>(split.vecs) * (rank + 1) / parts);
    aligned = kMask && reinterpret_cast<uintptr_t>(mask + split.lead) % V == 0;
  }
  __device__ __forceinline__ float single(int j) const { return kMask && !mask[j] ? ninf() : as_float(row[j]); }
  __device__ __forceinline__ void around(int j, float k) {
    const float x = single(j);
    take<1>(s, &x, k);
    if (kTop) note<1>(best, best_at, &x, j);
  }
  // vectors v, v + kThreads, ...: all there (kAll), or those below `to`
  template <bool kAll>
  __device__ __forceinline__ void load(Group& g, int v) const {
    const T* const p = row + split.lead + static_cast<long long>(v) * V;
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (kAll || v + q * kThreads < to) {
        g.x[q] = Vec<T, V>::load(p + q * kThreads * V);
        if (kMask) g.m[q].load(mask + split.lead + static_cast<long long>(v + q * kThreads) * V, aligned);
      }
  }
  template <bool kAll>
  __device__ __forceinline__ void use(const Group& g, int v, float k) {
    float x[kAhead * V];
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (kAll || v + q * kThreads < to) {
        g.x[q].unpack(x + q * V);
        if (kMask) g.m[q].apply(x + q * V, ninf());
        if (kTop) note<V>(best, best_at, x + q * V, split.lead + (v + q * kThreads) * V);
        if (!kAll) take<V>(s, x + q * V, k);
      }
    if (kAll) take<kAhead * V>(s, x, k);
  }
  __device__ __forceinline__ void begin(Group& a) const {
    if (to - from >= kStep) load<true>(a, from + tid); else load<false>(a, from + tid);
  }
  __device__ __forceinline__ void run(float k) {
    Group a;
    begin(a);
    run(a, k);
  }
  // a: as begin() left it
  __device__ __forceinline__ void run(Group& a, float k) {
    Group b;
    if (first && tid < split.lead) around(tid, k);
    const int groups = (to - from) / kStep;
    int v = from + tid;
    for (int i = 0; i < groups; i += 2, v += 2 * kStep) {           // two in turn, so that none has to be moved
      if (i + 1 < groups) load<true>(b, v + kStep); else load<false>(b, v + kStep);
      use<true>(a, v, k);
      if (i + 1 >= groups) {
        use<false>(b, v + kStep, k);
        break;
      }
      if (i + 2 < groups) load<true>(a, v + 2 * kStep); else load<false>(a, v + 2 * kStep);
      use<true>(b, v + kStep, k);
    }
    if (groups % 2 == 0) use<false>(a, v, k);
    const int behind = split.lead + split.vecs * V;
    if (first && behind + tid < vocab) around(behind + tid, k);
  }
  // its entries from `least` on (and NaN), once more; there are few, so what is done with one is not unrolled into all of them
  template <typename F>
  __device__ __forceinline__ void each(float least, F&& f) const {
    if (first && tid < split.lead) f(single(tid), tid);
    constexpr int kMany = 8;            // (loads that wait for one another would be most of the time)
    for (int v0 = from + tid; v0 < to; v0 += kThreads * kMany) {
      Vec<T, V> raw[kMany];
#pragma unroll
      for (int q = 0; q < kMany; ++q)
        if (v0 + q * kThreads < to) raw[q] = Vec<T, V>::load(row + split.lead + static_cast<long long>(v0 + q * kThreads) * V);
      unsigned long long large = 0;
#pragma unroll
      for (int q = 0; q < kMany; ++q) {
        float x[V];
        raw[q].unpack(x);
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) bits |= x[i] < least ? 0u : 1u << i;
        if (v0 + q * kThreads < to) large |= static_cast<unsigned long long>(bits) << q * V;
      }
      while (large) {
        const int at = __ffsll(large) - 1, j = split.lead + (v0 + at / V * kThreads) * V + at % V;
        large &= large - 1;
        const float x = single(j);       // (hidden ones come back as -inf)
        if (!(x < least)) f(x, j);
      }
    }
    const int behind = split.lead + split.vecs * V;
    if (first && behind + tid < vocab) f(single(behind + tid), behind + tid);
  }
};

// A warp a row.
template <typename T, bool kMask, int kEach>
__global__ void __launch_bounds__(128)
logprob_warp_kernel(const LogprobArgs a) {
  enter_kernel();
  const long long n = static_cast<long long>(blockIdx.x) * 4 + threadIdx.x / 32;
  if (n >= a.rows) return;
  const float k = a.inv_t * kLog2e;
  Scan<T, 32, false, kMask, kEach> scan(static_cast<const T*>(a.x) + n * a.ld, kMask ? a.mask + n * a.mask_ld : nullptr, a.vocab, threadIdx.x % 32, 0, 1);
  scan.run(k);
  const Row r = finish(join_lanes(scan.s, 32, k), a.inv_t);
  if (threadIdx.x % 32 == 0) leave_row<T>(a, n, r);
}

// As many blocks as are resident walk the rows: a row's first vectors are under way while the row before it is summed over the warps.
// These take turns at what is left to do for a row, its token's logit included.
constexpr int kWalkThreads = 128;
template <typename T, bool kMask> constexpr int kWalkBlocks = sizeof(T) == 4 ? (kMask ? 4 : 5) : kMask ? 5 : 8;      // of an SM, as the registers go
template <typename T, bool kMask>
__global__ void __launch_bounds__(kWalkThreads, kWalkBlocks<T, kMask>)
logprob_walk_kernel(const LogprobArgs a) {
  enter_kernel();
  constexpr int kWarps = kWalkThreads / 32;
  using Row_ = Scan<T, kWalkThreads, false, kMask>;
  __shared__ Sums warps[2][kWarps];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const float k = a.inv_t * kLog2e;
  const auto row_at = [&](long long n) {
    return Row_(static_cast<const T*>(a.x) + n * a.ld, kMask ? a.mask + n * a.mask_ld : nullptr, a.vocab, tid, 0, 1);
  };
  long long n = blockIdx.x;
  Row_ now = row_at(n);
  typename Row_::Group group;
  now.begin(group);
  for (int i = 0; n < a.rows; ++i) {
    now.run(group, k);
    const Sums mine = now.s;
    const long long next = n + gridDim.x;
    if (next < a.rows) {
      now = row_at(next);
      now.begin(group);
    }
    const Sums s = join_lanes(mine, 32, k);
    if (lane == 0) warps[i & 1][warp] = s;
    __syncthreads();                  // (the other half is written before the next one, read behind it)
    if (warp == (i & (kWarps - 1))) {
      const Row r = finish(join_lanes(lane < kWarps ? warps[i & 1][lane] : Sums{ninf(), 0.f, 0.f}, kWarps, k), a.inv_t);
      if (lane == 0) leave_row<T>(a, n, r);
    }
    n = next;
  }
}

template <typename T, int kThreads, bool kTop, bool kMask>
__global__ void __launch_bounds__(kThreads, kTop ? 1024 / kThreads : 1)
logprob_long_kernel(const LogprobArgs a) {
  enter_kernel();
  const cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const long long n = blockIdx.x / blocks;
  const float k = a.inv_t * kLog2e;
  constexpr int kWarps = kThreads / 32;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  Scan<T, kThreads, kTop, kMask> scan(static_cast<const T*>(a.x) + n * a.ld, kMask ? a.mask + n * a.mask_ld : nullptr, a.vocab, tid, rank, blocks);
  if (blocks > 1) cluster.barrier_arrive();
  scan.run(k);
  if (blocks > 1) cluster.barrier_wait();      // (the first block is there to be written to)

  __shared__ Sums warps[kWarps], parts[8];
  Sums s = join_lanes(scan.s, 32, k);
  if (lane == 0) warps[warp] = s;
  __syncthreads();
  if (warp == 0) {
    s = join_lanes(lane < kWarps ? warps[lane] : Sums{ninf(), 0.f, 0.f}, kWarps, k);
    // where the first block reads it
    if (lane == 0) *cluster.map_shared_rank(&parts[rank], 0) = s;
  }

  __shared__ __align__(16) unsigned long long best_keys[kMaxTop], found[kTop ? kFound : 2], all_keys[kTop ? 8 * kMaxTop : 2];
  __shared__ unsigned long long groups[32], bound, round_keys[kWarps];
  __shared__ int found_n;
  if constexpr (kTop) {
    const unsigned long long mine = scan.best_at >= 0 ? key_of(scan.best, scan.best_at) : 0;
    constexpr int width = kThreads / 32;      // threads of a group: 4 .. 16
    unsigned long long g = mine;
    for (int off = 1; off < width; off <<= 1) g = larger(g, __shfl_xor_sync(0xffffffffu, g, off));
    if (tid % width == 0) groups[tid / width] = g;
    if (tid == 0) found_n = 0;
    __syncthreads();
    if (warp == 0) {
      const unsigned long long key = groups[lane];
      int rank_of = 0;
      for (int i = 0; i < 32; ++i) {
        const unsigned long long other = __shfl_sync(0xffffffffu, key, i);
        rank_of += other > key || (other == key && i < lane);           // (empty groups share the key 0)
      }
      if (rank_of == a.top - 1) bound = key;
      if (lane < kMaxTop) best_keys[lane] = 0;
    }
    __syncthreads();
    const unsigned long long least = bound;
    if (mine >= least && mine)
      scan.each(key_value(least), [&](float x, int j) {
        const unsigned long long key = key_of(x, j);
        if (key >= least) {
          const int slot = atomicAdd(&found_n, 1);
          if (slot < kFound) found[slot] = key;
        }
      });
    __syncthreads();
    const int many = found_n;
    if (many <= kFound) {
      for (int i = tid; i < many; i += kThreads) {
        const unsigned long long key = found[i];
        const int rank_of = larger_ones(found, many, key);
        if (rank_of < a.top) best_keys[rank_of] = key;
      }
      __syncthreads();
    } else {                                    // many large entries fell to few threads: K rounds
      unsigned long long last = ~0ull;
      for (int q = 0; q < a.top; ++q) {
        unsigned long long b = 0;
        if (mine >= least && mine)
          scan.each(ninf(), [&](float x, int j) {
            const unsigned long long key = key_of(x, j);
            if (key < last) b = larger(b, key);
          });
        for (int off = 1; off < 32; off <<= 1) b = larger(b, __shfl_xor_sync(0xffffffffu, b, off));
        if (lane == 0) round_keys[warp] = b;
        __syncthreads();
        b = round_keys[0];
        for (int w = 1; w < kWarps; ++w) b = larger(b, round_keys[w]);
        last = b;
        if (tid == 0) best_keys[q] = b;
        __syncthreads();
      }
    }
  }

  if constexpr (kTop) {
    if (blocks > 1 && tid < a.top) *cluster.map_shared_rank(&all_keys[rank * a.top + tid], 0) = best_keys[tid];
  }
  // (nobody of the others is read from here on, and the first block is the last to leave)
  if (blocks > 1) cluster.sync(); else __syncthreads();
  if (rank != 0) return;
  if (kTop || warp == 0) {
    const Row done = finish(join_lanes(lane % 8 < blocks ? parts[lane % 8] : Sums{ninf(), 0.f, 0.f}, 8, k), a.inv_t);
    if (tid == 0) leave_row<T>(a, n, done);
    if constexpr (kTop) {
      const unsigned long long* const keys = blocks > 1 ? all_keys : best_keys;
      for (int i = tid; i < blocks * a.top; i += kThreads) {             // each block's are in order; all different but for zeros
        const unsigned long long key = keys[i];
        const int rank_of = larger_ones(keys, blocks * a.top, key);
        if (key && rank_of < a.top) {
          a.top_index[n * a.top + rank_of] = key_index(key);
          a.top_value[n * a.top + rank_of] = log_p(key_value(key), done, a.inv_t);
        }
      }
    }
  }
}

// A warp a chunk of a row (a block's would be emptier at a row's end: 60000 rows of 3001 bf16 logits 128 us against 206, 8000 of
// 50001 255 against 263).  V > 1: logits and gradient lie alike within 16 bytes in every row.
constexpr int kChunkThreads = 256, kChunkVecs = 4;
template <typename T, int V, bool kMask>
__global__ void __launch_bounds__(kChunkThreads)
logprob_long_bwd_kernel(const LogprobGradArgs a) {
  enter_kernel();
  const long long item = static_cast<long long>(blockIdx.x) * (kChunkThreads / 32) + threadIdx.x / 32, n = item / a.chunks;
  if (n >= a.rows) return;
  const int chunk = static_cast<int>(item - n * a.chunks), tid = threadIdx.x % 32;
  const T* const row = static_cast<const T*>(a.x) + n * a.ld;
  const uint8_t* const mask = kMask ? a.mask + n * a.mask_ld : nullptr;
  T* const out = static_cast<T*>(a.dx) + n * a.vocab;
  const Split<T, V> split(row, a.vocab);
  const int v0 = chunk * (32 * kChunkVecs) + tid;
  const bool aligned = kMask && reinterpret_cast<uintptr_t>(mask + split.lead) % V == 0;
  Vec<T, V> raw[kChunkVecs];
  MaskWord<V> words[kChunkVecs];
#pragma unroll
  for (int q = 0; q < kChunkVecs; ++q)
    if (v0 + q * 32 < split.vecs) {
      const long long at = split.lead + static_cast<long long>(v0 + q * 32) * V;
      raw[q] = Vec<T, V>::load_stream(row + at);
      if (kMask) words[q].load(mask + at, aligned);
    }
  const RowGrad g = row_grad(a, n);
  if (V > 1 && chunk == 0) {
    const int behind = split.lead + split.vecs * V;
    const auto single = [&](int j) {
      float d = 0.f;
      if (g.there && (!kMask || mask[j])) {
        d = entry_grad(as_float(row[j]), g, a.inv_t);
        if (j == g.token) d += g.at_token;
        d *= g.post;
      }
      out[j] = from_float<T>(d);
    };
    if (tid < split.lead) single(tid);
    else if (tid >= 16 && behind + tid - 16 < a.vocab) single(behind + tid - 16);      // (fewer than V of either)
  }
#pragma unroll
  for (int q = 0; q < kChunkVecs; ++q)
    if (v0 + q * 32 < split.vecs) {
      const int at = split.lead + (v0 + q * 32) * V;
      float x[V];
      raw[q].unpack(x);
      entry_grads<V>(x, g, a.inv_t);
      if (static_cast<unsigned>(g.token - at) < V) {
#pragma unroll
        for (int i = 0; i < V; ++i) if (g.token == at + i) x[i] += g.at_token;
      }
      if (g.post != 1.f) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] *= g.post;
      }
      if (kMask) words[q].apply(x, 0.f);
      if (!g.there) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = 0.f;
      }
      Vec<T, V>::pack(x).store_stream(out + at);
    }
}

// Lanes of a short row: four entries each, or eight where the rows are more than one wave then, since what a row costs besides is
// paid per lane (200000 float32 rows of 65: 46 and 42 us against 70 and 52 of four; 1000 rows of 100: 3.2 and 2.8 against 2.8 and 2.5).
int short_lanes(int vocab, long long rows) {
  const auto lanes_of = [&](int each) {
    int lanes = 1;
    while (lanes < 32 && lanes * each < vocab) lanes *= 2;
    return lanes;
  };
  return rows * lanes_of(4) > 2048ll * kNumSMs ? lanes_of(8) : lanes_of(4);
}
template <typename T, int kThreads, bool kMask>
void launch_long(const LogprobArgs& a, unsigned cluster, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(a.rows * cluster);
  if (a.top) launch_kernel_clusters(logprob_long_kernel<T, kThreads, true, kMask>, cluster, grid, kThreads, 0, s, a);
  else launch_kernel_clusters(logprob_long_kernel<T, kThreads, false, kMask>, cluster, grid, kThreads, 0, s, a);
}
template <typename T, bool kMask>
void forward_long(const LogprobArgs& a, cudaStream_t s) {
  // A warp a row: where a block's threads would have a few vectors each, if there are eight rows an SM, two vectors at a time (60000
  // x 5001 bf16: 130 us against 144 with four); and where there are two waves of them, 32 entries at a time (24000 x 16001 bf16: 159
  // against 172 of walking blocks, 8000 x 50001: 160 against 164; 2000 x 50001: 67 against 51).  Walking blocks: eight rows an SM
  // of the others (4000 x 100000 bf16: 158 against 199 of a block a row).
  const size_t bytes = a.vocab * sizeof(T);
  const auto warps = [&](auto kernel) { launch_kernel(kernel, static_cast<unsigned>((a.rows + 3) / 4), 128, 0, s, a); };
  if (!a.top && (a.vocab <= kShort || (bytes <= 16384 && a.rows >= 8 * kNumSMs))) return warps(logprob_warp_kernel<T, kMask, 32 / sizeof(T)>);
  if (!a.top && bytes <= 131072 && a.rows >= 40 * kNumSMs) return warps(logprob_warp_kernel<T, kMask, 32>);
  if (!a.top && a.rows >= 8 * kNumSMs) {
    constexpr int kBlocks = kWalkBlocks<T, kMask> * kNumSMs;
    launch_kernel(logprob_walk_kernel<T, kMask>, static_cast<unsigned>(a.rows < kBlocks ? a.rows : kBlocks), kWalkThreads, 0, s, a);
    return;
  }
  // a row to several blocks where rows alone leave SMs idle and a block's part stays a few vectors a thread
  unsigned cluster = 1;
  while (cluster < 8 && a.rows * cluster * 2 <= kNumSMs && a.vocab / (cluster * 2) >= 4096) cluster *= 2;
  // Threads of a block: what a row costs besides its entries is paid per thread, so there are only as many as fill the SMs with
  // the rows there are, and no more than have four vectors each.
  int threads = 128;
  while (threads < 512 && a.rows * cluster * threads < 1024ll * kNumSMs && a.vocab / static_cast<int>(cluster) >= threads * 64) threads *= 2;
  if (threads == 128) launch_long<T, 128, kMask>(a, cluster, s);
  else if (threads == 256) launch_long<T, 256, kMask>(a, cluster, s);
  else launch_long<T, 512, kMask>(a, cluster, s);
}
// Whether a row is held in registers.  Up to 128 entries (200000 float32 rows of 100 with a mask 71 us against 92 of a warp a row that
// goes by vectors, of 200 153 against 105).  With the largest entries, one of which costs a round over all that is held: up to 256; up to two of
// longer rows (20000 bf16 rows of 1000: 75 us against 84, four of them 96 against 88); and where a block's groups of threads
// are fewer than the wanted entries, which leaves its search without a bound (twenty of 500: 278 against 1029, of 1000: 281 against 107).
template <typename T>
bool held_row(int vocab, int top) {
  constexpr int kGroup = 4 * 16 / sizeof(T);      // entries of the smallest block's groups
  if (!top) return vocab <= kNarrow;
  return vocab <= 256 || (vocab <= kShort && (top <= 2 || (vocab + kGroup - 1) / kGroup < top));
}
unsigned short_blocks(int vocab, long long rows, int* lanes) {
  *lanes = short_lanes(vocab, rows);
  return static_cast<unsigned>((rows + 128 / *lanes - 1) / (128 / *lanes));
}
template <typename T>
void forward(LogprobArgs a, cudaStream_t s) {
  if (held_row<T>(a.vocab, a.top)) {
    const unsigned blocks = short_blocks(a.vocab, a.rows, &a.lanes);
    const auto go = [&](auto kernel) { launch_kernel(kernel, blocks, 128, 0, s, a); };
    if (a.vocab <= 4 * a.lanes) a.mask ? go(logprob_short_kernel<T, 4, true>) : go(logprob_short_kernel<T, 4, false>);
    else if (a.vocab <= 8 * a.lanes) a.mask ? go(logprob_short_kernel<T, 8, true>) : go(logprob_short_kernel<T, 8, false>);
    else a.mask ? go(logprob_short_kernel<T, 32, true>) : go(logprob_short_kernel<T, 32, false>);
    return;
  }
  if (a.mask) forward_long<T, true>(a, s);
  else forward_long<T, false>(a, s);
}
template <typename T>
void backward(LogprobGradArgs a, cudaStream_t s) {
  if (a.vocab <= kNarrow) {
    const unsigned blocks = short_blocks(a.vocab, a.rows, &a.lanes);
    const auto go = [&](auto kernel) { launch_kernel(kernel, blocks, 128, 0, s, a); };
    if (a.vocab <= 4 * a.lanes) a.mask ? go(logprob_short_bwd_kernel<T, 4, true>) : go(logprob_short_bwd_kernel<T, 4, false>);
    else a.mask ? go(logprob_short_bwd_kernel<T, 8, true>) : go(logprob_short_bwd_kernel<T, 8, false>);
    return;
  }
  constexpr int V = 16 / sizeof(T);
  const bool alike = (address(a.x) - address(a.dx)) % 16 == 0 && (a.ld - a.vocab) * static_cast<long long>(sizeof(T)) % 16 == 0;
  const int per_chunk = 32 * kChunkVecs * (alike ? V : 1);
  a.chunks = (a.vocab + per_chunk - 1) / per_chunk;
  const long long blocks = (a.rows * a.chunks + kChunkThreads / 32 - 1) / (kChunkThreads / 32);
  const auto go = [&](auto kernel) { launch_kernel(kernel, static_cast<unsigned>(blocks), kChunkThreads, 0, s, a); };
  if (alike) a.mask ? go(logprob_long_bwd_kernel<T, V, true>) : go(logprob_long_bwd_kernel<T, V, false>);
  else a.mask ? go(logprob_long_bwd_kernel<T, 1, true>) : go(logprob_long_bwd_kernel<T, 1, false>);
}

int check_rows(const void* x, long long ld, const void* mask, const void* tokens, int tokens_bytes, long long rows, int vocab, int type, float temperature) {
  if (!x) return MXK_ERR_NULL;
  if (rows <= 0 || vocab <= 0 || vocab > 0x3fffffff || ld < 0) return MXK_ERR_DIMS;
  // blocks of the longest grid: eight for a row, or one for 1024 entries
  if (rows > 0x7fffffffll / 8 || rows * ((vocab + 1023) / 1024) > 0x7fffffff) return MXK_ERR_DIMS;
  if (!known_type(type) || !(temperature >= kColdest && temperature <= kHottest)) return MXK_ERR_UNSUPPORTED;
  if (tokens && tokens_bytes != 4 && tokens_bytes != 8) return MXK_ERR_UNSUPPORTED;
  if (address(x) % type_bytes(type) || (tokens && address(tokens) % tokens_bytes)) return MXK_ERR_ALIGN;
  (void)mask;
  return MXK_OK;
}

}  // namespace
}  // namespace mxk

extern "C" {

int mxk_token_logprob_fwd(const void* logits, long long ld, const uint8_t* mask, long long mask_ld, const void* tokens, int tokens_bytes,
                          float* log_prob, float* entropy, float* top_value, long long* top_index, float* stats, long long rows, int vocab,
                          int top, int type, float temperature, mxk_stream_t stream) {
  using namespace mxk;
  if (const int status = check_rows(logits, ld, mask, tokens, tokens_bytes, rows, vocab, type, temperature)) return status;
  if ((tokens && !log_prob) || (top > 0 && (!top_value || !top_index))) return MXK_ERR_NULL;
  if (top < 0 || top > vocab) return MXK_ERR_DIMS;
  if (top > kMaxTop) return MXK_ERR_UNSUPPORTED;
  if (!aligned16(stats)) return MXK_ERR_ALIGN;
  LogprobArgs a{};
  a.x = logits; a.ld = ld; a.mask = mask; a.mask_ld = mask_ld;
  a.tokens = tokens; a.tokens_bytes = tokens_bytes;
  a.log_prob = log_prob; a.entropy = entropy; a.top_value = top_value; a.top_index = top_index;
  a.stats = reinterpret_cast<float4*>(stats);
  a.rows = rows; a.vocab = vocab; a.top = top;
  a.inv_t = 1.f / temperature;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (type == MXK_F32) forward<float>(a, s);
  else if (type == MXK_BF16) forward<__nv_bfloat16>(a, s);
  else forward<__half>(a, s);
  return launch_status();
}

int mxk_token_logprob_bwd(const void* logits, long long ld, const uint8_t* mask, long long mask_ld, const void* tokens, int tokens_bytes,
                          const float* stats, const float* g_log_prob, long long g_log_prob_ld, const float* g_entropy, long long g_entropy_ld,
                          void* dlogits, long long rows, int vocab, int type, float temperature, mxk_stream_t stream) {
  using namespace mxk;
  if (const int status = check_rows(logits, ld, mask, tokens, tokens_bytes, rows, vocab, type, temperature)) return status;
  if (!stats || !dlogits) return MXK_ERR_NULL;
  if (!aligned16(stats) || address(dlogits) % type_bytes(type)) return MXK_ERR_ALIGN;
  LogprobGradArgs a{};
  a.x = logits; a.ld = ld; a.mask = mask; a.mask_ld = mask_ld;
  a.tokens = tokens; a.tokens_bytes = tokens_bytes;
  a.stats = reinterpret_cast<const float4*>(stats);
  a.g_lp = g_log_prob; a.g_lp_ld = g_log_prob_ld; a.g_h = g_entropy; a.g_h_ld = g_entropy_ld;
  a.dx = dlogits;
  a.rows = rows; a.vocab = vocab;
  a.inv_t = 1.f / temperature;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (type == MXK_F32) backward<float>(a, s);
  else if (type == MXK_BF16) backward<__nv_bfloat16>(a, s);
  else backward<__half>(a, s);
  return launch_status();
}

}  // extern "C"
