// Rows of a table by token, out[n] = scale W[ids[n]], and the table's gradient, dW[v] = scale sum_{n: ids[n] = v} dy[n].
//
// The gradient is summed in float32 over the tokens' positions in ascending order, so it is the same in every run: positions
// are sorted by token (radix sort, stable), then the sorted list is cut into runs of kRun positions.  A group of threads owns a
// run and a column tile, keeps one token's sum in registers, and writes a token's row when the token ends.  A token that
// crosses the runs' borders (a frequent one) leaves a partial sum per run, and a second kernel adds these up in order.
//
// The sort is one cluster of up to sixteen blocks that hold the list in their shared memory, up to 262144 positions: each warp owns a
// stretch, counts and keys are exchanged through distributed shared memory, and the cluster's barrier stands where separate
// launches would.  (Through L2 instead, a pass of 65536 keys takes 16 us, and twice that while others write; longer lists do.)
// A key's place among its warp's equal ones comes from a ballot for each bit.  The forward pass sorts, since it has the tokens: the
// lookup neither needs the sort nor waits for it, and 130 SMs look up while it runs.  The sort also marks the tokens that there
// are, in a bit for each row of the table, and further blocks of the summing launch clear the rows that no position has: the
// gradient is written once.  (Clearing all of it while the sort runs takes longer: both launches are bound by what they write.)
//
// Bytes bound it: ids and the rows that are looked up, and dy and the table's size once.  65536 tokens of 1024 bf16 features into
// 131072 rows, both passes 117 us: the sort, 24 us, beside 35 of looking up (42 MB of distinct rows in, 134 out); 69 of summing
// and clearing (403 MB, 5.8 TB/s); 14.5 of joining, the chain of the most frequent token's runs.  16000 tokens of 512 into 50001 rows:
// the sort 14.8 (latency: two passes, two cluster barriers each), the sums 16.8, the join 4 to 7.  64 tokens: 2.1, a launch.
#include <cooperative_groups.h>

#include "elements.cuh"

namespace mxk {
namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------------------------------------------------- lookup
// `lanes` (a power of two) threads share a row of `vecs` vectors.  kBeside: behind the sort on the stream, but at work while it
// runs: that lets its successors come up only once everything in front of it has ended, so there is nothing to wait for in front.
// The last block waits for the sort's end instead, so that whoever waits for this launch has waited for both.
template <typename T, int V, typename I, bool kBeside>
__global__ void __launch_bounds__(128)
embedding_fwd_kernel(const I* ids, const T* table, T* __restrict__ out, long long rows, long long vocab, int dim,
                     int lanes, float scale) {
  if (!kBeside) enter_kernel();
  else if (blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per_block = 128 / lanes, lane = threadIdx.x % lanes;
  const long long n = static_cast<long long>(blockIdx.x) * per_block + threadIdx.x / lanes;
  if (n >= rows) return;
  const long long id = static_cast<long long>(ids[n]);
  const bool known = id >= 0 && id < vocab;
  const T* const src = table + (known ? id : 0) * dim;
  T* const dst = out + n * dim;
#pragma unroll 4
  for (int c = lane * V; c < dim; c += lanes * V) {
    float x[V];
    if (known) {
      Vec<T, V>::load(src + c).unpack(x);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] *= scale;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = 0.f;
    }
    Vec<T, V>::pack(x).store_stream(dst + c);
  }
}

// --------------------------------------------------------------------------------------------------------------- sort
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kMaxDigits = 9, kMaxBins = 1 << kMaxDigits;   // bits of a pass, and its bins
constexpr int kHeld = 16;                                    // keys a lane holds between the two walks over its warp's stretch
constexpr int kMaxShared = 16 * kSortThreads * kHeld;        // longest list in the cluster's shared memory
constexpr int kSortSmem = (kSortWarps * kMaxBins + 2 * kMaxBins + 64) * 4;
constexpr int kSharedSmem = kSortSmem + kSortThreads * kHeld * 8;

struct SortLists {
  uint2* pair[2];                  // (key, position)
};

// keys: tokens, `vocab` for those outside of the table (they sort last).  passes * digits cover vocab + 1 values.
// kShared: a block holds the keys of its warps' stretches; else they pass through the lists in global memory.
template <typename I, bool kShared>
__global__ void __launch_bounds__(kSortThreads)
sort_tokens_kernel(const I* ids, SortLists lists, int rows, uint32_t vocab, int passes, int digits, uint32_t inverse, uint32_t* __restrict__ present) {
  // (in this order: the lookup behind it starts with the second and does not wait)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ uint32_t sort_smem[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, bins = 1 << digits;
  uint32_t* const counts = sort_smem + warp * kMaxBins;      // [bin] of this warp: counts, then keys of the bin before its next one
  uint32_t* const total = sort_smem + kSortWarps * kMaxBins; // [bin] of this block, read by the others
  uint32_t* const start = total + kMaxBins;                  // [bin]: where this block's begin
  uint32_t* const sums = start + kMaxBins;                   // of warps, in the scan over bins
  uint2* const held = reinterpret_cast<uint2*>(sort_smem + kSortSmem / 4);   // (key, position), kShared
  const int stretches = blocks * kSortWarps;
  const int len = ((rows + stretches - 1) / stretches + 31) / 32 * 32;       // of a warp, in whole 32s
  const int part = len * kSortWarps;                                         // of a block
  const long long begin64 = static_cast<long long>(rank * kSortWarps + warp) * len;
  const int begin = begin64 < rows ? static_cast<int>(begin64) : rows;
  const int end = rows - begin < len ? rows : begin + len;
  for (int b = lane; b < bins; b += 32) counts[b] = 0;
  __syncwarp();
  for (long long i = rank * kSortThreads + threadIdx.x; i < (static_cast<long long>(vocab) + 31) / 32; i += blocks * kSortThreads) present[i] = 0;

  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digits;
    const uint2* const in = lists.pair[(pass + 1) & 1];
    uint2* const out = lists.pair[pass & 1];
    const auto read = [&](int i) {
      if (pass == 0) {
        const long long id = static_cast<long long>(ids[i]);
        return make_uint2(id >= 0 && id < static_cast<long long>(vocab) ? static_cast<uint32_t>(id) : vocab, i);
      }
      // (what other blocks of the cluster wrote in the pass before is read past L1, which would not know)
      return kShared ? held[i - rank * part] : __ldcg(in + i);
    };
    uint2 pair[kHeld];
    const auto count = [&](bool there, uint32_t k) {
      if (there) atomicAdd(&counts[(k >> shift) & (bins - 1)], 1u);
    };
    if (kShared) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j) {
        pair[j] = make_uint2(0, 0);
        if (begin + j * 32 + lane < end) pair[j] = read(begin + j * 32 + lane);
      }
#pragma unroll
      for (int j = 0; j < kHeld; ++j) count(begin + j * 32 + lane < end, pair[j].x);
    } else {
      for (int i = begin + lane; i < end; i += 32) count(true, read(i).x);
    }
    __syncthreads();
    // over the warps of the block: counts -> keys of the bin in the warps before; the block's total
    if (threadIdx.x < bins) {
      uint32_t mine = 0, c[8];
      for (int w = 0; w < kSortWarps; w += 8) {
#pragma unroll
        for (int q = 0; q < 8; ++q) c[q] = sort_smem[(w + q) * kMaxBins + threadIdx.x];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          sort_smem[(w + q) * kMaxBins + threadIdx.x] = mine;
          mine += c[q];
        }
      }
      total[threadIdx.x] = mine;
    }
    cluster.sync();                                          // (also: every key of the pass before is in registers)
    // over the blocks, and over the bins
    uint32_t before = 0, all = 0;
    if (threadIdx.x < bins) {
#pragma unroll 4
      for (int r = 0; r < blocks; ++r) {
        const uint32_t c = cluster.map_shared_rank(total, r)[threadIdx.x];
        before += r < rank ? c : 0;
        all += c;
      }
    }
    uint32_t scan = all;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, scan, off);
      if (lane >= off) scan += up;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    const uint32_t base = __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0);     // of the warps before this one, in every lane
    if (threadIdx.x < bins) start[threadIdx.x] = base + scan - all + before;
    __syncthreads();
    const auto place = [&](bool there, uint2 p) {
      const uint32_t digit = (p.x >> shift) & (bins - 1);
      uint32_t peers = __ballot_sync(0xffffffffu, there);
#pragma unroll
      for (int bit = 0; bit < kMaxDigits; ++bit) {           // (above the digit's bits: zero in every lane)
        const bool one = digit & (1u << bit);
        peers &= __ballot_sync(0xffffffffu, one) ^ (one ? 0u : 0xffffffffu);
      }
      uint32_t at = 0;
      if (there) {
        at = counts[digit];
        const uint32_t to = start[digit] + at + __popc(peers & ((1u << lane) - 1));
        if (kShared) {
          const uint32_t r = __umulhi(to, inverse);          // to / part
          cluster.map_shared_rank(held, r)[to - r * part] = p;
        } else {
          out[to] = p;
        }
      }
      __syncwarp();
      if (there && lane == __ffs(peers) - 1) counts[digit] = at + __popc(peers);
      __syncwarp();
    };
    if (kShared) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (begin + j * 32 < end) place(begin + j * 32 + lane < end, pair[j]);
    } else {
      for (int i = begin; i < end; i += 32) place(i + lane < end, i + lane < end ? read(i + lane) : make_uint2(0, 0));
      __threadfence();
    }
    for (int b = lane; b < bins; b += 32) counts[b] = 0;     // (this warp's own, for the next pass)
    cluster.sync();     // (also: nobody's totals are overwritten, or gone, while they are read)
  }
  uint2* const out = lists.pair[(passes - 1) & 1];
  for (int i = begin + lane; i < end; i += 32) {
    const uint2 p = kShared ? held[i - rank * part] : __ldcg(out + i);
    uint32_t before = ~p.x;                                  // (the first position of a block of the cluster marks its token once more)
    if (kShared ? i > rank * part : i > 0) before = kShared ? held[i - 1 - rank * part].x : __ldcg(out + i - 1).x;
    if (p.x < vocab && before != p.x) atomicOr(present + p.x / 32, 1u << p.x % 32);
    if (kShared) out[i] = p;
  }
}

// --------------------------------------------------------------------------------------------------------------- sums
constexpr int kRun = 32;           // sorted positions of a run
constexpr int kSumThreads = 256;
constexpr int kAhead = 8;          // rows that are fetched at once
constexpr int kClearRows = 32;     // table rows that a block looks after: a word of `present`

struct SumArgs {
  const uint32_t* present;         // a bit for each row of the table
  const uint2* pair;               // (key, position), sorted by key; keys of `vocab` are of no row
  const void* dy;
  void* dw;
  float* partial;                  // [run][2][dim]: of the token that began before the run, and of the one that goes on behind it
  int rows, dim, group, runs;      // group: threads of a run and column tile
  uint32_t vocab;
  int tiles;                       // column tiles
  unsigned run_blocks;
  uint32_t vecs, inverse;          // vectors of a row, ceil(2^32 / vecs)
  float scale;
};

template <typename T, int V>
__global__ void __launch_bounds__(kSumThreads, 3)
embedding_sum_kernel(const SumArgs a) {
  enter_kernel();
  T* const dw = static_cast<T*>(a.dw);
  if (blockIdx.x >= a.run_blocks) {
    const uint32_t word = blockIdx.x - a.run_blocks, have = a.present[word];
    const long long first = static_cast<long long>(word) * kClearRows;
    const uint32_t rows = a.vocab - first < kClearRows ? static_cast<uint32_t>(a.vocab - first) : kClearRows;
    float zero[V];
#pragma unroll
    for (int i = 0; i < V; ++i) zero[i] = 0.f;
    const Vec<T, V> z = Vec<T, V>::pack(zero);
    T* const base = dw + first * a.dim;
    // (a row of the block's at a time would leave lanes idle where rows are short)
    for (uint32_t i = threadIdx.x; i < rows * a.vecs; i += kSumThreads) {
      const uint32_t r = a.vecs == 1 ? i : a.inverse ? __umulhi(i, a.inverse) : i / a.vecs;
      if (!(have >> r & 1)) z.store_stream(base + static_cast<long long>(i) * V);
    }
    return;
  }
  const int per_block = kSumThreads / a.group;
  const long long item = static_cast<long long>(blockIdx.x) * per_block + threadIdx.x / a.group;
  const int run = static_cast<int>(item / a.tiles);
  const int c = (static_cast<int>(item % a.tiles) * a.group + threadIdx.x % a.group) * V;
  if (run >= a.runs || c >= a.dim) return;
  const int begin = run * kRun, many = a.rows - begin < kRun ? a.rows - begin : kRun;
  const T* const dy = static_cast<const T*>(a.dy) + c;
  float* const part = a.partial + static_cast<long long>(run) * 2 * a.dim + c;
  uint32_t token = a.pair[begin].x;
  bool whole = begin == 0 || a.pair[begin - 1].x != token;      // the token's first position is in this run
  const uint32_t behind = begin + many < a.rows ? a.pair[begin + many].x : ~0u;
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.f;
  const auto leave = [&](bool ends) {
    if (token >= a.vocab) return;
    if (whole && ends) {
      float x[V];
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = sum[i] * a.scale;
      Vec<T, V>::pack(x).store_stream(dw + static_cast<long long>(token) * a.dim + c);
    } else {
      constexpr int kWide = V < 4 ? V : 4;                   // (a thread's columns begin at a multiple of V)
      float* const to = part + (whole ? a.dim : 0);
#pragma unroll
      for (int i = 0; i < V; i += kWide) Vec<float, kWide>::pack(sum + i).store(to + i);
    }
  };
  uint2 next[kAhead];                                        // the tokens and positions of the rows that come next
  const auto look = [&](int i) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) next[j] = i + j < many ? a.pair[begin + i + j] : make_uint2(~0u, 0);
  };
  look(0);
  for (int i = 0; i < many; i += kAhead) {
    Vec<T, V> row[kAhead];
    uint32_t key[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      key[j] = next[j].x;
      if (key[j] < a.vocab) row[j] = Vec<T, V>::load_stream(dy + static_cast<long long>(next[j].y) * a.dim);
    }
    look(i + kAhead);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j < many) {
        if (key[j] != token) {
          leave(true);
          token = key[j];
          whole = true;
#pragma unroll
          for (int e = 0; e < V; ++e) sum[e] = 0.f;
        }
        if (token < a.vocab) {
          float x[V];
          row[j].unpack(x);
#pragma unroll
          for (int e = 0; e < V; ++e) sum[e] += x[e];
        }
      }
  }
  leave(behind != token);
}

// Tokens that cross a run's end: the partial sums of the runs they cover, added in order, by the blocks of the run in which such a
// token begins.  Over few runs a warp takes a column tile; over many the warps share the runs, each for four tiles at once, so
// that the most frequent token, which the launch waits for, has loads enough under way.
template <typename T, int V>
__global__ void __launch_bounds__(kSumThreads)
embedding_join_kernel(const SumArgs a) {
  enter_kernel();
  constexpr int kWarps = kSumThreads / 32, kTile = 32 * V, kTiles = 4;
  __shared__ float sums[kWarps][kTiles * kTile];
  const int run = blockIdx.x, last = run * kRun + kRun - 1;
  if (last + 1 >= a.rows) return;
  const uint32_t token = a.pair[last].x;
  const uint32_t behind = a.pair[last + 1].x, first = a.pair[run * kRun].x, before = run > 0 ? a.pair[run * kRun - 1].x : ~token;
  if (token >= a.vocab || behind != token || (first == token && before == token)) return;     // does not cross, or begins before
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int count = 1;                                             // runs with a part of it: this one, and those that begin with it
  for (bool more = true; more; ) {
    bool same[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = run + count + j * 32 + lane;
      same[j] = at < a.runs && a.pair[static_cast<long long>(at) * kRun].x == token;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t with = __ballot_sync(0xffffffffu, same[j]);
      if (more) count += with == 0xffffffffu ? 32 : __ffs(~with) - 1;
      more = more && with == 0xffffffffu;
    }
  }
  const bool few = count <= kWarps;
  const auto part = [&](int r, int c) { return a.partial + (static_cast<long long>(run + r) * 2 + (r == 0)) * a.dim + c; };
  const auto leave = [&](int c, const float* sum) {
    T* const row = static_cast<T*>(a.dw) + static_cast<long long>(token) * a.dim + c;
#pragma unroll
    for (int i = 0; i < V; ++i) row[i] = from_float<T>(sum[i] * a.scale);
  };
  if (few) {
    for (int c = (blockIdx.y * kWarps + warp) * kTile + lane * V; c < a.dim; c += gridDim.y * kWarps * kTile) {
      Vec<float, V> all[kWarps];      // (all on their way before the first is added)
#pragma unroll
      for (int r = 0; r < kWarps; ++r)
        if (r < count) all[r] = Vec<float, V>::load(part(r, c));
      float sum[V];
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] = 0.f;
#pragma unroll
      for (int r = 0; r < kWarps; ++r)
        if (r < count) {
          float x[V];
          all[r].unpack(x);
#pragma unroll
          for (int i = 0; i < V; ++i) sum[i] += x[i];
        }
      leave(c, sum);
    }
    return;
  }
  const int share = (count + kWarps - 1) / kWarps;
  const int from = warp * share < count ? warp * share : count, to = from + share < count ? from + share : count;
  for (int c0 = blockIdx.y * kTiles * kTile; c0 < a.dim; c0 += gridDim.y * kTiles * kTile) {
    float sum[kTiles][V];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[t][i] = 0.f;
#pragma unroll 4
    for (int r = from; r < to; ++r)
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int c = c0 + t * kTile + lane * V;
        if (c < a.dim) {
          float x[V];
          Vec<float, V>::load(part(r, c)).unpack(x);
#pragma unroll
          for (int i = 0; i < V; ++i) sum[t][i] += x[i];
        }
      }
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < V; ++i) sums[warp][t * kTile + lane * V + i] = sum[t][i];
    __syncthreads();
    for (int i = threadIdx.x * V; i < kTiles * kTile && c0 + i < a.dim; i += kSumThreads * V) {
      float all[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        all[e] = sums[0][i + e];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) all[e] += sums[w][i + e];
      }
      leave(c0 + i, all);
    }
    __syncthreads();
  }
}

int power_of_two(int n, int most) {
  int p = 1;
  while (p < n && p < most) p *= 2;
  return p;
}

template <typename T, int V, typename I>
void forward(const I* ids, const void* table, void* out, long long rows, long long vocab, int dim, float scale, bool beside, cudaStream_t s) {
  const int lanes = power_of_two(dim / V, 32), per_block = 128 / lanes;
  const auto go = [&](auto kernel) {
    launch_kernel(kernel, static_cast<unsigned>((rows + per_block - 1) / per_block), 128, 0, s, ids, static_cast<const T*>(table), static_cast<T*>(out), rows, vocab, dim, lanes,
                  scale);
  };
  beside ? go(embedding_fwd_kernel<T, V, I, true>) : go(embedding_fwd_kernel<T, V, I, false>);
}
template <typename T, typename I>
void forward_by_width(const I* ids, const void* table, void* out, long long rows, long long vocab, int dim, float scale, bool beside, cudaStream_t s) {
  const int width = access_bytes(address(table) | address(out) | static_cast<uintptr_t>(dim) * sizeof(T));
  if (width == 16) forward<T, 16 / sizeof(T)>(ids, table, out, rows, vocab, dim, scale, beside, s);
  else if (width == 8) forward<T, 8 / sizeof(T)>(ids, table, out, rows, vocab, dim, scale, beside, s);
  else forward<T, 1>(ids, table, out, rows, vocab, dim, scale, beside, s);
}
template <typename I>
void forward_by_type(int type, const I* ids, const void* table, void* out, long long rows, long long vocab, int dim, float scale, bool beside, cudaStream_t s) {
  if (type == MXK_F32) forward_by_width<float>(ids, table, out, rows, vocab, dim, scale, beside, s);
  else if (type == MXK_BF16) forward_by_width<__nv_bfloat16>(ids, table, out, rows, vocab, dim, scale, beside, s);
  else forward_by_width<__half>(ids, table, out, rows, vocab, dim, scale, beside, s);
}

template <typename T, int V>
void sum(SumArgs a, cudaStream_t s) {
  a.group = power_of_two(a.dim / V, kSumThreads);
  a.tiles = (a.dim / V + a.group - 1) / a.group;
  const int per_block = kSumThreads / a.group;
  const long long items = static_cast<long long>(a.runs) * a.tiles;
  a.run_blocks = static_cast<unsigned>((items + per_block - 1) / per_block);
  a.vecs = a.dim / V;
  a.inverse = a.vecs > 1 && a.vecs <= 8192 ? static_cast<uint32_t>(((1ull << 32) + a.vecs - 1) / a.vecs) : 0;     // exact for 32 rows of as many
  launch_kernel(embedding_sum_kernel<T, V>, a.run_blocks + (a.vocab + kClearRows - 1) / kClearRows, kSumThreads, 0, s, a);
  if (a.runs < 2) return;
  if (a.dim % 4 == 0) launch_kernel(embedding_join_kernel<T, 4>, dim3(a.runs, a.dim > 512 ? 2 : 1), kSumThreads, 0, s, a);
  else launch_kernel(embedding_join_kernel<T, 1>, a.runs, kSumThreads, 0, s, a);
}
template <typename T>
void sum_by_width(const SumArgs& a, cudaStream_t s) {
  const int width = access_bytes(address(a.dy) | address(a.dw) | static_cast<uintptr_t>(a.dim) * sizeof(T));
  if (width == 16) sum<T, 16 / sizeof(T)>(a, s);
  else if (width == 8) sum<T, 8 / sizeof(T)>(a, s);
  else sum<T, 1>(a, s);
}

int runs_of(long long rows) { return static_cast<int>((rows + kRun - 1) / kRun); }
size_t list_bytes(long long rows) { return (static_cast<size_t>(rows) * 8 + 255) / 256 * 256; }
size_t present_bytes(long long vocab) { return (static_cast<size_t>(vocab) + 31) / 32 * 4 / 256 * 256 + 256; }
int check_sizes(long long rows, long long vocab, int dim, int type) {
  if (rows < 0 || vocab <= 0 || dim <= 0 || dim > 1 << 24 || rows > 0x7fffffff - 65536 || vocab > 0x7fffffff - 65536) return MXK_ERR_DIMS;
  return known_type(type) ? MXK_OK : MXK_ERR_UNSUPPORTED;
}

// What the forward pass leaves for the backward: two lists (the sort's last pass writes one of them) and the marks.
struct Sorted {
  SortLists lists;
  uint32_t* present;
  int passes, digits;
  Sorted(void* p, long long rows, long long vocab) {
    uint8_t* const base = static_cast<uint8_t*>(p);
    for (int i = 0; i < 2; ++i) lists.pair[i] = reinterpret_cast<uint2*>(base + i * list_bytes(rows));
    present = reinterpret_cast<uint32_t*>(base + 2 * list_bytes(rows));
    int bits = 1;
    while ((static_cast<uint64_t>(vocab) >> bits) != 0) ++bits;     // of the values 0 .. vocab
    passes = (bits + kMaxDigits - 1) / kMaxDigits;
    digits = (bits + passes - 1) / passes;
  }
  const uint2* pairs() const { return lists.pair[(passes - 1) & 1]; }
};

template <typename I>
int sort_tokens(const I* ids, const Sorted& to, int rows, uint32_t vocab, cudaStream_t s) {
  const SortLists& lists = to.lists;
  const int passes = to.passes, digits = to.digits;
  const bool shared = rows <= kMaxShared;
  const int status = shared ? allow_smem<sort_tokens_kernel<I, true>, kSharedSmem>() : allow_smem<sort_tokens_kernel<I, false>, kSortSmem>();
  if (status) return status;
  // a short list is one block's: less than a barrier's worth of work for each of eight; a long one takes the largest cluster there
  // is (65536 keys: 31 us with eight blocks).  Sixteen blocks that each fill an SM need as many free ones side by side: a whole GPU has them, a
  // small partition of one may not, where the launch then fails.
  const int cluster = rows <= 2048 ? 1 : rows <= 32768 ? 8 : 16;
  if (cluster > 8) {
    const int wide = shared ? allow_wide_cluster<sort_tokens_kernel<I, true>>() : allow_wide_cluster<sort_tokens_kernel<I, false>>();
    if (wide) return wide;
  }
  const int stretches = cluster * kSortWarps, part = ((rows + stretches - 1) / stretches + 31) / 32 * 32 * kSortWarps;
  const uint32_t inverse = static_cast<uint32_t>(((1ull << 32) + part - 1) / part);     // exact for lists of up to 2^18 and parts of up to 2^14
  if (shared) launch_kernel_clusters(sort_tokens_kernel<I, true>, cluster, cluster, kSortThreads, kSharedSmem, s, ids, lists, rows, vocab, passes, digits, inverse, to.present);
  else launch_kernel_clusters(sort_tokens_kernel<I, false>, cluster, cluster, kSortThreads, kSortSmem, s, ids, lists, rows, vocab, passes, digits, inverse, to.present);
  return MXK_OK;
}

}  // namespace
}  // namespace mxk

extern "C" {

size_t mxk_embedding_sorted_bytes(long long rows, long long vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  return 2 * mxk::list_bytes(rows) + mxk::present_bytes(vocab);
}

int mxk_embedding_fwd(const void* ids, int ids_bytes, const void* table, void* out, void* sorted, size_t sorted_bytes, long long rows,
                      long long vocab, int dim, int type, float scale, mxk_stream_t stream) {
  using namespace mxk;
  if (!ids || !table || !out) return MXK_ERR_NULL;
  if (rows <= 0) return MXK_ERR_DIMS;
  if (const int status = check_sizes(rows, vocab, dim, type)) return status;
  if (ids_bytes != 4 && ids_bytes != 8) return MXK_ERR_UNSUPPORTED;
  if (address(ids) % ids_bytes || (address(table) | address(out)) % type_bytes(type) || !aligned16(sorted)) return MXK_ERR_ALIGN;
  if (sorted && sorted_bytes < mxk_embedding_sorted_bytes(rows, vocab)) return MXK_ERR_WORKSPACE;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto go = [&](const auto* tokens) {
    if (sorted) {
      if (const int status = sort_tokens(tokens, Sorted(sorted, rows, vocab), static_cast<int>(rows), static_cast<uint32_t>(vocab), s)) return status;
    }
    forward_by_type(type, tokens, table, out, rows, vocab, dim, scale, sorted != nullptr, s);
    return launch_status();
  };
  return ids_bytes == 8 ? go(static_cast<const long long*>(ids)) : go(static_cast<const int*>(ids));
}

size_t mxk_embedding_bwd_workspace_bytes(long long rows, int dim) {
  if (rows <= 0 || dim <= 0) return 0;
  return static_cast<size_t>(mxk::runs_of(rows)) * 2 * dim * 4;
}

int mxk_embedding_bwd(const void* sorted, size_t sorted_bytes, const void* dy, void* dw, void* workspace, size_t workspace_bytes, long long rows,
                      long long vocab, int dim, int type, float scale, mxk_stream_t stream) {
  using namespace mxk;
  if (!dw || (rows > 0 && (!sorted || !dy))) return MXK_ERR_NULL;
  if (const int status = check_sizes(rows, vocab, dim, type)) return status;
  if ((address(dy) | address(dw)) % type_bytes(type) || !aligned16(sorted) || !aligned16(workspace)) return MXK_ERR_ALIGN;
  if (rows > 0 && (!workspace || workspace_bytes < mxk_embedding_bwd_workspace_bytes(rows, dim) || sorted_bytes < mxk_embedding_sorted_bytes(rows, vocab))) return MXK_ERR_WORKSPACE;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (const cudaError_t e = cudaMemsetAsync(dw, 0, static_cast<size_t>(vocab) * dim * type_bytes(type), s)) return static_cast<int>(e);
    return MXK_OK;
  }
  const Sorted from(const_cast<void*>(sorted), rows, vocab);
  SumArgs a{};
  a.dy = dy; a.dw = dw;
  a.rows = static_cast<int>(rows); a.dim = dim; a.runs = runs_of(rows);
  a.vocab = static_cast<uint32_t>(vocab);
  a.scale = scale;
  a.pair = from.pairs();
  a.present = from.present;
  a.partial = static_cast<float*>(workspace);
  if (type == MXK_F32) sum_by_width<float>(a, s);
  else if (type == MXK_BF16) sum_by_width<__nv_bfloat16>(a, s);
  else sum_by_width<__half>(a, s);
  return launch_status();
}

}  // extern "C"
