// Rows of a table by token, out[n] = scale W[ids[n]], and the table's gradient, dW[v] = scale sum_{n: ids[n] = v} dy[n].
//
// The gradient is summed in float32 over the tokens' positions in ascending order, so it is the same in every run: positions
// are sorted by token (radix sort, stable), then the sorted list is cut into runs of kRun positions.  A group of threads owns a
// run and a column tile, keeps one token's sum in registers, and writes a token's row when the token ends.  A token that
// crosses the runs' borders (a frequent one) leaves a partial sum per run, and a second kernel adds these up in order.  Rows
// that no position has are zeroed by further blocks of the same launch, which look their tokens up in the sorted list: the
// gradient is written once, without a pass that clears it first.
//
// The sort is one cluster of eight blocks: each warp owns a stretch of the list, counts are exchanged through distributed
// shared memory, and the cluster's barrier stands where separate launches would; the lists themselves pass through L2.
//
// Bytes bound all of it but the sort: ids, dy once, and the table's size once.
#include <cooperative_groups.h>

#include "elements.cuh"

namespace mxk {
namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------------------------------------------------- lookup
// `lanes` (a power of two) threads share a row of `vecs` vectors.
template <typename T, int V, typename I>
__global__ void __launch_bounds__(128)
embedding_fwd_kernel(const I* __restrict__ ids, const T* __restrict__ table, T* __restrict__ out, long long rows, long long vocab, int dim,
                     int lanes, float scale) {
  enter_kernel();
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
constexpr int kHeld = 8;                                     // keys a lane keeps between the two walks over its warp's stretch
constexpr int kSortSmem = (kSortWarps * kMaxBins + 4 * kMaxBins + 64) * 4;

struct SortLists {
  uint32_t *key[2], *pos[2];
};

// keys: tokens, `vocab` for those outside of the table (they sort last).  passes * digits cover vocab + 1 values.
template <typename I>
__global__ void __launch_bounds__(kSortThreads)
sort_tokens_kernel(const I* __restrict__ ids, SortLists lists, int rows, uint32_t vocab, int passes, int digits) {
  enter_kernel();
  extern __shared__ uint32_t sort_smem[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, bins = 1 << digits;
  uint32_t* const counts = sort_smem;                        // [warp][bin]: counts, then where the warp's next key of a bin goes
  uint32_t* const total = counts + kSortWarps * kMaxBins;    // [bin] of this block, read by the others
  uint32_t* const start = total + kMaxBins;                  // [bin]
  uint32_t* const sums = start + kMaxBins;                   // of warps, in the scan over bins
  const int stretches = blocks * kSortWarps;
  const int len = ((rows + stretches - 1) / stretches + 31) / 32 * 32;      // of a warp, in whole 32s
  const long long begin64 = static_cast<long long>(rank * kSortWarps + warp) * len;
  const int begin = begin64 < rows ? static_cast<int>(begin64) : rows;
  const int end = rows - begin < len ? rows : begin + len;
  const bool held = len <= 32 * kHeld;

  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digits;
    const uint32_t* const key_in = lists.key[(pass + 1) & 1];
    const uint32_t* const pos_in = lists.pos[(pass + 1) & 1];
    uint32_t* const key_out = lists.key[pass & 1];
    uint32_t* const pos_out = lists.pos[pass & 1];
    // (what other blocks of the cluster wrote in the pass before is read past L1, which would not know)
    const auto read = [&](int i, uint32_t& key, uint32_t& pos) {
      if (pass == 0) {
        const long long id = static_cast<long long>(ids[i]);
        key = id >= 0 && id < static_cast<long long>(vocab) ? static_cast<uint32_t>(id) : vocab;
        pos = i;
      } else {
        key = __ldcg(key_in + i);
        pos = __ldcg(pos_in + i);
      }
    };
    for (int b = threadIdx.x; b < kSortWarps * bins; b += kSortThreads) counts[b / bins * kMaxBins + b % bins] = 0;
    __syncthreads();
    uint32_t key[kHeld], pos[kHeld];
    const auto count = [&](bool in, uint32_t k) {
      const uint32_t digit = in ? (k >> shift) & (bins - 1) : bins;      // those behind the end form a class of their own
      const uint32_t peers = __match_any_sync(0xffffffffu, digit);
      if (in && lane == __ffs(peers) - 1) counts[warp * kMaxBins + digit] += __popc(peers);
      __syncwarp();
    };
    if (held) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (begin + j * 32 + lane < end) read(begin + j * 32 + lane, key[j], pos[j]);
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (begin + j * 32 < end) count(begin + j * 32 + lane < end, key[j]);
    } else {
      for (int i = begin; i < end; i += 32) {
        uint32_t k = 0, p;
        if (i + lane < end) read(i + lane, k, p);
        count(i + lane < end, k);
      }
    }
    __syncthreads();
    // over the warps of the block: counts -> keys of the bin in the warps before; the block's total
    uint32_t mine = 0;
    if (threadIdx.x < bins) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = counts[w * kMaxBins + threadIdx.x];
        counts[w * kMaxBins + threadIdx.x] = mine;
        mine += c;
      }
      total[threadIdx.x] = mine;
    }
    cluster.sync();
    // over the blocks, and over the bins
    uint32_t before = 0, all = 0;
    if (threadIdx.x < bins) {
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
    if (threadIdx.x < bins) {
      uint32_t base = scan - all + before;
      for (int w = 0; w < warp; ++w) base += sums[w];
      start[threadIdx.x] = base;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < kSortWarps * bins; b += kSortThreads) counts[b / bins * kMaxBins + b % bins] += start[b % bins];
    __syncthreads();
    const auto place = [&](bool in, uint32_t k, uint32_t p) {
      const uint32_t digit = in ? (k >> shift) & (bins - 1) : bins;
      const uint32_t peers = __match_any_sync(0xffffffffu, digit);
      if (in) {
        const uint32_t to = counts[warp * kMaxBins + digit] + __popc(peers & ((1u << lane) - 1));
        key_out[to] = k;
        pos_out[to] = p;
      }
      __syncwarp();
      if (in && lane == __ffs(peers) - 1) counts[warp * kMaxBins + digit] += __popc(peers);
      __syncwarp();
    };
    if (held) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (begin + j * 32 < end) place(begin + j * 32 + lane < end, key[j], pos[j]);
    } else {
      for (int i = begin; i < end; i += 32) {
        uint32_t k = 0, p = 0;
        if (i + lane < end) read(i + lane, k, p);
        place(i + lane < end, k, p);
      }
    }
    __threadfence();
    cluster.sync();     // (also: nobody's totals are overwritten, or gone, while they are read)
  }
}

// --------------------------------------------------------------------------------------------------------------- sums
constexpr int kRun = 32;           // sorted positions of a run
constexpr int kSumThreads = 256;
constexpr int kAhead = 8;          // rows that are fetched at once
constexpr int kZeroRows = 32;      // table rows that a block looks after

struct SumArgs {
  const uint32_t *key, *pos;       // sorted; keys of `vocab` are of no row
  const void* dy;
  void* dw;
  float* partial;                  // [run][2][dim]: of the token that began before the run, and of the one that goes on behind it
  int rows, dim, group, runs;      // group: threads of a run and column tile
  uint32_t vocab;
  int tiles;                       // column tiles
  unsigned run_blocks;
  float scale;
};

// First index in the sorted keys that is not below `k`; the whole warp looks.
__device__ __forceinline__ int lower_bound_warp(const uint32_t* __restrict__ key, int n, uint32_t k) {
  int lo = 0, hi = n;              // key[lo - 1] < k <= key[hi]
  const int lane = threadIdx.x % 32;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const bool below = at < hi && key[at] < k;
    const int many = __popc(__ballot_sync(0xffffffffu, below));     // a prefix of the lanes
    if (many == 0) return lo;
    const int last = lo + (many - 1) * step;
    const int next = last + step;
    lo = last + 1;
    hi = next < hi ? next : hi;
  }
  return lo;
}

template <typename T, int V>
__global__ void __launch_bounds__(kSumThreads)
embedding_sum_kernel(const SumArgs a) {
  enter_kernel();
  T* const dw = static_cast<T*>(a.dw);
  if (blockIdx.x >= a.run_blocks) {    // rows of the table that no position has
    __shared__ uint32_t present;
    __shared__ int range[2];
    const long long first = static_cast<long long>(blockIdx.x - a.run_blocks) * kZeroRows;
    const int many = a.vocab - first < kZeroRows ? static_cast<int>(a.vocab - first) : kZeroRows;
    if (threadIdx.x == 0) present = 0;
    if (threadIdx.x < 64) {
      const int at = lower_bound_warp(a.key, a.rows, static_cast<uint32_t>(first) + (threadIdx.x < 32 ? 0 : many));
      if (threadIdx.x % 32 == 0) range[threadIdx.x / 32] = at;
    }
    __syncthreads();
    for (int i = range[0] + threadIdx.x; i < range[1]; i += kSumThreads) {
      const uint32_t bit = 1u << (a.key[i] - static_cast<uint32_t>(first));
      if (i == range[0] || a.key[i - 1] != a.key[i]) atomicOr(&present, bit);
    }
    __syncthreads();
    const uint32_t have = present;
    float zero[V];
#pragma unroll
    for (int i = 0; i < V; ++i) zero[i] = 0.f;
    const Vec<T, V> z = Vec<T, V>::pack(zero);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int r = warp; r < many; r += kSumThreads / 32) {
      if (have >> r & 1) continue;
      T* const row = dw + (first + r) * a.dim;
      for (int c = lane * V; c < a.dim; c += 32 * V) z.store_stream(row + c);
    }
    return;
  }
  const int per_block = kSumThreads / a.group;
  const long long item = static_cast<long long>(blockIdx.x) * per_block + threadIdx.x / a.group;
  const int run = static_cast<int>(item / a.tiles);
  const int c = (static_cast<int>(item % a.tiles) * a.group + threadIdx.x % a.group) * V;
  if (run >= a.runs || c >= a.dim) return;
  const int begin = run * kRun, end = a.rows - begin < kRun ? a.rows : begin + kRun;
  const T* const dy = static_cast<const T*>(a.dy) + c;
  float* const part = a.partial + static_cast<long long>(run) * 2 * a.dim + c;
  uint32_t token = a.key[begin];
  bool whole = begin == 0 || a.key[begin - 1] != token;      // the token's first position is in this run
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.f;
  const auto leave = [&](bool ends) {
    if (token < a.vocab) {
      if (whole && ends) {
        float x[V];
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = sum[i] * a.scale;
        Vec<T, V>::pack(x).store_stream(dw + static_cast<long long>(token) * a.dim + c);
      } else {
        float* const to = part + (whole ? a.dim : 0);
#pragma unroll
        for (int i = 0; i < V; ++i) to[i] = sum[i];
      }
    }
  };
  for (int i = begin; i < end; i += kAhead) {
    Vec<T, V> row[kAhead];
    uint32_t key[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j < end) {
        key[j] = a.key[i + j];
        if (key[j] < a.vocab) row[j] = Vec<T, V>::load_stream(dy + static_cast<long long>(a.pos[i + j]) * a.dim);
      }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j < end) {
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
  leave(end == a.rows || a.key[end] != token);
}

// Tokens that cross a run's end: the partial sums of the runs they cover.  A block per run in which such a token begins; its
// warps share the runs, in order, and their sums are added in order.
template <typename T>
__global__ void __launch_bounds__(kSumThreads)
embedding_join_kernel(const SumArgs a) {
  enter_kernel();
  constexpr int kWarps = kSumThreads / 32;
  __shared__ float sums[kWarps][32];
  const int run = blockIdx.x, last = run * kRun + kRun - 1;
  if (last + 1 >= a.rows) return;
  const uint32_t token = a.key[last];
  if (token >= a.vocab || a.key[last + 1] != token) return;
  // begins in this run: its first position is here
  if (a.key[run * kRun] == token && run > 0 && a.key[run * kRun - 1] == token) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int stop = lower_bound_warp(a.key, a.rows, token + 1);
  const int count = (stop - 1) / kRun - run + 1;             // runs with a part of it
  const int share = (count + kWarps - 1) / kWarps;
  for (int c0 = blockIdx.y * 32; c0 < a.dim; c0 += gridDim.y * 32) {
    const int c = c0 + lane;
    float sum = 0.f;
    if (c < a.dim) {
      const int from = warp * share, to = from + share < count ? from + share : count;
#pragma unroll 8
      for (int r = from; r < to; ++r) sum += a.partial[(static_cast<long long>(run + r) * 2 + (r == 0)) * a.dim + c];
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < a.dim) {
#pragma unroll
      for (int w = 1; w < kWarps; ++w) sum += sums[w][lane];
      static_cast<T*>(a.dw)[static_cast<long long>(token) * a.dim + c] = from_float<T>(sum * a.scale);
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
void forward(const I* ids, const void* table, void* out, long long rows, long long vocab, int dim, float scale, cudaStream_t s) {
  const int lanes = power_of_two(dim / V, 32), per_block = 128 / lanes;
  launch_kernel(embedding_fwd_kernel<T, V, I>, static_cast<unsigned>((rows + per_block - 1) / per_block), 128, 0, s, ids, static_cast<const T*>(table),
                static_cast<T*>(out), rows, vocab, dim, lanes, scale);
}
template <typename T, typename I>
void forward_by_width(const I* ids, const void* table, void* out, long long rows, long long vocab, int dim, float scale, cudaStream_t s) {
  const int width = access_bytes(address(table) | address(out) | static_cast<uintptr_t>(dim) * sizeof(T));
  if (width == 16) forward<T, 16 / sizeof(T)>(ids, table, out, rows, vocab, dim, scale, s);
  else if (width == 8) forward<T, 8 / sizeof(T)>(ids, table, out, rows, vocab, dim, scale, s);
  else forward<T, 1>(ids, table, out, rows, vocab, dim, scale, s);
}
template <typename I>
void forward_by_type(int type, const I* ids, const void* table, void* out, long long rows, long long vocab, int dim, float scale, cudaStream_t s) {
  if (type == MXK_F32) forward_by_width<float>(ids, table, out, rows, vocab, dim, scale, s);
  else if (type == MXK_BF16) forward_by_width<__nv_bfloat16>(ids, table, out, rows, vocab, dim, scale, s);
  else forward_by_width<__half>(ids, table, out, rows, vocab, dim, scale, s);
}

template <typename T, int V>
void sum(SumArgs a, cudaStream_t s) {
  a.group = power_of_two(a.dim / V, kSumThreads);
  a.tiles = (a.dim / V + a.group - 1) / a.group;
  const int per_block = kSumThreads / a.group;
  a.run_blocks = static_cast<unsigned>((static_cast<long long>(a.runs) * a.tiles + per_block - 1) / per_block);
  const unsigned zero_blocks = (a.vocab + kZeroRows - 1) / kZeroRows;
  launch_kernel(embedding_sum_kernel<T, V>, a.run_blocks + zero_blocks, kSumThreads, 0, s, a);
  if (a.runs > 1) {
    const int tiles = (a.dim + 31) / 32;
    launch_kernel(embedding_join_kernel<T>, dim3(a.runs, tiles < 4 ? tiles : 4), kSumThreads, 0, s, a);
  }
}
template <typename T>
void sum_by_width(const SumArgs& a, cudaStream_t s) {
  const int width = access_bytes(address(a.dy) | address(a.dw) | static_cast<uintptr_t>(a.dim) * sizeof(T));
  if (width == 16) sum<T, 16 / sizeof(T)>(a, s);
  else if (width == 8) sum<T, 8 / sizeof(T)>(a, s);
  else sum<T, 1>(a, s);
}

int runs_of(long long rows) { return static_cast<int>((rows + kRun - 1) / kRun); }
size_t list_bytes(long long rows) { return (static_cast<size_t>(rows) * 4 + 255) / 256 * 256; }
int check_sizes(long long rows, long long vocab, int dim, int type) {
  if (rows < 0 || vocab <= 0 || dim <= 0 || rows > 0x7fffffff - 65536 || vocab > 0x7fffffff - 65536) return MXK_ERR_DIMS;
  return known_type(type) ? MXK_OK : MXK_ERR_UNSUPPORTED;
}

template <typename I>
int sort_tokens(const I* ids, const SortLists& lists, int rows, uint32_t vocab, int* passes_out, cudaStream_t s) {
  int bits = 1;
  while ((static_cast<uint64_t>(vocab) >> bits) != 0) ++bits;       // of the values 0 .. vocab
  const int passes = (bits + kMaxDigits - 1) / kMaxDigits, digits = (bits + passes - 1) / passes;
  *passes_out = passes;
  const int status = allow_smem<sort_tokens_kernel<I>, kSortSmem>();
  if (status) return status;
  // a short list is one block's: less than a barrier's worth of work for each of eight
  const unsigned blocks = rows <= 2048 ? 1 : 8;
  launch_kernel_clusters(sort_tokens_kernel<I>, blocks, blocks, kSortThreads, kSortSmem, s, ids, lists, rows, vocab, passes, digits);
  return MXK_OK;
}

}  // namespace
}  // namespace mxk

extern "C" {

int mxk_embedding_fwd(const void* ids, int ids_bytes, const void* table, void* out, long long rows, long long vocab, int dim, int type,
                      float scale, mxk_stream_t stream) {
  using namespace mxk;
  if (!ids || !table || !out) return MXK_ERR_NULL;
  if (rows <= 0) return MXK_ERR_DIMS;
  if (const int status = check_sizes(rows, vocab, dim, type)) return status;
  if (ids_bytes != 4 && ids_bytes != 8) return MXK_ERR_UNSUPPORTED;
  if (address(ids) % ids_bytes || (address(table) | address(out)) % type_bytes(type)) return MXK_ERR_ALIGN;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (ids_bytes == 8) forward_by_type(type, static_cast<const long long*>(ids), table, out, rows, vocab, dim, scale, s);
  else forward_by_type(type, static_cast<const int*>(ids), table, out, rows, vocab, dim, scale, s);
  return launch_status();
}

size_t mxk_embedding_bwd_workspace_bytes(long long rows, int dim) {
  if (rows <= 0 || dim <= 0) return 0;
  return 4 * mxk::list_bytes(rows) + static_cast<size_t>(mxk::runs_of(rows)) * 2 * dim * 4;
}

int mxk_embedding_bwd(const void* ids, int ids_bytes, const void* dy, void* dw, void* workspace, size_t workspace_bytes, long long rows,
                      long long vocab, int dim, int type, float scale, mxk_stream_t stream) {
  using namespace mxk;
  if (!dw || (rows > 0 && (!ids || !dy))) return MXK_ERR_NULL;
  if (const int status = check_sizes(rows, vocab, dim, type)) return status;
  if (ids_bytes != 4 && ids_bytes != 8) return MXK_ERR_UNSUPPORTED;
  if (address(ids) % ids_bytes || (address(dy) | address(dw)) % type_bytes(type)) return MXK_ERR_ALIGN;
  if (rows > 0 && (!workspace || workspace_bytes < mxk_embedding_bwd_workspace_bytes(rows, dim))) return MXK_ERR_WORKSPACE;
  if (rows > 0 && !aligned16(workspace)) return MXK_ERR_ALIGN;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  SumArgs a{};
  a.dy = dy; a.dw = dw;
  a.rows = static_cast<int>(rows); a.dim = dim; a.runs = runs_of(rows);
  a.vocab = static_cast<uint32_t>(vocab);
  a.scale = scale;
  if (rows > 0) {
    uint8_t* const base = static_cast<uint8_t*>(workspace);
    SortLists lists;
    for (int i = 0; i < 2; ++i) {
      lists.key[i] = reinterpret_cast<uint32_t*>(base + i * list_bytes(rows));
      lists.pos[i] = reinterpret_cast<uint32_t*>(base + (2 + i) * list_bytes(rows));
    }
    a.partial = reinterpret_cast<float*>(base + 4 * list_bytes(rows));
    int passes = 0;
    const int status = ids_bytes == 8 ? sort_tokens(static_cast<const long long*>(ids), lists, a.rows, a.vocab, &passes, s)
                                      : sort_tokens(static_cast<const int*>(ids), lists, a.rows, a.vocab, &passes, s);
    if (status) return status;
    a.key = lists.key[(passes - 1) & 1];
    a.pos = lists.pos[(passes - 1) & 1];
  }
  if (type == MXK_F32) sum_by_width<float>(a, s);
  else if (type == MXK_BF16) sum_by_width<__nv_bfloat16>(a, s);
  else sum_by_width<__half>(a, s);
  return launch_status();
}

}  // extern "C"
