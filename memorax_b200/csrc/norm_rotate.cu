// Norms of query and key heads and the position rotation in one pass, and their gradients:
//   n = x r w,  r = 1 / sqrt(mean(x^2) + eps)  (rms)  or  1 / max(|x|, eps), no w  (l2)  or  1 (none)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * base^(-2 i / R)
// for the R / 2 pairs of a head's first R elements: (i, i + R / 2), or neighbours (2 i, 2 i + 1); the others stay n.
// Backward, with g the cotangents turned back by t and n' = x r:
//   dx = r (w g - n' mean(n' w g))  (l2: the sum in place of the mean; nothing of n' where eps took |x|'s place)
//   dw = sum over tokens and heads of n' g.
//
// Angles: a far position times a rate in float32 would lose the turn it is in.  The rates are held as turns in 64-bit fixed
// point (2^-64 of a turn), a position's phase is one integer product whose overflow drops the whole turns, and its top 32 bits
// go to sinpi / cospi.  A token's sines and cosines are computed once and serve all of its heads.
//
// A lane holds sixteen elements of a head: as many pairs of vectors as that makes, so that both halves of each rotated pair
// are its own and only the norm goes over lanes.  A warp takes one side (queries or keys) of a token, several heads at a time.
// The backward pass sums dw in registers over the tokens of a warp, then over a block's warps, and a second launch adds the
// blocks' rows in a fixed order.  Bytes bound it: x in, y out; backward x and dy in, dx out.
#include "elements.cuh"

namespace mxk {
namespace {

constexpr int kWarps = 4;            // of a block
constexpr int kMaxDim = 512;

struct Side {                        // queries or keys
  const void* x;
  long long sb, st, sh;              // strides of x in elements
  const void* dy;
  long long db, dt, dh;
  const void* w;                     // (d) or null
  void* out;                         // (B, T, heads, d): y, or dx
  int heads;
};
struct RotateArgs {
  Side side[2];
  const void* positions;             // int32 / int64, or null: 0 .. T - 1
  long long pb, pt;
  const unsigned long long* turns;   // (R / 2) turns per position, 2^-64
  float* partial;                    // backward: [block][2][d]
  long long tokens;
  int T, dim, rot, lanes, norm, parts[2];   // lanes of a head; warps that share a side's heads
  int positions_bytes;
  float eps;
};

// kNeighbours: pairs (2 i, 2 i + 1).  A lane's units are pairs of vectors of V; unit u of a head is made of
//   halves:      (u, u + R / 2V) where u < R / 2V, else the two vectors from R / V + 2 (u - R / 2V) on
//   neighbours:  (2 u, 2 u + 1)
template <typename T, int V, bool kNeighbours, bool kBwd, bool kWeights>
__global__ void __launch_bounds__(kWarps * 32)
norm_rotate_kernel(const RotateArgs a) {
  enter_kernel();
  constexpr int kUnits = 8 / V;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int L = a.lanes, per_turn = 32 / L, sub = lane / L, l = lane % L;
  const int half = a.rot / (2 * V);                       // rotated units of a head
  const int parts = a.parts[0] + a.parts[1];
  int first[kUnits], second[kUnits];                      // the units' elements
  bool in[kUnits], turned[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int unit = l + u * L;
    in[u] = unit < a.dim / (2 * V);
    turned[u] = in[u] && unit < half;
    if (kNeighbours) first[u] = 2 * unit * V, second[u] = first[u] + V;
    else if (unit < half) first[u] = unit * V, second[u] = first[u] + a.rot / 2;
    else first[u] = a.rot + 2 * (unit - half) * V, second[u] = first[u] + V;
  }
  float dw[2][16];
  if (kBwd && kWeights) {
#pragma unroll
    for (int i = 0; i < 16; ++i) dw[0][i] = dw[1][i] = 0.f;
  }
  const long long items = a.tokens * parts;
  for (long long item = static_cast<long long>(blockIdx.x) * kWarps + warp; item < items; item += static_cast<long long>(gridDim.x) * kWarps) {
    const long long token = item / parts;
    const int part = static_cast<int>(item - token * parts);
    const int k = part >= a.parts[0];
    const Side& s = a.side[k];
    const int share = part - (k ? a.parts[0] : 0), shares = a.parts[k];
    const long long b = token / a.T, t = token - b * a.T;
    unsigned long long position = t;
    if (a.positions) {
      const long long at = b * a.pb + t * a.pt;
      position = a.positions_bytes == 8 ? static_cast<const unsigned long long*>(a.positions)[at]
                                        : static_cast<unsigned long long>(static_cast<long long>(static_cast<const int*>(a.positions)[at]));
    }
    float cs[8], sn[8];
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float c = 1.f, v = 0.f;
        if (turned[u]) {
          // neighbours: the pairs of a unit's two vectors follow one another
          const unsigned long long phase = position * a.turns[(l + u * L) * V + i];
          // the top 32 bits, signed: half turns in [-1, 1)
          sincospif(static_cast<float>(static_cast<int>(phase >> 32)) * 0x1p-31f, &v, &c);
        }
        cs[u * V + i] = c;
        sn[u * V + i] = v;
      }
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = 1.f;
    if (kWeights) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
        if (in[u]) {
          const T* const wp = static_cast<const T*>(s.w);
          Vec<T, V>::load(wp + first[u]).unpack(w + 2 * u * V);
          Vec<T, V>::load(wp + second[u]).unpack(w + (2 * u + 1) * V);
        }
    }
    const T* const x0 = static_cast<const T*>(s.x) + b * s.sb + t * s.st;
    const T* const g0 = kBwd ? static_cast<const T*>(s.dy) + b * s.db + t * s.dt : nullptr;
    T* const y0 = static_cast<T*>(s.out) + token * s.heads * a.dim;
    const int step = per_turn * shares;
    const int turns = (s.heads + step - 1) / step;
#pragma unroll 2
    for (int turn = 0; turn < turns; ++turn) {
      const int h = (turn * shares + share) * per_turn + sub;
      const bool live = h < s.heads;
      float x[16], g[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = g[i] = 0.f;
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
        if (in[u] && live) {
          const T* const xp = x0 + h * s.sh;
          Vec<T, V>::load_stream(xp + first[u]).unpack(x + 2 * u * V);
          Vec<T, V>::load_stream(xp + second[u]).unpack(x + (2 * u + 1) * V);
          if (kBwd) {
            const T* const gp = g0 + h * s.dh;
            Vec<T, V>::load_stream(gp + first[u]).unpack(g + 2 * u * V);
            Vec<T, V>::load_stream(gp + second[u]).unpack(g + (2 * u + 1) * V);
          }
        }
      // pair i of unit u: elements (p, q) of the lane's sixteen
      const auto turn_pairs = [&](float* v, float sign) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          if (!turned[u]) continue;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int p = kNeighbours ? 2 * u * V + 2 * i : 2 * u * V + i, q = kNeighbours ? p + 1 : p + V;
            const float c = cs[u * V + i], d = sign * sn[u * V + i], e = v[p], f = v[q];
            v[p] = e * c - f * d;
            v[q] = f * c + e * d;
          }
        }
      };
      if (kBwd) turn_pairs(g, -1.f);
      float squares = 0.f, along = 0.f;
      if (a.norm != MXK_NORM_NONE) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          squares = fmaf(x[i], x[i], squares);
          if (kBwd) along = fmaf(x[i], g[i] * w[i], along);
        }
        for (int off = 1; off < L; off <<= 1) {
          squares += __shfl_xor_sync(0xffffffffu, squares, off);
          if (kBwd) along += __shfl_xor_sync(0xffffffffu, along, off);
        }
      }
      float r = 1.f;
      bool held = false;                                  // eps in the place of the length
      if (a.norm == MXK_NORM_RMS) r = 1.f / sqrtf(squares / a.dim + a.eps);
      if (a.norm == MXK_NORM_L2) {
        const float length = sqrtf(squares);
        held = !(length > a.eps);
        r = 1.f / (held ? a.eps : length);
      }
      if (kBwd) {
        const float back = a.norm == MXK_NORM_NONE || held ? 0.f : along * r * r / (a.norm == MXK_NORM_RMS ? a.dim : 1);
        if (kWeights) {           // (an index that is not known here would put the sums into memory)
          if (k == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) dw[0][i] = fmaf(x[i] * r, g[i], dw[0][i]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) dw[1][i] = fmaf(x[i] * r, g[i], dw[1][i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = r * (g[i] * w[i] - x[i] * back);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = x[i] * r * w[i];
        turn_pairs(g, 1.f);
      }
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
        if (in[u] && live) {
          T* const yp = y0 + static_cast<long long>(h) * a.dim;
          Vec<T, V>::pack(g + 2 * u * V).store_stream(yp + first[u]);
          Vec<T, V>::pack(g + (2 * u + 1) * V).store_stream(yp + second[u]);
        }
    }
  }
  if (kBwd && kWeights) {
    // lanes of the same elements, then the block's warps one after the other
    __shared__ float sums[kWarps][2][kMaxDim];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float v = dw[k][i];
        for (int off = L; off < 32; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        const int u = i / (2 * V);
        if (sub == 0 && in[u]) sums[warp][k][(i / V % 2 ? second[u] : first[u]) + i % V] = v;
      }
    }
    __syncthreads();
    float* const to = a.partial + static_cast<long long>(blockIdx.x) * 2 * a.dim;
    for (int i = threadIdx.x; i < 2 * a.dim; i += kWarps * 32) {
      const int k = i / a.dim, c = i % a.dim;
      float v = sums[0][k][c];
#pragma unroll
      for (int q = 1; q < kWarps; ++q) v += sums[q][k][c];
      to[i] = v;
    }
  }
}

// dw[c] = the sum of column c over the blocks' rows; a warp a column, lanes and then their sums in a fixed order
template <typename T>
__global__ void __launch_bounds__(256)
rotate_weights_kernel(const float* __restrict__ partial, int rows, int dim, T* dwq, T* dwk) {
  enter_kernel();
  const int c = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (c >= 2 * dim) return;
  float sum = 0.f;
#pragma unroll 4
  for (int r = lane; r < rows; r += 32) sum += partial[static_cast<long long>(r) * 2 * dim + c];
#pragma unroll
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  T* const to = c < dim ? dwq : dwk;
  if (lane == 0 && to) to[c % dim] = from_float<T>(sum);
}

constexpr int kBwdBlocks = 8 * kNumSMs;     // each leaves a row of partial sums

int blocks_of(long long items, bool rows) {
  const long long want = (items + kWarps - 1) / kWarps;
  const long long most = rows ? kBwdBlocks : 0x7fffffff;
  return static_cast<int>(want < most ? want : most);
}

template <typename T, int V, bool kBwd>
void launch(const RotateArgs& a, bool neighbours, bool weights, int blocks, cudaStream_t s) {
  const auto go = [&](auto kernel) { launch_kernel(kernel, blocks, kWarps * 32, 0, s, a); };
  if (neighbours) weights ? go(norm_rotate_kernel<T, V, true, kBwd, true>) : go(norm_rotate_kernel<T, V, true, kBwd, false>);
  else weights ? go(norm_rotate_kernel<T, V, false, kBwd, true>) : go(norm_rotate_kernel<T, V, false, kBwd, false>);
}
template <typename T, bool kBwd>
void launch_by_width(const RotateArgs& a, int width, bool neighbours, bool weights, int blocks, cudaStream_t s) {
  constexpr int kWide = 16 / sizeof(T);
  if (width >= kWide) launch<T, kWide, kBwd>(a, neighbours, weights, blocks, s);
  else if (sizeof(T) == 2 && width >= 4) launch<T, 4, kBwd>(a, neighbours, weights, blocks, s);
  else launch<T, 1, kBwd>(a, neighbours, weights, blocks, s);
}

size_t partial_bytes(int dim) { return static_cast<size_t>(kBwdBlocks) * 2 * dim * 4; }

int run(const mxk_rotate* r, bool bwd, void* dwq, void* dwk, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (!r || !r->turns) return MXK_ERR_NULL;
  if (r->batch <= 0 || r->steps <= 0 || r->dim <= 0 || r->dim > kMaxDim || r->rot <= 0 || r->rot > r->dim || r->batch > 0x7fffffff || r->steps > 0x7fffffff) return MXK_ERR_DIMS;
  if (r->dim % 2 || r->rot % 2 || !known_type(r->type) || r->norm < MXK_NORM_NONE || r->norm > MXK_NORM_L2) return MXK_ERR_UNSUPPORTED;
  if (r->positions && r->positions_bytes != 4 && r->positions_bytes != 8) return MXK_ERR_UNSUPPORTED;
  const int size = type_bytes(r->type);
  RotateArgs a{};
  uintptr_t bits = 0;
  const bool weights = r->side[0].w || r->side[1].w;
  for (int k = 0; k < 2; ++k) {
    const mxk_rotate_side& s = r->side[k];
    if (!s.x || !s.out || (bwd && !s.dy)) return MXK_ERR_NULL;
    if (s.heads <= 0 || s.heads > 65536) return MXK_ERR_DIMS;
    if (weights && (!s.w || r->norm != MXK_NORM_RMS)) return MXK_ERR_UNSUPPORTED;   // both or none, and of the rms norm
    // (a stride along an extent of one is never used)
    const long long sb = r->batch > 1 ? s.sb : 0, st = r->steps > 1 ? s.st : 0, sh = s.heads > 1 ? s.sh : 0;
    bits |= address(s.x) | address(s.out) | address(s.w) | static_cast<uintptr_t>(sb | st | sh) * size;
    a.side[k].x = s.x; a.side[k].sb = sb; a.side[k].st = st; a.side[k].sh = sh;
    if (bwd) {
      const long long db = r->batch > 1 ? s.db : 0, dt = r->steps > 1 ? s.dt : 0, dh = s.heads > 1 ? s.dh : 0;
      bits |= address(s.dy) | static_cast<uintptr_t>(db | dt | dh) * size;
      a.side[k].dy = s.dy; a.side[k].db = db; a.side[k].dt = dt; a.side[k].dh = dh;
    }
    a.side[k].w = s.w; a.side[k].out = s.out; a.side[k].heads = s.heads;
  }
  if (bits % size) return MXK_ERR_ALIGN;
  if (bwd && weights && (!workspace || workspace_bytes < partial_bytes(r->dim))) return MXK_ERR_WORKSPACE;
  a.positions = r->positions; a.pb = r->pb; a.pt = r->pt; a.positions_bytes = r->positions_bytes;
  a.turns = r->turns;
  a.tokens = static_cast<long long>(r->batch) * r->steps;
  a.T = static_cast<int>(r->steps); a.dim = r->dim; a.rot = r->rot; a.norm = r->norm; a.eps = r->eps;
  a.partial = static_cast<float*>(workspace);
  // elements of an access: both vectors of a unit have to be whole, in the rotated part and behind it
  int width = access_bytes(bits) / size;
  while (width > 1 && (r->dim % (2 * width) || r->rot % (2 * width))) width /= 2;
  a.lanes = 1;
  while (a.lanes * 16 < r->dim) a.lanes *= 2;
  // a side's heads are shared by several warps until there are about sixteen warps an SM; each computes the angles again
  const long long enough = 16ll * kNumSMs;
  for (int k = 0; k < 2; ++k) {
    const int turns = (a.side[k].heads + 32 / a.lanes - 1) / (32 / a.lanes);
    long long parts = (enough + 2 * a.tokens - 1) / (2 * a.tokens);
    a.parts[k] = static_cast<int>(parts < turns ? parts : turns);
  }
  const int blocks = blocks_of(a.tokens * (a.parts[0] + a.parts[1]), bwd && weights);
  const bool neighbours = r->interleaved != 0;
  const auto go = [&](auto one) {
    using T = decltype(one);
    if (bwd) {
      launch_by_width<T, true>(a, width, neighbours, weights, blocks, stream);
      if (weights)
        launch_kernel(rotate_weights_kernel<T>, (2 * r->dim + 7) / 8, 256, 0, stream, a.partial, blocks, r->dim, static_cast<T*>(dwq), static_cast<T*>(dwk));
    } else {
      launch_by_width<T, false>(a, width, neighbours, weights, blocks, stream);
    }
  };
  if (r->type == MXK_F32) go(float{});
  else if (r->type == MXK_BF16) go(__nv_bfloat16{});
  else go(__half{});
  return launch_status();
}

}  // namespace
}  // namespace mxk

extern "C" {

int mxk_norm_rotate_fwd(const mxk_rotate* args, mxk_stream_t stream) {
  return mxk::run(args, false, nullptr, nullptr, nullptr, 0, static_cast<cudaStream_t>(stream));
}

size_t mxk_norm_rotate_bwd_workspace_bytes(int dim) { return dim > 0 && dim <= mxk::kMaxDim ? mxk::partial_bytes(dim) : 0; }

int mxk_norm_rotate_bwd(const mxk_rotate* args, void* dw_query, void* dw_key, void* workspace, size_t workspace_bytes, mxk_stream_t stream) {
  return mxk::run(args, true, dw_query, dw_key, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
