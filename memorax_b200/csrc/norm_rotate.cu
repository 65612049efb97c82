// Norms of query and key heads and the position rotation in one pass, and their gradients:
//   n = x r w,  r = 1 / sqrt(mean(x^2) + eps)  (rms)  or  1 / max(|x|, eps), no w  (l2)  or  1 (none)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * base^(-2 i / R)
// for the R / 2 pairs of a head's first R elements: (i, i + R / 2), or neighbours (2 i, 2 i + 1); the others stay n.
// Backward, with g the cotangents turned back by t and n' = x r:
//   dx = r (w g - n' mean(n' w g))  (l2: the sum in place of the mean; nothing of n' where eps took |x|'s place)
//   dw = sum over tokens and heads of n' g.
//
// Angles: a far position times a rate in float32 would lose the turn it is in.  The rates are held as turns in 64-bit fixed
// point (2^-64 of a turn), a position's phase is one integer product whose overflow drops the whole turns.  Its top two bits say
// which quarter of the turn, the thirty behind them where in it; within half a quarter either side polynomials in the square do.
// A token's sines and cosines are computed once and serve all of its heads.
//
// A lane holds sixteen elements of a head: as many pairs of vectors as that makes, so that both halves of each rotated pair
// are its own and only the norm goes over lanes.  A block takes one side (queries or keys) of a tile of tokens: its threads
// compute the tile's sines and cosines once, into shared memory in the order in which lanes read them, then its warps walk the
// tile's heads, several at a time, across tokens (one key head a token fills a warp as well as 32), the next ones' loads under
// way while a warp works.  The backward pass sums dw in registers over all of a block's tiles, then over its warps, and a
// second launch adds the blocks' rows in a fixed order.
//
// Bytes bound it in float32: x in, y out; backward x and dy in, dx out (16384 tokens of 40 heads of 128: 108 and 161 us, 6.2 TB/s).
// In 16 bits it is latency: the same heads in bf16 take 71 and 98 us (4.7 and 5.1 TB/s) with the same instructions and half of the
// bytes under way, a turn of 1 KB for each of 18 and 14 warps an SM; loads are what warps wait for most, 60 and 55 % of the issue slots are
// in use.  65536 tokens of 8 + 8 heads of 128 without weights, as the delta rule takes them: 115 and 154 us (4.7 and 5.2 TB/s).  Slower were: rows through a
// ring in shared memory (cp.async, three turns ahead), blocks that walk several tiles in the forward pass, four warps a block.
// A tile's positions are loaded together before its angles (one behind the other: 75 and 102 us, and with one head a side 19 forward
// for 12).  64 tokens of 16 heads take 3.1 us, a launch.
#include "elements.cuh"
#include "packed.cuh"

namespace mxk {
namespace {

constexpr int kWarps = 2;            // of a block: a short prologue's worth of tiles, many blocks to level them (four: 5 us more on 5555 tokens x 12 heads)
constexpr int kMaxDim = 512;
constexpr int kTableBytes = 32 * 1024;

struct Side {                        // queries or keys
  const void* x;
  long long sb, st, sh;              // strides of x in elements
  const void* dy;
  long long db, dt, dh;
  const void* w;                     // (d) or null
  void* out;                         // (B, T, heads, d): y, or dx
  int heads;
  uint32_t inverse;                  // ceil(2^32 / heads): row / heads for rows below 2^16; 0 for one head
};
struct RotateArgs {
  Side side[2];
  const void* positions;             // int32 / int64, or null: 0 .. T - 1
  long long pb, pt;
  const unsigned long long* turns;   // (R / 2) turns per position, 2^-64
  float* partial;                    // backward: [block][d]
  int tokens, T, dim, rot, norm;
  int log_lanes;                     // of a head
  float inv_dim;
  int tile[2], first_key;            // tokens of a tile; the first block of the keys
  int positions_bytes;
  float eps;
};

// Sine and cosine of 2 pi u / 2^32.  Least-squares fits on Chebyshev nodes, reweighted towards equal errors: 5e-9 and 5e-11 off
// over the half quarter either side, below a float's step.
__device__ __forceinline__ void sine_cosine(uint32_t u, float* s, float* c) {
  const uint32_t quarter = (u + 0x20000000u) >> 30;
  const float x = static_cast<float>(static_cast<int>(u - (quarter << 30))) * 0x1p-30f, z = x * x;      // in quarters, -1/2 .. 1/2
  const float sine = x * fmaf(z, fmaf(z, fmaf(z, -0.00460217733472635f, 0.07968022821530597f), -0.6459634786602615f), 1.5707963219673886f);
  const float cosine = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 0.0009036317569995774f, -0.02086007134892384f), 0.2536692039449117f), -1.2337005406477641f), 1.f);
  const float a = quarter & 1 ? cosine : sine, b = quarter & 1 ? sine : cosine;
  *s = __uint_as_float(__float_as_uint(a) ^ (quarter & 2) << 30);
  *c = __uint_as_float(__float_as_uint(b) ^ (quarter + 1 & 2) << 30);
}

// kNeighbours: pairs (2 i, 2 i + 1).  A lane's units are pairs of vectors of V; unit u of a head is made of
//   halves:      (u, u + R / 2V) where u < R / 2V, else the two vectors from R / V + 2 (u - R / 2V) on
//   neighbours:  (2 u, 2 u + 1)
template <typename T, int V, bool kNeighbours, bool kBwd, bool kWeights>
__global__ void __launch_bounds__(kWarps * 32, kBwd ? 8 : 10)
norm_rotate_kernel(const RotateArgs a) {
  enter_kernel();
  constexpr int kUnits = 8 / V;
  extern __shared__ float4 rotate_smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int log_l = a.log_lanes, L = 1 << log_l, per_turn = 32 >> log_l, group = lane >> log_l, l = lane & (L - 1);
  const int half = a.rot / (2 * V);                       // rotated units of a head
  const int k = static_cast<int>(blockIdx.x) >= a.first_key;
  const Side& s = a.side[k];
  const int heads = s.heads, tile_tokens = a.tile[k], dim = a.dim;
  const T* const x0 = static_cast<const T*>(s.x);         // (parameters at an index that is not known here are loads)
  const T* const dy0 = static_cast<const T*>(s.dy);
  const long long sh = s.sh, dh = s.dh;
  const uint32_t inverse = s.inverse;
  float* const table = reinterpret_cast<float*>(rotate_smem);                 // [token][cos, cos, sin, sin][lane of a head] float4
  long long* const x_at = reinterpret_cast<long long*>(rotate_smem + (tile_tokens * 4 << log_l));   // [token]
  long long* const g_at = x_at + tile_tokens;
  unsigned long long* const position_of = reinterpret_cast<unsigned long long*>(g_at + tile_tokens);
  int first[kUnits], second[kUnits];                      // the units' elements
  bool in[kUnits], turned[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int unit = l + u * L;
    in[u] = unit < dim / (2 * V);
    turned[u] = in[u] && unit < half;
    if (kNeighbours) first[u] = 2 * unit * V, second[u] = first[u] + V;
    else if (unit < half) first[u] = unit * V, second[u] = first[u] + a.rot / 2;
    else first[u] = a.rot + 2 * (unit - half) * V, second[u] = first[u] + V;
  }
  // sixteen elements as eight pairs; units that a head does not have stay zero
  F2 w[8], dw[8];
  float w1[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w1[i] = 1.f;
  if (kWeights) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
      if (in[u]) {
        const T* const wp = static_cast<const T*>(s.w);
        Vec<T, V>::load(wp + first[u]).unpack(w1 + 2 * u * V);
        Vec<T, V>::load(wp + second[u]).unpack(w1 + (2 * u + 1) * V);
      }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = F2(w1[2 * i], w1[2 * i + 1]), dw[i] = F2(0.f);
  Vec<T, V> xr[2 * kUnits], gr[2 * kUnits];               // of the row that comes next
#pragma unroll
  for (int u = 0; u < 2 * kUnits; ++u) xr[u].bits = gr[u].bits = typename Vec<T, V>::raw{};

  const int blocks = k ? gridDim.x - a.first_key : a.first_key;
  for (long long t0 = static_cast<long long>(k ? blockIdx.x - a.first_key : blockIdx.x) * tile_tokens; t0 < a.tokens; t0 += static_cast<long long>(blocks) * tile_tokens) {
    const int many = a.tokens - t0 < tile_tokens ? static_cast<int>(a.tokens - t0) : tile_tokens;
    __syncthreads();                                      // (nobody reads the tile before any more)
    const unsigned b0 = static_cast<unsigned>(t0) / static_cast<unsigned>(a.T), from = static_cast<unsigned>(t0) - b0 * a.T;
    // (positions first, all of the tile's on their way together: each behind the one before took most of a tile with few heads)
    for (int token = threadIdx.x; token < many; token += kWarps * 32) {
      unsigned b = b0, t = from + token;
      if (t >= static_cast<unsigned>(a.T)) {
        const unsigned more = t / static_cast<unsigned>(a.T);
        b += more;
        t -= more * a.T;
      }
      x_at[token] = b * s.sb + t * s.st;
      g_at[token] = b * s.db + t * s.dt;
      unsigned long long position = t;
      if (a.positions) {
        const long long at = b * a.pb + t * a.pt;
        position = a.positions_bytes == 8 ? static_cast<const unsigned long long*>(a.positions)[at]
                                          : static_cast<unsigned long long>(static_cast<long long>(static_cast<const int*>(a.positions)[at]));
      }
      position_of[token] = position;
    }
    __syncthreads();
    // pair e of lane `of`, the same of every token
    for (int slot = threadIdx.x & ((8 << log_l) - 1); slot < 8 << log_l; slot += kWarps * 32) {
      const int e = slot >> log_l, of = slot & (L - 1), unit = of + e / V * L;
      const unsigned long long turns = unit < half ? a.turns[unit * V + e % V] : 0;
      float* to = table + ((e / 4 << log_l) + of) * 4 + e % 4;
      const int stride = 8 << log_l < kWarps * 32 ? kWarps * 32 >> (3 + log_l) : 1;
      for (int token = threadIdx.x >> (3 + log_l); token < many; token += stride) {
        float c, v;
        sine_cosine(static_cast<uint32_t>(position_of[token] * turns >> 32), &v, &c);
        to[token * 16 << log_l] = c;
        to[(token * 16 << log_l) + (8 << log_l)] = v;
      }
    }
    __syncthreads();

    const int rows = many * heads;
    T* const out = static_cast<T*>(s.out) + t0 * heads * dim;
    int token_next = 0, row_next = 0;
    const auto fetch = [&](int turn) {
      row_next = turn * per_turn + group;
      const int row = row_next < rows ? row_next : rows - 1;          // (behind the last: any row, which is not stored)
      const int token = inverse ? __umulhi(row, inverse) : row, h = row - token * heads;
      token_next = token;
      const T* const xp = x0 + x_at[token] + h * sh;
      const T* const gp = kBwd ? dy0 + g_at[token] + h * dh : nullptr;
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
        if (in[u]) {
          xr[2 * u] = Vec<T, V>::load_stream(xp + first[u]);
          xr[2 * u + 1] = Vec<T, V>::load_stream(xp + second[u]);
          if (kBwd) {
            gr[2 * u] = Vec<T, V>::load_stream(gp + first[u]);
            gr[2 * u + 1] = Vec<T, V>::load_stream(gp + second[u]);
          }
        }
    };
    fetch(warp);
    for (int turn = warp; turn * per_turn < rows; turn += kWarps) {
      float x1[16], g1[16];
#pragma unroll
      for (int u = 0; u < 2 * kUnits; ++u) {
        xr[u].unpack(x1 + u * V);
        if (kBwd) gr[u].unpack(g1 + u * V);
      }
      F2 x[8], g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = F2(x1[2 * i], x1[2 * i + 1]);
        if (kBwd) g[i] = F2(g1[2 * i], g1[2 * i + 1]);
      }
      const bool live = row_next < rows;
      const float4* const turns_of = rotate_smem + (token_next * 4 << log_l) + l;
      T* const yp = out + row_next * dim;
      fetch(turn + kWarps);
      float cs[8], sn[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 c = turns_of[j << log_l], v = turns_of[(j + 2) << log_l];
        cs[4 * j] = c.x, cs[4 * j + 1] = c.y, cs[4 * j + 2] = c.z, cs[4 * j + 3] = c.w;
        sn[4 * j] = v.x, sn[4 * j + 1] = v.y, sn[4 * j + 2] = v.z, sn[4 * j + 3] = v.w;
      }
      // (a, b) -> (a c - b s, b c + a s), backward by -s; what is not turned is not touched (infinities)
      const auto turn_pairs = [&](F2* v) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          if (!turned[u]) continue;
          if constexpr (kNeighbours || V == 1) {          // the pairs themselves are neighbours
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float c = cs[u * V + i], d = kBwd ? -sn[u * V + i] : sn[u * V + i];
              F2& p = v[u * V + i];
              p = fma(p.swapped(), F2(-d, d), mul(p, F2(c)));
            }
          } else {                                        // two rotated pairs at once
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              const int at = u * V + 2 * i;
              const F2 c(cs[at], cs[at + 1]), d(sn[at], sn[at + 1]);
              F2 &p = v[u * V + i], &q = v[u * V + V / 2 + i];
              const F2 e = p;
              p = kBwd ? fma(q, d, mul(e, c)) : sub(mul(e, c), mul(q, d));
              q = kBwd ? sub(mul(q, c), mul(e, d)) : fma(e, d, mul(q, c));
            }
          }
        }
      };
      if (kBwd) turn_pairs(g);
      F2 squares2(0.f), along2(0.f);
      float squares = 0.f, along = 0.f;
      F2 wg[8];
      if (kBwd) {
#pragma unroll
        for (int i = 0; i < 8; ++i) wg[i] = kWeights ? mul(g[i], w[i]) : g[i];
      }
      if (a.norm != MXK_NORM_NONE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          squares2 = fma(x[i], x[i], squares2);
          if (kBwd) along2 = fma(x[i], wg[i], along2);
        }
        squares = squares2.sum();
        if (kBwd) along = along2.sum();
        for (int off = 1; off < L; off <<= 1) {
          squares += __shfl_xor_sync(0xffffffffu, squares, off);
          if (kBwd) along += __shfl_xor_sync(0xffffffffu, along, off);
        }
      }
      float r = 1.f;
      bool held = false;                                  // eps in the place of the length
      if (a.norm == MXK_NORM_RMS) r = rsqrtf(fmaf(squares, a.inv_dim, a.eps));
      if (a.norm == MXK_NORM_L2) {
        const float length = sqrtf(squares);
        held = !(length > a.eps);
        r = 1.f / (held ? a.eps : length);
      }
      if (kBwd) {
        if (kWeights && !live) r = 0.f;                   // a row that is not there adds nothing to dw
        const float back = a.norm == MXK_NORM_NONE || held ? 0.f : -along * r * r * (a.norm == MXK_NORM_RMS ? a.inv_dim : 1.f);
        const F2 r2(r), back2(back);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const F2 n = mul(x[i], r2);
          if (kWeights) dw[i] = fma(n, g[i], dw[i]);
          g[i] = fma(n, back2, mul(wg[i], r2));
        }
      } else {
        const F2 r2(r);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = kWeights ? mul(mul(x[i], r2), w[i]) : mul(x[i], r2);
        turn_pairs(g);
      }
      if (live) {
        float y[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[2 * i] = g[i].lo(), y[2 * i + 1] = g[i].hi();
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
          if (in[u]) {
            Vec<T, V>::pack(y + 2 * u * V).store_stream(yp + first[u]);
            Vec<T, V>::pack(y + (2 * u + 1) * V).store_stream(yp + second[u]);
          }
      }
    }
  }
  if (kBwd && kWeights) {
    // lanes of the same elements, then the block's warps one after the other
    __shared__ float sums[kWarps][kMaxDim];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i % 2 ? dw[i / 2].hi() : dw[i / 2].lo();
      for (int off = L; off < 32; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      const int u = i / (2 * V);
      if (group == 0 && in[u]) sums[warp][(i / V % 2 ? second[u] : first[u]) + i % V] = v;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.dim; c += kWarps * 32) {
      float v = sums[0][c];
#pragma unroll
      for (int q = 1; q < kWarps; ++q) v += sums[q][c];
      a.partial[static_cast<long long>(blockIdx.x) * a.dim + c] = v;
    }
  }
}

// dw[c] = the sum of column c over the blocks' rows; a block takes 32 columns of a side, its warps share the rows in order
template <typename T>
__global__ void __launch_bounds__(1024)
rotate_weights_kernel(const float* partial, int first_key, int rows, int dim, T* dwq, T* dwk) {
  enter_kernel();
  __shared__ float sums[32][33];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, c = blockIdx.x * 32 + lane;
  const int from = blockIdx.y ? first_key : 0, to = blockIdx.y ? rows : first_key;
  float sum = 0.f;
  if (c < dim) {
#pragma unroll 8
    for (int r = from + warp; r < to; r += 32) sum += partial[static_cast<long long>(r) * dim + c];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp) return;
  for (int q = 1; q < 32; ++q) sum += sums[q][lane];
  T* const out = blockIdx.y ? dwk : dwq;
  if (c < dim && out) out[c] = from_float<T>(sum);
}

constexpr int kBwdBlocks = 8 * kNumSMs;     // each leaves a row of partial sums

template <typename T, int V, bool kBwd>
void launch(const RotateArgs& a, bool neighbours, bool weights, int blocks, size_t smem, cudaStream_t s) {
  const auto go = [&](auto kernel) { launch_kernel(kernel, blocks, kWarps * 32, smem, s, a); };
  if (neighbours) weights ? go(norm_rotate_kernel<T, V, true, kBwd, true>) : go(norm_rotate_kernel<T, V, true, kBwd, false>);
  else weights ? go(norm_rotate_kernel<T, V, false, kBwd, true>) : go(norm_rotate_kernel<T, V, false, kBwd, false>);
}
template <typename T, bool kBwd>
void launch_by_width(const RotateArgs& a, int width, bool neighbours, bool weights, int blocks, size_t smem, cudaStream_t s) {
  constexpr int kWide = 16 / sizeof(T);
  if (width >= kWide) launch<T, kWide, kBwd>(a, neighbours, weights, blocks, smem, s);
  else if (sizeof(T) == 2 && width >= 4) launch<T, 4, kBwd>(a, neighbours, weights, blocks, smem, s);
  else launch<T, 1, kBwd>(a, neighbours, weights, blocks, smem, s);
}

size_t partial_bytes(int dim) { return static_cast<size_t>(kBwdBlocks) * dim * 4; }

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
    if (s.heads <= 0 || s.heads > 65535) return MXK_ERR_DIMS;
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
    a.side[k].inverse = s.heads == 1 ? 0 : static_cast<uint32_t>(((1ull << 32) + s.heads - 1) / s.heads);
  }
  if (bits % size) return MXK_ERR_ALIGN;
  if (bwd && weights && (!workspace || workspace_bytes < partial_bytes(r->dim))) return MXK_ERR_WORKSPACE;
  a.positions = r->positions; a.pb = r->pb; a.pt = r->pt; a.positions_bytes = r->positions_bytes;
  a.turns = r->turns;
  if (r->batch * r->steps > 0x7fffffff) return MXK_ERR_DIMS;
  a.tokens = static_cast<int>(r->batch * r->steps);
  a.T = static_cast<int>(r->steps); a.dim = r->dim; a.inv_dim = 1.f / r->dim; a.rot = r->rot; a.norm = r->norm; a.eps = r->eps;
  a.partial = static_cast<float*>(workspace);
  // elements of an access: both vectors of a unit have to be whole, in the rotated part and behind it
  int width = access_bytes(bits) / size;
  while (width > 1 && (r->dim % (2 * width) || r->rot % (2 * width))) width /= 2;
  while ((16 << a.log_lanes) < r->dim) ++a.log_lanes;
  const int lanes = 1 << a.log_lanes;
  // Tiles: eight turns a warp where there are tokens for two blocks an SM of them, fewer where not; angles that fit the table,
  // rows that fit 16 bits.
  long long blocks[2], room = 0;
  for (int k = 0; k < 2; ++k) {
    const int heads = a.side[k].heads, per_turn = 32 / lanes;
    long long tile = (8ll * kWarps * per_turn + heads - 1) / heads;
    const long long spread = a.tokens / (2 * kNumSMs), most = kTableBytes / (64 * lanes), rows = 65535 / heads;
    for (const long long limit : {spread, most, rows}) tile = tile < limit ? tile : limit;
    if (tile < 1) tile = 1;
    a.tile[k] = static_cast<int>(tile);
    blocks[k] = (a.tokens + tile - 1) / tile;
    const long long bytes = tile * (64 * lanes + 24);
    room = room > bytes ? room : bytes;
  }
  // As many as are resident, each walks several tiles; shared by the sides' heads and the angles of a token, which take as long as
  // one and a half of them (backward pass of 16384 tokens with 32 heads and 1 of 128: 218 us where they are left out, 146 so).
  if (bwd && weights) {
    const long long queries_take = 2 * a.side[0].heads + 3, keys_take = 2 * a.side[1].heads + 3;
    long long keys = kBwdBlocks * keys_take / (queries_take + keys_take);
    keys = keys < 1 ? 1 : keys > kBwdBlocks - 1 ? kBwdBlocks - 1 : keys;
    blocks[0] = blocks[0] < kBwdBlocks - keys ? blocks[0] : kBwdBlocks - keys;
    blocks[1] = blocks[1] < keys ? blocks[1] : keys;
    for (int k = 0; k < 2; ++k) {                         // the same number of whole tiles to each
      const long long walks = ((a.tokens + a.tile[k] - 1) / a.tile[k] + blocks[k] - 1) / blocks[k] * blocks[k];
      a.tile[k] = static_cast<int>((a.tokens + walks - 1) / walks);
    }
  }
  if (blocks[0] + blocks[1] > 0x7fffffff) return MXK_ERR_DIMS;
  a.first_key = static_cast<int>(blocks[0]);
  const int all = static_cast<int>(blocks[0] + blocks[1]);
  const size_t smem = static_cast<size_t>(room);
  const bool neighbours = r->interleaved != 0;
  const auto go = [&](auto one) {
    using T = decltype(one);
    if (bwd) {
      launch_by_width<T, true>(a, width, neighbours, weights, all, smem, stream);
      if (weights)
        launch_kernel(rotate_weights_kernel<T>, dim3((r->dim + 31) / 32, 2), 1024, 0, stream, a.partial, a.first_key, all, r->dim, static_cast<T*>(dwq), static_cast<T*>(dwk));
    } else {
      launch_by_width<T, false>(a, width, neighbours, weights, all, smem, stream);
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
