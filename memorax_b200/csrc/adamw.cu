// One AdamW step over many tensors of one type in as few launches as their list fits, moments in 32 or in 8 bits:
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g g,
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// with g the gradient times a factor.  All of it is float32; only what is stored is rounded.
//
// The tensors' addresses travel in the kernel's parameters (40 bytes each of the 32 KB there are): gradients are elsewhere in
// every step, and a table in device memory would have to be copied there first.  Moments live in one buffer each, a tensor's
// at a multiple of kBlock elements, so that a warp's 256 elements are one block of 8-bit moments, all of one tensor.
//
// 8 bits: a block of m is held as e4m3 numbers c and a float scale s = max|m| / 448 with m = c s; of v the root is held (half
// the range in exponents), v = (c s)^2.  e4m3 rather than evenly spaced steps: the update is a quotient, so what counts is the
// relative error (at most 2^-4), over 2^17 of a block's largest; a root below that is held as the format's smallest number
// rather than as zero, which would leave eps alone under m.  The step itself uses the moments before they are rounded.  What is
// held must not turn on how a compiler pairs operations: a number next to a border of the format would be held 2^-4 away, and a
// step later be its block's largest.  So each operation behind a held number is rounded by itself; the additions are single ones,
// since two packed ones after each other were fused.
//
// A kernel of single operations has too many of them for its bytes when the moments are 8 bits wide: two floats go through
// each instruction, a block's largest comes from one reduction over the warp's bit patterns, and roots are an approximate
// reciprocal root times v with one correction by the residual v - r r, formed by a fused multiply-add (Markstein's form of
// Newton's step).  Reads of a warp's next elements are under way while it works on these: a turn ahead, in registers;
// where 8-bit moments meet 16-bit parameters and gradients, so that a turn is 48 bytes a thread, three turns ahead, copied to
// shared memory by the thread that reads them (5.7e8 bf16 parameters: 882 us against 1018 in registers; with float32 copies the
// ring of 1.2e8 parameters takes 334 us, registers 286).  Scales are read and written for all of a thread block's turns at once:
// one by one, between the other warps' reads of the same lines, they took as long as everything else (5.7e8 parameters 1538 us).
//
// Bytes bound it: 28 a parameter for bf16 with float32 copies and moments (1.5e7 parameters: 70 us, 5.9 TB/s), 10 for bf16 with
// 8-bit moments.  Those, 5.7e8 parameters, take 872 us (6.6 TB/s) with 80 % of the issue slots in use, while the clocks hold: in
// long runs the power limit lowers them, and it is 935 to 1040 us.  300 float32 tensors of up to 4001: 6.3 us, the host's 16.
#include <cuda_fp8.h>
#include <math.h>

#include <type_traits>

#include "elements.cuh"
#include "packed.cuh"

namespace mxk {
namespace {

constexpr int kBlock = 256;           // elements that share a scale: eight a lane
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTurn = kWarps * kBlock;   // elements of a thread block's turn
constexpr int kMostTurns = 16;
constexpr int kMost = 700;            // tensors of a launch: 700 * 44 bytes of parameters

struct Coefficients {
  float b1, b2, take_m, take_v, eps;   // take: (1 - b1) times the gradients' factor, (1 - b2) times its square
  float decay, step, root;   // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

template <int kCap>
struct Tensors {
  mxk_adamw_tensor t[kCap];
  int first[kCap];          // thread block at which each begins
  int count, turns;         // turns of a thread block
  void *m, *v;
  float *m_scale, *v_scale;
  const float* now;         // decay, step, root in device memory, or null
  Coefficients c;
};

// The coefficients of the step that a captured graph replays: counted and computed on the device.
__global__ void adamw_tick_kernel(long long* step, const float* lr, double b1, double b2, double weight_decay, float* now) {
  enter_kernel();
  const long long t = *step + 1;
  *step = t;
  const double rate = static_cast<double>(*lr);
  now[0] = static_cast<float>(1.0 - rate * weight_decay);
  now[1] = static_cast<float>(rate / (1.0 - pow(b1, static_cast<double>(t))));
  now[2] = static_cast<float>(1.0 / sqrt(1.0 - pow(b2, static_cast<double>(t))));
}

__device__ __forceinline__ float largest(const F2* x) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(x[i].lo()), fabsf(x[i].hi())));
  // of the warp: numbers that are not negative are in the order of their bits
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
}
__device__ __forceinline__ float reciprocal(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ void values_of(uint2 codes, F2* x) {
  const __nv_fp8x2_storage_t* c = reinterpret_cast<const __nv_fp8x2_storage_t*>(&codes);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(static_cast<__half2>(__nv_cvt_fp8x2_to_halfraw2(c[i], __NV_E4M3)));
    x[i] = F2(f.x, f.y);
  }
}
// The roots of v = -n, negative like n, so that no sign has to be turned; plain: v is positive, normal and finite throughout.
__device__ __forceinline__ void negative_roots(const F2* n, F2* root, bool plain) {
  if (plain) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(-n[i].lo()));
      asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(-n[i].hi()));
      const F2 y(a, b), r = mul(n[i], y), rest = fma(r, r, n[i]);
      root[i] = fma(rest, mul(y, F2(0.5f)), r);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) root[i] = F2(-sqrtf(-n[i].lo()), -sqrtf(-n[i].hi()));
  }
}
// A warp's 256 numbers -> codes (times `sign`) and scale.  kRoot: none of other sign, and none but zero held as zero: `least` is
// the square of this thread's smallest, plain: none is zero.
template <bool kRoot>
__device__ __forceinline__ uint2 hold(const F2* x, float sign, float* scale, float least = 0.f, bool plain = false) {
  float top = largest(x);
  if (top < 0x1p-100f) top = 0.f;    // (448 / top has to be finite)
  *scale = __fmul_rn(top, 1.f / 448.f);
  const float to = top > 0.f ? __fmul_rn(__frcp_rn(top), 448.f) : 0.f;
  F2 y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = mul(x[i], F2(sign * to));
  if (kRoot && top > 0.f && !(least * to * to >= 0x1p-18f)) {
    const auto floor = [&](float v) { return v < 0x1p-9f && (plain || v > 0.f) ? 0x1p-9f : v; };      // (NaN stays)
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = F2(floor(y[i].lo()), floor(y[i].hi()));
  }
  uint2 codes;
  __nv_fp8x2_storage_t* c = reinterpret_cast<__nv_fp8x2_storage_t*>(&codes);
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[i].lo(), y[i].hi()), __NV_SATFINITE, __NV_E4M3);
  return codes;
}

// Eight neighbours of a tensor, as they are in memory; those past its end (`left` elements from here) read as zero.
template <typename T>
struct Eight {
  static constexpr int kVec = 16 / sizeof(T);
  Vec<T, kVec> v[8 / kVec];
  __device__ __forceinline__ void load(const T* p, int left, bool wide) {
    if (wide && left >= 8) {
#pragma unroll
      for (int k = 0; k < 8 / kVec; ++k) v[k] = Vec<T, kVec>::load_stream(p + k * kVec);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const T zero = from_float<T>(0.f);
        reinterpret_cast<T*>(v)[k] = k < left ? p[k] : zero;
      }
    }
  }
  __device__ __forceinline__ void store(T* p, int left, bool wide) const {
    if (wide && left >= 8) {
#pragma unroll
      for (int k = 0; k < 8 / kVec; ++k) v[k].store_stream(p + k * kVec);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < left) p[k] = reinterpret_cast<const T*>(v)[k];
    }
  }
  __device__ __forceinline__ void values(F2* to) const {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8 / kVec; ++k) v[k].unpack(x + k * kVec);
#pragma unroll
    for (int k = 0; k < 4; ++k) to[k] = F2(x[2 * k], x[2 * k + 1]);
  }
  __device__ __forceinline__ void take(const F2* from) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[2 * k] = from[k].lo(), x[2 * k + 1] = from[k].hi();
#pragma unroll
    for (int k = 0; k < 8 / kVec; ++k) v[k] = Vec<T, kVec>::pack(x + k * kVec);
  }
};
// What a thread reads for eight elements, before anything is made of it: in registers,
template <typename W, typename G>
struct Ahead {
  Eight<W> x;
  Eight<G> g;
  Eight<float> m, v;
  uint2 cm, cv;                     // (which moments are used is known where they are: the others take no registers)
};
// or on its way through shared memory: planes of 16 (moments: 8) bytes a thread, so that neighbours do not meet in a bank.
template <int kBytes>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const uint32_t smem = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem), "l"(from) : "memory");
}
template <typename W, typename G>
struct Ring {
  static constexpr int kX = 8 * sizeof(W) / 16, kG = 8 * sizeof(G) / 16;      // planes
  static constexpr int kStage = kThreads * 16 * (kX + kG + 1);
  static constexpr int kStages = 4;
  static constexpr int kSmem = kStages * kStage;
  uint8_t* base;
  __device__ __forceinline__ uint8_t* plane(int stage, int i) const { return base + stage * kStage + (i * kThreads + threadIdx.x) * 16; }
  __device__ __forceinline__ uint8_t* moment(int stage, int i) const { return base + stage * kStage + (kX + kG) * kThreads * 16 + (i * kThreads + threadIdx.x) * 8; }
  __device__ __forceinline__ void fetch(int stage, const W* x, const G* g, const uint8_t* m, const uint8_t* v) const {
#pragma unroll
    for (int i = 0; i < kX; ++i) copy_async<16>(plane(stage, i), x + i * (16 / sizeof(W)));
#pragma unroll
    for (int i = 0; i < kG; ++i) copy_async<16>(plane(stage, kX + i), g + i * (16 / sizeof(G)));
    copy_async<8>(moment(stage, 0), m);
    copy_async<8>(moment(stage, 1), v);
  }
  template <typename T>
  __device__ __forceinline__ void take(int stage, int first, Eight<T>& to) const {
#pragma unroll
    for (int i = 0; i < static_cast<int>(8 * sizeof(T) / 16); ++i) to.v[i] = Vec<T, Eight<T>::kVec>::load(reinterpret_cast<const T*>(plane(stage, first + i)));
  }
};

template <typename P, typename G, bool k8, bool kMaster>
constexpr bool kRings = k8 && !kMaster && sizeof(P) == 2 && sizeof(G) == 2;

template <typename P, typename G, bool k8, bool kMaster, int kCap>
__global__ void __launch_bounds__(kThreads, kRings<P, G, k8, kMaster> ? 4 : k8 ? 3 : 2)
adamw_kernel(const __grid_constant__ Tensors<kCap> a) {
  enter_kernel();
  int lo = 0, hi = a.count - 1;       // the last tensor that begins at or before this block
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.first[mid] <= static_cast<int>(blockIdx.x)) lo = mid; else hi = mid - 1;
  }
  const mxk_adamw_tensor& t = a.t[lo];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long start = static_cast<long long>(blockIdx.x - a.first[lo]) * a.turns * kTurn;      // of the thread block
  const long long rest = t.n - start;
  const int many = static_cast<int>(min(rest, static_cast<long long>(a.turns) * kTurn));             // its elements
  const int turns = (many - warp * kBlock + kTurn - 1) / kTurn;                                      // a warp's, with any of them
  int left = many - threadIdx.x * 8;                                                                 // from this thread's on
  P* p = static_cast<P*>(t.p) + start + threadIdx.x * 8;
  const G* g = static_cast<const G*>(t.g) + start + threadIdx.x * 8;
  float* master = kMaster ? t.master + start + threadIdx.x * 8 : nullptr;
  const bool wide = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(master)) & 15) == 0;
  const long long at = t.state + start;
  uint8_t *pm = static_cast<uint8_t*>(a.m) + (at + threadIdx.x * 8) * (k8 ? 1 : 4), *pv = static_cast<uint8_t*>(a.v) + (at + threadIdx.x * 8) * (k8 ? 1 : 4);
  const float decay = a.now ? a.now[0] : a.c.decay, step = a.now ? a.now[1] : a.c.step, rs = a.now ? a.now[2] : a.c.root;
  __shared__ float scale[2][kMostTurns * kWarps];
  const int scales = (many + kBlock - 1) / kBlock;
  if (k8) {
    for (int i = threadIdx.x; i < scales; i += kThreads) {
      scale[0][i] = a.m_scale[at / kBlock + i];
      scale[1][i] = a.v_scale[at / kBlock + i];
    }
    __syncthreads();
  }
  using W = std::conditional_t<kMaster, float, P>;                    // what takes the update
  const W* own = kMaster ? reinterpret_cast<const W*>(master) : reinterpret_cast<const W*>(p);
  Ahead<W, G> next;
  const auto read = [&](int ahead) {
    next.x.load(own + ahead, left - ahead, wide);
    next.g.load(g + ahead, left - ahead, wide);
    if (k8) {
      next.cm = __ldcs(reinterpret_cast<const uint2*>(pm + ahead));
      next.cv = __ldcs(reinterpret_cast<const uint2*>(pv + ahead));
    } else {
      next.m.load(reinterpret_cast<const float*>(pm) + ahead, 8, true);
      next.v.load(reinterpret_cast<const float*>(pv) + ahead, 8, true);
    }
  };
  constexpr bool kRing = kRings<P, G, k8, kMaster>;
  constexpr int kStages = Ring<W, G>::kStages;
  extern __shared__ uint4 adamw_smem[];
  const Ring<W, G> ring{reinterpret_cast<uint8_t*>(adamw_smem)};
  const auto copy = [&](int turn, int ahead) {                       // (elements that are no whole vectors: when they are needed)
    if (turn < turns && wide && left - ahead >= 8) ring.fetch(turn % kStages, own + ahead, g + ahead, pm + ahead, pv + ahead);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (kRing) {
    for (int turn = 0; turn < kStages - 1; ++turn) copy(turn, turn * kTurn);
  } else if (turns > 0) {
    read(0);
  }
  for (int turn = 0; turn < turns; ++turn) {
    Ahead<W, G> in;
    if (kRing) {
      copy(turn + kStages - 1, (kStages - 1) * kTurn);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      if (wide && left >= 8) {
        ring.take(turn % kStages, 0, in.x);
        ring.take(turn % kStages, Ring<W, G>::kX, in.g);
        in.cm = *reinterpret_cast<const uint2*>(ring.moment(turn % kStages, 0));
        in.cv = *reinterpret_cast<const uint2*>(ring.moment(turn % kStages, 1));
      } else {
        in.x.load(own, left, wide);
        in.g.load(g, left, wide);
        in.cm = *reinterpret_cast<const uint2*>(pm);
        in.cv = *reinterpret_cast<const uint2*>(pv);
      }
    } else {
      in = next;
      if (turn + 1 < turns) read(kTurn);
    }
    F2 x[4], gr[4], m[4], v[4], n[4], root[4];                        // n: -v
    in.x.values(x);
    in.g.values(gr);
    if (k8) {
      const F2 sm(scale[0][turn * kWarps + warp]), sv(scale[1][turn * kWarps + warp]);
      values_of(in.cm, m);
      values_of(in.cv, v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        m[k] = mul(m[k], sm);
        v[k] = mul(v[k], sv);
        v[k] = mul(v[k], v[k]);
      }
    } else {
      in.m.values(m);
      in.v.values(v);
    }
    float least = -0x1p127f, most = 0.f;                              // of n: nearest to zero, and farthest
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const F2 old_m = mul(m[k], F2(a.c.b1)), new_m = mul(gr[k], F2(a.c.take_m));
      m[k] = F2(__fadd_rn(old_m.lo(), new_m.lo()), __fadd_rn(old_m.hi(), new_m.hi()));
      if (k8) {
        const F2 old_n = mul(v[k], F2(-a.c.b2)), new_n = mul(mul(gr[k], F2(-a.c.take_v)), gr[k]);
        n[k] = F2(__fadd_rn(old_n.lo(), new_n.lo()), __fadd_rn(old_n.hi(), new_n.hi()));
      } else {
        v[k] = fma(v[k], F2(a.c.b2), mul(mul(gr[k], F2(a.c.take_v)), gr[k]));
        n[k] = mul(v[k], F2(-1.f));
      }
      least = fmaxf(least, fmaxf(n[k].lo(), n[k].hi()));
      most = fminf(most, fminf(n[k].lo(), n[k].hi()));
    }
    const bool plain = least <= -0x1p-126f && most >= -0x1.fffffep127f;
    negative_roots(n, root, plain);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const F2 under = fma(root[k], F2(-rs), F2(a.c.eps));
      const F2 update = mul(m[k], F2(reciprocal(under.lo()), reciprocal(under.hi())));
      x[k] = fma(update, F2(-step), mul(x[k], F2(decay)));
    }
    if (kMaster) {
      Eight<float> w;
      w.take(x);
      w.store(master, left, wide);
    }
    Eight<P> y;
    y.take(x);
    y.store(p, left, wide);
    if (k8) {
      float sm, sv;
      const uint2 cm = hold<false>(m, 1.f, &sm), cv = hold<true>(root, -1.f, &sv, -least, plain);
      __stcs(reinterpret_cast<uint2*>(pm), cm);
      __stcs(reinterpret_cast<uint2*>(pv), cv);
      __syncwarp();
      if (lane == 0) scale[0][turn * kWarps + warp] = sm, scale[1][turn * kWarps + warp] = sv;
    } else {
      Eight<float> w;
      w.take(m);
      w.store(reinterpret_cast<float*>(pm), 8, true);
      w.take(v);
      w.store(reinterpret_cast<float*>(pv), 8, true);
    }
    p += kTurn; g += kTurn; own += kTurn; master += kMaster ? kTurn : 0;
    pm += k8 ? kTurn : 4 * kTurn; pv += k8 ? kTurn : 4 * kTurn;
    left -= kTurn;
  }
  if (k8) {
    __syncthreads();
    for (int i = threadIdx.x; i < scales; i += kThreads) {
      a.m_scale[at / kBlock + i] = scale[0][i];
      a.v_scale[at / kBlock + i] = scale[1][i];
    }
  }
}

template <typename P, typename G, bool k8, int kCap>
int launch(const mxk_adamw_tensor* t, int count, const mxk_adamw_state& s, const Coefficients& c, cudaStream_t stream) {
  Tensors<kCap> a;
  long long all = 0, blocks = 0;
  for (int i = 0; i < count; ++i) all += (t[i].n + kTurn - 1) / kTurn;
  // about eight blocks an SM, of as many turns as that takes: a block's way to its tensor is paid once
  a.turns = static_cast<int>(all / (8 * kNumSMs) < 1 ? 1 : all / (8 * kNumSMs) < kMostTurns ? all / (8 * kNumSMs) : kMostTurns);
  for (int i = 0; i < count; ++i) {
    a.t[i] = t[i];
    a.first[i] = static_cast<int>(blocks);
    blocks += t[i].n <= kTurn * a.turns ? 1 : (t[i].n + kTurn * a.turns - 1) / (kTurn * a.turns);
    if (blocks > 0x7fffffff) return MXK_ERR_DIMS;
  }
  a.count = count;
  a.m = s.m; a.v = s.v; a.m_scale = s.m_scale; a.v_scale = s.v_scale; a.now = s.now;
  a.c = c;
  constexpr bool kHalf = sizeof(P) == 2;
  if (kHalf && t[0].master) {
    launch_kernel(adamw_kernel<P, G, k8, kHalf, kCap>, static_cast<unsigned>(blocks), kThreads, 0, stream, a);
    return MXK_OK;
  }
  constexpr int kSmem = kRings<P, G, k8, false> ? Ring<P, G>::kSmem : 0;
  if constexpr (kSmem > 0) {
    if (const int status = allow_smem<adamw_kernel<P, G, k8, false, kCap>, kSmem>()) return status;
  }
  launch_kernel(adamw_kernel<P, G, k8, false, kCap>, static_cast<unsigned>(blocks), kThreads, kSmem, stream, a);
  return MXK_OK;
}
template <typename P, typename G>
int launch_all(const mxk_adamw_tensor* t, int count, const mxk_adamw_state& s, const Coefficients& c, cudaStream_t stream) {
  for (int i = 0; i < count; i += kMost) {
    const int some = count - i < kMost ? count - i : kMost;
    int status;
    if (some <= 48)    // (the parameters are copied with every launch: 31 KB cost the host 3 us)
      status = s.bits == 8 ? launch<P, G, true, 48>(t + i, some, s, c, stream) : launch<P, G, false, 48>(t + i, some, s, c, stream);
    else if (some <= kMost / 2)
      status = s.bits == 8 ? launch<P, G, true, kMost / 2>(t + i, some, s, c, stream) : launch<P, G, false, kMost / 2>(t + i, some, s, c, stream);
    else
      status = s.bits == 8 ? launch<P, G, true, kMost>(t + i, some, s, c, stream) : launch<P, G, false, kMost>(t + i, some, s, c, stream);
    if (status) return status;
  }
  return launch_status();
}

}  // namespace
}  // namespace mxk

extern "C" {

int mxk_adamw_tick(long long* step, const float* lr, double beta1, double beta2, double weight_decay, float* now, mxk_stream_t stream) {
  if (!step || !lr || !now) return MXK_ERR_NULL;
  mxk::launch_kernel(mxk::adamw_tick_kernel, 1, 1, 0, static_cast<cudaStream_t>(stream), step, lr, beta1, beta2, weight_decay, now);
  return mxk::launch_status();
}

int mxk_adamw(const mxk_adamw_tensor* tensors, int count, int param_type, int grad_type, const mxk_adamw_state* state, double lr,
              double beta1, double beta2, double eps, double weight_decay, double grad_scale, long long step, mxk_stream_t stream) {
  using namespace mxk;
  if (!tensors || !state || !state->m || !state->v) return MXK_ERR_NULL;
  if (count <= 0 || (step <= 0 && !state->now)) return MXK_ERR_DIMS;
  if (!known_type(param_type) || (grad_type != param_type && grad_type != MXK_F32) || (state->bits != 8 && state->bits != 32)) return MXK_ERR_UNSUPPORTED;
  if (state->bits == 8 && (!state->m_scale || !state->v_scale)) return MXK_ERR_NULL;
  if (!aligned16(state->m) || !aligned16(state->v)) return MXK_ERR_ALIGN;
  const uintptr_t param_low = type_bytes(param_type) - 1, grad_low = type_bytes(grad_type) - 1;
  for (int i = 0; i < count; ++i) {
    const mxk_adamw_tensor& t = tensors[i];
    if (!t.p || !t.g) return MXK_ERR_NULL;
    if (t.n <= 0 || t.state < 0) return MXK_ERR_DIMS;
    if (!t.master != !tensors[0].master || (t.master && param_type == MXK_F32)) return MXK_ERR_UNSUPPORTED;
    if ((t.state & (kBlock - 1)) || (address(t.p) & param_low) || (address(t.g) & grad_low) || (address(t.master) & 3)) return MXK_ERR_ALIGN;
  }
  Coefficients c;
  c.b1 = static_cast<float>(beta1); c.take_m = static_cast<float>((1.0 - beta1) * grad_scale);
  c.b2 = static_cast<float>(beta2); c.take_v = static_cast<float>((1.0 - beta2) * grad_scale * grad_scale);
  c.eps = static_cast<float>(eps);
  c.decay = c.step = c.root = 0.f;
  if (!state->now) {
    c.decay = static_cast<float>(1.0 - lr * weight_decay);
    c.step = static_cast<float>(lr / (1.0 - pow(beta1, static_cast<double>(step))));
    c.root = static_cast<float>(1.0 / sqrt(1.0 - pow(beta2, static_cast<double>(step))));
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = grad_type == MXK_F32;
  switch (param_type) {
    case MXK_F32: return launch_all<float, float>(tensors, count, *state, c, s);
    case MXK_BF16: return wide ? launch_all<__nv_bfloat16, float>(tensors, count, *state, c, s) : launch_all<__nv_bfloat16, __nv_bfloat16>(tensors, count, *state, c, s);
    default: return wide ? launch_all<__half, float>(tensors, count, *state, c, s) : launch_all<__half, __half>(tensors, count, *state, c, s);
  }
}

}  // extern "C"
