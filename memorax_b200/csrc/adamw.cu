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
// rather than as zero, which would leave eps alone under m.  The step itself uses the moments before they are rounded.  Each
// operation behind a held number is rounded by itself (__fmul_rn ...: no contraction), so that the number held does not turn on
// how the compiler pairs them.
//
// Bytes bound it: 10 a parameter for bf16 with 8-bit moments, 30 for bf16 with float32 copies and moments.
#include <cuda_fp8.h>
#include <math.h>

#include "elements.cuh"

namespace mxk {
namespace {

constexpr int kBlock = 256;           // elements that share a scale: eight a lane
constexpr int kThreads = 256;
constexpr int kTurn = kThreads * 8;   // elements of a block's turn
constexpr int kTurns = 4;             // turns of a thread block
constexpr int kMost = 700;            // tensors of a launch: 700 * 44 bytes of parameters

struct Coefficients {
  float b1, one_b1, b2, one_b2, eps, gscale;
  float decay, step, root;   // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

template <int kCap>
struct Tensors {
  mxk_adamw_tensor t[kCap];
  int first[kCap];          // thread block at which each begins
  int count;
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

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int off = 16; off; off >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
  return x;
}

__device__ __forceinline__ void values_of(uint2 codes, float scale, float* x) {
  const __nv_fp8x2_storage_t* c = reinterpret_cast<const __nv_fp8x2_storage_t*>(&codes);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(static_cast<__half2>(__nv_cvt_fp8x2_to_halfraw2(c[i], __NV_E4M3)));
    x[2 * i] = __fmul_rn(f.x, scale);
    x[2 * i + 1] = __fmul_rn(f.y, scale);
  }
}
// A warp's 256 numbers -> codes and scale; kRoot: none negative, and none but zero held as zero.
template <bool kRoot>
__device__ __forceinline__ uint2 hold(const float* x, float* scale) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
  top = warp_max(top);
  if (top < 0x1p-100f) top = 0.f;    // (448 / top has to be finite)
  *scale = __fmul_rn(top, 1.f / 448.f);
  const float to = top > 0.f ? __fmul_rn(__frcp_rn(top), 448.f) : 0.f;
  uint2 codes;
  __nv_fp8x2_storage_t* c = reinterpret_cast<__nv_fp8x2_storage_t*>(&codes);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f = make_float2(__fmul_rn(x[2 * i], to), __fmul_rn(x[2 * i + 1], to));
    if (kRoot && top > 0.f) {
      if (x[2 * i] > 0.f) f.x = fmaxf(f.x, 0x1p-9f);
      if (x[2 * i + 1] > 0.f) f.y = fmaxf(f.y, 0x1p-9f);
    }
    c[i] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
  }
  return codes;
}

// Eight neighbours from `i` on of a tensor of n; those past its end read as zero.
template <typename T>
__device__ __forceinline__ void load8(const T* p, long long i, long long n, bool wide, float* x) {
  if (wide && i + 8 <= n) {
    constexpr int kVec = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < 8; k += kVec) Vec<T, kVec>::load_stream(p + i + k).unpack(x + k);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = i + k < n ? as_float(p[i + k]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, long long i, long long n, bool wide, const float* x) {
  if (wide && i + 8 <= n) {
    constexpr int kVec = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < 8; k += kVec) Vec<T, kVec>::pack(x + k).store_stream(p + i + k);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) p[i + k] = from_float<T>(x[k]);
  }
}

template <typename P, typename G, bool k8, int kCap>
__global__ void __launch_bounds__(kThreads)
adamw_kernel(const __grid_constant__ Tensors<kCap> a) {
  enter_kernel();
  int lo = 0, hi = a.count - 1;       // the last tensor that begins at or before this block
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.first[mid] <= static_cast<int>(blockIdx.x)) lo = mid; else hi = mid - 1;
  }
  const mxk_adamw_tensor& t = a.t[lo];
  P* const p = static_cast<P*>(t.p);
  const G* const g = static_cast<const G*>(t.g);
  float* const master = t.master;
  const long long n = t.n;
  const bool wide = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(master)) & 15) == 0;
  const float decay = a.now ? a.now[0] : a.c.decay, step = a.now ? a.now[1] : a.c.step, rs = a.now ? a.now[2] : a.c.root;
  long long i = static_cast<long long>(blockIdx.x - a.first[lo]) * (kTurn * kTurns) + threadIdx.x * 8;
  for (int turn = 0; turn < kTurns; ++turn, i += kTurn) {
    const long long block = i / kBlock * kBlock;     // a warp's 256 elements
    if (block >= n) return;
    const long long at = t.state + i;
    float x[8], gr[8], m[8], v[8];
    if (master) load8(master, i, n, wide, x); else load8(p, i, n, wide, x);
    load8(g, i, n, wide, gr);
    if (k8) {
      const uint2 cm = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + at));
      const uint2 cv = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + at));
      const float sm = a.m_scale[at / kBlock], sv = a.v_scale[at / kBlock];
      values_of(cm, sm, m);
      values_of(cv, sv, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = __fmul_rn(v[k], v[k]);
    } else {
      const float* pm = static_cast<const float*>(a.m) + at;
      const float* pv = static_cast<const float*>(a.v) + at;
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        Vec<float, 4>::load_stream(pm + k).unpack(m + k);
        Vec<float, 4>::load_stream(pv + k).unpack(v + k);
      }
    }
    float root[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float e = __fmul_rn(gr[k], a.c.gscale);
      m[k] = __fadd_rn(__fmul_rn(m[k], a.c.b1), __fmul_rn(e, a.c.one_b1));
      v[k] = __fadd_rn(__fmul_rn(v[k], a.c.b2), __fmul_rn(__fmul_rn(e, a.c.one_b2), e));
      root[k] = __fsqrt_rn(v[k]);
      x[k] = __fsub_rn(__fmul_rn(x[k], decay), __fmul_rn(__fdividef(m[k], __fadd_rn(__fmul_rn(root[k], rs), a.c.eps)), step));
    }
    if (master) store8(master, i, n, wide, x);
    store8(p, i, n, wide, x);
    if (k8) {
      float sm, sv;
      const uint2 cm = hold<false>(m, &sm), cv = hold<true>(root, &sv);
      __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.m) + at), cm);
      __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + at), cv);
      if (threadIdx.x % 32 == 0) {
        a.m_scale[at / kBlock] = sm;
        a.v_scale[at / kBlock] = sv;
      }
    } else {
      float* pm = static_cast<float*>(a.m) + at;
      float* pv = static_cast<float*>(a.v) + at;
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        Vec<float, 4>::pack(m + k).store_stream(pm + k);
        Vec<float, 4>::pack(v + k).store_stream(pv + k);
      }
    }
  }
}

template <typename P, typename G, bool k8, int kCap>
int launch(const mxk_adamw_tensor* t, int count, const mxk_adamw_state& s, const Coefficients& c, cudaStream_t stream) {
  Tensors<kCap> a;
  long long blocks = 0;
  for (int i = 0; i < count; ++i) {
    a.t[i] = t[i];
    a.first[i] = static_cast<int>(blocks);
    blocks += (t[i].n + kTurn * kTurns - 1) / (kTurn * kTurns);
    if (blocks > 0x7fffffff) return MXK_ERR_DIMS;
  }
  a.count = count;
  a.m = s.m; a.v = s.v; a.m_scale = s.m_scale; a.v_scale = s.v_scale; a.now = s.now;
  a.c = c;
  launch_kernel(adamw_kernel<P, G, k8, kCap>, static_cast<unsigned>(blocks), kThreads, 0, stream, a);
  return MXK_OK;
}
template <typename P, typename G>
int launch_all(const mxk_adamw_tensor* t, int count, const mxk_adamw_state& s, const Coefficients& c, cudaStream_t stream) {
  for (int i = 0; i < count; i += kMost) {
    const int some = count - i < kMost ? count - i : kMost;
    int status;
    if (some <= 48)    // (the parameters are copied with every launch)
      status = s.bits == 8 ? launch<P, G, true, 48>(t + i, some, s, c, stream) : launch<P, G, false, 48>(t + i, some, s, c, stream);
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
  for (int i = 0; i < count; ++i) {
    const mxk_adamw_tensor& t = tensors[i];
    if (!t.p || !t.g) return MXK_ERR_NULL;
    if (t.n <= 0 || t.state < 0) return MXK_ERR_DIMS;
    if (t.state % kBlock || address(t.p) % type_bytes(param_type) || address(t.g) % type_bytes(grad_type) || address(t.master) % 4) return MXK_ERR_ALIGN;
  }
  Coefficients c;
  c.b1 = static_cast<float>(beta1); c.one_b1 = static_cast<float>(1.0 - beta1);
  c.b2 = static_cast<float>(beta2); c.one_b2 = static_cast<float>(1.0 - beta2);
  c.eps = static_cast<float>(eps); c.gscale = static_cast<float>(grad_scale);
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
