// AdamW over many tensors in one launch, the moments held in 32 or in 8 bits,
// and the global gradient norm that clips a step or calls it off.
//
// With g the gradient times the clip coefficient, t the tensor's step count
// and every value taken in f32:
//   m <- b1 m + (1 - b1) g             v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - lr / (1 - b1^t)  m / (sqrt(v / (1 - b2^t)) + eps)
//
// Layout.  Every tensor's state starts on a multiple of 256 slots of one flat
// array, so a block of 256 slots belongs to one tensor and one warp does one
// block: 8 elements a lane in two groups of four, each array read and written
// with whole 128-byte lines.  A table tells each block's tensor, its place in it
// and how much of it is used; a warp reads the record of its next block while it
// works on this one.  The parameters' and gradients' pointers travel in the
// launch itself, so gradients that move from step to step cost no copy.
//
// 8-bit moments.  A block holds 256 e4m3 codes and one f32 scale = max / 448.
// They are rounded stochastically, by a hash of (slot, step): with b2 = 0.999
// a step moves v by 0.1% or less, far under half a step of a 3-bit mantissa
// (3 to 6%), so rounding to nearest would hold v where it is for good, while
// this keeps its expectation.  The update itself uses the unrounded moments.
// A positive v is never held as 0 beside an m that is not: the element would
// next move by m / eps.  In a block with a v above 2^-100 it is held as the
// smallest code at least; in one without, v and m are zeros, and a step is then
// at most that from moments of zero, 3.2 lr (gradients below 3e-14 of which eps,
// 1e-8 as a rule, leaves nothing to see).
//
// Bound: with 32-bit moments HBM: an f32 parameter costs 28 bytes (p, m, v read
// and written, g read); 10.2 M take 51 us (5.6 TB/s; two sets of parameters in
// turn, so nothing of one is left in L2), 40 M 182 us (6.1).  With 8 bits it costs
// 16 (a bf16 one 10), but some 83 instructions, of which the hash and the rounding
// are half, and these bound it: 10.2 M f32 parameters 39 us, 160 M bf16 ones 518 us
// (3.1 TB/s); 3% of it is the root that is right for every v.  The norm adds 11 us
// at 10.2 M.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include <cuda_fp8.h>

#include "ow_common.cuh"
#include "ow_internal.h"

namespace ow {
namespace {

constexpr int BLK = OW_ADAMW_BLOCK;  // slots a warp works on, and that share a scale
constexpr int WARPS = 8;
constexpr float TINY = 7.888609052210118e-31f;  // 2^-100: a block whose values are all below it is held as zeros

template <int MAXT>
struct Ptrs {
  void* p[MAXT];
  const void* g[MAXT];
};

struct Tables {
  const int4* block;       // [blocks]: tensor, block of the tensor, elements in use
  int t0;                  // first tensor of this launch
  int64_t blk0, nblk;      // its blocks
};

// Scalars the norm leaves for the update.
struct Ctl {
  float coef;   // clip coefficient
  float found;  // 1: a gradient was not finite
  unsigned ticket_norm, ticket_step;
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, int i, int n, bool vec, float (&o)[4]) {
  if (vec && i + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p + i);
      const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = Elem<T>::to_f(h[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = i + k < n ? Elem<T>::to_f(p[i + k]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, int i, int n, bool vec, const float (&v)[4]) {
  if (vec && i + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p + i) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      uint2 o;
      T* h = reinterpret_cast<T*>(&o);
#pragma unroll
      for (int k = 0; k < 4; ++k) h[k] = Elem<T>::from(v[k]);
      *reinterpret_cast<uint2*>(p + i) = o;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[i + k] = Elem<T>::from(v[k]);
  }
}

template <typename T>
__device__ __forceinline__ bool aligned4(const void* p) {
  return ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0;
}

// sqrt(v) and m / d, each within two steps of f32.  The root is right for every
// v: below 2^-126 too (gradients of 1e-19 and less), which counts with a small eps,
// and inf for a v that overflowed, so that m / inf takes 0 off the parameter.
__device__ __forceinline__ float fast_sqrt(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float fast_div(float m, float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return m * r;
}

// Two 16-bit numbers from (slot, step), as the 20 bits below an e4m3 mantissa
// see them: 16 random bits and half of the last one.  ``seed``: of the block's
// first slot; the slots of a block differ in the low 8 bits only.  The mixing steps
// are a published 32-bit integer mixer's, found by search (C. Wellons, "Prospecting
// for hash functions", 2018); the seed's multipliers are 2^32 over the golden ratio
// (Knuth, TAOCP 6.4) and the two of A. Appleby's 32-bit finalizer (2011).
__device__ __forceinline__ uint32_t random_seed(int64_t slot, uint32_t step) {
  return (uint32_t)slot * 0x9E3779B1u + (uint32_t)((uint64_t)slot >> 32) * 0x85EBCA6Bu + step * 0xC2B2AE35u;
}
__device__ __forceinline__ void random20(uint32_t seed, uint32_t e, uint32_t& r1, uint32_t& r2) {
  uint32_t h = seed + e * 0x9E3779B1u;
  h = (h ^ (h >> 16)) * 0x7FEB352Du;
  h = (h ^ (h >> 15)) * 0x846CA68Bu;
  h ^= h >> 16;
  r1 = (h << 4 & 0xFFFF0u) | 8u;
  r2 = (h >> 12 & 0xFFFF0u) | 8u;
}

// |x| inv, at most 448, as an e4m3 magnitude.  Times 2^-120 the exponents of
// e4m3 (subnormals included) are those of f32, so the code is the top bits and
// adding a random number below them rounds.
__device__ __forceinline__ uint32_t hold8(float x, float inv, uint32_t r20) {
  const float y = __fmul_rn(fabsf(x), inv);
  return min((__float_as_uint(y * 7.52316384526264e-37f) + r20) >> 20, 126u);  // 2^-120
}

constexpr uint32_t INF = 0x7F800000u;

// A block whose v are not all finite, before it is held; a format with one scale
// has no room for them, and they are kept from the block's other elements.  An
// element that a gradient (or its own state) has made NaN or inf is marked by
// v = NaN and held so.  One with a finite m whose v overflowed took a step of 0;
// it goes on from m = 0 and the largest finite v of its block.  ``mmax`` and
// ``vtop`` (as bits): the largest of the finite ones, of the whole block.
__device__ __forceinline__ void mend_odd(float (&m)[2][4], float (&v)[2][4], float& mmax, uint32_t& vtop) {
  float mm = 0.f;
  uint32_t vt = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool lost = (__float_as_uint(m[j][k]) & INF) == INF || v[j][k] != v[j][k];
      if (lost) v[j][k] = __uint_as_float(0x7FFFFFFFu);
      else if (__float_as_uint(v[j][k]) == INF) m[j][k] = 0.f;
      else {
        mm = fmaxf(mm, fabsf(m[j][k]));
        vt = max(vt, __float_as_uint(v[j][k]));
      }
    }
  mmax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mm)));
  vtop = __reduce_max_sync(0xffffffffu, vt);
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (__float_as_uint(v[j][k]) == INF) v[j][k] = __uint_as_float(vtop);
}

__device__ __forceinline__ void unhold4(uint32_t codes, float scale, float (&o)[4]) {
  const __half2 a(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xFFFFu), __NV_E4M3));
  const __half2 b(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), __NV_E4M3));
  const float2 fa = __half22float2(a), fb = __half22float2(b);
  o[0] = fa.x * scale; o[1] = fa.y * scale; o[2] = fb.x * scale; o[3] = fb.y * scale;
}

struct StepArgs {
  Tables tab;
  void* m;             // flat: f32, or e4m3 codes
  void* v;
  float* ms;           // [blocks] scales of the 8-bit states
  float* vs;
  float* steps;        // [tensors] steps done
  const float* lr_ptr; // device learning rate, or NULL
  const float* found_in;
  Ctl* ctl;            // also the clip coefficient when ``use_ctl``
  int use_ctl;
  float lr, b1c, b2c, b1, b2, ln_b1, ln_b2, eps, wd;
  int ntensors;
};

// Where a block's values are and, with 32 bits, the values as they come from
// memory.  With 8 bits they come by asynchronous copies to the thread's own
// slots in shared memory: every thread reads back what it asked for itself.
template <typename T, bool EIGHT>
struct Fetched {
  int used;     // elements of the block in use
  const T* g;   // the block's first gradient; NULL: nothing to do
  T* p;
  bool vec;
  float t;      // the tensor's steps, this one included
  float ms, vs; // 8 bits
  using W = std::conditional_t<sizeof(T) == 4, float4, uint2>;
  W pw[EIGHT ? 1 : 2], gw[EIGHT ? 1 : 2];
  float4 mw[EIGHT ? 1 : 2], vw[EIGHT ? 1 : 2];
};

template <typename T>
struct Slots {
  using W = typename Fetched<T, true>::W;
  W p[2][WARPS * 32], g[2][WARPS * 32];
  uint32_t m[2][WARPS * 32], v[2][WARPS * 32];
};

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(BYTES)
               : "memory");
}

template <typename T, bool EIGHT, int MAXT>
__device__ __forceinline__ void fetch(Fetched<T, EIGHT>& f, Slots<T>* to, const Ptrs<MAXT>& ptr, const StepArgs& a, int64_t blk,
                                      int4 rec) {
  const int lane = threadIdx.x & 31;
  f.used = rec.z;
  const T* g = reinterpret_cast<const T*>(ptr.g[rec.x - a.tab.t0]);
  f.g = g;
  if (!g) return;
  f.g = g + (int64_t)rec.y * BLK;
  f.p = reinterpret_cast<T*>(ptr.p[rec.x - a.tab.t0]) + (int64_t)rec.y * BLK;
  f.vec = aligned4<T>(f.p) && aligned4<T>(f.g) && rec.z == BLK;
  f.t = a.steps[rec.x] + 1.f;
  const int64_t slot = blk * BLK;
  using W = typename Fetched<T, EIGHT>::W;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int e = j * 128 + lane * 4;
    if constexpr (EIGHT) {
      if (f.vec) {
        copy_async<sizeof(W)>(&to->p[j][threadIdx.x], f.p + e);
        copy_async<sizeof(W)>(&to->g[j][threadIdx.x], f.g + e);
      }
      copy_async<4>(&to->m[j][threadIdx.x], (const unsigned char*)a.m + slot + e);
      copy_async<4>(&to->v[j][threadIdx.x], (const unsigned char*)a.v + slot + e);
    } else {
      if (f.vec) {
        f.pw[j] = *reinterpret_cast<const W*>(f.p + e);
        f.gw[j] = *reinterpret_cast<const W*>(f.g + e);
      }
      f.mw[j] = *reinterpret_cast<const float4*>((const float*)a.m + slot + e);
      f.vw[j] = *reinterpret_cast<const float4*>((const float*)a.v + slot + e);
    }
  }
  if constexpr (EIGHT) {
    f.ms = a.ms[blk];
    f.vs = a.vs[blk];
  }
}

template <typename T, typename W>
__device__ __forceinline__ void widen(const W& w, float (&o)[4]) {
  if constexpr (sizeof(T) == 4) {
    o[0] = w.x; o[1] = w.y; o[2] = w.z; o[3] = w.w;
  } else {
    const T* h = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = Elem<T>::to_f(h[k]);
  }
}

// 8-bit moments take some 83 instructions and 10 to 16 bytes an element, so a
// warp asks for its next block before it works on this one, by copies that hold
// no registers; with 32 bits and 28 bytes the loads of the warps at hand fill
// the memory's pipe already.
template <typename T, bool EIGHT, int MAXT>
__global__ void __launch_bounds__(WARPS * 32, 3) adamw_kernel(const __grid_constant__ Ptrs<MAXT> ptr, const StepArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // A step that was called off leaves everything as it is.
  if (a.found_in && *a.found_in != 0.f) return;
  float coef = 1.f;
  if (a.use_ctl) {
    if (a.ctl->found != 0.f) return;
    coef = a.ctl->coef;
  }
  const float lr = a.lr_ptr ? *a.lr_ptr : a.lr;
  const float decay = 1.f - lr * a.wd;
  float t_have = -1.f, alpha = 0.f, rc2 = 0.f;
  const int64_t stride = (int64_t)gridDim.x * WARPS, nblk = a.tab.nblk;
  const int4* records = a.tab.block + a.tab.blk0;
  int64_t b = (int64_t)blockIdx.x * WARPS + warp;
  Fetched<T, EIGHT> now, next;
  __shared__ Slots<T> slots[EIGHT ? 2 : 1];
  int4 ahead = b < nblk ? records[b] : make_int4(0, 0, 0, 0);
  if (EIGHT && b < nblk) {
    fetch(now, slots, ptr, a, a.tab.blk0 + b, ahead);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (b + stride < nblk) ahead = records[b + stride];
  }
  auto work = [&](const Fetched<T, EIGHT>& f, const Slots<T>& in, int64_t blk) {
    if (f.g) {  // without a gradient a tensor takes no step
      const int64_t slot = blk * BLK;
      const int n = f.used;
      const bool vec = f.vec;
      float pv[2][4], gv[2][4], mv[2][4], vv[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (vec && EIGHT) {
          widen<T>(in.p[j][threadIdx.x], pv[j]);
          widen<T>(in.g[j][threadIdx.x], gv[j]);
        } else if (vec) {
          widen<T>(f.pw[EIGHT ? 0 : j], pv[j]);
          widen<T>(f.gw[EIGHT ? 0 : j], gv[j]);
        } else {
          load4(f.p, j * 128 + lane * 4, n, false, pv[j]);
          load4(f.g, j * 128 + lane * 4, n, false, gv[j]);
        }
        if constexpr (EIGHT) {
          unhold4(in.m[j][threadIdx.x], f.ms, mv[j]);
          unhold4(in.v[j][threadIdx.x], f.vs, vv[j]);
        } else {
          widen<float>(f.mw[j], mv[j]);
          widen<float>(f.vw[j], vv[j]);
        }
      }
      if (f.t != t_have) {  // most often all tensors are at the same step
        t_have = f.t;
        alpha = lr / -expm1f(t_have * a.ln_b1);
        rc2 = rsqrtf(-expm1f(t_have * a.ln_b2));
      }
      float mmax = 0.f;
      uint32_t vtop = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // Every product and sum of the moments is rounded on its own (no fused
          // multiply-add), so they, and with them the codes, are those of the
          // formula taken operation by operation in f32, on any machine.
          const float gg = __fmul_rn(gv[j][k], coef);
          const float m = __fadd_rn(__fmul_rn(a.b1, mv[j][k]), __fmul_rn(a.b1c, gg));
          const float v = __fadd_rn(__fmul_rn(a.b2, vv[j][k]), __fmul_rn(__fmul_rn(a.b2c, gg), gg));
          pv[j][k] = pv[j][k] * decay - alpha * fast_div(m, fast_sqrt(v) * rc2 + a.eps);
          mv[j][k] = m;
          vv[j][k] = v;
          if constexpr (EIGHT) {
            mmax = fmaxf(mmax, fabsf(m));
            vtop = max(vtop, __float_as_uint(v));  // v is not negative; an inf or a NaN is the largest
          }
        }
        store4(f.p, j * 128 + lane * 4, n, vec, pv[j]);
        if constexpr (!EIGHT) {
          store4((float*)a.m + slot, j * 128 + lane * 4, BLK, true, mv[j]);
          store4((float*)a.v + slot, j * 128 + lane * 4, BLK, true, vv[j]);
        }
      }
      if constexpr (EIGHT) {
        mmax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mmax)));  // not negative
        vtop = __reduce_max_sync(0xffffffffu, vtop);
        const bool odd = vtop >= INF;
        if (odd) mend_odd(mv, vv, mmax, vtop);
        const float vmax = __uint_as_float(vtop);
        const uint32_t seed = random_seed(slot, (uint32_t)t_have) + lane * 4 * 0x9E3779B1u;
        if (!(vmax > TINY)) mmax = 0.f;  // v held as zeros: an m held beside them would next move by m / eps
        const float minv = mmax > TINY ? __fdiv_rn(448.f, mmax) : 0.f, vinv = vmax > TINY ? __fdiv_rn(448.f, vmax) : 0.f;
        const uint32_t least = vinv > 0.f ? 1u : 0u;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t om = 0, ov = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t r1, r2;
            random20(seed, j * 128 + k, r1, r2);
            const uint32_t qm = hold8(mv[j][k], minv, r1) | (__float_as_uint(mv[j][k]) >> 24 & 128u);
            const uint32_t qv = max(hold8(vv[j][k], vinv, r2), min(__float_as_uint(vv[j][k]), least));
            om |= qm << (8 * k);
            ov |= qv << (8 * k);
          }
          if (odd) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (vv[j][k] != vv[j][k]) {
                om |= 127u << (8 * k);
                ov |= 127u << (8 * k);
              }
          }
          *reinterpret_cast<uint32_t*>((unsigned char*)a.m + slot + j * 128 + lane * 4) = om;
          *reinterpret_cast<uint32_t*>((unsigned char*)a.v + slot + j * 128 + lane * 4) = ov;
        }
        if (lane == 0) {
          a.ms[blk] = mmax > TINY ? __fmul_rn(mmax, 1.f / 448.f) : 0.f;
          a.vs[blk] = vmax > TINY ? __fmul_rn(vmax, 1.f / 448.f) : 0.f;
        }
      }
    }
  };
  if constexpr (EIGHT) {
    // two sets of slots in turn; the newest copies are left under way
    auto turn = [&](Fetched<T, EIGHT>& f, int at, Fetched<T, EIGHT>& g) {
      const int4 rec = ahead;
      if (b + 2 * stride < nblk) ahead = records[b + 2 * stride];
      if (b + stride < nblk) fetch(g, slots + (at ^ 1), ptr, a, a.tab.blk0 + b + stride, rec);
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      work(f, slots[at], a.tab.blk0 + b);
      b += stride;
      return b < nblk;
    };
    if (b < nblk)
      while (turn(now, 0, next) && turn(next, 1, now)) {
      }
  } else {
    for (; b < nblk; b += stride) {
      const int4 rec = ahead;
      if (b + stride < nblk) ahead = records[b + stride];
      fetch(now, slots, ptr, a, a.tab.blk0 + b, rec);
      work(now, slots[0], a.tab.blk0 + b);
    }
  }
  // The last block counts the step: every block has read the counts by then.
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(&a.ctl->ticket_step, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (last) {
    for (int i = threadIdx.x; i < a.ntensors; i += blockDim.x)
      if (ptr.g[i]) a.steps[a.tab.t0 + i] += 1.f;
    if (threadIdx.x == 0) a.ctl->ticket_step = 0;
  }
}

struct NormArgs {
  Tables tab;
  double* part;     // one sum of squares a block of every launch
  int part0;        // this launch's first
  int finish;       // the last launch: add up part[0 .. part0 + gridDim.x)
  float max_norm;   // <= 0: no clipping
  int skip;         // a norm that is not finite calls the step off
  float* norm;      // the norm, written when not NULL
  float* found;     // set to 1 as well when the step is called off, when not NULL
  Ctl* ctl;
};

// Sum of squares of every gradient.  The squares are added in f64: a finite
// gradient never overflows the sum, so the sum is finite exactly when every
// gradient is, and one pass serves the clipping and the finite check.  The
// order of the additions is fixed by the grid.
template <typename T, int MAXT>
__global__ void __launch_bounds__(WARPS * 32) grad_norm_kernel(const __grid_constant__ Ptrs<MAXT> ptr, const NormArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double s = 0.0;
  const int64_t stride = (int64_t)gridDim.x * WARPS;
  int64_t b = (int64_t)blockIdx.x * WARPS + warp;
  int4 next = b < a.tab.nblk ? a.tab.block[a.tab.blk0 + b] : make_int4(0, 0, 0, 0);
  for (; b < a.tab.nblk; b += stride) {
    const int4 rec = next;
    if (b + stride < a.tab.nblk) next = a.tab.block[a.tab.blk0 + b + stride];
    const T* g = reinterpret_cast<const T*>(ptr.g[rec.x - a.tab.t0]);
    if (!g) continue;
    g += (int64_t)rec.y * BLK;
    const bool vec = aligned4<T>(g);
    float v[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) load4(g, j * 128 + lane * 4, rec.z, vec, v[j]);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) s += (double)v[j][k] * (double)v[j][k];
  }
  __shared__ double sh[WARPS];
  __shared__ bool last;
  auto block_sum = [&](double x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    __syncthreads();
    if (lane == 0) sh[warp] = x;
    __syncthreads();
    double r = 0.0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) r += sh[i];
    return r;
  };
  s = block_sum(s);
  if (threadIdx.x == 0) {
    a.part[a.part0 + blockIdx.x] = s;
    __threadfence();
    last = a.finish && atomicAdd(&a.ctl->ticket_norm, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double tot = 0.0;
  const int np = a.part0 + (int)gridDim.x;
  for (int i = threadIdx.x; i < np; i += blockDim.x) tot += __ldcg(a.part + i);
  tot = block_sum(tot);
  if (threadIdx.x == 0) {
    const float norm = (float)sqrt(tot);
    const bool bad = !isfinite(tot);
    float c = 1.f;
    if (a.max_norm > 0.f) {
      const float r = (float)((double)a.max_norm / (sqrt(tot) + 1e-6));
      c = r >= 1.f ? 1.f : r;  // a NaN stays one
    }
    a.ctl->coef = c;
    a.ctl->found = a.skip && bad ? 1.f : 0.f;
    if (a.skip && bad && a.found) *a.found = 1.f;
    if (a.norm) *a.norm = norm;
    a.ctl->ticket_norm = 0;
  }
}

constexpr int MAX_FEW = 32, MAX_MANY = 512;  // tensors of one launch (their pointers are its arguments)

int grid_for(int64_t nblk, int per_sm) {
  return (int)std::min<int64_t>((nblk + WARPS - 1) / WARPS, (int64_t)device_sm_count() * per_sm);
}

int check(const ow_adamw_t* a) {
  OW_CHECK_ARG(a != nullptr, "ow_adamw: args is NULL");
  OW_CHECK_ARG(a->tensors > 0, "ow_adamw: tensors must be positive (got %d)", a->tensors);
  OW_CHECK_ARG(a->params && a->grads && a->slots, "ow_adamw: params, grads or slots is NULL");
  OW_CHECK_ARG(a->dev_blocks && a->control, "ow_adamw: a device table is NULL");
  if (a->dtype != OW_DTYPE_F32 && a->dtype != OW_DTYPE_BF16 && a->dtype != OW_DTYPE_F16) {
    set_error("ow_adamw: parameters must be float32, bfloat16 or float16 (dtype code %d)", a->dtype);
    return OW_ERR_UNSUPPORTED;
  }
  const size_t es = dtype_size(a->dtype);
  OW_CHECK_ARG((uintptr_t)a->dev_blocks % 16 == 0 && (uintptr_t)a->control % 4 == 0, "ow_adamw: a device table is not aligned");
  for (int i = 0; i < a->tensors; ++i)
    OW_CHECK_ARG(((uintptr_t)a->params[i] | (uintptr_t)a->grads[i]) % es == 0, "ow_adamw: tensor %d is not aligned", i);
  for (int i = 0; i < a->tensors; ++i)
    OW_CHECK_ARG(a->slots[i] >= 0 && a->slots[i] % BLK == 0 && a->slots[i + 1] % BLK == 0 && a->slots[i] < a->slots[i + 1],
                 "ow_adamw: slots of tensor %d must be a rising multiple of %d", i, BLK);
  return OW_OK;
}

// Calls f(pointers, tables, tensors of the launch) for each launch of the call.
template <class F>
int each_launch(const ow_adamw_t* a, F&& f) {
  for (int t0 = 0; t0 < a->tensors; t0 += MAX_MANY) {
    const int n = std::min(MAX_MANY, a->tensors - t0);
    Tables tab{(const int4*)a->dev_blocks, t0, a->slots[t0] / BLK, (a->slots[t0 + n] - a->slots[t0]) / BLK};
    const bool end = t0 + n == a->tensors;
    auto fill = [&](auto& ptr) {
      for (int i = 0; i < n; ++i) {
        ptr.g[i] = a->grads[t0 + i];
        ptr.p[i] = a->params[t0 + i];
      }
    };
    if (n <= MAX_FEW) {  // a launch with few pointers starts sooner than one with 8 KB of them
      Ptrs<MAX_FEW> ptr{};
      fill(ptr);
      OW_RETURN_IF(f(ptr, tab, n, end));
    } else {
      Ptrs<MAX_MANY> ptr{};
      fill(ptr);
      OW_RETURN_IF(f(ptr, tab, n, end));
    }
  }
  return OW_OK;
}

template <class F>
int by_type(int dtype, F&& f) {
  if (dtype == OW_DTYPE_F32) return f((float*)nullptr);
  if (dtype == OW_DTYPE_BF16) return f((__nv_bfloat16*)nullptr);
  return f((__half*)nullptr);
}

// Blocks an SM.  8-bit blocks are fetched ahead by warps that stay (three are
// what the registers let run); with 32 bits more blocks than run at once even
// out what the memory's channels take (10.2 M parameters: 46.5 against 49.5 us).
constexpr int NORM_PER_SM = 6, STEP_PER_SM = 8, STEP8_PER_SM = 3;

}  // namespace
}  // namespace ow

using namespace ow;

extern "C" {

int32_t ow_grad_norm_partials(const ow_adamw_t* a) {
  clear_error();
  if (!a || a->tensors <= 0 || !a->slots) {
    set_error("ow_grad_norm_partials: no tensors");
    return 0;
  }
  int32_t n = 0;
  for (int t0 = 0; t0 < a->tensors; t0 += MAX_MANY) {
    const int c = std::min(MAX_MANY, a->tensors - t0);
    n += grid_for((a->slots[t0 + c] - a->slots[t0]) / BLK, NORM_PER_SM);
  }
  return n;
}

int ow_grad_norm(const ow_adamw_t* a, const ow_grad_norm_t* o, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  OW_CHECK_ARG(o && o->partials, "ow_grad_norm: options or partials is NULL");
  OW_CHECK_ARG((uintptr_t)o->partials % 8 == 0 && ((uintptr_t)o->norm | (uintptr_t)o->found) % 4 == 0,
               "ow_grad_norm: an output is not aligned");
  OW_CHECK_ARG(o->first >= 0 && o->capacity >= o->first + ow_grad_norm_partials(a),
               "ow_grad_norm: room for %d partial sums from %d on is needed, got %d", ow_grad_norm_partials(a), o->first,
               o->capacity);
  int at = o->first;
  return by_type(a->dtype, [&](auto* tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    return each_launch(a, [&](auto& ptr, const Tables& tab, int, bool end) -> int {
      NormArgs k{tab, o->partials, at, o->finish && end, o->max_norm, o->skip_nonfinite, o->norm, o->found, (Ctl*)a->control};
      const int grid = grid_for(tab.nblk, NORM_PER_SM);
      at += grid;
      using P = std::remove_reference_t<decltype(ptr)>;
      launch(grad_norm_kernel<T, sizeof(ptr.p) / sizeof(void*)>, grid, WARPS * 32, 0, (cudaStream_t)stream, (const P&)ptr, k);
      OW_CHECK_LAUNCH("grad_norm_kernel");
      return OW_OK;
    });
  });
}

int ow_adamw_step(const ow_adamw_t* a, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  OW_CHECK_ARG(a->state_bits == 32 || a->state_bits == 8, "ow_adamw_step: state_bits must be 32 or 8 (got %d)", a->state_bits);
  OW_CHECK_ARG(a->exp_avg && a->exp_avg_sq && a->dev_steps, "ow_adamw_step: a state pointer is NULL");
  OW_CHECK_ARG(a->state_bits == 32 || (a->exp_avg_scale && a->exp_avg_sq_scale), "ow_adamw_step: 8-bit states need their scales");
  OW_CHECK_ARG(((uintptr_t)a->exp_avg | (uintptr_t)a->exp_avg_sq) % (a->state_bits == 32 ? 16 : 4) == 0 &&
                   ((uintptr_t)a->exp_avg_scale | (uintptr_t)a->exp_avg_sq_scale | (uintptr_t)a->dev_steps |
                    (uintptr_t)a->lr_ptr | (uintptr_t)a->found) % 4 == 0,
               "ow_adamw_step: the state is not aligned");
  OW_CHECK_ARG(a->state_bits == 32 || (float)a->eps > 0.f,
               "ow_adamw_step: 8-bit states need a positive eps (both moments may be held as 0)");
  OW_CHECK_ARG(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0, "ow_adamw_step: betas must be in [0, 1)");
  for (int i = 0; i < a->tensors; ++i)
    OW_CHECK_ARG(a->params[i] || !a->grads[i], "ow_adamw_step: parameter %d is NULL", i);
  StepArgs k{};
  k.m = a->exp_avg; k.v = a->exp_avg_sq;
  k.ms = a->exp_avg_scale; k.vs = a->exp_avg_sq_scale;
  k.steps = a->dev_steps;
  k.lr_ptr = a->lr_ptr;
  k.found_in = a->found;
  k.ctl = (Ctl*)a->control;
  k.use_ctl = a->use_norm;
  k.lr = (float)a->lr;
  k.b1 = (float)a->beta1; k.b2 = (float)a->beta2;
  k.b1c = (float)(1.0 - a->beta1); k.b2c = (float)(1.0 - a->beta2);
  k.ln_b1 = (float)log(a->beta1); k.ln_b2 = (float)log(a->beta2);  // -inf for 0: the correction is then 1
  k.eps = (float)a->eps; k.wd = (float)a->weight_decay;
  return by_type(a->dtype, [&](auto* tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    return each_launch(a, [&](auto& ptr, const Tables& tab, int n, bool) -> int {
      k.tab = tab;
      k.ntensors = n;
      const int grid = grid_for(tab.nblk, a->state_bits == 8 ? STEP8_PER_SM : STEP_PER_SM);
      using P = std::remove_reference_t<decltype(ptr)>;
      constexpr int MAXT = sizeof(ptr.p) / sizeof(void*);
      if (a->state_bits == 8)
        launch(adamw_kernel<T, true, MAXT>, grid, WARPS * 32, 0, (cudaStream_t)stream, (const P&)ptr, k);
      else
        launch(adamw_kernel<T, false, MAXT>, grid, WARPS * 32, 0, (cudaStream_t)stream, (const P&)ptr, k);
      OW_CHECK_LAUNCH("adamw_kernel");
      return OW_OK;
    });
  });
}

}  // extern "C"
