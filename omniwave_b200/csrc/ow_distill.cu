// The loss of a classifier that learns from a teacher's top logits and from
// labels, and the gradient of its logits z [rows, classes].
//
// With q_T = softmax(z / T) over all classes and p = softmax(t / T) over the
// row's entries (t_j, c_j):
//   soft = T^2 sum_j p_j (log p_j - log q_T[c_j]);   hard = -log q_1[label]
//   loss = weight soft + (1 - weight) hard            (mean, sum or row by row)
//   dz   = a T (q_T - sum_j p_j [c_j]) + b (q_1 - [label])
// with a and b the factors of soft and hard in the loss times its gradient.
// All in f32, exponentials to the base of 2: with k = log2(e) and the row's largest
// logit m,
//   s = sum 2^((z - m) k),   log q = ((z - m) k - log2 s) / k
// where z - m comes first: a softmax does not hang on what its logits have in common,
// and z k - m k would lose as many of its bits as that has, and overflow where z is its
// type's lowest value (a class masked so is 2^-inf = 0).  A row's own terms, which the
// sums leave out, are in 64 bits.
//
// The forward reads z once, with a running maximum that is looked at once for
// four vectors; the backward reads it again and writes dz, first as if there were
// neither teacher nor label, then the entries of those classes anew: each of them
// takes everything that falls on its class, is computed in f32 and rounded once,
// in an order that the row alone fixes.
//
// What bounds it is HBM, if the exponentials do not: the special-function units do
// 16 a cycle and SM, two for each logit of 16 bits are half as much again as the
// memory takes.  So with T = 2 or 4 the second is the first one's power (POW; k / T
// is exact then), and one serves where T = 1 or a term is left out.
//
// A row is a warp's, or a block's, of which the last warp has the teacher's entries
// while the others have the logits: its loads depend on one another.
//
// Measured (B200, device time in a CUDA graph): 4096 x 32000 bf16, T = 2, 64 entries,
// forward 67 us (3.9 TB/s; issue slots, half of them taken, and rows that end together; 65
// with one multiply-add, z k - m k, in the place of distance and product) and backward 86
// (6.2 TB/s, HBM); T = 3 94 and 106; 2048 x 32000 f32, any T, 54 to 57 and 94 to 97; 1531 x
// 40009 f16 forward 35; 128 x 1000 6.7 and 5.7.
// Asking for a row's vectors ahead, across rows too, cost a fourth of the blocks and 6 us.
#include <algorithm>
#include <type_traits>

#include "ow_common.cuh"
#include "ow_internal.h"
#include "ow_sm100.cuh"

namespace ow {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453;
constexpr int MOST_TOP = 1024;  // a lane's entries are 32 at most

struct Args {
  int64_t rows, ld;
  int V, K;
  const void* z;
  const void* t;         // [rows, K]
  int t_dt;
  const void* cls;       // [rows, K]
  int cls8;              // 64-bit indices
  const void* label;     // [rows], or NULL
  int label8;
  float kt;              // log2(e) / T
  float temp;
  float weight;
  // What a row's forward leaves: its largest logit m and 1 over the sums of 2^((z - m) kt) and of 2^((z - m) k), apart,
  // since a logarithm of a sum in one float with m would take the rounding of m to every probability.  A scale's sign
  // bit says that the row lacks its term, NaN that an index or an entry makes the term NaN.
  float* pivot;          // [rows]
  float* scale_t;
  float* scale_1;
  float* top_pivot;      // [rows] the same of the teacher's entries: the largest t, 1 over the sum of 2^((t - it) kt)
  float* top_scale;
  float* soft;           // [rows] or NULL
  float* hard;
  float* loss;           // [rows] or NULL
  // backward
  const float* dloss;
  int dloss_rows;        // a gradient for each row
  const float* coef;     // factors of soft and hard, or NULL: weight and 1 - weight
  void* dz;
  int slots;             // of a row's table of classes: a power of two, at least 2 K
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen(float v) { return v; }
template <> __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float ld_teacher(const Args& a, int64_t i) {
  return a.t_dt == OW_DTYPE_F32   ? ((const float*)a.t)[i]
         : a.t_dt == OW_DTYPE_F16 ? __half2float(((const __half*)a.t)[i])
                                  : __bfloat162float(((const __nv_bfloat16*)a.t)[i]);
}
__device__ __forceinline__ int64_t ld_index(const void* p, int wide, int64_t i) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// ---------------------------------------------------------------- a row's logits
using f2 = uint64_t;  // two floats
__device__ __forceinline__ f2 both(float v) { return sm100::f2pack(v, v); }

template <typename T>
constexpr int PER = 16 / sizeof(T);  // elements of a 16-byte vector

template <typename T>
__device__ __forceinline__ void widen(const uint4& r, float (&o)[PER<T>]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = sm100::unpack2<std::is_same_v<T, __nv_bfloat16>>(w[i]);
      o[2 * i] = f.x;
      o[2 * i + 1] = f.y;
    }
  }
}
// The same as pairs.
template <typename T>
__device__ __forceinline__ void widen(const uint4& r, f2 (&o)[PER<T> / 2]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  if constexpr (sizeof(T) == 4) {
    o[0] = (f2)w[0] | (f2)w[1] << 32;
    o[1] = (f2)w[2] | (f2)w[3] << 32;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = sm100::unpack2<std::is_same_v<T, __nv_bfloat16>>(w[i]);
      o[i] = sm100::f2pack(f.x, f.y);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 narrow(const f2 (&v)[PER<T> / 2]) {
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
    w[0] = (uint32_t)v[0]; w[1] = (uint32_t)(v[0] >> 32);
    w[2] = (uint32_t)v[1]; w[3] = (uint32_t)(v[1] >> 32);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = sm100::f2unpack(v[i]);
      w[i] = sm100::pack2<std::is_same_v<T, __nv_bfloat16>>(f.x, f.y);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The larger of two vectors, element by element.
template <typename T>
__device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      o[i] = __float_as_uint(fmaxf(__uint_as_float(x[i]), __uint_as_float(y[i])));
    } else if constexpr (std::is_same_v<T, __half>) {
      const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&x[i]), *reinterpret_cast<const __half2*>(&y[i]));
      o[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x[i]), *reinterpret_cast<const __nv_bfloat162*>(&y[i]));
      o[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
template <typename T>
__device__ __forceinline__ uint4 least() {  // a vector of -inf
  constexpr uint32_t w = sizeof(T) == 4 ? 0xFF800000u : std::is_same_v<T, __half> ? 0xFC00FC00u : 0xFF80FF80u;
  return make_uint4(w, w, w, w);
}
__device__ __forceinline__ f2 ex2(f2 v) {
  const float2 f = sm100::f2unpack(v);
  return sm100::f2pack(ex2(f.x), ex2(f.y));
}
// e^(POW - 1) and e^POW of what POW says (0: not used, 1: one exponential serves for both).
template <int POW>
__device__ __forceinline__ f2 power1(f2 e) {
  if constexpr (POW == 4) return sm100::mul2(sm100::mul2(e, e), e);
  return e;
}

// How a row's elements lie in 16-byte units: up to ``lead`` singly, then whole units, then the rest singly.
template <typename T>
struct Lay {
  int lead, units;
  __device__ __forceinline__ Lay(const T* z, int V) {
    lead = min(V, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(T));
    units = (V - lead) / PER<T>;
  }
  __device__ __forceinline__ int rest() const { return lead + units * PER<T>; }
};

// A maximum with the sums of 2^(x k - m k) around it: the running state of a softmax.
struct Run {
  float m, st, s1;
};
// The pivot of a maximum; a row of -inf has none, and sums to 0.
__device__ __forceinline__ float pivot(float m) { return m == -INFINITY ? 0.f : m; }
// What a sum around m is worth around the pivot p: a sum that has seen no logit yet is 0.
__device__ __forceinline__ float moved(float m, float p, float k) { return m == -INFINITY ? 0.f : ex2((m - p) * k); }
// 2^((v - p) k).  The distance first: it is at most 0 where p is the largest, so that no logit, a type's lowest
// value among them, can overflow on the way, and it does not lose what v k and p k have in common.
__device__ __forceinline__ float above(float v, float p, float k) { return ex2((v - p) * k); }
// The states of a warp's lanes as one: each sum is moved once, to the largest maximum.
__device__ __forceinline__ Run join(Run r, float kt) {
  const float mine = r.m;
#pragma unroll
  for (int o = 16; o; o >>= 1) r.m = fmaxf(r.m, __shfl_xor_sync(0xffffffffu, r.m, o));
  const float p = pivot(r.m);
  r.st *= moved(mine, p, kt);
  r.s1 *= moved(mine, p, LOG2E);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    r.st += __shfl_xor_sync(0xffffffffu, r.st, o);
    r.s1 += __shfl_xor_sync(0xffffffffu, r.s1, o);
  }
  return r;
}

// The softmax state of a thread's share of a row, every G-th unit from ``lane`` on.
template <typename T, int G, int POW>
__device__ __forceinline__ Run softmax_share(const T* z, int V, int lane, float kt) {
  constexpr int N = 4;  // vectors under way at once
  const Lay<T> lay(z, V);
  Run run{-INFINITY, 0.f, 0.f};
  auto single = [&](int i) {
    const float v = widen(z[i]), m = fmaxf(run.m, v), p = pivot(m);
    run.st = run.st * moved(run.m, p, kt) + above(v, p, kt);
    run.s1 = run.s1 * moved(run.m, p, LOG2E) + above(v, p, LOG2E);
    run.m = m;
  };
  for (int i = lane; i < lay.lead; i += G) single(i);
  for (int i = lay.rest() + lane; i < V; i += G) single(i);
  f2 st[2] = {sm100::f2pack(run.st, 0.f), 0}, s1[2] = {sm100::f2pack(run.s1, 0.f), 0};  // four chains of sums
  const uint4* u = reinterpret_cast<const uint4*>(z + lay.lead);
  auto step = [&](const uint4 (&v)[N]) {
    float x[PER<T>];
    widen<T>(larger<T>(larger<T>(v[0], v[1]), larger<T>(v[2], v[3])), x);
    float m = run.m;
#pragma unroll
    for (int j = 0; j < PER<T>; ++j) m = fmaxf(m, x[j]);
    const float p = pivot(m);
    if (m > run.m) {
      const float ft = moved(run.m, p, kt), f1 = POW != 1 ? moved(run.m, p, LOG2E) : 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        st[c] = sm100::mul2(st[c], both(ft));
        if constexpr (POW != 1) s1[c] = sm100::mul2(s1[c], both(f1));
      }
      run.m = m;
    }
    const f2 less = both(-p);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      f2 d[PER<T> / 2];
      widen<T>(v[n], d);
#pragma unroll
      for (int j = 0; j < PER<T> / 2; ++j) {
        d[j] = sm100::add2(d[j], less);
        const f2 e = ex2(sm100::mul2(d[j], both(kt)));
        st[j & 1] = sm100::add2(st[j & 1], e);
        if constexpr (POW == 2) s1[j & 1] = sm100::fma2(e, e, s1[j & 1]);
        if constexpr (POW == 4) s1[j & 1] = sm100::fma2(sm100::mul2(e, e), sm100::mul2(e, e), s1[j & 1]);
        if constexpr (POW == 0) s1[j & 1] = sm100::add2(s1[j & 1], ex2(sm100::mul2(d[j], both(LOG2E))));
      }
    }
  };
  int i = lane;
  for (; i + (N - 1) * G < lay.units; i += N * G) {
    uint4 v[N];
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = __ldg(u + i + n * G);
    step(v);
  }
  if (i < lay.units) {
    uint4 v[N];
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = i + n * G < lay.units ? __ldg(u + i + n * G) : least<T>();
    step(v);
  }
  auto whole = [](const f2 (&v)[2]) {
    const float2 f = sm100::f2unpack(sm100::add2(v[0], v[1]));
    return f.x + f.y;
  };
  run.st = whole(st);
  run.s1 = POW == 1 ? run.st : whole(s1);
  return run;
}

// A scale as it is left for the backward, and whether its row has the term.
__device__ __forceinline__ float leave(float s, bool has) { return __uint_as_float((__float_as_uint(s) & 0x7FFFFFFFu) | (has ? 0u : 0x80000000u)); }
__device__ __forceinline__ bool has_term(float s) { return __float_as_int(s) >= 0; }

template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Threads of a block: eight warps with a row each, or a row's G and the warp of its entries.
constexpr int block_of(int G) { return G == 32 ? 256 : G + 32; }
constexpr int rows_of(int G) { return G == 32 ? 8 : 1; }

// ---------------------------------------------------------------- forward
// What a row's entries and label have to say without its logits' sums, by one warp:
//   soft / (T^2 ln 2) = own + (m - r) kt + log2 of the sum of 2^((z - m) kt)
// with r the largest of the entries' logits, in 64 bits: what is common to them and m is taken off before the product.
struct Said {
  double own;
  float r;
  float top_pivot, top_scale;
  float label;           // the label's logit
  int has_soft;          // 1, 0: no entries, or -1: not to be used
  int has_label;         // 1, 0, or -1: not a class
};
template <typename T>
__device__ __forceinline__ Said listen(const Args& a, const T* z, int64_t row, int lane, float* sx, float* sz) {
  Said s{0., 0.f, 0.f, 0.f, 0.f, 0, 0};
  const int64_t at = row * a.K;
  int64_t label = -1;
  if (a.label && a.weight < 1.f) label = ld_index(a.label, a.label8, row);
  float tm = -INFINITY, r = -INFINITY;
  bool bad = false;
  if (a.weight > 0.f) {
#pragma unroll 4
    for (int j = lane; j < a.K; j += 32) {
      const int64_t c = ld_index(a.cls, a.cls8, at + j);
      const float t = ld_teacher(a, at + j);
      const bool on = c >= 0, in = on && c < a.V;
      bad |= on && (!in || t != t || t == INFINITY);
      sx[j] = on ? t : -INFINITY;
      sz[j] = in ? widen(z[c]) : 0.f;
      if (on) tm = fmaxf(tm, t);
      if (in) r = fmaxf(r, sz[j]);
    }
  }
  if (label >= 0) {
    s.has_label = label < a.V ? 1 : -1;
    if (label < a.V) s.label = widen(z[label]);
  }
  if (a.weight <= 0.f) return s;
  __syncwarp();
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, o));
    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, o));
  }
  if (__any_sync(0xffffffffu, bad)) {
    s.has_soft = -1;
    return s;
  }
  if (tm == -INFINITY) return s;
  s.has_soft = 1;
  s.r = pivot(r);
  float sd = 0.f;           // sum of e d
  double ts = 0., sq = 0.;  // of e, e (z - r)
  for (int j = lane; j < a.K; j += 32) {
    const float d = (sx[j] - tm) * a.kt, e = ex2(d);
    if (e > 0.f) {  // a probability of 0 has no part, whatever the student says
      ts += e;
      sd = fmaf(e, d, sd);
      sq = fma((double)e, (double)sz[j] - s.r, sq);
    }
  }
  ts = warp_sum(ts);
  sd = warp_sum(sd);
  sq = warp_sum(sq);
  s.own = (sd - sq * a.kt) / ts - log2f((float)ts);
  s.top_pivot = tm;
  s.top_scale = 1.f / (float)ts;
  return s;
}

// Writes down a row's results.
__device__ __forceinline__ void conclude(const Args& a, int64_t row, Run run, const Said& s) {
  const float p = pivot(run.m);
  float soft = 0.f, hard = 0.f;
  if (s.has_soft > 0) soft = (float)(LN2 * a.temp * a.temp * (s.own + (((double)p - s.r) * a.kt + log2f(run.st))));
  if (s.has_label > 0) hard = (float)((double)p - s.label + LN2 * log2f(run.s1));
  if (s.has_soft < 0) soft = run.st = NAN;
  if (s.has_label < 0) hard = run.s1 = NAN;
  a.pivot[row] = p;
  a.scale_t[row] = leave(1.f / run.st, s.has_soft != 0);
  a.scale_1[row] = leave(1.f / run.s1, s.has_label != 0);
  a.top_pivot[row] = s.top_pivot;
  a.top_scale[row] = s.top_scale;
  if (a.soft) {
    a.soft[row] = soft;
    a.hard[row] = hard;
  }
  if (a.loss) a.loss[row] = a.weight * soft + (1.f - a.weight) * hard;
}

template <int G, typename T, int POW>
__global__ void __launch_bounds__(block_of(G), G == 32 ? 4 : 1024 / block_of(G)) distill_fwd_kernel(const Args a) {
  extern __shared__ float dyn[];  // [rows][2][K]: the entries' logits, the student's there
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if constexpr (G == 32) {
    float* sx = dyn + warp * 2 * a.K;
    for (int64_t row = (int64_t)blockIdx.x * 8 + warp; row < a.rows; row += (int64_t)gridDim.x * 8) {
      const T* z = (const T*)a.z + row * a.ld;
      Run run = softmax_share<T, 32, POW>(z, a.V, lane, a.kt);
      const Said said = listen(a, z, row, lane, sx, sx + a.K);
      run = join(run, a.kt);
      if (lane == 0) conclude(a, row, run, said);
      __syncwarp();  // before the next row's entries overwrite these
    }
  } else {
    constexpr int W = G / 32;
    __shared__ Run sh[2][W];  // used in turn, so one barrier a row is enough
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
      const T* z = (const T*)a.z + row * a.ld;
      Said said;
      if (warp < W) {
        Run run = softmax_share<T, G, POW>(z, a.V, threadIdx.x, a.kt);
        run = join(run, a.kt);
        if (lane == 0) sh[turn][warp] = run;
      } else {
        said = listen(a, z, row, lane, dyn, dyn + a.K);
      }
      __syncthreads();
      if (warp == W) {
        Run run = lane < W ? sh[turn][lane] : Run{-INFINITY, 0.f, 0.f};
        run = join(run, a.kt);
        if (lane == 0) conclude(a, row, run, said);
      }
    }
  }
}

// The rows' sums, in an order that their number fixes: the loss, and the factors
// of soft and hard in it.
__global__ void __launch_bounds__(1024) distill_sum_kernel(const Args a, int mean, float* loss, float* coef) {
  __shared__ double sh[4][32];
  double v[4] = {0, 0, 0, 0};  // soft, its rows, hard, its rows
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < a.rows; i += 1024) {
    v[0] += a.soft[i];
    v[1] += has_term(a.scale_t[i]);
    v[2] += a.hard[i];
    v[3] += has_term(a.scale_1[i]);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if ((threadIdx.x & 31) == 0) sh[k][threadIdx.x >> 5] = v[k];
  }
  __syncthreads();
  if (threadIdx.x) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = 0;
    for (int i = 0; i < 32; ++i) v[k] += sh[k][i];
  }
  const double cs = (double)a.weight / (mean ? max(v[1], 1.0) : 1.0), ch = (1.0 - (double)a.weight) / (mean ? max(v[3], 1.0) : 1.0);
  loss[0] = (float)(cs * v[0] + ch * v[2]);
  coef[0] = (float)cs;
  coef[1] = (float)ch;
}

// ---------------------------------------------------------------- backward
// A row's gradient but for its entries and its label:
//   qs 2^((z - m) kt) + qh 2^((z - m) k),   e (qs + c e^(POW - 1)) where POW says so
// with qs and qh the factors ks and kh of the two probabilities times their scales.
template <int POW>
struct Slope {
  float kt, ks, kh, qs, qh, c;
  f2 less;
  bool soft, none;  // has a teacher; learns from nothing
  __device__ __forceinline__ Slope(const Args& a, int64_t row) : kt(a.kt), ks(0.f), kh(0.f), qs(0.f), qh(0.f), less(both(-a.pivot[row])) {
    const float scale_t = a.scale_t[row], scale_1 = a.scale_1[row], g = a.dloss[a.dloss_rows ? row : 0];
    soft = has_term(scale_t);
    none = !soft && !has_term(scale_1);
    if (soft) {
      ks = g * (a.coef ? a.coef[0] : a.weight) * a.temp;
      qs = ks * scale_t;
    }
    if (has_term(scale_1)) {
      kh = g * (a.coef ? a.coef[1] : 1.f - a.weight);
      qh = kh * scale_1;
    }
    c = POW == 1 ? qs + qh : qh;
  }
  __device__ __forceinline__ f2 operator()(f2 v) const {
    const f2 d = sm100::add2(v, less), e = ex2(sm100::mul2(d, both(kt)));
    if constexpr (POW == 1) return sm100::mul2(e, both(c));
    if constexpr (POW >= 2) return sm100::mul2(e, sm100::fma2(both(c), power1<POW>(e), both(qs)));
    const f2 f = ex2(sm100::mul2(d, both(LOG2E)));
    return sm100::fma2(e, both(qs), qh != 0.f ? sm100::mul2(f, both(qh)) : 0);
  }
  __device__ __forceinline__ float operator()(float v) const { return sm100::f2unpack((*this)(both(v))).x; }
};

// A thread's share of a row's gradient, every G-th unit from ``lane`` on.
template <typename T, int G, int POW>
__device__ __forceinline__ void slope_share(const T* z, T* dz, int V, int lane, const Slope<POW>& slope) {
  constexpr int N = 4, P = PER<T> / 2;
  const Lay<T> lay(dz, V);
  auto single = [&](int i) { dz[i] = narrow<T>(slope.none ? 0.f : slope(widen(z[i]))); };
  if (((uintptr_t)z ^ (uintptr_t)dz) & 15) {  // rows of z that start elsewhere in a unit
    for (int i = lane; i < V; i += G) single(i);
    return;
  }
  for (int i = lane; i < lay.lead; i += G) single(i);
  for (int i = lay.rest() + lane; i < V; i += G) single(i);
  const uint4* u = reinterpret_cast<const uint4*>(z + lay.lead);
  uint4* o = reinterpret_cast<uint4*>(dz + lay.lead);
  for (int i = lane; i < lay.units; i += N * G) {
    uint4 v[N];
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = !slope.none && i + n * G < lay.units ? __ldg(u + i + n * G) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      f2 x[P];
      widen<T>(v[n], x);
#pragma unroll
      for (int j = 0; j < P; ++j) x[j] = slope.none ? 0 : slope(x[j]);
      if (i + n * G < lay.units) o[i + n * G] = narrow<T>(x);
    }
  }
}

// What is to be written at a row's entries and its label, by one warp.
struct Amends {
  uint32_t first;  // of this lane's entries (every 32nd): those whose value is to be written
  int label;       // the label's class where no entry has it, or -1, and its value
  float value;
};
// ``mem``: [K] classes, [K] probabilities, [K] values, [slots] of a table of classes.
template <typename T, int POW>
__device__ __forceinline__ Amends amends(const Args& a, const T* z, int64_t row, int lane, const Slope<POW>& slope, float* mem) {
  int* sc = reinterpret_cast<int*>(mem);
  float *sp = mem + a.K, *sv = sp + a.K;
  int* table = reinterpret_cast<int*>(sv + a.K);
  Amends m{0u, -1, 0.f};
  if (a.label && slope.kh != 0.f) {
    const int64_t y = ld_index(a.label, a.label8, row);
    if (y >= 0 && y < a.V) {
      m.label = (int)y;
      m.value = slope(widen(z[y])) - slope.kh;
    }
  }
  if (!slope.soft) return m;
  for (int i = lane; i < a.slots; i += 32) table[i] = -1;
  const float tm = a.top_pivot[row], by = a.top_scale[row];
#pragma unroll 4
  for (int j = lane; j < a.K; j += 32) {
    const int64_t c = ld_index(a.cls, a.cls8, row * a.K + j);
    const float t = ld_teacher(a, row * a.K + j);
    const bool in = c >= 0 && c < a.V;
    const float p = in ? above(t, tm, a.kt) * by : 0.f;
    sc[j] = p > 0.f ? (int)c : -1;  // what has no probability takes nothing off
    sp[j] = p;
    sv[j] = in ? slope(widen(z[c])) : 0.f;
  }
  __syncwarp();
  // Whether a class is named twice: whichever entry comes to the table first, the answer is the same.
  bool twice = false;
  for (int j = lane; j < a.K; j += 32) {
    const int c = sc[j];
    if (c < 0) continue;
    for (uint32_t h = (uint32_t)c * 2654435761u >> 16;; ++h) {
      const int old = atomicCAS(table + (h & (a.slots - 1)), -1, c);
      twice |= old == c;
      if (old == -1 || old == c) break;
    }
  }
  twice = __any_sync(0xffffffffu, twice);
  bool met = false;  // the label is among the entries
  for (int j = lane, k = 0; j < a.K; j += 32, ++k) {
    const int c = sc[j];
    if (c < 0) continue;
    bool first = true;
    float d = sp[j];
    if (twice) {
      for (int i = 0; i < j; ++i) first &= sc[i] != c;
      for (int i = j + 1; i < a.K; ++i) d += sc[i] == c ? sp[i] : 0.f;
    }
    if (!first) continue;
    met |= c == m.label;
    sv[j] -= fmaf(slope.ks, d, c == m.label ? slope.kh : 0.f);
    m.first |= 1u << k;
  }
  if (__any_sync(0xffffffffu, met)) m.label = -1;
  return m;
}
template <typename T>
__device__ __forceinline__ void amend(const Args& a, T* dz, const Amends& m, int lane, const float* mem) {
  const int* sc = reinterpret_cast<const int*>(mem);
  const float* sv = mem + 2 * a.K;
  if (m.first)
    for (int j = lane, k = 0; j < a.K; j += 32, ++k)
      if (m.first >> k & 1) dz[sc[j]] = narrow<T>(sv[j]);
  if (lane == 0 && m.label >= 0) dz[m.label] = narrow<T>(m.value);
}

template <int G, typename T, int POW>
__global__ void __launch_bounds__(block_of(G), G == 32 ? 4 : 1024 / block_of(G)) distill_bwd_kernel(const Args a) {
  extern __shared__ float dyn[];  // [rows][3 K + slots]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if constexpr (G == 32) {
    float* mem = dyn + warp * (3 * a.K + a.slots);
    for (int64_t row = (int64_t)blockIdx.x * 8 + warp; row < a.rows; row += (int64_t)gridDim.x * 8) {
      const T* z = (const T*)a.z + row * a.ld;
      T* dz = (T*)a.dz + row * a.V;
      const Slope<POW> slope(a, row);
      const Amends m = amends<T>(a, z, row, lane, slope, mem);
      slope_share<T, 32>(z, dz, a.V, lane, slope);
      __syncwarp();
      amend(a, dz, m, lane, mem);
      __syncwarp();  // before the next row's entries overwrite these
    }
  } else {
    constexpr int W = G / 32;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
      const T* z = (const T*)a.z + row * a.ld;
      T* dz = (T*)a.dz + row * a.V;
      const Slope<POW> slope(a, row);
      Amends m{};
      if (warp < W) slope_share<T, G>(z, dz, a.V, threadIdx.x, slope);
      else m = amends<T>(a, z, row, lane, slope, dyn);
      __syncthreads();
      if (warp == W) {
        amend(a, dz, m, lane, dyn);
        __syncwarp();
      }
    }
  }
}

// ---------------------------------------------------------------- host
bool float_type(int dt) { return dt == OW_DTYPE_F32 || dt == OW_DTYPE_BF16 || dt == OW_DTYPE_F16; }

int check(const ow_distill_t* a) {
  OW_CHECK_ARG(a != nullptr, "ow_distill: args is NULL");
  OW_CHECK_ARG(a->rows >= 0 && a->rows < (1LL << 40) && a->classes > 0 && a->classes < (1 << 30) && a->top > 0,
               "ow_distill: bad shape [%lld, %d], %d entries", (long long)a->rows, a->classes, a->top);
  OW_CHECK_ARG(a->ld >= a->classes, "ow_distill: a row stride is shorter than its row");
  if (a->top > MOST_TOP) {
    set_error("ow_distill: at most %d entries a row (got %d)", MOST_TOP, a->top);
    return OW_ERR_UNSUPPORTED;
  }
  if (!float_type(a->dtype) || !float_type(a->top_dtype)) {
    set_error("ow_distill: dtypes must be float32, bfloat16 or float16");
    return OW_ERR_UNSUPPORTED;
  }
  OW_CHECK_ARG((a->class_bytes == 4 || a->class_bytes == 8) && (!a->labels || a->label_bytes == 4 || a->label_bytes == 8),
               "ow_distill: classes and labels must be 32- or 64-bit integers");
  OW_CHECK_ARG(a->temperature > 0.0 && a->temperature <= 1e4 && a->temperature >= 1e-4, "ow_distill: the temperature must be 1e-4 to 1e4");
  OW_CHECK_ARG(a->weight >= 0.0 && a->weight <= 1.0, "ow_distill: the weight must be 0 to 1");
  OW_CHECK_ARG(a->reduction >= OW_REDUCE_NONE && a->reduction <= OW_REDUCE_SUM, "ow_distill: unknown reduction %d", a->reduction);
  OW_CHECK_ARG(a->rows == 0 || (a->logits && a->top_logits && a->top_classes && a->stats), "ow_distill: a pointer is NULL");
  OW_CHECK_ARG((uintptr_t)a->logits % dtype_size(a->dtype) == 0 && (uintptr_t)a->top_logits % dtype_size(a->top_dtype) == 0 &&
                   (uintptr_t)a->top_classes % a->class_bytes == 0 && (!a->labels || (uintptr_t)a->labels % a->label_bytes == 0) &&
                   ((uintptr_t)a->stats | (uintptr_t)a->loss | (uintptr_t)a->factors) % 4 == 0,
               "ow_distill: a tensor is not aligned");
  return OW_OK;
}

Args base(const ow_distill_t* a) {
  Args k{};
  k.rows = a->rows; k.ld = a->ld; k.V = a->classes; k.K = a->top;
  k.z = a->logits;
  k.t = a->top_logits; k.t_dt = a->top_dtype;
  k.cls = a->top_classes; k.cls8 = a->class_bytes == 8;
  k.label = a->labels; k.label8 = a->label_bytes == 8;
  k.kt = (float)(1.4426950408889634 / a->temperature);
  k.temp = (float)a->temperature;
  k.weight = (float)a->weight;
  if (a->weight == 0.0) {  // T has no say
    k.kt = LOG2E;
    k.temp = 1.f;
  }
  k.pivot = a->stats;
  k.scale_t = a->stats + a->rows;
  k.scale_1 = a->stats + 2 * a->rows;
  k.top_pivot = a->stats + 3 * a->rows;
  k.top_scale = a->stats + 4 * a->rows;
  return k;
}

// Calls f<G, T, POW>: the threads of a row, its type and what serves for the second exponential.
template <class F>
int with(const ow_distill_t* a, F&& f) {
  const bool hard = a->labels && a->weight < 1.0, soft = a->weight > 0.0;
  const int pow = !hard || !soft || a->temperature == 1.0 ? 1 : a->temperature == 2.0 ? 2 : a->temperature == 4.0 ? 4 : 0;
  auto power = [&](auto g, auto t) -> int {
    switch (pow) {
      case 1: return f(g, t, std::integral_constant<int, 1>());
      case 2: return f(g, t, std::integral_constant<int, 2>());
      case 4: return f(g, t, std::integral_constant<int, 4>());
      default: return f(g, t, std::integral_constant<int, 0>());
    }
  };
  auto type = [&](auto t) -> int {
    // A warp a row where rows are many and not long, forward and backward of bf16, T = 2, 32 entries: 16384 x 2000 70 us
    // (a block a row 188), 4096 x 8000 50 (69), 2048 x 8000 36 (38; f32 54 and 51), 1024 x 2000 18 (20); but 1024 x 8000
    // 25 (23), 4096 x 16000 87 (98; f32 160 and 144), 128 x 1000 15 (13).  Its entries have to leave room for those of the
    // block's other rows.
    const int64_t rows = a->rows, sms = device_sm_count();
    const bool warps = a->top <= 256 && (a->classes <= 256 || (a->classes <= 8192 && rows >= (a->classes <= 4096 ? 6 : 14) * sms));
    return warps ? power(std::integral_constant<int, 32>(), t) : power(std::integral_constant<int, 224>(), t);
  };
  switch (a->dtype) {
    case OW_DTYPE_F32: return type(float());
    case OW_DTYPE_BF16: return type(__nv_bfloat16());
    default: return type(__half());
  }
}

// ``smem``: at most 40 KB, of eight rows with 256 entries each (one with 1024: 20 KB).
template <class K>
int launch_rows(K kern, const char* name, int G, size_t smem, const Args& k, cudaStream_t st) {
  const int rb = rows_of(G);
  const int64_t grid = std::min<int64_t>((k.rows + rb - 1) / rb, (int64_t)device_sm_count() * 8);
  launch(kern, (int)grid, block_of(G), smem, st, k);
  OW_CHECK_LAUNCH(name);
  return OW_OK;
}

}  // namespace
}  // namespace ow

using namespace ow;

extern "C" {

size_t ow_distill_workspace_size(const ow_distill_t* a) {
  clear_error();
  if (check(a) != OW_OK) return 0;
  return (size_t)a->rows * 2 * sizeof(float) + 256;
}

int ow_distill_fwd(const ow_distill_t* a, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  if (a->rows == 0) return OW_OK;
  OW_CHECK_ARG(a->loss && (a->reduction == OW_REDUCE_NONE || a->factors), "ow_distill_fwd: a pointer is NULL");
  const size_t need = ow_distill_workspace_size(a);
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("ow_distill_fwd needs %zu workspace bytes, got %zu", need, a->workspace_bytes);
    return OW_ERR_WORKSPACE;
  }
  Args k = base(a);
  if (a->reduction == OW_REDUCE_NONE) {
    k.loss = a->loss;
  } else {
    k.soft = (float*)(((uintptr_t)a->workspace + 255) & ~(uintptr_t)255);
    k.hard = k.soft + a->rows;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  OW_RETURN_IF(with(a, [&](auto G, auto t, auto pow) -> int {
    return launch_rows(distill_fwd_kernel<G.value, decltype(t), pow.value>, "distill_fwd_kernel", G.value,
                       (size_t)rows_of(G.value) * 2 * k.K * sizeof(float), k, st);
  }));
  if (a->reduction != OW_REDUCE_NONE) {
    launch(distill_sum_kernel, 1, 1024, 0, st, k, a->reduction == OW_REDUCE_MEAN, a->loss, a->factors);
    OW_CHECK_LAUNCH("distill_sum_kernel");
  }
  return OW_OK;
}

int ow_distill_bwd(const ow_distill_t* a, const ow_distill_grads_t* g, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  OW_CHECK_ARG(g != nullptr, "ow_distill_bwd: grads is NULL");
  if (a->rows == 0) return OW_OK;
  OW_CHECK_ARG(g->dloss && g->dlogits && (a->reduction == OW_REDUCE_NONE || a->factors), "ow_distill_bwd: a pointer is NULL");
  OW_CHECK_ARG((uintptr_t)g->dloss % 4 == 0 && (uintptr_t)g->dlogits % dtype_size(a->dtype) == 0,
               "ow_distill_bwd: a gradient is not aligned");
  Args k = base(a);
  k.dloss = g->dloss;
  k.dloss_rows = a->reduction == OW_REDUCE_NONE;
  k.coef = a->reduction == OW_REDUCE_NONE ? nullptr : a->factors;
  k.dz = g->dlogits;
  const cudaStream_t st = (cudaStream_t)stream;
  k.slots = 2;
  while (k.slots < 2 * k.K) k.slots *= 2;
  return with(a, [&](auto G, auto t, auto pow) -> int {
    return launch_rows(distill_bwd_kernel<G.value, decltype(t), pow.value>, "distill_bwd_kernel", G.value,
                       (size_t)rows_of(G.value) * (3 * k.K + k.slots) * sizeof(float), k, st);
  });
}

}  // extern "C"
