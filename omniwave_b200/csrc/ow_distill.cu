// The loss of a classifier that learns from a teacher's top logits and from
// labels, and the gradient of its logits z [rows, classes].
//
// With q_T = softmax(z / T) over all classes and p = softmax(t / T) over the
// row's entries (t_j, c_j):
//   soft = T^2 sum_j p_j (log p_j - log q_T[c_j]);   hard = -log q_1[label]
//   loss = weight soft + (1 - weight) hard            (mean, sum or row by row)
//   dz   = a T (q_T - sum_j p_j [c_j]) + b (q_1 - [label])
// with a and b the factors of soft and hard in the loss times its gradient.
// All in f32, exponentials to the base of 2: with k = log2(e), the row's largest
// logit m and mk = m k,
//   s = sum 2^(z k - mk),   log q = (z k - mk - log2 s) / k
// where z k - mk is one rounding and the rounding of mk drops out.
//
// G threads share a row: a block, or a warp where rows are short.  The forward
// reads z once, with a running maximum; the backward reads it again and writes
// dz, first as if there were neither teacher nor label, then the entries of
// those classes anew: each of them takes everything that falls on its class, is
// computed in f32 and rounded once, in an order that the row alone fixes.
#include <algorithm>
#include <type_traits>

#include "ow_common.cuh"
#include "ow_internal.h"

namespace ow {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int THREADS = 256;
constexpr int MOST_TOP = 1024;

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
  float* lse_t;          // [rows] log2 of the sum of 2^(z kt); only where not NULL
  float* lse_1;          // the same for T = 1
  float* top;            // the same of the teacher's entries; +inf: the row has none
  float* soft;           // [rows] or NULL
  float* hard;           // [rows] or NULL, NaN-free 0 and top / lse_1 tell whether the row has one
  float* loss;           // [rows] or NULL
  // backward
  const float* dloss;
  int dloss_rows;        // a gradient for each row
  const float* coef;     // factors of soft and hard, or NULL: weight and 1 - weight
  void* dz;
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

// Calls f(first element, its index, whether V elements follow) for a row's elements in 16-byte units where it can.
template <int G, typename T, class F>
__device__ __forceinline__ void over_row(const T* z, int V, int lane, F&& f) {
  constexpr int U = 16 / sizeof(T);
  const int lead = min(V, (int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(T));
  const int units = (V - lead) / U;
  for (int i = lane; i < lead; i += G) f(i, std::integral_constant<int, 1>());
  for (int i = lane; i < units; i += G) f(lead + i * U, std::integral_constant<int, U>());
  for (int i = lead + units * U + lane; i < V; i += G) f(i, std::integral_constant<int, 1>());
}
template <int N, typename T>
__device__ __forceinline__ void ldn(const T* p, float (&o)[N]) {
  if constexpr (N == 1) {
    o[0] = widen(p[0]);
  } else {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    T v[N];
    *reinterpret_cast<uint4*>(v) = r;
#pragma unroll
    for (int k = 0; k < N; ++k) o[k] = widen(v[k]);
  }
}
template <int N, typename T>
__device__ __forceinline__ void stn(T* p, const float (&o)[N]) {
  if constexpr (N == 1) {
    p[0] = narrow<T>(o[0]);
  } else {
    alignas(16) T v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = narrow<T>(o[k]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
  }
}

template <int G>
__device__ __forceinline__ void row_sync() {
  if constexpr (G == 32) __syncwarp();
  else __syncthreads();
}

// A maximum with the sums of 2^(x k - m k) around it: the running state of a softmax.
struct Run {
  float m, st, s1;
};
// The pivot of a maximum; a row of -inf has none, and sums to 0.
__device__ __forceinline__ float pivot(float m) { return m == -INFINITY ? 0.f : m; }
// What a sum around m is worth around the pivot p: a sum that has seen no logit yet is 0.
__device__ __forceinline__ float moved(float m, float p, float k) { return m == -INFINITY ? 0.f : ex2((m - p) * k); }
__device__ __forceinline__ Run join(const Run& a, const Run& b, float kt) {
  Run r;
  r.m = fmaxf(a.m, b.m);
  const float p = pivot(r.m);
  r.st = a.st * moved(a.m, p, kt) + b.st * moved(b.m, p, kt);
  r.s1 = a.s1 * moved(a.m, p, LOG2E) + b.s1 * moved(b.m, p, LOG2E);
  return r;
}

template <int G, typename T>
__global__ void __launch_bounds__(THREADS) distill_fwd_kernel(const Args a) {
  constexpr int RB = THREADS / G;
  __shared__ Run sh[THREADS / 32];
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  for (int64_t r0 = (int64_t)blockIdx.x * RB; r0 < a.rows; r0 += (int64_t)gridDim.x * RB) {
    const int64_t row = r0 + sub;
    const bool live = row < a.rows;
    const T* z = (const T*)a.z + row * a.ld;
    const int64_t label = live && a.label ? ld_index(a.label, a.label8, row) : -1;
    Run run{-INFINITY, 0.f, 0.f};
    if (live)
      over_row<G>(z, a.V, lane, [&](int i, auto n) {
        constexpr int N = decltype(n)::value;
        float v[N];
        ldn<N>(z + i, v);
        float m = run.m;
#pragma unroll
        for (int k = 0; k < N; ++k) m = fmaxf(m, v[k]);
        const float p = pivot(m);
        if (m > run.m) {
          run.st *= moved(run.m, p, a.kt);
          run.s1 *= moved(run.m, p, LOG2E);
          run.m = m;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
          run.st += ex2(fmaf(v[k], a.kt, -p * a.kt));
          run.s1 += ex2(fmaf(v[k], LOG2E, -p * LOG2E));
        }
      });
#pragma unroll
    for (int o = 16; o; o >>= 1)
      run = join(run, Run{__shfl_xor_sync(0xffffffffu, run.m, o), __shfl_xor_sync(0xffffffffu, run.st, o),
                          __shfl_xor_sync(0xffffffffu, run.s1, o)}, a.kt);
    if constexpr (G > 32) {
      if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = run;
      __syncthreads();
      run = sh[0];
#pragma unroll
      for (int i = 1; i < G / 32; ++i) run = join(run, sh[i], a.kt);
      __syncthreads();
    }
    if (!live || lane >= 32) continue;
    const float p = pivot(run.m), mt = p * a.kt, m1 = p * LOG2E;
    const float log_t = log2f(run.st), log_1 = log2f(run.s1);
    // The teacher's entries, by one warp.
    float soft = 0.f, top = INFINITY;
    if (a.weight > 0.f) {
      const int64_t at = row * a.K;
      float tm = -INFINITY, ts = 0.f;
      bool bad = false;
      for (int j = lane; j < a.K; j += 32) {
        const int64_t c = ld_index(a.cls, a.cls8, at + j);
        if (c < 0) continue;
        bad |= c >= a.V;
        const float t = ld_teacher(a, at + j);
        bad |= t != t;
        tm = fmaxf(tm, t);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, o));
      bad = __any_sync(0xffffffffu, bad);
      if (bad) {
        soft = top = NAN;
      } else if (tm > -INFINITY) {
        const float tk = tm * a.kt;
        for (int j = lane; j < a.K; j += 32)
          if (ld_index(a.cls, a.cls8, at + j) >= 0) ts += ex2(fmaf(ld_teacher(a, at + j), a.kt, -tk));
#pragma unroll
        for (int o = 16; o; o >>= 1) ts += __shfl_xor_sync(0xffffffffu, ts, o);
        const float log_s = log2f(ts), inv = 1.f / ts;
        for (int j = lane; j < a.K; j += 32) {
          const int64_t c = ld_index(a.cls, a.cls8, at + j);
          if (c < 0) continue;
          const float d = fmaf(ld_teacher(a, at + j), a.kt, -tk), pj = ex2(d) * inv;
          if (pj > 0.f) soft += pj * ((d - log_s) - (fmaf(widen(z[c]), a.kt, -mt) - log_t));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) soft += __shfl_xor_sync(0xffffffffu, soft, o);
        soft *= LN2 * a.temp * a.temp;
        top = tk + log_s;
        if (tm == INFINITY) soft = top = NAN;
      }
    }
    float hard = 0.f, lse_1 = INFINITY;
    if (label >= 0 && a.weight < 1.f) {
      hard = label < a.V ? LN2 * (log_1 - fmaf(widen(z[label]), LOG2E, -m1)) : NAN;
      lse_1 = label < a.V ? m1 + log_1 : NAN;
    }
    if (lane == 0) {
      a.lse_t[row] = mt + log_t;
      a.lse_1[row] = lse_1;
      a.top[row] = top;
      if (a.soft) {
        a.soft[row] = soft;
        a.hard[row] = hard;
      }
      if (a.loss) a.loss[row] = a.weight * soft + (1.f - a.weight) * hard;
    }
  }
}

// The rows' sums, in an order that their number fixes: the loss, and the factors
// of soft and hard in it.
__global__ void __launch_bounds__(1024) distill_sum_kernel(const Args a, int mean, float* loss, float* coef) {
  __shared__ double sh[4][32];
  double v[4] = {0, 0, 0, 0};  // soft, its rows, hard, its rows
  for (int64_t i = threadIdx.x; i < a.rows; i += 1024) {
    v[0] += a.soft[i];
    v[1] += a.top[i] != INFINITY;
    v[2] += a.hard[i];
    v[3] += a.lse_1[i] != INFINITY;
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

template <int G, typename T>
__global__ void __launch_bounds__(THREADS) distill_bwd_kernel(const Args a) {
  constexpr int RB = THREADS / G;
  extern __shared__ float dyn[];  // [RB][2][K]: the entries' classes and probabilities
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  int* sc = reinterpret_cast<int*>(dyn) + sub * 2 * a.K;
  float* sp = dyn + sub * 2 * a.K + a.K;
  for (int64_t r0 = (int64_t)blockIdx.x * RB; r0 < a.rows; r0 += (int64_t)gridDim.x * RB) {
    const int64_t row = r0 + sub;
    const bool live = row < a.rows;
    const T* z = (const T*)a.z + row * a.ld;
    T* dz = (T*)a.dz + row * a.V;
    float lse_t = 0.f, lse_1 = 0.f, top = INFINITY, ks = 0.f, kh = 0.f;
    int64_t label = -1;
    if (live) {
      lse_t = a.lse_t[row];
      lse_1 = a.lse_1[row];
      top = a.top[row];
      const float g = a.dloss[a.dloss_rows ? row : 0];
      if (top != INFINITY) ks = g * (a.coef ? a.coef[0] : a.weight) * a.temp;
      if (lse_1 != INFINITY) {
        kh = g * (a.coef ? a.coef[1] : 1.f - a.weight);
        label = ld_index(a.label, a.label8, row);
      }
      if (top != top) ks = NAN;
      const bool any = top != INFINITY || lse_1 != INFINITY;
      const bool has_t = top != INFINITY, has_1 = lse_1 != INFINITY;
      auto value = [&](float v) {
        float d = 0.f;
        if (has_t) d = ks * ex2(fmaf(v, a.kt, -lse_t));
        if (has_1) d = fmaf(kh, ex2(fmaf(v, LOG2E, -lse_1)), d);
        return d;
      };
      auto dense = [&](int i, auto n) {
        constexpr int N = decltype(n)::value;
        float v[N];
        if (any) ldn<N>(z + i, v);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = any ? value(v[k]) : 0.f;
        stn<N>(dz + i, v);
      };
      if (((uintptr_t)z & 15) == ((uintptr_t)dz & 15)) over_row<G>(z, a.V, lane, dense);
      else
        for (int i = lane; i < a.V; i += G) dense(i, std::integral_constant<int, 1>());
      if (has_t)
        for (int j = lane; j < a.K; j += G) {
          const int64_t c = ld_index(a.cls, a.cls8, row * a.K + j);
          sc[j] = c < 0 || c >= a.V ? -1 : (int)c;
          sp[j] = sc[j] < 0 ? 0.f : ex2(fmaf(ld_teacher(a, row * a.K + j), a.kt, -top));
        }
    }
    row_sync<G>();
    if (live) {
      auto anew = [&](int c, float d) {  // class c with d to take off
        const float v = widen(z[c]);
        float u = lse_1 != INFINITY ? kh * ex2(fmaf(v, LOG2E, -lse_1)) : 0.f;
        if (top != INFINITY) u = fmaf(ks, ex2(fmaf(v, a.kt, -lse_t)), u);
        dz[c] = narrow<T>(u - d);
      };
      const int y = label >= 0 && label < a.V ? (int)label : -1;
      bool met = false;  // the label is among the entries
      if (top != INFINITY)
        for (int j = lane; j < a.K; j += G) {
          const int c = sc[j];
          if (c < 0) continue;
          bool first = true;
          for (int i = 0; i < j; ++i) first &= sc[i] != c;
          if (!first) continue;
          float d = 0.f;
          for (int i = j; i < a.K; ++i) d += sc[i] == c ? sp[i] : 0.f;
          anew(c, ks * d + (c == y ? kh : 0.f));
        }
      if (y >= 0 && lane == 0) {
        if (top != INFINITY)
          for (int i = 0; i < a.K; ++i) met |= sc[i] == y;
        if (!met) anew(y, kh);
      }
    }
    row_sync<G>();
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
  k.lse_t = a->stats;
  k.lse_1 = a->stats + a->rows;
  k.top = a->stats + 2 * a->rows;
  return k;
}

constexpr int WARP_ROW = 1024;  // rows of up to this many classes are a warp's

int grid_of(int64_t rows, int rb) {
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + rb - 1) / rb, (int64_t)device_sm_count() * 8));
}

template <class F>
int with(const ow_distill_t* a, F&& f) {
  auto type = [&](auto t) {
    return a->classes <= WARP_ROW ? f(std::integral_constant<int, 32>(), t) : f(std::integral_constant<int, THREADS>(), t);
  };
  switch (a->dtype) {
    case OW_DTYPE_F32: return type(float());
    case OW_DTYPE_BF16: return type(__nv_bfloat16());
    default: return type(__half());
  }
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
  with(a, [&](auto G, auto t) -> int {
    launch(distill_fwd_kernel<G.value, decltype(t)>, grid_of(k.rows, THREADS / G.value), THREADS, 0, st, k);
    return OW_OK;
  });
  OW_CHECK_LAUNCH("distill_fwd_kernel");
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
  return with(a, [&](auto G, auto t) -> int {
    constexpr int RB = THREADS / G.value;
    auto kern = distill_bwd_kernel<G.value, decltype(t)>;
    const size_t smem = (size_t)RB * 2 * k.K * sizeof(float);  // at most 64 KB
    if (smem > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) {
        set_error("ow_distill: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
        return OW_ERR_CUDA;
      }
    }
    launch(kern, grid_of(k.rows, RB), THREADS, smem, st, k);
    OW_CHECK_LAUNCH("distill_bwd_kernel");
    return OW_OK;
  });
}

}  // extern "C"
