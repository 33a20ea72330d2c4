// RMSNorm before and after a block, fused with the block's gate, the
// per-sample residual scale and the residual add.
//
// A row is one token's C channels; sample b owns ``tokens`` rows.  With
// rms(v) = v rsqrt(mean(v^2) + eps), everything in f32:
//   d^ = rms(delta);  h = x + s_b q (d^ wp)          (post-norm, gate q, scale s)
//   h^ = rms(h);      n = h^ wn                      (the next block's pre-norm)
// Without delta h is x and only n is written.  Backward, from dh and dn:
//   u = dn wn;        D = dh + r_h (u - h^ mean(u h^))                dx = D
//   e = s q wp D;     ddelta = r_d (e - d^ mean(e d^))
//   dwn = sum dn h^;  dwp = sum s q D d^;  dq = sum s D d^ wp
// h is recomputed from x and delta, so the f32 sums see the f32 h and not the
// rounded one, and nothing but x, delta and two floats a row is kept.
//
// Split.  G threads share a row, each with NV vectors of V channels in
// registers, so a row is read once; rows of up to 32 lanes need only shuffles.
// A block stays within the rows that share a gate (all of them, or one
// sample's), so it keeps the channels' factors q wp and wn in shared memory
// instead of reading 8 to 12 bytes of weights an element again and again.
// The backward needs three sums a row, taken in one exchange: with
// A = sum e' (dh + r_h u), B = sum e' h^, S = sum u h^ (e' = s q wp d^),
// mean(e d^) = (A - B r_h S / C) / C.  Both of the post-norm's gradients follow
// from one sum, t = sum s D d^: dwp = q t and dq = wp t.  Each thread adds its
// channels' shares in registers over all its rows; a block leaves one partial
// row and a second kernel adds these in a fixed order.
//
// Bound: HBM.  Measured (B200, device time in a CUDA graph): 128 x 3136 x 128, f32
// stream, 16-bit branch, next norm, gate and scale, forward and backward 298 us
// for 1.75 GB (5.9 TB/s, 89% of the copy bandwidth); 50176 x 1024 bf16 forward
// 77 us (5.4 TB/s), with the backward 242 (4.3 TB/s); one token 3 us.
#include <algorithm>

#include "ow_common.cuh"
#include "ow_internal.h"

namespace ow {
namespace {

struct Args {
  int64_t rows, tokens;
  int C;
  const void* x;
  const void* delta;
  const void* dh;
  const void* dn;
  const void* wp;
  const void* q;
  const void* wn;
  int wp_dt, q_dt, wn_dt, n_dt;
  int x_dt, d_dt;
  int q_rows;            // 0: no gate, 1: one for all, else one for each sample
  const float* scale;    // [samples] or NULL
  float eps, inv_c;
  void* h;
  void* n;
  float* rd;             // [rows] 1 / rms(delta)
  float* rh;             // [rows] 1 / rms(h)
  void* dx;
  void* ddelta;
  float* part;           // [parts][arrays][C] partial sums: of dn h^ (with a next norm), of s D d^ (with delta)
  int arrays;
  int64_t groups;        // gate rows whose gradients are kept apart (1 or samples)
  int per_group;         // blocks that share a group's rows
  int64_t group_rows;
};

// V channels from p (an array of dtype dt) as floats.
template <int V>
__device__ __forceinline__ void ldv(const void* p, int dt, int64_t i, float (&o)[V]) {
  if (dt == OW_DTYPE_F32) {
    const float* f = (const float*)p + i;
    if constexpr (V == 8) {
      const float4 a = *reinterpret_cast<const float4*>(f), b = *reinterpret_cast<const float4*>(f + 4);
      o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
    } else {
      o[0] = f[0];
    }
  } else if constexpr (V == 8) {
    const uint4 r = *reinterpret_cast<const uint4*>((const uint16_t*)p + i);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float2 f;
      if (dt == OW_DTYPE_BF16) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
      else f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      o[2 * k] = f.x;
      o[2 * k + 1] = f.y;
    }
  } else {
    o[0] = dt == OW_DTYPE_BF16 ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : __half2float(((const __half*)p)[i]);
  }
}

// Eight 16-bit values as floats.
__device__ __forceinline__ void widen8(const uint4& r, int dt, float (&o)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float2 f;
    if (dt == OW_DTYPE_BF16) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
    else f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    o[2 * k] = f.x;
    o[2 * k + 1] = f.y;
  }
}

template <int V>
__device__ __forceinline__ void stv(void* p, int dt, int64_t i, const float (&v)[V]) {
  if (dt == OW_DTYPE_F32) {
    float* f = (float*)p + i;
    if constexpr (V == 8) {
      *reinterpret_cast<float4*>(f) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(f + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      f[0] = v[0];
    }
  } else if constexpr (V == 8) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (dt == OW_DTYPE_BF16) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&t);
      } else {
        const __half2 t = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&t);
      }
    }
    *reinterpret_cast<uint4*>((uint16_t*)p + i) = make_uint4(w[0], w[1], w[2], w[3]);
  } else if (dt == OW_DTYPE_BF16) {
    ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v[0]);
  } else {
    ((__half*)p)[i] = __float2half_rn(v[0]);
  }
}

__device__ __forceinline__ float ld1(const void* p, int dt, int64_t i) {
  float o[1];
  ldv<1>(p, dt, i, o);
  return o[0];
}

// Ragged rows: C is no multiple of 8, so a row starts anywhere in a 16-byte unit.
// Its threads take the aligned units that it touches and leave out what belongs
// to its neighbours: channel c of a unit's first element is then -7 to C - 1.
// Rows 8 apart start alike, so a thread whose rows are a multiple of 8 apart
// keeps its channels from row to row.  (777 channels, 64 x 784 rows of bf16,
// forward and backward: element by element 1066 us, in units 368.)
__device__ __forceinline__ bool inside(int c, int C) { return c >= 0 && c + 8 <= C; }
template <bool RAG>
__device__ __forceinline__ uint4 fetch8(const void* p, int64_t i, int64_t total) {
  const uint16_t* u = (const uint16_t*)p + i;
  if (!RAG || i + 8 <= total) return *reinterpret_cast<const uint4*>(u);
  uint32_t w[4] = {0, 0, 0, 0};  // the array's end
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (i + k < total) w[k / 2] |= (uint32_t)u[k] << (16 * (k & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <bool RAG, int V>
__device__ __forceinline__ void mask(float (&o)[V], int c, int C) {
  if constexpr (RAG) {
    if (!inside(c, C)) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (c + k < 0 || c + k >= C) o[k] = 0.f;
    }
  }
}
template <bool RAG, int V>
__device__ __forceinline__ void load(const void* p, int dt, int64_t i, int64_t total, int c, int C, float (&o)[V]) {
  if constexpr (RAG) {
    if (i + V <= total) ldv<V>(p, dt, i, o);
    else
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] = i + k < total ? ld1(p, dt, i + k) : 0.f;
    mask<RAG>(o, c, C);
  } else {
    ldv<V>(p, dt, i, o);
  }
}
template <bool RAG, int V>
__device__ __forceinline__ void store(void* p, int dt, int64_t i, int c, int C, const float (&v)[V]) {
  if (!RAG || inside(c, C)) {
    stv<V>(p, dt, i, v);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (c + k >= 0 && c + k < C) {
        const float one[1] = {v[k]};
        stv<1>(p, dt, i + k, one);
      }
  }
}

// Eight sums to a row of floats that starts on 16 bytes.
__device__ __forceinline__ void store_each(float* to, int c, int C, const float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (c + k >= 0 && c + k < C) to[c + k] = v[k];
}

// Sum of K values over the G threads of a row; every thread gets it.  Rows of
// more than a warp meet in shared memory (``sh``: [2][K][32] floats a block,
// used in turn, so one barrier an exchange is enough).
template <int G, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* sh, int& turn) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (G > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w0 = threadIdx.x / G * (G / 32);
    float* s = sh + turn * K * 32;
    turn ^= 1;
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k * 32 + warp] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < G / 32; ++i) t += s[k * 32 + w0 + i];
      v[k] = t;
    }
  }
}

// A block's channel factors in shared memory: q wp (with delta) and wn (with a
// next norm).  Vectors of 8 are kept as two planes of 4, so a warp's 16-byte
// reads do not conflict; for ragged rows as eight planes, with room for the
// channels before the first and behind the last, read value by value.
template <int V, bool RAG>
__host__ __device__ constexpr int factor_floats(int C) {
  return RAG ? 8 * ((C >> 3) + 3) : C;
}
template <int V, bool RAG>
__device__ __forceinline__ int plane(int c, int C) {
  if constexpr (RAG) return (c & 7) * ((C >> 3) + 3) + (c >> 3) + 1;
  else if constexpr (V == 8) return (c & 4) * (C >> 3) + (c >> 3) * 4 + (c & 3);
  else return c;
}
template <int V, bool RAG>
__device__ __forceinline__ void factors(const float* w, int c, int C, float (&o)[V]) {
  if constexpr (RAG) {
#pragma unroll
    for (int k = 0; k < V; ++k) o[k] = w[plane<V, RAG>(c + k, C)];
  } else if constexpr (V == 8) {
    const float4 a = *reinterpret_cast<const float4*>(w + (c >> 1)), b = *reinterpret_cast<const float4*>(w + (C >> 1) + (c >> 1));
    o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
  } else {
    o[0] = w[c];
  }
}
template <int V, bool DELTA, bool NEXT, bool RAG>
__device__ __forceinline__ void load_factors(const Args& a, int64_t group, float* kq, float* wn) {
  // beside the channels: zeros, which meet zeros
  for (int c = (int)threadIdx.x - (RAG ? 8 : 0); c < a.C + (RAG ? 8 : 0); c += blockDim.x) {
    const bool on = !RAG || (c >= 0 && c < a.C);
    if constexpr (DELTA) {
      float w = on ? ld1(a.wp, a.wp_dt, c) : 0.f;
      if (on && a.q_rows) w *= ld1(a.q, a.q_dt, (a.q_rows > 1 ? group * a.C : 0) + c);
      kq[plane<V, RAG>(c, a.C)] = w;
    }
    if constexpr (NEXT) wn[plane<V, RAG>(c, a.C)] = on ? ld1(a.wn, a.wn_dt, c) : 0.f;
  }
  __syncthreads();
}

__device__ __forceinline__ int64_t sample_of(const Args& a, int64_t row) {
  return a.rows < (1LL << 32) ? (int64_t)((uint32_t)row / (uint32_t)a.tokens) : row / a.tokens;
}

// Block (group, part) strides over its group's rows, ``blockDim / G`` at a time.
// H16: x, delta and n are 16-bit; a row is then half the bytes of an f32 one,
// too few in flight to fill the memory's pipe, so each row is asked for while
// the one before it is worked on (128 x 196 x 512: forward 34 -> 21 us, backward
// 62 -> 48).
template <int V, int G, int NV, bool DELTA, bool NEXT, bool H16, bool RAG>
__global__ void __launch_bounds__(G > 256 ? G : 256) norm_fwd_kernel(const Args a) {
  constexpr int T = G > 256 ? G : 256, RB = T / G;
  extern __shared__ float4 dyn4[];
  float* kq = reinterpret_cast<float*>(dyn4);
  float* wn = kq + (DELTA ? factor_floats<V, RAG>(a.C) : 0);
  __shared__ float sh[G > 32 ? 2 * 32 : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const int64_t group = blockIdx.x / a.per_group;
  const int part = blockIdx.x % a.per_group;
  const int64_t row_end = min(a.rows, (group + 1) * a.group_rows);
  const int64_t stride = (int64_t)a.per_group * RB;
  int64_t r0 = group * a.group_rows + (int64_t)part * RB;
  // RAG: where this thread's rows start in a 16-byte unit (stride is a multiple of 8)
  const int shift = RAG ? (int)((r0 + sub) * a.C & 7) : 0;
  const int64_t total = a.rows * a.C;
  uint4 fx[NV], fd[NV];  // H16: the next row
  auto fetch_row = [&](int64_t row) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * V - shift;
      fx[j] = fd[j] = make_uint4(0, 0, 0, 0);
      if (row < row_end && c < a.C && (!RAG || c > -8)) {
        fx[j] = fetch8<RAG>(a.x, row * a.C + c, total);
        if constexpr (DELTA) fd[j] = fetch8<RAG>(a.delta, row * a.C + c, total);
      }
    }
  };
  if constexpr (H16) fetch_row(r0 + sub);
  load_factors<V, DELTA, NEXT, RAG>(a, group, kq, wn);
  for (; r0 < row_end; r0 += stride) {
    const int64_t row = r0 + sub;
    const bool live = row < row_end;
    const int64_t at = row * a.C;
    float x[NV][V], d[NV][V];
    if constexpr (H16) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        widen8(fx[j], a.x_dt, x[j]);
        mask<RAG>(x[j], (j * G + lane) * V - shift, a.C);
        if constexpr (DELTA) widen8(fd[j], a.d_dt, d[j]);
        mask<RAG>(d[j], (j * G + lane) * V - shift, a.C);
      }
      fetch_row(row + stride);
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * G + lane) * V - shift;
#pragma unroll
        for (int k = 0; k < V; ++k) x[j][k] = d[j][k] = 0.f;
        if (live && c < a.C && (!RAG || c > -8)) {
          load<RAG>(a.x, a.x_dt, at + c, total, c, a.C, x[j]);
          if constexpr (DELTA) load<RAG>(a.delta, a.d_dt, at + c, total, c, a.C, d[j]);
        }
      }
    }
    if constexpr (DELTA) {
      float s[1] = {0.f};
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) s[0] += d[j][k] * d[j][k];
      row_sum<G>(s, sh, turn);
      const float rd = rsqrtf(s[0] * a.inv_c + a.eps);
      if (live && lane == 0 && a.rd) a.rd[row] = rd;
      const float sc = rd * (a.scale && live ? a.scale[sample_of(a, row)] : 1.f);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * G + lane) * V - shift;
        if (!live || c >= a.C || (RAG && c <= -8)) continue;
        float w[V];
        factors<V, RAG>(kq, c, a.C, w);
#pragma unroll
        for (int k = 0; k < V; ++k) x[j][k] += sc * d[j][k] * w[k];
        store<RAG>(a.h, a.x_dt, at + c, c, a.C, x[j]);
      }
    }
    if constexpr (NEXT) {
      float s[1] = {0.f};
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) s[0] += x[j][k] * x[j][k];
      row_sum<G>(s, sh, turn);
      const float rh = rsqrtf(s[0] * a.inv_c + a.eps);
      if (live && lane == 0 && a.rh) a.rh[row] = rh;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * G + lane) * V - shift;
        if (!live || c >= a.C || (RAG && c <= -8)) continue;
        float w[V];
        factors<V, RAG>(wn, c, a.C, w);
#pragma unroll
        for (int k = 0; k < V; ++k) w[k] *= x[j][k] * rh;
        store<RAG>(a.n, a.n_dt, at + c, c, a.C, w);
      }
    }
  }
}

// Block (group, part) strides over its group's rows; ``part`` gets its sums.
template <int V, int G, int NV, bool DELTA, bool NEXT, bool H16, bool RAG>
__global__ void __launch_bounds__(G > 256 ? G : 256, G == 512 && !H16 ? 2 : 0) norm_bwd_kernel(const Args a) {
  constexpr int T = G > 256 ? G : 256, RB = T / G;
  extern __shared__ float4 dyn4[];  // the channel factors, later the sums of the block's row groups
  float* kq = reinterpret_cast<float*>(dyn4);
  float* wn = kq + (DELTA ? factor_floats<V, RAG>(a.C) : 0);
  __shared__ float sh[G > 32 ? 2 * 3 * 32 : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const int64_t group = blockIdx.x / a.per_group;
  const int part = blockIdx.x % a.per_group;
  const int64_t row_end = min(a.rows, (group + 1) * a.group_rows);
  const int64_t stride = (int64_t)a.per_group * RB;
  int64_t r0 = group * a.group_rows + (int64_t)part * RB;
  // RAG: where this thread's rows start in a 16-byte unit (stride is a multiple of 8)
  const int shift = RAG ? (int)((r0 + sub) * a.C & 7) : 0;
  const int64_t total = a.rows * a.C;
  uint4 fx[NV], fd[NV], fh[NV], fn[NV];  // H16: the next row
  float fr[2];
  auto fetch_row = [&](int64_t row) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * V - shift;
      fx[j] = fd[j] = fh[j] = fn[j] = make_uint4(0, 0, 0, 0);
      if (row < row_end && c < a.C && (!RAG || c > -8)) {
        const int64_t i = row * a.C + c;
        if constexpr (NEXT) {
          fx[j] = fetch8<RAG>(a.x, i, total);
          fn[j] = fetch8<RAG>(a.dn, i, total);
        }
        if constexpr (DELTA) {
          fd[j] = fetch8<RAG>(a.delta, i, total);
          if (a.dh) fh[j] = fetch8<RAG>(a.dh, i, total);
        }
      }
    }
    fr[0] = DELTA && row < row_end ? a.rd[row] : 0.f;
    fr[1] = NEXT && row < row_end ? a.rh[row] : 0.f;
  };
  if constexpr (H16) fetch_row(r0 + sub);
  load_factors<V, DELTA, NEXT, RAG>(a, group, kq, wn);
  float an[NV][V], at_[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < V; ++k) an[j][k] = at_[j][k] = 0.f;

  for (; r0 < row_end; r0 += stride) {
    const int64_t row = r0 + sub;
    const bool live = row < row_end;
    const int64_t at = row * a.C;
    float x[NV][V], d[NV][V], gh[NV][V], gn[NV][V];
    float rd, rh;
    if constexpr (H16) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        widen8(fx[j], a.x_dt, x[j]);
        mask<RAG>(x[j], (j * G + lane) * V - shift, a.C);
        widen8(fd[j], a.d_dt, d[j]);
        mask<RAG>(d[j], (j * G + lane) * V - shift, a.C);
        widen8(fh[j], a.x_dt, gh[j]);
        mask<RAG>(gh[j], (j * G + lane) * V - shift, a.C);
        widen8(fn[j], a.n_dt, gn[j]);
        mask<RAG>(gn[j], (j * G + lane) * V - shift, a.C);
      }
      rd = fr[0];
      rh = fr[1];
      fetch_row(row + stride);
    } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * V - shift;
#pragma unroll
      for (int k = 0; k < V; ++k) x[j][k] = d[j][k] = gh[j][k] = gn[j][k] = 0.f;
      if (live && c < a.C && (!RAG || c > -8)) {
        if constexpr (NEXT) {
          load<RAG>(a.x, a.x_dt, at + c, total, c, a.C, x[j]);
          load<RAG>(a.dn, a.n_dt, at + c, total, c, a.C, gn[j]);
        }
        if constexpr (DELTA) load<RAG>(a.delta, a.d_dt, at + c, total, c, a.C, d[j]);
        if (DELTA && a.dh) load<RAG>(a.dh, a.x_dt, at + c, total, c, a.C, gh[j]);
      }
    }
    rd = DELTA && live ? a.rd[row] : 0.f;
    rh = NEXT && live ? a.rh[row] : 0.f;
    }
    const float sc = DELTA && a.scale && live ? a.scale[sample_of(a, row)] : 1.f;
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * V - shift;
      if (!live || c >= a.C || (RAG && c <= -8)) continue;
      float wp[V], w[V];
      if constexpr (DELTA) factors<V, RAG>(kq, c, a.C, wp);
      if constexpr (NEXT) factors<V, RAG>(wn, c, a.C, w);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float e = 0.f;
        if constexpr (DELTA) {
          d[j][k] *= rd;                 // d^
          e = sc * wp[k] * d[j][k];      // h - x
        }
        if constexpr (NEXT) {
          x[j][k] = (x[j][k] + e) * rh;  // h^
          const float u = gn[j][k] * w[k];
          an[j][k] += gn[j][k] * x[j][k];
          s[0] += u * x[j][k];
          if constexpr (DELTA) s[2] += e * x[j][k];
          gh[j][k] += rh * u;
        }
        if constexpr (DELTA) s[1] += e * gh[j][k];
      }
    }
    row_sum<G>(s, sh, turn);
    const float mu = s[0] * a.inv_c * rh;              // r_h mean(u h^)
    const float me = (s[1] - s[2] * mu) * a.inv_c;     // mean(e d^)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * V - shift;
      if (!live || c >= a.C || (RAG && c <= -8)) continue;
      float o[V], wp[V];
      if constexpr (DELTA) factors<V, RAG>(kq, c, a.C, wp);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float D = NEXT ? gh[j][k] - x[j][k] * mu : gh[j][k];
        gh[j][k] = D;
        if constexpr (DELTA) {
          at_[j][k] += sc * D * d[j][k];
          o[k] = rd * (sc * wp[k] * D - d[j][k] * me);
        }
      }
      store<RAG>(a.dx, a.x_dt, at + c, c, a.C, gh[j]);
      if constexpr (DELTA) store<RAG>(a.ddelta, a.d_dt, at + c, c, a.C, o);
    }
  }

  float* out = a.part + (int64_t)blockIdx.x * a.arrays * a.C;
  float* dyn = reinterpret_cast<float*>(dyn4);
  auto leave = [&](float (&v)[NV][V], int which) {
    float* to = out + (int64_t)which * a.C;
    if constexpr (RB > 1) {  // add the block's row groups in order
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const int c = (j * G + lane) * V - shift + k;
          if (c < a.C && (!RAG || c >= 0)) dyn[sub * a.C + c] = v[j][k];
        }
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += T) {
        float t = 0.f;
        for (int i = 0; i < RB; ++i) t += dyn[i * a.C + c];
        to[c] = t;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * G + lane) * V - shift;
        if (c < a.C && (!RAG || c > -8)) {
          if constexpr (RAG) store_each(to, c, a.C, v[j]);
          else stv<V>(to, OW_DTYPE_F32, c, v[j]);
        }
      }
    }
  };
  int which = 0;
  if constexpr (NEXT) leave(an, which++);
  if constexpr (DELTA) leave(at_, which++);
}

// Rows longer than the kernels above hold: one block a row, read again for
// each pass.  part is added by the same second kernel.
template <bool DELTA, bool NEXT>
__global__ void __launch_bounds__(256) norm_long_fwd_kernel(const Args a) {
  __shared__ float sh[2 * 32];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t at = row * a.C, b = row / a.tokens;
    float rd = 0.f;
    if constexpr (DELTA) {
      float s[1] = {0.f};
      for (int c = threadIdx.x; c < a.C; c += 256) {
        const float d = ld1(a.delta, a.d_dt, at + c);
        s[0] += d * d;
      }
      row_sum<256>(s, sh, turn);
      rd = rsqrtf(s[0] * a.inv_c + a.eps);
      if (threadIdx.x == 0 && a.rd) a.rd[row] = rd;
    }
    const float sc = DELTA ? rd * (a.scale ? a.scale[b] : 1.f) : 0.f;
    auto hval = [&](int c) {
      float h = ld1(a.x, a.x_dt, at + c);
      if constexpr (DELTA) {
        float w = ld1(a.wp, a.wp_dt, c);
        if (a.q_rows) w *= ld1(a.q, a.q_dt, (a.q_rows > 1 ? b * a.C : 0) + c);
        h += sc * ld1(a.delta, a.d_dt, at + c) * w;
      }
      return h;
    };
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float h[1] = {hval(c)};
      s[0] += h[0] * h[0];
      if constexpr (DELTA) stv<1>(a.h, a.x_dt, at + c, h);
    }
    if constexpr (NEXT) {
      row_sum<256>(s, sh, turn);
      const float rh = rsqrtf(s[0] * a.inv_c + a.eps);
      if (threadIdx.x == 0 && a.rh) a.rh[row] = rh;
      for (int c = threadIdx.x; c < a.C; c += 256) {
        const float o[1] = {hval(c) * rh * ld1(a.wn, a.wn_dt, c)};
        stv<1>(a.n, a.n_dt, at + c, o);
      }
    }
  }
}

template <bool DELTA, bool NEXT>
__global__ void __launch_bounds__(256) norm_long_bwd_kernel(const Args a) {
  __shared__ float sh[2 * 3 * 32];
  int turn = 0;
  const int64_t group = blockIdx.x / a.per_group;
  const int part = blockIdx.x % a.per_group;
  const int64_t row_end = min(a.rows, (group + 1) * a.group_rows);
  float* out = a.part + (int64_t)blockIdx.x * a.arrays * a.C;
  for (int c = threadIdx.x; c < a.C; c += 256)
    for (int i = 0; i < a.arrays; ++i) out[(int64_t)i * a.C + c] = 0.f;  // each thread adds to its own channels only
  for (int64_t row = group * a.group_rows + part; row < row_end; row += a.per_group) {
    const int64_t at = row * a.C, b = row / a.tokens;
    const float rd = DELTA ? a.rd[row] : 0.f, rh = NEXT ? a.rh[row] : 0.f;
    const float sc = DELTA && a.scale ? a.scale[b] : 1.f;
    struct El { float d, e, q, wp, hh, g, gn; };
    auto el = [&](int c) {
      El r{};
      r.q = 1.f;
      if constexpr (DELTA) {
        r.d = ld1(a.delta, a.d_dt, at + c) * rd;
        r.wp = ld1(a.wp, a.wp_dt, c);
        if (a.q_rows) r.q = ld1(a.q, a.q_dt, (a.q_rows > 1 ? b * a.C : 0) + c);
        r.e = sc * r.q * r.wp * r.d;
      }
      r.g = a.dh ? ld1(a.dh, a.x_dt, at + c) : 0.f;
      if constexpr (NEXT) {
        r.hh = (ld1(a.x, a.x_dt, at + c) + r.e) * rh;
        r.gn = ld1(a.dn, a.n_dt, at + c);
      }
      return r;
    };
    float s[3] = {0.f, 0.f, 0.f};
    for (int c = threadIdx.x; c < a.C; c += 256) {
      El r = el(c);
      if constexpr (NEXT) {
        const float u = r.gn * ld1(a.wn, a.wn_dt, c);
        s[0] += u * r.hh;
        s[2] += r.e * r.hh;
        r.g += rh * u;
      }
      s[1] += r.e * r.g;
    }
    row_sum<256>(s, sh, turn);
    const float mu = s[0] * a.inv_c * rh, me = (s[1] - s[2] * mu) * a.inv_c;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const El r = el(c);
      float D[1] = {r.g};
      int which = 0;
      if constexpr (NEXT) {
        D[0] += rh * r.gn * ld1(a.wn, a.wn_dt, c) - r.hh * mu;
        out[c] += r.gn * r.hh;
        which = 1;
      }
      stv<1>(a.dx, a.x_dt, at + c, D);
      if constexpr (DELTA) {
        out[(int64_t)which * a.C + c] += sc * D[0] * r.d;
        const float o[1] = {rd * (sc * r.q * r.wp * D[0] - r.d * me)};
        stv<1>(a.ddelta, a.d_dt, at + c, o);
      }
    }
  }
}

// Column sums of the partial rows, 32 channels a block, 32 threads a channel,
// added in an order that the shape alone fixes.  blockIdx.y: 0 the next norm's
// gradient, 1 the post-norm's (sum over the groups of q t), 2 and on the
// groups' gates (wp t).  One chain of loads is what this kernel takes, so each thread
// has four of them in flight.
struct SumArgs {
  const float* part;
  int C, arrays, per_group, at_t;   // at_t: the array of t (-1: none)
  int64_t groups;
  const void* wp;
  const void* q;
  int q_rows, wp_dt, q_dt, wn_dt;
  int few;        // the groups have few parts: a thread adds up a group's
  int64_t ys;
  void* dnext;
  void* dpost;
  void* dgate;
};

__global__ void __launch_bounds__(1024) norm_sum_kernel(const SumArgs a) {
  __shared__ float sh[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  const int64_t ys = a.ys;
  for (int64_t y = blockIdx.y; y < ys; y += gridDim.y) {
    void* out = y == 0 ? a.dnext : y == 1 ? a.dpost : a.dgate;
    if (!out) continue;
    if (y >= 2 && a.few) {  // 32 groups at once, a thread each
      const int64_t g = (y - 2) * 32 + ry;
      if (c < a.C && g < a.groups) {
        float v[1] = {0.f};
        const float* p = a.part + (g * a.per_group * a.arrays + a.at_t) * a.C + c;
#pragma unroll 4
        for (int i = 0; i < a.per_group; ++i) v[0] += p[(int64_t)i * a.arrays * a.C];
        v[0] *= ld1(a.wp, a.wp_dt, c);
        stv<1>(out, a.q_dt, g * a.C + c, v);
      }
      continue;
    }
    const int64_t stride = (int64_t)a.arrays * a.C;
    const float* p = a.part + (y == 0 ? 0 : (int64_t)a.at_t * a.C) + c;
    int64_t n = a.groups * a.per_group;
    if (y >= 2) {
      p += (y - 2) * a.per_group * stride;
      n = a.per_group;
    }
    const bool weigh = y == 1 && a.q_rows > 1;
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.C)
      for (int64_t i = ry; i < n; i += 128) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int64_t r = i + 32 * k;
          if (r < n) t[k] += p[r * stride] * (weigh ? ld1(a.q, a.q_dt, r / a.per_group * a.C + c) : 1.f);
        }
      }
    __syncthreads();
    sh[ry][cx] = (t[0] + t[1]) + (t[2] + t[3]);
    __syncthreads();
    if (ry == 0 && c < a.C) {
      float v[1] = {0.f};
#pragma unroll
      for (int i = 0; i < 32; ++i) v[0] += sh[i][cx];
      if (y == 1 && a.q_rows == 1) v[0] *= ld1(a.q, a.q_dt, c);
      if (y >= 2) v[0] *= ld1(a.wp, a.wp_dt, c);
      stv<1>(out, y == 0 ? a.wn_dt : y == 1 ? a.wp_dt : a.q_dt, (y >= 2 ? (y - 2) * a.C : 0) + c, v);
    }
  }
}

bool float_type(int dt) { return dt == OW_DTYPE_F32 || dt == OW_DTYPE_BF16 || dt == OW_DTYPE_F16; }

int check(const ow_norm_t* a) {
  OW_CHECK_ARG(a != nullptr, "ow_norm: args is NULL");
  OW_CHECK_ARG(a->samples >= 0 && a->tokens >= 0 && a->channels > 0, "ow_norm: bad shape [%lld, %lld, %d]",
               (long long)a->samples, (long long)a->tokens, a->channels);
  OW_CHECK_ARG(a->samples < (1LL << 31) && a->tokens < (1LL << 31) && a->samples * a->tokens < (1LL << 40), "ow_norm: too many rows");
  OW_CHECK_ARG(a->channels < (1 << 30), "ow_norm: too many channels (%d)", a->channels);
  const bool d = a->delta != nullptr;
  OW_CHECK_ARG(a->x && (!d || a->post_w) && (d || a->next_w), "ow_norm: an input pointer is NULL");
  OW_CHECK_ARG(a->gate_rows == 0 || (d && a->gate && (a->gate_rows == 1 || a->gate_rows == a->samples)),
               "ow_norm: the gate must have 1 row or one for each sample (got %lld)", (long long)a->gate_rows);
  OW_CHECK_ARG(d || !a->sample_scale, "ow_norm: a residual scale needs delta");
  if (!float_type(a->x_dtype) || (d && (!float_type(a->delta_dtype) || !float_type(a->post_dtype))) ||
      (a->gate_rows && !float_type(a->gate_dtype)) || (a->next_w && (!float_type(a->next_dtype) || !float_type(a->n_dtype)))) {
    set_error("ow_norm: dtypes must be float32, bfloat16 or float16");
    return OW_ERR_UNSUPPORTED;
  }
  OW_CHECK_ARG(a->eps >= 0.0, "ow_norm: eps must not be negative");
  auto at = [](const void* p, int dt) { return (uintptr_t)p % dtype_size(dt) == 0; };
  OW_CHECK_ARG(at(a->x, a->x_dtype) && (!d || (at(a->delta, a->delta_dtype) && at(a->post_w, a->post_dtype) && at(a->h, a->x_dtype))) &&
                   (!a->gate_rows || at(a->gate, a->gate_dtype)) &&
                   (!a->next_w || (at(a->next_w, a->next_dtype) && at(a->n, a->n_dtype))) &&
                   ((uintptr_t)a->sample_scale | (uintptr_t)a->rstd_delta | (uintptr_t)a->rstd_h) % 4 == 0,
               "ow_norm: a tensor is not aligned");
  return OW_OK;
}

Args base(const ow_norm_t* a) {
  Args k{};
  k.rows = a->samples * a->tokens;
  k.tokens = a->tokens;
  k.C = a->channels;
  k.x = a->x; k.delta = a->delta;
  k.wp = a->post_w; k.q = a->gate; k.wn = a->next_w;
  k.x_dt = a->x_dtype; k.d_dt = a->delta_dtype;
  k.wp_dt = a->post_dtype; k.q_dt = a->gate_dtype; k.wn_dt = a->next_dtype; k.n_dt = a->n_dtype;
  k.q_rows = a->gate_rows > 1 ? 2 : (int)a->gate_rows;
  k.scale = a->sample_scale;
  k.eps = (float)a->eps;
  k.inv_c = 1.f / (float)a->channels;
  k.rd = a->rstd_delta; k.rh = a->rstd_h;
  return k;
}

bool all16(const Args& k, bool delta, bool next) {
  return k.x_dt != OW_DTYPE_F32 && (!delta || k.d_dt != OW_DTYPE_F32) && (!next || k.n_dt != OW_DTYPE_F32);
}

constexpr int LONG_V = 8192, LONG_1 = 1024;  // channels a row may have in the register kernels

// Whether the rows are moved in aligned units of 8 channels: every array of
// rows starts on 16 bytes (the channels' vectors are read one by one), and, for
// ragged rows, it pays: it does for 16-bit arrays (100 channels: forward 75 us
// against 100 element by element, with the backward 218 against 439), and not for
// f32 alone (777: 90 against 74).  With f32 arrays beside 16-bit ones the backward
// gains and the forward loses; 112 channels is where training gains (20 M elements,
// f32 stream, forward and with the backward, in units and by elements: 92 channels
// 143, 314 and 75, 300; 108 123, 273 and 79, 310; 116 118, 258 and 76, 313; 150 162,
// 355 and 152, 563; 204 116, 259 and 127, 482).  Between 122 and 128, whose units
// take a split for 256 channels, elements would be better in both (124: 178, 398
// and 73, 298).
bool units(const Args& k, bool delta, bool next, const void* const* more, int n) {
  if ((uintptr_t)k.x % 16 || (uintptr_t)k.delta % 16) return false;
  for (int i = 0; i < n; ++i)
    if ((uintptr_t)more[i] % 16) return false;
  if (k.C % 8 == 0 || k.C > LONG_1 || all16(k, delta, next)) return true;
  const bool all32 = k.x_dt == OW_DTYPE_F32 && (!delta || k.d_dt == OW_DTYPE_F32) && (!next || k.n_dt == OW_DTYPE_F32);
  return !all32 && k.C > 112;
}


// Calls f<V, G, NV> with the split of a row of C channels.
template <class F>
int split_fwd(int C, bool vec, F&& f) {
#define OW_SPLIT(V, G, NV) return f(std::integral_constant<int, V>(), std::integral_constant<int, G>(), std::integral_constant<int, NV>())
  if (vec) {
    if (C <= 64) OW_SPLIT(8, 8, 1);
    if (C <= 128) OW_SPLIT(8, 16, 1);
    if (C <= 256) OW_SPLIT(8, 32, 1);
    if (C <= 512) OW_SPLIT(8, 32, 2);
    if (C <= 1024) OW_SPLIT(8, 128, 1);
    if (C <= 2048) OW_SPLIT(8, 256, 1);
    if (C <= 4096) OW_SPLIT(8, 256, 2);
    OW_SPLIT(8, 256, 4);
  }
  if (C <= 128) OW_SPLIT(1, 32, 4);
  if (C <= 512) OW_SPLIT(1, 128, 4);
  OW_SPLIT(1, 256, 4);
}

template <class F>
int split_bwd(int C, bool vec, F&& f) {
  if (vec) {
    if (C <= 64) OW_SPLIT(8, 8, 1);
    if (C <= 128) OW_SPLIT(8, 16, 1);
    if (C <= 256) OW_SPLIT(8, 32, 1);
    if (C <= 512) OW_SPLIT(8, 64, 1);
    if (C <= 1024) OW_SPLIT(8, 128, 1);
    if (C <= 2048) OW_SPLIT(8, 256, 1);
    if (C <= 4096) OW_SPLIT(8, 512, 1);
    OW_SPLIT(8, 1024, 1);
  }
  if (C <= 128) OW_SPLIT(1, 32, 4);
  if (C <= 512) OW_SPLIT(1, 128, 4);
  OW_SPLIT(1, 256, 4);
#undef OW_SPLIT
}

bool ragged(int C, bool vec) { return vec && C % 8 != 0; }
// channels that a row's threads must have room for
int room(int C, bool vec) { return ragged(C, vec) ? C + 7 : C; }
bool too_long(int C, bool vec) { return room(C, vec) > (vec ? LONG_V : LONG_1); }

// Blocks of a group for ragged rows: a block's rows ``parts`` x RB apart start
// alike when that is a multiple of 8.  Fewer blocks than that makes do when each
// takes its rows at once and has none further on.
int alike(int parts, int RB, int64_t rows) {
  const int m = RB >= 8 ? 1 : 8 / RB;
  if (parts < m && (int64_t)parts * RB >= rows) return parts;
  return std::max(m, parts / m * m);
}

int reserve(const void* kern, size_t smem) {
  if (smem <= 48 * 1024) return OW_OK;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) {
    set_error("ow_norm: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    return OW_ERR_CUDA;
  }
  return OW_OK;
}

template <class F>
int modes(bool delta, bool next, F&& f) {
  if (delta) return next ? f(std::true_type(), std::true_type()) : f(std::true_type(), std::false_type());
  return f(std::false_type(), std::true_type());
}

// The blocks: at most ``per_sm`` an SM, no more than there are rows, shared out
// over the groups of rows with a gate of their own.
void parts(const ow_norm_t* a, Args* k, int per_sm) {
  k->groups = a->gate_rows > 1 ? a->samples : 1;
  k->group_rows = k->rows / std::max<int64_t>(k->groups, 1);
  const int64_t want = (int64_t)device_sm_count() * per_sm;
  const int64_t per = std::max<int64_t>(1, want / std::max<int64_t>(k->groups, 1));
  k->per_group = (int)std::max<int64_t>(1, std::min<int64_t>(per, k->group_rows));
  k->arrays = (a->next_w ? 1 : 0) + (a->delta ? 1 : 0);
}

// Blocks an SM runs at once, by the registers of the kernels' threads (40 to 128
// forward, 80 to 121 backward): more would make a second, half empty wave.
constexpr int FWD_PER_SM = 6, BWD_PER_SM = 3;
constexpr int fwd_per_sm(int nv, bool h16, bool rag) {
  return rag ? (nv == 1 ? 4 : 2) : nv == 1 ? (h16 ? 5 : 6) : nv == 2 ? (h16 ? 3 : 4) : (h16 ? 2 : 3);
}
constexpr int bwd_per_sm(int T, bool h16) { return T > 512 ? 1 : T > 256 ? (h16 ? 1 : 2) : h16 ? 2 : 3; }
// With 1024 threads a row to come does not fit in their 64 registers.
constexpr bool bwd_ahead(int V, int T) { return V == 8 && T <= 512; }

// The blocks of the backward, rows moved in units or not, and with them the rows of its partial sums.
void bwd_parts(const ow_norm_t* a, Args* k, bool vec) {
  parts(a, k, BWD_PER_SM);
  if (too_long(k->C, vec)) return;
  split_bwd(room(k->C, vec), vec, [&](auto V, auto G, auto) -> int {
    constexpr int T = G.value > 256 ? G.value : 256, RB = T / G.value;
    parts(a, k, bwd_per_sm(T, bwd_ahead(V.value, T) && all16(*k, a->delta, a->next_w)));
    k->per_group = (int)std::min<int64_t>(k->per_group, std::max<int64_t>(1, (k->group_rows + RB - 1) / RB));
    if (ragged(k->C, vec)) k->per_group = alike(k->per_group, RB, k->group_rows);
    return OW_OK;
  });
}

}  // namespace
}  // namespace ow

using namespace ow;

extern "C" {

size_t ow_norm_bwd_workspace_size(const ow_norm_t* a) {
  clear_error();
  if (check(a) != OW_OK) return 0;
  Args k = base(a);
  // whether the rows are moved in units depends on the gradients' addresses too
  bwd_parts(a, &k, false);
  const int others = k.per_group;
  bwd_parts(a, &k, true);
  return (size_t)k.groups * std::max(k.per_group, others) * k.arrays * k.C * sizeof(float) + 256;
}

int ow_norm_fwd(const ow_norm_t* a, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  Args k = base(a);
  if (k.rows == 0) return OW_OK;
  const bool delta = a->delta, next = a->next_w;
  OW_CHECK_ARG((!delta || a->h) && (!next || a->n), "ow_norm_fwd: an output pointer is NULL");
  k.h = a->h;
  k.n = a->n;
  const void* outs[] = {k.h, k.n};
  const bool vec = units(k, delta, next, outs, 2), rag = ragged(k.C, vec);
  const cudaStream_t st = (cudaStream_t)stream;
  parts(a, &k, FWD_PER_SM);
  return modes(delta, next, [&](auto D, auto N) -> int {
    if (too_long(k.C, vec)) {
      const int64_t grid = std::min<int64_t>(k.rows, (int64_t)device_sm_count() * FWD_PER_SM);
      launch(norm_long_fwd_kernel<D.value, N.value>, (int)grid, 256, 0, st, k);
    } else {
      OW_RETURN_IF(split_fwd(room(k.C, vec), vec, [&](auto V, auto G, auto NV) -> int {
        constexpr int T = G.value > 256 ? G.value : 256, RB = T / G.value;
        const bool h16 = V.value == 8 && all16(k, D.value, N.value);
        parts(a, &k, V.value == 8 ? fwd_per_sm(NV.value, h16, rag) : FWD_PER_SM);
        k.per_group = (int)std::min<int64_t>(k.per_group, (k.group_rows + RB - 1) / RB);
        if (rag) k.per_group = alike(k.per_group, RB, k.group_rows);
        OW_CHECK_ARG(k.groups * k.per_group < (1LL << 31), "ow_norm_fwd: too many samples");
        const size_t smem = (size_t)(rag ? factor_floats<8, true>(k.C) : k.C) * sizeof(float) * (D.value + N.value);
        auto go = [&](auto kern) -> int {
          OW_RETURN_IF(reserve((const void*)kern, smem));
          launch(kern, (int)(k.groups * k.per_group), T, smem, st, k);
          return OW_OK;
        };
        if constexpr (V.value == 8) {
          if (rag)
            return h16 ? go(norm_fwd_kernel<8, G.value, NV.value, D.value, N.value, true, true>)
                       : go(norm_fwd_kernel<8, G.value, NV.value, D.value, N.value, false, true>);
          if (h16) return go(norm_fwd_kernel<8, G.value, NV.value, D.value, N.value, true, false>);
        }
        return go(norm_fwd_kernel<V.value, G.value, NV.value, D.value, N.value, false, false>);
      }));
    }
    OW_CHECK_LAUNCH("norm_fwd_kernel");
    return OW_OK;
  });
}

int ow_norm_bwd(const ow_norm_t* a, const ow_norm_grads_t* g, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  const bool delta = a->delta, next = a->next_w;
  OW_CHECK_ARG(g != nullptr, "ow_norm_bwd: grads is NULL");
  Args k = base(a);
  OW_CHECK_ARG(k.rows == 0 || (g->dx && (!next || g->dn) && (!delta || g->ddelta) && (g->dh || next) &&
                               (!delta || k.rd) && (!next || k.rh)),
               "ow_norm_bwd: a pointer is NULL");
  auto at = [](const void* p, int dt) { return !p || (uintptr_t)p % dtype_size(dt) == 0; };
  OW_CHECK_ARG(at(g->dh, a->x_dtype) && at(g->dx, a->x_dtype) && (!next || (at(g->dn, a->n_dtype) && at(g->dnext, a->next_dtype))) &&
                   (!delta || (at(g->ddelta, a->delta_dtype) && at(g->dpost, a->post_dtype))) &&
                   (!a->gate_rows || at(g->dgate, a->gate_dtype)),
               "ow_norm_bwd: a gradient is not aligned");
  const size_t need = ow_norm_bwd_workspace_size(a);
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("ow_norm_bwd needs %zu workspace bytes, got %zu", need, a->workspace_bytes);
    return OW_ERR_WORKSPACE;
  }
  k.dh = g->dh; k.dn = g->dn; k.dx = g->dx; k.ddelta = g->ddelta;
  k.part = (float*)(((uintptr_t)a->workspace + 255) & ~(uintptr_t)255);
  const void* more[] = {k.dh, k.dn, k.dx, k.ddelta};
  const bool vec = units(k, delta, next, more, 4), rag = ragged(k.C, vec);
  const cudaStream_t st = (cudaStream_t)stream;
  bwd_parts(a, &k, vec);
  const int64_t grid = k.groups * k.per_group;
  OW_CHECK_ARG(grid < (1LL << 31), "ow_norm_bwd: too many samples");
  if (grid > 0) OW_RETURN_IF(modes(delta, next, [&](auto D, auto N) -> int {
    if (too_long(k.C, vec)) {
      launch(norm_long_bwd_kernel<D.value, N.value>, (int)grid, 256, 0, st, k);
    } else {
      OW_RETURN_IF(split_bwd(room(k.C, vec), vec, [&](auto V, auto G, auto NV) -> int {
        constexpr int T = G.value > 256 ? G.value : 256, RB = T / G.value;
        constexpr bool AHEAD = bwd_ahead(V.value, T);
        const bool h16 = AHEAD && all16(k, D.value, N.value);
        const size_t smem = sizeof(float) * std::max<size_t>((size_t)(rag ? factor_floats<8, true>(k.C) : k.C) * (D.value + N.value),
                                                             RB > 1 ? (size_t)RB * k.C : 0);
        auto go = [&](auto kern) -> int {
          OW_RETURN_IF(reserve((const void*)kern, smem));
          launch(kern, (int)grid, T, smem, st, k);
          return OW_OK;
        };
        if constexpr (AHEAD) {
          if (h16)
            return rag ? go(norm_bwd_kernel<8, G.value, NV.value, D.value, N.value, true, true>)
                       : go(norm_bwd_kernel<8, G.value, NV.value, D.value, N.value, true, false>);
        }
        if constexpr (V.value == 8)
          if (rag) return go(norm_bwd_kernel<8, G.value, NV.value, D.value, N.value, false, true>);
        return go(norm_bwd_kernel<V.value, G.value, NV.value, D.value, N.value, false, false>);
      }));
    }
    OW_CHECK_LAUNCH("norm_bwd_kernel");
    return OW_OK;
  }));
  SumArgs s{};
  s.part = k.part; s.C = k.C; s.arrays = k.arrays; s.per_group = k.per_group; s.groups = k.groups;
  s.at_t = delta ? (next ? 1 : 0) : -1;
  s.wp = k.wp; s.q = k.q; s.q_rows = k.q_rows;
  s.wp_dt = k.wp_dt; s.q_dt = k.q_dt; s.wn_dt = k.wn_dt;
  s.dnext = next ? g->dnext : nullptr;
  s.dpost = delta ? g->dpost : nullptr;
  s.dgate = a->gate_rows ? g->dgate : nullptr;
  s.few = s.per_group <= 16;
  s.ys = s.at_t < 0 ? 1 : 2 + (!s.q_rows ? 0 : s.few ? (s.groups + 31) / 32 : s.groups);
  launch(norm_sum_kernel, dim3((k.C + 31) / 32, (unsigned)std::min<int64_t>(s.ys, 32768)), 1024, 0, st, s);
  OW_CHECK_LAUNCH("norm_sum_kernel");
  return OW_OK;
}

}  // extern "C"
