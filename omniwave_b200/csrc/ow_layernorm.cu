// Layer norm, forward and backward, with the gradients of weight and bias.
//
// A row is one token's C channels, all arithmetic in f32:
//   m = mean(x);  r = rsqrt(mean((x - m)^2) + eps);  x^ = (x - m) r;  n = x^ w + b
// Backward, from dn:
//   u = dn w;  dx = r (u - mean(u) - x^ mean(u x^));  dw = sum dn x^;  db = sum dn
// The squares are taken around the mean, from the row in registers: a sum of x^2
// less the mean's square loses the variance of rows that lie far from zero.
//
// G threads share a row, a thread E of its channels.  A thread meets the same
// channels in all its rows, so weight and bias stay in registers, and so do its
// shares of dw and db; a block leaves one partial row of each and a second kernel
// adds these in a fixed order.
//
// Many rows: a team of threads (a row's, or a warp where rows are shorter) works on
// its own and has its rows in chunks, which bulk copies bring to a ring of its own in
// shared memory some chunks ahead.  What is in flight then does not hang on
// registers, and a row may lie across few threads: E is 16 to 32, so that a row's two
// exchanges and the arithmetic, in pairs (f32x2), take few instructions an element.
// Few rows, and types or addresses that the copies do not take: straight from
// global memory, a row over as many threads as it has vectors.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "ow_common.cuh"
#include "ow_internal.h"
#include "ow_rows.cuh"
#include "ow_sm100.cuh"

namespace ow {
namespace {

struct Args {
  int64_t rows;
  int C;
  const void* x;
  const void* w;
  const void* b;     // or NULL
  const void* dn;
  int x_dt, w_dt, b_dt, n_dt;
  float eps, inv_c;
  void* n;
  float* mean;       // [rows], or NULL where nothing is kept
  float* rstd;
  void* dx;          // or NULL
  float* part;       // [blocks][2][C] sums of dn x^ and of dn, or NULL
};

// Threads of a block for rows of G threads.
constexpr int threads_of(int G) { return G > 256 ? G : 256; }

// The channel of a thread's element e.
template <int V, int G>
__device__ __forceinline__ int channel(int e, int lane) {
  if constexpr (V == 8) return ((e >> 3) * G + lane) * 8 + (e & 7);
  else return e * G + lane;
}

// A thread's share of a row (or of a vector of channels); 0 beside the channels.
template <int V, int G, int NV>
__device__ __forceinline__ void take(const void* p, int dt, int64_t at, int C, int lane, bool live, float (&o)[8 * NV]) {
#pragma unroll
  for (int j = 0; j < 8 * NV / V; ++j) {
    const int c = channel<V, G>(j * V, lane);
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.f;
    if (live && c < C) ldv<V>(p, dt, at + c, v);
#pragma unroll
    for (int k = 0; k < V; ++k) o[j * V + k] = v[k];
  }
}
template <int V, int G, int NV>
__device__ __forceinline__ void give(void* p, int dt, int64_t at, int C, int lane, const float (&o)[8 * NV]) {
#pragma unroll
  for (int j = 0; j < 8 * NV / V; ++j) {
    const int c = channel<V, G>(j * V, lane);
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = o[j * V + k];
    if (c < C) stv<V>(p, dt, at + c, v);
  }
}

template <int V, int G, int NV>
__global__ void __launch_bounds__(threads_of(G)) layernorm_fwd_kernel(const Args a) {
  constexpr int T = threads_of(G), RB = T / G, E = 8 * NV;
  __shared__ float sh[G > 32 ? 2 * 32 : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  float w[E], b[E];
  take<V, G, NV>(a.w, a.w_dt, 0, a.C, lane, true, w);
  take<V, G, NV>(a.b, a.b_dt, 0, a.C, lane, a.b != nullptr, b);
  for (int64_t r0 = (int64_t)blockIdx.x * RB; r0 < a.rows; r0 += (int64_t)gridDim.x * RB) {
    const int64_t row = r0 + sub;
    const bool live = row < a.rows;
    float x[E], s[1] = {0.f};
    take<V, G, NV>(a.x, a.x_dt, row * a.C, a.C, lane, live, x);
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += x[e];
    row_sum<G>(s, sh, turn);
    const float mean = s[0] * a.inv_c;
    s[0] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[e] -= mean;
      if (channel<V, G>(e, lane) < a.C) s[0] += x[e] * x[e];
    }
    row_sum<G>(s, sh, turn);
    const float r = rsqrtf(s[0] * a.inv_c + a.eps);
    if (!live) continue;
    if (lane == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = r;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] * r * w[e] + b[e];
    give<V, G, NV>(a.n, a.n_dt, row * a.C, a.C, lane, x);
  }
}

template <int V, int G, int NV>
__global__ void __launch_bounds__(threads_of(G)) layernorm_bwd_kernel(const Args a) {
  constexpr int T = threads_of(G), RB = T / G, E = 8 * NV;
  extern __shared__ float dyn[];  // [RB][C]: the block's row groups meet
  __shared__ float sh[G > 32 ? 2 * 2 * 32 : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  float w[E], dw[E], db[E];
  take<V, G, NV>(a.w, a.w_dt, 0, a.C, lane, true, w);
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
  for (int64_t r0 = (int64_t)blockIdx.x * RB; r0 < a.rows; r0 += (int64_t)gridDim.x * RB) {
    const int64_t row = r0 + sub;
    const bool live = row < a.rows;
    float x[E], g[E], s[2] = {0.f, 0.f};
    take<V, G, NV>(a.x, a.x_dt, row * a.C, a.C, lane, live, x);
    take<V, G, NV>(a.dn, a.n_dt, row * a.C, a.C, lane, live, g);
    const float mean = live ? a.mean[row] : 0.f, r = live ? a.rstd[row] : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[e] = channel<V, G>(e, lane) < a.C ? (x[e] - mean) * r : 0.f;  // x^
      dw[e] += g[e] * x[e];
      db[e] += g[e];
      g[e] *= w[e];                                                   // u
      s[0] += g[e];
      s[1] += g[e] * x[e];
    }
    row_sum<G>(s, sh, turn);
    if (!live || !a.dx) continue;
    const float mu = s[0] * a.inv_c, mx = s[1] * a.inv_c;
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = r * (g[e] - mu - x[e] * mx);
    give<V, G, NV>(a.dx, a.x_dt, row * a.C, a.C, lane, g);
  }
  if (!a.part) return;
  auto leave = [&](const float (&v)[E], int which) {
    float* to = a.part + ((int64_t)blockIdx.x * 2 + which) * a.C;
    if constexpr (RB > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (channel<V, G>(e, lane) < a.C) dyn[sub * a.C + channel<V, G>(e, lane)] = v[e];
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += T) {
        float t = 0.f;
        for (int i = 0; i < RB; ++i) t += dyn[i * a.C + c];
        to[c] = t;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (channel<V, G>(e, lane) < a.C) to[channel<V, G>(e, lane)] = v[e];
    }
  };
  leave(dw, 0);
  leave(db, 1);
}

// Rows longer than the kernels above hold: one block a row, read again for each
// pass.  The partial sums are added by the same second kernel.
__global__ void __launch_bounds__(256) layernorm_long_fwd_kernel(const Args a) {
  __shared__ float sh[2 * 32];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t at = row * a.C;
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < a.C; c += 256) s[0] += ld1(a.x, a.x_dt, at + c);
    row_sum<256>(s, sh, turn);
    const float mean = s[0] * a.inv_c;
    s[0] = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float d = ld1(a.x, a.x_dt, at + c) - mean;
      s[0] += d * d;
    }
    row_sum<256>(s, sh, turn);
    const float r = rsqrtf(s[0] * a.inv_c + a.eps);
    if (threadIdx.x == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = r;
    }
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float o[1] = {(ld1(a.x, a.x_dt, at + c) - mean) * r * ld1(a.w, a.w_dt, c) + (a.b ? ld1(a.b, a.b_dt, c) : 0.f)};
      stv<1>(a.n, a.n_dt, at + c, o);
    }
  }
}

__global__ void __launch_bounds__(256) layernorm_long_bwd_kernel(const Args a) {
  __shared__ float sh[2 * 2 * 32];
  int turn = 0;
  float* out = a.part ? a.part + (int64_t)blockIdx.x * 2 * a.C : nullptr;
  if (out)
    for (int c = threadIdx.x; c < 2 * a.C; c += 256) out[c] = 0.f;
  __syncthreads();
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t at = row * a.C;
    const float mean = a.mean[row], r = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float u = ld1(a.dn, a.n_dt, at + c) * ld1(a.w, a.w_dt, c);
      s[0] += u;
      s[1] += u * (ld1(a.x, a.x_dt, at + c) - mean) * r;
    }
    row_sum<256>(s, sh, turn);
    const float mu = s[0] * a.inv_c, mx = s[1] * a.inv_c;
    for (int c = threadIdx.x; c < a.C; c += 256) {  // each thread adds to its own channels only
      const float g = ld1(a.dn, a.n_dt, at + c), hat = (ld1(a.x, a.x_dt, at + c) - mean) * r;
      if (out) {
        out[c] += g * hat;
        out[a.C + c] += g;
      }
      const float o[1] = {r * (g * ld1(a.w, a.w_dt, c) - mu - hat * mx)};
      if (a.dx) stv<1>(a.dx, a.x_dt, at + c, o);
    }
  }
}

// Column sums of the partial rows, in an order that the shape alone fixes: 32
// channels a block, 32 threads a channel, each with four loads in flight.
// blockIdx.y: the weight's, the bias's.
__global__ void __launch_bounds__(1024) layernorm_sum_kernel(const float* __restrict__ part, int blocks, int C, void* dw, int w_dt,
                                                             void* db, int b_dt) {
  __shared__ float sh[32][33];
  void* out = blockIdx.y == 0 ? dw : db;
  if (!out) return;
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
  const float* p = part + (int64_t)blockIdx.y * C + c;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < C)
    for (int i = ry; i < blocks; i += 128) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + 32 * k < blocks) t[k] += p[(int64_t)(i + 32 * k) * 2 * C];
    }
  sh[ry][cx] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
  if (ry == 0 && c < C) {
    float v[1] = {0.f};
#pragma unroll
    for (int i = 0; i < 32; ++i) v[0] += sh[i][cx];
    stv<1>(out, blockIdx.y == 0 ? w_dt : b_dt, c, v);
  }
}

// ---------------------------------------------------------------- many rows
using f2 = uint64_t;  // two floats
__device__ __forceinline__ f2 both(float v) { return sm100::f2pack(v, v); }

// Two neighbouring elements of storage type T, and back.
template <typename T>
__device__ __forceinline__ f2 widen2(uint32_t lo, uint32_t hi) {
  if constexpr (sizeof(T) == 4) return (f2)lo | (f2)hi << 32;
  const float2 f = sm100::unpack2<std::is_same_v<T, __nv_bfloat16>>(lo);
  return sm100::f2pack(f.x, f.y);
}
template <typename T>
__device__ __forceinline__ uint32_t narrow2(f2 v) {
  const float2 f = sm100::f2unpack(v);
  return sm100::pack2<std::is_same_v<T, __nv_bfloat16>>(f.x, f.y);
}

struct Ring {
  int rows;          // of a chunk
  int stages;
  int x_bytes;       // room of a chunk of x, of dn
  int n_bytes;
  int bars;          // where the barriers are, behind the ring
  int* fault;
  uint32_t probe_ns;
};

constexpr int STREAM_T = 256;
constexpr int team_of(int G) { return G > 32 ? G : 32; }

__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
template <typename T>
__device__ __forceinline__ float lds1(uint32_t at) {
  if constexpr (sizeof(T) == 4) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
  } else {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
    return (float)*reinterpret_cast<T*>(&v);
  }
}

// A thread's share of a row in shared memory, in pairs; 0 beside the channels.
template <typename T, int V, int G, int E>
__device__ __forceinline__ void take2(uint32_t row, int C, int lane, bool live, f2 (&o)[E / 2]) {
  if constexpr (V == 8) {
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      const int c = (j * G + lane) * 8;
      uint4 a = make_uint4(0, 0, 0, 0), b = a;
      if (live && c < C) {
        a = lds16(row + c * (int)sizeof(T));
        if constexpr (sizeof(T) == 4) b = lds16(row + c * (int)sizeof(T) + 16);
      }
      if constexpr (sizeof(T) == 4) {
        o[4 * j] = widen2<T>(a.x, a.y); o[4 * j + 1] = widen2<T>(a.z, a.w);
        o[4 * j + 2] = widen2<T>(b.x, b.y); o[4 * j + 3] = widen2<T>(b.z, b.w);
      } else {
        o[4 * j] = widen2<T>(a.x, 0); o[4 * j + 1] = widen2<T>(a.y, 0);
        o[4 * j + 2] = widen2<T>(a.z, 0); o[4 * j + 3] = widen2<T>(a.w, 0);
      }
    }
  } else {
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = live && e * G + lane < C ? lds1<T>(row + (e * G + lane) * (int)sizeof(T)) : 0.f;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) o[i] = sm100::f2pack(v[2 * i], v[2 * i + 1]);
  }
}
template <typename T, int V, int G, int E>
__device__ __forceinline__ void give2(T* row, int C, int lane, const f2 (&o)[E / 2]) {
  if constexpr (V == 8) {
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      const int c = (j * G + lane) * 8;
      if (c >= C) continue;
      uint4* p = reinterpret_cast<uint4*>(row + c);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          p[h] = make_uint4((uint32_t)o[4 * j + 2 * h], (uint32_t)(o[4 * j + 2 * h] >> 32), (uint32_t)o[4 * j + 2 * h + 1],
                            (uint32_t)(o[4 * j + 2 * h + 1] >> 32));
      } else {
        p[0] = make_uint4(narrow2<T>(o[4 * j]), narrow2<T>(o[4 * j + 1]), narrow2<T>(o[4 * j + 2]), narrow2<T>(o[4 * j + 3]));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 f = sm100::f2unpack(o[i]);
      if ((2 * i) * G + lane < C) row[(2 * i) * G + lane] = (T)f.x;
      if ((2 * i + 1) * G + lane < C) row[(2 * i + 1) * G + lane] = (T)f.y;
    }
  }
}
// Whether a pair's elements are channels; for vectors both or neither.
template <int V, int G>
__device__ __forceinline__ f2 in_row(f2 v, int i, int lane, int C) {
  if constexpr (V == 8) return channel<8, G>(2 * i, lane) < C ? v : 0;
  const float2 f = sm100::f2unpack(v);
  return sm100::f2pack(channel<1, G>(2 * i, lane) < C ? f.x : 0.f, channel<1, G>(2 * i + 1, lane) < C ? f.y : 0.f);
}
// Weight or bias: once a block, so from any address.
template <int V, int G, int E>
__device__ __forceinline__ void take_vector(const void* p, int dt, int C, int lane, f2 (&o)[E / 2]) {
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const int c = channel<V, G>(2 * i, lane), d = channel<V, G>(2 * i + 1, lane);
    o[i] = sm100::f2pack(p && c < C ? ld1(p, dt, c) : 0.f, p && d < C ? ld1(p, dt, d) : 0.f);
  }
}

template <int G>
__device__ __forceinline__ void team_sync(int team) {
  if constexpr (G <= 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(G) : "memory");
}
// Sum of K values over the G threads of a row; every thread gets it.  Warps of a
// team meet in shared memory (``sh``: [2][K][32] floats a block, used in turn).
template <int G, int K>
__device__ __forceinline__ void team_sum(float (&v)[K], float* sh, int& turn, int team) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (G > 32) {
    const int warp = threadIdx.x >> 5, w0 = threadIdx.x / G * (G / 32);
    float* s = sh + turn * K * 32;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k * 32 + warp] = v[k];
    team_sync<G>(team);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < G / 32; ++i) t += s[k * 32 + w0 + i];
      v[k] = t;
    }
  } else {
    __syncwarp();
  }
}

// One array's part of a chunk: bytes [b0, b1) of it, in the 16-byte units that they
// touch (the array's address is one).  The array's last unit may not be whole: what
// is behind the last whole one comes by plain stores.
struct Span {
  const unsigned char* src;
  uint32_t copied;     // bytes of the copy
  uint32_t rest;       // bytes behind it
  __device__ __forceinline__ Span(const void* p, int64_t b0, int64_t b1, int64_t total) {
    const int64_t a0 = b0 & ~(int64_t)15, a1 = min((b1 + 15) & ~(int64_t)15, total & ~(int64_t)15);
    src = (const unsigned char*)p + a0;
    copied = a1 > a0 ? (uint32_t)(a1 - a0) : 0;
    rest = b1 > a0 + copied ? (uint32_t)(b1 - a0 - copied) : 0;
  }
  __device__ __forceinline__ void store_rest(unsigned char* to) const {
    for (uint32_t i = copied; i < copied + rest; i += 2)
      *reinterpret_cast<uint16_t*>(to + i) = *reinterpret_cast<const uint16_t*>(src + i);
  }
  __device__ __forceinline__ void copy(unsigned char* to, uint64_t* bar) const {
    if (copied) sm100::bulk_g2s(to, src, copied, bar);
  }
};

// A team's walk over its chunks, with the ring in front of it.  Rows are counted in
// 32 bits (there are fewer than 2^31 - 2^20, and no step is longer than 2^20).
template <typename XT, typename NT, int V, int G, bool TWO>
struct Walk {
  static constexpr int TEAM = team_of(G), TEAMS = STREAM_T / TEAM, XS = sizeof(XT), NS = sizeof(NT);
  const Args& a;
  const Ring& r;
  uint64_t* bar;                    // [stages] of this team
  unsigned char* ring;              // [stages][x | dn]
  volatile int* abort;
  const uint32_t rows, step;        // of the array; from a team's chunk to its next
  uint32_t row, ahead;              // the current chunk's first row; that of the next to be brought
  const unsigned char *xp, *np;     // V == 8: where that one lies
  int s = 0, phase = 0;

  __device__ __forceinline__ Walk(const Args& a_, const Ring& r_, unsigned char* smem, volatile int* abort_)
      : a(a_), r(r_), abort(abort_), rows((uint32_t)a_.rows), step(gridDim.x * TEAMS * r_.rows) {
    const int team = threadIdx.x / TEAM;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + r.bars);
    bar = bars + team * r.stages;
    ring = smem + team * r.stages * (r.x_bytes + r.n_bytes);
    row = ahead = (blockIdx.x * TEAMS + team) * r.rows;
    xp = (const unsigned char*)a.x + (int64_t)row * a.C * XS;
    np = (const unsigned char*)a.dn + (int64_t)row * a.C * NS;
    if (threadIdx.x == 0) {
      for (int i = 0; i <= TEAMS * r.stages; ++i) sm100::mbar_init(bars + i, 1);
      sm100::fence_mbar_init();
      *abort = 0;
      sm100::wait_probe(bars + TEAMS * r.stages, abort, r.probe_ns);
    }
    __syncthreads();
    if (threadIdx.x % TEAM == 0)
      for (int i = 0; i < r.stages; ++i) fill(i);
  }
  __device__ __forceinline__ bool more() const { return row < rows; }
  // Rows of the current chunk.
  __device__ __forceinline__ int here() const { return min((uint32_t)r.rows, rows - row); }
  __device__ __forceinline__ void fill(int i) {
    if (ahead >= rows || *abort) return;
    const int n = min((uint32_t)r.rows, rows - ahead);
    unsigned char* to = ring + i * (r.x_bytes + r.n_bytes);
    if constexpr (V == 8) {
      const uint32_t e = n * a.C;
      sm100::mbar_arrive_expect_tx(bar + i, e * (XS + (TWO ? NS : 0)));
      sm100::bulk_g2s(to, xp, e * XS, bar + i);
      if constexpr (TWO) sm100::bulk_g2s(to + r.x_bytes, np, e * NS, bar + i);
      xp += (int64_t)step * a.C * XS;
      np += (int64_t)step * a.C * NS;
    } else {
      const int64_t e0 = (int64_t)ahead * a.C, e1 = e0 + (int64_t)n * a.C, all = a.rows * a.C;
      const Span x(a.x, e0 * XS, e1 * XS, all * XS);
      x.store_rest(to);
      if constexpr (TWO) {
        const Span n(a.dn, e0 * NS, e1 * NS, all * NS);
        n.store_rest(to + r.x_bytes);
        sm100::mbar_arrive_expect_tx(bar + i, x.copied + n.copied);
        x.copy(to, bar + i);
        n.copy(to + r.x_bytes, bar + i);
      } else {
        sm100::mbar_arrive_expect_tx(bar + i, x.copied);
        x.copy(to, bar + i);
      }
    }
    ahead += step;
  }
  // The current chunk has landed.  A wait that gives up leaves garbage in the results and says so; no thread
  // leaves the walk early, so none is left behind at a team's barrier.
  __device__ __forceinline__ void wait() {
    if (!sm100::mbar_try_wait(bar + s, phase)) sm100::mbar_wait(bar + s, phase, abort);
  }
  // The first of the chunk's rows of x and of dn; rows lie densely behind it.
  __device__ __forceinline__ uint32_t x() const { return at(0, XS); }
  __device__ __forceinline__ uint32_t dn() const { return at(r.x_bytes, NS); }
  __device__ __forceinline__ uint32_t at(int off, int es) const {
    const uint32_t p = sm100::smem_u32(ring) + s * (r.x_bytes + r.n_bytes) + off;
    return V == 8 ? p : p + (row * a.C * es & 15);
  }
  // All threads of the team have read the chunk (and met since): its stage takes another.
  __device__ __forceinline__ void refill() {
    if (threadIdx.x % TEAM == 0) fill(s);
  }
  __device__ __forceinline__ void next() {
    row += step;
    if (++s == r.stages) {
      s = 0;
      phase ^= 1;
    }
  }
  __device__ __forceinline__ void end() {
    __syncthreads();
    sm100::report_abort(abort, r.fault);
    if (*abort)  // give copies in flight time to land before the shared memory they target is released
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
};

// Blocks of STREAM_T threads an SM runs at once, by the registers of E elements a thread.
constexpr int fwd_an_sm(int E) { return E <= 16 ? 3 : 2; }
constexpr int bwd_an_sm(int E) { return E <= 16 ? 2 : 1; }

template <typename XT, typename NT, int V, int G, int E>
__global__ void __launch_bounds__(STREAM_T, fwd_an_sm(E)) layernorm_stream_fwd_kernel(const Args a, const Ring r) {
  constexpr int PASS = team_of(G) / G, P = E / 2;
  extern __shared__ __align__(16) unsigned char room[];
  __shared__ float sh[G > 32 ? 2 * 32 : 1];
  __shared__ int abort;
  int turn = 0;
  const int lane = threadIdx.x % G, sub = threadIdx.x % team_of(G) / G;
  Walk<XT, NT, V, G, false> walk(a, r, room, &abort);
  const int team = threadIdx.x / team_of(G);
  f2 w[P], b[P];
  take_vector<V, G, E>(a.w, a.w_dt, a.C, lane, w);
  take_vector<V, G, E>(a.b, a.b_dt, a.C, lane, b);
  for (; walk.more(); walk.next()) {
    walk.wait();
    const int rows = walk.here();
    const uint32_t px = walk.x();
    for (int p = 0; p < rows; p += PASS) {
      const bool live = p + sub < rows;
      f2 x[P], t = 0;
      take2<XT, V, G, E>(px + (p + sub) * a.C * (int)sizeof(XT), a.C, lane, live, x);
#pragma unroll
      for (int i = 0; i < P; ++i) t = sm100::add2(t, x[i]);
      float2 h = sm100::f2unpack(t);
      float s[1] = {h.x + h.y};
      team_sum<G>(s, sh, turn, team);
      if (p + PASS >= rows) walk.refill();
      const float mean = s[0] * a.inv_c;
      const f2 less = both(-mean);
      t = 0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        x[i] = in_row<V, G>(sm100::add2(x[i], less), i, lane, a.C);
        t = sm100::fma2(x[i], x[i], t);
      }
      h = sm100::f2unpack(t);
      s[0] = h.x + h.y;
      team_sum<G>(s, sh, turn, team);
      const float rstd = rsqrtf(s[0] * a.inv_c + a.eps);
      if (!live) continue;
      const int64_t row = walk.row + p + sub;
      if (lane == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
      }
      const f2 by = both(rstd);
#pragma unroll
      for (int i = 0; i < P; ++i) x[i] = sm100::fma2(sm100::mul2(x[i], by), w[i], b[i]);
      give2<NT, V, G, E>((NT*)a.n + row * a.C, a.C, lane, x);
    }
  }
  walk.end();
}

template <typename XT, typename NT, int V, int G, int E>
__global__ void __launch_bounds__(STREAM_T, bwd_an_sm(E)) layernorm_stream_bwd_kernel(const Args a, const Ring r) {
  constexpr int PASS = team_of(G) / G, P = E / 2, RB = STREAM_T / G;
  extern __shared__ __align__(16) unsigned char room[];  // the ring, later [RB][C]: the block's row groups meet
  __shared__ float sh[G > 32 ? 2 * 2 * 32 : 1];
  __shared__ int abort;
  int turn = 0;
  const int lane = threadIdx.x % G, sub = threadIdx.x % team_of(G) / G;
  Walk<XT, NT, V, G, true> walk(a, r, room, &abort);
  const int team = threadIdx.x / team_of(G);
  f2 w[P], dw[P], db[P];
  take_vector<V, G, E>(a.w, a.w_dt, a.C, lane, w);
#pragma unroll
  for (int i = 0; i < P; ++i) dw[i] = db[i] = 0;
  for (; walk.more(); walk.next()) {
    const int rows = walk.here();
    float mean = sub < rows ? a.mean[walk.row + sub] : 0.f, rstd = sub < rows ? a.rstd[walk.row + sub] : 0.f;
    walk.wait();
    const uint32_t px = walk.x(), pn = walk.dn();
    for (int p = 0; p < rows; p += PASS) {
      const bool live = p + sub < rows;
      const int64_t row = walk.row + p + sub;
      f2 x[P], g[P], s0 = 0, s1 = 0;
      take2<XT, V, G, E>(px + (p + sub) * a.C * (int)sizeof(XT), a.C, lane, live, x);
      take2<NT, V, G, E>(pn + (p + sub) * a.C * (int)sizeof(NT), a.C, lane, live, g);
      const f2 less = both(-mean), by = both(rstd);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        x[i] = sm100::mul2(in_row<V, G>(sm100::add2(x[i], less), i, lane, a.C), by);  // x^
        dw[i] = sm100::fma2(g[i], x[i], dw[i]);
        db[i] = sm100::add2(db[i], g[i]);
        g[i] = sm100::mul2(g[i], w[i]);                                               // u
        s0 = sm100::add2(s0, g[i]);
        s1 = sm100::fma2(g[i], x[i], s1);
      }
      const float rs = rstd;
      if (p + PASS < rows) {  // the next row's
        const bool on = p + PASS + sub < rows;
        mean = on ? a.mean[row + PASS] : 0.f;
        rstd = on ? a.rstd[row + PASS] : 0.f;
      }
      const float2 h0 = sm100::f2unpack(s0), h1 = sm100::f2unpack(s1);
      float s[2] = {h0.x + h0.y, h1.x + h1.y};
      team_sum<G>(s, sh, turn, team);
      if (p + PASS >= rows) walk.refill();
      if (!live || !a.dx) continue;
      const f2 mu = both(-rs * (s[0] * a.inv_c)), mx = both(-rs * (s[1] * a.inv_c)), ra = both(rs);
#pragma unroll
      for (int i = 0; i < P; ++i) g[i] = sm100::fma2(x[i], mx, sm100::fma2(g[i], ra, mu));
      give2<XT, V, G, E>((XT*)a.dx + row * a.C, a.C, lane, g);
    }
  }
  walk.end();
  if (!a.part) return;
  float* meet = reinterpret_cast<float*>(room);
  auto leave = [&](const f2 (&v)[P], int which) {
    float* to = a.part + ((int64_t)blockIdx.x * 2 + which) * a.C;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 f = sm100::f2unpack(v[i]);
      const int c = channel<V, G>(2 * i, lane), d = channel<V, G>(2 * i + 1, lane);
      if (c < a.C) meet[threadIdx.x / G * a.C + c] = f.x;
      if (d < a.C) meet[threadIdx.x / G * a.C + d] = f.y;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += STREAM_T) {
      float t = 0.f;
      for (int i = 0; i < RB; ++i) t += meet[i * a.C + c];
      to[c] = t;
    }
  };
  leave(dw, 0);
  leave(db, 1);
}

// ---------------------------------------------------------------- host
constexpr int LONG = 8192;  // channels a row may have in the register kernels

bool float_type(int dt) { return dt == OW_DTYPE_F32 || dt == OW_DTYPE_BF16 || dt == OW_DTYPE_F16; }

int check(const ow_layernorm_t* a) {
  OW_CHECK_ARG(a != nullptr, "ow_layernorm: args is NULL");
  OW_CHECK_ARG(a->rows >= 0 && a->rows < (1LL << 40) && a->channels > 0 && a->channels < (1 << 30),
               "ow_layernorm: bad shape [%lld, %d]", (long long)a->rows, a->channels);
  if (!float_type(a->x_dtype) || !float_type(a->weight_dtype) || (a->bias && !float_type(a->bias_dtype)) || !float_type(a->n_dtype)) {
    set_error("ow_layernorm: dtypes must be float32, bfloat16 or float16");
    return OW_ERR_UNSUPPORTED;
  }
  OW_CHECK_ARG(a->eps >= 0.0, "ow_layernorm: eps must not be negative");
  OW_CHECK_ARG(a->rows == 0 || (a->x && a->weight), "ow_layernorm: an input pointer is NULL");
  auto at = [](const void* p, int dt) { return (uintptr_t)p % dtype_size(dt) == 0; };
  OW_CHECK_ARG(at(a->x, a->x_dtype) && at(a->weight, a->weight_dtype) && (!a->bias || at(a->bias, a->bias_dtype)) &&
                   at(a->n, a->n_dtype) && ((uintptr_t)a->mean | (uintptr_t)a->rstd) % 4 == 0,
               "ow_layernorm: a tensor is not aligned");
  return OW_OK;
}

Args base(const ow_layernorm_t* a) {
  Args k{};
  k.rows = a->rows;
  k.C = a->channels;
  k.x = a->x; k.w = a->weight; k.b = a->bias;
  k.x_dt = a->x_dtype; k.w_dt = a->weight_dtype; k.b_dt = a->bias_dtype; k.n_dt = a->n_dtype;
  k.eps = (float)a->eps;
  k.inv_c = 1.f / (float)a->channels;
  k.mean = a->mean;
  k.rstd = a->rstd;
  return k;
}

// Calls f<G, NV> with the split of a row of C channels, at most LONG.
template <class F>
int split(int C, F&& f) {
#define OW_SPLIT(G, NV) return f(std::integral_constant<int, G>(), std::integral_constant<int, NV>())
  if (C <= 64) OW_SPLIT(8, 1);
  if (C <= 128) OW_SPLIT(16, 1);
  if (C <= 256) OW_SPLIT(32, 1);
  if (C <= 512) OW_SPLIT(64, 1);
  if (C <= 1024) OW_SPLIT(128, 1);
  if (C <= 2048) OW_SPLIT(256, 1);
  if (C <= 4096) OW_SPLIT(512, 1);
  OW_SPLIT(512, 2);
#undef OW_SPLIT
}

constexpr int BLOCKS_AN_SM = 4;

// Blocks of the general kernels.
int blocks_of(const Args& k) {
  int64_t n = k.rows;
  if (k.C <= LONG)
    split(k.C, [&](auto G, auto) -> int {
      constexpr int RB = threads_of(G.value) / G.value;
      n = (k.rows + RB - 1) / RB;
      return OW_OK;
    });
  return (int)std::max<int64_t>(1, std::min<int64_t>(n, (int64_t)device_sm_count() * BLOCKS_AN_SM));
}

bool aligned(std::initializer_list<const void*> ps) {
  return std::all_of(ps.begin(), ps.end(), [](const void* p) { return (uintptr_t)p % 16 == 0; });
}

// Calls f<G, E> with the streaming kernels' split of a row of C channels, at most LONG.
template <class F>
int split_stream(int C, F&& f) {
#define OW_SPLIT(G, E) return f(std::integral_constant<int, G>(), std::integral_constant<int, E>())
  if (C <= 32) OW_SPLIT(4, 8);
  if (C <= 64) OW_SPLIT(8, 8);
  if (C <= 128) OW_SPLIT(8, 16);
  if (C <= 256) OW_SPLIT(16, 16);
  if (C <= 512) OW_SPLIT(32, 16);
  if (C <= 768) OW_SPLIT(32, 24);
  if (C <= 1024) OW_SPLIT(32, 32);
  if (C <= 2048) OW_SPLIT(64, 32);
  if (C <= 4096) OW_SPLIT(128, 32);
  OW_SPLIT(256, 32);
#undef OW_SPLIT
}

// How a launch streams its rows.
struct Stream {
  int grid;
  Ring r;
  size_t smem;
};
template <int G, int E>
Stream stream_of(const Args& k, bool bwd) {
  constexpr int TEAM = team_of(G), TEAMS = STREAM_T / TEAM, PASS = TEAM / G;
  Stream s{};
  const int an_sm = bwd ? bwd_an_sm(E) : fwd_an_sm(E);
  const int xs = k.x_dt == OW_DTYPE_F32 ? 4 : 2, ns = k.n_dt == OW_DTYPE_F32 ? 4 : 2;
  const int64_t most = (int64_t)device_sm_count() * an_sm;
  // 2 KB of x for each of a team's warps in a chunk, and no less than three chunks for a team
  const int64_t pass = (int64_t)PASS * k.C * xs;
  s.r.rows = PASS * (int)std::max<int64_t>(1, std::min<int64_t>(2048 * (TEAM / 32) / pass, k.rows / (most * TEAMS * PASS * 3)));
  // a chunk starts up to 15 bytes behind a 16-byte unit's start and ends as many before another's end
  s.r.x_bytes = (int)((s.r.rows * (int64_t)k.C * xs + 30) / 16 * 16);
  s.r.n_bytes = bwd ? (int)((s.r.rows * (int64_t)k.C * ns + 30) / 16 * 16) : 0;
  const int room = 220 * 1024 / an_sm - 2048;
  s.r.stages = std::max(2, std::min(6, room / (TEAMS * (s.r.x_bytes + s.r.n_bytes))));
  s.r.bars = TEAMS * s.r.stages * (s.r.x_bytes + s.r.n_bytes);
  s.smem = s.r.bars + (TEAMS * s.r.stages + 1) * 8;
  if (bwd) s.smem = std::max(s.smem, (size_t)(STREAM_T / G) * k.C * sizeof(float));
  const int64_t chunks = (k.rows + s.r.rows - 1) / s.r.rows;
  s.grid = (int)std::max<int64_t>(1, std::min<int64_t>((chunks + TEAMS - 1) / TEAMS, most));
  return s;
}

// Whether the streaming kernels serve: their types, addresses that bulk copies take, and rows enough to fill the SMs.
bool streams(const Args& k, bool at16) {
  const bool types = k.x_dt == OW_DTYPE_F32 || k.x_dt == k.n_dt;
  return types && at16 && k.C <= LONG && k.rows < (1LL << 31) - (1 << 20) && k.rows * k.C >= (int64_t)device_sm_count() * 16384;
}

int reserve(const void* kern, size_t smem) {
  if (smem <= 48 * 1024) return OW_OK;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) {
    set_error("ow_layernorm: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    return OW_ERR_CUDA;
  }
  return OW_OK;
}

template <bool BWD>
int run_stream(const Args& k, int* grid, cudaStream_t st) {
  return split_stream(k.C, [&](auto G, auto E) -> int {
    Stream s = stream_of<G.value, E.value>(k, BWD);
    OW_RETURN_IF(fault_word(&s.r.fault));
    s.r.probe_ns = wait_probe_ns();
    *grid = s.grid;
    auto go = [&](auto x, auto n, auto v) -> int {
      using XT = decltype(x);
      using NT = decltype(n);
      void (*kern)(const Args, const Ring);
      if constexpr (BWD) kern = layernorm_stream_bwd_kernel<XT, NT, v.value, G.value, E.value>;
      else kern = layernorm_stream_fwd_kernel<XT, NT, v.value, G.value, E.value>;
      OW_RETURN_IF(reserve((const void*)kern, s.smem));
      launch(kern, s.grid, STREAM_T, s.smem, st, k, s.r);
      OW_CHECK_LAUNCH("layernorm_stream_kernel");
      return OW_OK;
    };
    auto types = [&](auto v) -> int {
      const int x = k.x_dt, n = k.n_dt;
      if (x == OW_DTYPE_BF16) return go(__nv_bfloat16(), __nv_bfloat16(), v);
      if (x == OW_DTYPE_F16) return go(__half(), __half(), v);
      if (n == OW_DTYPE_BF16) return go(float(), __nv_bfloat16(), v);
      if (n == OW_DTYPE_F16) return go(float(), __half(), v);
      return go(float(), float(), v);
    };
    return k.C % 8 == 0 ? types(std::integral_constant<int, 8>()) : types(std::integral_constant<int, 1>());
  });
}

// Blocks of the backward, at most: each leaves a row of partial sums.
int most_blocks(const Args& k) {
  return std::max(blocks_of(k), (int)std::min<int64_t>(k.rows, (int64_t)device_sm_count() * bwd_an_sm(8)));
}

}  // namespace
}  // namespace ow

using namespace ow;

extern "C" {

size_t ow_layernorm_bwd_workspace_size(const ow_layernorm_t* a) {
  clear_error();
  if (check(a) != OW_OK) return 0;
  const Args k = base(a);
  return (size_t)most_blocks(k) * 2 * k.C * sizeof(float) + 256;
}

int ow_layernorm_fwd(const ow_layernorm_t* a, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  Args k = base(a);
  if (k.rows == 0) return OW_OK;
  OW_CHECK_ARG(a->n && !a->mean == !a->rstd, "ow_layernorm_fwd: a pointer is NULL");
  k.n = a->n;
  const cudaStream_t st = (cudaStream_t)stream;
  int grid = blocks_of(k);
  const bool at16 = aligned({k.x, k.n});
  if (streams(k, at16)) return run_stream<false>(k, &grid, st);
  if (k.C > LONG) {
    launch(layernorm_long_fwd_kernel, grid, 256, 0, st, k);
  } else {
    const bool vec = at16 && k.C % 8 == 0 && aligned({k.w, k.b});
    split(k.C, [&](auto G, auto NV) -> int {
      constexpr int T = threads_of(G.value);
      if (vec) launch(layernorm_fwd_kernel<8, G.value, NV.value>, grid, T, 0, st, k);
      else launch(layernorm_fwd_kernel<1, G.value, NV.value>, grid, T, 0, st, k);
      return OW_OK;
    });
  }
  OW_CHECK_LAUNCH("layernorm_fwd_kernel");
  return OW_OK;
}

int ow_layernorm_bwd(const ow_layernorm_t* a, const ow_layernorm_grads_t* g, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  OW_CHECK_ARG(g != nullptr, "ow_layernorm_bwd: grads is NULL");
  OW_CHECK_ARG(a->rows > 0, "ow_layernorm_bwd: no rows");
  OW_CHECK_ARG(g->dn && a->mean && a->rstd, "ow_layernorm_bwd: a pointer is NULL");
  OW_CHECK_ARG(!g->dbias || float_type(a->bias_dtype), "ow_layernorm_bwd: bias_dtype is not set");
  auto at = [](const void* p, int dt) { return (uintptr_t)p % dtype_size(dt) == 0; };
  OW_CHECK_ARG(at(g->dn, a->n_dtype) && at(g->dx, a->x_dtype) && at(g->dweight, a->weight_dtype) &&
                   (!g->dbias || at(g->dbias, a->bias_dtype)),
               "ow_layernorm_bwd: a gradient is not aligned");
  const size_t need = ow_layernorm_bwd_workspace_size(a);
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("ow_layernorm_bwd needs %zu workspace bytes, got %zu", need, a->workspace_bytes);
    return OW_ERR_WORKSPACE;
  }
  Args k = base(a);
  k.dn = g->dn;
  k.dx = g->dx;
  if (g->dweight || g->dbias) k.part = (float*)(((uintptr_t)a->workspace + 255) & ~(uintptr_t)255);
  if (!k.part && !k.dx) return OW_OK;
  const cudaStream_t st = (cudaStream_t)stream;
  int grid = blocks_of(k);
  const bool at16 = aligned({k.x, k.dn, k.dx});
  if (streams(k, at16)) {
    OW_RETURN_IF(run_stream<true>(k, &grid, st));
  } else if (k.C > LONG) {
    launch(layernorm_long_bwd_kernel, grid, 256, 0, st, k);
  } else {
    const bool vec = at16 && k.C % 8 == 0 && aligned({k.w});
    OW_RETURN_IF(split(k.C, [&](auto G, auto NV) -> int {
      constexpr int T = threads_of(G.value), RB = T / G.value;
      const size_t smem = RB > 1 ? (size_t)RB * k.C * sizeof(float) : 0;  // at most 256 threads of 8 channels: 8 KB
      if (vec) launch(layernorm_bwd_kernel<8, G.value, NV.value>, grid, T, smem, st, k);
      else launch(layernorm_bwd_kernel<1, G.value, NV.value>, grid, T, smem, st, k);
      return OW_OK;
    }));
  }
  OW_CHECK_LAUNCH("layernorm_bwd_kernel");
  if (k.part) {
    launch(layernorm_sum_kernel, dim3((k.C + 31) / 32, 2), 1024, 0, st, (const float*)k.part, grid, k.C, g->dweight, a->weight_dtype,
           g->dbias, a->bias_dtype);
    OW_CHECK_LAUNCH("layernorm_sum_kernel");
  }
  return OW_OK;
}

}  // extern "C"
