// Layer norm's kernels for many rows, shared by its two source files; what they
// compute and why they are built as they are stands in ow_layernorm.cu.
#pragma once

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "ow_common.cuh"
#include "ow_internal.h"
#include "ow_rows.cuh"
#include "ow_sm100.cuh"

namespace ow {

// One launch of the streaming backward (ow_layernorm_bwd.cu); *grid gets its blocks.
struct LayerNormArgs;
int layernorm_stream_backward(const LayerNormArgs& k, int* grid, cudaStream_t st);



struct LayerNormArgs {
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

namespace {

using Args = LayerNormArgs;

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

// A thread's share of a row in shared memory, in pairs; 0 beside the channels, or ``beside`` where they come singly.
template <typename T, int V, int G, int E, bool FULL>
__device__ __forceinline__ void take2(uint32_t row, int C, int lane, bool live, f2 (&o)[E / 2], float beside = 0.f) {
  if constexpr (V == 8) {
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      const int c = (j * G + lane) * 8;
      uint4 a = make_uint4(0, 0, 0, 0), b = a;
      if (live && (FULL || c < C)) {
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
    for (int e = 0; e < E; ++e) v[e] = live && e * G + lane < C ? lds1<T>(row + (e * G + lane) * (int)sizeof(T)) : beside;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) o[i] = sm100::f2pack(v[2 * i], v[2 * i + 1]);
  }
}
template <typename T, int V, int G, int E, bool FULL>
__device__ __forceinline__ void give2(T* row, int C, int lane, const f2 (&o)[E / 2]) {
  if constexpr (V == 8) {
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      const int c = (j * G + lane) * 8;
      if (!FULL && c >= C) continue;
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
template <int V, int G, bool FULL>
__device__ __forceinline__ f2 in_row(f2 v, int i, int lane, int C) {
  if constexpr (FULL) return v;
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
// 32 bits: there are fewer than 2^31, and a step is no longer than a third of them, or than
// the 2^15 rows of one pass of all teams (stream_of).
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

// ---------------------------------------------------------------- host
constexpr int LONG = 8192;  // channels a row may have in the register kernels

// Calls f<G, E> with the streaming kernels' split of a row of C channels, at most LONG.
template <class F>
int split_stream(int C, F&& f) {
#define OW_SPLIT(G, E) return f(std::integral_constant<int, G>(), std::integral_constant<int, E>())
  if (C % 8) {  // by single channels, in fewer splits; a thread's idle channels cost it their instructions
    if (C <= 64) OW_SPLIT(8, 8);
    if (C <= 256) OW_SPLIT(16, 16);
    if (C <= 512) OW_SPLIT(32, 16);
    if (C <= 1024) OW_SPLIT(32, 32);
    if (C <= 2048) OW_SPLIT(64, 32);
    if (C <= 4096) OW_SPLIT(128, 32);
    OW_SPLIT(256, 32);
  }
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

int reserve(const void* kern, size_t smem) {
  if (smem <= 48 * 1024) return OW_OK;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) {
    set_error("ow_layernorm: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    return OW_ERR_CUDA;
  }
  return OW_OK;
}

// Launches the streaming kernel that ``kernel_of(x's type, n's, V, G, E, FULL)`` names.
template <bool BWD, class F>
int run_stream(const Args& k, int* grid, cudaStream_t st, F&& kernel_of) {
  return split_stream(k.C, [&](auto G, auto E) -> int {
    Stream s = stream_of<G.value, E.value>(k, BWD);
    OW_RETURN_IF(fault_word(&s.r.fault));
    s.r.probe_ns = wait_probe_ns();
    *grid = s.grid;
    auto go = [&](auto x, auto n, auto v) -> int {
      void (*kern)(const Args, const Ring) =
          kernel_of(x, n, std::integral_constant<int, (v.value > 1 ? 8 : 1)>(), G, E, std::bool_constant<v.value == 16>());
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
    constexpr int g = G.value, e = E.value;
    if (k.C % 8 == 0) return k.C == g * e ? types(std::integral_constant<int, 16>()) : types(std::integral_constant<int, 8>());
    if constexpr ((g == 8 && e == 8) || (g == 16 && e == 16) || (g == 32 && e == 16) || (g >= 32 && e == 32))
      return types(std::integral_constant<int, 1>());
    return OW_ERR_INVALID;  // not a split of such rows
  });
}

}  // namespace
}  // namespace ow
