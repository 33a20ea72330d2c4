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
//
// Bound and measured (B200, device time in a CUDA graph): HBM.  401408 x 128, f32 in
// and bf16 out, forward 53 us (5.8 TB/s) and with the backward 142 (82 of it the
// backward's, 6.2 TB/s); 50176 x 1024 bf16 41 and 102 us (5.0 TB/s, the backward 62);
// 12544 x 4096 38 and 99.  Rows of single channels are bound by instructions: 50176 x
// 777 bf16 72 and 157 us.  One token of 1024 2.1 us.  Without the ring (every row
// straight from global memory, 8 channels a thread) these were 58 and 244, 64 and 236,
// 74 and 270, 174 and 594 us.
#include "ow_layernorm.cuh"

namespace ow {
namespace {

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

template <typename XT, typename NT, int V, int G, int E, bool FULL>
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
      take2<XT, V, G, E, FULL>(px + (p + sub) * a.C * (int)sizeof(XT), a.C, lane, live, x);
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
        x[i] = in_row<V, G, FULL>(sm100::add2(x[i], less), i, lane, a.C);
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
      give2<NT, V, G, E, FULL>((NT*)a.n + row * a.C, a.C, lane, x);
    }
  }
  walk.end();
}

// ---------------------------------------------------------------- host

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

// Whether the streaming kernels serve: their types, addresses that bulk copies take, and rows enough to fill the SMs.
bool streams(const Args& k, bool at16) {
  const bool types = k.x_dt == OW_DTYPE_F32 || k.x_dt == k.n_dt;
  return types && at16 && k.C <= LONG && k.rows < (1LL << 31) - (1 << 20) && k.rows * k.C >= (int64_t)device_sm_count() * 16384;
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
  if (streams(k, at16))
    return run_stream<false>(k, &grid, st, [](auto x, auto n, auto V, auto G, auto E, auto full) {
      return layernorm_stream_fwd_kernel<decltype(x), decltype(n), V.value, G.value, E.value, full.value>;
    });
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
    OW_RETURN_IF(layernorm_stream_backward(k, &grid, st));
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
