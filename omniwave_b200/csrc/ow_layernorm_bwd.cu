// Layer norm's backward for many rows (see ow_layernorm.cu).
#include "ow_layernorm.cuh"

namespace ow {
namespace {

template <typename XT, typename NT, int V, int G, int E, bool FULL>
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
  // a row's mean and deviation are asked for a row ahead
  float mean = 0.f, rstd = 0.f;
  if (walk.row + sub < walk.rows) {
    mean = a.mean[walk.row + sub];
    rstd = a.rstd[walk.row + sub];
  }
  for (; walk.more(); walk.next()) {
    const int rows = walk.here();
    walk.wait();
    const uint32_t px = walk.x(), pn = walk.dn();
    for (int p = 0; p < rows; p += PASS) {
      const bool live = p + sub < rows;
      const int64_t row = walk.row + p + sub;
      f2 x[P], g[P], s0 = 0, s1 = 0;
      take2<XT, V, G, E, FULL>(px + (p + sub) * a.C * (int)sizeof(XT), a.C, lane, live, x, mean);
      take2<NT, V, G, E, FULL>(pn + (p + sub) * a.C * (int)sizeof(NT), a.C, lane, live, g);
      const f2 less = both(-mean), by = both(rstd);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        // x^.  Beside the channels and behind the rows, where g is 0, it has to be 0 too: a mean times a deviation's
        // inverse may overflow, and 0 times that is NaN.
        const bool in = FULL || V == 1 || channel<8, G>(2 * i & ~7, lane) < a.C;
        x[i] = sm100::mul2(sm100::add2(x[i], less), in ? by : 0);
        dw[i] = sm100::fma2(g[i], x[i], dw[i]);
        db[i] = sm100::add2(db[i], g[i]);
        g[i] = sm100::mul2(g[i], w[i]);                                               // u
        s0 = sm100::add2(s0, g[i]);
        s1 = sm100::fma2(g[i], x[i], s1);
      }
      const float rs = rstd;
      const uint32_t then = (p + PASS < rows ? walk.row + p + PASS : walk.row + walk.step) + sub;
      mean = rstd = 0.f;  // of what is no row (only the last chunk ends inside a pass)
      if (then < walk.rows) {
        mean = a.mean[then];
        rstd = a.rstd[then];
      }
      const float2 h0 = sm100::f2unpack(s0), h1 = sm100::f2unpack(s1);
      float s[2] = {h0.x + h0.y, h1.x + h1.y};
      team_sum<G>(s, sh, turn, team);
      if (p + PASS >= rows) walk.refill();
      if (!live || !a.dx) continue;
      const f2 mu = both(-rs * (s[0] * a.inv_c)), mx = both(-rs * (s[1] * a.inv_c)), ra = both(rs);
#pragma unroll
      for (int i = 0; i < P; ++i) g[i] = sm100::fma2(x[i], mx, sm100::fma2(g[i], ra, mu));
      give2<XT, V, G, E, FULL>((XT*)a.dx + row * a.C, a.C, lane, g);
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

}  // namespace

int layernorm_stream_backward(const LayerNormArgs& k, int* grid, cudaStream_t st) {
  return run_stream<true>(k, grid, st, [](auto x, auto n, auto V, auto G, auto E, auto full) {
    return layernorm_stream_bwd_kernel<decltype(x), decltype(n), V.value, G.value, E.value, full.value>;
  });
}

}  // namespace ow
