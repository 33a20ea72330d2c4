// The gated feed-forward block, forward and backward, on the tensor cores (sm_100a):
//
//   g = x Wg^T + bg;  u = x Wu^T + bu;  h = act(g) u;  y = h Wd^T + bd + r
//   dh = dy Wd;  dg = dh u act'(g);  du = dh act(g)
//   dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dWd = dy^T h
//
// The products are the GEMM of the linear layer (ow_gemm.cuh) in three more forms:
// g, u and h by one launch, whose tiles hold as many columns of g as of u, so that
// the epilogue has both of an element at hand and x is read once; dx by one whose k
// blocks are those of dg Wg and then those of du Wu, so that the sum never leaves
// TMEM; dWg and dWu by one whose tiles are those of both.
//
// h, dg and du are held in 16 bits because the tensor core takes no other; act(g) and
// u act'(g), which the backward multiplies dh with, for their traffic.  Each is rounded
// once, and so dWg is off by what three roundings make, its own among them: 0.0029 of
// its norm in bf16, where its own makes 0.0017.  dh is rounded
// nowhere.  gate's and up's bias gradients are f32 sums of dg and du, as they are
// rounded where dh's product is whole (its epilogue sums what it has staged) and before
// that where it is split.
//
// Bound and measured (B200, device time in a CUDA graph): the tensor pipe under the
// power cap for 16384 x 4096 x 8192, forward 2120 to 2280 us, with the backward 7.6 to
// 8.1 ms (1230 to 1310 TFLOP/s); with k of 512 the epilogues (25088 x 512 x 1024 gelu,
// biases and residual 78 and 286 us); 12544 x 1024 x 2048 f16 silu forward 127 us; one
// token 1024 -> 2048 -> 1024 6.8 us, 12.6 MB at 1.9 TB/s in two launches.
#include "ow_gemm.cuh"

namespace ow {
namespace {

struct GradArgs {
  const float* dh;   // [splits][M, ldh] partial sums of dh
  const void* act;   // [M, ld] act(g)
  const void* slope; // [M, ld] u act'(g)
  void* dg;          // [M, ld]
  void* du;          // [M, ld]
  float* part;       // [chunks][2][N] column sums of dg and of du, or NULL
  int64_t M, ld, ldh, chunk;
  int N, splits;
};

// dg and du from the partial sums of dh, which stays in f32, rounded to the 16-bit type,
// and their f32 column sums for the biases.  A block does 256 columns of a chunk of rows.
template <bool BF16>
__global__ void __launch_bounds__(256) gate_grad_kernel(const GradArgs a) {
  __shared__ float sh[8][264];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n = blockIdx.x * 256 + tx * 8;
  const int64_t m1 = min(a.M, (int64_t)(blockIdx.y + 1) * a.chunk);
  float s[2][8];
#pragma unroll
  for (int k = 0; k < 8; ++k) s[0][k] = s[1][k] = 0.f;
  const bool whole = n + 8 <= a.N;
  for (int64_t m = blockIdx.y * a.chunk + ty; m < m1; m += 8) {
    if (n >= a.N) continue;
    float d[8], g[8], u[8];
    const float* part = a.dh + m * a.ldh + n;
#pragma unroll
    for (int k = 0; k < 8; ++k) d[k] = 0.f;
    if (whole) {
#pragma unroll 4
      for (int i = 0; i < a.splits; ++i, part += a.M * a.ldh) {
        const float4 p = *reinterpret_cast<const float4*>(part), q = *reinterpret_cast<const float4*>(part + 4);
        d[0] += p.x; d[1] += p.y; d[2] += p.z; d[3] += p.w;
        d[4] += q.x; d[5] += q.y; d[6] += q.z; d[7] += q.w;
      }
      const uint4 gv = *reinterpret_cast<const uint4*>((const uint16_t*)a.act + m * a.ld + n);
      const uint4 uv = *reinterpret_cast<const uint4*>((const uint16_t*)a.slope + m * a.ld + n);
      const uint32_t gq[4] = {gv.x, gv.y, gv.z, gv.w}, uq[4] = {uv.x, uv.y, uv.z, uv.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 i = unpack2<BF16>(gq[k]), j = unpack2<BF16>(uq[k]);
        g[2 * k] = i.x; g[2 * k + 1] = i.y;
        u[2 * k] = j.x; u[2 * k + 1] = j.y;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = n + k < a.N;
        for (int i = 0; in && i < a.splits; ++i) d[k] += part[i * a.M * a.ldh + k];
        g[k] = in ? ld16(a.act, m * a.ld + n + k, BF16) : 0.f;
        u[k] = in ? ld16(a.slope, m * a.ld + n + k, BF16) : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      u[k] *= d[k];   // dg
      d[k] *= g[k];   // du
      s[0][k] += u[k];
      s[1][k] += d[k];
    }
    // rows start on 16 bytes and have room for whole vectors
    *reinterpret_cast<uint4*>((uint16_t*)a.dg + m * a.ld + n) =
        make_uint4(pack2<BF16>(u[0], u[1]), pack2<BF16>(u[2], u[3]), pack2<BF16>(u[4], u[5]), pack2<BF16>(u[6], u[7]));
    *reinterpret_cast<uint4*>((uint16_t*)a.du + m * a.ld + n) =
        make_uint4(pack2<BF16>(d[0], d[1]), pack2<BF16>(d[2], d[3]), pack2<BF16>(d[4], d[5]), pack2<BF16>(d[6], d[7]));
  }
  if (!a.part) return;
  for (int i = 0; i < 2; ++i) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) sh[ty][tx * 8 + k] = i ? s[1][k] : s[0][k];
    __syncthreads();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c < a.N) {
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) t += sh[j][threadIdx.x];
      a.part[((int64_t)i * gridDim.y + blockIdx.y) * a.N + c] = t;
    }
  }
}

// ---------------------------------------------------------------- host
int check(const ow_ffn_t* a) {
  OW_CHECK_ARG(a != nullptr, "ow_ffn: args is NULL");
  OW_CHECK_ARG(a->rows >= 0 && a->in_features > 0 && a->hidden > 0 && a->out_features > 0, "ow_ffn: bad shape [%lld, %d] x [%d] x [%d]",
               (long long)a->rows, a->in_features, a->hidden, a->out_features);
  OW_CHECK_ARG(a->rows < (1LL << 31) - 256 && a->in_features < (1 << 30) && a->hidden < (1 << 29) && a->out_features < (1 << 30),
               "ow_ffn: too large");
  if (!is16(a->dtype)) {
    set_error("ow_ffn: dtype must be bfloat16 or float16 (code %d)", a->dtype);
    return OW_ERR_UNSUPPORTED;
  }
  OW_CHECK_ARG(a->activation >= OW_ACT_NONE && a->activation <= OW_ACT_GELU, "ow_ffn: unknown activation %d", a->activation);
  OW_CHECK_ARG(a->ldx >= a->in_features && a->ldg >= a->in_features && a->ldu >= a->in_features && a->ldd >= a->hidden &&
                   (!a->residual || a->ldr >= a->out_features),
               "ow_ffn: a row stride is shorter than its row");
  auto bias = [](const void* p, int dt) { return !p || is16(dt) || dt == OW_DTYPE_F32; };
  OW_CHECK_ARG(bias(a->gate_bias, a->gate_bias_dtype) && bias(a->up_bias, a->up_bias_dtype) && bias(a->down_bias, a->down_bias_dtype),
               "ow_ffn: a bias must be float32, bfloat16 or float16");
  OW_CHECK_ARG(!a->act == !a->slope, "ow_ffn: act and slope are kept both or neither");
  auto at = [](const void* p, int dt) { return !p || (uintptr_t)p % dtype_size(dt) == 0; };
  OW_CHECK_ARG(((uintptr_t)a->x | (uintptr_t)a->gate_weight | (uintptr_t)a->up_weight | (uintptr_t)a->down_weight |
                (uintptr_t)a->out | (uintptr_t)a->residual) % 2 == 0 &&
                   ((uintptr_t)a->h | (uintptr_t)a->act | (uintptr_t)a->slope) % 16 == 0 && at(a->gate_bias, a->gate_bias_dtype) &&
                   at(a->up_bias, a->up_bias_dtype) && at(a->down_bias, a->down_bias_dtype),
               "ow_ffn: a tensor is not aligned");
  return OW_OK;
}

Mat mat_x(const ow_ffn_t* a) { return Mat{a->x, a->rows, a->in_features, a->ldx}; }
Mat mat_g(const ow_ffn_t* a) { return Mat{a->gate_weight, a->hidden, a->in_features, a->ldg}; }
Mat mat_u(const ow_ffn_t* a) { return Mat{a->up_weight, a->hidden, a->in_features, a->ldu}; }

Mat mat_d(const ow_ffn_t* a) { return Mat{a->down_weight, a->out_features, a->hidden, a->ldd}; }
Mat mat_dy(const ow_ffn_t* a, const ow_ffn_grads_t* g) { return Mat{g->dout, a->rows, a->out_features, a->out_features}; }

bool in_units(const ow_ffn_t* a) {
  return a->in_features % 8 == 0 && tma_rows(a->x, a->ldx) && tma_rows(a->gate_weight, a->ldg) && tma_rows(a->up_weight, a->ldu);
}
// Whether the kernels for a few rows serve: as for the linear layer, of both weights.
bool few_rows(const ow_ffn_t* a) {
  if (!in_units(a)) return a->rows <= 4;
  return a->rows <= 16 || (a->rows <= 32 && (int64_t)a->in_features * a->hidden <= (1 << 23));
}

// The projection back, as the linear layer has it.
ow_linear_t down(const ow_ffn_t* a) {
  ow_linear_t d{};
  d.rows = a->rows;
  d.in_features = a->hidden;
  d.out_features = a->out_features;
  d.dtype = a->dtype;
  d.activation = OW_ACT_NONE;
  d.x = a->h;
  d.ldx = up8(a->hidden);
  d.weight = a->down_weight;
  d.ldw = a->ldd;
  d.bias = a->down_bias;
  d.bias_dtype = a->down_bias_dtype;
  d.residual = a->residual;
  d.ldr = a->ldr;
  d.out = a->out;
  return d;
}

Plan plan_gate(const ow_ffn_t* a) { return plan_gemm(a->rows, 2 * a->hidden, blocks_of(a->in_features)); }

// Everything a backward call needs, carved from its workspace.
struct BwdWs {
  bool fused;        // dg and du come from dh's product itself
  void *dg, *du;
  float* bias;       // [2][chunks][hidden]
  int chunks;
  int64_t chunk;
  Plan ph, px, pw;
  DualWs h, x, w;
  GemmWs hs;         // dh's product where it is split
  void* down;        // the projection back's own workspace
  size_t down_bytes;
};

bool wants_gate(const ow_ffn_grads_t* g) { return g->dx || g->dgate_weight || g->dup_weight || g->dgate_bias || g->dup_bias; }

BwdWs bwd_take(const ow_ffn_t* a, const ow_ffn_grads_t* g, Carver& ws) {
  BwdWs b{};
  const int64_t M = a->rows, ld = up8(a->hidden);
  const int F = a->hidden, K = a->in_features;
  if (wants_gate(g)) {
    // Where dh's product is split over k (few tiles), its sum is complete in another kernel only, which then makes dg and du.
    b.ph = plan_gemm(M, F, blocks_of(a->out_features));
    b.fused = b.ph.splits == 1;
    b.dg = ws.take((size_t)M * ld * 2);
    b.du = ws.take((size_t)M * ld * 2);
    if (b.fused) {
      b.h = dual_take<GRAD>(mat_dy(a, g), mat_d(a), Second{}, M, F, b.ph, ws);
      b.chunks = (int)((M + 31) / 32);
    } else {
      b.hs = gemm_take(mat_dy(a, g), mat_d(a), M, F, b.ph, ws);
      // chunks of rows: a few blocks an SM, at least 8 rows each
      const int64_t col_blocks = (F + 255) / 256;
      b.chunks = (int)std::max<int64_t>(1, std::min<int64_t>((M + 7) / 8, (int64_t)device_sm_count() * 8 / col_blocks));
      b.chunk = (M + b.chunks - 1) / b.chunks;
      b.chunks = (int)((M + b.chunk - 1) / b.chunk);
    }
    if (g->dgate_bias || g->dup_bias) b.bias = (float*)ws.take((size_t)b.chunks * 2 * F * 4);
    const Mat dg{nullptr, M, F, ld};
    if (g->dx) {
      b.px = plan_gemm(M, K, 2 * blocks_of(F));
      b.x = dual_take<CAT_K>(dg, mat_g(a), Second{dg, mat_u(a)}, M, K, b.px, ws);
    }
    if (g->dgate_weight || g->dup_weight) {
      b.pw = plan_gemm(2 * F, K, blocks_of(M));
      b.w = dual_take<CAT_M>(dg, mat_x(a), Second{dg}, F, K, b.pw, ws);
    }
  }
  const ow_linear_t d = down(a);
  const ow_linear_grads_t dgr{g->dout, nullptr, g->ddown_weight, g->ddown_dtype, g->ddown_bias};
  b.down_bytes = ow_linear_workspace_size(&d, &dgr);
  b.down = ws.take(b.down_bytes);
  return b;
}

}  // namespace
}  // namespace ow

using namespace ow;

extern "C" {

size_t ow_ffn_workspace_size(const ow_ffn_t* a, const ow_ffn_grads_t* g) {
  clear_error();
  if (check(a) != OW_OK) return 0;
  Carver c(nullptr);
  if (a->rows > 0) {
    if (g) {
      bwd_take(a, g, c);
    } else {
      if (!few_rows(a)) dual_take<GATE>(mat_x(a), mat_g(a), Second{Mat{}, mat_u(a)}, a->rows, a->hidden, plan_gate(a), c);
      const ow_linear_t d = down(a);
      c.take(ow_linear_workspace_size(&d, nullptr));
    }
  }
  return c.used + 256;
}

int ow_ffn_fwd(const ow_ffn_t* a, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  if (a->rows == 0) return OW_OK;
  OW_CHECK_ARG(a->x && a->gate_weight && a->up_weight && a->down_weight && a->h && a->out, "ow_ffn_fwd: a pointer is NULL");
  const size_t need = ow_ffn_workspace_size(a, nullptr);
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("ow_ffn_fwd needs %zu workspace bytes, got %zu", need, a->workspace_bytes);
    return OW_ERR_WORKSPACE;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  const bool bf = a->dtype == OW_DTYPE_BF16;
  const int F = a->hidden, K = a->in_features;
  Carver ws((void*)(((uintptr_t)a->workspace + 255) & ~(uintptr_t)255));
  Epi e{};
  e.bias = a->gate_bias; e.bias_dt = a->gate_bias_dtype; e.act = a->activation; e.bf16 = bf;
  e.z = a->act; e.ldz = up8(F); e.vz = 1;
  e.out = a->h; e.ldo = up8(F); e.vo = 1;
  const Second s{Mat{}, mat_u(a), a->up_bias, a->up_bias_dtype, a->slope};
  if (few_rows(a)) {
    const GateRowsArgs k{{a->x, a->ldx, a->gate_weight, a->ldg, (int)a->rows, F, K, e}, a->up_weight, a->ldu,
                         Gate{a->up_bias, a->up_bias_dtype, a->slope}};
    OW_RETURN_IF(in_units(a) ? run_units<true>(k, st) : run_rows<true>(k, st));
  } else {
    const Plan p = plan_gate(a);
    const DualWs w = dual_take<GATE>(mat_x(a), mat_g(a), s, a->rows, F, p, ws);
    OW_RETURN_IF((gemm_dual<GATE, false, false>(mat_x(a), mat_g(a), s, a->rows, F, K, p, w, e, bf, st)));
  }
  ow_linear_t d = down(a);
  d.workspace_bytes = ow_linear_workspace_size(&d, nullptr);
  d.workspace = ws.take(d.workspace_bytes);
  return ow_linear_fwd(&d, stream);
}

int ow_ffn_bwd(const ow_ffn_t* a, const ow_ffn_grads_t* g, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  OW_CHECK_ARG(g != nullptr, "ow_ffn_bwd: grads is NULL");
  OW_CHECK_ARG(a->rows > 0, "ow_ffn_bwd: no rows");
  auto out = [&](const void* p, int dt) { return !p || dt == a->dtype || dt == OW_DTYPE_F32; };
  if (!out(g->dgate_weight, g->dgate_dtype) || !out(g->dup_weight, g->dup_dtype) || !out(g->ddown_weight, g->ddown_dtype)) {
    set_error("ow_ffn_bwd: a weight's gradient must be of dtype or float32");
    return OW_ERR_UNSUPPORTED;
  }
  auto bias = [](const void* p, int dt) { return !p || is16(dt) || dt == OW_DTYPE_F32; };
  OW_CHECK_ARG(bias(g->dgate_bias, a->gate_bias_dtype) && bias(g->dup_bias, a->up_bias_dtype) && bias(g->ddown_bias, a->down_bias_dtype),
               "ow_ffn_bwd: a bias dtype is not set");
  const bool gate = wants_gate(g), weights = g->dgate_weight || g->dup_weight;
  OW_CHECK_ARG(g->dout && (!gate || (a->down_weight && a->act && a->slope)) && (!g->dx || (a->gate_weight && a->up_weight)) &&
                   (!weights || a->x) && (!g->ddown_weight || a->h) && !g->dgate_weight == !g->dup_weight &&
                   (!weights || g->dgate_dtype == g->dup_dtype),
               "ow_ffn_bwd: a pointer is NULL, or the gradients of gate and up are not asked for alike");
  auto at = [](const void* p, int dt) { return !p || (uintptr_t)p % dtype_size(dt) == 0; };
  OW_CHECK_ARG(((uintptr_t)g->dout | (uintptr_t)g->dx) % 2 == 0 && at(g->dgate_weight, g->dgate_dtype) && at(g->dup_weight, g->dup_dtype) &&
                   at(g->ddown_weight, g->ddown_dtype) && at(g->dgate_bias, a->gate_bias_dtype) && at(g->dup_bias, a->up_bias_dtype) &&
                   at(g->ddown_bias, a->down_bias_dtype),
               "ow_ffn_bwd: a gradient is not aligned");
  const size_t need = ow_ffn_workspace_size(a, g);
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("ow_ffn_bwd needs %zu workspace bytes, got %zu", need, a->workspace_bytes);
    return OW_ERR_WORKSPACE;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  const bool bf = a->dtype == OW_DTYPE_BF16;
  const int F = a->hidden, K = a->in_features;
  const int64_t M = a->rows, ld = up8(F);
  Carver ws((void*)(((uintptr_t)a->workspace + 255) & ~(uintptr_t)255));
  const BwdWs b = bwd_take(a, g, ws);
  if (g->ddown_weight || g->ddown_bias) {
    ow_linear_t d = down(a);
    d.workspace = b.down;
    d.workspace_bytes = b.down_bytes;
    const ow_linear_grads_t dgr{g->dout, nullptr, g->ddown_weight, g->ddown_dtype, g->ddown_bias};
    OW_RETURN_IF(ow_linear_bwd(&d, &dgr, stream));
  }
  if (!gate) return OW_OK;
  if (b.fused) {
    Epi e{};
    e.bf16 = bf;
    e.out = b.dg; e.ldo = ld; e.vo = 1;
    Second s{};
    s.c = b.du; s.kept = a->act; s.kept2 = a->slope; s.part = b.bias;
    // Up to 8 blocks of k a tile's epilogue takes longer than its products (25088 x 512 -> 1024 52 us, and 62 with the
    // other; with 16 blocks, 12544 x 1024 -> 2048, 83 and 74).
    const bool brief = blocks_of(a->out_features) <= 8;
    OW_RETURN_IF((brief ? gemm_dual<GRAD, false, true>(mat_dy(a, g), mat_d(a), s, M, F, a->out_features, b.ph, b.h, e, bf, st)
                        : gemm_dual<GRAD_LONG, false, true>(mat_dy(a, g), mat_d(a), s, M, F, a->out_features, b.ph, b.h, e, bf, st)));
  } else {
    OW_RETURN_IF((gemm<false, true>(mat_dy(a, g), mat_d(a), M, F, a->out_features, b.ph, b.hs, Epi{}, bf, st, true)));
    const GradArgs k{b.hs.part, a->act, a->slope, b.dg, b.du, b.bias, M, ld, b.hs.part_ld, b.chunk, F, b.ph.splits};
    launch(bf ? gate_grad_kernel<true> : gate_grad_kernel<false>, dim3((F + 255) / 256, b.chunks), 256, 0, st, k);
    OW_CHECK_LAUNCH("gate_grad_kernel");
  }
  if (b.bias) {
    launch(dbias_kernel, dim3((F + 31) / 32, 2), 1024, 0, st, (const float*)b.bias, b.chunks, F, g->dgate_bias, a->gate_bias_dtype,
           g->dup_bias, a->up_bias_dtype);
    OW_CHECK_LAUNCH("dbias_kernel");
  }
  const Mat dg{b.dg, M, F, ld}, du{b.du, M, F, ld};
  if (g->dx) {
    Epi e{};
    e.bf16 = bf;
    e.out = g->dx; e.ldo = K; e.vo = tma_rows(g->dx, K);
    OW_RETURN_IF((gemm_dual<CAT_K, false, true>(dg, mat_g(a), Second{du, mat_u(a)}, M, K, F, b.px, b.x, e, bf, st)));
  }
  if (weights) {
    Epi e{};
    e.bf16 = bf;
    e.out = g->dgate_weight; e.ldo = K;
    e.out32 = g->dgate_dtype == OW_DTYPE_F32;
    e.vo = ((uintptr_t)g->dgate_weight | (uintptr_t)g->dup_weight) % 16 == 0 && K % (e.out32 ? 4 : 8) == 0;
    OW_RETURN_IF((gemm_dual<CAT_M, true, true>(dg, mat_x(a), Second{du, Mat{}, nullptr, 0, g->dup_weight}, F, K, M, b.pw, b.w, e, bf, st)));
  }
  return OW_OK;
}

}  // extern "C"
