// Linear layer with bias, activation and residual in its epilogue, forward
// and backward, on the tensor cores (sm_100a):
//
//   z = x W^T + b;  y = act(z) + r;    dz = dy act'(z);  dx = dz W;  dW = dz^T x
//
// One GEMM kernel, D[m, n] = sum_k A[m, k] B[n, k], serves all three products.
// An operand is read where it lies, by TMA boxes of 64 elements (128 bytes)
// with the 128-byte swizzle: K-major when its rows run along k (x and W in
// the forward, dz in dx), MN-major when they run across (W in dx, dz and x in
// dW), so nothing is transposed in memory.
//
// Persistent, one CTA per SM, 576 threads: 16 epilogue warps, one thread that
// issues the copies and one that issues the tcgen05.mma (M = 128, N = 64 or 128,
// or M = 256, N = 256).  A ring of 64-wide k blocks feeds the MMA; the accumulator is
// double-buffered in TMEM, so a tile's epilogue runs under the next tile's
// products.  Tiles are walked in patches of 12 row blocks, so that the SMs at
// work share A and B blocks in L2.
//
// A 128 x 256 tile of one SM takes in 48 KB for every 512 cycles of products,
// more than an SM's 64 bytes a cycle.  So large products run on pairs of SMs
// (a cluster of two, cta_group::2): a 256 x 256 tile, each SM holding 128 rows
// of A and 128 of B and accumulating 128 rows of the tile, 32 KB for the same
// products.  The even CTA issues the MMAs of the pair; both load their own
// halves, counted on the even CTA's barriers.
//
// Where the tiles are few and k is long (dW: k is all tokens) the k blocks
// are split over CTAs; each leaves an f32 partial, and a second kernel adds
// them in a fixed order and does the epilogue.
//
// A few rows (serving) are a matter of reading W once, with no tile to stage:
// the warp-wide MMA straight from global memory where rows are 16-byte units,
// CUDA cores where they are not.
//
// Bound and measured (B200, device time in a CUDA graph; torch.matmul without an
// epilogue beside it): the tensor pipe for 8192^3, 713 us = 1542 TFLOP/s (675);
// 12544 x 2048 x 1024 39.7 us (38), its last wave two thirds full; HBM for
// 401408 x 128 x 256, 58 us (57); 25088 x 512 x 1024 25.3 us (25.7), with gelu,
// bias and kept z 41; one row 1024 -> 2048 2.7 us.
#include "ow_gemm.cuh"

namespace ow {
namespace {

// ---------------------------------------------------------------- backward of the epilogue
struct DzArgs {
  const void* dy;    // [M, N] contiguous
  const void* z;     // [M, ldz] or NULL
  void* dz;          // [M, ldz] or NULL (only the sums are wanted)
  float* part;       // [chunks][N] column sums, or NULL
  int64_t M, ldz, chunk;
  int N, vec;
};

// dz = dy act'(z), rounded to the 16-bit type (the tensor core takes no other), and
// its f32 column sums for the bias.  What that costs: a bf16 dW of 4096 x 512 x 256,
// gelu, is off by 0.0024 of its norm, where its own rounding makes 0.0017 and
// dz's as much again; z in 16 bits (half the traffic of f32 in both passes) is
// not seen in it: 0.00234 with an exact z, 0.00240 so.
// A block does 256 columns of a chunk of rows.
// HBM and arithmetic bound it together: 25088 x 1024 bf16 gelu 30.7 us, silu 28.0
// (5.5 TB/s), none (sums alone) 17; without the row ahead, and with the type
// a value instead of a parameter, 34.8, 30.6 and 17.
template <int ACT, bool BF16>
__global__ void __launch_bounds__(256) dz_kernel(const DzArgs a) {
  __shared__ float sh[8][264];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n = blockIdx.x * 256 + tx * 8;
  const int64_t m1 = min(a.M, (int64_t)(blockIdx.y + 1) * a.chunk);
  float s[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) s[k] = 0.f;
  const bool whole = a.vec && n + 8 <= a.N;
  // the row to come is asked for while the one before it is worked on
  uint4 gv = make_uint4(0, 0, 0, 0), zv = gv;
  auto fetch = [&](int64_t m) {
    if (!whole || m >= m1) return;
    gv = *reinterpret_cast<const uint4*>((const uint16_t*)a.dy + m * a.N + n);
    if constexpr (ACT != OW_ACT_NONE) zv = *reinterpret_cast<const uint4*>((const uint16_t*)a.z + m * a.ldz + n);
  };
  int64_t m = blockIdx.y * a.chunk + ty;
  fetch(m);
  for (; m < m1; m += 8) {
    if (n >= a.N) continue;
    float g[8], z[8];
    if (whole) {
      const uint32_t gq[4] = {gv.x, gv.y, gv.z, gv.w}, zq[4] = {zv.x, zv.y, zv.z, zv.w};
      fetch(m + 8);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2<BF16>(gq[k]), h = unpack2<BF16>(zq[k]);
        g[2 * k] = f.x; g[2 * k + 1] = f.y;
        z[2 * k] = h.x; z[2 * k + 1] = h.y;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        g[k] = n + k < a.N ? ld16(a.dy, m * a.N + n + k, BF16) : 0.f;
        z[k] = ACT != OW_ACT_NONE && n + k < a.N ? ld16(a.z, m * a.ldz + n + k, BF16) : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      g[k] *= act_slope<ACT>(z[k]);
      s[k] += g[k];
    }
    if (a.dz)  // rows of dz start on 16 bytes and have room for whole vectors
      *reinterpret_cast<uint4*>((uint16_t*)a.dz + m * a.ldz + n) =
          make_uint4(pack2<BF16>(g[0], g[1]), pack2<BF16>(g[2], g[3]), pack2<BF16>(g[4], g[5]), pack2<BF16>(g[6], g[7]));
  }
  if (!a.part) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) sh[ty][tx * 8 + k] = s[k];
  __syncthreads();
  const int c = threadIdx.x;
  if (blockIdx.x * 256 + c < a.N) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += sh[i][c];
    a.part[(int64_t)blockIdx.y * a.N + blockIdx.x * 256 + c] = t;
  }
}

int check(const ow_linear_t* a) {
  OW_CHECK_ARG(a != nullptr, "ow_linear: args is NULL");
  OW_CHECK_ARG(a->rows >= 0 && a->in_features > 0 && a->out_features > 0, "ow_linear: bad shape [%lld, %d] x [%d]",
               (long long)a->rows, a->in_features, a->out_features);
  OW_CHECK_ARG(a->rows < (1LL << 31) - 256 && a->in_features < (1 << 30) && a->out_features < (1 << 30), "ow_linear: too large");
  if (!is16(a->dtype)) {
    set_error("ow_linear: dtype must be bfloat16 or float16 (code %d)", a->dtype);
    return OW_ERR_UNSUPPORTED;
  }
  OW_CHECK_ARG(a->activation >= OW_ACT_NONE && a->activation <= OW_ACT_GELU, "ow_linear: unknown activation %d", a->activation);
  OW_CHECK_ARG(a->ldx >= a->in_features && a->ldw >= a->in_features && (!a->residual || a->ldr >= a->out_features),
               "ow_linear: a row stride is shorter than its row");
  OW_CHECK_ARG(!a->bias || is16(a->bias_dtype) || a->bias_dtype == OW_DTYPE_F32, "ow_linear: bias must be float32, bfloat16 or float16");
  return OW_OK;
}

bool in_units(const ow_linear_t* a) {
  return a->in_features % 8 == 0 && tma_rows(a->x, a->ldx) && tma_rows(a->weight, a->ldw);
}
// Whether the kernels for a few rows serve.  In units, against the GEMM: 16 rows
// 1024 -> 2048 3.3 and 7.5 us, 4096 -> 4096 10.6 and 14.1, 8192 -> 8192 32 and 30;
// 32 rows 4.1 and 7.6, 13.5 and 14.1, 42 and 31.  Other rows, where the GEMM
// copies x and W first: 4 rows 1001 -> 1000 3.8 and 14, 4090 -> 4096 22 and 57; 8 rows
// 9.5 and 14, 65 and 57.
bool few_rows(const ow_linear_t* a) {
  if (!in_units(a)) return a->rows <= 4;
  return a->rows <= 16 || (a->rows <= 32 && (int64_t)a->in_features * a->out_features <= (1 << 24));
}

Mat mat_x(const ow_linear_t* a) { return Mat{a->x, a->rows, a->in_features, a->ldx}; }
Mat mat_w(const ow_linear_t* a) { return Mat{a->weight, a->out_features, a->in_features, a->ldw}; }

// Everything a backward call needs, carved from its workspace.
struct BwdWs {
  bool own_dz;     // dz is made; else dout serves as it is
  void* dz;        // [rows, up8(N)] (NULL too where only the size is asked for)
  float* bias;     // [chunks][N]
  int chunks;
  int64_t chunk;
  Plan px, pw;
  GemmWs x, w;
};

BwdWs bwd_take(const ow_linear_t* a, const ow_linear_grads_t* g, Carver& ws) {
  BwdWs b{};
  const int N = a->out_features, K = a->in_features;
  const int64_t M = a->rows;
  b.own_dz = (g->dx || g->dweight) && (a->activation != OW_ACT_NONE || !tma_rows(g->dout, N));
  if (b.own_dz) b.dz = ws.take((size_t)M * up8(N) * 2);
  // chunks of rows: a few blocks an SM, at least 8 rows each
  const int64_t col_blocks = (N + 255) / 256;
  b.chunks = (int)std::max<int64_t>(1, std::min<int64_t>((M + 7) / 8, (int64_t)device_sm_count() * 8 / col_blocks));
  b.chunk = (M + b.chunks - 1) / b.chunks;
  b.chunks = (int)((M + b.chunk - 1) / b.chunk);
  if (g->dbias) b.bias = (float*)ws.take((size_t)b.chunks * N * 4);
  const Mat dz = b.own_dz ? Mat{nullptr, M, N, up8(N)} : Mat{g->dout, M, N, N};
  if (g->dx) {
    b.px = plan_gemm(M, K, blocks_of(N));
    b.x = gemm_take(dz, mat_w(a), M, K, b.px, ws);
  }
  if (g->dweight) {
    b.pw = plan_gemm(N, K, blocks_of(M));
    b.w = gemm_take(dz, mat_x(a), N, K, b.pw, ws);
  }
  return b;
}

}  // namespace
}  // namespace ow

using namespace ow;

extern "C" {

size_t ow_linear_workspace_size(const ow_linear_t* a, const ow_linear_grads_t* g) {
  clear_error();
  if (check(a) != OW_OK) return 0;
  Carver c(nullptr);
  if (a->rows > 0) {
    if (g) {
      bwd_take(a, g, c);
    } else if (!few_rows(a)) {
      gemm_take(mat_x(a), mat_w(a), a->rows, a->out_features, plan_gemm(a->rows, a->out_features, blocks_of(a->in_features)), c);
    }
  }
  return c.used + 256;
}

int ow_linear_fwd(const ow_linear_t* a, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  if (a->rows == 0) return OW_OK;
  OW_CHECK_ARG(a->x && a->weight && a->out, "ow_linear_fwd: a pointer is NULL");
  OW_CHECK_ARG(((uintptr_t)a->x | (uintptr_t)a->weight | (uintptr_t)a->out | (uintptr_t)a->residual) % 2 == 0 &&
                   (uintptr_t)a->z % 16 == 0 && (!a->bias || (uintptr_t)a->bias % dtype_size(a->bias_dtype) == 0),
               "ow_linear_fwd: a tensor is not aligned");
  const size_t need = ow_linear_workspace_size(a, nullptr);
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("ow_linear_fwd needs %zu workspace bytes, got %zu", need, a->workspace_bytes);
    return OW_ERR_WORKSPACE;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  const bool bf = a->dtype == OW_DTYPE_BF16;
  const int N = a->out_features, K = a->in_features;
  Epi e{};
  e.bias = a->bias; e.bias_dt = a->bias_dtype; e.act = a->activation; e.bf16 = bf;
  e.z = a->z; e.ldz = up8(N); e.vz = 1;
  e.res = a->residual; e.ldr = a->ldr; e.vr = tma_rows(a->residual, a->ldr);
  e.out = a->out; e.ldo = N; e.vo = tma_rows(a->out, N);
  if (few_rows(a)) {
    const RowsArgs k{a->x, a->ldx, a->weight, a->ldw, (int)a->rows, N, K, e};
    return in_units(a) ? run_units<false>(k, st) : run_rows<false>(k, st);
  }
  Carver ws((void*)(((uintptr_t)a->workspace + 255) & ~(uintptr_t)255));
  const Plan p = plan_gemm(a->rows, N, blocks_of(K));
  const GemmWs w = gemm_take(mat_x(a), mat_w(a), a->rows, N, p, ws);
  return gemm<false, false>(mat_x(a), mat_w(a), a->rows, N, K, p, w, e, bf, st);
}

int ow_linear_bwd(const ow_linear_t* a, const ow_linear_grads_t* g, void* stream) {
  clear_error();
  OW_RETURN_IF(check(a));
  OW_CHECK_ARG(g != nullptr, "ow_linear_bwd: grads is NULL");
  OW_CHECK_ARG(!g->dbias || is16(a->bias_dtype) || a->bias_dtype == OW_DTYPE_F32, "ow_linear_bwd: bias_dtype is not set");
  if (g->dweight && g->dweight_dtype != a->dtype && g->dweight_dtype != OW_DTYPE_F32) {
    set_error("ow_linear_bwd: dweight must be of dtype or float32 (code %d)", g->dweight_dtype);
    return OW_ERR_UNSUPPORTED;
  }
  OW_CHECK_ARG(a->rows > 0, "ow_linear_bwd: no rows");
  OW_CHECK_ARG(g->dout && (!g->dx || a->weight) && (!g->dweight || a->x) && (a->activation == OW_ACT_NONE || a->z),
               "ow_linear_bwd: a pointer is NULL");
  OW_CHECK_ARG(((uintptr_t)a->x | (uintptr_t)a->weight | (uintptr_t)g->dout | (uintptr_t)g->dx) % 2 == 0 &&
                   (uintptr_t)a->z % 16 == 0 && (uintptr_t)g->dweight % dtype_size(g->dweight ? g->dweight_dtype : a->dtype) == 0 &&
                   (!g->dbias || (uintptr_t)g->dbias % dtype_size(a->bias_dtype) == 0),
               "ow_linear_bwd: a tensor is not aligned");
  const size_t need = ow_linear_workspace_size(a, g);
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("ow_linear_bwd needs %zu workspace bytes, got %zu", need, a->workspace_bytes);
    return OW_ERR_WORKSPACE;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  const bool bf = a->dtype == OW_DTYPE_BF16;
  const int N = a->out_features, K = a->in_features;
  const int64_t M = a->rows;
  Carver ws((void*)(((uintptr_t)a->workspace + 255) & ~(uintptr_t)255));
  const BwdWs b = bwd_take(a, g, ws);
  if (b.dz || g->dbias) {
    DzArgs k{g->dout, a->activation == OW_ACT_NONE ? nullptr : a->z, b.dz, b.bias, M, up8(N), b.chunk, N, tma_rows(g->dout, N)};
    const dim3 grid((N + 255) / 256, b.chunks);
    auto go = [&](auto act) {
      if (bf) launch(dz_kernel<decltype(act)::value, true>, grid, 256, 0, st, k);
      else launch(dz_kernel<decltype(act)::value, false>, grid, 256, 0, st, k);
    };
    switch (a->activation) {
      case OW_ACT_NONE: go(std::integral_constant<int, OW_ACT_NONE>()); break;
      case OW_ACT_RELU: go(std::integral_constant<int, OW_ACT_RELU>()); break;
      case OW_ACT_SILU: go(std::integral_constant<int, OW_ACT_SILU>()); break;
      default: go(std::integral_constant<int, OW_ACT_GELU>());
    }
    OW_CHECK_LAUNCH("dz_kernel");
    if (g->dbias) {
      launch(dbias_kernel, (N + 31) / 32, 1024, 0, st, (const float*)b.bias, b.chunks, N, g->dbias, a->bias_dtype, nullptr, 0);
      OW_CHECK_LAUNCH("dbias_kernel");
    }
  }
  const Mat dz = b.dz ? Mat{b.dz, M, N, up8(N)} : Mat{g->dout, M, N, N};
  if (g->dx) {
    Epi e{};
    e.bf16 = bf;
    e.out = g->dx; e.ldo = K; e.vo = tma_rows(g->dx, K);
    OW_RETURN_IF((gemm<false, true>(dz, mat_w(a), M, K, N, b.px, b.x, e, bf, st)));
  }
  if (g->dweight) {
    Epi e{};
    e.bf16 = bf;
    e.out = g->dweight; e.ldo = K;
    e.out32 = g->dweight_dtype == OW_DTYPE_F32;
    e.vo = (uintptr_t)g->dweight % 16 == 0 && K % (e.out32 ? 4 : 8) == 0;
    OW_RETURN_IF((gemm<true, true>(dz, mat_x(a), N, K, M, b.pw, b.w, e, bf, st)));
  }
  return OW_OK;
}

}  // extern "C"

