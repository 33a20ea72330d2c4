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
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "ow_common.cuh"
#include "ow_internal.h"
#include "ow_sm100.cuh"

namespace ow {
namespace {

using namespace sm100;

constexpr int TM = 128, KE = 64;
constexpr int EPI_WARPS = 16, PROD_W = 16, MMA_W = 17, THREADS = 576;
constexpr int A_ST = TM * 128;
constexpr int BLOCK_ST = 2048;  // a 32 x 32 block of 16-bit values, or half a block of f32, in staging
constexpr int PATCH = 12;

// BN columns of a tile; CG CTAs share it (2: 256 rows, BN / 2 rows of B each).
template <int BN, int CG>
struct GC {
  static constexpr int B_ROWS = BN / CG;
  static constexpr int CW = BN == 256 ? 64 : 32;   // columns of an epilogue warp
  static constexpr int NBLK = CW / 32;
  static constexpr int ACTIVE = 4 * (BN / CW);     // epilogue warps at work
  static constexpr int STG_W = NBLK * BLOCK_ST;
  static constexpr int STAGES = BN == 256 ? 5 : BN == 128 ? 6 : 8;
  static constexpr int B_ST = B_ROWS * 128;
  static constexpr int OFF_B = STAGES * A_ST;
  static constexpr int OFF_STG = OFF_B + STAGES * B_ST;
  static constexpr int OFF_BAR = OFF_STG + ACTIVE * STG_W;
  static constexpr int NBAR = 2 * STAGES + 4 + 1 + EPI_WARPS;  // full, empty, tfull[2], tfree[2], probe, residual
  static constexpr int SMEM = OFF_BAR + NBAR * 8 + 16 + 1024;
  static constexpr int TMEM_COLS = 2 * BN;
  static_assert(SMEM <= 232448, "shared memory budget");
};

// What happens to a block of D on its way out.  Arrays whose rows TMA can
// address (vz, vr, vo) move as 32 x 32 boxes between staging and memory, the
// others element by element.
struct Epi {
  const void* bias;
  int bias_dt;
  int act;
  int bf16;          // 16-bit type of z, residual and out
  void* z;
  int64_t ldz;
  const void* res;
  int64_t ldr;
  void* out;         // 16-bit, or f32 (partials, an f32 weight gradient)
  int64_t ldo;
  int out32;
  int vz, vr, vo;
};

struct GemmArgs {
  int64_t M;
  int N;
  int kblocks;       // 64-wide blocks of k
  int mtiles, ntiles;
  int splits;        // of the k blocks; with more than one, out is the partials
  int kq, kr;        // kblocks / splits and the rest: the first kr splits have a block more
  Epi e;
  int* fault;
  uint32_t probe_ns;
};

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// mbar_wait for a whole warp, without a look at the abort flag where the phase
// is complete.  The lanes agree on the answer: if the wait of one gave up, all
// leave their loop together and none is left behind in a __syncwarp.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity) || mbar_wait(bar, parity, abort));
}
// Whether a phase is complete, without waiting; the same for all lanes.
__device__ __forceinline__ bool is_done(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return __all_sync(0xffffffffu, ok);
}
// One lane of a converged warp, the same one each time.
__device__ __forceinline__ bool elect_lane() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// ---------------------------------------------------------------- CTA pairs
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared-memory address of ``p`` in CTA ``rank`` of the cluster.
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_in(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void arrive_in(uint32_t bar) {
  // release at the scope of the CTA: what it orders is this thread's reads of
  // TMEM (a release at cluster scope waits for every global store before it)
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A load into this CTA that completes on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
template <int CG>
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  if constexpr (CG == 1) {
    umma_f16(d, a, b, id, acc);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
  }
}
// Arrive on ``bar`` (of both CTAs of a pair) once the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CG == 1) {
    umma_commit(bar);
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_take(uint32_t* holder, uint32_t ncols) {
  if constexpr (CG == 1) {
    tmem_alloc(holder, ncols);
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(holder)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_give(uint32_t taddr, uint32_t ncols) {
  if constexpr (CG == 1) tmem_dealloc(taddr, ncols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// Descriptor of an SW128 operand read MN-major: 64-element MN atoms ``lbo``
// bytes apart, 8-line K groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// ---------------------------------------------------------------- activations
// 2^x and 1 / x by the special-function units, subnormals taken as 0 (two
// instructions less each than without).  A quotient below 2^-126 is 0, which of
// silu drops values under 1.1e-36 (z < -87.3); all others keep their 22 bits.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float sigmoid(float z) { return rcp(1.f + ex2(z * -1.44269504f)); }

// gelu(z) = z Phi(z) for a result of the 16-bit type.  Phi's tail, Phi(-|z|), is
// 2^q(|z|): its logarithm is so near a parabola that a polynomial of degree 8
// serves, and its error is one of the tail relative to itself, so gelu keeps its
// bits where it is small (a form whose error is bounded absolutely was off by 8
// steps of f16 at z = -4).  q is this file's own fit, by a linear program over the
// coefficients, one for each type:
//   f16   off by 7e-6 of the tail up to |z| = 6, from where z Phi rounds to 0 (q
//         falls on without end), and by 4e-7 of 1;
//   bf16  by 3.1e-4 of the tail up to 6 and 6.3e-4 up to 13.5, by 6e-7 of 1; from
//         z = -12.9 on the exponential, and gelu below 1.6e-37 with it, is 0.
// One special-function result an element: with erff, or with an exponential and a
// quotient, the epilogue is slower (25088 x 512 x 1024 with bias and kept z 56 and
// 47 us, here 41).
template <bool BF16>
__device__ __forceinline__ float gelu(float z) {
  float q;
  if constexpr (BF16) {
    const float a = fminf(fabsf(z), 13.5f);
    q = fmaf(a, 3.98267339e-8f, -2.39384553e-6f);
    q = fmaf(q, a, 6.14833989e-5f);
    q = fmaf(q, a, -8.9382549e-4f);
    q = fmaf(q, a, 8.29635281e-3f);
    q = fmaf(q, a, -5.3509552e-2f);
    q = fmaf(q, a, -0.458847046f);
    q = fmaf(q, a, -1.15114152f);
    q = fmaf(q, a, -1.00000072f);
  } else {
    const float a = fabsf(z);
    q = fmaf(a, -1.39922733e-7f, 1.43002126e-6f);
    q = fmaf(q, a, 3.0813193e-5f);
    q = fmaf(q, a, -7.80530798e-4f);
    q = fmaf(q, a, 8.10782891e-3f);
    q = fmaf(q, a, -5.33918403e-2f);
    q = fmaf(q, a, -0.458847821f);
    q = fmaf(q, a, -1.15115714f);
    q = fmaf(q, a, -0.999998868f);
  }
  const float tail = ex2(q);
  return z * (z > 0.f ? 1.f - tail : tail);
}
template <int ACT, bool BF16>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == OW_ACT_RELU) return z > 0.f || z != z ? z : 0.f;
  if constexpr (ACT == OW_ACT_SILU) return z * sigmoid(z);
  if constexpr (ACT == OW_ACT_GELU) return gelu<BF16>(z);
  return z;
}
__device__ __forceinline__ float act_fwd(float z, int act, int bf16) {
  return act == OW_ACT_RELU   ? act_fwd<OW_ACT_RELU, false>(z)
         : act == OW_ACT_SILU ? act_fwd<OW_ACT_SILU, false>(z)
         : act == OW_ACT_GELU ? (bf16 ? gelu<true>(z) : gelu<false>(z))
                              : z;
}

// act'(z)
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == OW_ACT_RELU) return z > 0.f ? 1.f : z == z ? 0.f : z;
  if constexpr (ACT == OW_ACT_SILU) {
    const float s = sigmoid(z);
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if constexpr (ACT == OW_ACT_GELU) {
    // Phi(z) + z phi(z).  The density needs exp(-z^2 / 2) anyway, and the tail is
    // t P(t) times it with t = 1 / (1 + 0.35 |z|): this file's own fit again, off by
    // 1e-7 of 1, 3e-7 of the tail up to |z| = 6 and 3e-5 up to 14
    const float e = ex2(z * z * -0.72134752f);
    const float t = rcp(fmaf(fabsf(z), 0.35f, 1.f));
    float tail = fmaf(t, 0.0471570618f, -0.194429092f);
    tail = fmaf(tail, t, 0.226878741f);
    tail = fmaf(tail, t, -0.00380232154f);
    tail = fmaf(tail, t, 0.148624128f);
    tail = fmaf(tail, t, 0.135697883f);
    tail = fmaf(tail, t, 0.139873699f) * t * e;
    return fmaf(z * 0.39894228040143268f, e, z > 0.f ? 1.f - tail : tail);
  }
  return 1.f;
}

// z as it is kept for the backward: a finite value stays finite in f16 (an
// infinite one would make silu' and gelu' NaN).
__device__ __forceinline__ float keep_z(float z, int bf16) {
  return bf16 ? z : z > 65504.f ? 65504.f : z < -65504.f ? -65504.f : z;
}

__device__ __forceinline__ float ld16(const void* p, int64_t i, int bf16) {
  return bf16 ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : __half2float(((const __half*)p)[i]);
}
__device__ __forceinline__ void st16(void* p, int64_t i, int bf16, float v) {
  if (bf16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
  else ((__half*)p)[i] = __float2half_rn(v);
}
__device__ __forceinline__ float ld_any(const void* p, int dt, int64_t i) {
  return dt == OW_DTYPE_F32 ? ((const float*)p)[i] : ld16(p, i, dt == OW_DTYPE_BF16);
}
__device__ __forceinline__ uint32_t pk(float a, float b, int bf16) { return bf16 ? pack2<true>(a, b) : pack2<false>(a, b); }
__device__ __forceinline__ float2 upk(uint32_t v, int bf16) { return bf16 ? unpack2<true>(v) : unpack2<false>(v); }

// ---------------------------------------------------------------- epilogue
// A warp's block of 32 rows, a row a lane: 64-byte rows in staging under the
// 64-byte swizzle of the TMA boxes that carry it (conflict free for a warp that
// writes its rows 16 bytes at a time).
__device__ __forceinline__ uint32_t stg_at(int row, int u) { return row * 64 + ((u ^ ((row >> 1) & 3)) << 4); }

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int c0, int c1, int c2, const void* src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(src))
               : "memory");
}

// The lanes' rows of 32 16-bit values, staged and sent to rows m0.. and
// columns n0.. of an array.  The caller waits for the copy before it writes
// the staging again.
__device__ __forceinline__ void put16(unsigned char* stg, const float (&v)[32], int bf16, const CUtensorMap* map, bool boxes,
                                      void* out, int64_t ld, int64_t m0, int64_t M, int n0, int N) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    *reinterpret_cast<uint4*>(stg + stg_at(lane, u)) =
        make_uint4(pk(v[8 * u], v[8 * u + 1], bf16), pk(v[8 * u + 2], v[8 * u + 3], bf16),
                   pk(v[8 * u + 4], v[8 * u + 5], bf16), pk(v[8 * u + 6], v[8 * u + 7], bf16));
  if (boxes) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_3d(map, n0, (int)m0, 0, stg);
      bulk_commit();
    }
  } else {
    __syncwarp();
    uint16_t* o = reinterpret_cast<uint16_t*>(out);
    for (int row = 0; row < 32 && m0 + row < M; ++row)
      if (n0 + lane < N)
        o[(m0 + row) * ld + n0 + lane] =
            *reinterpret_cast<const uint16_t*>(stg + stg_at(row, lane >> 3) + (lane & 7) * 2);
    fence_proxy_async_smem();  // before a copy writes the staging again
    __syncwarp();
  }
}

// The same in f32, half a block of 16 columns at a time; waits for its copies.
__device__ __forceinline__ void put32(unsigned char* stg, const float (&v)[32], const CUtensorMap* map, bool boxes, float* out,
                                      int64_t ld, int64_t m0, int64_t M, int n0, int N, int split) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int nb = n0 + 16 * h;
    if (nb >= N) break;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      *reinterpret_cast<float4*>(stg + stg_at(lane, u)) =
          make_float4(v[16 * h + 4 * u], v[16 * h + 4 * u + 1], v[16 * h + 4 * u + 2], v[16 * h + 4 * u + 3]);
    if (boxes) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(map, nb, (int)m0, split, stg);
        bulk_commit();
        bulk_wait_read();
      }
    } else {
      __syncwarp();
      for (int row = lane >> 4; row < 32 && m0 + row < M; row += 2) {
        const int c = lane & 15;
        if (nb + c < N) out[(m0 + row) * ld + nb + c] = *reinterpret_cast<const float*>(stg + stg_at(row, c >> 2) + (c & 3) * 4);
      }
      fence_proxy_async_smem();
    }
    __syncwarp();
  }
}

// This lane's row of the staged residual.
__device__ __forceinline__ void take_res(const unsigned char* stg, uint4 (&r)[4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < 4; ++u) r[u] = *reinterpret_cast<const uint4*>(stg + stg_at(lane, u));
}
// A residual whose rows TMA cannot address, staged element by element.
__device__ __forceinline__ void stage_res(unsigned char* stg, const Epi& e, int64_t m0, int64_t M, int n0, int N) {
  const int lane = threadIdx.x & 31;
  for (int row = 0; row < 32; ++row)
    *reinterpret_cast<uint16_t*>(stg + stg_at(row, lane >> 3) + (lane & 7) * 2) =
        m0 + row < M && n0 + lane < N ? reinterpret_cast<const uint16_t*>(e.res)[(m0 + row) * e.ldr + n0 + lane] : 0;
  __syncwarp();
}

__device__ __forceinline__ void add_bias(float (&v)[32], const Epi& e, int n0, int N) {
  if (n0 + 32 <= N && e.bias_dt == OW_DTYPE_F32 && ((uintptr_t)e.bias & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 b = __ldg(reinterpret_cast<const float4*>((const float*)e.bias + n0) + i);
      v[4 * i] += b.x; v[4 * i + 1] += b.y; v[4 * i + 2] += b.z; v[4 * i + 3] += b.w;
    }
  } else if (n0 + 32 <= N && e.bias_dt != OW_DTYPE_F32 && ((uintptr_t)e.bias & 15) == 0) {
    const int bf = e.bias_dt == OW_DTYPE_BF16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 b = __ldg(reinterpret_cast<const uint4*>((const uint16_t*)e.bias + n0) + i);
      const uint32_t q[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = upk(q[k], bf);
        v[8 * i + 2 * k] += f.x;
        v[8 * i + 2 * k + 1] += f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (n0 + i < N) v[i] += ld_any(e.bias, e.bias_dt, n0 + i);
  }
}

// ---------------------------------------------------------------- GEMM
struct Unit {
  int mt, nt, split, kb0, kb1;
};

// Unit u: the splits outermost (CTAs at work then read the same k range),
// tiles in patches of PATCH row blocks.
__device__ __forceinline__ Unit unit_of(const GemmArgs& a, int u) {
  // a division here is a hundred cycles before the first copy; most launches need one
  const uint32_t tiles = (uint32_t)(a.mtiles * a.ntiles);
  Unit r;
  r.split = a.splits == 1 ? 0 : (int)((uint32_t)u / tiles);
  const uint32_t t = (uint32_t)u - (uint32_t)r.split * tiles;
  const uint32_t per = (uint32_t)(PATCH * a.ntiles), p = a.mtiles <= PATCH ? 0 : t / per, q = t - p * per;
  const uint32_t rows = (uint32_t)min(PATCH, a.mtiles - (int)p * PATCH);
  r.nt = (int)(q / rows);
  r.mt = (int)(p * PATCH + (q - (uint32_t)r.nt * rows));
  r.kb0 = r.split * a.kq + min(r.split, a.kr);
  r.kb1 = r.kb0 + a.kq + (r.split < a.kr ? 1 : 0);
  return r;
}

struct Maps {
  CUtensorMap a, b, out, z, res;
};

template <int BN, int CG, bool AMN, bool BMN, bool BF16, int ACT>
__global__ void __launch_bounds__(THREADS, 1) gemm_kernel(const __grid_constant__ Maps maps, const GemmArgs a) {
  using C = GC<BN, CG>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tfree = tfull + 2;
  uint64_t* probe = tfree + 2;
  uint64_t* rbar = probe + 1;  // [EPI_WARPS] a warp's residual has landed
  uint32_t* tmem = reinterpret_cast<uint32_t*>(full + C::NBAR);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = a.mtiles * a.ntiles * a.splits;
  const uint32_t rank = CG == 1 ? 0 : cluster_rank();
  const int first = blockIdx.x / CG, step = gridDim.x / CG;
  Unit t = unit_of(a, first);  // while the barriers are set up

  if (warp == 0) {  // a lane a barrier
    for (int i = lane; i < C::NBAR; i += 32) {
      uint64_t* b = full + i;
      mbar_init(b, b == tfree || b == tfree + 1 ? C::ACTIVE * CG : 1);
    }
    fence_mbar_init();
    __syncwarp();
    if (lane == 0) {
      *abort = 0;
      wait_probe(probe, abort, a.probe_ns);
    }
  } else if (threadIdx.x == PROD_W * 32) {
    prefetch_map(&maps.a);
    prefetch_map(&maps.b);
  }
  if (warp == MMA_W) tmem_take<CG>(tmem, C::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // the pair's barriers are set up
  tc_fence_after();
  const uint32_t tbase = *tmem;

  if (*abort) {
    // the wait-timeout self-check ran out: nothing is issued
  } else if (warp == PROD_W) {
    // This warp and the next run their loops with all lanes and let one issue:
    // what the instructions take (barriers, descriptors, coordinates) is then
    // computed once for the warp.  With a single lane in the loop, moving it to
    // the uniform registers cost 125 cycles an MMA, whatever its size.
    const bool one = elect_lane();
    int s = 0, turn = 0;
    for (int u = first; u < units;) {
      const int am0 = (t.mt * CG + (int)rank) * TM, bn0 = t.nt * BN + (int)rank * C::B_ROWS;
      for (int kb = t.kb0; kb < t.kb1; ++kb) {
        if (turn > 0 && !wait_for(empty + s, (turn - 1) & 1, abort)) break;
        unsigned char* sa = sm + s * A_ST;
        unsigned char* sb = sm + C::OFF_B + s * C::B_ST;
        if (one) {
          if (rank == 0) mbar_arrive_expect_tx(full + s, CG * (A_ST + C::B_ST));
          auto load = [&](void* dst, const CUtensorMap* map, int c0, int c1) {
            if constexpr (CG == 1) tma_load_2d(dst, map, c0, c1, full + s);
            else tma_load_2d_pair(dst, map, c0, c1, in_cta(full + s, 0));
          };
          if constexpr (AMN) {
#pragma unroll
            for (int i = 0; i < TM / 64; ++i) load(sa + i * 8192, &maps.a, am0 + i * 64, kb * KE);
          } else {
            load(sa, &maps.a, kb * KE, am0);
          }
          if constexpr (BMN) {
#pragma unroll
            for (int i = 0; i < C::B_ROWS / 64; ++i) load(sb + i * 8192, &maps.b, bn0 + i * 64, kb * KE);
          } else {
            load(sb, &maps.b, kb * KE, bn0);
          }
        }
        __syncwarp();
        if (++s == C::STAGES) {
          s = 0;
          ++turn;
        }
      }
      if ((u += step) < units) t = unit_of(a, u);
    }
  } else if (warp == MMA_W) {
    if (rank == 0) {
      constexpr uint32_t ID = idesc_f16(TM * CG, BN, BF16) | (AMN ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u);
      const uint32_t s0 = smem_u32(sm);
      const uint32_t tmem0 = __shfl_sync(0xffffffffu, tbase, 0);
      const bool one = elect_lane();
      int s = 0, tl = 0;
      uint32_t phase = 0;
      // Whether block s has landed, asked while the one before it is issued.  A block's
      // turn of this loop (432 cycles with the wait in front of its products, and as
      // many for 64 columns as for 256) bounds narrow tiles: 2048 x 1024 x 2048 12.0 -> 11.5 us.
      bool ready = false;
      for (int u = first; u < units; ++tl) {
        const int acc = tl & 1;
        if (tl >= 2 && !wait_for(tfree + acc, ((tl >> 1) - 1) & 1, abort)) break;
        tc_fence_after();
        const uint32_t tacc = tmem0 + acc * BN;
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          if (!ready && !wait_for(full + s, phase, abort)) break;
          const int s1 = s + 1 == C::STAGES ? 0 : s + 1;
          const uint32_t phase1 = s1 == 0 ? phase ^ 1 : phase;
          ready = is_done(full + s1, phase1);
          tc_fence_after();
          const uint32_t aA = s0 + s * A_ST, aB = s0 + C::OFF_B + s * C::B_ST;
          const uint64_t da = AMN ? sdesc_mn(aA, 8192) : sdesc_sw128(aA);
          const uint64_t db = BMN ? sdesc_mn(aB, 8192) : sdesc_sw128(aB);
          if (one) {
            // a 16-wide k step further: 2048 bytes (MN-major) or 32, in units of 16
#pragma unroll
            for (int kk = 0; kk < KE / 16; ++kk)
              umma<CG>(tacc, da + kk * (AMN ? 128 : 2), db + kk * (BMN ? 128 : 2), ID, (kb > t.kb0 || kk > 0) ? 1u : 0u);
            commit<CG>(empty + s);
          }
          __syncwarp();
          s = s1;
          phase = phase1;
        }
        if (one) commit<CG>(tfull + acc);
        __syncwarp();
        if ((u += step) < units) t = unit_of(a, u);
      }
    }
  } else if (warp < C::ACTIVE) {
    unsigned char* stg = sm + C::OFF_STG + warp * C::STG_W;
    const int q = warp & 3, group = warp >> 2;
    const Epi& e = a.e;
    int tl = 0, fetched = 0;
    for (int u = first; u < units; ++tl) {
      const int acc = tl & 1;
      const int64_t m0 = (int64_t)(t.mt * CG + (int)rank) * TM + q * 32;
      const int nb = t.nt * BN + group * C::CW;
      const bool some = m0 < a.M && nb < a.N;
      const int blocks = !some ? 0 : nb + 32 < a.N ? C::NBLK : 1;
      // The staging is free once the last tile's copies have read it; the
      // residual is on its way there while the products are still at work.
      if (lane == 0) {
        bulk_wait_read();
        if (e.res && e.vr && some) {
          mbar_arrive_expect_tx(rbar + warp, blocks * BLOCK_ST);
          for (int j = 0; j < blocks; ++j) tma_load_2d(stg + j * BLOCK_ST, &maps.res, nb + 32 * j, (int)m0, rbar + warp);
        }
      }
      __syncwarp();
      if (!wait_for(tfull + acc, (tl >> 1) & 1, abort)) break;
      __syncwarp();
      tc_fence_after();
      if (e.res && e.vr && some) {
        if (!wait_for(rbar + warp, fetched++ & 1, abort)) break;
        __syncwarp();
      }
#pragma unroll
      for (int j = 0; j < C::NBLK; ++j) {
        if (j >= blocks) break;
        const int n0 = nb + 32 * j;
        unsigned char* sj = stg + j * BLOCK_ST;
        uint32_t w[32];
        tmem_ld32(tbase + acc * BN + group * C::CW + j * 32 + ((uint32_t)(q * 32) << 16), w);
        tmem_ld_wait();
        if (j + 1 == blocks) {  // the accumulator is read: the next but one tile may have it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 1) mbar_arrive(tfree + acc);
            else arrive_in(in_cta(tfree + acc, 0));
          }
        }
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(w[i]);
        uint4 r[4];
        if (e.res) {
          if (!e.vr) stage_res(sj, e, m0, a.M, n0, a.N);
          take_res(sj, r);
          __syncwarp();
        }
        if (e.bias) add_bias(v, e, n0, a.N);
        if (e.z) {
          float z[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) z[i] = keep_z(v[i], BF16);
          put16(sj, z, BF16, &maps.z, true, nullptr, 0, m0, a.M, n0, a.N);
        }
        if constexpr (ACT != OW_ACT_NONE) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = act_fwd<ACT, BF16>(v[i]);
        }
        if (e.res) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t p[4] = {r[k].x, r[k].y, r[k].z, r[k].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = upk(p[i], BF16);
              v[8 * k + 2 * i] += f.x;
              v[8 * k + 2 * i + 1] += f.y;
            }
          }
        }
        if (e.z) {  // z's copy has left the staging
          if (lane == 0) bulk_wait_read();
          __syncwarp();
        }
        if (e.out32) put32(sj, v, &maps.out, e.vo, (float*)e.out, e.ldo, m0, a.M, n0, a.N, t.split);
        else put16(sj, v, BF16, &maps.out, e.vo, e.out, e.ldo, m0, a.M, n0, a.N);
      }
      if (blocks == 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 1) mbar_arrive(tfree + acc);
          else arrive_in(in_cta(tfree + acc, 0));
        }
      }
      if ((u += step) < units) t = unit_of(a, u);
    }
    if (lane == 0) bulk_wait_read();  // the staging stays until it is read
  }

  __syncwarp();
  __syncthreads();
  report_abort(abort, a.fault);
  if (*abort) {
    // A wait gave up: give in-flight copies and MMAs time to land before the
    // shared memory and TMEM they target are released.
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  // Neither CTA of a pair leaves while the other may still count on its barriers.
  if constexpr (CG == 2) cluster_sync();
  if (warp == MMA_W) {
    tc_fence_after();
    tmem_give<CG>(tbase, C::TMEM_COLS);
  }
}

// Adds the split-k partials of [M, N] (row stride ld) in order and finishes.
__global__ void __launch_bounds__(256) gemm_sum_kernel(const float* __restrict__ part, int splits, int64_t stride, int64_t ld,
                                                       int64_t M, int N, const Epi e) {
  const int64_t nv = (N + 3) / 4, total = M * nv;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t m = i / nv;
    const int n = (int)(i - m * nv) * 4;
    float4 s = *reinterpret_cast<const float4*>(part + m * ld + n);  // ld is a multiple of 4
    for (int p = 1; p < splits; ++p) {
      const float4 t = *reinterpret_cast<const float4*>(part + p * stride + m * ld + n);
      s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
    }
    float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (n + k >= N) break;
      float z = v[k];
      if (e.bias) z += ld_any(e.bias, e.bias_dt, n + k);
      if (e.z) st16(e.z, m * e.ldz + n + k, e.bf16, keep_z(z, e.bf16));
      z = act_fwd(z, e.act, e.bf16);
      if (e.res) z += ld16(e.res, m * e.ldr + n + k, e.bf16);
      if (e.out32) ((float*)e.out)[m * e.ldo + n + k] = z;
      else st16(e.out, m * e.ldo + n + k, e.bf16, z);
    }
  }
}

// ---------------------------------------------------------------- a few rows
struct RowsArgs {
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t ldw;
  int M, N, K;
  Epi e;
};

// One output from its sum: bias, the kept z, the activation, the residual.
__device__ __forceinline__ void finish_one(const Epi& e, float z, int64_t m, int n, int bf) {
  if (e.bias) z += ld_any(e.bias, e.bias_dt, n);
  if (e.z) st16(e.z, m * e.ldz + n, bf, keep_z(z, bf));
  z = act_fwd(z, e.act, bf);
  if (e.res) z += ld16(e.res, m * e.ldr + n, bf);
  st16(e.out, m * e.ldo + n, bf, z);
}

// Rows that are not 16-byte units.  Four warps share a feature (its k dealt out
// in turns of 32), a block of 8 warps does two; MR rows at once.
template <int MR>
__global__ void __launch_bounds__(256) linear_rows_kernel(const RowsArgs a) {
  __shared__ float sh[8][MR];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp & 3;
  const int n = blockIdx.x * 2 + (warp >> 2);
  const int bf = a.e.bf16;
  float s[MR];
#pragma unroll
  for (int r = 0; r < MR; ++r) s[r] = 0.f;
  if (n < a.N) {
    const uint16_t* w = reinterpret_cast<const uint16_t*>(a.w) + n * a.ldw;
    const uint16_t* x = reinterpret_cast<const uint16_t*>(a.x);
#pragma unroll 4
    for (int64_t k = part * 32 + lane; k < a.K; k += 128) {
      const float wk = ld16(w, k, bf);
#pragma unroll
      for (int r = 0; r < MR; ++r)
        if (r < a.M) s[r] = fmaf(wk, ld16(x, r * a.ldx + k, bf), s[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < MR; ++r)
#pragma unroll
    for (int o = 16; o; o >>= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
  if (lane == 0)
#pragma unroll
    for (int r = 0; r < MR; ++r) sh[warp][r] = s[r];
  __syncthreads();
  if (part == 0 && lane < MR && lane < a.M && n < a.N)
    finish_one(a.e, ((sh[warp][lane] + sh[warp + 1][lane]) + sh[warp + 2][lane]) + sh[warp + 3][lane], lane, n, bf);
}

template <bool BF16>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes that are read once: not kept in L1, which holds x.  These loads and
// the MMAs are volatile so that all loads of a pass stay ahead of its products.
__device__ __forceinline__ uint4 ld_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 ld_again(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Rows of 16-byte units, up to 8 NB of them, on the warp-wide MMA: a warp takes
// 16 features and, 64 of k a turn, a share of k.  A lane's 16 bytes are 8
// neighbouring k, where the MMA wants k 2t, 2t + 1, 2t + 8, 2t + 9 in lane t; a
// sum does not mind in which order its terms come, so the units go in as they
// lie, W's and x's alike: no shuffle, no shared memory.  Reading W bounds it;
// the loads of some turns are under way before the first product, as many as
// the registers hold beside x's: 4, 3 and 1 turns for NB = 1, 2 and 4 (16 rows,
// 4096 x 4096: 13.1 us with 2 turns, 10.6 with 3; 32 rows: 19 with 2, 13.5 with
// 1, whose blocks are more).  A block's warps meet in shared memory.  Where the
// features give too few blocks to fill the SMs, a cluster of blocks (along y)
// splits k and its first adds them.  All sums in a fixed order.
//
// On CUDA cores (a warp a feature) 8 rows of 4096 x 4096 took 38.7 us, here 8.7;
// one row 11.7 and 8.3; one row of 8192 x 8192 38.3 and 23.9 (5.6 TB/s).
constexpr int UNIT_WARPS = 8;
constexpr int unit_turns(int nb) { return nb == 1 ? 4 : nb == 2 ? 3 : 1; }

template <int NB, bool BF16>
__global__ void __launch_bounds__(UNIT_WARPS * 32) linear_units_kernel(const RowsArgs a) {
  constexpr int U = unit_turns(NB), warps = UNIT_WARPS, ROW = 8 * NB + 1;
  extern __shared__ float sh[];  // [warps][16][ROW], [8 NB][16]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, units = a.K >> 3, splits = gridDim.y, all = warps * splits * 8;
  const uint16_t* w = reinterpret_cast<const uint16_t*>(a.w) + t * 8;
  const uint16_t* x = reinterpret_cast<const uint16_t*>(a.x) + t * 8;
  // features and rows past the end repeat the last; what they give is not stored
  const uint16_t* w0 = w + min(n0 + g, a.N - 1) * a.ldw;
  const uint16_t* w1 = w + min(n0 + g + 8, a.N - 1) * a.ldw;
  const uint16_t* xr[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) xr[j] = x + min(8 * j + g, a.M - 1) * a.ldx;
  float c[NB][4];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j][i] = 0.f;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int q = (blockIdx.y * warps + warp) * 8; q < units; q += all * U) {
    uint4 p[U][2][2], v[U][2][NB];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = q + u * all + h * 4;  // in units; K < 2^30
        const bool in = k + t < units;
        p[u][h][0] = in ? ld_once(w0 + k * 8) : zero;
        p[u][h][1] = in ? ld_once(w1 + k * 8) : zero;
#pragma unroll
        for (int j = 0; j < NB; ++j) v[u][h][j] = in ? ld_again(xr[j] + k * 8) : zero;
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          mma16<BF16>(c[j], p[u][h][0].x, p[u][h][1].x, p[u][h][0].y, p[u][h][1].y, v[u][h][j].x, v[u][h][j].y);
          mma16<BF16>(c[j], p[u][h][0].z, p[u][h][1].z, p[u][h][0].w, p[u][h][1].w, v[u][h][j].z, v[u][h][j].w);
        }
  }
  float* mine = sh + warp * 16 * ROW;
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) mine[(g + 8 * (i >> 1)) * ROW + 8 * j + 2 * t + (i & 1)] = c[j][i];
  __syncthreads();
  float* sum = sh + warps * 16 * ROW;  // this block's sums, for the cluster's first block
  for (int i = threadIdx.x; i < 16 * a.M; i += warps * 32) {
    const int n = n0 + (i & 15), m = i >> 4;
    float z = 0.f;
#pragma unroll
    for (int p = 0; p < warps; ++p) z += sh[(p * 16 + (i & 15)) * ROW + m];
    if (splits > 1) sum[i] = z;
    else if (n < a.N) finish_one(a.e, z, m, n, BF16);
  }
  if (splits == 1) return;
  cluster_sync();
  if (blockIdx.y == 0) {
    for (int i = threadIdx.x; i < 16 * a.M; i += warps * 32) {
      const int n = n0 + (i & 15), m = i >> 4;
      float z = sum[i];
#pragma unroll 4
      for (int p = 1; p < splits; ++p) z += ld_in(in_cta(sum + i, p));
      if (n < a.N) finish_one(a.e, z, m, n, BF16);
    }
  }
  cluster_sync();  // a block's sums stay until the first has read them
}

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

__global__ void __launch_bounds__(1024) dbias_kernel(const float* __restrict__ part, int chunks, int N, void* out, int dt) {
  __shared__ float sh[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
  float t[4] = {0.f, 0.f, 0.f, 0.f};  // four loads in flight: a chain of them is what this kernel takes
  if (c < N)
    for (int p = ry; p < chunks; p += 128) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (p + 32 * k < chunks) t[k] += part[(int64_t)(p + 32 * k) * N + c];
    }
  sh[ry][cx] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
  if (ry == 0 && c < N) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += sh[i][cx];
    if (dt == OW_DTYPE_F32) ((float*)out)[c] = v;
    else st16(out, c, dt == OW_DTYPE_BF16, v);
  }
}

// Rows of ``cols`` 16-bit elements copied to rows of ``ldd`` (a multiple of 8),
// for an operand whose rows TMA cannot read in place.
__global__ void __launch_bounds__(256) pad_rows_kernel(const uint16_t* __restrict__ src, int64_t lds, uint16_t* __restrict__ dst,
                                                       int64_t ldd, int64_t rows, int cols) {
  const int64_t total = rows * cols;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t r = i / cols;
    const int c = (int)(i - r * cols);
    dst[r * ldd + c] = src[r * lds + c];
  }
}

// ---------------------------------------------------------------- host
int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }

bool tma_rows(const void* p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0; }

// An operand as the GEMM reads it: rows x cols 16-bit elements, row stride ld.
struct Mat {
  const void* p;
  int64_t rows;
  int cols;
  int64_t ld;
};

template <typename... KArgs, typename... Args>
int launch_cluster(const char* name, void (*kern)(KArgs...), dim3 grid, dim3 cluster, int threads, size_t smem, cudaStream_t st,
                   const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cluster.x;
  at.val.clusterDim.y = cluster.y;
  at.val.clusterDim.z = cluster.z;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  count_launches(1);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("%s: launch failed: %s", name, cudaGetErrorString(e));
    return OW_ERR_CUDA;
  }
  return OW_OK;
}

// Shape of one GEMM: the tile's width, whether pairs of SMs share it, and the
// k splits that a model finds fastest, in cycles of an SM.  Its figures are
// measured (B200, 1.75 GHz): a 64-wide k block takes 400 cycles in a 128 x 64
// tile, 460 in 128 x 128 and 600 in the pair's 256 x 256 (products alone: 128,
// 256, 512; an SM's copies at 64 bytes a cycle: 384, 512, 512); an epilogue
// 1300 + 9.5 a column, under the next tile's products; a launch with its first
// copies 6000; splits write and read f32 partials at about 3 KB a cycle and
// start one more kernel (5000).  With few tiles the narrow ones win by filling
// the SMs (2000 x 512 x 512: 6.3, 7.0, 8.9 us), with many the pair's
// (12544 x 2048 x 1024: 81, 52, 39 us).
struct Plan {
  int bn, cg, splits;
};
Plan plan_gemm(int64_t M, int N, int kblocks) {
  const int sms = device_sm_count();
  Plan best{128, 1, 1};
  double least = 1e300;
  struct Tile { int bn, cg, block; };
  for (const Tile t : {Tile{64, 1, 400}, Tile{128, 1, 460}, Tile{256, 2, 600}}) {
    const int64_t tiles = (M + TM * t.cg - 1) / (TM * t.cg) * ((N + t.bn - 1) / t.bn);
    const int slots = sms / t.cg;
    const double epilogue = 1300.0 + 9.5 * t.bn;
    // more splits than fill the SMs twice gain nothing
    const int smax = (int)std::min<int64_t>(std::min(kblocks, 64), 1 + 2 * slots / tiles);
    for (int s = 1; s <= smax; ++s) {
      const int64_t waves = (tiles * s + slots - 1) / slots;
      const int kb = (kblocks + s - 1) / s;
      double c = waves * std::max<double>((double)kb * t.block, epilogue) + epilogue + 6000.0;
      if (s > 1) c += 5000.0 + (double)s * M * N * 8.0 / 3000.0;
      if (c < least) {
        least = c;
        best = Plan{t.bn, t.cg, s};
      }
    }
  }
  return best;
}

// Workspace of one GEMM: padded copies of operands TMA cannot read, partials.
struct GemmWs {
  void* a;
  void* b;
  float* part;
  int64_t part_ld;
};

GemmWs gemm_take(const Mat& A, const Mat& B, int64_t M, int N, const Plan& p, Carver& ws) {
  GemmWs w{};
  if (!tma_rows(A.p, A.ld)) w.a = ws.take((size_t)A.rows * up8(A.cols) * 2);
  if (!tma_rows(B.p, B.ld)) w.b = ws.take((size_t)B.rows * up8(B.cols) * 2);
  w.part_ld = (N + 3) / 4 * 4;
  if (p.splits > 1) w.part = (float*)ws.take((size_t)p.splits * M * w.part_ld * 4);
  return w;
}

int pad_rows(Mat& m, void* to, cudaStream_t st) {
  const int64_t ld = up8(m.cols), total = m.rows * m.cols;
  const int grid = (int)std::min<int64_t>((total + 255) / 256, (int64_t)device_sm_count() * 16);
  launch(pad_rows_kernel, grid, 256, 0, st, (const uint16_t*)m.p, m.ld, (uint16_t*)to, ld, m.rows, m.cols);
  OW_CHECK_LAUNCH("pad_rows_kernel");
  m.p = to;
  m.ld = ld;
  return OW_OK;
}

int map_of(CUtensorMap* map, const Mat& m, bool bf16, uint32_t box_rows) {
  const uint64_t dims[2] = {(uint64_t)m.cols, (uint64_t)m.rows};
  const uint64_t strides[1] = {(uint64_t)m.ld * 2};
  const uint32_t box[2] = {(uint32_t)KE, box_rows};
  return encode_tiled_map(map, bf16, 2, m.p, dims, strides, box, "ow_linear");
}

// An output or residual as boxes of 32 rows x 64 bytes: [splits][rows][cols].
int block_map(CUtensorMap* map, int dtype, const void* p, int64_t rows, int cols, int64_t ld, int splits) {
  const uint64_t es = dtype == OW_DTYPE_F32 ? 4 : 2;
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)splits};
  const uint64_t strides[2] = {(uint64_t)ld * es, (uint64_t)ld * rows * es};
  const uint32_t box[3] = {(uint32_t)(64 / es), 32, 1};
  return encode_tiled_map64(map, dtype, splits > 0 ? 3 : 2, p, dims, strides, box, true, "ow_linear");
}

template <int BN, int CG, bool AMN, bool BMN, bool BF16, int ACT>
int run_gemm(const Maps& maps, const GemmArgs& k, int grid, cudaStream_t st) {
  using C = GC<BN, CG>;
  auto kern = gemm_kernel<BN, CG, AMN, BMN, BF16, ACT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) {
    set_error("ow_linear: cannot reserve %d bytes of shared memory: %s", C::SMEM, cudaGetErrorString(e));
    return OW_ERR_CUDA;
  }
  return launch_cluster("gemm_kernel", kern, dim3(grid), dim3(CG), THREADS, C::SMEM, st, maps, k);
}

// D[M, N] = sum_k A B with the epilogue ``e``.  AMN/BMN: the operand's rows
// run along M or N and its row index is k.
template <bool AMN, bool BMN>
int gemm(Mat A, Mat B, int64_t M, int N, int64_t K, const Plan& p, const GemmWs& w, const Epi& e, bool bf16, cudaStream_t st) {
  if (w.a) OW_RETURN_IF(pad_rows(A, w.a, st));
  if (w.b) OW_RETURN_IF(pad_rows(B, w.b, st));
  Maps maps{};
  OW_RETURN_IF(map_of(&maps.a, A, bf16, AMN ? KE : TM));
  OW_RETURN_IF(map_of(&maps.b, B, bf16, BMN ? KE : p.bn / p.cg));
  GemmArgs k{};
  k.M = M;
  k.N = N;
  k.kblocks = (int)((K + KE - 1) / KE);
  k.mtiles = (int)((M + TM * p.cg - 1) / (TM * p.cg));
  k.ntiles = (N + p.bn - 1) / p.bn;
  k.splits = p.splits;
  k.kq = k.kblocks / p.splits;
  k.kr = k.kblocks % p.splits;
  k.e = e;
  if (p.splits > 1) {
    k.e = Epi{};
    k.e.out = w.part;
    k.e.ldo = w.part_ld;
    k.e.out32 = 1;
    k.e.vo = 1;
  }
  const int t16 = bf16 ? OW_DTYPE_BF16 : OW_DTYPE_F16;
  if (k.e.vo) OW_RETURN_IF(block_map(&maps.out, k.e.out32 ? OW_DTYPE_F32 : t16, k.e.out, M, N, k.e.ldo, p.splits));
  if (k.e.z) OW_RETURN_IF(block_map(&maps.z, t16, k.e.z, M, N, k.e.ldz, 1));
  if (k.e.res && k.e.vr) OW_RETURN_IF(block_map(&maps.res, t16, k.e.res, M, N, k.e.ldr, 0));
  OW_RETURN_IF(fault_word(&k.fault));
  k.probe_ns = wait_probe_ns();
  const int64_t units = (int64_t)k.mtiles * k.ntiles * k.splits;
  OW_CHECK_ARG(units < (1LL << 31) - 1024, "ow_linear: too many tiles");
  const int grid = (int)std::min<int64_t>(units, device_sm_count() / p.cg) * p.cg;
  auto go = [&](auto act) -> int {
    constexpr int ACT = decltype(act)::value;
    auto tile = [&](auto bn, auto cg) -> int {
      constexpr int BN = decltype(bn)::value, CG = decltype(cg)::value;
      return bf16 ? run_gemm<BN, CG, AMN, BMN, true, ACT>(maps, k, grid, st) : run_gemm<BN, CG, AMN, BMN, false, ACT>(maps, k, grid, st);
    };
    if (p.cg == 2) return tile(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    if (p.bn == 64) return tile(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    return tile(std::integral_constant<int, 128>(), std::integral_constant<int, 1>());
  };
  if constexpr (!AMN && !BMN) {  // only the forward has an activation
    switch (k.e.act) {
      case OW_ACT_RELU: OW_RETURN_IF(go(std::integral_constant<int, OW_ACT_RELU>())); break;
      case OW_ACT_SILU: OW_RETURN_IF(go(std::integral_constant<int, OW_ACT_SILU>())); break;
      case OW_ACT_GELU: OW_RETURN_IF(go(std::integral_constant<int, OW_ACT_GELU>())); break;
      default: OW_RETURN_IF(go(std::integral_constant<int, OW_ACT_NONE>()));
    }
  } else {
    OW_RETURN_IF(go(std::integral_constant<int, OW_ACT_NONE>()));
  }
  if (p.splits > 1) {
    const int64_t total = M * ((N + 3) / 4);
    const int g2 = (int)std::min<int64_t>((total + 255) / 256, (int64_t)device_sm_count() * 16);
    launch(gemm_sum_kernel, g2, 256, 0, st, (const float*)w.part, p.splits, M * w.part_ld, w.part_ld, M, N, e);
    OW_CHECK_LAUNCH("gemm_sum_kernel");
  }
  return OW_OK;
}

bool is16(int dt) { return dt == OW_DTYPE_BF16 || dt == OW_DTYPE_F16; }

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
int blocks_of(int64_t k) { return (int)((k + KE - 1) / KE); }

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
    if (in_units(a)) {
      const int blocks = (N + 15) / 16;
      auto go = [&](auto nb, auto b16) -> int {
        constexpr int NB = decltype(nb)::value, W = UNIT_WARPS, turns = std::max(unit_turns(NB), 2);
        // A split costs 0.7 us (2048 -> 1024: 3.5 us whole, 3.9 in two), and pays where each
        // warp keeps the turns that it has under way at once (4096 -> 64: 4.5 whole, 4.0 in two).
        int splits = 1;
        while (splits < 8 && blocks * splits * 2 <= device_sm_count() && K >= 64 * W * turns * splits * 2) splits *= 2;
        const size_t smem = ((size_t)W * 16 * (8 * NB + 1) + 128 * NB) * 4;
        if (splits > 1)
          return launch_cluster("linear_units_kernel", linear_units_kernel<NB, decltype(b16)::value>, dim3(blocks, splits),
                                dim3(1, splits), W * 32, smem, st, k);
        launch(linear_units_kernel<NB, decltype(b16)::value>, blocks, W * 32, smem, st, k);
        OW_CHECK_LAUNCH("linear_units_kernel");
        return OW_OK;
      };
      auto of = [&](auto nb) { return bf ? go(nb, std::true_type()) : go(nb, std::false_type()); };
      if (a->rows <= 8) return of(std::integral_constant<int, 1>());
      if (a->rows <= 16) return of(std::integral_constant<int, 2>());
      return of(std::integral_constant<int, 4>());
    }
    auto go = [&](auto mr) -> int {
      launch(linear_rows_kernel<decltype(mr)::value>, (N + 1) / 2, 256, 0, st, k);
      OW_CHECK_LAUNCH("linear_rows_kernel");
      return OW_OK;
    };
    if (a->rows == 1) return go(std::integral_constant<int, 1>());
    if (a->rows == 2) return go(std::integral_constant<int, 2>());
    return go(std::integral_constant<int, 4>());
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
      launch(dbias_kernel, (N + 31) / 32, 1024, 0, st, (const float*)b.bias, b.chunks, N, g->dbias, a->bias_dtype);
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
