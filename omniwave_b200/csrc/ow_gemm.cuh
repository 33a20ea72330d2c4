// The products of the linear layer and of the feed-forward block on the tensor
// cores (sm_100a): the GEMM kernel that serves them all, the kernels for a few
// rows, and the host code that plans and launches them.  What they compute and
// why they are split as they are stands in ow_linear.cu and ow_ffn.cu.
#pragma once

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

// What a launch of the GEMM kernel computes.  PLAIN: one product.  GATE: two
// products of the same A, a tile holding half as many columns of each, whose
// epilogue joins them: act(A B1^T + b1) (A B2^T + b2).  CAT_K: the sum of two
// products, the second's k blocks behind the first's.  CAT_M: two products with the
// same B, the second's tiles behind the first's.  GRAD: one product d, whose epilogue
// reads what GATE kept, act(g) and u act'(g), and writes d times either; GRAD_LONG is
// the same for long k, with more of shared memory for the operands.
enum Kind { PLAIN, GATE, CAT_K, CAT_M, GRAD, GRAD_LONG };
constexpr bool is_grad(int kind) { return kind == GRAD || kind == GRAD_LONG; }

// BN columns of a tile; CG CTAs share it (2: 256 rows, BN / 2 rows of B each).
template <int BN, int CG, int KIND = PLAIN>
struct GC {
  static constexpr int B_ROWS = BN / CG;
  // GATE: a warp has 32 columns of either product
  static constexpr int CW = KIND == GATE ? 64 : BN == 256 ? 64 : 32;   // columns of an epilogue warp
  static constexpr int NBLK = CW / 32;
  static constexpr int ACTIVE = 4 * (BN / CW);     // epilogue warps at work
  // blocks of staging a warp: GATE three (its results leave together), GRAD two (what comes in and goes out in its
  // place) for each of its blocks, GRAD_LONG for all
  static constexpr int SETS = KIND == GRAD ? NBLK : 1;
  static constexpr int STG_W = (KIND == GATE ? 3 : is_grad(KIND) ? 2 * SETS : NBLK) * BLOCK_ST;
  static constexpr int STAGES = BN == 256 ? (KIND == GATE ? 4 : KIND == GRAD ? 3 : 5) : BN == 128 ? (KIND == GATE || is_grad(KIND) ? 5 : 6) : 8;
  static constexpr int B_ST = B_ROWS * 128;
  static constexpr int OFF_B = STAGES * A_ST;
  static constexpr int OFF_STG = OFF_B + STAGES * B_ST;
  static constexpr int OFF_BAR = OFF_STG + ACTIVE * STG_W;
  static constexpr int NBAR = 2 * STAGES + 4 + 1 + 2 * EPI_WARPS;  // full, empty, tfull[2], tfree[2], probe, residual[2]
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
  // GATE (N counts the columns of one product)
  const void* bias2;
  int bias2_dt;
  int raw;           // leave both products as f32 partials, side by side as in the tile
  // CAT_K: k blocks, CAT_M: rows of tiles of the first product
  int half;
  void* out2;        // CAT_M: the second product
  float* part;       // GRAD: [2][blocks of 32 rows][N] column sums of both rounded results, or NULL
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
__device__ __forceinline__ float gelu_tail(float x) {  // x = |z|
  float q;
  if constexpr (BF16) {
    q = fmaf(x, 3.98267339e-8f, -2.39384553e-6f);
    q = fmaf(q, x, 6.14833989e-5f);
    q = fmaf(q, x, -8.9382549e-4f);
    q = fmaf(q, x, 8.29635281e-3f);
    q = fmaf(q, x, -5.3509552e-2f);
    q = fmaf(q, x, -0.458847046f);
    q = fmaf(q, x, -1.15114152f);
    q = fmaf(q, x, -1.00000072f);
  } else {
    q = fmaf(x, -1.39922733e-7f, 1.43002126e-6f);
    q = fmaf(q, x, 3.0813193e-5f);
    q = fmaf(q, x, -7.80530798e-4f);
    q = fmaf(q, x, 8.10782891e-3f);
    q = fmaf(q, x, -5.33918403e-2f);
    q = fmaf(q, x, -0.458847821f);
    q = fmaf(q, x, -1.15115714f);
    q = fmaf(q, x, -0.999998868f);
  }
  return ex2(q);
}
template <bool BF16>
__device__ __forceinline__ float gelu(float z) {
  const float x = fabsf(z), tail = gelu_tail<BF16>(BF16 ? fminf(x, 13.5f) : x);
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

// The larger of z and 0, NaN where z is.
__device__ __forceinline__ float max0(float z) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(z));
  return r;
}

// An activation at z and, where it is used, its slope.  gelu is max(z, 0) - |z| tail
// with the tail of ``gelu``, an operation less than z Phi, and the slope takes Phi from
// the same tail; beyond the clamp the tail is 0.
template <int ACT, bool BF16>
__device__ __forceinline__ void act_both(float z, float& a, float& s) {
  if constexpr (ACT == OW_ACT_SILU) {
    const float g = sigmoid(z);
    a = z * g;
    s = fmaf(a, 1.f - g, g);
  } else if constexpr (ACT == OW_ACT_GELU) {
    const float x = fminf(fabsf(z), BF16 ? 13.5f : 100.f), tail = gelu_tail<BF16>(x);
    a = fmaf(-x, tail, max0(z));
    s = fmaf(z * 0.39894228040143268f, ex2(z * z * -0.72134752f), z > 0.f ? 1.f - tail : tail);
  } else {
    a = act_fwd<ACT, false>(z);
    s = act_slope<ACT>(z);
  }
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

__device__ __forceinline__ void stage16(unsigned char* stg, const float (&v)[32], int bf16) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    *reinterpret_cast<uint4*>(stg + stg_at(lane, u)) =
        make_uint4(pk(v[8 * u], v[8 * u + 1], bf16), pk(v[8 * u + 2], v[8 * u + 3], bf16),
                   pk(v[8 * u + 4], v[8 * u + 5], bf16), pk(v[8 * u + 6], v[8 * u + 7], bf16));
}

// The lanes' rows of 32 16-bit values, staged and sent to rows m0.. and
// columns n0.. of an array.  The caller waits for the copy before it writes
// the staging again.
__device__ __forceinline__ void put16(unsigned char* stg, const float (&v)[32], int bf16, const CUtensorMap* map, bool boxes,
                                      void* out, int64_t ld, int64_t m0, int64_t M, int n0, int N) {
  const int lane = threadIdx.x & 31;
  stage16(stg, v, bf16);
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

template <int C>
__device__ __forceinline__ void add_bias(float (&v)[C], const void* bias, int bias_dt, int n0, int N) {
  if (n0 + C <= N && bias_dt == OW_DTYPE_F32 && ((uintptr_t)bias & 15) == 0) {
#pragma unroll
    for (int i = 0; i < C / 4; ++i) {
      const float4 b = __ldg(reinterpret_cast<const float4*>((const float*)bias + n0) + i);
      v[4 * i] += b.x; v[4 * i + 1] += b.y; v[4 * i + 2] += b.z; v[4 * i + 3] += b.w;
    }
  } else if (n0 + C <= N && bias_dt != OW_DTYPE_F32 && ((uintptr_t)bias & 15) == 0) {
    const int bf = bias_dt == OW_DTYPE_BF16;
#pragma unroll
    for (int i = 0; i < C / 8; ++i) {
      const uint4 b = __ldg(reinterpret_cast<const uint4*>((const uint16_t*)bias + n0) + i);
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
    for (int i = 0; i < C; ++i)
      if (n0 + i < N) v[i] += ld_any(bias, bias_dt, n0 + i);
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
struct Maps2 : Maps {  // of the second product; c2 is GATE's second z, CAT_M's and GRAD's second output, GRAD's b2 act(g)
  CUtensorMap a2, b2, c2;
};
template <int KIND>
using MapsOf = std::conditional_t<KIND == PLAIN, Maps, Maps2>;

// The accumulator is read: the next but one tile may have it.
template <int CG>
__device__ __forceinline__ void give_back(uint64_t* tfree) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    if constexpr (CG == 1) mbar_arrive(tfree);
    else arrive_in(in_cta(tfree, 0));
  }
}

// GATE's epilogue: a warp has 32 rows and 32 columns of both products.  For the
// backward it keeps what that multiplies dh with, act(g) and u act'(g), rounded once
// each, rather than g and u: the slope costs less here, next to the activation, and
// the backward's epilogue is left with two products.  The three results are staged side
// by side and leave together, 16 columns at a time, which the registers hold beside the
// arithmetic.  With k of 512 the arithmetic of an epilogue is what a tile takes: 25088 x
// 512 -> 1024 gelu, with biases, 70 us and 43 with nothing kept, where the products
// alone take 32 (all 32 columns at once, spilling, 81; each result waiting for the one
// before it, 74 with gelu alone; written through the load and store units in the place
// of TMA, 78).
template <int BN, int CG, bool BF16, int ACT>
__device__ __forceinline__ void gate_epilogue(const Maps2& maps, const GemmArgs& a, Unit t, uint32_t rank, int first, int step, int units,
                                              uint32_t tbase, uint64_t* tfull, uint64_t* tfree, unsigned char* stg,
                                              volatile int* abort) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = warp & 3, group = warp >> 2;
  const Epi& e = a.e;
  int tl = 0;
  for (int u = first; u < units; ++tl) {
    const int acc = tl & 1;
    const int64_t m0 = (int64_t)(t.mt * CG + (int)rank) * TM + q * 32;
    const int n0 = t.nt * (BN / 2) + group * 32;
    const bool some = m0 < a.M && n0 < a.N;
    if (!wait_for(tfull + acc, (tl >> 1) & 1, abort)) break;
    __syncwarp();
    tc_fence_after();
    const uint32_t at = tbase + acc * BN + group * 32 + ((uint32_t)(q * 32) << 16);
    if (lane == 0) bulk_wait_read();  // the staging is free once the last tile's copies have read it
    __syncwarp();
    if (!some) {
      give_back<CG>(tfree + acc);
    } else if (a.raw) {
      const int nv = t.nt * BN + group * 32, all = a.ntiles * BN;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t c[32];
        tmem_ld32(at + h * (BN / 2), c);
        tmem_ld_wait();
        if (h == 1) give_back<CG>(tfree + acc);
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(c[i]);
        put32(stg, v, &maps.out, true, nullptr, 0, m0, a.M, nv + h * (BN / 2), all, t.split);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // 16 columns at a time, which the registers hold beside the arithmetic
        uint32_t c[2][16];
        tmem_ld16(at + 16 * h, c[0]);
        tmem_ld16(at + BN / 2 + 16 * h, c[1]);
        tmem_ld_wait();
        if (h == 1) give_back<CG>(tfree + acc);
        float v[16], w[16];  // the gate, its factor
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          v[i] = __uint_as_float(c[0][i]);
          w[i] = __uint_as_float(c[1][i]);
        }
        if (e.bias) add_bias(v, e.bias, e.bias_dt, n0 + 16 * h, a.N);
        if (a.bias2) add_bias(w, a.bias2, a.bias2_dt, n0 + 16 * h, a.N);
        auto block = [&](auto keep) {
          constexpr bool KEEP = decltype(keep)::value;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t o[3][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = 8 * k + 2 * i;
              float a0, s0, a1, s1;
              act_both<ACT, BF16>(v[j], a0, s0);
              act_both<ACT, BF16>(v[j + 1], a1, s1);
              o[0][i] = pack2<BF16>(keep_z(a0, BF16), keep_z(a1, BF16));
              o[1][i] = pack2<BF16>(keep_z(s0 * w[j], BF16), keep_z(s1 * w[j + 1], BF16));
              o[2][i] = pack2<BF16>(a0 * w[j], a1 * w[j + 1]);
            }
#pragma unroll
            for (int i = KEEP ? 0 : 2; i < 3; ++i)
              *reinterpret_cast<uint4*>(stg + i * BLOCK_ST + stg_at(lane, 2 * h + k)) = make_uint4(o[i][0], o[i][1], o[i][2], o[i][3]);
          }
        };
        if (e.z) block(std::true_type());
        else block(std::false_type());
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (e.z) {
          tma_store_3d(&maps.z, n0, (int)m0, 0, stg);
          tma_store_3d(&maps.c2, n0, (int)m0, 0, stg + BLOCK_ST);
        }
        tma_store_3d(&maps.out, n0, (int)m0, 0, stg + 2 * BLOCK_ST);
        bulk_commit();
      }
    }
    if ((u += step) < units) t = unit_of(a, u);
  }
  if (lane == 0) bulk_wait_read();  // the staging stays until it is read
}

// Column sums of a staged block of 32 x 32 16-bit values, to 32 floats of ``out`` of
// which ``cols`` are columns: ones times the block on the warp-wide MMA.  (By shuffles,
// from the registers, it took as many instructions as gelu and its slope.)
template <bool BF16>
__device__ __forceinline__ void column_sums(const unsigned char* stg, float* out, int cols) {
  const int lane = threadIdx.x & 31;
  const uint32_t one = BF16 ? 0x3F803F80u : 0x3C003C00u, at = smem_u32(stg);
  const uint32_t ones[4] = {one, one, one, one};
  float2 mine = make_float2(0.f, 0.f);
#pragma unroll
  for (int u = 0; u < 4; ++u) {  // 8 columns
    uint32_t b[4];
    ldsm_x4_trans(at + stg_at(lane, u), b[0], b[1], b[2], b[3]);
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    mma16816<BF16>(c, ones, b[0], b[1]);
    mma16816<BF16>(c, ones, b[2], b[3]);
    if (lane >> 2 == u) mine = make_float2(c[0], c[1]);
  }
  const int n = (lane >> 2) * 8 + (lane & 3) * 2;  // every row of the product is the sums
  if (lane >= 16) return;
  if (n < cols) out[n] = mine.x;
  if (n + 1 < cols) out[n + 1] = mine.y;
}

// GRAD's epilogue: u act'(g) and act(g) of a block of 32 rows and 32 columns come to
// the staging by copies, their products with d take their places there and leave.  A
// lane reads and writes its own row.  With short k a tile's time is the epilogue's: each
// of a warp's blocks has its own staging, and a tile's are asked for while the tile
// before it is worked on (25088 x 512 -> 1024 52 us, where its traffic takes 36; all in
// one staging 62; 8 warps with blocks of 64 columns 76; by the load and store units, with
// gelu, 109 and TMA 76).  That leaves three stages for the operands, which long k does
// not bear (16384 x 4096 -> 8192 1227 us, and 834 to 960 with five and one staging).
template <int BN, int CG, bool BF16, int KIND>
__device__ __forceinline__ void grad_epilogue(const Maps2& maps, const GemmArgs& a, Unit t, uint32_t rank, int first, int step, int units,
                                              uint32_t tbase, uint64_t* tfull, uint64_t* tfree, uint64_t* here, unsigned char* stg0,
                                              volatile int* abort) {
  using C = GC<BN, CG, KIND>;
  constexpr int SETS = C::SETS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = warp & 3, group = warp >> 2;
  auto row_of = [&](const Unit& t) { return (t.mt * CG + (int)rank) * TM + q * 32; };
  auto col_of = [&](const Unit& t) { return t.nt * BN + group * C::CW; };
  auto blocks_of = [&](const Unit& t) { return row_of(t) >= a.M || col_of(t) >= a.N ? 0 : col_of(t) + 32 < a.N ? C::NBLK : 1; };
  auto fetch = [&](const Unit& t, int j) {  // by lane 0, once the copies that left the block's staging have read it
    unsigned char* stg = stg0 + 2 * (j % SETS) * BLOCK_ST;
    uint64_t* bar = here + (j % SETS) * EPI_WARPS;
    mbar_arrive_expect_tx(bar, 2 * BLOCK_ST);
    tma_load_2d(stg, &maps.res, col_of(t) + 32 * j, row_of(t), bar);
    tma_load_2d(stg + BLOCK_ST, &maps.b2, col_of(t) + 32 * j, row_of(t), bar);
  };
  if (lane == 0)
    for (int j = 0; j < min(SETS, blocks_of(t)); ++j) fetch(t, j);
  int tl = 0;
  uint32_t phases = 0;  // of the stagings' barriers
  for (int u = first; u < units; ++tl) {
    const int acc = tl & 1, blocks = blocks_of(t);
    const int64_t m0 = row_of(t);
    const int nb = col_of(t);
    Unit next = t;
    const bool more = (u += step) < units;
    if (more) next = unit_of(a, u);
    const int then = more ? blocks_of(next) : 0;
    if (!wait_for(tfull + acc, (tl >> 1) & 1, abort)) break;
    __syncwarp();
    tc_fence_after();
#pragma unroll
    for (int j = 0; j < C::NBLK; ++j) {
      if (j >= blocks) break;
      const int n0 = nb + 32 * j;
      unsigned char* stg = stg0 + 2 * (j % SETS) * BLOCK_ST;
      uint32_t w[32];
      tmem_ld32(tbase + acc * BN + group * C::CW + j * 32 + ((uint32_t)(q * 32) << 16), w);
      tmem_ld_wait();
      if (j + 1 == blocks) give_back<CG>(tfree + acc);
      if (!wait_for(here + (j % SETS) * EPI_WARPS, phases >> (j % SETS) & 1, abort)) break;
      phases ^= 1u << (j % SETS);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4* at = reinterpret_cast<uint4*>(stg + h * BLOCK_ST + stg_at(lane, k));
          const uint4 r = *at;
          const uint32_t f[4] = {r.x, r.y, r.z, r.w};
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 c = unpack2<BF16>(f[i]);
            o[i] = pack2<BF16>(__uint_as_float(w[8 * k + 2 * i]) * c.x, __uint_as_float(w[8 * k + 2 * i + 1]) * c.y);
          }
          *at = make_uint4(o[0], o[1], o[2], o[3]);
        }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(&maps.out, n0, (int)m0, 0, stg);
        tma_store_3d(&maps.c2, n0, (int)m0, 0, stg + BLOCK_ST);
        bulk_commit();
      }
      if (a.part) {
        float* to = a.part + m0 / 32 * a.N + n0;
        column_sums<BF16>(stg, to, a.N - n0);
        column_sums<BF16>(stg + BLOCK_ST, to + (a.M + 31) / 32 * a.N, a.N - n0);
      }
      if constexpr (SETS > 1) {
        // the staging of the block before this one has been read by now, or soon
        if (j > 0 && lane == 0 && then > j - 1) {
          asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          fetch(next, j - 1);
        }
      } else if (lane == 0 && j + 1 < blocks) {
        bulk_wait_read();
        fetch(t, j + 1);
      }
      __syncwarp();
    }
    if (blocks == 0) give_back<CG>(tfree + acc);
    if (lane == 0) {
      // what is not asked for yet: the last block's, and all where this tile had none
      const int from = SETS == 1 || blocks == 0 ? 0 : blocks - 1, to = min(SETS, then);
      if (to > from) bulk_wait_read();
      for (int j = from; j < to; ++j) fetch(next, j);
    }
    __syncwarp();
    t = next;
  }
  if (lane == 0) bulk_wait_read();
}

template <int BN, int CG, bool AMN, bool BMN, bool BF16, int ACT, int KIND = PLAIN>
__global__ void __launch_bounds__(THREADS, 1) gemm_kernel(const __grid_constant__ MapsOf<KIND> maps, const GemmArgs a) {
  using C = GC<BN, CG, KIND>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tfree = tfull + 2;
  uint64_t* probe = tfree + 2;
  uint64_t* rbar = probe + 1;  // [EPI_WARPS] a warp's residual has landed; [2][EPI_WARPS] what GRAD's two blocks take
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
    if constexpr (KIND == GATE || KIND == CAT_K) prefetch_map(&maps.b2);
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
      int am0 = (t.mt * CG + (int)rank) * TM;
      const int bn0 = KIND == GATE ? t.nt * (BN / 2) : t.nt * BN + (int)rank * C::B_ROWS;
      const CUtensorMap *ma = &maps.a, *mb = &maps.b;
      if constexpr (KIND == CAT_M)
        if (t.mt >= a.half) {
          am0 -= a.half * CG * TM;
          ma = &maps.a2;
        }
      if constexpr (KIND == GATE && CG == 2)
        if (rank == 1) mb = &maps.b2;
      for (int kb = t.kb0; kb < t.kb1; ++kb) {
        if (turn > 0 && !wait_for(empty + s, (turn - 1) & 1, abort)) break;
        unsigned char* sa = sm + s * A_ST;
        unsigned char* sb = sm + C::OFF_B + s * C::B_ST;
        int k0 = kb * KE;
        if constexpr (KIND == CAT_K)
          if (kb >= a.half) {
            k0 -= a.half * KE;
            ma = &maps.a2;
            mb = &maps.b2;
          }
        if (one) {
          if (rank == 0) mbar_arrive_expect_tx(full + s, CG * (A_ST + C::B_ST));
          auto load = [&](void* dst, const CUtensorMap* map, int c0, int c1) {
            if constexpr (CG == 1) tma_load_2d(dst, map, c0, c1, full + s);
            else tma_load_2d_pair(dst, map, c0, c1, in_cta(full + s, 0));
          };
          if constexpr (AMN) {
#pragma unroll
            for (int i = 0; i < TM / 64; ++i) load(sa + i * 8192, ma, am0 + i * 64, k0);
          } else {
            load(sa, ma, k0, am0);
          }
          if constexpr (BMN) {
#pragma unroll
            for (int i = 0; i < C::B_ROWS / 64; ++i) load(sb + i * 8192, mb, bn0 + i * 64, k0);
          } else {
            load(sb, mb, k0, bn0);
            if constexpr (KIND == GATE && CG == 1) load(sb + BN / 2 * 128, &maps.b2, k0, bn0);
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
    if constexpr (KIND == GATE) gate_epilogue<BN, CG, BF16, ACT>(maps, a, t, rank, first, step, units, tbase, tfull, tfree, stg, abort);
    else if constexpr (is_grad(KIND)) grad_epilogue<BN, CG, BF16, KIND>(maps, a, t, rank, first, step, units, tbase, tfull, tfree, rbar + warp, stg, abort);
    else {
    const int q = warp & 3, group = warp >> 2;
    const Epi& e = a.e;
    int tl = 0, fetched = 0;
    for (int u = first; u < units; ++tl) {
      const int acc = tl & 1;
      int64_t m0 = (int64_t)(t.mt * CG + (int)rank) * TM + q * 32;
      const int nb = t.nt * BN + group * C::CW;
      const CUtensorMap* mo = &maps.out;
      void* out = e.out;
      int slice = t.split;
      if constexpr (KIND == CAT_M) {
        const bool second = t.mt >= a.half;
        if (second) m0 -= (int64_t)a.half * CG * TM;
        if (a.splits > 1) {
          slice = 2 * t.split + second;
        } else if (second) {
          mo = &maps.c2;
          out = a.out2;
        }
      }
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
        if (e.bias) add_bias(v, e.bias, e.bias_dt, n0, a.N);
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
        if (e.out32) put32(sj, v, mo, e.vo, (float*)out, e.ldo, m0, a.M, n0, a.N, slice);
        else put16(sj, v, BF16, mo, e.vo, out, e.ldo, m0, a.M, n0, a.N);
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
// blockIdx.y: the second of CAT_M's results, whose partials are ``second`` floats on.
__global__ void __launch_bounds__(256) gemm_sum_kernel(const float* __restrict__ part, int splits, int64_t stride, int64_t ld,
                                                       int64_t M, int N, Epi e, void* out2, int64_t second) {
  if (blockIdx.y) {
    part += second;
    e.out = out2;
  }
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

// What GATE's epilogue does with the two sums of one output.
struct Gate {
  const void* bias2;
  int bias2_dt;
  void* z2;          // u act'(g), beside e.z: act(g)
};
__device__ __forceinline__ float act_slope(float z, int act) {
  return act == OW_ACT_RELU   ? act_slope<OW_ACT_RELU>(z)
         : act == OW_ACT_SILU ? act_slope<OW_ACT_SILU>(z)
         : act == OW_ACT_GELU ? act_slope<OW_ACT_GELU>(z)
                              : 1.f;
}
__device__ __forceinline__ void finish_gate(const Epi& e, const Gate& g, float v, float w, int64_t m, int n, int bf) {
  if (e.bias) v += ld_any(e.bias, e.bias_dt, n);
  if (g.bias2) w += ld_any(g.bias2, g.bias2_dt, n);
  const float a = act_fwd(v, e.act, bf);
  if (e.z) {
    st16(e.z, m * e.ldz + n, bf, keep_z(a, bf));
    st16(g.z2, m * e.ldz + n, bf, keep_z(w * act_slope(v, e.act), bf));
  }
  st16(e.out, m * e.ldo + n, bf, a * w);
}

// The same for GATE's partials, whose rows hold tiles of ``bn`` columns, half of them of either product.
__global__ void __launch_bounds__(256) gate_sum_kernel(const float* __restrict__ part, int splits, int64_t stride, int64_t ld, int bn,
                                                       int64_t M, int N, const Epi e, const Gate g) {
  const int64_t total = M * N;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t m = i / N;
    const int n = (int)(i - m * N), h = bn / 2;
    const float* p = part + m * ld + n / h * bn + n % h;
    float v = 0.f, w = 0.f;
    for (int s = 0; s < splits; ++s) {
      v += p[s * stride];
      w += p[s * stride + h];
    }
    finish_gate(e, g, v, w, m, n, e.bf16);
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
struct GateRowsArgs : RowsArgs {
  const void* w2;
  int64_t ldw2;
  Gate g;
};
template <bool GATED>
using RowsOf = std::conditional_t<GATED, GateRowsArgs, RowsArgs>;

// One output from its sum: bias, the kept z, the activation, the residual.
__device__ __forceinline__ void finish_one(const Epi& e, float z, int64_t m, int n, int bf) {
  if (e.bias) z += ld_any(e.bias, e.bias_dt, n);
  if (e.z) st16(e.z, m * e.ldz + n, bf, keep_z(z, bf));
  z = act_fwd(z, e.act, bf);
  if (e.res) z += ld16(e.res, m * e.ldr + n, bf);
  st16(e.out, m * e.ldo + n, bf, z);
}

// Rows that are not 16-byte units.  Four warps share a feature (its k dealt out
// in turns of 32), a block of 8 warps does two; MR rows at once.  GATED: the
// block's two are a gate and its factor.
template <int MR, bool GATED = false>
__global__ void __launch_bounds__(256) linear_rows_kernel(const RowsOf<GATED> a) {
  __shared__ float sh[8][MR];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp & 3;
  const int n = GATED ? blockIdx.x : blockIdx.x * 2 + (warp >> 2);
  const int bf = a.e.bf16;
  float s[MR];
#pragma unroll
  for (int r = 0; r < MR; ++r) s[r] = 0.f;
  if (n < a.N) {
    const uint16_t* w = reinterpret_cast<const uint16_t*>(a.w) + n * a.ldw;
    if constexpr (GATED)
      if (warp >= 4) w = reinterpret_cast<const uint16_t*>(a.w2) + n * a.ldw2;
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
  if (part != 0 || lane >= MR || lane >= a.M || n >= a.N) return;
  auto sum = [&](int w0) { return ((sh[w0][lane] + sh[w0 + 1][lane]) + sh[w0 + 2][lane]) + sh[w0 + 3][lane]; };
  if constexpr (GATED) {
    if (warp == 0) finish_gate(a.e, a.g, sum(0), sum(4), lane, n, bf);
  } else {
    finish_one(a.e, sum(warp), lane, n, bf);
  }
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
// GATED: the 16 are 8 gates and the factors of these 8.
//
// On CUDA cores (a warp a feature) 8 rows of 4096 x 4096 took 38.7 us, here 8.7;
// one row 11.7 and 8.3; one row of 8192 x 8192 38.3 and 23.9 (5.6 TB/s).
constexpr int UNIT_WARPS = 8;
constexpr int unit_turns(int nb) { return nb == 1 ? 4 : nb == 2 ? 3 : 1; }

template <int NB, bool BF16, bool GATED = false>
__global__ void __launch_bounds__(UNIT_WARPS * 32) linear_units_kernel(const RowsOf<GATED> a) {
  constexpr int U = unit_turns(NB), warps = UNIT_WARPS, ROW = 8 * NB + 1;
  extern __shared__ float sh[];  // [warps][16][ROW], [8 NB][16]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * (GATED ? 8 : 16), units = a.K >> 3, splits = gridDim.y, all = warps * splits * 8;
  const uint16_t* w = reinterpret_cast<const uint16_t*>(a.w) + t * 8;
  const uint16_t* x = reinterpret_cast<const uint16_t*>(a.x) + t * 8;
  // features and rows past the end repeat the last; what they give is not stored
  const uint16_t* w0 = w + min(n0 + g, a.N - 1) * a.ldw;
  const uint16_t* w1 = w + min(n0 + g + 8, a.N - 1) * a.ldw;
  if constexpr (GATED) w1 = reinterpret_cast<const uint16_t*>(a.w2) + t * 8 + min(n0 + g, a.N - 1) * a.ldw2;
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
  if constexpr (GATED) {
    for (int i = threadIdx.x; i < 16 * a.M; i += warps * 32) {
      float z = 0.f;
#pragma unroll
      for (int p = 0; p < warps; ++p) z += sh[(p * 16 + (i & 15)) * ROW + (i >> 4)];
      sum[i] = z;
    }
    if (splits > 1) cluster_sync();
    else __syncthreads();
    if (blockIdx.y == 0)
      for (int i = threadIdx.x; i < 8 * a.M; i += warps * 32) {
        const int at = (i >> 3) * 16 + (i & 7), n = n0 + (i & 7);
        float v = sum[at], z = sum[at + 8];
#pragma unroll 4
        for (int p = 1; p < splits; ++p) {
          v += ld_in(in_cta(sum + at, p));
          z += ld_in(in_cta(sum + at + 8, p));
        }
        if (n < a.N) finish_gate(a.e, a.g, v, z, i >> 3, n, BF16);
      }
    if (splits > 1) cluster_sync();
    return;
  }
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

// blockIdx.y: the second of two arrays of partial sums.
__global__ void __launch_bounds__(1024) dbias_kernel(const float* __restrict__ part, int chunks, int N, void* out, int dt, void* out2 = nullptr,
                                                     int dt2 = 0) {
  __shared__ float sh[32][33];
  if (blockIdx.y) {
    part += (int64_t)chunks * N;
    out = out2;
    dt = dt2;
  }
  if (!out) return;
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

int blocks_of(int64_t k) { return (int)((k + KE - 1) / KE); }

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

template <int BN, int CG, bool AMN, bool BMN, bool BF16, int ACT, int KIND = PLAIN>
int run_gemm(const MapsOf<KIND>& maps, const GemmArgs& k, int grid, cudaStream_t st) {
  using C = GC<BN, CG, KIND>;
  auto kern = gemm_kernel<BN, CG, AMN, BMN, BF16, ACT, KIND>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) {
    set_error("ow_linear: cannot reserve %d bytes of shared memory: %s", C::SMEM, cudaGetErrorString(e));
    return OW_ERR_CUDA;
  }
  return launch_cluster("gemm_kernel", kern, dim3(grid), dim3(CG), THREADS, C::SMEM, st, maps, k);
}

// D[M, N] = sum_k A B with the epilogue ``e``.  AMN/BMN: the operand's rows
// run along M or N and its row index is k.  ``parts``: the f32 partials of a split
// product stay as they are, and there is no epilogue.
template <bool AMN, bool BMN>
int gemm(Mat A, Mat B, int64_t M, int N, int64_t K, const Plan& p, const GemmWs& w, const Epi& e, bool bf16, cudaStream_t st,
         bool parts = false) {
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
  if (p.splits > 1 && !parts) {
    const int64_t total = M * ((N + 3) / 4);
    const int g2 = (int)std::min<int64_t>((total + 255) / 256, (int64_t)device_sm_count() * 16);
    launch(gemm_sum_kernel, g2, 256, 0, st, (const float*)w.part, p.splits, M * w.part_ld, w.part_ld, M, N, e, nullptr, 0);
    OW_CHECK_LAUNCH("gemm_sum_kernel");
  }
  return OW_OK;
}

// A second product beside the first (GATE, CAT_K, CAT_M), with the arguments that come with it.
struct Second {
  Mat a, b;           // CAT_K both, CAT_M a, GATE b
  const void* bias;   // GATE
  int bias_dt;
  void* c;            // GATE: its z, beside e.z; CAT_M: its output; GRAD: d act(g), e.out being d u act'(g)
  const void* kept;   // GRAD: act(g) and u act'(g), rows of e.ldo, as the results'
  const void* kept2;
  float* part;        // GRAD: column sums, or NULL
};
struct DualWs {
  void *a, *b, *a2, *b2;
  float* part;
  int64_t part_ld;
};
// Columns of a GATE tile's partials, all of them.
int gate_cols(int N, int bn) { return (N + bn / 2 - 1) / (bn / 2) * bn; }

template <int KIND>
DualWs dual_take(const Mat& A, const Mat& B, const Second& s, int64_t M, int N, const Plan& p, Carver& ws) {
  DualWs w{};
  auto copy = [&](const Mat& m) { return tma_rows(m.p, m.ld) ? nullptr : ws.take((size_t)m.rows * up8(m.cols) * 2); };
  w.a = copy(A);
  w.b = copy(B);
  if (KIND == CAT_K || KIND == CAT_M) w.a2 = copy(s.a);
  if (KIND == CAT_K || KIND == GATE) w.b2 = copy(s.b);
  w.part_ld = KIND == GATE ? gate_cols(N, p.bn) : (N + 3) / 4 * 4;
  if (p.splits > 1) w.part = (float*)ws.take((size_t)p.splits * (KIND == CAT_M ? 2 : 1) * M * w.part_ld * 4);
  return w;
}

// The forms with a second product.  M and N are the size of one result, K of one product.
template <int KIND, bool AMN, bool BMN>
int gemm_dual(Mat A, Mat B, Second s, int64_t M, int N, int64_t K, const Plan& p, const DualWs& w, const Epi& e, bool bf16,
              cudaStream_t st) {
  if (w.a) OW_RETURN_IF(pad_rows(A, w.a, st));
  if (w.b) OW_RETURN_IF(pad_rows(B, w.b, st));
  if (w.a2) OW_RETURN_IF(pad_rows(s.a, w.a2, st));
  if (w.b2) OW_RETURN_IF(pad_rows(s.b, w.b2, st));
  Maps2 maps{};
  const uint32_t arows = AMN ? KE : TM, brows = BMN ? KE : KIND == GATE ? p.bn / 2 : p.bn / p.cg;
  OW_RETURN_IF(map_of(&maps.a, A, bf16, arows));
  OW_RETURN_IF(map_of(&maps.b, B, bf16, brows));
  if (KIND == CAT_K || KIND == CAT_M) OW_RETURN_IF(map_of(&maps.a2, s.a, bf16, arows));
  if (KIND == CAT_K || KIND == GATE) OW_RETURN_IF(map_of(&maps.b2, s.b, bf16, brows));
  GemmArgs k{};
  k.M = M;
  k.N = N;
  k.kblocks = blocks_of(K) * (KIND == CAT_K ? 2 : 1);
  k.mtiles = (int)((M + TM * p.cg - 1) / (TM * p.cg));
  k.ntiles = KIND == GATE ? (N + p.bn / 2 - 1) / (p.bn / 2) : (N + p.bn - 1) / p.bn;
  k.half = KIND == CAT_K ? k.kblocks / 2 : k.mtiles;
  if (KIND == CAT_M) k.mtiles *= 2;
  k.splits = p.splits;
  k.kq = k.kblocks / p.splits;
  k.kr = k.kblocks % p.splits;
  k.e = e;
  const int t16 = bf16 ? OW_DTYPE_BF16 : OW_DTYPE_F16;
  if (p.splits > 1) {
    k.e = Epi{};
    k.e.out = w.part;
    k.e.ldo = w.part_ld;
    k.e.out32 = 1;
    k.e.vo = 1;
    k.raw = 1;
    OW_RETURN_IF(block_map(&maps.out, OW_DTYPE_F32, w.part, M, KIND == GATE ? (int)w.part_ld : N, w.part_ld,
                           p.splits * (KIND == CAT_M ? 2 : 1)));
  } else {
    if (e.vo) OW_RETURN_IF(block_map(&maps.out, e.out32 ? OW_DTYPE_F32 : t16, e.out, M, N, e.ldo, 1));
    if (KIND == GATE) {
      k.bias2 = s.bias;
      k.bias2_dt = s.bias_dt;
      if (e.z) OW_RETURN_IF(block_map(&maps.z, t16, e.z, M, N, e.ldz, 1));
      if (e.z) OW_RETURN_IF(block_map(&maps.c2, t16, s.c, M, N, e.ldz, 1));
    }
    if (is_grad(KIND)) {
      k.part = s.part;
      OW_RETURN_IF(block_map(&maps.c2, t16, s.c, M, N, e.ldo, 1));
      OW_RETURN_IF(block_map(&maps.res, t16, s.kept2, M, N, e.ldo, 0));
      OW_RETURN_IF(block_map(&maps.b2, t16, s.kept, M, N, e.ldo, 0));
    }
    if (KIND == CAT_M) {
      k.out2 = s.c;
      if (e.vo) OW_RETURN_IF(block_map(&maps.c2, e.out32 ? OW_DTYPE_F32 : t16, s.c, M, N, e.ldo, 1));
    }
  }
  OW_RETURN_IF(fault_word(&k.fault));
  k.probe_ns = wait_probe_ns();
  const int64_t units = (int64_t)k.mtiles * k.ntiles * k.splits;
  OW_CHECK_ARG(units < (1LL << 31) - 1024, "ow_linear: too many tiles");
  const int grid = (int)std::min<int64_t>(units, device_sm_count() / p.cg) * p.cg;
  auto go = [&](auto act) -> int {
    constexpr int ACT = decltype(act)::value;
    auto tile = [&](auto bn, auto cg) -> int {
      constexpr int BN = decltype(bn)::value, CG = decltype(cg)::value;
      return bf16 ? run_gemm<BN, CG, AMN, BMN, true, ACT, KIND>(maps, k, grid, st) : run_gemm<BN, CG, AMN, BMN, false, ACT, KIND>(maps, k, grid, st);
    };
    if (p.cg == 2) return tile(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    if (p.bn == 64) return tile(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    return tile(std::integral_constant<int, 128>(), std::integral_constant<int, 1>());
  };
  if constexpr (KIND == GATE) {
    switch (e.act) {
      case OW_ACT_RELU: OW_RETURN_IF(go(std::integral_constant<int, OW_ACT_RELU>())); break;
      case OW_ACT_SILU: OW_RETURN_IF(go(std::integral_constant<int, OW_ACT_SILU>())); break;
      case OW_ACT_GELU: OW_RETURN_IF(go(std::integral_constant<int, OW_ACT_GELU>())); break;
      default: OW_RETURN_IF(go(std::integral_constant<int, OW_ACT_NONE>()));
    }
  } else {
    OW_RETURN_IF(go(std::integral_constant<int, OW_ACT_NONE>()));
  }
  if (p.splits > 1) {
    const int64_t stride = M * w.part_ld;
    auto blocks = [&](int64_t n) { return (int)std::min<int64_t>((n + 255) / 256, (int64_t)device_sm_count() * 16); };
    if (KIND == GATE) {
      launch(gate_sum_kernel, blocks(M * N), 256, 0, st, (const float*)w.part, p.splits, stride, w.part_ld, p.bn, M, N, e,
             Gate{s.bias, s.bias_dt, s.c});
    } else {
      const int both = KIND == CAT_M ? 2 : 1;
      launch(gemm_sum_kernel, dim3(blocks(M * ((N + 3) / 4)), both), 256, 0, st, (const float*)w.part, p.splits, stride * both, w.part_ld,
             M, N, e, s.c, stride);
    }
    OW_CHECK_LAUNCH("gemm_sum_kernel");
  }
  return OW_OK;
}

// The kernel for up to 32 rows of 16-byte units.
template <bool GATED>
int run_units(const RowsOf<GATED>& k, cudaStream_t st) {
  const int blocks = GATED ? (k.N + 7) / 8 : (k.N + 15) / 16;
  auto go = [&](auto nb, auto b16) -> int {
    constexpr int NB = decltype(nb)::value, W = UNIT_WARPS, turns = std::max(unit_turns(NB), 2);
    auto kern = linear_units_kernel<NB, decltype(b16)::value, GATED>;
    // A split costs 0.7 us (2048 -> 1024: 3.5 us whole, 3.9 in two), and pays where each
    // warp keeps the turns that it has under way at once (4096 -> 64: 4.5 whole, 4.0 in two).
    int splits = 1;
    while (splits < 8 && blocks * splits * 2 <= device_sm_count() && k.K >= 64 * W * turns * splits * 2) splits *= 2;
    const size_t smem = ((size_t)W * 16 * (8 * NB + 1) + 128 * NB) * 4;
    if (splits > 1)
      return launch_cluster("linear_units_kernel", kern, dim3(blocks, splits), dim3(1, splits), W * 32, smem, st, k);
    launch(kern, blocks, W * 32, smem, st, k);
    OW_CHECK_LAUNCH("linear_units_kernel");
    return OW_OK;
  };
  auto of = [&](auto nb) { return k.e.bf16 ? go(nb, std::true_type()) : go(nb, std::false_type()); };
  if (k.M <= 8) return of(std::integral_constant<int, 1>());
  if (k.M <= 16) return of(std::integral_constant<int, 2>());
  return of(std::integral_constant<int, 4>());
}
template <bool GATED>
int run_rows(const RowsOf<GATED>& k, cudaStream_t st) {
  auto go = [&](auto mr) -> int {
    launch(linear_rows_kernel<decltype(mr)::value, GATED>, GATED ? k.N : (k.N + 1) / 2, 256, 0, st, k);
    OW_CHECK_LAUNCH("linear_rows_kernel");
    return OW_OK;
  };
  if (k.M == 1) return go(std::integral_constant<int, 1>());
  if (k.M == 2) return go(std::integral_constant<int, 2>());
  return go(std::integral_constant<int, 4>());
}

bool is16(int dt) { return dt == OW_DTYPE_BF16 || dt == OW_DTYPE_F16; }


}  // namespace
}  // namespace ow
