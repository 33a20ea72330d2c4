// What the kernels over rows of channels share: vectors of a storage type as
// floats, and sums over the threads of a row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "omniwave_b200.h"

namespace ow {

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

}  // namespace ow
