// What the kernels for 4-bit weights share.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "m3_kernels.cuh"
#include "m3_lm.cuh"

namespace m3 {

struct W4Params {
  int M, N, K, tiles, blocks;  // tiles: 128-column tiles, blocks: 16-row blocks
  int wk, wn;                   // warps along K, row blocks at a time, of a CTA (m3_w4.cu)
  int mtiles;                   // batch tiles
  const void *x;
  int64_t ldx;
  int x_vec;  // every row of x starts on 16 bytes
  const uint4 *codes;
  uint32_t mask, magic;  // constants of w4_pair
  const void *scales;
  int64_t s_ld;
  int s_bf16, groups;
  const uint8_t *zeros;
  int64_t z_ld;
  void *y;
  int64_t ldy;
  int y_bf16;
};

// pair i of a word as bf16 (q - z), with zz = (128 + z, 128 + z): 128 + q is
// the bf16 whose mantissa ends in q, and the difference is exact
// (mask 0x000F000F and magic 0x43004300 are kernel parameters: as immediates
// the and and the or would be two instructions)
__device__ __forceinline__ uint32_t w4_pair(uint32_t w, int i, uint32_t zz, uint32_t mask, uint32_t magic) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w >> (4 * i)), "r"(mask), "r"(magic));  // (a & b) | c
  __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162 *>(&v), *reinterpret_cast<__nv_bfloat162 *>(&zz));
  return *reinterpret_cast<uint32_t *>(&d);
}

// 8 consecutive elements of a batch row as bf16 terms: one for bf16 x, three
// for fp32 x (head, middle, rest; each the truncation of what is left).  The
// 24 bits of an x of 2^-110 or more end at or above bf16's smallest subnormal
// number, 2^-133, so head + middle + rest is x; of a smaller x what lies below
// that is dropped.  An infinite x is its head alone.
template <typename XT>
struct W4X;

template <>
struct W4X<__nv_bfloat16> {
  static constexpr int kTerms = 1;
  uint4 t[1];
  __device__ __forceinline__ void load(const void *x, int64_t row, int k, int K, bool vec) {
    const __nv_bfloat16 *p = static_cast<const __nv_bfloat16 *>(x) + row + k;
    if (vec && k + 8 <= K) {
      t[0] = *reinterpret_cast<const uint4 *>(p);
      return;
    }
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? (uint32_t)__bfloat16_as_ushort(p[i]) : 0u;
    t[0] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
  __device__ __forceinline__ void zero() { t[0] = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void terms(uint4 (&o)[1]) const { o[0] = t[0]; }
};

template <>
struct W4X<float> {
  static constexpr int kTerms = 3;
  float v[8];
  __device__ __forceinline__ void load(const void *x, int64_t row, int k, int K, bool vec) {
    const float *p = static_cast<const float *>(x) + row + k;
    if (vec && k + 8 <= K) {
      const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? p[i] : 0.f;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
  __device__ __forceinline__ void terms(uint4 (&o)[3]) const {
    uint32_t h[8], m[8], l[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[i] = __float_as_uint(v[i]);
      const float r = isinf(v[i]) ? 0.f : v[i] - __uint_as_float(h[i] & 0xffff0000u);
      m[i] = __float_as_uint(r);
      l[i] = __float_as_uint(r - __uint_as_float(m[i] & 0xffff0000u));
    }
    auto pack = [](const uint32_t (&b)[8]) {
      return make_uint4(__byte_perm(b[0], b[1], 0x7632), __byte_perm(b[2], b[3], 0x7632),
                        __byte_perm(b[4], b[5], 0x7632), __byte_perm(b[6], b[7], 0x7632));
    };
    o[0] = pack(h), o[1] = pack(m), o[2] = pack(l);
  }
};

__device__ __forceinline__ void w4_store(const W4Params &p, int m, int n, float s) {
  if (p.y_bf16)
    static_cast<__nv_bfloat16 *>(p.y)[(int64_t)m * p.ldy + n] = __float2bfloat16_rn(s);
  else
    static_cast<float *>(p.y)[(int64_t)m * p.ldy + n] = s;
}

// The kernel for many batch rows of a bf16 x (m3_w4_tc.cu); not taken: x is
// laid out as TMA does not read it.
cudaError_t launch_w4_tc(const W4Params &p, int group, cudaStream_t stream, bool *taken);

}  // namespace m3
