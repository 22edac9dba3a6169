// The 4-bit KV cache: layout of a row, and what its kernels share.
//
// A row is one slot of one KV head: D codes of four bits, D / 2 bytes, the even column of a byte in its low half, and for
// every group of GROUP columns a pair of fp16 numbers (scale, minimum); a column stands for scale * code + minimum.  Codes
// are (sequence, KV head, slot, D / 2) and scales (sequence, KV head, slot, D / GROUP, 2): a head's slots lie one behind the
// other, so that any run of them is one contiguous piece of memory (in the order of the fp16 cache, slot before head, a head
// would own 64 of every 64 * KV bytes, and 16 of its scales).
#pragma once

#include "cq_common.cuh"

// Quantises one row that LANES = D / 16 neighbouring lanes hold, 8 columns of the lower half of the head and the same 8 of the
// upper half each (x[0..7] at 8 * lane, x[8..15] at D / 2 + 8 * lane; fp16 numbers).  minimum = min x, scale =
// fp16((max x - minimum) / 15), code = rint((x - minimum) / scale) within 0..15, and 0 where the scale is 0.  A group with an
// infinite or NaN column cannot be kept in 4 bits: it is NaN as a whole (scale 0, minimum NaN), so that nothing finite comes
// of it.  words: the two words of codes; pairs: scale | minimum << 16 of the groups of the two halves.
template <int D, int GROUP>
__device__ __forceinline__ void kv4_quantise(const float (&x)[16], uint32_t (&words)[2], uint32_t (&pairs)[2]) {
  constexpr int LANES = D / 16;
  constexpr bool WHOLE = GROUP == D;                       // a group spans both halves
  constexpr int REACH = GROUP / 8 < LANES ? GROUP / 8 : LANES;
  float lo[2], hi[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    lo[h] = INFINITY;
    hi[h] = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = x[8 * h + e];
      lo[h] = fminf(lo[h], v);
      hi[h] = fabsf(v) < INFINITY ? fmaxf(hi[h], v) : INFINITY;        // (NaN too; fmaxf keeps the infinity)
    }
  }
  if (WHOLE) {
    lo[0] = lo[1] = fminf(lo[0], lo[1]);
    hi[0] = hi[1] = fmaxf(hi[0], hi[1]);
  }
#pragma unroll
  for (int h = 0; h < (WHOLE ? 1 : 2); ++h)
#pragma unroll
    for (int d = 1; d < REACH; d *= 2) {
      lo[h] = fminf(lo[h], __shfl_xor_sync(0xffffffffu, lo[h], d));
      hi[h] = fmaxf(hi[h], __shfl_xor_sync(0xffffffffu, hi[h], d));
    }
  if (WHOLE) {
    lo[1] = lo[0];
    hi[1] = hi[0];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bool bad = hi[h] == INFINITY;
    const __half s16 = bad ? __ushort_as_half(0) : __float2half_rn(__fdiv_rn(__fsub_rn(hi[h], lo[h]), 15.f));
    const float s = __half2float(s16);
    pairs[h] = (uint32_t)__half_as_ushort(s16) | (bad ? 0x7FFF0000u : (uint32_t)__half_as_ushort(__float2half_rn(lo[h])) << 16);
    uint32_t w = 0;
    if (s > 0.f) {
      // the quotient as the division rounds it, by one residual step after the product with the reciprocal (Markstein)
      const float inv = __frcp_rn(s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = __fsub_rn(x[8 * h + e], lo[h]), q = __fmul_rn(d, inv), u = fminf(__fmaf_rn(__fmaf_rn(-q, s, d), inv, q), 15.f);
        // (rounded to a whole number, half to even, by adding 1.5 * 2^23)
        w |= (__float_as_uint(__fadd_rn(u, 12582912.f)) & 15u) << (4 * e);
      }
    }
    words[h] = w;
  }
}

// sixteen fp16 columns as kv4_quantise takes them, rotated by the angles of cos_p / sin_p (8 columns of the lower half):
// products and sums rounded one by one, then to fp16, as rope_cache leaves a row
__device__ __forceinline__ void kv4_rotate(float (&x)[16], const float* __restrict__ cos_p, const float* __restrict__ sin_p) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = x[e], b = x[8 + e], c = cos_p[e], s = sin_p[e];
    x[e] = __half2float(__float2half_rn(__fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s))));
    x[8 + e] = __half2float(__float2half_rn(__fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s))));
  }
}

__device__ __forceinline__ void kv4_load16(const __half* lower, const __half* upper, float (&x)[16]) {
  const uint4 a = *reinterpret_cast<const uint4*>(lower), b = *reinterpret_cast<const uint4*>(upper);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ uint4 kv4_halves(const float* x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename... KArgs, typename... Args>
cudaError_t kv4_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
