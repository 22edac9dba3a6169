// The 4-bit KV cache: layout of a row, and what its kernels share.
//
// A row is one slot of one KV head: D codes of four bits, D / 2 bytes, the even column of a byte in its low half, and for
// every group of GROUP columns a pair of fp16 numbers (scale, minimum); a column stands for scale * code + minimum.  Codes
// are (sequence, KV head, slot, D / 2) and scales (sequence, KV head, slot, D / GROUP, 2): a head's slots lie one behind the
// other, so that any run of them is one contiguous piece of memory (in the order of the fp16 cache, slot before head, a head
// would own 64 of every 64 * KV bytes, and 16 of its scales).
#pragma once

#include "cq_common.cuh"

// pairs of fp32 numbers in one instruction
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 apart(uint64_t a) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint32_t kv4_pair(uint64_t x) {
  const float2 f = apart(x);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint64_t kv4_two(uint32_t h) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return two(f.x, f.y);
}
__device__ __forceinline__ uint32_t kv4_min2(uint32_t a, uint32_t b) {      // NaN where one is
  const __half2 m = __hmin2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t kv4_max2(uint32_t a, uint32_t b) {
  const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

// Quantises one row that LANES = D / 16 neighbouring lanes hold, 8 columns of the lower half of the head and the same 8 of the
// upper half each (x[0..3] at 8 * lane, x[4..7] at D / 2 + 8 * lane, two fp16 numbers a word).  minimum = min x, scale =
// fp16((max x - minimum) / 15) (the fp16 number below it where 15 of them would leave fp16), code = rint((x - minimum) / scale)
// within 0..15, and 0 where the scale is 0.  A group with an
// infinite or NaN column cannot be kept in 4 bits: it is NaN as a whole (scale 0, minimum NaN), so that nothing finite comes
// of it.  words: the two words of codes; pairs: scale | minimum << 16 of the groups of the two halves.
template <int D, int GROUP>
__device__ __forceinline__ void kv4_quantise(const uint32_t (&x)[8], uint32_t (&words)[2], uint32_t (&pairs)[2]) {
  constexpr int LANES = D / 16;
  constexpr bool WHOLE = GROUP == D;                       // a group spans both halves
  constexpr int REACH = GROUP / 8 < LANES ? GROUP / 8 : LANES;
  uint32_t ends[2];                                        // (-min, max)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = kv4_min2(kv4_min2(x[4 * h], x[4 * h + 1]), kv4_min2(x[4 * h + 2], x[4 * h + 3]));
    const uint32_t hi = kv4_max2(kv4_max2(x[4 * h], x[4 * h + 1]), kv4_max2(x[4 * h + 2], x[4 * h + 3]));
    ends[h] = kv4_max2(__byte_perm(lo, hi, 0x5410) ^ 0x8000u, __byte_perm(lo, hi, 0x7632) ^ 0x8000u);
  }
  if (WHOLE) ends[0] = kv4_max2(ends[0], ends[1]);
#pragma unroll
  for (int h = 0; h < (WHOLE ? 1 : 2); ++h)
#pragma unroll
    for (int d = 1; d < REACH; d *= 2) ends[h] = kv4_max2(ends[h], __shfl_xor_sync(0xffffffffu, ends[h], d));
  if (WHOLE) ends[1] = ends[0];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bool bad = (ends[h] & 0x7C00u) == 0x7C00u || (ends[h] & 0x7C000000u) == 0x7C000000u;
    const float2 e = __half22float2(*reinterpret_cast<const __half2*>(&ends[h]));      // (-min, max)
    // Quotients as the division rounds them, by one residual step after the product with the reciprocal (Markstein).
    const float range = __fadd_rn(e.y, e.x), q15 = __fmul_rn(range, 1.f / 15.f);
    const __half near16 = __float2half_rn(__fmaf_rn(__fmaf_rn(-q15, 15.f, range), 1.f / 15.f, q15));
    // code 15 would stand for 65520 or more, which fp16 rounds to infinity: the next lower scale is below range / 15
    const bool beyond = __fmaf_rn(15.f, __half2float(near16), -e.x) >= 65520.f;
    const __half s16 = __ushort_as_half(bad ? 0 : (unsigned short)(__half_as_ushort(near16) - beyond));
    const float s = __half2float(s16);
    pairs[h] = (uint32_t)__half_as_ushort(s16) | (bad ? 0x7FFF0000u : (ends[h] ^ 0x8000u) << 16);
    uint32_t w = 0;
    if (s > 0.f) {
      const float inv = __frcp_rn(s);
      const uint64_t inv2 = two(inv, inv), s2 = two(-s, -s), low2 = two(e.x, e.x), whole = two(12582912.f, 12582912.f);
      uint32_t b[8];
      // 1.5 * 2^23 + code, rounded to a whole number, half to even, by the addition.  Beyond 15 only where the scale, below
      // fp16's normal numbers, was rounded by more than 2^-11 of it.
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t d = add2(kv4_two(x[4 * h + i]), low2), q = mul2(d, inv2), u = fma2(fma2(q, s2, d), inv2, q);
        const float2 r = apart(add2(u, whole));
        b[2 * i] = __float_as_uint(r.x);
        b[2 * i + 1] = __float_as_uint(r.y);
      }
      if (s < 6.103515625e-05f)
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = min(b[i], 0x4B40000Fu);
#pragma unroll
      for (int i = 7; i >= 0; --i) w = 16u * w + b[i];     // modulo 2^32: the exponents' part is one constant
      w -= 0x4B400000u * 0x11111111u;
    }
    words[h] = w;
  }
}

// sixteen fp16 columns as kv4_quantise takes them, rotated by the angles of cos_p / sin_p (8 columns of the lower half):
// products and sums rounded one by one, then to fp16, as rope_cache leaves a row.  PAIRS: the tables start on 8 bytes (any 4 will do
// without; rows of a prompt 24 us with, the single tokens' kernel is the same either way and reads them one by one)
template <bool PAIRS>
__device__ __forceinline__ void kv4_rotate(uint32_t (&x)[8], const float* __restrict__ cos_p, const float* __restrict__ sin_p) {
  const uint64_t minus = two(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t a = kv4_two(x[i]), b = kv4_two(x[4 + i]);
    float2 cf, sf;
    if (PAIRS) cf = reinterpret_cast<const float2*>(cos_p)[i], sf = reinterpret_cast<const float2*>(sin_p)[i];
    else cf = make_float2(cos_p[2 * i], cos_p[2 * i + 1]), sf = make_float2(sin_p[2 * i], sin_p[2 * i + 1]);
    const uint64_t c = two(cf.x, cf.y), s = two(sf.x, sf.y);
    x[i] = kv4_pair(fma2(mul2(b, s), minus, mul2(a, c)));
    x[4 + i] = kv4_pair(add2(mul2(b, c), mul2(a, s)));
  }
}

__device__ __forceinline__ void kv4_load16(const __half* lower, const __half* upper, uint32_t (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(lower), b = *reinterpret_cast<const uint4*>(upper);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
  x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
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

// whether a and b, that many bytes each, share none
inline bool kv4_apart(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
  return (uintptr_t)a + a_bytes <= (uintptr_t)b || (uintptr_t)b + b_bytes <= (uintptr_t)a;
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
