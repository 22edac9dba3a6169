// The paged KV cache: layout, and what its kernels share.
//
// A pool has pages of `page_size` slots of every KV head, keys and values (page, KV head, slot, D) in fp16 or bf16: a head's slots
// of a page are one contiguous piece of memory (4 KB for 16 slots of 128 columns), which one bulk copy or a warp's 16-byte
// loads take whole; with the slot before the head it would be 256 bytes of every 256 * KV.  A table (sequences, width) of int32
// names the page of every page_size slots of a sequence; an entry outside the pool stands for no page.
#pragma once

#include <cuda_bf16.h>

#include "cq_kv4.cuh"

namespace cq_paged {

template <typename T> struct Type;
template <> struct Type<__half> {
  static __device__ __forceinline__ float2 apart(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ uint32_t pair(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float one(__half x) { return __half2float(x); }
};
template <> struct Type<__nv_bfloat16> {
  static __device__ __forceinline__ float2 apart(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
  static __device__ __forceinline__ uint32_t pair(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
};

// rows (tokens, heads, D): contiguous columns, strides in elements
template <typename T> struct Rows {
  const T* at;
  int64_t token, head;
  __device__ __forceinline__ const T* row(int64_t t, int h) const { return at + t * token + (int64_t)h * head; }
};
template <typename T> struct Pool {
  T *k, *v;
  int pages, heads, log_page;
  // the first slot of a page's head, in rows of D columns
  __device__ __forceinline__ size_t rows(int page, int head) const { return ((size_t)page * heads + head) << log_page; }
};
struct Table {
  const int* entries;
  int64_t stride;
  int width;
  // the page of a slot (0 <= slot), -1 where there is none
  template <typename P> __device__ __forceinline__ int page_of(const P& pool, int sequence, long long slot) const {
    const long long i = slot >> pool.log_page;
    const int page = i < width ? __ldg(entries + (int64_t)sequence * stride + i) : -1;
    return page >= 0 && page < pool.pages ? page : -1;
  }
};

// eight columns of the lower half of a head (x1) and the same of the upper half (x2), rotated: products and sums rounded one by
// one in fp32, then to the type, as rope_cache and the 4-bit cache leave a row
template <typename T> __device__ __forceinline__ void rotate8(uint4& x1, uint4& x2, const float* __restrict__ cos_p, const float* __restrict__ sin_p) {
  uint32_t* w1 = reinterpret_cast<uint32_t*>(&x1);
  uint32_t* w2 = reinterpret_cast<uint32_t*>(&x2);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = Type<T>::apart(w1[i]), b = Type<T>::apart(w2[i]);
    const float c0 = cos_p[2 * i], c1 = cos_p[2 * i + 1], s0 = sin_p[2 * i], s1 = sin_p[2 * i + 1];
    w1[i] = Type<T>::pair(__fsub_rn(__fmul_rn(a.x, c0), __fmul_rn(b.x, s0)), __fsub_rn(__fmul_rn(a.y, c1), __fmul_rn(b.y, s1)));
    w2[i] = Type<T>::pair(__fadd_rn(__fmul_rn(b.x, c0), __fmul_rn(a.x, s0)), __fadd_rn(__fmul_rn(b.y, c1), __fmul_rn(a.y, s1)));
  }
}

template <typename T> Pool<T> pool_of(const cq_pages* p) {
  int log_page = 4;
  while ((1 << log_page) < p->page_size) ++log_page;
  return Pool<T>{(T*)p->k, (T*)p->v, p->pages, p->n_kv_heads, log_page};
}
inline Table table_of(const cq_table* t) { return Table{t->entries, t->stride, t->width}; }
template <typename T> Rows<T> rows_of(const cq_rows* r) { return r ? Rows<T>{(const T*)r->at, r->token_stride, r->head_stride} : Rows<T>{}; }

inline bool rows_fit(const cq_rows* r) {
  return r && r->at && ((uintptr_t)r->at & 15) == 0 && r->token_stride >= 0 && r->head_stride >= 0 && r->token_stride % 8 == 0 && r->head_stride % 8 == 0;
}
// no tables, or all of them
inline bool tables_fit(const float* cos_t, const float* sin_t, const long long* positions, int rows) {
  return !cos_t || (sin_t && positions && rows > 0 && (((uintptr_t)cos_t | (uintptr_t)sin_t) & 3) == 0 && ((uintptr_t)positions & 7) == 0);
}
int check(const cq_pages* pages, const cq_table* table);

}  // namespace cq_paged
