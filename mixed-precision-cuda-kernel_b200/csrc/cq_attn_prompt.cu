// Attention of prompts, causal, with a sliding window and first keys that stay visible, grouped heads and ragged lengths; and
// the weight that every key received from a prompt's last queries.  In the reference it is torch's attention without window
// or lengths (llama/modeling_llama_quant.py:371-419 of the reference project).
//
//   p = i + keys - queries;  visible(i, j): j <= p, j < length, and (no window, or j < sinks, or j > p - window)
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,  lse_i = ln sum_j exp(scale q_i . k_j)
//   weights_j = sum of exp(scale q_i . k_j - lse_i) over the observed queries i of the KV head
//
// mma.sync tiles: 64 queries of a head against 64 keys at a time, four warps of 16 queries, a running maximum and sum per row.
#include <algorithm>

#include "cq_kv4.cuh"

namespace {

constexpr int PR_THREADS = 128, PR_TILE = 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct PromptArgs {
  cq_prompt s;
  const __half *q, *k, *v;
  const long long* lengths;
};

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const __half* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_at(p)));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const __half* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_at(p)));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 64 rows of D halves into shared memory (row stride D + 8); rows from `rows` on are zeros
template <int D>
__device__ __forceinline__ void load_tile(__half* to, const __half* src, long long stride, int rows) {
  for (int i = threadIdx.x; i < PR_TILE * (D / 8); i += PR_THREADS) {
    const int r = i / (D / 8), c = 8 * (i % (D / 8));
    *reinterpret_cast<uint4*>(to + r * (D + 8) + c) = r < rows ? *reinterpret_cast<const uint4*>(src + r * stride + c) : make_uint4(0, 0, 0, 0);
  }
}
__device__ __forceinline__ bool sees(const cq_prompt& s, int pos, int key, int n) {
  return key <= pos && key < n && pos < n && (!s.window || key < s.sinks || key > pos - s.window);
}
__device__ __forceinline__ int length_of(const PromptArgs& a, int b) {
  if (!a.lengths) return a.s.keys;
  const long long n = a.lengths[b];
  return n < 0 ? 0 : (n > a.s.keys ? a.s.keys : (int)n);
}
// scores of this warp's 16 queries (fragments qf) against the 64 keys in shared memory, not scaled
template <int D>
__device__ __forceinline__ void scores64(float (&s)[8][4], const uint32_t (&qf)[D / 16][4], const __half* s_k, int lane) {
#pragma unroll
  for (int nt = 0; nt < 8; ++nt) {
    s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int kc = 0; kc < D / 16; kc += 2) {
      uint32_t r[4];
      ldsm4(r, s_k + (8 * nt + (lane & 7)) * (D + 8) + 16 * kc + 8 * (lane >> 3));
      mma16816(s[nt], qf[kc], r[0], r[1]);
      mma16816(s[nt], qf[kc + 1], r[2], r[3]);
    }
  }
}
template <int D>
__device__ __forceinline__ void query_fragments(uint32_t (&qf)[D / 16][4], const __half* s_q, int warp, int lane) {
#pragma unroll
  for (int kc = 0; kc < D / 16; ++kc) ldsm4(qf[kc], s_q + (16 * warp + (lane & 15)) * (D + 8) + 16 * kc + 8 * (lane >> 4));
}

template <int D>
__global__ void __launch_bounds__(PR_THREADS) prompt_kernel(const __grid_constant__ PromptArgs a, __half* __restrict__ out, float* __restrict__ lse) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ __align__(16) __half s_k[PR_TILE * (D + 8)], s_v[PR_TILE * (D + 8)];
  const cq_prompt& s = a.s;
  const int q0 = blockIdx.x * PR_TILE, h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kvh = h / (s.n_heads / s.n_kv_heads), off = s.keys - s.queries, n = length_of(a, b);
  const int rows = min(PR_TILE, s.queries - q0), pmin = q0 + off, pmax = pmin + rows - 1;
  uint32_t qf[D / 16][4];
  load_tile<D>(s_k, a.q + b * s.q_strides[0] + (long long)q0 * s.q_strides[1] + h * s.q_strides[2], s.q_strides[1], rows);
  __syncthreads();
  query_fragments<D>(qf, s_k, warp, lane);
  float o[D / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {};
  const float scale2 = s.scale * LOG2E;
  const int r0 = pmin + 16 * warp + (lane >> 2);           // positions r0 and r0 + 8
  const int end = pmin < n ? min(n, pmax + 1) : 0;
  for (int k0 = 0; k0 < end; k0 += PR_TILE) {
    if (s.window && k0 >= s.sinks && k0 + PR_TILE - 1 <= pmin - s.window) continue;
    __syncthreads();
    const __half* ks = a.k + b * s.k_strides[0] + (long long)k0 * s.k_strides[1] + kvh * s.k_strides[2];
    const __half* vs = a.v + b * s.v_strides[0] + (long long)k0 * s.v_strides[1] + kvh * s.v_strides[2];
    load_tile<D>(s_k, ks, s.k_strides[1], n - k0);
    load_tile<D>(s_v, vs, s.v_strides[1], n - k0);
    __syncthreads();
    float sc[8][4];
    scores64<D>(sc, qf, s_k, lane);
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = k0 + 8 * nt + 2 * (lane & 3) + (e & 1);
        sc[nt][e] = sees(s, r0 + 8 * (e >> 1), key, n) ? sc[nt][e] * scale2 : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], sc[nt][e]);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      const float ref = top[i] == -INFINITY ? 0.f : top[i], keep = exp2f(m[i] - ref);
      m[i] = top[i];
      l[i] *= keep;
#pragma unroll
      for (int nt = 0; nt < D / 8; ++nt) {
        o[nt][2 * i] *= keep;
        o[nt][2 * i + 1] *= keep;
      }
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int e = 2 * i; e < 2 * i + 2; ++e) {
          sc[nt][e] = exp2f(sc[nt][e] - ref);
          l[i] += sc[nt][e];
        }
    }
#pragma unroll
    for (int kc = 0; kc < 4; ++kc) {
      const uint32_t p[4] = {half_pair(sc[2 * kc][0], sc[2 * kc][1]), half_pair(sc[2 * kc][2], sc[2 * kc][3]),
                             half_pair(sc[2 * kc + 1][0], sc[2 * kc + 1][1]), half_pair(sc[2 * kc + 1][2], sc[2 * kc + 1][3])};
#pragma unroll
      for (int nt = 0; nt < D / 8; nt += 2) {
        uint32_t r[4];
        ldsm4t(r, s_v + (16 * kc + (lane & 15)) * (D + 8) + 8 * (nt + (lane >> 4)));
        mma16816(o[nt], p, r[0], r[1]);
        mma16816(o[nt + 1], p, r[2], r[3]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    const int r = q0 + 16 * warp + (lane >> 2) + 8 * i;
    if (r >= s.queries) continue;
    const bool empty = m[i] == -INFINITY && l[i] == 0.f;
    const float inv = empty ? 0.f : 1.f / l[i];
    __half* to = out + (((size_t)b * s.queries + r) * s.n_heads + h) * D + 2 * (lane & 3);
#pragma unroll
    for (int nt = 0; nt < D / 8; ++nt)
      *reinterpret_cast<uint32_t*>(to + 8 * nt) = empty ? 0u : half_pair(o[nt][2 * i] * inv, o[nt][2 * i + 1] * inv);
    if ((lane & 3) == 0) lse[((size_t)b * s.n_heads + h) * s.queries + r] = empty ? -INFINITY : ((m[i] == -INFINITY ? 0.f : m[i]) + log2f(l[i])) * LN2;
  }
}

// 64 keys of a KV head, all its query heads and observed queries one after another
template <int D>
__global__ void __launch_bounds__(PR_THREADS) prompt_weights_kernel(const __grid_constant__ PromptArgs a, const float* __restrict__ lse, int observe,
                                                                    float* __restrict__ weights) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ __align__(16) __half s_k[PR_TILE * (D + 8)], s_q[PR_TILE * (D + 8)];
  __shared__ float s_sum[4][PR_TILE];
  const cq_prompt& s = a.s;
  const int k0 = blockIdx.x * PR_TILE, kvh = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = s.n_heads / s.n_kv_heads, off = s.keys - s.queries, n = length_of(a, b);
  load_tile<D>(s_k, a.k + b * s.k_strides[0] + (long long)k0 * s.k_strides[1] + kvh * s.k_strides[2], s.k_strides[1], n - k0);
  const float scale2 = s.scale * LOG2E;
  float sum[8][2] = {};
  // positions of the queries that count: the observed ones from this tile's first key on, and within its last key's window
  const int first = max(max(off, n - observe), k0);
  const int last = s.window && k0 >= s.sinks ? min(n, min(k0 + PR_TILE, n) - 1 + s.window) : n;
  for (int g = 0; g < G; ++g)
    for (int p0 = first; p0 < last; p0 += PR_TILE) {
      const int h = kvh * G + g, q0 = p0 - off;
      __syncthreads();
      load_tile<D>(s_q, a.q + b * s.q_strides[0] + (long long)q0 * s.q_strides[1] + h * s.q_strides[2], s.q_strides[1], last - p0);
      __syncthreads();
      uint32_t qf[D / 16][4];
      query_fragments<D>(qf, s_q, warp, lane);
      float sc[8][4];
      scores64<D>(sc, qf, s_k, lane);
      float ref[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int p = p0 + 16 * warp + (lane >> 2) + 8 * i;
        ref[i] = p < last ? lse[((size_t)b * s.n_heads + h) * s.queries + p - off] * LOG2E : 0.f;
      }
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = k0 + 8 * nt + 2 * (lane & 3) + (e & 1), p = p0 + 16 * warp + (lane >> 2) + 8 * (e >> 1);
          if (p < last && sees(s, p, key, n)) sum[nt][e & 1] += exp2f(sc[nt][e] * scale2 - ref[e >> 1]);
        }
    }
#pragma unroll
  for (int nt = 0; nt < 8; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      for (int d = 4; d < 32; d *= 2) sum[nt][e] += __shfl_xor_sync(0xffffffffu, sum[nt][e], d);
      if (lane < 4) s_sum[warp][8 * nt + 2 * lane + e] = sum[nt][e];
    }
  __syncthreads();
  if (threadIdx.x < PR_TILE && k0 + threadIdx.x < s.keys)
    weights[((size_t)b * s.n_kv_heads + kvh) * s.keys + k0 + threadIdx.x] =
        (s_sum[0][threadIdx.x] + s_sum[1][threadIdx.x]) + (s_sum[2][threadIdx.x] + s_sum[3][threadIdx.x]);
}

int check(const cq_prompt* s, const void* q, const void* k, const void* v) {
  if (!s || !q || !k || (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) || s->window < 0 || s->sinks < 0) return CQ_ERR_BAD_ARG;
  if (s->sequences < 1 || s->sequences > 65535 || s->queries < 1 || s->keys < s->queries || s->keys > (1 << 24) || s->n_kv_heads < 1 ||
      s->n_heads < 1 || s->n_heads > 65535 || s->n_heads % s->n_kv_heads)
    return CQ_ERR_BAD_SHAPE;
  if (s->head_dim != 64 && s->head_dim != 128) return CQ_ERR_UNSUPPORTED;
  for (int i = 0; i < 3; ++i)
    if ((s->q_strides[i] | s->k_strides[i] | (v ? s->v_strides[i] : 0)) & 7) return CQ_ERR_BAD_ARG;
  return CQ_OK;
}

}  // namespace

extern "C" int cq_attn_prefill(const cq_prompt* shape, const void* q, const void* k, const void* v, const long long* lengths, void* out,
                               float* lse, cq_stream_t stream) {
  const int rc = check(shape, q, k, v);
  if (rc != CQ_OK) return rc;
  if (!v || !out || !lse || ((uintptr_t)out & 15)) return CQ_ERR_BAD_ARG;
  const PromptArgs a = {*shape, (const __half*)q, (const __half*)k, (const __half*)v, lengths};
  auto fn = shape->head_dim == 128 ? prompt_kernel<128> : prompt_kernel<64>;
  CQ_CUDA_TRY(kv4_launch(fn, dim3((shape->queries + PR_TILE - 1) / PR_TILE, shape->n_heads, shape->sequences), dim3(PR_THREADS), 0,
                         (cudaStream_t)stream, a, (__half*)out, lse));
  return CQ_OK;
}

extern "C" int cq_attn_prefill_weights(const cq_prompt* shape, const void* q, const void* k, const float* lse, const long long* lengths,
                                       int observe, float* weights, cq_stream_t stream) {
  const int rc = check(shape, q, k, nullptr);
  if (rc != CQ_OK) return rc;
  if (!lse || !weights || observe < 1) return CQ_ERR_BAD_ARG;
  const PromptArgs a = {*shape, (const __half*)q, (const __half*)k, nullptr, lengths};
  auto fn = shape->head_dim == 128 ? prompt_weights_kernel<128> : prompt_weights_kernel<64>;
  CQ_CUDA_TRY(kv4_launch(fn, dim3((shape->keys + PR_TILE - 1) / PR_TILE, shape->n_kv_heads, shape->sequences), dim3(PR_THREADS), 0,
                         (cudaStream_t)stream, a, lse, observe, weights));
  return CQ_OK;
}
