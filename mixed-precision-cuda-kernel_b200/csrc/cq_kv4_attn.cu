// Attention of single tokens over the 4-bit KV cache (layout: cq_kv4.cuh), with a sliding window and first slots that stay
// visible, and the weight that every slot received.  In the reference the cache is fp16 and attention torch's
// (llama/modeling_llama_quant.py:371-419 of the reference project).
//
//   out = sum_j p_j v_j,  p = softmax over the visible slots j of scale * q . k_j,
//   visible: j < n and (no window, or j < sinks, or j >= n - window)
//
// One CTA per query head, a warp per slot: dot product by shuffles, running maximum and sum per warp, the warps meet in
// shared memory.
#include <algorithm>

#include "cq_kv4.cuh"

namespace {

constexpr int AT_THREADS = 256, AT_WARPS = AT_THREADS / 32;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ int held(const long long* length, int b, int more, int slots) {
  const long long n = length[b];
  return n < 0 ? 0 : (n + more > slots ? slots : (int)n + more);
}

template <int D>
__global__ void __launch_bounds__(AT_THREADS) kv4_attend_kernel(const __half* __restrict__ q, cq_kv4 cache,
                                                                const long long* __restrict__ length, int more, __half* __restrict__ out,
                                                                float* __restrict__ scores, float2* __restrict__ stats, int H, int window,
                                                                int sinks, float scale) {
  constexpr int CPL = D / 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float s_o[AT_WARPS][D], s_m[AT_WARPS], s_l[AT_WARPS];
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int KV = cache.n_kv_heads, groups = D / cache.group, n = held(length, b, more, cache.slots);
  const size_t head = (size_t)b * KV + h / (H / KV), mine = (size_t)b * H + h;
  const int from = window ? max(0, n - window) : 0, c = CPL * lane;
  const int first = window ? min(sinks, from) : 0;         // slots [0, first) and [from, n)
  float qv[CPL], o[CPL] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < CPL; ++i) qv[i] = __half2float(q[mine * D + c + i]) * scale * LOG2E;
  auto row = [&](const void* codes, const void* scales, int slot, float* x) {
    const size_t at = head * cache.slots + slot;
    const float2 sm = __half22float2(((const __half2*)scales)[at * groups + c / cache.group]);
#pragma unroll
    for (int i = 0; i < CPL; ++i)
      x[i] = __fmaf_rn((float)((((const uint8_t*)codes)[at * (D / 2) + (c + i) / 2] >> (4 * (i & 1))) & 15), sm.x, sm.y);
  };
  for (int v = warp; v < first + n - from; v += AT_WARPS) {
    const int slot = v < first ? v : v - first + from;
    float x[CPL], s = 0.f;
    row(cache.k_codes, cache.k_scales, slot, x);
#pragma unroll
    for (int i = 0; i < CPL; ++i) s += qv[i] * x[i];
    for (int d = 16; d; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (scores && lane == 0) scores[mine * cache.slots + slot] = s;
    const float top = fmaxf(m, s), ref = top == -INFINITY ? 0.f : top, keep = exp2f(m - ref), w = exp2f(s - ref);
    m = top;
    l = l * keep + w;
    row(cache.v_codes, cache.v_scales, slot, x);
#pragma unroll
    for (int i = 0; i < CPL; ++i) o[i] = o[i] * keep + w * x[i];
  }
#pragma unroll
  for (int i = 0; i < CPL; ++i) s_o[warp][c + i] = o[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  float top = -INFINITY, tot = 0.f;
  for (int w = 0; w < AT_WARPS; ++w) top = fmaxf(top, s_m[w]);
  const float ref = top == -INFINITY ? 0.f : top;
  for (int w = 0; w < AT_WARPS; ++w) tot += s_l[w] * exp2f(s_m[w] - ref);
  if (threadIdx.x < D) {
    float sum = 0.f;
    for (int w = 0; w < AT_WARPS; ++w) sum += s_o[w][threadIdx.x] * exp2f(s_m[w] - ref);
    out[mine * D + threadIdx.x] = __float2half_rn(n > 0 ? sum / tot : 0.f);
  }
  if (stats && threadIdx.x == 0) stats[mine] = make_float2(ref, tot);
}

// weights_out = weights + the sum of the weights of the head's queries; 0 from slot n on.  A new slot (more) has none before.
__global__ void __launch_bounds__(AT_THREADS) kv4_weights_kernel(const float* __restrict__ scores, const float2* __restrict__ stats,
                                                                 const long long* __restrict__ length, int more, const float* weights,
                                                                 float* weights_out, int H, int KV, int slots, int window, int sinks) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int slot = blockIdx.x * AT_THREADS + threadIdx.x, kv = blockIdx.y, b = blockIdx.z, G = H / KV;
  if (slot >= slots) return;
  const int n = held(length, b, more, slots);
  const size_t at = ((size_t)b * KV + kv) * slots + slot;
  float w = 0.f;
  if (slot < n) {
    if (!(more && slot == length[b])) w = weights[at];
    if (!window || slot < sinks || slot >= n - window) {
      float sum = 0.f;
      for (int g = 0; g < G; ++g) {
        const size_t head = (size_t)b * H + kv * G + g;
        const float2 ml = stats[head];
        sum += exp2f(scores[head * slots + slot] - ml.x) / ml.y;
      }
      w += sum;
    }
  }
  weights_out[at] = w;
}

int attend(const cq_kv4* cache, const void* q, const long long* length, int more, void* out, int n_heads, int window, int sinks, float scale,
           const float* weights, float* weights_out, void* workspace, cudaStream_t stream) {
  const int B = cache->sequences, KV = cache->n_kv_heads;
  float2* stats = weights ? (float2*)workspace : nullptr;
  float* scores = weights ? (float*)(stats + (size_t)B * n_heads) : nullptr;
  auto fn = cache->head_dim == 128 ? kv4_attend_kernel<128> : kv4_attend_kernel<64>;
  CQ_CUDA_TRY(kv4_launch(fn, dim3(n_heads, B), dim3(AT_THREADS), 0, stream, (const __half*)q, *cache, length, more, (__half*)out, scores,
                         stats, n_heads, window, sinks, scale));
  if (weights)
    CQ_CUDA_TRY(kv4_launch(kv4_weights_kernel, dim3((cache->slots + AT_THREADS - 1) / AT_THREADS, KV, B), dim3(AT_THREADS), 0, stream,
                           (const float*)scores, (const float2*)stats, length, more, weights, weights_out, n_heads, KV, cache->slots, window,
                           sinks));
  return CQ_OK;
}

int check(const cq_kv4* cache, const void* q, const long long* length, const void* out, int n_heads, int window, int sinks,
          const float* weights, const float* weights_out, const void* workspace) {
  const int rc = cq_kv4_check(cache);
  if (rc != CQ_OK) return rc;
  if (!q || !length || !out || window < 0 || sinks < 0 || (!weights != !weights_out) || !workspace) return CQ_ERR_BAD_ARG;
  if (n_heads < 1 || n_heads % cache->n_kv_heads) return CQ_ERR_BAD_SHAPE;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15) return CQ_ERR_BAD_ARG;
  return CQ_OK;
}

}  // namespace

extern "C" size_t cq_kv4_attend_workspace_bytes(const cq_kv4* cache, int n_heads, int with_weights) {
  if (cq_kv4_check(cache) != CQ_OK || n_heads < 1) return 0;
  const size_t heads = (size_t)cache->sequences * n_heads;
  return heads * cache->head_dim * 2 + (with_weights ? heads * 8 + heads * cache->slots * 4 : 0) + 256;
}

extern "C" int cq_kv4_attend(const cq_kv4* cache, const void* q, const long long* length, void* out, int n_heads, int window, int sinks,
                             float scale, const float* weights, float* weights_out, void* workspace, cq_stream_t stream) {
  const int rc = check(cache, q, length, out, n_heads, window, sinks, weights, weights_out, workspace);
  if (rc != CQ_OK) return rc;
  return attend(cache, q, length, 0, out, n_heads, window, sinks, scale, weights, weights_out, workspace, (cudaStream_t)stream);
}

extern "C" int cq_kv4_step(const cq_kv4* cache, const void* q, const void* k, const void* v, const float* cos_table, const float* sin_table,
                           const long long* positions, int table_rows, const long long* length, void* out, int n_heads, int window,
                           int sinks, float scale, const float* weights, float* weights_out, void* workspace, cq_stream_t stream) {
  int rc = check(cache, q, length, out, n_heads, window, sinks, weights, weights_out, workspace);
  if (rc != CQ_OK) return rc;
  if (!k || !v || (((uintptr_t)k | (uintptr_t)v) & 15)) return CQ_ERR_BAD_ARG;
  void* rotated = workspace;
  const size_t own = ((size_t)cache->sequences * n_heads * cache->head_dim * 2 + 255) / 256 * 256;
  rc = cq_kv4_write(cache, q, rotated, k, v, cos_table, sin_table, positions, table_rows, length, 1, n_heads, stream);
  if (rc != CQ_OK) return rc;
  return attend(cache, rotated, length, 1, out, n_heads, window, sinks, scale, weights, weights_out, (uint8_t*)workspace + own,
                (cudaStream_t)stream);
}
