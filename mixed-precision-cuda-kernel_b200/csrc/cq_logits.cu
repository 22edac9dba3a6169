// Logits on their way to a token: penalties for tokens that occurred, biases of single tokens, a grammar's bit mask, and the largest.
//
// A cluster of CTAs takes a row, a CTA a part of the vocabulary.  How often its tokens occurred is counted in shared memory from the
// row's history (integer additions: their order changes nothing), where a part is larger than that memory one slice after
// another; then every logit is read once and written once.  The largest travels as one 64-bit key, its value in the order of
// unsigned numbers above the complement of its token: the maximum of keys is the lowest token of the largest value.
#include <algorithm>

#include <cooperative_groups.h>

#include "cq_pages.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int THREADS = 512;
constexpr int SLICE = 16384;                 // tokens counted at a time
constexpr uint32_t OCCURRED = 0x80000000u;   // anywhere in the history; the bits below count the generated part

struct Adjust {
  cq_adjust a;
  int rows, vocab;
};

template <typename T> __device__ __forceinline__ float value_of(T x);
template <> __device__ __forceinline__ float value_of(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float value_of(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float value_of(float x) { return x; }
template <typename T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ __half rounded(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ float rounded(float x) { return x; }

// fp32 numbers in the order of unsigned ones: NaN above all, both zeros alike
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long larger(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

template <typename T>
__global__ void __launch_bounds__(THREADS) adjust_logits_kernel(const Adjust p) {
  extern __shared__ __align__(16) uint32_t s_count[];      // [slice], and where there are biases [slice] 1 + the entry that counts
  __shared__ unsigned long long s_key[THREADS / 32];
  __shared__ unsigned long long s_best;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const cq_adjust& a = p.a;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = gridDim.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = (p.vocab + parts - 1) / parts, begin = min(p.vocab, (int)blockIdx.x * part), end = min(p.vocab, begin + part);
  const T* in = (const T*)a.logits + (int64_t)row * a.logits_stride;
  T* out = (T*)a.out + (int64_t)row * a.out_stride;
  uint32_t* s_bias = s_count + (a.tokens ? min(part, SLICE) : 0);

  long long n = 0, prompt = 0;
  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (a.tokens) {
    n = a.length ? a.length[row] : a.width;
    n = n < 0 ? 0 : (n > a.width ? a.width : n);
    prompt = a.prompt ? a.prompt[row] : 0;
    if (a.repetition) rep = a.repetition[row];
    if (a.presence) pres = a.presence[row];
    if (a.frequency) freq = a.frequency[row];
  }
  const long long* tokens = a.tokens ? a.tokens + (int64_t)row * a.tokens_stride : nullptr;
  const uint32_t* mask = nullptr;
  if (a.mask) {
    const long long m = a.mask_rows ? a.mask_rows[row] : row;
    if (m >= 0 && m < a.masks) mask = a.mask + m * a.mask_stride;
  }

  unsigned long long best = 0;
  for (int base = begin; base < end; base += SLICE) {
    const int size = min(SLICE, end - base);
    if (a.tokens)
      for (int i = tid; i < size; i += THREADS) s_count[i] = 0u;
    if (a.biases)
      for (int i = tid; i < size; i += THREADS) s_bias[i] = 0u;
    __syncthreads();
    for (long long i = tid; i < n; i += THREADS) {
      const long long v = tokens[i] - base;
      if (v < 0 || v >= size) continue;
      if (i < prompt) atomicOr(&s_count[v], OCCURRED);
      else {
        atomicOr(&s_count[v], OCCURRED);
        atomicAdd(&s_count[v], 1u);
      }
    }
    for (int i = tid; i < a.biases; i += THREADS) {        // of the same token's entries the last one counts
      const long long v = a.bias_ids[(int64_t)row * a.bias_ids_stride + i] - base;
      if (v >= 0 && v < size) atomicMax(&s_bias[v], (uint32_t)i + 1u);
    }
    __syncthreads();
    for (int i = tid; i < size; i += THREADS) {
      const int v = base + i;
      float x = value_of<T>(in[v]);
      const uint32_t c = a.tokens ? s_count[i] : 0u;
      if (c) {
        if (a.repetition) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        if (c & ~OCCURRED) {
          if (a.frequency) x = __fsub_rn(x, __fmul_rn(freq, (float)(c & ~OCCURRED)));
          if (a.presence) x = __fsub_rn(x, pres);
        }
      }
      if (a.biases && s_bias[i]) x = __fadd_rn(x, a.bias[(int64_t)row * a.bias_stride + s_bias[i] - 1u]);
      if (mask && !(mask[v >> 5] >> (v & 31) & 1u)) x = -INFINITY;
      out[v] = rounded<T>(x);
      best = larger(best, (unsigned long long)order_of(x) << 32 | (0xFFFFFFFFu - (uint32_t)v));
    }
    __syncthreads();
  }
  for (int d = 16; d; d /= 2) best = larger(best, __shfl_xor_sync(0xffffffffu, best, d));
  if (lane == 0) s_key[warp] = best;
  __syncthreads();
  if (warp == 0) {
    best = lane < THREADS / 32 ? s_key[lane] : 0ull;
    for (int d = 16; d; d /= 2) best = larger(best, __shfl_xor_sync(0xffffffffu, best, d));
    if (lane == 0) s_best = best;
  }
  if (parts > 1) cluster.sync();
  if (blockIdx.x == 0 && warp == 0) {
    if (parts > 1) best = lane < parts ? *cluster.map_shared_rank(&s_best, lane) : 0ull;
    for (int d = 16; d; d /= 2) best = larger(best, __shfl_xor_sync(0xffffffffu, best, d));
    if (lane == 0) a.next[row] = (long long)(0xFFFFFFFFu - (uint32_t)best);
  }
  if (parts > 1) cluster.sync();                           // (nobody leaves while its key may be read)
}

// bytes from the first to behind the last element of `rows` rows of `cols`
size_t span(int64_t rows, int64_t cols, int64_t stride, size_t item) { return (size_t)((rows - 1) * stride + cols) * item; }

}  // namespace

extern "C" int cq_adjust_logits(const cq_adjust* a, int rows, int vocab, cq_stream_t stream) {
  if (!a || !a->logits || !a->out || !a->next) return CQ_ERR_BAD_ARG;
  if (rows < 1 || rows > 65535 || vocab < 1 || vocab > (1 << 30) || a->width > INT32_MAX) return CQ_ERR_BAD_SHAPE;
  if (a->dtype < 0 || a->dtype > 2) return CQ_ERR_UNSUPPORTED;
  const size_t item = a->dtype == 1 ? 4 : 2;
  if (((uintptr_t)a->logits | (uintptr_t)a->out) & (item - 1)) return CQ_ERR_BAD_ARG;
  if (a->logits_stride < 0 || (rows > 1 && a->out_stride < vocab)) return CQ_ERR_BAD_ARG;
  if (a->tokens ? a->width < 0 || a->tokens_stride < 0 : (a->length || a->prompt || a->repetition || a->presence || a->frequency)) return CQ_ERR_BAD_ARG;
  if (a->biases < 0 || (a->biases > 0 && (!a->bias_ids || !a->bias || a->bias_ids_stride < 0 || a->bias_stride < 0))) return CQ_ERR_BAD_ARG;
  if (a->mask ? a->masks < 1 || a->mask_stride < 0 || (!a->mask_rows && a->masks < rows) : a->mask_rows != nullptr) return CQ_ERR_BAD_ARG;
  // in place, or apart
  const bool in_place = a->logits == a->out && (rows == 1 || a->logits_stride == a->out_stride);
  if (!in_place && !kv4_apart(a->logits, span(rows, vocab, a->logits_stride, item), a->out, span(rows, vocab, a->out_stride, item))) return CQ_ERR_BAD_ARG;
  const int sms = cq_sm_count();
  int parts = 1;
  while (parts < 8 && (vocab > parts * SLICE || rows * parts < sms) && vocab > parts * 1024) parts *= 2;
  const int part = (vocab + parts - 1) / parts, slice = std::min(part, SLICE), smem = 4 * slice * ((a->tokens ? 1 : 0) + (a->biases ? 1 : 0));
  auto fn = a->dtype == 0 ? adjust_logits_kernel<__half> : (a->dtype == 1 ? adjust_logits_kernel<float> : adjust_logits_kernel<__nv_bfloat16>);
  CQ_CUDA_TRY(cq_grant_smem((const void*)fn, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts, rows);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  CQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, Adjust{*a, rows, vocab}));
  return CQ_OK;
}
