// Writing, reading and thinning out the 4-bit KV cache (layout: cq_kv4.cuh; attention over it: cq_kv4_attn.cu).  In the
// reference the cache is the fp16 key and value tensors of its vendored LLaMA (llama/modeling_llama_quant.py:371-419 of the
// reference project).
#include <algorithm>

#include "cq_kv4.cuh"

namespace {

constexpr int WR_THREADS = 256;

// D / 16 lanes a row of q, k or v: rotated (q and k), q to q_out, k and v quantised into their slots.
template <int D, int GROUP>
__global__ void __launch_bounds__(WR_THREADS) kv4_write_kernel(
    const __half* __restrict__ q, __half* __restrict__ q_out, const __half* __restrict__ k, const __half* __restrict__ v,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, const long long* __restrict__ positions, int table_rows,
    const long long* __restrict__ first, cq_kv4 cache, int tokens, int H, long long rows) {
  constexpr int LANES = D / 16;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int KV = cache.n_kv_heads, per = H + 2 * KV, c = 8 * (threadIdx.x % LANES);
  const long long stride = (long long)gridDim.x * (WR_THREADS / LANES);
  // every lane of a warp stays in the loop to its end: the rows' lanes exchange their minima
  const long long turns = (rows + stride - 1) / stride;
  for (long long i = 0, row = (long long)blockIdx.x * (WR_THREADS / LANES) + threadIdx.x / LANES; i < turns; ++i, row += stride) {
    const bool in = row < rows;
    const long long t = in ? row / per : 0;
    const int j = in ? (int)(row - t * per) : 0;
    const bool is_q = j < H, is_k = !is_q && j < H + KV;
    const __half* src = is_q ? q + (t * H + j) * D : (is_k ? k + (t * KV + j - H) * D : v + (t * KV + j - H - KV) * D);
    float x[16];
    kv4_load16(src + c, src + c + D / 2, x);
    bool there = true;
    if (cos_t && (is_q || is_k)) {
      const long long p = positions[t];
      there = p >= 0 && p < table_rows;
      if (there) kv4_rotate(x, cos_t + p * (D / 2) + c, sin_t + p * (D / 2) + c);
    }
    uint32_t words[2], pairs[2];
    kv4_quantise<D, GROUP>(x, words, pairs);
    if (!in) continue;
    if (is_q) {
      *reinterpret_cast<uint4*>(q_out + (t * H + j) * D + c) = kv4_halves(x);
      *reinterpret_cast<uint4*>(q_out + (t * H + j) * D + c + D / 2) = kv4_halves(x + 8);
      continue;
    }
    const long long b = t / tokens, slot = first[b] + (t - b * tokens);
    if (!there || slot < 0 || slot >= cache.slots) continue;
    const size_t at = ((size_t)b * KV + (is_k ? j - H : j - H - KV)) * cache.slots + slot;
    uint8_t* codes = (uint8_t*)(is_k ? cache.k_codes : cache.v_codes) + at * (D / 2);
    uint32_t* scales = (uint32_t*)(is_k ? cache.k_scales : cache.v_scales) + at * (D / GROUP);
    *reinterpret_cast<uint32_t*>(codes + c / 2) = words[0];
    *reinterpret_cast<uint32_t*>(codes + (c + D / 2) / 2) = words[1];
    if (c % GROUP == 0) scales[c / GROUP] = pairs[0];
    if (GROUP != D && c % GROUP == 0) scales[(c + D / 2) / GROUP] = pairs[1];
  }
}

// One lane per eight columns of a row: k and v (sequence, count, KV, D) fp16.  Slots outside the cache read as zeros.
__global__ void __launch_bounds__(WR_THREADS) kv4_read_kernel(cq_kv4 cache, const long long* __restrict__ first, int count,
                                                              __half* __restrict__ k, __half* __restrict__ v, long long pieces) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int KV = cache.n_kv_heads, D = cache.head_dim, per = D / 8, groups = D / cache.group;
  const bool value = blockIdx.y;
  const uint32_t* codes = (const uint32_t*)(value ? cache.v_codes : cache.k_codes);
  const __half2* scales = (const __half2*)(value ? cache.v_scales : cache.k_scales);
  __half* to = value ? v : k;
  for (long long i = (long long)blockIdx.x * WR_THREADS + threadIdx.x; i < pieces; i += (long long)gridDim.x * WR_THREADS) {
    const long long row = i / per, tok = row / KV, b = tok / count;
    const int w = (int)(i - row * per), head = (int)(row - tok * KV);
    const long long slot = first[b] + (tok - b * count);
    uint4 out = make_uint4(0, 0, 0, 0);
    if (slot >= 0 && slot < cache.slots) {
      const size_t at = ((size_t)b * KV + head) * cache.slots + slot;
      const uint32_t word = codes[at * per + w];
      const float2 sm = __half22float2(scales[at * groups + 8 * w / cache.group]);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __fmaf_rn((float)((word >> (4 * e)) & 15u), sm.x, sm.y);
      out = kv4_halves(x);
    }
    *reinterpret_cast<uint4*>(to + 8 * i) = out;
  }
}

// ------------------------------------------------------------------ eviction
constexpr int SEL_THREADS = 1024;

// weights in the order of unsigned numbers; NaN above all, and both zeros alike
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The slots of one head that stay, in order: kept (keep) and -1 behind them; their weights.  The smallest key that stays is
// found eight bits at a time; of the slots with exactly that key the lowest stay.
__global__ void __launch_bounds__(SEL_THREADS) kv4_select_kernel(const float* __restrict__ weights, const long long* __restrict__ length,
                                                                 long long* __restrict__ length_out, int* __restrict__ kept,
                                                                 float* __restrict__ weights_out, int KV, int slots, int keep, int sinks,
                                                                 int recent) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ uint32_t hist[256];
  __shared__ uint32_t s_prefix, s_need;
  __shared__ uint32_t s_warp[2][32];
  const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long len = length[b];
  const int n = (int)(len < 0 ? 0 : (len > slots ? slots : len));
  const size_t row = (size_t)b * KV + head;
  const float* w = weights + row * slots;
  int* to = kept + row * keep;
  float* wto = weights_out + row * keep;
  if (head == 0 && tid == 0) length_out[b] = n < keep ? n : keep;
  if (n <= keep) {
    for (int j = tid; j < keep; j += SEL_THREADS) {
      to[j] = j < n ? j : -1;
      wto[j] = j < n ? w[j] : 0.f;
    }
    return;
  }
  const int beg = sinks, end = n - recent;                 // the candidates; end - beg > need, as n > keep
  if (tid == 0) {
    s_prefix = 0;
    s_need = (uint32_t)(keep - sinks - recent);
  }
  uint32_t mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    for (int j = beg + tid; j < end; j += SEL_THREADS) {
      const uint32_t key = weight_key(w[j]);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (warp == 0) {
      // from the largest digit down: the first at which the count reaches what is needed
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += hist[255 - (8 * lane + i)];
      uint32_t before = mine;
      for (int d = 1; d < 32; d *= 2) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += o;
      }
      before -= mine;
      const uint32_t need = s_need;
      __syncwarp();
      if (before < need && before + mine >= need) {
        for (int i = 0; i < 8; ++i) {
          const uint32_t c = hist[255 - (8 * lane + i)];
          if (before + c >= need) {
            s_prefix = prefix | (uint32_t)(255 - (8 * lane + i)) << shift;
            s_need = need - before;
            break;
          }
          before += c;
        }
      } else if (need == 0 && lane == 0) {
        s_prefix = 0xFFFFFFFFu;                            // nothing between the sinks and the recent ones stays
      }
    }
    __syncthreads();
    mask |= 255u << shift;
    if (s_need == 0) break;
  }
  const uint32_t limit = s_prefix, ties = s_need;           // keys above `limit` stay, and the first `ties` equal to it
  const bool none = ties == 0;
  // in order: slots of a block of SEL_THREADS at a time, ranks by ballots
  uint32_t above = 0, equal = 0;                            // before this block: kept because above or outside, equal
  for (int base = 0; base < n; base += SEL_THREADS) {
    const int j = base + tid;
    bool up = false, eq = false;
    if (j < n) {
      if (j < beg || j >= end) up = true;
      else if (!none) {
        const uint32_t key = weight_key(w[j]);
        up = key > limit;
        eq = key == limit;
      }
    }
    const uint32_t bu = __ballot_sync(0xffffffffu, up), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) {
      s_warp[0][warp] = __popc(bu);
      s_warp[1][warp] = __popc(be);
    }
    __syncthreads();
    uint32_t cu = s_warp[0][lane], ce = s_warp[1][lane];
    uint32_t pu = cu, pe = ce;
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t a = __shfl_up_sync(0xffffffffu, pu, d), c = __shfl_up_sync(0xffffffffu, pe, d);
      if (lane >= d) {
        pu += a;
        pe += c;
      }
    }
    const uint32_t tu = __shfl_sync(0xffffffffu, pu, 31), te = __shfl_sync(0xffffffffu, pe, 31);
    const uint32_t lt = (1u << lane) - 1u;
    const uint32_t mu = above + __shfl_sync(0xffffffffu, pu - cu, warp) + __popc(bu & lt);
    const uint32_t me = equal + __shfl_sync(0xffffffffu, pe - ce, warp) + __popc(be & lt);
    if (up || (eq && me < ties)) {
      const uint32_t at = mu + (me < ties ? me : ties);
      to[at] = j;
      wto[at] = w[j];
    }
    above += tu;
    equal += te;
    __syncthreads();
  }
}

// Rows kept[...] of `from` to the first slots of `to`, zeros behind them; a lane per 16 bytes of codes, 4 of scales.
struct MoveArgs {
  const void* src[4];
  void* dst[4];
  int bytes[4];              // of a row
  int src_slots, dst_slots, keep;
};
__global__ void __launch_bounds__(WR_THREADS) kv4_gather_kernel(MoveArgs a, const int* __restrict__ kept, long long rows) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int which = blockIdx.y, per = a.bytes[which] / 4;
  const uint32_t* src = (const uint32_t*)a.src[which];
  uint32_t* dst = (uint32_t*)a.dst[which];
  for (long long i = (long long)blockIdx.x * WR_THREADS + threadIdx.x; i < rows * per; i += (long long)gridDim.x * WR_THREADS) {
    const long long r = i / per, head = r / a.keep;
    const int w = (int)(i - r * per), at = kept ? kept[r] : (int)(r - head * a.keep);
    dst[((size_t)head * a.dst_slots + (r - head * a.keep)) * per + w] = at < 0 ? 0u : src[((size_t)head * a.src_slots + at) * per + w];
  }
}

int blocks_for(long long items, int threads, int most) {
  return (int)std::max<long long>(1, std::min<long long>((items + threads - 1) / threads, most));
}
int most_blocks() { return cq_sm_count() * 16; }

}  // namespace

extern "C" int cq_kv4_check(const cq_kv4* c) {
  if (!c || !c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales) return CQ_ERR_BAD_ARG;
  if (((uintptr_t)c->k_codes | (uintptr_t)c->k_scales | (uintptr_t)c->v_codes | (uintptr_t)c->v_scales) & 15) return CQ_ERR_BAD_ARG;
  if (c->sequences < 1 || c->sequences > 65535 || c->n_kv_heads < 1 || c->slots < 32 || c->slots % 32 || c->slots > (1 << 30))
    return CQ_ERR_BAD_SHAPE;
  if ((c->head_dim != 64 && c->head_dim != 128) || (c->group != 32 && c->group != 64)) return CQ_ERR_UNSUPPORTED;
  return CQ_OK;
}

extern "C" int cq_kv4_write(const cq_kv4* cache, const void* q, void* q_out, const void* k, const void* v, const float* cos_table,
                            const float* sin_table, const long long* positions, int table_rows, const long long* first, int tokens,
                            int n_heads, cq_stream_t stream) {
  const int rc = cq_kv4_check(cache);
  if (rc != CQ_OK) return rc;
  if (!k || !v || !first || tokens < 1 || n_heads < 0 || (n_heads > 0 && (!q || !q_out))) return CQ_ERR_BAD_ARG;
  if (cos_table && (!sin_table || !positions || table_rows < 1)) return CQ_ERR_BAD_ARG;
  if (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v) & 15) return CQ_ERR_BAD_ARG;
  const long long rows = (long long)cache->sequences * tokens * (n_heads + 2 * cache->n_kv_heads);
  const bool wide = cache->head_dim == 128, narrow = cache->group == 32;
  auto fn = wide ? (narrow ? kv4_write_kernel<128, 32> : kv4_write_kernel<128, 64>)
                 : (narrow ? kv4_write_kernel<64, 32> : kv4_write_kernel<64, 64>);
  const int blocks = blocks_for(rows * (cache->head_dim / 16), WR_THREADS, most_blocks());
  CQ_CUDA_TRY(kv4_launch(fn, dim3(blocks), dim3(WR_THREADS), 0, (cudaStream_t)stream, (const __half*)q, (__half*)q_out, (const __half*)k,
                         (const __half*)v, cos_table, sin_table, positions, table_rows, first, *cache, tokens, n_heads, rows));
  return CQ_OK;
}

extern "C" int cq_kv4_read(const cq_kv4* cache, const long long* first, int count, void* k, void* v, cq_stream_t stream) {
  const int rc = cq_kv4_check(cache);
  if (rc != CQ_OK) return rc;
  if (!first || !k || !v || count < 1 || (((uintptr_t)k | (uintptr_t)v) & 15)) return CQ_ERR_BAD_ARG;
  const long long pieces = (long long)cache->sequences * count * cache->n_kv_heads * (cache->head_dim / 8);
  CQ_CUDA_TRY(kv4_launch(kv4_read_kernel, dim3(blocks_for(pieces, WR_THREADS, most_blocks()), 2), dim3(WR_THREADS), 0,
                         (cudaStream_t)stream, *cache, first, count, (__half*)k, (__half*)v, pieces));
  return CQ_OK;
}

extern "C" size_t cq_kv4_evict_workspace_bytes(const cq_kv4* cache, int keep) {
  if (cq_kv4_check(cache) != CQ_OK || keep < 1) return 0;
  const size_t row = cache->head_dim / 2 + 4 * (cache->head_dim / cache->group);
  return (size_t)cache->sequences * cache->n_kv_heads * keep * 2 * row;
}

extern "C" int cq_kv4_evict(const cq_kv4* from, const cq_kv4* to, const float* weights, float* weights_out, const long long* length,
                            long long* length_out, int keep, int sinks, int recent, int* kept, void* workspace, cq_stream_t stream) {
  int rc = cq_kv4_check(from);
  if (rc == CQ_OK) rc = cq_kv4_check(to);
  if (rc != CQ_OK) return rc;
  if (!weights || !weights_out || !length || !length_out || !kept) return CQ_ERR_BAD_ARG;
  if (from->sequences != to->sequences || from->n_kv_heads != to->n_kv_heads || from->head_dim != to->head_dim || from->group != to->group)
    return CQ_ERR_BAD_SHAPE;
  if (sinks < 0 || recent < 0 || keep < 1 || keep > to->slots || (long long)sinks + recent > keep) return CQ_ERR_BAD_ARG;
  const void* fp[4] = {from->k_codes, from->k_scales, from->v_codes, from->v_scales};
  void* tp[4] = {to->k_codes, to->k_scales, to->v_codes, to->v_scales};
  const bool in_place = fp[0] == tp[0];
  for (int i = 0; i < 4; ++i)
    if ((fp[i] == tp[i]) != in_place) return CQ_ERR_BAD_ARG;
  if (in_place && (from->slots != to->slots || !workspace || ((uintptr_t)workspace & 15))) return CQ_ERR_BAD_ARG;
  const int B = from->sequences, KV = from->n_kv_heads, D = from->head_dim;
  CQ_CUDA_TRY(kv4_launch(kv4_select_kernel, dim3(KV, B), dim3(SEL_THREADS), 0, (cudaStream_t)stream, weights, length, length_out, kept,
                         weights_out, KV, from->slots, keep, sinks, recent));
  const long long rows = (long long)B * KV * keep;
  MoveArgs move = {}, back = {};
  const int bytes[4] = {D / 2, 4 * (D / from->group), D / 2, 4 * (D / from->group)};
  uint8_t* ws = (uint8_t*)workspace;
  for (int i = 0; i < 4; ++i) {
    move.src[i] = fp[i];
    move.dst[i] = in_place ? ws : tp[i];
    back.src[i] = ws;
    back.dst[i] = tp[i];
    move.bytes[i] = back.bytes[i] = bytes[i];
    if (in_place) ws += rows * bytes[i];
  }
  move.src_slots = from->slots;
  move.dst_slots = in_place ? keep : to->slots;
  move.keep = back.keep = back.src_slots = keep;
  back.dst_slots = to->slots;
  const dim3 grid(blocks_for(rows * (D / 8), WR_THREADS, most_blocks()), 4);
  CQ_CUDA_TRY(kv4_launch(kv4_gather_kernel, grid, dim3(WR_THREADS), 0, (cudaStream_t)stream, move, (const int*)kept, rows));
  if (in_place) CQ_CUDA_TRY(kv4_launch(kv4_gather_kernel, grid, dim3(WR_THREADS), 0, (cudaStream_t)stream, back, (const int*)nullptr, rows));
  return CQ_OK;
}
