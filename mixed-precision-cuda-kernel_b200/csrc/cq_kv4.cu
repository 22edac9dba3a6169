// Writing, reading and thinning out the 4-bit KV cache (layout: cq_kv4.cuh; attention over it: cq_kv4_attn.cu).  In the
// reference the cache is the fp16 key and value tensors of its vendored LLaMA (llama/modeling_llama_quant.py:371-419 of the
// reference project).
#include <algorithm>
#include <utility>

#include "cq_kv4.cuh"

namespace {

constexpr int WR_THREADS = 256, WR_TOKENS = 64;      // a block's rows of one head (reads, moves)

// D / 16 lanes a row of q, k or v: rotated (q and k), q to q_out, k and v quantised into their slots.  A block takes one head's
// rows of as many tokens as it has rows of lanes, so that nothing is divided but block indices.  63 MB of rows of 40 heads and
// 34 MB of results take 24 us, 4.0 TB/s, with reading them back 36: neither memory (DRAM 30 % busy under ncu, much of the results still in
// L2) nor instructions (62 % of the cycles issue one) are full, and warps wait for their loads (6.6 of 16 cycles an issue).  (Two tokens a lane: 39, and 6.4 instead of 4.9 for 5 x 77 tokens; four
// heads one after another, the angles kept in registers: 38 and 7.2.  Tables that start off 8 bytes (PAIRS false) have an instance of their
// own: a choice at run time costs the usual ones 24 -> 28 us of the rows' part.)
template <int D, int GROUP, bool PAIRS>
__global__ void __launch_bounds__(WR_THREADS, 6) kv4_write_kernel(
    const __half* __restrict__ q, __half* __restrict__ q_out, const __half* __restrict__ k, const __half* __restrict__ v,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, const long long* __restrict__ positions, int table_rows,
    const long long* __restrict__ first, cq_kv4 cache, int tokens, int H) {
  constexpr int LANES = D / 16, ROWS = WR_THREADS / LANES;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int KV = cache.n_kv_heads, j = blockIdx.y, b = blockIdx.z, c = 8 * (threadIdx.x % LANES), t = blockIdx.x * ROWS + threadIdx.x / LANES;
  const bool is_q = j < H, is_k = !is_q && j < H + KV;
  const int head = is_q ? j : (is_k ? j - H : j - H - KV), heads = is_q ? H : KV;
  const size_t row = (size_t)b * tokens + min(t, tokens - 1);      // (every lane stays to the end: a row's lanes exchange their minima)
  const __half* src = (is_q ? q : (is_k ? k : v)) + (row * heads + head) * D + c;
  uint32_t x[8];
  kv4_load16(src, src + D / 2, x);
  const long long pos = cos_t ? positions[row] : 0, slot = is_q ? 0 : first[b] + t;
  const bool turn = cos_t && pos >= 0 && pos < table_rows;
  if (turn && (is_q || is_k)) kv4_rotate<PAIRS>(x, cos_t + pos * (D / 2) + c, sin_t + pos * (D / 2) + c);
  if (is_q) {
    if (t >= tokens) return;
    __half* to = q_out + (row * H + head) * D + c;
    *reinterpret_cast<uint4*>(to) = make_uint4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<uint4*>(to + D / 2) = make_uint4(x[4], x[5], x[6], x[7]);
    return;
  }
  uint32_t words[2], pairs[2];
  kv4_quantise<D, GROUP>(x, words, pairs);
  // a key without a position in the tables is left out, and its value with it
  if (t >= tokens || (cos_t && !turn) || slot < 0 || slot >= cache.slots) return;
  const size_t at = ((size_t)b * KV + head) * cache.slots + slot;
  uint8_t* codes = (uint8_t*)(is_k ? cache.k_codes : cache.v_codes) + at * (D / 2);
  uint32_t* scales = (uint32_t*)(is_k ? cache.k_scales : cache.v_scales) + at * (D / GROUP);
  *reinterpret_cast<uint32_t*>(codes + c / 2) = words[0];
  *reinterpret_cast<uint32_t*>(codes + (c + D / 2) / 2) = words[1];
  if (c % GROUP == 0) {
    scales[c / GROUP] = pairs[0];
    if (GROUP != D) scales[(c + D / 2) / GROUP] = pairs[1];
  }
}

// D / 8 lanes a row, eight columns each: k and v (sequence, count, KV, D) fp16.  A block takes a head's rows of 64 tokens.  Slots
// outside the cache read as zeros.
template <int D, int GROUP>
__global__ void __launch_bounds__(WR_THREADS) kv4_read_kernel(cq_kv4 cache, const long long* __restrict__ first, int count,
                                                              __half* __restrict__ k, __half* __restrict__ v) {
  constexpr int LANES = D / 8, ROWS = WR_THREADS / LANES, FLIGHT = WR_TOKENS / ROWS;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int KV = cache.n_kv_heads, b = blockIdx.z, head = blockIdx.y >> 1, w = threadIdx.x % LANES;
  const bool value = blockIdx.y & 1;
  const uint32_t* codes = (const uint32_t*)(value ? cache.v_codes : cache.k_codes);
  const __half2* scales = (const __half2*)(value ? cache.v_scales : cache.k_scales);
  __half* to = value ? v : k;
  const size_t row0 = ((size_t)b * KV + head) * cache.slots;
  const long long slot0 = first[b];
  uint32_t word[FLIGHT];
  __half2 pair[FLIGHT];
#pragma unroll
  for (int f = 0; f < FLIGHT; ++f) {
    const int t = blockIdx.x * WR_TOKENS + f * ROWS + threadIdx.x / LANES;
    const long long slot = slot0 + t;
    const bool in = t < count && slot >= 0 && slot < cache.slots;
    word[f] = in ? codes[(row0 + slot) * LANES + w] : 0u;
    pair[f] = in ? scales[(row0 + slot) * (D / GROUP) + 8 * w / GROUP] : __half2half2(__ushort_as_half(0));
  }
#pragma unroll
  for (int f = 0; f < FLIGHT; ++f) {
    const int t = blockIdx.x * WR_TOKENS + f * ROWS + threadIdx.x / LANES;
    if (t >= count) break;
    // scale * code + minimum, rounded once: 1024 + code is what a code in the lowest bits of an fp16 1024 makes
    const __half2 s2 = __low2half2(pair[f]), m2 = __high2half2(pair[f]), less = __float2half2_rn(-1024.f);
    uint32_t x[4];                                         // columns (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = (word[f] >> (4 * e) & 0x000F000Fu) | 0x64006400u;
      const __half2 y = __hfma2(__hadd2(*reinterpret_cast<const __half2*>(&u), less), s2, m2);
      x[e] = *reinterpret_cast<const uint32_t*>(&y);
    }
    *reinterpret_cast<uint4*>(to + (((size_t)b * count + t) * KV + head) * D + 8 * w) =
        make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410), __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
  }
}

// ------------------------------------------------------------------ eviction
constexpr int SEL_THREADS = 1024, SEL_FEW = 128;

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
  const int threads = blockDim.x, head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long len = length[b];
  const int n = (int)(len < 0 ? 0 : (len > slots ? slots : len));
  const size_t row = (size_t)b * KV + head;
  const float* w = weights + row * slots;
  int* to = kept + row * keep;
  float* wto = weights_out + row * keep;
  if (head == 0 && tid == 0) length_out[b] = n < keep ? n : keep;
  if (n <= keep) {
    for (int j = tid; j < keep; j += threads) {
      to[j] = j < n ? j : -1;
      wto[j] = j < n ? w[j] : 0.f;
    }
    return;
  }
  const int beg = sinks, end = n - recent;                 // the candidates; end - beg > need, as n > keep
  if (n <= SEL_FEW) {
    // Few slots: a candidate's place among them is the count of those that come before it, a thread a slot.  (With the move, 32
    // heads of 34 slots 3.7 us, of 128 4.8; by digits 6.6 and 6.7.  256 slots would be about even.)
    __shared__ __align__(16) uint32_t s_key[SEL_FEW];
    const uint32_t mine = tid >= beg && tid < end ? weight_key(w[tid]) : 0u;      // (no weight's key is 0)
    if (tid < SEL_FEW) s_key[tid] = mine;
    __syncthreads();
    int before = 0;
    if (mine)
      for (int i = beg / 4; 4 * i < end; ++i) {
        const uint4 k = reinterpret_cast<const uint4*>(s_key)[i];
        const int at = 4 * i;
        before += at < tid ? k.x >= mine : k.x > mine;
        before += at + 1 < tid ? k.y >= mine : k.y > mine;
        before += at + 2 < tid ? k.z >= mine : k.z > mine;
        before += at + 3 < tid ? k.w >= mine : k.w > mine;
      }
    const bool stays = tid < n && (!mine || before < keep - sinks - recent);
    const uint32_t bits = __ballot_sync(0xffffffffu, stays);
    if (lane == 0) s_warp[0][warp] = __popc(bits);
    __syncthreads();
    const uint32_t at = __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[0][lane] : 0u) + __popc(bits & ((1u << lane) - 1u));
    if (stays) {
      to[at] = tid;
      wto[at] = w[tid];
    }
    return;
  }
  if (tid == 0) {
    s_prefix = 0;
    s_need = (uint32_t)(keep - sinks - recent);
  }
  uint32_t mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    for (int j = beg + tid; j < end; j += threads) {
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
  if (tid < 64) s_warp[tid >> 5][tid & 31] = 0;              // (of warps that a smaller block has not)
  __syncthreads();
  const uint32_t limit = s_prefix, ties = s_need;           // keys above `limit` stay, and the first `ties` equal to it
  const bool none = ties == 0;
  // in order: as many slots as threads at a time, ranks by ballots
  uint32_t above = 0, equal = 0;                            // before this block: kept because above or outside, equal
  for (int base = 0; base < n; base += threads) {
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

// Rows kept[...] of a head to its first slots, zeros behind them: 16 bytes of codes a lane, 64 rows a block.  kept null: the
// rows as they lie.
struct MoveArgs {
  const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  uint8_t *k_codes_to, *k_scales_to, *v_codes_to, *v_scales_to;
  int src_slots, dst_slots, keep;
};
template <int D, int GROUP>
__global__ void __launch_bounds__(WR_THREADS) kv4_gather_kernel(const MoveArgs a, const int* __restrict__ kept) {
  constexpr int ROW = D / 2, PIECES = ROW / 16, WORDS = D / GROUP;      // 16-byte pieces of codes, words of scales
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const size_t head = blockIdx.y + (size_t)gridDim.y * blockIdx.z, from = head * a.src_slots, to = head * a.dst_slots;
  const int r0 = blockIdx.x * WR_TOKENS;
  __shared__ int s_at[WR_TOKENS];
  if (threadIdx.x < WR_TOKENS) {
    const int r = r0 + threadIdx.x;
    s_at[threadIdx.x] = r < a.keep ? (kept ? kept[head * a.keep + r] : r) : -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < WR_TOKENS * PIECES; i += WR_THREADS) {
    const int r = i / PIECES, c = 16 * (i % PIECES), at = s_at[r];
    if (r0 + r >= a.keep) break;
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    if (at >= 0) {
      x = *reinterpret_cast<const uint4*>(a.k_codes + (from + at) * ROW + c);
      y = *reinterpret_cast<const uint4*>(a.v_codes + (from + at) * ROW + c);
    }
    *reinterpret_cast<uint4*>(a.k_codes_to + (to + r0 + r) * ROW + c) = x;
    *reinterpret_cast<uint4*>(a.v_codes_to + (to + r0 + r) * ROW + c) = y;
  }
  for (int i = threadIdx.x; i < WR_TOKENS * WORDS; i += WR_THREADS) {
    const int r = i / WORDS, c = 4 * (i % WORDS), at = s_at[r];
    if (r0 + r >= a.keep) break;
    *reinterpret_cast<uint32_t*>(a.k_scales_to + (to + r0 + r) * (4 * WORDS) + c) =
        at < 0 ? 0u : *reinterpret_cast<const uint32_t*>(a.k_scales + (from + at) * (4 * WORDS) + c);
    *reinterpret_cast<uint32_t*>(a.v_scales_to + (to + r0 + r) * (4 * WORDS) + c) =
        at < 0 ? 0u : *reinterpret_cast<const uint32_t*>(a.v_scales + (from + at) * (4 * WORDS) + c);
  }
}

// the instance for a cache's head width and group
#define KV4_PICK(kernel, c, ...)                                                                                     \
  ((c)->head_dim == 128 ? ((c)->group == 32 ? kernel<128, 32 __VA_ARGS__> : kernel<128, 64 __VA_ARGS__>)           \
                        : ((c)->group == 32 ? kernel<64, 32 __VA_ARGS__> : kernel<64, 64 __VA_ARGS__>))

}  // namespace

extern "C" int cq_kv4_check(const cq_kv4* c) {
  if (!c || !c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales) return CQ_ERR_BAD_ARG;
  if (((uintptr_t)c->k_codes | (uintptr_t)c->k_scales | (uintptr_t)c->v_codes | (uintptr_t)c->v_scales) & 15) return CQ_ERR_BAD_ARG;
  if (c->sequences < 1 || c->sequences > 65535 || c->n_kv_heads < 1 || c->n_kv_heads > 32767 || c->slots < 32 || c->slots % 32 || c->slots > (1 << 30))
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
  const long long kinds = n_heads + 2ll * cache->n_kv_heads;
  if (kinds > 65535) return CQ_ERR_BAD_SHAPE;
  const int rows = WR_THREADS / (cache->head_dim / 16);
  const bool pairs = (((uintptr_t)cos_table | (uintptr_t)sin_table) & 7) == 0;
  auto fn = pairs ? KV4_PICK(kv4_write_kernel, cache, , true) : KV4_PICK(kv4_write_kernel, cache, , false);
  CQ_CUDA_TRY(kv4_launch(fn, dim3((tokens + rows - 1) / rows, (unsigned)kinds, cache->sequences), dim3(WR_THREADS), 0,
                         (cudaStream_t)stream, (const __half*)q, (__half*)q_out, (const __half*)k, (const __half*)v, cos_table, sin_table, positions,
                         table_rows, first, *cache, tokens, n_heads));
  return CQ_OK;
}

extern "C" int cq_kv4_read(const cq_kv4* cache, const long long* first, int count, void* k, void* v, cq_stream_t stream) {
  const int rc = cq_kv4_check(cache);
  if (rc != CQ_OK) return rc;
  if (!first || !k || !v || count < 1 || (((uintptr_t)k | (uintptr_t)v) & 15)) return CQ_ERR_BAD_ARG;
  CQ_CUDA_TRY(kv4_launch(KV4_PICK(kv4_read_kernel, cache), dim3((count + WR_TOKENS - 1) / WR_TOKENS, 2 * cache->n_kv_heads, cache->sequences),
                         dim3(WR_THREADS), 0, (cudaStream_t)stream, *cache, first, count, (__half*)k, (__half*)v));
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
  if (sinks < 0 || recent < 0 || keep < 1 || keep > to->slots) return CQ_ERR_BAD_ARG;
  sinks = std::min(sinks, keep);                           // (where more than keep slots are to stay in any case)
  recent = std::min(recent, keep - sinks);
  const void* fp[4] = {from->k_codes, from->k_scales, from->v_codes, from->v_scales};
  void* tp[4] = {to->k_codes, to->k_scales, to->v_codes, to->v_scales};
  const bool in_place = fp[0] == tp[0];
  for (int i = 0; i < 4; ++i)
    if ((fp[i] == tp[i]) != in_place) return CQ_ERR_BAD_ARG;
  if (in_place && (from->slots != to->slots || !workspace || ((uintptr_t)workspace & 15))) return CQ_ERR_BAD_ARG;
  const int B = from->sequences, KV = from->n_kv_heads, D = from->head_dim;
  const size_t heads = (size_t)B * KV, row_bytes[2] = {(size_t)D / 2, 4 * (size_t)(D / from->group)};
  for (int i = 0; i < 4 && !in_place; ++i)
    for (int j = 0; j < 4; ++j)
      if (!kv4_apart(tp[i], heads * to->slots * row_bytes[i & 1], fp[j], heads * from->slots * row_bytes[j & 1])) return CQ_ERR_BAD_ARG;
  const std::pair<const void*, size_t> in[2] = {{weights, heads * from->slots * 4}, {length, (size_t)B * 8}},
                                       res[3] = {{weights_out, heads * keep * 4}, {length_out, (size_t)B * 8}, {kept, heads * keep * 4}};
  for (const auto& r : res)
    for (const auto& i : in)
      if (!kv4_apart(r.first, r.second, i.first, i.second)) return CQ_ERR_BAD_ARG;
  // The passes of a head are a chain: many threads for many slots, fewer for short ones or where heads fill the SMs anyway.  (With the
  // move, 256 / 512 / 1024 threads: 32 heads of 200 slots 5.9 / 6.1 / 6.7 us, 1000 9.3 / 7.4 / 7.5, 4000 24 / 20 / 13; 1080 heads of 200
  // 9.6 / 13.7 / 23.7, of 1000 36 / 38 / 45, of 4000 119 / 121 / 130.)
  const int threads = from->slots <= 512 || (from->slots <= 4096 && (long long)B * KV > 2 * cq_sm_count()) ? 256 : (from->slots <= 1024 ? 512 : SEL_THREADS);
  CQ_CUDA_TRY(kv4_launch(kv4_select_kernel, dim3(KV, B), dim3(threads), 0, (cudaStream_t)stream, weights, length, length_out, kept,
                         weights_out, KV, from->slots, keep, sinks, recent));
  const size_t rows = (size_t)B * KV * keep;
  const int code = D / 2, scale = 4 * (D / from->group);
  uint8_t* ws = (uint8_t*)workspace;
  // codes in front: they are moved in pieces of 16 bytes, a row of scales may have four
  uint8_t* mid[4] = {ws, ws + 2 * rows * code, ws + rows * code, ws + rows * (2 * code + scale)};
  auto args = [](const void* const* f, void* const* t, int src_slots, int dst_slots, int n) {
    return MoveArgs{(const uint8_t*)f[0], (const uint8_t*)f[1], (const uint8_t*)f[2], (const uint8_t*)f[3], (uint8_t*)t[0], (uint8_t*)t[1],
                    (uint8_t*)t[2], (uint8_t*)t[3], src_slots, dst_slots, n};
  };
  const dim3 grid((keep + WR_TOKENS - 1) / WR_TOKENS, KV, B);
  void* over[4] = {mid[0], mid[1], mid[2], mid[3]};
  auto fn = KV4_PICK(kv4_gather_kernel, from);
  CQ_CUDA_TRY(kv4_launch(fn, grid, dim3(WR_THREADS), 0, (cudaStream_t)stream, args(fp, in_place ? over : tp, from->slots, in_place ? keep : to->slots, keep),
                         (const int*)kept));
  if (in_place)
    CQ_CUDA_TRY(kv4_launch(fn, grid, dim3(WR_THREADS), 0, (cudaStream_t)stream, args(over, tp, keep, to->slots, keep), (const int*)nullptr));
  return CQ_OK;
}
