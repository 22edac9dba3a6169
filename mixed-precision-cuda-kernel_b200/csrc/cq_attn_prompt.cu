// Attention of prompts, causal, with a sliding window and first keys that stay visible, grouped heads and ragged lengths; and
// the weight that every key received from a prompt's last queries.  In the reference it is torch's attention without window
// or lengths (llama/modeling_llama_quant.py:371-419 of the reference project).
//
//   p = i + keys - queries;  visible(i, j): j <= p, j < length, and (no window, or j < sinks, or j > p - window)
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,  lse_i = ln sum_j exp(scale q_i . k_j)
//   weights_j = sum of exp(scale q_i . k_j - lse_i) over the observed queries i of the KV head
//
// Both are tcgen05 kernels, a persistent CTA on every SM: tiles come by TMA, products are 128 x 128 into tensor memory, and the
// exponentials bound them.
#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstring>
#include <type_traits>

#include "cq_kv4.cuh"
#include "cq_umma.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// n / d for 0 <= n < 2^31 by one multiplication: m = floor(2^32 (2^shift - d) / d) + 1 with 2^shift >= d.  (Every warp of a CTA works out
// for itself what an item is; with the compiler's divisions, and absent blocks read and summed, the weights of the last 64 of 8192 queries of 32 heads took 38 us, 25 without.)
struct Divisor {
  uint32_t d = 1, m = 1, shift = 0;
  Divisor() = default;
  explicit Divisor(uint32_t by) : d(by) {
    while ((1ull << shift) < by) ++shift;
    m = (uint32_t)((((1ull << shift) - by) << 32) / by + 1);
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi(m, (uint32_t)n) + (uint32_t)n) >> shift); }
};

struct PromptArgs {
  cq_prompt s;
  const __half *q, *k, *v;
  const long long* lengths;
  int group;                                               // query heads of a KV head
  Divisor by_group, by_heads, by_row, by_parts;            // (what they divide: PromptItem, KeysItem)
  int rows = 256, shift = 8, pack = 1;                     // queries of a head in an item (2^shift), heads in it
};

__device__ __forceinline__ uint32_t half_pair(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ int length_of(const PromptArgs& a, int b) {
  if (!a.lengths) return a.s.keys;
  const long long n = a.lengths[b];
  return n < 0 ? 0 : (n > a.s.keys ? a.s.keys : (int)n);
}
// ------------------------------------------------------------------ attention
// A CTA takes two tiles of 128 queries of a head, one for each group of four softmax warps, and goes through the keys 128 at a
// time.  S = Q . K^T and O += P . V are tcgen05.mma of one CTA (128 x 128 x 16 a step), all accumulators in tensor memory:
// S of the two tiles, O of the two tiles, 512 columns; P takes the place of its S, as fp16, and is the A operand from there.
// While the softmax warps of one tile take exponentials, the tensor core works on the other tile.
//   warps 0-3, 4-7  softmax of a tile, a thread a query: row maximum, exponentials, row sum, P; O / sum at the end
//   warp 8          TMA of Q, K, V (128-byte swizzle, boxes of 64 columns x 128 rows; what lies outside reads as zeros)
//   warp 9          issues the MMAs; owns the tensor memory
// The reference of a row's exponentials is a whole number and only raised when a score is 2^8 above it, so that O is rescaled
// (tensor memory -> registers -> tensor memory) a few times in the first tiles and hardly ever afterwards.  P is rounded to
// fp16 (2^-11 of each weight; the row sum is of the unrounded ones, in fp32).
// Bound by the softmax phases: 2000 cycles for a tile with a warp a scheduler, and a tile's next scores wait for its weights, in whose
// place they go; two tiles by 128 keys take 3900 cycles, their MMAs alone 2160.  8192 tokens of 32 heads 1.03 PFLOP/s, 2048 of 40 heads
// 65 us, 8192 of 64 / 8 heads with a window of 2048 527 us in a burst, 610 once the power cap holds the clock at 1.69 GHz (normal
// random inputs).  Keys with a few columns four times as large, whose scores make rows raise their reference and take tiles twice: 77, 654 and
// 691 us.  Sixteen softmax warps of half a row spill (0.69 to 0.92 PFLOP/s), two MMA warps 0.83, two score buffers of 64 keys 0.50 to 0.61.
constexpr int UM_THREADS = 320, UM_TILE = 128, UM_STAGES = 4, UM_CHUNK = 64 * 128 * 2;      // bytes of 64 columns of a tile
constexpr int W_LOAD = 8, W_MMA = 9;
constexpr int POLY_OF_8 = 1;                      // of eight pairs of exponentials, how many are polynomials
constexpr float HEADROOM = 8.f, LIFT = 7.f, LOWEST = -4.f;      // weights are 2^7 times the exponentials, at most 2^15

// the key tiles that the queries at positions pmin .. pmax (both inside the length n) of a CTA see
struct KeyTiles {
  int ns = 0, wt0 = 0, count = 0, from = 0;
  __device__ __forceinline__ KeyTiles(const cq_prompt& s, int pmin, int pmax) {
    if (pmax < pmin) return;
    const int key = s.window ? max(0, pmin - s.window + 1) : 0, first = s.window ? min(s.sinks, key) : 0;
    ns = (first + UM_TILE - 1) / UM_TILE;
    wt0 = key / UM_TILE;
    if (ns >= wt0) ns = wt0 = 0;
    count = ns + pmax / UM_TILE + 1 - wt0;
  }
  __device__ __forceinline__ void cut(int part, const Divisor& parts) {      // to one of as many parts as equal as they can be
    const int each = parts(count), more = count - each * (int)parts.d;
    from = part * each + min(part, more);
    count = each + (part < more);
  }
  __device__ __forceinline__ int base(int i) const { return UM_TILE * (i + from < ns ? i + from : i + from - ns + wt0); }
};
// whether any of the queries pmin .. pmax sees a key of the tile; whether all of them see all of it
__device__ __forceinline__ bool tile_seen(const cq_prompt& s, int base, int pmin, int pmax) {
  return pmin <= pmax && base <= pmax && (!s.window || base < s.sinks || base + UM_TILE - 1 > pmin - s.window);
}
__device__ __forceinline__ bool tile_whole(const cq_prompt& s, int base, int pmin, int pmax, int n) {
  const int last = base + UM_TILE - 1;
  return last <= pmin && last < n && (!s.window || last < s.sinks || base > pmax - s.window);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x of two numbers up to 2^7 (ANY: of any, infinity from 2^7 on) on the multiply-add pipe: x = n + f with a whole n and |f| <= 1/2, by adding and taking away
// 1.5 * 2^23, then 2^f by the polynomial of degree 5 whose largest relative error is the least (2.1e-7 in fp32; coefficients by
// Remez's exchange; degree 4 is 2.6e-6, which the weights of keys show, and takes 1 % off a prompt) and 2^n as a bit pattern.  x is held at -127, whose bit pattern is that of 0: below 2^-126.5 the
// result is exactly 0, a masked score's of -infinity too (a row or key that sees nothing is known by a sum of 0).  NaN stays NaN.
template <bool ANY> __device__ __forceinline__ uint64_t power2(float2 x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-127.f));
  if (ANY) {
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(128.f));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(128.f));
  }
  const uint64_t v = two(x.x, x.y), big = two(12582912.f, 12582912.f), less = two(-12582912.f, -12582912.f);
  const uint64_t t = add2(v, big), f = fma2(add2(t, less), two(-1.f, -1.f), v);
  uint64_t p = fma2(f, two(0.0013276472454890609f, 0.0013276472454890609f), two(0.009675540961325169f, 0.009675540961325169f));
  p = fma2(p, f, two(0.05550713092088699f, 0.05550713092088699f));
  p = fma2(p, f, two(0.24022120237350464f, 0.24022120237350464f));
  p = fma2(p, f, two(0.6931469440460205f, 0.6931469440460205f));
  p = fma2(p, f, two(1.0000001192092896f, 1.0000001192092896f));
  const float2 n = apart(t);
  return mul2(p, two(__uint_as_float((__float_as_uint(n.x) << 23) + 0x3F800000u), __uint_as_float((__float_as_uint(n.y) << 23) + 0x3F800000u)));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A mean of finite values is none of fp16's infinities, but where they are near its largest number the weights' roundings can carry it there.
// (Looking at a row's largest sum and holding it is 1 % of a prompt.)
constexpr float LARGEST = 65504.f;
__device__ __forceinline__ float within(float x, float most) { return fabsf(x) < INFINITY ? fminf(fmaxf(x, -most), most) : x; }

// which of the 32 keys from `first` on a query sees that sees lo .. hi and those below `sinks`: a bit each
__device__ __forceinline__ uint32_t below32(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u); }
__device__ __forceinline__ uint32_t visible32(int first, int lo, int hi, int sinks) {
  return below32(hi + 1 - first) & (~below32(lo - first) | below32(sinks - first));
}

struct PromptMaps {
  CUtensorMap q, k, v;
  int one[3][2];             // 0 where the heads (0) or sequences (1) of q, k, v are all the same rows
};

// The work of a CTA: every gridDim.x-th item, the longest first, forwards and backwards in turn.
__device__ __forceinline__ int item_at(int round, int items) {
  const int i = round * (int)gridDim.x + (int)(round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  return i < items ? i : -1;
}

// An item is 256 queries of a head,
// or where calls have few of them (FEW) one of several parts of such an item's keys, and where they have 128 at most the queries
// of several heads of a KV head, `rows` places each.
template <bool FEW>
struct PromptItem {
  int b, h, kvh, q0, n, pmin, pmax;          // positions of the queries that are inside the length
  int part = 0, heads = 1;
  __device__ __forceinline__ PromptItem(const PromptArgs& a, int item) {
    const cq_prompt& s = a.s;
    const int whole = FEW ? a.by_parts(item) : item, rows = FEW ? a.rows : 2 * UM_TILE;
    const int row = a.by_row(whole), rest = whole - row * (int)a.by_row.d;
    b = a.by_heads(rest);
    h = rest - b * (int)a.by_heads.d;
    kvh = a.by_group(h);
    if (FEW) {
      part = item - whole * (int)a.by_parts.d;
      const int first = (h - kvh * (int)a.by_group.d) * a.pack;
      h = kvh * a.group + first;
      heads = min(a.pack, a.group - first);
    }
    q0 = ((FEW ? (s.queries + rows - 1) >> a.shift : (s.queries + rows - 1) / (2 * UM_TILE)) - 1 - row) * rows;
    n = length_of(a, b);
    pmin = q0 + s.keys - s.queries;
    pmax = min(n, min(q0 + rows, s.queries) + s.keys - s.queries) - 1;
  }
  // of tile t
  __device__ __forceinline__ static bool packed(const PromptArgs& a) { return FEW && a.rows <= UM_TILE; }
  __device__ __forceinline__ int lowest(const PromptArgs& a, int t) const { return packed(a) ? pmin : pmin + UM_TILE * t; }
  __device__ __forceinline__ int highest(const PromptArgs& a, int t) const {
    if (packed(a)) return heads * a.rows > UM_TILE * t ? pmax : -1;
    return min(pmax, pmin + UM_TILE * t + UM_TILE - 1);
  }
  // of row x of the 256
  __device__ __forceinline__ int query(const PromptArgs& a, int x) const { return q0 + (packed(a) ? x & (a.rows - 1) : x); }
  __device__ __forceinline__ int head(const PromptArgs& a, int x) const { return packed(a) ? x >> a.shift : 0; }
};

// A value in a masked place has the weight 0, and 0 times infinity or NaN is NaN: where a row with a finite lse has a NaN, a warp
// sums its columns with one again, in fp32, over the keys that the row sees.  (Finite values never come here.)
template <int D>
__device__ __noinline__ void row_again(const PromptArgs& a, int b, int h, int q, __half* out, const float* lse) {
  constexpr int C = D / 32;                                // columns of a lane
  const cq_prompt& s = a.s;
  const int lane = threadIdx.x & 31, kvh = h / a.group;
  __half* to = out + (((size_t)b * s.queries + q) * s.n_heads + h) * D + C * lane;
  const float l = lse[((size_t)b * s.n_heads + h) * s.queries + q];
  bool mine = false;
#pragma unroll
  for (int i = 0; i < C; ++i) mine |= __hisnan(to[i]);
  if (!(fabsf(l) < INFINITY) || !__any_sync(0xffffffffu, mine)) return;
  const __half* ks = a.k + b * s.k_strides[0] + kvh * s.k_strides[2] + C * lane;
  const __half* vs = a.v + b * s.v_strides[0] + kvh * s.v_strides[2] + C * lane;
  const __half* qr = a.q + b * s.q_strides[0] + q * s.q_strides[1] + h * s.q_strides[2] + C * lane;
  float x[C], y[C] = {};
#pragma unroll
  for (int i = 0; i < C; ++i) x[i] = __half2float(qr[i]) * (s.scale * LOG2E);
  const int hi = q + s.keys - s.queries, lo = s.window ? max(0, hi - s.window + 1) : 0;
  bool done = false;                                   // NaN again: the row sees one
  for (int from = 0, to_key; from <= hi && !done; from = to_key) {
    if (from >= s.sinks && from < lo) from = lo;
    to_key = min(min(from + 128, hi + 1), from < min(s.sinks, lo) ? min(s.sinks, lo) : hi + 1);
#pragma unroll 4
    for (int j = from; j < to_key; ++j) {
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < C; ++i) dot = fmaf(x[i], __half2float(ks[j * s.k_strides[1] + i]), dot);
#pragma unroll
      for (int d = 16; d; d /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, d);
      const float p = exp2f(dot - l * LOG2E);
#pragma unroll
      for (int i = 0; i < C; ++i) y[i] = fmaf(p, __half2float(vs[j * s.v_strides[1] + i]), y[i]);
    }
    done = true;
#pragma unroll
    for (int i = 0; i < C; ++i) done = done && (y[i] != y[i] || !__hisnan(to[i]));
    done = __all_sync(0xffffffffu, done);
  }
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (__hisnan(to[i])) to[i] = __float2half_rn(y[i]);
}
// the rows of a softmax warp, at the CTA's end, where no other warp waits
template <int D, bool FEW>
__device__ __noinline__ void rows_again(const PromptArgs& a, int items, __half* out, const float* lse) {
  const int warp = threadIdx.x >> 5;
  for (int round = 0, item; (item = item_at(round, items)) >= 0; ++round) {
    const PromptItem<FEW> w(a, item);
    for (int x = 32 * warp; x < 32 * warp + 32; ++x)
      if (w.query(a, x) < a.s.queries && w.head(a, x) < w.heads) row_again<D>(a, w.b, w.h + w.head(a, x), w.query(a, x), out, lse);
  }
}

template <int D, bool FEW>
__global__ void __launch_bounds__(UM_THREADS, 1) prompt_kernel(const __grid_constant__ PromptArgs a, const __grid_constant__ PromptMaps maps,
                                                                    __half* __restrict__ out, float* __restrict__ lse, float* __restrict__ partial, int items,
                                                                    uint32_t* __restrict__ status) {
  using namespace umma;
  constexpr int CH = D / 64, TILE_BYTES = CH * UM_CHUNK;
  extern __shared__ __align__(1024) uint8_t um_smem[];
  __shared__ __align__(8) uint64_t s_bar[3 + 2 * UM_STAGES + 6];
  __shared__ uint32_t s_tmem;
  __shared__ int s_gone;
  __shared__ int s_nan[W_LOAD];                            // a softmax warp met a NaN in a sum
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t smem = (smem_at(um_smem) + 1023u) & ~1023u, s_q = smem, s_kv = smem + 2 * TILE_BYTES;
  const uint32_t bars = smem_at(s_bar);
  const uint32_t q_full = bars, q_free = bars + 8, drained = bars + 16;
  auto kv_full = [&](int st) { return bars + 8 * (3 + st); };
  auto kv_free = [&](int st) { return bars + 8 * (3 + UM_STAGES + st); };
  auto s_full = [&](int t) { return bars + 8 * (3 + 2 * UM_STAGES + t); };
  auto p_full = [&](int t) { return bars + 8 * (5 + 2 * UM_STAGES + t); };
  auto o_done = [&](int t) { return bars + 8 * (7 + 2 * UM_STAGES + t); };
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    bar_init(q_full, 1);
    bar_init(q_free, 1);
    bar_init(drained, 1);
    for (int i = 0; i < UM_STAGES; ++i) {
      bar_init(kv_full(i), 1);
      bar_init(kv_free(i), 1);
    }
    for (int t = 0; t < 2; ++t) {
      bar_init(s_full(t), 1);
      bar_init(p_full(t), 128);
      bar_init(o_done(t), 1);
    }
    s_gone = 0;
    for (int i = 0; i < W_LOAD; ++i) s_nan[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == W_MMA) alloc(&s_tmem, 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s_tmem;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const cq_prompt& s = a.s;

  if (warp >= W_LOAD) {
    if (warp == W_LOAD && lane == 0) {
      int loaded = 0, sent = 0;                            // query blocks, tiles of keys and values
      bool ok = true;
      for (int round = 0, item; ok && (item = item_at(round, items)) >= 0; ++round) {
        const PromptItem<FEW> w(a, item);
        KeyTiles tiles(s, w.pmin, w.pmax);
        if (FEW) tiles.cut(w.part, a.by_parts);
        if (!tiles.count) continue;
        if (loaded && !(ok = bar_wait(q_free, (loaded - 1) & 1, &s_gone, status))) break;
        if (w.packed(a)) {
          bar_expect(q_full, w.heads * a.rows * D * 2);
          for (int e = 0; e < w.heads; ++e)
            for (int c = 0; c < CH; ++c)
              tma(s_q + e * a.rows / UM_TILE * TILE_BYTES + c * UM_CHUNK + e * a.rows % UM_TILE * 128, &maps.q, 64 * c, w.q0, (w.h + e) * maps.one[0][0],
                  w.b * maps.one[0][1], q_full);
        } else {
          bar_expect(q_full, 2 * TILE_BYTES);
          for (int t = 0; t < 2; ++t)
            for (int c = 0; c < CH; ++c)
              tma(s_q + t * TILE_BYTES + c * UM_CHUNK, &maps.q, 64 * c, w.q0 + UM_TILE * t, w.h * maps.one[0][0], w.b * maps.one[0][1], q_full);
        }
        ++loaded;
        for (int i = 0; i < 2 * tiles.count; ++i, ++sent) {      // keys, values, keys, values ...
          const int st = sent % UM_STAGES, use = sent / UM_STAGES;
          if (use && !(ok = bar_wait(kv_free(st), (use - 1) & 1, &s_gone, status))) break;
          bar_expect(kv_full(st), TILE_BYTES);
          const int which = i & 1 ? 2 : 1;
          for (int c = 0; c < CH; ++c)
            tma(s_kv + st * TILE_BYTES + c * UM_CHUNK, which == 1 ? &maps.k : &maps.v, 64 * c, tiles.base(i / 2), w.kvh * maps.one[which][0],
                w.b * maps.one[which][1], kv_full(st));
        }
      }
      if (!ok) {                                           // copies in flight end before the CTA does
        for (int k = 0; loaded && k < 1000 && !bar_try(q_full, (loaded - 1) & 1); ++k) {}
        for (int i = max(0, sent - UM_STAGES); i < sent; ++i)
          for (int k = 0; k < 1000 && !bar_try(kv_full(i % UM_STAGES), (i / UM_STAGES) & 1); ++k) {}
      }
    } else if (warp == W_MMA) {
      constexpr uint32_t SHAPE_S = shape_of(128, 128, false), SHAPE_O = shape_of(128, D, true);
      int taken[2] = {0, 0};                               // tiles of keys that a query tile has taken, in all items
      int blocks = 0, sent = 0;
      bool ok = true;
      for (int round = 0, item; ok && (item = item_at(round, items)) >= 0; ++round) {
        const PromptItem<FEW> w(a, item);
        KeyTiles tiles(s, w.pmin, w.pmax);
        if (FEW) tiles.cut(w.part, a.by_parts);
        if (!tiles.count) continue;
        auto seen = [&](int t, int i) { return tile_seen(s, tiles.base(i), w.lowest(a, t), w.highest(a, t)); };
        auto scores = [&](int t, int i) {
          if (elected()) {
            const uint32_t kt = s_kv + ((sent + 2 * i) % UM_STAGES) * TILE_BYTES, qt = s_q + t * TILE_BYTES;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t at = (k / 4) * UM_CHUNK + (k % 4) * 32;
              mma_ss(tmem + 128 * t, operand(qt + at, 0), operand(kt + at, 0), SHAPE_S, k > 0);
            }
            commit(s_full(t));
          }
          __syncwarp();
        };
        bool first[2] = {true, true};
        ok = bar_wait_warp(q_full, blocks & 1, &s_gone, status) && bar_wait_warp(kv_full(sent % UM_STAGES), (sent / UM_STAGES) & 1, &s_gone, status);
        if (!ok) break;
        ++blocks;
        fence_after();
        for (int t = 0; t < 2; ++t)
          if (seen(t, 0)) scores(t, 0);
        if (elected()) {
          commit(kv_free(sent % UM_STAGES));
          if (tiles.count == 1) commit(q_free);
        }
        __syncwarp();
        for (int i = 0; i < tiles.count && ok; ++i) {
          const int vi = sent + 2 * i + 1, ki = vi + 1, sv = vi % UM_STAGES;
          const bool next = i + 1 < tiles.count;
          ok = bar_wait_warp(kv_full(sv), (vi / UM_STAGES) & 1, &s_gone, status);
          if (ok && next) ok = bar_wait_warp(kv_full(ki % UM_STAGES), (ki / UM_STAGES) & 1, &s_gone, status);
          if (!ok) break;
          const int base = tiles.base(i);
          if (base + UM_TILE > w.n && w.n < s.keys) {
            // Rows behind the sequence's end may hold anything, and 0 times NaN is NaN.
            uint8_t* vt = um_smem + (s_kv + sv * TILE_BYTES - smem_at(um_smem));
            for (int r = w.n - base; r < UM_TILE; ++r)
              for (int c = lane; c < CH * 8; c += 32) *reinterpret_cast<uint4*>(vt + (c / 8) * UM_CHUNK + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
            fence_async();
            __syncwarp();
          }
          for (int t = 0; t < 2 && ok; ++t) {
            if (seen(t, i)) {
              ok = bar_wait_warp(p_full(t), taken[t] & 1, &s_gone, status);
              if (!ok) break;
              fence_after();
              if (elected()) {
                const uint32_t vt = s_kv + sv * TILE_BYTES;
#pragma unroll
                for (int k = 0; k < UM_TILE / 16; ++k)
                  mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k, operand(vt + k * 2048, UM_CHUNK), SHAPE_O, !first[t] || k > 0);
                commit(o_done(t));
              }
              __syncwarp();
              first[t] = false;
              ++taken[t];
            }
            if (next && seen(t, i + 1)) scores(t, i + 1);
          }
          if (ok && elected()) {
            commit(kv_free(sv));
            if (next) commit(kv_free(ki % UM_STAGES));
            if (i + 2 == tiles.count) commit(q_free);      // the last scores of these queries are on their way
          }
          __syncwarp();
        }
        sent += 2 * tiles.count;
      }
      // nothing is in flight when the tensor memory is given back and the CTA ends
      if (elected()) commit(drained);
      for (int k = 0; k < 100000 && !bar_try(drained, 0); ++k) {}
      __syncwarp();
    }
  } else {
    const int t = warp >> 2, r = tid & 127;
    const uint32_t at_s = tmem + 128 * t + ((uint32_t)(warp & 3) << 21), at_o = at_s + 256;
    const float scale2 = s.scale * LOG2E;
    const uint64_t scale22 = two(scale2, scale2);
    int taken = 0;                                         // tiles of keys, in all items
    bool ok = true;
    for (int round = 0, item; (item = item_at(round, items)) >= 0; ++round) {
      const PromptItem<FEW> w(a, item);
      KeyTiles tiles(s, w.pmin, w.pmax);
      if (FEW) tiles.cut(w.part, a.by_parts);
      const int q = w.query(a, UM_TILE * t + r), p = q + s.keys - s.queries, head = w.h + w.head(a, UM_TILE * t + r);
      const int hi = min(p, w.n - 1), lo = s.window ? p - s.window + 1 : 0;
      float ref = -INFINITY;
      uint64_t sum = 0;                                    // two partial sums
      bool first = true;
      for (int i = 0; i < tiles.count && ok; ++i) {
        const int base = tiles.base(i);
        if (!tile_seen(s, base, w.lowest(a, t), w.highest(a, t))) continue;
        ok = bar_wait_warp(s_full(t), taken & 1, &s_gone, status);
        if (!ok) break;
        fence_after();
        const bool whole = tile_whole(s, base, w.lowest(a, t), w.highest(a, t), w.n);
        // Exponentials with the reference as it is, the maximum on the way: where it shows that the reference has to rise (or a
        // first guess of 0 was too high), the tile is taken again, once.  P leaves the registers when that is known.
        uint32_t pr[64];
        uint64_t here;
        for (;;) {
          const float minus = LIFT - (ref == -INFINITY ? 0.f : ref);
          const uint64_t minus2 = two(minus, minus);
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          here = 0;
#pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 64) {
            uint32_t x[64];
            load32(at_s + c0, x);
            load32(at_s + c0 + 32, x + 32);
            wait_load<32>(x);
            wait_load<32>(x + 32);
            if (!whole) {
#pragma unroll
              for (int g = 0; g < 64; g += 32) {
                const uint32_t vis = visible32(base + c0 + g, lo, hi, s.sinks);
#pragma unroll
                for (int c = 0; c < 32; ++c) x[g + c] = vis >> c & 1u ? x[g + c] : 0xFF800000u;
              }
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float2 f = apart(fma2(two(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), scale22, minus2));
              const uint64_t z = e % 8 < POLY_OF_8 ? power2<false>(f) : two(ex2(f.x), ex2(f.y));
              here = add2(here, z);
              const float2 g = apart(z);
              pr[c0 / 2 + e] = half_pair(g.x, g.y);
              top[e % 4] = max3(top[e % 4], __uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
            }
          }
          const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale2;
          const bool unset = ref == -INFINITY;
          const bool again = most > (unset ? 0.f : ref) + HEADROOM || (unset && most < LOWEST && most != -INFINITY);
          if (!__any_sync(0xffffffffu, again)) {
            if (unset && most != -INFINITY) ref = 0.f;
            break;
          }
          const float now = again ? ceilf(most) : ref, keep = again && !unset ? ex2(ref - now) : 1.f;
          ref = now;
          sum = mul2(sum, two(keep, keep));
          if (!first) {
            if (!(ok = bar_wait_warp(o_done(t), (taken - 1) & 1, &s_gone, status))) break;
            fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              uint32_t y[16];
              load16(at_o + c, y);
              wait_load<16>(y);
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * keep);
              store16(at_o + c, y);
            }
          }
        }
        if (!ok) break;
        sum = add2(sum, here);
        store32(at_s, pr);
        store32(at_s + 32, pr + 32);
        wait_store();
        fence_before();
        bar_arrive(p_full(t));
        first = false;
        ++taken;
      }
      const float2 parts = apart(sum);
      const float total = parts.x + parts.y;
      const bool row = q < s.queries && head < w.h + w.heads, empty = first || p >= w.n || (ref == -INFINITY && total == 0.f);
      if (ok && !first) ok = bar_wait_warp(o_done(t), (taken - 1) & 1, &s_gone, status);
      fence_after();
      const float inv = empty ? 0.f : 1.f / total;
      const size_t at_row = ((size_t)w.b * s.queries + q) * s.n_heads + head, rows = (size_t)s.sequences * s.queries * s.n_heads;
      const bool cut = FEW && a.by_parts.d > 1;            // a part of the row: fp32, and its sum
      float* to32 = partial + (w.part * rows + at_row) * D;
      __half* to = out + at_row * D;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t y[32];
        if (!first && ok) {
          load32(at_o + c, y);
          wait_load<32>(y);
        }
        if (!row) continue;
        if (cut) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = empty ? 0.f : __uint_as_float(y[e + k]) * inv;
            *reinterpret_cast<float4*>(to32 + c + e) = make_float4(v[0], v[1], v[2], v[3]);
          }
          continue;
        }
        uint64_t all[2] = {};
#pragma unroll
        for (int e = 0; e < 16; ++e) all[e & 1] = add2(all[e & 1], two(__uint_as_float(y[2 * e]), __uint_as_float(y[2 * e + 1])));
        const float2 any = apart(add2(all[0], all[1]));
        if (!empty && (any.x != any.x || any.y != any.y)) s_nan[warp] = 1;      // (an empty row's sums may be anything)
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < 32; ++e) most = fmaxf(most, fabsf(__uint_as_float(y[e])));
        if (most * inv > LARGEST)
#pragma unroll
          for (int e = 0; e < 32; ++e) y[e] = __float_as_uint(within(__uint_as_float(y[e]), LARGEST * total));
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint32_t v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = half_pair(__uint_as_float(y[e + 2 * k]) * inv, __uint_as_float(y[e + 2 * k + 1]) * inv);
          *reinterpret_cast<uint4*>(to + c + e) = !ok ? make_uint4(~0u, ~0u, ~0u, ~0u) : (empty ? make_uint4(0, 0, 0, 0) : make_uint4(v[0], v[1], v[2], v[3]));
        }
      }
      const float total2 = !ok ? NAN : (empty ? -INFINITY : (ref == -INFINITY ? 0.f : ref) - LIFT + log2f(total));
      if (row && cut) partial[a.by_parts.d * rows * D + w.part * rows + at_row] = total2;
      else if (row) lse[((size_t)w.b * s.n_heads + head) * s.queries + q] = total2 * LN2;
    }
  }
  fence_before();
  __syncthreads();
  if (warp == W_MMA) {
    fence_after();
    dealloc(tmem, 512);
  }
  if (warp < W_LOAD && s_nan[warp]) rows_again<D, FEW>(a, items, out, lse);
}

// a row's parts: out = sum 2^(l_p - l) out_p, l = log2 of the sum of 2^(l_p); a warp a row
template <int D>
__global__ void __launch_bounds__(256) prompt_sum_kernel(const __grid_constant__ PromptArgs a, const float* __restrict__ partial, __half* out, float* lse) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int C = D / 32;
  const cq_prompt& s = a.s;
  const int lane = threadIdx.x & 31, parts = (int)a.by_parts.d;
  const size_t rows = (size_t)s.sequences * s.queries * s.n_heads, row = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const float l = lane < parts ? partial[parts * rows * D + lane * rows + row] : -INFINITY;
  float top = l;
#pragma unroll
  for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float f = l == -INFINITY ? 0.f : exp2f(l - (top == -INFINITY ? 0.f : top));
  float sum = f;
#pragma unroll
  for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  float y[C] = {};
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const float w = __shfl_sync(0xffffffffu, f, p);
    const float* from = partial + (p * rows + row) * D + C * lane;
#pragma unroll
    for (int i = 0; i < C; ++i) y[i] = fmaf(w, from[i], y[i]);
  }
  const bool empty = sum == 0.f;
  const float inv = empty ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < C; i += 2)
    *reinterpret_cast<uint32_t*>(out + row * D + C * lane + i) = half_pair(within(y[i] * inv, LARGEST), within(y[i + 1] * inv, LARGEST));
  const int h = (int)(row % s.n_heads), q = (int)(row / s.n_heads % s.queries), b = (int)(row / s.n_heads / s.queries);
  if (lane == 0) lse[((size_t)b * s.n_heads + h) * s.queries + q] = empty ? -INFINITY : (top + log2f(sum)) * LN2;
  __syncwarp();
  bool broken = false;
#pragma unroll
  for (int i = 0; i < C; ++i) broken |= y[i] != y[i];
  if (__any_sync(0xffffffffu, broken)) row_again<D>(a, b, h, q, out, lse);
}

// The form of a call: queries of a head side by side (`rows`), heads in an item (`pack`), parts of its keys.
struct PromptForm {
  int rows = 256, pack = 1, parts = 1;
  int units(const cq_prompt* s) const { return (s->n_heads / s->n_kv_heads + pack - 1) / pack; }      // items of a KV head, a block of queries, a part
  long long items(const cq_prompt* s) const {
    return (long long)((s->queries + rows - 1) / rows) * s->n_kv_heads * units(s) * s->sequences * parts;
  }
};
// key tiles that the block's queries see
int tiles_of(const cq_prompt* s, int block, int rows) {
  const int off = s->keys - s->queries, pmin = block * rows + off, pmax = std::min((block + 1) * rows, s->queries) + off - 1;
  const int key = s->window ? std::max(0, pmin - s->window + 1) : 0, ns = (std::min(s->window ? s->sinks : 0, key) + UM_TILE - 1) / UM_TILE;
  const int wt0 = key / UM_TILE;
  return pmax / UM_TILE + 1 - (ns >= wt0 ? 0 : wt0 - ns);
}
// What the first and the last CTA have to do, the longer of the two, in tiles of 256 x 128 x 128 (about 1.9 us): 0.7 where one tile of
// 128 queries is all there is or heads are 64 wide, 2 for an item; and for joining the parts 2, and 0.5 for a million of numbers.  On 36 shapes of 1
// to 5000 queries its choice is 0.4 % slower than the best, 8 % at most.  (16 queries of 64 / 8 heads over 4000 keys: 60 us as whole heads, 18 so;
// 512 of 32 heads over 4096 72 and 55; 100 of 8 / 1 over 20000 273 and 34; 2048 over their own keys stay whole, 36 us, 40 in two.)
double prompt_cost(const cq_prompt* s, const PromptForm& f) {
  const int blocks = (s->queries + f.rows - 1) / f.rows, sms = cq_sm_count();
  const long long items = f.items(s), row = items / blocks;
  const bool one = s->queries <= UM_TILE && f.pack * f.rows <= 256 && (f.rows == 256 || f.pack * f.rows <= UM_TILE);
  const double tile = (one ? 0.7 : 1.0) * (s->head_dim == 128 ? 1.0 : 0.7);
  double most = 0;
  for (int last = 0; last < 2; ++last) {
    double t = 0;
    for (long long j = 0;; ++j) {
      const long long i = j * sms + ((j & 1) != last ? sms - 1 : 0);
      if (i >= items) break;
      t += (tiles_of(s, blocks - 1 - (int)(i / row), f.rows) + f.parts - 1) / f.parts * tile + 2;
    }
    most = std::max(most, t);
  }
  return most + (f.parts > 1 ? 2 + 0.5e-6 * f.parts * s->sequences * s->queries * s->n_heads * s->head_dim : 0);
}
PromptForm prompt_form(const cq_prompt* s) {
  static thread_local cq_prompt last = {};
  static thread_local PromptForm kept;                     // (of the last call's shape)
  if (!memcmp(&last, s, offsetof(cq_prompt, q_strides))) return kept;
  const int G = s->n_heads / s->n_kv_heads, sms = cq_sm_count();
  PromptForm best, f;
  if (best.items(s) < 4ll * sms) {                         // (more items fill the SMs as they are)
    double least = prompt_cost(s, best);
    for (int packed = 0; packed < 2; ++packed) {
      if (packed) {
        if (s->queries > UM_TILE || G == 1) break;
        for (f.rows = 8; f.rows < s->queries;) f.rows *= 2;
        f.pack = std::min(G, 256 / f.rows);
      }
      const int most = tiles_of(s, (s->queries + f.rows - 1) / f.rows - 1, f.rows);
      for (f.parts = 1; f.parts <= std::min(16, most) && (f.parts == 1 || f.items(s) <= 3ll * sms); ++f.parts) {
        const double t = prompt_cost(s, f);
        if (t < least) {
          least = t;
          best = f;
        }
      }
    }
  }
  last = *s;
  return kept = best;
}

// ------------------------------------------------------------------ weights of the keys
// S^T = K . Q^T of 128 keys (lanes of tensor memory, a thread each) and 128 queries (columns): a key's weight is a sum along
// its thread's own columns, so nothing is exchanged.  The columns are two blocks of 64 queries, of any two heads and places:
// queries of a head that are fewer than 128 do not leave a tile half empty.  Bound by the exponentials, one for each pair and
// 16 a cycle and SM (1024 cycles a tile, its MMAs 540); some of them are polynomials.
//   warps 0-15  four groups, every fourth tile each: sums of exponentials, joined by the group with an item's last tile
//   warp 16     TMA of K, Q;  warp 17  MMAs, up to four score buffers ahead
// (Two groups that met at every item's end were 47.6 us for 2048 tokens of 40 heads of 128 and 490 for 8192 of 64 / 8 heads with
// window and sinks, four are 36 and 363: two warps a scheduler leave most of their instructions' latency open.)
constexpr int KW_GROUPS = 4, KW_THREADS = 128 * KW_GROUPS + 64, KW_Q = 64, KW_BUFFERS = 4;
constexpr int KW_LOAD = 4 * KW_GROUPS, KW_MMA = KW_LOAD + 1, KW_SLOTS = 12;
static_assert(KW_GROUPS == KW_BUFFERS, "a group's tiles come in one buffer");
constexpr int KW_POLY_OF_8 = 1;                   // as POLY_OF_8

// An item: 128 keys of a KV head, the queries [first, last) of its heads in blocks of 64, and of those one of `parts` parts
struct KeysItem {
  int b, kvh, k0, n, first, last, per_head, begin, blocks, tiles, part;
  __device__ __forceinline__ KeysItem(const PromptArgs& a, int item, int observe) {
    const cq_prompt& s = a.s;
    const int row = a.by_row(item), in_row = item - row * (int)a.by_row.d, rest = a.by_parts(in_row);
    part = in_row - rest * (int)a.by_parts.d;
    k0 = row * UM_TILE;
    b = a.by_heads(rest);
    kvh = rest - b * s.n_kv_heads;
    n = length_of(a, b);
    first = max(max(s.keys - s.queries, n - observe), k0);
    last = s.window && k0 >= s.sinks ? (int)min((long long)n, min(k0 + UM_TILE, n) - 1 + (long long)s.window) : n;
    per_head = max(0, last - first + KW_Q - 1) / KW_Q;
    const int all = per_head * a.group, each = a.by_parts(all), more = all - each * (int)a.by_parts.d;
    begin = part * each + min(part, more);
    blocks = each + (part < more);
    tiles = (blocks + 1) / 2;
  }
};
// a block's head (of the KV head's) and place in it; steps forward without a division
struct Block {
  int head, at;
  __device__ __forceinline__ explicit Block(const KeysItem& w, int n) : head(0), at(0) {
    if (w.blocks) {
      head = (w.begin + n) / w.per_head;
      at = w.begin + n - head * w.per_head;
    }
  }
  __device__ __forceinline__ void step(const KeysItem& w, int n) {
    at += n;
    while (at >= w.per_head) {
      at -= w.per_head;
      ++head;
    }
  }
  __device__ __forceinline__ int position(const KeysItem& w) const { return w.first + KW_Q * at; }
};

template <int D>
__global__ void __launch_bounds__(KW_THREADS, 1) prompt_keys_kernel(const __grid_constant__ PromptArgs a, const __grid_constant__ PromptMaps maps,
                                                                    const float* __restrict__ lse, int observe, float* __restrict__ weights, int items,
                                                                    uint32_t* __restrict__ status) {
  using namespace umma;
  constexpr int CH = D / 64, TILE_BYTES = CH * UM_CHUNK;
  extern __shared__ __align__(1024) uint8_t um_smem[];
  __shared__ __align__(8) uint64_t s_bar[5 + 4 * KW_BUFFERS + KW_SLOTS];
  __shared__ __align__(16) float s_lse[2 * KW_GROUPS][UM_TILE];
  __shared__ float s_sum[KW_SLOTS][KW_GROUPS][UM_TILE];
  __shared__ uint32_t s_tmem;
  __shared__ int s_gone;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t smem = (smem_at(um_smem) + 1023u) & ~1023u, s_k = smem, s_q = smem + 2 * TILE_BYTES;
  const uint32_t bars = smem_at(s_bar), drained = bars;
  auto k_full = [&](int i) { return bars + 8 * (1 + i); };
  auto k_free = [&](int i) { return bars + 8 * (3 + i); };
  auto q_full = [&](int i) { return bars + 8 * (5 + i); };
  auto q_free = [&](int i) { return bars + 8 * (5 + KW_BUFFERS + i); };
  auto s_full = [&](int i) { return bars + 8 * (5 + 2 * KW_BUFFERS + i); };
  auto s_free = [&](int i) { return bars + 8 * (5 + 3 * KW_BUFFERS + i); };
  auto summed = [&](int i) { return bars + 8 * (5 + 4 * KW_BUFFERS + i); };
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    bar_init(drained, 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(k_full(i), 1);
      bar_init(k_free(i), 1);
    }
    for (int i = 0; i < KW_BUFFERS; ++i) {
      bar_init(q_full(i), 1);
      bar_init(q_free(i), 1);
      bar_init(s_full(i), 1);
      bar_init(s_free(i), 128);
    }
    for (int i = 0; i < KW_SLOTS; ++i) bar_init(summed(i), 4 * KW_GROUPS);
    s_gone = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == KW_MMA) alloc(&s_tmem, 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s_tmem;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const cq_prompt& s = a.s;
  const int off = s.keys - s.queries, G = a.group;

  if (warp == KW_LOAD) {
    if (lane == 0) {
      uint32_t loaded = 0, sent = 0;                       // key tiles, query tiles
      bool ok = true;
      for (int round = 0, item; ok && (item = item_at(round, items)) >= 0; ++round) {
        const KeysItem w(a, item, observe);
        if (!w.tiles) continue;
        const uint32_t kb = loaded & 1;
        if (loaded >= 2 && !(ok = bar_wait(k_free(kb), (loaded / 2 - 1) & 1, &s_gone, status))) break;
        bar_expect(k_full(kb), TILE_BYTES);
        for (int c = 0; c < CH; ++c)
          tma(s_k + kb * TILE_BYTES + c * UM_CHUNK, &maps.k, 64 * c, w.k0, w.kvh * maps.one[1][0], w.b * maps.one[1][1], k_full(kb));
        ++loaded;
        Block block(w, 0);
        for (int j = 0; j < w.tiles; ++j, ++sent) {
          const uint32_t st = sent % KW_BUFFERS, use = sent / KW_BUFFERS;
          if (use && !(ok = bar_wait(q_free(st), (use - 1) & 1, &s_gone, status))) break;
          const int here = min(2, w.blocks - 2 * j);       // (the last tile may have one block: the other place is not read)
          bar_expect(q_full(st), here * (TILE_BYTES / 2));
          for (int e = 0; e < here; ++e) {
            for (int c = 0; c < CH; ++c)
              tma(s_q + st * TILE_BYTES + c * UM_CHUNK + e * (UM_CHUNK / 2), &maps.q, 64 * c, block.position(w) - off,
                  (w.kvh * G + block.head) * maps.one[0][0], w.b * maps.one[0][1], q_full(st));
            block.step(w, 1);
          }
        }
      }
      if (!ok) {                                           // copies in flight end before the CTA does
        for (uint32_t i = loaded > 2 ? loaded - 2 : 0; i < loaded; ++i)
          for (int k = 0; k < 1000 && !bar_try(k_full(i & 1), (i / 2) & 1); ++k) {}
        for (uint32_t i = sent > KW_BUFFERS ? sent - KW_BUFFERS : 0; i < sent; ++i)
          for (int k = 0; k < 1000 && !bar_try(q_full(i % KW_BUFFERS), (i / KW_BUFFERS) & 1); ++k) {}
      }
    }
  } else if (warp == KW_MMA) {
    constexpr uint32_t SHAPE = shape_of(128, 128, false);
    uint32_t loaded = 0, sent = 0;
    bool ok = true;
    for (int round = 0, item; ok && (item = item_at(round, items)) >= 0; ++round) {
      const KeysItem w(a, item, observe);
      if (!w.tiles) continue;
      const uint32_t kb = loaded & 1;
      ok = bar_wait_warp(k_full(kb), (loaded / 2) & 1, &s_gone, status);
      for (int j = 0; j < w.tiles && ok; ++j, ++sent) {
        const uint32_t st = sent % KW_BUFFERS, use = sent / KW_BUFFERS;
        ok = bar_wait_warp(q_full(st), use & 1, &s_gone, status) && (!use || bar_wait_warp(s_free(st), (use - 1) & 1, &s_gone, status));
        if (!ok) break;
        fence_after();
        if (elected()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = (k / 4) * UM_CHUNK + (k % 4) * 32;
            mma_ss(tmem + 128 * st, operand(s_k + kb * TILE_BYTES + at, 0), operand(s_q + st * TILE_BYTES + at, 0), SHAPE, k > 0);
          }
          commit(q_free(st));
          commit(s_full(st));
        }
        __syncwarp();
      }
      if (ok && elected()) commit(k_free(kb));
      __syncwarp();
      ++loaded;
    }
    // nothing is in flight when the tensor memory is given back and the CTA ends
    if (elected()) commit(drained);
    for (int k = 0; k < 100000 && !bar_try(drained, 0); ++k) {}
    __syncwarp();
  } else {
    const uint32_t wg = warp >> 2;
    const int r = tid & 127;
    const float scale2 = s.scale * LOG2E;
    const uint64_t scale22 = two(scale2, scale2);
    uint32_t seen = 0, before = 0;                         // tiles, and items with any, before this one
    bool ok = true;
    for (int round = 0, item; (item = item_at(round, items)) >= 0; ++round) {
      const KeysItem w(a, item, observe);
      const int key = w.k0 + r;
      if (!w.tiles) {
        if (!wg && key < s.keys) weights[(((size_t)w.part * s.sequences + w.b) * s.n_kv_heads + w.kvh) * s.keys + key] = 0.f;
        continue;
      }
      // the positions of the queries that see this key
      const int lo = key < w.n ? max(w.first, key) : w.last;
      const int hi = min(w.last, s.window && key >= s.sinks ? (int)min((long long)w.last, key + (long long)s.window) : w.last) - 1;
      uint64_t sum[2] = {};
      // this group's tiles are every KW_GROUPS-th; their two blocks, and minus the lse (in powers of two) of column r a tile ahead
      const int own = (wg - seen) % KW_GROUPS;
      Block block[2] = {Block(w, min(2 * own, w.blocks - 1)), Block(w, min(2 * own + 1, w.blocks - 1))};
      auto minus_lse = [&](int j) {
        const Block& mine = block[r >> 6];
        const int p = mine.position(w) + (r & 63);
        return 2 * j + (r >> 6) < w.blocks && p < w.last ? -LOG2E * lse[((size_t)w.b * s.n_heads + w.kvh * G + mine.head) * s.queries + p - off] : -INFINITY;
      };
      float ahead = own < w.tiles ? minus_lse(own) : 0.f;
      for (int j = own; j < w.tiles; j += KW_GROUPS) {
        const uint32_t st = wg, use = (seen + j) / KW_BUFFERS;
        int place[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) place[e] = 2 * j + e < w.blocks ? block[e].position(w) : w.last;
        float* mine = s_lse[2 * wg + (use & 1)];
        mine[r] = ahead;
        if (j + KW_GROUPS < w.tiles) {
          block[0].step(w, 2 * KW_GROUPS);
          block[1].step(w, 2 * KW_GROUPS);
          ahead = minus_lse(j + KW_GROUPS);
        }
        asm volatile("barrier.cta.sync %0, 128;" ::"r"(2 + wg) : "memory");
        ok = ok && bar_wait_warp(s_full(st), use & 1, &s_gone, status);
        if (!ok) continue;
        fence_after();
        const uint32_t at = tmem + 128 * st + ((uint32_t)(warp & 3) << 21);
#pragma unroll
        for (int c0 = 0; c0 < 128; c0 += 32) {
          if (c0 == 64 && 2 * j + 1 == w.blocks) break;
          uint32_t x[32];
          load32(at + c0, x);
          wait_load<32>(x);
          const int p0 = place[c0 / 64] + c0 % 64;
          const bool whole = w.k0 + UM_TILE - 1 <= p0 && p0 + 32 <= w.last && (!s.window || w.k0 + UM_TILE - 1 < s.sinks || p0 + 31 - w.k0 < s.window);
          const ulonglong2* less = reinterpret_cast<const ulonglong2*>(mine + c0);
          const uint32_t vis = below32(hi + 1 - p0) & ~below32(lo - p0);
          // What is hidden is left out behind the subtraction of the lse: that of a query which does not see the key may be NaN.
          auto add = [&](auto all) {
            auto of = [&](int c, uint64_t x2, uint64_t m) {
              const float2 f = apart(fma2(x2, scale22, m));
              return decltype(all)::value ? f : make_float2(vis >> c & 1u ? f.x : -INFINITY, vis >> (c + 1) & 1u ? f.y : -INFINITY);
            };
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const ulonglong2 m = less[e / 2];
              const float2 f = of(2 * e, two(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), m.x);
              const float2 g = of(2 * e + 2, two(__uint_as_float(x[2 * e + 2]), __uint_as_float(x[2 * e + 3])), m.y);
              sum[0] = add2(sum[0], e % 8 < KW_POLY_OF_8 ? power2<true>(f) : two(ex2(f.x), ex2(f.y)));
              sum[1] = add2(sum[1], two(ex2(g.x), ex2(g.y)));
            }
          };
          if (whole) add(std::true_type());
          else add(std::false_type());
        }
        fence_before();
        bar_arrive(s_free(st));
      }
      const float2 halves = apart(add2(sum[0], sum[1]));
      // The group with the item's last tile adds the groups' sums; the others go on.  (Until it has, they come 10 items further at
      // most: its next tile, 4 on, is not taken, so that the tile 8 on is not made, and what a group goes through without one of
      // its own is fewer than 4.)
      const uint32_t slot = before % KW_SLOTS;
      s_sum[slot][wg][r] = ok ? halves.x + halves.y : NAN;
      __syncwarp();
      if (lane == 0) bar_arrive(summed(slot));
      seen += w.tiles;
      if ((seen - 1) % KW_GROUPS == wg) {
        ok = bar_wait_warp(summed(slot), before / KW_SLOTS & 1, &s_gone, status) && ok;
        float all = s_sum[slot][0][r];
        for (int g = 1; g < KW_GROUPS; ++g) all += s_sum[slot][g][r];
        if (key < s.keys) weights[(((size_t)w.part * s.sequences + w.b) * s.n_kv_heads + w.kvh) * s.keys + key] = ok ? all : NAN;
      }
      ++before;
    }
  }
  fence_before();
  __syncthreads();
  if (warp == KW_MMA) {
    fence_after();
    dealloc(tmem, 512);
  }
}

// the parts' sums, in order
__global__ void __launch_bounds__(256) prompt_join_kernel(const float* __restrict__ part, int parts, long long n, float* __restrict__ weights) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float sum = 0.f;
#pragma unroll 4
  for (int p = 0; p < parts; ++p) sum += part[p * n + i];
  weights[i] = sum;
}
// Into how many parts an item's queries are cut, by a model in tiles of 128 x 128 (about 0.7 us each): an SM's share of all of
// them, 2 for every item that it takes, more than half of the longest item where the work runs out, 2.5 for joining the parts.  On 28
// shapes its choice is 0.4 % slower than the best, 7 % at most.  (70B heads, 8192 tokens, a window of 2048 with sinks, whose tile all
// queries see: 1 part 592 us, 6 374, 16 404; 2048 tokens of 40 heads stay whole, 35 us, 39 in two.)
int parts_of(const cq_prompt* s, int observe) {
  const int tiles = (s->keys + UM_TILE - 1) / UM_TILE, G = s->n_heads / s->n_kv_heads, step = (tiles + 255) / 256;
  double sum = 0, longest = 0;
  for (int t = 0; t < tiles; t += step) {
    const long long k0 = (long long)t * UM_TILE, end = std::min<long long>(k0 + UM_TILE, s->keys);
    const long long first = std::max({(long long)s->keys - s->queries, (long long)s->keys - observe, k0});
    const long long last = s->window && k0 >= s->sinks ? std::min<long long>(s->keys, end - 1 + s->window) : s->keys;
    const double n = std::ceil(0.5 * G * ((std::max(0ll, last - first) + KW_Q - 1) / KW_Q));
    sum += n * step;
    longest = std::max(longest, n);
  }
  const double heads = (double)s->n_kv_heads * s->sequences, sms = cq_sm_count(), share = sum * heads / sms;
  int best = 1;
  double least = 0;
  for (int p = 1; p <= 16; ++p) {
    const double t = share + 2.0 * tiles * heads * p / sms + 0.6 * longest / p + (p > 1 ? 2.5 : 0.0);
    if (p == 1 || t < least) {
      least = t;
      best = p;
    }
  }
  return best;
}

// Tensor map of q, k or v (sequence, token, head strides in halves): boxes of 64 columns x `rows` tokens.  A broadcast sequence or
// head (stride 0) is one of them, addressed with the coordinate 0 (one[]).  False where the map cannot describe the tensor.
bool map_of(CUtensorMap* map, const void* at, const int64_t (&strides)[3], int sequences, int tokens, int heads, int D, int rows, int (&one)[2]) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = []() -> Encode {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      return nullptr;
    }
    return (Encode)fn;
  }();
  if (!encode) return false;
  one[0] = heads > 1 && strides[2] != 0;
  one[1] = sequences > 1 && strides[0] != 0;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)tokens, one[0] ? (cuuint64_t)heads : 1, one[1] ? (cuuint64_t)sequences : 1};
  const cuuint64_t steps[3] = {tokens > 1 ? (cuuint64_t)strides[1] * 2 : (cuuint64_t)D * 2, one[0] ? (cuuint64_t)strides[2] * 2 : (cuuint64_t)D * 2,
                               one[1] ? (cuuint64_t)strides[0] * 2 : (cuuint64_t)D * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, each[4] = {1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(at), dims, steps, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int check_shape(const cq_prompt* s) {
  if (!s) return CQ_ERR_BAD_ARG;
  if (s->sequences < 1 || s->sequences > 65535 || s->queries < 1 || s->keys < s->queries || s->keys > (1 << 24) || s->n_kv_heads < 1 ||
      s->n_heads < 1 || s->n_heads > 65535 || s->n_heads % s->n_kv_heads)
    return CQ_ERR_BAD_SHAPE;
  if (s->head_dim != 64 && s->head_dim != 128) return CQ_ERR_UNSUPPORTED;
  return s->window < 0 || s->sinks < 0 ? CQ_ERR_BAD_ARG : CQ_OK;
}
int check(const cq_prompt* s, const void* q, const void* k, const void* v) {
  if (!s || !q || !k || (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) || s->window < 0 || s->sinks < 0 || !(s->scale > 0.f)) return CQ_ERR_BAD_ARG;
  if (const int rc = check_shape(s)) return rc;
  for (int i = 0; i < 3; ++i)
    if ((s->q_strides[i] | s->k_strides[i] | (v ? s->v_strides[i] : 0)) & 7) return CQ_ERR_BAD_ARG;
  if ((s->queries > 1 && s->q_strides[1] < 8) || (s->keys > 1 && (s->k_strides[1] < 8 || (v && s->v_strides[1] < 8)))) return CQ_ERR_BAD_ARG;
  return CQ_OK;
}

}  // namespace

extern "C" size_t cq_attn_prefill_workspace_bytes(const cq_prompt* s) {
  if (check_shape(s) != CQ_OK) return 0;
  const int parts = prompt_form(s).parts;
  return parts > 1 ? (size_t)parts * s->sequences * s->queries * s->n_heads * (s->head_dim + 1) * sizeof(float) : 0;
}

extern "C" int cq_attn_prefill(const cq_prompt* shape, const void* q, const void* k, const void* v, const long long* lengths, void* out,
                               float* lse, void* workspace, uint32_t* status_word, cq_stream_t stream) {
  const int rc = check(shape, q, k, v);
  if (rc != CQ_OK) return rc;
  if (!v || !out || !lse || ((uintptr_t)out & 15)) return CQ_ERR_BAD_ARG;
  const int D = shape->head_dim, B = shape->sequences, G = shape->n_heads / shape->n_kv_heads;
  PromptArgs a = {*shape, (const __half*)q, (const __half*)k, (const __half*)v, lengths, G};
  const PromptForm form = prompt_form(shape);
  const int parts = form.parts, units = form.units(shape);
  a.rows = form.rows;
  a.pack = form.pack;
  if (parts > 1 && (!workspace || ((uintptr_t)workspace & 15))) return CQ_ERR_BAD_ARG;
  const bool few = a.rows < 256 || parts > 1;
  while (1 << a.shift > a.rows) --a.shift;
  a.by_group = Divisor(units);
  a.by_heads = Divisor((uint32_t)shape->n_kv_heads * units);
  a.by_row = Divisor((uint32_t)shape->n_kv_heads * units * B);
  a.by_parts = Divisor(parts);
  PromptMaps maps;
  if (!map_of(&maps.q, q, shape->q_strides, B, shape->queries, shape->n_heads, D, std::min(a.rows, UM_TILE), maps.one[0]) ||
      !map_of(&maps.k, k, shape->k_strides, B, shape->keys, shape->n_kv_heads, D, UM_TILE, maps.one[1]) ||
      !map_of(&maps.v, v, shape->v_strides, B, shape->keys, shape->n_kv_heads, D, UM_TILE, maps.one[2]))
    return CQ_ERR_UNSUPPORTED;
  auto fn = D == 128 ? (few ? prompt_kernel<128, true> : prompt_kernel<128, false>) : (few ? prompt_kernel<64, true> : prompt_kernel<64, false>);
  const int smem = (2 + UM_STAGES) * (D / 64) * UM_CHUNK + 1024;
  CQ_CUDA_TRY(cq_grant_smem((const void*)fn, smem));
  const long long items = form.items(shape);
  const size_t rows = (size_t)B * shape->queries * shape->n_heads;
  if (items > INT32_MAX / 2 || (rows + 7) / 8 > INT32_MAX) return CQ_ERR_BAD_SHAPE;
  CQ_CUDA_TRY(kv4_launch(fn, dim3((unsigned)std::min<long long>(items, cq_sm_count())), dim3(UM_THREADS), smem, (cudaStream_t)stream, a, maps,
                         (__half*)out, lse, (float*)workspace, (int)items, status_word));
  if (parts > 1)
    CQ_CUDA_TRY(kv4_launch(D == 128 ? prompt_sum_kernel<128> : prompt_sum_kernel<64>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0,
                           (cudaStream_t)stream, a, (const float*)workspace, (__half*)out, lse));
  return CQ_OK;
}

extern "C" size_t cq_attn_prefill_weights_workspace_bytes(const cq_prompt* s, int observe) {
  if (!s || s->sequences < 1 || s->queries < 1 || s->keys < s->queries || s->n_kv_heads < 1 || s->n_heads < s->n_kv_heads || observe < 1) return 0;
  const int parts = parts_of(s, observe);
  return parts > 1 ? (size_t)parts * s->sequences * s->n_kv_heads * s->keys * sizeof(float) : 16;
}

extern "C" int cq_attn_prefill_weights(const cq_prompt* shape, const void* q, const void* k, const float* lse, const long long* lengths,
                                       int observe, float* weights, void* workspace, uint32_t* status_word, cq_stream_t stream) {
  const int rc = check(shape, q, k, nullptr);
  if (rc != CQ_OK) return rc;
  if (!lse || !weights || !workspace || observe < 1) return CQ_ERR_BAD_ARG;
  PromptArgs a = {*shape, (const __half*)q, (const __half*)k, nullptr, lengths, shape->n_heads / shape->n_kv_heads};
  const int D = shape->head_dim, B = shape->sequences;
  PromptMaps maps;
  if (!map_of(&maps.q, q, shape->q_strides, B, shape->queries, shape->n_heads, D, KW_Q, maps.one[0]) ||
      !map_of(&maps.k, k, shape->k_strides, B, shape->keys, shape->n_kv_heads, D, UM_TILE, maps.one[1]))
    return CQ_ERR_UNSUPPORTED;
  maps.v = maps.k;
  auto fn = D == 128 ? prompt_keys_kernel<128> : prompt_keys_kernel<64>;
  const int smem = (2 + KW_BUFFERS) * (D / 64) * UM_CHUNK + 1024;
  CQ_CUDA_TRY(cq_grant_smem((const void*)fn, smem));
  const int parts = parts_of(shape, observe);
  const long long n = (long long)B * shape->n_kv_heads * shape->keys, items = (long long)((shape->keys + UM_TILE - 1) / UM_TILE) * shape->n_kv_heads * B * parts;
  if (items > INT32_MAX / 2) return CQ_ERR_BAD_SHAPE;
  a.by_heads = Divisor(shape->n_kv_heads);
  a.by_row = Divisor((uint32_t)shape->n_kv_heads * B * parts);
  a.by_parts = Divisor(parts);
  CQ_CUDA_TRY(kv4_launch(fn, dim3((unsigned)std::min<long long>(items, cq_sm_count())), dim3(KW_THREADS), smem, (cudaStream_t)stream, a, maps, lse,
                         observe, parts > 1 ? (float*)workspace : weights, (int)items, status_word));
  if (parts > 1)
    CQ_CUDA_TRY(kv4_launch(prompt_join_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (cudaStream_t)stream, (const float*)workspace, parts, n,
                           weights));
  return CQ_OK;
}
