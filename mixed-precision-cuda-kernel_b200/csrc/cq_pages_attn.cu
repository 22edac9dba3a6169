// Attention of single tokens over the paged KV cache (layout: cq_pages.cuh); in the reference a part of its vendored LLaMA
// (llama/modeling_llama_quant.py:371-419 of the reference project).
//
// The bound is the cache, read once.  As in cq_attn.cu all query heads of a KV head share one tile of mma.sync m16n8k16, rows 0-7
// of A: scores S = Q . K^T with keys straight from the pages (the order of the columns inside a step is free as long as both
// operands agree), then the weights as the A operand of P . V.  A weight is two numbers of the cache's type, its upper bits in rows
// 0-7 and what is left in rows 8-15, which the heads leave empty.  An MMA cuts its sums off instead of rounding them: each one
// sums its 16 products alone, fp32 additions do the rest.  A warp takes 16 slots a turn (they lie in one page) and keeps its own
// running maximum, a whole number of powers of two, sum and weighted values; warps meet in shared memory, CTAs that share a head
// in a cluster, or, where a head's slots are cut wherever the equal shares of all CTAs end, in a second kernel.
//
// Tried and not taken: rings of tiles copied asynchronously, each warp its own (three tiles of 8 KB a warp, eight warps an SM; 70B heads, 16
// sequences up to 4001 slots 42 us against 41, 13B heads with a window 38 against 33, four of 65531 slots 172 against 172), the next
// tile's loads between the sums (registers spill: 53 against 41), two tiles a warp in rings on three CTAs an SM (249 against 172).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cq_pages.cuh"

namespace {

using namespace cq_paged;

constexpr int AT_HEADS = 8;                  // query heads of a CTA
constexpr int AT_SLOTS = 16;                 // slots of a turn
constexpr int AT_WARPS = 4;
constexpr int MAX_CLUSTER = 8;
constexpr int per_sm(int head_dim) { return head_dim == 64 ? 4 : 3; }      // CTAs that an SM holds

// sums of 16 products without an addend, rows 0-7 and rows 8-15 in pairs
template <typename T> __device__ __forceinline__ void mma(uint64_t (&d)[2], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  float x[4];
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  d[0] = two(x[0], x[1]), d[1] = two(x[2], x[3]);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^d of a whole number d <= 0; 0 below the normal numbers (and 1 for NaN, whose sums are NaN)
__device__ __forceinline__ float whole_pow2(float d) { return __int_as_float(max(0, 127 + __float2int_rn(d)) << 23); }
// The maximum of scores of which none is above -infinity (NaN does not count): below all others, above that of no slot, which is -infinity
constexpr float LOWEST = -3.402823466e38f;
// The share of sums with maximum m in those that reach up to `top`: 0 where they have no slot.  Otherwise it is not 0, so that infinite sums
// stay infinite (2^-126 of other sums is nothing beside `top`'s own weight, which is 1/2 at least).
__device__ __forceinline__ float share_of(float m, float top) {
  return m == -INFINITY ? 0.f : __int_as_float(max(1, 127 + __float2int_rn(m - top)) << 23);
}
// two weights: their upper bits, and what is left of them
template <typename T> __device__ __forceinline__ uint2 split_weights(float a, float b) {
  const uint32_t hi = Type<T>::pair(a, b);
  const float2 f = Type<T>::apart(hi);
  return make_uint2(hi, Type<T>::pair(a - f.x, b - f.y));
}
// not as read-only data: the launch itself may write a row
__device__ __forceinline__ uint4 ld16(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void ld32(uint4& a, uint4& b, const void* p) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p) : "memory");
}

// What a query sees of n slots: j < first or from <= j < n, in tiles of TILE slots
template <int TILE> struct Visible {
  int n, first, from, low, second, tiles;    // tiles 0 .. low - 1 and second .. ; their number
  __device__ __forceinline__ Visible(int n, int window, int sinks) : n(n) {
    first = window > 0 ? min(sinks, n) : n;
    from = window > 0 ? max(first, n > window ? n - window : 0) : n;
    low = (first + TILE - 1) / TILE;
    second = max(low, from / TILE);
    tiles = low + (from < n ? max(0, (n + TILE - 1) / TILE - second) : 0);
  }
  __device__ __forceinline__ int tile(int i) const { return i < low ? i : second + i - low; }
  __device__ __forceinline__ bool sees(int j) const { return j < first || (j >= from && j < n); }
};

// slots that hold a row, a step's new one among them (more 1)
__device__ __forceinline__ int held(long long n, int more, int slots) {
  return n < 0 ? 0 : (n >= slots ? slots : (int)n + more);
}

// The step's new token: k, v (sequences, KV, D), not rotated
template <typename T> struct NewRow {
  Rows<T> k, v;
  const float *cos_t, *sin_t;
  const long long* positions;
  int table_rows;
};

// What the kernels get besides their tensors
struct Shape {
  int sequences, H, chunks, window, sinks;
  float scale;
};
constexpr int PART = 4;                      // in front of a head's D partial sums: maximum, sum of weights
// The partial results of a CTA: 0 of a head whose slots begin with an earlier CTA, 1 of a head that a later CTA goes on with
template <int D> __device__ __forceinline__ float* part_of(void* ws, int cta, int which) {
  return reinterpret_cast<float*>(ws) + (size_t)(2 * cta + which) * AT_HEADS * (D + PART);
}

// (most quotients fit 32 bits, whose division takes a quarter of the time)
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return (unsigned long long)(a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}
// All tiles of all sequences and tasks in a row, cut into equal ranges for `ctas` CTAs.  (By whole warps, 32 sequences at a time.)
// FAR: lengths past the first-level cache.
template <bool FAR> struct Tiles {
  const long long* length;
  const Shape& shape;
  const int slots, more, heads_each, lane;
  long long total, each;
  int n;                                     // slots of the lane's sequence in the last 32
  uint32_t mine, upto;                       // its tiles, and those of the ones in front of it too (2^26 each at most)
  __device__ __forceinline__ Tiles(const long long* length, const Shape& shape, int slots, int more, int heads_each, int ctas)
      : length(length), shape(shape), slots(slots), more(more), heads_each(heads_each), lane(threadIdx.x & 31), total(0) {
    for (int s = 0; s < shape.sequences; s += 32) total += scan(s);
    total *= heads_each;
    each = max((long long)AT_WARPS, quotient(total + ctas - 1, ctas));       // for each warp one at least
  }
  __device__ __forceinline__ Visible<AT_SLOTS> sees(int n) const { return Visible<AT_SLOTS>(n, shape.window, shape.sinks); }
  __device__ __forceinline__ int slots_of(int s) const { return held(FAR ? __ldcg(length + s) : length[s], more, slots); }
  __device__ __forceinline__ Visible<AT_SLOTS> visible(int s) const { return sees(slots_of(s)); }
  __device__ __forceinline__ long long scan(int s) {
    n = s + lane < shape.sequences ? slots_of(s + lane) : 0;
    mine = upto = s + lane < shape.sequences ? sees(n).tiles : 0;
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += y;
    }
    return (long long)__shfl_sync(0xffffffffu, upto, 31);
  }
  // the sequence with tile x < total; from: its first one; all: how many slots it has
  __device__ __forceinline__ int find(long long x, long long& from, int& all) {
    long long before = 0;
    for (int s = 0;; s += 32) {
      if (shape.sequences > 32) scan(s);
      const uint32_t found = __ballot_sync(0xffffffffu, x < (before + upto) * heads_each);
      if (found) {
        const int k = __ffs(found) - 1;
        from = (before + __shfl_sync(0xffffffffu, upto - mine, k)) * heads_each;
        all = __shfl_sync(0xffffffffu, n, k);
        return s + k;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  // a sequence's first tile; all: as above
  __device__ __forceinline__ long long front(int seq, int& all) {
    long long before = 0;
    for (int s = 0; s < seq - seq % 32; s += 32) before += scan(s);
    if (shape.sequences > 32) scan(seq - seq % 32);
    all = __shfl_sync(0xffffffffu, n, seq % 32);
    return (before + __shfl_sync(0xffffffffu, upto - mine, seq % 32)) * heads_each;
  }
};
// The infinite and NaN values of columns d .. d + 3 that a query sees in some tiles, summed without their weights, which are not 0; NaN where
// the score is -infinity, and 0 where there are none.  A thread's four columns wait for sixteen slots at a time (one infinite value in four sequences
// of 65531 slots: 1.05 ms in place of 0.17; with the weights summed again 26).  Out of line: its registers are none of the kernel's (inlined
// four sequences of 30000 slots 69.6 us, so 68.1; 64 of 16 / 4 heads 51.4, so 51.6, without either 50.6).
template <typename T, int D>
__device__ __noinline__ float4 infinities(const Pool<T> pool, const Table table, const Visible<AT_SLOTS> vis, int tile0, int tile1, int seq, int kvh,
                                          const T* query, int d, float scale2) {
  float odd[4] = {};
  for (int t = tile0; t < tile1; ++t) {
    const int base = vis.tile(t) * AT_SLOTS, page = table.page_of(pool, seq, base);
    if (page < 0) continue;
    const size_t row0 = pool.rows(page, kvh) + (base & ((1 << pool.log_page) - 1));
    uint2 raw[AT_SLOTS];
#pragma unroll
    for (int j = 0; j < AT_SLOTS; ++j) raw[j] = vis.sees(base + j) ? *reinterpret_cast<const uint2*>(pool.v + (row0 + j) * D + d) : make_uint2(0u, 0u);
#pragma unroll
    for (int j = 0; j < AT_SLOTS; ++j) {
      const float2 lo = Type<T>::apart(raw[j].x), hi = Type<T>::apart(raw[j].y);
      const float v[4] = {lo.x, lo.y, hi.x, hi.y};
      if (isfinite(v[0]) && isfinite(v[1]) && isfinite(v[2]) && isfinite(v[3])) continue;
      float dot = 0.f;
#pragma unroll 1
      for (int c = 0; c < D; ++c) dot += Type<T>::one(query[c]) * Type<T>::one(pool.k[(row0 + j) * D + c]);
      const bool none = dot * scale2 == -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (!isfinite(v[c])) odd[c] += none ? NAN : v[c];
    }
  }
  return make_float4(odd[0], odd[1], odd[2], odd[3]);
}

// Where the four columns 4 f .. of a head's sums are in shared memory: eight lanes with what one MMA gave them, and eight lanes
// with consecutive columns, meet different banks (one sequence of 32 heads, 256 slots: 5.4 us; in order 5.8).
__device__ __forceinline__ int place_of(int f) { return 4 * (f ^ (f >> 3 & 3)); }
// CLUSTER: a cluster of CTAs for the heads of a KV head and sequence, each with the same share of its tiles.  Otherwise all tiles of all
// sequences and KV heads in a row, cut into equal ranges for the CTAs that the device holds at once.  (168 registers a thread for 128 columns,
// 122 to 128 for 64; with equal ranges 48 to 64 bytes are spilled, 12 without a step for 64 columns.)
template <typename T, int D, bool STEP, bool CLUSTER>
__global__ void __launch_bounds__(AT_WARPS * 32, per_sm(D)) pages_attend_kernel(const Rows<T> q, const Pool<T> pool, const Table table, const NewRow<T> fresh,
                                                                        const long long* __restrict__ length, T* __restrict__ out, void* ws, const Shape shape) {
  constexpr int THREADS = AT_WARPS * 32;
  constexpr int KP = D / 32;                 // 16-byte pieces of a key per lane (four lanes a slot)
  // Narrow heads' keys come two pieces at a time, whole lines for four lanes (64 sequences of 16 / 4 heads up to 5000 slots 54.3 us, so 55.8;
  // wide ones 42.6 that way, also values 43.1, against 40.9).
  constexpr bool PAIRS = D == 64;
  auto piece = [](int i) { return PAIRS ? 64 * (i >> 1) + 8 * (i & 1) : 32 * i; };          // its columns, behind the lane's first
  constexpr int VS = D / 64;                 // of a value (eight lanes a slot)
  // Weights times a power of two: fp16's halves of their split then reach down to 2^-38 of the largest; in bf16, whose halves reach anywhere,
  // sums of 2^24 of the largest values stay finite.
  constexpr float LIFT = std::is_same<T, __half>::value ? 32768.f : 5.9604644775390625e-8f;
  if (CLUSTER) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ __align__(16) float s_sum[AT_WARPS][AT_HEADS][D + 8];
  __shared__ __align__(16) float s_part[CLUSTER ? AT_HEADS : 1][D + PART];
  __shared__ __align__(16) T s_q[AT_HEADS][D + (PAIRS ? 8 : 32)];
  __shared__ float s_m[AT_WARPS][AT_HEADS], s_l[AT_WARPS][AT_HEADS];
  const int KV = pool.heads, H = shape.H, G = H / KV, chunks = shape.chunks, heads_each = KV * chunks, slots = table.width << pool.log_page;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g8 = lane >> 2, t4 = lane & 3;
  const float scale2 = shape.scale * 1.4426950408889634f;  // scores in powers of two
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!CLUSTER) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");          // (the second kernel reads lengths before it waits)

  // Tiles tile0 .. tile1 - 1 of one sequence and task (a KV head and eight of its query heads at most): to `out`, or partial results to `part`.
  auto segment = [&](int seq, int task, const Visible<AT_SLOTS>& vis, int tile0, int tile1, float* part) {
    const int kvh = task / chunks, h0 = (task - kvh * chunks) * AT_HEADS, heads = min(AT_HEADS, G - h0), head0 = kvh * G + h0;
    long long at = -1;                       // the new row's slot, where it is written
    bool turn = false;
    long long pos = 0;
    if (STEP) {
      pos = fresh.cos_t ? fresh.positions[seq] : 0;
      turn = fresh.cos_t && pos >= 0 && pos < fresh.table_rows;
      at = !fresh.cos_t || turn ? length[seq] : -1;
      if (at < 0 || at >= slots) at = -1;
    }
    // queries in shared memory, rotated
    constexpr int PIECES = D / 16;
    for (int i = tid; i < AT_HEADS * PIECES; i += THREADS) {
      const int g = i / PIECES, c = 8 * (i - g * PIECES);
      uint4 x1 = make_uint4(0, 0, 0, 0), x2 = x1;
      if (g < heads) {
        const T* src = q.row(seq, head0 + g) + c;
        x1 = *reinterpret_cast<const uint4*>(src);
        x2 = *reinterpret_cast<const uint4*>(src + D / 2);
        if (turn) rotate8<T>(x1, x2, fresh.cos_t + pos * (D / 2) + c, fresh.sin_t + pos * (D / 2) + c);
      }
      *reinterpret_cast<uint4*>(&s_q[g][c]) = x1;
      *reinterpret_cast<uint4*>(&s_q[g][c + D / 2]) = x2;
    }
    // The new row, by the CTA that will read it (those of other query heads write the same).
    if (STEP && at >= 0 && tile0 < tile1 && tile1 == vis.tiles && tid < 2 * PIECES) {
      const int page = table.page_of(pool, seq, at), c = 8 * (tid % PIECES);
      if (page >= 0) {
        const bool value = tid >= PIECES;
        const T* src = (value ? fresh.v : fresh.k).row(seq, kvh) + c;
        T* dst = (value ? pool.v : pool.k) + (pool.rows(page, kvh) + (at & ((1 << pool.log_page) - 1))) * D + c;
        uint4 x1 = *reinterpret_cast<const uint4*>(src), x2 = *reinterpret_cast<const uint4*>(src + D / 2);
        if (turn && !value) rotate8<T>(x1, x2, fresh.cos_t + pos * (D / 2) + c, fresh.sin_t + pos * (D / 2) + c);
        *reinterpret_cast<uint4*>(dst) = x1;
        *reinterpret_cast<uint4*>(dst + D / 2) = x2;
      }
    }
    __syncthreads();
    const int first = (PAIRS ? 16 : 8) * t4; // of the lane's columns in queries and keys
    const T* mine_q = &s_q[g8][first];

    float m = -INFINITY, l = 0.f;
    uint64_t o2[8 * VS];                     // MMA j + 8 s: its column n is column 64 s + 8 n + j of the head; n = 2 t4 and 2 t4 + 1
#pragma unroll
    for (int i = 0; i < 8 * VS; ++i) o2[i] = 0;

#pragma unroll 1
    for (int i = tile0 + warp; i < tile1; i += AT_WARPS) {
      const int base = vis.tile(i) * AT_SLOTS, page = table.page_of(pool, seq, base);
      if (page < 0) continue;
      const size_t row0 = pool.rows(page, kvh) + (base & ((1 << pool.log_page) - 1));
      uint4 kk[2][KP], vv[4][VS];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < KP; e += PAIRS ? 2 : 1) {
          const T* from = pool.k + (row0 + 8 * h + g8) * D + first + piece(e);
          if constexpr (PAIRS) ld32(kk[h][e], kk[h][e + 1], from);
          else kk[h][e] = ld16(from);
        }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int p = 8 * (u >> 1) + 2 * t4 + (u & 1);
#pragma unroll
        for (int e = 0; e < VS; ++e) vv[u][e] = vis.sees(base + p) ? ld16(pool.v + (row0 + p) * D + 8 * g8 + 64 * e) : make_uint4(0, 0, 0, 0);
      }
      uint64_t pairs[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < KP; ++e) {
        const uint4 qa = *reinterpret_cast<const uint4*>(mine_q + piece(e));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint64_t d0[2], d1[2];
          mma<T>(d0, qa.x, 0u, qa.y, 0u, kk[h][e].x, kk[h][e].y);
          mma<T>(d1, qa.z, 0u, qa.w, 0u, kk[h][e].z, kk[h][e].w);
          pairs[h] = add2(pairs[h], add2(d0[0], d1[0]));
        }
      }
      float s[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 f = apart(pairs[h]);
        s[h][0] = f.x, s[h][1] = f.y;
      }
      // this lane: head g8, slots base + 8 h + 2 t4 + e
      bool sees[2][2];
      float top = m;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sees[h][e] = vis.sees(base + 8 * h + 2 * t4 + e);
          top = fmaxf(top, sees[h][e] ? __fmul_rn(s[h][e], scale2) : -INFINITY);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // A whole number at or above the maximum, so that rescaling sums is exact.  (A tile has a slot that all heads see.  No finite
      // score so far: weights 0, or NaN where a score is NaN, which no maximum shows.)
      const float ref = fmaxf(ceilf(top), LOWEST), keep = whole_pow2(m - ref);
      const uint64_t keep2 = two(keep, keep);
      m = ref;
      // From 2^23 on the maximum is a rounded product itself: the products that it is compared with are then rounded alike.  (Unrounded ones may
      // lie a power of two and more above it, whose weights fp16 does not hold, or all of them far below.)
      const bool coarse = fabsf(ref) >= 8388608.f;
      float w[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = coarse ? __fsub_rn(__fmul_rn(s[h][e], scale2), ref) : __fmaf_rn(s[h][e], scale2, -ref);
          w[h][e] = sees[h][e] ? LIFT * ex2(x) : 0.f;
        }
      l = l * keep + ((w[0][0] + w[0][1]) + (w[1][0] + w[1][1]));
      const uint2 w0 = split_weights<T>(w[0][0], w[0][1]), w1 = split_weights<T>(w[1][0], w[1][1]);
#pragma unroll
      for (int e = 0; e < VS; ++e) {
        const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vv[0][e]);
        const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vv[1][e]);
        const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vv[2][e]);
        const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vv[3][e]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
          uint64_t d[2];
          mma<T>(d, w0.x, w0.y, w1.x, w1.y, __byte_perm(v0[j >> 1], v1[j >> 1], sel), __byte_perm(v2[j >> 1], v3[j >> 1], sel));
          o2[8 * e + j] = fma2(o2[8 * e + j], keep2, add2(d[0], d[1]));
        }
      }
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t4 == 0) {
      s_m[warp][g8] = m;
      s_l[warp][g8] = l;
    }
#pragma unroll
    for (int e = 0; e < VS; ++e)
#pragma unroll
      for (int j = 0; j < 8; j += 4) {       // columns n = 2 t4 and 2 t4 + 1
        const float2 x0 = apart(o2[8 * e + j]), x1 = apart(o2[8 * e + j + 1]), x2 = apart(o2[8 * e + j + 2]), x3 = apart(o2[8 * e + j + 3]);
        *reinterpret_cast<float4*>(&s_sum[warp][g8][place_of(16 * e + 4 * t4 + j / 4)]) = make_float4(x0.x, x1.x, x2.x, x3.x);
        *reinterpret_cast<float4*>(&s_sum[warp][g8][place_of(16 * e + 4 * t4 + 2 + j / 4)]) = make_float4(x0.y, x1.y, x2.y, x3.y);
      }
    __syncthreads();
    for (int i = tid; i < heads * D / 4; i += THREADS) {
      const int g = i / (D / 4), d = 4 * (i - g * (D / 4));
      float top = s_m[0][g];
#pragma unroll
      for (int w = 1; w < AT_WARPS; ++w) top = fmaxf(top, s_m[w][g]);
      float tot = 0.f, sum[4] = {};
#pragma unroll
      for (int w = 0; w < AT_WARPS; ++w) {
        const float f = share_of(s_m[w][g], top);
        const float4 x = *reinterpret_cast<const float4*>(&s_sum[w][g][place_of(d / 4)]);
        tot += f * s_l[w][g];
        sum[0] += f * x.x, sum[1] += f * x.y, sum[2] += f * x.z, sum[3] += f * x.w;
      }
      if (!(fabsf(sum[0]) + fabsf(sum[1]) + fabsf(sum[2]) + fabsf(sum[3]) <= 3.0e38f) && tot == tot) {
        // An infinite or NaN value takes part.  What the halves of its weight and rescaled sums make of it may be NaN where the product
        // is infinite; no weight is 0, however small, but that of a score of -infinity: such values are added again without their weights.
        // (Columns without one are right as they are.)
        const float4 odd = infinities<T, D>(pool, table, vis, tile0, tile1, seq, kvh, s_q[g], d, scale2);
        sum[0] = odd.x != 0.f ? odd.x : sum[0], sum[1] = odd.y != 0.f ? odd.y : sum[1];
        sum[2] = odd.z != 0.f ? odd.z : sum[2], sum[3] = odd.w != 0.f ? odd.w : sum[3];
      }
      if (part) {
        float* mine = part + g * (D + PART);
        *reinterpret_cast<float4*>(mine + PART + d) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        if (d == 0) *reinterpret_cast<float2*>(mine) = make_float2(top, tot);
      } else {
        const bool none = top == -INFINITY;  // no slot is visible (where all scores are -infinity 0 / 0, as in the formula)
        *reinterpret_cast<uint2*>(out + ((size_t)seq * H + head0 + g) * D + d) =
            none ? make_uint2(0u, 0u) : make_uint2(Type<T>::pair(sum[0] / tot, sum[1] / tot), Type<T>::pair(sum[2] / tot, sum[3] / tot));
      }
    }
  };

  if constexpr (CLUSTER) {
    const int rank = blockIdx.x, n = gridDim.x, task = blockIdx.y, seq = blockIdx.z;
    const Visible<AT_SLOTS> vis(held(length[seq], STEP, slots), shape.window, shape.sinks);
    const int each = (vis.tiles + n - 1) / n, tile0 = min(vis.tiles, rank * each), tile1 = min(vis.tiles, tile0 + each);
    segment(seq, task, vis, tile0, tile1, n > 1 ? &s_part[0][0] : nullptr);
    if (n == 1) return;
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int kvh = task / chunks, h0 = (task - kvh * chunks) * AT_HEADS, heads = min(AT_HEADS, G - h0), head0 = kvh * G + h0;
    // an equal share of the columns for every CTA
    for (int i = rank * THREADS + tid; i < heads * D / 4; i += n * THREADS) {
      const int g = i / (D / 4), d = 4 * (i - g * (D / 4));
      auto from = [&](int r, int c) {
        uint32_t to;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(&s_part[g][c])), "r"(r));
        return to;
      };
      float m[MAX_CLUSTER], l[MAX_CLUSTER], top = -INFINITY, tot = 0.f, sum[4] = {};
      float4 x[MAX_CLUSTER];
#pragma unroll
      for (int r = 0; r < MAX_CLUSTER; ++r) {
        m[r] = -INFINITY, l[r] = 0.f, x[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n) {
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(m[r]), "=f"(l[r]) : "r"(from(r, 0)) : "memory");
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[r].x), "=f"(x[r].y), "=f"(x[r].z), "=f"(x[r].w) : "r"(from(r, PART + d)) : "memory");
        }
        top = fmaxf(top, m[r]);
      }
#pragma unroll
      for (int r = 0; r < MAX_CLUSTER; ++r)
        if (r < n) {
          const float f = share_of(m[r], top);
          tot += f * l[r];
          sum[0] += f * x[r].x, sum[1] += f * x[r].y, sum[2] += f * x[r].z, sum[3] += f * x[r].w;
        }
      const bool none = top == -INFINITY;
      *reinterpret_cast<uint2*>(out + ((size_t)seq * H + head0 + g) * D + d) =
          none ? make_uint2(0u, 0u) : make_uint2(Type<T>::pair(sum[0] / tot, sum[1] / tot), Type<T>::pair(sum[2] / tot, sum[3] / tot));
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    const int cta = blockIdx.x, ctas = gridDim.x, B = shape.sequences;
    Tiles<false> all(length, shape, slots, STEP, heads_each, ctas);
    const long long begin = min(all.total, all.each * cta), end = min(all.total, begin + all.each);
    if (begin < end) {
      long long x = begin, from;
      int held_by, seq = all.find(x, from, held_by);
      Visible<AT_SLOTS> vis = all.sees(held_by);
#pragma unroll 1
      while (true) {
        const int task = (int)quotient(x - from, vis.tiles);
        const long long begins = from + (long long)task * vis.tiles, ends = begins + vis.tiles;
        const int tile0 = (int)(x - begins), tile1 = (int)(min(end, ends) - begins);
        segment(seq, task, vis, tile0, tile1, tile0 > 0 ? part_of<D>(ws, cta, 0) : (tile1 < vis.tiles ? part_of<D>(ws, cta, 1) : nullptr));
        x = begins + tile1;
        if (x >= end) break;
        if (x == from + (long long)vis.tiles * heads_each) {
          from = x;
          do vis = all.visible(++seq);
          while (vis.tiles == 0);
        }
        __syncthreads();
      }
    }
    // (sequences that see nothing)
    for (int s = cta; s < B; s += ctas)
      if (all.visible(s).tiles == 0)
        for (int i = tid; i < H * D / 8; i += THREADS) reinterpret_cast<uint4*>(out + (size_t)s * H * D)[i] = make_uint4(0, 0, 0, 0);
  }
}

// Joins the partial results of heads that several CTAs share: a row of blocks for each task where there are few of them, otherwise for the one
// that begins in a CTA and goes on behind it; `heads` of the task's heads for a block, the more warps a head the fewer tasks there are.
// Which parts they are follows from the lengths alone, and is known before the first kernel ends: that one lets this one begin when its own
// wait is over, so that lengths may be read (past the first-level cache).  A warp has the shares of 32 parts in its
// lanes, and the first four parts' sums on their way, before it adds.  (One sequence of 64 / 8 heads, 32000 slots: 34.6 us with
// the attention, 29.2 without this kernel; as one block for a task's heads, which looked up the parts in memory, 42.3.)
constexpr int JOIN_WARPS = AT_HEADS;
template <typename T, int D>
__global__ void __launch_bounds__(32 * JOIN_WARPS) pages_join_kernel(const void* ws, const long long* __restrict__ length, const Shape shape, int slots, int more,
                                                                     int KV, int ctas, int heads, T* __restrict__ out) {
  constexpr int CPL = D / 32, EARLY = 4;
  using Columns = typename std::conditional<CPL == 4, float4, float2>::type;
  __shared__ __align__(16) float s_sum[JOIN_WARPS][D];
  __shared__ float s_top[JOIN_WARPS], s_tot[JOIN_WARPS];
  __shared__ int4 s_job;                     // sequence, task, first CTA, parts
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, H = shape.H, G = H / KV, heads_each = KV * shape.chunks;
  if (warp == 0) {
    const bool few = gridDim.x == (long long)shape.sequences * heads_each;        // a row of blocks for each task
    Tiles<true> all(length, shape, slots, more, heads_each, ctas);
    int seq = -1, task = 0, n = 0, parts = 0, cta = 0;
    long long from = 0;
    if (few) {
      seq = blockIdx.x / heads_each;
      task = blockIdx.x - seq * heads_each;
      from = all.front(seq, n);
    } else if (all.each * (blockIdx.x + 1ll) < all.total) {
      const long long x = all.each * (blockIdx.x + 1ll) - 1;
      seq = all.find(x, from, n);
      task = (int)quotient(x - from, all.sees(n).tiles);
    }
    if (const int tiles = seq < 0 ? 0 : all.sees(n).tiles) {
      const long long begins = from + (long long)task * tiles;
      cta = (int)quotient(begins, all.each);
      if (few || cta == blockIdx.x) parts = (int)quotient(begins + tiles - 1, all.each) - cta + 1;
    }
    if (lane == 0) s_job = make_int4(seq, task, cta, parts);
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int seq = s_job.x, task = s_job.y, cta = s_job.z, parts = s_job.w;
  const int kvh = task / shape.chunks, h0 = (task - kvh * shape.chunks) * AT_HEADS, first = blockIdx.y * heads;
  heads = min(heads, min(AT_HEADS, G - h0) - first);
  if (parts < 2 || heads <= 0) return;
  const int groups = JOIN_WARPS / heads, g = warp / groups, group = warp - g * groups;
  auto part = [&](int r) { return part_of<D>(const_cast<void*>(ws), cta + r, r == 0) + (first + g) * (D + PART); };
  auto columns = [&](int r) { return *reinterpret_cast<const Columns*>(part(r) + PART + CPL * lane); };
  float top = -INFINITY, tot = 0.f, sum[CPL] = {};
  if (g < heads)
    for (int r0 = group; r0 < parts; r0 += 32 * groups) {
      const int r = r0 + lane * groups, n = min(32, (parts - r0 + groups - 1) / groups);
      const float2 ml = r < parts ? *reinterpret_cast<const float2*>(part(r)) : make_float2(-INFINITY, 0.f);
      Columns x[EARLY];
#pragma unroll
      for (int k = 0; k < EARLY; ++k)
        if (k < n) x[k] = columns(r0 + k * groups);
      float next = fmaxf(top, ml.x);
      for (int d = 16; d; d /= 2) next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, d));
      const float keep = share_of(top, next), f = share_of(ml.x, next);
      top = next;
      float add = f * ml.y;
      for (int d = 16; d; d /= 2) add += __shfl_xor_sync(0xffffffffu, add, d);
      tot = tot * keep + add;
#pragma unroll
      for (int i = 0; i < CPL; ++i) sum[i] *= keep;
      auto more_of = [&](const Columns& c, int k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
        for (int i = 0; i < CPL; ++i) sum[i] = __fmaf_rn(fk, reinterpret_cast<const float*>(&c)[i], sum[i]);
      };
#pragma unroll
      for (int k = 0; k < EARLY; ++k)
        if (k < n) more_of(x[k], k);
#pragma unroll 8
      for (int k = EARLY; k < n; ++k) more_of(columns(r0 + k * groups), k);
    }
#pragma unroll
  for (int i = 0; i < CPL; ++i) s_sum[warp][CPL * lane + i] = sum[i];
  if (lane == 0) s_top[warp] = top, s_tot[warp] = tot;
  __syncthreads();
  if (g >= heads || group) return;
  float best = -INFINITY;
  for (int k = 0; k < groups; ++k) best = fmaxf(best, s_top[warp + k]);
  tot = 0.f;
#pragma unroll
  for (int i = 0; i < CPL; ++i) sum[i] = 0.f;
  for (int k = 0; k < groups; ++k) {
    if (s_top[warp + k] == -INFINITY) continue;
    const float f = share_of(s_top[warp + k], best);
    tot += f * s_tot[warp + k];
#pragma unroll
    for (int i = 0; i < CPL; ++i) sum[i] = __fmaf_rn(f, s_sum[warp + k][CPL * lane + i], sum[i]);
  }
  const bool none = best == -INFINITY;
  T* to = out + ((size_t)seq * H + kvh * G + h0 + first + g) * D + CPL * lane;
#pragma unroll
  for (int i = 0; i < CPL; i += 2) *reinterpret_cast<uint32_t*>(to + i) = none ? 0u : Type<T>::pair(sum[i] / tot, sum[i + 1] / tot);
}

// Clusters of 1 .. MAX_CLUSTER CTAs that the device holds at once (fewer than its CTAs / n: a cluster lies in one part of the device)
struct Held {
  int clusters[MAX_CLUSTER + 1];
  explicit Held(int head_dim) {
    for (int n = 1; n <= MAX_CLUSTER; ++n) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(n);
      cfg.blockDim = dim3(AT_WARPS * 32);
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = n;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      auto fn = head_dim == 64 ? pages_attend_kernel<__half, 64, false, true> : pages_attend_kernel<__half, 128, false, true>;
      if (cudaOccupancyMaxActiveClusters(&clusters[n], fn, &cfg) == cudaSuccess && clusters[n] > 0) continue;
      (void)cudaGetLastError();
      clusters[n] = per_sm(head_dim) * cq_sm_count() / n;
    }
  }
};
// (of the first device: those of one machine are alike)
const Held& held_by_device(int head_dim) {
  if (head_dim == 64) {
    static const Held held(64);
    return held;
  }
  static const Held held(128);
  return held;
}

// CTAs of a cluster for each sequence and task, 0: equal ranges.  The least time by a model (us): waves of clusters, each its start and the
// turns of a warp, which take longer the fuller the SMs are; joins; for ranges what all warps need together, a start for every task and
// the second kernel.  It goes by the table's width: lengths are known to the device alone.  Its numbers are those with which it lost
// least over 937 calls (1 to 128 sequences of 32 / 32, 64 / 8 and 16 / 4 heads, 60 to 65000 slots, equal and mixed lengths) with tables as wide as the
// longest sequence: the plan taken is 0.6 % behind the best on average, 12 % at most.  In wider tables it is further behind: 16 sequences of
// 32 / 32 heads with 110 slots take 8.7 us, in a table of 4096 slots 21.9, of 16384 15.4; 33 of 16 / 4 heads with 200 5.0, 5.0 and 10.2.  (16 sequences of 64 / 8 heads up to 4001 slots: 1 CTA 83 us, 2 53, 3 41, 4 50, 8 49, ranges
// 44; 8 of 40 heads, window 1021: 1 32, 2 39, ranges 38; 2 of 64 / 8 heads up to 20000 slots: 8 53, ranges 33; 24 of 16 / 4 heads, 1500 slots: 5
// 11.6, 6, of which the device does not hold 96, 16.8; 5 of them, 60 slots: 1 2.7, ranges 8.1.)
int plan_of(const cq_pages* pages, const cq_table* table, int n_heads, int window, int sinks) {
  const int KV = pages->n_kv_heads, chunks = (n_heads / KV + AT_HEADS - 1) / AT_HEADS, sms = cq_sm_count(), slots = per_sm(pages->head_dim) * sms;
  const bool narrow = pages->head_dim == 64;
  const double tasks = (double)table->sequences * KV * chunks;
  const long long all = (long long)table->width * pages->page_size;
  const long long most = window ? std::min<long long>(all, (long long)window + sinks + AT_SLOTS) : all, tiles = (most + AT_SLOTS - 1) / AT_SLOTS;
  const Held& device = held_by_device(pages->head_dim);
  double least = 13 + 3.4 * tasks / slots + std::max(1.0, tasks * tiles / (slots * AT_WARPS)) * (narrow ? 1.12 : 2.2);
  int best = 0;
  for (int n = 1; n <= MAX_CLUSTER; ++n) {
    if (n > 1 && (n - 1) * AT_WARPS >= tiles) break;
    const double held = device.clusters[n], each = std::min(held * n / sms, std::max(1.0, tasks * n / sms));
    const double turn = narrow ? std::max(0.97 + 0.11 * each, 0.31 * each) : std::max(0.82 + 0.45 * each, 0.7 * each);
    const double waves = tasks <= held ? 1.0 : 0.75 * tasks / held + 0.25 * std::ceil(tasks / held);
    const double t = 1.3 + waves * (((tiles + n * AT_WARPS - 1) / (n * AT_WARPS)) * turn + 2.0) + (n > 1 ? 1.35 + 0.085 * n : 0.0);
    if (t < least) {
      least = t;
      best = n;
    }
  }
  return best;
}

template <typename T, int D>
int attend(const cq_pages* pages, const cq_table* table, const cq_rows* q, const cq_rows* k, const cq_rows* v, const float* cos_t, const float* sin_t,
           const long long* positions, int table_rows, const long long* length, void* out, int H, int window, int sinks, float scale, void* workspace,
           cudaStream_t stream) {
  const int KV = pages->n_kv_heads, chunks = (H / KV + AT_HEADS - 1) / AT_HEADS, cluster = plan_of(pages, table, H, window, sinks), ctas = per_sm(D) * cq_sm_count();
  if (!cluster && !workspace) return CQ_ERR_BAD_ARG;
  const NewRow<T> fresh = {rows_of<T>(k), rows_of<T>(v), cos_t, sin_t, positions, table_rows};
  const Shape shape = {table->sequences, H, chunks, window, sinks, scale};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = cluster ? dim3(cluster, KV * chunks, table->sequences) : dim3(ctas);
  cfg.blockDim = dim3(AT_WARPS * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  auto fn = cluster ? (k ? pages_attend_kernel<T, D, true, true> : pages_attend_kernel<T, D, false, true>)
                    : (k ? pages_attend_kernel<T, D, true, false> : pages_attend_kernel<T, D, false, false>);
  CQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, rows_of<T>(q), pool_of<T>(pages), table_of(table), fresh, length, (T*)out, workspace, shape));
  if (!cluster) {
    // as many blocks as there are CTAs, or fewer
    const int tasks = std::min(table->sequences, ctas) * std::min(KV * chunks, ctas), most = std::min(AT_HEADS, H / KV);
    int heads = most;
    while (heads > 1 && tasks * ((most + heads / 2 - 1) / (heads / 2)) <= ctas) heads /= 2;
    CQ_CUDA_TRY(kv4_launch(pages_join_kernel<T, D>, dim3(std::min(tasks, ctas), (most + heads - 1) / heads), dim3(32 * JOIN_WARPS), 0, stream,
                           (const void*)workspace, length, shape, table->width * pages->page_size, (int)(k != nullptr), KV, ctas, heads, (T*)out));
  }
  return CQ_OK;
}

int call(const cq_pages* pages, const cq_table* table, const cq_rows* q, const cq_rows* k, const cq_rows* v, const float* cos_t, const float* sin_t,
         const long long* positions, int table_rows, const long long* length, void* out, int H, int window, int sinks, float scale, void* workspace,
         cudaStream_t stream) {
  const int rc = check(pages, table);
  if (rc != CQ_OK) return rc;
  if (!rows_fit(q) || !length || ((uintptr_t)length & 7) || !out || window < 0 || sinks < 0 || !(scale > 0.f) || (((uintptr_t)out | (uintptr_t)workspace) & 15)) return CQ_ERR_BAD_ARG;
  if (H < 1 || H % pages->n_kv_heads || (H + 7ll * pages->n_kv_heads) / 8 > 65535) return CQ_ERR_BAD_SHAPE;
  auto fn = pages->dtype == 0 ? (pages->head_dim == 128 ? attend<__half, 128> : attend<__half, 64>)
                              : (pages->head_dim == 128 ? attend<__nv_bfloat16, 128> : attend<__nv_bfloat16, 64>);
  return fn(pages, table, q, k, v, cos_t, sin_t, positions, table_rows, length, out, H, window, sinks, scale, workspace, stream);
}

}  // namespace

extern "C" size_t cq_pages_attend_workspace_bytes(const cq_pages* pages, const cq_table* table, int n_heads, int window, int sinks) {
  if (check(pages, table) != CQ_OK || n_heads < 1 || n_heads % pages->n_kv_heads || window < 0 || sinks < 0) return 0;
  if (plan_of(pages, table, n_heads, window, sinks)) return 0;
  return (size_t)per_sm(pages->head_dim) * cq_sm_count() * 2 * AT_HEADS * (pages->head_dim + PART) * sizeof(float);
}

extern "C" int cq_pages_attend(const cq_pages* pages, const cq_table* table, const cq_rows* q, const long long* length, void* out, int n_heads,
                               int window, int sinks, float scale, void* workspace, cq_stream_t stream) {
  return call(pages, table, q, nullptr, nullptr, nullptr, nullptr, nullptr, 0, length, out, n_heads, window, sinks, scale, workspace,
              (cudaStream_t)stream);
}

extern "C" int cq_pages_step(const cq_pages* pages, const cq_table* table, const cq_rows* q, const cq_rows* k, const cq_rows* v,
                             const float* cos_table, const float* sin_table, const long long* positions, int table_rows, const long long* length,
                             void* out, int n_heads, int window, int sinks, float scale, void* workspace, cq_stream_t stream) {
  if (!rows_fit(k) || !rows_fit(v)) return CQ_ERR_BAD_ARG;
  if (!tables_fit(cos_table, sin_table, positions, table_rows)) return CQ_ERR_BAD_ARG;
  return call(pages, table, q, k, v, cos_table, sin_table, positions, table_rows, length, out, n_heads, window, sinks, scale, workspace,
              (cudaStream_t)stream);
}
