// Attention of single tokens over the paged KV cache (layout: cq_pages.cuh); in the reference a part of its vendored LLaMA
// (llama/modeling_llama_quant.py:371-419 of the reference project).
//
// The bound is the cache, read once.  As in cq_attn.cu all query heads of a KV head share one tile of mma.sync m16n8k16, rows 0-7
// of A: scores S = Q . K^T with keys straight from the pages (the order of the columns inside a step is free as long as both
// operands agree), then the weights as the A operand of P . V.  A weight is two numbers of the cache's type, its upper bits in rows
// 0-7 and what is left in rows 8-15, which the heads leave empty.  An MMA cuts its sums off instead of rounding them: each one
// sums its 16 products alone, fp32 additions do the rest.  A warp takes 16 slots a turn (they lie in one page) and keeps its own
// running maximum, a whole number of powers of two, sum and weighted values; warps meet in shared memory, ranges of slots in the
// workspace.
#include <algorithm>
#include <cmath>

#include "cq_pages.cuh"

namespace {

using namespace cq_paged;

constexpr int AT_HEADS = 8;                  // query heads of a CTA
constexpr int AT_SLOTS = 16;                 // slots of a turn
constexpr int AT_WARPS = 4;

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^d of a whole number d <= 0; 0 below the normal numbers (and 1 for NaN, whose sums are NaN)
__device__ __forceinline__ float whole_pow2(float d) { return __int_as_float(max(0, 127 + __float2int_rn(d)) << 23); }
// the share of sums (maximum m, sum of weights l) in those that reach up to `top`: 0 where they have no slot, but 1 where their
// only scores are NaN
__device__ __forceinline__ float share_of(float m, float l, float top) { return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : whole_pow2(m - top); }
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
__device__ __forceinline__ int held(const long long* length, int s, int more, int slots) {
  const long long n = length[s];
  return n < 0 ? 0 : (n >= slots ? slots : (int)n + more);
}

// The step's new token: k, v (sequences, KV, D), not rotated
template <typename T> struct NewRow {
  Rows<T> k, v;
  const float *cos_t, *sin_t;
  const long long* positions;
  int table_rows;
};

template <typename T, int D, bool STEP>
__global__ void __launch_bounds__(AT_WARPS * 32, 3) pages_attend_kernel(const Rows<T> q, const Pool<T> pool, const Table table, const NewRow<T> fresh,
                                                                        const long long* __restrict__ length, T* __restrict__ out,
                                                                        float* __restrict__ part, int H, int chunks, int window, int sinks, float scale) {
  constexpr int THREADS = AT_WARPS * 32;
  constexpr int KP = D / 32;                 // 16-byte pieces of a key per lane (four lanes a slot)
  constexpr int VS = D / 64;                 // of a value (eight lanes a slot)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ __align__(16) float s_sum[AT_WARPS][AT_HEADS][D];
  __shared__ __align__(16) T s_q[AT_HEADS][D + 32];
  __shared__ float s_m[AT_WARPS][AT_HEADS], s_l[AT_WARPS][AT_HEADS];
  const int split = blockIdx.x, nsplit = gridDim.x, kvh = blockIdx.y / chunks, seq = blockIdx.z, KV = pool.heads;
  const int G = H / KV, h0 = (blockIdx.y - kvh * chunks) * AT_HEADS, heads = min(AT_HEADS, G - h0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g8 = lane >> 2, t4 = lane & 3;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int slots = table.width << pool.log_page;
  const Visible<AT_SLOTS> vis(held(length, seq, STEP, slots), window, sinks);
  const int each = (vis.tiles + nsplit - 1) / nsplit, tile0 = split * each, tile1 = min(vis.tiles, tile0 + each);
  const int head0 = kvh * G + h0;            // the CTA's first head, of a sequence's

  long long at = -1;                         // the new row's slot, where it is written
  bool turn = false;
  long long pos = 0;
  if (STEP) {
    pos = fresh.cos_t ? fresh.positions[seq] : 0;
    turn = fresh.cos_t && pos >= 0 && pos < fresh.table_rows;
    at = !fresh.cos_t || turn ? length[seq] : -1;
    if (at < 0 || at >= slots) at = -1;
  }
  // queries in shared memory, rotated: a lane's pieces 8 t4 + 32 i of head g8
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
  if (STEP && at >= 0 && tile1 == vis.tiles && tile0 < tile1 && tid < 2 * PIECES) {
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
  const T* mine_q = &s_q[g8][8 * t4];

  const float scale2 = scale * 1.4426950408889634f;        // scores in powers of two
  float m = -INFINITY, l = 0.f;
  float o[8 * VS][2];                        // MMA j + 8 s: its column n is column 64 s + 8 n + j of the head
#pragma unroll
  for (int i = 0; i < 8 * VS; ++i) o[i][0] = o[i][1] = 0.f;

#pragma unroll 1
  for (int i = tile0 + warp; i < tile1; i += AT_WARPS) {
    const int base = vis.tile(i) * AT_SLOTS, page = table.page_of(pool, seq, base);
    if (page < 0) continue;
    const size_t row0 = pool.rows(page, kvh) + (base & ((1 << pool.log_page) - 1));
    uint4 kk[2][KP], vv[4][VS];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < KP; ++e) kk[h][e] = ld16(pool.k + (row0 + 8 * h + g8) * D + 8 * t4 + 32 * e);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int p = 8 * (u >> 1) + 2 * t4 + (u & 1);
#pragma unroll
      for (int e = 0; e < VS; ++e) vv[u][e] = vis.sees(base + p) ? ld16(pool.v + (row0 + p) * D + 8 * g8 + 64 * e) : make_uint4(0, 0, 0, 0);
    }
    float s[2][2] = {};
#pragma unroll
    for (int e = 0; e < KP; ++e) {
      const uint4 qa = *reinterpret_cast<const uint4*>(mine_q + 32 * e);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float d0[4], d1[4];
        mma(d0, qa.x, 0u, qa.y, 0u, kk[h][e].x, kk[h][e].y, T());
        mma(d1, qa.z, 0u, qa.w, 0u, kk[h][e].z, kk[h][e].w, T());
        s[h][0] += d0[0] + d1[0];
        s[h][1] += d0[1] + d1[1];
      }
    }
    // this lane: head g8, slots base + 8 h + 2 t4 + e
    bool sees[2][2];
    float top = m;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sees[h][e] = vis.sees(base + 8 * h + 2 * t4 + e);
        top = fmaxf(top, sees[h][e] ? s[h][e] * scale2 : -INFINITY);
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // A whole number at or above the maximum, so that rescaling sums is exact.  (No finite score so far: weights 0, or NaN
    // where a score is NaN, which no maximum shows.)
    top = ceilf(top);
    const float ref = top == -INFINITY ? 0.f : top;
    const float keep = whole_pow2(m - ref);
    m = top;
    // weights times 2^15: fp16's halves of their split then reach down to 2^-38 of the largest
    float w[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) w[h][e] = sees[h][e] ? 32768.f * ex2(__fmaf_rn(s[h][e], scale2, -ref)) : 0.f;
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
        float d[4];
        mma(d, w0.x, w0.y, w1.x, w1.y, __byte_perm(v0[j >> 1], v1[j >> 1], sel), __byte_perm(v2[j >> 1], v3[j >> 1], sel), T());
        o[8 * e + j][0] = o[8 * e + j][0] * keep + (d[0] + d[2]);
        o[8 * e + j][1] = o[8 * e + j][1] * keep + (d[1] + d[3]);
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
    for (int c = 0; c < 2; ++c)              // columns n = 2 t4 + c
#pragma unroll
      for (int j = 0; j < 8; j += 4)
        *reinterpret_cast<float4*>(&s_sum[warp][g8][64 * e + 8 * (2 * t4 + c) + j]) =
            make_float4(o[8 * e + j][c], o[8 * e + j + 1][c], o[8 * e + j + 2][c], o[8 * e + j + 3][c]);
  __syncthreads();
  for (int i = tid; i < heads * D / 4; i += THREADS) {
    const int g = i / (D / 4), d = 4 * (i - g * (D / 4));
    float top = s_m[0][g];
#pragma unroll
    for (int w = 1; w < AT_WARPS; ++w) top = fmaxf(top, s_m[w][g]);
    float tot = 0.f, sum[4] = {};
#pragma unroll
    for (int w = 0; w < AT_WARPS; ++w) {
      const float f = share_of(s_m[w][g], s_l[w][g], top);
      const float4 x = *reinterpret_cast<const float4*>(&s_sum[w][g][d]);
      tot += f * s_l[w][g];
      sum[0] += f * x.x, sum[1] += f * x.y, sum[2] += f * x.z, sum[3] += f * x.w;
    }
    if (!(fabsf(sum[0]) + fabsf(sum[1]) + fabsf(sum[2]) + fabsf(sum[3]) <= 3.0e38f) && tot == tot) {
      // An infinite or NaN value takes part.  The two halves of a weight turn infinity into NaN where the product does
      // not: these columns are added again, weight by weight.
      sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
      for (int t = tile0; t < tile1; ++t)
        for (int j = vis.tile(t) * AT_SLOTS, end = j + AT_SLOTS; j < end; ++j) {
          const int page = vis.sees(j) ? table.page_of(pool, seq, j) : -1;
          if (page < 0) continue;
          const size_t row = pool.rows(page, kvh) + (j & ((1 << pool.log_page) - 1));
          float dot = 0.f;
          for (int c = 0; c < D; ++c) dot += Type<T>::one(s_q[g][c]) * Type<T>::one(pool.k[row * D + c]);
          const float w = 32768.f * ex2(__fmaf_rn(dot, scale2, top == -INFINITY ? 0.f : -top));
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[c] += w * Type<T>::one(pool.v[row * D + d + c]);
        }
    }
    const size_t head = (size_t)seq * H + head0 + g;
    if (nsplit == 1) {
      const bool none = tot == 0.f;          // no slot is visible (a visible one's weight is not 0)
      *reinterpret_cast<uint2*>(out + head * D + d) =
          none ? make_uint2(0u, 0u) : make_uint2(Type<T>::pair(sum[0] / tot, sum[1] / tot), Type<T>::pair(sum[2] / tot, sum[3] / tot));
    } else {
      float* mine = part + (head * nsplit + split) * (size_t)(D + 4);
      *reinterpret_cast<float4*>(mine + 4 + d) = make_float4(sum[0], sum[1], sum[2], sum[3]);
      if (d == 0) *reinterpret_cast<float2*>(mine) = make_float2(top, tot);
    }
  }
}

// joins a head's ranges: a warp a head, D / 32 columns a lane
template <typename T, int D>
__global__ void __launch_bounds__(256) pages_join_kernel(const float* __restrict__ part, int nsplit, long long heads, T* __restrict__ out) {
  constexpr int CPL = D / 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long head = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (head >= heads) return;
  const float* mine = part + (size_t)head * nsplit * (D + 4);
  const float2 ml = lane < nsplit ? *reinterpret_cast<const float2*>(mine + (size_t)lane * (D + 4)) : make_float2(-INFINITY, 0.f);
  float top = ml.x;
  for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float f = share_of(ml.x, ml.y, top);
  float tot = f * ml.y, sum[CPL] = {};
  for (int d = 16; d; d /= 2) tot += __shfl_xor_sync(0xffffffffu, tot, d);
#pragma unroll 8
  for (int r = 0; r < nsplit; ++r) {
    const float fr = __shfl_sync(0xffffffffu, f, r);
#pragma unroll
    for (int i = 0; i < CPL; i += 2) {
      const float2 x = *reinterpret_cast<const float2*>(mine + r * (D + 4) + 4 + CPL * lane + i);
      sum[i] = __fmaf_rn(fr, x.x, sum[i]);
      sum[i + 1] = __fmaf_rn(fr, x.y, sum[i + 1]);
    }
  }
  const bool none = tot == 0.f;
#pragma unroll
  for (int i = 0; i < CPL; i += 2)
    *reinterpret_cast<uint32_t*>(out + head * D + CPL * lane + i) = none ? 0u : Type<T>::pair(sum[i] / tot, sum[i + 1] / tot);
}

// ranges that a head's slots are cut into: what fills the SMs with three CTAs, four turns a warp at least
int splits_of(const cq_pages* pages, const cq_table* table, int n_heads, int window, int sinks) {
  const int KV = pages->n_kv_heads, chunks = (n_heads / KV + AT_HEADS - 1) / AT_HEADS;
  const long long tasks = (long long)table->sequences * KV * chunks, all = (long long)table->width * pages->page_size;
  const long long most = window ? std::min<long long>(all, (long long)window + sinks + AT_SLOTS) : all;
  return (int)std::max<long long>(1, std::min<long long>({32, 3 * cq_sm_count() / tasks, most / (4 * AT_WARPS * AT_SLOTS)}));
}

template <typename T, int D>
int attend(const cq_pages* pages, const cq_table* table, const cq_rows* q, const cq_rows* k, const cq_rows* v, const float* cos_t, const float* sin_t,
           const long long* positions, int table_rows, const long long* length, void* out, int H, int window, int sinks, float scale, void* workspace,
           cudaStream_t stream) {
  const int KV = pages->n_kv_heads, chunks = (H / KV + AT_HEADS - 1) / AT_HEADS, nsplit = splits_of(pages, table, H, window, sinks);
  const NewRow<T> fresh = {rows_of<T>(k), rows_of<T>(v), cos_t, sin_t, positions, table_rows};
  CQ_CUDA_TRY(kv4_launch(k ? pages_attend_kernel<T, D, true> : pages_attend_kernel<T, D, false>, dim3(nsplit, KV * chunks, table->sequences),
                         dim3(AT_WARPS * 32), 0, stream, rows_of<T>(q), pool_of<T>(pages), table_of(table), fresh, length, (T*)out, (float*)workspace, H,
                         chunks, window, sinks, scale));
  if (nsplit > 1) {
    const long long heads = (long long)table->sequences * H;
    CQ_CUDA_TRY(kv4_launch(pages_join_kernel<T, D>, dim3((unsigned)((heads + 7) / 8)), dim3(256), 0, stream, (const float*)workspace, nsplit, heads, (T*)out));
  }
  return CQ_OK;
}

int call(const cq_pages* pages, const cq_table* table, const cq_rows* q, const cq_rows* k, const cq_rows* v, const float* cos_t, const float* sin_t,
         const long long* positions, int table_rows, const long long* length, void* out, int H, int window, int sinks, float scale, void* workspace,
         cudaStream_t stream) {
  const int rc = check(pages, table);
  if (rc != CQ_OK) return rc;
  if (!rows_fit(q) || !length || !out || window < 0 || sinks < 0 || !(scale > 0.f) || (((uintptr_t)out | (uintptr_t)workspace) & 15)) return CQ_ERR_BAD_ARG;
  if (H < 1 || H % pages->n_kv_heads || (H + 7ll * pages->n_kv_heads) / 8 > 65535) return CQ_ERR_BAD_SHAPE;
  if (!workspace && cq_pages_attend_workspace_bytes(pages, table, H, window, sinks)) return CQ_ERR_BAD_ARG;
  auto fn = pages->dtype == 0 ? (pages->head_dim == 128 ? attend<__half, 128> : attend<__half, 64>)
                              : (pages->head_dim == 128 ? attend<__nv_bfloat16, 128> : attend<__nv_bfloat16, 64>);
  return fn(pages, table, q, k, v, cos_t, sin_t, positions, table_rows, length, out, H, window, sinks, scale, workspace, stream);
}

}  // namespace

extern "C" size_t cq_pages_attend_workspace_bytes(const cq_pages* pages, const cq_table* table, int n_heads, int window, int sinks) {
  if (check(pages, table) != CQ_OK || n_heads < 1 || n_heads % pages->n_kv_heads || window < 0 || sinks < 0) return 0;
  const int nsplit = splits_of(pages, table, n_heads, window, sinks);
  return nsplit > 1 ? (size_t)table->sequences * n_heads * nsplit * (pages->head_dim + 4) * 4 : 0;
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
  if (cos_table && (!sin_table || !positions || table_rows < 1)) return CQ_ERR_BAD_ARG;
  return call(pages, table, q, k, v, cos_table, sin_table, positions, table_rows, length, out, n_heads, window, sinks, scale, workspace,
              (cudaStream_t)stream);
}
