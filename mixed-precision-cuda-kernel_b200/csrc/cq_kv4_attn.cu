// Attention of single tokens over the 4-bit KV cache (layout: cq_kv4.cuh), with a sliding window and first slots that stay
// visible, and the weight that every slot received.  In the reference the cache is fp16 and attention torch's
// (llama/modeling_llama_quant.py:371-419 of the reference project).
//
//   out = sum_j p_j v_j,  p = softmax over the visible slots j of scale * q . k_j,
//   visible: j < n and (no window, or j < sinks, or j >= n - window)
//
// The bound is the cache, read once: 160 bytes a slot and KV head (D = 128, groups of 32), 222 cycles of an SM's share of HBM for 32
// slots of a head.  Taking the codes apart is what it costs beyond: 690 warp instructions for them (8 query heads), 172 cycles of
// the four schedulers if none ever waited; 60 % of their cycles issue one, tensor pipe 34 %.  4 sequences of 65536 slots with 8 KV
// heads: 81 us for 336 MB, a kernel that only copies them into shared memory 58.  So:
//   * slots are the M side of mma.sync.m16n8k16 and the (up to eight) query heads of a KV head its N side, in both products:
//     S^T = K Q^T and O^T = V^T P^T.  (With the heads on the M side half of every MMA and of its accumulators were empty.)
//     P^T is the accumulator of the first product, packed to fp16 and transposed by two movmatrix;
//   * keys: a masked word IS two fp16 numbers code * 2^-24 (below the normal range, exact), so codes go into the MMA with
//     five instructions a word and no conversion; an MMA sums the columns of one group alone, and its sums take the
//     group's scale in fp32.  The minima's part, sum over groups of minimum * (sum of the group's query columns), is one
//     MMA more, the query sums split into three fp16 numbers.  Nothing is rounded before the softmax but the sums;
//   * values: scale * code + minimum rounded to fp16 (three instructions for two), so that any column can ride with any
//     group, which costs an output about as much as its own rounding to fp16 does; weights are two fp16 numbers of 11 bits each and two
//     MMAs (rounded to one of them: error against 64 bits 3.5e-4 of the outputs' norm instead of 2.8e-4, 4 to 7 % less time);
//   * queries are scaled by a power of two, a head's largest to 16 .. 32, so that neither codes * 2^-24 nor a sixteenth of a
//     query (for the codes in the upper half of a byte) leaves fp16;
//   * a warp takes 32 slots a turn from a ring of its own in shared memory that cp.async fills (two turns), and keeps its own
//     running maximum, sum and weighted values; nothing waits for another warp until the end;
//   * several CTAs share a KV head's slots.  Where clusters of them fill the chip they meet in distributed shared memory, else
//     their sums go to the workspace and a small kernel joins them: no counters, nothing that two calls on one cache could confuse.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "cq_kv4.cuh"

namespace {

constexpr int AT_THREADS = 256;
constexpr int AT_HEADS = 8;                  // query heads of a CTA
constexpr int AT_SLOTS = 32;                 // slots of a turn
constexpr int AT_SM_WARPS = 16;              // warps an SM holds (128 registers a thread)
constexpr int AT_STAGES = 2;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float HEADROOM = 8.f, LIFT = 7.f;  // weights are 2^7 times the exponentials, at most 2^15, and fp16 reaches down to 2^-31 of them

__device__ __forceinline__ int held(const long long* length, int b, int more, int slots) {
  const long long n = length[b];
  return n < 0 ? 0 : (n >= slots ? slots : (int)n + (n < slots ? more : 0));
}

__device__ __forceinline__ void at_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with sums that start at 0
__device__ __forceinline__ void at_mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 16 bytes that are read once: they leave L2 first
__device__ __forceinline__ void copy16(uint32_t to, const void* from, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "l"(policy) : "memory");
}
__device__ __forceinline__ uint64_t evict_first() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint32_t hadd2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// (x & MASK) | y in one instruction
template <uint32_t MASK> __device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t y) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(x), "n"(MASK), "r"(y));
  return d;
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
template <int WORDS> __device__ __forceinline__ void lds(uint32_t at, uint32_t (&v)[WORDS]) {
  if constexpr (WORDS == 4) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
  else if constexpr (WORDS == 2) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(at));
  else v[0] = lds32(at);
}
// the same shared-memory address in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t in_cta(uint32_t at, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A turn's slots in shared memory: codes of keys and values in pieces of 16 bytes, their order within a row turned so that
// the lanes' words lie in different banks; then the scales of both.
template <int D, int NG> struct Turn {
  static constexpr int ROW = D / 2, CODES = AT_SLOTS * ROW, SCALES = AT_SLOTS * NG * 4, BYTES = 2 * (CODES + SCALES);
  __device__ __forceinline__ static int piece(int row, int c) {        // where piece c of a row lies
    return row * ROW + 16 * (c ^ (D == 128 ? (row >> 1) & 3 : (row >> 2) & 1));
  }
  // which of eight slots is row (column) 2 t + e of the MMAs: such that the value words of the four lanes t lie in different banks
  __device__ __forceinline__ static int slot(int t, int e) { return D == 128 ? (t & 1) + 4 * (t >> 1) + 2 * e : t + 4 * e; }
};

// the slots that are visible, as a list of turns: `ns` from the first on, then those from wt0 on
struct Visible {
  int n, first, from, ns, wt0, turns;
  __device__ __forceinline__ Visible(int n_, int window, int sinks) : n(n_) {
    from = window ? max(0, n - window) : 0;
    first = window ? min(sinks, from) : 0;
    const int all = (n + AT_SLOTS - 1) / AT_SLOTS;
    ns = (first + AT_SLOTS - 1) / AT_SLOTS;
    wt0 = from / AT_SLOTS;
    if (ns >= wt0) ns = wt0 = 0;             // one run from the first slot on
    turns = ns + all - wt0;
  }
  __device__ __forceinline__ int base(int v) const { return AT_SLOTS * (v < ns ? v : v - ns + wt0); }
  __device__ __forceinline__ bool sees(int slot) const { return slot < n && (slot < first || slot >= from); }
  __device__ __forceinline__ bool whole(int b) const { return b + AT_SLOTS <= n && (b >= from || b + AT_SLOTS <= first); }
};

struct NewRow {
  const __half *k, *v;                       // [sequence][KV][D]; null: no step
  const float *cos_t, *sin_t;                // null: no rotation
  const long long* positions;
  int table_rows;
};

template <int D, int NG, int WARPS, bool STEP, bool WEIGHTS>
__global__ void __launch_bounds__(WARPS * 32, AT_SM_WARPS / WARPS) kv4_attend_kernel(
    const __half* __restrict__ q, const cq_kv4 cache, const NewRow fresh, const long long* __restrict__ length, __half* __restrict__ out,
    float* __restrict__ scores, float2* __restrict__ stats, float* __restrict__ part, int H, int chunks, int window, int sinks, float scale) {
  using T = Turn<D, NG>;
  constexpr int THREADS = WARPS * 32, GROUP = D / NG, NW = D / 32, WG = GROUP / 32;     // words of a key per lane, of a group
  constexpr int VW = D / 64, LANES = D / 16;                                            // words of a value per lane; lanes of a row
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(128) uint8_t ring[];          // [warp][stage][turn]; then [warp][head][D] fp32
  __shared__ __align__(16) __half s_q[AT_HEADS][D + 8];
  __shared__ float s_unit[AT_HEADS];                       // 2^-e of each head's scaled queries
  __shared__ float s_m[WARPS][AT_HEADS], s_l[WARPS][AT_HEADS];
  __shared__ __align__(16) float s_part[AT_HEADS][D];
  __shared__ float s_pm[AT_HEADS], s_pl[AT_HEADS];
  __shared__ uint32_t s_const[4];
  __shared__ __align__(16) uint32_t s_row[2][D / 8], s_pairs[2][NG];                    // the new row: codes and scales of key, value
  const int kvh = blockIdx.y / chunks, chunk = blockIdx.y - kvh * chunks, b = blockIdx.z;
  const int split = blockIdx.x, nsplit = gridDim.x;        // (a cluster, where there is one, is the CTAs of one row of the grid)
  const int G = H / cache.n_kv_heads, heads = min(AT_HEADS, G - chunk * AT_HEADS);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g8 = lane >> 2, t4 = lane & 3;
  const size_t head0 = (size_t)b * H + (size_t)kvh * G + chunk * AT_HEADS, row0 = ((size_t)b * cache.n_kv_heads + kvh) * cache.slots;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Visible vis(held(length, b, STEP ? 1 : 0, cache.slots), window, sinks);
  if (tid < 3) s_const[tid] = tid == 0 ? 0x64006400u : (tid == 1 ? 0x2C002C00u : 0xD400D400u);

  const uint32_t my_ring = (uint32_t)__cvta_generic_to_shared(ring) + warp * (AT_STAGES * T::BYTES);
  const int stride = nsplit * WARPS;
  const uint64_t policy = evict_first();
  auto fetch = [&](int v, int stage) {
    if (v < vis.turns) {
      const int base = vis.base(v);
      const uint32_t to = my_ring + stage * T::BYTES;
      const uint8_t* kc = (const uint8_t*)cache.k_codes + (row0 + base) * T::ROW;
      const uint8_t* vc = (const uint8_t*)cache.v_codes + (row0 + base) * T::ROW;
#pragma unroll
      for (int i = 0; i < T::CODES / 512; ++i) {
        const int p = lane + 32 * i, at = T::piece(p / (T::ROW / 16), p % (T::ROW / 16));
        copy16(to + at, kc + 16 * p, policy);
        copy16(to + T::CODES + at, vc + 16 * p, policy);
      }
      if (NG == 4 || lane < 8 * NG) {
        copy16(to + 2 * T::CODES + 16 * lane, (const uint8_t*)cache.k_scales + (row0 + base) * (4 * NG) + 16 * lane, policy);
        copy16(to + 2 * T::CODES + T::SCALES + 16 * lane, (const uint8_t*)cache.v_scales + (row0 + base) * (4 * NG) + 16 * lane, policy);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int v = split * WARPS + warp;
#pragma unroll
  for (int i = 0; i < AT_STAGES; ++i) fetch(v + i * stride, i);

  // queries: rotated, scaled by a power of two, to shared memory; D / 16 lanes a head
  const long long pos = STEP && fresh.cos_t ? fresh.positions[b] : 0;
  const bool turn = STEP && fresh.cos_t && pos >= 0 && pos < fresh.table_rows;
  for (int i = tid; i < AT_HEADS * LANES; i += THREADS) {
    const int g = i / LANES, c = 8 * (i % LANES);
    uint32_t row[8] = {};
    if (g < heads) {
      const __half* src = q + (head0 + g) * D + c;
      kv4_load16(src, src + D / 2, row);
      if (turn) kv4_rotate<false>(row, fresh.cos_t + pos * (D / 2) + c, fresh.sin_t + pos * (D / 2) + c);
    }
    float x[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 f = apart(kv4_two(row[e]));
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const int up = top > 0.f && top < INFINITY ? 131 - (int)(__float_as_uint(top) >> 23) : 0;       // the largest to 2^4 .. 2^5
    const float by = __int_as_float((127 + up) << 23);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] *= by;
    *reinterpret_cast<uint4*>(&s_q[g][c]) = kv4_halves(x);
    *reinterpret_cast<uint4*>(&s_q[g][c + D / 2]) = kv4_halves(x + 8);
    if (c == 0) s_unit[g] = __int_as_float((127 - up) << 23);
  }
  // the new row, quantised where its turn is read; it goes to the cache after the last read of it here.  (Other CTAs of more
  // than eight query heads may still read the slot while the first one writes it: what they read there is not used.)
  const int last = vis.turns - 1;
  const bool owner = STEP && last >= 0 && last % stride / WARPS == split;
  const long long slot_new = STEP ? length[b] : -1;
  const bool writes = STEP && slot_new >= 0 && slot_new < cache.slots && (turn || !fresh.cos_t);
  if (STEP && owner && warp == WARPS - 1) {
    const int which = lane / LANES & 1, c = 8 * (lane % LANES);
    const __half* src = (which ? fresh.v : fresh.k) + ((size_t)b * cache.n_kv_heads + kvh) * D + c;
    uint32_t x[8];
    kv4_load16(src, src + D / 2, x);
    if (!which && turn) kv4_rotate<false>(x, fresh.cos_t + pos * (D / 2) + c, fresh.sin_t + pos * (D / 2) + c);
    uint32_t words[2], pairs[2];
    kv4_quantise<D, GROUP>(x, words, pairs);
    if (lane < 2 * LANES) {
      s_row[which][c / 8] = words[0];
      s_row[which][c / 8 + D / 16] = words[1];
      if (c % GROUP == 0) {
        s_pairs[which][c / GROUP] = pairs[0];
        if (GROUP != D) s_pairs[which][(c + D / 2) / GROUP] = pairs[1];
      }
    }
  }
  __syncthreads();

  // Numbers of the values' conversion: 1024 (a code in the lowest bits adds itself), 1 / 16 and -64.  Read back from shared
  // memory because the compiler, if it knows them, makes two instructions of one, an immediate in each.
  const uint32_t consts = (uint32_t)__cvta_generic_to_shared(s_const);
  const uint32_t magic = lds32(consts), sixteenth = lds32(consts + 4), minus64 = lds32(consts + 8);

  // B operands of the first product: head g8; word i holds columns 32 i + 8 t4 .. + 7
  uint32_t qb[NW][4], qs[2];
  float sums[NG] = {};
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const uint4 w = *reinterpret_cast<const uint4*>(&s_q[g8][32 * i + 8 * t4]);
    const uint32_t h[4] = {w.x, w.y, w.z, w.w};            // columns (0 1) (2 3) (4 5) (6 7)
    qb[i][0] = __byte_perm(h[0], h[2], 0x5410);            // 0, 4
    qb[i][1] = __byte_perm(h[1], h[3], 0x5410);            // 2, 6
    const __half2 part16 = __float2half2_rn(0.0625f);
    __half2 odd = __hmul2(__halves2half2(__ushort_as_half(h[0] >> 16), __ushort_as_half(h[2] >> 16)), part16);
    qb[i][2] = *reinterpret_cast<uint32_t*>(&odd);         // 1, 5
    odd = __hmul2(__halves2half2(__ushort_as_half(h[1] >> 16), __ushort_as_half(h[3] >> 16)), part16);
    qb[i][3] = *reinterpret_cast<uint32_t*>(&odd);         // 3, 7
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
      sums[i / WG] += f.x + f.y;
    }
  }
  {
    float part[4] = {};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
      sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
      // lane t4 = 0, 1, 2 has the first, second, third 11 bits
      float rest = sums[g];
      for (int i = 0; i < t4; ++i) rest -= __half2float(__float2half_rn(rest));
      part[g] = t4 < 3 ? rest : 0.f;
    }
    qs[0] = pair_of(part[0], part[1]);
    qs[1] = pair_of(part[2], part[3]);
  }
  const float unit[2] = {s_unit[2 * t4] * scale * LOG2E, s_unit[2 * t4 + 1] * scale * LOG2E};      // heads 2 t4, 2 t4 + 1

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {}, lifted[2] = {-LIFT, -LIFT};
  float o[4 * VW][4] = {};                   // MMA j: rows g8, g8 + 8 are the columns (16 or 8) g8 + 2 j, + 1; heads 2 t4, + 1
  // Where this lane's words lie in a turn.  (A row's bytes start at a multiple of its length, so that the turned order of its
  // pieces is an exclusive or with the address; what is added beyond is a constant of the instruction.)
  constexpr int R = T::ROW;
  const int row_k = T::slot(g8 >> 1, g8 & 1), row_v = T::slot(t4, 0), row_step = T::slot(0, 1);
  const uint32_t off_k = T::piece(row_k, 0) + 4 * t4;
  const int word_v = D == 128 ? 8 * (g8 & 1) : 4 * (g8 & 3), piece_v = g8 / (D == 128 ? 2 : 4);
  const uint32_t off_v[2] = {(uint32_t)(T::CODES + T::piece(row_v, piece_v) + word_v), (uint32_t)(T::CODES + T::piece(row_v + row_step, piece_v) + word_v)};
  const uint32_t off_ks = 2 * T::CODES + row_k * (4 * NG), off_vs = 2 * T::CODES + T::SCALES + (row_v * NG + g8 * (D / 8) / GROUP) * 4;
  auto take = [&](uint32_t at, int base, auto all) {
    constexpr bool ALL = decltype(all)::value;             // every slot of the turn is visible
    float s[2][4];                                         // [half of the turn][slot g8: 2 heads, slot g8 + 8: 2 heads]
    uint32_t at_k[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) at_k[i] = (at + off_k) ^ (16 * i);
    const uint32_t at_ks = at + off_ks, at_vs = at + off_vs, at_v[2] = {at + off_v[0], at + off_v[1]};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t k0[NG], k1[NG];
      lds<NG>(at_ks + (16 * u) * (4 * NG), k0);
      lds<NG>(at_ks + (16 * u + 8) * (4 * NG), k1);
      float sum[4];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float d[4];
#pragma unroll
        for (int i = g * WG; i < (g + 1) * WG; ++i) {
          const uint32_t w0 = lds32(at_k[i] + 16 * u * R), w1 = lds32(at_k[i] + (16 * u + 8) * R);
          const uint32_t x0 = w0 >> 8, x1 = w1 >> 8;
          if (i == g * WG) at_mma0(d, w0 & 0x000F000Fu, w1 & 0x000F000Fu, x0 & 0x000F000Fu, x1 & 0x000F000Fu, qb[i][0], qb[i][1]);
          else at_mma(d, w0 & 0x000F000Fu, w1 & 0x000F000Fu, x0 & 0x000F000Fu, x1 & 0x000F000Fu, qb[i][0], qb[i][1]);
          at_mma(d, w0 & 0x00F000F0u, w1 & 0x00F000F0u, x0 & 0x00F000F0u, x1 & 0x00F000F0u, qb[i][2], qb[i][3]);
        }
        const float f0 = __low2float(*reinterpret_cast<const __half2*>(&k0[g])), f1 = __low2float(*reinterpret_cast<const __half2*>(&k1[g]));
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = g == 0 ? (e < 2 ? f0 : f1) * d[e] : __fmaf_rn(e < 2 ? f0 : f1, d[e], sum[e]);
      }
      float low[4];
      const uint32_t a0 = NG > 1 ? __byte_perm(k0[0], k0[NG > 1], 0x7632) : k0[0] >> 16, a1 = NG > 1 ? __byte_perm(k1[0], k1[NG > 1], 0x7632) : k1[0] >> 16;
      const uint32_t a2 = NG > 2 ? __byte_perm(k0[NG > 2 ? 2 : 0], k0[NG > 2 ? 3 : 0], 0x7632) : 0u;
      const uint32_t a3 = NG > 2 ? __byte_perm(k1[NG > 2 ? 2 : 0], k1[NG > 2 ? 3 : 0], 0x7632) : 0u;
      at_mma0(low, a0, a1, a2, a3, qs[0], qs[1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[u][e] = __fmaf_rn(sum[e], 16777216.f, low[e]) * unit[e & 1];
        const int slot = base + 16 * u + row_k + (e < 2 ? 0 : 8);
        if (!ALL && !vis.sees(slot)) s[u][e] = -INFINITY;
        else if (WEIGHTS && 2 * t4 + (e & 1) < heads) scores[(head0 + 2 * t4 + (e & 1)) * cache.slots + slot] = s[u][e];
      }
    }
    // The reference of the weights is a whole number, so that sums are rescaled exactly, and is only raised when a score is 2^8
    // above it: the lanes' own maxima are enough to see that none is.
    float top[2];
    bool above = false;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = fmaxf(fmaxf(s[0][e], s[0][e + 2]), fmaxf(s[1][e], s[1][e + 2]));
      above |= top[e] > m[e] + HEADROOM;
    }
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], d));
        const float now = fmaxf(m[e], ceilf(top[e])), keep = ex2(m[e] - (now == -INFINITY ? 0.f : now));
        m[e] = now;
        lifted[e] = (now == -INFINITY ? 0.f : now) - LIFT;
        l[e] *= keep;
#pragma unroll
        for (int j = 0; j < 4 * VW; ++j) {
          o[j][e] *= keep;
          o[j][e + 2] *= keep;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = ex2(s[u][e] - lifted[e & 1]);
        l[e & 1] += w[e];
      }
      // the weights' upper 11 bits, and the next 11
      const uint32_t h0 = pair_of(w[0], w[1]), h1 = pair_of(w[2], w[3]);
      const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
      const uint32_t p0 = transposed(h0), p1 = transposed(h1);
      const uint32_t r0 = transposed(pair_of(w[0] - f0.x, w[1] - f0.y)), r1 = transposed(pair_of(w[2] - f1.x, w[3] - f1.y));
      // two slots' words side by side: [slots 0-7 | 8-15]
      uint32_t sc[2], mn[2], vw[2][2][VW];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pair[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 16 * u + 8 * h;
          lds<VW>(at_v[e] + r * R, vw[h][e]);
          pair[e] = lds32(at_vs + (r + e * row_step) * (4 * NG));
          if (!ALL && !vis.sees(base + r + row_v + e * row_step)) pair[e] = 0;      // (what is not visible may be anything, NaN too)
        }
        sc[h] = __byte_perm(pair[0], pair[1], 0x5410);
        mn[h] = __byte_perm(pair[0], pair[1], 0x7632);
      }
#pragma unroll
      for (int i = 0; i < VW; ++i)
#pragma unroll
        for (int y = 0; y < 2; ++y) {                      // codes 0-3, 4-7 of a word
          uint32_t a[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x = __byte_perm(vw[h][0][i], vw[h][1][i], y ? 0x7632 : 0x5410), z = x >> 8;
            a[h][0] = hfma2(hadd2(and_or<0x000F000Fu>(x, magic), 0xE400E400u), sc[h], mn[h]);
            a[h][1] = hfma2(hfma2(and_or<0x00F000F0u>(x, magic), sixteenth, minus64), sc[h], mn[h]);
            a[h][2] = hfma2(hadd2(and_or<0x000F000Fu>(z, magic), 0xE400E400u), sc[h], mn[h]);
            a[h][3] = hfma2(hfma2(and_or<0x00F000F0u>(z, magic), sixteenth, minus64), sc[h], mn[h]);
          }
          at_mma(o[4 * i + 2 * y], a[0][0], a[0][1], a[1][0], a[1][1], p0, p1);
          at_mma(o[4 * i + 2 * y + 1], a[0][2], a[0][3], a[1][2], a[1][3], p0, p1);
          at_mma(o[4 * i + 2 * y], a[0][0], a[0][1], a[1][0], a[1][1], r0, r1);
          at_mma(o[4 * i + 2 * y + 1], a[0][2], a[0][3], a[1][2], a[1][3], r0, r1);
        }
    }
  };

  int stage = 0;
#pragma unroll 1
  for (; v < vis.turns; v += stride) {
    asm volatile("cp.async.wait_group %0;" ::"n"(AT_STAGES - 1) : "memory");
    __syncwarp();
    const uint32_t at = my_ring + stage * T::BYTES;
    const int base = vis.base(v);
    if (STEP && v == last && writes) {
      const int r = (int)slot_new - base;                  // (the last slot of the last turn's)
      uint8_t* to = ring + (at - (uint32_t)__cvta_generic_to_shared(ring));
      for (int i = lane; i < 2 * (D / 8); i += 32) {
        const int which = i / (D / 8), w = i % (D / 8);
        *reinterpret_cast<uint32_t*>(to + which * T::CODES + T::piece(r, w / 4) + 4 * (w % 4)) = s_row[which][w];
      }
      if (lane < 2 * NG) *reinterpret_cast<uint32_t*>(to + 2 * T::CODES + lane / NG * T::SCALES + (r * NG + lane % NG) * 4) = s_pairs[lane / NG][lane % NG];
      __syncwarp();
    }
    if (vis.whole(base)) take(at, base, std::true_type());
    else take(at, base, std::false_type());
    __syncwarp();
    fetch(v + AT_STAGES * stride, stage);
    stage = stage == AT_STAGES - 1 ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();

  // the warps' sums meet
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int d = 4; d < 32; d *= 2) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
    if (g8 == 0) {
      s_m[warp][2 * t4 + e] = m[e];
      s_l[warp][2 * t4 + e] = l[e];
    }
    float* to = reinterpret_cast<float*>(ring + warp * (AT_STAGES * T::BYTES)) + (2 * t4 + e) * D + g8 * (D / 8);
#pragma unroll
    for (int j = 0; j < 4 * VW; j += 2)
      *reinterpret_cast<float4*>(to + 2 * j) = make_float4(o[j][e], o[j][e + 2], o[j + 1][e], o[j + 1][e + 2]);
  }
  __syncthreads();
  if (STEP && owner && writes && chunk == 0) {
    const size_t at = row0 + slot_new;
    for (int i = tid; i < 2 * (D / 8); i += THREADS) {
      const int which = i / (D / 8), w = i % (D / 8);
      reinterpret_cast<uint32_t*>((uint8_t*)(which ? cache.v_codes : cache.k_codes) + at * T::ROW)[w] = s_row[which][w];
    }
    if (tid < 2 * NG) reinterpret_cast<uint32_t*>(tid / NG ? cache.v_scales : cache.k_scales)[at * NG + tid % NG] = s_pairs[tid / NG][tid % NG];
  }
  if (tid < AT_HEADS) {
    float top = -INFINITY, tot = 0.f;
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_m[w][tid]);
    for (int w = 0; w < WARPS; ++w) {
      // a warp without a finite score: no share, or NaN where it met one (which no maximum shows)
      const float f = s_m[w][tid] == -INFINITY ? (s_l[w][tid] == 0.f ? 0.f : 1.f) : ex2(s_m[w][tid] - top);
      tot += f * s_l[w][tid];
      s_m[w][tid] = f;
    }
    s_pm[tid] = top;
    s_pl[tid] = tot;
  }
  __syncthreads();
  for (int i = tid; i < heads * D / 4; i += THREADS) {
    const int g = i / (D / 4), c = 4 * (i % (D / 4));
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int w = 0; w < WARPS; ++w) {
      const float f = s_m[w][g];
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(ring + w * (AT_STAGES * T::BYTES)) + g * D + c);
      sum.x += f * x.x;
      sum.y += f * x.y;
      sum.z += f * x.z;
      sum.w += f * x.w;
    }
    if (nsplit == 1) {
      const float inv = vis.n ? 1.f / s_pl[g] : 0.f;
      *reinterpret_cast<uint2*>(out + (head0 + g) * D + c) =
          vis.n ? make_uint2(pair_of(sum.x * inv, sum.y * inv), pair_of(sum.z * inv, sum.w * inv)) : make_uint2(0, 0);
    } else if (part) {
      *reinterpret_cast<float4*>(part + (((head0 + g) * nsplit + split) * (D + 4) + 4 + c)) = sum;
    } else {
      *reinterpret_cast<float4*>(&s_part[g][c]) = sum;
    }
  }
  if (nsplit == 1) {
    if (WEIGHTS && tid < heads) stats[head0 + tid] = make_float2((s_pm[tid] == -INFINITY ? 0.f : s_pm[tid]) - LIFT, s_pl[tid]);
    return;
  }
  if (part) {
    if (tid < heads) *reinterpret_cast<float2*>(part + ((head0 + tid) * nsplit + split) * (D + 4)) = make_float2(s_pm[tid], s_pl[tid]);
    return;
  }
  cluster_barrier();
  // every CTA joins its share of the columns, two a thread
  const uint32_t pm = (uint32_t)__cvta_generic_to_shared(s_pm), pl = (uint32_t)__cvta_generic_to_shared(s_pl);
  const uint32_t parts = (uint32_t)__cvta_generic_to_shared(s_part);
  const int pairs = heads * D / 2, mine = (pairs + nsplit - 1) / nsplit;
  for (int i = split * mine + tid; i < min(pairs, (split + 1) * mine); i += THREADS) {
    const int g = i / (D / 2), c = 2 * (i % (D / 2));
    float top = -INFINITY, tot = 0.f, x = 0.f, y = 0.f;
    for (int r = 0; r < nsplit; ++r) top = fmaxf(top, ld_cluster(in_cta(pm + 4 * g, r)));
#pragma unroll 4
    for (int r = 0; r < nsplit; ++r) {
      const float mr = ld_cluster(in_cta(pm + 4 * g, r)), lr = ld_cluster(in_cta(pl + 4 * g, r));
      const float f = mr == -INFINITY ? (lr == 0.f ? 0.f : 1.f) : ex2(mr - top);
      tot += f * lr;
      x += f * ld_cluster(in_cta(parts + 4 * (g * D + c), r));
      y += f * ld_cluster(in_cta(parts + 4 * (g * D + c + 1), r));
    }
    *reinterpret_cast<uint32_t*>(out + (head0 + g) * D + c) = vis.n ? pair_of(x / tot, y / tot) : 0u;
    if (WEIGHTS && c == 0) stats[head0 + g] = make_float2((top == -INFINITY ? 0.f : top) - LIFT, tot);
  }
  cluster_barrier();                                       // (nobody leaves while its sums are read)
}

// The parts of a query head's sums in the workspace, [head][part][maximum, sum, -, -, D values]: a warp per head.
template <int D>
__global__ void __launch_bounds__(AT_THREADS) kv4_join_kernel(const float* __restrict__ part, int nsplit, long long heads, __half* __restrict__ out, float2* __restrict__ stats) {
  constexpr int CPL = D / 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long head = (long long)blockIdx.x * (AT_THREADS / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (head >= heads) return;
  const float* mine = part + head * nsplit * (D + 4);
  const float2 ml = lane < nsplit ? *reinterpret_cast<const float2*>(mine + lane * (D + 4)) : make_float2(-INFINITY, 0.f);      // (at most 32 parts)
  float top = ml.x;
  for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2(ml.x - top);
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
  const bool none = tot == 0.f;                            // no slot is visible (a visible one's weight is not 0)
#pragma unroll
  for (int i = 0; i < CPL; i += 2)
    *reinterpret_cast<uint32_t*>(out + head * D + CPL * lane + i) = none ? 0u : pair_of(sum[i] / tot, sum[i + 1] / tot);
  if (stats && lane == 0) stats[head] = make_float2((top == -INFINITY ? 0.f : top) - LIFT, tot);
}

// weights_out = weights + the sum of the weights of the head's queries; 0 from slot n on.  A new slot (more) has none before.
// Four slots a thread.
__global__ void __launch_bounds__(AT_THREADS) kv4_weights_kernel(const float* __restrict__ scores, const float2* __restrict__ stats,
                                                                 const long long* __restrict__ length, int more, const float* weights,
                                                                 float* weights_out, int H, int KV, int slots, int window, int sinks) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int slot = 4 * (blockIdx.x * AT_THREADS + threadIdx.x), kv = blockIdx.y, b = blockIdx.z, G = H / KV;
  if (slot >= slots) return;
  const Visible vis(held(length, b, more, slots), window, sinks);
  const size_t at = ((size_t)b * KV + kv) * slots + slot;
  float sum[4] = {};
  if (slot < vis.n && (slot < vis.first || slot + 3 >= vis.from)) {
    const size_t head0 = (size_t)b * H + (size_t)kv * G;
#pragma unroll 8
    for (int g = 0; g < G; ++g) {
      const float2 ml = stats[head0 + g];
      const float4 s = *reinterpret_cast<const float4*>(scores + (head0 + g) * slots + slot);
      const float inv = 1.f / ml.y;
      sum[0] += ex2(s.x - ml.x) * inv;
      sum[1] += ex2(s.y - ml.x) * inv;
      sum[2] += ex2(s.z - ml.x) * inv;
      sum[3] += ex2(s.w - ml.x) * inv;
    }
  }
  const long long fresh = more ? length[b] : -1;
  const float4 old = slot < vis.n ? *reinterpret_cast<const float4*>(weights + at) : make_float4(0.f, 0.f, 0.f, 0.f);
  const float before[4] = {old.x, old.y, old.z, old.w};
  float w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = slot + e < vis.n ? (slot + e == fresh ? 0.f : before[e]) + (vis.sees(slot + e) ? sum[e] : 0.f) : 0.f;
  *reinterpret_cast<float4*>(weights_out + at) = make_float4(w[0], w[1], w[2], w[3]);
}

// The CTAs of a call: their warps, how many share a head's slots, and whether those are clusters.
struct Shape {
  int warps, splits;
  bool cluster;
};
constexpr int AT_MAX_SPLITS = 32;            // (a lane each where they are joined)
Shape plan_of(const cq_kv4* cache, int n_heads, int window, int sinks, int sms) {
  const int B = cache->sequences, KV = cache->n_kv_heads, chunks = (n_heads / KV + AT_HEADS - 1) / AT_HEADS;
  const long long tasks = (long long)B * KV * chunks;
  const long long most = window ? std::min<long long>(cache->slots, (long long)window + sinks + AT_SLOTS) : cache->slots;
  const int turns = (int)((most + AT_SLOTS - 1) / AT_SLOTS);
  // The least time by a model (us): waves of CTAs, each its start and the turns of a warp, which take longer the fuller the SM
  // is; joins as clusters (of 2, 4 or 8, which GPCs hold without a rest: 40 heads of 9984 slots with clusters of 7 33 us, with
  // 7 unclustered CTAs 24.6) or through the workspace.  Over 29 shapes (1 to 64 sequences, 1 to 40 KV heads, 128 to 131072
  // slots), each timed with every plan, the plans it takes are 2 % slower than the best ones on average, 15 % at most.
  // (16 sequences of 64 heads on 8 KV heads, 4096 slots: 16 warps, one CTA a head 26.1 us, 4 warps 31.2; 1 sequence of 65536:
  // 18 CTAs of 8 warps 31.2, clusters of 8 of 16 warps 42; 32 heads of 512 slots in 32 sequences: 4 warps 30.7, 16 68.6.)
  Shape best = {4, 1, false};
  double least = 0;
  for (int w : {4, 8, 16})
    for (int n = 1; n <= AT_MAX_SPLITS; ++n) {
      if (n > 1 && (long long)(n - 1) * w >= turns) break;
      const long long ctas = tasks * n;
      const double waves = (double)ctas / (sms * (AT_SM_WARPS / w)), whole = std::ceil(waves);
      const double part = w == 4 ? 0.37 : (w == 8 ? 0.73 : 0.87), filled = std::max(1.0, part * whole + (1 - part) * waves);
      const int per_sm = (int)std::min<long long>(AT_SM_WARPS, w * ((ctas + sms - 1) / sms));
      const double turn = (1.43 + 0.85 * std::max(0, per_sm - 4) / 12) * (cache->head_dim == 64 ? 0.47 : 1.0);
      const double body = filled * (((turns + n * w - 1) / (n * w)) * turn + 1.4 + 0.05 * w);
      const bool cluster = n == 2 || n == 4 || n == 8;
      const double t = body + (n == 1 ? 0.0 : (cluster ? 1.65 + 0.15 * n : 8.7 + 0.05 * n));
      if (least == 0 || t < least) {
        least = t;
        best = {w, n, n > 1 && cluster};
      }
    }
  return best;
}
// A program's calls are alike from one to the next, and the model takes 1 to 2 us of the host: the last plan of a thread stays.
Shape shape_of(const cq_kv4* cache, int n_heads, int window, int sinks) {
  struct Asked {
    int sequences, n_kv_heads, slots, head_dim, n_heads, window, sinks, sms;
  };
  thread_local Asked last = {};
  thread_local Shape plan = {};
  const Asked now = {cache->sequences, cache->n_kv_heads, cache->slots, cache->head_dim, n_heads, window, sinks, cq_sm_count()};
  if (std::memcmp(&now, &last, sizeof(now)) != 0) {
    plan = plan_of(cache, n_heads, window, sinks, now.sms);
    last = now;
  }
  return plan;
}
size_t sums_bytes(const cq_kv4* cache, int n_heads, const Shape& s) {
  return s.splits > 1 && !s.cluster ? (size_t)cache->sequences * n_heads * s.splits * (cache->head_dim + 4) * 4 : 0;
}

int attend(const cq_kv4* cache, const void* q, const NewRow& fresh, const long long* length, void* out, int n_heads, int window, int sinks,
           float scale, const float* weights, float* weights_out, void* workspace, cudaStream_t stream) {
  const int B = cache->sequences, KV = cache->n_kv_heads, D = cache->head_dim, NG = D / cache->group, more = fresh.k ? 1 : 0;
  const int chunks = (n_heads / KV + AT_HEADS - 1) / AT_HEADS;
  const Shape s = shape_of(cache, n_heads, window, sinks);
  float* part = s.splits > 1 && !s.cluster ? (float*)workspace : nullptr;
  float2* stats = weights ? (float2*)((uint8_t*)workspace + sums_bytes(cache, n_heads, s)) : nullptr;
  float* scores = weights ? (float*)(stats + ((size_t)B * n_heads + 1) / 2 * 2) : nullptr;
  using Kernel = void (*)(const __half*, const cq_kv4, const NewRow, const long long*, __half*, float*, float2*, float*, int, int, int, int, float);
  auto pick = [&](auto width, auto groups) -> Kernel {
    constexpr int W = decltype(width)::value, N = decltype(groups)::value;
    auto sized = [&](auto w) -> Kernel {
      constexpr int C = decltype(w)::value;
      if (weights) return more ? kv4_attend_kernel<W, N, C, true, true> : kv4_attend_kernel<W, N, C, false, true>;
      return more ? kv4_attend_kernel<W, N, C, true, false> : kv4_attend_kernel<W, N, C, false, false>;
    };
    return s.warps == 16 ? sized(std::integral_constant<int, 16>()) : (s.warps == 8 ? sized(std::integral_constant<int, 8>()) : sized(std::integral_constant<int, 4>()));
  };
  using std::integral_constant;
  const Kernel fn = D == 128 ? (NG == 4 ? pick(integral_constant<int, 128>(), integral_constant<int, 4>()) : pick(integral_constant<int, 128>(), integral_constant<int, 2>()))
                             : (NG == 2 ? pick(integral_constant<int, 64>(), integral_constant<int, 2>()) : pick(integral_constant<int, 64>(), integral_constant<int, 1>()));
  const int smem = s.warps * AT_STAGES * AT_SLOTS * (D + 8 * NG);
  CQ_CUDA_TRY(cq_grant_smem((const void*)fn, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(s.splits, KV * chunks, B);
  cfg.blockDim = dim3(s.warps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = s.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = s.cluster ? 2 : 1;
  CQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, (const __half*)q, *cache, fresh, length, (__half*)out, scores, stats, part, n_heads, chunks, window, sinks,
                                 scale));
  if (part) {
    const long long heads = (long long)B * n_heads;
    CQ_CUDA_TRY(kv4_launch(D == 128 ? kv4_join_kernel<128> : kv4_join_kernel<64>, dim3((unsigned)((heads + 7) / 8)), dim3(AT_THREADS), 0, stream,
                           (const float*)part, s.splits, heads, (__half*)out, stats));
  }
  if (weights)
    CQ_CUDA_TRY(kv4_launch(kv4_weights_kernel, dim3((cache->slots + 4 * AT_THREADS - 1) / (4 * AT_THREADS), KV, B), dim3(AT_THREADS), 0, stream,
                           (const float*)scores, (const float2*)stats, length, more, weights, weights_out, n_heads, KV, cache->slots, window,
                           sinks));
  return CQ_OK;
}

int check(const cq_kv4* cache, const void* q, const long long* length, const void* out, int n_heads, int window, int sinks,
          const float* weights, const float* weights_out, const void* workspace) {
  const int rc = cq_kv4_check(cache);
  if (rc != CQ_OK) return rc;
  if (!q || !length || !out || window < 0 || sinks < 0 || (!weights != !weights_out)) return CQ_ERR_BAD_ARG;
  if (n_heads < 1 || n_heads % cache->n_kv_heads || (n_heads + 7ll * cache->n_kv_heads) / 8 > 65535) return CQ_ERR_BAD_SHAPE;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)weights | (uintptr_t)weights_out | (uintptr_t)workspace) & 15) return CQ_ERR_BAD_ARG;
  const size_t bytes = (size_t)cache->sequences * cache->n_kv_heads * cache->slots * 4;
  if (weights != weights_out && !kv4_apart(weights, bytes, weights_out, bytes)) return CQ_ERR_BAD_ARG;
  if (!workspace && cq_kv4_attend_workspace_bytes(cache, n_heads, window, sinks, weights != nullptr)) return CQ_ERR_BAD_ARG;
  return CQ_OK;
}

}  // namespace

extern "C" size_t cq_kv4_attend_workspace_bytes(const cq_kv4* cache, int n_heads, int window, int sinks, int with_weights) {
  if (cq_kv4_check(cache) != CQ_OK || n_heads < 1 || n_heads % cache->n_kv_heads || window < 0 || sinks < 0) return 0;
  const size_t heads = (size_t)cache->sequences * n_heads;
  return sums_bytes(cache, n_heads, shape_of(cache, n_heads, window, sinks)) + (with_weights ? heads * 8 + heads * cache->slots * 4 + 16 : 0);
}

extern "C" int cq_kv4_attend(const cq_kv4* cache, const void* q, const long long* length, void* out, int n_heads, int window, int sinks,
                             float scale, const float* weights, float* weights_out, void* workspace, cq_stream_t stream) {
  const int rc = check(cache, q, length, out, n_heads, window, sinks, weights, weights_out, workspace);
  if (rc != CQ_OK) return rc;
  return attend(cache, q, NewRow{}, length, out, n_heads, window, sinks, scale, weights, weights_out, workspace, (cudaStream_t)stream);
}

extern "C" int cq_kv4_step(const cq_kv4* cache, const void* q, const void* k, const void* v, const float* cos_table, const float* sin_table,
                           const long long* positions, int table_rows, const long long* length, void* out, int n_heads, int window,
                           int sinks, float scale, const float* weights, float* weights_out, void* workspace, cq_stream_t stream) {
  const int rc = check(cache, q, length, out, n_heads, window, sinks, weights, weights_out, workspace);
  if (rc != CQ_OK) return rc;
  if (!k || !v || (((uintptr_t)k | (uintptr_t)v) & 15)) return CQ_ERR_BAD_ARG;
  if (cos_table && (!sin_table || !positions || table_rows < 1)) return CQ_ERR_BAD_ARG;
  const NewRow fresh = {(const __half*)k, (const __half*)v, cos_table, sin_table, positions, table_rows};
  return attend(cache, q, fresh, length, out, n_heads, window, sinks, scale, weights, weights_out, workspace, (cudaStream_t)stream);
}
