// Logits on their way to a token: penalties for tokens that occurred, biases of single tokens, a grammar's bit mask, and the largest.
//
// The bound is the logits' traffic, each read once and written once; penalties are the business of few tokens and are settled token by
// token, beside it.  The tokens that occurred or have a bias are marked in a bit map, occurrences are counted in shared memory (integer
// additions: their order changes nothing): in a place for every token where a CTA's part of the vocabulary is small, else in
// the marked tokens' places, a token's rank among them.  The pass over the logits leaves the marked ones out of the maximum;
// their values are written over its results.  (256 rows of 131071 bf16 logits, histories of 1500 and masks: 31 us; penalties in the pass take 57
// instructions a logit, 138 us; counters for all tokens, a slice of the vocabulary after the other, 87.  A row of 32000
// with a history of 300 4.7 us, without 3.4.)  Every thread has four pieces of 16 bytes on the way, copied asynchronously to places of its
// own, and waits for no other thread; what no mask changes is neither converted nor rounded.  Of eight logits only the largest
// meets the thread's best.  The largest travels as one 64-bit key, its value in the order of unsigned numbers above the
// complement of its token: the maximum of keys is the lowest token of the largest value.
#include <algorithm>
#include <type_traits>

#include "cq_pages.cuh"

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int STAGES = 4;                    // pieces of 16 bytes of a thread on their way
constexpr int PARTS = 8;                     // CTAs of a row, at most
constexpr int TOKENS = 4 * THREADS;          // of the history, loads in flight
constexpr int SLICE = 129 * 1024;            // tokens that the bit map holds
constexpr int PLACES = STAGES * THREADS * 16 / 12;          // marked tokens at a time, in the pieces' memory
// what is known of a token: whether it occurred in the prompt, whether it has a bias, and below how often it was generated
constexpr uint32_t PROMPT = 0x80000000u, BIAS = 0x40000000u, TIMES = 0x3FFFFFFFu;

struct Adjust {
  cq_adjust a;
  int vocab, part, slice;                    // logits of a row, of a CTA, and of the bit map
  int keep;                                  // tokens of the history in shared memory
  bool alike;                                // results lie as the logits do, by 16 bytes
};

template <typename T> __device__ __forceinline__ float value_of(T x) { return cq_paged::Type<T>::one(x); }
template <> __device__ __forceinline__ float value_of(float x) { return x; }
template <typename T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ __half rounded(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ float rounded(float x) { return x; }

// 16 bytes of logits.  largest(): NaN where one is; hide(): -infinity in the places whose bits are set, `lut` the 16-bit lanes of four bits
template <typename T> struct Piece {
  uint4 w;
  using Two = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  __device__ __forceinline__ float largest() const {
    const Two* t = reinterpret_cast<const Two*>(&w);
    const Two m = __hmax2_nan(__hmax2_nan(t[0], t[1]), __hmax2_nan(t[2], t[3]));
    const float2 f = cq_paged::Type<T>::apart(*reinterpret_cast<const uint32_t*>(&m));
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(f.x), "f"(f.y));
    return d;
  }
  __device__ __forceinline__ void hide(uint32_t bits, const uint2* lut) {
    constexpr uint32_t NONE = std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
    const uint2 a = lut[bits & 15u], b = lut[bits >> 4];
    w.x = (w.x & ~a.x) | (NONE & a.x), w.y = (w.y & ~a.y) | (NONE & a.y);
    w.z = (w.z & ~b.x) | (NONE & b.x), w.w = (w.w & ~b.y) | (NONE & b.y);
  }
  __device__ __forceinline__ T at(int e) const { return reinterpret_cast<const T*>(&w)[e]; }
};
template <> struct Piece<float> {
  uint4 w;
  __device__ __forceinline__ float largest() const {
    float d;
    asm("{\n\t.reg .f32 a, b;\n\tmax.NaN.f32 a, %1, %2;\n\tmax.NaN.f32 b, %3, %4;\n\tmax.NaN.f32 %0, a, b;\n\t}"
        : "=f"(d) : "f"(__uint_as_float(w.x)), "f"(__uint_as_float(w.y)), "f"(__uint_as_float(w.z)), "f"(__uint_as_float(w.w)));
    return d;
  }
  __device__ __forceinline__ void hide(uint32_t bits, const uint2*) {
    constexpr uint32_t NONE = 0xFF800000u;
    w.x = bits & 1u ? NONE : w.x, w.y = bits & 2u ? NONE : w.y, w.z = bits & 4u ? NONE : w.z, w.w = bits & 8u ? NONE : w.w;
  }
  __device__ __forceinline__ float at(int e) const { return reinterpret_cast<const float*>(&w)[e]; }
};

// fp32 numbers in the order of unsigned ones: NaN above all, both zeros alike
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long larger(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

template <int BYTES> __device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(BYTES) : "memory");
}

// the largest key of a warp's lanes
__device__ __forceinline__ unsigned long long largest_of_warp(unsigned long long key) {
  const uint32_t high = (uint32_t)(key >> 32), top = __reduce_max_sync(0xffffffffu, high);
  return (unsigned long long)top << 32 | __reduce_max_sync(0xffffffffu, high == top ? (uint32_t)key : 0u);
}

template <typename T, bool DIRECT>
__global__ void __launch_bounds__(THREADS, 2) adjust_logits_kernel(const Adjust p) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ unsigned long long s_key[THREADS / 32];
  __shared__ unsigned long long s_part[PARTS];
  __shared__ int s_sum[WARPS], s_count;
  __shared__ uint2 s_lut[16];                // what four bits are in 16-bit lanes
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const cq_adjust& a = p.a;
  const int parts = gridDim.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (parts > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // (this CTA runs: its memory may be written)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tid < 16) s_lut[tid] = make_uint2((tid & 1 ? 0xFFFFu : 0u) | (tid & 2 ? 0xFFFF0000u : 0u), (tid & 4 ? 0xFFFFu : 0u) | (tid & 8 ? 0xFFFF0000u : 0u));
  const bool counts = a.tokens != nullptr, known = counts || a.biases;
  uint4* s_piece = reinterpret_cast<uint4*>(smem) + tid;                     // [stage][thread]
  uint32_t* s_mask = reinterpret_cast<uint32_t*>(smem + 16 * STAGES * THREADS);             // numbered as the marks
  uint64_t* s_bits = reinterpret_cast<uint64_t*>(smem + 16 * STAGES * THREADS + (a.mask ? p.slice / 8 + 16 : 0));
  int* s_rank = reinterpret_cast<int*>(s_bits + p.slice / 64);               // of a word's first marked token
  int* s_history = s_rank + p.slice / 64;                                    // -1 outside the vocabulary
  // [place], DIRECT: a place for every token, otherwise after the pieces and in their memory
  uint32_t* s_known = DIRECT ? reinterpret_cast<uint32_t*>(s_bits) + p.slice / 32 : reinterpret_cast<uint32_t*>(smem);
  uint32_t* s_token = s_known + PLACES;                                      // (not DIRECT)
  uint32_t* s_bias = DIRECT ? s_known + p.slice : s_token + PLACES;          // 1 + the entry that counts
  uint16_t* s_list = reinterpret_cast<uint16_t*>(s_known + (a.biases ? 2 : 1) * p.slice);   // DIRECT: the marked tokens, in any order
  const T* in = (const T*)a.logits + (int64_t)row * a.logits_stride;
  T* out = (T*)a.out + (int64_t)row * a.out_stride;
  // Logits are numbered from the 16-byte boundary in front of the row's first, so that pieces are aligned.  (Where results lie otherwise,
  // they are written one by one.)
  const int skip = (int)(((uintptr_t)in / sizeof(T)) % VEC);
  in -= skip;
  out -= skip;
  const int total = p.vocab + skip, begin = min(total, (int)blockIdx.x * p.part), end = min(total, begin + p.part);
  auto whole = [&](int i) { return (unsigned)(i - skip) <= (unsigned)(p.vocab - VEC) && p.vocab >= VEC; };
  auto fetch = [&](int i, int stage) {
    if (whole(i)) {
      copy_async<16>(s_piece + stage * THREADS, in + i);
    } else {
      T* w = reinterpret_cast<T*>(s_piece + stage * THREADS);
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = i + e >= skip && i + e < total ? in[i + e] : T(-INFINITY);
    }
  };
  constexpr int STEP = THREADS * VEC;
  auto first_pieces = [&](int base, int stop) {
#pragma unroll
    for (int k = 0; k < STAGES; ++k) {
      if (base + k * STEP + tid * VEC < stop) fetch(base + k * STEP + tid * VEC, k);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  const long long* tokens = counts ? a.tokens + (int64_t)row * a.tokens_stride : nullptr;
  const long long* ids = a.biases ? a.bias_ids + (int64_t)row * a.bias_ids_stride : nullptr;
  auto token_of = [&](long long v) { return (unsigned long long)v < (unsigned)p.vocab ? (int)v : -1; };
  // all that the row says in one round of loads
  long long v0[TOKENS / THREADS] = {}, n64 = a.width, prompt64 = 0, mask_row = row;
  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (counts) {
#pragma unroll
    for (int k = 0; k < TOKENS / THREADS; ++k) v0[k] = tid + k * THREADS < a.width ? tokens[tid + k * THREADS] : -1;
    if (a.length) n64 = a.length[row];
    if (a.prompt) prompt64 = a.prompt[row];
    if (a.repetition) rep = a.repetition[row];
    if (a.presence) pres = a.presence[row];
    if (a.frequency) freq = a.frequency[row];
  }
  if (a.mask && a.mask_rows) mask_row = a.mask_rows[row];
  first_pieces(begin, min(end, begin + p.slice));
  const uint32_t* mask = a.mask && mask_row >= 0 && mask_row < a.masks ? a.mask + mask_row * a.mask_stride : nullptr;
  const int n = !counts || n64 < 0 ? 0 : (int)(n64 > a.width ? a.width : n64), prompt = (int)(prompt64 < 0 ? 0 : (prompt64 > n ? n : prompt64));

  float top = -INFINITY;                     // the thread's largest, the piece that has it and where that begins
  Piece<T> of_top = {};
  int at_top = -1;
  unsigned long long best = 0;
  auto key_of = [&](float x, int v) { return (unsigned long long)order_of(x) << 32 | (0xFFFFFFFFu - (uint32_t)v); };
#pragma unroll 1
  for (int base = begin; base < end; base += p.slice) {
    const int stop = min(end, base + p.slice), size = stop - base, words = (size + 63) / 64;
    if (base != begin) first_pieces(base, stop);
    if (known) {
      for (int i = tid; i < (size + 31) / 32; i += THREADS) reinterpret_cast<uint32_t*>(s_bits)[i] = 0u;
      if (!DIRECT && tid == 0 && (size + 31) / 32 % 2) reinterpret_cast<uint32_t*>(s_bits)[(size + 31) / 32] = 0u;      // (the last word's other half)
      if (DIRECT)
        for (int i = tid; i < size; i += THREADS) {
          s_known[i] = 0u;
          if (a.biases) s_bias[i] = 0u;
        }
      if (DIRECT && tid == 0) s_count = 0;
      __syncthreads();
    }
    // the place of a token in the slice, -1 outside
    auto place = [&](int v) {
      const int j = v < 0 ? -1 : v + skip - base;
      return j < size ? j : -1;
    };
    // what(place, number) of the history's tokens, and of those with a bias
    auto each_token = [&](auto find, auto what) {
#pragma unroll 1
      for (int j0 = tid; j0 < n; j0 += 4 * THREADS) {
        int at[4], i[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = j0 + k * THREADS;
          at[k] = j < n ? place(j < p.keep ? s_history[j] : token_of(tokens[j])) : -1;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) i[k] = find(at[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i[k] >= 0) what(i[k], at[k], j0 + k * THREADS);
      }
    };
    auto each_bias = [&](auto find, auto what) {
#pragma unroll 1
      for (int j = tid; j < a.biases; j += THREADS) {
        const int at = place(token_of(ids[j])), i = find(at);
        if (i >= 0) what(i, at, j);
      }
    };
    // what is known of the token in place i
    auto occurred = [&](int i, int j) {
      if (j < prompt) atomicOr(&s_known[i], PROMPT);
      else atomicAdd(&s_known[i], 1u);
    };
    auto biased = [&](int i, int j) {        // of the same token's entries the last one counts
      atomicOr(&s_known[i], BIAS);
      atomicMax(&s_bias[i], (uint32_t)j + 1u);
    };
    if (known) {
      uint32_t* bits = reinterpret_cast<uint32_t*>(s_bits);
      // Tokens at `at` (-1: none) of a lane, K at a time.  DIRECT: first(k) is whether that is the first that is known of the token, which then
      // goes on the list; a warp takes the list's next places for all of its lanes.
      auto note = [&](auto size, const int* at, auto first) {
        constexpr int K = decltype(size)::value;
        if constexpr (DIRECT) {
          uint32_t fresh[K];
          int all = 0;
#pragma unroll
          for (int k = 0; k < K; ++k) {
            fresh[k] = __ballot_sync(0xffffffffu, first(k));
            all += __popc(fresh[k]);
          }
          if (!all) return;
          int to = 0;
          if (lane == 0) to = atomicAdd(&s_count, all);
          to = __shfl_sync(0xffffffffu, to, 0);
#pragma unroll
          for (int k = 0; k < K; ++k) {
            if (fresh[k] >> lane & 1u) {
              s_list[to + __popc(fresh[k] & ((1u << lane) - 1u))] = (uint16_t)at[k];
              atomicOr(&bits[at[k] >> 5], 1u << (at[k] & 31));
            }
            to += __popc(fresh[k]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < K; ++k)
            if (at[k] >= 0 && !(*(volatile uint32_t*)&bits[at[k] >> 5] >> (at[k] & 31) & 1u)) atomicOr(&bits[at[k] >> 5], 1u << (at[k] & 31));
        }
      };
      using std::integral_constant;
      constexpr int K = TOKENS / THREADS;
      if (counts && (DIRECT || base == begin)) {
#pragma unroll 1
        for (int j0 = tid; j0 - tid < n; j0 += TOKENS) {
          int at[K];
          uint32_t old[K];
#pragma unroll
          for (int k = 0; k < K; ++k) {
            const int j = j0 + k * THREADS, v = token_of(v0[k]);
            at[k] = j < n ? place(v) : -1;
            if (!DIRECT && j < p.keep) s_history[j] = v;
          }
          // (the next ones are on their way meanwhile)
#pragma unroll
          for (int k = 0; k < K; ++k) v0[k] = j0 + TOKENS + k * THREADS < n ? tokens[j0 + TOKENS + k * THREADS] : -1;
          if (DIRECT)
#pragma unroll
            for (int k = 0; k < K; ++k) {
              old[k] = 1u;
              if (at[k] >= 0) old[k] = j0 + k * THREADS < prompt ? atomicOr(&s_known[at[k]], PROMPT) : atomicAdd(&s_known[at[k]], 1u);
            }
          note(integral_constant<int, K>(), at, [&](int k) { return old[k] == 0u; });
        }
      } else if (counts) {
#pragma unroll 1
        for (int j = tid; j < n; j += THREADS) {
          const int at = place(j < p.keep ? s_history[j] : token_of(tokens[j]));
          note(integral_constant<int, 1>(), &at, [](int) { return false; });
        }
      }
#pragma unroll 1
      for (int j0 = 0; j0 < a.biases; j0 += THREADS) {     // of the same token's entries the last one counts
        const int j = j0 + tid, at = j < a.biases ? place(token_of(ids[j])) : -1;
        uint32_t old = 1u;
        if (DIRECT && at >= 0) {
          old = atomicOr(&s_known[at], BIAS);
          atomicMax(&s_bias[at], (uint32_t)j + 1u);
        }
        note(integral_constant<int, 1>(), &at, [&](int) { return old == 0u; });
      }
    }
    // The mask's words, moved to where the marks of the same tokens are
    if (mask)
#pragma unroll 4
      for (int i = tid; i < (size + 31) / 32; i += THREADS) {
        const int v = base + 32 * i - skip, w = v >> 5;
        const uint32_t low = w >= 0 ? __ldg(mask + w) : 0u, high = 32 * (w + 1) < p.vocab ? __ldg(mask + w + 1) : 0u;
        s_mask[i] = __funnelshift_r(low, high, v & 31);
      }
    if (mask || known) __syncthreads();      // (the mask's words and the marks are there)
    // what is known of the marked tokens with ranks from rank0 on
    auto count = [&](int rank0, int here) {
      for (int i = tid; i < here; i += THREADS) {
        s_known[i] = 0u;
        if (a.biases) s_bias[i] = 0u;
      }
      __syncthreads();
      auto index = [&](int at) {             // -1: outside, or has its turn earlier or later
        const int w = max(at, 0) >> 6, i = s_rank[w] + __popcll(s_bits[w] & ((1ull << (at & 63)) - 1ull)) - rank0;
        return at >= 0 && i >= 0 && i < here ? i : -1;
      };
      if (counts)
        each_token(index, [&](int i, int at, int j) {
          s_token[i] = at;
          occurred(i, j);
        });
      each_bias(index, [&](int i, int at, int j) {
        s_token[i] = at;
        biased(i, j);
      });
      __syncthreads();
    };
    // (of a masked token the pass over the logits may have left -infinity in place of the logit, which changes nothing)
    auto put = [&](int i, int j) {
      const uint32_t c = s_known[i];
      const int at = base + j;
      float x = value_of<T>(DIRECT && size <= STAGES * STEP ? reinterpret_cast<const T*>(smem)[j] : in[at]);       // (a small slice's pieces are all there yet)
      if (a.repetition && (c & (PROMPT | TIMES))) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      if (c & TIMES) {
        if (a.frequency) x = __fsub_rn(x, __fmul_rn(freq, (float)(c & TIMES)));
        if (a.presence) x = __fsub_rn(x, pres);
      }
      if (c & BIAS) x = __fadd_rn(x, a.bias[(int64_t)row * a.bias_stride + s_bias[i] - 1u]);
      if (mask && !(s_mask[j >> 5] >> (j & 31) & 1u)) x = -INFINITY;
      out[at] = rounded<T>(x);
      best = larger(best, key_of(x, at - skip));
    };

    for (int i0 = base + tid * VEC; i0 < stop; i0 += STAGES * STEP) {
#pragma unroll
      for (int k = 0; k < STAGES; ++k) {
        const int i = i0 + k * STEP, j = i - base;
        if (i >= stop) break;
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        Piece<T> piece;
        piece.w = s_piece[k * THREADS];
        if (i + STAGES * STEP < stop) fetch(i + STAGES * STEP, k);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (mask) {
          const uint32_t hidden = ~(s_mask[j >> 5] >> (j & 31)) & ((1u << VEC) - 1u);
          if (hidden) piece.hide(hidden, s_lut);
        }
        if (p.alike && whole(i)) *reinterpret_cast<uint4*>(out + i) = piece.w;
        else
          for (int e = 0; e < VEC; ++e)
            if (i + e >= skip && i + e < total) out[i + e] = piece.at(e);
        if (known) {
          const uint32_t own = reinterpret_cast<const uint32_t*>(s_bits)[j >> 5] >> (j & 31) & ((1u << VEC) - 1u);
          if (own) piece.hide(own, s_lut);
        }
        const float m = piece.largest();
        if (at_top < 0 || (!(m <= top) && top == top)) {
          top = m;
          at_top = i;
          of_top = piece;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (known && DIRECT) {
      __syncthreads();                       // (results of the pass lie under those of the marked tokens)
      for (int i = tid; i < s_count; i += THREADS) put(s_list[i], s_list[i]);
    } else if (known) {
      // ranks: a thread takes consecutive words
      const int each = (words + THREADS - 1) / THREADS, w0 = min(words, tid * each), w1 = min(words, w0 + each);
      int mine = 0;
      for (int w = w0; w < w1; ++w) mine += __popcll(s_bits[w]);
      int before = mine;
      for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += o;
      }
      if (lane == 31) s_sum[warp] = before;
      __syncthreads();
      int all = lane < WARPS ? s_sum[lane] : 0;
      for (int d = 1; d < WARPS; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, all, d);
        if (lane >= d) all += o;
      }
      const int marked = __shfl_sync(0xffffffffu, all, WARPS - 1);
      const int in_front = __shfl_sync(0xffffffffu, all, max(0, warp - 1));
      before += (warp ? in_front : 0) - mine;
      for (int w = w0; w < w1; ++w) {
        s_rank[w] = before;
        before += __popcll(s_bits[w]);
      }
      __syncthreads();                       // (results of the pass lie under those of the marked tokens; the pieces' memory is free)
      for (int rank0 = 0; rank0 < marked; rank0 += PLACES) {
        const int here = min(PLACES, marked - rank0);
        if (rank0) __syncthreads();
        count(rank0, here);
        for (int i = tid; i < here; i += THREADS) put(i, s_token[i]);
      }
    }
    if (stop < end) __syncthreads();         // (the next slice takes the same memory)
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    if (at_top >= 0 && at_top + e >= skip && at_top + e < total) best = larger(best, key_of(value_of<T>(of_top.at(e)), at_top + e - skip));
  best = largest_of_warp(best);
  if (lane == 0) s_key[warp] = best;
  __syncthreads();
  if (warp == 0) {
    best = largest_of_warp(lane < THREADS / 32 ? s_key[lane] : 0ull);
  }
  if (parts > 1) {                           // to the cluster's first CTA
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid == 0) {
      uint32_t at;
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(&s_part[blockIdx.x])));
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(best) : "memory");
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (blockIdx.x) return;
    if (tid == 0)
      for (int i = 1; i < parts; ++i) best = larger(best, s_part[i]);
  }
  if (tid == 0) a.next[row] = (long long)(0xFFFFFFFFu - (uint32_t)best);
}

// bytes from the first to behind the last element of `rows` rows of `cols`
size_t span(int64_t rows, int64_t cols, int64_t stride, size_t item) { return (size_t)((rows - 1) * stride + cols) * item; }

}  // namespace

extern "C" int cq_adjust_logits(const cq_adjust* a, int rows, int vocab, cq_stream_t stream) {
  if (!a || !a->logits || !a->out || !a->next) return CQ_ERR_BAD_ARG;
  // (indices, and their steps behind the last entry, in 32 bits)
  if (rows < 1 || rows > 65535 || vocab < 1 || vocab > (1 << 30) || a->width >= (1 << 30) || a->biases >= (1 << 30)) return CQ_ERR_BAD_SHAPE;
  if (a->dtype < 0 || a->dtype > 2) return CQ_ERR_UNSUPPORTED;
  const size_t item = a->dtype == 1 ? 4 : 2;
  if (((uintptr_t)a->logits | (uintptr_t)a->out) & (item - 1)) return CQ_ERR_BAD_ARG;
  if (a->logits_stride < 0 || (rows > 1 && a->out_stride < vocab)) return CQ_ERR_BAD_ARG;
  if (a->tokens ? a->width < 0 || a->tokens_stride < 0 : (a->length || a->prompt || a->repetition || a->presence || a->frequency)) return CQ_ERR_BAD_ARG;
  if (a->biases < 0 || (a->biases > 0 && (!a->bias_ids || !a->bias || a->bias_ids_stride < 0 || a->bias_stride < 0))) return CQ_ERR_BAD_ARG;
  if (a->mask ? a->masks < 1 || a->mask_stride < 0 || (!a->mask_rows && a->masks < rows) : a->mask_rows != nullptr) return CQ_ERR_BAD_ARG;
  if (((uintptr_t)a->tokens | (uintptr_t)a->length | (uintptr_t)a->prompt | (uintptr_t)a->bias_ids | (uintptr_t)a->mask_rows | (uintptr_t)a->next) & 7)
    return CQ_ERR_BAD_ARG;
  if (((uintptr_t)a->repetition | (uintptr_t)a->presence | (uintptr_t)a->frequency | (uintptr_t)a->bias | (uintptr_t)a->mask) & 3) return CQ_ERR_BAD_ARG;
  // in place, or apart
  const bool in_place = a->logits == a->out && (rows == 1 || a->logits_stride == a->out_stride);
  if (!in_place && !kv4_apart(a->logits, span(rows, vocab, a->logits_stride, item), a->out, span(rows, vocab, a->out_stride, item))) return CQ_ERR_BAD_ARG;
  const int sms = cq_sm_count(), vec = 16 / (int)item;
  const bool known = a->tokens || a->biases;
  auto part_of = [&](int parts) { return ((vocab + vec - 1 + parts - 1) / parts + vec - 1) / vec * vec; };
  // bytes of a CTA with a place for every token of its part (64 bits: a part may be the whole vocabulary)
  auto places = [&](int parts) {
    const int64_t slice = (part_of(parts) + 31) / 32 * 32;
    return STAGES * THREADS * 16 + (a->mask ? slice / 8 + 16 : 0) + slice / 8 + slice * (a->biases ? 10 : 6);
  };
  // Two CTAs on an SM, or one where few run.  A place for every token, where there is room (a row of 128256 logits with a history of 8000 10.9 us,
  // with ranks 13.1); for that also half the CTAs, which then see a history half as often (64 rows of 50257 logits 7.2 us, so 8.0; 100 of
  // 25000 7.2, so 8.4).  More CTAs than fill the device lose (128 rows of 32000 14.0 against 9.9).
  constexpr int HALF = 112 * 1024 + 512, WHOLE = 225 * 1024;
  int parts = 1;
  while (parts < PARTS && rows * parts < sms && vocab > parts * 1024) parts *= 2;
  int room = rows * parts <= sms / 2 ? WHOLE : HALF;
  if (known && (parts == 2 || parts == 4) && rows * parts / 2 <= sms && places(parts / 2) <= WHOLE) parts /= 2, room = WHOLE;
  const bool direct = known && places(parts) <= room;
  const int part = part_of(parts), slice = direct ? (part + 31) / 32 * 32 : std::min((part + 63) / 64 * 64, SLICE);
  const int ring = STAGES * THREADS * 16 + (a->mask ? slice / 8 + 16 : 0), fixed = !known ? ring : (direct ? (int)places(parts) : ring + slice / 64 * 12);
  const int keep = a->tokens && !direct ? (int)std::min<int64_t>(a->width, (112 * 1024 - fixed) / 4) : 0, smem = fixed + 4 * keep;
  const bool alike = (((uintptr_t)a->logits ^ (uintptr_t)a->out) & 15) == 0 && (rows == 1 || (a->logits_stride - a->out_stride) % vec == 0);
  auto fn = a->dtype == 0   ? (direct ? adjust_logits_kernel<__half, true> : adjust_logits_kernel<__half, false>)
            : a->dtype == 1 ? (direct ? adjust_logits_kernel<float, true> : adjust_logits_kernel<float, false>)
                            : (direct ? adjust_logits_kernel<__nv_bfloat16, true> : adjust_logits_kernel<__nv_bfloat16, false>);
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
  cfg.numAttrs = parts > 1 ? 2 : 1;
  CQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, Adjust{*a, vocab, part, slice, keep, alike}));
  return CQ_OK;
}
