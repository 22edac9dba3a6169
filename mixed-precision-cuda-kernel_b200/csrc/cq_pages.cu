// Writing rows into the paged KV cache and reading them back (layout: cq_pages.cuh; attention over it: cq_pages_attn.cu).  In the
// reference the cache is the fp16 key and value tensors of its vendored LLaMA (llama/modeling_llama_quant.py:371-419 of the
// reference project).
#include "cq_pages.cuh"

namespace cq_paged {

int check(const cq_pages* p, const cq_table* t) {
  const int rc = cq_pages_check(p);
  if (rc != CQ_OK) return rc;
  if (!t || !t->entries || ((uintptr_t)t->entries & 3) || t->stride < 0) return CQ_ERR_BAD_ARG;
  if (t->sequences < 1 || t->sequences > 65535 || t->width < 1 || (long long)t->width * p->page_size > (1 << 30)) return CQ_ERR_BAD_SHAPE;
  return CQ_OK;
}

}  // namespace cq_paged

namespace {

using namespace cq_paged;

constexpr int THREADS = 256, TOKENS = 2, SLOTS = 2;

// The sequence of packed row t: the last one that starts at or before it, -1 in front of the first and behind the last.
__device__ __forceinline__ int sequence_of(const long long* __restrict__ starts, int sequences, long long t) {
  if (t < starts[0] || t >= starts[sequences]) return -1;
  int low = 0, high = sequences;                           // starts[low] <= t < starts[high]
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (starts[mid] <= t) low = mid;
    else high = mid;
  }
  return low;
}

// D / 16 lanes a row of q, k or v, eight columns of each half of the head a lane: q and k rotated, q to q_out, k and v to their
// slots.  The bound is memory: a block takes 16 or 32 heads of two tokens, whose angles, positions and slots it reads once, and writes
// beside one another what lies so (2048 tokens of 40 heads 21 us, 5.9 TB/s; with a block for the rows of one head, which reads
// 512 bytes of angles for 256 of a row, 32; one token 21, four 22, sixteen 25).
template <typename T, int D>
__global__ void __launch_bounds__(THREADS) pages_write_kernel(const Rows<T> q, T* __restrict__ q_out, const Rows<T> k, const Rows<T> v,
                                                              const float* __restrict__ cos_t, const float* __restrict__ sin_t,
                                                              const long long* __restrict__ positions, int table_rows,
                                                              const long long* __restrict__ first, const long long* __restrict__ starts, const Pool<T> pool,
                                                              const Table table, int sequences, int rows, int H) {
  constexpr int LANES = D / 16, HEADS = THREADS / LANES / TOKENS;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int r = threadIdx.x / LANES, j = blockIdx.y * HEADS + r % HEADS, KV = pool.heads, c = 8 * (threadIdx.x % LANES);
  const long long t = (long long)blockIdx.x * TOKENS + r / HEADS;
  if (t >= rows || j >= H + 2 * KV) return;
  const bool is_q = j < H, is_k = !is_q && j < H + KV;
  const int head = is_q ? j : (is_k ? j - H : j - H - KV);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const T* src = (is_q ? q : (is_k ? k : v)).row(t, head) + c;
  uint4 x1 = *reinterpret_cast<const uint4*>(src), x2 = *reinterpret_cast<const uint4*>(src + D / 2);
  const long long pos = cos_t ? positions[t] : 0;
  const bool turn = cos_t && pos >= 0 && pos < table_rows;
  T* to = nullptr;
  if (is_q) {
    to = q_out + (t * H + head) * D + c;
  } else if (!cos_t || turn) {               // (a key without a position in the tables is left out, and its value with it)
    const int each = rows / sequences, s = starts ? sequence_of(starts, sequences, t) : (int)(t / each);
    if (s >= 0) {
      const long long slot = first[s] + t - (starts ? starts[s] : (long long)s * each);
      const int page = slot < 0 ? -1 : table.page_of(pool, s, slot);
      if (page >= 0) to = (is_k ? pool.k : pool.v) + (pool.rows(page, head) + (slot & ((1 << pool.log_page) - 1))) * D + c;
    }
  }
  if (turn && (is_q || is_k)) rotate8<T>(x1, x2, cos_t + pos * (D / 2) + c, sin_t + pos * (D / 2) + c);
  if (!to) return;
  *reinterpret_cast<uint4*>(to) = x1;
  *reinterpret_cast<uint4*>(to + D / 2) = x2;
}

// D / 8 lanes a row, 16 bytes of its key and of its value each: k and v (sequence, count, KV, D).  Slots without a page read as zeros.
// A block takes the heads of two slots, whose rows lie one behind the other where they are written (5 x 2001 slots of 40 heads 64 us,
// 6.4 TB/s; a head's slots, one behind the other where they are read, 70).
template <typename T, int D>
__global__ void __launch_bounds__(THREADS) pages_read_kernel(const Pool<T> pool, const Table table, const long long* __restrict__ first, int count,
                                                             T* __restrict__ k, T* __restrict__ v) {
  constexpr int LANES = D / 8, HEADS = THREADS / LANES / SLOTS;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int s = blockIdx.z, r = threadIdx.x / LANES, head = blockIdx.y * HEADS + r % HEADS, c = 8 * (threadIdx.x % LANES);
  const long long i = (long long)blockIdx.x * SLOTS + r / HEADS;
  if (i >= count || head >= pool.heads) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long slot = first[s] + i;
  const int page = slot < 0 ? -1 : table.page_of(pool, s, slot);
  uint4 x = make_uint4(0, 0, 0, 0), y = x;
  if (page >= 0) {
    const size_t at = (pool.rows(page, head) + (slot & ((1 << pool.log_page) - 1))) * D + c;
    x = *reinterpret_cast<const uint4*>(pool.k + at);
    y = *reinterpret_cast<const uint4*>(pool.v + at);
  }
  const size_t to = (((size_t)s * count + i) * pool.heads + head) * D + c;
  *reinterpret_cast<uint4*>(k + to) = x;
  *reinterpret_cast<uint4*>(v + to) = y;
}

template <typename T, int D>
int write(const cq_pages* pages, const cq_table* table, const cq_rows* q, void* q_out, const cq_rows* k, const cq_rows* v, const float* cos_t,
          const float* sin_t, const long long* positions, int table_rows, const long long* first, const long long* starts, int rows, int H,
          cudaStream_t stream) {
  constexpr int HEADS = THREADS / (D / 16) / TOKENS;
  CQ_CUDA_TRY(kv4_launch(pages_write_kernel<T, D>, dim3((rows - 1) / TOKENS + 1, (H + 2 * pages->n_kv_heads + HEADS - 1) / HEADS), dim3(THREADS), 0, stream,
                         rows_of<T>(H ? q : nullptr), (T*)q_out, rows_of<T>(k), rows_of<T>(v), cos_t, sin_t, positions, table_rows, first, starts,
                         pool_of<T>(pages), table_of(table), table->sequences, rows, H));
  return CQ_OK;
}
template <typename T, int D>
int read(const cq_pages* pages, const cq_table* table, const long long* first, int count, void* k, void* v, cudaStream_t stream) {
  constexpr int HEADS = THREADS / (D / 8) / SLOTS;
  CQ_CUDA_TRY(kv4_launch(pages_read_kernel<T, D>, dim3((count - 1) / SLOTS + 1, (pages->n_kv_heads + HEADS - 1) / HEADS, table->sequences), dim3(THREADS), 0, stream,
                         pool_of<T>(pages), table_of(table), first, count, (T*)k, (T*)v));
  return CQ_OK;
}

}  // namespace

extern "C" int cq_pages_check(const cq_pages* p) {
  if (!p || !p->k || !p->v || (((uintptr_t)p->k | (uintptr_t)p->v) & 31)) return CQ_ERR_BAD_ARG;
  if (p->pages < 1 || p->n_kv_heads < 1 || p->n_kv_heads > 16383 || p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
    return CQ_ERR_BAD_SHAPE;
  if ((p->head_dim != 64 && p->head_dim != 128) || (p->dtype != 0 && p->dtype != 2)) return CQ_ERR_UNSUPPORTED;
  const size_t bytes = (size_t)p->pages * p->n_kv_heads * p->page_size * p->head_dim * 2;
  return kv4_apart(p->k, bytes, p->v, bytes) ? CQ_OK : CQ_ERR_BAD_ARG;
}

extern "C" int cq_pages_write(const cq_pages* pages, const cq_table* table, const cq_rows* q, void* q_out, const cq_rows* k, const cq_rows* v,
                              const float* cos_table, const float* sin_table, const long long* positions, int table_rows,
                              const long long* first, const long long* starts, int rows, int n_heads, cq_stream_t stream) {
  const int rc = check(pages, table);
  if (rc != CQ_OK) return rc;
  if (!rows_fit(k) || !rows_fit(v) || !first || rows < 1 || n_heads < 0 || (n_heads > 0 && (!rows_fit(q) || !q_out || ((uintptr_t)q_out & 15))))
    return CQ_ERR_BAD_ARG;
  if (!tables_fit(cos_table, sin_table, positions, table_rows) || (((uintptr_t)first | (uintptr_t)starts) & 7)) return CQ_ERR_BAD_ARG;
  if (n_heads + 2ll * pages->n_kv_heads > 65535 || (!starts && rows % table->sequences)) return CQ_ERR_BAD_SHAPE;
  auto fn = pages->dtype == 0 ? (pages->head_dim == 128 ? write<__half, 128> : write<__half, 64>)
                              : (pages->head_dim == 128 ? write<__nv_bfloat16, 128> : write<__nv_bfloat16, 64>);
  return fn(pages, table, q, q_out, k, v, cos_table, sin_table, positions, table_rows, first, starts, rows, n_heads, (cudaStream_t)stream);
}

extern "C" int cq_pages_read(const cq_pages* pages, const cq_table* table, const long long* first, int count, void* k, void* v, cq_stream_t stream) {
  const int rc = check(pages, table);
  if (rc != CQ_OK) return rc;
  if (!first || ((uintptr_t)first & 7) || !k || !v || count < 1 || (((uintptr_t)k | (uintptr_t)v) & 15)) return CQ_ERR_BAD_ARG;
  auto fn = pages->dtype == 0 ? (pages->head_dim == 128 ? read<__half, 128> : read<__half, 64>)
                              : (pages->head_dim == 128 ? read<__nv_bfloat16, 128> : read<__nv_bfloat16, 64>);
  return fn(pages, table, first, count, k, v, (cudaStream_t)stream);
}
