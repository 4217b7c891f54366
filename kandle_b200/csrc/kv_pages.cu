// Pages of a cache: copies to other places (kd_kv_pages_copy) and beams that take over their parents' pages (kd_kv_pages_fork).
//
// A pool is [pages,Hkv,128,D] with rows of a head side by side; a call works on all pools of a model at once (keys and values of every
// layer), whose addresses travel in the launch's parameters.  Bound: HBM, every moved byte read and written once: 300 pages of 18 pools (2.8 GB moved) 428 us, 6.6
// TB/s; 16 requests of 8 beams at 1000 positions 80 us, 6.1 TB/s.  Two pages 14 us, four beams 15 us: the launches.
#include "common.cuh"
#include "kernels.cuh"

namespace kd {

constexpr int KVP_POOLS = 128;      // pools of one launch: 1 KB of parameters

struct PagePools {
  void* base[KVP_POOLS];
  int64_t page_bytes, head_bytes;   // strides
  int heads, row_bytes, pages;
};

__device__ __forceinline__ bool page_ok(int page, int pages, int* err) {
  if ((unsigned)page < (unsigned)pages) return true;
  if (threadIdx.x == 0 && atomicCAS(err, 0, 103) == 0) { err[1] = blockIdx.x; err[2] = page; }
  return false;
}

// `bytes` (a multiple of 16) of one head of a page, by the block.
__device__ __forceinline__ void copy_head(const char* src, char* dst, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<const uint4*>(src + i);
}

// A page that is written twice, or written and read, would hold what came last: such pairs are left out and reported.
// Short lists are compared in every block of the copy, which costs it nothing (300 pairs of 8 pools of 256 KB: 195 us either way); long ones
// once, 256 pairs a block: lists of 4096 pairs of 8 KB in 8 pools 124 us in the copy and 132 apart, 16384 pairs 1226 and 534.
constexpr int KVP_CHECK = 4096;

__global__ void __launch_bounds__(256) kv_pages_check_kernel(const int* __restrict__ src, const int* __restrict__ dst, int n, uint8_t* clash, int* err) {
  pdl_wait();
  pdl_trigger();
  __shared__ int2 part[256];
  const int own = blockIdx.x * 256 + threadIdx.x, s = own < n ? src[own] : 0, d = own < n ? dst[own] : 0;
  int read = 0, written = 0;
  for (int a = 0; a < n; a += 256) {
    const int i = a + threadIdx.x;
    __syncthreads();
    part[threadIdx.x] = i < n ? make_int2(src[i], dst[i]) : make_int2(-1, -1);      // (no page)
    __syncthreads();
#pragma unroll 16
    for (int k = 0; k < 256; ++k) {
      read += part[k].x == d;
      written += part[k].y == d;
    }
  }
  const bool found = d >= 0 && (written > 1 || read > (s == d));                      // (others than the pair itself)
  if (own >= n) return;
  clash[own] = found;
  if (found && atomicCAS(err, 0, 105) == 0) { err[1] = own; err[2] = d; }
}

// Pair x of the lists, head y, pool z.  known: what the kernel above found, or null.
__global__ void __launch_bounds__(256) kv_pages_copy_kernel(const __grid_constant__ PagePools P, const int* __restrict__ src, const int* __restrict__ dst, int n,
                                                            const uint8_t* __restrict__ known, int* err) {
  pdl_wait();
  pdl_trigger();
  const int s = src[blockIdx.x], d = dst[blockIdx.x];
  if (known) {
    if (known[blockIdx.x]) return;
  } else {
    bool clash = false;
    for (int i = threadIdx.x; i < n; i += 256) clash |= i != (int)blockIdx.x && (dst[i] == d || src[i] == d);
    if (__syncthreads_or(clash)) {
      if (threadIdx.x == 0 && atomicCAS(err, 0, 105) == 0) { err[1] = blockIdx.x; err[2] = d; }
      return;
    }
  }
  if (s == d || !page_ok(s, P.pages, err) || !page_ok(d, P.pages, err)) return;
  char* base = static_cast<char*>(P.base[blockIdx.z]) + blockIdx.y * P.head_bytes;
  copy_head(base + s * P.page_bytes, base + d * P.page_bytes, 128 * P.row_bytes);
}

// One block per request of K beams.  Beam r goes on behind parents[r]: the columns of whole pages are gathered by reference, column by
// column (a thread reads a column before it writes it, so the table is updated in place).  The partly filled page of a parent stays with its
// first child; its other children take their spare pages, into which the next kernel copies the rows.  The pages of beams without
// children become the spare pages of the beams that used theirs: there are as many of one as of the other.
__global__ void __launch_bounds__(256) kv_fork_table_kernel(const int* __restrict__ parents, int K, int* __restrict__ table, int64_t table_row, int max_pages,
                                                            int* __restrict__ spare, const int* __restrict__ length, int* __restrict__ moves, int* err) {
  pdl_wait();
  pdl_trigger();
  __shared__ int par[32], tail[32], sp[32];
  __shared__ int cols[32][256];
  const int b = blockIdx.x, t = threadIdx.x;
  const int given = *length, len = min(max(given, 0), max_pages * 128), whole = len / 128, rest = len % 128;
  if (given != len && b == 0 && t == 0 && atomicCAS(err, 0, 102) == 0) { err[1] = given; err[2] = max_pages * 128; }
  int* rows = table + (int64_t)b * K * table_row;
  if (t < K) {
    int q = parents[b * K + t];
    if ((unsigned)q >= (unsigned)K) {
      if (atomicCAS(err, 0, 106) == 0) { err[1] = b * K + t; err[2] = q; }
      q = t;
    }
    par[t] = q;
    sp[t] = spare[b * K + t];
    if (rest) tail[t] = rows[t * table_row + whole];
  }
  __syncthreads();
  for (int c = t; c < whole; c += 256) {
    for (int r = 0; r < K; ++r) cols[r][t] = rows[r * table_row + c];
    for (int r = 0; r < K; ++r) rows[r * table_row + c] = cols[par[r]][t];
  }
  if (t < K) {
    int from = 0, to = 0;                                   // nothing to copy
    if (rest) {
      bool first = true;
      int before = 0;                                       // earlier beams that use their spare page
      for (int r = 0; r < t; ++r) {
        first &= par[r] != par[t];
        bool f = true;
        for (int u = 0; u < r; ++u) f &= par[u] != par[r];
        before += !f;
      }
      int page = tail[par[t]];
      if (!first) {
        from = page;
        to = page = sp[t];
        for (int q = 0, free = 0; q < K; ++q) {             // the page of the `before`-th beam without children
          bool child = false;
          for (int r = 0; r < K; ++r) child |= par[r] == q;
          if (!child && free++ == before) spare[b * K + t] = tail[q];
        }
      }
      rows[t * table_row + whole] = page;
    }
    moves[2 * (b * K + t)] = from;
    moves[2 * (b * K + t) + 1] = to;
  }
}

// Beam x, head y, pool z.
__global__ void __launch_bounds__(256) kv_fork_copy_kernel(const __grid_constant__ PagePools P, const int* __restrict__ moves, const int* __restrict__ length, int* err) {
  pdl_wait();
  pdl_trigger();
  const int s = moves[2 * blockIdx.x], d = moves[2 * blockIdx.x + 1];
  if (s == d || !page_ok(s, P.pages, err) || !page_ok(d, P.pages, err)) return;
  char* base = static_cast<char*>(P.base[blockIdx.z]) + blockIdx.y * P.head_bytes;
  copy_head(base + s * P.page_bytes, base + d * P.page_bytes, (*length % 128) * P.row_bytes);
}

// Pools are written while the lists and tables are read by other blocks.
static int apart_from_pools(const kd_tensor* const* pools, int n_pools, const kd_tensor* t, const char* what) {
  for (int i = 0; i < n_pools; ++i) KD_REQUIRE(!views_meet(pools[i], t), "%s must not share memory with a pool", what);
  return KD_OK;
}

static int page_pools(const kd_tensor* const* pools, int first, int count, PagePools* P) {
  const kd_tensor* a = pools[first];
  for (int i = 0; i < count; ++i) {
    const kd_tensor* t = pools[first + i];
    KD_REQUIRE(t, "null tensor");
    KD_REQUIRE(t->ndim == 4 && t->shape[2] == 128, "a pool must be [pages,Hkv,128,D]");
    const int64_t size = dtype_size(t->dtype);
    KD_REQUIRE(t->strides[3] == 1 && t->strides[2] == t->shape[3], "the 128 rows of a head must lie side by side");
    KD_REQUIRE(t->shape[3] * size % 16 == 0 && t->strides[0] * size % 16 == 0 && t->strides[1] * size % 16 == 0 && t->strides[0] >= 0 && t->strides[1] >= 0,
               "rows, heads and pages must begin on multiples of 16 bytes");
    KD_REQUIRE(t->shape[0] <= 0x7fffffff && t->shape[1] <= 65535 && t->shape[3] <= 65536, "the pool is too large");
    KD_REQUIRE(t->dtype == a->dtype, "the pools' types differ");
    for (int d = 0; d < 4; ++d) KD_REQUIRE(t->shape[d] == a->shape[d] && t->strides[d] == a->strides[d], "the pools' shapes or strides differ");
    KD_TRY(tensor_ptr(t, &P->base[i]));
    KD_REQUIRE((reinterpret_cast<uintptr_t>(P->base[i]) & 15) == 0, "pools must be 16-byte aligned");
  }
  const int64_t size = dtype_size(a->dtype);
  P->page_bytes = a->strides[0] * size;
  P->head_bytes = a->strides[1] * size;
  P->heads = (int)a->shape[1];
  P->row_bytes = (int)(a->shape[3] * size);
  P->pages = (int)a->shape[0];
  return KD_OK;
}

}  // namespace kd

using namespace kd;

KD_API int kd_kv_pages_copy(const kd_tensor* const* pools, int n_pools, const kd_tensor* src, const kd_tensor* dst) {
  KD_TRY(require_init());
  KD_REQUIRE(src && dst && n_pools >= 0 && (pools || n_pools == 0), "null tensor");
  KD_REQUIRE(src->dtype == KD_I32 && dst->dtype == KD_I32 && src->ndim == 1 && dst->ndim == 1 && is_contiguous(src) && is_contiguous(dst) && src->shape[0] == dst->shape[0],
             "src and dst must be contiguous int32 [n]");
  KD_REQUIRE(src->shape[0] <= 65536, "%lld pages: up to 65536 a call", (long long)src->shape[0]);
  const int n = (int)src->shape[0];
  void *ps, *pd, *known = nullptr;
  KD_TRY(tensor_ptr(src, &ps));
  KD_TRY(tensor_ptr(dst, &pd));
  PagePools P;
  for (int a = 0; a < n_pools; a += KVP_POOLS) KD_TRY(page_pools(pools, a, n_pools - a < KVP_POOLS ? n_pools - a : KVP_POOLS, &P));
  KD_TRY(apart_from_pools(pools, n_pools, src, "src"));
  KD_TRY(apart_from_pools(pools, n_pools, dst, "dst"));
  if (n > KVP_CHECK && n_pools > 0) {
    KD_TRY(get_workspace(n, &known));
    KD_CUDA_CHECK(launch_ex(kv_pages_check_kernel, dim3((n + 255) / 256), dim3(256), 0, (const int*)ps, (const int*)pd, n, (uint8_t*)known, ctx().error_flag));
    KD_TRY(after_launch("kv_pages_check_kernel"));
  }
  for (int a = 0; a < n_pools; a += KVP_POOLS) {
    const int count = n_pools - a < KVP_POOLS ? n_pools - a : KVP_POOLS;
    if (n_pools > KVP_POOLS) KD_TRY(page_pools(pools, a, count, &P));
    if (n == 0 || P.heads == 0 || P.row_bytes == 0) continue;
    KD_CUDA_CHECK(launch_ex(kv_pages_copy_kernel, dim3(n, P.heads, count), dim3(256), 0, P, (const int*)ps, (const int*)pd, n, (const uint8_t*)known, ctx().error_flag));
    KD_TRY(after_launch("kv_pages_copy_kernel"));
  }
  return KD_OK;
}

KD_API int kd_kv_pages_fork(const kd_tensor* const* pools, int n_pools, const kd_tensor* parents, const kd_tensor* block_table, const kd_tensor* spare,
                            const kd_tensor* length) {
  KD_TRY(require_init());
  KD_REQUIRE(parents && block_table && spare && length && n_pools >= 0 && (pools || n_pools == 0), "null tensor");
  KD_REQUIRE(parents->dtype == KD_I32 && parents->ndim == 2 && is_contiguous(parents) && parents->shape[1] >= 1 && parents->shape[1] <= 32,
             "parents must be contiguous int32 [requests, beams], of 1 to 32 beams");
  KD_REQUIRE(parents->shape[0] <= 65535 && numel(parents) <= 0x7fffffff, "too many requests");
  const int B = (int)parents->shape[0], K = (int)parents->shape[1];
  KD_REQUIRE(block_table->dtype == KD_I32 && block_table->ndim == 2 && block_table->shape[0] == (int64_t)B * K && block_table->strides[1] == 1 &&
                 block_table->strides[0] >= block_table->shape[1] && block_table->shape[1] < (1 << 24),
             "block_table must be int32 [requests x beams, max_pages] with rows in one piece");
  KD_REQUIRE(spare->dtype == KD_I32 && is_contiguous(spare) && numel(spare) == (int64_t)B * K, "spare must be contiguous int32 [requests x beams]");
  KD_REQUIRE(length->dtype == KD_I32 && numel(length) == 1, "length must be one int32");
  void *pp, *pt, *ps, *pl, *moves;
  KD_TRY(tensor_ptr(parents, &pp)); KD_TRY(tensor_ptr(block_table, &pt)); KD_TRY(tensor_ptr(spare, &ps)); KD_TRY(tensor_ptr(length, &pl));
  PagePools P;
  for (int a = 0; a < n_pools; a += KVP_POOLS) KD_TRY(page_pools(pools, a, n_pools - a < KVP_POOLS ? n_pools - a : KVP_POOLS, &P));
  KD_TRY(apart_from_pools(pools, n_pools, parents, "parents"));
  KD_TRY(apart_from_pools(pools, n_pools, block_table, "block_table"));
  KD_TRY(apart_from_pools(pools, n_pools, spare, "spare"));
  KD_TRY(apart_from_pools(pools, n_pools, length, "length"));
  KD_REQUIRE(!views_meet(block_table, spare) && !views_meet(block_table, parents) && !views_meet(block_table, length) && !views_meet(spare, parents) && !views_meet(spare, length),
             "block_table and spare must not share memory with one another or with what the call reads");
  if (B == 0) return KD_OK;
  KD_TRY(get_workspace(8 * (uint64_t)B * K, &moves));
  KD_CUDA_CHECK(launch_ex(kv_fork_table_kernel, dim3(B), dim3(256), 0, (const int*)pp, K, (int*)pt, (int64_t)block_table->strides[0], (int)block_table->shape[1], (int*)ps,
                          (const int*)pl, (int*)moves, ctx().error_flag));
  KD_TRY(after_launch("kv_fork_table_kernel"));
  for (int a = 0; a < n_pools && K > 1; a += KVP_POOLS) {
    const int count = n_pools - a < KVP_POOLS ? n_pools - a : KVP_POOLS;
    if (n_pools > KVP_POOLS) KD_TRY(page_pools(pools, a, count, &P));
    if (P.heads == 0 || P.row_bytes == 0) continue;
    KD_CUDA_CHECK(launch_ex(kv_fork_copy_kernel, dim3(B * K, P.heads, count), dim3(256), 0, P, (const int*)moves, (const int*)pl, ctx().error_flag));
    KD_TRY(after_launch("kv_fork_copy_kernel"));
  }
  return KD_OK;
}
