// Attention of new tokens over a paged cache: kd_attention_paged.
//
// Sequence b brings n_b new tokens (packed rows of q), whose keys and values are the last n_b of its ctx_b positions in the pages:
// token i sees positions 0 .. ctx_b - n_b + i.
#include "common.cuh"
#include "kernels.cuh"

namespace kd {

struct PagedParams {
  int T, B, Hq, Hkv, D, max_pages, pages;
  int even;                    // q_start null: this many tokens for every sequence
  int max_query;
  const int *q_start, *ctx, *table;
  int ctx_step;                // 0: one context length for all sequences
  int64_t table_row;
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  int64_t sq_t, sq_h, so_t, so_h, sk[3], sv[3];   // pools: page, head, row
  float scale_log2;
  int* err;
};

// A sequence's first row in q, its new tokens and its keys, whatever the tensors on the device say: rows stay inside q, positions
// inside the block table.
struct PagedSeq {
  int row0, n, ctx;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int b) {
  PagedSeq s;
  const int a = p.q_start ? p.q_start[b] : b * p.even, e = p.q_start ? p.q_start[b + 1] : a + p.even;
  s.row0 = min(max(a, 0), p.T);
  s.n = min(min(max(e, s.row0), p.T) - s.row0, p.max_query);
  const int c = p.ctx[(int64_t)b * p.ctx_step];
  s.ctx = min(max(c, 0), p.max_pages * 128);
  if ((s.row0 != a || s.row0 + s.n != e) && atomicCAS(p.err, 0, 104) == 0) { p.err[1] = b; p.err[2] = a; p.err[3] = e; }
  if (s.ctx != c && atomicCAS(p.err, 0, 102) == 0) { p.err[1] = c; p.err[2] = p.max_pages * 128; }
  return s;
}

// One warp per query row and head.
__global__ void __launch_bounds__(256) paged_attention_kernel(const PagedParams p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, h = blockIdx.y, b = blockIdx.z;
  const PagedSeq s = paged_seq(p, b);
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= s.n) return;
  const int hk = h / (p.Hq / p.Hkv), per = p.D / 32;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -1e30f, l = 0.f;
  for (int e = 0; e < per; ++e) q[e] = __bfloat162float(p.q[(s.row0 + i) * p.sq_t + h * p.sq_h + lane * per + e]);
  const int seen = s.ctx - s.n + i + 1;
  for (int j = 0; j < seen; ++j) {
    const int page = p.table[b * p.table_row + j / 128];
    if ((unsigned)page >= (unsigned)p.pages) {
      if (lane == 0 && atomicCAS(p.err, 0, 103) == 0) { p.err[1] = b; p.err[2] = page; }
      continue;
    }
    const __nv_bfloat16* k = p.k + page * p.sk[0] + hk * p.sk[1] + (j % 128) * p.sk[2] + lane * per;
    const __nv_bfloat16* v = p.v + page * p.sv[0] + hk * p.sv[1] + (j % 128) * p.sv[2] + lane * per;
    float d = 0.f;
    for (int e = 0; e < per; ++e) d += q[e] * __bfloat162float(k[e]);
    d = warp_sum(d) * p.scale_log2;
    const float m2 = fmaxf(m, d), a = exp2f(m - m2), w = exp2f(d - m2);
    for (int e = 0; e < per; ++e) o[e] = o[e] * a + w * __bfloat162float(v[e]);
    l = l * a + w;
    m = m2;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;     // a token that sees nothing gets a zero row
  for (int e = 0; e < per; ++e) p.o[(s.row0 + i) * p.so_t + h * p.so_h + lane * per + e] = __float2bfloat16_rn(o[e] * inv);
}

}  // namespace kd

using namespace kd;

KD_API int kd_attention_paged(const kd_tensor* q, const kd_tensor* k_pool, const kd_tensor* v_pool, const kd_tensor* block_table,
                              const kd_tensor* ctx_len, const kd_tensor* q_start, int max_query, float scale, const kd_tensor* out) {
  KD_TRY(require_init());
  KD_REQUIRE(q && k_pool && v_pool && block_table && ctx_len && out, "null tensor");
  KD_REQUIRE(q->ndim == 3 && out->ndim == 3 && k_pool->ndim == 4 && v_pool->ndim == 4, "q and out are [tokens,Hq,D], the pools [pages,Hkv,128,D]");
  KD_REQUIRE(q->dtype == KD_BF16 && out->dtype == KD_BF16 && k_pool->dtype == KD_BF16 && v_pool->dtype == KD_BF16, "q, pools and out must be bf16");
  KD_REQUIRE(q->shape[0] <= 0x7fffff00 && k_pool->shape[0] <= 0x7fffffff, "too many tokens or pages");
  const int T = (int)q->shape[0], Hq = (int)q->shape[1], D = (int)q->shape[2], Hkv = (int)k_pool->shape[1];
  KD_REQUIRE(D == 64 || D == 128, "head size %d: 64 or 128 are handled", D);
  KD_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 64, "%d query heads on %d key heads: a multiple of them, up to 64 times, is handled", Hq, Hkv);
  KD_REQUIRE(k_pool->shape[2] == 128 && k_pool->shape[3] == D, "pools must be [pages,Hkv,128,%d]", D);
  for (int i = 0; i < 4; ++i) KD_REQUIRE(v_pool->shape[i] == k_pool->shape[i], "the pools' shapes differ");
  for (int i = 0; i < 3; ++i) KD_REQUIRE(out->shape[i] == q->shape[i], "out must have q's shape");
  KD_REQUIRE(q->strides[2] == 1 && out->strides[2] == 1 && k_pool->strides[3] == 1 && v_pool->strides[3] == 1, "unit stride along the head dimension required");
  for (int i = 0; i < 2; ++i) KD_REQUIRE(q->strides[i] % 8 == 0 && out->strides[i] % 8 == 0, "strides must be multiples of 8 elements");
  for (int i = 0; i < 3; ++i)
    KD_REQUIRE(k_pool->strides[i] % 8 == 0 && v_pool->strides[i] % 8 == 0 && k_pool->strides[i] >= 0 && v_pool->strides[i] >= 0, "strides must be multiples of 8 elements");
  KD_REQUIRE(block_table->ndim == 2 && block_table->dtype == KD_I32 && block_table->strides[1] == 1 && block_table->strides[0] >= 0, "block_table must be int32 [B,max_pages] with rows in one piece");
  KD_REQUIRE(block_table->shape[0] <= 65535 && block_table->shape[1] < (1 << 24), "the block table is too large");
  const int B = (int)block_table->shape[0], max_pages = (int)block_table->shape[1];
  KD_REQUIRE(ctx_len->dtype == KD_I32 && is_contiguous(ctx_len) && (numel(ctx_len) == B || numel(ctx_len) == 1), "ctx_len must be int32 [B] or one number for all");
  KD_REQUIRE(scale > 0.f && scale < 1e30f, "scale must be positive");
  if (q_start) {
    KD_REQUIRE(q_start->dtype == KD_I32 && is_contiguous(q_start) && numel(q_start) == (int64_t)B + 1, "q_start must be int32 [B+1]");
  } else {
    KD_REQUIRE(B == 0 || T % B == 0, "%d tokens do not divide over %d sequences: q_start says where each begins", T, B);
  }
  KD_REQUIRE(max_query >= 0, "max_query must not be negative");
  if (T == 0 || B == 0) return KD_OK;
  PagedParams p{};
  p.T = T; p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.D = D; p.max_pages = max_pages;
  p.pages = (int)k_pool->shape[0];
  p.even = q_start ? 0 : T / B;
  p.max_query = !q_start ? p.even : max_query == 0 || max_query > T ? T : max_query;
  p.ctx_step = numel(ctx_len) == 1 ? 0 : 1;
  p.table_row = block_table->strides[0];
  void *pq, *pk, *pv, *po, *pt, *pc, *ps = nullptr;
  KD_TRY(tensor_ptr(q, &pq)); KD_TRY(tensor_ptr(k_pool, &pk)); KD_TRY(tensor_ptr(v_pool, &pv)); KD_TRY(tensor_ptr(out, &po));
  KD_TRY(tensor_ptr(block_table, &pt)); KD_TRY(tensor_ptr(ctx_len, &pc));
  if (q_start) KD_TRY(tensor_ptr(q_start, &ps));
  KD_REQUIRE(((reinterpret_cast<uintptr_t>(pq) | reinterpret_cast<uintptr_t>(pk) | reinterpret_cast<uintptr_t>(pv) | reinterpret_cast<uintptr_t>(po)) & 15) == 0,
             "q, pools and out must be 16-byte aligned");
  p.q = static_cast<const __nv_bfloat16*>(pq); p.k = static_cast<const __nv_bfloat16*>(pk); p.v = static_cast<const __nv_bfloat16*>(pv);
  p.o = static_cast<__nv_bfloat16*>(po);
  p.table = static_cast<const int*>(pt); p.ctx = static_cast<const int*>(pc); p.q_start = static_cast<const int*>(ps);
  p.sq_t = q->strides[0]; p.sq_h = q->strides[1]; p.so_t = out->strides[0]; p.so_h = out->strides[1];
  for (int i = 0; i < 3; ++i) { p.sk[i] = k_pool->strides[i]; p.sv[i] = v_pool->strides[i]; }
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = ctx().error_flag;
  KD_CUDA_CHECK(launch_ex(paged_attention_kernel, dim3((p.max_query + 7) / 8, Hq, B), dim3(256), 0, p));
  return after_launch("paged_attention_kernel");
}
