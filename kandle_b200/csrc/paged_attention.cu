// Attention of new tokens over a paged cache: kd_attention_paged.
//
// Sequence b brings n_b new tokens (packed rows of q), whose keys and values are the last n_b of its ctx_b positions in the pages:
// token i sees positions 0 .. ctx_b - n_b + i.
#include "common.cuh"
#include "kernels.cuh"
#include "sm100.cuh"

namespace kd {

using namespace sm100;

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
  int behind_tiles;            // the kernel before belongs to the same call, and has no part in what this one reads
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

// ----------------------------------------------------------------------------- what both kernels share
// A tile of 128 rows holds the query heads that share a KV head of 128 / group tokens, a token's heads side by side; a page is a key
// tile.  S = Q K^T and O += P V run on tcgen05 with S, P (over S, as packed bf16) and O in tensor memory; a thread owns a row.
constexpr int PA_ROWS = 128;

__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float pa_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// (x0, x1) = (a0, a1) * s + m
__device__ __forceinline__ void pa_fma2(float& x0, float& x1, float a0, float a1, float s, float m) {
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(x0), "=f"(x1) : "f"(a0), "f"(a1), "f"(s), "f"(m));
}
// (s0, s1) += (a0, a1)
__device__ __forceinline__ void pa_add2(float& s0, float& s1, float a0, float a1) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "+f"(s0), "+f"(s1) : "f"(a0), "f"(a1));
}

// One key tile of a thread's row, whose scores are complete: the running maximum m (of scores times scale_log2) and sum l, P for the MMA
// warp in two halves of 64 keys.  lim >= 0: only keys 0 .. lim of the tile are seen (masked; a row that sees none gets sums that its caller
// drops).  The maximum is raised only when it grew by more than 2^8: the sum uses the same one, so nothing is lost.  before_p() comes
// before P is handed over, o_ready() before O is touched; both return whether to go on, alike in a whole warp.
template <int D, typename Ready, typename Before>
__device__ __forceinline__ bool paged_softmax(uint32_t s_addr, uint32_t o_addr, bool masked, int lim, bool first, bool real, float scale_log2, float& m, float& l, uint64_t* p_ready,
                                              Ready o_ready, Before before_p) {
  tc_fence_after();
  uint32_t r[128];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_addr + c * 32, r + c * 32);
  tmem_wait_ld();
  if (masked) {
#pragma unroll
    for (int e = 0; e < 128; ++e)
      if (e > lim) r[e] = __float_as_uint(-1e30f);
  }
  float mx0 = -1e30f, mx1 = -1e30f, mx2 = -1e30f, mx3 = -1e30f;
#pragma unroll
  for (int e = 0; e < 128; e += 8) {
    mx0 = pa_max3(mx0, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
    mx1 = pa_max3(mx1, __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
    mx2 = pa_max3(mx2, __uint_as_float(r[e + 4]), __uint_as_float(r[e + 5]));
    mx3 = pa_max3(mx3, __uint_as_float(r[e + 6]), __uint_as_float(r[e + 7]));
  }
  const float m_blk = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * scale_log2;
  float alpha = 1.f;
  bool rescale = false;
  if (first || !real) {        // (nobody reads a padding row)
    m = m_blk;
  } else if (m_blk - m > 8.0f) {
    alpha = pa_exp2(m - m_blk);
    m = m_blk;
    rescale = true;
  }
  if (__any_sync(0xffffffffu, rescale)) {
    if (!o_ready()) return false;
    tc_fence_after();
#pragma unroll 1
    for (int c = 0; c < D / 16; ++c) {            // narrow pieces: the 128 scores stay in registers meanwhile
      uint32_t orr[16];
      tmem_ld_32x16(o_addr + c * 16, orr);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e) orr[e] = __float_as_uint(__uint_as_float(orr[e]) * alpha);
      tmem_st_32x16(o_addr + c * 16, orr);
    }
    l *= alpha;
  }
  if (!before_p()) return false;
  // P = 2^(s c - m) as packed bf16 over the first 64 columns of S.  (Probabilities meet the values as bf16, the type of the tensor
  // cores' other operand; their sum stays in fp32.)
  float sum0 = 0.f, sum1 = 0.f;
  const float neg_m = -m;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int e = 32 * half; e < 32 * half + 32; ++e) {
      float x0, x1;
      pa_fma2(x0, x1, __uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]), scale_log2, neg_m);
      const float e0 = pa_exp2(x0), e1 = pa_exp2(x1);
      pa_add2(sum0, sum1, e0, e1);
      r[e] = pack_bf16(e0, e1);
    }
    tmem_st_32x32(s_addr + half * 32, r + half * 32);
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(p_ready + half);
  }
  l += sum0 + sum1;
  return true;
}

// Behind the last key a page may hold anything, and 0 x NaN is none: those values become zeros before a product reads them.  By the
// four warps of a tile; `row` is the thread's key.
template <int D>
__device__ __forceinline__ void clear_values(uint8_t* tile, int row, int keys) {
  if (row >= keys) {
#pragma unroll
    for (int d = 0; d < D / 8; ++d) *reinterpret_cast<uint4*>(tile + (d / 8) * 16384 + row * 128 + (d % 8) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_proxy();
}

// ----------------------------------------------------------------------------- up to 128 query rows: one pass over the keys at HBM speed
// The key tiles of all sequences and KV heads stand in one row, and block x takes an equal share of it, from wherever it begins in one
// sequence to wherever it ends in another; a sequence that is cut leaves unnormalised sums that are joined.  So long and short
// sequences load every SM alike.
//   warps 0-3   softmax of the even key tiles of the block's piece of a sequence, and its output
//   warps 4-7   softmax of the odd ones: two chains of S, softmax and O, of which one computes while the other waits
//   warp 8      divides the work; TMA: queries, then pages through a ring
//   warp 9      tcgen05.mma
//   warps 10-11 complete the third warpgroup, which hands registers to the softmax (72 against 216 a thread)
// A warp whose rows are all padding only keeps step.  Bound: HBM; 128 exponentials a thread and tile are hidden behind the next pages.
constexpr int PR_THREADS = 384, PR_CACHE = 40;      // (sequences whose lengths are kept in shared memory)
struct RowSeq {
  int row0, n, ctx, tiles;            // tiles: of keys, 1 for tokens without keys; 0 where another kernel has the sequence
};
__device__ __forceinline__ RowSeq row_seq(const PagedParams& p, int b) {
  const PagedSeq s = paged_seq(p, b);
  const int rows = s.n * (p.Hq / p.Hkv);
  return RowSeq{s.row0, s.n, s.ctx, rows == 0 || rows > PA_ROWS ? 0 : max(1, (s.ctx + 127) / 128)};
}
struct PagedSplit {
  float* part_o;      // [place][rows][D] unnormalised sums
  float2* part_ml;    // [place][rows] (running maximum in the log2 domain, sum)
  int4* cut;          // the joining kernel's list: (sequence or first place, ..., parts)
  int* cuts;          // its length
  int slots;          // blocks of a head that run at a time
};
// Parts of a cut sequence that are through, by its first block; the last one sets it back.
constexpr int PA_BLOCKS = 1024;
static __device__ unsigned g_paged_through[PA_BLOCKS];
// A piece of a sequence.
struct Piece {
  int b, hk, j0, nb;                  // key tiles j0 .. j0 + nb - 1
  int parts, part, first;             // parts of the whole sequence, this one's number, the block of the first one
  RowSeq s;
};
// Goes through the pieces of block x; the same in every warp.
struct Walk {
  int64_t u, end, per;                // place in the row of tiles
  int b, hk, off;
  __device__ __forceinline__ bool next(const PagedParams& p, const int4* cache, Piece& w) {
    if (u >= end) return false;
    for (;;) {
      if (b == p.B) { b = 0; ++hk; }
      if (hk == p.Hkv) return false;
      if (b < PR_CACHE) { const int4 c = cache[b]; w.s = RowSeq{c.x, c.y, c.z, c.w}; }
      else w.s = row_seq(p, b);
      if (w.s.tiles) break;
      ++b;
    }
    const int64_t start = u - off, x = u / per;
    w.b = b; w.hk = hk; w.j0 = off;
    w.nb = (int)min((int64_t)(w.s.tiles - off), end - u);
    w.first = (int)(start / per);
    w.parts = (int)((start + w.s.tiles - 1) / per) - w.first + 1;
    w.part = (int)x - w.first;
    u += w.nb;
    ++b;
    off = 0;
    return true;
  }
};

// Four channels of a row from all parts of a sequence: sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k.  PIECES: part 0 ends block `first` (its
// second place), the others begin the blocks behind it (their first places); else places first, first + 1, ...
template <int D, bool PIECES>
__device__ __forceinline__ void join_parts(const PagedParams& p, const PagedSplit& in, const RowSeq& s, int hk, int r, int c, int64_t first, int parts, int part_rows, int token = -1,
                                           int head = 0) {
  const int group = p.Hq / p.Hkv;
  float m = -1e30f, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < parts; ++k) {
    const int64_t at = (PIECES ? 2 * (first + k) + (k == 0 ? 1 : 0) : first + k) * part_rows + r;
    const float2 x = __ldcg(in.part_ml + at);
    const float4 o = __ldcg(reinterpret_cast<const float4*>(in.part_o + at * D + c));
    if (x.y == 0.f) continue;            // nothing was seen there
    const float now = fmaxf(m, x.x), f0 = pa_exp2(m - now), f1 = pa_exp2(x.x - now);
    m = now;
    l = l * f0 + x.y * f1;
    acc.x = acc.x * f0 + o.x * f1; acc.y = acc.y * f0 + o.y * f1; acc.z = acc.z * f0 + o.z * f1; acc.w = acc.w * f0 + o.w * f1;
  }
  if (token < 0) { token = r / group; head = r % group; }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(p.o + (int64_t)(s.row0 + token) * p.so_t + (int64_t)(hk * group + head) * p.so_h + c) =
      make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

template <int D, int QROWS>
struct RowShape {
  static constexpr int TILE = 128 * D * 2, STAGES = 6 * 32768 / (2 * TILE);     // (keys and values)
  static constexpr int Q_BYTES = QROWS * D * 2, QBUF = QROWS < 128 ? 2 : 1;
  static constexpr int SMEM = 1024 + QBUF * Q_BYTES + STAGES * 2 * TILE + 256 + PR_CACHE * 16 + 128 + 1024;
  static_assert(SMEM <= 227 * 1024, "tiles exceed shared memory");
};

template <int D, int QROWS>
__global__ void __launch_bounds__(PR_THREADS, 1)
paged_rows_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                  const __grid_constant__ PagedParams p, const PagedSplit out) {
  using S = RowShape<D, QROWS>;
  constexpr int SLABS = D / 64, TILE = S::TILE, ST = S::STAGES, SLAB = 128 * 128, QSLAB = QROWS * 128, QBUF = S::QBUF;
  constexpr uint32_t IDESC_QK = make_idesc_bf16(128, 128, 0, 0), IDESC_PV = make_idesc_bf16(128, D, 0, 1);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;                                   // (an MMA reads 128 rows: what follows stands in for the missing ones)
  uint8_t* k_ring = q_smem + QBUF * S::Q_BYTES;
  uint8_t* v_ring = k_ring + ST * TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_ring + ST * TILE);
  uint64_t *q_full = bars, *q_empty = bars + 2, *s_full = bars + 4, *p_ready = bars + 6, *o_done = bars + 10, *o_free = bars + 12;
  uint64_t *k_full = bars + 13, *v_full = k_full + ST, *empty = v_full + ST;     // up to 6 each
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 31);
  int4* cache = reinterpret_cast<int4*>(bars + 32);
  float2* ml = reinterpret_cast<float2*>(cache + PR_CACHE); // odd chain's (maximum, sum) of every row
  Walk* walk_s = reinterpret_cast<Walk*>(ml + 128);
  int* flags = reinterpret_cast<int*>(walk_s + 1);          // abort, and one that stays 0; whether this block joins
  volatile int* abort_flag = flags;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.Hq / p.Hkv;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); mbar_init(&s_full[i], 1); mbar_init(&o_done[i], 1); }
    for (int i = 0; i < 4; ++i) mbar_init(&p_ready[i], 4);
    mbar_init(o_free, 4);
    for (int i = 0; i < ST; ++i) { mbar_init(&k_full[i], 1); mbar_init(&v_full[i], 1); mbar_init(&empty[i], 1); }
    flags[0] = flags[1] = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (!p.behind_tiles) pdl_wait();
  if (warp == 8) {
    // tiles of a head, and where this block begins
    int64_t sum = 0;
    for (int b = lane; b < p.B; b += 32) {
      const RowSeq s = row_seq(p, b);
      if (b < PR_CACHE) cache[b] = make_int4(s.row0, s.n, s.ctx, s.tiles);
      sum += s.tiles;
    }
    __syncwarp();
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    Walk w;
    const int64_t all = sum * p.Hkv;
    w.per = max((int64_t)1, (all + gridDim.x - 1) / gridDim.x);
    w.u = min(all, blockIdx.x * w.per);
    w.end = min(all, w.u + w.per);
    w.hk = w.b = w.off = 0;
    if (w.u < w.end) {
      w.hk = (int)(w.u / sum);
      int64_t left = w.u - w.hk * sum;
      for (int b0 = 0; b0 < p.B; b0 += 32) {
        int n = 0;
        if (b0 + lane < p.B) n = b0 + lane < PR_CACHE ? cache[b0 + lane].w : row_seq(p, b0 + lane).tiles;
        int64_t upto = n;
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, upto > left);
        if (hit) {
          const int who = __ffs(hit) - 1;
          w.b = b0 + who;
          w.off = (int)(left - __shfl_sync(0xffffffffu, upto - n, who));
          break;
        }
        left -= __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    if (lane == 0) *walk_s = w;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;      // S of chain t at 128 t, O at 256 + D t
  pdl_trigger();                              // after the TMEM allocation (see common.cuh)
  Walk walk = *walk_s;
  if (QROWS == PA_ROWS && threadIdx.x == 0) out.cut[blockIdx.x] = make_int4(0, 0, 0, 0);      // (thread 0 writes what is cut, too)
  Piece w;
  const int q_tokens = QROWS / group;
  int loaded = 0, q_loaded = 0;               // tiles (keys and values each) and queries asked for, by the copying warp
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.err, code)); };

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 8) {
    bool ok = true;
    for (; ok && walk.next(p, cache, w);) {
      if (w.s.ctx == 0) continue;
      const int qb = q_loaded % QBUF;
      if (!wait(&q_empty[qb], (uint32_t)(((q_loaded / QBUF) & 1) ^ 1), 321)) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(&q_full[qb], SLABS * q_tokens * group * 128);
#pragma unroll
        for (int d = 0; d < SLABS; ++d) tma_load_4d(q_smem + qb * S::Q_BYTES + d * QSLAB, &tmap_q, &q_full[qb], d * 64, w.hk * group, w.s.row0, 0);
      }
      __syncwarp();
      ++q_loaded;
      int page = 0;
      for (int j = 0; j < w.nb; ++j) {
        if (j % 32 == 0) {                    // 32 entries of the table at a time
          page = j + lane < w.nb ? p.table[w.b * p.table_row + w.j0 + j + lane] : 0;
          if ((unsigned)page >= (unsigned)p.pages && atomicCAS(p.err, 0, 103) == 0) { p.err[1] = w.b; p.err[2] = page; }
        }
        const int where = __shfl_sync(0xffffffffu, page, j % 32), slot = loaded % ST;
        if (!(ok = wait(&empty[slot], (uint32_t)(((loaded / ST) & 1) ^ 1), 322))) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&k_full[slot], TILE);
#pragma unroll
          for (int d = 0; d < SLABS; ++d) tma_load_4d(k_ring + slot * TILE + d * SLAB, &tmap_k, &k_full[slot], d * 64, 0, w.hk, where);
          mbar_arrive_expect_tx(&v_full[slot], TILE);
#pragma unroll
          for (int d = 0; d < SLABS; ++d) tma_load_4d(v_ring + slot * TILE + d * SLAB, &tmap_v, &v_full[slot], d * 64, 0, w.hk, where);
        }
        __syncwarp();
        ++loaded;
      }
    }
  } else if (warp == 9) {
    bool ok = true;
    int done = 0, q_done = 0, pieces = 0, turn[2] = {0, 0};      // tiles, queries, pieces with keys, tiles of a chain
    while (ok && walk.next(p, cache, w)) {
      if (w.s.ctx == 0) continue;
      const int qb = q_done % QBUF;
      if (!(ok = wait(&q_full[qb], (uint32_t)((q_done / QBUF) & 1), 323))) break;
      ++q_done;
      // S(g) = Q K(g)^T, g-th tile of the piece
      auto issue_qk = [&](int g) -> bool {
        const int slot = (done + g) % ST, t = g & 1;
        if (!wait(&k_full[slot], (uint32_t)(((done + g) / ST) & 1), 324)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t qdesc = make_smem_desc_sw128(smem_u32(q_smem + qb * S::Q_BYTES), 16, 1024), kdesc = make_smem_desc_sw128(smem_u32(k_ring + slot * TILE), 16, 1024);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_ss(tmem_base + (uint32_t)(t * 128), qdesc + ((uint32_t)((k / 4) * QSLAB + (k % 4) * 32) >> 4), kdesc + ((uint32_t)((k / 4) * SLAB + (k % 4) * 32) >> 4), IDESC_QK,
                    k != 0 ? 1u : 0u);
          umma_commit(&s_full[t]);
          if (g + 1 == w.nb) umma_commit(&q_empty[qb]);
        }
        __syncwarp();
        return true;
      };
      for (int g = 0; ok && g < 2 && g < w.nb; ++g) ok = issue_qk(g);
      // the sums of the piece before have been read
      if (ok && pieces > 0) ok = wait(o_free, (uint32_t)((pieces - 1) & 1), 325);
      for (int g = 0; ok && g < w.nb; ++g) {
        const int slot = (done + g) % ST, t = g & 1;
        if (!(ok = wait(&v_full[slot], (uint32_t)(((done + g) / ST) & 1), 326))) break;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!(ok = wait(&p_ready[2 * t + half], (uint32_t)(turn[t] & 1), 327))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t vdesc = make_smem_desc_sw128(smem_u32(v_ring + slot * TILE), SLAB, 1024);
#pragma unroll
            for (int k = 4 * half; k < 4 * half + 4; ++k)
              umma_ts(tmem_base + (uint32_t)(256 + t * D), tmem_base + (uint32_t)(t * 128 + k * 8), vdesc + (uint32_t)(k * 128), IDESC_PV, g > 1 || k != 0 ? 1u : 0u);
            if (half == 1) {
              umma_commit(&empty[slot]);
              umma_commit(&o_done[t]);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        ++turn[t];
        if (g + 2 < w.nb) ok = issue_qk(g + 2);
      }
      done += w.nb;
      ++pieces;
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = warp >> 2, q = warp & 3, row = q * 32 + lane, i = row / group;      // this row's token
    const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16), s_addr = lane_addr + (uint32_t)(t * 128), o_addr = lane_addr + (uint32_t)(256 + t * D);
    int done = 0, turn = 0, other = 0;      // tiles, this chain's, and for the even one those of the odd
    bool ok = true;
    while (ok && walk.next(p, cache, w)) {
      const int nb = w.s.ctx == 0 ? 0 : w.nb, hidden = w.s.ctx - w.s.n, rows = w.s.n * group;
      const bool real = row < rows, active = q * 32 < rows;
      const int last = real ? hidden + i : -1;                    // the last key that it sees
      float m = -1e30f, l = 0.f;
      for (int g = t; g < nb; g += 2, ++turn) {
        if (!(ok = wait(&s_full[t], (uint32_t)(turn & 1), 328))) break;
        const int kv0 = (w.j0 + g) * 128, slot = (done + g) % ST;
        auto before_p = [&] {
          if (kv0 + 128 <= w.s.ctx) return true;
          if (!wait(&v_full[slot], (uint32_t)(((done + g) / ST) & 1), 329)) return false;
          clear_values<D>(v_ring + slot * TILE, row, w.s.ctx - kv0);
          return true;
        };
        if (active) {
          ok = paged_softmax<D>(s_addr, o_addr, kv0 + 127 > hidden, last - kv0, g < 2, real, p.scale_log2, m, l, &p_ready[2 * t],
                                [&] { return wait(&o_done[t], (uint32_t)((turn - 1) & 1), 330); }, before_p);
          if (!ok) break;
        } else {
          if (!(ok = before_p())) break;
          __syncwarp();
          if (lane == 0) { mbar_arrive(&p_ready[2 * t]); mbar_arrive(&p_ready[2 * t + 1]); }
        }
      }
      if (!ok) break;
      done += nb;
      other += nb / 2;
      const int seen = min(last, (w.j0 + w.nb) * 128 - 1) - w.j0 * 128;        // the last key of the piece that the row sees
      if (nb <= t || seen < t * 128) { m = -1e30f; l = 0.f; }                  // (a row that sees none of a chain's keys has summed masked ones)
      if (nb > 1) {
        if (t == 1) ml[row] = make_float2(m, l);
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      if (t == 1) continue;
      // Both chains' sums.  (The odd one's next are behind the next product, which waits until these have been read.)
      if (nb > 0 && !(ok = wait(&o_done[0], (uint32_t)((turn - 1) & 1), 331))) break;
      if (nb > 1 && !(ok = wait(&o_done[1], (uint32_t)((other - 1) & 1), 331))) break;
      tc_fence_after();
      const float2 e = nb > 1 ? ml[row] : make_float2(-1e30f, 0.f);
      const float M = fmaxf(m, e.x), wa = l == 0.f ? 0.f : pa_exp2(m - M), we = e.y == 0.f ? 0.f : pa_exp2(e.x - M), L = wa * l + we * e.y;
      const bool direct = w.parts == 1;
      const int64_t at = (int64_t)(2 * blockIdx.x + (w.part == 0 ? 1 : 0)) * QROWS + row;
      const float f = !direct ? 1.f : L == 0.f ? 0.f : 1.f / L, fa = wa * f, fe = we * f;
      if (active) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          uint32_t x[32];
          __syncwarp();
          if (nb > 0) {
            tmem_ld_32x32(lane_addr + 256 + c * 32, x);
            tmem_wait_ld();
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = fa == 0.f ? 0.f : fa * __uint_as_float(x[k]);
          if (nb > 1) {
            tmem_ld_32x32(lane_addr + 256 + D + c * 32, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = fe == 0.f ? o[k] : fmaf(fe, __uint_as_float(x[k]), o[k]);
          }
          if (real && direct) {
            uint4* to = reinterpret_cast<uint4*>(p.o + (int64_t)(w.s.row0 + i) * p.so_t + (int64_t)(w.hk * group + row % group) * p.so_h + c * 32);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              to[k] = make_uint4(pack_bf16(o[8 * k], o[8 * k + 1]), pack_bf16(o[8 * k + 2], o[8 * k + 3]), pack_bf16(o[8 * k + 4], o[8 * k + 5]), pack_bf16(o[8 * k + 6], o[8 * k + 7]));
          } else if (real) {
            float4* to = reinterpret_cast<float4*>(out.part_o + at * D + c * 32);
#pragma unroll
            for (int k = 0; k < 8; ++k) to[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
        }
        if (real && !direct) out.part_ml[at] = make_float2(M, L);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && nb > 0) mbar_arrive(o_free);
      if (direct) continue;
      if constexpr (QROWS == PA_ROWS) {
        // 64 KB a part and more: a second kernel joins them
        if (threadIdx.x == 0 && w.part == 0) out.cut[blockIdx.x] = make_int4(w.b, w.hk, w.parts, 0);
      } else {
        // The part that is through last joins them all (in the parts' order, whoever is last).
        asm volatile("bar.sync 2, 128;" ::: "memory");
        if (threadIdx.x == 0) {
          unsigned before;
          asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(&g_paged_through[w.first]) : "memory");
          flags[2] = before == (unsigned)w.parts - 1;
          if (flags[2]) g_paged_through[w.first] = 0;
        }
        asm volatile("bar.sync 2, 128;" ::: "memory");
        if (flags[2]) {
          for (int n = threadIdx.x; n < rows * (D / 4); n += 128) {
            const int r = n / (D / 4);
            join_parts<D, true>(p, out, w.s, w.hk, r, n % (D / 4) * 4, w.first, w.parts, QROWS);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && warp == 8) {             // copies still on their way land before the block ends
    if (q_loaded > 0) mbar_wait(&q_full[(q_loaded - 1) % QBUF], (uint32_t)(((q_loaded - 1) / QBUF) & 1), flags + 1, p.err, 332);
    for (int k = max(0, loaded - ST); k < loaded; ++k) {
      mbar_wait(&k_full[k % ST], (uint32_t)((k / ST) & 1), flags + 1, p.err, 332);
      mbar_wait(&v_full[k % ST], (uint32_t)((k / ST) & 1), flags + 1, p.err, 332);
    }
  }
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  if (p.behind_tiles) pdl_wait();             // whoever waits for this kernel waits for the one before it
}

// Sequences with more than 32 rows that were cut.  Block x of the kernel above began with sequence cut[x] and did not end it; blocks of
// 32 rows, four channels a thread.
template <int D>
__global__ void __launch_bounds__(256) paged_rows_join_kernel(const __grid_constant__ PagedParams p, const PagedSplit in) {
  pdl_wait();
  pdl_trigger();
  const int4 c = in.cut[blockIdx.x];
  if (c.z <= 1) return;
  const RowSeq s = row_seq(p, c.x);
  const int rows = s.n * (p.Hq / p.Hkv);
  for (int n = threadIdx.x; n < 32 * (D / 4); n += 256) {
    const int r = blockIdx.y * 32 + n / (D / 4);
    if (r < rows) join_parts<D, true>(p, in, s, c.y, r, n % (D / 4) * 4, blockIdx.x, c.z, PA_ROWS);
  }
}

// ----------------------------------------------------------------------------- many query rows: tcgen05
// A block owns two tiles of 128 rows that share every key and passes over the pages of its part.
//   warps 0-3   softmax and output of tile A, a row per thread      warps 4-7   the same for tile B
//   warp 8      TMA: both query tiles, then the pages through two slots for keys and two for values
//   warp 9      tcgen05.mma: QK_A(0) QK_B(0) | PV_A(j) QK_A(j+1) PV_B(j) QK_B(j+1) | ..., one tile's products beside the other's softmax
//   warps 10-11 complete the third warpgroup, which hands registers to the softmax (72 against 216 a thread)
// Bound: the softmax's issued instructions beside the tensor pipe.
// How the work of every KV head is divided: per sequence `items` pairs of tiles with `len` key tiles each.  An item is cut into parts of at
// most L key tiles where there are too few to fill the GPU, or where one is longer than a block's even share.
struct PagedWork {
  int items, len;
};
constexpr int PT_CACHE = 256;       // sequences whose work is kept in shared memory while L is looked for
__device__ __forceinline__ PagedWork tile_work(const PagedParams& p, int b) {
  const PagedSeq s = paged_seq(p, b);
  const int group = p.Hq / p.Hkv, tokens = 2 * (PA_ROWS / group);
  if (s.n * group <= PA_ROWS) return PagedWork{0, 0};
  return PagedWork{(s.n + tokens - 1) / tokens, (s.ctx + 127) / 128};
}
__device__ __forceinline__ int parts_of(const PagedWork& w, int L) { return w.len <= L ? 1 : (w.len + L - 1) / L; }

// What block x of a head does: part `part` of `parts` of item `item` of sequence b (-1: nothing).  Items that are cut have more than L tiles, so
// there are at most `slots` of them and 2 x `slots` parts: `place` counts those before the item, `cut` the items, `cuts` all of them.
struct PagedPlan {
  int b, item, part, parts, place, cut, cuts;
};
// By one warp.  `slots`: blocks of a head that run at a time.
__device__ __forceinline__ PagedPlan paged_plan(const PagedParams& p, int x, int slots, int least, int2* cache) {
  const int lane = threadIdx.x & 31;
  auto of = [&](int b) {
    if (b < PT_CACHE) return PagedWork{cache[b].x, cache[b].y};
    return tile_work(p, b);
  };
  int64_t sum = 0;
  int longest = 0;
  for (int b = lane; b < p.B; b += 32) {
    const PagedWork w = tile_work(p, b);
    if (b < PT_CACHE) cache[b] = make_int2(w.items, w.len);
    sum += (int64_t)w.items * w.len;
    longest = max(longest, w.len);
  }
  __syncwarp();
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
  }
  const int even = max(least, (int)((sum + slots - 1) / slots));
  auto count = [&](int L) {
    int n = 0;
    for (int b = lane; b < p.B; b += 32) {
      const PagedWork w = of(b);
      n += w.items * parts_of(w, L);
    }
    return __reduce_add_sync(0xffffffffu, n);
  };
  // the smallest parts that run all at once; where that makes them a third longer than an even share, the even share
  int L = even;
  for (const int most = even + even / 3 + 1; L < longest && count(L) > slots;) {
    L += max(1, L / 16);
    if (L > most) {
      L = even;
      break;
    }
  }
  PagedPlan plan{-1, 0, 0, 0, 0, 0, 0};
  int before = 0, places = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const PagedWork w = b0 + lane < p.B ? of(b0 + lane) : PagedWork{0, 0};
    const int parts = w.items ? parts_of(w, L) : 0, n = w.items * parts;
    const int cut_parts = parts > 1 ? n : 0, cut_items = parts > 1 ? w.items : 0;
    int upto = n, cut_upto = cut_parts, items_upto = cut_items;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o), u = __shfl_up_sync(0xffffffffu, cut_upto, o), y = __shfl_up_sync(0xffffffffu, items_upto, o);
      if (lane >= o) { upto += v; cut_upto += u; items_upto += y; }
    }
    const int first = before + upto - n;
    const unsigned hit = __ballot_sync(0xffffffffu, x >= first && x < first + n);
    if (hit) {
      const int who = __ffs(hit) - 1;
      plan.b = b0 + who;
      plan.parts = __shfl_sync(0xffffffffu, parts, who);
      const int at = x - __shfl_sync(0xffffffffu, first, who);
      plan.item = at / plan.parts;
      plan.part = at % plan.parts;
      plan.place = places + __shfl_sync(0xffffffffu, cut_upto - cut_parts, who) + plan.item * plan.parts;
      plan.cut = plan.cuts + __shfl_sync(0xffffffffu, items_upto - cut_items, who) + plan.item;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    places += __shfl_sync(0xffffffffu, cut_upto, 31);
    plan.cuts += __shfl_sync(0xffffffffu, items_upto, 31);
  }
  return plan;
}

constexpr int PT_THREADS = 384, PT_ROWS = 256;

template <int D>
__global__ void __launch_bounds__(PT_THREADS, 1)
paged_tiles_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                   const __grid_constant__ PagedParams p, const PagedSplit out) {
  constexpr int SLABS = D / 64, NK = 2, NV = 2, TILE = 128 * D * 2, SLAB = 128 * 128;
  constexpr uint32_t TMEM_COLS = 512;     // scores of tile t at 128 t, sums at 256 + D t
  constexpr uint32_t IDESC_QK = make_idesc_bf16(128, 128, 0, 0), IDESC_PV = make_idesc_bf16(128, D, 0, 1);
  extern __shared__ uint8_t smem_raw[];
  __shared__ int2 cache[PT_CACHE];
  __shared__ PagedPlan plan_s;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;
  uint8_t* k_ring = q_smem + 2 * TILE;
  uint8_t* v_ring = k_ring + NK * TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_ring + NV * TILE);
  uint64_t* q_full = bars;          // 1
  uint64_t* t_full = bars + 1;      // 4: key slots, then value slots
  uint64_t* t_empty = bars + 5;     // 4
  uint64_t* s_full = bars + 9;      // 2
  uint64_t* p_ready = bars + 11;    // 4: [tile][half of the keys]
  uint64_t* o_done = bars + 15;     // 2
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);     // and behind it one that stays 0
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = blockIdx.y, group = p.Hq / p.Hkv, per_tile = 128 / group;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < NK + NV; ++i) { mbar_init(&t_full[i], 1); mbar_init(&t_empty[i], 1); }
    for (int t = 0; t < 2; ++t) { mbar_init(&s_full[t], 1); mbar_init(&o_done[t], 1); }
    for (int t = 0; t < 4; ++t) mbar_init(&p_ready[t], 4);
    abort_flag[0] = abort_flag[1] = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  pdl_wait();
  if (warp == 8) {
    const PagedPlan plan = paged_plan(p, blockIdx.x, out.slots, 2, cache);
    if (lane == 0) {
      plan_s = plan;
      if (hk == 0 && blockIdx.x == 0) *out.cuts = plan.cuts;
      if (hk == 0 && plan.b >= 0 && plan.part == 0 && plan.parts > 1) out.cut[plan.cut] = make_int4(plan.b, plan.item, plan.parts, plan.place);
    }
  }
  __syncthreads();
  const PagedPlan plan = plan_s;
  if (plan.b < 0) return;
  if (warp == 9) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();   // after the TMEM allocation (see common.cuh)

  const PagedSeq s = paged_seq(p, plan.b);
  const int hidden = s.ctx - s.n;                 // keys 0 .. hidden + i are seen by token i
  // the last tokens, which see the most keys, begin first
  const int items = (s.n + 2 * per_tile - 1) / (2 * per_tile), item = items - 1 - plan.item;
  int tok0[2], nblk[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    tok0[t] = (2 * item + t) * per_tile;
    nblk[t] = tok0[t] >= s.n ? 0 : (max(0, hidden + min(s.n, tok0[t] + per_tile)) + 127) / 128;
  }
  const int all = max(nblk[0], nblk[1]), j0 = (int)((int64_t)all * plan.part / plan.parts), n_blocks = (int)((int64_t)all * (plan.part + 1) / plan.parts) - j0;
#pragma unroll
  for (int t = 0; t < 2; ++t) nblk[t] = min(max(nblk[t] - j0, 0), n_blocks);     // block numbers below count from j0

  int issued = 0;                                 // pages' keys and values by the copying warp
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  // whole warps wait and an elected lane issues (see attention_prefill2.cu)
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.err, code)); };
  if (warp == 8) {
    if (n_blocks > 0) {
      if (elect_one()) {
        mbar_arrive_expect_tx(q_full, 2 * SLABS * per_tile * group * 128);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int d = 0; d < SLABS; ++d) tma_load_4d(q_smem + t * TILE + d * SLAB, &tmap_q, q_full, d * 64, hk * group, s.row0 + tok0[t], 0);
      }
      __syncwarp();
      int page = 0;
      for (int j = 0; j < n_blocks; ++j) {
        if (j % 32 == 0) {       // 32 entries of the table at a time
          page = j + lane < n_blocks ? p.table[plan.b * p.table_row + j0 + j + lane] : 0;
          if ((unsigned)page >= (unsigned)p.pages && atomicCAS(p.err, 0, 103) == 0) { p.err[1] = plan.b; p.err[2] = page; }
        }
        const int where = __shfl_sync(0xffffffffu, page, j % 32);
        if (!wait(&t_empty[j % NK], (uint32_t)(((j / NK) & 1) ^ 1), 421)) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&t_full[j % NK], TILE);
#pragma unroll
          for (int d = 0; d < SLABS; ++d) tma_load_4d(k_ring + (j % NK) * TILE + d * SLAB, &tmap_k, &t_full[j % NK], d * 64, 0, hk, where);
        }
        __syncwarp();
        issued = 2 * j + 1;
        if (!wait(&t_empty[NK + j % NV], (uint32_t)(((j / NV) & 1) ^ 1), 422)) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&t_full[NK + j % NV], TILE);
#pragma unroll
          for (int d = 0; d < SLABS; ++d) tma_load_4d(v_ring + (j % NV) * TILE + d * SLAB, &tmap_v, &t_full[NK + j % NV], d * 64, 0, hk, where);
        }
        __syncwarp();
        issued = 2 * j + 2;
      }
    }
  } else if (warp == 9) {
    bool ok = n_blocks == 0 || wait(q_full, 0, 423);
    auto commit = [&](uint64_t* bar) {
      if (elect_one()) umma_commit(bar);
      __syncwarp();
    };
    // S_t(j) = Q_t K(j)^T.  A page's keys are waited for by whichever tile comes first.
    auto issue_qk = [&](int t, int j, bool wait_k) -> bool {
      const int slot = j % NK;
      if (wait_k && !wait(&t_full[slot], (uint32_t)((j / NK) & 1), 424)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t qdesc = make_smem_desc_sw128(smem_u32(q_smem + t * TILE), 16, 1024), kdesc = make_smem_desc_sw128(smem_u32(k_ring + slot * TILE), 16, 1024);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (uint32_t)((k / 4) * SLAB + (k % 4) * 32) >> 4;
          umma_ss(tmem_base + (uint32_t)(t * 128), qdesc + off, kdesc + off, IDESC_QK, k != 0 ? 1u : 0u);
        }
        umma_commit(&s_full[t]);
      }
      __syncwarp();
      return true;
    };
    auto issue_pv = [&](int t, int j, bool wait_v) -> bool {
      const int slot = j % NV;
      if (wait_v && !wait(&t_full[NK + slot], (uint32_t)((j / NV) & 1), 426)) return false;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (!wait(&p_ready[2 * t + half], (uint32_t)(j & 1), 425)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vdesc = make_smem_desc_sw128(smem_u32(v_ring + slot * TILE), SLAB, 1024);
#pragma unroll
          for (int k = 4 * half; k < 4 * half + 4; ++k)
            umma_ts(tmem_base + (uint32_t)(256 + t * D), tmem_base + (uint32_t)(t * 128 + k * 8), vdesc + (uint32_t)(k * 128), IDESC_PV, (j | k) != 0 ? 1u : 0u);
          if (half == 1) umma_commit(&o_done[t]);
        }
        __syncwarp();
      }
      return true;
    };
    if (ok && n_blocks > 0) {
      if (nblk[0] > 0) ok = issue_qk(0, 0, true);
      if (ok && nblk[1] > 0) ok = issue_qk(1, 0, nblk[0] == 0);
      if (ok) commit(&t_empty[0]);
    }
    for (int j = 0; ok && j < n_blocks; ++j) {
      const bool a_now = j < nblk[0], b_now = j < nblk[1], a_next = j + 1 < nblk[0], b_next = j + 1 < nblk[1];
      if (a_now) ok = issue_pv(0, j, true);
      if (ok && a_next) ok = issue_qk(0, j + 1, true);
      if (ok && b_now) ok = issue_pv(1, j, !a_now);
      if (ok) commit(&t_empty[NK + j % NV]);
      if (ok && b_next) ok = issue_qk(1, j + 1, !a_next);
      if (ok && (a_next || b_next)) commit(&t_empty[(j + 1) % NK]);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = warp >> 2, q = warp & 3, row = q * 32 + lane, nb = t ? nblk[1] : nblk[0], first = t ? tok0[1] : tok0[0];
    const int i = first + row / group;            // this row's token; rows behind the tile's tokens see nothing
    const bool real = row < per_tile * group && i < s.n;
    const int last = real ? hidden + i : -1;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16), s_addr = lane_addr + (uint32_t)(t * 128), o_addr = lane_addr + (uint32_t)(256 + t * D);
    float m_used = -1e30f, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nb; ++j) {
      ok = mbar_wait(&s_full[t], (uint32_t)(j & 1), abort_flag, p.err, 427);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      const int kv0 = (j0 + j) * 128;
      auto o_ready = [&] { return (bool)__all_sync(0xffffffffu, mbar_wait(&o_done[t], (uint32_t)((j - 1) & 1), abort_flag, p.err, 428)); };
      auto before_p = [&] {
        // (by the tile whose product comes first)
        if (kv0 + 128 <= s.ctx || (t == 1 && j < nblk[0])) return true;
        if (!__all_sync(0xffffffffu, mbar_wait(&t_full[NK + j % NV], (uint32_t)((j / NV) & 1), abort_flag, p.err, 429))) return false;
        clear_values<D>(v_ring + (j % NV) * TILE, row, s.ctx - kv0);
        return true;
      };
      if (!(ok = paged_softmax<D>(s_addr, o_addr, kv0 + 127 > hidden + first, last - kv0, j == 0, real, p.scale_log2, m_used, l, &p_ready[2 * t], o_ready, before_p))) break;
    }
    if (ok && nb > 0) {
      ok = mbar_wait(&o_done[t], (uint32_t)((nb - 1) & 1), abort_flag, p.err, 430);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok) {
      tc_fence_after();
      const bool sees = nb > 0 && last >= j0 * 128;      // a row that sees none of these keys has summed masked ones
      const int h = hk * group + row % group;
      const bool direct = plan.parts == 1;
      const int64_t at = ((int64_t)hk * 2 * out.slots + plan.place + plan.part) * PT_ROWS + t * 128 + row;
      if (real && !direct) out.part_ml[at] = sees ? make_float2(m_used, l) : make_float2(-1e30f, 0.f);
      const float inv_l = sees ? 1.0f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t orr[32];
        __syncwarp();
        if (nb > 0) {
          tmem_ld_32x32(o_addr + c * 32, orr);
          tmem_wait_ld();
        }
        if (real && direct) {
          uint4* to = reinterpret_cast<uint4*>(p.o + (int64_t)(s.row0 + i) * p.so_t + (int64_t)h * p.so_h + c * 32);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (sees) {
              uint32_t* vv = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
              for (int e = 0; e < 4; ++e) vv[e] = pack_bf16(__uint_as_float(orr[g * 8 + 2 * e]) * inv_l, __uint_as_float(orr[g * 8 + 2 * e + 1]) * inv_l);
            }
            to[g] = v;
          }
        } else if (real && sees) {
          float4* to = reinterpret_cast<float4*>(out.part_o + at * D + c * 32);
#pragma unroll
          for (int g = 0; g < 8; ++g)
            to[g] = make_float4(__uint_as_float(orr[4 * g]), __uint_as_float(orr[4 * g + 1]), __uint_as_float(orr[4 * g + 2]), __uint_as_float(orr[4 * g + 3]));
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag && warp == 8) {      // copies still on their way land before the block ends
    if (n_blocks > 0) mbar_wait(q_full, 0, abort_flag + 1, p.err, 431);
    for (int k = max(0, issued - 4); k < issued; ++k) {
      const int j = k / 2, slot = k % 2 ? NK + j % NV : j % NK;
      mbar_wait(&t_full[slot], (uint32_t)((j / 2) & 1), abort_flag + 1, p.err, 431);
    }
  }
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Items that were cut: block (x, y, z) has 32 rows of the x-th of head y, four channels a thread.
template <int D>
__global__ void __launch_bounds__(256) paged_tiles_join_kernel(const __grid_constant__ PagedParams p, const PagedSplit in) {
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x >= *in.cuts) return;
  const int4 c = in.cut[blockIdx.x];
  const PagedSeq s = paged_seq(p, c.x);
  const int group = p.Hq / p.Hkv, per_tile = PA_ROWS / group, items = (s.n + 2 * per_tile - 1) / (2 * per_tile);
  for (int n = threadIdx.x; n < 32 * (D / 4); n += 256) {
    const int r = blockIdx.z * 32 + n / (D / 4), i = (2 * (items - 1 - c.y) + r / PA_ROWS) * per_tile + r % PA_ROWS / group;
    if (r % PA_ROWS < per_tile * group && i < s.n)
      join_parts<D, false>(p, in, RowSeq{s.row0, s.n, s.ctx, 0}, blockIdx.y, r, n % (D / 4) * 4, (int64_t)blockIdx.y * 2 * in.slots + c.w, c.z, PT_ROWS, i, r % PA_ROWS % group);
  }
}

// As launch_ex, always with a programmatic dependency on the kernel before: for kernels that belong to the same call.
template <typename... KArgs, typename... Args>
static cudaError_t launch_behind(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, Args&&... args) {
  const bool pdl = ctx().pdl;
  ctx().pdl = true;
  const cudaError_t e = launch_ex(kernel, grid, block, smem, std::forward<Args>(args)...);
  ctx().pdl = pdl;
  return e;
}

// [token][head][D] with a box of the query heads of `tokens` tokens on one KV head, 64 channels wide.
static int make_tmap_heads(CUtensorMap* out, const PagedParams& p, int tokens) {
  const int64_t ext[4] = {1, p.T, p.Hq, p.D}, st[3] = {p.T * p.sq_t, p.sq_t, p.sq_h};
  return make_tmap_bhsd(out, p.q, ext, st, p.Hq / p.Hkv, tokens);
}

struct PagedLaunch {
  PagedParams p;
  CUtensorMap k, v;
  PagedSplit rows, tiles;
};

template <int D>
static int launch_tiles(const PagedLaunch& a) {
  constexpr int SMEM = 6 * 128 * D * 2 + 1024 + 256;
  static bool configured[64] = {false};   // per device: kd_shutdown + kd_init may move the library to another GPU
  if (!configured[ctx().device & 63]) {
    KD_CUDA_CHECK(cudaFuncSetAttribute(paged_tiles_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    configured[ctx().device & 63] = true;
  }
  const PagedParams& p = a.p;
  const int per_tile = PA_ROWS / (p.Hq / p.Hkv);
  CUtensorMap tq;
  KD_TRY(make_tmap_heads(&tq, p, per_tile));
  const int64_t blocks = a.tiles.slots + (int64_t)p.T / (2 * per_tile) + p.B;     // items of all sequences, and one more for every cut
  KD_CUDA_CHECK(launch_ex(paged_tiles_kernel<D>, dim3((unsigned)blocks, p.Hkv), dim3(PT_THREADS), (size_t)SMEM, tq, a.k, a.v, p, a.tiles));
  return after_launch("paged_tiles_kernel");
}
template <int D, int QROWS>
static int launch_rows(const PagedLaunch& a) {
  using S = RowShape<D, QROWS>;
  static bool configured[64] = {false};
  if (!configured[ctx().device & 63]) {
    KD_CUDA_CHECK(cudaFuncSetAttribute(paged_rows_kernel<D, QROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    configured[ctx().device & 63] = true;
  }
  CUtensorMap tq;
  KD_TRY(make_tmap_heads(&tq, a.p, QROWS / (a.p.Hq / a.p.Hkv)));
  const dim3 grid(ctx().sm_count), block(PR_THREADS);
  if (a.p.behind_tiles) KD_CUDA_CHECK(launch_behind(paged_rows_kernel<D, QROWS>, grid, block, (size_t)S::SMEM, tq, a.k, a.v, a.p, a.rows));
  else KD_CUDA_CHECK(launch_ex(paged_rows_kernel<D, QROWS>, grid, block, (size_t)S::SMEM, tq, a.k, a.v, a.p, a.rows));
  KD_TRY(after_launch("paged_rows_kernel"));
  if constexpr (QROWS == PA_ROWS) {
    KD_CUDA_CHECK(launch_behind(paged_rows_join_kernel<D>, dim3(ctx().sm_count, 4), dim3(256), 0, a.p, a.rows));
    KD_TRY(after_launch("paged_rows_join_kernel"));
  }
  return KD_OK;
}

template <int D>
static int launch_paged(PagedLaunch& a) {
  PagedParams& p = a.p;
  const int64_t rows = (int64_t)p.max_query * (p.Hq / p.Hkv);
  const bool tiles = rows > PA_ROWS, few = rows <= PA_ROWS || p.q_start;
  const int sms = ctx().sm_count, part = rows <= 32 ? 32 : PA_ROWS;
  KD_REQUIRE(sms <= PA_BLOCKS, "%d multiprocessors", sms);
  a.tiles.slots = sms / p.Hkv > 0 ? sms / p.Hkv : 1;
  const uint64_t row_places = few ? 2 * (uint64_t)sms * part : 0, tile_places = tiles ? 2 * (uint64_t)a.tiles.slots * p.Hkv * PT_ROWS : 0;
  void* scratch;
  KD_TRY(get_workspace((row_places + tile_places) * (D * 4 + 8) + ((uint64_t)sms + a.tiles.slots + 1) * 16, &scratch));
  a.rows.part_o = static_cast<float*>(scratch);
  a.tiles.part_o = a.rows.part_o + row_places * D;
  a.rows.part_ml = reinterpret_cast<float2*>(a.tiles.part_o + tile_places * D);
  a.tiles.part_ml = a.rows.part_ml + row_places;
  a.rows.cut = reinterpret_cast<int4*>(a.tiles.part_ml + tile_places);
  a.tiles.cut = a.rows.cut + sms;
  a.tiles.cuts = reinterpret_cast<int*>(a.tiles.cut + a.tiles.slots);
  p.behind_tiles = tiles;
  if (tiles) KD_TRY(launch_tiles<D>(a));
  if (few) KD_TRY((rows <= 32 ? launch_rows<D, 32>(a) : launch_rows<D, PA_ROWS>(a)));
  if (!tiles) return KD_OK;
  KD_CUDA_CHECK(launch_behind(paged_tiles_join_kernel<D>, dim3(a.tiles.slots, p.Hkv, PT_ROWS / 32), dim3(256), 0, p, a.tiles));
  return after_launch("paged_tiles_join_kernel");
}

// After an error a sequence may have been left with some of its parts counted (context.cu, check_device_flag).
int paged_reset_counters() {
  void* at = nullptr;
  KD_CUDA_CHECK(cudaGetSymbolAddress(&at, g_paged_through));
  KD_CUDA_CHECK(cudaMemsetAsync(at, 0, sizeof(unsigned) * PA_BLOCKS, ctx().stream));
  return KD_OK;
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
  KD_REQUIRE(Hkv > 0 && Hq > 0 && Hq <= 65535 && Hq % Hkv == 0 && Hq / Hkv <= 64, "%d query heads on %d key heads: a multiple of them, up to 64 times, is handled", Hq, Hkv);
  KD_REQUIRE(k_pool->shape[2] == 128 && k_pool->shape[3] == D, "pools must be [pages,Hkv,128,%d]", D);
  for (int i = 0; i < 4; ++i) KD_REQUIRE(v_pool->shape[i] == k_pool->shape[i], "the pools' shapes differ");
  for (int i = 0; i < 3; ++i) KD_REQUIRE(out->shape[i] == q->shape[i], "out must have q's shape");
  KD_REQUIRE(q->strides[2] == 1 && out->strides[2] == 1 && k_pool->strides[3] == 1 && v_pool->strides[3] == 1, "unit stride along the head dimension required");
  for (int i = 0; i < 2; ++i) KD_REQUIRE(q->strides[i] % 8 == 0 && out->strides[i] % 8 == 0, "strides must be multiples of 8 elements");
  for (int i = 0; i < 3; ++i)
    KD_REQUIRE(k_pool->strides[i] % 8 == 0 && v_pool->strides[i] % 8 == 0 && k_pool->strides[i] >= 0 && v_pool->strides[i] >= 0, "strides must be multiples of 8 elements");
  KD_REQUIRE(k_pool->shape[0] >= 1, "the pools hold no page");
  KD_REQUIRE(block_table->ndim == 2 && block_table->dtype == KD_I32 && block_table->strides[1] == 1 && block_table->strides[0] >= 0, "block_table must be int32 [B,max_pages] with rows in one piece");
  KD_REQUIRE(block_table->shape[0] <= 65535 && block_table->shape[1] < (1 << 24), "the block table is too large");
  const int B = (int)block_table->shape[0], max_pages = (int)block_table->shape[1];
  KD_REQUIRE(ctx_len->dtype == KD_I32 && is_contiguous(ctx_len) && (numel(ctx_len) == B || numel(ctx_len) == 1), "ctx_len must be int32 [B] or one number for all");
  KD_REQUIRE(scale >= 1e-6f && scale <= 1e6f, "scale must lie between 1e-6 and 1e6");
  if (q_start) {
    KD_REQUIRE(q_start->dtype == KD_I32 && is_contiguous(q_start) && numel(q_start) == (int64_t)B + 1, "q_start must be int32 [B+1]");
  } else {
    KD_REQUIRE(B == 0 || T % B == 0, "%d tokens do not divide over %d sequences: q_start says where each begins", T, B);
  }
  KD_REQUIRE(max_query >= 0, "max_query must not be negative");
  if (T == 0 || B == 0) return KD_OK;
  PagedLaunch a{};
  PagedParams& p = a.p;
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
  KD_TRY(make_tmap_bhsd(&a.k, p.k, k_pool->shape, k_pool->strides, 128));
  KD_TRY(make_tmap_bhsd(&a.v, p.v, v_pool->shape, v_pool->strides, 128));
  return D == 128 ? launch_paged<128>(a) : launch_paged<64>(a);
}
