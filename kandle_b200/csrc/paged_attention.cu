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

// ----------------------------------------------------------------------------- how the work is divided
// Work of every KV head: per sequence `items` tiles of queries of `len` key tiles each.  An item is cut into parts of at most L key tiles,
// and a block takes a part, so that long and short sequences fill the GPU alike.
struct PagedWork {
  int items, len;
};
constexpr int PA_CACHE = 512;       // sequences whose work is kept in shared memory while L is looked for
constexpr int PA_FEW_ROWS = 64;     // rows (new tokens x query heads of a KV head) up to which a sequence is one item of the few-row kernel
constexpr int PA_KEYS = 64;         // keys of a tile there

__device__ __forceinline__ PagedWork few_work(const PagedParams& p, int b) {
  const PagedSeq s = paged_seq(p, b);
  const int rows = s.n * (p.Hq / p.Hkv);
  if (rows == 0 || rows > PA_FEW_ROWS) return PagedWork{0, 0};
  return PagedWork{1, (s.ctx + PA_KEYS - 1) / PA_KEYS};
}
// Two tiles of 128 rows an item; a tile holds the query heads of as many tokens as fit.
__device__ __forceinline__ PagedWork tile_work(const PagedParams& p, int b) {
  const PagedSeq s = paged_seq(p, b);
  const int group = p.Hq / p.Hkv, tokens = 2 * (128 / group);
  if (s.n * group <= PA_FEW_ROWS) return PagedWork{0, 0};
  return PagedWork{(s.n + tokens - 1) / tokens, (s.ctx + 127) / 128};
}
__device__ __forceinline__ int parts_of(const PagedWork& w, int L) { return w.len <= L ? 1 : (w.len + L - 1) / L; }

// What block x of a head does: part `part` of `parts` of item `item` of sequence b.  `place`: where the first part of the sequence's first item
// leaves its sums, counted over the items that are cut (these have more than L tiles each, so there are at most `slots` of them and
// 2 x `slots` parts).
struct PagedPlan {
  int b, item, part, parts, place;
};
// By one warp.  `slots`: blocks of a head that run at a time.  Returns b = -1 where there is no work for x.
template <typename Work>
__device__ __forceinline__ PagedPlan paged_plan(const PagedParams& p, Work work, int x, int slots, int least, int2* cache) {
  const int lane = threadIdx.x & 31;
  auto of = [&](int b) {
    if (b < PA_CACHE) return PagedWork{cache[b].x, cache[b].y};
    return work(p, b);
  };
  int64_t sum = 0;
  int longest = 0;
  for (int b = lane; b < p.B; b += 32) {
    const PagedWork w = work(p, b);
    if (b < PA_CACHE) cache[b] = make_int2(w.items, w.len);
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
  PagedPlan plan{-1, 0, 0, 0, 0};
  int before = 0, cut_before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const PagedWork w = b0 + lane < p.B ? of(b0 + lane) : PagedWork{0, 0};
    const int parts = w.items ? parts_of(w, L) : 0, n = w.items * parts;
    const int cut = parts > 1 ? n : 0;
    int upto = n, cut_upto = cut;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o), u = __shfl_up_sync(0xffffffffu, cut_upto, o);
      if (lane >= o) { upto += v; cut_upto += u; }
    }
    const int first = before + upto - n;
    const unsigned hit = __ballot_sync(0xffffffffu, x >= first && x < first + n);
    if (hit) {
      const int who = __ffs(hit) - 1;
      plan.b = b0 + who;
      plan.parts = __shfl_sync(0xffffffffu, parts, who);
      plan.place = __shfl_sync(0xffffffffu, cut_before + cut_upto - cut, who);
      const int at = x - __shfl_sync(0xffffffffu, first, who);
      plan.item = at / plan.parts;
      plan.part = at % plan.parts;
      return plan;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    cut_before += __shfl_sync(0xffffffffu, cut_upto, 31);
  }
  return plan;
}

// ----------------------------------------------------------------------------- few query rows: one pass over the keys at HBM speed
// The rows of a sequence and KV head (its new tokens times the query heads on it, at most 64) are one tile.  Keys and values come as tiles of 64
// through a ring of TMA copies.  Four groups of warps each take 16 keys of a tile, with a running maximum and sum of their own, so that
// no warp waits for another before the end; there they are joined in shared memory.  Tiles of 16 rows suit mma.sync (m16n8k16): with 2 to
// 16 live rows a tcgen05 tile of 128 would compute eight times as much and leave its softmax to as many threads.  Bound: HBM.
struct PagedSplit {
  float* part_o;      // [part][Hkv][rows][D] unnormalised sums
  float2* part_ml;    // [part][Hkv][rows] (running maximum in the log2 domain, sum)
  int2* plan;         // per sequence: place of its first part, parts of an item
  int slots;
};

__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// MT tiles of 16 rows a warp, RG groups of warps side by side over the rows.
template <int D, int MT, int RG>
struct FewShape {
  static constexpr int ROWS = 16 * MT * RG, WARPS = 4 * RG, THREADS = 32 * (WARPS + 1);
  static constexpr int TILE = PA_KEYS * D * 2, CTAS = RG == 1 ? 2 : 1;
  static constexpr int SLOTS = (CTAS == 2 ? 96 : 192) * 1024 / TILE;
  static constexpr int Q_BYTES = ROWS * D * 2;
  static constexpr int SMEM = 1024 + Q_BYTES + SLOTS * TILE + SLOTS * 16 + ROWS * 4 * 8 + 64;
  static_assert(4 * ROWS * D * 4 <= SLOTS * TILE, "the warps' sums are joined in the ring");
};

template <int D, int MT, int RG>
__global__ void __launch_bounds__(FewShape<D, MT, RG>::THREADS, FewShape<D, MT, RG>::CTAS)
paged_few_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ PagedParams p, const PagedSplit out) {
  using S = FewShape<D, MT, RG>;
  constexpr int SLAB = PA_KEYS * 128, QSLAB = S::ROWS * 128, NT = D / 8;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int2 cache[PA_CACHE];
  __shared__ PagedPlan plan_s;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem;
  uint8_t* q_smem = ring + S::SLOTS * S::TILE;
  uint64_t* full = reinterpret_cast<uint64_t*>(q_smem + S::Q_BYTES);
  uint64_t* empty = full + S::SLOTS;
  float2* ml = reinterpret_cast<float2*>(empty + S::SLOTS);        // [key group][row]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ml + 4 * S::ROWS);      // and behind it one that stays 0
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = blockIdx.y, group = p.Hq / p.Hkv;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::SLOTS; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], S::WARPS); }
    abort_flag[0] = abort_flag[1] = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  pdl_wait();
  if (warp == S::WARPS) {
    const PagedPlan plan = paged_plan(p, few_work, blockIdx.x, out.slots, 2, cache);
    if (lane == 0) {
      plan_s = plan;
      if (plan.b >= 0 && plan.part == 0 && hk == 0) out.plan[plan.b] = make_int2(plan.place, plan.parts);
    }
  }
  __syncthreads();
  const PagedPlan plan = plan_s;
  if (plan.b < 0) return;
  const PagedSeq s = paged_seq(p, plan.b);
  const int rows = s.n * group, tiles = (s.ctx + PA_KEYS - 1) / PA_KEYS;
  const int j0 = (int)((int64_t)tiles * plan.part / plan.parts), j1 = (int)((int64_t)tiles * (plan.part + 1) / plan.parts);
  const int hidden = s.ctx - s.n;                                  // keys 0 .. hidden + i are seen by token i

  int issued = 0;                                                  // by the copying warp
  if (warp == S::WARPS) {
    bool ok = true;
    int page = 0;
    for (int j = j0; ok && j < j1; ++j) {
      const int i = j - j0;
      // 32 entries of the table at a time
      if (i % 64 == 0 || (j % 2 == 0 && (j / 2 - j0 / 2) % 32 == 0)) {
        const int at = j / 2 + lane;
        page = at < p.max_pages ? p.table[plan.b * p.table_row + at] : 0;
        if (at <= (j1 - 1) / 2 && (unsigned)page >= (unsigned)p.pages && atomicCAS(p.err, 0, 103) == 0) { p.err[1] = plan.b; p.err[2] = page; }
      }
      const int where = __shfl_sync(0xffffffffu, page, (j / 2 - j0 / 2) % 32);
      for (int kv = 0; kv < 2; ++kv) {
        const int t = 2 * i + kv, slot = t % S::SLOTS;
        ok = mbar_wait(&empty[slot], (uint32_t)(((t / S::SLOTS) & 1) ^ 1), abort_flag, p.err, 321);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        if (elect_one()) {
          mbar_arrive_expect_tx(&full[slot], S::TILE);
#pragma unroll
          for (int d = 0; d < D / 64; ++d) tma_load_4d(ring + slot * S::TILE + d * SLAB, kv ? &tmap_v : &tmap_k, &full[slot], d * 64, (j % 2) * 64, hk, where);
        }
        __syncwarp();
        issued = t + 1;
      }
    }
  } else {
    // the rows of q, swizzled as the copies are
    for (int i = threadIdx.x; i < S::ROWS * (D / 8); i += 32 * S::WARPS) {
      const int r = i / (D / 8), c = i % (D / 8);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows) v = *reinterpret_cast<const uint4*>(p.q + (int64_t)(s.row0 + r / group) * p.sq_t + (int64_t)(hk * group + r % group) * p.sq_h + c * 8);
      *reinterpret_cast<uint4*>(q_smem + (c / 8) * QSLAB + r * 128 + (((c % 8) ^ (r & 7)) << 4)) = v;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * S::WARPS) : "memory");
    const int kg = warp & 3, rg = warp >> 2, lr = lane & 7, mi = lane >> 3, row_a = lane >> 2, col = (lane & 3) * 2;
    const int row0 = rg * 16 * MT;
    const uint32_t q_base = smem_u32(q_smem), ring_base = smem_u32(ring);
    auto q_frag = [&](uint32_t (&a)[4], int mt, int k) {
      const int r = row0 + mt * 16 + (mi & 1) * 8 + lr, c = 2 * k + (mi >> 1);
      ldsm4(a, q_base + (c / 8) * QSLAB + r * 128 + (((c % 8) ^ (r & 7)) << 4));
    };
    uint32_t qr[MT == 1 ? D / 16 : 1][4];
    if constexpr (MT == 1) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) q_frag(qr[k], 0, k);
    }
    float o[MT][NT][4], m[MT][2], l[MT][2];
    int last[MT][2];                                               // the last key that a row sees
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row0 + mt * 16 + h * 8 + row_a;
        m[mt][h] = -1e30f;
        l[mt][h] = 0.f;
        last[mt][h] = r < rows ? hidden + r / group : -1;
      }
    }
    bool ok = true;
    for (int j = j0; j < j1; ++j) {
      const int tk = 2 * (j - j0), sk = tk % S::SLOTS, sv = (tk + 1) % S::SLOTS;
      ok = mbar_wait(&full[sk], (uint32_t)((tk / S::SLOTS) & 1), abort_flag, p.err, 322);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      float sc[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[mt][n][e] = 0.f;
      {
        const int key = kg * 16 + (mi >> 1) * 8 + lr;
        const uint32_t base = ring_base + sk * S::TILE + key * 128;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int c = 2 * k + (mi & 1);
          uint32_t kb[4];
          ldsm4(kb, base + (c / 8) * SLAB + (((c % 8) ^ (key & 7)) << 4));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t qa[4];
            if constexpr (MT == 1) {
#pragma unroll
              for (int e = 0; e < 4; ++e) qa[e] = qr[k][e];
            } else {
              q_frag(qa, mt, k);
            }
            mma16(sc[mt][0], qa, kb[0], kb[1]);
            mma16(sc[mt][1], qa, kb[2], kb[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[sk]);
      const int key0 = j * PA_KEYS + kg * 16;
      uint32_t pa[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (key0 + 15 > hidden) {                                  // some token does not see all of these keys
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + n * 8 + col + (e & 1) > last[mt][e >> 1]) sc[mt][n][e] = -INFINITY;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(fmaxf(sc[mt][0][2 * h], sc[mt][0][2 * h + 1]), fmaxf(sc[mt][1][2 * h], sc[mt][1][2 * h + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float now = fmaxf(m[mt][h], mx * p.scale_log2);
          const float a = pa_exp2(m[mt][h] - now);
          m[mt][h] = now;
          l[mt][h] *= a;
          if (__any_sync(0xffffffffu, a != 1.f)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) { o[mt][n][2 * h] *= a; o[mt][n][2 * h + 1] *= a; }
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float e0 = pa_exp2(fmaf(sc[mt][n][2 * h], p.scale_log2, -now)), e1 = pa_exp2(fmaf(sc[mt][n][2 * h + 1], p.scale_log2, -now));
            l[mt][h] += e0 + e1;
            // probabilities meet the values as bf16, the type of the tensor cores' other operand; their sum stays in fp32
            pa[mt][2 * n + h] = pack_bf16(e0, e1);
          }
        }
      }
      ok = mbar_wait(&full[sv], (uint32_t)(((tk + 1) / S::SLOTS) & 1), abort_flag, p.err, 323);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      if (j * PA_KEYS + PA_KEYS > s.ctx) {
        // behind the last key the page may hold anything, and 0 x NaN is none: those values become zeros
        for (int r = max(s.ctx - j * PA_KEYS, kg * 16); r < kg * 16 + 16; ++r)
          for (int d = lane; d < D / 2; d += 32) *reinterpret_cast<uint32_t*>(ring + sv * S::TILE + (d / 32) * SLAB + r * 128 + (d % 32) * 4) = 0;
        __syncwarp();
      }
      {
        const int key = kg * 16 + (mi & 1) * 8 + lr;
        const uint32_t base = ring_base + sv * S::TILE + key * 128;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          const int c = 2 * n + (mi >> 1);
          uint32_t vb[4];
          ldsm4_t(vb, base + (c / 8) * SLAB + (((c % 8) ^ (key & 7)) << 4));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16(o[mt][2 * n], pa[mt], vb[0], vb[1]);
            mma16(o[mt][2 * n + 1], pa[mt], vb[2], vb[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[sv]);
    }
    // Join the key groups.  Every copy has landed and been read when all warps are here (a failed wait ends them all, and none is looked at).
    float* sums = reinterpret_cast<float*>(ring);                  // [key group][row][D]
    asm volatile("bar.sync 1, %0;" ::"n"(32 * S::WARPS) : "memory");
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row0 + mt * 16 + h * 8 + row_a;
        float x = l[mt][h];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        if ((lane & 3) == 0) ml[kg * S::ROWS + r] = make_float2(m[mt][h], x);
        if (r < rows) {
#pragma unroll
          for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(sums + (kg * S::ROWS + r) * D + n * 8 + col) = make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
        }
      }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * S::WARPS) : "memory");
    if (!*abort_flag) {
      // 8 channels a thread
      for (int i = threadIdx.x; i < rows * (D / 8); i += 32 * S::WARPS) {
        const int r = i / (D / 8), c = i % (D / 8) * 8;
        float w[4], M = -1e30f, L = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) M = fmaxf(M, ml[k * S::ROWS + r].x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = ml[k * S::ROWS + r];
          w[k] = pa_exp2(x.x - M);
          L += w[k] * x.y;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 a = *reinterpret_cast<const float4*>(sums + (k * S::ROWS + r) * D + c), e = *reinterpret_cast<const float4*>(sums + (k * S::ROWS + r) * D + c + 4);
          acc[0] += w[k] * a.x; acc[1] += w[k] * a.y; acc[2] += w[k] * a.z; acc[3] += w[k] * a.w;
          acc[4] += w[k] * e.x; acc[5] += w[k] * e.y; acc[6] += w[k] * e.z; acc[7] += w[k] * e.w;
        }
        if (plan.parts == 1) {
          const float inv = L > 0.f ? 1.f / L : 0.f;               // a token that sees nothing gets a zero row
          *reinterpret_cast<uint4*>(p.o + (int64_t)(s.row0 + r / group) * p.so_t + (int64_t)(hk * group + r % group) * p.so_h + c) =
              make_uint4(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv), pack_bf16(acc[4] * inv, acc[5] * inv), pack_bf16(acc[6] * inv, acc[7] * inv));
        } else {
          const int64_t at = ((int64_t)(plan.place + plan.part) * p.Hkv + hk) * S::ROWS + r;
          float4* to = reinterpret_cast<float4*>(out.part_o + at * D + c);
          to[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
          to[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
          if (c == 0) out.part_ml[at] = make_float2(M, L);
        }
      }
    }
  }
  __syncthreads();
  if (*abort_flag && warp == S::WARPS)                             // copies still on their way land before the block ends
    for (int t = max(0, issued - S::SLOTS); t < issued; ++t) mbar_wait(&full[t % S::SLOTS], (uint32_t)((t / S::SLOTS) & 1), abort_flag + 1, p.err, 324);
  pdl_trigger();
}

// ----------------------------------------------------------------------------- many query rows: tcgen05
// A block owns two tiles of 128 rows (a token's query heads side by side, so that a tile of 128 / group tokens shares every key of
// their KV head) and passes over the pages of its part; a page is a key tile, found through the block table.
//   warps 0-3   softmax and output of tile A, a row per thread      warps 4-7   the same for tile B
//   warp 8      TMA: both query tiles, then the pages through two slots for keys and two for values
//   warp 9      tcgen05.mma: QK_A(0) QK_B(0) | PV_A(j) QK_A(j+1) PV_B(j) QK_B(j+1) | ..., one tile's products beside the other's softmax
//   warps 10-11 complete the third warpgroup, which hands registers to the softmax (72 against 216 a thread)
// TMEM (512 columns): scores of A and B, overwritten by the probabilities as packed bf16, and both sums.  The running maximum is raised only
// when it grew by more than 2^8.  Bound: the softmax's issued instructions beside the tensor pipe.
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

constexpr int PT_THREADS = 384, PT_ROWS = 256;

template <int D>
__global__ void __launch_bounds__(PT_THREADS, 1)
paged_tiles_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                   const __grid_constant__ PagedParams p, const PagedSplit out) {
  constexpr int SLABS = D / 64, NK = 2, NV = 2, TILE = 128 * D * 2, SLAB = 128 * 128;
  constexpr uint32_t TMEM_COLS = 512;     // scores of tile t at 128 t, sums at 256 + D t
  constexpr uint32_t IDESC_QK = make_idesc_bf16(128, 128, 0, 0), IDESC_PV = make_idesc_bf16(128, D, 0, 1);
  extern __shared__ uint8_t smem_raw[];
  __shared__ int2 cache[PA_CACHE];
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
    const PagedPlan plan = paged_plan(p, tile_work, blockIdx.x, out.slots, 2, cache);
    if (lane == 0) {
      plan_s = plan;
      if (plan.b >= 0 && plan.item == 0 && plan.part == 0 && hk == 0) out.plan[plan.b] = make_int2(plan.place, plan.parts);
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
      tc_fence_after();
      const int kv0 = (j0 + j) * 128;
      uint32_t r[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_addr + c * 32, r + c * 32);
      tmem_wait_ld();
      if (kv0 + 127 > hidden + first) {           // some row does not see all of these keys
        const int lim = last - kv0;
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
      const float m_blk = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * p.scale_log2;
      float alpha = 1.f;
      bool rescale = false;
      if (j == 0) {
        m_used = m_blk;
      } else if (m_blk - m_used > 8.0f) {
        alpha = pa_exp2(m_used - m_blk);
        m_used = m_blk;
        rescale = true;
      }
      if (__any_sync(0xffffffffu, rescale)) {
        ok = mbar_wait(&o_done[t], (uint32_t)((j - 1) & 1), abort_flag, p.err, 428);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {        // narrow pieces: the 128 scores stay in registers meanwhile
          uint32_t orr[16];
          tmem_ld_32x16(o_addr + c * 16, orr);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) orr[e] = __float_as_uint(__uint_as_float(orr[e]) * alpha);
          tmem_st_32x16(o_addr + c * 16, orr);
        }
        l *= alpha;
      }
      if (kv0 + 128 > s.ctx && (t == 0 || j >= nblk[0])) {
        // Behind the last key the page may hold anything, and 0 x NaN is none: those values become zeros, by the tile whose
        // product comes first.
        ok = mbar_wait(&t_full[NK + j % NV], (uint32_t)((j / NV) & 1), abort_flag, p.err, 429);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        if (kv0 + row >= s.ctx) {
#pragma unroll
          for (int d = 0; d < SLABS * 8; ++d) *reinterpret_cast<uint4*>(v_ring + (j % NV) * TILE + (d / 8) * SLAB + row * 128 + (d % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_proxy();
      }
      // P = 2^(s c - m) as packed bf16 over the first 64 columns of S, handed over in two halves of 64 keys.  (Probabilities meet
      // the values as bf16, the type of the tensor cores' other operand; their sum stays in fp32.)
      float sum0 = 0.f, sum1 = 0.f;
      const float neg_m = -m_used;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int e = 32 * half; e < 32 * half + 32; ++e) {
          float x0, x1;
          pa_fma2(x0, x1, __uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]), p.scale_log2, neg_m);
          const float e0 = pa_exp2(x0), e1 = pa_exp2(x1);
          pa_add2(sum0, sum1, e0, e1);
          r[e] = pack_bf16(e0, e1);
        }
        tmem_st_32x32(s_addr + half * 32, r + half * 32);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[2 * t + half]);
      }
      l += sum0 + sum1;
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
      const int64_t at = (((int64_t)plan.place + (int64_t)plan.item * plan.parts + plan.part) * p.Hkv + hk) * PT_ROWS + t * 128 + row;
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

// Joins the parts of items that were cut: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.  A warp per token and head.  TILES: the
// items of the kernel above, else one item a sequence, with `part_rows` rows.
template <int D, bool TILES>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedParams p, const PagedSplit in, int part_rows) {
  constexpr int W = D / 32;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, b = blockIdx.z, h = blockIdx.y, group = p.Hq / p.Hkv, i = blockIdx.x * 8 + (threadIdx.x >> 5);
  const PagedSeq s = paged_seq(p, b);
  if (i >= s.n || (s.n * group > PA_FEW_ROWS) != TILES) return;
  const int2 plan = in.plan[b];
  if (plan.y <= 1) return;
  const int hk = h / group, per_tile = 128 / group;
  const int items = (s.n + 2 * per_tile - 1) / (2 * per_tile);
  const int64_t first = TILES ? plan.x + (int64_t)(items - 1 - i / (2 * per_tile)) * plan.y : plan.x;
  const int r = TILES ? i / per_tile % 2 * 128 + i % per_tile * group + h % group : i * group + h % group;
  auto place = [&](int k) { return ((first + k) * p.Hkv + hk) * part_rows + r; };
  float M = -1e30f;
  for (int k = lane; k < plan.y; k += 32) M = fmaxf(M, in.part_ml[place(k)].x);
  M = warp_max(M);
  float L = 0.f, acc[W] = {};
#pragma unroll 4
  for (int k = 0; k < plan.y; ++k) {
    const int64_t at = place(k);
    const float2 x = in.part_ml[at];
    if (x.y == 0.f) continue;            // nothing was seen there, and nothing written
    const float w = pa_exp2(x.x - M);
    L += w * x.y;
    const float* o = in.part_o + at * D + lane * W;
#pragma unroll
    for (int e = 0; e < W; ++e) acc[e] += w * o[e];
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  __nv_bfloat16* o = p.o + (int64_t)(s.row0 + i) * p.so_t + (int64_t)h * p.so_h + lane * W;
#pragma unroll
  for (int e = 0; e < W; e += 2) *reinterpret_cast<__nv_bfloat162*>(o + e) = __floats2bfloat162_rn(acc[e] * inv, acc[e + 1] * inv);
}

// Blocks of a head that run at a time, and room for the sums of cut items.
static int paged_split(const PagedParams& p, int ctas, int rows, PagedSplit* out) {
  out->slots = ctas / p.Hkv;
  if (out->slots < 1) out->slots = 1;
  const uint64_t places = 2 * (uint64_t)out->slots * p.Hkv * rows;
  void* scratch;
  KD_TRY(get_workspace(places * (p.D * 4 + 8) + (uint64_t)p.B * 8, &scratch));
  out->part_o = static_cast<float*>(scratch);
  out->part_ml = reinterpret_cast<float2*>(out->part_o + places * p.D);
  out->plan = reinterpret_cast<int2*>(out->part_ml + places);
  return KD_OK;
}

// [token][head][D] with a box of the query heads of `tokens` tokens on one KV head, 64 channels wide.
static int make_tmap_heads(CUtensorMap* out, const PagedParams& p, int group, int tokens) {
  const int64_t ext[4] = {1, p.T, p.Hq, p.D}, st[3] = {p.T * p.sq_t, p.sq_t, p.sq_h};
  return make_tmap_bhsd(out, p.q, ext, st, group, tokens);
}

template <int D>
static int launch_tiles(const kd_tensor* k_pool, const kd_tensor* v_pool, const PagedParams& p) {
  constexpr int SMEM = 6 * 128 * D * 2 + 1024 + 256;
  static bool configured[64] = {false};   // per device: kd_shutdown + kd_init may move the library to another GPU
  if (!configured[ctx().device & 63]) {
    KD_CUDA_CHECK(cudaFuncSetAttribute(paged_tiles_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    configured[ctx().device & 63] = true;
  }
  const int group = p.Hq / p.Hkv, per_tile = 128 / group;
  CUtensorMap tq, tk, tv;
  KD_TRY(make_tmap_heads(&tq, p, group, per_tile));
  KD_TRY(make_tmap_bhsd(&tk, p.k, k_pool->shape, k_pool->strides, 128));
  KD_TRY(make_tmap_bhsd(&tv, p.v, v_pool->shape, v_pool->strides, 128));
  PagedSplit out{};
  KD_TRY(paged_split(p, ctx().sm_count, PT_ROWS, &out));
  const int64_t blocks = out.slots + (int64_t)p.T / (2 * per_tile) + p.B;     // items of all sequences, and one more for every cut
  KD_CUDA_CHECK(launch_ex(paged_tiles_kernel<D>, dim3((unsigned)blocks, p.Hkv), dim3(PT_THREADS), (size_t)SMEM, tq, tk, tv, p, out));
  KD_TRY(after_launch("paged_tiles_kernel"));
  KD_CUDA_CHECK(launch_ex(paged_join_kernel<D, true>, dim3((p.max_query + 7) / 8, p.Hq, p.B), dim3(256), 0, p, out, PT_ROWS));
  return after_launch("paged_join_kernel");
}

template <int D, int MT, int RG>
static int launch_few(const CUtensorMap& tk, const CUtensorMap& tv, const PagedParams& p) {
  using S = FewShape<D, MT, RG>;
  static bool configured[64] = {false};   // per device: kd_shutdown + kd_init may move the library to another GPU
  if (!configured[ctx().device & 63]) {
    KD_CUDA_CHECK(cudaFuncSetAttribute(paged_few_kernel<D, MT, RG>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    configured[ctx().device & 63] = true;
  }
  PagedSplit out{};
  KD_TRY(paged_split(p, S::CTAS * ctx().sm_count, S::ROWS, &out));
  KD_CUDA_CHECK(launch_ex(paged_few_kernel<D, MT, RG>, dim3(out.slots + p.B, p.Hkv), dim3(S::THREADS), (size_t)S::SMEM, tk, tv, p, out));
  KD_TRY(after_launch("paged_few_kernel"));
  const int most = p.max_query * (p.Hq / p.Hkv) < S::ROWS ? p.max_query : S::ROWS / (p.Hq / p.Hkv);
  KD_CUDA_CHECK(launch_ex(paged_join_kernel<D, false>, dim3((most + 7) / 8, p.Hq, p.B), dim3(256), 0, p, out, S::ROWS));
  return after_launch("paged_join_kernel");
}
template <int D>
static int few_rows(const kd_tensor* k_pool, const kd_tensor* v_pool, const PagedParams& p) {
  CUtensorMap tk, tv;
  KD_TRY(make_tmap_bhsd(&tk, p.k, k_pool->shape, k_pool->strides, PA_KEYS));
  KD_TRY(make_tmap_bhsd(&tv, p.v, v_pool->shape, v_pool->strides, PA_KEYS));
  const int64_t rows = (int64_t)p.max_query * (p.Hq / p.Hkv);
  if (rows <= 16) return launch_few<D, 1, 1>(tk, tv, p);
  if (rows <= 32) return launch_few<D, 2, 1>(tk, tv, p);
  return launch_few<D, 2, 2>(tk, tv, p);
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
  if ((int64_t)p.max_query * (Hq / Hkv) > PA_FEW_ROWS) {
    KD_TRY(D == 128 ? launch_tiles<128>(k_pool, v_pool, p) : launch_tiles<64>(k_pool, v_pool, p));
    if (!q_start) return KD_OK;
  }
  return D == 128 ? few_rows<128>(k_pool, v_pool, p) : few_rows<64>(k_pool, v_pool, p);
}
