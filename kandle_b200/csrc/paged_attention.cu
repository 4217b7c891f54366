// Attention of new tokens over a paged cache: kd_attention_paged.
//
// Sequence b brings n_b new tokens (packed rows of q), whose keys and values are the last n_b of its ctx_b positions in the pages:
// token i sees positions 0 .. ctx_b - n_b + i.
//
// Tiles.  A tile of 128 rows holds the query heads that share a KV head of 128 / group tokens, a token's heads side by side; a page is a
// key tile, found through the block table.  S = Q K^T and O += P V run on tcgen05 with S, P (packed bf16) and O in tensor memory, in two
// chains of which one computes while the other waits.  An item of work is
//   a sequence of up to 128 rows: the chains take its even and odd pages, and their sums are added at the end (bound: HBM), or
//   two neighbouring tiles of a longer one: a chain each, both on every page (bound: exponentials beside the tensor pipe).
//
// Division.  The pages of all items of all KV heads stand in one row, and each of as many persistent blocks as SMs takes an equal share of it, from
// wherever it begins in one item to wherever it ends in another: long and short sequences, prompts and single tokens load every SM
// alike.  (Where items are few, whole items or equal pieces of them: paged_walk.)  An item that is cut leaves unnormalised sums, which are joined by the block that is through last if they are of one tile, else by a
// second kernel.
//
// Softmax.  A thread owns a row and loads its 128 scores at once; S is free from then on, so that the next Q K^T runs beside the exponentials
// (with P over S it waited for P V, and a chain's step was the sum of both: 4331 cycles for two tiles and a page, of which the exponential unit
// needs 2048 and the tensor pipe 2048).  Tensor memory holds one S for both chains, which they use in turn, two P and two O.  Two threads a
// row (and 16 warps) were slower: they have to exchange the maximum.  With up to 32 rows (FEW) one warp has a tile, and its instructions have to come
// for it alone: short loops over 32 scores at a time, P over S; with up to 16 rows a thread has a quarter of the scores of one or two rows, so that lanes
// without a row have no exponentials (32 single tokens: 84.1 us with a row's 128 scores in straight code, 80.3 in loops, 75.0 so).
//
// Measured: 32 single tokens on up to 6000 positions (16 heads on 8 of 128, 379 MB) 75 us, 5.1 TB/s, of which some 15 are the launch, the division,
// the blocks' change from one item to the next and the joins; 8 x 9 tokens on 9000 (32 on 8, 153 MB) 44 us; 4 x 2048 tokens on 6144 (32 on 8) 1015 us (1000 to
// 1030 from one machine to another), 948 TFLOP/s: a step of 3700 cycles, in which a softmax takes 3000 (load 440, maximum 450, exponentials 1800, store 400) and waits 600 for its S.
#include <initializer_list>
#include <type_traits>

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

constexpr int PA_ROWS = 128;            // rows of a tile
constexpr int PA_SOFTMAX = 8;           // warps 0-7: chain warp / 4, rows 32 (warp % 4) and on
constexpr int PA_THREADS = 384;
constexpr int PA_CACHE = 256;           // sequences whose lengths are kept in shared memory
constexpr int PA_PIECES = 4;            // pieces of work that the warps of a block may be apart

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

// 16 lanes x 32 columns: thread i receives, of lanes i / 4 and i / 4 + 8, columns 8 g + 2 (i % 4) and the next, as r[4 g .. 4 g + 1] and r[4 g + 2 .. 4 g + 3].
__device__ __forceinline__ void pa_ld_16x32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// 16 lanes x 16 columns: thread i has column 4 g + i % 4 of lanes i / 4 and i / 4 + 8 as r[2 g] and r[2 g + 1].
__device__ __forceinline__ void pa_st_16x16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// ----------------------------------------------------------------------------- the division of the work
// One warp goes through all of this while the others wait for it, an instruction after the other, and so with few divisions.
template <bool FEW>
struct ItemShape {
  int group, tokens;                  // query heads on a KV head, tokens of a tile
  __device__ __forceinline__ bool pair(int n) const { return !FEW && n > tokens; }
  __device__ __forceinline__ bool has(int n, int item) const { return pair(n) ? item * 2 * tokens < n : item < min(n, 1); }
  // Pages that an item's tokens see, and its units: a page of an item with two tiles counts twice, its two softmaxes take twice as long (and one
  // at least: tokens without keys get zero rows).
  __device__ __forceinline__ int pages(const PagedSeq& s, int item) const {
    const int upto = pair(s.n) ? min(s.n, (item + 1) * 2 * tokens) : s.n;
    return (max(0, s.ctx - s.n + upto) + 127) >> 7;
  }
  __device__ __forceinline__ int units(const PagedSeq& s, int item) const { return max(1, pages(s, item)) << (pair(s.n) ? 1 : 0); }
  __device__ __forceinline__ int64_t all_units(const PagedSeq& s, int& items, int& most) const {
    int64_t sum = 0;
    for (int i = 0; has(s.n, i); ++i) {
      const int u = units(s, i);
      sum += u;
      most = max(most, u);
      ++items;
    }
    return sum;
  }
};
// Items in equal pieces of at most `per` units (whole pages).
struct Pieces {
  unsigned most[2];                   // pages of a piece of one tile and of two
  uint64_t by[2];                     // 2^32 divided by them, rounded up: quotients of numbers up to 2^16 are exact
  __device__ __forceinline__ explicit Pieces(unsigned per) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      most[i] = max(1u, per >> i);
      by[i] = (uint64_t)(0xffffffffu / most[i]) + 1;
    }
  }
  template <bool FEW>
  __device__ __forceinline__ int of(const ItemShape<FEW>& shape, const PagedSeq& s, int item) const {
    const bool pair = shape.pair(s.n);
    return (int)(((max(1, shape.pages(s, item)) + (pair ? most[1] : most[0]) - 1) * (pair ? by[1] : by[0])) >> 32);
  }
  template <bool FEW>
  __device__ __forceinline__ int all(const ItemShape<FEW>& shape, const PagedSeq& s) const {
    int sum = 0;
    for (int i = 0; shape.has(s.n, i); ++i) sum += of(shape, s, i);
    return sum;
  }
};
struct CachedSeq {
  PagedSeq s;
  int64_t units;
};
__device__ __forceinline__ PagedSeq seq_of(const PagedParams& p, const CachedSeq* cache, int b) { return b < PA_CACHE ? cache[b].s : paged_seq(p, b); }
// A block's piece of an item: pages j0 .. j0 + nb - 1.
struct Piece {
  PagedSeq s;
  int b, hk, item, j0, nb;
  int parts, part, first;             // parts of the whole item, this one's number, the block of the first one
  bool pair;
  // pages of the two chains
  template <bool FEW>
  __device__ __forceinline__ void tiles(const ItemShape<FEW>& shape, int (&n)[2]) const {
    n[0] = (nb + 1) / 2;
    n[1] = nb / 2;
    if (!pair) return;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int token0 = (2 * item + t) * shape.tokens, keys = token0 >= s.n ? 0 : max(0, s.ctx - s.n + min(s.n, token0 + shape.tokens));
      n[t] = min(max((keys + 127) / 128 - j0, 0), nb);
    }
  }
};
// Goes through the pieces of a block: units u .. end - 1 of a row of fewer than 2^31, `per` a block; or the one piece `part` of `parts` that begins
// at `off` of its item and has up to `end` units.
struct Walk {
  unsigned u, end, per;
  int b, hk, item, off, block, parts, part;
  template <bool FEW>
  __device__ __forceinline__ bool next(const PagedParams& p, const ItemShape<FEW>& shape, const CachedSeq* cache, Piece& w) {
    if (u >= end) return false;
    for (;;) {
      if (b == p.B) { b = 0; ++hk; }
      if (hk == p.Hkv) return false;
      w.s = seq_of(p, cache, b);
      if (shape.has(w.s.n, item)) break;
      ++b;
      item = 0;
    }
    w.pair = shape.pair(w.s.n);
    const int pages = shape.pages(w.s, item), twice = w.pair ? 1 : 0, all = max(1, pages) << twice;
    const int take = min(all - off, (int)(end - u));
    const unsigned start = u - off;
    w.b = b; w.hk = hk; w.item = item;
    w.j0 = min(off >> twice, pages);
    w.nb = min((off + take) >> twice, pages) - w.j0;
    if (parts) {
      w.first = block - part;
      w.parts = parts;
      u = end;
    } else {
      w.first = off ? (int)(start / per) : block;
      w.parts = (start + all <= end ? block : (int)((start + all - 1) / per)) - w.first + 1;
      u += take;
    }
    w.part = block - w.first;
    off = 0;
    ++item;
    return true;
  }
};
// A cut in units: what the partial sums and the join of an item cost beside a page, with few rows and with more; and what a second item costs a block.
constexpr unsigned PA_CUT_FEW = 2, PA_CUT = 10, PA_SECOND = 4;

// Block x's share, by one warp: an equal share of all units, wherever that cuts an item; or, where there are no more items than blocks, an item or
// an equal piece of one, if the longest share is then longer by no more than what a cut or a second item costs (8 KV heads of 128, in a graph: 16 single
// tokens on 1000 positions 22.8 us in equal shares, 18.8 as whole items; 30 tokens on 900 29.3 and 21.7; 4 x 200 on 600 36.6 and 24.9; one token
// on 700, which is cut either way, 12.9 and 13.4: the choice itself).
template <bool FEW>
__device__ __forceinline__ Walk paged_walk(const PagedParams& p, const ItemShape<FEW>& shape, int x, int blocks, CachedSeq* cache) {
  constexpr unsigned ALL = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  uint64_t own = 0;
  int items = 0, most = 0;
  for (int b = lane; b < p.B; b += 32) {
    const PagedSeq s = paged_seq(p, b);
    const int64_t n = shape.all_units(s, items, most);
    if (b < PA_CACHE) cache[b] = CachedSeq{s, n};
    own += n;
  }
  __syncwarp();
  own = min(own, (uint64_t)1 << 42);
  items = min(items, 1 << 20);
  const uint64_t sum64 = ((uint64_t)__reduce_add_sync(ALL, (unsigned)(own >> 16)) << 16) + __reduce_add_sync(ALL, (unsigned)(own & 0xffff));
  Walk w;
  w.u = w.end = 0;
  w.per = 1;
  w.hk = w.b = w.item = w.off = w.parts = w.part = 0;
  w.block = x;
  if (sum64 * p.Hkv >= 0x80000000u) {
    if (lane == 0 && atomicCAS(p.err, 0, 107) == 0) { p.err[1] = (int)(sum64 >> 31); p.err[2] = (int)(sum64 & 0x7fffffff); }
    return w;
  }
  unsigned sum = (unsigned)sum64;
  const unsigned all = sum * p.Hkv;
  w.per = max(1u, (all + blocks - 1) / blocks);
  unsigned one = 0;                                  // one piece a block, of up to so many units
  const unsigned longest = __reduce_max_sync(ALL, most);
  if ((uint64_t)__reduce_add_sync(ALL, items) * p.Hkv <= blocks && longest < 32768) {
    // a lane tries one of up to eight lengths with a quarter of the sequences
    const unsigned more = min((unsigned)lane & 7, PA_SECOND), per = longest <= w.per + more + (FEW ? PA_CUT_FEW : PA_CUT) ? longest : w.per + more;
    const Pieces cut(per);
    int n = 0;
    for (int b = lane >> 3; b < p.B; b += 4) n += cut.all(shape, seq_of(p, cache, b));
    n += __shfl_xor_sync(ALL, n, 8);
    n += __shfl_xor_sync(ALL, n, 16);
    const unsigned fits = __ballot_sync(ALL, n * p.Hkv <= blocks);
    if (fits) {
      one = __shfl_sync(ALL, per, __ffs(fits) - 1);
      sum = __shfl_sync(ALL, n, __ffs(fits) - 1);
    }
  }
  const Pieces cut(max(1u, one));
  unsigned left;
  if (one) {
    if (x >= (int)(sum * p.Hkv)) return w;
    left = x;
  } else {
    w.u = (unsigned)min((uint64_t)all, (uint64_t)x * w.per);
    w.end = min(all, w.u + w.per);
    if (w.u >= w.end) return w;
    left = w.u;
  }
  w.hk = (int)(left / sum);
  left -= w.hk * sum;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + lane;
    unsigned n = 0;
    if (b < p.B) {
      int i = 0, m = 0;
      n = one ? cut.all(shape, seq_of(p, cache, b)) : (unsigned)(b < PA_CACHE ? cache[b].units : shape.all_units(paged_seq(p, b), i, m));
    }
    unsigned upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(ALL, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned hit = __ballot_sync(ALL, upto > left);
    if (hit) {
      const int who = __ffs(hit) - 1;
      w.b = b0 + who;
      left -= __shfl_sync(ALL, upto - n, who);
      break;
    }
    left -= __shfl_sync(ALL, upto, 31);
  }
  const PagedSeq s = seq_of(p, cache, w.b);
  if (!one) {
    for (; left >= (unsigned)shape.units(s, w.item); ++w.item) left -= shape.units(s, w.item);
    w.off = (int)left;
    return w;
  }
  for (; left >= (unsigned)cut.of(shape, s, w.item); ++w.item) left -= cut.of(shape, s, w.item);
  w.parts = cut.of(shape, s, w.item);
  w.part = (int)left;
  const int size = (max(1, shape.pages(s, w.item)) + w.parts - 1) / w.parts << (shape.pair(s.n) ? 1 : 0);
  w.off = w.part * size;
  w.end = size;
  return w;
}

// ----------------------------------------------------------------------------- sums of items that are cut
// Block x leaves the end of an item that began before it at place 2 x, and the beginning of one that goes on behind it at 2 x + 1.
struct PagedSplit {
  float* part_o;      // [place][rows][D] unnormalised sums, or [place][D / 4][rows][4] of items with two tiles
  float2* part_ml;    // [place][rows] (running maximum in the log2 domain, sum)
  int4* cut;          // what of two tiles began in block x and went on: (sequence, KV head, item, parts)
};
// Parts of a cut item that are through, by its first block; the last one sets it back.
constexpr int PA_BLOCKS = 1024;
static __device__ unsigned g_paged_through[PA_BLOCKS];

// Where the four channels from c on of a row stand in a place, in float4s.  A thread has a row: with two tiles' 256 rows whole warps store, in one
// piece if rows stand side by side (1 x 512 tokens on 16384: 96.3 -> 93.1 us); of few rows, the channels are read side by side (8 x 9 tokens:
// 57.5 us with rows side by side, 53.5 so).
template <int D>
__device__ __forceinline__ int part_at(bool pair, int r, int c) { return pair ? c / 4 * (2 * PA_ROWS) + r : r * (D / 4) + c / 4; }
// Four channels of a row of an item's parts: sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k.
struct JoinedRow {
  float m = -1e30f, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float2 x, float4 o) {
    const float now = fmaxf(m, x.x), f0 = pa_exp2(m - now), f1 = pa_exp2(x.x - now);
    const bool some = x.y != 0.f;        // (else nothing was seen there, and nothing written)
    m = now;
    l = l * f0 + (some ? x.y * f1 : 0.f);
    acc.x = acc.x * f0 + (some ? o.x * f1 : 0.f); acc.y = acc.y * f0 + (some ? o.y * f1 : 0.f);
    acc.z = acc.z * f0 + (some ? o.z * f1 : 0.f); acc.w = acc.w * f0 + (some ? o.w * f1 : 0.f);
  }
  __device__ __forceinline__ void put(__nv_bfloat16* to) const {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  }
};
// The place of part k of an item that began in block `first`.
__device__ __forceinline__ int64_t part_place(int first, int k) { return 2 * (int64_t)(first + k) + (k == 0 ? 1 : 0); }

// ----------------------------------------------------------------------------- the kernel
// FEW: no sequence has more than 32 rows; queries of two items and more pages fit, and a warp of its own writes the outputs.
//   warps 0-7   softmax (and outputs)
//   warp 8      FEW: outputs
//   warp 9      division; TMA: queries, then pages through rings of keys and of values
//   warps 10-11 tcgen05.mma: scores, products
template <int D, bool FEW>
struct PagedShape {
  static constexpr int TILE = 128 * D * 2, RING = (FEW ? 3 : 2) * 32768 / TILE;      // slots for keys, and as many for values
  static constexpr int QROWS = FEW ? 32 : PA_ROWS, Q_BYTES = QROWS * D * 2;
  static constexpr int Q_AT = 0, RING_AT = 2 * Q_BYTES, BARS_AT = RING_AT + 2 * RING * TILE;
  static constexpr int CACHE_AT = BARS_AT + 1024, ML_AT = CACHE_AT + PA_CACHE * (int)sizeof(CachedSeq), BYTES = ML_AT + 2 * 2 * PA_ROWS * 8;
  // tensor memory: scores, probabilities, sums
  // (FEW: scores of each chain, with the probabilities over them.  Else one buffer for the scores of both chains.  With heads of 64 there is room
  // for two; the chains' softmaxes then run side by side, both at their exponentials and both not, and a step takes 4400 cycles in place of
  // 4000: 73.8 us against 71.0 in a batch of 12 x 700 tokens.)
  static constexpr uint32_t S_STEP = FEW ? 128 : 0, P_COL = FEW ? 0 : 128, P_STEP = FEW ? 128 : 64, O_COL = 256;
  static_assert(O_COL + 2 * D <= 512, "tensor memory has 512 columns");
  // registers of a thread of warps 8-11 and of the others, which hold 128 scores (FEW: 32, and all have what they were launched with)
  static constexpr int OTHER_REGS = 72, SOFTMAX_REGS = 216;
  static_assert((PA_THREADS - PA_SOFTMAX * 32) * OTHER_REGS + PA_SOFTMAX * 32 * SOFTMAX_REGS <= PA_THREADS * 168, "registers of the launch");
  static constexpr int SMEM = BYTES + 1024;
  static_assert(SMEM <= 227 * 1024, "tiles exceed shared memory");
};

template <int D, bool FEW>
__global__ void __launch_bounds__(PA_THREADS, 1)
paged_attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                       const __grid_constant__ PagedParams p, const PagedSplit out) {
  using S = PagedShape<D, FEW>;
  constexpr int SLABS = D / 64, TILE = S::TILE, RING = S::RING, SLAB = 128 * 128, QROWS = S::QROWS, QSLAB = QROWS * 128, Q_BYTES = S::Q_BYTES;
  constexpr uint32_t S_STEP = S::S_STEP, P_COL = S::P_COL, P_STEP = S::P_STEP, O_COL = S::O_COL;
  constexpr uint32_t IDESC_QK = make_idesc_bf16(128, 128, 0, 0), IDESC_PV = make_idesc_bf16(128, D, 0, 1);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *q_smem = smem + S::Q_AT, *ring = smem + S::RING_AT;      // (an MMA reads 128 rows: what follows stands in for missing ones)
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BARS_AT);
  uint64_t *q_full = bars, *q_empty = bars + 2, *s_full = bars + 4, *s_free = bars + 8;      // scores are there [chain], have been loaded
  uint64_t *p_ready = bars + 12, *o_done = bars + 14, *o_free = bars + 16, *few_done = bars + 17, *y_bar = bars + 18;      // y_bar: sums of the two chains are there [quarter]
  uint64_t *full = bars + 26, *empty = full + 2 * RING;      // up to 12 each
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 50);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);      // and behind it one that stays 0
  int* joins = const_cast<int*>(abort_flag) + 2;                                  // items that this block joins at the end
  uint64_t *piece_full = bars + 52, *piece_empty = piece_full + PA_PIECES;
  Piece* piece_s = reinterpret_cast<Piece*>(piece_empty + PA_PIECES);             // what the warps work on; no parts: behind the last one
  Piece* join_s = piece_s + PA_PIECES;                                            // [2]
  static_assert((52 + 2 * PA_PIECES) * 8 + (PA_PIECES + 2) * sizeof(Piece) <= 1024, "barriers and what stands behind them");
  CachedSeq* cache = reinterpret_cast<CachedSeq*>(smem + S::CACHE_AT);
  float2* ml = reinterpret_cast<float2*>(smem + S::ML_AT);     // [piece & 1][chain][row] (maximum, sum)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const ItemShape<FEW> shape{p.Hq / p.Hkv, QROWS / (p.Hq / p.Hkv)};
  const int group = shape.group;

  // The copying warp sets up the barriers and goes on; the others meet it at a barrier that it only arrives at.
  if (warp == 9) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); mbar_init(&p_ready[i], 4); mbar_init(&o_done[i], 1); mbar_init(&s_full[i], 1); }
      mbar_init(s_free, 4);
      for (int i = 0; i < 4; ++i) mbar_init(&y_bar[i], 2);
      mbar_init(o_free, FEW ? 1 : PA_SOFTMAX);
      mbar_init(few_done, 2);
      for (int i = 0; i < 2 * RING; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
      for (int i = 0; i < PA_PIECES; ++i) { mbar_init(&piece_full[i], 1); mbar_init(&piece_empty[i], PA_SOFTMAX + 2 + (FEW ? 1 : 0)); }
      abort_flag[0] = abort_flag[1] = 0;
      *joins = 0;
      fence_mbar_init();
      prefetch_tmap(&tmap_q);
      prefetch_tmap(&tmap_k);
      prefetch_tmap(&tmap_v);
    }
    __syncwarp();
    asm volatile("bar.arrive 3, %0;" ::"n"(PA_THREADS) : "memory");
  } else {
    if (warp == 10) {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
      tc_fence_before();
    }
    asm volatile("bar.sync 3, %0;" ::"n"(PA_THREADS) : "memory");
  }
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, warp == 9 ? 0u : *tmem_slot, 0);      // (warp 9 may be ahead of it)  S at 0, P of chain t at P_COL + 64 t, O at O_COL + D t
  pdl_wait();
  if (warp == 10) pdl_trigger();              // after the TMEM allocation (see common.cuh): one thread's is the block's
  if (!FEW && threadIdx.x == 0) out.cut[blockIdx.x] = make_int4(0, 0, 0, 0);      // (thread 0 writes what is cut, too)
  int issued[2] = {0, 0}, q_loaded = 0;       // pages' keys and values and items' queries asked for, by the copying warp
  auto mbar_test = [](uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done != 0;
  };
  // As wait, asking without pause for a while: a step of the chains' loop hangs on it.
  auto wait_soon = [&](uint64_t* bar, uint32_t parity, int code) {
    bool ok = false;
    for (int spins = 0; !ok && spins < 4096; ++spins) ok = __all_sync(0xffffffffu, mbar_test(bar, parity));
    return ok || (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.err, code));
  };
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.err, code)); };
  // The k-th piece of the block's share, and that the warp is done with it.  nullptr: there are no more, or a wait ran out.
  auto piece_at = [&](int k) -> const Piece* {
    if (!wait(&piece_full[k % PA_PIECES], (uint32_t)((k / PA_PIECES) & 1), 341)) return nullptr;
    return piece_s[k % PA_PIECES].parts ? piece_s + k % PA_PIECES : nullptr;
  };
  auto piece_done = [&](int k) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&piece_empty[k % PA_PIECES]);
  };
  // A warp's part of a cut item is written.  The last of all its parts' warps leaves the item to be joined at the end of its block (in the parts'
  // order, whoever is last).
  auto part_through = [&](const Piece& w, int warps) {
    unsigned before;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(&g_paged_through[w.first]) : "memory");
    if (before == (unsigned)(w.parts * warps) - 1) {
      g_paged_through[w.first] = 0;
      join_s[atomicAdd(joins, 1)] = w;
    }
  };
  // Descriptors and addresses pass through a shuffle, which tells the compiler that they are alike in a warp: what was made of numbers read from memory
  // went through vector registers for every MMA and took 85 cycles each, whatever its size.
  auto uniform_desc = [](uint32_t addr, uint32_t lbo) { return make_smem_desc_sw128(__shfl_sync(0xffffffffu, addr, 0), lbo, 1024); };
  // where the outputs of a tile's row go
  auto out_row = [&](const PagedSeq& s, int hk, int token, int r) { return p.o + (int64_t)(s.row0 + token) * p.so_t + (int64_t)(hk * group + r % group) * p.so_h; };

  if (warp >= PA_SOFTMAX) {
  if constexpr (!FEW) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::OTHER_REGS));
  if (warp == 9) {
    // This warp alone goes through the division: its state does not fit beside the others' registers, and each began a piece some 4000 cycles late.
    Walk walk = paged_walk(p, shape, blockIdx.x, gridDim.x, cache);
    int page_first = 0;                                             // the next piece's first 32 entries of the table
    auto publish = [&](int k) {
      Piece w;
      const bool more = walk.next(p, shape, cache, w);
      if (!more) w.parts = w.nb = 0;
      if (!wait(&piece_empty[k % PA_PIECES], (uint32_t)(((k / PA_PIECES) & 1) ^ 1), 342)) return false;
      if (lane == 0) {
        piece_s[k % PA_PIECES] = w;
        mbar_arrive(&piece_full[k % PA_PIECES]);
      }
      __syncwarp();
      if (lane < w.nb) page_first = p.table[w.b * p.table_row + w.j0 + lane];
      return true;
    };
    bool ok = publish(0);
    for (int k = 0; ok; ++k) {
      const Piece w = piece_s[k % PA_PIECES];
      if (!w.parts) break;
      if (w.nb == 0) {
        ok = publish(k + 1);
        continue;
      }
      int page = 0, page_next = page_first;                         // entries of the table, 32 at a time
      // queries: one item's two tiles, or FEW: two items' one tile
      const int qb = FEW ? q_loaded & 1 : 0;
      if (!wait(&q_empty[qb], (uint32_t)(((FEW ? q_loaded >> 1 : q_loaded) & 1) ^ 1), 321)) break;
      const int tiles = w.pair ? 2 : 1, token0 = w.s.row0 + (w.pair ? w.item * 2 * shape.tokens : 0);
      if (elect_one()) {
        mbar_arrive_expect_tx(&q_full[qb], tiles * SLABS * shape.tokens * group * 128);
        for (int t = 0; t < tiles; ++t)
#pragma unroll
          for (int d = 0; d < SLABS; ++d)
            tma_load_4d(q_smem + (qb + t) * Q_BYTES + d * QSLAB, &tmap_q, &q_full[qb], d * 64, w.hk * group, token0 + t * shape.tokens, 0);
      }
      __syncwarp();
      ++q_loaded;
      // What is read behind the copies waits for them (three pages of them take some 8000 cycles): the next piece's entries come before them.
      if (!(ok = publish(k + 1))) break;
      for (int j = 0; j < w.nb; ++j) {
        if (j % 32 == 0) {
          page = j + lane < w.nb ? page_next : 0;
          if (j + 32 + lane < w.nb) page_next = p.table[w.b * p.table_row + w.j0 + j + 32 + lane];
          if ((unsigned)page >= (unsigned)p.pages && atomicCAS(p.err, 0, 103) == 0) { p.err[1] = w.b; p.err[2] = page; }
        }
        const int where = __shfl_sync(0xffffffffu, page, j % 32);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int slot = v * RING + issued[v] % RING;
          if (!(ok = wait(&empty[slot], (uint32_t)(((issued[v] / RING) & 1) ^ 1), 322))) break;
          if (elect_one()) {
            mbar_arrive_expect_tx(&full[slot], TILE);
#pragma unroll
            for (int d = 0; d < SLABS; ++d) tma_load_4d(ring + slot * TILE + d * SLAB, v ? &tmap_v : &tmap_k, &full[slot], d * 64, 0, w.hk, where);
          }
          __syncwarp();
          ++issued[v];
        }
        if (!ok) break;
      }
    }
  } else if (warp == 10) {
    // Scores: S_t = Q_t K(g)^T in the order of pages and chains.  (A warp for the scores and one for the products: a wait takes some 200 cycles
    // beside the operands that the tensor pipe reads from shared memory, and with ten waits and 32 MMAs for two tiles and a page one
    // warp took 5700 cycles, more than the softmax.  One warp for each chain would not see every phase of the barriers that it waits for.)
    bool ok = true;
    int page = 0, q_done = 0, tiles[2] = {0, 0};                // pages, items with keys, tiles of scores
    for (int k = 0; ok; ++k) {
      const Piece* at = piece_at(k);
      if (!at) break;
      const Piece w = *at;
      piece_done(k);
      if (w.nb == 0) continue;
      const int qb = FEW ? q_done & 1 : 0;
      const bool pair = !FEW && w.pair;
      int n[2];
      w.tiles(shape, n);
      if (!(ok = wait_soon(&q_full[qb], (uint32_t)((FEW ? q_done >> 1 : q_done) & 1), 324))) break;
#pragma unroll 1
      for (int g = 0; ok && g < w.nb; ++g, ++page) {
        const int slot = page % RING;
        if (!(ok = wait_soon(&full[slot], (uint32_t)((page / RING) & 1), 325))) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (pair ? g >= n[t] : (g & 1) != t) continue;
          const uint64_t qdesc = uniform_desc(smem_u32(q_smem + (qb + (pair ? t : 0)) * Q_BYTES), 16), kdesc = uniform_desc(smem_u32(ring + slot * TILE), 16);
          // the scores before have been loaded (FEW: and the probabilities in their place used)
          if (FEW) ok = tiles[t] == 0 || wait_soon(&o_done[t], (uint32_t)((tiles[t] - 1) & 1), 340);
          else ok = tiles[0] == 0 || wait_soon(s_free, (uint32_t)((tiles[0] - 1) & 1), 340);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              umma_ss(tmem_base + (uint32_t)t * S_STEP, qdesc + ((uint32_t)((k / 4) * QSLAB + (k % 4) * 32) >> 4), kdesc + ((uint32_t)((k / 4) * SLAB + (k % 4) * 32) >> 4), IDESC_QK,
                      k != 0 ? 1u : 0u);
            umma_commit(&s_full[t]);
          }
          __syncwarp();
          if (!ok) break;
          ++tiles[FEW ? t : 0];
        }
        if (!ok) break;
        if (elect_one()) {
          umma_commit(&empty[slot]);
          if (g + 1 == w.nb) umma_commit(&q_empty[qb]);
        }
        __syncwarp();
      }
      ++q_done;
    }
  } else if (warp == 11) {
    // Products: O_t += P_t V(g), in the same order.
    bool ok = true;
    int page = 0, q_done = 0, turn[2] = {0, 0};      // pages, items with keys, tiles of a chain
    for (int k = 0; ok; ++k) {
      const Piece* at = piece_at(k);
      if (!at) break;
      const Piece w = *at;
      piece_done(k);
      if (w.nb == 0) continue;
      const bool pair = !FEW && w.pair;
      int n[2];
      w.tiles(shape, n);
      // the sums of the piece before have been read
      if (q_done > 0 && !(ok = wait_soon(o_free, (uint32_t)((q_done - 1) & 1), 328))) break;
#pragma unroll 1
      for (int g = 0; ok && g < w.nb; ++g, ++page) {
        const int slot = RING + page % RING;
        if (!(ok = wait_soon(&full[slot], (uint32_t)((page / RING) & 1), 326))) break;
#pragma unroll
        for (int t = 0; ok && t < 2; ++t) {
          if (pair ? g >= n[t] : (g & 1) != t) continue;
          const uint64_t vdesc = uniform_desc(smem_u32(ring + slot * TILE), SLAB);
          const uint32_t more = __shfl_sync(0xffffffffu, (pair ? g : g >> 1) != 0 ? 1u : 0u, 0);
          if (!(ok = wait_soon(&p_ready[t], (uint32_t)(turn[t] & 1), 327))) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              umma_ts(tmem_base + O_COL + (uint32_t)(t * D), tmem_base + P_COL + (uint32_t)t * P_STEP + (uint32_t)(k * 8), vdesc + (uint32_t)(k * 128), IDESC_PV, k != 0 ? 1u : more);
            umma_commit(&o_done[t]);
          }
          __syncwarp();
          ++turn[t];
        }
        if (!ok) break;
        if (elect_one()) umma_commit(&empty[slot]);
        __syncwarp();
      }
      ++q_done;
    }
  } else if (FEW && warp == 8) {
    // Outputs of pieces with up to 32 rows, while the chains go on.
    int pieces = 0, turns[2] = {0, 0};
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const Piece* piece = piece_at(k);
      if (!piece) break;
      const Piece w = *piece;
      piece_done(k);
      const int rows = w.s.n * group;
      const bool real = lane < rows, direct = w.parts == 1;
      float f[2] = {0.f, 0.f}, M = -1e30f, L = 0.f;
      const bool use[2] = {w.nb > 0, w.nb > 1};
      if (w.nb > 0) {
        if (!(ok = wait(few_done, (uint32_t)(pieces & 1), 337))) break;
        const float2* now = ml + (pieces & 1) * 2 * PA_ROWS;
        const float2 a = now[lane], b = now[PA_ROWS + lane];
        M = fmaxf(a.x, b.x);
        f[0] = a.y == 0.f ? 0.f : pa_exp2(a.x - M);
        f[1] = b.y == 0.f ? 0.f : pa_exp2(b.x - M);
        L = f[0] * a.y + f[1] * b.y;
        if (direct) {
          const float inv = L == 0.f ? 0.f : 1.f / L;
          f[0] *= inv;
          f[1] *= inv;
        }
        turns[0] += (w.nb + 1) / 2;
        turns[1] += w.nb / 2;
        if (!(ok = wait(&o_done[0], (uint32_t)((turns[0] - 1) & 1), 338))) break;
        if (w.nb > 1 && !(ok = wait(&o_done[1], (uint32_t)((turns[1] - 1) & 1), 338))) break;
        tc_fence_after();
      }
      __nv_bfloat16* to = real ? out_row(w.s, w.hk, lane / group, lane) : nullptr;
      const int64_t at = (int64_t)(2 * blockIdx.x + (w.part == 0 ? 1 : 0)) * QROWS + lane;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t x[64];
        __syncwarp();
        if (use[0]) tmem_ld_32x32(tmem_base + O_COL + c, x);
        if (use[1]) tmem_ld_32x32(tmem_base + O_COL + D + c, x + 32);
        tmem_wait_ld();
        if (c + 32 == D && w.nb > 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(o_free);
        }
        if (!real) continue;
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float o[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            o[k] = f[0] == 0.f ? 0.f : f[0] * __uint_as_float(x[e + k]);
            if (f[1] != 0.f) o[k] = fmaf(f[1], __uint_as_float(x[32 + e + k]), o[k]);
          }
          if (direct) {
            *reinterpret_cast<uint4*>(to + c + e) = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
          } else {
            float4* part = reinterpret_cast<float4*>(out.part_o + at * D + c + e);
            part[0] = make_float4(o[0], o[1], o[2], o[3]);
            part[1] = make_float4(o[4], o[5], o[6], o[7]);
          }
        }
      }
      if (real && !direct) out.part_ml[at] = make_float2(M, L);
      __syncwarp();
      if (w.nb > 0) ++pieces;
      if (!direct && lane == 0) part_through(w, 1);
      __syncwarp();
    }
  }
  } else {
    if constexpr (!FEW) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::SOFTMAX_REGS));
    const int t = warp >> 2, q = warp & 3, row = q * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16), s_addr = lane_addr + (uint32_t)t * S_STEP, p_addr = lane_addr + P_COL + (uint32_t)t * P_STEP, o_addr = lane_addr + O_COL + (uint32_t)(t * D);
    const int row_token = row / group, slim_token1 = FEW ? (lane >> 2) / group : 0, slim_token2 = FEW ? ((lane >> 2) + 8) / group : 0;
    int done = 0, pieces = 0, turns[2] = {0, 0}, y_turn = 0;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const Piece* piece = piece_at(k);
      if (!piece) break;
      const Piece& w = *piece;                                      // (not copied: the registers are for scores)
      const bool pair = !FEW && w.pair;
      // this chain's tile
      const int token0 = pair ? (2 * w.item + t) * shape.tokens : 0, tokens = min(shape.tokens, w.s.n - token0), rows = tokens * group;
      const int hidden = w.s.ctx - w.s.n + token0;                  // keys 0 .. hidden + i are seen by the tile's token i
      const bool active = q * 32 < rows, real = row < rows;
      const int last = real ? hidden + row_token : -1;
      int n[2];
      w.tiles(shape, n);
      const int mine = t ? n[1] : n[0];
      int my_turn = t ? turns[1] : turns[0];
      float m = -1e30f, l = 0.f;
      // FEW, up to 16 rows: a thread has a quarter of the columns of rows lane / 4 and lane / 4 + 8 (whose statistics are m2 and l2)
      const bool slim = FEW && rows <= 16;
      const int last1 = (lane >> 2) < rows ? hidden + slim_token1 : -1, last2 = (lane >> 2) + 8 < rows ? hidden + slim_token2 : -1;
      float m2 = -1e30f, l2 = 0.f;
      // P, and values that were cleared, are there for the product
      auto hand_over = [&] {
        if (active) tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[t]);
      };
      for (int i = 0; i < mine; ++i, ++my_turn) {
        const int g = pair ? i : 2 * i + t, kv0 = (w.j0 + g) * 128;
        const bool masked = kv0 + 127 > hidden;                     // some row does not see all of these keys
        const int lim = last - kv0;
        float mx0 = -1e30f, mx1 = -1e30f, mx2 = -1e30f, mx3 = -1e30f, alpha = 1.f, neg_m = 0.f, sum0 = 0.f, sum1 = 0.f;
        bool rescale = false;
        // The maximum is raised only when it grew by more than 2^8: the sum uses the same one, so nothing is lost.
        auto raise = [&] {
          const float m_blk = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * p.scale_log2;
          if (i == 0 || !real) {                                    // (nobody reads a padding row)
            m = m_blk;
          } else if (m_blk - m > 8.0f) {
            alpha = pa_exp2(m - m_blk);
            m = m_blk;
            rescale = true;
          }
          neg_m = -m;
        };
        auto rescale_sums = [&] {
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {                     // narrow pieces: the scores stay in registers meanwhile
            uint32_t o[16];
            tmem_ld_32x16(o_addr + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st_32x16(o_addr + c, o);
          }
        };
        // Behind the last key a page may hold anything, and 0 x NaN is none: those values become zeros before a product reads them (by
        // the chain whose product comes first).
        auto clear_values = [&] {
          // (what stood in the slot before has been used, so that the parity is that of this page)
          if (i == 0 && pieces > 0 && !wait(o_free, (uint32_t)((pieces - 1) & 1), 333)) return false;
          const int slot = RING + (done + g) % RING;
          if (!wait(&full[slot], (uint32_t)(((done + g) / RING) & 1), 330)) return false;
          if (kv0 + row >= w.s.ctx) {
#pragma unroll
            for (int d = 0; d < D / 8; ++d) *reinterpret_cast<uint4*>(ring + slot * TILE + (d / 8) * SLAB + row * 128 + (d % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async_proxy();
          return true;
        };
        const bool unclean = kv0 + 128 > w.s.ctx && (!pair || t == 0 || i >= n[0]);
        if constexpr (FEW) {
          // One warp works on a tile here, and straight code for 128 scores comes to it at a few cycles an instruction (5300 a tile, with eight warps 3300):
          // short loops over 32 scores, which are read twice.  S of this chain is overwritten by P, and its next Q K^T waits for P V.
          if (!(ok = wait(&s_full[t], (uint32_t)(my_turn & 1), 329))) break;
          tc_fence_after();
          if (active) {
            // columns that no row of the tile, and that not every row sees, in whole 32s
            const int columns = min(128, (hidden - kv0 + w.s.n - 1) / 32 * 32 + 32), clear = hidden - kv0 - 31;
            auto mask = [&](int c, uint32_t* r) {
              if (c <= clear) return;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (e > lim - c) r[e] = __float_as_uint(-1e30f);
            };
            auto largest = [&](int c, uint32_t* r) {
              mask(c, r);
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                mx0 = pa_max3(mx0, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
                mx1 = pa_max3(mx1, __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
                mx2 = pa_max3(mx2, __uint_as_float(r[e + 4]), __uint_as_float(r[e + 5]));
                mx3 = pa_max3(mx3, __uint_as_float(r[e + 6]), __uint_as_float(r[e + 7]));
              }
            };
            auto exponentials = [&](int c, uint32_t* r) {
              mask(c, r);
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                float x0, x1;
                pa_fma2(x0, x1, __uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]), p.scale_log2, neg_m);
                const float e0 = pa_exp2(x0), e1 = pa_exp2(x1);
                pa_add2(sum0, sum1, e0, e1);
                r[e] = pack_bf16(e0, e1);
              }
              tmem_st_32x16(p_addr + c / 2, r);
            };
            auto columns_by = [&](auto&& work) {
#pragma unroll 1
              for (int c = 0; c < columns; c += 32) {
                uint32_t r[32];
                tmem_ld_32x32(s_addr + c, r);
                tmem_wait_ld();
                work(c, r);
              }
            };
            // As above for up to 16 rows, TWO: more than 8.
            auto slim_tile = [&](auto two) {
              constexpr bool TWO = decltype(two)::value;
              const int lim1 = last1 - kv0 - 2 * (lane & 3), lim2 = last2 - kv0 - 2 * (lane & 3);
              float x[2][2] = {{-1e30f, -1e30f}, {-1e30f, -1e30f}}, sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}}, alpha2 = 1.f;
              auto slim_mask = [&](int c, uint32_t* r) {
                if (c <= clear) return;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  if (e % 4 < 2 && 8 * (e / 4) + e % 2 > lim1 - c) r[e] = __float_as_uint(-1e30f);
                  if (TWO && e % 4 >= 2 && 8 * (e / 4) + e % 2 > lim2 - c) r[e] = __float_as_uint(-1e30f);
                }
              };
#pragma unroll 1
              for (int c = 0; c < columns; c += 32) {
                uint32_t r[16];
                pa_ld_16x32(s_addr + c, r);
                tmem_wait_ld();
                slim_mask(c, r);
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                  x[0][e / 4 % 2] = pa_max3(x[0][e / 4 % 2], __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
                  if (TWO) x[1][e / 4 % 2] = pa_max3(x[1][e / 4 % 2], __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
                }
              }
              auto slim_raise = [&](float (&y)[2], bool some, float& m, float& alpha) {
                float now = fmaxf(y[0], y[1]);
                now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 1));
                now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 2)) * p.scale_log2;
                if (i == 0 || !some) {
                  m = now;
                } else if (now - m > 8.0f) {
                  alpha = pa_exp2(m - now);
                  m = now;
                  rescale = true;
                }
              };
              slim_raise(x[0], last1 >= 0, m, alpha);
              if (TWO) slim_raise(x[1], last2 >= 0, m2, alpha2);
              if (__any_sync(0xffffffffu, rescale)) {
                l *= alpha;
                l2 *= alpha2;
                const float a1 = __shfl_sync(0xffffffffu, alpha, (lane & 7) * 4), a2 = __shfl_sync(0xffffffffu, alpha2, (lane & 7) * 4);
                alpha = lane < 8 ? a1 : a2;                           // of row `lane`
                rescale_sums();
              }
#pragma unroll 1
              for (int c = 0; c < columns; c += 32) {
                uint32_t r[16], y[8];
                pa_ld_16x32(s_addr + c, r);
                tmem_wait_ld();
                slim_mask(c, r);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  if (e % 2 == 1 && !TWO) { y[e] = 0; continue; }
                  float x0, x1;
                  pa_fma2(x0, x1, __uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]), p.scale_log2, e % 2 ? -m2 : -m);
                  const float e0 = pa_exp2(x0), e1 = pa_exp2(x1);
                  pa_add2(sum[e % 2][0], sum[e % 2][1], e0, e1);
                  y[e] = pack_bf16(e0, e1);
                }
                pa_st_16x16(p_addr + c / 2, y);
              }
              l += sum[0][0] + sum[0][1];
              l2 += sum[1][0] + sum[1][1];
            };
            if (rows <= 8) {
              slim_tile(std::false_type{});
            } else if (rows <= 16) {
              slim_tile(std::true_type{});
            } else {
              columns_by(largest);
              raise();
              if (__any_sync(0xffffffffu, rescale)) {                   // (the product before is complete, or there were no scores)
                rescale_sums();
                l *= alpha;
              }
              columns_by(exponentials);
              l += sum0 + sum1;
            }
#pragma unroll 1
            for (int c = columns; c < 128; c += 32) {
              uint32_t none[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) none[e] = 0;
              tmem_st_32x16(p_addr + c / 2, none);
            }
          }
          if (unclean && !(ok = clear_values())) break;
          hand_over();
          continue;
        }
        uint32_t r[128];
        // P of the tile before is handed over when its store is done: while the scores are waited for, or else behind their load
        bool handed = i == 0;
        if (!handed && !__all_sync(0xffffffffu, mbar_test(&s_full[t], (uint32_t)(my_turn & 1)))) {
          hand_over();
          handed = true;
        }
        if (!(ok = wait(&s_full[t], (uint32_t)(my_turn & 1), 329))) break;
        tc_fence_after();
        if (active) {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_addr + c * 32, r + c * 32);
        }
        if (!handed) hand_over();
        if (active) tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        if (active) {
          if (masked) {
#pragma unroll
            for (int e = 0; e < 128; ++e)
              if (e > lim) r[e] = __float_as_uint(-1e30f);
          }
#pragma unroll
          for (int e = 0; e < 128; e += 8) {
            mx0 = pa_max3(mx0, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
            mx1 = pa_max3(mx1, __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
            mx2 = pa_max3(mx2, __uint_as_float(r[e + 4]), __uint_as_float(r[e + 5]));
            mx3 = pa_max3(mx3, __uint_as_float(r[e + 6]), __uint_as_float(r[e + 7]));
          }
          raise();
        }
        // P = 2^(s c - m) as packed bf16.  (Probabilities meet the values as bf16, the type of the tensor cores' other operand; their sum stays in
        // fp32.)
        if (active) {
#pragma unroll
          for (int e = 0; e < 64; ++e) {
            float x0, x1;
            pa_fma2(x0, x1, __uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]), p.scale_log2, neg_m);
            const float e0 = pa_exp2(x0), e1 = pa_exp2(x1);
            pa_add2(sum0, sum1, e0, e1);
            r[e] = pack_bf16(e0, e1);
          }
        }
        // the product before has read P, and O is complete
        if (my_turn > 0 && !(ok = wait(&o_done[t], (uint32_t)((my_turn - 1) & 1), 332))) break;
        if (active && __any_sync(0xffffffffu, rescale)) {
          rescale_sums();
          l *= alpha;
        }
        if (unclean && !(ok = clear_values())) break;
        if (active) {
          tmem_st_32x32(p_addr, r);
          tmem_st_32x32(p_addr + 32, r + 32);
        }
        if (!ok) break;
        l += sum0 + sum1;
      }
      if (!FEW && ok && mine > 0) hand_over();
      if (!ok) break;
      done += w.nb;
      turns[0] += n[0];
      turns[1] += n[1];
      // a row that sees none of the chain's keys has summed masked ones
      const int first_key = (w.j0 + (pair ? 0 : t)) * 128;
      if (mine == 0 || (slim ? last1 : last) < first_key) { m = -1e30f; l = 0.f; }
      float2* now = ml + (pieces & 1) * 2 * PA_ROWS;
      if constexpr (FEW) {
        const bool some = w.nb > 0;
        piece_done(k);
        if (!some) continue;
        if (q == 0) {
          // (the outputs of the piece before have been read: nobody is two pieces ahead)
          if (pieces > 0 && !(ok = wait(o_free, (uint32_t)((pieces - 1) & 1), 333))) break;
          if (slim) {
            if (mine == 0 || last2 < first_key) { m2 = -1e30f; l2 = 0.f; }
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l2 += __shfl_xor_sync(0xffffffffu, l2, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            l2 += __shfl_xor_sync(0xffffffffu, l2, 2);
            if (lane % 4 == 0) {
              now[t * PA_ROWS + lane / 4] = make_float2(m, l);
              now[t * PA_ROWS + lane / 4 + 8] = make_float2(m2, l2);
            }
          } else {
            now[t * PA_ROWS + row] = make_float2(m, l);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(few_done);
        }
        ++pieces;
        continue;
      }
      const bool direct = w.parts == 1;
      const int place = 2 * blockIdx.x + (w.part == 0 ? 1 : 0);
      if (threadIdx.x == 0 && pair && !direct && w.part == 0) out.cut[blockIdx.x] = make_int4(w.b, w.hk, w.item, w.parts);
      // the chains' shares of an output; where both worked on the same rows, each needs the other's statistics
      float f[2] = {0.f, 0.f}, M = m, L = l;
      if (w.nb > 0 && active) {
        if (pair) {
          f[t] = !direct ? 1.f : L == 0.f ? 0.f : 1.f / L;
        } else {
          now[t * PA_ROWS + row] = make_float2(m, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(&y_bar[q]);
          if (!(ok = wait(&y_bar[q], (uint32_t)(y_turn & 1), 335))) break;
          ++y_turn;
          const float2 a = now[row], b = now[PA_ROWS + row];
          M = fmaxf(a.x, b.x);
          f[0] = a.y == 0.f ? 0.f : pa_exp2(a.x - M);
          f[1] = b.y == 0.f ? 0.f : pa_exp2(b.x - M);
          L = f[0] * a.y + f[1] * b.y;
          if (direct) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            f[0] *= inv;
            f[1] *= inv;
          }
        }
        if (n[0] > 0 && !(pair && t == 1) && !(ok = wait(&o_done[0], (uint32_t)((turns[0] - 1) & 1), 336))) break;
        if (n[1] > 0 && !(pair && t == 0) && !(ok = wait(&o_done[1], (uint32_t)((turns[1] - 1) & 1), 336))) break;
        tc_fence_after();
      }
      // this warp's channels: its own chain's, or half of both chains'
      const bool some = w.nb > 0;
      if (active) {
        const int width = pair ? D : D / 2, c0 = pair ? 0 : t * width;
        const bool use[2] = {some && n[0] > 0 && !(pair && t == 1), some && n[1] > 0 && !(pair && t == 0)};
        __nv_bfloat16* to = out_row(w.s, w.hk, token0 + row_token, row);
        const int part_row = (pair ? t * PA_ROWS : 0) + row;
        float4* parts = reinterpret_cast<float4*>(out.part_o) + (int64_t)place * (2 * PA_ROWS * D / 4);
#pragma unroll 1
        for (int c = c0; c < c0 + width; c += 16) {
          uint32_t x[32];
          __syncwarp();
          if (use[0]) tmem_ld_32x16(lane_addr + O_COL + c, x);
          if (use[1]) tmem_ld_32x16(lane_addr + O_COL + D + c, x + 16);
          tmem_wait_ld();
          if (!real) continue;
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              o[i] = f[0] == 0.f ? 0.f : f[0] * __uint_as_float(x[e + i]);      // (a share of 0: nothing was written there)
              if (f[1] != 0.f) o[i] = fmaf(f[1], __uint_as_float(x[16 + e + i]), o[i]);
            }
            if (direct) {
              *reinterpret_cast<uint4*>(to + c + e) = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
            } else if (some) {
              float4* part = parts + part_at<D>(pair, part_row, c + e);
              part[0] = make_float4(o[0], o[1], o[2], o[3]);
              part[pair ? 2 * PA_ROWS : 1] = make_float4(o[4], o[5], o[6], o[7]);
            }
          }
        }
        if (real && !direct && (pair || t == 0)) out.part_ml[(int64_t)place * (2 * PA_ROWS) + part_row] = make_float2(M, L);
      }
      if (!pair && !direct) {
        __syncwarp();
        if (lane == 0) part_through(w, PA_SOFTMAX);
      }
      piece_done(k);
      if (!some) continue;
      // (nobody counts twice in a phase: the piece before is over)
      if (pieces > 0 && !(ok = wait(o_free, (uint32_t)((pieces - 1) & 1), 333))) break;
      ++pieces;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (warp == 9) {                         // copies still on their way land before the block ends
      auto landed = [&](uint64_t* bar, int parity) { mbar_wait(bar, (uint32_t)(parity & 1), abort_flag + 1, p.err, 339); };
      for (int i = max(0, q_loaded - (FEW ? 2 : 1)); i < q_loaded; ++i) landed(&q_full[FEW ? i & 1 : 0], FEW ? i >> 1 : i);
      for (int v = 0; v < 2; ++v)
        for (int i = max(0, issued[v] - RING); i < issued[v]; ++i) landed(&full[v * RING + i % RING], i / RING);
    }
  } else {
    for (int i = 0; i < *joins; ++i) {
      const Piece& j = join_s[i];
      for (int n = threadIdx.x; n < j.s.n * group * (D / 4); n += PA_THREADS) {
        const int r = n / (D / 4), c = n % (D / 4) * 4;
        JoinedRow row;
        const int first = j.first, parts = j.parts;
#pragma unroll 4
        for (int k = 0; k < parts; ++k) {
          const int64_t at = part_place(first, k) * (FEW ? QROWS : 2 * PA_ROWS) + r;
          row.add(__ldcg(out.part_ml + at), __ldcg(reinterpret_cast<const float4*>(out.part_o + at * D + c)));
        }
        row.put(out_row(j.s, j.hk, r / group, r) + c);
      }
    }
  }
  if (warp == 10) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Items of two tiles that were cut by the kernel above: block (x, y) has 32 rows of what began in block x and went on, four channels of two or four
// rows a thread, whose loads go out together (100 tokens on 800 positions, 16 heads on 8 of 128,
// in a graph: 26.6 us one after the other, 24.3 so; 512 on 2048 30.5 and 28.3).
// (By one block, 256 rows of four to five parts would take as long as the launch.)
template <int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedParams p, const PagedSplit in) {
  pdl_wait();
  pdl_trigger();
  const int4 c = in.cut[blockIdx.x];
  if (c.w <= 1) return;
  constexpr int ROWS = 32 * (D / 4) / 256;
  const int group = p.Hq / p.Hkv, tokens = PA_ROWS / group, channel = threadIdx.x % (2 * D) / 8 * 4;
  auto row_of = [&](int j) { return (int)blockIdx.y * 32 + (j * 256 + (int)threadIdx.x) / (2 * D) * 8 + (int)threadIdx.x % 8; };      // (eight rows side by side)
  JoinedRow rows[ROWS];
#pragma unroll 2
  for (int k = 0; k < c.w; ++k) {
    const int64_t place = part_place(blockIdx.x, k);
    float2 x[ROWS];
    float4 o[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {                                  // (rows that nobody has are in the place, too)
      x[j] = __ldcg(in.part_ml + place * (2 * PA_ROWS) + row_of(j));
      o[j] = __ldcg(reinterpret_cast<const float4*>(in.part_o) + place * (2 * PA_ROWS * D / 4) + part_at<D>(true, row_of(j), channel));
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) rows[j].add(x[j], o[j]);
  }
  const PagedSeq s = paged_seq(p, c.x);
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int r = row_of(j), i = (2 * c.z + r / PA_ROWS) * tokens + r % PA_ROWS / group;
    if (r % PA_ROWS < tokens * group && i < s.n) rows[j].put(p.o + (int64_t)(s.row0 + i) * p.so_t + (int64_t)(c.y * group + r % PA_ROWS % group) * p.so_h + channel);
  }
}

// As launch_ex, always with a programmatic dependency on the kernel before: for a kernel that belongs to the same call.
template <typename... KArgs, typename... Args>
static cudaError_t launch_behind(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, Args&&... args) {
  const bool pdl = ctx().pdl;
  ctx().pdl = true;
  const cudaError_t e = launch_ex(kernel, grid, block, smem, std::forward<Args>(args)...);
  ctx().pdl = pdl;
  return e;
}

template <int D, bool FEW>
static int launch_paged(const CUtensorMap& tk, const CUtensorMap& tv, const PagedParams& p) {
  using S = PagedShape<D, FEW>;
  static bool configured[64] = {false};   // per device: kd_shutdown + kd_init may move the library to another GPU
  if (!configured[ctx().device & 63]) {
    KD_CUDA_CHECK(cudaFuncSetAttribute(paged_attention_kernel<D, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    configured[ctx().device & 63] = true;
  }
  // [token][head][D] with a box of the query heads of a tile's tokens on one KV head, 64 channels wide
  const int group = p.Hq / p.Hkv, blocks = ctx().sm_count;
  KD_REQUIRE(blocks <= PA_BLOCKS, "%d multiprocessors", blocks);
  const int64_t ext[4] = {1, p.T, p.Hq, D}, st[3] = {p.T * p.sq_t, p.sq_t, p.sq_h};
  CUtensorMap tq;
  KD_TRY(make_tmap_bhsd(&tq, p.q, ext, st, group, S::QROWS / group));
  const uint64_t places = 2 * (uint64_t)blocks * (FEW ? S::QROWS : 2 * PA_ROWS);
  void* scratch;
  KD_TRY(get_workspace(places * (D * 4 + 8) + (uint64_t)blocks * 16, &scratch));
  PagedSplit out{};
  out.part_o = static_cast<float*>(scratch);
  out.part_ml = reinterpret_cast<float2*>(out.part_o + places * D);
  out.cut = reinterpret_cast<int4*>(out.part_ml + places);
  KD_CUDA_CHECK(launch_ex(paged_attention_kernel<D, FEW>, dim3(blocks), dim3(PA_THREADS), (size_t)S::SMEM, tq, tk, tv, p, out));
  KD_TRY(after_launch("paged_attention_kernel"));
  if ((int64_t)p.max_query * group > PA_ROWS) {
    KD_CUDA_CHECK(launch_behind(paged_join_kernel<D>, dim3(blocks, 2 * PA_ROWS / 32), dim3(256), 0, p, out));
    KD_TRY(after_launch("paged_join_kernel"));
  }
  return KD_OK;
}

// After an error an item may have been left with some of its parts counted (context.cu, check_device_flag).
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
  // (a warp waits for all pages of a piece, at most 2 us each, and gives up after a second)
  KD_REQUIRE(block_table->shape[0] <= 65535 && block_table->shape[1] <= (1 << 18), "the block table is too large: up to 65535 sequences of 2^18 pages are handled");
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
  for (const kd_tensor* t : {q, k_pool, v_pool, block_table, ctx_len, q_start})
    KD_REQUIRE(!views_meet(out, t), "out must not share memory with what the call reads");
  p.q = static_cast<const __nv_bfloat16*>(pq); p.k = static_cast<const __nv_bfloat16*>(pk); p.v = static_cast<const __nv_bfloat16*>(pv);
  p.o = static_cast<__nv_bfloat16*>(po);
  p.table = static_cast<const int*>(pt); p.ctx = static_cast<const int*>(pc); p.q_start = static_cast<const int*>(ps);
  p.sq_t = q->strides[0]; p.sq_h = q->strides[1]; p.so_t = out->strides[0]; p.so_h = out->strides[1];
  for (int i = 0; i < 3; ++i) { p.sk[i] = k_pool->strides[i]; p.sv[i] = v_pool->strides[i]; }
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = ctx().error_flag;
  CUtensorMap tk, tv;
  KD_TRY(make_tmap_bhsd(&tk, p.k, k_pool->shape, k_pool->strides, 128));
  KD_TRY(make_tmap_bhsd(&tv, p.v, v_pool->shape, v_pool->strides, 128));
  const bool few = (int64_t)p.max_query * (Hq / Hkv) <= 32;
  if (D == 128) return few ? launch_paged<128, true>(tk, tv, p) : launch_paged<128, false>(tk, tv, p);
  return few ? launch_paged<64, true>(tk, tv, p) : launch_paged<64, false>(tk, tv, p);
}
