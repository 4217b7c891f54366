// Beam search: the best continuations of every request's beams (kd_beam_select).
//
// A request has K beams with scores s_j and logits x_j over V tokens; candidate (j, i) is worth v = s_j + x_ji - lse_j, where
// lse_j = log sum_i exp(x_ji).  One launch passes over the logits once: a block per segment of a row leaves the segment's maximum, its sum of
// exponentials and its K largest logits in order, and the block of a request that is through last joins the sums (in double) and takes
// the K largest candidates of the segments' lists.  Within a row the order of candidates is that of the logits, so the sums are not
// needed for the lists.  Equal candidates go by the lower beam, then the lower token.
//
// A segment is read 4096 logits at a time.  Those above a bound, the K-th largest so far, are put side by side in shared memory; after the first
// 4096 hardly any are.  The first bound: with q = 1, 2 or 4, the q-th largest of a warp's lanes' maxima, and of these the one
// that ceil(K / q) of the eight warps reach, so at least K logits reach it.
//
// Bound: HBM, 4 bytes a logit, where there are many rows: 32 requests of 4 beams over 151936 tokens (78 MB) 28 us, of which the pass takes 16 (4.9
// TB/s: four blocks an SM with 16 KB each on the way, which stop for the bound at their first step) and the join of a request 6, a chain of short
// steps by one block; the rest is the launch.  One request of 4 beams 13.7 us, all latency: 2.4 of them the pass.  Two launches (lists, then the
// join) took 110 and 20.5, with the lists ranked by every pair of a step.  Masked rows are slower where a step of 4096 logits is left with
// fewer than K that are not minus infinity: the bound is minus infinity then, and a segment is read K times more.  In a graph, 32 x 4 beams with all
// logits 26.9 us, with 1 % of them 27.0, with 0.01 % 249; 4 x 32 beams 125, 1372 and 1387.
#include "common.cuh"
#include "kernels.cuh"

namespace kd {

constexpr int BM_THREADS = 256, BM_CAP = 512, BM_CAND = 1024, BM_BEAMS = 32, BM_NE = 16, BM_STEP = BM_NE * BM_THREADS, BM_REQUESTS = 65536;

// Segments of a request that are through; the last one sets it back.
static __device__ unsigned int g_beam_through[BM_REQUESTS];

// Larger is better: the number in the upper half, the lower index in the lower one.  0: no candidate.
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t i) {
  const uint32_t b = __float_as_uint(x + 0.f);                      // -0 and 0 are equal
  return (uint64_t)((b & 0x80000000u) ? ~b : (b | 0x80000000u)) << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float beam_logit(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint32_t beam_token(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// Doubles as whole numbers of the same order (64-bit comparisons of doubles are slow).
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double value_of(uint64_t o) { return __longlong_as_double((long long)(o >> 63 ? o & 0x7fffffffffffffffull : ~o)); }
// A candidate's ordered value, and (beam, token) in the upper and lower half of `at`.
struct BeamBest {
  uint64_t v, at;
};
constexpr uint64_t BM_LOWEST = 0x000fffffffffffffull;      // ordered(-infinity)
constexpr uint64_t BM_NONE = ~0ull;
__device__ __forceinline__ bool better(const BeamBest& a, const BeamBest& b) { return a.v > b.v || (a.v == b.v && a.at < b.at); }
// A lane's value that is the q-th largest of the warp's (equal ones count singly).
template <typename T>
__device__ __forceinline__ T warp_nth(T x, int q, T least) {
  T top = least;
#pragma unroll 1
  for (int i = 0; i < q; ++i) {
    top = x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const unsigned who = __ballot_sync(0xffffffffu, x == top);
    if ((threadIdx.x & 31) == (unsigned)(__ffs(who) - 1)) x = least;
  }
  return top;
}
__device__ __forceinline__ int beam_quota(int K) { return K <= 8 ? 1 : K <= 16 ? 2 : 4; }
// Of eight values the one that n of them reach.  By whole warps.
template <typename T>
__device__ __forceinline__ T nth_of_eight(const T* x, int n) {
  const int lane = threadIdx.x & 7;
  const T own = x[lane];
  int above = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) above += x[j] > own || (x[j] == own && j < lane);
  return x[(__ffs(__ballot_sync(0xffffffffu, above == n - 1)) - 1) & 7];
}

struct BeamParams {
  const float* logits;
  int64_t ld;
  int V, K, eos, vec, segs, seg_len;
  float2* stats;                // per row and segment (maximum, sum of exponentials)
  uint64_t* lists;              // ... and its K best, 0 behind the last
  const float* scores;          // may be out_scores
  float* out_scores;
  int* parents;
  int64_t* tokens;
  float* ended;
};

struct BeamShared {
  float2 red[8];
  float least[8];
  uint64_t keys[BM_CAP], next[BM_BEAMS], best[8];
  int count, last;
  double lse[BM_BEAMS], score[BM_BEAMS];
  uint64_t heads[8];
  int dead[BM_BEAMS];           // every candidate of the beam is worth minus infinity
  BeamBest cand[BM_CAND], chosen[BM_BEAMS], ends[BM_BEAMS], top[8];
};

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float BM_LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp_of(float x) { return exp2_of(x * BM_LOG2E); }
// exp(a - m) of two numbers, added to two sums.  (The difference first: a times log2 e may be beyond fp32 where masks are its
// lowest number.  A fused multiply-add would save 1 us of 28 in the largest case.)
__device__ __forceinline__ void add_exp(float& s0, float& s1, float a0, float a1, float minus_m) {
  float x0, x1;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
      "add.rn.f32x2 d, a, c;\n\tmul.rn.f32x2 d, d, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(x0), "=f"(x1) : "f"(a0), "f"(a1), "f"(BM_LOG2E), "f"(minus_m));
  x0 = exp2_of(x0);
  x1 = exp2_of(x1);
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "+f"(s0), "+f"(s1) : "f"(x0), "f"(x1));
}
__device__ __forceinline__ float max_of(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The segments' lists of request b are there: its outputs.  By the whole block.  One block runs this once, out of a cold instruction cache: short
// loops, no double-precision functions (an lse in fp32 parts is off by less than the sum of the exponentials is).
__device__ __noinline__ void beam_join(const BeamParams& p, int64_t b, BeamShared& sh) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5, K = p.K, segs = p.segs;
  const bool ends = (unsigned)p.eos < (unsigned)p.V;
  // the lists' entries, K for each segment of each beam; a thread's first ones come while the sums are joined
  const uint64_t* lists = p.lists + b * K * segs * K;
  const int total = K * segs * K;
  const int own = lane * 8 + w;      // (few entries: some for every warp)
  uint64_t early[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) early[k] = own + k * BM_THREADS < total ? __ldcg(lists + own + k * BM_THREADS) : 0;
#pragma unroll 1
  for (int j = w; j < K; j += 8) {
    const float2* st = p.stats + (b * K + j) * segs;
    float m = -INFINITY, s = 0.f;
#pragma unroll 1
    for (int c = lane; c < segs; c += 32) {
      const float2 x = __ldcg(st + c);
      const float now = fmaxf(m, x.x), from = now == -INFINITY ? 0.f : now;
      s = s * exp_of(m - from) + x.y * exp_of(x.x - from);
      m = now;
    }
    const float all = warp_max(m), from = all == -INFINITY ? 0.f : all;
    s = warp_sum(s * exp_of(m - from));
    if (lane == 0) {
      const double l = (double)all + logf(s), g = p.scores[b * K + j];
      sh.lse[j] = l;
      sh.score[j] = g;
      sh.dead[j] = !(fabs(l) < INFINITY) || !(fabs(g) < INFINITY);
      BeamBest e{BM_LOWEST, BM_NONE};
      if (ends) {
        e.at = (uint64_t)j << 32 | p.eos;
        if (!sh.dead[j]) e.v = ordered(((double)p.logits[(b * K + j) * p.ld + p.eos] - l) + g);
      }
      sh.ends[j] = e;
    }
  }
  if (t == 0) sh.count = 0;
  __syncthreads();
  auto entry = [&](int i, uint64_t key) -> BeamBest {
    const int j = i / (segs * K);
    if (sh.dead[j]) {
      i -= j * segs * K;
      const int token = i + (ends && i >= p.eos);
      return BeamBest{BM_LOWEST, i < K && token < p.V ? (uint64_t)j << 32 | token : BM_NONE};
    }
    if (key == 0) return BeamBest{BM_LOWEST, BM_NONE};
    return BeamBest{ordered(((double)beam_logit(key) - sh.lse[j]) + sh.score[j]), (uint64_t)j << 32 | beam_token(key)};
  };
  // a bound that K candidates reach
  uint64_t top = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (own + k * BM_THREADS < total) top = max(top, entry(own + k * BM_THREADS, early[k]).v);
#pragma unroll 1
  for (int i = own + 4 * BM_THREADS; i < total; i += BM_THREADS) top = max(top, entry(i, __ldcg(lists + i)).v);
  const int quota = beam_quota(K);
  top = warp_nth(top, quota, (uint64_t)0);
  if (lane == 0) sh.heads[w] = top;
  __syncthreads();
  const uint64_t least = nth_of_eight(sh.heads, (K + quota - 1) / quota);
  auto collect = [&](const BeamBest& e) {
    if (e.at != BM_NONE && e.v >= least) {
      const int n = atomicAdd(&sh.count, 1);
      if (n < BM_CAND) sh.cand[n] = e;
    }
  };
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (own + k * BM_THREADS < total) collect(entry(own + k * BM_THREADS, early[k]));
#pragma unroll 1
  for (int i = own + 4 * BM_THREADS; i < total; i += BM_THREADS) collect(entry(i, __ldcg(lists + i)));
  __syncthreads();
  const int n = sh.count;
  if (t < K) sh.chosen[t] = BeamBest{BM_LOWEST, BM_NONE};
  __syncthreads();
  if (n <= BM_CAND) {
#pragma unroll 1
    for (int c = t; c < n; c += BM_THREADS) {
      const BeamBest e = sh.cand[c];
      int before = 0;
#pragma unroll 4
      for (int i = 0; i < n; ++i) before += better(sh.cand[i], e);
      if (before < K) sh.chosen[before] = e;
    }
  } else {
    // many candidates: one after the other, every thread with the best of its own behind the last one taken
    BeamBest mine, last{~0ull, 0};
    auto look = [&]() {
      mine = BeamBest{BM_LOWEST, BM_NONE};
#pragma unroll 1
      for (int i = t; i < total; i += BM_THREADS) {
        const BeamBest e = entry(i, __ldcg(lists + i));
        if (better(last, e) && better(e, mine)) mine = e;
      }
    };
    look();
#pragma unroll 1
    for (int k = 0; k < K; ++k) {
      BeamBest x = mine;
#pragma unroll 1
      for (int o = 16; o > 0; o >>= 1) {
        BeamBest y;
        y.v = __shfl_xor_sync(0xffffffffu, x.v, o);
        y.at = __shfl_xor_sync(0xffffffffu, x.at, o);
        if (better(y, x)) x = y;
      }
      if (lane == 0) sh.top[w] = x;
      __syncthreads();
      x = sh.top[0];
#pragma unroll 1
      for (int i = 1; i < 8; ++i)
        if (better(sh.top[i], x)) x = sh.top[i];
      if (t == 0) sh.chosen[k] = x;
      const bool taken = x.at == mine.at && x.at != BM_NONE;
      last = x;
      if (taken) look();
      __syncthreads();
    }
  }
  __syncthreads();
  if (t < K) {
    const BeamBest x = sh.chosen[t];
    const int64_t at = b * K + t;
    p.out_scores[at] = (float)value_of(x.v);
    p.parents[at] = x.at == BM_NONE ? 0 : (int)(x.at >> 32);
    p.tokens[at] = x.at == BM_NONE ? 0 : (int64_t)(x.at & 0xffffffffu);
    if (p.ended) {
      const BeamBest e = sh.ends[t];
      int before = 0;
#pragma unroll 1
      for (int i = 0; i < K; ++i) before += better(sh.chosen[i], e) + (i != t && better(sh.ends[i], e));
      p.ended[at] = e.at != BM_NONE && before < K ? (float)value_of(e.v) : -INFINITY;
    }
  }
}

__global__ void __launch_bounds__(BM_THREADS, 4) beam_kernel(const BeamParams p) {
  __shared__ BeamShared sh;
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x, lane = t & 31, w = t >> 5, K = p.K, quota = beam_quota(K);
  const int64_t row = blockIdx.y;
  const int lo = blockIdx.x * p.seg_len, hi = min(p.V, lo + p.seg_len);
  const float* x = p.logits + row * p.ld;
  // whole steps are read four logits at a time; the rest of a row goes round over all threads, so that every warp has some for the first bound
  auto whole = [&](int base) { return p.vec && base + BM_STEP <= hi; };
  auto index = [&](int base, int e) { return base + (whole(base) ? ((e >> 2) * BM_THREADS + t) * 4 + (e & 3) : e * BM_THREADS + t); };
  auto load = [&](int base, float (&r)[BM_NE]) {
    if (whole(base)) {
#pragma unroll
      for (int e = 0; e < BM_NE; e += 4) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(x + index(base, e)));
        r[e] = f.x; r[e + 1] = f.y; r[e + 2] = f.z; r[e + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < BM_NE; ++e) r[e] = index(base, e) < hi ? x[index(base, e)] : -INFINITY;
    }
  };
  // the best of keys[0 .. n), in order, to their front; how many there are
  auto order = [&](int n) {
#pragma unroll 1
    for (int c = t; c < n; c += BM_THREADS) {
      const uint64_t key = sh.keys[c];
      int before = 0;
#pragma unroll 8
      for (int i = 0; i < n; ++i) before += sh.keys[i] > key;
      if (before < K) sh.next[before] = key;
    }
    n = min(n, K);
    __syncthreads();
    if (t < n) sh.keys[t] = sh.next[t];
    if (t == 0) sh.count = n;
    __syncthreads();
    return n;
  };
  float r[BM_NE], ahead[BM_NE], m = -INFINITY, s = 0.f, s1 = 0.f, bound = -INFINITY;
  bool above = false;               // only logits above the bound count (else those that reach it)
  int kept = 0;
  if (t == 0) sh.count = 0;
  load(lo, ahead);
#pragma unroll 1
  for (int base = lo, step = 0; base < hi; base += BM_STEP, ++step) {
#pragma unroll
    for (int e = 0; e < BM_NE; ++e) r[e] = ahead[e];
    if (base + BM_STEP < hi) load(base + BM_STEP, ahead);
    float four[BM_NE / 4], top;
    auto tops = [&]() {
#pragma unroll
      for (int e = 0; e < BM_NE; e += 4) four[e / 4] = fmaxf(max_of(r[e], r[e + 1], r[e + 2]), r[e + 3]);
      top = fmaxf(max_of(four[0], four[1], four[2]), four[3]);
    };
    tops();
    // the thread's own maximum and sum; terms far below vanish, NaN and infinity stay
    const float now = fmaxf(m, top), from = now == -INFINITY ? 0.f : now, scale = exp_of(m - from);
    s *= scale;
    s1 *= scale;
    m = now;
#pragma unroll
    for (int e = 0; e < BM_NE; e += 2) add_exp(s, s1, r[e], r[e + 1], -from);
    if (p.eos >= base && p.eos < base + BM_STEP) {
#pragma unroll
      for (int e = 0; e < BM_NE; ++e)
        if (index(base, e) == p.eos) r[e] = -INFINITY;
      tops();
    }
    if (step == 0) {
      const float u = warp_nth(top, quota, -INFINITY);
      if (lane == 0) sh.least[w] = u;
      __syncthreads();
      bound = nth_of_eight(sh.least, (K + quota - 1) / quota);
    }
    if (above ? top > bound : top >= bound) {
#pragma unroll
      for (int g = 0; g < BM_NE; g += 4) {
        if (!(above ? four[g / 4] > bound : four[g / 4] >= bound)) continue;
#pragma unroll
        for (int e = g; e < g + 4; ++e) {
          const int i = index(base, e);
          if ((above ? r[e] > bound : r[e] >= bound) && i < hi && i != p.eos) {
            const int n = atomicAdd(&sh.count, 1);
            if (n < BM_CAP) sh.keys[n] = beam_key(r[e], i);
          }
        }
      }
    }
    // the bound is raised after the first step and now and then
    if ((step & 3) == 0) {
      __syncthreads();
      const int n = sh.count;
      __syncthreads();
      if (n <= BM_CAP && n > kept) {
        kept = order(n);
        if (kept == K) {
          bound = beam_logit(sh.keys[K - 1]);
          above = true;             // what comes later and is equal has a higher index
        }
      }
    }
  }
  __syncthreads();
  const int n = sh.count;
  __syncthreads();
  if (n <= BM_CAP) {
    kept = order(n);
  } else {
    // Many logits reach the bound: many equal ones, or fewer than K in a step that are not minus infinity (nearly every segment where few tokens may
    // come).  One after the other, from memory: K more passes over the segment.
    uint64_t last = ~0ull;
#pragma unroll 1
    for (int k = 0; k < K; ++k) {
      uint64_t mine = 0;
#pragma unroll 1
      for (int i = lo + t; i < hi; i += BM_THREADS) {
        const float f = x[i];
        const uint64_t key = f >= -INFINITY && i != p.eos ? beam_key(f, i) : 0;
        if (key < last && key > mine) mine = key;
      }
#pragma unroll 1
      for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
      if (lane == 0) sh.best[w] = mine;
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < 8; ++i) mine = max(mine, sh.best[i]);
      if (t == 0) sh.keys[k] = mine;
      last = mine;
      __syncthreads();
    }
    kept = K;
  }
  // the segment's maximum and sum
  const float all = warp_max(m), from = all == -INFINITY ? 0.f : all;
  s = warp_sum((s + s1) * exp_of(m - from));
  if (lane == 0) sh.red[w] = make_float2(all, s);
  __syncthreads();
  const int64_t place = row * p.segs + blockIdx.x;
  if (t < K) p.lists[place * K + t] = t < kept ? sh.keys[t] : 0;
  if (w == 0) {
    const float2 y = sh.red[lane & 7];
    const float top = warp_max(y.x), base = top == -INFINITY ? 0.f : top;
    const float sum = warp_sum(lane < 8 ? y.y * exp_of(y.x - base) : 0.f);
    if (lane == 0) p.stats[place] = make_float2(top, sum);
  }
  __syncthreads();
  const int64_t b = row / K;
  if (t == 0) {
    // the block's writes before it, those of the others' blocks behind it
    unsigned before;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(&g_beam_through[b]) : "memory");
    sh.last = before == (unsigned)(K * p.segs) - 1;
    if (sh.last) g_beam_through[b] = 0;
  }
  __syncthreads();
  if (sh.last) beam_join(p, b, sh);
}

// After an error of another kernel in between (context.cu, check_device_flag).
int beam_reset_counters() {
  void* at = nullptr;
  KD_CUDA_CHECK(cudaGetSymbolAddress(&at, g_beam_through));
  KD_CUDA_CHECK(cudaMemsetAsync(at, 0, sizeof(unsigned) * BM_REQUESTS, ctx().stream));
  return KD_OK;
}

}  // namespace kd

using namespace kd;

KD_API int kd_beam_select(const kd_tensor* logits, const kd_tensor* scores, int eos, const kd_tensor* out_scores, const kd_tensor* parents, const kd_tensor* tokens,
                          const kd_tensor* ended) {
  KD_TRY(require_init());
  KD_REQUIRE(logits && scores && out_scores && parents && tokens, "null tensor");
  KD_REQUIRE(scores->ndim == 2 && scores->dtype == KD_F32 && is_contiguous(scores) && scores->shape[1] >= 1 && scores->shape[1] <= BM_BEAMS,
             "scores must be contiguous fp32 [requests, beams], of 1 to %d beams", BM_BEAMS);
  const int64_t B = scores->shape[0], K = scores->shape[1];
  KD_REQUIRE(logits->dtype == KD_F32 && logits->ndim >= 2 && logits->ndim <= 3, "logits must be fp32 [requests, beams, V] or [requests x beams, V]");
  const int last = logits->ndim - 1;
  // from one row to the next (the stride of a dimension of one is none)
  const int64_t V = logits->shape[last], ld = logits->strides[logits->ndim == 3 && K == 1 ? 0 : last - 1];
  if (logits->ndim == 3)
    KD_REQUIRE(logits->shape[0] == B && logits->shape[1] == K && (logits->strides[0] == K * ld || B <= 1), "logits must hold evenly spaced rows, one for each of %lld x %lld beams", (long long)B, (long long)K);
  else
    KD_REQUIRE(logits->shape[0] == B * K, "logits must hold one row for each of %lld x %lld beams", (long long)B, (long long)K);
  KD_REQUIRE(logits->strides[last] == 1 || V == 1, "unit stride along the vocabulary required");
  KD_REQUIRE(V >= 2 && V <= (1 << 30) && eos < V, "a vocabulary of 2 to 2^30 tokens, among them the end token (or a negative one for none), is required");
  KD_REQUIRE(B * K <= 65535, "%lld beams: up to 65535 a call", (long long)(B * K));
  KD_REQUIRE(out_scores->dtype == KD_F32 && is_contiguous(out_scores) && numel(out_scores) == B * K && parents->dtype == KD_I32 && is_contiguous(parents) &&
                 numel(parents) == B * K && tokens->dtype == KD_I64 && is_contiguous(tokens) && numel(tokens) == B * K,
             "outputs must be contiguous [requests, beams]: scores fp32, parents int32, tokens int64");
  if (ended) KD_REQUIRE(ended->dtype == KD_F32 && is_contiguous(ended) && numel(ended) == B * K, "ended must be contiguous fp32 [requests, beams]");
  void *px, *ps, *po, *pp, *pt, *pe = nullptr, *scratch;
  KD_TRY(tensor_ptr(logits, &px)); KD_TRY(tensor_ptr(scores, &ps)); KD_TRY(tensor_ptr(out_scores, &po)); KD_TRY(tensor_ptr(parents, &pp)); KD_TRY(tensor_ptr(tokens, &pt));
  if (ended) KD_TRY(tensor_ptr(ended, &pe));
  // The block that joins a request reads its scores before it writes, and the logits are read by others meanwhile.
  const kd_tensor* outs[4] = {out_scores, parents, tokens, ended};
  for (int i = 0; i < 4; ++i) {
    KD_REQUIRE(!views_meet(outs[i], logits) && (!views_meet(outs[i], scores) || (i == 0 && po == ps)), "outputs must not share memory with what the call reads (out_scores may be scores)");
    for (int j = 0; j < i; ++j) KD_REQUIRE(!views_meet(outs[i], outs[j]), "outputs must not share memory with one another");
  }
  if (B == 0) return KD_OK;
  BeamParams p{};
  p.logits = static_cast<const float*>(px);
  p.ld = ld; p.V = (int)V; p.K = (int)K; p.eos = eos;
  p.vec = (reinterpret_cast<uintptr_t>(px) & 15) == 0 && ld % 4 == 0;
  // four blocks an SM: segments of several steps where there are rows enough
  const int64_t rows = B * K, steps = (V + BM_STEP - 1) / BM_STEP;
  int64_t segs = 4 * (int64_t)ctx().sm_count / rows;
  segs = segs < 1 ? 1 : segs > steps ? steps : segs;
  p.seg_len = (int)((steps + segs - 1) / segs) * BM_STEP;
  p.segs = (int)((V + p.seg_len - 1) / p.seg_len);
  const uint64_t places = (uint64_t)rows * p.segs;
  KD_TRY(get_workspace(places * 8 * (1 + K), &scratch));
  p.stats = static_cast<float2*>(scratch);
  p.lists = reinterpret_cast<uint64_t*>(p.stats + places);
  p.scores = static_cast<const float*>(ps);
  p.out_scores = static_cast<float*>(po); p.parents = static_cast<int*>(pp); p.tokens = static_cast<int64_t*>(pt); p.ended = static_cast<float*>(pe);
  KD_CUDA_CHECK(launch_ex(beam_kernel, dim3(p.segs, (unsigned)rows), dim3(BM_THREADS), 0, p));
  return after_launch("beam_kernel");
}
