// Beam search: the best continuations of every request's beams (kd_beam_select).
//
// A request has K beams with scores s_j and logits x_j over V tokens; candidate (j, i) is worth v = s_j + x_ji - lse_j, where
// lse_j = log sum_i exp(x_ji).  The first kernel passes over the logits once: a block per chunk of a row leaves the chunk's maximum, its sum
// of exponentials and its K largest logits in order.  The second, a block per request, joins the sums (in double), and takes the
// K largest candidates of the chunks' lists.  Within a row the order of candidates is that of the logits, so the sums are not needed for
// the lists.  Equal candidates go by the lower beam, then the lower token.
//
// A chunk's K largest: the K-th largest of the 256 threads' maxima is a bound that K elements reach and few others do; those that reach
// it are put side by side, and each counts the larger ones.  Bound: HBM, 4 bytes a logit.
#include "common.cuh"
#include "kernels.cuh"

namespace kd {

constexpr int BM_THREADS = 256, BM_CAP = 512, BM_BEAMS = 32;

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

template <int NE>
__global__ void __launch_bounds__(BM_THREADS) beam_rows_kernel(const float* __restrict__ logits, int64_t ld, int V, int K, int eos, int vec, float2* __restrict__ stats,
                                                               uint64_t* __restrict__ lists) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red[8];
  __shared__ __align__(16) float mx[BM_THREADS];
  __shared__ uint64_t keys[BM_CAP];
  __shared__ int count;
  __shared__ float bound;
  __shared__ uint64_t best[8];
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int64_t row = blockIdx.y;
  const int base = blockIdx.x * (NE * BM_THREADS);
  const float* x = logits + row * ld;
  auto index = [&](int e) { return base + ((e >> 2) * BM_THREADS + t) * 4 + (e & 3); };
  float r[NE];
#pragma unroll
  for (int e = 0; e < NE; e += 4) {
    const int i = index(e);
    if (vec && i + 3 < V) {
      const float4 f = *reinterpret_cast<const float4*>(x + i);
      r[e] = f.x; r[e + 1] = f.y; r[e + 2] = f.z; r[e + 3] = f.w;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) r[e + c] = i + c < V ? x[i + c] : -INFINITY;
    }
  }
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < NE; ++e) m = fmaxf(m, r[e]);
  m = warp_max(m);
  if (lane == 0) red[w] = m;
  if (t == 0) count = 0;
  __syncthreads();
  m = red[0];
  for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < NE; ++e) s += m == -INFINITY && r[e] == -INFINITY ? 0.f : expf(r[e] - m);
  s = warp_sum(s);
  if (lane == 0) red[w] = s;
  // the K-th largest of the threads' maxima
  float own = -INFINITY;
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    if (index(e) == eos) r[e] = -INFINITY;
    own = fmaxf(own, r[e]);
  }
  mx[t] = own;
  __syncthreads();
  const int64_t place = row * gridDim.x + blockIdx.x;
  if (t == 0) {
    s = 0.f;
    for (int i = 0; i < 8; ++i) s += red[i];
    stats[place] = make_float2(m, s);
  }
  int rank = 0;
  for (int i = 0; i < BM_THREADS; i += 4) {
    const float4 f = *reinterpret_cast<const float4*>(mx + i);
    rank += (f.x > own || (f.x == own && i < t)) + (f.y > own || (f.y == own && i + 1 < t)) + (f.z > own || (f.z == own && i + 2 < t)) +
            (f.w > own || (f.w == own && i + 3 < t));
  }
  if (rank == K - 1) bound = own;
  __syncthreads();
  const float least = bound;
  auto valid = [&](int e) { return index(e) < V && index(e) != eos; };
#pragma unroll
  for (int e = 0; e < NE; ++e)
    if (r[e] >= least && valid(e)) {
      const int n = atomicAdd(&count, 1);
      if (n < BM_CAP) keys[n] = beam_key(r[e], index(e));
    }
  __syncthreads();
  const int n = count;
  uint64_t* out = lists + place * K;
  if (n <= BM_CAP) {
    for (int c = t; c < n; c += BM_THREADS) {
      const uint64_t key = keys[c];
      int before = 0;
      for (int i = 0; i < n; ++i) before += keys[i] > key;
      if (before < K) out[before] = key;
    }
    if (t >= n && t < K) out[t] = 0;
    return;
  }
  // hardly ever: many logits are equal to the bound.  One after the other.
  uint64_t last = ~0ull;
  for (int k = 0; k < K; ++k) {
    uint64_t mine = 0;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const uint64_t key = r[e] >= least && valid(e) ? beam_key(r[e], index(e)) : 0;
      if (key < last && key > mine) mine = key;
    }
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, mine, o);
      mine = other > mine ? other : mine;
    }
    if (lane == 0) best[w] = mine;
    __syncthreads();
    for (int i = 0; i < 8; ++i) mine = best[i] > mine ? best[i] : mine;
    if (t == 0) out[k] = mine;
    last = mine;
    __syncthreads();
  }
}

// (value, place) with place = beam * V + token.
struct BeamBest {
  double v;
  int64_t at;
};
__device__ __forceinline__ bool better(const BeamBest& a, const BeamBest& b) { return a.v > b.v || (a.v == b.v && a.at < b.at); }

__global__ void __launch_bounds__(BM_THREADS) beam_merge_kernel(const float* __restrict__ logits, int64_t ld, int V, int K, int eos, int chunks, const float2* __restrict__ stats,
                                                                const uint64_t* __restrict__ lists, const float* scores, float* out_scores, int* __restrict__ parents,
                                                                int64_t* __restrict__ tokens, float* __restrict__ ended) {
  pdl_wait();
  pdl_trigger();
  __shared__ double lse[BM_BEAMS], score[BM_BEAMS];
  __shared__ int dead[BM_BEAMS];                 // every candidate of the beam is worth minus infinity
  __shared__ BeamBest red[8], chosen[BM_BEAMS], ends[BM_BEAMS];
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int64_t b = blockIdx.x, none = (int64_t)1 << 62;
  for (int j = w; j < K; j += 8) {
    const float2* st = stats + (b * K + j) * chunks;
    float m = -INFINITY;
    for (int c = lane; c < chunks; c += 32) m = fmaxf(m, st[c].x);
    m = warp_max(m);
    double s = 0.0;
    for (int c = lane; c < chunks; c += 32) s += st[c].x == -INFINITY ? (double)st[c].y : st[c].y * exp((double)st[c].x - m);
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      const double l = (double)m + log(s), g = scores[b * K + j];
      lse[j] = l;
      score[j] = g;
      dead[j] = !isfinite(l) || isnan(g) || isinf(g);
      BeamBest e{-INFINITY, none};
      if ((unsigned)eos < (unsigned)V) {
        e.at = (int64_t)j * V + eos;
        if (!dead[j]) e.v = ((double)logits[(b * K + j) * ld + eos] - l) + g;
      }
      ends[j] = e;
    }
  }
  __syncthreads();
  // entry k of list (j, c)
  auto entry = [&](int list, int k) -> BeamBest {
    const int j = list / chunks, c = list - j * chunks;
    if (k >= K) return BeamBest{-INFINITY, none};
    if (dead[j]) {
      int64_t i = k;
      if ((unsigned)eos < (unsigned)V && i >= eos) ++i;
      return BeamBest{-INFINITY, c == 0 && i < V ? (int64_t)j * V + i : none};
    }
    const uint64_t key = lists[((b * K + j) * chunks + c) * K + k];
    if (key == 0) return BeamBest{-INFINITY, none};
    return BeamBest{((double)beam_logit(key) - lse[j]) + score[j], (int64_t)j * V + beam_token(key)};
  };
  const int total = K * chunks;
  // the best of this thread's lists behind the last candidate taken
  BeamBest mine, last{INFINITY, -1};
  auto look = [&]() {
    mine = BeamBest{-INFINITY, none};
    for (int l = t; l < total; l += BM_THREADS)
      for (int k = 0; k < K; ++k) {
        const BeamBest e = entry(l, k);
        if (better(last, e)) {
          if (better(e, mine)) mine = e;
          break;
        }
      }
  };
  look();
  for (int k = 0; k < K; ++k) {
    BeamBest x = mine;
    for (int o = 16; o > 0; o >>= 1) {
      BeamBest y;
      y.v = __shfl_xor_sync(0xffffffffu, x.v, o);
      y.at = __shfl_xor_sync(0xffffffffu, x.at, o);
      if (better(y, x)) x = y;
    }
    if (lane == 0) red[w] = x;
    __syncthreads();
    x = red[0];
    for (int i = 1; i < 8; ++i)
      if (better(red[i], x)) x = red[i];
    if (t == 0) chosen[k] = x;
    const bool taken = x.at == mine.at && x.at != none;
    last = x;
    if (taken) look();
    __syncthreads();
  }
  if (t < K) {
    const BeamBest x = chosen[t];
    const int64_t n = b * K + t;
    out_scores[n] = (float)x.v;
    parents[n] = x.at == none ? 0 : (int)(x.at / V);
    tokens[n] = x.at == none ? 0 : x.at % V;
    if (ended) {
      const BeamBest e = ends[t];
      int before = 0;
      for (int i = 0; i < K; ++i) before += better(chosen[i], e) + (i != t && better(ends[i], e));
      ended[n] = e.at != none && before < K ? (float)e.v : -INFINITY;
    }
  }
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
  const int64_t V = logits->shape[last], ld = logits->strides[last - 1];
  if (logits->ndim == 3)
    KD_REQUIRE(logits->shape[0] == B && logits->shape[1] == K && (logits->strides[0] == K * ld || B <= 1), "logits must hold evenly spaced rows, one for each of %lld x %lld beams", (long long)B, (long long)K);
  else
    KD_REQUIRE(logits->shape[0] == B * K, "logits must hold one row for each of %lld x %lld beams", (long long)B, (long long)K);
  KD_REQUIRE(logits->strides[last] == 1 || V == 1, "unit stride along the vocabulary required");
  KD_REQUIRE(V >= 2 && V <= 0x7fffffff - 8192 && eos < V, "a vocabulary of at least two tokens, among them the end token (or a negative one for none), is required");
  KD_REQUIRE(B * K <= 65535, "%lld beams: up to 65535 a call", (long long)(B * K));
  KD_REQUIRE(out_scores->dtype == KD_F32 && is_contiguous(out_scores) && numel(out_scores) == B * K && parents->dtype == KD_I32 && is_contiguous(parents) &&
                 numel(parents) == B * K && tokens->dtype == KD_I64 && is_contiguous(tokens) && numel(tokens) == B * K,
             "outputs must be contiguous [requests, beams]: scores fp32, parents int32, tokens int64");
  if (ended) KD_REQUIRE(ended->dtype == KD_F32 && is_contiguous(ended) && numel(ended) == B * K, "ended must be contiguous fp32 [requests, beams]");
  void *px, *ps, *po, *pp, *pt, *pe = nullptr, *scratch;
  KD_TRY(tensor_ptr(logits, &px)); KD_TRY(tensor_ptr(scores, &ps)); KD_TRY(tensor_ptr(out_scores, &po)); KD_TRY(tensor_ptr(parents, &pp)); KD_TRY(tensor_ptr(tokens, &pt));
  if (ended) KD_TRY(tensor_ptr(ended, &pe));
  if (B == 0) return KD_OK;
  const int vec = (reinterpret_cast<uintptr_t>(px) & 15) == 0 && ld % 4 == 0;
  constexpr int NE = 16;
  const int chunks = (int)((V + NE * BM_THREADS - 1) / (NE * BM_THREADS));
  const uint64_t places = (uint64_t)B * K * chunks;
  KD_TRY(get_workspace(places * 8 * (1 + K), &scratch));
  float2* stats = static_cast<float2*>(scratch);
  uint64_t* lists = reinterpret_cast<uint64_t*>(stats + places);
  KD_CUDA_CHECK(launch_ex(beam_rows_kernel<NE>, dim3(chunks, (unsigned)(B * K)), dim3(BM_THREADS), 0, (const float*)px, ld, (int)V, (int)K, eos, vec, stats, lists));
  KD_TRY(after_launch("beam_rows_kernel"));
  KD_CUDA_CHECK(launch_ex(beam_merge_kernel, dim3((unsigned)B), dim3(BM_THREADS), 0, (const float*)px, ld, (int)V, (int)K, eos, chunks, (const float2*)stats,
                          (const uint64_t*)lists, (const float*)ps, (float*)po, (int*)pp, (int64_t*)pt, (float*)pe));
  return after_launch("beam_merge_kernel");
}
