// Beam search on the paged cache: selection over beams and vocabulary, and the reordering of the beams' pages.
//
// Selection.  cand(w, v) = score_w + x_wv - log sum_u exp x_wu; the K largest over the W * V candidates of a request, equal
// ones by the lowest w * V + v.  Inside a row the order is the logits' own, so a row's K best are found on the logits,
// exactly; only the few survivors are put on the common scale, in 64 bits.
//   beam_slice_kernel  one CTA per slice of a row, one pass: every thread keeps the maximum of its elements and the sum of
//                      their exponentials.  The K-th largest of 64 groups' maxima is a threshold that the slice's K best
//                      cannot lie below; only the threads whose own maximum reaches it (K and a few) have their
//                      elements read again, out of L2, and what reaches it there is ranked.
//   beam_merge_kernel  one CTA per request: log-sum-exps of its rows, then the same threshold over their candidates.
// HBM-bound: the logits are read once.  Nothing depends on the order in which threads arrive.
// Measured, bf16: 64 requests of 8 beams over 151936 tokens 54 us (2.9 TB/s; the slices alone 46), one request of 4 beams over
// 51200 tokens 13.7 us.  What bounds the slices is instruction issue: unpacking, maximum, fma, ex2 and add per logit.
//
// Sums.  exp x = 2^(x L' - e) 2^e with L' the fp32 log2(e) and e = ceil(max x L') a whole number, so that raising the maximum
// scales a sum by a power of two, exactly; 32 terms at a time in fp32, 64 bits from there on.  L' is off by 1.3e-8
// relatively; for the terms that matter x is close to e / L', and log sum exp x = e / L' + log sum 2^(x L' - e) takes that out.
#pragma once

#include "paged_prefill.cuh"   // packed fp32 arithmetic
#include "sampling.cuh"

namespace kb200 {

constexpr int kBeamThreads = 256;
constexpr int kBeamGroups = 64;        // of 4 neighbouring threads; at least kBeamMaxOut
constexpr int kBeamMaxOut = 64;
constexpr int kBeamMaxBeams = 64;
constexpr int kBeamKeep = 1024;        // survivors that are ranked at once; more (rows made for it) take the slow way
constexpr int kBeamCtasPerSm = 4;      // slices that are cut per SM when rows alone are too few
constexpr float kBeamLog2e = 1.4426950408889634f;
static_assert(kBeamGroups >= kBeamMaxOut, "the K-th largest group maximum must exist");

struct BeamSum { double s; float e; float pad; };   // s * 2^e; e = -inf: nothing

struct BeamParams {
  const char* logits;
  const float* scores;
  const uint8_t* finished;     // or nullptr
  unsigned long long* part;    // [rows][slices][K] keys: ordered logit << 32 | ~index
  BeamSum* part_sum;           // [rows][slices]
  int64_t* out_tokens;
  int64_t* out_parents;
  float* out_scores;
  int64_t row_stride, vocab, end_token;
  int batch, beams, n_out, n_slices, slice, vec_ok;
};

// floats ordered as unsigned integers
__device__ __forceinline__ uint32_t order_f32(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unorder_f32(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ unsigned long long order_f64(double x) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x);
  return (b >> 63) ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double unorder_f64(unsigned long long o) {
  return __longlong_as_double((long long)((o >> 63) ? o & ~(1ull << 63) : ~o));
}
// 2^(a - b) for whole numbers a <= b (0 below 2^-1000)
__device__ __forceinline__ double pow2_diff(float a, float b) {
  const float d = a - b;
  return d > -1000.f ? __hiloint2double((1023 + (int)d) << 20, 0) : 0.0;
}
__device__ __forceinline__ float beam_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// (-0 and 0 are equal, NaN counts as -inf)
__device__ __forceinline__ float beam_value(float x) { return x == x ? x + 0.f : -INFINITY; }
__device__ __forceinline__ unsigned long long beam_key(float x, uint32_t i) { return ((unsigned long long)order_f32(x) << 32) | (uint32_t)~i; }

template <typename LT>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_slice_kernel(const BeamParams p) {
  constexpr int N = SampleVec<LT>::N;      // elements of a 16-byte vector
  constexpr int U = 4;                     // vectors in flight
  constexpr int NW = kBeamThreads / 32;
  __shared__ __align__(16) unsigned long long group_key[kBeamGroups];
  __shared__ unsigned long long kept[kBeamKeep];
  __shared__ BeamSum red[NW];
  __shared__ unsigned long long threshold;
  __shared__ int picked[kBeamThreads];     // threads whose elements are read again
  __shared__ int n_picked, n_kept;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int64_t r = blockIdx.y;
  const int sl = blockIdx.x, K = p.n_out;
  const int64_t lo = (int64_t)sl * p.slice;
  const LT* row = reinterpret_cast<const LT*>(p.logits) + r * p.row_stride + lo;
  const int len = (int)(min(lo + p.slice, p.vocab) - lo);   // (elements are counted from the slice's start from here on)
  const bool vec = p.vec_ok != 0;
  // vector v of thread t starts at (v * threads + t) * N; what lies past the end is -inf
  const int nv = (len + kBeamThreads * N - 1) / (kBeamThreads * N);
  auto load = [&](int i, float (&x)[N]) {
    if (vec && i + N <= len) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + i));
      const LT* e = reinterpret_cast<const LT*>(&raw);
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = logit_to_float<LT>(e[k]);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = -INFINITY;
      if (i < len) {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (i + k < len) x[k] = logit_to_float<LT>(__ldg(row + i + k));
      }
    }
  };

  // One pass.  Of the maximum only the batch is kept that it was met in: its place is looked up at the end (some lane of a
  // warp meets a new maximum in nearly every batch, and a search there would cost more than everything else).
  float m = -INFINITY, e2 = -INFINITY;
  int best_v = 0;
  double sum = 0.0;
  // x[] in [.., top]: the running maximum and the sum of exponentials take a batch in
  auto take = [&](int v0, float top, const float (&x)[U * N]) {
    if (top > m) {
      m = top;
      best_v = v0;
      const float e_new = ceilf(m * kBeamLog2e);
      if (e_new > e2) {
        sum *= pow2_diff(e2, e_new);
        e2 = e_new;
      }
    }
    if (m > -INFINITY) {
      const uint64_t l2 = pack_f32x2(kBeamLog2e, kBeamLog2e), ne = pack_f32x2(-e2, -e2);
      uint64_t a0 = 0ull, a1 = 0ull;   // (bit pattern of 0.f, 0.f)
#pragma unroll
      for (int i = 0; i < U * N; i += 4) {
        float y0, y1, y2, y3;
        unpack_f32x2(fma_f32x2(pack_f32x2(x[i], x[i + 1]), l2, ne), y0, y1);
        unpack_f32x2(fma_f32x2(pack_f32x2(x[i + 2], x[i + 3]), l2, ne), y2, y3);
        a0 = add_f32x2(a0, pack_f32x2(beam_ex2(y0), beam_ex2(y1)));
        a1 = add_f32x2(a1, pack_f32x2(beam_ex2(y2), beam_ex2(y3)));
      }
      float s0, s1;
      unpack_f32x2(add_f32x2(a0, a1), s0, s1);
      sum += (double)(s0 + s1);
    }
  };
  const int nv_full = vec ? len / (kBeamThreads * N) / U * U : 0;   // vectors that every thread has in whole, in batches
  const LT* mine_at = row + tid * N;
  auto stream = [&](bool clean) {
    uint4 raw[U], next[U];   // the next batch is on its way while this one is summed up
    if (nv_full > 0) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = __ldg(reinterpret_cast<const uint4*>(mine_at + u * (kBeamThreads * N)));
    }
    for (int v0 = 0; v0 < nv_full; v0 += U) {
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = next[u];
      if (v0 + U < nv_full) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          next[u] = __ldg(reinterpret_cast<const uint4*>(mine_at + (v0 + U + u) * (kBeamThreads * N)));
      }
      float x[U * N], tops[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const LT* e = reinterpret_cast<const LT*>(&raw[u]);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float f = logit_to_float<LT>(e[k]);
          x[u * N + k] = clean ? beam_value(f) : f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        tops[u] = fmaxf(x[u * N], x[u * N + 1]);
#pragma unroll
        for (int k = 2; k < N; k += 2) tops[u] = max3(tops[u], x[u * N + k], x[u * N + k + 1]);
      }
      take(v0, fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), x);
    }
    for (int v0 = nv_full; v0 < nv; v0 += U) {
      float x[U * N], top = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float y[N];
        load(((v0 + u) * kBeamThreads + tid) * N, y);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          x[u * N + k] = clean ? beam_value(y[k]) : y[k];
          top = fmaxf(top, x[u * N + k]);
        }
      }
      take(v0, top, x);
    }
  };
  stream(false);
  if (!(sum == sum)) {   // a NaN or an infinity among the logits
    m = e2 = -INFINITY;
    best_v = 0;
    sum = 0.0;
    stream(true);
  }
  int best_i = tid * N;   // (a thread without a number above -inf: its first element)
  const bool any = best_i < len;
  if (m > -INFINITY) {
    bool found = false;
    for (int v = best_v; !found && v < nv; ++v) {
      const int i = (v * kBeamThreads + tid) * N;
      float x[N];
      load(i, x);
#pragma unroll
      for (int k = N - 1; k >= 0; --k)
        if (x[k] == m) { found = true; best_i = i + k; }   // (the lowest one stays)
    }
  }
  const uint32_t first = (uint32_t)lo;

  // sums and maxima across the CTA
  const unsigned long long mine = any ? beam_key(m + 0.f, first + best_i) : 0ull;
  {
    float e = e2;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) e = fmaxf(e, __shfl_xor_sync(0xffffffffu, e, d));
    double s = e2 > -INFINITY ? sum * pow2_diff(e2, e) : 0.0;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0) red[wid] = BeamSum{s, e, 0.f};
    unsigned long long g = mine;
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      const unsigned long long o = __shfl_xor_sync(0xffffffffu, g, d);
      g = o > g ? o : g;
    }
    if ((tid & 3) == 0) group_key[tid >> 2] = g;
  }
  if (tid == 0) { threshold = 0ull; n_picked = 0; n_kept = 0; }   // (fewer groups with elements than K: everything is kept)
  __syncthreads();
  if (tid < kBeamGroups) {
    const unsigned long long g = group_key[tid];
    int above = 0;
    const ulonglong2* k2 = reinterpret_cast<const ulonglong2*>(group_key);
#pragma unroll 8
    for (int i = 0; i < kBeamGroups / 2; ++i) {
      const ulonglong2 o = k2[i];
      above += (o.x > g) + (o.y > g);
    }
    if (g != 0ull && above == K - 1) threshold = g;
  } else if (wid == NW - 1 && lane == 0) {
    BeamSum t = red[0];
    for (int w = 1; w < NW; ++w) t.e = fmaxf(t.e, red[w].e);
    t.s = 0.0;
    for (int w = 0; w < NW; ++w) t.s += red[w].e > -INFINITY ? red[w].s * pow2_diff(red[w].e, t.e) : 0.0;
    p.part_sum[r * p.n_slices + sl] = t;
  }
  __syncthreads();
  const unsigned long long thr = threshold;
  if (mine != 0ull && mine >= thr) picked[atomicAdd(&n_picked, 1)] = tid;   // (any order: the survivors are ranked)
  __syncthreads();
  const int np = n_picked;
  const float thr_x = thr ? unorder_f32((uint32_t)(thr >> 32)) : -INFINITY;
  for (int j = wid; j < np; j += NW) {       // a warp per thread whose elements are read again
    const int t = picked[j];
    for (int v = lane; v < nv; v += 32) {
      const int i = (v * kBeamThreads + t) * N;
      float x[N];
      load(i, x);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (x[k] < thr_x || i + k >= len) continue;   // (nearly all; NaN goes on)
        const unsigned long long key = beam_key(beam_value(x[k]), first + i + k);
        if (key >= thr) {
          const int at = atomicAdd(&n_kept, 1);
          if (at < kBeamKeep) kept[at] = key;
        }
      }
    }
  }
  __syncthreads();
  const int n = n_kept;
  unsigned long long* out = p.part + (r * p.n_slices + sl) * K;
  if (n <= kBeamKeep) {
    for (int i = tid; i < n; i += kBeamThreads) {
      const unsigned long long key = kept[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += kept[j] > key;
      if (rank < K) out[rank] = key;
    }
    for (int i = n + tid; i < K; i += kBeamThreads) out[i] = 0ull;   // a slice shorter than K
    return;
  }
  // too many to rank: K rounds, each the best element behind the last one
  unsigned long long last = ~0ull;
  for (int rank = 0; rank < K; ++rank) {
    unsigned long long top = 0ull;
    for (int v = 0; v < nv; ++v) {
      const int i = (v * kBeamThreads + tid) * N;
      float x[N];
      load(i, x);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const unsigned long long key = beam_key(beam_value(x[k]), first + i + k);
        if (i + k < len && key < last && key > top) top = key;
      }
    }
    __syncthreads();
    kept[tid] = top;
    __syncthreads();
    for (int d = kBeamThreads / 2; d > 0; d >>= 1) {
      if (tid < d && kept[tid + d] > kept[tid]) kept[tid] = kept[tid + d];
      __syncthreads();
    }
    last = kept[0];
    if (tid == 0) out[rank] = last;
  }
}

// A candidate on the common scale.  Larger is better; equal values by the lower flat index.
struct BeamCand {
  unsigned long long v;   // ordered 64-bit value, 0: none
  unsigned long long i;   // flat index
  __device__ __forceinline__ bool before(const BeamCand& o) const { return v > o.v || (v == o.v && i < o.i); }
};

__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(const BeamParams p) {
  constexpr int NT = kBeamThreads;
  __shared__ double base[kBeamMaxBeams];      // score - log-sum-exp; the score itself for a finished beam
  __shared__ int kind[kBeamMaxBeams];         // 0 a live row, 1 finished, 2 nothing to offer
  __shared__ unsigned long long group_v[kBeamGroups], group_i[kBeamGroups];
  __shared__ unsigned long long kept_v[kBeamKeep], kept_i[kBeamKeep];
  __shared__ unsigned long long thr_v, thr_i;
  __shared__ int n_kept;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int64_t b = blockIdx.x;
  const int W = p.beams, K = p.n_out, S = p.n_slices;
  const int64_t V = p.vocab;
  // log-sum-exps: a warp per row
  for (int w = wid; w < W; w += NT / 32) {
    const BeamSum* ps = p.part_sum + (b * W + w) * S;
    float e = -INFINITY;
    for (int s = lane; s < S; s += 32) e = fmaxf(e, ps[s].e);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) e = fmaxf(e, __shfl_xor_sync(0xffffffffu, e, d));
    double sum = 0.0;
    for (int s = lane; s < S; s += 32) {
      const BeamSum t = ps[s];
      if (t.e > -INFINITY) sum += t.s * pow2_diff(t.e, e);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) {
      const float score = p.scores[b * W + w];
      const bool fin = p.finished && p.finished[b * W + w] != 0;
      const double lse = (double)e / (double)kBeamLog2e + log(sum);
      const bool finite = fabsf(score) < INFINITY && (fin || (lse - lse == 0.0));
      kind[w] = !finite ? 2 : fin ? 1 : 0;
      base[w] = (fin ? (double)score : (double)score - lse) + 0.0;
    }
  }
  if (tid == 0) { n_kept = 0; thr_v = 0ull; thr_i = ~0ull; }
  __syncthreads();

  // candidate c of the request: rank k of slice s of row w.  Neighbouring threads take different rows and slices of one
  // rank, so that the good ones are spread over the threads.
  const int WS = W * S, n_cand = WS * K;
  const unsigned long long kMinusInf = order_f64(-INFINITY);
  auto candidate = [&](int c) -> BeamCand {
    const int k = c / WS, ws = c - k * WS, w = ws / S, s = ws - w * S;
    BeamCand r{0ull, ~0ull};
    const int kd = kind[w];
    if (kd == 0) {
      const unsigned long long key = p.part[((b * W + w) * S + s) * K + k];
      if (key == 0ull) return r;
      const float x = unorder_f32((uint32_t)(key >> 32));
      r.v = order_f64((double)x + base[w]);
      r.i = (unsigned long long)w * V + (uint32_t)~(uint32_t)key;
    } else if (s == 0) {
      // a finished beam goes on by its end token alone; whatever else such a row has is -inf, lowest tokens first
      if (kd == 1 && k == 0) {
        r.v = order_f64(base[w]);
        r.i = (unsigned long long)w * V + p.end_token;
      } else {
        const long long j = kd == 1 ? k - 1 : k, tok = kd == 1 && j >= p.end_token ? j + 1 : j;
        if (tok >= V) return r;
        r.v = kMinusInf;
        r.i = (unsigned long long)w * V + tok;
      }
    }
    return r;
  };
  auto write = [&](int rank, const BeamCand& c) {
    const int64_t at = b * K + rank;
    const int64_t w = (int64_t)(c.i / (unsigned long long)V);
    p.out_tokens[at] = (int64_t)c.i - w * V;
    p.out_parents[at] = w;
    p.out_scores[at] = (float)unorder_f64(c.v);
  };

  const bool one = n_cand <= NT;   // a thread has one candidate at most: it stays in registers
  BeamCand best{0ull, ~0ull};
  for (int c = tid; c < n_cand; c += NT) {
    const BeamCand v = candidate(c);
    if (v.v != 0ull && v.before(best)) best = v;
  }
  BeamCand g = best;
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    const BeamCand o{__shfl_xor_sync(0xffffffffu, g.v, d), __shfl_xor_sync(0xffffffffu, g.i, d)};
    if (o.before(g)) g = o;
  }
  if ((tid & 3) == 0) { group_v[tid >> 2] = g.v; group_i[tid >> 2] = g.i; }
  __syncthreads();
  if (tid < kBeamGroups) {
    const BeamCand mine{group_v[tid], group_i[tid]};
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < kBeamGroups; ++i) above += BeamCand{group_v[i], group_i[i]}.before(mine);
    if (mine.v != 0ull && above == K - 1) { thr_v = mine.v; thr_i = mine.i; }
  }
  __syncthreads();
  const BeamCand thr{thr_v, thr_i};
  if (best.v != 0ull && !thr.before(best)) {
    for (int c = tid; c < n_cand; c += NT) {
      const BeamCand v = one ? best : candidate(c);
      if (v.v == 0ull || thr.before(v)) continue;
      const int at = atomicAdd(&n_kept, 1);
      if (at < kBeamKeep) { kept_v[at] = v.v; kept_i[at] = v.i; }
    }
  }
  __syncthreads();
  const int n = n_kept;
  if (n <= kBeamKeep) {
    for (int i = tid; i < n; i += NT) {
      const BeamCand c{kept_v[i], kept_i[i]};
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += BeamCand{kept_v[j], kept_i[j]}.before(c);
      if (rank < K) write(rank, c);
    }
    return;
  }
  // too many survivors to rank: K rounds, each the best candidate behind the last one
  BeamCand last{~0ull, 0ull};
  for (int rank = 0; rank < K; ++rank) {
    BeamCand mine{0ull, ~0ull};
    for (int c = tid; c < n_cand; c += NT) {
      const BeamCand v = candidate(c);
      if (v.v != 0ull && last.before(v) && v.before(mine)) mine = v;
    }
    __syncthreads();
    kept_v[tid] = mine.v;
    kept_i[tid] = mine.i;
    __syncthreads();
    for (int d = NT / 2; d > 0; d >>= 1) {
      if (tid < d) {
        const BeamCand o{kept_v[tid + d], kept_i[tid + d]};
        if (o.before(BeamCand{kept_v[tid], kept_i[tid]})) { kept_v[tid] = o.v; kept_i[tid] = o.i; }
      }
      __syncthreads();
    }
    last = BeamCand{kept_v[0], kept_i[0]};
    if (tid == 0) write(rank, last);
  }
}

// Slices per row: enough CTAs to fill every SM, none below 2048 elements (a vector of 16-bit logits per thread).
inline int beam_slice_len(int64_t rows, int64_t vocab, int sms) {
  int64_t n = (kBeamCtasPerSm * (int64_t)sms + rows - 1) / rows;
  if (n > (vocab + 2047) / 2048) n = (vocab + 2047) / 2048;
  if (n < 1) n = 1;
  return (int)(((vocab + n - 1) / n + 7) / 8 * 8);
}
inline uint64_t beam_workspace_need(int64_t batch, int64_t beams, int64_t vocab, int64_t n_out, int sms) {
  const int64_t rows = batch * beams, slice = beam_slice_len(rows, vocab, sms), S = (vocab + slice - 1) / slice;
  return (uint64_t)(rows * S * n_out * 8 + rows * S * sizeof(BeamSum));
}

template <typename LT>
inline int launch_beam_slices(const BeamParams& p, cudaStream_t stream) {
  const dim3 grid((unsigned)p.n_slices, (unsigned)(p.batch * p.beams));
  KB200_CUDA_OK(launch_kernel(beam_slice_kernel<LT>, grid, dim3(kBeamThreads), 0, stream, p));
  return KB200_OK;
}

// ---------------------------------------------------------------------------
// Reordering.  Beam w of a request goes on from beam parent[w].  Full pages are immutable: their table entries are gathered.
// The page that is still being filled is private to a beam: its first L mod P tokens are copied from the parent's,
// in every pool.  Parents permute and repeat, so a page is source and destination at once; one thread owns the same 16 bytes
// of all the beams' pages, reads what it needs and then writes, and no staging buffer or second launch is needed.
// HBM-bound: (distinct sources + moved beams) * (L mod P) tokens of every pool.  Measured: 32 requests of 8 beams, 24 int8 layers of
// 8 heads of 128 in pages of 16, 35 us = 4.5 TB/s; 2 requests of 4 beams, 24 bf16 layers, 3.7 us.
// ---------------------------------------------------------------------------
constexpr int kReorderPools = 96;
struct ReorderParams {
  char* pools[kReorderPools];     // [n_pages][heads][page_size][row]
  float* scales[kReorderPools];   // [n_pages][heads], one per block of an int8 pool
  int32_t* table;               // the beams' tables, rows b * W + w
  const int32_t* own;           // private pages, row own_rows[b * W + w] (or b * W + w)
  const int64_t* own_rows;
  const void* parents;
  const int32_t* lengths;
  int64_t table_rs, own_rs, own_n_rows, cols, n_pages;
  int64_t page_stride_b, head_stride_b;   // bytes
  int64_t scale_page_stride;              // elements
  int32_t n_pools, n_scales, n_heads, row_bytes, page_size, batch, beams, parents_is_i64;
  int32_t tables;                         // this launch gathers the tables too
};

__device__ __forceinline__ int reorder_parent(const ReorderParams& p, int64_t b, int w) {
  const int64_t i = b * p.beams + w;
  const int64_t q = p.parents_is_i64 ? static_cast<const int64_t*>(p.parents)[i] : static_cast<const int32_t*>(p.parents)[i];
  return q >= 0 && q < p.beams ? (int)q : -1;
}

// grid (planes, batch, parts of a plane): a plane for the tables, one per pool, one for all the scale arrays
template <typename Vec, int MAXW>
__global__ void __launch_bounds__(256) reorder_kernel(const ReorderParams p) {
  __shared__ int parent[MAXW];        // -1: stays as it is
  __shared__ int64_t page[MAXW];      // the private page that is being filled
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, W = p.beams;
  const int64_t b = blockIdx.y;
  const int L = p.lengths[b], P = p.page_size;
  const int full = L > 0 ? L / P : 0, rest = L > 0 ? L - full * P : 0;
  const bool table = p.tables && blockIdx.x == 0;
  if (tid < W) {
    int q = reorder_parent(p, b, tid);
    if (q < 0 && table) report(KB200_STATUS_BAD_ROW, (int)(b * W + tid), KID_REORDER);
    const int64_t r = p.own_rows ? p.own_rows[b * W + tid] : b * W + tid;
    const bool row_ok = r >= 0 && r < p.own_n_rows && full < p.cols;
    page[tid] = rest > 0 && row_ok ? p.own[r * p.own_rs + full] : -1;
    if (rest > 0 && (page[tid] < 0 || page[tid] >= p.n_pages)) {
      if (table) report(row_ok ? KB200_STATUS_BAD_PAGE : KB200_STATUS_BAD_ROW, (int)page[tid], KID_REORDER);
      page[tid] = -1;
    }
    parent[tid] = q == tid ? -1 : q;
  }
  __syncthreads();
  if (table) {   // a thread owns one column of the request's rows
    if (blockIdx.z != 0) return;
    if (full > p.cols) { if (tid == 0) report(KB200_STATUS_BAD_ROW, L, KID_REORDER); return; }
    int32_t* t = p.table + b * W * p.table_rs;
    for (int c = tid; c < full; c += 256) {
      int32_t v[MAXW];
#pragma unroll
      for (int w = 0; w < MAXW; ++w)
        if (w < W && parent[w] >= 0) v[w] = t[parent[w] * p.table_rs + c];
#pragma unroll
      for (int w = 0; w < MAXW; ++w)
        if (w < W && parent[w] >= 0) t[w * p.table_rs + c] = v[w];
    }
    return;
  }
  if (rest == 0) return;
  const int plane = (int)blockIdx.x - p.tables;
  if (plane == p.n_pools) {   // a block's scale goes with its codes
    for (int i = tid + 256 * blockIdx.z; i < p.n_scales * p.n_heads; i += 256 * gridDim.z) {
      float* at = p.scales[i / p.n_heads] + i % p.n_heads;
      float v[MAXW];
#pragma unroll
      for (int w = 0; w < MAXW; ++w)
        if (w < W && parent[w] >= 0 && page[w] >= 0 && page[parent[w]] >= 0) v[w] = at[page[parent[w]] * p.scale_page_stride];
#pragma unroll
      for (int w = 0; w < MAXW; ++w)
        if (w < W && parent[w] >= 0 && page[w] >= 0 && page[parent[w]] >= 0) at[page[w] * p.scale_page_stride] = v[w];
    }
    return;
  }
  char* pool = p.pools[plane];
  const int per_head = rest * p.row_bytes / (int)sizeof(Vec);   // vectors of one head's filled rows
  const int total = per_head * p.n_heads;
  for (int i = tid + 256 * blockIdx.z; i < total; i += 256 * gridDim.z) {
    const int h = i / per_head, c = i - h * per_head;
    char* at = pool + h * p.head_stride_b + (int64_t)c * sizeof(Vec);
    Vec v[MAXW];
#pragma unroll
    for (int w = 0; w < MAXW; ++w)
      if (w < W && parent[w] >= 0 && page[w] >= 0 && page[parent[w]] >= 0)
        v[w] = *reinterpret_cast<const Vec*>(at + page[parent[w]] * p.page_stride_b);
#pragma unroll
    for (int w = 0; w < MAXW; ++w)
      if (w < W && parent[w] >= 0 && page[w] >= 0 && page[parent[w]] >= 0)
        *reinterpret_cast<Vec*>(at + page[w] * p.page_stride_b) = v[w];
  }
}

inline int launch_beam_step(const void* logits, int logits_dtype, int64_t batch, int64_t beams, int64_t vocab, int64_t row_stride,
                            const float* scores, const uint8_t* finished, int64_t end_token, int64_t n_out, int64_t* out_tokens,
                            int64_t* out_parents, float* out_scores, void* workspace, uint64_t workspace_bytes, int device,
                            cudaStream_t stream) {
  KB200_REQUIRE(batch >= 0 && vocab > 0 && beams > 0 && n_out > 0, "batch must be non-negative, beams, vocab and n_out positive");
  if (batch == 0) return KB200_OK;
  if (beams > kBeamMaxBeams || n_out > kBeamMaxOut)
    return fail(KB200_ERR_UNSUPPORTED, "%lld beams with %lld candidates are not supported (at most %d and %d)", (long long)beams,
                (long long)n_out, kBeamMaxBeams, kBeamMaxOut);
  KB200_REQUIRE(vocab <= (1ll << 20), "vocab above 2^20 is not supported");
  KB200_REQUIRE(n_out <= beams * vocab, "more candidates than there are (beam, token) pairs");
  KB200_REQUIRE(batch * beams <= 65535, "too many rows");
  KB200_REQUIRE(logits && scores && out_tokens && out_parents && out_scores, "null pointer argument");
  KB200_REQUIRE(row_stride >= vocab, "row_stride is smaller than the vocabulary");
  KB200_REQUIRE(!finished || (end_token >= 0 && end_token < vocab), "end_token must be a token of the vocabulary");
  const int es = dtype_size(logits_dtype);
  KB200_REQUIRE(logits_dtype == KB200_DTYPE_F32 || logits_dtype == KB200_DTYPE_F16 || logits_dtype == KB200_DTYPE_BF16,
                "logits must be F32, F16 or BF16");
  int sms = 0;
  if (int rc = device_sm_count(device, &sms)) return rc;
  const uint64_t need = beam_workspace_need(batch, beams, vocab, n_out, sms);
  if (!workspace || workspace_bytes < need)
    return fail(KB200_ERR_WORKSPACE, "workspace too small: need %llu bytes, got %llu", (unsigned long long)need,
                (unsigned long long)workspace_bytes);
  KB200_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "workspace must be 16-byte aligned");
  BeamParams p;
  p.logits = static_cast<const char*>(logits);
  p.scores = scores;
  p.finished = finished;
  p.out_tokens = out_tokens;
  p.out_parents = out_parents;
  p.out_scores = out_scores;
  p.row_stride = row_stride;
  p.vocab = vocab;
  p.end_token = end_token;
  p.batch = (int)batch;
  p.beams = (int)beams;
  p.n_out = (int)n_out;
  p.slice = beam_slice_len(batch * beams, vocab, sms);
  p.n_slices = (int)((vocab + p.slice - 1) / p.slice);
  p.part_sum = static_cast<BeamSum*>(workspace);
  p.part = reinterpret_cast<unsigned long long*>(p.part_sum + batch * beams * p.n_slices);
  p.vec_ok = ((reinterpret_cast<uintptr_t>(logits) & 15) == 0 && (row_stride * es) % 16 == 0) ? 1 : 0;
  int rc;
  if (logits_dtype == KB200_DTYPE_F32) rc = launch_beam_slices<float>(p, stream);
  else if (logits_dtype == KB200_DTYPE_F16) rc = launch_beam_slices<__half>(p, stream);
  else rc = launch_beam_slices<__nv_bfloat16>(p, stream);
  if (rc) return rc;
  KB200_CUDA_OK(launch_kernel(beam_merge_kernel, dim3((unsigned)batch), dim3(kBeamThreads), 0, stream, p));
  return KB200_OK;
}

template <typename Vec>
inline int launch_reorder_vec(const ReorderParams& p, dim3 grid, cudaStream_t stream) {
  if (p.beams <= 4) KB200_CUDA_OK(launch_kernel(reorder_kernel<Vec, 4>, grid, dim3(256), 0, stream, p));
  else if (p.beams <= 8) KB200_CUDA_OK(launch_kernel(reorder_kernel<Vec, 8>, grid, dim3(256), 0, stream, p));
  else if (p.beams <= 16) KB200_CUDA_OK(launch_kernel(reorder_kernel<Vec, 16>, grid, dim3(256), 0, stream, p));
  else KB200_CUDA_OK(launch_kernel(reorder_kernel<Vec, 32>, grid, dim3(256), 0, stream, p));
  return KB200_OK;
}

inline int launch_reorder(void* const* pools, int n_pools, float* const* scales, int n_scales, int64_t page_stride_b,
                          int64_t head_stride_b, int row_bytes, int n_heads, int64_t scale_page_stride, int64_t n_pages,
                          int32_t* table, int64_t table_rs, int64_t table_cols, const int32_t* own, int64_t own_rs,
                          int64_t own_n_rows, int64_t own_cols, const int64_t* own_rows, const void* parents,
                          int parents_is_i64, const int32_t* lengths, int64_t batch, int beams, int page_size, int device,
                          cudaStream_t stream) {
  KB200_REQUIRE(batch >= 0 && beams > 0 && n_pools >= 0 && n_scales >= 0, "batch must be non-negative and beams positive");
  if (batch == 0) return KB200_OK;
  if (beams > 32) return fail(KB200_ERR_UNSUPPORTED, "%d beams are not supported (at most 32)", beams);
  KB200_REQUIRE(batch <= 65535, "batch out of range");
  KB200_REQUIRE(table && own && parents && lengths && (n_pools == 0 || pools) && (n_scales == 0 || scales), "null pointer argument");
  KB200_REQUIRE(page_size > 0 && n_pages > 0 && table_cols > 0 && own_cols > 0, "page_size, n_pages and the tables must not be empty");
  KB200_REQUIRE(n_pools == 0 || (n_heads > 0 && row_bytes > 0), "n_heads and row_bytes must be positive");
  KB200_REQUIRE((int64_t)page_size * row_bytes <= 0x7fffffff / (n_heads > 0 ? n_heads : 1), "pages are too large");
  int sms = 0;
  if (int rc = device_sm_count(device, &sms)) return rc;
  bool vec = page_stride_b % 16 == 0 && head_stride_b % 16 == 0 && row_bytes % 16 == 0;
  for (int i = 0; i < n_pools; ++i) {
    KB200_REQUIRE(pools[i], "null pointer argument");
    vec = vec && (reinterpret_cast<uintptr_t>(pools[i]) & 15) == 0;
  }
  for (int i = 0; i < n_scales; ++i) KB200_REQUIRE(scales[i], "null pointer argument");
  ReorderParams p;
  p.table = table;
  p.own = own;
  p.own_rows = own_rows;
  p.parents = parents;
  p.lengths = lengths;
  p.table_rs = table_rs;
  p.own_rs = own_rs;
  p.own_n_rows = own_n_rows;
  p.cols = table_cols < own_cols ? table_cols : own_cols;
  p.n_pages = n_pages;
  p.page_stride_b = page_stride_b;
  p.head_stride_b = head_stride_b;
  p.scale_page_stride = scale_page_stride;
  p.n_heads = n_heads;
  p.row_bytes = row_bytes;
  p.page_size = page_size;
  p.batch = (int)batch;
  p.beams = beams;
  p.parents_is_i64 = parents_is_i64;
  int done_p = 0, done_s = 0;
  do {   // (pools by value, 96 a launch: 24 layers of K and V take one)
    p.tables = done_p == 0 && done_s == 0 ? 1 : 0;
    p.n_pools = n_pools - done_p < kReorderPools ? n_pools - done_p : kReorderPools;
    p.n_scales = n_scales - done_s < kReorderPools ? n_scales - done_s : kReorderPools;
    for (int i = 0; i < p.n_pools; ++i) p.pools[i] = static_cast<char*>(pools[done_p + i]);
    for (int i = 0; i < p.n_scales; ++i) p.scales[i] = scales[done_s + i];
    const int planes = p.tables + p.n_pools + (p.n_scales > 0 ? 1 : 0);
    // enough CTAs to fill the GPU four times over, none with less than a vector per thread of a full page
    const int64_t vectors = p.n_pools > 0 ? (int64_t)page_size * row_bytes * n_heads / 16 : 256;
    int64_t z = ((int64_t)sms * 4 + planes * batch - 1) / (planes * batch);
    if (z > (vectors + 255) / 256) z = (vectors + 255) / 256;
    if (z < 1) z = 1;
    const dim3 grid((unsigned)planes, (unsigned)batch, (unsigned)z);
    if (int rc = vec ? launch_reorder_vec<uint4>(p, grid, stream) : launch_reorder_vec<uint8_t>(p, grid, stream)) return rc;
    done_p += p.n_pools;
    done_s += p.n_scales;
  } while (done_p < n_pools || done_s < n_scales);
  return KB200_OK;
}

}  // namespace kb200
