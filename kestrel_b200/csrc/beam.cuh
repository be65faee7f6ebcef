// Beam search on the paged cache: selection over beams and vocabulary, and the reordering of the beams' pages.
//
// Selection.  cand(w, v) = score_w + x_wv - log sum_u exp x_wu; the K largest over the W * V candidates of a request, equal
// ones by the lowest w * V + v.  Inside a row the order is the logits' own, so a row's K best are found on the logits
// (exactly, in one pass that also gathers maximum and sum); only the few survivors are put on the common scale, in 64 bits.
//   beam_slice_kernel  one CTA per slice of a row, the slice in registers.  The K-th largest of the 256 threads' own
//                      maxima is a threshold that the slice's K best cannot lie below, and what lies at or above it
//                      belongs to K threads: at most K * EPT elements to rank, K and a few as a rule.
//   beam_merge_kernel  one CTA per request: log-sum-exps of its rows, then the same threshold over their candidates.
// HBM-bound: the logits are read once.  Nothing depends on the order in which threads arrive.
#pragma once

#include "sampling.cuh"

namespace kb200 {

constexpr int kBeamThreads = 256;
constexpr int kBeamMaxOut = 64;
constexpr int kBeamMaxBeams = 64;
constexpr int kBeamMergeThreads = 512;
constexpr int kBeamMergeKeep = 1024;   // survivors that the merge ranks at once; more (never seen) take the slow way

struct BeamParams {
  const char* logits;
  const float* scores;
  const uint8_t* finished;     // or nullptr
  unsigned long long* part;    // [rows][slices][K] keys: ordered logit << 32 | ~index
  float2* part_ml;             // [rows][slices] maximum, sum of exp(x - maximum)
  int64_t* out_tokens;
  int64_t* out_parents;
  float* out_scores;
  int64_t row_stride, vocab, end_token;
  int batch, beams, n_out, n_slices, slice, vec_ok;
};

// floats ordered as unsigned integers, NaN below everything but 0
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

// EPT elements per thread, in vectors of 16 bytes
template <typename LT, int EPT>
__global__ void __launch_bounds__(kBeamThreads) beam_slice_kernel(const BeamParams p) {
  constexpr int N = SampleVec<LT>::N;
  constexpr int NV = EPT / N;
  __shared__ __align__(16) unsigned long long keys[kBeamThreads];
  __shared__ unsigned long long kept[kBeamMaxOut * EPT];
  __shared__ float red_m[kBeamThreads / 32];
  __shared__ double red_s[kBeamThreads / 32];
  __shared__ unsigned long long threshold;
  __shared__ int n_kept;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int64_t r = blockIdx.y;
  const int sl = blockIdx.x, K = p.n_out;
  const LT* row = reinterpret_cast<const LT*>(p.logits) + r * p.row_stride;
  const int64_t lo = (int64_t)sl * p.slice, hi = min(lo + p.slice, p.vocab);

  // the slice: vector j of this thread starts at lo + (j * threads + tid) * N; what lies past the end is -inf
  float x[EPT];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t i = lo + ((int64_t)j * kBeamThreads + tid) * N;
    if (p.vec_ok && i + N <= hi) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + i));
      const LT* e = reinterpret_cast<const LT*>(&raw);
#pragma unroll
      for (int k = 0; k < N; ++k) x[j * N + k] = logit_to_float<LT>(e[k]);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) x[j * N + k] = i + k < hi ? logit_to_float<LT>(__ldg(row + i + k)) : -INFINITY;
    }
  }
  auto index_of = [&](int e) { return (uint32_t)(lo + ((int64_t)(e / N) * kBeamThreads + tid) * N + e % N); };
  // this thread's best: largest value, then lowest index (indices ascend with e)
  float best = -INFINITY;
  int best_e = 0;
  if (tid == 0) n_kept = 0;
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    x[e] = x[e] == x[e] ? x[e] + 0.f : -INFINITY;   // NaN: never chosen before a number; -0 and 0 are equal
    if (x[e] > best) { best = x[e]; best_e = e; }
  }
  const uint32_t first_i = index_of(0);
  const bool any = first_i < hi;
  keys[tid] = any ? ((unsigned long long)order_f32(best) << 32) | (uint32_t)~index_of(best_e) : 0ull;
  float m = best;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (lane == 0) red_m[wid] = m;
  __syncthreads();
  m = red_m[0];
#pragma unroll
  for (int w = 1; w < kBeamThreads / 32; ++w) m = fmaxf(m, red_m[w]);

  // sum of exp(x - m): fp32 inside a thread (at most EPT terms), 64 bits across
  float s = 0.f;
  if (m > -INFINITY) {
#pragma unroll
    for (int e = 0; e < EPT; ++e) s += exp2f((x[e] - m) * 1.4426950408889634f);
  }
  double sd = s;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sd += __shfl_xor_sync(0xffffffffu, sd, d);
  if (lane == 0) red_s[wid] = sd;

  // rank of this thread's maximum among the threads' (keys are distinct, but for the zeros of empty threads)
  const unsigned long long mine = keys[tid];
  int above = 0;
  const ulonglong2* k2 = reinterpret_cast<const ulonglong2*>(keys);
#pragma unroll 8
  for (int i = 0; i < kBeamThreads / 2; ++i) {
    const ulonglong2 v = k2[i];
    above += (v.x > mine) + (v.y > mine);
  }
  if (tid == 0) threshold = 0ull;   // (fewer threads with elements than K: everything is kept)
  __syncthreads();
  if (mine != 0ull && above == K - 1) threshold = mine;
  if (tid == 0) {
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < kBeamThreads / 32; ++w) t += red_s[w];
    p.part_ml[r * p.n_slices + sl] = make_float2(m, (float)t);
  }
  __syncthreads();
  const unsigned long long thr = threshold;
  if (mine != 0ull && mine >= thr) {
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const uint32_t i = index_of(e);
      const unsigned long long key = ((unsigned long long)order_f32(x[e]) << 32) | (uint32_t)~i;
      if (i < hi && key >= thr) kept[atomicAdd(&n_kept, 1)] = key;   // (their order is settled by the ranks below)
    }
  }
  __syncthreads();
  const int n = n_kept;
  unsigned long long* out = p.part + (r * p.n_slices + sl) * K;
  for (int i = tid; i < n; i += kBeamThreads) {
    const unsigned long long key = kept[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += kept[j] > key;
    if (rank < K) out[rank] = key;
  }
  for (int i = n + tid; i < K; i += kBeamThreads) out[i] = 0ull;   // a slice shorter than K
}

// A candidate on the common scale.  Larger is better; equal values by the lower flat index.
struct BeamCand {
  unsigned long long v;   // ordered 64-bit value, 0: none
  unsigned long long i;   // flat index
  __device__ __forceinline__ bool before(const BeamCand& o) const { return v > o.v || (v == o.v && i < o.i); }
};

__global__ void __launch_bounds__(kBeamMergeThreads) beam_merge_kernel(const BeamParams p) {
  constexpr int NT = kBeamMergeThreads;
  __shared__ double base[kBeamMaxBeams];      // score - log-sum-exp; the score itself for a finished beam
  __shared__ int kind[kBeamMaxBeams];         // 0 a live row, 1 finished, 2 nothing to offer
  __shared__ unsigned long long top_v[NT], top_i[NT];
  __shared__ unsigned long long kept_v[kBeamMergeKeep], kept_i[kBeamMergeKeep];
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
    const float2* ml = p.part_ml + (b * W + w) * S;
    float m = -INFINITY;
    for (int s = lane; s < S; s += 32) m = fmaxf(m, ml[s].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    double sum = 0.0;
    for (int s = lane; s < S; s += 32) sum += ml[s].x > -INFINITY ? (double)ml[s].y * exp((double)ml[s].x - (double)m) : 0.0;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) {
      const float score = p.scores[b * W + w];
      const bool fin = p.finished && p.finished[b * W + w] != 0;
      const double lse = (double)m + log(sum);
      const bool finite = fabsf(score) < INFINITY && (fin || (lse - lse == 0.0));
      kind[w] = !finite ? 2 : fin ? 1 : 0;
      base[w] = (fin ? (double)score : (double)score - lse) + 0.0;
    }
  }
  if (tid == 0) { n_kept = 0; thr_v = 0ull; thr_i = ~0ull; }
  __syncthreads();

  // candidate c of the request: rank k of slice s of row w.  Neighbouring threads take different rows and slices of one
  // rank, so that the good ones are spread over the threads.
  const int n_cand = W * S * K;
  const unsigned long long kMinusInf = order_f64(-INFINITY);
  auto candidate = [&](int c) -> BeamCand {
    const int k = c / (W * S), ws = c - k * (W * S), w = ws / S, s = ws - w * S;
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

  BeamCand best{0ull, ~0ull};
  for (int c = tid; c < n_cand; c += NT) {
    const BeamCand v = candidate(c);
    if (v.v != 0ull && v.before(best)) best = v;
  }
  top_v[tid] = best.v;
  top_i[tid] = best.i;
  __syncthreads();
  if (best.v != 0ull) {
    int above = 0;
    for (int i = 0; i < NT; ++i) above += BeamCand{top_v[i], top_i[i]}.before(best);
    if (above == K - 1) { thr_v = best.v; thr_i = best.i; }
  }
  __syncthreads();
  const BeamCand thr{thr_v, thr_i};
  if (best.v != 0ull && !thr.before(best)) {
    for (int c = tid; c < n_cand; c += NT) {
      const BeamCand v = candidate(c);
      if (v.v == 0ull || thr.before(v)) continue;
      const int at = atomicAdd(&n_kept, 1);
      if (at < kBeamMergeKeep) { kept_v[at] = v.v; kept_i[at] = v.i; }
    }
  }
  __syncthreads();
  const int n = n_kept;
  if (n <= kBeamMergeKeep) {
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
    top_v[tid] = mine.v;
    top_i[tid] = mine.i;
    __syncthreads();
    for (int d = NT / 2; d > 0; d >>= 1) {
      if (tid < d) {
        const BeamCand o{top_v[tid + d], top_i[tid + d]};
        if (o.before(BeamCand{top_v[tid], top_i[tid]})) { top_v[tid] = o.v; top_i[tid] = o.i; }
      }
      __syncthreads();
    }
    last = BeamCand{top_v[0], top_i[0]};
    if (tid == 0) write(rank, last);
  }
}

// Elements per thread of the slice kernel: 32 (one wave of loads in flight, few partial lists), 8 when the rows
// alone would not give every SM a CTA.
inline int beam_slice_len(int64_t rows, int64_t vocab, int sms) {
  const int64_t big = 32 * kBeamThreads;
  return rows * ((vocab + big - 1) / big) >= sms ? (int)big : 8 * kBeamThreads;
}
inline uint64_t beam_workspace_need(int64_t batch, int64_t beams, int64_t vocab, int64_t n_out, int sms) {
  const int64_t rows = batch * beams, slice = beam_slice_len(rows, vocab, sms), S = (vocab + slice - 1) / slice;
  return (uint64_t)(rows * S * n_out * 8 + rows * S * 8);
}

template <typename LT>
inline int launch_beam_slices(const BeamParams& p, cudaStream_t stream) {
  const dim3 grid((unsigned)p.n_slices, (unsigned)(p.batch * p.beams));
  if (p.slice == 32 * kBeamThreads) KB200_CUDA_OK(launch_kernel(beam_slice_kernel<LT, 32>, grid, dim3(kBeamThreads), 0, stream, p));
  else KB200_CUDA_OK(launch_kernel(beam_slice_kernel<LT, 8>, grid, dim3(kBeamThreads), 0, stream, p));
  return KB200_OK;
}

// ---------------------------------------------------------------------------
// Reordering.  Beam w of a request goes on from beam parent[w].  Full pages are immutable: their table entries are gathered.
// The page that is still being filled is private to a beam: its first L mod P tokens are copied from the parent's,
// in every pool.  Parents permute and repeat, so a page is source and destination at once; one thread owns the same 16 bytes
// of all the beams' pages, reads what it needs and then writes, and no staging buffer or second launch is needed.
// HBM-bound: (distinct sources + moved beams) * (L mod P) tokens of every pool.
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
  p.part = static_cast<unsigned long long*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part + batch * beams * p.n_slices * n_out);
  p.vec_ok = ((reinterpret_cast<uintptr_t>(logits) & 15) == 0 && (row_stride * es) % 16 == 0) ? 1 : 0;
  int rc;
  if (logits_dtype == KB200_DTYPE_F32) rc = launch_beam_slices<float>(p, stream);
  else if (logits_dtype == KB200_DTYPE_F16) rc = launch_beam_slices<__half>(p, stream);
  else rc = launch_beam_slices<__nv_bfloat16>(p, stream);
  if (rc) return rc;
  KB200_CUDA_OK(launch_kernel(beam_merge_kernel, dim3((unsigned)batch), dim3(kBeamMergeThreads), 0, stream, p));
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
