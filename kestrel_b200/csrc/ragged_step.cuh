// The tables of one step built on the GPU from request lengths: page allocation from a free list in device memory, block
// tables, slot map, positions, packed row offsets.
//
//   need_i = ceil((L_i + n_i) / P) - ceil(L_i / P), C_i = need_0 + .. + need_i
//   page j that entry i takes = free[count - C_i + j]   (what PageTable.reserve hands out, called entry after entry)
//
// The whole step is one thread-block cluster.  Every CTA scans the (few) requests into its shared memory, so the tokens and
// table entries can be cut anywhere; a page that is being handed out is read from the free list, not from the table that
// another CTA is filling.  The cluster barrier stands between the reads of the inputs and the writes of the counts,
// so out_seqused_k may be `lengths` and out_free_count may be `free_count`: a captured graph advances its own state.
// No scratch memory and no counter that two graphs could share.
// Latency-bound: 16 bytes per token and 8 per table entry, a few MB at most; what counts is one launch and one scan.
// Measured: 256 decode requests of up to 8k tokens 5.4 us, 1000 requests with 128k new tokens 11 us (3.1 MB).
#pragma once

#include "common.cuh"

namespace kb200 {

struct RaggedParams {
  int32_t* page_table;
  const void* batch_idx;
  const int32_t* lengths;
  const int32_t* new_tokens;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* out_page_table;
  int32_t* out_seqused;
  int32_t* out_cu;
  int64_t* out_slots;
  int64_t* out_positions;
  int32_t* out_free_count;
  int32_t* out_taken;
  int64_t pt_rs, pt_rows, pt_cols, out_rs, out_cols, free_cap, n_pages, n_tokens;
  int32_t batch, page_size, batch_idx_is_i64;
};

constexpr int kRaggedThreads = 1024;
constexpr int kRaggedMaxBatch = 8192;
constexpr int kRaggedMaxCluster = 16;   // more than the portable 8 where the device can hold it

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// dynamic shared memory: four int arrays of batch + 1
__global__ void __launch_bounds__(kRaggedThreads, 1) ragged_step_kernel(const RaggedParams p) {
  extern __shared__ int ragged_smem[];
  __shared__ long long warp_n[32], warp_p[32], carry_n, carry_p;
  __shared__ int bad;
  int* cu = ragged_smem;                     // first packed token of an entry
  int* pc = cu + p.batch + 1;                // pages taken by the entries before
  int* len = pc + p.batch + 1;               // tokens held before, -1: an entry that cannot be served
  int* row = len + p.batch + 1;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int rank = blockIdx.x, n_cta = gridDim.x;
  const int P = p.page_size;
  if (tid == 0) { carry_n = 0; carry_p = 0; bad = 0; }
  __syncthreads();
  const long long most = min(p.pt_cols, p.out_cols) * P;
  for (int base = 0; base < p.batch; base += kRaggedThreads) {
    const int i = base + tid;
    long long n = 0, np = 0;
    if (i < p.batch) {
      const int64_t r = p.batch_idx_is_i64 ? static_cast<const int64_t*>(p.batch_idx)[i] : static_cast<const int32_t*>(p.batch_idx)[i];
      const long long L = p.lengths[i], want = p.new_tokens[i];
      const bool ok = r >= 0 && r < p.pt_rows && L >= 0 && want >= 0 && L + want <= most;
      if (!ok && rank == 0) report(KB200_STATUS_BAD_ROW, i, KID_RAGGED);
      n = ok ? want : 0;
      // (row 0 is the padding row: its tokens go to page 0, it is never given a page)
      np = ok && r != 0 ? (L + want + P - 1) / P - (L + P - 1) / P : 0;
      len[i] = ok ? (int)L : -1;
      row[i] = ok ? (int)r : 0;
    }
    long long sn = n, sp = np;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long un = __shfl_up_sync(0xffffffffu, sn, d), up = __shfl_up_sync(0xffffffffu, sp, d);
      if (lane >= d) { sn += un; sp += up; }
    }
    if (lane == 31) { warp_n[wid] = sn; warp_p[wid] = sp; }
    __syncthreads();
    if (wid == 0) {
      long long wn = warp_n[lane], wp = warp_p[lane];
      const long long n0 = wn, p0 = wp;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long un = __shfl_up_sync(0xffffffffu, wn, d), up = __shfl_up_sync(0xffffffffu, wp, d);
        if (lane >= d) { wn += un; wp += up; }
      }
      warp_n[lane] = carry_n + wn - n0;
      warp_p[lane] = carry_p + wp - p0;
      __syncwarp();
      if (lane == 31) { carry_n += wn; carry_p += wp; }
    }
    __syncthreads();
    if (i < p.batch) {
      const long long en = warp_n[wid] + sn - n, ep = warp_p[wid] + sp - np;
      if (en > 0x7fffffff || ep > 0x7fffffff) bad = 1;
      cu[i] = (int)en;
      pc[i] = (int)ep;
    }
    __syncthreads();
  }
  const long long all_n = carry_n, all_p = carry_p;
  const int count = *p.free_count;
  // all or nothing: a step that does not fit takes no page and has no tokens
  const bool fits = !bad && all_n <= p.n_tokens && count >= 0 && count <= p.free_cap && all_p <= count;
  if (tid == 0) { cu[p.batch] = fits ? (int)all_n : 0; pc[p.batch] = fits ? (int)all_p : 0; }
  __syncthreads();
  cluster_arrive();   // this CTA has read lengths and free_count for the last time

  // pages of P tokens: a shift where P is a power of two (a 32-bit division otherwise; lengths are below 2^31)
  const int shift = (P & (P - 1)) == 0 ? 31 - __clz(P) : -1;
  auto pages_of = [&](uint32_t x) { return (int)(shift >= 0 ? x >> shift : x / (uint32_t)P); };
  auto tokens_of = [&](int i) { return fits ? cu[i + 1] - cu[i] : 0; };
  auto held_by = [&](int i) { return pages_of((uint32_t)len[i] + P - 1); };
  // block tables: a warp per entry, kCopies loads of a lane in flight
  constexpr int kCopies = 8;
  for (int i = rank * 32 + wid; i < p.batch; i += n_cta * 32) {
    if (len[i] < 0) continue;
    const int held = held_by(i), want = pages_of((uint32_t)len[i] + tokens_of(i) + P - 1);
    const int n_new = fits ? pc[i + 1] - pc[i] : 0, n_old = want - n_new;   // (the padding row has no new pages)
    int32_t* src = p.page_table + (int64_t)row[i] * p.pt_rs;
    int32_t* dst = p.out_page_table + (int64_t)i * p.out_rs;
    for (int c0 = lane; c0 < n_old; c0 += 32 * kCopies) {
      int v[kCopies];
#pragma unroll
      for (int k = 0; k < kCopies; ++k)
        if (c0 + 32 * k < n_old) v[k] = src[c0 + 32 * k];
#pragma unroll
      for (int k = 0; k < kCopies; ++k)
        if (c0 + 32 * k < n_old) dst[c0 + 32 * k] = v[k];
    }
    const int32_t* taken = p.free_pages + (count - pc[i + 1]);
    for (int j = lane; j < n_new; j += 32) {
      const int page = taken[j];
      dst[held + j] = page;
      src[held + j] = page;
    }
  }
  // slots and positions: a warp takes consecutive tokens, kTokens of a lane at a time so that their table entries are on the
  // way together; from one to the next a lane's entry is a few steps further, or it is searched for
  constexpr int kTokens = 4;
  const uint32_t n_live = fits ? (uint32_t)all_n : 0u, n_tokens = (uint32_t)p.n_tokens;
  const uint32_t n_warps = n_cta * 32u, per_warp = (n_tokens / n_warps / 32 + 1) * 32;
  const uint32_t begin = min((rank * 32u + wid) * per_warp, n_tokens), end = min(begin + per_warp, n_tokens);
  int e = 0;
  for (uint32_t t0 = begin; t0 < end; t0 += 32 * kTokens) {
    int pos[kTokens], blk[kTokens], page[kTokens];
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      const uint32_t tok = t0 + 32 * u + lane;
      pos[u] = 0;
      page[u] = -1;
      if (tok < end && tok < n_live) {
        const int t = (int)tok;   // cu[e] <= t
        for (int k = 0; k < 3 && cu[e + 1] <= t; ++k) ++e;
        if (cu[e + 1] <= t) {
          int hi = p.batch;   // cu[e] <= t < cu[hi]
          while (hi - e > 1) {
            const int mid = (e + hi) >> 1;
            if (cu[mid] <= t) e = mid; else hi = mid;
          }
        }
        pos[u] = len[e] + (t - cu[e]);
        blk[u] = pages_of(pos[u]);
        const int held = held_by(e);
        // a page that this step hands out comes from the free list: another CTA may not have written its table entry yet
        page[u] = blk[u] >= held && pc[e + 1] > pc[e] ? p.free_pages[count - pc[e + 1] + (blk[u] - held)]
                                                       : p.page_table[(int64_t)row[e] * p.pt_rs + blk[u]];
        if (page[u] < 0 || page[u] >= p.n_pages) {
          report(KB200_STATUS_BAD_PAGE, page[u], KID_RAGGED);
          page[u] = -1;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      const uint32_t tok = t0 + 32 * u + lane;
      if (tok < end) {
        p.out_slots[tok] = page[u] < 0 ? -1 : (int64_t)page[u] * P + (pos[u] - blk[u] * P);
        p.out_positions[tok] = pos[u];
      }
    }
  }
  cluster_wait();   // every CTA has read its inputs: they may be overwritten
  if (rank == 0) {
    for (int i = tid; i <= p.batch; i += kRaggedThreads) {
      p.out_cu[i] = fits ? cu[i] : 0;
      if (i < p.batch) p.out_seqused[i] = len[i] < 0 ? 0 : len[i] + tokens_of(i);
    }
    if (tid == 0) {
      *p.out_free_count = fits ? count - (int)all_p : count;
      *p.out_taken = fits ? (int)all_p : -1;
      if (!fits) report(KB200_STATUS_NO_PAGES, (int)min(all_p, 0x7fffffffll), KID_RAGGED);
    }
  }
}

// The largest cluster of this kernel that the device can hold, asked once per device.
inline int ragged_max_cluster(int device) {
  static std::once_flag flags[64];
  static int most[64];
  const int i = device & 63;
  std::call_once(flags[i], [&] {
    most[i] = 8;
    if (cudaFuncSetAttribute(ragged_step_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(kRaggedMaxCluster);
      cfg.blockDim = dim3(kRaggedThreads);
      cfg.dynamicSmemBytes = 4 * (kRaggedMaxBatch + 1) * sizeof(int);
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = kRaggedMaxCluster;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, ragged_step_kernel, &cfg) == cudaSuccess && n > 0) most[i] = kRaggedMaxCluster;
    }
    (void)cudaGetLastError();   // (a device that refuses keeps the portable size)
  });
  return most[i];
}

inline int launch_ragged_step(const RaggedParams& p, int device, cudaStream_t stream) {
  KB200_REQUIRE(p.batch >= 0 && p.n_tokens >= 0, "batch and n_tokens must be non-negative");
  if (p.batch > kRaggedMaxBatch)
    return fail(KB200_ERR_UNSUPPORTED, "a step of %d requests is not supported (at most %d)", p.batch, kRaggedMaxBatch);
  KB200_REQUIRE(p.page_size > 0 && p.n_pages > 0, "page_size and n_pages must be positive");
  KB200_REQUIRE(p.n_tokens <= 0x7fffffff, "n_tokens out of range");
  KB200_REQUIRE(p.page_table && p.free_pages && p.free_count && p.out_cu && p.out_free_count && p.out_taken &&
                    (p.n_tokens == 0 || (p.out_slots && p.out_positions)) &&
                    (p.batch == 0 || (p.batch_idx && p.lengths && p.new_tokens && p.out_page_table && p.out_seqused)),
                "null pointer argument");
  KB200_REQUIRE(p.pt_cols > 0 && p.out_cols > 0 && p.pt_cols <= 0x7fffffff / p.page_size, "bad page-table width");
  const int smem = 4 * (p.batch + 1) * (int)sizeof(int);
  static SmemAttrOnce once;
  if (int rc = once.ensure(ragged_step_kernel, 4 * (kRaggedMaxBatch + 1) * (int)sizeof(int), device)) return rc;
  // a CTA per 32 requests or 4096 tokens, in one cluster.  1000 requests with 128k tokens: 16.5 us with 8 CTAs, 11.0 with 16
  int64_t ctas = (p.batch + 31) / 32;
  if ((p.n_tokens + 4095) / 4096 > ctas) ctas = (p.n_tokens + 4095) / 4096;
  if (ctas < 1) ctas = 1;
  if (ctas > 8) ctas = ragged_max_cluster(device);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kRaggedThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  KB200_CUDA_OK(cudaLaunchKernelEx(&cfg, ragged_step_kernel, p));
  return KB200_OK;
}

// ---------------------------------------------------------------------------
// The pages of finished requests go back to the free list, last page of a row first, row after row (PageTable.erase).
// The first keep[i] pages of a row belong to somebody else (a cached prefix) and stay out.  One CTA.
// ---------------------------------------------------------------------------
struct ReleaseParams {
  int32_t* page_table;
  const void* batch_idx;
  const int32_t* lengths;
  const int32_t* keep;       // or nullptr
  int32_t* free_pages;
  int32_t* free_count;
  int64_t pt_rs, pt_rows, pt_cols, free_cap, n_pages;
  int32_t batch, page_size, batch_idx_is_i64;
};

__global__ void __launch_bounds__(kRaggedThreads, 1) release_rows_kernel(const ReleaseParams p) {
  extern __shared__ int ragged_smem[];
  __shared__ long long warp_p[32], carry;
  int* first = ragged_smem;          // free-list place of the row's last page, relative to the count
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int count = *p.free_count;
  if (tid == 0) carry = 0;
  __syncthreads();
  auto span = [&](int i, int64_t& r, int& lo, int& hi) {   // the row's private pages [lo, hi)
    r = p.batch_idx_is_i64 ? static_cast<const int64_t*>(p.batch_idx)[i] : static_cast<const int32_t*>(p.batch_idx)[i];
    const long long L = p.lengths[i], k = p.keep ? p.keep[i] : 0, held = (L + p.page_size - 1) / p.page_size;
    const bool ok = r >= 0 && r < p.pt_rows && L >= 0 && held <= p.pt_cols && k >= 0;
    if (!ok) { lo = hi = -1; return; }
    lo = (int)min(k, held);
    hi = r == 0 ? lo : (int)held;
  };
  for (int base = 0; base < p.batch; base += kRaggedThreads) {
    const int i = base + tid;
    long long np = 0;
    if (i < p.batch) {
      int64_t r;
      int lo, hi;
      span(i, r, lo, hi);
      if (lo < 0) report(KB200_STATUS_BAD_ROW, i, KID_RAGGED);
      np = hi - lo;
    }
    long long sp = np;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, sp, d);
      if (lane >= d) sp += up;
    }
    if (lane == 31) warp_p[wid] = sp;
    __syncthreads();
    long long off = carry;
    for (int w = 0; w < wid; ++w) off += warp_p[w];
    if (i < p.batch) first[i] = (int)min(off + sp - np, 0x7fffffffll);
    __syncthreads();
    if (tid == kRaggedThreads - 1) carry = off + sp;
    __syncthreads();
  }
  const bool fits = count >= 0 && count + carry <= p.free_cap;
  if (!fits) {   // more pages than the list can hold: rows released twice; nothing is changed
    if (tid == 0) report(KB200_STATUS_NO_PAGES, count, KID_RAGGED);
    return;
  }
  for (int i = wid; i < p.batch; i += kRaggedThreads / 32) {
    int64_t r;
    int lo, hi;
    span(i, r, lo, hi);
    for (int c = lo + lane; c < hi; c += 32) {
      int32_t* at = p.page_table + r * p.pt_rs + c;
      p.free_pages[(int64_t)count + first[i] + (hi - 1 - c)] = *at;
      *at = -1;
    }
  }
  __syncthreads();
  if (tid == 0) *p.free_count = count + (int)carry;
}

inline int launch_release_rows(const ReleaseParams& p, int device, cudaStream_t stream) {
  KB200_REQUIRE(p.batch >= 0, "batch must be non-negative");
  if (p.batch == 0) return KB200_OK;
  if (p.batch > kRaggedMaxBatch)
    return fail(KB200_ERR_UNSUPPORTED, "a release of %d requests is not supported (at most %d)", p.batch, kRaggedMaxBatch);
  KB200_REQUIRE(p.page_size > 0, "page_size must be positive");
  KB200_REQUIRE(p.page_table && p.free_pages && p.free_count && p.batch_idx && p.lengths, "null pointer argument");
  static SmemAttrOnce once;
  if (int rc = once.ensure(release_rows_kernel, (kRaggedMaxBatch + 1) * (int)sizeof(int), device)) return rc;
  KB200_CUDA_OK(launch_kernel(release_rows_kernel, dim3(1), dim3(kRaggedThreads), (size_t)(p.batch + 1) * sizeof(int), stream, p));
  return KB200_OK;
}

}  // namespace kb200
