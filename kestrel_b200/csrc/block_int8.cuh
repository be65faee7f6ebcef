// Append to a cache held in 8 bits with one scale per block, a block being one page of one KV head.
//
// Arithmetic.  With a = max |x| over the block's rows the scale is the power of two s, 64 s <= a < 128 s (0 for a block
// of zeros, never below 2^-126), the code floor(x / s) in [-128, 127], and a code stands for (code + 1/2) s, at most s / 2
// away from x.  A later row with a larger maximum raises s by 2^k; the codes already there become code >> k, and
// because floor(floor(x / s) / 2^k) = floor(x / (s 2^k)) they are the codes that x would have got at once: the bytes of
// a block do not depend on how its tokens were split over calls, and no rounding is added to a rounding.  Rounding to the nearest
// code would lose both.  Everything is exact in fp32 (scaling by a power of two), one fma rounded down per element.
//
// Work.  HBM-bound: T * H * D * 2 * (in + 1) bytes.  The tokens of one block form a *run* of the slot mapping (the page stays
// the same); a run's first token decides who handles it, so a block has one owner per call and nothing is atomic.
//   append_block_int8_kernel        few tokens (a decode step, a short chunk): a CTA looks after `window` tokens of one head of K or V,
//                                   runs of up to 16 tokens that start there go to one warp each, longer ones to all of its warps
//                                   together; rows are asked for together with the block's old scale and stay in registers
//                                   between the maximum and the codes
//   append_block_int8_warps_kernel  many tokens: every warp has a window of its own
// Measured, 8 heads of 128, bf16 rows: 256 single tokens 6.4 us (latency: slots, then rows and scale, then codes); eight
// chunks of 1500 to 2600 tokens 34 us = 3.1 TB/s with a warp per window, 58 us with a CTA per window.  What is left: the
// second pass comes out of L2, and a run's passes wait for each other.
#pragma once

#include <type_traits>

#include "cache_ops.cuh"

namespace kb200 {

struct AppendI8Params {
  const char* rows[2];          // K, V
  char* cache[2];
  float* scale[2];
  const int64_t* slots;
  int64_t row_stride_b[2];      // bytes between tokens
  int64_t page_stride, token_stride, head_stride;   // elements (= bytes) of the cache view
  int64_t scale_page_stride;    // elements
  int64_t num_tokens, n_slots_total;
  int32_t page_size, head_dim, window;
};

constexpr int kI8Threads = 256;
constexpr int kI8MaxWindow = 64;
constexpr int kI8Ahead = 128;    // tokens behind the window whose pages are at hand: a run may reach past its window
constexpr int kI8WarpRun = 16;   // longest run that one warp takes
constexpr int kI8WarpsFrom = 8;  // windows of 64 tokens per SM from which every warp has its own
constexpr int kI8Chunks = 4;     // 16-element pieces of rows that a thread keeps

// s with 64 s <= a < 128 s; 0 for 0.  The exponent is clamped so that s and 1 / s are normal numbers.
__device__ __forceinline__ float block_scale_of(float a) {
  if (a == 0.f) return 0.f;
  const uint32_t e = __float_as_uint(a) & 0x7f800000u;
  return __uint_as_float(e > (7u << 23) ? e - (6u << 23) : (1u << 23));
}
__device__ __forceinline__ float pow2_reciprocal(float s) { return s == 0.f ? 0.f : __uint_as_float((254u << 23) - __float_as_uint(s)); }

// floor(x * inv) in the low byte: one fma rounded down onto the integers (ulp 1 at 1.5 * 2^23)
__device__ __forceinline__ uint32_t floor_code(float x, float inv) { return __float_as_uint(__fmaf_rd(x, inv, 12582912.f)); }
// the same for rows that hold NaN or infinities: NaN -> 0, infinities saturate
__device__ __forceinline__ uint32_t floor_code_any(float x, float inv) {
  if (x != x) return 0u;
  if (fabsf(x) == INFINITY) return x > 0.f ? 127u : 0x80u;
  return floor_code(x, inv);
}

// 16 consecutive elements as they lie in memory; VEC: 16-byte loads
template <typename In> struct Raw16 { uint4 v[sizeof(In)]; };   // (16 elements are sizeof(In) vectors of 16 bytes)
template <typename In, bool VEC>
__device__ __forceinline__ void load16(const In* src, Raw16<In>& raw) {
  if constexpr (VEC) {
#pragma unroll
    for (int v = 0; v < (int)sizeof(In); ++v) raw.v[v] = *(reinterpret_cast<const uint4*>(src) + v);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(raw.v);
#pragma unroll
    for (int i = 0; i < 4 * (int)sizeof(In); ++i) {
      if constexpr (sizeof(In) == 4) w[i] = __float_as_uint(src[i]);
      else {
        const uint16_t* s = reinterpret_cast<const uint16_t*>(src);
        w[i] = (uint32_t)s[2 * i] | ((uint32_t)s[2 * i + 1] << 16);
      }
    }
  }
}
// Largest magnitude so far as a bit pattern, which orders like the number; 16-bit types: two of them side by side.
// NaN and infinities lie above every number.
template <typename In>
__device__ __forceinline__ uint32_t max_bits(uint32_t m, const Raw16<In>& raw) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(raw.v);
#pragma unroll
  for (int i = 0; i < 4 * (int)sizeof(In); ++i) {
    if constexpr (sizeof(In) == 4) m = max(m, w[i] & 0x7fffffffu);
    else m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  }
  return m;
}
template <typename In>
__device__ __forceinline__ float bits_to_abs(uint32_t m) {   // NaN and infinities come out as such
  if constexpr (sizeof(In) == 4) return __uint_as_float(m);
  else {
    const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
    return to_float(*reinterpret_cast<const In*>(&h));
  }
}

// Arithmetic shift right of 16 codes
__device__ __forceinline__ uint4 shift_codes(uint4 v, int k) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t r = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) r |= ((uint32_t)((int)(int8_t)(w[i] >> (8 * b)) >> k) & 0xffu) << (8 * b);
    w[i] = r;
  }
  return v;
}

template <typename In>
__device__ __forceinline__ uint4 code16(const Raw16<In>& x, float inv, bool bad) {
  const In* e = reinterpret_cast<const In*>(x.v);
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = to_float(e[4 * q + k]);
      b[k] = bad ? floor_code_any(f, inv) : floor_code(f, inv);
    }
    w[q] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename In, bool VEC>
__global__ void __launch_bounds__(kI8Threads) append_block_int8_kernel(const AppendI8Params p) {
  constexpr int NW = kI8Threads / 32, J = kI8Chunks;
  constexpr int kSpan = kI8MaxWindow + kI8Ahead;
  __shared__ int page_of[kSpan + 1];         // [0]: the token before the window; -1: no page
  __shared__ int off_of[kSpan + 1];
  __shared__ int starts[kI8MaxWindow];       // window index of every run that starts here
  __shared__ int long_start[kI8MaxWindow], long_len[kI8MaxWindow];   // the long ones among them
  __shared__ int n_starts, n_long;
  __shared__ float red[NW];
  __shared__ int red_flags[NW];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int h = blockIdx.y, kv = blockIdx.z;
  const int64_t w0 = (int64_t)blockIdx.x * p.window;
  const int P = p.page_size, C = p.head_dim >> 4;   // 16-element chunks per row
  const int shift = (P & (P - 1)) == 0 ? 31 - __clz(P) : -1;
  auto split = [&](int64_t t, int& page, int& off) {   // page -1: a token without a slot
    page = -1;
    off = 0;
    if (t < 0 || t >= p.num_tokens) return;
    const int64_t s = p.slots[t];
    if (s < 0 || s >= p.n_slots_total) return;
    page = (int)(shift >= 0 ? s >> shift : s / P);
    off = (int)(s - (int64_t)page * P);
  };
  const int n_span = p.window + kI8Ahead;
  for (int i = tid; i <= n_span; i += kI8Threads) {
    const int64_t t = w0 + i - 1;
    split(t, page_of[i], off_of[i]);
    if (h == 0 && kv == 0 && i >= 1 && i <= p.window && t < p.num_tokens && p.slots[t] >= p.n_slots_total)
      report(KB200_STATUS_BAD_SLOT, (int)p.slots[t], KID_APPEND);
  }
  __syncthreads();
  if (wid == 0) {
    int n = 0;
    for (int i0 = 0; i0 < p.window; i0 += 32) {
      const int i = i0 + lane;
      const bool start = i < p.window && page_of[i + 1] >= 0 && page_of[i + 1] != page_of[i];
      const uint32_t m = __ballot_sync(0xffffffffu, start);
      if (start) starts[n + __popc(m & ((1u << lane) - 1u))] = i;
      n += __popc(m);
    }
    if (lane == 0) { n_starts = n; n_long = 0; }
  }
  __syncthreads();
  if (n_starts == 0) return;

  const char* rows = p.rows[kv] + (int64_t)h * p.head_dim * (int64_t)sizeof(In);
  const int64_t rs = p.row_stride_b[kv];
  char* cache = p.cache[kv] + (int64_t)h * p.head_stride;
  // offset in the block of the run's token r (i0: its start in the window)
  auto off_at = [&](int i0, int r) {
    if (i0 + r < n_span) return off_of[i0 + r + 1];
    int page, off;
    split(w0 + i0 + r, page, off);
    return off;
  };
  // one run, shared by `nt` threads (this one is number `me`); `agree` turns a thread's (maximum, flags) into the team's
  auto do_run = [&](int i0, int len, int me, int nt, auto agree, auto sync) {
    const int64_t t0 = w0 + i0, page = page_of[i0 + 1];
    const int n = len * C;   // chunks
    float* sp = p.scale[kv] + page * p.scale_page_stride + h;
    const float s_was = *sp;
    auto at = [&](int i) { const int r = i / C; return reinterpret_cast<const In*>(rows + (t0 + r) * rs) + 16 * (i - r * C); };
    Raw16<In> raw[J];
    uint32_t m = 0;
    int flags = 0;   // 1: not finite, 2: the block starts anew, 4: the slots do not ascend (one may come twice)
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (me + j * nt < n) load16<In, VEC>(at(me + j * nt), raw[j]);
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (me + j * nt < n) m = max_bits<In>(m, raw[j]);
    for (int i = me + J * nt; i < n; i += nt) {
      Raw16<In> x;
      load16<In, VEC>(at(i), x);
      m = max_bits<In>(m, x);
    }
    for (int r = me; r < len; r += nt) {
      const int o = off_at(i0, r);
      if (o == 0) flags |= 2;
      if (r + 1 < len && off_at(i0, r + 1) <= o) flags |= 4;
    }
    float a = bits_to_abs<In>(m);
    if (!(a < INFINITY)) {   // NaN or infinities: the largest number without them
      flags |= 1;
      a = 0.f;
      for (int i = me; i < n; i += nt) {
        const In* x = at(i);
        for (int e = 0; e < 16; ++e) {
          const float f = fabsf(to_float(x[e]));
          if (f < INFINITY) a = fmaxf(a, f);
        }
      }
    }
    agree(a, flags);
    const bool bad = flags & 1, dup = flags & 4;
    const float s_old = (flags & 2) ? 0.f : s_was;
    const float s_new = fmaxf(s_old, block_scale_of(a));
    const float inv = pow2_reciprocal(s_new);
    char* blk = cache + page * p.page_stride;
    if (s_old > 0.f && s_new > s_old) {   // the scale grew: what the block holds is coded again
      const int k = min(31, (int)((__float_as_uint(s_new) - __float_as_uint(s_old)) >> 23));
      for (int i = me; i < P * C; i += nt) {
        const int r = i / C, c = i - r * C;
        uint4* q = reinterpret_cast<uint4*>(blk + (int64_t)r * p.token_stride + 16 * c);
        *q = shift_codes(*q, k);
      }
    }
    sync();   // the old scale has been read and the old codes are in place before anything new is written
    auto code = [&](int i, const Raw16<In>& x) {
      const int r = i / C, c = i - r * C;
      const int o = off_at(i0, r);
      if (dup) {   // of two rows with the same slot the later one counts
        bool again = false;
        for (int q = r + 1; q < len; ++q) again |= off_at(i0, q) == o;
        if (again) return;
      }
      *reinterpret_cast<uint4*>(blk + (int64_t)o * p.token_stride + 16 * c) = code16<In>(x, inv, bad);
    };
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (me + j * nt < n) code(me + j * nt, raw[j]);
    for (int i = me + J * nt; i < n; i += nt) {
      Raw16<In> x;
      load16<In, VEC>(at(i), x);
      code(i, x);
    }
    if (me == 0) {
      if (s_new != s_was) *sp = s_new;
      if (bad) report(KB200_STATUS_NOT_FINITE, (int)t0, KID_APPEND_I8);
    }
  };

  // short runs: a warp each
  for (int i = wid; i < n_starts; i += NW) {
    const int i0 = starts[i], page = page_of[i0 + 1];
    int len = 0;
    for (;;) {   // the run ends at the first token of another page (past the pages at hand: looked up)
      const int j = i0 + len + lane;
      int pg, off;
      if (j < n_span) pg = page_of[j + 1];
      else split(w0 + j, pg, off);
      const uint32_t other = __ballot_sync(0xffffffffu, pg != page);
      if (other) { len += __ffs(other) - 1; break; }
      len += 32;
    }
    if (len > kI8WarpRun) {   // all warps, below
      if (lane == 0) {
        const int at = atomicAdd(&n_long, 1);   // (their order does not matter: different blocks)
        long_start[at] = i0;
        long_len[at] = len;
      }
      continue;
    }
    do_run(i0, len, lane, 32,
           [&](float& a, int& flags) {
             a = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a)));   // (non-negative: ordered as integers)
             flags = (int)__reduce_or_sync(0xffffffffu, (uint32_t)flags);
           },
           [] { __syncwarp(); });
  }
  __syncthreads();
  const int nl = n_long;
  for (int i = 0; i < nl; ++i)
    do_run(long_start[i], long_len[i], tid, kI8Threads,
           [&](float& a, int& flags) {
             const float wa = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a)));
             const int wf = (int)__reduce_or_sync(0xffffffffu, (uint32_t)flags);
             __syncthreads();   // (the previous run's values have been read)
             if (lane == 0) { red[wid] = wa; red_flags[wid] = wf; }
             __syncthreads();
             a = 0.f;
             flags = 0;
#pragma unroll
             for (int k = 0; k < NW; ++k) { a = fmaxf(a, red[k]); flags |= red_flags[k]; }
           },
           [] { __syncthreads(); });
}

// Many tokens (prompt chunks): every warp has a window of its own and takes its runs alone, whatever their length, in two passes
// over the rows (the second one out of L1 and L2).  No barriers, and as many runs on an SM as it holds warps.  A lane's
// piece is one 16-byte vector of a row, so that a warp reads whole lines; rows have 1, 2, 4, .. 32 of them, which keeps a lane
// in one column and its addresses a constant step apart.
template <typename In> struct Vec16 { static constexpr int N = 16 / (int)sizeof(In); };
template <typename In, bool VEC>
__device__ __forceinline__ uint4 load_vec(const In* src) {
  if constexpr (VEC) return *reinterpret_cast<const uint4*>(src);
  else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(In) == 4) w[i] = __float_as_uint(src[i]);
      else {
        const uint16_t* s = reinterpret_cast<const uint16_t*>(src);
        w[i] = (uint32_t)s[2 * i] | ((uint32_t)s[2 * i + 1] << 16);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <typename In>
__device__ __forceinline__ uint32_t max_bits_vec(uint32_t m, const uint4& v) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(In) == 4) m = max(m, w[i] & 0x7fffffffu);
    else m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  }
  return m;
}
template <typename In, bool ANY>
__device__ __forceinline__ void store_codes(char* dst, const uint4& v, float inv) {
  const In* e = reinterpret_cast<const In*>(&v);
  uint32_t w[Vec16<In>::N / 4];
#pragma unroll
  for (int q = 0; q < Vec16<In>::N / 4; ++q) {
    uint32_t b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = ANY ? floor_code_any(to_float(e[4 * q + k]), inv) : floor_code(to_float(e[4 * q + k]), inv);
    w[q] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  }
  if constexpr (Vec16<In>::N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(dst) = w[0];
}

template <typename In, bool VEC>
__global__ void __launch_bounds__(kI8Threads) append_block_int8_warps_kernel(const AppendI8Params p) {
  constexpr int NW = kI8Threads / 32, U = 4, N = Vec16<In>::N;   // U vectors of a lane in flight
  constexpr int kSpan = 2 * kI8MaxWindow;
  __shared__ int pages[NW][kSpan + 1], offs[NW][kSpan + 1];   // [0]: the token before the window; page -1: no page
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int h = blockIdx.y, kv = blockIdx.z;
  const int64_t w0 = ((int64_t)blockIdx.x * NW + wid) * kI8MaxWindow;
  if (w0 >= p.num_tokens) return;
  const int P = p.page_size, C = p.head_dim / N;   // vectors per row
  const int shift = (P & (P - 1)) == 0 ? 31 - __clz(P) : -1;
  int* page_of = pages[wid];
  int* off_of = offs[wid];
  auto split = [&](int64_t t, int& page, int& off) {
    page = -1;
    off = 0;
    if (t < 0 || t >= p.num_tokens) return;
    const int64_t s = p.slots[t];
    if (s < 0) return;
    if (s >= p.n_slots_total) {
      if (h == 0 && kv == 0 && t >= w0 && t < w0 + kI8MaxWindow) report(KB200_STATUS_BAD_SLOT, (int)s, KID_APPEND);
      return;
    }
    page = (int)(shift >= 0 ? s >> shift : s / P);
    off = (int)(s - (int64_t)page * P);
  };
  for (int i = lane; i <= kSpan; i += 32) split(w0 + i - 1, page_of[i], off_of[i]);
  __syncwarp();
  const char* rows = p.rows[kv] + (int64_t)h * p.head_dim * (int64_t)sizeof(In);
  const int64_t rs = p.row_stride_b[kv];
  char* cache = p.cache[kv] + (int64_t)h * p.head_stride;
  const int row_0 = lane / C, col = lane - row_0 * C, drow = 32 / C;   // a lane's rows: row_0, row_0 + drow, ..

  uint32_t starts[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = 32 * q + lane;
    starts[q] = __ballot_sync(0xffffffffu, page_of[i + 1] >= 0 && page_of[i + 1] != page_of[i]);
  }
  for (;;) {
    const int i0 = starts[0] ? __ffs(starts[0]) - 1 : starts[1] ? 31 + __ffs(starts[1]) : -1;
    if (i0 < 0) break;
    if (i0 < 32) starts[0] &= starts[0] - 1;
    else starts[1] &= starts[1] - 1;
    const int page = page_of[i0 + 1];
    int len = 0;
    for (;;) {   // the run ends at the first token of another page
      const int j = i0 + len + lane;
      int pg, off;
      if (j < kSpan) pg = page_of[j + 1];
      else split(w0 + j, pg, off);
      const uint32_t other = __ballot_sync(0xffffffffu, pg != page);
      if (other) { len += __ffs(other) - 1; break; }
      len += 32;
    }
    auto off_at = [&](int r) {
      if (i0 + r < kSpan) return off_of[i0 + r + 1];
      int pg, off;
      split(w0 + i0 + r, pg, off);
      return off;
    };
    float* sp = p.scale[kv] + (int64_t)page * p.scale_page_stride + h;
    const float s_was = *sp;
    const char* mine = rows + (w0 + i0 + row_0) * rs + 16 * col;
    const int64_t step = drow * rs;
    uint32_t m = 0;
    {
      const char* at = mine;
      int r = row_0;
      for (; r + (U - 1) * drow < len; r += U * drow, at += U * step) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load_vec<In, VEC>(reinterpret_cast<const In*>(at + u * step));
#pragma unroll
        for (int u = 0; u < U; ++u) m = max_bits_vec<In>(m, v[u]);
      }
      for (; r < len; r += drow, at += step) m = max_bits_vec<In>(m, load_vec<In, VEC>(reinterpret_cast<const In*>(at)));
    }
    int flags = 0;   // 1: not finite, 2: the block starts anew, 4: the slots do not ascend (one may come twice)
    for (int r = lane; r < len; r += 32) {
      const int o = off_at(r);
      if (o == 0) flags |= 2;
      if (r + 1 < len && off_at(r + 1) <= o) flags |= 4;
    }
    float a = bits_to_abs<In>(m);
    if (!(a < INFINITY)) {   // NaN or infinities: the largest number without them
      flags |= 1;
      a = 0.f;
      for (int r = row_0; r < len; r += drow) {
        const In* e = reinterpret_cast<const In*>(mine + (r - row_0) * rs);
        for (int k = 0; k < N; ++k) {
          const float f = fabsf(to_float(e[k]));
          if (f < INFINITY) a = fmaxf(a, f);
        }
      }
    }
    a = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a)));   // (non-negative: ordered as integers)
    flags = (int)__reduce_or_sync(0xffffffffu, (uint32_t)flags);
    const float s_old = (flags & 2) ? 0.f : s_was;
    const float s_new = fmaxf(s_old, block_scale_of(a));
    const float inv = pow2_reciprocal(s_new);
    char* blk = cache + (int64_t)page * p.page_stride;
    if (s_old > 0.f && s_new > s_old) {   // the scale grew: what the block holds is coded again
      const int k = min(31, (int)((__float_as_uint(s_new) - __float_as_uint(s_old)) >> 23));
      const int C16 = p.head_dim >> 4;
      for (int i = lane; i < P * C16; i += 32) {
        const int r = i / C16, c = i - r * C16;
        uint4* q = reinterpret_cast<uint4*>(blk + (int64_t)r * p.token_stride + 16 * c);
        *q = shift_codes(*q, k);
      }
    }
    __syncwarp();   // the old scale has been read and the old codes are in place before anything new is written
    char* dst = blk + col * N;
    if ((flags & 5) == 0) {
      const char* at = mine;
      int r = row_0;
      for (; r + (U - 1) * drow < len; r += U * drow, at += U * step) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load_vec<In, VEC>(reinterpret_cast<const In*>(at + u * step));
#pragma unroll
        for (int u = 0; u < U; ++u) store_codes<In, false>(dst + (int64_t)off_at(r + u * drow) * p.token_stride, v[u], inv);
      }
      for (; r < len; r += drow, at += step)
        store_codes<In, false>(dst + (int64_t)off_at(r) * p.token_stride, load_vec<In, VEC>(reinterpret_cast<const In*>(at)), inv);
    } else {
      for (int r = row_0; r < len; r += drow) {
        const int o = off_at(r);
        bool again = false;   // of two rows with the same slot the later one counts
        if (flags & 4)
          for (int q = r + 1; q < len; ++q) again |= off_at(q) == o;
        if (!again)
          store_codes<In, true>(dst + (int64_t)o * p.token_stride, load_vec<In, VEC>(reinterpret_cast<const In*>(mine + (r - row_0) * rs)), inv);
      }
    }
    if (lane == 0) {
      if (s_new != s_was) *sp = s_new;
      if (flags & 1) report(KB200_STATUS_NOT_FINITE, (int)(w0 + i0), KID_APPEND_I8);
    }
  }
}

template <typename In>
inline int launch_append_i8_typed(const AppendI8Params& p, bool vec, bool warps, dim3 grid, cudaStream_t stream) {
  if (warps) {
    if (vec) KB200_CUDA_OK(launch_kernel(append_block_int8_warps_kernel<In, true>, grid, dim3(kI8Threads), 0, stream, p));
    else KB200_CUDA_OK(launch_kernel(append_block_int8_warps_kernel<In, false>, grid, dim3(kI8Threads), 0, stream, p));
    return KB200_OK;
  }
  if (vec) KB200_CUDA_OK(launch_kernel(append_block_int8_kernel<In, true>, grid, dim3(kI8Threads), 0, stream, p));
  else KB200_CUDA_OK(launch_kernel(append_block_int8_kernel<In, false>, grid, dim3(kI8Threads), 0, stream, p));
  return KB200_OK;
}

inline int launch_append_block_int8(const void* key, const void* value, int64_t key_token_stride, int64_t value_token_stride,
                                    void* key_cache, void* value_cache, int64_t page_stride, int64_t token_stride,
                                    int64_t head_stride, float* key_scales, float* value_scales, int64_t scale_page_stride,
                                    const int64_t* slots, int64_t num_tokens, int64_t n_pages, int page_size, int n_heads,
                                    int head_dim, int in_dtype, cudaStream_t stream) {
  KB200_REQUIRE(num_tokens >= 0, "num_tokens must be non-negative");
  if (num_tokens == 0) return KB200_OK;
  KB200_REQUIRE(key && value && key_cache && value_cache && key_scales && value_scales && slots, "null pointer argument");
  KB200_REQUIRE(page_size > 0 && n_heads > 0 && n_pages > 0, "page_size, n_kv_heads and n_pages must be positive");
  KB200_REQUIRE(n_heads <= 65535, "too many KV heads");
  KB200_REQUIRE(n_pages <= 0x7fffffff, "too many pages");
  KB200_REQUIRE(num_tokens <= 0x7fffffff, "too many tokens");
  if (head_dim <= 0 || head_dim % 16 != 0)
    return fail(KB200_ERR_UNSUPPORTED, "head_dim %d is not supported by int8 pools (a multiple of 16)", head_dim);
  const int es = dtype_size(in_dtype);
  KB200_REQUIRE(in_dtype == KB200_DTYPE_F32 || in_dtype == KB200_DTYPE_F16 || in_dtype == KB200_DTYPE_BF16,
                "rows must be F32, F16 or BF16");
  KB200_REQUIRE(aligned16(key_cache) && aligned16(value_cache) && page_stride % 16 == 0 && token_stride % 16 == 0 &&
                    head_stride % 16 == 0,
                "int8 pools and their strides must be 16-byte aligned");
  AppendI8Params p;
  p.rows[0] = static_cast<const char*>(key);
  p.rows[1] = static_cast<const char*>(value);
  p.cache[0] = static_cast<char*>(key_cache);
  p.cache[1] = static_cast<char*>(value_cache);
  p.scale[0] = key_scales;
  p.scale[1] = value_scales;
  p.slots = slots;
  p.row_stride_b[0] = key_token_stride * es;
  p.row_stride_b[1] = value_token_stride * es;
  p.page_stride = page_stride; p.token_stride = token_stride; p.head_stride = head_stride;
  p.scale_page_stride = scale_page_stride;
  p.num_tokens = num_tokens;
  p.n_slots_total = n_pages * page_size;
  p.page_size = page_size;
  p.head_dim = head_dim;
  const bool vec = aligned16(key) && aligned16(value) && p.row_stride_b[0] % 16 == 0 && p.row_stride_b[1] % 16 == 0;
  // Windows of 64 tokens for every warp once that gives each SM its warps; below, windows of eight tokens for a CTA: eight warps
  // take a run each (a decode step), or one long run together.
  const int64_t windows = (num_tokens + kI8MaxWindow - 1) / kI8MaxWindow;
  const int row_vecs = head_dim * es / 16;
  const bool warps = windows * n_heads * 2 >= 148 * kI8WarpsFrom && row_vecs <= 32 && (row_vecs & (row_vecs - 1)) == 0;
  p.window = 8;
  const int64_t per_cta = warps ? kI8MaxWindow * (kI8Threads / 32) : p.window;
  const dim3 grid((unsigned)((num_tokens + per_cta - 1) / per_cta), (unsigned)n_heads, 2);
  if (in_dtype == KB200_DTYPE_F32) return launch_append_i8_typed<float>(p, vec, warps, grid, stream);
  if (in_dtype == KB200_DTYPE_F16) return launch_append_i8_typed<__half>(p, vec, warps, grid, stream);
  return launch_append_i8_typed<__nv_bfloat16>(p, vec, warps, grid, stream);
}

}  // namespace kb200
