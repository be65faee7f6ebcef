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
// A CTA looks after `window` tokens of one head of K or V: runs of up to 32 tokens that start there go to one warp each, longer
// ones to all of its warps together.  Two passes over a run's rows (maximum, then codes); the second one hits L1.
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
constexpr int kI8WarpRun = 32;   // longest run that one warp takes

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

// 16 consecutive elements as floats; VEC: 16-byte loads
template <typename In, bool VEC>
__device__ __forceinline__ void load16(const In* src, float (&x)[16]) {
  if constexpr (VEC) {
    uint4 raw[sizeof(In)];   // 16 elements = sizeof(In) vectors of 16 bytes
#pragma unroll
    for (int v = 0; v < (int)sizeof(In); ++v) raw[v] = *(reinterpret_cast<const uint4*>(src) + v);
    const In* e = reinterpret_cast<const In*>(raw);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = to_float(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = to_float(src[i]);
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

template <typename In, bool VEC>
__global__ void __launch_bounds__(kI8Threads) append_block_int8_kernel(const AppendI8Params p) {
  constexpr int NW = kI8Threads / 32;
  __shared__ int starts[kI8MaxWindow];       // window index of every run that starts here
  __shared__ int long_start[kI8MaxWindow];   // the long ones among them, and their lengths
  __shared__ int long_len[kI8MaxWindow];
  __shared__ int n_starts, n_long;
  __shared__ float red[NW];
  __shared__ int red_bad[NW], red_fresh[NW], red_dup[NW];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int h = blockIdx.y, kv = blockIdx.z;
  const int64_t w0 = (int64_t)blockIdx.x * p.window;
  const int P = p.page_size, C = p.head_dim >> 4;   // 16-element chunks per row
  auto page_of = [&](int64_t t) -> int64_t {        // page of token t, -1 where it has none
    const int64_t s = p.slots[t];
    return s < 0 || s >= p.n_slots_total ? -1 : s / P;
  };
  if (wid == 0) {
    int n = 0;
    for (int i0 = 0; i0 < p.window; i0 += 32) {
      const int64_t t = w0 + i0 + lane;
      bool start = false;
      if (i0 + lane < p.window && t < p.num_tokens) {
        const int64_t pg = page_of(t);
        start = pg >= 0 && (t == 0 || page_of(t - 1) != pg);
        if (pg < 0 && h == 0 && kv == 0 && p.slots[t] >= 0) report(KB200_STATUS_BAD_SLOT, (int)p.slots[t], KID_APPEND);
      }
      const uint32_t m = __ballot_sync(0xffffffffu, start);
      if (start) starts[n + __popc(m & ((1u << lane) - 1u))] = i0 + lane;
      n += __popc(m);
    }
    if (lane == 0) { n_starts = n; n_long = 0; }
  }
  __syncthreads();
  if (n_starts == 0) return;

  const char* rows = p.rows[kv] + (int64_t)h * p.head_dim * (int64_t)sizeof(In);
  const int64_t rs = p.row_stride_b[kv];
  char* cache = p.cache[kv] + (int64_t)h * p.head_stride;
  // one run, shared by `nt` threads (this one is number `me`); `agree` turns a thread's (maximum, non-finite, restart,
  // duplicate) into the team's
  auto do_run = [&](int64_t t0, int len, int me, int nt, auto agree, auto sync) {
    const int64_t slot0 = p.slots[t0], page = slot0 / P, base = page * P;
    float a = 0.f;
    int bad = 0, fresh = 0, dup = 0;
    for (int i = me; i < len * C; i += nt) {
      const int r = i / C, c = i - r * C;
      float x[16];
      load16<In, VEC>(reinterpret_cast<const In*>(rows + (t0 + r) * rs) + 16 * c, x);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float m = fabsf(x[e]);
        if (m < INFINITY) a = fmaxf(a, m);
        else bad = 1;
      }
      if (c == 0) {
        const int64_t s = p.slots[t0 + r];
        if (s == base) fresh = 1;                                    // the block's first token: it starts anew
        if (r + 1 < len && p.slots[t0 + r + 1] <= s) dup = 1;        // not ascending: a slot may come twice
      }
    }
    agree(a, bad, fresh, dup);
    float* sp = p.scale[kv] + page * p.scale_page_stride + h;
    const float s_old = fresh ? 0.f : *sp;
    const float s_new = fmaxf(s_old, block_scale_of(a));
    const float inv = pow2_reciprocal(s_new);
    char* blk = cache + page * p.page_stride;
    if (s_old > 0.f && s_new > s_old) {   // the scale grew: what the block holds is coded again
      const int k = min(31, (int)((__float_as_uint(s_new) - __float_as_uint(s_old)) >> 23));
      for (int i = me; i < P * C; i += nt) {
        const int r = i / C, c = i - r * C;
        uint4* at = reinterpret_cast<uint4*>(blk + (int64_t)r * p.token_stride + 16 * c);
        *at = shift_codes(*at, k);
      }
    }
    sync();   // the old scale has been read and the old codes are in place before anything new is written
    for (int i = me; i < len * C; i += nt) {
      const int r = i / C, c = i - r * C;
      const int64_t s = p.slots[t0 + r];
      if (dup) {   // of two rows with the same slot the later one counts
        bool again = false;
        for (int j = r + 1; j < len; ++j) again |= p.slots[t0 + j] == s;
        if (again) continue;
      }
      float x[16];
      load16<In, VEC>(reinterpret_cast<const In*>(rows + (t0 + r) * rs) + 16 * c, x);
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t b0, b1, b2, b3;
        if (bad) {
          b0 = floor_code_any(x[4 * q], inv); b1 = floor_code_any(x[4 * q + 1], inv);
          b2 = floor_code_any(x[4 * q + 2], inv); b3 = floor_code_any(x[4 * q + 3], inv);
        } else {
          b0 = floor_code(x[4 * q], inv); b1 = floor_code(x[4 * q + 1], inv);
          b2 = floor_code(x[4 * q + 2], inv); b3 = floor_code(x[4 * q + 3], inv);
        }
        w[q] = __byte_perm(__byte_perm(b0, b1, 0x0040), __byte_perm(b2, b3, 0x0040), 0x5410);
      }
      *reinterpret_cast<uint4*>(blk + (s - base) * p.token_stride + 16 * c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (me == 0) {
      *sp = s_new;
      if (bad) report(KB200_STATUS_NOT_FINITE, (int)t0, KID_APPEND_I8);
    }
  };

  // short runs: a warp each
  for (int i = wid; i < n_starts; i += NW) {
    const int64_t t0 = w0 + starts[i];
    const int64_t page = page_of(t0);
    const int64_t t = t0 + lane;
    const uint32_t other = __ballot_sync(0xffffffffu, t >= p.num_tokens || page_of(t) != page);
    int len = other ? __ffs(other) - 1 : 32;
    if (!other && t0 + 32 < p.num_tokens && page_of(t0 + 32) == page) {   // longer than a warp takes: all warps, below
      int64_t end = t0 + 32;
      for (;;) {
        const int64_t u = end + lane;
        const uint32_t o2 = __ballot_sync(0xffffffffu, u >= p.num_tokens || page_of(u) != page);
        if (o2) { end += __ffs(o2) - 1; break; }
        end += 32;
      }
      if (lane == 0) {
        const int at = atomicAdd(&n_long, 1);   // (their order does not matter: different blocks)
        long_start[at] = starts[i];
        long_len[at] = (int)(end - t0);
      }
      continue;
    }
    do_run(t0, len, lane, 32,
           [&](float& a, int& bad, int& fresh, int& dup) {
             a = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a)));   // (non-negative: ordered as integers)
             const uint32_t f = __reduce_or_sync(0xffffffffu, (uint32_t)(bad | (fresh << 1) | (dup << 2)));
             bad = f & 1; fresh = (f >> 1) & 1; dup = (f >> 2) & 1;
           },
           [] { __syncwarp(); });
  }
  __syncthreads();
  const int nl = n_long;
  for (int i = 0; i < nl; ++i)
    do_run(w0 + long_start[i], long_len[i], tid, kI8Threads,
           [&](float& a, int& bad, int& fresh, int& dup) {
             const float wa = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a)));
             const uint32_t f = __reduce_or_sync(0xffffffffu, (uint32_t)(bad | (fresh << 1) | (dup << 2)));
             __syncthreads();   // (the previous run's values have been read)
             if (lane == 0) { red[wid] = wa; red_bad[wid] = f & 1; red_fresh[wid] = (f >> 1) & 1; red_dup[wid] = (f >> 2) & 1; }
             __syncthreads();
             a = 0.f; bad = fresh = dup = 0;
#pragma unroll
             for (int k = 0; k < NW; ++k) { a = fmaxf(a, red[k]); bad |= red_bad[k]; fresh |= red_fresh[k]; dup |= red_dup[k]; }
           },
           [] { __syncthreads(); });
}

template <typename In>
inline int launch_append_i8_typed(const AppendI8Params& p, bool vec, dim3 grid, cudaStream_t stream) {
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
  // Eight warps take a run each in a window of eight single-token runs (a decode step).  Larger windows once that gives
  // every SM its eight CTAs anyway: fewer CTAs that find no run of their own.
  int window = 8;
  while (window < kI8MaxWindow && num_tokens * n_heads * 2 / (2 * window) >= 148 * 8) window *= 2;
  p.window = window;
  const bool vec = aligned16(key) && aligned16(value) && p.row_stride_b[0] % 16 == 0 && p.row_stride_b[1] % 16 == 0;
  const dim3 grid((unsigned)((num_tokens + window - 1) / window), (unsigned)n_heads, 2);
  if (in_dtype == KB200_DTYPE_F32) return launch_append_i8_typed<float>(p, vec, grid, stream);
  if (in_dtype == KB200_DTYPE_F16) return launch_append_i8_typed<__half>(p, vec, grid, stream);
  return launch_append_i8_typed<__nv_bfloat16>(p, vec, grid, stream);
}

}  // namespace kb200
