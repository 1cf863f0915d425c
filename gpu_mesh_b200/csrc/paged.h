// The paged KV cache (internal to the library): a pool of pages that the
// sequences of a ragged batch share, in the activation type or in e4m3.
#pragma once

#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace mg {

constexpr int kE4M3 = 2;             // cache type, next to kF32 / kBF16
constexpr int kErrPaged = 4;         // a page id, length or token range outside the pool or the batch
constexpr int kPagedMaxBatch = 2048; // sequences of one call (the kernels keep a prefix over them in shared memory)
constexpr int kPagedMinExp = -100;   // least exponent of a page's scale
constexpr int kPagedMaxExp = 100;    // largest: sums weighed by 2^-e do not overflow
constexpr int kPagedMaxTokens = 1 << 26;  // token rows of one call
constexpr int64_t kPagedMaxLen = 1 << 30; // tokens that a table row may hold: positions stay clear of 32 bits

// Page p, KV head h, token o (of page_size) is the D contiguous elements at
// k + p·kp + h·kh + o·kt (strides in elements, v likewise).  In an e4m3 pool
// an element's value is its code times the scale of its page and head, a
// power of two kept as fp32 in ks / vs [pages, nkv].
struct PagedPool {
  void *k, *v;
  float *ks, *vs;
  int64_t kp, kh, kt, vp, vh, vt;
  int64_t kse, vse;  // row strides of ks / vs
  int pages, ps, nkv, D, cdtype;
};

// Sequence b owns token rows q_start[b] .. q_start[b + 1] - 1 and, with them
// counted, kv_len[b] cached tokens; token j lives in page table[b][j / ps].
struct PagedBatch {
  const int32_t* table;
  int64_t ld;
  int max_pages;
  const int32_t* q_start;
  const int32_t* kv_len;
  int B, T, max_new;
};

struct PagedAppendArgs {
  PagedPool pool;
  PagedBatch batch;
  int dtype;
  const void* qkv;  // [T, (nq + 2 nkv) D], row stride ldqkv
  int64_t ldqkv;
  int nq;
  const int64_t* positions;  // [T] or NULL (the token's place in the cache)
  const float* cos;          // [max_pos, D/2] or NULL (no rotation)
  const float* sin;
  int max_pos;
  const void* q_norm;  // [D] or NULL
  const void* k_norm;
  float eps;
  void* q_out;  // [T, nq, D], token stride ldq, head stride D
  int64_t ldq;
  int* err;
};
cudaError_t launch_paged_append(const PagedAppendArgs& a, cudaStream_t s);

struct PagedAttnArgs {
  PagedPool pool;
  PagedBatch batch;
  int dtype;
  const void* q;  // token stride ldq, head stride hdq, D contiguous
  int64_t ldq, hdq;
  int nq;
  float scale;
  void* out;
  int64_t ldo, hdo;
  void* ws;
  size_t ws_bytes;
  int* err;
  int sms;  // CTAs of the persistent kernels, read once per call: workspace, offsets and grids follow it
};
size_t paged_attention_workspace(const PagedAttnArgs& a);

// Tensor-core kernel for the sequences with at most kPagedFewRows query rows
// ((token, head) pairs) per KV head (k_paged_decode.cu): it reads the cache
// once for two tiles of 8 rows, the kernel for more rows computes 128-row
// tiles however few they hold (16 sequences on 17 to 5,000 positions, 4 heads
// per KV head, e4m3, pages of 16: exactly 4 tokens each 50 us here, 5 tokens
// each 91 us there).
constexpr int kPagedFewRows = 16;
bool paged_decode_applicable(const PagedAttnArgs& a);
size_t paged_decode_workspace(const PagedAttnArgs& a);
cudaError_t launch_paged_decode(const PagedAttnArgs& a, cudaStream_t s);
// Tensor-core kernel for the sequences with more (k_paged_extend.cu), on the
// same types and head sizes.
size_t paged_extend_workspace(const PagedAttnArgs& a);
cudaError_t launch_paged_extend(const PagedAttnArgs& a, cudaStream_t s);
cudaError_t launch_paged_attention(const PagedAttnArgs& a, cudaStream_t s);

#ifdef __CUDACC__
// What a sequence brings: its first token row, its new tokens, the tokens
// cached before them (negative where the batch has more new than cached
// tokens: the first rows then see no key).  Ranges outside the batch or the
// table make `ok` false and are recorded; the sequence is then left out.
struct SeqSpan {
  int q0, n, past;
  bool ok;
};

__device__ __forceinline__ SeqSpan seq_span(const PagedBatch& b, int i, int ps) {
  const int q0 = b.q_start[i], q1 = b.q_start[i + 1], len = b.kv_len[i];
  SeqSpan s;
  s.ok = q0 >= 0 && q1 >= q0 && q1 <= b.T && q1 - q0 <= b.max_new && len >= 0 &&
         (int64_t)len <= (int64_t)b.max_pages * ps;
  s.q0 = q0;
  s.n = s.ok ? q1 - q0 : 0;
  s.past = s.ok ? len - s.n : 0;
  return s;
}

// 2^e as a float, 0 below the normal range.
__device__ __forceinline__ float pow2i(int e) {
  return e < -126 ? 0.f : __uint_as_float((uint32_t)(min(e, 127) + 127) << 23);
}
// The exponent of a scale (a power of two).
__device__ __forceinline__ int scale_exp(float s) { return (int)((__float_as_uint(s) >> 23) & 0xffu) - 127; }

// The least e >= kPagedMinExp with amax <= 448·2^e (448 = 1.75·2^8 is the
// largest e4m3 value), at most kPagedMaxExp; amax >= 0 and finite.
__device__ __forceinline__ int e4m3_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kPagedMinExp), kPagedMaxExp);
}

// Two floats to two e4m3 codes, to nearest even; beyond ±448 (infinities
// too) the largest value, NaN stays NaN.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// Two codes (low half first) to floats; every e4m3 value is a half.
__device__ __forceinline__ float2 from_e4m3x2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
#endif

}  // namespace mg
