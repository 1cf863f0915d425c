// Helpers shared by the tensor-core kernels over a paged KV cache: tensor
// maps of the pools, conversions of e4m3 codes, fp16 MMAs.
#pragma once

#include "attn_tc_common.cuh"
#include "paged.h"
#include "tc_common.cuh"

namespace mg {
namespace paged {

constexpr int kSlice = 16;  // token rows of the small box: a sequence's last page is loaded in such slices

// K and V of a pool as 4-D arrays {dim, token, head, page}: one box of a
// whole page, one of kSlice tokens.
struct PoolMaps {
  CUtensorMap k, v, k_tail, v_tail;
};

// The element of a pool that the tensor-core kernels read, and its row in
// shared memory: 64 bf16 dims to a 128-byte swizzled block, an e4m3 row of
// 128 or 64 bytes swizzled over its own width.
template <int D, bool E4>
struct PoolRow {
  static constexpr int kBlocks = E4 ? 1 : D / 64;         // boxes per token row
  static constexpr int kBlockDims = E4 ? D : 64;          // dims of a box
  static constexpr int kBytes = E4 ? D : 128;             // bytes of a box row
  static constexpr int kRowBytes = D * (E4 ? 1 : 2);
  // Byte offset of 16-byte piece c of token row r inside a block.
  static __device__ __forceinline__ uint32_t at(int r, int c) {
    if constexpr (kBytes == 128) return r * 128 + ((c ^ (r & 7)) << 4);
    return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  }
};

inline bool pool_map(CUtensorMap* tm, const PagedPool& p, const void* base, int64_t ps, int64_t hs, int64_t ts,
                     int box_dims, int box_rows) {
  tc_host::EncodeTiled enc = tc_host::encoder();
  if (!enc) return false;
  const bool e4 = p.cdtype == kE4M3;
  const cuuint64_t esz = e4 ? 1 : 2;
  const cuuint64_t dims[4] = {(cuuint64_t)p.D, (cuuint64_t)p.ps, (cuuint64_t)p.nkv, (cuuint64_t)p.pages};
  const cuuint64_t strides[3] = {(cuuint64_t)ts * esz, (cuuint64_t)hs * esz, (cuuint64_t)ps * esz};
  const cuuint32_t box[4] = {(cuuint32_t)box_dims, (cuuint32_t)box_rows, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(tm, e4 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base),
             dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             box_dims * (int)esz == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool E4>
inline bool pool_maps(PoolMaps* m, const PagedPool& p) {
  constexpr int dims = PoolRow<D, E4>::kBlockDims;
  return pool_map(&m->k, p, p.k, p.kp, p.kh, p.kt, dims, p.ps) && pool_map(&m->v, p, p.v, p.vp, p.vh, p.vt, dims, p.ps) &&
         pool_map(&m->k_tail, p, p.k, p.kp, p.kh, p.kt, dims, kSlice) &&
         pool_map(&m->v_tail, p, p.v, p.vp, p.vh, p.vt, dims, kSlice);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Over e4m3 pages the running maximum m of a row is one of s + e (2^e the scale
// of the values' page), while its sum l holds Σ 2^(s - m), the keys' own
// weights.
//   * A key is added as 2^(s + e - m + offset)·2^(-e - offset), offset at least
//     7, of which the first factor vanishes below 2^-126.  The key is then below
//     2^(span - 133) of l, `span` the difference of the row's largest and least
//     e: nothing up to a span of 108 (2^-25), but it can be all of l beyond, with
//     e > 8 on one page and a page of zeros, e = -100, on the other.  Rows that
//     see so wide a span are computed again by redo_row, whose maximum is one of
//     s: the kernels note whether a piece has met a scale above 2^8 (values
//     above 114,688), and wide_row then looks at the sequence's pages.
//   * l·2^d is taken in two steps, as 2^d alone may vanish where l does not.
constexpr int kSpan = 108;
__device__ __forceinline__ bool high_scale(float scale) { return scale > 256.f; }
static_assert(kSpan + kPagedMinExp == 8, "no wider span without a high scale");
// L + l·2^d with f = 2^d: a piece's sum joined to those of others.
template <bool E4>
__device__ __forceinline__ float add_sum(float L, float l, float d, float f) {
  if constexpr (E4) {
    if (d < -64.f) {
      const float h = ex2(0.5f * d);
      return L + l * h * h;
    }
  }
  return fmaf(f, l, L);
}

// Two e4m3 codes (the low half of `codes`) to two halves: exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}

// Two floats to a half pair, `lo` in the low half.
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// D (16x8, fp32) += A (16x16) B (16x8), halves.
__device__ __forceinline__ void mma16816_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The factor that brings a row of largest magnitude `amax` to [128, 256): a
// power of two, so a bf16 row becomes halves exactly, but for elements below
// 2^-21 of the largest, which are off by at most 2^-33 of it.
__device__ __forceinline__ int row_shift(float amax) {
  return amax > 0.f ? min(7 - ((int)(__float_as_uint(amax) >> 23) - 127), 126) : 0;
}

// The sequence of token row t (-1: none), by a whole warp, and the keys that t sees.
__device__ __forceinline__ int seq_of_row(const PagedAttnArgs& a, int t, int* vis) {
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < a.batch.B; b0 += 32) {
    SeqSpan s{0, 0, 0, false};
    if (b0 + lane < a.batch.B) s = seq_span(a.batch, b0 + lane, a.pool.ps);
    const unsigned found = __ballot_sync(0xffffffffu, s.ok && s.q0 <= t && t < s.q0 + s.n);
    if (found) {
      *vis = __shfl_sync(0xffffffffu, s.past + t - s.q0 + 1, __ffs(found) - 1);
      return b0 + __ffs(found) - 1;
    }
  }
  return -1;
}

// Whether the exponents of the value pages that token row t sees, of KV head h,
// span more than kSpan; by a whole warp.
static __device__ __noinline__ bool wide_row(const PagedAttnArgs& a, int t, int h) {
  const PagedPool& pool = a.pool;
  int vis = 0, lo = 127, hi = -127;
  const int b = seq_of_row(a, t, &vis);
  if (b < 0) return false;
  for (int i = threadIdx.x & 31; (int64_t)i * pool.ps < vis; i += 32) {
    const int page = a.batch.table[(int64_t)b * a.batch.ld + i];
    const int e = page >= 0 && page < pool.pages ? max(scale_exp(pool.vs[page * pool.vse + h]), kPagedMinExp) : 0;
    lo = min(lo, e);
    hi = max(hi, e);
  }
  return __reduce_max_sync(0xffffffffu, hi) - __reduce_min_sync(0xffffffffu, lo) > kSpan;
}

// One (token row, query head) again, by a whole warp, key
// by key in fp32.  The tensor-core kernels multiply all values of a block, a
// row's invisible ones by the weight 0, and 0 times an infinity or a NaN of a
// later token is NaN: a row that comes out with NaN is computed again from
// what it sees.  So is one that sees such a value, which then comes out as the
// formula has it; some 100 ns per key, paid by rows that are lost anyway.
template <int D, bool E4>
__device__ __noinline__ void redo_row(const PagedAttnArgs& a, int t, int head) {
  constexpr int N = D / 32;  // dims of a lane
  const PagedPool& pool = a.pool;
  const int lane = threadIdx.x & 31, h = head / (a.nq / pool.nkv);
  int vis = 0;
  const int b = seq_of_row(a, t, &vis);
  if (b < 0) return;
  float q[N], acc[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = __bfloat162float(((const __nv_bfloat16*)a.q)[(int64_t)t * a.ldq + (int64_t)head * a.hdq + lane * N + i]) *
           (a.scale * 1.4426950408889634f);
    acc[i] = 0.f;
  }
#pragma unroll 1
  for (int j = 0; j < vis; ++j) {
    const int page = a.batch.table[(int64_t)b * a.batch.ld + j / pool.ps], o = j % pool.ps;
    float k[N], v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) k[i] = v[i] = 0.f;
    if (page >= 0 && page < pool.pages) {
      const int64_t kat = page * pool.kp + h * pool.kh + o * pool.kt + lane * N;
      const int64_t vat = page * pool.vp + h * pool.vh + o * pool.vt + lane * N;
      const float fk = E4 ? pool.ks[page * pool.kse + h] : 1.f, fv = E4 ? pool.vs[page * pool.vse + h] : 1.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (E4) {
          k[i] = from_e4m3x2(((const uint8_t*)pool.k)[kat + i]).x * fk;
          v[i] = from_e4m3x2(((const uint8_t*)pool.v)[vat + i]).x * fv;
        } else {
          k[i] = __bfloat162float(((const __nv_bfloat16*)pool.k)[kat + i]);
          v[i] = __bfloat162float(((const __nv_bfloat16*)pool.v)[vat + i]);
        }
      }
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    const float top = fmaxf(m, s), keep = m == -INFINITY ? 0.f : ex2(m - top);
    const float w = s == -INFINITY ? 0.f : ex2(s - top);  // also where nothing lies above -inf yet
    m = top;
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = acc[i] * keep + w * v[i];
  }
  __nv_bfloat16* out = (__nv_bfloat16*)a.out + (int64_t)t * a.ldo + (int64_t)head * a.hdo;
#pragma unroll
  for (int i = 0; i < N; ++i) out[lane * N + i] = __float2bfloat16_rn(l == 0.f ? 0.f : acc[i] / l);
}

// The same for a row that this block has written, if it holds a NaN or its sequence's scales span too much (`wide`).
template <int D, bool E4>
__device__ __forceinline__ void redo_if_lost(const PagedAttnArgs& a, int t, int head, bool wide) {
  const __nv_bfloat16* out = (const __nv_bfloat16*)a.out + (int64_t)t * a.ldo + (int64_t)head * a.hdo;
  bool bad = false;
  for (int d = threadIdx.x & 31; d < D; d += 32) bad |= __hisnan(out[d]);
  if (wide || __any_sync(0xffffffffu, bad)) redo_row<D, E4>(a, t, head);
}

}  // namespace paged
}  // namespace mg
