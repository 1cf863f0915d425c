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

}  // namespace paged
}  // namespace mg
