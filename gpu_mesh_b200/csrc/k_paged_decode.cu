// Attention over a paged KV cache for sequences that bring few tokens: at
// most 16 query rows (new tokens x query heads) per KV head.  bf16
// activations, head_dim 64 or 128, pages in bf16 or e4m3.
//
// The cache is read once and every byte feeds at most 32 query rows' worth of
// FLOPs, so memory is the bound.  What the kernel does about it:
//   * Work split.  The units are (sequence, KV head, block of 32 keys, 16 over
//     bf16 pages) of the lengths as they are on the device.  Every CTA (one per
//     SM) takes an equal contiguous run of them, whose ends move to the end of
//     a (sequence, head) where one is near, and deals it to its warps the same
//     way; each warp streams its part by itself, without a barrier.  Then the
//     CTA joins what its warps' ends cut, once, in shared memory.  A (sequence,
//     head) that CTAs' ends cut leaves (max, sum, O) in the workspace, and a
//     second kernel joins those pieces in order: no counters to initialise, so
//     a captured call can be replayed and its result does not depend on timing.
//   * Loads.  Keys and values go from memory straight into the registers that
//     the MMAs read.  The order of the dims inside a score product is free,
//     so a thread's K fragments are 16 consecutive bytes of its keys; the
//     order of the output dims is free too, so its V fragments are D / 8
//     consecutive elements of four keys, paired by byte permutes.  Every load
//     instruction covers whole 64- or 128-byte rows whatever the page size
//     (16-token pages cost one table lookup more, not more requests), and
//     each warp has the next block's loads in flight while it computes.
//   * Compute.  Transposed products, so that the query rows sit on the MMA's N = 8
//     side: Sᵀ = K·Qᵀ (M = 16 keys), Oᵀ = Vᵀ·Pᵀ (M = 16 dims), fp32
//     accumulators, online softmax in base 2.
//       bf16 pages: bf16 MMAs, P split into bf16 high + low parts (2^-17).
//       e4m3 pages: codes become halves in registers (exact), Q as halves
//       scaled by a power of two per row (exact), K's scale multiplies the
//       fp32 scores.  V's scale 2^e goes into the exponent: with the running
//       maximum m of s + e, P' = 2^(s + e - m + 14) (rounded to half: 2^-11
//       relative, down to 2^-28 of the largest, and within 2^-39 of it below)
//       weighs the raw codes, while the sum adds P'·2^(-e - 14) = 2^(s - m) in
//       fp32 (scales far apart: kSpan); out = O / l · 2^-14.
//
// Measured (32 query, 8 KV heads of 128): 64 tokens on 7.9 to 8.2 K positions,
// e4m3, 204 us = 5.2 TB/s; 32 tokens, bf16, 182 us = 5.8 TB/s (a copy runs at
// 6.5); 32 tokens on 1 K, e4m3 27 us, bf16 37 us; one token on 130, 8.5 us.
// The long ones are bound by a warp's way through a block between its
// requests (issue slots 37 % active, 8 warps per SM), the short ones by their
// round trips: lengths, page, block, the CTA's join, the second kernel.
// Through a shared-memory ring, filled by TMA or cp.async, the long one took
// 266 us, and more with smaller pages.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "paged_tc.cuh"

namespace mg {
namespace {

using namespace attn;
using namespace paged;

constexpr int kWarps = 8;   // of a CTA (one per SM): 255 registers each; 12 or 16 warps spill, and were slower
constexpr int kRowsD = 16;  // most query rows of a (sequence, head)

// Keys of a block.
__host__ __device__ constexpr int block_keys(bool e4) { return e4 ? 32 : 16; }

// Blocks of a sequence and KV head that this kernel takes (0: none, or left
// to the kernel for many tokens).
__device__ __forceinline__ int decode_blocks(const SeqSpan& s, int G, int bk) {
  if (s.n < 1 || s.n * G > kRowsD) return 0;
  const int len = s.past + s.n;
  return len > 0 ? (len + bk - 1) / bk : 1;  // no keys at all: one block that writes zeros
}

// Blocks that a CTA's run's end moves to end with a (sequence, head).  0, 4, 8,
// 16: one token on 130 positions 12.1, 9.6, 8.5, 8.5 us; 16 sequences of up to
// 5 K with 2 to 4 tokens 49.2, 49.6, 43.7, 46.5 us; the others within 4 %.
constexpr int kSnap = 8;

// Blocks of a CTA's run at least, where there are few: its warps take one each,
// and the pieces to join get fewer (2 sequences of up to 1.2 K positions, 5
// tokens, 2 KV heads: 22.6 us, with runs of one block 29.1; runs of eight take
// one token on 130 positions from 8.5 to 11.4 us).
constexpr int kLeast = 4;

// What a CTA leaves for the join: the (sequence, head) that its run ends and
// earlier ones began, as its first token row, KV head, query rows (0: there
// is none) and number of pieces, this run's the last; and whether its piece in
// slot 0 or 1 has met a high_scale.
struct Cut {
  int q0, h, rows, pieces;
  int high[2], pad[2];
};

// What a warp's piece of a cut (sequence, head) is: rows 0 where there is none.
struct PieceMeta {
  int b, h, rows, ends, high;
};

// Floats of a run's piece of one (sequence, head): per row O [D], max, sum.
__host__ __device__ constexpr int piece_floats(int rows, int D) { return rows * (D + 2); }

// 16 (or 8) bytes of the cache, read once: not kept in L1.
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load_once8(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

template <int D, bool E4, int NT>
__global__ void __launch_bounds__(kWarps * 32, 1) paged_decode_kernel(const __grid_constant__ PagedAttnArgs a, int row_cap) {
  constexpr int KS = D / 16;                     // k-steps of the score MMA
  constexpr int DM = D / 16;                     // dim tiles of Oᵀ
  constexpr int BK = block_keys(E4), SUB = BK / 16;  // keys of a block, its 16-key tiles
  constexpr int KP = D * (E4 ? 1 : 2) / 64;      // 16-byte pieces of a key that a thread holds (four threads a key)
  constexpr int VW = D / 8 * (E4 ? 1 : 2) / 4;   // words of a value row that a thread holds (eight threads a row)
  constexpr int QW = KS / 2;       // 16-byte words of a query row that a thread holds
  constexpr int ES = E4 ? 1 : 2;
  const PagedPool& pool = a.pool;
  const PagedBatch& bt = a.batch;
  const int G = a.nq / pool.nkv, nkv = pool.nkv;
  // Two tiles of query rows keep their fragments in shared memory: in registers
  // (and requested a piece ahead) they spill (16 sequences of up to 5 K keys, 2
  // to 4 tokens each, e4m3: 57 us against 43).
  constexpr bool kQShared = NT == 2;
  __shared__ uint2 qs[kQShared ? kWarps : 1][kQShared ? NT * KS : 1][32];
  extern __shared__ __align__(16) float held[];  // [warp][2][row][O(D), max, sum]: pieces for the CTA's join
  __shared__ int lost;                           // a row came out with NaN, or its pages may span too much
  __shared__ PieceMeta meta[kWarps][2];          // 0: began in an earlier warp's part, 1: goes on in the next one's
  int* pre = (int*)(held + 2 * kWarps * piece_floats(row_cap, D));  // [B + 1] blocks before a sequence
  int* slen = pre + bt.B + 1;                                       // [B] cached tokens
  int* sqn = slen + bt.B;                                           // [B] first token row · 32 + new tokens

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  // This grid may be resident while the append before it writes pages, scales
  // and tables: everything is read behind this wait by ordinary loads, as the
  // non-coherent ones are for data that nothing writes in a kernel's lifetime.
  pdl_wait();
  for (int b = tid; b < bt.B; b += kWarps * 32) {
    const SeqSpan s = seq_span(bt, b, pool.ps);
    if (!s.ok && blockIdx.x == 0) flag_error(a.err, kErrPaged);
    pre[b + 1] = decode_blocks(s, G, BK);
    slen[b] = s.past + s.n;
    sqn[b] = s.q0 * 32 + (s.n & 31);
  }
  // The join kernel may start now: what it reads before its own wait was
  // written before this kernel.
  pdl_trigger();
  __syncthreads();
  if (warp == 0) {  // blocks before each sequence, over its KV heads, summed
    long long run = 0;
    for (int b0 = 0; b0 < bt.B; b0 += 32) {
      const int b = b0 + lane;
      long long x = b < bt.B ? (long long)pre[b + 1] * nkv : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      x += run;
      if (b < bt.B) pre[b + 1] = (int)(x < 0x7fffffffLL ? x : 0x7fffffffLL);
      run = __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) {
      pre[0] = 0;
      if (run >= 0x7fffffffLL) {  // 2^35 cached tokens: no pool holds them
        flag_error(a.err, kErrPaged);
        pre[bt.B] = 0;
      }
    }
  }
  __syncthreads();
  const int total = pre[bt.B], c = blockIdx.x, grid = min((int)gridDim.x, (total + kLeast - 1) / kLeast);
  auto seq_of = [&](int u) {
    int lo = 0, hi = bt.B;  // pre[lo] <= u < pre[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= u) lo = mid; else hi = mid;
    }
    return lo;
  };
  auto begin = [&](int k) {  // of CTA k's run
    const int u = (int)((long long)k * total / grid);
    if (u >= total) return total;
    const int b = seq_of(u), nb = max(1, (slen[b] + BK - 1) / BK), off = (u - pre[b]) % nb;
    return off <= kSnap ? u - off : nb - off <= kSnap ? u + nb - off : u;
  };
  // No workspace where no (sequence, head) can be cut.
  Cut* cuts = (Cut*)((float*)a.ws + (size_t)2 * gridDim.x * piece_floats(row_cap, D));
  if (a.ws && tid == 0) cuts[c] = Cut{};
  if (tid < 2 * kWarps) meta[tid >> 1][tid & 1].rows = 0;
  if (tid == 0) lost = 0;
  if (c >= grid) return;
  const int c0 = begin(c), c1 = begin(c + 1);
  if (c0 >= c1) return;
  __syncthreads();  // meta is cleared
  // The warp's part of the run; where there are fewer blocks than warps the last ones have none.
  const int parts = min(kWarps, c1 - c0), part_of = min(warp, parts);
  const int u0 = c0 + (int)((long long)(c1 - c0) * part_of / parts);
  const int u1 = c0 + (int)((long long)(c1 - c0) * min(part_of + 1, parts) / parts);

  // The part's blocks, in order.  Data is requested one block ahead of the
  // computation, pages are looked up two ahead.
  struct Block {
    int b, h, k0, len;  // keys k0 .. of the sequence's len
    int page[SUB];      // -1: no key there, or outside the pool (its keys read as zeros)
    bool valid, first, last;  // first / last block of its piece of the part
    bool full;          // every key of the block is there
  };
  const int page_shift = 31 - __clz(pool.ps);
  int cu = u0, cb, ch, cblk, cnb, clen;
  const int32_t* ctab;
  {
    cb = seq_of(min(cu, total - 1));
    clen = slen[cb];
    cnb = max(1, (clen + BK - 1) / BK);
    ch = (cu - pre[cb]) / cnb;
    cblk = (cu - pre[cb]) - ch * cnb;
    ctab = bt.table + (int64_t)cb * bt.ld;
  }
  bool fresh = true;
  auto next_block = [&]() {
    Block x;
    x.valid = cu < u1;
    x.b = cb;
    x.h = ch;
    x.k0 = cblk * BK;
    x.len = x.valid ? clen : 0;
    x.first = fresh || cblk == 0;
    x.last = cblk + 1 == cnb || cu + 1 == u1;
    fresh = false;
#pragma unroll
    for (int i = 0; i < SUB; ++i)
      x.page[i] = x.k0 + 16 * i < x.len ? ctab[(x.k0 + 16 * i) >> page_shift] : -1;
    ++cu;
    if (++cblk == cnb && cu < u1) {
      cblk = 0;
      if (++ch == nkv) {
        ch = 0;
        do ++cb; while (pre[cb + 1] == pre[cb]);
        clen = slen[cb];
        cnb = max(1, (clen + BK - 1) / BK);
        ctab = bt.table + (int64_t)cb * bt.ld;
      }
    }
    return x;
  };
  // The page numbers, a block later: they have arrived by then.
  auto check = [&](Block& x) {
    x.full = x.k0 + BK <= x.len;
#pragma unroll
    for (int i = 0; i < SUB; ++i)
      if ((unsigned)x.page[i] >= (unsigned)pool.pages) {
        if (x.k0 + 16 * i < x.len) flag_error(a.err, kErrPaged);
        x.page[i] = -1;
        x.full = false;
      }
  };
  uint4 kx[SUB][2][KP];       // keys g, g + 8 of each tile
  uint32_t vx[SUB][4][VW];    // values 2t, 2t + 1, 2t + 8, 2t + 9
  float ks[SUB], vs[SUB];
  uint4 qx[QW];               // query row g
  // Query row g of 8-row tile nt, its dims in the order of the K fragments: a
  // thread's 16 bytes of a key are 16 (bf16: 8) consecutive dims, k-steps of
  // four dims each.
  auto load_q = [&](const Block& x, int nt, uint4* to) {
    const int r = nt * 8 + g;
    const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + (int64_t)((sqn[x.b] >> 5) + r / G) * a.ldq +
                             (int64_t)(x.h * G + r % G) * a.hdq;
#pragma unroll
    for (int i = 0; i < QW; ++i)
      to[i] = r < (sqn[x.b] & 31) * G
                  ? *reinterpret_cast<const uint4*>(E4 ? q + 64 * (i / 2) + 16 * t + 8 * (i % 2) : q + 32 * i + 8 * t)
                  : make_uint4(0u, 0u, 0u, 0u);
  };
  // A block's keys (both scales, and the query rows of a new piece) and values:
  // each half is requested as soon as the registers of the block before are
  // free.  Offsets of a thread's rows inside a tile, in bytes; the tile lies in one page.
  const int64_t koff = (int64_t)g * pool.kt * ES + 16 * t, k8 = 8 * pool.kt * ES;
  const int64_t voff = (int64_t)2 * t * pool.vt * ES + g * (VW * 4), v1 = pool.vt * ES, v8 = 8 * v1;
  auto load_k = [&](const Block& x) {
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
      const int k0 = x.k0 + 16 * i, page = x.page[i];
      const uint8_t* kp = (const uint8_t*)pool.k + (page * pool.kp + x.h * pool.kh + (k0 & (pool.ps - 1)) * pool.kt) * ES + koff;
      if (x.full) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int p = 0; p < KP; ++p) kx[i][r][p] = load_once(kp + r * k8 + 64 * p);
      } else {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int p = 0; p < KP; ++p)
            kx[i][r][p] = page >= 0 && k0 + g + 8 * r < x.len ? load_once(kp + r * k8 + 64 * p) : make_uint4(0u, 0u, 0u, 0u);
      }
      if constexpr (E4) {
        ks[i] = page >= 0 ? pool.ks[page * pool.kse + x.h] : 0.f;
        vs[i] = page >= 0 ? pool.vs[page * pool.vse + x.h] : 1.f;
      }
    }
    if (!kQShared && x.valid && x.first) load_q(x, 0, qx);
  };
  auto load_v = [&](const Block& x) {
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
      const int k0 = x.k0 + 16 * i, page = x.page[i];
      const uint8_t* vp = (const uint8_t*)pool.v + (page * pool.vp + x.h * pool.vh + (k0 & (pool.ps - 1)) * pool.vt) * ES + voff;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool ok = page >= 0 && k0 + 2 * t + (r & 1) + 8 * (r >> 1) < x.len;
        const uint8_t* at = vp + (r & 1) * v1 + (r >> 1) * v8;
        if constexpr (VW == 2) {
          uint2 v = make_uint2(0u, 0u);
          if (x.full) v = load_once8(at);
          else if (ok) v = load_once8(at);
          vx[i][r][0] = v.x;
          vx[i][r][1] = v.y;
        } else {
#pragma unroll
          for (int p = 0; p < VW / 4; ++p) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (x.full) v = load_once(at + 16 * p);
            else if (ok) v = load_once(at + 16 * p);
            vx[i][r][4 * p] = v.x;
            vx[i][r][4 * p + 1] = v.y;
            vx[i][r][4 * p + 2] = v.z;
            vx[i][r][4 * p + 3] = v.w;
          }
        }
      }
    }
  };
  Block now = next_block();
  check(now);
  load_k(now);
  load_v(now);
  Block next = next_block();

  const float scale2 = a.scale * 1.4426950408889634f;
  // Thread (g, t) holds keys g, g + 8 (dims of Oᵀ by tile) for the query
  // rows 2t, 2t + 1 of each 8-row tile; vis: keys those rows see.
  int rows = 0, least = 0, from = 0, vis[NT][2];
  float mrow[NT][2], lrow[NT][2], rowf[NT][2];
  float top_vs = 0.f;  // largest scale of the piece's values (a flag took 2.3 % more: 209 us on 8 K)
  float o[NT][DM][4];
  uint32_t qb[KS][2] = {};  // of the only tile
  auto query = [&](int nt, int ks) {  // the B fragment of k-step ks
    if constexpr (kQShared) return qs[warp][nt * KS + ks][lane];
    return make_uint2(qb[ks][0], qb[ks][1]);
  };
  while (now.valid) {
    if (now.first) {
      const int n = sqn[now.b] & 31, past = now.len - n;
      rows = n * G;
      top_vs = 0.f;
      least = past + 1;  // keys that every row sees
      from = now.k0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + 2 * t + e;
          vis[nt][e] = r < rows ? past + r / G + 1 : 0;
          mrow[nt][e] = -INFINITY;
          lrow[nt][e] = 0.f;
          rowf[nt][e] = scale2;
        }
#pragma unroll
        for (int i = 0; i < DM; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        auto keep = [&](int ks, uint32_t b0, uint32_t b1) {
          if constexpr (kQShared) qs[warp][nt * KS + ks][lane] = make_uint2(b0, b1);
          else qb[ks][0] = b0, qb[ks][1] = b1;
        };
        if constexpr (kQShared) load_q(now, nt, qx);
        if constexpr (E4) {
          float amax = 0.f;
#pragma unroll
          for (int i = 0; i < QW; ++i) {
            const uint32_t x[4] = {qx[i].x, qx[i].y, qx[i].z, qx[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) amax = fmaxf(amax, fmaxf(fabsf(lo_bf16(x[k])), fabsf(hi_bf16(x[k]))));
          }
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          const int sh = row_shift(amax);
          const float f = pow2i(sh);
#pragma unroll
          for (int i = 0; i < QW; ++i) {
            const uint4 x = qx[i];
            keep(2 * i, pack_f16(lo_bf16(x.x) * f, hi_bf16(x.x) * f), pack_f16(lo_bf16(x.y) * f, hi_bf16(x.y) * f));
            keep(2 * i + 1, pack_f16(lo_bf16(x.z) * f, hi_bf16(x.z) * f), pack_f16(lo_bf16(x.w) * f, hi_bf16(x.w) * f));
          }
          // Row g's factor is needed by the threads that hold rows 2t, 2t + 1.
#pragma unroll
          for (int e = 0; e < 2; ++e) rowf[nt][e] = scale2 * pow2i(-__shfl_sync(0xffffffffu, sh, (2 * t + e) * 4));
        } else {
#pragma unroll
          for (int i = 0; i < QW; ++i) {
            keep(2 * i, qx[i].x, qx[i].y);
            keep(2 * i + 1, qx[i].z, qx[i].w);
          }
        }
      }
    }
    const int j0 = now.k0;
    float sc[NT][SUB][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < SUB; ++i) sc[nt][i][0] = sc[nt][i][1] = sc[nt][i][2] = sc[nt][i][3] = 0.f;
#pragma unroll
    for (int q = 0; q < KP; ++q) {
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        const uint32_t x[4] = {kx[i][0][q].x, kx[i][0][q].y, kx[i][0][q].z, kx[i][0][q].w};
        const uint32_t y[4] = {kx[i][1][q].x, kx[i][1][q].y, kx[i][1][q].z, kx[i][1][q].w};
        if constexpr (E4) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t a0 = e4m3x2_to_f16x2(x[w]), a1 = e4m3x2_to_f16x2(y[w]);
            const uint32_t a2 = e4m3x2_hi_to_f16x2(x[w]), a3 = e4m3x2_hi_to_f16x2(y[w]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint2 b = query(nt, 4 * q + w);
              mma16816_f16(sc[nt][i], a0, a1, a2, a3, b.x, b.y);
            }
          }
        } else {
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint2 b = query(nt, 2 * q + w);
              mma16816_full(sc[nt][i], x[2 * w], y[2 * w], x[2 * w + 1], y[2 * w + 1], b.x, b.y);
            }
        }
      }
    }
    float ksc[SUB], vw[SUB];  // vw: 2^(-e - 14)
    int ve[SUB];
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
      ksc[i] = E4 ? ks[i] : 1.f;
      ve[i] = E4 ? scale_exp(vs[i]) : 0;
      vw[i] = E4 ? pow2i(-ve[i] - 14) : 1.f;
      if (E4) top_vs = fmaxf(top_vs, vs[i]);
    }
    check(next);
    load_k(next);
    // Online softmax per query row (column): keys g (c0, c1), g + 8 (c2, c3) of each tile.
    uint32_t ph[NT][SUB][2], plo[NT][SUB][2];
    const bool clear = j0 + BK <= least;  // every key of the block is visible to every row
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx[2] = {mrow[nt][0], mrow[nt][1]};
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        float* s = sc[nt][i];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = rowf[nt][e] * ksc[i];
          s[e] = E4 ? fmaf(s[e], f, (float)ve[i]) : s[e] * f;
          s[2 + e] = E4 ? fmaf(s[2 + e], f, (float)ve[i]) : s[2 + e] * f;
          if (!clear) {
            s[e] = j0 + 16 * i + g < vis[nt][e] ? s[e] : -INFINITY;
            s[2 + e] = j0 + 16 * i + g + 8 < vis[nt][e] ? s[2 + e] : -INFINITY;
          }
          mx[e] = fmaxf(mx[e], fmaxf(s[e], s[2 + e]));
        }
      }
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
      }
      if (__any_sync(0xffffffffu, mx[0] != mrow[nt][0] || mx[1] != mrow[nt][1])) {
        float keep[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float d = mrow[nt][e] == -INFINITY ? -INFINITY : mrow[nt][e] - mx[e];
          mrow[nt][e] = mx[e];
          if constexpr (E4) {
            const float half = ex2(0.5f * d);
            keep[e] = half * half;
            lrow[nt][e] = lrow[nt][e] * half * half;
          } else {
            keep[e] = ex2(d);
            lrow[nt][e] *= keep[e];
          }
        }
#pragma unroll
        for (int i = 0; i < DM; ++i) {
          o[nt][i][0] *= keep[0];
          o[nt][i][1] *= keep[1];
          o[nt][i][2] *= keep[0];
          o[nt][i][3] *= keep[1];
        }
      }
      // A row that has seen no key yet keeps m = -inf: every weight is 0.
      const float base0 = mx[0] == -INFINITY ? 0.f : mx[0] - (E4 ? 14.f : 0.f);
      const float base1 = mx[1] == -INFINITY ? 0.f : mx[1] - (E4 ? 14.f : 0.f);
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        float* s = sc[nt][i];
        s[0] = ex2(s[0] - base0);
        s[1] = ex2(s[1] - base1);
        s[2] = ex2(s[2] - base0);
        s[3] = ex2(s[3] - base1);
        if constexpr (E4) {
          lrow[nt][0] = fmaf(s[0] + s[2], vw[i], lrow[nt][0]);
          lrow[nt][1] = fmaf(s[1] + s[3], vw[i], lrow[nt][1]);
          // Pᵀ as the B operand of Oᵀ += Vᵀ·Pᵀ: an 8x8 (keys x rows) matrix each, transposed in registers.
          ph[nt][i][0] = movm_trans(pack_f16(s[0], s[1]));
          ph[nt][i][1] = movm_trans(pack_f16(s[2], s[3]));
        } else {
          lrow[nt][0] += s[0] + s[2];
          lrow[nt][1] += s[1] + s[3];
          const uint32_t h01 = pack2(s[0], s[1]), h23 = pack2(s[2], s[3]);
          ph[nt][i][0] = movm_trans(h01);
          ph[nt][i][1] = movm_trans(h23);
          plo[nt][i][0] = movm_trans(pack2(s[0] - lo_bf16(h01), s[1] - hi_bf16(h01)));
          plo[nt][i][1] = movm_trans(pack2(s[2] - lo_bf16(h23), s[3] - hi_bf16(h23)));
        }
      }
    }
    // Tile j of Oᵀ: rows g and g + 8 are the thread's dims 2j and 2j + 1.
#pragma unroll
    for (int j = 0; j < DM; ++j) {
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        if constexpr (E4) {
          const int sel = j & 1 ? 0x7362 : 0x5140;
          const uint32_t y0 = __byte_perm(vx[i][0][j / 2], vx[i][1][j / 2], sel);
          const uint32_t y1 = __byte_perm(vx[i][2][j / 2], vx[i][3][j / 2], sel);
          const uint32_t a0 = e4m3x2_to_f16x2(y0), a1 = e4m3x2_hi_to_f16x2(y0);
          const uint32_t a2 = e4m3x2_to_f16x2(y1), a3 = e4m3x2_hi_to_f16x2(y1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816_f16(o[nt][j], a0, a1, a2, a3, ph[nt][i][0], ph[nt][i][1]);
        } else {
          const uint32_t a0 = __byte_perm(vx[i][0][j], vx[i][1][j], 0x5410), a1 = __byte_perm(vx[i][0][j], vx[i][1][j], 0x7632);
          const uint32_t a2 = __byte_perm(vx[i][2][j], vx[i][3][j], 0x5410), a3 = __byte_perm(vx[i][2][j], vx[i][3][j], 0x7632);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816_full(o[nt][j], a0, a1, a2, a3, ph[nt][i][0], ph[nt][i][1]);
            mma16816_full(o[nt][j], a0, a1, a2, a3, plo[nt][i][0], plo[nt][i][1]);
          }
        }
      }
    }
    load_v(next);
    if (now.last) {  // end of the piece: out, or kept for the CTA's join
      const bool ends = now.k0 + BK >= now.len, whole = from == 0 && ends;
      const int slot = from > 0 ? 0 : 1;
      if (!whole && lane == 0) meta[warp][slot] = PieceMeta{now.b, now.h, rows, ends, high_scale(top_vs)};
      if (E4 && whole && high_scale(top_vs)) lost = 1;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float l = lrow[nt][e];
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
          const int r = nt * 8 + 2 * t + e;
          if (r >= rows) continue;
          // The thread's D / 8 dims of the row.
          float x[D / 8];
#pragma unroll
          for (int j = 0; j < DM; ++j) x[2 * j] = o[nt][j][e], x[2 * j + 1] = o[nt][j][2 + e];
          const float unit = E4 ? 1.f / 16384.f : 1.f;
          if (whole) {
            const float f = l == 0.f ? 0.f : unit / l;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) x[i] *= f;
            __nv_bfloat16* out = (__nv_bfloat16*)a.out + (int64_t)((sqn[now.b] >> 5) + r / G) * a.ldo +
                                 (int64_t)(now.h * G + r % G) * a.hdo + g * (D / 8);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) store16_f<__nv_bfloat16>(out + 8 * i, x + 8 * i);
            float bad = 0.f;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) bad = fmaf(x[i], 0.f, bad);
            if (bad != 0.f) lost = 1;
          } else {
            float* part = held + (size_t)(2 * warp + slot) * piece_floats(row_cap, D) + r * (D + 2);
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
              *reinterpret_cast<float2*>(part + g * (D / 8) + 2 * i) = make_float2(x[2 * i] * unit, x[2 * i + 1] * unit);
            if (g == 0) *reinterpret_cast<float2*>(part + D) = make_float2(mrow[nt][e], l);
          }
        }
      }
    }
    now = next;
    next = next_block();
  }
  __syncthreads();
  // Chains of pieces of one (sequence, head): a slot 1, or warp 0's slot 0,
  // and the slots 0 of the warps behind it up to the one that ends it.
  for (int i = -1; i < kWarps; ++i) {
    const bool begun = i < 0;  // in an earlier CTA's run
    const PieceMeta head = begun ? meta[0][0] : meta[i][1];
    if (head.rows == 0) continue;
    int last = max(i, 0);
    bool ends = begun && head.ends, high = head.high;
    while (!ends && last + 1 < kWarps && meta[last + 1][0].rows > 0) ends = meta[++last][0].ends, high |= meta[last][0].high;
    if (E4 && high && tid == 0) {
      if (!begun && ends) lost = 1;
      else cuts[c].high[begun ? 0 : 1] = 1;
    }
    const int q0 = sqn[head.b] >> 5, np = last - i + (begun ? 0 : 1);  // pieces of the chain
    const int lowest = begun ? 0 : i;
    float* part = (float*)a.ws + (size_t)(2 * c + (begun ? 0 : 1)) * piece_floats(row_cap, D);
    for (int k = tid; k < head.rows * D; k += kWarps * 32) {
      const int r = k / D, d = k % D;
      const float* x = held + r * (D + 2);
      // piece j of the chain: slot 1 of its first warp unless the pair began earlier, then slots 0
      auto at = [&](int j) { return x + (size_t)(2 * (lowest + j) + (j == 0 && !begun ? 1 : 0)) * piece_floats(row_cap, D); };
      float M = -INFINITY, S = 0.f, acc = 0.f;
      for (int j = 0; j < np; ++j) M = fmaxf(M, at(j)[D]);
      for (int j = 0; j < np; ++j) {
        const float m = at(j)[D], f = m == -INFINITY ? 0.f : ex2(m - M);
        S = add_sum<E4>(S, at(j)[D + 1], m - M, f);
        acc += f * at(j)[d];
      }
      if (!begun && ends) {
        const float y = S == 0.f ? 0.f : acc / S;
        ((__nv_bfloat16*)a.out)[(int64_t)(q0 + r / G) * a.ldo + (int64_t)(head.h * G + r % G) * a.hdo + d] = __float2bfloat16_rn(y);
        if (y != y) lost = 1;
      } else {
        part[r * (D + 2) + d] = acc;
        if (d == 0) *reinterpret_cast<float2*>(part + r * (D + 2) + D) = make_float2(M, S);
      }
    }
    if (begun && ends && tid == 0) {  // the pair's last piece: find its first
      const int p0 = pre[head.b] + head.h * ((slen[head.b] + BK - 1) / BK);
      int k = min(c, (int)(((long long)p0 + 1) * grid / total));
      while (k > 0 && begin(k) > p0) --k;
      while (k + 1 < c && begin(k + 1) <= p0) ++k;
      *reinterpret_cast<int4*>(&cuts[c]) = make_int4(q0, head.h, head.rows, c - k + 1);
    }
  }
  __syncthreads();
  if (lost) {  // the lost rows of the (sequence, head)s that lie in this run, again
    for (int u = c0; u < c1;) {
      const int b = seq_of(u), nb = max(1, (slen[b] + BK - 1) / BK), h = (u - pre[b]) / nb, from = pre[b] + h * nb;
      if (from >= c0 && from + nb <= c1) {
        const int q0 = sqn[b] >> 5, n = sqn[b] & 31;
        const bool wide = E4 && wide_row(a, q0 + n - 1, h);
        for (int r = warp; r < n * G; r += kWarps) redo_if_lost<D, E4>(a, q0 + r / G, h * G + r % G, wide);
      }
      u = from + nb;
    }
  }
}

// Joins the pieces of the (sequence, KV head)s that CTAs' ends have cut, in
// order: CTA i the one that run i ends, its warps by query row, several to a
// row where there are few rows.
constexpr int kJoinWarps = 8;

template <int D, bool E4>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_decode_join_kernel(const __grid_constant__ PagedAttnArgs a,
                                                                           int row_cap) {
  constexpr int N = D / 32;
  __shared__ float part[kJoinWarps][32][N + 3];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.nq / a.pool.nkv;
  const float* ws = (const float*)a.ws;
  const int grid = gridDim.x, last = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  const Cut* cuts = (const Cut*)(ws + (size_t)2 * grid * piece_floats(row_cap, D));
  const int4 x = __ldcg(reinterpret_cast<const int4*>(cuts + last));
  const Cut cut{x.x, x.y, x.z, x.w};
  if (cut.rows == 0) return;
  bool high = false;
  if constexpr (E4) {
    for (int k = lane; k < cut.pieces; k += 32) high |= __ldcg(&cuts[last - cut.pieces + 1 + k].high[k == 0 ? 1 : 0]) != 0;
    high = __any_sync(0xffffffffu, high);
  }
  const int per = cut.rows >= kJoinWarps ? 1 : kJoinWarps / cut.rows;  // warps of a row
  for (int r0 = 0; r0 < cut.rows; r0 += kJoinWarps / per) {
    const int r = r0 + warp / per, sub = warp % per;
    const bool mine = warp / per < kJoinWarps / per && r < cut.rows;
    float M = -INFINITY, L = 0.f, acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    auto add = [&](float m, float l, const float* v) {
      const float top = fmaxf(M, m);
      const float keep = M == -INFINITY ? 0.f : ex2(M - top), f = m == -INFINITY ? 0.f : ex2(m - top);
      L = add_sum<E4>(add_sum<E4>(0.f, L, M - top, keep), l, m - top, f);
      M = top;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = acc[i] * keep + f * v[i];
    };
    if (mine) {
      for (int k0 = sub; k0 < cut.pieces; k0 += 8 * per) {
        float2 ml[8];
        float v[8][N];
#pragma unroll
        for (int k = 0; k < 8; ++k) {  // eight pieces' loads in flight
          const int i = min(k0 + k * per, cut.pieces - 1);
          // the first piece is its run's slot 1, the others their runs' slot 0
          const float* q = ws + (size_t)(2 * (last - cut.pieces + 1 + i) + (i == 0 ? 1 : 0)) * piece_floats(row_cap, D) + (size_t)r * (D + 2);
          ml[k] = __ldcg(reinterpret_cast<const float2*>(q + D));
#pragma unroll
          for (int j = 0; j < N / 2; ++j) {
            const float2 y = __ldcg(reinterpret_cast<const float2*>(q + lane * N + 2 * j));
            v[k][2 * j] = y.x, v[k][2 * j + 1] = y.y;
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k0 + k * per < cut.pieces) add(ml[k].x, ml[k].y, v[k]);
      }
    }
    if (per > 1) {  // then cut.rows < kJoinWarps: one round
      if (mine && sub > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) part[warp][lane][i] = acc[i];
        part[warp][lane][N] = M;
        part[warp][lane][N + 1] = L;
      }
      __syncthreads();
      if (mine && sub == 0)
        for (int k = 1; k < per; ++k) add(part[warp + k][lane][N], part[warp + k][lane][N + 1], part[warp + k][lane]);
    }
    if (mine && sub == 0) {
      const float f = L == 0.f ? 0.f : 1.f / L;
      __nv_bfloat16* out = (__nv_bfloat16*)a.out + (int64_t)(cut.q0 + r / G) * a.ldo + (int64_t)(cut.h * G + r % G) * a.hdo + lane * N;
      float bad = 0.f;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        *reinterpret_cast<uint32_t*>(out + 2 * i) = pack2(acc[2 * i] * f, acc[2 * i + 1] * f);
        bad = fmaf(acc[2 * i] * f, 0.f, fmaf(acc[2 * i + 1] * f, 0.f, bad));
      }
      if (__any_sync(0xffffffffu, bad != 0.f) || (high && wide_row(a, cut.q0 + r / G, cut.h))) redo_row<D, E4>(a, cut.q0 + r / G, cut.h * G + r % G);
    }
  }
}

int row_cap(const PagedAttnArgs& a) {
  return (int)std::min<int64_t>(kRowsD, (int64_t)std::max(a.batch.max_new, 1) * (a.nq / a.pool.nkv));
}

// Whether a CTA's run can end inside a (sequence, head): one of at most
// 2 kSnap blocks lies within kSnap of an end everywhere.
bool may_cut(const PagedAttnArgs& a) {
  return (int64_t)a.batch.max_pages * a.pool.ps > 2 * kSnap * block_keys(a.pool.cdtype == kE4M3);
}

template <int D, bool E4, int NT>
cudaError_t launch_decode(const PagedAttnArgs& a, cudaStream_t s) {
  auto kernel = paged_decode_kernel<D, E4, NT>;
  auto bytes = [](int rows, int B) { return (size_t)(2 * kWarps * piece_floats(rows, D) + 3 * B + 1) * 4; };
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes(8 * NT, kPagedMaxBatch));
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const int rows = row_cap(a), grid = a.sms;
  PagedAttnArgs args = a;
  if (!may_cut(a)) args.ws = nullptr;
  cudaError_t e = launch_pdl(kernel, dim3(grid), dim3(kWarps * 32), bytes(rows, a.batch.B), s, args, rows);
  if (e != cudaSuccess || !may_cut(a)) return e;
  return launch_pdl(paged_decode_join_kernel<D, E4>, dim3(grid), dim3(kJoinWarps * 32), 0, s, a, rows);
}

}  // namespace

// Whether the tensor-core kernels take the batch: this one the sequences with at
// most 16 query rows per KV head, its partner, which needs tensor maps, the others.
bool paged_decode_applicable(const PagedAttnArgs& a) {
  return a.dtype == kBF16 && (a.pool.D == 64 || a.pool.D == 128) && tc_host::encoder() != nullptr;
}

size_t paged_decode_workspace(const PagedAttnArgs& a) {
  if (!may_cut(a)) return 0;
  return (size_t)a.sms * (2 * piece_floats(row_cap(a), a.pool.D) * sizeof(float) + sizeof(Cut));
}

cudaError_t launch_paged_decode(const PagedAttnArgs& a, cudaStream_t s) {
  const bool two = row_cap(a) > 8;  // one tile of 8 query rows where every such sequence fits it
  const bool e4 = a.pool.cdtype == kE4M3;
  auto go = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (e4) return two ? launch_decode<D, true, 2>(a, s) : launch_decode<D, true, 1>(a, s);
    return two ? launch_decode<D, false, 2>(a, s) : launch_decode<D, false, 1>(a, s);
  };
  return a.pool.D == 128 ? go(std::integral_constant<int, 128>()) : go(std::integral_constant<int, 64>());
}

}  // namespace mg
