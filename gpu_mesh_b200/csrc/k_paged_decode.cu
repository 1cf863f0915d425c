// Attention over a paged KV cache for sequences that bring few tokens: at
// most 16 query rows (new tokens x query heads) per KV head.  bf16
// activations, head_dim 64 or 128, pages in bf16 or e4m3.
//
// The cache is read once and every byte feeds at most 32 query rows' worth of
// FLOPs, so memory is the bound.  What the kernel does about it:
//   * Work split.  The units are (sequence, KV head, 128-key chunk) of the
//     lengths as they are on the device; each persistent CTA counts them and
//     takes a contiguous run of equal length.  A run's end that lies near the
//     end of a (sequence, head) moves there; one that cuts it leaves (max,
//     sum, O) in the workspace, and a second kernel joins the pieces in order:
//     no counters to initialise, so a captured call can be replayed and its
//     result does not depend on timing.
//   * Loads.  Keys and values go from memory straight into the registers that
//     the MMAs read.  The order of the dims inside a score product is free,
//     so a thread's K fragments are 16 consecutive bytes of its keys; the
//     order of the output dims is free too, so its V fragments are D / 8
//     consecutive elements of four keys, paired by byte permutes.  Every load
//     instruction covers whole 64- or 128-byte rows whatever the page size
//     (16-token pages cost one table lookup more, not more requests), and
//     each warp has the next block's loads in flight while it computes.
//   * Compute.  Eight warps take 32-key (bf16: 16-key) blocks in turn.
//     Transposed products, so that the query rows sit on the MMA's N = 8
//     side: Sᵀ = K·Qᵀ (M = 16 keys), Oᵀ = Vᵀ·Pᵀ (M = 16 dims), fp32
//     accumulators, online softmax in base 2.
//       bf16 pages: bf16 MMAs, P split into bf16 high + low parts (2^-17).
//       e4m3 pages: codes become halves in registers (exact), Q as halves
//       scaled by a power of two per row (exact), K's scale multiplies the
//       fp32 scores.  V's scale 2^e goes into the exponent: with the running
//       maximum m of s + e, P' = 2^(s + e - m + 14) (rounded to half: 2^-11
//       relative, down to 2^-28 of the largest) weighs the raw codes, while
//       the sum adds P'·2^(-e - 14) = 2^(s - m) in fp32; out = O / l · 2^-14.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "paged_tc.cuh"

namespace mg {
namespace {

using namespace attn;
using namespace paged;

constexpr int kWarps = 8;
constexpr int kThreadsD = kWarps * 32;
constexpr int kChunkD = 128;     // keys of a unit
constexpr int kRowsD = 16;       // most query rows of a (sequence, head)
constexpr int kSnap = 4;         // units a run's end moves to end with a (sequence, head)
constexpr int kMaxPieces = 160;  // pieces of a cut pair (at most one per CTA)

// 128-key chunks of a sequence that this kernel takes (0: none, or left to
// the kernel for many tokens).
__device__ __forceinline__ int decode_chunks(const SeqSpan& s, int G) {
  if (s.n < 1 || s.n * G > kRowsD) return 0;
  const int len = s.past + s.n;
  return len > 0 ? (len + kChunkD - 1) / kChunkD : 1;  // no keys at all: one unit that writes zeros
}

// Runs of the `total` units over `grid` CTAs: equal ones, but for ends that
// lie within kSnap units of a (sequence, head)'s end and move there, which
// saves a cut (an empty run is possible then).
struct Runs {
  long long total;
  int grid;
  __device__ Runs(long long n, int most) : total(n), grid((int)(n < most ? n : most)) {}
  __device__ long long raw(int c) const { return (long long)c * total / grid; }
};

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
__global__ void __launch_bounds__(kThreadsD, 1)
    paged_decode_kernel(const __grid_constant__ PagedAttnArgs a, int merge_rows) {
  constexpr int KS = D / 16;                     // k-steps of the score MMA
  constexpr int DM = D / 16;                     // dim tiles of Oᵀ
  constexpr int SUB = E4 ? 2 : 1;                // 16-key tiles of a warp's block
  constexpr int BK = 16 * SUB;                   // keys of a block
  constexpr int KP = D * (E4 ? 1 : 2) / 64;      // 16-byte pieces of a key that a thread holds (four threads a key)
  constexpr int VW = D / 8 * (E4 ? 1 : 2) / 4;   // words of a value row that a thread holds (eight threads a key)
  using Elem = typename std::conditional<E4, uint8_t, __nv_bfloat16>::type;
  const PagedPool& pool = a.pool;
  const PagedBatch& bt = a.batch;
  const int G = a.nq / pool.nkv, nkv = pool.nkv;
  extern __shared__ float smem_f[];
  float* merge = smem_f;                               // [warp][row][m, l, O(D)]
  float* fac = merge + kWarps * merge_rows * (D + 2);  // [warp][row]
  float* msum = fac + kWarps * 8;                      // [row] max, [row] sum
  int* pre = (int*)(msum + 16);                        // [B + 1] units before a sequence
  int* slen = pre + bt.B + 1;                          // [B] cached tokens
  int* sqn = slen + bt.B;                              // [B] first token row · 32 + new tokens

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  pdl_wait();
  for (int b = tid; b < bt.B; b += kThreadsD) {
    const SeqSpan s = seq_span(bt, b, pool.ps);
    if (!s.ok && blockIdx.x == 0) flag_error(a.err, kErrPaged);
    pre[b + 1] = decode_chunks(s, G);
    slen[b] = s.past + s.n;
    sqn[b] = s.q0 * 32 + (s.n & 31);
  }
  // The join kernel may start now: what it reads before its own wait was
  // written before this kernel.
  pdl_trigger();
  __syncthreads();
  if (warp == 0) {  // units before each sequence: chunks · KV heads, summed
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
      if (run >= 0x7fffffffLL) {  // 2^38 cached tokens: no pool holds them
        flag_error(a.err, kErrPaged);
        pre[bt.B] = 0;
      }
    }
  }
  __syncthreads();
  const Runs runs(pre[bt.B], (int)gridDim.x);
  const int c = blockIdx.x;
  if (c >= runs.grid) return;
  // The sequence that unit u belongs to.
  auto seq_of = [&](int u) {
    int lo = 0, hi = bt.B;  // pre[lo] <= u < pre[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= u) lo = mid; else hi = mid;
    }
    return lo;
  };
  auto begin = [&](int k) {
    const int u = (int)runs.raw(k);
    if (u >= (int)runs.total) return u;
    const int b = seq_of(u), C = max(1, (slen[b] + kChunkD - 1) / kChunkD), off = (u - pre[b]) % C;
    return off <= kSnap ? u - off : C - off <= kSnap ? u + C - off : u;
  };
  const int u0 = begin(c), u1 = begin(c + 1);
  if (u0 >= u1) return;

  // A piece of the run: the part of one (sequence, KV head) that lies in it.
  struct Piece {
    int b, h, pu, C, ue, kb, ke;  // first unit of the pair, its units, the piece's end; its blocks
  };
  auto piece_at = [&](int u) {
    Piece p;
    p.b = seq_of(u);
    const int len = slen[p.b];
    p.C = max(1, (len + kChunkD - 1) / kChunkD);
    p.h = (u - pre[p.b]) / p.C;
    p.pu = pre[p.b] + p.h * p.C;
    p.ue = min(u1, p.pu + p.C);
    p.kb = (u - p.pu) * (kChunkD / BK);
    p.ke = min((p.ue - p.pu) * (kChunkD / BK), (len + BK - 1) / BK);
    return p;
  };

  // The blocks of this warp, in order, over all pieces: `ahead` runs two
  // blocks ahead of the computation for the page lookups, one for the data.
  // Blocks are dealt to the warps in turn across pieces.
  struct Block {
    int b, h, k0, len;  // len 0: none left
    int page[SUB];
  };
  Piece ap = piece_at(u0);
  int abase = 0, ablk = ap.kb + warp;
  auto next_block = [&]() {
    Block x;
    x.len = 0;
    x.b = x.h = x.k0 = 0;
    while (ablk >= ap.ke) {
      abase = (abase + max(0, ap.ke - ap.kb)) & (kWarps - 1);
      if (ap.ue >= u1) break;
      ap = piece_at(ap.ue);
      ablk = ap.kb + ((warp - abase) & (kWarps - 1));
    }
#pragma unroll
    for (int i = 0; i < SUB; ++i) x.page[i] = -1;
    if (ablk < ap.ke) {
      x.b = ap.b;
      x.h = ap.h;
      x.k0 = ablk * BK;
      x.len = slen[ap.b];
#pragma unroll
      for (int i = 0; i < SUB; ++i)
        if (x.k0 + 16 * i < x.len) x.page[i] = __ldg(bt.table + (int64_t)x.b * bt.ld + (x.k0 + 16 * i) / pool.ps);
      ablk += kWarps;
    }
    return x;
  };
  uint4 kx[SUB][2][KP];       // keys g, g + 8 of each tile
  uint32_t vx[SUB][4][VW];    // values 2t, 2t + 1, 2t + 8, 2t + 9
  float ks[SUB], vs[SUB];
  // A block's keys (and both scales) and values: each half is requested as soon
  // as the registers of the block before are free.
  auto load_k = [&](const Block& x) {
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
      const int k0 = x.k0 + 16 * i, page = x.page[i];
      const bool some = k0 < x.len, good = page >= 0 && page < pool.pages;
      if (some && !good) flag_error(a.err, kErrPaged);  // its keys read as zeros
      const Elem* kp = (const Elem*)pool.k + (int64_t)page * pool.kp + x.h * pool.kh + (k0 % pool.ps) * pool.kt;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const bool ok = good && k0 + g + 8 * r < x.len;
#pragma unroll
        for (int p = 0; p < KP; ++p)
          kx[i][r][p] = ok ? load_once((const uint8_t*)(kp + (g + 8 * r) * pool.kt) + 64 * p + 16 * t) : make_uint4(0u, 0u, 0u, 0u);
      }
      if constexpr (E4) {
        ks[i] = some && good ? __ldg(pool.ks + (int64_t)page * pool.kse + x.h) : 0.f;
        vs[i] = some && good ? __ldg(pool.vs + (int64_t)page * pool.vse + x.h) : 1.f;
      }
    }
  };
  auto load_v = [&](const Block& x) {
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
      const int k0 = x.k0 + 16 * i, page = x.page[i];
      const bool good = page >= 0 && page < pool.pages;
      const Elem* vp = (const Elem*)pool.v + (int64_t)page * pool.vp + x.h * pool.vh + (k0 % pool.ps) * pool.vt;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = 2 * t + (r & 1) + 8 * (r >> 1);
        const bool ok = good && k0 + key < x.len;
        const uint8_t* at = (const uint8_t*)(vp + key * pool.vt) + g * (VW * 4);
        if constexpr (VW == 2) {
          const uint2 v = ok ? load_once8(at) : make_uint2(0u, 0u);
          vx[i][r][0] = v.x;
          vx[i][r][1] = v.y;
        } else {
#pragma unroll
          for (int w = 0; w < VW / 4; ++w) {
            const uint4 v = ok ? load_once(at + 16 * w) : make_uint4(0u, 0u, 0u, 0u);
            vx[i][r][4 * w] = v.x;
            vx[i][r][4 * w + 1] = v.y;
            vx[i][r][4 * w + 2] = v.z;
            vx[i][r][4 * w + 3] = v.w;
          }
        }
      }
    }
  };
  Block now = next_block(), next = next_block();
  load_k(now);
  load_v(now);

  const float scale2 = a.scale * 1.4426950408889634f;
  int base = 0;
  for (int u = u0; u < u1;) {
    const Piece p = piece_at(u);
    const int len = slen[p.b], nq_tok = sqn[p.b] & 31, rows = nq_tok * G, past = len - nq_tok;
    const bool whole = p.pu >= u0 && p.pu + p.C <= u1;
    // Thread (g, t) holds keys g, g + 8 (dims of Oᵀ by tile) for the query
    // rows 2t, 2t + 1 of each 8-row tile; vis: keys those rows see.
    int vis[NT][2];
    float mrow[NT][2], lrow[NT][2], rowf[NT][2];
    float o[NT][DM][4];
    uint32_t qb[NT][KS][2];
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
      // Row g's dims in the order of the K fragments: thread t of a key's
      // four holds 16 consecutive bytes, k-steps of four dims each.
      const int r = nt * 8 + g;
      const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + (int64_t)((sqn[p.b] >> 5) + r / G) * a.ldq +
                               (int64_t)(p.h * G + r % G) * a.hdq;
      if constexpr (E4) {
        uint4 raw[KS / 4][2];
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < KS / 4; ++i)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            raw[i][w] = r < rows ? *reinterpret_cast<const uint4*>(q + 64 * i + 16 * t + 8 * w) : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t x[4] = {raw[i][w].x, raw[i][w].y, raw[i][w].z, raw[i][w].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) amax = fmaxf(amax, fmaxf(fabsf(lo_bf16(x[k])), fabsf(hi_bf16(x[k]))));
          }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int sh = row_shift(amax);
        const float f = pow2i(sh);
#pragma unroll
        for (int i = 0; i < KS / 4; ++i)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint4 x = raw[i][w];
            qb[nt][4 * i + 2 * w][0] = pack_f16(lo_bf16(x.x) * f, hi_bf16(x.x) * f);
            qb[nt][4 * i + 2 * w][1] = pack_f16(lo_bf16(x.y) * f, hi_bf16(x.y) * f);
            qb[nt][4 * i + 2 * w + 1][0] = pack_f16(lo_bf16(x.z) * f, hi_bf16(x.z) * f);
            qb[nt][4 * i + 2 * w + 1][1] = pack_f16(lo_bf16(x.w) * f, hi_bf16(x.w) * f);
          }
        // Row g's factor is needed by the threads that hold rows 2t, 2t + 1.
#pragma unroll
        for (int e = 0; e < 2; ++e) rowf[nt][e] = scale2 * pow2i(-__shfl_sync(0xffffffffu, sh, (2 * t + e) * 4));
      } else {
#pragma unroll
        for (int i = 0; i < KS / 2; ++i) {
          const uint4 x = r < rows ? *reinterpret_cast<const uint4*>(q + 32 * i + 8 * t) : make_uint4(0u, 0u, 0u, 0u);
          qb[nt][2 * i][0] = x.x;
          qb[nt][2 * i][1] = x.y;
          qb[nt][2 * i + 1][0] = x.z;
          qb[nt][2 * i + 1][1] = x.w;
        }
      }
    }
    const int least = past + 1;  // keys that every row sees
    for (int blk = p.kb + ((warp - base) & (kWarps - 1)); blk < p.ke; blk += kWarps) {
      const int j0 = blk * BK;
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
              for (int nt = 0; nt < NT; ++nt) mma16816_f16(sc[nt][i], a0, a1, a2, a3, qb[nt][4 * q + w][0], qb[nt][4 * q + w][1]);
            }
          } else {
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816_full(sc[nt][i], x[2 * w], y[2 * w], x[2 * w + 1], y[2 * w + 1], qb[nt][2 * q + w][0], qb[nt][2 * q + w][1]);
          }
        }
      }
      float ksc[SUB];
      int ve[SUB];
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        ksc[i] = E4 ? ks[i] : 1.f;
        ve[i] = E4 ? scale_exp(vs[i]) : 0;
      }
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
            keep[e] = mrow[nt][e] == -INFINITY ? 0.f : ex2(mrow[nt][e] - mx[e]);
            mrow[nt][e] = mx[e];
            lrow[nt][e] *= keep[e];
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
            const float w = pow2i(-ve[i] - 14);
            lrow[nt][0] = fmaf(s[0] + s[2], w, lrow[nt][0]);
            lrow[nt][1] = fmaf(s[1] + s[3], w, lrow[nt][1]);
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
      next = next_block();
    }
    base = (base + max(0, p.ke - p.kb)) & (kWarps - 1);

    // End of the piece: join the warps, eight query rows at a time.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int nr = min(8, rows - nt * 8);
      if (nt > 0 && nr <= 0) break;
      float* mw = merge + warp * merge_rows * (D + 2);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = lrow[nt][e];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
        const int hh = 2 * t + e;
        if (hh < nr) {
          if (g == 0) {
            mw[hh * (D + 2)] = mrow[nt][e];
            mw[hh * (D + 2) + 1] = l;
          }
#pragma unroll
          for (int j = 0; j < DM; ++j)
            *reinterpret_cast<float2*>(&mw[hh * (D + 2) + 2 + g * (D / 8) + 2 * j]) = make_float2(o[nt][j][e], o[nt][j][2 + e]);
        }
      }
      __syncthreads();
      if (tid < nr) {
        float M = -INFINITY, S = 0.f;
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, merge[(w * merge_rows + tid) * (D + 2)]);
        for (int w = 0; w < kWarps; ++w) {
          const float mv = merge[(w * merge_rows + tid) * (D + 2)];
          const float f = mv == -INFINITY ? 0.f : ex2(mv - M);
          fac[w * 8 + tid] = f;
          S += f * merge[(w * merge_rows + tid) * (D + 2) + 1];
        }
        msum[tid] = M;
        msum[8 + tid] = S;
      }
      __syncthreads();
      float* part = (float*)a.ws + (size_t)(2 * c + (p.pu < u0 ? 0 : 1)) * kRowsD * (D + 2);
      for (int i = tid; i < nr * D; i += kThreadsD) {
        const int hh = i / D, d = i % D, r = nt * 8 + hh;
        float acc = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) acc += fac[w * 8 + hh] * merge[(w * merge_rows + hh) * (D + 2) + 2 + d];
        if constexpr (E4) acc *= 1.f / 16384.f;
        if (whole) {
          const float S = msum[8 + hh];
          ((__nv_bfloat16*)a.out)[(int64_t)((sqn[p.b] >> 5) + r / G) * a.ldo + (int64_t)(p.h * G + r % G) * a.hdo + d] =
              __float2bfloat16_rn(S == 0.f ? 0.f : acc / S);
        } else {
          part[r * (D + 2) + 2 + d] = acc;
          if (d == 0) {
            part[r * (D + 2)] = msum[hh];
            part[r * (D + 2) + 1] = msum[8 + hh];
          }
        }
      }
      __syncthreads();  // the join area is rewritten
    }
    u = p.ue;
  }
}

// Joins the pieces of a (sequence, KV head) that CTA runs have cut.
template <int D>
__global__ void __launch_bounds__(128) paged_decode_join_kernel(PagedAttnArgs a, int grid) {
  __shared__ long long before_s, total_s;
  __shared__ float fac[kRowsD][kMaxPieces];
  __shared__ float sum[kRowsD];
  const PagedBatch& bt = a.batch;
  const int tid = threadIdx.x, nkv = a.pool.nkv, G = a.nq / nkv;
  const int b = blockIdx.x / nkv, h = blockIdx.x % nkv;
  pdl_trigger();
  if (tid == 0) before_s = total_s = 0;
  __syncthreads();
  // Lengths were written before the attention kernel began, which allows this
  // kernel to start only after its own wait.
  long long before = 0, total = 0;
  for (int i = tid; i < bt.B; i += 128) {
    const long long x = (long long)decode_chunks(seq_span(bt, i, a.pool.ps), G) * nkv;
    total += x;
    if (i < b) before += x;
  }
  atomicAdd((unsigned long long*)&total_s, (unsigned long long)total);
  atomicAdd((unsigned long long*)&before_s, (unsigned long long)before);
  const SeqSpan sp = seq_span(bt, b, a.pool.ps);
  const int C = decode_chunks(sp, G);
  __syncthreads();
  pdl_wait();
  if (C == 0 || total_s >= 0x7fffffffLL) return;
  const Runs runs(total_s, grid);
  // The ends of runs that cut this pair (none of them moved): c_lo + 1 .. c_hi.
  const long long p0 = before_s + (long long)h * C;
  if (C <= 2 * kSnap) return;
  int c_lo = (int)((p0 + kSnap) * runs.grid / runs.total);  // the last run that begins at p0 + kSnap or before
  while (c_lo + 1 < runs.grid && runs.raw(c_lo + 1) <= p0 + kSnap) ++c_lo;
  while (c_lo > 0 && runs.raw(c_lo) > p0 + kSnap) --c_lo;
  int c_hi = c_lo;
  while (c_hi + 1 < runs.grid && runs.raw(c_hi + 1) < p0 + C - kSnap) ++c_hi;
  if (c_lo == c_hi) return;
  const int rows = sp.n * G, np = c_hi - c_lo + 1;
  // A CTA's first pair is its slot 0 if an earlier run begins it, else slot 1.
  auto piece = [&](int k) { return (const float*)a.ws + (size_t)(2 * (c_lo + k) + (k > 0 ? 0 : 1)) * kRowsD * (D + 2); };
  for (int i = tid; i < rows * np; i += 128) fac[i / np][i % np] = __ldcg(piece(i % np) + (i / np) * (D + 2));
  __syncthreads();
  if (tid < rows) {
    float M = -INFINITY, S = 0.f;
    for (int k = 0; k < np; ++k) M = fmaxf(M, fac[tid][k]);
    for (int k = 0; k < np; ++k) {
      const float f = fac[tid][k] == -INFINITY ? 0.f : ex2(fac[tid][k] - M);
      fac[tid][k] = f;
      S += f * __ldcg(piece(k) + tid * (D + 2) + 1);
    }
    sum[tid] = S;
  }
  __syncthreads();
  for (int i = tid; i < rows * D; i += 128) {
    const int r = i / D, d = i % D;
    float acc = 0.f;
    for (int k0 = 0; k0 < np; k0 += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = k0 + k < np ? __ldcg(piece(k0 + k) + r * (D + 2) + 2 + d) : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < np) acc += fac[r][k0 + k] * v[k];
    }
    ((__nv_bfloat16*)a.out)[(int64_t)(sp.q0 + r / G) * a.ldo + (int64_t)(h * G + r % G) * a.hdo + d] =
        __float2bfloat16_rn(sum[r] == 0.f ? 0.f : acc / sum[r]);
  }
}

int decode_grid(const PagedAttnArgs& a) {
  const int64_t most = (int64_t)a.batch.B * a.pool.nkv *
                       std::max<int64_t>(1, ((int64_t)a.batch.max_pages * a.pool.ps + kChunkD - 1) / kChunkD);
  return (int)std::min<int64_t>(std::min<int64_t>(usable_sms(), kMaxPieces), most);
}

int row_cap(const PagedAttnArgs& a) {
  return (int)std::min<int64_t>(kRowsD, (int64_t)std::max(a.batch.max_new, 1) * (a.nq / a.pool.nkv));
}

template <int D, bool E4, int NT>
cudaError_t launch_decode(const PagedAttnArgs& a, cudaStream_t s) {
  auto kernel = paged_decode_kernel<D, E4, NT>;
  const int rows = std::min(8, row_cap(a));
  const size_t smem = (size_t)(kWarps * rows * (D + 2) + kWarps * 8 + 16 + 3 * a.batch.B + 1) * 4;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const size_t most = (size_t)(kWarps * 8 * (D + 2) + kWarps * 8 + 16 + 3 * kPagedMaxBatch + 1) * 4;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const int grid = decode_grid(a);
  cudaError_t e = launch_pdl(kernel, dim3(grid), dim3(kThreadsD), smem, s, a, rows);
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_decode_join_kernel<D>, dim3((unsigned)(a.batch.B * a.pool.nkv)), dim3(128), 0, s, a, grid);
}

}  // namespace

// Whether this kernel takes the sequences with at most 16 query rows per KV head.
bool paged_decode_applicable(const PagedAttnArgs& a) {
  return a.dtype == kBF16 && (a.pool.D == 64 || a.pool.D == 128) && tc_host::encoder() != nullptr;
}

size_t paged_decode_workspace(const PagedAttnArgs& a) {
  return (size_t)2 * decode_grid(a) * kRowsD * (a.pool.D + 2) * sizeof(float);
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
