// Attention over a paged KV cache for sequences that bring few tokens: at
// most 16 query rows (new tokens x query heads) per KV head.  bf16
// activations, head_dim 64 or 128, pages in bf16 or e4m3.
//
// The cache is read once and every byte feeds at most 32 query rows' worth of
// FLOPs, so memory is the bound.  What the kernel does about it:
//   * Work split.  The units are (sequence, KV head, 128-key chunk) of the
//     lengths as they are on the device; each persistent CTA counts them,
//     takes an equal contiguous run, and streams it.  A (sequence, head) that
//     a run's end cuts leaves its (max, sum, O) in the workspace, and a second
//     kernel joins the pieces in order: no counters to initialise, so a
//     captured call can be replayed and its result does not depend on timing.
//   * Loads.  A producer warp looks up four chunks' pages and scales at a
//     time (lane = (chunk, page)), ahead of their use, and requests each page
//     with 4-D TMA into a ring of stages; a sequence's last page comes in
//     16-token slices, so at most 15 invisible tokens are read.
//   * Compute.  Two groups of four warps take chunks in turn, 32 keys a warp.
//     Transposed products, so that the query rows sit on the MMA's N = 8
//     side: Sᵀ = K·Qᵀ (M = 16 keys), Oᵀ = Vᵀ·Pᵀ (M = 16 dims), fp32
//     accumulators, online softmax in base 2.
//       bf16 pages: bf16 MMAs, P split into bf16 high + low parts (2^-17).
//       e4m3 pages: codes become halves in registers (exact), Q as halves
//       scaled by a power of two per row (exact), K's scale multiplies the
//       fp32 scores.  V's scale 2^e goes into the exponent: with the running
//       maximum m of s + e, P' = 2^(s + e - m + 14) (rounded to half: 2^-11
//       relative, down to 2^-28 of the largest) weighs the raw codes, while
//       the sum adds P'·2^-e-14 = 2^(s - m) in fp32; out = O / l · 2^-14.
//       ldmatrix takes two codes as one 16-bit element: the dims of a K
//       fragment come out permuted, which Q's fragments match, and V's
//       transposed fragments hold even dims in rows 0-7 and odd in 8-15.
// Every wait is bounded (code 3 in the error word on expiry); on a timeout
// the CTA stops, lets the copies it issued land and returns.
#include <math.h>

#include <algorithm>

#include "kernels.h"
#include "paged_tc.cuh"

namespace mg {
namespace {

using namespace tc;
using namespace attn;
using namespace paged;

constexpr int kWarps = 8;                     // consumer warps, in two groups that take chunks in turn
constexpr int kGroup = kWarps / 2;            // warps of a group
constexpr int kThreadsD = (kWarps + 1) * 32;  // + the producer warp
constexpr int kKeysW = 32;                    // keys per consumer warp
constexpr int kSub = kKeysW / 16;             // its 16-key tiles
constexpr int kChunkD = kGroup * kKeysW;      // keys per unit (128)
constexpr int kSnap = 4;                      // units a run's end moves to end with a (sequence, head)
constexpr int kMaxStagesD = 8;
constexpr int kSmemD = 227 * 1024;
constexpr int kRowsD = 16;                    // most query rows of a (sequence, head)
constexpr int kMaxPieces = 160;               // pieces of a cut pair (at most one per CTA)

__device__ __forceinline__ void consumers_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool consumers_any(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.red.or.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)pred)
      : "memory");
  return r != 0;
}

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

// Shared memory: `stages` ring stages (K, V, the piece's query rows, the
// scales of the chunk's pages), the warps' join area for up to eight rows at
// a time, the barriers, the sequences of the batch.  `rows` is the most query
// rows of a (sequence, head) of this launch.
template <int D, bool E4>
struct DecodeLayout {
  using Row = PoolRow<D, E4>;
  static constexpr int kKV = kChunkD * Row::kRowBytes;  // K (or V) bytes of a chunk
  static constexpr int kBlock = kChunkD * Row::kBytes;  // one box column of a chunk
  static constexpr int kScales = 64;                    // 8 K scales, 8 V exponents
  static constexpr int kBars = 2 * kMaxStagesD * 8 + 16;
  int stage, merge_rows, merge, meta;
  __host__ __device__ DecodeLayout(int rows, int B) {
    stage = (2 * kKV + rows * D * 2 + kScales + 1023) / 1024 * 1024;
    merge_rows = rows < 8 ? rows : 8;
    merge = (kWarps * merge_rows * (D + 2) + kWarps * 8 + 16) * 4;
    meta = (3 * B + 2 + 3) / 4 * 16;
  }
  __host__ __device__ int bytes(int stages) const { return stages * stage + (merge + 15) / 16 * 16 + kBars + meta + 1024; }
};

template <int D, bool E4, int NT>
__global__ void __launch_bounds__(kThreadsD, 1)
    paged_decode_kernel(const __grid_constant__ PoolMaps maps, PagedAttnArgs a, int stages, int row_cap) {
  using L = DecodeLayout<D, E4>;
  using Row = PoolRow<D, E4>;
  constexpr int KS = D / 16;  // k-steps of the score MMA
  constexpr int DM = D / 16;  // dim tiles of Oᵀ
  const PagedPool& pool = a.pool;
  const PagedBatch& bt = a.batch;
  const int G = a.nq / pool.nkv, nkv = pool.nkv;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const L lay(row_cap, bt.B);
  const int MR = lay.merge_rows;
  float* merge = (float*)(smem + stages * lay.stage);  // [warp][row][m, l, O(D)]
  float* fac = merge + kWarps * MR * (D + 2);          // [warp][row]
  float* msum = fac + kWarps * 8;                      // [row] max, [row] sum
  uint64_t* full = (uint64_t*)((uint8_t*)merge + (lay.merge + 15) / 16 * 16);
  uint64_t* empty = full + kMaxStagesD;
  volatile int* abort_flag = (volatile int*)(empty + kMaxStagesD);
  int* pre = (int*)((uint8_t*)full + L::kBars);  // [B + 1] units before a sequence
  int* slen = pre + bt.B + 1;                    // [B] cached tokens
  int* sqn = slen + bt.B;                        // [B] first token row · 32 + new tokens

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], E4 ? 2 : 1);  // the loads, and the scales
      mbar_init(&empty[s], kGroup);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
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

  if (warp == kWarps) {
    const int ppc = kChunkD / pool.ps;  // pages per chunk
    struct Fetch {
      int page, keys, b, h, chunk;
      float ks, vs;
    };
    // Lane (j, i) = (lane / 8, lane % 8): page i of the chunk of unit ub + j.
    auto fetch = [&](int ub) {
      Fetch f{-1, 0, 0, 0, 0, 0.f, 1.f};
      const int u = ub + (lane >> 3), i = lane & 7;
      if (u < u1) {
        f.b = seq_of(u);
        const int len = slen[f.b], C = max(1, (len + kChunkD - 1) / kChunkD), local = u - pre[f.b];
        f.h = local / C;
        f.chunk = local - f.h * C;
        const int first = f.chunk * kChunkD + i * pool.ps;
        if (i < ppc && first < len) {
          f.keys = min(pool.ps, len - first);
          f.page = bt.table[(int64_t)f.b * bt.ld + first / pool.ps];
        }
      }
      return f;
    };
    // Its scales, a step later: the page's number has arrived by then.
    auto fetch_scales = [&](Fetch& f) {
      if (f.keys > 0 && (f.page < 0 || f.page >= pool.pages)) {
        flag_error(a.err, kErrPaged);
        f.page = -1;  // outside the pool: the box is filled with zeros
      } else if (E4 && f.keys > 0) {
        f.ks = pool.ks[(int64_t)f.page * pool.kse + f.h];
        f.vs = pool.vs[(int64_t)f.page * pool.vse + f.h];
      }
    };
    int n = 0;
    bool stop = false;
    Fetch next = fetch(u0);
    fetch_scales(next);
    for (int ub = u0; ub < u1 && !stop; ub += 4) {
      const Fetch f = next;
      next = fetch(ub + 4);
      for (int j = 0; j < 4 && ub + j < u1; ++j, ++n) {
        const int s = n % stages;
        bool ok = true;
        if (n >= stages && lane == 0) ok = mbar_wait(&empty[s], ((n / stages) - 1) & 1, a.err);
        ok = __shfl_sync(0xffffffffu, (int)(ok && !*abort_flag), 0);
        if (!ok) {
          stop = true;
          break;
        }
        uint8_t* st = smem + s * lay.stage;
        const bool mine = (lane >> 3) == j && f.keys > 0;
        const int nsl = (f.keys + kSlice - 1) / kSlice;  // 16-token slices that hold keys
        const int src = j * 8;
        const int b = __shfl_sync(0xffffffffu, f.b, src), h = __shfl_sync(0xffffffffu, f.h, src);
        const int chunk = __shfl_sync(0xffffffffu, f.chunk, src);
        const int qn = sqn[b], rows = (qn & 31) * G;
        // The query rows come with the first chunk that each warp group sees of a piece.
        const bool with_q = chunk <= 1 || n <= 1;
        if (lane == 0) {
          const int keys = min(kChunkD, slen[b] - chunk * kChunkD);
          mbar_expect_tx(&full[s], 2u * ((max(keys, 0) + kSlice - 1) / kSlice) * kSlice * Row::kRowBytes +
                                       (with_q ? (uint32_t)rows * D * 2 : 0u));
        }
        __syncwarp();
        if (mine) {
          const int i = lane & 7;
          uint8_t* kd = st + i * pool.ps * Row::kBytes;
          if (nsl * kSlice >= pool.ps) {
#pragma unroll
            for (int db = 0; db < Row::kBlocks; ++db) {
              tma_load_4d(kd + db * L::kBlock, &maps.k, &full[s], db * 64, 0, f.h, f.page);
              tma_load_4d(kd + L::kKV + db * L::kBlock, &maps.v, &full[s], db * 64, 0, f.h, f.page);
            }
          } else {
            for (int q = 0; q < nsl; ++q)
#pragma unroll
              for (int db = 0; db < Row::kBlocks; ++db) {
                tma_load_4d(kd + q * kSlice * Row::kBytes + db * L::kBlock, &maps.k_tail, &full[s], db * 64,
                            q * kSlice, f.h, f.page);
                tma_load_4d(kd + q * kSlice * Row::kBytes + L::kKV + db * L::kBlock, &maps.v_tail, &full[s], db * 64,
                            q * kSlice, f.h, f.page);
              }
          }
        }
        if (with_q && lane < rows)
          bulk_load(st + 2 * L::kKV + L::kScales + lane * D * 2,
                    (const __nv_bfloat16*)a.q + (int64_t)((qn >> 5) + lane / G) * a.ldq + (int64_t)(h * G + lane % G) * a.hdq,
                    D * 2, &full[s]);
        if constexpr (E4) {
          if ((lane >> 3) == j) {
            ((float*)(st + 2 * L::kKV))[lane & 7] = f.ks;
            ((int*)(st + 2 * L::kKV))[8 + (lane & 7)] = scale_exp(f.vs);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
        }
      }
      fetch_scales(next);
    }
    if (*abort_flag || stop) {  // let every issued copy land before shared memory is released
      if (lane == 0) {
        *abort_flag = 1;
        for (int i = n > stages ? n - stages : 0; i < n; ++i) mbar_wait(&full[i % stages], (i / stages) & 1, a.err);
      }
    }
  } else {
    const int g = lane >> 2, t = lane & 3;
    const int grp = warp / kGroup, wk = warp % kGroup;
    const int page_shift = 31 - __clz(pool.ps);
    const float scale2 = a.scale * 1.4426950408889634f;
    int n = 0;
    bool stop = false;  // set by a vote only, so that all warps leave together
    for (int u = u0; u < u1 && !stop;) {
      const int b = seq_of(u);
      const int len = slen[b], C = max(1, (len + kChunkD - 1) / kChunkD);
      const int h = (u - pre[b]) / C, pu = pre[b] + h * C;  // the pair's first unit
      const int ue = min(u1, pu + C);
      const int nq_tok = sqn[b] & 31, rows = nq_tok * G, past = len - nq_tok;
      const bool whole = pu >= u0 && pu + C <= u1;

      // Thread (g, t) holds keys g, g + 8 (dims of Oᵀ by tile) for the query
      // rows 2t, 2t + 1 of each 8-row tile; vis: keys those rows see.
      int vis[NT][2];
      float mrow[NT][2], lrow[NT][2], rowf[NT][2];
      float o[NT][DM][4];
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
      }
      const int least = past + 1;  // keys that every row sees
      uint32_t qb[NT][KS][2];
      bool have_q = false;
      for (int uc = u; uc < ue; ++uc, ++n) {
        if ((n & 1) != grp) continue;
        const int s = n % stages;
        if (!mbar_wait(&full[s], (n / stages) & 1, a.err)) *abort_flag = 1;
        if (*abort_flag) break;  // the vote at the end of the piece stops every warp
        uint8_t* st = smem + s * lay.stage;
        if (!have_q) {
          have_q = true;
          const __nv_bfloat16* Qs = (const __nv_bfloat16*)(st + 2 * L::kKV + L::kScales);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + g;
            if constexpr (E4) {
              float amax = 0.f;
              uint2 raw[KS];
#pragma unroll
              for (int ks = 0; ks < KS; ++ks) {
                raw[ks] = r < rows ? *reinterpret_cast<const uint2*>(Qs + r * D + 16 * ks + 4 * t) : make_uint2(0u, 0u);
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(lo_bf16(raw[ks].x)), fabsf(hi_bf16(raw[ks].x))),
                                         fmaxf(fabsf(lo_bf16(raw[ks].y)), fabsf(hi_bf16(raw[ks].y)))));
              }
              amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
              amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
              const int sh = row_shift(amax);
              const float f = pow2i(sh);
#pragma unroll
              for (int ks = 0; ks < KS; ++ks) {
                qb[nt][ks][0] = pack_f16(lo_bf16(raw[ks].x) * f, hi_bf16(raw[ks].x) * f);
                qb[nt][ks][1] = pack_f16(lo_bf16(raw[ks].y) * f, hi_bf16(raw[ks].y) * f);
              }
              // Row g's factor is needed by the threads that hold rows 2t, 2t + 1.
#pragma unroll
              for (int e = 0; e < 2; ++e)
                rowf[nt][e] = scale2 * pow2i(-__shfl_sync(0xffffffffu, sh, (2 * t + e) * 4));
            } else {
#pragma unroll
              for (int ks = 0; ks < KS; ++ks) {
                qb[nt][ks][0] = r < rows ? *reinterpret_cast<const uint32_t*>(Qs + r * D + 16 * ks + 2 * t) : 0u;
                qb[nt][ks][1] = r < rows ? *reinterpret_cast<const uint32_t*>(Qs + r * D + 16 * ks + 8 + 2 * t) : 0u;
              }
            }
          }
        }
        const int j0 = (uc - pu) * kChunkD + wk * kKeysW;  // the warp's first key
        const int nk = min(kKeysW, len - j0);
        if (nk > 0) {
          float ksc[kSub];
          int ve[kSub];
#pragma unroll
          for (int u2 = 0; u2 < kSub; ++u2) {
            ksc[u2] = 1.f;
            ve[u2] = 0;
            if constexpr (E4) {
              const int pg = (wk * kKeysW + 16 * u2) >> page_shift;
              ksc[u2] = ((const float*)(st + 2 * L::kKV))[pg];
              ve[u2] = ((const int*)(st + 2 * L::kKV))[8 + pg];
            }
          }
          float sc[NT][kSub][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int u2 = 0; u2 < kSub; ++u2) sc[nt][u2][0] = sc[nt][u2][1] = sc[nt][u2][2] = sc[nt][u2][3] = 0.f;
          const uint32_t kbase = smem_u32(st);
          const int kr = wk * kKeysW + (lane & 7) + 8 * ((lane >> 3) & 1);
          if constexpr (E4) {
#pragma unroll
            for (int jj = 0; jj < KS / 2; ++jj) {
#pragma unroll
              for (int u2 = 0; u2 < kSub; ++u2) {
                uint32_t x[4];
                ldsm_x4(kbase + Row::at(kr + 16 * u2, 2 * jj + (lane >> 4)), x);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint32_t a0 = e4m3x2_to_f16x2(x[2 * e]), a1 = e4m3x2_to_f16x2(x[2 * e + 1]);
                  const uint32_t a2 = e4m3x2_hi_to_f16x2(x[2 * e]), a3 = e4m3x2_hi_to_f16x2(x[2 * e + 1]);
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
                    mma16816_f16(sc[nt][u2], a0, a1, a2, a3, qb[nt][2 * jj + e][0], qb[nt][2 * jj + e][1]);
                }
              }
            }
          } else {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              const int cc = 2 * ks + (lane >> 4);
#pragma unroll
              for (int u2 = 0; u2 < kSub; ++u2) {
                uint32_t x[4];
                ldsm_x4(kbase + (cc >> 3) * L::kBlock + Row::at(kr + 16 * u2, cc & 7), x);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma16816_full(sc[nt][u2], x[0], x[1], x[2], x[3], qb[nt][ks][0], qb[nt][ks][1]);
              }
            }
          }
          // Online softmax per query row (column): keys g (c0, c1), g + 8 (c2, c3) of each tile.
          uint32_t ph[NT][kSub][2], plo[NT][kSub][2];
          const bool clear = j0 + kKeysW <= least;  // every key of the warp is visible to every row
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float mx[2] = {mrow[nt][0], mrow[nt][1]};
#pragma unroll
            for (int u2 = 0; u2 < kSub; ++u2) {
              float* p = sc[nt][u2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float f = rowf[nt][e] * ksc[u2];
                p[e] = E4 ? fmaf(p[e], f, (float)ve[u2]) : p[e] * f;
                p[2 + e] = E4 ? fmaf(p[2 + e], f, (float)ve[u2]) : p[2 + e] * f;
                if (!clear) {
                  p[e] = j0 + 16 * u2 + g < vis[nt][e] ? p[e] : -INFINITY;
                  p[2 + e] = j0 + 16 * u2 + g + 8 < vis[nt][e] ? p[2 + e] : -INFINITY;
                }
                mx[e] = fmaxf(mx[e], fmaxf(p[e], p[2 + e]));
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
            for (int u2 = 0; u2 < kSub; ++u2) {
              float* p = sc[nt][u2];
              p[0] = ex2(p[0] - base0);
              p[1] = ex2(p[1] - base1);
              p[2] = ex2(p[2] - base0);
              p[3] = ex2(p[3] - base1);
              if constexpr (E4) {
                const float w = pow2i(-ve[u2] - 14);
                lrow[nt][0] = fmaf(p[0] + p[2], w, lrow[nt][0]);
                lrow[nt][1] = fmaf(p[1] + p[3], w, lrow[nt][1]);
                // Pᵀ as the B operand of Oᵀ += Vᵀ·Pᵀ: an 8x8 (keys x rows) matrix each, transposed in registers.
                ph[nt][u2][0] = movm_trans(pack_f16(p[0], p[1]));
                ph[nt][u2][1] = movm_trans(pack_f16(p[2], p[3]));
              } else {
                lrow[nt][0] += p[0] + p[2];
                lrow[nt][1] += p[1] + p[3];
                const uint32_t h01 = pack2(p[0], p[1]), h23 = pack2(p[2], p[3]);
                ph[nt][u2][0] = movm_trans(h01);
                ph[nt][u2][1] = movm_trans(h23);
                plo[nt][u2][0] = movm_trans(pack2(p[0] - lo_bf16(h01), p[1] - hi_bf16(h01)));
                plo[nt][u2][1] = movm_trans(pack2(p[2] - lo_bf16(h23), p[3] - hi_bf16(h23)));
              }
            }
          }
          // Value rows behind the sequence can hold anything (P is 0 there,
          // but 0 · NaN is not): their halves of the fragments are cleared.
          const bool full_keys = nk == kKeysW;
          uint32_t m01[kSub], m89[kSub];
#pragma unroll
          for (int u2 = 0; u2 < kSub; ++u2) {
            const int kk = 16 * u2 + 2 * t;
            m01[u2] = (kk < nk ? 0x0000ffffu : 0u) | (kk + 1 < nk ? 0xffff0000u : 0u);
            m89[u2] = (kk + 8 < nk ? 0x0000ffffu : 0u) | (kk + 9 < nk ? 0xffff0000u : 0u);
          }
          const uint32_t vbase = smem_u32(st + L::kKV);
          if constexpr (E4) {
#pragma unroll
            for (int jj = 0; jj < DM / 2; ++jj) {
#pragma unroll
              for (int u2 = 0; u2 < kSub; ++u2) {
                uint32_t x[4];
                ldsm_x4_t(vbase + Row::at(kr + 16 * u2, 2 * jj + (lane >> 4)), x);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  // bytes (key 2t: dims 2g, 2g + 1; key 2t + 1: the same) to one key pair per dim
                  const uint32_t y0 = __byte_perm(x[2 * e], 0u, 0x3120), y1 = __byte_perm(x[2 * e + 1], 0u, 0x3120);
                  uint32_t a0 = e4m3x2_to_f16x2(y0), a1 = e4m3x2_hi_to_f16x2(y0);
                  uint32_t a2 = e4m3x2_to_f16x2(y1), a3 = e4m3x2_hi_to_f16x2(y1);
                  if (!full_keys) a0 &= m01[u2], a1 &= m01[u2], a2 &= m89[u2], a3 &= m89[u2];
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
                    mma16816_f16(o[nt][2 * jj + e], a0, a1, a2, a3, ph[nt][u2][0], ph[nt][u2][1]);
                }
              }
            }
          } else {
            const int mi = lane >> 3;
            const int vr = wk * kKeysW + (lane & 7) + 8 * (mi >> 1);
#pragma unroll
            for (int dm = 0; dm < DM; ++dm) {
              const int cc = 2 * dm + (mi & 1);
#pragma unroll
              for (int u2 = 0; u2 < kSub; ++u2) {
                uint32_t x[4];
                ldsm_x4_t(vbase + (cc >> 3) * L::kBlock + Row::at(vr + 16 * u2, cc & 7), x);
                if (!full_keys) x[0] &= m01[u2], x[1] &= m01[u2], x[2] &= m89[u2], x[3] &= m89[u2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  mma16816_full(o[nt][dm], x[0], x[1], x[2], x[3], ph[nt][u2][0], ph[nt][u2][1]);
                  mma16816_full(o[nt][dm], x[0], x[1], x[2], x[3], plo[nt][u2][0], plo[nt][u2][1]);
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }

      // End of the piece: join the warps, eight query rows at a time.
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int nr = min(8, rows - nt * 8);
        if (nt > 0 && nr <= 0) break;
        float* mw = merge + warp * MR * (D + 2);
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
            for (int dm = 0; dm < DM; ++dm) {
              if constexpr (E4) {  // rows g and g + 8 of the tile are dims 2g and 2g + 1
                *reinterpret_cast<float2*>(&mw[hh * (D + 2) + 2 + 16 * dm + 2 * g]) =
                    make_float2(o[nt][dm][e], o[nt][dm][2 + e]);
              } else {
                mw[hh * (D + 2) + 2 + 16 * dm + g] = o[nt][dm][e];
                mw[hh * (D + 2) + 2 + 16 * dm + g + 8] = o[nt][dm][2 + e];
              }
            }
          }
        }
        if (consumers_any(*abort_flag)) {  // also orders the writes above
          *abort_flag = 1;
          stop = true;
          break;
        }
        if (tid < nr) {
          float M = -INFINITY, S = 0.f;
          for (int w = 0; w < kWarps; ++w) M = fmaxf(M, merge[(w * MR + tid) * (D + 2)]);
          for (int w = 0; w < kWarps; ++w) {
            const float mv = merge[(w * MR + tid) * (D + 2)];
            const float f = mv == -INFINITY ? 0.f : ex2(mv - M);
            fac[w * 8 + tid] = f;
            S += f * merge[(w * MR + tid) * (D + 2) + 1];
          }
          msum[tid] = M;
          msum[8 + tid] = S;
        }
        consumers_bar();
        float* part = (float*)a.ws + (size_t)(2 * c + (pu < u0 ? 0 : 1)) * kRowsD * (D + 2);
        for (int i = tid; i < nr * D; i += kWarps * 32) {
          const int hh = i / D, d = i % D, r = nt * 8 + hh;
          float acc = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) acc += fac[w * 8 + hh] * merge[(w * MR + hh) * (D + 2) + 2 + d];
          if constexpr (E4) acc *= 1.f / 16384.f;
          if (whole) {
            const float S = msum[8 + hh];
            ((__nv_bfloat16*)a.out)[(int64_t)((sqn[b] >> 5) + r / G) * a.ldo + (int64_t)(h * G + r % G) * a.hdo + d] =
                __float2bfloat16_rn(S == 0.f ? 0.f : acc / S);
          } else {
            part[r * (D + 2) + 2 + d] = acc;
            if (d == 0) {
              part[r * (D + 2)] = msum[hh];
              part[r * (D + 2) + 1] = msum[8 + hh];
            }
          }
        }
        consumers_bar();  // the merge area is rewritten
      }
      u = ue;
    }
  }
  __syncthreads();
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
  PoolMaps maps;
  if (!pool_maps<D, E4>(&maps, a.pool)) return cudaErrorInvalidValue;
  auto kernel = paged_decode_kernel<D, E4, NT>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemD);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const int rows = row_cap(a);
  const DecodeLayout<D, E4> lay(rows, a.batch.B);
  // An even ring: a stage always belongs to the same warp group, whose waits
  // then see every phase of its barriers.
  int stages = kMaxStagesD;
  while (stages > 2 && lay.bytes(stages) > kSmemD) stages -= 2;
  if (lay.bytes(stages) > kSmemD) return cudaErrorInvalidValue;
  const int grid = decode_grid(a);
  cudaError_t e = launch_pdl(kernel, dim3(grid), dim3(kThreadsD), lay.bytes(stages), s, maps, a, stages, rows);
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
