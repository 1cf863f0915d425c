// Attention over a paged KV cache for sequences that bring many tokens
// (prompts and prompt chunks; more than 16 query rows per KV head), on
// tcgen05.  bf16 activations, head_dim 64 or 128, pages in bf16 or e4m3.
//
// A query tile is 128 / G tokens x the G query heads that share a KV head
// (row r = token r / G, head r % G); an item is two adjacent tiles of one
// (sequence, head), which share every key and value chunk they both see, and
// a unit is an item's 128-key chunk.  Persistent CTAs (one per SM) count the
// batch's units from the lengths on the device and take equal contiguous
// runs, so chunks of long contexts fill the GPU however few items they make;
// an item that a run's end cuts leaves (max, sum, O) of its rows in the
// workspace, and a second kernel joins the pieces in order.
//
// Warp roles:
//   * softmax (8 warps per tile): two threads per query row (its TMEM lane),
//     half of the chunk's keys each; they exchange maxima through shared
//     memory.  Online softmax in base 2; the maximum moves only when a row's
//     scores outgrow it by 2^8, and only then is the row of O in TMEM rescaled.
//     P goes back into TMEM over the scores.  The time from scores to P is
//     what a tile waits for, with one thread per row twice as long.
//   * MMA issuer: S_X = Q_X·Kᵀ and O_X += P_X·V per tile X, ping-ponging, P
//     read from TMEM, V read MN-major.
//   * producer: the tiles' query rows by 3-D TMA over {dim, head, token}; the
//     chunks' keys and values, each with a ring of its own (keys are free for
//     the next chunk long before values), by 4-D TMA over the pages, looked up
//     four chunks at a time.
// e4m3 pages:
//   * Scores by fp8 MMAs straight on the codes.  Q, brought to [128, 256) per
//     row by a power of two, is the sum of two e4m3 numbers: a bf16 has eight
//     significant bits, and the nearest e4m3 leaves a remainder of at most
//     four.  That is exact for elements down to 2^-10 of the row's largest; a
//     smaller one is off by at most 2^-17 of it (the remainder is subnormal).
//   * K's scale multiplies the fp32 scores; V's scale 2^e joins the exponent:
//     P' = 2^(s + e - m + 7) in half (2^-11 relative, down to 2^-21 of the
//     largest, and within 2^-31 of it below), while the sum adds 2^(s - m) in
//     fp32 (scales far apart: kSpan).  P in e4m3 would be 2^-4, so the
//     values are not multiplied as codes: two converter warps turn them into
//     halves (exact), MN-major; rows behind the sequence become zeros.
// P is bf16 over bf16 pages (half a step: 2^-8 relative): the precision in
// which the stage's own prefill multiplies the values.
//
// Bound: the chain of a tile, whose next score product goes over the P that
// its value product reads: scores → softmax → value product → scores, some
// 4,300 cycles per chunk with two tiles in flight (2,050 of them the
// exponentials of both; the MMA pipe is 34 to 40 % busy).  Measured: chunks of
// 700 to 1024 tokens on 5 to 8 K positions (4 sequences, 32 query, 8 KV heads
// of 128) 410 us over bf16 pages, 830 TFLOP/s, 508 us over e4m3 ones; 8
// prompts of 801 to 1024 (32 query, 4 KV heads of 64) 117 us.  The softmax warps
// use all 96 registers of a thread and spill 120 to 210 bytes.
// Slower were steps of 64 keys with the next scores under the softmax (655 us
// for the bf16 chunks: twice the issue and barrier work per key), an issuing
// warp per tile (503 us), one softmax thread per row (553 us).
// Every wait is bounded (code 3 in the error word on expiry); on expiry the
// roles stop, issued loads and MMAs drain, and TMEM is freed.
#include <math.h>

#include <algorithm>

#include "kernels.h"
#include "paged_tc.cuh"

namespace mg {
namespace {

using namespace tc;
using namespace attn;
using namespace paged;
using bf16 = __nv_bfloat16;

constexpr int kChunkE = 128;     // keys of a unit
constexpr int kTile = 128;       // query rows of a tile = TMEM lanes
constexpr int kBoxE = 128 * 128; // a 128-row x 128-byte swizzled block
constexpr int kColSE = 0;        // TMEM: tile X's scores (then P) at 128·X, its output at 256 + D·X
constexpr int kColOE = 256;
constexpr int kSmemE = 227 * 1024;

// Warps of a CTA.
template <bool E4>
struct Roles {
  static constexpr int kTileWarps = 8;          // softmax warps of a tile: two threads of a query row
  static constexpr int kSoft = 2 * kTileWarps;
  static constexpr int kConv = E4 ? 2 : 0;
  static constexpr int kProducer = kSoft + kConv;
  static constexpr int kMma = kProducer + 1;
  static constexpr int kThreads = 32 * (kMma + 1);
};

template <int D, bool E4>
struct ExtendLayout {
  using Row = PoolRow<D, E4>;
  static constexpr int kDB = D / 64;
  static constexpr int kQ = kDB * kBoxE;                       // one tile's query rows (e4m3: as bf16, then as two code tiles)
  static constexpr int kCodes = kChunkE * D;                   // a chunk's keys (or values, or a tile's rows) as codes
  static constexpr int kK = E4 ? kCodes : kDB * kBoxE;         // a chunk's keys
  static constexpr int kV = kDB * kBoxE;                       // a chunk's values, 16-bit
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = 2 * kQ;
  static constexpr int kOffV = kOffK + 2 * kK;
  static constexpr int kOffRaw = kOffV + 2 * kV;               // e4m3: the values' codes, two chunks
  static constexpr int kOffBar = kOffRaw + (E4 ? 2 * kCodes : 0);
  static constexpr int kOffScale = kOffBar + 256;              // [4][8] K scales, [4][8] V exponents
  static constexpr int kOffRow = kOffScale + 256;              // [2][tile][half][row] what a row's two threads exchange
  static constexpr int kOffPre = kOffRow + 2 * 2 * 2 * kTile * 4;  // [B + 1] units before a sequence
  static int bytes(int B) { return kOffPre + (B + 1 + 3) / 4 * 16 + 1024; }
};

// The tile pairs of one sequence.
struct Pairs {
  SeqSpan s;
  int tq, n_pairs;  // tokens of a tile, tile pairs
  __device__ Pairs(const SeqSpan& sp, int G) : s(sp) {
    tq = kTile / G;
    n_pairs = sp.n * G > kPagedFewRows ? (sp.n + 2 * tq - 1) / (2 * tq) : 0;
  }
  // Chunks that tile qt sees (0 for a tile past the sequence).
  __device__ int tile_chunks(int qt) const {
    if (qt * tq >= s.n) return 0;
    return (max(0, s.past + min((qt + 1) * tq, s.n)) + kChunkE - 1) / kChunkE;
  }
  __device__ int units(int j) const { return max(1, max(tile_chunks(2 * j), tile_chunks(2 * j + 1))); }
};

// Units of a sequence and KV head, by a whole warp.
__device__ __forceinline__ long long seq_units(const Pairs& p) {
  long long n = 0;
  for (int j = threadIdx.x & 31; j < p.n_pairs; j += 32) n += p.units(j);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

// Fills pre[0 .. B] (units before each sequence, saturated) with all warps of
// the CTA; pre[B] is 0 where the batch is too large to count.
__device__ __forceinline__ void count_units(const PagedAttnArgs& a, int* pre, bool report) {
  const int G = a.nq / a.pool.nkv, warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  for (int b = warp; b < a.batch.B; b += warps) {
    const SeqSpan sp = seq_span(a.batch, b, a.pool.ps);
    if (report && !sp.ok && lane == 0) flag_error(a.err, kErrPaged);
    const long long n = seq_units(Pairs(sp, G)) * a.pool.nkv;
    if (lane == 0) pre[b + 1] = (int)min(n, 0x7fffffffLL);
  }
  __syncthreads();
  if (warp == 0) {
    long long run = 0;
    for (int b0 = 0; b0 < a.batch.B; b0 += 32) {
      const int b = b0 + lane;
      long long x = b < a.batch.B ? pre[b + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      x += run;
      if (b < a.batch.B) pre[b + 1] = (int)min(x, 0x7fffffffLL);
      run = __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) {
      pre[0] = 0;
      if (run >= 0x7fffffffLL) {
        if (report) flag_error(a.err, kErrPaged);
        pre[a.batch.B] = 0;
      }
    }
  }
  __syncthreads();
}

struct RunsE {
  long long total;
  int grid;
  __device__ RunsE(long long n, int most) : total(n), grid((int)(n < most ? n : most)) {}
  __device__ int begin(int c) const { return (int)((long long)c * total / grid); }
};

// Where a unit lies: sequence, KV head, tile pair, chunk inside the item.
struct Place {
  int b, h, j, chunk;
};

// By a whole warp (all lanes get the result).
__device__ __forceinline__ Place place_of(const PagedAttnArgs& a, const int* pre, int u) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = a.batch.B;  // pre[lo] <= u < pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= u) lo = mid; else hi = mid;
  }
  const Pairs p(seq_span(a.batch, lo, a.pool.ps), a.nq / a.pool.nkv);
  const int per = (pre[lo + 1] - pre[lo]) / a.pool.nkv;
  Place r{lo, (u - pre[lo]) / per, 0, 0};
  int rem = (u - pre[lo]) % per;
  for (int j0 = 0;; j0 += 32) {
    const int n = j0 + lane < p.n_pairs ? p.units(j0 + lane) : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, x > rem);
    if (past || j0 + 32 >= p.n_pairs) {
      const int at = past ? __ffs(past) - 1 : 31;
      r.j = j0 + at;
      r.chunk = rem - __shfl_sync(0xffffffffu, x - n, at);
      return r;
    }
    rem -= __shfl_sync(0xffffffffu, x, 31);
  }
}

// The pieces of a CTA's run, one after another: item (b, h, j), its chunks
// [lo, hi) that lie in the run, and the share of them that each tile sees.
struct Walk {
  const PagedAttnArgs& a;
  const int* pre;
  int u, u1, first;
  Place at;
  Pairs p;
  int lo, hi, units, ca, cb, nch;  // ca, cb: chunks of each tile in this piece; nch: the larger
  bool whole;
  __device__ Walk(const PagedAttnArgs& args, const int* pre_, int u0, int u1_)
      : a(args), pre(pre_), u(u0), u1(u1_), first(u0), at(place_of(args, pre_, u0)),
        p(seq_span(args.batch, at.b, args.pool.ps), args.nq / args.pool.nkv) {
    set();
  }
  __device__ void set() {
    units = p.units(at.j);
    lo = at.chunk;
    hi = min(units, lo + (u1 - u));
    whole = lo == 0 && hi == units;
    ca = max(0, min(hi, p.tile_chunks(2 * at.j)) - lo);
    cb = max(0, min(hi, p.tile_chunks(2 * at.j + 1)) - lo);
    nch = max(ca, cb);
  }
  __device__ int c(int x) const { return x ? cb : ca; }
  __device__ bool done() const { return u >= u1; }
  __device__ void next() {
    u += hi - lo;
    if (u >= u1) return;
    at.chunk = 0;
    if (++at.j == p.n_pairs) {
      at.j = 0;
      if (++at.h == a.pool.nkv) {
        at.h = 0;
        do ++at.b; while (pre[at.b + 1] == pre[at.b]);
        p = Pairs(seq_span(a.batch, at.b, a.pool.ps), a.nq / a.pool.nkv);
      }
    }
    set();
  }
};

// Rows of a partial: O [256][D], then the maxima and the sums.
template <int D>
__host__ __device__ constexpr size_t partial_floats() {
  return (size_t)2 * kTile * (D + 2);
}

// What a CTA leaves for the join: the item that its run ends and earlier ones
// began, as its sequence's first token row and new tokens, its KV head and
// tile pair, and its pieces (0: there is none), this run's the last; whether a
// row of a whole item in its run came out with NaN or its pages may span too
// much; and whether its piece in slot 0 or 1 has met a high_scale.
struct CutItem {
  int q0, n, h, j, pieces, redo, high[2];
};

__device__ __forceinline__ uint64_t desc_mn(const void* p, uint32_t lbo) {
  const uint64_t addr = smem_u32(p);
  return ((addr & 0x3FFFFull) >> 4) | ((uint64_t)(lbo >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// The issuing warp runs converged, its operands the same in every lane, and
// one lane (`one`) issues: the operands then stay in uniform registers.  Inside
// a branch of one lane each product cost about 90 cycles to issue.
__device__ __forceinline__ void mma_16bit(bool one, uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"((uint32_t)one));
}
__device__ __forceinline__ void mma_ta(bool one, uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(b), "r"(idesc), "r"(acc), "r"((uint32_t)one));
}
// D (fp32) += A·Bᵀ, both e4m3 codes in shared memory, K = 32.
__device__ __forceinline__ void mma_codes(bool one, uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"((uint32_t)one));
}
__device__ __forceinline__ void commit(bool one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"((uint32_t)one)
      : "memory");
}

// Shared-memory descriptor of a K-major tile of codes: rows of 128 bytes
// swizzled over 128, or of 64 over 64; eight rows to a group (SBO).
template <int D>
__device__ __forceinline__ uint64_t desc_codes(const void* p) {
  const uint64_t addr = smem_u32(p);
  return ((addr & 0x3FFFFull) >> 4) | (1ull << 16) | ((uint64_t)(8 * D >> 4) << 32) | (1ull << 46) |
         ((D == 128 ? 2ull : 4ull) << 61);
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* tm, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(tm), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ bool warp_waits(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}

// Barrier over the (eight) softmax warps of tile x that returns the OR of
// `pred`, so that they all take the same branch afterwards.
__device__ __forceinline__ bool tile_any(int x, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.red.or.pred q, %2, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)pred), "r"(1 + x)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two fp32 operations in one instruction; a pair is two consecutive registers.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void split_pair(uint64_t p, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int D, bool E4>
__global__ void __launch_bounds__(Roles<E4>::kThreads, 1)
    paged_extend_kernel(const __grid_constant__ PoolMaps maps, const __grid_constant__ CUtensorMap tm_q,
                        const __grid_constant__ PagedAttnArgs a) {
  using L = ExtendLayout<D, E4>;
  using R = Roles<E4>;
  const PagedPool& pool = a.pool;
  const PagedBatch& bt = a.batch;
  const int G = a.nq / pool.nkv;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sq = smem + L::kOffQ;    // tile X's query rows at sq + X·kQ
  uint8_t* sk = smem + L::kOffK;    // stage s: a chunk's keys at sk + s·kK
  uint8_t* sv = smem + L::kOffV;    // its values at sv + s·kV
  uint8_t* sraw = smem + L::kOffRaw;  // e4m3: its values' codes at sraw + s·kCodes
  uint64_t* bars = (uint64_t*)(smem + L::kOffBar);
  uint64_t* kfull = bars;         // [2] a chunk's keys in shared memory
  uint64_t* kempty = bars + 2;    // [2] its score products done
  uint64_t* vfull = bars + 4;     // [2] its values in shared memory
  uint64_t* vempty = bars + 6;    // [2] its value products done
  uint64_t* sfull = bars + 8;     // [tile] scores ready in TMEM
  uint64_t* pready = bars + 10;   // [tile] P written, O rescaled
  uint64_t* odone = bars + 12;    // [tile] value product done
  uint64_t* qfull = bars + 14;    // [tile] query rows landed
  uint64_t* qempty = bars + 16;   // [tile] the piece's score products read them
  uint64_t* qconv = bars + 18;    // [tile] query rows are halves (e4m3)
  uint64_t* sready = bars + 20;   // [4] a chunk's scales written (e4m3)
  uint64_t* rfull = bars + 24;    // [2] a chunk's values as codes landed (e4m3)
  uint64_t* rempty = bars + 26;   // [2] converted
  uint64_t* drain = bars + 28;    // every MMA finished
  uint32_t* tmem_holder = (uint32_t*)(bars + 29);
  volatile int* abort_flag = (volatile int*)(tmem_holder + 1);
  volatile int* redo = abort_flag + 1;  // a row came out with NaN, or its pages may span too much
  // The scales of chunk n in slot n & 3: the keys' stage is free again before
  // the softmax of the chunk has ended, but chunk n + 4 is not converted before.
  float* sks = (float*)(smem + L::kOffScale);  // [4][8]
  int* sve = (int*)(sks + 32);                 // [4][8]
  float* srow = (float*)(smem + L::kOffRow);
  int* pre = (int*)(smem + L::kOffPre);

  // By a shuffle, so that the compiler knows a role's branch to be the same for
  // every lane (bf16 chunks on 5-8 K: 420 -> 411 us, e4m3: 518 -> 503 us).
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&kfull[s], 1);
      mbar_init(&kempty[s], 1);
      mbar_init(&vfull[s], E4 ? R::kConv : 1);
      mbar_init(&vempty[s], 1);
      mbar_init(&rfull[s], 1);
      mbar_init(&rempty[s], E4 ? R::kConv : 1);
      mbar_init(&sfull[s], 1);
      mbar_init(&pready[s], R::kTileWarps);
      mbar_init(&odone[s], 1);
      mbar_init(&qfull[s], 1);
      mbar_init(&qempty[s], 1);
      mbar_init(&qconv[s], R::kTileWarps);
    }
    for (int s = 0; s < 4; ++s) mbar_init(&sready[s], 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (E4 && threadIdx.x < 64) ((int*)sks)[threadIdx.x] = 0;  // sks and sve: finite where no page writes them
  pdl_wait();
  pdl_trigger();  // the join kernel reads, before its own wait, only what was written before this kernel
  count_units(a, pre, blockIdx.x == 0);
  const RunsE runs(pre[bt.B], (int)gridDim.x);
  const int c = blockIdx.x;
  CutItem* cut = (CutItem*)((float*)a.ws + (size_t)2 * gridDim.x * partial_floats<D>()) + c;
  if (threadIdx.x == 0) *redo = cut->pieces = cut->redo = cut->high[0] = cut->high[1] = 0;
  if (c >= runs.grid) return;
  if (warp == R::kProducer) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_holder;
  const int u0 = runs.begin(c), u1 = runs.begin(c + 1);

  int issued = 0, issued_v = 0;  // chunks whose keys, values were requested (producer)
  int qn[2] = {0, 0};     // query tiles requested (producer)
  if (warp < R::kSoft) {
    const int x = warp / R::kTileWarps, hf = (warp >> 2) & 1, q4 = warp & 3;
    const int r = q4 * 32 + lane;
    const uint32_t lanes = (uint32_t)(q4 * 32) << 16;
    const uint32_t tS = tmem + lanes + kColSE + 128 * x;
    const float scale2 = a.scale * 1.4426950408889634f;
    int n = 0;     // ring position of the piece's first chunk
    int cnt = 0;   // this tile's chunks so far (its sfull / pready / odone phases)
    int qm = 0;    // query tiles so far
    int turn = 0;  // exchanges so far: they alternate between two slots, with a barrier in each
    bool ok = true;  // of this warp; the tile's warps stop together, after a vote
    // Exchanges v with the row's other thread; false if any of the tile's warps gave up a wait.
    auto exchange = [&](float v, float& other) -> bool {
      float* slot = srow + ((turn & 1) * 2 + x) * 2 * kTile;
      ++turn;
      slot[hf * kTile + r] = v;
      const bool bad = tile_any(x, !ok);
      other = slot[(1 - hf) * kTile + r];
      return !bad;
    };
    for (Walk w(a, pre, u0, u1); !w.done() && ok; w.next()) {
      const int qt = 2 * w.at.j + x;
      const int s_tok = qt * w.p.tq + r / G;  // this row's token
      const bool valid = r / G < w.p.tq && s_tok < w.p.s.n;
      const int vis = valid ? w.p.s.past + s_tok + 1 : 0;
      const int len = w.p.s.past + w.p.s.n;
      const int nchx = w.c(x);
      float rowf = scale2;
      if (E4 && nchx > 0) {
        // The tile's rows, half a row per thread: scaled to [128, 256) and
        // split into two codes per element, over the bf16 rows (all of which
        // have been read at the exchange).
        ok = warp_waits(&qfull[x], qm & 1, a.err);
        ++qm;
        constexpr int NP = D / 16;  // 16-byte pieces of half a row
        uint8_t* tile = sq + x * L::kQ;
        uint4 v[NP];
        float amax = 0.f, other;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const int k = hf * NP + p;
          v[p] = *reinterpret_cast<const uint4*>(tile + (k >> 3) * kBoxE + r * 128 + (((k & 7) ^ (r & 7)) << 4));
          const uint32_t wv[4] = {v[p].x, v[p].y, v[p].z, v[p].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(fabsf(lo_bf16(wv[i])), fabsf(hi_bf16(wv[i]))));
        }
        if (!exchange(amax, other)) {
          ok = false;
          break;
        }
        amax = fmaxf(amax, other);
        const int sh = row_shift(amax);
        const float f = amax < INFINITY ? pow2i(sh) : NAN;  // a code would saturate an infinity
        rowf = scale2 * pow2i(-sh);
#pragma unroll
        for (int p = 0; p < NP / 2; ++p) {  // 16 elements: a 16-byte piece of codes
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 q = v[2 * p + i / 2];
            const uint32_t w0 = i % 2 ? q.z : q.x, w1 = i % 2 ? q.w : q.y;
            const float e0 = lo_bf16(w0) * f, e1 = hi_bf16(w0) * f, e2 = lo_bf16(w1) * f, e3 = hi_bf16(w1) * f;
            hi[i] = to_e4m3x2(e0, e1) | (to_e4m3x2(e2, e3) << 16);
            const float2 a01 = from_e4m3x2(hi[i]), a23 = from_e4m3x2(hi[i] >> 16);
            lo[i] = to_e4m3x2(e0 - a01.x, e1 - a01.y) | (to_e4m3x2(e2 - a23.x, e3 - a23.y) << 16);
          }
          const uint32_t at = L::Row::at(r, hf * (NP / 2) + p);
          *reinterpret_cast<uint4*>(tile + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(tile + L::kCodes + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&qconv[x]);
      }

      float m = -INFINITY, l = 0.f;  // base-2 maximum that P is taken against, sum of this thread's keys
      for (int ch = 0; ch < nchx; ++ch, ++cnt) {
        const int pos = n + ch, k0 = (w.lo + ch) * kChunkE;
        ok = warp_waits(&sfull[x], (int)(cnt & 1), a.err);
        if constexpr (E4) ok = ok && warp_waits(&sready[pos & 3], (int)(pos >> 2) & 1, a.err);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int nv = vis - k0 - 64 * hf;  // visible keys of this half chunk for this row
        float sc[64];
        tmem_ld64(tS + 64 * hf, sc);
        if (!__all_sync(0xffffffffu, nv >= 64)) {
#pragma unroll
          for (int k = 0; k < 64; ++k) sc[k] = k < nv ? sc[k] : -INFINITY;
        }
        // Score k in base 2 is sc·f + e with f > 0 and e the same for 16 keys
        // (a page's K scale and V exponent; bf16: the softmax scale and 0), so
        // the maximum is taken of the raw scores, 16 at a time.
        const int at0 = (pos & 3) * 8 + 4 * hf;
        auto factor = [&](int g) { return fmaxf(rowf * sks[at0 + g], 1.17549435e-38f); };  // never 0: -inf · 0 is NaN
        float mt = -INFINITY, other;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float v = max3(sc[16 * g], sc[16 * g + 1], sc[16 * g + 2]), y = max3(sc[16 * g + 3], sc[16 * g + 4], sc[16 * g + 5]);
          v = max3(v, sc[16 * g + 6], sc[16 * g + 7]);
          y = max3(y, sc[16 * g + 8], sc[16 * g + 9]);
          v = max3(v, sc[16 * g + 10], sc[16 * g + 11]);
          y = max3(y, sc[16 * g + 12], sc[16 * g + 13]);
          v = max3(v, sc[16 * g + 14], sc[16 * g + 15]);
          if constexpr (E4) {
            mt = fmaxf(mt, fmaf(fmaxf(v, y), factor(g), (float)sve[at0 + g]));
          } else {
            mt = max3(mt, v, y);
          }
        }
        if constexpr (!E4) mt *= scale2;
        if (!exchange(mt, other)) {
          ok = false;
          break;
        }
        mt = fmaxf(mt, other);
        float m_new = m;
        bool moved = false;
        if (m == -INFINITY) {
          m_new = mt;
        } else if (mt - m > 8.f) {
          m_new = mt;
          moved = true;
        }
        const float half = moved ? ex2((E4 ? 0.5f : 1.f) * (m - m_new)) : 1.f, alpha = E4 ? half * half : half;
        const float mb = m_new == -INFINITY ? 0.f : m_new - (E4 ? 7.f : 0.f);
        m = m_new;
        float add = 0.f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float f = E4 ? factor(g) : scale2, e = E4 ? (float)sve[at0 + g] - mb : -mb;
          const uint64_t ff = pair_of(f, f), ee = pair_of(e, e);
          uint64_t sum = 0;  // two zeros
#pragma unroll
          for (int k = 16 * g; k < 16 * g + 16; k += 2) {
            float y0, y1;
            split_pair(fma_pair(pair_of(sc[k], sc[k + 1]), ff, ee), y0, y1);
            y0 = ex2(y0);
            y1 = ex2(y1);
            sum = add_pair(sum, pair_of(y0, y1));
            sc[k / 2] = __uint_as_float(E4 ? pack_f16(y0, y1) : bf16_pair(y0, y1));
          }
          float s0, s1;
          split_pair(sum, s0, s1);
          add = E4 ? fmaf(s0 + s1, pow2i(-7 - sve[at0 + g]), add) : add + (s0 + s1);
        }
        // P over the scores, two keys per column: both threads of the row have
        // read theirs (the exchange).
        tmem_st32(tS + 32 * hf, sc);
        l = E4 ? l * half * half + add : l * alpha + add;
        // The previous value product of this tile has finished (the score
        // product just read was issued after it).
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll 1
          for (int c4 = 0; c4 < D / 64; ++c4) {
            const uint32_t tO = tmem + lanes + kColOE + D * x + (D / 2) * hf + c4 * 32;
            float o[32];
            tmem_ld32(tO, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= alpha;
            tmem_st32(tO, o);
          }
        }
        // bf16: value rows behind the sequence were not loaded (P is 0 there,
        // but 0 · NaN is not): cleared before the value products.  (A wait that
        // runs out is voted on at the next exchange.)
        if constexpr (!E4) {
          if (k0 + kChunkE > len && k0 + r >= len) {
            if (!mbar_wait(&vfull[pos & 1], (int)(pos >> 1) & 1, a.err)) *abort_flag = 1;
            uint8_t* v = sv + (pos & 1) * L::kV;
#pragma unroll
            for (int p = 0; p < D / 16; ++p) {
              const int k = hf * (D / 16) + p;
              *reinterpret_cast<uint4*>(v + (k >> 3) * kBoxE + r * 128 + (k & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&pready[x]);
      }
      if (!ok) break;
      if (nchx > 0) {
        ok = warp_waits(&odone[x], (int)((cnt - 1) & 1), a.err);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      float other;
      if (!exchange(l, other)) {
        ok = false;
        break;
      }
      l = hf == 0 ? l + other : other + l;
      {
        const float unit = E4 ? 1.f / 128.f : 1.f;
        const float f = !w.whole ? unit : l == 0.f ? 0.f : unit / l;
        bf16* out = (bf16*)a.out + (int64_t)(w.p.s.q0 + s_tok) * a.ldo + (int64_t)(w.at.h * G + r % G) * a.hdo;
        float* part = (float*)a.ws + (size_t)(2 * c + (w.lo > 0 ? 0 : 1)) * partial_floats<D>();
        const int row = x * kTile + r;
        bool bad = false;
#pragma unroll
        for (int c4 = 0; c4 < D / 64; ++c4) {
          const int d0 = (D / 2) * hf + c4 * 32;
          float o[32];
          if (nchx > 0) {
            tmem_ld32(tmem + lanes + kColOE + D * x + d0, o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            o[e] *= f;
            bad |= o[e] != o[e];
          }
          if (!w.whole && valid) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<float4*>(part + (size_t)row * D + d0 + 4 * e) =
                  make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          } else if (valid) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(out + d0 + 8 * e) =
                  make_uint4(bf16_pair(o[8 * e], o[8 * e + 1]), bf16_pair(o[8 * e + 2], o[8 * e + 3]),
                             bf16_pair(o[8 * e + 4], o[8 * e + 5]), bf16_pair(o[8 * e + 6], o[8 * e + 7]));
          }
        }
        if (w.whole && valid && bad) *redo = 1;
        if (!w.whole && valid && hf == 0) {
          part[2 * kTile * D + row] = m;
          part[2 * kTile * D + 2 * kTile + row] = l;
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      n += w.nch;
    }
    if (!ok) *abort_flag = 1;
  } else if (E4 && warp < R::kProducer) {
    // Converters: a thread takes 16 codes (piece pc of a row) of rows rr +
    // RPI·i of a chunk's values.  Eight lanes hold four pieces of two rows, so
    // that their halves go to eight different groups of banks.
    constexpr int PPR = D / 16, RPI = 32 * (E4 ? R::kConv : 2) / PPR, NI = kChunkE / RPI;
    const int cw = warp - R::kSoft;
    const int pc = D == 128 ? (lane & 3) + 4 * ((lane >> 3) & 1) : lane & 3;
    const int rr = D == 128 ? cw * 4 + ((lane >> 2) & 1) + 2 * (lane >> 4) : cw * 8 + (lane >> 2);
    // 16 codes are 32 bytes of halves: two pieces of the row's 64-dim block.
    const uint32_t from = L::Row::at(rr, pc);
    const uint32_t to0 = (pc >> 2) * kBoxE + rr * 128 + ((((pc & 3) * 2) ^ (rr & 7)) << 4), to1 = to0 ^ 16;
    int n = 0;
    bool ok = true;
    for (Walk w(a, pre, u0, u1); !w.done() && ok; w.next()) {
      const int len = w.p.s.past + w.p.s.n;
      for (int ch = 0; ch < w.nch; ++ch, ++n) {
        const int s = n & 1, left = len - (w.lo + ch) * kChunkE;  // keys from this chunk on
        ok = warp_waits(&rfull[s], (int)(n >> 1) & 1, a.err);
        if (ok && n >= 2) ok = warp_waits(&vempty[s], (int)((n >> 1) - 1) & 1, a.err);
        if (*abort_flag) ok = false;
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        const uint8_t* src = sraw + s * L::kCodes + from;
        uint8_t* dst = sv + s * L::kV;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          uint4 v = *reinterpret_cast<const uint4*>(src + i * RPI * D);  // RPI is a multiple of 8: the swizzle is the same
          if (rr + RPI * i >= left) v = make_uint4(0u, 0u, 0u, 0u);
          const uint32_t c4[4] = {v.x, v.y, v.z, v.w};
          uint32_t f[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            f[2 * k] = e4m3x2_to_f16x2(c4[k]);
            f[2 * k + 1] = e4m3x2_hi_to_f16x2(c4[k]);
          }
          *reinterpret_cast<uint4*>(dst + to0 + i * RPI * 128) = make_uint4(f[0], f[1], f[2], f[3]);
          *reinterpret_cast<uint4*>(dst + to1 + i * RPI * 128) = make_uint4(f[4], f[5], f[6], f[7]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&rempty[s]);
          mbar_arrive(&vfull[s]);
        }
      }
    }
    if (!ok) *abort_flag = 1;
  } else if (warp == R::kProducer) {
    int n = 0;
    bool ok = true;
    const int ppc = kChunkE / pool.ps;
    for (Walk w(a, pre, u0, u1); !w.done() && ok; w.next()) {
      if (w.lo > 0 && w.hi == w.units && lane == 0) {  // the last piece of a cut item
        const int start = w.u - w.lo, first = (int)((((long long)start + 1) * runs.grid - 1) / runs.total);
        *reinterpret_cast<int4*>(cut) = make_int4(w.p.s.q0, w.p.s.n, w.at.h, w.at.j);
        cut->pieces = c - first + 1;
      }
      // The tiles' query rows, once the previous piece's score products have read theirs.
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (w.c(x) == 0 || !ok) continue;
        if (lane == 0) {
          if (qn[x] > 0) ok = mbar_wait(&qempty[x], (qn[x] - 1) & 1, a.err);
          if (ok) {
            mbar_expect_tx(&qfull[x], L::kDB * 128 * G * w.p.tq);
            for (int db = 0; db < L::kDB; ++db)
              tma_load_3d(sq + x * L::kQ + db * kBoxE, &tm_q, &qfull[x], db * 64, w.at.h * G,
                          w.p.s.q0 + (2 * w.at.j + x) * w.p.tq);
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0);
        if (ok) ++qn[x];
      }
      {
        const int len = w.p.s.past + w.p.s.n;
        bool high = false;
        for (int c0 = 0; c0 < w.nch && ok; c0 += 4) {
          // Lane (j, i): page i of chunk c0 + j.
          const int i = lane & 7, cj = c0 + (lane >> 3);
          const int first = (w.lo + cj) * kChunkE + i * pool.ps;
          int keys = 0, page = -1;
          if (cj < w.nch && i < ppc && first < len) {
            keys = min(pool.ps, len - first);
            page = bt.table[(int64_t)w.at.b * bt.ld + first / pool.ps];
            if (page < 0 || page >= pool.pages) {
              flag_error(a.err, kErrPaged);
              page = -1;  // outside the pool: the box is filled with zeros
            }
          }
          float ks = 1.f, vs = 1.f;
          if (E4 && page >= 0) {
            ks = pool.ks[page * pool.kse + w.at.h];
            vs = pool.vs[page * pool.vse + w.at.h];
            high |= high_scale(vs);
          }
          const int nsl = (keys + kSlice - 1) / kSlice;
          for (int j = 0; j < 4 && c0 + j < w.nch; ++j, ++n) {
            const int s = n & 1;
            const bool mine = (lane >> 3) == j && keys > 0;
            uint32_t bytes = mine ? (uint32_t)nsl * kSlice * L::Row::kRowBytes : 0u;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) bytes += __shfl_xor_sync(0xffffffffu, bytes, o);
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {  // the chunk's keys, then its values (e4m3: their codes)
              uint64_t* full = kv == 0 ? &kfull[s] : E4 ? &rfull[s] : &vfull[s];
              uint64_t* empty = kv == 0 ? &kempty[s] : E4 ? &rempty[s] : &vempty[s];
              if (n >= 2 && lane == 0) ok = mbar_wait(empty, (int)((n >> 1) - 1) & 1, a.err);
              ok = __shfl_sync(0xffffffffu, (int)(ok && !*abort_flag), 0);
              if (!ok) break;
              if (lane == 0) mbar_expect_tx(full, bytes);
              __syncwarp();
              uint8_t* st = kv == 0 ? sk + s * L::kK : E4 ? sraw + s * L::kCodes : sv + s * L::kV;
              for (int pi = 0; pi < ppc; ++pi, st += pool.ps * L::Row::kBytes) {  // the same in every lane, one issues
                const int slices = __shfl_sync(0xffffffffu, nsl, j * 8 + pi), pg = __shfl_sync(0xffffffffu, page, j * 8 + pi);
                if (slices == 0) break;
                if (slices * kSlice >= pool.ps) {
#pragma unroll
                  for (int db = 0; db < L::Row::kBlocks; ++db)
                    if (lane == 0) tma_load_4d(st + db * kBoxE, kv ? &maps.v : &maps.k, full, db * 64, 0, w.at.h, pg);
                } else {  // the sequence's last page: its slices that hold keys
                  for (int q = 0; q < slices; ++q)
#pragma unroll
                    for (int db = 0; db < L::Row::kBlocks; ++db)
                      if (lane == 0)
                        tma_load_4d(st + q * kSlice * L::Row::kBytes + db * kBoxE, kv ? &maps.v_tail : &maps.k_tail, full, db * 64,
                                    q * kSlice, w.at.h, pg);
                }
              }
              issued += kv == 0 ? 1 : 0;
              issued_v += kv;
            }
            if (!ok) break;
            if constexpr (E4) {  // 16 keys at a time; groups behind the sequence keep what they had
              if (mine)
                for (int q = 0; q < pool.ps / 16; ++q) {
                  sks[(n & 3) * 8 + i * (pool.ps / 16) + q] = ks;
                  sve[(n & 3) * 8 + i * (pool.ps / 16) + q] = max(scale_exp(vs), kPagedMinExp);
                }
              __syncwarp();
              if (lane == 0) mbar_arrive(&sready[n & 3]);
            }
          }
        }
        if constexpr (E4) {
          if (__any_sync(0xffffffffu, high) && lane == 0) {
            if (w.whole) *redo = 1;
            else cut->high[w.lo > 0 ? 0 : 1] = 1;
          }
        }
      }
      if (*abort_flag) ok = false;
      ok = __all_sync(0xffffffffu, ok);
    }
    if (!ok) *abort_flag = 1;
  } else if (warp == R::kMma) {
    // Scores: bf16, or codes; values: bf16, or halves (MN-major).
    constexpr uint32_t kTypes = (1u << 7) | (1u << 10);
    constexpr uint32_t idS = E4 ? instr_desc(kChunkE) & ~kTypes : instr_desc(kChunkE);
    constexpr uint32_t idPV = (E4 ? instr_desc(D) & ~kTypes : instr_desc(D)) | (1u << 16);
    const bool one = lane == 0;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    int n = 0, k_seen = 0, v_seen = 0;  // ring positions whose keys, values this warp has waited for
    int cnt[2] = {0, 0}, qm[2] = {0, 0};
    bool ok = true;
    auto wait_ring = [&](uint64_t* full, int& seen, int upto) -> bool {
      for (; seen < upto; ++seen)
        if (!warp_waits(&full[seen & 1], (int)(seen >> 1) & 1, a.err)) return false;
      return true;
    };
    auto score = [&](int x, int pos) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int st = __shfl_sync(0xffffffffu, pos & 1, 0);
      const uint8_t* k = sk + st * L::kK;
      const uint8_t* q = sq + x * L::kQ;
      if constexpr (E4) {
#pragma unroll
        for (int half = 0; half < 2; ++half)  // Q's codes, then its remainders'
#pragma unroll
          for (int kd = 0; kd < D / 32; ++kd)
            mma_codes(one, tm + kColSE + 128 * x, desc_codes<D>(q + half * L::kCodes) + (uint64_t)(2 * kd),
                      desc_codes<D>(k) + (uint64_t)(2 * kd), idS, half + kd > 0 ? 1u : 0u);
      } else {
#pragma unroll
        for (int kd = 0; kd < D / 16; ++kd)
          mma_16bit(one, tm + kColSE + 128 * x, smem_desc(q + (kd >> 2) * kBoxE) + (uint64_t)((kd & 3) * 2),
                    smem_desc(k + (kd >> 2) * kBoxE) + (uint64_t)((kd & 3) * 2), idS, kd > 0 ? 1u : 0u);
      }
      commit(one, &sfull[x]);
    };
    auto value = [&](int x, int pos, bool first) -> bool {
      if (!warp_waits(&pready[x], (int)(cnt[x] & 1), a.err)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int st = __shfl_sync(0xffffffffu, pos & 1, 0);
      const uint8_t* v = sv + st * L::kV;
#pragma unroll
      for (int kk = 0; kk < kChunkE / 16; ++kk)
        mma_ta(one, tm + kColOE + D * x, tm + kColSE + 128 * x + kk * 8, desc_mn(v + kk * 16 * 128, kBoxE), idPV,
               (first && kk == 0) ? 0u : 1u);
      commit(one, &odone[x]);
      // The next score product overwrites the columns that P is read from.
      const bool done = warp_waits(&odone[x], (int)(cnt[x] & 1), a.err);
      ++cnt[x];
      return done;
    };
    for (Walk w(a, pre, u0, u1); !w.done() && ok; w.next()) {
      // The last tile that sees chunk ch frees its keys (after its score
      // product) and values (after its value product).
      auto last_of = [&](int x, int ch) { return x == (ch < w.cb ? 1 : 0); };
      if (w.nch > 0) ok = wait_ring(kfull, k_seen, n + 1);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (w.c(x) == 0 || !ok) continue;
        if (!warp_waits(E4 ? &qconv[x] : &qfull[x], qm[x] & 1, a.err)) {
          ok = false;
          continue;
        }
        score(x, n);
        if (last_of(x, 0)) commit(one, &kempty[n & 1]);
        if (w.c(x) == 1) commit(one, &qempty[x]);  // the tile's last score product
        ++qm[x];
      }
      for (int ch = 0; ch < w.nch && ok; ++ch) {
        if (!wait_ring(vfull, v_seen, n + ch + 1)) {
          ok = false;
          break;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (ch >= w.c(x) || !ok) continue;
          if (!value(x, n + ch, ch == 0) || __any_sync(0xffffffffu, *abort_flag)) {
            ok = false;
            continue;
          }
          if (last_of(x, ch)) commit(one, &vempty[(n + ch) & 1]);
          if (ch + 1 < w.c(x)) {
            if (!wait_ring(kfull, k_seen, n + ch + 2)) {
              ok = false;
              continue;
            }
            score(x, n + ch + 1);
            if (last_of(x, ch + 1)) commit(one, &kempty[(n + ch + 1) & 1]);
            if (ch + 2 == w.c(x)) commit(one, &qempty[x]);
          }
        }
      }
      n += w.nch;
      if (__any_sync(0xffffffffu, *abort_flag)) ok = false;
    }
    if (!ok) *abort_flag = 1;
    commit(one, drain);  // arrives once every MMA issued above has finished
  }

  __syncthreads();
  if (warp == R::kProducer && lane == 0 && *abort_flag) {
    // Let the loads this CTA issued land before its shared memory goes away.
    for (int i = issued > 2 ? issued - 2 : 0; i < issued; ++i) mbar_wait(&kfull[i & 1], (int)(i >> 1) & 1, a.err);
    for (int i = issued_v > 2 ? issued_v - 2 : 0; i < issued_v; ++i) mbar_wait(E4 ? &rfull[i & 1] : &vfull[i & 1], (int)(i >> 1) & 1, a.err);
    for (int x = 0; x < 2; ++x)
      if (qn[x] > 0) mbar_wait(&qfull[x], (qn[x] - 1) & 1, a.err);
  }
  if (warp == R::kMma) mbar_wait(drain, 0, a.err);
  if (threadIdx.x == 0 && *redo) cut->redo = 1;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == R::kProducer) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// Joins the pieces of cut items, in order: block (c, y) 32 of the 256 rows of
// the item that CTA c's run ends, eight lanes per row; and computes lost rows
// of its run's whole items again (here, since the first kernel's roles
// wait for one another with a limit).
template <int D, bool E4>
__global__ void __launch_bounds__(256) paged_extend_join_kernel(const __grid_constant__ PagedAttnArgs a) {
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x;
  const CutItem* cut = (const CutItem*)((const float*)a.ws + (size_t)2 * gridDim.x * partial_floats<D>()) + c;
  const int2 todo = __ldcg(reinterpret_cast<const int2*>(&cut->pieces));
  const int pieces = todo.x, G = a.nq / a.pool.nkv, tq = kTile / G;
  if (todo.y != 0) {
    extern __shared__ int pre[];
    count_units(a, pre, false);
    const RunsE runs(pre[a.batch.B], (int)gridDim.x);
    for (Walk w(a, pre, runs.begin(c), runs.begin(c + 1)); !w.done(); w.next()) {
      if (!w.whole) continue;
      const bool wide = E4 && wide_row(a, w.p.s.q0 + w.p.s.n - 1, w.at.h);
      for (int i = threadIdx.x >> 5; i < 32; i += 8) {
        const int row = blockIdx.y * 32 + i, r = row % kTile, s_tok = (2 * w.at.j + row / kTile) * tq + r / G;
        if (r / G < tq && s_tok < w.p.s.n) redo_if_lost<D, E4>(a, w.p.s.q0 + s_tok, w.at.h * G + r % G, wide);
      }
    }
  }
  if (pieces == 0) return;
  const int4 it = __ldcg(reinterpret_cast<const int4*>(cut));  // q0, n, h, j
  const int row = blockIdx.y * 32 + (threadIdx.x >> 3), d0 = (threadIdx.x & 7) * (D / 8);
  const int r = row % kTile, s_tok = (2 * it.w + row / kTile) * tq + r / G;
  const bool valid = r / G < tq && s_tok < it.y;
  if (!__any_sync(0xffffffffu, valid)) return;
  // The item's first run left it in its slot 1, the others in their slots 0.
  auto piece = [&](int k) {
    return (const float*)a.ws + (size_t)(2 * (c - pieces + 1 + k) + (k == 0 ? 1 : 0)) * partial_floats<D>();
  };
  bool high = false;
  float M = -INFINITY, L = 0.f, o[D / 8];
#pragma unroll
  for (int e = 0; e < D / 8; ++e) o[e] = 0.f;
  for (int k0 = 0; k0 < pieces; k0 += 2) {  // two pieces' loads in flight
    float m[2], l[2];
    float4 v[2][D / 32];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float* q = piece(min(k0 + k, pieces - 1));
      m[k] = __ldcg(q + 2 * kTile * D + row);
      l[k] = __ldcg(q + 2 * kTile * D + 2 * kTile + row);
      if constexpr (E4) {
        const int i = min(k0 + k, pieces - 1);
        high |= __ldcg(&(cut - pieces + 1 + i)->high[i == 0 ? 1 : 0]) != 0;
      }
#pragma unroll
      for (int e = 0; e < D / 32; ++e) v[k][e] = __ldcg(reinterpret_cast<const float4*>(q + (size_t)row * D + d0 + 4 * e));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k0 + k >= pieces) continue;
      // One that saw no key has O = 0, or NaN from values that the row does not
      // see: such a row is computed again below.
      const float top = fmaxf(M, m[k]), keep = M == -INFINITY ? 0.f : ex2(M - top);
      const float f = m[k] == -INFINITY ? 0.f : ex2(m[k] - top);
      L = add_sum<E4>(add_sum<E4>(0.f, L, M - top, keep), l[k], m[k] - top, f);
      M = top;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) {
        o[4 * e] = o[4 * e] * keep + f * v[k][e].x;
        o[4 * e + 1] = o[4 * e + 1] * keep + f * v[k][e].y;
        o[4 * e + 2] = o[4 * e + 2] * keep + f * v[k][e].z;
        o[4 * e + 3] = o[4 * e + 3] * keep + f * v[k][e].w;
      }
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  bf16* out = (bf16*)a.out + (int64_t)(it.x + s_tok) * a.ldo + (int64_t)(it.z * G + r % G) * a.hdo + d0;
  float bad = 0.f;
#pragma unroll
  for (int e = 0; e < D / 8; ++e) {
    o[e] *= inv;
    bad = fmaf(o[e], 0.f, bad);
  }
  if (valid) {
#pragma unroll
    for (int e = 0; e < D / 64; ++e)
      *reinterpret_cast<uint4*>(out + 8 * e) = make_uint4(bf16_pair(o[8 * e], o[8 * e + 1]), bf16_pair(o[8 * e + 2], o[8 * e + 3]),
                                                          bf16_pair(o[8 * e + 4], o[8 * e + 5]), bf16_pair(o[8 * e + 6], o[8 * e + 7]));
  }
  unsigned again = __ballot_sync(0xffffffffu, valid && (bad != 0.f || high)), nan = __ballot_sync(0xffffffffu, bad != 0.f);
  while (again) {  // eight lanes are a row
    const int lane = __ffs(again) - 1;
    const unsigned row_lanes = 0xffu << (lane & ~7);
    again &= ~row_lanes;
    if ((nan & row_lanes) == 0 && !wide_row(a, __shfl_sync(0xffffffffu, it.x + s_tok, lane), it.z)) continue;
    redo_row<D, E4>(a, __shfl_sync(0xffffffffu, it.x + s_tok, lane), __shfl_sync(0xffffffffu, it.z * G + r % G, lane));
  }
}

template <int D, bool E4>
cudaError_t launch_extend(const PagedAttnArgs& a, cudaStream_t s) {
  PoolMaps maps{};
  if (!pool_maps<D, E4>(&maps, a.pool)) return cudaErrorInvalidValue;
  const int G = a.nq / a.pool.nkv, tq = kTile / G;
  CUtensorMap tq_map;
  {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a.nq, (cuuint64_t)a.batch.T};
    const cuuint64_t strides[2] = {(cuuint64_t)a.hdq * 2, (cuuint64_t)a.ldq * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)tq};
    const cuuint32_t estr[3] = {1, 1, 1};
    if (tc_host::encoder()(&tq_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), dims, strides, box,
                           estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  auto kernel = paged_extend_kernel<D, E4>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemE);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const int grid = a.sms;
  cudaError_t e = launch_pdl(kernel, dim3(grid), dim3(Roles<E4>::kThreads), ExtendLayout<D, E4>::bytes(a.batch.B), s, maps,
                             tq_map, a);
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_extend_join_kernel<D, E4>, dim3(grid, 2 * kTile / 32), dim3(256), (size_t)(a.batch.B + 1) * 4, s, a);
}

}  // namespace

size_t paged_extend_workspace(const PagedAttnArgs& a) {
  return (size_t)a.sms * (2 * (a.pool.D == 128 ? partial_floats<128>() : partial_floats<64>()) * sizeof(float) + sizeof(CutItem));
}

cudaError_t launch_paged_extend(const PagedAttnArgs& a, cudaStream_t s) {
  const bool e4 = a.pool.cdtype == kE4M3;
  if (a.pool.D == 128) return e4 ? launch_extend<128, true>(a, s) : launch_extend<128, false>(a, s);
  return e4 ? launch_extend<64, true>(a, s) : launch_extend<64, false>(a, s);
}

}  // namespace mg
