// Append to a paged KV cache: per-head RMSNorm of queries and keys, rotary
// positions, and the store of keys and values into their sequence's pages, in
// one pass over the fused q/k/v rows.
//
// For token row t of sequence b, its s-th new token, with j = past + s:
//   x <- x · w / sqrt(mean(x²) + eps)                     (q, k; optional)
//   y_i = x_i cos(p, i) - x_{i+D/2} sin(p, i),  y_{i+D/2} = x_{i+D/2} cos(p, i) + x_i sin(p, i)
//   q_out[t] = y_q;  K, V of token j = y_k, x_v           (p = positions[t] or j)
// computed in fp32 and rounded once to the destination's type.
//
// e4m3 pages: the codes of a (page, head) share the scale 2^e with the least
// e that holds its largest finite magnitude, so scaling is exact and the only
// rounding is the code's own (at most 2^-4 relative above the subnormals).
// Tokens arrive over several calls: a page that already holds tokens keeps
// max(e_old, e_new), and where it grows its old codes move by 2^(e_old - e_new),
// which is exact too until they reach the subnormals.
//
// Bound: memory, T·(2 nq + 2 nkv)·D·e bytes read or written plus the codes.
// A thread holds 16 bytes of a head, a head's D / N lanes reduce its norm and
// swap rotate-half partners by shuffles, so a row is read once.  A warp takes
// one token, whose table entries stay in its registers over all heads (eight
// warps share a token where there are few); its rows are requested before the
// sequence is looked up.
// Measured: 24 ragged fp32 chunks (83 MB) 13.3 us = 6.2 TB/s; 8 x 1024 bf16
// tokens into e4m3 pages (189 MB) 52.4 us = 3.6 TB/s, where norm and rotation run
// twice, once for the page's scale, and registers spill (issue slots 60 % active,
// DRAM 42 %: neither is full); the same rows into bf16 pages 41.5 us = 5.0 TB/s,
// fp32 rows into e4m3 pages (357 MB) 81.9 us = 4.4 TB/s; 32 tokens 4.9 us, one
// token 3.1 us.
#include <math.h>

#include <algorithm>

#include "kernels.h"
#include "paged.h"

namespace mg {
namespace {

constexpr int kThreads = 256;
constexpr int kWarpsA = kThreads / 32;
constexpr int kAhead = 4;     // 16-byte vectors of a token row that a thread requests at once
// Most new tokens per sequence for which a token's CTA also stores its run of
// rows (32 sequences, 8 KV heads of 128, pages of 64: 3 tokens 7.2 us against
// 7.8 with a CTA per run, 4 tokens 8.6 against 8.0; 128 sequences 12.4 against
// 25.4, pages of 16 8.6 against 12.2; 8 tokens 14.0 against 8.9).
constexpr int kThinNew = 4;

template <typename T, int D>
struct Shape {
  static constexpr int N = 16 / sizeof(T);  // elements of a vector
  static constexpr int LPH = D / N;         // lanes of a head
  static constexpr int HPW = 32 / LPH;      // heads that a warp holds at once
  static constexpr int K = N < D / 2 ? N : D / 2;  // table entries of a vector's dims
  static_assert(LPH >= 1 && LPH <= 32, "a head lies inside a warp");
};

template <typename T>
__device__ __forceinline__ void widen(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      x[i] = __uint_as_float(w[i]);
    }
  }
}

// The sequence of token row t (-1: behind the last one) and its span, by a
// whole warp: the lanes look at the batch's ranges side by side, one round
// trip to memory for 32 sequences.
__device__ __forceinline__ int find_seq(const PagedBatch& bt, int t, int ps, SeqSpan* span) {
  const int lane = threadIdx.x & 31;
  for (int i0 = 0; i0 < bt.B; i0 += 32) {
    const int i = min(i0 + lane, bt.B - 1);
    const SeqSpan s = seq_span(bt, i, ps);
    const unsigned hit = __ballot_sync(0xffffffffu, s.ok && s.q0 <= t && t < s.q0 + s.n);
    if (hit) {
      const int at = __ffs(hit) - 1;
      span->ok = true;
      span->q0 = __shfl_sync(0xffffffffu, s.q0, at);
      span->n = __shfl_sync(0xffffffffu, s.n, at);
      span->past = __shfl_sync(0xffffffffu, s.past, at);
      return min(i0 + at, bt.B - 1);
    }
  }
  return -1;
}

// Rotary row of token row t at cache position j.
__device__ __forceinline__ int64_t rope_pos(const PagedAppendArgs& a, int t, int j) {
  int64_t pos = a.positions ? a.positions[t] : (int64_t)j;
  if (pos < 0 || pos >= a.max_pos) {
    flag_error(a.err, kErrPositionRange);
    pos = pos < 0 ? 0 : a.max_pos - 1;
  }
  return pos;
}

// The table entries of the dims at d0.
template <typename T, int D>
struct Rope {
  float c[Shape<T, D>::K], s[Shape<T, D>::K];
  __device__ __forceinline__ void load(const PagedAppendArgs& a, int64_t pos, int d0) {
    const size_t at = (size_t)pos * (D / 2) + d0 % (D / 2);
#pragma unroll
    for (int i = 0; i < Shape<T, D>::K / 4; ++i) {
      load16_f<float>(a.cos + at + 4 * i, c + 4 * i);
      load16_f<float>(a.sin + at + 4 * i, s + 4 * i);
    }
  }
};

// Norm (by the weights w, or NULL) and rotation (where `rotate`) of the N elements at dims d0 of a head; every lane of the warp
// takes part in the shuffles.
template <typename T, int D>
__device__ __forceinline__ void norm_rotate(const PagedAppendArgs& a, float* x, int d0, const void* w, bool rotate,
                                            const Rope<T, D>& rope) {
  constexpr int N = Shape<T, D>::N, LPH = Shape<T, D>::LPH, K = Shape<T, D>::K, half = D / 2;
  if (a.q_norm || a.k_norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w) {
      const float r = 1.0f / sqrtf(ss / (float)D + a.eps);
      float g[N];
      load16_f<T>((const T*)w + d0, g);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = x[i] * r * g[i];
    }
  }
  if (a.cos == nullptr) return;
  float other[N];
  if constexpr (LPH > 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) other[i] = __shfl_xor_sync(0xffffffffu, x[i], LPH / 2);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) other[i] = x[(i + N / 2) % N];
  }
  if (!rotate) return;
#pragma unroll
  for (int i = 0; i < N; ++i)
    x[i] = fmaf(x[i], rope.c[i % K], d0 + i < half ? -other[i] * rope.s[i % K] : other[i] * rope.s[i % K]);
}

// The N values at p as e4m3 codes of scale 1 / inv.
template <int N>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* x, float inv) {
  uint32_t w[N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    w[i] = to_e4m3x2(x[4 * i] * inv, x[4 * i + 1] * inv) | (to_e4m3x2(x[4 * i + 2] * inv, x[4 * i + 3] * inv) << 16);
  if constexpr (N == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
    *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// Codes of rows [0, rows) of one (page, head) times f, by `nthreads` threads
// (thread `id`): 8 codes at a time, kMove loads in flight per thread.
__device__ __forceinline__ void move_codes(uint8_t* base, int64_t kt, int D, int rows, float f, int id, int nthreads) {
  constexpr int kMove = 8;
  const int per_row = D / 8, total = rows * per_row;
  for (int i0 = id; i0 < total; i0 += nthreads * kMove) {
    uint2 v[kMove];
#pragma unroll
    for (int k = 0; k < kMove; ++k) {
      const int i = i0 + k * nthreads;
      if (i < total) v[k] = *reinterpret_cast<const uint2*>(base + (int64_t)(i / per_row) * kt + (i % per_row) * 8);
    }
#pragma unroll
    for (int k = 0; k < kMove; ++k) {
      const int i = i0 + k * nthreads;
      if (i >= total) continue;
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = from_e4m3x2((e < 2 ? v[k].x : v[k].y) >> (16 * (e & 1)));
        w[e] = to_e4m3x2(x.x * f, x.y * f);
      }
      *reinterpret_cast<uint2*>(base + (int64_t)(i / per_row) * kt + (i % per_row) * 8) =
          make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
    }
  }
}

__device__ __forceinline__ float finite_abs(float x) {
  const float m = fabsf(x);
  return m <= 3.402823466e38f ? m : 0.f;  // not an infinity, not NaN
}

// One run of rows, the new tokens of a sequence in one page, for one (head, K
// or V) of an e4m3 pool, or several where the pages are small, by a whole
// CTA: the largest magnitude of all rows gives the scale, so the rows are held
// as they were read and the norm and rotation run twice, which takes fewer
// registers than their results as fp32.  At four CTAs per SM (64 registers) part
// of the rows is spilled all the same: 216 bytes written and 468 read per thread
// with bf16 and head_dim 128, 1380 and 3012 with fp32.
template <typename T, int D>
struct RunShape {
  static constexpr int RPI = kThreads / Shape<T, D>::LPH;  // rows per round
  static constexpr int IT = RPI >= 128 ? 1 : 128 / RPI;    // rounds of a CTA: the largest page
  __host__ __device__ static constexpr int rounds(int ps) { return (ps + RPI - 1) / RPI; }  // of one unit
  // (Head, K or V)s of a CTA: four of 16-token pages, of 64-token pages one.
  __host__ __device__ static constexpr int units(int ps) { return ps >= 64 ? 1 : IT / rounds(ps) < 64 / ps ? IT / rounds(ps) : 64 / ps; }
};

// `rounds` and `IT` (the rounds of all units) are the page size's.
template <typename T, int D, int rounds, int IT>
__device__ __forceinline__ void store_run(const PagedAppendArgs& a, int slot, int u0) {
  constexpr int N = Shape<T, D>::N, LPH = Shape<T, D>::LPH, RPI = RunShape<T, D>::RPI;
  __shared__ float run_amax[IT], run_old[IT];
  const PagedPool& pool = a.pool;
  const PagedBatch& bt = a.batch;
  const int tid = threadIdx.x, lane = tid & 31, d0 = tid % LPH * N, r0 = tid / LPH;
  const int units = min(IT / rounds, 2 * pool.nkv - u0);
  // Sequence b's runs are the slots q_start[b] / ps + 2 b + r; it has at most
  // n / ps + 2 of them.  Every warp looks it up by itself, as find_seq does.
  SeqSpan sp;
  int b = -1;
  for (int i0 = 0; i0 < bt.B && b < 0; i0 += 32) {
    const int i = min(i0 + lane, bt.B - 1);
    const SeqSpan s = seq_span(bt, i, pool.ps);
    const bool in = s.ok && s.q0 / pool.ps + 2 * i <= slot && slot < (s.q0 + s.n) / pool.ps + 2 * (i + 1);
    const unsigned hit = __ballot_sync(0xffffffffu, in);
    if (hit) {
      const int at = __ffs(hit) - 1;
      b = min(i0 + at, bt.B - 1);
      sp.q0 = __shfl_sync(0xffffffffu, s.q0, at);
      sp.n = __shfl_sync(0xffffffffu, s.n, at);
      sp.past = __shfl_sync(0xffffffffu, s.past, at);
    }
  }
  if (b < 0 || sp.past < 0) return;
  const int pi = sp.past / pool.ps + slot - (sp.q0 / pool.ps + 2 * b);  // page of the sequence
  const int j0 = max(sp.past, pi * pool.ps), j1 = min(sp.past + sp.n, (pi + 1) * pool.ps);
  if (j0 >= j1) return;
  const int nr = j1 - j0, off = j0 - pi * pool.ps, t0 = sp.q0 + j0 - sp.past;
  const int page = bt.table[(int64_t)b * bt.ld + pi];
  // Round `it` is rows (it % rounds)·RPI .. of unit u0 + it / rounds.
  uint4 raw[IT];
  const T* rows = (const T*)a.qkv + (int64_t)t0 * a.ldqkv + (size_t)(a.nq + u0) * D + d0;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int u = it / rounds, r = (it - u * rounds) * RPI + r0;
    raw[it] = r < nr && u < units ? *reinterpret_cast<const uint4*>(rows + (int64_t)r * a.ldqkv + u * D) : make_uint4(0u, 0u, 0u, 0u);
  }
  if (page < 0 || page >= pool.pages) {
    if (tid == 0) flag_error(a.err, kErrPaged);
    return;
  }
  auto scale_at = [&](int u) {
    return u >= pool.nkv ? pool.vs + (int64_t)page * pool.vse + u - pool.nkv : pool.ks + (int64_t)page * pool.kse + u;
  };
  auto codes_at = [&](int u) {
    return u >= pool.nkv ? (uint8_t*)pool.v + page * pool.vp + (u - pool.nkv) * pool.vh
                         : (uint8_t*)pool.k + page * pool.kp + u * pool.kh;
  };
  if (tid < units) {
    run_amax[tid] = 0.f;
    run_old[tid] = off > 0 ? *scale_at(u0 + tid) : 0.f;
  }
  __syncthreads();
  auto value = [&](int it, float* x) {
    const int u = it / rounds, r = min((it - u * rounds) * RPI + r0, nr - 1);
    widen<T>(raw[it], x);
    if (u0 + u >= pool.nkv) return;  // values: as they are
    Rope<T, D> rope;
    if (a.cos) rope.load(a, rope_pos(a, t0 + r, j0 + r), d0);
    norm_rotate<T, D>(a, x, d0, a.k_norm, true, rope);
  };
#pragma unroll
  for (int u = 0; u < IT / rounds; ++u) {
    if (u >= units) break;  // uniform over the CTA
    float amax = 0.f;
#pragma unroll
    for (int it = u * rounds; it < (u + 1) * rounds; ++it) {
      if ((it - u * rounds) * RPI >= nr) break;
      float x[N];
      value(it, x);
#pragma unroll
      for (int i = 0; i < N; ++i) amax = fmaxf(amax, finite_abs(x[i]));
    }
    amax = warp_max(amax);
    if (lane == 0) atomicMax((int*)&run_amax[u], __float_as_int(amax));  // magnitudes order as integers
  }
  __syncthreads();
  for (int u = 0; u < units && off > 0; ++u) {
    const int e = e4m3_exp(run_amax[u]), eo = scale_exp(run_old[u]);
    if (e > eo) move_codes(codes_at(u0 + u), u0 + u >= pool.nkv ? pool.vt : pool.kt, D, off, pow2i(eo - e), tid, kThreads);
  }
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int u = it / rounds, r = (it - u * rounds) * RPI + r0;
    if ((it - u * rounds) * RPI >= nr || u >= units) continue;
    int e = e4m3_exp(run_amax[u]);
    if (off > 0) e = max(e, scale_exp(run_old[u]));
    if (r == 0 && d0 == 0) *scale_at(u0 + u) = pow2i(e);
    float x[N];
    value(it, x);
    if (r < nr) store_codes<N>(codes_at(u0 + u) + (int64_t)(off + r) * (u0 + u >= pool.nkv ? pool.vt : pool.kt) + d0, x, pow2i(-e));
  }
}

// kMode 0: the pool holds the activation type.  1: e4m3, a token's CTA also
// stores the run of rows (new tokens in one page) that it begins.  2: e4m3,
// CTAs below `tiles` store a run's units each and the others rotate the queries only.
// `per`: warps of a token (8 in mode 1).
template <typename T, int D, int kMode>
__global__ void __launch_bounds__(kThreads, kMode == 1 ? 2 : 4)
    paged_append_kernel(const __grid_constant__ PagedAppendArgs a, int tiles, int per) {
  using S = Shape<T, D>;
  constexpr int N = S::N, LPH = S::LPH, HPW = S::HPW;
  pdl_trigger();
  pdl_wait();
  const PagedPool& pool = a.pool;
  const PagedBatch& bt = a.batch;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int block = blockIdx.x;
  if (kMode == 2) {
    if (block < tiles) {
      const int units = RunShape<T, D>::units(pool.ps), per_slot = (2 * pool.nkv + units - 1) / units;
      const int slot = block / per_slot, u0 = block % per_slot * units;
      using RS = RunShape<T, D>;
      switch (pool.ps) {
        case 16: store_run<T, D, RS::rounds(16), RS::rounds(16) * RS::units(16)>(a, slot, u0); break;
        case 32: store_run<T, D, RS::rounds(32), RS::rounds(32) * RS::units(32)>(a, slot, u0); break;
        case 64: store_run<T, D, RS::rounds(64), RS::rounds(64) * RS::units(64)>(a, slot, u0); break;
        default: store_run<T, D, RS::rounds(128), RS::rounds(128) * RS::units(128)>(a, slot, u0); break;
      }
      return;
    }
    block -= tiles;
  }
  if (block == (int)gridDim.x - tiles - 1) {  // the last CTA looks the batch over: a range that does not fit may own no row
    for (int i = tid; i < bt.B; i += kThreads) {
      const SeqSpan sp = seq_span(bt, i, pool.ps);
      if (!sp.ok || (sp.n > 0 && sp.past < 0)) flag_error(a.err, kErrPaged);
    }
    return;
  }
  const int t = block * (kWarpsA / per) + warp / per, sub = warp % per;
  if (t >= bt.T) return;
  const int hl = lane % LPH, d0 = hl * N;
  // Queries (kMode 0: keys and values too): groups of HPW heads, every per-th
  // of them, kAhead at a time; the first are requested before the lookups.
  const int heads = kMode == 0 ? a.nq + 2 * pool.nkv : a.nq;
  const T* row = (const T*)a.qkv + (int64_t)t * a.ldqkv;
  uint4 raw[kAhead];
  auto request = [&](int g0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int hh = (g0 + k * per) * HPW + lane / LPH;
      raw[k] = hh < heads ? *reinterpret_cast<const uint4*>(row + (size_t)hh * D + d0) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  request(sub);
  SeqSpan sp;
  const int b = find_seq(bt, t, pool.ps, &sp);
  if (b < 0 || sp.past < 0) return;  // a row behind the last sequence, or of one that does not fit
  const int j = sp.past + t - sp.q0;
  const int pi = j / pool.ps, off = j - pi * pool.ps;
  const int page = bt.table[(int64_t)b * bt.ld + pi];
  Rope<T, D> rope;
  if (a.cos) rope.load(a, rope_pos(a, t, j), d0);
  const bool page_ok = page >= 0 && page < pool.pages;
  if (!page_ok && lane == 0) flag_error(a.err, kErrPaged);

  for (int g0 = sub; g0 * HPW < heads; g0 += kAhead * per) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if ((g0 + k * per) * HPW >= heads) break;  // uniform over the warp
      const int hh = (g0 + k * per) * HPW + lane / LPH;
      const bool is_q = hh < a.nq, is_v = hh >= a.nq + pool.nkv;
      float x[N];
      widen<T>(raw[k], x);
      norm_rotate<T, D>(a, x, d0, is_v ? nullptr : is_q ? a.q_norm : a.k_norm, !is_v, rope);
      if (hh >= heads) continue;
      if (is_q) {
        store16_f<T>((T*)a.q_out + (int64_t)t * a.ldq + (size_t)hh * D + d0, x);
      } else if (page_ok) {
        const int h = hh - a.nq - (is_v ? pool.nkv : 0);
        T* dst = is_v ? (T*)pool.v + page * pool.vp + h * pool.vh + off * pool.vt
                      : (T*)pool.k + page * pool.kp + h * pool.kh + off * pool.kt;
        store16_f<T>(dst + d0, x);
      }
    }
    if ((g0 + kAhead * per) * HPW < heads) request(g0 + kAhead * per);
  }
  if constexpr (kMode == 1) {
    // A run begins at the sequence's first new token and at each page's start.
    if (!page_ok || (t != sp.q0 && off != 0)) return;
    const int nr = min(min(sp.n - (t - sp.q0), pool.ps - off), kThinNew);
    for (int u0 = warp * HPW; u0 < 2 * pool.nkv; u0 += kWarpsA * HPW) {  // units: (head, K or V)
      const int u = u0 + lane / LPH;
      const bool valid = u < 2 * pool.nkv;
      const bool is_v = valid && u >= pool.nkv;
      const int h = is_v ? u - pool.nkv : u;
      uint4 rw[kThinNew];
#pragma unroll
      for (int r = 0; r < kThinNew; ++r)
        rw[r] = valid && r < nr ? *reinterpret_cast<const uint4*>(row + (int64_t)r * a.ldqkv + (size_t)(a.nq + u) * D + d0)
                                : make_uint4(0u, 0u, 0u, 0u);
      float* sc = is_v ? pool.vs + (int64_t)page * pool.vse + h : pool.ks + (int64_t)page * pool.kse + h;
      const float old = valid && off > 0 ? *sc : 0.f;
      auto value = [&](int r, float* x) {
        widen<T>(rw[r], x);
        Rope<T, D> at = rope;
        if (a.cos && r > 0) at.load(a, rope_pos(a, t + r, j + r), d0);
        norm_rotate<T, D>(a, x, d0, valid && !is_v ? a.k_norm : nullptr, valid && !is_v, at);
      };
      float amax = 0.f;
#pragma unroll
      for (int r = 0; r < kThinNew; ++r) {
        if (r >= nr) break;  // uniform over the CTA
        float x[N];
        value(r, x);
#pragma unroll
        for (int i = 0; i < N; ++i) amax = fmaxf(amax, finite_abs(x[i]));
      }
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      __syncwarp();  // every lane has read the old scale
      int e = e4m3_exp(amax);
      uint8_t* base = is_v ? (uint8_t*)pool.v + page * pool.vp + h * pool.vh
                           : (uint8_t*)pool.k + page * pool.kp + h * pool.kh;
      const int64_t ts = is_v ? pool.vt : pool.kt;
      int shift = 0;
      if (valid && off > 0) {
        const int eo = scale_exp(old);
        if (e > eo) shift = eo - e;
        e = max(e, eo);
      }
      // Where a scale grew, the whole warp moves that unit's old codes.
      for (unsigned grew = __ballot_sync(0xffffffffu, shift != 0 && hl == 0); grew; grew &= grew - 1) {
        const int src = __ffs(grew) - 1;
        uint8_t* bs = (uint8_t*)__shfl_sync(0xffffffffu, (unsigned long long)base, src);
        const int64_t st = (int64_t)__shfl_sync(0xffffffffu, (long long)ts, src);
        move_codes(bs, st, D, off, pow2i(__shfl_sync(0xffffffffu, shift, src)), lane, 32);
      }
      if (valid && hl == 0) *sc = pow2i(e);
      const float inv = pow2i(-e);
#pragma unroll
      for (int r = 0; r < kThinNew; ++r) {
        if (r >= nr) break;
        float x[N];
        value(r, x);
        if (valid) store_codes<N>(base + (int64_t)(off + r) * ts + d0, x, inv);
      }
    }
  }
}

template <typename T, int D>
cudaError_t launch_d(const PagedAppendArgs& a, cudaStream_t s) {
  const int rows = a.batch.T;
  // As many warps per token as 16 warps per SM allow (32 rows: 8, 1000 rows: 2
  // warps were fastest of 1, 2, 4 and 8).
  int per = kWarpsA;
  while (per > 1 && (int64_t)rows * per > 16 * usable_sms()) per /= 2;
  const int blocks = (rows + kWarpsA / per - 1) / (kWarpsA / per) + 1;
  if (a.pool.cdtype != kE4M3)
    return launch_pdl(paged_append_kernel<T, D, 0>, dim3(blocks), dim3(kThreads), 0, s, a, 0, per);
  if (a.batch.max_new <= kThinNew)
    return launch_pdl(paged_append_kernel<T, D, 1>, dim3(rows + 1), dim3(kThreads), 0, s, a, 0, kWarpsA);
  const int units = RunShape<T, D>::units(a.pool.ps);
  const int64_t tiles = (int64_t)(rows / a.pool.ps + 2 * a.batch.B) * ((2 * a.pool.nkv + units - 1) / units);
  if (tiles + blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_pdl(paged_append_kernel<T, D, 2>, dim3((unsigned)(tiles + blocks)), dim3(kThreads), 0, s, a, (int)tiles, per);
}

template <typename T>
cudaError_t launch_t(const PagedAppendArgs& a, cudaStream_t s) {
  switch (a.pool.D) {
    case 8: return launch_d<T, 8>(a, s);
    case 16: return launch_d<T, 16>(a, s);
    case 32: return launch_d<T, 32>(a, s);
    case 64: return launch_d<T, 64>(a, s);
    case 128: return launch_d<T, 128>(a, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendArgs& a, cudaStream_t s) {
  if (a.batch.T == 0 || a.batch.B == 0) return cudaSuccess;
  const cudaError_t e = a.dtype == kBF16 ? launch_t<__nv_bfloat16>(a, s) : launch_t<float>(a, s);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace mg
