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
// One thread holds 16 bytes of a head, a head's D / N lanes reduce its norm
// and swap rotate-half partners by shuffles, so a row is read once.
#include <math.h>

#include <algorithm>

#include "kernels.h"
#include "paged.h"

namespace mg {
namespace {

constexpr int kThreads = 256;
constexpr int kRowVecs = 4;   // 16-byte vectors of a token row that a thread loads before it computes
constexpr int kThinNew = 8;   // most new tokens per sequence for which a token's CTA also stores its run of rows

template <typename T, int D>
struct Shape {
  static constexpr int N = 16 / sizeof(T);  // elements of a vector
  static constexpr int LPH = D / N;         // lanes of a head
  static_assert(LPH >= 1 && LPH <= 32, "a head lies inside a warp");
};

// The sequence that token row t belongs to (-1: behind the last one).  The
// CTA's threads look at the batch's ranges side by side: one round trip to
// memory where a bisection makes log2(B).
__device__ __forceinline__ int find_seq(const PagedBatch& b, int t, int* found) {
  if (threadIdx.x == 0) *found = -1;
  __syncthreads();
  for (int i = threadIdx.x; i < b.B; i += kThreads)
    if (b.q_start[i] <= t && t < b.q_start[i + 1]) *found = i;
  __syncthreads();
  return *found;
}

// Rotary row of token row t at cache position j.
__device__ __forceinline__ int64_t rope_pos(const PagedAppendArgs& a, int t, int j) {
  int64_t pos = a.positions ? a.positions[t] : (int64_t)j;
  if (pos < 0 || pos >= a.max_pos) {
    if (a.cos) flag_error(a.err, kErrPositionRange);
    pos = pos < 0 ? 0 : a.max_pos - 1;
  }
  return pos;
}

// Norm and rotation of the N elements at dims d0.. of a head; every lane of
// the warp takes part in the shuffles.
template <typename T, int D>
__device__ __forceinline__ void norm_rotate(const PagedAppendArgs& a, float* x, int d0, const T* w, bool rotate,
                                            int64_t pos) {
  constexpr int N = Shape<T, D>::N, LPH = Shape<T, D>::LPH, half = D / 2;
  if (a.q_norm || a.k_norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w) {
      const float r = 1.0f / sqrtf(ss / (float)D + a.eps);
      float g[N];
      load16_f<T>(w + d0, g);
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
  const float* c = a.cos + (size_t)pos * half;
  const float* s = a.sin + (size_t)pos * half;
  constexpr int K = N < half ? N : half;  // table entries of these dims
  const int k0 = d0 % half;
  float cv[K], sv[K];
#pragma unroll
  for (int i = 0; i < K / 4; ++i) {
    load16_f<float>(c + k0 + 4 * i, cv + 4 * i);
    load16_f<float>(s + k0 + 4 * i, sv + 4 * i);
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    x[i] = fmaf(x[i], cv[i % K], d0 + i < half ? -other[i] * sv[i % K] : other[i] * sv[i % K]);
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

// kMode 0: the pool holds the activation type.  1: e4m3, a token's CTA also
// stores the run of rows (new tokens in one page) that it begins.  2: e4m3,
// tile CTAs store the runs and token CTAs rotate the queries only.
template <typename T, int D, int kMode>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(PagedAppendArgs a, int slots) {
  constexpr int N = Shape<T, D>::N, LPH = Shape<T, D>::LPH;
  __shared__ int found;
  __shared__ float warp_amax[kThreads / 32];
  pdl_trigger();
  pdl_wait();
  const PagedPool& pool = a.pool;
  const PagedBatch& bt = a.batch;
  const int tid = threadIdx.x;
  const int hl = tid % LPH, d0 = hl * N;
  const int nh = a.nq + 2 * pool.nkv;

  if (kMode == 2 && blockIdx.x < (unsigned)(slots * 2 * pool.nkv)) {
    // One run: (sequence, page) x (head, K or V).  Sequence b's runs are the
    // slots q_start[b] / ps + 2 b + r; it has at most n / ps + 2 of them.
    const int slot = blockIdx.x / (2 * pool.nkv), u = blockIdx.x % (2 * pool.nkv);
    const int h = u % pool.nkv;
    const bool is_v = u >= pool.nkv;
    if (tid == 0) found = -1;
    __syncthreads();
    for (int i = tid; i < bt.B; i += kThreads) {
      const int lo = bt.q_start[i] / pool.ps + 2 * i, hi = bt.q_start[i + 1] / pool.ps + 2 * (i + 1);
      if (lo <= slot && slot < hi) found = i;
    }
    __syncthreads();
    const int b = found;
    if (b < 0) return;
    const SeqSpan sp = seq_span(bt, b, pool.ps);
    if (!sp.ok || sp.past < 0) return;
    const int pi = sp.past / pool.ps + slot - (sp.q0 / pool.ps + 2 * b);  // page of the sequence
    const int j0 = max(sp.past, pi * pool.ps), j1 = min(sp.past + sp.n, (pi + 1) * pool.ps);
    if (j0 >= j1) return;
    const int page = bt.table[(int64_t)b * bt.ld + pi];
    if (page < 0 || page >= pool.pages) {
      if (tid == 0) flag_error(a.err, kErrPaged);
      return;
    }
    constexpr int RPI = kThreads / LPH;                    // rows per round
    constexpr int IT = RPI >= 128 ? 1 : 128 / RPI;         // rounds of the largest page
    const int r0 = tid / LPH, nr = j1 - j0, off = j0 - pi * pool.ps;
    float x[IT][N];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int r = it * RPI + r0;
      if (r < nr) {
        load16_f<T>((const T*)a.qkv + (int64_t)(sp.q0 + j0 - sp.past + r) * a.ldqkv + (size_t)(a.nq + u) * D + d0, x[it]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[it][i] = 0.f;
      }
    }
    float* sc = is_v ? pool.vs + (int64_t)page * pool.vse + h : pool.ks + (int64_t)page * pool.kse + h;
    const float old = off > 0 ? *sc : 0.f;
    float amax = 0.f;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      if (it * RPI >= nr) break;  // uniform over the CTA
      const int r = it * RPI + r0;
      if (!is_v) {
        const int t = sp.q0 + j0 - sp.past + (r < nr ? r : 0);
        norm_rotate<T, D>(a, x[it], d0, (const T*)a.k_norm, true, a.cos ? rope_pos(a, t, j0 + (r < nr ? r : 0)) : 0);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) amax = fmaxf(amax, finite_abs(x[it][i]));
    }
    amax = warp_max(amax);
    if ((tid & 31) == 0) warp_amax[tid >> 5] = amax;
    __syncthreads();  // also: every thread has read the old scale
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) amax = fmaxf(amax, warp_amax[w]);
    int e = e4m3_exp(amax);
    uint8_t* base = is_v ? (uint8_t*)pool.v + page * pool.vp + h * pool.vh : (uint8_t*)pool.k + page * pool.kp + h * pool.kh;
    const int64_t ts = is_v ? pool.vt : pool.kt;
    if (off > 0) {
      const int eo = scale_exp(old);
      if (e > eo) move_codes(base, ts, D, off, pow2i(eo - e), tid, kThreads);
      e = max(e, eo);
    }
    if (tid == 0) *sc = pow2i(e);
    const float inv = pow2i(-e);
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int r = it * RPI + r0;
      if (r < nr) store_codes<N>(base + (int64_t)(off + r) * ts + d0, x[it], inv);
    }
    return;
  }

  const int t = kMode == 2 ? blockIdx.x - slots * 2 * pool.nkv : blockIdx.x;
  if (t == bt.T) {  // the last CTA looks the batch over: a range that does not fit may own no CTA above
    for (int i = tid; i < bt.B; i += kThreads) {
      const SeqSpan sp = seq_span(bt, i, pool.ps);
      if (!sp.ok || (sp.n > 0 && sp.past < 0)) flag_error(a.err, kErrPaged);
    }
    return;
  }
  const int b = find_seq(bt, t, &found);
  if (b < 0) return;  // a row behind the last sequence
  const SeqSpan sp = seq_span(bt, b, pool.ps);
  if (!sp.ok || sp.past < 0) return;
  const int j = sp.past + t - sp.q0;
  const int64_t pos = a.cos ? rope_pos(a, t, j) : 0;
  const int pi = j / pool.ps, off = j - pi * pool.ps;
  const int page = bt.table[(int64_t)b * bt.ld + pi];
  const bool page_ok = page >= 0 && page < pool.pages;
  if (!page_ok && tid == 0) flag_error(a.err, kErrPaged);

  // Queries (kMode 0: keys and values too), vector by vector.
  const int vecs = (kMode == 0 ? nh : a.nq) * LPH;
  const T* row = (const T*)a.qkv + (int64_t)t * a.ldqkv;
  for (int v0 = 0; v0 < vecs; v0 += kRowVecs * kThreads) {
    float x[kRowVecs][N];
#pragma unroll
    for (int k = 0; k < kRowVecs; ++k) {
      const int v = v0 + k * kThreads + tid;
      if (v < vecs) {
        load16_f<T>(row + (size_t)v * N, x[k]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[k][i] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < kRowVecs; ++k) {
      const int v = v0 + k * kThreads + tid;
      if (v0 + k * kThreads >= vecs) break;  // uniform over the CTA
      const int hh = v / LPH;
      const bool is_q = hh < a.nq, is_v = hh >= a.nq + pool.nkv;
      norm_rotate<T, D>(a, x[k], d0, is_v ? nullptr : is_q ? (const T*)a.q_norm : (const T*)a.k_norm, !is_v, pos);
      if (v >= vecs) continue;
      if (is_q) {
        store16_f<T>((T*)a.q_out + (int64_t)t * a.ldq + (size_t)hh * D + d0, x[k]);
      } else if (page_ok) {
        const int h = hh - a.nq - (is_v ? pool.nkv : 0);
        T* dst = is_v ? (T*)pool.v + page * pool.vp + h * pool.vh + off * pool.vt
                      : (T*)pool.k + page * pool.kp + h * pool.kh + off * pool.kt;
        store16_f<T>(dst + d0, x[k]);
      }
    }
  }
  if constexpr (kMode == 1) {
    // A run begins at the sequence's first new token and at each page's start.
    if (!page_ok || (t != sp.q0 && off != 0)) return;
    const int nr = min(min(sp.n - (t - sp.q0), pool.ps - off), kThinNew);
    constexpr int UPR = kThreads / LPH;  // units (head, K or V) per round
    for (int u0 = 0; u0 < 2 * pool.nkv; u0 += UPR) {
      const int u = u0 + tid / LPH;
      const bool valid = u < 2 * pool.nkv;
      const bool is_v = valid && u >= pool.nkv;
      const int h = is_v ? u - pool.nkv : u;
      float x[kThinNew][N];
#pragma unroll
      for (int r = 0; r < kThinNew; ++r) {
        if (valid && r < nr) {
          load16_f<T>((const T*)a.qkv + (int64_t)(t + r) * a.ldqkv + (size_t)(a.nq + u) * D + d0, x[r]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) x[r][i] = 0.f;
        }
      }
      float* sc = is_v ? pool.vs + (int64_t)page * pool.vse + h : pool.ks + (int64_t)page * pool.kse + h;
      const float old = valid && off > 0 ? *sc : 0.f;
      float amax = 0.f;
#pragma unroll
      for (int r = 0; r < kThinNew; ++r) {
        if (r >= nr) break;  // uniform over the CTA
        norm_rotate<T, D>(a, x[r], d0, valid && !is_v ? (const T*)a.k_norm : nullptr, valid && !is_v,
                          a.cos ? rope_pos(a, t + r, j + r) : 0);
#pragma unroll
        for (int i = 0; i < N; ++i) amax = fmaxf(amax, finite_abs(x[r][i]));
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
        move_codes(bs, st, D, off, pow2i(__shfl_sync(0xffffffffu, shift, src)), tid & 31, 32);
      }
      if (!valid) continue;
      if (hl == 0) *sc = pow2i(e);
      const float inv = pow2i(-e);
#pragma unroll
      for (int r = 0; r < kThinNew; ++r)
        if (r < nr) store_codes<N>(base + (int64_t)(off + r) * ts + d0, x[r], inv);
    }
  }
}

template <typename T, int D>
cudaError_t launch_d(const PagedAppendArgs& a, cudaStream_t s) {
  const int T_rows = a.batch.T;
  if (a.pool.cdtype != kE4M3)
    return launch_pdl(paged_append_kernel<T, D, 0>, dim3(T_rows + 1), dim3(kThreads), 0, s, a, 0);
  if (a.batch.max_new <= kThinNew)
    return launch_pdl(paged_append_kernel<T, D, 1>, dim3(T_rows + 1), dim3(kThreads), 0, s, a, 0);
  const int slots = T_rows / a.pool.ps + 2 * a.batch.B;
  return launch_pdl(paged_append_kernel<T, D, 2>, dim3((unsigned)(slots * 2 * a.pool.nkv + T_rows + 1)), dim3(kThreads), 0,
                    s, a, slots);
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
