// Attention over a paged KV cache on the CUDA cores: every type, head size
// and group that the pool can hold, and the launch rule between this kernel
// and the tensor-core ones.
//
//   out[t, h] = Σ_j softmax_j(scale · q[t, h]·K[j]) V[j],   j <= past + s
// for the s-th new token t of a sequence with `past` tokens before; a row
// that sees no key gives 0.
//
// A CTA takes 16 query rows ((token, head) pairs that share a KV head; 8 or 4
// where no sequence has more) and a range of keys, 32 keys at a time through
// shared memory in fp32, with the running maximum and sum of the softmax in
// base 2.  Where the rows alone do not fill the GPU the keys are cut into
// ranges, whose (max, sum, O) go to the workspace and are joined in order by a
// second kernel.
//
// Bound: the fp32 FMA rate next to the shared-memory reads (each K and V
// element read from memory once per CTA's rows); in decode steps the round
// trips of a CTA's few rounds.  Measured: 8 fp32 tokens on up to 2 K positions
// (32 query, 4 KV heads of 64) 18.6 us, 24.8 with 16 rows to a CTA; 16 tokens
// with 8 KV heads 31 us = 2.0 TB/s, 57 with 16 rows; chunks of up to 20 tokens
// on the same lengths 88 us.
#include <math.h>

#include <algorithm>

#include "kernels.h"
#include "paged.h"

namespace mg {
namespace {

constexpr int kRows = 16;     // most query rows of a CTA
constexpr int kKeys = 32;     // keys of a round
constexpr int kSimt = 128;    // threads
constexpr int kMaxSplits = 64;
constexpr float kUnseen = -1.f;  // in place of a weight: the row does not see the key

// One 16-byte (e4m3: 8-code) piece of a cached row, widened.
template <typename C>
struct Cached;
template <>
struct Cached<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const float* p, float* v) { load16_f<float>(p, v); }
};
template <>
struct Cached<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* v) { load16_f<__nv_bfloat16>(p, v); }
};
template <>
struct Cached<uint8_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const uint8_t* p, float* v) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = from_e4m3x2((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};

// The workspace holds a part of D + 2 floats (maximum, sum, O) per key range
// of each (new token, head): the s-th new token of sequence b is its row
// part_row(a, b) + s.  By the batch's bounds, not by token rows, of which a
// padded batch may have many more.
__device__ __forceinline__ int64_t part_row(const PagedAttnArgs& a, int b) { return (int64_t)b * max(a.batch.max_new, 1); }

template <typename T, typename C, int D, int ROWS>
__global__ void __launch_bounds__(kSimt) paged_attn_simt_kernel(const __grid_constant__ PagedAttnArgs a, int tiles, int splits) {
  constexpr int RPT = ROWS * D / kSimt;           // output rows of a thread
  constexpr int TPR = kSimt / ROWS;                // threads of a query row
  constexpr int KPT = kKeys / TPR;                 // keys of a thread in a round
  static_assert(RPT >= 1 && TPR <= 32, "a query row lies in a warp");
  constexpr int P4 = Cached<C>::N;
  // Rows 4 floats apart in the banks: eight keys' 16-byte reads do not collide.
  __shared__ __align__(16) float sq[ROWS][D + 4];
  __shared__ __align__(16) float sk[kKeys][D + 4];
  __shared__ __align__(16) float sv[kKeys][D];
  __shared__ __align__(16) float sp[ROWS][kKeys];
  __shared__ float keep[ROWS], sum[ROWS], top[ROWS];
  pdl_trigger();
  pdl_wait();
  const PagedPool& pool = a.pool;
  const PagedBatch& bt = a.batch;
  const int tid = threadIdx.x, h = blockIdx.y, z = blockIdx.z;
  const int b = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  const int G = a.nq / pool.nkv;
  const SeqSpan span = seq_span(bt, b, pool.ps);
  if (!span.ok) {
    if (tid == 0) flag_error(a.err, kErrPaged);
    return;
  }
  const int rows = span.n * G, r0 = tile * ROWS;
  if (r0 >= rows) return;
  const int nr = min(ROWS, rows - r0);
  const int most = min(span.past + (r0 + nr - 1) / G + 1, span.past + span.n);  // keys the last row sees
  const int step = most > 0 ? (int)(((long long)(most + kKeys - 1) / kKeys + splits - 1) / splits) * kKeys : 0;
  const long long first = (long long)z * step;
  const int k_lo = (int)min(first, (long long)max(most, 0)), k_hi = (int)min(first + step, (long long)max(most, 0));

  for (int i = tid; i < ROWS * D; i += kSimt) {
    const int r = i / D, d = i % D;
    float x = 0.f;
    if (r < nr)
      x = ldf<T>((const T*)a.q + (int64_t)(span.q0 + (r0 + r) / G) * a.ldq + (int64_t)(h * G + (r0 + r) % G) * a.hdq + d);
    sq[r][d] = x;
  }
  const float scale2 = a.scale * 1.4426950408889634f;
  const int qr = tid / TPR, kq = tid % TPR;               // score row, first key
  const int vis = qr < nr ? span.past + (r0 + qr) / G + 1 : 0;
  float m = -INFINITY, l = 0.f;                           // of row qr (the same in its threads)
  const int od = tid % D, og = tid / D;                   // output dim, first output row / RPT
  float acc[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) acc[i] = 0.f;

  // A round's keys and values, requested a round ahead, its pages two.
  constexpr int NV = (kKeys * D / P4 + kSimt - 1) / kSimt;  // pieces of a thread
  const int page_shift = 31 - __clz(pool.ps);
  int page[NV];
  float kx[NV][P4], vx[NV][P4];
  auto look_up = [&](int k0) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int j = k0 + (tid + v * kSimt) / (D / P4);
      page[v] = j < k_hi && tid + v * kSimt < kKeys * D / P4 ? bt.table[(int64_t)b * bt.ld + (j >> page_shift)] : -1;
    }
  };
  auto request = [&](int k0) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = tid + v * kSimt, j = k0 + i / (D / P4), d = i % (D / P4) * P4, o = j & (pool.ps - 1);
#pragma unroll
      for (int e = 0; e < P4; ++e) kx[v][e] = vx[v][e] = 0.f;
      if (j >= k_hi || i >= kKeys * D / P4) continue;
      if (page[v] < 0 || page[v] >= pool.pages) {
        flag_error(a.err, kErrPaged);
        continue;
      }
      Cached<C>::load((const C*)pool.k + page[v] * pool.kp + h * pool.kh + o * pool.kt + d, kx[v]);
      Cached<C>::load((const C*)pool.v + page[v] * pool.vp + h * pool.vh + o * pool.vt + d, vx[v]);
      if constexpr (sizeof(C) == 1) {
        const float fk = pool.ks[page[v] * pool.kse + h], fv = pool.vs[page[v] * pool.vse + h];
#pragma unroll
        for (int e = 0; e < P4; ++e) kx[v][e] *= fk, vx[v][e] *= fv;
      }
    }
  };
  look_up(k_lo);
  request(k_lo);
  look_up(k_lo + kKeys);
  for (int k0 = k_lo; k0 < k_hi; k0 += kKeys) {
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = tid + v * kSimt, r = i / (D / P4), d = i % (D / P4) * P4;
      if (i >= kKeys * D / P4) continue;
#pragma unroll
      for (int e = 0; e < P4; e += 4) {
        *reinterpret_cast<float4*>(&sk[r][d + e]) = make_float4(kx[v][e], kx[v][e + 1], kx[v][e + 2], kx[v][e + 3]);
        *reinterpret_cast<float4*>(&sv[r][d + e]) = make_float4(vx[v][e], vx[v][e + 1], vx[v][e + 2], vx[v][e + 3]);
      }
    }
    __syncthreads();
    if (k0 + kKeys < k_hi) {
      request(k0 + kKeys);
      look_up(k0 + 2 * kKeys);
    }
    float s[KPT];
#pragma unroll
    for (int i = 0; i < KPT; ++i) s[i] = 0.f;
    for (int d = 0; d < D; d += 4) {
      const float4 x = *reinterpret_cast<const float4*>(&sq[qr][d]);
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        const float4 y = *reinterpret_cast<const float4*>(&sk[kq + TPR * i][d]);
        s[i] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s[i]))));
      }
    }
    float mx = m;
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      s[i] = k0 + kq + TPR * i < vis ? s[i] * scale2 : -INFINITY;
      mx = fmaxf(mx, s[i]);
    }
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - mx);
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const float p = s[i] == -INFINITY ? 0.f : exp2f(s[i] - mx);
      sp[qr][kq + TPR * i] = k0 + kq + TPR * i < vis ? p : kUnseen;
      part += p;
    }
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    m = mx;
    l = l * alpha + part;
    if (kq == 0) keep[qr] = alpha;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RPT; ++i) acc[i] *= keep[og * RPT + i];
    // Keys that no row of the tile sees were loaded as zeros; a row's own
    // invisible keys weigh 0, but 0 · NaN is not 0, so they are left out (and
    // only they: a visible key's NaN counts, however little it weighs).
    for (int k = 0; k < kKeys; k += 4) {
      const float v[4] = {sv[k][od], sv[k + 1][od], sv[k + 2][od], sv[k + 3][od]};
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float4 p4 = *reinterpret_cast<const float4*>(&sp[og * RPT + i][k]);
        const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i] = p[e] != kUnseen ? fmaf(p[e], v[e], acc[i]) : acc[i];
      }
    }
  }
  if (kq == 0) {
    sum[qr] = l;
    top[qr] = m;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = og * RPT + i;
    if (r >= nr) continue;
    const int64_t t = span.q0 + (r0 + r) / G;
    const int head = h * G + (r0 + r) % G;
    if (splits == 1) {
      stf<T>((T*)a.out + t * a.ldo + (int64_t)head * a.hdo + od, sum[r] == 0.f ? 0.f : acc[i] / sum[r]);
    } else {
      float* w = (float*)a.ws + (((part_row(a, b) - span.q0 + t) * a.nq + head) * splits + z) * (D + 2);
      w[2 + od] = acc[i];
      if (od == 0) {
        w[0] = top[r];
        w[1] = sum[r];
      }
    }
  }
}

// Join of the key ranges of one (new token, head): block (x, head) the
// x % max_new-th new token of sequence x / max_new, a thread per dim in each of
// kJoinParts parts, which take every kJoinParts-th range in their order and
// are then joined in theirs.
constexpr int kJoinParts = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinParts * D) paged_attn_join_kernel(const __grid_constant__ PagedAttnArgs a, int splits) {
  __shared__ float part[kJoinParts][D + 2];
  pdl_trigger();
  pdl_wait();
  const int most = max(a.batch.max_new, 1), b = blockIdx.x / most, s = blockIdx.x % most;
  const int head = blockIdx.y, d = threadIdx.x % D, mine = threadIdx.x / D;
  const SeqSpan span = seq_span(a.batch, b, a.pool.ps);  // on its way beside the ranges
  const float* w = (const float*)a.ws + ((part_row(a, b) + s) * a.nq + head) * splits * (D + 2);
  float M = -INFINITY, l = 0.f, o = 0.f;
  auto add = [&](float m, float sum, float v) {
    if (sum == 0.f) {  // it saw no key (v is 0), or its keys weigh nothing (v is 0 or NaN)
      o = fmaf(0.f, v, o);
      return;
    }
    const float top = fmaxf(M, m), keep = M == -INFINITY ? 0.f : exp2f(M - top), f = exp2f(m - top);
    M = top;
    l = l * keep + f * sum;
    o = o * keep + f * v;
  };
  for (int z0 = mine; z0 < splits; z0 += 8 * kJoinParts) {  // eight ranges' loads in flight
    float m[8], sum[8], v[8];
#pragma unroll
    for (int z = 0; z < 8; ++z) {
      const float* q = w + min(z0 + z * kJoinParts, splits - 1) * (D + 2);
      m[z] = __ldcg(q);
      sum[z] = __ldcg(q + 1);
      v[z] = __ldcg(q + 2 + d);
    }
#pragma unroll
    for (int z = 0; z < 8; ++z)
      if (z0 + z * kJoinParts < splits) add(m[z], sum[z], v[z]);
  }
  if (s >= span.n) return;  // (the same in the whole block)
  part[mine][d] = o;
  if (d == 0) {
    part[mine][D] = M;
    part[mine][D + 1] = l;
  }
  __syncthreads();
  if (mine > 0) return;
  for (int k = 1; k < kJoinParts; ++k) add(part[k][D], part[k][D + 1], part[k][d]);
  stf<T>((T*)a.out + (int64_t)(span.q0 + s) * a.ldo + (int64_t)head * a.hdo + d, l == 0.f ? 0.f : o / l);
}

int64_t most_rows(const PagedAttnArgs& a) { return (int64_t)std::max(a.batch.max_new, 1) * (a.nq / a.pool.nkv); }
int64_t simt_tiles(const PagedAttnArgs& a) { return (most_rows(a) + kRows - 1) / kRows; }

// Key ranges per row: enough CTAs for nine per SM, at least a round each (with
// 16 rows to a CTA and 4, 6, 8, 9, 10, 13 per SM: 8 tokens 26.4, 22.7, 24.8,
// 24.8, 24.8, 28.3 us, chunks of up to 20 tokens 145, 117, 98, 88, 88, 90 us, of
// up to 60 at 8, 9, 10: 137, 137, 148 us).
int simt_splits(const PagedAttnArgs& a) {
  const int64_t ctas = a.batch.B * simt_tiles(a) * a.pool.nkv;
  const int64_t keys = (int64_t)a.batch.max_pages * a.pool.ps;
  int64_t n = ctas > 0 ? (9LL * a.sms + ctas - 1) / ctas : 1;
  n = std::min<int64_t>(n, (keys + kKeys - 1) / kKeys);
  return (int)std::max<int64_t>(1, std::min<int64_t>(n, kMaxSplits));
}

template <typename T, typename C, int D>
cudaError_t launch_simt_d(const PagedAttnArgs& a, cudaStream_t s) {
  const int64_t tiles = simt_tiles(a), ctas = a.batch.B * tiles;
  const int splits = simt_splits(a);
  if (ctas > INT32_MAX) return cudaErrorInvalidConfiguration;  // (B · max_new beyond any batch that fits the GPU)
  const dim3 grid((unsigned)ctas, (unsigned)a.pool.nkv, (unsigned)splits);
  // A CTA's rows: no more than a sequence has, but a thread owns at least one output.
  constexpr int few = 4 < kSimt / D ? kSimt / D : 4, some = 8 < kSimt / D ? kSimt / D : 8;
  const int64_t rows = most_rows(a);
  auto kernel = rows <= few ? paged_attn_simt_kernel<T, C, D, few>
                : rows <= some ? paged_attn_simt_kernel<T, C, D, some> : paged_attn_simt_kernel<T, C, D, kRows>;
  cudaError_t e = launch_pdl(kernel, grid, dim3(kSimt), 0, s, a, (int)tiles, splits);
  if (e == cudaSuccess && splits > 1)
    e = launch_pdl(paged_attn_join_kernel<T, D>, dim3((unsigned)(a.batch.B * std::max(a.batch.max_new, 1)), (unsigned)a.nq),
                   dim3(kJoinParts * D), 0, s, a, splits);
  return e;
}

template <typename T, typename C>
cudaError_t launch_simt(const PagedAttnArgs& a, cudaStream_t s) {
  switch (a.pool.D) {
    case 8: return launch_simt_d<T, C, 8>(a, s);
    case 16: return launch_simt_d<T, C, 16>(a, s);
    case 32: return launch_simt_d<T, C, 32>(a, s);
    case 64: return launch_simt_d<T, C, 64>(a, s);
    case 128: return launch_simt_d<T, C, 128>(a, s);
  }
  return cudaErrorInvalidValue;
}

size_t simt_workspace(const PagedAttnArgs& a) {
  const int splits = simt_splits(a);
  return splits > 1 ? (size_t)a.batch.B * std::max(a.batch.max_new, 1) * a.nq * splits * (a.pool.D + 2) * sizeof(float) : 0;
}

bool only_few(const PagedAttnArgs& a) {
  return (int64_t)a.batch.max_new * (a.nq / a.pool.nkv) <= kPagedFewRows;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

size_t paged_attention_workspace(const PagedAttnArgs& a) {
  if (!paged_decode_applicable(a)) return simt_workspace(a);
  const size_t few = align256(paged_decode_workspace(a));
  return only_few(a) ? few : few + paged_extend_workspace(a);
}

// bf16 with head_dim 64 or 128 runs on the tensor cores: each sequence on the
// kernel for few or for many query rows, by its new tokens as the device has
// them (the host's bound says whether the second can be left out).  Other
// types and sizes run on the CUDA cores.
cudaError_t launch_paged_attention(const PagedAttnArgs& a, cudaStream_t s) {
  if (a.batch.T == 0 || a.batch.B == 0) return cudaSuccess;
  if (a.ws_bytes < paged_attention_workspace(a)) return cudaErrorInvalidValue;
  cudaError_t e;
  if (paged_decode_applicable(a)) {
    e = launch_paged_decode(a, s);
    if (e == cudaSuccess && !only_few(a)) {
      PagedAttnArgs many = a;
      many.ws = (uint8_t*)a.ws + align256(paged_decode_workspace(a));
      e = launch_paged_extend(many, s);
    }
  } else if (a.dtype == kBF16) {
    e = a.pool.cdtype == kE4M3 ? launch_simt<__nv_bfloat16, uint8_t>(a, s) : launch_simt<__nv_bfloat16, __nv_bfloat16>(a, s);
  } else {
    e = a.pool.cdtype == kE4M3 ? launch_simt<float, uint8_t>(a, s) : launch_simt<float, float>(a, s);
  }
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace mg
