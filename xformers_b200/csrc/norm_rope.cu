// Norms of queries and keys per head, rotary embeddings and KV-cache emplacement in one pass.
//
//   r = 1 / sqrt(mean_j x_j^2 + eps);  y_j = x_j * r * (w_j + offset);  then y is turned by the token's angles (rope_padded.cu)
//
// for every row (token, head) of xq and xk; rows of xv are copied.  HBM-bound: every row is read once and written once, statistics and
// products are taken in fp32 and rounded once to the type of the inputs.
//
// A row of D elements is held by L lanes of a warp (L the power of two from D / (2 E) on, E = 16 bytes of elements), each with a
// vector of the row's first half and the same vector of its second half, so the sum of squares is a few shuffles and a pair of
// split halves needs no exchange.  A warp works on 32 / L rows of one token side by side and walks down its heads.  Weights and the token's sines and
// cosines make four factors per pair,
//   z_re = r (x_re w_re cos - x_im w_im sin),   z_im = r (x_im w_im cos + x_re w_re sin),
// which stay in registers over the rows, and two pairs share an instruction.
//   Three kernels: norm_rope_few_kernel for what fits the SMs at a token to a CTA, norm_rope_kernel for more, norm_rope_any_kernel for rows that do not start on
// 16-byte boundaries.  Frequencies (a double-precision exponential each) are formed once per CTA, before it waits for the kernel ahead of it in the stream.
// Measured (bf16, 64 + 2 x 8 rows of 128 a token): 26939 tokens of 9 sequences 185 us (6.0 TB/s; the memory, half of whose traffic are writes, is what bounds it), 8096
// of 2 sequences 62 (5.3), 2048 of 2048 sequences 18.8 (4.5), 256 of 256 sequences 5.2 (latency).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "internal.h"
#include "ptx.cuh"
#include "rope.cuh"

namespace xfb {

constexpr int kNormThreads = 256, kNormWarps = kNormThreads / 32;
constexpr int kNormMaxDim = 512;

struct NormRopeArgs {
  xfb200_rope_params p;
  const void* q_weight;
  const void* k_weight;
  int32_t weight_dtype;
  float eps, weight_offset;
  int32_t lanes;  // that hold a row (vector path)
  int64_t cache_rows;
  double log2_theta;
  // Elements (words of a quantised cache) from a row to the next one of xq, xk, xv, out_q, cache_k, cache_v, where (group, head) flatten to
  // one stride in all of them (flat)
  int32_t flat;
  int32_t row[6];

  // offset of row i of a tensor (`which`: its place in `row`)
  __device__ __forceinline__ int64_t at(int i, int which, int heads, int64_t sg, int64_t sh) const {
    if (flat) return int64_t(i) * row[which];
    const int g = i / heads, h = i - g * heads;
    return g * sg + h * sh;
  }
  __device__ __forceinline__ int64_t xq_at(int i) const { return at(i, 0, p.q_heads, p.xq_g, p.xq_h); }
  __device__ __forceinline__ int64_t xk_at(int i) const { return at(i, 1, p.kv_heads, p.xk_g, p.xk_h); }
  __device__ __forceinline__ int64_t xv_at(int i) const { return at(i, 2, p.kv_heads, p.xv_g, p.xv_h); }
  __device__ __forceinline__ int64_t oq_at(int i) const { return at(i, 3, p.q_heads, p.oq_g, p.oq_h); }
  __device__ __forceinline__ int64_t ck_at(int i) const { return at(i, 4, p.kv_heads, p.ck_g, p.ck_h); }
  __device__ __forceinline__ int64_t cv_at(int i) const { return at(i, 5, p.kv_heads, p.cv_g, p.cv_h); }
};

__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
  if (w == nullptr) return 1.f;
  if (dtype == XFB200_F32) return reinterpret_cast<const float*>(w)[i];
  if (dtype == XFB200_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(reinterpret_cast<const __half*>(w)[i]);
}

// Where a token's keys and values go, and its position.  A key position outside the sequence's slot, or a page outside the pool, is not written: row -1.
struct __align__(16) Place {
  long long row;
  double pos;
};
__device__ __forceinline__ Place place_of(const NormRopeArgs& a, int tok, int b) {
  const xfb200_rope_params& p = a.p;
  const int slot = p.seqlen_k[b] - (p.seqstart_q[b + 1] - tok);  // the queries are the last keys of the sequence
  const int cache_start = p.seqstart_k[b];
  const int slot_rows = p.block_tables != nullptr ? p.pages_per_seq * p.page_size : p.seqstart_k[b + 1] - cache_start;
  auto position = [&](const void* base, int64_t i) -> long long {
    return p.seqpos_i64 ? reinterpret_cast<const long long*>(base)[i * p.seqpos_stride] : reinterpret_cast<const int*>(base)[i * p.seqpos_stride];
  };
  long long row = -1;
  if (slot >= 0 && slot < slot_rows) {
    row = p.block_tables != nullptr ? int64_t(p.block_tables[int64_t(b) * p.block_tables_stride + slot / p.page_size]) * p.page_size + slot % p.page_size
                                    : int64_t(cache_start) + slot;
    if (row < 0 || row >= a.cache_rows) row = -1;
  }
  return {row, double(p.seqpos != nullptr ? position(p.seqpos, tok) : slot + (p.first_seqpos != nullptr ? position(p.first_seqpos, b) : 0))};
}

// Shared memory: frequencies (double), weights of q and k (fp32), sines and cosines of the token of each warp, places of its next 32 tokens, and the rings.
constexpr int kNormDepth = 3;  // batches of a warp's ring, a row for every L lanes
constexpr int kNormRingBytes = kNormDepth * 2 * 32 * 16;  // of a warp
template <typename T>
struct NormShared {
  double* freq;   // [pairs]
  float* weight;  // [2][dim]
  float2* cs;     // [pairs], of the warp
  Place* places;  // [32], of the warp
  uint4* ring;    // [depth][2][32], of the warp, at the lane's place
  __device__ __forceinline__ NormShared(uint8_t* smem, int dim, int warp, int lane) {
    places = reinterpret_cast<Place*>(smem) + warp * 32;
    freq = reinterpret_cast<double*>(smem + kNormWarps * 32 * sizeof(Place));
    weight = reinterpret_cast<float*>(freq + dim / 2);
    cs = reinterpret_cast<float2*>(weight + 2 * dim) + warp * (dim / 2);
    ring = reinterpret_cast<uint4*>(smem + bytes(dim, false) + warp * kNormRingBytes) + lane;
  }
  __host__ __device__ static constexpr size_t bytes(int dim, bool rings) {
    return ((kNormWarps * 32 * sizeof(Place) + size_t(dim / 2) * 8 + size_t(2 * dim) * 4 + size_t(kNormWarps) * (dim / 2) * 8 + 15) & ~size_t(15)) + (rings ? kNormWarps * kNormRingBytes : 0);
  }
  // By the whole CTA; frequencies are formed before it waits for the kernel ahead of it in the stream.
  __device__ __forceinline__ void fill(const NormRopeArgs& a) {
    const int dim = a.p.dim;
    for (int j = threadIdx.x; j < dim / 2; j += kNormThreads)
      freq[j] = rope_rescale<double>(a.p, exp2(double(-2 * j) / double(dim) * a.log2_theta)) / double(a.p.linear_scale);
    grid_dep_wait();
    grid_dep_launch();
    for (int i = threadIdx.x; i < 2 * dim; i += kNormThreads)
      weight[i] = weight_at(i < dim ? a.q_weight : a.k_weight, a.weight_dtype, i < dim ? i : i - dim) + a.weight_offset;
  }
  // Sines and cosines of a token, by its warp.  The angle is formed in double precision and reduced there, to [-pi, pi]: single-precision sine and cosine are only
  // good on a small range.  Their fast forms are off by 2^-21, which 16-bit outputs do not show; fp32 ones get sincospif (417 tokens of 48 rows of 80: error
  // 1.8e-7 -> 7.8e-8 of the outputs' norm, 7.5 -> 7.6 us).  internal_f64 takes them in double precision.
  __device__ __forceinline__ void angles(const NormRopeArgs& a, double pos, int lane) {
    __syncwarp();
    for (int j = lane; j < a.p.dim / 2; j += 32) {
      const double ang = pos * freq[j];
      float sn, cn;
      if (a.p.internal_f64) {
        sn = float(sin(ang)), cn = float(cos(ang));
      } else if constexpr (std::is_same<T, float>::value) {
        const double half_turns = ang * 0.318309886183790671537767526745;
        sincospif(float(half_turns - 2.0 * rint(half_turns * 0.5)), &sn, &cn);
      } else {
        const double two_pi = 6.283185307179586476925286766559;
        __sincosf(float(ang - two_pi * rint(ang * (1.0 / two_pi))), &sn, &cn);
      }
      cs[j] = make_float2(cn, sn);
    }
    __syncwarp();
  }
};

// What a lane does to its part of a row: E pairs, with their factors two to a register pair.
template <typename T, bool kAdj>
struct NormPairs {
  static constexpr int E = RopeVec<T>::kElems;
  uint64_t rc[E / 2], is[E / 2], ic[E / 2], rs[E / 2];
  __device__ __forceinline__ void set(const float* w, const float2* cs, bool has, int x_off, int pairs) {
    const int y_off = pairs + x_off;
    float f[4][E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = kAdj ? (i >= E / 2 ? y_off + 2 * (i - E / 2) : x_off + 2 * i) : x_off + i;  // element of the real part
      const int pair = kAdj ? e / 2 : e;
      const float w_re = has ? w[e] : 0.f, w_im = has ? w[kAdj ? e + 1 : e + pairs] : 0.f;
      const float2 c = has ? cs[pair] : make_float2(1.f, 0.f);
      f[0][i] = w_re * c.x, f[1][i] = -(w_im * c.y), f[2][i] = w_im * c.x, f[3][i] = w_re * c.y;
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      rc[i] = f2_pack(f[0][2 * i], f[0][2 * i + 1]), is[i] = f2_pack(f[1][2 * i], f[1][2 * i + 1]);
      ic[i] = f2_pack(f[2][2 * i], f[2][2 * i + 1]), rs[i] = f2_pack(f[3][2 * i], f[3][2 * i + 1]);
    }
  }
  // (U rows at a time, whose chains run side by side; what does not depend on the norm comes before it)
  template <int U>
  __device__ __forceinline__ void apply(uint4 (&xw)[U], uint4 (&yw)[U], int L, float inv_dim, float eps) const {
    uint64_t z_re[U][E / 2], z_im[U][E / 2];
    float sq[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[E], y[E];
      RopeVec<T>::unpack(xw[u], x);
      RopeVec<T>::unpack(yw[u], y);
      uint64_t s2 = f2_pack(0.f, 0.f), t2 = s2;
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        uint64_t re, im;
        if constexpr (kAdj) {
          const float* z = i < E / 4 ? x + 4 * i : y + 4 * (i - E / 4);
          re = f2_pack(z[0], z[2]), im = f2_pack(z[1], z[3]);
        } else {
          re = f2_pack(x[2 * i], x[2 * i + 1]), im = f2_pack(y[2 * i], y[2 * i + 1]);
        }
        s2 = ffma2(re, re, s2), t2 = ffma2(im, im, t2);
        z_re[u][i] = ffma2(re, rc[i], fmul2(im, is[i])), z_im[u][i] = ffma2(im, ic[i], fmul2(re, rs[i]));
      }
      float s, t;
      f2_unpack(fadd2(s2, t2), s, t);
      sq[u] = s + t;
    }
    for (int o = 1; o < L; o <<= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) sq[u] += __shfl_xor_sync(0xffffffffu, sq[u], o);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float r = rsqrtf(sq[u] * inv_dim + eps);
      const uint64_t r2 = f2_pack(r, r);
      float x[E], y[E];
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        if constexpr (kAdj) {
          float* z = i < E / 4 ? x + 4 * i : y + 4 * (i - E / 4);
          f2_unpack(fmul2(z_re[u][i], r2), z[0], z[2]), f2_unpack(fmul2(z_im[u][i], r2), z[1], z[3]);
        } else {
          f2_unpack(fmul2(z_re[u][i], r2), x[2 * i], x[2 * i + 1]), f2_unpack(fmul2(z_im[u][i], r2), y[2 * i], y[2 * i + 1]);
        }
      }
      xw[u] = RopeVec<T>::pack(x), yw[u] = RopeVec<T>::pack(y);
    }
  }
};

// The rows of a token in the cache of k or v.
template <typename T, int kQuant>
__device__ __forceinline__ void* cache_rows(const NormRopeArgs& a, bool of_v, long long row) {
  using C = typename std::conditional<kQuant == 0, T, int32_t>::type;  // an element of the caches
  return of_v ? reinterpret_cast<C*>(a.p.cache_v) + row * a.p.cv_m : reinterpret_cast<C*>(a.p.cache_k) + row * a.p.ck_m;
}
// One of them into its cache; the whole warp calls it.  kQuant as in rope_padded_kernel: 1 int4 row-wise caches, 2 fp8 row-wise caches.  (The rows of a
// quantised cache fill their lanes; what a 16-bit cache would hold is what is quantised.)
template <typename T, int kQuant>
__device__ __forceinline__ void to_cache(const NormRopeArgs& a, bool of_v, void* rows, long long cache_row, int r, bool live, uint4 xw, uint4 yw, int x_off, int y_off, int L, int v) {
  const xfb200_rope_params& p = a.p;
  using C = typename std::conditional<kQuant == 0, T, int32_t>::type;
  C* const dst = reinterpret_cast<C*>(rows) + (of_v ? a.cv_at(r) : a.ck_at(r));
  if constexpr (kQuant != 0) {
    constexpr int E = RopeVec<T>::kElems;
    float x[E], y[E];
    RopeVec<T>::unpack(xw, x);
    RopeVec<T>::unpack(yw, y);
    int32_t* ss = nullptr;
    if (kQuant == 2 && live) {
      const int g = r / p.kv_heads, h = r - g * p.kv_heads;
      ss = of_v ? reinterpret_cast<int32_t*>(p.v_scale_shift) + cache_row * p.vss_m + g * p.vss_g + h * p.vss_h
                : reinterpret_cast<int32_t*>(p.k_scale_shift) + cache_row * p.kss_m + g * p.kss_g + h * p.kss_h;
    }
    quantise_row<E, kQuant>(x, y, L, v, p.dim, live, dst, ss);
  } else if (live) {
    RopeVec<T>::store(dst + x_off, xw);
    RopeVec<T>::store(dst + y_off, yw);
  }
}

// ---------------------------------------------------------------------------
// A token to a CTA (blockIdx = token of the sequence, sequence), all of them at once.  Latency is what counts: a warp asks for the first rows of each kind before
// page table, position and angles are known (256 sequences, paged: 5.1 us; through the ring of norm_rope_kernel 6.7).
// ---------------------------------------------------------------------------
template <int U>
struct RowBatch {  // U rows of a lane on their way
  uint4 x[U], y[U];
  template <typename T, typename At>
  __device__ __forceinline__ void load(int r0, int step, int n_rows, bool has, const T* src, At&& row_at, int x_off, int y_off) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * step;
      x[u] = y[u] = make_uint4(0, 0, 0, 0);
      if (has && r < n_rows) {
        const T* row = src + row_at(r);
        x[u] = RopeVec<T>::load(row + x_off);
        y[u] = RopeVec<T>::load(row + y_off);
      }
    }
  }
};

template <typename T, bool kAdj, int kQuant>
__global__ void __launch_bounds__(kNormThreads, 2) norm_rope_few_kernel(const __grid_constant__ NormRopeArgs a) {
  constexpr int E = RopeVec<T>::kElems;
  extern __shared__ __align__(16) uint8_t norm_smem[];
  const xfb200_rope_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pairs = p.dim / 2;
  NormShared<T> sm(norm_smem, p.dim, warp, lane);
  sm.fill(a);
  const int b = blockIdx.y, tok = p.seqstart_q[b] + int(blockIdx.x);
  if (tok >= p.seqstart_q[b + 1]) return;
  const int nq = p.q_heads * p.groups, nkv = p.kv_heads * p.groups;
  const int L = a.lanes, v = lane % L, rpw = 32 / L, step = kNormWarps * rpw, r_q = warp * rpw + lane / L;
  const int r_v = (warp + kNormWarps / 2) % kNormWarps * rpw + lane / L;  // (the rows of v go to warps that have none of k, as far as there are such)
  const bool has = v < pairs / E;  // (a lane behind the end of a row takes part in the exchanges only)
  const int x_off = v * E, y_off = pairs + x_off;
  const T* const src_q = reinterpret_cast<const T*>(p.xq) + int64_t(tok) * p.xq_m;
  const T* const src_k = reinterpret_cast<const T*>(p.xk) + int64_t(tok) * p.xk_m;
  const T* const src_v = reinterpret_cast<const T*>(p.xv) + int64_t(tok) * p.xv_m;
  auto xq_at = [&](int i) { return a.xq_at(i); };
  auto xk_at = [&](int i) { return a.xk_at(i); };
  auto xv_at = [&](int i) { return a.xv_at(i); };
  RowBatch<2> q;
  RowBatch<1> k, vv;
  q.load(r_q, step, nq, has, src_q, xq_at, x_off, y_off);
  k.load(r_q, step, nkv, has, src_k, xk_at, x_off, y_off);
  vv.load(r_v, step, nkv, has, src_v, xv_at, x_off, y_off);
  const Place at = place_of(a, tok, b);
  __syncthreads();
  sm.angles(a, at.pos, lane);
  const float inv_dim = 1.f / float(p.dim);
  // (r - lane / L: the warp's first row of a round, the same for all lanes)
  if (at.row >= 0) {
    for (int r = r_v; r - lane / L < nkv; r += step) {
      if (r != r_v) vv.load(r, step, nkv, has, src_v, xv_at, x_off, y_off);
      to_cache<T, kQuant>(a, true, cache_rows<T, kQuant>(a, true, at.row), at.row, r, has && r < nkv, vv.x[0], vv.y[0], x_off, y_off, L, v);
    }
    NormPairs<T, kAdj> f;
    if (r_q - lane / L < nkv) f.set(sm.weight + p.dim, sm.cs, has, x_off, pairs);
    for (int r = r_q; r - lane / L < nkv; r += step) {
      if (r != r_q) k.load(r, step, nkv, has, src_k, xk_at, x_off, y_off);
      f.apply(k.x, k.y, L, inv_dim, a.eps);
      to_cache<T, kQuant>(a, false, cache_rows<T, kQuant>(a, false, at.row), at.row, r, has && r < nkv, k.x[0], k.y[0], x_off, y_off, L, v);
    }
  }
  NormPairs<T, kAdj> f;
  f.set(sm.weight, sm.cs, has, x_off, pairs);
  T* const dst_q = reinterpret_cast<T*>(p.out_q) + int64_t(tok) * p.oq_m;
  for (int r0 = r_q; r0 - lane / L < nq; r0 += 2 * step) {
    if (r0 != r_q) q.load(r0, step, nq, has, src_q, xq_at, x_off, y_off);
    f.apply(q.x, q.y, L, inv_dim, a.eps);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = r0 + u * step;
      if (has && r < nq) {
        T* const dst = dst_q + a.oq_at(r);
        RopeVec<T>::store(dst + x_off, q.x[u]);
        RopeVec<T>::store(dst + y_off, q.y[u]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Many tokens: CTAs that are resident all the time, whose warps go through the tokens of the call as one row of them, whatever the lengths of its sequences.
// (With CTAs that have up to 16 tokens of one sequence each: 8096 tokens of 2 sequences 81 us instead of 62, a prompt of 2048 beside 63 single tokens, 32 heads, 33.5 instead of 12.8.)
// ---------------------------------------------------------------------------
// How many warps of a CTA share a token, so that the slowest is through soonest: a token costs a warp as much as kTokenRows steps of rows
// before the first one.  (1 / 2 / 4 / 8 warps, and as this has it: 8096 tokens of 80 rows of 128 62.9 / 61.0 / 68.0 / 88.4, 61.6 us; 1024 of them 13.2 / 10.9 / 12.8 / 16.0, 11.5;
// 540 12.9 / 8.9 / 8.1 / 9.8, 8.7; 2048 tokens of 48 rows 11.6 / 13.4 / 16.0 / 21.0, 12.2.)
constexpr int kTokenRows = 3;
__device__ __forceinline__ int warps_per_token(int64_t tokens, int steps) {
  int best = kNormWarps;
  int64_t best_cost = -1;
#pragma unroll
  for (int w = kNormWarps; w >= 1; w >>= 1) {
    const int64_t at_once = int64_t(gridDim.x) * (kNormWarps / w), cost = (tokens + at_once - 1) / at_once * (kTokenRows + (steps + w - 1) / w);
    if (best_cost < 0 || cost < best_cost) best = w, best_cost = cost;
  }
  return best;
}

struct WarpTokens {
  int tok, end, stride, wpt, share, start, batch;
  __device__ __forceinline__ WarpTokens(const NormRopeArgs& a, int warp, int steps) {
    start = a.p.seqstart_q[0], end = a.p.seqstart_q[a.p.batch], batch = a.p.batch;
    wpt = warps_per_token(int64_t(end) - start, steps);
    tok = start + warp / wpt * int(gridDim.x) + int(blockIdx.x), stride = int(gridDim.x) * (kNormWarps / wpt), share = warp % wpt;
  }
  // The places of this token and the warp's next 31, a lane each.  The sequence of a token is the last one that starts at or before it: where it would be if
  // all were as long, or else by bisection.
  __device__ __forceinline__ void places(const NormRopeArgs& a, Place* to, int lane) const {
    const int32_t* const starts = a.p.seqstart_q;
    const int64_t t64 = int64_t(tok) + int64_t(lane) * stride;
    __syncwarp();
    if (t64 < end) {
      const int t = int(t64);
      int b = int((t64 - start) * batch / (end - start));
      if (starts[b] > t || starts[b + 1] <= t) {
        b = 0;
        for (int n = batch; n > 1;) {
          const int half = n / 2;
          if (starts[b + half] <= t) b += half, n -= half;
          else n = half;
        }
      }
      to[lane] = place_of(a, t, b);
    }
    __syncwarp();
  }
};

// CTAs to an SM: what the registers of 16-bit rows, twice as many elements to a lane, allow (three with spilt registers: 26939 tokens 198 us instead of 185; f32,
// 17981 tokens of 24 rows of 80: two 70 us, three 63).
template <typename T>
constexpr int norm_ctas() { return sizeof(T) == 4 ? 3 : 2; }

// Rows start on 16-byte boundaries and dim is a multiple of two vectors.  A warp's rows come through a ring in shared memory, kNormDepth - 1 batches ahead and across tokens;
// every lane copies and reads back its own vectors, so no barrier is involved.  Nothing reads the rows again, so the L2 is told to drop them first, which
// leaves it to what is written (without: 2048 single tokens 19.5 us instead of 18.8, 3563 tokens of 48 rows 21.2 instead of 20.4; 26939 of 80 rows, far beyond the L2, 181
// instead of 185).  More on the way at once does not help the longest calls (rings of 3 / 4 batches: 26939 tokens 185 / 194 us, 8096 61.6 / 59.4).
template <typename T, bool kAdj, int kQuant>
__global__ void __launch_bounds__(kNormThreads, norm_ctas<T>()) norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  constexpr int E = RopeVec<T>::kElems;
  extern __shared__ __align__(16) uint8_t norm_smem[];
  const xfb200_rope_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pairs = p.dim / 2;
  NormShared<T> sm(norm_smem, p.dim, warp, lane);
  sm.fill(a);
  const int nq = p.q_heads * p.groups, nkv = p.kv_heads * p.groups;
  const int L = a.lanes, v = lane % L, rpw = 32 / L, rg = lane / L;  // lanes of a row, rows that a warp has side by side
  WarpTokens mine(a, warp, (nq + 2 * nkv + rpw - 1) / rpw);
  const int step = mine.wpt * rpw;
  const bool has = v < pairs / E;  // (a lane behind the end of a row takes part in the exchanges only)
  const int x_off = v * E, y_off = pairs + x_off;

  // The kinds of a token in the order in which they are gone through: q, v, k.  The first row of a kind that this warp has:
  const int first_qk = mine.share * rpw, first_v = (mine.share + (mine.wpt >> 1)) % mine.wpt * rpw;  // (the rows of v go to warps that have none of k, as far as there are such)
  auto first_of = [&](int kind) { return kind == 1 ? first_v : first_qk; };
  auto rows_of = [&](int kind) { return kind == 0 ? nq : nkv; };
  int ask_tok = mine.tok, ask_kind = 0, ask_row = first_qk, ask_n = nq, ask_slot = 0;  // the next batch to ask for
  const T* ask_src = reinterpret_cast<const T*>(p.xq) + ask_tok * p.xq_m + x_off;
  const uint64_t keep_none = l2_evict_first();
  auto ask = [&]() {
    while (ask_tok < mine.end && ask_row >= ask_n) {  // (on to the next kind; some have no row for this warp)
      if (++ask_kind == 3) ask_kind = 0, ask_tok = int(min(int64_t(ask_tok) + mine.stride, int64_t(mine.end)));
      ask_row = first_of(ask_kind), ask_n = rows_of(ask_kind);
      ask_src = (ask_kind == 0   ? reinterpret_cast<const T*>(p.xq) + ask_tok * p.xq_m
                 : ask_kind == 1 ? reinterpret_cast<const T*>(p.xv) + ask_tok * p.xv_m
                                 : reinterpret_cast<const T*>(p.xk) + ask_tok * p.xk_m) + x_off;
    }
    if (ask_tok < mine.end) {
      const int r = ask_row + rg;
      const bool ok = has && r < ask_n;
      const T* const row = ask_src + (!ok ? -x_off : ask_kind == 0 ? a.xq_at(r) : ask_kind == 1 ? a.xv_at(r) : a.xk_at(r));
      uint4* const to = sm.ring + ask_slot * 64;
      cp_async_16(to, row, ok, keep_none);
      cp_async_16(to + 32, row + (ok ? pairs : 0), ok, keep_none);
      ask_row += step;
    }
    cp_async_commit();
    ask_slot = ask_slot + 1 == kNormDepth ? 0 : ask_slot + 1;
  };
#pragma unroll 1
  for (int i = 0; i < kNormDepth - 1; ++i) ask();
  int slot = 0;
  __syncthreads();

  const float inv_dim = 1.f / float(p.dim);
  for (int i = 0; mine.tok < mine.end; ++i) {
    if ((i & 31) == 0) mine.places(a, sm.places, lane);
    const Place at = sm.places[i & 31];
    sm.angles(a, at.pos, lane);
#pragma unroll 1
    for (int kind = 0; kind < 3; ++kind) {
      const int n = rows_of(kind);
      int r0 = first_of(kind);
      if (r0 >= n) continue;
      void* const dst = kind == 0 ? reinterpret_cast<T*>(p.out_q) + mine.tok * p.oq_m : cache_rows<T, kQuant>(a, kind == 1, at.row);
      NormPairs<T, kAdj> f;
      if (kind != 1) f.set(sm.weight + (kind == 0 ? 0 : p.dim), sm.cs, has, x_off, pairs);
#pragma unroll 1
      for (; r0 < n; r0 += step) {
        cp_async_wait<kNormDepth - 2>();
        const uint4* const from = sm.ring + slot * 64;
        uint4 xw[1] = {from[0]}, yw[1] = {from[32]};
        slot = slot + 1 == kNormDepth ? 0 : slot + 1;
        ask();  // (into the slot of the batch before this one, whose values are long used)
        if (kind != 1) f.apply(xw, yw, L, inv_dim, a.eps);
        const int r = r0 + rg;
        const bool live = has && r < n;
        if (kind != 0) {
          to_cache<T, kQuant>(a, kind == 1, dst, at.row, r, live && at.row >= 0, xw[0], yw[0], x_off, y_off, L, v);
        } else if (live) {
          T* const row = reinterpret_cast<T*>(dst) + a.oq_at(r);
          RopeVec<T>::store(row + x_off, xw[0]);
          RopeVec<T>::store(row + y_off, yw[0]);
        }
      }
    }
    mine.tok = int(min(int64_t(mine.tok) + mine.stride, int64_t(mine.end)));
  }
}

// Any other shape: a lane has the pairs lane, lane + 32, ... of a row.
template <typename T, bool kAdj>
__global__ void __launch_bounds__(kNormThreads, 4) norm_rope_any_kernel(const __grid_constant__ NormRopeArgs a) {
  extern __shared__ __align__(16) uint8_t norm_smem[];
  const xfb200_rope_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pairs = p.dim / 2;
  NormShared<T> sm(norm_smem, p.dim, warp, lane);
  sm.fill(a);
  const int nq = p.q_heads * p.groups, nkv = p.kv_heads * p.groups;
  WarpTokens mine(a, warp, nq + 2 * nkv);
  __syncthreads();
  const float inv_dim = 1.f / float(p.dim);
  constexpr int N = kNormMaxDim / 64;  // pairs of a lane
  for (int i = 0; mine.tok < mine.end; ++i) {
    if ((i & 31) == 0) mine.places(a, sm.places, lane);
    const Place to = sm.places[i & 31];
    sm.angles(a, to.pos, lane);
    for (int r = mine.share; r < nq + 2 * nkv; r += mine.wpt) {
      const int kind = (r >= nq) + (r >= nq + nkv), j = r - (kind == 0 ? 0 : kind == 1 ? nq : nq + nkv);
      if (kind != 0 && to.row < 0) continue;
      const T* src = kind == 0   ? reinterpret_cast<const T*>(p.xq) + mine.tok * p.xq_m + a.xq_at(j)
                     : kind == 1 ? reinterpret_cast<const T*>(p.xk) + mine.tok * p.xk_m + a.xk_at(j)
                                 : reinterpret_cast<const T*>(p.xv) + mine.tok * p.xv_m + a.xv_at(j);
      T* dst = kind == 0   ? reinterpret_cast<T*>(p.out_q) + mine.tok * p.oq_m + a.oq_at(j)
               : kind == 1 ? reinterpret_cast<T*>(p.cache_k) + to.row * p.ck_m + a.ck_at(j)
                           : reinterpret_cast<T*>(p.cache_v) + to.row * p.cv_m + a.cv_at(j);
      float re[N], im[N], sq = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int j = lane + 32 * n;
        re[n] = im[n] = 0.f;
        if (j < pairs) {
          re[n] = RopeIo<T>::ld(src + (kAdj ? 2 * j : j));
          im[n] = RopeIo<T>::ld(src + (kAdj ? 2 * j + 1 : j + pairs));
        }
        sq += re[n] * re[n] + im[n] * im[n];
      }
      for (int o = 1; o < 32; o <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      const float rs = rsqrtf(sq * inv_dim + a.eps);
      const float* wr = sm.weight + (kind == 0 ? 0 : p.dim);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int j = lane + 32 * n;
        if (j >= pairs) continue;
        const int c_re = kAdj ? 2 * j : j, c_im = kAdj ? 2 * j + 1 : j + pairs;
        float x = re[n], y = im[n];
        if (kind != 2) {
          const float2 w = sm.cs[j];
          const float s = x * rs * wr[c_re], z = y * rs * wr[c_im];
          x = s * w.x - z * w.y, y = z * w.x + s * w.y;
        }
        RopeIo<T>::st(dst + c_re, x);
        RopeIo<T>::st(dst + c_im, y);
      }
    }
    mine.tok = int(min(int64_t(mine.tok) + mine.stride, int64_t(mine.end)));
  }
}

template <typename T>
static int launch_norm_rope(NormRopeArgs a, cudaStream_t st) {
  constexpr int E = RopeVec<T>::kElems;
  const xfb200_rope_params& p = a.p;
  auto aligned = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  const int64_t strides[] = {p.xq_m, p.xq_g, p.xq_h, p.xk_m, p.xk_g, p.xk_h, p.xv_m, p.xv_g, p.xv_h,
                             p.oq_m, p.oq_g, p.oq_h, p.ck_m, p.ck_g, p.ck_h, p.cv_m, p.cv_g, p.cv_h};
  const bool quant = p.cache_format != 0;
  const int per_row = p.dim / 2 / E;
  bool vec = p.dim % (2 * E) == 0 && per_row <= 32 && aligned(p.xq) && aligned(p.xk) && aligned(p.xv) && aligned(p.out_q) &&
             (quant || (aligned(p.cache_k) && aligned(p.cache_v)));
  for (int i = 0; i < 18; ++i) vec = vec && ((quant && i >= 12) || strides[i] % E == 0);
  for (a.lanes = 1; a.lanes < per_row;) a.lanes <<= 1;
  {
    a.flat = 1;
    auto flatten = [&](int heads, int64_t g, int64_t h) {
      if (p.groups > 1 && heads > 1 && g != heads * h) a.flat = 0;
      const int64_t stride = heads > 1 ? h : g;
      if (stride != int32_t(stride)) a.flat = 0;
      return int32_t(stride);
    };
    a.row[0] = flatten(p.q_heads, p.xq_g, p.xq_h), a.row[1] = flatten(p.kv_heads, p.xk_g, p.xk_h), a.row[2] = flatten(p.kv_heads, p.xv_g, p.xv_h);
    a.row[3] = flatten(p.q_heads, p.oq_g, p.oq_h), a.row[4] = flatten(p.kv_heads, p.ck_g, p.ck_h), a.row[5] = flatten(p.kv_heads, p.cv_g, p.cv_h);
  }
  const int64_t tokens = int64_t(p.batch) * p.max_q_per_seq;  // at most
  const bool few = vec && tokens <= 2 * sm_count();
  auto go = [&](auto* kernel, int per_sm, bool rings) -> int {
    const dim3 grid = few ? dim3(unsigned(p.max_q_per_seq), unsigned(p.batch), 1) : dim3(unsigned(std::min<int64_t>(tokens, int64_t(per_sm) * sm_count())), 1, 1);
    const cudaError_t e = launch_early(kernel, grid, kNormThreads, NormShared<T>::bytes(p.dim, rings), st, a);
    return e != cudaSuccess ? cuda_fail("norm_rope_kernel launch", e) : XFB200_OK;
  };
  auto vectors = [&](auto format, auto adjacents) -> int {
    constexpr int kQuant = decltype(format)::value;
    constexpr bool kAdj = decltype(adjacents)::value;
    if (few) return go(norm_rope_few_kernel<T, kAdj, kQuant>, 2, false);
    auto* kernel = norm_rope_kernel<T, kAdj, kQuant>;
    static bool configured[kMaxDevices] = {false};  // the attribute belongs to the device's context
    if (first_use_on_device(configured)) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(NormShared<T>::bytes(kNormMaxDim, true)));
      if (e != cudaSuccess) return cuda_fail("norm_rope_padded: cudaFuncSetAttribute", e);
    }
    return go(kernel, norm_ctas<T>(), true);
  };
  auto pick = [&](auto format) -> int { return p.adjacents ? vectors(format, std::true_type()) : vectors(format, std::false_type()); };
  static_assert(NormShared<T>::bytes(kNormMaxDim, false) <= 48 * 1024, "shared memory without an opt-in");
  if (quant) {
    if constexpr (sizeof(T) != 2) {
      return set_error(XFB200_E_UNSUPPORTED, "norm_rope_padded: a quantised cache needs bf16 or f16 inputs");
    } else {
      if (!vec || per_row != a.lanes || per_row < 2)
        return set_error(XFB200_E_UNSUPPORTED, "norm_rope_padded: a quantised cache needs dim 32, 64, 128, 256 or 512 and 16-byte aligned input rows");
      return p.cache_format == 2 ? pick(std::integral_constant<int, 2>()) : pick(std::integral_constant<int, 1>());
    }
  }
  if (vec) return pick(std::integral_constant<int, 0>());
  return p.adjacents ? go(norm_rope_any_kernel<T, true>, 4, false) : go(norm_rope_any_kernel<T, false>, 4, false);
}

}  // namespace xfb

extern "C" int xfb200_norm_rope_padded(const xfb200_norm_rope_params* p, void* stream) {
  using namespace xfb;
  if (p == nullptr) return set_error(XFB200_E_INVALID, "norm_rope_padded: null params");
  bool empty;
  const int rc = check_rope_params(&p->rope, "norm_rope_padded", &empty);
  if (rc != XFB200_OK || empty) return rc;
  if (p->rope.dim > kNormMaxDim) return set_error(XFB200_E_UNSUPPORTED, "norm_rope_padded: dim %d (at most %d)", p->rope.dim, kNormMaxDim);
  if (!(p->eps >= 0.f)) return set_error(XFB200_E_INVALID, "norm_rope_padded: eps must not be negative");
  if (p->weight_dtype != XFB200_BF16 && p->weight_dtype != XFB200_F16 && p->weight_dtype != XFB200_F32)
    return set_error(XFB200_E_INVALID, "norm_rope_padded: bad weight_dtype %d", p->weight_dtype);
  if (p->cache_rows < 0) return set_error(XFB200_E_INVALID, "norm_rope_padded: cache_rows must not be negative");
  NormRopeArgs a{};
  a.p = p->rope;
  a.q_weight = p->q_weight, a.k_weight = p->k_weight, a.weight_dtype = p->weight_dtype;
  a.eps = p->eps, a.weight_offset = p->weight_offset;
  a.cache_rows = p->cache_rows;
  a.log2_theta = std::log2(double(p->rope.theta));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->rope.dtype == XFB200_BF16) return launch_norm_rope<__nv_bfloat16>(a, st);
  if (p->rope.dtype == XFB200_F16) return launch_norm_rope<__half>(a, st);
  return launch_norm_rope<float>(a, st);
}
