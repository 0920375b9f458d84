// Softmax cross entropy of z = x W^T + b over a large vocabulary, from the hidden states on, without keeping the logits.
//   forward   lse_t = log sum_v exp z_tv, in one pass over the vocabulary: every 128 x 128 tile of logits leaves (max, sum of
//             exp) per token, a second launch joins them;  loss_t = lse_t - (1 - e) z_t,y - e/V sum_v z_tv
//   backward  in pieces of the vocabulary: G = w_t (exp(z - lse_t) - (1 - e)[v = y_t] - e/V) for one piece, recomputed, in 16-bit
//             planes; dx += G W and dW = G^T x of that piece; db = column sums of G
// The tile computes z transposed (r = vocabulary, c = token): a lane holds 32 logits of one token, so the softmax statistics
// need one exchange between lane halves instead of five steps for each of 32 rows.
// bf16 tensors go to the matrix cores as they are, G is rounded to bf16 (2^-9 relative, unbiased, T V of them to a sum: below the
// rounding of the bf16 gradients themselves).  fp32 tensors are split into two fp16 planes scaled by a power of two taken from the
// tensor's largest element (gemm16.h); G likewise.  Statistics, sums and partial gradients are fp32.
// Rows whose target is ignore_index are packed as zeros and weighted zero: whatever they hold (NaN, Inf) reaches nothing.
// Bound by the matrix cores: 8 T V D operations, of which the recomputation is 2 T V D; for few tokens by the reading of W.
#include "gemm16.h"

#define CE_AMAX_X 128                    // partial maxima of x and of W
#define CE_AMAX_W 384
#define CE_PIECE_BYTES (128ll << 20)     // of G: half of the 256 MB last-level cache

struct CeDims {
  int64_t T, D, V, Tp, Dp, tiles_v, tiles_t;
  int np;
  bool pack_w;
};
static bool ce_dims(int64_t T, int64_t D, int64_t V, int bf16, int w_aligned, CeDims* d) {
  if (T <= 0 || D <= 0 || V <= 0 || T > (1 << 24) || D > (1 << 20) || V > (1 << 24)) return false;
  auto pad = [](int64_t v) { return (v + G16_PAD - 1) / G16_PAD * G16_PAD; };
  d->T = T; d->D = D; d->V = V; d->Tp = pad(T); d->Dp = pad(D);
  d->tiles_v = ceil_div(V, G16_T); d->tiles_t = ceil_div(T, G16_T);
  d->np = bf16 ? 1 : 2;
  d->pack_w = !bf16 || d->Dp != D || !w_aligned;
  return true;
}
static size_t ce_up(size_t b) { return (b + 255) & ~(size_t)255; }

// what the forward pass leaves for the backward: [scales][x planes][W planes]
struct CeKept { float* scale; unsigned short* x; unsigned short* w; size_t bytes; };
static CeKept ce_kept(void* base, const CeDims& d) {
  CeKept k;
  char* p = (char*)base;
  size_t at = 0;
  k.scale = (float*)p; at += 256;
  k.x = (unsigned short*)(p + at); at += ce_up((size_t)d.np * d.Tp * d.Dp * 2);
  k.w = (unsigned short*)(p + at); if (d.pack_w) at += ce_up((size_t)d.np * d.V * d.Dp * 2);
  k.bytes = at;
  return k;
}
// scale: [0] 2^Ex, [1] 2^Ew, [2] number of live rows

__device__ __forceinline__ float ce_block_max(float m, float* red) {
  m = ofq_wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  const float r = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  return r;
}

// the power of two that brings m into [2^13, 2^14): two planes hold every element down to m 2^-13 with 2^-22 of it, and a
// rounding up stays far below fp16's 65504; 1 for 0, Inf and NaN
__device__ __forceinline__ float ce_scale(float m) {
  const int ex = (int)((__float_as_uint(m) >> 23) & 0xffu) - 127;
  if (!(m > 0.f) || ex == 128) return 1.f;
  const int e = min(max(13 - ex, -100), 100);
  return __uint_as_float((unsigned)(e + 127) << 23);
}

__global__ __launch_bounds__(256) void ce_amax_kernel(const float* __restrict__ x, const int64_t* __restrict__ y, int64_t ignore, int64_t T,
                                                      int64_t D, const float* __restrict__ w, int64_t nw, float* __restrict__ parts) {
  __shared__ float red[4];
  float m = 0.f;
  if (blockIdx.x < CE_AMAX_X) {
    for (int64_t t = blockIdx.x * 4 + (threadIdx.x >> 6); t < T; t += CE_AMAX_X * 4) {
      if (y[t] == ignore) continue;
      for (int64_t i = threadIdx.x & 63; i < D; i += 64) m = fmaxf(m, fabsf(x[t * D + i]));
    }
  } else {
    const int64_t n4 = ((uintptr_t)w & 15) == 0 ? nw / 4 : 0;
    const int64_t b = blockIdx.x - CE_AMAX_X;
    for (int64_t i = b * 256 + threadIdx.x; i < n4; i += CE_AMAX_W * 256) {
      const float4 v = reinterpret_cast<const float4*>(w)[i];
      m = ofq_absmax4(m, v.x, v.y, v.z, v.w);
    }
    for (int64_t i = n4 * 4 + b * 256 + threadIdx.x; i < nw; i += CE_AMAX_W * 256) m = fmaxf(m, fabsf(w[i]));
  }
  m = ce_block_max(m, red);
  if (threadIdx.x == 0) parts[blockIdx.x] = m;
}

// x (rows with ignored targets as zeros, padding as zeros) and, where it cannot be used in place, W into planes; one thread to
// eight elements of a row
template <int NP>
__global__ __launch_bounds__(256) void ce_pack_kernel(const void* __restrict__ x, const int64_t* __restrict__ y, int64_t ignore,
                                                      const void* __restrict__ w, CeDims d, const float* __restrict__ parts, CeKept k) {
  __shared__ float red[4];
  float sx = 1.f, sw = 1.f;
  if (NP == 2) {
    float m = threadIdx.x < CE_AMAX_X ? parts[threadIdx.x] : 0.f;
    sx = ce_scale(ce_block_max(m, red));
    m = parts[CE_AMAX_X + threadIdx.x];
    if (threadIdx.x < CE_AMAX_W - 256) m = fmaxf(m, parts[CE_AMAX_X + 256 + threadIdx.x]);
    sw = ce_scale(ce_block_max(m, red));
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) { k.scale[0] = sx; k.scale[1] = sw; }
  const int64_t per = d.Dp / 8, rows = d.Tp + (d.pack_w ? d.V : 0), n = rows * per;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t row = i / per;
    const int64_t c = (i - row * per) * 8;
    const bool isx = row < d.Tp;
    const int64_t t = isx ? row : row - d.Tp;
    const bool live = isx ? t < d.T && y[t] != ignore : true;
    const int64_t nv = live ? (d.D - c < 8 ? d.D - c : 8) : 0;
    unsigned short* dst = (isx ? k.x : k.w) + t * d.Dp + c;
    if (NP == 1) {
      const unsigned short* src = reinterpret_cast<const unsigned short*>(isx ? x : w) + t * d.D + c;
      g16_u32x4 v = {0u, 0u, 0u, 0u};
      if (nv == 8 && ((uintptr_t)src & 15) == 0) v = *reinterpret_cast<const g16_u32x4*>(src);
      else {
        unsigned short h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = e < nv ? src[e] : (unsigned short)0;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (unsigned)h[2 * e] | ((unsigned)h[2 * e + 1] << 16);
      }
      *reinterpret_cast<g16_u32x4*>(dst) = v;
    } else {
      const float* src = reinterpret_cast<const float*>(isx ? x : w) + t * d.D + c;
      const float s = isx ? sx : sw;
      float v[8];
      if (nv == 8 && ((uintptr_t)src & 15) == 0) {
        const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < nv ? src[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= s;
      g16_u32x4 hi, lo;
      g16_split8(v, hi, lo);
      *reinterpret_cast<g16_u32x4*>(dst) = hi;
      *reinterpret_cast<g16_u32x4*>(dst + (isx ? d.Tp : d.V) * d.Dp) = lo;
    }
  }
}

struct CeLogits {
  G16Op w, x;                  // P, Q
  const void* bias; const int64_t* y; const float* scale;
  int bias16, T, Tp, V, Dp, v0, tiles_r, tiles_c;
  float eps;
  float2* part; float* zsum; float* zy;              // forward: [tiles_v][Tp] (max, sum exp), sum of logits; the target's logit
  const float* lse; const float* wrow; unsigned short* G; int64_t ldg;       // backward
};

template <int NP, bool GRAD>
__global__ __launch_bounds__(256) void ce_logits_kernel(CeLogits p) {
  G16_SHARED
  __shared__ float sbias[G16_T];
  __shared__ float stat[3][2][G16_T];
  int tr, tc;
  g16_tile_of(blockIdx.x, p.tiles_r, p.tiles_c, tr, tc);
  const int r0 = p.v0 + tr * G16_T, c0 = tc * G16_T;            // the vocabulary is absolute here
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wid & 1, wc = wid >> 1, lh = lane >> 5;
  if (tid < G16_T) {
    float b = 0.f;
    if (p.bias && r0 + tid < p.V)
      b = p.bias16 ? g16_f32(reinterpret_cast<const unsigned short*>(p.bias)[r0 + tid]) : reinterpret_cast<const float*>(p.bias)[r0 + tid];
    sbias[tid] = b;
  }
  g16_f32x16 acc[2][2];
  g16_tile<NP, false, false>(acc, p.w, p.x, r0, c0, 0, p.Dp, g16_p0, g16_q0, g16_p1, g16_q1);
  const float ix = NP == 2 ? 1.f / p.scale[0] : 1.f, iw = NP == 2 ? 1.f / p.scale[1] : 1.f;       // powers of two: exact
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int eb = 0; eb < 4; ++eb) {
      const float4 b = *reinterpret_cast<const float4*>(sbias + g16_r(wr, i, eb * 4, lane));
      const float bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][eb * 4 + e] = (NP == 2 ? acc[i][j][eb * 4 + e] * ix * iw : acc[i][j][eb * 4 + e]) + bb[e];
    }
  const int nv = p.V - r0;                                      // rows of this tile inside the vocabulary
  int yl[2];                                                    // the target's row in this tile, or none
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int c = c0 + g16_c(wc, j, lane);
    const int64_t y = c < p.T ? p.y[c] : -1;
    yl[j] = y >= r0 && y < r0 + G16_T && y < p.V ? (int)(y - r0) : -1;
  }
  if constexpr (!GRAD) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float m = -INFINITY, z = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int r = g16_r(wr, i, e, lane);
          const float v = acc[i][j][e];
          if (r < nv) { m = v > m || v != v ? v : m; z += v; }
          if (r == yl[j]) p.zy[c0 + g16_c(wc, j, lane)] = v;
        }
      const float om = __shfl_xor(m, 32, 64);
      m = om > m || om != om ? om : m;
      const float safe = m == -INFINITY ? 0.f : m;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) s += g16_r(wr, i, e, lane) < nv ? __expf(acc[i][j][e] - safe) : 0.f;
      s += __shfl_xor(s, 32, 64);
      z += __shfl_xor(z, 32, 64);
      if (lh == 0) {
        const int c = g16_c(wc, j, lane);
        stat[0][wr][c] = m; stat[1][wr][c] = s; stat[2][wr][c] = z;
      }
    }
    __syncthreads();
    if (tid < G16_T && c0 + tid < p.T) {
      const float m0 = stat[0][0][tid], m1 = stat[0][1][tid];
      const float m = m1 > m0 || m1 != m1 ? m1 : m0;
      const float safe = m == -INFINITY ? 0.f : m;
      const float s = stat[1][0][tid] * __expf(m0 - safe) + stat[1][1][tid] * __expf(m1 - safe);
      const int64_t at = (int64_t)tr * p.Tp + c0 + tid;
      p.part[at] = make_float2(m, s);
      if (p.zsum) p.zsum[at] = stat[2][0][tid] + stat[2][1][tid];
    }
  } else {
    float w[2], lse[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = c0 + g16_c(wc, j, lane);
      w[j] = c < p.T ? p.wrow[c] : 0.f;
      lse[j] = c < p.T ? p.lse[c] : 0.f;
    }
    const float ev = p.eps / (float)p.V, on = 1.f - p.eps;
    g16_store_tile(
        [&](int i, int j, int e) {
          const int r = g16_r(wr, i, e, lane);
          const float g = (__expf(acc[i][j][e] - lse[j]) - (r == yl[j] ? on : 0.f) - ev) * w[j];
          return r < nv && w[j] != 0.f ? g : 0.f;
        },
        [&](int c, int r, const float (&v)[8]) {
          const int64_t row = c0 + c, col = tr * G16_T + r;
          if (row >= p.Tp || col >= p.ldg) return;
          unsigned short* dst = p.G + row * p.ldg + col;
          if constexpr (NP == 1) {
            *reinterpret_cast<g16_u32x4*>(dst) = g16_bf16x8_of(v);
          } else {
            g16_u32x4 hi, lo;
            g16_split8(v, hi, lo);
            *reinterpret_cast<g16_u32x4*>(dst) = hi;
            *reinterpret_cast<g16_u32x4*>(dst + (int64_t)p.Tp * p.ldg) = lo;
          }
        },
        g16_p0, g16_q0, g16_p1, g16_q1);
  }
}

// joins the tiles' statistics: 64 tokens to a workgroup, four threads to a token
__global__ __launch_bounds__(256) void ce_join_kernel(const float2* __restrict__ part, const float* __restrict__ zsum, const float* __restrict__ zy,
                                                      const int64_t* __restrict__ y, int64_t ignore, int T, int64_t Tp, int V, int tiles,
                                                      float eps, float* __restrict__ lse, float* __restrict__ rows) {
  __shared__ float sm[3][4][64];
  const int l = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int t = blockIdx.x * 64 + l;
  float m = -INFINITY, s = 0.f, z = 0.f;
  if (t < T)
    for (int k = q; k < tiles; k += 4) {
      const float2 p = part[(int64_t)k * Tp + t];
      const float nm = p.x > m || p.x != p.x ? p.x : m;
      const float safe = nm == -INFINITY ? 0.f : nm;
      s = s * __expf(m - safe) + p.y * __expf(p.x - safe);
      m = nm;
      if (zsum) z += zsum[(int64_t)k * Tp + t];
    }
  sm[0][q][l] = m; sm[1][q][l] = s; sm[2][q][l] = z;
  __syncthreads();
  if (q != 0 || t >= T) return;
#pragma unroll
  for (int k = 1; k < 4; ++k) {
    const float om = sm[0][k][l];
    const float nm = om > m || om != om ? om : m;
    const float safe = nm == -INFINITY ? 0.f : nm;
    s = s * __expf(m - safe) + sm[1][k][l] * __expf(om - safe);
    m = nm;
    z += sm[2][k][l];
  }
  const float L = m + logf(s);
  const int64_t yt = y[t];
  float loss;
  if (yt == ignore) loss = 0.f;
  else if (yt < 0 || yt >= V) loss = NAN;                   // a target outside the vocabulary: loud, but no read out of range
  else {
    loss = L - (1.f - eps) * zy[t];
    if (eps != 0.f) loss -= eps * (z / (float)V);
  }
  lse[t] = L;
  rows[t] = loss;
}

// number of live rows and, for mean / sum, the loss: one workgroup, a fixed order
__global__ __launch_bounds__(1024) void ce_reduce_kernel(const float* __restrict__ rows, const int64_t* __restrict__ y, int64_t ignore, int T,
                                                         int reduction, float* __restrict__ loss, float* __restrict__ scale) {
  __shared__ double rs[16];
  __shared__ int rn[16];
  double s = 0.0;
  int n = 0;
  for (int t = threadIdx.x; t < T; t += 1024) {
    s += rows[t];
    n += y[t] != ignore;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    n += __shfl_xor(n, o, 64);
  }
  if ((threadIdx.x & 63) == 0) { rs[threadIdx.x >> 6] = s; rn[threadIdx.x >> 6] = n; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) { s += rs[i]; n += rn[i]; }
    scale[2] = (float)n;
    if (reduction == 1) *loss = (float)(s / (double)n);      // no live row: 0 / 0, a NaN, as a mean over nothing is
    else if (reduction == 2) *loss = (float)s;
  }
}

// w_t = dL/dloss_t (mean: g / live rows; sum: g; none: g_t), zero where the row does not count; two planes: times the power of two that
// brings the largest into [2^13, 2^14) (|G| <= |w|).  One workgroup; scal[0] = the power's reciprocal
__global__ __launch_bounds__(1024) void ce_weight_kernel(const float* __restrict__ grad, const int64_t* __restrict__ y, int64_t ignore, int T,
                                                         int64_t Tp, int V, int reduction, int planes, const float* __restrict__ scale,
                                                         float* __restrict__ wrow, float* __restrict__ scal) {
  __shared__ float red[16];
  const float n = scale[2];
  const float g0 = reduction ? grad[0] : 0.f;
  const float f = reduction == 1 ? (n > 0.f ? g0 / n : 0.f) : g0;
  auto weight = [&](int64_t t) {
    if (t >= T) return 0.f;
    const int64_t yt = y[t];
    if (yt == ignore || yt < 0 || yt >= V) return 0.f;
    return reduction ? f : grad[t];
  };
  float m = 0.f;
  if (planes == 2) {
    for (int64_t t = threadIdx.x; t < T; t += 1024) m = fmaxf(m, fabsf(weight(t)));
    m = ofq_wave_max(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int i = 0; i < 16; ++i) m = fmaxf(m, red[i]);
  }
  const float s = planes == 2 ? ce_scale(m) : 1.f;
  for (int64_t t = threadIdx.x; t < Tp; t += 1024) wrow[t] = weight(t) * s;
  if (threadIdx.x == 0) scal[0] = 1.f / s;
}

struct CeOut {
  G16Op P, Q;
  int R, C, K, tiles_r, tiles_c, split;
  float* part; int64_t slot;               // fp32 [split][C][R], accumulated into where acc is set
  int acc;
  void* out; int out16; int64_t ldo;       // else the final tensor, typed, times 1 / (scale * G's scale)
  const float* scale; const float* scal;
};

// n of eight values (n <= 8) to element `at` of a typed tensor, 16 bytes at a time where aligned
__device__ __forceinline__ void ce_put(void* out, int out16, int64_t at, int n, const float (&v)[8]) {
  if (out16) {
    unsigned short* o = reinterpret_cast<unsigned short*>(out) + at;
    if (n >= 8 && ((uintptr_t)o & 15) == 0) { *reinterpret_cast<g16_u32x4*>(o) = g16_bf16x8_of(v); return; }
#pragma unroll
    for (int e = 0; e < 8; ++e) if (e < n) o[e] = g16_bf16(v[e]);
  } else {
    float* o = reinterpret_cast<float*>(out) + at;
    if (n >= 8 && ((uintptr_t)o & 15) == 0) {
      *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) if (e < n) o[e] = v[e];
  }
}

// dx (QCOL false: P = W [k = v][r = d], Q = G [c = t][k = v]) and dW (QCOL true: P = x [k = t][r = d], Q = G [k = t][c = v])
template <int NP, bool QCOL>
__global__ __launch_bounds__(256) void ce_grad_kernel(CeOut p) {
  G16_SHARED
  int tr, tc;
  g16_tile_of(blockIdx.x, p.tiles_r, p.tiles_c, tr, tc);
  constexpr int BK = G16<NP>::BK;
  const int nk = p.K / BK, per = (nk + p.split - 1) / p.split;
  const int kb = min((int)blockIdx.y * per, nk), ke = min(kb + per, nk);
  g16_f32x16 acc[2][2];
  g16_tile<NP, true, QCOL>(acc, p.P, p.Q, tr * G16_T, tc * G16_T, kb * BK, ke * BK, g16_p0, g16_q0, g16_p1, g16_q1);
  const float a = NP == 2 ? 1.f / p.scale[0] : 1.f, b = p.part ? 1.f : p.scal[0];
  g16_store_tile([&](int i, int j, int e) { return acc[i][j][e]; },
                 [&](int c, int r, const float (&v0)[8]) {
                   const int64_t row = tc * G16_T + c;
                   const int col = tr * G16_T + r;
                   if (row >= p.C || col >= p.R) return;
                   float v[8];
                   if (p.part) {
                     float* o = p.part + blockIdx.y * p.slot + row * p.R + col;       // R and slot are multiples of 64
#pragma unroll
                     for (int e = 0; e < 8; ++e) v[e] = v0[e];
                     if (p.acc) {
                       const float4 x = *reinterpret_cast<const float4*>(o), y = *reinterpret_cast<const float4*>(o + 4);
                       v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
                     }
                     ce_put(o, 0, 0, 8, v);
                   } else {
#pragma unroll
                     for (int e = 0; e < 8; ++e) v[e] = v0[e] * a * b;
                     ce_put(p.out, p.out16, row * p.ldo + col, p.R - col, v);
                   }
                 },
                 g16_p0, g16_q0, g16_p1, g16_q1);
}

// dx = sum of the split's partials, in order, scaled and typed
__global__ __launch_bounds__(256) void ce_dx_kernel(const float* __restrict__ part, int64_t slot, int split, CeDims d, int planes,
                                                    const float* __restrict__ scale, const float* __restrict__ scal, void* __restrict__ dx,
                                                    int out16) {
  const int64_t per = d.Dp / 8, n = d.T * per;
  const float a = planes == 2 ? 1.f / scale[1] : 1.f, b = scal[0];
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t t = i / per, c = (i - t * per) * 8;
    if (c >= d.D) continue;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < split; ++s) {
      const float* p = part + s * slot + t * d.Dp + c;
      const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * a * b;
    ce_put(dx, out16, t * d.D + c, (int)min((int64_t)8, d.D - c), v);
  }
}

// column sums of G over the tokens: partials [gridDim.y][ldg], then the bias gradient
template <int NP>
__global__ __launch_bounds__(256) void ce_db_part_kernel(const unsigned short* __restrict__ G, int64_t Tp, int64_t ldg, float* __restrict__ part) {
  __shared__ float red[8][256];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int64_t col = (blockIdx.x * 32ll + cl) * 8;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (col < ldg)
    for (int64_t t = blockIdx.y * 8 + rl; t < Tp; t += gridDim.y * 8) {
      const g16_u32x4 a = *reinterpret_cast<const g16_u32x4*>(G + t * ldg + col);
      float v[8];
      if constexpr (NP == 2) {
        g16_join8(a, *reinterpret_cast<const g16_u32x4*>(G + (Tp + t) * ldg + col), v);
      } else {
        const g16_bf16x8 h = __builtin_bit_cast(g16_bf16x8, a);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)h[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += v[e];
    }
#pragma unroll
  for (int e = 0; e < 8; ++e) red[rl][cl * 8 + e] = s[e];
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) sum += red[k][threadIdx.x];
  const int64_t c = blockIdx.x * 256ll + threadIdx.x;
  if (c < ldg) part[blockIdx.y * ldg + c] = sum;
}
__global__ __launch_bounds__(256) void ce_db_kernel(const float* __restrict__ part, int64_t ldg, int ny, int n, const float* __restrict__ scal,
                                                    void* __restrict__ db, int out16, int64_t at) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  float s = 0.f;
  for (int k = 0; k < ny; ++k) s += part[k * ldg + c];
  s *= scal[0];
  if (out16) reinterpret_cast<unsigned short*>(db)[at + c] = g16_bf16(s);
  else reinterpret_cast<float*>(db)[at + c] = s;
}

static int ce_w_aligned(const void* w) { return ((uintptr_t)w & 15) == 0; }

extern "C" size_t ofq_linear_ce_kept_bytes(int64_t T, int64_t D, int64_t V, int bf16, int w_aligned) {
  CeDims d;
  if (!ce_dims(T, D, V, bf16, w_aligned, &d)) return 0;
  return ce_kept(nullptr, d).bytes;
}

struct CeFwdWs { float* amax; float2* part; float* zsum; float* zy; float* rows; size_t bytes; };
static CeFwdWs ce_fwd_ws(void* base, const CeDims& d) {
  CeFwdWs w;
  char* p = (char*)base;
  size_t at = 0;
  w.amax = (float*)(p + at); at += ce_up((CE_AMAX_X + CE_AMAX_W) * 4);
  w.zy = (float*)(p + at); at += ce_up(d.Tp * 4);
  w.rows = (float*)(p + at); at += ce_up(d.Tp * 4);
  w.part = (float2*)(p + at); at += ce_up((size_t)d.tiles_v * d.Tp * 8);
  w.zsum = (float*)(p + at); at += ce_up((size_t)d.tiles_v * d.Tp * 4);
  w.bytes = at;
  return w;
}

extern "C" size_t ofq_linear_ce_fwd_ws_bytes(int64_t T, int64_t D, int64_t V, int bf16) {
  CeDims d;
  if (!ce_dims(T, D, V, bf16, 1, &d)) return 0;
  return ce_fwd_ws(nullptr, d).bytes;
}

static G16Op ce_w_op(const CeDims& d, const CeKept& k, const void* w, int64_t v0, bool col) {
  const unsigned short* p = d.pack_w ? k.w : (const unsigned short*)w;
  return G16Op{p + (col ? v0 * d.Dp : 0), d.Dp, d.V * d.Dp, (int)(col ? d.V - v0 : d.V), (int)d.Dp};
}

// reduction: 0 none (loss [T]), 1 mean, 2 sum (loss: one float)
extern "C" int ofq_linear_ce_fwd(const void* x, const void* w, const void* bias, const int64_t* target, int64_t T, int64_t D, int64_t V,
                                 int bf16, int bias16, int64_t ignore_index, float smoothing, int reduction, float* loss, float* lse,
                                 void* kept, size_t kept_bytes, void* ws, size_t ws_bytes, ofq_stream_t stream) {
  CeDims d;
  if (!x || !w || !target || !loss || !lse || !kept || !ws || reduction < 0 || reduction > 2 || !(smoothing >= 0.f && smoothing <= 1.f) ||
      !ce_dims(T, D, V, bf16, ce_w_aligned(w), &d) || ((uintptr_t)kept & 255) || ((uintptr_t)ws & 255))
    return OFQ_EINVAL;
  const CeKept k = ce_kept(kept, d);
  const CeFwdWs f = ce_fwd_ws(ws, d);
  if (kept_bytes < k.bytes || ws_bytes < f.bytes) return OFQ_ENOWS;
  const int64_t tiles = d.tiles_v * d.tiles_t;
  if (tiles >= (1ll << 31)) return OFQ_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  if (!bf16) {
    hipLaunchKernelGGL(ce_amax_kernel, dim3(CE_AMAX_X + CE_AMAX_W), dim3(256), 0, st, (const float*)x, target, ignore_index, T, D,
                       (const float*)w, V * D, f.amax);
    OFQ_LAUNCH_CHECK();
  }
  const int64_t chunks = (d.Tp + (d.pack_w ? V : 0)) * (d.Dp / 8);
  const dim3 pg((unsigned)std::min<int64_t>(ceil_div(chunks, 256), 4096));
  if (bf16) hipLaunchKernelGGL(ce_pack_kernel<1>, pg, dim3(256), 0, st, x, target, ignore_index, w, d, f.amax, k);
  else hipLaunchKernelGGL(ce_pack_kernel<2>, pg, dim3(256), 0, st, x, target, ignore_index, w, d, f.amax, k);
  OFQ_LAUNCH_CHECK();
  CeLogits a = {};
  a.w = ce_w_op(d, k, w, 0, false);
  a.x = G16Op{k.x, d.Dp, d.Tp * d.Dp, (int)d.Tp, (int)d.Dp};
  a.bias = bias; a.bias16 = bias16; a.y = target; a.scale = k.scale;
  a.T = (int)T; a.Tp = (int)d.Tp; a.V = (int)V; a.Dp = (int)d.Dp; a.eps = smoothing;
  a.tiles_r = (int)d.tiles_v; a.tiles_c = (int)d.tiles_t;
  a.part = f.part; a.zsum = smoothing != 0.f ? f.zsum : nullptr; a.zy = f.zy;
  if (bf16) hipLaunchKernelGGL((ce_logits_kernel<1, false>), dim3((unsigned)tiles), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((ce_logits_kernel<2, false>), dim3((unsigned)tiles), dim3(256), 0, st, a);
  OFQ_LAUNCH_CHECK();
  float* rows = reduction == 0 ? loss : f.rows;
  hipLaunchKernelGGL(ce_join_kernel, dim3((unsigned)ceil_div(T, 64)), dim3(256), 0, st, f.part, a.zsum, f.zy, target, ignore_index, (int)T,
                     d.Tp, (int)V, (int)d.tiles_v, smoothing, lse, rows);
  OFQ_LAUNCH_CHECK();
  hipLaunchKernelGGL(ce_reduce_kernel, dim3(1), dim3(1024), 0, st, rows, target, ignore_index, (int)T, reduction, loss, k.scale);
  OFQ_LAUNCH_CHECK();
  return 0;
}

struct CeBwd { int64_t piece, pieces; int split, ny; float* scal; float* wrow; unsigned short* G; float* part; int64_t slot; float* db; size_t bytes; };
static CeBwd ce_bwd_ws(void* base, const CeDims& d, bool want_dx, bool want_db) {
  CeBwd b;
  const int64_t vp = ceil_div(d.V, G16_T) * G16_T;
  b.piece = std::min(vp, std::max<int64_t>(CE_PIECE_BYTES / (d.Tp * 2 * d.np) / G16_T * G16_T, G16_T));
  b.pieces = ceil_div(vp, b.piece);
  b.piece = ceil_div(ceil_div(vp, b.pieces), G16_T) * G16_T;             // pieces of one size
  b.pieces = ceil_div(vp, b.piece);
  // dx has few tiles and a long k: split it until two workgroups to a CU have work, at no less than eight k-steps each
  const int64_t tiles = d.tiles_t * ceil_div(d.D, G16_T), steps = b.piece / (d.np == 1 ? 64 : 32);
  b.split = tiles >= 384 ? 1 : (int)std::max<int64_t>(1, std::min(ceil_div(512, tiles), steps / 8));
  b.ny = (int)std::max<int64_t>(1, std::min<int64_t>(d.Tp / 64, 32));
  char* p = (char*)base;
  size_t at = 0;
  b.scal = (float*)p; at += 256;
  b.wrow = (float*)(p + at); at += ce_up(d.Tp * 4);
  b.G = (unsigned short*)(p + at); at += ce_up((size_t)d.np * d.Tp * b.piece * 2);
  b.slot = d.T * d.Dp;
  b.part = (float*)(p + at); if (want_dx) at += ce_up((size_t)b.split * b.slot * 4);
  b.db = (float*)(p + at); if (want_db) at += ce_up((size_t)b.ny * b.piece * 4);
  b.bytes = at;
  return b;
}

extern "C" size_t ofq_linear_ce_bwd_ws_bytes(int64_t T, int64_t D, int64_t V, int bf16, int want_dx, int want_db) {
  CeDims d;
  if (!ce_dims(T, D, V, bf16, 1, &d)) return 0;
  return ce_bwd_ws(nullptr, d, want_dx != 0, want_db != 0).bytes;
}

// grad: the incoming gradient, one float or (reduction 0) [T]; lse and kept as the forward pass left them; dx / dw / db: any may be NULL
extern "C" int ofq_linear_ce_bwd(const float* grad, const void* w, const void* bias, const int64_t* target, const float* lse, const void* kept,
                                 int64_t T, int64_t D, int64_t V, int bf16, int bias16, int64_t ignore_index, float smoothing, int reduction,
                                 void* dx, void* dw, void* db, void* ws, size_t ws_bytes, ofq_stream_t stream) {
  CeDims d;
  if (!grad || !w || !target || !lse || !kept || !ws || reduction < 0 || reduction > 2 || !(smoothing >= 0.f && smoothing <= 1.f) ||
      !ce_dims(T, D, V, bf16, ce_w_aligned(w), &d) || ((uintptr_t)kept & 255) || ((uintptr_t)ws & 255))
    return OFQ_EINVAL;
  const CeKept k = ce_kept((void*)kept, d);
  const CeBwd b = ce_bwd_ws(ws, d, dx != nullptr, db != nullptr);
  if (ws_bytes < b.bytes) return OFQ_ENOWS;
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(ce_weight_kernel, dim3(1), dim3(1024), 0, st, grad, target, ignore_index, (int)T, d.Tp, (int)V, reduction, d.np, k.scale,
                     b.wrow, b.scal);
  OFQ_LAUNCH_CHECK();
  for (int64_t i = 0; i < b.pieces; ++i) {
    const int64_t v0 = i * b.piece, nv = std::min(b.piece, V - v0);
    const int64_t np64 = ceil_div(nv, G16_PAD) * G16_PAD;                 // k extent of dx, whole k-steps: G is zero behind the vocabulary
    CeLogits a = {};
    a.w = ce_w_op(d, k, w, 0, false);
    a.x = G16Op{k.x, d.Dp, d.Tp * d.Dp, (int)d.Tp, (int)d.Dp};
    a.bias = bias; a.bias16 = bias16; a.y = target; a.scale = k.scale;
    a.T = (int)T; a.Tp = (int)d.Tp; a.V = (int)V; a.Dp = (int)d.Dp; a.eps = smoothing; a.v0 = (int)v0;
    a.tiles_r = (int)ceil_div(nv, G16_T); a.tiles_c = (int)d.tiles_t;
    a.lse = lse; a.wrow = b.wrow; a.G = b.G; a.ldg = b.piece;
    const dim3 lg((unsigned)(a.tiles_r * a.tiles_c));
    if (bf16) hipLaunchKernelGGL((ce_logits_kernel<1, true>), lg, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((ce_logits_kernel<2, true>), lg, dim3(256), 0, st, a);
    OFQ_LAUNCH_CHECK();
    const int64_t gpl = d.Tp * b.piece;
    if (dw) {
      CeOut o = {};
      o.P = G16Op{k.x, d.Dp, d.Tp * d.Dp, (int)d.Tp, (int)d.Dp};
      o.Q = G16Op{b.G, b.piece, gpl, (int)d.Tp, (int)b.piece};
      o.R = (int)D; o.C = (int)nv; o.K = (int)d.Tp; o.split = 1;
      o.tiles_r = (int)ceil_div(D, G16_T); o.tiles_c = (int)ceil_div(nv, G16_T);
      o.out = (char*)dw + v0 * D * (bf16 ? 2 : 4); o.out16 = bf16; o.ldo = D; o.scale = k.scale; o.scal = b.scal;
      const dim3 g((unsigned)(o.tiles_r * o.tiles_c));
      if (bf16) hipLaunchKernelGGL((ce_grad_kernel<1, true>), g, dim3(256), 0, st, o);
      else hipLaunchKernelGGL((ce_grad_kernel<2, true>), g, dim3(256), 0, st, o);
      OFQ_LAUNCH_CHECK();
    }
    if (dx) {
      CeOut o = {};
      o.P = ce_w_op(d, k, w, v0, true);
      o.Q = G16Op{b.G, b.piece, gpl, (int)d.Tp, (int)b.piece};
      o.R = (int)d.Dp; o.C = (int)T; o.K = (int)np64; o.split = b.split;
      o.tiles_r = (int)ceil_div(d.Dp, G16_T); o.tiles_c = (int)d.tiles_t;
      o.part = b.part; o.slot = b.slot; o.acc = i > 0; o.scale = k.scale; o.scal = b.scal;
      const dim3 g((unsigned)(o.tiles_r * o.tiles_c), (unsigned)b.split);
      if (bf16) hipLaunchKernelGGL((ce_grad_kernel<1, false>), g, dim3(256), 0, st, o);
      else hipLaunchKernelGGL((ce_grad_kernel<2, false>), g, dim3(256), 0, st, o);
      OFQ_LAUNCH_CHECK();
    }
    if (db) {
      const dim3 g((unsigned)ceil_div(b.piece, 256), (unsigned)b.ny);
      if (bf16) hipLaunchKernelGGL(ce_db_part_kernel<1>, g, dim3(256), 0, st, b.G, d.Tp, b.piece, b.db);
      else hipLaunchKernelGGL(ce_db_part_kernel<2>, g, dim3(256), 0, st, b.G, d.Tp, b.piece, b.db);
      OFQ_LAUNCH_CHECK();
      hipLaunchKernelGGL(ce_db_kernel, dim3((unsigned)ceil_div(nv, 256)), dim3(256), 0, st, b.db, b.piece, b.ny, (int)nv, b.scal, db, bias16, v0);
      OFQ_LAUNCH_CHECK();
    }
  }
  if (dx) {
    const dim3 g((unsigned)std::min<int64_t>(ceil_div(T * (d.Dp / 8), 256), 8192));
    hipLaunchKernelGGL(ce_dx_kernel, g, dim3(256), 0, st, b.part, b.slot, b.split, d, d.np, k.scale, b.scal, dx, bf16);
    OFQ_LAUNCH_CHECK();
  }
  return 0;
}
