// Softmax cross entropy of z = x W^T + b over a large vocabulary, from the hidden states on, without keeping the logits.
//   forward   lse_t = log sum_v exp z_tv, in one pass over the vocabulary: every tile of logits leaves (max, sum of
//             exp) per token, a second launch joins them;  loss_t = lse_t - (1 - e) z_t,y - e/V sum_v z_tv
//   backward  in pieces of the vocabulary: G = w_t (exp(z - lse_t) - (1 - e)[v = y_t] - e/V) for one piece, recomputed, in 16-bit
//             planes; dx += G W and dW = G^T x of that piece; db = column sums of G
// The tile computes z transposed (r = vocabulary, c = token): a lane holds 32 logits of one token, so the softmax statistics
// need one exchange between lane halves instead of five steps for each of 32 rows.
// bf16 tensors go to the matrix cores as they are, G is rounded to bf16 (off by up to 2^-8 relative, as the gradients themselves are; what
// all its rows have in common is left out of it, CeGrad; up to 64 rows it has two planes, ce_dims).  fp32 tensors are split into two fp16 planes scaled by a power of two taken from the
// tensor's largest element (gemm16.h); G's are scaled by 2^13.  Statistics, sums and partial gradients are fp32; exponentials are __expf's, off
// by 2^-22 (1 + |z - lse| / 4) of themselves, below the logits' own errors in them.
// Rows whose target is ignore_index are left out of all of it (CeRows): they cost nothing and what they hold (NaN, Inf) reaches nothing.
// Bound by the matrix cores: 8 n V D operations for n rows that count, of which the recomputation is 2 n V D (6 where the logits are kept,
// ce_z); for few rows by the reading of W.
#include "gemm16.h"

#define CE_AMAX_X 128                    // partial maxima of x and of W
#define CE_AMAX_W 384
#define CE_FINE G16_PAD                  // rows up to which G of bf16 tensors has two planes
// Rows up to which W is read as it is, without the matrix cores.  Few / not, us, both directions, V 65536, D 2048: bf16 1 row 191 / 225, 4 rows
// 246 / 310, 8 rows 464 / 313; fp32 (whose W would be packed) 1 row 362 / 850, 4 rows 387, 8 rows 542 / 857.
#define CE_FEW_16 4
#define CE_FEW 8
#define CE_PIECE_BYTES (128ll << 20)     // of G: half of the 256 MB last-level cache

static int ce_form(int64_t R, int64_t C, int split) {
  auto tiles = [&](int t) { return ceil_div(R, t) * ceil_div(C, t) * split; };
  return g16_form(tiles(64), tiles(128), tiles(256));
}

struct CeDims {
  int64_t T, D, V, Tp, Dp, Vp, tiles_v, tiles_t;
  int np, gp;                // planes of the operands, of G
  bool pack_w, few;
};
static bool ce_dims(int64_t T, int64_t D, int64_t V, int bf16, int w_aligned, CeDims* d) {
  if (T <= 0 || D <= 0 || V <= 0 || T > (1 << 24) || D > (1 << 20) || V > (1 << 24)) return false;
  auto pad = [](int64_t v) { return (v + G16_PAD - 1) / G16_PAD * G16_PAD; };
  d->T = T; d->D = D; d->V = V; d->Tp = pad(T); d->Dp = pad(D); d->Vp = pad(V);
  d->few = T <= (bf16 ? CE_FEW_16 : CE_FEW);
  d->tiles_v = ceil_div(V, d->few ? 64 : g16_t(ce_form(V, T, 1)));   // of the forward pass
  d->tiles_t = ceil_div(T, 64);                                      // at most
  d->np = bf16 ? 1 : 2;
  // G of few bf16 rows is held to 16 bits: where one row's rounding is not averaged with others' it showed in the whole gradient (two rows of
  // three classes: dx 2.3e-3 off, the rounding of the outputs alone 1.6e-3).  The second plane is a second k loop over the same W: 8 and 64
  // rows of 65536 x 2048 take 302 and 321 us with it, 1.9 and 2.0 times what three passes over W take (157).
  d->gp = bf16 && T > CE_FINE ? 1 : 2;
  d->pack_w = !d->few && (!bf16 || d->Dp != D || !w_aligned);
  return true;
}
static size_t ce_up(size_t b) { return (b + 255) & ~(size_t)255; }

// Pieces of the vocabulary in the backward pass, and the columns of one: all of it, or as many as give whole rounds of 256 tiles to the 256
// CUs in dW (and, for as many rows, in G), the last one what is left.  100000 columns of 4096, 4096 rows: seven of 14336 are 3.5 rounds
// each, 12.9 ms; six of 16384 and a rest 12.0.
static int64_t ce_pieces(const CeDims& d, int64_t* piece) {
  const int64_t vp = ceil_div(d.V, 128) * 128, most = std::max<int64_t>(CE_PIECE_BYTES / (d.Tp * 2 * d.gp) / 128 * 128, 128);
  const int64_t round = std::max<int64_t>(256 / ceil_div(d.D, 256), 1) * 256;
  *piece = vp <= most ? vp : most >= round ? most / round * round : most;
  return ceil_div(vp, *piece);
}
// Logits of a single piece are kept (its G takes as much again for a while) where the product takes longer than their way to memory and
// back; else they are computed a second time.  Kept / not, us, 2 directions: bf16, 64 x 65536, D 2048: 267 / 306; 509 x 21841, D 768:
// 160 / 168; 1024 x 16000, D 256: 112 / 104; fp32, D 768: 331 / 385; 1024 x 16000, D 256: 190 / 195; 700 x 20000, D 64: 123 / 115.
// Whole tiles, as they lie in the registers; 0: not kept.
static int64_t ce_z(const CeDims& d) {
  int64_t piece;
  if (ce_pieces(d, &piece) > 1 || d.Dp * (d.np == 2 ? 3 : 1) < 512) return 0;
  const int t = g16_t(ce_form(d.V, d.T, 1));
  const int64_t n = ceil_div(d.V, t) * ceil_div(d.T, t) * t * t;
  return n * 4 <= CE_PIECE_BYTES ? n : 0;
}

// What the forward pass leaves for the backward.  Rows whose target is ignore_index take no part in anything: the others are packed in
// their order, n of them.  Few rows (d.few): x in fp32, the logits [T][V].  Else W planes: zero padded to Vp rows; where W is used in place and its last rows do not fill G16_PAD, those, zero
// padded.
// [1]; row -> packed row or -1; packed -> row; target or -1; lse; fp32 in planes: a row's largest element (by row, those that count)
struct CeRows { int* n; int* pos; int* idx; int* y; float* lse; float* xmax; };
__host__ __device__ static inline int64_t ce_w_rows(const CeDims& d) { return d.pack_w ? d.Vp : d.Vp != d.V ? G16_PAD : 0; }
struct CeKept { float* scale; CeRows rows; unsigned short* x; unsigned short* w; float* z; size_t bytes; };
static CeKept ce_kept(void* base, const CeDims& d, bool backward) {
  CeKept k;
  char* p = (char*)base;
  size_t at = 0;
  k.scale = (float*)p; k.rows.n = (int*)p + 2; at += 256;            // scale: 2^Ex, 2^Ew
  k.rows.pos = (int*)(p + at); at += ce_up(d.Tp * 4);
  k.rows.idx = (int*)(p + at); at += ce_up(d.Tp * 4);
  k.rows.y = (int*)(p + at); at += ce_up(d.Tp * 4);
  k.rows.lse = (float*)(p + at); at += ce_up(d.Tp * 4);
  k.rows.xmax = (float*)(p + at); at += d.np == 2 && !d.few ? ce_up(d.Tp * 4) : 0;
  k.x = (unsigned short*)(p + at); at += d.few ? ce_up((size_t)CE_FEW * d.D * 4) : ce_up((size_t)d.np * d.Tp * d.Dp * 2);
  k.w = (unsigned short*)(p + at); at += d.few ? 0 : ce_up((size_t)d.np * ce_w_rows(d) * d.Dp * 2);
  const int64_t z = !backward ? 0 : d.few ? d.T * d.V : ce_z(d);
  k.z = z ? (float*)(p + at) : nullptr; at += ce_up((size_t)z * 4);
  k.bytes = at;
  return k;
}
// packed rows that are zero filled and multiplied
__device__ __forceinline__ int ce_padded(int n) { return max((n + G16_PAD - 1) / G16_PAD * G16_PAD, G16_PAD); }

__device__ __forceinline__ float ce_block_max(float m, float* red) {
  m = ofq_wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  const float r = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  return r;
}

// the power of two that brings m into [2^13, 2^14): two planes hold every element down to m 2^-13 with 2^-22 of it, and a
// rounding up stays far below fp16's 65504; 1 for 0, Inf and NaN.  It and its reciprocal are normal numbers.
__device__ __forceinline__ float ce_scale(float m) {
  const int ex = (int)((__float_as_uint(m) >> 23) & 0xffu) - 127;
  if (!(m > 0.f) || ex == 128) return 1.f;
  const int e = min(13 - ex, 126);                        // (-114 for the largest m)
  return __uint_as_float((unsigned)(e + 127) << 23);
}

// Numbers the rows that count, in order; one workgroup, eight times 64 rows to a wave a time.  rows_out: losses of reduction none, zero for
// the others (else NULL)
// One workgroup, 5 us up to 8192 rows, each further 8192 about 2: beside the launches around it the numbering by many workgroups and a
// second launch would be slower.
template <int NT>
__device__ __forceinline__ void ce_number(const int64_t* __restrict__ y, int64_t ignore, int64_t T, int V, CeRows k, float* __restrict__ rows_out) {
  __shared__ int count[NT / 64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  int first = 0;
  for (int64_t t0 = 0; t0 < T; t0 += NT * 8) {
    const int64_t at = t0 + wid * 512 + lane;
    int64_t v[8];
    int before[8], n = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = at + u * 64 < T ? y[at + u * 64] : ignore;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const unsigned long long live = __ballot(v[u] != ignore);
      before[u] = n + __popcll(live & ((1ull << lane) - 1));
      n += __popcll(live);
    }
    __syncthreads();
    if (lane == 0) count[wid] = n;
    __syncthreads();
    int base = first;
    for (int w = 0; w < NT / 64; ++w) {
      if (w < wid) base += count[w];
      first += count[w];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t t = at + u * 64;
      if (t >= T) continue;
      const bool live = v[u] != ignore;
      const int c = base + before[u];
      k.pos[t] = live ? c : -1;
      if (live) {
        k.idx[c] = (int)t;
        k.y[c] = v[u] < 0 || v[u] >= V ? -1 : (int)v[u];
      } else if (rows_out) {
        rows_out[t] = 0.f;
      }
    }
  }
  if (threadIdx.x == 0) *k.n = first;
}
__global__ __launch_bounds__(1024) void ce_number_kernel(const int64_t* __restrict__ y, int64_t ignore, int64_t T, int V, CeRows k,
                                                         float* __restrict__ rows_out) {
  ce_number<1024>(y, ignore, T, V, k, rows_out);
}

// Largest elements of x and W (fp32), and the numbering in one workgroup more.  Bound by memory: W of 21841 x 768 in 23 us, half of it
// from the last-level cache.
__global__ __launch_bounds__(256) void ce_amax_kernel(const float* __restrict__ x, const int64_t* __restrict__ y, int64_t ignore, int64_t T,
                                                      int64_t D, int V, const float* __restrict__ w, int64_t nw, float* __restrict__ parts,
                                                      CeRows k, float* __restrict__ rows_out) {
  __shared__ float red[4];
  float m = 0.f;
  if (blockIdx.x == CE_AMAX_X + CE_AMAX_W) {
    ce_number<256>(y, ignore, T, V, k, rows_out);
    return;
  }
  if (blockIdx.x < CE_AMAX_X) {
    for (int64_t t = blockIdx.x * 4 + (threadIdx.x >> 6); t < T; t += CE_AMAX_X * 4) {
      if (y[t] == ignore) continue;
      float r = 0.f;
      for (int64_t i = threadIdx.x & 63; i < D; i += 64) r = fmaxf(r, fabsf(x[t * D + i]));
      r = ofq_wave_max(r);
      if ((threadIdx.x & 63) == 0) k.xmax[t] = r;
      m = fmaxf(m, r);
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

// x (the rows that count, and zeros up to ce_padded of them) and, where it cannot be used in place, W into planes; one thread to eight
// elements of a row.  Bound by memory: 67 MB read and 67 written (21841 x 768 fp32) in 23 us, 5.9 TB/s.
template <int NP>
__global__ __launch_bounds__(256) void ce_pack_kernel(const void* __restrict__ x, const void* __restrict__ w, CeDims d, const float* __restrict__ parts,
                                                      CeKept k) {
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
  const int live_rows = *k.rows.n, padded = ce_padded(live_rows);
  const int64_t per = d.Dp / 8, rows = padded + ce_w_rows(d), n = rows * per;
  const int64_t wfirst = d.pack_w ? 0 : d.Vp - G16_PAD;       // the packed rows of W begin here
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t row = i / per;
    const int64_t c = (i - row * per) * 8;
    const bool isx = row < padded;
    const int64_t to = isx ? row : row - padded;
    const bool live = isx ? to < live_rows : to + wfirst < d.V;
    const int64_t t = !live ? 0 : isx ? k.rows.idx[to] : to + wfirst;
    const int64_t nv = live ? (d.D - c < 8 ? d.D - c : 8) : 0;
    unsigned short* dst = (isx ? k.x : k.w) + to * d.Dp + c;
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
      *reinterpret_cast<g16_u32x4*>(dst + (isx ? d.Tp : d.Vp) * d.Dp) = lo;
    }
  }
}

// The incoming gradient as the backward launches see it.  reduction mean / sum: one float for all rows; none: one a row.
// What all rows have in common is multiplied in fp32 at the end: G holds (exp(z - lse) - (1 - e)[v = y] - e/V) / unit.  A target's element,
// the one that carries a gradient, is then -1 for a class that is not learnt yet, which 16 bits hold exactly; 1/n or 1 - e rounded to bf16
// would be one relative error, up to 2^-9, common to all rows, that no sum averages (dW and dx of 4096 rows in bf16: 2.8e-3 from
// the formula in 64 bits, against 1.8e-3 so).
// A row's own gradient: bf16 G, whose exponents are fp32's, takes it along, over the largest (shared[0]).  fp32's two fp16 planes hold an
// element down to 2^-17 of the largest in full and none below 2^-38: rows' gradients of unlike size would cost the small rows of dx
// their digits (1e-6 of the largest: 2e-4 of that row's dx).  There G is without it; dx, a row at a time, is multiplied by it in
// fp32 at the end, and dW, db are sums over rows of it times x, times 1: x is packed once more with it (ce_weighted_kernel), scaled by what
// the largest of the products needs.  shared: [0] a power of two next to the largest gradient, [1] the packed products' scale, [2] that
// over x's own.
struct CeGrad {
  const float* grad; const int* n; const float* shared;
  int reduction;
  float eps;
};
__device__ __forceinline__ float ce_unit(float eps) { return eps <= 0.5f ? 1.f - eps : 1.f; }
// two planes: |G| <= 2^14, as the scaled operands are
template <int NP> __device__ __forceinline__ constexpr float ce_gscale() { return NP == 2 ? 8192.f : 1.f; }
// what the sums are multiplied by at the end (behind the planes' scales, which come off first: a power of two more next to a small factor would
// take its last places)
__device__ __forceinline__ float ce_factor(const CeGrad& g) {
  const float n = (float)*g.n;
  const float common = g.reduction == 0 ? g.shared[0] : g.reduction == 2 ? g.grad[0] : n > 0.f ? g.grad[0] / n : 0.f;
  return common * ce_unit(g.eps);
}
// of row t of dx
template <int NP> __device__ __forceinline__ float ce_factor_row(const CeGrad& g, int64_t t) {
  return NP == 2 && g.reduction == 0 ? g.grad[t] * ce_unit(g.eps) : ce_factor(g);
}
// a sum of nothing stays zero under an infinite gradient: rows that are ignored, classes behind a mask
__device__ __forceinline__ float ce_times(float v, float f) { return v == 0.f ? 0.f : v * f; }

struct CeLogits {
  G16Op w, x;                  // P, Q
  CeRows rows;
  const void* bias; const float* scale;
  float* z;                                          // tiles of logits as they lie in the registers, or NULL
  int bias16, Tp, V, Dp, v0, tiles_r, tiles_c;
  float eps;
  float2* part; float* zsum; float* zy;              // forward: [tiles_v][Tp] (max, sum exp), sum of logits; the target's logit
  CeGrad g; unsigned short* G; int64_t ldg;          // backward
  int gp;                                            // G's planes
  float* db;                                         // column sums of G's tiles [tiles_c][ldg], or NULL
};

// One tile of logits (r: classes, c: rows): their statistics, or (GRAD) G in planes and (DB) its column sums.  Bound by the matrix cores, with
// few features by the epilogue: 4096 x 100000 of 4096 bf16 2.8 ms (1140 TFLOP/s, 3891 rows count), G of 4096 x 16384 439 us; 1740 x
// 50021 of 1024 bf16 230 us (775); 509 x 21841 of 768 fp32 70 us (730 of the three products), G from kept logits 24 us.
template <int NP, int CFG, bool GRAD, bool DB>
__global__ __launch_bounds__(g16_nt(CFG)) void ce_logits_kernel(CeLogits p) {
  using C = G16<NP, CFG>;
  constexpr int TL = C::T;
  G16_SHARED(NP, CFG)
  __shared__ float sbias[TL];
  __shared__ float stat[3][2][TL];
  int tr, tc;
  g16_group(g16_xcd(blockIdx.x, gridDim.x, gridDim.x), p.tiles_r, p.tiles_c, tr, tc);
  const int r0 = p.v0 + tr * TL, c0 = tc * TL;            // the vocabulary is absolute here
  const int n = *p.rows.n;
  if (c0 >= ce_padded(n)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wid & 1, wc = wid >> 1, lh = lane >> 5;
  if (p.bias && tid < TL) {
    float b = 0.f;
    if (r0 + tid < p.V)
      b = p.bias16 ? g16_f32(reinterpret_cast<const unsigned short*>(p.bias)[r0 + tid]) : reinterpret_cast<const float*>(p.bias)[r0 + tid];
    sbias[tid] = b;
  }
  G16Acc<NP, CFG> acc;
  float* z = nullptr;                                     // (waves of no row have nothing to keep)
  if (p.z && c0 + g16_c<CFG>(wc, 0, 0) < n)
    z = p.z + (((int64_t)tr * p.tiles_c + tc) * (g16_nt(CFG) / 64) + wid) * (C::RB * C::CB * 1024) + lane * 4;
  if (GRAD && p.z) {
#pragma unroll
    for (int i = 0; i < C::RB; ++i)
#pragma unroll
      for (int j = 0; j < C::CB; ++j)
#pragma unroll
        for (int eb = 0; eb < 4; ++eb) {
          const float4 v = z ? *reinterpret_cast<const float4*>(z + ((i * C::CB + j) * 4 + eb) * 256) : make_float4(0.f, 0.f, 0.f, 0.f);
          acc[i][j][eb * 4] = v.x; acc[i][j][eb * 4 + 1] = v.y; acc[i][j][eb * 4 + 2] = v.z; acc[i][j][eb * 4 + 3] = v.w;
        }
    __syncthreads();
  } else {
    g16_tile<NP, CFG, false, false>(acc, p.w, p.x, r0, c0, 0, p.Dp, lds);
  }
  if (!GRAD && z) {
#pragma unroll
    for (int i = 0; i < C::RB; ++i)
#pragma unroll
      for (int j = 0; j < C::CB; ++j)
#pragma unroll
        for (int eb = 0; eb < 4; ++eb)
          *reinterpret_cast<float4*>(z + ((i * C::CB + j) * 4 + eb) * 256) =
              make_float4(acc[i][j][eb * 4], acc[i][j][eb * 4 + 1], acc[i][j][eb * 4 + 2], acc[i][j][eb * 4 + 3]);
  }
  // What few tiles need (a bias, rows past the vocabulary, a target) is passed over as a whole where it is not there: the epilogue of
  // 256 x 256 logits takes a wave's instructions as long as three k-steps.
  if constexpr (NP == 2) {
    // powers of two, taken off in one step: their product may lie outside fp32's range where the logit does not
    const int off = 254 - (int)(__float_as_uint(p.scale[0]) >> 23) - (int)(__float_as_uint(p.scale[1]) >> 23);
#pragma unroll
    for (int i = 0; i < C::RB; ++i)
#pragma unroll
      for (int j = 0; j < C::CB; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = ldexpf(acc[i][j][e], off);
  }
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < C::RB; ++i)
#pragma unroll
      for (int eb = 0; eb < 4; ++eb) {
        const float4 b = *reinterpret_cast<const float4*>(sbias + g16_r<CFG>(wr, i, eb * 4, lane));
        const float bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < C::CB; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][eb * 4 + e] += bb[e];
      }
  }
  const int nv = p.V - r0;                                          // rows of this tile inside the vocabulary
  int yl[C::CB];                                                    // the target's row in this tile where this lane holds it, or -1
#pragma unroll
  for (int j = 0; j < C::CB; ++j) {
    const int c = c0 + g16_c<CFG>(wc, j, lane);
    const int y = (c < n ? p.rows.y[c] : -1) - r0;
    yl[j] = y >= 0 && y < TL && y / (C::RB * 32) == wr && (y >> 2 & 1) == lh && y < nv ? y : -1;
  }
  if constexpr (!GRAD) {
    if (nv < TL) {
#pragma unroll
      for (int i = 0; i < C::RB; ++i)
#pragma unroll
        for (int j = 0; j < C::CB; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] = g16_r<CFG>(wr, i, e, lane) < nv ? acc[i][j][e] : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < C::CB; ++j) {
      float m = -INFINITY, s = 0.f, t = 0.f;
      // the largest that is no NaN; a NaN gets into the sum of exponentials by itself
#pragma unroll
      for (int i = 0; i < C::RB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float safe = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < C::RB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) s += __expf(acc[i][j][e] - safe);
      s += __shfl_xor(s, 32, 64);
      if (p.zsum) {
#pragma unroll
        for (int i = 0; i < C::RB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) t += g16_r<CFG>(wr, i, e, lane) < nv ? acc[i][j][e] : 0.f;
        t += __shfl_xor(t, 32, 64);
      }
      if (__any(yl[j] >= 0)) {
        float zy = 0.f;
#pragma unroll
        for (int i = 0; i < C::RB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) zy = g16_r<CFG>(wr, i, e, lane) == yl[j] ? acc[i][j][e] : zy;
        if (yl[j] >= 0) p.zy[c0 + g16_c<CFG>(wc, j, lane)] = zy;
      }
      if (lh == 0) {
        const int c = g16_c<CFG>(wc, j, lane);
        stat[0][wr][c] = m; stat[1][wr][c] = s; stat[2][wr][c] = t;
      }
    }
    __syncthreads();
    if (tid < TL && c0 + tid < n) {
      const float m0 = stat[0][0][tid], m1 = stat[0][1][tid];
      const float m = fmaxf(m0, m1);
      const float safe = m == -INFINITY ? 0.f : m;
      const float s = stat[1][0][tid] * __expf(m0 - safe) + stat[1][1][tid] * __expf(m1 - safe);
      const int64_t at = (int64_t)tr * p.Tp + c0 + tid;
      p.part[at] = make_float2(m, s);
      if (p.zsum) p.zsum[at] = stat[2][0][tid] + stat[2][1][tid];
    }
  } else {
    const bool weighted = NP == 2 && p.g.reduction == 0;
    const float unit = 1.f / ce_unit(p.eps), gs = NP == 2 || p.g.reduction ? ce_gscale<NP>() : 1.f / p.g.shared[0];
    float* srow = stat[0][0];                             // the rows' own gradients, for the column sums (a barrier lies in the store below)
    if (DB && weighted && tid < TL) srow[tid] = c0 + tid < n && p.rows.y[c0 + tid] >= 0 ? p.g.grad[p.rows.idx[c0 + tid]] * (1.f / p.g.shared[0]) : 0.f;
    const float ev = p.eps / (float)p.V * unit, on = (1.f - p.eps) * unit;
#pragma unroll
    for (int j = 0; j < C::CB; ++j) {
      const int c = c0 + g16_c<CFG>(wc, j, lane);
      const bool live = c < n && p.rows.y[c] >= 0;
      float w = !live ? 0.f : p.g.reduction ? gs : p.g.grad[p.rows.idx[c]] * gs, lse = live ? p.rows.lse[c] : 0.f;
      if (NP == 2 && !p.g.reduction) w = w == 0.f ? 0.f : gs;
      const float wu = w * unit, we = -ev * w, wy = -on * w;
#pragma unroll
      for (int i = 0; i < C::RB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = fmaf(__expf(acc[i][j][e] - lse), wu, we);
      if (__any(yl[j] >= 0)) {
#pragma unroll
        for (int i = 0; i < C::RB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] += g16_r<CFG>(wr, i, e, lane) == yl[j] ? wy : 0.f;
      }
      if (nv < TL || __any(w == 0.f)) {
#pragma unroll
        for (int i = 0; i < C::RB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] = g16_r<CFG>(wr, i, e, lane) < nv && w != 0.f ? acc[i][j][e] : 0.f;
      }
    }
    float colsum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    g16_store_tile<NP, CFG, false>(
        [&](int i, int j, int e) { return acc[i][j][e]; },
        [&](int c, int r, const float (&v)[8]) {
          const int64_t row = c0 + c, col = tr * TL + r;
          if constexpr (DB) {
            const float own = weighted ? srow[c] : 1.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) colsum[e] += v[e] * own;
          }
          if (row >= p.Tp || col >= p.ldg) return;
          unsigned short* dst = p.G + row * p.ldg + col;
          if constexpr (NP == 1) {
            const g16_u32x4 hi = g16_bf16x8_of(v);
            *reinterpret_cast<g16_u32x4*>(dst) = hi;
            if (p.gp == 2) {
              float rest[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) rest[e] = v[e] - __uint_as_float(e & 1 ? hi[e >> 1] & 0xffff0000u : hi[e >> 1] << 16);
              *reinterpret_cast<g16_u32x4*>(dst + (int64_t)p.Tp * p.ldg) = g16_bf16x8_of(rest);
            }
          } else {
            g16_u32x4 hi, lo;
            g16_split8(v, hi, lo);
            *reinterpret_cast<g16_u32x4*>(dst) = hi;
            *reinterpret_cast<g16_u32x4*>(dst + (int64_t)p.Tp * p.ldg) = lo;
          }
        },
        [](int, int, const float (&)[8]) {}, lds);
    if constexpr (DB) {
      // every thread has eight columns of the rows it stored; the sixteen threads of the same columns meet in LDS
      constexpr int PER = TL / 8, RR = g16_nt(CFG) / PER;
      g16_ldsf* red = (g16_ldsf*)lds.p[0];
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) red[(tid / PER) * TL + (tid % PER) * 8 + e] = colsum[e];
      __syncthreads();
      if (tid < TL && tr * TL + tid < p.ldg) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < RR; ++k) s += red[k * TL + tid];
        p.db[(int64_t)tc * p.ldg + tr * TL + tid] = s;
      }
    }
  }
}

// Joins the tiles' statistics, TOK tokens to a workgroup a time and NT / TOK threads to a token; ONE: one workgroup for all of it, and with
// it the reduction.
struct CeJoin {
  const float2* part; const float* zsum; const float* zy;
  CeRows k;
  int64_t Tp;
  int V, tiles, reduction;
  float eps;
  float* rows; float* loss;                          // rows: losses of the packed rows; reduction none: loss, of all rows
};

// the loss of mean / sum: one workgroup, a fixed order
template <int NT>
__device__ __forceinline__ void ce_reduce(const CeJoin& p) {
  __shared__ double rs[NT / 64];
  const int n = *p.k.n;
  double s = 0.0;
  for (int t = threadIdx.x; t < n; t += NT) s += p.rows[t];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) rs[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < NT / 64; ++i) s += rs[i];
    *p.loss = (float)(p.reduction == 1 ? s / (double)n : s);        // no row: 0 / 0, a NaN, as a mean over nothing is
  }
}

// 4 to 12 us: a latency, of one load and one exchange through LDS.  ONE up to 8192 statistics: 4.4 us where two launches take 9.
template <int NT, int TOK, bool ONE>
__global__ __launch_bounds__(NT) void ce_join_kernel(CeJoin p) {
  constexpr int PER = NT / TOK;
  __shared__ float sm[3][PER][TOK];
  const int l = threadIdx.x % TOK, q = threadIdx.x / TOK;
  const int n = *p.k.n;
  for (int t0 = blockIdx.x * TOK; t0 < n; t0 += gridDim.x * TOK) {
    const int t = t0 + l;
    float m = -INFINITY, s = 0.f, z = 0.f;
    if (t < n)
      for (int k = q; k < p.tiles; k += PER) {
        const float2 v = p.part[(int64_t)k * p.Tp + t];
        const float nm = fmaxf(m, v.x);
        const float safe = nm == -INFINITY ? 0.f : nm;
        s = s * __expf(m - safe) + v.y * __expf(v.x - safe);
        m = nm;
        if (p.zsum) z += p.zsum[(int64_t)k * p.Tp + t];
      }
    __syncthreads();
    sm[0][q][l] = m; sm[1][q][l] = s; sm[2][q][l] = z;
    for (int half = PER / 2; half > 0; half >>= 1) {
      __syncthreads();
      if (q < half) {
        const float om = sm[0][q + half][l];
        const float nm = fmaxf(m, om);
        const float safe = nm == -INFINITY ? 0.f : nm;
        s = s * __expf(m - safe) + sm[1][q + half][l] * __expf(om - safe);
        m = nm;
        z += sm[2][q + half][l];
        sm[0][q][l] = m; sm[1][q][l] = s; sm[2][q][l] = z;
      }
    }
    if (q == 0 && t < n) {
      const float L = m + logf(s);
      float loss = NAN;                              // a target outside the vocabulary: loud, but no read out of range
      if (p.k.y[t] >= 0) {
        loss = L - (1.f - p.eps) * p.zy[t];
        if (p.eps != 0.f) loss -= p.eps * (z / (float)p.V);
      }
      p.k.lse[t] = L;
      if (p.reduction) p.rows[t] = loss;
      else p.loss[p.k.idx[t]] = loss;
    }
  }
  if constexpr (ONE) {
    __syncthreads();
    if (p.reduction) ce_reduce<NT>(p);
  }
}
__global__ __launch_bounds__(1024) void ce_reduce_kernel(CeJoin p) { ce_reduce<1024>(p); }

// The largest of rows' own gradients (1 where that is 0, Inf or NaN, or it or its reciprocal no normal number): one workgroup
__global__ __launch_bounds__(1024) void ce_weight_kernel(const float* __restrict__ grad, CeRows k, float* __restrict__ shared) {
  __shared__ float red[16];
  float m = 0.f;
  for (int t = threadIdx.x; t < *k.n; t += 1024)
    if (k.y[t] >= 0) m = fmaxf(m, fabsf(grad[k.idx[t]]));
  m = ofq_wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) m = fmaxf(m, red[i]);
    shared[0] = m >= 0x1p-126f && m <= 0x1p126f ? m : 1.f;
  }
}

// The same for rows in planes: two passes over the rows, the second for the largest product of a row's gradient and its largest element.
// 333 rows: 3.7 us, a latency.
__global__ __launch_bounds__(1024) void ce_weight_rows_kernel(const float* __restrict__ grad, CeRows k, const float* __restrict__ scale, float* __restrict__ shared) {
  __shared__ float red[16];
  const int n = *k.n;
  auto largest = [&](auto&& of) {
    float m = 0.f;
    for (int t = threadIdx.x; t < n; t += 1024)
      if (k.y[t] >= 0) m = fmaxf(m, of(k.idx[t]));
    m = ofq_wave_max(m);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int i = 0; i < 16; ++i) m = fmaxf(m, red[i]);
    return m;
  };
  const float m = largest([&](int t) { return fabsf(grad[t]); });
  const int ex = (int)((__float_as_uint(m) >> 23) & 0xffu);
  const float w = !(m > 0.f) || ex == 255 ? 1.f : __uint_as_float((unsigned)min(max(ex, 1), 253) << 23);      // (its reciprocal is a float too)
  const float s = scale[0], xw = largest([&](int t) { return fabsf(grad[t]) * (1.f / w) * (k.xmax[t] * s); });
  const float f = fminf(ce_scale(xw), 0x1p126f / s);
  if (threadIdx.x == 0) { shared[0] = w; shared[1] = s * f; shared[2] = f; }
}

// x's planes times the rows' own gradients, for dW; rows without one (or with a target outside the vocabulary) are zeros, whatever x holds.
// 333 x 197: 3.9 us, a launch's latency; bound by memory, 4 bytes an element each way, where there are many rows.
__global__ __launch_bounds__(256) void ce_weighted_kernel(const float* __restrict__ grad, const unsigned short* __restrict__ x, CeDims d, CeRows k,
                                                          const float* __restrict__ shared, unsigned short* __restrict__ out) {
  const int rows = *k.n;
  const int64_t per = d.Dp / 8, n = ce_padded(rows) * per, plane = d.Tp * d.Dp;
  const float inv = 1.f / shared[0], f = shared[2];
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t row = i / per;
    const float w = row < rows && k.y[row] >= 0 ? grad[k.idx[row]] * inv : 0.f;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (w != 0.f) {
      g16_join8(*reinterpret_cast<const g16_u32x4*>(x + i * 8), *reinterpret_cast<const g16_u32x4*>(x + plane + i * 8), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * w * f;
    }
    g16_u32x4 hi, lo;
    g16_split8(v, hi, lo);
    *reinterpret_cast<g16_u32x4*>(out + i * 8) = hi;
    *reinterpret_cast<g16_u32x4*>(out + plane + i * 8) = lo;
  }
}

struct CeOut {
  G16Op P, Q;
  CeRows rows;
  const unsigned short* tail;              // dx: P's last G16_PAD rows of k where K ends in front of them, or NULL
  int R, C, K, tiles_r, tiles_c, split;
  int gp;                                  // G's planes: bf16 with two takes them one after the other
  float* part; int64_t slot;               // fp32 [split][C][R], accumulated into where acc is set
  int acc;
  void* out; int out16; int64_t ldo;       // else the final tensor, typed, times 1 / (scale * G's scale)
  const float* scale; CeGrad g;            // scale: of P
  const float* cols; int cols_tl;          // dW: the column sums that G's tiles of cols_tl rows left, or NULL; db: their sum
  void* db; int db16;
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

// one element of the bias gradient: the sums of a column over ce_padded(n) / TL tiles, in order
template <int NP>
__device__ __forceinline__ void ce_put_db(const float* __restrict__ cols, int64_t ldg, int TL, int c, const CeGrad& g, void* __restrict__ db, int out16) {
  float s = 0.f;
  const int ny = (ce_padded(*g.n) + TL - 1) / TL;
#pragma unroll 8
  for (int k = 0; k < ny; ++k) s += cols[k * ldg + c];
  s = ce_times(s * (1.f / ce_gscale<NP>()), ce_factor(g));
  if (out16) reinterpret_cast<unsigned short*>(db)[c] = g16_bf16(s);
  else reinterpret_cast<float*>(db)[c] = s;
}
// where no dW product takes it along
template <int NP>
__global__ __launch_bounds__(256) void ce_db_kernel(const float* __restrict__ cols, int64_t ldg, int TL, int n, CeGrad g, void* __restrict__ db, int out16) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c < n) ce_put_db<NP>(cols, ldg, TL, c, g, db, out16);
}

// dx (QCOL false: P = W [k = v][r = d], Q = G [c = t][k = v]) and dW (QCOL true: P = x [k = t][r = d], Q = G [k = t][c = v]); t: packed rows.
// A part of a split k has consecutive workgroups of one XCD, so that they take whole rows of W.  Bound by the matrix cores: 4096 x 16384 of
// 4096 bf16 dx 475 and dW 490 us (1100 and 1070 TFLOP/s); fp32 509 x 21841 of 768 61 and 80 us (840 and 640 of the three products: dW has
// 1026 tiles for 512 places).
template <int NP, int CFG, bool QCOL>
__global__ __launch_bounds__(g16_nt(CFG)) void ce_grad_kernel(CeOut p) {
  using C = G16<NP, CFG>;
  G16_SHARED(NP, CFG)
  const int id = g16_xcd(blockIdx.x, gridDim.x, gridDim.x), tiles = p.tiles_r * p.tiles_c, sp = id / tiles, n = *p.rows.n;
  int tr, tc;
  g16_group(id - sp * tiles, p.tiles_r, p.tiles_c, tr, tc);
  if constexpr (!QCOL) {
    if (!p.part) {                                   // dx itself: this tile's share of the rows that do not count
      constexpr int PER = C::T / 8;
      const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int i = threadIdx.x; i < C::T * PER; i += g16_nt(CFG)) {
        const int t = tc * C::T + i / PER, col = tr * C::T + i % PER * 8;
        if (t < p.C && col < p.R && p.rows.pos[t] < 0) ce_put(p.out, p.out16, t * p.ldo + col, p.R - col, zero);
      }
    }
    if (tc * C::T >= n) return;
  }
  constexpr int BK = C::BK;
  const int nk = (QCOL ? ce_padded(n) : p.K) / BK, per = (nk + p.split - 1) / p.split;
  const int kb = min(sp * per, nk), ke = min(kb + per, nk);
  G16Acc<NP, CFG> acc;
  g16_tile<NP, CFG, true, QCOL>(acc, p.P, p.Q, tr * C::T, tc * C::T, kb * BK, ke * BK, lds);
  if (NP == 1 && p.gp == 2) {
    const G16Op lo = {p.Q.p + p.Q.plane, p.Q.ld, 0, p.Q.rows, p.Q.cols};
    g16_tile<NP, CFG, true, QCOL, true>(acc, p.P, lo, tr * C::T, tc * C::T, kb * BK, ke * BK, lds);
  }
  if constexpr (!QCOL) {
    if (p.tail && sp + 1 == p.split) {
      const G16Op tp = {p.tail, p.P.ld, 0, G16_PAD, p.P.cols}, tq = {p.Q.p + p.K, p.Q.ld, p.Q.plane, p.Q.rows, p.Q.cols};
      g16_tile<NP, CFG, true, false, true>(acc, tp, tq, tr * C::T, tc * C::T, 0, G16_PAD, lds);
      if (NP == 1 && p.gp == 2) {
        const G16Op lo = {tq.p + tq.plane, tq.ld, 0, tq.rows, tq.cols};
        g16_tile<NP, CFG, true, false, true>(acc, tp, lo, tr * C::T, tc * C::T, 0, G16_PAD, lds);
      }
    }
  }
  const float a = NP == 2 ? 1.f / p.scale[0] * (1.f / ce_gscale<NP>()) : 1.f, b = ce_factor(p.g);
  g16_store_tile<NP, CFG, false>([&](int i, int j, int e) { return acc[i][j][e]; },
                 [&](int c, int r, const float (&v0)[8]) {
                   const int64_t row = tc * C::T + c;
                   const int col = tr * C::T + r;
                   if (row >= (QCOL ? p.C : n) || col >= p.R) return;
                   float v[8];
                   if (p.part) {
                     float* o = p.part + sp * p.slot + row * p.R + col;       // R and slot are multiples of 64
#pragma unroll
                     for (int e = 0; e < 8; ++e) v[e] = v0[e];
                     if (p.acc) {
                       const float4 x = *reinterpret_cast<const float4*>(o), y = *reinterpret_cast<const float4*>(o + 4);
                       v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
                     }
                     ce_put(o, 0, 0, 8, v);
                   } else {
                     const int64_t to = QCOL ? row : (int64_t)p.rows.idx[row];
                     const float f = QCOL || NP == 1 ? b : ce_factor_row<NP>(p.g, to);
#pragma unroll
                     for (int e = 0; e < 8; ++e) v[e] = ce_times(v0[e] * a, f);
                     ce_put(p.out, p.out16, to * p.ldo + col, p.R - col, v);
                   }
                 },
                 [](int, int, const float (&)[8]) {}, lds);
  if constexpr (QCOL) {
    const int c = tc * C::T + threadIdx.x;
    if (p.cols && tr == 0 && threadIdx.x < C::T && c < p.C) ce_put_db<NP>(p.cols, p.Q.ld, p.cols_tl, c, p.g, p.db, p.db16);
  }
}

// ---- few rows: without the matrix cores, W read as it is.  Bound by memory: W once for the logits, once for both gradients.
template <bool BF16> __device__ __forceinline__ float ce_load(const void* p, int64_t i) {
  if constexpr (BF16) return g16_f32(reinterpret_cast<const unsigned short*>(p)[i]);
  else return reinterpret_cast<const float*>(p)[i];
}
// N consecutive elements (8 or 16 bytes, aligned), as fp32
template <bool BF16, int N> __device__ __forceinline__ void ce_load_n(const void* p, int64_t i, float (&v)[N]) {
  if constexpr (BF16) {
    unsigned q[N / 2];
    const unsigned short* a = reinterpret_cast<const unsigned short*>(p) + i;
    if constexpr (N == 8) *reinterpret_cast<g16_u32x4*>(q) = *reinterpret_cast<const g16_u32x4*>(a);
    else *reinterpret_cast<uint2*>(q) = *reinterpret_cast<const uint2*>(a);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = __uint_as_float(e & 1 ? q[e >> 1] & 0xffff0000u : q[e >> 1] << 16);
  } else {
    const float* a = reinterpret_cast<const float*>(p) + i;
#pragma unroll
    for (int e = 0; e < N; e += 4) *reinterpret_cast<float4*>(v + e) = *reinterpret_cast<const float4*>(a + e);
  }
}

struct CeFew {
  const void* x; const void* w; const void* bias;
  CeRows k;
  float* xs; float* z;                               // kept: the rows that count in fp32 [CE_FEW][D]; logits [T][V], or NULL
  int64_t D;
  int bias16, Tp, T, V;
  float2* part; float* zsum; float* zy;
  CeGrad g;                                          // backward
  float* dxp; int64_t slot; void* dw; void* db;
  int per;
};

// Logits and their statistics, 64 classes to a workgroup, a wave to four classes a time, its lanes along D.  VEC: 16 bytes a load (every row of
// W and x is a multiple of that), else an element.  65536 x 2048 bf16, one row: 68 to 75 us, 3.6 to 3.9 TB/s.
template <bool BF16, bool VEC, int TT>
__global__ __launch_bounds__(256) void ce_few_logits_kernel(CeFew p) {
  constexpr int N = VEC ? (BF16 ? 8 : 4) : 1, U = TT > 2 ? 4 : 8;
  __shared__ float zs[TT][64];
  const int n = *p.k.n, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  if (blockIdx.x == 0)
    for (int t = 0; t < TT; ++t)
      for (int64_t i = threadIdx.x; i < p.D; i += 256) p.xs[t * p.D + i] = t < n ? ce_load<BF16>(p.x, (int64_t)p.k.idx[t] * p.D + i) : 0.f;
  int64_t row[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) row[t] = t < n ? (int64_t)p.k.idx[t] * p.D : -1;
  const int v0 = blockIdx.x * 64 + wid * 16;
  for (int g = 0; g < 16; g += U) {
    float acc[U][TT];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[u][t] = 0.f;
    int64_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = (int64_t)min(v0 + g + u, p.V - 1) * p.D;
#pragma unroll 2
    for (int64_t d = lane * N; d < p.D; d += 64 * N) {
      float w[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if constexpr (VEC) ce_load_n<BF16, N>(p.w, at[u] + d, w[u]);
        else w[u][0] = ce_load<BF16>(p.w, at[u] + d);
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        if (row[t] < 0) continue;
        float x[N];
        if constexpr (VEC) ce_load_n<BF16, N>(p.x, row[t] + d, x);
        else x[0] = ce_load<BF16>(p.x, row[t] + d);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < N; ++e) acc[u][t] = fmaf(w[u][e], x[e], acc[u][t]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        float a = acc[u][t];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
        if (lane == 0) zs[t][wid * 16 + g + u] = a;
      }
  }
  __syncthreads();
  const int v = blockIdx.x * 64 + lane;
  float b = 0.f;
  if (p.bias && v < p.V) b = p.bias16 ? ce_load<true>(p.bias, v) : ce_load<false>(p.bias, v);
  for (int t = wid; t < n; t += 4) {
    const float z = v < p.V ? zs[t][lane] + b : -INFINITY;
    if (v < p.V && p.z) p.z[(int64_t)t * p.V + v] = z;
    if (v < p.V && v == p.k.y[t]) p.zy[t] = z;
    float m = z, sum = v < p.V ? z : 0.f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    float e = __expf(z - (m == -INFINITY ? 0.f : m));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { e += __shfl_xor(e, o, 64); sum += __shfl_xor(sum, o, 64); }
    if (lane == 0) {
      const int64_t at = (int64_t)blockIdx.x * p.Tp + t;
      p.part[at] = make_float2(m, e);
      if (p.zsum) p.zsum[at] = sum;
    }
  }
}

// All gradients in one pass over W.  A thread has eight columns (four, with more than four rows) of x and of dx in registers and walks over the
// vocabulary: reads its columns of a row of W, adds G times them to dx, writes G times x to dW.  512 / per rows of W to a workgroup a time,
// `per` threads to a row (a power of two; blockIdx.y: further columns); every row group leaves a partial dx.  VEC: a thread's columns are
// consecutive (D is a multiple of 8); else they are `per` apart.  The loads have no conditions (columns past the end read column 0), or each would be waited for.
// One row against 65536 x 2048 bf16 reads and writes 268 MB each in 87 to 90 us, half of the reading from the last-level cache (a copy of as
// much through memory takes 105; two products on the matrix cores take 71 + 88).
template <int TT> constexpr int ce_few_columns() { return TT > 4 ? 4 : 8; }
template <bool BF16, bool VEC, int TT>
__global__ __launch_bounds__(512) void ce_few_kernel(CeFew p) {
  constexpr int N = ce_few_columns<TT>(), U = 4;
  const int r = threadIdx.x / p.per, rp = 512 / p.per, l = threadIdx.x % p.per, n = *p.k.n, D = (int)p.D;
  const int first = blockIdx.y * p.per * N;
  int col[N];
#pragma unroll
  for (int e = 0; e < N; ++e) col[e] = VEC ? first + l * N + e : first + e * p.per + l;
  float xs[TT][N], dx[TT][N], w[TT], lse[TT];
  int y[TT];
  const float unit = 1.f / ce_unit(p.g.eps), ev = p.g.eps / (float)p.V * unit, on = (1.f - p.g.eps) * unit, f = ce_factor(p.g);
  const bool finite = fabsf(f) <= 3e38f;             // (else the products are scaled one by one, zeros left alone)
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    y[t] = t < n ? p.k.y[t] : -1;
    const bool live = t < n && y[t] >= 0;
    w[t] = !live ? 0.f : p.g.reduction ? 1.f : p.g.grad[p.k.idx[t]] / p.g.shared[0];
    lse[t] = live ? p.k.lse[t] : 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      xs[t][e] = col[e] < D ? p.xs[t * p.D + col[e]] * (finite ? f : 1.f) : 0.f;
      dx[t][e] = 0.f;
    }
  }
  const int step = gridDim.x * rp;
  for (int v0 = blockIdx.x * rp + r; v0 < p.V; v0 += U * step) {
    float q[U][N], z[U][TT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * step < p.V ? v0 + u * step : v0;
      const int64_t at = v * p.D;
      if constexpr (VEC) {
        ce_load_n<BF16, N>(p.w, at + (col[0] < D ? col[0] : 0), q[u]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) q[u][e] = ce_load<BF16>(p.w, at + (col[e] < D ? col[e] : 0));
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) z[u][t] = p.z[(int64_t)(t < n ? t : 0) * p.V + v];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * step;
      if (v >= p.V) break;
      const int64_t at = v * p.D;
      float o[N], sum = 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = 0.f;
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        float gt = (__expf(z[u][t] - lse[t]) * unit - (v == y[t] ? on : 0.f) - ev) * w[t];
        gt = w[t] == 0.f ? 0.f : gt;
        sum += gt;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          dx[t][e] = fmaf(gt, q[u][e], dx[t][e]);
          o[e] = fmaf(gt, xs[t][e], o[e]);
        }
      }
      if (p.dw) {
        if (!finite) {
#pragma unroll
          for (int e = 0; e < N; ++e) o[e] = ce_times(o[e], f);
        }
        if constexpr (VEC) {
          if (col[0] < D) {                          // (D is a multiple of 8)
            if constexpr (BF16 && N == 8) {
              *reinterpret_cast<g16_u32x4*>(reinterpret_cast<unsigned short*>(p.dw) + at + col[0]) = g16_bf16x8_of(o);
            } else if constexpr (BF16) {
              const float o8[8] = {o[0], o[1], o[2], o[3], 0.f, 0.f, 0.f, 0.f};
              const g16_u32x4 h = g16_bf16x8_of(o8);
              *reinterpret_cast<uint2*>(reinterpret_cast<unsigned short*>(p.dw) + at + col[0]) = make_uint2(h[0], h[1]);
            } else {
#pragma unroll
              for (int e = 0; e < N; e += 4)
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.dw) + at + col[e]) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            if (col[e] >= D) continue;
            if constexpr (BF16) reinterpret_cast<unsigned short*>(p.dw)[at + col[e]] = g16_bf16(o[e]);
            else reinterpret_cast<float*>(p.dw)[at + col[e]] = o[e];
          }
        }
      }
      if (p.db && blockIdx.y == 0 && l == 0) {
        const float s = ce_times(sum, f);
        if (p.bias16) reinterpret_cast<unsigned short*>(p.db)[v] = g16_bf16(s);
        else reinterpret_cast<float*>(p.db)[v] = s;
      }
    }
  }
  if (!p.dxp) return;
#pragma unroll
  for (int t = 0; t < TT; ++t)
    if (t < n) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (col[e] < D) p.dxp[(int64_t)(blockIdx.x * rp + r) * p.slot + t * p.D + col[e]] = dx[t][e];
    }
}

// dx of few rows: 32 groups of threads share the many partials of eight columns and meet in LDS
__global__ __launch_bounds__(256) void ce_dx_few_kernel(const float* __restrict__ part, int64_t slot, int split, int64_t T, int64_t D, CeRows k, CeGrad g,
                                                        void* __restrict__ dx, int out16) {
  __shared__ float sums[32][8];
  const int64_t i = blockIdx.x * 8ll + threadIdx.x % 8, t = i / D, c = i - t * D;
  const int l = threadIdx.x % 8, q = threadIdx.x / 8;
  const int at = t < T ? k.pos[t] : -1, ns = at < 0 ? 0 : split;
  float v = 0.f;
  const float* p = part + at * D + c;
#pragma unroll 8
  for (int s = q; s < ns; s += 32) v += p[s * slot];
  sums[q][l] = v;
  for (int half = 16; half > 0; half >>= 1) {
    __syncthreads();
    if (q < half) sums[q][l] = v += sums[q + half][l];
  }
  if (q == 0 && t < T) {
    v = ce_times(v, ce_factor(g));
    if (out16) reinterpret_cast<unsigned short*>(dx)[i] = g16_bf16(v);
    else reinterpret_cast<float*>(dx)[i] = v;
  }
}

// dx = sum of the split's partials, in order, scaled and typed, and zeros in the rows that do not count
template <int NP>
__global__ __launch_bounds__(256) void ce_dx_kernel(const float* __restrict__ part, int64_t slot, int split, CeDims d, const float* __restrict__ scale,
                                                    CeRows k, CeGrad g, void* __restrict__ dx, int out16) {
  const int64_t per = d.Dp / 8, n = d.T * per;
  const float a = NP == 2 ? 1.f / scale[0] * (1.f / ce_gscale<NP>()) : 1.f;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t t = i / per, c = (i - t * per) * 8;
    if (c >= d.D) continue;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const int at = k.pos[t];
    const float* p = part + at * d.Dp + c;
    const int ns = at < 0 ? 0 : split;
#pragma unroll 8
    for (int s = 0; s < ns; ++s) {
      const float4 x = *reinterpret_cast<const float4*>(p + s * slot), y = *reinterpret_cast<const float4*>(p + s * slot + 4);
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
    const float b = ce_factor_row<NP>(g, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ce_times(v[e] * a, b);
    ce_put(dx, out16, t * d.D + c, (int)min((int64_t)8, d.D - c), v);
  }
}

static int ce_w_aligned(const void* w) { return ((uintptr_t)w & 15) == 0; }

extern "C" size_t ofq_linear_ce_kept_bytes(int64_t T, int64_t D, int64_t V, int bf16, int w_aligned, int backward) {
  CeDims d;
  if (!ce_dims(T, D, V, bf16, w_aligned, &d)) return 0;
  return ce_kept(nullptr, d, backward != 0).bytes;
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

static G16Op ce_w_op(const CeDims& d, const CeKept& k, const void* w, int64_t v0) {
  const unsigned short* p = d.pack_w ? k.w : (const unsigned short*)w;
  return G16Op{p + v0 * d.Dp, d.Dp, d.Vp * d.Dp, (int)(d.V - v0), (int)d.Dp};
}

// launches with the tile form of their grid: logits of V' columns (tv: tiles along them), gradient products
template <bool GRAD>
static int ce_logits(CeLogits& a, int64_t V, int64_t T, int bf16, int* tv, hipStream_t st) {
  const int form = ce_form(V, T, 1), t = g16_t(form);
  a.tiles_r = (int)ceil_div(V, t); a.tiles_c = (int)ceil_div(T, t);
  if (tv) *tv = a.tiles_r;
  const dim3 g((unsigned)(a.tiles_r * a.tiles_c));
#define CE_LOGITS(NP, CFG)                                                                                                    \
  do {                                                                                                                        \
    if (GRAD && a.db) hipLaunchKernelGGL((ce_logits_kernel<NP, CFG, GRAD, GRAD>), g, dim3(g16_nt(CFG)), 0, st, a);             \
    else hipLaunchKernelGGL((ce_logits_kernel<NP, CFG, GRAD, false>), g, dim3(g16_nt(CFG)), 0, st, a);                         \
  } while (0)
  if (bf16) { if (form == G16_BIG) CE_LOGITS(1, G16_BIG); else if (form == G16_MID) CE_LOGITS(1, G16_MID); else if (form == G16_DEEP) CE_LOGITS(1, G16_DEEP); else CE_LOGITS(1, G16_TINY); }
  else { if (form == G16_BIG) CE_LOGITS(2, G16_BIG); else if (form == G16_MID) CE_LOGITS(2, G16_MID); else if (form == G16_DEEP) CE_LOGITS(2, G16_DEEP); else CE_LOGITS(2, G16_TINY); }
#undef CE_LOGITS
  OFQ_LAUNCH_CHECK();
  return 0;
}
template <bool QCOL>
static int ce_grad(CeOut& o, int bf16, hipStream_t st) {
  const int form = ce_form(o.R, o.C, o.split), t = g16_t(form);
  o.tiles_r = (int)ceil_div(o.R, t); o.tiles_c = (int)ceil_div(o.C, t);
  const dim3 g((unsigned)(o.tiles_r * o.tiles_c * o.split));
#define CE_GRAD(NP, CFG) hipLaunchKernelGGL((ce_grad_kernel<NP, CFG, QCOL>), g, dim3(g16_nt(CFG)), 0, st, o)
  if (bf16) { if (form == G16_BIG) CE_GRAD(1, G16_BIG); else if (form == G16_MID) CE_GRAD(1, G16_MID); else if (form == G16_DEEP) CE_GRAD(1, G16_DEEP); else CE_GRAD(1, G16_TINY); }
  else { if (form == G16_BIG) CE_GRAD(2, G16_BIG); else if (form == G16_MID) CE_GRAD(2, G16_MID); else if (form == G16_DEEP) CE_GRAD(2, G16_DEEP); else CE_GRAD(2, G16_TINY); }
#undef CE_GRAD
  OFQ_LAUNCH_CHECK();
  return 0;
}

template <bool BF16, bool VEC>
static void ce_few_launch(const CeFew& a, bool backward, dim3 g, hipStream_t st) {
#define CE_FEW_ROWS(TT)                                                                                              \
  do {                                                                                                               \
    if (backward) hipLaunchKernelGGL((ce_few_kernel<BF16, VEC, TT>), g, dim3(512), 0, st, a);                         \
    else hipLaunchKernelGGL((ce_few_logits_kernel<BF16, VEC, TT>), g, dim3(256), 0, st, a);                           \
  } while (0)
  if (a.T == 1) CE_FEW_ROWS(1); else if (a.T == 2) CE_FEW_ROWS(2); else if (BF16 || a.T <= CE_FEW_16) CE_FEW_ROWS(4); else if constexpr (!BF16) CE_FEW_ROWS(8);
#undef CE_FEW_ROWS
}
static int ce_few(const CeFew& a, int bf16, const void* other, bool backward, dim3 g, hipStream_t st) {
  const bool vec = a.D % (bf16 || backward ? 8 : 4) == 0 && (((uintptr_t)a.w | (uintptr_t)other) & 15) == 0;
  if (bf16) { if (vec) ce_few_launch<true, true>(a, backward, g, st); else ce_few_launch<true, false>(a, backward, g, st); }
  else { if (vec) ce_few_launch<false, true>(a, backward, g, st); else ce_few_launch<false, false>(a, backward, g, st); }
  OFQ_LAUNCH_CHECK();
  return 0;
}

// reduction: 0 none (loss [T]), 1 mean, 2 sum (loss: one float)
extern "C" int ofq_linear_ce_fwd(const void* x, const void* w, const void* bias, const int64_t* target, int64_t T, int64_t D, int64_t V,
                                 int bf16, int bias16, int64_t ignore_index, float smoothing, int reduction, int backward, float* loss,
                                 void* kept, size_t kept_bytes, void* ws, size_t ws_bytes, ofq_stream_t stream) {
  CeDims d;
  if (!x || !w || !target || !loss || !kept || !ws || reduction < 0 || reduction > 2 || !(smoothing >= 0.f && smoothing <= 1.f) ||
      !ce_dims(T, D, V, bf16, ce_w_aligned(w), &d) || ((uintptr_t)kept & 255) || ((uintptr_t)ws & 255))
    return OFQ_EINVAL;
  const CeKept k = ce_kept(kept, d, backward != 0);
  const CeFwdWs f = ce_fwd_ws(ws, d);
  if (kept_bytes < k.bytes || ws_bytes < f.bytes) return OFQ_ENOWS;
  if (ceil_div(V, 64) * d.tiles_t >= (1ll << 31)) return OFQ_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  float* rows_out = reduction == 0 ? loss : nullptr;
  if (bf16 || d.few) hipLaunchKernelGGL(ce_number_kernel, dim3(1), dim3(1024), 0, st, target, ignore_index, T, (int)V, k.rows, rows_out);
  else hipLaunchKernelGGL(ce_amax_kernel, dim3(CE_AMAX_X + CE_AMAX_W + 1), dim3(256), 0, st, (const float*)x, target, ignore_index, T, D,
                          (int)V, (const float*)w, V * D, f.amax, k.rows, rows_out);
  OFQ_LAUNCH_CHECK();
  float* zsum = smoothing != 0.f ? f.zsum : nullptr;
  int tv;
  if (d.few) {
    CeFew a = {};
    a.x = x; a.w = w; a.bias = bias; a.bias16 = bias16; a.k = k.rows; a.xs = (float*)k.x; a.z = k.z;
    a.D = D; a.Tp = (int)d.Tp; a.T = (int)T; a.V = (int)V; a.part = f.part; a.zsum = zsum; a.zy = f.zy;
    tv = (int)d.tiles_v;
    if (int rc = ce_few(a, bf16, x, false, dim3((unsigned)tv), st)) return rc;
  } else {
    const int64_t chunks = (d.Tp + ce_w_rows(d)) * (d.Dp / 8);
    const dim3 pg((unsigned)std::min<int64_t>(ceil_div(chunks, 256), 4096));
    if (bf16) hipLaunchKernelGGL(ce_pack_kernel<1>, pg, dim3(256), 0, st, x, w, d, f.amax, k);
    else hipLaunchKernelGGL(ce_pack_kernel<2>, pg, dim3(256), 0, st, x, w, d, f.amax, k);
    OFQ_LAUNCH_CHECK();
    CeLogits a = {};
    a.w = ce_w_op(d, k, w, 0);
    a.x = G16Op{k.x, d.Dp, d.Tp * d.Dp, (int)d.Tp, (int)d.Dp};
    a.rows = k.rows; a.bias = bias; a.bias16 = bias16; a.scale = k.scale; a.z = k.z;
    a.Tp = (int)d.Tp; a.V = (int)V; a.Dp = (int)d.Dp; a.eps = smoothing;
    a.part = f.part; a.zsum = zsum; a.zy = f.zy;
    if (int rc = ce_logits<false>(a, V, T, bf16, &tv, st)) return rc;
  }
  const CeJoin j = {f.part, zsum, f.zy, k.rows, d.Tp, (int)V, tv, reduction, smoothing, f.rows, loss};
  // little to join: one workgroup does that and the sum, one launch less
  if (T * tv <= 8192) {
    if (tv <= 64) hipLaunchKernelGGL((ce_join_kernel<1024, 128, true>), dim3(1), dim3(1024), 0, st, j);
    else hipLaunchKernelGGL((ce_join_kernel<1024, 8, true>), dim3(1), dim3(1024), 0, st, j);
  } else {
    hipLaunchKernelGGL((ce_join_kernel<256, 8, false>), dim3((unsigned)std::min<int64_t>(ceil_div(T, 8), 65536)), dim3(256), 0, st, j);
    OFQ_LAUNCH_CHECK();
    if (reduction) hipLaunchKernelGGL(ce_reduce_kernel, dim3(1), dim3(1024), 0, st, j);
  }
  OFQ_LAUNCH_CHECK();
  return 0;
}

struct CeBwd {
  int64_t piece, pieces;
  int split, per, columns, blocks;
  float* shared; unsigned short* G; float* part; int64_t slot; float* db; unsigned short* xw; size_t bytes;
};
// want_weighted: dW of rows with gradients of their own
static CeBwd ce_bwd_ws(void* base, const CeDims& d, bool want_dx, bool want_db, bool want_weighted) {
  CeBwd b = {};
  if (d.few) {                                       // `per` threads to a row of W, at least four rows to each
    b.columns = d.T > 4 ? ce_few_columns<CE_FEW>() : ce_few_columns<1>();
    for (b.per = 8; b.per < 512 && b.per * b.columns < d.D; b.per *= 2) {}
    b.blocks = (int)std::max<int64_t>(1, std::min<int64_t>(256, ceil_div(d.V, 4 * (512 / b.per))));
    b.split = b.blocks * (512 / b.per);
    b.shared = (float*)base;
    b.part = (float*)((char*)base + 256);
    b.slot = d.T * d.D;
    b.bytes = 256 + (want_dx ? ce_up((size_t)b.split * b.slot * 4) : 0);
    return b;
  }
  b.pieces = ce_pieces(d, &b.piece);
  // dx has few tiles and a long k: split it so that two workgroups to a CU have work, and none waits for a place (24 tiles, k 21888, two
  // planes: 528 workgroups 86 us, 504 61), at no less than eight k-steps each
  const int64_t tiles = ceil_div(d.T, 128) * ceil_div(d.D, 128), steps = b.piece / (d.np == 1 ? 64 : 32);
  // (32 steps of the fp32 head of 1000 classes: 25 us at once, three parts 8 and 5 for the launch that joins them)
  b.split = (int)std::max<int64_t>(1, std::min(512 / tiles, steps / 8));
  char* p = (char*)base;
  size_t at = 0;
  b.shared = (float*)p; at += 256;
  b.G = (unsigned short*)(p + at); at += ce_up((size_t)d.gp * d.Tp * b.piece * 2);
  b.slot = d.T * d.Dp;
  b.part = b.split > 1 || b.pieces > 1 ? (float*)(p + at) : nullptr;                    // else dx is written by its product
  if (want_dx && b.part) at += ce_up((size_t)b.split * b.slot * 4);
  b.db = (float*)(p + at); if (want_db) at += ce_up((size_t)d.tiles_t * b.piece * 4);
  b.xw = (unsigned short*)(p + at); if (want_weighted && d.np == 2) at += ce_up((size_t)d.np * d.Tp * d.Dp * 2);
  b.bytes = at;
  return b;
}

extern "C" size_t ofq_linear_ce_bwd_ws_bytes(int64_t T, int64_t D, int64_t V, int bf16, int want_dx, int want_db) {
  CeDims d;
  if (!ce_dims(T, D, V, bf16, 1, &d)) return 0;
  return ce_bwd_ws(nullptr, d, want_dx != 0, want_db != 0, true).bytes;
}
extern "C" size_t ofq_linear_ce_bwd_call_ws_bytes(int64_t T, int64_t D, int64_t V, int bf16, int reduction, int want_dx, int want_dw, int want_db) {
  CeDims d;
  if (!ce_dims(T, D, V, bf16, 1, &d)) return 0;
  return ce_bwd_ws(nullptr, d, want_dx != 0, want_db != 0, reduction == 0 && want_dw != 0).bytes;
}

// grad: the incoming gradient, one float or (reduction 0) [T]; kept as a forward pass with backward != 0 left it; dx / dw / db: any may be NULL
extern "C" int ofq_linear_ce_bwd(const float* grad, const void* w, const void* bias, const void* kept, size_t kept_bytes, int64_t T, int64_t D,
                                 int64_t V, int bf16, int bias16, float smoothing, int reduction, void* dx, void* dw, void* db, void* ws,
                                 size_t ws_bytes, ofq_stream_t stream) {
  CeDims d;
  if (!grad || !w || !kept || !ws || reduction < 0 || reduction > 2 || !(smoothing >= 0.f && smoothing <= 1.f) ||
      !ce_dims(T, D, V, bf16, ce_w_aligned(w), &d) || ((uintptr_t)kept & 255) || ((uintptr_t)ws & 255))
    return OFQ_EINVAL;
  const CeKept k = ce_kept((void*)kept, d, true);
  if (kept_bytes != k.bytes) return OFQ_EINVAL;          // another size, or weights that moved to another alignment since
  const bool own = reduction == 0 && !bf16 && !d.few;    // rows' own gradients beside G, not in it
  const CeBwd b = ce_bwd_ws(ws, d, dx != nullptr, db != nullptr, own && dw != nullptr);
  if (ws_bytes < b.bytes) return OFQ_ENOWS;
  hipStream_t st = (hipStream_t)stream;
  if (own) {
    hipLaunchKernelGGL(ce_weight_rows_kernel, dim3(1), dim3(1024), 0, st, grad, k.rows, k.scale, b.shared);
    OFQ_LAUNCH_CHECK();
    if (dw) {
      const dim3 g((unsigned)std::min<int64_t>(ceil_div(d.Tp * (d.Dp / 8), 256), 4096));
      hipLaunchKernelGGL(ce_weighted_kernel, g, dim3(256), 0, st, grad, k.x, d, k.rows, b.shared, b.xw);
      OFQ_LAUNCH_CHECK();
    }
  } else if (reduction == 0) {
    hipLaunchKernelGGL(ce_weight_kernel, dim3(1), dim3(1024), 0, st, grad, k.rows, b.shared);
    OFQ_LAUNCH_CHECK();
  }
  const CeGrad cg = {grad, k.rows.n, b.shared, reduction, smoothing};
  if (d.few) {
    CeFew a = {};
    a.w = w; a.bias16 = bias16; a.k = k.rows; a.xs = (float*)k.x; a.z = k.z; a.D = D; a.T = (int)T; a.V = (int)V; a.g = cg;
    a.dxp = dx ? b.part : nullptr; a.slot = b.slot; a.dw = dw; a.db = db; a.per = b.per;
    if (int rc = ce_few(a, bf16, dw, true, dim3((unsigned)b.blocks, (unsigned)ceil_div(D, b.per * b.columns)), st)) return rc;
    if (dx) {
      hipLaunchKernelGGL(ce_dx_few_kernel, dim3((unsigned)ceil_div(T * D, 8)), dim3(256), 0, st, b.part, b.slot, b.split, T, D, k.rows, cg, dx, bf16);
      OFQ_LAUNCH_CHECK();
    }
    return 0;
  }
  for (int64_t i = 0; i < b.pieces; ++i) {
    const int64_t v0 = i * b.piece, nv = std::min(b.piece, V - v0);
    const bool tail = !d.pack_w && nv % G16_PAD;                          // (of the last piece: the others are whole tiles)
    const int64_t kdx = tail ? nv / G16_PAD * G16_PAD : ceil_div(nv, G16_PAD) * G16_PAD;       // G is zero behind the vocabulary
    CeLogits a = {};
    a.w = ce_w_op(d, k, w, 0);
    a.x = G16Op{k.x, d.Dp, d.Tp * d.Dp, (int)d.Tp, (int)d.Dp};
    a.rows = k.rows; a.bias = bias; a.bias16 = bias16; a.scale = k.scale; a.z = k.z;
    a.Tp = (int)d.Tp; a.V = (int)V; a.Dp = (int)d.Dp; a.eps = smoothing; a.v0 = (int)v0;
    a.g = cg; a.gp = d.gp; a.G = b.G; a.ldg = b.piece; a.db = db ? b.db : nullptr;
    if (int rc = ce_logits<true>(a, nv, T, bf16, nullptr, st)) return rc;
    const int64_t gpl = d.Tp * b.piece;
    if (dw) {
      CeOut o = {};
      o.rows = k.rows; o.gp = d.gp;
      o.P = G16Op{own ? b.xw : k.x, d.Dp, d.Tp * d.Dp, (int)d.Tp, (int)d.Dp};
      o.Q = G16Op{b.G, b.piece, gpl, (int)d.Tp, (int)b.piece};
      o.R = (int)D; o.C = (int)nv; o.K = (int)d.Tp; o.split = 1;
      o.out = (char*)dw + v0 * D * (bf16 ? 2 : 4); o.out16 = bf16; o.ldo = D; o.scale = own ? b.shared + 1 : k.scale; o.g = cg;
      if (db) {
        o.cols = b.db; o.cols_tl = g16_t(ce_form(nv, T, 1));
        o.db = (char*)db + v0 * (bias16 ? 2 : 4); o.db16 = bias16;
      }
      if (int rc = ce_grad<true>(o, bf16, st)) return rc;
    }
    if (dx) {
      CeOut o = {};
      o.rows = k.rows; o.gp = d.gp;
      o.P = ce_w_op(d, k, w, v0);
      o.Q = G16Op{b.G, b.piece, gpl, (int)d.Tp, (int)b.piece};
      o.C = (int)T; o.K = (int)kdx; o.split = b.split; o.tail = tail ? k.w : nullptr; o.scale = k.scale + 1; o.g = cg;
      if (b.part) { o.R = (int)d.Dp; o.part = b.part; o.slot = b.slot; o.acc = i > 0; }
      else { o.R = (int)D; o.out = dx; o.out16 = bf16; o.ldo = D; }
      if (int rc = ce_grad<false>(o, bf16, st)) return rc;
    }
    if (db && !dw) {
      const dim3 g((unsigned)ceil_div(nv, 256));
      const int tl = g16_t(ce_form(nv, T, 1));
      char* to = (char*)db + v0 * (bias16 ? 2 : 4);
      if (bf16) hipLaunchKernelGGL(ce_db_kernel<1>, g, dim3(256), 0, st, b.db, b.piece, tl, (int)nv, cg, to, bias16);
      else hipLaunchKernelGGL(ce_db_kernel<2>, g, dim3(256), 0, st, b.db, b.piece, tl, (int)nv, cg, to, bias16);
      OFQ_LAUNCH_CHECK();
    }
  }
  if (dx && b.part) {
    const int64_t chunks = T * (d.Dp / 8);
    const dim3 g((unsigned)std::min<int64_t>(ceil_div(chunks, 256), 8192));
    if (bf16) hipLaunchKernelGGL(ce_dx_kernel<1>, g, dim3(256), 0, st, b.part, b.slot, b.split, d, k.scale + 1, k.rows, cg, dx, bf16);
    else hipLaunchKernelGGL(ce_dx_kernel<2>, g, dim3(256), 0, st, b.part, b.slot, b.split, d, k.scale + 1, k.rows, cg, dx, bf16);
    OFQ_LAUNCH_CHECK();
  }
  return 0;
}
