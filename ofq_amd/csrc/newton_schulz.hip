// Orthogonalising an update by Newton-Schulz products, for many matrices in each launch, and the optimiser step around it.
//   X = U / max(|U|_F, eps), rows <= columns (transposed otherwise);  steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X
// X, A and B live as two fp16 planes of the value times 2^10 (gemm16.h: fp32's precision; one plane lost 1e-2 of the result on a
// gradient of low rank, whose small singular values the chain multiplies by up to a^steps).  A and B are symmetric: only the
// tiles on and below the diagonal are computed, and written twice.
// Bound by the matrix cores from about 512 x 512 on (3 x 16-bit products for fp32's precision), by the launches' latency below.
#include "gemm16.h"

#define NS_SCALE 1024.f
#define NS_BLK 64                        // block of the elementwise passes
#define NS_PARTS 256                     // partial sums of squares of one matrix, at most
#define NS_UPLOAD 24                     // records to an upload launch (they travel in its arguments)

struct NsTensor {          // one entry per matrix of the host array handed to ofq_newton_schulz
  const void* g;           // [rows][cols] gradient / update, contiguous
  float* mom;              // momentum buffer, updated in place (optimiser form), or NULL
  void* out;               // the orthogonalised matrix (mom == NULL) or the parameter, updated in place
  int64_t rows, cols;
  float wscale, pad_;      // the parameter's own factor of the learning rate
};

struct NsRec {
  const void* g; float* mom; void* out;
  int64_t x0, x1, a, b;    // offsets of the planes in the workspace, in halves (x0 / x1 are swapped by the step's parity)
  int64_t part;            // first partial sum
  int rows, cols, m, n, mp, np;
  float wscale;
  int e0, p0;              // prefix sums over the matrices: elementwise blocks, partials,
  int s[3], u[3];          // symmetric tiles and X tiles of 64, 128 and 256
  int nparts, per;         // partial sums of this matrix, blocks to each
};

struct NsUpload { NsRec r[NS_UPLOAD]; };
__global__ void ns_upload_kernel(NsRec* dst, NsUpload u, int n) {
  const int words = n * (int)(sizeof(NsRec) / 4);
  for (int i = threadIdx.x; i < words; i += blockDim.x) reinterpret_cast<unsigned*>(dst)[i] = reinterpret_cast<const unsigned*>(u.r)[i];
}

// the matrix that workgroup `id` works on: the last record whose prefix is <= id
template <class F>
__device__ __forceinline__ const NsRec& ns_find(const NsRec* t, int n, int id, F&& first) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first(t[mid]) <= id) lo = mid; else hi = mid - 1;
  }
  return t[lo];
}

struct NsStep { float lr, decay, omm; int nesterov; };      // omm = 1 - momentum
struct NsChain { float a, b, c, eps; int steps; };

// |U|_F of a matrix, from its partial sums; all 256 threads
__device__ __forceinline__ double ns_norm_of(const NsRec& r, const double* __restrict__ parts) {
  __shared__ double red[4];
  double s = (int)threadIdx.x < r.nparts ? parts[r.part + threadIdx.x] : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return sqrt((red[0] + red[1]) + (red[2] + red[3]));
}
__device__ __forceinline__ double ns_divisor(double norm, float eps) { return norm > (double)eps || norm != norm ? norm : (double)eps; }

template <bool BF16>
__device__ __forceinline__ float ns_load(const void* g, int64_t i) {
  return BF16 ? g16_f32(reinterpret_cast<const unsigned short*>(g)[i]) : reinterpret_cast<const float*>(g)[i];
}

// m <- m + (1 - mu)(g - m), and the sum of squares of u = m or (Nesterov) m - (1 - mu)(m - g); doubles, so that neither tiny nor huge
// gradients leave the range of their squares.  HBM-bound: reads g and m, writes m: 25 million elements in 55 us, 5.4 TB/s.
template <bool BF16>
__global__ __launch_bounds__(256) void ns_norm_kernel(const NsRec* __restrict__ t, int n, NsStep st, const unsigned* __restrict__ guard,
                                                      double* __restrict__ parts) {
  if (guard != nullptr && (__hip_atomic_load(guard, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & 0x7fffffffu) != 0u) return;
  const NsRec r = ns_find(t, n, blockIdx.x, [](const NsRec& r) { return r.p0; });
  const int64_t total = (int64_t)r.rows * r.cols;
  const int64_t chunk = (int64_t)r.per * (NS_BLK * NS_BLK);
  const int64_t first = (int64_t)(blockIdx.x - r.p0) * chunk, end = min(total, first + chunk);
  double s = 0.0;
  const bool vec = !BF16 && ((((uintptr_t)r.g | (uintptr_t)r.mom) & 15) == 0);
  int64_t i = first + threadIdx.x;
  if (vec) {
    const int64_t end4 = first + ((end - first) & ~(int64_t)3);
    for (int64_t k = first + threadIdx.x * 4; k < end4; k += 1024) {
      const float4 g = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(r.g) + k);
      float u[4] = {g.x, g.y, g.z, g.w};
      if (r.mom) {
        const float4 m4 = *reinterpret_cast<const float4*>(r.mom + k);
        float m[4] = {m4.x, m4.y, m4.z, m4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m[e] = m[e] + st.omm * (u[e] - m[e]);
          u[e] = st.nesterov ? m[e] - st.omm * (m[e] - u[e]) : m[e];
        }
        *reinterpret_cast<float4*>(r.mom + k) = make_float4(m[0], m[1], m[2], m[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s += (double)u[e] * u[e];
    }
    i = end4 + threadIdx.x;
  }
  if (BF16 && ((uintptr_t)r.g & 15) == 0) {
    const int64_t end8 = first + ((end - first) & ~(int64_t)7);
    for (int64_t k = first + threadIdx.x * 8; k < end8; k += 2048) {
      const g16_u32x4 w = *reinterpret_cast<const g16_u32x4*>(reinterpret_cast<const unsigned short*>(r.g) + k);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = __uint_as_float(w[e] << 16), b = __uint_as_float(w[e] & 0xffff0000u);
        s += (double)a * a;
        s += (double)b * b;
      }
    }
    i = end8 + threadIdx.x;
  }
  for (; i < end; i += 256) {
    float u = ns_load<BF16>(r.g, i);
    if (r.mom) {
      const float m = r.mom[i] + st.omm * (u - r.mom[i]);
      r.mom[i] = m;
      u = st.nesterov ? m - st.omm * (m - u) : m;
    }
    s += (double)u * u;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  __shared__ double red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) parts[r.part + blockIdx.x - r.p0] = (red[0] + red[1]) + (red[2] + red[3]);
}

// Of a vector (one row or column) the chain is a scalar's, X = f U: f <- f (a + b A + c A A) with A = (f |U|)^2, here in 64 bits.  In planes and
// fp32 its error is one factor, common to all of the vector, that nothing averages: 1.1e-6 where plain fp32 products have 0.5e-6.
__device__ __forceinline__ double ns_vector_factor(double norm, const NsChain& ch) {
  double f = 1.0 / ns_divisor(norm, ch.eps);
  for (int k = 0; k < ch.steps; ++k) {
    const double q = (f * norm) * (f * norm);
    f *= ch.a + q * (ch.b + q * ch.c);
  }
  return f;
}

// X planes = u / max(|u|_F, eps) * 2^10, transposed where rows > columns, zero padded to [mp][np].  64 x 64 blocks through LDS.  25 million
// elements in 67 us, 3 TB/s: scalar loads, as either side may be the transposed one.
template <bool BF16>
__global__ __launch_bounds__(256) void ns_pack_kernel(const NsRec* __restrict__ t, int n, NsStep st, float eps,
                                                      const double* __restrict__ parts, _Float16* __restrict__ ws) {
  __shared__ float blk[NS_BLK][NS_BLK + 1];
  const NsRec r = ns_find(t, n, blockIdx.x, [](const NsRec& r) { return r.e0; });
  if (r.m == 1) return;
  const double norm = ns_norm_of(r, parts);
  // the factor as a power of two and a float in [0.5, 1): as one float it is Inf where norm and eps lie below 3e-36 (and 0 Inf a NaN), and has
  // no digits left where norm lies above 1e41
  int ex;
  const float inv = (float)frexp((double)NS_SCALE / ns_divisor(norm, eps), &ex);
  const int bc = r.np / NS_BLK, id = blockIdx.x - r.e0;
  const int xr = (id / bc) * NS_BLK, xc = (id % bc) * NS_BLK;          // block of X [mp][np]
  const bool tr = r.rows > r.cols;
  const int gr = tr ? xc : xr, gc = tr ? xr : xc;
  const int lc = threadIdx.x & 63;
#pragma unroll 4
  for (int lr = threadIdx.x >> 6; lr < NS_BLK; lr += 4) {
    const int i = gr + lr, j = gc + lc;
    float u = 0.f;
    if (i < r.rows && j < r.cols) {
      const int64_t at = (int64_t)i * r.cols + j;
      u = ns_load<BF16>(r.g, at);
      if (r.mom) {
        const float m = r.mom[at];
        u = st.nesterov ? m - st.omm * (m - u) : m;
      }
    }
    blk[lr][lc] = u;
  }
  __syncthreads();
  _Float16* hi = ws + r.x0;
  _Float16* lo = hi + (int64_t)r.mp * r.np;
  const int q = (threadIdx.x & 7) * 8;
#pragma unroll
  for (int row = threadIdx.x >> 3; row < NS_BLK; row += 32) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ldexpf(tr ? blk[q + e][row] : blk[row][q + e], ex) * inv;
    g16_u32x4 h, l;
    g16_split8(v, h, l);
    const int64_t at = (int64_t)(xr + row) * r.np + xc + q;
    *reinterpret_cast<g16_u32x4*>(hi + at) = h;
    *reinterpret_cast<g16_u32x4*>(lo + at) = l;
  }
}

// One tile (tr >= tc) of a symmetric matrix: A = X X^T (SQUARE false: k along X's rows) or B = b A + c A A (k along A's).
// Matrices of unlike lengths in one launch of X X^T wait for the longest tiles: cut along k into pieces (added up by the last to
// arrive) they were no faster, the pieces' way through memory costs what the balance gains.
// Matrix cores: twelve of 1024 x 1024 / 4096 113 us (X X^T, 690 TFLOP/s of plane products: its longest tiles are 128 k-steps) and 75 us
// (squares, 515: 432 tiles for 512 places); thirty of 384 / 1536 36 and 23 us, of which a tile's start and end are about half.
// Taking short matrices a product behind the long ones, so that one launch mixes short and long tiles, gained 2 % there and lost 20 % on
// the larger ones.
template <int CFG, bool SQUARE>
__global__ __launch_bounds__(g16_nt(CFG)) void ns_sym_kernel(const NsRec* __restrict__ t, int n, float fb, float fc, int odd, int run,
                                                             _Float16* __restrict__ ws) {
  using C = G16<2, CFG>;
  G16_SHARED(2, CFG)
  const int id = g16_xcd(blockIdx.x, gridDim.x, run);
  const NsRec& r = ns_find(t, n, id, [](const NsRec& r) { return r.s[C::SIZE]; });
  const int mp = r.mp;
  int tr, tc;
  g16_tri(id - r.s[C::SIZE], (mp + C::T - 1) / C::T, tr, tc);
  const int64_t pl = (int64_t)mp * (SQUARE ? mp : r.np);
  const unsigned short* src = reinterpret_cast<const unsigned short*>(ws) + (SQUARE ? r.a : odd ? r.x1 : r.x0);
  const int ld = SQUARE ? mp : r.np;
  const G16Op P = {src, ld, pl, mp, 0};
  G16Acc<2, CFG> acc;
  g16_tile<2, CFG, false, false>(acc, P, P, tr * C::T, tc * C::T, 0, ld, lds);
  const int64_t po = (int64_t)mp * mp;
  _Float16* out = ws + (SQUARE ? r.b : r.a);
  const _Float16* in = ws + r.a;
  const float alpha = (SQUARE ? fc : 1.f) / NS_SCALE;
  auto value = [&](int i, int j, int e) { return acc[i][j][e] * alpha; };
  auto put = [&](int row, int col, const float (&v0)[8]) {      // out[row][col .. col + 7]
    if (row >= mp || col >= mp) return;
    const int64_t at = (int64_t)row * mp + col;
    float v[8];
    if (SQUARE) {
      g16_join8(*reinterpret_cast<const g16_u32x4*>(in + at), *reinterpret_cast<const g16_u32x4*>(in + po + at), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fb * v[e] + v0[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v0[e];
    }
    g16_u32x4 h, l;
    g16_split8(v, h, l);
    *reinterpret_cast<g16_u32x4*>(out + at) = h;
    *reinterpret_cast<g16_u32x4*>(out + po + at) = l;
  };
  auto direct = [&](int c, int q, const float (&v)[8]) { put(tc * C::T + c, tr * C::T + q, v); };
  auto mirror = [&](int q, int c, const float (&v)[8]) { put(tr * C::T + q, tc * C::T + c, v); };
  if (tr == tc) g16_store_tile<2, CFG, false>(value, direct, mirror, lds);
  else g16_store_tile<2, CFG, true>(value, direct, mirror, lds);
}

// X <- a X + B X: r runs along the columns of X, c along its rows.  Matrix cores: twelve of 1024 x 1024 / 4096 181 us, 860 TFLOP/s of plane
// products; six of 2048 x 2048 / 8192 640 us, 970.
template <int CFG>
__global__ __launch_bounds__(g16_nt(CFG)) void ns_update_kernel(const NsRec* __restrict__ t, int n, float fa, int odd, _Float16* __restrict__ ws) {
  using C = G16<2, CFG>;
  G16_SHARED(2, CFG)
  const int id = g16_xcd(blockIdx.x, gridDim.x, CFG == G16_MID ? 64 : 32);
  const NsRec& r = ns_find(t, n, id, [](const NsRec& r) { return r.u[C::SIZE]; });
  const int mp = r.mp, np = r.np;
  int tr, tc;
  g16_group(id - r.u[C::SIZE], (np + C::T - 1) / C::T, (mp + C::T - 1) / C::T, tr, tc);
  const int64_t pl = (int64_t)mp * np;
  const _Float16* x = ws + (odd ? r.x1 : r.x0);
  _Float16* out = ws + (odd ? r.x0 : r.x1);
  const G16Op P = {reinterpret_cast<const unsigned short*>(x), np, pl, mp, np};
  const G16Op Q = {reinterpret_cast<const unsigned short*>(ws) + r.b, mp, (int64_t)mp * mp, mp, 0};
  G16Acc<2, CFG> acc;
  g16_tile<2, CFG, true, false>(acc, P, Q, tr * C::T, tc * C::T, 0, mp, lds);
  auto put = [&](int c, int q, const float (&v0)[8]) {
    const int row = tc * C::T + c, col = tr * C::T + q;
    if (row >= mp || col >= np) return;
    const int64_t at = (int64_t)row * np + col;
    float v[8];
    g16_join8(*reinterpret_cast<const g16_u32x4*>(x + at), *reinterpret_cast<const g16_u32x4*>(x + pl + at), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fa * v[e] + v0[e];
    g16_u32x4 h, l;
    g16_split8(v, h, l);
    *reinterpret_cast<g16_u32x4*>(out + at) = h;
    *reinterpret_cast<g16_u32x4*>(out + pl + at) = l;
  };
  g16_store_tile<2, CFG, false>([&](int i, int j, int e) { return acc[i][j][e] * (1.f / NS_SCALE); }, put, put, lds);
}

// out = O (the update's own type), or the parameter p <- p decay - lr wscale O; hyper: {lr, decay} from device memory (a captured
// step), guard: the step's guard word (see adamw.hip).  HBM-bound: 25 million elements in 64 us, 4.6 TB/s.
template <bool BF16>
__global__ __launch_bounds__(256) void ns_apply_kernel(const NsRec* __restrict__ t, int n, NsStep st, NsChain ch, const float* __restrict__ hyper,
                                                       const unsigned* __restrict__ guard, const double* __restrict__ parts,
                                                       const _Float16* __restrict__ ws) {
  if (guard != nullptr && (__hip_atomic_load(guard, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & 0x7fffffffu) != 0u) return;
  __shared__ float blk[NS_BLK][NS_BLK + 1];
  const NsRec r = ns_find(t, n, blockIdx.x, [](const NsRec& r) { return r.e0; });
  const float lr = hyper ? hyper[0] : st.lr, decay = hyper ? hyper[1] : st.decay;
  auto put = [&](int64_t at, float o) {
    if (r.mom) {
      float* p = reinterpret_cast<float*>(r.out) + at;
      *p = *p * decay - lr * r.wscale * o;
    } else if (BF16) {
      reinterpret_cast<unsigned short*>(r.out)[at] = g16_bf16(o);
    } else {
      reinterpret_cast<float*>(r.out)[at] = o;
    }
  };
  if (r.m == 1) {
    const double f = ns_vector_factor(ns_norm_of(r, parts), ch);
    const int at = (blockIdx.x - r.e0) * NS_BLK + (int)threadIdx.x;
    if (threadIdx.x < NS_BLK && at < r.n) {
      float u = ns_load<BF16>(r.g, at);
      if (r.mom) {
        const float m = r.mom[at];
        u = st.nesterov ? m - st.omm * (m - u) : m;
      }
      put(at, (float)(u * f));
    }
    return;
  }
  const int odd = ch.steps & 1;
  const int bc = r.np / NS_BLK, id = blockIdx.x - r.e0;
  const int xr = (id / bc) * NS_BLK, xc = (id % bc) * NS_BLK;
  const bool tr = r.rows > r.cols;
  const _Float16* hi = ws + (odd ? r.x1 : r.x0);
  const _Float16* lo = hi + (int64_t)r.mp * r.np;
  const int q = (threadIdx.x & 7) * 8;
#pragma unroll
  for (int row = threadIdx.x >> 3; row < NS_BLK; row += 32) {
    const int64_t at = (int64_t)(xr + row) * r.np + xc + q;
    float v[8];
    g16_join8(*reinterpret_cast<const g16_u32x4*>(hi + at), *reinterpret_cast<const g16_u32x4*>(lo + at), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (tr) blk[q + e][row] = v[e]; else blk[row][q + e] = v[e];
    }
  }
  __syncthreads();
  const int gr = tr ? xc : xr, gc = tr ? xr : xc;
  const int lc = threadIdx.x & 63;
#pragma unroll 4
  for (int l = threadIdx.x >> 6; l < NS_BLK; l += 4) {
    const int i = gr + l, j = gc + lc;
    if (i >= r.rows || j >= r.cols) continue;
    put((int64_t)i * r.cols + j, blk[l][lc] * (1.f / NS_SCALE));
  }
}

struct NsPlan {
  std::vector<NsRec> recs;
  int64_t halves = 0, parts = 0;
  bool alike = true;       // one length (of the matrices; vectors have no products)
  int blocks = 0, sym[3] = {0, 0, 0}, upd[3] = {0, 0, 0};        // tiles of 64, 128 and 256
};

// the workspace: [records][partial sums of squares][planes]
static int ns_plan(const NsTensor* ts, int64_t n, NsPlan* out) {
  if (!ts || n <= 0 || n > 65536) return OFQ_EINVAL;
  std::vector<int> order(n);
  for (int i = 0; i < n; ++i) {
    if (ts[i].rows <= 0 || ts[i].cols <= 0 || ts[i].rows > (1 << 20) || ts[i].cols > (1 << 20)) return OFQ_EINVAL;
    order[i] = i;
  }
  // long k loops first: a launch ends with its short tiles
  std::stable_sort(order.begin(), order.end(), [&](int x, int y) {
    return std::max(ts[x].rows, ts[x].cols) > std::max(ts[y].rows, ts[y].cols);
  });
  auto pad = [](int64_t v) { return (int)((v + G16_PAD - 1) / G16_PAD * G16_PAD); };
  int64_t blocks = 0, sym[3] = {0, 0, 0}, upd[3] = {0, 0, 0};
  int length = 0;
  for (int64_t k = 0; k < n; ++k) {
    const NsTensor& s = ts[order[k]];
    NsRec r = {};
    r.g = s.g; r.mom = s.mom; r.out = s.out; r.wscale = s.wscale;
    r.rows = (int)s.rows; r.cols = (int)s.cols;
    r.m = std::min(r.rows, r.cols); r.n = std::max(r.rows, r.cols);
    r.mp = pad(r.m); r.np = pad(r.n);
    const bool vector = r.m == 1;                        // (no planes and no products)
    const int64_t x = vector ? 0 : 2 * (int64_t)r.mp * r.np, a = vector ? 0 : 2 * (int64_t)r.mp * r.mp;
    r.x0 = out->halves; r.x1 = r.x0 + x; r.a = r.x1 + x; r.b = r.a + a;
    out->halves = r.b + a;
    const int64_t nb = (int64_t)(r.mp / NS_BLK) * (r.np / NS_BLK);
    r.per = (int)ceil_div(nb, NS_PARTS);
    r.nparts = (int)ceil_div((int64_t)r.rows * r.cols, (int64_t)r.per * NS_BLK * NS_BLK);
    r.part = out->parts;
    r.p0 = (int)out->parts;
    out->parts += r.nparts;
    r.e0 = (int)blocks; blocks += nb;
    for (int k3 = 0; k3 < 3; ++k3) {
      const int64_t tm = vector ? 0 : ceil_div(r.mp, 64 << k3), tn = vector ? 0 : ceil_div(r.np, 64 << k3);
      r.s[k3] = (int)sym[k3]; r.u[k3] = (int)upd[k3];
      sym[k3] += tm * (tm + 1) / 2;
      upd[k3] += tm * tn;
    }
    if (!vector && length && r.np != length) out->alike = false;
    if (!vector) length = r.np;
    if (blocks >= (1ll << 30) || sym[0] >= (1ll << 30) || upd[0] >= (1ll << 30)) return OFQ_EINVAL;
    out->recs.push_back(r);
  }
  out->blocks = (int)blocks;
  for (int k3 = 0; k3 < 3; ++k3) { out->sym[k3] = (int)sym[k3]; out->upd[k3] = (int)upd[k3]; }
  return 0;
}
static size_t ns_up(size_t b) { return (b + 255) & ~(size_t)255; }

static size_t ns_bytes(const NsPlan& p) {
  return ns_up(p.recs.size() * sizeof(NsRec)) + ns_up(p.parts * sizeof(double)) + ns_up(p.halves * 2);
}

extern "C" int64_t ofq_newton_schulz_entry_bytes(void) { return (int64_t)sizeof(NsTensor); }

extern "C" size_t ofq_newton_schulz_ws_bytes(const void* tensors, int64_t n) {
  try {
    NsPlan p;
    if (ns_plan((const NsTensor*)tensors, n, &p)) return 0;
    return ns_bytes(p);
  } catch (...) { return 0; }
}

// tensors: HOST array of n entries (NsTensor); bf16: the updates' (and, without momentum, the outputs') type.  See include/ofq_hip.h.
extern "C" int ofq_newton_schulz(const void* tensors, int64_t n, int bf16, int steps, float fa, float fb, float fc, float eps,
                                 float lr, float weight_decay, double momentum, int nesterov, const void* hyper_dev, const void* guard,
                                 void* ws, size_t ws_bytes, ofq_stream_t stream) {
  try {
    const NsTensor* ts = (const NsTensor*)tensors;
    NsPlan p;
    if (steps < 0 || steps > 100 || !(eps > 0.f)) return OFQ_EINVAL;
    if (int rc = ns_plan(ts, n, &p)) return rc;
    for (int64_t i = 0; i < n; ++i) {
      if (!ts[i].g || !ts[i].out || (bf16 && ts[i].mom) || (ts[i].mom != nullptr) != (ts[0].mom != nullptr)) return OFQ_EINVAL;
    }
    if (!ws || ((uintptr_t)ws & 255) || ws_bytes < ns_bytes(p)) return OFQ_ENOWS;
    char* at = (char*)ws;
    NsRec* recs = (NsRec*)at; at += ns_up(n * sizeof(NsRec));
    double* parts = (double*)at; at += ns_up(p.parts * sizeof(double));
    _Float16* planes = (_Float16*)at;
    hipStream_t st = (hipStream_t)stream;
    for (int64_t i = 0; i < n; i += NS_UPLOAD) {
      NsUpload u;
      const int k = (int)std::min<int64_t>(NS_UPLOAD, n - i);
      memset(&u, 0, sizeof(u));
      for (int j = 0; j < k; ++j) u.r[j] = p.recs[i + j];
      hipLaunchKernelGGL(ns_upload_kernel, dim3(1), dim3(256), 0, st, recs + i, u, k);
      OFQ_LAUNCH_CHECK();
    }
    NsStep s = {lr, 1.f - lr * weight_decay, (float)(1.0 - momentum), nesterov};
    const float* hyper = (const float*)hyper_dev;
    const int nn = (int)n;
    const unsigned* gd = (const unsigned*)guard;
    if (bf16) hipLaunchKernelGGL(ns_norm_kernel<true>, dim3((unsigned)p.parts), dim3(256), 0, st, recs, nn, s, gd, parts);
    else hipLaunchKernelGGL(ns_norm_kernel<false>, dim3((unsigned)p.parts), dim3(256), 0, st, recs, nn, s, gd, parts);
    OFQ_LAUNCH_CHECK();
    if (bf16) hipLaunchKernelGGL(ns_pack_kernel<true>, dim3(p.blocks), dim3(256), 0, st, recs, nn, s, eps, parts, planes);
    else hipLaunchKernelGGL(ns_pack_kernel<false>, dim3(p.blocks), dim3(256), 0, st, recs, nn, s, eps, parts, planes);
    OFQ_LAUNCH_CHECK();
    // unlike lengths: DEEP, in which a long tile alone on a CU is fastest, and short runs (thirty matrices of 384 x 384 and 384 x 1536:
    // 40 us, MID 50; six of 2048 x 2048 and 2048 x 8192: 390, MID 505, BIG 565)
    const int cs = g16_form(p.sym[0], p.sym[1], p.sym[2]), ca = p.alike || cs == G16_TINY ? cs : G16_DEEP, cu = g16_form(p.upd[0], p.upd[1], p.upd[2]);
    auto grid = [](const int (&tiles)[3], int form) { return dim3((unsigned)tiles[form == G16_TINY ? 0 : form == G16_BIG ? 2 : 1]); };
    const dim3 ga = grid(p.sym, ca), gs = grid(p.sym, cs), gu = grid(p.upd, cu);
    const int ra = p.alike ? 32 : 4;
    for (int k = 0; k < (p.upd[0] ? steps : 0); ++k) {
#define NS_SYM(CFG, SQ, GRID, RUN) hipLaunchKernelGGL((ns_sym_kernel<CFG, SQ>), GRID, dim3(g16_nt(CFG)), 0, st, recs, nn, fb, fc, k & 1, RUN, planes)
      if (ca == G16_BIG) NS_SYM(G16_BIG, false, ga, 32); else if (ca == G16_MID) NS_SYM(G16_MID, false, ga, 64);
      else if (ca == G16_DEEP) NS_SYM(G16_DEEP, false, ga, ra); else NS_SYM(G16_TINY, false, ga, ra);
      OFQ_LAUNCH_CHECK();
      if (cs == G16_BIG) NS_SYM(G16_BIG, true, gs, 32); else if (cs == G16_MID) NS_SYM(G16_MID, true, gs, 64);
      else if (cs == G16_DEEP) NS_SYM(G16_DEEP, true, gs, 32); else NS_SYM(G16_TINY, true, gs, 32);
      OFQ_LAUNCH_CHECK();
#undef NS_SYM
#define NS_UPD(CFG) hipLaunchKernelGGL(ns_update_kernel<CFG>, gu, dim3(g16_nt(CFG)), 0, st, recs, nn, fa, k & 1, planes)
      if (cu == G16_BIG) NS_UPD(G16_BIG); else if (cu == G16_MID) NS_UPD(G16_MID); else if (cu == G16_DEEP) NS_UPD(G16_DEEP); else NS_UPD(G16_TINY);
      OFQ_LAUNCH_CHECK();
#undef NS_UPD
    }
    const NsChain ch = {fa, fb, fc, eps, steps};
    if (bf16) hipLaunchKernelGGL(ns_apply_kernel<true>, dim3(p.blocks), dim3(256), 0, st, recs, nn, s, ch, hyper, gd, parts, planes);
    else hipLaunchKernelGGL(ns_apply_kernel<false>, dim3(p.blocks), dim3(256), 0, st, recs, nn, s, ch, hyper, gd, parts, planes);
    OFQ_LAUNCH_CHECK();
    return 0;
  } catch (...) { return OFQ_EINVAL; }
}
