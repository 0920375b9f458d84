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
  int e0, s0, x0t, p0;     // prefix sums over the matrices: elementwise blocks, symmetric tiles, X tiles, partials
  int nparts, per;         // partial sums of this matrix, blocks to each
};

struct NsUpload { NsRec r[NS_UPLOAD]; };
__global__ void ns_upload_kernel(NsRec* dst, NsUpload u, int n) {
  const int words = n * (int)(sizeof(NsRec) / 4);
  for (int i = threadIdx.x; i < words; i += blockDim.x) reinterpret_cast<unsigned*>(dst)[i] = reinterpret_cast<const unsigned*>(u.r)[i];
}

// the matrix that workgroup `id` works on: the last record whose prefix is <= id
template <int NsRec::*F>
__device__ __forceinline__ const NsRec& ns_find(const NsRec* t, int n, int id) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t[mid].*F <= id) lo = mid; else hi = mid - 1;
  }
  return t[lo];
}

struct NsStep { float lr, decay, omm; int nesterov; };      // omm = 1 - momentum

template <bool BF16>
__device__ __forceinline__ float ns_load(const void* g, int64_t i) {
  return BF16 ? g16_f32(reinterpret_cast<const unsigned short*>(g)[i]) : reinterpret_cast<const float*>(g)[i];
}

// m <- m + (1 - mu)(g - m), and the sum of squares of u = m or (Nesterov) m - (1 - mu)(m - g); doubles, so that neither tiny nor huge
// gradients leave the range of their squares.  HBM-bound: reads g and m, writes m.
template <bool BF16>
__global__ __launch_bounds__(256) void ns_norm_kernel(const NsRec* __restrict__ t, int n, NsStep st, const unsigned* __restrict__ guard,
                                                      double* __restrict__ parts) {
  if (guard != nullptr && (__hip_atomic_load(guard, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & 0x7fffffffu) != 0u) return;
  const NsRec r = ns_find<&NsRec::p0>(t, n, blockIdx.x);
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

// X planes = u / max(|u|_F, eps) * 2^10, transposed where rows > columns, zero padded to [mp][np].  64 x 64 blocks through LDS.
template <bool BF16>
__global__ __launch_bounds__(256) void ns_pack_kernel(const NsRec* __restrict__ t, int n, NsStep st, float eps,
                                                      const double* __restrict__ parts, _Float16* __restrict__ ws) {
  __shared__ float blk[NS_BLK][NS_BLK + 1];
  __shared__ double red[4];
  const NsRec r = ns_find<&NsRec::e0>(t, n, blockIdx.x);
  double s = (int)threadIdx.x < r.nparts ? parts[r.part + threadIdx.x] : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  const float inv = (float)((double)NS_SCALE / (norm > (double)eps || norm != norm ? norm : (double)eps));
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
    for (int e = 0; e < 8; ++e) v[e] = (tr ? blk[q + e][row] : blk[row][q + e]) * inv;
    g16_u32x4 h, l;
    g16_split8(v, h, l);
    const int64_t at = (int64_t)(xr + row) * r.np + xc + q;
    *reinterpret_cast<g16_u32x4*>(hi + at) = h;
    *reinterpret_cast<g16_u32x4*>(lo + at) = l;
  }
}

// A = X X^T (SQUARE false: K = np) or B = b A + c A A (SQUARE true: K = mp): one tile (tr >= tc) of a symmetric matrix
template <bool SQUARE>
__global__ __launch_bounds__(256) void ns_sym_kernel(const NsRec* __restrict__ t, int n, float fb, float fc, int odd, _Float16* __restrict__ ws) {
  G16_SHARED
  const NsRec& r = ns_find<&NsRec::s0>(t, n, blockIdx.x);
  const int id = blockIdx.x - r.s0;
  int tr = (int)((sqrtf(8.f * id + 1.f) - 1.f) * 0.5f);
  while ((tr + 1) * (tr + 2) / 2 <= id) ++tr;
  while (tr * (tr + 1) / 2 > id) --tr;
  const int tc = id - tr * (tr + 1) / 2;
  const int mp = r.mp;
  const int64_t pl = (int64_t)mp * (SQUARE ? mp : r.np);
  const unsigned short* src = reinterpret_cast<const unsigned short*>(ws) + (SQUARE ? r.a : odd ? r.x1 : r.x0);
  const int ld = SQUARE ? mp : r.np;
  const G16Op P = {src, ld, pl, mp, 0};
  g16_f32x16 acc[2][2];
  g16_tile<2, false, false>(acc, P, P, tr * G16_T, tc * G16_T, 0, ld, g16_p0, g16_q0, g16_p1, g16_q1);
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
  g16_store_tile(value, [&](int c, int q, const float (&v)[8]) { put(tc * G16_T + c, tr * G16_T + q, v); }, g16_p0, g16_q0, g16_p1, g16_q1);
  if (tr == tc) return;
  // the mirrored tile: eight consecutive c of one r, gathered from the tile in LDS (whole since the barrier in g16_store_tile)
  const float* quarter[4] = {reinterpret_cast<const float*>(g16_p0), reinterpret_cast<const float*>(g16_q0),
                             reinterpret_cast<const float*>(g16_p1), reinterpret_cast<const float*>(g16_q1)};
#pragma unroll
  for (int pass = 0; pass < 8; ++pass) {
    const int rr = (threadIdx.x & 63) + 64 * (pass & 1), c0 = (threadIdx.x >> 6) * 8;        // c0 within the quarter
    const float* q = quarter[pass >> 1];
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = q[(c0 + e) * 128 + (((rr >> 2) ^ (c0 + e)) << 2) + (rr & 3)];
    put(tr * G16_T + rr, tc * G16_T + (pass >> 1) * 32 + c0, v);
  }
}

// X <- a X + B X: r runs along the columns of X, c along its rows
__global__ __launch_bounds__(256) void ns_update_kernel(const NsRec* __restrict__ t, int n, float fa, int odd, _Float16* __restrict__ ws) {
  G16_SHARED
  const NsRec& r = ns_find<&NsRec::x0t>(t, n, blockIdx.x);
  const int nr = (r.np + G16_T - 1) / G16_T;
  const int id = blockIdx.x - r.x0t;
  const int tc = id / nr, tr = id % nr;
  const int mp = r.mp, np = r.np;
  const int64_t pl = (int64_t)mp * np;
  const _Float16* x = ws + (odd ? r.x1 : r.x0);
  _Float16* out = ws + (odd ? r.x0 : r.x1);
  const G16Op P = {reinterpret_cast<const unsigned short*>(x), np, pl, mp, np};
  const G16Op Q = {reinterpret_cast<const unsigned short*>(ws) + r.b, mp, (int64_t)mp * mp, mp, 0};
  g16_f32x16 acc[2][2];
  g16_tile<2, true, false>(acc, P, Q, tr * G16_T, tc * G16_T, 0, mp, g16_p0, g16_q0, g16_p1, g16_q1);
  g16_store_tile([&](int i, int j, int e) { return acc[i][j][e] * (1.f / NS_SCALE); },
                 [&](int c, int q, const float (&v0)[8]) {
                   const int row = tc * G16_T + c, col = tr * G16_T + q;
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
                 },
                 g16_p0, g16_q0, g16_p1, g16_q1);
}

// out = O (the update's own type), or the parameter p <- p decay - lr wscale O; hyper: {lr, decay} from device memory (a captured
// step), guard: the step's guard word (see adamw.hip)
template <bool BF16>
__global__ __launch_bounds__(256) void ns_apply_kernel(const NsRec* __restrict__ t, int n, NsStep st, const float* __restrict__ hyper,
                                                       const unsigned* __restrict__ guard, int odd, const _Float16* __restrict__ ws) {
  if (guard != nullptr && (__hip_atomic_load(guard, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & 0x7fffffffu) != 0u) return;
  __shared__ float blk[NS_BLK][NS_BLK + 1];
  const NsRec r = ns_find<&NsRec::e0>(t, n, blockIdx.x);
  const float lr = hyper ? hyper[0] : st.lr, decay = hyper ? hyper[1] : st.decay;
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
  const float f = lr * r.wscale;
#pragma unroll 4
  for (int l = threadIdx.x >> 6; l < NS_BLK; l += 4) {
    const int i = gr + l, j = gc + lc;
    if (i >= r.rows || j >= r.cols) continue;
    const int64_t at = (int64_t)i * r.cols + j;
    const float o = blk[l][lc] * (1.f / NS_SCALE);
    if (r.mom) {
      float* p = reinterpret_cast<float*>(r.out) + at;
      *p = *p * decay - f * o;
    } else if (BF16) {
      reinterpret_cast<unsigned short*>(r.out)[at] = g16_bf16(o);
    } else {
      reinterpret_cast<float*>(r.out)[at] = o;
    }
  }
}

struct NsPlan {
  std::vector<NsRec> recs;
  int64_t halves = 0, parts = 0;
  int blocks = 0, sym = 0, upd = 0;
};

// the workspace: [records][partial sums][planes]
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
  int64_t blocks = 0, sym = 0, upd = 0;
  for (int64_t k = 0; k < n; ++k) {
    const NsTensor& s = ts[order[k]];
    NsRec r = {};
    r.g = s.g; r.mom = s.mom; r.out = s.out; r.wscale = s.wscale;
    r.rows = (int)s.rows; r.cols = (int)s.cols;
    r.m = std::min(r.rows, r.cols); r.n = std::max(r.rows, r.cols);
    r.mp = pad(r.m); r.np = pad(r.n);
    const int64_t x = 2 * (int64_t)r.mp * r.np, a = 2 * (int64_t)r.mp * r.mp;
    r.x0 = out->halves; r.x1 = r.x0 + x; r.a = r.x1 + x; r.b = r.a + a;
    out->halves = r.b + a;
    const int64_t nb = (int64_t)(r.mp / NS_BLK) * (r.np / NS_BLK);
    r.per = (int)ceil_div(nb, NS_PARTS);
    r.nparts = (int)ceil_div((int64_t)r.rows * r.cols, (int64_t)r.per * NS_BLK * NS_BLK);
    r.part = out->parts;
    r.p0 = (int)out->parts;
    out->parts += r.nparts;
    r.e0 = (int)blocks; blocks += nb;
    const int64_t tm = ceil_div(r.mp, G16_T), tn = ceil_div(r.np, G16_T);
    r.s0 = (int)sym; sym += tm * (tm + 1) / 2;
    r.x0t = (int)upd; upd += tm * tn;
    if (blocks >= (1ll << 30) || sym >= (1ll << 24) || upd >= (1ll << 30)) return OFQ_EINVAL;
    out->recs.push_back(r);
  }
  out->blocks = (int)blocks; out->sym = (int)sym; out->upd = (int)upd;
  return 0;
}
static size_t ns_up(size_t b) { return (b + 255) & ~(size_t)255; }

extern "C" int64_t ofq_newton_schulz_entry_bytes(void) { return (int64_t)sizeof(NsTensor); }

extern "C" size_t ofq_newton_schulz_ws_bytes(const void* tensors, int64_t n) {
  try {
    NsPlan p;
    if (ns_plan((const NsTensor*)tensors, n, &p)) return 0;
    return ns_up(n * sizeof(NsRec)) + ns_up(p.parts * sizeof(double)) + ns_up(p.halves * 2);
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
    const size_t rb = ns_up(n * sizeof(NsRec)), pb = ns_up(p.parts * sizeof(double));
    if (!ws || ((uintptr_t)ws & 255) || ws_bytes < rb + pb + ns_up(p.halves * 2)) return OFQ_ENOWS;
    NsRec* recs = (NsRec*)ws;
    double* parts = (double*)((char*)ws + rb);
    _Float16* planes = (_Float16*)((char*)ws + rb + pb);
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
    for (int k = 0; k < steps; ++k) {
      hipLaunchKernelGGL(ns_sym_kernel<false>, dim3(p.sym), dim3(256), 0, st, recs, nn, fb, fc, k & 1, planes);
      OFQ_LAUNCH_CHECK();
      hipLaunchKernelGGL(ns_sym_kernel<true>, dim3(p.sym), dim3(256), 0, st, recs, nn, fb, fc, k & 1, planes);
      OFQ_LAUNCH_CHECK();
      hipLaunchKernelGGL(ns_update_kernel, dim3(p.upd), dim3(256), 0, st, recs, nn, fa, k & 1, planes);
      OFQ_LAUNCH_CHECK();
    }
    if (bf16) hipLaunchKernelGGL(ns_apply_kernel<true>, dim3(p.blocks), dim3(256), 0, st, recs, nn, s, hyper, gd, steps & 1, planes);
    else hipLaunchKernelGGL(ns_apply_kernel<false>, dim3(p.blocks), dim3(256), 0, st, recs, nn, s, hyper, gd, steps & 1, planes);
    OFQ_LAUNCH_CHECK();
    return 0;
  } catch (...) { return OFQ_EINVAL; }
}
