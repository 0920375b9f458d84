#pragma once
// The matrix product behind the linear cross entropy and the Newton-Schulz chain: D[r][c] = sum_k P[r, k] Q[c, k] on 16-bit planes,
// fp32 accumulation, with the epilogue of the caller.
//   NP = 1  bf16 operands as they are: one v_mfma_f32_32x32x16_bf16 per 16 k.
//   NP = 2  fp32 operands as two fp16 planes hi = rne(x 2^E), lo = rne(x 2^E - hi): hi hi + hi lo + lo hi, three
//           v_mfma_f32_32x32x16_f16 per 16 k.  The dropped lo lo and the rounding of lo are <= 2^-22 of the product for every
//           element within 2^-13 of the planes' full scale: fp32's own precision at 3/16 of the fp32 MFMA's cost.
// An operand is stored with k contiguous ("row": element (r, k) at r ld + k) or with r contiguous ("col": k ld + r).  Both go
// from global memory into LDS without a register in between (16 bytes a lane); a col tile is read with the transposing LDS
// read, so no transposed copy of an operand exists anywhere.
// Tile 128 x 128, 256 threads = 2 x 2 waves of 64 x 64, k-step 64 (NP = 1) or 32 (NP = 2): 32 KB a stage, two stages, two
// workgroups to a CU.  The LDS DMA writes linearly, so the 16-byte chunks of a row are permuted at the source: row tiles
// by XOR with the bits of the row that share a 256-byte bank line, col tiles by XOR of the chunk with 4 (k & 3), which puts the four
// k rows of a transposing read on different banks.
// The accumulator's lanes run along c and its registers along r (four consecutive r): outputs are stored [c][r].
#include "common.h"

typedef _Float16 g16_f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 g16_bf16x8 __attribute__((ext_vector_type(8)));
typedef short g16_s16x4 __attribute__((ext_vector_type(4)));
typedef short g16_s16x8 __attribute__((ext_vector_type(8)));
typedef float g16_f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned g16_u32x4 __attribute__((ext_vector_type(4)));

#define G16_T 128                        // tile rows and columns
#define G16_PAD 64                       // what packed operands are padded to, in both directions

// rows: r extent of a row operand / k extent of a col operand (loads past it repeat its last row);
// cols: of a col operand, its r extent rounded up to 8 (chunks past it repeat chunk 0)
struct G16Op {
  const unsigned short* p;
  int64_t ld, plane;
  int rows, cols;
};

template <int NP> struct G16 {
  static constexpr int BK = NP == 1 ? 64 : 32;
  static constexpr int CPR = BK / 8;                    // 16-byte chunks of a row tile's row
  static constexpr int RPL = 16 / CPR;                  // rows to a 256-byte bank line
  static constexpr int HALVES = NP * G16_T * BK;        // of one operand's stage: 8192
};

// the four 16 KB stage buffers; separate arrays, so that the compiler knows which of them an outstanding DMA writes
#define G16_SHARED                                                                       \
  __shared__ __attribute__((aligned(1024))) unsigned short g16_p0[8192];                 \
  __shared__ __attribute__((aligned(1024))) unsigned short g16_q0[8192];                 \
  __shared__ __attribute__((aligned(1024))) unsigned short g16_p1[8192];                 \
  __shared__ __attribute__((aligned(1024))) unsigned short g16_q1[8192];

template <int NP, bool COL>
struct G16Loader {
  const unsigned short* at[4];
  int64_t step;
  const unsigned short* base;
  int64_t ld;
  int k_last, kl[4];
  // wave w issues chunks [w * 256, w * 256 + 256) of the stage's 1024, 64 a time
  __device__ __forceinline__ void init(const G16Op& o, int r0, int k0, int wid, int lane) {
    constexpr int BK = G16<NP>::BK, CPR = G16<NP>::CPR, RPL = G16<NP>::RPL;
    ld = o.ld;
    base = o.p;
    k_last = o.rows - 1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int L = (wid * 4 + u) * 64 + lane;
      const int pl = NP == 1 ? 0 : L >> 9, l = NP == 1 ? L : L & 511;
      if (!COL) {
        const int row = l / CPR, c = (l % CPR) ^ ((row / RPL) % CPR);
        const int r = min(r0 + row, o.rows - 1);
        at[u] = o.p + pl * o.plane + (int64_t)r * o.ld + k0 + c * 8;
        kl[u] = 0;
      } else {
        const int k = l >> 4, c = (l & 15) ^ ((k & 3) << 2);
        const int r = r0 + c * 8 < o.cols ? r0 + c * 8 : 0;
        at[u] = o.p + pl * o.plane + (int64_t)(k0 + k) * o.ld + r;
        kl[u] = k0 + k;
      }
    }
    step = COL ? (int64_t)BK * o.ld : BK;
  }
  __device__ __forceinline__ void issue(unsigned short* lds, int wid) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned short* g = at[u];
      if (COL) {                                         // past the last k row: that row again (the other operand is zero there)
        const int over = kl[u] - k_last;
        if (over > 0) g -= (int64_t)over * ld;
        kl[u] += G16<NP>::BK;
      }
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)g,
                                       (__attribute__((address_space(3))) unsigned*)(lds + (wid * 4 + u) * 512), 16, 0, 0);
      at[u] += step;
    }
  }
};

template <int NP, bool COL>
__device__ __forceinline__ g16_s16x8 g16_frag(const unsigned short* s, int pl, int half, int blk, int ks, int lane) {
  constexpr int BK = G16<NP>::BK, CPR = G16<NP>::CPR, RPL = G16<NP>::RPL;
  const int l31 = lane & 31, lh = lane >> 5;
  if (!COL) {
    const int row = half * 64 + blk * 32 + l31;
    const int c = (ks * 2 + lh) ^ ((l31 / RPL) % CPR);
    return *reinterpret_cast<const g16_s16x8*>(s + pl * (G16_T * BK) + row * BK + c * 8);
  } else {
    const int p16 = lane & 15;
    const int k = ks * 16 + 8 * lh + (p16 >> 2);
    const int chunk = (half * 8 + blk * 4 + 2 * ((lane >> 4) & 1) + ((p16 & 3) >> 1)) ^ ((p16 >> 2) << 2);
    const unsigned short* a = s + pl * (G16_T * BK) + k * G16_T + chunk * 8 + (p16 & 1) * 4;
    const g16_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) g16_s16x4*)(a));
    const g16_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) g16_s16x4*)(a + 4 * G16_T));
    return g16_s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
}

template <int NP>
__device__ __forceinline__ g16_f32x16 g16_mfma(g16_s16x8 a, g16_s16x8 b, g16_f32x16 c) {
  if constexpr (NP == 1)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(g16_bf16x8, a), __builtin_bit_cast(g16_bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(g16_f16x8, a), __builtin_bit_cast(g16_f16x8, b), c, 0, 0, 0);
}

// all of a wave's LDS reads returned and its DMA landed, then the barrier.  The wait is the builtin, which the compiler's own wait
// counting sees: behind an inline-asm wait it still takes the DMA for outstanding and waits for the next stage's in front of this one's reads.
__device__ __forceinline__ void g16_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);                    // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// One stage.  Inside an MFMA products are cut off some bits below the accumulator's last place (its final rounding is to nearest).
// Accumulators of 32 k each, added up with v_add_f32, halved the error of the sums but took 9 % of the time; as it is the
// Newton-Schulz chain is 1.1e-6 to 2.9e-6 off where fp32 products are 1.5e-6 to 3.9e-6 off, so it is left out.
template <int NP, bool PCOL, bool QCOL>
__device__ __forceinline__ void g16_compute(g16_f32x16 (&acc)[2][2], const unsigned short* sp, const unsigned short* sq, int wr, int wc,
                                            int lane) {
#pragma unroll
  for (int ks = 0; ks < G16<NP>::BK / 16; ++ks) {
    g16_s16x8 a[NP][2], b[NP][2];
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[q][i] = g16_frag<NP, PCOL>(sp, q, wr, i, ks, lane);
        b[q][i] = g16_frag<NP, QCOL>(sq, q, wc, i, ks, lane);
      }
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int s = 0; s < NP - q; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = g16_mfma<NP>(a[q][i], b[s][j], acc[i][j]);
  }
}

// the k loop of one tile: k in [kb, ke), both multiples of G16<NP>::BK
template <int NP, bool PCOL, bool QCOL>
__device__ __forceinline__ void g16_tile(g16_f32x16 (&acc)[2][2], const G16Op& P, const G16Op& Q, int r0, int c0, int kb, int ke,
                                         unsigned short* p0, unsigned short* q0, unsigned short* p1, unsigned short* q1) {
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wid & 1, wc = wid >> 1;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  const int nk = (ke - kb) / G16<NP>::BK;
  if (nk <= 0) return;
  G16Loader<NP, PCOL> lp;
  G16Loader<NP, QCOL> lq;
  lp.init(P, r0, kb, wid, lane);
  lq.init(Q, c0, kb, wid, lane);
  lp.issue(p0, wid);
  lq.issue(q0, wid);
  g16_barrier();
  int t = 0;
  for (; t + 2 <= nk; t += 2) {
    lp.issue(p1, wid);
    lq.issue(q1, wid);
    __builtin_amdgcn_sched_barrier(0);                   // the next stage's loads go out ahead of this one's LDS reads
    g16_compute<NP, PCOL, QCOL>(acc, p0, q0, wr, wc, lane);
    g16_barrier();
    if (t + 2 < nk) {
      lp.issue(p0, wid);
      lq.issue(q0, wid);
    }
    __builtin_amdgcn_sched_barrier(0);
    g16_compute<NP, PCOL, QCOL>(acc, p1, q1, wr, wc, lane);
    g16_barrier();
  }
  if (t < nk) {
    g16_compute<NP, PCOL, QCOL>(acc, p0, q0, wr, wc, lane);
    g16_barrier();
  }
}

// r of register e of block i, relative to the tile
__device__ __forceinline__ int g16_r(int wr, int i, int e, int lane) { return wr * 64 + i * 32 + (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5); }
__device__ __forceinline__ int g16_c(int wc, int j, int lane) { return wc * 64 + j * 32 + (lane & 31); }

// The tile in LDS as [c][r] fp32, a quarter (32 c) in each of the stage buffers; then every thread gets eight consecutive r of eight
// rows c: f(c, r, v) with c, r relative to the tile.  Chunks of four r are XORed with c (bank conflicts).
template <class V, class F>
__device__ __forceinline__ void g16_store_tile(V&& val, F&& f, unsigned short* p0, unsigned short* q0, unsigned short* p1,
                                               unsigned short* q1) {
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wid & 1, wc = wid >> 1, l31 = lane & 31, lh = lane >> 5;
  float* quarter[4] = {reinterpret_cast<float*>(p0), reinterpret_cast<float*>(q0), reinterpret_cast<float*>(p1),
                       reinterpret_cast<float*>(q1)};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float* q = wc == 0 ? quarter[j] : quarter[2 + j];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int eb = 0; eb < 4; ++eb) {
        const int ch = (wr * 16 + i * 8 + eb * 2 + lh) ^ l31;
        *reinterpret_cast<float4*>(q + l31 * 128 + ch * 4) =
            make_float4(val(i, j, eb * 4), val(i, j, eb * 4 + 1), val(i, j, eb * 4 + 2), val(i, j, eb * 4 + 3));
      }
  }
  g16_barrier();
  const int rg = threadIdx.x & 15, cr = threadIdx.x >> 4;
#pragma unroll
  for (int pass = 0; pass < 8; ++pass) {
    const float* q = quarter[pass >> 1];
    const int cl = (pass & 1) * 16 + cr;
    const float4 a = *reinterpret_cast<const float4*>(q + cl * 128 + ((rg * 2) ^ cl) * 4);
    const float4 b = *reinterpret_cast<const float4*>(q + cl * 128 + ((rg * 2 + 1) ^ cl) * 4);
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    f((pass >> 1) * 32 + cl, rg * 8, v);
  }
}

// eight values as two fp16 planes (rounded to nearest even: hi is off by half a step of fp16, lo by half a step of what is left).  The
// value is pinned in a register: where it is a product the compiler otherwise rounds it to fp16 in one step for hi (v_fma_mixlo_f16) and
// through fp32 for lo, and one element in 10^4, a tie of the two, is off by a step of hi.
__device__ __forceinline__ void g16_split8(const float (&v)[8], g16_u32x4& hi, g16_u32x4& lo) {
  _Float16 h[8], l[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float x = v[e];
    asm("" : "+v"(x));
    h[e] = (_Float16)x;
    l[e] = (_Float16)(x - (float)h[e]);
  }
  hi = __builtin_bit_cast(g16_u32x4, *reinterpret_cast<g16_f16x8*>(h));
  lo = __builtin_bit_cast(g16_u32x4, *reinterpret_cast<g16_f16x8*>(l));
}
__device__ __forceinline__ void g16_join8(g16_u32x4 hi, g16_u32x4 lo, float (&v)[8]) {
  const g16_f16x8 h = __builtin_bit_cast(g16_f16x8, hi), l = __builtin_bit_cast(g16_f16x8, lo);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)h[e] + (float)l[e];
}
// fp32 -> bf16, to nearest even; a NaN stays one
__device__ __forceinline__ unsigned short g16_bf16(float x) { return __builtin_bit_cast(unsigned short, (__bf16)x); }
__device__ __forceinline__ g16_u32x4 g16_bf16x8_of(const float (&v)[8]) {
  g16_bf16x8 h;
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = (__bf16)v[e];
  return __builtin_bit_cast(g16_u32x4, h);
}
__device__ __forceinline__ float g16_f32(unsigned short b) { return __uint_as_float((unsigned)b << 16); }

// Workgroup -> tile: workgroups go round robin over the eight XCDs, each with its own L2; every XCD gets a contiguous run of tiles,
// and within it the tiles go in groups of eight rows of c, r fastest over the group, so that the run's operands stay in the L2
__device__ __forceinline__ void g16_tile_of(int id, int tr, int tc, int& r, int& c) {
  const int total = tr * tc;
  const int q = total >> 3, rem = total & 7, xcd = id & 7, loc = id >> 3;
  const int t = (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + loc;
  const int per = 8 * tr, g = t / per, first = g * 8, size = min(8, tc - first), in = t - g * per;
  c = first + in % size;
  r = in / size;
}
