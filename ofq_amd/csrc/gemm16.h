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
// The LDS DMA writes linearly, so the 16-byte chunks of a row are permuted at the source: row tiles
// by XOR with the bits of the row that share a 256-byte bank line, col tiles by XOR of the chunk with 4 (k & 3), which puts the four
// k rows of a transposing read on different banks.
// The accumulator's lanes run along c and its registers along r (four consecutive r): outputs are stored [c][r].
#include "common.h"
#include <type_traits>
#include <utility>

typedef _Float16 g16_f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 g16_bf16x8 __attribute__((ext_vector_type(8)));
typedef short g16_s16x4 __attribute__((ext_vector_type(4)));
typedef short g16_s16x8 __attribute__((ext_vector_type(8)));
typedef float g16_f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned g16_u32x4 __attribute__((ext_vector_type(4)));
typedef float g16_f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) float g16_ldsf;
typedef __attribute__((address_space(3))) g16_f32x4 g16_ldsf4;

#define G16_PAD 64                       // what packed operands are padded to, in both directions

// The tile forms:
//   BIG   256 x 256, 2 x 4 waves of 128 x 64: half the operand traffic per product.  For grids that fill the chip with it.
//   MID   128 x 128, 2 x 2 waves, two workgroups to a CU, the one's loads and barriers behind the other's MFMAs.
//   DEEP  128 x 128, 2 x 2 waves, four stages, one workgroup to a CU: for grids that have no second one to give it, or whose longest tile
//         is what everything waits for.  One wave to a SIMD hides nothing by itself, so its LDS reads and DMA loads are spread one by one
//         behind the MFMAs (a burst of eight loads stalls a wave by 340 cycles, and the MFMAs with it): 24 k-steps of two planes 20 us
//         where MID takes 25.
//   TINY  64 x 64 in the same manner: for grids whose time is one tile's latency.
// A 256 x 256 form of four waves in that manner (512 registers, 64 bytes a clock of LDS reads) was no faster on rows and 2 to 3 times
// slower on columns.
enum { G16_MID = 0, G16_DEEP = 1, G16_BIG = 2, G16_TINY = 3 };

// rows: r extent of a row operand (loads past it repeat its last row); a col operand has every k row of the loop
// cols: of a col operand, its r extent rounded up to 8 (chunks past it repeat chunk 0)
struct G16Op {
  const unsigned short* p;
  int64_t ld, plane;
  int rows, cols;
};

constexpr int g16_nt(int cfg) { return cfg == G16_BIG ? 512 : 256; }     // threads
constexpr int g16_t(int cfg) { return cfg == G16_BIG ? 256 : cfg == G16_TINY ? 64 : 128; }

template <int NP, int CFG> struct G16 {
  static constexpr int BK = NP == 1 ? 64 : 32;
  static constexpr int T = g16_t(CFG);                  // tile rows and columns
  static constexpr int SIZE = T / 128;                  // 0, 1, 2
  static constexpr int WC = CFG == G16_BIG ? 4 : 2;     // waves along c; two along r
  static constexpr int RB = T / 64, CB = T / (32 * WC); // 32 x 32 blocks of a wave
  static constexpr int KS = BK / 16;                    // phases (of 16 k) in a stage
  static constexpr int CPR = BK / 8;                    // 16-byte chunks of a row tile's row
  static constexpr int RPL = 16 / CPR;                  // rows to a 256-byte bank line
  static constexpr int HALVES = NP * T * BK;            // of one operand's stage: 8 KB (TINY), 16 or 32 (BIG)
  static constexpr int LOADS = HALVES / 1024 / WC;      // DMA loads of a wave and operand for a stage: four (TINY: two)
  // the XOR of a col tile's chunks: four k rows on different banks (a row of T = 64 is half a bank line)
  static __device__ constexpr int colx(int k) { return T >= 128 ? (k & 3) << 2 : (k >> 1 & 1) << 2; }
  static constexpr int DEPTH = CFG == G16_DEEP || CFG == G16_TINY ? 4 : 2;       // stages
};
template <int NP, int CFG> using G16Acc = g16_f32x16[G16<NP, CFG>::RB][G16<NP, CFG>::CB];

// the stage buffers; separate arrays, so that the compiler knows which of them an outstanding DMA writes
typedef __attribute__((address_space(3))) unsigned short g16_lds;
struct G16Lds { g16_lds *p[4], *q[4]; };
#define G16_SHARED(NP, CFG)                                                                                                            \
  constexpr int g16_n = G16<NP, CFG>::HALVES, g16_m = G16<NP, CFG>::DEPTH > 2 ? g16_n : 8;                                             \
  __shared__ __attribute__((aligned(1024))) unsigned short g16_p0[g16_n], g16_q0[g16_n], g16_p1[g16_n], g16_q1[g16_n];                 \
  __shared__ __attribute__((aligned(1024))) unsigned short g16_p2[g16_m], g16_q2[g16_m], g16_p3[g16_m], g16_q3[g16_m];                 \
  G16Lds lds;      /* (stored one by one: an initialiser of constants would become a table in memory) */                                 \
  lds.p[0] = (g16_lds*)g16_p0; lds.p[1] = (g16_lds*)g16_p1; lds.p[2] = (g16_lds*)g16_p2; lds.p[3] = (g16_lds*)g16_p3;                                                          \
  lds.q[0] = (g16_lds*)g16_q0; lds.q[1] = (g16_lds*)g16_q1; lds.q[2] = (g16_lds*)g16_q2; lds.q[3] = (g16_lds*)g16_q3;

// A wave's loads of a stage: a scalar base that moves with the stage, and one 32-bit offset a load and lane that never changes
template <int NP, int CFG, bool COL>
struct G16Loader {
  using C = G16<NP, CFG>;
  unsigned off[C::LOADS];                                // bytes
  const char* base;
  int64_t step;                                          // bytes a stage
  // wave w issues chunks [w * LOADS * 64, (w + 1) * LOADS * 64) of the stage, 64 a time; they lie in one plane
  __device__ __forceinline__ void init(const G16Op& o, int r0, int k0, int wid, int lane) {
    constexpr int PC = C::HALVES / 8 / NP;               // chunks of a plane
    const int pl = NP == 1 ? 0 : wid * C::LOADS * 64 / PC;
    static_assert(NP == 1 || PC % (C::LOADS * 64) == 0, "a wave's chunks lie in one plane");
    base = reinterpret_cast<const char*>(o.p + pl * o.plane + (COL ? (int64_t)k0 * o.ld : (int64_t)r0 * o.ld + k0));
    step = (COL ? (int64_t)C::BK * o.ld : C::BK) * 2;
#pragma unroll
    for (int u = 0; u < C::LOADS; ++u) {
      const int l = ((wid * C::LOADS + u) * 64 + lane) % PC;
      if (!COL) {
        const int row = l / C::CPR, c = (l % C::CPR) ^ ((row / C::RPL) % C::CPR);
        off[u] = (unsigned)min(row, o.rows - 1 - r0) * (unsigned)(o.ld * 2) + c * 16;
      } else {
        const int k = l / (C::T / 8), c = (l % (C::T / 8)) ^ C::colx(k);
        off[u] = (unsigned)k * (unsigned)(o.ld * 2) + (r0 + c * 8 < o.cols ? r0 + c * 8 : 0) * 2;
      }
    }
  }
  __device__ __forceinline__ void issue(g16_lds* lds, int wid, int u, int t) const {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)(base + t * step + off[u]),
                                     (__attribute__((address_space(3))) unsigned*)(lds + (wid * C::LOADS + u) * 512), 16, 0, 0);
  }
};

// eight k of one row: block `blk` (32 rows) of the tile
template <int NP, int CFG, bool COL>
__device__ __forceinline__ g16_s16x8 g16_frag(const g16_lds* s, int pl, int blk, int ks, int lane) {
  using C = G16<NP, CFG>;
  const int l31 = lane & 31, lh = lane >> 5;
  if (!COL) {
    const int c = (ks * 2 + lh) ^ ((l31 / C::RPL) % C::CPR);
    return *(const __attribute__((address_space(3))) g16_s16x8*)(s + pl * (C::T * C::BK) + (blk * 32 + l31) * C::BK + c * 8);
  } else {
    const int p16 = lane & 15;
    const int k = ks * 16 + 8 * lh + (p16 >> 2);
    const int chunk = (blk * 4 + 2 * ((lane >> 4) & 1) + ((p16 & 3) >> 1)) ^ C::colx(p16 >> 2);
    const g16_lds* a = s + pl * (C::T * C::BK) + k * C::T + chunk * 8 + (p16 & 1) * 4;
    const g16_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) g16_s16x4*)(a));
    const g16_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) g16_s16x4*)(a + 4 * C::T));
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

// at most N of a wave's DMA loads outstanding and all of its LDS reads returned, then the barrier.  The wait is the builtin, which the
// compiler's own wait counting sees: behind an inline-asm wait it still takes the DMA for outstanding and waits for the next stage's
// in front of this one's reads.
template <int N>
__device__ __forceinline__ void g16_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0070);        // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// f(integral_constant<0>) ... f(integral_constant<N - 1>)
template <class F, int... I>
__device__ __forceinline__ void g16_for_impl(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F> __device__ __forceinline__ void g16_for(F&& f) { g16_for_impl(f, std::make_integer_sequence<int, N>{}); }

// The fragments of 16 k: what a wave's MFMAs of one phase take; read number n of NP (RB + CB)
template <int NP, int CFG> struct G16Frags { g16_s16x8 a[NP][G16<NP, CFG>::RB], b[NP][G16<NP, CFG>::CB]; };
template <int NP, int CFG, bool PCOL, bool QCOL, int N>
__device__ __forceinline__ void g16_read(G16Frags<NP, CFG>& f, const G16Lds& s, int buf, int ks, int wr, int wc, int lane) {
  constexpr int RB = G16<NP, CFG>::RB, CB = G16<NP, CFG>::CB, q = N / (RB + CB), i = N % (RB + CB);
  if constexpr (i < RB) f.a[q][i] = g16_frag<NP, CFG, PCOL>(s.p[buf], q, wr * RB + i, ks, lane);
  else f.b[q][i - RB] = g16_frag<NP, CFG, QCOL>(s.q[buf], q, wc * CB + i - RB, ks, lane);
}
// MFMA number n of RB CB (NP = 1) or 3 RB CB (hi hi, hi lo, lo hi).  Inside an MFMA products are cut off some bits below the accumulator's
// last place (its final rounding is to nearest).  Accumulators of four stages each (128 k of two planes, 256 of one), added up
// with v_add_f32, halve the error of long sums.  TINY has them: its time is a latency.  In the other forms they took 9 %; there the Newton-Schulz chain is 1.1e-6 to 2.9e-6 off where
// fp32 products are 1.5e-6 to 3.9e-6 off, so they are left out.
template <int NP, int CFG, int N>
__device__ __forceinline__ void g16_mma(G16Acc<NP, CFG>& acc, const G16Frags<NP, CFG>& f) {
  constexpr int RB = G16<NP, CFG>::RB, CB = G16<NP, CFG>::CB, m = N / (RB * CB), i = N / CB % RB, j = N % CB, pa = m == 2, pb = m == 1;
  acc[i][j] = g16_mfma<NP>(f.a[pa][i], f.b[pb][j], acc[i][j]);
}

// The k loop of one tile: k in [kb, ke), both multiples of BK.
// DEEP: the fragments of the next 16 k are read while the MFMAs of the current ones run, across the stages too: the barrier that
// makes stage t + 1 readable comes in front of the last phase of stage t, when all of stage t is in registers; its buffer is free from
// there on and takes the loads of stage t + DEPTH, which are spread over SPREAD phases.
// ADD: on top of what acc holds.
template <int NP, int CFG, bool PCOL, bool QCOL, bool ADD = false>
__device__ __forceinline__ void g16_tile(G16Acc<NP, CFG>& acc, const G16Op& P, const G16Op& Q, int r0, int c0, int kb, int ke, const G16Lds& s) {
  using C = G16<NP, CFG>;
  constexpr int D = C::DEPTH, KS = C::KS, NL = 2 * C::LOADS, NM = C::RB * C::CB * (NP == 2 ? 3 : 1), NR = (C::RB + C::CB) * NP;
  static_assert(KS % 2 == 0, "two fragment sets in turn");
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wid & 1, wc = wid >> 1;
  if constexpr (!ADD) {
#pragma unroll
    for (int i = 0; i < C::RB; ++i)
#pragma unroll
      for (int j = 0; j < C::CB; ++j) acc[i][j] = g16_f32x16{};
  }
  const int nk = (ke - kb) / C::BK;
  if (nk <= 0) return;
  G16Loader<NP, CFG, PCOL> lp;
  G16Loader<NP, CFG, QCOL> lq;
  lp.init(P, r0, kb, wid, lane);
  lq.init(Q, c0, kb, wid, lane);
  // load n of NL of stage t into buffer b; past the last stage that one's again (the loop has no conditions)
  auto load1 = [&](int b, int n, int t) {
    if (n < C::LOADS) lp.issue(s.p[b], wid, n, min(t, nk - 1));
    else lq.issue(s.q[b], wid, n - C::LOADS, min(t, nk - 1));
  };
  auto load = [&](int b, int t) {
#pragma unroll
    for (int n = 0; n < NL; ++n) load1(b, n, t);
  };
  if constexpr (C::DEPTH == 2) {
    auto use = [&](int b) {
      __builtin_amdgcn_sched_barrier(0);                 // the next stage's loads go out ahead of this one's LDS reads
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        G16Frags<NP, CFG> f;
        g16_for<NR>([&](auto n) { g16_read<NP, CFG, PCOL, QCOL, n()>(f, s, b, ks, wr, wc, lane); });
        g16_for<NM>([&](auto n) { g16_mma<NP, CFG, n()>(acc, f); });
      }
    };
    load(0, 0);
    g16_barrier<0>();
    int t = 0;
    for (; t + 2 <= nk; t += 2) {
      load(1, t + 1);
      use(0);
      g16_barrier<0>();
      if (t + 2 < nk) load(0, t + 2);
      use(1);
      g16_barrier<0>();
    }
    if (t < nk) {
      use(0);
      g16_barrier<0>();
    }
  } else {
    constexpr int SPREAD = NM >= 2 * NL ? 1 : NM >= NL ? 2 : KS;               // phases that take the loads, an MFMA or two to each
    constexpr int FIRST = NL / SPREAD;                                         // loads of a phase
    static_assert(SPREAD <= KS && NL % SPREAD == 0, "the loads are out before the next barrier");
    G16Frags<NP, CFG> f[2];
    // TINY: accumulators of D stages each
    constexpr bool PART = CFG == G16_TINY;
    G16Acc<NP, CFG> part;
    auto& sum = *[&] { if constexpr (PART) return &part; else return &acc; }();
    auto flush = [&](bool add) {
#pragma unroll
      for (int i = 0; i < C::RB; ++i)
#pragma unroll
        for (int j = 0; j < C::CB; ++j) {
          if (add) acc[i][j] += part[i][j];
          part[i][j] = g16_f32x16{};
        }
    };
    if constexpr (PART) flush(false);
    // The MFMAs of phase ks, and behind them the reads of the next one (rks of buffer rb) and loads [L0, L0 + N) of stage lt into buffer lb
    auto phase = [&](int ks, int rb, int rks, int lb, int lt, auto l0_, auto n_) {
      constexpr int L0 = l0_(), N = n_();
      g16_for<NM>([&](auto m_) {
        constexpr int m = m_();
        g16_mma<NP, CFG, m>(sum, f[ks & 1]);
        constexpr int ra = m * NR / NM, re = (m + 1) * NR / NM, la = m * N / NM, le = (m + 1) * N / NM;
        g16_for<re - ra>([&](auto d) { g16_read<NP, CFG, PCOL, QCOL, ra + d()>(f[(ks + 1) & 1], s, rb, rks, wr, wc, lane); });
        g16_for<le - la>([&](auto d) { load1(lb, L0 + la + d(), lt); });
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    using I0 = std::integral_constant<int, 0>;
    using IF = std::integral_constant<int, FIRST>;
#pragma unroll
    for (int u = 0; u < D - 1; ++u) load(u, u);
#pragma unroll
    for (int n = 0; n < FIRST; ++n) load1(D - 1, n, D - 1);
    g16_barrier<NL * (D - 2) + FIRST>();
    g16_for<NR>([&](auto n) { g16_read<NP, CFG, PCOL, QCOL, n()>(f[0], s, 0, 0, wr, wc, lane); });
    for (int t = 0;; t += D) {
      bool done = false;
      g16_for<D>([&](auto u_) {
        constexpr int u = u_();
        if (done) return;
        if constexpr (PART && u == 0) flush(true);
        // all phases of stage t + u but the last, with what is left of the loads of the stage before
        g16_for<KS - 1>([&](auto ks_) {
          constexpr int ks = ks_();
          if constexpr (ks + 1 < SPREAD) phase(ks, u, ks + 1, (u + D - 1) % D, t + u + D - 1, std::integral_constant<int, (ks + 1) * FIRST>{}, IF{});
          else phase(ks, u, ks + 1, 0, 0, I0{}, I0{});
        });
        if (t + u + 1 >= nk) { done = true; return; }
        g16_barrier<NL * (D - 2)>();
        phase(KS - 1, (u + 1) % D, 0, u, t + u + D, I0{}, IF{});
      });
      if (done) break;
    }
    g16_for<NM>([&](auto n) { g16_mma<NP, CFG, n()>(sum, f[(KS - 1) & 1]); });
    if constexpr (PART) flush(true);
    g16_barrier<0>();                                    // the repeated loads land before the buffers serve the epilogue
  }
}

// r of register e of block i and c of block j, relative to the tile
template <int CFG> __device__ __forceinline__ int g16_r(int wr, int i, int e, int lane) {
  return wr * (G16<1, CFG>::RB * 32) + i * 32 + (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5);
}
template <int CFG> __device__ __forceinline__ int g16_c(int wc, int j, int lane) { return wc * (G16<1, CFG>::CB * 32) + j * 32 + (lane & 31); }

// The tile in LDS as [c][r] fp32, four blocks of 32 c a time (BIG: two rounds); every thread gets eight consecutive r of rows c:
// f(c, r, v) with c, r relative to the tile.  Chunks of four r are XORed with c (bank conflicts).  MIRROR: and, behind it, eight
// consecutive c of rows r: m(r, c, v).
template <int NP, int CFG, bool MIRROR, class V, class F, class M>
__device__ __forceinline__ void g16_store_tile(V&& val, F&& f, M&& m, const G16Lds& s) {
  using C = G16<NP, CFG>;
  constexpr int TR = C::T, JR = 4 / C::WC < C::CB ? 4 / C::WC : C::CB, NB = JR * C::WC, ROUNDS = C::CB / JR, NT = g16_nt(CFG);        // JR: blocks of a wave in a round
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wid & 1, wc = wid >> 1, l31 = lane & 31, lh = lane >> 5;
  // row c of 32 of block blk of four; blk is a constant wherever this is called (an index of run time would move the table of buffers to
  // memory, and the k loop's reads of it with it)
  auto row = [&](int blk, int c) { return (g16_ldsf*)(blk & 1 ? s.q[blk >> 1] : s.p[blk >> 1]) + c * TR; };
  g16_for<ROUNDS>([&](auto round_) {
    constexpr int round = round_();
    if (round) __syncthreads();
#pragma unroll
    for (int jr = 0; jr < JR; ++jr) {
      const int at = wc * JR + jr;
      g16_ldsf* q = at == 0 ? row(0, l31) : at == 1 ? row(1, l31) : at == 2 ? row(2, l31) : row(3, l31);
#pragma unroll
      for (int i = 0; i < C::RB; ++i)
#pragma unroll
        for (int eb = 0; eb < 4; ++eb) {
          const int ch = (wr * (C::RB * 8) + i * 8 + eb * 2 + lh) ^ (l31 % (TR / 4));
          const int j = round * JR + jr;
          *(g16_ldsf4*)(q + ch * 4) = g16_f32x4{val(i, j, eb * 4), val(i, j, eb * 4 + 1), val(i, j, eb * 4 + 2), val(i, j, eb * 4 + 3)};
        }
    }
    __syncthreads();
    auto cbase = [&](int blk) { return blk / JR * (C::CB * 32) + (round * JR + blk % JR) * 32; };
    constexpr int PER = TR / 8, STEP = NT / PER;     // threads to a row c, rows to a pass
    const int rg = threadIdx.x % PER, cr = threadIdx.x / PER;
    g16_for<NB * 32 / STEP>([&](auto pass_) {
      constexpr int blk = pass_() / (32 / STEP);
      const int cl = pass_() % (32 / STEP) * STEP + cr;
      const g16_ldsf* q = row(blk, cl);
      const g16_f32x4 a = *(const g16_ldsf4*)(q + ((rg * 2) ^ (cl % (TR / 4))) * 4), b = *(const g16_ldsf4*)(q + ((rg * 2 + 1) ^ (cl % (TR / 4))) * 4);
      const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      f(cbase(blk) + cl, rg * 8, v);
    });
    if constexpr (MIRROR) {
      constexpr int W = NT / 4;                          // r of a pass; four groups of eight c
      g16_for<NB * TR / W>([&](auto pass_) {
        constexpr int blk = pass_() / (TR / W);
        const int rr = threadIdx.x % W + pass_() % (TR / W) * W, cl = threadIdx.x / W * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = row(blk, cl + e)[(((rr >> 2) ^ ((cl + e) % (TR / 4))) << 2) + (rr & 3)];
        m(rr, cbase(blk) + cl, v);
      });
    }
  });
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

// Workgroup -> tile: workgroups go round robin over the eight XCDs, each with its own L2.  Every XCD gets runs of `run` consecutive tiles
// (what it has in flight at a time; or, run = total, one run: as good where all tiles are alike), and consecutive tiles share
// operands: they go in groups of eight c, c fastest.
__device__ __forceinline__ int g16_xcd(int id, int total, int run) {
  const int whole = total / (8 * run) * (8 * run);
  if (id < whole) {
    const int slot = id >> 3;
    return ((slot / run) * 8 + (id & 7)) * run + slot % run;
  }
  id -= whole;
  total -= whole;
  const int q = total >> 3, rem = total & 7, xcd = id & 7, loc = id >> 3;
  return whole + (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + loc;
}
__device__ __forceinline__ void g16_group(int t, int tr, int tc, int& r, int& c) {
  const int per = 8 * tr, g = t / per, first = g * 8, size = min(8, tc - first), in = t - g * per;
  c = first + in % size;
  r = in / size;
}
// Of the tiles r >= c of a symmetric matrix: bands of eight r, r fastest
__device__ __forceinline__ void g16_tri(int t, int n, int& r, int& c) {
  int first = 0;
  for (;; first += 8) {
    const int g = min(8, n - first), count = first * g + g * (g + 1) / 2;
    if (t < count) break;
    t -= count;
  }
  const int g = min(8, n - first);
  if (t < first * g) { r = first + t % g; c = t / g; return; }
  t -= first * g;
  int k = 0;                                             // column k of the band's triangle has g - k tiles
  while (t >= g - k) { t -= g - k; ++k; }
  c = first + k;
  r = c + t;
}

// The tile form for a grid of so many tiles of 64, 128 and 256.  In units of a 128 tile's time on a CU that has two of them, a 256 tile takes
// 3.4; every CU takes whole tiles.  Measured (MID / BIG, us): 1024 tiles of 128, k 14336: 495 / 412; 96 x 32, two planes, k 2048: 639 / 590;
// 1026, i.e. 260 of 256, two planes: 81 / 93; 512: 125 / 173.  TINY / MID, two planes: 10 tiles of 64, k 192: 6 / 10; 180, k 192 and 768:
// 12 / 19; 474, k 197: 11 / 14; 540, k 192: 16 / 14; 2160: 63 / 45.  DEEP / MID: 180 of 128, k 384: 23 / 25.
static inline int g16_form(int64_t t64, int64_t t128, int64_t t256) {
  if (t64 <= 512) return G16_TINY;
  if (t128 <= 256) return G16_DEEP;
  return 3.4 * ceil_div(t256, 256) <= (double)ceil_div(t128, 256) ? G16_BIG : G16_MID;
}
