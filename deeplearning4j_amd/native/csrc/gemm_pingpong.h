// The ping-pong 256 x 256 loop of gemm_core.h (mainloop_pingpong_deep: wave groups, staging order and hazards are those) for operands in
// either layout, and product sources that take an operand as the sum of two 16-bit halves.
//
// Phases of a k-tile read 8, 4, 8 and 4 fragments (32, 16, 32, 16 KiB for the four waves of a group; LDS gives 128 bytes a cycle, a phase's
// MFMAs take 256 cycles): A-lo | B-hi | A-hi | B-lo of the NEXT k-tile, into the registers that B-hi has left. (With B-lo read beside A-lo, 12 / 4 / 8 / 0, the first phase waits for LDS.)
//
//   K-contiguous operand   the core's image: 256 rows x 128 bytes, half-tile h = rows g * 128 + h * 64 + 0..63 (A) / cols wn * 64 + h * 32 + 0..31 (B)
//   K-major operand        each half-tile is an image of its own, [64 k][128 x] with a pitch of 256 bytes: 16 KiB, two 1-KiB pieces per
//                          wave like the other, so the counted waits hold unchanged; the fragments come from transposing LDS reads
//
// A product of fp32 operands runs on the 16-bit matrix cores as three products of halves, a = a1 + a2 with a1 = fp16(a), a2 = fp16(a - a1)
// (operands scaled by a power of two so that the largest is below 2^14):  a . b = a1 b1 + a1 b2 + a2 b1, what is left out is 2^-24 of |a||b|.
// The three are one long product: k-tile t of 3 KT reads halves (t / KT == 2, t / KT == 1) of A and B.
#pragma once
#include "gemm_trans.h"

namespace gemmcore {

template <class C, bool TA, bool TB, class Src>
__device__ __forceinline__ void mainloop_pp(char* smem, const Src& src, int KT, typename C::acc_t (&acc)[C::TM][C::TN], const float (&init)[C::TN]) {
  static_assert(C::BM == 256 && C::BN == 256 && C::WM == 2 && C::WN == 4 && C::MF == 16 && C::STAGES == 2 && C::ESZ == 2, "ping-pong geometry");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wid >> 2, wn = wid & 3;
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = init[j];

  constexpr int HALF = 16384;
  int oa[2][2], ob[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      oa[h][s] = TA ? h * HALF + (wid * 2 + s) * 1024 : pp_piece_a<C>(wid, h, s) * 1024;
      ob[h][s] = C::A_BYTES + (TB ? h * HALF + (wid * 2 + s) * 1024 : pp_piece_b<C>(wid, h, s) * 1024);
    }
  auto stage_ah = [&](int h, int t) {
    char* sb = smem + (t & 1) * C::STAGE_BYTES;
    glds16(src.a_half(h, 0, t), sb + oa[h][0]);
    glds16(src.a_half(h, 1, t), sb + oa[h][1]);
  };
  auto stage_bh = [&](int h, int t) {
    char* sb = smem + (t & 1) * C::STAGE_BYTES;
    glds16(src.b_half(h, 0, t), sb + ob[h][0]);
    glds16(src.b_half(h, 1, t), sb + ob[h][1]);
  };
  const int lr = lane & 15, lq = lane >> 4, sw = (lr >> 1) & 7;
  int foff[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) foff[ks] = lr * 128 + (((ks * 4 + lq) ^ sw) << 4);
  const int a_wave = grp * 128 * 128;
  const int b_wave = C::A_BYTES + wn * 64 * 128;
  constexpr int BLK = 16 * 128;
  auto frag_a = [&](const char* cs, int h, int i, int ks) -> bf16x8_t {
    if constexpr (TA) return tr_frag16<C, 128>(cs + h * HALF, grp * 64 + i * 16, ks, lane);
    else return *reinterpret_cast<const bf16x8_t*>(cs + a_wave + (h * 4 + i) * BLK + foff[ks]);
  };
  auto frag_b = [&](const char* cs, int h, int j, int ks) -> bf16x8_t {
    if constexpr (TB) return tr_frag16<C, 128>(cs + C::A_BYTES + h * HALF, wn * 32 + j * 16, ks, lane);
    else return *reinterpret_cast<const bf16x8_t*>(cs + b_wave + (h * 2 + j) * BLK + foff[ks]);
  };

#define PP_BAR() do { __builtin_amdgcn_sched_barrier(0); __builtin_amdgcn_s_barrier(); __builtin_amdgcn_sched_barrier(0); } while (0)
#define PP_LOAD_END() do { __builtin_amdgcn_sched_barrier(0); asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); PP_BAR(); } while (0)
#define PP_MMA(I0, J0, BF) do { \
    __builtin_amdgcn_s_setprio(1); \
    _Pragma("unroll") for (int ks = 0; ks < 2; ++ks) \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) \
    _Pragma("unroll") for (int j = 0; j < 2; ++j) mma<C>(af[i][ks], BF[j][ks], acc[I0 + i][J0 + j]); \
    __builtin_amdgcn_s_setprio(0); \
    PP_BAR(); } while (0)
  stage_ah(0, 0); stage_bh(0, 0); stage_bh(1, 0); stage_ah(1, 0);
  stage_ah(0, 1); stage_bh(0, 1); stage_bh(1, 1);
  wait_vmcnt<6>();                        // k-tile 0 landed
  PP_BAR();
  bf16x8_t af[4][2], bx[2][2], by[2][2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) bx[j][ks] = frag_b(smem, 0, j, ks);
  if (grp == 1) PP_BAR();                 // stagger: group 1 runs one barrier behind group 0

  // bx holds the k-tile's B-lo fragments; by takes its B-hi ones and, once those are used, B-lo of the next k-tile
  for (int t = 0; t < KT; ++t) {
    const char* cs = smem + (t & 1) * C::STAGE_BYTES;
    // ---- phase 0
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) af[i][ks] = frag_a(cs, 0, i, ks);
    stage_ah(1, t + 1);
    wait_vmcnt<10>();                     // B-hi(t) landed
    PP_LOAD_END();
    PP_MMA(0, 0, bx);
    // ---- phase 1
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) by[j][ks] = frag_b(cs, 1, j, ks);
    stage_ah(0, t + 2);
    wait_vmcnt<10>();                     // A-hi(t)
    PP_LOAD_END();
    PP_MMA(0, 2, by);
    // ---- phase 2
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) af[i][ks] = frag_a(cs, 1, i, ks);
    stage_bh(0, t + 2);
    wait_vmcnt<8>();                      // A-lo(t + 1) and B-lo(t + 1)
    PP_LOAD_END();
    PP_MMA(4, 2, by);
    // ---- phase 3
    const char* ns = smem + ((t + 1) & 1) * C::STAGE_BYTES;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) by[j][ks] = frag_b(ns, 0, j, ks);
    stage_bh(1, t + 2);
    PP_LOAD_END();
    PP_MMA(4, 0, bx);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) bx[j][ks] = by[j][ks];
  }
  wait_vmcnt<0>();                        // the stages past the end: the epilogue reuses the staging memory
  if (grp == 0) PP_BAR();                 // re-align the two groups: every LDS read of the main loop is complete behind this
  PP_BAR();
#undef PP_BAR
#undef PP_LOAD_END
#undef PP_MMA
}

// An operand of a product: `p` is element (x = 0, k = 0) of its first half, `ld` the bytes from one row to the next (rows are x for a
// K-contiguous operand, k for a K-major one), `lo` the bytes from the first half to the second. x >= xlim is not read: a K-contiguous
// operand repeats its last row, a K-major one gives zeros (whole 16-byte chunks). `rows`: x -> row of a K-contiguous operand, or null.
struct Operand {
  const char* p;
  int64_t ld, lo;
  int xlim;
  const int* rows;
};

// k-tiles of a product over K: SEG * ceil(K / BK); SEG 3: both operands are pairs of halves, SEG 2: one is (the other's `lo` is 0)
template <class C, int SEG> __host__ __device__ __forceinline__ int k_tiles(int K) { return SEG * ((K + C::BK - 1) / C::BK); }

// Source of both loops: k-tiles [t0, ..) of the product; k >= K reads zeros, whatever the tile index.
template <class C, bool TA, bool TB, int SEG, bool PP> struct ProductSrc {
  static constexpr int NA = PP ? 4 : C::PA, NB = PP ? 4 : C::PB;
  const char* ap[NA];
  const char* bp[NB];
  int ak[NA], bk[NB];              // first k of this lane's chunk inside a k-tile
  int64_t aks, bks;                // bytes per k
  int64_t alo, blo;
  int K, KT1, t0;
  struct At { int k; int64_t a, b; };
  __device__ __forceinline__ At tile(int t) const {
    t += t0;
    At at;
    if constexpr (SEG == 1) { at.k = t * C::BK; at.a = at.b = 0; }
    else if constexpr (SEG == 2) {
      const int seg = t >= KT1 ? 1 : 0;
      at.k = (t - seg * KT1) * C::BK;
      at.a = seg ? alo : 0;
      at.b = seg ? blo : 0;
    } else {
      const int seg = t >= 2 * KT1 ? 2 : t >= KT1 ? 1 : 0;
      at.k = (t - seg * KT1) * C::BK;
      at.a = seg == 2 ? alo : 0;
      at.b = seg == 1 ? blo : 0;
    }
    return at;
  }
  __device__ __forceinline__ const void* a(int i, const At& at) const {
    const int k = at.k + ak[i];
    return (k < K && (!TA || ap[i])) ? (const void*)(ap[i] + at.a + k * aks) : (const void*)g_zero_page;
  }
  __device__ __forceinline__ const void* b(int i, const At& at) const {
    const int k = at.k + bk[i];
    return (k < K && (!TB || bp[i])) ? (const void*)(bp[i] + at.b + k * bks) : (const void*)g_zero_page;
  }
  __device__ __forceinline__ const void* a_half(int h, int s, int t) const { return a(h * 2 + s, tile(t)); }
  __device__ __forceinline__ const void* b_half(int h, int s, int t) const { return b(h * 2 + s, tile(t)); }

  // x of piece i of one side; geometry of the loops: a piece is 8 rows of 128 bytes (K-contiguous) or whole k-rows (K-major)
  template <bool T, bool SIDE_A> static __device__ __forceinline__ void place(int i, int& x, int& k) {
    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if constexpr (PP) {
      const int h = i >> 1, s = i & 1;
      if constexpr (T) {
        const int row = (wid * 2 + s) * 4 + (lane >> 4);
        const int xi = ((lane & 15) ^ tr_swz<C, 128>(row)) * C::CH;
        k = row;
        x = SIDE_A ? (xi >> 6) * 128 + h * 64 + (xi & 63) : (xi >> 5) * 64 + h * 32 + (xi & 31);
      } else {
        x = (SIDE_A ? pp_piece_a<C>(wid, h, s) : pp_piece_b<C>(wid, h, s)) * 8 + (lane >> 3);
        k = ((lane & 7) ^ (s * 4 + (lane >> 4))) * C::CH;
      }
    } else if constexpr (T) {
      tr_stage_pos<C, SIDE_A ? C::BM : C::BN>(i, k, x);
    } else {
      x = stage_row<C>(i);
      k = stage_chunk(stage_row<C>(0)) * C::CH;
    }
  }
  template <bool T, bool SIDE_A, int NP> static __device__ __forceinline__ void side(const Operand& o, int x0, const char* (&p)[NP], int (&kk)[NP], int64_t& ks) {
    ks = T ? o.ld : (int64_t)C::ESZ;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      int x;
      place<T, SIDE_A>(i, x, kk[i]);
      x += x0;
      if constexpr (T) p[i] = x < o.xlim ? o.p + (int64_t)x * C::ESZ : nullptr;
      else {
        if (x > o.xlim - 1) x = o.xlim - 1;
        p[i] = o.p + (int64_t)(o.rows ? o.rows[x] : x) * o.ld;
      }
    }
  }
  __device__ __forceinline__ void set(const Operand& A, const Operand& B, int m0, int n0, int K_, int first) {
    side<TA, true>(A, m0, ap, ak, aks);
    side<TB, false>(B, n0, bp, bk, bks);
    alo = A.lo; blo = B.lo; K = K_; KT1 = (K_ + C::BK - 1) / C::BK; t0 = first;
  }
};

template <class C> constexpr bool is_pp() { return C::BM == 256 && C::BN == 256; }

// acc = init (a value per column of the lane) + k-tiles [t0, t1) of A . B^T at rows m0.., columns n0..
template <class C, bool TA, bool TB, int SEG>
__device__ __forceinline__ void product(char* smem, const Operand& A, const Operand& B, int m0, int n0, int K, int t0, int t1,
                                        typename C::acc_t (&acc)[C::TM][C::TN], const float (&init)[C::TN]) {
  ProductSrc<C, TA, TB, SEG, is_pp<C>()> src;
  src.set(A, B, m0, n0, K, t0);
  if constexpr (is_pp<C>()) mainloop_pp<C, TA, TB>(smem, src, t1 - t0, acc, init);
  else {
    mainloop_flex<C, decltype(src), TA, TB>(smem, src, t1 - t0, acc);
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int i = 0; i < C::TM; ++i) acc[i][j] += init[j];
  }
}
template <class C, bool TA, bool TB, int SEG>
__device__ __forceinline__ void product(char* smem, const Operand& A, const Operand& B, int m0, int n0, int K, int t0, int t1,
                                        typename C::acc_t (&acc)[C::TM][C::TN]) {
  float zero[C::TN];
#pragma unroll
  for (int j = 0; j < C::TN; ++j) zero[j] = 0.f;
  product<C, TA, TB, SEG>(smem, A, B, m0, n0, K, t0, t1, acc, zero);
}

}  // namespace gemmcore
