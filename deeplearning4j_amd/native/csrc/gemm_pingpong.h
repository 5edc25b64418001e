// Products on the LDS-DMA core for operands in either layout, and for operands given as the sum of two 16-bit halves.
//
// Large tile, 256 x 256 x 64, 8 waves as 2 (M) x 4 (N), ping-pong as in gemm_core.h (the two wave groups run one barrier apart, one reads
// fragments while the other keeps the matrix pipe busy; half-tiles are staged again as soon as both groups have read them) with two changes:
//
//   * TWO phases of 32 MFMAs to a k-tile instead of four of 16: {A-lo, all of B} and {A-hi}. Half the barriers; a phase reads 16 or 8
//     fragments (64 / 32 KiB for the four waves of a group; LDS gives 128 bytes a cycle, 32 MFMAs take 512).
//   * staging through buffer instructions: a lane's offset inside the tile is one register for the whole product, the walk along k moves the
//     scalar base, and what lies outside is an offset past the buffer's end, for which the hardware writes zeros. (Pointers cost two registers
//     each and a 64-bit add, a compare and two selects per load.)
//
//   8192 x 16384 x 2048 bf16, both operands K-contiguous, without an epilogue: 401 us (1372 TF/s) with four phases and pointers, 370 us with
//   four phases and buffers, 342 us (1605 TF/s) with two; phases by halves of k instead 366 us; B-lo read a phase ahead 353 us.
//
//   issue order: phase 0: A-hi(t+1)   phase 1: A-lo, B-lo, B-hi (t+2)       waits: phase 0 vmcnt(8) -> A-hi(t), phase 1 vmcnt(8) -> A-lo, B (t+1)
//   A slot is staged at least one barrier behind the lgkmcnt(0) that closes its last read by both groups: A-hi(t-1) is read in phase 1 of t-1,
//   A-lo / B(t) in phase 0 of t. Data is read one phase, hence one barrier of every wave, behind the wait for it.
//
//   K-contiguous operand   the core's image: 256 rows x 128 bytes, half-tile h = rows g * 128 + h * 64 + 0..63 (A) / cols wn * 64 + h * 32 + 0..31 (B)
//   K-major operand        each half-tile is an image of its own, [64 k][128 x] with a pitch of 256 bytes: 16 KiB, two 1-KiB pieces per
//                          wave like the other, so the counted waits hold unchanged; the fragments come from transposing LDS reads
//                          (one such operand: up to 20 % longer than K-contiguous ones, at 8192 x 2048 x 32768; two: 40 %)
//
// A product of fp32 operands runs on the 16-bit matrix cores as three products of halves, a = a1 + a2 with a1 = fp16(a), a2 = fp16(a - a1)
// (operands scaled by powers of two so that the largest is below 2^15):  a . b = a1 b1 + a1 b2 + a2 b1. What is left out of an element is 2^-24 of it,
// or 2^-40 of the largest element that shares its factor (the second half's smallest step) where that is more.
// The three are one long product whose k-tiles come in threes, (a1, b1), (a1, b2), (a2, b1), so that what a k-tile reads again is still in L2.
#pragma once
#include "gemm_trans.h"

namespace gemmcore {

template <class C> constexpr bool is_pp() { return C::BM == 256 && C::BN == 256; }

// An operand of a product: `p` is element (x = 0, k = 0) of its first half, `ld` the bytes from one row to the next (rows are x for a
// K-contiguous operand, k for a K-major one), `lo` the bytes from the first half to the second. x >= xlim is not read: a K-contiguous
// operand repeats its last row, a K-major one gives zeros (whole 16-byte chunks). `rows`: x -> row of a K-contiguous operand, or null.
// The large tile takes rows of less than BUF_LD bytes, and row indirections inside the first BUF_SPAN bytes.
struct Operand {
  const char* p;
  int64_t ld, lo;
  int xlim;
  const int* rows;
};
constexpr int64_t BUF_LD = 1 << 22, BUF_SPAN = (1ll << 31) - (1 << 23);

// k-tiles of a product over K: SEG * ceil(K / BK); SEG 3: both operands are pairs of halves, SEG 2: one is (the other's `lo` is 0)
template <class C, int SEG> __host__ __device__ __forceinline__ int k_tiles(int K) { return SEG * ((K + C::BK - 1) / C::BK); }

// k-tile t of the product: first k, and the halves' byte offsets
template <class C, int SEG> struct KWalk {
  int64_t alo, blo;
  int K, t0;
  struct At { int k; int64_t a, b; };
  __device__ __forceinline__ At tile(int t) const {
    t += t0;
    At at;
    const int k = t / SEG, seg = t - k * SEG;
    at.k = k * C::BK;
    at.a = seg == SEG - 1 && SEG > 1 ? alo : 0;
    at.b = seg == 1 ? blo : 0;
    return at;
  }
  __device__ __forceinline__ void walk(const Operand& A, const Operand& B, int K_, int first) {
    alo = A.lo; blo = B.lo; K = K_; t0 = first;
  }
};

// ------------------------------------------------------------------------------------------------------------- 256 x 256 tile
template <class C, bool TA, bool TB, int SEG> struct BufSrc : KWalk<C, SEG> {
  typedef typename KWalk<C, SEG>::At At;
  const char *ap, *bp;             // uniform
  int64_t ald, bld;
  int av[4], bv[4];                // byte offset of this lane's chunk of piece (half, s) from the tile's first k; -1: not there
  int ak[4], bk[4];                // its first k inside a k-tile

  template <bool T, bool SIDE_A> static __device__ __forceinline__ void place(int i, int& x, int& k) {
    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63, h = i >> 1, s = i & 1;
    if constexpr (T) {
      const int row = (wid * 2 + s) * 4 + (lane >> 4);
      const int xi = ((lane & 15) ^ tr_swz<C, 128>(row)) * C::CH;
      k = row;
      x = SIDE_A ? (xi >> 6) * 128 + h * 64 + (xi & 63) : (xi >> 5) * 64 + h * 32 + (xi & 31);
    } else {
      x = (SIDE_A ? pp_piece_a<C>(wid, h, s) : pp_piece_b<C>(wid, h, s)) * 8 + (lane >> 3);
      k = ((lane & 7) ^ (s * 4 + (lane >> 4))) * C::CH;
    }
  }
  template <bool T, bool SIDE_A> static __device__ __forceinline__ void side(const Operand& o, int x0, const char*& base, int (&v)[4], int (&kk)[4]) {
    base = o.rows ? o.p : o.p + (int64_t)x0 * (T ? (int64_t)C::ESZ : o.ld);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int x;
      place<T, SIDE_A>(i, x, kk[i]);
      if constexpr (T) v[i] = x0 + x < o.xlim ? kk[i] * (int)o.ld + x * C::ESZ : -1;
      else {
        if (x0 + x > o.xlim - 1) x = o.xlim - 1 - x0;
        v[i] = (o.rows ? o.rows[x0 + x] : x) * (int)o.ld + kk[i] * C::ESZ;
      }
    }
  }
  __device__ __forceinline__ void set(const Operand& A, const Operand& B, int m0, int n0, int K, int first) {
    side<TA, true>(A, m0, ap, av, ak);
    side<TB, false>(B, n0, bp, bv, bk);
    ald = A.ld; bld = B.ld;
    this->walk(A, B, K, first);
  }
  static __device__ __forceinline__ void load(const char* base, int off, char* lds) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00027000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_vptr_t)lds, 16, off, 0, 0, 0);
  }
  // both pieces of half h of k-tile t; k >= K (the tail, and tiles past the end) as zeros
  __device__ __forceinline__ void a_half(int h, int t, char* l0, char* l1) const {
    const At at = this->tile(t);
    const char* base = ap + at.a + (TA ? at.k * ald : (int64_t)at.k * C::ESZ);
    load(base, at.k + ak[h * 2] < this->K ? av[h * 2] : -1, l0);
    load(base, at.k + ak[h * 2 + 1] < this->K ? av[h * 2 + 1] : -1, l1);
  }
  __device__ __forceinline__ void b_half(int h, int t, char* l0, char* l1) const {
    const At at = this->tile(t);
    const char* base = bp + at.b + (TB ? at.k * bld : (int64_t)at.k * C::ESZ);
    load(base, at.k + bk[h * 2] < this->K ? bv[h * 2] : -1, l0);
    load(base, at.k + bk[h * 2 + 1] < this->K ? bv[h * 2 + 1] : -1, l1);
  }
};

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
  auto stage_a = [&](int h, int t) {
    char* sb = smem + (t & 1) * C::STAGE_BYTES;
    src.a_half(h, t, sb + oa[h][0], sb + oa[h][1]);
  };
  auto stage_b = [&](int h, int t) {
    char* sb = smem + (t & 1) * C::STAGE_BYTES;
    src.b_half(h, t, sb + ob[h][0], sb + ob[h][1]);
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
#define PP_MMA(I0) do { \
    __builtin_amdgcn_s_setprio(1); \
    _Pragma("unroll") for (int h = 0; h < 2; ++h) \
    _Pragma("unroll") for (int ks = 0; ks < 2; ++ks) \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) \
    _Pragma("unroll") for (int j = 0; j < 2; ++j) mma<C>(af[i][ks], bf[h][j][ks], acc[I0 + i][h * 2 + j]); \
    __builtin_amdgcn_s_setprio(0); \
    PP_BAR(); } while (0)
  stage_a(0, 0); stage_b(0, 0); stage_b(1, 0); stage_a(1, 0);
  stage_a(0, 1); stage_b(0, 1); stage_b(1, 1);
  wait_vmcnt<6>();                        // k-tile 0 landed
  PP_BAR();
  if (grp == 1) PP_BAR();                 // stagger: group 1 runs one barrier behind group 0

  bf16x8_t af[4][2], bf[2][2][2];
#pragma unroll 1
  for (int t = 0; t < KT; ++t) {
    const char* cs = smem + (t & 1) * C::STAGE_BYTES;
    // ---- phase 0
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) af[i][ks] = frag_a(cs, 0, i, ks);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) bf[h][j][ks] = frag_b(cs, h, j, ks);
    stage_a(1, t + 1);
    wait_vmcnt<8>();                      // A-hi(t): A-lo, B-lo, B-hi (t+1) and A-hi(t+1) may be in flight
    PP_LOAD_END();
    PP_MMA(0);
    // ---- phase 1
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) af[i][ks] = frag_a(cs, 1, i, ks);
    stage_a(0, t + 2); stage_b(0, t + 2); stage_b(1, t + 2);
    wait_vmcnt<8>();                      // A-lo, B-lo, B-hi (t+1): A-hi(t+1) and the six above may be in flight
    PP_LOAD_END();
    PP_MMA(4);
  }
  wait_vmcnt<0>();                        // the stages past the end: the epilogue reuses the staging memory
  if (grp == 0) PP_BAR();                 // re-align the two groups: every LDS read of the main loop is complete behind this
  PP_BAR();
#undef PP_BAR
#undef PP_LOAD_END
#undef PP_MMA
}

// ------------------------------------------------------------------------------------------------------------- smaller tiles
// Source of the loop below: a pointer per piece.
template <class C, bool TA, bool TB, int SEG> struct PtrSrc : KWalk<C, SEG> {
  typedef typename KWalk<C, SEG>::At At;
  const char* ap[C::PA];
  const char* bp[C::PB];
  int ak[C::PA], bk[C::PB];        // first k of this lane's chunk inside a k-tile
  int64_t aks, bks;                // bytes per k
  __device__ __forceinline__ const void* a(int i, const At& at) const {
    const int k = at.k + ak[i];
    return (k < this->K && (!TA || ap[i])) ? (const void*)(ap[i] + at.a + k * aks) : (const void*)g_zero_page;
  }
  __device__ __forceinline__ const void* b(int i, const At& at) const {
    const int k = at.k + bk[i];
    return (k < this->K && (!TB || bp[i])) ? (const void*)(bp[i] + at.b + k * bks) : (const void*)g_zero_page;
  }
  template <bool T, int BX, int NP> static __device__ __forceinline__ void side(const Operand& o, int x0, const char* (&p)[NP], int (&kk)[NP], int64_t& ks) {
    ks = T ? o.ld : (int64_t)C::ESZ;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      int x;
      if constexpr (T) tr_stage_pos<C, BX>(i, kk[i], x);
      else { x = stage_row<C>(i); kk[i] = stage_chunk(stage_row<C>(0)) * C::CH; }
      x += x0;
      if constexpr (T) p[i] = x < o.xlim ? o.p + (int64_t)x * C::ESZ : nullptr;
      else {
        if (x > o.xlim - 1) x = o.xlim - 1;
        p[i] = o.p + (int64_t)(o.rows ? o.rows[x] : x) * o.ld;
      }
    }
  }
  __device__ __forceinline__ void set(const Operand& A, const Operand& B, int m0, int n0, int K, int first) {
    side<TA, C::BM>(A, m0, ap, ak, aks);
    side<TB, C::BN>(B, n0, bp, bk, bks);
    this->walk(A, B, K, first);
  }
};

// The multi-stage loop of gemm_trans.h (mainloop_flex). fp32 operands: a matrix instruction adds four products, so a sum over K is a chain of
// K / 4 roundings; every four k-tiles (128 k) the chain ends in a second set of accumulators, which leaves 32 + K / 128 of them.
template <class C, class Src, bool TA, bool TB>
__device__ __forceinline__ void mainloop_stages(char* smem, const Src& src, int KT, typename C::acc_t (&acc)[C::TM][C::TN]) {
  static_assert(C::MF == 16 && C::STAGES > 1, "16x16 MFMA geometry");
  constexpr bool FLUSH = C::DT == DT_F32;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid / C::WN, wn = wid - wm * C::WN;
  typename C::acc_t part[FLUSH ? C::TM : 1][FLUSH ? C::TN : 1];
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int e = 0; e < C::ACC; ++e) { acc[i][j][e] = 0.f; if constexpr (FLUSH) part[i][j][e] = 0.f; }
  auto stage = [&](int t) {
    char* sb = smem + (t % C::STAGES) * C::STAGE_BYTES;
    const auto ts = src.tile(t);
#pragma unroll
    for (int i = 0; i < C::PA; ++i) glds16(src.a(i, ts), sb + (wid + i * C::NW) * 1024);
#pragma unroll
    for (int i = 0; i < C::PB; ++i) glds16(src.b(i, ts), sb + C::A_BYTES + (wid + i * C::NW) * 1024);
  };
  const int lr = lane & 15, lq = lane >> 4, sw = (lr >> 1) & 7;
  int foff[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) foff[ks] = lr * 128 + (((ks * 4 + lq) ^ sw) << 4);
  const int a_row0 = wm * (C::BM / C::WM), b_row0 = wn * (C::BN / C::WN);
  constexpr int BLK = 16 * 128;
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s)
    if (s < KT) stage(s);
  for (int t = 0; t < KT; ++t) {
    const int ahead = KT - 1 - t;                 // k-tiles issued behind this one may stay in flight
    if (C::STAGES >= 4 && ahead >= 2) wait_vmcnt<2 * C::LPT>();
    else if (C::STAGES >= 3 && ahead >= 1) wait_vmcnt<C::LPT>();
    else wait_vmcnt<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slot staged below has been read by this wave
    __builtin_amdgcn_s_barrier();
    if (t + C::STAGES - 1 < KT) stage(t + C::STAGES - 1);
    const char* cs = smem + (t % C::STAGES) * C::STAGE_BYTES;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      bf16x8_t af[C::TM], bfr[C::TN];
#pragma unroll
      for (int i = 0; i < C::TM; ++i) {
        if constexpr (TA) af[i] = tr_frag16<C, C::BM>(cs, a_row0 + i * 16, ks, lane);
        else af[i] = *reinterpret_cast<const bf16x8_t*>(cs + a_row0 * 128 + i * BLK + foff[ks]);
      }
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        if constexpr (TB) bfr[j] = tr_frag16<C, C::BN>(cs + C::A_BYTES, b_row0 + j * 16, ks, lane);
        else bfr[j] = *reinterpret_cast<const bf16x8_t*>(cs + C::A_BYTES + b_row0 * 128 + j * BLK + foff[ks]);
      }
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
          if constexpr (FLUSH) mma<C>(af[i], bfr[j], part[i][j]);
          else mma<C>(af[i], bfr[j], acc[i][j]);
        }
    }
    if constexpr (FLUSH)
      if ((t & 3) == 3 || t == KT - 1) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int j = 0; j < C::TN; ++j)
#pragma unroll
            for (int e = 0; e < C::ACC; ++e) { acc[i][j][e] += part[i][j][e]; part[i][j][e] = 0.f; }
      }
  }
  __builtin_amdgcn_s_barrier();
}

// acc = init (a value per column of the lane) + k-tiles [t0, t1) of A . B^T at rows m0.., columns n0..
template <class C, bool TA, bool TB, int SEG>
__device__ __forceinline__ void product(char* smem, const Operand& A, const Operand& B, int m0, int n0, int K, int t0, int t1,
                                        typename C::acc_t (&acc)[C::TM][C::TN], const float (&init)[C::TN]) {
  if constexpr (is_pp<C>()) {
    BufSrc<C, TA, TB, SEG> src;
    src.set(A, B, m0, n0, K, t0);
    mainloop_pp<C, TA, TB>(smem, src, t1 - t0, acc, init);
  } else {
    PtrSrc<C, TA, TB, SEG> src;
    src.set(A, B, m0, n0, K, t0);
    mainloop_stages<C, decltype(src), TA, TB>(smem, src, t1 - t0, acc);
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
