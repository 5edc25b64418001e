// Losses over a large vocabulary straight from the hidden states (ops/vocab_loss.py): the logits z = h W^T + b are never written to
// memory. Two losses share the kernels:
//
//   cross entropy    loss_n = lse_n - (1 - e) z[n, y_n] - (e / V) sum_j z[n, j]                       dz = c_n (q - (1 - e) [j = y_n] - e / V)
//   distillation     loss_n = T^2 (sum_k p_k log p_k - sum_k p_k z'[n, i_k] + P_n lse_n), z' = z / T  dz = c_n T (P_n q - sum_{k: i_k = j} p_k)
//
// with q = exp(z - lse), p = softmax over the K teacher logits / T and P_n = sum_k p_k (1, or 0 for a row without entries).
//
// Forward: a product tile h W^T stays in the accumulators; its epilogue leaves one (max, sum of exp) pair per row and column tile, which
// combine_kernel joins. Backward: the same product again, piece by piece of the vocabulary; the epilogue turns the accumulators into dz
// (a piece of at most some hundred MiB), and two products consume it: dh += dz W and dW = dz^T h. Rows without a label / teacher entry
// are left out of all products: rows_kernel writes the list of the others, the kernels read their number on the device.
#include "gemm_trans.h"

using namespace gemmcore;

namespace {

constexpr float NEG_INF = -__builtin_inff();

__device__ __forceinline__ float load_f(const void* p, int64_t i, int dt) {
  if (dt == DT_F32) return reinterpret_cast<const float*>(p)[i];
  const uint16_t v = reinterpret_cast<const uint16_t*>(p)[i];
  return dt == DT_BF16 ? bf2f(v) : (float)__builtin_bit_cast(_Float16, v);
}
__device__ __forceinline__ void store_f(void* p, int64_t i, int dt, float v) {
  if (dt == DT_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dt == DT_BF16) reinterpret_cast<uint16_t*>(p)[i] = f2bf(v);
  else reinterpret_cast<uint16_t*>(p)[i] = __builtin_bit_cast(uint16_t, (_Float16)v);
}

// all-lanes reductions over the 16 lanes that share the accumulator rows of a 16x16 block: rotations inside a DPP row, no LDS traffic
template <int ROR> __device__ __forceinline__ float dpp_ror(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x120 + ROR, 0xf, 0xf, true));
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, dpp_ror<8>(v)); v = fmaxf(v, dpp_ror<4>(v)); v = fmaxf(v, dpp_ror<2>(v)); return fmaxf(v, dpp_ror<1>(v));
}
__device__ __forceinline__ float sum16(float v) {
  v += dpp_ror<8>(v); v += dpp_ror<4>(v); v += dpp_ror<2>(v); return v + dpp_ror<1>(v);
}

// ------------------------------------------------------------------------------------------------------------------------ rows
// rows[0 .. count) = rows that take part, in order; rows[count .. N) = the others; loss of the others = 0.
// One workgroup: a scan of N flags, 1024 at a time.
__global__ void __launch_bounds__(1024) rows_kernel(const int64_t* __restrict__ lab64, const int* __restrict__ lab32, int64_t ignore,
                                                    const float* __restrict__ mass, int N, int* __restrict__ rows, int* __restrict__ count,
                                                    float* __restrict__ loss) {
  __shared__ int wsum[16];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  int done = 0;
  for (int base = 0; base < N; base += 1024) {
    const int n = base + tid;
    bool ok = false;
    if (n < N) ok = lab64 ? lab64[n] != ignore : lab32 ? (int64_t)lab32[n] != ignore : mass[n] != 0.f;
    const unsigned long long b = __ballot(ok);
    if (lane == 0) wsum[wid] = __popcll(b);
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < 16; ++w) { if (w < wid) before += wsum[w]; all += wsum[w]; }
    const int at = done + before + __popcll(b & ((1ull << lane) - 1));
    if (n < N) {
      if (ok) rows[at] = n;
      else { rows[N - 1 - (n - at)] = n; loss[n] = 0.f; }      // n - at rows before this one do not take part
    }
    done += all;
    __syncthreads();
  }
  if (tid == 0) *count = done;
}

// ------------------------------------------------------------------------------------------------------------------------ teacher
// One wave per row: p = softmax(teacher / T) over the entries with an index >= 0, ent = sum p log p, mass = sum p as 1 or 0 (0: no entry
// with a finite weight), and psum_k = the summed p of all entries with entry k's index (an index may come twice). K <= 1024.
__global__ void __launch_bounds__(256) teacher_kernel(const void* __restrict__ idx, int idx64, const void* __restrict__ t, int tdt, int N, int K,
                                                      float invT, float* __restrict__ p, float* __restrict__ psum, float* __restrict__ ent,
                                                      float* __restrict__ mass) {
  __shared__ int si[4][1024];
  __shared__ float sp[4][1024];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int n = blockIdx.x * 4 + wid;
  if (n >= N) return;                                   // waves work alone below: no block barrier
  float m = NEG_INF;
  bool bad = false;
  for (int k = lane; k < K; k += 64) {
    const int64_t o = (int64_t)n * K + k;
    const int64_t i = idx64 ? reinterpret_cast<const int64_t*>(idx)[o] : (int64_t)reinterpret_cast<const int*>(idx)[o];
    const float v = i < 0 ? NEG_INF : load_f(t, o, tdt) * invT;
    si[wid][k] = i > 0x7fffffff ? 0x7fffffff : (int)i;
    sp[wid][k] = v;
    bad |= !(v < __builtin_inff());                     // NaN or +inf
    m = fmaxf(m, v);
  }
  bad = __any(bad);
  m = wave_max(m);
  float s = 0.f;
  for (int k = lane; k < K; k += 64) {
    const float e = m == NEG_INF ? 0.f : __expf(sp[wid][k] - m);
    s += e;
  }
  s = wave_sum(s);
  const float inv = s > 0.f ? 1.f / s : 0.f, ls = s > 0.f ? __logf(s) : 0.f;
  float h = 0.f;
  for (int k = lane; k < K; k += 64) {
    const float d = sp[wid][k] - m;
    float w = m == NEG_INF ? 0.f : __expf(d) * inv;
    if (w > 0.f) h += w * (d - ls);
    if (bad) w = __builtin_nanf("");
    sp[wid][k] = w;
    p[(int64_t)n * K + k] = w;
  }
  h = wave_sum(h);
  if (lane == 0) {
    ent[n] = bad ? __builtin_nanf("") : h;
    mass[n] = bad || s > 0.f ? 1.f : 0.f;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (int k = lane; k < K; k += 64) {
    const int mine = si[wid][k];
    float q = 0.f;
    for (int j = 0; j < K; ++j) q += si[wid][j] == mine ? sp[wid][j] : 0.f;
    psum[(int64_t)n * K + k] = q;
  }
}

// z'[m, i_k] for the entries that count, and cross_n = sum_k p_k z'[n, i_k]: one wave per row, dot products along the hidden axis
// (W rows are contiguous here; `vstride` 1 and `dstride` V walk the [D, V] layout). An index >= V makes the row NaN.
__global__ void __launch_bounds__(256) gather_kernel(const void* __restrict__ h, int64_t ldh, const void* __restrict__ W, int64_t vstride,
                                                     int64_t dstride, const void* __restrict__ bias, int bdt, int dt, int D, int V,
                                                     const void* __restrict__ idx, int idx64, int K, float invT, const float* __restrict__ p,
                                                     const int* __restrict__ rows, const int* __restrict__ count, float* __restrict__ zk,
                                                     float* __restrict__ cross) {
  const int lane = threadIdx.x & 63;
  const int m = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= *count) return;
  const int n = rows[m];
  float acc = 0.f;
  for (int k = 0; k < K; ++k) {
    const int64_t o = (int64_t)n * K + k;
    const float pk = p[o];
    if (pk == 0.f) continue;
    const int64_t i = idx64 ? reinterpret_cast<const int64_t*>(idx)[o] : (int64_t)reinterpret_cast<const int*>(idx)[o];
    float z = __builtin_nanf("");
    if (i >= 0 && i < V) {
      float s = 0.f;
      for (int d = lane; d < D; d += 64) s += load_f(h, n * ldh + d, dt) * load_f(W, i * vstride + d * dstride, dt);
      z = (wave_sum(s) + (bias ? load_f(bias, i, bdt) : 0.f)) * invT;
    }
    if (lane == 0) zk[o] = z;
    acc += pk * z;
  }
  if (lane == 0) cross[n] = acc;
}

// ------------------------------------------------------------------------------------------------------------------------ scores
struct ScoreP {
  const void* H; int64_t ldh;            // [N, D]
  const void* W; int64_t ldw;            // [V, D], or [D, V] (TB)
  const void* bias; int bdt;
  const int* rows; const int* count;
  const int64_t* lab64; const int* lab32;
  int N, D, V, v0, v1;                   // columns [v0, v1) of the vocabulary
  float invT, smooth_v;                  // 1 / T;  e / V
  // statistics
  float2* part; float* tz; float* zs;    // part [ntiles][N]; target score [N]; zs [ntiles][N] = sum of z * e / V (or null)
  // gradient
  const float* lse; const float* coef; const float* mass;   // per position in `rows` (mass per row, or null = 1)
  float keep;                            // 1 - e
  void* G; int64_t ldg;                  // [rows up to a tile][ldg], column v at v - v0
};

__device__ __forceinline__ int64_t label_of(const ScoreP& p, int n) {
  return p.lab64 ? p.lab64[n] : p.lab32 ? (int64_t)p.lab32[n] : -1;
}

template <class C, bool TB> __device__ __forceinline__ void score_src(FlexSrc<C, false, TB>& src, const ScoreP& p, int m0, int n0, int count) {
  src.kb = 0; src.ke = p.D;
  src.kchunk = stage_chunk(stage_row<C>(0)) * C::CH;
  src.a_kstride = 0;
  src.b_kstride = p.ldw * C::ESZ;
#pragma unroll
  for (int i = 0; i < C::PA; ++i) {
    int m = m0 + stage_row<C>(i);
    if (m > count - 1) m = count - 1;                   // results of the rows past the end are not used
    src.ap[i] = (const char*)p.H + (int64_t)p.rows[m] * p.ldh * C::ESZ;
  }
#pragma unroll
  for (int i = 0; i < C::PB; ++i) {
    if constexpr (TB) {
      int row, x;
      tr_stage_pos<C, C::BN>(i, row, x);
      src.brow[i] = row;
      src.bp[i] = (n0 + x < p.v1) ? (const char*)p.W + (int64_t)(n0 + x) * C::ESZ : nullptr;
    } else {
      int n = n0 + stage_row<C>(i);
      if (n > p.V - 1) n = p.V - 1;
      src.bp[i] = (const char*)p.W + (int64_t)n * p.ldw * C::ESZ;
    }
  }
}

template <class C, bool TB, bool GRAD>
__global__ void __launch_bounds__(C::NT) score_kernel(const ScoreP p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int count = *p.count;
  const int mtiles = (count + C::BM - 1) / C::BM, ntiles = (p.v1 - p.v0 + C::BN - 1) / C::BN;
  if ((int)blockIdx.x >= mtiles * ntiles) return;
  int mt, nt;
  tile_coords(xcd_remap(blockIdx.x, mtiles * ntiles), mtiles, ntiles, 8, mt, nt);
  const int m0 = mt * C::BM, n0 = p.v0 + nt * C::BN;
  typename C::acc_t acc[C::TM][C::TN];
  {
    FlexSrc<C, false, TB> src;
    score_src<C, TB>(src, p, m0, n0, count);
    mainloop_flex<C, FlexSrc<C, false, TB>, false, TB>(smem, src, (p.D + C::BK - 1) / C::BK, acc);
  }
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int wm = wid / C::WN, wn = wid - wm * C::WN, lc = lane & 15;
  const int row0 = wm * (C::BM / C::WM) + (lane >> 4) * 4, col0 = wn * (C::BN / C::WN) + lc;
  float bv[C::TN];
#pragma unroll
  for (int j = 0; j < C::TN; ++j) {
    const int col = n0 + col0 + j * 16;
    bv[j] = col < p.v1 ? (p.bias ? load_f(p.bias, col, p.bdt) * p.invT : 0.f) : NEG_INF;
  }
  constexpr int OSZ = C::ESZ, PITCH = C::BN * OSZ + 16;
  float* sf = reinterpret_cast<float*>(smem + (GRAD ? C::BM * PITCH : 0));
  int* slab = reinterpret_cast<int*>(sf);                        // label's column inside the tile, or -1
  for (int r = tid; r < C::BM; r += C::NT) {
    const int m = m0 + r;
    int lab = -1;
    float c = 0.f, l = 0.f;
    if (m < count) {
      const int n = p.rows[m];
      const int64_t y = label_of(p, n) - n0;
      lab = y >= 0 && y < C::BN && y + n0 < p.v1 ? (int)y : -1;
      if constexpr (GRAD) { c = p.coef[m]; l = p.lse[m]; if (p.mass) sf[3 * C::BM + r] = c * p.mass[n]; else sf[3 * C::BM + r] = c; }
    } else if constexpr (GRAD) sf[3 * C::BM + r] = 0.f;
    slab[r] = lab;
    if constexpr (GRAD) { sf[C::BM + r] = c; sf[2 * C::BM + r] = l; }
  }
  __syncthreads();
  if constexpr (!GRAD) {
    float* sM = sf + C::BM;                                      // [WN][BM]
    float* sS = sM + C::WN * C::BM;
    float* sZ = sS + C::WN * C::BM;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = row0 + i * 16 + q;
        const int lab = slab[r] - col0;
        float z[C::TN], m = NEG_INF, zsum = 0.f;
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
          z[j] = acc[i][j][q] * p.invT + bv[j];
          m = fmaxf(m, z[j]);
          if (lab == j * 16) p.tz[m0 + r] = z[j];
          if (p.zs && n0 + col0 + j * 16 < p.v1) zsum += z[j] * p.smooth_v;
        }
        float mm = max16(m);
        const float ref = mm == NEG_INF ? 0.f : mm;
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < C::TN; ++j) s += __expf(z[j] - ref);  // the maximum passes over a NaN score, the sum keeps it
        s = sum16(s);
        if (p.zs) zsum = sum16(zsum);
        if (lc == 0) { sM[wn * C::BM + r] = mm; sS[wn * C::BM + r] = s; if (p.zs) sZ[wn * C::BM + r] = zsum; }
      }
    __syncthreads();
    for (int r = tid; r < C::BM; r += C::NT) {
      if (m0 + r >= count) continue;
      float m = NEG_INF, s = 0.f, z = 0.f;
#pragma unroll
      for (int w = 0; w < C::WN; ++w) m = fmaxf(m, sM[w * C::BM + r]);
#pragma unroll
      for (int w = 0; w < C::WN; ++w) {
        const float mw = sM[w * C::BM + r], sw = sS[w * C::BM + r];
        s += mw == NEG_INF ? sw : sw * __expf(mw - m);
        if (p.zs) z += sZ[w * C::BM + r];
      }
      p.part[(int64_t)nt * p.N + m0 + r] = make_float2(m, s);
      if (p.zs) p.zs[(int64_t)nt * p.N + m0 + r] = z;
    }
  } else {
    typedef typename Out<C::DT == DT_F32 ? OT_F32 : C::DT == DT_F16 ? OT_F16 : OT_BF16>::T OTy;
    typedef Out<C::DT == DT_F32 ? OT_F32 : C::DT == DT_F16 ? OT_F16 : OT_BF16> O;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = row0 + i * 16 + q;
        const int lab = slab[r] - col0;
        const float c = sf[C::BM + r], l = sf[2 * C::BM + r], cm = sf[3 * C::BM + r];
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
          float g = cm * __expf(acc[i][j][q] * p.invT + bv[j] - l) - c * p.smooth_v;
          if (lab == j * 16) g -= c * p.keep;
          if (n0 + col0 + j * 16 >= p.v1 || m0 + r >= count) g = 0.f;
          *reinterpret_cast<OTy*>(smem + r * PITCH + (col0 + j * 16) * OSZ) = O::cv(g);
        }
      }
    __syncthreads();
    constexpr int CPR = C::BN * OSZ / 16;
    char* out = (char*)p.G + ((int64_t)m0 * p.ldg + (n0 - p.v0)) * OSZ;
    for (int idx = tid; idx < C::BM * CPR; idx += C::NT) {
      const int r = idx / CPR, ch = idx - r * CPR;
      *reinterpret_cast<f32x4*>(out + (int64_t)r * p.ldg * OSZ + ch * 16) = *reinterpret_cast<const f32x4*>(smem + r * PITCH + ch * 16);
    }
  }
}

// joins the (max, sum) pairs of a row's column tiles; R rows x 256 / R tile groups per workgroup
struct CombineP {
  const float2* part; const float* zs; const float* tz;
  const int* rows; const int* count;
  const int64_t* lab64; const int* lab32;
  const float* ent; const float* cross; const float* mass;      // distillation (ent != null)
  int N, V, ntiles;
  float keep, T;
  float* lse; float* loss;
};
template <int R>
__global__ void __launch_bounds__(256) combine_kernel(const CombineP p) {
  constexpr int GR = 256 / R;
  __shared__ float sm[GR][R], ss[GR][R], sz[GR][R];
  const int r = threadIdx.x % R, g = threadIdx.x / R;
  const int m = blockIdx.x * R + r, count = *p.count;
  if ((int)blockIdx.x * R >= count) return;
  float mx = NEG_INF, s = 0.f, z = 0.f;
  if (m < count) {
#pragma unroll 4
    for (int t = g; t < p.ntiles; t += GR) {
      const float2 v = p.part[(int64_t)t * p.N + m];
      const float nm = fmaxf(mx, v.x);
      if (nm == NEG_INF) s += v.y;
      else s = s * __expf(mx - nm) + v.y * __expf(v.x - nm);     // exp(-inf) = 0 for a tile without a finite score
      mx = nm;
      if (p.zs) z += p.zs[(int64_t)t * p.N + m];
    }
  }
  sm[g][r] = mx; ss[g][r] = s; sz[g][r] = z;
  __syncthreads();
  if (g != 0 || m >= count) return;
  for (int w = 1; w < GR; ++w) {
    const float mw = sm[w][r], nm = fmaxf(mx, mw);
    if (nm == NEG_INF) s += ss[w][r];
    else s = s * __expf(mx - nm) + ss[w][r] * __expf(mw - nm);
    mx = nm;
    z += sz[w][r];
  }
  const int n = p.rows[m];
  float lse = mx + __logf(s), loss;
  if (p.ent) {
    loss = p.T * p.T * (p.ent[n] - p.cross[n] + lse * p.mass[n]);
    if (p.cross[n] != p.cross[n]) lse = p.cross[n];
  } else {
    const int64_t y = p.lab64 ? p.lab64[n] : (int64_t)p.lab32[n];
    if (y < 0 || y >= p.V) lse = __builtin_nanf("");            // a label outside the vocabulary: loss and gradient of the row are NaN
    loss = lse - p.keep * (y < 0 || y >= p.V ? 0.f : p.tz[m]) - z;
  }
  p.lse[m] = lse;
  p.loss[n] = loss;
}

// ------------------------------------------------------------------------------------------------------------------------ backward
// coef[m] = dloss[rows[m]] * T * s,  scale = 1 / s.  s = 1, or for fp16 the power of two that puts the largest coefficient into
// [2^13, 2^14): dz is at most that large then, and entries down to 2^-38 of it stay above fp16's smallest step.
__global__ void __launch_bounds__(1024) coef_kernel(const float* __restrict__ dloss, const int* __restrict__ rows, const int* __restrict__ count,
                                                    float T, int scaled, float* __restrict__ coef, float* __restrict__ scale) {
  __shared__ float red[16];
  const int c = *count;
  float s = 1.f;
  if (scaled) {
    float mx = 0.f;
    for (int m = threadIdx.x; m < c; m += 1024) {
      const float v = fabsf(dloss[rows[m]] * T);
      if (v < __builtin_inff()) mx = fmaxf(mx, v);
    }
    mx = block_max(mx, red);
    if (mx > 0.f) {
      int e;
      frexpf(mx, &e);                                            // mx in [2^(e-1), 2^e)
      e = min(max(14 - e, -100), 100);
      s = ldexpf(1.f, e);
    }
  }
  for (int m = threadIdx.x; m < c; m += 1024) coef[m] = dloss[rows[m]] * T * s;
  if (threadIdx.x == 0) *scale = 1.f / s;
}

// the rows that take part, packed; zeros up to the next multiple of 256 rows
__global__ void __launch_bounds__(256) pack_kernel(const char* __restrict__ h, int64_t ldh_bytes, const int* __restrict__ rows,
                                                   const int* __restrict__ count, char* __restrict__ out, int64_t row_bytes) {
  const int c = *count, m = blockIdx.x;
  if (m >= (c + 255) / 256 * 256) return;
  const char* src = m < c ? h + rows[m] * ldh_bytes : nullptr;
  for (int64_t b = threadIdx.x * 16; b < row_bytes; b += 256 * 16) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (src) v = *reinterpret_cast<const f32x4*>(src + b);
    *reinterpret_cast<f32x4*>(out + m * row_bytes + b) = v;
  }
}

// the teacher's entries of a piece of dz: dz[m, i_k] = c_m (P q - psum_k), from the exact scores (entries with the same index write the
// same value)
__global__ void __launch_bounds__(256) entries_kernel(const void* __restrict__ idx, int idx64, int K, const float* __restrict__ p,
                                                      const float* __restrict__ psum, const float* __restrict__ zk, const float* __restrict__ lse,
                                                      const float* __restrict__ coef, const float* __restrict__ mass,
                                                      const int* __restrict__ rows, const int* __restrict__ count, int v0, int v1, void* G,
                                                      int64_t ldg, int dt) {
  const int lane = threadIdx.x & 63, m = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= *count) return;
  const int n = rows[m];
  for (int k = lane; k < K; k += 64) {
    const int64_t o = (int64_t)n * K + k;
    const int64_t i = idx64 ? reinterpret_cast<const int64_t*>(idx)[o] : (int64_t)reinterpret_cast<const int*>(idx)[o];
    if (i < v0 || i >= v1 || p[o] == 0.f) continue;
    store_f(G, (int64_t)m * ldg + (i - v0), dt, coef[m] * (mass[n] * __expf(zk[o] - lse[m]) - psum[o]));
  }
}

// db[v0 + v] = scale * column sum of dz: 8 columns per thread, 32 row lanes, one workgroup per 64 columns
__global__ void __launch_bounds__(256) colsum_kernel(const void* __restrict__ G, int64_t ldg, int dt, int vc, const int* __restrict__ count,
                                                     const float* __restrict__ scale, void* __restrict__ db, int bdt) {
  __shared__ float red[32][65];
  const int cg = threadIdx.x & 7, rl = threadIdx.x >> 3, c = *count;
  const int v = blockIdx.x * 64 + cg * 8;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (v < vc)                                                    // dz is zero between vc and its row stride (a multiple of 64)
    for (int m = rl; m < c; m += 32)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += load_f(G, (int64_t)m * ldg + v + e, dt);
#pragma unroll
  for (int e = 0; e < 8; ++e) red[rl][cg * 8 + e] = s[e];
  __syncthreads();
  if (threadIdx.x < 64 && (int)(blockIdx.x * 64 + threadIdx.x) < vc) {
    float a = 0.f;
    for (int r = 0; r < 32; ++r) a += red[r][threadIdx.x];
    store_f(db, blockIdx.x * 64 + threadIdx.x, bdt, a * *scale);
  }
}

// dh partial products: unit u of the grid owns output tile u % tiles and share u / tiles of the piece's columns; its fp32 tile lives in
// slab u and is added to by the following pieces. Which unit owns what depends on the number of rows alone, so the sum's order is fixed.
struct DhP {
  const void* G; int64_t ldg;
  const void* W; int64_t ldw;            // first row (column) of the piece
  const int* count;
  int D, vc, units, accum;
  float* slab;
};
__device__ __forceinline__ int dh_shares(int tiles, int units) { return tiles >= units ? 1 : units / tiles; }

template <class C, bool TB>
__global__ void __launch_bounds__(C::NT) dh_kernel(const DhP p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int count = *p.count;
  const int mtiles = (count + C::BM - 1) / C::BM, ntiles = (p.D + C::BN - 1) / C::BN, tiles = mtiles * ntiles;
  if (tiles == 0) return;
  const int shares = dh_shares(tiles, p.units);
  if ((int)blockIdx.x >= tiles * shares) return;
  const int u = xcd_remap(blockIdx.x, tiles * shares);
  const int share = u / tiles, t = u - share * tiles;
  int mt, nt;
  tile_coords(t, mtiles, ntiles, 8, mt, nt);
  const int m0 = mt * C::BM, n0 = nt * C::BN;
  const int ktiles = (p.vc + C::BK - 1) / C::BK, per = (ktiles + shares - 1) / shares;
  const int k0 = min(ktiles, share * per), k1 = min(ktiles, k0 + per);
  FlexSrc<C, false, TB> src;
  src.kb = k0 * C::BK; src.ke = min(p.vc, k1 * C::BK);
  src.kchunk = stage_chunk(stage_row<C>(0)) * C::CH;
  src.a_kstride = 0; src.b_kstride = p.ldw * C::ESZ;
#pragma unroll
  for (int i = 0; i < C::PA; ++i) src.ap[i] = (const char*)p.G + (int64_t)(m0 + stage_row<C>(i)) * p.ldg * C::ESZ;
#pragma unroll
  for (int i = 0; i < C::PB; ++i) {
    if constexpr (TB) {
      int row, x;
      tr_stage_pos<C, C::BN>(i, row, x);
      src.brow[i] = row;
      src.bp[i] = (n0 + x < p.D) ? (const char*)p.W + (int64_t)(n0 + x) * C::ESZ : nullptr;
    } else {
      int n = n0 + stage_row<C>(i);
      if (n > p.D - 1) n = p.D - 1;
      src.bp[i] = (const char*)p.W + (int64_t)n * p.ldw * C::ESZ;
    }
  }
  typename C::acc_t acc[C::TM][C::TN];
  mainloop_flex<C, FlexSrc<C, false, TB>, false, TB>(smem, src, k1 - k0, acc);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wm = wid / C::WN, wn = wid - wm * C::WN;
  float* out = p.slab + (int64_t)u * C::BM * C::BN + (wm * (C::BM / C::WM) + (lane >> 4) * 4) * C::BN + wn * (C::BN / C::WN) + (lane & 15);
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float* o = out + (i * 16 + q) * C::BN + j * 16;
        *o = p.accum ? *o + acc[i][j][q] : acc[i][j][q];
      }
}

// dh rows from the slabs, in the order of the shares; rows that take no part get zeros. One workgroup per row.
template <int BM, int BN>
__global__ void __launch_bounds__(256) dh_rows_kernel(const float* __restrict__ slab, const int* __restrict__ rows, const int* __restrict__ count,
                                                      const float* __restrict__ scale, int D, int units, void* __restrict__ dh, int64_t ldo, int dt) {
  const int m = blockIdx.x, c = *count, n = rows[m];
  const int mtiles = (c + BM - 1) / BM, ntiles = (D + BN - 1) / BN, tiles = mtiles * ntiles;
  const int shares = tiles ? dh_shares(tiles, units) : 1;
  const float s = *scale;
  for (int d = threadIdx.x; d < D; d += 256) {
    float v = 0.f;
    if (m < c) {
      const int mt = m / BM, nt = d / BN;
      const int g = mt / 8, rowsg = min(8, mtiles - g * 8);       // tile_coords with 8 row tiles to a group
      const int t = g * 8 * ntiles + nt * rowsg + (mt - g * 8);
      for (int k = 0; k < shares; ++k) v += slab[(int64_t)(k * tiles + t) * BM * BN + (m - mt * BM) * BN + (d - nt * BN)];
      v *= s;
    }
    store_f(dh, (int64_t)n * ldo + d, dt, v);
  }
}

// dW[v0 .. v0 + vc) = scale * dz^T h (SWAP 0, [V, D]) or its transpose (SWAP 1, [D, V]): both operands are walked along their rows
struct DwP {
  const void* G; int64_t ldg;
  const void* H; int64_t ldh;            // packed rows
  const int* count; const float* scale;
  void* out; int64_t ldo;
  int D, vc;
};
template <class C, int OT, bool SWAP>
__global__ void __launch_bounds__(C::NT) dw_kernel(const DwP p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int K = (*p.count + 63) / 64 * 64;
  const int M = SWAP ? p.D : p.vc, N = SWAP ? p.vc : p.D;
  const int mtiles = (M + C::BM - 1) / C::BM, ntiles = (N + C::BN - 1) / C::BN;
  int mt, nt;
  tile_coords(xcd_remap(blockIdx.x, gridDim.x), mtiles, ntiles, 8, mt, nt);
  const int m0 = mt * C::BM, n0 = nt * C::BN;
  const char* A = (const char*)(SWAP ? p.H : p.G);
  const char* B = (const char*)(SWAP ? p.G : p.H);
  const int mlim = SWAP ? p.D : (int)p.ldg, nlim = SWAP ? (int)p.ldg : p.D;   // dz is zero from vc to ldg
  FlexSrc<C, true, true> src;
  src.kb = 0; src.ke = K; src.kchunk = 0;
  src.a_kstride = (SWAP ? p.ldh : p.ldg) * C::ESZ;
  src.b_kstride = (SWAP ? p.ldg : p.ldh) * C::ESZ;
#pragma unroll
  for (int i = 0; i < C::PA; ++i) {
    int row, x;
    tr_stage_pos<C, C::BM>(i, row, x);
    src.arow[i] = row;
    src.ap[i] = m0 + x < mlim ? A + (int64_t)(m0 + x) * C::ESZ : nullptr;
  }
#pragma unroll
  for (int i = 0; i < C::PB; ++i) {
    int row, x;
    tr_stage_pos<C, C::BN>(i, row, x);
    src.brow[i] = row;
    src.bp[i] = n0 + x < nlim ? B + (int64_t)(n0 + x) * C::ESZ : nullptr;
  }
  typename C::acc_t acc[C::TM][C::TN];
  mainloop_flex<C, FlexSrc<C, true, true>, true, true>(smem, src, K / C::BK, acc);
  EpiP e;
  e.out = p.out; e.residual = nullptr; e.bias = nullptr; e.stats = nullptr; e.stat_shift = nullptr;
  e.alpha = *p.scale; e.act = ACT_NONE; e.accum = 0;
  const int64_t ldo = p.ldo;
  epilogue_impl<C, OT, ACT_NONE, 0>(smem, acc, mt, n0, N, M - m0, e, [=](int r) -> int64_t {
    return m0 + r < M ? (int64_t)(m0 + r) * ldo + n0 : (int64_t)-1;
  });
}

template <int DT> using Tile = Cfg<128, 128, 2, 2, 2, 16, DT>;

template <typename F> void allow_lds(F* fn, int bytes, DeviceOnceLds& once) { once.ensure(reinterpret_cast<const void*>(fn), bytes); }

template <int DT, bool TB, bool GRAD> int launch_score(const ScoreP& p, hipStream_t st) {
  typedef Tile<DT> C;
  const int64_t grid = (int64_t)((p.N + C::BM - 1) / C::BM) * ((p.v1 - p.v0 + C::BN - 1) / C::BN);
  constexpr int EPI = GRAD ? C::BM * (C::BN * C::ESZ + 16) + 4 * C::BM * 4 : C::BM * 4 * (1 + 3 * C::WN);
  constexpr int MAIN = C::STAGES * C::STAGE_BYTES, LDS = MAIN > EPI ? MAIN : EPI;
  static DeviceOnceLds once;
  allow_lds(&score_kernel<C, TB, GRAD>, LDS, once);
  hipLaunchKernelGGL((score_kernel<C, TB, GRAD>), dim3(grid), dim3(C::NT), LDS, st, p);
  return (int)hipGetLastError();
}
template <bool GRAD> int dispatch_score(const ScoreP& p, int dt, int tb, hipStream_t st) {
  switch (dt) {
    case DT_BF16: return tb ? launch_score<DT_BF16, true, GRAD>(p, st) : launch_score<DT_BF16, false, GRAD>(p, st);
    case DT_F16: return tb ? launch_score<DT_F16, true, GRAD>(p, st) : launch_score<DT_F16, false, GRAD>(p, st);
    case DT_F32: return tb ? launch_score<DT_F32, true, GRAD>(p, st) : launch_score<DT_F32, false, GRAD>(p, st);
  }
  return -2;
}

template <int DT, bool TB> int launch_dh(const DhP& p, int grid, hipStream_t st) {
  typedef Tile<DT> C;
  constexpr int LDS = C::STAGES * C::STAGE_BYTES;
  static DeviceOnceLds once;
  allow_lds(&dh_kernel<C, TB>, LDS, once);
  hipLaunchKernelGGL((dh_kernel<C, TB>), dim3(grid), dim3(C::NT), LDS, st, p);
  return (int)hipGetLastError();
}
template <int DT, bool SWAP> int launch_dw(const DwP& p, hipStream_t st) {
  typedef Tile<DT> C;
  constexpr int OT = DT == DT_F32 ? OT_F32 : DT == DT_F16 ? OT_F16 : OT_BF16;
  const int M = SWAP ? p.D : p.vc, N = SWAP ? p.vc : p.D;
  constexpr int LDS = C::lds_bytes(Out<OT>::SZ);
  static DeviceOnceLds once;
  allow_lds(&dw_kernel<C, OT, SWAP>, LDS, once);
  hipLaunchKernelGGL((dw_kernel<C, OT, SWAP>), dim3(((M + C::BM - 1) / C::BM) * ((N + C::BN - 1) / C::BN)), dim3(C::NT), LDS, st, p);
  return (int)hipGetLastError();
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

// rows that take part: label != ignore (labels64 / labels32), or mass != 0
DL4J_API int dl4j_vl_rows(const int64_t* labels64, const int* labels32, int64_t ignore, const float* mass, int N, int* rows, int* count,
                          float* loss, hipStream_t st) {
  if (N <= 0 || !rows || !count || !loss || (!labels64 && !labels32 && !mass)) return -2;
  hipLaunchKernelGGL(rows_kernel, dim3(1), dim3(1024), 0, st, labels64, labels32, ignore, mass, N, rows, count, loss);
  return (int)hipGetLastError();
}

DL4J_API int dl4j_vl_teacher(const void* idx, int idx64, const void* t, int tdt, int N, int K, float invT, float* p, float* psum, float* ent,
                             float* mass, hipStream_t st) {
  if (N <= 0 || K <= 0 || K > 1024 || tdt < 0 || tdt > 2 || !idx || !t || !p || !psum || !ent || !mass) return -2;
  hipLaunchKernelGGL(teacher_kernel, dim3((N + 3) / 4), dim3(256), 0, st, idx, idx64, t, tdt, N, K, invT, p, psum, ent, mass);
  return (int)hipGetLastError();
}

// sizes: N D V ldh vstride dstride dt bdt idx64 K
DL4J_API int dl4j_vl_gather(const void* h, const void* W, const void* bias, const void* idx, const float* p, const int* rows, const int* count,
                            float invT, float* zk, float* cross, const int64_t* d, hipStream_t st) {
  if (d[0] <= 0 || d[1] <= 0 || d[2] <= 0 || d[9] <= 0 || !h || !W || !idx) return -2;
  hipLaunchKernelGGL(gather_kernel, dim3((d[0] + 3) / 4), dim3(256), 0, st, h, d[3], W, d[4], d[5], bias, (int)d[7], (int)d[6], (int)d[1], (int)d[2],
                     idx, (int)d[8], (int)d[9], invT, p, rows, count, zk, cross);
  return (int)hipGetLastError();
}

// column tiles that the statistics of V columns take (rows of `part`)
DL4J_API int dl4j_vl_tiles(int V, int dt) { return (V + Tile<DT_BF16>::BN - 1) / Tile<DT_BF16>::BN; }

// d: N D V v0 v1 ldh ldw ldg dt wt bdt (wt: W is [D, V]);  f: 1/T, e/V, 1-e
// grad = 0: part / tz / zs are written; grad = 1: G [N rounded up to 128 rows][ldg]
DL4J_API int dl4j_vl_scores(int grad, const void* H, const void* W, const void* bias, const int* rows, const int* count, const int64_t* labels64,
                            const int* labels32, float* part, float* tz, float* zs, const float* lse, const float* coef, const float* mass, void* G,
                            const int64_t* d, const float* f, hipStream_t st) {
  ScoreP p;
  p.H = H; p.W = W; p.bias = bias; p.rows = rows; p.count = count; p.lab64 = labels64; p.lab32 = labels32;
  p.N = (int)d[0]; p.D = (int)d[1]; p.V = (int)d[2]; p.v0 = (int)d[3]; p.v1 = (int)d[4];
  p.ldh = d[5]; p.ldw = d[6]; p.ldg = d[7]; p.bdt = (int)d[10];
  p.invT = f[0]; p.smooth_v = f[1]; p.keep = f[2];
  p.part = (float2*)part; p.tz = tz; p.zs = zs; p.lse = lse; p.coef = coef; p.mass = mass; p.G = G;
  const int dt = (int)d[8], wt = (int)d[9], ch = dt == DT_F32 ? 4 : 8;
  if (p.N <= 0 || p.D <= 0 || p.V <= 0 || p.v0 < 0 || p.v1 > p.V || p.v0 >= p.v1 || dt < 0 || dt > 2) return -2;
  const int Dp = (p.D + ch - 1) / ch * ch;                       // rows are read in 16-byte chunks, zeros behind D (V)
  if (p.ldh % ch || p.ldh < Dp || p.ldw % ch || !aligned16(H) || !aligned16(W)) return -2;
  if (wt ? p.ldw < (p.V + ch - 1) / ch * ch || p.v0 % ch : p.ldw < Dp) return -2;
  if (grad ? (!G || !lse || !coef || p.ldg % Tile<DT_BF16>::BN || p.ldg < p.v1 - p.v0 || !aligned16(G)) : (!part || !tz)) return -2;
  return grad ? dispatch_score<true>(p, dt, wt, st) : dispatch_score<false>(p, dt, wt, st);
}

DL4J_API int dl4j_vl_combine(const float* part, const float* zs, const float* tz, const int* rows, const int* count, const int64_t* labels64,
                             const int* labels32, const float* ent, const float* cross, const float* mass, int N, int V, int ntiles, float keep,
                             float T, float* lse, float* loss, hipStream_t st) {
  if (N <= 0 || ntiles <= 0 || !part || !lse || !loss || (!ent && !labels64 && !labels32)) return -2;
  CombineP p{(const float2*)part, zs, tz, rows, count, labels64, labels32, ent, cross, mass, N, V, ntiles, keep, T, lse, loss};
  if (N <= 256) hipLaunchKernelGGL((combine_kernel<1>), dim3(N), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((combine_kernel<8>), dim3((N + 7) / 8), dim3(256), 0, st, p);
  return (int)hipGetLastError();
}

DL4J_API int dl4j_vl_coef(const float* dloss, const int* rows, const int* count, float T, int scaled, float* coef, float* scale, hipStream_t st) {
  if (!dloss || !rows || !count || !coef || !scale) return -2;
  hipLaunchKernelGGL(coef_kernel, dim3(1), dim3(1024), 0, st, dloss, rows, count, T, scaled, coef, scale);
  return (int)hipGetLastError();
}

// out: [N rounded up to 256][row_bytes]
DL4J_API int dl4j_vl_pack(const void* h, int64_t ldh_bytes, const int* rows, const int* count, void* out, int64_t row_bytes, int N, hipStream_t st) {
  if (N <= 0 || row_bytes % 16 || ldh_bytes % 16 || !aligned16(h) || !aligned16(out)) return -2;
  hipLaunchKernelGGL(pack_kernel, dim3((N + 255) / 256 * 256), dim3(256), 0, st, (const char*)h, ldh_bytes, rows, count, (char*)out, row_bytes);
  return (int)hipGetLastError();
}

DL4J_API int dl4j_vl_entries(const void* idx, int idx64, int K, const float* p, const float* psum, const float* zk, const float* lse,
                             const float* coef, const float* mass, const int* rows, const int* count, int N, int v0, int v1, void* G, int64_t ldg,
                             int dt, hipStream_t st) {
  if (N <= 0 || K <= 0 || !G || !zk) return -2;
  hipLaunchKernelGGL(entries_kernel, dim3((N + 3) / 4), dim3(256), 0, st, idx, idx64, K, p, psum, zk, lse, coef, mass, rows, count, v0, v1, G, ldg, dt);
  return (int)hipGetLastError();
}

DL4J_API int dl4j_vl_colsum(const void* G, int64_t ldg, int dt, int vc, const int* count, const float* scale, void* db, int bdt, hipStream_t st) {
  if (vc <= 0 || ldg % 64 || ldg < vc || !db) return -2;
  hipLaunchKernelGGL(colsum_kernel, dim3((vc + 63) / 64), dim3(256), 0, st, G, ldg, dt, vc, count, scale, db, bdt);
  return (int)hipGetLastError();
}

// units of the dh product's grid for N rows at most; the slab takes units * 128 * 128 floats
DL4J_API int dl4j_vl_dh_units(int N, int D) {
  const int tiles = ((N + 127) / 128) * ((D + 127) / 128);
  return tiles > 512 ? tiles : 512;
}

// d: N D vc ldg ldw dt wt accum units ; W points at the piece's first row (column)
DL4J_API int dl4j_vl_dh(const void* G, const void* W, const int* count, float* slab, const int64_t* d, hipStream_t st) {
  DhP p;
  p.G = G; p.W = W; p.count = count; p.slab = slab;
  p.D = (int)d[1]; p.vc = (int)d[2]; p.ldg = d[3]; p.ldw = d[4]; p.accum = (int)d[7]; p.units = (int)d[8];
  const int dt = (int)d[5], wt = (int)d[6], ch = dt == DT_F32 ? 4 : 8;
  if (d[0] <= 0 || p.D <= 0 || p.vc <= 0 || p.ldw % ch || p.ldg % 128 || p.ldg < p.vc || !aligned16(G) || !aligned16(W)) return -2;
  if (p.ldw < ((wt ? p.vc : p.D) + ch - 1) / ch * ch) return -2;
  if (p.units != dl4j_vl_dh_units((int)d[0], p.D) || !slab) return -2;
  switch (dt * 2 + wt) {
    case DT_BF16 * 2: return launch_dh<DT_BF16, true>(p, p.units, st);
    case DT_BF16 * 2 + 1: return launch_dh<DT_BF16, false>(p, p.units, st);
    case DT_F16 * 2: return launch_dh<DT_F16, true>(p, p.units, st);
    case DT_F16 * 2 + 1: return launch_dh<DT_F16, false>(p, p.units, st);
    case DT_F32 * 2: return launch_dh<DT_F32, true>(p, p.units, st);
    case DT_F32 * 2 + 1: return launch_dh<DT_F32, false>(p, p.units, st);
  }
  return -2;
}

DL4J_API int dl4j_vl_dh_rows(const float* slab, const int* rows, const int* count, const float* scale, int N, int D, void* dh, int64_t ldo, int dt,
                             hipStream_t st) {
  if (N <= 0 || D <= 0 || !slab || !dh) return -2;
  hipLaunchKernelGGL((dh_rows_kernel<128, 128>), dim3(N), dim3(256), 0, st, slab, rows, count, scale, D, dl4j_vl_dh_units(N, D), dh, ldo, dt);
  return (int)hipGetLastError();
}

// d: D vc ldg ldh ldo dt wt ; out points at the piece's first row (column)
DL4J_API int dl4j_vl_dw(const void* G, const void* H, const int* count, const float* scale, void* out, const int64_t* d, hipStream_t st) {
  DwP p;
  p.G = G; p.H = H; p.count = count; p.scale = scale; p.out = out;
  p.D = (int)d[0]; p.vc = (int)d[1]; p.ldg = d[2]; p.ldh = d[3]; p.ldo = d[4];
  const int dt = (int)d[5], wt = (int)d[6], ch = dt == DT_F32 ? 4 : 8;
  if (p.D <= 0 || p.vc <= 0 || p.ldg % 128 || p.ldg < p.vc || p.ldh % ch || p.ldh < (p.D + ch - 1) / ch * ch || !aligned16(G) || !aligned16(H)) return -2;
  switch (dt * 2 + wt) {
    case DT_BF16 * 2: return launch_dw<DT_BF16, false>(p, st);
    case DT_BF16 * 2 + 1: return launch_dw<DT_BF16, true>(p, st);
    case DT_F16 * 2: return launch_dw<DT_F16, false>(p, st);
    case DT_F16 * 2 + 1: return launch_dw<DT_F16, true>(p, st);
    case DT_F32 * 2: return launch_dw<DT_F32, false>(p, st);
    case DT_F32 * 2 + 1: return launch_dw<DT_F32, true>(p, st);
  }
  return -2;
}
