// Losses over a large vocabulary straight from the hidden states (ops/vocab_loss.py): the logits z = h W^T + b are never written to
// memory. Two losses share the kernels:
//
//   cross entropy    loss_n = lse_n - (1 - e) z[n, y_n] - (e / V) sum_j z[n, j]                       dz = c_n (q - (1 - e) [j = y_n] - e / V)
//   distillation     loss_n = T^2 (sum_k p_k log p_k - sum_k p_k z'[n, i_k] + P_n lse_n), z' = z / T  dz = c_n T (P_n q - sum_{k: i_k = j} p_k)
//
// with q = exp(z - lse), p = softmax over the K teacher logits / T and P_n = sum_k p_k (1, or 0 for a row without entries).
//
// What bounds it: the products. A step is four of 2 N D V operations (scores twice, since they are not kept, and the two gradients). bf16, 8192 x
// 2048 of 65536 words: 8.8 TFLOP, 6.95 ms (1265 TF/s; the loop alone reaches 1605). One forward of a few rows reads W once: 1 x 768 of 30522 words,
// 47 MB, 12 us (3.9 TB/s) of 19.
//
// Forward: a product tile h W^T stays in the accumulators; its epilogue leaves one (max, sum of exp) pair per row and column tile, which
// combine_kernel joins. Backward: the same product again, piece by piece of the vocabulary; the epilogue turns the accumulators into dz
// (a piece of at most some hundred MiB), and two products consume it: dh += dz W and dW = dz^T h. Rows without a label / teacher entry
// are left out of all products: rows_kernel writes the list of the others, the kernels read their number on the device.
//
// fp32 operands go through the 16-bit matrix cores as scaled pairs of halves (gemm_pingpong.h); small calls keep the fp32 matrix cores,
// which need no conversion of W.
#include "gemm_pingpong.h"

using namespace gemmcore;

namespace {

constexpr float NEG_INF = -__builtin_inff();
// Scores are kept in units of log 2 (z' = z / T / ln 2): every exponential is one v_exp_f32, every normaliser one v_log_f32.
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }
// A score x * scale against a reference that is one. In one instruction the exact product stands against a rounded one: what is off by half a step of
// the reference is the same for a whole row and leaves its softmax as it is, as long as an exponential holds it. Beyond LARGE (a step of 1/2; at
// 2^30 half a step is 64) the score is rounded first, so that it is 0 at most. (Always rounding first made the statistics kernel 4 % longer.)
constexpr float LARGE = 0x1p22f;
template <bool ROUND> __device__ __forceinline__ float below(float x, float scale, float ref) {
  if constexpr (ROUND) {
#pragma clang fp contract(off)
    const float z = x * scale;
    return z - ref;
  } else return __builtin_fmaf(x, scale, -ref);
}
template <bool B> struct Bool { static constexpr bool value = B; };
constexpr int KMAX = 1024;                              // teacher entries per row
typedef int i32x4 __attribute__((ext_vector_type(4)));

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
__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int*>(p)[i];
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

// (max, sum of exp) pairs: the join of two; a pair without a finite score has max -inf and sum 0 (or NaN)
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float nm = fmaxf(m, m2);
  if (nm == NEG_INF) s += s2;
  else s = s * exp2_(m - nm) + s2 * exp2_(m2 - nm);
  m = nm;
}

// fp32 operands in halves: a row of H is scaled by a power of two of its own, 2^eh, that puts its largest value into [2^14, 2^15), so that no
// row costs another one its low bits (one factor for all of H: a row 10^6 times as large as the others left their scores off by 5e-5, 10^9 by
// 0.05). A score is 2^-(eh + ew) * product + bias.
// A word of W has 2^ew, with 2^lo, the largest word's, unless its largest value lies NEAR powers of two below that word's: such a word's exponent
// goes up to WORD beyond lo. The gradient of the hidden states sums over the words, and takes the rest, 2^(lo - ew), with a copy of the scores'
// gradient that is written for it alone, where there is such a word (`wide`). A score of halves is off by 2^-40 of the factors' range, so a word
// 10^6 times smaller than the largest keeps 2^-32 of its own largest value, one 10^9 times smaller 2^-22; the gradient's copy keeps 2^-27 of a row's
// coefficient.
constexpr int NEAR = 8, WORD = 12, ZERO_ROW = 127;                 // ZERO_ROW: the exponent of a row of zeros
struct Scales { float top; int wide; };                            // top: the largest finite |w|
// the exponent that puts m into [2^14, 2^15)
__device__ __forceinline__ int scale_for(float m) {
  if (!(m > 0.f)) return 0;
  int e;
  frexpf(m, &e);
  return min(15 - e, 126);
}
__device__ __forceinline__ int lowest_word(const Scales* sc) { return scale_for(sc->top); }
__device__ __forceinline__ int word_scale(float m, int lo) { return m > 0.f ? lo + min(max(scale_for(m) - lo - NEAR, 0), min(WORD, 126 - lo)) : lo; }
// What the backward pass multiplies its products with.
struct Grad {
  float inv;        // gradients = inv * product (sum)
  int hlo;          // dW: exponent of the rows' factors, all brought to the one of the row that counts most
};
constexpr int NO_ROW = 254;                                        // the exponent of a row that adds nothing to dW
__device__ __forceinline__ float pow2(float v, int e) { return __builtin_amdgcn_ldexpf(v, e); }

// ------------------------------------------------------------------------------------------------------------------------ rows
// rows[0 .. count) = rows that take part, in order, lab their labels (-1: outside the vocabulary, or none); rows[count .. N) = the others;
// loss of the others = 0.
// One workgroup: a scan of N flags, 1024 at a time behind the loads of 8192 (bound by their latency: 4096 rows 7 us, 8192 rows 11 us).
constexpr int SCAN = 8;
__global__ void __launch_bounds__(1024) rows_kernel(const void* __restrict__ labels, int lab64, int64_t ignore, const float* __restrict__ mass, int N,
                                                    int V, int* __restrict__ rows, int* __restrict__ lab, int* __restrict__ count,
                                                    Scales* __restrict__ sc, float* __restrict__ loss) {
  __shared__ int wsum[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  int done = 0;
  for (int64_t base = 0; base < N; base += 1024 * SCAN) {
    int y[SCAN];                                                     // label; -1: none inside the vocabulary; -2: takes no part
#pragma unroll
    for (int j = 0; j < SCAN; ++j) {
      const int64_t n = base + j * 1024 + tid;
      y[j] = -2;
      if (n < N && labels) {
        const int64_t l = load_index(labels, n, lab64);
        if (l != ignore) y[j] = l >= 0 && l < V ? (int)l : -1;
      } else if (n < N && mass[n] != 0.f) y[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < SCAN; ++j) {
      const int64_t n = base + j * 1024 + tid;
      if (n - tid >= N) break;
      const unsigned long long b = __ballot(y[j] != -2);
      if (lane == 0) wsum[j & 1][wid] = __popcll(b);
      __syncthreads();                                               // (the other array was read in front of the barrier before this one)
      int before = 0, all = 0;
#pragma unroll
      for (int w = 0; w < 16; ++w) { const int c = wsum[j & 1][w]; if (w < wid) before += c; all += c; }
      const int at = done + before + __popcll(b & ((1ull << lane) - 1));
      if (n < N) {
        if (y[j] != -2) { rows[at] = (int)n; lab[at] = y[j]; }
        else { rows[N - 1 - (n - at)] = (int)n; loss[n] = 0.f; }   // n - at rows before this one do not take part
      }
      done += all;
    }
  }
  if (tid == 0) { *count = done; *sc = Scales{0.f, 0}; }
}

// ------------------------------------------------------------------------------------------------------------------------ teacher
struct TeacherP {
  const void* idx; int idx64;
  const void* t; int tdt;
  int N, V, K, P2;                       // P2: K rounded up to a power of two
  float invT;
  int tile, tiles;                       // column tiles of the score kernels
  int* sidx; float* sp; float* psum;     // [N][K], by index
  unsigned short* first;                 // [tiles + 1][N]: entries before column tile t
  float* ent; float* mass;
};
// One wave per row: p = softmax(teacher / T) over the entries with an index >= 0, ent = sum p log p, mass = 1, or 0 where no entry has a
// weight. The entries are sorted by index (a bitonic sort in LDS), so that a column tile finds its own between first[t] and first[t + 1],
// and psum, the summed p of all entries with one index, is a run. K log^2 K steps of LDS: 4096 rows x 64 entries 18 us. An index outside the vocabulary, a NaN or +inf makes ent NaN.
__global__ void __launch_bounds__(256) teacher_kernel(const TeacherP p) {
  extern __shared__ char smem[];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int n = blockIdx.x * 4 + wid;
  uint64_t* key = reinterpret_cast<uint64_t*>(smem) + wid * p.P2;            // index << 10 | entry
  float* w = reinterpret_cast<float*>(smem + 4 * 8 * p.P2) + wid * p.P2;
  if (n >= p.N) return;                                 // waves work alone: no block barrier below
  float m = NEG_INF;
  bool bad = false;
  for (int k = lane; k < p.P2; k += 64) {
    uint64_t q = ~0ull;
    float v = NEG_INF;
    if (k < p.K) {
      const int64_t o = (int64_t)n * p.K + k, i = load_index(p.idx, o, p.idx64);
      if (i >= 0) {
        const float l = load_f(p.t, o, p.tdt);
        v = l * p.invT;
        bad |= !(v < __builtin_inff()) || (i >= p.V && l != NEG_INF);
        if (i < p.V) q = (uint64_t)i << 10 | (uint64_t)k;
      }
    }
    key[k] = q;
    w[k] = v;
    m = fmaxf(m, v);
  }
  bad = __any(bad);
  m = wave_max(m);
  float s = 0.f;
  if (m != NEG_INF)
    for (int k = lane; k < p.P2; k += 64) s += __expf(w[k] - m);
  s = wave_sum(s);
  const float inv = s > 0.f ? 1.f / s : 0.f, ls = s > 0.f ? __logf(s) : 0.f;
  float h = 0.f;
  for (int k = lane; k < p.P2; k += 64) {
    const float d = w[k] - m;
    const float e = m == NEG_INF ? 0.f : __expf(d) * inv;
    if (e > 0.f) h += e * (d - ls);
    w[k] = e;
  }
  h = wave_sum(h);
  if (lane == 0) {
    p.ent[n] = bad ? __builtin_nanf("") : h;
    p.mass[n] = bad || s > 0.f ? 1.f : 0.f;
  }
  for (int size = 2; size <= p.P2; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (int c = lane; c < p.P2 / 2; c += 64) {
        const int i = (c / step) * 2 * step + (c % step), j = i + step;
        const uint64_t a = key[i], b = key[j];
        if ((a > b) == ((i & size) == 0)) { key[i] = b; key[j] = a; }
      }
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (int k = lane; k < p.K; k += 64) {
    const uint64_t q = key[k];
    const bool there = q != ~0ull;
    const int i = there ? (int)(q >> 10) : 0x7fffffff;
    float sum = 0.f;
    if (there) {
      int a = k;
      while (a > 0 && (int)(key[a - 1] >> 10) == i) --a;
      for (; a < p.K && key[a] != ~0ull && (int)(key[a] >> 10) == i; ++a) sum += w[key[a] & 1023];
    }
    const int64_t o = (int64_t)n * p.K + k;
    p.sidx[o] = i;
    p.sp[o] = there ? w[q & 1023] : 0.f;
    p.psum[o] = sum;
  }
  for (int t = lane; t <= p.tiles; t += 64) {
    const uint64_t lim = (uint64_t)t * p.tile << 10;
    int lo = 0, hi = p.K;                               // entries below the tile's first column
    while (lo < hi) { const int mid = (lo + hi) >> 1; if (key[mid] < lim) lo = mid + 1; else hi = mid; }
    p.first[(int64_t)t * p.N + n] = (unsigned short)lo;
  }
}

// ------------------------------------------------------------------------------------------------------------------------ operands
// Values and halves, four at a time; columns [C, ..) are zeros. (Vector loads from global memory take any multiple of 4 bytes.)
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void load4(const float* x, int c, int C, float (&v)[4]) {
  if (c + 4 <= C) {
    const f32x4 f = *reinterpret_cast<const f32x4_any*>(x);
    v[0] = f[0]; v[1] = f[1]; v[2] = f[2]; v[3] = f[3];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = c + j < C ? x[j] : 0.f;
  }
}
__device__ __forceinline__ float finite_max(float m, float x) { const float t = fabsf(x); return fmaxf(m, t < __builtin_inff() ? t : 0.f); }
__device__ __forceinline__ void halves(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  const float d = v - (float)hi;
  lo = (_Float16)(d == d ? d : 0.f);                    // inf - inf: an infinity stays in the first half alone
}

__device__ __forceinline__ int64_t up4(int n) { return ((int64_t)n + 3) / 4 * 4; }   // words of a cut's maxima
struct SplitP {
  const float* W; int64_t ldw; int wt, V, D;             // [V, D], or [D, V] with wt
  _Float16* wo; int64_t wcp;                             // halves of W, rows of wcp
  const float* H; int64_t ldh; _Float16* ho; int64_t dp, hcap;   // the rows that take part, packed; hcap: rows of one half
  const int* rows; const int* count;
  Scales* sc; int *eh, *ew;
  float* wmax; int cuts;                                 // largest finite |w| of every word ([D, V]: of each of `cuts` cuts of the rows)
  int chunks;                                            // [D, V]: cuts of the rows among the kernel's workgroups
  float* tops;                                           // the same of every workgroup of W in amax_kernel
  int gw, tw;                                            // workgroups of W, the others are H's; values of tops
};
constexpr int CUTS = 32, TOPS = 2048;
// Bound by reading W (30522 x 768 fp32, 94 MB: 27 us, 3.5 TB/s); the same pass cannot convert, since a word's factor depends on the largest word.
// Rows of H and words of a [V, D] table: a wave to four rows at a time. Words of a [D, V] table: a lane to four columns, workgroups of 256 columns x a cut
// of the rows.
__global__ void __launch_bounds__(256) amax_kernel(const SplitP p) {
  __shared__ float red[16];
  __shared__ f32x4 part[4][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const bool is_w = (int)blockIdx.x < p.gw;
  float top = 0.f;
  if (is_w && p.wt) {
    const int per = (p.D + p.chunks - 1) / p.chunks, units = (p.V + 255) / 256 * p.chunks;
    for (int u = blockIdx.x; u < units; u += p.gw) {
      const int strip = u / p.chunks, chunk = u - strip * p.chunks, c = strip * 256 + lane * 4, r1 = min(p.D, (chunk + 1) * per);
      float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
      for (int r = chunk * per + wid; r < r1; r += 4) {
        float v[4];
        load4(p.W + r * p.ldw + c, c, p.V, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = finite_max(m[j], v[j]);
      }
      part[wid][lane] = f32x4{m[0], m[1], m[2], m[3]};
      __syncthreads();
      if (wid == 0 && c < p.V) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = fmaxf(fmaxf(part[0][lane][j], part[1][lane][j]), fmaxf(part[2][lane][j], part[3][lane][j]));
          m[j] = x;
          top = fmaxf(top, x);
        }
        *reinterpret_cast<f32x4*>(p.wmax + chunk * up4(p.V) + c) = f32x4{m[0], m[1], m[2], m[3]};
      }
      __syncthreads();
    }
  } else {
    constexpr int G = 4;                                           // rows of a wave at a time: their loads are in flight together
    const int R = is_w ? p.V : *p.count, step = (is_w ? p.gw : gridDim.x - p.gw) * 4 * G;
    const bool whole = ((reinterpret_cast<uintptr_t>(is_w ? p.W : p.H) | (uintptr_t)((is_w ? p.ldw : p.ldh) * 4) | (uintptr_t)p.D * 4) & 15) == 0;   // 16 bytes at a time
    for (int64_t r0 = ((is_w ? blockIdx.x : blockIdx.x - p.gw) * 4 + wid) * G; r0 < R; r0 += step) {
      const float* x[G];
      float m[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int64_t r = r0 + g < R ? r0 + g : R - 1;
        x[g] = is_w ? p.W + r * p.ldw : p.H + p.rows[r] * p.ldh;
        m[g] = 0.f;
      }
      if (whole) {
#pragma unroll 4
        for (int c = lane * 4; c < p.D; c += 256)
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(x[g] + c);
            m[g] = finite_max(finite_max(finite_max(finite_max(m[g], v[0]), v[1]), v[2]), v[3]);
          }
      } else {
        for (int c = lane * 4; c < p.D; c += 256)
#pragma unroll
          for (int g = 0; g < G; ++g) {
            float v[4];
            load4(x[g] + c, c, p.D, v);
            m[g] = finite_max(finite_max(finite_max(finite_max(m[g], v[0]), v[1]), v[2]), v[3]);
          }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float t = wave_max(m[g]);
        if (lane == 0 && r0 + g < R) {
          if (is_w) p.wmax[r0 + g] = t;
          else p.eh[r0 + g] = t > 0.f ? scale_for(t) : ZERO_ROW;
        }
        top = fmaxf(top, t);
      }
    }
  }
  if (!is_w) return;
  top = block_max(top, red);
  if (threadIdx.x == 0) p.tops[blockIdx.x] = top;
}

// Bound by memory: W read once, written once in halves (30522 x 768: 188 MB, 37 us, 5.1 TB/s from what the caches keep of the pass before).
// W and the packed rows of H as scaled halves.
__global__ void __launch_bounds__(256) split_kernel(const SplitP p) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  __shared__ float red[16];
  const bool is_w = (int)blockIdx.x < p.gw;
  float top = 0.f;
  for (int i = threadIdx.x; i < p.tw; i += 256) top = fmaxf(top, p.tops[i]);
  top = block_max(top, red);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.sc->top = top;
  const int lo = scale_for(top);
  auto store4 = [](_Float16* out, int64_t half, const float (&v)[4], const float (&f)[4]) {
    _Float16 a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) halves(v[j] * f[j], a[j], b[j]);
    __builtin_memcpy(out, a, 8);
    __builtin_memcpy(out + half, b, 8);
  };
  if (is_w && p.wt) {
    const int per = (p.D + p.chunks - 1) / p.chunks, units = (p.V + 255) / 256 * p.chunks;
    for (int u = blockIdx.x; u < units; u += p.gw) {
      const int strip = u / p.chunks, chunk = u - strip * p.chunks, c = strip * 256 + lane * 4, r1 = min(p.D, (chunk + 1) * per);
      if (c >= p.wcp) continue;
      float f[4];
      f32x4 m = {0.f, 0.f, 0.f, 0.f};
      if (c < p.V) {
#pragma unroll 8
        for (int k = 0; k < p.cuts; ++k) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(p.wmax + k * up4(p.V) + c);
#pragma unroll
          for (int j = 0; j < 4; ++j) m[j] = fmaxf(m[j], x[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = word_scale(m[j], lo);
        f[j] = pow2(1.f, e);
        if (chunk == 0 && wid == 0 && c + j < p.V) {
          p.ew[c + j] = e;
          if (e != lo) p.sc->wide = 1;
        }
      }
#pragma unroll 4
      for (int r = chunk * per + wid; r < r1; r += 4) {
        float v[4];
        load4(p.W + r * p.ldw + c, c, p.V, v);
        store4(p.wo + r * p.wcp + c, (int64_t)p.D * p.wcp, v, f);
      }
    }
    return;
  }
  // a wave to 1024 values of a row, all its loads ahead of its stores
  const int64_t ldo = is_w ? p.wcp : p.dp, half = is_w ? p.V * p.wcp : p.hcap * p.dp;
  const int parts = (int)((ldo + 1023) / 1024);
  const int64_t n = (int64_t)(is_w ? p.V : *p.count) * parts, step = (int64_t)(is_w ? p.gw : gridDim.x - p.gw) * 4;
  for (int64_t u = (int64_t)(is_w ? blockIdx.x : blockIdx.x - p.gw) * 4 + wid; u < n; u += step) {
    const int64_t r = u / parts;
    const int c0 = (int)(u - r * parts) * 1024 + lane * 4;
    const float* x = is_w ? p.W + r * p.ldw : p.H + p.rows[r] * p.ldh;
    float v[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) load4(x + c0 + k * 256, c0 + k * 256, p.D, v[k]);
    const int e = is_w ? word_scale(p.wmax[r], lo) : p.eh[r] == ZERO_ROW ? 0 : p.eh[r];
    const float s = pow2(1.f, e), f[4] = {s, s, s, s};
    if (is_w && c0 == 0) {
      p.ew[r] = e;
      if (e != lo) p.sc->wide = 1;
    }
    _Float16* out = (is_w ? p.wo : p.ho) + r * ldo + c0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c0 + k * 256 < ldo) store4(out + k * 256, half, v[k], f);
  }
}

// Copies of operands whose rows do not start on 16 bytes or do not end on them: rows of Cp elements with zeros behind C. Workgroups [0, gw)
// take W, the others the rows of H that take part, one after the other. (Bound by memory; 1600 rows x 512 and 512 x 98 words in fp32: 3 us.)
struct PadP {
  const char* W; int64_t ldw; int wr, wc; char* wo; int64_t wcp;       // elements
  const char* H; int64_t ldh; int D; char* ho; int64_t dp;
  const int* rows; const int* count;
  int gw;
};
template <int ESZ>
__global__ void __launch_bounds__(256) pad_kernel(const PadP p) {
  constexpr int CH = 16 / ESZ;
  const bool is_w = (int)blockIdx.x < p.gw;
  const int count = *p.count;
  if (count == 0) return;                                          // nothing reads the copies then
  const int R = is_w ? p.wr : count, C = is_w ? p.wc : p.D;
  const int64_t q = (is_w ? p.wcp : p.dp) / CH;
  const int lane = threadIdx.x & 63, step = (is_w ? p.gw : gridDim.x - p.gw) * 4;
  for (int r = (is_w ? blockIdx.x : blockIdx.x - p.gw) * 4 + (threadIdx.x >> 6); r < R; r += step) {   // a wave to a row
    const char* row = is_w ? p.W + r * p.ldw * ESZ : p.H + p.rows[r] * p.ldh * ESZ;
    char* out = is_w ? p.wo + r * p.wcp * ESZ : p.ho + r * p.dp * ESZ;
    for (int64_t i = lane; i < q; i += 64) {
      const int c = (int)i * CH;
      const char* x = row + i * 16;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if constexpr (ESZ == 4) {
#pragma unroll
        for (int j = 0; j < CH; ++j) v[j] = c + j < C ? reinterpret_cast<const float*>(x)[j] : 0.f;
      } else {
        s16x8 t = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < CH; ++j) t[j] = c + j < C ? reinterpret_cast<const short*>(x)[j] : (short)0;
        v = __builtin_bit_cast(f32x4, t);
      }
      *reinterpret_cast<f32x4*>(out + i * 16) = v;
    }
  }
}

// The rows that take part, packed, for the weights' gradient. fp16 values and halves are brought to one factor, 2^hlo, since the product sums
// over the rows (a row's low bits are lost against the row's that counts most where it counts less, as in the sum itself).
struct PackP {
  const char* h; int64_t ldh, half_in;                             // bytes
  const int* rows;                                                 // or null: packed already
  char* out; int64_t ldo, half_out, row_bytes;
  int halves;                                                      // 1 or 2
};
__device__ __forceinline__ s16x8 halves_pow2(s16x8 v, int e) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const short x = v[j];                                          // (a bit cast of the vector's element itself reads element 0)
    v[j] = __builtin_bit_cast(short, (_Float16)pow2((float)__builtin_bit_cast(_Float16, x), e));
  }
  return v;
}
__device__ __forceinline__ void pack_row(const PackP& p, int m, int e) {
  const char* src = p.h + (p.rows ? p.rows[m] : m) * p.ldh;
  char* out = p.out + m * p.ldo;
  for (int half = 0; half < p.halves; ++half)
    for (int64_t b = threadIdx.x * 16; b < p.row_bytes; b += 256 * 16) {
      const s16x8 v = *reinterpret_cast<const s16x8*>(src + half * p.half_in + b);
      *reinterpret_cast<s16x8*>(out + half * p.half_out + b) = e == 0 ? v : halves_pow2(v, e);
    }
}
__global__ void __launch_bounds__(256) pack_kernel(const PackP p, const int* __restrict__ count, const int* __restrict__ t, const Grad* __restrict__ gr) {
  const int m = blockIdx.x;
  if (m < *count) pack_row(p, m, t ? gr->hlo - t[m] : 0);
}

// Bound by memory (65536 x 2048 bf16, 537 MB: 190 us, 2.9 TB/s).
// out[c][r] = in[row r][c] of 16-bit values, R x C, 64 x 64 at a time through LDS; blockIdx.z: the halves of a pair. `count`: R on the device,
// and `rows` the row of position r (both or none); positions from R to the next multiple of 64 become zeros. `gate`: only where *gate >= least. `t`: exponents of
// positions that are brought to one factor, 2^hlo (pack_kernel), or null.
struct TransposeP {
  const uint16_t* in; int64_t ldi, half_in;
  uint16_t* out; int64_t ldo, half_out;
  int R, C;
  const int* count; const int* rows;
  const int* gate; int least;
  const int* t; const Grad* gr;
};
__global__ void __launch_bounds__(256) transpose_kernel(const TransposeP p) {
  __shared__ uint16_t tile[64][64 + 2];
  if (p.gate && *p.gate < p.least) return;
  const int R = p.count ? *p.count : p.R, r0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
  if (r0 >= R) return;
  const uint16_t* in = p.in + blockIdx.z * p.half_in;
  uint16_t* out = p.out + blockIdx.z * p.half_out;
  const int r = threadIdx.x >> 2, q = (threadIdx.x & 3) * 16;      // 16 values of a row
  const uint16_t* src = r0 + r < R ? in + (int64_t)(p.rows ? p.rows[r0 + r] : r0 + r) * p.ldi + c0 + q : nullptr;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (src && c0 + q + h * 8 < p.C) v = *reinterpret_cast<const s16x8*>(src + h * 8);      // rows are readable in whole chunks
    if (src && p.t) v = halves_pow2(v, p.gr->hlo - p.t[r0 + r]);
#pragma unroll
    for (int e = 0; e < 8; ++e) tile[r][q + h * 8 + e] = (uint16_t)v[e];
  }
  __syncthreads();
  const int c = threadIdx.x >> 2;
  if (c0 + c >= p.C) return;
  uint16_t* dst = out + (c0 + c) * p.ldo + r0 + q;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    s16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (short)tile[q + h * 8 + e][c];
    *reinterpret_cast<s16x8*>(dst + h * 8) = v;
  }
}

// ------------------------------------------------------------------------------------------------------------------------ scores
struct ScoreP {
  Operand H, W;                          // H: [rows, D] (xlim is the count, set on the device); W: columns of the vocabulary
  const void* bias; int bdt;
  const int* rows; const int* count;
  const Scales* sc; const int *eh, *ew;  // operands in halves: exponents per position in `rows` and per word
  const int* lab;                        // per position in `rows`
  int N, D, v0, v1;                      // columns [v0, v1) of the vocabulary
  float invT, smooth_v;                  // 1 / T;  e / V
  float2* part; float* tz; float* zs;    // statistics: part [ntiles][N]; target score [N]; zs [ntiles][N] = sum of z * e / V (or null)
  // gradient, per position in `rows`: coefficient; q = exp2(z - ref) * inv
  const float* ref; const float* inv; const float* coef; const int* g;   // g: exponents inside the coefficients (fp16, halves)
  float keep;                            // 1 - e
  char* G; int64_t ldg, glo;             // [v - v0][ldg bytes]: position m at element m; second half glo bytes behind
  char* R; int64_t ldr, rlo;             // the gradient once more, row by row: [m][v - v0] (or null; 256 x 256 tiles)
  char* G2;                              // operands in halves, smaller tiles: the copy like G for the hidden states' gradient (or null)
  float* colsum; int64_t ldc;            // [row tiles][ldc] column sums of the gradient, or null
  // teacher entries (first != null)
  const unsigned short* first; const int* sidx; const float* psum; float* zk; int K;
};

// pitch of a vocabulary row of the staged gradient: 4 positions of 16 columns leave the accumulators at a time, 8 banks (of fp32 16) apart
template <class C> constexpr int grad_pitch() { return C::BM * C::ESZ + 16 * C::ESZ; }
constexpr int larger(int a, int b) { return a > b ? a : b; }
// The epilogue lays over the operand stages: the gradient; or the lanes' sums of exponentials, then the scores of the teacher's entries.
// Behind them: the rows' side arrays.
template <class C> constexpr int score_over(bool grad) {
  return larger(C::STAGES * C::STAGE_BYTES, grad ? C::BN * grad_pitch<C>() : larger(C::WN * 16 * (C::BM + 16), C::BM / C::WM * (C::BN + 4)) * 4);
}
template <class C> constexpr int score_side(bool grad) { return grad ? 4 * C::BM + C::WM * C::BN : C::BM * (1 + 3 * C::WN) + 4 * C::NW + 4; }
template <class C> constexpr int score_lds(bool grad, int seg) {
  return score_over<C>(grad) + (score_side<C>(grad) + (seg == 3 ? C::BM : 0) + (grad && C::DT == DT_F16 ? C::BM : 0)) * 4;
}

// The bias is where the accumulators start (-inf for columns past the vocabulary), so that a score is accumulator * zscale. (Operands in halves:
// the accumulators are brought to 2^-(eh + ew) * accumulator + bias behind the product.)
//
// Statistics: every exponential is taken against ONE reference per quarter wave, the largest score of its 32 rows x 64 columns (on the large
// tile), instead of the row's maximum: four cross-lane steps in all instead of four per row, and no row waits for its own maximum. A sum of
// exponentials down to 2^-64 below the reference keeps what words 2^-62 of it add (at 2^-100 a row that is sure of its word lost all the others,
// 1.7e-4 of its loss); a row that lies lower, or a reference beyond LARGE, makes the workgroup take the tile again with a reference per row and
// rounded scores. The 16 lanes that share a row leave their partial sums in LDS, where one thread per row adds them.
// (A maximum and a sum reduced over the lanes for every row, as the fallback does it, made the epilogue of a 256 x 256 tile as long as seven
// of its k-tiles.)
// Bound by the matrix cores: forward of 8192 x 2048 of 65536 words in bf16 1.72 ms (1280 TF/s), 4096 x 1024 of 32000 0.31 ms (860 TF/s: 16 k-tiles
// to an epilogue). With the gradient (exponentials, 2 or 4 bytes per score written through LDS) 1.94 and 0.35 ms.
// SEG 3: operands and gradient in halves; 2: the gradient in halves (its rounding to 16 bits then counts for nothing: few rows do not
// average it out, and for them a second pass over the gradient costs little beside W).
template <class C, bool TB, bool GRAD, int SEG>
__global__ void __launch_bounds__(C::NT) score_kernel(const ScoreP p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int count = *p.count;
  const int mtiles = (count + C::BM - 1) / C::BM, ntiles = (p.v1 - p.v0 + C::BN - 1) / C::BN;
  if ((int)blockIdx.x >= mtiles * ntiles) return;
  int mt, nt;
  tile_coords(xcd_remap(blockIdx.x, mtiles * ntiles), mtiles, ntiles, 8, mt, nt);
  const int m0 = mt * C::BM, n0 = p.v0 + nt * C::BN;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int wm = wid / C::WN, wn = wid - wm * C::WN, lc = lane & 15;
  const int row0 = wm * (C::BM / C::WM) + (lane >> 4) * 4, col0 = wn * (C::BN / C::WN) + lc;
  constexpr int OSZ = C::ESZ, PITCH = grad_pitch<C>(), RW = C::BM / C::WM, CW = C::BN / C::WN;
  const float zscale = p.invT * LOG2E;
  // the rows' label, coefficient and normaliser: on their way while the product runs
  int lab = -1;
  float rc = 0.f, rl = 3e38f, rq = 0.f;                            // rows past the end: exp2(z - ref) = 0
  int re = 0;
  float rg = 1.f;
  if (SEG == 3 && tid < C::BM) re = p.eh[min(m0 + tid, count - 1)];    // (rows past the end repeat the last one)
  if (tid < C::BM && m0 + tid < count) {
    lab = p.lab[m0 + tid] - n0;
    if constexpr (GRAD) { rc = p.coef[m0 + tid]; rl = p.ref[m0 + tid]; rq = rc * p.inv[m0 + tid]; }
    if (GRAD && C::DT == DT_F16) rg = pow2(1.f, -p.g[m0 + tid]);
  }
  typename C::acc_t acc[C::TM][C::TN];
  float bj[C::TN];                                                 // the columns' bias
  int ej[C::TN];                                                   // and exponents
#pragma unroll
  for (int j = 0; j < C::TN; ++j) {
    const int col = n0 + col0 + j * 16;
    bj[j] = col < p.v1 ? (p.bias ? load_f(p.bias, col, p.bdt) : 0.f) : NEG_INF;
    ej[j] = SEG == 3 && col < p.v1 ? p.ew[col] : 0;
  }
  {
    Operand H = p.H;
    H.xlim = count;
    if constexpr (SEG == 3) product<C, false, TB, 3>(smem, H, p.W, m0, n0, p.D, 0, k_tiles<C, 3>(p.D), acc);
    else product<C, false, TB, 1>(smem, H, p.W, m0, n0, p.D, 0, k_tiles<C, 1>(p.D), acc, bj);
  }
  float* sf = reinterpret_cast<float*>(smem + score_over<C>(GRAD));
  int* slab = reinterpret_cast<int*>(sf);                          // label's column inside the tile, or none of them
  int* sE = slab + score_side<C>(GRAD);                            // exponents of the rows
  float* sG = sf + score_side<C>(GRAD) + (SEG == 3 ? C::BM : 0);   // 2^-g
  if (tid < C::BM) {
    if constexpr (SEG == 3) sE[tid] = re;
    if constexpr (GRAD && C::DT == DT_F16) sG[tid] = rg;
    slab[tid] = lab < C::BN && lab + n0 < p.v1 ? lab : -1;
    if constexpr (GRAD) { sf[C::BM + tid] = rc; sf[2 * C::BM + tid] = rl; sf[3 * C::BM + tid] = rq; }
  }
  __syncthreads();
  if constexpr (SEG == 3) {
#pragma unroll
    for (int i = 0; i < C::TM; ++i) {
      const i32x4 e = *reinterpret_cast<const i32x4*>(sE + row0 + i * 16);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int j = 0; j < C::TN; ++j) acc[i][j][q] = pow2(acc[i][j][q], -(e[q] + ej[j])) + bj[j];
    }
  }
  // a label's score is rare in a wave's part of the tile: whether there is one at all is asked once
  bool labelled = false;
  for (int r = lane; r < RW; r += 64) labelled |= (unsigned)(slab[wm * RW + r] - wn * CW) < (unsigned)CW;
  labelled = __any(labelled);
  if constexpr (!GRAD) {
    float* sM = sf + C::BM;                                        // [WN][BM] maximum (reference) and sum of a row in a wave's columns
    float* sS = sM + C::WN * C::BM;
    float* sZ = sS + C::WN * C::BM;
    float* sR = sZ + C::WN * C::BM;                                // [NW][4] references
    int* again = reinterpret_cast<int*>(sR + 4 * C::NW);
    float* sP = reinterpret_cast<float*>(smem);                    // [WN][16][BM + 16] partial sums
    float m = NEG_INF;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int j = 0; j < C::TN; ++j) m = fmaxf(fmaxf(fmaxf(m, acc[i][j][0]), fmaxf(acc[i][j][1], acc[i][j][2])), acc[i][j][3]);
    m = max16(m) * zscale;
    const float ref = m == NEG_INF ? 0.f : m;
    if (lc == 0) sR[wid * 4 + (lane >> 4)] = ref;
    if (tid == 0) *again = 0;
#pragma unroll
    for (int i = 0; i < C::TM; ++i) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] += exp2_(below<false>(acc[i][j][q], zscale, ref));   // (the reference passes over a NaN score, the sum keeps it)
      *reinterpret_cast<f32x4*>(sP + (wn * 16 + lc) * (C::BM + 16) + row0 + i * 16) = s;
    }
    __syncthreads();
    if (tid < C::BM && m0 + tid < count) {
      bool low = false;
#pragma unroll
      for (int w = 0; w < C::WN; ++w) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) s += sP[(w * 16 + k) * (C::BM + 16) + tid];
        const float r = sR[(tid / RW * C::WN + w) * 4 + ((tid >> 2) & 3)];
        sM[w * C::BM + tid] = r;
        sS[w * C::BM + tid] = s;
        low |= (s < 0x1p-64f && n0 + w * CW < p.v1) || fabsf(r) >= LARGE;
      }
      if (low) *again = 1;
    }
    __syncthreads();
    if (*again) {                                                  // a reference per row
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float mr = NEG_INF, s = 0.f;
#pragma unroll
          for (int j = 0; j < C::TN; ++j) mr = fmaxf(mr, acc[i][j][q]);
          mr = max16(mr) * zscale;
          const float rr = mr == NEG_INF ? 0.f : mr;
#pragma unroll
          for (int j = 0; j < C::TN; ++j) s += exp2_(below<true>(acc[i][j][q], zscale, rr));
          s = sum16(s);
          if (lc == 0) { sM[wn * C::BM + row0 + i * 16 + q] = mr; sS[wn * C::BM + row0 + i * 16 + q] = s; }
        }
    }
    if (labelled) {
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = row0 + i * 16 + q, at = slab[r] - col0;
#pragma unroll
          for (int j = 0; j < C::TN; ++j)
            if (at == j * 16) p.tz[m0 + r] = acc[i][j][q] * zscale;
        }
    }
    if (p.zs) {                                                    // label smoothing
      const float k = zscale * p.smooth_v;
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float zsum = 0.f;
#pragma unroll
          for (int j = 0; j < C::TN; ++j)
            if (n0 + col0 + j * 16 < p.v1) zsum += acc[i][j][q] * k;
          zsum = sum16(zsum);
          if (lc == 0) sZ[wn * C::BM + row0 + i * 16 + q] = zsum;
        }
    }
    __syncthreads();
    if (tid < C::BM && m0 + tid < count) {
      float mx = NEG_INF, s = 0.f, z = 0.f;
#pragma unroll
      for (int w = 0; w < C::WN; ++w) {
        join(mx, s, sM[w * C::BM + tid], sS[w * C::BM + tid]);
        if (p.zs) z += sZ[w * C::BM + tid];
      }
      p.part[(int64_t)nt * p.N + m0 + tid] = make_float2(mx, s);
      if (p.zs) p.zs[(int64_t)nt * p.N + m0 + tid] = z;
    }
    if (p.first) {
      // the scores of the teacher's entries: the tile passes through LDS, one row of waves at a time, and every row picks its own
      constexpr int P4 = C::BN + 4, TPR = C::NT / RW;
      float* sz = reinterpret_cast<float*>(smem);
      for (int half = 0; half < C::WM; ++half) {
        if (wm == half) {
#pragma unroll
          for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int j = 0; j < C::TN; ++j) sz[(row0 - wm * RW + i * 16 + q) * P4 + col0 + j * 16] = acc[i][j][q];
        }
        __syncthreads();
        const int r = tid / TPR, at = m0 + half * RW + r;
        if (at < count) {
          const int n = p.rows[at];
          const int64_t t = nt + p.v0 / C::BN;
          const int e1 = p.first[(t + 1) * p.N + n];
          for (int e = p.first[t * p.N + n] + tid % TPR; e < e1; e += TPR) {
            const int64_t o = (int64_t)n * p.K + e;
            p.zk[o] = sz[r * P4 + p.sidx[o] - n0];
          }
        }
        __syncthreads();
      }
    }
  } else {
    typedef Out<C::DT == DT_F32 ? OT_F32 : C::DT == DT_F16 ? OT_F16 : OT_BF16> O;
    typedef typename O::T OTy;
    typedef OTy Pack __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < C::TM; ++i) {
      const f32x4 c = *reinterpret_cast<const f32x4*>(sf + 3 * C::BM + row0 + i * 16), l = *reinterpret_cast<const f32x4*>(sf + 2 * C::BM + row0 + i * 16);
      auto probabilities = [&](auto round) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int j = 0; j < C::TN; ++j) acc[i][j][q] = c[q] * exp2_(below<decltype(round)::value>(acc[i][j][q], zscale, l[q]));
      };
      // (rows past the end have a reference of 3e38: either way a probability of 0)
      bool large = false;
#pragma unroll
      for (int q = 0; q < 4; ++q) large |= fabsf(l[q]) >= LARGE && l[q] < 3e38f;
      if (__any(large)) probabilities(Bool<true>()); else probabilities(Bool<false>());
    }
    if (p.smooth_v != 0.f) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        const float sv = n0 + col0 + j * 16 < p.v1 ? p.smooth_v : 0.f;
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][j][q] -= sf[C::BM + row0 + i * 16 + q] * sv;
      }
    }
    if (labelled) {
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = row0 + i * 16 + q, at = slab[r] - col0;
          const float ck = sf[C::BM + r] * p.keep;
#pragma unroll
          for (int j = 0; j < C::TN; ++j)
            if (at == j * 16) acc[i][j][q] -= ck;
        }
    }
    if (p.colsum) {                                                // a lane's rows, the four lane groups of a column, the wave rows
      float* sC = sf + 4 * C::BM;
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
          if constexpr (C::DT == DT_F16) {
            const f32x4 g = *reinterpret_cast<const f32x4*>(sG + row0 + i * 16);
            s += (acc[i][j][0] * g[0] + acc[i][j][1] * g[1]) + (acc[i][j][2] * g[2] + acc[i][j][3] * g[3]);
          } else s += (acc[i][j][0] + acc[i][j][1]) + (acc[i][j][2] + acc[i][j][3]);
        }
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (lane < 16) sC[wm * C::BN + col0 + j * 16] = s;
      }
    }
    char* out = p.G + (int64_t)(n0 - p.v0) * p.ldg + (int64_t)m0 * OSZ;
    // a gradient that outlives the caches anyway passes them by (4096 x 32000: step 1.07 -> 1.04 ms; 614 x 30522, where the products find it
    // there: 255 -> 264 us)
    const bool stream = (int64_t)count * (p.v1 - p.v0) > (32 << 20);
    constexpr int CPR = C::BM * OSZ / 16;
    // copy 0: the gradient; copy 1 (where words have factors): the hidden states' own, times 2^(lo - ew)
    const bool wide = SEG == 3 && p.sc->wide && (p.R || p.G2);
    const int lo = SEG == 3 ? lowest_word(p.sc) : 0;
#pragma unroll 1
    for (int copy = 0; copy < (SEG == 3 && wide ? 2 : 1); ++copy) {
      if (SEG == 3 && copy == 1) {
        __syncthreads();
        out = p.G2 ? p.G2 + (out - p.G) : nullptr;
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
          const float f = n0 + col0 + j * 16 < p.v1 ? pow2(1.f, lo - p.ew[n0 + col0 + j * 16]) : 0.f;
#pragma unroll
          for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][j][q] *= f;
        }
      }
#pragma unroll
      for (int half = 0; half < (SEG > 1 ? 2 : 1); ++half) {
        if (half == 1) __syncthreads();
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int j = 0; j < C::TN; ++j) {
            Pack v;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              v[q] = O::cv(acc[i][j][q]);
              if constexpr (SEG == 2) acc[i][j][q] -= O::fl(v[q]);
              else if (half == 1) v[q] = O::cv(acc[i][j][q] - O::fl(v[q]));   // (the accumulators are needed again)
            }
            *reinterpret_cast<Pack*>(smem + (col0 + j * 16) * PITCH + (row0 + i * 16) * OSZ) = v;
          }
        __syncthreads();
        if (p.first) {
          // the teacher's entries of this tile, from their exact scores: entries with one index write the same value
          if (tid < C::BM && m0 + tid < count) {
            const int n = p.rows[m0 + tid];
            const int64_t t = nt + p.v0 / C::BN;
            const int e1 = p.first[(t + 1) * p.N + n];
            for (int e = p.first[t * p.N + n]; e < e1; ++e) {
              const int64_t o = (int64_t)n * p.K + e;
              const float l = sf[2 * C::BM + tid], z = fabsf(l) >= LARGE ? below<true>(p.zk[o], zscale, l) : below<false>(p.zk[o], zscale, l);
              float g = sf[3 * C::BM + tid] * exp2_(z) - sf[C::BM + tid] * p.psum[o];
              if (SEG == 3 && copy == 1) g = pow2(g, lo - p.ew[p.sidx[o]]);
              if (half == 1) g -= O::fl(O::cv(g));
              *reinterpret_cast<OTy*>(smem + (p.sidx[o] - n0) * PITCH + tid * OSZ) = O::cv(g);
            }
          }
          __syncthreads();
        }
        if (out) {
          char* o = out + half * p.glo;
          const int rows_there = min(C::BN, p.v1 - n0) * CPR;
          if (stream) {
            for (int idx = tid; idx < rows_there; idx += C::NT) {
              const int v = idx / CPR, ch = idx - v * CPR;
              __builtin_nontemporal_store(*reinterpret_cast<const f32x4*>(smem + v * PITCH + ch * 16), reinterpret_cast<f32x4*>(o + v * p.ldg + ch * 16));
            }
          } else {
            for (int idx = tid; idx < rows_there; idx += C::NT) {
              const int v = idx / CPR, ch = idx - v * CPR;
              *reinterpret_cast<f32x4*>(o + v * p.ldg + ch * 16) = *reinterpret_cast<const f32x4*>(smem + v * PITCH + ch * 16);
            }
          }
        }
        if constexpr (is_pp<C>()) {
          if (p.R && (!wide || copy == 1)) {
            // rows again: transposing LDS reads give a lane 4 + 4 words of one position; a wave writes 16 positions x 32 words at a time
            char* orow = p.R + half * p.rlo + (int64_t)m0 * p.ldr + (int64_t)(n0 - p.v0) * OSZ;
            const int x = lane & 15, g4 = lane >> 4;
            const char* base = smem + (g4 * 8 + (x >> 2)) * PITCH + (x & 3) * 8;
#pragma unroll 4
            for (int b = wid; b < 128; b += 8) {
              const int v = (b & 7) * 32, m = (b >> 3) * 16;
              const char* a0 = base + v * PITCH + m * 2;
              typedef s16x4 __attribute__((address_space(3))) * lds_ptr_t;
              const s16x4 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr_t)(a0));
              const s16x4 t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr_t)(a0 + 4 * PITCH));
              s16x8 t;
              t[0] = t0[0]; t[1] = t0[1]; t[2] = t0[2]; t[3] = t0[3]; t[4] = t1[0]; t[5] = t1[1]; t[6] = t1[2]; t[7] = t1[3];
              *reinterpret_cast<s16x8*>(orow + (int64_t)(m + x) * p.ldr + (v + g4 * 8) * 2) = t;
            }
          }
        }
      }
    }
    if (p.colsum) {
      const float* sC = sf + 4 * C::BM;
      for (int v = tid; v < C::BN; v += C::NT) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < C::WM; ++w) s += sC[w * C::BN + v];
        if (n0 + v < p.v1) p.colsum[mt * p.ldc + n0 + v] = s;
      }
    }
  }
}

// Bound by latency: 8 bytes per row and column tile (4096 rows x 125 tiles 8 us, one row x 239 tiles 4 us).
// joins the (max, sum) pairs of a row's column tiles; R rows x 256 / R tile groups per workgroup
struct CombineP {
  const float2* part; const float* zs; const float* tz;
  const int* rows; const int* count;
  const int* lab;
  const float* ent; const float* sp; const float* zk; int K;    // distillation (ent != null)
  int N, ntiles;
  float keep, T, zscale;                                        // zscale: of the entries' scores zk
  float* ref; float* inv; float* loss;
};
template <int R>
__global__ void __launch_bounds__(256) combine_kernel(const CombineP p) {
  constexpr int GR = 256 / R;
  __shared__ float sm[GR][R], ss[GR][R], sz[GR][R];
  const int r = threadIdx.x % R, g = threadIdx.x / R;
  const int m = blockIdx.x * R + r, count = *p.count;
  if ((int)blockIdx.x * R >= count) return;
  float mx = NEG_INF, s = 0.f, z = 0.f;                          // z: smoothing term, or sum of p * score over the teacher's entries
  int n = 0;
  if (m < count) {
    n = p.rows[m];
#pragma unroll 4
    for (int t = g; t < p.ntiles; t += GR) {
      const float2 v = p.part[(int64_t)t * p.N + m];
      join(mx, s, v.x, v.y);
    }
    if (p.zs)
      for (int t = g; t < p.ntiles; t += GR) z += p.zs[(int64_t)t * p.N + m];
    if (p.ent)
      for (int k = g; k < p.K; k += GR) {
        const float w = p.sp[(int64_t)n * p.K + k];
        if (w > 0.f) z += w * (p.zk[(int64_t)n * p.K + k] * p.zscale);
      }
  }
  sm[g][r] = mx; ss[g][r] = s; sz[g][r] = z;
  for (int w = GR / 2; w > 0; w >>= 1) {
    __syncthreads();
    if (g < w) {
      join(mx, s, sm[g + w][r], ss[g + w][r]);
      z += sz[g + w][r];
      sm[g][r] = mx; ss[g][r] = s; sz[g][r] = z;
    }
  }
  if (g != 0 || m >= count) return;
  // The normaliser is kept as (reference, 1 / sum): as one number of the size of the scores its rounding would be the row's, some 2^-24 |lse|
  // of every probability at once.
  // The reference may lie up to 2^64 above the row: the sum's exponent goes to it (exactly, towards the row's own scores), the mantissa has the logarithm.
  float loss;
  const float top = mx + (float)__builtin_amdgcn_frexp_expf(s), ls = log2_(__builtin_amdgcn_frexp_mantf(s));
  if (p.ent) {
    const float h = p.ent[n];
    loss = p.T * p.T * (h + LN2 * ((top - z) + ls));
    if (h != h) mx = h;                                          // nothing sound to distil from: the row's gradient is NaN too
  } else {
    const bool in = p.lab[m] >= 0;
    loss = in ? LN2 * ((top - p.keep * p.tz[m] - z) + ls) : __builtin_nanf("");
    if (!in) mx = loss;                                          // a label outside the vocabulary: loss and gradient of the row are NaN
  }
  p.ref[m] = mx;
  p.inv[m] = 1.f / s;
  p.loss[n] = loss;
}

// ------------------------------------------------------------------------------------------------------------------------ backward
// Bound by the latency of one workgroup (4096 rows: 7 us).
// coef[m] = dloss[rows[m]] * T * s with the largest at `top` (0: s = 1). The scores' gradient is rounded to 16 bits: at a label it is close to
// its coefficient, and with the largest coefficient at a power of two the large ones sit at the end of their binade, where a rounding counts
// least.
// fp16 takes top = 2^14, and its smallest step, 2^-24, is what is left of a row whose coefficient is small. So a row has a power of two
// of its own, 2^g, which the sums over the words carry and give back: halves (slack 0) put every coefficient into [2^14, 2^15), fp16 operands,
// whose gradients keep 11 bits, only those below 2^-12 of the largest (raised to that). With one factor for all, a row weighted 10^-6 of the
// largest had its hidden states' gradient off by 2e-4 in fp32, one weighted 10^-7 by 5e-3 in fp16. For dW, which sums over the rows, t = g + eh is
// the whole exponent of a row, and the rows of H are brought to the lowest t. (A value of dW so holds 2^-40 of the largest |coefficient| |h| of a row.)
struct CoefP {
  const float* dloss; const int* rows; const int* count;
  float T, top;
  const int* eh;                         // exponents of operands in halves, or null
  float* coef; int *g, *t; int slack;    // g, t: or null (bf16, fp32)
  Grad* gr;
};
__device__ __forceinline__ int row_scale(const CoefP& p, float c) {
  const float x = fabsf(c);
  if (!p.g || !(x > 0.f && x < __builtin_inff())) return 0;
  int e;
  frexpf(x, &e);
  return min(max(15 - e - p.slack, 0), 126);
}
__device__ __forceinline__ int row_total(const CoefP& p, int m, float c, int g) {
  if (!p.t) return 0;
  const int e = p.eh ? p.eh[m] : 0;
  return c == 0.f || e == ZERO_ROW ? NO_ROW : g + e;
}
// Bound by the latency of one workgroup (4096 rows: 7 us).
__global__ void __launch_bounds__(1024) coef_kernel(const CoefP p) {
  __shared__ float red[16];
  const int c = *p.count;
  float s = 1.f, v[8];                                             // the first 8192 rows stay in registers
#pragma unroll
  for (int j = 0; j < 8; ++j) { const int m = j * 1024 + threadIdx.x; v[j] = m < c ? p.dloss[p.rows[m]] * p.T : 0.f; }
  if (p.top > 0.f) {
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (fabsf(v[j]) < __builtin_inff()) mx = fmaxf(mx, fabsf(v[j]));
    for (int m = 8192 + threadIdx.x; m < c; m += 1024) {
      const float x = fabsf(p.dloss[p.rows[m]] * p.T);
      if (x < __builtin_inff()) mx = fmaxf(mx, x);
    }
    mx = block_max(mx, red);
    if (mx > 0.f) s = fminf(p.top / mx, 1e37f);
  }
  int low = NO_ROW;
  auto row = [&](int m, float x) {
    const int g = row_scale(p, x * s);
    p.coef[m] = pow2(x * s, g);
    if (p.g) {
      const int t = row_total(p, m, x, g);
      p.g[m] = g;
      p.t[m] = t;
      low = min(low, t);
    }
  };
#pragma unroll
  for (int j = 0; j < 8; ++j) { const int m = j * 1024 + threadIdx.x; if (m < c) row(m, v[j]); }
  for (int m = 8192 + threadIdx.x; m < c; m += 1024) row(m, p.dloss[p.rows[m]] * p.T);
  if (p.g) low = -(int)block_max((float)-low, red);
  if (threadIdx.x == 0) *p.gr = Grad{1.f / s, p.g ? low : 0};
}

// coef_kernel and pack_kernel in one launch for few rows: a workgroup per row, each finds the largest coefficient and the lowest t for itself
__global__ void __launch_bounds__(256) prepare_kernel(const CoefP p, const PackP pk) {
  __shared__ float red[16];
  const int c = *p.count, m = blockIdx.x;
  if (m >= c && m > 0) return;
  float s = 1.f;
  if (p.top > 0.f) {
    float mx = 0.f;
    for (int k = threadIdx.x; k < c; k += 256) {
      const float v = fabsf(p.dloss[p.rows[k]] * p.T);
      if (v < __builtin_inff()) mx = fmaxf(mx, v);
    }
    mx = block_max(mx, red);
    if (mx > 0.f) s = fminf(p.top / mx, 1e37f);
  }
  int low = 0;
  if (p.g) {
    low = NO_ROW;
    for (int k = threadIdx.x; k < c; k += 256) {
      const float v = p.dloss[p.rows[k]] * p.T;
      low = min(low, row_total(p, k, v, row_scale(p, v * s)));
    }
    low = -(int)block_max((float)-low, red);
  }
  if (m == 0 && threadIdx.x == 0) *p.gr = Grad{1.f / s, low};
  if (m >= c) return;
  const float x = p.dloss[p.rows[m]] * p.T;
  const int g = row_scale(p, x * s), t = row_total(p, m, x, g);
  if (threadIdx.x == 0) {
    p.coef[m] = pow2(x * s, g);
    if (p.g) { p.g[m] = g; p.t[m] = t; }
  }
  if (pk.out) pack_row(pk, m, low - t);
}

// db from the gradient itself (both halves): with teacher entries the tiles' column sums do not hold them. Eight lanes to a word, 16 bytes each at a
// time. Bound by reading the gradient (96 rows x 30522 words in halves: 7.2 us; a wave to a word, two bytes a lane, took 10.4).
__global__ void __launch_bounds__(256) bias_rows_kernel(const char* __restrict__ G, int64_t ldg, int64_t glo, int dt, int vc, const int* __restrict__ count,
                                                        const int* __restrict__ g, const Grad* __restrict__ gr, void* __restrict__ db, int bdt) {
  const int v = blockIdx.x * 32 + (threadIdx.x >> 3), c = *count, ch = dt == DT_F32 ? 4 : 8;
  float s = 0.f;
  auto add = [&](const char* at, int m) {
    const f32x4 raw = *reinterpret_cast<const f32x4*>(at);
    if (dt == DT_F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s += m + e < c ? raw[e] : 0.f;
    } else {
      const s16x8 x = __builtin_bit_cast(s16x8, raw);
      i32x4 g0 = {0, 0, 0, 0}, g1 = {0, 0, 0, 0};
      if (dt == DT_F16) { g0 = *reinterpret_cast<const i32x4*>(g + m); g1 = *reinterpret_cast<const i32x4*>(g + m + 4); }   // (readable in 64s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t u = (uint16_t)x[e];
        s += m + e < c ? (dt == DT_BF16 ? bf2f(u) : pow2((float)__builtin_bit_cast(_Float16, u), -(e < 4 ? g0[e & 3] : g1[e & 3]))) : 0.f;
      }
    }
  };
  if (v < vc) {
    const char* row = G + v * ldg;
#pragma unroll 2
    for (int m = (threadIdx.x & 7) * ch; m < c; m += 8 * ch) {
      const char* at = row + (int64_t)m * (16 / ch);
      add(at, m);
      if (glo) add(at + glo, m);
    }
  }
  s += __shfl_xor(s, 4, 64);
  s += __shfl_xor(s, 2, 64);
  s += __shfl_xor(s, 1, 64);
  if (v < vc && (threadIdx.x & 7) == 0) store_f(db, v, bdt, s * gr->inv);
}

// dh: unit u of the grid owns output tile u % tiles and share u / tiles of the piece's columns; its fp32 tile lives in slab u and is added
// to by the following pieces. 8192 x 2048 of 65536 words in bf16 1.69 ms in four pieces (1300 TF/s; 1.54 in two), 4096 x 1024 of 32000 0.238 ms (1130 TF/s). Which unit owns what depends on the number of rows alone, so the sum's order is fixed.
//
// Large tile, W by rows ([V, D]): read as it is (K-major, transposing LDS reads), or transposed first where `many` rows pay for that.
struct DhP {
  Operand G, W, WT;
  const char* wide_g; const Scales* sc;  // operands in halves: the gradient's copy for words with factors (or null)
  int many;
  const int* count;
  int D, vc, units, most, accum;         // most: shares at most (each has some k-tiles to work on)
  float* slab;
};
__device__ __forceinline__ int shares_of(int tiles, int units, int most) { return tiles >= units ? 1 : min(most, units / tiles); }

// accumulators to (or onto) a tile of a slab
template <class C> __device__ __forceinline__ void to_slab(float* tile, typename C::acc_t (&acc)[C::TM][C::TN], bool add) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wm = wid / C::WN, wn = wid - wm * C::WN;
  float* out = tile + (wm * (C::BM / C::WM) + (lane >> 4) * 4) * C::BN + wn * (C::BN / C::WN) + (lane & 15);
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float* o = out + (i * 16 + q) * C::BN + j * 16;
        *o = add ? *o + acc[i][j][q] : acc[i][j][q];
      }
}

template <class C, bool TA, bool TB, int SEG>
__global__ void __launch_bounds__(C::NT) dh_kernel(const DhP p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int count = *p.count;
  const int mtiles = (count + C::BM - 1) / C::BM, ntiles = (p.D + C::BN - 1) / C::BN, tiles = mtiles * ntiles;
  if (tiles == 0) return;
  const int shares = shares_of(tiles, p.units, p.most);
  if ((int)blockIdx.x >= tiles * shares) return;
  const int u = xcd_remap(blockIdx.x, tiles * shares);
  const int share = u / tiles;
  int mt, nt;
  tile_coords(u - share * tiles, mtiles, ntiles, 8, mt, nt);
  const int ktiles = k_tiles<C, SEG>(p.vc), per = (ktiles + shares - 1) / shares;
  const int k0 = min(ktiles, share * per), k1 = min(ktiles, k0 + per);
  typename C::acc_t acc[C::TM][C::TN];
  Operand G = p.G;
  if (SEG == 3 && p.wide_g && p.sc->wide) G.p = p.wide_g;
  G.xlim = (count + 7) & ~7;                                       // (whole chunks; what lies behind is not read)
  if (is_pp<C>() && TB && count >= p.many) product<C, TA, false, SEG>(smem, G, p.WT, mt * C::BM, nt * C::BN, p.vc, k0, k1, acc);
  else product<C, TA, TB, SEG>(smem, G, p.W, mt * C::BM, nt * C::BN, p.vc, k0, k1, acc);
  to_slab<C>(p.slab + (int64_t)u * C::BM * C::BN, acc, p.accum);
}

// What is left, bound by memory (8192 x 2048: 100 MB, 26 us): workgroups [0, N * blocks) dh from the slabs, in the order of the shares
// (rows that take no part get zeros): 1024 columns of a row, or, where a call of few rows leaves many shares, 256 columns with a quarter of the shares
// to each wave (96 rows x 768 from 85 shares 12.9 and 8.0 us; 4096 x 1024 from 4 shares 20.6 and 24.7).
// Those behind them 256 words of db = scale * sum over the row tiles' column sums.
struct FinishP {
  const float* slab; const int* rows; const int* count;
  const Scales* sc; const int* g; const Grad* gr;   // sc: of operands in halves, or null; g: or null
  int N, D, units, most, blocks;         // blocks of a row
  void* dh; int dt;
  const float* colsum; int bm; int V;
  void* db; int bdt;
};
template <int BM, int BN, bool QUARTERS>
__global__ void __launch_bounds__(256) finish_kernel(const FinishP p) {
  __shared__ f32x4 quarter[QUARTERS ? 3 : 1][64];
  const int c = *p.count;
  if ((int)blockIdx.x >= p.N * p.blocks) {
    const int v = ((int)blockIdx.x - p.N * p.blocks) * 256 + threadIdx.x, tiles = (c + p.bm - 1) / p.bm;
    if (v >= p.V) return;
    float s = 0.f;
#pragma unroll 4
    for (int t = 0; t < tiles; ++t) s += p.colsum[(int64_t)t * p.V + v];
    store_f(p.db, v, p.bdt, s * p.gr->inv);
    return;
  }
  const int m = blockIdx.x / p.blocks, b = blockIdx.x - m * p.blocks;
  const int mtiles = (c + BM - 1) / BM, ntiles = (p.D + BN - 1) / BN, tiles = mtiles * ntiles;
  const int shares = m < c ? shares_of(tiles, p.units, p.most) : 1;
  const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int d = QUARTERS ? b * 256 + lane * 4 : b * 1024 + (int)threadIdx.x * 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (m < c && d < p.D) {
    const int mt = m / BM, nt = d / BN;
    const int g = mt / 8, rowsg = min(8, mtiles - g * 8);         // tile_coords with 8 row tiles to a group
    const int t = g * 8 * ntiles + nt * rowsg + (mt - g * 8);
    const float* x = p.slab + ((int64_t)t * BM + (m - mt * BM)) * BN + (d - nt * BN);
    const int per = QUARTERS ? (shares + 3) / 4 : shares, k0 = QUARTERS ? wid * per : 0, k1 = min(shares, k0 + per);
#pragma unroll 4
    for (int k = k0; k < k1; ++k) v += *reinterpret_cast<const f32x4*>(x + (int64_t)k * tiles * BM * BN);
  }
  if constexpr (QUARTERS) {
    if (wid > 0) quarter[wid - 1][lane] = v;
    __syncthreads();
    if (wid > 0) return;
    v = (v + quarter[0][lane]) + (quarter[1][lane] + quarter[2][lane]);
  }
  const int e = (p.sc ? lowest_word(p.sc) : 0) + (p.g && m < c ? p.g[m] : 0);
  const float inv = p.gr->inv;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = pow2(v[j], -e) * inv;
  const int64_t o = (int64_t)p.rows[m] * p.D + d;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (d + j < p.D) store_f(p.dh, o + j, p.dt, v[j]);
}

// dW[v0 .. v0 + vc) = scale * dz^T h (SWAP 0, [V, D]) or its transpose (SWAP 1, [D, V]): the gradient is read along its
// rows (the sum's axis; 8192 x 2048 of 65536 words in bf16 1.5 ms, 1470 TF/s); h is walked row by row by the 128 x 128 tiles, and read along the rows of its transpose by the 256 x 256 ones.
// shares > 1 (small outputs): the rows' range is cut, fp32 tiles go to a slab and dw_sum_kernel adds them in order.
struct DwP {
  Operand G, H;
  const int* count;
  const Grad* gr;
  void* out; int64_t ldo;
  int D, vc, shares;
  float* slab;
};
template <class C, int OT, bool SWAP, int SEG>
__global__ void __launch_bounds__(C::NT) dw_kernel(const DwP p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int K = *p.count;                                        // rows past it are not read
  const int M = SWAP ? p.D : p.vc, N = SWAP ? p.vc : p.D;
  const int mtiles = (M + C::BM - 1) / C::BM, ntiles = (N + C::BN - 1) / C::BN, tiles = mtiles * ntiles;
  const int u = xcd_remap(blockIdx.x, gridDim.x), share = u / tiles;
  int mt, nt;
  tile_coords(u - share * tiles, mtiles, ntiles, 8, mt, nt);
  const int m0 = mt * C::BM, n0 = nt * C::BN;
  const int ktiles = k_tiles<C, SEG>(K), per = (ktiles + p.shares - 1) / p.shares;
  const int k0 = min(ktiles, share * per), k1 = min(ktiles, k0 + per);
  typename C::acc_t acc[C::TM][C::TN];
  product<C, SWAP && !is_pp<C>(), !SWAP && !is_pp<C>(), SEG>(smem, SWAP ? p.H : p.G, SWAP ? p.G : p.H, m0, n0, K, k0, k1, acc);
  if (p.shares > 1) { to_slab<C>(p.slab + (int64_t)u * C::BM * C::BN, acc, false); return; }
  if constexpr (C::DT == DT_F16) {                                 // the rows' factor
    const int e = -p.gr->hlo;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][j][q] = pow2(acc[i][j][q], e);
  }
  if constexpr (is_pp<C>() && OT == OT_F32) {                      // an fp32 tile is more than LDS: stores of 16 columns from the accumulators
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, wm = wid / C::WN, wn = wid - wm * C::WN;
    const int r0 = m0 + wm * (C::BM / C::WM) + (lane >> 4) * 4, c0 = n0 + wn * (C::BN / C::WN) + (lane & 15);
    const float s = p.gr->inv;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
          if (r0 + i * 16 + q < M && c0 + j * 16 < N) reinterpret_cast<float*>(p.out)[(r0 + i * 16 + q) * p.ldo + c0 + j * 16] = acc[i][j][q] * s;
    return;
  }
  EpiP e;
  e.out = p.out; e.residual = nullptr; e.bias = nullptr; e.stats = nullptr; e.stat_shift = nullptr;
  e.alpha = p.gr->inv; e.act = ACT_KEEP; e.accum = 0;
  const int64_t ldo = p.ldo;
  epilogue_impl<C, OT, ACT_KEEP, 0>(smem, acc, mt, n0, N, M - m0, e, [=](int r) -> int64_t {
    return m0 + r < M ? (int64_t)(m0 + r) * ldo + n0 : (int64_t)-1;
  });
}
template <int BM, int BN>
__global__ void __launch_bounds__(256) dw_sum_kernel(const float* __restrict__ slab, int shares, int M, int N, const Grad* __restrict__ gr,
                                                     void* __restrict__ out, int64_t ldo, int dt) {
  const int mtiles = (M + BM - 1) / BM, ntiles = (N + BN - 1) / BN, tiles = mtiles * ntiles;
  const int m = blockIdx.x, mt = m / BM, g = mt / 8, rowsg = min(8, mtiles - g * 8);
  for (int n = threadIdx.x; n < N; n += 256) {
    const int nt = n / BN, t = g * 8 * ntiles + nt * rowsg + (mt - g * 8);
    const float* x = slab + ((int64_t)t * BM + (m - mt * BM)) * BN + (n - nt * BN);
    float v = 0.f;
#pragma unroll 4
    for (int k = 0; k < shares; ++k) v += x[(int64_t)k * tiles * BM * BN];
    store_f(out, (int64_t)m * ldo + n, dt, pow2(v, -gr->hlo) * gr->inv);
  }
}

// ------------------------------------------------------------------------------------------------------------------------ host side
template <int DT> using Big = Cfg<256, 256, 2, 4, 2, 16, DT>;
template <int DT> using Mid = Cfg<128, 128, 2, 4, 2, 16, DT>;   // eight waves: step of 32 rows x 1024, 50000 words 138 us with four, 132 with eight
template <int DT> using Few = Cfg<32, 128, 1, 4, 4, 16, DT>;
template <int DT> using Small = Cfg<64, 64, 2, 2, 4, 16, DT>;
enum { TILE_BIG = 0, TILE_MID = 1, TILE_FEW = 2, TILE_SMALL = 3 };
int tile_rows(int tile) { return tile == TILE_BIG ? 256 : tile == TILE_FEW ? 32 : tile == TILE_SMALL ? 64 : 128; }
int tile_cols(int tile) { return tile == TILE_BIG ? 256 : tile == TILE_SMALL ? 64 : 128; }

// One call: sizes, layout and pointers (ops/vocab_loss.py _ARGS lists the same fields in the same order)
struct Args {
  int64_t N, D, V, dt, split, wt, bdt, ldh, ldw, lab64, ignore, idx64, tdt, K, want_h, want_w, want_b;
  int64_t pad_h, pad_w;                  // operands that are copied to whole 16-byte chunks (H: packed) by the forward call: set by layout()
  const void *H, *W, *bias, *labels, *idx, *t;
  float* loss; char* state; char* ws;
  const float* dloss; void *dh, *dw, *db;
};

int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Plan {
  int tile, dh_tile, dw_tile;            // TILE_*
  int op;                                // operand type of the products
  bool pad_w, pad_h;
  bool pair;                             // 16-bit operands: the scores' gradient in two halves
  int copies;                            // of the scores' gradient: two halves, two layouts, or one copy for each product that reads it
  bool nt;                               // backward products on 256 x 256 tiles from operands laid out along the sum's axis
  bool wtr; int many;                    // dh: W is transposed first, for calls of `many` rows that take part
  int bm, bn, tiles;                     // tiles of the scores
  int64_t np, dp, wcp, wrows, vp;           // padded rows / columns of the packed H and of the halves of W
  int pieces, step;
  int units, most, shares;
  bool quarters;                         // finish_kernel
  bool pack;                             // dW: the rows of H that take part are packed first (fp16, halves: brought to one factor)
  int64_t gcols;
};

// What the operands' addresses decide. The forward call's decision, since the backward call may get the same values at another place.
void layout(Args& a) {
  const int64_t ch = a.dt == DT_F32 ? 4 : 8, wc = a.wt ? a.V : a.D;
  a.pad_w = !a.split && (wc % ch || a.ldw % ch || !aligned16(a.W));
  a.pad_h = !a.split && (a.D % ch || a.ldh % ch || !aligned16(a.H));
}

Plan plan(const Args& a) {
  Plan p;
  p.op = a.split ? DT_F16 : (int)a.dt;
  const bool bits16 = p.op != DT_F32;
  const int64_t big_tiles = up(a.N, 256) / 256 * (up(a.V, 256) / 256);
  // (its operands are addressed with 32-bit offsets: rows of all of them, and H's indirect ones together, have to be short of that)
  const bool near = up(a.N, 256) * 2 < BUF_LD && up(a.V, 256) * 2 < BUF_LD && a.ldh * 4 < BUF_LD && a.ldw * 4 < BUF_LD && up(a.D, 8) * 4 < BUF_LD && (a.split || a.N * a.ldh * 2 < BUF_SPAN);
  const int64_t mid_tiles = up(a.N, 128) / 128 * (up(a.V, 128) / 128);
  // Tile of the scores (times of calls with D = 1024 in bf16, 128 x 128 against the other):
  //   256 x 256 once such tiles cover two thirds of the 256 CUs: forward of 300 rows x 22500 words (176 tiles) 41.8 and 39.2 us, x 16000 (126) 30.5
  //   and 37.3; step of 1000 x 11300 159 and 151 us; not for half a tile of rows: 100 x 50000 30.1 and 36.3
  //   32 x 128, four stages, where few rows meet a large vocabulary and W streams through: 1 x 768 of 30522 words 22.2 and 18.4 us, fp32 32 x 50000
  //   150 and 67 (64 x 64: 18.6 and 96)
  //   64 x 64, four stages, where 128 x 128 ones leave CUs idle and the time is one chain of k-tiles: 300 x 5000 (120 tiles) 22.5 and 19.0 us, x 7000
  //   (165) 22.6 and 26.8; fp32, whose chains are longer: 300 x 300 of 12000 (282) 59.3 and 44.3, of 20000 (471) 51.7 and 67.0
  p.tile = bits16 && big_tiles >= 176 && a.N > 128 && near ? TILE_BIG : a.N <= 32 && a.V >= 16384 ? TILE_FEW : mid_tiles < (bits16 ? 144 : 384) ? TILE_SMALL : TILE_MID;
  if (a.split && p.tile == TILE_FEW) p.tile = TILE_MID;
  if (!bits16 && p.tile == TILE_BIG) p.tile = TILE_MID;
  p.bm = tile_rows(p.tile);
  p.bn = tile_cols(p.tile);
  p.tiles = (int)(up(a.V, p.bn) / p.bn);
  p.np = up(a.N, 256);
  p.vp = up(a.V, 64);
  p.dp = up(a.D, 8);
  p.wrows = a.wt ? a.D : a.V;
  p.pad_w = a.pad_w;
  p.pad_h = a.pad_h;
  p.wcp = up(a.wt ? a.V : a.D, 8);
  const int64_t esz = a.dt == DT_F32 ? 4 : 2;                    // halves take as much as fp32
  // The backward products on 256 x 256 tiles, for which the scores' gradient is written a second time, row by row, and H transposed; against
  // 128 x 128 tiles without that: step of 600 rows x 4096 of 40000 words 841 against 939 us, x 1024 277 and 285, 4096 x 512 of 32000 634 and 683,
  // 2048 x 256 271 and 244, 400 x 1024 of 40000 243 and 240.
  p.nt = p.tile == TILE_BIG && a.N >= 512 && a.D >= 512;
  p.pair = bits16 && !a.split && a.N <= 256;                       // (see score_kernel)
  // A piece's gradient with all its copies: 640 MiB. Step of 8192 x 2048 of 65536 words, two copies: 6.95 ms with 256 MiB, 6.82 with 512, 6.76 with 1024
  // (its 16-bit logits: 1024 MiB); 3001 x 1000 of 50001: 0.99 ms in one piece of 588 MiB, 1.09 in two.
  p.copies = p.nt || p.pair || (a.split && a.want_h) ? 2 : 1;
  const int64_t most = ((int64_t)640 << 20) / (p.np * esz * p.copies) / 256 * 256;
  p.pieces = (int)(most >= 256 ? (a.V + most - 1) / most : up(a.V, 256) / 256);
  p.step = (int)up((a.V + p.pieces - 1) / p.pieces, 256);
  p.pieces = (int)((a.V + p.step - 1) / p.step);
  p.gcols = up(a.V < p.step ? a.V : p.step, 256);
  // W as it lies, through transposing LDS reads, against W transposed first: 2100 rows x 1000 of 50001 words 231 us against 207 + 98; 4096 x 1024 of
  // 32000: 242 and 226 + 47; 8192 x 2048 of 65536: 1820 and 1520 + 188. The transpose costs the same for any number of rows.
  p.many = 6144;
  p.wtr = a.want_h && p.nt && !a.wt && a.N >= p.many;
  p.pack = a.want_w && !p.nt && (!p.pad_h || p.op == DT_F16);
  const int seg = a.split ? 3 : p.pair ? 2 : 1, bk = bits16 ? 64 : 32;
  const int64_t vk = seg * (up(p.step, bk) / bk), nk = seg * (up(a.N, bk) / bk);   // k-tiles of the two products' sums
  const int64_t cols = p.gcols < a.V ? p.gcols : a.V;
  auto tiles = [](int64_t m, int64_t n, int t) { return up(m, t) / t * (up(n, t) / t); };
  // 64 x 64 tiles in the backward products by the same reasoning; their sums can be cut into shares of four k-tiles. Step of 700 rows x 304 of
  // 400 words: dh 40.8 (128 x 128) and 38.6 us, dw 41.6 and 38.5; 30 x 2048 of 10000, dw: 81 and 95.
  p.dh_tile = p.nt ? TILE_BIG : tiles(a.N, a.D, 128) * (vk / 4 + 1) < 256 ? TILE_SMALL : TILE_MID;
  p.dw_tile = p.nt ? TILE_BIG : tiles(cols, a.D, 128) * (nk / 4 + 1) < 256 ? TILE_SMALL : TILE_MID;
  const int want_h = p.dh_tile == TILE_BIG ? 256 : p.dh_tile == TILE_SMALL ? 1024 : 512, want_w = p.dw_tile == TILE_SMALL ? 1024 : 512;
  const int64_t ht = tiles(a.N, a.D, tile_rows(p.dh_tile)), wt = tiles(cols, a.D, tile_rows(p.dw_tile));
  p.units = (int)(ht > want_h ? ht : want_h);
  p.most = (int)((vk + 3) / 4);
  p.quarters = (ht >= p.units ? 1 : p.units / ht < p.most ? p.units / ht : p.most) >= 16;
  int64_t sh = p.dw_tile == TILE_BIG ? 1 : want_w / wt;
  if (sh > nk / 4) sh = nk / 4;
  p.shares = (int)(sh < 1 ? 1 : sh);
  return p;
}

// buffers carved from one allocation each: state (kept from forward to backward), forward and backward workspace
struct Carve {
  char* base; int64_t at = 0;
  explicit Carve(char* b) : base(b) {}
  template <typename T> T* take(int64_t n) {
    T* r = reinterpret_cast<T*>(base + at);
    at += up(n * (int64_t)sizeof(T), 256);
    return r;
  }
};
struct State {
  Scales* sc; int *count, *rows, *lab; float *ref, *inv; int *eh, *ew;
  int* sidx; float *sp, *psum, *zk, *ent, *mass; unsigned short* first;
  char *wo, *ho;
  int64_t bytes;
  State(const Args& a, const Plan& p) {
    Carve c(a.state);
    sc = c.take<Scales>(1); count = c.take<int>(1); rows = c.take<int>(a.N); lab = c.take<int>(a.N); ref = c.take<float>(a.N); inv = c.take<float>(a.N);
    const int64_t nk = a.K ? a.N * a.K : 0;
    sidx = c.take<int>(nk); sp = c.take<float>(nk); psum = c.take<float>(nk); zk = c.take<float>(nk);
    ent = c.take<float>(a.K ? a.N : 0); mass = c.take<float>(a.K ? a.N : 0);
    first = c.take<unsigned short>(a.K ? (int64_t)(p.tiles + 1) * a.N : 0);
    const int64_t esz = a.dt == DT_F32 ? 4 : 2;                    // (two halves take as much as an fp32 value)
    eh = c.take<int>(a.split ? a.N : 0); ew = c.take<int>(a.split ? a.V : 0);
    wo = c.take<char>(a.split || p.pad_w ? p.wrows * p.wcp * esz : 0);
    ho = c.take<char>(a.split || p.pad_h ? p.np * p.dp * esz : 0);
    bytes = c.at;
  }
};
struct Work {
  float2* part; float *tz, *zs, *wmax, *tops;                         // forward
  Grad* gr; int *g, *t; float *coef, *colsum; char* G; char* packed; uint16_t *ht, *wtr; float *dh_slab, *dw_slab;  // backward
  int64_t fwd, bwd;
  Work(const Args& a, const Plan& p) {
    Carve c(a.ws);
    part = c.take<float2>((int64_t)p.tiles * a.N); tz = c.take<float>(a.N); zs = c.take<float>((int64_t)p.tiles * a.N);
    wmax = c.take<float>(a.split ? up(a.V, 4) * (a.wt ? CUTS : 1) : 0);
    tops = c.take<float>(a.split ? TOPS : 0);
    fwd = c.at;
    c.at = 0;
    const int64_t esz = a.dt == DT_F32 ? 4 : 2;
    gr = c.take<Grad>(1); g = c.take<int>(p.op == DT_F16 ? a.N : 0); t = c.take<int>(p.op == DT_F16 ? a.N : 0); coef = c.take<float>(a.N); G = c.take<char>(p.np * p.gcols * esz * p.copies);
    colsum = c.take<float>(a.want_b && !a.K ? (a.N + p.bm - 1) / p.bm * a.V : 0);
    packed = c.take<char>(p.pack ? a.N * p.dp * esz : 0);
    ht = c.take<uint16_t>(a.want_w && p.nt ? a.D * p.np * (a.split ? 2 : 1) : 0);
    wtr = c.take<uint16_t>(p.wtr ? a.D * p.vp * (a.split ? 2 : 1) : 0);
    const int64_t ht = tile_rows(p.dh_tile), wt = tile_rows(p.dw_tile), cols = p.gcols < a.V ? p.gcols : a.V;
    dh_slab = c.take<float>(a.want_h ? p.units * ht * ht : 0);
    dw_slab = c.take<float>(a.want_w && p.shares > 1 ? up(cols, wt) * up(a.D, wt) * p.shares : 0);
    bwd = c.at;
  }
};

#define VL_CHECK() do { const int e_ = (int)hipGetLastError(); if (e_) return e_; } while (0)

template <class C, bool TB, bool GRAD, int SEG> int launch_score(const ScoreP& p, hipStream_t st) {
  const int64_t grid = (int64_t)((p.N + C::BM - 1) / C::BM) * ((p.v1 - p.v0 + C::BN - 1) / C::BN);
  if (grid > 0x7fffffff) return -2;
  constexpr int LDS = score_lds<C>(GRAD, SEG);
  static_assert(LDS <= 160 * 1024, "tile does not fit the 160 KiB LDS");
  static DeviceOnceLds once;
  once.ensure(reinterpret_cast<const void*>(&score_kernel<C, TB, GRAD, SEG>), LDS);
  hipLaunchKernelGGL((score_kernel<C, TB, GRAD, SEG>), dim3((unsigned)grid), dim3(C::NT), LDS, st, p);
  return (int)hipGetLastError();
}
template <int DT, bool TB, bool GRAD, int SEG> int score_tile(const ScoreP& p, int tile, hipStream_t st) {
  if (tile == TILE_FEW) return launch_score<Few<DT>, TB, GRAD, SEG>(p, st);
  return tile == TILE_SMALL ? launch_score<Small<DT>, TB, GRAD, SEG>(p, st) : launch_score<Mid<DT>, TB, GRAD, SEG>(p, st);
}
template <int DT, bool TB, bool GRAD> int score16(const ScoreP& p, int tile, bool pair, hipStream_t st) {
  if constexpr (GRAD)
    if (pair) return tile == TILE_BIG ? launch_score<Big<DT>, TB, GRAD, 2>(p, st) : score_tile<DT, TB, GRAD, 2>(p, tile, st);
  if (tile == TILE_BIG) return launch_score<Big<DT>, TB, GRAD, 1>(p, st);
  if (GRAD || tile != TILE_FEW) return tile == TILE_SMALL ? launch_score<Small<DT>, TB, GRAD, 1>(p, st) : launch_score<Mid<DT>, TB, GRAD, 1>(p, st);
  return launch_score<Few<DT>, TB, false, 1>(p, st);
}
template <bool TB, bool GRAD> int dispatch_score(const ScoreP& p, int tile, int op, bool split, bool pair, hipStream_t st) {
  if (split)
    return tile == TILE_BIG ? launch_score<Big<DT_F16>, TB, GRAD, 3>(p, st) : tile == TILE_SMALL ? launch_score<Small<DT_F16>, TB, GRAD, 3>(p, st)
                            : launch_score<Mid<DT_F16>, TB, GRAD, 3>(p, st);
  if (op == DT_F32) return score_tile<DT_F32, TB, GRAD, 1>(p, tile, st);
  return op == DT_BF16 ? score16<DT_BF16, TB, GRAD>(p, tile, pair, st) : score16<DT_F16, TB, GRAD>(p, tile, pair, st);
}
template <bool GRAD> int scores(const ScoreP& p, int tile, int op, bool split, bool pair, bool tb, hipStream_t st) {
  return tb ? dispatch_score<true, GRAD>(p, tile, op, split, pair, st) : dispatch_score<false, GRAD>(p, tile, op, split, pair, st);
}

template <class C, bool TA, bool TB, int SEG> int launch_dh(const DhP& p, hipStream_t st) {
  constexpr int LDS = C::STAGES * C::STAGE_BYTES;
  static DeviceOnceLds once;
  once.ensure(reinterpret_cast<const void*>(&dh_kernel<C, TA, TB, SEG>), LDS);
  hipLaunchKernelGGL((dh_kernel<C, TA, TB, SEG>), dim3(p.units), dim3(C::NT), LDS, st, p);
  return (int)hipGetLastError();
}
// 256 x 256: the gradient K-contiguous (p.nt); smaller tiles: the gradient and the [V, D] table are walked row by row
template <int DT, int SEG> int rows_dh(const DhP& p, int tile, bool wt, hipStream_t st) {
  if (tile == TILE_SMALL) return wt ? launch_dh<Small<DT>, true, false, SEG>(p, st) : launch_dh<Small<DT>, true, true, SEG>(p, st);
  return wt ? launch_dh<Mid<DT>, true, false, SEG>(p, st) : launch_dh<Mid<DT>, true, true, SEG>(p, st);
}
template <bool TB> int big_dh(const DhP& p, int op, bool split, hipStream_t st) {
  return split ? launch_dh<Big<DT_F16>, false, TB, 3>(p, st) : op == DT_BF16 ? launch_dh<Big<DT_BF16>, false, TB, 1>(p, st) : launch_dh<Big<DT_F16>, false, TB, 1>(p, st);
}
int dispatch_dh(const DhP& p, int tile, int op, bool split, bool pair, bool wt, hipStream_t st) {
  if (tile == TILE_BIG) return wt ? big_dh<false>(p, op, split, st) : big_dh<true>(p, op, split, st);
  if (split) return rows_dh<DT_F16, 3>(p, tile, wt, st);
  if (op == DT_F32) return rows_dh<DT_F32, 1>(p, tile, wt, st);
  if (op == DT_BF16) return pair ? rows_dh<DT_BF16, 2>(p, tile, wt, st) : rows_dh<DT_BF16, 1>(p, tile, wt, st);
  return pair ? rows_dh<DT_F16, 2>(p, tile, wt, st) : rows_dh<DT_F16, 1>(p, tile, wt, st);
}

template <class C, int OT, bool SWAP, int SEG> int launch_dw(const DwP& p, hipStream_t st) {
  const int M = SWAP ? p.D : p.vc, N = SWAP ? p.vc : p.D;
  const int tiles = ((M + C::BM - 1) / C::BM) * ((N + C::BN - 1) / C::BN);
  constexpr int LDS = is_pp<C>() && OT == OT_F32 ? C::STAGES * C::STAGE_BYTES : C::lds_bytes(Out<OT>::SZ);
  static_assert(LDS <= 160 * 1024, "tile does not fit the 160 KiB LDS");
  static DeviceOnceLds once;
  once.ensure(reinterpret_cast<const void*>(&dw_kernel<C, OT, SWAP, SEG>), LDS);
  hipLaunchKernelGGL((dw_kernel<C, OT, SWAP, SEG>), dim3(tiles * p.shares), dim3(C::NT), LDS, st, p);
  VL_CHECK();
  if (p.shares > 1)
    hipLaunchKernelGGL((dw_sum_kernel<C::BM, C::BN>), dim3(M), dim3(256), 0, st, p.slab, p.shares, M, N, p.gr, p.out, p.ldo,
                       OT == OT_F32 ? (int)DT_F32 : OT == OT_F16 ? (int)DT_F16 : (int)DT_BF16);
  return (int)hipGetLastError();
}
template <int DT, int OT, bool SWAP, int SEG> int rows_dw(const DwP& p, int tile, hipStream_t st) {
  return tile == TILE_SMALL ? launch_dw<Small<DT>, OT, SWAP, SEG>(p, st) : launch_dw<Mid<DT>, OT, SWAP, SEG>(p, st);
}
template <bool SWAP> int dispatch_dw(const DwP& p, int tile, int op, bool split, bool pair, hipStream_t st) {
  const bool big = tile == TILE_BIG;
  if (split) return big ? launch_dw<Big<DT_F16>, OT_F32, SWAP, 3>(p, st) : rows_dw<DT_F16, OT_F32, SWAP, 3>(p, tile, st);
  if (op == DT_F32) return rows_dw<DT_F32, OT_F32, SWAP, 1>(p, tile, st);
  if (op == DT_BF16)
    return big ? launch_dw<Big<DT_BF16>, OT_BF16, SWAP, 1>(p, st) : pair ? rows_dw<DT_BF16, OT_BF16, SWAP, 2>(p, tile, st) : rows_dw<DT_BF16, OT_BF16, SWAP, 1>(p, tile, st);
  return big ? launch_dw<Big<DT_F16>, OT_F16, SWAP, 1>(p, st) : pair ? rows_dw<DT_F16, OT_F16, SWAP, 2>(p, tile, st) : rows_dw<DT_F16, OT_F16, SWAP, 1>(p, tile, st);
}

// 0 where the arguments are what the kernels assume
int check(const Args& a, bool bwd) {
  if (a.N <= 0 || a.N > 0x7fffffff - 512 || a.D <= 0 || a.D > 0x7fffffff - 512 || a.V <= 0 || a.V > 0x7fffffff - 512) return -2;
  if (a.dt < 0 || a.dt > 2 || a.bdt < 0 || a.bdt > 2 || (a.split && a.dt != DT_F32) || a.K < 0 || a.K > KMAX) return -2;
  if (!a.H || !a.W || !a.state || !a.ws || !aligned16(a.state) || !aligned16(a.ws)) return -2;
  if (!bwd && (!a.loss || (a.K ? !a.idx || !a.t || a.tdt < 0 || a.tdt > 2 : !a.labels))) return -2;
  if (a.ldh < a.D || a.ldw < (a.wt ? a.V : a.D)) return -2;
  Args now = a;
  layout(now);
  if ((now.pad_w && !a.pad_w) || (now.pad_h && !a.pad_h)) return -2;
  if (bwd && (!a.dloss || (a.want_h && !a.dh) || (a.want_w && !a.dw) || (a.want_b && (!a.db || !a.bias)))) return -2;
  return 0;
}

void operands(const Args& a, const Plan& p, const State& s, Operand& H, Operand& W) {
  const int esz = a.dt == DT_F32 ? 4 : 2;
  if (a.split) {
    H = Operand{(const char*)s.ho, p.dp * 2, p.np * p.dp * 2, 0, nullptr};
    W = Operand{(const char*)s.wo, p.wcp * 2, p.wrows * p.wcp * 2, 0, nullptr};
  } else {
    H = p.pad_h ? Operand{s.ho, p.dp * esz, 0, 0, nullptr} : Operand{(const char*)a.H, a.ldh * esz, 0, 0, s.rows};
    W = p.pad_w ? Operand{s.wo, p.wcp * esz, 0, 0, nullptr} : Operand{(const char*)a.W, a.ldw * esz, 0, 0, nullptr};
  }
}

ScoreP score_args(const Args& a, const State& s, const float* f) {
  ScoreP q = {};
  q.bias = a.bias; q.bdt = (int)a.bdt; q.rows = s.rows; q.count = s.count; q.sc = s.sc; q.eh = s.eh; q.ew = s.ew;
  q.lab = s.lab;
  q.N = (int)a.N; q.D = (int)a.D;
  q.invT = 1.f / f[0]; q.smooth_v = f[1] / (float)a.V; q.keep = 1.f - f[1];
  if (a.K) { q.first = s.first; q.sidx = s.sidx; q.psum = s.psum; q.zk = s.zk; q.K = (int)a.K; q.keep = 0.f; q.smooth_v = 0.f; }
  return q;
}

int forward(const Args& a, const float* f, hipStream_t st) {
  if (const int e = check(a, false)) return e;
  if (!(f[0] > 0.f)) return -2;
  const Plan p = plan(a);
  const State s(a, p);
  const Work w(a, p);
  if (a.K) {
    int p2 = 2;
    while (p2 < a.K) p2 <<= 1;
    TeacherP t{a.idx, (int)a.idx64, a.t, (int)a.tdt, (int)a.N, (int)a.V, (int)a.K, p2, 1.f / f[0], p.bn, p.tiles, s.sidx, s.sp, s.psum, s.first, s.ent, s.mass};
    hipLaunchKernelGGL(teacher_kernel, dim3((unsigned)((a.N + 3) / 4)), dim3(256), 4 * 12 * p2, st, t);
    VL_CHECK();
  }
  hipLaunchKernelGGL(rows_kernel, dim3(1), dim3(1024), 0, st, a.K ? nullptr : a.labels, (int)a.lab64, a.ignore, s.mass, (int)a.N, (int)a.V, s.rows, s.lab, s.count, s.sc, a.loss);
  VL_CHECK();
  if (a.split) {
    // [D, V]: as many cuts of the rows as fill the chip once for the largest values (2368 x 20592: 58 us with 25 cuts, 68 with 16), fewer for the
    // conversion (84 us with 25, 75 with 16)
    const int64_t strips = up(a.V, 256) / 256, fit = strips < 2048 ? 2048 / strips : 1, most = a.D < 64 ? 1 : CUTS;
    const int cuts = (int)(fit < most ? fit : most);
    auto groups = [&](int n) { return (int)(strips * n < TOPS ? strips * n : TOPS); };
    SplitP q{(const float*)a.W, a.ldw, (int)a.wt, (int)a.V, (int)a.D, (_Float16*)s.wo, p.wcp, (const float*)a.H, a.ldh, (_Float16*)s.ho, p.dp, p.np,
             s.rows, s.count, s.sc, s.eh, s.ew, w.wmax, cuts, cuts, w.tops, a.wt ? groups(cuts) : 1024, 0};
    hipLaunchKernelGGL(amax_kernel, dim3(q.gw + 256), dim3(256), 0, st, q);
    VL_CHECK();
    q.tw = q.gw;
    q.chunks = cuts < 16 ? cuts : 16;
    q.gw = a.wt ? groups(q.chunks) : 2048;
    hipLaunchKernelGGL(split_kernel, dim3(q.gw + 256), dim3(256), 0, st, q);
    VL_CHECK();
  }
  if (p.pad_w || p.pad_h) {
    const PadP q{(const char*)a.W, a.ldw, (int)p.wrows, (int)(a.wt ? a.V : a.D), s.wo, p.wcp, (const char*)a.H, a.ldh, (int)a.D, s.ho, p.dp, s.rows, s.count,
                 p.pad_w ? 1024 : 0};
    const dim3 grid(q.gw + (p.pad_h ? 256 : 0));
    if (a.dt == DT_F32) hipLaunchKernelGGL((pad_kernel<4>), grid, dim3(256), 0, st, q);
    else hipLaunchKernelGGL((pad_kernel<2>), grid, dim3(256), 0, st, q);
    VL_CHECK();
  }
  ScoreP q = score_args(a, s, f);
  operands(a, p, s, q.H, q.W);
  q.W.xlim = (int)a.V;
  q.v0 = 0; q.v1 = (int)a.V;
  q.part = w.part; q.tz = w.tz; q.zs = q.smooth_v != 0.f ? w.zs : nullptr;
  if (const int e = scores<false>(q, p.tile, p.op, a.split, false, a.wt, st)) return e;
  CombineP c{w.part, q.zs, w.tz, s.rows, s.count, s.lab, a.K ? s.ent : nullptr, s.sp, s.zk, (int)a.K, (int)a.N, p.tiles, q.keep, f[0],
             q.invT * LOG2E, s.ref, s.inv, a.loss};
  if (a.N <= 256) hipLaunchKernelGGL((combine_kernel<1>), dim3((unsigned)a.N), dim3(256), 0, st, c);
  else hipLaunchKernelGGL((combine_kernel<8>), dim3((unsigned)((a.N + 7) / 8)), dim3(256), 0, st, c);
  return (int)hipGetLastError();
}

template <int B> void launch_finish(const FinishP& q, bool quarters, dim3 grid, hipStream_t st) {
  if (quarters) hipLaunchKernelGGL((finish_kernel<B, B, true>), grid, dim3(256), 0, st, q);
  else hipLaunchKernelGGL((finish_kernel<B, B, false>), grid, dim3(256), 0, st, q);
}

int backward(const Args& a, const float* f, hipStream_t st) {
  if (const int e = check(a, true)) return e;
  const Plan p = plan(a);
  const State s(a, p);
  const Work w(a, p);
  const int esz = a.dt == DT_F32 ? 4 : 2, gsz = a.split ? 2 : esz;
  const float top = p.op == DT_F16 ? 16384.f : p.op == DT_BF16 ? 1.f : 0.f;
  Operand H, W;
  operands(a, p, s, H, W);
  Operand packed = H;
  const bool f16 = p.op == DT_F16;
  const CoefP cp{a.dloss, s.rows, s.count, f[0], top, a.split ? s.eh : nullptr, w.coef, f16 ? w.g : nullptr, f16 ? w.t : nullptr, a.split ? 0 : 12, w.gr};
  PackP pk{H.p, H.ld, H.lo, H.rows, p.pack ? w.packed : nullptr, p.dp * gsz, a.split ? a.N * p.dp * 2 : 0, a.split || p.pad_h ? p.dp * gsz : up(a.D, 16 / esz) * esz,
           a.split ? 2 : 1};
  if (a.N <= 1024) {
    hipLaunchKernelGGL(prepare_kernel, dim3((unsigned)a.N), dim3(256), 0, st, cp, pk);
    VL_CHECK();
  } else {
    hipLaunchKernelGGL(coef_kernel, dim3(1), dim3(1024), 0, st, cp);
    VL_CHECK();
    if (p.pack) {
      hipLaunchKernelGGL(pack_kernel, dim3((unsigned)a.N), dim3(256), 0, st, pk, s.count, cp.t, w.gr);
      VL_CHECK();
    }
  }
  if (p.pack) packed = Operand{w.packed, pk.ldo, pk.half_out, 0, nullptr};
  if (a.want_w && p.nt) {
    TransposeP t{(const uint16_t*)H.p, H.ld / 2, H.lo / 2, w.ht, p.np, a.D * p.np, (int)a.N, (int)a.D, s.count, H.rows, nullptr, 0, cp.t, w.gr};
    hipLaunchKernelGGL(transpose_kernel, dim3((unsigned)((a.N + 63) / 64), (unsigned)((a.D + 63) / 64), a.split ? 2 : 1), dim3(256), 0, st, t);
    VL_CHECK();
    packed = Operand{(const char*)w.ht, p.np * 2, a.split ? a.D * p.np * 2 : 0, 0, nullptr};
  }
  packed.xlim = (int)a.D;
  Operand wt = W;                                                  // W along the sum's axis of the dh product
  if (p.wtr) {
    TransposeP t{(const uint16_t*)W.p, W.ld / 2, W.lo / 2, w.wtr, p.vp, a.D * p.vp, (int)a.V, (int)a.D, nullptr, nullptr, s.count, p.many, nullptr, nullptr};
    hipLaunchKernelGGL(transpose_kernel, dim3((unsigned)((a.V + 63) / 64), (unsigned)((a.D + 63) / 64), a.split ? 2 : 1), dim3(256), 0, st, t);
    VL_CHECK();
    wt = Operand{(const char*)w.wtr, p.vp * 2, a.split ? a.D * p.vp * 2 : 0, (int)a.D, nullptr};
  }
  const int64_t ldg = p.np * gsz, glo = a.split || p.pair ? p.gcols * ldg : 0;
  const int64_t ldr = p.gcols * gsz, rlo = a.split ? p.np * ldr : 0;   // the same row by row (p.nt)
  char* rows_g = w.G + p.np * p.gcols * esz;                       // that layout, or the copy G2
  for (int k = 0; k < p.pieces; ++k) {
    const int v0 = k * p.step, v1 = (int)(a.V < v0 + (int64_t)p.step ? a.V : v0 + p.step), vc = v1 - v0;
    ScoreP q = score_args(a, s, f);
    q.H = H; q.W = W;
    q.W.xlim = (int)a.V;
    q.v0 = v0; q.v1 = v1; q.ref = s.ref; q.inv = s.inv; q.coef = w.coef; q.g = w.g; q.G = w.G; q.ldg = ldg; q.glo = glo;
    if (p.nt && a.want_h) { q.R = rows_g; q.ldr = ldr; q.rlo = rlo; }
    else if (a.split && a.want_h) q.G2 = rows_g;
    if (a.want_b && !a.K) { q.colsum = w.colsum; q.ldc = a.V; }
    if (const int e = scores<true>(q, p.tile, p.op, a.split, p.pair, a.wt, st)) return e;
    if (a.want_b && a.K) {
      hipLaunchKernelGGL(bias_rows_kernel, dim3((vc + 31) / 32), dim3(256), 0, st, w.G, ldg, glo, a.split ? (int)DT_F16 : (int)a.dt, vc, s.count, w.g, w.gr,
                         (char*)a.db + (int64_t)v0 * (a.bdt == DT_F32 ? 4 : 2), (int)a.bdt);
      VL_CHECK();
    }
    Operand G{w.G, ldg, glo, 0, nullptr};
    if (a.want_h) {
      DhP d;
      d.G = p.nt ? Operand{rows_g, ldr, rlo, 0, nullptr} : G;
      d.wide_g = q.G2; d.sc = s.sc;
      d.W = W;
      d.W.p += a.wt ? (int64_t)v0 * gsz : v0 * W.ld;
      d.W.xlim = (int)a.D;
      d.WT = wt;
      d.WT.p += (int64_t)v0 * gsz;
      d.many = p.wtr ? p.many : 0x7fffffff;
      d.count = s.count; d.D = (int)a.D; d.vc = vc; d.units = p.units; d.most = p.most; d.accum = k > 0; d.slab = w.dh_slab;
      const int e = dispatch_dh(d, p.dh_tile, p.op, a.split, p.pair, a.wt, st);
      if (e) return e;
    }
    if (a.want_w) {
      DwP d;
      d.G = G; d.G.xlim = vc;
      d.H = packed; d.count = s.count; d.gr = w.gr;
      d.out = (char*)a.dw + (a.wt ? (int64_t)v0 : v0 * a.D) * esz;
      d.ldo = a.wt ? a.V : a.D;
      d.D = (int)a.D; d.vc = vc; d.shares = p.shares; d.slab = w.dw_slab;
      const int e = a.wt ? dispatch_dw<true>(d, p.dw_tile, p.op, a.split, p.pair, st) : dispatch_dw<false>(d, p.dw_tile, p.op, a.split, p.pair, st);
      if (e) return e;
    }
  }
  const bool sums = a.want_b && !a.K;
  if (a.want_h || sums) {
    const int64_t cols = p.quarters ? 256 : 1024, blocks = (a.D + cols - 1) / cols;
    if (a.N * blocks + (a.V + 255) / 256 > 0x7fffffff) return -2;
    const FinishP q{w.dh_slab, s.rows, s.count, a.split ? s.sc : nullptr, cp.g, w.gr, a.want_h ? (int)a.N : 0, (int)a.D, p.units, p.most, (int)blocks, a.dh, (int)a.dt, w.colsum, p.bm, (int)a.V, a.db, (int)a.bdt};
    const dim3 grid((unsigned)(q.N * blocks + (sums ? (a.V + 255) / 256 : 0)));
    if (p.dh_tile == TILE_BIG) launch_finish<256>(q, p.quarters, grid, st);
    else if (p.dh_tile == TILE_SMALL) launch_finish<64>(q, p.quarters, grid, st);
    else launch_finish<128>(q, p.quarters, grid, st);
  }
  return (int)hipGetLastError();
}

}  // namespace

// bytes of the state, the forward workspace and the backward workspace; sets the fields of the call that layout() decides
DL4J_API void dl4j_linear_loss_bytes(int64_t* args, int64_t* out) {
  Args& a = *reinterpret_cast<Args*>(args);
  layout(a);
  const Plan p = plan(a);
  const Work w(a, p);
  out[0] = State(a, p).bytes;
  out[1] = w.fwd;
  out[2] = w.bwd;
}
// loss [N] of cross entropy (K = 0) or of distillation; f: temperature, label smoothing
DL4J_API int dl4j_linear_loss_fwd(const int64_t* args, const float* f, hipStream_t st) {
  return forward(*reinterpret_cast<const Args*>(args), f, st);
}
// dh [N, D], dw [V, D] ([D, V] with wt), db [V] from dloss [N] and the forward call's state
DL4J_API int dl4j_linear_loss_bwd(const int64_t* args, const float* f, hipStream_t st) {
  return backward(*reinterpret_cast<const Args*>(args), f, st);
}
