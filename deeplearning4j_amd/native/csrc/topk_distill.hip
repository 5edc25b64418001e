// Distillation from a teacher's top logits on logits that are there already (ops/vocab_loss.py topk_distillation):
//
//   p = softmax over the K teacher logits / T (entries with an index < 0 left out), z' = z / T, lse = log sum_j exp z'_j, P = sum_k p_k
//   loss = T^2 (sum_k p_k log p_k - sum_k p_k z'[i_k] + P lse)        dz_j = dloss T (P exp(z'_j - lse) - sum_{k: i_k = j} p_k)
//
// Bound by the logits: forward reads them once (running maximum and sum of the softmax), backward reads them once and writes dz. One
// workgroup per row; 16-byte loads behind a peeled head, since rows of an odd vocabulary start anywhere. The teacher's softmax is K
// values: both directions compute it in LDS instead of passing it through memory. 8192 x 65536 bf16, 128 entries: forward 238 us (4.5 TB/s),
// backward 478 us (4.5 TB/s; a copy reaches 5.0); 4096 x 30522, a fifth of the rows without entries: 60 and 93 us.
#include "common.h"

namespace {

constexpr float NEG_INF = -__builtin_inff();
constexpr int KMAX = 1024;

template <typename T> struct El;
template <> struct El<float> {
  static __device__ __forceinline__ float ld(float v) { return v; }
  static __device__ __forceinline__ float st(float v) { return v; }
};
template <> struct El<bf16_t> {
  static __device__ __forceinline__ float ld(bf16_t v) { return bf2f(v); }
  static __device__ __forceinline__ bf16_t st(float v) { return f2bf(v); }
};
template <> struct El<_Float16> {
  static __device__ __forceinline__ float ld(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 st(float v) { return (_Float16)v; }
};

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dt) {   // 0 fp32, 1 bf16, 2 fp16
  if (dt == 0) return reinterpret_cast<const float*>(p)[i];
  const uint16_t v = reinterpret_cast<const uint16_t*>(p)[i];
  return dt == 1 ? bf2f(v) : (float)__builtin_bit_cast(_Float16, v);
}

// exp(z / T - ref) of a rounded z / T against a reference that is one: 1 at most. Fused to one instruction, the exact product stands against a
// rounded one, and half a step of a logit of 2^30 is more than an exponential holds.
__device__ __forceinline__ float exp_below(float z, float invT, float ref) {
#pragma clang fp contract(off)
  const float t = z * invT;
  return __expf(t - ref);
}

// the teacher's weights of row n in LDS: si[k] index (-1: none), sp[k] = p_k; returns (P, sum p log p) to all threads. NaN or +inf among
// the row's logits, or an entry outside the vocabulary (with any logit but -inf), makes both NaN.
template <int NT>
__device__ __forceinline__ float2 teacher_row(const void* idx, int idx64, const void* t, int tdt, int64_t n, int V, int K, float invT, int* si,
                                              float* sp, float* red) {
  const int tid = threadIdx.x;
  float m = NEG_INF, bad = 0.f;
  for (int k = tid; k < K; k += NT) {
    const int64_t o = n * K + k;
    const int64_t i = idx64 ? reinterpret_cast<const int64_t*>(idx)[o] : (int64_t)reinterpret_cast<const int*>(idx)[o];
    const float l = i < 0 ? NEG_INF : load_any(t, o, tdt), v = l * invT;
    si[k] = i < 0 ? -1 : i > 0x7fffffff ? 0x7fffffff : (int)i;
    sp[k] = v;
    if (!(v < __builtin_inff()) || (i >= V && l != NEG_INF)) bad = 1.f;
    m = fmaxf(m, v);
  }
  m = block_max(m, red);
  bad = block_max(bad, red);
  float s = 0.f;
  for (int k = tid; k < K; k += NT) s += m == NEG_INF ? 0.f : __expf(sp[k] - m);
  s = block_sum(s, red);
  const float inv = s > 0.f ? 1.f / s : 0.f, ls = s > 0.f ? __logf(s) : 0.f;
  float h = 0.f;
  for (int k = tid; k < K; k += NT) {
    const float d = sp[k] - m;
    const float w = m == NEG_INF ? 0.f : __expf(d) * inv;
    if (w > 0.f) h += w * (d - ls);
    sp[k] = bad != 0.f ? __builtin_nanf("") : w;
  }
  h = block_sum(h, red);                                // (its barriers also publish sp)
  if (bad != 0.f) return make_float2(__builtin_nanf(""), __builtin_nanf(""));
  return make_float2(s > 0.f ? 1.f : 0.f, h);
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_fwd_kernel(const T* __restrict__ z, int64_t ldz, const void* __restrict__ idx, int idx64,
                                                         const void* __restrict__ t, int tdt, int V, int K, float Tm, float invT,
                                                         float* __restrict__ loss, float* __restrict__ lse) {
  __shared__ int si[KMAX];
  __shared__ float sp[KMAX];
  __shared__ float red[16];
  constexpr int E = 16 / (int)sizeof(T);
  const int64_t n = blockIdx.x;
  const T* zr = z + n * ldz;
  const int tid = threadIdx.x;
  const float2 pt = teacher_row<NT>(idx, idx64, t, tdt, n, V, K, invT, si, sp, red);
  if (pt.x == 0.f) {                                    // no entry: the row takes no part
    if (tid == 0) { loss[n] = 0.f; lse[n] = 0.f; }
    return;
  }
  const int head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(zr) & 15)) & 15) / sizeof(T)));
  const int nv = (V - head) / E, tail = head + nv * E;
  float m = NEG_INF, s = 0.f;
  auto one = [&](float z) {
    const float nm = fmaxf(m, z * invT);
    if (nm != NEG_INF) s = s * __expf(m - nm) + exp_below(z, invT, nm); else s += z != z ? z : 0.f;
    m = nm;
  };
  if (tid < head) one(El<T>::ld(zr[tid]));
  if (tail + tid < V) one(El<T>::ld(zr[tail + tid]));
  const f32x4* vp = reinterpret_cast<const f32x4*>(zr + head);
#pragma unroll 4
  for (int i = tid; i < nv; i += NT) {
    const f32x4 raw = vp[i];
    T e[E];
    __builtin_memcpy(e, &raw, 16);
    float f[E], mx = NEG_INF;
#pragma unroll
    for (int j = 0; j < E; ++j) { f[j] = El<T>::ld(e[j]); mx = fmaxf(mx, f[j] * invT); }
    const float nm = fmaxf(m, mx), ref = nm == NEG_INF ? 0.f : nm;
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) a += exp_below(f[j], invT, ref);
    s = s * __expf(m - ref) + a;                        // m = -inf: s is 0 (or NaN) there
    m = nm;
  }
  const float M = block_max(m, red), ref = M == NEG_INF ? 0.f : M;
  s = block_sum(m == NEG_INF ? s : s * __expf(m - ref), red);
  const float L = M + __logf(s);
  float c = 0.f;
  for (int k = tid; k < K; k += NT) {
    const float w = sp[k];
    if (w == 0.f) continue;
    c += si[k] < V ? w * (El<T>::ld(zr[si[k]]) * invT) : __builtin_nanf("");   // (w is NaN too)
  }
  c = block_sum(c, red);
  if (tid == 0) {
    loss[n] = Tm * Tm * (pt.y - c + pt.x * L);
    lse[n] = c != c ? c : L;
  }
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_bwd_kernel(const T* __restrict__ z, int64_t ldz, const void* __restrict__ idx, int idx64,
                                                         const void* __restrict__ t, int tdt, int V, int K, float Tm, float invT,
                                                         const float* __restrict__ lse, const float* __restrict__ dloss, T* __restrict__ dz) {
  __shared__ int si[KMAX];
  __shared__ float sp[KMAX];
  __shared__ float red[16];
  constexpr int E = 16 / (int)sizeof(T);
  const int64_t n = blockIdx.x;
  const T* zr = z + n * ldz;
  T* out = dz + n * V;
  const int tid = threadIdx.x;
  const float2 pt = teacher_row<NT>(idx, idx64, t, tdt, n, V, K, invT, si, sp, red);
  const bool none = pt.x == 0.f;
  const float c = dloss[n] * Tm, cp = c * pt.x, L = lse[n];
  // the heads of the two rows differ where ldz is not V: whole 16-byte pieces only where both are aligned alike
  const bool alike = ((reinterpret_cast<uintptr_t>(zr) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const int head = alike ? min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(zr) & 15)) & 15) / sizeof(T))) : V;
  const int nv = (V - head) / E, tail = head + nv * E;
  auto one = [&](int j) { out[j] = El<T>::st(none ? 0.f : cp * exp_below(El<T>::ld(zr[j]), invT, L)); };
  for (int j = tid; j < head; j += NT) one(j);
  if (tail + tid < V) one(tail + tid);
  const f32x4* vp = reinterpret_cast<const f32x4*>(zr + head);
  f32x4* op = reinterpret_cast<f32x4*>(out + head);
  if (none) {
    for (int i = tid; i < nv; i += NT) op[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    return;
  }
#pragma unroll 4
  for (int i = tid; i < nv; i += NT) {
    f32x4 raw = vp[i];
    T e[E];
    __builtin_memcpy(e, &raw, 16);
#pragma unroll
    for (int j = 0; j < E; ++j) e[j] = El<T>::st(cp * exp_below(El<T>::ld(e[j]), invT, L));
    __builtin_memcpy(&raw, e, 16);
    op[i] = raw;
  }
  __syncthreads();
  for (int k = tid; k < K; k += NT) {
    const int i = si[k];
    if (i < 0 || i >= V || sp[k] == 0.f) continue;
    float q = 0.f;
    for (int j = 0; j < K; ++j) q += si[j] == i ? sp[j] : 0.f;     // an index may come twice: all its entries write the same value
    out[i] = El<T>::st(c * (pt.x * exp_below(El<T>::ld(zr[i]), invT, L) - q));
  }
}

template <typename T>
int launch(bool bwd, const void* z, int64_t ldz, const void* idx, int idx64, const void* t, int tdt, int N, int V, int K, float T_, float* loss,
           float* lse, const float* dloss, void* dz, hipStream_t st) {
  constexpr int NT = 256;
  if (bwd) hipLaunchKernelGGL((distill_bwd_kernel<T, NT>), dim3(N), dim3(NT), 0, st, (const T*)z, ldz, idx, idx64, t, tdt, V, K, T_, 1.f / T_, lse, dloss, (T*)dz);
  else hipLaunchKernelGGL((distill_fwd_kernel<T, NT>), dim3(N), dim3(NT), 0, st, (const T*)z, ldz, idx, idx64, t, tdt, V, K, T_, 1.f / T_, loss, lse);
  return (int)hipGetLastError();
}

int dispatch(bool bwd, const void* z, int64_t ldz, const void* idx, int idx64, const void* t, int tdt, int N, int V, int K, int dt, float T,
             float* loss, float* lse, const float* dloss, void* dz, hipStream_t st) {
  if (N <= 0 || V <= 0 || K <= 0 || K > KMAX || ldz < V || !(T > 0.f) || tdt < 0 || tdt > 2 || !z || !idx || !t || !lse) return -2;
  if (bwd ? !dloss || !dz : !loss) return -2;
  switch (dt) {
    case 0: return launch<float>(bwd, z, ldz, idx, idx64, t, tdt, N, V, K, T, loss, lse, dloss, dz, st);
    case 1: return launch<bf16_t>(bwd, z, ldz, idx, idx64, t, tdt, N, V, K, T, loss, lse, dloss, dz, st);
    case 2: return launch<_Float16>(bwd, z, ldz, idx, idx64, t, tdt, N, V, K, T, loss, lse, dloss, dz, st);
  }
  return -2;
}

}  // namespace

// One call (ops/vocab_loss.py lists the same fields in the same order). Types: 0 fp32, 1 bf16, 2 fp16.
// loss != null: loss [N] and lse [N] (of z / T, for the backward call); else dz [N][V] from dloss [N] and lse.
struct DistillArgs {
  int64_t N, V, K, ldz, dt, idx64, tdt;
  const void *z, *idx, *t;
  float *loss, *lse; const float* dloss; void* dz;
};
DL4J_API int dl4j_topk_distill(const int64_t* args, const float* f, hipStream_t st) {
  const DistillArgs& a = *reinterpret_cast<const DistillArgs*>(args);
  if (a.N > 0x7fffffff || a.V > 0x7fffffff || a.K > KMAX) return -2;
  return dispatch(a.loss == nullptr, a.z, a.ldz, a.idx, (int)a.idx64, a.t, (int)a.tdt, (int)a.N, (int)a.V, (int)a.K, (int)a.dt, f[0], a.loss, a.lse, a.dloss,
                  a.dz, st);
}
