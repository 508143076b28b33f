// What the kernels on rows of logits share that are neither the cross entropy's nor bound to whole vectors: scores, streaming
// softmax statistics, 16-byte access to rows of any alignment.
//
// Scores z = cap(x) / temperature, cap(x) = softcap * tanh(x / softcap) or x.  A thread's statistics are of what it has seen:
//   m   largest level (what exponentials are taken against: a logit, or with a soft-cap its score), s = sum exp(z - m), t = sum exp(z - m) (z - m)
// so that ln sum exp z = m + ln s, and the entropy of softmax(z) is ln s - t / s.  Everything is fp32.  z - m is formed from the difference of the
// logits, so that rows at the type's lowest value or about 1e30 are exact where scores near the largest are, at any temperature; a score of minus
// infinity has exp = 0 and adds nothing to t (z - m is cut at -200, where exp is 0 in fp32).
#pragma once
#include "common.h"

namespace rows {

constexpr int64_t LAST_CACHE = 256ll << 20;  // bytes that the cache behind the L2s holds

typedef u32x4 __attribute__((aligned(2))) u32x4_any;  // 16 bytes at any element
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// 16 bytes of a row as numbers
template <typename T> struct Vec;
template <> struct Vec<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const u32x4& w, float* f) {
    Pack8 t;
    t.u = w;
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = bf2f(t.e[e]);
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    Pack8 t;
#pragma unroll
    for (int e = 0; e < 8; e++) t.e[e] = f2bf(f[e]);
    return t.u;
  }
};
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const u32x4& w, float* f) {
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] = __uint_as_float(w[e]);
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = __float_as_uint(f[e]);
    return w;
  }
};
// N numbers of a row as they are loaded: 16 or (N fp32 numbers for 16 bytes of bf16) 32 bytes
template <typename T, int N> struct Raw {
  static constexpr int W = N / Vec<T>::N;
  u32x4 w[W];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = *reinterpret_cast<const u32x4_any*>(p + i * Vec<T>::N);
  }
  __device__ __forceinline__ void load_once(const T* p) {
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p + i * Vec<T>::N));
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int i = 0; i < W; i++) Vec<T>::unpack(w[i], f + i * Vec<T>::N);
  }
};

// A row of n elements as `head` single ones, nvec vectors of N that begin at 16-byte boundaries of T, and the rest
struct Cut {
  int head, nvec, edges;  // edges: head and rest
  __device__ __forceinline__ int edge(int e, int n) const { return e < head ? e : n - (edges - e); }  // element of edge e
};
template <typename T, int N> __device__ __forceinline__ Cut cut(const T* row, int n) {
  Cut c;
  c.head = min(n, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T));
  c.nvec = (n - c.head) / N;
  c.edges = n - c.nvec * N;
  return c;
}

// tanh(x / softcap) = 1 - 2 r, r = 1 / (exp(2 x / softcap) + 1), so that a capped score is one fma on r, and its slope dy / dx is 4 r (1 - r).  That is off by softcap 2^-21 / temperature
// whatever the score, so that a soft-cap far above the logits would leave nothing of them: above WIDE_CAP scores of |x| < softcap / 4 are x (1 - y^2 / 3 + 2 y^4 / 15 - ..) / temperature, y = x /
// softcap (the series left off behind y^8: 8.4e-9 of it at most), and all are as exact as they are large: 2^-19 of themselves.  The series and the choice are ten more issue slots a logit; us
// with scores of the first kind | of the second, bf16: 1500 x 256000 with 64 alternatives 203 | 214, its gradient 308 | 367, distillation of 4096 x 100352 407 | 533, the LM head's scores of 2048 x 4096
// x 100352 1237 | 1260, x 256 227 | 257.
constexpr float WIDE_CAP = 64.f;
struct Scale {
  int kind;                   // of the kernels that run: 0 no soft-cap, 1 up to WIDE_CAP, 2 above (CAP)
  float cap, cap_k, inv_tau;  // cap_k = 2 log2(e) / cap; cap 0: none
  float inv_cap;
  float r_k, top;             // a capped score is r_k r + top: r_k = -2 cap / temperature, top = cap / temperature
  float unit, unit2;          // of a level (see level), in scores: 1, or 1 / temperature; and in powers of two
};
// (a soft-cap below 8.5e-39 has no factor of x in fp32: 0 would become NaN)
inline bool takes(float temperature, float softcap) { return temperature >= 1e-6f && temperature <= 1e6f && (softcap == 0.f || (softcap >= 1e-30f && softcap <= 1e30f)); }
inline Scale scale_of(float temperature, float softcap) {
  Scale c;
  c.kind = softcap > WIDE_CAP ? 2 : softcap > 0.f ? 1 : 0;
  c.cap = softcap;
  c.inv_cap = softcap > 0.f ? 1.f / softcap : 0.f;
  c.cap_k = softcap > 0.f ? 2.f * LOG2E / softcap : 0.f;
  c.inv_tau = 1.f / temperature;
  c.top = softcap * c.inv_tau;
  c.r_k = -2.f * c.top;
  c.unit = softcap > 0.f ? 1.f : c.inv_tau;
  c.unit2 = c.unit * LOG2E;
  return c;
}
__device__ __forceinline__ float tail_of_tanh(float x, const Scale& c) { return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * c.cap_k) + 1.f); }
// What rows are compared by, and exponentials are taken against: capped scores, or the logits themselves, whose scores may have no room in fp32 (the type's lowest value at a
// temperature below 1) where their differences have.
template <int CAP> __device__ __forceinline__ float level(float x, const Scale& c) {
  if (CAP == 0) return x;
  const float far = __builtin_fmaf(tail_of_tanh(x, c), c.r_k, c.top);
  if (CAP == 1) return far;
  const float y = x * c.inv_cap, y2 = y * y, z = x * c.inv_tau;
  const float p = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(62.f / 2835.f, y2, -17.f / 315.f), y2, 2.f / 15.f), y2, -1.f / 3.f) * y2;
  return fabsf(y) < 0.25f ? __builtin_fmaf(z, p, z) : far;
}
// a value that all threads of the workgroup have, in a scalar register
__device__ __forceinline__ float uniform(float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); }
// z - m, m the score of level m
template <int CAP> __device__ __forceinline__ float behind(float x, const Scale& c, float m) {
  if (CAP == 1) return __builtin_fmaf(tail_of_tanh(x, c), c.r_k, c.top - m);
  if (CAP == 2) return level<2>(x, c) - m;
  const float d = (x - m) * c.unit;
  return d == -INFINITY && x > -INFINITY ? __builtin_fmaf(x, c.unit, -m * c.unit) : d;  // (at a temperature above 1 the scores may have the room that the logits have not)
}
// dz / dx
template <int CAP> __device__ __forceinline__ float slope(float x, const Scale& c) {
  if (!CAP) return c.inv_tau;
  const float r = tail_of_tanh(x, c);
  return 4.f * r * (1.f - r) * c.inv_tau;
}
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }
// exp(z - m)
template <int CAP> __device__ __forceinline__ float exp_behind(float x, const Scale& c, float m) {
  return CAP ? exp_of(behind<CAP>(x, c, m)) : __builtin_amdgcn_exp2f((x - m) * c.unit2);
}
__device__ __forceinline__ float log_of(float s) { return __builtin_amdgcn_logf(s) * LN2; }

// Statistics of what a thread has seen: the largest level, the sum of exponentials behind it, that sum weighted by z - m; m = -inf: nothing above minus infinity yet.
struct Stat {
  float m, s, t;
  static __device__ __forceinline__ Stat none() { return Stat{-INFINITY, 0.f, 0.f}; }
  __device__ __forceinline__ float ref() const { return m == -INFINITY ? 0.f : m; }  // against which every exponential of such a thread is 0
  // the largest level is m2 now
  __device__ __forceinline__ void raise(float m2, float unit) {
    if (m != -INFINITY) {
      const float d = (m - m2) * unit, f = exp_of(d);
      t = f * (t + s * fmaxf(d, -200.f));
      s *= f;
    }
    m = m2;
  }
  __device__ __forceinline__ void join(const Stat& o, float unit) {
    Stat b = o;
    if (b.m > m) raise(b.m, unit);
    else if (m > b.m) b.raise(m, unit);
    s += b.s;
    t += b.t;
  }
};
// Largest value and sum of a workgroup of NW waves (a power of two), with one register for the waves' results, which each lane has one of.
template <int NW, bool MAX> __device__ __forceinline__ float block_reduce(float v, float* red) {
  auto both = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
  v = MAX ? wave_max(v) : wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[threadIdx.x & (NW - 1)];
#pragma unroll
  for (int o = NW / 2; o > 0; o >>= 1) v = both(v, __shfl_xor(v, o, 64));
  return v;
}
template <int NW> __device__ __forceinline__ Stat block_join(Stat a, Stat* red, float unit) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor(a.m, o, 64);
    b.s = __shfl_xor(a.s, o, 64);
    b.t = __shfl_xor(a.t, o, 64);
    a.join(b, unit);
  }
  if (NW == 1) return a;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int i = 1; i < NW; i++) a.join(red[i], unit);
  return a;
}

// d / d x of g ln p[target] + h entropy: (g (i == target) - p (g + h (ln p + H))) dz/dx, from the row's m (a score, as
// stats hold it), ln S and H
template <int CAP, bool ENT>
__device__ __forceinline__ float score_grad(float x, const Scale& c, float m, float log_sum, float entropy, float g, float h, bool target) {
  const float logp = (CAP ? behind<CAP>(x, c, m) : __builtin_fmaf(x, c.inv_tau, -m)) - log_sum;
  float d = -exp_of(logp) * (ENT ? __builtin_fmaf(h, fmaxf(logp, -200.f) + entropy, g) : g);
  if (target) d += g;
  return d * slope<CAP>(x, c);
}

// Whether rows of n numbers of `size` bytes at a and b share memory in another way than being the same (a + b in place is each element over itself).
inline bool overlap(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t rows, int64_t n, int size) {
  const int64_t d = ((const char*)b - (const char*)a) / size;  // (both are aligned to their type)
  if (a == b || !b || d >= (rows - 1) * lda + n || -d >= (rows - 1) * ldb + n) return false;
  const int64_t at = lda == ldb ? ((d % lda) + lda) % lda : 0;
  return at < n || at + n > lda;
}

}  // namespace rows

// gemm.hip: the LM head's product with a row's part of its softmax in the epilogue (logprobs.hip): logits leave the kernel only as what is formed of them.
struct HeadRows {
  const int32_t* targets;     // [rows]
  int32_t ignore_index, V;    // V: of the whole product; a target from there on has no logit
  int32_t rows;               // that there are: up to M, those behind pad the product (their gradients are zeros)
  rows::Scale scale;
  float *parts, *target_logit;  // statistics: [ceil(N / 256)][M][3], (Stat) of 256 columns; the
                                // logit x of each target that is one of the columns
  const float *stats, *dlogprobs, *dentropy;  // gradients: from [M, 3], [M], [M] (optional)
};
// Whether the forms run on a product of that size (operands 16-byte aligned, rows of K numbers), and how many of the N columns they take: whole rounds of tiles, or all;
// 0: the plain product does better.
int olmax_gemm_head_columns(int M, int N, int K);
int olmax_gemm_head_stats(hipStream_t s, const bf16* h, const bf16* w, int M, int N, int K, const HeadRows& rows);
// d [M, ldd] (16-byte aligned, ldd a multiple of 8): columns 0 .. N
int olmax_gemm_head_grads(hipStream_t s, const bf16* h, const bf16* w, bf16* d, int64_t ldd, int M, int N, int K, const HeadRows& rows);

// lmhead_rows.hip: the LM head's products on fewer tokens than a tile of 256 has rows.  Whether large tiles do better with the tokens padded to 256 (for the logits of more than
// 64 tokens, and for the gradients):
bool olmax_lmhead_pads(int64_t T, int32_t d, int32_t V);
// Whether, where that is not so, the gradients do better with the tokens padded to 64:
bool olmax_lmhead_pads_64(int64_t T, int32_t d, int32_t V);
// dst [padded, d] = src [rows, d] and zeros; d is a multiple of 8 and both are 16-byte aligned
void olmax_pad_rows(hipStream_t s, const bf16* src, bf16* dst, int64_t rows, int64_t padded, int d);
// columns [0, n) of rows [from, to) of d = 0
void olmax_zero_rows(hipStream_t s, bf16* d, int64_t from, int64_t to, int64_t n, int64_t ld);
// olmax_lmhead_products of T tokens padded to `rows`, 64 or 256, that dlogits and tmp [rows, d], for dh, have memory of.  h_pad is h and zeros up to row 63; where T < 64 so is dlogits
// (other rows of it may hold anything).
int olmax_lmhead_products_few(hipStream_t stream, const bf16* dlogits, const bf16* W, const bf16* h, const bf16* h_pad, bf16* dh, void* dW, int T, int d, int V, int64_t ldl,
                              bool dw_f32, bf16* tmp, int rows, GemmScratch scratch);

// What the LM head's calls are given, for their checks ahead of any launch (olmax_model_logprobs and its like make them ahead of the model's).
struct HeadScore {
  const void *h, *W;
  const int32_t* targets;
  float *logprobs, *entropy, *stats;
  int32_t* top_ids;
  float* top_logprobs;
  void* workspace;
  int64_t workspace_bytes, T;
  int32_t d, V, top, ignore_index;
  float temperature, softcap;
};
struct HeadScoreGrad {
  const void *h, *W;
  const int32_t* targets;
  const float *stats, *dlogprobs, *dentropy;
  void *dh, *dW, *workspace;
  int64_t workspace_bytes, T;
  int32_t d, V;
  float temperature, softcap;
};
struct HeadDistill {
  const void *h, *W;
  const int32_t* top_ids;
  const float* top_logprobs;
  float* loss;
  void *dh, *workspace;
  int64_t workspace_bytes, T;
  int32_t d, V, k, tail;
  float temperature, softcap;
};
int olmax_lmhead_logprobs_check(const HeadScore& a);
int olmax_lmhead_logprobs_bwd_check(const HeadScoreGrad& a);
int olmax_lmhead_distill_check(const HeadDistill& a);
