// Distillation from a teacher's top logits: the divergence of the student's softmax from what the teacher says about its k best tokens, with the gradient.
//
// p = softmax(z), z = cap(x) / temperature of the student (rows.h); the teacher gives k tokens id_j and numbers t_j of a row.
//   tail 0 (renormalize): q = softmax_k(t / temperature), the teacher's distribution over its k tokens alone (t: logits or log probabilities)
//     L = sum_j q_j (ln q_j - ln p_j)                     dL/dz_i = p_i - q_i
//   tail 1 (bucket): q_j = exp(t_j), and all other tokens are one event of probability r = 1 - sum q, s = sum of the others' p
//     L = sum_j q_j (ln q_j - ln p_j) + r ln(r / s)       dL/dz_i = p_i - q_i for the k tokens, p_i (1 - r / s) for the others
// s is summed over the others by themselves (1 - sum p_j would leave nothing of a small one): a bit of LDS per token says which those are.
#include "rows.h"
#include <algorithm>
#include <mutex>

using namespace rows;

namespace {

constexpr int MAX_TOP = 128;
constexpr int COUNT_IN_ROWS = 1024;  // up to so many rows each workgroup counts them itself
constexpr float LEAST_TAIL = 0x1p-20f;  // fp32 log probabilities leave less than this undetermined: a tail below it is none (a student without other tokens would lose infinitely by it)
constexpr int MAX_BITS = 1 << 20;    // tokens that a workgroup can keep a bit of (128 KB)

template <int NW> __device__ __forceinline__ float counted_rows(const int32_t* ids, int64_t T, int k, float* red) {
  float n = 0.f;
  for (int64_t i = threadIdx.x; i < T; i += NW * 64) n += ids[i * k] >= 0 ? 1.f : 0.f;
  return block_sum<NW>(n, red);
}

__global__ __launch_bounds__(1024) void distill_count_kernel(const int32_t* __restrict__ ids, int64_t T, int k, float* __restrict__ n) {
  __shared__ float red[16];
  const float c = counted_rows<16>(ids, T, k, red);
  if (threadIdx.x == 0) *n = c;
}

__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ row_loss, const int32_t* __restrict__ ids, int64_t T, int k, float* __restrict__ loss,
                                                           int mean) {
  __shared__ float red[16];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < T; i += 1024) s += row_loss[i];
  s = block_sum<16>(s, red);
  const float n = mean ? counted_rows<16>(ids, T, k, red) : 1.f;
  if (threadIdx.x == 0) *loss = n > 0.f ? s / n : 0.f;
}

struct Teacher {
  const int32_t* ids;
  const float* t;
  int k;
};

// One workgroup a row.  The first pass takes the statistics and the loss, the second writes the gradient of all tokens, and the k tokens' own follow.
template <typename T, typename TO, bool CAP, bool BUCKET, int TH>
__global__ __launch_bounds__(TH) void distill_rows_kernel(const T* __restrict__ logits, TO* __restrict__ dlogits, Teacher teacher, float* __restrict__ row_loss,
                                                          const float* __restrict__ drow, const float* __restrict__ n_counted, int64_t rows, int V, int64_t ld,
                                                          int64_t ldd, Scale c, float dloss, int mean, int pad) {
  constexpr int N = Vec<TO>::N, NW = TH / 64, UNROLL = 4, SPAN = TH * UNROLL;
  extern __shared__ unsigned bits[];  // BUCKET: of the k tokens, element i at i + shift
  __shared__ int ids[MAX_TOP];
  __shared__ Stat red[NW];
  __shared__ float sums[NW];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, k = teacher.k;
  const T* zr = logits + row * ld;
  TO* dr = dlogits ? dlogits + row * ldd : nullptr;
  const Cut cutting = dr ? cut<TO, N>(dr, V) : cut<T, N>(zr, V);
  if (teacher.ids[row * k] < 0) {  // left out
    if (tid == 0) row_loss[row] = 0.f;
    if (dr) {
      float zero[N] = {};
      for (int v = tid; v < cutting.nvec; v += TH) *reinterpret_cast<u32x4*>(dr + cutting.head + v * N) = Vec<TO>::pack(zero);
      if (tid < cutting.edges) dr[cutting.edge(tid, V)] = (TO)0.f;
      if (tid < pad) dr[V + tid] = (TO)0.f;
    }
    return;
  }
  // ---- the teacher's side; thread j has token j
  const int id = tid < k ? teacher.ids[row * k + tid] : -1;
  bool mine = id >= 0 && id < V;
  const float t = mine ? teacher.t[row * k + tid] : -INFINITY;
  const float xj = mine ? (float)zr[id] : 0.f;
  if (tid < MAX_TOP) ids[tid] = mine ? id : -1;
  const int shift = (N - cutting.head) & (N - 1);
  if (BUCKET)
    for (int i = tid; i < (V + N + 31) / 32; i += TH) bits[i] = 0;
  __syncthreads();
  for (int j = 0; j < tid && mine; j++) mine = ids[j] != id;  // a token that is named again counts once
  if (BUCKET && mine) atomicOr(&bits[(id + shift) >> 5], 1u << ((id + shift) & 31));
  float q, logq, r = 0.f;
  if (BUCKET) {
    q = mine ? __expf(t) : 0.f;
    logq = t;
    r = 1.f - block_sum<NW>(q, sums);
    if (r < LEAST_TAIL) r = 0.f;
  } else {
    const float best = block_max<NW>(mine ? t : -INFINITY, sums);
    const float d = (t - best) * c.inv_tau, e = mine && best > -INFINITY ? exp_of(d) : 0.f;
    const float sum = block_sum<NW>(e, sums);
    q = sum > 0.f ? e / sum : 0.f;
    logq = d - log_of(sum);
  }
  const float weight = block_sum<NW>(q, sums) + r;  // 1, but for rounding; 0: nothing to learn
  float n = 1.f;
  if (mean && dr) n = n_counted ? *n_counted : counted_rows<NW>(teacher.ids, rows, k, sums);

  // ---- pass 1: largest score, sum of exponentials (BUCKET: of the other tokens)
  const T* body = zr + cutting.head;
  const unsigned char* byte_of = reinterpret_cast<const unsigned char*>(bits);
  auto inside = [&](int v) {  // which elements of a vector are among the k
    const int at = cutting.head + v * N + shift;
    return N == 8 ? (unsigned)byte_of[at >> 3] : (byte_of[at >> 3] >> (at & 4)) & 15u;
  };
  Raw<T, N> next[UNROLL];
  auto fetch = [&](int at) {
#pragma unroll
    for (int u = 0; u < UNROLL; u++)
      if (at + u * TH + tid < cutting.nvec) next[u].load(body + (int64_t)(at + u * TH + tid) * N);
  };
  fetch(0);
  Stat a = Stat::none();
  const bool has_edge = tid < cutting.edges;
  const int edge = has_edge ? cutting.edge(tid, V) : 0;
  const float edge_x = has_edge ? (float)zr[edge] : -INFINITY;
  if (has_edge && (CAP || edge_x > -INFINITY)) a.m = score<CAP>(edge_x, c);
  if (has_edge && !(BUCKET && (bits[(edge + shift) >> 5] >> ((edge + shift) & 31) & 1))) a.s = exp_of(behind<CAP>(edge_x, c, a.ref()));
  for (int at = 0; at < cutting.nvec; at += SPAN) {
    Raw<T, N> now[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) now[u] = next[u];
    fetch(at + SPAN);
    float cm = -INFINITY;
    bool any = false;
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      if (at + u * TH + tid >= cutting.nvec) continue;
      any = true;
      float x[N];
      now[u].unpack(x);
#pragma unroll
      for (int e = 0; e < N; e++) cm = fmaxf(cm, x[e]);
    }
    const float top = score<CAP>(cm, c);
    if (any && top > a.m) a.raise(top);
    const float ref = a.ref();
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const int v = at + u * TH + tid;
      if (v >= cutting.nvec) continue;
      float x[N];
      now[u].unpack(x);
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = exp_of(behind<CAP>(x[e], c, ref));
      if (BUCKET) {
        const unsigned in = inside(v);
        if (in)
#pragma unroll
          for (int e = 0; e < N; e++) x[e] = in >> e & 1 ? 0.f : x[e];
      }
#pragma unroll
      for (int w = N / 2; w > 0; w >>= 1)
#pragma unroll
        for (int e = 0; e < w; e++) x[e] += x[e + w];
      a.s += x[0];
    }
  }
  a = block_join<NW>(a, red);
  const float dj = behind<CAP>(xj, c, a.ref()), ej = mine ? exp_of(dj) : 0.f;
  const float rest = a.s, sum = BUCKET ? rest + block_sum<NW>(ej, sums) : rest;
  const bool none = sum == 0.f;  // no score above minus infinity: no distribution, nothing to learn from
  const float log_sum = log_of(sum);
  float loss = block_sum<NW>(q > 0.f ? q * (logq - (dj - log_sum)) : 0.f, sums);
  if (BUCKET && r > 0.f) loss += r * (log_of(r) - (log_of(rest) - log_sum));
  if (tid == 0) row_loss[row] = none ? 0.f : loss;
  if (!dr) return;

  // ---- pass 2: the gradient, in place allowed (every thread reads what it writes, the k logits are in registers)
  const float scale = none || weight == 0.f ? 0.f : dloss * (drow ? drow[row] : 1.f) / n;
  const float inv_sum = none ? 0.f : 1.f / sum;
  const float out_scale = scale * (weight * inv_sum - (BUCKET && rest > 1e-30f ? r / rest : 0.f)) * c.inv_tau;
  auto chain = [&](float x) {
    if (!CAP) return 1.f;
    const float y = 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * c.cap_k) + 1.f);
    return 1.f - y * y;
  };
  const float m = a.ref();
  for (int v = tid; v < cutting.nvec; v += TH) {
    const int i = cutting.head + v * N;
    Raw<T, N> w;
    w.load(zr + i);
    float x[N];
    w.unpack(x);
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = exp_of(behind<CAP>(x[e], c, m)) * out_scale * chain(x[e]);
    *reinterpret_cast<u32x4*>(dr + i) = Vec<TO>::pack(x);
  }
  if (has_edge) dr[edge] = (TO)(exp_of(behind<CAP>(edge_x, c, m)) * out_scale * chain(edge_x));
  if (tid < pad) dr[V + tid] = (TO)0.f;
  __syncthreads();  // behind the vectors that hold them
  if (mine) dr[id] = (TO)((ej * inv_sum * weight - q) * scale * c.inv_tau * chain(xj));
}

}  // namespace

// Workspace: T floats (row losses) and the number of counted rows.
extern "C" int64_t olmax_distill_workspace_bytes(int64_t T) { return ((T * 4 + 15) / 16) * 16 + 16; }

static int distill_check(const char* name, int64_t T, int32_t V, int32_t k, int32_t tail, float temperature, float softcap) {
  OLMAX_CHECK(T > 0 && V > 0 && T < (1LL << 24), OLMAX_ERR_SHAPE, "%s: bad shape T=%ld V=%d", name, (long)T, V);
  OLMAX_CHECK(k >= 1 && k <= MAX_TOP, OLMAX_ERR_ARG, "%s: 1 to %d tokens of the teacher a row (got %d)", name, MAX_TOP, k);
  OLMAX_CHECK(tail == 0 || (tail == 1 && V <= MAX_BITS - 32), OLMAX_ERR_ARG, "%s: tail must be 0 (renormalize) or 1 (bucket, up to %d logits)", name, MAX_BITS - 32);
  OLMAX_CHECK(temperature >= 1e-6f && temperature <= 1e6f && softcap >= 0.f && softcap <= 1e30f, OLMAX_ERR_ARG, "%s: temperature within 1e-6 and 1e6, softcap not negative", name);
  return OLMAX_OK;
}

// grads_bf16: the gradient of fp32 logits as bf16 (the LM head's products take it); pad: zeros behind each of its rows
static int distill(hipStream_t stream, const void* logits, void* dlogits, const int32_t* ids, const float* t, float* loss, const float* dloss_rows,
                   void* workspace, int64_t T, int32_t V, int32_t k, int64_t ld, int64_t ldd, bool logits_f32, bool grads_f32, int32_t tail, float temperature,
                   float softcap, float dloss, int32_t reduction, int pad) {
  Scale c;
  c.cap = softcap;
  c.cap_k = softcap > 0.f ? 2.f * LOG2E / softcap : 0.f;
  c.inv_tau = 1.f / temperature;
  float* row_loss = reduction == 2 ? loss : (float*)workspace;
  float* n = nullptr;
  if (reduction == 0 && dlogits && T > COUNT_IN_ROWS) {
    n = (float*)((char*)workspace + ((T * 4 + 15) / 16) * 16);
    hipLaunchKernelGGL(distill_count_kernel, dim3(1), dim3(1024), 0, stream, ids, T, k, n);
  }
  const Teacher teacher{ids, t, k};
#define ROWS(TY, TO, CAPV, BUCKETV, THV)                                                                                                               \
  do {                                                                                                                                                 \
    auto kern = distill_rows_kernel<TY, TO, CAPV, BUCKETV, THV>;                                                                                       \
    static std::once_flag attr_once; /* per instantiation */                                                                                           \
    std::call_once(attr_once, [&] { (void)hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, MAX_BITS / 8); });        \
    hipLaunchKernelGGL(kern, dim3((unsigned)T), dim3(THV), BUCKETV ? (V + 8 + 31) / 32 * 4 : 0, stream, (const TY*)logits, (TO*)dlogits, teacher, row_loss, \
                       dloss_rows, (const float*)n, T, V, ld, ldd, c, dloss, (int)(reduction == 0), pad);                                              \
  } while (0)
#define ROWS_H(TY, TO, CAPV, BUCKETV) do { if (V <= 16384) ROWS(TY, TO, CAPV, BUCKETV, 256); else ROWS(TY, TO, CAPV, BUCKETV, 512); } while (0)
#define ROWS_B(TY, TO, CAPV) do { if (tail) ROWS_H(TY, TO, CAPV, true); else ROWS_H(TY, TO, CAPV, false); } while (0)
#define ROWS_C(TY, TO) do { if (softcap > 0.f) ROWS_B(TY, TO, true); else ROWS_B(TY, TO, false); } while (0)
  if (logits_f32 && grads_f32) ROWS_C(float, float); else if (logits_f32) ROWS_C(float, bf16); else ROWS_C(bf16, bf16);
#undef ROWS
#undef ROWS_H
#undef ROWS_B
#undef ROWS_C
  if (reduction != 2) hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, (const float*)row_loss, ids, T, k, loss, (int)(reduction == 0));
  OLMAX_LAUNCH_CHECK();
  return OLMAX_OK;
}

extern "C" int32_t olmax_distill(hipStream_t stream, const void* logits, void* dlogits, const int32_t* top_ids, const float* top_logprobs, float* loss,
                                 const float* dloss_rows, void* workspace, int64_t workspace_bytes, int64_t T, int32_t V, int32_t k, int64_t ld,
                                 int64_t ldd, int32_t logits_f32, int32_t tail, float temperature, float softcap, float dloss, int32_t reduction) {
  OLMAX_CHECK(logits && top_ids && top_logprobs && loss && workspace, OLMAX_ERR_ARG, "olmax_distill: null pointer");
  if (int rc = distill_check("olmax_distill", T, V, k, tail, temperature, softcap)) return rc;
  OLMAX_CHECK(ld >= V && (!dlogits || ldd >= V), OLMAX_ERR_SHAPE, "olmax_distill: row strides of %ld and %ld are shorter than %d logits", (long)ld, (long)ldd, V);
  OLMAX_CHECK(reduction >= 0 && reduction <= 2, OLMAX_ERR_ARG, "olmax_distill: reduction must be 0 (mean), 1 (sum) or 2 (none)");
  OLMAX_CHECK(!dloss_rows || reduction == 2, OLMAX_ERR_ARG, "olmax_distill: a per-row cotangent only goes with reduction none");
  OLMAX_CHECK((((uintptr_t)logits | (uintptr_t)dlogits) & (logits_f32 ? 3 : 1)) == 0, OLMAX_ERR_ALIGN, "olmax_distill: operands not aligned to their type");
  OLMAX_CHECK(logits != dlogits || ld == ldd, OLMAX_ERR_ARG, "olmax_distill: in place wants one row stride");
  OLMAX_CHECK(workspace_bytes >= olmax_distill_workspace_bytes(T) && aligned16(workspace), OLMAX_ERR_WORKSPACE, "olmax_distill: workspace needs %ld bytes, 16-byte aligned",
              (long)olmax_distill_workspace_bytes(T));
  return distill(stream, logits, dlogits, top_ids, top_logprobs, loss, dloss_rows, workspace, T, V, k, ld, ldd, logits_f32 != 0, logits_f32 != 0, tail,
                 temperature, softcap, dloss, reduction, 0);
}

// ---- with the LM head's product, forward and backward in one call.  Logits fp32 in the workspace, their gradient bf16 behind them.
static int64_t head_stride(int32_t V) { return ((int64_t)V + 63) / 64 * 64; }
static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

extern "C" int64_t olmax_lmhead_distill_workspace_bytes(int64_t T, int32_t d, int32_t V) {
  if (T <= 0 || V <= 0) return 0;
  return up256(T * head_stride(V) * 4) + up256(T * head_stride(V) * 2) + olmax_distill_workspace_bytes(T);
}

extern "C" int32_t olmax_lmhead_distill(hipStream_t stream, const void* h, const void* W, const int32_t* top_ids, const float* top_logprobs, float* loss,
                                        void* dh, void* dW, void* workspace, int64_t workspace_bytes, int64_t T, int32_t d, int32_t V, int32_t k,
                                        int32_t tail, float temperature, float softcap, float dloss, int32_t dw_f32) {
  OLMAX_CHECK(h && W && top_ids && top_logprobs && loss && workspace, OLMAX_ERR_ARG, "olmax_lmhead_distill: null pointer");
  if (int rc = distill_check("olmax_lmhead_distill", T, V, k, tail, temperature, softcap)) return rc;
  OLMAX_CHECK(d > 0, OLMAX_ERR_SHAPE, "olmax_lmhead_distill: bad shape d=%d", d);
  OLMAX_CHECK(workspace_bytes >= olmax_lmhead_distill_workspace_bytes(T, d, V) && (((uintptr_t)workspace) & 255) == 0, OLMAX_ERR_WORKSPACE,
              "olmax_lmhead_distill: workspace needs %ld bytes, 256-byte aligned", (long)olmax_lmhead_distill_workspace_bytes(T, d, V));
  const int64_t ld = head_stride(V);
  const bf16 *hp = (const bf16*)h, *wp = (const bf16*)W;
  bf16* grads = (bf16*)((char*)workspace + up256(T * ld * 4));
  void* row_ws = (char*)grads + up256(T * ld * 2);
  if (int rc = olmax_gemm_padded(stream, hp, wp, workspace, nullptr, (int)T, V, d, d, d, ld, 0, true, true, true, false)) return rc;
  if (int rc = distill(stream, workspace, dh || dW ? grads : nullptr, top_ids, top_logprobs, loss, nullptr, row_ws, T, V, k, ld, ld, true, false, tail, temperature,
                       softcap, dloss, 0, (8 - V % 8) % 8))
    return rc;
  return olmax_lmhead_products(stream, grads, wp, hp, (bf16*)dh, dW, (int)T, d, V, ld, dw_f32 != 0, GemmScratch{workspace, std::min<int64_t>(T * ld * 4, PRODUCT_SCRATCH)});
}
