// Distillation from a teacher's top logits: the divergence of the student's softmax from what the teacher says about its k best tokens, with the gradient.
//
// p = softmax(z), z = cap(x) / temperature of the student (rows.h); the teacher gives k tokens id_j and numbers t_j of a row.
//   tail 0 (renormalize): q = softmax_k(t / temperature), the teacher's distribution over its k tokens alone (t: logits or log probabilities)
//     L = sum_j q_j (ln q_j - ln p_j)                     dL/dz_i = p_i - q_i
//   tail 1 (bucket): q_j = exp(t_j), and all other tokens are one event of probability r = 1 - sum q, s = sum of the others' p
//     L = sum_j q_j (ln q_j - ln p_j) + r ln(r / s)       dL/dz_i = p_i - q_i for the k tokens, p_i (1 - r / s) for the others
// s is summed over the others by themselves (1 - sum p_j would leave nothing of a small one): a bit of LDS per token says which those are.  Their sum is kept against their own largest
// score m' (or one at most 46 above it), S' = sum exp(z - m'): a student that is sure of the teacher's tokens leaves s far below what fp32 holds, but ln s = m' - m + ln S' - ln S
// and p_i r / s = exp(z_i - m') r / S' are ordinary numbers, and the only ones that still pull such a student back.
#include "rows.h"
#include <algorithm>
#include <mutex>
#include <type_traits>

using namespace rows;

namespace {

constexpr int MAX_TOP = 128;
constexpr int COUNTERS = 64;
constexpr int COUNT_IN_ROWS = 1024;  // up to so many rows each workgroup counts them itself
constexpr float LEAST_TAIL = 0x1p-20f;  // fp32 log probabilities leave less than this undetermined: a tail below it is none (a student without other tokens would lose infinitely by it)
constexpr int MAX_BITS = 1 << 20;    // tokens that a workgroup can keep a bit of (128 KB)
constexpr float FAR_BEHIND = 1e-20f;  // a sum of exponentials below it (46 nats) may have lost terms that count: one of 2^-24 of it is still 10^10 times fp32's least normal number.  Taking it
                                      // again costs a row two passes over its registers: 4096 x 100352 bf16 329 us where no row does, 371 where all do

// Rows that are not left out, in COUNTERS shares (a line of memory a row: one workgroup takes 10 us for 4096 rows, these 5).
__global__ __launch_bounds__(256) void distill_count_kernel(const int32_t* __restrict__ ids, int64_t T, int k, float* __restrict__ n) {
  __shared__ float red[4];
  float c = 0.f;
  for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < T; i += COUNTERS * 256) c += ids[i * k] >= 0 ? 1.f : 0.f;
  c = block_sum<4>(c, red);
  if (threadIdx.x == 0) n[blockIdx.x] = c;
}

// loss = sum of the rows' (/ rows that are not left out); one workgroup, whose loads of both are in flight together.
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ row_loss, const int32_t* __restrict__ ids, const float* __restrict__ counted, int64_t T, int k,
                                                           float* __restrict__ loss, int mean) {
  __shared__ float sums[16], counts[16];
  float s = 0.f, n = 0.f;
  const bool count = mean && !counted;
  for (int64_t i = threadIdx.x; i < T; i += blockDim.x) {
    const int id = count ? ids[i * k] : 0;
    s += row_loss[i];
    n += id >= 0 ? 1.f : 0.f;
  }
  s = wave_sum(s);
  n = wave_sum(n);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s, counts[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int waves = blockDim.x >> 6;
  s = wave_sum((int)threadIdx.x < waves ? sums[threadIdx.x] : 0.f);
  n = !mean ? 1.f : wave_sum(counted ? counted[threadIdx.x] : (int)threadIdx.x < waves ? counts[threadIdx.x] : 0.f);
  if (threadIdx.x == 0) *loss = n > 0.f ? s / n : 0.f;
}

struct Teacher {
  const int32_t* ids;
  const float* t;
  int k;
  float* x;  // the student's logits of the tokens, kept by a launch ahead of the one that may overwrite them; null: from the row
};

// What a workgroup knows of its row's teacher: tokens (-1: dropped), probabilities, their logarithms, the student's logits.  (In LDS, so that they take no registers while a
// row is held there.)
template <int NW> struct Lds {
  int id[MAX_TOP];
  float q[MAX_TOP], logq[MAX_TOP], x[MAX_TOP];
  float weight, rest, counted;
  Stat red[NW];
  float sums[NW];
};

// The teacher's side of a row, by one wave, two tokens a lane (with `bits` its tokens' too, element i at i + shift; they are zero).  Others read it behind a barrier.
template <typename T, bool BUCKET, int NW>
__device__ __forceinline__ void teacher_of(const Teacher& teacher, int64_t row, const T* zr, int V, float inv_tau, unsigned* bits, int shift, Lds<NW>& l) {
  const int lane = threadIdx.x & 63, k = teacher.k;
  int id[2];
  bool mine[2];
  float t[2], q[2], logq[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int j = lane + 64 * i;
    id[i] = j < k ? teacher.ids[row * k + j] : -1;
    t[i] = j < k ? teacher.t[row * k + j] : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
    mine[i] = id[i] >= 0 && id[i] < V;
    l.x[lane + 64 * i] = !mine[i] ? 0.f : teacher.x ? teacher.x[row * k + lane + 64 * i] : (float)zr[id[i]];
    if (!mine[i]) t[i] = -INFINITY;
  }
  for (int j = 0; j < min(k, 64); j++) {  // a token that is named again counts once
    const int other = __builtin_amdgcn_readlane(id[0], j);
    mine[0] = mine[0] && !(j < lane && id[0] == other);
    mine[1] = mine[1] && id[1] != other;
  }
  for (int j = 0; j < k - 64; j++) mine[1] = mine[1] && !(j < lane && id[1] == __builtin_amdgcn_readlane(id[1], j));
  float sum = 0.f, best = 0.f;
  if (!BUCKET) best = wave_max(fmaxf(mine[0] ? t[0] : -INFINITY, mine[1] ? t[1] : -INFINITY));
#pragma unroll
  for (int i = 0; i < 2; i++) {
    logq[i] = BUCKET ? t[i] : (t[i] - best) * inv_tau;
    q[i] = mine[i] && best > -INFINITY ? exp_of(logq[i]) : 0.f;
    sum += q[i];
  }
  sum = wave_sum(sum);
  const float r = BUCKET && 1.f - sum >= LEAST_TAIL ? 1.f - sum : 0.f;
  const float part = BUCKET ? 1.f : sum > 0.f ? 1.f / sum : 0.f, log_part = BUCKET ? 0.f : log_of(sum);
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int j = lane + 64 * i;
    l.id[j] = mine[i] ? id[i] : -1;
    l.q[j] = q[i] * part;
    l.logq[j] = logq[i] - log_part;
    if (BUCKET && bits && mine[i]) atomicOr(&bits[(id[i] + shift) >> 5], 1u << ((id[i] + shift) & 31));
  }
  if (lane == 0) l.weight = BUCKET ? sum + r : sum > 0.f ? 1.f : 0.f, l.rest = r;  // sum of all probabilities; 0: nothing to learn
}

// A row's loss from its statistics (BUCKET: of the other tokens alone), and what its gradient is made of: exp(z - m_out) * out dz/dx for the other tokens,
// (exp(z - m) * in - q * scale) dz/dx for the teacher's.  Every wave sums the tokens by itself.  m: the largest level of all, m_out: what the statistics are against.
struct Factors {
  float m, m_out, out, in, scale;
};
template <int CAP, bool BUCKET, int NW>
__device__ __forceinline__ Factors factors_of(const Stat& a, const Lds<NW>& l, const Scale& c, float scale, float* row_loss) {
  const int lane = threadIdx.x & 63;
  const float weight = l.weight, r = l.rest;
  Factors f;
  float most = a.m;
  if (BUCKET) {
    float own = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; i++) own = fmaxf(own, l.id[lane + 64 * i] >= 0 ? level<CAP>(l.x[lane + 64 * i], c) : -INFINITY);
    most = fmaxf(most, wave_max(own));
  }
  f.m = uniform(most == -INFINITY ? 0.f : most);
  f.m_out = uniform(a.ref());
  const float apart = !BUCKET ? 0.f : CAP ? a.m - f.m : behind<0>(a.m, c, f.m);  // of the two, in scores
  float d[2], inside = 0.f, loss = 0.f;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const bool mine = l.id[lane + 64 * i] >= 0;
    d[i] = behind<CAP>(l.x[lane + 64 * i], c, f.m);
    if (BUCKET && mine) inside += exp_of(d[i]);
  }
  const float sum = uniform(BUCKET ? __builtin_fmaf(a.s, exp_of(apart), wave_sum(inside)) : a.s);
  const bool none = sum == 0.f;  // no score above minus infinity: no distribution, nothing to learn from
  const float log_sum = log_of(sum);
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const float q = l.q[lane + 64 * i];
    if (q > 0.f) loss += q * (l.logq[lane + 64 * i] - (d[i] - log_sum));
  }
  loss = wave_sum(loss);
  if (BUCKET && r > 0.f) {  // r (ln r - ln s); a lead that has no room in fp32 (behind masks of the type's lowest value, at a temperature below 1) may have it times r
    const float lead = CAP || apart > -INFINITY || a.m == -INFINITY ? r * apart : (r * a.m - r * f.m) * c.unit;
    loss += r * (log_of(r) - (log_of(a.s) - log_sum)) - lead;
  }
  if (threadIdx.x == 0) *row_loss = none ? 0.f : loss;
  f.scale = none || weight == 0.f ? 0.f : scale;
  const float inv_sum = none ? 0.f : 1.f / sum;
  f.in = uniform(f.scale * weight * inv_sum);
  // (without others above minus infinity there is nothing to pull on)
  f.out = uniform(f.scale * (BUCKET ? weight * inv_sum * exp_of(apart) - (a.s > 0.f ? r / a.s : 0.f) : weight * inv_sum));
  return f;
}
template <int CAP> __device__ __forceinline__ float outside(float x, const Scale& c, const Factors& f) {
  return exp_behind<CAP>(x, c, f.m_out) * f.out * slope<CAP>(x, c);
}
template <int CAP> __device__ __forceinline__ float inside(float x, float q, const Scale& c, const Factors& f) {
  return (exp_behind<CAP>(x, c, f.m) * f.in - q * f.scale) * slope<CAP>(x, c);
}

// (past_cache) Held rows' gradients of more bytes than LAST_CACHE are stored past it, where rows that are being read leave them no room.  us, through it | past it, bf16:
// 4096 x 100352 346 | 329, with a product of the gradients behind it 1320 | 1290; 2048 x 100352 181 | 172, 862 | 874; 4000 x 50304 163 | 155, 604 | 577; fp32 4000 x 50304 313 | 303; nor are logits kept there that are read once, for the loss alone: 700 x 128256 fp32 69.7 | 65.1.
// Below it: 500 x 50304 32 | 28, with a product 234 | 261; fp32 500 x 100278 81 | 91.
struct RowArgs {
  Teacher teacher;
  float* row_loss;
  const float *drow, *n_counted;
  int64_t rows;
  int V;
  int64_t ld, ldd;
  float dloss;
  int mean, pad, past_cache;
};

// The number of rows that are not left out, by the second wave.
template <int NW> __device__ __forceinline__ void count_rows(const RowArgs& p, Lds<NW>& l) {
  float n = 0.f;
  if (p.n_counted) n = p.n_counted[threadIdx.x & 63];
  else
    for (int i = threadIdx.x & 63; i < p.rows; i += 64) n += p.teacher.ids[(int64_t)i * p.teacher.k] >= 0 ? 1.f : 0.f;
  n = wave_sum(n);
  if (threadIdx.x == 64) l.counted = n;
}
template <typename TO, int TH> __device__ __forceinline__ void write_zeros(TO* dr, const Cut& cutting, int v0, int v1, bool ends, int V, int pad) {
  constexpr int N = Vec<TO>::N;
  const float zero[N] = {};
  for (int v = v0 + threadIdx.x; v < v1; v += TH) *reinterpret_cast<u32x4*>(dr + cutting.head + v * N) = Vec<TO>::pack(zero);
  if (ends && (int)threadIdx.x < cutting.edges) dr[cutting.edge(threadIdx.x, V)] = (TO)0.f;
  if (ends && (int)threadIdx.x < pad) dr[V + threadIdx.x] = (TO)0.f;
}

// Rows that no workgroup holds, and few rows: two launches of shares of rows.  The first leaves statistics (BUCKET: sums of the other tokens) of each share, and the teacher's tokens'
// logits; or (part_stat null) the loss of whole rows, and there is no second.  700 x 128256 fp32: 60 us, 6.0 TB/s.
template <typename T, int CAP, bool BUCKET, int TH>
__global__ __launch_bounds__(TH) void distill_stats_kernel(const T* __restrict__ logits, const RowArgs p, const Scale c, Stat* __restrict__ part_stat, int parts) {
  constexpr int N = Vec<T>::N, UNROLL = 4, SPAN = TH * UNROLL;
  extern __shared__ unsigned bits[];  // BUCKET: of the teacher's tokens in the share, the row's single elements behind its vectors
  __shared__ Lds<TH / 64> l;
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts, tid = threadIdx.x, V = p.V;
  const int32_t* ids = p.teacher.ids + row * p.teacher.k;
  if (ids[0] < 0) {
    if (!part_stat && tid == 0) p.row_loss[row] = 0.f;
    return;
  }
  const T* zr = logits + row * p.ld;
  const Cut cutting = cut<T, N>(zr, V);
  const T* body = zr + cutting.head;
  const int per = (cutting.nvec + parts - 1) / parts;
  const int v0 = min(part * per, cutting.nvec), v1 = min(v0 + per, cutting.nvec);
  Raw<T, N> next[UNROLL];
  const bool once = !part_stat && p.past_cache;  // (no second launch reads them)
  auto fetch = [&](int at) {
    if (once) {  // (between barriers, or the compiler makes one load of both)
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < UNROLL; u++)
        if (at + u * TH + tid < v1) next[u].load_once(body + (int64_t)(at + u * TH + tid) * N);
      __builtin_amdgcn_sched_barrier(0);
    } else {
#pragma unroll
      for (int u = 0; u < UNROLL; u++)
        if (at + u * TH + tid < v1) next[u].load(body + (int64_t)(at + u * TH + tid) * N);
    }
  };
  fetch(v0);
  if (!part_stat && tid < 64) teacher_of<T, BUCKET, TH / 64>(p.teacher, row, zr, V, c.inv_tau, nullptr, 0, l);  // (beside the others' first loads)
  if (part_stat && part == 0 && tid < p.teacher.k) p.teacher.x[row * p.teacher.k + tid] = ids[tid] >= 0 && ids[tid] < V ? (float)zr[ids[tid]] : 0.f;
  if (BUCKET) {
    for (int i = tid; i < (per * N + 2 * N + 31) / 32; i += TH) bits[i] = 0;
    __syncthreads();
    if (tid < p.teacher.k) {
      const int id = ids[tid], in = id - cutting.head;
      int at = -1;
      if (id >= 0 && id < V) at = in < 0 ? per * N + id : in >= cutting.nvec * N ? per * N + id - cutting.nvec * N : in >= v0 * N && in < v1 * N ? in - v0 * N : -1;
      if (at >= 0) atomicOr(&bits[at >> 5], 1u << (at & 31));
    }
    __syncthreads();
  }
  const unsigned char* byte_of = reinterpret_cast<const unsigned char*>(bits);
  Stat a = Stat::none();
  if (part == 0 && tid < cutting.edges) {
    const float x = (float)zr[cutting.edge(tid, V)];
    const int at = per * N + tid;
    if (!(BUCKET && (bits[at >> 5] >> (at & 31) & 1))) {
      if (CAP || x > -INFINITY) a.m = level<CAP>(x, c);
      a.s = exp_behind<CAP>(x, c, a.ref());
    }
  }
  for (int at = v0; at < v1; at += SPAN) {
    Raw<T, N> now[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) now[u] = next[u];
    fetch(at + SPAN);
    float most = -INFINITY;
    unsigned in[UNROLL];  // BUCKET: which elements are the teacher's
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const int v = at + u * TH + tid, b = v - v0;
      if (v >= v1) continue;
      float x[N];
      now[u].unpack(x);
      if (BUCKET) {
        in[u] = N == 8 ? (unsigned)byte_of[b] : (byte_of[b >> 1] >> (b & 1) * 4) & 15u;
        if (in[u])
#pragma unroll
          for (int e = 0; e < N; e++) x[e] = in[u] >> e & 1 ? -INFINITY : x[e];
      }
#pragma unroll
      for (int e = 0; e < N; e++) most = fmaxf(most, x[e]);
    }
    const float top = level<CAP>(most, c);
    if (at + tid < v1 && top > a.m) a.raise(top, c.unit);
    const float ref = a.ref();
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const int v = at + u * TH + tid;
      if (v >= v1) continue;
      float x[N];
      now[u].unpack(x);
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = exp_behind<CAP>(x[e], c, ref);
      if (BUCKET && in[u])
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = in[u] >> e & 1 ? 0.f : x[e];
#pragma unroll
      for (int w = N / 2; w > 0; w >>= 1)
#pragma unroll
        for (int e = 0; e < w; e++) x[e] += x[e + w];
      a.s += x[0];
    }
  }
  a = block_join<TH / 64>(a, l.red, c.unit);
  if (part_stat && tid == 0) part_stat[blockIdx.x] = a;
  if (!part_stat) factors_of<CAP, BUCKET, TH / 64>(a, l, c, 0.f, p.row_loss + row);
}

// The second joins them (every workgroup for itself), writes the loss, and the gradient of one of `shares` shares of the row.
template <typename T, typename TO, int CAP, bool BUCKET>
__global__ __launch_bounds__(256) void distill_grads_kernel(const T* __restrict__ logits, TO* __restrict__ dlogits, const RowArgs p, const Scale c,
                                                            const Stat* __restrict__ part_stat, int parts, int shares) {
  constexpr int N = Vec<TO>::N, TH = 256, NW = TH / 64;
  __shared__ Lds<NW> l;
  __shared__ float unused;
  const int64_t row = blockIdx.x / shares;
  const int share = blockIdx.x % shares, tid = threadIdx.x, V = p.V;
  const T* zr = logits + row * p.ld;
  TO* dr = dlogits ? dlogits + row * p.ldd : nullptr;
  const Cut cutting = dr ? cut<TO, N>(dr, V) : cut<T, N>(zr, V);
  const int per = (cutting.nvec + shares - 1) / shares;
  const int v0 = min(share * per, cutting.nvec), v1 = min(v0 + per, cutting.nvec);
  if (p.teacher.ids[row * p.teacher.k] < 0) {  // left out
    if (share == 0 && tid == 0) p.row_loss[row] = 0.f;
    if (dr) write_zeros<TO, TH>(dr, cutting, v0, v1, share == 0, V, p.pad);
    return;
  }
  if (tid < 64) {
    Stat a = Stat::none();
    if (tid < parts) a = part_stat[row * parts + tid];
    a = block_join<1>(a, nullptr, c.unit);
    if (tid == 0) l.red[0] = a;
    teacher_of<T, BUCKET, NW>(p.teacher, row, zr, V, c.inv_tau, nullptr, 0, l);
  }
  if (tid >> 6 == 1 && dr && p.mean) count_rows(p, l);
  __syncthreads();
  float scale = 0.f;
  if (dr) scale = uniform(p.dloss * (p.drow ? p.drow[row] : 1.f) / (p.mean ? l.counted : 1.f));
  const Factors f = factors_of<CAP, BUCKET, NW>(l.red[0], l, c, scale, share == 0 ? p.row_loss + row : &unused);
  if (!dr) return;
  for (int v = v0 + tid; v < v1; v += TH) {
    const int i = cutting.head + v * N;
    Raw<T, N> w;
    w.load(zr + i);
    float x[N];
    w.unpack(x);
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = outside<CAP>(x[e], c, f);
    *reinterpret_cast<u32x4*>(dr + i) = Vec<TO>::pack(x);
  }
  if (share == 0 && tid < cutting.edges) {
    const int i = cutting.edge(tid, V);
    dr[i] = (TO)outside<CAP>((float)zr[i], c, f);
  }
  if (share == 0 && tid < p.pad) dr[V + tid] = (TO)0.f;
  __syncthreads();  // behind the vectors that hold them
  if (tid < MAX_TOP && l.id[tid] >= 0) {
    const int in = l.id[tid] - cutting.head;
    if (in >= 0 && in < cutting.nvec * N ? in >= v0 * N && in < v1 * N : share == 0) dr[l.id[tid]] = (TO)inside<CAP>(l.x[tid], l.q[tid], c, f);
  }
}

// One workgroup a row, of which a thread keeps HELD vectors in registers: statistics and the loss, then the gradient of all tokens, then the k tokens' own.
// Each logit is read once and its gradient written once, and no exponential is kept: those of the gradient are taken again.  4096 x 100352 bf16 to bf16: 329 us with the count and the sum, 5.0 TB/s (a copy:
// 5.2), the vector unit busy for 60 %: the rows of a CU, of which registers hold two, read and write in turns that overlap only with each other's.
template <typename T, typename TO, int CAP, bool BUCKET, int TH, int HELD>
__global__ __launch_bounds__(TH, 4) void distill_rows_kernel(const T* __restrict__ logits, TO* __restrict__ dlogits, const RowArgs p, const Scale c) {
  constexpr int N = Vec<TO>::N, NW = TH / 64;
  extern __shared__ unsigned bits[];  // BUCKET
  __shared__ Lds<NW> l;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, V = p.V;
  const T* zr = logits + row * p.ld;
  TO* dr = dlogits ? dlogits + row * p.ldd : nullptr;
  const Cut cutting = dr ? cut<TO, N>(dr, V) : cut<T, N>(zr, V);
  if (p.teacher.ids[row * p.teacher.k] < 0) {  // left out
    if (tid == 0) p.row_loss[row] = 0.f;
    if (dr) write_zeros<TO, TH>(dr, cutting, 0, cutting.nvec, true, V, p.pad);
    return;
  }
  const T* body = zr + cutting.head;
  Raw<T, N> held[HELD];
#pragma unroll
  for (int i = 0; i < HELD; i++)
    if (i * TH + tid < cutting.nvec) held[i].load_once(body + (int64_t)(i * TH + tid) * N);
  const int shift = (N - cutting.head) & (N - 1);
  if (BUCKET) {
    for (int i = tid; i < (V + 8 + 31) / 32; i += TH) bits[i] = 0;
    __syncthreads();
  }
  if (tid < 64) teacher_of<T, BUCKET, NW>(p.teacher, row, zr, V, c.inv_tau, bits, shift, l);
  if (tid >> 6 == 1 && dr && p.mean) count_rows(p, l);
  if (BUCKET) __syncthreads();

  // ---- largest score, sum of exponentials (BUCKET: of the other tokens)
  const unsigned char* byte_of = reinterpret_cast<const unsigned char*>(bits);
  auto hide = [&](float* x, int first, float by) {  // those elements of vector first + tid that are the teacher's; first is even
    const int at = tid + (cutting.head ? 1 : 0);
    const unsigned in = N == 8 ? (unsigned)byte_of[at + first] : (byte_of[(at >> 1) + (first >> 1)] >> (at & 1) * 4) & 15u;
    if (in)
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = in >> e & 1 ? by : x[e];
  };
  auto summed = [&](const Raw<T, N>& w, int first, float ref) {  // of vector first + tid
    float x[N];
    w.unpack(x);
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = exp_behind<CAP>(x[e], c, ref);
    if (BUCKET) hide(x, first, 0.f);
#pragma unroll
    for (int w2 = N / 2; w2 > 0; w2 >>= 1)
#pragma unroll
      for (int e = 0; e < w2; e++) x[e] += x[e + w2];
    return x[0];
  };
  auto largest = [&](const Raw<T, N>& w, float most) {
    float x[N];
    w.unpack(x);
#pragma unroll
    for (int e = 0; e < N; e++) most = fmaxf(most, x[e]);
    return most;
  };
  // each pass unpacks a vector when its turn comes: hidden from the compiler, which otherwise keeps all unpacked logits of a pass for the next
  auto keep = [](Raw<T, N>& w) {
#pragma unroll
    for (int i = 0; i < Raw<T, N>::W; i++) asm volatile("" : "+v"(w.w[i]));
    __builtin_amdgcn_sched_barrier(0);
  };
  // the row's single elements, one to a thread, as max, sum and gradient
  auto edge_value = [&](int* at) {
    *at = cutting.edge(tid, V);
    return (float)zr[*at];
  };
  auto is_other = [&](int at) { return !(BUCKET && (bits[(at + shift) >> 5] >> ((at + shift) & 31) & 1)); };
  const bool has_edge = tid < cutting.edges;
  int edge;
  float most = -INFINITY;
  if (has_edge) most = fmaxf(most, edge_value(&edge));
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    keep(held[i]);
    if (i * TH + tid < cutting.nvec) most = largest(held[i], most);
  }
  most = uniform(block_reduce<NW, true>(most, l.sums));
  Stat a = Stat::none();
  auto sum_behind = [&](float most) {
    a.m = -INFINITY;
    if (CAP || most > -INFINITY) a.m = level<CAP>(most, c);
    const float ref = a.ref();
    float sum = 0.f;
    if (has_edge) {
      const float x = edge_value(&edge);
      if (is_other(edge)) sum = exp_behind<CAP>(x, c, ref);
    }
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      keep(held[i]);
      if (i * TH + tid < cutting.nvec) sum += summed(held[i], i * TH, ref);
    }
    a.s = uniform(block_reduce<NW, false>(sum, l.sums));
  };
  sum_behind(most);
  if (BUCKET && a.s < FAR_BEHIND) {  // (the same for all threads) the teacher's tokens lead by far, so that the others' sum is taken again, against their own largest
    most = -INFINITY;
    if (has_edge) {
      const float x = edge_value(&edge);
      if (is_other(edge)) most = fmaxf(most, x);
    }
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      keep(held[i]);
      if (i * TH + tid < cutting.nvec) {
        float x[N];
        held[i].unpack(x);
        hide(x, i * TH, -INFINITY);
#pragma unroll
        for (int e = 0; e < N; e++) most = fmaxf(most, x[e]);
      }
    }
    sum_behind(uniform(block_reduce<NW, true>(most, l.sums)));
  }
  // (a barrier of the reduction lies between the teacher's wave and here)
  float scale = 0.f;
  if (dr) scale = uniform(p.dloss * (p.drow ? p.drow[row] : 1.f) / (p.mean ? l.counted : 1.f));
  const Factors f = factors_of<CAP, BUCKET, NW>(a, l, c, scale, p.row_loss + row);
  if (!dr) return;

  // ---- the gradient, in place allowed (every thread reads what it writes, the k logits are in LDS)
  auto write = [&](const Raw<T, N>& w, int v) {
    float x[N];
    w.unpack(x);
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = outside<CAP>(x[e], c, f);
    u32x4* to = reinterpret_cast<u32x4*>(dr + cutting.head + v * N);
    const u32x4 all = Vec<TO>::pack(x);
    if (p.past_cache) {  // (between barriers, or the compiler makes one store of both)
      __builtin_amdgcn_sched_barrier(0);
      __builtin_nontemporal_store(all, to);
      __builtin_amdgcn_sched_barrier(0);
    } else {
      *to = all;
    }
  };
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    int at = tid;
    asm volatile("" : "+v"(at));  // (the offsets, which would be kept from the loads, are computed again)
    keep(held[i]);
    if (i * TH + at < cutting.nvec) write(held[i], i * TH + at);
  }
  if (has_edge) {
    const float x = edge_value(&edge);
    dr[edge] = (TO)outside<CAP>(x, c, f);
  }
  if (tid < p.pad) dr[V + tid] = (TO)0.f;
  __syncthreads();  // behind the vectors that hold them
  if (tid < MAX_TOP && l.id[tid] >= 0) dr[l.id[tid]] = (TO)inside<CAP>(l.x[tid], l.q[tid], c, f);
}

}  // namespace

// How a call runs: held = vectors and threads that hold a row, or 0 and the shares of a row for statistics and gradient.
// The fewest threads that hold the row, which is then read once; shares are read twice, by two launches, and keep more CUs busy where rows are few and long.
// us with the gradient, shares | held, bf16: 1 x 128256 15.9 | 23.6, 64 x 128256 24.2 | 29.1, 250 x 128256 43 | 36, 800 x 128256 152 | 125, 64 x 50304 19.0 | 17.1; fp32 800 x 50304
// 121 | 71.  The loss alone, streamed | held: 1600 x 128256 88 | 138, 400 x 128256 26 | 40, 128 x 50304 15.3 | 12.9.
struct Form {
  int threads, held, parts, shares;
};
static Form form_of(int64_t T, int V, bool logits_f32, bool grads_f32, bool grad) {
  const int vecs = V / (grads_f32 ? 4 : 8), reads = V / (logits_f32 ? 4 : 8);
  const bool wide = logits_f32 && !grads_f32;  // a vector takes eight registers
  const int most = wide ? 13 : grads_f32 ? 25 : 20;
  if (vecs <= 256 * 8) return {256, 8, 1, 1};
  // the loss alone: a row has to be read once anyway, and 256 threads that stream it leave a CU to more rows
  const bool hold = grad ? T > 128 || vecs <= 512 * 25 : T < 400 && vecs <= 512 * 25;
  if (hold && vecs <= 512 * (wide ? 13 : 25)) return {512, wide ? 13 : 25, 1, 1};
  if (hold && vecs <= 1024 * most) return {1024, most, 1, 1};
  const int64_t parts = T > 256 ? 1 : std::min<int64_t>(std::min<int64_t>(reads / 1024, 1024 / T), 32);
  const int64_t shares = grad ? std::min<int64_t>(vecs / 2048, 4096 / T) : 1;
  return {0, 0, (int)std::max<int64_t>(1, parts), (int)std::max<int64_t>(1, shares)};
}

// Workspace: T floats (row losses), the shares of the number of counted rows, statistics of the shares of rows, the tokens' logits.
static int64_t stats_at(int64_t T) { return ((T * 4 + 15) / 16) * 16 + COUNTERS * 4; }
extern "C" int64_t olmax_distill_workspace_bytes(int64_t T, int32_t V, int32_t k, int32_t logits_f32) {
  if (T <= 0 || V <= 0 || k <= 0) return 0;
  int64_t parts = 1;
  for (int grad = 0; grad < 4; grad++) parts = std::max<int64_t>(parts, form_of(T, V, logits_f32 != 0, logits_f32 && grad < 2, grad & 1).parts);
  return stats_at(T) + T * (parts * (int64_t)sizeof(Stat) + k * 4ll);
}

static int distill_check(const char* name, int64_t T, int32_t V, int32_t k, int32_t tail, float temperature, float softcap) {
  OLMAX_CHECK(T > 0 && V > 0 && V < (1 << 30) && T < (1LL << 24), OLMAX_ERR_SHAPE, "%s: bad shape T=%ld V=%d", name, (long)T, V);
  OLMAX_CHECK(k >= 1 && k <= MAX_TOP, OLMAX_ERR_ARG, "%s: 1 to %d tokens of the teacher a row (got %d)", name, MAX_TOP, k);
  OLMAX_CHECK(tail == 0 || (tail == 1 && V <= MAX_BITS - 32), OLMAX_ERR_ARG, "%s: tail must be 0 (renormalize) or 1 (bucket, up to %d logits)", name, MAX_BITS - 32);
  OLMAX_CHECK(takes(temperature, softcap), OLMAX_ERR_ARG, "%s: temperature within 1e-6 and 1e6, softcap 0 or within 1e-30 and 1e30", name);
  return OLMAX_OK;
}

// grads_bf16: the gradient of fp32 logits as bf16 (the LM head's products take it); pad: zeros behind each of its rows
static int distill(hipStream_t stream, const void* logits, void* dlogits, const int32_t* ids, const float* t, float* loss, const float* dloss_rows,
                   void* workspace, int64_t T, int32_t V, int32_t k, int64_t ld, int64_t ldd, bool logits_f32, bool grads_f32, int32_t tail, float temperature,
                   float softcap, float dloss, int32_t reduction, int pad) {
  const Scale c = scale_of(temperature, softcap);
  float* row_loss = reduction == 2 ? loss : (float*)workspace;
  float* n = nullptr;
  if (reduction == 0 && T > COUNT_IN_ROWS) {
    n = (float*)((char*)workspace + ((T * 4 + 15) / 16) * 16);
    hipLaunchKernelGGL(distill_count_kernel, dim3(COUNTERS), dim3(256), 0, stream, ids, T, k, n);
  }
  const Form form = form_of(T, V, logits_f32, grads_f32, dlogits != nullptr);
  OLMAX_CHECK(T * std::max(form.parts, form.shares) < (1LL << 31), OLMAX_ERR_SHAPE, "olmax_distill: T=%ld rows of V=%d are too many", (long)T, V);
  Stat* part_stat = (Stat*)((char*)workspace + stats_at(T));
  const bool alone = form.parts == 1 && !dlogits;
  const RowArgs args{{ids, t, k, form.threads || alone ? nullptr : (float*)(part_stat + T * form.parts)}, row_loss, dloss_rows, n, T, V, ld, ldd, dloss, (int)(reduction == 0), pad, (int)(T * V * (dlogits && !grads_f32 || !logits_f32 ? 2 : 4) > LAST_CACHE)};
#define LAUNCH(K, GRID, THV, LDS, ...)                                                                                                          \
  do {                                                                                                                                          \
    auto kern = K;                                                                                                                              \
    static std::once_flag attr_once; /* per instantiation */                                                                                    \
    std::call_once(attr_once, [&] { (void)hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, MAX_BITS / 8); }); \
    hipLaunchKernelGGL(kern, dim3((unsigned)(GRID)), dim3(THV), LDS, stream, (const TY*)logits, __VA_ARGS__);                                   \
  } while (0)
#define HELD(THV, HELDV) LAUNCH((distill_rows_kernel<TY, TO, CAP, BUCKET, THV, (HELDV)>), T, THV, BUCKET ? (V + 8 + 31) / 32 * 4 : 0, (TO*)dlogits, args, c)
  auto go = [&](auto in, auto out, auto capped, auto bucket) {
    using TY = decltype(in);
    using TO = decltype(out);
    constexpr int CAP = decltype(capped)::value;
    constexpr bool BUCKET = decltype(bucket)::value, WIDE = sizeof(TY) != sizeof(TO);
    if (form.threads == 256) HELD(256, 8);
    else if (form.threads == 512) HELD(512, WIDE ? 13 : 25);
    else if (form.threads == 1024) HELD(1024, WIDE ? 13 : sizeof(TO) == 2 ? 20 : 25);
    else {
      constexpr int N = Vec<TY>::N;
      const size_t lds = BUCKET ? ((V / N + form.parts) / form.parts * N + 2 * N + 31) / 32 * 4 : 0;
      Stat* stat = alone ? nullptr : part_stat;
      if (form.parts > 1) LAUNCH((distill_stats_kernel<TY, CAP, BUCKET, 256>), T * form.parts, 256, lds, args, c, stat, form.parts);
      else LAUNCH((distill_stats_kernel<TY, CAP, BUCKET, 512>), T, 512, lds, args, c, stat, 1);
      if (!alone) LAUNCH((distill_grads_kernel<TY, TO, CAP, BUCKET>), T * form.shares, 256, 0, (TO*)dlogits, args, c, (const Stat*)part_stat, form.parts, form.shares);
    }
  };
#undef HELD
#undef LAUNCH
  auto kind = [&](auto in, auto out) {
    auto tails = [&](auto capped) { tail ? go(in, out, capped, std::true_type()) : go(in, out, capped, std::false_type()); };
    if (c.kind == 0) tails(std::integral_constant<int, 0>());
    else if (c.kind == 1) tails(std::integral_constant<int, 1>());
    else tails(std::integral_constant<int, 2>());
  };
  if (logits_f32 && grads_f32) kind(0.f, 0.f);
  else if (logits_f32) kind(0.f, bf16());
  else kind(bf16(), bf16());
  if (reduction != 2) hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(T <= 256 ? 256 : 1024), 0, stream, (const float*)row_loss, ids, (const float*)n, T, k, loss, (int)(reduction == 0));
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
  OLMAX_CHECK(!overlap(logits, ld, dlogits, ldd, T, V, logits_f32 ? 4 : 2), OLMAX_ERR_ARG, "olmax_distill: the gradient overlaps the logits, but is not in their place");
  OLMAX_CHECK(workspace_bytes >= olmax_distill_workspace_bytes(T, V, k, logits_f32) && aligned16(workspace), OLMAX_ERR_WORKSPACE, "olmax_distill: workspace needs %ld bytes, 16-byte aligned",
              (long)olmax_distill_workspace_bytes(T, V, k, logits_f32));
  return distill(stream, logits, dlogits, top_ids, top_logprobs, loss, dloss_rows, workspace, T, V, k, ld, ldd, logits_f32 != 0, logits_f32 != 0, tail,
                 temperature, softcap, dloss, reduction, 0);
}

// ---- with the LM head's product, forward and backward in one call.  Logits fp32 in the workspace, their gradient bf16 behind them.
static int64_t head_stride(int32_t V) { return ((int64_t)V + 63) / 64 * 64; }
static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

struct HeadPlan {
  bool few;       // tokens fewer than a tile has rows: the gradients' products pad them, and the logits' those of more than 64
  bool in64;      // gradients of 64 tokens
  int64_t rows, ld, grads_at, rows_at, h_at, dh_at, bytes;
};
static HeadPlan head_plan(int64_t T, int32_t d, int32_t V, int32_t k) {
  HeadPlan p;
  p.few = olmax_lmhead_pads(T, d, V);
  p.in64 = olmax_lmhead_pads_64(T, d, V);
  p.rows = p.few && T > 64 ? 256 : T;
  p.ld = head_stride(V);
  p.grads_at = up256(std::max<int64_t>(p.rows * p.ld * 4, p.few ? PRODUCT_SCRATCH : 0));
  p.rows_at = p.grads_at + up256((p.few ? 256 : p.in64 ? 64 : T) * p.ld * 2);
  p.h_at = p.rows_at + up256(olmax_distill_workspace_bytes(T, V, k, 1));
  p.dh_at = p.h_at + (p.few || p.in64 ? up256((p.few ? 256ll : 64ll) * d * 2) : 0);
  p.bytes = p.dh_at + (p.few || p.in64 ? up256((p.few ? 256ll : 64ll) * d * 2) : 0);
  return p;
}
extern "C" int64_t olmax_lmhead_distill_workspace_bytes(int64_t T, int32_t d, int32_t V, int32_t k) {
  return T <= 0 || V <= 0 || d <= 0 || k <= 0 || T >= (1 << 24) ? 0 : head_plan(T, d, V, k).bytes;
}

int olmax_lmhead_distill_check(const HeadDistill& a) {
  OLMAX_CHECK(a.h && a.W && a.top_ids && a.top_logprobs && a.loss && a.workspace, OLMAX_ERR_ARG, "olmax_lmhead_distill: null pointer");
  if (int rc = distill_check("olmax_lmhead_distill", a.T, a.V, a.k, a.tail, a.temperature, a.softcap)) return rc;
  OLMAX_CHECK(a.d > 0, OLMAX_ERR_SHAPE, "olmax_lmhead_distill: bad shape d=%d", a.d);
  OLMAX_CHECK(aligned16(a.h) && aligned16(a.W) && aligned16(a.dh), OLMAX_ERR_ALIGN, "olmax_lmhead_distill: h, W and dh must be 16-byte aligned");
  const int64_t need = head_plan(a.T, a.d, a.V, a.k).bytes;
  OLMAX_CHECK(a.workspace_bytes >= need && (((uintptr_t)a.workspace) & 255) == 0, OLMAX_ERR_WORKSPACE, "olmax_lmhead_distill: workspace needs %ld bytes, 256-byte aligned", (long)need);
  return OLMAX_OK;
}

extern "C" int32_t olmax_lmhead_distill(hipStream_t stream, const void* h, const void* W, const int32_t* top_ids, const float* top_logprobs, float* loss,
                                        void* dh, void* dW, void* workspace, int64_t workspace_bytes, int64_t T, int32_t d, int32_t V, int32_t k,
                                        int32_t tail, float temperature, float softcap, float dloss, int32_t dw_f32) {
  if (int rc = olmax_lmhead_distill_check({h, W, top_ids, top_logprobs, loss, dh, workspace, workspace_bytes, T, d, V, k, tail, temperature, softcap})) return rc;
  const HeadPlan p = head_plan(T, d, V, k);
  const bf16 *hp = (const bf16*)h, *wp = (const bf16*)W;
  char* ws = (char*)workspace;
  bf16 *grads = (bf16*)(ws + p.grads_at), *h_pad = (bf16*)(ws + p.h_at);
  const bool grad = dh || dW;
  const int pad = (8 - V % 8) % 8;
  if (p.few && (dW || p.rows > T)) olmax_pad_rows(stream, hp, h_pad, T, 256, d);
  if (int rc = olmax_gemm_padded(stream, p.rows > T ? h_pad : hp, wp, workspace, nullptr, (int)p.rows, V, d, d, d, p.ld, 0, true, true, true, false)) return rc;
  if (int rc = distill(stream, workspace, grad ? grads : nullptr, top_ids, top_logprobs, loss, nullptr, ws + p.rows_at, T, V, k, p.ld, p.ld, true, false, tail, temperature, softcap,
                       dloss, 0, pad))
    return rc;
  const GemmScratch scratch{workspace, std::min(p.grads_at, PRODUCT_SCRATCH)};  // (the logits are done with)
  if (p.in64 && dW) olmax_pad_rows(stream, hp, h_pad, T, 64, d);
  else if (!p.few) return olmax_lmhead_products(stream, grads, wp, hp, (bf16*)dh, dW, (int)T, d, V, p.ld, dw_f32 != 0, scratch);
  if (dW) olmax_zero_rows(stream, grads, T, 64, V + pad, p.ld);
  return olmax_lmhead_products_few(stream, grads, wp, hp, h_pad, (bf16*)dh, dW, (int)T, d, V, p.ld, dw_f32 != 0, (bf16*)(ws + p.dh_at), p.few ? 256 : 64, scratch);
}
