// Log probabilities of given tokens, the entropy of their distributions and the most likely alternatives, with the gradient.
//
// z = cap(x) / temperature (rows.h), p = softmax(z):  logprob = z[target] - m - ln S,  entropy = ln S - sum p (z - m),
// alternatives = the `top` largest logits, in order, ties to the lowest index.
#include "rows.h"
#include <type_traits>
#include <algorithm>

using namespace rows;

namespace {

constexpr int GROUPS = 256;   // of threads whose largest logits bound the alternatives
constexpr int UNROLL = 4;     // vectors of a thread that are in flight, and reduced against one maximum
constexpr int MAX_TOP = 128;
constexpr int CAND = 1024;    // candidates for the alternatives that a workgroup can hold
constexpr int JOINED = 2048;  // of all parts of a row

// Rises with the value; -0 is 0.
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
constexpr unsigned KEY_NEG_INF = 0x007fffffu;
// A candidate: larger for a larger value, and among equal ones for a lower index; 0: none.
__device__ __forceinline__ uint64_t entry_of(unsigned key, int index) { return ((uint64_t)key << 32) | (0xffffffffu - (unsigned)index); }
__device__ __forceinline__ int index_of(uint64_t e) { return (int)(0xffffffffu - (unsigned)e); }

template <int TH> struct Lds {
  alignas(16) unsigned best[GROUPS];  // key of the largest of each group of threads
  uint64_t cand[CAND];
  unsigned hist[256];
  Stat red[TH / 64];
  int n, sums[TH / 64];
};

// A lower bound of the k-th largest value that the workgroup has seen, from the largest of each group of threads: at least k values are not below the k-th
// largest of those.  Found on the upper 16 bits of the keys, by bits: each wave counts all groups, four a lane.  *seen = *noted as it is between two barriers, the same
// for all threads (behind the second one of them may already note more).
template <int TH>
__device__ __forceinline__ unsigned kth_best(unsigned* best, unsigned own, int k, const int* noted, int* seen) {
  static_assert(TH == GROUPS || TH == 2 * GROUPS || TH == 4 * GROUPS, "up to four threads to a group");
  if (TH > GROUPS) own = max(own, (unsigned)__shfl_xor((int)own, 1, 64));
  if (TH > 2 * GROUPS) own = max(own, (unsigned)__shfl_xor((int)own, 2, 64));
  __syncthreads();
  if (noted) *seen = *noted;
  if ((threadIdx.x & (TH / GROUPS - 1)) == 0) best[threadIdx.x / (TH / GROUPS)] = own;
  __syncthreads();
  const u32x4 q = *reinterpret_cast<const u32x4*>(best + (threadIdx.x & 63) * 4);
  unsigned at = 0;
#pragma unroll
  for (int bit = 15; bit >= 0; bit--) {
    const unsigned tried = at | (1u << bit);
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) n += __popcll(__ballot((q[j] >> 16) >= tried));
    if (n >= k) at = tried;
  }
  return max(at << 16, KEY_NEG_INF);
}

// The exact way, for rows with more values that tie at the bound than there is room: the k largest of elements [lo, hi) above minus infinity go
// to cand, in any order; returns how many.  The k-th largest key by four passes of 8 bits, then all above it, then as many equal ones as are
// missing, from the lowest index on.
template <typename T, int TH>
__device__ int select_exact(const T* zr, int lo, int hi, int k, Lds<TH>& l) {
  unsigned at = 0;
  int need = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) l.hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = lo + threadIdx.x; i < hi; i += TH) {
      const float x = (float)zr[i];
      if (!(x > -INFINITY)) continue;
      const unsigned key = key_of(x);
      if (shift == 24 || (key >> (shift + 8)) == (at >> (shift + 8))) atomicAdd(&l.hist[(key >> shift) & 255], 1u);
    }
    __syncthreads();
    int b = 255, above = 0;
    for (; b > 0; b--) {
      const int n = (int)l.hist[b];
      if (above + n >= need) break;
      above += n;
    }
    need -= above;
    at |= (unsigned)b << shift;
  }
  __syncthreads();
  if (threadIdx.x == 0) l.n = 0;
  __syncthreads();
  for (int i = lo + threadIdx.x; i < hi; i += TH) {
    const float x = (float)zr[i];
    if (x > -INFINITY && key_of(x) > at) l.cand[atomicAdd(&l.n, 1)] = entry_of(key_of(x), i);
  }
  __syncthreads();
  const int above = l.n;
  int got = 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int base = lo; base < hi && got < need; base += TH) {
    const int i = base + threadIdx.x;
    const float x = i < hi ? (float)zr[i] : -INFINITY;
    const bool eq = x > -INFINITY && key_of(x) == at;
    const uint64_t votes = __ballot(eq);
    __syncthreads();
    if (lane == 0) l.sums[wave] = __popcll(votes);
    __syncthreads();
    int before = got + __popcll(votes & ((1ull << lane) - 1));
    for (int w = 0; w < wave; w++) before += l.sums[w];
    if (eq && before < need) l.cand[above + before] = entry_of(at, i);
    for (int w = 0; w < TH / 64; w++) got += l.sums[w];
  }
  __syncthreads();
  return above + min(got, need);
}

// Leaves of cand[0 .. n) those whose key is at least `bound`, in any order, and returns how many.  Each thread holds its share meanwhile.
template <int ROOM, int TH>
__device__ __forceinline__ int narrow(uint64_t* cand, int n, unsigned bound, int* counter) {
  uint64_t own[ROOM / TH];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ROOM / TH; i++) {
    const int at = i * TH + threadIdx.x;
    own[i] = at < n ? cand[at] : 0;
  }
  if (threadIdx.x == 0) *counter = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ROOM / TH; i++)
    if (own[i] && (unsigned)(own[i] >> 32) >= bound) cand[atomicAdd(counter, 1)] = own[i];
  __syncthreads();
  return *counter;
}

// emit(rank, entry) for the k largest of cand[0 .. n): an entry's rank is the number of larger ones (all are different).  Room for a multiple of 8; eight are read at a
// time (one by one 128 of them take 5 us).
template <int TH, typename F>
__device__ __forceinline__ void ranked(uint64_t* cand, int n, int k, F emit) {
  if (threadIdx.x < 8 && (n & 7) && (n & ~7) + (int)threadIdx.x >= n) cand[(n & ~7) + threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += TH) {
    const uint64_t e = cand[i];
    int rank = 0;
    for (int j = 0; j < n; j += 8) {
      uint64_t o[8];
#pragma unroll
      for (int u = 0; u < 8; u++) o[u] = cand[j + u];
#pragma unroll
      for (int u = 0; u < 8; u++) rank += o[u] > e;
    }
    if (rank < k) emit(rank, e);
  }
}

// What a row's outputs are written from.
struct Out {
  float *logprobs, *entropy, *stats, *top_logprobs;  // logprobs and the top ones may be null
  int32_t* top_ids;
};
__device__ __forceinline__ void write_skipped(const Out& o, int64_t row, int k) {
  if (threadIdx.x == 0) {
    if (o.logprobs) o.logprobs[row] = 0.f;
    o.entropy[row] = 0.f;
  }
  if (threadIdx.x < 3) o.stats[row * 3 + threadIdx.x] = 0.f;
  if (o.top_ids && (int)threadIdx.x < k) {
    o.top_ids[row * k + threadIdx.x] = -1;
    o.top_logprobs[row * k + threadIdx.x] = -INFINITY;
  }
}
// a: statistics of the whole row, x: the target's logit, if there is one.  A row without a score above minus infinity has no distribution: log probabilities of minus
// infinity, entropy 0.  By one thread.
template <int CAP>
__device__ __forceinline__ void write_row(const Out& o, int64_t row, bool has_target, float x, const Scale& c, const Stat& a) {
  const bool none = a.s == 0.f;
  const float log_sum = log_of(a.s), entropy = none ? 0.f : log_sum - a.t / a.s;
  if (o.logprobs) o.logprobs[row] = !has_target ? 0.f : none ? -INFINITY : behind<CAP>(x, c, a.m) - log_sum;
  o.entropy[row] = entropy;
  // the level as a score, and what its rounding leaves in the logarithm
  const float m = CAP ? a.m : a.m * c.inv_tau, left = CAP || __builtin_isinf(m) ? 0.f : __builtin_fmaf(a.m, c.inv_tau, -m);
  o.stats[row * 3] = m;
  o.stats[row * 3 + 1] = none ? 0.f : log_sum + left;
  o.stats[row * 3 + 2] = entropy;
}
// The n <= k largest logits above minus infinity are cand[0 .. n) or are the largest of them; the rest of k slots gets the lowest indices that are not among them.
template <int CAP, int TH>
__device__ __forceinline__ void write_top(const Out& o, int64_t row, int k, uint64_t* cand, int n, const Scale& c, const Stat& a) {
  int32_t* ids = o.top_ids + row * k;
  float* lp = o.top_logprobs + row * k;
  const float log_sum = log_of(a.s);
  const bool none = a.s == 0.f;
  ranked<TH>(cand, n, k, [&](int rank, uint64_t e) {
    ids[rank] = index_of(e);
    lp[rank] = none ? -INFINITY : behind<CAP>(value_of((unsigned)(e >> 32)), c, a.m) - log_sum;
  });
  if (n < k && (int)threadIdx.x < k) {  // (the first k indices hold at least k - n others)
    int below = 0;
    bool there = false;
    for (int j = 0; j < n; j++) {
      const int id = index_of(cand[j]);
      below += id < (int)threadIdx.x;
      there |= id == (int)threadIdx.x;
    }
    const int rank = n + (int)threadIdx.x - below;
    if (!there && rank < k) {
      ids[rank] = threadIdx.x;
      lp[rank] = none ? -INFINITY : behind<CAP>(-INFINITY, c, a.m) - log_sum;
    }
  }
}

// One workgroup to a row, or to one of `parts` equal shares of it; with part_stat a share leaves its statistics and its candidates for a kernel that joins them.
// The row is read once, a chunk of four vectors a thread ahead of the one in work; the largest score of a chunk is known before its exponentials, which are taken against the
// largest so far.  3596 x 100352 bf16: 124 us, 5.8 TB/s, the vector unit busy for 90 % of it (a copy on the card reads and writes 5.2).  1500 x 256000 with a soft-cap and 64
// alternatives: 196 us, 3.9 TB/s; 19 issue slots a logit, six of them its three transcendental instructions, keep the vector unit busy for 88 %.
template <typename T, int CAP, bool TOP, int TH>
__global__ __launch_bounds__(TH) void score_rows_kernel(const T* __restrict__ logits, const int32_t* __restrict__ targets, Out out, uint64_t* __restrict__ part_top,
                                                        Stat* __restrict__ part_stat, int V, int64_t ld, int32_t ignore_index, Scale c, int k, int parts, bool once) {
  constexpr int N = Vec<T>::N, SPAN = TH * UNROLL;
  __shared__ Lds<TH> l;
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const int target = targets ? targets[row] : -1;
  if (targets && target == ignore_index) {  // (the join writes for a row in parts)
    if (!part_stat) write_skipped(out, row, k);
    return;
  }
  const T* zr = logits + row * ld;
  const Cut cutting = cut<T, N>(zr, V);
  const T* body = zr + cutting.head;
  const int per = (cutting.nvec + parts - 1) / parts;
  const int v0 = min(part * per, cutting.nvec), v1 = min(v0 + per, cutting.nvec);
  if (TOP && threadIdx.x == 0) l.n = 0;
  Raw<T, N> next[UNROLL];
  auto fetch = [&](int at) {
    if (once) {  // (between barriers, or the compiler makes one load of both)
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < UNROLL; u++) {
        const int v = at + u * TH + threadIdx.x;
        if (v < v1) next[u].load_once(body + (int64_t)v * N);
      }
      __builtin_amdgcn_sched_barrier(0);
    } else {
#pragma unroll
      for (int u = 0; u < UNROLL; u++) {
        const int v = at + u * TH + threadIdx.x;
        if (v < v1) next[u].load(body + (int64_t)v * N);
      }
    }
  };
  fetch(v0);
  Stat a = Stat::none();
  float most = -INFINITY;  // of the logits themselves
  unsigned bound = KEY_NEG_INF;
  float bound_value = -INFINITY;
  // the single elements at the row's ends, one to a thread
  const bool has_edge = part == 0 && (int)threadIdx.x < cutting.edges;
  const int edge = has_edge ? cutting.edge(threadIdx.x, V) : 0;
  const float edge_x = has_edge ? (float)zr[edge] : -INFINITY;
  if (has_edge) {
    if (edge_x > -INFINITY) most = edge_x;
    if (CAP || edge_x > -INFINITY) a.m = level<CAP>(edge_x, c);
    const float d = behind<CAP>(edge_x, c, a.ref()), e = exp_of(d);
    a.s = e;
    a.t = e * fmaxf(d, -200.f);
  }
  const int chunks = max(1, (v1 - v0 + SPAN - 1) / SPAN);
  for (int ch = 0; ch < chunks; ch++) {
    const int at = v0 + ch * SPAN;
    Raw<T, N> now[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) now[u] = next[u];
    if (ch + 1 < chunks) fetch(at + SPAN);
    float cm = -INFINITY, vm[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      vm[u] = -INFINITY;
      if (at + u * TH + (int)threadIdx.x >= v1) continue;
      float x[N];
      now[u].unpack(x);
#pragma unroll
      for (int e = 0; e < N; e++) vm[u] = fmaxf(vm[u], x[e]);
      cm = fmaxf(cm, vm[u]);
    }
    if (cm > most || (CAP && a.m == -INFINITY)) {  // (a soft-cap makes a score of minus infinity too)
      most = fmaxf(most, cm);
      a.raise(level<CAP>(most, c), c.unit);
    }
    const float ref = a.ref();
    const float cap_r = c.r_k * LOG2E, cap_top = (c.top - ref) * LOG2E;
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      if (at + u * TH + (int)threadIdx.x >= v1) continue;
      float x[N], t[2] = {0.f, 0.f};  // (two chains of fma)
      now[u].unpack(x);
#pragma unroll
      for (int e = 0; e < N; e++) {
        if (CAP) {  // scores are finite: in units of log 2, without a cut (three of 22 issue slots of a logit; these rows are bound by them)
          const float d = CAP == 1 ? __builtin_fmaf(tail_of_tanh(x[e], c), cap_r, cap_top) : behind<CAP>(x[e], c, ref) * LOG2E;
          x[e] = __builtin_amdgcn_exp2f(d);
          t[e & 1] = __builtin_fmaf(x[e], d, t[e & 1]);
        } else {
          const float d = (x[e] - ref) * c.unit2;
          x[e] = __builtin_amdgcn_exp2f(d);
          t[e & 1] = __builtin_fmaf(x[e], fmaxf(d, -200.f), t[e & 1]);
        }
      }
#pragma unroll
      for (int w = N / 2; w > 0; w >>= 1)
#pragma unroll
        for (int e = 0; e < w; e++) x[e] += x[e + w];
      a.s += x[0];
      a.t = __builtin_fmaf(t[0] + t[1], LN2, a.t);
    }
    if (TOP) {
      if ((ch & (ch + 1)) == 0) {  // 1, 2, 4, .. chunks seen: about k candidates between two bounds, and those below the new one go where many ties came with them
        int noted;
        bound = kth_best<TH>(l.best, key_of(most), k, &l.n, &noted);
        bound_value = value_of(bound);
        if (noted > CAND / 2 && noted <= CAND) narrow<CAND, TH>(l.cand, noted, bound, &l.n);
      }
      // vectors with a candidate are noted, with their largest; which of their elements are is seen at the end, against the last bound.  (Element by element here: 1600 x 128256
      // with 20 alternatives 120 us, so 96.)
      if (cm >= bound_value && cm > -INFINITY) {
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
          if (vm[u] >= bound_value && vm[u] > -INFINITY) {
            const int to = atomicAdd(&l.n, 1);
            if (to < CAND) l.cand[to] = entry_of(key_of(vm[u]), at + u * TH + threadIdx.x);
          }
      }
    }
  }
  const Stat all = block_join<TH / 64>(a, l.red, c.unit);
  int n = 0;
  if (TOP) {
    if (((chunks - 1) & chunks) != 0) bound = kth_best<TH>(l.best, key_of(most), k, nullptr, nullptr);  // of all that was seen
    __syncthreads();
    n = l.n;
    __syncthreads();
    if (n <= CAND) {
      bound_value = value_of(bound);
      auto offer = [&](float x, int i) {
        if (x >= bound_value && x > -INFINITY) {
          const int to = atomicAdd(&l.n, 1);
          if (to < CAND) l.cand[to] = entry_of(key_of(x), i);
        }
      };
      uint64_t own[CAND / TH];
#pragma unroll
      for (int i = 0; i < CAND / TH; i++) own[i] = i * TH + (int)threadIdx.x < n ? l.cand[i * TH + threadIdx.x] : 0;
      if (threadIdx.x == 0) l.n = 0;
      __syncthreads();
      Raw<T, N> r[CAND / TH];
#pragma unroll
      for (int i = 0; i < CAND / TH; i++)
        if ((unsigned)(own[i] >> 32) >= bound) r[i].load(body + (int64_t)index_of(own[i]) * N);
#pragma unroll
      for (int i = 0; i < CAND / TH; i++)
        if ((unsigned)(own[i] >> 32) >= bound) {
          float x[N];
          r[i].unpack(x);
#pragma unroll
          for (int e = 0; e < N; e++) offer(x[e], cutting.head + index_of(own[i]) * N + e);
        }
      if (has_edge) offer(edge_x, edge);
      __syncthreads();
      n = l.n;
    }
    if (n > CAND) {
      const int first = part == 0 ? 0 : cutting.head + v0 * N;  // part 0 has the edges: the row's first elements and its last
      const int last = cutting.head + v1 * N;
      if (parts == 1) {
        n = select_exact(zr, 0, V, k, l);
      } else {
        n = select_exact(zr, first, last, k, l);
        if (part == 0) {  // the rest behind the last vector joins the k largest of the others (cand has room: k + 7 <= CAND)
          const int rest = cutting.edges - cutting.head;
          __syncthreads();
          if (threadIdx.x == 0) l.n = n;
          __syncthreads();
          if ((int)threadIdx.x < rest) {
            const int i = V - rest + threadIdx.x;
            const float x = (float)zr[i];
            if (x > -INFINITY) l.cand[atomicAdd(&l.n, 1)] = entry_of(key_of(x), i);
          }
          __syncthreads();
          n = l.n;
        }
      }
    }
  }
  if (!part_stat) {
    const bool has_target = target >= 0 && target < V;
    if (threadIdx.x == 0) write_row<CAP>(out, row, has_target, has_target ? (float)zr[target] : 0.f, c, all);
    if (TOP) write_top<CAP, TH>(out, row, k, l.cand, n, c, all);
    return;
  }
  if (threadIdx.x == 0) part_stat[blockIdx.x] = all;
  if (TOP) {
    uint64_t* mine = part_top + (int64_t)blockIdx.x * k;
    ranked<TH>(l.cand, n, k, [&](int rank, uint64_t e) { mine[rank] = e; });
    for (int i = n + threadIdx.x; i < k; i += TH) mine[i] = 0;
  }
}

// The parts of a row, one workgroup a row.
template <typename T, int CAP, bool TOP, int TH = 256>
__global__ __launch_bounds__(TH) void score_join_kernel(const T* __restrict__ logits, const int32_t* __restrict__ targets, Out out,
                                                        const uint64_t* __restrict__ part_top, const Stat* __restrict__ part_stat, int V, int64_t ld,
                                                        int32_t ignore_index, Scale c, int k, int parts) {
  __shared__ uint64_t cand[JOINED];
  __shared__ alignas(16) unsigned best[GROUPS];
  __shared__ Stat red[TH / 64];
  __shared__ int counter;
  const int64_t row = blockIdx.x;
  const int target = targets ? targets[row] : -1;
  if (targets && target == ignore_index) {
    write_skipped(out, row, k);
    return;
  }
  Stat a = Stat::none();
  if ((int)threadIdx.x < parts) a = part_stat[row * parts + threadIdx.x];
  uint64_t most = 0;
  if (TOP)
    for (int i = threadIdx.x; i < parts * k; i += TH) {
      const uint64_t e = part_top[row * parts * k + i];
      cand[i] = e;
      most = max(most, e);
    }
  a = block_join<TH / 64>(a, red, c.unit);
  const bool has_target = target >= 0 && target < V;
  if (threadIdx.x == 0) write_row<CAP>(out, row, has_target, has_target ? (float)logits[row * ld + target] : 0.f, c, a);
  if (TOP) {
    const unsigned bound = kth_best<TH>(best, max((unsigned)(most >> 32), KEY_NEG_INF), k, nullptr, nullptr);
    const int n = narrow<JOINED, TH>(cand, parts * k, bound, &counter);
    write_top<CAP, TH>(out, row, k, cand, n, c, a);
  }
}

// The rows of an LM head whose product left statistics of 256 columns a tile (olmax_gemm_head_stats), [tiles][ld_tiles], and, for the last columns, logits (`rest`, from column
// `fused` on) with statistics of their own: 16 rows a workgroup, each sixteenth of a wave takes every 64th tile.  (64 rows a workgroup, a lane each: 20 us for 2048 rows of
// 384 tiles, so 8.)
template <int CAP>
__global__ __launch_bounds__(1024) void head_join_kernel(const Stat* __restrict__ tiles, int n_tiles, const Stat* __restrict__ rest_stat, const float* __restrict__ rest,
                                                         int64_t ld_rest, const float* __restrict__ target_logit, const int32_t* __restrict__ targets, Out out, int64_t rows,
                                                         int64_t ld_tiles, int V, int fused, int32_t ignore_index, Scale c) {
  __shared__ Stat part[16][16];
  const int wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x * 16ll + (threadIdx.x & 15);
  Stat a = Stat::none();
  if (row < rows)
    for (int i = threadIdx.x >> 4; i < n_tiles; i += 64) a.join(tiles[(int64_t)i * ld_tiles + row], c.unit);
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    Stat b;
    b.m = __shfl_xor(a.m, o, 64);
    b.s = __shfl_xor(a.s, o, 64);
    b.t = __shfl_xor(a.t, o, 64);
    a.join(b, c.unit);
  }
  if ((threadIdx.x & 63) < 16) part[wave][threadIdx.x & 15] = a;
  __syncthreads();
  if (threadIdx.x >= 16 || row >= rows) return;
  const int target = targets ? targets[row] : -1;
  if (targets && target == ignore_index) {
    if (out.logprobs) out.logprobs[row] = 0.f;
    out.entropy[row] = 0.f;
    for (int i = 0; i < 3; i++) out.stats[row * 3 + i] = 0.f;
    return;
  }
  for (int w = 1; w < 16; w++) a.join(part[w][threadIdx.x], c.unit);
  if (fused < V) a.join(rest_stat[row], c.unit);
  const bool has_target = target >= 0 && target < V;
  write_row<CAP>(out, row, has_target, !has_target ? 0.f : target < fused ? target_logit[row] : rest[row * ld_rest + target - fused], c, a);
}

__global__ __launch_bounds__(256) void zero_columns_kernel(bf16* __restrict__ d, int64_t rows, int64_t ld, int n) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i < rows * n) d[i / n * ld + i % n] = (bf16)0.f;
}

// d loss / d logits of logprob and entropy: dz_i = g (delta_it - p_i) - h p_i (ln p_i + H), from the statistics that the forward pass kept.
// Reads and writes each logit once, without any wait between threads: 4096 x 50304 bf16 159 us, 5.2 TB/s, as a copy; 333 x 100278 fp32 46 us, 5.8 TB/s.
// A workgroup takes one of `parts` shares of a row.  first: the column of the whole row that these logits begin with (they are its last).
template <typename T, typename TO, int CAP, bool ENT, bool ONCE, int TH = 256>
__global__ __launch_bounds__(TH) void score_grad_kernel(const T* __restrict__ logits, TO* __restrict__ dlogits, const int32_t* __restrict__ targets,
                                                        const float* __restrict__ stats, const float* __restrict__ dlogprobs,
                                                        const float* __restrict__ dentropy, int V, int64_t ld, int64_t ldd, int32_t ignore_index, Scale c,
                                                        int parts, int pad, int first) {
  constexpr int N = Vec<TO>::N;
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const T* zr = logits + row * ld;
  TO* dr = dlogits + row * ldd;
  const Cut cutting = cut<TO, N>(dr, V);
  const int per = (cutting.nvec + parts - 1) / parts;
  const int v0 = min(part * per, cutting.nvec), v1 = min(v0 + per, cutting.nvec);
  const int target = targets[row];
  const float m = stats[row * 3], log_sum = stats[row * 3 + 1], entropy = stats[row * 3 + 2];
  const bool skipped = target == ignore_index || m == -INFINITY;  // no distribution: no gradient
  const float g = skipped || target < 0 || target >= first + V ? 0.f : dlogprobs[row], h = skipped || !ENT ? 0.f : dentropy[row];
  auto grad = [&](float x, int i) { return score_grad<CAP, ENT>(x, c, m, log_sum, entropy, g, h, first + i == target); };
  for (int v = v0 + threadIdx.x; v < v1; v += TH) {
    float x[N];
    const int i = cutting.head + v * N;
    if (!skipped) {
      Raw<T, N> r;
      if (ONCE) r.load_once(zr + i);
      else r.load(zr + i);
      r.unpack(x);
    }
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = skipped ? 0.f : grad(x[e], i + e);
    *reinterpret_cast<u32x4*>(dr + i) = Vec<TO>::pack(x);
  }
  if (part == 0 && (int)threadIdx.x < cutting.edges) {
    const int i = cutting.edge(threadIdx.x, V);
    dr[i] = (TO)(skipped ? 0.f : grad((float)zr[i], i));
  }
  if (part == 0 && (int)threadIdx.x < pad) dr[V + threadIdx.x] = (TO)0.f;
}

// Loads past the last-level cache.  Forward, of logits that it cannot hold: us, 3596 x 100352 bf16 134.4 | 124.6, 1600 x 100352 70 | 64, 1600 x 100278 fp32 123 | 115, and with the
// gradient behind it 489 | 462 for 4096 x 100352; logits that it can hold may be there from the product: 200 x 100278 fp32 17.3 | 19.3.  Backward, where gradients, which
// somebody reads next, fit, but not easily beside the logits: 333 x 100278 fp32 57.6 | 46.2, 800 x 50304 bf16 forward, backward and a product behind them 315 | 294, in place
// 1600 x 50304 64 | 58 (800 x 50304: 30 | 34); where they do not fit: 4096 x 50304 159.1 | 161.1.

// Threads of a workgroup and shares of a row in the forward pass.
struct Form {
  int threads, parts;
};
// Rows that fill the GPU by themselves take a workgroup of 256 threads each, up to 256 long ones one of 512; few ones come in shares of at least one round of loads (1024 vectors; 128256 bf16 in
// 15 of 1069, whose second round is 45), whose candidates a second launch joins: many of those cost more than longer shares of 1024 threads.  us in a graph, bf16, 256 threads x 1 | 512 x 1 | 1024 x 1 | 256 x 16 | 1024 x 4: 1 x 128256
// without alternatives 17.0 | - | 13.5 | 7.4 | 10.2, with 20 28.8 | - | 23.2 | 13.4 | 17, with 128 35.8 | - | 25.7 | 45 | 20.9; 200 x 100352 with 20 27.3 | 22.6 | 24.1; 400 x 100352 with
// 20 33.1 | 31.8 | 44.8, without 21.1 | 21.7 | 24.7; 1600 x 50304 with 20 49.7 | 54.8 | 104; 100 x 4096 without 4.7 | - | 6.2.
Form form_of(int64_t T, int V, int top, bool f32) {
  const int64_t vecs = V / (f32 ? 4 : 8);
  if (T > 256 || vecs < 2048) return {256, 1};
  if (T > 128) return {vecs < 6000 ? 256 : 512, 1};
  const int64_t shares = std::min<int64_t>(std::min<int64_t>(vecs / 1024, 1024 / T), 32);
  if (shares * top <= 640) return {256, (int)shares};
  return {1024, (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(vecs / 4096, 512 / top), 256 / T))};
}

}  // namespace

extern "C" int64_t olmax_token_logprobs_workspace_bytes(int64_t T, int32_t V, int32_t top, int32_t logits_f32) {
  if (T <= 0 || V <= 0) return 0;
  const int parts = form_of(T, V, top, logits_f32 != 0).parts;
  return parts == 1 ? 0 : T * parts * ((int64_t)std::max(top, 0) * 8 + (int64_t)sizeof(Stat));
}

extern "C" int32_t olmax_token_logprobs(hipStream_t stream, const void* logits, const int32_t* targets, float* logprobs, float* entropy, float* stats,
                                        int32_t* top_ids, float* top_logprobs, void* workspace, int64_t workspace_bytes, int64_t T, int32_t V,
                                        int64_t ld, int32_t top, int32_t logits_f32, int32_t ignore_index, float temperature, float softcap) {
  OLMAX_CHECK(logits && entropy && stats && (!logprobs || targets), OLMAX_ERR_ARG, "olmax_token_logprobs: null pointer");
  OLMAX_CHECK(T > 0 && V > 0 && V < (1 << 30) && ld >= V && T < (1LL << 24), OLMAX_ERR_SHAPE, "olmax_token_logprobs: bad shape T=%ld V=%d ld=%ld", (long)T, V, (long)ld);
  OLMAX_CHECK(top >= 0 && top <= MAX_TOP && top <= V && (top == 0 || (top_ids && top_logprobs)), OLMAX_ERR_ARG,
              "olmax_token_logprobs: 0 to %d alternatives, not more than there are logits, with both outputs (got %d)", MAX_TOP, top);
  OLMAX_CHECK(takes(temperature, softcap), OLMAX_ERR_ARG, "olmax_token_logprobs: temperature within 1e-6 and 1e6, softcap 0 or within 1e-30 and 1e30");
  OLMAX_CHECK(((uintptr_t)logits & (logits_f32 ? 3 : 1)) == 0, OLMAX_ERR_ALIGN, "olmax_token_logprobs: logits not aligned to their type");
  const Form form = form_of(T, V, top, logits_f32 != 0);
  const int parts = form.parts;
  OLMAX_CHECK(workspace_bytes >= olmax_token_logprobs_workspace_bytes(T, V, top, logits_f32) && (parts == 1 || (workspace && aligned16(workspace))), OLMAX_ERR_WORKSPACE,
              "olmax_token_logprobs: workspace needs %ld bytes, 16-byte aligned", (long)olmax_token_logprobs_workspace_bytes(T, V, top, logits_f32));
  uint64_t* part_top = (uint64_t*)workspace;
  Stat* part_stat = parts == 1 ? nullptr : (Stat*)((char*)workspace + T * parts * (int64_t)top * 8);
  const Out out{logprobs, entropy, stats, top ? top_logprobs : nullptr, top ? top_ids : nullptr};
  const Scale c = scale_of(temperature, softcap);
  const bool past_cache = T * V * (logits_f32 ? 4 : 2) > LAST_CACHE;
#define ROWS(TY, CAPV, TOPV, THV)                                                                                                                             \
  hipLaunchKernelGGL((score_rows_kernel<TY, CAPV, TOPV, THV>), dim3((unsigned)(T * parts)), dim3(THV), 0, stream, (const TY*)logits, targets, out, part_top, \
                     part_stat, V, ld, ignore_index, c, top, parts, past_cache)
#define SCORE(TY, CAPV, TOPV)                                                                                                                             \
  do {                                                                                                                                                    \
    if (form.threads == 256) ROWS(TY, CAPV, TOPV, 256); else if (form.threads == 512) ROWS(TY, CAPV, TOPV, 512); else ROWS(TY, CAPV, TOPV, 1024);                                                                  \
    if (parts > 1)                                                                                                                                        \
      hipLaunchKernelGGL((score_join_kernel<TY, CAPV, TOPV>), dim3((unsigned)T), dim3(256), 0, stream, (const TY*)logits, targets, out,                   \
                         (const uint64_t*)part_top, (const Stat*)part_stat, V, ld, ignore_index, c, top, parts);                                          \
  } while (0)
#define SCORE_T(TY, CAPV) do { if (top) SCORE(TY, CAPV, true); else SCORE(TY, CAPV, false); } while (0)
#define SCORE_C(TY) do { if (c.kind == 0) SCORE_T(TY, 0); else if (c.kind == 1) SCORE_T(TY, 1); else SCORE_T(TY, 2); } while (0)
  if (logits_f32) SCORE_C(float); else SCORE_C(bf16);
#undef ROWS
#undef SCORE
#undef SCORE_T
#undef SCORE_C
  OLMAX_LAUNCH_CHECK();
  return OLMAX_OK;
}

// grads_bf16: the gradient of fp32 logits as bf16 (the LM head's products take it); pad: zeros behind each of its rows
static int token_logprobs_bwd(hipStream_t stream, const void* logits, const int32_t* targets, const float* stats, const float* dlogprobs,
                              const float* dentropy, void* dlogits, int64_t T, int32_t V, int64_t ld, int64_t ldd, bool logits_f32, bool grads_f32,
                              int32_t ignore_index, float temperature, float softcap, int pad, int first = 0) {
  const Scale c = scale_of(temperature, softcap);
  const int parts = (int)std::max<int64_t>(1, V / (grads_f32 ? 4 : 8) / 2048);
  OLMAX_CHECK(T * parts < (1LL << 31), OLMAX_ERR_SHAPE, "olmax_token_logprobs_bwd: T=%ld rows of V=%d are too many", (long)T, V);
  const int64_t bytes = T * V * (grads_f32 ? 4 : 2);
  const bool past_cache = bytes <= LAST_CACHE && (logits == dlogits ? bytes : 2 * bytes) > LAST_CACHE / 2;
  auto go = [&](auto in, auto out, auto capped, auto entropies, auto once) {
    using TY = decltype(in);
    using TO = decltype(out);
    hipLaunchKernelGGL((score_grad_kernel<TY, TO, decltype(capped)::value, decltype(entropies)::value, decltype(once)::value>), dim3((unsigned)(T * parts)), dim3(256), 0, stream,
                       (const TY*)logits, (TO*)dlogits, targets, stats, dlogprobs, dentropy, V, ld, ldd, ignore_index, c, parts, pad, first);
  };
  auto kind = [&](auto in, auto out) {
    const std::true_type yes;
    const std::false_type no;
    auto loads = [&](auto capped, auto entropies) { past_cache ? go(in, out, capped, entropies, yes) : go(in, out, capped, entropies, no); };
    auto entropies = [&](auto capped) { dentropy ? loads(capped, yes) : loads(capped, no); };
    if (c.kind == 0) entropies(std::integral_constant<int, 0>());
    else if (c.kind == 1) entropies(std::integral_constant<int, 1>());
    else entropies(std::integral_constant<int, 2>());
  };
  if (logits_f32 && grads_f32) kind(0.f, 0.f);
  else if (logits_f32) kind(0.f, bf16());
  else kind(bf16(), bf16());
  OLMAX_LAUNCH_CHECK();
  return OLMAX_OK;
}

extern "C" int32_t olmax_token_logprobs_bwd(hipStream_t stream, const void* logits, const int32_t* targets, const float* stats, const float* dlogprobs,
                                            const float* dentropy, void* dlogits, int64_t T, int32_t V, int64_t ld, int64_t ldd, int32_t logits_f32,
                                            int32_t ignore_index, float temperature, float softcap) {
  OLMAX_CHECK(logits && targets && stats && dlogprobs && dlogits, OLMAX_ERR_ARG, "olmax_token_logprobs_bwd: null pointer");
  OLMAX_CHECK(T > 0 && V > 0 && V < (1 << 30) && ld >= V && ldd >= V && T < (1LL << 24), OLMAX_ERR_SHAPE, "olmax_token_logprobs_bwd: bad shape T=%ld V=%d", (long)T, V);
  OLMAX_CHECK(takes(temperature, softcap), OLMAX_ERR_ARG, "olmax_token_logprobs_bwd: temperature within 1e-6 and 1e6, softcap 0 or within 1e-30 and 1e30");
  OLMAX_CHECK((((uintptr_t)logits | (uintptr_t)dlogits) & (logits_f32 ? 3 : 1)) == 0, OLMAX_ERR_ALIGN, "olmax_token_logprobs_bwd: operands not aligned to their type");
  OLMAX_CHECK(logits != dlogits || ld == ldd, OLMAX_ERR_ARG, "olmax_token_logprobs_bwd: in place wants one row stride");
  OLMAX_CHECK(!overlap(logits, ld, dlogits, ldd, T, V, logits_f32 ? 4 : 2), OLMAX_ERR_ARG, "olmax_token_logprobs_bwd: the gradient overlaps the logits, but is not in their place");
  return token_logprobs_bwd(stream, logits, targets, stats, dlogprobs, dentropy, dlogits, T, V, ld, ldd, logits_f32 != 0, logits_f32 != 0, ignore_index,
                            temperature, softcap, 0);
}

// ---- with the LM head's product.  The logits are fp32: the framework's bf16 ones are off by 2^-9 of themselves, as much in a
// log probability as policies of two steps may be apart.  Their gradient is rounded to bf16 in front of its two products, which are the matrix cores' only so (fp32 ones would be two or three
// times as many): dh and dW are off by two roundings, 0.0023 of themselves in the mean at 1024 x 4096 x 100352, and by one, 0.0017, if only they were rounded.  Where the product runs in large tiles they stay in its accumulators (HeadRows), but for the columns behind the last whole
// round of tiles, which are a product of their own; where it does not, or alternatives are asked for, all of them go through the workspace.  us, logits in the workspace -> not: 2048
// x 4096 x 100352 1443 -> 1195 (the product alone, fp32 logits written, 1335), gradients of 1024 x 4096 x 100352 2080 -> 1977.
static int64_t head_stride(int32_t V) { return ((int64_t)V + 63) / 64 * 64; }  // whole lines of bf16 and fp32
static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// Memory of the forward call: fp32 logits of the columns from `fused` on, then (fused > 0) statistics of its tiles, of the other columns, target logits, and tokens that are
// padded (to `rows`)
struct HeadPlan {
  int fused;
  int64_t rows, ld, stats_at, rest_at, target_at, h_at, bytes;
};
static HeadPlan head_plan(int64_t T, int32_t d, int32_t V, int32_t top) {
  HeadPlan p;
  p.rows = top == 0 && T > 64 && olmax_lmhead_pads(T, d, V) ? 256 : T;
  p.fused = top > 0 ? 0 : olmax_gemm_head_columns((int)p.rows, V, d);
  p.ld = head_stride(V - p.fused);
  p.stats_at = up256(p.rows * p.ld * 4);
  p.rest_at = p.stats_at + up256((int64_t)((p.fused + 255) / 256) * p.rows * sizeof(Stat));
  p.target_at = p.rest_at + up256(T * sizeof(Stat));
  p.h_at = p.target_at + up256(T * 4);
  p.bytes = p.fused ? p.h_at + (p.rows > T ? up256(p.rows * d * 2) : 0) : p.stats_at + olmax_token_logprobs_workspace_bytes(T, V, top, 1);
  return p;
}

extern "C" int64_t olmax_lmhead_logprobs_workspace_bytes(int64_t T, int32_t d, int32_t V, int32_t top) {
  return T <= 0 || V <= 0 || d <= 0 || T >= (1 << 24) ? 0 : head_plan(T, d, V, top).bytes;
}

int olmax_lmhead_logprobs_check(const HeadScore& a) {
  OLMAX_CHECK(a.h && a.W && a.workspace && a.entropy && a.stats && (!a.logprobs || a.targets), OLMAX_ERR_ARG, "olmax_lmhead_logprobs: null pointer");
  OLMAX_CHECK(a.T > 0 && a.d > 0 && a.V > 0 && a.V < (1 << 30) && a.T < (1LL << 24), OLMAX_ERR_SHAPE, "olmax_lmhead_logprobs: bad shape T=%ld d=%d V=%d", (long)a.T, a.d, a.V);
  OLMAX_CHECK(a.top >= 0 && a.top <= MAX_TOP && a.top <= a.V && (a.top == 0 || (a.top_ids && a.top_logprobs)), OLMAX_ERR_ARG,
              "olmax_lmhead_logprobs: 0 to %d alternatives, not more than there are logits, with both outputs (got %d)", MAX_TOP, a.top);
  OLMAX_CHECK(takes(a.temperature, a.softcap), OLMAX_ERR_ARG,
              "olmax_lmhead_logprobs: temperature within 1e-6 and 1e6, softcap 0 or within 1e-30 and 1e30");
  OLMAX_CHECK(aligned16(a.h) && aligned16(a.W), OLMAX_ERR_ALIGN, "olmax_lmhead_logprobs: h and W must be 16-byte aligned");
  const int64_t need = head_plan(a.T, a.d, a.V, a.top).bytes;
  OLMAX_CHECK(a.workspace_bytes >= need && (((uintptr_t)a.workspace) & 255) == 0, OLMAX_ERR_WORKSPACE, "olmax_lmhead_logprobs: workspace needs %ld bytes, 256-byte aligned", (long)need);
  return OLMAX_OK;
}

extern "C" int32_t olmax_lmhead_logprobs(hipStream_t stream, const void* h, const void* W, const int32_t* targets, float* logprobs, float* entropy,
                                         float* stats, int32_t* top_ids, float* top_logprobs, void* workspace, int64_t workspace_bytes, int64_t T,
                                         int32_t d, int32_t V, int32_t top, int32_t ignore_index, float temperature, float softcap) {
  if (int rc = olmax_lmhead_logprobs_check({h, W, targets, logprobs, entropy, stats, top_ids, top_logprobs, workspace, workspace_bytes, T, d, V, top, ignore_index, temperature,
                                            softcap}))
    return rc;
  const HeadPlan p = head_plan(T, d, V, top);
  const bf16 *hp = (const bf16*)h, *wp = (const bf16*)W;
  char* ws = (char*)workspace;
  if (p.rows > T) {
    olmax_pad_rows(stream, hp, (bf16*)(ws + p.h_at), T, p.rows, d);
    hp = (bf16*)(ws + p.h_at);
  }
  const int rest = V - p.fused;
  if (rest) {
    if (int rc = olmax_gemm_padded(stream, hp, wp + (int64_t)p.fused * d, ws, nullptr, (int)p.rows, rest, d, d, d, p.ld, 0, true, true, true, false)) return rc;
  }
  if (!p.fused)
    return olmax_token_logprobs(stream, ws, targets, logprobs, entropy, stats, top_ids, top_logprobs, ws + p.stats_at, workspace_bytes - p.stats_at, T, V, p.ld, top, 1,
                                ignore_index, temperature, softcap);
  const Scale c = scale_of(temperature, softcap);
  const Out out{logprobs, entropy, stats, nullptr, nullptr};
  Stat *tiles = (Stat*)(ws + p.stats_at), *rest_stat = (Stat*)(ws + p.rest_at);
  float* target_logit = (float*)(ws + p.target_at);
  HeadRows rows{};
  rows.targets = targets;
  rows.ignore_index = ignore_index;
  rows.V = V;
  rows.rows = (int)T;
  rows.scale = c;
  rows.parts = (float*)tiles;
  rows.target_logit = target_logit;
  if (int rc = olmax_gemm_head_stats(stream, hp, wp, (int)p.rows, p.fused, d, rows)) return rc;
  auto join = [&](auto capped) {
    constexpr int CAP = decltype(capped)::value;
    if (rest)
      hipLaunchKernelGGL((score_rows_kernel<float, CAP, false, 256>), dim3((unsigned)T), dim3(256), 0, stream, (const float*)ws, targets, out, (uint64_t*)nullptr, rest_stat, rest,
                         p.ld, ignore_index, c, 0, 1, false);
    hipLaunchKernelGGL((head_join_kernel<CAP>), dim3((unsigned)((T + 15) / 16)), dim3(1024), 0, stream, (const Stat*)tiles, (p.fused + 255) / 256, (const Stat*)rest_stat,
                       (const float*)ws, p.ld, (const float*)target_logit, targets, out, T, p.rows, V, p.fused, ignore_index, c);
  };
  if (c.kind == 0) join(std::integral_constant<int, 0>());
  else if (c.kind == 1) join(std::integral_constant<int, 1>());
  else join(std::integral_constant<int, 2>());
  OLMAX_LAUNCH_CHECK();
  return OLMAX_OK;
}

// The backward call's: bf16 gradients, then fp32 logits of the columns from `fused` on and, in the same place afterwards, room for the products' partial sums; then (tokens
// padded to `rows`) the padded tokens, and room for dh
struct HeadGradPlan {
  int fused;
  bool in64;  // gradients of 64 tokens
  int64_t rows, ld, logits_at, room, h_at, dh_at, bytes;
};
static HeadGradPlan head_grad_plan(int64_t T, int32_t d, int32_t V) {
  HeadGradPlan p;
  p.rows = olmax_lmhead_pads(T, d, V) ? 256 : T;
  p.fused = olmax_gemm_head_columns((int)p.rows, V, d);
  p.ld = head_stride(V);
  p.in64 = olmax_lmhead_pads_64(T, d, V);
  p.logits_at = up256((p.in64 ? 64 : p.rows) * p.ld * 2);
  p.room = std::max(up256(p.rows * head_stride(V - p.fused) * 4), p.fused ? PRODUCT_SCRATCH : 0);
  p.h_at = p.logits_at + p.room;
  p.dh_at = p.h_at + (p.rows > T ? up256(p.rows * d * 2) : p.in64 ? up256(64ll * d * 2) : 0);
  p.bytes = p.dh_at + (p.rows > T ? up256(p.rows * d * 2) : p.in64 ? up256(64ll * d * 2) : 0);
  return p;
}
extern "C" int64_t olmax_lmhead_logprobs_bwd_workspace_bytes(int64_t T, int32_t d, int32_t V) {
  return T <= 0 || V <= 0 || d <= 0 || T >= (1 << 24) ? 0 : head_grad_plan(T, d, V).bytes;
}

int olmax_lmhead_logprobs_bwd_check(const HeadScoreGrad& a) {
  OLMAX_CHECK(a.h && a.W && a.targets && a.stats && a.dlogprobs && a.workspace && (a.dh || a.dW), OLMAX_ERR_ARG, "olmax_lmhead_logprobs_bwd: null pointer");
  OLMAX_CHECK(a.T > 0 && a.d > 0 && a.V > 0 && a.V < (1 << 30) && a.T < (1LL << 24), OLMAX_ERR_SHAPE, "olmax_lmhead_logprobs_bwd: bad shape T=%ld d=%d V=%d", (long)a.T, a.d, a.V);
  OLMAX_CHECK(takes(a.temperature, a.softcap), OLMAX_ERR_ARG,
              "olmax_lmhead_logprobs_bwd: temperature within 1e-6 and 1e6, softcap 0 or within 1e-30 and 1e30");
  OLMAX_CHECK(aligned16(a.h) && aligned16(a.W) && aligned16(a.dh), OLMAX_ERR_ALIGN, "olmax_lmhead_logprobs_bwd: h, W and dh must be 16-byte aligned");
  const int64_t need = head_grad_plan(a.T, a.d, a.V).bytes;
  OLMAX_CHECK(a.workspace_bytes >= need && (((uintptr_t)a.workspace) & 255) == 0, OLMAX_ERR_WORKSPACE, "olmax_lmhead_logprobs_bwd: workspace needs %ld bytes, 256-byte aligned",
              (long)need);
  return OLMAX_OK;
}

extern "C" int32_t olmax_lmhead_logprobs_bwd(hipStream_t stream, const void* h, const void* W, const int32_t* targets, const float* stats,
                                             const float* dlogprobs, const float* dentropy, void* dh, void* dW, void* workspace, int64_t workspace_bytes,
                                             int64_t T, int32_t d, int32_t V, int32_t ignore_index, float temperature, float softcap, int32_t dw_f32) {
  if (int rc = olmax_lmhead_logprobs_bwd_check({h, W, targets, stats, dlogprobs, dentropy, dh, dW, workspace, workspace_bytes, T, d, V, temperature, softcap})) return rc;
  const HeadGradPlan p = head_grad_plan(T, d, V);
  const int rest = V - p.fused, pad = (8 - V % 8) % 8, rows_of = (int)p.rows;
  const bf16 *hp = (const bf16*)h, *wp = (const bf16*)W;
  char* ws = (char*)workspace;
  bf16* grads = (bf16*)ws;
  float* logits = (float*)(ws + p.logits_at);
  const bool padded = p.rows > T, in64 = p.in64 && dW;  // (dh alone gains nothing by it)
  bf16* h_pad = (bf16*)(ws + p.h_at);
  if (padded || in64) olmax_pad_rows(stream, hp, h_pad, T, padded ? p.rows : 64, d);
  const bf16* tokens = padded ? h_pad : hp;
  if (p.fused) {
    HeadRows rows{};
    rows.targets = targets;
    rows.ignore_index = ignore_index;
    rows.V = V;
    rows.rows = (int)T;
    rows.scale = scale_of(temperature, softcap);
    rows.stats = stats, rows.dlogprobs = dlogprobs, rows.dentropy = dentropy;
    if (int rc = olmax_gemm_head_grads(stream, tokens, wp, grads, p.ld, rows_of, p.fused, d, rows)) return rc;
  }
  if (rest) {
    const int64_t ldr = head_stride(rest);
    if (int rc = olmax_gemm_padded(stream, tokens, wp + (int64_t)p.fused * d, logits, nullptr, rows_of, rest, d, d, d, ldr, 0, true, true, true, false)) return rc;
    if (int rc = token_logprobs_bwd(stream, logits, targets, stats, dlogprobs, dentropy, grads + p.fused, T, rest, ldr, p.ld, true, false, ignore_index, temperature, softcap, pad,
                                    p.fused))
      return rc;
    if (padded || in64) olmax_zero_rows(stream, grads + p.fused, T, 64, rest + pad, p.ld);
  } else if (pad) {
    hipLaunchKernelGGL(zero_columns_kernel, dim3((unsigned)((p.rows * pad + 255) / 256)), dim3(256), 0, stream, grads + V, p.rows, p.ld, pad);
  }
  const GemmScratch scratch{logits, std::min(p.room, PRODUCT_SCRATCH)};
  if (padded || in64)
    return olmax_lmhead_products_few(stream, grads, wp, hp, h_pad, (bf16*)dh, dW, (int)T, d, V, p.ld, dw_f32 != 0, (bf16*)(ws + p.dh_at), padded ? 256 : 64, scratch);
  // (without shared reductions the few long ones of dh take 60 % more: dh and dW of 1024 x 4096 x 100352 1.78 -> 1.34 ms)
  return olmax_lmhead_products(stream, grads, wp, hp, (bf16*)dh, dW, (int)T, d, V, p.ld, dw_f32 != 0, scratch);
}
