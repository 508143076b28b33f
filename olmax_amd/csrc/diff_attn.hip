// Differential attention for gfx950: the difference of two causal softmax maps, with its gradients.  GQA, optional sliding window, BSHD layout, bf16 in and out, fp32
// statistics.  No counterpart in the reference; beside its attention (src/olmax/nn/attention.py:96-103, attn.hip).
//
// A query head h has two queries q_1, q_2 of width D side by side in 2D columns, its key head two keys, and values of width W = 2D (a head of 128 columns is two maps of 64):
//   s_m = q_m k_m^T / sqrt(D),  P_m = softmax(s_m),  O_m = P_m v,   o = O_1 - lambda_h O_2
// Key j is visible to query i iff j <= i and (window < 0 or j >= i - window).  With dP = do v^T and delta_m = do . O_m (a row's sum of P_m dP):
//   dS_1 = P_1 (dP - delta_1),  dS_2 = -lambda P_2 (dP - delta_2),  dq_m = dS_m k_m / sqrt(D),  dk_m = dS_m^T q_m / sqrt(D),
//   dv = (P_1 - lambda P_2)^T do,  dlambda = - sum of delta_2 over the head's queries
// so that the gradients take no more products than one map of width W does, but the exponentials of two.
// D is 32 or 64.  Maps of 128 have values of 256: a wave's accumulators of 32 queries would be 128 registers in the forward pass and 256 in dK/dV's, and three stages of K and V 192 KB of the 160 that
// there are, so that they would want kernels of another layout.
//
// The kernels are laid out as those of attn.hip: score tiles are transposed, a lane owns one query (forward, dQ) or one key (dK/dV), and a [rows][W] tile of K or Q holds both
// maps' halves of a row, k-steps 0 .. W/32 - 1 of the products the first one's.
#include "attn_tiles.h"
#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>
#include <utility>

namespace {

// 4 B per lane straight into LDS, as dma16
__device__ __forceinline__ void dma4(const void* g, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds_addr), "v"(g) : "m0", "memory");
}

// Where workgroups would be few and their chains long, a chain is dealt to n workgroups, size steps to each; what they have goes to memory in fp32, [row][n], and a second kernel joins it.  See plan_of.
constexpr int MOST_CHUNKS = 64;
struct Chunks {
  float* to;
  int size, n;
  int upto[MOST_CHUNKS];  // chains that have a chunk p are the longest upto[p] - upto[p - 1]: workgroup w of a head has the chunk p with w in between, of one of these
};
struct Place { int chain, part; };
template <bool PART>
__device__ __forceinline__ Place place_of(const Chunks& ch, int w) {
  if constexpr (!PART) return {w, 0};
  int p = 0, before = 0;
  while (p + 1 < ch.n && w >= ch.upto[p]) before = ch.upto[p++];
  return {w - before, p};
}

struct Sizes {
  int S, H, KH, window;
  int64_t ldq, ldk, ldv, ldo, ldo2;
  float scale;
  int shared;  // one lambda for all heads
};

// ---- Rows that come out infinite or NaN: see redo_rows.  What a row does not see must not reach it, and the tile products take hidden pairs along as zeros, which an infinity
// or a NaN turns into NaN.  A wave that finds such values among those it has stored does their rows over, over visible pairs only: lane l has key or query l of 64 for the scores, columns l and
// l + 64 of the row for the sums.  Speed does not matter here.
__device__ __forceinline__ float dot(const bf16* a, const bf16* b, int n) {
  float s = 0.f;
#pragma unroll 1
  for (int c = 0; c < n; c += 8) {
    Pack8 x, y;
    x.u = *reinterpret_cast<const u32x4*>(a + c);
    y.u = *reinterpret_cast<const u32x4*>(b + c);
#pragma unroll
    for (int e = 0; e < 8; e++) s += bf2f(x.e[e]) * bf2f(y.e[e]);
  }
  return s;
}

// second: whether something of the second map's is not finite either.  Otherwise its o2 and log-normaliser stand, and
// stay as they are: another wave may still be storing them.  A log-normaliser that is finite stands as well.
template <int W>
__device__ __forceinline__ void redo_fwd(const bf16* q, const bf16* K, int64_t ldk, const bf16* V, int64_t ldv, float lam, bf16* o, bf16* o2, float* lse, int S, int i, int window,
                                         float scale, int lane, bool second) {
  constexpr int D = W / 2;
  const int first = window >= 0 ? max(0, i - window) : 0;
  float l[2];
#pragma unroll 1
  for (int m = 0; m < 2; m++) {
    float mx = -INFINITY, sm = 0.f;
#pragma unroll 1
    for (int j = first + lane; j <= i; j += 64) mx = fmaxf(mx, dot(q + m * D, K + j * ldk + m * D, D) * scale);
    mx = wave_max(mx);
#pragma unroll 1
    for (int j = first + lane; j <= i; j += 64) sm += __expf(dot(q + m * D, K + j * ldk + m * D, D) * scale - mx);
    l[m] = mx + __logf(wave_sum(sm));
    if (lane == 0 && (m == 0 || second) && !(fabsf(lse[m * S]) < INFINITY)) lse[m * S] = l[m];
  }
  float acc[2][W / 64] = {};
#pragma unroll 1
  for (int j0 = first; j0 <= i; j0 += 64) {
    const int n = min(64, i - j0 + 1);
    float p1 = 0.f, p2 = 0.f;
    if (lane < n) {
      p1 = __expf(dot(q, K + (j0 + lane) * ldk, D) * scale - l[0]);
      p2 = __expf(dot(q + D, K + (j0 + lane) * ldk + D, D) * scale - l[1]);
    }
#pragma unroll 1
    for (int t = 0; t < n; t++) {
      const float a = __shfl(p1, t, 64), b = __shfl(p2, t, 64);
#pragma unroll
      for (int c = 0; c < W / 64; c++) {
        const float v = bf2f(V[(j0 + t) * ldv + c * 64 + lane]);
        acc[0][c] += a * v;
        acc[1][c] += b * v;
      }
    }
  }
#pragma unroll
  for (int c = 0; c < W / 64; c++) {
    const int at = c * 64 + lane;
    o[at] = f2bf(acc[0][c] - lam * acc[1][c]);
    if (o2 && second) o2[at] = f2bf(acc[1][c]);
  }
}

// What gradients of queries and keys are multiplied by: a query that sees one key alone has P = 1 whatever they are, and gradients of exactly 0, where an exponential, and dP in two places, leave
// roundings; so has a key that only such queries see, where there are no others.  (Not a select: what is not finite stays so.)
__device__ __forceinline__ float query_moves(int i, int window) { return i == 0 || window == 0 ? 0.f : 1.f; }
__device__ __forceinline__ float key_moves(int S, int window) { return S == 1 || window == 0 ? 0.f : 1.f; }

// p_m and dP of a pair
template <int W>
__device__ __forceinline__ void pair_of(const bf16* q, const bf16* k, const bf16* d_o, const bf16* v, float l1, float l2, float scale, float& p1, float& p2, float& dp) {
  constexpr int D = W / 2;
  p1 = __expf(dot(q, k, D) * scale - l1);
  p2 = __expf(dot(q + D, k + D, D) * scale - l2);
  dp = dot(d_o, v, W);
}

// columns [lo, hi) of the row; sum1, sum2: the row's sums of P_m dP, which are its delta
template <int W>
__device__ __forceinline__ void redo_dq(const bf16* q, const bf16* K, int64_t ldk, const bf16* V, int64_t ldv, const bf16* d_o, float l1, float l2, float lam, bf16* dq, int i, int window,
                                        float scale, int lane, int lo, int hi, float& sum1, float& sum2) {
  constexpr int D = W / 2;
  const int first = window >= 0 ? max(0, i - window) : 0;
  float acc[W / 64] = {};
  sum1 = sum2 = 0.f;
#pragma unroll 1
  for (int j = first + lane; j <= i; j += 64) {
    float p1, p2, dp;
    pair_of<W>(q, K + j * ldk, d_o, V + j * ldv, l1, l2, scale, p1, p2, dp);
    sum1 += p1 * dp;
    sum2 += p2 * dp;
  }
  sum1 = wave_sum(sum1);
  sum2 = wave_sum(sum2);
#pragma unroll 1
  for (int j0 = first; j0 <= i; j0 += 64) {
    const int n = min(64, i - j0 + 1);
    float s1 = 0.f, s2 = 0.f;
    if (lane < n) {
      float p1, p2, dp;
      pair_of<W>(q, K + (j0 + lane) * ldk, d_o, V + (j0 + lane) * ldv, l1, l2, scale, p1, p2, dp);
      s1 = p1 * (dp - sum1);
      s2 = -lam * p2 * (dp - sum2);
    }
#pragma unroll 1
    for (int t = 0; t < n; t++) {
      const float a = __shfl(s1, t, 64), b = __shfl(s2, t, 64);
#pragma unroll
      for (int c = 0; c < W / 64; c++) acc[c] += (c * 64 + lane < D ? a : b) * bf2f(K[(j0 + t) * ldk + c * 64 + lane]);
    }
  }
#pragma unroll
  for (int c = 0; c < W / 64; c++)
    if (c * 64 + lane >= lo && c * 64 + lane < hi) dq[c * 64 + lane] = f2bf(acc[c] * (scale * query_moves(i, window)));
}

// key j, columns [lo, hi); Q, dO, stats, lam of the first of its rep query heads
template <int W>
__device__ __forceinline__ void redo_dkv(const bf16* Q, int64_t ldq, const bf16* dO, int64_t lddo, const float* stats, const float* lam, int lam_step, const bf16* k, const bf16* v,
                                         bf16* dk, bf16* dv, int j, int S, int rep, int window, float scale, int lane, int lo, int hi) {
  constexpr int D = W / 2;
  const int last = window >= 0 ? min(S - 1, j + window) : S - 1;
  float ak[W / 64] = {}, av[W / 64] = {};
#pragma unroll 1
  for (int r = 0; r < rep; r++, Q += W, dO += W, stats += 4 * (int64_t)S, lam += lam_step)
#pragma unroll 1
    for (int i0 = j; i0 <= last; i0 += 64) {
      const int n = min(64, last - i0 + 1);
      float p = 0.f, s1 = 0.f, s2 = 0.f;
      if (lane < n) {
        const int64_t i = i0 + lane;
        const float* st = stats + i;
        float p1, p2, dp;
        pair_of<W>(Q + i * ldq, k, dO + i * lddo, v, st[0] * LN2, st[S] * LN2, scale, p1, p2, dp);
        dp += st[2 * (int64_t)S];
        s1 = p1 * dp;
        s2 = p2 * (st[3 * (int64_t)S] - *lam * dp);
        p = p1 - *lam * p2;
      }
#pragma unroll 1
      for (int t = 0; t < n; t++) {
        const float a = __shfl(s1, t, 64), b = __shfl(s2, t, 64), pt = __shfl(p, t, 64);
#pragma unroll
        for (int c = 0; c < W / 64; c++) {
          ak[c] += (c * 64 + lane < D ? a : b) * bf2f(Q[(i0 + t) * ldq + c * 64 + lane]);
          av[c] += pt * bf2f(dO[(i0 + t) * lddo + c * 64 + lane]);
        }
      }
    }
#pragma unroll
  for (int c = 0; c < W / 64; c++) {
    const int at = c * 64 + lane;
    if (at < lo || at >= hi) continue;
    dk[at] = f2bf(ak[c] * (scale * key_moves(S, window)));
    dv[at] = f2bf(av[c]);
  }
}

// Fragments that have been loaded, and that the compiler knows to have been: it counts no transfer of inline assembly, and where it finds a load of its own unfinished on some way into a loop it waits
// there, in every round, for as many as were behind that load, which are the tiles under way.  (Gradients of 1 x 4096 tokens, 32/8 heads of 32: 422 us, 407 with this; heads of 64, whose rounds are longer, the same.)
template <int N>
__device__ __forceinline__ void arrived(bf16x8 (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+v"(f[i]));
}

// The lane, formed where it is needed rather than kept in a register
__device__ __forceinline__ int lane_id() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}

// f(0) .. f(N - 1) with the index as a constant (a loop of 48 products is not unrolled before its arrays would have to be registers)
template <typename F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
  each_of(f, std::make_integer_sequence<int, N>());
}

// Scores of pairs that are not visible become -3e38 (s + I M): two more k-steps, of the identity and a mask with M[k][column] = 0 or -3e38 (hides(k, column)), into the accumulators where they
// are, so that tiles inside pay nothing.  (As selects on the scores every tile pays; in a branch or a second copy of the tile the accumulators of the two ways meet in copies and spill.)
// Lane and column are hidden from the compiler, which otherwise keeps what is formed of them through the loop.
template <typename F>
__device__ __forceinline__ void hide(f32x16& s1, f32x16& s2, int lane, int column, F hides) {
  asm volatile("" : "+v"(lane), "+v"(column));
#pragma unroll
  for (int u = 0; u < 2; u++) {
    bf16x8 one, mask;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int k = u * 16 + (lane >> 5) * 8 + e;
      one[e] = f2bf(k == (lane & 31) ? 1.f : 0.f);
      mask[e] = f2bf(hides(k, column) ? -3e38f : 0.f);
    }
    s1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(one, mask, s1, 0, 0, 0);
    s2 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(one, mask, s2, 0, 0, 0);
  }
}

// ---------------------------------------------------------------------------------------
// Forward.  grid = ceil(S / 32 QW) H B workgroups of 2 QW waves; wave (qw, m) owns 32 queries and one map, and the two waves of a SIMD (QW = 4), qw of either map, take turns: a key tile is two parts, the softmax
// (vector unit) and the products (matrix unit: this tile's probabilities with V, the next tile's scores), a barrier ends each, and map 1 is one part behind map 0.
// LDS: 3 stages of K, then of V.  Map 0's waves fetch K, map 1's V.  K(t) is read in parts 2t - 1 and 2t, V(t) in 2t + 1 and 2t + 2 (counted as map 0 does), so that K(t + 3) is issued in 2t + 1 and
// V(t + 2) too, and each has four parts to land; past the end the last tile is fetched again.
// 2 x 4096 tokens, 32 heads of 64: 470 us, 412 GFLOP of products at 880 TFLOP/s, 1.9 GHz; a map's 32 x 64 tile takes a SIMD 1560 clk, 768 of them matrix instructions.  Bound by what a wave can
// issue, and by the power: without the products 380 us, without the exponentials' part 510 (its own latencies then stand alone), without the LDS reads 7 % less, without the transfers 2 %.
// No gain: one barrier a tile with the maps half a tile apart (496), 64 queries to a wave on tiles of 32 keys (538; it spills 12 registers), scores ahead of the values' products with the maximum in
// their shadow (500), addresses moved by steps (472; heads of 32: 3 % less, heads of 64 1 % more).
// ---------------------------------------------------------------------------------------
template <int N>
__device__ __forceinline__ void part_ends() {  // at most the newest N transfers of this wave are under way; its LDS reads are done
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
constexpr int smem_fwd(int W) { return 2 * 3 * 64 * W * 2; }
template <int W, int QW, bool PART>
__global__ __launch_bounds__(QW * 128, 2) void diff_attn_fwd_kernel(const bf16* __restrict__ Q, const bf16* __restrict__ K, const bf16* __restrict__ V, const float* __restrict__ LAM,
                                                               bf16* __restrict__ O, bf16* __restrict__ O2, float* __restrict__ LSE, const Sizes z, const Chunks ch) {
  constexpr int TILE = 64 * W * 2;  // bytes of a K or V tile of 64 keys
  constexpr int KS = W / 32;        // k-steps of a map
  constexpr int QR = QW * 32;       // queries of the workgroup
  constexpr int SHARES = 4 / QW;    // of a tile's four that a wave fetches
  constexpr int INS = 64 * W / 2048 * SHARES;  // its transfers
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];  // [3] K, [3] V
  const int S = z.S, H = z.H, KH = z.KH, window = z.window;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, lhi = lane >> 5;
  const int qw = wave % QW, m = wave / QW;
  const int nqt = (S + QR - 1) / QR;
  const WgCoord wg = decode_wg(blockIdx.x, (int)(gridDim.x / ((PART ? ch.upto[ch.n - 1] : nqt) * (H / KH))), H / KH);
  const Place place = place_of<PART>(ch, wg.rank);
  const int qt = nqt - 1 - place.chain, part = place.part;  // longest rows first
  const int b = wg.group / KH, kh = wg.group % KH;
  const int h = kh * (H / KH) + wg.r;
  const int i0 = qt * QR;
  const int iw0 = i0 + qw * 32;
  const int qi = iw0 + l32;  // this lane's query
  const int qic = min(qi, S - 1);

  bf16x8 qf[KS];
  {
    const bf16* qp = Q + ((int64_t)b * S + qic) * z.ldq + h * W + m * (W / 2) + lhi * 8;
#pragma unroll
    for (int s = 0; s < KS; s++) qf[s] = *reinterpret_cast<const bf16x8*>(qp + s * 16);
  }
  int t_lo = (window >= 0 ? max(0, i0 - window) : 0) >> 6;
  int t_hi = min(i0 + QR - 1, S - 1) >> 6;  // inclusive
  if constexpr (PART) {
    t_lo += part * ch.size;
    if (t_lo > t_hi) return;
    t_hi = min(t_hi, t_lo + ch.size - 1);
  }

  f32x16 o[W / 32], st[2];
#pragma unroll
  for (int dt = 0; dt < W / 32; dt++)
#pragma unroll
    for (int r = 0; r < 16; r++) o[dt][r] = 0.f;
  float mx = -INFINITY, sum = 0.f;

  const bf16* kbase = K + (int64_t)b * S * z.ldk + kh * W;
  const bf16* vbase = V + (int64_t)b * S * z.ldv + kh * W;
  const unsigned lds0 = lds_addr_of(smem);
  const bf16* base = m ? vbase : kbase;
  const int64_t ld = m ? z.ldv : z.ldk;
  TileDma<64, W> dma[SHARES];
#pragma unroll
  for (int i = 0; i < SHARES; i++) dma[i].init(ld, qw + i * QW, lane);
  auto load = [&](int t, int stage) {  // of this wave's operand
    t = min(t, t_hi);
    const unsigned dst = lds0 + (m * 3 + stage) * TILE;
#pragma unroll
    for (int i = 0; i < SHARES; i++) {
      if (t * 64 + 64 <= S) dma[i].issue(base + (int64_t)t * 64 * ld, dst, qw + i * QW);
      else dma_tile<64, W>(base, ld, t * 64, S, dst, qw + i * QW, lane);
    }
  };
  const float sc2 = z.scale * LOG2E;
  FragAddr<W> fa;
  fa.init(lane);
  const int kmap = (m * KS) << 5;  // of the swizzled chunk index: this map's k-steps (KS is 2 or 4: the bits are apart)
  auto visible = [&](int t) { return t * 64 <= iw0 + 31 && (window < 0 || t * 64 + 63 >= iw0 - window); };
  auto scores = [&](int stage) {
    const unsigned char* sk = smem + stage * TILE;
#pragma unroll
    for (int jt = 0; jt < 2; jt++)
#pragma unroll
      for (int r = 0; r < 16; r++) st[jt][r] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int jt = 0; jt < 2; jt++) {
        const bf16x8 kf = *reinterpret_cast<const bf16x8*>(sk + (fa.kc[s] ^ kmap) + jt * 32 * (2 * W));
        st[jt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[s], st[jt], 0, 0, 0);
      }
  };

  load(t_lo, 0);
  load(t_lo + 1, 1);
  if (m == 0) load(t_lo + 2, 2);
  arrived(qf);
  part_ends<0>();
  if (visible(t_lo)) scores(0);
  if (m == 1) part_ends<0>();
  int stage = 0;  // of tile t
  for (int t = t_lo; t <= t_hi; t++) {
    const int next = stage == 2 ? 0 : stage + 1, after = next == 2 ? 0 : next + 1;
    const bool vis = visible(t);
    // ---- softmax
    if (m == 1) load(t + 2, after);
    bf16x8 pb[4];
    if (vis) {
      const int j0 = t * 64;
      const bool need_mask = (j0 + 63 > iw0) || (window >= 0 && j0 < iw0 + 31 - window);
      if (need_mask) {
        int i = qi, half = lhi;
        asm volatile("" : "+v"(i), "+v"(half));  // a branch, and nothing formed of them is kept through the loop
#pragma unroll
        for (int jt = 0; jt < 2; jt++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const int j = j0 + jt * 32 + (r >> 2) * 8 + half * 4 + (r & 3);
            const bool ok = (j <= i) && (window < 0 || j >= i - window);
            st[jt][r] = ok ? st[jt][r] : -INFINITY;
          }
      }
      float mt = -INFINITY;
#pragma unroll
      for (int jt = 0; jt < 2; jt++)
#pragma unroll
        for (int r = 0; r < 16; r++) mt = fmaxf(mt, st[jt][r]);
      mt = half_swap_max(mt * sc2);
      // the reference of the exponentials moves when a row's maximum has grown by 2^8 (as in attn.hip)
      if (__builtin_amdgcn_ballot_w64(mt > mx + 8.f) != 0) {
        const float m_new = fmaxf(mx, mt);
        const float alpha = fexp2(mx - (m_new == -INFINITY ? 0.f : m_new));
        sum *= alpha;
        mx = m_new;
#pragma unroll
        for (int dt = 0; dt < W / 32; dt++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[dt][r] *= alpha;
      }
      const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int jt = 0; jt < 2; jt++)
#pragma unroll
        for (int r = 0; r < 16; r++) st[jt][r] = fexp2(__builtin_fmaf(st[jt][r], sc2, -ref));
#pragma unroll
      for (int u = 0; u < 4; u++) pb[u] = pack_bf16x8(st[u >> 1], (u & 1) * 8);
      float ps[16];  // the sum in fp32, pairwise
#pragma unroll
      for (int r = 0; r < 16; r++) ps[r] = st[0][r] + st[1][r];
#pragma unroll
      for (int w = 8; w > 0; w >>= 1)
#pragma unroll
        for (int r = 0; r < w; r++) ps[r] += ps[r + w];
      sum += ps[0];
    }
    part_ends<INS>();
    // ---- products
    if (m == 0) load(t + 3, stage);
    if (vis) {
      const unsigned char* sv = smem + (3 + stage) * TILE;
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int dt = 0; dt < W / 32; dt++) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa.load_tr(sv, u * 16, dt), pb[u], o[dt], 0, 0, 0);
    }
    if (t < t_hi && visible(t + 1)) scores(next);
    part_ends<INS>();
    stage = next;
  }
  if (m == 0) part_ends<0>();
  dma_wait_all();
  __syncthreads();

  const float total = half_swap_sum(sum);
  if constexpr (PART) {
    if (qi < S) {
      float* to = ch.to + ((((int64_t)b * H + h) * S + qi) * ch.n + part) * (2 * W + 4);
#pragma unroll
      for (int u = 0; u < W / 8; u++)
        *reinterpret_cast<f32x4*>(to + m * W + u * 8 + lhi * 4) = f32x4{o[u >> 2][(u & 3) * 4], o[u >> 2][(u & 3) * 4 + 1], o[u >> 2][(u & 3) * 4 + 2], o[u >> 2][(u & 3) * 4 + 3]};
      if (lhi == 0) {
        to[2 * W + m] = mx;
        to[2 * W + 2 + m] = total;
      }
    }
    return;
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
  const float lse = (mx + log2f(total)) * LN2;
  float zeros = lse * 0.f;  // NaN where something of a row is not finite; rows behind the sequence are none
  const float lam = LAM[z.shared ? 0 : h];
  float* lse_row = LSE + ((int64_t)b * H + h) * 2 * S;
  if (lhi == 0 && qi < S) lse_row[m * S + qi] = lse;
  // the second map's rows through LDS (its lanes own what the first one's do)
  f32x4* park = reinterpret_cast<f32x4*>(smem) + qw * (W / 8 * 64) + lane;
  if (m == 1) {
    bf16* o2p = O2 ? O2 + ((int64_t)b * S + qic) * z.ldo2 + h * W : nullptr;
#pragma unroll
    for (int u = 0; u < W / 8; u++) {
      f32x4 y;
      Pack4 pk;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        y[e] = o[u >> 2][(u & 3) * 4 + e] * inv;
        pk.e[e] = f2bf(y[e]);
        zeros = __builtin_fmaf(y[e], 0.f, zeros);
      }
      park[u * 64] = y;
      if (O2 && qi < S) *reinterpret_cast<u32x2*>(o2p + u * 8 + lhi * 4) = pk.u;
    }
    if (qi >= S) zeros = 0.f;
    reinterpret_cast<float*>(smem + QW * 32 * W * 4)[qw * 64 + lane] = zeros;
    if (__builtin_amdgcn_ballot_w64(zeros != 0.f)) dma_wait_all();  // the other wave of these rows is going to store them over
  }
  __syncthreads();
  if (m == 1) return;
  const float zeros2 = reinterpret_cast<float*>(smem + QW * 32 * W * 4)[qw * 64 + lane];
  zeros += zeros2;
  if (qi < S) {
    bf16* op = O + ((int64_t)b * S + qi) * z.ldo + h * W;
#pragma unroll
    for (int u = 0; u < W / 8; u++) {
      const f32x4 y = park[u * 64];
      Pack4 pk;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float x = __builtin_fmaf(o[u >> 2][(u & 3) * 4 + e], inv, -lam * y[e]);
        zeros = __builtin_fmaf(x, 0.f, zeros);
        pk.e[e] = f2bf(x);
      }
      *reinterpret_cast<u32x2*>(op + u * 8 + lhi * 4) = pk.u;
    }
  } else {
    zeros = 0.f;
  }
  const uint64_t bad2 = __builtin_amdgcn_ballot_w64(zeros2 != 0.f);
  redo_rows(zeros, [&](int r) {
    const int i = iw0 + r;
    const int64_t at = (int64_t)b * S + i;
    redo_fwd<W>(Q + at * z.ldq + h * W, kbase, z.ldk, vbase, z.ldv, lam, O + at * z.ldo + h * W, O2 ? O2 + at * z.ldo2 + h * W : nullptr, lse_row + i, S, i, window, z.scale, lane, ((bad2 | bad2 >> 32) >> r & 1) != 0);
  });
}

// Joins a row's chunks: a wave to a row, a lane to columns l and l + 64.  qr: queries of a workgroup of the first kernel.  Bound by the latency of loads that mostly hit the caches: 10 us for 1 x 8192
// tokens of one head of 64 (38 MB).
template <int W>
__global__ __launch_bounds__(256) void diff_attn_fwd_join_kernel(const bf16* __restrict__ Q, const bf16* __restrict__ K, const bf16* __restrict__ V, const float* __restrict__ LAM,
                                                                 bf16* __restrict__ O, bf16* __restrict__ O2, float* __restrict__ LSE, const Sizes z, const Chunks ch, int qr) {
  const int S = z.S, H = z.H, window = z.window, lane = threadIdx.x & 63;
  const int per = (S + 3) / 4, bh = blockIdx.x / per, i = blockIdx.x % per * 4 + (threadIdx.x >> 6);
  if (i >= S) return;
  const int b = bh / H, h = bh % H, kh = h / (H / z.KH);
  const int i0 = i / qr * qr;
  const int n = ((min(i0 + qr, S) - 1) / 64 - (window >= 0 ? max(0, i0 - window) : 0) / 64) / ch.size + 1;
  const float* from = ch.to + ((int64_t)bh * S + i) * ch.n * (2 * W + 4);
  const float lam = LAM[z.shared ? 0 : h];
  // lane c has the statistics of chunk c (there are at most 64); the chunks' loads do not wait for each other
  float y[2][W / 64] = {}, w[2], lse[2];
#pragma unroll
  for (int m = 0; m < 2; m++) {
    const float* st = from + min(lane, n - 1) * (2 * W + 4) + 2 * W + m;
    const float mine = lane < n ? st[0] : -INFINITY, mx = wave_max(mine);
    w[m] = fexp2(mine - mx);
    const float sum = wave_sum(lane < n ? w[m] * st[2] : 0.f);
    w[m] /= sum;
    lse[m] = (mx + log2f(sum)) * LN2;
  }
#pragma unroll 4
  for (int c = 0; c < n; c++) {
    const float* p = from + c * (2 * W + 4) + lane;
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
      for (int x = 0; x < W / 64; x++) y[m][x] = __builtin_fmaf(__shfl(w[m], c, 64), p[m * W + x * 64], y[m][x]);
  }
  const int64_t at = (int64_t)b * S + i;
  bf16 *o = O + at * z.ldo + h * W, *o2 = O2 ? O2 + at * z.ldo2 + h * W : nullptr;
  float* lse_row = LSE + (int64_t)bh * 2 * S + i;
  float zeros = lse[0] * 0.f, zeros2 = lse[1] * 0.f;
#pragma unroll
  for (int x = 0; x < W / 64; x++) {
    const float v = __builtin_fmaf(-lam, y[1][x], y[0][x]);
    zeros = __builtin_fmaf(v, 0.f, zeros);
    zeros2 = __builtin_fmaf(y[1][x], 0.f, zeros2);
    o[x * 64 + lane] = f2bf(v);
    if (O2) o2[x * 64 + lane] = f2bf(y[1][x]);
  }
  if (lane < 2) lse_row[lane * S] = lane ? lse[1] : lse[0];
  const bool bad2 = __builtin_amdgcn_ballot_w64(zeros2 != 0.f) != 0;
  if (__builtin_amdgcn_ballot_w64(zeros != 0.f) || bad2) {
    dma_wait_all();
    redo_fwd<W>(Q + at * z.ldq + h * W, K + (int64_t)b * S * z.ldk + kh * W, z.ldk, V + (int64_t)b * S * z.ldv + kh * W, z.ldv, lam, o, o2, lse_row, S, i, window, z.scale, lane, bad2);
  }
}

// ---------------------------------------------------------------------------------------
// dQ, dlambda and delta.  grid = ceil(S / 32 QW) H B workgroups of QW x KG waves; wave (qw, kg) owns 32 queries and every KG-th of their key tiles.  KG = 1 (QW = 4): two workgroups per CU, no merge.
// KG > 1 (QW = 2): a workgroup of 64 queries, four waves for heads of 64 (KG = 2; its LDS leaves room for one on a CU) and eight for heads of 32 (KG = 4), a wave with 1 / KG of the chain of tiles;
// what they have is added through LDS, in key-group order.  See q_split.
// The sums of P_m dP come out of the same sweep in fp32: dK/dV takes its delta from them, and dlambda is their sum: terms of both signs, that an error of 2^-9 in each would leave three digits of.
// dQ: 1 x 4096 tokens, 32/8 heads of 64: 255 us, 206 GFLOP at 810 TFLOP/s, bound by issue as the forward; fragments one product ahead 10 us more, four spill.
// For dQ they come too late, and it takes delta from the outputs as they were rounded, as dQ of attn.hip does; but where a workgroup has SWEEP key tiles or fewer, a sweep ahead forms them first.
// A row that sees few keys has most to lose: its dP - delta is small beside delta, and its gradients are the largest.  dQ's error as a share of its norm, and us of a backward pass, without the sweep,
// with, and with it everywhere (rounding dS and the result alone makes 0.0023): 5 tokens 0.0069, 0.0022; 3 x 333, 4/2 heads of 32 0.0031, 0.0025; 25.8, 29.4 us (30.9 where the tiles are fetched again); 1 x 1000, 8/4, window 333
// 0.0029, 0.0024; 46, 56 us; 1 x 4096, 32/8 0.0027, 0.0026, 0.0024; 609, 613, 777 us.
// STATS [B, H, 4, S]: what dK/dV takes of a row: lse_1 and lse_2 in powers of two, -delta_1, and -lambda (delta_1 - delta_2) (-lambda (dP - delta_2) is -lambda times what it has of the first map, plus this).  DLAM: a number for
// each workgroup, [B, H, tiles].
// ---------------------------------------------------------------------------------------
// A log-normaliser in powers of two is rounded, by up to 2^-24 of itself, and all of its row's probabilities are off by that: what their sums are multiplied by for it.
// (log2(e) is off as much in the scores' factor: the two cancel.)
__device__ __forceinline__ float mend(float lse, float l) { return __builtin_fmaf(-LN2, __builtin_fmaf(lse, LOG2E, -l), 1.f); }
struct Grad {
  int64_t lddo, lddq, lddk, lddv;
};
struct Lambda {
  const float* parts;
  float* dlam;
  int batch, tiles;
};
constexpr int SWEEP = 8;
// And where |lambda| is above SWEEP_WEIGHT: delta_1 is do . (o + lambda O_2), whose roundings are as large as lambda O_2 however small O_1 is.  Error of dq_1 as a share of its norm, by outputs and by
// the sweep, 4096 tokens, queries and keys of deviation 3 (1.5): lambda 0.5: 0.0059 (0.0027), 0.0024 (0.0024); 1: 0.0076 (0.0028); 2: 0.012 (0.0031); 5: 0.027 (0.0048); 30: 0.16 (0.024), with the
// sweep 0.0024 (0.0024) at any lambda.  us of a backward pass whose heads all sweep: 1 x 4096, 32/8 heads: 584, 752; 1 x 5000, 16/8, window 1024: 242, 301; dealt out, where each part sweeps the
// whole chain: 1 x 8192, 1/1: 132, 399.
constexpr float SWEEP_WEIGHT = 1.f;
template <int W, int QW, int KG, bool PART>
__global__ __launch_bounds__(QW * KG * 64, 2) void diff_attn_dq_kernel(const bf16* __restrict__ Q, const bf16* __restrict__ K, const bf16* __restrict__ V, const float* __restrict__ LAM,
                                                              const bf16* __restrict__ O, const bf16* __restrict__ O2, const float* __restrict__ LSE, const bf16* __restrict__ dO,
                                                              bf16* __restrict__ dQ, float* __restrict__ STATS, float* __restrict__ DLAM, const Sizes z, const Grad gr, const Chunks ch) {
  constexpr int TILE = 64 * W * 2, KS = W / 32;
  constexpr int QR = QW * 32;         // queries of the workgroup
  constexpr int TEAMS = QW * KG / 4;  // tiles are fetched by teams of 4 waves
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];  // [KG][2][K | V]
  __shared__ float red[QW * KG], sums[KG > 1 ? KG : 1][QR][2];
  const int S = z.S, H = z.H, KH = z.KH, window = z.window;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, lhi = lane >> 5;
  const int qw = wave % QW, kg = wave / QW, wv = wave & 3, team = wave >> 2;
  const int nqt = (S + QR - 1) / QR;
  const WgCoord wg = decode_wg(blockIdx.x, (int)(gridDim.x / ((PART ? ch.upto[ch.n - 1] : nqt) * (H / KH))), H / KH);
  const Place place = place_of<PART>(ch, wg.rank);
  const int qt = nqt - 1 - place.chain, part = place.part;
  const int b = wg.group / KH, kh = wg.group % KH;
  const int h = kh * (H / KH) + wg.r;
  const int i0 = qt * QR;
  const int iw0 = i0 + qw * 32;
  const int qi = iw0 + l32;
  const int qic = min(qi, S - 1);
  const float lam = LAM[z.shared ? 0 : h];
  int t_lo = (window >= 0 ? max(0, i0 - window) : 0) >> 6;
  int t_hi = min(i0 + QR - 1, S - 1) >> 6;
  const int all_lo = t_lo, all_hi = t_hi;
  if constexpr (PART) {
    t_lo += part * ch.size;
    if (t_lo > t_hi) return;
    t_hi = min(t_hi, t_lo + ch.size - 1);
  }

  const bf16* kbase = K + (int64_t)b * S * z.ldk + kh * W;
  const bf16* vbase = V + (int64_t)b * S * z.ldv + kh * W;
  const unsigned lds0 = lds_addr_of(smem);
  TileDma<64, W> dk, dv;
  dk.init(z.ldk, wv, lane);
  dv.init(z.ldv, wv, lane);
  // K/V tiles of round r: tile t_lo + r KG + g for key group g
  auto load_kv = [&](int t_lo, int t_hi, int round, int stage) {
#pragma unroll
    for (int g0 = 0; g0 < KG / TEAMS; g0++) {
      const int g = g0 * TEAMS + team, t = t_lo + round * KG + g;
      if (KG > 1 && t > t_hi) break;
      const unsigned dst = lds0 + (g * 2 + stage) * (2 * TILE);
      if (t * 64 + 64 <= S) {
        dk.issue(kbase + (int64_t)t * 64 * z.ldk, dst, wv);
        dv.issue(vbase + (int64_t)t * 64 * z.ldv, dst + TILE, wv);
      } else {
        dma_tile<64, W>(kbase, z.ldk, t * 64, S, dst, wv, lane);
        dma_tile<64, W>(vbase, z.ldv, t * 64, S, dst + TILE, wv, lane);
      }
    }
  };
  const bool sweeps = all_hi - all_lo < SWEEP || fabsf(lam) > SWEEP_WEIGHT;
  const int first_lo = sweeps ? all_lo : t_lo, first_hi = sweeps ? all_hi : t_hi;
  load_kv(first_lo, first_hi, 0, 0);

  bf16x8 qf[W / 16], dof[W / 16];
  float d1 = 0.f, d2 = 0.f;
  {
    const int64_t at = (int64_t)b * S + qic;
    const bf16* qp = Q + at * z.ldq + h * W + lhi * 8;
    const bf16* dp = dO + at * gr.lddo + h * W + lhi * 8;
    const bf16* op = O + at * z.ldo + h * W + lhi * 8;
    const bf16* o2p = O2 + at * z.ldo2 + h * W + lhi * 8;
#pragma unroll
    for (int s = 0; s < W / 16; s++) {
      qf[s] = *reinterpret_cast<const bf16x8*>(qp + s * 16);
      dof[s] = *reinterpret_cast<const bf16x8*>(dp + s * 16);
      const bf16x8 of = *reinterpret_cast<const bf16x8*>(op + s * 16), o2f = *reinterpret_cast<const bf16x8*>(o2p + s * 16);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        d1 += bf2f(of[e]) * bf2f(dof[s][e]);
        d2 += bf2f(o2f[e]) * bf2f(dof[s][e]);
      }
    }
  }
  arrived(qf);
  arrived(dof);
  d2 = half_swap_sum(d2);
  d1 = __builtin_fmaf(lam, d2, half_swap_sum(d1));  // o + lambda O_2 = O_1
  const int64_t row0 = ((int64_t)b * H + h) * 2 * S;
  const float l1 = LSE[row0 + qic] * LOG2E, l2 = LSE[row0 + S + qic] * LOG2E;
  const float sc2 = z.scale * LOG2E;
  FragAddr<W, W == 128> fa;  // (short of registers)
  fa.init(lane);

  float sum1 = 0.f, sum2 = 0.f;  // of P_m dP
  auto add_groups = [&] {  // the halves' sums, and the key groups', in their order
    sum1 = half_swap_sum(sum1);
    sum2 = half_swap_sum(sum2);
    if constexpr (KG > 1) {
      if (lhi == 0) {
        sums[kg][qw * 32 + l32][0] = sum1;
        sums[kg][qw * 32 + l32][1] = sum2;
      }
      __syncthreads();
      sum1 = sum2 = 0.f;
#pragma unroll
      for (int g = 0; g < KG; g++) {
        sum1 += sums[g][qw * 32 + l32][0];
        sum2 += sums[g][qw * 32 + l32][1];
      }
    }
  };
  dma_wait_all();
  __syncthreads();
  const int rounds = (t_hi - t_lo + KG) / KG;
  bool there = false;  // whether both stages have what the chain takes
  if (sweeps) {        // delta by a sweep ahead
    const int rounds = (all_hi - all_lo + KG) / KG;
    for (int round = 0; round < rounds; round++) {
      const int cur = round & 1;
      if (round + 1 < rounds) load_kv(all_lo, all_hi, round + 1, cur ^ 1);
      const int t = all_lo + round * KG + kg, j0 = t * 64;
      if ((KG == 1 || t <= all_hi) && j0 <= iw0 + 31 && (window < 0 || j0 + 63 >= iw0 - window)) {
        const unsigned char* sk = smem + (kg * 2 + cur) * (2 * TILE);
        const unsigned char* sv = sk + TILE;
        const bool need_mask = (j0 + 63 > iw0) || (window >= 0 && j0 < iw0 + 31 - window);
#pragma unroll 1
        for (int jt = 0; jt < 2; jt++) {
          f32x16 s1, s2, dp;
#pragma unroll
          for (int r = 0; r < 16; r++) s1[r] = s2[r] = dp[r] = 0.f;
#pragma unroll
          for (int s = 0; s < KS; s++) {
            s1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa.load_kc(sk, jt * 32, s), qf[s], s1, 0, 0, 0);
            s2 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa.load_kc(sk, jt * 32, KS + s), qf[KS + s], s2, 0, 0, 0);
          }
#pragma unroll
          for (int s = 0; s < 2 * KS; s++) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa.load_kc(sv, jt * 32, s), dof[s], dp, 0, 0, 0);
          if (need_mask)
            hide(s1, s2, lane, qi, [&](int k, int i) {
              const int j = j0 + jt * 32 + k;
              return j > i || (window >= 0 && j < i - window);
            });
          float t1 = 0.f, t2 = 0.f;
#pragma unroll
          for (int r = 0; r < 16; r++) {
            t1 = __builtin_fmaf(fexp2(__builtin_fmaf(s1[r], sc2, -l1)), dp[r], t1);
            t2 = __builtin_fmaf(fexp2(__builtin_fmaf(s2[r], sc2, -l2)), dp[r], t2);
          }
          sum1 += t1;
          sum2 += t2;
        }
      }
      dma_wait_all();
      __syncthreads();
    }
    add_groups();
    d1 = sum1;
    d2 = sum2;
    there = !PART && rounds <= 2;
    if (!there) {
      load_kv(t_lo, t_hi, 0, 0);
      dma_wait_all();
      __syncthreads();
    }
  }

  f32x16 dq[W / 32];
#pragma unroll
  for (int dt = 0; dt < W / 32; dt++)
#pragma unroll
    for (int r = 0; r < 16; r++) dq[dt][r] = 0.f;
  sum1 = sum2 = 0.f;


  for (int round = 0; round < rounds; round++) {
    const int cur = round & 1;
    if (round + 1 < rounds && !there) load_kv(t_lo, t_hi, round + 1, cur ^ 1);
    const int t = t_lo + round * KG + kg, j0 = t * 64;
    const bool visible = (KG == 1 || t <= t_hi) && j0 <= iw0 + 31 && (window < 0 || j0 + 63 >= iw0 - window);
    if (visible) {
      const unsigned char* sk = smem + (kg * 2 + cur) * (2 * TILE);
      const unsigned char* sv = sk + TILE;
      const bool need_mask = (j0 + 63 > iw0) || (window >= 0 && j0 < iw0 + 31 - window);
      // 48 products (W = 128) in six runs: scores and dP of either half of the tile's keys, then dQ of either.  The exponentials go between the products of dP, what is left of dS between those of
      // the next half's scores, or of dQ; each product's fragment is read two ahead, in a pinned order, as in dK/dV.
      constexpr int STEPS = 2 * KS, EL = 16 / STEPS, AHEAD = 2;
      f32x16 s1[2], s2[2], dp[2];
      bf16x8 ds1[2][2], ds2[2][2], fr[AHEAD + 1];
      float t1 = 0.f, t2 = 0.f;  // the sums of half a tile
      auto pin = [] { __builtin_amdgcn_sched_barrier(0); };
      auto fetch = [&](int n) {  // the fragment of product n
        const int run = n / STEPS, s = n % STEPS;
        if (run >= 4) return fa.load_tr(sk, (run - 4) * 32 + s / (W / 32) * 16, s % (W / 32));
        return fa.load_kc(run & 1 ? sv : sk, run / 2 * 32, s);
      };
      auto left = [&](int jt, int s) {
#pragma unroll
        for (int r = s * EL; r < (s + 1) * EL; r++) {
          t1 = r == 0 ? s1[jt][r] * dp[jt][r] : __builtin_fmaf(s1[jt][r], dp[jt][r], t1);
          t2 = r == 0 ? s2[jt][r] * dp[jt][r] : __builtin_fmaf(s2[jt][r], dp[jt][r], t2);
          ds1[jt][r >> 3][r & 7] = f2bf(s1[jt][r] * (dp[jt][r] - d1));
          ds2[jt][r >> 3][r & 7] = f2bf(s2[jt][r] * (dp[jt][r] - d2));
        }
        if (s + 1 == STEPS) {
          sum1 += t1;
          sum2 += t2;
        }
      };
      pin();
      each<AHEAD>([&](auto at) { fr[at] = fetch(at); });
      each<6 * STEPS>([&](auto at) {
        constexpr int n = decltype(at)::value, run = n / STEPS, s = n % STEPS, jt = run >= 4 ? run - 4 : run / 2;
        if (n + AHEAD < 6 * STEPS) fr[(n + AHEAD) % (AHEAD + 1)] = fetch(n + AHEAD);
        if (run >= 4) {
          constexpr int u = s / (W / 32), dt = s % (W / 32);
          dq[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[n % (AHEAD + 1)], dt < W / 64 ? ds1[jt][u] : ds2[jt][u], dq[dt], 0, 0, 0);
          if (run == 4) left(1, s);
        } else if (run & 1) {
          if (s == 0)
#pragma unroll
            for (int r = 0; r < 16; r++) dp[jt][r] = 0.f;
          dp[jt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[n % (AHEAD + 1)], dof[s], dp[jt], 0, 0, 0);
#pragma unroll
          for (int r = s * EL; r < (s + 1) * EL; r++) {
            s1[jt][r] = fexp2(__builtin_fmaf(s1[jt][r], sc2, -l1));
            s2[jt][r] = fexp2(__builtin_fmaf(s2[jt][r], sc2, -l2));
          }
          if (s + 1 == STEPS) asm volatile("" : "+v"(s1[jt]), "+v"(s2[jt]));  // (here: else they move behind the next branch)
        } else {
          if (s == 0)
#pragma unroll
            for (int r = 0; r < 16; r++) { s1[jt][r] = 0.f; s2[jt][r] = 0.f; }
          if (s < KS) s1[jt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[n % (AHEAD + 1)], qf[s], s1[jt], 0, 0, 0);
          else s2[jt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[n % (AHEAD + 1)], qf[s], s2[jt], 0, 0, 0);
          if (run == 2) left(0, s);
          if (run == 2 && s + 1 == STEPS) asm volatile("" : "+v"(ds1[0][0]), "+v"(ds1[0][1]), "+v"(ds2[0][0]), "+v"(ds2[0][1]), "+v"(sum1), "+v"(sum2));
        }
        pin();
        if (run < 4 && !(run & 1) && s + 1 == STEPS && need_mask)
          hide(s1[jt], s2[jt], lane, qi, [&](int k, int i) {
            const int j = j0 + jt * 32 + k;
            return j > i || (window >= 0 && j < i - window);
          });
      });
    }
    dma_wait_all();
    __syncthreads();
  }
  add_groups();
  if constexpr (PART) {
    if (qi < S) {
      float* to = ch.to + ((((int64_t)b * H + h) * S + qi) * ch.n + part) * (W + 4);
#pragma unroll
      for (int u = 0; u < W / 8; u++)
        *reinterpret_cast<f32x4*>(to + u * 8 + lhi * 4) = f32x4{dq[u >> 2][(u & 3) * 4], dq[u >> 2][(u & 3) * 4 + 1], dq[u >> 2][(u & 3) * 4 + 2], dq[u >> 2][(u & 3) * 4 + 3]};
      if (lhi == 0) {
        to[W] = sum1;
        to[W + 1] = sum2;
      }
    }
    return;
  }
  {
    const float* lse = LSE + row0 + min(iw0 + (lane_id() & 31), S - 1);
    sum1 *= mend(lse[0], l1);
    sum2 *= mend(lse[S], l2);
  }
  float zeros = 0.f;
  const float moves = z.scale * query_moves(qi, window);
  auto store4 = [&](int u, const f32x4& v) {
    Pack4 pk;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float x = v[e] * (u < W / 16 ? moves : -lam * moves);
      zeros = __builtin_fmaf(x, 0.f, zeros);
      pk.e[e] = f2bf(x);
    }
    *reinterpret_cast<u32x2*>(dQ + ((int64_t)b * S + qic) * gr.lddq + h * W + u * 8 + lhi * 4) = pk.u;
  };
  if constexpr (KG == 1) {
    if (qi < S) {
#pragma unroll
      for (int u = 0; u < W / 8; u++) store4(u, f32x4{dq[u >> 2][(u & 3) * 4], dq[u >> 2][(u & 3) * 4 + 1], dq[u >> 2][(u & 3) * 4 + 2], dq[u >> 2][(u & 3) * 4 + 3]});
    }
  } else {
    add_partials<W, KG>(smem, dq, qw, kg, lane, [&](int u, const f32x4& v) {
      if (qi < S) store4(u, v);
    });
  }
  if (qi < S) zeros = __builtin_fmaf(sum1, 0.f, __builtin_fmaf(sum2, 0.f, zeros));
  redo_rows(zeros, [&](int r) {
    const int i = iw0 + r;
    const int64_t at = (int64_t)b * S + i;
    float a, c;
    redo_dq<W>(Q + at * z.ldq + h * W, kbase, z.ldk, vbase, z.ldv, dO + at * gr.lddo + h * W, LSE[row0 + i], LSE[row0 + S + i], lam,
               dQ + at * gr.lddq + h * W, i, window, z.scale, lane, kg * (W / KG), (kg + 1) * (W / KG), a, c);
    sum1 = l32 == r ? a : sum1;
    sum2 = l32 == r ? c : sum2;
  });
  const bool counts = lhi == 0 && kg == 0 && qi < S;
  if (counts) {
    float* st = STATS + 2 * row0 + qi;
    st[0] = l1;
    st[S] = l2;
    st[2 * (int64_t)S] = -sum1;
    st[3 * (int64_t)S] = lam * (sum2 - sum1);
  }
  const float dl = block_sum<QW * KG>(counts ? sum2 : 0.f, red);
  if (tid == 0) DLAM[((int64_t)b * H + h) * nqt + qt] = -dl;
}

// Joins dQ's chunks: 16 waves, of 4 rows each, to 64 queries; a lane to columns l and l + 64.
template <int W>
__global__ __launch_bounds__(1024) void diff_attn_dq_join_kernel(const bf16* __restrict__ Q, const bf16* __restrict__ K, const bf16* __restrict__ V, const float* __restrict__ LAM,
                                                                const float* __restrict__ LSE, const bf16* __restrict__ dO,
                                                                bf16* __restrict__ dQ, float* __restrict__ STATS, float* __restrict__ DLAM, const Sizes z, const Grad gr, const Chunks ch, int qr) {
  __shared__ float red[16];
  const int S = z.S, H = z.H, window = z.window, lane = threadIdx.x & 63;
  const int per = (S + 63) / 64, bh = blockIdx.x / per;
  const int b = bh / H, h = bh % H, kh = h / (H / z.KH);
  const float lam = LAM[z.shared ? 0 : h];
  float total = 0.f;
  for (int r = 0; r < 4; r++) {
    const int i = blockIdx.x % per * 64 + r * 16 + (threadIdx.x >> 6);
    if (i >= S) break;
    const int i0 = i / qr * qr;
    const int n = ((min(i0 + qr, S) - 1) / 64 - (window >= 0 ? max(0, i0 - window) : 0) / 64) / ch.size + 1;
    const float* from = ch.to + ((int64_t)bh * S + i) * ch.n * (W + 4);
    float y[W / 64] = {}, sum1 = 0.f, sum2 = 0.f;
#pragma unroll 4
    for (int c = 0; c < n; c++, from += W + 4) {
#pragma unroll
      for (int x = 0; x < W / 64; x++) y[x] += from[x * 64 + lane];
      sum1 += from[W];
      sum2 += from[W + 1];
    }
    const int64_t at = (int64_t)b * S + i;
    bf16* dq = dQ + at * gr.lddq + h * W;
    const float* lse = LSE + (int64_t)bh * 2 * S + i;
    const float l1 = lse[0], l2 = lse[S];
    sum1 *= mend(l1, l1 * LOG2E);
    sum2 *= mend(l2, l2 * LOG2E);
    float zeros = (sum1 + sum2) * 0.f;
#pragma unroll
    for (int x = 0; x < W / 64; x++) {
      const float moves = z.scale * query_moves(i, window), v = y[x] * (x * 64 + lane < W / 2 ? moves : -lam * moves);
      zeros = __builtin_fmaf(v, 0.f, zeros);
      dq[x * 64 + lane] = f2bf(v);
    }
    if (__builtin_amdgcn_ballot_w64(zeros != 0.f)) {
      dma_wait_all();
      redo_dq<W>(Q + at * z.ldq + h * W, K + (int64_t)b * S * z.ldk + kh * W, z.ldk, V + (int64_t)b * S * z.ldv + kh * W, z.ldv, dO + at * gr.lddo + h * W, l1, l2, lam, dq, i, window, z.scale,
                 lane, 0, W, sum1, sum2);
    }
    if (lane < 4) STATS[((int64_t)bh * 4 + lane) * S + i] = lane == 0 ? l1 * LOG2E : lane == 1 ? l2 * LOG2E : lane == 2 ? -sum1 : lam * (sum2 - sum1);
    total += sum2;
  }
  const float dl = block_sum<16>(lane == 0 ? total : 0.f, red);
  if (threadIdx.x == 0) DLAM[blockIdx.x] = -dl;
}


// ---------------------------------------------------------------------------------------
// dK/dV.  grid = ceil(S / 32 KW) KH B workgroups of KW x QS waves; wave (kw, qs) owns 32 keys and every QS-th of the pairs of a query head of the group and one of its 32-row
// tiles from the diagonal on.  LDS: per query group 2 stages of (Q | dO | the 32 rows' statistics), then the fragments of V and K.
// 1 x 4096 tokens, 32/8 heads of 64 (2 x 4): 345 us, 275 GFLOP at 800 TFLOP/s, bound by issue: 272 vector and matrix instructions to 32 products.
// KW = 4, QS = 1: two workgroups per CU, no reduction.  KW = 2, QS = 4: one workgroup of eight waves per CU, half the keys and a quarter of the chain; the four partial sums are added through LDS
// in group order.  See dkv_split.
// ---------------------------------------------------------------------------------------
constexpr int smem_q(int W, int KG) { return KG * 2 * 2 * 64 * W * 2; }
// k-steps of K that lie in LDS, the last of the second map's (W = 128: with all in registers the loop spills, and a reload waits for the tiles under way; two workgroups of 4 x 1 find room on a CU with 3)
constexpr int k_parked(int W, int KW) { return W != 128 ? 0 : KW == 4 ? 3 : 4; }
constexpr int smem_kv(int W, int KW, int QS) {
  const int run = QS * 2 * (2 * 32 * W * 2 + 512) + KW * (W / 16 + k_parked(W, KW)) * 1024, sums = QS > 1 ? KW * QS * 32 * W * 4 : 0;
  return run > sums ? run : sums;
}
// dlambda of a head (or of all): dQ's sums, [B][H][tiles], in their order; the last workgroups, which have the least to do
template <int WAVES>
__device__ __forceinline__ void add_dlambda(const Lambda& la, int H, int shared, int wave) {
  __shared__ float red[WAVES];
  for (int64_t n = gridDim.x - 1 - blockIdx.x; n < (shared ? 1 : H); n += gridDim.x) {
    const int64_t per = (int64_t)la.tiles * (shared ? H : 1);
    const int lane = lane_id();
    float sum = 0.f;
    for (int c = 0; c < la.batch; c++) {
      const float* p = la.parts + ((int64_t)c * H + n) * la.tiles;
      for (int64_t i = wave * 64 + lane; i < per; i += WAVES * 64) sum += p[i];
    }
    sum = wave_sum(sum);
    __syncthreads();
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    sum = red[0];
    for (int w = 1; w < WAVES; w++) sum += red[w];
    if (wave == 0 && lane == 0) la.dlam[n] = sum;
  }
}
template <int W, int KW, int QS, bool PART>
__global__ __launch_bounds__(KW * QS * 64, 2) void diff_attn_dkv_kernel(const bf16* __restrict__ Q, const bf16* __restrict__ K, const bf16* __restrict__ V, const float* __restrict__ LAM,
                                                                        const float* __restrict__ STATS, const bf16* __restrict__ dO,
                                                                        bf16* __restrict__ dK, bf16* __restrict__ dV, const Sizes z, const Grad gr, const Lambda la, const Chunks ch) {
  constexpr int QT = 32, KS = W / 32;
  constexpr int TILE = QT * W * 2, STAGE = 2 * TILE + 512;
  constexpr int KT = KW * 32;         // keys of the workgroup
  constexpr int TEAMS = KW * QS / 4;  // tiles are fetched by teams of 4 waves
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int S = z.S, H = z.H, KH = z.KH, window = z.window;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, lhi = lane >> 5;
  const int kw = wave % KW, qs = wave / KW, wv = wave & 3, team = wave >> 2;
  const WgCoord wg = decode_wg(blockIdx.x, (int)(gridDim.x / (PART ? ch.upto[ch.n - 1] : (S + KT - 1) / KT)), 1);  // key tile 0 is seen by every query: longest first
  const int b = wg.group / KH, kh = wg.group % KH;
  const int rep = H / KH;
  const Place place = place_of<PART>(ch, wg.rank);
  const int j0 = place.chain * KT, part = place.part;
  const int jw0 = j0 + kw * 32;
  const int kj = jw0 + l32;  // this lane's key
  const int kjc = min(kj, S - 1);

  const int i_hi = window >= 0 ? min(S - 1, j0 + KT - 1 + window) : S - 1;
  const int t_lo = j0 / QT, t_hi = i_hi / QT;  // inclusive
  int total = (t_hi - t_lo + 1) * rep;
  if constexpr (PART) {
    if (part * ch.size >= total) return;
    total = min(total - part * ch.size, ch.size);
  }

  // K's and V's fragments of these keys: K's first in registers, the others in LDS, each the 1 KB that a read takes
  constexpr int PARKED = k_parked(W, KW), HELD = 2 * KS - PARKED, FIXED = 2 * KS + PARKED;
  const unsigned lds0 = lds_addr_of(smem);
  bf16x8 kf[HELD];
  {
    const bf16* kp = K + ((int64_t)b * S + kjc) * z.ldk + kh * W + lhi * 8;
    const bf16* vp = V + ((int64_t)b * S + kjc) * z.ldv + kh * W + lhi * 8;
    const unsigned dst = lds0 + QS * 2 * STAGE + kw * (FIXED * 1024);
#pragma unroll
    for (int s = 0; s < HELD; s++) kf[s] = *reinterpret_cast<const bf16x8*>(kp + s * 16);
    if (qs == 0) {
#pragma unroll
      for (int s = 0; s < 2 * KS; s++) dma16(vp + s * 16, dst + s * 1024);
#pragma unroll
      for (int s = 0; s < PARKED; s++) dma16(kp + (HELD + s) * 16, dst + (2 * KS + s) * 1024);
    }
  }
  f32x16 dk[W / 32], dv[W / 32];
#pragma unroll
  for (int dt = 0; dt < W / 32; dt++)
#pragma unroll
    for (int r = 0; r < 16; r++) { dk[dt][r] = 0.f; dv[dt][r] = 0.f; }

  const float sc2 = z.scale * LOG2E;
  const unsigned char* sgrp = smem + qs * (2 * STAGE);  // this query group's stages

  TileDma<QT, W> tq, tdo;
  tq.init(z.ldq, wv, lane);
  tdo.init(gr.lddo, wv, lane);
  // (tile, head) pairs, the last tile first and its heads next to each other: the workgroups of a K/V head, which begin at different tiles, read the same ones at the same time, out of one L2.
  // A group takes every QS-th pair; addresses move by a step, or by another one where the heads of a tile are done.
  struct Pair { int h, t; };
  const int dh = QS % rep, dt = QS / rep, n0 = PART ? place.part * ch.size : 0;
  auto first = [&](int n) { return Pair{(n0 + n) % rep, t_hi - (n0 + n) / rep}; };
  auto advance = [&](Pair& x) {
    x.h += dh;
    x.t -= dt;
    const bool next = x.h >= rep;
    if (next) {
      x.h -= rep;
      --x.t;
    }
    return next;
  };
  const int64_t q_step = dh * W - dt * QT * z.ldq, q_next = q_step - rep * W - QT * z.ldq, do_step = dh * W - dt * QT * gr.lddo, do_next = do_step - rep * W - QT * gr.lddo;
  const int64_t st_step = (int64_t)dh * 4 * S - dt * QT, st_next = st_step - (int64_t)rep * 4 * S - QT;
  // the next one to load of each query group this team fetches for, and of this wave's own group (its rows' statistics)
  Pair own = first(qs), ld[QS / TEAMS];
  const bf16 *q_at[QS / TEAMS], *do_at[QS / TEAMS];
  const float* st_at = STATS + ((int64_t)b * H + kh * rep + own.h) * 4 * S + own.t * QT;
#pragma unroll
  for (int g = 0; g < QS / TEAMS; g++) {
    ld[g] = first(g * TEAMS + team);
    const int64_t row = (int64_t)b * S + ld[g].t * QT, column = (kh * rep + ld[g].h) * W;
    q_at[g] = Q + row * z.ldq + column;
    do_at[g] = dO + row * gr.lddo + column;
  }
  auto load_tile = [&](int round, int stage) {
#pragma unroll
    for (int g = 0; g < QS / TEAMS; g++) {
      const int grp = g * TEAMS + team;
      if (QS > 1 && round * QS + grp >= total) break;
      const int t = ld[g].t;
      const unsigned dst = lds0 + (grp * 2 + stage) * STAGE;
      if (t * QT + QT <= S) {
        tq.issue(q_at[g], dst, wv);
        tdo.issue(do_at[g], dst + TILE, wv);
      } else {
        const int l = lane_id();
        dma_tile<QT, W>(q_at[g] - t * QT * z.ldq, z.ldq, t * QT, S, dst, wv, l);
        dma_tile<QT, W>(do_at[g] - t * QT * gr.lddo, gr.lddo, t * QT, S, dst + TILE, wv, l);
      }
      const bool next = advance(ld[g]);
      q_at[g] += next ? q_next : q_step;
      do_at[g] += next ? do_next : do_step;
    }
    if (kw == 0 && (QS == 1 || round * QS + qs < total)) {  // the rows' statistics: lanes 0 .. 31 the first of two, 32 .. 63 the second
      const int l = lane_id();
      const float* st = st_at + (int64_t)(l >> 5) * S + min(l & 31, S - 1 - own.t * QT);
      const unsigned dst = lds0 + (qs * 2 + stage) * STAGE + 2 * TILE;
      dma4(st, dst);
      dma4(st + 2 * (int64_t)S, dst + 256);
      st_at += advance(own) ? st_next : st_step;
    }
  };

  FragAddr<W, W == 128> fa;
  fa.init(lane);
  const unsigned char* fixed = smem + QS * 2 * STAGE + kw * (FIXED * 1024) + lane * 16;
  auto v_step = [&](int s) { return *reinterpret_cast<const bf16x8*>(fixed + s * 1024); };
  auto k_step = [&](int s) { return s < HELD ? kf[s < HELD ? s : 0] : v_step(2 * KS + s - HELD); };
  load_tile(0, 0);
  arrived(kf);
  dma_wait_all();
  __syncthreads();
  const int rounds = (total + QS - 1) / QS;
  Pair cur_it = first(qs);  // being consumed
  for (int round = 0; round < rounds; round++) {
    const int cur = round & 1;
    const bool more = round + 1 < rounds;
    if (more) load_tile(round + 1, cur ^ 1);
    const int ib = cur_it.t * QT;  // first query of the tile
    const bool visible = (QS == 1 || round * QS + qs < total) && (ib + QT - 1 >= jw0) && (window < 0 || ib <= jw0 + 31 + window);
    if (visible) {
      const float nlam = -LAM[z.shared ? 0 : kh * rep + cur_it.h];
      const unsigned char* sq = sgrp + cur * STAGE;
      const unsigned char* so = sq + TILE;
      const float* stats = reinterpret_cast<const float*>(sq + 2 * TILE);
      const bool need_mask = (ib < jw0 + 31) || (ib + QT > S) || (window >= 0 && ib + QT - 1 > jw0 + window);
      // A tile is 32 products (W = 128) in four runs: scores, dP, dV, dK.  The exponentials go between those of dP, what is left of dS between those of dV, and each product's fragments are read
      // some products ahead; the order is pinned, since the compiler's own reads so far ahead that it spills, and a reload waits for the tiles under way.
      constexpr int STEPS = 2 * KS, EL = 16 / STEPS;  // products of a run, rows of the vector work beside each
      constexpr int AP = 1, AV = 1, AK = 2;  // products that fragments are read ahead by, of dP, dV and dK
      static_assert(AV <= AP && AK < STEPS, "the first fragments of a run are read beside the last products of the one before");
      f32x16 s1, s2, dp;  // rows are queries ib + 8 (r / 4) + 4 lhi + r % 4; column: key kj
      bf16x8 w[2], ds1[2], ds2[2];
      auto pin = [] { __builtin_amdgcn_sched_barrier(0); };
      auto of4 = [&](int row, int r) { return stats[row * 32 + (r >> 2) * 8 + lhi * 4 + (r & 3)]; };
      auto tr_step = [&](const unsigned char* tile, int i) { return fa.load_tr(tile, i / (W / 32) * 16, i % (W / 32)); };
#pragma unroll
      for (int r = 0; r < 16; r++) { s1[r] = 0.f; s2[r] = 0.f; }
      pin();
      bf16x8 fq[STEPS], f2[KS], fo[AP + 1], fv[AP + 1], ft[AV + 1], fd[AK + 1];
#pragma unroll
      for (int s = 0; s < STEPS; s++) fq[s] = fa.load_kc(sq, 0, s);
#pragma unroll
      for (int s = 0; s < KS; s++) f2[s] = k_step(KS + s);
      pin();
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        if (s < KS) s1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fq[s], kf[s], s1, 0, 0, 0);
        else s2 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fq[s], f2[s - KS], s2, 0, 0, 0);
        if (s >= STEPS - AP) {
          fo[s - (STEPS - AP)] = fa.load_kc(so, 0, s - (STEPS - AP));
          fv[s - (STEPS - AP)] = v_step(s - (STEPS - AP));
        }
        pin();
      }
      if (need_mask) {
        const int l = lane_id();
        hide(s1, s2, l, jw0 + (l & 31), [&](int k, int j) {
          const int i = ib + k;
          return j > i || i >= S || (window >= 0 && j < i - window);
        });
      }
#pragma unroll
      for (int r = 0; r < 16; r++) dp[r] = of4(2, r);  // -delta_1
      pin();
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        if (s + AP < STEPS) {
          fo[(s + AP) % (AP + 1)] = fa.load_kc(so, 0, s + AP);
          fv[(s + AP) % (AP + 1)] = v_step(s + AP);
        } else if (s + AP - STEPS < AV) {
          ft[s + AP - STEPS] = tr_step(so, s + AP - STEPS);
        }
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fo[s % (AP + 1)], fv[s % (AP + 1)], dp, 0, 0, 0);
#pragma unroll
        for (int r = s * EL; r < (s + 1) * EL; r++) {
          s1[r] = fexp2(__builtin_fmaf(s1[r], sc2, -of4(0, r)));
          s2[r] = fexp2(__builtin_fmaf(s2[r], sc2, -of4(1, r)));
          w[r >> 3][r & 7] = f2bf(__builtin_fmaf(nlam, s2[r], s1[r]));
        }
        pin();
      }
#pragma unroll
      for (int i = 0; i < STEPS; i++) {
        if (i + AV < STEPS) ft[(i + AV) % (AV + 1)] = tr_step(so, i + AV);
        dv[i % (W / 32)] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ft[i % (AV + 1)], w[i / (W / 32)], dv[i % (W / 32)], 0, 0, 0);
#pragma unroll
        for (int r = i * EL; r < (i + 1) * EL; r++) {
          ds1[r >> 3][r & 7] = f2bf(s1[r] * dp[r]);
          ds2[r >> 3][r & 7] = f2bf(s2[r] * __builtin_fmaf(nlam, dp[r], of4(3, r)));
        }
        if (i >= STEPS - AK) fd[i - (STEPS - AK)] = tr_step(sq, i - (STEPS - AK));
        pin();
      }
#pragma unroll
      for (int i = 0; i < STEPS; i++) {
        const int dt = i % (W / 32);
        if (i + AK < STEPS) fd[(i + AK) % (AK + 1)] = tr_step(sq, i + AK);
        dk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fd[i % (AK + 1)], dt < W / 64 ? ds1[i / (W / 32)] : ds2[i / (W / 32)], dk[dt], 0, 0, 0);
        pin();
      }
    }
    advance(cur_it);
    dma_wait_all();
    __syncthreads();
  }
  const int le = lane_id(), ke = jw0 + (le & 31);
  if constexpr (PART) {
    if (ke < S) {
      float* to = ch.to + ((((int64_t)b * KH + kh) * S + ke) * ch.n + part) * (2 * W) + (le >> 5) * 4;
#pragma unroll
      for (int u = 0; u < W / 8; u++) {
        *reinterpret_cast<f32x4*>(to + u * 8) = f32x4{dk[u >> 2][(u & 3) * 4], dk[u >> 2][(u & 3) * 4 + 1], dk[u >> 2][(u & 3) * 4 + 2], dk[u >> 2][(u & 3) * 4 + 3]};
        *reinterpret_cast<f32x4*>(to + W + u * 8) = f32x4{dv[u >> 2][(u & 3) * 4], dv[u >> 2][(u & 3) * 4 + 1], dv[u >> 2][(u & 3) * 4 + 2], dv[u >> 2][(u & 3) * 4 + 3]};
      }
    }
    return;
  }
  bf16* kp = dK + ((int64_t)b * S + min(ke, S - 1)) * gr.lddk + kh * W;
  bf16* vp = dV + ((int64_t)b * S + min(ke, S - 1)) * gr.lddv + kh * W;
  float zeros = 0.f;
  const float moves = z.scale * key_moves(S, window);
  auto store4 = [&](bf16* p, int dt, int g, const f32x4& v, float mul) {
    Pack4 pk;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float x = v[e] * mul;
      zeros = __builtin_fmaf(x, 0.f, zeros);
      pk.e[e] = f2bf(x);
    }
    *reinterpret_cast<u32x2*>(p + dt * 32 + g * 8 + (le >> 5) * 4) = pk.u;
  };
  if constexpr (QS == 1) {
    if (ke < S) {
#pragma unroll
      for (int dt = 0; dt < W / 32; dt++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          store4(kp, dt, g, f32x4{dk[dt][g * 4], dk[dt][g * 4 + 1], dk[dt][g * 4 + 2], dk[dt][g * 4 + 3]}, moves);
          store4(vp, dt, g, f32x4{dv[dt][g * 4], dv[dt][g * 4 + 1], dv[dt][g * 4 + 2], dv[dt][g * 4 + 3]}, 1.f);
          __builtin_amdgcn_sched_barrier(0);  // a row leaves in order (see attn.hip)
        }
    }
  } else {
    // the stages are free: the last round ended in a barrier; dK first, then dV in the same space
    add_partials<W, QS>(smem, dk, kw, qs, le, [&](int u, const f32x4& v) {
      if (ke < S) store4(kp, u >> 2, u & 3, v, moves);
    });
    __syncthreads();
    add_partials<W, QS>(smem, dv, kw, qs, le, [&](int u, const f32x4& v) {
      if (ke < S) store4(vp, u >> 2, u & 3, v, 1.f);
    });
  }
  redo_rows(ke < S ? zeros : 0.f, [&](int r) {
    const int64_t seq = (int64_t)b * S, at = seq + jw0 + r, row = ((int64_t)b * H + kh * rep) * 4 * S;
    redo_dkv<W>(Q + seq * z.ldq + kh * rep * W, z.ldq, dO + seq * gr.lddo + kh * rep * W, gr.lddo, STATS + row, LAM + (z.shared ? 0 : kh * rep), z.shared ? 0 : 1,
                K + at * z.ldk + kh * W, V + at * z.ldv + kh * W, dK + at * gr.lddk + kh * W, dV + at * gr.lddv + kh * W, jw0 + r, S, rep, window, z.scale, le,
                qs * (W / QS), (qs + 1) * (W / QS));
  });
  add_dlambda<KW * QS>(la, H, z.shared, wave);
}

// Joins dK's and dV's chunks: a wave to a key.  kt: keys of a workgroup of the first kernel.
template <int W>
__global__ __launch_bounds__(256) void diff_attn_dkv_join_kernel(const bf16* __restrict__ Q, const bf16* __restrict__ K, const bf16* __restrict__ V, const float* __restrict__ LAM,
                                                                 const float* __restrict__ STATS, const bf16* __restrict__ dO, bf16* __restrict__ dK, bf16* __restrict__ dV, const Sizes z,
                                                                 const Grad gr, const Lambda la, const Chunks ch, int kt) {
  const int S = z.S, H = z.H, KH = z.KH, window = z.window, rep = H / KH, lane = threadIdx.x & 63;
  const int per = (S + 3) / 4, bk = blockIdx.x / per, j = blockIdx.x % per * 4 + (threadIdx.x >> 6);
  const int b = bk / KH, kh = bk % KH;
  if (j < S) {
    const int j0 = j / kt * kt, i_hi = window >= 0 ? min(S - 1, j0 + kt - 1 + window) : S - 1;
    const int n = ((i_hi / 32 - j0 / 32 + 1) * rep + ch.size - 1) / ch.size;
    const float* from = ch.to + ((int64_t)bk * S + j) * ch.n * (2 * W) + lane;
    float yk[W / 64] = {}, yv[W / 64] = {}, zeros = 0.f;
#pragma unroll 4
    for (int c = 0; c < n; c++, from += 2 * W)
#pragma unroll
      for (int x = 0; x < W / 64; x++) {
        yk[x] += from[x * 64];
        yv[x] += from[W + x * 64];
      }
    const int64_t seq = (int64_t)b * S, at = seq + j;
    bf16 *dk = dK + at * gr.lddk + kh * W, *dv = dV + at * gr.lddv + kh * W;
#pragma unroll
    for (int x = 0; x < W / 64; x++) {
      const float k = yk[x] * (z.scale * key_moves(S, window));
      zeros = __builtin_fmaf(k, 0.f, __builtin_fmaf(yv[x], 0.f, zeros));
      dk[x * 64 + lane] = f2bf(k);
      dv[x * 64 + lane] = f2bf(yv[x]);
    }
    if (__builtin_amdgcn_ballot_w64(zeros != 0.f)) {
      dma_wait_all();
      redo_dkv<W>(Q + seq * z.ldq + kh * rep * W, z.ldq, dO + seq * gr.lddo + kh * rep * W, gr.lddo, STATS + ((int64_t)b * H + kh * rep) * 4 * S, LAM + (z.shared ? 0 : kh * rep), z.shared ? 0 : 1,
                  K + at * z.ldk + kh * W, V + at * z.ldv + kh * W, dk, dv, j, S, rep, window, z.scale, lane, 0, W);
    }
  }
  add_dlambda<4>(la, H, z.shared, threadIdx.x >> 6);
}



int64_t tiles_of(int32_t S) { return ((int64_t)S + 127) / 128; }  // of 128 queries
// a number for 64 queries at least
int64_t parts_bytes(int32_t B, int32_t S, int32_t H) { return ((int64_t)B * H * (((int64_t)S + 63) / 64) * 4 + 255) / 256 * 256; }
int64_t stats_bytes(int32_t B, int32_t S, int32_t H) { return ((int64_t)B * H * 4 * S * 4 + 255) / 256 * 256; }

constexpr int64_t MAX_LD = 1 << 24;  // of a row, in elements: 64 rows are within reach of a 32-bit offset in bytes
// Whether rows of na and nb bf16 numbers at a and b share memory: exact for one row stride, as views of one buffer have it, otherwise whether their ranges meet.
bool meet(const void* a, int64_t lda, int64_t na, const void* b, int64_t ldb, int64_t nb, int64_t rows) {
  if (!a || !b) return false;
  const int64_t d = ((const char*)b - (const char*)a) / 2;
  if (d >= (rows - 1) * lda + na || -d >= (rows - 1) * ldb + nb) return false;
  const int64_t at = lda == ldb ? ((d % lda) + lda) % lda : 0;
  return at < na || at + nb > lda;
}
// The same of rows and a range of bytes, and of two ranges.
bool meet(const void* a, int64_t lda, int64_t na, int64_t rows, const void* range, int64_t bytes) {
  if (!a || !range || bytes <= 0) return false;
  const int64_t d = (const char*)range - (const char*)a, first = d > 0 ? d : 0, ld = 2 * lda, n = 2 * na, end = std::min(d + bytes, (rows - 1) * ld + n);
  return first < end && (first % ld < n || (first / ld + 1) * ld < end);
}
bool meet(const void* a, int64_t na, const void* b, int64_t nb) {
  return a && b && na > 0 && nb > 0 && (const char*)a < (const char*)b + nb && (const char*)b < (const char*)a + na;
}
bool rows_ok(const void* p, int64_t ld, int64_t width) { return aligned16(p) && ld % 8 == 0 && ld >= width && ld < MAX_LD; }

// rows, threads: queries and threads of a workgroup of the call's largest grid, which holds fewer than 2^32 threads
int check_shape(const char* name, int32_t B, int32_t S, int32_t H, int32_t KH, int32_t D, int rows, int threads) {
  OLMAX_CHECK(B > 0 && S > 0 && H > 0 && KH > 0 && H % KH == 0 && S <= (1 << 24) && H <= (1 << 16), OLMAX_ERR_SHAPE, "%s: bad shape B=%d S=%d H=%d KH=%d", name, B, S, H, KH);
  OLMAX_CHECK(((int64_t)S / 32 + 2) * (H / KH) < (1LL << 31), OLMAX_ERR_SHAPE, "%s: S=%d tokens of %d query heads to a key head are too many", name, S, H / KH);
  OLMAX_CHECK(D == 32 || D == 64, OLMAX_ERR_SHAPE, "%s: D must be 32 or 64 (got %d)", name, D);
  OLMAX_CHECK(((int64_t)S + rows - 1) / rows * H < (1LL << 32) / threads && ((int64_t)S + rows - 1) / rows * H * B < (1LL << 32) / threads, OLMAX_ERR_SHAPE,
              "%s: B=%d S=%d H=%d are too many rows", name, B, S, H);
  return OLMAX_OK;
}

// Forms of dQ and dK/dV.  us of a backward pass that takes one and the other of the two forms, bf16, causal, B x S, H/KH heads:
// dQ split over key groups (two of them, four for D = 32) where the workgroups of 128 queries would not fill 256 CUs: it halves the queries of a workgroup and its chain of key tiles, and its merge and one more
// barrier per tile are then free.  D = 64: 117 split, 133 whole (1 x 1000, 16/4); 122, 142 (1 x 2048, 16/16, 256 workgroups); with 512 of them 218, 196 (1 x 2048, 32/16).
// D = 32: 105, 121; 172, 158; 30.5, 33 (3 x 333, 4/2).
constexpr int QSW = 2;
constexpr int qs_groups(int W) { return W == 128 ? 2 : 4; }
bool q_split(int B, const Sizes& z) { return tiles_of(z.S) * z.H * B <= 256; }

// dK/dV split over query groups where the longest chain, of key tile 0 through all queries and heads of the group, would outlast the others' share of work: 4 x 1 has S / 128 KH B workgroups on
// 512 places, of half the longest chain's work on average.
// D = 64, 2 x 4 and 4 x 1: 617, 1053 (1 x 4096, 32/8: 256 workgroups of 4 x 1); 1209, 1349 (2 x 4096, 32/8: 512); 667, 586 (1 x 4096, 32/32: 1024); 1234, 1107 (1 x 8192, 16/16: 1024);
// window 512: 170, 178 (1 x 5000, 16/8: 320); 512, 431 (2 x 4000, 32/32: 2048).  D = 32: 418, 760; 797, 899; 457, 368; 849, 693.
// About the border, 1 x 4096 with 18/18, 20/20 and 22/22 heads (576, 640, 704): 387, 388; 414, 405; 451, 423; window 1024: 236, 219; 250, 251; 267, 267.  D = 32: 251, 254; 271, 263; 291, 270;
// window 1024: 153, 141; 163, 161; 176, 176.
bool dkv_split(int B, const Sizes& z) { return (int64_t)((z.S + 127) / 128) * z.KH * B <= 640; }
// and with one block of keys to eight query groups (D = 32: they find room in LDS) where the workgroups of two would not fill the GPU, or only just, and with chains of every length.
// 1 x 8 and 2 x 4: 43, 57 (1 x 600, 8/2: 20 workgroups of 2 x 4); 280, 341 (1 x 4096, 16/4: 256); 121, 97 (1 x 2048, 16/16: 512); window 512: 87, 78 (1 x 2000, 32/8: 256).
bool dkv_narrow(int B, const Sizes& z) { return (int64_t)((z.S + 63) / 64) * z.KH * B * (z.window < 0 ? 1 : 2) <= 256; }

// Form of the forward pass: workgroups of 64 queries (a wave to a SIMD; the turns are then between SIMDs and cost nothing) where those of 128 would leave half of the GPU empty, and for D = 32 always:
// a CU's LDS and registers hold three of those, and one of 128 queries.  us, 64 and 128 queries, B x S, H/KH heads: D = 64: 17.8, 21.0 (1 x 512, 8/8: 32 workgroups of 128);
// 29.3, 32.1 (1 x 1000, 16/4: 128); 57.1, 53.4 (1 x 2048, 16/16: 256); 120, 76 (1 x 2048, 32/8: 512).  D = 32: 23.1, 25.4 (1 x 1024, 8/8); 51.3, 52.7 (1 x 2048, 32/8); 162, 168 (1 x 4096, 32/8);
// 36.6, 42.1 (1 x 4000, 16/8, window 512).
template <int W>
bool fwd_halves(int B, const Sizes& z) { return W == 64 || tiles_of(z.S) * z.H * B <= 128; }

// Dealing chains out.  `tiles` chains of steps(i) steps to each of `heads`, on `places` workgroups that the GPU holds at once: chunks of `size` steps, the smallest size (4 at least) with which no
// workgroup waits for a place, since a second round costs as much as the first.  It is done where the longest chain, which without it is shared by `groups` groups of waves of one workgroup, gets
// shorter by `margin` steps, or else the chunks' way through memory and the second launch cost more.  us, dealt out and not, B x S, H/KH heads of 64 (32):
// forward, margin 20: 54, 162 (49, 136) 1 x 8192, 1/1; 39, 85 (36, 71) 1 x 4096, 2/1; 33, 47 (29, 39) 1 x 2048, 4/4; 43, 48 (40, 39) 1 x 2048, 8/2; below it 37, 29 (34, 24) 1 x 1000, 16/4.
// A backward pass with only dQ's dealt out, margin 12: 233, 327 (145, 179) 1 x 8192, 1/1; 211, 246 1 x 4096, 2/1; below it 115, 112 (65, 61) 1 x 1000, 4/1; 131, 121 (97, 81) 1 x 2048, 16/16.
// With only dK/dV's, margin 6 (steps of half the size): 375, 484 1 x 4096, 16/4; 106, 210 (67, 106) 1 x 2048, 8/2; 75, 116 (51, 61) 1 x 1000, 16/4; 38, 48 1 x 300, 4/1; below it
// 226, 206 (142, 131) 1 x 4096, 8/8; 687, 633 1 x 4096, 32/8; (92, 86) 1 x 4000, 8/2 of 32 with a window of 1024, where heads of 64, above it, take 137 dealt out and 157 not.
template <typename F>
Chunks plan_of(int64_t tiles, int64_t heads, int places, int groups, int margin, F steps) {  // steps(0) the longest chain's
  Chunks ch{nullptr, 0, 1, {}};
  ch.upto[0] = (int)tiles;
  if (tiles * heads > 2 * places) return ch;
  int64_t total = 0, longest = 0;
  for (int64_t i = 0; i < tiles; i++) {
    const int64_t n = steps(i);
    total += n * heads;
    longest = std::max(longest, n);
  }
  int64_t size = std::max({(total + places - 1) / places, (int64_t)4, (longest + MOST_CHUNKS - 1) / MOST_CHUNKS});
  for (; longest / groups - size >= margin; size += (size + 15) / 16) {
    int n = (int)((longest + size - 1) / size), sum = 0;
    for (int p = 0; p < n; p++) {
      int64_t last = tiles;
      while (last > 0 && steps(last - 1) <= p * size) last--;
      ch.upto[p] = sum += (int)last;
    }
    if (sum * heads > places) continue;
    ch.size = (int)size;
    ch.n = n;
    return ch;
  }
  ch.upto[0] = (int)tiles;
  return ch;
}
int64_t key_tiles(const Sizes& z, int64_t i0, int64_t qr) {  // of the workgroup of queries i0 .. i0 + qr - 1
  const int64_t hi = i0 + qr < z.S ? i0 + qr - 1 : z.S - 1, lo = z.window >= 0 && i0 > z.window ? i0 - z.window : 0;
  return hi / 64 - lo / 64 + 1;
}
int fwd_queries(int W) { return W == 64 ? 64 : 128; }
Chunks fwd_plan(int B, const Sizes& z, int W) {
  const int64_t qr = fwd_queries(W);
  return plan_of((z.S + qr - 1) / qr, (int64_t)z.H * B, W == 64 ? 512 : 256, 1, 20, [&](int64_t i) { return key_tiles(z, ((z.S + qr - 1) / qr - 1 - i) * qr, qr); });
}
Chunks dq_plan(int B, const Sizes& z, int W) {
  return plan_of(((int64_t)z.S + 127) / 128, (int64_t)z.H * B, 512, qs_groups(W), 12, [&](int64_t i) { return key_tiles(z, (((int64_t)z.S + 127) / 128 - 1 - i) * 128, 128); });
}
Chunks dkv_plan(int B, const Sizes& z, int W) {
  return plan_of(((int64_t)z.S + 127) / 128, (int64_t)z.KH * B, 512, W == 64 && dkv_narrow(B, z) ? 8 : 4, 6, [&](int64_t i) {
    const int64_t j0 = i * 128, hi = z.window >= 0 && j0 + 127 + z.window < z.S ? j0 + 127 + z.window : z.S - 1;
    return (hi / 32 - j0 / 32 + 1) * (z.H / z.KH);
  });
}
int64_t fwd_chunk_bytes(int B, const Sizes& z, int W) {
  const Chunks c = fwd_plan(B, z, W);
  return c.n < 2 ? 0 : (int64_t)B * z.H * z.S * c.n * (2 * W + 4) * 4;
}
int64_t bwd_chunk_bytes(int B, const Sizes& z, int W) {
  const Chunks q = dq_plan(B, z, W), k = dkv_plan(B, z, W);
  const int64_t nq = q.n < 2 ? 0 : (int64_t)B * z.H * z.S * q.n * (W + 4) * 4, nk = k.n < 2 ? 0 : (int64_t)B * z.KH * z.S * k.n * 2 * W * 4;
  return nq > nk ? nq : nk;
}

template <int W>
void fwd(hipStream_t stream, const bf16* q, const bf16* k, const bf16* v, const float* lam, bf16* o, bf16* o2, float* lse, float* workspace, int B, const Sizes& z) {
  constexpr int QW = W == 64 ? 2 : 4;
  static std::once_flag once;
  std::call_once(once, [] {
    (void)hipFuncSetAttribute((const void*)diff_attn_fwd_kernel<W, QW, false>, hipFuncAttributeMaxDynamicSharedMemorySize, smem_fwd(W));
    (void)hipFuncSetAttribute((const void*)diff_attn_fwd_kernel<W, 2, false>, hipFuncAttributeMaxDynamicSharedMemorySize, smem_fwd(W));
    (void)hipFuncSetAttribute((const void*)diff_attn_fwd_kernel<W, QW, true>, hipFuncAttributeMaxDynamicSharedMemorySize, smem_fwd(W));
  });
  Chunks ch = fwd_plan(B, z, W);
  ch.to = workspace;
  auto run = [&](auto kern, int qw) {
    hipLaunchKernelGGL(kern, dim3((unsigned)((ch.n > 1 ? ch.upto[ch.n - 1] : (int64_t)((z.S + 32 * qw - 1) / (32 * qw))) * z.H * B)), dim3(128 * qw), smem_fwd(W), stream, q, k, v, lam, o, o2, lse, z, ch);
  };
  if (ch.n > 1) {
    run(diff_attn_fwd_kernel<W, QW, true>, QW);
    hipLaunchKernelGGL(diff_attn_fwd_join_kernel<W>, dim3((unsigned)((int64_t)((z.S + 3) / 4) * z.H * B)), dim3(256), 0, stream, q, k, v, lam, o, o2, lse, z, ch, 32 * QW);
  } else if (fwd_halves<W>(B, z)) run(diff_attn_fwd_kernel<W, 2, false>, 2);
  else run(diff_attn_fwd_kernel<W, QW, false>, QW);
}

template <int W>
void bwd(hipStream_t stream, const bf16* q, const bf16* k, const bf16* v, const float* lam, const bf16* o, const bf16* o2, const float* lse, const bf16* d_o, bf16* dq, bf16* dk,
         bf16* dv, float* dlam, float* stats, float* parts, float* chunks, int B, const Sizes& z, const Grad& gr) {
  constexpr int QG = qs_groups(W);
  static std::once_flag once;
  std::call_once(once, [] {
    auto room = [](auto kern, int bytes) { (void)hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes); };
    room(diff_attn_dq_kernel<W, 4, 1, false>, smem_q(W, 1));
    room(diff_attn_dq_kernel<W, 4, 1, true>, smem_q(W, 1));
    room(diff_attn_dq_kernel<W, QSW, QG, false>, smem_q(W, QG));
    room(diff_attn_dkv_kernel<W, 4, 1, false>, smem_kv(W, 4, 1));
    room(diff_attn_dkv_kernel<W, 4, 1, true>, smem_kv(W, 4, 1));
    room(diff_attn_dkv_kernel<W, 2, 4, false>, smem_kv(W, 2, 4));
    if constexpr (W == 64) room(diff_attn_dkv_kernel<W, 1, 8, false>, smem_kv(W, 1, 8));
  });
  Chunks cq = dq_plan(B, z, W), ck = dkv_plan(B, z, W);
  cq.to = ck.to = chunks;  // (dK/dV's are written when dQ's have been joined)
  int tiles = 0;
  auto dq_of = [&](auto kern, int qw, int kg) {
    tiles = (z.S + 32 * qw - 1) / (32 * qw);
    hipLaunchKernelGGL(kern, dim3((unsigned)((int64_t)(cq.n > 1 ? cq.upto[cq.n - 1] : tiles) * z.H * B)), dim3(64 * qw * kg), smem_q(W, kg), stream, q, k, v, lam, o, o2, lse, d_o, dq, stats, parts, z, gr, cq);
  };
  if (cq.n > 1) {
    dq_of(diff_attn_dq_kernel<W, 4, 1, true>, 4, 1);
    tiles = (z.S + 63) / 64;
    hipLaunchKernelGGL(diff_attn_dq_join_kernel<W>, dim3((unsigned)((int64_t)tiles * z.H * B)), dim3(1024), 0, stream, q, k, v, lam, lse, d_o, dq, stats, parts, z, gr, cq, 128);
  } else if (q_split(B, z)) dq_of(diff_attn_dq_kernel<W, QSW, QG, false>, QSW, QG);
  else dq_of(diff_attn_dq_kernel<W, 4, 1, false>, 4, 1);
  const Lambda la{parts, dlam, B, tiles};
  auto kv = [&](auto kern, int kw, int qs) {
    hipLaunchKernelGGL(kern, dim3((unsigned)((ck.n > 1 ? ck.upto[ck.n - 1] : (int64_t)((z.S + 32 * kw - 1) / (32 * kw))) * z.KH * B)), dim3(64 * kw * qs), smem_kv(W, kw, qs), stream, q, k, v, lam, (const float*)stats, d_o,
                       dk, dv, z, gr, la, ck);
  };
  if (ck.n > 1) {
    kv(diff_attn_dkv_kernel<W, 4, 1, true>, 4, 1);
    hipLaunchKernelGGL(diff_attn_dkv_join_kernel<W>, dim3((unsigned)((int64_t)((z.S + 3) / 4) * z.KH * B)), dim3(256), 0, stream, q, k, v, lam, (const float*)stats, d_o, dk, dv, z, gr, la, ck, 128);
    return;
  }
  if constexpr (W == 64) {
    if (dkv_narrow(B, z)) return kv(diff_attn_dkv_kernel<W, 1, 8, false>, 1, 8);
  }
  if (dkv_split(B, z)) kv(diff_attn_dkv_kernel<W, 2, 4, false>, 2, 4);
  else kv(diff_attn_dkv_kernel<W, 4, 1, false>, 4, 1);
}

}  // namespace

// (shapes that the calls refuse need none)
static bool sizes_of(int32_t B, int32_t S, int32_t H, int32_t KH, int32_t D, int32_t window, Sizes& z) {
  if (B <= 0 || S <= 0 || H <= 0 || KH <= 0 || H % KH || (D != 32 && D != 64)) return false;
  z = Sizes{S, H, KH, window < 0 || window >= S ? -1 : window, 0, 0, 0, 0, 0, 0.f, 0};
  return true;
}
extern "C" int64_t olmax_diff_attn_fwd_workspace_bytes(int32_t B, int32_t S, int32_t H, int32_t KH, int32_t D, int32_t window) {
  Sizes z;
  return sizes_of(B, S, H, KH, D, window, z) ? fwd_chunk_bytes(B, z, 2 * D) : 0;
}
extern "C" int32_t olmax_diff_attn_fwd(hipStream_t stream, const void* q, const void* k, const void* v, const float* lam, void* o, void* o2, float* lse, void* workspace, int64_t workspace_bytes, int32_t B, int32_t S,
                                       int32_t H, int32_t KH, int32_t D, int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo, int64_t ldo2, int32_t lam_shared, int32_t window) {
  OLMAX_CHECK(q && k && v && lam && o && lse, OLMAX_ERR_ARG, "olmax_diff_attn_fwd: null pointer");
  if (int rc = check_shape("olmax_diff_attn_fwd", B, S, H, KH, D, D == 32 ? 64 : 128, D == 32 ? 256 : 512)) return rc;
  const int64_t W = 2 * D, rows = (int64_t)B * S;
  OLMAX_CHECK(rows_ok(q, ldq, H * W) && rows_ok(k, ldk, KH * W) && rows_ok(v, ldv, KH * W) && rows_ok(o, ldo, H * W) && (!o2 || rows_ok(o2, ldo2, H * W)), OLMAX_ERR_ALIGN,
              "olmax_diff_attn_fwd: operands must be 16-byte aligned, with row strides that are multiples of 8, at least heads * 2D and below 2^24");
  OLMAX_CHECK((((uintptr_t)lam | (uintptr_t)lse) & 3) == 0, OLMAX_ERR_ALIGN, "olmax_diff_attn_fwd: lam and lse not aligned to their type");
  const void* ins[] = {q, k, v};
  const int64_t ld_in[] = {ldq, ldk, ldv}, n_in[] = {H * W, KH * W, KH * W};
  for (int i = 0; i < 3; i++)
    OLMAX_CHECK(!meet(ins[i], ld_in[i], n_in[i], o, ldo, H * W, rows) && !meet(ins[i], ld_in[i], n_in[i], o2, ldo2, H * W, rows), OLMAX_ERR_ARG,
                "olmax_diff_attn_fwd: an output shares memory with an input");
  OLMAX_CHECK(!meet(o, ldo, H * W, o2, ldo2, H * W, rows), OLMAX_ERR_ARG, "olmax_diff_attn_fwd: o and o2 share memory");
  const Sizes z{S, H, KH, window < 0 || window >= S ? -1 : window, ldq, ldk, ldv, ldo, ldo2, 1.f / sqrtf((float)D), lam_shared != 0};
  const int64_t need = fwd_chunk_bytes(B, z, (int)W);
  OLMAX_CHECK(need == 0 || (workspace && workspace_bytes >= need && (((uintptr_t)workspace) & 15) == 0), OLMAX_ERR_WORKSPACE,
              "olmax_diff_attn_fwd: workspace needs %ld bytes, 16-byte aligned", (long)need);
  // what is not rows of heads
  struct { const void* p; int64_t n; } const flat[] = {{lse, (int64_t)B * H * 2 * S * 4}, {workspace, need}, {lam, (lam_shared ? 1 : H) * 4ll}};
  bool apart = !meet(lse, flat[0].n, workspace, need) && !meet(lse, flat[0].n, lam, flat[2].n) && !meet(workspace, need, lam, flat[2].n);
  for (const auto& f : flat) apart = apart && !meet(o, ldo, H * W, rows, f.p, f.n) && !meet(o2, ldo2, H * W, rows, f.p, f.n);
  for (int i = 0; i < 3; i++)
    for (int f = 0; f < 2; f++) apart = apart && !meet(ins[i], ld_in[i], n_in[i], rows, flat[f].p, flat[f].n);
  OLMAX_CHECK(apart, OLMAX_ERR_ARG, "olmax_diff_attn_fwd: lse, lam or the workspace shares memory with an output or an input");
  (D == 64 ? fwd<128> : fwd<64>)(stream, (const bf16*)q, (const bf16*)k, (const bf16*)v, lam, (bf16*)o, (bf16*)o2, lse, (float*)workspace, B, z);
  OLMAX_LAUNCH_CHECK();
  return OLMAX_OK;
}

// Workspace: the rows' statistics [B, H, 4, S], then dlambda's parts, up to [B, H, ceil(S / 64)], then the chunks of chains that are dealt out (dQ's, and in the same place dK/dV's), fp32
extern "C" int64_t olmax_diff_attn_bwd_workspace_bytes(int32_t B, int32_t S, int32_t H, int32_t KH, int32_t D, int32_t window) {
  Sizes z;
  return sizes_of(B, S, H, KH, D, window, z) ? stats_bytes(B, S, H) + parts_bytes(B, S, H) + bwd_chunk_bytes(B, z, 2 * D) : 0;
}

extern "C" int32_t olmax_diff_attn_bwd(hipStream_t stream, const void* q, const void* k, const void* v, const float* lam, const void* o, const void* o2, const float* lse,
                                       const void* d_o, void* dq, void* dk, void* dv, float* dlam, void* workspace, int64_t workspace_bytes, int32_t B, int32_t S, int32_t H,
                                       int32_t KH, int32_t D, int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo, int64_t ldo2, int64_t lddo, int64_t lddq, int64_t lddk,
                                       int64_t lddv, int32_t lam_shared, int32_t window) {
  OLMAX_CHECK(q && k && v && lam && o && o2 && lse && d_o && dq && dk && dv && dlam && workspace, OLMAX_ERR_ARG, "olmax_diff_attn_bwd: null pointer");
  if (int rc = check_shape("olmax_diff_attn_bwd", B, S, H, KH, D, 128, 256)) return rc;
  const int64_t W = 2 * D, rows = (int64_t)B * S;
  const void *ins[] = {q, k, v, o, o2, d_o}, *outs[] = {dq, dk, dv};
  const int64_t ld_in[] = {ldq, ldk, ldv, ldo, ldo2, lddo}, n_in[] = {H * W, KH * W, KH * W, H * W, H * W, H * W};
  const int64_t ld_out[] = {lddq, lddk, lddv}, n_out[] = {H * W, KH * W, KH * W};
  bool ok = true, apart = true;
  for (int i = 0; i < 6; i++) ok = ok && rows_ok(ins[i], ld_in[i], n_in[i]);
  for (int i = 0; i < 3; i++) ok = ok && rows_ok(outs[i], ld_out[i], n_out[i]);
  OLMAX_CHECK(ok, OLMAX_ERR_ALIGN, "olmax_diff_attn_bwd: operands must be 16-byte aligned, with row strides that are multiples of 8, at least heads * 2D and below 2^24");
  OLMAX_CHECK((((uintptr_t)lam | (uintptr_t)lse | (uintptr_t)dlam) & 3) == 0, OLMAX_ERR_ALIGN, "olmax_diff_attn_bwd: lam, lse and dlam not aligned to their type");
  const int64_t need = olmax_diff_attn_bwd_workspace_bytes(B, S, H, KH, D, window);
  OLMAX_CHECK(workspace_bytes >= need && (((uintptr_t)workspace) & 255) == 0, OLMAX_ERR_WORKSPACE, "olmax_diff_attn_bwd: workspace needs %ld bytes, 256-byte aligned", (long)need);
  for (int x = 0; x < 3; x++) {
    for (int i = 0; i < 6; i++) apart = apart && !meet(ins[i], ld_in[i], n_in[i], outs[x], ld_out[x], n_out[x], rows);
    for (int y = 0; y < x; y++) apart = apart && !meet(outs[y], ld_out[y], n_out[y], outs[x], ld_out[x], n_out[x], rows);
  }
  struct { const void* p; int64_t n; } const flat[] = {{dlam, (lam_shared ? 1 : H) * 4ll}, {workspace, need}, {lam, (lam_shared ? 1 : H) * 4ll}, {lse, (int64_t)B * H * 2 * S * 4}};  // two that are written
  for (int f = 0; f < 4; f++) {
    for (int x = 0; x < 3; x++) apart = apart && !meet(outs[x], ld_out[x], n_out[x], rows, flat[f].p, flat[f].n);
    for (int i = 0; i < 6 && f < 2; i++) apart = apart && !meet(ins[i], ld_in[i], n_in[i], rows, flat[f].p, flat[f].n);
    for (int g = 0; g < f && g < 2; g++) apart = apart && !meet(flat[g].p, flat[g].n, flat[f].p, flat[f].n);
  }
  OLMAX_CHECK(apart, OLMAX_ERR_ARG, "olmax_diff_attn_bwd: an output shares memory with an input or another output");
  const Sizes z{S, H, KH, window < 0 || window >= S ? -1 : window, ldq, ldk, ldv, ldo, ldo2, 1.f / sqrtf((float)D), lam_shared != 0};
  const Grad gr{lddo, lddq, lddk, lddv};
  (D == 64 ? bwd<128> : bwd<64>)(stream, (const bf16*)q, (const bf16*)k, (const bf16*)v, lam, (const bf16*)o, (const bf16*)o2, lse, (const bf16*)d_o, (bf16*)dq, (bf16*)dk, (bf16*)dv,
                                 dlam, (float*)workspace, (float*)((char*)workspace + stats_bytes(B, S, H)), (float*)((char*)workspace + stats_bytes(B, S, H) + parts_bytes(B, S, H)), B, z, gr);
  OLMAX_LAUNCH_CHECK();
  return OLMAX_OK;
}

extern "C" int32_t olmax_diff_attn_form(int32_t B, int32_t S, int32_t H, int32_t KH, int32_t D, int32_t window) {
  Sizes z;
  if (!sizes_of(B, S, H, KH, D, window, z)) return -1;
  const int W = 2 * D;
  const bool q_parts = dq_plan(B, z, W).n > 1, kv_parts = dkv_plan(B, z, W).n > 1, split = !q_parts && q_split(B, z), narrow = !kv_parts && D == 32 && dkv_narrow(B, z);
  const int64_t qr = split ? 32 * QSW : 128;
  int64_t chain = 0;
  for (int64_t i0 = 0; i0 < S; i0 += qr) chain = std::max(chain, key_tiles(z, i0, qr));
  const bool fwd_parts = fwd_plan(B, z, W).n > 1;
  const bool bits[] = {!fwd_parts && (D == 32 || fwd_halves<128>(B, z)), fwd_parts, split, q_parts, chain > SWEEP, !kv_parts && !narrow && dkv_split(B, z), narrow, kv_parts};
  int32_t form = 0;
  for (int i = 0; i < 8; i++) form |= bits[i] << i;
  return form;
}
