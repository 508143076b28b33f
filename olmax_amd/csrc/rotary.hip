// Rotary positions beyond the reference's (half layout, whole head, fp32 angles, position = row % seq_len; norm_rope.hip): tables for contexts longer than a model was
// trained on, half and interleaved pairs, part of a head, given positions.
//
// A pair (a, b) of columns turns by angle(p, i) = p f_i: (a cos - b sin, b cos + a sin); its gradient turns back.  Pairs are (i, i + R/2) in the half layout and
// (2i, 2i + 1) in the interleaved one, i < R/2; columns of a head from R on pass.  Rows are bf16 or fp32, tables and arithmetic fp32, rounded once.
#include "rows.h"
#include <algorithm>
#include <cmath>

namespace {

// ---- tables.  f_i = theta^(-2i/R), slowed down by kind:
//   1 all by the factor;  2 (llama3) those that turn less than `low` times in the original context by the factor, those that turn more than `high` times not, linearly in the
//   turns between;  3 (yarn) by the index, linearly between those of so many turns, `low` and `high` then (not up to low, by the factor from high on).
// The angle is formed in quarters of a turn and in 64 bits: at position 131072 fp32 leaves an error of 0.004.  A quarter's fraction, to the nearest, is exact, so that what fp32 adds is
// two Taylor polynomials on [-pi/4, pi/4], whose next terms are 2e-9 and 1.2e-10.
struct Scaling {
  int kind;
  double log_theta, factor, turns, low, high;  // turns: of an angle of 1 in the original context, L / 2 pi
};
__device__ __forceinline__ double quarters_per_position(int i, int rotary, const Scaling& c) {
  constexpr double TWO_OVER_PI = 0.63661977236758134308;
  const double f = exp(-2.0 * i / rotary * c.log_theta);
  double keep = 1.0;  // share that is not slowed down
  if (c.kind == 1) keep = 0.0;
  if (c.kind == 2) keep = fmin(fmax((f * c.turns - c.low) / (c.high - c.low), 0.0), 1.0);
  if (c.kind == 3) keep = 1.0 - fmin(fmax((i - c.low) / fmax(c.high - c.low, 0.001), 0.0), 1.0);
  return (keep * f + (1.0 - keep) * (f / c.factor)) * TWO_OVER_PI;
}

// The workgroup's frequencies lie in LDS; a thread has VEC columns and takes positions a grid apart.  Bound by the writes: 13.6 us for 131072 x 64 columns (67 MB, 4.9 TB/s; 15.9
// with a column and its frequency to a thread, 4 bytes a store); 13.9 to 14.2 with 1024 or 4096 workgroups.
template <int VEC>
__global__ __launch_bounds__(256) void rotary_tables_kernel(float* __restrict__ cos_t, float* __restrict__ sin_t, int64_t length, int half, const Scaling c, float size) {
  __shared__ double freq[256];  // (half is 256 at most)
  if (threadIdx.x < half) freq[threadIdx.x] = quarters_per_position(threadIdx.x, 2 * half, c);
  __syncthreads();
  const int across = half / VEC, per = 256 / across;  // threads and rows of a workgroup
  const int i = threadIdx.x % across * VEC, r = threadIdx.x / across;
  if (r >= per) return;
  double f[VEC];
#pragma unroll
  for (int e = 0; e < VEC; e++) f[e] = freq[i + e];
  for (int64_t p = (int64_t)blockIdx.x * per + r; p < length; p += (int64_t)gridDim.x * per) {
    float cs[VEC], sn[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      const double t = (double)p * f[e], quarter = rint(t);  // below 2^31: positions are, and f at most 2 / pi
      const float x = (float)((t - quarter) * 1.57079632679489661923), y = x * x;
      const float s = x + x * y * (-1.f / 6 + y * (1.f / 120 + y * (-1.f / 5040 + y * (1.f / 362880))));
      const float k = 1.f + y * (-0.5f + y * (1.f / 24 + y * (-1.f / 720 + y * (1.f / 40320 + y * (-1.f / 3628800)))));
      const int q = (int)quarter & 3;
      const float a = q & 1 ? s : k, b = q & 1 ? k : s;
      cs[e] = size * (q == 1 || q == 2 ? -a : a);
      sn[e] = size * (q >= 2 ? -b : b);
    }
    float *to_c = cos_t + p * half + i, *to_s = sin_t + p * half + i;
    if constexpr (VEC == 4) {
      *reinterpret_cast<f32x4*>(to_c) = f32x4{cs[0], cs[1], cs[2], cs[3]};
      *reinterpret_cast<f32x4*>(to_s) = f32x4{sn[0], sn[1], sn[2], sn[3]};
    } else {
      *to_c = cs[0];
      *to_s = sn[0];
    }
  }
}

// ---- rotation
struct Turn {
  const float *cos_t, *sin_t;  // [rows, half]
  const int32_t* positions;    // [tokens], or null: token % seq_len
  int64_t tokens, ldx, ldy;
  int heads, head_dim, half, rows, seq_len;
  float sign;                  // 1, or -1: back
};
// Position of a token: negative ones (padding) are not turned; one that the tables do not have comes out as NaN (`off`), and reads the last row.
__device__ __forceinline__ int position_of(const Turn& a, int64_t token, bool& off) {
  const int p = a.positions ? a.positions[token] : (int)(token % a.seq_len);
  off = p >= a.rows;
  return off ? a.rows - 1 : p;
}
__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
  const float t = x;
  x = __builtin_fmaf(t, c, -(y * s));
  y = __builtin_fmaf(y, c, t * s);
}

// Vectors of 16 bytes.  A unit is a place in a head: a vector pair (half layout) or a vector (interleaved) that turns, or a vector that passes.  A thread keeps a unit's cosines and sines in
// registers and takes every slots-th head, UNROLL at a time, so that the tables are read once for them and that many loads are in flight.
// Bound by HBM: 8192 tokens, 64 heads of 128 in bf16 (268 MB) 46 us, 5.8 TB/s; 1 token 2.3 us.
template <typename T, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(const T* x, T* y, const Turn a, int turning, int units, int slots, int per, int copies) {
  constexpr int N = rows::Vec<T>::N, UNROLL = 4, PAIRS = HALF ? N : N / 2;
  const int u = threadIdx.x % units, slot = threadIdx.x / units % slots, row = threadIdx.x / (units * slots);
  const int64_t token = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * per + row;
  if (row >= per || token >= a.tokens) return;
  bool off;
  const int p = position_of(a, token, off);
  const bool turns = u < turning;
  const T* xr = x + token * a.ldx;
  T* yr = y + token * a.ldy;
  if (!turns || p < 0) {
    if (!copies) return;
    const int at = turns ? u * N : 2 * a.half + (u - turning) * N;
    for (int h = slot; h < a.heads; h += slots) {
      const int64_t c = (int64_t)h * a.head_dim + at;
      *reinterpret_cast<u32x4*>(yr + c) = *reinterpret_cast<const u32x4*>(xr + c);
      if (HALF && turns) *reinterpret_cast<u32x4*>(yr + c + a.half) = *reinterpret_cast<const u32x4*>(xr + c + a.half);
    }
    return;
  }
  float c[PAIRS], s[PAIRS];
  const int64_t entry = (int64_t)p * a.half + u * PAIRS;
#pragma unroll
  for (int e = 0; e < PAIRS; e++) {
    c[e] = off ? NAN : a.cos_t[entry + e];
    s[e] = a.sign * a.sin_t[entry + e];
  }
  for (int h0 = slot; h0 < a.heads; h0 += UNROLL * slots) {
    u32x4 v[UNROLL], w[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; i++) {
      const int64_t at = (int64_t)min(h0 + i * slots, a.heads - 1) * a.head_dim + u * N;
      v[i] = *reinterpret_cast<const u32x4*>(xr + at);
      if (HALF) w[i] = *reinterpret_cast<const u32x4*>(xr + at + a.half);
    }
#pragma unroll
    for (int i = 0; i < UNROLL; i++) {
      if (h0 + i * slots >= a.heads) break;
      const int64_t at = (int64_t)(h0 + i * slots) * a.head_dim + u * N;
      float f[N], g[N];
      rows::Vec<T>::unpack(v[i], f);
      if (HALF) rows::Vec<T>::unpack(w[i], g);
#pragma unroll
      for (int e = 0; e < PAIRS; e++) turn(HALF ? f[e] : f[2 * e], HALF ? g[e] : f[2 * e + 1], c[e], s[e]);
      *reinterpret_cast<u32x4*>(yr + at) = rows::Vec<T>::pack(f);
      if (HALF) *reinterpret_cast<u32x4*>(yr + at + a.half) = rows::Vec<T>::pack(g);
    }
  }
}

// Any widths and alignment: a thread has one pair, or one column that passes.
template <typename T>
__global__ __launch_bounds__(256) void rotary_any_kernel(const T* x, T* y, const Turn a, bool half_layout) {
  const int per_head = a.head_dim - a.half;
  const int64_t n = a.tokens * a.heads * per_head;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < n; id += (int64_t)gridDim.x * 256) {
    const int i = (int)(id % per_head);
    const int64_t head = id / per_head, token = head / a.heads;
    const int64_t h = (head % a.heads) * a.head_dim;
    const T* xr = x + token * a.ldx + h;
    T* yr = y + token * a.ldy + h;
    if (i >= a.half) {
      yr[a.half + i] = xr[a.half + i];
      continue;
    }
    bool off;
    const int p = position_of(a, token, off);
    const int at = half_layout ? i : 2 * i, bt = half_layout ? i + a.half : 2 * i + 1;
    float f = (float)xr[at], g = (float)xr[bt];
    if (p >= 0) {
      const int64_t entry = (int64_t)p * a.half + i;
      turn(f, g, off ? NAN : a.cos_t[entry], a.sign * a.sin_t[entry]);
    }
    yr[at] = (T)f;
    yr[bt] = (T)g;
  }
}

constexpr int64_t MOST_GROUPS = 1 << 23;  // workgroups of 256 in a dimension of the grid
template <typename T>
void launch(hipStream_t stream, const T* x, T* y, const Turn& a, bool half_layout) {
  constexpr int N = rows::Vec<T>::N;
  const bool vec = aligned16(x) && aligned16(y) && a.ldx % N == 0 && a.ldy % N == 0 && a.head_dim % N == 0 && (half_layout ? a.half : 2 * a.half) % N == 0;
  const int turning = half_layout ? a.half / N : 2 * a.half / N, units = turning + (a.head_dim - 2 * a.half) / N;
  if (!vec || units > 256) {
    const int64_t n = a.tokens * a.heads * (a.head_dim - a.half);
    hipLaunchKernelGGL((rotary_any_kernel<T>), dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 16)), dim3(256), 0, stream, x, y, a, half_layout);
    return;
  }
  const int slots = std::min((a.heads + 3) / 4, 256 / units), per = 256 / (units * slots);
  const int64_t groups = (a.tokens + per - 1) / per;  // below 2^31; a dimension of the grid has room for 2^32 threads, less one
  const dim3 grid((unsigned)std::min(groups, MOST_GROUPS), (unsigned)((groups + MOST_GROUPS - 1) / MOST_GROUPS));
  const int copies = (const void*)x != (const void*)y;
  if (half_layout) hipLaunchKernelGGL((rotary_kernel<T, true>), grid, dim3(256), 0, stream, x, y, a, turning, units, slots, per, copies);
  else hipLaunchKernelGGL((rotary_kernel<T, false>), grid, dim3(256), 0, stream, x, y, a, turning, units, slots, per, copies);
}

int rotate(const char* name, float sign, hipStream_t stream, const void* x, void* y, const float* cos_t, const float* sin_t, const int32_t* positions, int64_t tokens, int32_t heads,
           int32_t head_dim, int32_t rotary_dim, int32_t table_rows, int32_t seq_len, int64_t ldx, int64_t ldy, int32_t layout, int32_t f32) {
  OLMAX_CHECK(tokens >= 0 && tokens < (1LL << 31) && heads > 0 && head_dim > 0 && heads <= (1 << 24) / head_dim, OLMAX_ERR_SHAPE, "%s: bad shape tokens=%ld heads=%d head_dim=%d",
              name, (long)tokens, heads, head_dim);
  OLMAX_CHECK(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim, OLMAX_ERR_SHAPE, "%s: rotary_dim must be even and up to head_dim=%d (got %d)", name, head_dim, rotary_dim);
  OLMAX_CHECK(layout == 0 || layout == 1, OLMAX_ERR_ARG, "%s: layout must be 0 (half) or 1 (interleaved)", name);
  OLMAX_CHECK(table_rows > 0 && (positions || (seq_len > 0 && seq_len <= table_rows)), OLMAX_ERR_SHAPE,
              "%s: without positions seq_len must be within 1 and the tables' %d rows (got %d)", name, table_rows, seq_len);
  if (tokens == 0) return OLMAX_OK;
  OLMAX_CHECK(x && y && cos_t && sin_t, OLMAX_ERR_ARG, "%s: null pointer", name);
  const int64_t width = (int64_t)heads * head_dim;
  if (tokens == 1) ldx = ldy = width;
  OLMAX_CHECK(ldx >= width && ldy >= width && ldx < (1LL << 31) && ldy < (1LL << 31), OLMAX_ERR_SHAPE, "%s: rows of %d x %d overlap, or are 2^31 and more apart (row strides %ld, %ld)",
              name, heads, head_dim, (long)ldx, (long)ldy);
  const int size = f32 ? 4 : 2;
  OLMAX_CHECK((((uintptr_t)x | (uintptr_t)y) & (size - 1)) == 0 && (((uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)positions) & 3) == 0, OLMAX_ERR_ALIGN,
              "%s: operands not aligned to their type", name);
  OLMAX_CHECK(x != y || ldx == ldy, OLMAX_ERR_ARG, "%s: in place wants one row stride", name);
  OLMAX_CHECK(!rows::overlap(x, ldx, y, ldy, tokens, width, size), OLMAX_ERR_ARG, "%s: the result overlaps the input, but is not in its place", name);
  const Turn a{cos_t, sin_t, positions, tokens, ldx, ldy, heads, head_dim, rotary_dim / 2, table_rows, seq_len, sign};
  if (f32) launch(stream, (const float*)x, (float*)y, a, layout == 0);
  else launch(stream, (const bf16*)x, (bf16*)y, a, layout == 0);
  OLMAX_LAUNCH_CHECK();
  return OLMAX_OK;
}

}  // namespace

extern "C" int32_t olmax_rotary_tables(hipStream_t stream, float* cos_t, float* sin_t, int64_t length, int32_t rotary_dim, double theta, int32_t kind, double factor,
                                       double original_length, double low, double high, float size) {
  OLMAX_CHECK(cos_t && sin_t, OLMAX_ERR_ARG, "olmax_rotary_tables: null pointer");
  OLMAX_CHECK(length > 0 && length < (1LL << 31) && rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= 512, OLMAX_ERR_SHAPE,
              "olmax_rotary_tables: length within 1 and 2^31 - 1 and an even rotary_dim up to 512 (got %ld, %d)", (long)length, rotary_dim);
  OLMAX_CHECK(theta > 1.0 && theta <= 1e30 && size > 0.f && size <= 1e30f, OLMAX_ERR_ARG, "olmax_rotary_tables: theta within 1 and 1e30, size positive");
  OLMAX_CHECK(kind >= 0 && kind <= 3, OLMAX_ERR_ARG, "olmax_rotary_tables: kind must be 0 (none), 1 (linear), 2 (llama3) or 3 (yarn)");
  OLMAX_CHECK(kind == 0 || (factor >= 1.0 && factor <= 1e6), OLMAX_ERR_ARG, "olmax_rotary_tables: factor within 1 and 1e6");
  OLMAX_CHECK(kind < 2 || (original_length >= 1.0 && original_length <= 2147483648.0), OLMAX_ERR_ARG, "olmax_rotary_tables: original_length within 1 and 2^31");
  OLMAX_CHECK(kind < 2 || (low > 0.0 && high > low && high <= 1e30), OLMAX_ERR_ARG, "olmax_rotary_tables: llama3 and yarn want 0 < low < high (turns in the original context)");
  constexpr double TWO_PI = 6.283185307179586477;
  Scaling c{kind, std::log(theta), factor, original_length / TWO_PI, low, high};
  if (kind == 3) {  // indices at which the original context has so many turns
    auto index = [&](double turns) { return rotary_dim * std::log(original_length / (turns * TWO_PI)) / (2.0 * c.log_theta); };
    c.low = std::max(std::floor(index(high)), 0.0);
    c.high = std::min(std::ceil(index(low)), rotary_dim - 1.0);
  }
  const int half = rotary_dim / 2;
  const bool wide = half % 4 == 0 && ((uintptr_t)cos_t & 15) == 0 && ((uintptr_t)sin_t & 15) == 0;
  const int per = 256 / (wide ? half / 4 : half);
  const dim3 grid((unsigned)std::min<int64_t>((length + per - 1) / per, 2048));
  if (wide) hipLaunchKernelGGL(rotary_tables_kernel<4>, grid, dim3(256), 0, stream, cos_t, sin_t, length, half, c, size);
  else hipLaunchKernelGGL(rotary_tables_kernel<1>, grid, dim3(256), 0, stream, cos_t, sin_t, length, half, c, size);
  OLMAX_LAUNCH_CHECK();
  return OLMAX_OK;
}

extern "C" int32_t olmax_rotary_fwd(hipStream_t stream, const void* x, void* y, const float* cos_t, const float* sin_t, const int32_t* positions, int64_t tokens, int32_t heads,
                                    int32_t head_dim, int32_t rotary_dim, int32_t table_rows, int32_t seq_len, int64_t ldx, int64_t ldy, int32_t layout, int32_t f32) {
  return rotate("olmax_rotary_fwd", 1.f, stream, x, y, cos_t, sin_t, positions, tokens, heads, head_dim, rotary_dim, table_rows, seq_len, ldx, ldy, layout, f32);
}

extern "C" int32_t olmax_rotary_bwd(hipStream_t stream, const void* dy, void* dx, const float* cos_t, const float* sin_t, const int32_t* positions, int64_t tokens, int32_t heads,
                                    int32_t head_dim, int32_t rotary_dim, int32_t table_rows, int32_t seq_len, int64_t lddy, int64_t lddx, int32_t layout, int32_t f32) {
  return rotate("olmax_rotary_bwd", -1.f, stream, dy, dx, cos_t, sin_t, positions, tokens, heads, head_dim, rotary_dim, table_rows, seq_len, lddy, lddx, layout, f32);
}
