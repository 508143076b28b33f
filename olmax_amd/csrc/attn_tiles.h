// What the attention kernels share: rows of K, V, Q and dO as swizzled tiles in LDS, the fragments of v_mfma_f32_32x32x16_bf16 that are read from
// them in and against their storage order, and which workgroup takes which tile.
#pragma once
#include "common.h"

namespace {

__device__ __forceinline__ float fexp2(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// 16-byte chunk swizzle of the [rows][D] tiles.  ds_read_b128 serves the lane groups
// {0-3,12-15,20-23,24-27} / {4-7,8-11,16-19,28-31} (one row per lane, same logical chunk) per clock
// and the transposing ds_read_b64 serves lanes 0-31 (4 consecutive rows x 4 chunks); these masks give
// 16 distinct chunks modulo the 256-byte line of the 64 banks in both cases.  D = 128: a row is a
// line; D = 64: two rows share one, so the row's lowest bit already separates them, and bit 1 moves
// the transposed read's other two rows to the other half of their own.
template <int D>
__device__ __forceinline__ int swz(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row & 2) << 1) | ((row >> 2) & 3);
}

// Per-lane byte offsets of the operand fragments inside a [rows][D] tile.  The swizzle only
// looks at row bits 0-3, so stepping rows by 16 or 32 is a plain immediate offset and the
// D/16 (k-contiguous) plus D/16 (transposed) lane-dependent offsets are loop invariant.
// LEAN: the k-contiguous offsets are formed at each read from the first one (kc[s] = kc[0] ^ 32 s:
// the k-step only enters the XOR-swizzled chunk index) instead of living in registers, for a
// kernel that would otherwise spill them.
template <int D, bool LEAN = false>
struct FragAddr {
  int kc[LEAN ? 1 : D / 16];  // row (lane % 32), k-step s
  int tr[D / 32][2];          // column tile dt, half h of the transposed read
  __device__ __forceinline__ void init(int lane) {
    const int l32 = lane & 31, lhi = lane >> 5;
#pragma unroll
    for (int s = 0; s < (LEAN ? 1 : D / 16); s++) kc[s] = l32 * (2 * D) + (((2 * s + lhi) ^ swz<D>(l32)) << 4);
    const int j16 = lane & 15, g16 = lane >> 4;
#pragma unroll
    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int col = dt * 32 + ((g16 & 1) << 4) + ((j16 & 3) << 2);
        const int row = ((g16 >> 1) << 2) + (h << 3) + (j16 >> 2);
        tr[dt][h] = row * (2 * D) + (((col >> 3) ^ swz<D>(row)) << 4) + ((col & 7) << 1);
      }
  }
  // k-contiguous fragment: rows row0 + lane%32 (row0 multiple of 16), k-step s
  __device__ __forceinline__ bf16x8 load_kc(const unsigned char* tile, int row0, int s) const {
    int off = kc[LEAN ? 0 : s];
    if (LEAN) {
      asm volatile("" : "+v"(off));  // keeps the XOR at the read: hoisted out of the loop it is a register again
      off ^= s << 5;
    }
    return *reinterpret_cast<const bf16x8*>(tile + off + row0 * (2 * D));
  }
  // transposed fragment: MFMA rows = storage columns dt*32 + lane%32, k = storage rows r0 + {..}
  __device__ __forceinline__ bf16x8 load_tr(const unsigned char* tile, int r0, int dt) const {
    Pack8 p;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(tile + tr[dt][h] + r0 * (2 * D)));
      p.u[h * 2 + 0] = ((u32x2&)t)[0];
      p.u[h * 2 + 1] = ((u32x2&)t)[1];
    }
    return p.v;
  }
};

// Stream ROWS rows of D bf16 (global row r0 + i, clamped to S-1, row stride ld) into the
// swizzled LDS tile at lds_addr: DMA instructions of 1 KB (512/D rows) shared by 4 waves.
template <int ROWS, int D>
__device__ __forceinline__ void dma_tile(const bf16* base, int64_t ld, int r0, int S, unsigned lds_addr, int wave, int lane) {
#pragma unroll
  for (int i = 0; i < ROWS * D / 2048; i++) {
    const int blk = i * 4 + wave;
    const int p = blk * 64 + lane;
    const int row = p / (D / 8), ph = p % (D / 8);
    const int gr = min(r0 + row, S - 1);
    dma16(base + (int64_t)gr * ld + ((ph ^ swz<D>(row)) << 3), lds_addr + blk * 1024);
  }
}

// Workgroup id -> (tile rank, K/V group, head inside the group).  Hardware deals consecutive
// ids round-robin to the 8 XCDs and every XCD starts its ids in order, so the tile rank (the
// amount of causal work) is the SLOWEST index: each XCD gets the same mix of long and short
// tiles and starts the longest first (with the rank fastest, one XCD got 54 % more work than
// another and the CUs idled 39 % of the kernel).  When the group count divides by 8 the
// heads sharing a K/V head also land on one XCD, i.e. one L2.
struct WgCoord { int rank, group, r; };
__device__ __forceinline__ WgCoord decode_wg(int id, int ngroups, int rep) {
  const int level = ngroups * rep;
  WgCoord c;
  c.rank = id / level;
  const int u = id % level;
  if ((ngroups & 7) == 0) {
    const int blk = u / (8 * rep), rem = u % (8 * rep);
    c.r = rem >> 3;
    c.group = blk * 8 + (rem & 7);
  } else {
    c.group = u / rep;
    c.r = u % rep;
  }
  return c;
}

// The same tile transfer with everything lane-dependent hoisted out of the loop: a lane's byte
// offset (row * ld + swizzled chunk) inside the rows of one instruction of the four waves is computed
// once, and since the swizzle only looks at row bits 0-3 the DMA instructions of a transfer differ by
// a wave-uniform 2048/D rows, which go into the scalar base: one vector register per
// operand whatever the tile height.  Only for tiles that lie entirely inside the sequence (no
// row clamping).
template <int ROWS, int D>
struct TileDma {
  unsigned off;
  int64_t step;
  __device__ __forceinline__ void init(int64_t ld, int wave, int lane) {
    const int p = wave * 64 + lane;
    const int row = p / (D / 8), ph = p % (D / 8);
    off = (unsigned)((row * ld + ((ph ^ swz<D>(row)) << 3)) * 2);
    step = (2048 / D) * ld;
  }
  __device__ __forceinline__ void issue(const bf16* row0, unsigned lds_addr, int wave) const {
#pragma unroll
    for (int i = 0; i < ROWS * D / 2048; i++) dma16_s(row0 + i * step, off, lds_addr + (i * 4 + wave) * 1024);
  }
};

// acc + sum of the two bf16 values in dword w of a packed fragment
__device__ __forceinline__ float dot2_ones(const bf16x8& v, int w, float acc) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  const bf2 pair = {v[2 * w], v[2 * w + 1]};
  const bf2 ones = {(__bf16)1.0f, (__bf16)1.0f};
  return __builtin_amdgcn_fdot2_f32_bf16(pair, ones, acc, false);
}

__device__ __forceinline__ bf16x8 pack_bf16x8(const f32x16& a, int base) {
  bf16x8 r;
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = f2bf(a[base + e]);
  return r;
}


// Sum over the GROUPS waves that hold partial accumulators of the same 32 columns (column block c): every wave parks its D/8 units of 4 floats per lane in LDS, [c][group][unit][lane], and after a
// barrier adds its share of the units in group order and hands them to `out`.
template <int D, int GROUPS, typename Out>
__device__ __forceinline__ void add_partials(unsigned char* smem, const f32x16 (&acc)[D / 32], int c, int group, int lane, Out out) {
  constexpr int UNITS = D / 8, MINE = UNITS / GROUPS;
  static_assert(UNITS % GROUPS == 0, "units are dealt evenly to the groups");
  f32x4* park = reinterpret_cast<f32x4*>(smem) + c * (GROUPS * UNITS * 64) + lane;
#pragma unroll
  for (int u = 0; u < UNITS; u++)
    park[(group * UNITS + u) * 64] = f32x4{acc[u >> 2][(u & 3) * 4], acc[u >> 2][(u & 3) * 4 + 1], acc[u >> 2][(u & 3) * 4 + 2], acc[u >> 2][(u & 3) * 4 + 3]};
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MINE; i++) {
    const int u = group * MINE + i;
    f32x4 v = park[u * 64];
#pragma unroll
    for (int g = 1; g < GROUPS; g++) v += park[(g * UNITS + u) * 64];
    out(u, v);
  }
}

// calls row(r) for the rows r of a wave's 32 in which a lane's sum of zeros is not zero
template <typename Row>
__device__ __forceinline__ void redo_rows(float zeros, Row row) {
  const uint64_t bad = __builtin_amdgcn_ballot_w64(zeros != 0.f);
  if (bad) dma_wait_all();  // the wave's stores to the same rows, made by other lanes
  for (uint32_t rows = (uint32_t)bad | (uint32_t)(bad >> 32); rows; rows &= rows - 1) row(__builtin_ctz(rows));
}

}  // namespace
