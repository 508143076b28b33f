// The LM head's products on fewer tokens than a tile of 256 has rows: the tokens are padded to a tile.
//
// 822 MB of weights at 4096 x 100352 take 160 us to read; below 256 tokens the forms that need no whole tile read them at 2 to 2.7 TB/s in dh (long reductions, few tiles) and write
// dW at 1.3 TB/s where there are fewer tokens than a k-tile has.  us as they are | padded, 4096 x 100352: logits of 192 tokens 307 | 216, gradients of 16
// tokens 1216 | 659, of 64 819 | 657, of 192 1113 | 748, distillation of 192 1115 | 802.
#include "rows.h"

namespace {

__global__ __launch_bounds__(256) void pad_rows_kernel(const bf16* __restrict__ src, bf16* __restrict__ dst, int64_t given, int64_t all) {  // in chunks of 8
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= all) return;
  u32x4 v = {0u, 0u, 0u, 0u};
  if (i < given) v = *(reinterpret_cast<const u32x4*>(src) + i);
  *(reinterpret_cast<u32x4*>(dst) + i) = v;
}

__global__ __launch_bounds__(256) void zero_rows_kernel(bf16* __restrict__ d, int64_t n, int64_t ld) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i < n) d[blockIdx.y * ld + i] = (bf16)0.f;
}

}  // namespace

// us, distillation of 63 tokens as they are | with gradients of 64: 9402 x 4096 118 | 84, 20000 x 4096 236 | 159, 2000 x 4096 41 | 38, 9402 x 1024 61 | 56, 20000 x 1024 103 | 79; narrow and small ones
// gain less (64 tokens for 63: 36000 x 256 70 for 72, 4096 x 1024 23 for 31) than the three launches that pad cost.
bool olmax_lmhead_pads_64(int64_t T, int32_t d, int32_t V) { return T < 64 && d % 8 == 0 && d >= 1024 && (int64_t)V * d >= 8000000 && !olmax_lmhead_pads(T, d, V); }

bool olmax_lmhead_pads(int64_t T, int32_t d, int32_t V) { return T < 256 && olmax_gemm_head_columns(256, V, d) > 0; }

void olmax_pad_rows(hipStream_t s, const bf16* src, bf16* dst, int64_t rows, int64_t padded, int d) {
  const int64_t all = padded * d / 8;
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)((all + 255) / 256)), dim3(256), 0, s, src, dst, rows * d / 8, all);
}

void olmax_zero_rows(hipStream_t s, bf16* d, int64_t from, int64_t to, int64_t n, int64_t ld) {
  if (to <= from || n <= 0) return;
  hipLaunchKernelGGL(zero_rows_kernel, dim3((unsigned)((n + 255) / 256), (unsigned)(to - from)), dim3(256), 0, s, d + from * ld, n, ld);
}

int olmax_lmhead_products_few(hipStream_t stream, const bf16* dlogits, const bf16* W, const bf16* h, const bf16* h_pad, bf16* dh, void* dW, int T, int d, int V, int64_t ldl,
                              bool dw_f32, bf16* tmp, int rows, GemmScratch scratch) {
  if (rows == 64) {
    if (int rc = olmax_lmhead_products(stream, dlogits, W, h_pad, dh ? tmp : nullptr, dW, 64, d, V, ldl, dw_f32, scratch)) return rc;
    if (dh) olmax_pad_rows(stream, tmp, dh, T, T, d);
    OLMAX_LAUNCH_CHECK();
    return OLMAX_OK;
  }
  if (dh) {  // (rows behind the tokens are products of whatever is there, and are left behind)
    if (int rc = olmax_gemm_padded(stream, dlogits, W, tmp, nullptr, 256, d, V, ldl, d, d, 0, true, false, false, true, scratch)) return rc;
    olmax_pad_rows(stream, tmp, dh, T, T, d);
  }
  if (dW) {
    const bool few = T < 64;
    if (int rc = olmax_gemm_padded(stream, dlogits, few ? h_pad : h, dW, nullptr, V, d, few ? 64 : T, ldl, d, d, 0, false, false, dw_f32, true, scratch)) return rc;
  }
  OLMAX_LAUNCH_CHECK();
  return OLMAX_OK;
}
