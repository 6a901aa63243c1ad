// liboxb, entry points of products on 8-bit integers (gemm_int8.cuh).
#include "common.cuh"
#include "gemm_int8.cuh"
using namespace oxb;

// Rows of x [T, K] bf16 as int8 codes q (rows ld_q >= K bytes apart) with a scale per row
OXB_API int oxb_quantize_tokens(const void* x, int T, int K, void* q, int ld_q, float* scales, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (K <= 0 || ld_q < K) return (int)cudaErrorInvalidValue;
  oxb_launch(quantize_tokens_kernel, dim3(T), dim3(256), 0, stream, reinterpret_cast<const __nv_bfloat16*>(x), K, reinterpret_cast<int8_t*>(q),
             ld_q, scales);
  OXB_CHECK_LAUNCH();
  return 0;
}

template <int TN>
static int int8_go(const CUtensorMap& tw, const CUtensorMap& tx, const I8Args& a, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_int8_kernel<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, I8Tile<TN>::SMEM);
    if (e != cudaSuccess) return (int)e;
    configured[dev] = true;
  }
  const dim3 grid((a.N + I8_BM - 1) / I8_BM, 1, (a.T + TN - 1) / TN);
  if (grid.z > 65535) return (int)cudaErrorInvalidValue;
  const cudaError_t e = oxb_launch(gemm_int8_kernel<TN>, grid, dim3(I8_THREADS), (size_t)I8Tile<TN>::SMEM, stream, tw, tx, a);
  if (e != cudaSuccess) return (int)e;
  OXB_CHECK_LAUNCH();
  return 0;
}

// Y [T, N] bf16 (rows ld_y apart) from int8 codes xq [T, K] and w [N, K] (rows on 16-byte boundaries, ld bytes apart) with scales per
// row; bias [N] or null.  The sums are 32-bit: K <= 131072.
OXB_API int oxb_gemm_int8(const void* xq, int ld_x, const float* sx, const void* w, int ld_w, const float* sw, const float* bias, void* y,
                          int ld_y, int T, int N, int K, cudaStream_t stream) {
  if (T <= 0 || N <= 0) return 0;
  if (K <= 0 || K > 131072 || ld_y < N) return (int)cudaErrorInvalidValue;
  const int tn = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : T <= 128 ? 128 : 256;
  CUtensorMap tw, tx;
  int e = oxb_make_tmap_2d(&tw, w, N, K, ld_w, I8_BM, I8_BK, 1);
  if (!e) e = oxb_make_tmap_2d(&tx, xq, T, K, ld_x, tn, I8_BK, 1);
  if (e) return e;
  const I8Args a{reinterpret_cast<__nv_bfloat16*>(y), sx, sw, bias, N, T, K, ld_y, N % 8 == 0 && ld_y % 8 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0};
  switch (tn) {
    case 16: return int8_go<16>(tw, tx, a, stream);
    case 32: return int8_go<32>(tw, tx, a, stream);
    case 64: return int8_go<64>(tw, tx, a, stream);
    case 128: return int8_go<128>(tw, tx, a, stream);
    default: return int8_go<256>(tw, tx, a, stream);
  }
}
