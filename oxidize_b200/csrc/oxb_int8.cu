// liboxb, entry points of products on 8-bit integers (gemm_int8.cuh).
#include "common.cuh"
#include "gemm_int8.cuh"
using namespace oxb;

// Attributes of a kernel, set once per device; 0 or an error
template <typename F>
static int int8_configure(F* kernel, int smem, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
  if (!done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    done[dev] = true;
  }
  return 0;
}

static int quantize_launch(const __nv_bfloat16* x, int T, int K, int8_t* q, int ld_q, float* scales, cudaStream_t stream) {
  const int wide = K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const cudaError_t e = K <= 4096   ? oxb_launch(quantize_tokens_kernel<2>, dim3(T), dim3(256), 0, stream, x, K, wide, q, ld_q, scales)
                        : K <= 8192 ? oxb_launch(quantize_tokens_kernel<4>, dim3(T), dim3(256), 0, stream, x, K, wide, q, ld_q, scales)
                                    : oxb_launch(quantize_tokens_kernel<8>, dim3(T), dim3(256), 0, stream, x, K, wide, q, ld_q, scales);
  return (int)e;
}

// Tiles of 256 x 256 that come as halves: those of a last wave that would leave half of the SMs and more idle (4096 tokens of 14336 x 4096,
// 6 waves and 8 tiles: 244 us in a graph, 254 without)
static int int8_halved(long long tiles) {
  const int sms = oxb_sm_count(), last = (int)(tiles % sms);
  return tiles > sms && 2 * last <= sms ? last : 0;
}

template <int TN, int RB = 1>
static int int8_go(const CUtensorMap& tw, const CUtensorMap& tx, I8Args a, int splits, cudaStream_t stream) {
  static bool done[64] = {false};
  const int e = int8_configure(gemm_int8_kernel<TN, RB>, I8Tile<TN, RB>::SMEM, done);
  if (e) return e;
  a.token_tiles = (a.T + TN - 1) / TN;
  const long long tiles = (long long)((a.N + RB * I8_BM - 1) / (RB * I8_BM)) * a.token_tiles;
  if (tiles > (1 << 30)) return (int)cudaErrorInvalidValue;
  a.whole = RB == 2 ? (int)(tiles - int8_halved(tiles)) : 0;
  const dim3 grid(RB == 2 ? (int)(2 * tiles) - a.whole : (int)tiles, splits);
  return (int)(splits > 1 ? oxb_launch_cluster(gemm_int8_kernel<TN, RB>, grid, dim3(I8_THREADS), dim3(1, splits, 1), (size_t)I8Tile<TN, RB>::SMEM, stream, tw, tx, a)
                          : oxb_launch(gemm_int8_kernel<TN, RB>, grid, dim3(I8_THREADS), (size_t)I8Tile<TN, RB>::SMEM, stream, tw, tx, a));
}

// Tokens and blocks of 128 weight rows of a tile, CTAs that share its K
struct I8Plan {
  int tn, rb, splits;
};
static I8Plan int8_plan(int T, int N, int K) {
  const int sms = oxb_sm_count(), n_tiles = (N + 127) / 128, kbs = (K + I8_BK - 1) / I8_BK;
  if (T > 128) {
    // One CTA to an SM, in waves.  A tile's time in those of 128 x 256: 128 x 128 0.62, 256 x 256 1.75 (us with the three, 128 x 128
    // first: 512 tokens of 4096 x 4096 17.5, 22.4, 38; 1024 of 4096 x 4096 32, 26, 40; 1024 of 14336 x 4096 96, 84, 76; 8192 of
    // 8192 x 8192 623, 575, 474).
    auto waves = [&](int rows, int tokens) { return (int)(((long long)((N + rows - 1) / rows) * ((T + tokens - 1) / tokens) + sms - 1) / sms); };
    const int halved = int8_halved((long long)((N + 255) / 256) * ((T + 255) / 256));
    const double w1 = 0.62 * waves(128, 128), w2 = waves(128, 256), w4 = 1.75 * waves(256, 256) - (halved > 0 ? 0.75 : 0);
    return w4 <= w2 && w4 <= w1 ? I8Plan{256, 2, 1} : w2 <= w1 ? I8Plan{256, 1, 1} : I8Plan{128, 1, 1};
  }
  const int tn = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128;
  // Splits: as many as the SMs hold at a time (two CTAs of up to 64 tokens each), of 8 k-blocks and more; none where the weight tiles
  // alone nearly fill the SMs.  us with 1, 2, 4, 8: 16 tokens of 4096 x 14336 35, 22, 17, 16; 64 of 4096 x 4096 11.8, 12.0, 10.4,
  // 11.8; of 8192 x 8192 25, 21, 19, 29; of 14336 x 4096 16.4, 18.0, 25, 39.  128 tokens: large sums, so only for few tiles (4096 x 4096
  // 13.9, 16.9, 15.2, 36).
  int splits = 1;
  if (4 * n_tiles <= 3 * sms) splits = tn <= 64 ? 2 * sms / n_tiles : sms / (4 * n_tiles);
  splits = splits < kbs / 8 ? splits : kbs / 8;
  return {tn, 1, splits < 1 ? 1 : splits > 8 ? 8 : splits};
}

// Y [T, N] bf16 (rows ld_y apart) from x [T, K] bf16 (contiguous) and int8 codes w [N, K] (rows on 16-byte boundaries, ld_w bytes apart)
// with scales per row; bias [N] or null.  The sums are 32-bit: K <= 131072.  rows: scratch of T rows of K codes, each padded to 16 bytes, and
// T float scales behind them (may be null where oxb_int8_needs_rows is 0: one token of up to 40960 values); quantized: they are there from an
// earlier call on the same x.
OXB_API int oxb_int8_needs_rows(int T, int K) { return T > 1 || K > 40960; }
OXB_API int oxb_linear_int8(const void* x, int T, int K, void* rows, int quantized, const void* w, int ld_w, const float* sw, const float* bias,
                            void* y, int ld_y, int N, cudaStream_t stream) {
  if (T <= 0 || N <= 0) return 0;
  if (K <= 0 || K > 131072 || ld_y < N || ld_w % 16 != 0 || (reinterpret_cast<uintptr_t>(w) & 15) != 0) return (int)cudaErrorInvalidValue;
  const __nv_bfloat16* xb = reinterpret_cast<const __nv_bfloat16*>(x);
  __nv_bfloat16* yb = reinterpret_cast<__nv_bfloat16*>(y);
  int e = 0;
  if (!oxb_int8_needs_rows(T, K)) {
    const int wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    e = (int)oxb_launch(gemv_int8_kernel<4>, dim3((N + 31) / 32), dim3(256), (size_t)((K + 511) / 512 * 512), stream, xb, wide,
                        reinterpret_cast<const int8_t*>(w), ld_w, sw, bias, yb, N, K);
    if (e) return e;
    OXB_CHECK_LAUNCH();
    return 0;
  }
  if (rows == nullptr) return (int)cudaErrorInvalidValue;
  const int ld_q = (K + 15) / 16 * 16;
  int8_t* q = reinterpret_cast<int8_t*>(rows);
  float* scales = reinterpret_cast<float*>(q + (size_t)T * ld_q);
  if (!quantized) {
    e = quantize_launch(xb, T, K, q, ld_q, scales, stream);
    if (e) return e;
  }
  const I8Plan p = int8_plan(T, N, K);
  CUtensorMap tw, tx;
  e = oxb_make_tmap_2d(&tw, w, N, K, ld_w, I8_BM, I8_BK, 1);
  if (!e) e = oxb_make_tmap_2d(&tx, q, T, K, ld_q, p.tn, I8_BK, 1);
  if (e) return e;
  const I8Args a{yb, scales, sw, bias, N, T, K, ld_y, N % 8 == 0 && ld_y % 8 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0, 1, 0};
  switch (p.tn) {
    case 16: e = int8_go<16>(tw, tx, a, p.splits, stream); break;
    case 32: e = int8_go<32>(tw, tx, a, p.splits, stream); break;
    case 64: e = int8_go<64>(tw, tx, a, p.splits, stream); break;
    case 128: e = int8_go<128>(tw, tx, a, p.splits, stream); break;
    default: e = p.rb == 2 ? int8_go<256, 2>(tw, tx, a, 1, stream) : int8_go<256>(tw, tx, a, 1, stream); break;
  }
  if (e) return e;
  OXB_CHECK_LAUNCH();
  return 0;
}
