// liboxb, entry point of state-space layers' convolution (causal_conv.cuh).
#include "causal_conv.cuh"
using namespace oxb;

template <typename TX, typename TY, int V, int K>
static int conv_go(const ConvArgs& a, int longest, cudaStream_t stream) {
  // single rows: one to a thread (decoding sequences share nothing); else the longest tiles that leave every SM threads (7 prompts, 4096
  // channels: 48 us with tiles of 32 to 256 rows, 51 with 16), eight rows of a thread at a time in up to 64 bytes
  const int blocks = (a.C + 128 * V - 1) / (128 * V), most = longest == 1 ? 1 : 64;
  int tt = most;
  while (tt > 8 && (long long)blocks * ((a.s.T + tt - 1) / tt) < 8LL * oxb_sm_count()) tt /= 2;
  const dim3 grid((a.s.T + tt - 1) / tt, blocks);
  if (blocks > 65535) return (int)cudaErrorInvalidValue;
  const cudaError_t e = tt == 1 ? oxb_launch(causal_conv_kernel<TX, TY, V, K, 1>, grid, dim3(128), 0, stream, a, tt)
                                : oxb_launch(causal_conv_kernel<TX, TY, V, K, V * sizeof(TX) == 16 ? 4 : 8>, grid, dim3(128), 0, stream, a, tt);
  if (e != cudaSuccess) return (int)e;
  OXB_CHECK_LAUNCH();
  return 0;
}
template <typename TX, typename TY, int V>
static int conv_taps(const ConvArgs& a, int longest, cudaStream_t stream) {
  switch (a.taps) {
    case 1: return conv_go<TX, TY, V, 1>(a, longest, stream);
    case 2: return conv_go<TX, TY, V, 2>(a, longest, stream);
    case 3: return conv_go<TX, TY, V, 3>(a, longest, stream);
    default: return conv_go<TX, TY, V, 4>(a, longest, stream);
  }
}
template <typename TX, typename TY>
static int conv_types(const ConvArgs& a, int longest, cudaStream_t stream) {
  const bool wide = a.C % 4 == 0 && a.x.ld % 4 == 0 && a.y.ld % 4 == 0 && a.slot_stride % 4 == 0 &&
                    (reinterpret_cast<uintptr_t>(a.x.p) % (4 * sizeof(TX))) == 0 && (reinterpret_cast<uintptr_t>(a.y.p) % (4 * sizeof(TY))) == 0 &&
                    ((reinterpret_cast<uintptr_t>(a.window) | reinterpret_cast<uintptr_t>(a.w)) & 15) == 0;
  return wide ? conv_taps<TX, TY, 4>(a, longest, stream) : conv_taps<TX, TY, 1>(a, longest, stream);
}

// Short causal convolution of a step: x [T, ld_x] and y [T, ld_y] of C channels (dtype codes 0 float32, 2 bfloat16), w [C, taps],
// bias [C] or null, the ring [num_slots, taps, C] float32 (slots `slot_stride` values apart) read and updated; longest: rows of
// the sequence that feeds most.
OXB_API int oxb_causal_conv(const void* x, int ld_x, int x_dtype, const float* w, const float* bias, const int* query_start,
                            const int* seq_lens, const int* slots, float* window, long long slot_stride, int num_slots, void* y, int ld_y,
                            int y_dtype, int B, int T, int C, int taps, int silu, int longest, cudaStream_t stream) {
  if (B <= 0 || T <= 0 || C <= 0) return 0;
  if (B > 65535 || taps <= 0 || num_slots <= 0 || !ssm_dtype(x_dtype) || !ssm_dtype(y_dtype) || slots == nullptr)
    return (int)cudaErrorInvalidValue;
  const ConvArgs a{{query_start, seq_lens, slots, B, T, num_slots}, {x, ld_x, x_dtype}, {y, ld_y, y_dtype}, w, bias, window, slot_stride, C, taps, silu};
  if (taps <= 4) {
    if (x_dtype == 0) return y_dtype == 0 ? conv_types<float, float>(a, longest, stream) : conv_types<float, __nv_bfloat16>(a, longest, stream);
    return y_dtype == 0 ? conv_types<__nv_bfloat16, float>(a, longest, stream) : conv_types<__nv_bfloat16, __nv_bfloat16>(a, longest, stream);
  }
  const int tiles = (C + 255) / 256;
  if (tiles > 65535) return (int)cudaErrorInvalidValue;
  oxb_launch(causal_conv_any_kernel, dim3(T, tiles), dim3(256), 0, stream, a);
  OXB_CHECK_LAUNCH();
  oxb_launch(conv_window_kernel, dim3(tiles, B), dim3(256), 0, stream, a);
  OXB_CHECK_LAUNCH();
  return 0;
}
