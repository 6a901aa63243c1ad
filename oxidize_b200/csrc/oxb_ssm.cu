// liboxb, entry points of state-space layers (ssm.cuh).
#include "common.cuh"
#include "ssm.cuh"
using namespace oxb;

static bool ssm_dtype(int d) { return d == 0 || d == 2; }

template <typename TX, typename TY, int V, int K>
static int conv_go(const ConvArgs& a, int longest, cudaStream_t stream) {
  // single rows: one to a thread (decoding sequences share nothing); else the longest tiles that leave every SM threads
  const int blocks = (a.C + 128 * V - 1) / (128 * V), most = longest == 1 ? 1 : 64;
  int tt = most;
  while (tt > 8 && (long long)blocks * ((a.s.T + tt - 1) / tt) < 8LL * oxb_sm_count()) tt /= 2;
  const dim3 grid((a.s.T + tt - 1) / tt, blocks);
  if (blocks > 65535) return (int)cudaErrorInvalidValue;
  const cudaError_t e = tt == 1 ? oxb_launch(causal_conv_kernel<TX, TY, V, K, 1>, grid, dim3(128), 0, stream, a, tt)
                                : oxb_launch(causal_conv_kernel<TX, TY, V, K, 8>, grid, dim3(128), 0, stream, a, tt);
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

// Whether `cols` values of a row are whole 16-byte pieces on their boundaries, wherever the row starts
static bool ssm_wide(const SsmRows& m, int cols) {
  const int size = m.dtype == 0 ? 4 : 2;
  return m.p != nullptr && (reinterpret_cast<uintptr_t>(m.p) & 15) == 0 && ((long long)m.ld * size) % 16 == 0 && ((long long)cols * size) % 16 == 0;
}

template <int S>
static int scan_go(ScanArgs a, int longest, cudaStream_t stream) {
  const int channels = SCAN_THREADS / SCAN_L, blocks = (a.C + channels - 1) / channels;
  const SsmRows* rows[6] = {&a.u, &a.dt, &a.z, &a.b, &a.c, &a.y};
  a.wide = 0;
  for (int i = 0; i < 6; ++i) a.wide |= (ssm_wide(*rows[i], i == 3 || i == 4 ? a.N : a.C) ? 1 : 0) << i;
  constexpr int PIECE = S < 4 ? S : 4;
  if (a.N == SCAN_L * S && a.slot_stride % PIECE == 0 && (reinterpret_cast<uintptr_t>(a.state) % (4 * PIECE)) == 0) a.wide |= 64;
  cudaError_t e;
  if (longest == 1) {
    e = oxb_launch(selective_step_kernel<S>, dim3(blocks, (a.s.B + SCAN_L - 1) / SCAN_L), dim3(SCAN_THREADS), 0, stream, a);
  } else {
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
    if (!configured[dev]) {
      e = cudaFuncSetAttribute(selective_scan_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, ScanTile<S>::SMEM);
      if (e != cudaSuccess) return (int)e;
      configured[dev] = true;
    }
    e = oxb_launch(selective_scan_kernel<S>, dim3(blocks, a.s.B), dim3(SCAN_THREADS), (size_t)ScanTile<S>::SMEM, stream, a);
  }
  if (e != cudaSuccess) return (int)e;
  OXB_CHECK_LAUNCH();
  return 0;
}

// Selective scan of a step: u, dt, z, y of C channels and b, c of N <= 128 states, each a matrix of T rows with its own stride and
// dtype; a [C, N]; d, dt_bias [C] or null; z null: no gate.  The state [num_slots, C, N] float32 is read and updated.
// longest 1: every sequence feeds one row at most.
OXB_API int oxb_selective_scan(const void* u, int ld_u, int u_dtype, const void* dt, int ld_dt, int dt_dtype, const void* z, int ld_z,
                               int z_dtype, const void* b, int ld_b, int b_dtype, const void* c, int ld_c, int c_dtype, const float* a,
                               const float* d, const float* dt_bias, const int* query_start, const int* seq_lens, const int* slots,
                               float* state, long long slot_stride, int num_slots, void* y, int ld_y, int y_dtype, int B, int T, int C,
                               int N, int longest, cudaStream_t stream) {
  if (B <= 0 || T <= 0 || C <= 0) return 0;
  if (B > 65535 || N <= 0 || N > 128 || num_slots <= 0 || slots == nullptr || !ssm_dtype(u_dtype) || !ssm_dtype(dt_dtype) ||
      !ssm_dtype(z_dtype) || !ssm_dtype(b_dtype) || !ssm_dtype(c_dtype) || !ssm_dtype(y_dtype))
    return (int)cudaErrorInvalidValue;
  const ScanArgs s{{query_start, seq_lens, slots, B, T, num_slots}, {u, ld_u, u_dtype}, {dt, ld_dt, dt_dtype}, {z, ld_z, z_dtype},
                   {b, ld_b, b_dtype}, {c, ld_c, c_dtype}, {y, ld_y, y_dtype}, a, d, dt_bias, state, slot_stride, C, N, 0};
  if (N <= 8) return scan_go<1>(s, longest, stream);
  if (N <= 16) return scan_go<2>(s, longest, stream);
  if (N <= 32) return scan_go<4>(s, longest, stream);
  if (N <= 64) return scan_go<8>(s, longest, stream);
  return scan_go<16>(s, longest, stream);
}
