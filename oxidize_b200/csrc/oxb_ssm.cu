// liboxb, entry points of state-space layers (ssm.cuh).
#include "common.cuh"
#include "ssm.cuh"
using namespace oxb;

static bool ssm_dtype(int d) { return d == 0 || d == 2; }

// Short causal convolution of a step: x [T, ld_x] and y [T, ld_y] of C channels (dtype codes 0 float32, 2 bfloat16), w [C, taps],
// bias [C] or null, the ring [num_slots, taps, C] float32 (slots `slot_stride` values apart) read and updated.
OXB_API int oxb_causal_conv(const void* x, int ld_x, int x_dtype, const float* w, const float* bias, const int* query_start,
                            const int* seq_lens, const int* slots, float* window, long long slot_stride, int num_slots, void* y, int ld_y,
                            int y_dtype, int B, int T, int C, int taps, int silu, cudaStream_t stream) {
  if (B <= 0 || T <= 0 || C <= 0) return 0;
  if (B > 65535 || taps <= 0 || num_slots <= 0 || !ssm_dtype(x_dtype) || !ssm_dtype(y_dtype) || slots == nullptr)
    return (int)cudaErrorInvalidValue;
  const ConvArgs a{{query_start, seq_lens, slots, B, T, num_slots}, {x, ld_x, x_dtype}, {y, ld_y, y_dtype}, w, bias, window, slot_stride, C, taps, silu};
  const int tiles = (C + 255) / 256;
  if (tiles > 65535) return (int)cudaErrorInvalidValue;
  oxb_launch(causal_conv_kernel, dim3(T, tiles), dim3(256), 0, stream, a);
  OXB_CHECK_LAUNCH();
  oxb_launch(conv_window_kernel, dim3(tiles, B), dim3(256), 0, stream, a);
  OXB_CHECK_LAUNCH();
  return 0;
}

template <int L, int S>
static int scan_go(const ScanArgs& a, cudaStream_t stream) {
  oxb_launch(selective_scan_kernel<L, S>, dim3((a.C + 128 / L - 1) / (128 / L), a.s.B), dim3(128), 0, stream, a);
  OXB_CHECK_LAUNCH();
  return 0;
}

// Selective scan of a step: u, dt, z, y of C channels and b, c of N <= 128 states, each a matrix of T rows with its own stride and
// dtype; a [C, N]; d, dt_bias [C] or null; z null: no gate.  The state [num_slots, C, N] float32 is read and updated.
OXB_API int oxb_selective_scan(const void* u, int ld_u, int u_dtype, const void* dt, int ld_dt, int dt_dtype, const void* z, int ld_z,
                               int z_dtype, const void* b, int ld_b, int b_dtype, const void* c, int ld_c, int c_dtype, const float* a,
                               const float* d, const float* dt_bias, const int* query_start, const int* seq_lens, const int* slots,
                               float* state, long long slot_stride, int num_slots, void* y, int ld_y, int y_dtype, int B, int T, int C,
                               int N, cudaStream_t stream) {
  if (B <= 0 || T <= 0 || C <= 0) return 0;
  if (B > 65535 || N <= 0 || N > 128 || num_slots <= 0 || slots == nullptr || !ssm_dtype(u_dtype) || !ssm_dtype(dt_dtype) ||
      !ssm_dtype(z_dtype) || !ssm_dtype(b_dtype) || !ssm_dtype(c_dtype) || !ssm_dtype(y_dtype))
    return (int)cudaErrorInvalidValue;
  const ScanArgs s{{query_start, seq_lens, slots, B, T, num_slots}, {u, ld_u, u_dtype}, {dt, ld_dt, dt_dtype}, {z, ld_z, z_dtype},
                   {b, ld_b, b_dtype}, {c, ld_c, c_dtype}, {y, ld_y, y_dtype}, a, d, dt_bias, state, slot_stride, C, N};
  if (N <= 4) return scan_go<4, 1>(s, stream);
  if (N <= 8) return scan_go<4, 2>(s, stream);
  if (N <= 16) return scan_go<4, 4>(s, stream);
  if (N <= 32) return scan_go<8, 4>(s, stream);
  if (N <= 64) return scan_go<16, 4>(s, stream);
  return scan_go<16, 8>(s, stream);
}
