// liboxb, entry point of state-space layers' selective scan (ssm.cuh).
#include "common.cuh"
#include "ssm.cuh"
using namespace oxb;

static bool scan_direct(const ScanArgs& a) {
  return a.N % 4 == 0 && a.b.dtype == 0 && a.c.dtype == 0 && a.b.ld % 4 == 0 && a.c.ld % 4 == 0 &&
         ((reinterpret_cast<uintptr_t>(a.b.p) | reinterpret_cast<uintptr_t>(a.c.p)) & 15) == 0;
}

template <int L, int S, bool ALL, typename TU, typename TZ>
static int scan_typed(const ScanArgs& a, cudaStream_t stream) {
  constexpr int CH = ScanTile<L, S>::CH;
  return (int)oxb_launch(selective_scan_kernel<L, S, ALL, TU, TZ>, dim3((a.C + CH - 1) / CH, a.s.B), dim3(128), 0, stream, a);
}
template <int NP, bool ALL, typename TU, typename TZ>
static int scan_wide_typed(const ScanArgs& a, cudaStream_t stream) {
  constexpr int CW = ScanWide<NP>::CW;
  return (int)oxb_launch(selective_scan_wide_kernel<NP, ALL, TU, TZ>, dim3((a.C + CW - 1) / CW, a.s.B), dim3(CW), 0, stream, a);
}
// by the types of u, dt and of the gate
#define SCAN_TYPES(F, ...)                                                                          \
  (a.u.dtype == 0 ? (a.z.p == nullptr   ? F<__VA_ARGS__, float, NoGate>(a, stream)                  \
                     : a.z.dtype == 0   ? F<__VA_ARGS__, float, float>(a, stream)                   \
                                        : F<__VA_ARGS__, float, __nv_bfloat16>(a, stream))          \
                  : (a.z.p == nullptr   ? F<__VA_ARGS__, __nv_bfloat16, NoGate>(a, stream)          \
                     : a.z.dtype == 0   ? F<__VA_ARGS__, __nv_bfloat16, float>(a, stream)           \
                                        : F<__VA_ARGS__, __nv_bfloat16, __nv_bfloat16>(a, stream)))

template <int L, int S>
static int scan_go(ScanArgs a, cudaStream_t stream) {
  a.wide = scan_direct(a);
  const int e = a.N == L * S ? SCAN_TYPES(scan_typed, L, S, true) : SCAN_TYPES(scan_typed, L, S, false);
  if (e != 0) return e;
  OXB_CHECK_LAUNCH();
  return 0;
}
template <int L, int S>
static int scan_step_go(ScanArgs a, cudaStream_t stream) {
  a.whole = S >= 4 && a.N == L * S && a.slot_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a.state) & 15) == 0;
  a.wide = S >= 4 && a.N == L * S && scan_direct(a);
  constexpr int CH = 128 / L;
  const dim3 grid((a.C + CH - 1) / CH, (a.s.B + L - 1) / L);
  if (a.N == L * S) oxb_launch(selective_step_kernel<L, S, true>, grid, dim3(128), 0, stream, a);
  else oxb_launch(selective_step_kernel<L, S, false>, grid, dim3(128), 0, stream, a);
  OXB_CHECK_LAUNCH();
  return 0;
}
template <int NP>
static int scan_wide_go(ScanArgs a, cudaStream_t stream) {
  a.wide = scan_direct(a);
  const int e = a.N == NP ? SCAN_TYPES(scan_wide_typed, NP, true) : SCAN_TYPES(scan_wide_typed, NP, false);
  if (e != 0) return e;
  OXB_CHECK_LAUNCH();
  return 0;
}

// Lanes that share a channel, by the channels of all sequences that run at a time.  One lane is the most economical, but its warps take
// 155 ns a token whoever runs beside them.  us with 16, 8 and 1 lanes, 16 states: 1 x 2048 rows of 256 channels 62, 86, 320; of 1536:
// 111, 118, 323; of 2048: 142, 126, 324; of 5120: 258, 229, 326; 2 x 1024 of 5120: 225, 172, 193; 4 x 1024: 425, 281, 251; 9 x 1024:
// 916, 576, 406; 32 x 256 of 2048: 328, 208, 133.  (Four lanes: never ahead of both neighbours.)
static int scan_lanes(int C, int T, int longest) {
  const long long channels = (long long)C * (longest > 0 ? (T + longest - 1) / longest : 1), sms = oxb_sm_count();
  return channels < 12 * sms ? 16 : channels < 110 * sms ? 8 : 1;
}

// Selective scan of a step: u, dt, z, y of C channels and b, c of N <= 128 states, each a matrix of T rows with its own stride and
// dtype (u and dt: the same one); a [C, N]; d, dt_bias [C] or null; z null: no gate.  The state [num_slots, C, N] float32 is read and updated.
// longest 1: every sequence feeds one row at most (one with more is reported: its rows become zeros, its state stays).
OXB_API int oxb_selective_scan(const void* u, int ld_u, int u_dtype, const void* dt, int ld_dt, int dt_dtype, const void* z, int ld_z,
                               int z_dtype, const void* b, int ld_b, int b_dtype, const void* c, int ld_c, int c_dtype, const float* a,
                               const float* d, const float* dt_bias, const int* query_start, const int* seq_lens, const int* slots,
                               float* state, long long slot_stride, int num_slots, void* y, int ld_y, int y_dtype, int B, int T, int C,
                               int N, int longest, cudaStream_t stream) {
  if (B <= 0 || T <= 0 || C <= 0) return 0;
  if (B > 65535 || u_dtype != dt_dtype || N <= 0 || N > 128 || num_slots <= 0 || slots == nullptr || !ssm_dtype(u_dtype) || !ssm_dtype(dt_dtype) ||
      !ssm_dtype(z_dtype) || !ssm_dtype(b_dtype) || !ssm_dtype(c_dtype) || !ssm_dtype(y_dtype))
    return (int)cudaErrorInvalidValue;
  const ScanArgs s{{query_start, seq_lens, slots, B, T, num_slots}, {u, ld_u, u_dtype}, {dt, ld_dt, dt_dtype}, {z, ld_z, z_dtype},
                   {b, ld_b, b_dtype}, {c, ld_c, c_dtype}, {y, ld_y, y_dtype}, a, d, dt_bias, state, slot_stride, C, N, 0, 0};
  if (longest == 1) {
    if (N <= 8) return scan_step_go<4, 2>(s, stream);
    if (N <= 16) return scan_step_go<4, 4>(s, stream);
    if (N <= 32) return scan_step_go<8, 4>(s, stream);
    if (N <= 64) return scan_step_go<16, 4>(s, stream);
    return scan_step_go<8, 16>(s, stream);
  }
  const int lanes = scan_lanes(C, T, longest);
  if (N <= 8) return lanes == 1 ? scan_wide_go<8>(s, stream) : scan_go<8, 1>(s, stream);
  if (N <= 16) return lanes == 1 ? scan_wide_go<16>(s, stream) : lanes == 8 ? scan_go<8, 2>(s, stream) : scan_go<16, 1>(s, stream);
  if (N <= 32) return lanes <= 8 ? scan_go<8, 4>(s, stream) : scan_go<16, 2>(s, stream);
  if (N <= 64) return scan_go<16, 4>(s, stream);
  return scan_go<8, 16>(s, stream);
}
