// State-space layers: the short causal convolution and the selective scan of a step's rows.
//
//   convolution  y[t, c] = act(sum_i w[c, i] x[t - (taps - 1) + i, c] + bias[c])
//   scan         s = softplus(dt + dt_bias);  h[n] <- exp(s A[c, n]) h[n] + s u B[n];  y = (sum_n h[n] C[n] + D u) silu(z)
//
// A step feeds ragged sequences; what a sequence carries from step to step lies in a slot: the ring of its last `taps` inputs
// (position p's row is row p % taps, so that the row a decoded token writes is none of those it reads) and the state h [C, N], both
// float32.  A sequence whose rows start at position 0 starts from nothing, whatever its slot holds.
#pragma once
#include "common.cuh"

namespace oxb {

// Rows and slots of a step's sequences.
struct SsmStep {
  const int* query_start;  // [B + 1]
  const int* seq_lens;     // [B], with this step's rows
  const int* slots;        // [B], < 0: none (rows of zeros come out)
  int B, T, num_slots;
};

// A row-major matrix of float32 (dtype 0) or bfloat16 (2) values.
struct SsmRows {
  const void* p;
  int ld, dtype;
};
__device__ __forceinline__ float ssm_load(const SsmRows& m, size_t row, int col) {
  const size_t at = row * (size_t)m.ld + col;
  return m.dtype == 0 ? reinterpret_cast<const float*>(m.p)[at] : bf16_to_f32(reinterpret_cast<const __nv_bfloat16*>(m.p)[at]);
}
__device__ __forceinline__ void ssm_store(const SsmRows& m, size_t row, int col, float v) {
  const size_t at = row * (size_t)m.ld + col;
  if (m.dtype == 0) reinterpret_cast<float*>(const_cast<void*>(m.p))[at] = v;
  else reinterpret_cast<__nv_bfloat16*>(const_cast<void*>(m.p))[at] = __float2bfloat16(v);
}

__device__ __forceinline__ float ssm_silu(float x) { return x / (1.f + expf(-x)); }
__device__ __forceinline__ float ssm_softplus(float x) { return x > 20.f ? x : log1pf(expf(x)); }

// A sequence's rows [t0, t1) of the step, its slot (< 0: none) and the position of its first row.
struct SsmSeq {
  int t0, t1, slot, pos0;
};
__device__ __forceinline__ SsmSeq ssm_seq(const SsmStep& s, int b) {
  SsmSeq q;
  q.t0 = max(s.query_start[b], 0);
  q.t1 = min(s.query_start[b + 1], s.T);
  q.slot = s.slots[b];
  q.pos0 = s.seq_lens[b] - (q.t1 - q.t0);
  if (q.slot >= s.num_slots) {
    if (threadIdx.x == 0) oxb_report(OXB_BAD_SLOT, q.slot);
    q.slot = -1;
  }
  return q;
}

struct ConvArgs {
  SsmStep s;
  SsmRows x, y;
  const float* w;     // [C, taps]
  const float* bias;  // [C] or null
  float* window;      // [num_slots, taps, C]
  long long slot_stride;
  int C, taps, silu;
};

// grid (T, channels / 256)
__global__ void __launch_bounds__(256) causal_conv_kernel(const ConvArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x, c = blockIdx.y * 256 + threadIdx.x;
  if (c >= a.C || t >= a.s.query_start[a.s.B]) return;
  const SsmSeq q = ssm_seq(a.s, sequence_of(a.s.query_start, a.s.B, t));
  if (q.slot < 0) return ssm_store(a.y, t, c, 0.f);
  const float* ring = a.window + q.slot * a.slot_stride;
  float v = 0.f;
  for (int i = 0; i < a.taps; ++i) {
    const int r = t - (a.taps - 1) + i, p = q.pos0 + r - q.t0;
    if (p < 0) continue;
    v = fmaf(a.w[(size_t)c * a.taps + i], r >= q.t0 ? ssm_load(a.x, r, c) : ring[(size_t)(p % a.taps) * a.C + c], v);
  }
  if (a.bias != nullptr) v += a.bias[c];
  ssm_store(a.y, t, c, a.silu ? ssm_silu(v) : v);
}

// grid (channels / 256, B), after the convolution: its last inputs
__global__ void __launch_bounds__(256) conv_window_kernel(const ConvArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int c = blockIdx.x * 256 + threadIdx.x;
  const SsmSeq q = ssm_seq(a.s, blockIdx.y);
  if (c >= a.C || q.slot < 0) return;
  float* ring = a.window + q.slot * a.slot_stride;
  for (int t = max(q.t0, q.t1 - a.taps); t < q.t1; ++t) ring[(size_t)((q.pos0 + t - q.t0) % a.taps) * a.C + c] = ssm_load(a.x, t, c);
}

struct ScanArgs {
  SsmStep s;
  SsmRows u, dt, z, b, c, y;  // z.p null: no gate
  const float* a;             // [C, N]
  const float* d;             // [C] or null
  const float* dt_bias;       // [C] or null
  float* state;               // [num_slots, C, N]
  long long slot_stride;
  int C, N;
};

// grid (channels * L / 128, B): L lanes share a channel, S states to a lane
template <int L, int S>
__global__ void __launch_bounds__(128) selective_scan_kernel(const ScanArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const SsmSeq q = ssm_seq(a.s, blockIdx.y);
  if (q.t1 <= q.t0) return;
  const int lane = threadIdx.x % L, c = blockIdx.x * (128 / L) + threadIdx.x / L, cc = min(c, a.C - 1);
  if (q.slot < 0) {
    if (c < a.C)
      for (int t = q.t0 + lane; t < q.t1; t += L) ssm_store(a.y, t, c, 0.f);
    return;
  }
  float* state = a.state + q.slot * a.slot_stride + (size_t)cc * a.N;
  float A[S], h[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int n = lane * S + i;
    A[i] = n < a.N ? a.a[(size_t)cc * a.N + n] : 0.f;
    h[i] = n < a.N && q.pos0 > 0 ? state[n] : 0.f;
  }
  const float D = a.d != nullptr ? a.d[cc] : 0.f, bias = a.dt_bias != nullptr ? a.dt_bias[cc] : 0.f;
  for (int t = q.t0; t < q.t1; ++t) {
    const float u = ssm_load(a.u, t, cc), dt = ssm_softplus(ssm_load(a.dt, t, cc) + bias);
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int n = lane * S + i;
      if (n < a.N) {
        h[i] = fmaf(expf(dt * A[i]), h[i], dt * u * ssm_load(a.b, t, n));
        y = fmaf(h[i], ssm_load(a.c, t, n), y);
      }
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (lane == 0 && c < a.C) {
      y = fmaf(D, u, y);
      if (a.z.p != nullptr) y *= ssm_silu(ssm_load(a.z, t, c));
      ssm_store(a.y, t, c, y);
    }
  }
  if (c < a.C)
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (lane * S + i < a.N) state[lane * S + i] = h[i];
}

}  // namespace oxb
