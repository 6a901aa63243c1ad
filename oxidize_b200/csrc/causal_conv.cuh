// The short causal convolution of state-space layers (ssm.cuh: its formula, the ring of a sequence's last inputs).
#pragma once
#include "ssm.cuh"

namespace oxb {

struct ConvArgs {
  SsmStep s;
  SsmRows x, y;
  const float* w;     // [C, taps]
  const float* bias;  // [C] or null
  float* window;      // [num_slots, taps, C]
  long long slot_stride;
  int C, taps, silu;
};

template <typename T, int V>
struct ConvRow {  // V neighbouring channels of a row as they are stored
  static constexpr int WORDS = V * sizeof(T) >= 4 ? V * (int)sizeof(T) / 4 : 1;
  uint32_t v[WORDS];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1 && sizeof(T) == 2) v[0] = *reinterpret_cast<const uint16_t*>(p);
    else if constexpr (WORDS == 1) v[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (WORDS == 2) *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(p);
    else *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(v[j]);
    else return j & 1 ? __uint_as_float(v[j >> 1] & 0xFFFF0000u) : __uint_as_float(v[j >> 1] << 16);
  }
};
template <int V>
__device__ __forceinline__ void conv_load_floats(float* to, const float* p) {
  if constexpr (V == 4) *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(p);
  else to[0] = p[0];
}
template <typename T, int V>
__device__ __forceinline__ void conv_store(T* p, const float* v) {
  if constexpr (V == 1 && sizeof(T) == 2) *p = __float2bfloat16(v[0]);
  else if constexpr (V == 1) *p = v[0];
  else if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// grid (tiles of TT rows, channels / (128 V)).  A thread owns V neighbouring channels and goes through the tile's rows with the K - 1
// (K: taps) rows ahead in registers; U rows are loaded at a time.
//
// The rows of a sequence that read its ring (the first K - 1) all belong to the tile of its first row, wherever the tile ends: the
// thread that reads a ring is then also the one that writes it, afterwards.
//
// Bound by memory: a row is read and written once, but for the K - 1 rows ahead of a tile (L2 has them); its instructions fill 45 % of
// the issue slots, half of them silu's.  What counts are warps and plain code for whole groups of rows: 7 prompts of 300 to 1900 rows,
// 4096 channels, bf16 to float32 48 us, 4.4 TB/s (52 with five blocks to an SM and every row guarded, 55 with the next group's rows loaded
// ahead, which costs registers).
template <typename TX, typename TY, int V, int K, int U>
__global__ void __launch_bounds__(128, U == 1 ? 1 : V == 1 ? 10 : 6) causal_conv_kernel(const ConvArgs a, int TT) {
  pdl_launch_dependents();
  pdl_wait();
  const int c = (blockIdx.y * 128 + threadIdx.x) * V;
  float w[K][V], bias[V];
  if (c < a.C) {
    float all[K * V];
#pragma unroll
    for (int i = 0; i < K; ++i) conv_load_floats<V>(all + i * V, a.w + (size_t)c * K + i * V);
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) w[i][j] = all[j * K + i];
#pragma unroll
    for (int j = 0; j < V; ++j) bias[j] = a.bias != nullptr ? a.bias[c + j] : 0.f;
  }
  const int begin = blockIdx.x * TT, upto = min(a.s.query_start[a.s.B], a.s.T), end = min(begin + TT, upto);
  if (c >= a.C || begin >= end) return;
  const TX* X = reinterpret_cast<const TX*>(a.x.p) + c;
  TY* Y = reinterpret_cast<TY*>(const_cast<void*>(a.y.p)) + c;
  int b = sequence_of(a.s.query_start, a.s.B, begin);
  for (int t = begin; t < end;) {
    const SsmSeq q = ssm_seq(a.s, b, c == 0);
    ++b;
    if (q.t1 <= t) continue;  // (of no rows)
    const bool first = q.t0 >= begin;
    int stop = min(q.t1, end);
    if (q.slot < 0) {
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      for (; t < stop; ++t) conv_store<TY, V>(Y + (size_t)t * a.y.ld, zero);
      continue;
    }
    float* ring = a.window + q.slot * a.slot_stride + c;
    if (first) stop = max(stop, min(q.t1, q.t0 + K - 1));
    else t = max(t, q.t0 + K - 1);
    float past[K > 1 ? K - 1 : 1][V];  // the rows ahead, oldest first
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      const int back = K - 1 - i, p = q.pos0 + t - q.t0 - back;
#pragma unroll
      for (int j = 0; j < V; ++j) past[i][j] = 0.f;
      if (t - back >= q.t0 && t < stop) {
        ConvRow<TX, V> r;
        r.load(X + (size_t)(t - back) * a.x.ld);
#pragma unroll
        for (int j = 0; j < V; ++j) past[i][j] = r.at(j);
      } else if (first && p >= 0) {
        conv_load_floats<V>(past[i], ring + (size_t)(p % K) * a.C);
      }
    }
    const TX* from = X + (size_t)t * a.x.ld;
    TY* to = Y + (size_t)t * a.y.ld;
    auto row = [&](const ConvRow<TX, V>& r, TY* to) {
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = r.at(j);
        float v = bias[j];
#pragma unroll
        for (int i = 0; i < K - 1; ++i) v = fmaf(w[i][j], past[i][j], v);
        v = fmaf(w[K - 1][j], x, v);
        y[j] = a.silu ? ssm_silu(v) : v;
#pragma unroll
        for (int i = 0; i + 1 < K - 1; ++i) past[i][j] = past[i + 1][j];
        if constexpr (K > 1) past[K - 2][j] = x;
      }
      conv_store<TY, V>(to, y);
    };
    for (; t + U <= stop; t += U) {
      ConvRow<TX, V> r[U];
#pragma unroll
      for (int k = 0; k < U; ++k, from += a.x.ld) r[k].load(from);
#pragma unroll
      for (int k = 0; k < U; ++k, to += a.y.ld) row(r[k], to);
    }
    if (t < stop) {
      ConvRow<TX, V> r[U];
#pragma unroll
      for (int k = 0; k < U; ++k, from += a.x.ld)
        if (t + k < stop) r[k].load(from);
#pragma unroll
      for (int k = 0; k < U; ++k, to += a.y.ld)
        if (t + k < stop) row(r[k], to);
    }
    t = stop;
    if (first) {  // the sequence's last rows stay for its next step
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const int row = q.t1 - K + i;
        if (row >= q.t0) {
          ConvRow<TX, V> r;
          r.load(X + (size_t)row * a.x.ld);
          float v[V];
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = r.at(j);
          conv_store<float, V>(ring + (size_t)((q.pos0 + row - q.t0) % K) * a.C, v);
        }
      }
    }
  }
}

// More taps than that kernel has, row by row.  grid (T, channels / 256)
__global__ void __launch_bounds__(256) causal_conv_any_kernel(const ConvArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x, c = blockIdx.y * 256 + threadIdx.x;
  if (c >= a.C || t >= a.s.query_start[a.s.B]) return;
  const SsmSeq q = ssm_seq(a.s, sequence_of(a.s.query_start, a.s.B, t), c == 0);
  if (q.slot < 0) return ssm_store(a.y, t, c, 0.f);
  const float* ring = a.window + q.slot * a.slot_stride;
  float v = a.bias != nullptr ? a.bias[c] : 0.f;
  for (int i = 0; i < a.taps; ++i) {
    const int r = t - (a.taps - 1) + i, p = q.pos0 + r - q.t0;
    if (p < 0) continue;
    v = fmaf(a.w[(size_t)c * a.taps + i], r >= q.t0 ? ssm_load(a.x, r, c) : ring[(size_t)(p % a.taps) * a.C + c], v);
  }
  ssm_store(a.y, t, c, a.silu ? ssm_silu(v) : v);
}

// grid (channels / 256, B), after causal_conv_any_kernel: a sequence's last inputs
__global__ void __launch_bounds__(256) conv_window_kernel(const ConvArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int c = blockIdx.x * 256 + threadIdx.x;
  const SsmSeq q = ssm_seq(a.s, blockIdx.y, false);
  if (c >= a.C || q.slot < 0) return;
  float* ring = a.window + q.slot * a.slot_stride;
  for (int t = max(q.t0, q.t1 - a.taps); t < q.t1; ++t) ring[(size_t)((q.pos0 + t - q.t0) % a.taps) * a.C + c] = ssm_load(a.x, t, c);
}

}  // namespace oxb
