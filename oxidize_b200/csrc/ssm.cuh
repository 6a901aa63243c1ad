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

__device__ __forceinline__ float ssm_softplus(float x) { return x > 20.f ? x : log1pf(expf(x)); }

// A sequence's rows [t0, t1) of the step, its slot (< 0: none) and the position of its first row.
struct SsmSeq {
  int t0, t1, slot, pos0;
};
__device__ __forceinline__ SsmSeq ssm_seq(const SsmStep& s, int b, bool report) {
  SsmSeq q;
  q.t0 = max(s.query_start[b], 0);
  q.t1 = min(s.query_start[b + 1], s.T);
  q.slot = s.slots[b];
  q.pos0 = s.seq_lens[b] - (q.t1 - q.t0);
  if (q.slot >= s.num_slots) {
    if (report) oxb_report(OXB_BAD_SLOT, q.slot);
    q.slot = -1;
  }
  return q;
}

// Exponential of x and silu with the special function unit: the part of x log2(e) that float32 drops is put back, so that the
// relative error stays at some 2^-22 wherever x is (without it, it grows with |x|: 2^-20 at 8).
__device__ __forceinline__ float ssm_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ssm_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ssm_exp(float x) {
  constexpr float L = 1.4426950408889634f, L_LO = 1.925963033500e-8f;  // log2(e) and what its float32 leaves out
  const float t = x * L;
  const float e = ssm_ex2(t);
  // (nothing is put back where the exponential is 0 or infinite, or t is not a number)
  return fabsf(t) < 126.f ? fmaf(e, 0.6931471805599453f * fmaf(x, L_LO, fmaf(x, L, -t)), e) : e;
}
__device__ __forceinline__ float ssm_silu_fast(float x) { return x * ssm_rcp(1.f + ssm_exp(-x)); }

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
// Bound by memory: a row is read and written once, but for the K - 1 rows ahead of a tile (L2 has them).
template <typename TX, typename TY, int V, int K, int U>
__global__ void __launch_bounds__(128) causal_conv_kernel(const ConvArgs a, int TT) {
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
    for (; t < stop; t += U) {
      ConvRow<TX, V> r[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (t + k < stop) r[k].load(X + (size_t)(t + k) * a.x.ld);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (t + k < stop) {
          float y[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float x = r[k].at(j);
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < K - 1; ++i) v = fmaf(w[i][j], past[i][j], v);
            v = fmaf(w[K - 1][j], x, v) + bias[j];
            y[j] = a.silu ? ssm_silu_fast(v) : v;
#pragma unroll
            for (int i = 0; i + 1 < K - 1; ++i) past[i][j] = past[i + 1][j];
            if constexpr (K > 1) past[K - 2][j] = x;
          }
          conv_store<TY, V>(Y + (size_t)(t + k) * a.y.ld, y);
        }
      }
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
  float v = 0.f;
  for (int i = 0; i < a.taps; ++i) {
    const int r = t - (a.taps - 1) + i, p = q.pos0 + r - q.t0;
    if (p < 0) continue;
    v = fmaf(a.w[(size_t)c * a.taps + i], r >= q.t0 ? ssm_load(a.x, r, c) : ring[(size_t)(p % a.taps) * a.C + c], v);
  }
  if (a.bias != nullptr) v += a.bias[c];
  ssm_store(a.y, t, c, a.silu ? ssm_silu_fast(v) : v);
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

struct ScanArgs {
  SsmStep s;
  SsmRows u, dt, z, b, c, y;  // z.p null: no gate
  const float* a;             // [C, N]
  const float* d;             // [C] or null
  const float* dt_bias;       // [C] or null
  float* state;               // [num_slots, C, N]
  long long slot_stride;
  int C, N;
  // bits: u, dt, z, b, c, y lie on 16-byte boundaries and their rows are whole 16-byte pieces; 64: a lane's states do and are
  int wide;
};

// L neighbouring lanes share a channel, S neighbouring states to a lane (N <= L S; states past N are zeros that stay zeros).  The
// states of a lane and then the lanes' sums are added up in one order for every kernel and every step, so that a sequence's bits
// do not depend on how its rows are portioned or on what runs beside it.
constexpr int SCAN_L = 8;

// One token: the decays are exponentials of base two (A2 = A log2(e)).  The lane's share of h . c.
template <int S>
__device__ __forceinline__ float scan_token(float (&h)[S], const float (&A2)[S], float dt, float du, const float (&bv)[S], const float (&cv)[S]) {
  float y = 0.f;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    h[i] = fmaf(ssm_ex2(dt * A2[i]), h[i], du * bv[i]);
    y = fmaf(h[i], cv[i], y);
  }
  return y;
}

// From each lane's shares of L tokens to lane l's whole of token l: pairs of lanes swap halves of what they hold.
template <int L>
__device__ __forceinline__ float scan_join(float (&v)[L], int lane) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = up ? v[i + o] : v[i], give = up ? v[i] : v[i + o];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  return v[0];
}

template <int S>
__device__ __forceinline__ void scan_floats(float (&to)[S], const float* p) {  // shared memory, S floats on their own boundary
  if constexpr (S >= 4) {
#pragma unroll
    for (int i = 0; i < S; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      to[i] = v.x, to[i + 1] = v.y, to[i + 2] = v.z, to[i + 3] = v.w;
    }
  } else if constexpr (S == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    to[0] = v.x, to[1] = v.y;
  } else {
    to[0] = p[0];
  }
}

__device__ __forceinline__ void cp_async16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

constexpr int SCAN_THREADS = 128, SCAN_TT = 32, SCAN_STAGES = 3;
template <int S>
struct ScanTile {
  static constexpr int CH = SCAN_THREADS / SCAN_L, NP = SCAN_L * S;
  // bytes of a staged row of channels: float32's, and 16 more so that the rows that a warp reads at once lie in different banks
  static constexpr int PITCH = CH * 4 + 16, ROWS = SCAN_TT * PITCH;
  static constexpr int STAGE = 3 * ROWS + 2 * SCAN_TT * NP * 4;
  static constexpr int STEPS = SCAN_TT * 2 + 4;  // floats of a channel's (dt, dt u) pairs
  static constexpr int SMEM = SCAN_STAGES * STAGE + CH * STEPS * 4 + 2 * ROWS;
};

// Rows [r0, r0 + n) and `cols` columns from c0 on into shared memory, asynchronously where their boundaries allow it (WIDE: whole
// 16-byte pieces).  FLOATS: as float32 (rows of float32 values only are copied asynchronously then).
template <bool FLOATS>
__device__ __forceinline__ void scan_stage(uint8_t* to, int pitch, const SsmRows& m, bool wide, int r0, int n, int c0, int cols) {
  const int size = m.dtype == 0 ? 4 : 2;
  const uint8_t* from = reinterpret_cast<const uint8_t*>(m.p) + ((size_t)r0 * m.ld + c0) * size;
  const size_t ld = (size_t)m.ld * size;
  if (wide && (!FLOATS || size == 4)) {
    const int pieces = cols * size / 16;
    for (int i = threadIdx.x; i < n * pieces; i += SCAN_THREADS) {
      const int r = i / pieces, p = i % pieces;
      cp_async16(to + r * pitch + p * 16, from + r * ld + p * 16);
    }
  } else if (size == 4) {
    for (int i = threadIdx.x; i < n * cols; i += SCAN_THREADS) {
      const int r = i / cols, c = i % cols;
      cp_async4(to + r * pitch + c * 4, from + r * ld + c * 4);
    }
  } else {
    for (int i = threadIdx.x; i < n * cols; i += SCAN_THREADS) {
      const int r = i / cols, c = i % cols;
      const uint16_t v = *reinterpret_cast<const uint16_t*>(from + r * ld + c * 2);
      if (FLOATS) *reinterpret_cast<uint32_t*>(to + r * pitch + c * 4) = (uint32_t)v << 16;
      else *reinterpret_cast<uint16_t*>(to + r * pitch + c * 2) = v;
    }
  }
}
__device__ __forceinline__ float scan_staged(const uint8_t* row, int c, int dtype) {
  return dtype == 0 ? reinterpret_cast<const float*>(row)[c] : __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(row)[c] << 16);
}

// grid (channels / CH, B): CTA (i, b) takes CH channels of sequence b through its rows, SCAN_TT at a time.
template <int S>
__global__ void __launch_bounds__(SCAN_THREADS) selective_scan_kernel(const ScanArgs a) {
  using Tile = ScanTile<S>;
  constexpr int L = SCAN_L, CH = Tile::CH, NP = Tile::NP, TT = SCAN_TT, PITCH = Tile::PITCH;
  extern __shared__ __align__(16) uint8_t scan_smem[];
  pdl_launch_dependents();
  pdl_wait();
  const SsmSeq q = ssm_seq(a.s, blockIdx.y, blockIdx.x == 0 && threadIdx.x == 0);
  if (q.t1 <= q.t0) return;
  const int tid = threadIdx.x, lane = tid % L, ch = tid / L, c0 = blockIdx.x * CH, c = c0 + ch, cc = min(c, a.C - 1), cols = min(CH, a.C - c0);
  if (q.slot < 0) {
    for (int i = tid; i < (q.t1 - q.t0) * cols; i += SCAN_THREADS) ssm_store(a.y, q.t0 + i / cols, c0 + i % cols, 0.f);
    return;
  }
  float* steps = reinterpret_cast<float*>(scan_smem + SCAN_STAGES * Tile::STAGE) + ch * Tile::STEPS;
  uint8_t* ybuf = scan_smem + SCAN_STAGES * Tile::STAGE + CH * Tile::STEPS * 4;
  const int tiles = (q.t1 - q.t0 + TT - 1) / TT;
  auto issue = [&](int i) {
    if (i < tiles) {
      uint8_t* st = scan_smem + (i % SCAN_STAGES) * Tile::STAGE;
      const int r0 = q.t0 + i * TT, n = min(TT, q.t1 - r0);
      scan_stage<false>(st, PITCH, a.u, a.wide & 1, r0, n, c0, cols);
      scan_stage<false>(st + Tile::ROWS, PITCH, a.dt, a.wide & 2, r0, n, c0, cols);
      if (a.z.p != nullptr) scan_stage<false>(st + 2 * Tile::ROWS, PITCH, a.z, a.wide & 4, r0, n, c0, cols);
      scan_stage<true>(st + 3 * Tile::ROWS, NP * 4, a.b, a.wide & 8, r0, n, 0, a.N);
      scan_stage<true>(st + 3 * Tile::ROWS + TT * NP * 4, NP * 4, a.c, a.wide & 16, r0, n, 0, a.N);
    }
    cp_async_commit();
  };
  if (a.N < NP)  // states that are not there
    for (int i = tid; i < SCAN_STAGES * 2 * TT * NP; i += SCAN_THREADS) {
      const int st = i / (2 * TT * NP), k = i % (2 * TT * NP);
      if (k % NP >= a.N) reinterpret_cast<float*>(scan_smem + st * Tile::STAGE + 3 * Tile::ROWS)[k] = 0.f;
    }
#pragma unroll
  for (int i = 0; i < SCAN_STAGES - 1; ++i) issue(i);
  float* state = a.state + q.slot * a.slot_stride + (size_t)cc * a.N;
  float A2[S], h[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int n = lane * S + i;
    A2[i] = n < a.N ? a.a[(size_t)cc * a.N + n] * 1.4426950408889634f : 0.f;
    h[i] = n < a.N && q.pos0 > 0 ? state[n] : 0.f;
  }
  const float D = a.d != nullptr ? a.d[cc] : 0.f, bias = a.dt_bias != nullptr ? a.dt_bias[cc] : 0.f;
  // a tile's results, written one tile later by all threads together
  auto flush = [&](int i) {
    const int r0 = q.t0 + i * TT, n = min(TT, q.t1 - r0), size = a.y.dtype == 0 ? 4 : 2;
    const uint8_t* from = ybuf + (i & 1) * Tile::ROWS;
    uint8_t* to = reinterpret_cast<uint8_t*>(const_cast<void*>(a.y.p)) + ((size_t)r0 * a.y.ld + c0) * size;
    const size_t ld = (size_t)a.y.ld * size;
    if (a.wide & 32) {
      const int pieces = cols * size / 16;
      for (int k = tid; k < n * pieces; k += SCAN_THREADS)
        *reinterpret_cast<uint4*>(to + (k / pieces) * ld + (k % pieces) * 16) = *reinterpret_cast<const uint4*>(from + (k / pieces) * PITCH + (k % pieces) * 16);
    } else if (size == 4) {
      for (int k = tid; k < n * cols; k += SCAN_THREADS)
        *reinterpret_cast<float*>(to + (k / cols) * ld + (k % cols) * 4) = *reinterpret_cast<const float*>(from + (k / cols) * PITCH + (k % cols) * 4);
    } else {
      for (int k = tid; k < n * cols; k += SCAN_THREADS)
        *reinterpret_cast<uint16_t*>(to + (k / cols) * ld + (k % cols) * 2) = *reinterpret_cast<const uint16_t*>(from + (k / cols) * PITCH + (k % cols) * 2);
    }
  };
  for (int i = 0; i < tiles; ++i) {
    cp_async_wait<SCAN_STAGES - 2>();
    __syncthreads();
    issue(i + SCAN_STAGES - 1);
    if (i > 0) flush(i - 1);
    const uint8_t* st = scan_smem + (i % SCAN_STAGES) * Tile::STAGE;
    const float *Bt = reinterpret_cast<const float*>(st + 3 * Tile::ROWS) + lane * S, *Ct = Bt + TT * NP;
    uint8_t* yt = ybuf + (i & 1) * Tile::ROWS;
    const int n = min(TT, q.t1 - q.t0 - i * TT);
    // each lane prepares every L-th token of its channel
    for (int t = lane; t < n; t += L) {
      const float dt = ssm_softplus(scan_staged(st + Tile::ROWS + t * PITCH, ch, a.dt.dtype) + bias);
      *reinterpret_cast<float2*>(steps + 2 * t) = make_float2(dt, dt * scan_staged(st + t * PITCH, ch, a.u.dtype));
    }
    __syncwarp();
    for (int g = 0; g < n; g += L) {
      float acc[L];
#pragma unroll
      for (int j = 0; j < L; ++j) {
        acc[j] = 0.f;
        if (g + j < n) {
          const float2 d = *reinterpret_cast<const float2*>(steps + 2 * (g + j));
          float bv[S], cv[S];
          scan_floats<S>(bv, Bt + (g + j) * NP);
          scan_floats<S>(cv, Ct + (g + j) * NP);
          acc[j] = scan_token<S>(h, A2, d.x, d.y, bv, cv);
        }
      }
      float y = scan_join<L>(acc, lane);
      const int t = g + lane;
      if (t < n) {
        y = fmaf(D, scan_staged(st + t * PITCH, ch, a.u.dtype), y);
        if (a.z.p != nullptr) y *= ssm_silu_fast(scan_staged(st + 2 * Tile::ROWS + t * PITCH, ch, a.z.dtype));
        if (a.y.dtype == 0) reinterpret_cast<float*>(yt + t * PITCH)[ch] = y;
        else reinterpret_cast<__nv_bfloat16*>(yt + t * PITCH)[ch] = __float2bfloat16(y);
      }
    }
    __syncwarp();  // (steps are written again)
  }
  __syncthreads();
  flush(tiles - 1);
  if (c < a.C)
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (lane * S + i < a.N) state[lane * S + i] = h[i];
}

// Steps of one row per sequence.  grid (channels / CH, B / L): a thread takes its states of L sequences through their tokens, lane l
// prepares and ends sequence l's.  Bound by memory: the states are read and written once.
template <int S>
__global__ void __launch_bounds__(SCAN_THREADS) selective_step_kernel(const ScanArgs a) {
  constexpr int L = SCAN_L;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x % L, c = blockIdx.x * (SCAN_THREADS / L) + threadIdx.x / L, cc = min(c, a.C - 1), b = blockIdx.y * L + lane;
  SsmSeq q{0, 0, -1, 0};
  if (b < a.s.B) q = ssm_seq(a.s, b, blockIdx.x == 0 && threadIdx.x < L);
  const bool on = q.t1 == q.t0 + 1, live = on && q.slot >= 0;
  float u = 0.f, dt = 0.f;
  if (live) {
    u = ssm_load(a.u, q.t0, cc);
    dt = ssm_load(a.dt, q.t0, cc) + (a.dt_bias != nullptr ? a.dt_bias[cc] : 0.f);
  }
  const float z = live && a.z.p != nullptr ? ssm_load(a.z, q.t0, cc) : 0.f, D = a.d != nullptr ? a.d[cc] : 0.f;
  const int slot = live ? q.slot : -1;
  float A2[S], h[L][S];
#pragma unroll
  for (int i = 0; i < S; ++i) A2[i] = lane * S + i < a.N ? a.a[(size_t)cc * a.N + lane * S + i] * 1.4426950408889634f : 0.f;
  const bool whole = a.wide & 64;  // S states are one piece in memory
#pragma unroll
  for (int j = 0; j < L; ++j) {
    const int s = __shfl_sync(0xffffffffu, slot, j, L), p = __shfl_sync(0xffffffffu, q.pos0, j, L);
    const float* from = a.state + s * a.slot_stride + (size_t)cc * a.N + lane * S;
#pragma unroll
    for (int i = 0; i < S; ++i) h[j][i] = 0.f;
    if (s >= 0 && p > 0) {
      if (whole) {
        scan_floats<S>(h[j], from);
      } else {
#pragma unroll
        for (int i = 0; i < S; ++i)
          if (lane * S + i < a.N) h[j][i] = from[i];
      }
    }
  }
  dt = ssm_softplus(dt);
  const float du = dt * u;
  float acc[L];
#pragma unroll
  for (int j = 0; j < L; ++j) {
    const int s = __shfl_sync(0xffffffffu, slot, j, L), t = __shfl_sync(0xffffffffu, q.t0, j, L);
    const float dtj = __shfl_sync(0xffffffffu, dt, j, L), duj = __shfl_sync(0xffffffffu, du, j, L);
    acc[j] = 0.f;
    if (s < 0) continue;
    float bv[S], cv[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const bool in = lane * S + i < a.N;
      bv[i] = in ? ssm_load(a.b, t, lane * S + i) : 0.f;
      cv[i] = in ? ssm_load(a.c, t, lane * S + i) : 0.f;
    }
    acc[j] = scan_token<S>(h[j], A2, dtj, duj, bv, cv);
    if (c < a.C) {
      float* to = a.state + s * a.slot_stride + (size_t)cc * a.N + lane * S;
      if (whole) {
        if constexpr (S >= 4) {
#pragma unroll
          for (int i = 0; i < S; i += 4) *reinterpret_cast<float4*>(to + i) = make_float4(h[j][i], h[j][i + 1], h[j][i + 2], h[j][i + 3]);
        } else if constexpr (S == 2) {
          *reinterpret_cast<float2*>(to) = make_float2(h[j][0], h[j][1]);
        } else {
          to[0] = h[j][0];
        }
      } else {
#pragma unroll
        for (int i = 0; i < S; ++i)
          if (lane * S + i < a.N) to[i] = h[j][i];
      }
    }
  }
  float y = scan_join<L>(acc, lane);
  if (on && c < a.C) {
    y = fmaf(D, u, y);
    if (a.z.p != nullptr) y *= ssm_silu_fast(z);
    ssm_store(a.y, q.t0, c, live ? y : 0.f);
  }
}

}  // namespace oxb
