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

// Dtype codes of the rows of these kernels: 0 float32, 2 bfloat16.
inline bool ssm_dtype(int d) { return d == 0 || d == 2; }

// Rows and slots of a step's sequences.
struct SsmStep {
  const int* query_start;  // [B + 1]
  const int* seq_lens;     // [B], with this step's rows (a smaller one is reported, and the sequence has no slot then)
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
// The bits of a value as they are stored, and the value: loads that are not converted at once do not wait for one another (and,
// volatile, are not put off until their values are wanted).
__device__ __forceinline__ uint32_t ssm_bits(const float* p) {
  uint32_t v;
  asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ssm_bits(const __nv_bfloat16* p) {
  uint32_t v;
  asm volatile("ld.global.u16 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
template <typename T>
__device__ __forceinline__ float ssm_value(uint32_t bits) {
  return __uint_as_float(sizeof(T) == 4 ? bits : bits << 16);
}
// (of a type that is not known to the compiler; not for loads that others follow)
__device__ __forceinline__ uint32_t ssm_bits(const SsmRows& m, size_t row, int col) {
  const size_t at = row * (size_t)m.ld + col;
  return m.dtype == 0 ? ssm_bits(reinterpret_cast<const float*>(m.p) + at) : ssm_bits(reinterpret_cast<const __nv_bfloat16*>(m.p) + at);
}
__device__ __forceinline__ float ssm_value(const SsmRows& m, uint32_t bits) { return __uint_as_float(m.dtype == 0 ? bits : bits << 16); }
// Two values of a column, stored where `first`, `second`
__device__ __forceinline__ void ssm_store2(const SsmRows& m, size_t row0, size_t row1, int col0, int col1, float2 v, bool first, bool second) {
  const int size = m.dtype == 0 ? 4 : 2;
  uint8_t* p = reinterpret_cast<uint8_t*>(const_cast<void*>(m.p));
  asm volatile(
      "{\n\t.reg .pred f, a, b, p, q;\n\t.reg .b16 lo, hi;\n\t.reg .b32 both;\n\t"
      "setp.eq.s32 f, %4, 0;\n\t"
      "setp.ne.s32 a, %5, 0;\n\t"
      "setp.ne.s32 b, %6, 0;\n\t"
      "cvt.rn.bf16x2.f32 both, %3, %2;\n\t"
      "mov.b32 {lo, hi}, both;\n\t"
      "and.pred p, a, f;\n\t"
      "and.pred q, b, f;\n\t"
      "@p st.global.f32 [%0], %2;\n\t"
      "@q st.global.f32 [%1], %3;\n\t"
      "not.pred f, f;\n\t"
      "and.pred p, a, f;\n\t"
      "and.pred q, b, f;\n\t"
      "@p st.global.b16 [%0], lo;\n\t"
      "@q st.global.b16 [%1], hi;\n\t}"
      ::"l"(p + (row0 * (size_t)m.ld + col0) * size), "l"(p + (row1 * (size_t)m.ld + col1) * size), "f"(v.x), "f"(v.y), "r"(m.dtype), "r"((int)first),
        "r"((int)second)
      : "memory");
}
__device__ __forceinline__ void ssm_store(const SsmRows& m, size_t row, int col, float v) {
  const size_t at = row * (size_t)m.ld + col;
  if (m.dtype == 0) reinterpret_cast<float*>(const_cast<void*>(m.p))[at] = v;
  else reinterpret_cast<__nv_bfloat16*>(const_cast<void*>(m.p))[at] = __float2bfloat16(v);
}


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
  if (q.slot >= 0 && q.pos0 < 0 && q.t1 > q.t0) {  // (rows of negative positions would lie ahead of the ring)
    if (report) oxb_report(OXB_BAD_ARGUMENT, s.seq_lens[b]);
    q.slot = -1;
  }
  return q;
}

// Exponential and silu with the special function unit: the part of w log2(e) that float32 drops is put back, so that the
// relative error stays at some 2^-22 wherever w is (without it, it grows with |w|: 2^-20 at 8).
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
__device__ __forceinline__ float ssm_exp_neg(float w) {  // exp(-w)
  constexpr float L = 1.4426950408889634f, L_LO = 1.92596299e-8f;  // log2(e) and what its float32 leaves out
  const float t = w * -L;
  const float e = ssm_ex2(t);
  // (nothing is put back where the exponential is 0 or infinite, or t is not a number)
  return fabsf(t) < 126.f ? fmaf(e, __fmul_rn(fmaf(w, L_LO, fmaf(w, L, t)), -0.6931471805599453f), e) : e;
}
__device__ __forceinline__ float ssm_silu(float x) { return __fmul_rn(x, ssm_rcp(__fadd_rn(ssm_exp_neg(x), 1.f))); }
// softplus(x) = max(x, 0) + log(1 + e) with e = exp(-|x|); log(1 + e) = e P(e) on [0, 1], P a polynomial fitted to the least relative
// error (2^-22.6 with its float32 coefficients and sums), so that small results keep their digits.
__device__ __forceinline__ float ssm_softplus(float x) {
  const float e = ssm_exp_neg(fabsf(x));
  float p = -0.00324402121f;
  p = fmaf(p, e, 0.0198514443f);
  p = fmaf(p, e, -0.0569594987f);
  p = fmaf(p, e, 0.106036514f);
  p = fmaf(p, e, -0.153055906f);
  p = fmaf(p, e, 0.196759388f);
  p = fmaf(p, e, -0.249541342f);
  p = fmaf(p, e, 0.333299637f);
  p = fmaf(p, e, -0.499999017f);
  p = fmaf(p, e, 1.f);
  return fmaf(e, p, fmaxf(x, 0.f));
}

// The y-th longest of a step's sequences: long ones start first, so that short ones fill the gaps (9 of 331 to 1650 rows, 5120
// channels: 398 us, 501 in their own order).  More than 32 stay in their order, also where a long one comes last: 200 single rows ahead of
// a portion of 2048 take 668 us, where the portion alone takes 193.  Whole warps.
__device__ __forceinline__ int scan_sequence(const SsmStep& s, int y) {
  if (s.B > 32) return y;
  const int lane = threadIdx.x & 31, n = lane < s.B ? s.query_start[lane + 1] - s.query_start[lane] : -1;
  int rank = 0;
  for (int i = 0; i < s.B; ++i) {
    const int m = __shfl_sync(0xffffffffu, n, i);
    rank += m > n || (m == n && i < lane);
  }
  return __ffs(__ballot_sync(0xffffffffu, lane < s.B && rank == y)) - 1;
}

struct NoGate {};  // (in the place of the gate's type)
template <typename T>
struct ScanGate {
  using type = T;
};
template <>
struct ScanGate<NoGate> {
  using type = float;
};

struct ScanArgs {
  SsmStep s;
  SsmRows u, dt, z, b, c, y;  // u and dt of one type; z.p null: no gate
  const float* a;             // [C, N]
  const float* d;             // [C] or null
  const float* dt_bias;       // [C] or null
  float* state;               // [num_slots, C, N]
  long long slot_stride;
  int C, N;
  int whole;  // four states and more to a lane, on 16-byte boundaries in memory
  int wide;   // b and c are float32 and their rows whole 16-byte pieces on their boundaries
};

// L neighbouring lanes share a channel, S states to a lane (N <= L S; states past N are zeros that stay zeros).  The products of h . c
// are added up in one order whatever L: states that differ in bit 1 of their number, then the sums that differ in bit 0, 2, 3 and so
// on, so that a sequence's bits do not depend on how its rows are portioned or on what runs beside it.  Four states and more to a
// lane are neighbours, two lie two apart.
template <int S>
__device__ __forceinline__ int scan_state(int lane, int i) {
  return S == 2 ? (lane >> 1) * 4 + (lane & 1) + 2 * i : lane * S + i;
}

// A lane's states of one channel: h <- exp(s A) h + s u b (decays as exponentials of base two, A2 = A log2(e)) and the lane's share of
// h . c.  (Instructions on pairs of float32 values take twice the clocks of single ones here: nothing is gained by them.)
template <int S>
struct ScanState {
  float h[S], A2[S];
  // The decays of one token, and, with them, the token: two calls, so that several tokens' exponentials can be under way.
  __device__ __forceinline__ void decays(float s, float (&e)[S]) const {
#pragma unroll
    for (int i = 0; i < S; ++i) e[i] = ssm_ex2(__fmul_rn(s, A2[i]));
  }
  __device__ __forceinline__ float token(const float (&e)[S], float su, const float (&b)[S], const float (&c)[S]) {
    float p[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      h[i] = fmaf(e[i], h[i], __fmul_rn(su, b[i]));
      p[i] = __fmul_rn(h[i], c[i]);
    }
    return sum(p);
  }
  // The token's share once more, after a step that is not finite: it has turned the zeros past state N into NaN, which do not count and
  // become zeros again.
  __device__ __forceinline__ float without_rest(const float (&c)[S], int lane, int N) {
    float p[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const bool on = scan_state<S>(lane, i) < N;
      p[i] = on ? __fmul_rn(h[i], c[i]) : 0.f;
      if (!on) h[i] = 0.f;
    }
    return sum(p);
  }
  // states that differ in bit 1, then 0, then 2 and so on (two states to a lane differ in bit 1)
  static __device__ __forceinline__ float sum(float (&p)[S]) {
    if constexpr (S >= 4) {
#pragma unroll
      for (int i = 0; i < S; i += 4) p[i] = __fadd_rn(__fadd_rn(p[i], p[i + 2]), __fadd_rn(p[i + 1], p[i + 3]));
#pragma unroll
      for (int w = 4; w < S; w *= 2)
#pragma unroll
        for (int i = 0; i < S; i += 2 * w) p[i] = __fadd_rn(p[i], p[i + w]);
    } else if constexpr (S == 2) {
      p[0] = __fadd_rn(p[0], p[1]);
    }
    return p[0];
  }
};

// Whether a step times its input is not finite
__device__ __forceinline__ bool scan_strange(float su) { return !(fabsf(su) < __int_as_float(0x7F800000)); }

// From each lane's shares of L tokens to the whole of one token: lanes that differ in one bit swap halves of what they hold, bit
// after bit.  Lane l ends with token scan_turn(l).
template <int S>
__host__ __device__ constexpr int scan_bit(int step) {  // (one state to a lane: bits 1, 0, 2, 3)
  return S == 1 && step < 2 ? 2 >> step : 1 << step;
}
template <int L, int S, int STEP = 0>
__device__ __forceinline__ float scan_join(float (&v)[L], int lane) {
  constexpr int N = (L / 2) >> STEP;
  if constexpr (N > 0) {
    constexpr int O = scan_bit<S>(STEP);
    const bool up = lane & O;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float keep = up ? v[i + N] : v[i], give = up ? v[i] : v[i + N];
      v[i] = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, give, O));
    }
    return scan_join<L, S, STEP + 1>(v, lane);
  }
  return v[0];
}
template <int L, int S>
__device__ __forceinline__ constexpr int scan_turn(int lane) {
  int t = 0;
#pragma unroll
  for (int step = 0; (L / 2) >> step > 0; ++step) t |= lane & scan_bit<S>(step) ? (L / 2) >> step : 0;
  return t;
}
template <int L, int S>
__device__ __forceinline__ constexpr int scan_owner(int token) {  // the lane that ends with it
  int l = 0;
#pragma unroll
  for (int step = 0; (L / 2) >> step > 0; ++step) l |= token & ((L / 2) >> step) ? scan_bit<S>(step) : 0;
  return l;
}

// A lane's values of a row of states that lie in one piece from p on
template <int S>
__device__ __forceinline__ void scan_floats(float (&to)[S], const float* p, int lane) {
  if constexpr (S >= 4) {
#pragma unroll
    for (int i = 0; i < S; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + lane * S + i);
      to[i] = v.x, to[i + 1] = v.y, to[i + 2] = v.z, to[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < S; ++i) to[i] = p[scan_state<S>(lane, i)];
  }
}

__device__ __forceinline__ void cp_async16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// Rows r0, r0 + STEP, ... of a column (past `last`: that one again)
template <int G, int STEP, typename T>
__device__ __forceinline__ void scan_load(const T* m, int ld, int r0, int last, uint32_t (&to)[G]) {
#pragma unroll
  for (int g = 0; g < G; ++g) to[g] = ssm_bits(m + (size_t)min(r0 + g * STEP, last) * ld);
}

// Tokens that a warp takes at a time: G groups of L, a lane prepares and ends one token of each (fewer where b and c are wide).
template <int L, int S>
struct ScanTile {
  static constexpr int NP = L * S, CH = 128 / L, G = L * NP >= 1024 ? 1 : L * NP >= 512 ? 2 : 4, TT = G * L, STAGES = 3;
  float bc[STAGES][2][TT * NP];
  float4 steps[4][2][TT / 2][32 / L];  // (s, s u) of two tokens; each warp's own, this tile's and the next one's
};

// ALL: there are NP states.  Otherwise those past N have to stay zeros whatever the steps are: one that is not finite takes its warp's tile
// through the code that leaves them out.
//
// grid (channels / CH, B): CTA (i, b) takes CH channels of sequence b through its rows, a tile of tokens at a time; L lanes share a
// channel.  For steps with few channels, all sequences' together.
//
// Warps run by themselves but for b and c, which lie in shared memory for all of them.  A lane loads u, dt and z of its tokens into
// registers (as they are stored: a conversion would wait for its load) a tile ahead of their use, makes its tokens' steps, hands them
// to the other lanes of the channel, and ends the tokens whose sums it gets.
//
// Alone on its quarter of an SM a warp takes as long as its instructions' latencies (the recurrence itself is one fused multiply-add a
// token): 58 ns a token of 16 states with L = 8, 30 with 16 (2048 rows of 1536 channels 101 us, of 256 channels 62).  With more warps it is bound by what shared memory can put into registers, 32
// values a clock and SM: the step and b and c for every lane of every channel, some 3 clocks per token and channel, against 1.2 for the
// 19 special functions (16 decays, the step's, two for the gate).
//
// Parts of a sequence beside one another (each one's end from zeros, joined, and then again from its first states) were measured as well:
// 70 us for 2048 rows of 1536 channels, but from 512 rows or 5120 channels on the other side of it nothing (27 for 28, 194 for 184),
// and results that depend on how a sequence is portioned.
template <int L, int S, bool ALL, typename TU, typename TZ>
__global__ void __launch_bounds__(128) selective_scan_kernel(const ScanArgs a) {
  using Tile = ScanTile<L, S>;
  constexpr int NP = Tile::NP, G = Tile::G, TT = Tile::TT, STAGES = Tile::STAGES, PARTS = 2 * TT * NP / 128;
  static_assert(PARTS % 4 == 0 || PARTS == 1 || PARTS == 2, "whole pieces of b and c for every thread");
  __shared__ __align__(16) Tile sm;
  pdl_wait();
  const SsmSeq q = ssm_seq(a.s, scan_sequence(a.s, blockIdx.y), blockIdx.x == 0 && threadIdx.x == 0);
  if (q.t1 <= q.t0) return;
  const int tid = threadIdx.x, lane = tid % L, turn = scan_turn<L, S>(lane), wc = tid % 32 / L, c = blockIdx.x * Tile::CH + tid / L, cc = min(c, a.C - 1);
  if (q.slot < 0) {
    if (c < a.C)
      for (int t = q.t0 + lane; t < q.t1; t += L) ssm_store(a.y, t, c, 0.f);
    return;
  }
  const int tiles = (q.t1 - q.t0 + TT - 1) / TT;
  uint32_t bits[PARTS];
  auto load_bc = [&](int i) {
    const int r0 = q.t0 + i * TT, n = min(TT, q.t1 - r0);
    if (a.wide) {
      float* to = sm.bc[i % STAGES][0];
      const float *b = reinterpret_cast<const float*>(a.b.p) + (size_t)r0 * a.b.ld, *c = reinterpret_cast<const float*>(a.c.p) + (size_t)r0 * a.c.ld;
#pragma unroll
      for (int k = 0; k < (PARTS + 3) / 4; ++k) {
        const int at = tid + 128 * k, w = at % (TT * NP / 4), t = w / (NP / 4), m = w % (NP / 4) * 4;
        if (at < 2 * TT * NP / 4 && t < n && m < a.N) cp_async16(to + at * 4, (at < TT * NP / 4 ? b + (size_t)t * a.b.ld : c + (size_t)t * a.c.ld) + m);
      }
    } else {
#pragma unroll
      for (int k = 0; k < PARTS; ++k) {
        const int at = tid + 128 * k, t = at % (TT * NP) / NP, m = at % NP;
        bits[k] = 0;
        if (t < n && m < a.N) bits[k] = ssm_bits(at < TT * NP ? a.b : a.c, r0 + t, m);
      }
    }
  };
  auto keep_bc = [&](int i) {
    if (!a.wide)
#pragma unroll
      for (int k = 0; k < PARTS; ++k) sm.bc[i % STAGES][0][tid + 128 * k] = ssm_value(tid + 128 * k < TT * NP ? a.b : a.c, bits[k]);
  };
  if (a.wide && a.N < NP)  // states that are not there
    for (int i = tid; i < STAGES * 2 * TT * NP; i += 128)
      if (i % NP >= a.N) sm.bc[0][0][i] = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (i < tiles) load_bc(i), keep_bc(i);
    cp_async_commit();
  }
  constexpr bool GATE = sizeof(TZ) > 1;
  using ZT = typename ScanGate<TZ>::type;
  const TU *U = reinterpret_cast<const TU*>(a.u.p) + cc, *DT = reinterpret_cast<const TU*>(a.dt.p) + cc;
  const ZT* Z = reinterpret_cast<const ZT*>(a.z.p) + cc;
  const int last = q.t1 - 1;
  float* state = a.state + q.slot * a.slot_stride + (size_t)cc * a.N;
  ScanState<S> h;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int n = scan_state<S>(lane, i);
    h.h[i] = n < a.N && q.pos0 > 0 ? state[n] : 0.f;
    h.A2[i] = n < a.N ? a.a[(size_t)cc * a.N + n] * 1.4426950408889634f : 0.f;
  }
  const float D = a.d != nullptr ? a.d[cc] : 0.f, bias = a.dt_bias != nullptr ? a.dt_bias[cc] : 0.f;
  // What does not wait for the recurrence is done beside it: in turn i the steps of tile i + 1 are made and the tokens of tile i - 1
  // ended, and what they need was loaded a turn before.
  uint32_t pu[G], pd[G], eu[G], ez[G];  // u and dt of the tile whose steps are made, u and z of the one that is ended
  float y[G];
  auto prepare = [&](float2 (&step)[G]) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      step[g].x = ssm_softplus(ssm_value<TU>(pd[g]) + bias);
      step[g].y = __fmul_rn(step[g].x, ssm_value<TU>(pu[g]));
    }
  };
  auto keep_steps = [&](int i, const float2 (&step)[G]) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int t = g * L + turn;
      reinterpret_cast<float2*>(&sm.steps[tid / 32][i & 1][t / 2][wc])[t & 1] = step[g];
    }
  };
  auto end = [&](float (&r)[G]) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      r[g] = fmaf(D, ssm_value<TU>(eu[g]), y[g]);
      if constexpr (GATE) r[g] = __fmul_rn(r[g], ssm_silu(ssm_value<TZ>(ez[g])));
    }
  };
  auto store = [&](int i, const float (&r)[G]) {
    const int r0 = q.t0 + i * TT + turn;
    if constexpr (G == 1) {
      if (i >= 0 && r0 < q.t1 && c < a.C) ssm_store(a.y, r0, c, r[0]);
    } else {
#pragma unroll
      for (int g = 0; g < G; g += 2) {
        const int r1 = r0 + g * L, r2 = r1 + L;
        ssm_store2(a.y, r1, r2, c, c, make_float2(r[g], r[g + 1]), i >= 0 && r1 < q.t1 && c < a.C, i >= 0 && r2 < q.t1 && c < a.C);
      }
    }
  };
  // Whether a warp's tile has steps that only the code for any step takes right
  auto odd = [&](const float2 (&step)[G]) {
    if constexpr (ALL) return false;
    bool any = false;
#pragma unroll
    for (int g = 0; g < G; ++g) any |= scan_strange(step[g].y);
    return __any_sync(0xffffffffu, any) != 0;
  };
  bool strange;
  scan_load<G, L>(U, a.u.ld, q.t0 + turn, last, pu);
  scan_load<G, L>(DT, a.dt.ld, q.t0 + turn, last, pd);
  {
    uint32_t nu[G], nd[G];
    scan_load<G, L>(U, a.u.ld, q.t0 + TT + turn, last, nu);
    scan_load<G, L>(DT, a.dt.ld, q.t0 + TT + turn, last, nd);
    float2 step[G];
    prepare(step);
    keep_steps(0, step);
    strange = odd(step);
#pragma unroll
    for (int g = 0; g < G; ++g) pu[g] = nu[g], pd[g] = nd[g], eu[g] = ez[g] = 0, y[g] = 0.f;
  }
  for (int i = 0; i < tiles; ++i) {
    cp_async_wait<1>();
    __syncthreads();  // tile i of b and c is there, tile i - 1 is not read any more
    if (i + 2 < tiles) load_bc(i + 2);
    cp_async_commit();
    uint32_t nu[G], nd[G], fu[G], fz[G];
    const int row = q.t0 + i * TT + turn;
    scan_load<G, L>(U, a.u.ld, row + 2 * TT, last, nu);
    scan_load<G, L>(DT, a.dt.ld, row + 2 * TT, last, nd);
    scan_load<G, L>(U, a.u.ld, row, last, fu);
    if constexpr (GATE) scan_load<G, L>(Z, a.z.ld, row, last, fz);
    float2 step[G];
    float done[G], sums[G];
    const float *Bt = sm.bc[i % STAGES][0], *Ct = sm.bc[i % STAGES][1];
    const float4(*steps)[32 / L] = sm.steps[tid / 32][i & 1];
    const int n = q.t1 - q.t0 - i * TT;
    if (n >= TT && !strange) {  // (all in one block of code, for the compiler to interleave)
      prepare(step);
      end(done);
      constexpr int P = S > 4 ? 2 : 4;  // tokens at a time: first all that does not depend on the token before
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float acc[L];
#pragma unroll
        for (int j = 0; j < L; j += P) {
          const int t = g * L + j;
          float bv[P][S], cv[P][S], e[P][S];
          float4 st[P / 2];
#pragma unroll
          for (int p = 0; p < P; p += 2) st[p / 2] = steps[(t + p) / 2][wc];
#pragma unroll
          for (int p = 0; p < P; ++p) {
            scan_floats<S>(bv[p], Bt + (t + p) * NP, lane);
            scan_floats<S>(cv[p], Ct + (t + p) * NP, lane);
          }
#pragma unroll
          for (int p = 0; p < P; ++p) h.decays(p & 1 ? st[p / 2].z : st[p / 2].x, e[p]);
#pragma unroll
          for (int p = 0; p < P; ++p) acc[j + p] = h.token(e[p], p & 1 ? st[p / 2].w : st[p / 2].y, bv[p], cv[p]);
        }
        sums[g] = scan_join<L, S>(acc, lane);
      }
    } else {  // the sequence's last tokens, or any steps
      prepare(step);
      end(done);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float acc[L];
#pragma unroll
        for (int j = 0; j < L; ++j) {
          const int t = g * L + j;
          acc[j] = 0.f;
          if (t < n) {
            float bv[S], cv[S], e[S];
            scan_floats<S>(bv, Bt + t * NP, lane);
            scan_floats<S>(cv, Ct + t * NP, lane);
            const float2 st = reinterpret_cast<const float2*>(&steps[t / 2][wc])[t & 1];
            h.decays(st.x, e);
            acc[j] = h.token(e, st.y, bv, cv);
            if (strange) acc[j] = h.without_rest(cv, lane, a.N);
          }
        }
        sums[g] = scan_join<L, S>(acc, lane);
      }
    }
    store(i - 1, done);
    keep_steps(i + 1, step);
    strange = odd(step);
    if (i + 2 < tiles) keep_bc(i + 2);
#pragma unroll
    for (int g = 0; g < G; ++g) pu[g] = nu[g], pd[g] = nd[g], eu[g] = fu[g], ez[g] = GATE ? fz[g] : 0, y[g] = sums[g];
  }
  // (only now: CTAs of the next kernel that came before would be spread over the SMs by where this one's are)
  pdl_launch_dependents();
  {
    float done[G];
    end(done);
    store(tiles - 1, done);
  }
  if (c < a.C)
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (scan_state<S>(lane, i) < a.N) state[scan_state<S>(lane, i)] = h.h[i];
}

// The same with a lane to a channel and all of its states in registers, where there are channels enough to fill the SMs so: nothing is
// handed from lane to lane, u, dt, z and y are whole lines of memory, and b and c come from shared memory to all lanes at once.
// grid (channels / CW, B), CW threads; SB tokens of b and c at a time, TT of the rest.
//
// Bound by its instructions: 174 of them for a token and warp, which fill 64 % of the issue slots, and 20 special functions a channel (the
// 16 decays among them), 56 % of that unit's; 248 registers leave two warps to a scheduler (with 168, three, 404 us).  9 sequences
// of 331 to 1650 rows, 5120 channels: 402 us where the special functions alone take 189 and memory 60.  Lengths that differ are part of it:
// 1440 one-warp blocks on 1184 places, and the longest sequence runs to the end.
template <int NP>
struct ScanWide {
  static constexpr int CW = 32, SB = 32, TT = 8, STAGES = 3;
};
// One channel of a sequence, from its start, token by token: where a step was not finite and there are states past N, which it turned into
// NaN.  Only the state's end shows it: a look at every step cost up to 12 %.
template <int NP>
__device__ __forceinline__ void scan_channel(const ScanArgs& a, const SsmSeq& q, int c) {
  float* state = a.state + q.slot * a.slot_stride + (size_t)c * a.N;
  ScanState<NP> h;
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    h.h[n] = n < a.N && q.pos0 > 0 ? state[n] : 0.f;
    h.A2[n] = n < a.N ? a.a[(size_t)c * a.N + n] * 1.4426950408889634f : 0.f;
  }
  const float D = a.d != nullptr ? a.d[c] : 0.f, bias = a.dt_bias != nullptr ? a.dt_bias[c] : 0.f;
#pragma unroll 1
  for (int r = q.t0; r < q.t1; ++r) {
    const float u = ssm_load(a.u, r, c), s = ssm_softplus(ssm_load(a.dt, r, c) + bias);
    float e[NP], bv[NP], cv[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      bv[n] = n < a.N ? ssm_load(a.b, r, n) : 0.f;
      cv[n] = n < a.N ? ssm_load(a.c, r, n) : 0.f;
    }
    h.decays(s, e);
    h.token(e, __fmul_rn(s, u), bv, cv);
    float v = fmaf(D, u, h.without_rest(cv, 0, a.N));
    if (a.z.p != nullptr) v = __fmul_rn(v, ssm_silu(ssm_load(a.z, r, c)));
    ssm_store(a.y, r, c, v);
  }
#pragma unroll
  for (int n = 0; n < NP; ++n)
    if (n < a.N) state[n] = h.h[n];
}
template <int NP, bool ALL, typename TU, typename TZ>
__global__ void __launch_bounds__(ScanWide<NP>::CW) selective_scan_wide_kernel(const ScanArgs a) {
  using W = ScanWide<NP>;
  constexpr int CW = W::CW, SB = W::SB, TT = W::TT, STAGES = W::STAGES, PARTS = 2 * SB * NP / CW;
  __shared__ __align__(16) float bc[STAGES][2][SB * NP];
  pdl_wait();
  const SsmSeq q = ssm_seq(a.s, scan_sequence(a.s, blockIdx.y), blockIdx.x == 0 && threadIdx.x == 0);
  if (q.t1 <= q.t0) return;
  const int tid = threadIdx.x, c = blockIdx.x * CW + tid, cc = min(c, a.C - 1);
  if (q.slot < 0) {
    if (c < a.C)
      for (int t = q.t0; t < q.t1; ++t) ssm_store(a.y, t, c, 0.f);
    return;
  }
  const int blocks = (q.t1 - q.t0 + SB - 1) / SB;
  uint32_t bits[PARTS];
  auto load_bc = [&](int i) {
    const int r0 = q.t0 + i * SB, n = min(SB, q.t1 - r0);
    if (a.wide) {
      float* to = bc[i % STAGES][0];
      const float *b = reinterpret_cast<const float*>(a.b.p) + (size_t)r0 * a.b.ld, *c = reinterpret_cast<const float*>(a.c.p) + (size_t)r0 * a.c.ld;
#pragma unroll
      for (int k = 0; k < PARTS / 4; ++k) {
        const int at = tid + CW * k, w = at % (SB * NP / 4), t = w / (NP / 4), m = w % (NP / 4) * 4;
        if (t < n && m < a.N) cp_async16(to + at * 4, (at < SB * NP / 4 ? b + (size_t)t * a.b.ld : c + (size_t)t * a.c.ld) + m);
      }
    } else {
#pragma unroll
      for (int k = 0; k < PARTS; ++k) {
        const int at = (tid + CW * k) % (SB * NP), t = at / NP, m = at % NP;
        bits[k] = 0;
        if (t < n && m < a.N) bits[k] = ssm_bits(k < PARTS / 2 ? a.b : a.c, r0 + t, m);
      }
    }
  };
  auto keep_bc = [&](int i) {
    if (!a.wide)
#pragma unroll
      for (int k = 0; k < PARTS; ++k) bc[i % STAGES][0][tid + CW * k] = ssm_value(k < PARTS / 2 ? a.b : a.c, bits[k]);
  };
  if (a.wide && a.N < NP)  // states that are not there
    for (int i = tid; i < STAGES * 2 * SB * NP; i += CW)
      if (i % NP >= a.N) bc[0][0][i] = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (i < blocks) load_bc(i), keep_bc(i);
    cp_async_commit();
  }
  constexpr bool GATE = sizeof(TZ) > 1;
  const TU *U = reinterpret_cast<const TU*>(a.u.p) + cc, *DT = reinterpret_cast<const TU*>(a.dt.p) + cc;
  using ZT = typename ScanGate<TZ>::type;
  const ZT* Z = reinterpret_cast<const ZT*>(a.z.p) + cc;
  float* state = a.state + q.slot * a.slot_stride + (size_t)cc * a.N;
  ScanState<NP> h;
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    h.h[n] = n < a.N && q.pos0 > 0 ? state[n] : 0.f;
    h.A2[n] = n < a.N ? a.a[(size_t)cc * a.N + n] * 1.4426950408889634f : 0.f;
  }
  const float D = a.d != nullptr ? a.d[cc] : 0.f, bias = a.dt_bias != nullptr ? a.dt_bias[cc] : 0.f;
  uint32_t u[TT], dt[TT], z[TT];
  auto load = [&](int r0, uint32_t (&u)[TT], uint32_t (&dt)[TT], uint32_t (&z)[TT]) {
    if (r0 + TT <= q.t1) {
      const TU *pu = U + (size_t)r0 * a.u.ld, *pd = DT + (size_t)r0 * a.dt.ld;
      const ZT* pz = Z + (GATE ? (size_t)r0 * a.z.ld : 0);
#pragma unroll
      for (int t = 0; t < TT; ++t, pu += a.u.ld, pd += a.dt.ld, pz += GATE ? a.z.ld : 0) {
        u[t] = ssm_bits(pu), dt[t] = ssm_bits(pd);
        if constexpr (GATE) z[t] = ssm_bits(pz);
      }
    } else {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const size_t r = min(r0 + t, q.t1 - 1);  // (past the last row: that one again)
        u[t] = ssm_bits(U + r * a.u.ld), dt[t] = ssm_bits(DT + r * a.dt.ld);
        if constexpr (GATE) z[t] = ssm_bits(Z + r * a.z.ld);
      }
    }
  };
  load(q.t0, u, dt, z);
  for (int i = 0; i < blocks; ++i) {
    cp_async_wait<1>();
    __syncthreads();  // b and c of these tokens are there, those of the block before are not read any more
    if (i + 2 < blocks) load_bc(i + 2);
    cp_async_commit();
    const float *Bt = bc[i % STAGES][0], *Ct = bc[i % STAGES][1];
    const int r1 = min(q.t0 + (i + 1) * SB, q.t1);
#pragma unroll 1
    for (int r0 = q.t0 + i * SB; r0 < r1; r0 += TT, Bt += TT * NP, Ct += TT * NP) {
      uint32_t nu[TT], nd[TT], nz[TT];
      load(r0 + TT, nu, nd, nz);
      float step[TT], y[TT];
      auto token = [&](int t) {
        float e[NP], bv[NP], cv[NP];
        scan_floats<NP>(bv, Bt + t * NP, 0);
        scan_floats<NP>(cv, Ct + t * NP, 0);
        h.decays(step[t], e);
        return h.token(e, __fmul_rn(step[t], ssm_value<TU>(u[t])), bv, cv);
      };
      auto end = [&](int t) {
        float v = fmaf(D, ssm_value<TU>(u[t]), y[t]);
        if constexpr (GATE) v = __fmul_rn(v, ssm_silu(ssm_value<TZ>(z[t])));
        return v;
      };
#pragma unroll
      for (int t = 0; t < TT; ++t) step[t] = ssm_softplus(ssm_value<TU>(dt[t]) + bias);
      if (r0 + TT <= r1) {
#pragma unroll
        for (int t = 0; t < TT; ++t) y[t] = token(t);
#pragma unroll
        for (int t = 0; t < TT; t += 2)
          ssm_store2(a.y, r0 + t, r0 + t + 1, c, c, make_float2(end(t), end(t + 1)), c < a.C, c < a.C);
      } else {
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (r0 + t < r1) {
            y[t] = token(t);
            if (c < a.C) ssm_store(a.y, r0 + t, c, end(t));
          }
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) u[t] = nu[t], dt[t] = nd[t], z[t] = GATE ? nz[t] : 0;
    }
    if (i + 2 < blocks) keep_bc(i + 2);
  }
  pdl_launch_dependents();
  if (!ALL && h.h[NP - 1] != 0.f) {  // (NaN)
    if (c < a.C) scan_channel<NP>(a, q, c);
    return;
  }
  if (c < a.C)
#pragma unroll
    for (int n = 0; n < NP; ++n)
      if (n < a.N) state[n] = h.h[n];
}

// Steps of one row per sequence.  grid (channels / (128 / L), B / L): a thread takes its states of L sequences through their tokens,
// lane l prepares and ends one sequence's.  Bound by memory: the states are read and written once (256 sequences of 5120 channels with
// 16 states: 40.6 us, 4.5 TB/s; with nine blocks to an SM 43, with a group's loads ahead of the one before it, which takes registers, 49).
template <int L, int S, bool ALL>
__global__ void __launch_bounds__(128, L * S <= 16 ? 10 : 1) selective_step_kernel(const ScanArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x % L, c = blockIdx.x * (128 / L) + threadIdx.x / L, cc = min(c, a.C - 1);
  const int b = blockIdx.y * L + scan_turn<L, S>(lane);
  SsmSeq q{0, 0, -1, 0};
  if (b < a.s.B) q = ssm_seq(a.s, b, blockIdx.x == 0 && threadIdx.x < L);
  const bool on = q.t1 == q.t0 + 1, live = on && q.slot >= 0;
  if (q.t1 > q.t0 + 1) {  // more rows than the caller said
    if (blockIdx.x == 0 && threadIdx.x < L) oxb_report(OXB_BAD_ARGUMENT, q.t1 - q.t0);
    if (c < a.C)
      for (int t = q.t0; t < q.t1; ++t) ssm_store(a.y, t, c, 0.f);
  }
  uint32_t ub = 0, db = 0, zb = 0;
  if (live) {
    ub = ssm_bits(a.u, q.t0, cc);
    db = ssm_bits(a.dt, q.t0, cc);
    if (a.z.p != nullptr) zb = ssm_bits(a.z, q.t0, cc);
  }
  const float D = a.d != nullptr ? a.d[cc] : 0.f, bias = a.dt_bias != nullptr ? a.dt_bias[cc] : 0.f;
  const int slot = live ? q.slot : -1;
  float A2[S], first[L][S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int n = scan_state<S>(lane, i);
    A2[i] = n < a.N ? a.a[(size_t)cc * a.N + n] * 1.4426950408889634f : 0.f;
  }
#pragma unroll
  for (int j = 0; j < L; ++j) {
    const int s = __shfl_sync(0xffffffffu, slot, scan_owner<L, S>(j), L), p = __shfl_sync(0xffffffffu, q.pos0, scan_owner<L, S>(j), L);
    const float* from = a.state + s * a.slot_stride + (size_t)cc * a.N;
#pragma unroll
    for (int i = 0; i < S; ++i) first[j][i] = 0.f;
    if (s >= 0 && p > 0) {
      if (a.whole) {
        scan_floats<S>(first[j], from, lane);
      } else {
#pragma unroll
        for (int i = 0; i < S; ++i)
          if (scan_state<S>(lane, i) < a.N) first[j][i] = from[scan_state<S>(lane, i)];
      }
    }
  }
  const float u = ssm_value(a.u, ub), dt = ssm_softplus(ssm_value(a.dt, db) + bias), du = __fmul_rn(dt, u);
  float acc[L];
#pragma unroll
  for (int j = 0; j < L; ++j) {
    const int owner = scan_owner<L, S>(j), s = __shfl_sync(0xffffffffu, slot, owner, L), t = __shfl_sync(0xffffffffu, q.t0, owner, L);
    const float dtj = __shfl_sync(0xffffffffu, dt, owner, L), duj = __shfl_sync(0xffffffffu, du, owner, L);
    acc[j] = 0.f;
    if (s < 0) continue;
    float bv[S], cv[S];
    if (S >= 4 && a.wide) {
      scan_floats<S>(bv, reinterpret_cast<const float*>(a.b.p) + (size_t)t * a.b.ld, lane);
      scan_floats<S>(cv, reinterpret_cast<const float*>(a.c.p) + (size_t)t * a.c.ld, lane);
    } else {
      uint32_t bb[S], cb[S];
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const int n = scan_state<S>(lane, i);
        bb[i] = n < a.N ? ssm_bits(a.b, t, n) : 0u;
        cb[i] = n < a.N ? ssm_bits(a.c, t, n) : 0u;
      }
#pragma unroll
      for (int i = 0; i < S; ++i) bv[i] = ssm_value(a.b, bb[i]), cv[i] = ssm_value(a.c, cb[i]);
    }
    ScanState<S> h;
#pragma unroll
    for (int i = 0; i < S; ++i) h.h[i] = first[j][i], h.A2[i] = A2[i];
    float e[S];
    h.decays(dtj, e);
    acc[j] = h.token(e, duj, bv, cv);
    if constexpr (!ALL)
      if (scan_strange(duj)) acc[j] = h.without_rest(cv, lane, a.N);
    if (c < a.C) {
      float* to = a.state + s * a.slot_stride + (size_t)cc * a.N;
      if (S >= 4 && a.whole) {
#pragma unroll
        for (int i = 0; i + 3 < S; i += 4) __stcs(reinterpret_cast<float4*>(to + lane * S + i), make_float4(h.h[i], h.h[i + 1], h.h[i + 2], h.h[i + 3]));
      } else {
#pragma unroll
        for (int i = 0; i < S; ++i)
          if (scan_state<S>(lane, i) < a.N) to[scan_state<S>(lane, i)] = h.h[i];
      }
    }
  }
  float y = scan_join<L, S>(acc, lane);
  if (on && c < a.C) {
    y = fmaf(D, u, y);
    if (a.z.p != nullptr) y = __fmul_rn(y, ssm_silu(ssm_value(a.z, zb)));
    ssm_store(a.y, q.t0, c, live ? y : 0.f);
  }
}

}  // namespace oxb
