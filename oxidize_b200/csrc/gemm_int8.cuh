// Y[T, N] = (Xq[T, K] . Wq[N, K]^T) * sx[T] * sw[N] (+ bias[N]) on 8-bit integers, whole-number sums in tensor memory, bf16 out.
//
// Weights are int8 codes with a scale per output channel; activations get theirs here, one scale per token:
// sx = max|x| / 127, code = rint(127 x / max|x|).  For bf16 values 127 x is exact in float32 and a quotient of such values is
// either a half or further from one than a division's rounding, so rint of the float32 division is the exact code.
//
// Orientation as in gemm_tcgen05.cuh: the MMA's M (128) runs over weight rows, its N over tokens.
#pragma once
#include "common.cuh"

namespace oxb {

// ------------------------------------------------------------------------------------------------ tokens to integers
// A token's largest value (m, scaled by `by` so that neither 127 x nor 127 / m leaves float32's range) and what its codes need.
struct I8Scale {
  float m, by, r;  // r = 127 / m
  bool zero;       // codes are 0: a row of zeros, or one that is not finite
};
// From the largest of the bf16 values' bits without their signs, which order as the values do, infinity and NaN (>= 0x7F80) on top;
// *scale: max|x| / 127, or NaN.
__device__ __forceinline__ I8Scale int8_scale(uint32_t most, float* scale) {
  I8Scale s;
  const float m = __uint_as_float(most << 16);
  s.zero = most == 0 || most >= 0x7F80;
  s.by = m > 1e30f ? 0x1p-64f : m < 1e-30f ? 0x1p64f : 1.f;
  s.m = m * s.by;
  s.r = __fdiv_rn(127.f, s.m);
  *scale = most >= 0x7F80 ? __uint_as_float(0x7FC00000u) : __fdiv_rn(m, 127.f);
  return s;
}
// rint(127 x / max|x|), ties to even, exactly: a first guess from the rounded reciprocal is off by one at most, next to halves, and its
// remainder 127 x - code m (exact: few bits on either side) says where.
__device__ __forceinline__ int int8_code(float x, const I8Scale& s) {
  x *= s.by;
  const float t = fmaf(x, s.r, 12582912.f), q = t - 12582912.f;  // 1.5 * 2^23: rounds to a whole number
  const float e = 2.f * fmaf(-q, s.m, 127.f * x);
  int c = (int)(__float_as_uint(t) - 0x4B400000u);
  if (fabsf(e) > s.m || (fabsf(e) == s.m && (c & 1))) c += e > 0.f ? 1 : -1;
  return s.zero ? 0 : c;
}
__device__ __forceinline__ uint32_t int8_codes4(uint32_t lo, uint32_t hi, const I8Scale& s) {  // four bf16 values
  const float2 a = unpack_bf16x2(lo), b = unpack_bf16x2(hi);
  return (uint32_t)(int8_code(a.x, s) & 255) | (uint32_t)(int8_code(a.y, s) & 255) << 8 | (uint32_t)(int8_code(b.x, s) & 255) << 16 |
         (uint32_t)int8_code(b.y, s) << 24;
}
__device__ __forceinline__ uint32_t int8_max2(uint32_t most, uint32_t v) {  // of the halves' bits without their signs
  return __vmaxu2(most, v & 0x7FFF7FFFu);
}
// The largest of a block's values; `red`: a word for each warp
__device__ __forceinline__ uint32_t int8_block_max(uint32_t most, uint32_t* red) {
  most = max(most & 0xFFFF, most >> 16);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
  __syncthreads();
  for (int i = 0; i < (int)blockDim.x / 32; ++i) most = max(most, red[i]);
  return most;
}

// grid (T): one token to a block.  Bound by memory: a token's values stay in registers between their maximum and their codes (up to
// 256 * 8 * HELD of them, the rest is read twice, the second time from L2).  wide: rows on 16-byte boundaries of whole 16-byte pieces.
template <int HELD>
__global__ void __launch_bounds__(256) quantize_tokens_kernel(const __nv_bfloat16* __restrict__ x, int K, int wide, int8_t* __restrict__ q, int ld_q,
                                                              float* __restrict__ scales) {
  __shared__ uint32_t red[8];
  pdl_launch_dependents();
  pdl_wait();
  const __nv_bfloat16* row = x + (size_t)blockIdx.x * K;
  int8_t* out = q + (size_t)blockIdx.x * ld_q;
  const int tid = threadIdx.x;
  uint32_t most = 0;
  if (wide) {
    const uint4* from = reinterpret_cast<const uint4*>(row);
    const int n = K / 8;
    uint4 v[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      v[i] = make_uint4(0, 0, 0, 0);
      if (tid + 256 * i < n) v[i] = from[tid + 256 * i];
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) most = int8_max2(int8_max2(int8_max2(int8_max2(most, v[i].x), v[i].y), v[i].z), v[i].w);
    for (int i = tid + 256 * HELD; i < n; i += 256) {
      const uint4 w = from[i];
      most = int8_max2(int8_max2(int8_max2(int8_max2(most, w.x), w.y), w.z), w.w);
    }
    most = int8_block_max(most, red);
    float scale;
    const I8Scale s = int8_scale(most, &scale);
    if (tid == 0) scales[blockIdx.x] = scale;
    uint2* to = reinterpret_cast<uint2*>(out);
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (tid + 256 * i < n) to[tid + 256 * i] = make_uint2(int8_codes4(v[i].x, v[i].y, s), int8_codes4(v[i].z, v[i].w, s));
    for (int i = tid + 256 * HELD; i < n; i += 256) {
      const uint4 w = from[i];
      to[i] = make_uint2(int8_codes4(w.x, w.y, s), int8_codes4(w.z, w.w, s));
    }
  } else {
    for (int k = tid; k < K; k += 256) most = int8_max2(most, __bfloat16_as_ushort(row[k]));
    most = int8_block_max(most, red);
    float scale;
    const I8Scale s = int8_scale(most, &scale);
    if (tid == 0) scales[blockIdx.x] = scale;
    for (int k = tid; k < K; k += 256) out[k] = (int8_t)int8_code(__bfloat162float(row[k]), s);
  }
}

// --------------------------------------------------------------------------------------------------------- one token
// grid (N / (8 ROWS)): a warp takes ROWS weight rows with dot products of four codes; every block makes the token's codes for itself
// (from L2, which saves a launch) while its first weights are on their way.  Bound by the weights' bytes (10240 x 2560: 6.7 us, 3.9 TB/s, 10.7 with
// two launches and tensor cores; two tokens here 10.4, there 8.1, so only one comes here).  Shared memory: K codes, padded to 512.
template <int ROWS>
__global__ void __launch_bounds__(256) gemv_int8_kernel(const __nv_bfloat16* __restrict__ x, int wide, const int8_t* __restrict__ w, int ld_w,
                                                        const float* __restrict__ sw, const float* __restrict__ bias, __nv_bfloat16* __restrict__ y, int N,
                                                        int K) {
  extern __shared__ __align__(16) int8_t gv_codes[];
  __shared__ uint32_t red[8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row0 = (blockIdx.x * 8 + warp) * ROWS, padded = (K + 511) / 512 * 512;
  const int8_t* rows[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) rows[r] = w + (size_t)min(row0 + r, N - 1) * ld_w;
  // 512 values of a row at a time, 16 to a lane
  auto load = [&](int k0, uint4 (&v)[ROWS]) {
    const int k = k0 + lane * 16;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      v[r] = make_uint4(0, 0, 0, 0);
      if (k + 16 <= K) {
        v[r] = __ldcs(reinterpret_cast<const uint4*>(rows[r] + k));
      } else if (k < K) {  // the last ones, one by one
        uint32_t b[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k + i < K) b[i / 4] |= (uint32_t)(uint8_t)rows[r][k + i] << (i % 4 * 8);
        v[r] = make_uint4(b[0], b[1], b[2], b[3]);
      }
    }
  };
  uint4 v0[ROWS], v1[ROWS];
  load(0, v0);  // (weights: no kernel writes them)
  load(512, v1);
  pdl_launch_dependents();
  pdl_wait();
  float scale;
  {
    const uint4* from = reinterpret_cast<const uint4*>(x);
    const int n = wide ? K / 8 : 0;
    uint4 held = make_uint4(0, 0, 0, 0);  // a thread's first eight values
    if (tid < n) held = from[tid];
    uint32_t most = int8_max2(int8_max2(int8_max2(int8_max2(0, held.x), held.y), held.z), held.w);
    for (int i = tid + 256; i < n; i += 256) {
      const uint4 v = from[i];
      most = int8_max2(int8_max2(int8_max2(int8_max2(most, v.x), v.y), v.z), v.w);
    }
    for (int k = n * 8 + tid; k < K; k += 256) most = int8_max2(most, __bfloat16_as_ushort(x[k]));
    const I8Scale s = int8_scale(int8_block_max(most, red), &scale);
    uint2* to = reinterpret_cast<uint2*>(gv_codes);
    if (tid < n) to[tid] = make_uint2(int8_codes4(held.x, held.y, s), int8_codes4(held.z, held.w, s));
    for (int i = tid + 256; i < n; i += 256) {
      const uint4 v = from[i];
      to[i] = make_uint2(int8_codes4(v.x, v.y, s), int8_codes4(v.z, v.w, s));
    }
    for (int k = n * 8 + tid; k < padded; k += 256) gv_codes[k] = k < K ? (int8_t)int8_code(__bfloat162float(x[k]), s) : 0;
  }
  __syncthreads();
  int acc[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) acc[r] = 0;
  for (int k0 = 0; k0 < K; k0 += 512) {
    uint4 next[ROWS];
    load(k0 + 1024, next);
    const uint4 c = *reinterpret_cast<const uint4*>(gv_codes + k0 + lane * 16);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      acc[r] = __dp4a((int)c.x, (int)v0[r].x, __dp4a((int)c.y, (int)v0[r].y, __dp4a((int)c.z, (int)v0[r].z, __dp4a((int)c.w, (int)v0[r].w, acc[r]))));
#pragma unroll
    for (int r = 0; r < ROWS; ++r) v0[r] = v1[r], v1[r] = next[r];
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    int a = acc[r];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (lane == 0 && row0 + r < N)
      y[row0 + r] = __float2bfloat16(__int2float_rn(a) * sw[row0 + r] * scale + (bias != nullptr ? bias[row0 + r] : 0.f));
  }
}

// ----------------------------------------------------------------------------------------------------------- product
// A wait of at most a second (a thread's polls pause in hardware for a time that is not ours to say, so the bound is on the clock):
// then the status word gets `code`, the CTA's flag goes up, and every later wait returns at once.
__device__ __forceinline__ bool int8_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int code, int detail) {
  if (mbar_try_wait(bar, parity)) return true;
  uint64_t begin, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(begin));
  do {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
  } while (now - begin < 1000000000ull);
  *abort_flag = 1;
  oxb_report(code, detail);
  return false;
}

// instruction descriptor for kind::i8, signed x signed -> s32, both operands K-major
__host__ __device__ constexpr uint32_t umma_idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

constexpr int I8_BM = 128, I8_BK = 128;  // weight rows of an MMA; values of a k-block (one 128-byte swizzle row)
constexpr int I8_THREADS = 192;          // warps 0-3: epilogue, 4: TMA, 5: MMA (which owns the tensor memory)

// A tile of 128 RB weight rows x TN tokens.  A tile of 128 x 256 wants 48 KB per 512 clocks of products on every SM (27 TB/s over all of them),
// so many tokens take tiles of 256 x 256, which fill the tensor memory with their two accumulators: a third less per product (8192
// tokens of 8192 x 8192: 445 to 474 us, 2.3 to 2.5 P operations a second; 575 with 128 x 256).  Which limit those meet is not established:
// 64 bytes a clock come into each SM (some 11 TB/s over all of them at the measured time), and shared memory takes those and gives the
// products 96 more, with 128 a clock.
template <int TN, int RB>
struct I8Tile {
  static constexpr int A_BYTES = RB * I8_BM * I8_BK, B_BYTES = TN * I8_BK, STAGE_BYTES = A_BYTES + B_BYTES;
  // tiles of up to 64 tokens leave room for a second CTA on the SM: the next kernel's, or another split
  static constexpr int STAGES = TN <= 64 ? 4 : TN == 128 ? 6 : RB == 1 ? 4 : 3;
  static constexpr int COLS = (TN < 32 ? 32 : TN) * RB;  // of tensor memory
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 /*alignment*/ + 256 /*barriers*/ + TN * 4 /*token scales*/;
};

struct I8Args {
  __nv_bfloat16* y;
  const float *sx, *sw, *bias;
  int N, T, K, ld_y, wide;  // wide: rows of y start on 16-byte boundaries and hold whole groups of 8
  int token_tiles;
  int whole;  // RB = 2: tiles ahead of this one are whole, the others halves of 128 weight rows
};

// A sum with its row's and its token's scale, in this order: a large token's scale alone would take the sum past float32's range.  The
// sum's two halves become float32 by their bits and are joined with one rounding: as the conversion instruction, which is one of the slow
// special function unit's.
__device__ __forceinline__ float int8_result(int sum, float sx, float sw, float b) {
  const float hi = __uint_as_float(0x4B400000u + (uint32_t)(sum >> 16)) - 12582912.f, lo = __uint_as_float(0x4B000000u | ((uint32_t)sum & 0xFFFF)) - 8388608.f;
  return fmaf(hi, 65536.f, lo) * sw * sx + b;
}

// [token][128 rows] of bf16 in shared memory to y's rows, by 128 threads
__device__ __forceinline__ void int8_store_rows(const __nv_bfloat16* stage, int tokens, int t0, int n0, const I8Args& a, int tid) {
  if (a.wide) {
    const int chunk = tid & 15;
    if (n0 + chunk * 8 < a.N)
      for (int t = tid >> 4; t < tokens; t += 8)
        *reinterpret_cast<uint4*>(a.y + (size_t)(t0 + t) * a.ld_y + n0 + chunk * 8) = *reinterpret_cast<const uint4*>(stage + t * I8_BM + chunk * 8);
  } else if (n0 + tid < a.N) {
    for (int t = 0; t < tokens; ++t) a.y[(size_t)(t0 + t) * a.ld_y + n0 + tid] = stage[t * I8_BM + tid];
  }
}

// grid (tiles, splits).  RB = 2: the tiles of a last wave that fills less than half of the SMs come as halves.  With splits the CTAs of a
// tile are a cluster along K: whole-number sums meet in distributed shared memory, each CTA ends its share of the tokens (in any order
// the same sum; RB = 1 only).
template <int TN, int RB>
__global__ void __launch_bounds__(I8_THREADS, 1)
gemm_int8_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const I8Args a) {
  using Cfg = I8Tile<TN, RB>;
  extern __shared__ uint8_t i8_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8_smem) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::STAGES * Cfg::STAGE_BYTES);
  uint64_t *empty = full + Cfg::STAGES, *accum = empty + Cfg::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* tok_scale = reinterpret_cast<float*>(smem + Cfg::STAGES * Cfg::STAGE_BYTES + 256);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, splits = gridDim.y;
  // token tiles innermost: a weight tile is fetched from HBM once
  int tile = blockIdx.x, half = 0, rb = RB;
  if (RB == 2 && tile >= a.whole) half = (tile - a.whole) & 1, tile = a.whole + (tile - a.whole) / 2, rb = 1;
  const int tile_n = tile / a.token_tiles, tile_t = tile % a.token_tiles;
  const int n0 = (tile_n * RB + half) * I8_BM, t0 = tile_t * TN, kbs = (a.K + I8_BK - 1) / I8_BK;
  const int kb0 = (int)((long long)blockIdx.y * kbs / splits), nkb = (int)((long long)(blockIdx.y + 1) * kbs / splits) - kb0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Cfg::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(accum, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, Cfg::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  if (warp == 4) {
    const bool leader = elect_one();
    const int npre = nkb < Cfg::STAGES ? nkb : Cfg::STAGES;
    const uint64_t once = l2_policy_evict_first();
    auto load_w = [&](int i, int st) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        if (r >= rb) break;
        uint8_t* to = smem + st * Cfg::STAGE_BYTES + r * (I8_BM * I8_BK);
        // (weights that one token tile reads need not stay in L2)
        if (TN <= 128 && a.token_tiles == 1) tma_load_2d_hint(to, &tmW, &full[st], (kb0 + i) * I8_BK, n0 + r * I8_BM, once);
        else tma_load_2d(to, &tmW, &full[st], (kb0 + i) * I8_BK, n0 + r * I8_BM);
      }
    };
    auto load_x = [&](int i, int st) { tma_load_2d(smem + st * Cfg::STAGE_BYTES + Cfg::A_BYTES, &tmX, &full[st], (kb0 + i) * I8_BK, t0); };
    if (leader)  // weights are static: they need not wait for the tokens
      for (int i = 0; i < npre; ++i) {
        mbar_expect_tx(&full[i], rb * (I8_BM * I8_BK) + Cfg::B_BYTES);
        load_w(i, i);
      }
    pdl_wait();
    if (leader)
      for (int i = 0; i < npre; ++i) load_x(i, i);
    int st = npre == Cfg::STAGES ? 0 : npre;
    uint32_t ph = 0;
    for (int i = npre; i < nkb; ++i) {
      if (!__all_sync(0xffffffffu, int8_wait(&empty[st], ph, abort_flag, OXB_TIMEOUT_TMA_EMPTY, blockIdx.x))) break;
      if (leader) {
        mbar_expect_tx(&full[st], rb * (I8_BM * I8_BK) + Cfg::B_BYTES);
        load_w(i, st);
        load_x(i, st);
      }
      if (++st == Cfg::STAGES) st = 0, ph ^= 1;
    }
  } else if (warp == 5) {
    const bool leader = elect_one();
    const uint32_t base = smem_u32(smem);
    // No operands come before the tokens do: ahead of this the bound on waits would count what earlier kernels still have to do (an
    // all-reduce may wait for its peers longer than that).
    pdl_wait();
    int st = 0;
    uint32_t ph = 0;
    for (int i = 0; i < nkb; ++i) {
      if (!__all_sync(0xffffffffu, int8_wait(&full[st], ph, abort_flag, OXB_TIMEOUT_TMA_FULL, blockIdx.x))) break;
      tc_fence_after();
      if (leader) {
        const uint64_t ad = umma_desc_k_sw128(base + st * Cfg::STAGE_BYTES), bd = umma_desc_k_sw128(base + st * Cfg::STAGE_BYTES + Cfg::A_BYTES);
#pragma unroll
        for (int k = 0; k < I8_BK / 32; ++k)  // 32 values = 32 bytes of the swizzle row: +2 in the (address >> 4) field
#pragma unroll
          for (int r = 0; r < RB; ++r)
            if (r < rb) umma_i8(tmem + r * TN, ad + r * (I8_BM * I8_BK >> 4) + 2 * k, bd + 2 * k, umma_idesc_i8(I8_BM, TN), i > 0 || k > 0);
        umma_commit(&empty[st]);
      }
      if (++st == Cfg::STAGES) st = 0, ph ^= 1;
    }
    if (leader) {
      umma_commit(accum);
      int8_wait(accum, 0, abort_flag, OXB_TIMEOUT_ACCUM, blockIdx.x);
    }
    __syncwarp();
    asm volatile("bar.arrive 3, 160;" ::: "memory");
  } else {
    pdl_wait();  // the tokens' scales
    const int tvalid = min(TN, a.T - t0);
    for (int j = threadIdx.x; j < tvalid; j += 128) tok_scale[j] = a.sx[t0 + j];
    const int row = warp * 32 + lane;
    asm volatile("bar.sync 3, 160;" ::: "memory");
    tc_fence_after();
    // over the ring, which is idle: [token][128 rows] in bf16, or, with splits, the sums of all tokens and then those results
    __nv_bfloat16* stage = reinterpret_cast<__nv_bfloat16*>(smem + (splits > 1 ? TN * I8_BM * 4 : 0));
    int* sums = reinterpret_cast<int*>(smem);
    const bool fine = !*abort_flag;
#pragma unroll 1
    for (int r = 0; r < rb; ++r) {
      const int n1 = n0 + r * I8_BM, n = n1 + row;
      const float sw = n < a.N ? a.sw[n] : 0.f, b = n < a.N && a.bias != nullptr ? a.bias[n] : 0.f;
      if (fine) {
        for (int c = 0; c * 16 < tvalid; ++c) {
          uint32_t v[16];
          tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + r * TN + c * 16, v);
          tmem_ld_wait();
          if (splits > 1) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (c * 16 + j < tvalid) sums[(c * 16 + j) * I8_BM + row] = (int)v[j];
          } else {  // (past the last token: whatever the scales' place holds, and nobody's)
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const int t = c * 16 + j;
              const __nv_bfloat162 y = __floats2bfloat162_rn(int8_result((int)v[j], tok_scale[t], sw, b), int8_result((int)v[j + 1], tok_scale[t + 1], sw, b));
              stage[t * I8_BM + row] = y.x;
              stage[(t + 1) * I8_BM + row] = y.y;
            }
          }
        }
      }
      if (splits > 1) {  // (RB = 1)
        cluster_sync_all();
        const int share = (tvalid + splits - 1) / splits, j0 = min(tvalid, (int)blockIdx.y * share), j1 = min(tvalid, j0 + share);
        if (fine)
          for (int t = j0; t < j1; t += 8) {  // (eight tokens' loads under way together)
            int sum[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) sum[u] = 0;
            for (int s = 0; s < splits; ++s) {
              const uint32_t from = dsmem_map(smem_u32(sums + t * I8_BM + row), s);
              int v[8];
#pragma unroll
              for (int u = 0; u < 8; ++u) v[u] = t + u < j1 ? __float_as_int(dsmem_ld_f32(from + u * (I8_BM * 4))) : 0;
#pragma unroll
              for (int u = 0; u < 8; ++u) sum[u] += v[u];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
              if (t + u < j1) stage[(t + u) * I8_BM + row] = __float2bfloat16(int8_result(sum[u], tok_scale[t + u], sw, b));
          }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (fine) int8_store_rows(stage + j0 * I8_BM, j1 - j0, t0 + j0, n1, a, threadIdx.x);
      } else {
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (fine) int8_store_rows(stage, tvalid, t0, n1, a, threadIdx.x);
        if (r + 1 < rb) asm volatile("bar.sync 1, 128;" ::: "memory");  // (the stage is written again)
      }
    }
  }
  if (splits > 1) {
    __syncwarp();
    if (warp >= 4) cluster_sync_all();
    cluster_sync_all();  // (the others may still be reading this CTA's sums)
  }
  if (*abort_flag)  // a wait gave up: copies in flight get time to land
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  tc_fence_before();
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem, Cfg::COLS);
}

}  // namespace oxb
