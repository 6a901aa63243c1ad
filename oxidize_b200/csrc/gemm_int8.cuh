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
// Bits of |x| of two bf16 values order as the values do, with infinity and NaN (>= 0x7F80) on top.
__device__ __forceinline__ uint32_t abs_bits_x2(uint32_t v) { return v & 0x7FFF7FFFu; }

__device__ __forceinline__ int int8_code(float x, float most) { return __float2int_rn(__fdiv_rn(127.f * x, most)); }

// grid (T): one token to a block
__global__ void __launch_bounds__(256) quantize_tokens_kernel(const __nv_bfloat16* __restrict__ x, int K, int8_t* __restrict__ q, int ld_q,
                                                              float* __restrict__ scales) {
  __shared__ uint32_t red[8];
  pdl_launch_dependents();
  pdl_wait();
  const __nv_bfloat16* row = x + (size_t)blockIdx.x * K;
  int8_t* out = q + (size_t)blockIdx.x * ld_q;
  uint32_t most = 0;
  for (int k = threadIdx.x; k < K; k += 256) most = max(most, (uint32_t)(__bfloat16_as_ushort(row[k]) & 0x7FFF));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, red[i]);
  float m = __uint_as_float(most << 16);
  const bool fine = most < 0x7F80;
  if (threadIdx.x == 0) scales[blockIdx.x] = fine ? __fdiv_rn(m, 127.f) : __uint_as_float(0x7FC00000u);
  // (127 x of the largest values would pass float32's range: both sides of the quotient are scaled)
  const float by = m > 1e30f ? 0.0009765625f : 1.f;
  m *= by;
  for (int k = threadIdx.x; k < K; k += 256) out[k] = fine && most > 0 ? (int8_t)int8_code(__bfloat162float(row[k]) * by, m) : 0;
}

// ----------------------------------------------------------------------------------------------------------- product
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

constexpr int I8_BM = 128, I8_BK = 128;  // weight rows of a tile; values of a k-block (one 128-byte swizzle row)
constexpr int I8_THREADS = 192;          // warps 0-3: epilogue, 4: TMA, 5: MMA

template <int TN>
struct I8Tile {
  static constexpr int A_BYTES = I8_BM * I8_BK, B_BYTES = TN * I8_BK, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = TN <= 64 ? 4 : TN == 128 ? 6 : 4;
  static constexpr int COLS = TN < 32 ? 32 : TN;  // of tensor memory
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 /*alignment*/ + 256 /*barriers*/ + TN * 4 /*token scales*/;
};

struct I8Args {
  __nv_bfloat16* y;
  const float *sx, *sw, *bias;
  int N, T, K, ld_y, wide;  // wide: rows of y start on 16-byte boundaries and hold whole groups of 8
};

// grid (weight tiles, 1, token tiles)
template <int TN>
__global__ void __launch_bounds__(I8_THREADS, 1)
gemm_int8_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const I8Args a) {
  using Cfg = I8Tile<TN>;
  extern __shared__ uint8_t i8_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8_smem) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::STAGES * Cfg::STAGE_BYTES);
  uint64_t *empty = full + Cfg::STAGES, *accum = empty + Cfg::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* tok_scale = reinterpret_cast<float*>(smem + Cfg::STAGES * Cfg::STAGE_BYTES + 256);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // token tiles innermost: a weight tile is fetched from HBM once
  const int lin = blockIdx.z * gridDim.x + blockIdx.x, tile_n = lin / (int)gridDim.z, tile_t = lin % (int)gridDim.z;
  const int n0 = tile_n * I8_BM, t0 = tile_t * TN, nkb = (a.K + I8_BK - 1) / I8_BK;
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
    if (leader)  // weights are static: they need not wait for the tokens
      for (int i = 0; i < npre; ++i) {
        mbar_expect_tx(&full[i], Cfg::STAGE_BYTES);
        tma_load_2d(smem + i * Cfg::STAGE_BYTES, &tmW, &full[i], i * I8_BK, n0);
      }
    pdl_wait();
    if (leader)
      for (int i = 0; i < npre; ++i) tma_load_2d(smem + i * Cfg::STAGE_BYTES + Cfg::A_BYTES, &tmX, &full[i], i * I8_BK, t0);
    int st = npre == Cfg::STAGES ? 0 : npre;
    uint32_t ph = 0;
    for (int i = npre; i < nkb; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&empty[st], ph, abort_flag, OXB_TIMEOUT_TMA_EMPTY, blockIdx.x))) break;
      if (leader) {
        mbar_expect_tx(&full[st], Cfg::STAGE_BYTES);
        tma_load_2d(smem + st * Cfg::STAGE_BYTES, &tmW, &full[st], i * I8_BK, n0);
        tma_load_2d(smem + st * Cfg::STAGE_BYTES + Cfg::A_BYTES, &tmX, &full[st], i * I8_BK, t0);
      }
      if (++st == Cfg::STAGES) st = 0, ph ^= 1;
    }
  } else if (warp == 5) {
    const bool leader = elect_one();
    const uint32_t base = smem_u32(smem);
    int st = 0;
    uint32_t ph = 0;
    for (int i = 0; i < nkb; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[st], ph, abort_flag, OXB_TIMEOUT_TMA_FULL, blockIdx.x))) break;
      tc_fence_after();
      if (leader) {
        const uint64_t ad = umma_desc_k_sw128(base + st * Cfg::STAGE_BYTES), bd = umma_desc_k_sw128(base + st * Cfg::STAGE_BYTES + Cfg::A_BYTES);
#pragma unroll
        for (int k = 0; k < I8_BK / 32; ++k)  // 32 values = 32 bytes of the swizzle row: +2 in the (address >> 4) field
          umma_i8(tmem, ad + 2 * k, bd + 2 * k, umma_idesc_i8(I8_BM, TN), i > 0 || k > 0);
        umma_commit(&empty[st]);
      }
      if (++st == Cfg::STAGES) st = 0, ph ^= 1;
    }
    if (leader) {
      umma_commit(accum);
      mbar_wait_bounded(accum, 0, abort_flag, OXB_TIMEOUT_ACCUM, blockIdx.x);
    }
    __syncwarp();
    asm volatile("bar.arrive 3, 160;" ::: "memory");
  } else {
    pdl_wait();  // the tokens' scales
    const int tvalid = min(TN, a.T - t0);
    for (int j = threadIdx.x; j < tvalid; j += 128) tok_scale[j] = a.sx[t0 + j];
    const int row = warp * 32 + lane, n = n0 + row;
    const float sw = n < a.N ? a.sw[n] : 0.f, b = n < a.N && a.bias != nullptr ? a.bias[n] : 0.f;
    asm volatile("bar.sync 3, 160;" ::: "memory");
    tc_fence_after();
    if (!*abort_flag) {
      // [token][128 rows] in bf16 over the idle ring, then rows of 16 bytes
      __nv_bfloat16* stage = reinterpret_cast<__nv_bfloat16*>(smem);
      for (int c = 0; c < TN / 16; ++c) {
        if (c * 16 >= tvalid) break;
        uint32_t r[16];
        tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c * 16, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int t = c * 16 + j;
          if (t < tvalid) stage[t * I8_BM + row] = __float2bfloat16(__int2float_rn((int)r[j]) * tok_scale[t] * sw + b);
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const int tid = threadIdx.x;
      if (a.wide) {
        const int chunk = tid & 15;
        if (n0 + chunk * 8 < a.N)
          for (int t = tid >> 4; t < tvalid; t += 8)
            *reinterpret_cast<uint4*>(a.y + (size_t)(t0 + t) * a.ld_y + n0 + chunk * 8) =
                *reinterpret_cast<const uint4*>(stage + t * I8_BM + chunk * 8);
      } else if (n < a.N) {
        for (int t = 0; t < tvalid; ++t) a.y[(size_t)(t0 + t) * a.ld_y + n] = stage[t * I8_BM + row];
      }
    }
  }
  if (*abort_flag)  // a wait gave up: copies in flight get time to land
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  tc_fence_before();
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem, Cfg::COLS);
}

}  // namespace oxb
