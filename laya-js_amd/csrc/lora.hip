// Low-rank adapters of many requests beside a shared projection
// (hb_lora_linear, hb_lora_qlinear):
//
//   y_m = x_m . w^T (+ bias) + scale_i * (x_m . A_i^T) . B_i^T,   i = index[m]
//
// with a bank of n adapters A [n, R, K], B [n, N, R]; a row whose index is
// outside [0, n) has none.
//
// lora_shrink: s = scale_i x_m . A_i^T of f16 / bf16 rows on v_mfma_f32_16x16x32,
// rounded to the 16-bit type for the second product, which the projection's own
// GEMM takes as ranks beyond K (gemm_ring with LoraExt): y is rounded once.
//
// lora_shrink_any, lora_expand_any: the inner products s = scale_i x_m . A_i^T
// in f32, then y = round(y + s . B_i^T) on top of the projection, any type and
// size.
#include <algorithm>
#include <stdexcept>

#include "gemm_kernels.h"

namespace hb {

// ------------------------------------------------------------------ f16 / bf16

// A block takes 16 MT rows and 64 ranks; its four waves share out K by 64 and
// their sums meet in LDS.  The rows' distinct adapters are gone through one after
// another, for all rows of the block, and a row keeps its own adapter's sums;
// with few row blocks those are shared out over gridDim.z.  Bound by reading x
// once (and A from the caches); at few rows by the chain of loads.
template <bool BF16, int MT>
__global__ __launch_bounds__(256) void lora_shrink(const uint16_t* __restrict__ X, int64_t ldx,
                                                   const uint16_t* __restrict__ A, const float* __restrict__ scales,
                                                   const int32_t* __restrict__ index, int n, int M, int R, int K,
                                                   uint16_t* __restrict__ S) {
  __shared__ __attribute__((aligned(16))) float red[4][MT * 16][68];  // 64 ranks, padded against bank conflicts
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = blockIdx.x * 16 * MT, r0 = blockIdx.y * 64;
  int a = lane < 16 * MT && m0 + lane < M ? index[m0 + lane] : -1;
  if (a >= n) a = -1;
  uint64_t left = __ballot(a >= 0);
  const uint16_t* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; i++) xr[i] = X + (int64_t)min(m0 + 16 * i + l16, M - 1) * ldx + 8 * g;
  for (int turn = 0; left != 0; turn++) {
    const int cur = __builtin_amdgcn_readlane(a, __builtin_ctzll(left));
    const uint64_t same = __ballot(a == cur);
    left &= ~same;
    if (turn % gridDim.z != blockIdx.z) continue;  // (the same in every wave)
    const uint16_t* ar[4];
#pragma unroll
    for (int t = 0; t < 4; t++) ar[t] = A + ((int64_t)cur * R + min(r0 + 16 * t + l16, R - 1)) * K + 8 * g;
    float4v acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int t = 0; t < 4; t++) acc[i][t] = float4v{0.f, 0.f, 0.f, 0.f};
    const int nt = min((R - r0 + 15) >> 4, 4);  // rank blocks there are
    for (int k = wave * 64; k < K; k += 256) {
      uint4v xf[MT][2];
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int s = 0; s < 2; s++) xf[i][s] = *(const uint4v*)(xr[i] + k + 32 * s);
#pragma unroll
      for (int t = 0; t < 4; t++) {
        if (t >= nt) break;
#pragma unroll
        for (int s = 0; s < 2; s++) {
          const uint4v af = *(const uint4v*)(ar[t] + k + 32 * s);
#pragma unroll
          for (int i = 0; i < MT; i++) {
            if constexpr (BF16)
              acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, af),
                                                                  __builtin_bit_cast(bf16x8, xf[i][s]), acc[i][t], 0, 0, 0);
            else
              acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, af),
                                                                 __builtin_bit_cast(half8, xf[i][s]), acc[i][t], 0, 0, 0);
          }
        }
      }
    }
    // lane: row l16 of its block, ranks 16 t + 4 g ..
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int t = 0; t < 4; t++) *(float4v*)&red[wave][16 * i + l16][16 * t + 4 * g] = acc[i][t];
    __syncthreads();
    const float sc = scales[cur];
    for (int q = tid; q < 16 * MT * 16; q += 256) {  // four ranks of a row
      const int row = q >> 4, r = (q & 15) * 4;
      if (!((same >> row) & 1) || r0 + r >= R) continue;  // (R % 8 == 0)
      float4v v = *(const float4v*)&red[0][row][r];
#pragma unroll
      for (int w = 1; w < 4; w++) v += *(const float4v*)&red[w][row][r];
      const uint32_t h[4] = {from_f<BF16>(v[0] * sc), from_f<BF16>(v[1] * sc), from_f<BF16>(v[2] * sc),
                             from_f<BF16>(v[3] * sc)};
      *(uint2v*)(S + (int64_t)(m0 + row) * R + r0 + r) = uint2v{h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
    }
    __syncthreads();  // the sums are written again
  }
}

// The ring's tile for the projection with adapters.
template <bool BF16>
static void lora_ring(hipStream_t st, int cus, const uint16_t* x, int64_t ldx, const uint16_t* w, const uint16_t* bias,
                      uint16_t* y, int64_t ldy, int M, int N, int K, const LoraExt& ext) {
  auto go = [&](auto launch) { launch(st, 0u, x, ldx, w, bias, (const uint16_t*)nullptr, (int64_t)0, y, ldy, M, N, K, ext); };
  LinearKernel tile = LinearKernel::kRing64x64x3;
  ring_tile(cus, M, N, K, false, true, false, &tile);
  if (M >= 4096) tile = LinearKernel::kRing128x256;
  switch (tile) {
    case LinearKernel::kRing32x64: return go(launch_ring_t<32, 64, 1, 2, 6, BF16, false, LoraExt>);
    case LinearKernel::kRing64x64: return go(launch_ring_t<64, 64, 2, 2, 4, BF16, false, LoraExt>);
    case LinearKernel::kRing64x64k: return go(launch_ring_t<64, 64, 2, 2, 5, BF16, false, LoraExt>);
    case LinearKernel::kRing128x64: return go(launch_ring_t<128, 64, 4, 2, 4, BF16, false, LoraExt>);
    case LinearKernel::kRing128x256: return go(launch_ring_t<128, 256, 4, 4, 3, BF16, false, LoraExt>);
    default: return go(launch_ring_t<64, 64, 2, 2, 3, BF16, false, LoraExt>);
  }
}

// ------------------------------------------------------------------ any type

// One wave per row and rank.
__global__ __launch_bounds__(256) void lora_shrink_any(int dt, const void* __restrict__ X, int64_t ldx,
                                                       const void* __restrict__ A, const float* __restrict__ scales,
                                                       const int32_t* __restrict__ index, int n, int64_t M, int R,
                                                       int K, float* __restrict__ S) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= M * R) return;
  const int64_t m = i / R;
  const int r = (int)(i - m * R), a = index[m];
  float s = 0.f;
  if (a >= 0 && a < n) {
    const int64_t row = ((int64_t)a * R + r) * K;
    for (int k = lane; k < K; k += 64) s = fmaf(load_f(X, m * ldx + k, dt), load_f(A, row + k, dt), s);
    s = wave_sum(s) * scales[a];
  }
  if (lane == 0) S[i] = s;
}

// One thread per output.
__global__ __launch_bounds__(256) void lora_expand_any(int dt, const float* __restrict__ S, const void* __restrict__ Bk,
                                                       const int32_t* __restrict__ index, int n, int64_t M, int N,
                                                       int R, void* __restrict__ Y, int64_t ldy) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
    const int a = index[m];
    if (a < 0 || a >= n) continue;
    const int64_t row = ((int64_t)a * N + c) * R;
    float d = 0.f;
    for (int r = 0; r < R; r++) d = fmaf(S[m * R + r], load_f(Bk, row + r, dt), d);
    store_f(Y, m * ldy + c, dt, load_f(Y, m * ldy + c, dt) + d);
  }
}

struct LoraArgs {
  uintptr_t a, b, scales, index;
  int64_t n, R;
};

static void check_lora(const char* op, int dt, int64_t M, int64_t N, int64_t K, const LoraArgs& l) {
  auto need = [&](bool ok, const char* what) {
    if (!ok) throw std::runtime_error(std::string(op) + ": " + what);
  };
  need(dt == HB_F32 || dt == HB_F16 || dt == HB_BF16, "dtype must be f32, f16 or bf16");
  need(M >= 0 && N >= 0 && K >= 0 && M < (1ll << 31) && N < (1ll << 30) && K < (1ll << 30), "bad sizes");
  need(l.n >= 0 && l.n < (1ll << 30) && l.R >= 0 && l.R <= 1024, "bad adapter count or rank (at most 1024)");
  need(l.n * l.R == 0 || M == 0 || N == 0 || K == 0 || (l.a && l.b && l.scales && l.index), "null adapter argument");
}

// The MFMA path: 16-bit types, K and the operands as the ring takes them, whole
// chunks of ranks, a bank that 32-bit offsets reach.
static bool lora_takes_ring(int dt, uintptr_t x, int64_t ldx, uintptr_t w, uintptr_t y, int64_t ldy, int64_t M, int64_t N,
                            int64_t K, const LoraArgs& l) {
  return (dt == HB_F16 || dt == HB_BF16) && M > 0 && N > 0 && K > 0 && l.n > 0 && l.R > 0 && ring_ok(ldx, K) &&
         l.R % 8 == 0 && ldx % 8 == 0 && ldy % 8 == 0 && (x | w | y | l.a | l.b) % 16 == 0 &&
         l.n * l.R * N * 2 < (1ll << 31);
}

// The projection with adapters on 16-bit weights; false: no memory for the inner
// products.
static bool lora_fused(uintptr_t ctx, int dt, const uint16_t* x, int64_t ldx, const uint16_t* w, const uint16_t* bias,
                       uint16_t* y, int64_t ldy, int M, int N, int K, const LoraArgs& l) {
  CallScratch held(ctx);
  if (!held.take((size_t)M * l.R * 2)) return false;
  uint16_t* S = (uint16_t*)held.p;
  hipStream_t st = stream_of(ctx);
  const int cus = cu_count(ctx);
  auto shrink = [&](auto kern, int rows) {
    const unsigned gx = (unsigned)((M + rows - 1) / rows), gy = (unsigned)((l.R + 63) / 64);
    const int64_t blocks = (int64_t)gx * gy;
    const unsigned gz = (unsigned)std::max<int64_t>(1, std::min<int64_t>({l.n, rows, cus / blocks}));
    kern<<<dim3(gx, gy, gz), 256, 0, st>>>(x, ldx, (const uint16_t*)l.a, (const float*)l.scales, (const int32_t*)l.index,
                                           (int)l.n, M, (int)l.R, K, S);
  };
  const bool bf = dt == HB_BF16;
  if (M >= 8192) shrink(bf ? lora_shrink<true, 2> : lora_shrink<false, 2>, 32);
  else shrink(bf ? lora_shrink<true, 1> : lora_shrink<false, 1>, 16);
  check_launch("hb_lora_linear");
  const LoraExt ext{S, (const uint16_t*)l.b, (const int32_t*)l.index, (int)l.n, (int)l.R};
  if (bf) lora_ring<true>(st, cus, x, ldx, w, bias, y, ldy, M, N, K, ext);
  else lora_ring<false>(st, cus, x, ldx, w, bias, y, ldy, M, N, K, ext);
  check_launch("hb_lora_linear");
  return true;
}

static void add_adapters(uintptr_t ctx, const char* op, int dt, uintptr_t x, int64_t ldx, uintptr_t y, int64_t ldy,
                         int64_t M, int64_t N, int64_t K, const LoraArgs& l) {
  if (M == 0 || N == 0 || K == 0 || l.n * l.R == 0) return;
  CallScratch s(ctx);
  if (!s.take((size_t)(M * l.R * 4)))
    throw std::runtime_error(std::string(op) + ": out of device memory for the adapters' inner products");
  hipStream_t st = stream_of(ctx);
  HB_REQUIRE((M * l.R + 3) / 4 < (1ll << 31), "hb_lora_linear: too many rows and ranks");
  lora_shrink_any<<<(unsigned)((M * l.R + 3) / 4), 256, 0, st>>>(dt, (const void*)x, ldx, (const void*)l.a,
                                                                 (const float*)l.scales, (const int32_t*)l.index,
                                                                 (int)l.n, M, (int)l.R, (int)K, (float*)s.p);
  const dim3 grid((unsigned)((N + 255) / 256), (unsigned)(M < 65535 ? M : 65535));
  lora_expand_any<<<grid, 256, 0, st>>>(dt, (const float*)s.p, (const void*)l.b, (const int32_t*)l.index, (int)l.n, M,
                                        (int)N, (int)l.R, (void*)y, ldy);
  check_launch(op);
}

}  // namespace hb

using namespace hb;

extern "C" {

int hb_lora_linear(uintptr_t ctx, int dt, uintptr_t x, int64_t ldx, uintptr_t w, uintptr_t bias, uintptr_t y,
                   int64_t ldy, int64_t M, int64_t N, int64_t K, uintptr_t a, uintptr_t b, uintptr_t scales, int64_t n,
                   int64_t R, uintptr_t index) {
  HB_API_BEGIN
  const LoraArgs l{a, b, scales, index, n, R};
  check_lora("hb_lora_linear", dt, M, N, K, l);
  HB_REQUIRE(ldx >= K && ldy >= N, "hb_lora_linear: leading dimension smaller than the row");
  if (lora_takes_ring(dt, x, ldx, w, y, ldy, M, N, K, l) &&
      lora_fused(ctx, dt, (const uint16_t*)x, ldx, (const uint16_t*)w, (const uint16_t*)bias, (uint16_t*)y, ldy, (int)M,
                 (int)N, (int)K, l))
    return 0;
  if (hb_linear(ctx, dt, x, ldx, w, bias, 0, 0, y, ldy, M, N, K, bias ? HB_EPI_BIAS : 0)) return -1;
  add_adapters(ctx, "hb_lora_linear", dt, x, ldx, y, ldy, M, N, K, l);
  HB_API_END
}

int hb_lora_qlinear(uintptr_t ctx, int dt, uintptr_t x, int64_t ldx, uintptr_t qw, uintptr_t qscales, uintptr_t zeros,
                    uintptr_t bias, uintptr_t y, int64_t ldy, int64_t M, int64_t N, int64_t K, int bits, int group,
                    int mode, uintptr_t a, uintptr_t b, uintptr_t scales, int64_t n, int64_t R, uintptr_t index) {
  HB_API_BEGIN
  const LoraArgs l{a, b, scales, index, n, R};
  check_lora("hb_lora_qlinear", dt, M, N, K, l);
  HB_REQUIRE(ldx >= K && ldy >= N, "hb_lora_qlinear: leading dimension smaller than the row");
  HB_REQUIRE((bits == 8 || bits == 4) && (mode == 0 || mode == 1) && group > 0, "hb_lora_qlinear: bad bits, mode or group");
  HB_REQUIRE(qw && qscales && (mode == 0 || zeros), "hb_lora_qlinear: missing weight tensors");
  if (lora_takes_ring(dt, x, ldx, 0, y, ldy, M, N, K, l) && group % 8 == 0 && qw % 8 == 0 && qscales % 2 == 0 &&
      zeros % 2 == 0) {
    // the weight dequantized into a 16-bit copy, as hb_qlinear does
    CallScratch copy(ctx);
    if (copy.take((size_t)(N * K * 2))) {
      const QW q{(const uint8_t*)qw, (const void*)qscales, (const void*)zeros, (int)((K + group - 1) / group), group};
      dequantize_rows(stream_of(ctx), cu_count(ctx), dt, bits, mode, q, (uint16_t*)copy.p, N, (int)K);
      check_launch("hb_lora_qlinear (dequantize)");
      if (lora_fused(ctx, dt, (const uint16_t*)x, ldx, (const uint16_t*)copy.p, (const uint16_t*)bias, (uint16_t*)y, ldy,
                     (int)M, (int)N, (int)K, l))
        return 0;
    }
  }
  if (hb_qlinear(ctx, dt, x, ldx, qw, qscales, zeros, bias, 0, 0, y, ldy, M, N, K, bits, group, mode,
                 bias ? HB_EPI_BIAS : 0))
    return -1;
  add_adapters(ctx, "hb_lora_qlinear", dt, x, ldx, y, ldy, M, N, K, l);
  HB_API_END
}

}  // extern "C"
