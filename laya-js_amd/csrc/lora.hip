// Low-rank adapters of many requests beside a shared projection
// (hb_lora_linear, hb_lora_qlinear):
//
//   y_m = x_m . w^T (+ bias) + scale_i * (x_m . A_i^T) . B_i^T,   i = index[m]
//
// with a bank of n adapters A [n, R, K], B [n, N, R]; a row whose index is
// outside [0, n) has none.
//
// lora_shrink_any, lora_expand_any: the inner products s = scale_i x_m . A_i^T
// in f32, then y = round(y + s . B_i^T) on top of the projection, any type and
// size.
#include <stdexcept>

#include "common.h"

namespace hb {

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
  if (hb_qlinear(ctx, dt, x, ldx, qw, qscales, zeros, bias, 0, 0, y, ldy, M, N, K, bits, group, mode,
                 bias ? HB_EPI_BIAS : 0))
    return -1;
  add_adapters(ctx, "hb_lora_qlinear", dt, x, ldx, y, ldy, M, N, K, l);
  HB_API_END
}

}  // extern "C"
