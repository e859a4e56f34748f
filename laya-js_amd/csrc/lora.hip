// Low-rank adapters of many requests beside a shared projection
// (hb_lora_linear, hb_lora_qlinear):
//
//   y_m = x_m . w^T (+ bias) + scale_i * (x_m . A_i^T) . B_i^T,   i = index[m]
//
// with a bank of n adapters A [n, R, K], B [n, N, R]; a row whose index is
// outside [0, n) has none.
//
// lora_prepare: s = scale_i x_m . A_i^T on v_mfma_f32_16x16x32 (f32: 16x16x4).  Of f16 /
// bf16 rows it is rounded to the 16-bit type for the second product, which the
// projection's own GEMM takes as ranks beyond K: gemm_ring with LoraExt, lora_stream
// for large M, lora_few for few tiles.  y is rounded once.  An element of s past the
// type's range (f16: 65504) makes the row's outputs infinite or NaN there; they are
// computed again one by one with its f32 value, a slow path for rows that are rare.
//
// lora_expand_f32: y += s . B_i^T of f32 rows past lora_few, on top of the projection.
//
// lora_shrink_any, lora_expand_any: the inner products in f32, then y = round(y + s .
// B_i^T), any type and size.
#include <algorithm>
#include <stdexcept>

#include "gemm_kernels.h"

namespace hb {

// ------------------------------------------------------------------ f16 / bf16

// lora_stream: rows and columns of a tile, stages of its ring, their width, waves
constexpr int kStTile = 256, kStStages = 4, kStBK = 32, kStWaves = 8;
constexpr int kStStage = 2 * kStTile * kStBK;  // u16 of a stage
constexpr int kStLds = kStStages * kStStage * 2;

// The adapters of lora_stream's tiles of rows, as LoraExt describes them.
struct Numbers {
  int16_t* number;        // [tiles * 256]: each row's adapter's number in its tile of 256 rows, or -1
  int32_t *list, *count;  // [tiles * 256]: the adapters by number; [tiles]
  int tiles;              // 0: gemm_ring numbers them itself (48 rows of 24 adapters: 17 us, with numbers from here 19)
};

// A quantized weight [N, K] and its 16-bit copy.
struct Codes {
  QW q;
  uint16_t* copy;
  int bits, mode;    // 8 or 4, 1: affine
  int N, K, blocks;  // 0 blocks: none
};

// What the projection's GEMM needs beforehand, in one launch (runs of blocks): the
// rows' inner products with their adapters, the numbers, and the weight's copy, as
// hb_qlinear makes it.  (With a launch of its own for the copy: 54
// rows x 1024 x 2624 35 -> 30 us.)
struct Prepare {
  const char* x;
  int64_t ldx;
  const char* a;
  const float* scales;
  const int32_t* index;
  int n, M, R, K;
  void* s;                   // [M, R], of x's type
  float* wide;               // [M, R], 16-bit types: four elements of s where one of them is past the type's range
  Numbers num;
  Codes codes;
  int gx, gy, gz;            // inner products: row blocks, rank blocks, turns
};

// Rows of 128 bytes in LDS, written by direct-to-LDS loads (8 rows a load: 8 lanes a
// row, so that it reads whole lines; fragments loaded straight into registers, 16 rows
// by 64 bytes, take a CU's L1 longer: 16k x 1024, rank 64, 24 us against 17; 48 rows x 1024
// x 2624, 24 adapters of rank 64, 19 against 13 with the projection), read as MFMA fragments: chunk c of
// row r at c ^ row_f(r), so that the 16 rows of a pass cover all banks.
__device__ __forceinline__ int row_f(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ uint4v lora_records(const void* p) {
  const uint64_t a = (uint64_t)p;
  return uint4v{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a),
                (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu), 0x80000000u, 0x00020000u};
}
// Byte offset of the lane's chunk of piece i of rows of `bytes`, those behind `last`
// clamped to it
__device__ __forceinline__ uint32_t piece_offset(int i, int lane, int last, uint32_t bytes) {
  const int r = i * 8 + (lane >> 3);
  return (uint32_t)min(r, last) * bytes + (((lane & 7) ^ row_f(r)) << 4);
}
__device__ __forceinline__ uint4v row_chunk(const char* rows, int r, int c) {
  return *(const uint4v*)(rows + r * 128 + ((c ^ row_f(r)) << 4));
}
template <int DT>
__device__ __forceinline__ float4v mfma16(uint4v a, uint4v b, float4v c) {
  if constexpr (DT == HB_F32) {  // of a lane's four k each product takes one
    const float4v av = __builtin_bit_cast(float4v, a), bv = __builtin_bit_cast(float4v, b);
#pragma unroll
    for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(av[e], bv[e], c, 0, 0, 0);
    return c;
  } else if constexpr (DT == HB_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  }
}

// Inner products.  A block takes 16 MT rows and 16 NT ranks; its four waves share out K
// by 128 bytes, each through two buffers of its own with no barrier, and their sums meet
// in LDS.  The rows' distinct adapters are gone through one after another, for all rows
// of the block, and a row keeps its own adapter's sums; with few row blocks those are
// shared out over gz blocks.  Bound by reading x once (and A from the caches); at few
// rows by the chain of loads and one CU's reading of A, so that blocks take 16 ranks
// then (48 x 2624, 29 adapters of rank 64: 14.9 -> 8.3 us).
template <int DT, int MT, int NT>
__device__ __forceinline__ void lora_inner(const Prepare& p, int bx, int by, int bz, char* lds) {
  constexpr int NW = 4, ES = DT == HB_F32 ? 4 : 2, KC = 128 / ES, BUF = (MT + NT) * 2048, L = 2 * (MT + NT);
  auto red = (float(*)[MT * 16][NT * 16 + 4])lds;  // [NW], padded against bank conflicts
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = bx * 16 * MT, r0 = by * 16 * NT, R = p.R, K = p.K;
  int a = lane < 16 * MT && m0 + lane < p.M ? p.index[m0 + lane] : -1;
  if (a >= p.n) a = -1;
  uint64_t left = __ballot(a >= 0);
  uint32_t xo[2 * MT], ao[2 * NT];
#pragma unroll
  for (int i = 0; i < 2 * MT; i++) xo[i] = piece_offset(i, lane, p.M - 1 - m0, (uint32_t)p.ldx * ES);
#pragma unroll
  for (int i = 0; i < 2 * NT; i++) ao[i] = piece_offset(i, lane, R - 1 - r0, (uint32_t)K * ES);
  const uint4v xs = lora_records(p.x + (int64_t)m0 * p.ldx * ES);
  const char* mine = lds + wave * 2 * BUF;
  const uint32_t at0 = (uint32_t)__builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)mine);
  for (int turn = 0; left != 0; turn++) {
    const int cur = __builtin_amdgcn_readlane(a, __builtin_ctzll(left));
    const uint64_t same = __ballot(a == cur);
    left &= ~same;
    if (turn % p.gz != bz) continue;  // (the same in every wave)
    const float sc = p.scales[cur];
    const uint4v as = lora_records(p.a + ((int64_t)cur * R + r0) * K * ES);
    float4v acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int t = 0; t < NT; t++) acc[i][t] = float4v{0.f, 0.f, 0.f, 0.f};
    auto request = [&](int k, int slot) __attribute__((always_inline)) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's reads of the buffer are done
      const uint32_t to = at0 + (uint32_t)(slot * BUF);
#pragma unroll
      for (int i = 0; i < 2 * MT; i++) buffer_lds16(xs, xo[i], (uint32_t)k * ES, to + 1024u * i);
#pragma unroll
      for (int i = 0; i < 2 * NT; i++) buffer_lds16(as, ao[i], (uint32_t)k * ES, to + 1024u * (2 * MT + i));
    };
    int slot = 0;
    if (wave * KC < K) request(wave * KC, 0);
    for (int k = wave * KC; k < K; k += NW * KC, slot ^= 1) {
      if (k + NW * KC < K) {
        request(k + NW * KC, slot ^ 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      const char* rows = mine + slot * BUF;
#pragma unroll
      for (int s = 0; s < 2; s++) {
        uint4v xf[MT], af[NT];
#pragma unroll
        for (int i = 0; i < MT; i++) xf[i] = row_chunk(rows, 16 * i + l16, 4 * s + g);
#pragma unroll
        for (int t = 0; t < NT; t++) af[t] = row_chunk(rows + MT * 2048, 16 * t + l16, 4 * s + g);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int i = 0; i < MT; i++) acc[i][t] = mfma16<DT>(af[t], xf[i], acc[i][t]);
      }
    }
    __syncthreads();  // everybody is done with the buffers
    // lane: row l16 of its block, ranks 16 t + 4 g ..
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int t = 0; t < NT; t++) *(float4v*)&red[wave][16 * i + l16][16 * t + 4 * g] = acc[i][t];
    __syncthreads();
    for (int q = tid; q < 16 * MT * 4 * NT; q += 64 * NW) {  // four ranks of a row
      const int row = q / (4 * NT), r = q % (4 * NT) * 4;
      if (!((same >> row) & 1) || r0 + r >= R) continue;  // (R % 4 == 0)
      float4v v = *(const float4v*)&red[0][row][r];
#pragma unroll
      for (int w = 1; w < NW; w++) v += *(const float4v*)&red[w][row][r];
      v *= sc;
      const int64_t at = (int64_t)(m0 + row) * R + r0 + r;
      if constexpr (DT == HB_F32) {
        *(float4v*)((float*)p.s + at) = v;
      } else {
        constexpr bool BF16 = DT == HB_BF16;
        const uint32_t h[4] = {from_f<BF16>(v[0]), from_f<BF16>(v[1]), from_f<BF16>(v[2]), from_f<BF16>(v[3])};
        *(uint2v*)((uint16_t*)p.s + at) = uint2v{h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
        float z = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) z = fmaf(to_f<BF16>((uint16_t)h[e]), 0.f, z);
        if (z != 0.f) *(float4v*)(p.wide + at) = v;
      }
    }
    __syncthreads();  // the buffers are filled again
  }
}

// Numbers a tile's adapters as they first occur (one wave, up to 256 rows).
__device__ __forceinline__ void lora_number(const Prepare& p, int tile) {
  const int lane = threadIdx.x;
  if (lane >= 64) return;
  const int64_t m0 = (int64_t)tile * kStTile;
  int a[4], num[4];
  uint64_t left[4], any = 0;
#pragma unroll
  for (int q = 0; q < 4; q++) {
    const int r = q * 64 + lane;
    a[q] = r < kStTile && m0 + r < p.M ? p.index[m0 + r] : -1;
    if (a[q] >= p.n) a[q] = -1;
    num[q] = -1;
    left[q] = __ballot(a[q] >= 0);
    any |= left[q];
  }
  int nd = 0;
  while (any != 0) {  // (at most one round per row)
    int cur = 0;
#pragma unroll
    for (int q = 3; q >= 0; q--)
      if (left[q] != 0) cur = __builtin_amdgcn_readlane(a[q], __builtin_ctzll(left[q]));
    any = 0;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      if (a[q] == cur) num[q] = nd;
      left[q] &= ~__ballot(a[q] == cur);
      any |= left[q];
    }
    if (lane == 0) p.num.list[m0 + nd] = cur;
    nd++;
  }
#pragma unroll
  for (int q = 0; q < 4; q++)
    if (q * 64 + lane < kStTile) p.num.number[m0 + q * 64 + lane] = (int16_t)num[q];
  if (lane == 0) p.num.count[tile] = nd;
}

// 8 codes at a time, four of them requested together.
template <int QB, bool AFF, bool BF16>
__device__ __forceinline__ void lora_dequantize(const Codes& c, int block) {
  const int threads = blockDim.x, cpr = c.K >> 3, n = c.N * cpr, step = c.blocks * threads;
  for (int i0 = block * threads + (int)threadIdx.x; i0 < n; i0 += 4 * step) {
    uint32_t w0[4], w1[4], sb[4], zb[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int i = min(i0 + u * step, n - 1), r = i / cpr, k = 8 * (i - r * cpr);
      if constexpr (QB == 8) {
        const uint2v w = *(const uint2v*)(c.q.q + (int64_t)i * 8);
        w0[u] = w.x;
        w1[u] = w.y;
      } else {
        w0[u] = *(const uint32_t*)(c.q.q + (int64_t)i * 4);
        w1[u] = 0;
      }
      const int64_t gi = (int64_t)r * c.q.G + k / c.q.group;
      sb[u] = ((const uint16_t*)c.q.scales)[gi];
      zb[u] = AFF ? ((const uint16_t*)c.q.zeros)[gi] : 0u;
    }
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (i0 + u * step < n)
        *(uint4v*)(c.copy + (int64_t)(i0 + u * step) * 8) = dequant8<QB, AFF, false, BF16>(w0[u], w1[u], sb[u], zb[u], 0.f, 0.f);
  }
}

template <int DT, int MT, int NT>
__global__ __launch_bounds__(256) void lora_prepare(Prepare p) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  int b = blockIdx.x;
  const int inner = p.gx * p.gy * p.gz;
  if constexpr (DT != HB_F32) {
    if (b < p.num.tiles) return lora_number(p, b);
    b -= p.num.tiles;
  }
  if (b < inner) {
    const int bx = b % p.gx, q = b / p.gx;
    return lora_inner<DT, MT, NT>(p, bx, q % p.gy, q / p.gy, lds);
  }
  if constexpr (DT != HB_F32) {
    constexpr bool BF16 = DT == HB_BF16;
    const Codes& c = p.codes;
    b -= inner;
    if (c.bits == 8 && c.mode == 0) lora_dequantize<8, false, BF16>(c, b);
    else if (c.bits == 8) lora_dequantize<8, true, BF16>(c, b);
    else if (c.mode == 0) lora_dequantize<4, false, BF16>(c, b);
    else lora_dequantize<4, true, BF16>(c, b);
  }
}

static void launch_prepare(hipStream_t st, int cus, int dt, Prepare& p) {
  const bool large = p.M >= 8192;
  const int rows = large ? 64 : 16;
  auto turns = [&] { return std::max(2, std::min({p.n, rows, cus / (int)std::min<int64_t>((int64_t)p.gx * p.gy, cus)})); };
  p.gx = (p.M + rows - 1) / rows;
  p.gy = (p.R + 63) / 64;
  p.gz = turns();
  const bool narrow = p.R <= 16 || (!large && (int64_t)p.gx * p.gy * p.gz < cus);  // 16 ranks a block
  if (narrow) p.gy = (p.R + 15) / 16;
  const int64_t blocks = (int64_t)p.gx * p.gy * p.gz + p.num.tiles + p.codes.blocks;
  HB_REQUIRE(blocks < (1ll << 24), "hb_lora_linear: too many rows and ranks");  // (2^32 threads)
  auto go = [&](auto kernel, std::atomic<uint64_t>& attr, int mt, int nt) {
    const int lds = 4 * 2 * (mt + nt) * 2048;
    if (lds > 64 * 1024)
      once_per_device(attr, [&] {
        HB_CHECK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
      });
    kernel<<<(unsigned)blocks, 256, lds, st>>>(p);
  };
  auto type = [&](auto t) {
    constexpr int DT = decltype(t)::value;
    static std::atomic<uint64_t> attr[4];
    if (large && narrow) go(lora_prepare<DT, 4, 1>, attr[0], 4, 1);
    else if (large) go(lora_prepare<DT, 4, 4>, attr[1], 4, 4);
    else if (narrow) go(lora_prepare<DT, 1, 1>, attr[2], 1, 1);
    else go(lora_prepare<DT, 1, 4>, attr[3], 1, 4);
  };
  if (dt == HB_F32) type(std::integral_constant<int, HB_F32>{});
  else if (dt == HB_F16) type(std::integral_constant<int, HB_F16>{});
  else type(std::integral_constant<int, HB_BF16>{});
}

// The projection with adapters for few rows: tiles of up to 32 x 32, whose NW waves share out
// K, then the adapters' axis (LoraExt), by chunks of 64, each through two buffers of its
// own with no barrier, and meet in LDS.  Bound by the chain of loads (the tile's
// adapters, operands, s and B), of which a wave has two chunks' on their way.  K's sum
// has another order than the other kernels' (a wave per tile in theirs: 12.5 us at the
// first of these sizes).  Taken up to 2 tiles a CU (f16; here and on gemm_ring's tiles,
// with lora_prepare: 48 x 2304 x 768, 24 adapters of rank 16, 8.6 and 14.5 us; 256 x 1024
// x 2624, 256 tiles, 11.5 and 19; 512 x 768 x 1152, 384 tiles, 11.7 and 13.7; 256 x 2304
// x 768, 576 tiles, 13.8 and 13.3; 128 x 5248 x 1024, 656 tiles, 16.0 and 14.9).  The
// tiles are of 16 columns while they leave CUs idle, so that a CU reads less (48 x 1024
// x 2624, 24 adapters of rank 64: 22.5 -> 19.2 us before its loads were of whole lines,
// 13.3 with them), and of 16 rows where there are no more.  Tiles of 64 x 64 take over while
// they go round the CUs once (400 x 2304 x 768, 252 tiles: 12.9 us, gemm_ring's 14.2; 1200 x
// 1024 x 1024, 304 tiles: 20.3 and 15.6).
template <int DT, int TM, int TN, int NW>
__global__ __launch_bounds__(NW * 64) void lora_few(const char* __restrict__ X, int64_t ldx, const char* __restrict__ W,
                                                    const char* __restrict__ bias, char* __restrict__ Y, int64_t ldy,
                                                    int M, int N, int K, int tiles_m, LoraExt ext) {
  constexpr int ES = DT == HB_F32 ? 4 : 2, KC = 128 / ES, V = 16 / ES;  // bytes, k of a chunk, ranks of 16 bytes
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  auto red = (float(*)[TM * 16][TN * 16 + 4])lds;  // [NW], padded against bank conflicts
  __shared__ int adapter[TM * 16];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile = xcd_tile(blockIdx.x, gridDim.x), tn = tile / tiles_m;
  const int m0 = (tile - tn * tiles_m) * TM * 16, n0 = tn * TN * 16, R = ext.R;
  int a = lane < TM * 16 && m0 + lane < M ? ext.index[m0 + lane] : -1;
  constexpr int BUF = (TM + TN) * 2048, L = 2 * (TM + TN);
  uint32_t xo[2 * TM], wo[2 * TN];
#pragma unroll
  for (int i = 0; i < 2 * TM; i++) xo[i] = piece_offset(i, lane, M - 1 - m0, (uint32_t)ldx * ES);
#pragma unroll
  for (int i = 0; i < 2 * TN; i++) wo[i] = piece_offset(i, lane, N - 1 - n0, (uint32_t)K * ES);
  const uint4v xs = lora_records(X + (int64_t)m0 * ldx * ES), ws = lora_records(W + (int64_t)n0 * K * ES);
  const char* buffers = lds + wave * 2 * BUF;
  const uint32_t at0 = (uint32_t)__builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)buffers);
  float4v acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = float4v{0.f, 0.f, 0.f, 0.f};
  auto request = [&](int c) __attribute__((always_inline)) {  // chunk wave + NW c of K
    const uint32_t to = at0 + (uint32_t)((c & 1) * BUF), k = (uint32_t)(wave + NW * c) * 128u;
#pragma unroll
    for (int i = 0; i < 2 * TM; i++) buffer_lds16(xs, xo[i], k, to + 1024u * i);
#pragma unroll
    for (int j = 0; j < 2 * TN; j++) buffer_lds16(ws, wo[j], k, to + 1024u * (2 * TM + j));
  };
  auto multiply = [&](int c) __attribute__((always_inline)) {
    const char* rows = buffers + (c & 1) * BUF;
#pragma unroll
    for (int s = 0; s < 2; s++) {
      uint4v xf[TM], wf[TN];
#pragma unroll
      for (int i = 0; i < TM; i++) xf[i] = row_chunk(rows, 16 * i + l16, 4 * s + g);
#pragma unroll
      for (int j = 0; j < TN; j++) wf[j] = row_chunk(rows + TM * 2048, 16 * j + l16, 4 * s + g);
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = mfma16<DT>(wf[j], xf[i], acc[i][j]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the buffer is requested again)
  };
  const int kc = (K / KC - wave + NW - 1) / NW;  // this wave's chunks of K, from 0 on
  if (kc > 0) request(0);
  if (kc > 1) request(1);
  // the tile's adapters by number, as they first occur: lane o has number o's
  if (a >= ext.n) a = -1;
  int num = -1, mine = 0, nd = 0;
  for (uint64_t left = __ballot(a >= 0); left != 0; nd++) {  // (at most one round per row)
    const int cur = __builtin_amdgcn_readlane(a, __builtin_ctzll(left));
    const uint64_t same = __ballot(a == cur);
    left &= ~same;
    num = a == cur ? nd : num;
    mine = lane == nd ? cur : mine;
  }
  if (tid < TM * 16) adapter[tid] = mine;
  const int rv = R / V, chunks = (nd * rv + 7) >> 3;   // 16 bytes of ranks of an adapter; chunks of 8 such
  const int ec = (chunks - wave + NW - 1) / NW;              // this wave's of those, numbered from kc on
  const float inv = (float)V / (float)R;
  const uint4v ss = lora_records(ext.s), bs = lora_records(ext.b);
  int xnum[2 * TM];  // of the rows of the lane's pieces
#pragma unroll
  for (int i = 0; i < 2 * TM; i++) xnum[i] = __shfl(num, 8 * i + (lane >> 3));
  auto request_ranks = [&](int c) __attribute__((always_inline)) {
    const uint32_t to = at0 + (uint32_t)((c & 1) * BUF);
    auto piece = [&](int i, auto rows) __attribute__((always_inline)) {  // of i's rows
      const int r = i * 8 + (lane >> 3), ch = (wave + NW * (c - kc)) * 8 + ((lane & 7) ^ row_f(r));
      const int o = (int)(((float)ch + 0.5f) * inv);
      rows(r, o, (uint32_t)(ch - o * rv) * V);
    };
    // past the records: zeros
#pragma unroll
    for (int i = 0; i < 2 * TM; i++)
      piece(i, [&](int r, int o, uint32_t rank) {
        buffer_lds16(ss, o == xnum[i] ? ((uint32_t)min(m0 + r, M - 1) * (uint32_t)R + rank) * ES : 0xfffffff0u, to + 1024u * i);
      });
#pragma unroll
    for (int j = 0; j < 2 * TN; j++)
      piece(j, [&](int r, int o, uint32_t rank) {
        const uint32_t who = (uint32_t)__shfl(mine, o & 63), n = (uint32_t)min(n0 + r, N - 1);
        buffer_lds16(bs, o < nd ? ((who * (uint32_t)N + n) * (uint32_t)R + rank) * ES : 0xfffffff0u,
                     to + 1024u * (2 * TM + j));
      });
  };
  const int all = max(kc, 0) + max(ec, 0);
  auto ask = [&](int c) __attribute__((always_inline)) {
    if (c < kc) request(c);
    else request_ranks(c);
  };
  if (max(kc, 0) < 1 && all > 0) ask(0);
  if (max(kc, 0) < 2 && all > 1) ask(1);
  for (int c = 0; c < all; c++) {
    if (c + 1 < all) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    multiply(c);
    if (c + 2 < all) ask(c + 2);
  }
  __syncthreads();  // everybody is done with the buffers
  // lane: row 16 i + l16, columns 16 j + 4 g ..
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) *(float4v*)&red[wave][16 * i + l16][16 * j + 4 * g] = acc[i][j];
  __syncthreads();
  constexpr int CW = TN * 8;  // threads of a row
  static_assert(NW * 64 % CW == 0, "a thread has the same two columns in every row");
  int dirty[2] = {kUnknown, kUnknown};
  for (int at = tid; at < TM * 16 * CW; at += NW * 64) {
    const int row = at / CW, col = at % CW * 2, m = m0 + row, n = n0 + col;
    if (m >= M || n >= N) continue;
    float v[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; w++)
#pragma unroll
      for (int q = 0; q < 2; q++) v[q] += red[w][row][col + q];
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const int nq = min(n + q, N - 1);
      // the zeros of other rows do not keep a non-finite B out of a row's sums (0 * inf), and
      // an inner product may be past the type's range
      bool alone = false;
      if (v[q] * 0.f != 0.f) {
        alone = lora_past<DT>(ext, m);
        if (!alone && dirty[q] == kUnknown) dirty[q] = lora_dirty<DT>(ext, adapter, nd, N, nq);
        alone = alone || lora_mixed(ext, dirty[q], m);
      }
      v[q] += bias != nullptr ? load_f(bias, nq, DT) : 0.f;
      if (alone) v[q] = lora_output<DT>(X, ldx, W, bias, N, K, ext, m, nq);
    }
    char* y = Y + ((int64_t)m * ldy + n) * ES;
    if constexpr (DT == HB_F32) {
      if (n + 1 < N) *(float2*)y = float2{v[0], v[1]};
      else *(float*)y = v[0];
    } else {
      const uint32_t lo = from_f<DT == HB_BF16>(v[0]), hi = from_f<DT == HB_BF16>(v[1]);
      if (n + 1 < N) *(uint32_t*)y = lo | (hi << 16);
      else *(uint16_t*)y = (uint16_t)lo;
    }
  }
}

// Its tiles, if it takes the call; false: it does not.
template <int DT>
static bool lora_few_tiles(hipStream_t st, int cus, const void* x, int64_t ldx, const void* w, const void* bias, void* y,
                           int64_t ldy, int M, int N, int K, const LoraExt& ext, bool launch) {
  auto run = [&](auto kernel, std::atomic<uint64_t>& attr, int bm, int bn, int nw) {
    if (!launch) return true;
    const int tm = (M + bm - 1) / bm, lds = nw * 2 * (bm + bn) * 128;
    if (lds >= 64 * 1024)  // (with its static LDS past the 64 KB that a launch has without the attribute)
      once_per_device(attr, [&] {
        HB_CHECK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
      });
    kernel<<<(unsigned)((int64_t)tm * ((N + bn - 1) / bn)), nw * 64, lds, st>>>(
        (const char*)x, ldx, (const char*)w, (const char*)bias, (char*)y, ldy, M, N, K, tm, ext);
    return true;
  };
  static std::atomic<uint64_t> attr[5];
  auto tiles = [&](int t) { return (int64_t)((M + t - 1) / t) * ((N + t - 1) / t); };
  const bool half = 2 * tiles(32) <= cus;
  if (tiles(32) <= 2 * cus) {
    if (M <= 16) return half ? run(lora_few<DT, 1, 1, 8>, attr[0], 16, 16, 8) : run(lora_few<DT, 1, 2, 8>, attr[1], 16, 32, 8);
    return half ? run(lora_few<DT, 2, 1, 8>, attr[2], 32, 16, 8) : run(lora_few<DT, 2, 2, 8>, attr[3], 32, 32, 8);
  }
  return tiles(64) <= cus && run(lora_few<DT, 4, 4, 4>, attr[4], 64, 64, 4);
}

// The projection with adapters for large M: 256 x 256 tiles (or 192 wide, 8 waves of 64
// x 96), 8 waves of 128 x 64 (6
// fragment reads per 8 products; 16 waves of 64 x 64 read 8, 16k x 5248 x 1024 rank 64
// 257 -> 273 us; 4 of 128 x 128 do not fit the registers, 305), a ring of four 32-wide
// stages as gemm_ring's, and one block per CU that streams its tiles without a pause:
// the ring is filled with the next tile's first stages during a tile's last ones, and
// the outputs go from registers to memory (the lane halves exchange 4 columns, so that
// a lane stores 8 of a row) while those loads are on their way.  On gemm_ring's blocks
// of one tile each the same tiles took 269 us, its tiles of 128 x 256 338.
// What bounds it (242 us with lora_prepare, then 24): without the loads into LDS 197, without
// the fragment reads too 187: the products alone, at the clock that the card holds under
// them, and behind them the 32 KB per stage from the L2.
// Of its numbering only whole-wave scalars are read, by scalar loads (kept in their
// address space), which the waits for the ring do not count.
using ScalarInts = const __attribute__((address_space(4))) int32_t*;
__device__ __forceinline__ ScalarInts scalar_ints(const void* p) {
  const uint64_t a = (uint64_t)p;
  return (ScalarInts)(((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) << 32) |
                      (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a));
}

__device__ __forceinline__ int stream_f(int r) { return (r >> 2) & 3; }  // swizzle of a row's 4 chunks

template <bool BF16, int BN>
__global__ __launch_bounds__(kStWaves * 64) void lora_stream(const uint16_t* __restrict__ X, int64_t ldx,
                                                             const uint16_t* __restrict__ W,
                                                             const uint16_t* __restrict__ bias, uint16_t* __restrict__ Y,
                                                             int64_t ldy, int M, int N, int K, int tiles_m, int tiles_n,
                                                             LoraExt ext, Numbers num) {
  constexpr int NST = kStStages, NW = kStWaves, WM = BN == 256 ? 2 : 4, WN = NW / WM, TM = kStTile / WM / 32, TN = BN / WN / 32;
  static_assert(TN * WN * 32 == BN && BN <= kStTile, "whole blocks of 32");
  constexpr int PW = 2 * kStTile / 16 / NW;  // 1 KB pieces (16 rows) of a stage per wave
  constexpr int ST = TM * TN * 2;            // stores of a tile per lane
  extern __shared__ __attribute__((aligned(16))) uint16_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, lg = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const bool xwave = wave < NW / 2;  // requests pieces of X, else of W
  const int KT0 = K / kStBK;
  const float inv8 = 8.f / (float)ext.R;

  // An XCD has one contiguous run of tiles, its blocks take them in turn; tiles are
  // numbered down 4 row tiles, then along N, so that the XCD's 32 share 4 x 8 operands
  // in its L2.
  const int ntiles = tiles_m * tiles_n, xcd = blockIdx.x & 7, nb = (int)((gridDim.x - xcd + 7) >> 3);
  const int run0 = (int)((int64_t)ntiles * xcd >> 3), run1 = (int)((int64_t)ntiles * (xcd + 1) >> 3);
  auto place = [&](int t, int* tm, int* tn) {
    constexpr int G = 4;
    const int grp = t / (G * tiles_n), rem = t - grp * G * tiles_n, gm = min(G, tiles_m - grp * G);
    *tn = rem / gm;
    *tm = grp * G + rem - *tn * gm;
  };

  // ---- requests: the tile they are at, its stage, and this wave's pieces of it
  int rt = run0 + (int)(blockIdx.x >> 3), rk = 0, rKT = 0, rn0 = 0;
  uint4v rsrc{};
  uint32_t off[PW];
  int xnum[PW];
  const int slot4 = (lane & 3), prow = lane >> 2;  // slot and row within a piece
  auto enter = [&]() __attribute__((always_inline)) {
    int tm, tn;
    place(rt, &tm, &tn);
    const int nd = scalar_ints(num.count)[tm];
    rKT = KT0 + (nd * ext.R + kStBK - 1) / kStBK;
    rk = 0;
    rn0 = tn * BN;
    const uint64_t base = xwave ? (uint64_t)(X + (int64_t)tm * kStTile * ldx) : (uint64_t)(W + (int64_t)rn0 * K);
    rsrc = uint4v{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base),
                  (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32) & 0xffffu), 0x80000000u, 0x00020000u};
#pragma unroll
    for (int i = 0; i < PW; i++) {
      const int r = (wave % (NW / 2) * PW + i) * 16 + prow;  // of X or of W
      const uint32_t c = (slot4 ^ stream_f(r)) * 16;
      // (rows past the operand are clamped: their outputs are never stored)
      off[i] = xwave ? (uint32_t)min(r, M - 1 - tm * kStTile) * (uint32_t)ldx * 2u + c
                     : r < BN ? (uint32_t)min(r, N - 1 - rn0) * (uint32_t)K * 2u + c : 0xfffffff0u;
      xnum[i] = nd;
      if (xwave) {  // the piece's 16 rows' numbers, two to a word: scalar loads, which no wait for the ring counts
        const ScalarInts nums = scalar_ints(num.number + (int64_t)tm * kStTile + (wave % (NW / 2) * PW + i) * 16);
        int v = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          int w = nums[e];
          asm("" : "+s"(w));  // (or the compiler loads a chosen address per lane)
          v = (lane >> 3) == e ? w : v;
        }
        xnum[i] = (int)(int16_t)(v >> (16 * ((lane >> 2) & 1)));
      }
    }
  };
  const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint16_t*)smem);
  // the next stage into ring slot `slot`; the last one of a tile moves on to the next
  auto request = [&](int slot) __attribute__((always_inline)) {
    const uint32_t to = lds0 + (uint32_t)(slot * kStStage * 2 + wave * PW * 1024);
    if (rk < KT0) {
#pragma unroll
      for (int i = 0; i < PW; i++) buffer_lds16(rsrc, off[i], (uint32_t)rk * 64u, to + 1024u * i);
    } else {
      // 4 chunks of 8 ranks of the adapters' axis (LoraExt)
      const int ch0 = (rk - KT0) * 4, r8 = ext.R >> 3;
      const uint64_t base = xwave ? (uint64_t)ext.s : (uint64_t)ext.b;
      const uint4v rs = {(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base),
                         (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32) & 0xffffu), 0x80000000u,
                         0x00020000u};
      int tm, tn;
      place(rt, &tm, &tn);
      const ScalarInts list = scalar_ints(num.list + (int64_t)tm * kStTile);
      int who[4];  // the chunks' adapters
      if (!xwave) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          who[j] = list[min(__builtin_amdgcn_readfirstlane((int)(((float)(ch0 + j) + 0.5f) * inv8)), kStTile - 1)];
      }
#pragma unroll
      for (int i = 0; i < PW; i++) {
        const int r = (wave % (NW / 2) * PW + i) * 16 + prow, j = slot4 ^ stream_f(r);
        const int o = (int)(((float)(ch0 + j) + 0.5f) * inv8), c = ch0 + j - o * r8;
        uint32_t at = 0xfffffff0u;  // past the records: zeros
        if (xwave) {
          if (o == xnum[i]) at = ((uint32_t)(tm * kStTile + r) * (uint32_t)ext.R + (uint32_t)c * 8u) * 2u;
        } else if (o < xnum[i] && r < BN) {
          const int a = j == 0 ? who[0] : j == 1 ? who[1] : j == 2 ? who[2] : who[3];
          const int n = min(rn0 + r, N - 1);
          at = (((uint32_t)a * (uint32_t)N + (uint32_t)n) * (uint32_t)ext.R + (uint32_t)c * 8u) * 2u;
        }
        buffer_lds16(rs, at, to + 1024u * i);
      }
    }
    if (++rk == rKT) {
      rt += nb;
      if (rt < run1) enter();
    }
  };

  // ---- products
  float16v acc[TM][TN];
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
  };
  int fo[2];
#pragma unroll
  for (int s = 0; s < 2; s++) fo[s] = l32 * kStBK + (((2 * s + lg) ^ stream_f(l32)) << 3);
  uint4v xf[2][TM], wf[2][TN];
  auto read = [&](int slot, int s, int d) __attribute__((always_inline)) {
    const uint16_t* b = smem + slot * kStStage;
#pragma unroll
    for (int i = 0; i < TM; i++) xf[d][i] = *(const uint4v*)(b + fo[s] + (wm * TM + i) * 32 * kStBK);
#pragma unroll
    for (int j = 0; j < TN; j++) wf[d][j] = *(const uint4v*)(b + fo[s] + (kStTile + (wn * TN + j) * 32) * kStBK);
  };
  auto multiply = [&](int d) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) acc[i][j] = mfma32<BF16>(wf[d][j], xf[d][i], acc[i][j]);
  };

  if (rt >= run1) return;  // (the whole block: more blocks than tiles)
  int ct = rt;             // the tile whose products are made
  enter();
  // total stages of this block's tiles are at least 2 (K >= 64)
  int ahead = 0;  // stages requested and not yet multiplied
#pragma unroll
  for (int s = 0; s < NST - 1; s++)
    if (rt < run1) {
      request(s);
      ahead++;
    }
  ring_wait_stages<PW, NST - 2>(ahead - 1);
  read(0, 0, 0);
  clear();
  int slot = 0;
  bool stored = false;  // the stores lie between the requests of this tile's stages 2 and 3
  while (true) {
    int tm, tn;
    place(ct, &tm, &tn);
    const int KT = KT0 + (scalar_ints(num.count)[tm] * ext.R + kStBK - 1) / kStBK;
    for (int kt = 0; kt < KT; kt++) {
      // the stage after this one has landed (if there is one) and everybody is done
      // with the one before, whose slot takes the third from here
      if (ahead >= NST - 1) {
        if (stored && kt < NST - 2) ring_wait_barrier<(NST - 3) * PW + ST>();
        else ring_wait_barrier<(NST - 3) * PW>();
      } else {
        ring_wait_barrier<0>();
      }
      read(slot, 1, 1);
      multiply(0);
      if (rt < run1) request(slot == 0 ? NST - 1 : slot - 1);
      else ahead--;
      slot = slot == NST - 1 ? 0 : slot + 1;
      if (ahead > 0) read(slot, 0, 0);
      multiply(1);
    }
    // ---- write-out: lane l32 holds row l32 of a 32 x 32 block, columns 8 g + 4 lg ..
    const int m0 = tm * kStTile + wm * TM * 32, n0 = tn * BN + wn * TN * 32;
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) z = fmaf(acc[i][j][r], 0.f, z);
    const bool odd = __any(z != 0.f);  // (a non-finite output: below)
    float bv[TN][4][4];
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        uint2v b = {0u, 0u};
        if (bias != nullptr) b = *(const uint2v*)(bias + min(n0 + 32 * j + 8 * g + 4 * lg, N - 4));
#pragma unroll
        for (int e = 0; e < 4; e++) bv[j][g][e] = to_f<BF16>((uint16_t)(b[e >> 1] >> (16 * (e & 1))));
      }
    const auto ys = __builtin_amdgcn_make_buffer_rsrc((void*)(Y + (int64_t)(tm * kStTile) * ldy + tn * BN), 0,
                                                      0x80000000u, 0x00020000u);
#pragma unroll
    for (int i = 0; i < TM; i++) {
      const int m = m0 + 32 * i + l32;
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t lo[2], hi[2];
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const int x = 8 * h + 4 * g;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = acc[i][j][x + e] + bv[j][2 * h + g][e];
            lo[g] = (uint32_t)from_f<BF16>(v[0]) | ((uint32_t)from_f<BF16>(v[1]) << 16);
            hi[g] = (uint32_t)from_f<BF16>(v[2]) | ((uint32_t)from_f<BF16>(v[3]) << 16);
          }
          // lane half lg now takes all 8 columns of group 2 h + lg
          const auto a = __builtin_amdgcn_permlane32_swap(lo[0], lo[1], false, false);
          const auto c = __builtin_amdgcn_permlane32_swap(hi[0], hi[1], false, false);
          const uint4v o = {(uint32_t)a[0], (uint32_t)c[0], (uint32_t)a[1], (uint32_t)c[1]};
          const int n = n0 + 32 * j + 16 * h + 8 * lg;
          // as many stores whatever the edges: those past them fall outside the records
          const uint32_t at = m < M && n < N
                                  ? (uint32_t)(m - tm * kStTile) * (uint32_t)ldy * 2u + (uint32_t)(n - tn * BN) * 2u
                                  : 0xfffffff0u;
          __builtin_amdgcn_raw_buffer_store_b128(o, ys, at, 0, 0);
        }
    }
    stored = !odd;
    if (__builtin_expect(odd, 0)) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      // the zeros of other rows do not keep a non-finite B out of a row's sums (0 *
      // inf), and an inner product may be past the type's range: an output that has come
      // out non-finite is computed again with its own row's adapter alone
      const int* list = num.list + (int64_t)tm * kStTile;
      const int nd = num.count[tm];
#pragma unroll 1
      for (int n = n0 + lane; n < min(n0 + TN * 32, N); n += 64) {
        int dirty = kUnknown;
#pragma unroll 1
        for (int m = m0; m < min(m0 + TM * 32, M); m++) {
          const float v = to_f<BF16>(__builtin_nontemporal_load(Y + (int64_t)m * ldy + n));
          constexpr int DT = BF16 ? HB_BF16 : HB_F16;
          if (v * 0.f == 0.f) continue;
          if (!lora_past<DT>(ext, m)) {
            if (dirty == kUnknown) dirty = lora_dirty<DT>(ext, list, nd, N, n);
            if (!lora_mixed(ext, dirty, m)) continue;
          }
          Y[(int64_t)m * ldy + n] = from_f<BF16>(lora_output<DT>(X, ldx, W, bias, N, K, ext, m, n));
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    ct += nb;
    if (ct >= run1) return;
    clear();
  }
}

// lora_stream's width of tile: 192 columns where the rounds that the CUs take with them are shorter
// by a fifth, which their operands, 17% more a product, leave a gain of (f16: 4096 x 5248
// x 1024, two rounds of either, 75 -> 69 us; 8192 x 2304 x 768 61 -> 56; 16.2k x 5248 x
// 1024, 7 rounds of 192 against 6 of 256, 262 and 274).
static int lora_stream_width(int cus, int M, int N) {
  auto cost = [&](int bn) {
    const int64_t tiles = (int64_t)((M + kStTile - 1) / kStTile) * ((N + bn - 1) / bn);
    return (tiles + cus - 1) / cus * bn;
  };
  return 5 * cost(192) <= 4 * cost(256) ? 192 : 256;
}
// The GEMM's tile, by the rules of the plain projection (ring_tile); on the streaming
// kernel, which stores 16 bytes at a time, once its tiles occupy half of the CUs
// (f16, 4 adapters in runs of 512 rows, streaming and by ring_tile: 4096 x 2304 x 768, 144
// tiles, 36 and 45 us; 3000 x 5248 x 1024 47 and 102; 16384 x 768 x 1152 51 and 81; 16k x
// 5248 x 1024 262 and 502).
// Its tiles of 256 rows suit rows that come in runs of one request: a tile of all
// different adapters multiplies 256 R ranks, gemm_ring's tile of 64 rows 64 R.
static bool lora_streams(int cus, int64_t M, int64_t N, const uint16_t* bias, const uint16_t* y, int64_t ldy) {
  if (M <= kStTile || N % 8 != 0 || ldy % 8 != 0 || (uintptr_t)y % 16 != 0 || (uintptr_t)bias % 8 != 0) return false;
  return 2 * ((M + kStTile - 1) / kStTile) * ((N + kStTile - 1) / kStTile) >= cus;
}
template <bool BF16>
static void lora_gemm(hipStream_t st, int cus, const uint16_t* x, int64_t ldx, const uint16_t* w, const uint16_t* bias,
                      uint16_t* y, int64_t ldy, int M, int N, int K, const LoraExt& ext, const Numbers& num) {
  if (num.tiles > 0) {
    static std::atomic<uint64_t> attr[2];
    auto run = [&](auto kernel, std::atomic<uint64_t>& at, int bn) {
      once_per_device(at, [&] {
        HB_CHECK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kStLds));
      });
      const int tm = (M + kStTile - 1) / kStTile, tn = (N + bn - 1) / bn;
      kernel<<<(unsigned)cus, kStWaves * 64, kStLds, st>>>(x, ldx, w, bias, y, ldy, M, N, K, tm, tn, ext, num);
    };
    if (lora_stream_width(cus, M, N) == 256) run(lora_stream<BF16, 256>, attr[0], 256);
    else run(lora_stream<BF16, 192>, attr[1], 192);
    return;
  }
  if (lora_few_tiles<BF16 ? HB_BF16 : HB_F16>(st, cus, x, ldx, w, bias, y, ldy, M, N, K, ext, true)) return;
  auto go = [&](auto launch) { launch(st, 0u, x, ldx, w, bias, (const uint16_t*)nullptr, (int64_t)0, y, ldy, M, N, K, ext); };
  LinearKernel tile = LinearKernel::kRing64x64x3;
  ring_tile(cus, M, N, K, false, true, false, &tile);
  switch (tile) {
    case LinearKernel::kRing32x64: return go(launch_ring_t<32, 64, 1, 2, 6, BF16, false, LoraExt>);
    case LinearKernel::kRing64x64: return go(launch_ring_t<64, 64, 2, 2, 4, BF16, false, LoraExt>);
    case LinearKernel::kRing64x64k: return go(launch_ring_t<64, 64, 2, 2, 5, BF16, false, LoraExt>);
    case LinearKernel::kRing128x64: return go(launch_ring_t<128, 64, 4, 2, 4, BF16, false, LoraExt>);
    case LinearKernel::kRing128x256: return go(launch_ring_t<128, 256, 4, 4, 3, BF16, false, LoraExt>);
    default: return go(launch_ring_t<64, 64, 2, 2, 3, BF16, false, LoraExt>);
  }
}

// ------------------------------------------------------------------ f32

// y += s . B^T of f32 rows on v_mfma_f32_16x16x4, onto the projection: 4 waves of 32
// rows and 64 columns, the rows' distinct adapters one after another (of few tiles shared
// out over blocks), each row's columns read and written in its own adapter's turn.  Bound by that, 8 bytes an output.
__global__ __launch_bounds__(256) void lora_expand_f32(const float* __restrict__ S, const float* __restrict__ Bk,
                                                       const int32_t* __restrict__ index, int n, int M, int N, int R,
                                                       float* __restrict__ Y, int64_t ldy) {
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = blockIdx.y * 32, n0 = (blockIdx.x * 4 + wave) * 64;
  int a = lane < 32 && m0 + lane < M ? index[m0 + lane] : -1;
  if (a >= n) a = -1;
  if (n0 >= N) return;
  const float* sr[2];
  int own[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    sr[i] = S + (int64_t)min(m0 + 16 * i + l16, M - 1) * R + 4 * g;
    own[i] = __shfl(a, 16 * i + l16);
  }
  int turn = 0;
  for (uint64_t left = __ballot(a >= 0); left != 0; turn++) {
    const int cur = __builtin_amdgcn_readlane(a, __builtin_ctzll(left));
    left &= ~__ballot(a == cur);
    if (turn % (int)gridDim.z != (int)blockIdx.z) continue;  // (a row is in one turn)
    const float* br[4];
#pragma unroll
    for (int t = 0; t < 4; t++) br[t] = Bk + ((int64_t)cur * N + min(n0 + 16 * t + l16, N - 1)) * R + 4 * g;
    float4v acc[2][4];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int t = 0; t < 4; t++) acc[i][t] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int r = 0; r < R; r += 16) {
      const bool in = r + 4 * g < R;
      float4v x[2], b[4];
#pragma unroll
      for (int i = 0; i < 2; i++) x[i] = in ? *(const float4v*)(sr[i] + r) : float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 4; t++) b[t] = in ? *(const float4v*)(br[t] + r) : float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int t = 0; t < 4; t++) acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[t][e], x[i][e], acc[i][t], 0, 0, 0);
    }
    // lane: row 16 i + l16, columns 16 t + 4 g ..
#pragma unroll
    for (int i = 0; i < 2; i++) {
      if (own[i] != cur) continue;  // (cur >= 0: no row behind M)
      float* y = Y + (int64_t)(m0 + 16 * i + l16) * ldy + n0 + 4 * g;
#pragma unroll
      for (int t = 0; t < 4; t++)
        if (n0 + 16 * t + 4 * g < N) *(float4v*)(y + 16 * t) += acc[i][t];  // (N % 4 == 0)
    }
  }
}

// ------------------------------------------------------------------ any type

// One wave per row and rank.
__global__ __launch_bounds__(256) void lora_shrink_any(int dt, const void* __restrict__ X, int64_t ldx,
                                                       const void* __restrict__ A, const float* __restrict__ scales,
                                                       const int32_t* __restrict__ index, int n, int64_t M, int R,
                                                       int K, float* __restrict__ S) {
  const int lane = threadIdx.x & 63;
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < M * R; i += (int64_t)gridDim.x * 4) {
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

static void check_lora(const char* op, int dt, uintptr_t x, uintptr_t w, uintptr_t y, int64_t M, int64_t N, int64_t K,
                       const LoraArgs& l) {
  auto need = [&](bool ok, const char* what) {
    if (!ok) throw std::runtime_error(std::string(op) + ": " + what);
  };
  need(dt == HB_F32 || dt == HB_F16 || dt == HB_BF16, "dtype must be f32, f16 or bf16");
  need(M >= 0 && N >= 0 && K >= 0 && M < (1ll << 31) && N < (1ll << 30) && K < (1ll << 30), "bad sizes");
  need(l.n >= 0 && l.n < (1ll << 30) && l.R >= 0 && l.R <= 1024, "bad adapter count or rank (at most 1024)");
  need(l.n * l.R == 0 || M == 0 || N == 0 || K == 0 || (l.a && l.b && l.scales && l.index), "null adapter argument");
  need(M == 0 || N == 0 || (y && (K == 0 || (x && w))), "null argument");
}

// The MFMA path: 16-bit types, K and the operands as the ring takes them, whole
// chunks of ranks, a bank that 32-bit offsets reach.
static bool lora_takes_ring(int dt, uintptr_t x, int64_t ldx, uintptr_t w, uintptr_t y, int64_t ldy, int64_t M, int64_t N,
                            int64_t K, const LoraArgs& l) {
  return (dt == HB_F16 || dt == HB_BF16) && M > 0 && N > 0 && K > 0 && l.n > 0 && l.R > 0 && ring_ok(ldx, K) &&
         l.R % 8 == 0 && ldx % 8 == 0 && ldy % 8 == 0 && (x | w | y | l.a | l.b) % 16 == 0 &&
         l.n * l.R * N * 2 < (1ll << 31) && M * l.R * 2 < (1ll << 31) && K < (1 << 22) && ldx < (1 << 22) && ldy < (1 << 22);
}

// The projection with adapters on 16-bit weights w, or on quantized ones (`codes`);
// false: no memory for the inner products, or for the weights' copy.
static bool lora_fused(uintptr_t ctx, int dt, const uint16_t* x, int64_t ldx, const uint16_t* w, Codes codes,
                       const uint16_t* bias, uint16_t* y, int64_t ldy, int M, int N, int K, const LoraArgs& l) {
  const int cus = cu_count(ctx);
  const int tiles = lora_streams(cus, M, N, bias, y, ldy) ? (M + kStTile - 1) / kStTile : 0;
  const int64_t rows = (int64_t)tiles * kStTile, s_bytes = ((int64_t)M * l.R * 2 + 255) / 256 * 256;
  const int64_t wide_bytes = 2 * s_bytes;
  CallScratch held(ctx);
  const int64_t w_bytes = codes.bits ? (int64_t)N * K * 2 : 0;  // (K % 64 == 0)
  if (!held.take((size_t)(w_bytes + s_bytes + wide_bytes + rows * 6 + tiles * 4))) return false;
  Prepare p{(const char*)x, ldx, (const char*)l.a, (const float*)l.scales, (const int32_t*)l.index, (int)l.n, M, (int)l.R, K};
  if (codes.bits) {
    codes.blocks = (int)std::min<int64_t>(((int64_t)N * K / 8 + 1023) / 1024, (int64_t)cus * 16);
    codes.N = N;
    codes.K = K;
    w = codes.copy = (uint16_t*)held.p;
  }
  p.codes = codes;
  p.s = (char*)held.p + w_bytes;
  p.wide = (float*)((char*)p.s + s_bytes);
  p.num.list = (int32_t*)((char*)p.wide + wide_bytes);
  p.num.count = p.num.list + rows;
  p.num.number = (int16_t*)(p.num.count + tiles);
  p.num.tiles = tiles;
  hipStream_t st = stream_of(ctx);
  launch_prepare(st, cus, dt, p);
  check_launch("hb_lora_linear");
  const LoraExt ext{p.s, p.wide, (const void*)l.b, p.index, p.n, p.R};
  if (dt == HB_BF16) lora_gemm<true>(st, cus, x, ldx, w, bias, y, ldy, M, N, K, ext, p.num);
  else lora_gemm<false>(st, cus, x, ldx, w, bias, y, ldy, M, N, K, ext, p.num);
  check_launch("hb_lora_linear");
  return true;
}

// f32 rows on the matrix cores: whole 128 bytes of K, 16 bytes of ranks and of y.
static bool lora_takes_f32(int dt, uintptr_t x, int64_t ldx, uintptr_t y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                           const LoraArgs& l) {
  return dt == HB_F32 && M > 0 && N > 0 && K > 0 && l.n > 0 && l.R > 0 && K % 32 == 0 && N % 4 == 0 && l.R % 4 == 0 &&
         ldx % 4 == 0 && ldy % 4 == 0 && K < (1 << 22) && ldx < (1 << 22) && (x | y | l.a | l.b) % 16 == 0 &&
         (M + 31) / 32 < 65536;
}
static Prepare prepare_f32(uintptr_t x, int64_t ldx, int64_t M, int64_t K, const LoraArgs& l, void* s) {
  Prepare p{(const char*)x, ldx, (const char*)l.a, (const float*)l.scales, (const int32_t*)l.index, (int)l.n, (int)M,
            (int)l.R, (int)K};
  p.s = s;
  return p;
}
// The projection of f32 rows with adapters where lora_few takes it (76 x 1024 x 2624, 21
// adapters of rank 16: 21.4 us, hb_linear and lora_expand_f32 33.5; 300 x 768 x 768, rank
// 64: 13.4 and 21.5; 256 x 5248 x 1024, past it, 48); false: it does not, or there is no
// memory for the inner products.
static bool lora_few_f32(uintptr_t ctx, uintptr_t x, int64_t ldx, uintptr_t w, uintptr_t bias, uintptr_t y, int64_t ldy,
                         int64_t M, int64_t N, int64_t K, const LoraArgs& l) {
  if (w % 16 != 0 || l.n * l.R * N * 4 >= (1ll << 31) || M * l.R * 4 >= (1ll << 31)) return false;
  const int cus = cu_count(ctx);
  hipStream_t st = stream_of(ctx);
  LoraExt ext{nullptr, nullptr, (const void*)l.b, (const int32_t*)l.index, (int)l.n, (int)l.R};
  auto few = [&](bool launch) {
    return lora_few_tiles<HB_F32>(st, cus, (const void*)x, ldx, (const void*)w, (const void*)bias, (void*)y, ldy, (int)M,
                                  (int)N, (int)K, ext, launch);
  };
  CallScratch s(ctx);
  if (!few(false) || !s.take((size_t)(M * l.R * 4))) return false;
  Prepare p = prepare_f32(x, ldx, M, K, l, s.p);
  launch_prepare(st, cus, HB_F32, p);
  check_launch("hb_lora_linear");
  ext.s = s.p;
  few(true);
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
  if (lora_takes_f32(dt, x, ldx, y, ldy, M, N, K, l)) {
    Prepare p = prepare_f32(x, ldx, M, K, l, s.p);
    launch_prepare(st, cu_count(ctx), dt, p);
    const int64_t tiles = (N + 255) / 256 * ((M + 31) / 32);
    const dim3 blocks((unsigned)((N + 255) / 256), (unsigned)((M + 31) / 32),
                      (unsigned)std::max<int64_t>(1, std::min<int64_t>({l.n, 32, 2 * cu_count(ctx) / std::max<int64_t>(tiles, 1)})));
    lora_expand_f32<<<blocks, 256, 0, st>>>((const float*)s.p, (const float*)l.b, (const int32_t*)l.index, (int)l.n, (int)M,
                                            (int)N, (int)l.R, (float*)y, ldy);
    return check_launch(op);
  }
  lora_shrink_any<<<capped_grid((M * l.R + 3) / 4, 256), 256, 0, st>>>(dt, (const void*)x, ldx, (const void*)l.a,
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
  check_lora("hb_lora_linear", dt, x, w, y, M, N, K, l);
  HB_REQUIRE(ldx >= K && ldy >= N, "hb_lora_linear: leading dimension smaller than the row");
  if (lora_takes_ring(dt, x, ldx, w, y, ldy, M, N, K, l) &&
      lora_fused(ctx, dt, (const uint16_t*)x, ldx, (const uint16_t*)w, Codes{}, (const uint16_t*)bias, (uint16_t*)y, ldy,
                 (int)M, (int)N, (int)K, l))
    return 0;
  if (lora_takes_f32(dt, x, ldx, y, ldy, M, N, K, l) && lora_few_f32(ctx, x, ldx, w, bias, y, ldy, M, N, K, l)) return 0;
  if (hb_linear(ctx, dt, x, ldx, w, bias, 0, 0, y, ldy, M, N, K, bias ? HB_EPI_BIAS : 0)) return -1;
  add_adapters(ctx, "hb_lora_linear", dt, x, ldx, y, ldy, M, N, K, l);
  HB_API_END
}

int hb_lora_qlinear(uintptr_t ctx, int dt, uintptr_t x, int64_t ldx, uintptr_t qw, uintptr_t qscales, uintptr_t zeros,
                    uintptr_t bias, uintptr_t y, int64_t ldy, int64_t M, int64_t N, int64_t K, int bits, int group,
                    int mode, uintptr_t a, uintptr_t b, uintptr_t scales, int64_t n, int64_t R, uintptr_t index) {
  HB_API_BEGIN
  const LoraArgs l{a, b, scales, index, n, R};
  check_lora("hb_lora_qlinear", dt, x, qw, y, M, N, K, l);
  HB_REQUIRE(ldx >= K && ldy >= N, "hb_lora_qlinear: leading dimension smaller than the row");
  HB_REQUIRE((bits == 8 || bits == 4) && (mode == 0 || mode == 1) && group > 0, "hb_lora_qlinear: bad bits, mode or group");
  HB_REQUIRE(qw && qscales && (mode == 0 || zeros), "hb_lora_qlinear: missing weight tensors");
  if (lora_takes_ring(dt, x, ldx, 0, y, ldy, M, N, K, l) && group % 8 == 0 && N * K < (1ll << 33) && qw % 8 == 0 && qscales % 2 == 0 &&
      zeros % 2 == 0) {
    Codes codes{};
    codes.q = QW{(const uint8_t*)qw, (const void*)qscales, (const void*)zeros, (int)((K + group - 1) / group), group};
    codes.bits = bits;
    codes.mode = mode;
    if (lora_fused(ctx, dt, (const uint16_t*)x, ldx, nullptr, codes, (const uint16_t*)bias, (uint16_t*)y, ldy, (int)M,
                   (int)N, (int)K, l))
      return 0;
  }
  if (hb_qlinear(ctx, dt, x, ldx, qw, qscales, zeros, bias, 0, 0, y, ldy, M, N, K, bits, group, mode,
                 bias ? HB_EPI_BIAS : 0))
    return -1;
  add_adapters(ctx, "hb_lora_qlinear", dt, x, ldx, y, ldy, M, N, K, l);
  HB_API_END
}

}  // extern "C"
