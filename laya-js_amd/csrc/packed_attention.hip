// Attention over packed documents (hb_sdpa_packed): every document's queries see
// that document's keys alone, within a window, causally, behind a prefix that
// all of them see; scores may be capped by a tanh and fall with distance.
//
//   pos(i) = i + n_k - n_q     (a document's queries are its last tokens)
//   x_ij   = scale * q_i . k_j
//   x_ij   = cap * tanh(x_ij / cap)                  with a cap
//   x_ij   = x_ij - slope_h * |pos(i) - j|           with slopes
//   o_i    = sum_j softmax_j(x_ij) v_j over the visible j
//   visible: j < prefix, or j <= pos(i) if causal and |pos(i) - j| <= half with
//   a window
//
// A query without a visible key gives zeros, and so do rows behind the last
// document.
//
// packed_attn_rows, packed_attn_few: f16 / bf16 with head dimension 64, flash
// attention on v_mfma_f32_32x32x16 with 32 rows per wave.  A row is a query and
// one of the G heads that share a key head, G rows a query, so grouped heads
// share what they read.  A block finds its document by its slot: document b has
// slots from off_b G / R + b on (R rows a block, rounded down), which leaves every
// document enough of them without a table, whatever the lengths.
// Both go through the 64-key tiles that some row of the block can see: those of
// the prefix, then the run from the first row's lowest key to the last row's
// highest.  A long run may be split over `splits` blocks; packed_attn_join adds up
// their parts.
//
// packed_attn_f32: f32, on v_mfma_f32_32x32x2_f32.
//
// packed_attn_any: any head dimension, type and strides.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <stdexcept>
#include <type_traits>

#include "attention_common.h"

namespace hb {

struct Packed {
  const void *Q, *K, *V;
  void* O;                 // [Tq, H, D]
  int64_t qs[3], ks[3], vs[3];  // element strides: token, head, column
  const int32_t *qoff, *koff;  // [B + 1]
  const int32_t* prefix;   // [B], or null
  const float* slopes;     // [H], or null
  int B, Tq, Tk, H, G, D;  // G: query heads of a key head
  int causal, half;        // half < 0: no window
  float scale, cap;        // cap <= 0: none
};

// A document's queries [q0, q0 + nq) and keys [k0, k0 + nk); document B stands
// for the rows behind the last one, and has no keys.
struct Doc {
  int q0, nq, k0, nk, prefix;
};
__device__ __forceinline__ Doc packed_doc(const Packed& p, int b) {
  Doc d;
  d.q0 = min(max(p.qoff[b], 0), p.Tq);
  if (b >= p.B) {
    d.nq = p.Tq - d.q0;
    d.k0 = d.nk = d.prefix = 0;
    return d;
  }
  d.nq = min(max(p.qoff[b + 1], d.q0), p.Tq) - d.q0;
  d.k0 = min(max(p.koff[b], 0), p.Tk);
  d.nk = min(max(p.koff[b + 1], d.k0), p.Tk) - d.k0;
  d.prefix = p.prefix == nullptr ? 0 : min(max(p.prefix[b], 0), d.nk);
  return d;
}

// The keys that a query at `pos` sees besides the prefix: [lo, hi]
__device__ __forceinline__ void packed_range(const Packed& p, int nk, int pos, int* lo, int* hi) {
  *lo = p.half >= 0 ? max(pos - p.half, 0) : 0;
  *hi = p.half >= 0 ? min(pos + p.half, nk - 1) : nk - 1;  // (both below 2^30)
  if (p.causal) *hi = min(*hi, pos);
}

// ------------------------------------------------------------------ rows and tiles

// The document of slot `slot`: the last b with off_b * G / R + b <= slot (the
// documents' first slots; document B holds the rows behind the last one).  All
// 64 lanes probe at once, so up to 63 documents take one round of loads.
template <int R>
__device__ __forceinline__ int slot_doc(const Packed& p, int64_t slot, int lane, int64_t* first) {
  auto base = [&](int b) { return (int64_t)min(max(p.qoff[b], 0), p.Tq) * p.G / R + b; };
  int lo = 0, n = p.B + 1;
  while (n > 1) {
    const int step = (n + 63) >> 6, at = lane * step;
    const int cnt = __popcll(__ballot(at < n && base(lo + (at < n ? at : 0)) <= slot));
    lo += (cnt - 1) * step;
    n = min(step, n - (cnt - 1) * step);
  }
  *first = base(lo);
  return lo;
}

// The tiles of KT keys that rows at positions pb0 .. pb1 can see: `pre` tiles of
// the prefix, then those from run0 on, `n` in all.
struct Tiles {
  int pre, run0, n;
  __device__ __forceinline__ int at(int i) const { return i < pre ? i : run0 + i - pre; }
};
template <int KT>
__device__ __forceinline__ Tiles row_tiles(const Packed& p, const Doc& d, int pb0, int pb1) {
  Tiles t;
  int lo, hi, x;
  packed_range(p, d.nk, pb0, &lo, &x);
  packed_range(p, d.nk, pb1, &x, &hi);
  t.pre = (d.prefix + KT - 1) / KT;
  t.run0 = max(lo / KT, t.pre);
  t.n = t.pre + (hi >= lo ? max(hi / KT + 1 - t.run0, 0) : 0);
  return t;
}

// One lane's row, and the visibility of a tile for all rows of its wave
struct Row {
  int pos, lo, span;  // key j is visible if j < prefix or j - lo <= span, unsigned
  int lo0, lo1, hi0, hi1;  // ranges of the wave's first and last rows' positions
  float slope;
};
__device__ __forceinline__ Row packed_row(const Packed& p, const Doc& d, int r, int rw0, int rows, int hk) {
  // (a wave without rows, rw0 >= rows, repeats the last one: its caller skips it)
  Row w;
  const int shift = d.nk - d.nq, last = min(rw0 + 31, rows - 1);
  int hi, x;
  w.pos = r / p.G + shift;
  packed_range(p, d.nk, w.pos, &w.lo, &hi);
  if (hi < w.lo) w.lo = 1 << 30, hi = w.lo;  // sees nothing of the run: keys are below 2^30
  w.span = hi - w.lo;
  packed_range(p, d.nk, min(rw0, rows - 1) / p.G + shift, &w.lo0, &w.hi0);
  packed_range(p, d.nk, last / p.G + shift, &w.lo1, &w.hi1);
  w.slope = p.slopes == nullptr ? 0.f : p.slopes[hk * p.G + r % p.G];
  return w;
}
// 0: no row sees a key of the tile, 1: every row sees every key, 2: neither
template <int KT>
__device__ __forceinline__ int tile_class(const Doc& d, const Row& w, int k0) {
  if (k0 + KT <= d.prefix) return 1;
  if (k0 >= d.prefix && (k0 > w.hi1 || k0 + KT - 1 < w.lo0)) return 0;
  return k0 + KT <= d.nk && k0 >= w.lo1 && k0 + KT - 1 <= w.hi0 ? 1 : 2;
}
__device__ __forceinline__ bool key_seen(const Doc& d, const Row& w, int j) {
  return j < d.prefix || (uint32_t)(j - w.lo) <= (uint32_t)w.span;
}

// Parts of a split run: per split and row (token * H + head) the unscaled output,
// its maximum score and its sum of weights.
struct Parts {
  float* o;    // [splits][rows][64]
  float2* ml;  // [splits][rows]
};

// ------------------------------------------------------------------ f16 / bf16 (D = 64)

constexpr float kLog2e = 1.4426950408889634f;

// A wave's 32 rows (lane l holds row l % 32; the halves split its columns and its
// keys).  Scores are in base 2 once `mul` is applied: mul is 1 where a cap or a
// slope has made them so beforehand.
struct Wave {
  uint4v qf[4];   // columns 16 s + 8 lg .. of the query per MFMA step s
  float16v o[2];  // columns 32 d + 8 (r / 4) + 4 lg + r % 4
  float m, l;     // running maximum (before mul), the lane's sum of weights
};
struct Score {
  float mul, c1, c2;  // capped: c2 tanh, computed as c2 - 2 c2 / (1 + 2^(c1 score))
  uint32_t flip;      // a negative scale turns the query round instead
};
__device__ __forceinline__ Score score_of(const Packed& p, bool cap, bool bias) {
  Score s;
  // (scale 0: any tiny factor; 0 * -inf would not be a maximum)
  const float sl = fmaxf(fabsf(p.scale), 1e-30f) * kLog2e;
  s.mul = cap || bias ? 1.f : sl;
  s.c1 = cap ? 2.f * sl / p.cap : sl;
  s.c2 = p.cap * kLog2e;
  s.flip = p.scale < 0.f ? 0x80008000u : 0u;
  return s;
}
template <bool CAP, bool BIAS>
__device__ __forceinline__ float score(const Score& s, float slope, int pos, int key, float x) {
  if constexpr (CAP) x = fmaf(-2.f * s.c2, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * s.c1)), s.c2);
  else if constexpr (BIAS) x *= s.c1;
  if constexpr (BIAS) x = fmaf(-slope, fabsf((float)(pos - key)), x);
  return x;
}

__device__ __forceinline__ void wave_init(Wave& w, const Score& sc, const uint16_t* qrow, int lg) {
#pragma unroll
  for (int s = 0; s < 4; s++) {
    w.qf[s] = *(const uint4v*)(qrow + 8 * lg + 16 * s);
#pragma unroll
    for (int e = 0; e < 4; e++) w.qf[s][e] ^= sc.flip;
  }
#pragma unroll
  for (int d = 0; d < 2; d++)
#pragma unroll
    for (int r = 0; r < 16; r++) w.o[d][r] = 0.f;
  w.m = -INFINITY;
  w.l = 0.f;
}

// One tile of 64 keys in LDS: scores, mask (`mixed`), online softmax, O += P V.
// Weights are rounded to the 16-bit type for the second product, as MFMA takes
// them; their sum is of the unrounded ones.
template <bool BF16, bool CAP, bool BIAS>
__device__ __forceinline__ void wave_tile(Wave& w, const Frag32& f, const uint16_t* Kc, const uint16_t* Vc, int k0,
                                          const Doc& d, const Row& row, bool mixed, const Score& sc, int lg) {
  float16v st[2];
#pragma unroll
  for (int kb = 0; kb < 2; kb++) {
#pragma unroll
    for (int r = 0; r < 16; r++) st[kb][r] = 0.f;
#pragma unroll
    for (int s = 0; s < 4; s++) st[kb] = mfma32x16<BF16>(*(const uint4v*)(Kc + f.ka[s] + kb * 2048), w.qf[s], st[kb]);
  }
  if constexpr (CAP || BIAS) {
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 16; r++)
        st[kb][r] = score<CAP, BIAS>(sc, row.slope, row.pos, k0 + 32 * kb + 8 * (r >> 2) + 4 * lg + (r & 3), st[kb][r]);
  }
  if (mixed) {
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 16; r++)
        st[kb][r] = key_seen(d, row, k0 + 32 * kb + 8 * (r >> 2) + 4 * lg + (r & 3)) ? st[kb][r] : -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int kb = 0; kb < 2; kb++)
#pragma unroll
    for (int r = 0; r < 16; r++) mx = fmaxf(mx, st[kb][r]);
  mx = max_xor32(mx);
  const float mnew = fmaxf(w.m, mx);
  const float mc = mnew == -INFINITY ? 0.f : mnew * sc.mul;
  const float alpha = __builtin_amdgcn_exp2f(w.m * sc.mul - mc);
  w.m = mnew;
  float psum = 0.f;
  uint4v pf[4];
#pragma unroll
  for (int t = 0; t < 4; t++) {
    uint32_t pk[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(st[t >> 1][8 * (t & 1) + e], sc.mul, -mc));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(st[t >> 1][8 * (t & 1) + e + 1], sc.mul, -mc));
      psum += p0 + p1;
      pk[e >> 1] = pack2<BF16>(p0, p1);
    }
    pf[t] = uint4v{pk[0], pk[1], pk[2], pk[3]};
  }
  w.l = w.l * alpha + psum;
  if (!__all(alpha == 1.0f)) {  // rescale O only when some row max of this wave moved
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int r = 0; r < 16; r++) w.o[e][r] *= alpha;
  }
#pragma unroll
  for (int t = 0; t < 4; t++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const uint2v v0 = lds_tr16(Vc + f.va[0][e] + t * 1024), v1 = lds_tr16(Vc + f.va[1][e] + t * 1024);
      w.o[e] = mfma32x16<BF16>(uint4v{v0.x, v0.y, v1.x, v1.y}, pf[t], w.o[e]);
    }
}

// A non-finite value must not reach a row whose weight for its key is 0 (hidden,
// or underflowed), as 0 * inf in the product does.  Where a wave's output has
// come out non-finite it is computed again, key by key, zero weights skipped:
// slow, and never run on finite data.  tiles [i0, i1) in steps of `step`.
template <bool BF16, bool CAP, bool BIAS>
__device__ __forceinline__ Wave wave_again(Wave w, const uint16_t* Kb, int64_t kst, const uint16_t* Vb, int64_t vst,
                                        Doc d, Row row, Tiles ti, int i0, int i1, int step,
                                        Score sc, int lg) {
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int r = 0; r < 16; r++) w.o[e][r] = 0.f;
  w.m = -INFINITY;
  w.l = 0.f;
#pragma unroll 1
  for (int i = i0; i < i1; i += step) {
    const int k0 = ti.at(i) * 64, k1 = min(k0 + 64, d.nk);
#pragma unroll 1
    for (int j = k0; j < k1; j++) {
      const uint16_t* kr = Kb + j * kst + 8 * lg;
      float x = 0.f;
#pragma unroll
      for (int s = 0; s < 4; s++) {
        const uint4v kv = *(const uint4v*)(kr + 16 * s);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x = fmaf(tof<BF16>(kv[e] & 0xffff), tof<BF16>(w.qf[s][e] & 0xffff), x);
          x = fmaf(tof<BF16>(kv[e] >> 16), tof<BF16>(w.qf[s][e] >> 16), x);
        }
      }
      x = score<CAP, BIAS>(sc, row.slope, row.pos, j, sum_xor32(x));
      x = key_seen(d, row, j) ? x : -INFINITY;
      const float mnew = fmaxf(w.m, x), mc = mnew == -INFINITY ? 0.f : mnew * sc.mul;
      const float alpha = __builtin_amdgcn_exp2f(w.m * sc.mul - mc), pr = __builtin_amdgcn_exp2f(fmaf(x, sc.mul, -mc));
      w.m = mnew;
      w.l = w.l * alpha + (lg == 0 ? pr : 0.f);  // (the halves' sums are added up later)
      const float p16 = tof<BF16>(fromf<BF16>(pr));
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++) {
          const uint2v vv = *(const uint2v*)(Vb + j * vst + 32 * e + 8 * r4 + 4 * lg);
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const float v = tof<BF16>(((c & 2) ? vv.y : vv.x) >> (16 * (c & 1)) & 0xffff);
            const float o = w.o[e][4 * r4 + c] * alpha;
            w.o[e][4 * r4 + c] = p16 == 0.f ? o : fmaf(p16, v, o);
          }
        }
    }
  }
  return w;
}
__device__ __forceinline__ bool wave_finite(const Wave& w) {
  float z = w.l * 0.f;
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int r = 0; r < 16; r++) z = fmaf(w.o[e][r], 0.f, z);
  return !__any(z != 0.f);  // 0 * finite = 0, 0 * (inf or NaN) = NaN
}

__device__ __forceinline__ int64_t row_index(const Packed& p, const Doc& d, int r, int hk) {
  return (int64_t)(d.q0 + r / p.G) * p.H + hk * p.G + r % p.G;
}

// 128 rows a block, four waves of 32, K and V tiles in a two-buffer LDS ring with
// one barrier per tile.
constexpr int kRowsB = 128;
template <bool BF16, bool CAP, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) void packed_attn_rows(Packed p, Parts part,
                                                                                                int splits) {
  __shared__ __attribute__((aligned(16))) uint16_t Ks[2][64 * 64];
  __shared__ __attribute__((aligned(16))) uint16_t Vs[2][64 * 64];
  const int tid = threadIdx.x, lane = tid & 63, lg = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hk = p.H / p.G, hk = blockIdx.x % Hk;
  const int64_t slot = blockIdx.x / Hk;
  int64_t first;
  const int b = slot_doc<kRowsB>(p, slot, lane, &first);
  const Doc d = packed_doc(p, b);
  const int64_t at = (slot - first) * kRowsB;
  if (at >= (int64_t)d.nq * p.G) return;  // (the whole block)
  const int rows = d.nq * p.G, r0 = (int)at, rw0 = r0 + 32 * wave;
  const int r = rw0 + (lane & 31), rc = min(r, rows - 1);
  const Score sc = score_of(p, CAP, BIAS);
  Row row = packed_row(p, d, rc, rw0, rows, hk);
  row.slope *= kLog2e;
  const int shift = d.nk - d.nq;
  const Tiles ti = row_tiles<64>(p, d, r0 / p.G + shift, min(r0 + kRowsB - 1, rows - 1) / p.G + shift);
  const int s = blockIdx.y, i0 = (int)((int64_t)ti.n * s / splits), i1 = (int)((int64_t)ti.n * (s + 1) / splits);
  const uint16_t* Kb = (const uint16_t*)p.K + d.k0 * p.ks[0] + hk * p.ks[1];
  const uint16_t* Vb = (const uint16_t*)p.V + d.k0 * p.vs[0] + hk * p.vs[1];
  Wave w;
  wave_init(w, sc, (const uint16_t*)p.Q + (d.q0 + rc / p.G) * p.qs[0] + (hk * p.G + rc % p.G) * p.qs[1], lg);
  auto fetch = [&](int i, int bf) __attribute__((always_inline)) {
    const int k0 = ti.at(i) * 64;
#pragma unroll
    for (int q = 0; q < 2; q++) dma_piece(Vb, p.vs[0], k0, wave * 2 + q, d.nk, Vs[bf], lane);
#pragma unroll
    for (int q = 0; q < 2; q++) dma_piece(Kb, p.ks[0], k0, wave * 2 + q, d.nk, Ks[bf], lane);
  };
  if (i0 < i1) fetch(i0, 0);
  const Frag32 f = frag32(lane);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int bf = 0;
  for (int i = i0; i < i1; i++) {
    // the next tile into the other buffer (free since the last barrier)
    if (i + 1 < i1) fetch(i + 1, bf ^ 1);
    const int k0 = ti.at(i) * 64, cl = rw0 < rows ? tile_class<64>(d, row, k0) : 0;
    if (cl != 0) wave_tile<BF16, CAP, BIAS>(w, f, Ks[bf], Vs[bf], k0, d, row, cl == 2, sc, lg);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    bf ^= 1;
    __syncthreads();
  }
  if (!wave_finite(w)) w = wave_again<BF16, CAP, BIAS>(w, Kb, p.ks[0], Vb, p.vs[0], d, row, ti, i0, i1, 1, sc, lg);
  const float lt = sum_xor32(w.l);
  if (r >= rows) return;
  const int64_t ri = row_index(p, d, r, hk);
  if (splits > 1) {
    const int64_t pr = (int64_t)s * p.Tq * p.H + ri;
    if (lg == 0) part.ml[pr] = float2{w.m * sc.mul, lt};
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        *(float4v*)(part.o + pr * 64 + 32 * e + 8 * j + 4 * lg) =
            float4v{w.o[e][4 * j], w.o[e][4 * j + 1], w.o[e][4 * j + 2], w.o[e][4 * j + 3]};
    return;
  }
  const float inv = lt == 0.f ? 0.f : 1.0f / lt;
  uint16_t* op = (uint16_t*)p.O + ri * 64 + 4 * lg;
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int j = 0; j < 4; j++)
      *(uint2v*)(op + 32 * e + 8 * j) = uint2v{pack2<BF16>(w.o[e][4 * j] * inv, w.o[e][4 * j + 1] * inv),
                                               pack2<BF16>(w.o[e][4 * j + 2] * inv, w.o[e][4 * j + 3] * inv)};
}

// 32 rows a block, for few queries a document: the block's four waves hold the
// same rows and take its tiles in turn, each through an LDS ring of its own with
// no barrier, so the block has 64 KB of keys and values on their way; then the
// waves' parts are joined.  Bound by reading K and V once.
constexpr int kRowsF = 32, kFewLds = 4 * 2 * 2 * 64 * 64 * 2;  // four rings of two K and V tiles
template <bool BF16, bool CAP, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1))) void packed_attn_few(Packed p, Parts part,
                                                                                               int splits) {
  extern __shared__ __attribute__((aligned(16))) uint16_t ring[];
  __shared__ float part_m[4][kRowsF], part_l[4][kRowsF];
  const int tid = threadIdx.x, lane = tid & 63, lg = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hk = p.H / p.G, hk = blockIdx.x % Hk;
  const int64_t slot = blockIdx.x / Hk;
  int64_t first;
  const int b = slot_doc<kRowsF>(p, slot, lane, &first);
  const Doc d = packed_doc(p, b);
  const int64_t at = (slot - first) * kRowsF;
  if (at >= (int64_t)d.nq * p.G) return;  // (the whole block)
  const int rows = d.nq * p.G, r0 = (int)at, r = r0 + l32, rc = min(r, rows - 1);
  const Score sc = score_of(p, CAP, BIAS);
  Row row = packed_row(p, d, rc, r0, rows, hk);
  row.slope *= kLog2e;
  const int shift = d.nk - d.nq;
  const Tiles ti = row_tiles<64>(p, d, r0 / p.G + shift, min(r0 + kRowsF - 1, rows - 1) / p.G + shift);
  const int s = blockIdx.y, i0 = (int)((int64_t)ti.n * s / splits) + wave, i1 = (int)((int64_t)ti.n * (s + 1) / splits);
  const uint16_t* Kb = (const uint16_t*)p.K + d.k0 * p.ks[0] + hk * p.ks[1];
  const uint16_t* Vb = (const uint16_t*)p.V + d.k0 * p.vs[0] + hk * p.vs[1];
  uint16_t* mine = ring + wave * (4 * 64 * 64);  // K, V, K, V
  auto fetch = [&](int i, int bf) __attribute__((always_inline)) {
    const int k0 = ti.at(i) * 64;
    // this wave's reads of the tile that was there are done
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int q = 0; q < 8; q++) dma_piece(Kb, p.ks[0], k0, q, d.nk, mine + bf * 8192, lane);
#pragma unroll
    for (int q = 0; q < 8; q++) dma_piece(Vb, p.vs[0], k0, q, d.nk, mine + bf * 8192 + 4096, lane);
  };
  Wave w;
  wave_init(w, sc, (const uint16_t*)p.Q + (d.q0 + rc / p.G) * p.qs[0] + (hk * p.G + rc % p.G) * p.qs[1], lg);
  const Frag32 f = frag32(lane);
  if (i0 < i1) fetch(i0, 0);
  int bf = 0;
  for (int i = i0; i < i1; i += 4) {
    if (i + 4 < i1) {
      fetch(i + 4, bf ^ 1);
      asm volatile("s_waitcnt vmcnt(16)" ::: "memory");  // all but the 16 loads just requested
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const int k0 = ti.at(i) * 64, cl = tile_class<64>(d, row, k0);
    if (cl != 0)
      wave_tile<BF16, CAP, BIAS>(w, f, mine + bf * 8192, mine + bf * 8192 + 4096, k0, d, row, cl == 2, sc, lg);
    bf ^= 1;
  }
  if (!wave_finite(w)) w = wave_again<BF16, CAP, BIAS>(w, Kb, p.ks[0], Vb, p.vs[0], d, row, ti, i0, i1, 4, sc, lg);
  // join the waves: weights 2^(m_w - max); wave w finishes registers [8 w, 8 w + 8)
  // of the 32
  const float lw = sum_xor32(w.l);
  if (lg == 0) {
    part_m[wave][l32] = w.m * sc.mul;
    part_l[wave][l32] = lw;
  }
  float* buf = (float*)ring;
  __syncthreads();  // every wave is done with its ring
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int i = 0; i < 16; i++) buf[wave * 2048 + (e * 16 + i) * 64 + lane] = w.o[e][i];
  __syncthreads();
  float mt = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; i++) mt = fmaxf(mt, part_m[i][l32]);
  const float mc = mt == -INFINITY ? 0.f : mt;
  float wt[4], lt = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    wt[i] = __builtin_amdgcn_exp2f(part_m[i][l32] - mc);
    lt += part_l[i][l32] * wt[i];
  }
  if (r >= rows) return;
  const float inv = lt == 0.f ? 0.f : 1.0f / lt;
  const int64_t ri = row_index(p, d, r, hk), pr = (int64_t)s * p.Tq * p.H + ri;
  if (splits > 1 && wave == 0 && lg == 0) part.ml[pr] = float2{mt, lt};
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int x = wave * 8 + h * 4, col = 32 * (x >> 4) + 8 * ((x & 15) >> 2) + 4 * lg;
    float4v ov;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < 4; i++) a += wt[i] == 0.f ? 0.f : buf[i * 2048 + (x + e) * 64 + lane] * wt[i];
      ov[e] = a;
    }
    if (splits > 1) {
      *(float4v*)(part.o + pr * 64 + col) = ov;
    } else {
      *(uint2v*)((uint16_t*)p.O + ri * 64 + col) =
          uint2v{pack2<BF16>(ov[0] * inv, ov[1] * inv), pack2<BF16>(ov[2] * inv, ov[3] * inv)};
    }
  }
}

// ------------------------------------------------------------------ f32 (D = 64)

// 32 rows a block; its four waves take the 32-key tiles those rows can see in
// turn, each with its own maximum, sum and output, and join them in LDS at the
// end.  Bound by the f32 matrix rate: a tile is 64 MFMAs of 64 cycles.  K goes
// through a wave-private LDS tile, V straight into operand registers, a whole
// 128-byte line per 32 lanes.  S^T = K . Q^T leaves lane l with the scores of row
// l % 32 for keys 8 (r / 4) + 4 (l / 32) + r % 4, which are the columns that the
// B operand of O^T += V^T . P^T takes when MFMA step r multiplies keys 8 (r / 4) +
// r % 4 and + 4: weights stay in registers, in f32.
constexpr int kRows32 = 32, kKeys32 = 32;
template <bool CAP, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void packed_attn_f32(Packed p, Parts part,
                                                                                               int splits) {
  __shared__ __attribute__((aligned(16))) float buf[4][kKeys32 * 64];  // K tiles; the waves' outputs at the end
  __shared__ float part_m[4][kRows32], part_l[4][kRows32];
  const int tid = threadIdx.x, lane = tid & 63, lg = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hk = p.H / p.G, hk = blockIdx.x % Hk;
  const int64_t slot = blockIdx.x / Hk;
  int64_t first;
  const int b = slot_doc<kRows32>(p, slot, lane, &first);
  const Doc d = packed_doc(p, b);
  const int64_t at = (slot - first) * kRows32;
  if (at >= (int64_t)d.nq * p.G) return;  // (the whole block)
  const int rows = d.nq * p.G, r0 = (int)at, r = r0 + l32, rc = min(r, rows - 1);
  const Row row = packed_row(p, d, rc, r0, rows, hk);
  const int shift = d.nk - d.nq;
  const Tiles ti = row_tiles<kKeys32>(p, d, r0 / p.G + shift, min(r0 + kRows32 - 1, rows - 1) / p.G + shift);
  const int s = blockIdx.y, i0 = (int)((int64_t)ti.n * s / splits) + wave, i1 = (int)((int64_t)ti.n * (s + 1) / splits);
  const float* Kb = (const float*)p.K + d.k0 * p.ks[0] + hk * p.ks[1];
  const float* Vb = (const float*)p.V + d.k0 * p.vs[0] + hk * p.vs[1];

  // element e of qf[i] is column 8 i + 4 lg + e, the columns its half supplies to
  // MFMA steps e of chunk pair i
  float4v qf[8];
  {
    const float* qp = (const float*)p.Q + (d.q0 + rc / p.G) * p.qs[0] + (hk * p.G + rc % p.G) * p.qs[1] + 4 * lg;
#pragma unroll
    for (int i = 0; i < 8; i++) qf[i] = *(const float4v*)(qp + 8 * i);
  }
  // K tile: 8 lanes a row, chunk c of row r at c ^ (r & 15): a 16-lane pass of the
  // fragment reads (16 rows, one chunk) covers all 64 banks.  Keys past the
  // document repeat its last one: their scores are hidden.
  const int kr = lane >> 3, c8 = lane & 7;
  float4v klo[4], khi[4];
  auto load_k = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float* kp = Kb + min(k0 + i * 8 + kr, d.nk - 1) * p.ks[0] + 4 * c8;
      klo[i] = *(const float4v*)kp;
      khi[i] = *(const float4v*)(kp + 32);
    }
  };
  auto kslot = [](int r_, int c) { return r_ * 64 + ((c ^ (r_ & 15)) << 2); };
  float* kb = buf[wave];
  float16v o[2];
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[e][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  if (i0 < i1) load_k(ti.at(i0) * kKeys32);
  for (int i = i0; i < i1; i += 4) {
    const int k0 = ti.at(i) * kKeys32, cl = tile_class<kKeys32>(d, row, k0);
#pragma unroll
    for (int q = 0; q < 4; q++) {
      *(float4v*)(kb + kslot(q * 8 + kr, c8)) = klo[q];
      *(float4v*)(kb + kslot(q * 8 + kr, c8 + 8)) = khi[q];
    }
    // the tile is this wave's own: its LDS stores and loads only need to stay in
    // order
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // V of the tile, the next tile's K
    float v[2][16];
#pragma unroll
    for (int q = 0; q < 16; q++) {
      const float* vp = Vb + min(k0 + 8 * (q >> 2) + 4 * lg + (q & 3), d.nk - 1) * p.vs[0] + l32;
      v[0][q] = vp[0];
      v[1][q] = vp[32];
    }
    if (i + 4 < i1) load_k(ti.at(i + 4) * kKeys32);
    float16v st;
#pragma unroll
    for (int q = 0; q < 16; q++) st[q] = 0.f;
#pragma unroll
    for (int q = 0; q < 8; q++) {
      const float4v kf = *(const float4v*)(kb + kslot(l32, 2 * q + lg));
#pragma unroll
      for (int e = 0; e < 4; e++) st = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], qf[q][e], st, 0, 0, 0);
    }
    // (the next tile's stores must not overtake these reads)
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float mx = -INFINITY;
#pragma unroll
    for (int q = 0; q < 16; q++) {
      const int key = k0 + 8 * (q >> 2) + 4 * lg + (q & 3);
      float x = st[q] * p.scale;
      if constexpr (CAP) x = p.cap * tanhf(x / p.cap);
      if constexpr (BIAS) x = fmaf(-row.slope, fabsf((float)(row.pos - key)), x);
      if (cl != 1) x = key_seen(d, row, key) ? x : -INFINITY;
      st[q] = x;
      mx = fmaxf(mx, x);
    }
    mx = max_xor32(mx);
    const float mnew = fmaxf(m, mx), mc = mnew == -INFINITY ? 0.f : mnew, alpha = expf(m - mc);
    m = mnew;
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < 16; q++) {
      st[q] = expf(st[q] - mc);
      sum += st[q];
    }
    l = l * alpha + sum;
    if (!__all(alpha == 1.0f)) {
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int q = 0; q < 16; q++) o[e][q] *= alpha;
    }
    // A non-finite V must not reach a row whose weight for that key is 0, as 0 *
    // inf in the product would: such a tile is added key by key, zero weights
    // skipped.
    float fin = 0.f;
#pragma unroll
    for (int q = 0; q < 16; q++) fin += v[0][q] * 0.f + v[1][q] * 0.f;
    if (__any(fin != 0.f)) {  // 0 * finite = 0, 0 * (inf or NaN) = NaN
#pragma unroll
      for (int q = 0; q < 16; q++) kb[(8 * (q >> 2) + 4 * lg + (q & 3)) * 32 + l32] = st[q];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll 1
      for (int j = 0; j < kKeys32; j++) {
        const float w = kb[j * 32 + l32];
        if (w == 0.f) continue;  // keys past the document among them
        const float* vp = Vb + (k0 + j) * p.vs[0] + 4 * lg;
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
          for (int q = 0; q < 16; q++) o[e][q] = fmaf(w, vp[32 * e + 8 * (q >> 2) + (q & 3)], o[e][q]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      continue;
    }
#pragma unroll
    for (int q = 0; q < 16; q++)
#pragma unroll
      for (int e = 0; e < 2; e++) o[e] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[e][q], st[q], o[e], 0, 0, 0);
  }
  // join the waves: weights exp(m_w - max); wave w finishes registers [8 w, 8 w + 8)
  const float lw = sum_xor32(l);
  if (lg == 0) {
    part_m[wave][l32] = m;
    part_l[wave][l32] = lw;
  }
  __syncthreads();  // every wave is done with its K tile
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int q = 0; q < 16; q++) buf[wave][(e * 16 + q) * 64 + lane] = o[e][q];
  __syncthreads();
  float mt = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; w++) mt = fmaxf(mt, part_m[w][l32]);
  const float mc = mt == -INFINITY ? 0.f : mt;
  float wt[4], lt = 0.f;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    wt[w] = expf(part_m[w][l32] - mc);
    lt += part_l[w][l32] * wt[w];
  }
  if (r >= rows) return;
  const float inv = splits > 1 ? 1.f : lt == 0.f ? 0.f : 1.0f / lt;
  const int64_t ri = row_index(p, d, r, hk), pr = (int64_t)s * p.Tq * p.H + ri;
  if (splits > 1 && wave == 0 && lg == 0) part.ml[pr] = float2{mt, lt};
  float* op = splits > 1 ? part.o + pr * 64 : (float*)p.O + ri * 64;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int x = wave * 8 + h * 4;  // register x: column 32 (x / 16) + 8 (x % 16 / 4) + 4 lg
    float4v ov;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < 4; w++) a += wt[w] == 0.f ? 0.f : buf[w][(x + e) * 64 + lane] * wt[w];
      ov[e] = a * inv;
    }
    *(float4v*)(op + 32 * (x >> 4) + 8 * ((x & 15) >> 2) + 4 * lg) = ov;
  }
}

// Joins the parts of split runs: one wave a row, a lane per column.  E2: maxima in
// base 2 (the 16-bit kernels), else natural.
template <bool E2>
__global__ __launch_bounds__(256) void packed_attn_join(int dt, Parts part, int splits, int64_t rows,
                                                        void* __restrict__ O) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= rows) return;
  float m = -INFINITY;
  for (int s = 0; s < splits; s++) m = fmaxf(m, part.ml[s * rows + r].x);
  const float mc = m == -INFINITY ? 0.f : m;
  float l = 0.f, o = 0.f;
  for (int s = 0; s < splits; s++) {
    const float2 ml = part.ml[s * rows + r];
    const float w = E2 ? __builtin_amdgcn_exp2f(ml.x - mc) : expf(ml.x - mc);
    l = fmaf(ml.y, w, l);
    if (w != 0.f) o = fmaf(part.o[(s * rows + r) * 64 + lane], w, o);
  }
  store_f(O, r * 64 + lane, dt, l == 0.f ? 0.f : o / l);
}

// ------------------------------------------------------------------ any type

// One wave per query and head: 64 keys at a time, a score per lane, then the
// lanes share out the columns of the output.
constexpr int kAnyCols = 8;  // columns per lane: D <= 512
__global__ __launch_bounds__(64) void packed_attn_any(Packed p, int dt) {
  extern __shared__ float sh[];  // [D] query, [64] weights
  float* w = sh + p.D;
  const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y, D = p.D;
  int b = 0, e = p.B + 1;  // the last document that begins at or before t
  while (e - b > 1) {
    const int m = (b + e) >> 1;
    if (p.qoff[m] <= t) b = m;
    else e = m;
  }
  const Doc d = packed_doc(p, b);
  const int pos = t - d.q0 + d.nk - d.nq;
  int lo, hi;
  packed_range(p, d.nk, pos, &lo, &hi);
  for (int c = lane; c < D; c += 64) sh[c] = load_f(p.Q, t * p.qs[0] + h * p.qs[1] + c * p.qs[2], dt);
  __syncthreads();
  const float slope = p.slopes == nullptr ? 0.f : p.slopes[h];
  float o[kAnyCols] = {}, m = -INFINITY, l = 0.f;
  const int64_t kh = (h / p.G) * p.ks[1], vh = (h / p.G) * p.vs[1];
  for (int j0 = 0; j0 < d.nk; j0 += 64) {
    // (the same in every lane: nothing of these keys is visible)
    if (j0 >= d.prefix && (j0 > hi || j0 + 63 < lo)) continue;
    const int j = j0 + lane;
    const bool seen = j < d.nk && (j < d.prefix || (j >= lo && j <= hi));
    float x = -INFINITY;
    if (seen) {
      const int64_t row = (int64_t)(d.k0 + j) * p.ks[0] + kh;
      float a = 0.f;
      for (int c = 0; c < D; c++) a = fmaf(sh[c], load_f(p.K, row + c * p.ks[2], dt), a);
      x = a * p.scale;
      if (p.cap > 0.f) x = p.cap * tanhf(x / p.cap);
      x -= slope * fabsf((float)(pos - j));
    }
    const float mn = fmaxf(m, wave_max(x));
    const float mc = mn == -INFINITY ? 0.f : mn, alpha = expf(m - mc);
    m = mn;
    const float pr = seen ? expf(x - mc) : 0.f;  // (NaN scores stay NaN)
    l = l * alpha + wave_sum(pr);
    __syncthreads();  // the last keys' weights are used up
    w[lane] = pr;
    __syncthreads();
    for (int i = 0; i < kAnyCols && i * 64 + lane < D; i++) {
      float a = o[i] * alpha;
      const int64_t col = vh + (i * 64 + lane) * p.vs[2];
      for (int k = 0; k < 64 && j0 + k < d.nk; k++)
        if (w[k] != 0.f) a = fmaf(w[k], load_f(p.V, (int64_t)(d.k0 + j0 + k) * p.vs[0] + col, dt), a);
      o[i] = a;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int i = 0; i < kAnyCols && i * 64 + lane < D; i++)
    store_f(p.O, ((int64_t)t * p.H + h) * D + i * 64 + lane, dt, o[i] * inv);
}

// ------------------------------------------------------------------ dispatch

// The MFMA kernels' conditions: D = 64, unit column strides, 16-byte aligned rows
// (`per` elements), and K / V row strides that 32-bit offsets within a tile reach.
static bool packed_takes_mfma(const Packed& p, int per) {
  auto rows16 = [&](const void* t, const int64_t* s) {
    return (uintptr_t)t % 16 == 0 && s[2] == 1 && s[0] % per == 0 && s[1] % per == 0;
  };
  auto near = [](int64_t s) { return s >= 0 && s < (1 << 23); };
  return p.D == 64 && (int64_t)p.Tq * p.G < (1ll << 30) && rows16(p.Q, p.qs) && rows16(p.K, p.ks) && rows16(p.V, p.vs) && near(p.ks[0]) && near(p.vs[0]) &&
         (uintptr_t)p.O % 16 == 0;
}

static void packed_any(uintptr_t ctx, int dt, const Packed& p) {
  packed_attn_any<<<dim3((unsigned)p.Tq, (unsigned)p.H), 64, (size_t)(p.D + 64) * 4, stream_of(ctx)>>>(p, dt);
}

template <class K>
static void packed_launch(uintptr_t ctx, K kern, std::atomic<uint64_t>& attr, int lds, int rows, const Packed& p, int splits,
                          const Parts& part) {
  if (lds > 64 * 1024)
    once_per_device(attr, [&] {
      HB_CHECK_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    });
  const int64_t grid = ((int64_t)p.Tq * p.G / rows + p.B + 1) * (p.H / p.G);
  HB_REQUIRE(grid < (1ll << 31), "hb_sdpa_packed: too many rows and heads");
  kern<<<dim3((unsigned)grid, (unsigned)splits), 256, (size_t)lds, stream_of(ctx)>>>(p, part, splits);
}

static void packed_mfma(uintptr_t ctx, int dt, const Packed& p) {
  const int64_t rows = (int64_t)p.Tq * p.G;
  const bool f32 = dt == HB_F32, few = f32 || rows <= 64 * (int64_t)p.B;
  const int per = few ? kRowsF : kRowsB, Hk = p.H / p.G, cus = cu_count(ctx);
  // Keys of an average document's rows, and the blocks they make
  int64_t keys = p.B ? p.Tk / p.B : 0;
  if (p.half >= 0) keys = std::min<int64_t>(keys, 2 * (int64_t)p.half + per / p.G + 64);
  const int64_t blocks = std::max<int64_t>((rows + per - 1) / per, p.B) * Hk;
  const int64_t want = 4 * (int64_t)cus, most = keys / 512;
  int splits = (int)std::max<int64_t>(1, std::min<int64_t>({most, (want + blocks - 1) / std::max<int64_t>(blocks, 1), 32}));
  CallScratch held(ctx);
  Parts part{nullptr, nullptr};
  const int64_t all = (int64_t)p.Tq * p.H;
  if (splits > 1) {
    if (held.take((size_t)(splits * all * (64 * 4 + 8)))) {
      part.o = (float*)held.p;
      part.ml = (float2*)(part.o + splits * all * 64);
    } else {
      splits = 1;  // no memory for the parts: unsplit
    }
  }
  auto go = [&](auto cap, auto bias) {
    constexpr bool CAP = decltype(cap)::value, BIAS = decltype(bias)::value;
    auto half = [&](auto bf) {
      constexpr bool BF = decltype(bf)::value;
      static std::atomic<uint64_t> attr{0};
      if (few) packed_launch(ctx, packed_attn_few<BF, CAP, BIAS>, attr, kFewLds, kRowsF, p, splits, part);
      else packed_launch(ctx, packed_attn_rows<BF, CAP, BIAS>, attr, 0, kRowsB, p, splits, part);
    };
    std::atomic<uint64_t> none{0};
    if (f32) packed_launch(ctx, packed_attn_f32<CAP, BIAS>, none, 0, kRows32, p, splits, part);
    else if (dt == HB_BF16) half(std::true_type{});
    else half(std::false_type{});
  };
  const std::true_type yes{};
  const std::false_type no{};
  if (p.cap > 0.f && p.slopes) go(yes, yes);
  else if (p.cap > 0.f) go(yes, no);
  else if (p.slopes) go(no, yes);
  else go(no, no);
  if (splits > 1) {
    check_launch("hb_sdpa_packed");
    auto join = f32 ? packed_attn_join<false> : packed_attn_join<true>;
    join<<<(unsigned)((all + 3) / 4), 256, 0, stream_of(ctx)>>>(dt, part, splits, all, p.O);
  }
}

}  // namespace hb

using namespace hb;

extern "C" int hb_sdpa_packed(uintptr_t ctx, int dt, uintptr_t q, const int64_t* qs, uintptr_t k, const int64_t* ks,
                              uintptr_t v, const int64_t* vs, uintptr_t o, uintptr_t q_offsets, uintptr_t k_offsets,
                              int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hk, int64_t D, float scale,
                              int causal, int64_t window, uintptr_t prefix, float cap, uintptr_t slopes) {
  HB_API_BEGIN
  HB_REQUIRE(dt == HB_F32 || dt == HB_F16 || dt == HB_BF16, "hb_sdpa_packed: dtype must be f32, f16 or bf16");
  HB_REQUIRE(B >= 0 && Tq >= 0 && Tk >= 0 && B < (1ll << 30) && Tq < (1ll << 30) && Tk < (1ll << 30),
             "hb_sdpa_packed: bad sizes");
  HB_REQUIRE(H >= 1 && Hk >= 1 && H % Hk == 0 && H < 65536, "hb_sdpa_packed: heads must be a multiple of the key heads");
  HB_REQUIRE(D >= 1 && D <= 64 * kAnyCols, "hb_sdpa_packed: head dimension must be 1 to 512");
  HB_REQUIRE(qs && ks && vs, "hb_sdpa_packed: null strides");
  HB_REQUIRE(std::isfinite(scale) && std::isfinite(cap) && cap >= 0.f, "hb_sdpa_packed: scale and cap must be finite");
  HB_REQUIRE(window >= -1, "hb_sdpa_packed: a window is not negative (-1: none)");
  if (Tq == 0) return 0;
  HB_REQUIRE(q && o && q_offsets && k_offsets && (Tk == 0 || (k && v)), "hb_sdpa_packed: null argument");
  Packed p;
  p.Q = (const void*)q;
  p.K = (const void*)k;
  p.V = (const void*)v;
  p.O = (void*)o;
  for (int i = 0; i < 3; i++) {
    p.qs[i] = qs[i];
    p.ks[i] = ks[i];
    p.vs[i] = vs[i];
  }
  p.qoff = (const int32_t*)q_offsets;
  p.koff = (const int32_t*)k_offsets;
  p.prefix = (const int32_t*)prefix;
  p.slopes = (const float*)slopes;
  p.B = (int)B;
  p.Tq = (int)Tq;
  p.Tk = (int)Tk;
  p.H = (int)H;
  p.G = (int)(H / Hk);
  p.D = (int)D;
  p.causal = causal ? 1 : 0;
  p.half = window < 0 ? -1 : (int)(window / 2 < (1ll << 30) ? window / 2 : (1ll << 30) - 1);
  p.scale = scale;
  p.cap = cap;
  if (packed_takes_mfma(p, dt == HB_F32 ? 4 : 8)) packed_mfma(ctx, dt, p);
  else packed_any(ctx, dt, p);
  check_launch("hb_sdpa_packed");
  HB_API_END
}
