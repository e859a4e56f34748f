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
// packed_attn_rows, packed_attn_few: f16 / bf16 with head dimension 64, one pass over
// the keys on v_mfma_f32_32x32x16 with 32 rows per wave.  A row is a query and
// one of the G heads that share a key head, G rows a query, so grouped heads
// share what they read.  Blocks of 128 rows are those of the plan's table; blocks of 32
// find their document by their slot (slot_doc).
// Both go through the 64-key tiles that some row of the block can see (tiles_of).
// A long run may be split over `splits` blocks; packed_attn_join adds up
// their parts.
//
// packed_attn_f32_rows, packed_attn_f32: the same for f32, on v_mfma_f32_32x32x2_f32.
//
// packed_attn_any: any head dimension, type and strides.
#include <float.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <stdexcept>
#include <type_traits>

#include "attention_common.h"

namespace hb {

constexpr float kLog2e = 1.4426950408889634f;

// Scores to base 2 (the 16-bit kernels).
struct Score {
  float mul, c1, c2;  // mul: the factor left once a cap or slope has been applied (1), else of the products
  float g, odd[5], far;      // score / cap of a product; coefficients of the capped score in that, and the products they hold for
  float poly[5], near;       // coefficients in the product itself
  float tiny[3], tiny_near;  // fewer of them for smaller products
  uint32_t flip;      // a negative scale turns the query round instead
};

struct Packed {
  const void *Q, *K, *V;
  void* O;                 // [Tq, H, D]
  int64_t qs[3], ks[3], vs[3];  // element strides: token, head, column
  const int32_t *qoff, *koff;  // [B + 1]
  const int32_t* doc;      // [Tq], outside [0, B) behind the last document
  const int32_t* blocks;   // [nblocks, 2]: document (below 0: none) and first row of each block of tokens
  int nblocks;
  const int32_t* prefix;   // [B], or null
  const float* slopes;     // [H], or null
  int B, Tq, Tk, H, G, D;  // G: query heads of a key head
  int causal, half;        // half < 0: no window
  float scale, cap;        // cap <= 0: none
  Score sc;
};

// A document's queries [q0, q0 + nq) and keys [k0, k0 + nk); document B stands
// for the rows behind the last one, and has no keys.
struct Doc {
  int q0, nq, k0, nk, prefix;
};
__device__ __forceinline__ Doc packed_doc(const Packed& p, int b) {
  Doc d;
  if (b >= p.B) {
    d.q0 = min(max(p.qoff[p.B], 0), p.Tq);
    d.nq = p.Tq - d.q0;
    d.k0 = min(max(p.koff[p.B], 0), p.Tk);  // (behind the last key, so that nothing behind it is visited)
    d.nk = d.prefix = 0;
    return d;
  }
  d.q0 = min(max(p.qoff[b], 0), p.Tq);
  d.nq = min(max(p.qoff[b + 1], d.q0), p.Tq) - d.q0;
  d.k0 = min(max(p.koff[b], 0), p.Tk);
  d.nk = min(max(p.koff[b + 1], d.k0), p.Tk) - d.k0;
  d.prefix = p.prefix == nullptr ? 0 : min(max(p.prefix[b], 0), d.nk);
  return d;
}

// What query t of document d sees, as rows of the packed keys: [lo, end), and the
// prefix [p0, pend).  All four grow with t, across documents too.
struct Seen {
  int pos, lo, end, p0, pend;
};
__device__ __forceinline__ Seen seen_by(const Packed& p, const Doc& d, int t) {
  Seen s;
  const int pos = t - d.q0 + d.nk - d.nq;
  int hi = p.half >= 0 ? min(pos + p.half, d.nk - 1) : d.nk - 1;  // (both terms below 2^30)
  if (p.causal) hi = min(hi, pos);
  s.pos = d.k0 + pos;
  s.lo = d.k0 + (p.half >= 0 ? max(pos - p.half, 0) : 0);
  s.end = d.k0 + max(hi + 1, 0);
  s.p0 = d.k0;
  s.pend = d.k0 + d.prefix;
  return s;
}

static_assert(kBlockTokens == 128, "a block of tokens is G blocks of rows");

// ------------------------------------------------------------------ rows and tiles

__device__ __forceinline__ int by_g(const Packed& p, int r) { return p.G == 1 ? r : r / p.G; }
__device__ __forceinline__ int mod_g(const Packed& p, int r) { return p.G == 1 ? 0 : r % p.G; }

// The document and the first row in it of block slot `slot`, of blocks that take R
// rows of one document; false: none, the block has nothing to do.
// Up to 63 documents: lane b counts document b's blocks, and the slots are dealt
// out exactly (lane B stands for the rows behind the last document).  Else
// document b has the slots from off_b G / R + b on, rounded down, which leaves each
// enough of them; all 64 lanes probe at once for the last b that begins at or
// before the slot.
template <int R>
__device__ __forceinline__ bool slot_doc(const Packed& p, int64_t slot, int lane, Doc* d, int* r0) {
  if (p.B < 64) {
    Doc x{0, 0, 0, 0, 0};
    if (lane <= p.B) x = packed_doc(p, lane);
    const int cnt = (x.nq * p.G + R - 1) / R;
    int start = cnt;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(start, o, 64);
      if (lane >= o) start += up;
    }
    start -= cnt;
    const uint64_t hit = __ballot(slot >= start && slot < (int64_t)start + cnt);
    if (hit == 0) return false;
    const int b = __builtin_ctzll(hit);
    d->q0 = __builtin_amdgcn_readlane(x.q0, b);
    d->nq = __builtin_amdgcn_readlane(x.nq, b);
    d->k0 = __builtin_amdgcn_readlane(x.k0, b);
    d->nk = __builtin_amdgcn_readlane(x.nk, b);
    d->prefix = __builtin_amdgcn_readlane(x.prefix, b);
    *r0 = ((int)slot - __builtin_amdgcn_readlane(start, b)) * R;
    return true;
  }
  auto base = [&](int b) { return (int64_t)min(max(p.qoff[b], 0), p.Tq) * p.G / R + b; };
  int lo = 0, n = p.B + 1;
  while (n > 1) {
    const int step = (n + 63) >> 6, at = lane * step;
    const int cnt = __popcll(__ballot(at < n && base(lo + (at < n ? at : 0)) <= slot));
    lo += (cnt - 1) * step;
    n = min(step, n - (cnt - 1) * step);
  }
  *d = packed_doc(p, lo);
  const int64_t at = (slot - base(lo)) * R;
  *r0 = (int)at;
  return at < (int64_t)d->nq * p.G;
}

// The tiles of KT keys that some of a document's rows can see, from what the first
// and the last of them see: those of the prefix, then the run from the first row's
// first key to the last row's last.  bound: the end of both.
struct Tiles {
  int a0, na, b0, n, bound;
  template <int KT>
  __device__ __forceinline__ int at(int i) const { return i < na ? a0 + KT * i : b0 + KT * (i - na); }
};
template <int KT>
__device__ __forceinline__ Tiles tiles_of(const Seen& f, const Seen& l) {
  Tiles t;
  t.a0 = l.p0;
  t.na = (l.pend - l.p0 + KT - 1) / KT;
  t.b0 = max(f.lo, t.a0 + KT * t.na);
  t.bound = max(l.end, l.pend);
  t.n = t.na + (max(l.end - t.b0, 0) + KT - 1) / KT;
  return t;
}

// One lane's row, and what its wave's first and last rows see
struct Row : Seen {
  Seen f, l;
  float slope;
};
// 0: no row sees a key of the tile, 1: every row sees every key, 2: neither
template <int KT>
__device__ __forceinline__ int tile_class(const Row& w, int k0) {
  if ((k0 >= w.l.lo && k0 + KT <= w.f.end) || (k0 >= w.l.p0 && k0 + KT <= w.f.pend)) return 1;
  return (k0 >= w.l.end || k0 + KT <= w.f.lo) && (k0 >= w.l.pend || k0 + KT <= w.f.p0) ? 0 : 2;
}
// ones in the bits below n
__device__ __forceinline__ uint32_t bits_below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }
// Bit i: the row sees key k0 + i
__device__ __forceinline__ uint32_t seen_bits(const Seen& w, int k0) {
  return (bits_below(w.pend - k0) & ~bits_below(w.p0 - k0)) | (bits_below(w.end - k0) & ~bits_below(w.lo - k0));
}
// x where the bit of `seen` is set, else -inf (the bit sign-extended to a word: one
// extract and one bit-field insert a score)
__device__ __forceinline__ float seen_or(uint32_t seen, int bit, float x) {
  const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)seen, bit, 1);
  return __uint_as_float((__float_as_uint(x) & m) | (~m & 0xff800000u));
}

// Parts of a split run: per split and row (token * H + head) the unscaled output,
// the score its weights are relative to and their sum.
struct Parts {
  float* o;    // [splits][rows][64]
  float2* ml;  // [splits][rows]
  int tiles;   // of a split; the last one takes what is left
};

// ------------------------------------------------------------------ f16 / bf16 (D = 64)

// A wave's 32 rows (lane l holds row l % 32; the halves split its columns and its
// keys).  Scores are in base 2 once `mul` is applied: mul is 1 where a cap or a
// slope has made them so beforehand.
struct Wave {
  uint4v qf[4];   // columns 16 s + 8 lg .. of the query per MFMA step s
  float16v o[2];  // columns 32 d + 8 (r / 4) + 4 lg + r % 4
  float m, l;     // running maximum (before mul), the lane's sum of weights
};
// A capped score c2 tanh(c1 x / 2) is c2 - 2 c2 / (1 + 2^(c1 x)) (c1 in base 2), which
// cancels for scores that are small against the cap (off by 2e-7 c2): it is taken past
// 0.75 cap alone, score by score, since a tile may hold hidden scores of any size beside
// small ones.  Within 0.75 cap the odd polynomial of degree 9 through tanh's Chebyshev
// points there, off by 3.6e-7 at most, in y = score / cap, whose square is in range
// whatever the products.  Where every score of a tile is within 0.75 cap, the same in the
// product itself, if its squares and the coefficients are normal numbers: 6 instructions
// instead of an exponential and a reciprocal at a lower rate (chunks of 1000 queries over
// up to 8192 keys: 164 -> 153 us).  Within 0.25 cap that of degree 5, off by 1e-7 at most,
// does, whose last product is one with the subtraction of the maximum (153 -> 135 us).
__device__ __forceinline__ float odd_polynomial(const float (&c)[5], float u, float x) {
  float r = fmaf(u, c[4], c[3]);
#pragma unroll
  for (int i = 2; i >= 0; i--) r = fmaf(u, r, c[i]);
  return x * r;
}
__device__ __forceinline__ float capped_near(const Score& s, float x) { return odd_polynomial(s.poly, x * x, x); }
__device__ __forceinline__ float capped(const Score& s, float x) {
  const float y = x * s.g;
  const float far = fmaf(-2.f * s.c2, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * s.c1)), s.c2);
  return fabsf(x) <= s.far ? odd_polynomial(s.odd, y * y, x) : far;
}
template <bool CAP, bool BIAS>
__device__ __forceinline__ float score(const Score& s, float slope, int pos, int key, float x) {
  if constexpr (CAP) x = capped(s, x);
  else if constexpr (BIAS) x *= s.c1;
  if constexpr (BIAS) x = fmaf(-slope, fabsf((float)(pos - key)), x);
  return x;
}
// The factor of x in its capped score, |x| <= tiny_near
__device__ __forceinline__ float tiny_factor(const Score& s, float x) {
  const float u = x * x;
  return fmaf(u, fmaf(u, s.tiny[2], s.tiny[1]), s.tiny[0]);
}
static Score score_of(float scale, float cap, bool bias) {
  Score s{};
  // (scale 0: the smallest number, since 0 * -inf would not be a maximum; no product gives it
  // a score that counts.  Finite times log2 e.)
  constexpr float kTiny = 0x1p-149f;
  const float sl = fminf(fmaxf(fabsf(scale), kTiny), 0x1p126f);
  const bool capped = cap > 0.f;
  s.mul = capped || bias ? 1.f : sl * kLog2e;
  s.c1 = sl * kLog2e;
  s.c2 = cap * kLog2e;
  s.flip = scale < 0.f ? 0x80008000u : 0u;
  if (!capped) return s;
  const double c[5] = {0.99999942, -0.33328192, 0.13258462, -0.05004161, 0.01291665};  // tanh(y) / y in y^2 on [0, 0.75^2]
  const double c3[3] = {0.9999996, -0.33321897, 0.12841434};                           // on [0, 0.25^2]
  // (finite, so that 0 * c1 is 0 under the smallest caps, and inf * c1 inf under the largest)
  const double g = std::min((double)sl / cap, (double)FLT_MAX / 4);
  s.g = (float)g;
  s.c1 = fmaxf((float)(2 * g * kLog2e), kTiny);
  double f = sl * kLog2e;
  bool normal = true;
  for (int i = 0; i < 5; i++, f *= g * g) {
    s.odd[i] = (float)(sl * kLog2e * c[i]);
    s.poly[i] = (float)(f * c[i]);
    if (i < 3) s.tiny[i] = (float)(f * c3[i]);
    normal = normal && std::isnormal(s.poly[i]);
    if (i == 2) s.tiny_near = normal ? 1.f : -1.f;
  }
  // (finite: an infinite product takes the exponential)
  s.far = (float)std::min(0.75 / g, (double)FLT_MAX);
  s.near = normal && s.far < 0x1p63f ? s.far : -1.f;
  s.tiny_near = s.tiny_near > 0.f && s.far < 0x1p63f ? (float)(0.25 / g) : -1.f;
  return s;
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

// sum + both halves of a packed pair, in f32
template <bool BF16>
__device__ __forceinline__ float add_pair(uint32_t p, float sum) {
  if constexpr (BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum,
                                           false);
  } else {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, p), __builtin_bit_cast(half2v, 0x3c003c00u), sum, false);
  }
}

// One tile of 64 keys in LDS, in three parts: the products of queries and keys,
template <bool BF16>
__device__ __forceinline__ void wave_products(const Wave& w, const Frag32& f, const uint16_t* Kc, float16v (&st)[2]) {
#pragma unroll
  for (int kb = 0; kb < 2; kb++) {
    uint4v kf[4];
#pragma unroll
    for (int s = 0; s < 4; s++) kf[s] = *(const uint4v*)(Kc + f.ka[s] + kb * 2048);
#pragma unroll
    for (int r = 0; r < 16; r++) st[kb][r] = 0.f;
#pragma unroll
    for (int s = 0; s < 4; s++) st[kb] = mfma32x16<BF16>(kf[s], w.qf[s], st[kb]);
  }
}
__device__ __forceinline__ float max_of(const float16v (&st)[2]) {
  float mx = -INFINITY;
#pragma unroll
  for (int kb = 0; kb < 2; kb++)
#pragma unroll
    for (int r = 0; r < 16; r++) mx = fmaxf(mx, st[kb][r]);
  return mx;
}
// their weights (cap, slope, mask if `mixed`, online softmax).  Weights are relative to
// w.m, which follows the maximum once it is left behind by a factor of 2^8 for some row
// of the wave: up to there they fit the 16-bit types as well, and O and the sum need no
// rescaling.  `top`: no less than the lane's scores; `mx`: their maximum.
template <class Max>
__device__ __forceinline__ void follow_maximum(Wave& w, const Score& sc, float top, Max mx) {
  if (__all(top * sc.mul <= fmaf(w.m, sc.mul, 8.f))) return;
  const float mnew = fmaxf(w.m, max_xor32(mx())), mc = mnew == -INFINITY ? 0.f : mnew * sc.mul;
  const float alpha = __builtin_amdgcn_exp2f(w.m * sc.mul - mc);
  w.m = mnew;
  w.l *= alpha;
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int r = 0; r < 16; r++) w.o[e][r] *= alpha;
}
// Weights are rounded to the 16-bit type for the second product, as MFMA takes them, and
// their sum is of the rounded ones (one dot product a pair).  exponent(x, mc): a score's
// distance to mc in base 2
template <bool BF16, class Exponent>
__device__ __forceinline__ void wave_exps(Wave& w, const float16v (&st)[2], const Score& sc, uint4v (&pf)[4],
                                          Exponent exponent) {
  const float mc = w.m == -INFINITY ? 0.f : w.m * sc.mul;
#pragma unroll
  for (int t = 0; t < 4; t++) {
    uint32_t pk[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f(exponent(st[t >> 1][8 * (t & 1) + e], mc));
      const float p1 = __builtin_amdgcn_exp2f(exponent(st[t >> 1][8 * (t & 1) + e + 1], mc));
      pk[e >> 1] = pack2<BF16>(p0, p1);
      w.l = add_pair<BF16>(pk[e >> 1], w.l);
    }
    pf[t] = uint4v{pk[0], pk[1], pk[2], pk[3]};
  }
}
template <bool BF16, bool CAP, bool BIAS>
__device__ __forceinline__ void wave_weights(Wave& w, float16v (&st)[2], int k0, const Row& row, bool mixed,
                                             const Score& sc, int lg, uint4v (&pf)[4]) {
  if constexpr (CAP) {
    float far = 0.f;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 16; r++) far = fmaxf(far, fabsf(st[kb][r]));
    if (!BIAS && !mixed && __all(far <= sc.tiny_near)) {
      auto tiny = [&](float x) { return x * tiny_factor(sc, x); };
      follow_maximum(w, sc, tiny(far), [&] { return tiny(max_of(st)); });  // (the cap keeps the order)
      wave_exps<BF16>(w, st, sc, pf, [&](float x, float mc) { return fmaf(x, tiny_factor(sc, x), -mc); });
      return;
    }
    if (__all(far <= sc.near)) {
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int r = 0; r < 16; r++) st[kb][r] = capped_near(sc, st[kb][r]);
    } else {
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int r = 0; r < 16; r++) st[kb][r] = capped(sc, st[kb][r]);
    }
  }
  if constexpr (BIAS) {
    const float d0 = (float)(row.pos - k0 - 4 * lg);
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const float x = CAP ? st[kb][r] : st[kb][r] * sc.c1;
        st[kb][r] = fmaf(-row.slope, fabsf(d0 - (float)(32 * kb + 8 * (r >> 2) + (r & 3))), x);
      }
  }
  if (mixed) {
#pragma unroll
    for (int kb = 0; kb < 2; kb++) {
      const uint32_t seen = seen_bits(row, k0 + 32 * kb) >> (4 * lg);
#pragma unroll
      for (int r = 0; r < 16; r++) st[kb][r] = seen_or(seen, 8 * (r >> 2) + (r & 3), st[kb][r]);
    }
  }
  const float mx = max_of(st);
  follow_maximum(w, sc, mx, [&] { return mx; });
  wave_exps<BF16>(w, st, sc, pf, [&](float x, float mc) { return fmaf(x, sc.mul, -mc); });
}
// and O += weights . V.
template <bool BF16>
__device__ __forceinline__ void wave_values(Wave& w, const Frag32& f, const uint16_t* Vc, const uint4v (&pf)[4]) {
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
                                           const Row& row, const Tiles& ti, int i0, int i1, int step,
                                           const Score& sc, int lg) {
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int r = 0; r < 16; r++) w.o[e][r] = 0.f;
  w.m = -INFINITY;
  w.l = 0.f;
#pragma unroll 1
  for (int i = i0; i < i1; i += step) {
    const int k0 = ti.at<64>(i), k1 = min(k0 + 64, ti.bound);
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
      x = seen_bits(row, j) & 1u ? x : -INFINITY;
      const float mnew = fmaxf(w.m, x), mc = mnew == -INFINITY ? 0.f : mnew * sc.mul;
      const float alpha = __builtin_amdgcn_exp2f(w.m * sc.mul - mc), pr = __builtin_amdgcn_exp2f(fmaf(x, sc.mul, -mc));
      w.m = mnew;
      const float p16 = tof<BF16>(fromf<BF16>(pr));
      w.l = w.l * alpha + (lg == 0 ? p16 : 0.f);  // (the halves' sums are added up later)
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

// The output row of a row (a query and one of its G heads)
__device__ __forceinline__ int64_t row_index(const Packed& p, int t, int r, int hk) {
  return (int64_t)t * p.H + hk * p.G + mod_g(p, r);
}
// A lane's row among rows of one document, r of them from rw0 on.
__device__ __forceinline__ Row doc_row(const Packed& p, const Doc& d, int r, int rw0, int rows, int hk) {
  Row w;
  static_cast<Seen&>(w) = seen_by(p, d, d.q0 + by_g(p, r));
  w.f = seen_by(p, d, d.q0 + by_g(p, rw0));
  w.l = seen_by(p, d, d.q0 + by_g(p, min(rw0 + 31, rows - 1)));
  w.slope = p.slopes == nullptr ? 0.f : p.slopes[hk * p.G + mod_g(p, r)];
  return w;
}

// 128 rows a block, four waves of 32, K and V tiles in a two-buffer LDS ring with
// one barrier per tile.  The plan's table of blocks of 128 tokens says where each
// works, so that its set-up is two scalar loads deep (the entry, then its document's
// offsets): a search among the documents took 2 us a block.
// 32 documents of up to 512 tokens, 12 heads, f16: 29 us; one of 4096, 24 heads: 162 us,
// 636 TFLOP/s.  Bound by its VALU (800 cycles a wave and tile: exponentials half) and
// MFMAs (512), which lie under one another for a fifth: a block alone takes 1.04 us a
// tile, three on a CU 0.84 each.
constexpr int kRowsB = 128;
template <bool BF16, bool CAP, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) void packed_attn_rows(Packed p, Parts part,
                                                                                                int splits) {
  __shared__ __attribute__((aligned(16))) uint16_t Ks[2][64 * 64];
  __shared__ __attribute__((aligned(16))) uint16_t Vs[2][64 * 64];
  const int tid = threadIdx.x, lane = tid & 63, lg = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hk = p.H / p.G;
  int slot = blockIdx.x / Hk;
  const int hk = blockIdx.x - slot * Hk;
  if (p.causal) slot = (int)(gridDim.x / Hk) - 1 - slot;  // a document's last rows, which see the most, first
  const int entry = by_g(p, slot), b = p.blocks[2 * entry];
  if (b < 0) return;  // (the whole block, here and below)
  const Doc d = packed_doc(p, b);
  const int t0 = min(max(p.blocks[2 * entry + 1], d.q0), d.q0 + d.nq), rows = min(d.q0 + d.nq - t0, kBlockTokens) * p.G;
  const int r0 = mod_g(p, slot) * kRowsB, rw0 = r0 + 32 * wave;
  if (r0 >= rows) return;
  const int r = rw0 + (lane & 31), rc = min(r, rows - 1), t = t0 + by_g(p, rc);
  const Score& sc = p.sc;
  Wave w;
  wave_init(w, sc, (const uint16_t*)p.Q + t * p.qs[0] + (hk * p.G + mod_g(p, rc)) * p.qs[1], lg);
  auto seen = [&](int q) { return seen_by(p, d, t0 + by_g(p, min(q, rows - 1))); };
  const Tiles ti = tiles_of<64>(seen(r0), seen(r0 + kRowsB - 1));
  const int s = blockIdx.y, i0 = min(s * part.tiles, ti.n), i1 = s + 1 < splits ? min(i0 + part.tiles, ti.n) : ti.n;
  if (splits > 1 && i0 >= i1) {  // nothing left for this split
    if (r < rows && lg == 0) part.ml[(int64_t)s * p.Tq * p.H + row_index(p, t, r, hk)] = float2{-INFINITY, 0.f};
    return;
  }
  const uint16_t* Kb = (const uint16_t*)p.K + hk * p.ks[1];
  const uint16_t* Vb = (const uint16_t*)p.V + hk * p.vs[1];
  auto fetch = [&](int i, int bf) __attribute__((always_inline)) {
    const int k0 = ti.at<64>(i);
#pragma unroll
    for (int q = 0; q < 2; q++) dma_piece(Vb, p.vs[0], k0, wave * 2 + q, ti.bound, Vs[bf], lane);
#pragma unroll
    for (int q = 0; q < 2; q++) dma_piece(Kb, p.ks[0], k0, wave * 2 + q, ti.bound, Ks[bf], lane);
  };
  if (i0 < i1) fetch(i0, 0);
  Row row;
  static_cast<Seen&>(row) = seen_by(p, d, t);
  row.f = seen(rw0);
  row.l = seen(rw0 + 31);
  row.slope = p.slopes == nullptr ? 0.f : p.slopes[hk * p.G + mod_g(p, rc)] * kLog2e;
  const Frag32 f = frag32(lane);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int at = 0;
  for (int i = i0; i < i1; i++) {
    // the next tile into the other buffer (free since the last barrier)
    if (i + 1 < i1) fetch(i + 1, at ^ 1);
    const int k0 = ti.at<64>(i), cl = rw0 < rows ? tile_class<64>(row, k0) : 0;
    if (cl != 0) {
      float16v st[2];
      uint4v pf[4];
      wave_products<BF16>(w, f, Ks[at], st);
      wave_weights<BF16, CAP, BIAS>(w, st, k0, row, cl == 2, sc, lg, pf);
      wave_values<BF16>(w, f, Vs[at], pf);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    at ^= 1;
    __syncthreads();
  }
  if (!wave_finite(w)) w = wave_again<BF16, CAP, BIAS>(w, Kb, p.ks[0], Vb, p.vs[0], row, ti, i0, i1, 1, sc, lg);
  const float lt = sum_xor32(w.l);
  if (r >= rows) return;
  const int64_t ri = row_index(p, t, r, hk);
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
// same rows and take its tiles in turn, each through a K and a V tile of its own in
// LDS with no barrier; a tile's K is requested once the last one's products are
// made, its V once that one's values are, so a wave has 8 to 16 KB on their way
// whatever it does, and two blocks share a CU.  Then the waves' parts are joined.
// Bound by reading K and V once (a token each of 48 documents of up to 4096, 4 key heads:
// 36 us, 3.2 TB/s, the longest documents' blocks at the end).
constexpr int kRowsF = 32, kFewLds = 4 * 2 * 64 * 64 * 2;
template <bool BF16, bool CAP, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void packed_attn_few(Packed p, Parts part,
                                                                                               int splits) {
  extern __shared__ __attribute__((aligned(16))) uint16_t ring[];
  __shared__ float part_m[4][kRowsF], part_l[4][kRowsF];
  const int tid = threadIdx.x, lane = tid & 63, lg = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hk = p.H / p.G, hk = blockIdx.x % Hk;
  const int64_t slot = blockIdx.x / Hk;
  Doc d;
  int r0;
  if (!slot_doc<kRowsF>(p, slot, lane, &d, &r0)) return;  // (the whole block)
  const int rows = d.nq * p.G, r = r0 + l32, rc = min(r, rows - 1);
  const Score& sc = p.sc;
  Row row = doc_row(p, d, rc, r0, rows, hk);
  row.slope *= kLog2e;
  const Tiles ti = tiles_of<64>(row.f, row.l);
  const int s = blockIdx.y, s0 = min(s * part.tiles, ti.n), i1 = s + 1 < splits ? min(s0 + part.tiles, ti.n) : ti.n;
  const int i0 = s0 + wave;
  if (splits > 1 && s0 >= i1) {  // nothing left for this split
    if (wave == 0 && r < rows && lg == 0)
      part.ml[(int64_t)s * p.Tq * p.H + row_index(p, d.q0 + by_g(p, r), r, hk)] = float2{-INFINITY, 0.f};
    return;
  }
  const uint16_t* Kb = (const uint16_t*)p.K + hk * p.ks[1];
  const uint16_t* Vb = (const uint16_t*)p.V + hk * p.vs[1];
  uint16_t *Kt = ring + wave * (2 * 64 * 64), *Vt = Kt + 64 * 64;
  auto fetch = [&](const uint16_t* base, int64_t stride, int i, uint16_t* tile) __attribute__((always_inline)) {
    // this wave's reads of the tile that was there are done
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int q = 0; q < 8; q++) dma_piece(base, stride, ti.at<64>(i), q, ti.bound, tile, lane);
  };
  Wave w;
  wave_init(w, sc, (const uint16_t*)p.Q + (d.q0 + by_g(p, rc)) * p.qs[0] + (hk * p.G + mod_g(p, rc)) * p.qs[1], lg);
  const Frag32 f = frag32(lane);
  if (i0 < i1) {
    fetch(Kb, p.ks[0], i0, Kt);
    fetch(Vb, p.vs[0], i0, Vt);
  }
  for (int i = i0; i < i1; i += 4) {
    const int k0 = ti.at<64>(i);
    const bool more = i + 4 < i1;
    float16v st[2];
    uint4v pf[4];
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // all but the 8 loads of V
    wave_products<BF16>(w, f, Kt, st);
    if (more) fetch(Kb, p.ks[0], i + 4, Kt);
    wave_weights<BF16, CAP, BIAS>(w, st, k0, row, tile_class<64>(row, k0) != 1, sc, lg, pf);
    if (more) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // all but the next K
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    wave_values<BF16>(w, f, Vt, pf);
    if (more) fetch(Vb, p.vs[0], i + 4, Vt);
  }
  if (!wave_finite(w)) w = wave_again<BF16, CAP, BIAS>(w, Kb, p.ks[0], Vb, p.vs[0], row, ti, i0, i1, 4, sc, lg);
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
  const int64_t ri = row_index(p, d.q0 + by_g(p, r), r, hk), pr = (int64_t)s * p.Tq * p.H + ri;
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
// (3 documents of up to 333 tokens, 12 heads, window: 17 us, a chain of the offsets, Q and
// K, two rounds of tiles and the join; eight waves a block: 21.6.)
constexpr int kRows32 = 32, kKeys32 = 32;
// exp of a difference: its rounding before the exponential is below 2^-23 |x|.
__device__ __forceinline__ float exp32(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
// A tile's scores into weights (scale, cap, slope, mask, online softmax); maximum,
// sum and output follow.
template <bool CAP, bool BIAS>
__device__ __forceinline__ void weigh32(const Packed& p, const Row& row, int k0, int cl, int lg, float16v& st,
                                        float16v (&o)[2], float& m, float& l) {
  float mx = -INFINITY;
  const float icap = 1.f / p.cap;  // (read with a cap alone)
  const uint32_t seen = cl != 1 ? seen_bits(row, k0) >> (4 * lg) : ~0u;
#pragma unroll
  for (int q = 0; q < 16; q++) {
    const int key = k0 + 8 * (q >> 2) + 4 * lg + (q & 3);
    float x = st[q] * p.scale;
    if constexpr (CAP) x = p.cap * tanhf(x * icap);
    if constexpr (BIAS) x = fmaf(-row.slope, fabsf((float)(row.pos - key)), x);
    if (cl != 1) x = seen_or(seen, 8 * (q >> 2) + (q & 3), x);
    st[q] = x;
    mx = fmaxf(mx, x);
  }
  mx = max_xor32(mx);
  const float mnew = fmaxf(m, mx), mc = mnew == -INFINITY ? 0.f : mnew, alpha = exp32(m - mc);
  m = mnew;
  float sum = 0.f;
#pragma unroll
  for (int q = 0; q < 16; q++) {
    st[q] = exp32(st[q] - mc);
    sum += st[q];
  }
  l = l * alpha + sum;
  if (!__all(alpha == 1.0f)) {
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int q = 0; q < 16; q++) o[e][q] *= alpha;
  }
}
// O += weights . V of one tile, key by key, from memory.
__device__ __forceinline__ void add_values32(const float* Vb, int64_t vstride, int k0, int lg, int l32, const float16v& st,
                                             float* kb, float16v (&o)[2]) {
#pragma unroll
  for (int q = 0; q < 16; q++) kb[(8 * (q >> 2) + 4 * lg + (q & 3)) * 32 + l32] = st[q];
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll 1
  for (int j = 0; j < kKeys32; j++) {
    const float w = kb[j * 32 + l32];
    if (w == 0.f) continue;  // keys past the document among them
    const float* vp = Vb + (k0 + j) * vstride + 4 * lg;
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int q = 0; q < 16; q++) o[e][q] = fmaf(w, vp[32 * e + 8 * (q >> 2) + (q & 3)], o[e][q]);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <bool CAP, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void packed_attn_f32(Packed p, Parts part,
                                                                                               int splits) {
  __shared__ __attribute__((aligned(16))) float buf[4][kKeys32 * 64];  // K tiles; the waves' outputs at the end
  __shared__ float part_m[4][kRows32], part_l[4][kRows32];
  const int tid = threadIdx.x, lane = tid & 63, lg = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hk = p.H / p.G, hk = blockIdx.x % Hk;
  const int64_t slot = blockIdx.x / Hk;
  Doc d;
  int r0;
  if (!slot_doc<kRows32>(p, slot, lane, &d, &r0)) return;  // (the whole block)
  const int rows = d.nq * p.G, r = r0 + l32, rc = min(r, rows - 1);
  const Row row = doc_row(p, d, rc, r0, rows, hk);
  const Tiles ti = tiles_of<kKeys32>(row.f, row.l);
  const int s = blockIdx.y, s0 = min(s * part.tiles, ti.n), i1 = s + 1 < splits ? min(s0 + part.tiles, ti.n) : ti.n;
  const int i0 = s0 + wave;
  if (splits > 1 && s0 >= i1) {  // nothing left for this split
    if (wave == 0 && r < rows && lg == 0)
      part.ml[(int64_t)s * p.Tq * p.H + row_index(p, d.q0 + by_g(p, r), r, hk)] = float2{-INFINITY, 0.f};
    return;
  }
  const float* Kb = (const float*)p.K + hk * p.ks[1];
  const float* Vb = (const float*)p.V + hk * p.vs[1];

  // element e of qf[i] is column 8 i + 4 lg + e, the columns its half supplies to
  // MFMA steps e of chunk pair i
  float4v qf[8];
  {
    const float* qp = (const float*)p.Q + (d.q0 + by_g(p, rc)) * p.qs[0] + (hk * p.G + mod_g(p, rc)) * p.qs[1] + 4 * lg;
#pragma unroll
    for (int i = 0; i < 8; i++) qf[i] = *(const float4v*)(qp + 8 * i);
  }
  // K tile: 8 lanes a row, chunk c of row r at c ^ (r & 15): a 16-lane pass of the
  // fragment reads (16 rows, one chunk) covers all 64 banks.  Keys past the
  // rows' last one repeat it: their scores are hidden.
  const int kr = lane >> 3, c8 = lane & 7;
  float4v klo[4], khi[4];
  auto load_k = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float* kp = Kb + min(k0 + i * 8 + kr, ti.bound - 1) * p.ks[0] + 4 * c8;
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
  if (i0 < i1) load_k(ti.at<kKeys32>(i0));
  for (int i = i0; i < i1; i += 4) {
    const int k0 = ti.at<kKeys32>(i), cl = tile_class<kKeys32>(row, k0);
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
      const float* vp = Vb + min(k0 + 8 * (q >> 2) + 4 * lg + (q & 3), ti.bound - 1) * p.vs[0] + l32;
      v[0][q] = vp[0];
      v[1][q] = vp[32];
    }
    if (i + 4 < i1) load_k(ti.at<kKeys32>(i + 4));
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
    weigh32<CAP, BIAS>(p, row, k0, cl, lg, st, o, m, l);
    // A non-finite V must not reach a row whose weight for that key is 0, as 0 *
    // inf in the product would: such a tile is added key by key, zero weights
    // skipped.
    float fin = 0.f;
#pragma unroll
    for (int q = 0; q < 16; q++) fin += v[0][q] * 0.f + v[1][q] * 0.f;
    if (__any(fin != 0.f)) {  // 0 * finite = 0, 0 * (inf or NaN) = NaN
      add_values32(Vb, p.vs[0], k0, lg, l32, st, kb, o);
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
  const int64_t ri = row_index(p, d.q0 + by_g(p, r), r, hk), pr = (int64_t)s * p.Tq * p.H + ri;
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

// 128 rows a block, four waves of 32 that share K and V tiles of 32 keys in a
// two-buffer LDS ring, for enough blocks to fill the GPU: a quarter of the reads of K
// and V and of the blocks' set-ups, and no joining (2 documents of up to 2000, 16 heads:
// 258 us, of 32 rows 281; the f32 matrix rate allows 166).
__device__ __forceinline__ void dma_piece32(const float* base, int64_t stride, int k0, int piece, int bound, float* dst,
                                            int lane, bool keys) {
  const uint64_t a = (uint64_t)(base + (int64_t)k0 * stride);
  const uint4v rs = {(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a),
                     (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu), 0x80000000u, 0x00020000u};
  // 4 rows of 16 chunks; chunk c of K's row r at c ^ (r & 15) as above, of V's at c ^ 8
  // in every second group of 4 rows, so that the lane halves' rows meet other banks
  const int r = piece * 4 + (lane >> 4), c = (lane & 15) ^ (keys ? r & 15 : (r & 4) * 2);
  const uint32_t off = __umul24(r, (uint32_t)stride) * 4u + (c << 4);
  const uint32_t lds = (uint32_t)__builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) float*)(dst + piece * 256));
  buffer_lds16(rs, k0 + r < bound ? off : 0xfffffff0u, lds);
}

template <bool CAP, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void packed_attn_f32_rows(Packed p, Parts part,
                                                                                                    int splits) {
  __shared__ __attribute__((aligned(16))) float Ks[2][kKeys32 * 64];
  __shared__ __attribute__((aligned(16))) float Vs[2][kKeys32 * 64];
  __shared__ float weights[4][kKeys32 * 32];
  const int tid = threadIdx.x, lane = tid & 63, lg = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hk = p.H / p.G;
  int slot = blockIdx.x / Hk;
  const int hk = blockIdx.x - slot * Hk;
  if (p.causal) slot = (int)(gridDim.x / Hk) - 1 - slot;
  const int entry = by_g(p, slot), b = p.blocks[2 * entry];
  if (b < 0) return;  // (the whole block, here and below)
  const Doc d = packed_doc(p, b);
  const int t0 = min(max(p.blocks[2 * entry + 1], d.q0), d.q0 + d.nq), rows = min(d.q0 + d.nq - t0, kBlockTokens) * p.G;
  const int r0 = mod_g(p, slot) * kRowsB, rw0 = r0 + 32 * wave;
  if (r0 >= rows) return;
  const int r = rw0 + l32, rc = min(r, rows - 1), t = t0 + by_g(p, rc);
  auto seen = [&](int q) { return seen_by(p, d, t0 + by_g(p, min(q, rows - 1))); };
  const Tiles ti = tiles_of<kKeys32>(seen(r0), seen(r0 + kRowsB - 1));
  const int s = blockIdx.y, i0 = min(s * part.tiles, ti.n), i1 = s + 1 < splits ? min(i0 + part.tiles, ti.n) : ti.n;
  if (splits > 1 && i0 >= i1) {  // nothing left for this split
    if (r < rows && lg == 0) part.ml[(int64_t)s * p.Tq * p.H + row_index(p, t, r, hk)] = float2{-INFINITY, 0.f};
    return;
  }
  const float* Kb = (const float*)p.K + hk * p.ks[1];
  const float* Vb = (const float*)p.V + hk * p.vs[1];
  auto fetch = [&](int i, int bf) __attribute__((always_inline)) {
    const int k0 = ti.at<kKeys32>(i);
#pragma unroll
    for (int q = 0; q < 2; q++) dma_piece32(Kb, p.ks[0], k0, wave * 2 + q, ti.bound, Ks[bf], lane, true);
#pragma unroll
    for (int q = 0; q < 2; q++) dma_piece32(Vb, p.vs[0], k0, wave * 2 + q, ti.bound, Vs[bf], lane, false);
  };
  if (i0 < i1) fetch(i0, 0);
  float4v qf[8];
  {
    const float* qp = (const float*)p.Q + t * p.qs[0] + (hk * p.G + mod_g(p, rc)) * p.qs[1] + 4 * lg;
#pragma unroll
    for (int i = 0; i < 8; i++) qf[i] = *(const float4v*)(qp + 8 * i);
  }
  Row row;
  static_cast<Seen&>(row) = seen_by(p, d, t);
  row.f = seen(rw0);
  row.l = seen(rw0 + 31);
  row.slope = p.slopes == nullptr ? 0.f : p.slopes[hk * p.G + mod_g(p, rc)];
  float16v o[2];
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[e][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int at = 0;
  for (int i = i0; i < i1; i++) {
    if (i + 1 < i1) fetch(i + 1, at ^ 1);
    const int k0 = ti.at<kKeys32>(i), cl = rw0 < rows ? tile_class<kKeys32>(row, k0) : 0;
    if (cl != 0) {
      const float* kt = Ks[at] + l32 * 64;
      float16v st;
#pragma unroll
      for (int q = 0; q < 16; q++) st[q] = 0.f;
#pragma unroll
      for (int q = 0; q < 8; q++) {
        const float4v kf = *(const float4v*)(kt + (((2 * q + lg) ^ (l32 & 15)) << 2));
#pragma unroll
        for (int e = 0; e < 4; e++) st = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], qf[q][e], st, 0, 0, 0);
      }
      weigh32<CAP, BIAS>(p, row, k0, cl, lg, st, o, m, l);
      // (row key, column half e ^ lg: the swizzle)
      const float* vt = Vs[at] + 4 * lg * 64 + l32;
      float v[2][16], fin = 0.f;
#pragma unroll
      for (int q = 0; q < 16; q++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          v[e][q] = vt[(8 * (q >> 2) + (q & 3)) * 64 + 32 * (e ^ lg)];
          fin = fmaf(v[e][q], 0.f, fin);
        }
      if (__any(fin != 0.f)) {
        add_values32(Vb, p.vs[0], k0, lg, l32, st, weights[wave], o);
      } else {
#pragma unroll
        for (int q = 0; q < 16; q++)
#pragma unroll
          for (int e = 0; e < 2; e++) o[e] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[e][q], st[q], o[e], 0, 0, 0);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    at ^= 1;
    __syncthreads();
  }
  const float lt = sum_xor32(l);
  if (r >= rows) return;
  const float inv = splits > 1 ? 1.f : lt == 0.f ? 0.f : 1.0f / lt;
  const int64_t ri = row_index(p, t, r, hk), pr = (int64_t)s * p.Tq * p.H + ri;
  if (splits > 1 && lg == 0) part.ml[pr] = float2{m, lt};
  float* op = (splits > 1 ? part.o + pr * 64 : (float*)p.O + ri * 64) + 4 * lg;
#pragma unroll
  for (int e = 0; e < 2; e++)
#pragma unroll
    for (int j = 0; j < 4; j++)
      *(float4v*)(op + 32 * e + 8 * j) =
          float4v{o[e][4 * j] * inv, o[e][4 * j + 1] * inv, o[e][4 * j + 2] * inv, o[e][4 * j + 3] * inv};
}

// Joins the parts of split runs: 16 lanes a row, four columns a lane.  E2: scores in
// base 2 (the 16-bit kernels), else natural.
template <bool E2>
__global__ __launch_bounds__(256) void packed_attn_join(int dt, Parts part, int splits, int64_t rows,
                                                        void* __restrict__ O) {
  const int c = (threadIdx.x & 15) * 4;
  const int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (r >= rows) return;
  float m = -INFINITY;
  for (int s = 0; s < splits; s++) m = fmaxf(m, part.ml[s * rows + r].x);
  const float mc = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4v o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; s++) {
    const float2 ml = part.ml[s * rows + r];
    const float w = E2 ? __builtin_amdgcn_exp2f(ml.x - mc) : expf(ml.x - mc);
    l = fmaf(ml.y, w, l);
    if (w == 0.f) continue;  // (a split without tiles has written no output)
    const float4v v = *(const float4v*)(part.o + (s * rows + r) * 64 + c);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = fmaf(v[e], w, o[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (dt == HB_F32) {
    *(float4v*)((float*)O + r * 64 + c) = float4v{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  } else {
    uint2v x;
    if (dt == HB_BF16) x = uint2v{pack2<true>(o[0] * inv, o[1] * inv), pack2<true>(o[2] * inv, o[3] * inv)};
    else x = uint2v{pack2<false>(o[0] * inv, o[1] * inv), pack2<false>(o[2] * inv, o[3] * inv)};
    *(uint2v*)((uint16_t*)O + r * 64 + c) = x;
  }
}

// ------------------------------------------------------------------ any type

// One wave per query and head: 64 keys at a time, a score per lane, then the
// lanes share out the columns of the output.
constexpr int kAnyCols = 8;  // columns per lane: D <= 512
__global__ __launch_bounds__(64) void packed_attn_any(Packed p, int dt) {
  extern __shared__ float sh[];  // [D] query, [64] weights
  float* w = sh + p.D;
  const int lane = threadIdx.x, h = blockIdx.y, D = p.D;
  for (int64_t t64 = blockIdx.x; t64 < p.Tq; t64 += gridDim.x) {
    const int t = (int)t64;
    __syncthreads();  // the last query and weights are used up
    const uint32_t b = (uint32_t)p.doc[t];
    const Seen d = seen_by(p, packed_doc(p, b < (uint32_t)p.B ? (int)b : p.B), t);
    for (int c = lane; c < D; c += 64) sh[c] = load_f(p.Q, t * p.qs[0] + h * p.qs[1] + c * p.qs[2], dt);
    __syncthreads();
    const float slope = p.slopes == nullptr ? 0.f : p.slopes[h];
    float o[kAnyCols] = {}, m = -INFINITY, l = 0.f;
    const int64_t kh = (h / p.G) * p.ks[1], vh = (h / p.G) * p.vs[1];
    const int bound = max(d.end, d.pend);
    for (int j0 = d.p0; j0 < bound; j0 += 64) {
      // (the same in every lane: nothing of these keys is visible)
      if (j0 >= d.pend && (j0 >= d.end || j0 + 64 <= d.lo)) continue;
      const int j = j0 + lane;
      const bool seen = j < d.pend || (j >= d.lo && j < d.end);
      float x = -INFINITY;
      if (seen) {
        const int64_t row = (int64_t)j * p.ks[0] + kh;
        float a = 0.f;
        for (int c = 0; c < D; c++) a = fmaf(sh[c], load_f(p.K, row + c * p.ks[2], dt), a);
        x = a * p.scale;
        if (p.cap > 0.f) x = p.cap * tanhf(x / p.cap);
        x -= slope * fabsf((float)(d.pos - j));
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
        for (int k = 0; k < 64 && j0 + k < bound; k++)
          if (w[k] != 0.f) a = fmaf(w[k], load_f(p.V, (int64_t)(j0 + k) * p.vs[0] + col, dt), a);
        o[i] = a;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int i = 0; i < kAnyCols && i * 64 + lane < D; i++)
      store_f(p.O, ((int64_t)t * p.H + h) * D + i * 64 + lane, dt, o[i] * inv);
  }
}

// ------------------------------------------------------------------ dispatch

// The MFMA kernels' conditions: D = 64, unit column strides, 16-byte aligned rows
// (`per` elements), K / V row strides that 32-bit offsets within a tile reach, and fewer
// than 2^32 threads in their grids.
static bool packed_takes_mfma(const Packed& p, int per) {
  auto rows16 = [&](const void* t, const int64_t* s) {
    return (uintptr_t)t % 16 == 0 && s[2] == 1 && s[0] % per == 0 && s[1] % per == 0;
  };
  auto near = [](int64_t s) { return s >= 0 && s < (1 << 23); };
  const int64_t blocks = std::max((int64_t)p.Tq * p.G / 32 + p.B + 1, (int64_t)p.nblocks * p.G) * (p.H / p.G);
  return p.D == 64 && (int64_t)p.Tq * p.G < (1ll << 30) && blocks < (1ll << 24) && rows16(p.Q, p.qs) && rows16(p.K, p.ks) && rows16(p.V, p.vs) && near(p.ks[0]) && near(p.vs[0]) &&
         (uintptr_t)p.O % 16 == 0;
}

static void packed_any(uintptr_t ctx, int dt, const Packed& p) {
  packed_attn_any<<<dim3(capped_grid(p.Tq, 64), (unsigned)p.H), 64, (size_t)(p.D + 64) * 4, stream_of(ctx)>>>(p, dt);
}

template <class K>
static void packed_launch(uintptr_t ctx, K kern, int lds, int64_t blocks, const Packed& p, int splits, const Parts& part) {
  const int64_t grid = blocks * (p.H / p.G);
  HB_REQUIRE(grid < (1ll << 24), "hb_sdpa_packed: too many rows and heads");  // (packed_takes_mfma)
  kern<<<dim3((unsigned)grid, (unsigned)splits), 256, (size_t)lds, stream_of(ctx)>>>(p, part, splits);
}

static void packed_mfma(uintptr_t ctx, int dt, const Packed& p) {
  const int64_t rows = (int64_t)p.Tq * p.G;
  const bool f32 = dt == HB_F32;
  const int Hk = p.H / p.G, cus = cu_count(ctx);
  // Blocks of 32 rows where documents have few, and for f32 where those of 128 would
  // not go round the CUs (12 heads, 8 documents of up to 400 tokens: 35 us, of 128 rows
  // 42; 16 heads, 2 of up to 2000, 288 blocks: 281 and 258; 35 of up to 481, windows
  // with a cap: 143 and 100).
  const bool few = rows <= 64 * (int64_t)p.B ||
                   (f32 && std::max<int64_t>((rows + kRowsB - 1) / kRowsB, p.B) * Hk <= cus);
  const int per = few ? kRowsF : kRowsB;
  // An average document's tiles, and the blocks there are
  const int tile = f32 ? kKeys32 : 64;
  int64_t keys = p.B ? p.Tk / p.B : 0;
  if (p.half >= 0) keys = std::min<int64_t>(keys, 2 * (int64_t)p.half + per / p.G + tile);
  const int64_t tiles = keys / tile, blocks = std::max<int64_t>((rows + per - 1) / per, p.B) * Hk;
  // A run is split where the blocks would leave the GPU short of work: into pieces
  // of so many tiles that there are `want` of them, at least `least` each, since fewer do
  // not pay for writing and joining the parts, and twice as many as an average document
  // has (the last piece takes what is left of a longer one).
  // 128-row blocks: 7 documents of up to 1286 tokens, 16 heads, 47 us in pieces of 8
  // tiles, 39 whole.  32-row blocks, whose waves share out the tiles anyway: a token each
  // of 48 documents of up to 4096, 192 blocks, 40.5 in 6 pieces, 36.5 whole; 8 such
  // documents, 32 blocks, 24.9 whole, 20.2 in 3; 16 tokens each of 16, 128 blocks, 25.9
  // whole, 32.7 in 6.  f32, whose tiles take longer: a token each of 11 of up to 1605, 16
  // heads, 46.7 whole, 37.8 in 4 pieces, 47.2 in 7.
  const int64_t want = f32 && few ? 2 * (int64_t)cus : few ? cus / 2 : 4 * (int64_t)cus;
  const int64_t least = f32 && few ? 16 : few ? 32 : 24;
  Parts part{nullptr, nullptr, (int)std::max<int64_t>(least, blocks * tiles / want)};
  int splits = (int)std::min<int64_t>(32, (2 * tiles + part.tiles - 1) / part.tiles);
  if (blocks >= want || part.tiles >= tiles) splits = 1;
  CallScratch held(ctx);
  const int64_t all = (int64_t)p.Tq * p.H;
  if (splits > 1) {
    if (held.take((size_t)(splits * all * (64 * 4 + 8)))) {
      part.o = (float*)held.p;
      part.ml = (float2*)(part.o + splits * all * 64);
    } else {
      splits = 1;  // no memory for the parts: unsplit
    }
  }
  static_assert(kRowsF == kRows32, "slots of both");
  const int64_t slots = rows / kRowsF + p.B + 1;  // enough for every document's last, partly filled block
  auto go = [&](auto cap, auto bias) {
    constexpr bool CAP = decltype(cap)::value, BIAS = decltype(bias)::value;
    auto half = [&](auto bf) {
      constexpr bool BF = decltype(bf)::value;
      if (few) {
        // (with its static LDS past the 64 KB that a launch has without the attribute)
        static std::atomic<uint64_t> attr{0};
        const auto kern = packed_attn_few<BF, CAP, BIAS>;
        once_per_device(attr, [&] {
          HB_CHECK_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, kFewLds));
        });
        packed_launch(ctx, kern, kFewLds, slots, p, splits, part);
      } else {
        packed_launch(ctx, packed_attn_rows<BF, CAP, BIAS>, 0, (int64_t)p.nblocks * p.G, p, splits, part);
      }
    };
    if (f32 && few) packed_launch(ctx, packed_attn_f32<CAP, BIAS>, 0, slots, p, splits, part);
    else if (f32) packed_launch(ctx, packed_attn_f32_rows<CAP, BIAS>, 0, (int64_t)p.nblocks * p.G, p, splits, part);
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
    join<<<(unsigned)((all + 15) / 16), 256, 0, stream_of(ctx)>>>(dt, part, splits, all, p.O);
  }
}

}  // namespace hb

using namespace hb;

extern "C" int hb_sdpa_packed(uintptr_t ctx, int dt, uintptr_t q, const int64_t* qs, uintptr_t k, const int64_t* ks,
                              uintptr_t v, const int64_t* vs, uintptr_t o, uintptr_t q_doc, uintptr_t q_blocks,
                              uintptr_t q_offsets, uintptr_t k_offsets, int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hk, int64_t D, float scale,
                              int causal, int64_t window, uintptr_t prefix, float cap, uintptr_t slopes) {
  HB_API_BEGIN
  HB_REQUIRE(dt == HB_F32 || dt == HB_F16 || dt == HB_BF16, "hb_sdpa_packed: dtype must be f32, f16 or bf16");
  HB_REQUIRE(B >= 0 && Tq >= 0 && Tk >= 0 && B < (1ll << 30) && Tq < (1ll << 30) && Tk < (1ll << 30),
             "hb_sdpa_packed: bad sizes");
  HB_REQUIRE(H >= 1 && Hk >= 1 && H % Hk == 0 && H < 65536, "hb_sdpa_packed: heads must be a multiple of the key heads");
  HB_REQUIRE(D >= 1 && D <= 64 * kAnyCols, "hb_sdpa_packed: head dimension must be 1 to 512");
  HB_REQUIRE(qs && ks && vs, "hb_sdpa_packed: null strides");
  HB_REQUIRE(std::isfinite(scale) && std::isfinite(cap) && cap >= 0.f, "hb_sdpa_packed: scale and cap must be finite");
  HB_REQUIRE(cap == 0.f || cap >= FLT_MIN, "hb_sdpa_packed: a cap is 0 (none) or a normal number");
  HB_REQUIRE(window >= -1, "hb_sdpa_packed: a window is not negative (-1: none)");
  if (Tq == 0) return 0;
  HB_REQUIRE(q && o && q_doc && q_blocks && q_offsets && k_offsets && (Tk == 0 || (k && v)), "hb_sdpa_packed: null argument");
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
  p.doc = (const int32_t*)q_doc;
  p.blocks = (const int32_t*)q_blocks;
  p.nblocks = (int)plan_blocks(B, Tq);
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
  // (its reciprocal is normal and twice its score to base 2 finite; scores below 2^114 round to themselves under either)
  p.cap = fminf(cap, 0x1p126f);
  p.sc = score_of(scale, p.cap, slopes != 0);
  if (packed_takes_mfma(p, dt == HB_F32 ? 4 : 8)) packed_mfma(ctx, dt, p);
  else packed_any(ctx, dt, p);
  check_launch("hb_sdpa_packed");
  HB_API_END
}
