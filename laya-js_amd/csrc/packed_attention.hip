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
// packed_attn_any: any head dimension, type and strides.
#include <math.h>

#include <stdexcept>

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

// One wave per query and head: 64 keys at a time, a score per lane, then the
// lanes share out the columns of the output.
constexpr int kAnyCols = 8;  // columns per lane: D <= 512
__global__ __launch_bounds__(64) void packed_attn_any(Packed p, int dt) {
  extern __shared__ float sh[];  // [D] query, [64] weights, [64] visibility
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
    w[64 + lane] = seen ? 1.f : 0.f;
    __syncthreads();
    for (int i = 0; i < kAnyCols && i * 64 + lane < D; i++) {
      float a = o[i] * alpha;
      const int64_t col = vh + (i * 64 + lane) * p.vs[2];
      for (int k = 0; k < 64 && j0 + k < d.nk; k++)
        if (w[64 + k] != 0.f) a = fmaf(w[k], load_f(p.V, (int64_t)(d.k0 + j0 + k) * p.vs[0] + col, dt), a);
      o[i] = a;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int i = 0; i < kAnyCols && i * 64 + lane < D; i++)
    store_f(p.O, ((int64_t)t * p.H + h) * D + i * 64 + lane, dt, o[i] * inv);
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
  packed_attn_any<<<dim3((unsigned)Tq, (unsigned)H), 64, (size_t)(D + 128) * 4, stream_of(ctx)>>>(p, dt);
  check_launch("hb_sdpa_packed");
  HB_API_END
}
