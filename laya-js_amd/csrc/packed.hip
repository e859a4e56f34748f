// Packed batches: the documents of a batch laid end to end, [T, ...] with T the
// sum of their lengths, instead of each padded to the longest.  The plan of
// such a batch from the documents' lengths (hb_pack_plan), rows moved between
// the padded and the packed layout (hb_pack_rows, hb_unpack_rows), and rotary
// positions given per token (hb_rope_at).
#include <math.h>

#include <stdexcept>

#include "common.h"

namespace hb {

// ------------------------------------------------------------------ plan

// off_b = min(T, sum of the lengths before b), lengths below 0 counting as 0
// and above L (if L > 0) as L; token t belongs to the last b with off_b <= t,
// at position t - off_b.
//
// The table of blocks: document b has ceil(n_b / kBlockTokens) entries, in order,
// then come those of the rows behind the last document (as document B), then -1.
//
// One launch: every block scans the lengths, 1024 at a time, as far as its own
// 1024 tokens need, and finds their documents by bisection among the 1024
// offsets in LDS; block 0 also writes the offsets, and the last block the end of the
// table.  Scanning B lengths again in each block costs less than a second launch
// would (B / 1024 rounds of one 16-byte read a thread); what bounds it is the
// launch itself, then the 12 bytes written a token (3 us for 300 tokens, 5 for 37k).
constexpr int kPlanDocs = 1024, kPlanTokens = 1024;

// Exclusive sums over the block's 256 threads, and their total.
__device__ __forceinline__ int64_t scan256(int64_t v, int64_t* wsum, int64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t incl = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t up = __shfl_up(incl, o, 64);
    if (lane >= o) incl += up;
  }
  if (lane == 63) wsum[wave] = incl;
  __syncthreads();
  int64_t base = incl - v;
  *total = 0;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    if (w < wave) base += wsum[w];
    *total += wsum[w];
  }
  return base;
}

__global__ __launch_bounds__(256) void pack_plan_kernel(const int32_t* __restrict__ lengths, int B, int T, int L,
                                                        int nblocks, int32_t* __restrict__ offsets,
                                                        int32_t* __restrict__ doc, int32_t* __restrict__ pos,
                                                        int32_t* __restrict__ slots, int2* __restrict__ blocks) {
  __shared__ int off[kPlanDocs + 1], boff[kPlanDocs];
  __shared__ int64_t wsum[2][4];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * kPlanTokens, t1 = T - t0 < kPlanTokens ? T : t0 + kPlanTokens;
  const bool first = blockIdx.x == 0, last = blockIdx.x == gridDim.x - 1;
  int64_t carry = 0;  // sum of the lengths before this round
  int bcarry = 0;     // and of their blocks
  for (int b0 = 0; b0 < B; b0 += kPlanDocs) {
    int64_t n[4], sum = 0, total;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int b = b0 + 4 * tid + e;
      int v = b < B ? lengths[b] : 0;
      v = v < 0 ? 0 : (L > 0 && v > L ? L : v);
      n[e] = sum;
      sum += v;
    }
    const int64_t base = carry + scan256(sum, wsum[0], &total);
    total += carry;
    int nb = 0, bn[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {  // (cut off at T)
      const int64_t o = base + n[e], x = base + (e < 3 ? n[e + 1] : sum);
      const int a = o < T ? (int)o : T, c = x < T ? (int)x : T;
      off[4 * tid + e] = a;
      bn[e] = nb;
      nb += (c - a + kBlockTokens - 1) / kBlockTokens;
    }
    int64_t btotal;
    const int bbase = bcarry + (int)scan256(nb, wsum[1], &btotal);
#pragma unroll
    for (int e = 0; e < 4; e++) boff[4 * tid + e] = bbase + bn[e];
    const int end = total < T ? (int)total : T;  // of this round's documents
    if (tid == 0) off[kPlanDocs] = end;
    __syncthreads();
    const int nd = B - b0 < kPlanDocs ? B - b0 : kPlanDocs;
    if (first)
      for (int i = tid; i < nd; i += 256) offsets[b0 + i] = off[i];
    const int lo = off[0] > t0 ? off[0] : t0, hi = end < t1 ? end : t1;
    for (int t = lo + tid; t < hi; t += 256) {
      int a = 0, c = nd;  // off[a] <= t, and the answer is in [a, c)
      while (c - a > 1) {
        const int m = (a + c) >> 1;
        if (off[m] <= t) a = m;
        else c = m;
      }
      const int d = b0 + a, q = t - off[a];
      doc[t] = d;
      pos[t] = q;
      if (slots != nullptr) slots[t] = d * L + q;
      if (q % kBlockTokens == 0) blocks[boff[a] + q / kBlockTokens] = int2{d, t};
    }
    carry = total;
    bcarry += (int)btotal;
    if (!first && !last && end >= t1) break;  // (the same in every thread)
    __syncthreads();  // off, boff and wsum are written again
  }
  const int end = carry < T ? (int)carry : T;
  if (first && tid == 0) offsets[B] = end;
  for (int t = (end > t0 ? end : t0) + tid; t < t1; t += 256) {  // behind the last document
    doc[t] = -1;
    pos[t] = 0;
    if (slots != nullptr) slots[t] = -1;
    if ((t - end) % kBlockTokens == 0) blocks[bcarry + (t - end) / kBlockTokens] = int2{B, t};
  }
  if (last)
    for (int i = bcarry + (T - end + kBlockTokens - 1) / kBlockTokens + tid; i < nblocks; i += 256) blocks[i] = int2{-1, 0};
}

// ------------------------------------------------------------------ rows

// Moves whole rows, one wave each: the row's source index is the same in all
// lanes, which take its vectors in turn.  Bound by reading and writing the rows (64 x
// 1024 x 1024 in f16: 37 us, 5 TB/s with what the caches hold).
// UNPACK: row b * L + l of the padded batch is row off_b + l of the packed one;
// else row t of the packed batch is row idx[t] of the padded one.  Rows without
// a source are zeros.
template <class V, bool UNPACK>
__global__ __launch_bounds__(256) void move_rows_kernel(const V* __restrict__ src, int64_t nsrc, int64_t vecs,
                                                        const int32_t* __restrict__ idx, int L, int64_t rows,
                                                        V* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); r < rows;
       r += (int64_t)gridDim.x * 4) {
    int64_t s;
    if constexpr (UNPACK) {
      const int64_t b = r / L, l = r - b * L, o = idx[b], n = idx[b + 1] - o;
      s = l < n ? o + l : -1;
    } else {
      s = idx[r];
    }
    const bool ok = s >= 0 && s < nsrc;
    const V* from = src + (ok ? s : 0) * vecs;
    V* to = out + r * vecs;
    for (int64_t i = lane; i < vecs; i += 64) to[i] = ok ? from[i] : V{};
  }
}

template <bool UNPACK>
static void launch_move_rows(hipStream_t st, uintptr_t src, int64_t nsrc, int64_t row_bytes, const int32_t* idx, int L,
                             int64_t rows, uintptr_t out) {
  const unsigned grid = capped_grid((rows + 3) / 4, 256);
  auto go = [&](auto v) {
    using V = decltype(v);
    move_rows_kernel<V, UNPACK><<<grid, 256, 0, st>>>((const V*)src, nsrc, row_bytes / (int64_t)sizeof(V), idx, L, rows,
                                                      (V*)out);
  };
  const int64_t al = src | out | row_bytes;
  if (al % 16 == 0) go(uint4v{});
  else if (al % 4 == 0) go(uint32_t{});
  else if (al % 2 == 0) go(uint16_t{});
  else go(uint8_t{});
}

// ------------------------------------------------------------------ rotary positions

constexpr int kMaxAxes = 4, kMaxRopeD = 512;
struct RopeAt {
  float inv[kMaxRopeD / 2];  // angle per position of each rotation pair
  int end[kMaxAxes];         // axis a rotates pairs end[a - 1] .. end[a] - 1
};

// cos and sin of pair i's angle at token t: the product of position and
// frequency rounded to f32, as the table of hb_rope holds it, its cosine and
// sine evaluated in f64 and rounded to f32.
__device__ __forceinline__ float2 rope_at_cs(const RopeAt& f, const int32_t* positions, int64_t T, int64_t t, int i) {
  int a = 0;
  while (i >= f.end[a]) a++;
  const float th = (float)((double)positions[a * T + t] * (double)f.inv[i]);
  double s, c;
  sincos((double)th, &s, &c);
  return float2{(float)c, (float)s};
}

// Rows of 16-byte aligned chunks (V values each, D / 2 a multiple of V): a block
// takes TB tokens, computes the cosines and sines of their D / 2 angles once for
// all heads, and rotates the chunk pairs (c, c + D / 2) of its heads, four loads
// of a thread in flight.  Bound by reading and writing the heads; a sine and
// cosine in f64 cost a block about as much as 16 KB of traffic, so TB tokens
// share a block where there are enough of them (32768 rows x 32 heads on three axes, bf16:
// 60 us, 4.5 TB/s; a block a token: 226).
constexpr int kRopeTokens = 8;  // 256 threads: one angle each at D = 64
template <class T, int V, bool BF16>
__device__ __forceinline__ void rope_load(const T* p, float (&v)[V]) {
  if constexpr (V == 4) {
    const float4v x = *(const float4v*)p;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = x[e];
  } else {
    const uint4v x = *(const uint4v*)p;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint16_t h = (uint16_t)(x[e >> 1] >> (16 * (e & 1)));
      v[e] = BF16 ? bf16_to_f32(h) : f16_bits_to_f32(h);
    }
  }
}
template <class T, int V, bool BF16>
__device__ __forceinline__ void rope_store(T* p, const float (&v)[V]) {
  if constexpr (V == 4) {
    *(float4v*)p = float4v{v[0], v[1], v[2], v[3]};
  } else {
    uint4v x;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t a = BF16 ? f32_to_bf16(v[2 * e]) : f32_to_f16_bits(v[2 * e]);
      const uint32_t c = BF16 ? f32_to_bf16(v[2 * e + 1]) : f32_to_f16_bits(v[2 * e + 1]);
      x[e] = a | (c << 16);
    }
    *(uint4v*)p = x;
  }
}
template <class T, int V, bool BF16>
__global__ __launch_bounds__(256) void rope_at_vec_kernel(const T* __restrict__ x, int64_t s0, int64_t s1,
                                                          T* __restrict__ y, int T_, int H, int D, int tb,
                                                          const int32_t* __restrict__ positions, RopeAt f) {
  extern __shared__ float2 cs[];  // [tb][D / 2]
  const int64_t first = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * tb;
  if (first >= T_) return;  // (the whole block)
  const int half = D / 2, C = half / V, t0 = (int)first, nt = T_ - t0 < tb ? T_ - t0 : tb;
  for (int i = threadIdx.x; i < nt * half; i += 256) cs[i] = rope_at_cs(f, positions, T_, t0 + i / half, i % half);
  __syncthreads();
  const int per = H * C, n = nt * per;
  constexpr int U = 4;
  for (int i0 = threadIdx.x; i0 < n; i0 += 256 * U) {
    float a[U][V], b[U][V];
    int at[U];  // angle of the chunk's first pair, or -1
    int64_t to[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + 256 * u;
      at[u] = -1;
      if (i >= n) continue;
      const int t = i / per, q = i - t * per, h = q / C, c = (q - h * C) * V;
      const T* from = x + (int64_t)(t0 + t) * s0 + h * s1 + c;
      rope_load<T, V, BF16>(from, a[u]);
      rope_load<T, V, BF16>(from + half, b[u]);
      at[u] = t * half + c;
      to[u] = ((int64_t)(t0 + t) * H + h) * D + c;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (at[u] < 0) continue;
      float lo[V], hi[V];
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float2 w = cs[at[u] + e];
        lo[e] = pin_f32(fmaf(-b[u][e], w.y, a[u][e] * w.x));
        hi[e] = pin_f32(fmaf(a[u][e], w.y, b[u][e] * w.x));
      }
      rope_store<T, V, BF16>(y + to[u], lo);
      rope_store<T, V, BF16>(y + to[u] + half, hi);
    }
  }
}

// Any type, head dimension and strides: one thread per rotation pair.
__global__ __launch_bounds__(256) void rope_at_kernel(int dt, const void* __restrict__ x, int64_t s0, int64_t s1,
                                                      int64_t s2, void* __restrict__ y, int64_t T, int64_t H, int D,
                                                      const int32_t* __restrict__ positions, RopeAt f) {
  const int half = D / 2;
  const int64_t n = T * H * half;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / half, t = r / H, h = r - t * H;
    const int j = (int)(i - r * half);
    const float2 cs = rope_at_cs(f, positions, T, t, j);
    const int64_t src = t * s0 + h * s1;
    const float x0 = load_f(x, src + j * s2, dt), x1 = load_f(x, src + (j + half) * s2, dt);
    store_f(y, r * D + j, dt, fmaf(-x1, cs.y, x0 * cs.x));
    store_f(y, r * D + j + half, dt, fmaf(x0, cs.y, x1 * cs.x));
  }
}

}  // namespace hb

using namespace hb;

extern "C" {

int hb_pack_plan(uintptr_t ctx, uintptr_t lengths, int64_t B, int64_t T, int64_t L, uintptr_t offsets, uintptr_t doc,
                 uintptr_t pos, uintptr_t slots, uintptr_t blocks) {
  HB_API_BEGIN
  HB_REQUIRE(B >= 0 && T >= 0 && L >= 0 && B < (1ll << 30) && T < (1ll << 30) && L < (1ll << 30),
             "hb_pack_plan: bad sizes");
  HB_REQUIRE((B == 0 || lengths) && offsets && blocks && (T == 0 || (doc && pos)), "hb_pack_plan: null argument");
  HB_REQUIRE(!slots || (L > 0 && B * L < (1ll << 31)), "hb_pack_plan: slots need L > 0 and B * L below 2^31");
  const unsigned grid = (unsigned)((T + kPlanTokens - 1) / kPlanTokens);
  pack_plan_kernel<<<grid < 1 ? 1 : grid, 256, 0, stream_of(ctx)>>>((const int32_t*)lengths, (int)B, (int)T, (int)L,
                                                                    (int)plan_blocks(B, T), (int32_t*)offsets, (int32_t*)doc,
                                                                    (int32_t*)pos, (int32_t*)slots, (int2*)blocks);
  check_launch("hb_pack_plan");
  HB_API_END
}

int hb_pack_rows(uintptr_t ctx, uintptr_t x, int64_t rows, int64_t row_bytes, uintptr_t slots, int64_t T,
                 uintptr_t out) {
  HB_API_BEGIN
  HB_REQUIRE(rows >= 0 && row_bytes >= 0 && T >= 0 && T < (1ll << 30), "hb_pack_rows: bad sizes");
  if (T == 0 || row_bytes == 0) return 0;
  HB_REQUIRE((rows == 0 || x) && slots && out, "hb_pack_rows: null argument");
  launch_move_rows<false>(stream_of(ctx), x, rows, row_bytes, (const int32_t*)slots, 1, T, out);
  check_launch("hb_pack_rows");
  HB_API_END
}

int hb_unpack_rows(uintptr_t ctx, uintptr_t x, int64_t T, int64_t row_bytes, uintptr_t offsets, int64_t B, int64_t L,
                   uintptr_t out) {
  HB_API_BEGIN
  HB_REQUIRE(T >= 0 && row_bytes >= 0 && B >= 0 && L >= 0 && B < (1ll << 30) && L < (1ll << 30) && B * L < (1ll << 31),
             "hb_unpack_rows: bad sizes");
  if (B * L == 0 || row_bytes == 0) return 0;
  HB_REQUIRE((T == 0 || x) && offsets && out, "hb_unpack_rows: null argument");
  launch_move_rows<true>(stream_of(ctx), x, T, row_bytes, (const int32_t*)offsets, (int)L, B * L, out);
  check_launch("hb_unpack_rows");
  HB_API_END
}

int hb_rope_at(uintptr_t ctx, int dt, uintptr_t x, const int64_t* xs, uintptr_t y, int64_t T, int64_t H, int64_t D,
               uintptr_t positions, int64_t axes, const int64_t* sections, double base) {
  HB_API_BEGIN
  HB_REQUIRE(dt == HB_F32 || dt == HB_F16 || dt == HB_BF16, "hb_rope_at: dtype must be f32, f16 or bf16");
  HB_REQUIRE(T >= 0 && H >= 0 && T < (1ll << 30) && H < (1ll << 20), "hb_rope_at: bad sizes");
  HB_REQUIRE(D > 0 && D % 2 == 0 && D <= kMaxRopeD, "hb_rope_at: the head dimension must be even and at most 512");
  HB_REQUIRE(axes >= 1 && axes <= kMaxAxes && sections && xs, "hb_rope_at: one to four axes with their sections");
  HB_REQUIRE(base > 0 && std::isfinite(base), "hb_rope_at: base must be positive");
  RopeAt f{};
  int64_t end = 0;
  for (int a = 0; a < axes; a++) {
    HB_REQUIRE(sections[a] >= 0 && sections[a] <= D / 2, "hb_rope_at: bad section");
    end += sections[a];
    f.end[a] = (int)end;
  }
  HB_REQUIRE(end == D / 2, "hb_rope_at: the sections must add up to half the head dimension");
  // (the frequencies of rope_table: the contract's f32 rule)
  const float lb = (float)log2(base);
  for (int64_t i = 0; i < D / 2; i++) {
    const float frac = (float)((double)i / (double)(D / 2));
    f.inv[i] = (float)exp2((double)(float)(-(double)frac * (double)lb));
  }
  if (T * H == 0) return 0;
  HB_REQUIRE(x && y && positions, "hb_rope_at: null argument");
  const int per = dt == HB_F32 ? 4 : 8;  // values of a 16-byte chunk
  if (D / 2 % per == 0 && xs[2] == 1 && xs[0] % per == 0 && xs[1] % per == 0 && x % 16 == 0 && y % 16 == 0) {
    const int tb = T >= 2048 ? kRopeTokens : 1;
    const int64_t blocks = (T + tb - 1) / tb;
    const unsigned gx = capped_grid(blocks, 256);
    const dim3 grid(gx, (unsigned)((blocks + gx - 1) / gx));
    const size_t lds = (size_t)tb * (D / 2) * sizeof(float2);
    auto go = [&](auto kern, auto v) {
      using E = decltype(v);
      kern<<<grid, 256, lds, stream_of(ctx)>>>((const E*)x, xs[0], xs[1], (E*)y, (int)T, (int)H, (int)D, tb,
                                               (const int32_t*)positions, f);
    };
    if (dt == HB_F32) go(rope_at_vec_kernel<float, 4, false>, 0.f);
    else if (dt == HB_F16) go(rope_at_vec_kernel<uint16_t, 8, false>, (uint16_t)0);
    else go(rope_at_vec_kernel<uint16_t, 8, true>, (uint16_t)0);
  } else {
    rope_at_kernel<<<capped_grid((T * H * (D / 2) + 255) / 256, 256), 256, 0, stream_of(ctx)>>>(
        dt, (const void*)x, xs[0], xs[1], xs[2], (void*)y, T, H, (int)D, (const int32_t*)positions, f);
  }
  check_launch("hb_rope_at");
  HB_API_END
}

}  // extern "C"
