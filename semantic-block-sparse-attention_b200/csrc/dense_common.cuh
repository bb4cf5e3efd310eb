// What the two prompt-attention kernels share: which document and query tile a block works on, which key
// tiles that tile sees, the mask of a row, the scores' transformation, and the packing of P.
#pragma once
#include <cuda_fp16.h>

#include "sm100.cuh"

namespace dense {

using namespace sm100;

constexpr float LN2F = 0.6931471805599453f;
constexpr float LOG2EF = 1.4426950408889634f;

struct Args {
  const void* q;                  // [Tq, Hq, D], strides in elements
  int64_t q_token, q_head;
  void* out;                      // [Tq, Hq, D] contiguous
  float* lse;                     // [Tq, Hq] or null
  const int32_t* cu_q;            // [docs + 1]
  const int32_t* cu_k;
  const int32_t* prefix;          // [docs] or null
  const float* slopes;            // [Hq] or null
  int docs, group, num_q_heads;
  int queries_per_tile, num_kv_heads;
  int64_t tokens_q, tokens_k;
  int causal, window;
  int zero_tail;                  // write zeros to the rows that no document has
  float score_scale;              // raw product -> log2 units, or -> 8/3 of the capping tanh's argument
  float cap_log2;                 // cap * log2(e)
  int* status;
  int splits, piece_keys;         // pieces that a tile's keys may be cut into, a block each, and their least size
  float* partial;                 // with splits > 1: [tile][KV head][splits][record_floats(D)]
};

// The block's share: queries [q0, q0 + nq) of a document (token of query 0: tok0), keys k0 ... of length lk.
struct Tile {
  int doc;
  int first;                      // index of the tile's first query in its document
  int count;                      // its queries
  int64_t token;                  // its first token
  int k0, lk;                     // the document's first key row and its keys
  int pos;                        // position of the tile's first query
  int prefix;
};

// Tile number `want` (0 ...).  Blocks start in this order, so the tiles with the most keys come first: by level, the
// position of a tile's first query in units of queries_per_tile (a document's last tiles see the most keys), and
// inside a level by document.  One KV head after the other and document by document, the last long tiles ran
// alone (32 heads over 8, D = 128: 4096 tokens 175 us against 153, two documents in 8192 361 against 326).
// doc = -1 behind the last tile; then `first` counts the tiles behind it.  For up to 64 documents, two a lane;
// warp-collective, and every warp of the block computes the same answer.
constexpr int WARP_DOCS = 64;
__device__ __forceinline__ Tile find_tile(const Args& a, int want) {
  const int lane = threadIdx.x & 31;
  const int qt = a.queries_per_tile;
  int64_t c0[2], c1[2];
  int k0[2], lk[2], n[2], off[2], pre[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {                    // all that may be needed, in one round trip
    const int d = 32 * i + lane;
    c0[i] = c1[i] = 0;
    k0[i] = lk[i] = pre[i] = 0;
    if (d < a.docs) {
      c0[i] = a.cu_q[d];
      c1[i] = a.cu_q[d + 1];
      k0[i] = a.cu_k[d];
      lk[i] = a.cu_k[d + 1];
      if (a.prefix) pre[i] = a.prefix[d];
    }
  }
  int all = 0, top = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    c0[i] = min(max(c0[i], (int64_t)0), a.tokens_q);
    c1[i] = min(max(c1[i], c0[i]), a.tokens_q);
    k0[i] = (int)min(max((int64_t)k0[i], (int64_t)0), a.tokens_k);
    lk[i] = (int)min(max((int64_t)lk[i], (int64_t)k0[i]), a.tokens_k) - k0[i];
    const int lq = (int)(c1[i] - c0[i]);
    n[i] = (lq + qt - 1) / qt;
    off[i] = max(lk[i] - lq, 0) / qt;              // level of the document's first tile
    all += n[i];
    if (n[i]) top = max(top, off[i] + n[i]);
  }
  all = __reduce_add_sync(0xffffffffu, all);
  Tile t{};
  t.doc = -1;
  t.first = want - all;
  if (want >= all) return t;
  // the largest level that has no more than `want` tiles above it
  auto from = [&](int level) {                     // tiles of `level` and above
    return (int)__reduce_add_sync(0xffffffffu, min(max(off[0] + n[0] - level, 0), n[0]) + min(max(off[1] + n[1] - level, 0), n[1]));
  };
  int lo = 0, hi = __reduce_max_sync(0xffffffffu, top);       // from(lo) > want >= from(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (from(mid) > want) lo = mid; else hi = mid;
  }
  int nth = want - from(lo + 1);
  const uint32_t in0 = __ballot_sync(0xffffffffu, off[0] <= lo && lo < off[0] + n[0]);
  const uint32_t in1 = __ballot_sync(0xffffffffu, off[1] <= lo && lo < off[1] + n[1]);
  const int half = nth >= __popc(in0);
  if (half) nth -= __popc(in0);
  const int at = __fns(half ? in1 : in0, 0, nth + 1);
  auto pick = [&](auto (&x)[2]) { return __shfl_sync(0xffffffffu, half ? x[1] : x[0], at); };
  const int64_t q0 = pick(c0), q1 = pick(c1);
  t.doc = 32 * half + at;
  t.first = (lo - pick(off)) * qt;
  t.count = (int)min((int64_t)qt, q1 - q0 - t.first);
  t.token = q0 + t.first;
  t.k0 = pick(k0);
  t.lk = pick(lk);
  t.pos = t.lk - (int)(q1 - q0) + t.first;
  t.prefix = min(max(pick(pre), 0), t.lk);
  return t;
}

// For more documents, in their order (and a document's last tiles first): all threads of the block, a run of documents
// each.  Two barriers, which every thread has to reach.
constexpr int FIND_BYTES = 128;                    // of shared memory
template <int THREADS>
__device__ __forceinline__ Tile find_tile_block(const Args& a, int want, void* scratch) {
  static_assert(sizeof(Tile) % 8 == 0 && sizeof(Tile) + THREADS / 8 <= FIND_BYTES, "scratch");
  Tile& found = *static_cast<Tile*>(scratch);
  int* totals = reinterpret_cast<int*>(&found + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, qt = a.queries_per_tile;
  const int per = (a.docs + THREADS - 1) / THREADS;
  const int d0 = min((int)threadIdx.x * per, a.docs), d1 = min(d0 + per, a.docs);
  auto start_of = [&](int d) { return min(max((int64_t)a.cu_q[d], (int64_t)0), a.tokens_q); };
  auto end_of = [&](int d, int64_t from) { return min(max((int64_t)a.cu_q[d + 1], from), a.tokens_q); };
  int mine = 0;
  for (int d = d0; d < d1; ++d) {
    const int64_t c0 = start_of(d);
    mine += (int)((end_of(d, c0) - c0 + qt - 1) / qt);
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) totals[warp] = upto;
  __syncthreads();
  int before = upto - mine, all = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += totals[w];
    all += totals[w];
  }
  if (want >= all) {
    Tile t{};
    t.doc = -1;
    t.first = want - all;
    return t;                                      // the same answer in every thread
  }
  if (want >= before && want < before + mine) {
    int rest = want - before, d = d0;
    int64_t c0 = 0, c1 = 0;
    int tiles = 0;
    for (;; ++d) {
      c0 = start_of(d);
      c1 = end_of(d, c0);
      tiles = (int)((c1 - c0 + qt - 1) / qt);
      if (rest < tiles) break;
      rest -= tiles;
    }
    Tile t;
    t.doc = d;
    t.first = (tiles - 1 - rest) * qt;
    t.count = (int)min((int64_t)qt, c1 - c0 - t.first);
    t.token = c0 + t.first;
    t.k0 = (int)min(max((int64_t)a.cu_k[d], (int64_t)0), a.tokens_k);
    t.lk = (int)min(max((int64_t)a.cu_k[d + 1], (int64_t)t.k0), a.tokens_k) - t.k0;
    t.pos = t.lk - (int)(c1 - c0) + t.first;
    t.prefix = a.prefix ? min(max(a.prefix[d], 0), t.lk) : 0;
    found = t;
  }
  __syncthreads();
  return found;
}

// Rows that no document has, those behind the last one and then those in front of the first, as zeros with a log-sum-exp
// of -inf: the spare blocks share them by tiles (there are enough: a grid of T / qt + docs tiles has at least the rest's).
template <int D>
__device__ __forceinline__ void zero_rest(const Args& a, int nth, int kv_head, int threads) {
  const int64_t front = min(max((int64_t)a.cu_q[0], (int64_t)0), a.tokens_q);
  const int64_t last = min(max((int64_t)a.cu_q[a.docs], front), a.tokens_q);
  const int64_t behind = a.tokens_q - last;
  const int64_t r0 = (int64_t)nth * a.queries_per_tile, r1 = min(behind + front, r0 + a.queries_per_tile);
  constexpr int CH = D / 8;
  for (int64_t i = threadIdx.x; i < (r1 - r0) * a.group * CH; i += threads) {
    const int64_t row = i / CH, r = r0 + row / a.group;
    const int64_t at = (r < behind ? last + r : r - behind) * a.num_q_heads + kv_head * a.group + row % a.group;
    reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at * D)[i % CH] = make_uint4(0u, 0u, 0u, 0u);
    if (a.lse && i % CH == 0) a.lse[at] = -INFINITY;
  }
}

// Keys that a row at position p sees: [lo, hi) and [0, pre).
struct Seen { int lo, hi, pre; };
__device__ __forceinline__ Seen seen_by(const Args& a, const Tile& t, int p) {
  Seen s;
  s.hi = a.causal ? min(t.lk, max(p + 1, 0)) : t.lk;
  s.lo = a.causal && a.window > 0 ? max(0, p - a.window + 1) : 0;
  s.pre = a.causal ? t.prefix : 0;
  return s;
}

// Bit i: key i of 32 is seen, for limits relative to the first of them; and what is not seen becomes -inf.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t seen_bits(int lo, int hi, int pre) { return (below(hi) & ~below(lo)) | below(pre); }
__device__ __forceinline__ void hide32(uint32_t* x, uint32_t bits) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (!(bits & (1u << i))) x[i] = 0xff800000u;
}

// The key tiles of BN rows that any row of the block's tile sees: [0, gp) then [glo, ...), n in all.
template <int BN>
struct KeyTiles {
  int gp, glo, n, base = 0;
  __device__ __forceinline__ KeyTiles(const Args& a, const Tile& t) {
    const Seen lo = seen_by(a, t, t.pos), hi = seen_by(a, t, t.pos + t.count - 1);
    gp = (lo.pre + BN - 1) / BN;
    const int end = max(gp, (hi.hi + BN - 1) / BN);
    glo = min(max(gp, lo.lo / BN), end);
    n = gp + end - glo;
  }
  __device__ __forceinline__ int at(int j) const { j += base; return (j < gp ? j : j - gp + glo) * BN; }
};

// ---- keys cut into pieces, where there are too few tiles for the multiprocessors.  A piece's block leaves O, the
// reference and the sum of each of its 128 rows, and a second launch joins them.
__host__ __device__ constexpr int record_floats(int d) { return 128 * (d + 3); }       // O [128][D], m, l, lr [128]
__device__ __forceinline__ int pieces_of(const Args& a, int n, int bn) { return min(a.splits, max(1, n * bn / a.piece_keys)); }

// The block's share of the grid: tile number `want` of KV head h, piece `split`.
struct Share {
  int want, h, split;
  __device__ __forceinline__ Share(const Args& a, int splits) {
    const int unit = splits > 1 ? blockIdx.x / splits : blockIdx.x;
    split = blockIdx.x - unit * splits;
    want = unit / a.num_kv_heads;
    h = unit - want * a.num_kv_heads;
  }
  __device__ __forceinline__ float* record(const Args& a, int d, int s) const {
    return a.partial + (((int64_t)want * a.num_kv_heads + h) * a.splits + s) * record_floats(d);
  }
};

// ---- two floats in a 64-bit register: one instruction for both
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 join(float x, float y) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ void split(f32x2 v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ float fmin3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// tanh(x) = 1 - 2 / (1 + e^2x): exact at both ends, absolute error a few 2^-24; two special-function operations.  For caps up
// to 52 that is enough; under higher ones tanh_any keeps small scores relative beside a row that reaches the cap.
__device__ __forceinline__ float tanh_exp(float x) {
  return 1.f - __fdividef(2.f, 1.f + fast_exp2(x * (2.f * LOG2EF)));
}

// tanh(3/8 y) as y P(y^2) on the multiply-add pipe (the exponentials of the softmax fill the special-function
// unit), P fitted for the smallest largest error: of degree 4 for |y| < 2 (2.5e-7 as evaluated in 32 bits), of
// degree 7 for |y| < 4 (5e-7; near 0 relative to y, 4e-6).  Scores beyond 1.5 caps are rare and take an exponential.
constexpr float TANH_ARG = 8.f / 3.f, TANH_FAR = 4.f;
__device__ __forceinline__ constexpr float near_coefficient(int i) {
  const float c[5] = {0.374998957f, -0.0175727159f, 0.000980816782f, -5.13917694e-05f, 1.80655456e-06f};
  return c[i];
}
__device__ __forceinline__ constexpr float far_coefficient(int i) {
  const float c[8] = {0.37499851f, -0.0175732356f, 0.000984045211f, -5.41848349e-05f,
                      2.69307429e-06f, -1.0540262e-07f, 2.68661982e-09f, -3.18844812e-11f};
  return c[i];
}
// factor * tanh(3/8 y) = y P(y^2) with the factor in the N coefficients (5: near, 8: far).
template <int N>
struct TanhPoly {
  f32x2 c[N];
  __device__ __forceinline__ explicit TanhPoly(float factor) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = factor * (N == 5 ? near_coefficient(i) : far_coefficient(i));
      c[i] = join(v, v);
    }
  }
  // y P(y^2) + add
  __device__ __forceinline__ f32x2 operator()(f32x2 y, f32x2 add) const {
    const f32x2 u = mul2(y, y);
    f32x2 r = c[N - 1];
#pragma unroll
    for (int i = N - 2; i >= 0; --i) r = fma2(r, u, c[i]);
    return fma2(r, y, add);
  }
};
// What happens to a raw score: 0 scaled only, 1 capped, 2 biased by distance (and capped, if there is a cap), 3
// capped so low that no running maximum is needed.
enum Mode { LINEAR = 0, CAPPED = 1, BIASED = 2, BOUNDED = 3 };

// A cap bounds the scores, so with bf16 P (float's range) a fixed reference will do where 2^(score - reference)
// stays between 2^-92 and 2^60: no maximum, no rescale of O, and the products P V stay inside float for |v| from
// 2^-34 (rows whose scores are all at the lower end) to 2^43 (over 2^24 keys).  That is caps up to 52.
constexpr float BOUNDED_TOP = 60.f, BOUNDED_LOG2 = 76.f;
__host__ __device__ inline float bounded_reference(float cap_log2) { return cap_log2 > BOUNDED_TOP ? cap_log2 - BOUNDED_TOP : 0.f; }

// A score behind which there is no query and key of the document (a key that the row does not see may be another
// document's, or what an earlier launch left) must not decide on a warp's form of tanh: it counts as 0, and a row of
// another document has no vote.  So a document's bits do not depend on what is packed beside it.
struct Vote {
  uint32_t near;                  // the bit that tells |y| >= 2, or none
  float near_most, far;           // 2 and TANH_FAR, or beyond every score
  __device__ __forceinline__ explicit Vote(bool mine)
      : near(mine ? 0x40000000u : 0u), near_most(mine ? 2.f : INFINITY), far(mine ? TANH_FAR : INFINITY) {}
};
__device__ __forceinline__ void clear32(uint32_t* x, uint32_t bits) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (!(bits & (1u << i))) x[i] = 0u;
}

// 32 raw scores in place -> what the exponential's scale multiplies; `bits` are the seen ones unless all are.  All lanes of a
// warp take part.
template <int MODE>
__device__ __forceinline__ void transform32(uint32_t* x, const Args& a, float slope, int p, int key0, bool all, uint32_t bits,
                                            const Vote& vote) {
  if constexpr (MODE == LINEAR) return;
  if (MODE == CAPPED || a.cap_log2 > 0.f) {
    if (!all) clear32(x, bits);
    const f32x2 arg2 = join(a.score_scale, a.score_scale);
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float y0, y1;
      split(mul2(join(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), arg2), y0, y1);
      most = fmax3(most, fabsf(y0), fabsf(y1));
      x[i] = __float_as_uint(y0);
      x[i + 1] = __float_as_uint(y1);
    }
    if (__all_sync(0xffffffffu, most < vote.far)) {
      const TanhPoly<8> poly(1.f);
      const f32x2 zero2 = join(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        float y0, y1;
        split(poly(join(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), zero2), y0, y1);
        x[i] = __float_as_uint(y0);
        x[i + 1] = __float_as_uint(y1);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(tanh_any(__uint_as_float(x[i]) * (1.f / TANH_ARG)));
    }
  }
  if constexpr (MODE == BIASED) {
    const float scale = a.cap_log2 > 0.f ? a.cap_log2 : a.score_scale;
    const float dist = (float)(p - key0);            // a conversion per key would cost as much as its exponential
#pragma unroll
    for (int i = 0; i < 32; ++i)
      x[i] = __float_as_uint(fmaf(-slope, fabsf(dist - (float)i), __uint_as_float(x[i]) * scale));
  }
}

// The factor that turns transformed scores into log2 units (positive: the maximum commutes with it).
template <int MODE> __device__ __forceinline__ float scale_of(const Args& a) {
  return MODE == LINEAR ? a.score_scale : MODE == BIASED ? 1.f : a.cap_log2;
}

// Largest and smallest of 32 values (the smallest only where it is asked for).
template <bool LEAST>
__device__ __forceinline__ void range32(const uint32_t* x, float& most, float& least) {
  float t0 = most, t1 = -INFINITY, u0 = least, u1 = INFINITY;
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    t0 = fmax3(t0, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
    t1 = fmax3(t1, __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
    if constexpr (LEAST) {
      u0 = fmin3(u0, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
      u1 = fmin3(u1, __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
    }
  }
  most = fmaxf(t0, t1);
  if constexpr (LEAST) least = fminf(u0, u1);
}

// 32 raw scores in place -> arguments of the exponential under a fixed reference.  All lanes of a warp take part.
__device__ __forceinline__ void bounded32(uint32_t* x, const Args& a, const TanhPoly<5>& capped, bool all, uint32_t bits,
                                          float neg_m, const Vote& vote) {
  const f32x2 arg2 = join(a.score_scale, a.score_scale), neg2 = join(neg_m, neg_m);
  uint32_t seen = 0;
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    float y0, y1;
    split(mul2(join(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), arg2), y0, y1);
    x[i] = __float_as_uint(y0);
    x[i + 1] = __float_as_uint(y1);
    seen |= x[i] | x[i + 1];
  }
  auto all_by = [&](const auto& poly) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float e0, e1;
      split(poly(join(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), neg2), e0, e1);
      x[i] = __float_as_uint(e0);
      x[i + 1] = __float_as_uint(e1);
    }
  };
  // every |y| < 2: the top bit of the exponent is clear in all of them.  Where that fails, perhaps by unseen ones only, it
  // is looked at again without them, in code of its own: cleared in front of the first vote they cost every tile 4 %, in
  // front of a shared second one 5 % where scores beyond 3/4 of the cap are common, here 2 % (8192 tokens x 32 heads over
  // 8 x 128 capped at 20: 846 us with the unseen ones in the vote, 891, 860; capped at 50: 670 each way)
  if (__all_sync(0xffffffffu, !(seen & vote.near))) {
    all_by(capped);
  } else {
    auto beyond = [&](bool masked) {
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < 32; i += 2) most = fmax3(most, fabsf(__uint_as_float(x[i])), fabsf(__uint_as_float(x[i + 1])));
      if (masked && __all_sync(0xffffffffu, most < vote.near_most)) {
        all_by(capped);
      } else if (__all_sync(0xffffffffu, most < vote.far)) {
        all_by(TanhPoly<8>(a.cap_log2));
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          x[i] = __float_as_uint(fmaf(tanh_exp(__uint_as_float(x[i]) * (1.f / TANH_ARG)), a.cap_log2, neg_m));
      }
    };
    if (all) {
      beyond(false);
    } else {
      clear32(x, bits);
      beyond(true);
    }
  }
  if (!all) hide32(x, bits);
}

template <bool F16> __device__ __forceinline__ uint32_t pack_pair(float x, float y) {
  if constexpr (F16) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// The running reference moves (and O is rescaled) only when a score passes it by more than this many log2 units.
// fp16 holds P up to 2^(8 + 6): what underflows at its lower end is then below 2^-31 of the largest term.  bf16
// has float's range, so 24 cost no accuracy, and P V up to 2^24 * keys * |v| stays far inside it; with 8, scores of
// a spread of 9 units (6 nats) made some row of a warp rescale in every second tile.
template <bool F16> __host__ __device__ constexpr float p_bias() { return F16 ? 6.f : 0.f; }
template <bool F16> __host__ __device__ constexpr float rescale_gap() { return F16 ? 8.f : 24.f; }

// Instruction descriptor for kind::f16 with an fp32 accumulator.
template <bool F16>
__host__ __device__ constexpr uint32_t idesc_of(int m, int n, bool b_mn_major) {
  const uint32_t d = make_idesc_bf16(m, n, false, b_mn_major);
  return F16 ? d & ~((1u << 7) | (1u << 10)) : d;
}

// A row's sum of P, twice where P is bf16: as computed, for the log-sum-exp, and as rounded, which divides O.  So the
// weights sum to 1 as the products see them: a row that sees one key gives its V whatever the reference is, and
// dominant weights lose nothing.  fp16's rounding is an eighth of bf16's and is left.
template <bool F16>
struct RowSum {
  f32x2 exact[2], rounded[2];
  __device__ __forceinline__ RowSum() {
    exact[0] = exact[1] = rounded[0] = rounded[1] = join(0.f, 0.f);
  }
  __device__ __forceinline__ void add(int i, float e0, float e1, uint32_t packed) {
    exact[i & 1] = add2(exact[i & 1], join(e0, e1));
    if constexpr (!F16)
      rounded[i & 1] = add2(rounded[i & 1], join(__uint_as_float(packed << 16), __uint_as_float(packed & 0xffff0000u)));
  }
  __device__ __forceinline__ void into(float& l, float& lr) const {
    float x, y;
    split(add2(exact[0], exact[1]), x, y);
    l += x + y;
    if constexpr (F16) { lr = l; return; }
    split(add2(rounded[0], rounded[1]), x, y);
    lr += x + y;
  }
};

// A warp's share of the output: each lane holds 32 values of its row (16-byte pieces piece0 ... + 3 as packed
// words) and has put them into `stage` (32 rows of PIECES 16-byte pieces, permuted so that neither side
// collides); this writes `rows` rows of it, PIECES lanes to a row, so that whole lines leave at once.
template <int PIECES>
__device__ __forceinline__ void stage_pieces(uint8_t* stage, int piece0, const uint32_t (&w)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    reinterpret_cast<uint4*>(stage)[lane * PIECES + ((piece0 + i) ^ (lane & (PIECES - 1)))] =
        make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}

// Zero rows [from, to) of a swizzled 128-byte-row tile of D columns (all of a row, so the permutation inside it
// does not matter).  One warp; the caller fences before the tensor core reads.
template <int D, int BN>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from, int to) {
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < (to - from) * 8 * (D / 64); i += 32) {
    const int slab = i / ((to - from) * 8), r = i % ((to - from) * 8);
    reinterpret_cast<uint4*>(tile + slab * BN * 128 + (from + r / 8) * 128)[r % 8] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// 32 accumulators of a lane's row from tensor memory to its partial.  Warp-collective; `keep`: the row exists.
__device__ __forceinline__ void store_partial(uint32_t tmem, float* to, bool keep) {
  uint32_t o[32];
  tmem_ld32(tmem, o);
  tmem_ld_wait();
  if (keep) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      reinterpret_cast<uint4*>(to)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
  }
}

// Joins the pieces of a tile: blockIdx.x is its share without a split; 8 dimensions of a row per thread.
template <int D, int BN, bool F16>
__global__ void __launch_bounds__(256) join_pieces_kernel(const Args a) {
  __shared__ __align__(8) uint8_t scratch[FIND_BYTES];
  const Share share(a, 1);
  const Tile tile = a.docs <= WARP_DOCS ? find_tile(a, share.want) : find_tile_block<256>(a, share.want, scratch);
  pdl_wait();                                        // every block waits: this launch must not end before the other
  if (tile.doc < 0) return;
  const KeyTiles<BN> keys(a, tile);
  const int pieces = pieces_of(a, keys.n, BN);
  if (pieces == 1) return;
  const float* first = share.record(a, D, 0);
  constexpr int CH = D / 8;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < tile.count * a.group * CH; i += gridDim.y * 256) {
    const int r = i / CH, c = i - r * CH;
    float m = -INFINITY;
    for (int s = 0; s < pieces; ++s) m = fmaxf(m, __ldcg(first + s * record_floats(D) + 128 * D + r));
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, l = 0.f, lr = 0.f;
#pragma unroll 4
    for (int s = 0; s < pieces; ++s) {
      const float* record = first + s * record_floats(D);
      const float ms = __ldcg(record + 128 * D + r), f = ms == m ? 1.f : fast_exp2(ms - m);
      const float4 x = __ldcg(reinterpret_cast<const float4*>(record + r * D + c * 8));
      const float4 y = __ldcg(reinterpret_cast<const float4*>(record + r * D + c * 8) + 1);
      l += f * __ldcg(record + 128 * D + 128 + r);
      lr += f * __ldcg(record + 128 * D + 256 + r);
      acc[0] += f * x.x; acc[1] += f * x.y; acc[2] += f * x.z; acc[3] += f * x.w;
      acc[4] += f * y.x; acc[5] += f * y.y; acc[6] += f * y.z; acc[7] += f * y.w;
    }
    const float inv = lr == 0.f ? 0.f : 1.f / lr;
    const int q = r / a.group;
    const int64_t at = (tile.token + q) * a.num_q_heads + share.h * a.group + r - q * a.group;
    uint4 w;
    w.x = pack_pair<F16>(acc[0] * inv, acc[1] * inv);
    w.y = pack_pair<F16>(acc[2] * inv, acc[3] * inv);
    w.z = pack_pair<F16>(acc[4] * inv, acc[5] * inv);
    w.w = pack_pair<F16>(acc[6] * inv, acc[7] * inv);
    if (lr == 0.f) w = make_uint4(0u, 0u, 0u, 0u);
    reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at * D)[c] = w;
    if (a.lse && c == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + __log2f(l) - p_bias<F16>()) * LN2F;
  }
}

}  // namespace dense
