// Rotary positions: q_post, k_post from q_pre, k_pre (the layer keeps both: routing reads the
// vectors before the rotation, attention the ones after it).
//
//   angle(t, i) = position_t * f_i,  c = a cos(angle), s = a sin(angle)   (a: the attention scale)
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s                                   (inverse: s -> -s)
//
// with (x1, x2) = (x_i, x_{i + R/2}) in the half layout and (x_2i, x_2i+1) in the interleaved one;
// dimensions from R on are copied.  Frequencies are doubles and the angle is reduced to a fraction of a
// turn in double: at position 1e6 and f = 1 a float product is off by up to 0.03 radians, which no later step
// can repair.  sincospi takes the fraction rounded to a float (off by up to 2^-25 of a half turn, 1e-7 radians); the rest of
// it turns the result once more, to first order (its square is below 2^-46).
//
// Bound: HBM, one read and one write of every element.  A cos/sin costs ~50 instructions and serves all
// heads of a token, so a block walks over tiles of whole tokens and keeps two of everything: while a thread
// turns the rows it holds, its next rows (2 x 16 bytes each, 2 rows) travel and the next tile's cos/sin go
// to the other half of shared memory; one barrier per tile.  A block per token instead of a walk spent a
// third of its time waiting at that barrier for a chain of divisions, position loads and sines.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../../include/semblo_b200.h"
#include "host_common.h"

using semblo::ceil_div;

namespace {

constexpr int THREADS = 256;
constexpr int MAX_HEAD_DIM = 512;           // a block holds the columns of one row at least

struct RotaryArgs {
  // scalars, not arrays of two: a select between array elements becomes a constant-bank load with an index
  // that differs in the warp, and those serialise (half of all issue slots of an earlier form)
  const void *q_in, *k_in;
  void *q_out, *k_out;
  int64_t q_in_token, q_in_head, q_out_token, q_out_head;       // strides in elements
  int64_t k_in_token, k_in_head, k_out_token, k_out_head;
  int heads0, heads;            // query heads, query + key heads
  int64_t tokens;
  int tokens_per_block, head_lanes;     // threads per block: tokens x head lanes x columns
  int head_dim, rotary_dim;
  int cols;                     // threads per (token, head): rotating columns, then copying ones
  int rot_cols;
  const void* positions;
  int pos64;
  const double* inv_freq;
  float scale;                  // on cos and sin
  float sin_sign;
};

// A pack is NP elements held as 32-bit words (16-bit elements two to a word), or one element (NP = 1).
template <typename T, int NP>
struct alignas(NP * sizeof(T) >= 16 ? 16 : NP * sizeof(T)) Pack { uint32_t w[NP * sizeof(T) / 4]; };
template <typename T> struct Pack<T, 1> { T v; };

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
  const __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// (x1, x2) <- (x1 c - x2 s, x2 c + x1 s) for the NP pairs of two packs; t(i) is pair i's (c, s).
template <typename T, int NP, bool INTERLEAVED, typename F>
__device__ __forceinline__ void turn_packs(Pack<T, NP>& p0, Pack<T, NP>& p1, F t) {
  if constexpr (NP == 1) {
    const float x = static_cast<float>(p0.v), y = static_cast<float>(p1.v);
    const float2 cs = t(0);
    p0.v = static_cast<T>(x * cs.x - y * cs.y);
    p1.v = static_cast<T>(y * cs.x + x * cs.y);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      uint32_t& a = INTERLEAVED ? (i < NP / 2 ? p0.w[2 * i] : p1.w[2 * i - NP]) : p0.w[i];
      uint32_t& b = INTERLEAVED ? (i < NP / 2 ? p0.w[2 * i + 1] : p1.w[2 * i + 1 - NP]) : p1.w[i];
      const float x = __uint_as_float(a), y = __uint_as_float(b);
      const float2 cs = t(i);
      a = __float_as_uint(x * cs.x - y * cs.y);
      b = __float_as_uint(y * cs.x + x * cs.y);
    }
  } else if constexpr (INTERLEAVED) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      uint32_t& a = i < NP / 2 ? p0.w[i] : p1.w[i - NP / 2];
      const float2 x = unpack2<T>(a), cs = t(i);
      a = pack2<T>(x.x * cs.x - x.y * cs.y, x.y * cs.x + x.x * cs.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NP; i += 2) {
      const float2 x = unpack2<T>(p0.w[i / 2]), y = unpack2<T>(p1.w[i / 2]);
      const float2 c0 = t(i), c1 = t(i + 1);
      p0.w[i / 2] = pack2<T>(x.x * c0.x - y.x * c0.y, x.y * c1.x - y.y * c1.y);
      p1.w[i / 2] = pack2<T>(y.x * c0.x + x.x * c0.y, y.y * c1.x + x.y * c1.y);
    }
  }
}

constexpr int AHEAD = 2;        // rows of a thread that travel together

// NP: pairs per thread and row.  A rotating column c covers the pairs [NP c, NP (c + 1)): two packs of NP
// elements, R/2 apart (half) or adjacent (interleaved).  A copying column covers 2 NP elements from R on
// (NP = 1: two single elements, the second may lie past the head).
template <typename T, int NP, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS, NP * sizeof(T) > 16 ? 2 : 3) rotary_kernel(const RotaryArgs a) {
  // cos, sin: [buffer][token][i][column] for pair NP column + i, so that a warp's reads do not collide
  extern __shared__ float2 turn[];
  const int pairs = a.rotary_dim >> 1;
  const int tile_pairs = a.tokens_per_block * pairs;
  const int row = threadIdx.x / a.cols, col = threadIdx.x - row * a.cols;
  const int tk = row / a.head_lanes, lane = row - tk * a.head_lanes;
  const bool mine = tk < a.tokens_per_block, rotating = col < a.rot_cols;
  const int e0 = rotating ? (INTERLEAVED ? 2 * NP * col : NP * col) : a.rotary_dim + 2 * NP * (col - a.rot_cols);
  int step = rotating && !INTERLEAVED ? pairs : NP;            // to the second pack; 0 at the odd end of a tail
  if (e0 + step + NP > a.head_dim) step = 0;
  const int span = AHEAD * a.head_lanes;                       // heads of one batch
  const int64_t advance = (int64_t)gridDim.x * a.tokens_per_block;

  struct Batch { Pack<T, NP> x0[AHEAD], x1[AHEAD]; };
  auto load = [&](Batch& b, int64_t token, int h0) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int h = h0 + u * a.head_lanes;
      if (h < a.heads) {
        const bool key = h >= a.heads0;
        const T* src = (key ? static_cast<const T*>(a.k_in) + token * a.k_in_token + (h - a.heads0) * a.k_in_head
                            : static_cast<const T*>(a.q_in) + token * a.q_in_token + h * a.q_in_head) + e0;
        b.x0[u] = *reinterpret_cast<const Pack<T, NP>*>(src);
        b.x1[u] = *reinterpret_cast<const Pack<T, NP>*>(src + step);
      }
    }
  };
  auto angles = [&](float2* buf, int64_t token0) {
    for (int i = threadIdx.x; i < tile_pairs; i += THREADS) {
      const int t = a.tokens_per_block == 1 ? 0 : i / pairs, p = i - t * pairs;
      if (token0 + t >= a.tokens) break;
      const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[token0 + t]
                                 : (double)static_cast<const int32_t*>(a.positions)[token0 + t];
      double turns = pos * a.inv_freq[p] * 0.15915494309189535;      // 1 / (2 pi)
      turns -= rint(turns);
      const double half_turns = 2.0 * turns;
      const float whole = (float)half_turns, rest = (float)((half_turns - whole) * 3.14159265358979324);
      float s0, c0;
      sincospif(whole, &s0, &c0);
      const float cs = fmaf(-s0, rest, c0), sn = fmaf(c0, rest, s0);
      buf[t * pairs + (p % NP) * a.rot_cols + p / NP] = make_float2(cs * a.scale, sn * a.scale * a.sin_sign);
    }
  };

  int64_t token0 = (int64_t)blockIdx.x * a.tokens_per_block;
  Batch now, next;
  if (mine && token0 + tk < a.tokens) load(now, token0 + tk, lane);
  angles(turn, token0);
  __syncthreads();
  for (int half = 0; token0 < a.tokens; token0 += advance, half ^= 1) {
    const int64_t token = token0 + tk;
    const bool have = mine && token < a.tokens;
    const bool more = mine && token + advance < a.tokens;
    float2 cs[NP];
    if (rotating) {
      const float2* c = turn + half * tile_pairs + (mine ? tk : 0) * pairs + col;
#pragma unroll
      for (int i = 0; i < NP; ++i) cs[i] = c[i * a.rot_cols];
    }
    for (int h0 = lane; h0 < a.heads; h0 += span) {
      if (h0 + span < a.heads) {
        if (have) load(next, token, h0 + span);
      } else if (more) {
        load(next, token + advance, lane);
      }
      if (have) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int h = h0 + u * a.head_lanes;
          if (h < a.heads) {
            if (rotating) turn_packs<T, NP, INTERLEAVED>(now.x0[u], now.x1[u], [&](int i) { return cs[i]; });
            const bool key = h >= a.heads0;
            T* dst = (key ? static_cast<T*>(a.k_out) + token * a.k_out_token + (h - a.heads0) * a.k_out_head
                          : static_cast<T*>(a.q_out) + token * a.q_out_token + h * a.q_out_head) + e0;
            *reinterpret_cast<Pack<T, NP>*>(dst) = now.x0[u];
            if (step) *reinterpret_cast<Pack<T, NP>*>(dst + step) = now.x1[u];
          }
        }
      }
      now = next;
    }
    if (token0 + advance < a.tokens) angles(turn + (half ^ 1) * tile_pairs, token0 + advance);
    __syncthreads();
  }
}

template <typename T, int NP>
int launch(RotaryArgs& a, bool interleaved, cudaStream_t st) {
  a.rot_cols = a.rotary_dim / (2 * NP);
  a.cols = a.rot_cols + (int)ceil_div(a.head_dim - a.rotary_dim, 2 * NP);
  // a block's threads are tokens x head lanes x columns: the split that leaves the fewest of them idle, with no more
  // tokens than leave two blocks for every multiprocessor
  const int rows = THREADS / a.cols;
  const int sms = semblo::sm_count();
  const int most_tokens = (int)std::min<int64_t>(std::max(1, 1024 / std::max(1, a.rotary_dim / 2)),   // 2 x 8 KB of cos/sin
                                                 std::max<int64_t>(1, a.tokens / (2 * sms)));
  int tb = 1, lanes = std::min(rows, a.heads);
  double best = 0;
  for (int l = 1; l <= std::min(rows, a.heads); ++l) {
    const int t = std::min(rows / l, most_tokens);
    const int64_t slots = ceil_div(ceil_div(a.heads, l), AHEAD) * AHEAD;
    const double used = (double)t * a.heads / ((double)rows * slots);
    if (used >= best) { best = used; tb = t; lanes = l; }
  }
  a.tokens_per_block = tb;
  a.head_lanes = lanes;
  const size_t smem = 2 * (size_t)tb * (a.rotary_dim / 2) * sizeof(float2);
  // many more blocks than fit at once, each with a handful of tiles: with one resident wave the blocks step
  // through memory in lockstep (131072 tokens x 20 heads x 256: 398 us at 64 per multiprocessor, 415 at 16, 500
  // at 3; 8192 x 40 x 128: 30.8, 30.9 and 30.3)
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(a.tokens, tb), (int64_t)sms * 64);
  if (interleaved) rotary_kernel<T, NP, true><<<grid, THREADS, smem, st>>>(a);
  else rotary_kernel<T, NP, false><<<grid, THREADS, smem, st>>>(a);
  SEMBLO_LAUNCH_CHECK();
  return 0;
}

// The widest pack that every row start and every pack offset allows.
template <typename T>
int dispatch(RotaryArgs& a, bool interleaved, cudaStream_t st) {
  uint64_t bits = 0;                                 // of every byte offset that a row can start at
  bits |= (uint64_t)(uintptr_t)a.q_in | (uint64_t)(uintptr_t)a.q_out | (uint64_t)(uintptr_t)a.k_in |
          (uint64_t)(uintptr_t)a.k_out;
  bits |= (uint64_t)(a.q_in_token | a.q_in_head | a.q_out_token | a.q_out_head) * sizeof(T);
  if (a.k_in) bits |= (uint64_t)(a.k_in_token | a.k_in_head | a.k_out_token | a.k_out_head) * sizeof(T);
  auto fits = [&](int np) {
    const uint64_t align = std::min<uint64_t>(16, np * sizeof(T));
    return a.rotary_dim % (2 * np) == 0 && a.head_dim % (2 * np) == 0 && bits % align == 0;
  };
  if (fits(8)) return launch<T, 8>(a, interleaved, st);
  if (fits(4)) return launch<T, 4>(a, interleaved, st);
  return launch<T, 1>(a, interleaved, st);
}

// ---------------------------------------------------------------- which rows share memory
// The dimensions of [tokens, heads, head_dim] that move, widest step first, in bytes.
struct Steps {
  int n = 0;
  bool still = false;             // a dimension of several indices does not move
  int64_t count[3], step[3];
  void add(int64_t c, int64_t s) {
    if (c <= 1) return;
    if (s == 0) { still = true; return; }
    int i = n++;
    for (; i > 0 && step[i - 1] < s; --i) { count[i] = count[i - 1]; step[i] = step[i - 1]; }
    count[i] = c;
    step[i] = s;
  }
  int64_t extent(int from, int64_t size) const {
    int64_t e = size;
    for (int i = from; i < n; ++i) e += (count[i] - 1) * step[i];
    return e;
  }
};

struct Rows {
  const char* at;
  Steps steps;
  Rows(const void* p, int64_t tokens, int64_t token_stride, int heads, int64_t head_stride, int head_dim, int size)
      : at(static_cast<const char*>(p)) {
    steps.add(tokens, token_stride * size);
    steps.add(heads, head_stride * size);
    steps.add(head_dim, size);
  }
};

// Whether elements of a, from dimension ia on, and of b, `offset` bytes on, meet.  Slices of one fused buffer, whose
// spans overlap, are told apart; rows that reach into each other count as meeting.
bool meet(int64_t offset, const Steps& a, int ia, const Steps& b, int ib, int64_t size) {
  if (offset >= a.extent(ia, size) || -offset >= b.extent(ib, size)) return false;
  if (ia == a.n && ib == b.n) return true;
  const int64_t step = std::max(ia < a.n ? a.step[ia] : 0, ib < b.n ? b.step[ib] : 0);
  int64_t na = 1, nb = 1;
  if (ia < a.n && a.step[ia] == step) na = a.count[ia++];
  if (ib < b.n && b.step[ib] == step) nb = b.count[ib++];
  const int64_t ea = a.extent(ia, size), eb = b.extent(ib, size);
  if (ea > step || eb > step) return true;
  // row i of a starts at i steps, row j of b at offset + j steps: they meet for -eb < offset + (j - i) steps < ea only,
  // which is at most three values of j - i
  auto below = [&](int64_t x) { return x >= 0 ? x / step : -((-x + step - 1) / step); };
  const int64_t last = std::min(nb - 1, below(ea - offset - 1));
  for (int64_t k = std::max(1 - na, below(-eb - offset) + 1); k <= last; ++k)
    if (meet(offset + k * step, a, ia, b, ib, size)) return true;
  return false;
}
bool meet(const Rows& a, const Rows& b, int64_t size) { return meet(b.at - a.at, a.steps, 0, b.steps, 0, size); }

bool repeats(const Rows& a, int64_t size) {
  if (a.steps.still) return true;
  for (int i = 0; i < a.steps.n; ++i)
    if (a.steps.extent(i + 1, size) > a.steps.step[i]) return true;
  return false;
}

}  // namespace

extern "C" int semblo_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                             int64_t qo_token_stride, int64_t qo_head_stride, int num_q_heads, const void* k,
                             int64_t k_token_stride, int64_t k_head_stride, void* k_out,
                             int64_t ko_token_stride, int64_t ko_head_stride, int num_kv_heads, int64_t tokens,
                             int head_dim, int rotary_dim, int dtype, const void* positions, int pos_is_int64,
                             const double* inv_freq, float attention_scale, int interleaved, int inverse,
                             void* stream) {
  SEMBLO_REQUIRE(tokens >= 0 && num_q_heads > 0 && num_kv_heads >= 0, "bad token or head count");
  SEMBLO_REQUIRE(rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
                 "rotary_dim must be even and at most head_dim (got %d of %d)", rotary_dim, head_dim);
  SEMBLO_REQUIRE(head_dim > 0 && head_dim <= MAX_HEAD_DIM, "head_dim must be at most %d (got %d)", MAX_HEAD_DIM, head_dim);
  SEMBLO_REQUIRE((k == nullptr) == (k_out == nullptr), "k and k_out come together");
  if (tokens == 0) return 0;
  SEMBLO_REQUIRE(q != nullptr && q_out != nullptr && positions != nullptr, "q, q_out and positions are required");
  SEMBLO_REQUIRE(rotary_dim == 0 || inv_freq != nullptr, "inv_freq is required");
  SEMBLO_REQUIRE(tokens < (int64_t)1 << 31, "too many tokens");
  SEMBLO_REQUIRE(std::min({q_token_stride, q_head_stride, qo_token_stride, qo_head_stride}) >= 0 &&
                     (!k || std::min({k_token_stride, k_head_stride, ko_token_stride, ko_head_stride}) >= 0),
                 "strides must not be negative");
  // one launch turns query and key heads in any order
  const int size = dtype == SEMBLO_F32 ? 4 : 2;
  const Rows qi(q, tokens, q_token_stride, num_q_heads, q_head_stride, head_dim, size);
  const Rows qo(q_out, tokens, qo_token_stride, num_q_heads, qo_head_stride, head_dim, size);
  SEMBLO_REQUIRE(!repeats(qo, size), "q_out must not repeat memory");
  SEMBLO_REQUIRE((q == q_out && q_token_stride == qo_token_stride && q_head_stride == qo_head_stride) || !meet(qi, qo, size),
                 "q_out overlaps its input without being it");
  if (k && num_kv_heads) {
    const Rows ki(k, tokens, k_token_stride, num_kv_heads, k_head_stride, head_dim, size);
    const Rows ko(k_out, tokens, ko_token_stride, num_kv_heads, ko_head_stride, head_dim, size);
    SEMBLO_REQUIRE(!repeats(ko, size), "k_out must not repeat memory");
    SEMBLO_REQUIRE((k == k_out && k_token_stride == ko_token_stride && k_head_stride == ko_head_stride) || !meet(ki, ko, size),
                   "k_out overlaps its input without being it");
    SEMBLO_REQUIRE(!meet(qo, ki, size) && !meet(ko, qi, size) && !meet(qo, ko, size),
                   "q_out and k_out must not overlap each other or the other's input");
  }
  RotaryArgs a{};
  a.q_in = q; a.q_out = q_out; a.k_in = k; a.k_out = k_out;
  a.q_in_token = q_token_stride; a.q_in_head = q_head_stride;
  a.q_out_token = qo_token_stride; a.q_out_head = qo_head_stride;
  a.k_in_token = k_token_stride; a.k_in_head = k_head_stride;
  a.k_out_token = ko_token_stride; a.k_out_head = ko_head_stride;
  a.heads0 = num_q_heads;
  a.heads = num_q_heads + (k ? num_kv_heads : 0);
  a.tokens = tokens;
  a.head_dim = head_dim; a.rotary_dim = rotary_dim;
  a.positions = positions; a.pos64 = pos_is_int64;
  a.inv_freq = inv_freq;
  a.scale = attention_scale;
  a.sin_sign = inverse ? -1.f : 1.f;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == SEMBLO_BF16) return dispatch<__nv_bfloat16>(a, interleaved, st);
  if (dtype == SEMBLO_F16) return dispatch<__half>(a, interleaved, st);
  if (dtype == SEMBLO_F32) return dispatch<float>(a, interleaved, st);
  return semblo::fail(semblo::SEMBLO_EINVAL, "rotary takes bf16, fp16 or fp32 (got dtype code %d)", dtype);
}
