// Attention of generated tokens over the 8-bit paged K/V cache (one query, or a few, per request).
//
//   s_j = cap tanh(q . k_j sm / cap)  (or q . k_j sm) - slope |p - j|,  k_j = code_j * k_scale(block of j)
//   o   = sum_j 2^(s_j log2e - m) v_j / sum_j 2^(s_j log2e - m),          p = length - queries + query index
//   key j is seen when j < length and ((j <= p and p - j < window) or j < prefix).
//
// Bound: HBM, 2 D bytes per key and KV head.  What has to keep up with 24 bytes per clock and
// multiprocessor is the way of a byte through it:
//   * a warp takes 16 keys at a time through a private ring in shared memory, copied (cp.async) in the order
//     of memory, 512 consecutive bytes an instruction: the same copies with each lane fetching the pieces that
//     it will need itself reached 4.7 TB/s, in memory order 6.2.  The 16-byte pieces are permuted inside their
//     128-byte lines so that the fragments are read back without bank conflicts;
//   * e4m3 becomes fp16 by the hardware's pair conversion and is exact there, as is the query after a power
//     of two per row is taken out (bf16 elements down to 2^-16 of the row's largest, fp16 ones down to 2^-13; fp16 ends at
//     2^-24, so that a smaller one is off by 2^-24 of the largest at most, a 32-bit sum's own rounding).  The products
//     S^T = K Q^T of m16n8k16 are exact up to that and the fp32 sums.
//     The order of the 16 values inside a k-step is free as long as K and Q agree: a lane's 16 consecutive
//     bytes are its elements of four k-steps.  The same freedom over the rows of O^T = V^T P^T turns 16
//     consecutive bytes of four keys into eight A fragments with two byte permutes per four values;
//   * P^T is S^T's accumulator transposed by movmatrix; heads are the n dimension of both products, so that
//     8 rows (queries x heads of a KV head) cost one n-tile.  A row tile has up to four of them (two at D = 256, where
//     O fills the registers): 80 x 3071 keys x 8 heads x 64 with 24 rows each 166 us in tiles of 16, 104 in one of 24
//     (90 in two blocks of four warps per multiprocessor instead of one of eight).
//     There the latency of the products and the softmax between them bounds it, not HBM.
// V's scale changes from block to block, so P carries it: P' = 2^(s + log2 scale - M + 11) in fp16 with its own
// running reference M next to the softmax's m (a block of large values with little weight must not push the
// others under fp16's range).  Both move only when a score passes them by 2^4: P' stays below 2^15, and what
// fp16 drops at its lower end is below 2^-36 of the largest term.
//
// Work is split evenly whatever the lengths: the 16-key groups of all (request, KV head, row tile) segments
// form one line, every block takes an equal piece of it, writes the segments that lie inside its piece and
// leaves partials of those that do not; a second launch (a programmatic dependent) merges them.  Where the
// lengths turn out short, blocks take whole segments, and where the table allows no segment of more than
// 8 groups per warp of a block, there is no second launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../../include/semblo_b200.h"
#include "host_common.h"
#include "sm100.cuh"

using semblo::ceil_div;

namespace {

constexpr int GROUP = 16;                 // keys per step of a warp
constexpr int DIRECT_STEPS = 8;           // steps of a block's warps that one block takes for a whole segment
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float GAP = 4.f;                // log2 units by which a score may pass a reference
constexpr float P_BIAS = 11.f;            // P' reaches 2^(P_BIAS + GAP) = 2^15

struct DecodeArgs {
  const void* q;                          // [B, n, Hq, D]
  int q_f16;
  void* out;                              // as q
  float* lse;                             // [B, n, Hq] or null
  const uint8_t* data;                    // [2, blocks, Hkv, block, D]
  const float* scales;                    // [2, blocks, Hkv]
  int64_t cache_blocks;
  int block_log2;
  const int32_t* table;
  int64_t table_stride;
  int table_len;
  const int32_t* lengths;                 // [B]
  const int32_t* prefix;                  // [B] or null
  const float* slopes;                    // [Hq] or null
  int batch, queries, num_q_heads, num_kv_heads, group;     // group: query heads per KV head
  int rows, row_tiles;                    // queries * group, tiles of 8 NT rows
  int window;                             // 0: none
  float sm_scale, softcap;
  int direct;
  float* partial;                         // [grid][2][record]
  int* status;
};

// ---------------------------------------------------------------- pieces
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Two e4m3 codes (low byte first) to two fp16.
__device__ __forceinline__ uint32_t widen_lo(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(d) : "r"(w));
  return d;
}
__device__ __forceinline__ uint32_t widen_hi(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(d) : "r"(w));
  return d;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t half2_bits(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 2^(a - b) where equal references (both -inf among them) give 1.
__device__ __forceinline__ float ratio2(float a, float b) { return a == b ? 1.f : sm100::fast_exp2(a - b); }

// The groups of one request: prefix groups [0, gp), then [glo, ...).
struct Span {
  int length, first, lo, prefix;          // keys, position of the first query, first key of the window, prefix keys
  int gp, glo, groups;
  __device__ __forceinline__ int group_of(int i) const { return i < gp ? i : i - gp + glo; }
};

__device__ __forceinline__ Span span_of(const DecodeArgs& a, int b) {
  Span s;
  const int64_t room = (int64_t)a.table_len << a.block_log2;
  const int given = a.lengths[b];
  s.length = (int)min((int64_t)max(given, 0), room);
  s.first = given - a.queries;
  s.prefix = a.prefix ? min(max(a.prefix[b], 0), s.length) : 0;
  s.lo = a.window > 0 ? max(0, s.first - a.window + 1) : 0;
  s.gp = (s.prefix + GROUP - 1) / GROUP;
  const int end = (s.length + GROUP - 1) / GROUP;
  s.glo = min(max(s.gp, s.lo / GROUP), end);
  s.groups = s.gp + end - s.glo;
  return s;
}

template <int D, int NT>
struct Cfg {
  static constexpr int STAGES = D == 256 ? 3 : D == 128 ? (NT > 2 ? 4 : 3) : 4;
  // two blocks per multiprocessor, of fewer warps where their registers are many (and the ring is large)
  static constexpr int WARPS = D == 256 || NT > 2 || (D == 128 && NT == 2) ? 4 : 8;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int PER_SM = 2;
  static constexpr int DIRECT = DIRECT_STEPS * WARPS;           // groups
  static constexpr int KV_BYTES = GROUP * D;                    // K or V of a group
  static constexpr int RING = STAGES * 2 * KV_BYTES;            // per warp
  static constexpr int KC = D / 32;                             // 16-byte pieces of K per lane
  static constexpr int VI = D == 256 ? 2 : 1;                   // pieces of V per lane and key (16 bytes, 8 for D = 64)
  static constexpr int KSTEPS = D / 16;
  static constexpr int ROWS = 8 * NT;
  static constexpr bool Q_SMEM = D * NT > 256;                  // the query's fragments do not fit in registers
  static constexpr int ACC = KSTEPS * NT * 4;                   // accumulators of O^T per lane
  static constexpr int RECORD = ACC * 32 + 3 * ROWS;            // floats: O fragments, then m, M, l of each row
  static constexpr int META_OFF = WARPS * RING;                 // float [WARPS][STAGES][2]: the group's scales
  static constexpr int ML_OFF = META_OFF + WARPS * STAGES * 8;  // float [3][WARPS][ROWS]
  static constexpr int FAC_OFF = ML_OFF + 3 * WARPS * ROWS * 4; // float [WARPS][ROWS] factors, [3][ROWS] totals
  static constexpr int Q_OFF = FAC_OFF + (WARPS + 3) * ROWS * 4;
  static constexpr int SUM_OFF = Q_OFF + (Q_SMEM ? KSTEPS * NT * 32 * 8 : 0);   // int [batch + 1], then [2 WARPS + 1]
  static_assert(ACC * 32 * 4 <= RING, "a warp's O must fit its ring");
};

// Inclusive sums of groups * segments-per-request over the batch into sums[1 ...]; sums[0] = 0.  Returns the most
// groups of a segment.
__device__ __forceinline__ int line_sums(const DecodeArgs& a, int segs, int* sums, int* scratch) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  int carry = 0, longest = 0;
  for (int b0 = 0; b0 < a.batch; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    const int groups = b < a.batch ? span_of(a, b).groups : 0;
    longest = max(longest, groups);
    int v = groups * segs;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += t;
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 31) { scratch[warp] = v; scratch[warps + warp] = longest; }
    __syncthreads();
    int before = carry;
    for (int w = 0; w < warps; ++w) {
      const int t = scratch[w];
      if (w < warp) before += t;
      carry += t;
      longest = max(longest, scratch[warps + w]);
    }
    if (b < a.batch) sums[b + 1] = before + v;
    __syncthreads();
  }
  if (threadIdx.x == 0) sums[0] = 0;
  __syncthreads();
  return longest;
}

// Groups of a block's piece: no fewer than give each of its warps one.
__device__ __forceinline__ int quota_of(int total, int blocks, int warps) {
  return max(warps, (total + blocks - 1) / blocks);
}

// Whether a block takes whole segments: where the rounds that this needs cost less than even pieces with their
// merge, which is worth `direct` groups.  Tables are as wide as the longest request may grow, so that what
// the launch is sized for says little about the lengths in it.
__device__ __forceinline__ bool takes_whole(int segments, int longest, int quota, int blocks, int direct) {
  return (int64_t)((segments + blocks - 1) / blocks) * longest <= quota + direct;
}

// Element e of a record in fragment order -> row of the tile and dimension.
template <int D, int NT>
__device__ __forceinline__ void element_of(int e, int& row, int& dim) {
  const int lane = e & 31, c = (e >> 5) & 3, j = (e >> 7) % (D / 16), nt = (e >> 7) / (D / 16);
  const int g = lane >> 2, t = lane & 3;
  row = nt * 8 + 2 * t + (c & 1);
  const int x = 2 * j + (c >> 1);                               // which of the lane's values of V
  if constexpr (D == 64) dim = 8 * g + x;
  else dim = 16 * g + (x & 15) + 128 * (x >> 4);
}

// Row of the output [B, n, Hq] of row `row` (query, head of the group) of KV head h.
__device__ __forceinline__ int64_t output_row(const DecodeArgs& a, int b, int h, int row) {
  const int qi = row / a.group;
  return ((int64_t)b * a.queries + qi) * a.num_q_heads + h * a.group + row - qi * a.group;
}

// From the sum of P' codes to the output, by the references.
__device__ __forceinline__ float finish_factor(float m, float mv, float l) {
  return sm100::fast_exp2(mv - m - P_BIAS) / l;
}

// ---------------------------------------------------------------- attention
template <int D, int NT, bool CAP>
__global__ void __launch_bounds__((Cfg<D, NT>::THREADS), (Cfg<D, NT>::PER_SM)) kv8_decode_kernel(const DecodeArgs a) {
  using C = Cfg<D, NT>;
  constexpr int WARPS = C::WARPS, THREADS = C::THREADS;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  int* sums = reinterpret_cast<int*>(smem + C::SUM_OFF);
  int* scratch = sums + a.batch + 1;
  float* meta = reinterpret_cast<float*>(smem + C::META_OFF) + warp * C::STAGES * 2;
  float* ml = reinterpret_cast<float*>(smem + C::ML_OFF);
  float* factors = reinterpret_cast<float*>(smem + C::FAC_OFF);
  float* totals = factors + WARPS * C::ROWS;
  uint2* q_frag = reinterpret_cast<uint2*>(smem + C::Q_OFF);
  uint8_t* ring = smem + warp * C::RING;
  const uint32_t ring_u32 = sm100::smem_u32(ring), meta_u32 = sm100::smem_u32(meta);
  const int segs = a.num_kv_heads * a.row_tiles;

  // positions are segments where blocks take whole ones, groups on the line otherwise
  int pos = blockIdx.x, end = a.batch * segs;
  int* const whole = scratch + 2 * WARPS;                           // read again for every segment: no register through its loop
  if (!a.direct) {
    const int longest = line_sums(a, segs, sums, scratch), total = sums[a.batch], quota = quota_of(total, gridDim.x, WARPS);
    const bool w = takes_whole(end, longest, quota, gridDim.x, C::DIRECT);
    if (threadIdx.x == 0) *whole = w;
    __syncthreads();
    if (!w) {
      pos = (int)min((int64_t)total, (int64_t)blockIdx.x * quota);
      end = min(total, pos + quota);
    }
  }

  while (pos < end) {
    // ---- the segment at pos
    int b, seg, i0, i1;
    Span sp;
    if (a.direct || *whole) {
      b = pos / segs; seg = pos - b * segs;
      sp = span_of(a, b);
      i0 = 0; i1 = sp.groups;
      pos += gridDim.x;
    } else {
      int lo = 0, hi = a.batch;                                 // the last request that starts at or before pos
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= pos) lo = mid; else hi = mid;
      }
      b = lo;
      sp = span_of(a, b);
      const int off = pos - sums[b];
      seg = off / sp.groups;
      i0 = off - seg * sp.groups;
      i1 = min(sp.groups, i0 + end - pos);
      pos += i1 - i0;
    }
    const int h = seg / a.row_tiles, row0 = (seg - h * a.row_tiles) * C::ROWS;
    if (a.lengths[b] > sp.length && threadIdx.x == 0) atomicCAS(a.status, 0, sm100::STATUS_OVERFLOW);

    // ---- the query's rows, on their way while the first groups are looked up
    uint2 raw[NT][C::KSTEPS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + nt * 8 + g;
      const bool have = r < a.rows;
      const int qi = have ? r / a.group : 0;
      const int64_t qrow = ((int64_t)b * a.queries + qi) * a.num_q_heads + h * a.group + (have ? r - qi * a.group : 0);
#pragma unroll
      for (int s = 0; s < C::KSTEPS; ++s) {
        raw[nt][s] = make_uint2(0u, 0u);
        if (have) raw[nt][s] = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) + qrow * D +
                                                                    64 * (s >> 2) + 16 * t + 4 * (s & 3)));
      }
    }

    // ---- pipeline over this warp's groups
    const int count = max(0, (i1 - i0 - warp + WARPS - 1) / WARPS);
    const int64_t table_row = (int64_t)b * a.table_stride;
    // the table entry of the group to be issued next is read while the one before it is issued
    auto page_for = [&](int it) -> int {
      if (it >= count) return 0;
      return a.table[table_row + ((sp.group_of(i0 + warp + it * WARPS) * GROUP) >> a.block_log2)];
    };
    int page_ahead = page_for(0);
    uint32_t bad = 0;                                           // per stage: its block does not exist
    const int64_t part = a.cache_blocks * a.num_kv_heads;       // cells of K, then those of V
    const int64_t v_off = (part << a.block_log2) * D;
    // instruction i of a copy takes row i (512 / D) + lane / (D / 16), piece lane % (D / 16).  Where a piece goes
    // in its line: K's reader has 2 rows x 4 pieces per quarter warp, V's 4 even or odd rows x 2 pieces
    const uint8_t* const k_lane = a.data + ((int64_t)h << a.block_log2) * D + lane * 16;
    const uint8_t* const v_lane = k_lane + v_off;
    const uint32_t k_dst = ring_u32 + (lane * 16 ^ (D == 64 ? 0 : D == 128 ? (lane >> 3 & 1) * 64 : (lane >> 4) * 64));
    const uint32_t v_dst = ring_u32 + C::KV_BYTES + (lane * 16 ^ (D == 64 ? (lane >> 3) * 32 : D == 128 ? (lane >> 4) * 32 : 0));
    const int copy_row = lane / (D / 16);
    const float* const scale_lane = a.scales + (lane & 1) * part + h;
    const int64_t block_bytes = (int64_t)D << a.block_log2, page_bytes = a.num_kv_heads * block_bytes;
    const int in_block = (1 << a.block_log2) - 1;
    int issue_stage = 0;
    auto issue = [&](int it) {
      const int page = page_ahead;
      page_ahead = page_for(it + 1);
      if (it < count) {
        const int st = issue_stage;
        const int key0 = sp.group_of(i0 + warp + it * WARPS) * GROUP;
        if (page < 0 || page >= a.cache_blocks) {
          bad |= 1u << st;
          if (lane == 0) atomicCAS(a.status, 0, sm100::STATUS_OVERFLOW);
        } else {
          bad &= ~(1u << st);
          const int64_t at = page * page_bytes + (key0 & in_block) * D;
          const uint8_t* k = k_lane + at;
          const uint8_t* v = v_lane + at;
          const uint32_t so = st * 2 * C::KV_BYTES;
          // bytes(r): what to copy of the group's key r, the rest of the 16 is filled with zeros
          auto copy = [&](auto bytes) {
#pragma unroll
            for (int i = 0; i < C::KC; ++i) {
              const uint32_t n = bytes(copy_row + i * (512 / D));
              // V's permutation depends on (row >> 1) & 3; what of it comes from i is a constant
              const uint32_t turn = D == 128 ? (i & 1) * 64 : D == 256 ? (i & 3) * 32 : 0;
              cp16(k_dst + so + i * 512, k + i * 512, n);
              cp16((v_dst ^ turn) + so + i * 512, v + i * 512, n);
            }
          };
          if (key0 + GROUP <= sp.length && (key0 >= sp.lo || key0 + GROUP <= sp.prefix)) {
            copy([](int) -> uint32_t { return 16; });
          } else {
            // rows that no query sees are not read: zeros, since 0 * NaN would not vanish in P V
            copy([&](int r) -> uint32_t {
              const int key = key0 + r;
              return key < sp.length && (key >= sp.lo || key < sp.prefix) ? 16 : 0;
            });
          }
          if (lane < 2) cp4(meta_u32 + (st * 2 + lane) * 4, scale_lane + (int64_t)page * a.num_kv_heads);
        }
      }
      issue_stage = issue_stage == C::STAGES - 1 ? 0 : issue_stage + 1;
      cp_commit();
    };
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) issue(s);

    // ---- the query: a power of two taken out of each row, fragments of fp16
    uint2 qf[C::Q_SMEM ? 1 : C::KSTEPS * NT];
    float coef[NT][2];
    int qpos[NT][2];
    float slope[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top = 0.f;
      auto pair = [&](uint32_t w) -> float2 {
        if (a.q_f16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      };
#pragma unroll
      for (int s = 0; s < C::KSTEPS; ++s) {
        const float2 x = pair(raw[nt][s].x), y = pair(raw[nt][s].y);
        top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      int e = (int)(__float_as_uint(top) >> 23) - 126;          // top < 2^e
      if (e == 129 || top == 0.f) e = 0;                        // infinities pass as they are
      e = min(max(e, -120), 126);                               // 2^e and 2^-e are normal numbers, as is sm_scale 2^e
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int s = 0; s < C::KSTEPS; ++s) {
        const float2 x = pair(raw[nt][s].x), y = pair(raw[nt][s].y);
        const uint2 f = make_uint2(half2_bits(x.x * down, x.y * down), half2_bits(y.x * down, y.y * down));
        if constexpr (C::Q_SMEM) {
          if (warp == 0) q_frag[(s * NT + nt) * 32 + lane] = f;
        } else {
          qf[s * NT + nt] = f;
        }
      }
      const float up = a.sm_scale * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
      for (int c = 0; c < 2; ++c) {                             // the rows of this lane's accumulator columns
        const float u = __shfl_sync(0xffffffffu, up, (2 * t + c) * 4);
        coef[nt][c] = CAP ? u / a.softcap : u * LOG2E;
        const int rr = row0 + nt * 8 + 2 * t + c;
        const int qq = rr < a.rows ? rr / a.group : 0;
        qpos[nt][c] = sp.first + qq;
        slope[nt][c] = a.slopes && rr < a.rows ? a.slopes[h * a.group + rr - qq * a.group] * LOG2E : 0.f;
      }
    }
    if constexpr (C::Q_SMEM) __syncthreads();

    float o[NT][C::KSTEPS][4];
    float m[NT][2], mv[NT][2], l[NT][2];                        // mv: the reference of P'
    float ms[NT][2], mvs[NT][2];                                // as subtracted: a row without keys has 0 and inf
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < C::KSTEPS; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nt][j][c] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) { m[nt][c] = mv[nt][c] = -INFINITY; l[nt][c] = 0.f; ms[nt][c] = 0.f; mvs[nt][c] = INFINITY; }
    }

    int stage = 0;
    for (int it = 0; it < count; ++it) {
      issue(it + C::STAGES - 1);
      cp_wait<C::STAGES - 1>();
      __syncwarp();
      const int st = stage;
      stage = stage == C::STAGES - 1 ? 0 : stage + 1;
      if (bad >> st & 1) continue;
      const int key0 = sp.group_of(i0 + warp + it * WARPS) * GROUP;
      const uint8_t* kp = ring + st * 2 * C::KV_BYTES;
      const float ks = meta[st * 2], vs = meta[st * 2 + 1];
      // ---- S^T = K Q^T
      // independent chains of products: one would put D / 16 latencies of the tensor core in a row
      constexpr int CHAINS = D / 64;
      float sc[NT][CHAINS][4], s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < CHAINS; ++i) sc[nt][i][0] = sc[nt][i][1] = sc[nt][i][2] = sc[nt][i][3] = 0.f;
#pragma unroll
      for (int i = 0; i < C::KC / 2; ++i) {
        const uint8_t* x = kp + (D == 64 ? g * D + 16 * t : g * D + 16 * t + (i >> 1) * 128 + ((i ^ g) & 1) * 64);
        const uint4 k0 = *reinterpret_cast<const uint4*>(x);
        const uint4 k8 = *reinterpret_cast<const uint4*>(x + 8 * D);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w8[4] = {k8.x, k8.y, k8.z, k8.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t a0 = widen_lo(w0[u]), a1 = widen_lo(w8[u]), a2 = widen_hi(w0[u]), a3 = widen_hi(w8[u]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint2 q;
            if constexpr (C::Q_SMEM) q = q_frag[((4 * i + u) * NT + nt) * 32 + lane];
            else q = qf[(4 * i + u) * NT + nt];
            mma16816(sc[nt][i], a0, a1, a2, a3, q.x, q.y);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if constexpr (CHAINS == 4) s[nt][c] = (sc[nt][0][c] + sc[nt][1][c]) + (sc[nt][2][c] + sc[nt][3][c]);
          else if constexpr (CHAINS == 2) s[nt][c] = sc[nt][0][c] + sc[nt][1][c];
          else s[nt][c] = sc[nt][0][c];
        }
      // ---- scores in log2 units; accumulator c: key g + 8 (c >> 1), row 2 t + (c & 1)
      const float lv = __log2f(vs);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[nt][c] *= ks * coef[nt][c & 1];
      if constexpr (CAP) {
        // a value's form depends on the value alone; the vote leaves out the second one where no value takes it
        float most = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) most = fmaxf(most, sm100::fmax3(fmaxf(fabsf(s[nt][0]), fabsf(s[nt][1])), fabsf(s[nt][2]), fabsf(s[nt][3])));
        const float cap = a.softcap * LOG2E;
        if (__all_sync(0xffffffffu, most < sm100::TANH_NEAR)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[nt][c] = cap * sm100::tanh_near(s[nt][c]);
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[nt][c] = cap * sm100::tanh_any(s[nt][c]);
        }
      }
      const bool all_seen = key0 + GROUP - 1 <= sp.first &&
                            (a.window == 0 || key0 >= sp.first + a.queries - a.window || key0 + GROUP <= sp.prefix) &&
                            key0 + GROUP <= sp.length;
      if (!all_seen || a.slopes) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int key = key0 + g + 8 * (c >> 1), d = qpos[nt][c & 1] - key;
            const bool seen = key < sp.length && ((d >= 0 && (a.window == 0 || d < a.window)) || key < sp.prefix);
            s[nt][c] = seen ? s[nt][c] - slope[nt][c & 1] * fabsf((float)d) : -INFINITY;
          }
      }
      bool need = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float x = fmaxf(s[nt][c], s[nt][c + 2]);
          need |= x > fminf(m[nt][c] + GAP, mv[nt][c] + (GAP - lv));
        }
      if (__any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = fmaxf(s[nt][c], s[nt][c + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            const float m1 = fmaxf(m[nt][c], x), mv1 = fmaxf(mv[nt][c], x + lv);
            l[nt][c] *= ratio2(m[nt][c], m1);
            const float f = ratio2(mv[nt][c], mv1);
            m[nt][c] = m1;
            mv[nt][c] = mv1;
            ms[nt][c] = m1 == -INFINITY ? 0.f : m1;
            mvs[nt][c] = mv1 == -INFINITY ? INFINITY : mv1;
#pragma unroll
            for (int j = 0; j < C::KSTEPS; ++j) { o[nt][j][c] *= f; o[nt][j][c + 2] *= f; }
          }
        }
      }
      uint32_t p[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];                                             // P', by an exponential of its own: it cannot overflow
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          l[nt][c & 1] += sm100::fast_exp2(s[nt][c] - ms[nt][c & 1]);
          w[c] = sm100::fast_exp2(s[nt][c] + ((lv + P_BIAS) - mvs[nt][c & 1]));
        }
        p[nt][0] = transpose8x8(half2_bits(w[0], w[1]));
        p[nt][1] = transpose8x8(half2_bits(w[2], w[3]));
      }
      // ---- O^T += V^T P^T
      const uint8_t* vp = kp + C::KV_BYTES;
#pragma unroll
      for (int i = 0; i < C::VI; ++i) {
        uint32_t w[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (D == 64) {
            const uint2 x = *reinterpret_cast<const uint2*>(vp + (t + 4 * (r >> 1)) * 128 +
                                                            16 * ((g >> 1) ^ (2 * t) ^ (4 * (r & 1))) + 8 * (g & 1));
            w[r][0] = x.x; w[r][1] = x.y; w[r][2] = w[r][3] = 0u;
          } else {
            const uint4 x = *reinterpret_cast<const uint4*>(vp + (2 * t + (r & 1) + 8 * (r >> 1)) * D + 16 * (g ^ (2 * t)) +
                                                            128 * i);
            w[r][0] = x.x; w[r][1] = x.y; w[r][2] = x.z; w[r][3] = x.w;
          }
        }
#pragma unroll
        for (int u = 0; u < (D == 64 ? 2 : 4); ++u) {
          const uint32_t x01 = __byte_perm(w[0][u], w[1][u], 0x5140), y01 = __byte_perm(w[0][u], w[1][u], 0x7362);
          const uint32_t x23 = __byte_perm(w[2][u], w[3][u], 0x5140), y23 = __byte_perm(w[2][u], w[3][u], 0x7362);
          const uint32_t ax[4] = {widen_lo(x01), widen_hi(x01), widen_lo(x23), widen_hi(x23)};
          const uint32_t ay[4] = {widen_lo(y01), widen_hi(y01), widen_lo(y23), widen_hi(y23)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816(o[nt][8 * i + 2 * u], ax[0], ax[1], ax[2], ax[3], p[nt][0], p[nt][1]);
            mma16816(o[nt][8 * i + 2 * u + 1], ay[0], ay[1], ay[2], ay[3], p[nt][0], p[nt][1]);
          }
        }
      }
      __syncwarp();
    }
    cp_wait<0>();

    // ---- the warps' states into one
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], d);
        if (g == 0) {
          const int r = nt * 8 + 2 * t + c;
          ml[warp * C::ROWS + r] = m[nt][c];
          ml[(WARPS + warp) * C::ROWS + r] = mv[nt][c];
          ml[(2 * WARPS + warp) * C::ROWS + r] = l[nt][c];
        }
      }
    __syncwarp();
    float* frag = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < C::KSTEPS; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) frag[((nt * C::KSTEPS + j) * 4 + c) * 32 + lane] = o[nt][j][c];
    __syncthreads();
    if (threadIdx.x < C::ROWS) {
      const int r = threadIdx.x;
      float mt = -INFINITY, mvt = -INFINITY, lt = 0.f;
      for (int w = 0; w < WARPS; ++w) {
        mt = fmaxf(mt, ml[w * C::ROWS + r]);
        mvt = fmaxf(mvt, ml[(WARPS + w) * C::ROWS + r]);
      }
      for (int w = 0; w < WARPS; ++w) {
        lt += ml[(2 * WARPS + w) * C::ROWS + r] * ratio2(ml[w * C::ROWS + r], mt);
        factors[w * C::ROWS + r] = ratio2(ml[(WARPS + w) * C::ROWS + r], mvt);
      }
      totals[r] = mt; totals[C::ROWS + r] = mvt; totals[2 * C::ROWS + r] = lt;
    }
    __syncthreads();
    const bool complete = i0 == 0 && i1 == sp.groups;
    float* record = complete ? nullptr : a.partial + ((int64_t)blockIdx.x * 2 + (i0 == 0 ? 1 : 0)) * C::RECORD;
    // a thread takes 8 consecutive dimensions of a row: values c and c + 2 of a lane's four fragments
    constexpr int QUADS = C::KSTEPS / 4;
    for (int i = threadIdx.x; i < NT * QUADS * 64; i += THREADS) {
      const int e0 = (i >> 6) * 512 + (i & 63);
      int r, dim;
      element_of<D, NT>(e0, r, dim);
      float acc[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) acc[x] = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = factors[w * C::ROWS + r];
#pragma unroll
        for (int x = 0; x < 8; ++x)
          acc[x] += reinterpret_cast<const float*>(smem + w * C::RING)[e0 + (x >> 1) * 128 + (x & 1) * 64] * f;
      }
      if (!complete) {
#pragma unroll
        for (int x = 0; x < 8; ++x) record[e0 + (x >> 1) * 128 + (x & 1) * 64] = acc[x];
      } else if (row0 + r < a.rows) {
        const float lt = totals[2 * C::ROWS + r], f = finish_factor(totals[r], totals[C::ROWS + r], lt);
        const int64_t at = output_row(a, b, h, row0 + r);
        uint4 o8;
        uint32_t* const words = reinterpret_cast<uint32_t*>(&o8);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float lo = lt == 0.f ? 0.f : acc[2 * x] * f, hi = lt == 0.f ? 0.f : acc[2 * x + 1] * f;
          if (a.q_f16) {
            words[x] = half2_bits(lo, hi);
          } else {
            const __nv_bfloat162 y = __floats2bfloat162_rn(lo, hi);
            words[x] = *reinterpret_cast<const uint32_t*>(&y);
          }
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at * D + dim) = o8;
        if (dim == 0 && a.lse) a.lse[at] = lt == 0.f ? -INFINITY : (totals[r] + __log2f(lt)) * LN2;
      }
    }
    if (!complete && threadIdx.x < 3 * C::ROWS) record[C::ACC * 32 + threadIdx.x] = totals[threadIdx.x];
    __syncthreads();
  }
  sm100::pdl_launch_dependents();
}

// ---------------------------------------------------------------- segments that more than one block worked on
// blockIdx: segment; of its fragments of 16 dimensions every gridDim.y-th; 8 of its rows.  The 8 warps take the
// parts in turn, a lane 4 of a fragment's 128 values; the first of them are on their way while the references and
// sums of all parts become a factor each.  One thread per value with the parts one after the other took 16 us
// for 524288 keys x 4 heads x 256 (of 186 in all), this takes 6.
constexpr int MERGE_AHEAD = 4, MERGE_WARPS = 8, MERGE_THREADS = MERGE_WARPS * 32;

template <int D, int NT>
__global__ void __launch_bounds__(MERGE_THREADS) kv8_merge_kernel(const DecodeArgs a, int blocks) {
  using C = Cfg<D, NT>;
  extern __shared__ __align__(16) uint8_t smem[];
  float4* slots = reinterpret_cast<float4*>(smem);              // [MERGE_WARPS][32]
  float* most = reinterpret_cast<float*>(slots + MERGE_WARPS * 32);   // [2][MERGE_WARPS][8]
  float* sum_l = most + 2 * MERGE_WARPS * 8;                          // [MERGE_WARPS][8]
  float* state = sum_l + MERGE_WARPS * 8;                             // [3][blocks][8]: m, M (then the factor), l of each part
  int* sums = reinterpret_cast<int*>(state + 3 * blocks * 8);
  int* scratch = sums + a.batch + 1;
  const int segs = a.num_kv_heads * a.row_tiles;
  const int b = blockIdx.x / segs, seg = blockIdx.x - b * segs;
  const int longest = line_sums(a, segs, sums, scratch);
  const Span sp = span_of(a, b);
  const int quota = quota_of(sums[a.batch], blocks, C::WARPS);
  const int s0 = sums[b] + seg * sp.groups, s1 = s0 + sp.groups;
  const int c0 = s0 / quota, c1 = sp.groups ? (s1 - 1) / quota : c0;
  sm100::pdl_wait();                                  // every block waits: this launch must not end before the other
  // one block had it whole
  if ((sp.groups > 0 && c0 == c1) || takes_whole(a.batch * segs, longest, quota, blocks, C::DIRECT)) return;
  const int parts = sp.groups ? c1 - c0 + 1 : 0;
  // the block where the segment starts left it in its slot 1, the others in their slot 0
  auto record = [&](int i) { return a.partial + ((int64_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * C::RECORD; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nt = blockIdx.z;
  auto values = [&](int j, int i) {
    return __ldcg(reinterpret_cast<const float4*>(record(i) + (nt * C::KSTEPS + j) * 128) + lane);
  };
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  float4 ahead[MERGE_AHEAD];
#pragma unroll
  for (int x = 0; x < MERGE_AHEAD; ++x) ahead[x] = warp + x * MERGE_WARPS < parts ? values(blockIdx.y, warp + x * MERGE_WARPS) : zero;

  // ---- a factor for each part and row; thread: row tid & 7, parts tid / 8, + 32, ...
  const int row = threadIdx.x & 7;
  float* const state_m = state, * const state_mv = state + blocks * 8, * const state_l = state + 2 * blocks * 8;
  float mt = -INFINITY, mvt = -INFINITY;
  for (int i = threadIdx.x >> 3; i < parts; i += MERGE_THREADS / 8) {
    const float* x = record(i) + C::ACC * 32 + nt * 8 + row;
    const float m = __ldcg(x), mv = __ldcg(x + C::ROWS), l = __ldcg(x + 2 * C::ROWS);
    state_m[i * 8 + row] = m; state_mv[i * 8 + row] = mv; state_l[i * 8 + row] = l;
    mt = fmaxf(mt, m);
    mvt = fmaxf(mvt, mv);
  }
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) {
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
    mvt = fmaxf(mvt, __shfl_xor_sync(0xffffffffu, mvt, o));
  }
  if (lane < 8) { most[warp * 8 + lane] = mt; most[(MERGE_WARPS + warp) * 8 + lane] = mvt; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < MERGE_WARPS; ++w) {
    mt = fmaxf(mt, most[w * 8 + row]);
    mvt = fmaxf(mvt, most[(MERGE_WARPS + w) * 8 + row]);
  }
  float lt = 0.f;
  for (int i = threadIdx.x >> 3; i < parts; i += MERGE_THREADS / 8) {
    lt += state_l[i * 8 + row] * ratio2(state_m[i * 8 + row], mt);
    state_mv[i * 8 + row] = ratio2(state_mv[i * 8 + row], mvt);
  }
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) lt += __shfl_xor_sync(0xffffffffu, lt, o);
  if (lane < 8) sum_l[warp * 8 + lane] = lt;
  __syncthreads();
  lt = 0.f;
#pragma unroll
  for (int w = 0; w < MERGE_WARPS; ++w) lt += sum_l[w * 8 + row];

  // ---- the values: of fragment lane 4 (lane & 7) + k, accumulator lane >> 3, that is of row 2 k + (lane >> 3 & 1)
  const int h = seg / a.row_tiles, out_row = (seg - h * a.row_tiles) * C::ROWS + nt * 8 + row;
  for (int j = blockIdx.y; j < C::KSTEPS; j += gridDim.y) {
    float4 acc = zero;
    auto add = [&](const float4& v, int i) {
      const float* f = state_mv + i * 8 + (lane >> 3 & 1);
      acc.x += v.x * f[0]; acc.y += v.y * f[2]; acc.z += v.z * f[4]; acc.w += v.w * f[6];
    };
#pragma unroll
    for (int x = 0; x < MERGE_AHEAD; ++x)
      if (warp + x * MERGE_WARPS < parts) add(ahead[x], warp + x * MERGE_WARPS);
#pragma unroll 4
    for (int i = warp + MERGE_AHEAD * MERGE_WARPS; i < parts; i += MERGE_WARPS) add(values(j, i), i);
    const int next = j + gridDim.y;
    if (next < C::KSTEPS) {
#pragma unroll
      for (int x = 0; x < MERGE_AHEAD; ++x) if (warp + x * MERGE_WARPS < parts) ahead[x] = values(next, warp + x * MERGE_WARPS);
    }
    slots[warp * 32 + lane] = acc;
    __syncthreads();
    // thread: row tid & 7, dimensions of fragment row tid / 8: accumulators row & 1 and that + 2
    if (threadIdx.x < 64 && out_row < a.rows) {
      const int g = threadIdx.x >> 3;
      const float* at0 = reinterpret_cast<const float*>(slots) + (row & 1) * 32 + g * 4 + (row >> 1);
      float lo = 0.f, hi = 0.f;
#pragma unroll
      for (int w = 0; w < MERGE_WARPS; ++w) { lo += at0[w * 128]; hi += at0[w * 128 + 64]; }
      const float f = finish_factor(mt, mvt, lt);
      lo = lt == 0.f ? 0.f : lo * f;
      hi = lt == 0.f ? 0.f : hi * f;
      const int dim = D == 64 ? 8 * g + 2 * j : 16 * g + 2 * (j & 7) + 128 * (j >> 3);
      const int64_t at = output_row(a, b, h, out_row);
      uint32_t word;
      if (a.q_f16) {
        word = half2_bits(lo, hi);
      } else {
        const __nv_bfloat162 y = __floats2bfloat162_rn(lo, hi);
        word = *reinterpret_cast<const uint32_t*>(&y);
      }
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at * D + dim) = word;
      if (dim == 0 && a.lse) a.lse[at] = lt == 0.f ? -INFINITY : (mt + __log2f(lt)) * LN2;
    }
    __syncthreads();
  }
}

struct Plan {
  int blocks, direct;
  int64_t bytes;
};

template <int D, int NT>
Plan plan_for(int64_t segments, int64_t longest) {
  using C = Cfg<D, NT>;
  Plan p;
  p.direct = longest <= C::DIRECT;
  // no more blocks than there can be pieces
  p.blocks = (int)(p.direct ? segments
                            : std::min<int64_t>((int64_t)semblo::sm_count() * C::PER_SM, ceil_div(segments * longest, C::WARPS)));
  p.bytes = p.direct ? 0 : (int64_t)p.blocks * 2 * C::RECORD * 4;
  return p;
}

int64_t longest_segment(int queries, int window, int table_len, int block_size, bool prefix) {
  int64_t keys = (int64_t)table_len * block_size;
  if (window > 0 && !prefix) keys = std::min<int64_t>(keys, (int64_t)window + queries + GROUP);
  return ceil_div(keys, GROUP);
}

// Shared memory of the line's sums, and of the merge.
constexpr int MAX_BATCH = 4096;
template <int D, int NT> constexpr int sum_bytes(int batch) { return (batch + 2 + 2 * std::max(Cfg<D, NT>::WARPS, MERGE_WARPS)) * 4; }
constexpr int merge_bytes(int blocks, int sums) { return MERGE_WARPS * 32 * 16 + (3 * MERGE_WARPS + 3 * blocks) * 8 * 4 + sums; }

template <int D, int NT, bool CAP>
int launch(DecodeArgs& a, const Plan& plan, cudaStream_t st) {
  using C = Cfg<D, NT>;
  const int sums = sum_bytes<D, NT>(a.batch);
  auto kern = kv8_decode_kernel<D, NT, CAP>;
  // the limits are a kernel's, not a launch's: set to the same value by every call, since another thread may be between
  // its own two lines
  SEMBLO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SUM_OFF + sum_bytes<D, NT>(MAX_BATCH)));
  const int smem = C::SUM_OFF + sums;
  a.direct = plan.direct;
  kern<<<plan.blocks, C::THREADS, smem, st>>>(a);
  SEMBLO_LAUNCH_CHECK();
  if (plan.direct) return 0;
  cudaLaunchConfig_t cfg{};
  // a block per fragment of 16 dimensions while there are few segments to merge
  const int segments = a.batch * a.num_kv_heads * a.row_tiles;
  const int slices = std::max(1, std::min(C::KSTEPS, 8 * semblo::sm_count() / (segments * NT)));
  cfg.gridDim = dim3((unsigned)segments, (unsigned)slices, NT);
  cfg.blockDim = dim3(MERGE_THREADS);
  cfg.dynamicSmemBytes = merge_bytes(plan.blocks, sums);
  SEMBLO_CUDA(cudaFuncSetAttribute(kv8_merge_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   merge_bytes(semblo::sm_count() * C::PER_SM, sum_bytes<D, NT>(MAX_BATCH))));
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  SEMBLO_CUDA(cudaLaunchKernelEx(&cfg, kv8_merge_kernel<D, NT>, (const DecodeArgs)a, plan.blocks));
  return 0;
}

int check_shape(int batch, int queries, int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                int table_len, int window, int* rows, int* nt, int* tiles) {
  SEMBLO_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "head_dim must be 64, 128 or 256 (got %d)",
                 head_dim);
  SEMBLO_REQUIRE(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
                 "query heads must be a multiple of the KV heads");
  SEMBLO_REQUIRE(block_size >= 16 && block_size <= 256 && (block_size & (block_size - 1)) == 0,
                 "block_size must be 16, 32, 64, 128 or 256 (got %d)", block_size);
  SEMBLO_REQUIRE(queries >= 1 && queries <= 16, "1 to 16 queries per request (got %d)", queries);
  SEMBLO_REQUIRE(batch >= 0 && batch <= MAX_BATCH, "at most %d requests (got %d)", MAX_BATCH, batch);
  SEMBLO_REQUIRE(table_len >= 0 && window >= 0, "negative table length or window");
  *rows = queries * (num_q_heads / num_kv_heads);
  // the widest tiles whose O stays in registers (the cache is read and widened once per tile), as narrow as
  // that number of tiles allows
  *tiles = (int)ceil_div(*rows, head_dim == 256 ? 16 : 32);
  *nt = (int)ceil_div(ceil_div(*rows, *tiles), 8);
  const int64_t groups = std::max<int64_t>(1, ceil_div((int64_t)table_len * block_size, 16));
  SEMBLO_REQUIRE(groups * batch * num_kv_heads * *tiles < ((int64_t)1 << 31), "batch x context is too large for one call");
  return 0;
}

Plan plan_of(int head_dim, int nt, int64_t segments, int64_t longest) {
#define SEMBLO_PLAN(DD, NN) if (head_dim == DD && nt == NN) return plan_for<DD, NN>(segments, longest);
  SEMBLO_PLAN(64, 1) SEMBLO_PLAN(64, 2) SEMBLO_PLAN(128, 1) SEMBLO_PLAN(128, 2) SEMBLO_PLAN(256, 1)
  SEMBLO_PLAN(64, 3) SEMBLO_PLAN(64, 4) SEMBLO_PLAN(128, 3) SEMBLO_PLAN(128, 4)
#undef SEMBLO_PLAN
  return plan_for<256, 2>(segments, longest);
}

}  // namespace

extern "C" int64_t semblo_kv8_decode_workspace_bytes(int batch, int queries, int num_q_heads, int num_kv_heads,
                                                     int head_dim, int block_size, int table_len, int window,
                                                     int has_prefix) {
  int rows, nt, tiles;
  const int rc = check_shape(batch, queries, num_q_heads, num_kv_heads, head_dim, block_size, table_len, window,
                             &rows, &nt, &tiles);
  if (rc) return rc;
  return plan_of(head_dim, nt, (int64_t)batch * num_kv_heads * tiles,
                 longest_segment(queries, window, table_len, block_size, has_prefix)).bytes;
}

extern "C" int semblo_kv8_decode(const void* q, int dtype, int batch, int queries, int num_q_heads,
                                 int num_kv_heads, int head_dim, const void* cache, const float* scales,
                                 int64_t cache_blocks, int block_size, const int32_t* block_table,
                                 int64_t table_stride, int table_len, const int32_t* lengths,
                                 const int32_t* prefix_lens, int window, float sm_scale, float softcap,
                                 const float* alibi_slopes, void* out, float* lse, void* workspace,
                                 int64_t workspace_bytes, int32_t* status, void* stream) {
  int rows, nt, tiles;
  const int rc = check_shape(batch, queries, num_q_heads, num_kv_heads, head_dim, block_size, table_len, window,
                             &rows, &nt, &tiles);
  if (rc) return rc;
  SEMBLO_REQUIRE(dtype == SEMBLO_BF16 || dtype == SEMBLO_F16, "queries are bf16 or fp16 (got dtype code %d)", dtype);
  SEMBLO_REQUIRE(semblo::cap_in_range(softcap), "the soft cap must be 0 or lie in [2^-100, 2^100] (got %g)", (double)softcap);
  if (batch == 0) return 0;
  SEMBLO_REQUIRE(q && cache && scales && block_table && lengths && out && status, "null pointer");
  SEMBLO_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
                 "q, the cache and out must be 16-byte aligned");
  const Plan plan = plan_of(head_dim, nt, (int64_t)batch * num_kv_heads * tiles,
                            longest_segment(queries, window, table_len, block_size, prefix_lens != nullptr));
  SEMBLO_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "the workspace must be 16-byte aligned");
  if (plan.bytes > workspace_bytes || (plan.bytes && !workspace))
    return semblo::fail(semblo::SEMBLO_ENOSPC, "workspace of %lld bytes needed, %lld given", (long long)plan.bytes,
                        (long long)workspace_bytes);
  DecodeArgs a{};
  a.q = q; a.q_f16 = dtype == SEMBLO_F16;
  a.out = out; a.lse = lse;
  a.data = (const uint8_t*)cache; a.scales = scales; a.cache_blocks = cache_blocks;
  while ((1 << a.block_log2) < block_size) ++a.block_log2;
  a.table = block_table; a.table_stride = table_stride; a.table_len = table_len;
  a.lengths = lengths; a.prefix = prefix_lens; a.slopes = alibi_slopes;
  a.batch = batch; a.queries = queries; a.num_q_heads = num_q_heads; a.num_kv_heads = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.rows = rows; a.row_tiles = tiles;
  a.window = window; a.sm_scale = sm_scale; a.softcap = softcap;
  a.partial = (float*)workspace;
  a.status = status;
  cudaStream_t st = (cudaStream_t)stream;
  const bool cap = softcap > 0.f;
#define SEMBLO_DECODE(DD, NN)                                                                     \
  if (head_dim == DD && nt == NN)                                                                 \
    return cap ? launch<DD, NN, true>(a, plan, st) : launch<DD, NN, false>(a, plan, st);
  SEMBLO_DECODE(64, 1) SEMBLO_DECODE(64, 2) SEMBLO_DECODE(128, 1) SEMBLO_DECODE(128, 2) SEMBLO_DECODE(256, 1)
  SEMBLO_DECODE(256, 2) SEMBLO_DECODE(64, 3) SEMBLO_DECODE(64, 4) SEMBLO_DECODE(128, 3) SEMBLO_DECODE(128, 4)
#undef SEMBLO_DECODE
  return semblo::fail(semblo::SEMBLO_EINVAL, "unreachable");
}
