// Attention of packed prompts for head dimensions 64 and 128 (the mathematics is in dense_prefill.cu).
//
// Two tiles of 128 rows (queries x the heads of a KV head) take turns on a multiprocessor: while the tensor core
// works on one tile (P V of a key tile, then S of the next), a warpgroup runs the softmax of the other, one
// thread per row.  At D = 128 the two S buffers and the two O accumulators are all of
// tensor memory; P lies over the S it came from.  Q, K and V are in shared memory (Q and a ring of
// K, V tiles by TMA).  P is handed over in halves, so that P V starts when half the exponentials are done.
// The two tiles belong to one block, which loads K and V once for both, or to two blocks (one_tile() below).
// Where scores are capped or biased or two blocks share the registers, a half is a step of the running maximum of
// its own: the 128 scores of a whole row, the polynomial's coefficients and its chains do not fit together.
#include <algorithm>

#include "dense_pair.h"
#include "host_common.h"

using namespace dense;
using semblo::ceil_div;

namespace {

constexpr int BN = PAIR_BN;
constexpr int PAGE = 16;

template <int D, int MODE, int TILES>
struct Cfg {
  // threads per row.  With a running maximum one: two would have to meet for every tile and, with half the
  // registers each, read the scores twice (16384 causal 1.4 times as long).  Under a fixed reference two pay where
  // the softmax outweighs the products (8192 capped, windowed: D = 64 797 -> 666 us, D = 128 752 -> 780)
  static constexpr int HALVES = MODE == BOUNDED && D == 64 ? 2 : 1;
  static constexpr int WARPS = 4 * TILES * HALVES;               // of the softmax; then the loading and the issuing warp
  static constexpr int THREADS = (WARPS + 2) * 32;
  static constexpr int SLABS = D / 64;                         // 128-byte wide slabs of a 16-bit tile
  static constexpr int TILE = BN * D * 2;                      // a tile of Q, K or V
  static constexpr int SLOTS = D == 128 ? (TILES == 2 ? 5 : 2) : TILES == 2 ? 8 : 5;
  static constexpr int Q_OFF = 0;
  static constexpr int KV_OFF = TILES * TILE;
  static constexpr int SUM_OFF = KV_OFF + SLOTS * TILE;        // float [2 tiles][2 halves][128]
  static constexpr int BAR_OFF = SUM_OFF + (HALVES == 2 ? 2048 : 0);
  static constexpr int TOTAL = BAR_OFF + 256;
  static constexpr int S_COL = 0;                              // + 128 x: S and P of tile x
  static constexpr int O_COL = 128 * TILES;                    // + D x
  static constexpr int TMEM_COLS = 256 * TILES;
  // P of a half lies over logits that the half's own threads have read
  static constexpr int P_HALF = HALVES == 2 ? 64 : 32;
};

enum { B_Q = 0, B_S = 1, B_P = 3, B_H = 7, B_O = 9, B_FULL = 11 };     // B_S + x, B_P + 2 x + half, B_H + x, B_O + x

// Which key tiles the block walks over and which of its row tiles sees each.
template <int TILES>
struct Walk {
  int gp, first, n;                       // prefix tiles, first tile of the main part, tiles in all
  int base = 0;                           // first of the block's, where the keys are cut into pieces (one row tile)
  int glo[TILES], end[TILES];
  bool any[TILES];
  __device__ __forceinline__ Walk(const Args& a, const Tile& t) {
    const int qt = a.queries_per_tile / TILES;
    int last = 0;
    first = 1 << 30;
    gp = 0;
#pragma unroll
    for (int x = 0; x < TILES; ++x) {
      Tile s = t;
      s.pos += x * qt;
      s.count = min(qt, t.count - x * qt);
      any[x] = s.count > 0;
      glo[x] = end[x] = 0;
      if (!any[x]) continue;
      const KeyTiles<BN> k(a, s);
      gp = k.gp;
      glo[x] = k.glo;
      end[x] = k.glo + k.n - k.gp;
      if (end[x] > glo[x]) {
        first = min(first, glo[x]);
        last = max(last, end[x]);
      }
    }
    n = gp + max(0, last - first);
  }
  __device__ __forceinline__ int tile(int j) const {
    if (TILES == 1) j += base;
    return j < gp ? j : j - gp + first;
  }
  __device__ __forceinline__ bool sees(int x, int j) const {
    if (TILES == 1) return j < n;
    const int i = tile(j);
    return any[x] && j < n && (j < gp || (i >= glo[x] && i < end[x]));
  }
};

template <int D, bool F16, int MODE, int TILES>
__global__ void __launch_bounds__(Cfg<D, MODE, TILES>::THREADS, 3 - TILES)
dense_pair_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                  const __grid_constant__ CUtensorMap tmap_v, const Args a) {
  using C = Cfg<D, MODE, TILES>;
  constexpr int SLOTS = C::SLOTS, HALVES = C::HALVES;
  constexpr int B_EMPTY = B_FULL + SLOTS;
  static_assert(8 * (B_EMPTY + SLOTS) + 8 <= 256, "barrier area");
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Share share(a, a.splits);
  const int h = share.h;
  if (smem_u32(smem) & 1023u) {                    // the swizzled tiles need 1024-byte alignment
    if (threadIdx.x == 0) atomicCAS(a.status, 0, STATUS_SMEM_ALIGN);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::TOTAL - 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  // barriers by the warp that loads, which need not wait for anybody with its first loads; tensor memory by the
  // warp that issues, while the others look for their tile
  if (warp == C::WARPS && lane == 0) {
    mbar_init(bar(B_Q), 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(bar(B_S + x), 1);
      mbar_init(bar(B_P + 2 * x), 4);              // the warps of the tile's softmax
      mbar_init(bar(B_P + 2 * x + 1), 4);
      mbar_init(bar(B_H + x), 1);                  // P V of a first half is complete
      mbar_init(bar(B_O + x), 1);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(bar(B_FULL + s), 1);
      mbar_init(bar(B_EMPTY + s), 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  __syncwarp();
  // the same answer in every warp
  const Tile tile = a.docs <= WARP_DOCS ? find_tile(a, share.want) : find_tile_block<C::THREADS>(a, share.want);
  if (tile.doc < 0) {
    if (a.zero_tail && share.split == 0) zero_tail<D>(a, tile.first, h, blockDim.x);
    return;
  }
  Walk<TILES> walk(a, tile);
  int pieces = 1;
  if constexpr (TILES == 1) {
    pieces = pieces_of(a, walk.n, BN);
    if (share.split >= pieces) return;
    walk.base = (int)((int64_t)walk.n * share.split / pieces);
    walk.n = (int)((int64_t)walk.n * (share.split + 1) / pieces) - walk.base;
  }
  const int qt = a.queries_per_tile / TILES;
  auto load_kv = [&](int i) {                      // K(i / 2) or V(i / 2) into its slot, which is free
    const int s = i % SLOTS, row = tile.k0 + walk.tile(i >> 1) * BN;
    mbar_arrive_expect_tx(bar(B_FULL + s), (uint32_t)C::TILE);
    for (int sl = 0; sl < C::SLABS; ++sl)
      tma_load_3d(smem_u32(smem + C::KV_OFF + s * C::TILE + sl * BN * 128), (i & 1) ? &tmap_v : &tmap_k, bar(B_FULL + s),
                  sl * 64, h, row);
  };
  if (warp == C::WARPS && lane == 0 && walk.n > 0) {
    const int tiles = walk.any[TILES - 1] ? TILES : 1;
    mbar_arrive_expect_tx(bar(B_Q), (uint32_t)(tiles * C::SLABS * qt * a.group * 128));
    for (int x = 0; x < tiles; ++x)
      for (int sl = 0; sl < C::SLABS; ++sl)
        tma_load_3d(smem_u32(smem + C::Q_OFF + x * C::TILE + sl * BN * 128), &tmap_q, bar(B_Q), sl * 64, h * a.group,
                    (int)tile.token + x * qt);
    load_kv(0);
    load_kv(1);
  }
  if (warp == C::WARPS + 1) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == C::WARPS) {
    // ------------------------------------------------------------ producer: after Q, K(0), V(0): K(1), V(1), ...
    if (lane == 0) {
      for (int i = 2; i < 2 * walk.n; ++i) {
        if (!mbar_wait(bar(B_EMPTY + i % SLOTS), ((i / SLOTS) & 1) ^ 1, abort_flag, a.status, STATUS_TIMEOUT_LOAD)) break;
        load_kv(i);
      }
    }
  } else if (warp == C::WARPS + 1) {
    // ------------------------------------------------------------ UMMA issuer
    // UMMAs of one thread execute in order: S(j + 1) may overwrite the P that the P V before it reads.
    if (elect_one()) {
      constexpr uint32_t idesc_pv = idesc_of<F16>(128, D, true);
      const int n = walk.n;
      bool ok = n == 0 || mbar_wait(bar(B_Q), 0, abort_flag, a.status, STATUS_TIMEOUT_MMA);
      auto keys_of = [&](int j) { return min(BN, tile.lk - walk.tile(j) * BN); };
      auto wait_slot = [&](int i) {
        ok = ok && mbar_wait(bar(B_FULL + i % SLOTS), (i / SLOTS) & 1, abort_flag, a.status, STATUS_TIMEOUT_MMA);
        return ok;
      };
      auto issue_s = [&](int x, int j) {           // K(j) has arrived
        tc_fence_after();
        const uint32_t q_base = smem_u32(smem + C::Q_OFF + x * C::TILE);
        const uint32_t k_base = smem_u32(smem + C::KV_OFF + (2 * j) % SLOTS * C::TILE);
        const uint32_t idesc = idesc_of<F16>(128, (keys_of(j) + PAGE - 1) / PAGE * PAGE, false);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * BN * 128 + (kk & 3) * 32;
          umma_ss(tmem_base + C::S_COL + x * 128, make_smem_desc(q_base + off, 16, 1024), make_smem_desc(k_base + off, 16, 1024),
                  idesc, kk > 0 ? 1u : 0u);
        }
        umma_commit(bar(B_S + x));
      };
      int done[2] = {0, 0};                        // P V products of each tile
      auto issue_pv = [&](int x, int j) {          // V(j) has arrived
        const int pages = (keys_of(j) + PAGE - 1) / PAGE;
        const uint32_t v_base = smem_u32(smem + C::KV_OFF + (2 * j + 1) % SLOTS * C::TILE);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ok = ok && mbar_wait(bar(B_P + 2 * x + half), done[x] & 1, abort_flag, a.status, STATUS_TIMEOUT_MMA);
          if (!ok) return;
          tc_fence_after();
#pragma unroll
          for (int kk = half * 4; kk < half * 4 + 4; ++kk)
            if (kk < pages)
              umma_ts(tmem_base + C::O_COL + x * D, tmem_base + C::S_COL + x * 128 + half * C::P_HALF + (kk & 3) * 8,
                      make_smem_desc(v_base + kk * PAGE * 128, BN * 128, 1024), idesc_pv, (done[x] > 0 || kk > 0) ? 1u : 0u);
          if (half == 0) umma_commit(bar(B_H + x));
        }
        ++done[x];
      };
      if (ok && n > 0 && wait_slot(0)) {
#pragma unroll
        for (int x = 0; x < TILES; ++x)
          if (walk.sees(x, 0)) issue_s(x, 0);
        umma_commit(bar(B_EMPTY));
      }
      for (int j = 0; ok && j < n; ++j) {
        if (!wait_slot(2 * j + 1)) break;
        const bool more = j + 1 < n;
#pragma unroll
        for (int x = 0; x < TILES; ++x) {
          if (ok && walk.sees(x, j)) issue_pv(x, j);
          if (x == TILES - 1 && ok) umma_commit(bar(B_EMPTY + (2 * j + 1) % SLOTS));
          if (more && ok) {
            if (x == 0) wait_slot(2 * j + 2);
            if (ok && walk.sees(x, j + 1)) issue_s(x, j + 1);
            if (x == TILES - 1 && ok) umma_commit(bar(B_EMPTY + (2 * j + 2) % SLOTS));
          }
        }
      }
      if (ok) {
        umma_commit(bar(B_O));
        umma_commit(bar(B_O + 1));
      }
    }
  } else {
    // ------------------------------------------------------------ softmax + epilogue: one or two threads per row
    const int x = TILES == 2 ? warp / (C::WARPS / 2) : 0, hf = HALVES == 2 ? (warp >> 2) & 1 : 0;
    const int row = threadIdx.x & 127;
    const int qi = row / a.group, hg = row - qi * a.group;
    const bool valid = qi < qt && x * qt + qi < tile.count;
    const int p = tile.pos + x * qt + qi;
    const Seen seen = valid ? seen_by(a, tile, p) : Seen{0, 0, 0};
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_addr + C::S_COL + x * 128;
    const uint32_t o_addr = tmem_base + lane_addr + C::O_COL + x * D + hf * (D / 2);
    const int head = h * a.group + hg;
    const float slope = a.slopes && valid ? a.slopes[head] * LOG2EF : 0.f;
    const float scale = scale_of<MODE>(a);
    const TanhPoly<MODE == BOUNDED ? 5 : 8> capped(a.cap_log2);
    float m_ref = MODE == BOUNDED ? bounded_reference(a.cap_log2) : -INFINITY, l = 0.f;
    bool ok = true;
    int count = 0;
    // this tile's walk: [0, gp), then [j0, j1)
    constexpr int LAST = TILES - 1;
    const bool any = x ? walk.any[LAST] : walk.any[0];
    const int glo = x ? walk.glo[LAST] : walk.glo[0], gend = x ? walk.end[LAST] : walk.end[0];
    const int gp = TILES == 2 && any ? walk.gp : 0;
    const int j0 = TILES == 2 && any && gend > glo ? walk.gp + glo - walk.first : gp;
    const int j1 = TILES == 1 ? walk.n : any && gend > glo ? j0 + gend - glo : gp;
    for (int j = gp > 0 ? 0 : j0; j < gp || (j >= j0 && j < j1); j = j + 1 == gp ? j0 : j + 1) {
      const int key0 = walk.tile(j) * BN;
      ok = mbar_wait_warp(bar(B_S + x), (uint32_t)(count & 1), abort_flag, a.status, STATUS_TIMEOUT_SOFTMAX);
      if (!ok) break;
      tc_fence_after();
      // P of chunk c (32 keys) of the tile to tensor memory: keys 2 i, 2 i + 1 share a column, P lies over logits that
      // have been read.  After every second chunk a half is handed over
      auto store = [&](int c, const uint32_t (&packed)[16]) {
        tmem_st16(s_addr + (c >> 1) * C::P_HALF + (c & 1) * 16, packed);
        if (!(c & 1)) return;
        // V's rows behind the document's end (another document's, or anything) are cleared: their P is 0, but 0 * NaN
        // would not vanish.  Both tiles' warps may do it; the stage stays until both are multiplied
        const int left = tile.lk - key0;
        if (c >> 1 == (HALVES == 2 ? left >> 6 : 0) && (warp & 3) == 0 && left < BN && (left & (PAGE - 1))) {
          ok = mbar_wait_warp(bar(B_FULL + (2 * j + 1) % SLOTS), ((2 * j + 1) / SLOTS) & 1, abort_flag, a.status,
                              STATUS_TIMEOUT_SOFTMAX);
          if (ok) zero_rows<D, BN>(smem + C::KV_OFF + (2 * j + 1) % SLOTS * C::TILE, left, (left + PAGE - 1) / PAGE * PAGE);
          fence_proxy_async_smem();
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_P + 2 * x + (c >> 1)));
      };
      constexpr int STEPS = MODE == BOUNDED ? 0 : MODE == LINEAR && TILES == 2 ? 1 : 2, CH = STEPS == 1 ? 4 : 2;   // chunks in a step
      if constexpr (MODE == BOUNDED) {
        // no maximum: chunk by chunk (with registers to spare the next one's scores on their way)
        constexpr int CHUNKS = 4 / HALVES, BUFFERS = HALVES == 1 ? 2 : 1;
        f32x2 sum0 = join(0.f, 0.f), sum1 = sum0;
        uint32_t held[BUFFERS][32];
        if constexpr (BUFFERS == 2) tmem_ld32(s_addr, held[0]);
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
          const int c = 2 * hf + i;
          uint32_t (&s)[32] = held[i % BUFFERS];
          if constexpr (BUFFERS == 1) tmem_ld32(s_addr + c * 32, s);
          tmem_ld_wait();
          if (BUFFERS == 2 && i + 1 < CHUNKS) tmem_ld32(s_addr + (c + 1) * 32, held[(i + 1) % BUFFERS]);
          const int lo = seen.lo - key0 - 32 * c, hi = seen.hi - key0 - 32 * c, pre = seen.pre - key0 - 32 * c;
          const bool all = __all_sync(0xffffffffu, (lo <= 0 && hi >= 32) || pre >= 32);
          bounded32(s, a, capped, all, seen_bits(lo, hi, pre), -m_ref);
          uint32_t packed[16];
#pragma unroll
          for (int n = 0; n < 16; ++n) {
            const float e0 = fast_exp2(__uint_as_float(s[2 * n])), e1 = fast_exp2(__uint_as_float(s[2 * n + 1]));
            packed[n] = pack_pair<F16>(e0, e1);
            if (n & 1) sum1 = add2(sum1, join(e0, e1)); else sum0 = add2(sum0, join(e0, e1));
          }
          store(c, packed);
        }
        float s0, s1;
        split(add2(sum0, sum1), s0, s1);
        l += s0 + s1;
      }
#pragma unroll 1
      for (int step = 0; step < STEPS; ++step) {
        const int k0 = key0 + 64 * step;
        uint32_t s[CH][32];
#pragma unroll
        for (int c = 0; c < CH; ++c) tmem_ld32(s_addr + step * 64 + c * 32, s[c]);
        tmem_ld_wait();
        const int lo = seen.lo - k0, hi = seen.hi - k0, pre = seen.pre - k0;
        const bool all = __all_sync(0xffffffffu, (lo <= 0 && hi >= 32 * CH) || pre >= 32 * CH);
        float tmax = -INFINITY, least = INFINITY;
        bool poly = false;                             // tanh by polynomial, in the exponential's pass
        if constexpr (MODE != BIASED) {
#pragma unroll
          for (int c = 0; c < CH; ++c) range32<MODE == CAPPED>(s[c], tmax, least);
        }
        if constexpr (MODE == CAPPED) {
          poly = all && __all_sync(0xffffffffu, fmaxf(tmax, -least) * a.score_scale < TANH_FAR);
          if (poly) tmax = tanh_exp(tmax * (a.score_scale * (1.f / TANH_ARG)));
        }
        if (MODE == BIASED || (MODE == CAPPED && !poly) || (MODE == LINEAR && !all)) {
          tmax = -INFINITY;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            transform32<MODE>(s[c], a, slope, p, k0 + 32 * c);
            if (!all) {
              hide32(s[c], seen_bits(lo - 32 * c, hi - 32 * c, pre - 32 * c));
            }
            range32<false>(s[c], tmax, least);
          }
        }
        tmax *= scale;
        // lazy rescale: only when the running reference falls far behind
        const bool need = m_ref != -INFINITY && tmax > m_ref + rescale_gap<F16>();
        float alpha = 1.f;
        if (need) {
          alpha = fast_exp2(m_ref - tmax);
          m_ref = tmax;
          l *= alpha;
        } else if (m_ref == -INFINITY) {
          m_ref = tmax;
        }
        if (__any_sync(0xffffffffu, need)) {
          // O is quiescent in the first step (S's barrier covers the P V issued before it), in the second when
          // the first half's P V has completed
          if (step == 1) {
            ok = mbar_wait_warp(bar(B_H + x), (uint32_t)(count & 1), abort_flag, a.status, STATUS_TIMEOUT_SOFTMAX);
            if (!ok) break;
            tc_fence_after();
          }
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(o_addr + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(o_addr + c * 32, o);
          }
        }
        const float neg_m = m_ref == -INFINITY ? 0.f : p_bias<F16>() - m_ref;
        const f32x2 scale2 = join(scale, scale), neg2 = join(neg_m, neg_m);
        f32x2 sum0 = join(0.f, 0.f), sum1 = sum0;
        auto exponentials = [&](auto argument) {
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            uint32_t packed[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float e0, e1;
              split(argument(join(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1]))), e0, e1);
              e0 = fast_exp2(e0);
              e1 = fast_exp2(e1);
              packed[i] = pack_pair<F16>(e0, e1);
              if (i & 1) sum1 = add2(sum1, join(e0, e1)); else sum0 = add2(sum0, join(e0, e1));
            }
            store(2 * step + c, packed);
          }
        };
        if (MODE == CAPPED && poly) {
          const f32x2 arg2 = join(a.score_scale, a.score_scale);
          exponentials([&](f32x2 v) { return capped(mul2(v, arg2), neg2); });
        } else {
          exponentials([&](f32x2 v) { return fma2(v, scale2, neg2); });
        }
        float s0, s1;
        split(add2(sum0, sum1), s0, s1);
        l += s0 + s1;
      }
      if (!ok) break;
      ++count;
    }
    if (ok) ok = mbar_wait_warp(bar(B_O + x), 0, abort_flag, a.status, STATUS_TIMEOUT_EPILOGUE);
    tc_fence_after();
    if constexpr (HALVES == 2) {
      float* sums = reinterpret_cast<float*>(smem + C::SUM_OFF) + x * 256;
      sums[hf * 128 + row] = l;
      asm volatile("bar.sync %0, 256;" ::"r"(1 + x) : "memory");     // all of the tile's threads, whatever became of them
      l += sums[(hf ^ 1) * 128 + row];
    }
    if (TILES == 1 && pieces > 1) {
      if (ok) {
        float* record = share.record(a, D, share.split);
#pragma unroll 1
        for (int c = 0; c < D / 32 / HALVES; ++c) store_partial(o_addr + c * 32, record + row * D + hf * (D / 2) + c * 32, valid);
        if (valid && hf == 0) {
          record[128 * D + row] = m_ref;
          record[128 * D + 128 + row] = l;
        }
      }
    } else if (ok && any) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t at = (tile.token + x * qt + qi) * a.num_q_heads + head;
      // through Q's shared memory (no product is in flight any more), a warp's own part of it
      constexpr int PIECES = D / 8 / HALVES;
      uint8_t* stage = smem + C::Q_OFF + warp * 32 * PIECES * 16;
#pragma unroll 1
      for (int c = 0; c < D / 32 / HALVES; ++c) {
        uint32_t o[32];
        if (count > 0) {
          tmem_ld32(o_addr + c * 32, o);
          tmem_ld_wait();
        }
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          w[i] = l == 0.f ? 0u : pack_pair<F16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
        stage_pieces<PIECES>(stage, c * 4, w);
      }
      __syncwarp();
#pragma unroll 4
      for (int i = lane; i < 32 * PIECES; i += 32) {
        const int r = i / PIECES, piece = i % PIECES, rr = (warp & 3) * 32 + r;
        const int q = rr / a.group;
        if (q < qt && x * qt + q < tile.count)
          reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) +
                                   ((tile.token + x * qt + q) * a.num_q_heads + h * a.group + rr - q * a.group) * D + hf * (D / 2))[piece] =
              reinterpret_cast<const uint4*>(stage)[r * PIECES + (piece ^ (r & (PIECES - 1)))];
      }
      if (valid && a.lse && hf == 0) a.lse[at] = l == 0.f ? -INFINITY : (m_ref + __log2f(l) - p_bias<F16>()) * LN2F;
    }
    tc_fence_before();
  }
  __syncthreads();
  if (*abort_flag) __nanosleep(50000);
  if (warp == C::WARPS + 1) tmem_dealloc(tmem_base, C::TMEM_COLS);
}

template <int D, bool F16, int MODE, int TILES>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, Args a, cudaStream_t st) {
  using C = Cfg<D, MODE, TILES>;
  auto kern = dense_pair_kernel<D, F16, MODE, TILES>;
  SEMBLO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::TOTAL));
  a.queries_per_tile = TILES * (128 / a.group);
  const unsigned grid = (unsigned)((ceil_div(a.tokens_q, a.queries_per_tile) + a.docs) * a.num_kv_heads * a.splits);
  kern<<<grid, C::THREADS, C::TOTAL, st>>>(mq, mk, mv, a);
  SEMBLO_LAUNCH_CHECK();
  return 0;
}

// One row tile per block, two blocks per multiprocessor, instead of two tiles that take turns in one block: twice
// the loads of K and V, but a block's beginning and end (about 6 us without products) overlap the other block's
// work.  us, 32 heads over 8, two tiles against one: 64 tokens x 128 10.6 : 7.6; 64 documents in 8192 tokens 108 :
// 79, 16 of them 126 : 113, 8 of them 190 : 188, one 508 : 559; a window of 512 in 16384 271 : 232; at head
// dimension 64 with 16 documents 104 : 100, with 8 166 : 174.  Where the softmax weighs most (a bias by
// distance; a cap in fp16) one tile is no slower at any length: biased, 16384 tokens x 128 3457 : 3057 us; capped,
// fp16, 8 heads over 2 x 64 830 : 822.
bool one_tile(const Args& a, int head_dim, int mode) {
  if (mode == BIASED || mode == CAPPED || a.splits > 1) return true;
  int64_t reach = a.tokens_k / std::max(1, a.docs);
  if (a.window > 0) reach = std::min<int64_t>(reach, a.window + BN);
  return reach <= (head_dim == 128 ? 1024 : 640);
}

}  // namespace

namespace dense {

int launch_pair(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, const Args& a, int head_dim,
                bool f16, int mode, cudaStream_t st) {
  const bool single = one_tile(a, head_dim, mode);
#define SEMBLO_PAIR(DD, FF, MM)                                                          \
  if (head_dim == DD && f16 == FF && mode == MM) {                                       \
    if constexpr (MM == LINEAR || MM == BOUNDED)                                         \
      if (!single) return launch<DD, FF, MM, 2>(mk, mv, mq, a, st);                      \
    return launch<DD, FF, MM, 1>(mk, mv, mq, a, st);                                     \
  }
  SEMBLO_PAIR(64, false, LINEAR) SEMBLO_PAIR(64, false, CAPPED) SEMBLO_PAIR(64, false, BIASED)
  SEMBLO_PAIR(64, false, BOUNDED) SEMBLO_PAIR(128, false, BOUNDED)
  SEMBLO_PAIR(64, true, LINEAR) SEMBLO_PAIR(64, true, CAPPED) SEMBLO_PAIR(64, true, BIASED)
  SEMBLO_PAIR(128, false, LINEAR) SEMBLO_PAIR(128, false, CAPPED) SEMBLO_PAIR(128, false, BIASED)
  SEMBLO_PAIR(128, true, LINEAR) SEMBLO_PAIR(128, true, CAPPED) SEMBLO_PAIR(128, true, BIASED)
#undef SEMBLO_PAIR
  return semblo::fail(semblo::SEMBLO_EINVAL, "unreachable");
}

}  // namespace dense
