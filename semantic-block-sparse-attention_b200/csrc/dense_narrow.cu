// Attention of packed prompts for head dimensions 64 and 128 (the mathematics is in dense_prefill.cu).
//
// A block owns 128 rows (queries x the heads of a KV head); two blocks share a multiprocessor, so that one's
// beginning, end and waits overlap the other's work.  S has two buffers of 64 keys and O the other half of a block's
// tensor memory (D = 128): S(t + 1) is complete before the softmax of S(t) ends, which is what has to keep up (16384
// exponentials per 128 x 128 scores at 16 a clock are as many clocks as both products).  One thread per row; P lies
// over the S it came from, Q, K and V are in shared memory (Q, and a ring of 64-key K, V tiles by TMA).
// Before that a block owned two such tiles with one S of 128 keys each and the softmax waited for the products:
// 32 heads over 8 x 128, us: 8192 tokens 503 -> 472, biased 920 -> 705, capped at 50 with a window of 4096
// 758 -> 651, 64 documents in 8192 tokens 107 -> 76 (495, 750, 703 and 77 since O is divided by the rounded sum).
#include <algorithm>

#include "dense_narrow.h"
#include "host_common.h"

using namespace dense;
using semblo::ceil_div;

namespace {

constexpr int BN = NARROW_BN;
constexpr int PAGE = 16;

template <int D>
struct Cfg {
  static constexpr int WARPS = 4;                              // of the softmax; then the loading and the issuing warp
  static constexpr int THREADS = (WARPS + 2) * 32;
  static constexpr int SLABS = D / 64;                         // 128-byte wide slabs of a 16-bit tile
  static constexpr int TILE = 128 * D * 2;                     // of Q
  static constexpr int KV = BN * D * 2;                        // of K or V
  static constexpr int SLOTS = D == 128 ? 5 : 8;
  static constexpr int Q_OFF = 0;
  static constexpr int KV_OFF = TILE;
  static constexpr int BAR_OFF = KV_OFF + SLOTS * KV;
  static constexpr int FIND_OFF = BAR_OFF + 320;               // of the search among many documents
  static constexpr int TOTAL = BAR_OFF + 512;
  static constexpr int S_COL = 0;                              // + 64 b: S and P, buffer b
  static constexpr int O_COL = 2 * BN;
  static constexpr int TMEM_COLS = 256;
};

enum { B_Q = 0, B_S = 1, B_P = 3, B_V = 5, B_O = 7, B_FULL = 8 };      // S full, P full, P V complete: + buffer

template <int D, bool F16, int MODE>
__global__ void __launch_bounds__(Cfg<D>::THREADS, 2)
dense_narrow_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                  const __grid_constant__ CUtensorMap tmap_v, const Args a) {
  using C = Cfg<D>;
  constexpr int SLOTS = C::SLOTS;
  constexpr int B_EMPTY = B_FULL + SLOTS;
  static_assert(8 * (B_EMPTY + SLOTS) <= 320, "barrier area");
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
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(B_S + b), 1);
      mbar_init(bar(B_P + b), C::WARPS);
      mbar_init(bar(B_V + b), 1);
    }
    mbar_init(bar(B_O), 1);
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
  const Tile tile = a.docs <= WARP_DOCS ? find_tile(a, share.want) : find_tile_block<C::THREADS>(a, share.want, smem + C::FIND_OFF);
  if (tile.doc < 0) {
    if (a.zero_tail && share.split == 0) zero_rest<D>(a, tile.first, h, blockDim.x);
    return;
  }
  KeyTiles<BN> keys(a, tile);
  const int pieces = pieces_of(a, keys.n, BN);
  if (share.split >= pieces) return;
  keys.base = (int)((int64_t)keys.n * share.split / pieces);
  keys.n = (int)((int64_t)keys.n * (share.split + 1) / pieces) - keys.base;
  auto load_kv = [&](int i) {                      // K(i / 2) or V(i / 2) into its slot, which is free
    const int s = i % SLOTS, row = tile.k0 + keys.at(i >> 1);
    mbar_arrive_expect_tx(bar(B_FULL + s), (uint32_t)C::KV);
    for (int sl = 0; sl < C::SLABS; ++sl)
      tma_load_3d(smem_u32(smem + C::KV_OFF + s * C::KV + sl * BN * 128), (i & 1) ? &tmap_v : &tmap_k, bar(B_FULL + s),
                  sl * 64, h, row);
  };
  if (warp == C::WARPS && lane == 0 && keys.n > 0) {
    mbar_arrive_expect_tx(bar(B_Q), (uint32_t)(C::SLABS * a.queries_per_tile * a.group * 128));
    for (int sl = 0; sl < C::SLABS; ++sl)
      tma_load_3d(smem_u32(smem + C::Q_OFF + sl * 128 * 128), &tmap_q, bar(B_Q), sl * 64, h * a.group, (int)tile.token);
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
      for (int i = 2; i < 2 * keys.n; ++i) {
        if (!mbar_wait(bar(B_EMPTY + i % SLOTS), ((i / SLOTS) & 1) ^ 1, abort_flag, a.status, STATUS_TIMEOUT_LOAD)) break;
        load_kv(i);
      }
    }
  } else if (warp == C::WARPS + 1) {
    // ------------------------------------------------------------ UMMA issuer
    // UMMAs of one thread execute in order: S(j + 2) may overwrite the P that the P V before it reads.
    if (elect_one()) {
      constexpr uint32_t idesc_pv = idesc_of<F16>(128, D, true);
      const int n = keys.n;
      bool ok = n == 0 || mbar_wait(bar(B_Q), 0, abort_flag, a.status, STATUS_TIMEOUT_MMA);
      auto keys_of = [&](int j) { return min(BN, tile.lk - keys.at(j)); };
      auto wait_slot = [&](int i) {
        ok = ok && mbar_wait(bar(B_FULL + i % SLOTS), (i / SLOTS) & 1, abort_flag, a.status, STATUS_TIMEOUT_MMA);
        return ok;
      };
      auto issue_s = [&](int j) {
        tc_fence_after();
        const uint32_t q_base = smem_u32(smem + C::Q_OFF), k_base = smem_u32(smem + C::KV_OFF + (2 * j) % SLOTS * C::KV);
        const uint32_t idesc = idesc_of<F16>(128, (keys_of(j) + PAGE - 1) / PAGE * PAGE, false);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_ss(tmem_base + C::S_COL + (j & 1) * BN, make_smem_desc(q_base + (kk >> 2) * 128 * 128 + (kk & 3) * 32, 16, 1024),
                  make_smem_desc(k_base + (kk >> 2) * BN * 128 + (kk & 3) * 32, 16, 1024), idesc, kk > 0 ? 1u : 0u);
        umma_commit(bar(B_S + (j & 1)));
        umma_commit(bar(B_EMPTY + (2 * j) % SLOTS));
      };
      for (int j = 0; j < 2 && j < n && wait_slot(2 * j); ++j) issue_s(j);
      for (int j = 0; ok && j < n; ++j) {
        const int pages = (keys_of(j) + PAGE - 1) / PAGE, b = j & 1;
        const uint32_t v_base = smem_u32(smem + C::KV_OFF + (2 * j + 1) % SLOTS * C::KV);
        if (!wait_slot(2 * j + 1)) break;
        ok = mbar_wait(bar(B_P + b), (j >> 1) & 1, abort_flag, a.status, STATUS_TIMEOUT_MMA);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < BN / PAGE; ++kk)
          if (kk < pages)
            umma_ts(tmem_base + C::O_COL, tmem_base + C::S_COL + b * BN + kk * 8,
                    make_smem_desc(v_base + kk * PAGE * 128, BN * 128, 1024), idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
        umma_commit(bar(B_V + b));
        umma_commit(bar(B_EMPTY + (2 * j + 1) % SLOTS));
        if (j + 2 < n && wait_slot(2 * j + 4)) issue_s(j + 2);
      }
      if (ok) umma_commit(bar(B_O));
    }
  } else {
    // ------------------------------------------------------------ softmax + epilogue: one thread per row
    const int row = threadIdx.x & 127;
    const int qi = row / a.group, hg = row - qi * a.group;
    const bool valid = qi < tile.count;
    // a row that no query has counts as the last query's, so that its warp need not mask more than that
    const int p = tile.pos + min(qi, tile.count - 1);
    const Seen seen = seen_by(a, tile, p);
    const bool idle = warp * 32 >= tile.count * a.group;     // no row of this warp has a query
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_addr + C::S_COL;
    const uint32_t o_addr = tmem_base + lane_addr + C::O_COL;
    const int head = h * a.group + hg;
    const float slope = a.slopes && valid ? a.slopes[head] * LOG2EF : 0.f;
    const float scale = scale_of<MODE>(a);
    const Vote vote(valid);
    const TanhPoly<MODE == BOUNDED ? 5 : 8> capped(a.cap_log2);
    float m_ref = MODE == BOUNDED ? bounded_reference(a.cap_log2) : -INFINITY, l = 0.f, lr = 0.f;
    bool ok = true;
    for (int j = 0; j < keys.n; ++j) {
      const int key0 = keys.at(j), b = j & 1;
      ok = mbar_wait_warp(bar(B_S + b), (uint32_t)((j >> 1) & 1), abort_flag, a.status, STATUS_TIMEOUT_SOFTMAX);
      if (!ok) break;
      if (idle) {                                  // whatever P is
        if (lane == 0) mbar_arrive(bar(B_P + b));
        continue;
      }
      tc_fence_after();
      const uint32_t s_buf = s_addr + b * BN;
      if constexpr (MODE == BOUNDED) {
        // no maximum: 32 keys, with the next ones' scores on their way
        RowSum<F16> sum;
        uint32_t held[2][32];
        tmem_ld32(s_buf, held[0]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t (&s)[32] = held[c];
          tmem_ld_wait();
          if (c == 0) tmem_ld32(s_buf + 32, held[1]);
          const int lo = seen.lo - key0 - 32 * c, hi = seen.hi - key0 - 32 * c, pre = seen.pre - key0 - 32 * c;
          const bool all = __all_sync(0xffffffffu, (lo <= 0 && hi >= 32) || pre >= 32);
          bounded32(s, a, capped, all, seen_bits(lo, hi, pre), -m_ref, vote);
          uint32_t packed[16];
#pragma unroll
          for (int n = 0; n < 16; ++n) {
            const float e0 = fast_exp2(__uint_as_float(s[2 * n])), e1 = fast_exp2(__uint_as_float(s[2 * n + 1]));
            packed[n] = pack_pair<F16>(e0, e1);
            sum.add(n, e0, e1, packed[n]);
          }
          tmem_st16(s_buf + c * 16, packed);
        }
        sum.into(l, lr);
      } else {
        constexpr int CH = 2;
        uint32_t s[CH][32];
#pragma unroll
        for (int c = 0; c < CH; ++c) tmem_ld32(s_buf + c * 32, s[c]);
        tmem_ld_wait();
        const int lo = seen.lo - key0, hi = seen.hi - key0, pre = seen.pre - key0;
        const bool all = __all_sync(0xffffffffu, (lo <= 0 && hi >= 32 * CH) || pre >= 32 * CH);
        float tmax = -INFINITY, least = INFINITY;
        bool poly = false;                             // tanh by polynomial, in the exponential's pass
        if constexpr (MODE != BIASED) {
#pragma unroll
          for (int c = 0; c < CH; ++c) range32<MODE == CAPPED>(s[c], tmax, least);
        }
        if constexpr (MODE == CAPPED) {
          poly = all && __all_sync(0xffffffffu, fmaxf(tmax, -least) * a.score_scale < vote.far);
          if (poly) tmax = tanh_any(tmax * (a.score_scale * (1.f / TANH_ARG)));
        }
        if (MODE == BIASED || (MODE == CAPPED && !poly) || (MODE == LINEAR && !all)) {
          tmax = -INFINITY;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const uint32_t bits = seen_bits(lo - 32 * c, hi - 32 * c, pre - 32 * c);
            transform32<MODE>(s[c], a, slope, p, key0 + 32 * c, all, bits, vote);
            if (!all) hide32(s[c], bits);
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
          lr *= alpha;
        } else if (m_ref == -INFINITY) {
          m_ref = tmax;
        }
        if (__any_sync(0xffffffffu, need)) {
          // O must be quiescent: the step before's P V has to be complete
          ok = mbar_wait_warp(bar(B_V + (b ^ 1)), (uint32_t)(((j - 1) >> 1) & 1), abort_flag, a.status,
                              STATUS_TIMEOUT_SOFTMAX);
          if (!ok) break;
          tc_fence_after();
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
        RowSum<F16> sum;
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
              sum.add(i, e0, e1, packed[i]);
            }
            tmem_st16(s_buf + c * 16, packed);
          }
        };
        if (MODE == CAPPED && poly) {
          const f32x2 arg2 = join(a.score_scale, a.score_scale);
          exponentials([&](f32x2 v) { return capped(mul2(v, arg2), neg2); });
        } else {
          exponentials([&](f32x2 v) { return fma2(v, scale2, neg2); });
        }
        sum.into(l, lr);
      }
      // V's rows behind the document's end (another document's, or anything) are cleared: their P is 0, but 0 * NaN
      // would not vanish
      const int left = tile.lk - key0;
      if (warp == 0 && left < BN && (left & (PAGE - 1))) {
        ok = mbar_wait_warp(bar(B_FULL + (2 * j + 1) % SLOTS), ((2 * j + 1) / SLOTS) & 1, abort_flag, a.status,
                            STATUS_TIMEOUT_SOFTMAX);
        if (!ok) break;
        zero_rows<D, BN>(smem + C::KV_OFF + (2 * j + 1) % SLOTS * C::KV, left, (left + PAGE - 1) / PAGE * PAGE);
        fence_proxy_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_P + b));
    }
    if (ok) ok = mbar_wait_warp(bar(B_O), 0, abort_flag, a.status, STATUS_TIMEOUT_EPILOGUE);
    tc_fence_after();
    if (ok && pieces > 1) {
      float* record = share.record(a, D, share.split);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) store_partial(o_addr + c * 32, record + row * D + c * 32, valid);
      if (valid) {
        record[128 * D + row] = m_ref;
        record[128 * D + 128 + row] = l;
        record[128 * D + 256 + row] = lr;
      }
    } else if (ok) {
      const float inv = lr == 0.f ? 0.f : 1.f / lr;
      const int64_t at = (tile.token + qi) * a.num_q_heads + head;
      // through Q's shared memory (no product is in flight any more), a warp's own part of it
      constexpr int PIECES = D / 8;
      uint8_t* stage = smem + C::Q_OFF + warp * 32 * PIECES * 16;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (keys.n > 0) {
          tmem_ld32(o_addr + c * 32, o);
          tmem_ld_wait();
        }
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          w[i] = lr == 0.f ? 0u : pack_pair<F16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
        stage_pieces<PIECES>(stage, c * 4, w);
      }
      __syncwarp();
#pragma unroll 4
      for (int i = lane; i < 32 * PIECES; i += 32) {
        const int r = i / PIECES, piece = i % PIECES, rr = (warp & 3) * 32 + r;
        const int q = rr / a.group;
        if (q < tile.count)
          reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) +
                                   ((tile.token + q) * a.num_q_heads + h * a.group + rr - q * a.group) * D)[piece] =
              reinterpret_cast<const uint4*>(stage)[r * PIECES + (piece ^ (r & (PIECES - 1)))];
      }
      if (valid && a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m_ref + __log2f(l) - p_bias<F16>()) * LN2F;
    }
    tc_fence_before();
  }
  __syncthreads();
  if (*abort_flag) __nanosleep(50000);
  if (warp == C::WARPS + 1) tmem_dealloc(tmem_base, C::TMEM_COLS);
}

template <int D, bool F16, int MODE>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, const Args& a, cudaStream_t st) {
  using C = Cfg<D>;
  auto kern = dense_narrow_kernel<D, F16, MODE>;
  SEMBLO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::TOTAL));
  const unsigned grid = (unsigned)((ceil_div(a.tokens_q, a.queries_per_tile) + a.docs) * a.num_kv_heads * a.splits);
  kern<<<grid, C::THREADS, C::TOTAL, st>>>(mq, mk, mv, a);
  SEMBLO_LAUNCH_CHECK();
  return 0;
}

}  // namespace

namespace dense {

int launch_narrow(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, const Args& a, int head_dim,
                  bool f16, int mode, cudaStream_t st) {
#define SEMBLO_NARROW(DD, FF, MM) \
  if (head_dim == DD && f16 == FF && mode == MM) return launch<DD, FF, MM>(mk, mv, mq, a, st);
  SEMBLO_NARROW(64, false, LINEAR) SEMBLO_NARROW(64, false, CAPPED) SEMBLO_NARROW(64, false, BIASED)
  SEMBLO_NARROW(64, false, BOUNDED) SEMBLO_NARROW(128, false, BOUNDED)
  SEMBLO_NARROW(64, true, LINEAR) SEMBLO_NARROW(64, true, CAPPED) SEMBLO_NARROW(64, true, BIASED)
  SEMBLO_NARROW(128, false, LINEAR) SEMBLO_NARROW(128, false, CAPPED) SEMBLO_NARROW(128, false, BIASED)
  SEMBLO_NARROW(128, true, LINEAR) SEMBLO_NARROW(128, true, CAPPED) SEMBLO_NARROW(128, true, BIASED)
#undef SEMBLO_NARROW
  return semblo::fail(semblo::SEMBLO_EINVAL, "unreachable");
}

}  // namespace dense
