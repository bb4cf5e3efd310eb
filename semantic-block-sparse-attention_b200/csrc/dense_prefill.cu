// Attention of packed prompts (documents) on tcgen05 / TMEM, with a soft cap on the scores, a bias by
// distance, a local window and a prefix that every query of a document sees.
//
//   s_ij = cap tanh(q_i . k_j sm / cap)  (or q_i . k_j sm) - slope_h |p_i - j|,   p_i = Lk - Lq + i
//   key j of the document is seen when (j <= p_i and p_i - j < window) or j < prefix   (causal; else always)
//   o_i  = sum_j 2^(s_ij log2e - m_i) v_j / sum_j 2^(s_ij log2e - m_i), one pass with a running m_i
//
// This file: the entry point, and the kernel for D = 256.  One block owns 128 rows (queries x the heads of a KV
// head, heads adjacent) and walks over the 64-key tiles that any of them sees.  Q, P, S (two buffers) and O
// fill tensor memory, K and V come by TMA.  Softmax: 8 warps, two threads per row; one thread issues the
// products in the fixed order S(0), S(1), then P V(t), S(t + 2).
#include <algorithm>

#include "../../include/semblo_b200.h"
#include "dense_common.cuh"
#include "dense_narrow.h"
#include "host_common.h"

using namespace dense;
using semblo::ceil_div;

namespace {

constexpr int BN = 64;
constexpr int PAGE = 16;

template <int D>
struct Cfg {
  static constexpr int STAGES = 3;
  static constexpr int KV_BYTES = BN * D * 2;
  static constexpr int K_OFF = 0;
  static constexpr int V_OFF = K_OFF + STAGES * KV_BYTES;
  static constexpr int EPI_OFF = V_OFF + STAGES * KV_BYTES;   // float [2][2][128]
  static constexpr int MX_OFF = EPI_OFF + 2048;               // float [2][2][128]: half-row maxima
  static constexpr int BAR_OFF = MX_OFF + 2048;
  static constexpr int SLOT_OFF = BAR_OFF + 256;
  static constexpr int FIND_OFF = SLOT_OFF + 64;              // of the search among many documents
  static constexpr int TOTAL = FIND_OFF + FIND_BYTES;
  static constexpr int O_COL = 2 * BN;                        // S/P buffers, then O, then Q
  static constexpr int Q_COL = O_COL + D;
  static constexpr int TMEM_COLS = 512;
  static_assert(Q_COL + D / 2 <= 512, "tensor memory budget");
};

enum { B_QFULL = 0, B_OREADY = 1, B_SFULL = 2, B_PFULL = 4, B_PVDONE = 6, B_EPI = 8, B_PAIR = 9, B_KVFULL = 13 };

template <int D, bool F16, int MODE>
__global__ void __launch_bounds__(320, 1)
dense_prefill_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                     const Args a) {
  using C = Cfg<D>;
  constexpr int STAGES = C::STAGES;
  constexpr int B_KVEMPTY = B_KVFULL + STAGES;
  static_assert(8 * (B_KVEMPTY + STAGES) <= 256, "barrier area");
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Share share(a, a.splits);
  const int h = share.h;
  if (smem_u32(smem) & 1023u) {                    // the swizzled tiles need 1024-byte alignment
    if (threadIdx.x == 0) atomicCAS(a.status, 0, STATUS_SMEM_ALIGN);
    return;
  }
  const Tile tile = a.docs <= WARP_DOCS ? find_tile(a, share.want) : find_tile_block<320>(a, share.want, smem + C::FIND_OFF);
  if (tile.doc < 0) {
    if (a.zero_tail && share.split == 0) zero_rest<D>(a, tile.first, h, blockDim.x);
    return;
  }
  KeyTiles<BN> keys(a, tile);
  const int pieces = pieces_of(a, keys.n, BN);
  if (share.split >= pieces) return;
  keys.base = (int)((int64_t)keys.n * share.split / pieces);
  keys.n = (int)((int64_t)keys.n * (share.split + 1) / pieces) - keys.base;

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::SLOT_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  if (threadIdx.x == 0) {
    mbar_init(bar(B_QFULL), 256);
    mbar_init(bar(B_OREADY), 1);
    mbar_init(bar(B_EPI), 256);
    for (int i = 0; i < 4; ++i) mbar_init(bar(B_PAIR + i), 2);    // the two warps that share 32 rows
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(B_SFULL + b), 1);
      mbar_init(bar(B_PFULL + b), 8);         // the softmax warps
      mbar_init(bar(B_PVDONE + b), 1);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar(B_KVFULL + s), 1);
      mbar_init(bar(B_KVEMPTY + s), 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 8) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&tmap_k);
      tma_prefetch_desc(&tmap_v);
      bool ok = true;
      for (int j = 0; j < keys.n && ok; ++j) {
        const int s = j % STAGES;
        ok = mbar_wait(bar(B_KVEMPTY + s), ((j / STAGES) & 1) ^ 1, abort_flag, a.status, STATUS_TIMEOUT_LOAD);
        if (!ok) break;
        const int row = tile.k0 + keys.at(j);
        mbar_arrive_expect_tx(bar(B_KVFULL + s), (uint32_t)C::KV_BYTES * 2);
        for (int sl = 0; sl < D / 64; ++sl) {
          tma_load_3d(smem_u32(smem + C::K_OFF + s * C::KV_BYTES + sl * BN * 128), &tmap_k, bar(B_KVFULL + s), sl * 64, h, row);
          tma_load_3d(smem_u32(smem + C::V_OFF + s * C::KV_BYTES + sl * BN * 128), &tmap_v, bar(B_KVFULL + s), sl * 64, h, row);
        }
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ UMMA issuer
    // inside elect_one() as a whole: issued from `if (lane == 0)` between warp barriers the same products ran 30 %
    // slower
    if (elect_one()) {
      constexpr uint32_t idesc_pv = idesc_of<F16>(128, D, true);
      bool ok = mbar_wait(bar(B_QFULL), 0, abort_flag, a.status, STATUS_TIMEOUT_MMA);
      tc_fence_after();
      const int n = keys.n;
      int qs = 0;                                      // stage of the next S product
      uint32_t q_par = 0;
      auto pages_of = [&](int j) { return min(BN / PAGE, (tile.lk - keys.at(j) + PAGE - 1) / PAGE); };
      auto issue_s = [&](int j) {
        ok = mbar_wait(bar(B_KVFULL + qs), q_par, abort_flag, a.status, STATUS_TIMEOUT_MMA);
        if (!ok) return;
        tc_fence_after();
        const int b = j & 1;
        const uint32_t k_base = smem_u32(smem + C::K_OFF + qs * C::KV_BYTES);
        const uint32_t idesc_qk = idesc_of<F16>(128, pages_of(j) * PAGE, false);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t sl = kk >> 2, ko = (kk & 3) * 32;
          umma_ts(tmem_base + b * BN, tmem_base + C::Q_COL + kk * 8,
                  make_smem_desc(k_base + sl * BN * 128 + ko, 16, 1024), idesc_qk, kk > 0 ? 1u : 0u);
        }
        umma_commit(bar(B_SFULL + b));
        if (++qs == STAGES) { qs = 0; q_par ^= 1; }
      };
      for (int j = 0; j < 2 && j < n && ok; ++j) issue_s(j);
      int vs = 0;
      for (int t = 0; ok && t < n; ++t) {
        const int b = t & 1;
        ok = mbar_wait(bar(B_PFULL + b), (uint32_t)((t >> 1) & 1), abort_flag, a.status, STATUS_TIMEOUT_MMA);
        if (!ok) break;
        tc_fence_after();
        const int np = pages_of(t);
        const uint32_t v_base = smem_u32(smem + C::V_OFF + vs * C::KV_BYTES);
        for (int kk = 0; kk < np; ++kk)
          umma_ts(tmem_base + C::O_COL, tmem_base + b * BN + (kk >> 1) * 32 + (kk & 1) * 8,
                  make_smem_desc(v_base + kk * PAGE * 128, BN * 128, 1024), idesc_pv, (t > 0 || kk > 0) ? 1u : 0u);
        umma_commit(bar(B_KVEMPTY + vs));
        umma_commit(bar(B_PVDONE + b));
        if (++vs == STAGES) vs = 0;
        if (t + 2 < n) issue_s(t + 2);
      }
      if (ok) umma_commit(bar(B_OREADY));
    }
  } else {
    // ------------------------------------------------------------ softmax + epilogue
    // warps 0-3 take columns [0, 32) of every tile and warps 4-7 columns [32, 64); thread = row
    const int hf = warp >> 2;
    const int row = threadIdx.x & 127;
    const int qi = row / a.group, hg = row - qi * a.group;
    const bool valid = qi < tile.count;
    // a row that no query has counts as the last query's, so that its warp need not mask more than that
    const int p = tile.pos + min(qi, tile.count - 1);
    const Seen seen = seen_by(a, tile, p);
    const bool idle = (warp & 3) * 32 >= tile.count * a.group;     // no row of this warp has a query
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const int head = h * a.group + hg;
    const float slope = a.slopes && valid ? a.slopes[head] * LOG2EF : 0.f;
    {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                                        (tile.token + qi) * a.q_token + head * a.q_head + hf * (D / 2));
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {           // 32 elements of this half: 16 columns
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 v = valid ? __ldg(src + c * 4 + i) : make_uint4(0u, 0u, 0u, 0u);
          w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
        tmem_st16(tmem_base + lane_addr + C::Q_COL + hf * (D / 4) + c * 16, w);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(bar(B_QFULL));
    }
    const float scale = scale_of<MODE>(a);
    const Vote vote(valid);
    const TanhPoly<MODE == BOUNDED ? 5 : 8> capped(a.cap_log2);
    float m_ref = MODE == BOUNDED ? bounded_reference(a.cap_log2) : -INFINITY, l_part = 0.f, lr_part = 0.f;
    bool ok = true;
    float* mx = reinterpret_cast<float*>(smem + C::MX_OFF);
    for (int j = 0; j < keys.n; ++j) {
      const int b = j & 1, key0 = keys.at(j) + 32 * hf;
      ok = mbar_wait_warp(bar(B_SFULL + b), (uint32_t)((j >> 1) & 1), abort_flag, a.status, STATUS_TIMEOUT_SOFTMAX);
      if (!ok) break;
      if (idle) {                                  // whatever P is
        if (lane == 0) mbar_arrive(bar(B_PFULL + b));
        continue;
      }
      tc_fence_after();
      const uint32_t s_addr = tmem_base + lane_addr + b * BN + hf * 32;
      const bool active = tile.lk > key0;                // the product wrote at least one page of this half
      uint32_t x[32];
      if constexpr (MODE == BOUNDED) {
        if (active) {
          tmem_ld32(s_addr, x);
          tmem_ld_wait();
          const int lo = seen.lo - key0, hi = seen.hi - key0, pre = seen.pre - key0;
          const bool all = __all_sync(0xffffffffu, (lo <= 0 && hi >= 32) || pre >= 32);
          bounded32(x, a, capped, all, seen_bits(lo, hi, pre), -m_ref, vote);
          uint32_t packed[16];
          RowSum<F16> sum;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float e0 = fast_exp2(__uint_as_float(x[2 * i])), e1 = fast_exp2(__uint_as_float(x[2 * i + 1]));
            packed[i] = pack_pair<F16>(e0, e1);
            sum.add(i, e0, e1, packed[i]);
          }
          sum.into(l_part, lr_part);
          tmem_st16(s_addr, packed);
        }
      } else {
        float hm = -INFINITY, least = INFINITY;
        bool poly = MODE == CAPPED;                        // this half's tanh by polynomial, in the exponential's pass
        if (active) {
          tmem_ld32(s_addr, x);
          tmem_ld_wait();
          const int lo = seen.lo - key0, hi = seen.hi - key0, pre = seen.pre - key0;
          const bool all = __all_sync(0xffffffffu, (lo <= 0 && hi >= 32) || pre >= 32);
          if constexpr (MODE == CAPPED) {
            range32<true>(x, hm, least);
            poly = all && __all_sync(0xffffffffu, fmaxf(hm, -least) * a.score_scale < vote.far);
            if (poly) hm = tanh_any(hm * (a.score_scale * (1.f / TANH_ARG)));
          }
          if (!poly) {
            const uint32_t bits = seen_bits(lo, hi, pre);
            transform32<MODE>(x, a, slope, p, key0, all, bits, vote);
            if (!all) hide32(x, bits);
            hm = -INFINITY;
            range32<false>(x, hm, least);
          }
        }
        float* slot = mx + b * 256;
        slot[hf * 128 + row] = hm;
        __syncwarp();                                      // one arrival per warp: the barrier counts warps
        if (lane == 0) mbar_arrive(bar(B_PAIR + (warp & 3)));
        ok = mbar_wait_warp(bar(B_PAIR + (warp & 3)), (uint32_t)(j & 1), abort_flag, a.status, STATUS_TIMEOUT_SOFTMAX);
        if (!ok) break;
        const float tmax = fmaxf(hm, slot[(hf ^ 1) * 128 + row]) * scale;
        // lazy rescale: only when the running reference falls far behind
        const bool need = m_ref != -INFINITY && tmax > m_ref + rescale_gap<F16>();
        float alpha = 1.f;
        if (need) {
          alpha = fast_exp2(m_ref - tmax);
          m_ref = tmax;
          l_part *= alpha;
          lr_part *= alpha;
        } else if (m_ref == -INFINITY) {
          m_ref = tmax;
        }
        if (__any_sync(0xffffffffu, need)) {
          // O must be quiescent: the previous tile's P V has to be complete
          ok = mbar_wait_warp(bar(B_PVDONE + ((j - 1) & 1)), (uint32_t)(((j - 1) >> 1) & 1), abort_flag, a.status,
                              STATUS_TIMEOUT_SOFTMAX);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 64; ++c) {
            uint32_t o[32];
            const uint32_t addr = tmem_base + lane_addr + C::O_COL + hf * (D / 2) + c * 32;
            tmem_ld32(addr, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(addr, o);
          }
        }
        if (active) {
          const float neg_m = m_ref == -INFINITY ? 0.f : p_bias<F16>() - m_ref;
          uint32_t packed[16];
          RowSum<F16> sum;
          auto exponentials = [&](auto argument) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float e0, e1;
              split(argument(join(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]))), e0, e1);
              e0 = fast_exp2(e0);
              e1 = fast_exp2(e1);
              packed[i] = pack_pair<F16>(e0, e1);
              sum.add(i, e0, e1, packed[i]);
            }
          };
          const f32x2 neg2 = join(neg_m, neg_m), scale2 = join(scale, scale);
          if (MODE == CAPPED && poly) {
            const f32x2 arg2 = join(a.score_scale, a.score_scale);
            exponentials([&](f32x2 v) { return capped(mul2(v, arg2), neg2); });
          } else {
            exponentials([&](f32x2 v) { return fma2(v, scale2, neg2); });
          }
          sum.into(l_part, lr_part);
          // P lies over this half's own logits; P V takes its 16-key slices from columns 0, 8, 32 and 40
          tmem_st16(s_addr, packed);
        }
      }
      // V's rows behind the document's end (another document's, or anything) are cleared: their P is 0, but 0 * NaN
      // would not vanish.  S's barrier says that the stage has arrived
      const int left = tile.lk - keys.at(j);
      if (warp == 0 && left < BN && (left & (PAGE - 1))) {
        zero_rows<D, BN>(smem + C::V_OFF + j % STAGES * C::KV_BYTES, left, (left + PAGE - 1) / PAGE * PAGE);
        fence_proxy_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_PFULL + b));
    }
    if (ok) ok = mbar_wait_warp(bar(B_OREADY), 0, abort_flag, a.status, STATUS_TIMEOUT_EPILOGUE);
    tc_fence_after();
    float* xchg = reinterpret_cast<float*>(smem + C::EPI_OFF);
    xchg[hf * 128 + row] = l_part;
    xchg[256 + hf * 128 + row] = lr_part;
    mbar_arrive(bar(B_EPI));
    if (ok) ok = mbar_wait_warp(bar(B_EPI), 0, abort_flag, a.status, STATUS_TIMEOUT_EPILOGUE);
    if (ok && pieces > 1) {
      const float l = l_part + xchg[(hf ^ 1) * 128 + row], lr = lr_part + xchg[256 + (hf ^ 1) * 128 + row];
      float* record = share.record(a, D, share.split);
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c)
        store_partial(tmem_base + lane_addr + C::O_COL + hf * (D / 2) + c * 32, record + row * D + hf * (D / 2) + c * 32, valid);
      if (valid && hf == 0) {
        record[128 * D + row] = m_ref;
        record[128 * D + 128 + row] = l;
        record[128 * D + 256 + row] = lr;
      }
    } else if (ok) {
      const float l = l_part + xchg[(hf ^ 1) * 128 + row], lr = lr_part + xchg[256 + (hf ^ 1) * 128 + row];
      const float inv = lr == 0.f ? 0.f : 1.f / lr;
      const int64_t at = (tile.token + qi) * a.num_q_heads + head;
      uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at * D + hf * (D / 2));
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
        uint32_t o[32];
        if (keys.n > 0) {
          tmem_ld32(tmem_base + lane_addr + C::O_COL + hf * (D / 2) + c * 32, o);
          tmem_ld_wait();
        }
        if (valid) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            w[i] = lr == 0.f ? 0u : pack_pair<F16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
#pragma unroll
          for (int i = 0; i < 4; ++i) dst[c * 4 + i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
      }
      if (valid && a.lse && hf == 0) a.lse[at] = l == 0.f ? -INFINITY : (m_ref + __log2f(l) - p_bias<F16>()) * LN2F;
    }
    tc_fence_before();
  }
  __syncthreads();
  if (*abort_flag) __nanosleep(50000);
  if (warp == 0) tmem_dealloc(tmem_base, C::TMEM_COLS);
}

template <int D, bool F16, int MODE>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, cudaStream_t st) {
  using C = Cfg<D>;
  auto kern = dense_prefill_kernel<D, F16, MODE>;
  SEMBLO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::TOTAL));
  const unsigned grid = (unsigned)((ceil_div(a.tokens_q, a.queries_per_tile) + a.docs) * a.num_kv_heads * a.splits);
  kern<<<grid, 320, C::TOTAL, st>>>(mk, mv, a);
  SEMBLO_LAUNCH_CHECK();
  return 0;
}

template <int D, int BN_, bool F16>
int join_pieces(const Args& a, cudaStream_t st) {
  const int64_t units = (ceil_div(a.tokens_q, a.queries_per_tile) + a.docs) * a.num_kv_heads;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)units, (unsigned)std::max<int64_t>(1, std::min<int64_t>(D / 16, 4 * semblo::sm_count() / units)));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  SEMBLO_CUDA(cudaLaunchKernelEx(&cfg, join_pieces_kernel<D, BN_, F16>, a));
  return 0;
}

// Into how many pieces a tile's keys may be cut, and the least keys of a piece.  Pieces of 512 keys: as many as bring
// the longest tile down to what each multiprocessor would get of an even share (causal tiles differ, so that is up to
// twice the free room).  A tile's mean number of keys is what a document has less half its queries.  Where even half
// the blocks that fit are not there, pieces of 256: the join, which reads every piece, is small then.  us without
// and with, D = 128: 16 tokens x 32 heads over 8 behind 8192 others 139 -> 22, 128 behind 30000 463 -> 71, 512 behind
// 30000 469 -> 242, 8192 tokens x 4 heads over 1 136 -> 105, 11 tokens of 2 documents behind 1250 20 -> 13 (in pieces
// of 512: 20).  1024 tokens x 8 heads over 2 20 -> 24, so a tile of few keys is not cut: the mean tile (the longest is
// `skew` of it) has to have 1.5 large pieces, 768 keys, or 2 small ones, 512, since with fewer the second launch and the
// partials cost what the cut saves.
struct Split { int pieces, keys; };
Split split_for(int64_t tokens_q, int64_t tokens_k, int group, int num_kv_heads, int head_dim, int documents, int causal,
                int window, bool prefix) {
  if (documents == 0 || tokens_q == 0) return {1, 512};
  const int64_t qt = 128 / group, tiles = (tokens_q + documents * (qt - 1)) / qt;      // no more than these have queries
  const int64_t slots = (int64_t)semblo::sm_count() * (head_dim == 256 ? 1 : 2), units = tiles * num_kv_heads;
  int64_t keys = tokens_k / documents;
  if (window > 0 && !prefix) keys = std::min<int64_t>(keys, window + qt);
  // the longest tile's keys over the mean of all
  const double skew = causal && tokens_q < tokens_k ? 2.0 * tokens_k / (2.0 * tokens_k - tokens_q) : causal ? 2.0 : 1.0;
  int64_t large = keys < 768 * skew ? 1 : std::min<int64_t>((int64_t)(skew * slots / units), keys / 512);
  int64_t small = keys < 512 * skew ? 1 : std::min(slots / (2 * units), keys / 256);
  large = std::min<int64_t>(std::max<int64_t>(large, 1), 32);
  small = std::min<int64_t>(small, 32);
  return small > large ? Split{(int)small, 256} : Split{(int)large, 512};
}

int64_t split_bytes(int64_t tokens_q, int group, int num_kv_heads, int head_dim, int documents, int splits) {
  if (splits == 1) return 0;
  return (ceil_div(tokens_q, 128 / group) + documents) * num_kv_heads * splits * record_floats(head_dim) * 4;
}

int check_shape(int64_t tokens_q, int64_t tokens_k, int num_q_heads, int num_kv_heads, int head_dim, int documents,
                int causal, int window, bool prefix) {
  SEMBLO_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "head_dim must be 64, 128 or 256 (got %d)",
                 head_dim);
  SEMBLO_REQUIRE(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
                 "query heads must be a multiple of the KV heads");
  const int group = num_q_heads / num_kv_heads;
  SEMBLO_REQUIRE(group <= 128, "at most 128 query heads per KV head (got %d)", group);
  SEMBLO_REQUIRE(tokens_q >= 0 && tokens_k >= 0 && documents >= 0, "negative token or document count");
  SEMBLO_REQUIRE(tokens_q < ((int64_t)1 << 30) && tokens_k < ((int64_t)1 << 30) && documents < (1 << 30), "too many tokens");
  SEMBLO_REQUIRE((ceil_div(tokens_q, 128 / group) + documents) * num_kv_heads < ((int64_t)1 << 31),
                 "tokens x KV heads is too large for one call");
  SEMBLO_REQUIRE(window >= 0, "negative window");
  SEMBLO_REQUIRE(causal || (window == 0 && !prefix), "a window or a prefix needs the causal mask");
  return 0;
}

}  // namespace

extern "C" int64_t semblo_dense_prefill_workspace_bytes(int64_t tokens_q, int64_t tokens_k, int num_q_heads,
                                                        int num_kv_heads, int head_dim, int documents, int causal,
                                                        int window, int has_prefix) {
  const int rc = check_shape(tokens_q, tokens_k, num_q_heads, num_kv_heads, head_dim, documents, causal, window, has_prefix);
  if (rc) return rc;
  const int group = num_q_heads / num_kv_heads;
  return split_bytes(tokens_q, group, num_kv_heads, head_dim, documents,
                     split_for(tokens_q, tokens_k, group, num_kv_heads, head_dim, documents, causal, window, has_prefix).pieces);
}

extern "C" int semblo_dense_prefill(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                    int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                    int64_t v_token_stride, int64_t v_head_stride, int64_t tokens_q,
                                    int64_t tokens_k, int num_q_heads, int num_kv_heads, int head_dim, int dtype,
                                    const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int documents,
                                    int causal, int window, const int32_t* prefix_lens, float sm_scale,
                                    float softcap, const float* alibi_slopes, void* out, int zero_tail, float* lse,
                                    void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  const int rc0 = check_shape(tokens_q, tokens_k, num_q_heads, num_kv_heads, head_dim, documents, causal, window,
                              prefix_lens != nullptr);
  if (rc0) return rc0;
  const int group = num_q_heads / num_kv_heads;
  SEMBLO_REQUIRE(dtype == SEMBLO_BF16 || dtype == SEMBLO_F16, "prompts are bf16 or fp16 (got dtype code %d)", dtype);
  SEMBLO_REQUIRE(semblo::cap_in_range(softcap), "the soft cap must be 0 or lie in [2^-100, 2^100] (got %g)", (double)softcap);
  SEMBLO_REQUIRE(sm_scale > 0.f, "the score scale must be positive");
  if (tokens_q == 0 || (documents == 0 && !zero_tail)) return 0;
  SEMBLO_REQUIRE(q && out && status && cu_seqlens_q && cu_seqlens_k && (tokens_k == 0 || (k && v)), "null pointer");
  SEMBLO_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
                 "q and out must be 16-byte aligned");
  SEMBLO_REQUIRE(((q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) == 0,
                 "strides must be multiples of 8 elements");
  Args a{};
  a.q = q; a.q_token = q_token_stride; a.q_head = q_head_stride;
  a.out = out; a.lse = lse;
  a.cu_q = cu_seqlens_q; a.cu_k = cu_seqlens_k; a.prefix = prefix_lens; a.slopes = alibi_slopes;
  a.docs = documents; a.group = group; a.num_q_heads = num_q_heads;
  a.queries_per_tile = 128 / group;
  a.num_kv_heads = num_kv_heads;
  a.tokens_q = tokens_q; a.tokens_k = tokens_k;
  a.causal = causal; a.window = window; a.zero_tail = zero_tail;
  a.score_scale = softcap > 0.f ? sm_scale / softcap * TANH_ARG : sm_scale * LOG2EF;
  a.cap_log2 = softcap * LOG2EF;
  a.status = status;
  const Split split = split_for(tokens_q, tokens_k, group, num_kv_heads, head_dim, documents, causal, window, prefix_lens != nullptr);
  a.splits = split.pieces;
  a.piece_keys = split.keys;
  a.partial = (float*)workspace;
  const int64_t bytes = split_bytes(tokens_q, group, num_kv_heads, head_dim, documents, a.splits);
  SEMBLO_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "the workspace must be 16-byte aligned");
  if (bytes > workspace_bytes || (bytes && !workspace))
    return semblo::fail(semblo::SEMBLO_ENOSPC, "workspace of %lld bytes needed, %lld given", (long long)bytes,
                        (long long)workspace_bytes);
  // no keys at all: the maps are not read, but have to describe something
  CUtensorMap mk, mv;
  const uint64_t dims[3] = {(uint64_t)head_dim, (uint64_t)num_kv_heads, (uint64_t)std::max<int64_t>(tokens_k, 1)};
  const uint64_t sk[2] = {(uint64_t)k_head_stride * 2, (uint64_t)k_token_stride * 2};
  const uint64_t sv[2] = {(uint64_t)v_head_stride * 2, (uint64_t)v_token_stride * 2};
  const int bn = head_dim <= 128 ? NARROW_BN : BN;
  const uint32_t box[3] = {64, 1, (uint32_t)bn};
  const uint64_t dense_stride[2] = {(uint64_t)head_dim * 2, (uint64_t)head_dim * num_kv_heads * 2};
  int rc = semblo::make_tensor_map_bf16(&mk, tokens_k ? k : q, 3, dims, tokens_k ? sk : dense_stride, box);
  if (rc) return rc;
  rc = semblo::make_tensor_map_bf16(&mv, tokens_k ? v : q, 3, dims, tokens_k ? sv : dense_stride, box);
  if (rc) return rc;
  CUtensorMap mq;
  if (head_dim <= 128) {
    const uint64_t qd[3] = {(uint64_t)head_dim, (uint64_t)num_q_heads, (uint64_t)tokens_q};
    const uint64_t qs[2] = {(uint64_t)q_head_stride * 2, (uint64_t)q_token_stride * 2};
    const uint32_t qbox[3] = {64, (uint32_t)group, (uint32_t)(128 / group)};
    rc = semblo::make_tensor_map_bf16(&mq, q, 3, qd, qs, qbox);
    if (rc) return rc;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const bool f16 = dtype == SEMBLO_F16;
  const int mode = alibi_slopes ? BIASED : softcap > 0.f ? (!f16 && a.cap_log2 <= BOUNDED_LOG2 ? BOUNDED : CAPPED) : LINEAR;
  if (head_dim <= 128) rc = dense::launch_narrow(mk, mv, mq, a, head_dim, f16, mode, st);
  else if (mode == LINEAR) rc = f16 ? launch<256, true, LINEAR>(mk, mv, a, st) : launch<256, false, LINEAR>(mk, mv, a, st);
  else if (mode == BOUNDED) rc = launch<256, false, BOUNDED>(mk, mv, a, st);
  else if (mode == CAPPED) rc = f16 ? launch<256, true, CAPPED>(mk, mv, a, st) : launch<256, false, CAPPED>(mk, mv, a, st);
  else rc = f16 ? launch<256, true, BIASED>(mk, mv, a, st) : launch<256, false, BIASED>(mk, mv, a, st);
  if (rc || a.splits == 1) return rc;
  if (head_dim == 64) return f16 ? join_pieces<64, NARROW_BN, true>(a, st) : join_pieces<64, NARROW_BN, false>(a, st);
  if (head_dim == 128) return f16 ? join_pieces<128, NARROW_BN, true>(a, st) : join_pieces<128, NARROW_BN, false>(a, st);
  return f16 ? join_pieces<256, BN, true>(a, st) : join_pieces<256, BN, false>(a, st);
}
