// Rotary positions: q_post, k_post from q_pre, k_pre (the layer keeps both: routing reads the
// vectors before the rotation, attention the ones after it).
//
//   angle(t, i) = position_t * f_i,  c = a cos(angle), s = a sin(angle)   (a: the attention scale)
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s                                   (inverse: s -> -s)
//
// with (x1, x2) = (x_i, x_{i + R/2}) in the half layout and (x_2i, x_2i+1) in the interleaved one;
// dimensions from R on are copied.  Frequencies are doubles and the angle is reduced to a fraction of a
// turn in double: a float product is off by half a radian at position 1e6 * f = 1, which no later step
// can repair.  sincospi of the reduced fraction is then as accurate as a float can be.
//
// Bound: HBM, one read and one write of every element.  A cos/sin costs ~40 instructions against the 8
// bytes that a bf16 pair moves, so a thread keeps the cos/sin of its 8 (or 4) pairs in registers and takes
// them through all heads of its head group: 4 loads of 2 x 16 bytes are requested before the first is used.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../../include/semblo_b200.h"
#include "host_common.h"

using semblo::ceil_div;

namespace {

struct RotaryArgs {
  const void* in[2];            // q, k
  void* out[2];
  int64_t in_token[2], in_head[2], out_token[2], out_head[2];   // strides in elements
  int heads0, heads;            // query heads, query + key heads
  int heads_per_group;
  int64_t tokens;
  int head_dim, rotary_dim;
  int cols;                     // threads per (token, head): rotating columns, then copying ones
  int rot_cols;
  const void* positions;
  int pos64;
  const double* inv_freq;
  float scale;                  // on cos and sin
  float sin_sign;
};

template <typename T> struct Conv;
template <> struct Conv<__nv_bfloat16> {
  static __device__ __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Conv<__half> {
  static __device__ __forceinline__ float to(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
};
template <> struct Conv<float> {
  static __device__ __forceinline__ float to(float x) { return x; }
  static __device__ __forceinline__ float from(float x) { return x; }
};

// N elements moved as the widest aligned words (N * sizeof(T) is a multiple of 8, or N is 1).
template <typename T, int N>
struct alignas(N * sizeof(T) >= 16 ? 16 : N * sizeof(T)) Pack { T v[N]; };

// NP: pairs per thread and head.  A rotating column c covers the pairs [NP c, NP (c + 1)): two packs of NP
// elements, R/2 apart (half) or adjacent (interleaved).  A copying column covers 2 NP elements from R on
// (NP = 1: two single elements, the second may lie past the head).
template <typename T, int NP, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  constexpr int AHEAD = NP * (int)sizeof(T) > 16 ? 2 : 4;      // heads whose loads are in flight
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t token = idx / a.cols;
  if (token >= a.tokens) return;
  const int col = (int)(idx - token * a.cols);
  const bool rotating = col < a.rot_cols;
  int e0, e1;                                                  // element offsets of the two packs
  if (rotating) {
    e0 = INTERLEAVED ? 2 * NP * col : NP * col;
    e1 = INTERLEAVED ? e0 + NP : e0 + a.rotary_dim / 2;
  } else {
    e0 = a.rotary_dim + 2 * NP * (col - a.rot_cols);
    e1 = e0 + NP;
  }
  const bool second = e1 + NP <= a.head_dim;                   // false only for the odd end of a copied tail
  float c[NP], s[NP];
  if (rotating) {
    const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[token]
                               : (double)static_cast<const int32_t*>(a.positions)[token];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      double turns = pos * a.inv_freq[NP * col + i] * 0.15915494309189535;      // 1 / (2 pi)
      turns -= rint(turns);
      float sn, cs;
      sincospif((float)(2.0 * turns), &sn, &cs);
      c[i] = cs * a.scale;
      s[i] = sn * a.scale * a.sin_sign;
    }
  }
  const int h_begin = blockIdx.y * a.heads_per_group;
  const int h_end = min(a.heads, h_begin + a.heads_per_group);
  for (int h0 = h_begin; h0 < h_end; h0 += AHEAD) {
    Pack<T, NP> x0[AHEAD], x1[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int h = h0 + u;
      if (h < h_end) {
        const int which = h >= a.heads0;
        const T* src = static_cast<const T*>(a.in[which]) + token * a.in_token[which] +
                       (int64_t)(which ? h - a.heads0 : h) * a.in_head[which];
        x0[u] = *reinterpret_cast<const Pack<T, NP>*>(src + e0);
        if (second) x1[u] = *reinterpret_cast<const Pack<T, NP>*>(src + e1);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int h = h0 + u;
      if (h >= h_end) break;
      if (rotating) {
        if constexpr (INTERLEAVED && NP > 1) {
          // pairs sit next to each other inside the packs
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            T* p = i < NP / 2 ? &x0[u].v[2 * i] : &x1[u].v[2 * i - NP];
            const float p1 = Conv<T>::to(p[0]), p2 = Conv<T>::to(p[1]);
            p[0] = Conv<T>::from(p1 * c[i] - p2 * s[i]);
            p[1] = Conv<T>::from(p2 * c[i] + p1 * s[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const float p1 = Conv<T>::to(x0[u].v[i]), p2 = Conv<T>::to(x1[u].v[i]);
            x0[u].v[i] = Conv<T>::from(p1 * c[i] - p2 * s[i]);
            x1[u].v[i] = Conv<T>::from(p2 * c[i] + p1 * s[i]);
          }
        }
      }
      const int which = h >= a.heads0;
      T* dst = static_cast<T*>(a.out[which]) + token * a.out_token[which] +
               (int64_t)(which ? h - a.heads0 : h) * a.out_head[which];
      *reinterpret_cast<Pack<T, NP>*>(dst + e0) = x0[u];
      if (second) *reinterpret_cast<Pack<T, NP>*>(dst + e1) = x1[u];
    }
  }
}

template <typename T, int NP>
int launch(RotaryArgs& a, bool interleaved, cudaStream_t st) {
  a.rot_cols = a.rotary_dim / (2 * NP);
  a.cols = a.rot_cols + (int)ceil_div(a.head_dim - a.rotary_dim, 2 * NP);
  // all heads in one thread once there are enough (token, column) threads to fill the part, else the heads
  // are spread over threads, which recompute the cos/sin: 1 token of 20 heads takes one wave of one head each
  const int64_t threads = a.tokens * a.cols;
  const int64_t want = (int64_t)semblo::sm_count() * 2048;
  const int64_t groups = std::min<int64_t>(a.heads, std::max<int64_t>(1, want / std::max<int64_t>(threads, 1)));
  a.heads_per_group = (int)ceil_div(a.heads, groups);
  dim3 grid((unsigned)ceil_div(threads, 256), (unsigned)ceil_div(a.heads, a.heads_per_group));
  if (interleaved) rotary_kernel<T, NP, true><<<grid, 256, 0, st>>>(a);
  else rotary_kernel<T, NP, false><<<grid, 256, 0, st>>>(a);
  SEMBLO_LAUNCH_CHECK();
  return 0;
}

// The widest pack that every row start and every pack offset allows.
template <typename T>
int dispatch(RotaryArgs& a, bool interleaved, cudaStream_t st) {
  uint64_t bits = 0;                                 // of every byte offset that a row can start at
  for (int w = 0; w < 2; ++w) {
    if (!a.in[w]) continue;
    bits |= (uint64_t)(uintptr_t)a.in[w] | (uint64_t)(uintptr_t)a.out[w];
    bits |= (uint64_t)(a.in_token[w] | a.in_head[w] | a.out_token[w] | a.out_head[w]) * sizeof(T);
  }
  auto fits = [&](int np) {
    const uint64_t align = std::min<uint64_t>(16, np * sizeof(T));
    return a.rotary_dim % (2 * np) == 0 && a.head_dim % (2 * np) == 0 && bits % align == 0;
  };
  if (fits(8)) return launch<T, 8>(a, interleaved, st);
  if (fits(4)) return launch<T, 4>(a, interleaved, st);
  return launch<T, 1>(a, interleaved, st);
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
  SEMBLO_REQUIRE((k == nullptr) == (k_out == nullptr), "k and k_out come together");
  if (tokens == 0) return 0;
  SEMBLO_REQUIRE(q != nullptr && q_out != nullptr && positions != nullptr, "q, q_out and positions are required");
  SEMBLO_REQUIRE(rotary_dim == 0 || inv_freq != nullptr, "inv_freq is required");
  SEMBLO_REQUIRE(tokens <= (int64_t)1 << 31, "too many tokens");
  RotaryArgs a{};
  a.in[0] = q; a.out[0] = q_out; a.in[1] = k; a.out[1] = k_out;
  a.in_token[0] = q_token_stride; a.in_head[0] = q_head_stride;
  a.out_token[0] = qo_token_stride; a.out_head[0] = qo_head_stride;
  a.in_token[1] = k_token_stride; a.in_head[1] = k_head_stride;
  a.out_token[1] = ko_token_stride; a.out_head[1] = ko_head_stride;
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
