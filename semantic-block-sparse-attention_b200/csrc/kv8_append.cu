// Appending to the 8-bit paged K/V cache: e4m3 codes [2, blocks, Hkv, block, D] with one fp32 scale for
// each block of tokens and KV head, [2, blocks, Hkv].
//
//   need   = the power of two 2^e with max |x| / 2^e in (224, 448] over the block's new finite values,
//            e clamped to [-100, 120]
//   scale' = need for a block that starts with this call, max(scale, need) for one that is continued
//   code   = e4m3(x / scale') (round to nearest even, saturating);  rows already there: e4m3(code scale / scale')
//
// e4m3 keeps three mantissa bits at every magnitude, so a power of two costs no accuracy against max / 448,
// a new maximum inside the same octave changes nothing, and the codes of rows already written move by whole
// exponents: they are rounded a second time only where they fall below 2^-6.  One thread block owns one
// (cache block, head, K or V): no atomics, the same bytes on every run.
//
// Bound: HBM, 2 bytes read and 1 written per value.  The maximum is needed before the first code, so a
// thread holds its share of the block in registers between the two steps and the input is read once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "../../include/semblo_b200.h"
#include "host_common.h"
#include "sm100.cuh"

using semblo::ceil_div;

namespace {

struct AppendArgs {
  const void* src[2];                   // k, v [T, Hkv, D]
  int64_t src_token[2], src_head[2];    // strides in elements
  int64_t tokens;
  uint8_t* data;
  float* scales;
  int64_t cache_blocks;
  int block_log2;
  int num_kv_heads, head_dim, col_log2; // 16-value columns of a row, a power of two
  const int32_t* table;
  int64_t table_stride;
  int table_len;
  const int32_t* cu;                    // [batch + 1]
  const int32_t* start;                 // [batch]
  int batch;
  int* status;
};

constexpr float E4M3_MAX_MANTISSA = 1.75f;           // 448 = 1.75 * 2^8

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

template <typename T2>
__device__ __forceinline__ float2 widen(uint32_t w) {
  if constexpr (sizeof(T2) == 4 && std::is_same<T2, __nv_bfloat162>::value)
    return make_float2(__int_as_float(w << 16), __int_as_float(w & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ uint32_t code4(float2 a, float2 b) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
  const __half2_raw r0 = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
  const __half2_raw r1 = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
  float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&r0));
  float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&r1));
  f0.x *= ratio; f0.y *= ratio; f1.x *= ratio; f1.y *= ratio;
  return code4(f0, f1);
}

// Maximum over the thread block of a non-negative value (compared as bits).
__device__ __forceinline__ float block_max(float v, uint32_t* slots) {
  const uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = b;
  __syncthreads();
  uint32_t m = 0;
  for (int i = 0; i < (int)blockDim.x >> 5; ++i) m = max(m, slots[i]);
  __syncthreads();
  return __uint_as_float(m);
}

// T2: the packed pair type of the input.  NL: 16-value pieces of the cache block per thread.
template <typename T2, int NL>
__global__ void __launch_bounds__(512) kv8_append_kernel(const AppendArgs a) {
  __shared__ uint32_t slots[16];
  const int lane = threadIdx.x & 31;
  const int block = 1 << a.block_log2;
  const int piece0 = threadIdx.x, piece_step = blockDim.x;
  // ---- which request and cache block: every warp walks the requests, 32 at a time
  int want = (int)blockIdx.x, seq = -1, n = 0, start = 0, nth = 0;
  int64_t row0 = 0;
  for (int b0 = 0; b0 < a.batch && seq < 0; b0 += 32) {
    const int b = b0 + lane;
    int bn = 0, bs = 0, blocks = 0;
    int64_t c0 = 0;
    if (b < a.batch) {
      c0 = a.cu[b];
      const int64_t c1 = min((int64_t)a.cu[b + 1], a.tokens);
      bs = a.start[b];
      bn = c0 < 0 ? 0 : (int)max((int64_t)0, c1 - c0);
      if (bn > 0 && bs < 0) {
        if (blockIdx.x == 0 && threadIdx.x == lane) atomicCAS(a.status, 0, sm100::STATUS_OVERFLOW);
        bn = 0;
      }
      if (bn > 0) blocks = (int)(((int64_t)bs + bn - 1) >> a.block_log2) - (bs >> a.block_log2) + 1;
    }
    int upto = blocks;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    const int total = __shfl_sync(0xffffffffu, upto, 31);
    if (want < total) {
      const uint32_t above = __ballot_sync(0xffffffffu, upto > want);
      const int at = __ffs(above) - 1;
      seq = b0 + at;
      nth = want - __shfl_sync(0xffffffffu, upto - blocks, at);
      n = __shfl_sync(0xffffffffu, bn, at);
      start = __shfl_sync(0xffffffffu, bs, at);
      row0 = __shfl_sync(0xffffffffu, c0, at);
    } else {
      want -= total;
    }
  }
  if (seq < 0) return;                                // the grid covers the largest possible number of blocks
  const int slot = (start >> a.block_log2) + nth;
  const int off = nth == 0 ? start & (block - 1) : 0;
  const int64_t pos0 = ((int64_t)slot << a.block_log2) + off;
  const int m = (int)min((int64_t)(block - off), (int64_t)start + n - pos0);
  const int64_t page = slot < a.table_len ? a.table[seq * a.table_stride + slot] : -1;
  const int h = blockIdx.y, part = blockIdx.z;
  const uint16_t* src = static_cast<const uint16_t*>(a.src[part]) + (row0 + pos0 - start) * a.src_token[part] +
                        (int64_t)h * a.src_head[part];
  // ---- the new rows into registers, their largest magnitude
  const int pieces = m << a.col_log2, colmask = (1 << a.col_log2) - 1;
  uint4 x[NL][2];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int p = i * piece_step + piece0;
    x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
    if (p < pieces) {
      const uint4* s = reinterpret_cast<const uint4*>(src + (int64_t)(p >> a.col_log2) * a.src_token[part] +
                                                      (p & colmask) * 16);
      x[i][0] = __ldg(s);
      x[i][1] = __ldg(s + 1);
    }
  }
  if (page < 0 || page >= a.cache_blocks) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, sm100::STATUS_OVERFLOW);
    return;
  }
  const int64_t cell = ((int64_t)part * a.cache_blocks + page) * a.num_kv_heads + h;
  uint8_t* dst = a.data + (cell << a.block_log2) * a.head_dim;
  const float before = off ? a.scales[cell] : 0.f;
  T2 top2;
  *reinterpret_cast<uint32_t*>(&top2) = 0u;
#pragma unroll
  for (int i = 0; i < NL; ++i)
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const uint4& q = x[i][w >> 2];
      uint32_t u = (w & 3) == 0 ? q.x : (w & 3) == 1 ? q.y : (w & 3) == 2 ? q.z : q.w;
      top2 = __hmax2(top2, __habs2(*reinterpret_cast<T2*>(&u)));
    }
  const float2 t2 = widen<T2>(*reinterpret_cast<uint32_t*>(&top2));
  float amax = block_max(fmaxf(t2.x, t2.y), slots);
  if (!(amax <= 3.4e38f)) {
    // infinities saturate and NaN stay NaN, but neither sets the scale of the others
    float f = 0.f;
#pragma unroll
    for (int i = 0; i < NL; ++i)
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const uint4& q = x[i][w >> 2];
        const float2 v = widen<T2>((w & 3) == 0 ? q.x : (w & 3) == 1 ? q.y : (w & 3) == 2 ? q.z : q.w);
        if (fabsf(v.x) <= 3.4e38f) f = fmaxf(f, fabsf(v.x));
        if (fabsf(v.y) <= 3.4e38f) f = fmaxf(f, fabsf(v.y));
      }
    amax = block_max(f, slots);
  }
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8;                // 2^e * 256 <= max < 2^e * 512
  if (__uint_as_float((bits & 0x7fffffu) | 0x3f800000u) > E4M3_MAX_MANTISSA) ++e;
  e = min(max(e, -100), 120);
  float scale = pow2(e);
  if (off) {
    if (before >= scale) {
      scale = before;
    } else {
      // the rows of earlier calls follow the new scale
      const float ratio = before / scale;
      uint4* rows = reinterpret_cast<uint4*>(dst);
      const int held = off << a.col_log2;
      for (int p = piece0; p < held; p += 4 * piece_step) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (p + u * piece_step < held) v[u] = rows[p + u * piece_step];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (p + u * piece_step >= held) break;
          rows[p + u * piece_step] = make_uint4(recode4(v[u].x, ratio), recode4(v[u].y, ratio),
                                                recode4(v[u].z, ratio), recode4(v[u].w, ratio));
        }
      }
    }
  }
  if (threadIdx.x == 0) a.scales[cell] = scale;
  // ---- the codes
  const bool exact_inverse = (__float_as_uint(scale) & 0x7fffffu) == 0 && scale >= pow2(-126) && scale <= pow2(126);
  const float inv = exact_inverse ? __int_as_float((254 << 23) - __float_as_int(scale)) : 0.f;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int p = i * piece_step + piece0;
    if (p >= pieces) break;
    uint32_t out[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint4& q = x[i][w >> 1];
      float2 f0 = widen<T2>((w & 1) ? q.z : q.x), f1 = widen<T2>((w & 1) ? q.w : q.y);
      if (exact_inverse) {
        f0.x *= inv; f0.y *= inv; f1.x *= inv; f1.y *= inv;
      } else {                                        // a scale set by the caller: divided as written
        f0.x /= scale; f0.y /= scale; f1.x /= scale; f1.y /= scale;
      }
      out[w] = code4(f0, f1);
    }
    reinterpret_cast<uint4*>(dst)[(off << a.col_log2) + p] = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

template <typename T2>
int launch(AppendArgs& a, cudaStream_t st) {
  const int64_t block = (int64_t)1 << a.block_log2;
  const int64_t most = std::min<int64_t>(a.tokens, a.tokens / block + 2 * (int64_t)a.batch);
  const int64_t rows = std::min<int64_t>(block, a.tokens);        // new rows that a block can hold
  const int64_t pieces = rows << a.col_log2, held = block << a.col_log2;
  // 256 threads where the new rows fill them, or a continued block may have to be rounded again; 512 of 8
  // pieces for the largest blocks (128 KB of input)
  int64_t threads = std::min<int64_t>(256, std::max<int64_t>(64, held));
  if (pieces > 2048) threads = 512;
  const int64_t per_thread = ceil_div(pieces, threads);
  dim3 grid((unsigned)most, (unsigned)a.num_kv_heads, 2);
  if (per_thread <= 1) kv8_append_kernel<T2, 1><<<grid, (unsigned)threads, 0, st>>>(a);
  else if (per_thread <= 2) kv8_append_kernel<T2, 2><<<grid, (unsigned)threads, 0, st>>>(a);
  else if (per_thread <= 4) kv8_append_kernel<T2, 4><<<grid, (unsigned)threads, 0, st>>>(a);
  else kv8_append_kernel<T2, 8><<<grid, (unsigned)threads, 0, st>>>(a);
  SEMBLO_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" int semblo_kv8_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                 int64_t v_token_stride, int64_t v_head_stride, int64_t tokens, int dtype,
                                 void* cache, float* scales, int64_t cache_blocks, int block_size,
                                 int num_kv_heads, int head_dim, const int32_t* block_table,
                                 int64_t table_stride, int table_len, const int32_t* cu_seqlens,
                                 const int32_t* start_positions, int batch, int32_t* status, void* stream) {
  SEMBLO_REQUIRE(block_size >= 16 && block_size <= 256 && (block_size & (block_size - 1)) == 0,
                 "block_size must be 16, 32, 64, 128 or 256 (got %d)", block_size);
  SEMBLO_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "head_dim must be 64, 128 or 256 (got %d)",
                 head_dim);
  SEMBLO_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65535 && batch >= 0 && tokens >= 0, "bad head, batch or token count");
  if (tokens == 0 || batch == 0) return 0;
  SEMBLO_REQUIRE(k && v && cache && scales && block_table && cu_seqlens && start_positions && status,
                 "null pointer");
  SEMBLO_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                   reinterpret_cast<uintptr_t>(cache)) & 15) == 0, "k, v and the cache must be 16-byte aligned");
  SEMBLO_REQUIRE(((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) == 0,
                 "strides of k and v must be multiples of 8 elements");
  SEMBLO_REQUIRE(tokens < ((int64_t)1 << 31), "too many tokens");
  AppendArgs a{};
  a.src[0] = k; a.src[1] = v;
  a.src_token[0] = k_token_stride; a.src_head[0] = k_head_stride;
  a.src_token[1] = v_token_stride; a.src_head[1] = v_head_stride;
  a.tokens = tokens;
  a.data = (uint8_t*)cache;
  a.scales = scales;
  a.cache_blocks = cache_blocks;
  while ((1 << a.block_log2) < block_size) ++a.block_log2;
  while ((16 << a.col_log2) < head_dim) ++a.col_log2;
  a.num_kv_heads = num_kv_heads; a.head_dim = head_dim;
  a.table = block_table; a.table_stride = table_stride; a.table_len = table_len;
  a.cu = cu_seqlens; a.start = start_positions; a.batch = batch;
  a.status = status;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == SEMBLO_BF16) return launch<__nv_bfloat162>(a, st);
  if (dtype == SEMBLO_F16) return launch<__half2>(a, st);
  return semblo::fail(semblo::SEMBLO_EINVAL, "the cache is filled from bf16 or fp16 (got dtype code %d)", dtype);
}
