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
// thread holds its share of the block in registers between the two steps and the input is read once.  A few
// tokens of each request take a warp per head (kv8_token_kernel), more of them one thread block per cache block
// and head (kv8_append_kernel); a prompt's blocks are a stream (kv8_stream_kernel): while a group of threads works
// on one block from registers, the next one's rows travel into shared memory.  131072 tokens x 4 heads x 256:
// 126 us, 6.4 TB/s; 163 us block by block, and no less as a stream while the rare cases were unrolled in the loop.
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
  int num_kv_heads, head_dim, col_log2; // 8-value columns of a row, a power of two
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

// One cache block of one head that a call writes: rows [off, off + m) of it, from token row `row`.
struct Unit {
  bool have;
  int off, m;
  int64_t row;
  int64_t page;                          // -1: not in the pool or the table
};

// Cache block number `want` (0 ...) of the call, requests in order; warp-collective.  A caller that asks with
// rising numbers passes the same Cursor again.
struct Cursor { int request, before; };  // before: cache blocks of the requests in front of it
__device__ __forceinline__ Unit find_unit(const AppendArgs& a, int64_t want, Cursor& from) {
  const int lane = threadIdx.x & 31;
  const int block = 1 << a.block_log2;
  Unit u{};
  int64_t rest = want - from.before;
  for (int b0 = from.request; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    int bn = 0, bs = 0, blocks = 0;
    int64_t c0 = 0;
    if (b < a.batch) {
      c0 = a.cu[b];
      const int64_t c1 = min((int64_t)a.cu[b + 1], a.tokens);
      bs = a.start[b];
      bn = c0 < 0 ? 0 : (int)max((int64_t)0, c1 - c0);
      if (bn > 0 && bs < 0) {
        atomicCAS(a.status, 0, sm100::STATUS_OVERFLOW);
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
    if (rest < total) {
      const int at = __ffs(__ballot_sync(0xffffffffu, upto > rest)) - 1;
      const int ahead = __shfl_sync(0xffffffffu, upto - blocks, at);
      const int nth = (int)rest - ahead;
      const int n = __shfl_sync(0xffffffffu, bn, at), start = __shfl_sync(0xffffffffu, bs, at);
      const int64_t row0 = __shfl_sync(0xffffffffu, c0, at);
      const int slot = (start >> a.block_log2) + nth;
      u.have = true;
      u.off = nth == 0 ? start & (block - 1) : 0;
      const int64_t pos0 = ((int64_t)slot << a.block_log2) + u.off;
      u.m = (int)min((int64_t)(block - u.off), (int64_t)start + n - pos0);
      u.row = row0 + pos0 - start;
      u.page = slot < a.table_len ? a.table[(int64_t)(b0 + at) * a.table_stride + slot] : -1;
      if (u.page >= a.cache_blocks) u.page = -1;
      from.before = (int)(want - nth);
      from.request = b0 + at;
      return u;
    }
    rest -= total;
  }
  return u;                              // behind the last one
}

// The same for a call with many requests: all threads of the block, a run of requests each.
__device__ __forceinline__ Unit find_unit_block(const AppendArgs& a, int64_t want, uint32_t* slots) {
  __shared__ Unit found;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int per = (a.batch + blockDim.x - 1) / blockDim.x;
  const int b0 = min((int)threadIdx.x * per, a.batch), b1 = min(b0 + per, a.batch);
  struct Run { int64_t row; int n, start, blocks; };
  auto run_of = [&](int b) {
    Run r{a.cu[b], 0, a.start[b], 0};
    r.n = r.row < 0 ? 0 : (int)max((int64_t)0, min((int64_t)a.cu[b + 1], a.tokens) - r.row);
    if (r.n > 0 && r.start < 0) {
      atomicCAS(a.status, 0, sm100::STATUS_OVERFLOW);
      r.n = 0;
    }
    if (r.n > 0) r.blocks = (int)(((int64_t)r.start + r.n - 1) >> a.block_log2) - (r.start >> a.block_log2) + 1;
    return r;
  };
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += run_of(b).blocks;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += t;
  }
  if (lane == 31) slots[warp] = upto;
  if (threadIdx.x == 0) found.have = false;
  __syncthreads();
  int64_t rest = want - (upto - mine);
  for (int w = 0; w < warp; ++w) rest -= slots[w];
  if (rest >= 0 && rest < mine) {
    int b = b0;
    Run r = run_of(b);
    while (rest >= r.blocks) {
      rest -= r.blocks;
      r = run_of(++b);
    }
    const int block = 1 << a.block_log2, slot = (r.start >> a.block_log2) + (int)rest;
    Unit u;
    u.have = true;
    u.off = rest == 0 ? r.start & (block - 1) : 0;
    const int64_t pos0 = ((int64_t)slot << a.block_log2) + u.off;
    u.m = (int)min((int64_t)(block - u.off), (int64_t)r.start + r.n - pos0);
    u.row = r.row + pos0 - r.start;
    u.page = slot < a.table_len ? a.table[(int64_t)b * a.table_stride + slot] : -1;
    if (u.page >= a.cache_blocks) u.page = -1;
    found = u;
  }
  __syncthreads();
  return found;
}
constexpr int WARP_REQUESTS = 64;        // up to here every warp searches for itself

// 2^e * 256 <= largest < 2^e * 512 with 448 as the limit: the exponent of the scale a block needs.
__device__ __forceinline__ int exponent_for(float largest) {
  const uint32_t bits = __float_as_uint(largest);
  int e = (int)(bits >> 23) - 127 - 8;
  if (__uint_as_float((bits & 0x7fffffu) | 0x3f800000u) > E4M3_MAX_MANTISSA) ++e;
  return min(max(e, -100), 120);
}

template <typename T2, int NL>
__device__ __forceinline__ float largest_of(const uint4 (&x)[NL]) {
  T2 top2;
  *reinterpret_cast<uint32_t*>(&top2) = 0u;
#pragma unroll
  for (int i = 0; i < NL; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint4& q = x[i];
      uint32_t u = w == 0 ? q.x : w == 1 ? q.y : w == 2 ? q.z : q.w;
      top2 = __hmax2(top2, __habs2(*reinterpret_cast<T2*>(&u)));
    }
  const float2 t2 = widen<T2>(*reinterpret_cast<uint32_t*>(&top2));
  return fmaxf(t2.x, t2.y);
}

// The rare cases read the input again, in loops of their own and out of line: unrolled beside the common ones
// they filled the instruction cache (131072 tokens x 4 heads x 256: 166 us).
// The largest magnitude without infinities and NaN, which saturate and stay but do not set the scale of others.
template <typename T2>
__device__ __noinline__ float largest_finite_of(const uint16_t* src, int64_t row_stride, int pieces, int col_log2, int tid,
                                                int threads) {
  float f = 0.f;
#pragma unroll 1
  for (int p = tid; p < pieces; p += threads) {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(src + (p >> col_log2) * row_stride + (p & ((1 << col_log2) - 1)) * 8));
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    for (int i = 0; i < 4; ++i) {
      const float2 v = widen<T2>(w[i]);
      if (fabsf(v.x) <= 3.4e38f) f = fmaxf(f, fabsf(v.x));
      if (fabsf(v.y) <= 3.4e38f) f = fmaxf(f, fabsf(v.y));
    }
  }
  return f;
}

// Codes under a scale that is not a power of two (set by the caller): divided as written.
template <typename T2>
__device__ __noinline__ void divide_rows(const uint16_t* src, int64_t row_stride, int pieces, int col_log2, uint2* dst,
                                         float scale, int tid, int threads) {
#pragma unroll 1
  for (int p = tid; p < pieces; p += threads) {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(src + (p >> col_log2) * row_stride + (p & ((1 << col_log2) - 1)) * 8));
    const float2 a = widen<T2>(x.x), b = widen<T2>(x.y), c = widen<T2>(x.z), d = widen<T2>(x.w);
    dst[p] = make_uint2(code4(make_float2(a.x / scale, a.y / scale), make_float2(b.x / scale, b.y / scale)),
                        code4(make_float2(c.x / scale, c.y / scale), make_float2(d.x / scale, d.y / scale)));
  }
}

// The rows of earlier calls follow a new scale: `held` 16-byte pieces of them.
__device__ __forceinline__ void recode_rows(uint8_t* dst, int held, float ratio, int tid, int threads) {
  uint4* rows = reinterpret_cast<uint4*>(dst);
  for (int p = tid; p < held; p += 4 * threads) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p + i * threads < held) v[i] = rows[p + i * threads];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p + i * threads >= held) break;
      rows[p + i * threads] = make_uint4(recode4(v[i].x, ratio), recode4(v[i].y, ratio), recode4(v[i].z, ratio),
                                         recode4(v[i].w, ratio));
    }
  }
}

__device__ __forceinline__ bool power_of_two(float scale) {
  return (__float_as_uint(scale) & 0x7fffffu) == 0 && scale >= pow2(-126) && scale <= pow2(126);
}

// Scale, earlier rows and codes of one unit, by `threads` threads of which this is number `tid`; x are its
// pieces tid, tid + threads, ... of the new rows and `largest` their largest magnitude over the unit.
template <typename T2, int NL>
__device__ __forceinline__ void write_unit(const AppendArgs& a, const Unit& u, int64_t cell, float before, float largest,
                                           const uint4 (&x)[NL], const uint16_t* src, int64_t row_stride, int tid,
                                           int threads) {
  uint8_t* dst = a.data + (cell << a.block_log2) * a.head_dim;
  float scale = pow2(exponent_for(largest));
  if (u.off) {
    if (before >= scale) {
      scale = before;
    } else {
      recode_rows(dst, u.off << (a.col_log2 - 1), before / scale, tid, threads);
    }
  }
  if (tid == 0) a.scales[cell] = scale;
  const int pieces = u.m << a.col_log2;
  uint2* out = reinterpret_cast<uint2*>(dst) + (u.off << a.col_log2);
  if (!power_of_two(scale)) {
    divide_rows<T2>(src, row_stride, pieces, a.col_log2, out, scale, tid, threads);
    return;
  }
  const float inv = __int_as_float((254 << 23) - __float_as_int(scale));
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int p = i * threads + tid;
    if (p >= pieces) break;
    float2 f[4] = {widen<T2>(x[i].x), widen<T2>(x[i].y), widen<T2>(x[i].z), widen<T2>(x[i].w)};
#pragma unroll
    for (int w = 0; w < 4; ++w) { f[w].x *= inv; f[w].y *= inv; }
    out[p] = make_uint2(code4(f[0], f[1]), code4(f[2], f[3]));
  }
}

// A few tokens of each request: a thread block takes a cache block's K or V, a warp one head after the other.  Where
// a scale grew, all of the block's threads round that head's earlier rows again.
constexpr int TOKEN_THREADS = 256, TOKEN_HEADS = 256;
template <typename T2>
__global__ void __launch_bounds__(TOKEN_THREADS) kv8_token_kernel(const AppendArgs a) {
  __shared__ uint32_t slots[TOKEN_THREADS / 32];
  __shared__ float grown[TOKEN_HEADS];               // old / new scale of a head whose scale grew (it may round to 0), else KEPT
  constexpr float KEPT = 2.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = blockIdx.z;
  Cursor cursor{0, 0};
  const Unit u = a.batch <= WARP_REQUESTS ? find_unit(a, blockIdx.x, cursor) : find_unit_block(a, blockIdx.x, slots);
  if (!u.have) return;                                // the grid covers the largest possible number of blocks
  if (u.page < 0) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, sm100::STATUS_OVERFLOW);
    return;
  }
  const int pieces = u.m << a.col_log2, colmask = (1 << a.col_log2) - 1;
  const int64_t row_stride = a.src_token[part], cell0 = ((int64_t)part * a.cache_blocks + u.page) * a.num_kv_heads;
  for (int h = warp; h < a.num_kv_heads; h += TOKEN_THREADS / 32) {
    const uint16_t* src = static_cast<const uint16_t*>(a.src[part]) + u.row * row_stride + (int64_t)h * a.src_head[part];
    auto piece = [&](int p) {
      return __ldg(reinterpret_cast<const uint4*>(src + (p >> a.col_log2) * row_stride + (p & colmask) * 8));
    };
    const int64_t cell = cell0 + h;
    const float before = u.off ? a.scales[cell] : 0.f;
    float top = 0.f;
    for (int p = lane; p < pieces; p += 32) {
      const uint4 x[1] = {piece(p)};
      const float t = largest_of<T2, 1>(x);
      top = t <= 3.4e38f ? fmaxf(top, t) : INFINITY;
      if (!(t <= 3.4e38f)) break;
    }
    float largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    if (!(largest <= 3.4e38f))
      largest = __uint_as_float(__reduce_max_sync(
          0xffffffffu, __float_as_uint(largest_finite_of<T2>(src, row_stride, pieces, a.col_log2, lane, 32))));
    float scale = pow2(exponent_for(largest)), ratio = KEPT;
    if (u.off) {
      if (before >= scale) scale = before;
      else ratio = before / scale;
    }
    if (lane == 0) {
      a.scales[cell] = scale;
      grown[h] = ratio;
    }
    uint2* out = reinterpret_cast<uint2*>(a.data + (cell << a.block_log2) * a.head_dim) + (u.off << a.col_log2);
    if (power_of_two(scale)) {
      const float inv = __int_as_float((254 << 23) - __float_as_int(scale));
      for (int p = lane; p < pieces; p += 32) {
        const uint4 x = piece(p);
        float2 f[4] = {widen<T2>(x.x), widen<T2>(x.y), widen<T2>(x.z), widen<T2>(x.w)};
#pragma unroll
        for (int w = 0; w < 4; ++w) { f[w].x *= inv; f[w].y *= inv; }
        out[p] = make_uint2(code4(f[0], f[1]), code4(f[2], f[3]));
      }
    } else {
      divide_rows<T2>(src, row_stride, pieces, a.col_log2, out, scale, lane, 32);
    }
  }
  if (u.off == 0) return;
  __syncthreads();
  for (int h = 0; h < a.num_kv_heads; ++h)
    if (grown[h] != KEPT)
      recode_rows(a.data + ((cell0 + h) << a.block_log2) * a.head_dim, u.off << (a.col_log2 - 1), grown[h], threadIdx.x,
                  TOKEN_THREADS);
}

// T2: the packed pair type of the input.  NL: 8-value pieces of the cache block per thread.
template <typename T2, int NL>
__global__ void __launch_bounds__(512) kv8_append_kernel(const AppendArgs a) {
  __shared__ uint32_t slots[16];
  const int h = blockIdx.y, part = blockIdx.z;
  Cursor cursor{0, 0};
  const Unit u = a.batch <= WARP_REQUESTS ? find_unit(a, blockIdx.x, cursor) : find_unit_block(a, blockIdx.x, slots);
  if (!u.have) return;                                // the grid covers the largest possible number of blocks
  const uint16_t* src = static_cast<const uint16_t*>(a.src[part]) + u.row * a.src_token[part] + (int64_t)h * a.src_head[part];
  // ---- the new rows into registers, their largest magnitude
  const int pieces = u.m << a.col_log2, colmask = (1 << a.col_log2) - 1;
  uint4 x[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int p = i * blockDim.x + threadIdx.x;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (p < pieces)
      x[i] = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)(p >> a.col_log2) * a.src_token[part] + (p & colmask) * 8));
  }
  if (u.page < 0) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, sm100::STATUS_OVERFLOW);
    return;
  }
  const int64_t cell = ((int64_t)part * a.cache_blocks + u.page) * a.num_kv_heads + h;
  const float before = u.off ? a.scales[cell] : 0.f;
  float largest = block_max(largest_of<T2, NL>(x), slots);
  if (!(largest <= 3.4e38f))
    largest = block_max(largest_finite_of<T2>(src, a.src_token[part], pieces, a.col_log2, threadIdx.x, blockDim.x), slots);
  write_unit<T2, NL>(a, u, cell, before, largest, x, src, a.src_token[part], threadIdx.x, blockDim.x);
}

// A stream of cache blocks: GROUP threads take one (cache block, head, part) after the other, NL pieces a thread.
// A thread copies (cp.async) exactly the pieces that it reads back, so the shared memory needs no barrier.
constexpr int STREAM_THREADS = 512;
template <typename T2, int NL, int GROUP>
__global__ void __launch_bounds__(STREAM_THREADS, NL == 4 ? 2 : 1) kv8_stream_kernel(const AppendArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];    // [NL][STREAM_THREADS] 16-byte pieces, then the maxima
  constexpr int GROUPS = STREAM_THREADS / GROUP;
  uint32_t* slots = reinterpret_cast<uint32_t*>(smem + NL * STREAM_THREADS * 16);
  const int group = threadIdx.x / GROUP, tid = threadIdx.x % GROUP;
  const int colmask = (1 << a.col_log2) - 1;
  const uint32_t mine = sm100::smem_u32(smem) + threadIdx.x * 16;
  const int heads2 = 2 * a.num_kv_heads;
  const int64_t step = (int64_t)gridDim.x * GROUPS;

  auto group_max = [&](float v) {
    uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
    if constexpr (GROUP > 32) {
      if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = b;
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(GROUP) : "memory");
      b = 0;
#pragma unroll
      for (int i = 0; i < GROUP / 32; ++i) b = max(b, slots[group * (GROUP / 32) + i]);
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(GROUP) : "memory");
    }
    return __uint_as_float(b);
  };
  auto source = [&](const Unit& u, int h, int part) {
    return static_cast<const uint16_t*>(a.src[part]) + u.row * a.src_token[part] + (int64_t)h * a.src_head[part];
  };
  auto request = [&](const Unit& u, int h, int part) {        // the new rows of a unit on their way
    if (u.have && u.page >= 0) {
      const uint16_t* src = source(u, h, part);
      const int pieces = u.m << a.col_log2;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int p = i * GROUP + tid;
        const bool in = p < pieces;
        const uint16_t* s = in ? src + (int64_t)(p >> a.col_log2) * a.src_token[part] + (p & colmask) * 8 : src;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(mine + i * STREAM_THREADS * 16), "l"(s),
                     "r"(in ? 16 : 0)
                     : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  Cursor cursor{0, 0};
  int64_t n = (int64_t)blockIdx.x * GROUPS + group;
  auto look = [&](int64_t i) { return find_unit(a, i / heads2, cursor); };
  Unit next = look(n);
  int h = (int)(n % heads2) >> 1, part = (int)(n & 1);
  request(next, h, part);
  while (next.have) {
    const Unit u = next;
    const uint16_t* src = source(u, h, part);
    const int64_t row_stride = a.src_token[part];
    const int64_t cell = ((int64_t)part * a.cache_blocks + max(u.page, (int64_t)0)) * a.num_kv_heads + h;
    const float before = u.off && u.page >= 0 ? a.scales[cell] : 0.f;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    uint4 x[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) x[i] = *reinterpret_cast<const uint4*>(smem + i * STREAM_THREADS * 16 + threadIdx.x * 16);
    const float own = largest_of<T2, NL>(x);          // every piece is in its register before its place is reused
    n += step;
    next = look(n);
    h = (int)(n % heads2) >> 1;
    part = (int)(n & 1);
    request(next, h, part);
    float largest = group_max(own);
    if (u.page < 0) {
      if (tid == 0) atomicCAS(a.status, 0, sm100::STATUS_OVERFLOW);
      continue;
    }
    if (!(largest <= 3.4e38f))
      largest = group_max(largest_finite_of<T2>(src, row_stride, u.m << a.col_log2, a.col_log2, tid, GROUP));
    write_unit<T2, NL>(a, u, cell, before, largest, x, src, row_stride, tid, GROUP);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename T2, int NL, int GROUP>
int launch_stream(const AppendArgs& a, int64_t units, cudaStream_t st) {
  auto kern = kv8_stream_kernel<T2, NL, GROUP>;
  const int smem = NL * STREAM_THREADS * 16 + STREAM_THREADS / 32 * 4;
  SEMBLO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int64_t blocks = std::min<int64_t>(ceil_div(units, STREAM_THREADS / GROUP), (int64_t)semblo::sm_count() * (NL == 4 ? 2 : 1));
  kern<<<(unsigned)blocks, STREAM_THREADS, smem, st>>>(a);
  SEMBLO_LAUNCH_CHECK();
  return 0;
}

template <typename T2>
int launch(AppendArgs& a, cudaStream_t st) {
  const int64_t block = (int64_t)1 << a.block_log2;
  const int64_t most = std::min<int64_t>(a.tokens, a.tokens / block + 2 * (int64_t)a.batch);
  const int64_t rows = std::min<int64_t>(block, a.tokens);        // new rows that a block can hold
  const int64_t pieces = rows << a.col_log2, held = block << a.col_log2;
  // a warp per head while a head's new rows are a few (64 requests of one token: 128 blocks of 256 threads instead of
  // 1024, 5.8 -> 3.7 us; 2000 of them: 473 -> 45 us)
  if (a.tokens <= 4 * (int64_t)a.batch && a.num_kv_heads <= TOKEN_HEADS) {
    kv8_token_kernel<T2><<<dim3((unsigned)most, 1, 2), TOKEN_THREADS, 0, st>>>(a);
    SEMBLO_LAUNCH_CHECK();
    return 0;
  }
  // enough new rows for every group of threads to overlap one cache block with the next: a stream
  const int64_t units = ceil_div(a.tokens, block) * a.num_kv_heads * 2;
  const int64_t per_thread = held <= 128 ? 4 : held <= 256 ? 8 : 16;
  const int64_t groups = (int64_t)semblo::sm_count() * STREAM_THREADS * (per_thread == 4 ? 2 : 1) / std::max<int64_t>(32, held / 16);
  if (units >= 2 * groups) {
    if (held <= 128) return launch_stream<T2, 4, 32>(a, units, st);
    if (held <= 256) return launch_stream<T2, 8, 32>(a, units, st);
    if (held <= 512) return launch_stream<T2, 16, 32>(a, units, st);
    if (held <= 1024) return launch_stream<T2, 16, 64>(a, units, st);
    if (held <= 2048) return launch_stream<T2, 16, 128>(a, units, st);
    if (held <= 4096) return launch_stream<T2, 16, 256>(a, units, st);
    return launch_stream<T2, 16, 512>(a, units, st);
  }
  // 256 threads where the new rows fill them, or a continued block may have to be rounded again; 512 for the
  // largest blocks (128 KB of input)
  int64_t threads = std::min<int64_t>(256, std::max<int64_t>(64, held / 2));
  if (pieces > 4096) threads = 512;
  const int64_t nl = ceil_div(pieces, threads);
  dim3 grid((unsigned)most, (unsigned)a.num_kv_heads, 2);
  if (nl <= 1) kv8_append_kernel<T2, 1><<<grid, (unsigned)threads, 0, st>>>(a);
  else if (nl <= 2) kv8_append_kernel<T2, 2><<<grid, (unsigned)threads, 0, st>>>(a);
  else if (nl <= 4) kv8_append_kernel<T2, 4><<<grid, (unsigned)threads, 0, st>>>(a);
  else if (nl <= 8) kv8_append_kernel<T2, 8><<<grid, (unsigned)threads, 0, st>>>(a);
  else kv8_append_kernel<T2, 16><<<grid, (unsigned)threads, 0, st>>>(a);
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
  // blocks write while others still read: the rows lie apart from the codes and the scales
  const uintptr_t codes0 = reinterpret_cast<uintptr_t>(cache), scales0 = reinterpret_cast<uintptr_t>(scales);
  const int64_t cells = 2 * cache_blocks * num_kv_heads;
  auto apart = [&](const void* rows, int64_t token_stride, int64_t head_stride) {
    const uintptr_t r0 = reinterpret_cast<uintptr_t>(rows);
    const uintptr_t r1 = r0 + 2 * ((tokens - 1) * token_stride + (num_kv_heads - 1) * head_stride + head_dim);
    return (r1 <= codes0 || r0 >= codes0 + (uintptr_t)(cells * block_size * head_dim)) &&
           (r1 <= scales0 || r0 >= scales0 + (uintptr_t)(cells * 4));
  };
  SEMBLO_REQUIRE(apart(k, k_token_stride, k_head_stride) && apart(v, v_token_stride, v_head_stride),
                 "k and v must not overlap the cache or its scales");
  AppendArgs a{};
  a.src[0] = k; a.src[1] = v;
  a.src_token[0] = k_token_stride; a.src_head[0] = k_head_stride;
  a.src_token[1] = v_token_stride; a.src_head[1] = v_head_stride;
  a.tokens = tokens;
  a.data = (uint8_t*)cache;
  a.scales = scales;
  a.cache_blocks = cache_blocks;
  while ((1 << a.block_log2) < block_size) ++a.block_log2;
  while ((8 << a.col_log2) < head_dim) ++a.col_log2;
  a.num_kv_heads = num_kv_heads; a.head_dim = head_dim;
  a.table = block_table; a.table_stride = table_stride; a.table_len = table_len;
  a.cu = cu_seqlens; a.start = start_positions; a.batch = batch;
  a.status = status;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == SEMBLO_BF16) return launch<__nv_bfloat162>(a, st);
  if (dtype == SEMBLO_F16) return launch<__half2>(a, st);
  return semblo::fail(semblo::SEMBLO_EINVAL, "the cache is filled from bf16 or fp16 (got dtype code %d)", dtype);
}
