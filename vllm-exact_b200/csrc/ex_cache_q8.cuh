// The 8-bit paged cache: rows of keys and values quantised as they are written, and read back.
//
// One row is the D numbers of one token and KV head. Its scale is s = max|x| / Q in float32 (Q = 127 for int8, 448 for
// e4m3, the largest code) and its codes are c = x / s rounded to nearest even, so x is stood for by c * s. The division
// is the correctly rounded one in both places: codes and scales are then the same numbers on any device that rounds
// as IEEE 754 says. s = 0 (a row of zeros, or of numbers so small that max|x| / Q rounds to 0) gives codes 0. A row
// that holds an infinity or a NaN gets codes 0 and that scale, so it reads back as NaN and not as wrong numbers.
// Codes: (block, place in page, KV head, D), any strides that keep 16-byte rows. Scales: (block, KV head, place), so
// that the scales of consecutive tokens of a head lie side by side for the attention kernels.
#pragma once
#include "ex_common.cuh"

#include <cuda_fp8.h>

namespace ex {

enum { CODE_NONE = -1, CODE_INT8 = 0, CODE_E4M3 = 1 };
template <int CODE>
__host__ __device__ constexpr float code_max() { return CODE == CODE_INT8 ? 127.0f : 448.0f; }

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t v, float& a, float& b) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value) {
    a = __uint_as_float(v << 16);
    b = __uint_as_float(v & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
    a = f.x;
    b = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// four codes of y (already divided by the scale) in a word, and the numbers that they are
template <int CODE>
__device__ __forceinline__ uint32_t encode4(const float (&y)[4], float (&back)[4]) {
  uint32_t w = 0;
  if constexpr (CODE == CODE_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = fminf(fmaxf(y[i], -127.0f), 127.0f);
      // 1.5 * 2^23 leaves no bits behind the point: the sum is c rounded to nearest even, its low byte the code
      const uint32_t u = __float_as_uint(c + 12582912.0f);
      w |= (u & 0xffu) << (8 * i);
      back[i] = __uint_as_float(u) - 12582912.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const __nv_fp8x2_storage_t p = __nv_cvt_float2_to_fp8x2(make_float2(y[i], y[i + 1]), __NV_SATFINITE, __NV_E4M3);
      w |= (uint32_t)p << (8 * i);
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(p, __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      back[i] = f.x;
      back[i + 1] = f.y;
    }
  }
  return w;
}

template <int CODE>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
  if constexpr (CODE == CODE_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int)(int8_t)(w >> (8 * i));
  } else {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (8 * i)), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      x[i] = f.x;
      x[i + 1] = f.y;
    }
  }
}

struct CacheView {      // strides in elements
  uint8_t* key;
  uint8_t* value;
  int64_t s_block, s_page, s_head;  // of both code arrays
  float* key_scale;
  float* value_scale;
  int64_t ss_block, ss_head;        // of both scale arrays (places are contiguous)
  int64_t blocks;
  int page;
};

constexpr int CQ_THREADS = 256;

// One row per D/8 lanes, 8 numbers (16 bytes) a lane. Rows are numbered (token, key or value, head).
template <int D, int CODE, typename T>
__global__ void __launch_bounds__(CQ_THREADS)
    k_cache_write(const T* __restrict__ key, const T* __restrict__ value, int64_t sk_t, int64_t sk_h, int64_t sv_t,
                  int64_t sv_h, CacheView c, const int64_t* __restrict__ slots, int64_t tokens, int KV,
                  T* __restrict__ key_out, T* __restrict__ value_out, int64_t sko_t, int64_t sko_h, int64_t svo_t,
                  int64_t svo_h) {
  constexpr int LANES = D / 8;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = ((int64_t)blockIdx.x * CQ_THREADS + threadIdx.x) / LANES;
  const int lane = threadIdx.x % LANES;
  const bool real = row < tokens * 2 * KV;  // every lane stays for the shuffles
  const int64_t t = real ? row / (2 * KV) : 0;
  const int r = real ? (int)(row - t * 2 * KV) : 0;
  const bool is_v = r >= KV;
  const int h = is_v ? r - KV : r;
  uint4 v = make_uint4(0, 0, 0, 0);
  int64_t slot = -1;
  if (real) {
    const T* src = is_v ? value + t * sv_t + h * sv_h : key + t * sk_t + h * sk_h;
    v = *reinterpret_cast<const uint4*>(src + lane * 8);
    slot = slots[t];
  }
  float x[8];
  unpack2<T>(v.x, x[0], x[1]);
  unpack2<T>(v.y, x[2], x[3]);
  unpack2<T>(v.z, x[4], x[5]);
  unpack2<T>(v.w, x[6], x[7]);
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max_nan(a, fabsf(x[i]));
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  const float s = __fdiv_rn(a, code_max<CODE>());
  const bool some = s > 0.0f && s < INFINITY;
  float y[2][4], b[2][4];
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i / 4][i % 4] = some ? __fdiv_rn(x[i], s) : 0.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = encode4<CODE>(y[i], b[i]);
  if (!real) return;
  if (slot >= 0 && slot < c.blocks * c.page) {  // -1: a padded token, not written
    const int64_t blk = slot / c.page;
    const int place = (int)(slot - blk * c.page);
    uint8_t* dst = (is_v ? c.value : c.key) + blk * c.s_block + place * c.s_page + h * c.s_head;
    *reinterpret_cast<uint2*>(dst + lane * 8) = make_uint2(w[0], w[1]);
    if (lane == 0) (is_v ? c.value_scale : c.key_scale)[blk * c.ss_block + h * c.ss_head + place] = s;
  }
  if (key_out != nullptr) {
    T* dst = is_v ? value_out + t * svo_t + h * svo_h : key_out + t * sko_t + h * sko_h;
    uint4 o;
    o.x = pack2<T>(b[0][0] * s, b[0][1] * s);
    o.y = pack2<T>(b[0][2] * s, b[0][3] * s);
    o.z = pack2<T>(b[1][0] * s, b[1][1] * s);
    o.w = pack2<T>(b[1][2] * s, b[1][3] * s);
    *reinterpret_cast<uint4*>(dst + lane * 8) = o;
  }
}

// The sequence that packed row r belongs to: the number of ends cu[1..n] that are <= r (n if r is behind the last).
// A search with 32 probes a step; every lane of the warp calls it and gets the answer.
__device__ __forceinline__ int find_sequence(const int32_t* __restrict__ cu, int n, int64_t r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, len = n;  // the answer is in [lo, lo + len]
  while (len > 0) {
    const int step = (len + 31) / 32;
    const int at = lo + min((lane + 1) * step, len);  // cu index of this lane's probe
    const unsigned below = __ballot_sync(0xffffffffu, (int64_t)cu[at] <= r);
    const int k = __popc(below);  // the ends are in order: probes 0..k-1 are <= r
    const int passed = min(k * step, len);
    if (k == 32 || passed == len) return lo + len;
    lo += passed;
    len = min(step, len - passed) - 1;  // the end at lo + step is > r
  }
  return lo;
}

// One warp per packed token: its sequence, page and place are looked up once for all its rows; 16 codes a lane.
template <int D, int CODE, typename T>
__global__ void __launch_bounds__(CQ_THREADS)
    k_cache_read(CacheView c, const int32_t* __restrict__ bt, int64_t sbt, int width, const int32_t* __restrict__ cu,
                 int n, int64_t rows, int KV, T* __restrict__ key_out, T* __restrict__ value_out, int64_t sko_t,
                 int64_t sko_h, int64_t svo_t, int64_t svo_h) {
  constexpr int LANES = D / 16;
  constexpr int ROWS = 32 / LANES;  // rows a pass
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t = (int64_t)blockIdx.x * (CQ_THREADS / 32) + threadIdx.x / 32;
  if (t >= rows) return;
  const int b = find_sequence(cu, n, t);
  if (b >= n || t < cu[0]) return;  // rows outside the sequences are left as they were
  const int64_t i = t - cu[b];
  if (i / c.page >= width) return;
  const int64_t blk = bt[(int64_t)b * sbt + i / c.page];
  const int place = (int)(i % c.page);
  if (blk < 0 || blk >= c.blocks) return;
  const int lane = threadIdx.x % LANES, sub = (threadIdx.x & 31) / LANES;
#pragma unroll 4
  for (int r0 = 0; r0 < 2 * KV; r0 += ROWS) {
    const int r = r0 + sub;
    if (r >= 2 * KV) continue;
    const bool is_v = r >= KV;
    const int h = is_v ? r - KV : r;
    const uint8_t* src = (is_v ? c.value : c.key) + blk * c.s_block + place * c.s_page + h * c.s_head;
    const uint4 w = *reinterpret_cast<const uint4*>(src + lane * 16);
    const float s = (is_v ? c.value_scale : c.key_scale)[blk * c.ss_block + h * c.ss_head + place];
    T* dst = (is_v ? value_out + t * svo_t + h * svo_h : key_out + t * sko_t + h * sko_h) + lane * 16;
    float x[4][4];
    decode4<CODE>(w.x, x[0]);
    decode4<CODE>(w.y, x[1]);
    decode4<CODE>(w.z, x[2]);
    decode4<CODE>(w.w, x[3]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint4 o;
      o.x = pack2<T>(x[2 * j][0] * s, x[2 * j][1] * s);
      o.y = pack2<T>(x[2 * j][2] * s, x[2 * j][3] * s);
      o.z = pack2<T>(x[2 * j + 1][0] * s, x[2 * j + 1][1] * s);
      o.w = pack2<T>(x[2 * j + 1][2] * s, x[2 * j + 1][3] * s);
      reinterpret_cast<uint4*>(dst)[j] = o;
    }
  }
}

}  // namespace ex
