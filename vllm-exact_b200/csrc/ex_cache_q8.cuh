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

// four codes of y (already divided by the scale, |y| < Q + 1/2) in a word, and the numbers that they are
template <int CODE>
__device__ __forceinline__ uint32_t encode4(const float (&y)[4], float (&back)[4]) {
  uint32_t w = 0;
  if constexpr (CODE == CODE_INT8) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // 1.5 * 2^23 leaves no bits behind the point: the sum is y rounded to nearest even, its low byte the code
      u[i] = __float_as_uint(y[i] + 12582912.0f);
      back[i] = __uint_as_float(u[i]) - 12582912.0f;
    }
    w = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
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

// A warp takes PASSES (4) passes of one token's rows (keys' heads, then values'), D / 8 lanes a row and 16 bytes a lane: 4 loads in
// flight a lane, and the token's slot looked up once. What bounds it is instructions: the quotients are therefore not
// divisions but (Markstein, 1990) q = q0 + r (x - q0 s) with r = 1 / s and q0 = x r, all rounded to nearest, which is the
// correctly rounded x / s as long as x - q0 s is exact: its last bit is at least 2^-46 |q| s, so it is for s >= 2^-80 where
// |q| is not so small (under 2^-10) that its code is 0 anyway. Smaller scales take the division.
// 16000 tokens of 8 heads of 128 with values read back, bf16 to e4m3: 34 us, 4.8 TB/s (one pass a warp and a division per value: 56 us).
// PASSES = 1 where all warps run at once even so: it is a chain of latencies then (16 tokens of 8 heads of 128: 2.3 us, with 4
// passes 3.1 us).
template <int D, int CODE, typename T, int PASSES>
__global__ void __launch_bounds__(CQ_THREADS)
    k_cache_write(const T* __restrict__ key, const T* __restrict__ value, int64_t sk_t, int64_t sk_h, int64_t sv_t,
                  int64_t sv_h, CacheView c, const int64_t* __restrict__ slots, uint32_t items, uint32_t per_token, int KV,
                  T* __restrict__ key_out, T* __restrict__ value_out, int64_t sko_t, int64_t sko_h, int64_t svo_t,
                  int64_t svo_h) {
  constexpr int LANES = D / 8, ROWS = 32 / LANES;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t item = blockIdx.x * (CQ_THREADS / 32) + threadIdx.x / 32;
  if (item >= items) return;
  const uint32_t token = item / per_token;
  const int64_t t = token;
  const int first = (int)(item - token * per_token) * (ROWS * PASSES) + (threadIdx.x & 31) / LANES;
  const int lane = threadIdx.x % LANES;
  const int64_t slot = slots[t];
  uint4 v[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = first + i * ROWS;
    v[i] = make_uint4(0, 0, 0, 0);  // (every lane stays for the shuffles)
    if (r < 2 * KV) {
      const T* src = r >= KV ? value + t * sv_t + (r - KV) * sv_h : key + t * sk_t + r * sk_h;
      v[i] = *reinterpret_cast<const uint4*>(src + lane * 8);
    }
  }
  const bool written = slot >= 0 && slot < c.blocks * c.page;  // -1: a padded token, not written
  int64_t blk = 0;
  int place = 0;
  if (written) {
    blk = slot <= 0xffffffffll ? (int64_t)((uint32_t)slot / (uint32_t)c.page) : slot / c.page;
    place = (int)(slot - blk * c.page);
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = first + i * ROWS;
    const bool is_v = r >= KV;
    const int h = is_v ? r - KV : r;
    float x[8];
    unpack2<T>(v[i].x, x[0], x[1]);
    unpack2<T>(v[i].y, x[2], x[3]);
    unpack2<T>(v[i].z, x[4], x[5]);
    unpack2<T>(v[i].w, x[6], x[7]);
    float a = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) a = max_nan(a, fabsf(x[k]));
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
    if (r >= 2 * KV) continue;  // (the rows behind the last one are a whole pass, or the warp's last lanes)
    const float s = __fdiv_rn(a, code_max<CODE>());
    float y[2][4], b[2][4];
    uint32_t w[2];
    if (s >= 0x1p-80f && s < INFINITY) {
      const float inv = __frcp_rn(s);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float q = __fmul_rn(x[k], inv);
        y[k / 4][k % 4] = __fmaf_rn(__fmaf_rn(-q, s, x[k]), inv, q);
      }
    } else {
      const bool some = s > 0.0f && s < INFINITY;
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k / 4][k % 4] = some ? fminf(fmaxf(__fdiv_rn(x[k], s), -code_max<CODE>()), code_max<CODE>()) : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) w[k] = encode4<CODE>(y[k], b[k]);
    if (written) {
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

// One warp per packed token: its sequence, page and place are looked up once for all its rows; 16 codes a lane. Bound by the
// bytes: 48 sequences of 100 to 2100 tokens, 4 heads of 256, int8 to bf16: 64 us, 5.1 TB/s (8 codes a lane, whole rows a store: 90 us).
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
  if (b >= n || t < cu[b]) return;  // rows outside the sequences are left as they were
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
