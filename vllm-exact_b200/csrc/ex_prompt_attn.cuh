// Causal attention of packed prompts with grouped heads: sequence b has queries cu_q[b] .. cu_q[b + 1] and keys
// cu_k[b] .. cu_k[b + 1] of the packed arrays; its last query is its last key's token, so query i sees the keys
// j <= i + Lk - Lq. A query that sees none (Lk < Lq) gives zeros.
#pragma once
#include "ex_paged_rows.cuh"

namespace ex {

struct PaArgs {
  const void *q, *k, *v;
  int64_t sq_t, sq_h, sk_t, sk_h, sv_t, sv_h;
  const int32_t *cu_q, *cu_k;
  int n, H, G;
  int64_t tokens, keys;  // rows of q and of k, v
  float scale_log2;
  void* out;
  int64_t so_t, so_h;
};

constexpr int PS_ROWS = 64, PS_KEYS = 64;

// The tile'th tile of `rows` queries over all sequences: its sequence and first query in it; false if there is none.
__device__ __forceinline__ bool pa_find_tile(const int32_t* __restrict__ cu, int n, int rows, int tile, int& b, int& row0) {
  const int lane = threadIdx.x & 31;
  int seen = 0;
  for (int base = 0; base < n; base += 32) {
    int c = 0;
    if (base + lane < n) c = (max(0, cu[base + lane + 1] - cu[base + lane]) + rows - 1) / rows;
    int incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned m = __ballot_sync(0xffffffffu, seen + incl > tile);
    if (m) {
      const int l = __ffs(m) - 1;
      b = base + l;
      row0 = (tile - seen - __shfl_sync(0xffffffffu, incl - c, l)) * rows;
      return true;
    }
    seen += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// Queries and keys of sequence b; offsets that leave the arrays (or run backwards) are not followed.
__device__ __forceinline__ void pa_sequence(const PaArgs& a, int b, int& q0, int& Lq, int& k0, int& Lk) {
  q0 = a.cu_q[b];
  k0 = a.cu_k[b];
  const int64_t q1 = a.cu_q[b + 1], k1 = a.cu_k[b + 1];
  Lq = q0 >= 0 && q1 <= a.tokens ? (int)max((int64_t)0, q1 - q0) : 0;
  Lk = k0 >= 0 && k1 <= a.keys ? (int)max((int64_t)0, k1 - k0) : 0;
}

template <int D, bool F16>
__global__ void __launch_bounds__(128) k_prompt_attn(const __grid_constant__ PaArgs a) {
  extern __shared__ __align__(1024) uint8_t ps_smem[];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int b, row0;
  if (!pa_find_tile(a.cu_q, a.n, PS_ROWS, blockIdx.x / a.H, b, row0)) return;
  const int h = blockIdx.x % a.H, g = h / a.G;
  int q0, Lq, k0, Lk;
  pa_sequence(a, b, q0, Lq, k0, Lk);
  const int off = Lk - Lq;  // query i sees keys j <= i + off
  const int last = min(Lk, min(row0 + PS_ROWS, Lq) + off);  // keys that some row of the tile sees
  const uint32_t s0 = ex_smem_u32(ps_smem);
  constexpr int CH = D / 8;
  auto load = [&](uint32_t dst, const uint16_t* base, int64_t st, int r0, int rmax) {
    for (int c = tid; c < 64 * CH; c += 128) {
      const int r = c / CH, ch = c % CH;
      const bool ok = r0 + r < rmax;
      cp_async16(dst + pd_swz(r, ch, D), ok ? base + (int64_t)(r0 + r) * st + ch * 8 : base, ok);
    }
    cp_async_commit();
  };
  const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)q0 * a.sq_t + (int64_t)h * a.sq_h;
  const uint16_t* kp = reinterpret_cast<const uint16_t*>(a.k) + (int64_t)k0 * a.sk_t + (int64_t)g * a.sk_h;
  const uint16_t* vp = reinterpret_cast<const uint16_t*>(a.v) + (int64_t)k0 * a.sv_t + (int64_t)g * a.sv_h;
  const uint32_t sQ = s0, sK = s0 + 64 * D * 2, sV = sK + 64 * D * 2;
  load(sQ, qp, a.sq_t, row0, Lq);
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  for (int kb = 0; kb < last; kb += PS_KEYS) {
    __syncthreads();
    load(sK, kp, a.sk_t, kb, Lk);
    load(sV, vp, a.sv_t, kb, Lk);
    cp_async_wait<0>();
    __syncthreads();
    float sc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
#pragma unroll
    for (int kt = 0; kt < D / 16; ++kt) {
      uint32_t af[4];
      ldsm_x4(sQ + pd_swz(warp * 16 + (lane & 15), kt * 2 + (lane >> 4), D), af);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        uint32_t bf[4];
        ldsm_x4(sK + pd_swz(j * 8 + (lane & 7) + (lane >> 4) * 8, kt * 2 + ((lane >> 3) & 1), D), bf);
        mma_16816<F16>(sc[j], af, bf[0], bf[1]);
        mma_16816<F16>(sc[j + 1], af, bf[2], bf[3]);
      }
    }
    uint32_t pa[8][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // rows lane/4 and lane/4 + 8
      const int row = row0 + warp * 16 + (lane >> 2) + 8 * e;
      float mx = m[e];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int key = kb + j * 8 + (lane & 3) * 2 + f;
          float& x = sc[j][2 * e + f];
          x = key < Lk && key <= row + off ? x * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, x);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float sub = mx == -INFINITY ? 0.0f : mx;
      const float al = ex2(m[e] - sub);
      m[e] = mx;
      l[e] *= al;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p0 = ex2(sc[j][2 * e] - sub), p1 = ex2(sc[j][2 * e + 1] - sub);
        l[e] += p0 + p1;
        pa[j][e] = F16 ? pack2<__half>(p0, p1) : pack_bf16(p0, p1);
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][2 * e] *= al;
        o[i][2 * e + 1] *= al;
      }
    }
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const uint32_t af[4] = {pa[2 * kt][0], pa[2 * kt][1], pa[2 * kt + 1][0], pa[2 * kt + 1][1]};
#pragma unroll
      for (int i = 0; i < D / 8; i += 2) {
        uint32_t bf[4];
        ldsm_x4_t(sV + pd_swz(kt * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), i + (lane >> 4), D), bf);
        mma_16816<F16>(o[i], af, bf[0], bf[1]);
        mma_16816<F16>(o[i + 1], af, bf[2], bf[3]);
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    const int row = row0 + warp * 16 + (lane >> 2) + 8 * e;
    if (row >= Lq) continue;
    const float inv = l[e] > 0.0f ? 1.0f / l[e] : (l[e] == 0.0f ? 0.0f : l[e]);
    uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(q0 + row) * a.so_t + (int64_t)h * a.so_h + (lane & 3) * 2;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      *reinterpret_cast<uint32_t*>(dst + i * 8) = F16 ? pack2<__half>(o[i][2 * e] * inv, o[i][2 * e + 1] * inv)
                                                     : pack_bf16(o[i][2 * e] * inv, o[i][2 * e + 1] * inv);
  }
}

}  // namespace ex
