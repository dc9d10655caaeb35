// Attention of a few query rows per sequence over a paged cache: one token over an 8-bit cache (paged_decode_q8), or
// up to 64 drafted tokens under an ancestor mask over a 16-bit or 8-bit cache (tree_attention).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - m),  x_j = (q . k_j) scale log2 e,  m the largest x_j so far
//
// The rows of a KV head are the (token, query head) pairs of its group, token-major. Keys are taken in segments whose
// length depends on the request's own length only, in blocks of 64 inside a segment, and segments are merged in order:
// a row's bits do not depend on the other requests, the other rows, or where pages lie.
//
// Work: items (request, segment, KV head, tile of 8 NT rows), numbered by walking the requests' lengths on the device
// (no host sync); CTA c takes items c, c + gridDim.x, ... Neighbouring items share keys or their pages' DRAM rows.
//   warp 4     producer: TMA boxes of 8 or 16 tokens (one page each) into an mbarrier ring that runs ahead across
//              items; scales of an 8-bit cache by bulk copies.
//   warps 0-3  S^T = K Q^T: warp w owns keys 16w .. 16w + 15 of the block (MMA rows), the query rows are MMA columns.
//              The block's row maxima are exchanged through shared memory, P goes there in 16 bits, and
//              O^T += V^T P^T: warp w owns a quarter of the head dimension over all 64 keys, so O never needs a merge
//              and an 8-bit code is converted once.
// 8-bit codes become float16 (exact). The key scale multiplies the score; the value scale goes into P, divided by the
// largest value scale so far, which multiplies O in the end: float16 P keeps 11 bits of every weight that counts.
// Queries are brought to float16 by a power of two per row, exact for all elements above 2^-14 of the row's largest.
#pragma once
#include "ex_cache_q8.cuh"
#include "ex_paged_decode.cuh"
#include "ex_paged_decode_tma.cuh"

#ifndef XSEG_A
#define XSEG_A 256
#define XSEG_B 512
#endif
#ifndef XNW
#define XNW ((CODE == CODE_NONE ? 2 : 1) * D <= 128 ? 12 : (CODE == CODE_NONE ? 2 : 1) * D <= 256 ? 8 : 4)
#endif
#ifndef XMK
#define XMK ((CODE == CODE_NONE ? 2 : 1) * D <= 128 ? 2 : 1)
#endif
#ifndef XPER
#define XPER (D == 256 && (NT == 2 || CODE == CODE_NONE) ? 1 : 2)
#endif
namespace ex {

constexpr int PR_THREADS = 160;
constexpr int PR_BLK = 64;       // keys a block
constexpr int PR_MAX_TOKENS = 64;  // drafted tokens of a request (bits of a mask word)
constexpr float PR_LOG2E = 1.4426950408889634f;

// Keys a segment, by the request's own length.
__host__ __device__ inline int pr_segment(int64_t L) { return L <= 2048 ? XSEG_A : XSEG_B; }
__host__ __device__ inline int pr_segments(int64_t L) {
  const int s = pr_segment(L);
  const int n = (int)((L + s - 1) / s);
  return n < 1 ? 1 : n;
}
// most segments of any request of at most max_len keys
__host__ inline int pr_max_segments(int64_t max_len) {
  const int a = pr_segments(max_len < 2048 ? max_len : 2048), b = pr_segments(max_len);
  return a > b ? a : b;
}

template <int D, int CODE, int NT, int BLK = PR_BLK>
struct PrCfg {
  static constexpr int ESZ = CODE == CODE_NONE ? 2 : 1;
  static constexpr int ROW = D * ESZ;                       // bytes of a key
  static constexpr int PITCH = ROW < 128 ? ROW : 128;       // bytes of a row of a TMA box
  static constexpr int NH = ROW / PITCH;                    // boxes across the head dimension
  static constexpr int HALF = BLK * PITCH;
  static constexpr int TILE = BLK * ROW;                 // K or V of a block
  static constexpr int STAGE = 2 * TILE + (CODE == CODE_NONE ? 0 : 1024);  // + scales of the keys and of the values, padded
  static constexpr int Q_BYTES = 8 * NT * D * 2;
  static constexpr int P_BYTES = 8 * NT * 128;
  static constexpr int MISC = 4 * 8 * NT * 4 /* maxima */ + 8 * NT * 4 /* row factors or sums */ + 512;
  static constexpr int FIXED = Q_BYTES + P_BYTES + MISC + 1024;
  static constexpr int PER_SM = (D == 256 && CODE == CODE_NONE) ? 1 : 2;
  static constexpr int ROOM = (PER_SM == 1 ? 225 : 112) * 1024 - FIXED;
  static constexpr int STAGES = ROOM / STAGE < 8 ? ROOM / STAGE : 8;
  static constexpr int SMEM = FIXED + STAGES * STAGE;
  static_assert(STAGES >= 2, "ring");
};

struct PrArgs {
  const void* q;
  int64_t sq_t, sq_h;
  int q_is_f16;
  const int32_t* bt;
  int64_t sbt;
  const int32_t* seq_lens;
  const int32_t* qsl;        // null: one token per request
  const uint64_t* mask;      // null: a chain (each drafted token sees those before it and itself)
  int n, H, G, KV, BS, group_log2, max_tokens;  // TMA boxes of 2^group_log2 tokens
  int max_keys;              // keys of a request behind this many are not read
  int64_t blocks, tokens;    // pages of the cache, rows of q
  float scale_log2;
  const float* k_scale;
  const float* v_scale;
  int64_t ss_block, ss_head;
  int NS;
  int rows_lo, rows_hi;      // requests with rows_lo < T G <= rows_hi are this kernel's
  float* ws_m;
  float* ws_l;
  float* ws_acc;
  void* out;
  int64_t so_t, so_h;
};

// the tokens and keys of request b as the kernels count them
__device__ __forceinline__ void pr_request(const PrArgs& a, int b, int& first, int& T, int& L) {
  first = a.qsl ? a.qsl[b] : b;
  T = a.qsl ? a.qsl[b + 1] - first : 1;
  // more tokens than the caller said, or rows that q does not have: left untouched
  if (T < 0 || T > a.max_tokens || first < 0 || (int64_t)first + T > a.tokens) T = 0;
  L = max(0, a.seq_lens[b]);
}
__device__ __forceinline__ int pr_keys(const PrArgs& a, int L) { return min(L, a.max_keys); }

// Items in request order; all lanes of a warp walk together.
struct PrWalk {
  int base = -32, total = 0, start = 0;  // window of 32 requests, its items, its first item
  int cnt = 0, incl = 0, first = 0, T = 0, L = 0;
  // request, token rows and item within the request of item `it` (increasing from call to call); false: no such item
  __device__ __forceinline__ bool find(const PrArgs& a, int rows_per_tile, int it, int& b, int& b_first, int& b_T,
                                       int& b_L, int& rem) {
    const int lane = threadIdx.x & 31;
    while (it >= start + total) {
      start += total;
      base += 32;
      if (base >= a.n) return false;
      cnt = 0;
      const int r = base + lane;
      if (r < a.n) {
        pr_request(a, r, first, T, L);
        if (T > 0 && T * a.G > a.rows_lo && T * a.G <= a.rows_hi)
          cnt = pr_segments(pr_keys(a, L)) * a.KV * ((T * a.G + rows_per_tile - 1) / rows_per_tile);
      }
      incl = cnt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      total = __shfl_sync(0xffffffffu, incl, 31);
    }
    const int at = it - start;
    const int l = __ffs(__ballot_sync(0xffffffffu, incl > at)) - 1;
    b = base + l;
    b_first = __shfl_sync(0xffffffffu, first, l);
    b_T = __shfl_sync(0xffffffffu, T, l);
    b_L = __shfl_sync(0xffffffffu, L, l);
    rem = at - __shfl_sync(0xffffffffu, incl - cnt, l);
    return true;
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool F16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16) mma_f16_16816(d, a, b0, b1);
  else mma_bf16_16816(d, a, b0, b1);
}

// two codes (bytes 0, 1 and bytes 2, 3 of w) as two pairs of float16, exact
template <int CODE>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CODE == CODE_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;  // code + 128 as an unsigned byte; 0x6400 + u is the float16 1024 + u
    lo = __byte_perm(u, 0x64646464u, 0x4140);
    hi = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0xe480));  // -1152
    *reinterpret_cast<__half2*>(&lo) = __hadd2(*reinterpret_cast<__half2*>(&lo), off);
    *reinterpret_cast<__half2*>(&hi) = __hadd2(*reinterpret_cast<__half2*>(&hi), off);
  }
}

// byte offset of (row, 16-byte chunk of the row) of a tile written by TMA in boxes of PITCH bytes a row
template <int PITCH, int HALF>
__device__ __forceinline__ uint32_t pr_at(int row, int chunk) {
  if constexpr (PITCH == 128) {
    return (uint32_t)((chunk >> 3) * HALF + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
  } else {  // 64-byte rows, 64-byte swizzle
    return (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
  }
}

#define PR_BAR() asm volatile("bar.sync 1, 128;" ::: "memory")

// The producer warp: every block of the CTA's items through the ring, running ahead of the consumers.
template <int D, int CODE, int NT, int STAGES, int BLK = PR_BLK>
__device__ __forceinline__ void pr_produce(const PrArgs& a, const CUtensorMap* tm_k, const CUtensorMap* tm_v, uint8_t* smem,
                                           uint64_t* full_bar, uint64_t* empty_bar, uint32_t* sgood) {
  using C = PrCfg<D, CODE, NT, BLK>;
  constexpr bool Q8 = CODE != CODE_NONE;
  const int lane = threadIdx.x & 31;
  PrWalk walk;
  uint32_t blkno = 0;
  const int group = 1 << a.group_log2, per = BLK >> a.group_log2;  // at most 16 groups a block
  // an item's keys and, a window of 32 groups at a time, where they lie: lane l holds the page of group l (-1: none)
  int it = blockIdx.x, g = 0, start = 0, end = 0;
  const int32_t* btr = a.bt;
  auto next_item = [&]() {
    int b, first, T, L, rem;
    if (!walk.find(a, 8 * NT, it, b, first, T, L, rem)) return false;
    it += gridDim.x;
    const int tiles = (T * a.G + 8 * NT - 1) / (8 * NT);
    const int keys = pr_keys(a, L), seg = pr_segment(keys);
    g = (rem / tiles) % a.KV;
    start = rem / (tiles * a.KV) * seg;
    end = min(keys, start + seg);
    btr = a.bt + (int64_t)b * a.sbt;
    return true;
  };
  auto window = [&](int key, int last, int& page, int& off) {
    const int key0 = key + lane * group;
    page = -1;
    if (key0 < last) {
      page = btr[key0 / a.BS];
      off = key0 % a.BS;
    }
  };
  bool ok = true, have = next_item();
  int page = -1, off = 0;
  if (have) window(start, end, page, off);
  while (have && ok) {
    const int cg = g, cend = end;
    int wkey = start;
    bool more = true;
    // the window after this one is looked up while this one is loaded: of this item, or the first of the next
    while (more && ok) {
      const int after = wkey + 32 * group;
      int npage = -1, noff = 0;
      more = after < cend;
      if (more) {
        window(after, cend, npage, noff);
      } else {
        have = next_item();
        if (have) window(start, end, npage, noff);
      }
      const unsigned goods = __ballot_sync(0xffffffffu, page >= 0 && page < a.blocks);
      for (int base = 0; base < 32; base += per) {
        if (wkey + base * group >= cend) break;
        const int st = blkno % STAGES;
        ok = mbar_wait(empty_bar + st, ((blkno / STAGES) & 1u) ^ 1u, EX_DEVERR_WAIT_SLOT);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const unsigned good = (goods >> base) & ((1u << per) - 1u);
        if (lane == 0) {
          sgood[st] = good;
          mbar_arrive_expect_tx(full_bar + st, (uint32_t)(__popc(good) * group * (2 * C::ROW)));
        }
        __syncwarp();
        const int sub = lane - base;
        if (sub >= 0 && sub < per && ((good >> sub) & 1u)) {
          uint8_t* ks = smem + st * C::STAGE;
          uint8_t* vs = ks + C::TILE;
#pragma unroll
          for (int h = 0; h < C::NH; ++h) {
            tma_load_4d(ks + h * C::HALF + sub * group * C::PITCH, tm_k, full_bar + st, h * (C::PITCH / C::ESZ), cg, off, page);
            tma_load_4d(vs + h * C::HALF + sub * group * C::PITCH, tm_v, full_bar + st, h * (C::PITCH / C::ESZ), cg, off, page);
          }
        }
        if constexpr (Q8) {
          // scales: 16 bytes of four tokens a lane. Not by bulk copies: as many of them as of the codes' boxes, 64 bytes
          // each, would take as much of the TMA unit as the codes.
          const int from = min(base + ((lane * 4) >> a.group_log2), 31);
          const int pg = __shfl_sync(0xffffffffu, page, from), po = __shfl_sync(0xffffffffu, off, from);
          if (lane < BLK / 4 && ((goods >> from) & 1u)) {
            float* ss = reinterpret_cast<float*>(smem + st * C::STAGE + 2 * C::TILE) + lane * 4;
            const int64_t so = (int64_t)pg * a.ss_block + cg * a.ss_head + po + ((lane * 4) & (group - 1));
            cp_async16(ex_smem_u32(ss), a.k_scale + so, true);
            cp_async16(ex_smem_u32(ss + BLK), a.v_scale + so, true);
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ex_smem_u32(full_bar + st)) : "memory");
        }
        __syncwarp();
        ++blkno;
      }
      wkey = after;
      page = npage;
      off = noff;
    }
  }
  // every load has landed before the CTA ends (also after a wait that ran out)
  if (lane == 0) {
    for (uint32_t i = blkno > (uint32_t)STAGES ? blkno - STAGES : 0; i < blkno; ++i)
      mbar_wait(full_bar + i % STAGES, (i / STAGES) & 1u, EX_DEVERR_WAIT_TMA);
  }
  __syncwarp();
}

// 1 / f and f = 2^e with m in [f, 2f): what a row with largest element m is divided by on its way to float16. Exponents
// are kept where both are normal numbers.
__device__ __forceinline__ float pr_query_scale(float m, float& f) {
  int e = (int)((__float_as_uint(m) >> 23) & 255u);
  e = e == 255 ? 127 : min(max(e, 2), 252);
  f = __uint_as_float((uint32_t)e << 23);
  return __uint_as_float((uint32_t)(254 - e) << 23);
}

// a word of the transposing load: dims 2x, 2x + 1 of two keys, as the two keys' dim 2x and their dim 2x + 1
template <int CODE>
__device__ __forceinline__ void transposed_to_f16(uint32_t w, uint32_t& even, uint32_t& odd) {
  if constexpr (CODE == CODE_E4M3) {
    codes_to_f16<CODE>(__byte_perm(w, 0, 0x3120), even, odd);
  } else {
    const uint32_t u = w ^ 0x80808080u;
    even = __byte_perm(u, 0x64646464u, 0x4240);
    odd = __byte_perm(u, 0x64646464u, 0x4341);
    const __half2 off = __half2half2(__ushort_as_half(0xe480));  // -1152
    *reinterpret_cast<__half2*>(&even) = __hadd2(*reinterpret_cast<__half2*>(&even), off);
    *reinterpret_cast<__half2*>(&odd) = __hadd2(*reinterpret_cast<__half2*>(&odd), off);
  }
}

template <int D, int CODE, bool F16, int NT>
__global__ void __launch_bounds__(PR_THREADS, PrCfg<D, CODE, NT>::PER_SM)
    k_paged_rows(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                 const __grid_constant__ PrArgs a) {
  using C = PrCfg<D, CODE, NT>;
  constexpr bool Q8 = CODE != CODE_NONE;
  constexpr bool MF16 = Q8 || F16;  // MMA type
  constexpr int ROWS = 8 * NT;
  constexpr int MT = D / 64;        // 16-dim tiles of a warp's quarter
  extern __shared__ uint8_t pr_smem_raw[];
  uint8_t* smem = pr_smem_raw + ((0u - ex_smem_u32(pr_smem_raw)) & 1023u);
  uint8_t* sq = smem + C::STAGES * C::STAGE;
  uint8_t* sp = sq + C::Q_BYTES;
  float* smax = reinterpret_cast<float*>(sp + C::P_BYTES);  // [4][ROWS]
  float* sfac = smax + 4 * ROWS;                            // [ROWS]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sfac + ROWS);
  uint64_t* empty_bar = full_bar + 8;
  uint32_t* sgood = reinterpret_cast<uint32_t*>(empty_bar + 8);  // groups of a stage whose page exists
  volatile int* sfail = reinterpret_cast<int*>(sgood + 8);       // a wait ran out
  volatile int* sbad = reinterpret_cast<int*>(sgood + 9);        // [4] a warp's keys have values that are not finite

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  if (tid == 0) {
    *sfail = 0;
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(full_bar + i, Q8 ? 33 : 1);  // codes: and every producer lane's copies of scales
      mbar_init(empty_bar + i, 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_wait();

  if (warp == 4) {
    pr_produce<D, CODE, NT, C::STAGES>(a, &tm_k, &tm_v, smem, full_bar, empty_bar, sgood);
    return;
  }
  PrWalk walk;
  uint32_t blkno = 0;  // blocks through the ring so far
  // -------------------------------------------------------------------------------------------------- consumers
  const int qr = lane >> 2, qc = (lane & 3) * 2;
  const uint32_t sq0 = ex_smem_u32(sq), sp0 = ex_smem_u32(sp);
  bool alive = true;
  for (int it = blockIdx.x; alive; it += gridDim.x) {
    int b, first, T, L, rem;
    if (!walk.find(a, ROWS, it, b, first, T, L, rem)) break;
    const int R = T * a.G;
    const int tiles = (R + ROWS - 1) / ROWS;
    const int row0 = (rem % tiles) * ROWS;
    const int g = (rem / tiles) % a.KV, s = rem / (tiles * a.KV);
    const int keys = pr_keys(a, L), seg = pr_segment(keys);
    const int start = s * seg, end = min(keys, start + seg);
    const int ctx = L - T;  // keys before the drafted tokens

    // queries to shared memory: row-major, 16-byte chunks swizzled; a row takes D/8 lanes
    PR_BAR();  // the last item's readers are done
    {
      constexpr int LANES = D / 8;
      const int c = tid % LANES;
      for (int r = tid / LANES; r < ROWS; r += 128 / LANES) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row0 + r < R) {
          const int t = (row0 + r) / a.G, h = (row0 + r) % a.G;
          v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(first + t) * a.sq_t +
                                              (int64_t)(g * a.G + h) * a.sq_h + c * 8);
        }
        if constexpr (!Q8) {
          *reinterpret_cast<uint4*>(sq + r * D * 2 + ((c ^ (r & 7)) << 4)) = v;
        } else {
          float f = 1.0f;
          if (!a.q_is_f16) {
            float x[8];
            unpack2<__nv_bfloat16>(v.x, x[0], x[1]);
            unpack2<__nv_bfloat16>(v.y, x[2], x[3]);
            unpack2<__nv_bfloat16>(v.z, x[4], x[5]);
            unpack2<__nv_bfloat16>(v.w, x[6], x[7]);
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float inv = pr_query_scale(m, f);
            v.x = pack2<__half>(x[0] * inv, x[1] * inv);
            v.y = pack2<__half>(x[2] * inv, x[3] * inv);
            v.z = pack2<__half>(x[4] * inv, x[5] * inv);
            v.w = pack2<__half>(x[6] * inv, x[7] * inv);
          }
          if (c == 0) sfac[r] = f * a.scale_log2;
          // A thread's four code bytes are four consecutive dims, MMA slots 2i, 2i+1, 2i+8, 2i+9 of a 16-dim step: the
          // query dims are stored in slot order. Dims 8c' .. 8c'+7 of the step: pairs go to slots (4c'+0, 4c'+8, 4c'+2, 4c'+10).
          uint8_t* base = sq + r * D * 2;
          const int step = c >> 1, half = c & 1;  // this chunk holds dims 8 half .. of the 16-dim step
          auto put = [&](int slot, uint32_t val) {
            const int chunk = step * 2 + (slot >> 3);
            *reinterpret_cast<uint32_t*>(base + ((chunk ^ (r & 7)) << 4) + (slot & 7) * 2) = val;
          };
          put(4 * half, v.x);
          put(4 * half + 8, v.y);
          put(4 * half + 2, v.z);
          put(4 * half + 10, v.w);
        }
      }
    }
    PR_BAR();
    float fac[2 * NT];  // score factors of this thread's columns
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) fac[i] = Q8 ? sfac[(i >> 1) * 8 + qc + (i & 1)] : a.scale_log2;

    float m_run[2 * NT], l_run[2 * NT];
    float o[MT][NT][4];
    float vm = 0.0f;  // largest value scale so far
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      m_run[i] = -INFINITY;
      l_run[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.0f;

    for (int kb = start; kb < end; kb += PR_BLK, ++blkno) {
      const int st = blkno % C::STAGES;
      if (!mbar_wait(full_bar + st, (blkno / C::STAGES) & 1u, EX_DEVERR_WAIT_TMA)) *sfail = 1;
      uint8_t* ks = smem + st * C::STAGE;
      uint8_t* vs = ks + C::TILE;
      const uint32_t ks0 = ex_smem_u32(ks), vs0 = ex_smem_u32(vs);
      const float* kscale = reinterpret_cast<const float*>(ks + 2 * C::TILE);
      const float* vscale = kscale + PR_BLK;
      const uint32_t good = sgood[st];
      const int per = PR_BLK >> a.group_log2;
      const bool whole = kb + PR_BLK <= min(end, ctx) && good == (1u << per) - 1u;  // every row sees every key

      // S^T: 16 keys x ROWS
      float sc[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
#pragma unroll
      for (int kt = 0; kt < D / 16; kt += (Q8 ? 2 : 1)) {
        uint32_t af[2][4];
        if constexpr (Q8) {
          uint32_t w[4];  // keys 0-7 | 8-15 of dims 16 kt .., then of the next 16 dims
          const int row = warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
          ldsm_x4(ks0 + pr_at<C::PITCH, C::HALF>(row, kt + (lane >> 4)), w);
          codes_to_f16<CODE>(w[0], af[0][0], af[0][2]);
          codes_to_f16<CODE>(w[1], af[0][1], af[0][3]);
          codes_to_f16<CODE>(w[2], af[1][0], af[1][2]);
          codes_to_f16<CODE>(w[3], af[1][1], af[1][3]);
        } else {
          ldsm_x4(ks0 + pr_at<C::PITCH, C::HALF>(warp * 16 + (lane & 15), kt * 2 + (lane >> 4)), af[0]);
        }
#pragma unroll
        for (int u = 0; u < (Q8 ? 2 : 1); ++u) {
          const int k2 = (kt + u) * 2;
          if constexpr (NT == 1) {
            uint32_t b0, b1;
            const uint32_t ad = sq0 + (lane & 7) * D * 2 + (((k2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
            asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(ad));
            mma_16816<MF16>(sc[0], af[u], b0, b1);
          } else {
#pragma unroll
            for (int j = 0; j < NT; j += 2) {
              uint32_t bf[4];
              const int r = j * 8 + (lane & 7) + (lane >> 4) * 8;
              ldsm_x4(sq0 + r * D * 2 + (((k2 + ((lane >> 3) & 1)) ^ (r & 7)) << 4), bf);
              mma_16816<MF16>(sc[j], af[u], bf[0], bf[1]);
              mma_16816<MF16>(sc[j + 1], af[u], bf[2], bf[3]);
            }
          }
        }
      }
      // scale, mask, block maxima
      const int k0 = warp * 16 + qr;  // this thread's keys are kb + k0 and kb + k0 + 8
      float ksc[2] = {1.0f, 1.0f}, vsc[2] = {1.0f, 1.0f};
      if constexpr (Q8) {
        ksc[0] = kscale[k0];
        ksc[1] = kscale[k0 + 8];
        vsc[0] = vscale[k0];
        vsc[1] = vscale[k0 + 8];
      }
      float mx[2 * NT];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[j][e] *= Q8 ? fac[2 * j + (e & 1)] * ksc[e >> 1] : fac[2 * j + (e & 1)];
      uint32_t bits = 0xffffffffu;  // visible: bit (2 * j + (e & 1)) * 2 + (e >> 1)
      if (!whole) {
        bits = 0;
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
          const int r = row0 + (i >> 1) * 8 + qc + (i & 1);
          const int t = r / a.G;
          uint64_t w = 0;
          if (r < R) w = a.mask ? a.mask[first + t] : (t >= 63 ? ~0ull : (2ull << t) - 1ull);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int kk = k0 + 8 * h, key = kb + kk;
            const int d = key - ctx;
            const bool see = r < R && key < end && ((good >> (kk >> a.group_log2)) & 1u) && (d < 0 || ((w >> d) & 1ull));
            if (see) bits |= 1u << (2 * i + h);
          }
        }
        // values of keys that may not be read: zeroed, since 0 * NaN would reach O
        int bad = 0;
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
          const int kk = warp * 16 + i;
          const bool none = kb + kk >= end || !((good >> (kk >> a.group_log2)) & 1u);
          for (int c = lane; c < C::ROW / 16; c += 32) {
            uint4* x = reinterpret_cast<uint4*>(vs + pr_at<C::PITCH, C::HALF>(kk, c));
            if (none) {
              *x = make_uint4(0, 0, 0, 0);
            } else if constexpr (!Q8) {  // (codes are finite; a scale that is not only reaches rows that see it)
              const uint32_t e = F16 ? 0x7c00u : 0x7f80u;
              const uint32_t w[4] = {x->x, x->y, x->z, x->w};
#pragma unroll
              for (int k = 0; k < 4; ++k) bad |= (w[k] & e) == e || ((w[k] >> 16) & e) == e;
            }
          }
        }
        if constexpr (!Q8) {
          bad = __any_sync(0xffffffffu, bad);
          if (lane == 0) sbad[warp] = bad;
        }
        fence_proxy_async_shared();  // the ring slot is written by TMA next
      }
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) {
        float& s0 = sc[i >> 1][i & 1];
        float& s1 = sc[i >> 1][2 + (i & 1)];
        if (!((bits >> (2 * i)) & 1u)) s0 = -INFINITY;
        if (!((bits >> (2 * i + 1)) & 1u)) s1 = -INFINITY;
        float v = fmaxf(s0, s1);
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
        mx[i] = v;
      }
      if (qr == 0) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
          *reinterpret_cast<float2*>(smax + warp * ROWS + j * 8 + qc) = make_float2(mx[2 * j], mx[2 * j + 1]);
      }
      float beta = 1.0f, vinv = 1.0f;
      if constexpr (Q8) {  // the largest finite value scale among the keys that may be read
        float v = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int kk = lane + 32 * h;
          if (kb + kk < end && ((good >> (kk >> a.group_log2)) & 1u) && vscale[kk] < INFINITY) v = fmaxf(v, vscale[kk]);
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
        const float vn = fmaxf(vm, v);
        const bool tiny = vn < 1.2e-38f;  // such values are zero next to any output type's smallest step
        beta = tiny ? 1.0f : __fdividef(vm, vn);
        vinv = tiny ? 0.0f : __frcp_rn(vn);
        vm = vn;
      }
      PR_BAR();
      if (*sfail) {  // the same for every thread here: the flag is only set before the barrier
        alive = false;
        break;
      }
      float alpha[2 * NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float2 v = *reinterpret_cast<const float2*>(smax + j * 8 + qc);
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          const float2 u = *reinterpret_cast<const float2*>(smax + w * ROWS + j * 8 + qc);
          v.x = fmaxf(v.x, u.x);
          v.y = fmaxf(v.y, u.y);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * j + e;
          const float mn = fmaxf(m_run[i], e ? v.y : v.x);
          const float sub = mn == -INFINITY ? 0.0f : mn;
          alpha[i] = mn == -INFINITY ? 1.0f : ex2(m_run[i] - mn);
          m_run[i] = mn;
          const float p0 = ex2(sc[j][e] - sub), p1 = ex2(sc[j][2 + e] - sub);
          l_run[i] = l_run[i] * alpha[i] + (p0 + p1);
          sc[j][e] = p0;
          sc[j][2 + e] = p1;
          if constexpr (Q8) {  // a key that is not seen has a scale that may be anything
            sc[j][e] = ((bits >> (2 * i)) & 1u) ? p0 * (vsc[0] * vinv) : 0.0f;
            sc[j][2 + e] = ((bits >> (2 * i + 1)) & 1u) ? p1 * (vsc[1] * vinv) : 0.0f;
          }
        }
        // P^T (rows x keys): 8 x 8 blocks transposed on the way, so that a B fragment is one ldmatrix row
        const uint32_t p01 = movmatrix_t(MF16 ? pack2<__half>(sc[j][0], sc[j][1]) : pack_bf16(sc[j][0], sc[j][1]));
        const uint32_t p23 = movmatrix_t(MF16 ? pack2<__half>(sc[j][2], sc[j][3]) : pack_bf16(sc[j][2], sc[j][3]));
        const int r = j * 8 + qr;
        *reinterpret_cast<uint32_t*>(sp + r * 128 + (((warp * 2) ^ (r & 7)) << 4) + qc * 2) = p01;
        *reinterpret_cast<uint32_t*>(sp + r * 128 + (((warp * 2 + 1) ^ (r & 7)) << 4) + qc * 2) = p23;
      }
      PR_BAR();
      // O^T: this warp's quarter of the head dimension
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          o[i][j][0] *= alpha[2 * j] * beta;
          o[i][j][1] *= alpha[2 * j + 1] * beta;
          o[i][j][2] *= alpha[2 * j] * beta;
          o[i][j][3] *= alpha[2 * j + 1] * beta;
        }
      bool slow = false;
      if constexpr (!Q8) {
        // values that are not finite behind a row's mask: a product of tensor cores would give 0 * inf to rows that
        // do not see them, so such a block's products are made one by one
        slow = !whole && (sbad[0] | sbad[1] | sbad[2] | sbad[3]);
        if (slow) {
#pragma unroll 1
          for (int kk = 0; kk < PR_BLK; ++kk) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int d = (warp * MT + i) * 16 + qr + (e >> 1) * 8;
                const uint16_t vr = *reinterpret_cast<const uint16_t*>(vs + pr_at<C::PITCH, C::HALF>(kk, d >> 3) + (d & 7) * 2);
                const float v = F16 ? __half2float(__ushort_as_half(vr)) : __uint_as_float((uint32_t)vr << 16);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                  const int r = j * 8 + qc + (e & 1);
                  const uint16_t pr = *reinterpret_cast<const uint16_t*>(sp + r * 128 + (((kk >> 3) ^ (r & 7)) << 4) + (kk & 7) * 2);
                  const float p = F16 ? __half2float(__ushort_as_half(pr)) : __uint_as_float((uint32_t)pr << 16);
                  if (p != 0.0f) o[i][j][e] += p * v;
                }
              }
            }
          }
        }
      }
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {  // 16 keys a step
        if (slow) break;
        uint32_t va[MT][4];
        const int mi = lane >> 3;
        if constexpr (!Q8) {
#pragma unroll
          for (int i = 0; i < MT; ++i)  // 16 dims: chunks 2x, 2x + 1; dims qr and qr + 8
            ldsm_x4_t(vs0 + pr_at<C::PITCH, C::HALF>(kt * 16 + (mi >> 1) * 8 + (lane & 7), (warp * MT + i) * 2 + (mi & 1)), va[i]);
        } else {
          // one 16-byte chunk is 16 dims; after the transposing load a word holds dims 2 qr, 2 qr + 1 of two keys
          if constexpr (MT == 1) {
            uint32_t w0, w1;
            const uint32_t ad = vs0 + pr_at<C::PITCH, C::HALF>(kt * 16 + (mi & 1) * 8 + (lane & 7), warp);
            asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(w0), "=r"(w1) : "r"(ad));
            transposed_to_f16<CODE>(w0, va[0][0], va[0][1]);
            transposed_to_f16<CODE>(w1, va[0][2], va[0][3]);
          } else {
#pragma unroll
            for (int i = 0; i < MT; i += 2) {
              uint32_t w[4];
              ldsm_x4_t(vs0 + pr_at<C::PITCH, C::HALF>(kt * 16 + (mi & 1) * 8 + (lane & 7), warp * MT + i + (mi >> 1)), w);
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                transposed_to_f16<CODE>(w[2 * u], va[i + u][0], va[i + u][1]);
                transposed_to_f16<CODE>(w[2 * u + 1], va[i + u][2], va[i + u][3]);
              }
            }
          }
        }
        if constexpr (NT == 1) {
          uint32_t b0, b1;
          const uint32_t ad = sp0 + (lane & 7) * 128 + (((kt * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
          asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(ad));
#pragma unroll
          for (int i = 0; i < MT; ++i) mma_16816<MF16>(o[i][0], va[i], b0, b1);
        } else {
#pragma unroll
          for (int j = 0; j < NT; j += 2) {
            uint32_t bf[4];
            const int r = j * 8 + (lane & 7) + (lane >> 4) * 8;
            ldsm_x4(sp0 + r * 128 + (((kt * 2 + ((lane >> 3) & 1)) ^ (r & 7)) << 4), bf);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              mma_16816<MF16>(o[i][j], va[i], bf[0], bf[1]);
              mma_16816<MF16>(o[i][j + 1], va[i], bf[2], bf[3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty_bar + st);
    }

    if (!alive) break;
    // the segment's sums: a warp holds those of its own keys
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      float v = l_run[i];
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      l_run[i] = v;
    }
    PR_BAR();  // the last block's maxima have been read
    if (qr == 0) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
        *reinterpret_cast<float2*>(smax + warp * ROWS + j * 8 + qc) = make_float2(l_run[2 * j], l_run[2 * j + 1]);
    }
    PR_BAR();
    const bool single = pr_segments(keys) == 1;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      const int c = (i >> 1) * 8 + qc + (i & 1);
      const int r = row0 + c;
      if (r >= R) continue;
      const float l = (smax[c] + smax[ROWS + c]) + (smax[2 * ROWS + c] + smax[3 * ROWS + c]);
      const int t = r / a.G, h = g * a.G + r % a.G;
      const float up = Q8 ? vm : 1.0f;
      if (single) {
        const float inv = l > 0.0f ? up / l : (l == 0.0f ? 0.0f : l);  // nothing seen: zeros; NaN stays NaN
        const int64_t at = (int64_t)(first + t) * a.so_t + (int64_t)h * a.so_h;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float x = o[mt][i >> 1][i & 1] * inv, y = o[mt][i >> 1][2 + (i & 1)] * inv;
          const int d0 = (warp * MT + mt) * 16;
          if constexpr (Q8) {
            uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + at + d0 + 2 * qr);
            *dst = a.q_is_f16 ? pack2<__half>(x, y) : pack_bf16(x, y);
          } else {
            ex_store_out<F16 ? EX_DTYPE_F16 : EX_DTYPE_BF16>(a.out, at + d0 + qr, x);
            ex_store_out<F16 ? EX_DTYPE_F16 : EX_DTYPE_BF16>(a.out, at + d0 + qr + 8, y);
          }
        }
      } else {
        const int64_t pi = ((int64_t)(first + t) * a.H + h) * a.NS + s;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float x = o[mt][i >> 1][i & 1] * up, y = o[mt][i >> 1][2 + (i & 1)] * up;
          float* dst = a.ws_acc + pi * D + (warp * MT + mt) * 16;
          if constexpr (Q8) {
            *reinterpret_cast<float2*>(dst + 2 * qr) = make_float2(x, y);
          } else {
            dst[qr] = x;
            dst[qr + 8] = y;
          }
        }
        if (warp == 0 && qr == 0) {
          a.ws_m[pi] = m_run[i];
          a.ws_l[pi] = l;
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// At most 16 rows of a KV head: a decode step, or a few drafted tokens.
//
// Every warp streams its own items: it loads blocks of 16 MK keys into its own ring, S blocks ahead and on into its next
// item, and computes S^T = K Q^T, P and O^T += V^T P^T on what has arrived. No thread waits for another warp. m is taken up
// only when a score passes it by more than 6 (a factor of 64; p stays small enough for float16), and the reference of
// the value scales when one is 64 times it: the common path has two votes and no shuffles. Both are decided for
// every row (every key) alone.
// ------------------------------------------------------------------------------------------------------------------
template <int D, int CODE, int NT>
struct PfCfg {
  static constexpr int MK = XMK;                       // 16-key tiles of a block
  static constexpr int NW = XNW;                       // warps of a CTA, one CTA per SM
  static constexpr int BLK = 16 * MK;
  using R = PrCfg<D, CODE, NT, BLK>;
  static constexpr int STAGE = 2 * R::TILE;
  static constexpr int SCALES = CODE == CODE_NONE ? 0 : 8 * BLK;  // bytes of a block's scales, keys' first
  static constexpr int ROOM = (225 * 1024) / NW;
  static constexpr int STAGES = ROOM / (STAGE + SCALES) < 8 ? ROOM / (STAGE + SCALES) : 8;
  static constexpr int SMEM = NW * STAGES * (STAGE + SCALES) + 1024 + NW * 8 * (8 + 4);
  static_assert(STAGES >= 2, "ring");
};

template <int D, int CODE, bool F16, int NT>
__global__ void __launch_bounds__(32 * PfCfg<D, CODE, NT>::NW, 1)
    k_paged_few(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ PrArgs a) {
  using F = PfCfg<D, CODE, NT>;
  using C = typename F::R;
  constexpr int MK = F::MK, BLK = F::BLK, NW = F::NW, STAGES = F::STAGES;
  constexpr bool Q8 = CODE != CODE_NONE;
  constexpr bool MF16 = Q8 || F16;
  constexpr int ROWS = 8 * NT;
  constexpr int KT = D / 16;
  extern __shared__ uint8_t pr_smem_raw[];
  uint8_t* smem = pr_smem_raw + ((0u - ex_smem_u32(pr_smem_raw)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* ring = smem + warp * STAGES * F::STAGE;
  uint8_t* behind = smem + NW * STAGES * F::STAGE;
  float* scales = reinterpret_cast<float*>(behind + warp * STAGES * F::SCALES);
  behind += NW * STAGES * F::SCALES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(behind) + warp * 8;
  uint32_t* sgood = reinterpret_cast<uint32_t*>(behind + NW * 64) + warp * 8;  // groups whose page exists

  pdl_launch_dependents();
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(full_bar + i, Q8 ? 33 : 1);  // codes: and every lane's copies of scales
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  pdl_wait();

  const int stride = gridDim.x * NW;
  const int glog = a.group_log2, group = 1 << glog, per = BLK >> glog;  // groups of a block
  // ---- what is loaded next: an item's keys and, for groups lane and lane + 32 of it, where they lie
  PrWalk lwalk;
  int lit = warp * gridDim.x + blockIdx.x, lg = 0, lkey = 0, lend = 0, lgi = 0, page[2] = {-1, -1}, off[2] = {0, 0};
  bool lhave = true;
  int lslot = 0;
  auto load_item = [&]() {  // the next item that has keys
    do {
      int b, first, T, L, rem;
      lhave = lwalk.find(a, ROWS, lit, b, first, T, L, rem);
      if (!lhave) return;
      lit += stride;
      const int keys = pr_keys(a, L), seg = pr_segment(keys);
      lg = rem % a.KV;
      lkey = rem / a.KV * seg;
      lend = min(keys, lkey + seg);
      lgi = 0;
      const int32_t* btr = a.bt + (int64_t)b * a.sbt;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = lkey + (lane + 32 * i) * group;
        page[i] = -1;
        if (key < lend) {
          page[i] = btr[key / a.BS];
          off[i] = key % a.BS;
        }
      }
    } while (lkey >= lend);
  };
  auto load_block = [&]() {
    if (!lhave) return;
    const int pg = lgi < 32 ? page[0] : page[1], po = lgi < 32 ? off[0] : off[1];
    const unsigned goods = __ballot_sync(0xffffffffu, pg >= 0 && pg < a.blocks);
    const int base = lgi & 31;
    const unsigned good = (goods >> base) & ((1u << per) - 1u);
    uint8_t* ks = ring + lslot * F::STAGE;
    uint64_t* bar = full_bar + lslot;
    if (lane == 0) {
      sgood[lslot] = good;
      mbar_arrive_expect_tx(bar, (uint32_t)(__popc(good) * group * 2 * C::ROW));
    }
    __syncwarp();
    const int sub = lane - base;
    if (sub >= 0 && sub < per && ((good >> sub) & 1u)) {
#pragma unroll
      for (int h = 0; h < C::NH; ++h) {
        tma_load_4d(ks + h * C::HALF + sub * group * C::PITCH, &tm_k, bar, h * (C::PITCH / C::ESZ), lg, po, pg);
        tma_load_4d(ks + C::TILE + h * C::HALF + sub * group * C::PITCH, &tm_v, bar, h * (C::PITCH / C::ESZ), lg, po, pg);
      }
    }
    if constexpr (Q8) {
      // scales: 16 bytes of four tokens a lane. Not by bulk copies: as many of them as of the codes' boxes would take as
      // much of the TMA unit as the codes.
      const int tok = (lane * 4) & (BLK - 1);
      const int from = base + (tok >> glog);
      const int p2 = __shfl_sync(0xffffffffu, pg, from), o2 = __shfl_sync(0xffffffffu, po, from);
      if (lane < BLK / 2 && ((goods >> from) & 1u)) {
        float* ss = scales + lslot * 2 * BLK + lane * 4;
        const float* src = lane < BLK / 4 ? a.k_scale : a.v_scale;
        cp_async16(ex_smem_u32(ss), src + (int64_t)p2 * a.ss_block + lg * a.ss_head + o2 + (tok & (group - 1)), true);
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ex_smem_u32(bar)) : "memory");
    }
    if (++lslot == STAGES) lslot = 0;
    lkey += BLK;
    lgi += per;
    if (lkey >= lend) load_item();
  };
  load_item();
#pragma unroll 1
  for (int i = 0; i < STAGES; ++i) load_block();

  // ---- what is computed
  PrWalk walk;
  int st = 0;  // ring slot of the next block and its phase
  uint32_t phase = 0;
  const int qr = lane >> 2, qc = (lane & 3) * 2;
  bool ok = true;
  for (int it = warp * gridDim.x + blockIdx.x; ok; it += stride) {
    int b, first, T, L, rem;
    if (!walk.find(a, ROWS, it, b, first, T, L, rem)) break;
    const int R = T * a.G;  // one tile: at most ROWS
    const int g = rem % a.KV, s = rem / a.KV;
    const int keys = pr_keys(a, L), seg = pr_segment(keys);
    const int start = s * seg, end = min(keys, start + seg);
    const int ctx = L - T;

    // query fragments of the MMA's second operand: row qr of each 8, dims 16 kt + 2 (lane % 4) + {0, 1, 8, 9} for a 16-bit
    // cache; for codes the four dims 16 kt + 4 (lane % 4) .., since a word of four codes takes those slots
    uint32_t qf[NT][KT][2];
    float qs[NT];  // what a row was divided by
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = j * 8 + qr;
      const bool have = r < R;
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(first + (have ? r / a.G : 0)) * a.sq_t +
                           (int64_t)(g * a.G + (have ? r % a.G : 0)) * a.sq_h;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        if constexpr (Q8) {
          const uint2 v = *reinterpret_cast<const uint2*>(qp + kt * 16 + 2 * qc);
          qf[j][kt][0] = have ? v.x : 0u;
          qf[j][kt][1] = have ? v.y : 0u;
        } else {
          const uint32_t v0 = *reinterpret_cast<const uint32_t*>(qp + kt * 16 + qc);
          const uint32_t v1 = *reinterpret_cast<const uint32_t*>(qp + kt * 16 + qc + 8);
          qf[j][kt][0] = have ? v0 : 0u;
          qf[j][kt][1] = have ? v1 : 0u;
        }
      }
      qs[j] = 1.0f;
      if (Q8 && !a.q_is_f16) {
        float m = 0.0f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float x, y;
            unpack2<__nv_bfloat16>(qf[j][kt][i], x, y);
            m = fmaxf(m, fmaxf(fabsf(x), fabsf(y)));
          }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const float inv = pr_query_scale(m, qs[j]);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float x, y;
            unpack2<__nv_bfloat16>(qf[j][kt][i], x, y);
            qf[j][kt][i] = pack2<__half>(x * inv, y * inv);
          }
      }
    }
    float fac[2 * NT];  // score factors of columns qc, qc + 1 of each 8
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i)
      fac[i] = Q8 ? __shfl_sync(0xffffffffu, qs[i >> 1], (qc + (i & 1)) * 4) * a.scale_log2 : a.scale_log2;

    float m[2 * NT], l[2 * NT], o[KT][NT][4];
    float vref = 0.0f, vinv = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.0f;

    for (int kb = start; kb < end; kb += BLK) {
      ok = mbar_wait(full_bar + st, phase, EX_DEVERR_WAIT_TMA);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint8_t* ks = ring + st * F::STAGE;
      uint8_t* vs = ks + C::TILE;
      const float* kscale = scales + st * 2 * BLK + qr;  // then those of the values
      const uint32_t good = sgood[st];
      const bool whole = kb + BLK <= min(end, ctx) && good == (1u << per) - 1u;
      // S^T, 16 keys a tile: a column's chunk c of the tile's rows lies at (base ^ (c % 8) * 16) + c / 8 * HALF for even c
      float sc[MK][NT][4];
#pragma unroll
      for (int i = 0; i < MK; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) sc[i][j][0] = sc[i][j][1] = sc[i][j][2] = sc[i][j][3] = 0.0f;
      uint32_t kbase[MK];
#pragma unroll
      for (int i = 0; i < MK; ++i)
        kbase[i] = ex_smem_u32(ks) +
                   (Q8 ? pr_at<C::PITCH, C::HALF>(16 * i + (lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4)
                       : pr_at<C::PITCH, C::HALF>(16 * i + (lane & 15), lane >> 4));
#pragma unroll
      for (int kt = 0; kt < KT; kt += (Q8 ? 2 : 1)) {
        const int c = Q8 ? kt : 2 * kt;
#pragma unroll
        for (int i = 0; i < MK; ++i) {
          uint32_t af[2][4];
          uint32_t w[4];
          ldsm_x4((kbase[i] ^ ((c & 7) << 4)) + (c >> 3) * C::HALF, w);
          if constexpr (Q8) {
            codes_to_f16<CODE>(w[0], af[0][0], af[0][2]);
            codes_to_f16<CODE>(w[1], af[0][1], af[0][3]);
            codes_to_f16<CODE>(w[2], af[1][0], af[1][2]);
            codes_to_f16<CODE>(w[3], af[1][1], af[1][3]);
          } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) af[0][x] = w[x];
          }
#pragma unroll
          for (int u = 0; u < (Q8 ? 2 : 1); ++u)
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_16816<MF16>(sc[i][j], af[u], qf[j][kt + u][0], qf[j][kt + u][1]);
        }
      }
      float vsc[MK][2];
#pragma unroll
      for (int i = 0; i < MK; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float ksc = Q8 ? kscale[16 * i + 8 * e] : 1.0f;
          vsc[i][e] = Q8 ? kscale[BLK + 16 * i + 8 * e] : 1.0f;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            sc[i][j][2 * e] *= Q8 ? fac[2 * j] * ksc : fac[2 * j];
            sc[i][j][2 * e + 1] *= Q8 ? fac[2 * j + 1] * ksc : fac[2 * j + 1];
          }
        }
      bool slow = false;  // 16-bit: a value that is not finite and that some row may not see
      uint32_t hidden = 0;  // bit ((i NT + j) 4 + e): the row does not see the key
      if (!whole) {
        int bad = 0;
#pragma unroll
        for (int i = 0; i < MK; ++i) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int kk = 16 * i + qr + 8 * e, d = kb + kk - ctx;
            const bool readable = kb + kk < end && ((good >> (kk >> a.group_log2)) & 1u);
            if (!readable) vsc[i][e] = 0.0f;
#pragma unroll
            for (int x = 0; x < 2 * NT; ++x) {
              const int r = (x >> 1) * 8 + qc + (x & 1);
              bool see = r < R && readable;
              if (see && d >= 0) {
                const int t = r / a.G;
                const uint64_t w = a.mask ? a.mask[first + t] : (t >= 63 ? ~0ull : (2ull << t) - 1ull);
                see = (w >> d) & 1ull;
              }
              if (!see) {
                hidden |= 1u << ((i * NT + (x >> 1)) * 4 + 2 * e + (x & 1));
                sc[i][x >> 1][2 * e + (x & 1)] = -INFINITY;
              }
            }
          }
        }
#pragma unroll 1
        for (int i = 0; i < 16 * MK; ++i) {
          const bool none = kb + i >= end || !((good >> ((i) >> a.group_log2)) & 1u);
          for (int c = lane; c < C::ROW / 16; c += 32) {
            uint4* x = reinterpret_cast<uint4*>(vs + pr_at<C::PITCH, C::HALF>(i, c));
            if (none) {
              *x = make_uint4(0, 0, 0, 0);  // values that may not be read: 0 * NaN would reach O
            } else if constexpr (!Q8) {
              const uint32_t e = F16 ? 0x7c00u : 0x7f80u;
              const uint32_t w[4] = {x->x, x->y, x->z, x->w};
#pragma unroll
              for (int k = 0; k < 4; ++k) bad |= (w[k] & e) == e || ((w[k] >> 16) & e) == e;
            }
          }
        }
        fence_proxy_async_shared();  // the ring slot is written by TMA next
        __syncwarp();
        if constexpr (!Q8) slow = __any_sync(0xffffffffu, bad);
      }
      // references: taken up for the rows that need it
      float top[2 * NT];
      bool need = false;
#pragma unroll
      for (int x = 0; x < 2 * NT; ++x) {
        float v = fmaxf(sc[0][x >> 1][x & 1], sc[0][x >> 1][2 + (x & 1)]);
#pragma unroll
        for (int i = 1; i < MK; ++i) v = fmaxf(v, fmaxf(sc[i][x >> 1][x & 1], sc[i][x >> 1][2 + (x & 1)]));
        top[x] = v;
        need |= v > m[x] + 6.0f;
      }
      if (__any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int x = 0; x < 2 * NT; ++x) {
          float v = top[x];
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          if (v > m[x] + 6.0f) {  // (for m = -inf as well)
            const float al = ex2(m[x] - v);
            m[x] = v;
            l[x] *= al;
#pragma unroll
            for (int mt = 0; mt < KT; ++mt) {
              o[mt][x >> 1][x & 1] *= al;
              o[mt][x >> 1][2 + (x & 1)] *= al;
            }
          }
        }
      }
      if constexpr (Q8) {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < MK; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) v = fmaxf(v, vsc[i][e] < INFINITY ? vsc[i][e] : 0.0f);  // (NaN: 0)
        if (__any_sync(0xffffffffu, v > 64.0f * vref)) {
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          const bool tiny = v < 1.2e-38f;  // such values are zero next to any output type's smallest step
          const float be = tiny ? 1.0f : __fdividef(vref, v);
          vinv = tiny ? 0.0f : __frcp_rn(v);
          vref = v;
#pragma unroll
          for (int mt = 0; mt < KT; ++mt)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[mt][j][e] *= be;
        }
      }
      uint32_t pb[MK][NT][2];
#pragma unroll
      for (int i = 0; i < MK; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float ref = m[2 * j + (e & 1)];
            p[e] = ex2(sc[i][j][e] - (ref == -INFINITY ? 0.0f : ref));
          }
          l[2 * j] += p[0] + p[2];
          l[2 * j + 1] += p[1] + p[3];
          if constexpr (Q8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] *= vsc[i][e >> 1] * vinv;
            if (!whole) {  // a key that is not seen has a scale that may be anything
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((hidden >> ((i * NT + j) * 4 + e)) & 1u) p[e] = 0.0f;
            }
          }
          pb[i][j][0] = movmatrix_t(MF16 ? pack2<__half>(p[0], p[1]) : pack_bf16(p[0], p[1]));
          pb[i][j][1] = movmatrix_t(MF16 ? pack2<__half>(p[2], p[3]) : pack_bf16(p[2], p[3]));
        }
      }
      const int mi = lane >> 3;
      if (!Q8 && slow) {
        // one product at a time: a weight of 0 leaves a value out that is not finite
#pragma unroll 1
        for (int kk = 0; kk < 16 * MK; ++kk) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // weight of (row 8 j + qc + e, key kk): in pb[kk / 16][j][kk / 8 % 2] of lane (qc + e) * 4 + kk % 8 / 2
              uint32_t w = 0;
#pragma unroll
              for (int x = 0; x < 2 * MK; ++x)
                if ((kk >> 3) == x) w = pb[x >> 1][j][x & 1];
              w = __shfl_sync(0xffffffffu, w, (qc + e) * 4 + ((kk & 7) >> 1));
              const uint32_t w16 = (kk & 1) ? w >> 16 : w & 0xffffu;
              const float p = F16 ? __half2float(__ushort_as_half((uint16_t)w16)) : __uint_as_float(w16 << 16);
#pragma unroll
              for (int mt = 0; mt < KT; ++mt)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  const int d = mt * 16 + qr + 8 * u;
                  const uint16_t vr = *reinterpret_cast<const uint16_t*>(vs + pr_at<C::PITCH, C::HALF>(kk, d >> 3) + (d & 7) * 2);
                  const float v = F16 ? __half2float(__ushort_as_half(vr)) : __uint_as_float((uint32_t)vr << 16);
                  if (p != 0.0f) o[mt][j][2 * u + e] += p * v;
                }
            }
        }
      } else {
#pragma unroll
        for (int i = 0; i < MK; ++i) {
          const uint32_t vbase = ex_smem_u32(vs) +
                                 (Q8 ? pr_at<C::PITCH, C::HALF>(16 * i + (mi & 1) * 8 + (lane & 7), mi >> 1)
                                     : pr_at<C::PITCH, C::HALF>(16 * i + (mi >> 1) * 8 + (lane & 7), mi & 1));
#pragma unroll
          for (int mt = 0; mt < KT; mt += (Q8 ? 2 : 1)) {
            const int c = Q8 ? mt : 2 * mt;
            uint32_t va[2][4], w[4];  // codes: keys 0-7 | 8-15 of a 16-byte chunk (16 dims), then of the next
            ldsm_x4_t((vbase ^ ((c & 7) << 4)) + (c >> 3) * C::HALF, w);
            if constexpr (Q8) {
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                transposed_to_f16<CODE>(w[2 * u], va[u][0], va[u][1]);
                transposed_to_f16<CODE>(w[2 * u + 1], va[u][2], va[u][3]);
              }
            } else {
#pragma unroll
              for (int x = 0; x < 4; ++x) va[0][x] = w[x];
            }
#pragma unroll
            for (int u = 0; u < (Q8 ? 2 : 1); ++u)
#pragma unroll
              for (int j = 0; j < NT; ++j) mma_16816<MF16>(o[mt + u][j], va[u], pb[i][j][0], pb[i][j][1]);
          }
        }
      }
      __syncwarp();
      if (++st == STAGES) st = 0, phase ^= 1;
      load_block();  // into the slot that was just read
    }
    if (!ok) break;
    const bool single = pr_segments(keys) == 1;
#pragma unroll
    for (int x = 0; x < 2 * NT; ++x) {
      float lx = l[x];
      lx += __shfl_xor_sync(0xffffffffu, lx, 4);
      lx += __shfl_xor_sync(0xffffffffu, lx, 8);
      lx += __shfl_xor_sync(0xffffffffu, lx, 16);
      const int c = (x >> 1) * 8 + qc + (x & 1);
      if (c >= R) continue;
      const int t = c / a.G, h = g * a.G + c % a.G;
      const float up = Q8 ? vref : 1.0f;
      // 16 dims a tile: codes 2 qr, 2 qr + 1; 16-bit qr, qr + 8
      if (single) {
        const float inv = lx > 0.0f ? up / lx : (lx == 0.0f ? 0.0f : lx);  // nothing seen: zeros; NaN stays NaN
        uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(first + t) * a.so_t + (int64_t)h * a.so_h;
#pragma unroll
        for (int mt = 0; mt < KT; ++mt) {
          const float u = o[mt][x >> 1][x & 1] * inv, v = o[mt][x >> 1][2 + (x & 1)] * inv;
          if constexpr (Q8) {
            *reinterpret_cast<uint32_t*>(dst + mt * 16 + 2 * qr) = a.q_is_f16 ? pack2<__half>(u, v) : pack_bf16(u, v);
          } else {
            ex_store_out<F16 ? EX_DTYPE_F16 : EX_DTYPE_BF16>(dst, mt * 16 + qr, u);
            ex_store_out<F16 ? EX_DTYPE_F16 : EX_DTYPE_BF16>(dst, mt * 16 + qr + 8, v);
          }
        }
      } else {
        const int64_t pi = ((int64_t)(first + t) * a.H + h) * a.NS + s;
        float* dst = a.ws_acc + pi * D;
#pragma unroll
        for (int mt = 0; mt < KT; ++mt) {
          const float u = o[mt][x >> 1][x & 1] * up, v = o[mt][x >> 1][2 + (x & 1)] * up;
          if constexpr (Q8) {
            *reinterpret_cast<float2*>(dst + mt * 16 + 2 * qr) = make_float2(u, v);
          } else {
            dst[mt * 16 + qr] = u;
            dst[mt * 16 + qr + 8] = v;
          }
        }
        if (qr == 0) {
          a.ws_m[pi] = m[x];
          a.ws_l[pi] = lx;
        }
      }
    }
  }
  // after a wait that ran out: the loads in flight land before the CTA ends (each slot's own last phase, bounded)
  if (!ok) {
    for (int i = 0; i < STAGES; ++i) mbar_wait(full_bar + (st + i) % STAGES, phase ^ (st + i >= STAGES ? 1u : 0u), EX_DEVERR_WAIT_TMA);
  }
}

// Segments of a row merged in order. D/2 threads a (token, query head), two numbers each: many loads in flight, and no
// shared memory, so that the grid is resident before the first kernel, which takes all of it, has ended.
template <int D, bool F16>
__global__ void __launch_bounds__(128) k_paged_rows_merge(const __grid_constant__ PrArgs a) {
  constexpr int WARPS = D / 64;  // of a row
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) / WARPS;
  const int lane = threadIdx.x & 31, d = ((threadIdx.x >> 5) % WARPS * 32 + lane) * 2;
  if (row >= a.tokens * a.H) return;
  const int64_t tok = row / a.H;
  const int h = (int)(row % a.H);
  int b = (int)tok;
  if (a.qsl) {
    b = find_sequence(a.qsl, a.n, tok);
    if (b >= a.n || tok < a.qsl[0]) return;
  }
  int first, T, L;
  pr_request(a, b, first, T, L);
  const int ns = pr_segments(pr_keys(a, L));
  if (T == 0 || ns == 1) return;  // untouched, or written by the first kernel
  const float* pm = a.ws_m + row * a.NS;
  const float* pl = a.ws_l + row * a.NS;
  const float* src = a.ws_acc + row * a.NS * D + d;
  float m = -INFINITY, l = 0.0f, x = 0.0f, y = 0.0f;
  for (int s0 = 0; s0 < ns; s0 += 32) {  // 32 segments at a time: their factors first, a segment a lane
    const bool have = s0 + lane < ns;
    const float ms = have ? pm[s0 + lane] : -INFINITY, ls = have ? pl[s0 + lane] : 0.0f;
    float mn = ms;
#pragma unroll
    for (int o = 16; o; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mn = fmaxf(mn, m);
    const float sub = mn == -INFINITY ? 0.0f : mn;
    const float c = ex2(ms - sub), old = ex2(m - sub);
    m = mn;
    l *= old;
    x *= old;
    y *= old;
    const int cnt = min(32, ns - s0);
#pragma unroll 16
    for (int s = 0; s < cnt; ++s) {
      const float cs = __shfl_sync(0xffffffffu, c, s);
      l += __shfl_sync(0xffffffffu, ls, s) * cs;
      const float2 v = *reinterpret_cast<const float2*>(src + (int64_t)(s0 + s) * D);
      x += v.x * cs;
      y += v.y * cs;
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
  *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + tok * a.so_t + (int64_t)h * a.so_h + d) =
      F16 ? pack2<__half>(x * inv, y * inv) : pack_bf16(x * inv, y * inv);
}

}  // namespace ex
