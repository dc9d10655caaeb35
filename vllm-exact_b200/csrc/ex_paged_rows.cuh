// Attention of a few query rows per sequence over a paged cache: one token over an 8-bit cache (paged_decode_q8), or
// up to 64 drafted tokens under an ancestor mask over a 16-bit or 8-bit cache (tree_attention).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - m),  x_j = (q . k_j) scale log2 e,  m the largest x_j so far
//
// The rows of a KV head are the (token, query head) pairs of its group, token-major. Keys are taken in segments whose
// length depends on the request's own length only, and segments are merged in order:
// a row's bits do not depend on the other requests, the other rows, or where pages lie.
//
// Work: items (request, segment, KV head, tile of rows), numbered by walking the requests' lengths on the device (no host
// sync), dealt out in turn: neighbouring items share keys' pages. Requests of at most 16 rows a KV head are k_paged_few's,
// the others k_tree_tc's (ex_tree_tc.cuh), by their own number of rows.
//
// 8-bit codes become float16 (exact). The key scale multiplies the score; the value scale goes into P: P is p_j vs_j over a
// reference of the row's own, the largest p_j vs_j of the keys that it sees so far. So float16 P keeps 11 bits of every product
// that counts, and what a hidden key or one of next to no weight has for a value scale is nothing to the row. (A finite
// weight under 2^-126 of the largest is 0, as float32's normal numbers end there: with values 2^122 times the others' even such a
// one would count.)
//
// P is rounded to the 16 bits of V (codes: to float16), since one product takes both in one type: half a step, 2^-8 of a weight
// over bf16, 2^-11 over float16 and codes, with sums of unrounded weights below it. ex_paged_decode holds P as two bf16 numbers,
// which costs a second product for V: its results are the finer ones, and other bits than these.
// Queries are brought to float16 by a power of two per row, exact for all elements above 2^-14 of the row's largest.
#pragma once
#include "ex_cache_q8.cuh"
#include "ex_paged_decode.cuh"
#include "ex_paged_decode_tma.cuh"

namespace ex {

constexpr int PR_MAX_TOKENS = 64;  // drafted tokens of a request (bits of a mask word)
constexpr float PR_LOG2E = 1.4426950408889634f;

// Keys a segment, by the request's own length alone: the order of its sums must not depend on the batch. Short segments spread
// a request over more SMs; every segment costs its partial results' traffic, and with many rows a CTA's start and end.
// At most 16 rows a KV head: 256 up to 2048 keys (256 requests of 1024 keys, e4m3: 120 us; 128: 131; 64: 160; one request of
// 1000 keys: 19, 16, 16 us), 512 behind (16 requests of 16384 keys, int8: 130 us; 256: 142; 1024: 136; one such request:
// 31, 31, 44 us).
__host__ __device__ inline int pr_segment(int64_t L) { return L <= 2048 ? 256 : 512; }
// More rows: 512 up to 2048 keys, behind them equal quarters of the request in whole blocks of 128 keys, of at least 2048 and at
// most 4096. Long segments cost a batch least, short ones spread a single request. 32 heads over 8 of 128, 16 tokens,
// bf16 | e4m3, microseconds with segments of 512, 1024, 2048, 4096 keys:
//   one request of  2500 keys   25   27   36   43 |  29   33   48   55      64 of 8192   729  532  458  411 | 973  709  577  504
//                   4096        24   28   37   56 |  30   36   49   72      32 of 3000   171  141  137  127 | 216  174  162  139
//                   16384       49   37   46   63 |  55   42   54   78      4 of 16384   121   99   82   67 | 150  118   98   83
//                   65536      155  116   89   71 | 178  133  104   86
__host__ __device__ inline int pr_segment_many(int64_t L) {
  const int quarter = L < 16384 ? (int)((L + 511) >> 9) << 7 : 4096;
  return L <= 2048 ? 512 : quarter < 2048 ? 2048 : quarter;
}
__host__ __device__ inline int pr_segments(int64_t L) {
  const int s = pr_segment(L), n = (int)((L + s - 1) / s);
  return n < 1 ? 1 : n;
}
__host__ __device__ inline int pr_segments_many(int64_t L) {
  const int s = pr_segment_many(L), n = (int)((L + s - 1) / s);
  return n < 1 ? 1 : n;
}
constexpr int PR_FEW = 16;  // rows a KV head
// most segments of any request of at most max_len keys
__host__ inline int pr_max_segments(int64_t max_len) {
  const int a = pr_segments(max_len < 2048 ? max_len : 2048), b = pr_segments(max_len);
  return a > b ? a : b;
}

// a block of keys in shared memory, as TMA writes it
template <int D, int CODE, int BLK>
struct PrTile {
  static constexpr int ESZ = CODE == CODE_NONE ? 2 : 1;
  static constexpr int ROW = D * ESZ;                  // bytes of a key
  static constexpr int PITCH = ROW < 128 ? ROW : 128;  // bytes of a row of a TMA box
  static constexpr int NH = ROW / PITCH;               // boxes across the head dimension
  static constexpr int HALF = BLK * PITCH;
  static constexpr int TILE = BLK * ROW;               // K or V
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
  uint32_t g_inv;            // ceil(2^16 / G): x / G is x g_inv >> 16 for x < 4096 (G <= 16)
  int rows_lo, rows_hi;      // requests with rows_lo < T G <= rows_hi are this kernel's
  const void* v;             // the values as the tensor map reads them, for those that are not finite
  int64_t sv_block, sv_page, sv_head;
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
template <bool MANY>
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
          cnt = (MANY ? pr_segments_many(pr_keys(a, L)) : pr_segments(pr_keys(a, L))) * a.KV * ((T * a.G + rows_per_tile - 1) / rows_per_tile);
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

__device__ __forceinline__ float lg2(float x) {  // (-infinity for what is below the normal numbers)
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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


// 1 / f and f = 2^e with m in [f, 2f): what a row with largest element m is divided by on its way to float16. Exponents
// are kept where both are normal numbers.
__device__ __forceinline__ float pr_query_scale(float m, float& f) {
  int e = (int)((__float_as_uint(m) >> 23) & 255u);
  e = e == 255 ? 127 : min(max(e, 2), 252);
  f = __uint_as_float((uint32_t)e << 23);
  return __uint_as_float((uint32_t)(254 - e) << 23);
}

// Two 16-bit values or four codes in a word: a bit (15, 31; e4m3 7, 15, 23, 31) for each that is not finite. One more than the
// largest exponent (e4m3: than the NaN code, which is all ones) carries into the place of the sign, and no further.
template <int CODE, bool F16>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if constexpr (CODE == CODE_E4M3) return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  return ((w & (F16 ? 0x7c007c00u : 0x7f807f80u)) + (F16 ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}
template <int CODE, bool F16>
__device__ __forceinline__ uint32_t only_finite(uint32_t w) {  // zeros for the others
  const uint32_t n = not_finite<CODE, F16>(w);
  return w & ~(CODE == CODE_E4M3 ? (n >> 7) * 0xffu : (n >> 15) * 0xffffu);
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

// ------------------------------------------------------------------------------------------------------------------
// At most 16 rows of a KV head: a decode step, or a few drafted tokens.
//
// Every warp streams its own items: it loads blocks of 16 MK keys into its own ring, S blocks ahead and on into its next
// item, and computes S^T = K Q^T, P and O^T += V^T P^T on what has arrived. No thread waits for another warp. References are taken
// up only when a score (16-bit) or a weight times its value scale (codes) is more than 64 times them (p stays small enough
// for float16): the common path has one vote and no shuffles. It is decided for every row alone.
// Near the cache's bytes where there are many requests (64 of 8192 keys, int8: 207 us, 5.3 TB/s of 6.56 measured; 256 of
// 768 to 1280, e4m3: 121 us, 4.6 TB/s; 16-bit, 4 tokens: 381 us, 5.6 TB/s). No unit is full (64 of 4096, e4m3: DRAM 80 % of a
// copy, issue slots 40 %, products 16 %): three warps a scheduler wait on their own chains of load, product, weights, product.
// One request of 1000 keys takes 19 us: two launches, and four blocks a warp one after another.
// ------------------------------------------------------------------------------------------------------------------
template <int D, int CODE, int NT>
struct PfCfg {
  static constexpr int ROW = (CODE == CODE_NONE ? 2 : 1) * D;  // bytes of a key
  // 16-key tiles of a block: two where the registers have room for them (256 requests of 1024 keys, e4m3: 119 us, with one 133)
  static constexpr int MK = ROW <= 128 ? 2 : 1;
  // Warps of a CTA, one CTA per SM: as many as rings of enough blocks fit in shared memory and results in registers. At most 8
  // rows (NT = 1): the same batch with 12 warps 119 us, 8 124, 4 186; 64 requests of 8192 keys, D = 256: 8 warps 207 us, 4
  // 294. 16 rows: codes of D = 128 do not fit the registers of 12 warps (64 requests of 8192 keys, e4m3, 4 tokens: 8 warps
  // 248 us, 10 311, 12 302), of D = 64 they do (8 warps 196 us, 12 164); D = 256: 8 warps 296 us, 6 367 (some spills in both).
  static constexpr int NW = ROW > 256 ? 4 : ROW > 128 || (NT == 2 && CODE != CODE_NONE && D == 128) ? 8 : 12;
  static constexpr int BLK = 16 * MK;
  using R = PrTile<D, CODE, BLK>;
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
  PrWalk<false> lwalk;
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
  PrWalk<false> walk;
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
    float vtop[2 * NT];  // codes: O is the sum of 2^(x - vtop) vs c
    bool apart = false;  // of some row m and vtop differ
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
      vtop[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.0f;

    bool noted = false;
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
      uint32_t hidden = 0;  // bit ((i NT + j) 4 + e): the row does not see the key
      if (!whole) {
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
            } else if constexpr (CODE != CODE_INT8) {
              // values that are not finite and that some row may not see: taken out, and in the end added to the rows that do
              if (not_finite<CODE, F16>(x->x) | not_finite<CODE, F16>(x->y) | not_finite<CODE, F16>(x->z) | not_finite<CODE, F16>(x->w)) {
                *x = make_uint4(only_finite<CODE, F16>(x->x), only_finite<CODE, F16>(x->y), only_finite<CODE, F16>(x->z), only_finite<CODE, F16>(x->w));
                noted = true;
              }
            }
          }
        }
        fence_proxy_async_shared();  // the ring slot is written by TMA next
        __syncwarp();
      }
      // references: taken up for the rows that need it. No product of a lane passes its largest score with its largest value
      // scale (but for roundings, hence 5.9): so one vote decides for scores and products, before a weight is made. Which other
      // rows of the warp need it makes no difference to a row.
      float top[2 * NT], lv = -INFINITY;
      bool need = false;
      if constexpr (Q8) {
        float v = fmaxf(vsc[0][0], vsc[0][1]);  // (NaN: left out)
#pragma unroll
        for (int i = 1; i < MK; ++i) v = fmaxf(v, fmaxf(vsc[i][0], vsc[i][1]));
        lv = lg2(v);
      }
#pragma unroll
      for (int x = 0; x < 2 * NT; ++x) {
        float v = fmaxf(sc[0][x >> 1][x & 1], sc[0][x >> 1][2 + (x & 1)]);
#pragma unroll
        for (int i = 1; i < MK; ++i) v = fmaxf(v, fmaxf(sc[i][x >> 1][x & 1], sc[i][x >> 1][2 + (x & 1)]));
        top[x] = v;
        need |= Q8 ? v > m[x] + 60.0f || v + lv > vtop[x] + 5.9f : v > m[x] + 6.0f;
      }
      if (__any_sync(0xffffffffu, need)) {
        float be[2 * NT];  // what O is scaled by
        bool some = false, differ = false;
#pragma unroll
        for (int x = 0; x < 2 * NT; ++x) {
          float v = top[x], vb = -INFINITY;  // the row's largest score, and the largest with the value scale in it
          if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < MK; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) vb = fmaxf(vb, sc[i][x >> 1][2 * e + (x & 1)] + lg2(vsc[i][e]));
          }
#pragma unroll
          for (int d = 4; d <= 16; d <<= 1) {
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
            if constexpr (Q8) vb = fmaxf(vb, __shfl_xor_sync(0xffffffffu, vb, d));
          }
          be[x] = 1.0f;
          if constexpr (Q8) {
            if (v > m[x] + 60.0f || vb > vtop[x] + 6.0f) {  // (the row's own: what other rows need does not matter)
              // Weights are over the products' reference, so that these need no factor, as long as that is not above the largest
              // score and at most 60 below it (weights and their sum stay far from the largest numbers). The products' is at
              // least 126 below it: what they lose then (2^-25 times 2^-126 times a code) is below bf16's smallest step.
              const float most = fmaxf(v, m[x]), high = vb > vtop[x] + 6.0f ? vb : vtop[x];
              const float mn = fmaxf(m[x], fminf(fmaxf(high, most - 60.0f), most)), to = fmaxf(high, mn - 66.0f);
              l[x] *= ex2(m[x] - mn);
              m[x] = mn;
              be[x] = ex2(vtop[x] - to);
              vtop[x] = to;
            }
            differ |= m[x] != vtop[x];
          } else if (v > m[x] + 6.0f) {  // (for m = -inf as well)
            be[x] = ex2(m[x] - v);
            m[x] = v;
            l[x] *= be[x];
          }
          some |= be[x] != 1.0f;
        }
        if constexpr (Q8) apart = __any_sync(0xffffffffu, differ);
        if (kb > start && __any_sync(0xffffffffu, some)) {  // (the first block's O is 0)
#pragma unroll
          for (int x = 0; x < 2 * NT; ++x)
#pragma unroll
            for (int mt = 0; mt < KT; ++mt) {
              o[mt][x >> 1][x & 1] *= be[x];
              o[mt][x >> 1][2 + (x & 1)] *= be[x];
            }
        }
      }
      // weights; for codes times the keys' value scales (of a key that is not seen it may be anything)
#pragma unroll
      for (int i = 0; i < MK; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float ref = m[2 * j + (e & 1)];
            sc[i][j][e] = ex2(sc[i][j][e] - (ref == -INFINITY ? 0.0f : ref));
          }
          l[2 * j] += sc[i][j][0] + sc[i][j][2];
          l[2 * j + 1] += sc[i][j][1] + sc[i][j][3];
          if constexpr (Q8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[i][j][e] *= vsc[i][e >> 1];
            if (!whole) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((hidden >> ((i * NT + j) * 4 + e)) & 1u) sc[i][j][e] = 0.0f;
            }
          }
        }
      if (Q8 && apart) {
#pragma unroll
        for (int x = 0; x < 2 * NT; ++x) {
          const float half = ex2(0.5f * (m[x] - vtop[x])), f = m[x] == vtop[x] ? 1.0f : half * half;  // (may be below the normal numbers)
#pragma unroll
          for (int i = 0; i < MK; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) sc[i][x >> 1][2 * e + (x & 1)] *= f;
        }
      }
      uint32_t pb[MK][NT][2];
#pragma unroll
      for (int i = 0; i < MK; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          pb[i][j][0] = movmatrix_t(MF16 ? pack2<__half>(sc[i][j][0], sc[i][j][1]) : pack_bf16(sc[i][j][0], sc[i][j][1]));
          pb[i][j][1] = movmatrix_t(MF16 ? pack2<__half>(sc[i][j][2], sc[i][j][3]) : pack_bf16(sc[i][j][2], sc[i][j][3]));
        }
      const int mi = lane >> 3;
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
      __syncwarp();
      if (++st == STAGES) st = 0, phase ^= 1;
      load_block();  // into the slot that was just read
    }
    if (!ok) break;
    if (CODE != CODE_INT8 && __any_sync(0xffffffffu, noted)) {
      // Values that are not finite: added as they are (their weight is positive, however small) to the rows that see them; what
      // blocks that are seen whole have made of them stays. Dims of a lane: 16-bit qr, qr + 8 of every 16, codes 2 qr, 2 qr + 1.
#pragma unroll 1
      for (int key = start; key < end; ++key) {
        const int pg = a.bt[(int64_t)b * a.sbt + key / a.BS], d = key - ctx;
        if (pg < 0 || pg >= a.blocks) continue;
        const int64_t at = (int64_t)pg * a.sv_block + (int64_t)(key % a.BS) * a.sv_page + (int64_t)g * a.sv_head;
#pragma unroll
        for (int mt = 0; mt < KT; ++mt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float v;
            if constexpr (Q8) {
              v = (reinterpret_cast<const uint8_t*>(a.v)[at + mt * 16 + 2 * qr + u] & 0x7f) == 0x7f ? NAN : 0.0f;
            } else {
              const uint16_t w = reinterpret_cast<const uint16_t*>(a.v)[at + mt * 16 + qr + 8 * u];
              v = F16 ? __half2float(__ushort_as_half(w)) : __uint_as_float((uint32_t)w << 16);
            }
            if (fabsf(v) < INFINITY) continue;
#pragma unroll
            for (int x = 0; x < 2 * NT; ++x) {
              const int r = (x >> 1) * 8 + qc + (x & 1), t = r / a.G;
              if (r >= R) continue;
              if (d >= 0 && !(((a.mask ? a.mask[first + t] : (t >= 63 ? ~0ull : (2ull << t) - 1ull)) >> d) & 1ull)) continue;
              o[mt][x >> 1][2 * u + (x & 1)] += v;
            }
          }
      }
    }
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
      const float half = ex2(0.5f * (vtop[x] - m[x])), up = !Q8 || vtop[x] == m[x] ? 1.0f : half * half;
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
  const int ns = T * a.G > PR_FEW ? pr_segments_many(pr_keys(a, L)) : pr_segments(pr_keys(a, L));
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
