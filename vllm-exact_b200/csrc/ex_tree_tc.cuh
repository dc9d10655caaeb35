// Attention of many query rows per KV head (more than 16: drafted tokens times grouped heads) over a 16-bit or 8-bit
// paged cache, on tcgen05. The mathematics and the masks are those of ex_paged_rows.cuh. Over codes m and the products' reference
// are both kept: P is 2^(x - m) vs 2^(m - vtop), so that a key's weight is made once for the sum and the product.
//
// One CTA per SM takes items (request, segment of its keys, KV head, tile of 128 rows) and walks the segment in blocks
// of 128 keys: S = Q K^T with both operands in shared memory, O += P V with P in tensor memory over the S it came
// from. D <= 128: blocks alternate between two streams, each with its own S, O, m and l and its own four softmax warps, so
// that one stream's softmax runs beside the other's products; the streams are added up at the end of the segment.
// D = 256: one O, two S buffers.
//   warps 0-3, 4-7  softmax (they also bring Q to shared memory and write the results). A thread has one row of the tile and,
//                   where the request has at most 64 (32) rows, 64 (32) of the block's keys: Q is then there two (four)
//                   times, every copy weighs its own keys and has zeros for the others, and the copies are added up
//                   at the end. A row's exponentials are what takes longest, and this spreads them over all schedulers.
//   warp 8          issues the products
//   warps 12-15, for codes 9-11   producers: TMA boxes of 8 or 16 tokens through the block table into a ring of slots. Issuing
//                   a box takes a warp about 75 cycles (its operands are uniform registers), 16 boxes of a 32 KB tile longer
//                   than HBM takes to deliver it: so several warps share the boxes of every tile.
//   warps 10, 11    16-bit: blocks with drafted tokens or the request's end; values behind the end are zeroed, values that
//                   are not finite are zeroed and noted, and added in the end to the rows that see them
//   warps 12-15     for codes: codes to float16 tiles (exact; values behind the end to zeros, and in blocks with drafted tokens or
//                   the end codes that are NaN, noted as 10 and 11 do)
// 16-bit: bound by reading the cache once (a block of 128 keys is 64 KB for D = 128, 1.5 us of an SM's share of HBM) and by an
// item's start and end, when only as much is read as the ring holds (of 45000 cycles for 2048 keys 13000 by clock readings in
// the kernel: queries 600, first scores 1400, last products 3000, results 8000). 64 requests of 6144 to 10240 keys, 16 tokens:
// 465 us, 4.6 TB/s, at 1965 MHz; 531 us called for seconds, when the power limit leaves 1650 MHz.
// Codes: no unit is full (counters of 16 requests of 16384 keys, 7 tokens: shared memory's pipe 53 % with the products' reads,
// issue slots 45 %, products 32 %, DRAM 36 % of a copy); it is each block's chain of load, conversion, product, softmax. Four
// converter warps more change nothing. 16 requests of 12288 to 20480 keys, 7 tokens: 240 us, 2.3 TB/s.
//
// P has the 16 bits of V (codes: float16), as in ex_paged_rows.cuh: one rounding of half a step, 2^-8 of a weight over bf16.
#pragma once
#include "ex_paged_rows.cuh"
#include "ex_prompt_attn.cuh"
#include "ex_tree_ring.h"

namespace ex {

template <int D, int CODE>
struct PtcCfg {
  static constexpr bool Q8 = CODE != CODE_NONE;
  static constexpr int STREAMS = D == 256 ? 1 : 2;
  static constexpr int THREADS = 512;
  static constexpr int FEEDERS = ptc_feeders(Q8);    // producer warps
  static constexpr int LOADED = ptc_loaded_count(Q8);  // arrivals on a loaded tile
  // registers a thread: at launch, of the softmax warps and of the others, which give theirs up
  static constexpr int REGS = 128, REGS_SOFTMAX = 168, REGS_OTHER = 88;
  static_assert(256 * REGS_SOFTMAX + (THREADS - 256) * REGS_OTHER <= THREADS * REGS, "register shares");
  static constexpr int SW = D < 128 ? D : 128;       // dims of a 16-bit slot
  static constexpr int PARTS = D / SW;               // slots of a block's K or V
  static constexpr int SUB = 128 * 128;              // 128 rows x 64 dims of 16 bits, one swizzled column
  static constexpr int SLOT = SW / 64 * SUB;
  static constexpr int Q_BYTES = (D / 64) * SUB;
  static constexpr int RAW = Q8 ? 128 * SW : 0;      // bytes of a slot of codes: 128 keys, SW dims
  static constexpr int SLOTS = D == 64 ? (Q8 ? 6 : 8) : (Q8 ? 3 : 5);
  static constexpr int RAWS = !Q8 ? 0 : D == 64 ? 6 : D == 128 ? 5 : 3;  // slots of codes
  // Blocks whose scales and pages are kept. While block j's weights are made, its values are the first tile not used up:
  // number 2 j + 2 in the order K0 K1 V0 K2 V1 .. of loading. The rings hold SLOTS + RAWS more, keys of block m being number
  // 2 m - 1: m < j + 8 as long as they are at most 13.
  static constexpr int SCALE_BLOCKS = 8;
  static_assert((SLOTS + RAWS) / PARTS <= 13, "blocks ahead");
  static constexpr int SMEM = 1024 + Q_BYTES + SLOTS * SLOT + RAWS * RAW + (Q8 ? SCALE_BLOCKS * 1024 + 512 : 0) + 768;
  static_assert(SMEM <= 232448, "shared memory of a CTA");
};

// N (a multiple of 32) columns of a row's scores, scaled by the keys' scales where they have some.
template <bool Q8, int N>
__device__ __forceinline__ void ptc_scores(uint32_t s_addr, const float* ks, float (&x)[N]) {
#pragma unroll
  for (int c = 0; c < N; c += 32) tmem_ld32(s_addr + c, reinterpret_cast<uint32_t*>(x) + c);
  tmem_ld_wait();
  if constexpr (Q8) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 k = *reinterpret_cast<const float4*>(ks + i);
      x[i] *= k.x;
      x[i + 1] *= k.y;
      x[i + 2] *= k.z;
      x[i + 3] *= k.w;
    }
  }
}
template <int N>
__device__ __forceinline__ float ptc_max(const float (&x)[N]) {
  float m[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int i = 4; i < N; ++i) m[i & 3] = fmaxf(m[i & 3], x[i]);
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// The largest x fac + log2 of the value scale: what a row's reference has to reach. (NaN, and keys that are not seen: left out.)
template <int N>
__device__ __forceinline__ float ptc_high(const float (&x)[N], const float* vs, float fac) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, __fmaf_rn(x[i], fac, __log2f(vs[i])));
  return m;
}
// Their weights 2^(x fac - sub) in 16 bits to tensor memory at p_addr (over scores that have been read); returns the weights'
// sum. Codes: times the values' scales over the row's reference (the scale times the weight first: neither that over the
// reference nor the scale over it need be a number).
template <bool Q8, bool MF16, int N>
__device__ __forceinline__ float ptc_weights(uint32_t p_addr, const float* vs, float fac, float sub, float vinv, float (&x)[N]) {
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int c = 0; c < N; c += 32) {
    uint32_t p[16];
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      float w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[k] = ex2(__fmaf_rn(x[c + i + k], fac, -sub));
        sum[k] += w[k];
      }
      if constexpr (Q8) {
        const float4 v = *reinterpret_cast<const float4*>(vs + c + i);
        w[0] = w[0] * v.x * vinv;
        w[1] = w[1] * v.y * vinv;
        w[2] = w[2] * v.z * vinv;
        w[3] = w[3] * v.w * vinv;
      }
      p[i / 2] = MF16 ? pack2<__half>(w[0], w[1]) : pack_bf16(w[0], w[1]);
      p[i / 2 + 1] = MF16 ? pack2<__half>(w[2], w[3]) : pack_bf16(w[2], w[3]);
    }
    tmem_st16(p_addr + c / 2, p);
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// 16-bit values of the context that are not finite, where a row stands in the tile more than once: a copy's weights of 0 for
// the other copies' keys have made NaN of them. The first `keys` keys from `start` on, which every row sees (values of edge
// blocks have been taken out), are looked at again: an element of the 16 in o that is not finite because of them becomes the
// sum of the copy's own, those of columns col .. col + W of a block.
template <bool F16>
__device__ __noinline__ void ptc_context_infinities(float* o, const int32_t* pages, int BS, int64_t blocks, const uint16_t* values,
                                                    int64_t s_block, int64_t s_page, int start, int keys, int col, int W) {
  float own[16] = {};
  uint32_t others = 0;
#pragma unroll 1
  for (int x = 0; x < keys; ++x) {
    const int key = start + x, page = pages[key / BS];
    if (page < 0 || page >= blocks) continue;
    const uint4* e = reinterpret_cast<const uint4*>(values + (int64_t)page * s_block + (int64_t)(key % BS) * s_page);
    const uint4 lo = e[0], hi = e[1];
    const uint32_t z[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    uint32_t some = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) some |= not_finite<CODE_NONE, F16>(z[i]);
    if (some == 0) continue;
    const bool mine = (x & 127) >= col && (x & 127) < col + W;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint16_t h = (uint16_t)(z[i >> 1] >> (16 * (i & 1)));
      const float y = F16 ? __half2float(__ushort_as_half(h)) : __uint_as_float((uint32_t)h << 16);
      if (!(fabsf(y) < INFINITY)) {
        if (mine) own[i] += y;
        else others |= 1u << i;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (!(fabsf(o[i]) < INFINITY) && (own[i] != 0.0f || ((others >> i) & 1u))) o[i] = own[i];
}

constexpr int PTC_EDGES = 8;   // edge blocks in flight: each takes a slot of the ring
constexpr int PTC_POISON = 8;  // items with edge blocks whose notes of values that are not finite are kept (the rings, of at most 8
                               // tiles or of 6 behind the conversion, and two or more an item, run ahead of the rows, which clear
                               // the notes that they have read)

template <int D, int CODE, bool F16>
__global__ void __launch_bounds__((PtcCfg<D, CODE>::THREADS), 1)
    k_tree_tc(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
              const __grid_constant__ PrArgs a) {
  using C = PtcCfg<D, CODE>;
  constexpr bool Q8 = C::Q8;
  constexpr bool MF16 = Q8 || F16;
  constexpr bool NOTES = CODE != CODE_INT8;  // some values may not be finite
  constexpr int ESZ = Q8 ? 1 : 2;
  constexpr int TM_S = 0, TM_O = 256;
  constexpr int CD = D == 64 ? 16 : 32;  // dims of a piece of the results: two pieces of 128 rows fit where Q was
  extern __shared__ uint8_t pr_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pr_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + C::Q_BYTES;
  uint8_t* raw = ring + C::SLOTS * C::SLOT;
  float* sscale = reinterpret_cast<float*>(raw + C::RAWS * C::RAW);  // [SCALE_BLOCKS][128 of keys, 128 of values]
  float* sfac = sscale + (Q8 ? C::SCALE_BLOCKS * 256 : 0);          // [128] 8-bit: score factors of the rows
  uint64_t* bar = reinterpret_cast<uint64_t*>(sfac + (Q8 ? 128 : 0));
  uint64_t* full_bar = bar;             // [8] 16-bit slots
  uint64_t* empty_bar = bar + 8;        // [8]
  uint64_t* rfull_bar = bar + 16;       // [8] slots of codes
  uint64_t* rempty_bar = bar + 24;      // [8]
  uint64_t* s_bar = bar + 32;           // [2]
  uint64_t* p_bar = bar + 34;           // [2]
  uint64_t* q_bar = bar + 36;
  uint64_t* o_bar = bar + 37;
  uint64_t* end_bar = bar + 38;
  uint64_t* done_bar = bar + 39;
  uint64_t* ask_bar = bar + 40;         // [PTC_EDGES] by number of the edge block: its values' loads have been issued
  uint64_t* fix_bar = bar + 48;         // [PTC_EDGES] they have been looked at
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 56);
  volatile int* sfail = reinterpret_cast<int*>(tmem_slot + 1);  // a wait of the softmax warps ran out
  uint32_t* sgood = tmem_slot + 3;      // [8] by block: groups whose page exists
  uint32_t* poison = sgood + 8;         // [PTC_POISON][8]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  if (tid == 0) {
    *sfail = 0;
    for (int i = 0; i < PTC_POISON * 8; ++i) poison[i] = 0;
    for (int i = 0; i < 8; ++i) {
      mbar_init(full_bar + i, Q8 ? 128 : C::LOADED);
      mbar_init(empty_bar + i, 1);
      mbar_init(rfull_bar + i, C::LOADED);
      mbar_init(rempty_bar + i, 128);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_bar + i, 1);
      mbar_init(p_bar + i, 128);
    }
    for (int i = 0; i < PTC_EDGES; ++i) {
      mbar_init(ask_bar + i, C::FEEDERS);
      mbar_init(fix_bar + i, 64);
    }
    mbar_init(done_bar, 1);
    mbar_init(q_bar, 256);
    mbar_init(o_bar, 1);
    mbar_init(end_bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  PrWalk<true> walk;
  // item `it`: everything the roles need; false: no such item
  int it = blockIdx.x, b, first, T, L, g, s, row0, R, start, end, ctx, nblk, jedge;
  auto next = [&]() {
    int rem;
    if (!walk.find(a, 128, it, b, first, T, L, rem)) return false;
    it += gridDim.x;
    R = T * a.G;
    const int tiles = (R + 127) / 128;
    row0 = rem % tiles * 128;
    g = rem / tiles % a.KV;
    s = rem / (tiles * a.KV);
    const int keys = pr_keys(a, L), seg = pr_segment_many(keys);
    start = s * seg;
    end = min(keys, start + seg);
    ctx = L - T;
    nblk = max(0, end - start + 127) >> 7;
    jedge = min(max(min(ctx, end) - start, 0) >> 7, nblk);  // blocks before it are seen by every row
    return true;
  };

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_OTHER));
  constexpr int FEED0 = Q8 ? 9 : 12;
  if (warp >= FEED0 && warp < FEED0 + C::FEEDERS) {
    // ------------------------------------------------------------------------------------------------ producers
    // Every producer follows all groups; it issues those of its own, the first one also announces each tile.
    const int feeder = warp - FEED0;
    const int group = 1 << a.group_log2, per = 128 >> a.group_log2;
    int slot = 0, made = 0;
    uint32_t ph = 1, blocks = 0, edges = 0;  // blocks, edge blocks of all items so far
    uint64_t* fulls = Q8 ? rfull_bar : full_bar;
    uint64_t* empties = Q8 ? rempty_bar : empty_bar;
    constexpr int SLOTS = Q8 ? C::RAWS : C::SLOTS;
    constexpr int PITCH = C::SW * ESZ < 128 ? C::SW * ESZ : 128;  // bytes of a box row
    constexpr int NB = C::SW * ESZ / PITCH;
    bool ok = true;
    while (ok && next()) {
      // where the groups lie: a window of 32 groups, a group a lane, and the next one looked up ahead
      int wpage = -1, woff = 0, npage = -1, noff = 0;
      auto look = [&](int key, int& page, int& off) {
        page = -1;
        if (key < end) {
          const int i = key / a.BS;
          page = a.bt[(int64_t)b * a.sbt + i];
          off = key - i * a.BS;
        }
      };
      // keys are loaded a block ahead of values: pages (lane: group) of the block whose keys were last loaded, and the one before
      int page[2] = {-1, -1}, off[2] = {0, 0};
      int key = start + lane * group;  // of the next look-up
#pragma unroll 1
      for (int n = 0; n < 2 * nblk && ok; ++n) {
        int j;
        const bool is_v = ptc_tile(n, nblk, j);
        if (!is_v) {
          const int at = (j * per) & 31;  // the block's first group in the window
          if (at == 0) {
            if (n == 0) {
              look(key, npage, noff);
              key += 32 * group;
            }
            wpage = npage;
            woff = noff;
            look(key, npage, noff);
            key += 32 * group;
          }
          page[0] = page[1];
          off[0] = off[1];
          page[1] = __shfl_sync(0xffffffffu, wpage, (at + lane) & 31);
          off[1] = __shfl_sync(0xffffffffu, woff, (at + lane) & 31);
          if (lane >= per) page[1] = -1;
        }
        const bool before = is_v && j < nblk - 1;  // (the last block's values follow its own keys)
        const int pg = before ? page[0] : page[1], po = before ? off[0] : off[1];
        const uint32_t there = __ballot_sync(0xffffffffu, lane < per && start + (j * per + lane) * group < end);
        const uint32_t good = __ballot_sync(0xffffffffu, pg >= 0 && pg < a.blocks) & there;
#pragma unroll 1
        for (int p = 0; p < C::PARTS; ++p) {
          ok = mbar_wait_idle(empties + slot, ph, EX_DEVERR_WAIT_SLOT);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          uint8_t* dst = Q8 ? raw + slot * C::RAW : ring + slot * C::SLOT;
          if (feeder == 0) {
            if (good != there) {  // tokens on pages that do not exist: zeros
#pragma unroll 1
              for (int i = 0; i < per; ++i) {
                if (!((there & ~good) >> i & 1)) continue;
#pragma unroll 1
                for (int c = lane; c < NB * group * PITCH / 16; c += 32) {
                  const int h = c / (group * PITCH / 16), x = c % (group * PITCH / 16);
                  *reinterpret_cast<uint4*>(dst + h * 128 * PITCH + i * group * PITCH + x * 16) = make_uint4(0, 0, 0, 0);
                }
              }
              fence_proxy_async_shared();
              __syncwarp();
            }
            if (lane == 0) {
              if (!is_v) sgood[(blocks + j) & 7] = good;
              mbar_arrive_expect_tx(fulls + slot, (uint32_t)(__popc(good) * group * C::SW * ESZ));
            }
          }
          if (((good >> lane) & 1u) && lane % C::FEEDERS == feeder) {
            const CUtensorMap* m = is_v ? &tm_v : &tm_k;
#pragma unroll
            for (int h = 0; h < NB; ++h)
              tma_load_4d(dst + h * 128 * PITCH + lane * group * PITCH, m, fulls + slot, (p * C::SW * ESZ + h * PITCH) / ESZ, g,
                          po, pg);
          }
          __syncwarp();
          // every producer arrives on every tile (feeder 0 has; the last one for codes with its copies of scales): see ptc_arrivals
          if (feeder != 0 && !(Q8 && feeder == C::FEEDERS - 1) && lane == 0) mbar_arrive(fulls + slot);
          if constexpr (Q8) {
            if (feeder == C::FEEDERS - 1) {
              if (!is_v && p == 0) {  // both scales come with the keys: the weights need them before the values
                float* ss = sscale + ((blocks + j) & (C::SCALE_BLOCKS - 1)) * 256 + lane * 4;
                const int from = (lane * 4) >> a.group_log2;
                const int p2 = __shfl_sync(0xffffffffu, pg, from), o2 = __shfl_sync(0xffffffffu, po, from);
                if ((good >> from) & 1u) {
                  const int64_t so = (int64_t)p2 * a.ss_block + g * a.ss_head + o2 + ((lane * 4) & (group - 1));
                  cp_async16(ex_smem_u32(ss), a.k_scale + so, true);
                  cp_async16(ex_smem_u32(ss + 128), a.v_scale + so, true);
                }
              }
              asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ex_smem_u32(fulls + slot)) : "memory");
            }
          }
          ++made;
          if (++slot == SLOTS) slot = 0, ph ^= 1;
        }
        if (!Q8 && is_v && j >= jedge) {
          if (ok && lane == 0) mbar_arrive(ask_bar + (edges & (PTC_EDGES - 1)));
          ++edges;
        }
      }
      blocks += nblk;
      __syncwarp();
    }
    // every load has landed before the CTA ends (also after a wait that ran out)
    for (int i = max(0, made - SLOTS); i < made; ++i)
      mbar_wait(fulls + i % SLOTS, (uint32_t)(i / SLOTS) & 1u, EX_DEVERR_WAIT_TMA);
  } else if (warp == 8) {
    // ------------------------------------------------------------------------------------------------ products
    constexpr uint32_t id_s = make_idesc_16(128, 128, MF16, false), id_o = make_idesc_16(128, C::SW, MF16, true);
    // The whole warp walks and waits, one lane issues. A wait that ran out is not looked at: what is issued then is wrong and
    // harmless, the error is recorded, and every later wait ends at once.
    const uint32_t dq = warp_uniform((uint32_t)make_sw128_desc(ex_smem_u32(smem))),
                   dr = warp_uniform((uint32_t)make_sw128_desc(ex_smem_u32(ring))),
                   dv = warp_uniform((uint32_t)make_sw128_desc_n(ex_smem_u32(ring), C::SUB)), tm = warp_uniform(tmem);
    uint32_t slot = 0, ph = 0, php = 0, phq = 0, edges = 0;
    auto commit = [&](uint64_t* b) { tc_commit_warp(b); };
    while (next()) {
      const int nb = (int)warp_uniform((uint32_t)nblk), je = (int)warp_uniform((uint32_t)jedge);
      if (nb == 0) continue;
      mbar_wait(q_bar, phq, EX_DEVERR_WAIT_TMEM);
      phq ^= 1;
#pragma unroll 1
      for (int n = 0; n < 2 * nb; ++n) {
        int j;
        const bool is_v = ptc_tile(n, nb, j);
        const uint32_t sbuf = tm + TM_S + (j & 1) * 128;
        if (is_v) {
          if (!Q8 && j >= je) {
            mbar_wait(fix_bar + (edges & (PTC_EDGES - 1)), (edges / PTC_EDGES) & 1u, EX_DEVERR_WAIT_MMA);
            ++edges;
          }
          mbar_wait(p_bar + (j & 1), (php >> (j & 1)) & 1u, EX_DEVERR_WAIT_TMEM);
          php ^= 1u << (j & 1);
        }
#pragma unroll
        for (int p = 0; p < C::PARTS; ++p) {
          mbar_wait(full_bar + slot, ph, EX_DEVERR_WAIT_TMA);
          __syncwarp();
          tc_fence_after();
          {
            if (is_v) {
              const uint32_t d = tm + TM_O + (C::STREAMS == 2 ? (j & 1) * D : p * C::SW), db = dv + slot * (C::SLOT >> 4);
              const uint32_t acc = j >= C::STREAMS ? 1u : 0u;
#pragma unroll
              for (int k = 0; k < 8; ++k) tc_mma_16_ta(d, sbuf + k * 8, db + k * (2048 >> 4), id_o, k > 0 ? 1u : acc);
            } else {
              const uint32_t db = dr + slot * (C::SLOT >> 4);
#pragma unroll
              for (int x = 0; x < C::SW / 64; ++x)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  tc_mma_16(sbuf, dq + (p * (C::SW / 64) + x) * (C::SUB >> 4) + 2 * k, db + x * (C::SUB >> 4) + 2 * k, id_s,
                            (p | x | k) != 0);
            }
            commit(empty_bar + slot);
          }
          if (++slot == C::SLOTS) slot = 0, ph ^= 1u;
        }
        if (!is_v) commit(s_bar + (j & 1));
        else if (C::STREAMS == 1) commit(o_bar);
      }
      commit(end_bar);
    }
    // every product is done before tensor memory is given back
    commit(done_bar);
    mbar_wait(done_bar, 0, EX_DEVERR_WAIT_MMA);
    __syncwarp();
  } else if ((warp == 10 || warp == 11) && !Q8) {
    // ---------------------------------------------------------------------------------------------- edge values
    int base = 0;   // slots of the items before
    uint32_t edges = 0;
    int item = 0;
    bool ok = true;
    while (ok && next()) {
      uint32_t* mine = poison + (item & (PTC_POISON - 1)) * 8;
      if (jedge < nblk) ++item;
      for (int j = jedge; j < nblk && ok; ++j) {
        const int e = j - jedge;
        // the producer's word that the slots are this block's
        ok = mbar_wait_idle(ask_bar + (edges & (PTC_EDGES - 1)), (edges / PTC_EDGES) & 1u, EX_DEVERR_WAIT_SLOT);
        for (int p = 0; p < C::PARTS && ok; ++p) {
          const int at = base + (min(j + 2, nblk) + j) * C::PARTS + p;  // in the order of loading
          uint8_t* vs = ring + (at % C::SLOTS) * C::SLOT;
          ok = mbar_wait(full_bar + at % C::SLOTS, (uint32_t)(at / C::SLOTS) & 1u, EX_DEVERR_WAIT_TMA);
          ok = __all_sync(0xffffffffu, ok);
          if (ok) clean_values<F16, 64>(vs, C::SW / 64, tid & 63, end - start - j * 128, mine + e * 4);
        }
        fence_proxy_async_shared();  // the products read shared memory through the async proxy
        if (ok) mbar_arrive(fix_bar + (edges & (PTC_EDGES - 1)));
        ++edges;
      }
      base += 2 * nblk * C::PARTS;
    }
  } else if (Q8 && warp >= 12) {
    // ------------------------------------------------------------------------------------------------ converters
    if constexpr (Q8) {
      const int t = tid - 384;
      int rslot = 0, slot = 0;
      uint32_t rph = 0, ph = 1;
      int item = 0;
      bool ok = true;
      while (ok && next()) {
        uint32_t* mine = poison + (item & (PTC_POISON - 1)) * 8;
        if (jedge < nblk) ++item;
#pragma unroll 1
        for (int n = 0; n < 2 * nblk && ok; ++n) {
          int j;
          const bool is_v = ptc_tile(n, nblk, j);
#pragma unroll 1
          for (int p = 0; p < C::PARTS; ++p) {
            ok = mbar_wait(rfull_bar + rslot, rph, EX_DEVERR_WAIT_TMA) && mbar_wait(empty_bar + slot, ph, EX_DEVERR_WAIT_SLOT);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            uint8_t* src = raw + rslot * C::RAW;
            uint8_t* dst = ring + slot * C::SLOT;
            // 8 lanes take the same 16 codes of 8 keys (no bank twice), then the keys STEP on: the swizzle stays the same
            constexpr int CH = C::SW / 16, STEP = 128 / CH;
            const int r0 = (t & 7) + t / (8 * CH) * 8, c = (t >> 3) % CH, c2 = (c & 3) * 2;
            src += C::SW == 128 ? r0 * 128 + ((c ^ (r0 & 7)) << 4) : r0 * 64 + ((c ^ ((r0 >> 1) & 3)) << 4);
            dst += (c >> 2) * C::SUB + r0 * 128;
            const int d0 = (c2 ^ (r0 & 7)) << 4, d1 = ((c2 + 1) ^ (r0 & 7)) << 4;
            if (is_v && j >= jedge) {  // values behind the end: zeros; codes that are NaN: zeros, noted
              const int left = end - (start + j * 128 + r0);
#pragma unroll 1
              for (int i = 0; i < CH; ++i) {
                uint4* x = reinterpret_cast<uint4*>(src + i * STEP * C::SW);
                if (i * STEP >= left) {
                  *x = make_uint4(0, 0, 0, 0);
                } else if constexpr (NOTES) {
                  const uint4 w = *x;
                  if ((not_finite<CODE, F16>(w.x) | not_finite<CODE, F16>(w.y) | not_finite<CODE, F16>(w.z) | not_finite<CODE, F16>(w.w)) == 0) continue;
                  *x = make_uint4(only_finite<CODE, F16>(w.x), only_finite<CODE, F16>(w.y), only_finite<CODE, F16>(w.z), only_finite<CODE, F16>(w.w));
                  const int key = r0 + i * STEP;
                  atomicOr(mine + (j - jedge) * 4 + (key >> 5), 1u << (key & 31));
                }
              }
            }
#pragma unroll 4
            for (int i = 0; i < CH; ++i) {
              const uint4 w = *reinterpret_cast<const uint4*>(src + i * STEP * C::SW);
              uint32_t o[8];
              codes_to_f16<CODE>(w.x, o[0], o[1]);
              codes_to_f16<CODE>(w.y, o[2], o[3]);
              codes_to_f16<CODE>(w.z, o[4], o[5]);
              codes_to_f16<CODE>(w.w, o[6], o[7]);
              *reinterpret_cast<uint4*>(dst + i * STEP * 128 + d0) = make_uint4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<uint4*>(dst + i * STEP * 128 + d1) = make_uint4(o[4], o[5], o[6], o[7]);
            }
            fence_proxy_async_shared();
            mbar_arrive(full_bar + slot);
            mbar_arrive(rempty_bar + rslot);
            if (++rslot == C::RAWS) rslot = 0, rph ^= 1;
            if (++slot == C::SLOTS) slot = 0, ph ^= 1;
          }
        }
      }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SOFTMAX));
    // -------------------------------------------------------------------------------------------------- softmax
    const int wg = warp >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the tile
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t phs[2] = {0, 0}, pho = 0, phe = 0, blocks = 0;
    int item = 0;
    // The queries of an item: row-major in swizzled columns of 64 dims, D / 8 lanes a row. Up to D = 128 they are loaded (QN
    // pieces a thread) while the products of the item before still run; codes leave no registers for it (with it 3 % slower).
    constexpr int LANES = D / 8, QSTEP = 256 / LANES, QN = 128 / QSTEP;
    constexpr bool AHEAD = D <= 128 && !Q8;
    const int qc = tid % LANES, qx = tid / LANES;
    uint4 qv[AHEAD ? QN : 1];
    auto load_q = [&](int x) {
      const int copies = R <= 32 ? 4 : R <= 64 ? 2 : 1, xl = copies == 1 ? row0 + x : x & (128 / copies - 1);
      if (xl >= R) return make_uint4(0, 0, 0, 0);
      const int t = (int)((uint32_t)xl * a.g_inv >> 16);
      return *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(first + t) * a.sq_t +
                                             (int64_t)(g * a.G + xl - t * a.G) * a.sq_h + qc * 8);
    };
    auto put_q = [&](int x, uint4 v) {
      if constexpr (Q8) {
        float f = 1.0f;
        if (!a.q_is_f16) {
          float y[8];
          unpack2<__nv_bfloat16>(v.x, y[0], y[1]);
          unpack2<__nv_bfloat16>(v.y, y[2], y[3]);
          unpack2<__nv_bfloat16>(v.z, y[4], y[5]);
          unpack2<__nv_bfloat16>(v.w, y[6], y[7]);
          float mq = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) mq = fmaxf(mq, fabsf(y[i]));
#pragma unroll
          for (int o = LANES / 2; o; o >>= 1) mq = fmaxf(mq, __shfl_xor_sync(0xffffffffu, mq, o));
          const float inv = pr_query_scale(mq, f);
          v.x = pack2<__half>(y[0] * inv, y[1] * inv);
          v.y = pack2<__half>(y[2] * inv, y[3] * inv);
          v.z = pack2<__half>(y[4] * inv, y[5] * inv);
          v.w = pack2<__half>(y[6] * inv, y[7] * inv);
        }
        if (qc == 0) sfac[x] = fmaxf(f * fabsf(a.scale_log2), 1e-45f);  // (0 times the -infinity of a hidden key would be NaN)
      }
      if (a.scale_log2 < 0.0f) {  // the largest score is looked for before it is scaled
        v.x ^= 0x80008000u;
        v.y ^= 0x80008000u;
        v.z ^= 0x80008000u;
        v.w ^= 0x80008000u;
      }
      *reinterpret_cast<uint4*>(smem + (qc >> 3) * C::SUB + x * 128 + (((qc & 7) ^ (x & 7)) << 4)) = v;
    };
    auto next_item = [&]() {  // the next item and, in registers, its queries
      const bool more = next();
      if constexpr (AHEAD) {
        if (more && nblk > 0) {
#pragma unroll
          for (int i = 0; i < QN; ++i) qv[i] = load_q(qx + i * QSTEP);
        }
      }
      return more;
    };
    bool more = next_item();
    while (more) {
      uint32_t* mine = poison + (item & (PTC_POISON - 1)) * 8;
      if (jedge < nblk) ++item;
      // copies of the rows: each weighs W keys of a block
      const int copies = R <= 32 ? 4 : R <= 64 ? 2 : 1, rows = 128 / copies, W = 128 / copies;
      const int rl = copies == 1 ? row0 + r : r & (rows - 1);  // row of the request (at least R: none)
      const int col = copies == 1 ? 0 : r / rows * W;
      const bool active = copies > 1 || row0 + (warp & 3) * 32 < R;  // some row of this warp is real
      // codes: O is the sum of the weights times value scales times codes over 2^(vtop - m); vinv = 2^(m - vtop)
      float m = -INFINITY, l = 0.0f, vtop = -INFINITY, vinv = 0.0f;
      if (nblk > 0) {
        if constexpr (AHEAD) {
#pragma unroll
          for (int i = 0; i < QN; ++i) put_q(qx + i * QSTEP, qv[i]);
        } else {
#pragma unroll 1
          for (int i = 0; i < QN; i += 4) {
            uint4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = load_q(qx + (i + k) * QSTEP);
#pragma unroll
            for (int k = 0; k < 4; ++k) put_q(qx + (i + k) * QSTEP, v[k]);
          }
        }
        fence_proxy_async_shared();
        tc_fence_before();  // the last item's O has been read
        mbar_arrive(q_bar);
        if constexpr (Q8) asm volatile("bar.sync 2, 256;" ::: "memory");  // sfac
      }
      const float fac = Q8 ? sfac[r] : fabsf(a.scale_log2);
      uint64_t word = 0;
      if (rl < R) {
        const int t = (int)((uint32_t)rl * a.g_inv >> 16);
        word = (a.mask ? a.mask[first + t] : ~0ull >> (63 - min(t, 63))) & (~0ull >> (64 - T));  // (T >= 1)
      }
      const uint32_t all_good = (uint32_t)((1ull << (128 >> a.group_log2)) - 1ull);
      for (int j = (C::STREAMS == 2 ? wg : 0); j < (C::STREAMS == 2 || wg == 0 ? nblk : 0); j += C::STREAMS) {
        const int buf = j & 1;
        if (!mbar_wait(s_bar + buf, phs[buf], EX_DEVERR_WAIT_MMA)) *sfail = 1;
        phs[buf] ^= 1;
        __syncwarp();
        tc_fence_after();
        if (active) {
          const uint32_t s_addr = tmem + lanes + TM_S + buf * 128;
          const uint32_t o_addr = tmem + lanes + TM_O + (C::STREAMS == 2 ? wg * D : 0);
          const int kb = start + j * 128;
          const uint32_t good = sgood[(blocks + j) & 7];
          const float* ks = sscale + ((blocks + j) & (C::SCALE_BLOCKS - 1)) * 256;
          const bool whole = j < jedge && good == all_good;
          auto see = [&](int q) {  // 32 columns from col + 32 q on
            const int at = kb + col + 32 * q, d = at - ctx;  // key, drafted token of the first
            uint32_t v = d >= 64 ? 0u : d >= 0 ? (uint32_t)(word >> d) : d > -32 ? (uint32_t)(word << -d) | ((1u << -d) - 1u) : ~0u;
            const int left = end - at;
            if (left < 32) v &= left > 0 ? (1u << left) - 1u : 0u;
            uint32_t pages = 0;
            for (int i = 0; i < 32 >> a.group_log2; ++i)
              if ((good >> (((col + 32 * q) >> a.group_log2) + i)) & 1u) pages |= ((1u << (1 << a.group_log2)) - 1u) << (i << a.group_log2);
            return v & pages;
          };
          // One step of 32 or 64 columns keeps its scores; more are read twice. Blocks that are not seen whole take a loop of
          // their own, in steps of 32.
          constexpr int STEP = Q8 ? 32 : 64;
          float x[STEP];
          auto masked = [&](int q) {
            float (&y)[32] = reinterpret_cast<float (&)[32]>(x);
            ptc_scores<Q8>(s_addr + col + q * 32, ks + col + q * 32, y);
            const uint32_t v = see(q);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((v >> i) & 1u)) y[i] = -INFINITY;
          };
          float most = 0.0f;  // log2 of the block's largest value scale (numbers of one sign are in order as their bits are)
          if constexpr (Q8) {
            const float4 v = *reinterpret_cast<const float4*>(ks + 128 + lane * 4);
            const uint32_t bits = __float_as_uint(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
            most = __log2f(__uint_as_float(__reduce_max_sync(0xffffffffu, bits)));
          }
          float mb = -INFINITY, vb = -INFINITY;  // the largest score, and the largest with the value scale in it
          const float* vs = ks + 128 + col;
          if (!whole) {
#pragma unroll 1
            for (int q = 0; q < W / 32; ++q) {
              masked(q);
              mb = fmaxf(mb, ptc_max(reinterpret_cast<float (&)[32]>(x)));
              if constexpr (Q8) vb = fmaxf(vb, ptc_high(reinterpret_cast<float (&)[32]>(x), vs + q * 32, fac));
            }
          } else if (W == 32) {
            ptc_scores<Q8>(s_addr + col, ks + col, reinterpret_cast<float (&)[32]>(x));
            mb = ptc_max(reinterpret_cast<float (&)[32]>(x));
          } else {
#pragma unroll 1
            for (int q = W / STEP - 1; q >= 0; --q) {  // (the first step last: it is kept)
              ptc_scores<Q8>(s_addr + col + q * STEP, ks + col + q * STEP, x);
              mb = fmaxf(mb, ptc_max(x));
            }
          }
          mb *= fac;
          if constexpr (Q8) {
            // No product passes the largest score with the largest scale (but for roundings, hence 11.9): the products are looked
            // at only if that would matter. Whether they are may depend on the warp's other rows, what is then decided does not.
            // (Products of up to 2^12 references are far from float16's largest number; with 2^6 the bound of 32 rows calls for a
            // look in most blocks: 64 requests of 8192 keys, e4m3, 16 tokens, 710 us instead of 577.)
            if (whole) {
              if (__any_sync(0xffffffffu, !(mb + most <= vtop + 11.9f))) {
                if (W == 32) {
                  vb = ptc_high(x, vs, fac);
                } else {
#pragma unroll 1
                  for (int q = W / STEP - 1; q >= 0; --q) {
                    ptc_scores<Q8>(s_addr + col + q * STEP, ks + col + q * STEP, x);
                    vb = fmaxf(vb, ptc_high(x, vs + q * STEP, fac));
                  }
                }
              }
            }
          }
          // (m = -inf: any finite score; codes: a weight of 2^6 times a value scale of at most 2^121 is a number)
          const bool grows = mb > m + (Q8 ? 6.0f : 8.0f);
          const bool vgrows = Q8 && vb > vtop + 12.0f;
          if (__any_sync(0xffffffffu, grows || vgrows)) {
            const float mn = grows ? mb : m;
            float al = mn == -INFINITY ? 1.0f : ex2(m - mn);
            m = mn;
            l *= al;
            if constexpr (Q8) {  // O stays where only m has grown: it is over the reference
              const float to = fmaxf(vgrows ? vb : vtop, m - 126.0f);  // (what it is divided by stays a normal number)
              al = to == -INFINITY ? 1.0f : ex2(vtop - to);
              vtop = to;
              const float half = ex2(0.5f * (m - vtop));  // (2^(m - vtop) may be below the normal numbers)
              vinv = vtop > -INFINITY ? half * half : 0.0f;
            }
            if (j >= C::STREAMS && (!Q8 || __any_sync(0xffffffffu, al != 1.0f))) {  // (else nothing is on O yet)
              // the last product on this O is done: it was issued before this S (D = 256: after it)
              if (C::STREAMS == 1) {
                if (!mbar_wait(o_bar, (pho + j - 1) & 1u, EX_DEVERR_WAIT_MMA)) *sfail = 1;
                __syncwarp();
                tc_fence_after();
              }
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
                tmem_ld16(o_addr + c, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
                tmem_st16(o_addr + c, o);
              }
            }
          }
          const float sub = m == -INFINITY ? 0.0f : m;
          const uint32_t p_addr = s_addr + (col >> 1);
          if (!whole) {
#pragma unroll 1
            for (int q = 0; q < W / 32; ++q) {
              masked(q);
              float y[32];  // scales of the keys that are seen (of others they may be anything)
              if constexpr (Q8) {
                const uint32_t v = see(q);
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] = (v >> i) & 1u ? vs[q * 32 + i] : 0.0f;
              }
              l += ptc_weights<Q8, MF16>(p_addr + q * 16, Q8 ? y : nullptr, fac, sub, vinv, reinterpret_cast<float (&)[32]>(x));
            }
          } else if (W == 32) {
            l += ptc_weights<Q8, MF16>(p_addr, vs, fac, sub, vinv, reinterpret_cast<float (&)[32]>(x));
          } else {
#pragma unroll 1
            for (int q = 0; q < W / STEP; ++q) {
              if (q > 0) ptc_scores<Q8>(s_addr + col + q * STEP, ks + col + q * STEP, x);
              l += ptc_weights<Q8, MF16>(p_addr + q * (STEP / 2), vs + q * STEP, fac, sub, vinv, x);
            }
          }
          if (copies > 1) {  // no weight of this copy for the other keys
            const uint32_t z[16] = {};
#pragma unroll 1
            for (int q = 0; q < 4; ++q)
              if (q * 32 < col || q * 32 >= col + W) tmem_st16(s_addr + q * 16, z);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(p_bar + buf);
      }
      // the item as the results need it; the next one is looked up, and its queries are loaded, while the last products run
      struct { int b, first, T, L, g, s, row0, R, start, end, ctx, nblk, jedge; } const w = {b, first, T, L, g, s, row0, R, start, end, ctx, nblk, jedge};
      more = next_item();
      // the streams and copies of each row, CD dims at a time through shared memory (over the queries); four warps each
      // take every other piece of the head dimension
      if (w.nblk > 0 && !mbar_wait(end_bar, phe, EX_DEVERR_WAIT_MMA)) *sfail = 1;
      if (w.nblk > 0) phe ^= 1;
      asm volatile("bar.sync 2, 256;" ::: "memory");  // (every product is done: the queries may be written over)
      if (*sfail) break;  // the same for every thread here: the flag is only set before the barrier
      tc_fence_after();
      float* sm = reinterpret_cast<float*>(smem);  // [2 streams][128]: m, then l, then 2^(vtop - m)
      sm[wg * 128 + r] = m;
      sm[256 + wg * 128 + r] = l;
      if constexpr (Q8) {
        const float half = ex2(0.5f * (vtop - m));
        sm[512 + wg * 128 + r] = vtop > -INFINITY ? half * half : 0.0f;
      }
      asm volatile("bar.sync 2, 256;" ::: "memory");
      pho += w.nblk;
      blocks += w.nblk;
      float mall = -INFINITY, lall = 0.0f, f[2];
      for (int k = 0; k < copies; ++k) {
        const int x = copies == 1 ? r : (r & (rows - 1)) + k * rows;
        mall = fmaxf(mall, fmaxf(sm[x], sm[128 + x]));
      }
      const float sub = mall == -INFINITY ? 0.0f : mall;
      for (int k = 0; k < copies; ++k) {
        const int x = copies == 1 ? r : (r & (rows - 1)) + k * rows;
        lall += sm[256 + x] * ex2(sm[x] - sub) + sm[256 + 128 + x] * ex2(sm[128 + x] - sub);
      }
      bool some[2];  // (a stream that weighed nothing may hold anything; one with a factor of 0 may hold NaN, which stays)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        some[i] = sm[i * 128 + r] > -INFINITY;
        f[i] = some[i] ? ex2(sm[i * 128 + r] - sub) * (Q8 ? sm[512 + i * 128 + r] : 1.0f) : 0.0f;
      }
      const bool have1 = C::STREAMS == 2 && w.nblk > 1;
      const bool single = pr_segments_many(pr_keys(a, w.L)) == 1;
      bool any = false;
      if (NOTES && w.jedge < w.nblk)
        for (int i = 0; i < 8; ++i) any |= mine[i] != 0;
      const float inv = lall > 0.0f ? 1.0f / lall : (lall == 0.0f ? 0.0f : lall);  // nothing seen: zeros; NaN stays NaN
      asm volatile("bar.sync 2, 256;" ::: "memory");  // sm has been read
      float* piece = reinterpret_cast<float*>(smem) + wg * 128 * CD;  // [128][CD], 4 floats a chunk, swizzled
      const int t2 = tid & 127;
#pragma unroll 1
      for (int c = wg * CD; c < D; c += 2 * CD) {
        if (active) {
#pragma unroll 1
          for (int k = 0; k < CD; k += 16) {
            uint32_t u[16] = {}, v[16] = {};
            if (w.nblk > 0) tmem_ld16(tmem + lanes + TM_O + c + k, u);
            if (have1) tmem_ld16(tmem + lanes + TM_O + D + c + k, v);
            tmem_ld_wait();
            float o[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              o[i] = some[0] ? __uint_as_float(u[i]) * f[0] : 0.0f;
              o[i] += some[1] ? __uint_as_float(v[i]) * f[1] : 0.0f;
            }
            if constexpr (!Q8) {
              if (copies > 1 && lall < INFINITY) {  // (NaN weights are NaN whatever the values)
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i += 2) top = max3_nan(top, fabsf(o[i]), fabsf(o[i + 1]));
                if (!(top < INFINITY)) {
                  float y[16];
#pragma unroll
                  for (int i = 0; i < 16; ++i) y[i] = o[i];
                  ptc_context_infinities<F16>(y, a.bt + (int64_t)w.b * a.sbt, a.BS, a.blocks,
                                              reinterpret_cast<const uint16_t*>(a.v) + (int64_t)w.g * a.sv_head + c + k, a.sv_block,
                                              a.sv_page, w.start, w.jedge * 128, col, W);
#pragma unroll
                  for (int i = 0; i < 16; ++i) o[i] = y[i];
                }
              }
            }
            if (single) {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= inv;
            }
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<float4*>(piece + r * CD + ((((k + i) >> 2) ^ (r & (CD / 4 - 1))) << 2)) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        if (wg == 0) asm volatile("bar.sync 4, 128;" ::: "memory");
        else asm volatile("bar.sync 5, 128;" ::: "memory");
        const int real = copies == 1 ? min(128, w.R - w.row0) : w.R, q = t2 % (CD / 4), d0 = c + q * 4;
#pragma unroll 2
        for (int x = t2 / (CD / 4); x < real; x += 128 / (CD / 4)) {
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int k = 0; k < copies; ++k) {
            const int y = x + k * rows;
            const float4 z = *reinterpret_cast<const float4*>(piece + y * CD + ((q ^ (y & (CD / 4 - 1))) << 2));
            v.x += z.x;
            v.y += z.y;
            v.z += z.z;
            v.w += z.w;
          }
          const int row = w.row0 + x, t = (int)((uint32_t)row * a.g_inv >> 16), h = w.g * a.G + row - t * a.G;
          if (NOTES && any) {  // values that were taken out: added as they are (their weight is positive) to the rows that see them
            const uint64_t rw = (a.mask ? a.mask[w.first + t] : ~0ull >> (63 - min(t, 63))) & (~0ull >> (64 - w.T));
#pragma unroll 1
            for (int k = 0; k < 256; ++k) {
              if (!((mine[k >> 5] >> (k & 31)) & 1u)) continue;
              const int key = w.start + w.jedge * 128 + k, d = key - w.ctx;
              if (key >= w.end || (d >= 0 && !((rw >> d) & 1ull))) continue;
              const int page = a.bt[(int64_t)w.b * a.sbt + key / a.BS];
              if (page < 0 || page >= a.blocks) continue;
              const int64_t at = (int64_t)page * a.sv_block + (int64_t)(key % a.BS) * a.sv_page + (int64_t)w.g * a.sv_head + d0;
              float y[4];
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                if constexpr (Q8) {
                  y[n] = (reinterpret_cast<const uint8_t*>(a.v)[at + n] & 0x7f) == 0x7f ? NAN : 0.0f;
                } else {
                  const uint16_t e = reinterpret_cast<const uint16_t*>(a.v)[at + n];
                  y[n] = F16 ? __half2float(__ushort_as_half(e)) : __uint_as_float((uint32_t)e << 16);
                  if (fabsf(y[n]) < INFINITY) y[n] = 0.0f;
                }
              }
              v.x += y[0];
              v.y += y[1];
              v.z += y[2];
              v.w += y[3];
            }
          }
          if (single) {
            const bool f16 = Q8 ? a.q_is_f16 != 0 : F16;
            uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + (int64_t)(w.first + t) * a.so_t +
                                                        (int64_t)h * a.so_h + d0);
            dst[0] = f16 ? pack2<__half>(v.x, v.y) : pack_bf16(v.x, v.y);
            dst[1] = f16 ? pack2<__half>(v.z, v.w) : pack_bf16(v.z, v.w);
          } else {
            *reinterpret_cast<float4*>(a.ws_acc + (((int64_t)(w.first + t) * a.H + h) * a.NS + w.s) * D + d0) = v;
          }
        }
        if (wg == 0) asm volatile("bar.sync 4, 128;" ::: "memory");
        else asm volatile("bar.sync 5, 128;" ::: "memory");
      }
      if (wg == 0 && !single && rl < w.R && (copies == 1 || r < rows)) {
        const int rt = (int)((uint32_t)rl * a.g_inv >> 16);
        const int64_t pi = ((int64_t)(w.first + rt) * a.H + w.g * a.G + rl - rt * a.G) * a.NS + w.s;
        a.ws_m[pi] = mall;
        a.ws_l[pi] = lall;
      }
      asm volatile("bar.sync 2, 256;" ::: "memory");  // before the queries and sfac are written again
      if (NOTES && any && tid < 8) mine[tid] = 0;     // for the item PTC_POISON on
    }
    __syncwarp();
    tc_fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ex
