// Causal attention of packed prompts with grouped heads: sequence b has queries cu_q[b] .. cu_q[b + 1] and keys
// cu_k[b] .. cu_k[b + 1] of the packed arrays; its last query is its last key's token, so query i sees the keys
// j <= i + Lk - Lq. A query that sees none (Lk < Lq) gives zeros.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^((s_j - m) scale log2 e),  s_j = q . k_j
//
// m is a reference: the largest score of the row's first block, taken up again only when a score passes it by a factor of
// 2^20 (2^14 for float16 weights, which end at 2^16): the precision of the weights and sums is relative and does not
// depend on it, and O is almost never rescaled. It depends on the row alone.
//
// One CTA takes 256 queries of one head (128 where D = 256) and walks their keys in blocks of 128. tcgen05 products:
// S = Q K^T with both operands in shared memory, O += P V with P in tensor memory, over the S it came from.
//   warps 0-3, 4-7  softmax of query tiles 0 and 1, one row a thread; the S row is read to registers, P written back
//   warp 8          issues the products; while one tile's softmax runs, the other tile's products do
//   warp 9          TMA producer: Q once, then K and V of every block through one ring of slots
//   warps 10, 11    edge blocks (those not visible to every row): values behind the sequence's end, which belong to
//                   another sequence or to nobody, are zeroed, since 0 * NaN would reach O; values that are not finite
//                   are zeroed and noted, and the rows that see such a key get it added at the end.
// D = 256: one query tile and two S buffers (tensor memory holds no more), S of the next block issued before P V.
// Bound by the products and the exponentials together (busy 50 and 45 % of the cycles, in turn), at the clock that the board's
// power leaves. Three prompts of 2048 to 8192 tokens (32 heads of 128 over 8) take 710 us, 1.13 PFLOP/s, at 1965 MHz, and called
// for seconds, at 1657 MHz, 812 us, 0.98 PFLOP/s; one of 16384 tokens 1765 and 2058 us, and without its softmax 1554, without its
// products 1352 us. Steps of 64 keys with two S buffers a tile, so that no softmax waits for its S: 1810 to 1980 us (a product of
// 64 columns reads Q as often as one of 128). Two threads a row: no faster, and spills.
//
// P has the 16 bits of V, since a product takes both in one type: one rounding of half a step, 2^-8 of a weight over bf16, with
// the sum of the unrounded weights below it. Relative error of the long prompts against 64 bits 0.0022, of which the
// outputs' own rounding is 0.0016.
#pragma once
#include "ex_paged_rows.cuh"

namespace ex {

struct PaArgs {
  const void* v;  // as the tensor map reads it, for values that are not finite
  int64_t sv_t, sv_h;
  const int32_t *cu_q, *cu_k;
  int n, H, G;
  int64_t tokens, keys;  // rows of q and of k, v
  int tiles;             // at least as many query tiles as there are
  float scale_log2;
  void* out;
  int64_t so_t, so_h;
};

constexpr int PA_THREADS = 384;
constexpr int PA_KEYS = 128;
constexpr int PA_EDGES = 4;  // 256 rows reach over at most 3 blocks that are not visible to all of them
// Of eight pairs of weights PA_POLY are 2^x by polynomial (ex2_pair): prompts of 2048 to 8192 tokens, D = 128, take 770, 731,
// 774 and 807 us with 0, 1, 2 and 3. (Measured at D = 128, used for every head size.)
constexpr int PA_POLY = 1;
constexpr int PA_REGS_LAUNCH = 168, PA_REGS_SOFTMAX = 208, PA_REGS_OTHER = 88;
static_assert(256 * PA_REGS_SOFTMAX + 128 * PA_REGS_OTHER <= PA_THREADS * PA_REGS_LAUNCH, "register shares");

template <int D>
struct PaCfg {
  static constexpr int NQ = D == 256 ? 1 : 2;      // query tiles of 128 rows
  static constexpr int ROWS = 128 * NQ;
  static constexpr int SW = D < 128 ? D : 128;     // dims of a ring slot
  static constexpr int PARTS = D / SW;             // slots of one block's K or V
  static constexpr int SUB = 128 * 128;            // bytes of 128 rows x 64 dims, one swizzled column
  static constexpr int SLOT = SW / 64 * SUB;
  static constexpr int Q_BYTES = NQ * (D / 64) * SUB;
  static constexpr int SLOTS = D == 64 ? 8 : 5;
  static constexpr int SMEM = Q_BYTES + SLOTS * SLOT + 1024 + 512;
  static constexpr int TM_S = 0, TM_O = 256;       // columns: two S buffers of 128, then O (NQ x D)
};

// Instruction descriptor of tcgen05.mma kind::f16 with float32 accumulation: D format in bits [4,6) (1 = f32), A and B
// formats in [7,10) and [10,13) (0 = f16, 1 = bf16), B's major dimension in bit 16 (0 = K, 1 = N), N >> 3 in [17,23),
// M >> 4 in [24,29).
__host__ __device__ constexpr uint32_t make_idesc_16(int M, int N, bool f16, bool b_n_major) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | (b_n_major ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// Descriptor of an N-major operand in 128-byte swizzled columns of 64 elements: 8 rows of K are 1024 bytes, the next
// 64 elements of N lie `column` bytes on.
__device__ __forceinline__ uint64_t make_sw128_desc_n(uint32_t smem_addr, uint32_t column) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFF) | ((uint64_t)(column >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// Products of one tile, issued by a warp that is here as a whole and does not branch: one lane is elected in the instruction's
// own predicate. Where every operand is uniform over the warp (and the compiler can see it: see warp_uniform), operands are
// then made and held in uniform registers; in a branch of one lane each would be moved there, 50 to 80 cycles a product
// of 64.
// D[tmem] (+)= A B^T over 64 elements of K, operands in shared memory: low words of the descriptors (the high words, 1024
// bytes between groups of 8 rows, version 1, 128-byte swizzle, are the same for every operand here).
constexpr uint32_t SW128_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void tc_mma_16(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t.reg .b32 r;\n\telect.sync r|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "r"(SW128_DESC_HI)
      : "memory");
}
// the same with A in tensor memory
__device__ __forceinline__ void tc_mma_16_ta(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t.reg .b32 r;\n\telect.sync r|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(acc), "r"(SW128_DESC_HI)
      : "memory");
}
__device__ __forceinline__ void tc_commit_warp(uint64_t* bar) {  // tc_commit by one lane of a whole warp
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b32 r;\n\telect.sync r|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(ex_smem_u32(bar))
      : "memory");
}
// The value that every lane has, in a register the compiler knows to be uniform.
__device__ __forceinline__ uint32_t warp_uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

#define EX_R8(r, i) "=r"((r)[i]), "=r"((r)[i + 1]), "=r"((r)[i + 2]), "=r"((r)[i + 3]), "=r"((r)[i + 4]), "=r"((r)[i + 5]), "=r"((r)[i + 6]), "=r"((r)[i + 7])
#define EX_I8(r, i) "r"((r)[i]), "r"((r)[i + 1]), "r"((r)[i + 2]), "r"((r)[i + 3]), "r"((r)[i + 4]), "r"((r)[i + 5]), "r"((r)[i + 6]), "r"((r)[i + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : EX_R8(r, 0), EX_R8(r, 8), EX_R8(r, 16), EX_R8(r, 24)
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::EX_I8(r, 0),
      EX_I8(r, 8), EX_I8(r, 16), EX_I8(r, 24), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::EX_I8(
          r, 0),
      EX_I8(r, 8), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          ex_smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(ex_smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// The tile'th tile of `rows` queries over all sequences: its first query in its sequence, and that sequence's first query
// and key and numbers of both (a sequence whose offsets leave the arrays or run backwards, of queries or of keys, is taken to
// have no tiles: nothing of it is read or written); false if there is none.
// Every offset is loaded in the one pass: a second, dependent round of loads would cost 700 cycles.
__device__ __forceinline__ bool pa_find_tile(const PaArgs& a, int rows, int tile, int& row0, int& q0, int& Lq, int& k0, int& Lk) {
  const int lane = threadIdx.x & 31;
  int seen = 0;
  for (int base = 0; base < a.n; base += 32) {
    int c = 0, qa = 0, qb = 0, ka = 0, kb = 0;
    if (base + lane < a.n) {
      qa = a.cu_q[base + lane];
      qb = a.cu_q[base + lane + 1];
      ka = a.cu_k[base + lane];
      kb = a.cu_k[base + lane + 1];
      if (qa >= 0 && qa <= qb && qb <= a.tokens && ka >= 0 && ka <= kb && kb <= a.keys) c = (int)(((int64_t)qb - qa + rows - 1) / rows);
    }
    int incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned m = __ballot_sync(0xffffffffu, seen + incl > tile);
    if (m) {
      const int l = __ffs(m) - 1;
      row0 = (tile - seen - __shfl_sync(0xffffffffu, incl - c, l)) * rows;
      q0 = __shfl_sync(0xffffffffu, qa, l);
      k0 = __shfl_sync(0xffffffffu, ka, l);
      Lq = __shfl_sync(0xffffffffu, qb, l) - q0;
      Lk = __shfl_sync(0xffffffffu, kb, l) - k0;
      return true;
    }
    seen += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

struct f32x2 {
  uint64_t v;
};
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(f32x2 p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if any is
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x of a pair, x < 127, on the multiply-add units, which have time left where the exponential unit (16 a cycle and SM, a
// quarter of what a block of scores asks for) has none: x = i + f with i the nearest integer (1.5 2^23 leaves no bits behind the
// point), 2^f by a polynomial, i into the exponent. The polynomial is the least-maximum-error one of degree 4 on
// [-0.5, 0.5], fitted by iteratively reweighted least squares (Lawson's method): relative error 2.7e-6 = 2^-18.5 in
// float32, a hundredth of a rounding step of float16. Below 2^-126 it stays there: next to the largest weight (at least 1 when
// it was made the reference) that is nothing, and keys that are not seen have weight 0 from elsewhere.
__device__ __forceinline__ void ex2_pair(f32x2 x, float& a, float& b) {
  float x0, x1;
  split(x, x0, x1);
  x = pair(fmaxf(x0, -126.0f), fmaxf(x1, -126.0f));
  const f32x2 t = add2(x, pair(12582912.0f, 12582912.0f));
  const f32x2 f = add2(x, fma2(t, pair(-1.0f, -1.0f), pair(12582912.0f, 12582912.0f)));  // x - (t - 1.5 2^23)
  f32x2 p = fma2(f, pair(0.009570102207362652f, 0.009570102207362652f), pair(0.05591786280274391f, 0.05591786280274391f));
  p = fma2(f, p, pair(0.240247443318367f, 0.240247443318367f));
  p = fma2(f, p, pair(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(f, p, pair(0.9999992847442627f, 0.9999992847442627f));
  float t0, t1, p0, p1;
  split(t, t0, t1);
  split(p, p0, p1);
  a = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
  b = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}

// The 128 values of a slot (`columns` swizzled columns of 64 dims): those from number `live` on become zeros, and so do numbers
// that are not finite, whose keys are noted. 16 bytes of a key a thread, eight threads along a key's 128 bytes (no bank
// conflict; with a key a thread a block took 7000 cycles), four keys in flight.
template <bool F16, int THREADS>
__device__ __forceinline__ void clean_values(uint8_t* vs, int columns, int t, int live, uint32_t* noted) {
  constexpr int STEP = THREADS / 8;  // keys side by side
#pragma unroll 1
  for (int r = t >> 3; r < 128 * columns; r += 4 * STEP) {
    uint4* x = reinterpret_cast<uint4*>(vs + r * 128 + (t & 7) * 16);
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 w = x[i * STEP * 8];
      bad |= not_finite<CODE_NONE, F16>(w.x) | not_finite<CODE_NONE, F16>(w.y) | not_finite<CODE_NONE, F16>(w.z) | not_finite<CODE_NONE, F16>(w.w);
    }
    if (live >= 128 && bad == 0) continue;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      const int key = (r + i * STEP) & 127;
      const uint4 v = x[i * STEP * 8];
      if (key >= live) {
        x[i * STEP * 8] = make_uint4(0, 0, 0, 0);
      } else if (not_finite<CODE_NONE, F16>(v.x) | not_finite<CODE_NONE, F16>(v.y) | not_finite<CODE_NONE, F16>(v.z) | not_finite<CODE_NONE, F16>(v.w)) {
        x[i * STEP * 8] = make_uint4(only_finite<CODE_NONE, F16>(v.x), only_finite<CODE_NONE, F16>(v.y), only_finite<CODE_NONE, F16>(v.z), only_finite<CODE_NONE, F16>(v.w));
        atomicOr(noted + (key >> 5), 1u << (key & 31));
      }
    }
  }
}

template <int D, bool F16>
__global__ void __launch_bounds__(PA_THREADS, 1)
    k_prompt_attn(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PaArgs a) {
  using C = PaCfg<D>;
  extern __shared__ uint8_t pa_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pa_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + C::Q_BYTES;
  uint64_t* bar = reinterpret_cast<uint64_t*>(ring + C::SLOTS * C::SLOT);
  uint64_t* full_bar = bar;            // [8] ring slots
  uint64_t* empty_bar = bar + 8;       // [8]
  uint64_t* q_bar = bar + 16;          // [2] the queries of a tile
  uint64_t* s_bar = bar + 18;          // [2] S of a tile (D = 256: of a buffer) is there
  uint64_t* p_bar = bar + 20;          // [2] P of a tile (buffer) is there
  uint64_t* o_bar = bar + 22;          // D = 256: P V of a block is done
  uint64_t* end_bar = bar + 23;        // every product is done
  uint64_t* ask_bar = bar + 24;        // [PA_EDGES] loads of an edge block's values have been issued
  uint64_t* fix_bar = ask_bar + PA_EDGES;  // [PA_EDGES] they have been looked at
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fix_bar + PA_EDGES);
  uint32_t* poison = tmem_slot + 1;    // [16] edge keys with a value that is not finite

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  if (tid == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(full_bar + i, 1);
      mbar_init(empty_bar + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_bar + i, 1);
      mbar_init(s_bar + i, 1);
      mbar_init(p_bar + i, 128);
    }
    mbar_init(o_bar, 1);
    mbar_init(end_bar, 1);
    for (int i = 0; i < PA_EDGES; ++i) {
      mbar_init(ask_bar + i, 1);
      mbar_init(fix_bar + i, 64);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = 0; i < 16; ++i) poison[i] = 0;
  }
  pdl_wait();
  int row0, q0, Lq, k0, Lk;
  // the last tiles have the most keys: they start first
  if (!pa_find_tile(a, C::ROWS, a.tiles - 1 - (int)(blockIdx.x / a.H), row0, q0, Lq, k0, Lk) || row0 >= Lq) return;
  const int h = blockIdx.x % a.H, g = h / a.G;
  const int off = Lk - Lq;  // row i sees the keys j <= i + off
  int nblk[2];              // blocks of each tile
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int first = row0 + 128 * i, last = min(first + 127, Lq - 1);
    nblk[i] = (i < C::NQ && first < Lq) ? max(0, (min(Lk, last + off + 1) + PA_KEYS - 1) / PA_KEYS) : 0;
  }
  const int nmax = max(nblk[0], nblk[1]);
  const int edge = max(0, min(Lk, row0 + off + 1)) / PA_KEYS;  // blocks before it are seen by every row
  __syncthreads();  // the barriers are there: the first loads are under way while tensor memory is taken
  if (warp <= 8) {
    if (warp == 8) {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
    tc_fence_before();
    asm volatile("bar.sync 1, 288;" ::: "memory");
    tc_fence_after();
  }
  const uint32_t tmem = warp <= 8 ? *(volatile uint32_t*)tmem_slot : 0u;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_REGS_OTHER));
    if (warp == 9) {
      // -------------------------------------------------------------------------------------------- TMA producer
      if (lane == 0 && nmax > 0) {
        auto load_q = [&](int tile) {
          mbar_arrive_expect_tx(q_bar + tile, C::Q_BYTES / C::NQ);
#pragma unroll
          for (int i = 0; i < D / 64; ++i)
            tma_load_3d(smem + (tile * (D / 64) + i) * C::SUB, &tm_q, q_bar + tile, i * 64, h, q0 + row0 + tile * 128);
        };
        load_q(0);
        int slot = 0, made = 0;
        uint32_t ph = 1;
        bool ok = true;
        auto load = [&](const CUtensorMap* m, int j) {
          for (int p = 0; p < C::PARTS && ok; ++p) {
            ok = mbar_wait_idle(empty_bar + slot, ph, EX_DEVERR_WAIT_SLOT);
            if (!ok) return;
            mbar_arrive_expect_tx(full_bar + slot, C::SLOT);
#pragma unroll
            for (int s = 0; s < C::SW / 64; ++s)
              tma_load_3d(ring + slot * C::SLOT + s * C::SUB, m, full_bar + slot, p * C::SW + s * 64, g, k0 + j * PA_KEYS);
            ++made;
            if (++slot == C::SLOTS) slot = 0, ph ^= 1;
          }
        };
        // in the order of use: S of a block is issued one block ahead of P V
        load(&tm_k, 0);
        if (C::NQ == 2) load_q(C::NQ - 1);
        if (C::NQ == 1 && nmax > 1) load(&tm_k, 1);
        for (int j = 0; j < nmax && ok; ++j) {
          load(&tm_v, j);
          if (j >= edge && ok) mbar_arrive(ask_bar + (j - edge));
          const int k = j + (C::NQ == 1 ? 2 : 1);
          if (k < nmax) load(&tm_k, k);
        }
        for (int i = 0; i < C::NQ; ++i) mbar_wait(q_bar + i, 0, EX_DEVERR_WAIT_TMA);  // every load has landed before the CTA ends
        for (int i = max(0, made - C::SLOTS); i < made; ++i)
          mbar_wait(full_bar + i % C::SLOTS, (uint32_t)(i / C::SLOTS) & 1u, EX_DEVERR_WAIT_TMA);
      }
    } else if (warp == 8) {
      // -------------------------------------------------------------------------------------------- products
      // The whole warp walks and waits, one lane issues. A wait that ran out is not looked at: what is issued then is wrong and
      // harmless, the error is recorded, and every later wait ends at once.
      constexpr uint32_t id_s = make_idesc_16(128, 128, F16, false), id_o = make_idesc_16(128, C::SW, F16, true);
      const uint32_t dq = warp_uniform((uint32_t)make_sw128_desc(ex_smem_u32(smem))),
                     dr = warp_uniform((uint32_t)make_sw128_desc(ex_smem_u32(ring))),
                     dv = warp_uniform((uint32_t)make_sw128_desc_n(ex_smem_u32(ring), C::SUB)), tm = warp_uniform(tmem);
      const int n0 = (int)warp_uniform((uint32_t)nblk[0]), n1 = (int)warp_uniform((uint32_t)nblk[1]), nm = max(n0, n1);
      const int first_edge = (int)warp_uniform((uint32_t)edge);
      uint32_t slot = 0, ph = 0;  // next slot to be used
      // S (buffer) = Q (tile) K^T over the dims of the slot
      auto issue_s = [&](uint32_t at, int tile, int buf, int part) {
        {
#pragma unroll
          for (int x = 0; x < C::SW / 64; ++x)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc_mma_16(tm + C::TM_S + buf * 128, dq + ((tile * (D / 64) + part * (C::SW / 64) + x) * (C::SUB >> 4) + 2 * k),
                        dr + at * (C::SLOT >> 4) + (x * (C::SUB >> 4) + 2 * k), id_s, (part | x | k) != 0);
        }
      };
      auto issue_o = [&](uint32_t at, int tile, int buf, int part, uint32_t acc) {
        {
#pragma unroll
          for (int k = 0; k < PA_KEYS / 16; ++k)
            tc_mma_16_ta(tm + C::TM_O + tile * D + part * C::SW, tm + C::TM_S + buf * 128 + k * 8,
                         dv + at * (C::SLOT >> 4) + k * (2048 >> 4), id_o, k > 0 ? 1u : acc);
        }
      };
      auto commit = [&](uint64_t* b) { tc_commit_warp(b); };
      auto wait_full = [&](uint32_t at, uint32_t p) {
        mbar_wait(full_bar + at, p, EX_DEVERR_WAIT_TMA);
        __syncwarp();
        tc_fence_after();
      };
      if (nm > 0) {
        mbar_wait(q_bar, 0, EX_DEVERR_WAIT_TMA);
        if constexpr (C::NQ == 2) {
          wait_full(0, 0);
          if (n0 > 0) {
            issue_s(0, 0, 0, 0);
            commit(s_bar);
          }
          mbar_wait(q_bar + 1, 0, EX_DEVERR_WAIT_TMA);
          __syncwarp();
          tc_fence_after();
          if (n1 > 0) {
            issue_s(0, 1, 1, 0);
            commit(s_bar + 1);
          }
          commit(empty_bar);
          slot = 1;
#pragma unroll 1
          for (int j = 0; j < nm; ++j) {
            const bool more = j + 1 < nm;
            const uint32_t kslot = slot + 1 == C::SLOTS ? 0 : slot + 1, kph = kslot == 0 ? ph ^ 1u : ph;
            wait_full(slot, ph);
            if (j >= first_edge) mbar_wait(fix_bar + (j - first_edge), 0, EX_DEVERR_WAIT_MMA);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (j >= (i ? n1 : n0)) continue;
              mbar_wait(p_bar + i, (uint32_t)j & 1u, EX_DEVERR_WAIT_TMEM);
              __syncwarp();
              tc_fence_after();
              issue_o(slot, i, i, 0, j > 0 ? 1u : 0u);
              if (j + 1 < (i ? n1 : n0)) {
                if (i == 0 || j + 1 >= n0) wait_full(kslot, kph);
                issue_s(kslot, i, i, 0);
                commit(s_bar + i);
              }
            }
            commit(empty_bar + slot);
            if (more) commit(empty_bar + kslot);
            slot = kslot;
            ph = kph;
            if (more) {
              ++slot;
              if (slot == C::SLOTS) slot = 0, ph ^= 1u;
            }
          }
        } else {
          auto advance = [&]() { if (++slot == C::SLOTS) slot = 0, ph ^= 1u; };
          // K0 K1 V0 K2 V1 ..: S of a block is issued a block ahead of its P V
#pragma unroll 1
          for (int n = 0; n < 2 * nm; ++n) {
            const bool is_v = n == 2 * nm - 1 || (n > 0 && !(n & 1));
            const int j = n == 2 * nm - 1 ? nm - 1 : is_v ? (n >> 1) - 1 : (n + 1) >> 1;
            if (is_v) {
              if (j >= first_edge) mbar_wait(fix_bar + (j - first_edge), 0, EX_DEVERR_WAIT_MMA);
              mbar_wait(p_bar + (j & 1), (uint32_t)(j >> 1) & 1u, EX_DEVERR_WAIT_TMEM);
            }
#pragma unroll
            for (int p = 0; p < C::PARTS; ++p) {
              wait_full(slot, ph);
              if (is_v) issue_o(slot, 0, j & 1, p, j > 0 ? 1u : 0u);
              else issue_s(slot, 0, j & 1, p);
              commit(empty_bar + slot);
              advance();
            }
            commit(is_v ? o_bar : s_bar + (j & 1));
          }
        }
        commit(end_bar);
        mbar_wait(end_bar, 0, EX_DEVERR_WAIT_MMA);
      }
    } else {
      // -------------------------------------------------------------------------------------------- edge values
      const int t = tid - 320;  // 64 threads
      bool ok = true;
      for (int j = edge; j < nmax && ok; ++j) {
        // the producer may be any number of blocks behind: its word that the slots are this block's comes first
        ok = mbar_wait_idle(ask_bar + (j - edge), 0, EX_DEVERR_WAIT_SLOT);
        for (int p = 0; p < C::PARTS && ok; ++p) {
          // number of the slot in the order of loading: K of min(j + 2, nmax) or j + 1 blocks and V of j came before
          const int at = C::NQ == 1 ? (min(j + 2, nmax) + j) * C::PARTS + p : 2 * j + 1;
          uint8_t* vs = ring + (at % C::SLOTS) * C::SLOT;
          ok = mbar_wait(full_bar + at % C::SLOTS, (uint32_t)(at / C::SLOTS) & 1u, EX_DEVERR_WAIT_TMA);
          if (ok) clean_values<F16, 64>(vs, C::SW / 64, t, Lk - j * PA_KEYS, poison + (j - edge) * 4);
        }
        fence_proxy_async_shared();  // the products read shared memory through the async proxy
        if (ok) mbar_arrive(fix_bar + (j - edge));
      }
    }
  } else {
    // ---------------------------------------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PA_REGS_SOFTMAX));
    const int tile = warp >> 2;
    const int nb = nblk[tile & 1];
    const int whole = max(0, min(Lk, row0 + (tile & (C::NQ - 1)) * 128 + off + 1)) / PA_KEYS;  // blocks before it are seen by every row of the tile
    const int row = row0 + tile * 128 + (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_addr = tmem + lanes + C::TM_O + tile * D;
    const float sc = a.scale_log2;
    const float grow = (F16 ? 14.0f : 20.0f) / sc;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < nb; ++j) {
      const int buf = C::NQ == 2 ? tile : (j & 1);
      const uint32_t s_addr = tmem + lanes + C::TM_S + buf * 128;
      ok = mbar_wait(s_bar + buf, (uint32_t)(C::NQ == 2 ? j : j >> 1) & 1u, EX_DEVERR_WAIT_MMA);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      float s[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + c * 32, reinterpret_cast<uint32_t*>(s) + c * 32);
      tmem_ld_wait();
      // A block that is seen whole is weighed with the reference that there is, while its largest score is still being looked
      // for: nothing waits for it. If a score of the warp passes its row's reference by too much (or is NaN), or a row has none
      // yet (every score so far was -infinity), or the block is an edge, or the first, the block is weighed (again) below.
      bool again = j >= whole || j == 0;
      f32x2 sum0 = pair(0.0f, 0.0f), sum1 = sum0;
      // The weights of the block against the reference, written over S, and their sums. Both callers have the same arithmetic
      // in the same order, so that a row does not depend on which one its warp needs.
      auto weigh = [&](float sub, auto any) {  // any: scores that are -infinity (or not seen) or NaN too
        const f32x2 sc2 = pair(sc, sc), sub2 = pair(-sub, -sub);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const f32x2 x = fma2(pair(s[c * 32 + 2 * i], s[c * 32 + 2 * i + 1]), sc2, sub2);
            float a0, a1, x0, x1;
            split(x, x0, x1);
            if ((i & 7) < PA_POLY) {
              ex2_pair(x, a0, a1);
              if (decltype(any)::value) {
                a0 = x0 > -INFINITY ? a0 : ex2(x0);
                a1 = x1 > -INFINITY ? a1 : ex2(x1);
              }
            } else {
              a0 = ex2(x0);
              a1 = ex2(x1);
            }
            if (i & 1) sum1 = add2(sum1, pair(a0, a1));
            else sum0 = add2(sum0, pair(a0, a1));
            p[i] = F16 ? pack2<__half>(a0, a1) : pack_bf16(a0, a1);
          }
          tmem_st16(s_addr + c * 16, p);
        }
      };
      if (!again) {
        float mx[2] = {s[0], s[1]};
#pragma unroll
        for (int c = 2; c < 126; c += 4) {
          mx[0] = max3_nan(mx[0], s[c], s[c + 1]);
          mx[1] = max3_nan(mx[1], s[c + 2], s[c + 3]);
        }
        const float mb = max_nan(max3_nan(mx[0], s[126], s[127]), mx[1]);
        weigh(m * sc, std::false_type{});
        again = !(mb <= m + grow) || m == -INFINITY;  // (no reference yet: the weights just made are not numbers)
      }
      if (__any_sync(0xffffffffu, again)) {
        if (j >= whole) {
          const int limit = min(Lk - 1, row + off) - j * PA_KEYS;  // columns behind it are not seen
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = c <= limit ? s[c] : -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < 128; ++c) mx[c & 3] = fmaxf(mx[c & 3], s[c]);
        const float mb = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const bool take = mb > m + grow || m == -INFINITY;
        if (j == 0) {
          m = mb;
        } else if (__any_sync(0xffffffffu, take)) {
          // the next product on O waits for P, the last one is done: it was issued before this S (D = 256: after it)
          if (C::NQ == 1) {
            ok = mbar_wait(o_bar, (uint32_t)(j - 1) & 1u, EX_DEVERR_WAIT_MMA);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
          }
          const float mn = take ? fmaxf(m, mb) : m;
          const float al = m == -INFINITY ? (mn == -INFINITY ? 1.0f : 0.0f) : ex2((m - mn) * sc);
          m = mn;
          l *= al;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(o_addr + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
            tmem_st32(o_addr + c, o);
          }
        }
        sum0 = sum1 = pair(0.0f, 0.0f);
        weigh(m == -INFINITY ? 0.0f : m * sc, std::true_type{});
      }
      float a0, a1;
      split(add2(sum0, sum1), a0, a1);
      l += a0 + a1;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_bar + buf);
    }
    if (tile < C::NQ) {
      if (nmax > 0) {
        if (ok) ok = mbar_wait(end_bar, 0, EX_DEVERR_WAIT_MMA);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (ok) {
        const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // nothing seen: zeros; NaN stays NaN
        // the warp's 32 rows go through shared memory (over its queries), so that a row is written as a whole
        uint8_t* mine = smem + (tile * 128 + (warp & 3) * 32) * (2 * D);
        bool any = false;
        for (int i = 0; i < 16; ++i) any |= poison[i] != 0;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          __syncwarp();
          if (nb > 0) {
            tmem_ld32(o_addr + c, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          if (any) {  // values that were taken out: added as they are (their weight is positive) to the rows that see them
            const int seen = min(Lk, row + off + 1);
#pragma unroll 1
            for (int key = edge * PA_KEYS; key < seen; ++key) {
              const int k = key - edge * PA_KEYS;
              if (k >= 512 || !((poison[k >> 5] >> (k & 31)) & 1u)) continue;
              const uint16_t* v = reinterpret_cast<const uint16_t*>(a.v) + (int64_t)(k0 + key) * a.sv_t + (int64_t)g * a.sv_h + c;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float x = F16 ? __half2float(__ushort_as_half(v[i])) : __uint_as_float((uint32_t)v[i] << 16);
                if (!(fabsf(x) < INFINITY)) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float x = __uint_as_float(o[i + 2 * k]) * inv, y = __uint_as_float(o[i + 2 * k + 1]) * inv;
              w[k] = F16 ? pack2<__half>(x, y) : pack_bf16(x, y);
            }
            *reinterpret_cast<uint4*>(mine + lane * (2 * D) + ((((c + i) >> 3) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
        constexpr int PER = D / 8;  // 16-byte pieces of a row
        const int rows = min(32, Lq - (row - lane));
        uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + (int64_t)(q0 + row - lane) * a.so_t + (int64_t)h * a.so_h;
#pragma unroll 4
        for (int i = lane; i < rows * PER; i += 32) {
          const int r = i / PER, c = i % PER;
          *reinterpret_cast<uint4*>(dst + r * a.so_t + c * 8) = *reinterpret_cast<const uint4*>(mine + r * (2 * D) + ((c ^ (r & 7)) << 4));
        }
      }
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
