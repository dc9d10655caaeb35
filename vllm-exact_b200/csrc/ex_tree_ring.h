// The ring of key and value tiles of k_tree_tc (ex_tree_tc.cuh), as its host check sees it: the order of the tiles and who
// arrives on the barrier of a slot. Plain C++, so that the protocol can be run step by step on a CPU.
#pragma once

#ifdef __CUDACC__
#define EX_RING_FN __host__ __device__ __forceinline__
#else
#define EX_RING_FN inline
#endif

namespace ex {

constexpr int ptc_feeders(bool codes) { return codes ? 3 : 4; }  // producer warps

// Arrivals of a producer warp on the "loaded" barrier of the slot of every tile, whether any box of the tile is its own or
// not: a slot that completed without a warp could be used up and filled again behind its back, and the warp would then wait on
// the parity of a later lap. For codes the last warp's 32 lanes arrive one by one, with their copies of scales.
constexpr int ptc_arrivals(bool codes, int feeder) { return codes && feeder == ptc_feeders(codes) - 1 ? 32 : 1; }
constexpr int ptc_loaded_count(bool codes) {
  int n = 0;
  for (int f = 0; f < ptc_feeders(codes); ++f) n += ptc_arrivals(codes, f);
  return n;
}

// The tiles of a segment of nblk blocks in the order of use, K0 K1 V0 K2 V1 .. (S of a block is made one block ahead of its
// P V): tile n of 2 nblk is block j's values or keys.
EX_RING_FN bool ptc_tile(int n, int nblk, int& j) {
  const bool v = n == 2 * nblk - 1 || (n > 0 && !(n & 1));
  j = n == 2 * nblk - 1 ? nblk - 1 : v ? (n >> 1) - 1 : (n + 1) >> 1;
  return v;
}

}  // namespace ex
