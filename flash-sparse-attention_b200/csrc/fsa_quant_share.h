// How the tiles of an item fall to the warps of a cluster (fsa_quant_dec.cuh), for the host too.
#pragma once

#ifdef __CUDACC__
#define FSA_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define FSA_HOST_DEVICE inline
#endif

namespace fsa {

// Warp w's piece of `tiles` tiles: how many, and the first of them. Pieces of equal size, but for one tile, in the order of the warps, none of them empty before
// the last that is not. Everything follows from one number of tiles, so that a piece ends where its item does or before.
FSA_HOST_DEVICE int quant_cluster_share(int tiles, int warps, int w, int* first) {
  *first = 0;
  if (warps > tiles) warps = tiles;
  if (w >= warps) return 0;
  const int each = tiles / warps, more = tiles - each * warps;
  *first = each * w + more * w / warps;
  return each * (w + 1) + more * (w + 1) / warps - *first;
}

}  // namespace fsa
