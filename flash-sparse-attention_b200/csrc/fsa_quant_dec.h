// What the decode over a cache with scales of its rows takes, and how its kernels are chosen (fsa_quant_dec_sm100.cu, and a source for
// each format beside it).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "fsa_quant_cache.h"
#include "fsa_quant_share.h"

namespace fsa {

constexpr int QUANT_TILE = 32;  // keys that a warp takes at a time

struct alignas(64) QuantDecParams {
  CUtensorMap map_k, map_v;    // codes: bytes of a row, heads, slots, blocks
  CUtensorMap map_ks, map_vs;  // scales, where a head's lie side by side: words of its slots, heads, blocks
  FsaQuantCache c;
  const void* q;
  void* out;
  float* lse;
  const int* used;
  const int* gather;
  float* pieces;   // [ctas][2][piece]: what the CTA's first item and its last one came to, where others share them
  int2* shared;    // [ctas]: (0: no first piece, 1: the item ends here, 2: it goes on), (item that begins here and goes on, or -1)
  int* status;
  long long q_sb, q_sh, o_sb, o_sh, l_sb, l_sh, g_sb;
  int batch, heads_q, group_heads;  // query heads of a KV head
  int blocks, items;                // of query heads a KV head, and of a sequence
  int topk, keys;                   // keys: slots of a sequence
  int chunks, words;                // of a row: 16-byte pieces, scales
  int page_shift;                   // log2 of the slots of a page
  int cache_blocks;                 // pages of the pool, or sequences
  int ctas;
  int cluster;                      // CTAs that share an item and meet in shared memory; 0: the work is one list
  bool scales_by_tma;
  float scale_log2;
};

// Sizes that a launch follows from: warps of a CTA, floats of a piece, query heads that an item takes.
struct QuantDecShape {
  int warps, piece, heads;
};
template <int FMT>
QuantDecShape quant_decode_shape(const FsaQuantCache& c, int dtype, int group_heads);
template <int FMT>
cudaError_t launch_quant_decode(const QuantDecParams& p, int dtype, cudaStream_t stream);

// f with an integral constant for the format.
template <typename F>
auto for_quant_format(int format, F&& f) {
  switch (format) {
    case FSA_QC_INT8: return f(std::integral_constant<int, FSA_QC_INT8>{});
    case FSA_QC_E4M3: return f(std::integral_constant<int, FSA_QC_E4M3>{});
    default: return f(std::integral_constant<int, FSA_QC_INT4>{});
  }
}

}  // namespace fsa
