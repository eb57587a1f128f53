// Layout of a key-value cache whose rows carry their own scales, as the kernels see it (fsa_quant_cache.cu, fsa_quant_dec_sm100.cu).
#pragma once
#include <stdint.h>

#include "../../include/fsa_b200.h"

namespace fsa {

inline int quant_row_bytes(const FsaQuantCache& c) { return c.format == FSA_QC_INT4 ? c.head_dim / 2 : c.head_dim; }
inline int quant_row_words(const FsaQuantCache& c) { return c.format == FSA_QC_INT4 ? c.head_dim / c.group : 1; }

// What every entry point asks of a cache: FSA_OK, or why not.
inline int check_quant_cache(const FsaQuantCache& c) {
  if (!c.k || !c.v || !c.k_scales || !c.v_scales || c.heads_kv <= 0 || c.head_dim <= 0) return FSA_ERR_INVALID_ARG;
  if (c.format != FSA_QC_INT8 && c.format != FSA_QC_E4M3 && c.format != FSA_QC_INT4) return FSA_ERR_UNSUPPORTED;
  if (c.head_dim > 128 || c.head_dim % 16) return FSA_ERR_UNSUPPORTED;
  if (c.format == FSA_QC_INT4 && ((c.group != 32 && c.group != 64) || c.head_dim % c.group)) return FSA_ERR_UNSUPPORTED;
  if (c.page_table ? (c.page_size <= 0 || c.max_pages <= 0 || c.num_pages <= 0) : c.capacity <= 0) return FSA_ERR_INVALID_ARG;
  if (((uintptr_t)c.k | (uintptr_t)c.v) & 15) return FSA_ERR_INVALID_ARG;
  if (((uintptr_t)c.k_scales | (uintptr_t)c.v_scales) & 3) return FSA_ERR_INVALID_ARG;
  for (int64_t s : {c.k_stride_b, c.k_stride_s, c.k_stride_h, c.v_stride_b, c.v_stride_s, c.v_stride_h})
    if (s % 16) return FSA_ERR_INVALID_ARG;
  return FSA_OK;
}

}  // namespace fsa
