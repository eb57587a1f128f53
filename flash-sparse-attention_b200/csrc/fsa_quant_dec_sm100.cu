// Entry points of the decode over a cache with scales of its rows; the kernels are in fsa_quant_dec.cuh.
#include "fsa_aux.h"
#include "fsa_params.h"
#include "fsa_quant_dec.h"

namespace fsa {

extern template QuantDecShape quant_decode_shape<FSA_QC_INT8>(const FsaQuantCache&, int, int);
extern template QuantDecShape quant_decode_shape<FSA_QC_E4M3>(const FsaQuantCache&, int, int);
extern template QuantDecShape quant_decode_shape<FSA_QC_INT4>(const FsaQuantCache&, int, int);
extern template cudaError_t launch_quant_decode<FSA_QC_INT8>(const QuantDecParams&, int, cudaStream_t);
extern template cudaError_t launch_quant_decode<FSA_QC_E4M3>(const QuantDecParams&, int, cudaStream_t);
extern template cudaError_t launch_quant_decode<FSA_QC_INT4>(const QuantDecParams&, int, cudaStream_t);

namespace {

// CTAs that take an item together and meet in shared memory, or 0: the work as one list, whose pieces meet in a kernel of their own. That kernel
// costs 4 us, which a cluster saves (one sequence of 8 KV heads of 128, int8: 200 keys 11.1 us, so 6.6; 2000 11.2 and 7.8; 8000 14.5 and 12.7); on
// the other side its CTAs are some of the GPU's and do not help one another, at about 1 us for each tile that a warp has more. So: as many CTAs as
// can all run (a cluster lies in one GPC, whose SMs need not be a multiple of it: 15 clusters of 8 ran at once, 33 of 4, 74 of 2, and a second turn
// doubles the time), and at most 4 tiles a warp where lengths are not known here and one sequence may have all the keys, else at most 3 tiles more
// than in the list (32 sequences x 2048 chosen keys: 24.4 us, so 21.1).
int cluster_of(long long items, long long tiles, int warps, bool alike, int sms) {
  int c = 8;
  while (c > 0 && (c > tiles || items * c > (c > 1 ? sms - 5 * c : sms))) c /= 2;
  if (c == 0) return 0;
  return (alike ? tiles * (sms - items * c) <= 3ll * c * warps * sms : tiles <= 4ll * c * warps) ? c : 0;
}

// What follows from sizes alone; a FSA_ERR_* code where they do not fit.
int plan(const FsaQuantDecodeArgs* a, QuantDecParams* p, int* warps, int* piece) {
  const FsaQuantCache& c = a->cache;
  const int rc = check_quant_cache(c);
  if (rc != FSA_OK) return rc;
  if (a->batch <= 0 || a->heads_q <= 0 || a->heads_q % c.heads_kv || a->topk < 0 || a->topk > 0x7fffff00) return FSA_ERR_INVALID_ARG;
  // the keys of a tile lie in one page
  if (c.page_table && (c.page_size < QUANT_TILE || (c.page_size & (c.page_size - 1)))) return FSA_ERR_UNSUPPORTED;
  for (p->page_shift = 0; c.page_table && 1 << p->page_shift < c.page_size;) ++p->page_shift;
  const long long keys = c.page_table ? (long long)c.max_pages * c.page_size : c.capacity;
  p->keys = (int)(keys < 0x7fffff00ll ? keys : 0x7fffff00ll);
  p->batch = a->batch;
  p->heads_q = a->heads_q;
  p->group_heads = a->heads_q / c.heads_kv;
  const QuantDecShape shape = for_quant_format(c.format, [&](auto f) { return quant_decode_shape<f()>(c, a->dtype, p->group_heads); });
  const int heads = shape.heads;
  *warps = shape.warps;
  *piece = shape.piece;
  p->blocks = (p->group_heads + heads - 1) / heads;
  if ((long long)p->blocks * c.heads_kv * a->batch > 0x7fffffffll) return FSA_ERR_UNSUPPORTED;
  p->items = p->blocks * c.heads_kv;
  p->topk = a->topk;
  p->chunks = quant_row_bytes(c) / 16;
  p->words = quant_row_words(c);
  const long long most = a->gather_kv_indices ? a->topk : p->keys, tiles = most > 0 ? (most + QUANT_TILE - 1) / QUANT_TILE : 1;
  const long long ctas = ((long long)p->items * a->batch * tiles + *warps - 1) / *warps;  // no warp without a tile
  const int sms = device_sm_count();
  p->ctas = (int)(ctas < sms ? ctas : sms);
  p->cluster = cluster_of((long long)p->items * a->batch, tiles, *warps, a->gather_kv_indices || !a->seqused_k, sms);
  return FSA_OK;
}

int64_t shared_bytes(const QuantDecParams& p) { return ((int64_t)p.ctas * sizeof(int2) + 15) / 16 * 16; }

}  // namespace

}  // namespace fsa

extern "C" int64_t fsa_decode_quantized_workspace_bytes(const FsaQuantDecodeArgs* a) {
  using namespace fsa;
  if (!a) return FSA_ERR_INVALID_ARG;
  QuantDecParams p = {};
  int warps, piece;
  const int rc = plan(a, &p, &warps, &piece);
  if (rc != FSA_OK) return rc;
  return p.cluster ? 16 : shared_bytes(p) + (int64_t)p.ctas * (2 + warps) * piece * (int64_t)sizeof(float);
}

extern "C" int fsa_decode_quantized(const FsaQuantDecodeArgs* a, void* stream_) {
  using namespace fsa;
  if (!a || !a->q || !a->out || !a->lse || !a->ws || !a->status) return FSA_ERR_INVALID_ARG;
  if (a->dtype != FSA_DT_BF16 && a->dtype != FSA_DT_FP16) return FSA_ERR_UNSUPPORTED;
  if (!(a->softmax_scale > 0.f) || a->softmax_scale > 3e38f) return FSA_ERR_INVALID_ARG;
  QuantDecParams p = {};
  int warps, piece;
  const int rc = plan(a, &p, &warps, &piece);
  if (rc != FSA_OK) return rc;
  if (((uintptr_t)a->q & 15) || ((uintptr_t)a->ws & 15) || ((uintptr_t)a->out & 3) || a->q_stride_b % 8 || a->q_stride_h % 8 || a->o_stride_b % 2 ||
      a->o_stride_h % 2)
    return FSA_ERR_INVALID_ARG;
  p.c = a->cache;
  p.q = a->q;
  p.out = a->out;
  p.lse = a->lse;
  p.used = a->seqused_k;
  p.gather = a->gather_kv_indices;
  p.shared = reinterpret_cast<int2*>(a->ws);
  p.pieces = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a->ws) + shared_bytes(p));
  p.status = a->status;
  p.q_sb = a->q_stride_b; p.q_sh = a->q_stride_h;
  p.o_sb = a->o_stride_b; p.o_sh = a->o_stride_h;
  p.l_sb = a->lse_stride_b; p.l_sh = a->lse_stride_h;
  p.g_sb = a->gather_stride;
  {
    const FsaQuantCache& c = p.c;
    const int wide = c.head_dim > 64 ? 128 : 64, bytes = c.format == FSA_QC_INT4 ? wide / 2 : wide;
    const uint64_t slots = c.page_table ? c.page_size : c.capacity, blocks = c.page_table ? c.num_pages : a->batch;
    p.cache_blocks = (int)blocks;
    auto map = [&](CUtensorMap* m, const void* base, int64_t sb, int64_t ss, int64_t sh) {
      return make_byte_map(m, base, quant_row_bytes(c), c.heads_kv, sh, slots, ss, blocks, sb, bytes, QUANT_TILE);
    };
    if (const int e = map(&p.map_k, c.k, c.k_stride_b, c.k_stride_s, c.k_stride_h); e != FSA_OK) return e;
    if (const int e = map(&p.map_v, c.v, c.v_stride_b, c.v_stride_s, c.v_stride_h); e != FSA_OK) return e;
    // a tile's scales come by TMA too where they are one piece that it can fetch, else lane by lane
    const int64_t groups = c.format == FSA_QC_INT4 ? wide / c.group : 1;
    auto one_piece = [&](const void* base, int64_t sb, int64_t ss, int64_t sh) {
      return ss == groups && p.words == groups && !((uintptr_t)base & 15) && (blocks == 1 || sb % 4 == 0) && (c.heads_kv == 1 || sh % 4 == 0) &&
             slots * groups < (1ull << 31);
    };
    p.scales_by_tma = !p.gather && one_piece(c.k_scales, c.ks_stride_b, c.ks_stride_s, c.ks_stride_h) &&
                      one_piece(c.v_scales, c.vs_stride_b, c.vs_stride_s, c.vs_stride_h);
    if (p.scales_by_tma) {
      const uint32_t box = (uint32_t)(QUANT_TILE * groups);
      if (const int e = make_word_map(&p.map_ks, c.k_scales, slots * groups, c.heads_kv, c.ks_stride_h, blocks, c.ks_stride_b, box); e != FSA_OK) return e;
      if (const int e = make_word_map(&p.map_vs, c.v_scales, slots * groups, c.heads_kv, c.vs_stride_h, blocks, c.vs_stride_b, box); e != FSA_OK) return e;
    }
  }
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  const cudaError_t e =
      for_quant_format(p.c.format, [&](auto f) { return launch_quant_decode<f()>(p, a->dtype, reinterpret_cast<cudaStream_t>(stream_)); });
  return e == cudaSuccess ? FSA_OK : FSA_ERR_LAUNCH;
}
