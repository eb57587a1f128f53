// Decode attention over a cache whose rows carry their own scales (fsa_quant_cache.cu): one query position per sequence.
//
// With codes k^, v^ and a row's scales a_j (keys), b_j (values)
//   s_jh = c (q_h . k^_j) a_j            8 bits            c = softmax_scale log2(e)
//   s_jh = c sum_g (q_hg . (k^_jg - 8)) a_jg + (sum q_hg) z_jg     4 bits, group by group
//   o_h  = sum_j p_jh b_j v^_j / sum_j p_jh,  p_jh = 2^(s_jh - m_h)
// so no value is ever rounded on its way: codes are exact in fp16, products and sums are those of the matrix instructions in fp32, scales are
// applied to scores and to probabilities. The queries enter as fp16 too: a row is multiplied by a power of two that brings its largest element
// to [2^10, 2^11) (exact but for elements 2^-24 and more below it, which lose less than 2^-34 of the largest), probabilities times b_j are rounded to
// fp16 (2^-11 of each; of fp16 results what that leaves goes in as well) in a unit of each head and group of columns that follows the largest of
// these products so far, so that what a key adds is held by what it weighs: a large b_j that nobody attends to, a key far above the others without a
// value, or a group of small columns beside large ones take nothing from the rest. Running maxima, sums and outputs are fp32.
//
// Bound by memory: a key is read once, at 2 * 8 * (heads per KV head) operations a byte. (int8, 64 chats of up to 8192 tokens: 102 us, 5.2 TB/s, 0.80 of a
// copy's rate; 4 bits, 8 x 100000: 112 us, 3.95 TB/s, where instructions bound it, 650 a tile; one sequence of 2001 keys 6.9 us.) What a warp does with a tile of 32 keys has to fit
// into the time that its bytes take, so: products run transposed (keys or value columns on the M = 16 side of mma.m16n8k16, up to eight query
// heads on the N = 8 side); columns of keys are dealt to lanes so that a lane's codes are neighbours in memory (the sum over columns has no order),
// values are transposed on their way out of shared memory (ldmatrix on bytes); and codes become fp16 numbers by being taken for the bits of one:
// n below 1024 in the low bits is the subnormal n 2^-24, which the matrix instructions multiply exactly. Codes are made positive for that (+128, of 4
// bits they are), and what this adds is taken off where it cannot grow: of scores, a sum over columns, in the first accumulator (-128 2^-24 sum q);
// of outputs, whose sums over keys run on and on, by a product of the same probabilities with the constant, tile by tile, once for the columns of a
// group (once for each sixteen columns took 1.5 us more of 8 x 100000 keys in 4 bits).
//
// The work is one list of tiles (sequence, KV head and block of query heads, 32 keys), cut into equal pieces for all warps of the grid whatever the
// lengths are. A warp streams its piece through a ring of its own in shared memory: TMA brings a tile's codes (cp.async, where positions are
// chosen one by one), the warp's own mbarriers say when, and no barrier of the CTA is in the loop. Whole tiles that follow in a page (or in a contiguous
// cache) are counted out when the first is sent, so that the walk and the page table are gone to once for all of them (3 us of
// 8 x 100000 keys in 4 bits). A piece that is a whole item is written out, the
// others meet inside the CTA and then, for items that several CTAs share, in quant_merge_kernel. Calls of few
// tiles are cut by items instead, each for a cluster of CTAs, and meet in its shared memory: one launch.
#pragma once
#include <cooperative_groups.h>
#include <math_constants.h>

#include <atomic>

#include "fsa_params.h"
#include "fsa_ptx.cuh"
#include "fsa_quant_dec.h"

namespace fsa {

constexpr int TILE = QUANT_TILE;
constexpr uint32_t ALL = 0xffffffffu;
constexpr int STATUS_WAIT = 1, STATUS_BAD_PAGE = 3;
// How far (base 2) a score may be above the reference maximum before that moves. (What lies 2^-126 below the reference is lost in fp32: of probabilities
// below 2^-120 of the largest some count as none.)
constexpr float LAG = 6.f;
// Units of a probability times a value scale as fp16: where one is chosen, the largest product is brought to [2^8, 2^9), and products may grow to fp16's
// end before it is chosen anew (2^6 of that are the lag's). What fp16 loses below its normal numbers is then at most 2^-33 of the largest for each key.
// (One unit for all heads and groups, chosen by scales alone, rounds away what lies 2^-14 below a scale that nobody attends to. It takes 29.8 us where
// this takes 32.3 of 37 ragged sequences with three groups, 146 and 160 of 8 x 100000 keys with four, 134.8 and 138.2 of 64 chats with 16 heads, and as
// long with up to two groups and eight heads; divisions in place of inverse_fast, which each item comes to once, cost 3 to 7 us more.)
constexpr int UNIT_TO = 8;
constexpr float FINEST = 8.507059173023462e37f;  // 2^126

template <int HD_, int FMT_, int GROUPS_, int NT_, bool HALF_>
struct Shape {
  static constexpr int HD = HD_, FMT = FMT_, GROUPS = GROUPS_, NT = NT_;  // NT: blocks of eight query heads
  static constexpr bool HALF = HALF_;              // queries and results are fp16, not bf16
  static constexpr bool INT4 = FMT == FSA_QC_INT4;
  static constexpr int GS = HD / GROUPS;           // columns of a group
  static constexpr int RB = INT4 ? HD / 2 : HD;    // bytes of a row
  static constexpr int CH = RB / 16;
  static constexpr int KSTEPS = HD / 16, MTILES = HD / 16;
  // One of a code's units, as it enters the products, and what was added to it. (Of 4 bits every other column comes 16 times as large: of
  // keys the others are multiplied, of values the result is divided.)
  static constexpr float UNIT = FMT == FSA_QC_E4M3 ? 1.f : 1.f / 16777216.f, K_UNIT = INT4 ? 16.f * UNIT : UNIT;
  static constexpr float ADDED = FMT == FSA_QC_E4M3 ? 0.f : (FMT == FSA_QC_INT8 ? 128.f : 8.f);
  static constexpr int HEADS = 8 * NT;
  static constexpr int TILE_BYTES = TILE * RB, SCALE_BYTES = TILE * GROUPS * 4;
  // a stage: keys and values, and elsewhere (swizzled tiles begin where their pattern does) their scales and what the tile is
  static constexpr int CODES = 2 * TILE_BYTES, EXTRA = 2 * SCALE_BYTES + 128;
  // (When it was chosen, before the later steps: int8, 64 chats of up to 8192 tokens, 8 warps 109.5 us, 10 99.4, 12 107; 4 bits, 8 x 100000, 133, 124
  // and 117.)
  static constexpr int WARPS = NT == 2 ? 8 : (RB == 128 ? 10 : 12), THREADS = 32 * WARPS;
  static constexpr int ALIGN = 8 * RB;             // the swizzle's pattern
  static constexpr int ROOM = 222 * 1024 / WARPS / ALIGN * ALIGN;
  static constexpr int STAGES = ROOM / (CODES + EXTRA) > 6 ? 6 : ROOM / (CODES + EXTRA);
  static constexpr int PIECE = HEADS * (HD + 2);   // floats: outputs, maxima, sums
  static constexpr int RING = (STAGES * (CODES + EXTRA) + ALIGN - 1) / ALIGN * ALIGN;
  static constexpr int SMEM = WARPS * RING + 1024;
  static_assert(STAGES >= 2 && RING >= 2 * PIECE * 4 && SMEM <= 225 * 1024, "ring");
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// The barrier counts this lane in when its copies so far have landed.
__device__ __forceinline__ void arrive_with_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void add2(float* d, const float* a) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(d[0]), "+f"(d[1])
      : "f"(a[0]), "f"(a[1]));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ float inverse_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Four codes of eight bits as two pairs of fp16: of int8 bytes (0, 2) and (1, 3) as (code + 128) 2^-24, of e4m3 (0, 1) and (2, 3).
template <int FMT>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t* lo, uint32_t* hi) {
  if constexpr (FMT == FSA_QC_INT8) {
    w ^= 0x80808080u;
    *lo = __byte_perm(w, 0, 0x4240);
    *hi = __byte_perm(w, 0, 0x4341);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(*lo), "=r"(*hi) : "r"(w));
  }
}
// Eight codes of four bits as pairs (0, 4), (1, 5), (2, 6), (3, 7) of fp16: n 2^-24, the second and fourth 16 n 2^-24.
__device__ __forceinline__ void widen8(uint32_t w, uint32_t* out) {
  const uint32_t v = w >> 8;
  out[0] = w & 0x000f000fu;
  out[1] = w & 0x00f000f0u;
  out[2] = v & 0x000f000fu;
  out[3] = v & 0x00f000f0u;
}
__device__ __forceinline__ uint32_t by16(uint32_t two) {
  const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&two), __float2half2_rn(16.f));
  return *reinterpret_cast<const uint32_t*>(&y);
}
// The same with all of them 16 n 2^-24: the matrix instructions align products by the exponents of their factors, of which a subnormal has the least
// there is, and what lies 2^-24 below the largest is lost. Of scores that was up to 4e-6 (2^-24 n: log-sum-exps off by up to 9e-7 of themselves, so by
// 1e-7); of outputs it is far below their rounding.
__device__ __forceinline__ void widen8_high(uint32_t w, uint32_t* out) {
  widen8(w, out);
  out[0] = by16(out[0]);
  out[2] = by16(out[2]);
}
// Two tiles of 16 rows x 16 bytes, transposed: lane's row address; registers 0, 1 hold bytes lane / 4 and that + 8 of rows 4 (lane % 4) .. + 3 of the
// first tile, 2 and 3 of the second.
__device__ __forceinline__ void load_transposed(uint32_t at, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

// Where a 16-byte piece of a row lies in a tile's shared memory: TMA's swizzle for rows of that many bytes. Lanes read keys by rows of lane / 4,
// pieces 2 (lane % 4) and the next (of 128 bytes), values by rows 2 (lane % 4) and so on, pieces of lane / 4: neither meets a bank twice at 128
// bytes a row; narrower rows of values twice.
template <typename S>
__device__ __forceinline__ int place_of(int row, int ch) {
  if constexpr (S::RB == 128) ch ^= row & 7;
  else if constexpr (S::RB == 64) ch ^= row >> 1 & 3;
  else ch ^= row >> 2 & 1;
  return row * S::RB + ch * 16;
}

__device__ __forceinline__ int keys_of(const QuantDecParams& p, int b) { return p.used ? min(max(p.used[b], 0), p.keys) : p.keys; }
__device__ __forceinline__ int tiles_of(int keys) { return keys > 0 ? (keys + TILE - 1) / TILE : 1; }  // (an empty sequence has its zeros written)

// A value that is the same in all lanes, for the compiler to know: branches on it are the warp's, and TMA's operands need no detour.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(ALL, x, 0); }

// Walk over the list: tile t of item (b, i), `left` of the item with this one; `keys` of the sequence, `count` of them (or of the chosen ones) to
// look at. Behind the last item b is the batch.
template <bool GATHER>
struct Walk {
  int b, i, t, left, tiles, keys, count;
  __device__ __forceinline__ void sequence(const QuantDecParams& p) {
    keys = uniform(keys_of(p, b));
    count = GATHER ? p.topk : keys;
    tiles = tiles_of(count);
  }
  __device__ __forceinline__ void next(const QuantDecParams& p) {
    ++t;
    if (--left > 0) return;
    t = 0;
    if (++i == p.items) {
      i = 0;
      if (++b < p.batch) sequence(p);
    }
    left = tiles;
  }
};

// The position that this lane's row of a tile is chosen to have, or -1.
__device__ __forceinline__ int chosen(const QuantDecParams& p, const Walk<true>& w, int lane) {
  const int at = w.t * TILE + lane;
  return w.b < p.batch && at < w.count ? p.gather[w.b * p.g_sb + at] : -1;
}

// Where the rows of a tile lie, fetched one tile ahead: of this lane's row (gather), or of the tile's first key.
struct Place {
  int position, block;
};
template <bool GATHER>
__device__ __forceinline__ Place look_up(const QuantDecParams& p, const Walk<GATHER>& w, int position) {
  Place at;
  at.position = GATHER ? position : w.t * TILE;
  if (w.b >= p.batch || at.position < 0 || at.position >= w.keys) at.position = -1;
  at.block = w.b;
  if (p.c.page_table) at.block = at.position >= 0 ? p.c.page_table[w.b * p.c.page_table_stride + (at.position >> p.page_shift)] : -1;
  return at;
}

// A tile on its way: `left` of item (b, i) with this one; of a KV head h; rows: a bit each that is there. Where positions are chosen, block and slot
// are those of the lane's row.
struct Tile {
  int block, slot, h, left, b, i, run;  // run: whole tiles that follow side by side with it
  uint32_t rows;
};

// The tile that the walk has come to. Pages hold a multiple of 32 slots, so that without gather the keys of a tile lie in one.
template <bool GATHER>
__device__ __forceinline__ void find_tile(const QuantDecParams& p, const Walk<GATHER>& w, const Place& at, Tile& tile) {
  tile.h = p.blocks == 1 ? w.i : w.i / p.blocks;
  tile.block = GATHER ? at.block : uniform(at.block);
  const bool there = at.position >= 0, known = there && (unsigned)tile.block < (unsigned)p.cache_blocks;
  if (there && !known) report_status(p.status, STATUS_BAD_PAGE);
  tile.slot = p.c.page_table ? at.position & (p.c.page_size - 1) : at.position;
  tile.left = w.left;
  tile.b = min(w.b, p.batch - 1);
  tile.i = w.i;
  tile.run = 0;
  if constexpr (GATHER) {
    tile.rows = __ballot_sync(ALL, known);
  } else {
    const int left = w.count - w.t * TILE;
    tile.rows = !known ? 0u : (left >= TILE ? ALL : (1u << left) - 1);
    const int end = p.c.page_table ? min(left, p.c.page_size - tile.slot) : left;
    if (known && end >= 2 * TILE) tile.run = end / TILE - 1;
  }
}

// Sends for a tile.
template <typename S, bool GATHER>
__device__ __forceinline__ void fetch(const QuantDecParams& p, const Tile& tile, uint8_t* stage, uint8_t* extra, uint64_t* full, int lane) {
  const FsaQuantCache& c = p.c;
  const int block = tile.block, slot = tile.slot, h = tile.h;
  const uint32_t rows = tile.rows;
  const bool lead = elect_one();
  if (lead) *reinterpret_cast<int4*>(extra + 2 * S::SCALE_BYTES) = make_int4((int)rows, tile.left, tile.b, tile.i);
  const bool here = rows >> lane & 1;  // this lane's row
  if constexpr (!GATHER) {
    if (lead) {
      if (rows) {
        mbar_arrive_expect_tx(full, 2 * S::TILE_BYTES + (p.scales_by_tma ? 2 * S::SCALE_BYTES : 0));
        tma_load_4d(stage, &p.map_k, full, 0, h, slot, block);
        tma_load_4d(stage + S::TILE_BYTES, &p.map_v, full, 0, h, slot, block);
        if (p.scales_by_tma) {
          tma_load_3d(extra, &p.map_ks, full, slot * S::GROUPS, h, block);
          tma_load_3d(extra + S::SCALE_BYTES, &p.map_vs, full, slot * S::GROUPS, h, block);
        }
      } else {
        mbar_arrive(full);
      }
    }
    if (p.scales_by_tma) return;
  } else {
    const long long k_row = here ? (long long)block * c.k_stride_b + (long long)slot * c.k_stride_s + h * c.k_stride_h : 0;
    const long long v_row = here ? (long long)block * c.v_stride_b + (long long)slot * c.v_stride_s + h * c.v_stride_h : 0;
    constexpr int ROWS = 32 / S::CH;  // that an instruction of the warp covers
    const uint32_t k_at = smem_u32(stage), v_at = k_at + S::TILE_BYTES;
    const int ch = lane % S::CH;
#pragma unroll 4
    for (int it = 0; it < TILE / ROWS; ++it) {
      const int row = it * ROWS + lane / S::CH;
      const long long k_from = __shfl_sync(ALL, k_row, row), v_from = __shfl_sync(ALL, v_row, row);
      const bool take = (rows >> row & 1) && ch < p.chunks;
      copy16(k_at + place_of<S>(row, ch), reinterpret_cast<const uint8_t*>(c.k) + (take ? k_from + ch * 16 : 0), take ? 16 : 0);
      copy16(v_at + place_of<S>(row, ch), reinterpret_cast<const uint8_t*>(c.v) + (take ? v_from + ch * 16 : 0), take ? 16 : 0);
    }
    if (lead) mbar_arrive(full);
  }
  // scales: a lane those of its own row
  const int row_slot = GATHER ? slot : slot + lane;
  const long long ks_row = block * c.ks_stride_b + row_slot * c.ks_stride_s + h * c.ks_stride_h;
  const long long vs_row = block * c.vs_stride_b + row_slot * c.vs_stride_s + h * c.vs_stride_h;
  const uint32_t ks_at = smem_u32(extra) + lane * S::GROUPS * 4, vs_at = ks_at + S::SCALE_BYTES;
#pragma unroll
  for (int g = 0; g < S::GROUPS; ++g) {
    const bool take = here && g < p.words;
    copy4(ks_at + 4 * g, reinterpret_cast<const uint32_t*>(c.k_scales) + (take ? ks_row + g : 0), take ? 4 : 0);
    copy4(vs_at + 4 * g, reinterpret_cast<const uint32_t*>(c.v_scales) + (take ? vs_row + g : 0), take ? 4 : 0);
  }
  arrive_with_copies(full);
}

// The queries of an item as B operands, with what scores are multiplied by, and their sums (of 4 bits by groups) in units of the codes.
template <typename S>
struct Queries {
  uint32_t f[S::NT][S::KSTEPS][2];
  float scale[S::NT][2];
  float sum[S::GROUPS][S::NT][2];
};

template <typename S>
__device__ __forceinline__ void load_queries(const QuantDecParams& p, int b, int item, int lane, Queries<S>& q) {
  const int r = lane >> 2, c = lane & 3, h = item / p.blocks, first = (item - h * p.blocks) * S::HEADS;
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt) {
    const int head = first + nt * 8 + r;
    const bool there = head < p.group_heads;
    const uint16_t* row = reinterpret_cast<const uint16_t*>(p.q) + b * p.q_sb + (long long)(h * p.group_heads + (there ? head : 0)) * p.q_sh;
    uint4 raw[S::KSTEPS / 2];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < S::KSTEPS / 2; ++i) {  // eight neighbouring columns
      constexpr int RUNS = S::INT4 ? S::GS / 32 : 2;  // of a group or a piece
      const int col = S::INT4 ? i / RUNS * S::GS + c * (S::GS / 4) + 8 * (i % RUNS)
                              : 16 * (S::RB == 128 ? 2 * c + i / 2 : c) + 8 * (i % 2);
      raw[i] = there && col < p.c.head_dim ? *reinterpret_cast<const uint4*>(row + col) : uint4{};
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) most = max(most, max(w[j] & 0x7fffu, w[j] >> 16 & 0x7fffu));
    }
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // the largest element goes to [2^10, 2^11); rows of zeros, and with an infinity or a NaN, stay as they are
    constexpr int MANTISSA = S::HALF ? 10 : 7, BIAS = S::HALF ? 15 : 127;
    int e = max((int)(most >> MANTISSA), 1) - BIAS - 10;
    if (most == 0 || most >= ((2u * BIAS + 1) << MANTISSA)) e = 0;
    e = min(max(e, -100), 100);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
    float sums[S::GROUPS] = {};
#pragma unroll
    for (int i = 0; i < S::KSTEPS / 2; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      uint32_t x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __half2 in = *reinterpret_cast<const __half2*>(&w[j]);
        const float a = S::HALF ? __low2float(in) : __uint_as_float(w[j] << 16), b = S::HALF ? __high2float(in) : __uint_as_float(w[j] & 0xffff0000u);
        x[j] = pack2<__half>(a * down, b * down);
        const __half2 two = *reinterpret_cast<const __half2*>(&x[j]);
        sums[S::INT4 ? i / (S::GS / 32) : 0] += __low2float(two) + __high2float(two);
      }
      uint32_t* f0 = q.f[nt][2 * i];
      uint32_t* f1 = q.f[nt][2 * i + 1];
      if constexpr (S::FMT == FSA_QC_E4M3) {
        f0[0] = x[0]; f0[1] = x[1]; f1[0] = x[2]; f1[1] = x[3];
      } else if constexpr (S::FMT == FSA_QC_INT8) {
        f0[0] = __byte_perm(x[0], x[1], 0x5410); f0[1] = __byte_perm(x[0], x[1], 0x7632);
        f1[0] = __byte_perm(x[2], x[3], 0x5410); f1[1] = __byte_perm(x[2], x[3], 0x7632);
      } else {
        f0[0] = __byte_perm(x[0], x[2], 0x5410); f0[1] = __byte_perm(x[0], x[2], 0x7632);
        f1[0] = __byte_perm(x[1], x[3], 0x5410); f1[1] = __byte_perm(x[1], x[3], 0x7632);
      }
    }
    const float mine = up * p.scale_log2 * (1.f / S::K_UNIT);
#pragma unroll
    for (int x = 0; x < 2; ++x) q.scale[nt][x] = __shfl_sync(0xffffffffu, mine, 4 * (2 * c + x));
    if constexpr (S::ADDED != 0.f) {
#pragma unroll
      for (int g = 0; g < S::GROUPS; ++g) {
        float sum = sums[g] * S::K_UNIT;
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int x = 0; x < 2; ++x) q.sum[g][nt][x] = __shfl_sync(0xffffffffu, sum, 4 * (2 * c + x));
      }
    }
  }
}

// What a warp knows about an item so far. Lanes: value columns of lane / 4, query heads 2 (lane % 4) and the next.
template <typename S>
struct State {
  float o[S::MTILES][S::NT][4];
  float centre[S::INT4 ? S::GROUPS : 1][S::NT][2];  // sum p z of this lane's keys
  float m[S::NT][2], l[S::NT][2];                   // reference maximum; sum of this lane's keys
  // What probabilities times value scales are multiplied by, and outputs with them: of each head, as what a key weighs is its probability times its
  // scale, neither alone; and of each group of columns, whose scales need not be alike.
  float unit[S::GROUPS][S::NT][2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int nt = 0; nt < S::NT; ++nt) {
#pragma unroll
      for (int t = 0; t < S::MTILES; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][nt][i] = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m[nt][x] = -CUDART_INF_F;
        l[nt][x] = 0.f;
#pragma unroll
        for (int g = 0; g < (S::INT4 ? S::GROUPS : 1); ++g) centre[g][nt][x] = 0.f;
#pragma unroll
        for (int g = 0; g < S::GROUPS; ++g) unit[g][nt][x] = FINEST;
      }
    }
  }
};

__device__ __forceinline__ float scale_of(uint32_t word, bool int4) { return __uint_as_float(int4 ? word << 16 : word); }
__device__ __forceinline__ float centre_of(uint32_t word) { return __uint_as_float(word & 0xffff0000u); }

template <typename S>
__device__ __forceinline__ void scale_outputs(State<S>& st, int g, int nt, int x, float by) {
#pragma unroll
  for (int t = g * (S::MTILES / S::GROUPS); t < (g + 1) * (S::MTILES / S::GROUPS); ++t) {
    st.o[t][nt][x] *= by;
    st.o[t][nt][x + 2] *= by;
  }
}

// Moves the reference maxima to what the tile brings. What has been added up shrinks by as much: the units take that up, so that sums of products stay
// as they are and later keys are held as finely as they deserve.
template <typename S>
__device__ __forceinline__ void move_reference(State<S>& st, const float (*s)[S::NT][4]) {
  float by[S::NT][2], back[S::NT][2];  // back: 1 where nothing has been added up
  bool beyond = false;
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float m = fmaxf(fmaxf(s[0][nt][x], s[0][nt][x + 2]), fmaxf(s[1][nt][x], s[1][nt][x + 2]));
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      m = fmaxf(m, st.m[nt][x]);
      const float down = m == -CUDART_INF_F ? 0.f : st.m[nt][x] - m;
      by[nt][x] = exp2_fast(down);
      back[nt][x] = st.m[nt][x] == -CUDART_INF_F ? 1.f : exp2_fast(-down);
      st.m[nt][x] = m;
      st.l[nt][x] *= by[nt][x];
#pragma unroll
      for (int g = 0; g < (S::INT4 ? S::GROUPS : 1); ++g) st.centre[g][nt][x] *= by[nt][x];
#pragma unroll
      for (int g = 0; g < S::GROUPS; ++g) beyond = beyond || !(st.unit[g][nt][x] * back[nt][x] <= FINEST);
    }
  }
  if (__any_sync(ALL, beyond)) {  // there is no finer one: what is left over shrinks after all
#pragma unroll
    for (int g = 0; g < S::GROUPS; ++g)
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (!(st.unit[g][nt][x] * back[nt][x] <= FINEST)) scale_outputs<S>(st, g, nt, x, by[nt][x] * FINEST * inverse_fast(st.unit[g][nt][x]));
  }
#pragma unroll
  for (int g = 0; g < S::GROUPS; ++g)
#pragma unroll
    for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) st.unit[g][nt][x] = fminf(st.unit[g][nt][x] * back[nt][x], FINEST);
}

// Chooses the units of group g by the tile's largest products of a probability and a value scale. (Their exponents are what counts: two heads a word.)
template <typename S>
__device__ __forceinline__ void choose_unit(State<S>& st, int g, const float (*e)[S::NT][4], const uint32_t (*b_words)[S::GROUPS]) {
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt) {
    float most[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x) most[x] = fmaxf(most[x], e[i >> 1][nt][x + 2 * (i & 1)] * scale_of(b_words[i][g], S::INT4));
    uint32_t both = __byte_perm(__float_as_uint(most[0]), __float_as_uint(most[1]), 0x7632);
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, d));
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float old = st.unit[g][nt][x];
      const uint32_t exponent = max(both >> (7 + 16 * x) & 0xffu, 128u + UNIT_TO - 127u);  // (no unit above FINEST)
      const float unit = fminf(old, __uint_as_float((254u + UNIT_TO - exponent) << 23));
      scale_outputs<S>(st, g, nt, x, unit < old ? unit * inverse_fast(old) : 1.f);
      st.unit[g][nt][x] = unit;
    }
  }
}

// One tile: its two halves of sixteen keys. groups: that the row has (of 96 columns in groups of 32 three).
template <typename S>
__device__ __forceinline__ void take_tile(State<S>& st, const Queries<S>& q, uint8_t* stage, const uint8_t* extra, uint32_t rows, int groups, int lane) {
  const int r = lane >> 2, c = lane & 3;
  uint32_t a_words[4][S::GROUPS], b_words[4][S::GROUPS];  // scales of rows r, r + 8, ..
  const uint32_t* scales = reinterpret_cast<const uint32_t*>(extra);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int g = 0; g < S::GROUPS; ++g) {
      a_words[i][g] = scales[(r + 8 * i) * S::GROUPS + g];
      b_words[i][g] = scales[(TILE + r + 8 * i) * S::GROUPS + g];
    }
  // ---- scores: keys r and r + 8 of each half, heads 2 c and 2 c + 1 of each block --------------------------------------
  float s[2][S::NT][4];
  constexpr int KWORDS = S::RB / 16 / S::GROUPS;  // of a group, of a lane
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[half][nt][i] = 0.f;
#pragma unroll
    for (int g = 0; g < S::GROUPS; ++g) {
      if (S::GS == 32 && g >= groups) continue;
      uint32_t w[2][KWORDS];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 16 * half + r + 8 * i;
        if constexpr (!S::INT4) {
#pragma unroll
          for (int j = 0; j < KWORDS / 4; ++j) {
            const uint4 x = *reinterpret_cast<const uint4*>(stage + place_of<S>(row, S::RB == 128 ? 2 * c + j : c));
            w[i][4 * j] = x.x; w[i][4 * j + 1] = x.y; w[i][4 * j + 2] = x.z; w[i][4 * j + 3] = x.w;
          }
        } else if constexpr (KWORDS == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(stage + place_of<S>(row, 2 * g + (c >> 1)) + 8 * (c & 1));
          w[i][0] = x.x; w[i][1] = x.y;
        } else {
          w[i][0] = *reinterpret_cast<const uint32_t*>(stage + place_of<S>(row, g) + 4 * c);
        }
      }
      float acc[S::NT][4];
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] = S::INT4 || S::ADDED == 0.f ? 0.f : -S::ADDED * q.sum[g][nt][i & 1];
#pragma unroll
      for (int j = 0; j < KWORDS; ++j) {
        if constexpr (!S::INT4) {
          uint32_t lo0, hi0, lo1, hi1;
          widen4<S::FMT>(w[0][j], &lo0, &hi0);
          widen4<S::FMT>(w[1][j], &lo1, &hi1);
#pragma unroll
          for (int nt = 0; nt < S::NT; ++nt) mma(acc[nt], lo0, lo1, hi0, hi1, q.f[nt][j][0], q.f[nt][j][1]);
        } else {
          uint32_t x0[4], x1[4];
          widen8_high(w[0][j], x0);
          widen8_high(w[1][j], x1);
          const int k = 2 * (g * KWORDS + j);
#pragma unroll
          for (int nt = 0; nt < S::NT; ++nt) {
            mma(acc[nt], x0[0], x1[0], x0[1], x1[1], q.f[nt][k][0], q.f[nt][k][1]);
            mma(acc[nt], x0[2], x1[2], x0[3], x1[3], q.f[nt][k + 1][0], q.f[nt][k + 1][1]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t word = a_words[2 * half + (i >> 1)][g];
          const float by = scale_of(word, S::INT4);
          if constexpr (S::INT4)
            s[half][nt][i] = fmaf(acc[nt][i], by, fmaf(q.sum[g][nt][i & 1], fmaf(-S::ADDED, by, centre_of(word)), s[half][nt][i]));  // (the codes' 8)
          else
            s[half][nt][i] = acc[nt][i] * by;
        }
    }
#pragma unroll
    for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[half][nt][i] *= q.scale[nt][i & 1];
  }
  const bool partial = __any_sync(ALL, rows != ALL);
  if (partial) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(rows >> (16 * half + r + 8 * (i >> 1)) & 1)) s[half][nt][i] = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int g = 0; g < S::GROUPS; ++g)
        if (!(rows >> (r + 8 * i) & 1)) b_words[i][g] = 0;
    if constexpr (S::FMT == FSA_QC_E4M3) {  // what lies in rows that are not there may be no number
      if (!(rows >> lane & 1)) {
#pragma unroll
        for (int ch = 0; ch < S::CH; ++ch) *reinterpret_cast<uint4*>(stage + S::TILE_BYTES + place_of<S>(lane, ch)) = uint4{};
      }
      fence_proxy_async_smem();  // in front of TMA's next writes
      __syncwarp();
    }
  }
  bool move = false;
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
    for (int x = 0; x < 2; ++x)
      move = move || fmaxf(fmaxf(s[0][nt][x], s[0][nt][x + 2]), fmaxf(s[1][nt][x], s[1][nt][x + 2])) > st.m[nt][x] + LAG;
  const bool moved = __any_sync(ALL, move);
  if (moved) move_reference<S>(st, s);

  // ---- probabilities -------------------------------------------------------------------------------------------------
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float m = st.m[nt][x] == -CUDART_INF_F ? 0.f : st.m[nt][x];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float& e = s[i >> 1][nt][x + 2 * (i & 1)];
        e = exp2_fast(e - m);
        st.l[nt][x] += e;
        if constexpr (S::INT4) {
#pragma unroll
          for (int g = 0; g < S::GROUPS; ++g) st.centre[g][nt][x] = fmaf(e, centre_of(b_words[i][g]), st.centre[g][nt][x]);
        }
      }
    }
  // ---- outputs: value bytes of lane / 4 and that + 8 of each piece, keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 of each half ------------
  // Row of a half that the lane names to the transposing load: such that what comes out in a register is keys (2 c, 2 c + 8, 2 c + 1, 2 c + 9), or of
  // e4m3, whose conversion takes neighbouring bytes, (2 c, 2 c + 1, 2 c + 8, 2 c + 9).
  const int kappa = lane & 15, first = S::FMT == FSA_QC_E4M3 ? kappa : kappa >> 1, second = S::FMT == FSA_QC_E4M3 ? kappa >> 1 : kappa;
  const int v_row = 16 * (lane >> 4) + 2 * (kappa >> 2) + (first & 1) + 8 * (second & 1);
  const uint32_t values = smem_u32(stage + S::TILE_BYTES) + place_of<S>(v_row, 0);
  constexpr int PIECES = S::CH / S::GROUPS;  // of sixteen bytes, of a group
  // Probabilities times scales, of fp16 results with what the rounding to fp16 leaves (else it would be as large as the result's own); of several groups
  // at a time, as far as registers go, since a vote is a wait.
  constexpr int FIT = 4 / (S::NT * (S::HALF ? 2 : 1)), AT_ONCE = S::GROUPS < FIT ? S::GROUPS : FIT;
  uint32_t pb_of[AT_ONCE][2][S::NT][2], rest_of[AT_ONCE][2][S::HALF ? S::NT : 1][2];
#pragma unroll
  for (int g = 0; g < S::GROUPS; ++g) {
    if (g % AT_ONCE == 0) {
      auto products = [&]() {  // whether one of them is beyond fp16 (or their sum, or is no number)
        __half2 sum = __float2half2_rn(0.f);
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float by = scale_of(b_words[i][g + k], S::INT4);
#pragma unroll
            for (int nt = 0; nt < S::NT; ++nt) {
              const float x = s[i >> 1][nt][2 * (i & 1)] * by * st.unit[g + k][nt][0], y = s[i >> 1][nt][2 * (i & 1) + 1] * by * st.unit[g + k][nt][1];
              const uint32_t two = pack2<__half>(x, y);
              const __half2 h = *reinterpret_cast<const __half2*>(&two);
              sum = __hadd2(sum, h);
              pb_of[k][i >> 1][nt][i & 1] = two;
              if constexpr (S::HALF) rest_of[k][i >> 1][nt][i & 1] = pack2<__half>(x - __low2float(h), y - __high2float(h));
            }
          }
        return ((*reinterpret_cast<const uint32_t*>(&sum) & 0x7fff7fffu) + 0x04000400u & 0x80008000u) != 0;
      };
      bool choose = moved;
      if (!choose) choose = __any_sync(ALL, products());
      if (choose) {
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) choose_unit<S>(st, g + k, s, b_words);
        products();
      }
    }
    if (S::GS == 32 && g >= groups) continue;
    uint32_t (&pb)[2][S::NT][2] = pb_of[g % AT_ONCE];
    uint32_t (&rest)[2][S::HALF ? S::NT : 1][2] = rest_of[g % AT_ONCE];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          pb[half][nt][i] = transposed(pb[half][nt][i]);
          if constexpr (S::HALF) rest[half][nt][i] = transposed(rest[half][nt][i]);
        }
    if constexpr (S::ADDED != 0.f) {
      // less what was added to the codes: the same products with that, which no rounding of probabilities changes; columns of a group share them
      constexpr uint32_t LESS0 = S::INT4 ? 0x80088008u : 0x80808080u, LESS1 = 0x80808080u;
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt) {
        float less[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          mma(less, LESS0, LESS1, LESS0, LESS1, pb[half][nt][0], pb[half][nt][1]);
          if constexpr (S::HALF) mma(less, LESS0, LESS1, LESS0, LESS1, rest[half][nt][0], rest[half][nt][1]);
        }
#pragma unroll
        for (int t = g * (S::MTILES / S::GROUPS); t < (g + 1) * (S::MTILES / S::GROUPS); ++t) {
          add2(st.o[t][nt], less);
          add2(st.o[t][nt] + 2, less + 2);
        }
      }
    }
    auto add = [&](int t, int half, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt) {
        mma(st.o[t][nt], a0, a1, a2, a3, pb[half][nt][0], pb[half][nt][1]);
        if constexpr (S::HALF) mma(st.o[t][nt], a0, a1, a2, a3, rest[half][nt][0], rest[half][nt][1]);
      }
    };
#pragma unroll
    for (int piece = g * PIECES; piece < (g + 1) * PIECES; ++piece) {
      uint32_t w[4];
      load_transposed(values ^ (piece * 16), w);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if constexpr (!S::INT4) {
          uint32_t lo0, hi0, lo1, hi1;
          widen4<S::FMT>(w[2 * half], &lo0, &hi0);
          widen4<S::FMT>(w[2 * half + 1], &lo1, &hi1);
          add(piece, half, lo0, lo1, hi0, hi1);
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t f[4];  // even and odd columns of keys 2 c and 2 c + 1, of 2 c + 8 and 2 c + 9
            widen8(w[2 * half + k], f);
            add(2 * piece + k, half, f[0], f[1], f[2], f[3]);
          }
        }
      }
    }
  }
}

// Sums over the lanes that share heads, and the outputs in the values' own units, two neighbouring columns in each pair (column_of).
template <typename S>
__device__ __forceinline__ void settle(State<S>& st, int lane) {
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) st.l[nt][x] += __shfl_xor_sync(0xffffffffu, st.l[nt][x], d);
      if constexpr (S::INT4) {
#pragma unroll
        for (int g = 0; g < S::GROUPS; ++g)
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) st.centre[g][nt][x] += __shfl_xor_sync(0xffffffffu, st.centre[g][nt][x], d);
      }
#pragma unroll
      for (int t = 0; t < S::MTILES; ++t) {
        const float by = inverse_fast(st.unit[t / (S::MTILES / S::GROUPS)][nt][x]);
        const float z = S::INT4 ? st.centre[S::INT4 ? t / (S::GS / 16) : 0][nt][x] : 0.f;
        // (one after the other: of values from 2^111 on their product is beyond fp32)
        float a = fmaf(st.o[t][nt][x] * (1.f / S::UNIT), by, z), b = fmaf(st.o[t][nt][x + 2] * (1.f / S::K_UNIT), by, z);
        if constexpr (!S::INT4) {  // columns r and r + 8: even rows take the neighbour's first, odd ones its second
          const float other = __shfl_xor_sync(ALL, lane & 4 ? a : b, 4);
          if (lane & 4) a = other; else b = other;
        }
        st.o[t][nt][x] = a;
        st.o[t][nt][x + 2] = b;
      }
    }
}

// The first of this lane's two columns in tile t, once settled.
template <typename S>
__device__ __forceinline__ int column_of(int t, int r) {
  return 16 * t + (S::INT4 ? 2 * r : (r & 6) + 8 * (r & 1));
}

__device__ __forceinline__ void store_two(const QuantDecParams& p, bool half, uint16_t* row, int col, float a, float b) {
  if (col < p.c.head_dim) *reinterpret_cast<uint32_t*>(row + col) = half ? pack2<__half>(a, b) : pack2<__nv_bfloat16>(a, b);
}

// A whole item.
template <typename S>
__device__ __forceinline__ void write_out(const QuantDecParams& p, const State<S>& st, int b, int item, int lane) {
  const int r = lane >> 2, c = lane & 3, h = item / p.blocks, first = (item - h * p.blocks) * S::HEADS;
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int head = first + nt * 8 + 2 * c + x;
      if (head >= p.group_heads) continue;
      const float l = st.l[nt][x], by = l == 0.f ? 0.f : 1.f / l;
      const long long hq = (long long)h * p.group_heads + head;
      uint16_t* row = reinterpret_cast<uint16_t*>(p.out) + b * p.o_sb + hq * p.o_sh;
#pragma unroll
      for (int t = 0; t < S::MTILES; ++t) store_two(p, S::HALF, row, column_of<S>(t, r), st.o[t][nt][x] * by, st.o[t][nt][x + 2] * by);
      if (r == 0) p.lse[b * p.l_sb + hq * p.l_sh] = l == 0.f ? -CUDART_INF_F : (st.m[nt][x] + log2f(l)) * CUDART_LN2_F;
    }
}

// A part of one: outputs as they are, maxima, sums.
template <typename S>
__device__ __forceinline__ void write_piece(float* to, const State<S>& st, int lane) {
  const int r = lane >> 2, c = lane & 3;
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int head = nt * 8 + 2 * c + x;
#pragma unroll
      for (int t = 0; t < S::MTILES; ++t)
        *reinterpret_cast<float2*>(to + head * S::HD + column_of<S>(t, r)) = make_float2(st.o[t][nt][x], st.o[t][nt][x + 2]);
      if (r == 0) {
        to[S::HEADS * S::HD + head] = st.m[nt][x];
        to[S::HEADS * (S::HD + 1) + head] = st.l[nt][x];
      }
    }
}

// Four columns of a head out of several parts. `part(i)`: where part i lies. AT_ONCE parts are fetched at a time: one by one their latencies were
// most of what a merge took.
template <int HD, int HEADS, int AT_ONCE, typename F>
__device__ __forceinline__ float4 join(int parts, int head, int col, F&& part, float* m_out, float* l_out) {
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -CUDART_INF_F, l = 0.f;
  for (int i0 = 0; i0 < parts; i0 += AT_ONCE) {
    float mi[AT_ONCE], li[AT_ONCE];
    float4 v[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      mi[i] = -CUDART_INF_F;
      li[i] = 0.f;
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + i < parts) {
        const float* x = part(i0 + i);
        mi[i] = x[HEADS * HD + head];
        li[i] = x[HEADS * (HD + 1) + head];
        v[i] = *reinterpret_cast<const float4*>(x + head * HD + col);
      }
    }
    float now = m;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) now = fmaxf(now, mi[i]);
    const float before = m == -CUDART_INF_F ? 0.f : exp2_fast(m - now);  // (0 times a NaN is one)
    m = now;
    l *= before;
    o.x *= before;
    o.y *= before;
    o.z *= before;
    o.w *= before;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const float by = mi[i] == -CUDART_INF_F ? 0.f : exp2_fast(mi[i] - m);
      o.x = fmaf(v[i].x, by, o.x);
      o.y = fmaf(v[i].y, by, o.y);
      o.z = fmaf(v[i].z, by, o.z);
      o.w = fmaf(v[i].w, by, o.w);
      l = fmaf(li[i], by, l);
    }
  }
  *m_out = m;
  *l_out = l;
  return o;
}

__device__ __forceinline__ void finish(const QuantDecParams& p, bool half, int b, int item, int heads, int head, int col, float4 o, float m, float l) {
  const int h = item / p.blocks, at = (item - h * p.blocks) * heads + head;
  if (at >= p.group_heads) return;
  const float by = l == 0.f ? 0.f : 1.f / l;
  const long long hq = (long long)h * p.group_heads + at;
  uint16_t* row = reinterpret_cast<uint16_t*>(p.out) + b * p.o_sb + hq * p.o_sh;
  store_two(p, half, row, col, o.x * by, o.y * by);
  store_two(p, half, row, col + 2, o.z * by, o.w * by);
  if (col == 0) p.lse[b * p.l_sb + hq * p.l_sh] = l == 0.f ? -CUDART_INF_F : (m + log2f(l)) * CUDART_LN2_F;
}

template <typename S, bool GATHER>
__global__ void __launch_bounds__(S::THREADS, 1) quant_decode_kernel(const __grid_constant__ QuantDecParams p) {
  after_previous();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full_s[S::WARPS][S::STAGES];
  __shared__ int abort_s;
  // what a warp's first piece (of an item that began before it) and its last one (of an item that goes on behind it) are
  __shared__ const float* part_s[S::WARPS][2];
  __shared__ int2 item_s[S::WARPS];  // of the last piece: sequence, item
  __shared__ unsigned pieces_s[3];
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

  uint64_t* full = full_s[warp];
  // a stage is there when its codes are (lane 0, with TMA's bytes) and its scales (the same, or each lane's copies)
  if (lane < S::STAGES) mbar_init(full + lane, p.scales_by_tma ? 1 : 33);
  if (!GATHER && tid == 0) {
    tma_prefetch_desc(&p.map_k);
    tma_prefetch_desc(&p.map_v);
    if (p.scales_by_tma) {
      tma_prefetch_desc(&p.map_ks);
      tma_prefetch_desc(&p.map_vs);
    }
  }
  if (tid == 0) abort_s = 0;
  if (tid < 3) pieces_s[tid] = 0;
  if (tid < 2 * S::WARPS) part_s[tid >> 1][tid & 1] = reinterpret_cast<const float*>(smem + (tid >> 1) * S::RING);
  mbar_fence_init();
  __syncthreads();

  // ---- where this warp begins ------------------------------------------------------------------------------------------
  // The first `warps` warps of the grid have equal pieces of the list, of at least a tile; the others none. Every warp adds up the
  // lengths by itself, a lane those of neighbouring sequences: no warp waits for another before it has its first tiles under way.
  // (Should someone write lengths meanwhile, which spoils the results, every index still stays in bounds and every loop ends. A cluster's warp reads its
  // sequence's once, so that it has no more than one piece, which its ring holds. In the list a warp reads them more than once and may come to another
  // cut than its neighbour: its walk ends by its own count, behind the last sequence there are no keys, and pieces that a neighbour expects and nobody
  // wrote are looked for where there is memory.)
  const long long g_warp = (long long)blockIdx.x * S::WARPS + warp;
  Walk<GATHER> walk;
  int mine = 0;
  if (p.cluster) {
    // an item's tiles go round the CTAs of its cluster first, then round their warps
    const int n = (int)blockIdx.x / p.cluster, w = warp * p.cluster + (int)blockIdx.x % p.cluster;
    walk.b = n / p.items;
    walk.i = n - walk.b * p.items;
    walk.sequence(p);
    mine = quant_cluster_share(walk.tiles, p.cluster * S::WARPS, w, &walk.t);
  } else {
    auto tiles_at = [&](int b) { return tiles_of(GATHER ? p.topk : keys_of(p, b)); };
    const bool alike = GATHER || !p.used;
    const int per = (p.batch + 31) / 32, b1 = min(min(lane * per, p.batch) + per, p.batch);
    int b0 = min(lane * per, p.batch);
    long long own = 0;
    // (of more than 32 sequences a lane the warp reads the lengths of each lane's in turn, side by side: 4096 sequences of up to 64 keys 182.7 us, so
    // 168.5; 1024 of up to 256 103 and 111)
    constexpr int FEW = 32;
    if (alike) {
      own = (long long)(b1 - b0) * tiles_at(0);
    } else if (per <= FEW) {
      for (int b = b0; b < b1; ++b) own += tiles_at(b);
    } else {
      for (int of = 0; of < 32; ++of) {
        const int end = min((of + 1) * per, p.batch);
        unsigned low = 0, high = 0;
        for (int b = of * per + lane; b < end; b += 32) {
          const unsigned n = tiles_at(b);
          low += n & 0xffff;
          high += n >> 16;
        }
        low = __reduce_add_sync(ALL, low);
        high = __reduce_add_sync(ALL, high);
        if (lane == of) own = ((long long)high << 16) + low;
      }
    }
    long long upto = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(ALL, upto, d);
      if (lane >= d) upto += o;
    }
    const long long total = __shfl_sync(ALL, upto, 31) * p.items, warps = min(total, (long long)p.ctas * S::WARPS);
    if (g_warp < warps) {
      // total * g_warp / warps and that of the next warp, without a division in 64 bits where none is needed
      long long at;
      if (total < 0x7fffffffll) {
        const unsigned w = (unsigned)warps, g = (unsigned)g_warp, each = (unsigned)total / w, more = (unsigned)total - each * w;
        at = each * g + more * g / w;
        mine = (int)(each * (g + 1) + more * (g + 1) / w - (unsigned)at);
      } else {
        at = total * g_warp / warps;
        mine = (int)min(total * (g_warp + 1) / warps - at, 0x7fffffffll);
      }
      long long from = (upto - own) * p.items;
      bool have = at >= from && at < upto * p.items;
      int where[3] = {0, 0, 0};
      if (!alike && per > FEW) {  // the lane's sequences, 32 at a time
        const int of = __ffs(__ballot_sync(ALL, have)) - 1, end = min((of + 1) * per, p.batch);
        from = __shfl_sync(ALL, from, of);
        for (int first = of * per; first < end; first += 32) {
          b0 = first + lane;
          const long long mine_too = b0 < end ? (long long)tiles_at(b0) * p.items : 0;
          long long until = mine_too;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const long long o = __shfl_up_sync(ALL, until, d);
            if (lane >= d) until += o;
          }
          have = at >= from + until - mine_too && at < from + until;
          if (__any_sync(ALL, have)) {
            from += until - mine_too;
            break;
          }
          from += __shfl_sync(ALL, until, 31);
        }
      }
      if (have) {
        int b = b0, tiles = tiles_at(b);
        if (alike) {
          const long long skip = (at - from) / ((long long)tiles * p.items);
          b += (int)skip;
          from += skip * tiles * p.items;
        } else {
          while (b + 1 < b1 && at >= from + (long long)tiles * p.items) {
            from += (long long)tiles * p.items;
            tiles = tiles_at(++b);
          }
        }
        where[0] = b;
        // (below tiles * items, which fits 31 bits but for sequences that no pool holds)
        const unsigned long long rest = (unsigned long long)(at - from);
        where[1] = rest < 0x7fffffffull ? (int)((unsigned)rest / (unsigned)tiles) : (int)(rest / (unsigned)tiles);
        where[2] = (int)(rest - (unsigned long long)where[1] * (unsigned)tiles);
        where[1] = min(where[1], p.items - 1);
      }
      const int src = __ffs(__ballot_sync(ALL, have)) - 1;
      walk.b = __shfl_sync(ALL, where[0], src);
      walk.i = __shfl_sync(ALL, where[1], src);
      walk.t = __shfl_sync(ALL, where[2], src);
    }
  }

  // ---- this warp's tiles -----------------------------------------------------------------------------------------------
  uint8_t* ring = smem + warp * S::RING;
  uint8_t* extras = ring + S::STAGES * S::CODES;
  float* own_pieces = p.pieces + (long long)blockIdx.x * 2 * S::PIECE;
  if (mine > 0) {
    if (!p.cluster) walk.sequence(p);
    walk.left = max(walk.tiles - walk.t, 1);
    int sent = 0, into = 0, chosen_next = -1;  // into: the stage that the next copies take
    Place place;
    Tile tile;
    tile.run = 0;
    if constexpr (GATHER) {
      place = look_up(p, walk, chosen(p, walk, lane));
      Walk<GATHER> ahead = walk;
      ahead.next(p);
      chosen_next = chosen(p, ahead, lane);
    } else {
      place = look_up(p, walk, 0);
    }
    auto send = [&]() {
      if (sent == mine) return;
      ++sent;
      if (!GATHER && tile.run > 0) {
        --tile.run;
        --tile.left;
        tile.slot += TILE;
      } else {
        find_tile(p, walk, place, tile);
        walk.t += tile.run;
        walk.left -= tile.run;
        walk.next(p);
        place = look_up(p, walk, chosen_next);
        if constexpr (GATHER) {
          Walk<GATHER> ahead = walk;
          ahead.next(p);
          chosen_next = chosen(p, ahead, lane);
        }
      }
      fetch<S, GATHER>(p, tile, ring + into * S::CODES, extras + into * S::EXTRA, full + into, lane);
      into = into + 1 == S::STAGES ? 0 : into + 1;
    };
    int2 item = make_int2(walk.b, walk.i);
    int left = walk.left, done = 0, at = 0;
    uint32_t phase = 0;
    bool whole = walk.t == 0;  // the item began in this warp
#pragma unroll 1
    for (int i = 0; i < S::STAGES - 1; ++i) send();
    Queries<S> q;
    State<S> st;
    auto arrived = [&]() { return mbar_wait_uniform(full + at, phase, &abort_s); };
    bool ok = true;
    for (;;) {
      load_queries<S>(p, item.x, item.y, lane, q);
      st.clear();
      const int n = min(left, mine - done);
      for (int i = 0; i < n; ++i) {
        // all lanes see the tile, and are done with the one whose place the next copies take
        ok = arrived();
        if (!ok) break;
        __syncwarp();
        send();
        uint8_t* extra = extras + at * S::EXTRA;
        take_tile<S>(st, q, ring + at * S::CODES, extra, *reinterpret_cast<const uint32_t*>(extra + 2 * S::SCALE_BYTES), p.words, lane);
        ++done;
        if (++at == S::STAGES) {
          at = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      const bool ends = n == left, last = done == mine;
      settle<S>(st, lane);
      if (whole && ends && !p.cluster) {
        write_out<S>(p, st, item.x, item.y, lane);
      } else {
        // the ring is free behind the last tile; a first piece that is done before goes through the workspace
        float* to = last ? reinterpret_cast<float*>(ring) : p.pieces + ((long long)p.ctas * 2 + g_warp) * S::PIECE;
        __syncwarp();
        write_piece<S>(to, st, lane);
        if (lane == 0) {
          const bool begins = whole && !p.cluster;
          part_s[warp][begins] = to;
          atomicOr(&pieces_s[begins], 1u << warp);
          if (begins)
            item_s[warp] = item;
          else if (ends)
            atomicOr(&pieces_s[2], 1u << warp);
        }
      }
      if (last) break;
      whole = true;
      ok = arrived();  // the next item says what it is
      if (!ok) break;
      const int4 what = *reinterpret_cast<const int4*>(extras + at * S::EXTRA + 2 * S::SCALE_BYTES);
      left = uniform(what.y);
      item = make_int2(what.z, what.w);
    }
    if (!ok) {  // a wait ran out: say so, and wait for what else is under way
      report_status(p.status, STATUS_WAIT);
      for (int i = done + 1; i < sent; ++i) mbar_wait_uniform(full + i % S::STAGES, i / S::STAGES & 1, &abort_s);
    }
  }
  __syncthreads();
  if (p.cluster) {  // the CTA's warps join their pieces behind warp 0's, the cluster's CTAs a share of the columns each
    auto cluster = cooperative_groups::this_cluster();
    float* joined = reinterpret_cast<float*>(smem) + S::PIECE;
    const int parts = abort_s ? 0 : __popc(pieces_s[0]), share = S::HEADS * S::HD / 4 / p.cluster, rank = (int)blockIdx.x % p.cluster;
    const int n = (int)blockIdx.x / p.cluster;
#pragma unroll 1
    for (int last = 0; last < 2; ++last) {
      auto part = [&](int i) { return last ? static_cast<const float*>(cluster.map_shared_rank(joined, i)) : part_s[i][0]; };
      const int j0 = last ? rank * share : 0, j1 = last ? j0 + share : S::HEADS * S::HD / 4;
#pragma unroll 1
      for (int j = j0 + tid; j < j1; j += S::THREADS) {
        const int head = j / (S::HD / 4), col = 4 * (j % (S::HD / 4));
        float m, l;
        const float4 o = join<S::HD, S::HEADS, 8>(last ? p.cluster : parts, head, col, part, &m, &l);
        if (last) {
          finish(p, S::HALF, n / p.items, n % p.items, S::HEADS, head, col, o, m, l);
        } else {
          *reinterpret_cast<float4*>(joined + head * S::HD + col) = o;
          if (col == 0) {
            joined[S::HEADS * S::HD + head] = m;
            joined[S::HEADS * (S::HD + 1) + head] = l;
          }
        }
      }
      cluster.sync();  // behind the last one nobody leaves while another CTA may still read its shared memory
    }
    return;
  }
  if (abort_s) {  // a wait ran out: nothing to join
    if (tid == 0) p.shared[blockIdx.x] = make_int2(0, -1);
    return;
  }

  // ---- items that several warps share ------------------------------------------------------------------------------------
  // Runs of pieces of one item, in the order of the warps.
  const unsigned firsts = pieces_s[0], lasts = pieces_s[1], ends_in = pieces_s[2];  // a bit a warp: first piece, last piece, the first one's item ends
  int2 told = make_int2(0, -1);
  const int highest = 31 - __clz(firsts | lasts);
  // a run goes from a warp's last piece (an item that begins there), or from the CTA's first piece of all, to the next warp in which an item ends
#pragma unroll 1
  for (int w0 = firsts & 1 ? -1 : (lasts ? __ffs(lasts) - 1 : 32); w0 < 32;) {
    const int k0 = w0 >= 0, begin = max(w0, 0);
    const unsigned later = ends_in & (k0 ? ~0u << begin << 1 : ~0u);
    const bool ends = later != 0, whole = k0 && ends;
    const int last = ends ? __ffs(later) - 1 : highest;
    auto part = [&](int i) { return i == 0 ? part_s[begin][k0] : part_s[begin + i][0]; };
    const int2 item = k0 ? item_s[begin] : make_int2(0, 0);
    float* to = own_pieces + (k0 ? S::PIECE : 0);
    {
#pragma unroll 1
      for (int j = tid; j < S::HEADS * S::HD / 4; j += S::THREADS) {
        const int head = j / (S::HD / 4), col = 4 * (j % (S::HD / 4));
        float m, l;
        const float4 o = join<S::HD, S::HEADS, 8>(last - begin + 1, head, col, part, &m, &l);
        if (whole) {
          finish(p, S::HALF, item.x, item.y, S::HEADS, head, col, o, m, l);
        } else {
          *reinterpret_cast<float4*>(to + head * S::HD + col) = o;
          if (col == 0) {
            to[S::HEADS * S::HD + head] = m;
            to[S::HEADS * (S::HD + 1) + head] = l;
          }
        }
      }
      if (!k0) told.x = ends ? 1 : 2;
      else if (!ends) told.y = item.x * p.items + item.y;
    }
    const unsigned next = lasts & (k0 ? ~0u << begin << 1 : ~0u);
    w0 = next ? __ffs(next) - 1 : 32;
  }
  if (tid == 0) p.shared[blockIdx.x] = told;
}

// Items that several CTAs share: a block takes a quarter of the columns of the item that begins in its CTA, if it goes on in others.
constexpr int MERGE_THREADS = 128, SLICES = 4;

template <int HD, int HEADS, bool HALF>
__global__ void __launch_bounds__(MERGE_THREADS) quant_merge_kernel(const __grid_constant__ QuantDecParams p) {
  after_previous();
  __shared__ int end_s;
  const int cta = blockIdx.x / SLICES, slice = blockIdx.x % SLICES;
  if (threadIdx.x == 0) end_s = p.ctas;
  // (what the next CTAs say is asked for with the item: two trips to memory in one)
  auto says = [&](int c) { return c < p.ctas ? p.shared[c].x : 0; };
  int c = cta + 1 + threadIdx.x, said = says(c);
  const int item = p.shared[cta].y;
  if (item < 0) return;
  __syncthreads();
  for (int c0 = cta + 1; c0 < p.ctas; c0 += MERGE_THREADS) {
    const bool ends = said == 1;
    if (ends) atomicMin(&end_s, c);
    if (__syncthreads_or(ends)) break;
    c += MERGE_THREADS;
    said = says(c);
  }
  constexpr int PIECE = HEADS * (HD + 2);
  const int last = min(end_s, p.ctas - 1);
  auto part = [&](int i) { return p.pieces + ((long long)(cta + i) * 2 + (i == 0)) * PIECE; };
  constexpr int WIDE = HD / 4 / SLICES;  // groups of four columns of a slice
  for (int j = threadIdx.x; j < HEADS * WIDE; j += MERGE_THREADS) {
    const int head = j / WIDE, col = 4 * (slice * WIDE + j % WIDE);
    float m, l;
    const float4 o = join<HD, HEADS, 8>(last - cta + 1, head, col, part, &m, &l);
    finish(p, HALF, item / p.items, item % p.items, HEADS, head, col, o, m, l);
  }
}

// ----------------------------------------------------------------------------------------------
// Launches
// ----------------------------------------------------------------------------------------------
template <typename S, bool GATHER>
cudaError_t launch_both(const QuantDecParams& p, cudaStream_t stream) {
  static std::atomic<unsigned long long> opted_in{0};
  auto kern = quant_decode_kernel<S, GATHER>;
  if (cudaError_t e = smem_opt_in(kern, S::SMEM, opted_in); e != cudaSuccess) return e;
  if (p.cluster) return launch_early(kern, (unsigned)(p.batch * p.items * p.cluster), S::THREADS, S::SMEM, stream, p.cluster, p);
  cudaError_t e = launch_early(kern, (unsigned)p.ctas, S::THREADS, S::SMEM, stream, 1, p);
  if (e != cudaSuccess) return e;
  return launch_early(quant_merge_kernel<S::HD, S::HEADS, S::HALF>, (unsigned)(p.ctas * SLICES), MERGE_THREADS, 0, stream, 1, p);
}

// f with the shape that a cache and a number of query heads a KV head need.
template <int FMT, typename F>
auto for_shape(const FsaQuantCache& c, int dtype, int group_heads, F&& f) {
  auto with_heads = [&](auto hd, auto groups) {
    if (dtype == FSA_DT_FP16)
      return group_heads > 8 ? f(Shape<hd(), FMT, groups(), 2, true>{}) : f(Shape<hd(), FMT, groups(), 1, true>{});
    return group_heads > 8 ? f(Shape<hd(), FMT, groups(), 2, false>{}) : f(Shape<hd(), FMT, groups(), 1, false>{});
  };
  auto with_width = [&](auto hd) {
    using std::integral_constant;
    if constexpr (FMT != FSA_QC_INT4)
      return with_heads(hd, integral_constant<int, 1>{});
    else
      return c.group == 32 ? with_heads(hd, integral_constant<int, hd() / 32>{}) : with_heads(hd, integral_constant<int, hd() / 64>{});
  };
  return c.head_dim <= 64 ? with_width(std::integral_constant<int, 64>{}) : with_width(std::integral_constant<int, 128>{});
}

template <int FMT>
QuantDecShape quant_decode_shape(const FsaQuantCache& c, int dtype, int group_heads) {
  return for_shape<FMT>(c, dtype, group_heads, [](auto s) { return QuantDecShape{decltype(s)::WARPS, decltype(s)::PIECE, decltype(s)::HEADS}; });
}
template <int FMT>
cudaError_t launch_quant_decode(const QuantDecParams& p, int dtype, cudaStream_t stream) {
  return for_shape<FMT>(p.c, dtype, p.group_heads, [&](auto s) {
    return p.gather ? launch_both<decltype(s), true>(p, stream) : launch_both<decltype(s), false>(p, stream);
  });
}

}  // namespace fsa
