// Decode attention over a cache whose rows carry their own scales (fsa_quant_cache.cu): one query position per sequence.
//
// With codes k^, v^ and a row's scales a_j (keys), b_j (values)
//   s_jh = c (q_h . k^_j) a_j            8 bits            c = softmax_scale log2(e)
//   s_jh = c sum_g (q_hg . (k^_jg - 8)) a_jg + (sum q_hg) z_jg     4 bits, group by group
//   o_h  = sum_j p_jh b_j v^_j / sum_j p_jh,  p_jh = 2^(s_jh - m_h)
// so no value is ever rounded on its way: codes are exact in fp16, products and sums are those of the matrix instructions in fp32, scales are
// applied to scores and to probabilities. The queries enter as fp16 too: a bf16 row is multiplied by a power of two that brings its largest
// element to [1, 2) (exact but for elements 2^-14 below it, whose lost bits are below the fp32 sum's own), probabilities as fp16 (2^-12) times b_j times a power
// of two that keeps them in range. Running maxima, sums and outputs are fp32.
//
// Bound by memory: a key is read once, at 2 * 8 * (heads per KV head) operations a byte. What a warp does with a tile of 32 keys has to fit
// into the time that its bytes take, so: products run transposed (keys or value columns on the M = 16 side of mma.m16n8k16, up to eight query
// heads on the N = 8 side); columns are dealt to lanes so that a lane's codes are neighbours in memory (the sum over columns has no order), and
// value columns so that the two keys of a register pair are two words of one lane; codes become fp16 by inserting them into the bits of 1024.
//
// The work is one list of tiles (sequence, KV head and block of query heads, 32 keys), cut into equal pieces for all warps of the grid whatever the
// lengths are. A warp streams its piece through a ring of its own in shared memory: TMA brings a tile's codes (cp.async, where positions are
// chosen one by one), the warp's own mbarriers say when, and no barrier of the CTA is in the loop. A piece that is a whole item is written out, the
// others meet inside the CTA and then, for items that several CTAs share, in quant_merge_kernel.
#include <math_constants.h>

#include <atomic>
#include <type_traits>

#include "fsa_aux.h"
#include "fsa_params.h"
#include "fsa_ptx.cuh"
#include "fsa_quant_cache.h"

namespace fsa {

namespace {

constexpr int TILE = 32;             // keys
constexpr uint32_t ALL = 0xffffffffu;
constexpr int STATUS_WAIT = 1, STATUS_BAD_PAGE = 3;
constexpr float LAG = 6.f;           // how far (base 2) a score may be above the reference maximum before that moves
constexpr float MOST_SCALE = 512.f;  // and a value scale above 1: 2^6 * 2^9 is within fp16

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
  bool scales_by_tma;
  float scale_log2;
};

template <int HD_, int FMT_, int GROUPS_, int NT_, bool HALF_>
struct Shape {
  static constexpr int HD = HD_, FMT = FMT_, GROUPS = GROUPS_, NT = NT_;  // NT: blocks of eight query heads
  static constexpr bool HALF = HALF_;              // queries and results are fp16, not bf16
  static constexpr bool INT4 = FMT == FSA_QC_INT4;
  static constexpr int GS = HD / GROUPS;           // columns of a group
  static constexpr int RB = INT4 ? HD / 2 : HD;    // bytes of a row
  static constexpr int CH = RB / 16;
  static constexpr int KSTEPS = HD / 16, MTILES = HD / 16;
  static constexpr int HEADS = 8 * NT;
  static constexpr int TILE_BYTES = TILE * RB, SCALE_BYTES = TILE * GROUPS * 4;
  // a stage: keys and values, and elsewhere (swizzled tiles begin where their pattern does) their scales and what the tile is
  static constexpr int CODES = 2 * TILE_BYTES, EXTRA = 2 * SCALE_BYTES + 128;
  static constexpr int WARPS = NT == 1 ? 12 : 8, THREADS = 32 * WARPS;
  static constexpr int ALIGN = 8 * RB;             // the swizzle's pattern
  static constexpr int ROOM = 222 * 1024 / WARPS / ALIGN * ALIGN;
  static constexpr int STAGES = ROOM / (CODES + EXTRA) > 6 ? 6 : ROOM / (CODES + EXTRA);
  static constexpr int PIECE = HEADS * (HD + 2);   // floats: outputs, maxima, sums
  static constexpr int RING = (STAGES * (CODES + EXTRA) + ALIGN - 1) / ALIGN * ALIGN;
  static constexpr int SMEM = WARPS * RING + 1024;
  static_assert(STAGES >= 2 && RING >= PIECE * 4 && SMEM <= 225 * 1024, "ring");
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
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// Four codes of eight bits as two pairs, bytes (0, 1) and (2, 3).
template <int FMT>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t* lo, uint32_t* hi) {
  if constexpr (FMT == FSA_QC_INT8) {
    w ^= 0x80808080u;  // code + 128
    *lo = sub2(__byte_perm(w, 0x64646464u, 0x4140), 0x64806480u);  // 1024 + code + 128, less 1152
    *hi = sub2(__byte_perm(w, 0x64646464u, 0x4342), 0x64806480u);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(*lo), "=r"(*hi) : "r"(w));
  }
}
// Eight codes of four bits, less 8, as pairs (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ void widen8(uint32_t w, uint32_t* out) {
  const uint32_t v = w >> 8;
  out[0] = sub2((w & 0x000f000fu) | 0x64006400u, 0x64086408u);                // 1024 + n, less 1032
  out[1] = fma2((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u);   // (1024 + 16 n) / 16 - 72
  out[2] = sub2((v & 0x000f000fu) | 0x64006400u, 0x64086408u);
  out[3] = fma2((v & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u);
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

// Walk over the list: tile t of item (b, i); `keys` of the sequence, `count` of them (or of the chosen ones) to look at.
template <bool GATHER>
struct Walk {
  int b, i, t, tiles, keys, count;
  __device__ __forceinline__ void sequence(const QuantDecParams& p) {
    keys = uniform(keys_of(p, b));
    count = GATHER ? p.topk : keys;
    tiles = tiles_of(count);
  }
  __device__ __forceinline__ void next(const QuantDecParams& p) {
    if (++t < tiles) return;
    t = 0;
    if (++i < p.items) return;
    i = 0;
    if (++b < p.batch) sequence(p);
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

// Sends for a tile. Pages hold a multiple of 32 slots, so that without gather the keys of a tile lie in one.
template <typename S, bool GATHER>
__device__ __forceinline__ void fetch(const QuantDecParams& p, const Walk<GATHER>& w, const Place& at, uint8_t* stage, uint8_t* extra, uint64_t* full,
                                      int lane) {
  const FsaQuantCache& c = p.c;
  const int h = p.blocks == 1 ? w.i : w.i / p.blocks;
  const int block = GATHER ? at.block : uniform(at.block);
  const bool there = at.position >= 0, known = there && (unsigned)block < (unsigned)p.cache_blocks;
  if (there && !known) report_status(p.status, STATUS_BAD_PAGE);
  const int slot = c.page_table ? at.position & (c.page_size - 1) : at.position;
  uint32_t rows;
  if constexpr (GATHER) {
    rows = __ballot_sync(ALL, known);
  } else {
    const int left = w.count - w.t * TILE;
    rows = !known ? 0u : (left >= TILE ? ALL : (1u << left) - 1);
  }
  const bool lead = elect_one();
  if (lead) *reinterpret_cast<int4*>(extra + 2 * S::SCALE_BYTES) = make_int4((int)rows, w.t + 1 == w.tiles, w.b, w.i);
  const bool here = rows >> lane & 1;  // this lane's row
  if constexpr (!GATHER) {
    if (lead) {
      if (known) {
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

// The queries of an item as B operands, with what scores are multiplied by; of 4 bits their sums by groups.
template <typename S>
struct Queries {
  uint32_t f[S::NT][S::KSTEPS][2];
  float scale[S::NT][2];
  float sum[S::INT4 ? S::GROUPS : 1][S::NT][2];
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
    // bf16: the exponent of the largest element; rows of zeros, and with an infinity or a NaN, as they are
    int e = 0;
    if constexpr (!S::HALF) {
      e = (int)(most >> 7) - 127;
      if (most < 0x80u || most >= 0x7f80u) e = 0;
      e = min(max(e, -100), 126);
    }
    const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
    float sums[S::GROUPS] = {};
#pragma unroll
    for (int i = 0; i < S::KSTEPS / 2; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      uint32_t x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = w[j];
        if constexpr (!S::HALF) x[j] = pack2<__half>(__uint_as_float(w[j] << 16) * down, __uint_as_float(w[j] & 0xffff0000u) * down);
        if constexpr (S::INT4) {
          const __half2 two = *reinterpret_cast<const __half2*>(&x[j]);
          sums[i / (S::GS / 32)] += __low2float(two) + __high2float(two);
        }
      }
      uint32_t* f0 = q.f[nt][2 * i];
      uint32_t* f1 = q.f[nt][2 * i + 1];
      if constexpr (!S::INT4) {
        f0[0] = x[0]; f0[1] = x[1]; f1[0] = x[2]; f1[1] = x[3];
      } else {
        f0[0] = __byte_perm(x[0], x[2], 0x5410); f0[1] = __byte_perm(x[0], x[2], 0x7632);
        f1[0] = __byte_perm(x[1], x[3], 0x5410); f1[1] = __byte_perm(x[1], x[3], 0x7632);
      }
    }
    const float mine = up * p.scale_log2;
#pragma unroll
    for (int x = 0; x < 2; ++x) q.scale[nt][x] = __shfl_sync(0xffffffffu, mine, 4 * (2 * c + x));
    if constexpr (S::INT4) {
#pragma unroll
      for (int g = 0; g < S::GROUPS; ++g) {
        float sum = sums[g];
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
  float v_inv;                                      // power of two that value scales are multiplied by; 0: none chosen yet
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
      }
    }
    v_inv = 0.f;
  }
};

__device__ __forceinline__ float scale_of(uint32_t word, bool int4) { return __uint_as_float(int4 ? word << 16 : word); }
__device__ __forceinline__ float centre_of(uint32_t word) { return __uint_as_float(word & 0xffff0000u); }

// Moves the reference maxima to what the tile brings, and the power of two of the value scales.
template <typename S>
__device__ __forceinline__ void move_reference(State<S>& st, const float (*s)[S::NT][4], float most_scale) {
#pragma unroll
  for (int d = 4; d < 32; d <<= 1) most_scale = fmaxf(most_scale, __shfl_xor_sync(0xffffffffu, most_scale, d));
  float ratio = 1.f;
  if (st.v_inv == 0.f || most_scale * st.v_inv > MOST_SCALE) {
    int e = (int)(__float_as_uint(most_scale) >> 23) - 127;
    e = min(max(e, -126), 126);
    const float now = __uint_as_float((uint32_t)(127 - e) << 23);
    if (st.v_inv != 0.f) ratio = now / st.v_inv;  // both powers of two
    st.v_inv = now;
  }
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float m = fmaxf(fmaxf(s[0][nt][x], s[0][nt][x + 2]), fmaxf(s[1][nt][x], s[1][nt][x + 2]));
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      m = fmaxf(m, st.m[nt][x]);
      const float by = m == -CUDART_INF_F ? 1.f : exp2_fast(st.m[nt][x] - m);
      st.m[nt][x] = m;
      st.l[nt][x] *= by;
#pragma unroll
      for (int g = 0; g < (S::INT4 ? S::GROUPS : 1); ++g) st.centre[g][nt][x] *= by;
#pragma unroll
      for (int t = 0; t < S::MTILES; ++t) {
        st.o[t][nt][x] *= by * ratio;
        st.o[t][nt][x + 2] *= by * ratio;
      }
    }
  }
}

// One tile: its two halves of sixteen keys.
template <typename S>
__device__ __forceinline__ void take_tile(State<S>& st, const Queries<S>& q, const uint8_t* stage, const uint8_t* extra, uint32_t rows, int lane) {
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
        for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
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
          widen8(w[0][j], x0);
          widen8(w[1][j], x1);
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
            s[half][nt][i] = fmaf(acc[nt][i], by, fmaf(q.sum[g][nt][i & 1], centre_of(word), s[half][nt][i]));
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
  }
  bool move = false;
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
    for (int x = 0; x < 2; ++x)
      move = move || fmaxf(fmaxf(s[0][nt][x], s[0][nt][x + 2]), fmaxf(s[1][nt][x], s[1][nt][x + 2])) > st.m[nt][x] + LAG;
  float most_scale = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int g = 0; g < S::GROUPS; ++g) most_scale = fmaxf(most_scale, scale_of(b_words[i][g], S::INT4));
  move = move || most_scale * st.v_inv > MOST_SCALE;
  if (__any_sync(ALL, move)) move_reference<S>(st, s, most_scale);

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
  // ---- outputs: value columns of lane / 4, keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 of each half -----------------------------
  const uint8_t* values = stage + S::TILE_BYTES;
  constexpr int GT = S::GS / 16;                        // tiles of sixteen columns of a group
  constexpr int VWORDS = S::INT4 ? 1 : S::GS / 32;
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int g = 0; g < S::GROUPS; ++g) {
      // Probabilities times scales, of fp16 results with what the rounding to fp16 leaves (else it would be as large as the result's own).
      uint32_t pb[S::NT][2], rest[S::HALF ? S::NT : 1][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float by = scale_of(b_words[2 * half + i][g], S::INT4) * st.v_inv;
#pragma unroll
        for (int nt = 0; nt < S::NT; ++nt) {
          const float x = s[half][nt][2 * i] * by, y = s[half][nt][2 * i + 1] * by;
          const uint32_t two = pack2<__half>(x, y);
          pb[nt][i] = transposed(two);
          if constexpr (S::HALF) {
            const __half2 h = *reinterpret_cast<const __half2*>(&two);
            rest[nt][i] = transposed(pack2<__half>(x - __low2float(h), y - __high2float(h)));
          }
        }
      }
      // columns g GS + r GS / 8 + i, i = 0 .. GS / 8: of tile t the two i = 2 t and 2 t + 1
      uint32_t w[4][VWORDS];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = 16 * half + 2 * c + (k & 1) + 8 * (k >> 1);
        if constexpr (!S::INT4 && S::RB == 128) {
          const uint4 x = *reinterpret_cast<const uint4*>(values + place_of<S>(row, r));
          w[k][0] = x.x; w[k][1] = x.y; w[k][2] = x.z; w[k][3] = x.w;
        } else if constexpr (!S::INT4) {
          const uint2 x = *reinterpret_cast<const uint2*>(values + place_of<S>(row, r >> 1) + 8 * (r & 1));
          w[k][0] = x.x; w[k][1] = x.y;
        } else if constexpr (S::GS == 64) {
          w[k][0] = *reinterpret_cast<const uint32_t*>(values + place_of<S>(row, 2 * g + (r >> 2)) + 4 * (r & 3));
        } else {
          w[k][0] = *reinterpret_cast<const uint16_t*>(values + place_of<S>(row, g) + 2 * r);
        }
        if constexpr (S::FMT == FSA_QC_E4M3) {  // what lies in rows that are not there may be no number
          if (partial && !(rows >> row & 1)) {
#pragma unroll
            for (int x = 0; x < VWORDS; ++x) w[k][x] = 0;
          }
        }
      }
      auto add = [&](int t, const uint32_t* f0, const uint32_t* f1) {
#pragma unroll
        for (int nt = 0; nt < S::NT; ++nt) {
          mma(st.o[t][nt], f0[0], f0[1], f1[0], f1[1], pb[nt][0], pb[nt][1]);
          if constexpr (S::HALF) mma(st.o[t][nt], f0[0], f0[1], f1[0], f1[1], rest[nt][0], rest[nt][1]);
        }
      };
      if constexpr (!S::INT4) {
#pragma unroll
        for (int x = 0; x < VWORDS; ++x) {
          uint32_t f[2][4];  // keys 2 c and 2 c + 1, 2 c + 8 and 2 c + 9; columns 4 x ..
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            widen4<S::FMT>(__byte_perm(w[2 * k][x], w[2 * k + 1][x], 0x5140), &f[k][0], &f[k][1]);
            widen4<S::FMT>(__byte_perm(w[2 * k][x], w[2 * k + 1][x], 0x7362), &f[k][2], &f[k][3]);
          }
          add(2 * x, f[0], f[1]);
          add(2 * x + 1, f[0] + 2, f[1] + 2);
        }
      } else {
#pragma unroll
        for (int four = 0; four < S::GS / 32; ++four) {  // four columns
          uint32_t f[2][4];
#pragma unroll
          for (int k = 0; k < 2; ++k) widen8(__byte_perm(w[2 * k][0], w[2 * k + 1][0], four ? 0x7632 : 0x5410), f[k]);  // columns 0 .. 3 of the two keys
          add(g * GT + 2 * four, f[0], f[1]);
          add(g * GT + 2 * four + 1, f[0] + 2, f[1] + 2);
        }
      }
    }
}

// Sums over the lanes that share heads, and the outputs in the values' own units.
template <typename S>
__device__ __forceinline__ void settle(State<S>& st) {
  const float by = st.v_inv == 0.f ? 1.f : 1.f / st.v_inv;
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
        const float z = S::INT4 ? st.centre[S::INT4 ? t / (S::GS / 16) : 0][nt][x] : 0.f;
        st.o[t][nt][x] = fmaf(st.o[t][nt][x], by, z);
        st.o[t][nt][x + 2] = fmaf(st.o[t][nt][x + 2], by, z);
      }
    }
}

// The first of this lane's columns in tile t; the next one is its other.
template <typename S>
__device__ __forceinline__ int column_of(int t, int r) {
  constexpr int GT = S::GS / 16;
  return t / GT * S::GS + r * (S::GS / 8) + 2 * (t % GT);
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

// Four columns of a head out of several parts. `part(i)`: where part i lies.
template <int HD, int HEADS, typename F>
__device__ __forceinline__ float4 join(int parts, int head, int col, F&& part, float* m_out, float* l_out) {
  float m = -CUDART_INF_F;
  for (int i = 0; i < parts; ++i) m = fmaxf(m, part(i)[HEADS * HD + head]);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int i = 0; i < parts; ++i) {
    const float* x = part(i);
    const float mi = x[HEADS * HD + head], by = mi == -CUDART_INF_F ? 0.f : exp2_fast(mi - m);  // (0 times a NaN is one)
    const float4 v = *reinterpret_cast<const float4*>(x + head * HD + col);
    o.x = fmaf(v.x, by, o.x);
    o.y = fmaf(v.y, by, o.y);
    o.z = fmaf(v.z, by, o.z);
    o.w = fmaf(v.w, by, o.w);
    l = fmaf(x[HEADS * (HD + 1) + head], by, l);
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
  __shared__ int ends_s[S::WARPS];   // whether the first piece's item ends in this warp
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

  uint64_t* full = full_s[warp];
  // a stage is there when its codes are (lane 0, with TMA's bytes) and its scales (the same, or each lane's copies)
  if (lane < S::STAGES) mbar_init(full + lane, p.scales_by_tma ? 1 : 33);
  if (tid == 0) abort_s = 0;
  mbar_fence_init();
  if (lane == 0) {
    part_s[warp][0] = part_s[warp][1] = nullptr;
    ends_s[warp] = 0;
  }
  __syncthreads();

  // ---- where this warp begins ------------------------------------------------------------------------------------------
  // The first `warps` warps of the grid have equal pieces of the list, of at least a tile; the others none. Every warp adds up the
  // lengths by itself, a lane those of neighbouring sequences: no warp waits for another before it has its first tiles under way.
  const long long g_warp = (long long)blockIdx.x * S::WARPS + warp;
  Walk<GATHER> walk;
  int mine = 0;
  {
    auto tiles_at = [&](int b) { return tiles_of(GATHER ? p.topk : keys_of(p, b)); };
    const bool alike = GATHER || !p.used;
    const int per = (p.batch + 31) / 32, b0 = min(lane * per, p.batch), b1 = min(b0 + per, p.batch);
    long long own = 0;
    if (alike) own = (long long)(b1 - b0) * tiles_at(0);
    else for (int b = b0; b < b1; ++b) own += tiles_at(b);
    long long upto = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(ALL, upto, d);
      if (lane >= d) upto += o;
    }
    const long long total = __shfl_sync(ALL, upto, 31) * p.items, warps = min(total, (long long)p.ctas * S::WARPS);
    if (g_warp < warps) {
      const long long at = total * g_warp / warps;
      mine = (int)min(total * (g_warp + 1) / warps - at, 0x7fffffffll);
      long long from = (upto - own) * p.items;
      const bool have = at >= from && at < upto * p.items;
      int where[3] = {0, 0, 0};
      if (have) {
        int b = b0, tiles = tiles_at(b);
        if (alike) {
          const long long skip = (at - from) / ((long long)tiles * p.items);
          b += (int)skip;
          from += skip * tiles * p.items;
        } else {
          while (at >= from + (long long)tiles * p.items) {
            from += (long long)tiles * p.items;
            tiles = tiles_at(++b);
          }
        }
        where[0] = b;
        where[1] = (int)((at - from) / tiles);
        where[2] = (int)((at - from) % tiles);
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
    walk.sequence(p);
    const bool begun = walk.t == 0;
    int sent = 0, into = 0, chosen_next = -1;  // into: the stage that the next copies take
    Place place;
    if constexpr (GATHER) {
      place = look_up(p, walk, chosen(p, walk, lane));
      Walk<GATHER> ahead = walk;
      ahead.next(p);
      chosen_next = chosen(p, ahead, lane);
    } else {
      place = look_up(p, walk, 0);
    }
    auto send = [&]() {
      if (sent < mine) {
        fetch<S, GATHER>(p, walk, place, ring + into * S::CODES, extras + into * S::EXTRA, full + into, lane);
        ++sent;
        into = into + 1 == S::STAGES ? 0 : into + 1;
        walk.next(p);
        place = look_up(p, walk, chosen_next);
        if constexpr (GATHER) {
          Walk<GATHER> ahead = walk;
          if (ahead.b < p.batch) ahead.next(p);
          chosen_next = chosen(p, ahead, lane);
        }
      }
    };
    int2 item = make_int2(walk.b, walk.i);
    for (int i = 0; i < S::STAGES - 1; ++i) send();
    Queries<S> q;
    State<S> st;
    load_queries<S>(p, item.x, item.y, lane, q);
    st.clear();
    bool fresh = false, whole = begun;  // whole: the item began in this warp
    int at = 0;
    uint32_t phase = 0;
    for (int i = 0; i < mine; ++i) {
      // all lanes see the tile, and are done with the one whose place the next copies take
      if (!mbar_wait_uniform(full + at, phase, &abort_s)) {
        report_status(p.status, STATUS_WAIT);
        for (int j = i + 1; j < sent; ++j) mbar_wait_uniform(full + j % S::STAGES, j / S::STAGES & 1, &abort_s);
        break;
      }
      __syncwarp();
      send();
      const uint8_t* stage = ring + at * S::CODES;
      const uint8_t* extra = extras + at * S::EXTRA;
      if (++at == S::STAGES) {
        at = 0;
        phase ^= 1;
      }
      const int4 what = *reinterpret_cast<const int4*>(extra + 2 * S::SCALE_BYTES);
      if (fresh) {
        item = make_int2(what.z, what.w);
        load_queries<S>(p, item.x, item.y, lane, q);
        st.clear();
        fresh = false;
      }
      take_tile<S>(st, q, stage, extra, (uint32_t)what.x, lane);
      const bool ends = __any_sync(ALL, what.y);
      if (ends || i + 1 == mine) {
        settle<S>(st);
        if (whole && ends) {
          write_out<S>(p, st, item.x, item.y, lane);
        } else {
          // the ring is free behind the last tile; a first piece that is done before goes through the workspace
          float* to = i + 1 == mine ? reinterpret_cast<float*>(ring) : p.pieces + ((long long)p.ctas * 2 + g_warp) * S::PIECE;
          __syncwarp();
          write_piece<S>(to, st, lane);
          if (lane == 0) {
            part_s[warp][whole] = to;
            if (whole)
              item_s[warp] = item;
            else
              ends_s[warp] = ends;
          }
        }
        fresh = true;
        whole = true;
      }
    }
  }
  __syncthreads();
  if (abort_s) {  // a wait ran out: nothing to join
    if (tid == 0) p.shared[blockIdx.x] = make_int2(0, -1);
    return;
  }

  // ---- items that several warps share ------------------------------------------------------------------------------------
  // Runs of pieces of one item, in the order of the warps.
  int2 told = make_int2(0, -1);
  int from = -1, kind = 0;  // the run's first warp and which of its pieces
  auto close = [&](int last, bool ends) {
    const int w0 = from, k0 = kind;
    auto part = [&](int i) { return i == 0 ? part_s[w0][k0] : part_s[w0 + i][0]; };
    const int2 item = k0 ? item_s[w0] : make_int2(0, 0);
    const bool whole = k0 && ends;
    float* to = own_pieces + (k0 ? S::PIECE : 0);
    for (int j = tid; j < S::HEADS * S::HD / 4; j += S::THREADS) {
      const int head = j / (S::HD / 4), col = 4 * (j % (S::HD / 4));
      float m, l;
      const float4 o = join<S::HD, S::HEADS>(last - w0 + 1, head, col, part, &m, &l);
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
    from = -1;
  };
  int last = 0;
  for (int w = 0; w < S::WARPS; ++w) {
    if (part_s[w][0]) {
      if (from < 0) {
        from = w;
        kind = 0;
      }
      last = w;
      if (ends_s[w]) close(w, true);
    }
    if (part_s[w][1]) {
      from = last = w;
      kind = 1;
    }
  }
  if (from >= 0) close(last, false);
  if (tid == 0) p.shared[blockIdx.x] = told;
}

// Items that several CTAs share: a block takes a quarter of the columns of the item that begins in its CTA, if it goes on in others.
constexpr int MERGE_THREADS = 128, SLICES = 4;

template <int HD, int HEADS, bool HALF>
__global__ void __launch_bounds__(MERGE_THREADS) quant_merge_kernel(const __grid_constant__ QuantDecParams p) {
  after_previous();
  __shared__ int end_s;
  const int cta = blockIdx.x / SLICES, slice = blockIdx.x % SLICES;
  const int item = p.shared[cta].y;
  if (item < 0) return;
  if (threadIdx.x == 0) end_s = p.ctas;
  __syncthreads();
  for (int c0 = cta + 1; c0 < p.ctas; c0 += MERGE_THREADS) {
    const int c = c0 + threadIdx.x;
    const bool ends = c < p.ctas && p.shared[c].x == 1;
    if (ends) atomicMin(&end_s, c);
    if (__syncthreads_or(ends)) break;
  }
  constexpr int PIECE = HEADS * (HD + 2);
  const int last = min(end_s, p.ctas - 1);
  auto part = [&](int i) { return p.pieces + ((long long)(cta + i) * 2 + (i == 0)) * PIECE; };
  constexpr int WIDE = HD / 4 / SLICES;  // groups of four columns of a slice
  for (int j = threadIdx.x; j < HEADS * WIDE; j += MERGE_THREADS) {
    const int head = j / WIDE, col = 4 * (slice * WIDE + j % WIDE);
    float m, l;
    const float4 o = join<HD, HEADS>(last - cta + 1, head, col, part, &m, &l);
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
  cudaError_t e = launch_early(kern, (unsigned)p.ctas, S::THREADS, S::SMEM, stream, 1, p);
  if (e != cudaSuccess || p.ctas == 1) return e;
  return launch_early(quant_merge_kernel<S::HD, S::HEADS, S::HALF>, (unsigned)(p.ctas * SLICES), MERGE_THREADS, 0, stream, 1, p);
}

// Calls f with the shape that a cache and a number of query heads a KV head need.
template <typename F>
auto for_shape(const FsaQuantCache& c, int dtype, int group_heads, F&& f) {
  auto with_heads = [&](auto hd, auto fmt, auto groups) {
    if (dtype == FSA_DT_FP16) return group_heads > 8 ? f(Shape<hd(), fmt(), groups(), 2, true>{}) : f(Shape<hd(), fmt(), groups(), 1, true>{});
    return group_heads > 8 ? f(Shape<hd(), fmt(), groups(), 2, false>{}) : f(Shape<hd(), fmt(), groups(), 1, false>{});
  };
  auto with_width = [&](auto hd) {
    using std::integral_constant;
    switch (c.format) {
      case FSA_QC_INT8: return with_heads(hd, integral_constant<int, FSA_QC_INT8>{}, integral_constant<int, 1>{});
      case FSA_QC_E4M3: return with_heads(hd, integral_constant<int, FSA_QC_E4M3>{}, integral_constant<int, 1>{});
      default:
        return c.group == 32 ? with_heads(hd, integral_constant<int, FSA_QC_INT4>{}, integral_constant<int, hd() / 32>{})
                             : with_heads(hd, integral_constant<int, FSA_QC_INT4>{}, integral_constant<int, hd() / 64>{});
    }
  };
  return c.head_dim <= 64 ? with_width(std::integral_constant<int, 64>{}) : with_width(std::integral_constant<int, 128>{});
}

// What follows from sizes alone; a FSA_ERR_* code where they do not fit.
int plan(const FsaQuantDecodeArgs* a, QuantDecParams* p, int* warps, int* piece) {
  const FsaQuantCache& c = a->cache;
  const int rc = check_quant_cache(c);
  if (rc != FSA_OK) return rc;
  if (a->batch <= 0 || a->heads_q <= 0 || a->heads_q % c.heads_kv || a->topk < 0) return FSA_ERR_INVALID_ARG;
  // the keys of a tile lie in one page
  if (c.page_table && (c.page_size < TILE || (c.page_size & (c.page_size - 1)))) return FSA_ERR_UNSUPPORTED;
  for (p->page_shift = 0; c.page_table && 1 << p->page_shift < c.page_size;) ++p->page_shift;
  const long long keys = c.page_table ? (long long)c.max_pages * c.page_size : c.capacity;
  p->keys = (int)(keys < 0x7fffff00ll ? keys : 0x7fffff00ll);
  p->batch = a->batch;
  p->heads_q = a->heads_q;
  p->group_heads = a->heads_q / c.heads_kv;
  const int heads = for_shape(c, a->dtype, p->group_heads, [&](auto s) {
    *warps = decltype(s)::WARPS;
    *piece = decltype(s)::PIECE;
    return (int)decltype(s)::HEADS;
  });
  p->blocks = (p->group_heads + heads - 1) / heads;
  if ((long long)p->blocks * c.heads_kv * a->batch > 0x7fffffffll) return FSA_ERR_UNSUPPORTED;
  p->items = p->blocks * c.heads_kv;
  p->topk = a->topk;
  p->chunks = quant_row_bytes(c) / 16;
  p->words = quant_row_words(c);
  const long long most = a->gather_kv_indices ? a->topk : p->keys, tiles = most > 0 ? (most + TILE - 1) / TILE : 1;
  const long long ctas = ((long long)p->items * a->batch * tiles + *warps - 1) / *warps;  // no warp without a tile
  p->ctas = (int)(ctas < device_sm_count() ? ctas : device_sm_count());
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
  return shared_bytes(p) + (int64_t)p.ctas * (2 + warps) * piece * (int64_t)sizeof(float);
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
      return make_byte_map(m, base, quant_row_bytes(c), c.heads_kv, sh, slots, ss, blocks, sb, bytes, TILE);
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
      const uint32_t box = (uint32_t)(TILE * groups);
      if (const int e = make_word_map(&p.map_ks, c.k_scales, slots * groups, c.heads_kv, c.ks_stride_h, blocks, c.ks_stride_b, box); e != FSA_OK) return e;
      if (const int e = make_word_map(&p.map_vs, c.v_scales, slots * groups, c.heads_kv, c.vs_stride_h, blocks, c.vs_stride_b, box); e != FSA_OK) return e;
    }
  }
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  const cudaError_t e =
      for_shape(p.c, a->dtype, p.group_heads, [&](auto s) { 
        const auto stream = reinterpret_cast<cudaStream_t>(stream_);
        return p.gather ? launch_both<decltype(s), true>(p, stream) : launch_both<decltype(s), false>(p, stream);
      });
  return e == cudaSuccess ? FSA_OK : FSA_ERR_LAUNCH;
}
