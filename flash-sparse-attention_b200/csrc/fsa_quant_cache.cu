// A key-value cache whose rows carry their own scales: rows are quantised as they are appended (their keys turned by their positions on
// the way) and read back as 16-bit rows. The decode over it is in fsa_quant_dec_sm100.cu.
//
//   8 bits   s = max|x| / top (127, or 448 for e4m3)           code = round(x * (1 / s))             value = code * s
//   4 bits   per group: s = bf16((max - min) / 15), z = bf16(min + 8 s)   code = clamp(round((x - z) * (1 / s)) + 8, 0, 15)
//                                                                                             value = z + (code - 8) s
// Every step is one fp32 operation rounded to nearest (no contraction), so that the codes do not depend on the launch or on who computes
// them. z is the value of code 8, the middle of the group, and not its minimum: a decode that keeps sums of codes and of z apart then adds
// numbers of the size of the result. Rounding z and s to bf16 costs at most half a step of what a bf16 input has already lost: codes are
// taken from the rounded pair.
//
// Both directions are bound by memory. Append: a group of 2, 4 or 8 (the next power of two of head_dim / 16) neighbouring lanes holds a row, two
// chunks of eight columns each - the partners of each other's pairs - and finds the row's or its groups' extremes by shuffles; nothing goes
// through shared memory. Read: a block takes eight tokens, looks their slots up once, and every thread widens sixteen columns at a time.
#include <initializer_list>

#include "fsa_axes.cuh"
#include "fsa_quant_cache.h"

namespace fsa {

namespace {

constexpr int V = 8;  // columns of a chunk

struct QuantPut {
  AppendParams a;  // places, rows and strides; the cache's own are below
  AxisMap m;       // positions given token by token (ids null: those of the slots)
  FsaQuantCache c;
  int lanes, lane_shift;  // of a row, and its log2
  int groups;      // of a row: words of scales
  int chunk_shift; // log2 of the chunks of a group
};

// Extremes that a NaN does not get lost in.
__device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float smaller(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr float TINY = 1.17549435e-38f;  // 2^-126

// Scale of a row whose largest magnitude is `most`, and what its values are multiplied by.
__device__ __forceinline__ float row_scale(float most, float top, float* inverse) {
  const float s = __fdiv_rn(most, top);
  *inverse = 0.f;
  if (!(most < INFINITY)) return NAN;
  if (s < TINY) return 0.f;
  *inverse = __frcp_rn(s);
  return s;
}

template <int FMT>
__device__ __forceinline__ uint2 codes8(const float* y, float inverse, bool finite) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (FMT == FSA_QC_INT8) {
      // clamped and rounded to the nearest even integer by an addition that leaves no bits for less; the low byte is the code
      uint32_t n[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        n[j] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(y[4 * i + j], inverse), -127.f), 127.f), 12582912.f));
      w[i] = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
    } else {
      w[i] = pack4_fp8<__nv_fp8_e4m3>(__fmul_rn(y[4 * i], inverse), __fmul_rn(y[4 * i + 1], inverse), __fmul_rn(y[4 * i + 2], inverse),
                                      __fmul_rn(y[4 * i + 3], inverse));
    }
    if (!finite) w[i] = 0;
  }
  return make_uint2(w[0], w[1]);
}

// Scale s and middle z of a group, as stored and as numbers.
struct Pair4 {
  uint32_t word;
  float z, inverse;
};
__device__ __forceinline__ Pair4 group_pair(float low, float high) {
  Pair4 p;
  const float width = __fdiv_rn(__fsub_rn(0.5f * high, 0.5f * low), 7.5f);  // (halves: the difference may be beyond fp32)
  float s = __bfloat162float(__float2bfloat16_rn(width));
  if (s < TINY) s = 0.f;
  // (of extremes near the end of fp32 8 s is beyond it, its sum with the least number is not)
  const float z = s < 1.3292279957849159e36f ? __fadd_rn(low, 8.f * s) : 2.f * __fadd_rn(0.5f * low, 4.f * s);  // (2^120)
  p.z = __bfloat162float(__float2bfloat16_rn(z));
  p.inverse = s > 0.f ? __frcp_rn(s) : 0.f;
  p.word = (__float_as_uint(s) >> 16) | (__float_as_uint(p.z) & 0xffff0000u);
  if (!(s < INFINITY) || !(fabsf(p.z) < INFINITY)) {  // an infinity or a NaN among the values
    p.word = 0x7fff7fffu;
    p.z = NAN;
  }
  return p;
}
__device__ __forceinline__ uint32_t codes4(const float* y, const Pair4& p) {
  // as above, and eight such numbers put together by their sum, less what they have in common
  constexpr uint32_t COMMON = 0x4b400000u;  // 12582912
  uint32_t r = 0, common = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float x = fminf(fmaxf(__fmul_rn(__fsub_rn(y[i], p.z), p.inverse), -8.f), 7.f);
    r += __float_as_uint(__fadd_rn(x, 12582920.f)) << (4 * i);
    common += COMMON << (4 * i);
  }
  return r - common;
}

// Quantises a row that `lanes` neighbouring lanes hold (all of the warp come here) and stores it if `live`.
template <int FORM>
__device__ __forceinline__ void put_row(const QuantPut& p, const float* ya, const float* yb, int a, int b, bool has_a, bool has_b, bool live, int u,
                                        uint8_t* codes, uint32_t* scales) {
  constexpr int FMT = FORM & 3, GROUPS = FORM >> 2;  // at most so many groups
  if constexpr (FMT != FSA_QC_INT4) {
    float most = 0.f;  // (columns that this lane does not have are zeros)
#pragma unroll
    for (int i = 0; i < V; ++i) most = larger(most, larger(fabsf(ya[i]), fabsf(yb[i])));
#pragma unroll
    for (int d = 4; d; d >>= 1)
      if (d < p.lanes) most = larger(most, __shfl_xor_sync(0xffffffffu, most, d));
    float inverse;
    const float s = row_scale(most, FMT == FSA_QC_INT8 ? 127.f : 448.f, &inverse);
    if (!live) return;
    const bool finite = most < INFINITY;
    if (has_a) *reinterpret_cast<uint2*>(codes + a) = codes8<FMT>(ya, inverse, finite);
    if (has_b) *reinterpret_cast<uint2*>(codes + b) = codes8<FMT>(yb, inverse, finite);
    if (u == 0) *scales = __float_as_uint(s);
  } else {
    float low_a = ya[0], high_a = ya[0], low_b = yb[0], high_b = yb[0];
#pragma unroll
    for (int i = 1; i < V; ++i) {
      low_a = smaller(low_a, ya[i]);
      high_a = larger(high_a, ya[i]);
      low_b = smaller(low_b, yb[i]);
      high_b = larger(high_b, yb[i]);
    }
    // Lane u finds the pair of group u for all.
    const int ga = has_a ? a / V >> p.chunk_shift : -1, gb = has_b ? b / V >> p.chunk_shift : -1;
    float low_u = 0.f, high_u = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      float low = smaller(ga == g ? low_a : INFINITY, gb == g ? low_b : INFINITY);
      float high = larger(ga == g ? high_a : -INFINITY, gb == g ? high_b : -INFINITY);
#pragma unroll
      for (int d = 4; d; d >>= 1)
        if (d < p.lanes) {
          low = smaller(low, __shfl_xor_sync(0xffffffffu, low, d));
          high = larger(high, __shfl_xor_sync(0xffffffffu, high, d));
        }
      if (u == g) {
        low_u = low;
        high_u = high;
      }
    }
    const Pair4 mine = group_pair(low_u, high_u);
    const int first = (threadIdx.x & 31) - u;  // the row's first lane
    Pair4 of_a, of_b;
    of_a.z = __shfl_sync(0xffffffffu, mine.z, first + max(ga, 0));
    of_a.inverse = __shfl_sync(0xffffffffu, mine.inverse, first + max(ga, 0));
    of_b.z = __shfl_sync(0xffffffffu, mine.z, first + max(gb, 0));
    of_b.inverse = __shfl_sync(0xffffffffu, mine.inverse, first + max(gb, 0));
    if (!live) return;
    if (has_a) *reinterpret_cast<uint32_t*>(codes + a / 2) = isnan(of_a.z) ? 0x88888888u : codes4(ya, of_a);
    if (has_b) *reinterpret_cast<uint32_t*>(codes + b / 2) = isnan(of_b.z) ? 0x88888888u : codes4(yb, of_b);
    if (u < p.groups) scales[u] = mine.word;
  }
}

// Where a token's rows lie in the cache, and its positions.
struct TokenPlace {
  long long block;
  int slot;
  bool live, turned;  // stored; has angles
  int pos[FSA_MAX_AXES];
};

__device__ __forceinline__ void find_place(const QuantPut& p, int seq, int slot, long long bi, long long si, TokenPlace* t) {
  t->slot = slot;
  t->block = seq;
  if (p.c.page_table) {
    t->block = p.c.page_table[seq * p.c.page_table_stride + slot / p.c.page_size];
    t->slot = slot % p.c.page_size;
  }
  if (p.m.ids) {
    t->turned = load_positions(p.m, bi, si, t->pos);
    if (!t->turned) report_status(p.a.status, STATUS_NO_ANGLES);
  } else {
    t->turned = true;
    t->pos[0] = slot + p.a.offset + (p.a.offsets ? p.a.offsets[seq] : 0);
  }
}

template <typename T, bool IL>
__device__ __forceinline__ void angles_of(const QuantPut& p, const TokenPlace& t, int a, int b, float* c, float* s) {
  if (p.m.ids)
    load_axis_angles<V, IL>(p.a.r, p.m, t.pos, a, b, c, s);
  else
    load_angles<V, IL>(p.a.r, t.pos[0], a, b, c, s);
}

// Head h of a token: query heads, then key heads, then value heads. `there`: this lane has columns of it.
template <typename T>
__device__ __forceinline__ void load_row(const AppendParams& p, long long bi, long long si, int h, int a, int b, bool has_a, bool has_b, Chunk<T, V>& xa,
                                         Chunk<T, V>& xb) {
  const T* src;
  if (h < p.heads_q)
    src = reinterpret_cast<const T*>(p.q) + bi * p.q_sb + si * p.q_ss + (long long)h * p.q_sh;
  else if (h < p.heads_q + p.heads_kv)
    src = reinterpret_cast<const T*>(p.k) + bi * p.k_sb + si * p.k_ss + (long long)(h - p.heads_q) * p.k_sh;
  else
    src = reinterpret_cast<const T*>(p.v) + bi * p.v_sb + si * p.v_ss + (long long)(h - p.heads_q - p.heads_kv) * p.v_sh;
  xa.raw = has_a ? __ldcs(reinterpret_cast<const uint4*>(src + a)) : uint4{};
  xb.raw = has_b ? __ldcs(reinterpret_cast<const uint4*>(src + b)) : uint4{};
}

// A row's two chunks as numbers, turned or as they are; zeros if it is not to be there.
template <typename T, bool IL>
__device__ __forceinline__ void row_values(const Chunk<T, V>& xa, const Chunk<T, V>& xb, bool turns, bool there, const float* c, const float* s, float* ya,
                                           float* yb) {
  if (turns && there) {
    // (each product and sum rounded: the same numbers whoever computes them)
    if constexpr (IL) {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const float a0 = float(xa.e[2 * j]), a1 = float(xa.e[2 * j + 1]), b0 = float(xb.e[2 * j]), b1 = float(xb.e[2 * j + 1]);
        const float cb = c[V / 2 + j], sb = s[V / 2 + j];
        ya[2 * j] = __fsub_rn(__fmul_rn(a0, c[j]), __fmul_rn(a1, s[j]));
        ya[2 * j + 1] = __fadd_rn(__fmul_rn(a1, c[j]), __fmul_rn(a0, s[j]));
        yb[2 * j] = __fsub_rn(__fmul_rn(b0, cb), __fmul_rn(b1, sb));
        yb[2 * j + 1] = __fadd_rn(__fmul_rn(b1, cb), __fmul_rn(b0, sb));
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float x1 = float(xa.e[i]), x2 = float(xb.e[i]);
        ya[i] = __fsub_rn(__fmul_rn(x1, c[i]), __fmul_rn(x2, s[i]));
        yb[i] = __fadd_rn(__fmul_rn(x2, c[i]), __fmul_rn(x1, s[i]));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      ya[i] = there ? float(xa.e[i]) : 0.f;
      yb[i] = there ? float(xb.e[i]) : 0.f;
    }
  }
}

// All lanes of the warp come here, those without a row with h < 0.
template <typename T, int FORM, bool IL>
__device__ __forceinline__ void store_row(const QuantPut& p, long long bi, long long si, int h, int a, int b, bool has_a, bool has_b, bool turns, int u,
                                          const TokenPlace& t, const float* c, const float* s, const Chunk<T, V>& xa, const Chunk<T, V>& xb) {
  const AppendParams& q = p.a;
  const bool is_q = h >= 0 && h < q.heads_q, is_v = h >= q.heads_q + q.heads_kv;
  float ya[V], yb[V];
  row_values<T, IL>(xa, xb, turns && !is_v, t.live && (is_v || t.turned), c, s, ya, yb);
  if (is_q) {
    T* out = reinterpret_cast<T*>(q.q_out) + bi * q.qo_sb + si * q.qo_ss + (long long)h * q.qo_sh;
    if (has_a) store16<T, V>(out, a, ya);
    if (has_b) store16<T, V>(out, b, yb);
  }
  const bool live = t.live && h >= q.heads_q;
  if (!__any_sync(0xffffffffu, live)) return;
  uint8_t* codes = nullptr;
  uint32_t* scales = nullptr;
  if (live) {
    const int hk = h - q.heads_q - (is_v ? q.heads_kv : 0);
    const FsaQuantCache& k = p.c;
    if (is_v) {
      codes = reinterpret_cast<uint8_t*>(k.v) + t.block * k.v_stride_b + t.slot * k.v_stride_s + hk * k.v_stride_h;
      scales = reinterpret_cast<uint32_t*>(k.v_scales) + t.block * k.vs_stride_b + t.slot * k.vs_stride_s + hk * k.vs_stride_h;
    } else {
      codes = reinterpret_cast<uint8_t*>(k.k) + t.block * k.k_stride_b + t.slot * k.k_stride_s + hk * k.k_stride_h;
      scales = reinterpret_cast<uint32_t*>(k.k_scales) + t.block * k.ks_stride_b + t.slot * k.ks_stride_s + hk * k.ks_stride_h;
    }
  }
  put_row<FORM>(p, ya, yb, a, b, has_a, has_b, live, u, codes, scales);
}

// This lane's columns of a row.
template <bool IL>
__device__ __forceinline__ void my_columns(const QuantPut& p, int u, int& a, int& b, bool& has_a, bool& has_b) {
  has_a = u < p.a.r.units;
  has_b = false;
  a = b = 0;
  if (has_a) chunk_columns<V, IL>(p.a.r, u, a, b, has_b);
}

// Few tokens: a thread has one row's share.
template <typename T, int FORM, bool IL>
__global__ void __launch_bounds__(THREADS) quant_rows_kernel(const __grid_constant__ QuantPut p) {
  after_previous();
  const AppendParams& q = p.a;
  const unsigned per_token = (unsigned)(q.slots * p.lanes);
  const unsigned idx = blockIdx.x * blockDim.x + threadIdx.x;
  const unsigned t = idx / per_token;
  const bool in = t < (unsigned)q.total;
  const unsigned rest = idx - t * per_token;
  const int slot = (int)(rest / (unsigned)p.lanes), u = (int)(rest - slot * (unsigned)p.lanes);
  int a, b;
  bool has_a, has_b;
  my_columns<IL>(p, u, a, b, has_a, has_b);
  long long bi = 0, si = t;
  if (!q.cu) {
    bi = t / (unsigned)q.new_tokens;
    si = t - bi * q.new_tokens;
  }
  Chunk<T, V> xa, xb;
  if (in) load_row<T>(q, bi, si, slot, a, b, has_a, has_b, xa, xb);

  TokenPlace place;
  place.live = false;
  if (in) {
    int seq = (int)bi, row = (int)si;
    place.live = true;
    if (q.cu) {
      seq = sequence_of(q.cu, q.batch, (int)t);
      place.live = seq < q.batch;
      if (place.live) row -= q.cu[seq];
    }
    if (place.live) {
      const int2 at = q.place[seq];
      place.live = row >= 0 && row < at.y;
      if (place.live) find_place(p, seq, at.x + row, bi, si, &place);
    }
  }
  const bool turns = has_a && u < q.r.turned;
  float c[V], s[V];
  if (turns && place.live && place.turned) angles_of<T, IL>(p, place, a, b, c, s);
  store_row<T, FORM, IL>(p, bi, si, in ? slot : -1, a, b, has_a, has_b, turns, u, place, c, s, xa, xb);
}

// Many tokens: a warp takes a token, so that its place and angles are found once for all heads; 32 / lanes rows at a time. (41 k packed tokens, 48
// heads of 128, 4 bits: threads with four rows of a token each 387 us; this with 104 registers 245, with five blocks an SM 206, with six, which
// spills, 243; keys and values of eight heads loaded ahead of everything, at 166 registers, 281. Without queries 121: the quantising itself, about
// 350 instructions for four rows.)
template <typename T, int FORM, bool IL>
__global__ void __launch_bounds__(THREADS, 5) quant_tokens_kernel(const __grid_constant__ QuantPut p) {
  after_previous();
  const AppendParams& q = p.a;
  const unsigned t = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  if (t >= (unsigned)q.total) return;
  const int lane = threadIdx.x & 31, slot = lane >> p.lane_shift, u = lane & (p.lanes - 1), rows = 32 >> p.lane_shift;
  int a, b;
  bool has_a, has_b;
  my_columns<IL>(p, u, a, b, has_a, has_b);
  long long bi = 0, si = t;
  int seq = 0, row = (int)t;
  if (!q.cu) {
    seq = (int)(t / (unsigned)q.new_tokens);
    row = (int)(t - (unsigned)seq * (unsigned)q.new_tokens);
    bi = seq;
    si = row;
  }
  auto load = [&](const T* from, Chunk<T, V>& xa, Chunk<T, V>& xb) {
    xa.raw = has_a ? __ldcs(reinterpret_cast<const uint4*>(from + a)) : uint4{};
    xb.raw = has_b ? __ldcs(reinterpret_cast<const uint4*>(from + b)) : uint4{};
  };
  TokenPlace place;
  place.live = true;
  place.turned = true;
  if (q.cu) {  // the sequence that the token is in: bounds at or in front of it, counted by all lanes
    int behind = 0;
    for (int b0 = 0; b0 <= q.batch; b0 += 32) behind += __popc(__ballot_sync(0xffffffffu, b0 + lane <= q.batch && q.cu[b0 + lane] <= row));
    seq = behind - 1;  // (of empty sequences the last)
    place.live = seq >= 0 && seq < q.batch;
    if (place.live) row -= q.cu[seq];
  }
  if (place.live) {
    const int2 at = q.place[seq];
    place.live = row >= 0 && row < at.y;
    if (place.live) find_place(p, seq, at.x + row, bi, si, &place);
  }
  const bool turns = has_a && u < q.r.turned, turned = place.live && place.turned;
  float c[V], s[V];
  if (turns && turned) angles_of<T, IL>(p, place, a, b, c, s);

  constexpr int BATCH = 4, PAIR = 2;  // rows of queries, and of keys or values, that a lane has under way
  {
    const T* from = reinterpret_cast<const T*>(q.q) + bi * q.q_sb + si * q.q_ss;
    T* to = reinterpret_cast<T*>(q.q_out) + bi * q.qo_sb + si * q.qo_ss;
    for (int h0 = slot; h0 < q.heads_q; h0 += BATCH * rows) {
      Chunk<T, V> xa[BATCH], xb[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i)
        if (h0 + i * rows < q.heads_q) load(from + (long long)(h0 + i * rows) * q.q_sh, xa[i], xb[i]);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (h0 + i * rows >= q.heads_q) continue;
        float ya[V], yb[V];
        row_values<T, IL>(xa[i], xb[i], turns, turned, c, s, ya, yb);
        T* out = to + (long long)(h0 + i * rows) * q.qo_sh;
        if (has_a) store16<T, V>(out, a, ya);
        if (has_b) store16<T, V>(out, b, yb);
      }
    }
  }
  if (!place.live) return;  // (the token's warp as one)
  const FsaQuantCache& k = p.c;
#pragma unroll 1
  for (int is_v = 0; is_v < 2; ++is_v) {
    const T* from = is_v ? reinterpret_cast<const T*>(q.v) + bi * q.v_sb + si * q.v_ss : reinterpret_cast<const T*>(q.k) + bi * q.k_sb + si * q.k_ss;
    const long long sh = is_v ? q.v_sh : q.k_sh, ch = is_v ? k.v_stride_h : k.k_stride_h, wh = is_v ? k.vs_stride_h : k.ks_stride_h;
    uint8_t* codes = is_v ? reinterpret_cast<uint8_t*>(k.v) + place.block * k.v_stride_b + place.slot * k.v_stride_s
                          : reinterpret_cast<uint8_t*>(k.k) + place.block * k.k_stride_b + place.slot * k.k_stride_s;
    uint32_t* scales = is_v ? reinterpret_cast<uint32_t*>(k.v_scales) + place.block * k.vs_stride_b + place.slot * k.vs_stride_s
                            : reinterpret_cast<uint32_t*>(k.k_scales) + place.block * k.ks_stride_b + place.slot * k.ks_stride_s;
#pragma unroll 1
    for (int h0 = 0; h0 < q.heads_kv; h0 += PAIR * rows) {  // all lanes: those of a row talk to one another
      Chunk<T, V> xa[PAIR], xb[PAIR];
#pragma unroll
      for (int i = 0; i < PAIR; ++i) {
        const int h = h0 + i * rows + slot;
        xa[i].raw = xb[i].raw = uint4{};
        if (h < q.heads_kv) load(from + h * sh, xa[i], xb[i]);
      }
#pragma unroll
      for (int i = 0; i < PAIR; ++i) {
        if (h0 + i * rows >= q.heads_kv) continue;
        const int h = h0 + i * rows + slot;
        float ya[V], yb[V];
        row_values<T, IL>(xa[i], xb[i], turns && !is_v, is_v || place.turned, c, s, ya, yb);
        put_row<FORM>(p, ya, yb, a, b, has_a, has_b, h < q.heads_kv, u, codes + h * ch, scales + h * wh);
      }
    }
  }
}

// Few tokens, pages assigned: a block per sequence finds its slots, stores its rows and advances its length, in one launch.
constexpr int STEP_PAGES = 4;  // that the new rows of a sequence may touch
constexpr int STEP_THREADS = 512;

template <typename T, int FORM, bool IL>
__global__ void __launch_bounds__(STEP_THREADS) quant_step_kernel(const __grid_constant__ QuantPut p) {
  after_previous();
  const AppendParams& q = p.a;
  const int b = blockIdx.x, heads = q.heads_q + 2 * q.heads_kv, items = q.new_tokens * heads * p.lanes;
  const int first = q.used[b];
  int n = rows_in_reach(q, b, first, q.new_tokens, threadIdx.x == 0);
  if (q.page_table && n > 0) {
    const int lo = first / q.page_size, hi = (first + n - 1) / q.page_size;
    int page[STEP_PAGES];
#pragma unroll
    for (int i = 0; i < STEP_PAGES; ++i) page[i] = lo + i <= hi ? q.page_table[b * q.pt_stride + lo + i] : 0;
    int bad = hi + 1;
#pragma unroll
    for (int i = STEP_PAGES - 1; i >= 0; --i)
      if (lo + i <= hi && (page[i] < 0 || page[i] >= q.num_pages)) bad = lo + i;
    if (bad <= hi) {
      n = max(0, bad * q.page_size - first);
      if (threadIdx.x == 0) report_status(q.status, STATUS_NO_ROOM);
    }
  }
  if (q.advance) {
    __syncthreads();  // every thread has read the length
    if (threadIdx.x == 0 && n > 0) q.used[b] = first + n;
  }
  const int round = (items + blockDim.x - 1) / blockDim.x;
  for (int i = 0; i < round; ++i) {  // whole warps: lanes of a row talk to one another
    const int k = i * blockDim.x + threadIdx.x;
    const bool in = k < items;
    const int row = in ? k / (heads * p.lanes) : 0, rest = k - row * (heads * p.lanes), h = rest / p.lanes, u = rest - h * p.lanes;
    int ca, cb;
    bool has_a, has_b;
    my_columns<IL>(p, u, ca, cb, has_a, has_b);
    Chunk<T, V> xa, xb;
    TokenPlace place;
    place.live = in && row < n;
    if (in) load_row<T>(q, b, row, h, ca, cb, has_a, has_b, xa, xb);
    if (place.live) find_place(p, b, first + row, b, row, &place);
    const bool turns = has_a && u < q.r.turned && h < q.heads_q + q.heads_kv;
    float c[V], s[V];
    if (turns && place.live && place.turned) angles_of<T, IL>(p, place, ca, cb, c, s);
    store_row<T, FORM, IL>(p, b, row, in ? h : -1, ca, cb, has_a, has_b, turns, u, place, c, s, xa, xb);
  }
}

// ----------------------------------------------------------------------------------------------
// Reading back
// ----------------------------------------------------------------------------------------------
// Small blocks with little under way each: what a read writes is two to four times what it fetches, and the GPU takes writes alone at 3.9 TB/s. 58 k
// tokens of 8 heads of 128, int8: 32 tokens, 256 threads, four pieces a thread under way 84.4 us; 128 threads 77.2; two pieces 71.3; 16 tokens
// 66.3; 8 tokens 64.5, with one piece 63.7 (4 bits: 56 k tokens 62.8, 59.3, 56.4, 51.8, 53.3, 58.8).
constexpr int READ_TOKENS = 8, READ_THREADS = 128, COLUMNS = 16;

struct QuantGet {
  FsaQuantCache c;
  void* k_out;
  void* v_out;
  const int* used;
  const int* cu;
  int* status;
  long long ko_sb, ko_ss, ko_sh, vo_sb, vo_ss, vo_sh;
  int batch, seqlen, total, pieces;  // pieces: of sixteen columns, of a head
  int group_shift;                   // log2 of the pieces of a group
  int of_head;                       // 2^16 / pieces, rounded up
  int step_tokens, step_rest;        // READ_THREADS in tokens and pieces
};

// Sixteen values.
template <int FMT>
__device__ __forceinline__ void widen(uint4 raw, uint32_t scale, float* y) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (FMT == FSA_QC_INT4) {
    const float s = __uint_as_float(scale << 16), z = __uint_as_float(scale & 0xffff0000u);
#pragma unroll
    for (int i = 0; i < COLUMNS; ++i)  // 2^23 + code, less that and 8
      y[i] = __fmaf_rn(__uint_as_float(0x4b000000u | (w[i >> 3] >> (4 * (i & 7)) & 15u)) - 8388616.f, s, z);
  } else if constexpr (FMT == FSA_QC_INT8) {
    const float s = __uint_as_float(scale);
#pragma unroll
    for (int i = 0; i < COLUMNS; ++i)  // 2^23 + 128 + code
      y[i] = __fmul_rn(__uint_as_float(__byte_perm(w[i >> 2] ^ 0x80808080u, 0x4b000000u, 0x7650 | (i & 3))) - 8388736.f, s);
  } else {
    const float s = __uint_as_float(scale);
#pragma unroll
    for (int i = 0; i < COLUMNS; i += 2) {
      uint32_t two;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"((uint16_t)(w[i >> 2] >> (8 * (i & 2)))));
      const __half2 h = *reinterpret_cast<const __half2*>(&two);
      y[i] = __fmul_rn(__low2float(h), s);
      y[i + 1] = __fmul_rn(__high2float(h), s);
    }
  }
}

template <typename T, int FMT>
__global__ void __launch_bounds__(READ_THREADS) quant_read_kernel(const __grid_constant__ QuantGet p) {
  after_previous();
  // of each token: where its rows' codes and scales begin (-1: zeros), and its result's
  __shared__ long long code_at[READ_TOKENS], scale_at[READ_TOKENS], out_at[READ_TOKENS];
  const unsigned t0 = (blockIdx.x >> 1) * (unsigned)READ_TOKENS;
  const int here = (int)min((unsigned)READ_TOKENS, (unsigned)p.total - t0);
  const bool is_v = blockIdx.x & 1;
  if (threadIdx.x < here) {
    const unsigned t = t0 + threadIdx.x;
    int seq, slot;
    bool in = true;
    long long to;
    if (p.cu) {
      seq = sequence_of(p.cu, p.batch, (int)t);
      in = seq < p.batch;
      slot = in ? (int)t - p.cu[seq] : 0;
      to = t * (is_v ? p.vo_ss : p.ko_ss);
    } else {
      seq = (int)(t / (unsigned)p.seqlen);
      slot = (int)(t - seq * (unsigned)p.seqlen);
      to = seq * (is_v ? p.vo_sb : p.ko_sb) + slot * (is_v ? p.vo_ss : p.ko_ss);
    }
    const long long cap = p.c.page_table ? (long long)p.c.max_pages * p.c.page_size : p.c.capacity;
    in = in && slot >= 0 && slot < cap && (!p.used || slot < p.used[seq]);
    long long block = seq;
    if (in && p.c.page_table) {
      block = p.c.page_table[seq * p.c.page_table_stride + slot / p.c.page_size];
      slot %= p.c.page_size;
      if (block < 0 || block >= p.c.num_pages) {
        in = false;
        report_status(p.status, STATUS_NO_ROOM);
      }
    }
    code_at[threadIdx.x] = in ? block * (is_v ? p.c.v_stride_b : p.c.k_stride_b) + slot * (is_v ? p.c.v_stride_s : p.c.k_stride_s) : -1;
    scale_at[threadIdx.x] = block * (is_v ? p.c.vs_stride_b : p.c.ks_stride_b) + slot * (is_v ? p.c.vs_stride_s : p.c.ks_stride_s);
    out_at[threadIdx.x] = to;
  }
  __syncthreads();
  const int per_token = p.pieces * p.c.heads_kv;
  const long long sh = is_v ? p.c.v_stride_h : p.c.k_stride_h, wh = is_v ? p.c.vs_stride_h : p.c.ks_stride_h, oh = is_v ? p.vo_sh : p.ko_sh;
  const uint8_t* codes = reinterpret_cast<const uint8_t*>(is_v ? p.c.v : p.c.k);
  const uint32_t* scales = reinterpret_cast<const uint32_t*>(is_v ? p.c.v_scales : p.c.k_scales);
  T* out = reinterpret_cast<T*>(is_v ? p.v_out : p.k_out);
  // Piece e of head h of token t: a thread's pieces are READ_THREADS apart, which it counts out without dividing.
  constexpr int BATCH = 2;  // pieces a thread has under way
  int t = threadIdx.x / per_token, rest = threadIdx.x - t * per_token;
  while (t < here) {
    uint4 raw[BATCH];
    uint32_t scale[BATCH];
    T* to[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      raw[j] = uint4{};
      scale[j] = 0;
      to[j] = nullptr;
      if (t < here) {
        const int h = rest * p.of_head >> 16, e = rest - h * p.pieces;
        const long long at = code_at[t];
        if (at >= 0) {
          const uint8_t* row = codes + at + h * sh;
          if constexpr (FMT == FSA_QC_INT4) {
            const uint2 half = __ldcs(reinterpret_cast<const uint2*>(row) + e);
            raw[j].x = half.x;
            raw[j].y = half.y;
          } else {
            raw[j] = __ldcs(reinterpret_cast<const uint4*>(row) + e);
          }
          scale[j] = __ldg(scales + scale_at[t] + h * wh + (FMT == FSA_QC_INT4 ? e >> p.group_shift : 0));
        }
        to[j] = out + out_at[t] + h * oh + e * COLUMNS;
        t += p.step_tokens;
        rest += p.step_rest;
        if (rest >= per_token) {
          rest -= per_token;
          ++t;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      if (!to[j]) continue;
      float y[COLUMNS];
      widen<FMT>(raw[j], scale[j], y);
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = pack2<T>(y[2 * i], y[2 * i + 1]);
      __stcs(reinterpret_cast<uint4*>(to[j]), make_uint4(w[0], w[1], w[2], w[3]));
      __stcs(reinterpret_cast<uint4*>(to[j]) + 1, make_uint4(w[4], w[5], w[6], w[7]));
    }
  }
}

// ----------------------------------------------------------------------------------------------
// Launches
// ----------------------------------------------------------------------------------------------
// f with the type and the format (and, in bits above, how many groups a row may have).
template <typename F>
cudaError_t for_format(int dtype, const FsaQuantCache& c, F&& f) {
  auto with_format = [&](auto t) {
    using std::integral_constant;
    switch (c.format) {
      case FSA_QC_INT8: return f(t, integral_constant<int, FSA_QC_INT8>{});
      case FSA_QC_E4M3: return f(t, integral_constant<int, FSA_QC_E4M3>{});
      default: return c.group == 32 ? f(t, integral_constant<int, FSA_QC_INT4 + 4 * 4>{}) : f(t, integral_constant<int, FSA_QC_INT4 + 4 * 2>{});
    }
  };
  return dtype == FSA_DT_BF16 ? with_format(__nv_bfloat16{}) : with_format(__half{});
}

// Whether quant_step_kernel takes the call, by the same bound as append_step_kernel's: rows of equal number, few enough that a block per sequence
// is no longer at them than a second launch takes, and nothing to be taken off a stack.
constexpr long long STEP_ELEMENTS = 192 * 128;
bool in_one_step(const FsaKvAppendQuantArgs* a) {
  if (a->cu_seqlens_new || a->free_pages || (long long)a->new_tokens * (a->heads_q + 2ll * a->cache.heads_kv) * a->cache.head_dim > STEP_ELEMENTS)
    return false;
  return !a->cache.page_table || (a->new_tokens - 1) / a->cache.page_size + 2 <= STEP_PAGES;
}

constexpr long long MANY_TOKENS = 148 * 16;  // from which on a warp a token fills the GPU

bool multiples_of(int64_t n, std::initializer_list<int64_t> values) {
  for (int64_t v : values)
    if (v % n) return false;
  return true;
}

}  // namespace

}  // namespace fsa

extern "C" int64_t fsa_kv_append_quantized_workspace_ints(const FsaKvAppendQuantArgs* a) {
  if (!a || a->batch <= 0 || (a->cache.page_table && a->cache.page_size <= 0)) return 0;
  return fsa::in_one_step(a) ? 0 : 2 * (int64_t)a->batch;
}

extern "C" int fsa_kv_append_quantized(const FsaKvAppendQuantArgs* a, void* stream_) {
  using namespace fsa;
  if (!a || !a->status || !a->k_new || !a->v_new || !a->seqused_k || (a->heads_q > 0 && (!a->q || !a->q_out))) return FSA_ERR_INVALID_ARG;
  const FsaQuantCache& c = a->cache;
  const int rc = check_quant_cache(c);
  if (rc != FSA_OK) return rc;
  if (a->batch <= 0 || a->heads_q < 0 || a->new_tokens < 0) return FSA_ERR_INVALID_ARG;
  if (a->dtype != FSA_DT_BF16 && a->dtype != FSA_DT_FP16) return FSA_ERR_UNSUPPORTED;
  if (a->rotary_dim != 0) {
    if (!table_ok(a->cos, a->sin, a->table_rows, a->table_dtype, c.head_dim, a->rotary_dim)) return FSA_ERR_INVALID_ARG;
    if (a->rotary_dim % 16) return FSA_ERR_UNSUPPORTED;
    if (a->table_dtype == FSA_DT_F32 && (!aligned_to(a->cos, 16) || !aligned_to(a->sin, 16) || a->table_stride % 4)) return FSA_ERR_UNSUPPORTED;
    if (a->position_ids && !axis_bits_ok(a->axis_bits, a->rotary_dim / 2, a->axes)) return FSA_ERR_INVALID_ARG;
  } else if (a->position_ids || a->heads_q > 0) {
    return FSA_ERR_INVALID_ARG;
  }
  if ((a->free_pages != nullptr) != (a->free_count != nullptr) || (a->free_pages && !c.page_table)) return FSA_ERR_INVALID_ARG;
  if (fsa_kv_append_quantized_workspace_ints(a) > 0 && !a->place_ws) return FSA_ERR_INVALID_ARG;
  const long long total = a->cu_seqlens_new ? (long long)a->total : (long long)a->batch * a->new_tokens;
  if (total < 0 || total > 0x7fffffffll) return FSA_ERR_INVALID_ARG;
  if (total == 0) return FSA_OK;
  for (const void* x : {a->q, a->k_new, a->v_new, (const void*)a->q_out})
    if (!aligned_to(x, 16)) return FSA_ERR_INVALID_ARG;
  if (!multiples_of(8, {a->k_stride_b, a->k_stride_s, a->k_stride_h, a->v_stride_b, a->v_stride_s, a->v_stride_h})) return FSA_ERR_INVALID_ARG;
  if (a->heads_q > 0 && !multiples_of(8, {a->q_stride_b, a->q_stride_s, a->q_stride_h, a->q_out_stride_b, a->q_out_stride_s, a->q_out_stride_h}))
    return FSA_ERR_INVALID_ARG;

  QuantPut p = {};
  AppendParams& q = p.a;
  RotaryShape& r = q.r;
  r.cos = a->cos;
  r.sin = a->sin;
  r.table_stride = a->table_stride;
  // (whether rows that are not turned by their slots have angles does not follow from where they lie)
  r.table_rows = a->rotary_dim && !a->position_ids ? a->table_rows : 0x7fffffff;
  r.table_dtype = a->table_dtype;
  r.turned = a->rotary_dim / (2 * V);
  r.chunks = c.head_dim / V;
  r.units = r.turned + (r.chunks - 2 * r.turned + 1) / 2;
  if (a->position_ids)
    make_axis_map(&p.m, a->axis_bits, a->position_ids, a->position_stride_a, a->position_stride_b, a->position_stride_s, a->axes,
                  a->position_ids_int64, a->table_rows);
  p.c = c;
  for (p.lanes = 1, p.lane_shift = 0; p.lanes < r.units; ++p.lane_shift) p.lanes *= 2;
  p.groups = quant_row_words(c);
  p.chunk_shift = c.group == 32 ? 2 : 3;
  q.q = a->q; q.k = a->k_new; q.v = a->v_new;
  q.q_out = a->q_out;
  q.used = a->seqused_k;
  q.page_table = c.page_table;
  q.free_pages = a->free_pages;
  q.free_count = a->free_count;
  q.cu = a->cu_seqlens_new;
  q.offsets = a->position_ids || !a->rotary_dim ? nullptr : a->seqlen_offsets;
  q.offset = a->position_ids || !a->rotary_dim ? 0 : a->offset;
  q.place = reinterpret_cast<int2*>(a->place_ws);
  q.status = a->status;
  q.q_sb = a->q_stride_b; q.q_ss = a->q_stride_s; q.q_sh = a->q_stride_h;
  q.k_sb = a->k_stride_b; q.k_ss = a->k_stride_s; q.k_sh = a->k_stride_h;
  q.v_sb = a->v_stride_b; q.v_ss = a->v_stride_s; q.v_sh = a->v_stride_h;
  q.qo_sb = a->q_out_stride_b; q.qo_ss = a->q_out_stride_s; q.qo_sh = a->q_out_stride_h;
  q.pt_stride = c.page_table_stride;
  q.batch = a->batch;
  q.new_tokens = a->new_tokens;
  q.total = (int)total;
  q.heads_q = a->heads_q;
  q.heads_kv = c.heads_kv;
  q.capacity = c.capacity;
  q.page_size = c.page_size;
  q.max_pages = c.max_pages;
  q.num_pages = c.num_pages;
  q.advance = a->advance;
  const int heads = a->heads_q + 2 * c.heads_kv;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (in_one_step(a)) {
    const long long items = (long long)a->new_tokens * heads * p.lanes;
    const int threads = items >= STEP_THREADS ? STEP_THREADS : (int)((items + 31) & ~31ll);
    const cudaError_t e = for_format(a->dtype, c, [&](auto t, auto fmt) {
      return a->interleaved ? launch_early(quant_step_kernel<decltype(t), fmt(), true>, (unsigned)a->batch, threads, 0, stream, 1, p)
                            : launch_early(quant_step_kernel<decltype(t), fmt(), false>, (unsigned)a->batch, threads, 0, stream, 1, p);
    });
    return e == cudaSuccess ? FSA_OK : FSA_ERR_LAUNCH;
  }
  const bool many = total >= MANY_TOKENS;
  q.slots = heads;
  const long long blocks = many ? (total + THREADS / 32 - 1) / (THREADS / 32) : (total * heads * p.lanes + THREADS - 1) / THREADS;
  if (!many && total * heads * p.lanes > 0x7fffffffll) return FSA_ERR_UNSUPPORTED;  // threads are counted in 32 bits
  // a warp looks at a sequence's slots where it may have many
  const int lanes = c.page_table && total / c.page_size > 2ll * a->batch ? 32 : 1;
  cudaError_t e = launch_append_place(q, lanes, stream);
  if (e != cudaSuccess) return FSA_ERR_LAUNCH;
  e = for_format(a->dtype, c, [&](auto t, auto fmt) {
    using T = decltype(t);
    if (a->interleaved)
      return many ? launch_early(quant_tokens_kernel<T, fmt(), true>, (unsigned)blocks, THREADS, 0, stream, 1, p)
                  : launch_early(quant_rows_kernel<T, fmt(), true>, (unsigned)blocks, THREADS, 0, stream, 1, p);
    return many ? launch_early(quant_tokens_kernel<T, fmt(), false>, (unsigned)blocks, THREADS, 0, stream, 1, p)
                : launch_early(quant_rows_kernel<T, fmt(), false>, (unsigned)blocks, THREADS, 0, stream, 1, p);
  });
  return e == cudaSuccess ? FSA_OK : FSA_ERR_LAUNCH;
}

extern "C" int fsa_kv_read_quantized(const FsaKvReadQuantArgs* a, void* stream_) {
  using namespace fsa;
  if (!a || !a->status || !a->k_out || !a->v_out || a->batch <= 0) return FSA_ERR_INVALID_ARG;
  const FsaQuantCache& c = a->cache;
  const int rc = check_quant_cache(c);
  if (rc != FSA_OK) return rc;
  if (a->dtype != FSA_DT_BF16 && a->dtype != FSA_DT_FP16) return FSA_ERR_UNSUPPORTED;
  const long long total = a->cu_seqlens ? (long long)a->total : (long long)a->batch * a->seqlen;
  if (total < 0 || total > 0x7fffffffll) return FSA_ERR_INVALID_ARG;
  if (total == 0) return FSA_OK;
  if (!aligned_to(a->k_out, 16) || !aligned_to(a->v_out, 16)) return FSA_ERR_INVALID_ARG;
  if (!multiples_of(8, {a->k_out_stride_b, a->k_out_stride_s, a->k_out_stride_h, a->v_out_stride_b, a->v_out_stride_s, a->v_out_stride_h}))
    return FSA_ERR_INVALID_ARG;
  QuantGet p = {};
  p.c = c;
  p.k_out = a->k_out;
  p.v_out = a->v_out;
  p.used = a->seqused_k;
  p.cu = a->cu_seqlens;
  p.status = a->status;
  p.ko_sb = a->k_out_stride_b; p.ko_ss = a->k_out_stride_s; p.ko_sh = a->k_out_stride_h;
  p.vo_sb = a->v_out_stride_b; p.vo_ss = a->v_out_stride_s; p.vo_sh = a->v_out_stride_h;
  p.batch = a->batch;
  p.seqlen = a->seqlen;
  p.total = (int)total;
  p.pieces = c.head_dim / COLUMNS;
  p.group_shift = c.group == 32 ? 1 : 2;
  const int per_token = p.pieces * c.heads_kv;
  if (per_token > 8192) return FSA_ERR_UNSUPPORTED;  // what of_head divides exactly
  p.of_head = (65536 + p.pieces - 1) / p.pieces;
  p.step_tokens = READ_THREADS / per_token;
  p.step_rest = READ_THREADS % per_token;
  const unsigned blocks = (unsigned)((total + READ_TOKENS - 1) / READ_TOKENS);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const cudaError_t e = for_format(a->dtype, c, [&](auto t, auto fmt) {
    return launch_early(quant_read_kernel<decltype(t), (fmt() & 3)>, 2 * blocks, READ_THREADS, 0, stream, 1, p);
  });
  return e == cudaSuccess ? FSA_OK : FSA_ERR_LAUNCH;
}
