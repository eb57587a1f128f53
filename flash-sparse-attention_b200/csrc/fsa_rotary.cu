// Rotary positions: y = R(p) x for the first `rotary_dim` columns of every head, as an operator with its gradient and on the way
// into a KV cache.
//
//   pair i of a head, (x1, x2) = columns (i, i + rotary_dim / 2), or (2i, 2i + 1) when interleaved, at position p:
//     y1 = x1 cos[p, i] - x2 sin[p, i]      y2 = x2 cos[p, i] + x1 sin[p, i]
//   gradient: the transposed rotation, i.e. the same kernel with -sin.
//
// Both are bound by memory: every element is read once and written once, for three operations. A thread takes two chunks of V elements of a
// head that hold V whole pairs (chunk u and chunk u + rotary_dim / 2V, which hold the partners of each other's pairs where those are
// halves apart), so that it needs V angles, and does that for HPT heads of the same token, so that it loads the angles once. V is the
// widest of 8, 4, 2, 1 elements that sizes, strides and addresses allow. Angles, products and sums are fp32 and rounded once.
// Measured (copy of as many bytes: 6538 GB/s): 4 x 4096 tokens, 40 heads of 128, both directions 115 us = 5870 GB/s; appending 16 chunks of up to
// 4000 tokens to a paged cache, 48 heads, 178 us = 5790 GB/s; blocks of 128 threads, of 256 118 and 181; append with six blocks an SM, as many as
// its registers would leave it (four) 218, eight 208.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fsa_b200.h"
#include "fsa_params.h"
#include "fsa_ptx.cuh"

namespace fsa {

namespace {

constexpr int THREADS = 128;
constexpr int STATUS_NO_ROOM = 3;    // new rows found no page, or lie behind the end of the cache
constexpr int STATUS_NO_ANGLES = 5;  // a position outside the tables

// What both kernels share: the tables and how a head's columns fall to threads.
struct RotaryShape {
  const void* cos;
  const void* sin;
  long long table_stride;
  int table_rows, table_dtype;
  int units, turned;  // threads a head; the first `turned` of them hold pairs
  int chunks;         // head_dim / V
};

template <int BYTES>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };
template <>
struct Raw<1> { using type = uint8_t; };

template <typename T, int V>
union Chunk {
  typename Raw<V * (int)sizeof(T)>::type raw;
  T e[V];
  __device__ Chunk() {}
};

// N angles from `first` on.
template <int N>
__device__ __forceinline__ void load_some(const RotaryShape& r, long long row, int first, float* c, float* s) {
  const long long at = row * r.table_stride + first;
  if (r.table_dtype == FSA_DT_F32) {
    const float* pc = reinterpret_cast<const float*>(r.cos) + at;
    const float* ps = reinterpret_cast<const float*>(r.sin) + at;
    if constexpr (N >= 4) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 a = *reinterpret_cast<const float4*>(pc + i), b = *reinterpret_cast<const float4*>(ps + i);
        c[i] = a.x; c[i + 1] = a.y; c[i + 2] = a.z; c[i + 3] = a.w;
        s[i] = b.x; s[i + 1] = b.y; s[i + 2] = b.z; s[i + 3] = b.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        c[i] = pc[i];
        s[i] = ps[i];
      }
    }
  } else if (r.table_dtype == FSA_DT_BF16) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(r.cos)[at + i]);
      s[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(r.sin)[at + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c[i] = __half2float(reinterpret_cast<const __half*>(r.cos)[at + i]);
      s[i] = __half2float(reinterpret_cast<const __half*>(r.sin)[at + i]);
    }
  }
}

// The V angles of a thread's two chunks at elements a and b.
template <int V, bool IL>
__device__ __forceinline__ void load_angles(const RotaryShape& r, long long row, int a, int b, float* c, float* s) {
  if constexpr (IL && V > 1) {
    load_some<V / 2>(r, row, a / 2, c, s);
    load_some<V / 2>(r, row, b / 2, c + V / 2, s + V / 2);
  } else {
    load_some<V>(r, row, IL ? a / 2 : a, c, s);
  }
}

// Element offsets of a thread's two chunks; the second may lie behind the last column (an odd number of columns to copy).
template <int V, bool IL>
__device__ __forceinline__ void chunk_columns(const RotaryShape& r, int u, int& a, int& b, bool& has_b) {
  // neighbouring threads take neighbouring chunks: with both chunks of a thread side by side a warp's requests were full of holes
  // (packed tokens of 64 columns, neighbouring pairs, both directions: 46.8 us, so 41.4)
  if (IL && V == 1) {  // a pair is two chunks
    a = 2 * u;
    b = a + 1;
  } else if (u < r.turned) {
    a = u;
    b = u + r.turned;
  } else {
    a = u + r.turned;  // 2 * turned chunks are rotated
    b = a + r.units - r.turned;
  }
  has_b = b < r.chunks;
  a *= V;
  b *= V;
}

// The pairs of two chunks, turned.
template <typename T, int V, bool IL>
__device__ __forceinline__ void turn(const Chunk<T, V>& xa, const Chunk<T, V>& xb, const float* c, const float* s, float* ya,
                                     float* yb) {
  if constexpr (IL && V > 1) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float a0 = float(xa.e[2 * j]), a1 = float(xa.e[2 * j + 1]), b0 = float(xb.e[2 * j]), b1 = float(xb.e[2 * j + 1]);
      ya[2 * j] = a0 * c[j] - a1 * s[j];
      ya[2 * j + 1] = a1 * c[j] + a0 * s[j];
      yb[2 * j] = b0 * c[V / 2 + j] - b1 * s[V / 2 + j];
      yb[2 * j + 1] = b1 * c[V / 2 + j] + b0 * s[V / 2 + j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float a = float(xa.e[i]), b = float(xb.e[i]);
      ya[i] = a * c[i] - b * s[i];
      yb[i] = b * c[i] + a * s[i];
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void store16(void* base, long long at, const float* y) {
  Chunk<T, V> o;
  if constexpr (V >= 2) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&o.raw);
#pragma unroll
    for (int i = 0; i < V; i += 2) w[i >> 1] = pack2<T>(y[i], y[i + 1]);
  } else {
    o.e[0] = T(y[0]);
  }
  *reinterpret_cast<typename Raw<V * 2>::type*>(reinterpret_cast<T*>(base) + at) = o.raw;
}
template <int V>
__device__ __forceinline__ void store8(void* base, long long at, const float* y, float scale, bool e4m3) {
  Chunk<uint8_t, V> o;
#pragma unroll
  for (int i = 0; i < V; ++i)
    o.e[i] = (uint8_t)__nv_cvt_float_to_fp8(__fdiv_rn(y[i], scale), __NV_SATFINITE, e4m3 ? __NV_E4M3 : __NV_E5M2);
  *reinterpret_cast<typename Raw<V>::type*>(reinterpret_cast<uint8_t*>(base) + at) = o.raw;
}

// The sequence that packed token t belongs to (cu[b] <= t < cu[b + 1]), or `batch` behind the last one. In front of the first one: 0, in
// which it has a negative place.
__device__ __forceinline__ int sequence_of(const int* cu, int batch, int t) {
  if (t >= cu[batch]) return batch;
  int lo = 0, hi = batch;  // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// ----------------------------------------------------------------------------------------------
// The operator
// ----------------------------------------------------------------------------------------------
struct RotaryParams {
  RotaryShape r;
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  const int* cu;
  const int* offsets;
  const void* position_ids;
  int* status;
  long long q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, qo_sb, qo_ss, qo_sh, ko_sb, ko_ss, ko_sh, id_sb, id_ss;
  int batch, seqlen, total;  // total: tokens of the call
  int heads_q, heads, slots; // heads: of q and k; slots: threads' groups of heads a token
  int offset, ids64;
  float sign;                // -1: the gradient
};

template <typename T, int V, bool IL, int HPT>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const RotaryParams p) {
  after_previous();
  const unsigned per_token = (unsigned)(p.slots * p.r.units);
  const unsigned idx = blockIdx.x * blockDim.x + threadIdx.x;
  const unsigned t = idx / per_token;
  if (t >= (unsigned)p.total) return;
  const unsigned rest = idx - t * per_token;
  const int slot = (int)(rest / (unsigned)p.r.units), u = (int)(rest - slot * (unsigned)p.r.units);
  int a, b;
  bool has_b;
  chunk_columns<V, IL>(p.r, u, a, b, has_b);

  long long bi = 0, si = t;  // where the token's row lies
  if (!p.cu && p.batch > 1) {
    bi = t / (unsigned)p.seqlen;
    si = t - bi * p.seqlen;
  }
  Chunk<T, V> xa[HPT], xb[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = slot + i * p.slots;
    if (h >= p.heads) continue;
    const bool is_q = h < p.heads_q;
    const T* src = is_q ? reinterpret_cast<const T*>(p.q) + bi * p.q_sb + si * p.q_ss + (long long)h * p.q_sh
                        : reinterpret_cast<const T*>(p.k) + bi * p.k_sb + si * p.k_ss + (long long)(h - p.heads_q) * p.k_sh;
    xa[i].raw = __ldcs(reinterpret_cast<const decltype(xa[i].raw)*>(src + a));
    if (has_b) xb[i].raw = __ldcs(reinterpret_cast<const decltype(xa[i].raw)*>(src + b));
  }

  long long pos;
  bool live = true;
  if (p.position_ids) {
    const long long at = bi * p.id_sb + si * p.id_ss;
    pos = p.ids64 ? reinterpret_cast<const long long*>(p.position_ids)[at] : reinterpret_cast<const int*>(p.position_ids)[at];
  } else {
    int seq = (int)bi;
    pos = si;
    if (p.cu) {
      seq = sequence_of(p.cu, p.batch, (int)t);
      live = seq < p.batch;
      if (live) pos -= p.cu[seq];
      live = live && pos >= 0;
    }
    pos += p.offset;
    if (p.offsets && live) pos += p.offsets[seq];
  }
  if (live && (pos < 0 || pos >= p.r.table_rows)) {
    live = false;
    report_status(p.status, STATUS_NO_ANGLES);
  }
  const bool turns = u < p.r.turned;
  float c[V], s[V];
  if (live && turns) {
    load_angles<V, IL>(p.r, pos, a, b, c, s);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] *= p.sign;
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = slot + i * p.slots;
    if (h >= p.heads) continue;
    const bool is_q = h < p.heads_q;
    T* dst = is_q ? reinterpret_cast<T*>(p.q_out) + bi * p.qo_sb + si * p.qo_ss + (long long)h * p.qo_sh
                  : reinterpret_cast<T*>(p.k_out) + bi * p.ko_sb + si * p.ko_ss + (long long)(h - p.heads_q) * p.ko_sh;
    if (live && turns) {
      float ya[V], yb[V];
      turn<T, V, IL>(xa[i], xb[i], c, s, ya, yb);
      store16<T, V>(dst, a, ya);
      store16<T, V>(dst, b, yb);
    } else {
      if (!live) {  // tokens outside every sequence, or without angles: zeros
        xa[i].raw = {};
        xb[i].raw = {};
      }
      *reinterpret_cast<decltype(xa[i].raw)*>(dst + a) = xa[i].raw;
      if (has_b) *reinterpret_cast<decltype(xa[i].raw)*>(dst + b) = xb[i].raw;
    }
  }
}

// ----------------------------------------------------------------------------------------------
// On the way into a cache
// ----------------------------------------------------------------------------------------------
struct AppendParams {
  RotaryShape r;
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_cache;
  void* v_cache;
  int* used;
  int* page_table;
  const int* free_pages;
  int* free_count;
  const int* cu;
  const int* offsets;
  const float* q_scale;
  const float* k_scale;
  const float* v_scale;
  int2* place;  // per sequence: first slot, rows that are stored
  int* status;
  long long q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, qo_sb, qo_ss, qo_sh, c_sb, c_ss, c_sh, vc_sb, vc_ss, vc_sh;
  long long pt_stride;
  int batch, new_tokens, total, heads_q, heads_kv, slots;
  int capacity, page_size, max_pages, num_pages, offset, advance, cache_dtype;
};

__device__ __forceinline__ int new_rows(const AppendParams& p, int b) {
  return p.cu ? min(p.cu[b + 1], p.total) - p.cu[b] : p.new_tokens;
}

// Rows of sequence b that have a slot and angles, by its length alone; what is missing is reported.
__device__ __forceinline__ int rows_in_reach(const AppendParams& p, int b, int first, int rows, bool report) {
  const long long cap = p.page_table ? (long long)p.max_pages * p.page_size : p.capacity;
  long long n = min((long long)rows, cap - first);
  int why = n < rows ? STATUS_NO_ROOM : 0;
  const long long at = (long long)first + p.offset + (p.offsets ? p.offsets[b] : 0);
  if (at < 0 || at + n > p.r.table_rows) {
    n = at < 0 ? 0 : min(n, (long long)p.r.table_rows - at);
    why = STATUS_NO_ANGLES;
  }
  if (first < 0 || n < 0) n = 0;
  if (first < 0) why = STATUS_NO_ROOM;
  if (why && rows > 0 && report) report_status(p.status, why);
  return (int)n;
}

// Where every sequence's rows go, in one block: pages that are missing come off the stack in the order of sequences and
// slots (the result does not depend on which thread is first), a page number outside the pool ends a sequence's rows, and
// lengths advance. `lanes` threads (1 or 32) look at the slots of a sequence.
__global__ void __launch_bounds__(1024) append_place_kernel(const AppendParams p, int lanes) {
  after_previous();
  __shared__ int warp_sum[32];
  __shared__ int carry_s;
  const int tid = threadIdx.x, lane = tid & 31;
  const int sub = lanes == 32 ? lane : 0, per_round = 1024 / lanes;
  const unsigned group = lanes == 32 ? 0xffffffffu : 1u << lane;
  const int have = p.free_count ? *p.free_count : 0;
  int taken = 0;  // pages asked for by the sequences of earlier rounds
  for (int b0 = 0; b0 < p.batch; b0 += per_round) {
    const int b = b0 + tid / lanes;
    int first = 0, n = 0, lo = 0, hi = -1, want = 0;
    if (b < p.batch) {
      first = p.used[b];
      const int rows = new_rows(p, b);
      n = rows > 0 ? rows_in_reach(p, b, first, rows, sub == 0) : 0;
      if (p.page_table && n > 0) {
        lo = first / p.page_size;
        hi = (first + n - 1) / p.page_size;
        for (int i = lo + sub; i <= hi; i += lanes) want += p.page_table[b * p.pt_stride + i] < 0;
      }
    }
    if (lanes == 32) want = __reduce_add_sync(0xffffffffu, want);
    // exclusive sum over the sequences of the round
    const int mine = sub == 0 ? want : 0;
    int incl = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, s);
      if (lane >= s) incl += o;
    }
    if (lane == 31) warp_sum[tid >> 5] = incl;
    __syncthreads();
    if (tid < 32) {
      int w = warp_sum[tid];
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, w, s);
        if (lane >= s) w += o;
      }
      warp_sum[tid] = w;
      if (tid == 31) carry_s = w;
    }
    __syncthreads();
    int rank = taken + (tid >= 32 ? warp_sum[(tid >> 5) - 1] : 0) + incl - mine;
    if (lanes == 32) rank = __shfl_sync(0xffffffffu, rank, 0);
    taken += carry_s;
    __syncthreads();

    if (b < p.batch) {
      int bad = hi + 1;  // the first slot without a page
      if (p.page_table && n > 0) {
        for (int i0 = lo; i0 <= hi; i0 += lanes) {
          const int i = i0 + sub;
          int page = 0;
          bool missing = false;
          if (i <= hi) {
            page = p.page_table[b * p.pt_stride + i];
            missing = page < 0;
          }
          int before = 0;
          if (lanes == 32) {
            const unsigned m = __ballot_sync(group, missing);
            before = __popc(m & ((1u << lane) - 1u));
            rank += before;
            if (missing) {
              if (rank < have) page = p.free_pages[have - 1 - rank];
            }
            rank += __popc(m) - before;
          } else if (missing) {
            if (rank < have) page = p.free_pages[have - 1 - rank];
            ++rank;
          }
          if (missing && page >= 0) p.page_table[b * p.pt_stride + i] = page;
          if (i <= hi && (page < 0 || page >= p.num_pages)) bad = min(bad, i);
        }
        if (lanes == 32) bad = __reduce_min_sync(0xffffffffu, bad);
        if (bad <= hi) {
          n = max(0, bad * p.page_size - first);
          if (sub == 0) report_status(p.status, STATUS_NO_ROOM);
        }
      }
      if (sub == 0) {
        p.place[b] = make_int2(first, n);
        if (p.advance && n > 0) p.used[b] = first + n;
      }
    }
  }
  if (p.free_count && tid == 0) *p.free_count = have - min(taken, max(have, 0));
}

// The two chunks of head h of a token (q heads, then k heads, then v heads).
template <typename T, int V>
__device__ __forceinline__ void append_load(const AppendParams& p, long long bi, long long si, int h, int a, int b, bool has_b,
                                            Chunk<T, V>& xa, Chunk<T, V>& xb) {
  const T* src;
  if (h < p.heads_q)
    src = reinterpret_cast<const T*>(p.q) + bi * p.q_sb + si * p.q_ss + (long long)h * p.q_sh;
  else if (h < p.heads_q + p.heads_kv)
    src = reinterpret_cast<const T*>(p.k) + bi * p.k_sb + si * p.k_ss + (long long)(h - p.heads_q) * p.k_sh;
  else
    src = reinterpret_cast<const T*>(p.v) + bi * p.v_sb + si * p.v_ss + (long long)(h - p.heads_q - p.heads_kv) * p.v_sh;
  xa.raw = __ldcs(reinterpret_cast<const decltype(xa.raw)*>(src + a));
  if (has_b) xb.raw = __ldcs(reinterpret_cast<const decltype(xa.raw)*>(src + b));
}

// Token (bi, si) is row `place` of the cache (c0 elements from its start, -1: not stored) at rotary position pos.
template <typename T, int V, bool IL>
__device__ __forceinline__ void append_store(const AppendParams& p, long long bi, long long si, int h, int a, int b, bool has_b,
                                             bool turns, bool live, long long k_row, long long v_row, const float* c, const float* s,
                                             Chunk<T, V>& xa, Chunk<T, V>& xb) {
  const bool is_q = h < p.heads_q, is_k = !is_q && h < p.heads_q + p.heads_kv;
  if (!live && !is_q) return;
  float ya[V], yb[V];
  if (live && turns && (is_q || is_k)) {
    turn<T, V, IL>(xa, xb, c, s, ya, yb);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      ya[i] = live ? float(xa.e[i]) : 0.f;
      yb[i] = live && has_b ? float(xb.e[i]) : 0.f;
    }
  }
  void* base;
  long long at;
  const float* scale;
  if (is_q) {
    base = p.q_out;
    at = bi * p.qo_sb + si * p.qo_ss + (long long)h * p.qo_sh;
    scale = p.q_scale;
  } else if (is_k) {
    base = p.k_cache;
    at = k_row + (long long)(h - p.heads_q) * p.c_sh;
    scale = p.k_scale;
  } else {
    base = p.v_cache;
    at = v_row + (long long)(h - p.heads_q - p.heads_kv) * p.vc_sh;
    scale = p.v_scale;
  }
  if (p.cache_dtype == FSA_DT_E4M3 || p.cache_dtype == FSA_DT_E5M2) {
    const float sc = *scale;
    store8<V>(base, at + a, ya, sc, p.cache_dtype == FSA_DT_E4M3);
    if (has_b) store8<V>(base, at + b, yb, sc, p.cache_dtype == FSA_DT_E4M3);
  } else {
    store16<T, V>(base, at + a, ya);
    if (has_b) store16<T, V>(base, at + b, yb);
  }
}

__device__ __forceinline__ void cache_rows(const AppendParams& p, int b, int slot, long long& k_row, long long& v_row) {
  if (p.page_table) {
    const long long page = p.page_table[b * p.pt_stride + slot / p.page_size];
    k_row = page * p.c_sb + (long long)(slot % p.page_size) * p.c_ss;
    v_row = page * p.vc_sb + (long long)(slot % p.page_size) * p.vc_ss;
  } else {
    k_row = (long long)b * p.c_sb + (long long)slot * p.c_ss;
    v_row = (long long)b * p.vc_sb + (long long)slot * p.vc_ss;
  }
}

template <typename T, int V, bool IL, int HPT>
__global__ void __launch_bounds__(THREADS, 6) append_rows_kernel(const AppendParams p) {
  after_previous();
  const unsigned per_token = (unsigned)(p.slots * p.r.units);
  const unsigned idx = blockIdx.x * blockDim.x + threadIdx.x;
  const unsigned t = idx / per_token;
  if (t >= (unsigned)p.total) return;
  const unsigned rest = idx - t * per_token;
  const int slot = (int)(rest / (unsigned)p.r.units), u = (int)(rest - slot * (unsigned)p.r.units);
  const int heads = p.heads_q + 2 * p.heads_kv;
  int a, b;
  bool has_b;
  chunk_columns<V, IL>(p.r, u, a, b, has_b);
  long long bi = 0, si = t;
  if (!p.cu) {
    bi = t / (unsigned)p.new_tokens;
    si = t - bi * p.new_tokens;
  }
  Chunk<T, V> xa[HPT], xb[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (slot + i * p.slots < heads) append_load<T, V>(p, bi, si, slot + i * p.slots, a, b, has_b, xa[i], xb[i]);

  int seq = (int)bi, row = (int)si;
  bool live = true;
  if (p.cu) {
    seq = sequence_of(p.cu, p.batch, (int)t);
    live = seq < p.batch;
    if (live) row -= p.cu[seq];
  }
  float c[V], s[V];
  long long k_row = 0, v_row = 0;
  const bool turns = u < p.r.turned;
  if (live) {
    const int2 place = p.place[seq];
    live = row >= 0 && row < place.y;
    if (live) {
      cache_rows(p, seq, place.x + row, k_row, v_row);
      if (turns)
        load_angles<V, IL>(p.r, (long long)place.x + row + p.offset + (p.offsets ? p.offsets[seq] : 0), a, b, c, s);
    }
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (slot + i * p.slots < heads)
      append_store<T, V, IL>(p, bi, si, slot + i * p.slots, a, b, has_b, turns, live, k_row, v_row, c, s, xa[i], xb[i]);
}

// Few tokens, pages assigned: a block per sequence finds its slots, stores its rows and advances its length by itself. One launch, where the
// two kernels above wait for one another (one token each of 64 sequences, 48 heads of 128: 5.3 us, so 3.3; one sequence 4.9 and 3.0).
constexpr int STEP_PAGES = 4;  // that the new rows of a sequence may touch

template <typename T, int V, bool IL>
__global__ void __launch_bounds__(1024) append_step_kernel(const AppendParams p) {
  after_previous();
  const int b = blockIdx.x, heads = p.heads_q + 2 * p.heads_kv, items = p.new_tokens * heads * p.r.units;
  const int first = p.used[b];
  int n = rows_in_reach(p, b, first, p.new_tokens, threadIdx.x == 0);
  if (p.page_table && n > 0) {
    const int lo = first / p.page_size, hi = (first + n - 1) / p.page_size;
    int page[STEP_PAGES];
#pragma unroll
    for (int i = 0; i < STEP_PAGES; ++i) page[i] = lo + i <= hi ? p.page_table[b * p.pt_stride + lo + i] : 0;
    int bad = hi + 1;
#pragma unroll
    for (int i = STEP_PAGES - 1; i >= 0; --i)
      if (lo + i <= hi && (page[i] < 0 || page[i] >= p.num_pages)) bad = lo + i;
    if (bad <= hi) {
      n = max(0, bad * p.page_size - first);
      if (threadIdx.x == 0) report_status(p.status, STATUS_NO_ROOM);
    }
  }
  const int at = first + p.offset + (p.offsets ? p.offsets[b] : 0);
  if (p.advance) {
    __syncthreads();  // every thread has read the length
    if (threadIdx.x == 0 && n > 0) p.used[b] = first + n;
  }
  for (int k = threadIdx.x; k < items; k += blockDim.x) {
    const int row = k / (heads * p.r.units), rest = k - row * (heads * p.r.units), h = rest / p.r.units, u = rest - h * p.r.units;
    int ca, cb;
    bool has_b;
    chunk_columns<V, IL>(p.r, u, ca, cb, has_b);
    Chunk<T, V> xa, xb;
    append_load<T, V>(p, b, row, h, ca, cb, has_b, xa, xb);
    const bool live = row < n, turns = u < p.r.turned;
    float c[V], s[V];
    long long k_row = 0, v_row = 0;
    if (live) {
      cache_rows(p, b, first + row, k_row, v_row);
      if (turns && h < p.heads_q + p.heads_kv) load_angles<V, IL>(p.r, at + row, ca, cb, c, s);
    }
    append_store<T, V, IL>(p, b, row, h, ca, cb, has_b, turns, live, k_row, v_row, c, s, xa, xb);
  }
}

// ----------------------------------------------------------------------------------------------
// Launches
// ----------------------------------------------------------------------------------------------
// The widest chunk that everything allows: `bytes` collects the lowest set bits of what has to be a multiple of it.
struct Width {
  unsigned long long elems = 8;  // of strides, sizes and addresses in elements
  void also(long long n) { elems |= (unsigned long long)n; }
  void address(const void* ptr, int elem_bytes) {
    elems |= reinterpret_cast<uintptr_t>(ptr) / (unsigned)elem_bytes;
  }
  int v() const { return (int)(elems & (~elems + 1)); }  // lowest set bit, at most 8
};

bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

int make_shape(RotaryShape* r, Width w, const void* cos, const void* sin, long long table_stride, int table_rows, int table_dtype,
               int head_dim, int rotary_dim) {
  w.also(rotary_dim / 2);
  w.also(head_dim);
  int v = w.v();
  // tables are read four fp32 values at a time by chunks of four and more
  if (v >= 4 && table_dtype == FSA_DT_F32 && (!aligned_to(cos, 16) || !aligned_to(sin, 16) || table_stride % 4)) v = 2;
  r->cos = cos;
  r->sin = sin;
  r->table_stride = table_stride;
  r->table_rows = table_rows;
  r->table_dtype = table_dtype;
  r->turned = rotary_dim / (2 * v);
  r->chunks = head_dim / v;
  r->units = r->turned + (r->chunks - 2 * r->turned + 1) / 2;
  return v;
}

bool table_ok(const void* cos, const void* sin, int rows, int dtype, int head_dim, int rotary_dim) {
  if (!cos || !sin || rows <= 0 || rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim) return false;
  const int es = dtype == FSA_DT_F32 ? 4 : 2;
  return (dtype == FSA_DT_F32 || dtype == FSA_DT_BF16 || dtype == FSA_DT_FP16) && aligned_to(cos, es) && aligned_to(sin, es);
}

template <typename F>
cudaError_t for_each_form(int dtype, int v, bool interleaved, bool many, F&& f) {
  auto with_hpt = [&](auto t, auto vv, auto il) {
    return many ? f(t, vv, il, std::integral_constant<int, 4>{}) : f(t, vv, il, std::integral_constant<int, 1>{});
  };
  auto with_il = [&](auto t, auto vv) {
    return interleaved ? with_hpt(t, vv, std::true_type{}) : with_hpt(t, vv, std::false_type{});
  };
  auto with_v = [&](auto t) {
    switch (v) {
      case 8: return with_il(t, std::integral_constant<int, 8>{});
      case 4: return with_il(t, std::integral_constant<int, 4>{});
      case 2: return with_il(t, std::integral_constant<int, 2>{});
      default: return with_il(t, std::integral_constant<int, 1>{});
    }
  };
  return dtype == FSA_DT_BF16 ? with_v(__nv_bfloat16{}) : with_v(__half{});
}

constexpr int HEADS_PER_THREAD = 4;

// Whether append_step_kernel takes the call: rows of equal number, few enough that a block per sequence is no longer at them than a second
// launch takes, and nothing to be taken off a stack. Replayed calls, us in one launch and in two, by sequences and rows of 128 columns (query, key
// and value heads times tokens) of each:
//          48 rows        96             192            384
//     1    3.0  4.9       3.7  4.9       5.0  4.9       7.3  5.3
//    16    3.1  5.2       3.8  5.3       5.3  5.3       7.4  5.6
//    64    3.3  5.3       4.0  5.6       5.3  5.8       7.6  7.8
//   128    3.2  5.3       4.3  6.0       5.5  7.7       7.8  8.4
//   256    4.0  5.8       7.2  8.2      10.6  9.2      14.8 13.8
// The bound is one for all numbers of sequences: at 192 rows one launch loses with 256 of them and wins with 64 and 128.
constexpr long long STEP_ELEMENTS = 192 * 128;
bool append_in_one_step(const FsaKvAppendRotaryArgs* a) {
  if (a->cu_seqlens_new || a->free_pages || (long long)a->new_tokens * (a->heads_q + 2ll * a->heads_kv) * a->head_dim > STEP_ELEMENTS) return false;
  return !a->page_table || (a->new_tokens - 1) / a->page_size + 2 <= STEP_PAGES;
}

}  // namespace

}  // namespace fsa

extern "C" int fsa_rotary(const FsaRotaryArgs* a, void* stream_) {
  using namespace fsa;
  if (!a || !a->status || (a->heads_q > 0 && (!a->q || !a->q_out)) || (a->heads_k > 0 && (!a->k || !a->k_out))) return FSA_ERR_INVALID_ARG;
  if (a->heads_q < 0 || a->heads_k < 0 || a->heads_q + a->heads_k <= 0 || a->head_dim <= 0 || a->batch <= 0) return FSA_ERR_INVALID_ARG;
  if (a->dtype != FSA_DT_BF16 && a->dtype != FSA_DT_FP16) return FSA_ERR_UNSUPPORTED;
  if (!table_ok(a->cos, a->sin, a->table_rows, a->table_dtype, a->head_dim, a->rotary_dim)) return FSA_ERR_INVALID_ARG;
  const long long total = a->cu_seqlens ? (long long)a->total : (long long)a->batch * a->seqlen;
  if (total < 0 || total > 0x7fffffffll) return FSA_ERR_INVALID_ARG;
  if (total == 0) return FSA_OK;
  const void* ptrs[4] = {a->q, a->k, a->q_out, a->k_out};
  for (const void* x : ptrs)
    if (x && !aligned_to(x, 2)) return FSA_ERR_INVALID_ARG;

  RotaryParams p = {};
  Width w;
  if (a->heads_q > 0) {
    w.address(a->q, 2);
    w.address(a->q_out, 2);
    for (int64_t s : {a->q_stride_b, a->q_stride_s, a->q_stride_h, a->q_out_stride_b, a->q_out_stride_s, a->q_out_stride_h}) w.also(s);
  }
  if (a->heads_k > 0) {
    w.address(a->k, 2);
    w.address(a->k_out, 2);
    for (int64_t s : {a->k_stride_b, a->k_stride_s, a->k_stride_h, a->k_out_stride_b, a->k_out_stride_s, a->k_out_stride_h}) w.also(s);
  }
  const int v = make_shape(&p.r, w, a->cos, a->sin, a->table_stride, a->table_rows, a->table_dtype, a->head_dim, a->rotary_dim);
  p.q = a->q;
  p.k = a->k;
  p.q_out = a->q_out;
  p.k_out = a->k_out;
  p.cu = a->cu_seqlens;
  p.offsets = a->seqlen_offsets;
  p.position_ids = a->position_ids;
  p.status = a->status;
  p.q_sb = a->q_stride_b; p.q_ss = a->q_stride_s; p.q_sh = a->q_stride_h;
  p.k_sb = a->k_stride_b; p.k_ss = a->k_stride_s; p.k_sh = a->k_stride_h;
  p.qo_sb = a->q_out_stride_b; p.qo_ss = a->q_out_stride_s; p.qo_sh = a->q_out_stride_h;
  p.ko_sb = a->k_out_stride_b; p.ko_ss = a->k_out_stride_s; p.ko_sh = a->k_out_stride_h;
  p.id_sb = a->position_stride_b; p.id_ss = a->position_stride_s;
  p.batch = a->batch;
  p.seqlen = a->seqlen;
  p.total = (int)total;
  p.heads_q = a->heads_q;
  p.heads = a->heads_q + a->heads_k;
  p.offset = a->offset;
  p.ids64 = a->position_ids_int64;
  p.sign = a->transposed ? -1.f : 1.f;
  const bool many = total * p.heads * p.r.units >= 148ll * 2048;
  p.slots = many ? (p.heads + HEADS_PER_THREAD - 1) / HEADS_PER_THREAD : p.heads;
  const long long blocks = (total * p.slots * p.r.units + THREADS - 1) / THREADS;
  if (blocks * THREADS > 0xffffffffll) return FSA_ERR_UNSUPPORTED;  // threads are counted in 32 bits
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const cudaError_t e = for_each_form(a->dtype, v, a->interleaved, many, [&](auto t, auto vv, auto il, auto hpt) {
    return launch_early(rotary_kernel<decltype(t), vv(), il(), hpt()>, (unsigned)blocks, THREADS, 0, stream, 1, p);
  });
  return e == cudaSuccess ? FSA_OK : FSA_ERR_LAUNCH;
}

extern "C" int64_t fsa_kv_append_rotary_workspace_ints(const FsaKvAppendRotaryArgs* a) {
  if (!a || a->batch <= 0 || (a->page_table && a->page_size <= 0)) return 0;
  return fsa::append_in_one_step(a) ? 0 : 2 * (int64_t)a->batch;
}

extern "C" int fsa_kv_append_rotary(const FsaKvAppendRotaryArgs* a, void* stream_) {
  using namespace fsa;
  if (!a || !a->status || !a->k_new || !a->v_new || !a->k_cache || !a->v_cache || !a->seqused_k ||
      (a->heads_q > 0 && (!a->q || !a->q_out)))
    return FSA_ERR_INVALID_ARG;
  if (a->batch <= 0 || a->heads_q < 0 || a->heads_kv <= 0 || a->head_dim <= 0) return FSA_ERR_INVALID_ARG;
  if (a->dtype != FSA_DT_BF16 && a->dtype != FSA_DT_FP16) return FSA_ERR_UNSUPPORTED;
  const bool fp8 = a->cache_dtype == FSA_DT_E4M3 || a->cache_dtype == FSA_DT_E5M2;
  if (!fp8 && a->cache_dtype != a->dtype) return FSA_ERR_UNSUPPORTED;
  if (fp8 && (!a->k_scale || !a->v_scale || (a->heads_q > 0 && !a->q_scale))) return FSA_ERR_INVALID_ARG;
  if (!table_ok(a->cos, a->sin, a->table_rows, a->table_dtype, a->head_dim, a->rotary_dim)) return FSA_ERR_INVALID_ARG;
  if (a->page_table ? (a->page_size <= 0 || a->max_pages <= 0 || a->num_pages <= 0) : a->capacity <= 0) return FSA_ERR_INVALID_ARG;
  if ((a->free_pages != nullptr) != (a->free_count != nullptr) || (a->free_pages && !a->page_table)) return FSA_ERR_INVALID_ARG;
  if (fsa_kv_append_rotary_workspace_ints(a) > 0 && !a->place_ws) return FSA_ERR_INVALID_ARG;
  const long long total = a->cu_seqlens_new ? (long long)a->total : (long long)a->batch * a->new_tokens;
  if (total < 0 || total > 0x7fffffffll) return FSA_ERR_INVALID_ARG;
  if (total == 0) return FSA_OK;
  const void* ptrs[4] = {a->q, a->k_new, a->v_new, a->q_out};
  for (int i = 0; i < 4; ++i)
    if (ptrs[i] && !aligned_to(ptrs[i], i == 3 && fp8 ? 1 : 2)) return FSA_ERR_INVALID_ARG;
  const int cs = fp8 ? 1 : 2;
  if (!aligned_to(a->k_cache, cs) || !aligned_to(a->v_cache, cs)) return FSA_ERR_INVALID_ARG;

  AppendParams p = {};
  Width w;
  if (a->heads_q > 0) {
    w.address(a->q, 2);
    w.address(a->q_out, cs);
    for (int64_t s : {a->q_stride_b, a->q_stride_s, a->q_stride_h, a->q_out_stride_b, a->q_out_stride_s, a->q_out_stride_h}) w.also(s);
  }
  w.address(a->k_new, 2);
  w.address(a->v_new, 2);
  w.address(a->k_cache, cs);
  w.address(a->v_cache, cs);
  for (int64_t s : {a->k_stride_b, a->k_stride_s, a->k_stride_h, a->v_stride_b, a->v_stride_s, a->v_stride_h, a->k_cache_stride_b,
                    a->k_cache_stride_s, a->k_cache_stride_h, a->v_cache_stride_b, a->v_cache_stride_s, a->v_cache_stride_h})
    w.also(s);
  const int v = make_shape(&p.r, w, a->cos, a->sin, a->table_stride, a->table_rows, a->table_dtype, a->head_dim, a->rotary_dim);
  p.q = a->q; p.k = a->k_new; p.v = a->v_new;
  p.q_out = a->q_out; p.k_cache = a->k_cache; p.v_cache = a->v_cache;
  p.used = a->seqused_k;
  p.page_table = a->page_table;
  p.free_pages = a->free_pages;
  p.free_count = a->free_count;
  p.cu = a->cu_seqlens_new;
  p.offsets = a->seqlen_offsets;
  p.q_scale = a->q_scale; p.k_scale = a->k_scale; p.v_scale = a->v_scale;
  p.place = reinterpret_cast<int2*>(a->place_ws);
  p.status = a->status;
  p.q_sb = a->q_stride_b; p.q_ss = a->q_stride_s; p.q_sh = a->q_stride_h;
  p.k_sb = a->k_stride_b; p.k_ss = a->k_stride_s; p.k_sh = a->k_stride_h;
  p.v_sb = a->v_stride_b; p.v_ss = a->v_stride_s; p.v_sh = a->v_stride_h;
  p.qo_sb = a->q_out_stride_b; p.qo_ss = a->q_out_stride_s; p.qo_sh = a->q_out_stride_h;
  p.c_sb = a->k_cache_stride_b; p.c_ss = a->k_cache_stride_s; p.c_sh = a->k_cache_stride_h;
  p.vc_sb = a->v_cache_stride_b; p.vc_ss = a->v_cache_stride_s; p.vc_sh = a->v_cache_stride_h;
  p.pt_stride = a->page_table_stride;
  p.batch = a->batch;
  p.new_tokens = a->new_tokens;
  p.total = (int)total;
  p.heads_q = a->heads_q;
  p.heads_kv = a->heads_kv;
  p.capacity = a->capacity;
  p.page_size = a->page_size;
  p.max_pages = a->max_pages;
  p.num_pages = a->num_pages;
  p.offset = a->offset;
  p.advance = a->advance;
  p.cache_dtype = a->cache_dtype;
  const int heads = a->heads_q + 2 * a->heads_kv;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (append_in_one_step(a)) {
    const long long items = (long long)a->new_tokens * heads * p.r.units;
    const int threads = items >= 1024 ? 1024 : (int)((items + 31) & ~31ll);
    const cudaError_t e = for_each_form(a->dtype, v, a->interleaved, false, [&](auto t, auto vv, auto il, auto) {
      return launch_early(append_step_kernel<decltype(t), vv(), il()>, (unsigned)a->batch, threads, 0, stream, 1, p);
    });
    return e == cudaSuccess ? FSA_OK : FSA_ERR_LAUNCH;
  }
  const bool many = total * heads * p.r.units >= 148ll * 2048;
  p.slots = many ? (heads + HEADS_PER_THREAD - 1) / HEADS_PER_THREAD : heads;
  const long long blocks = (total * p.slots * p.r.units + THREADS - 1) / THREADS;
  if (blocks * THREADS > 0xffffffffll) return FSA_ERR_UNSUPPORTED;  // threads are counted in 32 bits
  // a warp looks at a sequence's slots where it may have many
  const int lanes = a->page_table && total / a->page_size > 2ll * a->batch ? 32 : 1;
  cudaError_t e = launch_early(append_place_kernel, 1u, 1024, 0, stream, 1, p, lanes);
  if (e != cudaSuccess) return FSA_ERR_LAUNCH;
  e = for_each_form(a->dtype, v, a->interleaved, many, [&](auto t, auto vv, auto il, auto hpt) {
    return launch_early(append_rows_kernel<decltype(t), vv(), il(), hpt()>, (unsigned)blocks, THREADS, 0, stream, 1, p);
  });
  return e == cudaSuccess ? FSA_OK : FSA_ERR_LAUNCH;
}
