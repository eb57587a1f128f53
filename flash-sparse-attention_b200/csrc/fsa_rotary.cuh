// What the kernels that turn rows by their positions share: how a head's columns fall to threads, the angles, and where new rows lie in
// a cache (fsa_rotary.cu, fsa_quant_cache.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fsa_b200.h"
#include "fsa_params.h"
#include "fsa_ptx.cuh"

namespace fsa {

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

// New rows on their way into a cache.
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

// Where the rows of every sequence go (append_place_kernel), in one block.
cudaError_t launch_append_place(const AppendParams& p, int lanes, cudaStream_t stream);

// The widest chunk that everything allows: `bytes` collects the lowest set bits of what has to be a multiple of it.
struct Width {
  unsigned long long elems = 8;  // of strides, sizes and addresses in elements
  void also(long long n) { elems |= (unsigned long long)n; }
  void address(const void* ptr, int elem_bytes) {
    elems |= reinterpret_cast<uintptr_t>(ptr) / (unsigned)elem_bytes;
  }
  int v() const { return (int)(elems & (~elems + 1)); }  // lowest set bit, at most 8
};

inline bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

inline int make_shape(RotaryShape* r, Width w, const void* cos, const void* sin, long long table_stride, int table_rows, int table_dtype,
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

inline bool table_ok(const void* cos, const void* sin, int rows, int dtype, int head_dim, int rotary_dim) {
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

constexpr int HEADS_PER_THREAD = 4;  // of a call large enough to keep the GPU busy

}  // namespace fsa
