// Angles of tokens that have a position on each of several axes: pair i is turned by the position on axis(i).
#pragma once
#include "fsa_rotary.cuh"

namespace fsa {

// Which axis a pair belongs to, two bits a pair; positions of a call's tokens.
struct AxisMap {
  uint32_t bits[8];
  const void* ids;
  long long id_sa, id_sb, id_ss;
  int axes, ids64, rows;  // rows: of the tables
};

// The positions of token (bi, si) on all axes; false where one lies outside the tables.
__device__ __forceinline__ bool load_positions(const AxisMap& m, long long bi, long long si, int pos[FSA_MAX_AXES]) {
  bool ok = true;
#pragma unroll
  for (int a = 0; a < FSA_MAX_AXES; ++a) {
    pos[a] = 0;
    if (a < m.axes) {
      const long long at = a * m.id_sa + bi * m.id_sb + si * m.id_ss;
      const long long x = m.ids64 ? reinterpret_cast<const long long*>(m.ids)[at] : reinterpret_cast<const int*>(m.ids)[at];
      ok = ok && x >= 0 && x < m.rows;
      pos[a] = (int)x;
    }
  }
  return ok;
}

__device__ __forceinline__ int on_axis(const int pos[FSA_MAX_AXES], uint32_t axis) {
  const int low = axis & 1 ? pos[1] : pos[0], high = axis & 1 ? pos[3] : pos[2];
  return axis & 2 ? high : low;
}

// N angles from pair `first` on (a multiple of N). Neighbouring pairs mostly share their axis, and then one row of the tables holds them.
template <int N>
__device__ __forceinline__ void load_axis_some(const RotaryShape& r, const AxisMap& m, const int pos[FSA_MAX_AXES], int first, float* c, float* s) {
  const uint32_t w = m.bits[first >> 4] >> (2 * (first & 15)), one = w & 3;
  constexpr uint32_t FIELDS = 0x55555555u & ((1u << (2 * N)) - 1);
  if (((w ^ one * FIELDS) & (3 * FIELDS)) == 0) {
    load_some<N>(r, on_axis(pos, one), first, c, s);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) load_some<1>(r, on_axis(pos, w >> (2 * i) & 3), first + i, c + i, s + i);
  }
}

// load_angles of fsa_rotary.cuh with the positions of several axes.
template <int V, bool IL>
__device__ __forceinline__ void load_axis_angles(const RotaryShape& r, const AxisMap& m, const int pos[FSA_MAX_AXES], int a, int b, float* c, float* s) {
  if constexpr (IL && V > 1) {
    load_axis_some<V / 2>(r, m, pos, a / 2, c, s);
    load_axis_some<V / 2>(r, m, pos, b / 2, c + V / 2, s + V / 2);
  } else {
    load_axis_some<V>(r, m, pos, IL ? a / 2 : a, c, s);
  }
}

inline void make_axis_map(AxisMap* m, const uint32_t* bits, const void* ids, int64_t sa, int64_t sb, int64_t ss, int axes, int ids64, int rows) {
  for (int i = 0; i < 8; ++i) m->bits[i] = bits[i];
  m->ids = ids;
  m->id_sa = sa;
  m->id_sb = sb;
  m->id_ss = ss;
  m->axes = axes;
  m->ids64 = ids64;
  m->rows = rows;
}

// Every pair's axis is one of the call's.
inline bool axis_bits_ok(const uint32_t* bits, int pairs, int axes) {
  if (axes < 1 || axes > FSA_MAX_AXES || pairs > 128) return false;
  for (int i = 0; i < pairs; ++i)
    if ((int)(bits[i >> 4] >> (2 * (i & 15)) & 3) >= axes) return false;
  return true;
}

}  // namespace fsa
