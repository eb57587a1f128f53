// Rotary positions with several axes, forward and gradient: fsa_rotary's rotation, with the angle of pair i at the position that the token
// has on the pair's axis,
//   y1 = x1 cos[p_axis(i), i] - x2 sin[p_axis(i), i]      y2 = x2 cos[p_axis(i), i] + x1 sin[p_axis(i), i]
//
// Bound by memory as that one is, and laid out like it: a thread turns two chunks of V elements of up to four heads of a token, so that it
// fetches its V angles once for four heads. Angles come from up to four rows of the tables; chunks whose pairs lie on one axis (runs of pairs)
// fetch them four at a time, others (axes dealt out pair by pair) one by one. (4 x 4096 tokens, 32 + 8 heads of 128, three runs: 58.5 us a direction, 5.7 TB/s,
// 0.88 of a copy's rate; 20 k packed tokens, 32 heads of 80, two axes dealt out, neighbouring pairs: 42 us, 4.9 TB/s.)
#include "fsa_axes.cuh"

namespace fsa {

namespace {

struct AxesParams {
  RotaryShape r;
  AxisMap m;
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int* status;
  long long q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, qo_sb, qo_ss, qo_sh, ko_sb, ko_ss, ko_sh;
  int batch, seqlen, total;   // total: tokens of the call
  int heads_q, heads, slots;  // heads: of q and k; slots: threads' groups of heads a token
  float sign;                 // -1: the gradient
};

template <typename T, int V, bool IL, int HPT>
__global__ void __launch_bounds__(THREADS) rotary_axes_kernel(const __grid_constant__ AxesParams p) {
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
  if (p.batch > 1) {
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
  int pos[FSA_MAX_AXES];
  const bool live = load_positions(p.m, bi, si, pos);
  if (!live) report_status(p.status, STATUS_NO_ANGLES);
  const bool turns = u < p.r.turned;
  float c[V], s[V];
  if (live && turns) {
    load_axis_angles<V, IL>(p.r, p.m, pos, a, b, c, s);
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
      if (!live) {  // without angles: zeros
        xa[i].raw = {};
        xb[i].raw = {};
      }
      *reinterpret_cast<decltype(xa[i].raw)*>(dst + a) = xa[i].raw;
      if (has_b) *reinterpret_cast<decltype(xa[i].raw)*>(dst + b) = xb[i].raw;
    }
  }
}

}  // namespace

}  // namespace fsa

extern "C" int fsa_rotary_axes(const FsaRotaryAxesArgs* a, void* stream_) {
  using namespace fsa;
  if (!a || !a->status || !a->position_ids || (a->heads_q > 0 && (!a->q || !a->q_out)) || (a->heads_k > 0 && (!a->k || !a->k_out)))
    return FSA_ERR_INVALID_ARG;
  if (a->heads_q < 0 || a->heads_k < 0 || a->heads_q + a->heads_k <= 0 || a->head_dim <= 0 || a->batch <= 0 || a->seqlen < 0)
    return FSA_ERR_INVALID_ARG;
  if ((a->dtype != FSA_DT_BF16 && a->dtype != FSA_DT_FP16) || a->head_dim > 256) return FSA_ERR_UNSUPPORTED;
  if (!table_ok(a->cos, a->sin, a->table_rows, a->table_dtype, a->head_dim, a->rotary_dim)) return FSA_ERR_INVALID_ARG;
  if (!axis_bits_ok(a->axis_bits, a->rotary_dim / 2, a->axes)) return FSA_ERR_INVALID_ARG;
  const long long total = (long long)a->batch * a->seqlen;
  if (total > 0x7fffffffll) return FSA_ERR_INVALID_ARG;
  if (total == 0) return FSA_OK;
  const void* ptrs[4] = {a->q, a->k, a->q_out, a->k_out};
  for (const void* x : ptrs)
    if (x && !aligned_to(x, 2)) return FSA_ERR_INVALID_ARG;

  AxesParams p = {};
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
  make_axis_map(&p.m, a->axis_bits, a->position_ids, a->position_stride_a, a->position_stride_b, a->position_stride_s, a->axes,
                a->position_ids_int64, a->table_rows);
  p.q = a->q;
  p.k = a->k;
  p.q_out = a->q_out;
  p.k_out = a->k_out;
  p.status = a->status;
  p.q_sb = a->q_stride_b; p.q_ss = a->q_stride_s; p.q_sh = a->q_stride_h;
  p.k_sb = a->k_stride_b; p.k_ss = a->k_stride_s; p.k_sh = a->k_stride_h;
  p.qo_sb = a->q_out_stride_b; p.qo_ss = a->q_out_stride_s; p.qo_sh = a->q_out_stride_h;
  p.ko_sb = a->k_out_stride_b; p.ko_ss = a->k_out_stride_s; p.ko_sh = a->k_out_stride_h;
  p.batch = a->batch;
  p.seqlen = a->seqlen;
  p.total = (int)total;
  p.heads_q = a->heads_q;
  p.heads = a->heads_q + a->heads_k;
  p.sign = a->transposed ? -1.f : 1.f;
  const bool many = total * p.heads * p.r.units >= 148ll * 2048;
  p.slots = many ? (p.heads + HEADS_PER_THREAD - 1) / HEADS_PER_THREAD : p.heads;
  const long long blocks = (total * p.slots * p.r.units + THREADS - 1) / THREADS;
  if (blocks * THREADS > 0xffffffffll) return FSA_ERR_UNSUPPORTED;  // threads are counted in 32 bits
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const cudaError_t e = for_each_form(a->dtype, v, a->interleaved, many, [&](auto t, auto vv, auto il, auto hpt) {
    return launch_early(rotary_axes_kernel<decltype(t), vv(), il(), hpt()>, (unsigned)blocks, THREADS, 0, stream, 1, p);
  });
  return e == cudaSuccess ? FSA_OK : FSA_ERR_LAUNCH;
}
