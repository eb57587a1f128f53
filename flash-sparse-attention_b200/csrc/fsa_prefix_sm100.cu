// Attention of a batch of single queries over a prefix that all sequences share, sm_100a.
//
//   s[r, n] = q[r] . k[n],  o[r] = sum_n 2^(c (s[r, n] - m)) v[n] / l[r],  c = softmax_scale * log2(e),
//
// for the rows r = (sequence, query head of the group) of one KV head against the same keys: with the batch on the M side the
// prefix is read once for all sequences and its products run on tcgen05, where a decode of each sequence would read it
// `batch` times. What it leaves are partial results (normalised, with base-2 log-sum-exps), which prefix_merge_kernel joins
// with those of the sequences' own keys (dec_kernel).
//
// One CTA an SM; every CTA takes an equal share of the work, counted in (query tile of 128 rows) x (key tile of 128 keys): the
// items (KV head, pair of query tiles) lie behind one another, cut into as many pieces as there are CTAs, so a piece may end inside one
// item and begin the next, and every piece of an item leaves a partial result. Inside a CTA two softmax warpgroups, each with a score
// tile and an output accumulator in TMEM, alternate on the tensor pipe: on two query tiles that use the same key tile, or, where the item
// has one query tile, on even and odd key tiles of it.
//
// Bound: few rows - the prefix's bytes (64 KB a key tile and KV head); from about 400 rows a KV head on the chain
// S -> softmax -> P V of the two groups, as in the forward.
#include <type_traits>

#include "fsa_aux.h"
#include "fsa_params.h"
#include "fsa_ptx.cuh"

namespace fsa {

namespace {

constexpr int PM = 128;        // rows of a query tile
constexpr int PN = 128;        // keys of a key tile
constexpr int P_THREADS = 384; // two softmax warpgroups, and K producer, MMA issuer, V producer, one idle warp
constexpr int W_K = 8, W_ISSUE = 9, W_V = 10;

template <int HD>
struct PrefixSmem {
  static constexpr int kTile = 128 * HD * 2;            // bytes of a Q, K or V tile
  static constexpr int kStages = HD == 64 ? 4 : 2;      // of K and of V
  static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + kStages * kTile, kBars = kV + kStages * kTile;
  static constexpr int kTotal = kBars + 256 + 1024;     // 1024: the base is aligned by hand
};

struct PrefixBars {
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t v_fixed;                      // rows behind the prefix's end are cleared
  uint64_t q_full[2], s_full[2], p_full[2], o_final[2];
  uint64_t done;                         // everything the tensor pipe was given
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(PrefixBars) <= 256, "fits its room");

// Bounded wait that does not look at the abort flag: for what has been started and will come to its end.
__device__ __forceinline__ void wait_out(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - t0 < FSA_WAIT_CYCLES) {
  }
}

// The key tiles [t0, t1) of an item that a CTA computes.
struct PrefixSegment {
  int hkv, pair, t0, t1;
};

// Work is counted in query tiles x key tiles: an item has `tiles` key tiles, each counting as many as the item has query tiles (one or two).
struct PrefixWork {
  int q_tiles;      // query tiles of a KV head
  int pairs;        // items of a KV head
  int tiles;        // key tiles
  int ctas;         // CTAs that have work
  long long total;

  __device__ __forceinline__ PrefixWork(const PrefixParams& p) {
    const int keys = p.used ? max(0, min(*p.used, p.keys)) : p.keys;
    q_tiles = p.q_tiles;
    pairs = (q_tiles + 1) >> 1;
    tiles = (keys + PN - 1) / PN;
    total = (long long)p.Hkv * q_tiles * tiles;
    ctas = (int)min((long long)p.ctas, total);
  }
  __device__ __forceinline__ int weight(int pair) const { return 2 * pair + 1 < q_tiles ? 2 : 1; }
  __device__ __forceinline__ long long item_start(int item) const {  // item = hkv * pairs + pair
    return (long long)(item / pairs) * q_tiles * tiles + 2ll * (item % pairs) * tiles;
  }
  __device__ __forceinline__ long long share_start(int cta) const { return total * cta / ctas; }
  // The first key tile of an item that does not begin before place x; a key tile belongs to the CTA that holds its start.
  __device__ __forceinline__ int first_tile(int item, long long x) const {
    const int w = weight(item % pairs);
    const long long off = x - item_start(item);
    return off <= 0 ? 0 : (int)min((off + w - 1) / w, (long long)tiles);
  }
  __device__ __forceinline__ int item_at(long long x) const {
    const long long per_head = (long long)q_tiles * tiles;
    const int h = (int)(x / per_head);
    return h * pairs + min((int)((x - h * per_head) / (2ll * tiles)), pairs - 1);
  }
  __device__ __forceinline__ int cta_at(long long x) const { return (int)(((x + 1) * ctas - 1) / total); }  // the share that holds place x
};

template <int HD, typename T>
__global__ void __launch_bounds__(P_THREADS, 1) prefix_kernel(const __grid_constant__ PrefixParams p) {
  using SM = PrefixSmem<HD>;
  constexpr int STAGES = SM::kStages;
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t TMEM_S = 0, TMEM_O = 256;  // two tiles of 128 columns each; O of group q at 256 + 128 q
  after_previous();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  PrefixBars* bars = reinterpret_cast<PrefixBars*>(smem + SM::kBars);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &bars->abort_flag;

  const PrefixWork work(p);
  if ((int)blockIdx.x >= work.ctas) return;  // nothing for this CTA: before any barrier or TMEM exists
  const long long x0 = work.share_start(blockIdx.x), x1 = work.share_start(blockIdx.x + 1);
  const int item0 = work.item_at(x0), item1 = work.item_at(x1 - 1);
  const int keys = p.used ? max(0, min(*p.used, p.keys)) : p.keys;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], 1);
    }
    mbar_init(&bars->v_fixed, 1);
    mbar_init(&bars->done, 1);
    for (int q = 0; q < 2; ++q) {
      mbar_init(&bars->q_full[q], 4);
      mbar_init(&bars->s_full[q], 1);
      mbar_init(&bars->p_full[q], 4);
      mbar_init(&bars->o_final[q], 1);
    }
    bars->abort_flag = (*reinterpret_cast<volatile int*>(p.status) != 0) ? 1 : 0;
    mbar_fence_init();
  }
  if (warp == W_K) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  // One segment of this CTA's share: false when the rounding to whole key tiles leaves nothing of the item.
  auto segment = [&](int item, PrefixSegment& g) {
    g.hkv = item / work.pairs;
    g.pair = item % work.pairs;
    g.t0 = work.first_tile(item, x0);
    g.t1 = work.first_tile(item, x1);
    return g.t0 < g.t1;
  };

  if (warp >= W_K) {
    // 384 x 168 registers at launch = 256 x 216 + 128 x 72
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == W_K || warp == W_V) {
      // =============================== K and V producers ========================================
      const bool is_v = warp == W_V;
      const CUtensorMap* map = is_v ? &p.map_v : &p.map_k;
      uint64_t* full = is_v ? bars->v_full : bars->k_full;
      uint64_t* empty = is_v ? bars->v_empty : bars->k_empty;
      uint8_t* ring = smem + (is_v ? SM::kV : SM::kK);
      if (lane == 0) tma_prefetch_desc(map);
      bool ok = !*abort_flag;
      int n = 0;  // tiles requested so far
      PrefixSegment g;
      for (int item = item0; item <= item1 && ok; ++item) {
        if (!segment(item, g)) continue;
        for (int t = g.t0; t < g.t1 && ok; ++t, ++n) {
          const int s = n % STAGES;
          if (n >= STAGES) ok = mbar_wait(&empty[s], (n / STAGES - 1) & 1, abort_flag);
          if (!ok) break;
          uint8_t* dst = ring + s * SM::kTile;
          if (lane == 0) {
            mbar_arrive_expect_tx(&full[s], SM::kTile);
            if (p.page_table) {
              const int page_shift = 31 - __clz(p.page_size), row_shift = min(page_shift, 7);
              for (int r = 0; r < PN; r += 1 << row_shift) {
                const int n0 = t * PN + r;
                int page = -1;  // outside the pool: TMA fills zeros
                if (n0 < keys) {
                  page = p.page_table[n0 >> page_shift];
                  if (page < 0 || page >= p.num_pages) {
                    page = -1;
                    atomicExch(p.status, 3);
                  }
                }
                for (int d = 0; d < HD; d += 64)
                  tma_load_4d(dst + (d / 64) * (PN * 128) + r * 128, map, &full[s], d, g.hkv, n0 & (p.page_size - 1), page);
              }
            } else {
              for (int d = 0; d < HD; d += 64) tma_load_4d(dst + (d / 64) * (PN * 128), map, &full[s], d, g.hkv, t * PN, 0);
            }
          }
          __syncwarp();
          if (is_v && (t + 1) * PN > keys) {
            // Keys behind the end carry probability 0, but what lies in their V rows may be anything, and 0 * NaN is NaN.
            ok = mbar_wait(&full[s], (n / STAGES) & 1, abort_flag);
            if (!ok) break;
            const int r0 = keys - t * PN;
            constexpr int CPR = HD / 8;
            for (int i = lane; i < (PN - r0) * CPR; i += 32) {
              const int r = r0 + i / CPR, c = i % CPR;
              *reinterpret_cast<uint4*>(dst + (c >> 3) * (PN * 128) + sw128_offset(r, c & 7)) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->v_fixed);
          }
        }
      }
      // no copy is in flight when the CTA ends, whatever ended the loop
      for (int i = max(0, n - STAGES); i < n; ++i) wait_out(&full[i % STAGES], (i / STAGES) & 1);
    } else if (warp == W_ISSUE) {
      // =============================== MMA issuer ===============================================
      constexpr uint32_t idesc_s = umma_idesc_f16(PM, PN, IS_BF16, false, false);
      constexpr uint32_t idesc_o = umma_idesc_f16(PM, HD, IS_BF16, false, true);
      constexpr int KK_QK = HD / 16, KK_PV = PN / 16;
      const uint32_t lead = elect_one();
      const uint32_t dq = umma_desc_lo(smem_u32(smem + SM::kQ), 16), dk = umma_desc_lo(smem_u32(smem + SM::kK), 16);
      const uint32_t dv = umma_desc_lo(smem_u32(smem + SM::kV), PN * 128);
      bool ok = !*abort_flag;
      int nk = 0, nv = 0, n_fixed = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};
      auto wait_k = [&]() { return mbar_wait(&bars->k_full[nk % STAGES], (nk / STAGES) & 1, abort_flag); };
      auto issue_s = [&](int q) {
        const uint32_t a = dq + ((q * SM::kTile) >> 4), b = dk + (((nk % STAGES) * SM::kTile) >> 4);
#pragma unroll
        for (int kk = 0; kk < KK_QK; ++kk) {
          const uint32_t off = (kk >> 2) * (PN * 128) + (kk & 3) * 32;
          umma_ss_lead(lead, tmem + TMEM_S + q * 128, umma_desc_at(a, off), umma_desc_at(b, off), idesc_s, kk > 0);
        }
        umma_commit_lead(lead, &bars->s_full[q]);
      };
      auto release_k = [&]() {
        umma_commit_lead(lead, &bars->k_empty[nk % STAGES]);
        ++nk;
      };
      auto issue_pv = [&](int q, bool first) {
        const uint32_t b = dv + (((nv % STAGES) * SM::kTile) >> 4);
#pragma unroll
        for (int kk = 0; kk < KK_PV; ++kk)
          umma_ts_lead(lead, tmem + TMEM_O + q * 128, tmem + TMEM_S + q * 128 + kk * 8, umma_desc_at(b, kk * 2048), idesc_o,
                       (kk > 0 || !first) ? 1u : 0u);
      };
      auto wait_q = [&](int q) { return mbar_wait(&bars->q_full[q], n_q[q]++ & 1, abort_flag); };
      auto wait_p = [&](int q) { return mbar_wait(&bars->p_full[q], n_p[q]++ & 1, abort_flag); };
      PrefixSegment g;
      for (int item = item0; item <= item1 && ok; ++item) {
        if (!segment(item, g)) continue;
        const int n = g.t1 - g.t0;
        const bool two = work.weight(g.pair) == 2;
        // the first score tile of each group
        if (two) {
          ok = wait_k() && wait_q(0) && wait_q(1);
          if (!ok) break;
          tc_fence_after();
          issue_s(0);
          issue_s(1);
          release_k();
        } else {
          for (int q = 0; q < min(n, 2) && ok; ++q) {
            ok = wait_k() && wait_q(q);
            if (!ok) break;
            tc_fence_after();
            issue_s(q);
            release_k();
          }
        }
        for (int i = 0; i < n && ok; ++i) {
          ok = mbar_wait(&bars->v_full[nv % STAGES], (nv / STAGES) & 1, abort_flag);
          if (ok && (g.t0 + i + 1) * PN > keys) ok = mbar_wait(&bars->v_fixed, n_fixed++ & 1, abort_flag);
          if (!ok) break;
          if (two) {
            const bool more = i + 1 < n;
            if (more) ok = wait_k();
            for (int q = 0; q < 2 && ok; ++q) {
              ok = wait_p(q);
              if (!ok) break;
              tc_fence_after();
              issue_pv(q, i == 0);
              if (more)
                issue_s(q);
              else
                umma_commit_lead(lead, &bars->o_final[q]);
            }
            if (!ok) break;
            umma_commit_lead(lead, &bars->v_empty[nv % STAGES]);
            if (more) release_k();
          } else {
            const int q = i & 1;
            ok = wait_p(q);
            if (!ok) break;
            tc_fence_after();
            issue_pv(q, i < 2);
            umma_commit_lead(lead, &bars->v_empty[nv % STAGES]);
            if (i + 2 < n) {
              ok = wait_k();
              if (!ok) break;
              tc_fence_after();
              issue_s(q);
              release_k();
            } else {
              umma_commit_lead(lead, &bars->o_final[q]);
            }
          }
          ++nv;
        }
      }
      umma_commit_lead(lead, &bars->done);
      wait_out(&bars->done, 0);
    }
  } else {
    // =============================== softmax groups =============================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int q = warp >> 2, wq = warp & 3, row = wq * 32 + lane;
    const uint32_t lane_addr = uint32_t(wq * 32) << 16;
    const uint32_t tS = tmem + lane_addr + TMEM_S + q * 128, tO = tmem + lane_addr + TMEM_O + q * 128;
    const float c = p.scale_log2;
    bool ok = !*abort_flag;
    int n_s = 0, n_o = 0;
    PrefixSegment g;
    for (int item = item0; item <= item1 && ok; ++item) {
      if (!segment(item, g)) continue;
      const bool two = work.weight(g.pair) == 2;
      const int first = two ? g.t0 : g.t0 + q, step = two ? 1 : 2;
      if (first >= g.t1) continue;  // a segment of one key tile has nothing for the second group
      // ---- the group's query tile: rows (sequence, head of the group) -> shared memory, 128-byte swizzle ----
      // (all score tiles of the segment before have been waited for, so no MMA reads the old one)
      const int r = (2 * g.pair + (two ? q : 0)) * PM + row;
      const bool live = r < p.rows;
      const int b = live ? r / p.G : 0, head = g.hkv * p.G + (live ? r - b * p.G : 0);
      {
        const T* src = reinterpret_cast<const T*>(p.q) + (long long)b * p.q_sb + (long long)head * p.q_sh;
        uint8_t* dst = smem + SM::kQ + q * SM::kTile;
        uint4 v[HD / 8];
#pragma unroll
        for (int i = 0; i < HD / 8; ++i)
          v[i] = live && i * 8 < p.D ? *reinterpret_cast<const uint4*>(src + i * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < HD / 8; ++i)
          *reinterpret_cast<uint4*>(dst + (i >> 3) * (PM * 128) + sw128_offset(row, i & 7)) = v[i];
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->q_full[q]);
      }
      const bool idle = !__any_sync(0xffffffffu, live);  // no row of this warp exists: what it leaves in P is never read out
      float m_ref = -INFINITY;  // what the exponentials are relative to; it moves when the maximum has grown by 2^8
      float l = 0.f;            // their sum
      for (int t = first; t < g.t1; t += step) {
        ok = mbar_wait(&bars->s_full[q], n_s++ & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (!idle) {
          uint32_t sr[PN];
#pragma unroll
          for (int ch = 0; ch < PN / 32; ++ch) tmem_ld32(tS + ch * 32, &sr[ch * 32]);
          tmem_ld_wait();
          if ((t + 1) * PN > keys) {
            const int n_live = keys - t * PN;
#pragma unroll
            for (int i = 0; i < PN; ++i)
              if (i >= n_live) sr[i] = 0xff800000u;
          }
          float mx[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mx[j] = fmaxf(__uint_as_float(sr[j * 32]), __uint_as_float(sr[j * 32 + 1]));
#pragma unroll
            for (int i = 2; i < 32; i += 2)
              mx[j] = max3(mx[j], __uint_as_float(sr[j * 32 + i]), __uint_as_float(sr[j * 32 + i + 1]));
          }
          const float m_cand = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), m_ref);
          const bool none = m_cand == -INFINITY;  // every score so far is -inf: no reference yet, the exponentials are zeros
          const bool need = !none && !((m_cand - m_ref) * c <= 8.0f);
          float scale = 1.0f;
          if (need) {
            scale = ex2_approx((m_ref - m_cand) * c);
            m_ref = m_cand;
            l *= scale;
          }
          // (this tile's scores were issued behind the P V product before them, so O is at rest)
          if (t != first && __any_sync(0xffffffffu, need)) {
            constexpr int RC = HD == 64 ? 16 : 32;
#pragma unroll 1
            for (int ch = 0; ch < HD / RC; ++ch) {
              uint32_t o[RC];
              if constexpr (RC == 32)
                tmem_ld32(tO + ch * RC, o);
              else
                tmem_ld16(tO + ch * RC, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < RC; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * scale);
              if constexpr (RC == 32)
                tmem_st32(tO + ch * RC, o);
              else
                tmem_st16(tO + ch * RC, o);
            }
          }
          const float2 c2 = make_float2(c, c);
          const float neg = none ? 0.f : -(m_ref * c);
          const float2 nm2 = make_float2(neg, neg);
          float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int ch = 0; ch < PN / 32; ++ch) {
            uint32_t pk[16];
            const uint32_t* src = &sr[ch * 32];
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float2 ta = fma2(make_float2(__uint_as_float(src[i]), __uint_as_float(src[i + 1])), c2, nm2);
              const float2 tb = fma2(make_float2(__uint_as_float(src[i + 2]), __uint_as_float(src[i + 3])), c2, nm2);
              const float2 ea = make_float2(ex2_approx(ta.x), ex2_approx(ta.y)), eb = make_float2(ex2_approx(tb.x), ex2_approx(tb.y));
              sum2[0] = add2(sum2[0], ea);
              sum2[1] = add2(sum2[1], eb);
              // P is rounded to the inputs' type, the sum is not: the rounding errors of a row are independent and average out
              pk[i >> 1] = pack2<T>(ea.x, ea.y);
              pk[(i >> 1) + 1] = pack2<T>(eb.x, eb.y);
            }
            tmem_st16(tS + ch * 16, pk);
          }
          tmem_st_wait();
          l += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[q]);
      }
      if (!ok) break;
      // ---- the segment's partial result ----
      ok = mbar_wait(&bars->o_final[q], n_o++ & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      if (!idle) {
        const int piece = (int)blockIdx.x - work.cta_at(work.item_start(item));
        const long long slot = 2 * piece + (two ? 0 : q);
        const bool dead = l == 0.f || l != l;
        const float inv = dead ? 1.f : 1.f / l;
        float* dst = p.out_partial + slot * p.op_ss + ((long long)b * p.Hq + head) * p.D;
#pragma unroll
        for (int ch = 0; ch < HD / 32; ++ch) {
          uint32_t o[32];
          tmem_ld32(tO + ch * 32, o);
          tmem_ld_wait();
          if (live) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              if (ch * 32 + i < p.D)
                *reinterpret_cast<float4*>(dst + ch * 32 + i) =
                    make_float4(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv, __uint_as_float(o[i + 2]) * inv,
                                __uint_as_float(o[i + 3]) * inv);
          }
        }
        // (a row with NaN among its scores has l = NaN and is NaN as a whole)
        if (live) p.lse_partial[slot * p.lp_ss + (long long)head * p.B + b] = l == 0.f ? -INFINITY : m_ref * c + log2f(l);
      }
      tc_fence_before();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicExch(p.status, 1);
  if (warp == W_K) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One warp joins the partial results of a (sequence, query head): the pieces of its item over the prefix - which shares of the work
// they are follows from the same arithmetic - and the splits over the sequence's own keys. Weights 2^(lse - max); 32 at a time.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) prefix_merge_kernel(const PrefixParams p) {
  after_previous();
  const int lane = threadIdx.x & 31;
  const long long at = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (at >= (long long)p.B * p.Hq || *reinterpret_cast<volatile int*>(p.status) != 0) return;
  const int b = (int)(at / p.Hq), head = (int)(at - (long long)b * p.Hq);
  const int hkv = head / p.G, r = b * p.G + head - hkv * p.G;
  const PrefixWork work(p);
  const int item = hkv * work.pairs + r / (2 * PM);
  const bool two = work.weight(item % work.pairs) == 2;
  int c_first = 0, pieces = 0;
  if (work.total > 0) {
    const long long start = work.item_start(item);
    c_first = work.cta_at(start);
    pieces = work.cta_at(start + (long long)work.weight(item % work.pairs) * work.tiles - 1) - c_first + 1;
  }
  const int slots = 2 * pieces, count = slots + p.splits;
  const float* lp = p.lse_partial + (long long)head * p.B + b;
  const float* op = p.out_partial + at * p.D;
  // slot i of the prefix is written when its piece has key tiles for that group
  auto lse_of = [&](int i) {
    if (i >= count) return -INFINITY;
    if (i >= slots) return __ldcg(lp + (long long)(p.slots + i - slots) * p.lp_ss);
    const int cta = c_first + (i >> 1);
    const int t0 = work.first_tile(item, work.share_start(cta)), t1 = work.first_tile(item, work.share_start(cta + 1));
    if ((i & 1) ? (two || t1 - t0 < 2) : t1 <= t0) return -INFINITY;
    return __ldcg(lp + (long long)i * p.lp_ss);
  };
  float top = -INFINITY, sum = 0.f, acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  const int d0 = lane * VEC;
  const bool active = d0 < p.D;
  for (int s0 = 0; s0 < count; s0 += 32) {
    const float lse = lse_of(s0 + lane);
    float m = lse;
    unsigned used = __ballot_sync(0xffffffffu, lse != -INFINITY);  // NaN counts
    const bool nan = __any_sync(0xffffffffu, lse != lse);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = fmaxf(m, top);
    if (nan) m = __int_as_float(0x7fffffff);
    if (m == -INFINITY) continue;
    const float old = top == -INFINITY ? 0.f : exp2f(top - m);
    const float w = lse == -INFINITY ? 0.f : exp2f(lse - m);
    float ws = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
    sum = sum * old + ws;
    top = m;
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] *= old;
    while (used) {
      const int j = __ffs(used) - 1;
      used &= used - 1;
      const int i = s0 + j;
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const float* src = op + (long long)(i < slots ? i : p.slots + i - slots) * p.op_ss + d0;
      if (active) {
        if constexpr (VEC == 4) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
          acc[0] += wj * v.x;
          acc[1] += wj * v.y;
          acc[2] += wj * v.z;
          acc[3] += wj * v.w;
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
          acc[0] += wj * v.x;
          acc[1] += wj * v.y;
        }
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (active) {
    T* dst = reinterpret_cast<T*>(p.out) + (long long)b * p.o_sb + (long long)head * p.o_sh + d0;
#pragma unroll
    for (int i = 0; i < VEC; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack2<T>(acc[i] * inv, acc[i + 1] * inv);
  }
  if (lane == 0)
    p.lse[(long long)b * p.l_sb + (long long)head * p.l_sh] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

template <int HD, typename T>
cudaError_t launch_one(const PrefixParams& p, cudaStream_t stream) {
  auto kern = prefix_kernel<HD, T>;
  constexpr int smem = PrefixSmem<HD>::kTotal;
  static std::atomic<unsigned long long> opted_in{0};
  if (cudaError_t e = smem_opt_in(kern, smem, opted_in); e != cudaSuccess) return e;
  if (p.ctas > 0)  // a prefix without positions leaves no pieces
    if (cudaError_t e = launch_early(kern, (unsigned)p.ctas, P_THREADS, smem, stream, 1, p); e != cudaSuccess) return e;
  const unsigned grid = (unsigned)(((long long)p.B * p.Hq + 7) / 8);
  return launch_early(prefix_merge_kernel<T, HD / 32>, grid, 256, 0, stream, 1, p);
}

}  // namespace

cudaError_t launch_prefix(const PrefixParams& p, int dtype, int head_dim, cudaStream_t stream) {
  if (head_dim == 64) return dtype == DT_BF16 ? launch_one<64, __nv_bfloat16>(p, stream) : launch_one<64, __half>(p, stream);
  return dtype == DT_BF16 ? launch_one<128, __nv_bfloat16>(p, stream) : launch_one<128, __half>(p, stream);
}

}  // namespace fsa
