// Attention of a batch of single queries over a prefix that all sequences share and over each sequence's own keys, sm_100a.
//
//   s[r, n] = q[r] . k[n],  o[r] = sum_n 2^(c (s[r, n] - m)) v[n] / l[r],  c = softmax_scale * log2(e)
//
// Over the prefix, the rows r = (sequence, query head of the group) of one KV head meet the same keys: with them on the M side of tcgen05 the
// prefix is read once for all sequences, where a decode of each would read it `batch` times. Over a sequence's own keys only the G heads
// of the group share them; those tiles run through the same pipeline with G of 128 rows filled: a key tile's 64 KB take an SM's share of
// HBM about 2900 cycles where all SMs ask for them, its two products and one warp's softmax fewer.
//
// The work is a list of units of one key tile each (128 keys of one KV head):
//   pairs     prefix tile x two query tiles, for every KV head and pair of query tiles (a tile: the rows of as many sequences as
//             fit 128, or 128 heads of one)
//   singles   prefix tile x the last query tile, where their number is odd; own tile x the G rows of its sequence
// It is cut into shares of equal cost, one per CTA (one CTA an SM): items of pairs (an item: the units of the same rows and KV head)
// in equal pieces where that comes out, otherwise at any unit, so that a share may end inside an item and begin the next. Every piece
// of an item leaves a partial result - its O, reference maximum and sum - that prefix_merge_kernel joins. Lengths live on the device:
// every CTA works its share out from them.
//
// In a CTA two softmax warpgroups, each with a score tile and an accumulator in TMEM, alternate on the tensor pipe. They share the
// key tile of a pair; of the singles each walks its own half of the share ("stream"), tile by tile in turn.
//
// Bound: the keys' bytes, except where many sequences share a prefix (from about 400 rows a KV head): there the chain
// S -> softmax -> P V of the two groups, as in the forward.
#include <type_traits>

#include "fsa_aux.h"
#include "fsa_params.h"
#include "fsa_ptx.cuh"

namespace fsa {

namespace {

constexpr int PM = 128;         // rows of a query tile
constexpr int PN = 128;         // keys of a key tile
constexpr int OWN_BOX = 32;     // rows of the copies at the end of a sequence's own keys: no more than that is read in vain behind it
constexpr int DIRECT_ROWS = 8;  // of results that lanes write themselves; pieces of more have whole boxes of 32 rows
constexpr int P_THREADS = 384;  // two softmax warpgroups, and one warp each that requests K, issues the MMAs, requests V, plans
constexpr int W_K = 8, W_ISSUE = 9, W_V = 10, W_PLAN = 11;
constexpr int BATCH = 16;       // steps that the planner works out at a time, one a lane; it is two batches ahead at most
// What an SM's time goes to, in units of about 220 cycles: a pair of query tiles on a key tile (3900), a single one (1950 while others work on pairs
// and leave HBM to it: own keys alone come at 6.0 TB/s on 96 SMs, 1950 cycles a tile, at 3.6 on 48, 1640, and at 6.3 on 148), and what an item adds (results on
// their way out, and the next item's first scores): of own keys, and of a pair, whose 128 KB take 2000 to 2700 cycles to be written. In a call where 100 SMs
// work on own keys beside 48 on pairs a single takes 1.47 us with its share of items, where these make 1.2.
// Replayed calls of 32 query heads over 8 KV heads of 128, pages of 64, us, for 18 / 9 / 4 / 32, a single at 10, at 8, an item at 8, a pair's item at 16 and at 0:
//   64 sequences over 8192 + up to 1024 keys   45.6   45.8   49.8   45.9   45.6   45.8
//   256 over 1000 + up to 100                  43.1   43.3   43.4   47.0   47.9   46.1
//   100 over 20 000 + up to 1000               83.3   80.7   88.3   80.4   82.1   81.9
//   256 over 32 768 + up to 256                159    158    170    158    158    156
//   40 over 4000 + up to 200                   28.5   26.2   28.6   25.9   27.0   27.2
//   64 over 500 + up to 200                    20.8   20.8   20.8   20.5   20.8   25.8
//   235 over 2 + up to 645                     73.4   73.4   73.1   73.4   73.6   74.8
constexpr int COST_PAIR = 18, COST_SINGLE = 9, COST_ITEM = 4, COST_PAIR_ITEM = 32;

// What a softmax group has to know about the units of one item that it walks.
struct GroupSegment {
  int n;     // key tiles; 0: the group is done
  int keys;  // of the item from the first of these tiles on
  int rows;  // of the group's query tile that exist: the first ones
  int row0;  // of the workspaces: the piece's first row
  int shift; // place of the first row in the tile
  int gap;   // rows behind row0 at which the next piece is left out (0: it is not)
};
// A step: one key tile, with word of the segment that it begins, if it does. The planner's lanes work sixteen out at a time, ahead of the
// copies: step by step in the lane that also requests the tiles, indexes, lengths and pages took 5000 cycles a step, where a tile's bytes
// take 2900, and by a lane of its own the first came 10 000 cycles after the plan, most of them waits for instructions.
struct alignas(16) StepRecord {
  uint32_t info;  // STEP_*, keys in the tile (from bit 8), own: tile of the group's heads (from bit 16)
  int h, n0;      // KV head; first key
  int b;          // own: the sequence; prefix: the (first) query tile
  int page[4];    // of the tile's boxes, or of the one that holds them all
  int n, keys;    // of the segment, when this is its first step: key tiles; keys from here on
  int row0, gap;  // first row of its piece in the workspaces; see GroupSegment
};
static_assert(sizeof(StepRecord) == 48, "two batches fit");
struct PrefixBars {
  StepRecord rec[2 * BATCH];
  uint64_t rec_full[2], rec_empty[2];
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t seg_full[2][2], s_full[2], p_full[2], o_final[2];
  GroupSegment seg[2][2];
  uint64_t v_tail[4];    // V tiles with rows behind the last key: when those are cleared, v_full is told
  uint64_t done;         // everything the tensor pipe was given
  uint32_t v_info[4];
  uint32_t tmem_base;
  int abort_flag;
  // this CTA's share: pairs [a0, a1), singles [s[0], s[1]) and [s[1], s[2]) of the two streams, the sequence in which a stream
  // begins among the own keys and the tiles in front of it
  int a0, a1, s[3], b_at[2], cum_at[2];
  int ctas, tiles, keys, singles_prefix;
  int pair_id;  // number of this CTA's piece of pairs: those of an item follow one another
};
template <int HD>
struct PrefixSmem {
  static constexpr int kTile = 128 * HD * 2;        // bytes of a Q, K or V tile
  static constexpr int kStages = HD == 64 ? 4 : 2;  // of K and of V
  static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + kStages * kTile, kOut = kV + kStages * kTile, kBars = kOut + 8 * 4096;
  static constexpr int kTotal = kBars + (int)sizeof(PrefixBars) + 1024;  // 1024: the base is aligned by hand
};

enum : uint32_t { STEP_FIRST = 1u, STEP_LAST = 2u, STEP_OWN = 4u };  // of a segment; own keys

// Bounded wait that does not look at the abort flag: for what has been started and will come to its end.
__device__ __forceinline__ void wait_out(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - t0 < FSA_WAIT_CYCLES) {
  }
}

__device__ __forceinline__ int own_keys(const PrefixParams& p, int b) { return p.used ? max(0, min(p.used[b], p.own_keys)) : p.own_keys; }
__device__ __forceinline__ int tiles_of(int keys) { return (keys + PN - 1) / PN; }

// This CTA's share of the work, by all threads.
__device__ __forceinline__ void make_plan(const PrefixParams& p, PrefixBars* s, int2* warp_sum) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int prefix_keys = warp == 0 && p.prefix_used ? *p.prefix_used : p.prefix_keys;
  const int chunk = (p.B + P_THREADS - 1) / P_THREADS, b0 = tid * chunk, b1 = min(p.B, b0 + chunk);
  int mine = 0, some = 0;  // tiles, and sequences that have any
  for (int b = b0; b < b1; ++b) {
    const int u = tiles_of(own_keys(p, b));
    mine += u;
    some += u > 0;
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  some = __reduce_add_sync(0xffffffffu, some);
  if (lane == 31) warp_sum[warp] = make_int2(incl, some);
  __syncthreads();
  int cum = incl - mine, total_own = 0, sequences = 0;
#pragma unroll
  for (int w = 0; w < P_THREADS / 32; ++w) {
    const int2 v = warp_sum[w];
    if (w < warp) cum += v.x;
    total_own += v.x;
    sequences += v.y;
  }
  if (warp == 0) {
    const int keys = max(0, min(prefix_keys, p.prefix_keys)), tiles = tiles_of(keys);
    const int pairs = p.Hkv * p.pairs * tiles, odd = (p.q_tiles & 1) ? p.Hkv * tiles : 0, singles = odd + total_own * p.items_b;
    // Equal shares of the cost, in which items' share is spread over the units of their kind. Every CTA works the same bounds out, so they need not be
    // exact; a share is more than any unit's cost, so that every share between two that hold units of a kind holds one, too.
    const float pair_cost = pairs > 0 ? (float)COST_PAIR * pairs + (float)COST_PAIR_ITEM * p.Hkv * p.pairs : 0.f;
    const float single_cost = (float)COST_SINGLE * singles + (float)COST_ITEM * sequences * p.items_b, cost = pair_cost + single_cost;
    const float pairs_per = pairs > 0 ? __fdividef((float)pairs, pair_cost) : 1.f, singles_per = singles > 0 ? __fdividef((float)singles, single_cost) : 1.f;
    const float most = fmaxf(cost * fminf(pairs_per, singles_per) * 0.95f, 1.f);
    int ctas = cost > 0.f ? (int)fminf((float)p.ctas, most) : 0;
    const int cta = blockIdx.x, items = p.Hkv * p.pairs;
    float share = ctas > 0 ? __fdividef(cost, (float)ctas) : 0.f;
    // Where there are no more items of pairs than CTAs, each is cut into `cuts` equal pieces, one a CTA, and the pieces of a KV head over the same keys go to
    // neighbours, that read them at the same time. What their shares have left is singles, if it is some for each; if not, the other CTAs take
    // those. It is not done where the pieces come out too uneven. 256 sequences over 32 768 + up to 256 keys 171 us where pieces lie anywhere, so 159;
    // 256 over 16 000 + up to 64 107 and 98, 64 over 8192 + up to 1024 46.4 and 45.6, 256 over 1000 + up to 100 46.2 and 43.1, 64 over 500 + up to 200 24.0
    // and 20.8. One of the calls above loses, 40 over 4000 + up to 200, 27.0 and 28.5; no condition was found that leaves it out. (Pieces' bounds go
    // through an approximate quotient, which may give a piece a tile of its neighbour's.)
    int cuts = 0, own_from = 0;  // own_from: CTAs that have no singles
    float cut_tiles = 0.f;
    if (pairs > 0 && items <= ctas && cost < 16777216.f) {  // (sums of costs are exact)
      cuts = min(min((int)ceilf(__fdividef((float)(COST_PAIR * tiles), fmaxf(share - 0.5f * COST_PAIR_ITEM, 1.f))), tiles), (int)__fdividef((float)ctas + 0.5f, (float)items));
      cut_tiles = tiles == cuts ? 1.f : __fdividef((float)tiles, (float)cuts);  // (more than one by more than its error)
      const float piece = COST_PAIR * ceilf(cut_tiles) + COST_PAIR_ITEM, even = __fdividef(cost + (float)COST_PAIR_ITEM * items * (cuts - 1), (float)ctas);
      const int rest = min(ctas - cuts * items, max(singles - (singles + 15) / 16, min(singles, 1)));  // CTAs for singles alone: more than one each
      const float alone = singles > 0 ? (rest > 0 ? __fdividef(single_cost, (float)rest) : cost) : 0.f, limit = even + 0.5f * COST_PAIR_ITEM;
      if ((even - piece) * singles_per >= 4.f) {
        share = even;
      } else if (fmaxf(piece, alone) <= limit) {
        own_from = cuts * items;
        ctas = own_from + rest;
        share = alone;
      } else {
        cuts = 0;
      }
    }
    // lane 0: this CTA's bounds, lane 1: the next one's
    const int c = cta + (lane & 1);
    int a = 0, x, id = cta;
    float behind = share * c - pair_cost;  // of the cost, what is singles'
    if (cuts == 0) {
      a = c == ctas ? pairs : min(pairs, (int)ceilf(share * c * pairs_per));
    } else {
      auto start = [&](int cut) { return cut == cuts ? tiles : (int)(cut * cut_tiles); };  // first tile of a piece
      const int n = min(c, cuts * items), group = p.pairs * cuts, h = (int)__fdividef(n + 0.5f, (float)group), left = n - h * group;
      const int cut = (int)__fdividef(left + 0.5f, (float)p.pairs), pair = left - cut * p.pairs, item = h * p.pairs + pair, from = start(cut);
      // pairs of the CTAs in front; the piece itself, as units of its item (lane 1 has its end)
      const int before = (h * tiles + from) * p.pairs + (n < cuts * items ? pair * (start(cut + 1) - from) : 0);
      behind = own_from > 0 ? share * (c - own_from) : share * c - (float)COST_PAIR * before - (float)COST_PAIR_ITEM * n;
      id = item * cuts + cut;
      a = item * tiles + from;
      const int end = item * tiles + start(cut + 1), end0 = __shfl_sync(0xffffffffu, end, 0);
      if (lane & 1) a = end0;
      if (cta >= cuts * items) a = 0;
    }
    x = c == ctas ? singles : (behind <= 0.f ? 0 : min(singles, (int)ceilf(behind * singles_per)));
    const int a1 = __shfl_sync(0xffffffffu, a, 1), x1 = __shfl_sync(0xffffffffu, x, 1);
    if (lane == 0) {
      s->ctas = ctas;
      s->tiles = tiles;
      s->keys = keys;
      s->singles_prefix = odd;
      s->b_at[0] = s->b_at[1] = 0;  // (a stream that begins in front of the own keys begins them with the first sequence)
      s->cum_at[0] = s->cum_at[1] = 0;
      s->a0 = a;
      s->a1 = a1;
      s->pair_id = id;
      s->s[0] = x;
      s->s[1] = x + (x1 - x + 1) / 2;
      s->s[2] = x1;
    }
  }
  __syncthreads();
  if ((int)blockIdx.x < s->ctas && total_own > 0) {
    // the sequences in which the streams begin
    const int at0 = s->s[0] - s->singles_prefix, at1 = s->s[1] - s->singles_prefix;
    int c = cum;
    for (int b = b0; b < b1; ++b) {
      const int u = tiles_of(own_keys(p, b)), from = c * p.items_b, to = (c + u) * p.items_b;
      if (at0 >= from && at0 < to) s->b_at[0] = b, s->cum_at[0] = c;
      if (at1 >= from && at1 < to) s->b_at[1] = b, s->cum_at[1] = c;
      c += u;
    }
  }
}

template <int HD, typename T>
__global__ void __launch_bounds__(P_THREADS, 1) prefix_kernel(const __grid_constant__ PrefixParams p) {
  using SM = PrefixSmem<HD>;
  constexpr int STAGES = SM::kStages;
  static_assert(SM::kTotal <= 232448, "shared memory of an SM");
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t TMEM_S = 0, TMEM_O = 256;  // two tiles of 128 columns each; O of group q at 256 + 128 q
  after_previous();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  PrefixBars* bars = reinterpret_cast<PrefixBars*>(smem + SM::kBars);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &bars->abort_flag;

  // what has to be there before the roles begin, each by a warp of its own: the waits add up otherwise
  if (warp == W_K) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
    tc_fence_before();
  } else if (warp == W_ISSUE && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], 1);
      mbar_init(&bars->v_tail[s], 1);
    }
    for (int q = 0; q < 2; ++q) {
      mbar_init(&bars->seg_full[q][0], 1);
      mbar_init(&bars->seg_full[q][1], 1);
      mbar_init(&bars->s_full[q], 1);
      mbar_init(&bars->p_full[q], 4);
      mbar_init(&bars->o_final[q], 1);
      mbar_init(&bars->rec_full[q], 1);
      mbar_init(&bars->rec_empty[q], 2);
    }
    mbar_init(&bars->done, 1);
    mbar_fence_init();
  } else if (warp == W_V && lane == 0) {
    bars->abort_flag = *reinterpret_cast<volatile int*>(p.status);
    tma_prefetch_desc(&p.map_q);
    tma_prefetch_desc(&p.map_pq);
    if (p.prefix_keys > 0) {
      tma_prefetch_desc(&p.map_pk);
      tma_prefetch_desc(&p.map_pv);
    }
    if (p.own_keys > 0) {
      for (int i = 0; i < 2; ++i) {
        tma_prefetch_desc(&p.map_k[i]);
        tma_prefetch_desc(&p.map_v[i]);
      }
    }
  }
  make_plan(p, bars, reinterpret_cast<int2*>(smem + SM::kOut));
  __syncthreads();
  tc_fence_after();
  // no work for this CTA; shares of whole units may also come out empty
  if ((int)blockIdx.x >= bars->ctas || bars->a0 + bars->s[0] == bars->a1 + bars->s[2]) {
    if (warp == W_K) tmem_dealloc(bars->tmem_base, 512);
    return;
  }
  const uint32_t tmem = bars->tmem_base;
  const int n_pairs = bars->a1 - bars->a0, n_singles = bars->s[2] - bars->s[0], n_steps = n_pairs + n_singles;

  if (warp >= W_K) {
    // 384 x 168 registers at launch = 256 x 216 + 128 x 72. (With 72 the issuer's and the copy warps' code spills: at head size 128 116 bytes are
    // stored and 188 read back, at 64 52 and 708. What that costs has not been measured.)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == W_PLAN) {
      // =============================== planner ==================================================
      // (A warp that goes on together waits together: were some lanes to see the phase and others the abort, those that go on would wait
      // in their next vote or TMEM access for lanes that never come.)
      bool ok = !__any_sync(0xffffffffu, *abort_flag);
      const int q = lane & 1;  // (of the singles; batches begin with a single of the first stream once the pairs are through)
      int b = bars->b_at[q], cum = bars->cum_at[q];  // this stream's place among the own keys: sequence, tiles in front of it
      int m0 = 0;
      // A batch: steps m0 .. m0 + count - 1, pairs or singles, in lanes 0 .. count - 1.
      auto publish = [&](int batch) {
        const bool pair = m0 < n_pairs;
        const int count = min(BATCH, (pair ? n_pairs : n_steps) - m0), m = m0 + lane;
        StepRecord r;
        int item = 0, id = 0, keys_all = 0, tiles_all = 0, t = 0, left = 0;  // left: units of the item that are this CTA's from here on
        bool own = false, first = false;
        if (lane < count) {
          r.info = 0;
          if (pair) {
            const int pos = bars->a0 + m, tiles = bars->tiles;
            item = pos / tiles;
            t = pos - item * tiles;
            r.h = item / p.pairs;
            r.b = 2 * (item - r.h * p.pairs);
            id = bars->pair_id;
            r.row0 = (item + id) * (2 * PM);
            keys_all = bars->keys;
            tiles_all = tiles;
            left = min(tiles - t, bars->a1 - pos);
            first = m == 0;
          } else {
            const int pos = bars->s[q] + ((m - n_pairs) >> 1), end = bars->s[q + 1];
            const int y = pos - bars->singles_prefix;
            id = 2 * (int)blockIdx.x + q;
            own = y >= 0;
            if (!own) {
              tiles_all = bars->tiles;
              item = r.h = pos / tiles_all;
              t = pos - item * tiles_all;
              r.b = p.q_tiles - 1;
              r.row0 = (int)p.single_rows + (item + id) * PM;
              keys_all = bars->keys;
              item += p.Hkv * p.pairs;
            } else {
              // (The share was worked out from the lengths as they were. Were another stream to change them meanwhile, against the rules, the search
              // could pass the last sequence: it ends there, with a place that exists, and the call with a wait that expires.)
              int u;
              for (;;) {
                keys_all = own_keys(p, b);
                u = tiles_of(keys_all);
                if (y < (cum + u) * p.items_b || b + 1 >= p.B) break;
                cum += u;
                ++b;
              }
              const int per = max(u, 1), at = min(y - cum * p.items_b, per * p.items_b - 1), i = at / per;
              t = at - i * per;
              r.h = i / p.head_tiles;
              r.info = STEP_OWN | (uint32_t)(i - r.h * p.head_tiles) << 16;
              r.b = b;
              item = b * p.items_b + i;
              r.row0 = (int)p.own_rows + (item + id) * p.own_pitch;
              tiles_all = u;
              item += p.Hkv * (p.pairs + 1);
            }
            left = min(tiles_all - t, end - pos);
            first = m - n_pairs < 2;
          }
          first = first || t == 0;
          // which pieces of the item there are, for the merge; a CTA with a single unit has no second stream
          if (t == 0) p.plan_ws[2 * item] = id;
          if (t == tiles_all - 1) p.plan_ws[2 * item + 1] = id;
          r.gap = !pair && n_singles == 1 && t < tiles_all - 1 ? (own ? p.own_pitch : PM) : 0;
          const int keys = min(PN, keys_all - t * PN);
          r.n = left;
          r.keys = keys_all - t * PN;
          r.n0 = t * PN;
          r.info |= (first ? STEP_FIRST : 0u) | (left == 1 ? STEP_LAST : 0u) | ((uint32_t)keys << 8);
          const int* table = own ? p.page_table : p.prefix_table;
          if (table) {
            const int size = own ? p.page_size : p.prefix_page_size, box = min(size, PN), shift = 31 - __clz(size), pages = own ? p.num_pages : p.prefix_pages;
            if (own) table += (long long)b * p.max_pages;
#pragma unroll
            for (int i = 0; i < 4; ++i) r.page[i] = i * box < keys ? table[(r.n0 + i * box) >> shift] : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (r.page[i] < 0 || r.page[i] >= pages) {  // outside the pool: -1, for which TMA fills zeros
                r.page[i] = -1;
                report_status(p.status, 3);
              }
          }
        }
        // the streams' places for the next batch are those of their last lanes
        const int last = pair ? q : max((count - 1) - ((count - 1 - q) & 1), q);
        b = __shfl_sync(0xffffffffu, b, last);
        cum = __shfl_sync(0xffffffffu, cum, last);
        if (batch >= 2) ok = mbar_wait_uniform(&bars->rec_empty[batch & 1], ((batch >> 1) - 1) & 1, abort_flag);
        if (!ok) return;
        if (lane < count) bars->rec[(batch & 1) * BATCH + lane] = r;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->rec_full[batch & 1]);
        m0 += count;
      };
      if (ok) publish(0);
      if (ok && m0 < n_steps) publish(1);
      uint32_t n_tail = 0;  // parity of the tiles that were cleared, per place in the ring
      for (int batch = 0, n = 0; n < n_steps && ok; ++batch) {
        // Keys behind the end carry probability 0, but what lies in their V rows may be anything, and 0 * NaN is NaN: they are cleared here,
        // when the tile has come (by the warp that issues the MMAs that took 600 to 900 cycles in which nothing was issued).
        const int count = min(BATCH, (n < n_pairs ? n_pairs : n_steps) - n);
        for (int i = 0; i < count && ok; ++i, ++n) {
          const int r0 = (int)(bars->rec[(batch & 1) * BATCH + i].info >> 8) & 255, s = n % STAGES;
          if (r0 == PN) continue;
          ok = mbar_wait_uniform(&bars->v_tail[s], (n_tail >> s) & 1, abort_flag);
          if (!ok) break;
          n_tail ^= 1u << s;
          uint8_t* vt = smem + SM::kV + s * SM::kTile;
          constexpr int CPR = HD / 8;
          for (int k = lane; k < (PN - r0) * CPR; k += 32) {
            const int r = r0 + k / CPR, c = k % CPR;
            *reinterpret_cast<uint4*>(vt + (c >> 3) * (PN * 128) + sw128_offset(r, c & 7)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->v_full[s]);
        }
        if (ok && m0 < n_steps) publish(batch + 2);
      }
    } else if (warp == W_K || warp == W_V) {
      // =============================== requests of K and V ======================================
      // With the first key tile of a segment come the query rows, and word for the groups of what they are about to walk.
      if (lane == 0 && !*abort_flag) {
        const bool is_v = warp == W_V;
        uint64_t* const full = is_v ? bars->v_full : bars->k_full;
        uint64_t* const empty = is_v ? bars->v_empty : bars->k_empty;
        uint8_t* const ring = smem + (is_v ? SM::kV : SM::kK);
        const CUtensorMap* const own_map = is_v ? p.map_v : p.map_k;
        const CUtensorMap* const prefix_map = is_v ? &p.map_pv : &p.map_pk;
        const int own_shift = p.page_table ? min(31 - __clz(p.page_size | 1), 7) : 7;  // rows of a box, of a tile at most
        const int prefix_shift = p.prefix_table ? min(31 - __clz(p.prefix_page_size | 1), 7) : 7;
        const int q_bytes = p.q_box * (HD / 64), pq_bytes = p.pq_box * (HD / 64);
        bool ok = true;
        int n = 0;                                // tiles requested so far
        int n_seg[2] = {0, 0}, q_used[2] = {-1, -1};  // q_used: the last step whose scores read the group's rows
        auto wait_for_rows = [&](int q) {  // until the last scores with the group's rows are there
          if (q_used[q] >= 0) ok = ok && mbar_wait(&bars->k_empty[q_used[q] % STAGES], (q_used[q] / STAGES) & 1, abort_flag);
        };
        auto tell = [&](int q, const GroupSegment& x) {
          // (The scores of all that was told before are there. Those of the last segment were issued behind the product of the one
          // before it, and that behind the group's reading of this slot.)
          const int slot = n_seg[q]++ & 1;
          bars->seg[q][slot] = x;
          mbar_arrive(&bars->seg_full[q][slot]);
        };
        auto request_q = [&](int q, bool own, int shift, int head, int b, int h, uint64_t* bar) {
          uint8_t* dst = smem + SM::kQ + q * SM::kTile + shift * 128;
#pragma unroll
          for (int d = 0; d < HD; d += 64) tma_load_4d(dst + (d / 64) * (PM * 128), own ? &p.map_q : &p.map_pq, bar, d, head, b, h);
        };
        // Rows of a query tile that exist, and where they begin.
        auto rows_of = [&](bool own, int q_tile, int heads_from, int& head, int& b) {
          head = own ? heads_from : 0;
          b = own ? q_tile : q_tile * p.tile_seqs;
          if (own || p.G > PM) {
            if (!own) {
              b = q_tile / p.head_tiles;
              head = (q_tile - b * p.head_tiles) * PM;
            }
            return min(PM, p.G - head);
          }
          return min(p.tile_seqs, p.B - b) * p.G;
        };
        for (int batch = 0; n < n_steps && ok; ++batch) {
          const int count = min(BATCH, (n < n_pairs ? n_pairs : n_steps) - n);
          ok = mbar_wait(&bars->rec_full[batch & 1], (batch >> 1) & 1, abort_flag);
          if (!ok) break;
          for (int i = 0; i < count; ++i, ++n) {
            const int s = n % STAGES;
            if (n >= STAGES) ok = mbar_wait(&empty[s], (n / STAGES - 1) & 1, abort_flag);
            if (!ok) break;
            const StepRecord& r = bars->rec[(batch & 1) * BATCH + i];
            const uint32_t info = r.info;
            const int keys = (int)(info >> 8) & 255, h = r.h, n0 = r.n0, b = r.b;
            const bool own = info & STEP_OWN;
            const int shift = own ? own_shift : prefix_shift;
            // whole boxes, except at the end of a sequence's own keys: boxes of OWN_BOX rows
            const int unit = own ? OWN_BOX : 1 << shift;
            const uint32_t bytes = (uint32_t)((keys + unit - 1) & ~(unit - 1)) * (HD * 2);
            uint64_t* bar = &full[s];
            if (is_v) {
              bars->v_info[s] = info;
              if (keys < PN) bar = &bars->v_tail[s];
              mbar_arrive_expect_tx(bar, bytes);
            } else {
              const bool pair = n < n_pairs;
              const int q = pair ? 0 : (n - n_pairs) & 1;
              if (info & STEP_FIRST) {
                wait_for_rows(q);
                if (pair) wait_for_rows(1);
                if (!ok) break;
                mbar_arrive_expect_tx(&full[s], bytes + (own ? q_bytes : (pair ? 2 * pq_bytes : pq_bytes)));
                GroupSegment x;
                x.n = r.n;
                x.keys = r.keys;
                x.row0 = r.row0;
                x.gap = r.gap;
                // own rows sit in other lanes of the second group, so that the two groups' warps with rows are on different schedulers
                x.shift = own && p.item_rows <= 64 ? q * 64 : 0;
                int head, first_b;
                x.rows = rows_of(own, b, (int)(info >> 16) * PM, head, first_b);
                tell(q, x);
                request_q(q, own, x.shift, head, first_b, h, &full[s]);
                if (pair) {
                  x.rows = rows_of(false, b + 1, 0, head, first_b);
                  x.row0 += PM;
                  tell(1, x);
                  request_q(1, false, 0, head, first_b, h, &full[s]);
                }
              } else {
                mbar_arrive_expect_tx(&full[s], bytes);
              }
              if (pair || q == 0) q_used[0] = n;
              if (pair || q == 1) q_used[1] = n;
            }
            uint8_t* const dst = ring + s * SM::kTile;
            const bool paged = (own ? p.page_table : p.prefix_table) != nullptr;
            const int mask = (own ? p.page_size : p.prefix_page_size) - 1;
            for (int at = 0; at < keys;) {
              const bool whole = !own || keys - at > (1 << shift) - OWN_BOX;
              const int row = paged ? (n0 + at) & mask : n0 + at, last = paged ? r.page[at >> shift] : (own ? b : 0);
              const CUtensorMap* map = own ? (whole ? own_map : own_map + 1) : prefix_map;
#pragma unroll
              for (int d = 0; d < HD; d += 64) tma_load_4d(dst + (d / 64) * (PN * 128) + at * 128, map, bar, d, h, row, last);
              at += whole ? 1 << shift : OWN_BOX;
            }
          }
          if (ok) mbar_arrive(&bars->rec_empty[batch & 1]);
        }
        if (!is_v)
          for (int q = 0; q < 2 && ok; ++q) {
            GroupSegment none;
            none.n = 0;
            wait_for_rows(q);
            if (ok) tell(q, none);
          }
        // no copy is in flight when the CTA ends, whatever ended the loop
        for (int i = max(0, n - STAGES); i < n; ++i) wait_out(&full[i % STAGES], (i / STAGES) & 1);
      }
      __syncwarp();
    } else if (warp == W_ISSUE) {
      // =============================== MMA issuer ===============================================
      constexpr uint32_t idesc_s = umma_idesc_f16(PM, PN, IS_BF16, false, false);
      constexpr uint32_t idesc_o = umma_idesc_f16(PM, HD, IS_BF16, false, true);
      constexpr int KK_QK = HD / 16, KK_PV = PN / 16;
      const uint32_t lead = elect_one();
      const uint32_t dq = umma_desc_lo(smem_u32(smem + SM::kQ), 16), dk = umma_desc_lo(smem_u32(smem + SM::kK), 16);
      const uint32_t dv = umma_desc_lo(smem_u32(smem + SM::kV), PN * 128);
      bool ok = !*abort_flag;
      int nk = 0, nv = 0, n_p[2] = {0, 0};
      // The scores of group q with the next key tile; a pair's tile serves both groups before it is given back.
      auto issue_s = [&](int q, bool fetch, bool release) {
        const int s = nk % STAGES;
        if (fetch) ok = mbar_wait(&bars->k_full[s], (nk / STAGES) & 1, abort_flag);
        if (!ok) return;
        tc_fence_after();
        const uint32_t a = dq + ((q * SM::kTile) >> 4), b = dk + ((s * SM::kTile) >> 4);
#pragma unroll
        for (int kk = 0; kk < KK_QK; ++kk) {
          const uint32_t off = (kk >> 2) * (PN * 128) + (kk & 3) * 32;
          umma_ss_lead(lead, tmem + TMEM_S + q * 128, umma_desc_at(a, off), umma_desc_at(b, off), idesc_s, kk > 0);
        }
        umma_commit_lead(lead, &bars->s_full[q]);
        if (release) {
          umma_commit_lead(lead, &bars->k_empty[s]);
          ++nk;
        }
      };
      uint32_t info = 0;
      auto wait_v = [&]() {
        const int s = nv % STAGES;
        ok = mbar_wait(&bars->v_full[s], (nv / STAGES) & 1, abort_flag);
        if (!ok) return;
        info = *reinterpret_cast<volatile uint32_t*>(&bars->v_info[s]);
      };
      auto issue_pv = [&](int q) {
        ok = mbar_wait(&bars->p_full[q], n_p[q]++ & 1, abort_flag);
        if (!ok) return;
        tc_fence_after();
        const uint32_t b = dv + (((nv % STAGES) * SM::kTile) >> 4);
#pragma unroll
        for (int kk = 0; kk < KK_PV; ++kk)
          umma_ts_lead(lead, tmem + TMEM_O + q * 128, tmem + TMEM_S + q * 128 + kk * 8, umma_desc_at(b, kk * 2048), idesc_o,
                       (kk > 0 || !(info & STEP_FIRST)) ? 1u : 0u);
        if (info & STEP_LAST) umma_commit_lead(lead, &bars->o_final[q]);
      };
      auto release_v = [&]() {
        umma_commit_lead(lead, &bars->v_empty[nv % STAGES]);
        ++nv;
      };
      if (ok) {
        if (n_pairs > 0) {
          issue_s(0, true, false);
          if (ok) issue_s(1, false, true);
        } else {
          issue_s(0, true, true);
          if (ok && n_singles > 1) issue_s(1, true, true);
        }
      }
      for (int i = 0; i < n_pairs && ok; ++i) {
        wait_v();
        for (int q = 0; q < 2 && ok; ++q) {
          issue_pv(q);
          if (!ok) break;
          if (i + 1 < n_pairs)
            issue_s(q, q == 0, q == 1);
          else if (q < n_singles)
            issue_s(q, true, true);
        }
        if (ok) release_v();
      }
      for (int k = 0; k < n_singles && ok; ++k) {
        wait_v();
        if (ok) issue_pv(k & 1);
        if (!ok) break;
        release_v();
        if (k + 2 < n_singles) issue_s(k & 1, true, true);
      }
      umma_commit_lead(lead, &bars->done);
      wait_out(&bars->done, 0);
    }
  } else {
    // =============================== softmax groups =============================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int q = warp >> 2, wq = warp & 3;
    const uint32_t lane_addr = uint32_t(wq * 32) << 16;
    const uint32_t tS = tmem + lane_addr + TMEM_S + q * 128, tO = tmem + lane_addr + TMEM_O + q * 128;
    const float c = p.scale_log2;
    bool ok = !__any_sync(0xffffffffu, *abort_flag);  // (waits are the warp's: see the planner)
    int n_s = 0, n_seg = 0;
    while (ok) {
      ok = mbar_wait_uniform(&bars->seg_full[q][n_seg & 1], (n_seg >> 1) & 1, abort_flag);
      if (!ok) break;
      const GroupSegment g = bars->seg[q][n_seg & 1];
      if (g.n == 0) break;
      const int row = ((wq * 32 - g.shift) & 127) + lane;  // of the query tile
      const bool live = row < g.rows;
      const bool idle = row - lane >= g.rows;              // no row of this warp exists: what it leaves in P is never read out
      float m_ref = -INFINITY;  // what the exponentials are relative to; it moves when the maximum has grown by 2^8
      float l = 0.f;            // their sum
      for (int t = 0; t < g.n; ++t) {
        ok = mbar_wait_uniform(&bars->s_full[q], n_s++ & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (!idle) {
          uint32_t sr[PN];
#pragma unroll
          for (int ch = 0; ch < PN / 32; ++ch) tmem_ld32(tS + ch * 32, &sr[ch * 32]);
          tmem_ld_wait();
          const int n_live = g.keys - t * PN;
          if (n_live < PN) {
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
          const bool need = live && !none && !((m_cand - m_ref) * c <= 8.0f);  // (rows that do not exist hold what lay there)
          float scale = 1.0f;
          if (need) {
            scale = ex2_approx((m_ref - m_cand) * c);
            m_ref = m_cand;
            l *= scale;
          }
          // (this tile's scores were issued behind the P V product before them, so O is at rest)
          if (t > 0 && __any_sync(0xffffffffu, need)) {
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
      ok = mbar_wait_uniform(&bars->o_final[q], n_seg++ & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      if (!idle) {
        // as it is: the merge divides by the sum of all pieces
        const long long at = (long long)g.row0 + row;
        if (live) {
          p.ml_partial[at] = make_float2(l == 0.f ? -INFINITY : m_ref * c, l);
          if (g.gap) p.ml_partial[at + g.gap] = make_float2(-INFINITY, 0.f);
        }
        float* const mine = p.out_partial + at * p.D;  // this lane's row
        if (g.rows <= DIRECT_ROWS) {  // a group's few heads: each lane writes its row
          uint32_t o[HD];
#pragma unroll
          for (int ch = 0; ch < HD / 32; ++ch) tmem_ld32(tO + ch * 32, &o[ch * 32]);
          tmem_ld_wait();
          if (live) {
#pragma unroll
            for (int i = 0; i < HD; i += 4)
              if (i < p.D) *reinterpret_cast<uint4*>(mine + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        } else {
          // 32 columns at a time through shared memory and TMA; the rows of the warp that do not exist belong to the piece, too. (Written by the lanes,
          // the rows went through L1 three times.) The loop stays rolled: a CTA comes here once or twice, and its instructions have to arrive.
          uint8_t* stage = smem + SM::kOut + warp * 4096;
#pragma unroll 1
          for (int c0 = 0; c0 < p.D; c0 += 32) {
            uint32_t o[32];
            tmem_ld32(tO + c0, o);
            tmem_ld_wait();
            if (lane == 0) bulk_wait_read0();
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&p.map_o, stage, c0, g.row0 + row, 0);
              bulk_commit();
            }
          }
        }
      }
      tc_fence_before();
    }
    if (lane == 0) bulk_wait0();
  }

  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) report_status(p.status, *abort_flag);  // the reason it was launched with, or 1
  if (warp == W_K) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// WPR warps join the partial results of a (sequence, query head): the pieces of its item over the prefix and of its own keys' item, from
// the first to the last that the kernel in front noted. A piece has its
// reference maximum m, its sum l and its O, so o = sum 2^(m - max) O / sum 2^(m - max) l. 32 pieces a warp at a time, four rows under way.
template <typename T, int VEC, int WPR>
__global__ void __launch_bounds__(256) prefix_merge_kernel(const PrefixParams p) {
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % WPR;
  const int spare = blockIdx.x * (8 / WPR) + warp / WPR, at = min(spare, p.B * p.Hq - 1);  // (spare warps: the last row again)
  const int b = at / p.Hq, head = at - b * p.Hq, h = head / p.G, gi = head - h * p.G, gt = gi / PM;
  // pieces first .. last of the two items: all that is needed to find them is asked for at once
  const int q_tile = p.G > PM ? b * p.head_tiles + gt : b / p.tile_seqs, r = p.G > PM ? gi - gt * PM : (b - q_tile * p.tile_seqs) * p.G + gi;
  const bool pair = q_tile < 2 * p.pairs;
  const int pre = pair ? h * p.pairs + q_tile / 2 : h, own = b * p.items_b + h * p.head_tiles + gt;
  const int2 pre_at = p.prefix_keys > 0 ? __ldcg(reinterpret_cast<const int2*>(p.plan_ws) + (pair ? pre : pre + p.Hkv * p.pairs)) : make_int2(0, -1);
  const int2 own_at = p.own_keys > 0 ? __ldcg(reinterpret_cast<const int2*>(p.plan_ws) + own + p.Hkv * (p.pairs + 1)) : make_int2(0, -1);
  const bool skip = *reinterpret_cast<volatile int*>(p.status) != 0;
  // Numbers of pieces that there can be, and no others: where the kernel in front left because of the status word, what it has not noted is
  // whatever lay there, and the word may have been cleared since.
  auto pieces = [](int2 at, int limit) { return at.x >= 0 && at.y < limit ? max(at.y - at.x + 1, 0) : 0; };
  const int n_pre = min(p.prefix_used ? *p.prefix_used : p.prefix_keys, p.prefix_keys) > 0 ? pieces(pre_at, pair ? p.ctas : 2 * p.ctas) : 0;
  const int n_own = own_keys(p, b) > 0 ? pieces(own_at, 2 * p.ctas) : 0;
  if (WPR == 1 && skip) return;
  const int pre_pitch = pair ? 2 * PM : PM, pre_row = (pair ? 0 : (int)p.single_rows) + (pre + pre_at.x) * pre_pitch + r + (pair ? (q_tile & 1) * PM : 0);
  const int own_row = (int)p.own_rows + (own + own_at.x) * p.own_pitch + gi - gt * PM;
  const int count = skip ? 0 : n_pre + n_own;
  float top = -INFINITY, sum = 0.f, acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  const int d0 = lane * VEC;
  const bool active = d0 < p.D;
  using Row = typename std::conditional<VEC == 4, float4, float2>::type;
  // this warp's pieces: part, part + WPR, ...
  for (int s0 = 0; s0 < count; s0 += 32 * WPR) {
    const int i = s0 + lane * WPR + part, cnt = min(32, (count - s0 - part + WPR - 1) / WPR);
    const int mine = i < n_pre ? pre_row + i * pre_pitch : own_row + (i - n_pre) * p.own_pitch;
    const float2 ml = i < count ? __ldcg(p.ml_partial + mine) : make_float2(-INFINITY, 0.f);
    Row v[4];
    auto load4 = [&](int first) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = __shfl_sync(0xffffffffu, mine, (first + j) & 31);
        if (first + j < cnt && active) v[j] = __ldcg(reinterpret_cast<const Row*>(p.out_partial + (long long)row * p.D + d0));
      }
    };
    load4(0);
    float m = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = fmaxf(m, top);
    const float old = top == -INFINITY ? 0.f : exp2f(top - m), w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
    float ws = w * ml.y;  // (NaN among a piece's scores: its sum is NaN, and so is the row)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
    sum = sum * old + ws;
    top = m;
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] *= old;
    for (int first = 0; first < cnt; first += 4) {
      if (first > 0) load4(first);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float wj = __shfl_sync(0xffffffffu, w, (first + j) & 31);
        if (first + j >= cnt || wj == 0.f) continue;  // a piece without weight adds nothing, whatever its row holds
        const float* e = reinterpret_cast<const float*>(&v[j]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += wj * e[k];
      }
    }
  }
  if constexpr (WPR > 1) {  // the warps' sums, relative to the row's maximum
    __shared__ float parts[8][32 * VEC + 2];
    if (lane == 0) {
      parts[warp][32 * VEC] = top;
      parts[warp][32 * VEC + 1] = sum;
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) parts[warp][k * 32 + lane] = acc[k];
    __syncthreads();
    if (part != 0 || skip) return;
    float m = top, total = 0.f;
#pragma unroll
    for (int w = 1; w < WPR; ++w) m = fmaxf(m, parts[warp + w][32 * VEC]);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) {
      const float tw = parts[warp + w][32 * VEC];
      const float f = tw == -INFINITY ? 0.f : exp2f(tw - m);  // (without weight, but its sum may be a NaN: 0 * NaN is one)
      total += parts[warp + w][32 * VEC + 1] * f;
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += parts[warp + w][k * 32 + lane] * f;
    }
    top = m;
    sum = total;
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
  if (p.ctas > 0)  // otherwise there is no place for a key
    if (cudaError_t e = launch_early(kern, (unsigned)p.ctas, P_THREADS, smem, stream, 1, p); e != cudaSuccess) return e;
  // Few rows have many pieces: four warps a row where that still is one wave of blocks (6 sequences x 64 heads, 37 pieces, from a cold
  // L2: 14.5 us, so 8.2; 64 x 32 heads, 8 pieces: the whole call 49.8 us, so 55.7).
  const long long rows = (long long)p.B * p.Hq;
  if (rows <= 2ll * 4 * device_sm_count()) return launch_early(prefix_merge_kernel<T, HD / 32, 4>, (unsigned)((rows + 1) / 2), 256, 0, stream, 1, p);
  return launch_early(prefix_merge_kernel<T, HD / 32, 1>, (unsigned)((rows + 7) / 8), 256, 0, stream, 1, p);
}

}  // namespace

// Shares of the work: one CTA an SM, and no more than there can be units.
bool prefix_shape(PrefixParams* p) {
  p->head_tiles = (p->G + PM - 1) / PM;
  p->tile_seqs = p->G <= PM ? PM / p->G : 1;
  p->q_tiles = p->G <= PM ? (p->B + p->tile_seqs - 1) / p->tile_seqs : p->B * p->head_tiles;
  p->pairs = p->q_tiles / 2;
  p->items_b = p->Hkv * p->head_tiles;
  p->item_rows = p->G < PM ? p->G : PM;
  p->own_pitch = p->item_rows <= DIRECT_ROWS ? p->item_rows : (p->item_rows + 31) & ~31;
  p->q_box = 64 * p->item_rows * 2;
  p->pq_box = p->q_box * p->tile_seqs;
  auto tiles = [](long long keys) { return (keys + PN - 1) / PN; };
  const long long units = (long long)p->Hkv * (p->pairs + (p->q_tiles & 1)) * tiles(p->prefix_keys) + (long long)p->B * p->items_b * tiles(p->own_keys);
  if (units >= (1ll << 30)) return false;  // units are counted in 32 bits
  const int sms = device_sm_count();
  p->ctas = units < sms ? (int)units : sms;
  p->single_rows = p->prefix_keys > 0 ? ((long long)p->Hkv * p->pairs + p->ctas) * (2 * PM) : 0;
  if (p->pairs == 0) p->single_rows = 0;
  p->own_rows = p->single_rows + ((p->q_tiles & 1) && p->prefix_keys > 0 ? ((long long)p->Hkv + 2 * p->ctas) * PM : 0);
  p->partial_rows = p->own_rows + (p->own_keys > 0 ? ((long long)p->B * p->items_b + 2 * p->ctas) * p->own_pitch : 0);
  if (p->partial_rows >= (1ll << 31)) return false;
  p->plan_ints = 2 * ((long long)p->Hkv * (p->pairs + 1) + (long long)p->B * p->items_b);
  return true;
}

cudaError_t launch_prefix(const PrefixParams& p, int dtype, int head_dim, cudaStream_t stream) {
  if (head_dim == 64) return dtype == DT_BF16 ? launch_one<64, __nv_bfloat16>(p, stream) : launch_one<64, __half>(p, stream);
  return dtype == DT_BF16 ? launch_one<128, __nv_bfloat16>(p, stream) : launch_one<128, __half>(p, stream);
}

}  // namespace fsa
