// row_attention.cu -- attention of many query rows against a shared run of keys: whole prompts (packed rows,
// causal) and batches whose sequences share their first cache pages.
//
//   o[r] = sum_j softmax_j(scale q[r] . k[j]) v[j],   j < limit[r]
//
// A *unit* is up to 256 query rows of one KV head -- two row tiles of 128, which are TMEM lanes -- against a run of
// keys.  The query heads of a KV head are rows of their own (row = token * n_rep + head), so a tile holds
// 128 / n_rep tokens whose causal limits lie close together, and a decode step's few rows share a tile.  In a
// shared prefix the tokens of all member sequences are the rows of one part; every sequence's own keys are a part of
// their own with its rows only, and the results of both are joined.
//
// Work: parts (prefix groups, then sequences) are cut into units, a unit costs its 128-key blocks plus kUnitCost,
// and the concatenated costs are cut into equal ranges, one a CTA (make_plan, worked out by every CTA for itself).  A
// unit that a boundary cuts becomes several items, whose unnormalised rows, maxima and sums go to the workspace and are
// joined by a second kernel; the others are written to the output at once.
//
// One CTA an SM, 12 warps (E4M3 16), each role walking the same items:
//   warp 0          K/V tiles by TMA into a ring (K 0, V 0, K 1, V 1): packed rows as {64 dims, 128 rows} boxes,
//                   pages as four-row gathers; both give [dim half][128 keys][128 B] in the 128-byte swizzle
//   warps 1, 2      MMA issue (one lane), one for each row tile
//   warp 3          query rows of the next item, as boxes of n_rep heads x 128 / n_rep tokens (or one token, where a
//                   group's rows do not follow one another)
//   warps 4-7, 8-11 softmax and epilogue of row tile 0, 1: a thread owns a row, so maxima and sums need no exchange;
//                   and the washing of V (below)
//   warps 12-15     (E4M3 V) the block's codes to f16 by moving bits; the keys' scales are multiplied into P
// A block of 128 keys is two halves of 64, each with scores S_t[h] of its own in TMEM:
//   S_t[h] = Q_t K^T  ->  P = 2^((S - m) scale) as bf16 (E4M3 f16) over the same columns  ->  O_t += P V (A operand from TMEM)
// Half h + 1's products and half h's softmax run at the same time, and so do the two tiles.
//
// The running maximum is a stale one: m is a row's maximum over its first half block and moves only when a half block's
// sum passes 2^30 (2^x has the range for it), so that O is almost never rescaled.  P is rounded to bf16 (2^-8 of each weight
// at most, independent between keys); sums, maxima, O and the joined rows stay fp32.
// A quarter of the exponentials are a cubic on the FMA units (relative error 1.0e-4), the rest the exponential unit's: 64 a
// thread and half would take 544 clocks a warp there.
//
// E4M3: what is rounded is P times its key's scale, to f16 (2^-11), as paged_attention does it.  f16 has not bf16's
// range: scales count in units of a power of two that puts the geometric mean of an item's first 32 keys (those that
// all its rows see) between 2^2 and 2^3, O is multiplied by that unit at the end, and m also moves where a half block's
// sum times the largest scale that the row sees passes 2^15, so that no weight reaches f16's end.  A weight below 2^-14
// is off by up to 2^-25: its bits are missed only where the keys that carry a row have scales some 2^15 below that mean,
// or 2^25 below another key's that the row sees.
//
// What a masked key's zero probability meets in V must be finite.  The MMAs take none of the 16-key steps past an item's
// last key, and what is left of the keys that some row does not see is washed in shared memory: an infinity or a NaN
// becomes zero and its key is noted, and a row that does see it gets it added after the epilogue.  So an infinity or a NaN
// of a key that a row sees leaves the row's value not finite, whatever the key weighs: where the weight underflows to zero it
// is 0 times an infinity (NaN) or the added infinity, by where the key lies.
//
// Bound: the softmax warps.  A half block of both tiles takes about 1900 clocks, of which the tensor cores are busy for
// 1290 (ncu: 53 % of the cycles; exponential unit 39 %; issue slots 42 %; DRAM 2 %): 1200 are exponentials, the rest
// the way of the scores from TMEM and of P back.  Four prompts of 8192 tokens (12 heads over 2, 128 dims) take 820 to
// 870 us, 950 to 1000 TFLOP/s (of 1632 measured); 16 of 1024 tokens 99 to 105 us (500); 64 x 5 rows over a shared
// 8192-token prefix and 1024 tokens each 48 to 54 us against 78 us by paged_attention, which reads the prefix for every sequence.
// What small calls cost: the plan 5 us (its code is fetched and run once; later layers reuse it), an item's start and
// end 2 to 3 us (first block, epilogue), the join 3 us and up.
#include <initializer_list>
#include <type_traits>

#include "sd_common.cuh"
#include "sd_internal.h"
#include "umma.cuh"

namespace sd {

constexpr int kRowTile = 128;      // rows of a tile: TMEM lanes
constexpr int kUnitRows = 256;     // two tiles
constexpr int kKeyBlock = 128;     // keys of a block
constexpr int kUnitCost = 2;       // what a unit costs beside its blocks (query load, epilogue), in blocks
constexpr int kMinQuota = 3;       // smallest range of a CTA, in blocks: 9, 6, 4 and 3 take 24.6, 20.3, 20.1 and 19.4 us for 4 decode steps
constexpr int kMergeParts = 8;     // blocks of the cut-unit merge for each CTA of the grid
constexpr float kGrow = 1073741824.f;  // 2^30: a half block's sum past it moves the row's reference
constexpr float kGrowF16 = 32768.f;    // 2^15: the same of the sum times the block's largest scale (E4M3)
constexpr int kScaleMean = 2;          // E4M3: the mean scale of an item's first keys is counted as 2^2 .. 2^3
constexpr float kLargeScore = 4096.f;  // in units of log2
constexpr float kNoPart = -1.f;        // sum of a partial row that was not computed
constexpr float kExpC1 = 0.693282962f, kExpC2 = 0.242210999f, kExpC3 = 0.0550089143f;

enum RowSource { kPacked = 0, kPaged = 1, kPagedE4M3 = 2 };
constexpr int kLoadWarp = 0, kIssueWarp = 1, kQueryWarp = 3, kSoftmaxWarp = 4, kWidenWarp = 12;
constexpr int kSoftmaxWarps = 8;  // four a row tile
// Threads, and registers a thread of the softmax warps and of the others: the launch's own are what
// __launch_bounds__ leaves (168, E4M3 128), and the shares add up to them.
template <int SRC>
struct RowRoles {
  static constexpr bool V8 = SRC == kPagedE4M3;
  static constexpr int THREADS = 32 * (kSoftmaxWarps + 4 + (V8 ? 4 : 0));
  static constexpr int ITEMS = V8 ? 4 : 12;  // items of a CTA that it keeps in shared memory (E4M3 has less room)
  static constexpr int SOFTMAX_REGS = V8 ? 176 : 208, OTHER_REGS = V8 ? 80 : 88;
  static_assert(32 * kSoftmaxWarps * SOFTMAX_REGS + (THREADS - 32 * kSoftmaxWarps) * OTHER_REGS <= THREADS * (V8 ? 128 : 168),
                "register shares");
};

struct alignas(16) RowItem {
  int32_t src;     // sequence, or ~group
  int32_t vt0;     // first token of the unit, in the part
  int32_t n_vt;    // tokens of the part
  int32_t head;    // KV head
  int32_t k0, k1;  // keys of this item
  int32_t slot;    // first workspace row of the partial, or -1: the output itself
  int32_t nblk;    // blocks (0: nothing to do)
  int32_t row0;    // query row of token 0 (group: -1 where its members' rows do not follow one another)
  int32_t first;   // sequence: keys before its first new token; group: not 0 if every member has q_max tokens
  int32_t kv;      // packed: first key row; paged: sequence whose page table is read
  int32_t member0; // group: first member
};
static_assert(sizeof(RowItem) == 48, "three 16-byte loads");

// What the join needs of a unit that a CTA boundary cuts / of a sequence, in as few loads as can be.
struct alignas(16) CutUnit {
  int32_t slot, pieces;             // pieces 0: none is cut here
  int32_t row0, vt0, n_vt, head, pad[2];
};
struct alignas(16) SeqRows {
  int32_t row0, len;                // first query row, valid tokens
  int32_t own, pre;                 // first unit of its own part and of its group's (-1: no group, or no prefix)
  int32_t vt, pad[3];               // its first token in the group's part
};

struct RowParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  int64_t q_st, q_sh, o_st, o_sh;
  const int32_t *q_row0, *q_len, *ctx_len, *kv_row0;
  const int32_t *group_start, *members, *prefix_len;
  const int32_t* page_table;
  const float* v_scale;
  const uint8_t* v_pool;         // paged: V blocks; packed: V rows, strides in elements
  int64_t v_st, v_sh;
  int64_t q_rows, kv_rows;
  int32_t B, H, KV, n_rep, tpt, q_max, G, M;
  int32_t num_pages, max_pages, paged;
  int32_t plan;                 // 1: work the plan out, 0: it is in the workspace
  int32_t grid, min_quota, compact;  // CTAs of the plan, its smallest range; compact: slots only for cut units
  int32_t cap_seq, cap_group;   // workspace rows of a sequence's / a group's slot
  int32_t group_rows;           // workspace rows before the sequences' slots
  float scale_log2;
  uint64_t key;                 // of this launch shape
  uint64_t wait_ns;             // limit of a wait; 0: the softmax warps give up without looking
  int32_t* status;
  // workspace
  int32_t *cta_first, *cta_last;                // [grid]
  CutUnit* cut_unit;                            // [grid]
  uint64_t* plan_key;                           // the launch shape that the plan is for
  SeqRows* seq_rows;                            // [B]
  int2* member_row;                             // [M] {first query row, tokens}
  int2* unit_info;                              // [units] {first slot row, pieces}
  RowItem* items;                               // [units + grid]
  float2* part_ml;                              // [slot rows] {max (log2), sum}
  float4* part_o;                               // [slot rows / 32][D / 4][32]: a warp stores 32 rows' four columns at once
};

// ---------------------------------------------------------------- plan
// Every CTA of the attention kernel works the plan out for itself before it starts, in the shared memory that its
// blocks will take, and keeps its own items (they are written down, too: the workspace then serves the next layers,
// and the join).  That is a round trip to L2, some barriers and two scans, 3 to 6 us; a kernel of its own before this one
// took 5 to 10.  A thread a sequence, member or unit row.
constexpr int kPlanMost = 2048;  // sequences, members or groups of a call
struct PlanSpace {
  int32_t *rows, *len, *first, *group, *vt, *listed, *prefix, *table, *flags;
  __host__ __device__ static constexpr size_t bytes(int B, int G) {
    return sizeof(int32_t) * (static_cast<size_t>(G) + B + 1 + 5 * static_cast<size_t>(B) + 3 * static_cast<size_t>(G));
  }
  SD_DEV PlanSpace(uint8_t* at, int B, int G) {
    rows = reinterpret_cast<int32_t*>(at);  // [G + B + 1] first unit row of a part
    len = rows + G + B + 1;                 // [B] valid new tokens
    first = len + B;                        // keys before them
    group = first + B;
    vt = group + B;                         // first token in its group's part
    listed = vt + B;                        // where a sequence is listed first
    prefix = listed + B;                    // [G]
    table = prefix + G;                     // first member with rows
    flags = table + G;                      // kGroupRows, kGroupFull
  }
};
constexpr int kGroupRows = 1;  // the members' rows follow one another: token vt is row (first member's row) + vt
constexpr int kGroupFull = 2;  // and every token is one: no member has fewer than q_max
struct PartInfo {
  int n_vt, k0, first;  // tokens; keys k0 .. first + i (a sequence's token i) or k0 .. first - 1
  bool group;
};
// (A group's members count q_max tokens each, whether or not they have so many: token vt is row vt % q_max of member
// vt / q_max, with nothing to look up.)
SD_DEV PartInfo part_info(const RowParams& p, const PlanSpace& w, int part) {
  PartInfo f;
  f.group = part < p.G;
  if (f.group) {
    f.k0 = 0;
    f.first = w.prefix[part];  // 0 where the group is empty or its start bad
    f.n_vt = f.first > 0 ? (p.group_start[part + 1] - p.group_start[part]) * p.q_max : 0;
  } else {
    const int b = part - p.G;
    f.n_vt = w.len[b];
    f.first = w.first[b];
    const int g = f.n_vt > 0 ? w.group[b] : -1;
    f.k0 = g >= 0 ? w.prefix[g] : 0;
  }
  return f;
}
// last key + 1 of the part's unit row r (all KV heads alike)
SD_DEV int unit_end(const RowParams& p, const PartInfo& f, int r) {
  return f.group ? f.first : f.first + min((r + 1) * 2 * p.tpt, f.n_vt);
}
SD_DEV int unit_blocks(const RowParams& p, const PartInfo& f, int r) {
  return (unit_end(p, f, r) - f.k0 + kKeyBlock - 1) / kKeyBlock;
}
// Sum of v over the threads before this one, and over all.  `tot`: two sets of [32], used in turn.
SD_DEV int64_t plan_scan(int64_t v, int64_t& all, int64_t (*tot)[32], int& turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) tot[turn][warp] = x;
  __syncthreads();
  int64_t before = 0;
  all = 0;
  for (int i = 0; i < warps; ++i) {
    const int64_t t = tot[turn][i];
    if (i < warp) before += t;
    all += t;
  }
  turn ^= 1;
  return before + x - v;
}

// All threads of the CTA; `at`: PlanSpace::bytes() of shared memory.  range[0 .. 1] (shared): numbers of this CTA's first
// and last item; kept[i % ITEMS] holds them where that is all of them (returns whether).
template <int ITEMS>
SD_DEV bool make_plan(const RowParams& p, uint8_t* at, int64_t (*tot)[32], int* range, RowItem* kept) {
  const PlanSpace w(at, p.B, p.G);
  const int tid = threadIdx.x, nthr = blockDim.x;
  const bool writes = blockIdx.x == 0;  // what the join and later calls read of the whole batch
  int turn = 0;
  if (tid < 2) range[tid] = -tid;  // 0, -1: no items
  if (tid == 2) p.cut_unit[blockIdx.x].pieces = 0;
  if (tid == 3 && writes) *p.plan_key = p.key;
  // the first loads of everything, under way together
  const int member = tid < p.M ? p.members[tid] : 0;
  int start = 0, stop = 0, share = 0;
  if (tid < p.G) {
    start = p.group_start[tid];
    stop = p.group_start[tid + 1];
    share = p.prefix_len[tid];
  }
  for (int b = tid; b < p.B; b += nthr) {
    const int n = p.q_len[b], c = p.ctx_len[b], r0 = p.q_row0[b], k0 = p.paged ? 0 : p.kv_row0[b];
    int bad = 0;
    if (n < 0 || n > p.q_max || (n > 0 && (c < n || r0 < 0 || static_cast<int64_t>(r0) + n > p.q_rows)))
      bad = SPECDEC_STATUS_BAD_LENGTH;
    else if (n > 0 && p.paged && c > static_cast<int64_t>(p.max_pages) * kPage)
      bad = SPECDEC_STATUS_PAGE_OVERFLOW;
    else if (n > 0 && !p.paged && (k0 < 0 || static_cast<int64_t>(k0) + c > p.kv_rows))
      bad = SPECDEC_STATUS_BAD_LENGTH;
    if (bad && writes) raise_status(p.status, bad);
    const int v = bad ? 0 : n;
    w.len[b] = v;
    w.first[b] = v > 0 ? c - v : 0;
    w.group[b] = -1;
    w.listed[b] = 0x7fffffff;
  }
  if (p.G > 0) {
    int bad = 0;
    for (int g = tid; g < p.G; g += nthr) {
      if (g != tid) start = p.group_start[g], stop = p.group_start[g + 1], share = p.prefix_len[g];
      bad |= start < 0 || stop < start || stop > p.M;
      if (share < 0 && writes) raise_status(p.status, SPECDEC_STATUS_BAD_GROUP);
      w.prefix[g] = max(share, 0);
      w.table[g] = 0x7fffffff;
      w.flags[g] = kGroupRows | kGroupFull;
    }
    // starts that do not ascend within the member list: nobody is in a group, everything is attended to alone
    bad = __syncthreads_or(bad);
    if (bad && tid == 0 && writes) raise_status(p.status, SPECDEC_STATUS_BAD_GROUP);
    const int M = bad ? 0 : p.M;
    for (int i = tid; i < M; i += nthr) {
      const int b = i == tid ? member : p.members[i];
      if (b >= 0 && b < p.B) atomicMin(&w.listed[b], i);  // a sequence listed twice counts where it is listed first
    }
    __syncthreads();
    for (int i = tid; i < M; i += nthr) {
      const int b = i == tid ? member : p.members[i];
      int lo = 0, hi = p.G;  // the last group that starts at or before i, and holds it
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.group_start[mid] <= i) lo = mid; else hi = mid;
      }
      const int gs = p.group_start[lo], ge = p.group_start[lo + 1];
      int2 mr = make_int2(0, 0);
      if (b < 0 || b >= p.B || w.listed[b] != i) {
        if (writes) raise_status(p.status, SPECDEC_STATUS_BAD_GROUP);
        if (i >= gs && i < ge) atomicAnd(&w.flags[lo], 0);
      } else if (i >= gs && i < ge) {
        const int n = w.len[b], lead = p.members[gs];
        w.group[b] = lo;
        w.vt[b] = (i - gs) * p.q_max;
        mr = make_int2(p.q_row0[b], n);
        const bool follows = lead >= 0 && lead < p.B && mr.x >= 0 && mr.x == p.q_row0[lead] + (i - gs) * p.q_max;
        const int keep = (follows ? kGroupRows : 0) | (n == p.q_max ? kGroupFull : 0);
        if (keep != (kGroupRows | kGroupFull)) atomicAnd(&w.flags[lo], keep);
        if (n > 0) {
          atomicMin(&w.prefix[lo], w.first[b]);  // keys that all of the group's rows see
          atomicMin(&w.table[lo], i);
        }
      }
      p.member_row[i] = mr;  // (by every CTA, the same: each reads it from here on)
    }
    __syncthreads();
    for (int g = tid; g < p.G; g += nthr) {
      const int i = w.table[g];
      const int n = i == 0x7fffffff ? 0 : w.prefix[g] / kPage * kPage;  // whole pages
      w.prefix[g] = n;
      w.table[g] = i == 0x7fffffff ? 0 : p.members[i];
    }
  }
  __syncthreads();
  // first unit row of every part
  const int parts = p.G + p.B;
  int rows = 0;
  for (int base = 0; base < parts; base += nthr) {
    const int part = base + tid;
    int n = 0;
    if (part < parts) n = (part_info(p, w, part).n_vt + 2 * p.tpt - 1) / (2 * p.tpt);
    int64_t all;
    const int at_row = rows + static_cast<int>(plan_scan(n, all, tot, turn));
    if (part < parts) w.rows[part] = at_row;
    rows += static_cast<int>(all);
  }
  if (tid == 0) w.rows[parts] = rows;
  __syncthreads();
  if (writes)
    for (int b = tid; b < p.B; b += nthr) {
      const int g = w.group[b];
      SeqRows r = {};
      r.row0 = p.q_row0[b];
      r.len = w.len[b];
      r.own = w.rows[p.G + b] * p.KV;
      r.pre = g >= 0 && w.prefix[g] > 0 ? w.rows[g] * p.KV : -1;
      r.vt = g >= 0 ? w.vt[b] : 0;
      p.seq_rows[b] = r;
    }
  auto part_of = [&](int row) {  // the last part that starts at or before the row and has rows
    int lo = 0, hi = parts;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (w.rows[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
  };
  // a unit row's cost (one KV head's unit); rows beyond the threads are counted first, for the total
  int64_t total = 0, all;
  if (rows > nthr) {
    int64_t sum = 0;
    for (int row = tid; row < rows; row += nthr) {
      const int part = part_of(row);
      sum += unit_blocks(p, part_info(p, w, part), row - w.rows[part]) + kUnitCost;
    }
    (void)plan_scan(sum * p.KV, total, tot, turn);
    __syncthreads();
  }
  int64_t run = 0, quota = 0, from = 0, to = 0;
  bool direct_items = false;
  for (int base = 0; base < rows; base += nthr) {
    const int row = base + tid;
    int part = 0, r = 0, nb = 0, cost = 0;
    PartInfo f = {};
    if (row < rows) {
      part = part_of(row);
      r = row - w.rows[part];
      f = part_info(p, w, part);
      nb = unit_blocks(p, f, r);
      cost = nb + kUnitCost;
    }
    const int64_t us0 = run + plan_scan(static_cast<int64_t>(cost) * p.KV, all, tot, turn);
    run += all;
    if (base == 0) {
      if (rows <= nthr) total = all;
      if (total >= 0x7fffffff) {  // 2^31 blocks are half a minute of this device's tensor cores
        if (writes && tid == 0) {
          raise_status(p.status, SPECDEC_STATUS_BAD_LENGTH);
          *p.plan_key = ~p.key;  // nothing to join, and nothing to use again
        }
        total = 0;
      }
      quota = max(static_cast<int>((static_cast<uint32_t>(total) + p.grid - 1) / p.grid), p.min_quota);
      from = blockIdx.x * quota;
      to = min(from + quota, total);
      direct_items = quota <= (1 + kUnitCost) * (ITEMS - 2);
    }
    if (row >= rows || total == 0 || us0 >= to || us0 + static_cast<int64_t>(cost) * p.KV <= from) continue;
    auto cta_of = [&](int64_t x) { return static_cast<int>(static_cast<uint32_t>(x) / static_cast<uint32_t>(quota)); };
    const int c = blockIdx.x, b = part - p.G, end = unit_end(p, f, r), cap = f.group ? p.cap_group : p.cap_seq;
    RowItem it = {};
    it.src = f.group ? ~part : b;
    it.n_vt = f.n_vt;
    it.vt0 = r * 2 * p.tpt;
    if (f.group) {
      it.member0 = p.group_start[part];
      it.row0 = w.flags[part] & kGroupRows ? p.q_row0[p.members[it.member0]] : -1;
      it.first = w.flags[part] & kGroupFull;
      it.kv = w.table[part];
    } else {
      it.row0 = p.q_row0[b];
      it.first = f.first;
      it.kv = p.paged ? b : p.kv_row0[b];
    }
    for (int h = 0; h < p.KV; ++h) {
      const int u = row * p.KV + h;
      const int64_t us = us0 + static_cast<int64_t>(h) * cost, ue = us + cost;
      if (us >= to || ue <= from) continue;
      it.head = h;
      // pieces that hold blocks: a CTA whose range ends in the unit's own cost has none
      const int cb = cta_of(us + kUnitCost);  // first CTA with a block
      const int pieces = cta_of(ue - 1) - cb + 1;
      const int slot0 = p.compact ? 2 * cb + 1 : u + cb;
      const int64_t row0 = (f.group ? 0 : p.group_rows) + static_cast<int64_t>(slot0) * cap;
      // a sequence without shared keys writes its uncut rows itself
      const bool direct = !f.group && f.k0 == 0 && pieces == 1;
      if (c == cb) {
        p.unit_info[u] = make_int2(static_cast<int>(row0), pieces);
        if (pieces > 1) p.cut_unit[cb] = {static_cast<int>(row0), pieces, it.row0, it.vt0, it.n_vt, h, {}};
      }
      const int a = static_cast<int>(max(from - us - kUnitCost, static_cast<int64_t>(0)));
      const int e = static_cast<int>(min(to - us - kUnitCost, static_cast<int64_t>(nb)));
      const int step = c - cb;
      it.nblk = max(e - a, 0);
      it.k0 = f.k0 + a * kKeyBlock;
      it.k1 = min(f.k0 + e * kKeyBlock, end);
      it.slot = direct ? -1 : static_cast<int>(row0 + static_cast<int64_t>(p.compact && step > 0 ? 2 * step - 1 : step) * cap);
      p.items[u + c] = it;
      if (direct_items) kept[(u + c) % ITEMS] = it;
      if (from >= us) range[0] = p.cta_first[c] = u + c;
      if (to <= ue) range[1] = p.cta_last[c] = u + c;
    }
  }
  if (tid == 0 && from >= total) {  // nothing for this CTA
    p.cta_first[blockIdx.x] = 0;
    p.cta_last[blockIdx.x] = -1;
  }
  return direct_items;
}

// ---------------------------------------------------------------- geometry
template <int D, bool V8>
struct RowGeom {
  static_assert(!V8 || D == 128, "E4M3 V needs head_dim 128");
  static constexpr int KH = D / 64;               // 128-byte dim halves
  static constexpr int TILE = 16384 * KH;         // one K or V block, one query tile
  // ring slots, a K or a V block each: K in 0 and 2, V in 1 and 3
  static constexpr int NS = 4;
  static constexpr int RING = 2 * TILE;           // the ring lies behind the two query tiles
  static constexpr int RAW = RING + NS * TILE;
  static constexpr int STAGED = RAW + (V8 ? 16384 : 0);  // rows on their way out, STAGE bytes a softmax warp
  static constexpr int STAGE = 2048;
  static constexpr int SMEM = STAGED + kSoftmaxWarps * STAGE + 1024;
  static constexpr int S_COL = 0, O_COL = 256, TMEM_COLS = 512;
  static_assert(PlanSpace::bytes(kPlanMost, kPlanMost) <= STAGED, "a plan fits");
  static_assert(SMEM <= 227 * 1024 - 2048, "shared memory budget, 2 KB of static variables aside");
};

SD_DEV RowItem load_item(const RowItem* at) {
  RowItem it;
  const int4* s = reinterpret_cast<const int4*>(at);
  int4* d = reinterpret_cast<int4*>(&it);
#pragma unroll
  for (int i = 0; i < 3; ++i) d[i] = s[i];
  return it;
}
// Keys from here on are hidden from some of the unit's rows (its first row sees those before).
SD_DEV int first_hidden(const RowItem& it) { return it.src < 0 ? it.k1 : min(it.first + it.vt0 + 1, it.k1); }
// First block of the item with keys that some row does not see or that do not exist (none: past the last block).
SD_DEV int first_washed(const RowItem& it) { return max(first_hidden(it) - it.k0, 0) / kKeyBlock; }
// Some row of a tile with `halves` half blocks of the item sees a key that another row does not see.  (A tile that ends
// before the first such block neither waits for the washing nor looks at what it noted: it may be done before.)
SD_DEV bool sees_washed(const RowItem& it, int halves) {
  return first_hidden(it) < it.k1 && halves > 2 * first_washed(it);
}
// The halves of a bf16 pair that are infinite or NaN, as a mask of ones over them.
SD_DEV uint32_t not_finite(uint32_t w) {
  const uint32_t hi = ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
  return (hi >> 15) * 0xffffu;
}

// Two E4M3 codes, each in the upper byte of a half, as f16: the bits moved to f16's exponent and mantissa are the value
// times 2^-8 (f16's bias is 15, E4M3's 7; subnormals are subnormals in both), and the product with 2^8 is exact.
// (The NaN codes come out as 480.)
SD_DEV uint32_t e4m3_f16(uint32_t x) {
  const uint32_t v = (x & 0x80008000u) | ((x >> 1) & 0x3f803f80u);
  uint32_t y;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(v), "r"(0x5c005c00u));
  return y;
}

// half blocks (64 keys) of row tile t of an item
SD_DEV int tile_halves(const RowParams& p, const RowItem& it, int t) {
  const int v0 = it.vt0 + t * p.tpt;
  if (v0 >= it.n_vt) return 0;
  const int end = it.src < 0 ? it.k1 : min(it.first + min(v0 + p.tpt, it.n_vt), it.k1);
  return end <= it.k0 ? 0 : (end - it.k0 + kKeyBlock / 2 - 1) / (kKeyBlock / 2);
}

// Bounded waits of this kernel's warps, most of which wait most of the time: the hint lets the hardware put a warp
// to sleep for up to a millisecond instead of having it poll beside the softmax warps.  A wait that runs out (one second)
// ends the CTA's work: its warps leave their loops, the status says so, and the rows that they stood for are NaN.  Copies
// and products under way are waited for by the warps that issued them, whether or not a wait of their own ran out: the
// warp that would have used them may have left.
SD_DEV bool mbar_try_sleep(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}
SD_DEV bool row_wait(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  bool got = mbar_try_sleep(bar, parity);
  if (!got) {
    const uint64_t t0 = globaltimer_ns();
    do {
      got = mbar_try_sleep(bar, parity);
    } while (!got && globaltimer_ns() - t0 < limit_ns);
  }
  return __all_sync(0xffffffffu, got);
}

// A wait whose failure is looked at later: most of these barriers are complete when their turn comes, and a vote a wait
// would be most of its cost.
SD_DEV void lazy_wait(uint64_t* bar, uint32_t parity, bool& dead, uint64_t limit_ns) {
  if (mbar_try_sleep(bar, parity) || dead) return;
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_sleep(bar, parity)) {
    if (globaltimer_ns() - t0 > limit_ns) {
      dead = true;
      break;
    }
  }
}

// 3-D tiled load that stays in L2 as the hardware sees fit (K/V blocks are read again by other CTAs)
SD_DEV void tma_tile_3d(void* dst, const CUtensorMap* map, int32_t c0, int32_t c1, int32_t c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
SD_DEV void tma_rows4(void* dst, const CUtensorMap* map, int32_t r0, int32_t r1, int32_t r2, int32_t r3,
                      uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(smem_u32(bar))
      : "memory");
}

// ---------------------------------------------------------------- main kernel
template <int N>
SD_DEV void more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
SD_DEV void fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// One lane of a converged warp; the loops around it stay warp-uniform, so that descriptors and counters live in
// uniform registers.
SD_DEV bool elect_one() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(ok));
  return ok != 0;
}

// Two fp32 values in a 64-bit register: the packed arithmetic issues both at once.  The assembly here is volatile so
// that it is issued in the order written: a warp issues in order, and only an order that alternates between the
// exponential unit and the FMA units keeps both busy (scheduled by the compiler the two took turns, 1.3 times as long).
SD_DEV uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
SD_DEV void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
SD_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
SD_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm volatile("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SD_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm volatile("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SD_DEV float fma_sat(float a, float b, float c) {  // clamped to [0, 1]
  float r;
  asm volatile("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
SD_DEV float exp2_unit(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two weights as the P V product takes them: bf16, beside E4M3 V f16
template <bool V8>
SD_DEV uint32_t round_weights(float lo, float hi) {
  uint32_t r;
  if constexpr (V8)
    asm volatile("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm volatile("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
SD_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
SD_DEV float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x on the FMA units: x = n + f with f in [-1/2, 1/2], 2^f by the cubic through 1 at 0 with the least largest relative
// error on that interval (1.0e-04, against the 2^-8, or 2^-11, that P is rounded to), n added to the exponent.  x is clamped to
// [-127, 127] as z = (x + 127) / 254 in [0, 1], which costs nothing beside the scaling; z's rounding moves x by less
// than 2^-16.  At -127 the exponent and the mantissa of 1 cancel: masked keys and all that is smaller give exactly 0.
// (The clamp hides a NaN: the caller looks for one.)
constexpr float kPolyLow = -127.f, kPolySpan = 254.f;
constexpr float kRound = 12582912.f;  // 1.5 x 2^23: the low mantissa bits of x + kRound are the nearest integer
struct Poly2 {
  uint64_t z, t, f, y;
  template <int STEP>
  SD_DEV void step(float s0, float s1, float zs, float zn) {
    if constexpr (STEP == 0) {
      const float a = fma_sat(s0, zs, zn), b = fma_sat(s1, zs, zn);
      z = pack2(a, b);
    } else if constexpr (STEP == 1) {
      t = fma2(z, pack2(kPolySpan, kPolySpan), pack2(kRound + kPolyLow, kRound + kPolyLow));
    } else if constexpr (STEP == 2) {  // -(n - kPolyLow)
      f = fma2(t, pack2(-1.f, -1.f), pack2(kRound + kPolyLow, kRound + kPolyLow));
    } else if constexpr (STEP == 3) {
      f = fma2(z, pack2(kPolySpan, kPolySpan), f);
    } else if constexpr (STEP == 4) {
      y = fma2(f, pack2(kExpC3, kExpC3), pack2(kExpC2, kExpC2));
    } else if constexpr (STEP == 5) {
      y = fma2(y, f, pack2(kExpC1, kExpC1));
    } else {
      y = fma2(y, f, pack2(1.f, 1.f));
    }
  }
  SD_DEV void result(float& a, float& b) {
    float tl, th, yl, yh;
    unpack2(t, tl, th);
    unpack2(y, yl, yh);
    // (one multiply-add: the compiler's shift and addition are two instructions)
    uint32_t ra, rb;
    asm volatile("mad.lo.u32 %0, %1, 8388608, %2;" : "=r"(ra) : "r"(__float_as_uint(tl)), "r"(__float_as_uint(yl)));
    asm volatile("mad.lo.u32 %0, %1, 8388608, %2;" : "=r"(rb) : "r"(__float_as_uint(th)), "r"(__float_as_uint(yh)));
    a = __uint_as_float(ra);
    b = __uint_as_float(rb);
  }
};

// Eight pairs of scores at once: six take the exponential unit (12 x 8.5 clocks a warp), two the polynomial, whose
// steps lie between the others'.  A pair costs about 8 issue slots by the unit and 24 by the polynomial, so a quarter
// of the pairs balances the two.  Probabilities as pairs of 16 bits in w[0 .. 7], their sums added to `sum`.
template <bool V8>
SD_DEV void eight_pairs(const float* s, uint64_t sc, uint64_t ng, float zs, float zn, uint64_t (&sum)[2], float& seen,
                        const float* vs, uint32_t* w) {
  Poly2 p[2];
  float x[12], y[12], a, b;
  // E4M3: the keys' scales, two a pair
  ulonglong2 g[V8 ? 4 : 1];
  if constexpr (V8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] = reinterpret_cast<const ulonglong2*>(vs)[e];
  }
  auto weigh = [&](int e, float p0, float p1) {
    uint64_t v = pack2(p0, p1);
    sum[e & 1] = add2(sum[e & 1], v);
    if constexpr (V8) {
      v = mul2(v, e & 1 ? g[e >> 1].y : g[e >> 1].x);
      unpack2(v, p0, p1);
    }
    w[e] = round_weights<V8>(p0, p1);
  };
#define SD_X(E) unpack2(fma2(pack2(s[2 * (E)], s[2 * (E) + 1]), sc, ng), x[2 * (E)], x[2 * (E) + 1]);
#define SD_Y(E) y[E] = exp2_unit(x[E]);
#define SD_P(I, K) p[I].step<K>(s[12 + 2 * (I)], s[13 + 2 * (I)], zs, zn);
#define SD_W(E) weigh(E, y[2 * (E)], y[2 * (E) + 1]);
  SD_X(0) SD_Y(0) SD_P(0, 0)
  seen = max3_nan(seen, s[12], s[13]);
  SD_Y(1) SD_X(1) SD_P(1, 0)
  seen = max3_nan(seen, s[14], s[15]);
  SD_Y(2) SD_P(0, 1) SD_X(2)
  SD_Y(3) SD_P(1, 1) SD_P(0, 2)
  SD_Y(4) SD_W(0) SD_P(1, 2) SD_X(3)
  SD_Y(5) SD_P(0, 3) SD_P(1, 3)
  SD_Y(6) SD_W(1) SD_X(4) SD_P(0, 4)
  SD_Y(7) SD_P(1, 4) SD_X(5)
  SD_Y(8) SD_W(2) SD_P(0, 5) SD_P(1, 5)
  SD_Y(9) SD_W(3) SD_P(0, 6) SD_P(1, 6)
  SD_Y(10)
  p[0].result(a, b);
  weigh(6, a, b);
  SD_Y(11)
  p[1].result(a, b);
  weigh(7, a, b);
  SD_W(4) SD_W(5)
#undef SD_X
#undef SD_Y
#undef SD_P
#undef SD_W
}
// The rare way: exact where the scores are large, whatever they are (infinities and NaNs too).
template <bool V8>
SD_DEV void one_pair(const float* s, uint64_t sc, uint64_t minus_m, uint64_t& sum, const float* vs, uint32_t* w) {
  float a, b;
  unpack2(fma2(add2(pack2(s[0], s[1]), minus_m), sc, pack2(0.f, 0.f)), a, b);
  a = exp2_unit(a);
  b = exp2_unit(b);
  sum = add2(sum, pack2(a, b));
  if (V8) a *= vs[0], b *= vs[1];
  *w = round_weights<V8>(a, b);
}

// P = 2^((s - m) scale) of 64 scores as bf16 (V8: f16) in 32 TMEM columns; returns the sum, and in `seen` a NaN if there is one
// among the scores that took the polynomial.  USUAL: as s scale - m scale, eight of the 32 pairs by the polynomial.
// V8: each P is rounded after a multiplication by its key's scale (the codes themselves are exact in f16).
// `before_last` is called when a quarter is left.  Not USUAL: what is there already stays for rows that are not `mine`,
// so that no row's bits depend on what its neighbours' scores are.
template <bool USUAL, bool V8, typename Hook>
SD_DEV float row_probabilities(const float* s, float scale, float m, uint32_t ta, float& seen, const float* vs, bool mine,
                               Hook before_last) {
  const float neg = USUAL ? -m * scale : -m;
  const uint64_t sc = pack2(scale, scale), ng = pack2(neg, neg);
  const float zs = scale * (1.f / kPolySpan), zn = (neg - kPolyLow) * (1.f / kPolySpan);
  uint64_t sum[2] = {0, 0};
  uint32_t w[32];
  seen = -INFINITY;
  auto store = [&](int at) {
    if constexpr (!USUAL) {
      float old[16];
      umma::tmem_ld16(ta + at, old);
      umma::tmem_wait_ld16(old);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!mine) w[at + e] = __float_as_uint(old[e]);
    }
    umma::tmem_st16_words(ta + at, reinterpret_cast<const uint32_t(&)[16]>(w[at]));
  };
  if (!USUAL) umma::tmem_wait_st();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (q == 3) before_last();
    if (USUAL) {
      eight_pairs<V8>(s + 16 * q, sc, ng, zs, zn, sum, seen, vs + 16 * q, w + 8 * q);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) one_pair<V8>(s + 16 * q + 2 * e, sc, ng, sum[e & 1], vs + 16 * q + 2 * e, w + 8 * q + e);
    }
    if (q == 1) store(0);
  }
  store(16);
  float a, b;
  unpack2(add2(sum[0], sum[1]), a, b);
  return a + b;
}

// A half of a block known at run time only, where std::integral_constant is one known to the compiler.
struct Half {
  static constexpr int value = 0;
  int h;
  SD_DEV operator int() const { return h; }
};

template <int D, int SRC>
__global__ void __launch_bounds__(RowRoles<SRC>::THREADS, 1) row_attention_kernel(
    const RowParams p, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap tmap,
    const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  constexpr bool V8 = RowRoles<SRC>::V8;
  using Geo = RowGeom<D, V8>;
  constexpr int NS = Geo::NS, KH = Geo::KH, ITEMS = RowRoles<SRC>::ITEMS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[NS], empty[NS], raw_full, raw_empty;
  __shared__ uint64_t q_full, q_empty, s_full[2][2], p_full[2][2], pv_done[2], o_full[2], v_clean[2], bad_read[2][2], fin[2];
  // [tile][its item % 2]: keys past first_hidden whose V holds an infinity or a NaN.  A tile's items here are those of
  // sees_washed: only those are waited for by both sides.
  __shared__ uint32_t s_bad[2][2][4][8];  // (a washing warp its own eight words)
  __shared__ RowItem s_items[ITEMS];  // the CTA's first items
  __shared__ int s_range[2];
  __shared__ int s_lost;  // first item that a softmax warp gave up on
  // E4M3: scales of the keys in V's ring slots, in units of s_unit, and the largest finite one of each widening warp's keys
  __shared__ alignas(16) float s_vs[V8 ? 2 : 1][kKeyBlock], s_vs_top[V8 ? 2 : 1][4];
  __shared__ float s_unit[2];
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], V8 && (s & 1) ? 4 : 1);  // a TMA block, or the four widening warps
      mbar_init(&empty[s], 2);  // both MMA warps have read it
    }
    for (int t = 0; t < 2; ++t) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&s_full[t][h], 1);
        mbar_init(&p_full[t][h], 4);
      }
      mbar_init(&pv_done[t], 1);
      mbar_init(&o_full[t], 1);
      mbar_init(&v_clean[t], 4);
      mbar_init(&bad_read[t][0], 4);
      mbar_init(&bad_read[t][1], 4);
    }
    mbar_init(&raw_full, 1);
    mbar_init(&raw_empty, 4);
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 2);
    mbar_init(&fin[0], 1);
    mbar_init(&fin[1], 1);
    fence_barrier_init();
  }
  if (tid == 0) s_lost = 0x7fffffff;
  if (warp == kIssueWarp) {
    umma::tmem_alloc(&s_tmem, Geo::TMEM_COLS);
    umma::tmem_relinquish();
  }
  if (warp == kLoadWarp && lane == 0) {
    prefetch_tmap(&qmap);
    if (p.G > 0) prefetch_tmap(&tmap);
    prefetch_tmap(&kmap);
    prefetch_tmap(&vmap);
  }
  grid_dep_wait();
  grid_dep_launch();
  bool have_items = false;
  if (p.plan) {
    have_items = make_plan<ITEMS>(p, smem, reinterpret_cast<int64_t(*)[32]>(smem + Geo::STAGED), s_range, s_items);
    fence_proxy_async();  // its generic writes are over before the copies into the same memory begin
  } else if (tid == 0) {
    const bool same = *p.plan_key == p.key;
    if (!same && blockIdx.x == 0) raise_status(p.status, SPECDEC_STATUS_PLAN_MISMATCH);
    s_range[0] = same ? p.cta_first[blockIdx.x] : 0;
    s_range[1] = same ? p.cta_last[blockIdx.x] : -1;
  }
  __syncthreads();
  const int i0 = s_range[0], i1 = s_range[1];
  if (!have_items)
    for (int e = tid; e < 3 * min(i1 - i0 + 1, ITEMS); e += blockDim.x)
      reinterpret_cast<int4*>(s_items + (i0 + e / 3) % ITEMS)[e % 3] = reinterpret_cast<const int4*>(p.items + i0)[e];
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = s_tmem;
  auto item_at = [&](int i) { return i - i0 < ITEMS ? s_items[i % ITEMS] : load_item(p.items + i); };

  if (warp >= kSoftmaxWarp && warp < kWidenWarp) {
    more_regs<RowRoles<SRC>::SOFTMAX_REGS>();
    // ------------------------------------------------------------ softmax and epilogue: a thread a row
    const int t = (warp - kSoftmaxWarp) >> 2, row = tid & 127;
    const int tok = row / p.n_rep, rep = row - tok * p.n_rep;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 5;
    const uint32_t s_ta = umma::taddr(tmem, lanes, Geo::S_COL + t * 128);
    const uint32_t o_ta = umma::taddr(tmem, lanes, Geo::O_COL + t * D);
    const float scale = p.scale_log2;
    uint32_t sn = 0, pv = 0, on = 0;  // sn: phase bits of s_full; pv: halves handed over
    uint32_t blk = 0, rd[2] = {0, 0};  // blocks before this item; items of each tile that read s_bad
    bool dead = p.wait_ns == 0, idle = false;  // idle: no work in the item before
    for (int i = i0; i <= i1; ++i) {
      const RowItem it = item_at(i);
      if (it.nblk == 0) continue;
      // this row's visible keys end at `limit` (0: no row here)
      const int vt = it.vt0 + t * p.tpt + tok;
      int limit = 0;
      if (tok < p.tpt && vt < it.n_vt) {
        if (it.src >= 0) {
          limit = min(it.first + vt + 1, it.k1);
        } else if (it.first) {
          limit = it.k1;
        } else {
          const int mb = vt / p.q_max;
          if (vt - mb * p.q_max < p.member_row[it.member0 + mb].y) limit = it.k1;
        }
      }
      const int nh = tile_halves(p, it, t), nh_other = tile_halves(p, it, t ^ 1);
      const int hidden = first_hidden(it), blk0 = blk;
      blk += (max(nh, nh_other) + 1) / 2;
      const bool reads = sees_washed(it, nh), other_reads = sees_washed(it, nh_other);
      const uint32_t rd_mine = rd[t] & 1, rd_other = rd[t ^ 1];
      rd[t] += reads;
      rd[t ^ 1] += other_reads;
      if (nh == 0) {  // no tile, or a piece past the tile's keys: the row's other pieces are all of it
        if (it.slot >= 0 && limit > 0) p.part_ml[it.slot + t * kRowTile + row] = make_float2(-INFINITY, kNoPart);
        idle = true;
        continue;
      }
      const bool was_idle = idle;
      idle = false;
      const bool any_row = __any_sync(0xffffffffu, limit > 0);
      const int least = __reduce_min_sync(0xffffffffu, limit > 0 ? limit : 0x7fffffff);
      float m = -INFINITY, l = 0.f;
      float unit = 1.f;  // E4M3: of the item's scales
      // At head_dim 64 one half's scores are loaded while the other's are worked on; at 128 the next half's products
      // are not done by then, and a warp that waits for them works on nothing.
      constexpr bool AHEAD = D == 64;
      float s[AHEAD ? 2 : 1][64];
      auto load = [&](auto half) {
        const int H = half;
        lazy_wait(&s_full[t][H], (sn >> H) & 1, dead, p.wait_ns);
        sn ^= 1u << H;
        umma::fence_after_sync();
        if (any_row) {
          umma::tmem_ld32(s_ta + 64 * H, s[AHEAD ? H : 0]);
          umma::tmem_ld32(s_ta + 64 * H + 32, s[AHEAD ? H : 0] + 32);
        }
      };
      // Washing: what a masked key's zero probability meets must be finite.  V rows past the last key (the next
      // sequence's, a page's old contents) become zero as far as the products reach; an infinity or a NaN in a key that
      // only some rows see becomes zero, too, and its key is noted for the rows that do see it (after the epilogue).
      // The tile that has work in every block does it, a quarter of the rows a warp; the MMA warps wait for it.
      // (E4M3: the widening warps do.)
      const int wash = V8 || nh < nh_other || (nh == nh_other && t == 1) ? 0x7fffffff : first_washed(it);
      auto wash_block = [&](int j) {
        uint32_t* const bad = s_bad[t][rd_mine][warp & 3];
        uint32_t* const bad_other = s_bad[t ^ 1][rd_other & 1][warp & 3];
        const uint32_t slot = ((blk0 + j) & 1) * 2 + 1;
        if (j == first_washed(it) && other_reads && rd_other >= 2)
          lazy_wait(&bad_read[t ^ 1][rd_other & 1], (rd_other / 2 - 1) & 1, dead, p.wait_ns);
        lazy_wait(&full[slot], ((blk0 + j) >> 1) & 1, dead, p.wait_ns);
        if (__any_sync(0xffffffffu, dead)) return;  // what is not washed is not announced
        if (j == first_washed(it)) {
          if (lane < 8 && reads) bad[lane] = 0;
          if (lane < 8 && other_reads) bad_other[lane] = 0;
          __syncwarp();
        }
        uint8_t* const v = smem + Geo::RING + slot * Geo::TILE;
        const int key0 = it.k0 + j * kKeyBlock;
        // (the MMAs take 16 keys a step, and none of the steps past the last key's)
        const int o0 = max(hidden - key0, 0) * 128, o1 = min(it.k1 - key0, kKeyBlock) * 128;
        // (small code: what runs once an item is bound by fetching its instructions)
#pragma unroll 1
        for (int x = 0; x < KH; ++x) {
#pragma unroll 1
          for (int o = o0 + (warp & 3) * 512 + lane * 16; o < ((o1 + 2047) & ~2047); o += 2048) {
            uint4* const chunk = reinterpret_cast<uint4*>(v + x * 16384 + o);
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (o < o1) {
              w = *chunk;
              const uint4 b = make_uint4(not_finite(w.x), not_finite(w.y), not_finite(w.z), not_finite(w.w));
              if (!(b.x | b.y | b.z | b.w)) continue;
              w = make_uint4(w.x & ~b.x, w.y & ~b.y, w.z & ~b.z, w.w & ~b.w);
              const int bit = key0 + o / 128 - hidden;
              if (reads) atomicOr(&bad[bit >> 5], 1u << (bit & 31));
              if (other_reads) atomicOr(&bad_other[bit >> 5], 1u << (bit & 31));
            }
            *chunk = w;
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_clean[slot >> 1]);
      };
      auto work = [&](auto half, int k) {
        const int H = half;
        const bool more = k + 1 < nh;
        if (H == 0 && k / 2 >= wash) wash_block(k / 2);
        if (!AHEAD) load(half);
        if (!any_row) {
          if (AHEAD && more) load(std::integral_constant<int, AHEAD ? 1 - decltype(half)::value : 0>{});
        } else {
          float(&x)[64] = s[AHEAD ? H : 0];
          umma::tmem_wait_ld32(x);
          umma::tmem_wait_ld32(x + 32);
          const int key0 = it.k0 + k * (kKeyBlock / 2);
          const bool masked = least < key0 + kKeyBlock / 2;
          if (masked) {
            const int vis = limit - key0;
#pragma unroll
            for (int c = 0; c < 64; ++c) x[c] = c < vis ? x[c] : -INFINITY;
          }
          auto row_max = [&]() {
            float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int c = 4; c < 60; c += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e) mx[e] = max3_nan(mx[e], x[c + e], x[c + 4 + e]);
            return max3_nan(max3_nan(mx[0], mx[1], x[60]), max3_nan(mx[2], mx[3], x[61]), max_nan(x[62], x[63]));
          };
          if (k == 0) m = row_max();
          float seen, vs_top = 0.f;  // E4M3: the block's largest scale
          const float* vs = nullptr;
          if constexpr (V8) {  // the block's scales are there when its codes are widened
            const int b = blk0 + k / 2;
            vs = s_vs[b & 1] + 64 * H;
            if (H == 0) lazy_wait(&full[(b & 1) * 2 + 1], (b >> 1) & 1, dead, p.wait_ns);
            if (k == 0) unit = s_unit[b & 1];
          }
          auto next = [&]() {
            if (AHEAD && more) load(std::integral_constant<int, AHEAD ? 1 - decltype(half)::value : 0>{});
          };
          float sum = row_probabilities<true, V8>(x, scale, m == -INFINITY ? 0.f : m, s_ta + 64 * H, seen, vs, true, next);
          // Past the reference by more than 2^30 (or no reference yet, every key so far being masked): the
          // reference takes in this half block's maximum, O and l are rescaled and it is done again, once.  So it is
          // for NaN and infinite scores, and where the reference is so large that the roundings of m scale and of the
          // polynomial's argument (3 2^-24 of it) would show beside P's own.  A NaN stays one.
          // (Rows of the tile that are no token's hold anything; rows that see nothing here add nothing.)
          if constexpr (V8) {
            const float4 y = *reinterpret_cast<const float4*>(s_vs_top[(blk0 + k / 2) & 1]);
            vs_top = fmaxf(fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)), kGrowF16 / kGrow);
          }
          // E4M3: nor may a weight pass f16's range; where the scales themselves would, the reference goes that much higher.
          // (Whose keys' scales these are is asked only here.)
          auto moves = [&](float scales) {
            const bool grown = V8 ? !(sum * scales < kGrowF16) : !(sum < kGrow);
            return limit > key0 && (grown || seen != seen || !(fabsf(m) * scale < kLargeScore));
          };
          bool redo = moves(vs_top);
          if (__any_sync(0xffffffffu, redo)) {
            float top = row_max();
            if constexpr (V8) {
              float scales = vs_top;
              if (masked) {
                scales = kGrowF16 / kGrow;
#pragma unroll 1
                for (int c = 0; c < min(limit - key0, kKeyBlock / 2); ++c)
                  if (fabsf(vs[c]) < INFINITY) scales = fmaxf(scales, fabsf(vs[c]));
                __syncwarp();
                redo = moves(scales);
              }
              if (scales > kGrowF16 / 2) top += __log2f(scales * (2 / kGrowF16)) / scale;
            }
            const float to = redo ? max_nan(m, top) : m;
            const float alpha = to == m ? 1.f : fast_exp2((m - to) * scale);  // (no reference yet: 0 of nothing)
            m = to;
            l *= alpha;
            if (k > 0) {
              lazy_wait(&pv_done[t], (pv - 1) & 1, dead, p.wait_ns);  // the MMAs over the half before this add to O
              umma::fence_after_sync();
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                float o[16];
                umma::tmem_ld16(o_ta + c, o);
                umma::tmem_wait_ld16(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= alpha;
                umma::tmem_st16(o_ta + c, o);
              }
            }
            const float again = row_probabilities<false, V8>(x, scale, m == -INFINITY ? 0.f : m, s_ta + 64 * H, seen, vs,
                                                             redo, []() {});
            if (redo) sum = again;
          }
          l += sum;
          umma::tmem_wait_st();
        }
        ++pv;
        umma::fence_before_sync();
        __syncwarp();
        // (after a wait that ran out an arrival might complete a phase that another warp's rows are missing from)
        if (lane == 0 && !dead) mbar_arrive(&p_full[t][H]);
      };
      constexpr std::integral_constant<int, 0> even{};
      constexpr std::integral_constant<int, 1> odd{};
      // (A slot's phases can be told apart only by a warp that is no more than one behind or ahead: a tile that had no
      // work in the item before may be far ahead, until the item's first scores are there.)
      if (!AHEAD && wash == 0 && was_idle) lazy_wait(&s_full[t][0], sn & 1, dead, p.wait_ns);
      if (AHEAD) load(even);
      // Pages at head_dim 128: one body for both halves, half the instructions to fetch, which items of few blocks wait for
      // (E4M3 64 requests x 5 rows over 8192 74.6 -> 65.0 us, 3 groups of 16 43.1 -> 40.9).  Long prompts are better off with two
      // (4 x 8192 tokens 838 us against 875).
      if constexpr (AHEAD || SRC == kPacked) {
        for (int k = 0; k < nh; k += 2) {
          work(even, k);
          if (k + 1 < nh) work(odd, k + 1);
          if (__any_sync(0xffffffffu, dead)) break;
        }
      } else {
        for (int k = 0; k < nh; ++k) {
          work(Half{k & 1}, k);
          if (__any_sync(0xffffffffu, dead)) break;
        }
      }
      if (__any_sync(0xffffffffu, dead) || !row_wait(&o_full[t], on & 1, p.wait_ns)) {
        atomicMin(&s_lost, i);
        break;
      }
      ++on;
      umma::fence_after_sync();
      // keys whose V is not finite and that some row does not see: the MMAs had zeros for it
      const bool any_bad = reads && __any_sync(0xffffffffu, (&s_bad[t][rd_mine][0][0])[lane] != 0);
      if (any_row) {
        if (it.slot >= 0) {
          const int64_t r = it.slot + t * kRowTile + row;
          if (limit > 0) p.part_ml[r] = make_float2(m * scale, l);
          // (a slot has room for whole warps of the rows that there may be)
          if (t * kRowTile + (row & ~31) < (it.src < 0 ? p.cap_group : p.cap_seq)) {
            float4* const to = p.part_o + (r >> 5) * (8 * D) + lane;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float o[32];
              umma::tmem_ld32(o_ta + c, o);
              umma::tmem_wait_ld32(o);
              if constexpr (V8) {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= unit;
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) to[(c / 4 + e) * 32] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          }
        } else {
          // Rows leave through shared memory, 64 bytes of a row at a time, so that a store covers whole sectors.
          uint8_t* const stage = smem + Geo::STAGED + (warp - kSoftmaxWarp) * Geo::STAGE;
          const float inv = l == 0.f ? 0.f : V8 ? unit / l : 1.f / l;
          int64_t at = -1;  // this row's first value
          if (limit > 0)
            at = static_cast<int64_t>(it.row0 + vt) * p.o_st + static_cast<int64_t>(it.head * p.n_rep + rep) * p.o_sh;
          int64_t to[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) to[g] = __shfl_sync(0xffffffffu, at, g * 8 + lane / 4);
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            float o[32];
            umma::tmem_ld32(o_ta + c, o);
            umma::tmem_wait_ld32(o);
            // 16-byte chunk e of row r lies at place e ^ (r / 2 % 4): no bank conflicts either way
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(stage + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4)) =
                  make_uint4(pack_bf16(o[8 * e] * inv, o[8 * e + 1] * inv), pack_bf16(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                             pack_bf16(o[8 * e + 4] * inv, o[8 * e + 5] * inv),
                             pack_bf16(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
            __syncwarp();
            const int ch = lane & 3;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int r = g * 8 + lane / 4;
              const uint4 y = *reinterpret_cast<const uint4*>(stage + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4));
              if (to[g] >= 0) *reinterpret_cast<uint4*>(p.out + to[g] + c + ch * 8) = y;
            }
            __syncwarp();
          }
        }
        umma::fence_before_sync();  // O is read: the arrival for the next item's first block lets its MMAs write it
        if (any_bad) {
          // A row that sees such a key gets its infinities and NaNs here, added to what has just been stored (weighed
          // by anything above zero they stay what they are).
          __threadfence_block();
          __syncwarp();
          for (int w = 0; w < 32 && limit > 0; ++w) {
            for (uint32_t bits = (&s_bad[t][rd_mine][0][0])[w]; bits != 0; bits &= bits - 1) {
              const int key = hidden + 32 * (w & 7) + __ffs(bits) - 1;
              if (key >= limit) continue;
              int64_t at = 0;  // packed: the row's first value; paged: the block
              float vs = 1.f;
              if (SRC == kPacked) {
                at = (it.kv + static_cast<int64_t>(key)) * p.v_st + it.head * p.v_sh;
              } else {
                int page = p.page_table[static_cast<int64_t>(it.kv) * p.max_pages + key / kPage];
                if (page < 0 || page >= p.num_pages) page = 0;
                at = static_cast<int64_t>(page) * p.KV + it.head;
                if (SRC == kPagedE4M3) vs = p.v_scale[at * kPage + key % kPage];
              }
#pragma unroll 1
              for (int d = 0; d < D; ++d) {
                float v;
                if (SRC == kPacked) {
                  v = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.v_pool)[at + d]);
                } else if (SRC == kPaged) {
                  v = __bfloat162float(
                      *reinterpret_cast<const __nv_bfloat16*>(p.v_pool + at * (kPage * D * 2) + kblock_offset(key % kPage, d)));
                } else {
                  const uint32_t h = e4m3x2_to_f16x2(p.v_pool[at * (kPage * D) + key % kPage * D + d]);
                  v = __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xffffu))) * vs;
                }
                if (fabsf(v) < INFINITY) continue;
                if (it.slot >= 0) {
                  const int64_t r = it.slot + t * kRowTile + row;
                  float* const o = reinterpret_cast<float*>(p.part_o + (r >> 5) * (8 * D) + d / 4 * 32 + lane) + d % 4;
                  *o += v;
                } else {
                  __nv_bfloat16* const o = p.out + static_cast<int64_t>(it.row0 + vt) * p.o_st +
                                           static_cast<int64_t>(it.head * p.n_rep + rep) * p.o_sh + d;
                  *o = __float2bfloat16(__bfloat162float(*o) + v);
                }
              }
            }
          }
        }
      }
      if (reads) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bad_read[t][rd_mine]);
      }
    }
  } else {
    fewer_regs<RowRoles<SRC>::OTHER_REGS>();
    if (warp == kLoadWarp) {
      // ---------------------------------------------------------- K/V blocks
      uint32_t n = 0;  // blocks issued (K and V each count)
      bool ok = true;
      for (int i = i0; i <= i1 && ok; ++i) {
        const RowItem it = item_at(i);
        if (it.nblk == 0) continue;
        const int nb = (max(tile_halves(p, it, 0), tile_halves(p, it, 1)) + 1) / 2;
        int ids = 0;  // paged: lane l holds the page of keys 16 (32 (j / 4) + l) ..
        for (int j = 0; j < nb && ok; ++j) {
          if (SRC != kPacked && (j & 3) == 0) {
            const int last = (it.k1 - 1) / kPage;
            const int pg = min(it.k0 / kPage + 8 * j + lane, last);
            ids = p.page_table[static_cast<int64_t>(it.kv) * p.max_pages + pg];
            if (ids < 0 || ids >= p.num_pages) {
              raise_status(p.status, SPECDEC_STATUS_BAD_PAGE);
              ids = 0;
            }
          }
#pragma unroll
          for (int kv = 0; kv < 2; ++kv, ++n) {
            const uint32_t s = n % NS, round = n / NS;
            if (V8 && kv) {  // codes; the widening warps take care of the block's ring slot
              const uint32_t r = n >> 1;
              if (r > 0 && !row_wait(&raw_empty, (r - 1) & 1, p.wait_ns)) {
                ok = false;
                break;
              }
              int pg[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) pg[e] = __shfl_sync(0xffffffffu, ids, 8 * (j & 3) + e) * p.KV + it.head;
              if (lane == 0) {
                mbar_arrive_expect_tx(&raw_full, 16384);
#pragma unroll
                for (int e = 0; e < 8; e += 4)
                  tma_rows4(smem + Geo::RAW + e * 2048, &vmap, pg[e], pg[e + 1], pg[e + 2], pg[e + 3],
                            &raw_full);
              }
              __syncwarp();
              continue;
            }
            if (round > 0 && !row_wait(&empty[s], (round - 1) & 1, p.wait_ns)) {
              ok = false;
              break;
            }
            uint8_t* dst = smem + Geo::RING + s * Geo::TILE;
            const CUtensorMap* map = kv ? &vmap : &kmap;
            if (SRC == kPacked) {
              if (lane == 0) {
                mbar_arrive_expect_tx(&full[s], Geo::TILE);
#pragma unroll
                for (int x = 0; x < KH; ++x)
                  tma_tile_3d(dst + x * 16384, map, x * 64, it.head, it.kv + it.k0 + j * kKeyBlock, &full[s]);
              }
            } else {
              int pg[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) pg[e] = __shfl_sync(0xffffffffu, ids, 8 * (j & 3) + e);
              if (lane == 0) {
                mbar_arrive_expect_tx(&full[s], Geo::TILE);
#pragma unroll
                for (int x = 0; x < KH; ++x)
#pragma unroll
                  for (int e = 0; e < 8; e += 4) {
                    auto row = [&](int k) { return (pg[k] * p.KV + it.head) * KH + x; };
                    tma_rows4(dst + x * 16384 + e * 2048, map, row(e), row(e + 1), row(e + 2), row(e + 3), &full[s]);
                  }
              }
            }
            __syncwarp();
          }
        }
      }
      if (!ok && lane == 0) raise_status(p.status, SPECDEC_STATUS_TIMEOUT);
      // copies under way land before the CTA leaves: the last of every slot (of the one for codes, the last)
      for (uint32_t k = n > NS ? n - NS : 0; k < n; ++k) {
        if (!V8 || (k & 1) == 0)
          (void)row_wait(&full[k % NS], (k / NS) & 1, kWaitLimitNs);
        else if (k + 2 >= n)
          (void)row_wait(&raw_full, (k >> 1) & 1, kWaitLimitNs);
      }
    } else if (warp < kQueryWarp) {
      // ---------------------------------------------------------- MMA issue, a warp a row tile
      // What such a warp does between two products is time that its tile waits for, and the tensor cores hold few
      // products ahead: one warp for both tiles was the bound (4300 clocks a block against 2600 of products).
      const int t = warp - kIssueWarp;
      constexpr uint32_t id_qk = umma::idesc_f16(128, kKeyBlock / 2, true, true, false, false);
      constexpr uint32_t id_pv = umma::idesc_f16(128, D, !V8, !V8, false, true);
      constexpr uint32_t high = umma::desc_high(1024, umma::kSwizzle128B);
      const uint32_t q_low = umma::desc_low(smem_u32(smem) + t * Geo::TILE, 16);
      const uint32_t k_low = umma::desc_low(smem_u32(smem + Geo::RING), 16);
      const uint32_t v_low = umma::desc_low(smem_u32(smem + Geo::RING), 16384);
      const uint32_t s_col = tmem + Geo::S_COL + t * 128, o_col = tmem + Geo::O_COL + t * D;
      uint32_t pn = 0, items = 0, cleaned = 0;  // pn, cleaned: phase bits of p_full, v_clean
      uint32_t ks = 0, kp = 0;  // ring slot of the next block in the ring, and its phase
      bool ok = true;
      auto next = [&](uint32_t& s, uint32_t& ph) {
        if (++s == NS) s = 0, ph ^= 1;
      };
      auto qk = [&](int h, uint32_t slot) {  // keys 64 h .. of the block
        const uint32_t kl = k_low + slot * (Geo::TILE >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t at = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
            umma::mma_f16_ss_low<id_qk, high>(s_col + 64 * h, q_low, at, kl, h * (8192 >> 4) + at, kk > 0);
          }
          umma::commit(&s_full[t][h]);
        }
        __syncwarp();
      };
      auto pv = [&](int h, uint32_t slot, bool acc, int steps) {  // steps of 16 keys
        const uint32_t vl = v_low + slot * (Geo::TILE >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            if (kk < steps)
              umma::mma_f16_ts_low<id_pv, high>(o_col, s_col, 64 * h + kk * 8, vl, h * (8192 >> 4) + kk * (2048 >> 4),
                                              acc || kk > 0);
          umma::commit(&pv_done[t]);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) umma::commit(bar);
        __syncwarp();
      };
      for (int i = i0; i <= i1 && ok; ++i) {
        const RowItem it = item_at(i);
        if (it.nblk == 0) continue;
        // (a reduction's result is known to be the same in all lanes: loops and descriptors stay in uniform registers)
        const int nh = __reduce_max_sync(0xffffffffu, tile_halves(p, it, t));
        const int nb = (max(nh, __reduce_max_sync(0xffffffffu, tile_halves(p, it, t ^ 1))) + 1) / 2;
        const int last_key = __reduce_max_sync(0xffffffffu, it.k1 - it.k0);
        const int wash = V8 ? 0x7fffffff : __reduce_max_sync(0xffffffffu, first_washed(it));
        ok = row_wait(&q_full, items & 1, p.wait_ns) && row_wait(&full[ks], kp, p.wait_ns);
        if (!ok) break;
        umma::fence_after_sync();
        if (nh > 0) qk(0, ks);
        if (nh > 1) qk(1, ks);
        if (nb == 1) commit(&q_empty);
        commit(&empty[ks]);
        next(ks, kp);
        for (int j = 0; j < nb; ++j) {
          const uint32_t vs = ks, vp = kp;  // this block's V; then the next block's K
          next(ks, kp);
          const bool last = j == nb - 1;
          ok = row_wait(&full[vs], vp, p.wait_ns);
          if (!last) ok = ok && row_wait(&full[ks], kp, p.wait_ns);
          if (!ok) break;
          umma::fence_after_sync();
          if (j >= wash) {  // the softmax warps wash this block's V
            ok = row_wait(&v_clean[vs >> 1], (cleaned >> (vs >> 1)) & 1, p.wait_ns);
            cleaned ^= 1u << (vs >> 1);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = 2 * j + h;
            if (k < nh) {
              ok = ok && row_wait(&p_full[t][h], (pn >> h) & 1, p.wait_ns);
              if (!ok) break;
              pn ^= 1u << h;
              umma::fence_after_sync();
              pv(h, vs, k > 0, (last_key - k * (kKeyBlock / 2) + 15) / 16);
              if (k == nh - 1) commit(&o_full[t]);
              if (k + 2 < nh) qk(h, ks);
            }
          }
          if (!ok) break;
          commit(&empty[vs]);
          if (!last) {
            commit(&empty[ks]);
            if (j + 2 == nb) commit(&q_empty);
            next(ks, kp);
          }
        }
        ++items;
      }
      if (!ok && lane == 0) raise_status(p.status, SPECDEC_STATUS_TIMEOUT);
      commit(&fin[t]);
      (void)row_wait(&fin[t], 0, kWaitLimitNs);  // products under way
    } else if (warp == kQueryWarp) {
      // ---------------------------------------------------------- query rows
      uint32_t items = 0;
      bool ok = true;
      for (int i = i0; i <= i1 && ok; ++i) {
        const RowItem it = item_at(i);
        if (it.nblk == 0) continue;
        const int tiles = it.vt0 + p.tpt < it.n_vt ? 2 : 1;
        if (items > 0) ok = row_wait(&q_empty, (items - 1) & 1, p.wait_ns);
        if (!ok) break;
        ++items;
        if (it.row0 >= 0) {
          // rows that follow one another are a box of n_rep heads x tpt tokens a tile; rows past them meet no other row
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full, static_cast<uint32_t>(tiles * KH * 128 * p.n_rep * p.tpt));
            for (int e = 0; e < tiles; ++e)
#pragma unroll
              for (int x = 0; x < KH; ++x)
                tma_tile_3d(smem + e * Geo::TILE + x * 16384, &qmap, x * 64, it.head * p.n_rep,
                            it.row0 + it.vt0 + e * p.tpt, &q_full);
          }
        } else {
          // a group's rows may be anywhere: a box of n_rep heads a token (the swizzle goes by the address, so that a
          // token may start in the middle of its pattern)
          const int tokens = min(2 * p.tpt, it.n_vt - it.vt0);
          int mine = 0;
          for (int base = 0; base < tokens; base += 32) {
            const int vt = it.vt0 + base + lane, mb = vt / p.q_max;
            if (base + lane < tokens) mine += vt - mb * p.q_max < p.member_row[it.member0 + mb].y;
          }
          mine = __reduce_add_sync(0xffffffffu, mine);
          if (lane == 0) mbar_arrive_expect_tx(&q_full, static_cast<uint32_t>(mine * KH * 128 * p.n_rep));
          __syncwarp();
          for (int base = 0; base < tokens; base += 32) {
            const int in = base + lane, vt = it.vt0 + in, mb = vt / p.q_max, e = vt - mb * p.q_max;
            if (in >= tokens) continue;
            const int2 mr = p.member_row[it.member0 + mb];
            if (e >= mr.y) continue;
            const int tile = in / p.tpt;
            uint8_t* dst = smem + tile * Geo::TILE + (in - tile * p.tpt) * p.n_rep * 128;
#pragma unroll
            for (int x = 0; x < KH; ++x)
              tma_tile_3d(dst + x * 16384, &tmap, x * 64, it.head * p.n_rep, mr.x + e, &q_full);
          }
        }
        __syncwarp();
      }
      if (!ok && lane == 0) raise_status(p.status, SPECDEC_STATUS_TIMEOUT);
      if (items > 0) (void)row_wait(&q_full, (items - 1) & 1, kWaitLimitNs);  // the last item's rows land before the CTA leaves
    } else {
      // ---------------------------------------------------------- E4M3: codes to f16, a thread a key
      if constexpr (V8) {
        const int r = tid - 32 * kWidenWarp;
        uint32_t n = 1, rd[2] = {0, 0};
        bool ok = true;
        for (int i = i0; i <= i1 && ok; ++i) {
          const RowItem it = item_at(i);
          if (it.nblk == 0) continue;
          const int nb = (max(tile_halves(p, it, 0), tile_halves(p, it, 1)) + 1) / 2;
          // the scale of the item's key x; 0 past the last key, where the codes (clamped pages) are finite or NaN
          auto scale_of = [&](int x) {
            const int key = it.k0 + x;
            if (key >= it.k1) return 0.f;
            int page = p.page_table[static_cast<int64_t>(it.kv) * p.max_pages + key / kPage];
            if (page < 0 || page >= p.num_pages) page = 0;  // the loading warp reports it
            return p.v_scale[(static_cast<int64_t>(page) * p.KV + it.head) * kPage + key % kPage];
          };
          // (washing, as the softmax warps do it for bf16)
          const int hidden = first_hidden(it);
          bool reads[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            reads[t] = sees_washed(it, tile_halves(p, it, t));
            if (!reads[t]) continue;
            if (rd[t] >= 2) ok = ok && row_wait(&bad_read[t][rd[t] & 1], (rd[t] / 2 - 1) & 1, p.wait_ns);
            if (lane < 8) s_bad[t][rd[t] & 1][r >> 5][lane] = 0;
          }
          __syncwarp();
          if (!ok) break;
          // For the unit of the item's scales every warp looks at its first 32 keys for itself, as far as all rows see them
          // that see anything of the item.
          float next = scale_of(r), unit = 1.f, per_unit = 1.f;
          const float first = lane < max(hidden - it.k0, 1) ? scale_of(lane) : 0.f;
          for (int j = 0; j < nb; ++j, n += 2) {
            const float sc = next;
            const int key = it.k0 + j * kKeyBlock + r;
            const bool in = key < it.k1;
            if (j + 1 < nb) next = scale_of((j + 1) * kKeyBlock + r);
            const uint32_t s = n % NS;
            ok = row_wait(&raw_full, (n >> 1) & 1, p.wait_ns);
            if (ok && n >= NS) ok = row_wait(&empty[s], (n / NS - 1) & 1, p.wait_ns);
            if (!ok) break;
            const uint8_t* src = smem + Geo::RAW + r * 128;
            uint8_t* dst = smem + Geo::RING + s * Geo::TILE + r * 128;
            uint32_t nan = 0;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const int ch = (c + r) & 7;  // rotated, so that neighbouring keys use different banks
              const uint4 x = *reinterpret_cast<const uint4*>(src + ch * 16);
              const uint32_t w[4] = {x.x, x.y, x.z, x.w};
              uint32_t y[8];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                nan |= (w[e] & 0x7f7f7f7fu) + 0x01010101u;
                y[2 * e] = in ? e4m3_f16(__byte_perm(w[e], 0, 0x1404)) : 0u;
                y[2 * e + 1] = in ? e4m3_f16(__byte_perm(w[e], 0, 0x3424)) : 0u;
              }
              uint8_t* d = dst + (ch >> 2) * 16384;
              const int g = (ch & 3) * 2;
              *reinterpret_cast<uint4*>(d + ((g ^ (r & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
              *reinterpret_cast<uint4*>(d + (((g + 1) ^ (r & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
            }
            const bool strange = in && ((nan & 0x80808080u) || !(fabsf(sc) < INFINITY));
            if (j == 0) {  // (here, so that the scales' loads and the codes' have the same time)
              const int x = (__float_as_int(first) >> 23) & 255;
              const bool fine = x != 0 && x != 255;
              const int sum = __reduce_add_sync(0xffffffffu, fine ? x - 127 : 0);
              const int of = __popc(__ballot_sync(0xffffffffu, fine));
              // (the clamp keeps the unit, its reciprocal and their products with scales up to 2^45 away in fp32's range)
              const int mean = of > 0 ? min(max(__float2int_rd(__fdividef(sum, of)), -80), 80) : 0;
              unit = __int_as_float((127 + mean - kScaleMean) << 23);
              per_unit = __int_as_float((127 - mean + kScaleMean) << 23);
            }
            // a key that some row does not see adds nothing that is not finite here
            const bool sc_fine = fabsf(sc) < INFINITY;
            const float counted = sc_fine ? fminf(fmaxf(sc * per_unit, -3.4e38f), 3.4e38f) : key >= hidden ? 0.f : sc;
            s_vs[s >> 1][r] = counted;
            const uint32_t top = __reduce_max_sync(0xffffffffu, sc_fine ? __float_as_uint(fabsf(counted)) : 0u);
            if (lane == 0) s_vs_top[s >> 1][r >> 5] = __uint_as_float(top);
            if (r == 0) s_unit[s >> 1] = unit;
            if (strange) {
#pragma unroll 1
              for (int d = 0; d < D; ++d)
                if ((src[d] & 0x7f) == 0x7f)
                  *reinterpret_cast<uint16_t*>(dst + (d >> 6) * 16384 + ((((d >> 3) & 7) ^ (r & 7)) << 4) + (d & 7) * 2) =
                      key >= hidden ? 0 : 0x7fff;
              if (key >= hidden) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
                  if (reads[t]) atomicOr(&s_bad[t][rd[t] & 1][r >> 5][(key - hidden) >> 5], 1u << ((key - hidden) & 31));
              }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&full[s]);
              mbar_arrive(&raw_empty);
            }
          }
          rd[0] += reads[0];
          rd[1] += reads[1];
        }
        if (!ok && lane == 0) raise_status(p.status, SPECDEC_STATUS_TIMEOUT);
      }
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  if (warp == kIssueWarp) {
    umma::fence_after_sync();
    umma::tmem_dealloc(tmem, Geo::TMEM_COLS);
  }
  // Where a wait ran out: NaN for the rows of that item and of those behind it (the join hands a part's NaN on), so that
  // nothing that the output or the workspace held before passes for a result.
  const int lost = tid < 2 * kRowTile ? s_lost : 0x7fffffff;
  if (lost <= i1 && tid == 0) raise_status(p.status, SPECDEC_STATUS_TIMEOUT);
#pragma unroll 1
  for (int i = lost; i <= i1; ++i) {
    const RowItem it = load_item(p.items + i);
    const int t = tid / kRowTile, row = tid % kRowTile, tok = row / p.n_rep, vt = it.vt0 + t * p.tpt + tok;
    if (it.nblk == 0 || tok >= p.tpt || vt >= it.n_vt) continue;
    if (it.slot >= 0) {  // (it has these rows' places, whether or not a group's member has so many tokens)
      p.part_ml[it.slot + tid] = make_float2(NAN, NAN);
      continue;
    }
    uint4* const o = reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(it.row0 + vt) * p.o_st +
                                              static_cast<int64_t>(it.head * p.n_rep + row - tok * p.n_rep) * p.o_sh);
#pragma unroll 1
    for (int c = 0; c < D / 8; ++c) o[c] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
  }
}

// ---------------------------------------------------------------- joining partial rows
// One warp two rows that lie next to each other in their slots (a lane pair reads a whole sector): the pieces of up
// to two units, each a run of slots.  A piece that saw no key of the row has sum 0 (kNoPart where its row was not written)
// and maximum -inf and weighs nothing.
// Bound by the latency of L2, so the loads of several pieces, sums and rows alike, are under way together.
struct Pieces {
  int64_t row;  // workspace row of the first piece
  int n, cap;
  bool compact;
  SD_DEV int64_t at(int i) const { return row + static_cast<int64_t>(compact && i > 0 ? 2 * i - 1 : i) * cap; }
};
// Lane l: row l % 2 of the pair, columns 4 (l / 2) .. + 3, and 64 further.  `out` NULL: no such row.
template <int D>
SD_DEV void join_pair(const RowParams& p, const Pieces& a, const Pieces& b, __nv_bfloat16* out, int lane) {
  constexpr int PER = D / 64, AT_ONCE = D == 64 ? 8 : 6;
  const int n = out ? a.n + b.n : 0, c = lane >> 1;
  float4 acc[PER] = {};
  float m = -INFINITY, l = 0.f;
  for (int base = 0; base < n; base += AT_ONCE) {
    float2 ml[AT_ONCE];
    float4 v[AT_ONCE][PER];
#pragma unroll
    for (int e = 0; e < AT_ONCE; ++e) {
      const int i = base + e;
      if (i >= n) {
        ml[e] = make_float2(-INFINITY, kNoPart);
        continue;
      }
      const int64_t r = i < a.n ? a.at(i) : b.at(i - a.n);
      ml[e] = p.part_ml[r];
      const float4* from = p.part_o + (r >> 5) * (8 * D) + (r & 31);
#pragma unroll
      for (int x = 0; x < PER; ++x) v[e][x] = from[(c + 16 * x) * 32];
    }
    float to = m;
#pragma unroll
    for (int e = 0; e < AT_ONCE; ++e) to = max_nan(to, ml[e].x);
    const float mu = to == -INFINITY ? 0.f : to, keep = fast_exp2(m - mu);
    m = to;
    l *= keep;
#pragma unroll
    for (int x = 0; x < PER; ++x) acc[x].x *= keep, acc[x].y *= keep, acc[x].z *= keep, acc[x].w *= keep;
#pragma unroll
    for (int e = 0; e < AT_ONCE; ++e) {
      if (ml[e].y == kNoPart) continue;  // (what such a piece's row holds may be anything)
      const float w = fast_exp2(ml[e].x - mu);  // (0 times what is not finite stays not finite)
      l += w * ml[e].y;
#pragma unroll
      for (int x = 0; x < PER; ++x) {
        acc[x].x += w * v[e][x].x;
        acc[x].y += w * v[e][x].y;
        acc[x].z += w * v[e][x].z;
        acc[x].w += w * v[e][x].w;
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (out) {
#pragma unroll
    for (int x = 0; x < PER; ++x)
      reinterpret_cast<uint2*>(out)[c + 16 * x] = make_uint2(pack_bf16(acc[x].x * inv, acc[x].y * inv),
                                                             pack_bf16(acc[x].z * inv, acc[x].w * inv));
  }
}

// rows of the units that a CTA boundary cuts (no groups): block (c, y) takes a share of the unit that is cut in CTA c
template <int D>
__global__ void __launch_bounds__(256) join_cut_kernel(const RowParams p) {
  grid_dep_wait();
  grid_dep_launch();
  const int4* from = reinterpret_cast<const int4*>(p.cut_unit + blockIdx.x);
  const int4 x = from[0], y = from[1];
  if (x.y == 0 || *p.plan_key != p.key) return;
  const int slot = x.x, row0 = x.z, vt0 = x.w, n_vt = y.x, head = y.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r2 = (blockIdx.y * 8 + warp) * 2; r2 < kUnitRows; r2 += gridDim.y * 16) {
    const int r = r2 + (lane & 1);
    const int t = r / kRowTile, e = r % kRowTile, tok = e / p.n_rep, vt = vt0 + t * p.tpt + tok;
    const bool in = tok < p.tpt && vt < n_vt;
    if (!__any_sync(0xffffffffu, in)) continue;
    const Pieces a{slot + r, x.y, p.cap_seq, p.compact != 0}, none{0, 0, 0, false};
    join_pair<D>(p, a, none,
                 in ? p.out + static_cast<int64_t>(row0 + vt) * p.o_st +
                          static_cast<int64_t>(head * p.n_rep + e - tok * p.n_rep) * p.o_sh
                    : nullptr,
                 lane);
  }
}

// rows of every sequence: its group's pieces and its own
template <int D>
__global__ void __launch_bounds__(256) join_rows_kernel(const RowParams p) {
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, pairs = (p.n_rep + 1) / 2;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t bi = w / (p.KV * pairs);
  const int hp = static_cast<int>(w - bi * (p.KV * pairs)), kvh = hp / pairs;
  const int rep = (hp - kvh * pairs) * 2 + (lane & 1);
  const int b = static_cast<int>(bi / p.q_max), i = static_cast<int>(bi - static_cast<int64_t>(b) * p.q_max);
  if (b >= p.B) return;
  const int4* from = reinterpret_cast<const int4*>(p.seq_rows + b);
  const int4 rec = from[0];
  const int first_vt = from[1].x;
  if (*p.plan_key != p.key || i >= rec.y) return;
  auto pieces = [&](int units, int vt, int cap) {
    const int2 info = p.unit_info[units + vt / (2 * p.tpt) * p.KV + kvh];
    const int in = vt % (2 * p.tpt), t = in / p.tpt;
    return Pieces{info.x + t * kRowTile + (in - t * p.tpt) * p.n_rep + rep, info.y, cap, p.compact != 0};
  };
  Pieces own = pieces(rec.z, i, p.cap_seq), pre{0, 0, 0, false};
  if (rec.w >= 0)
    pre = pieces(rec.w, first_vt + i, p.cap_group);
  else if (own.n == 1)
    return;  // written already
  join_pair<D>(p, pre, own,
               rep < p.n_rep ? p.out + static_cast<int64_t>(rec.x + i) * p.o_st +
                                   static_cast<int64_t>(kvh * p.n_rep + rep) * p.o_sh
                             : nullptr,
               lane);
}

// ---------------------------------------------------------------- host side
struct RowShape {
  int B, H, KV, D, q_max, G, M, sms;
};
struct RowSpace {
  int64_t units_most;
  size_t key, first, last, cut, seqs, mrow, info, items, ml, o, bytes;
  int cap_seq, cap_group;
  int64_t group_rows, rows;
};

static int row_sms(int requested) {
  const int dev = device_sm_count();
  return requested > 0 && requested < dev ? requested : dev;
}

static RowSpace row_space(const RowShape& s) {
  RowSpace w;
  const int n_rep = s.H / s.KV, tpt = kRowTile / n_rep;
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t seq_units = s.B * up(s.q_max, 2 * tpt) * s.KV;
  // groups' members: every group rounds its own rows up
  const int64_t group_units = s.G > 0 ? (up(static_cast<int64_t>(s.M) * s.q_max, 2 * tpt) + s.G) * s.KV : 0;
  auto cap = [&](int64_t tokens) {
    return static_cast<int>(tokens <= tpt ? up(tokens * n_rep, 32) * 32 : kUnitRows);
  };
  w.units_most = seq_units + group_units;
  w.cap_seq = cap(s.q_max);
  w.cap_group = s.G > 0 ? cap(static_cast<int64_t>(s.M) * s.q_max) : 0;
  w.group_rows = s.G > 0 ? (group_units + s.sms) * w.cap_group : 0;
  // without groups a slot is taken by cut units only, two a CTA; else by every unit and one more a CTA
  w.rows = w.group_rows + (s.G > 0 ? group_units + seq_units + s.sms + 1 : 2 * static_cast<int64_t>(s.sms) + 2) * w.cap_seq;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at = align_up(at + n, 256);
    return o;
  };
  w.key = take(8);
  w.first = take(4 * s.sms);
  w.last = take(4 * s.sms);
  w.cut = take(sizeof(CutUnit) * s.sms);
  w.seqs = take(sizeof(SeqRows) * s.B);
  w.mrow = take(8 * (s.M + 1));
  w.info = take(8 * (seq_units + group_units));
  w.items = take(sizeof(RowItem) * (seq_units + group_units + s.sms));
  w.ml = take(8 * w.rows);
  w.o = take(4 * w.rows * s.D);
  w.bytes = at;
  return w;
}

static bool row_shape_ok(const RowShape& s) {
  return s.B > 0 && s.H > 0 && s.KV > 0 && s.H % s.KV == 0 && s.H / s.KV <= kRowTile && (s.D == 64 || s.D == 128) &&
         s.q_max > 0 && s.G >= 0 && s.M >= 0 && s.B <= kPlanMost && s.G <= kPlanMost && s.M <= kPlanMost;
}

static int check_shape(const RowShape& s) {
  if (s.B <= 0 || s.H <= 0 || s.KV <= 0)
    return fail(SPECDEC_ERR_INVALID, "num_seqs, num_q_heads and num_kv_heads must be positive");
  if (s.H % s.KV != 0) return fail(SPECDEC_ERR_INVALID, "query heads must divide KV heads");
  if (s.H / s.KV > kRowTile) return fail(SPECDEC_ERR_UNSUPPORTED, "at most 128 query heads per KV head");
  if (s.D != 64 && s.D != 128) return fail(SPECDEC_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (s.q_max <= 0) return fail(SPECDEC_ERR_INVALID, "max_q_len must be positive");
  if (s.G < 0 || s.M < 0 || (s.G == 0 && s.M != 0)) return fail(SPECDEC_ERR_INVALID, "bad group or member count");
  if (s.B > kPlanMost || s.G > kPlanMost || s.M > kPlanMost)
    return fail(SPECDEC_ERR_UNSUPPORTED, "at most %d sequences, groups or members a call", kPlanMost);
  // item and slot numbers are 32-bit
  const RowSpace w = row_space(s);
  if (w.rows > 0x7fffffff || w.units_most > (1 << 30) || s.q_max > (1 << 30) ||
      static_cast<int64_t>(s.M) * s.q_max > (1 << 30) || w.bytes > (size_t(1) << 40))
    return fail(SPECDEC_ERR_UNSUPPORTED, "batch of %d sequences x %d tokens is too large for one call", s.B, s.q_max);
  return SPECDEC_OK;
}

static int check_rows(const void* q, const void* out, int64_t qs, int64_t qh, int64_t os, int64_t oh) {
  if (!q || !out) return fail(SPECDEC_ERR_INVALID, "q and out must be device pointers");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u)
    return fail(SPECDEC_ERR_INVALID, "q/out must be 16-byte aligned");
  if ((qs | qh | os | oh) & 7 || qs <= 0 || qh <= 0 || qs >= (int64_t(1) << 38) || qh >= (int64_t(1) << 38))
    return fail(SPECDEC_ERR_INVALID, "q/out strides must be positive multiples of 8 elements");
  return SPECDEC_OK;
}

static int fill_row_params(RowParams& p, const RowShape& s, void* ws, size_t ws_bytes, float sm_scale) {
  if (!(sm_scale > 0.f) || sm_scale > 1e30f) return fail(SPECDEC_ERR_INVALID, "sm_scale must be positive and finite");
  const RowSpace w = row_space(s);
  if (!ws || ws_bytes < w.bytes)
    return fail(SPECDEC_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws ? ws_bytes : 0, w.bytes);
  if (reinterpret_cast<uintptr_t>(ws) & 255u) return fail(SPECDEC_ERR_INVALID, "workspace must be 256-byte aligned");
  uint8_t* base = static_cast<uint8_t*>(ws);
  p.B = s.B;
  p.H = s.H;
  p.KV = s.KV;
  p.n_rep = s.H / s.KV;
  p.tpt = kRowTile / p.n_rep;
  p.q_max = s.q_max;
  p.G = s.G;
  p.M = s.M;
  p.grid = s.sms;
  p.compact = s.G == 0;
  p.min_quota = kMinQuota;
  p.cap_seq = w.cap_seq;
  p.cap_group = w.cap_group;
  p.group_rows = static_cast<int32_t>(w.group_rows);
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.wait_ns = wait_limit_ns();
  p.cta_first = reinterpret_cast<int32_t*>(base + w.first);
  p.cta_last = reinterpret_cast<int32_t*>(base + w.last);
  p.cut_unit = reinterpret_cast<CutUnit*>(base + w.cut);
  p.plan_key = reinterpret_cast<uint64_t*>(base + w.key);
  p.seq_rows = reinterpret_cast<SeqRows*>(base + w.seqs);
  p.member_row = reinterpret_cast<int2*>(base + w.mrow);
  p.unit_info = reinterpret_cast<int2*>(base + w.info);
  p.items = reinterpret_cast<RowItem*>(base + w.items);
  p.part_ml = reinterpret_cast<float2*>(base + w.ml);
  p.part_o = reinterpret_cast<float4*>(base + w.o);
  return SPECDEC_OK;
}

template <int D, int SRC>
static int launch_row_attention(RowParams& p, const CUtensorMap& qmap, const CUtensorMap& tmap, const CUtensorMap& kmap,
                                const CUtensorMap& vmap,
                                bool reuse_plan, cudaStream_t st) {
  p.plan = reuse_plan ? 0 : 1;
  p.key = 14695981039346656037ull;  // FNV-1a over what a plan's rows, keys and places in the workspace depend on
  for (const int64_t x : {static_cast<int64_t>(D), static_cast<int64_t>(SRC), static_cast<int64_t>(p.B),
                          static_cast<int64_t>(p.H), static_cast<int64_t>(p.KV), static_cast<int64_t>(p.q_max),
                          static_cast<int64_t>(p.G), static_cast<int64_t>(p.M), static_cast<int64_t>(p.grid), p.q_rows,
                          p.kv_rows, static_cast<int64_t>(p.num_pages), static_cast<int64_t>(p.max_pages)})
    for (int b = 0; b < 64; b += 8) p.key = (p.key ^ ((x >> b) & 255)) * 1099511628211ull;
  // the attribute belongs to the function on each device; setting it again is cheap and needs no state of its own
  const cudaError_t e = cudaFuncSetAttribute(row_attention_kernel<D, SRC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             RowGeom<D, RowRoles<SRC>::V8>::SMEM);
  if (e != cudaSuccess) return fail(SPECDEC_ERR_CUDA, "row_attention_kernel: %s", cudaGetErrorString(e));
  if (int rc = launch_pdl("row_attention_kernel", row_attention_kernel<D, SRC>, dim3(p.grid), dim3(RowRoles<SRC>::THREADS),
                          RowGeom<D, RowRoles<SRC>::V8>::SMEM, st, p, qmap, tmap, kmap, vmap))
    return rc;
  // keys of one block: no unit is cut (a launch less is 2 of the 12 us of one prompt of 60 tokens)
  if (p.G == 0 && !p.paged && p.kv_rows <= kKeyBlock) return SPECDEC_OK;
  if (p.G == 0)
    return launch_pdl("join_cut_kernel", join_cut_kernel<D>, dim3(p.grid, kMergeParts), dim3(256), 0, st, p);
  const int64_t warps = static_cast<int64_t>(p.B) * p.q_max * p.KV * ((p.n_rep + 1) / 2);
  return launch_pdl("join_rows_kernel", join_rows_kernel<D>, dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(256),
                    0, st, p);
}

// 3-D map {D, heads, rows} over packed rows with a {64, box_heads, box_rows} box and 128-byte swizzle; rows past the
// end read as zero
static int encode_packed_map(CUtensorMap* map, const void* base, int64_t rows, int heads, int D, int64_t st, int64_t sh,
                             int box_heads, int box_rows) {
  auto fn = get_encode_fn();
  if (!fn) return fail(SPECDEC_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(st) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SPECDEC_ERR_INVALID, "cuTensorMapEncodeTiled (packed) failed (%d)", static_cast<int>(r));
  return SPECDEC_OK;
}

}  // namespace sd

using namespace sd;

extern "C" size_t specdec_prompt_workspace_bytes(int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads,
                                                 int32_t head_dim, int32_t max_q_len, int32_t num_sms) {
  const RowShape s{num_seqs, num_q_heads, num_kv_heads, head_dim, max_q_len, 0, 0, row_sms(num_sms)};
  return row_shape_ok(s) ? row_space(s).bytes : 0;
}

extern "C" int specdec_prompt_attention(const SpecdecPromptArgs* a, specdec_stream_t stream) {
  if (!a) return fail(SPECDEC_ERR_INVALID, "args is NULL");
  const SpecdecBatch& bt = a->batch;
  const RowShape s{bt.num_seqs, bt.num_q_heads, a->num_kv_heads, a->head_dim, bt.max_q_len, 0, 0, row_sms(a->num_sms)};
  if (int rc = check_shape(s)) return rc;
  if (int rc = check_rows(a->q, a->out, a->q_stride_tok, a->q_stride_head, a->o_stride_tok, a->o_stride_head)) return rc;
  if (!a->k || !a->v) return fail(SPECDEC_ERR_INVALID, "k and v must be device pointers");
  if (!bt.q_row0 || !bt.q_len || !bt.ctx_len || !a->kv_row0) return fail(SPECDEC_ERR_INVALID, "batch arrays must be set");
  if (a->q_rows <= 0 || a->kv_rows <= 0 || a->q_rows > 0x7fffffff || a->kv_rows > 0x7fffffff)
    return fail(SPECDEC_ERR_INVALID, "row counts out of range");
  if ((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) & 15u)
    return fail(SPECDEC_ERR_INVALID, "k/v must be 16-byte aligned");
  const int64_t strides[4] = {a->k_stride_tok, a->k_stride_head, a->v_stride_tok, a->v_stride_head};
  for (const int64_t x : strides)
    if (x <= 0 || x % 8 || x >= (int64_t(1) << 38))
      return fail(SPECDEC_ERR_INVALID, "k/v strides must be positive multiples of 8 elements");
  RowParams p = {};
  if (int rc = fill_row_params(p, s, a->workspace, a->workspace_bytes, a->sm_scale)) return rc;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.q_st = a->q_stride_tok;
  p.q_sh = a->q_stride_head;
  p.o_st = a->o_stride_tok;
  p.o_sh = a->o_stride_head;
  p.q_row0 = bt.q_row0;
  p.q_len = bt.q_len;
  p.ctx_len = bt.ctx_len;
  p.kv_row0 = a->kv_row0;
  p.v_pool = static_cast<const uint8_t*>(a->v);
  p.v_st = a->v_stride_tok;
  p.v_sh = a->v_stride_head;
  p.q_rows = a->q_rows;
  p.kv_rows = a->kv_rows;
  p.status = a->status;
  CUtensorMap qm, tm, km, vm;
  if (int rc = encode_packed_map(&qm, a->q, a->q_rows, s.H, s.D, a->q_stride_tok, a->q_stride_head, p.n_rep, p.tpt)) return rc;
  tm = qm;  // whole prompts have no groups
  if (int rc = encode_packed_map(&km, a->k, a->kv_rows, s.KV, s.D, a->k_stride_tok, a->k_stride_head, 1, kKeyBlock)) return rc;
  if (int rc = encode_packed_map(&vm, a->v, a->kv_rows, s.KV, s.D, a->v_stride_tok, a->v_stride_head, 1, kKeyBlock)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return s.D == 128 ? launch_row_attention<128, kPacked>(p, qm, tm, km, vm, a->reuse_plan != 0, st)
                    : launch_row_attention<64, kPacked>(p, qm, tm, km, vm, a->reuse_plan != 0, st);
}

extern "C" size_t specdec_shared_prefix_workspace_bytes(int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads,
                                                        int32_t head_dim, int32_t max_q_len, int32_t num_groups,
                                                        int32_t num_members, int32_t num_sms) {
  const RowShape s{num_seqs, num_q_heads, num_kv_heads, head_dim, max_q_len, num_groups, num_members, row_sms(num_sms)};
  return row_shape_ok(s) ? row_space(s).bytes : 0;
}

extern "C" int specdec_shared_prefix_attention(const SpecdecSharedPrefixArgs* a, specdec_stream_t stream) {
  if (!a) return fail(SPECDEC_ERR_INVALID, "args is NULL");
  const SpecdecBatch& bt = a->batch;
  const SpecdecPagedKV& kv = a->kv;
  const RowShape s{bt.num_seqs, bt.num_q_heads, kv.num_kv_heads, kv.head_dim, bt.max_q_len, a->num_groups,
                   a->num_members, row_sms(a->num_sms)};
  if (int rc = check_shape(s)) return rc;
  if (int rc = check_rows(a->q, a->out, a->q_stride_tok, a->q_stride_head, a->o_stride_tok, a->o_stride_head)) return rc;
  if (!bt.q_row0 || !bt.q_len || !bt.ctx_len) return fail(SPECDEC_ERR_INVALID, "batch arrays must be set");
  if (s.G > 0 && (!a->group_start || !a->prefix_len || (s.M > 0 && !a->members)))
    return fail(SPECDEC_ERR_INVALID, "group arrays must be set");
  if (!kv.k_pool || !kv.v_pool || !kv.page_table) return fail(SPECDEC_ERR_INVALID, "kv pool pointers must be set");
  if (kv.num_pages <= 0 || kv.max_pages_per_seq <= 0) return fail(SPECDEC_ERR_INVALID, "empty page pool");
  if ((reinterpret_cast<uintptr_t>(kv.k_pool) | reinterpret_cast<uintptr_t>(kv.v_pool)) & 15u)
    return fail(SPECDEC_ERR_INVALID, "pool pointers must be 16-byte aligned");
  if (kv.v_dtype != SPECDEC_BF16 && kv.v_dtype != SPECDEC_E4M3)
    return fail(SPECDEC_ERR_UNSUPPORTED, "v_dtype must be SPECDEC_BF16 or SPECDEC_E4M3");
  const bool v8 = kv.v_dtype == SPECDEC_E4M3;
  if (v8 && s.D != 128) return fail(SPECDEC_ERR_UNSUPPORTED, "E4M3 V needs head_dim 128 (one scale group per head)");
  if (v8 && !kv.v_scale) return fail(SPECDEC_ERR_INVALID, "E4M3 V needs v_scale");
  if (a->q_rows <= 0 || a->q_rows > 0x7fffffff) return fail(SPECDEC_ERR_INVALID, "row counts out of range");
  const int64_t page_rows = static_cast<int64_t>(kv.num_pages) * s.KV * (s.D / 64);
  if (page_rows > 0x7fffffff || static_cast<int64_t>(kv.max_pages_per_seq) * kPage > (1 << 30))
    return fail(SPECDEC_ERR_UNSUPPORTED, "page pool too large");
  RowParams p = {};
  if (int rc = fill_row_params(p, s, a->workspace, a->workspace_bytes, a->sm_scale)) return rc;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.q_st = a->q_stride_tok;
  p.q_sh = a->q_stride_head;
  p.o_st = a->o_stride_tok;
  p.o_sh = a->o_stride_head;
  p.q_row0 = bt.q_row0;
  p.q_len = bt.q_len;
  p.ctx_len = bt.ctx_len;
  p.group_start = a->group_start;
  p.members = a->members;
  p.prefix_len = a->prefix_len;
  p.page_table = kv.page_table;
  p.num_pages = kv.num_pages;
  p.max_pages = kv.max_pages_per_seq;
  p.paged = 1;
  p.v_scale = kv.v_scale;
  p.v_pool = static_cast<const uint8_t*>(kv.v_pool);
  p.q_rows = a->q_rows;
  p.status = a->status;
  CUtensorMap qm, tm, km, vm;
  if (int rc = encode_packed_map(&qm, a->q, a->q_rows, s.H, s.D, a->q_stride_tok, a->q_stride_head, p.n_rep, p.tpt)) return rc;
  if (int rc = encode_packed_map(&tm, a->q, a->q_rows, s.H, s.D, a->q_stride_tok, a->q_stride_head, p.n_rep, 1)) return rc;
  if (int rc = encode_rows_map(&km, kv.k_pool, static_cast<uint64_t>(page_rows), 2048)) return rc;
  if (int rc = encode_rows_map(&vm, kv.v_pool, static_cast<uint64_t>(v8 ? page_rows / 2 : page_rows), 2048)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (v8) return launch_row_attention<128, kPagedE4M3>(p, qm, tm, km, vm, a->reuse_plan != 0, st);
  return s.D == 128 ? launch_row_attention<128, kPaged>(p, qm, tm, km, vm, a->reuse_plan != 0, st)
                    : launch_row_attention<64, kPaged>(p, qm, tm, km, vm, a->reuse_plan != 0, st);
}
