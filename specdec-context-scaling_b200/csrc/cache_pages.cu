// cache_pages.cu -- pages of a cache between sequences: copy, fork, reserve, free and compact.
//
// A page id names the same slots in every layer.  Who holds a page is counted: refs[page] sequences have it in their
// row of the page table; a page with count 0 is free.  A row holds its pages in its first entries, -1 behind
// them.  New pages are always the lowest free ids, in the order of the request, so the same calls give the same
// tables whatever ran at the same time on the GPU.
//
// What takes an order (which page is free next) is one CTA's work: counts and scans over the tables in L2, a few
// microseconds.  It leaves a list of (from, to) page pairs, and a last kernel moves those pages in all layers: a warp
// takes 2 KB at a time, four 16-byte loads a lane under way before the first store.  Copies are bound by HBM.
#include "sd_common.cuh"
#include "sd_internal.h"

namespace sd {

constexpr int kPoolsPerLaunch = 192;  // K, V and scale pools (64 layers of three) that a launch's parameters hold

struct PagePools {
  uint8_t* base[kPoolsPerLaunch];
  int32_t bytes[3];   // a page of K, V, scales
  int32_t pieces[4];  // first 2 KB piece of each of them in a layer's page, and the number of all
  int32_t kinds;      // 2 or 3 pools a layer
  int32_t layers;
};
constexpr int kPiece = 2048;

// ---------------------------------------------------------------- moving pages
// A warp a (pair, layer, 2 KB piece).  Both pages of a pair lie in the pool, or the pair is left out and reported.
__global__ void __launch_bounds__(256) move_pages_kernel(const __grid_constant__ PagePools pools, const int32_t* src,
                                                         const int32_t* dst, const int32_t* count, int32_t n,
                                                         int32_t num_pages, int32_t* status) {
  grid_dep_wait();
  grid_dep_launch();
  const int pairs = count != nullptr ? min(*count, n) : n;
  const int lane = threadIdx.x & 31, per_page = pools.pieces[3] * pools.layers;
  const int64_t all = static_cast<int64_t>(pairs) * per_page, step = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); u < all; u += step) {
    const int i = static_cast<int>(u / per_page), rest = static_cast<int>(u - static_cast<int64_t>(i) * per_page);
    const int a = src[i], b = dst[i];
    if (a < 0 || a >= num_pages || b < 0 || b >= num_pages) {
      if (lane == 0 && rest == 0) raise_status(status, SPECDEC_STATUS_BAD_PAGE);
      continue;
    }
    if (a == b) continue;
    const int layer = rest / pools.pieces[3], piece = rest - layer * pools.pieces[3];
    const int kind = piece >= pools.pieces[2] ? 2 : piece >= pools.pieces[1] ? 1 : 0;
    const int bytes = pools.bytes[kind], at = (piece - pools.pieces[kind]) * kPiece;
    uint8_t* base = pools.base[layer * pools.kinds + kind] + at;
    const uint4* from = reinterpret_cast<const uint4*>(base + static_cast<int64_t>(a) * bytes);
    uint4* to = reinterpret_cast<uint4*>(base + static_cast<int64_t>(b) * bytes);
    const int words = min(bytes - at, kPiece) / 16;
    uint4 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 32 * e < words) x[e] = from[lane + 32 * e];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 32 * e < words) to[lane + 32 * e] = x[e];
  }
}

// ---------------------------------------------------------------- bookkeeping
struct PageBook {
  int32_t* table;
  int32_t* refs;
  int32_t* lengths;
  int32_t num_seqs, max_pages, num_pages;
  const int32_t* a;  // fork: source sequences; reserve: tokens; free: sequences
  const int32_t* b;  // fork: target sequences
  const int32_t* c;  // fork: tokens
  int32_t n;
  int32_t* n_live;     // compact
  int32_t *from, *to;  // pages to move
  int32_t* count;
  int32_t* scratch;    // [4 * num_seqs + num_pages + 2 * n]
  int32_t* status;
};

constexpr int kBookThreads = 1024;

// Sum of v over the CTA before this thread (exclusive) and in all.
SD_DEV int block_scan(int v, int& total) {
  __shared__ int s_sum[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) s_sum[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = s_sum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    s_sum[lane] = w;
  }
  __syncthreads();
  total = s_sum[31];
  return (warp ? s_sum[warp - 1] : 0) + x - v;
}

// The lowest `want` free pages, ascending, into list; returns how many there are (at most want).
SD_DEV int lowest_free(const PageBook& p, int want, int32_t* list) {
  int have = 0;
  for (int base = 0; base < p.num_pages && have < want; base += kBookThreads) {
    const int page = base + threadIdx.x;
    const int free = page < p.num_pages && p.refs[page] <= 0;
    int total;
    const int at = have + block_scan(free, total);
    if (free && at < want) list[at] = page;
    have += total;
  }
  __syncthreads();
  return min(have, want);
}

SD_DEV bool page_ok(const PageBook& p, int page) { return page >= 0 && page < p.num_pages; }

// Row s of the table gives up its pages.
SD_DEV void drop_row(const PageBook& p, int s, int lane) {
  int32_t* row = p.table + static_cast<int64_t>(s) * p.max_pages;
  for (int base = lane; base < p.max_pages; base += 8 * 32) {
    int page[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) page[e] = base + 32 * e < p.max_pages ? row[base + 32 * e] : -1;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (page_ok(p, page[e])) atomicSub(&p.refs[page[e]], 1);
      if (base + 32 * e < p.max_pages) row[base + 32 * e] = -1;
    }
  }
}

// Fork: target d = b[i] gives up its pages, takes over the full pages of source s = a[i]'s first c[i] tokens, and
// gets a page of its own for the started one.  A CTA a request does all but the last, taking eight entries a thread at
// a time; fork_pages_kernel then hands out the started ones' pages, in the order of the requests.
constexpr int kForkThreads = 256;
__global__ void __launch_bounds__(kForkThreads) fork_kernel(const PageBook p) {
  grid_dep_wait();
  grid_dep_launch();
  const int i = blockIdx.x, tid = threadIdx.x;
  const int s = p.a[i], d = p.b[i], len = p.c[i];
  auto in_range = [&](int x) { return x >= 0 && x < p.num_seqs; };
  const bool fine = in_range(s) && in_range(d) && s != d;
  // What is forked from stays as it is while others read it: a request whose source is another's target is left out (that
  // other one runs), and so is one whose target was listed before.  So nobody reads a row that this block writes.
  int bad = !fine || len < 0 || len > p.max_pages * kPage;
  if (!bad) bad = len > p.lengths[s];
  for (int k = tid; k < p.n && fine; k += kForkThreads) {
    const int ks = p.a[k], kd = p.b[k];
    const bool other = in_range(ks) && in_range(kd) && ks != kd;
    bad |= other && ((kd == d && k < i) || kd == s);
  }
  bad = __syncthreads_or(bad);
  const int32_t* from = p.table + static_cast<int64_t>(fine ? s : 0) * p.max_pages;
  const int need = (len + kPage - 1) / kPage, full = len / kPage;
  int lost = 0;
  for (int j = tid; !bad && j < need; j += kForkThreads) lost |= !page_ok(p, from[j]);
  lost = __syncthreads_or(lost);
  if (tid == 0) {
    p.scratch[i] = !bad && !lost;
    if (bad) raise_status(p.status, SPECDEC_STATUS_BAD_SEQUENCE);
    if (lost) raise_status(p.status, SPECDEC_STATUS_BAD_PAGE);
  }
  if (bad || lost) return;
  int32_t* to = p.table + static_cast<int64_t>(d) * p.max_pages;
  for (int base = tid; base < p.max_pages; base += 8 * kForkThreads) {
    int old[8], now[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = base + e * kForkThreads;
      old[e] = j < p.max_pages ? to[j] : -1;
      now[e] = j < full ? from[j] : -1;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = base + e * kForkThreads;
      if (page_ok(p, old[e])) atomicSub(&p.refs[old[e]], 1);
      if (now[e] >= 0) atomicAdd(&p.refs[now[e]], 1);
      if (j < p.max_pages) to[j] = now[e];
    }
  }
  if (tid == 0) p.lengths[d] = len;
}

__global__ void __launch_bounds__(kBookThreads) fork_pages_kernel(const PageBook p) {
  grid_dep_wait();
  grid_dep_launch();
  const int32_t* ok = p.scratch;
  int32_t* fresh = p.scratch + p.n;  // [n] free pages
  int want = 0;
  for (int base = 0; base < p.n; base += kBookThreads) {
    const int i = base + threadIdx.x;
    int total;
    (void)block_scan(i < p.n && ok[i] && p.c[i] % kPage != 0, total);
    want += total;
  }
  const int have = lowest_free(p, want, fresh);
  int seen = 0;
  for (int base = 0; base < p.n; base += kBookThreads) {
    const int i = base + threadIdx.x;
    const bool started = i < p.n && ok[i] && p.c[i] % kPage != 0;
    int total;
    const int at = seen + block_scan(started, total);
    if (started) {
      const int j = p.c[i] / kPage;
      if (at < have) {
        p.table[static_cast<int64_t>(p.b[i]) * p.max_pages + j] = fresh[at];
        p.refs[fresh[at]] = 1;
        p.from[at] = p.table[static_cast<int64_t>(p.a[i]) * p.max_pages + j];
        p.to[at] = fresh[at];
      } else {  // no page left: the target keeps the full pages only
        p.lengths[p.b[i]] = j * kPage;
        raise_status(p.status, SPECDEC_STATUS_NO_PAGES);
      }
    }
    seen += total;
  }
  if (threadIdx.x == 0) *p.count = have;
}

// Reserve: row s gets pages for a[s] tokens.  Pages that it goes on writing into (from its length on) and that others
// hold, too, are replaced by new ones, the started page's contents being copied.  (Counts are those before the call, so
// that no row's answer depends on another's place: a page that only writers hold is replaced for all of them.)  Requests are met in the order of
// the sequences until the pages run out; one that cannot be met is left as it was, and so is everyone's after it.
__global__ void __launch_bounds__(kBookThreads) reserve_kernel(const PageBook p) {
  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int32_t* held = p.scratch;            // [num_seqs] entries in use
  int32_t* swaps = held + p.num_seqs;   // [num_seqs] held pages to be replaced, from entry length / 16 on
  int32_t* start = swaps + p.num_seqs;  // [num_seqs] place of its first new page, or -1
  int32_t* copy = start + p.num_seqs;   // [num_seqs] the first of them has contents to keep
  int32_t* left = copy + p.num_seqs;    // [num_pages] page given up for the new page at the same place, or -1
  int32_t* fresh = p.to;
  auto end_of = [&](int s) { return min(held[s], (p.a[s] + kPage - 1) / kPage); };
  for (int s = warp; s < p.num_seqs; s += kBookThreads / 32) {
    const int32_t* row = p.table + static_cast<int64_t>(s) * p.max_pages;
    int have = 0;
    for (int base = 0; base < p.max_pages; base += 32) {
      const bool in = base + lane < p.max_pages && row[base + lane] >= 0;
      const int k = __popc(__ballot_sync(0xffffffffu, in));
      have += k;
      if (k < 32) break;
    }
    const int want = p.a[s], len = p.lengths[s];
    const bool fine = want >= 0 && want <= p.max_pages * kPage && len >= 0;
    int shared = 0;
    if (fine && want > len) {
      const int end = min(have, (want + kPage - 1) / kPage);
      for (int j = len / kPage + lane; j < end; j += 32) shared += page_ok(p, row[j]) && p.refs[row[j]] > 1;
      shared = __reduce_add_sync(0xffffffffu, shared);
    }
    if (lane == 0) {
      if (!fine) raise_status(p.status, SPECDEC_STATUS_PAGE_OVERFLOW);
      held[s] = have;
      swaps[s] = shared;
      start[s] = fine ? max((want + kPage - 1) / kPage - have, 0) : 0;
      copy[s] = 0;
    }
  }
  __syncthreads();
  int asked = 0;
  for (int base = 0; base < p.num_seqs; base += kBookThreads) {
    const int s = base + threadIdx.x;
    const int k = s < p.num_seqs ? min(start[s] + swaps[s], p.num_pages + 1) : 0;
    int total;
    const int at = min(asked + block_scan(k, total), 0x3fffffff);
    if (s < p.num_seqs) {
      start[s] = k == 0 ? -1 : at;
      copy[s] = k;
    }
    asked = min(asked + total, 0x3fffffff);
  }
  __syncthreads();
  const int have = lowest_free(p, min(asked, p.num_pages), fresh);
  for (int i = threadIdx.x; i < have; i += kBookThreads) left[i] = -1;
  __syncthreads();
  for (int s = warp; s < p.num_seqs; s += kBookThreads / 32) {
    const int at = start[s], k = copy[s];
    __syncwarp();
    if (at < 0 || at + k > have) {
      if (lane == 0) {
        if (at >= 0) raise_status(p.status, SPECDEC_STATUS_NO_PAGES);
        copy[s] = 0;
      }
      continue;
    }
    int32_t* row = p.table + static_cast<int64_t>(s) * p.max_pages;
    const int len = p.lengths[s], more = k - swaps[s];
    int done = 0;  // replaced so far
    bool keeps = false;
    for (int base = len / kPage; done < swaps[s] && base < end_of(s); base += 32) {
      const int j = base + lane;
      const int page = j < end_of(s) ? row[j] : -1;
      // counts of held pages do not change before every row has looked
      const bool swap = page_ok(p, page) && p.refs[page] > 1;
      const uint32_t who = __ballot_sync(0xffffffffu, swap);
      if (swap) {
        const int f = at + done + __popc(who & ((1u << lane) - 1));
        left[f] = page;
        row[j] = fresh[f];
        p.refs[fresh[f]] = 1;
      }
      if (base == len / kPage) keeps = (who & 1u) && len % kPage != 0;
      done += __popc(who);
    }
    for (int j = lane; j < more; j += 32) {
      const int page = fresh[at + swaps[s] + j];
      row[held[s] + j] = page;
      p.refs[page] = 1;
    }
    __syncwarp();
    if (lane == 0) copy[s] = keeps;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < have; i += kBookThreads)
    if (left[i] >= 0) atomicSub(&p.refs[left[i]], 1);
  // (old, new) pairs of the started pages, in the order of the rows
  int copies = 0;
  for (int base = 0; base < p.num_seqs; base += kBookThreads) {
    const int s = base + threadIdx.x;
    const bool c = s < p.num_seqs && copy[s] != 0;
    int total;
    const int at = copies + block_scan(c, total);
    if (c) {
      p.from[at] = left[start[s]];
      held[at] = fresh[start[s]];  // entries before s are done with: at <= s
    }
    copies += total;
    __syncthreads();
  }
  for (int i = threadIdx.x; i < copies; i += kBookThreads) p.to[i] = held[i];
  if (threadIdx.x == 0) *p.count = copies;
}

// Free: the sequences' rows give up their pages, their lengths become 0.
__global__ void __launch_bounds__(kBookThreads) free_kernel(const PageBook p) {
  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int32_t* mark = p.scratch;  // [num_seqs] the first request that names the sequence
  for (int s = threadIdx.x; s < p.num_seqs; s += kBookThreads) mark[s] = 0x7fffffff;
  __syncthreads();
  for (int i = threadIdx.x; i < p.n; i += kBookThreads) {
    const int s = p.a[i];
    if (s < 0 || s >= p.num_seqs)
      raise_status(p.status, SPECDEC_STATUS_BAD_SEQUENCE);
    else
      atomicMin(&mark[s], i);
  }
  __syncthreads();
  for (int i = warp; i < p.n; i += kBookThreads / 32) {
    const int s = p.a[i];
    if (s < 0 || s >= p.num_seqs || mark[s] != i) continue;  // named twice: once is enough
    drop_row(p, s, lane);
    if (lane == 0) p.lengths[s] = 0;
  }
}

// Compact: live pages at or past the number of live pages move to the free ids below it, both ascending.
__global__ void __launch_bounds__(kBookThreads) compact_kernel(const PageBook p) {
  grid_dep_wait();
  grid_dep_launch();
  int32_t* place = p.scratch;  // [num_pages] where a page goes
  int live = 0;
  for (int base = 0; base < p.num_pages; base += kBookThreads) {
    const int page = base + threadIdx.x;
    int total;
    (void)block_scan(page < p.num_pages && p.refs[page] > 0, total);
    live += total;
    if (page < p.num_pages) place[page] = page;
  }
  int holes = 0, moves = 0;
  for (int base = 0; base < p.num_pages; base += kBookThreads) {
    const int page = base + threadIdx.x;
    const bool hole = page < live && p.refs[page] <= 0;
    const bool move = page >= live && page < p.num_pages && p.refs[page] > 0;
    int total;
    const int h = holes + block_scan(hole, total);
    holes += total;
    const int m = moves + block_scan(move, total);
    moves += total;
    if (hole) p.to[h] = page;
    if (move) p.from[m] = page;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moves; i += kBookThreads) {
    place[p.from[i]] = p.to[i];
    p.refs[p.to[i]] = p.refs[p.from[i]];
    p.refs[p.from[i]] = 0;
  }
  __syncthreads();
  const int64_t entries = static_cast<int64_t>(p.num_seqs) * p.max_pages;
  for (int64_t e = threadIdx.x; e < entries; e += kBookThreads) {
    const int page = p.table[e];
    if (page_ok(p, page) && place[page] != page) p.table[e] = place[page];
  }
  if (threadIdx.x == 0) {
    *p.count = moves;
    *p.n_live = live;
  }
}

// ---------------------------------------------------------------- host side
static int check_pool(const SpecdecPagePool* a) {
  if (!a) return fail(SPECDEC_ERR_INVALID, "pool is NULL");
  if (a->num_layers <= 0 || a->num_pages <= 0 || a->num_kv_heads <= 0)
    return fail(SPECDEC_ERR_INVALID, "empty page pool");
  if (a->head_dim != 64 && a->head_dim != 128) return fail(SPECDEC_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (a->v_dtype != SPECDEC_BF16 && a->v_dtype != SPECDEC_E4M3)
    return fail(SPECDEC_ERR_UNSUPPORTED, "v_dtype must be SPECDEC_BF16 or SPECDEC_E4M3");
  if (!a->k_pools || !a->v_pools || (a->v_dtype == SPECDEC_E4M3 && !a->v_scales))
    return fail(SPECDEC_ERR_INVALID, "kv pool pointers must be set");
  if (a->num_kv_heads > (1 << 14)) return fail(SPECDEC_ERR_UNSUPPORTED, "at most 16384 KV heads");
  for (int l = 0; l < a->num_layers; ++l) {
    const void* v = a->v_dtype == SPECDEC_E4M3 ? a->v_scales[l] : a->v_pools[l];
    if (!a->k_pools[l] || !a->v_pools[l] || !v) return fail(SPECDEC_ERR_INVALID, "kv pool pointers must be set");
    if ((reinterpret_cast<uintptr_t>(a->k_pools[l]) | reinterpret_cast<uintptr_t>(a->v_pools[l]) |
         reinterpret_cast<uintptr_t>(v)) & 15u)
      return fail(SPECDEC_ERR_INVALID, "pool pointers must be 16-byte aligned");
  }
  return SPECDEC_OK;
}

static int move_pages(const SpecdecPagePool* a, const int32_t* src, const int32_t* dst, const int32_t* count, int32_t n,
                      int32_t* status, cudaStream_t st) {
  const bool v8 = a->v_dtype == SPECDEC_E4M3;
  PagePools pp;
  pp.kinds = v8 ? 3 : 2;
  const int k_bytes = a->num_kv_heads * kPage * a->head_dim * 2;
  pp.bytes[0] = k_bytes;
  pp.bytes[1] = v8 ? k_bytes / 2 : k_bytes;
  pp.bytes[2] = v8 ? a->num_kv_heads * kPage * 4 : 0;
  pp.pieces[0] = 0;
  for (int k = 0; k < 3; ++k) pp.pieces[k + 1] = pp.pieces[k] + (pp.bytes[k] + kPiece - 1) / kPiece;
  const int layers_a_launch = kPoolsPerLaunch / 3;
  for (int l0 = 0; l0 < a->num_layers; l0 += layers_a_launch) {
    pp.layers = a->num_layers - l0 < layers_a_launch ? a->num_layers - l0 : layers_a_launch;
    for (int l = 0; l < pp.layers; ++l) {
      pp.base[l * pp.kinds] = static_cast<uint8_t*>(a->k_pools[l0 + l]);
      pp.base[l * pp.kinds + 1] = static_cast<uint8_t*>(a->v_pools[l0 + l]);
      if (v8) pp.base[l * pp.kinds + 2] = reinterpret_cast<uint8_t*>(a->v_scales[l0 + l]);
    }
    // every warp of the device a piece, and up to four more in turn
    const int64_t blocks = (static_cast<int64_t>(n) * pp.layers * pp.pieces[3] + 7) / 8;
    const int64_t most = static_cast<int64_t>(device_sm_count()) * 8 * 4;
    if (int rc = launch_pdl("move_pages_kernel", move_pages_kernel, dim3(static_cast<unsigned>(blocks < most ? blocks : most)),
                            dim3(256), 0, st, pp, src, dst, count, n, a->num_pages, status))
      return rc;
  }
  return SPECDEC_OK;
}

static int64_t book_words(int64_t num_seqs, int64_t num_pages, int64_t n) {
  return 4 * num_seqs + num_pages + 2 * n + 2 * num_pages + 64;
}

static int check_book(const SpecdecPageTable* t, const SpecdecPagePool* a, int64_t n, PageBook& p) {
  if (!t) return fail(SPECDEC_ERR_INVALID, "table is NULL");
  if (!t->page_table || !t->page_refs || !t->lengths)
    return fail(SPECDEC_ERR_INVALID, "page_table, page_refs and lengths must be device pointers");
  if (t->num_seqs <= 0 || t->max_pages_per_seq <= 0 || t->max_pages_per_seq > (1 << 26))
    return fail(SPECDEC_ERR_INVALID, "bad page table shape");
  const size_t need = static_cast<size_t>(book_words(t->num_seqs, a->num_pages, n)) * 4;
  if (!t->workspace || t->workspace_bytes < need)
    return fail(SPECDEC_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", t->workspace ? t->workspace_bytes : 0, need);
  if (reinterpret_cast<uintptr_t>(t->workspace) & 15u) return fail(SPECDEC_ERR_INVALID, "workspace must be 16-byte aligned");
  p = PageBook{};
  p.table = t->page_table;
  p.refs = t->page_refs;
  p.lengths = t->lengths;
  p.num_seqs = t->num_seqs;
  p.max_pages = t->max_pages_per_seq;
  p.num_pages = a->num_pages;
  p.n = static_cast<int32_t>(n);
  p.status = t->status;
  int32_t* w = static_cast<int32_t*>(t->workspace);
  p.count = w;
  p.from = w + 32;
  p.to = p.from + a->num_pages;
  p.scratch = p.to + a->num_pages;
  return SPECDEC_OK;
}

}  // namespace sd

using namespace sd;

extern "C" int specdec_copy_pages(const SpecdecPagePool* pool, const int32_t* src, const int32_t* dst, int32_t n,
                                  int32_t* status, specdec_stream_t stream) {
  if (int rc = check_pool(pool)) return rc;
  if (n < 0) return fail(SPECDEC_ERR_INVALID, "page count out of range");
  if (n == 0) return SPECDEC_OK;
  if (!src || !dst) return fail(SPECDEC_ERR_INVALID, "src and dst must be device pointers");
  return move_pages(pool, src, dst, nullptr, n, status, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t specdec_page_workspace_bytes(int32_t num_seqs, int32_t num_pages, int32_t n) {
  if (num_seqs <= 0 || num_pages <= 0 || n < 0) return 0;
  return static_cast<size_t>(book_words(num_seqs, num_pages, n)) * 4;
}

extern "C" int specdec_fork_sequences(const SpecdecPagePool* pool, const SpecdecPageTable* table, const int32_t* src,
                                      const int32_t* dst, const int32_t* length, int32_t n, specdec_stream_t stream) {
  if (int rc = check_pool(pool)) return rc;
  if (n < 0) return fail(SPECDEC_ERR_INVALID, "sequence count out of range");
  PageBook p;
  if (int rc = check_book(table, pool, n, p)) return rc;
  if (n == 0) return SPECDEC_OK;
  if (!src || !dst || !length) return fail(SPECDEC_ERR_INVALID, "src, dst and length must be device pointers");
  p.a = src;
  p.b = dst;
  p.c = length;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (int rc = launch_pdl("fork_kernel", fork_kernel, dim3(n), dim3(kForkThreads), 0, st, p)) return rc;
  if (int rc = launch_pdl("fork_pages_kernel", fork_pages_kernel, dim3(1), dim3(kBookThreads), 0, st, p)) return rc;
  const int most = n < pool->num_pages ? n : pool->num_pages;
  return move_pages(pool, p.from, p.to, p.count, most, p.status, st);
}

extern "C" int specdec_reserve_pages(const SpecdecPagePool* pool, const SpecdecPageTable* table, const int32_t* tokens,
                                     specdec_stream_t stream) {
  if (int rc = check_pool(pool)) return rc;
  PageBook p;
  if (int rc = check_book(table, pool, 0, p)) return rc;
  if (!tokens) return fail(SPECDEC_ERR_INVALID, "tokens must be a device pointer");
  p.a = tokens;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (int rc = launch_pdl("reserve_kernel", reserve_kernel, dim3(1), dim3(kBookThreads), 0, st, p)) return rc;
  const int most = p.num_seqs < pool->num_pages ? p.num_seqs : pool->num_pages;
  return move_pages(pool, p.from, p.to, p.count, most, p.status, st);
}

extern "C" int specdec_free_sequences(const SpecdecPagePool* pool, const SpecdecPageTable* table, const int32_t* seqs,
                                      int32_t n, specdec_stream_t stream) {
  if (int rc = check_pool(pool)) return rc;
  if (n < 0) return fail(SPECDEC_ERR_INVALID, "sequence count out of range");
  PageBook p;
  if (int rc = check_book(table, pool, n, p)) return rc;
  if (n == 0) return SPECDEC_OK;
  if (!seqs) return fail(SPECDEC_ERR_INVALID, "seqs must be a device pointer");
  p.a = seqs;
  return launch_pdl("free_kernel", free_kernel, dim3(1), dim3(kBookThreads), 0, reinterpret_cast<cudaStream_t>(stream), p);
}

extern "C" int specdec_compact_pages(const SpecdecPagePool* pool, const SpecdecPageTable* table, int32_t* n_live,
                                     specdec_stream_t stream) {
  if (int rc = check_pool(pool)) return rc;
  PageBook p;
  if (int rc = check_book(table, pool, 0, p)) return rc;
  if (!n_live) return fail(SPECDEC_ERR_INVALID, "n_live must be a device pointer");
  p.n_live = n_live;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (int rc = launch_pdl("compact_kernel", compact_kernel, dim3(1), dim3(kBookThreads), 0, st, p)) return rc;
  const int most = (pool->num_pages + 1) / 2;
  return move_pages(pool, p.from, p.to, p.count, most, p.status, st);
}
