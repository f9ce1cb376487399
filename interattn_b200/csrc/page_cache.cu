// The pages of a K/V cache that sequences share: extend (hand out pages), write (keys and values of new tokens), fork,
// free, compact.  The state is three int32 arrays on the device: the table rows, the sequence lengths, and per page the
// number of table entries that hold it; a page is free when its count is zero.
//
// There is no free list: a page is handed out by its rank among the free ones, lowest first, so the result depends on the
// counts alone and not on the order in which threads or earlier calls ran.  Ranks are prefix sums over the counts, taken in
// one launch: by one CTA where list and pool are short, a chain of barriers and round trips to memory either way, and by a
// cluster of eight where they are long (8192 threads, the cluster's hardware barrier between the phases, the CTAs' totals
// through distributed shared memory).  Whatever moves data (the copies, the table rows of a fork, the remapped entries)
// follows in a second launch on the whole GPU and reads what to do from the scratch that the first left.
//
// A warp looks at 128 consecutive counts at a time, so they are read once and in order, and pages are granted in two steps, free
// page to rank and rank to list entry, so that they spread over all threads wherever in the pool they lie (with a run of pages
// per thread, 256 rows' pages out of 65536 took 153 us instead of 17).
//
// A write goes to the end of whatever its row holds, so it has to know when that is not where its tokens belong: the scratch keeps
// for every row whether its last extend was refused, and how many of its tokens lie in pages that a fork shared (see Guard).
//
// Measured: moving 1.14 GB of pages 182 us (0.97 of the copy peak), a plan over 16,384 pages 9 us, 64 forks of 8k tokens 15 us with
// the free before them; the plan is a chain of dependent loads and barriers.
#include <algorithm>

#include "dense_attention.cuh"
#include "page_cache.cuh"

namespace ia {
namespace {

constexpr int kPage = 16;
constexpr int kPlanCtas = 8, kPlanThreads = 1024;  // of the large plan; the small one is one CTA
// One CTA needs no cluster barrier, eight read the counts faster.  Handing out 4 pages to 4 / 256 rows and taking them back, one
// CTA and eight, us: 1024 pages 8.0 / 12.1 and 14.0 / 16.2, 32768 pages 12.6 / 17.6 and 14.7 / 16.4, 65536 pages 17.2 / 21.7 and
// 14.2 / 16.6, 262144 pages 46 / 50 and 19 / 20.  The compaction's plan with few pages to move: 4096 pages 6.1 and 8.7, 16384
// pages 9.0 and 9.0, 32768 pages 12.7 and 8.8.  A list is short while a thread can hold its row against all before it.
constexpr int kSmallList = 256, kSmallPool = 32768, kSmallCompact = 16384;
constexpr int kMoveThreads = 256;

// What a write to the row may not touch; all zero at first.
struct Guard {
  int shared;   // the row's first tokens, whole pages, that a fork shared: not while another count holds the page
  int refused;  // the row's last extend that asked for tokens was refused: nothing
};
// scratch: counters, then per entry of a list the inclusive sum of the pages wanted and what was granted, then the moves; the rows'
// guards, which outlive a call
struct Scratch {
  int* n_moves;      // [4]: moves, live pages, unused
  int* owner;        // [n_rows] first entry of the list that names the row
  int* upto;         // [n_entries] inclusive sums
  int* kept;         // [n_entries] pages of the row before, or taken over from the parent; -1: the entry was refused, -2: it names
                     // no row, or one that an entry before it names
  int* new_len;      // [n_entries]
  int2* moves;       // [n_pages] (from, to)
  int* remap;        // [n_pages]
  Guard* guard;      // [n_rows]
};
int64_t scratch_layout(char* base, int64_t n_rows, int64_t n_pages, Scratch* s) {
  int64_t off = 0;
  auto take = [&](int64_t bytes) {
    char* r = base ? base + off : nullptr;
    off += (bytes + 255) / 256 * 256;
    return r;
  };
  char* a[8] = {take(16),         take(n_rows * 4),  take(n_rows * 4),  take(n_rows * 4),
                take(n_rows * 4), take(n_pages * 8), take(n_pages * 4), take(n_rows * 8)};  // no list is longer than the table
  if (s) *s = Scratch{(int*)a[0], (int*)a[1], (int*)a[2], (int*)a[3], (int*)a[4], (int2*)a[5], (int*)a[6], (Guard*)a[7]};
  return off;
}

struct State {
  int* table;   // [n_rows, max_pages]
  int* lens;    // [n_rows]
  int* refs;    // [n_pages]
  int* status;
  int n_rows, max_pages, n_pages;
};
__device__ __forceinline__ int pages_of(int len) { return (len + kPage - 1) / kPage; }
__device__ __forceinline__ int len_of(const State& st, int row) {
  return max(0, min(st.lens[row], st.max_pages * kPage));
}
__device__ __forceinline__ void report(const State& st, int bits) { atomicOr(st.status, bits); }

// ---- prefix sums over the whole cluster -----------------------------------------------------------------------------
template <int CTAS> __device__ __forceinline__ void sync_all() {
  if constexpr (CTAS == 1) __syncthreads();
  else asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int CTAS> __device__ __forceinline__ int cta_rank() { return CTAS == 1 ? 0 : (int)blockIdx.x; }
__device__ __forceinline__ int peer_word(const int* smem, int rank) {
  uint32_t addr = (uint32_t)__cvta_generic_to_shared(smem), remote;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
  return v;
}
struct Sums { int before, total; };
// exclusive sum of v over all threads in order of (CTA, thread), and the sum of all
template <int CTAS> __device__ Sums scan(int v, int* warp_sums, int* cta_sum) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int upto = v;
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, w);
    if (lane >= w) upto += x;
  }
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, s, w);
      if (lane >= w) s += x;
    }
    warp_sums[lane] = s;
    if (lane == 31) *cta_sum = s;
  }
  __syncthreads();
  int before = upto - v + (warp > 0 ? warp_sums[warp - 1] : 0), total = 0;
  if constexpr (CTAS == 1) {
    total = *cta_sum;
  } else {
    sync_all<CTAS>();  // every CTA's sum is there
#pragma unroll
    for (int c = 0; c < CTAS; ++c) {
      const int x = peer_word(cta_sum, c);
      if (c < cta_rank<CTAS>()) before += x;
      total += x;
    }
  }
  sync_all<CTAS>();  // and has been read by all: the words may be used again
  return {before, total};
}

// A warp takes a run of consecutive pages, 128 at a time, a lane four of them: run w of all is [p0, p1).
struct Run { int p0, p1; };
template <int CTAS> __device__ __forceinline__ Run run_of(int n_pages) {
  constexpr int kWarps = CTAS * kPlanThreads / 32;
  const int per = ((n_pages + kWarps - 1) / kWarps + 127) & ~127, w = cta_rank<CTAS>() * (kPlanThreads / 32) + (threadIdx.x >> 5);
  const int64_t p0 = (int64_t)w * per;
  return {(int)min((int64_t)n_pages, p0), (int)min((int64_t)n_pages, p0 + per)};
}
// bit c: page at + c is in use
__device__ __forceinline__ int used_bits(const int* refs, int at, int end) {
  if (at + 4 <= end && (reinterpret_cast<uintptr_t>(refs) & 15) == 0) {
    const int4 r = *reinterpret_cast<const int4*>(refs + at);
    return (r.x != 0) | (r.y != 0) << 1 | (r.z != 0) << 2 | (r.w != 0) << 3;
  }
  int bits = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (at + c < end && refs[at + c] != 0) bits |= 1 << c;
  return bits;
}
// bit c: page at + c exists before `end`
__device__ __forceinline__ int page_bits(int at, int end) { return (1 << max(0, min(4, end - at))) - 1; }
__device__ __forceinline__ int count_used(const int* refs, Run run) {  // the lane's share
  int n = 0;
#pragma unroll 4
  for (int g = run.p0 + (threadIdx.x & 31) * 4; g < run.p1; g += 128) n += __popc(used_bits(refs, g, run.p1));
  return n;
}
// of the lane's up to four bits: how many set bits lie before them in the warp, and how many there are
__device__ __forceinline__ int2 rank_bits(int bits) {
  const unsigned below = (1u << (threadIdx.x & 31)) - 1;
  int2 r = {0, 0};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const unsigned m = __ballot_sync(0xffffffffu, bits >> c & 1);
    r.x += __popc(m & below);
    r.y += __popc(m);
  }
  return r;
}

// ---- who gets which page --------------------------------------------------------------------------------------------
struct PlanParams {
  State st;
  Scratch sc;
  const int* rows;   // extend: the rows; fork: the children
  const int* other;  // extend: tokens to add; fork: the parents
  int n;
  int fork, share;
};

template <int CTAS> __global__ void __launch_bounds__(kPlanThreads) pages_plan_kernel(const PlanParams p) {
  __shared__ int warp_sums[32];
  __shared__ int cta_sum;
  __shared__ __align__(16) int named[CTAS == 1 ? kSmallList : 4];  // the rows, then the sums
  constexpr int kAll = CTAS * kPlanThreads;
  const State& st = p.st;
  const int me = cta_rank<CTAS>() * kPlanThreads + threadIdx.x;
  const int per = (p.n + kAll - 1) / kAll, i0 = min(p.n, me * per), i1 = min(p.n, i0 + per);
  if constexpr (CTAS > 1) sync_all<CTAS>();  // the whole cluster runs before anyone reads a peer's shared memory
  grid_dependency_wait();
  if (p.fork) grid_launch_dependents();  // the copies follow; what follows an extend is not known here
  const Run run = run_of<CTAS>(st.n_pages);
  int n_free = -count_used(st.refs, run);
  if ((threadIdx.x & 31) == 0) n_free += run.p1 - run.p0;  // the lanes' sum is what counts
  // a row that the list names twice belongs to its first entry
  bool again = false;
  if constexpr (CTAS == 1) {
    if (me < kSmallList) named[me] = me < p.n ? p.rows[me] : 0;
    __syncthreads();
    if (me < p.n) {
      const int mine = named[me];
#pragma unroll 4
      for (int i = 0; i < (me | 31); i += 4) {
        const int4 x = *reinterpret_cast<const int4*>(named + i);
        again |= (i < me && x.x == mine) || (i + 1 < me && x.y == mine) || (i + 2 < me && x.z == mine) || (i + 3 < me && x.w == mine);
      }
    }
  } else {
    for (int i = i0; i < i1; ++i)
      if ((unsigned)p.rows[i] < (unsigned)st.n_rows) p.sc.owner[p.rows[i]] = 0x7fffffff;
    __threadfence();
    sync_all<CTAS>();
    for (int i = i0; i < i1; ++i)
      if ((unsigned)p.rows[i] < (unsigned)st.n_rows) atomicMin(p.sc.owner + p.rows[i], i);
    __threadfence();
    sync_all<CTAS>();
  }
  int wanted = 0, row = 0, other = 0, kept = 0;  // of the thread's entry, if it has one only
  for (int i = i0; i < i1; ++i) {
    row = p.rows[i];
    other = p.other[i];
    kept = -2;
    int need = 0;
    if constexpr (CTAS > 1)
      if ((unsigned)row < (unsigned)st.n_rows) again = __ldcg(p.sc.owner + row) != i;
    if ((unsigned)row < (unsigned)st.n_rows && !again) {
      const int len = len_of(st, row);
      kept = -1;
      if (p.fork) {
        if ((unsigned)other < (unsigned)st.n_rows && other != row && len == 0) {
          const int parent = len_of(st, other);
          kept = p.share ? parent / kPage : 0;
          need = pages_of(parent) - kept;
          p.sc.new_len[i] = parent;
        }
      } else if (other >= 0 && other <= st.max_pages * kPage - len) {
        kept = pages_of(len);
        need = pages_of(len + other) - kept;
        p.sc.new_len[i] = len + other;
      }
    }
    if (kept < 0) report(st, DEV_STATUS_BAD_INDEX);
    p.sc.kept[i] = kept;
    wanted += need;
    p.sc.upto[i] = need;
  }
  const Sums want = scan<CTAS>(wanted, warp_sums, &cta_sum);
  const Sums free_pages = scan<CTAS>(n_free, warp_sums, &cta_sum);
  // from the first entry on that does not fit, none is served
  int upto = want.before, granted = 0;
  for (int i = i0; i < i1; ++i) {
    const int need = p.sc.upto[i];
    upto += need;
    const bool fits = upto <= free_pages.total;
    p.sc.upto[i] = upto;
    if constexpr (CTAS == 1) named[i] = upto;
    if (per > 1) kept = p.sc.kept[i];
    if (!fits && kept >= 0) {
      p.sc.kept[i] = kept = -1;
      report(st, IA_DEV_STATUS_NO_PAGES);
    }
    if (fits) granted += need;
  }
  __threadfence();
  const Sums grants = scan<CTAS>(granted, warp_sums, &cta_sum);  // also: the sums above are visible to all
  // new lengths; all lengths were read before the barriers above
  for (int i = i0; i < i1; ++i)
    if (p.sc.kept[i] >= 0) st.lens[p.rows[i]] = p.sc.new_len[i];
  // the free page of rank r ...
  int rank = __shfl_sync(0xffffffffu, free_pages.before, 0);
  for (int g = run.p0; g < run.p1 && rank < grants.total; g += 128) {
    const int at = g + (threadIdx.x & 31) * 4, bits = page_bits(at, run.p1) & ~used_bits(st.refs, at, run.p1);
    const int2 r = rank_bits(bits);
    int k = rank + r.x;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (!(bits >> c & 1)) continue;
      if (k < grants.total) {
        p.sc.moves[k].y = at + c;
        st.refs[at + c] = 1;
      }
      ++k;
    }
    rank += r.y;
  }
  __threadfence();
  sync_all<CTAS>();
  // ... goes to the first entry whose sum is above r
  for (int r = me; r < grants.total; r += kAll) {
    const int page = __ldcg(&p.sc.moves[r].y);
    int lo = 0, hi = p.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((CTAS == 1 ? named[mid] : __ldcg(p.sc.upto + mid)) > r) hi = mid;
      else lo = mid + 1;
    }
    const int before = lo > 0 ? (CTAS == 1 ? named[lo - 1] : __ldcg(p.sc.upto + lo - 1)) : 0;
    const int at = __ldcg(p.sc.kept + lo) + r - before;
    st.table[(int64_t)p.rows[lo] * st.max_pages + at] = page;
    if (p.fork) p.sc.moves[r].x = st.table[(int64_t)p.other[lo] * st.max_pages + at];
  }
  if (me == 0) p.sc.n_moves[0] = p.fork ? grants.total : 0;
  for (int i = i0; i < i1; ++i) {  // here no barrier waits for these stores
    if (per > 1) {
      row = p.rows[i];
      other = p.other[i];
      kept = p.sc.kept[i];
    }
    if (!p.fork) {
      if (kept >= -1 && other != 0) p.sc.guard[row].refused = kept < 0;
    } else if (kept >= 0) {  // a parent of whole pages is no child, and all its entries say the same
      const int shared = p.share ? kept * kPage : 0;
      p.sc.guard[row] = Guard{shared, 0};
      if (shared > 0) p.sc.guard[other].shared = shared;
    }
  }
}

// Live pages at or past the number of live pages move into the holes below it, in order.
struct CompactParams { State st; Scratch sc; };
template <int CTAS> __global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(const CompactParams p) {
  __shared__ int warp_sums[32];
  __shared__ int cta_sum;
  const State& st = p.st;
  const Scratch& sc = p.sc;
  const int me = cta_rank<CTAS>() * kPlanThreads + threadIdx.x;
  if constexpr (CTAS > 1) sync_all<CTAS>();
  grid_dependency_wait();
  grid_launch_dependents();
  const Run run = run_of<CTAS>(st.n_pages);
  const Sums all = scan<CTAS>(count_used(st.refs, run), warp_sums, &cta_sum);
  const int n_live = all.total;
  // holes below n_live and movers at or past it pair off by rank
  const Run low_run = {run.p0, max(run.p0, min(run.p1, n_live))};
  const Sums low = scan<CTAS>(count_used(st.refs, low_run), warp_sums, &cta_sum);
  const int live_before = __shfl_sync(0xffffffffu, all.before, 0), low_before = __shfl_sync(0xffffffffu, low.before, 0);
  int hole = run.p0 - live_before, mover = live_before - low_before;
  for (int g = run.p0; g < run.p1; g += 128) {
    const int at = g + (threadIdx.x & 31) * 4, used = used_bits(st.refs, at, run.p1);
    const int below = page_bits(at, min(run.p1, n_live)), holes = below & ~used, movers = used & ~below;
    const int2 h = rank_bits(holes), m = rank_bits(movers);
    int to = hole + h.x, from = mover + m.x;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (holes >> c & 1) sc.moves[to++].y = at + c;
      if (movers >> c & 1) {
        sc.remap[at + c] = from;  // the move that takes this page
        sc.moves[from++].x = at + c;
      }
    }
    hole += h.y;
    mover += m.y;
  }
  if (me == 0) {
    sc.n_moves[0] = n_live - low.total;
    sc.n_moves[1] = n_live;
  }
}

// ---- moving ---------------------------------------------------------------------------------------------------------
struct MoveParams {
  State st;
  Scratch sc;
  const void* const* pools;  // n_pools base addresses
  int64_t page_bytes, head_bytes;  // strides
  int n_pools, n_heads, run_bytes; // one (page, head): a contiguous run, a multiple of 16 bytes
  const int *children, *parents;   // a fork's lists, else null
  int n;
};

// A warp copies one (move, pool, head) run of 2 to 8 KB at a time, eight 16-byte words a lane in flight.
__device__ __forceinline__ void copy_runs(const MoveParams& p) {
  const int lane = threadIdx.x & 31, warps = gridDim.x * (kMoveThreads / 32);
  const int64_t total = (int64_t)p.sc.n_moves[0] * p.n_pools * p.n_heads;
  const int words = p.run_bytes / 16;
  for (int64_t u = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); u < total; u += warps) {
    const int head = (int)(u % p.n_heads), pool = (int)(u / p.n_heads % p.n_pools);
    const int2 mv = p.sc.moves[u / p.n_heads / p.n_pools];
    if ((unsigned)mv.x >= (unsigned)p.st.n_pages || (unsigned)mv.y >= (unsigned)p.st.n_pages) {
      if (lane == 0) report(p.st, DEV_STATUS_BAD_INDEX);  // a table entry that was never a page
      continue;
    }
    char* base = (char*)p.pools[pool] + head * p.head_bytes;
    const uint4* src = reinterpret_cast<const uint4*>(base + mv.x * p.page_bytes);
    uint4* dst = reinterpret_cast<uint4*>(base + mv.y * p.page_bytes);
    for (int w = lane; w < words; w += 256) {
      uint4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (w + 32 * i < words) x[i] = __ldcs(src + w + 32 * i);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (w + 32 * i < words) __stcs(dst + w + 32 * i, x[i]);
    }
  }
}

__global__ void __launch_bounds__(kMoveThreads) pages_fork_kernel(const MoveParams p) {
  grid_dependency_wait();
  const State& st = p.st;
  // table rows and counts of what parent and child share: a warp takes 32 pages of an entry of the list
  const int pieces = (st.max_pages + 31) / 32;
  for (int64_t u = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); u < (int64_t)p.n * pieces;
       u += gridDim.x * (kMoveThreads / 32)) {
    const int i = (int)(u % p.n), j = (int)(u / p.n) * 32 + (threadIdx.x & 31);
    if (j >= p.sc.kept[i]) continue;
    const int page = st.table[(int64_t)p.parents[i] * st.max_pages + j];
    st.table[(int64_t)p.children[i] * st.max_pages + j] = page;
    if ((unsigned)page < (unsigned)st.n_pages) atomicAdd(st.refs + page, 1);
    else report(st, DEV_STATUS_BAD_INDEX);
  }
  copy_runs(p);
}

__global__ void __launch_bounds__(kMoveThreads) pages_compact_kernel(const MoveParams p) {
  grid_dependency_wait();
  const State& st = p.st;
  const int n_live = p.sc.n_moves[1];
  const int64_t entries = (int64_t)st.n_rows * st.max_pages;
  for (int64_t i = blockIdx.x * kMoveThreads + threadIdx.x; i < entries; i += (int64_t)gridDim.x * kMoveThreads) {
    const int row = (int)(i / st.max_pages), j = (int)(i % st.max_pages);
    if (j >= pages_of(len_of(st, row))) continue;
    const int page = st.table[i];
    if (page >= 0 && page < n_live) continue;
    const int move = (unsigned)page < (unsigned)st.n_pages ? p.sc.remap[page] : -1;
    if ((unsigned)move < (unsigned)p.sc.n_moves[0] && p.sc.moves[move].x == page) st.table[i] = p.sc.moves[move].y;
    else report(st, DEV_STATUS_BAD_INDEX);  // never a page, or one that the counts call free
  }
  for (int i = blockIdx.x * kMoveThreads + threadIdx.x; i < p.sc.n_moves[0]; i += gridDim.x * kMoveThreads) {
    const int2 mv = p.sc.moves[i];
    st.refs[mv.y] = st.refs[mv.x];
    st.refs[mv.x] = 0;
  }
  copy_runs(p);
}

// One CTA per entry: whoever takes the row's length away gives its pages back, so a row named twice is freed once.
struct FreeParams { State st; Guard* guard; const int* rows; };
__global__ void __launch_bounds__(512) pages_free_kernel(const FreeParams p) {
  __shared__ int len_s;
  const State& st = p.st;
  grid_dependency_wait();
  const int row = p.rows[blockIdx.x];
  if ((unsigned)row >= (unsigned)st.n_rows) {
    if (threadIdx.x == 0) report(st, DEV_STATUS_BAD_INDEX);
    return;
  }
  if (threadIdx.x == 0) {
    len_s = max(0, min(atomicExch(st.lens + row, 0), st.max_pages * kPage));
    p.guard[row] = Guard{0, 0};
  }
  __syncthreads();
  for (int j = threadIdx.x; j < pages_of(len_s); j += 512) {
    int* entry = st.table + (int64_t)row * st.max_pages + j;
    const int page = *entry;
    *entry = -1;
    if ((unsigned)page >= (unsigned)st.n_pages) report(st, DEV_STATUS_BAD_INDEX);
    else if (atomicSub(st.refs + page, 1) <= 0) {  // not held by anyone: the counts were wrong before
      atomicAdd(st.refs + page, 1);
      report(st, DEV_STATUS_BAD_INDEX);
    }
  }
}

// ---- writing --------------------------------------------------------------------------------------------------------
struct WriteParams {
  State st;
  const Guard* guard;
  const int *rows, *starts;  // [n], [n + 1]
  int n, n_tokens;
  const char *k, *v;
  char *k_pool, *v_pool;
  int64_t k_tok, k_head, v_tok, v_head, page_bytes, head_bytes;  // strides in bytes
  int n_heads, run_words;                                        // 16-byte words of one (token, head)
};

// A warp per token: the token's heads are n_heads runs of run_words 16-byte words in keys and values.
__global__ void __launch_bounds__(kMoveThreads) pages_write_kernel(const WriteParams p) {
  grid_dependency_wait();
  const State& st = p.st;
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * (kMoveThreads / 32), me = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5);
  const int words = p.n_heads * p.run_words;
  // Whose a token is is found by halves, which asks for starts that do not fall.  One CTA reports, also what no token would meet.
  const int mine = lane < p.n ? p.starts[lane] : 0x7fffffff;  // the whole list, if a warp holds it (4 rows 3.08 us, by halves 3.27)
  bool falls = false, outside = false;
  for (int i = threadIdx.x; i < p.n; i += kMoveThreads) {
    const int a = p.starts[i], b = p.starts[i + 1];
    falls |= a > b;
    outside |= a < 0 || b > p.n_tokens;
  }
  if (outside && blockIdx.x == 0) report(st, DEV_STATUS_BAD_INDEX);
  if (__syncthreads_or(falls)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) report(st, DEV_STATUS_BAD_INDEX);
    return;
  }
  int entry = -1, row = 0, start = 0, end = 0, first = 0;  // the entry at hand: tokens [start, end), positions from `first`
  bool good = false;
  for (int t = me; t < p.n_tokens; t += warps) {
    if (entry < 0 || t < start || t >= end) {
      int lo = 0, hi = p.n - 1;  // last entry with starts[entry] <= t
      if (p.n <= 32) {
        lo = max(0, __popc(__ballot_sync(0xffffffffu, mine <= t)) - 1);
      } else {
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (p.starts[mid] <= t) lo = mid;
          else hi = mid - 1;
        }
      }
      entry = lo;
      start = p.starts[lo];
      end = p.starts[lo + 1];
      if (t < start || t >= end) {  // a token that no entry names stays unwritten
        entry = -1;
        continue;
      }
      row = p.rows[lo];
      good = (unsigned)row < (unsigned)st.n_rows && start >= 0 && end <= p.n_tokens;
      const int len = good ? len_of(st, row) : 0;
      const Guard g = good ? p.guard[row] : Guard{0, 0};
      bool again = false;
      for (int i = lane; good && i < lo; i += 32) again |= p.rows[i] == row;
      good = good && !__any_sync(0xffffffffu, again);  // a row named twice: the first entry counts
      if (good) {
        first = len - (end - start);
        good = first >= 0 && g.refused == 0;
        const int shared = min(g.shared, first + end - start);
        if (good && first < shared) {  // no page of these may be another row's too
          bool held = false;
          for (int j = first / kPage + lane; j < pages_of(shared); j += 32) {
            const int page = st.table[(int64_t)row * st.max_pages + j];
            held |= (unsigned)page < (unsigned)st.n_pages && st.refs[page] > 1;
          }
          good = !__any_sync(0xffffffffu, held);
        }
      }
      if (!good && lane == 0) report(st, DEV_STATUS_BAD_INDEX);
    }
    if (!good) continue;
    const int pos = first + t - start;
    const int page = st.table[(int64_t)row * st.max_pages + pos / kPage];
    if ((unsigned)page >= (unsigned)st.n_pages) {
      if (lane == 0) report(st, DEV_STATUS_BAD_INDEX);
      continue;
    }
    const int64_t to = page * p.page_bytes + (int64_t)(pos % kPage) * p.run_words * 16;
    for (int w = lane; w < words; w += 128) {
      uint4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (w + 32 * i < words) {
          const int h = (w + 32 * i) / p.run_words, c = (w + 32 * i) % p.run_words * 16;
          a[i] = __ldcs(reinterpret_cast<const uint4*>(p.k + t * p.k_tok + h * p.k_head + c));
          b[i] = __ldcs(reinterpret_cast<const uint4*>(p.v + t * p.v_tok + h * p.v_head + c));
        }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (w + 32 * i < words) {
          const int h = (w + 32 * i) / p.run_words, c = (w + 32 * i) % p.run_words * 16;
          *reinterpret_cast<uint4*>(p.k_pool + to + h * p.head_bytes + c) = a[i];
          *reinterpret_cast<uint4*>(p.v_pool + to + h * p.head_bytes + c) = b[i];
        }
    }
  }
}

// None of the kernels that end a call lets its successor start early: that may be a kernel which reads tables, lengths
// or pages before it waits.
template <typename Params>
int launch(void (*kern)(Params), unsigned grid, unsigned block, cudaStream_t stream, const char* what, const Params& p, int cluster = 1) {
  const cudaError_t e = launch_overlapped(kern, grid, block, 0, stream, p, cluster);
  return e == cudaSuccess ? check_launch(what) : fail(IA_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
}

int state_of(const ia_page_cache& c, State* st) {
  *st = State{c.block_table, c.seq_lens, c.refs, device_status_address(), c.n_rows, c.max_pages, c.n_pages};
  return st->status ? IA_OK : IA_ERR_LAUNCH;
}
Scratch scratch_of(const ia_page_cache& c) {
  Scratch s;
  scratch_layout((char*)c.scratch, c.n_rows, c.n_pages, &s);
  return s;
}
MoveParams moves_of(const ia_page_cache& c, const State& st, const Scratch& sc) {
  const int size = c.dtype == IA_BF16 ? 2 : 4;
  MoveParams m{};
  m.st = st;
  m.sc = sc;
  m.pools = (const void* const*)c.pools;
  m.page_bytes = c.page_stride * size;
  m.head_bytes = c.head_stride * size;
  m.n_pools = c.n_pools;
  m.n_heads = c.n_kv_heads;
  m.run_bytes = kPage * c.head_dim * size;
  return m;
}

}  // namespace

int64_t page_cache_scratch_bytes(int64_t n_rows, int64_t n_pages) { return scratch_layout(nullptr, n_rows, n_pages, nullptr); }

static int plan(const ia_page_cache& c, const int32_t* rows, const int32_t* other, int n, int fork, int share, State* st,
                Scratch* sc, cudaStream_t stream) {
  if (int s = state_of(c, st)) return s;
  *sc = scratch_of(c);
  const PlanParams p{*st, *sc, rows, other, n, fork, share};
  if (n <= kSmallList && c.n_pages <= kSmallPool)
    return launch(pages_plan_kernel<1>, 1u, (unsigned)kPlanThreads, stream, "pages_plan_kernel", p);
  return launch(pages_plan_kernel<kPlanCtas>, (unsigned)kPlanCtas, (unsigned)kPlanThreads, stream, "pages_plan_kernel", p, kPlanCtas);
}

int launch_pages_extend(const ia_page_cache& c, const int32_t* rows, const int32_t* n_tokens, int n, cudaStream_t stream) {
  State st;
  Scratch sc;
  return plan(c, rows, n_tokens, n, 0, 0, &st, &sc, stream);
}

int launch_pages_fork(const ia_page_cache& c, const int32_t* parents, const int32_t* children, int n, int share,
                      cudaStream_t stream) {
  State st;
  Scratch sc;
  if (int s = plan(c, children, parents, n, 1, share, &st, &sc, stream)) return s;
  MoveParams m = moves_of(c, st, sc);
  m.children = children;
  m.parents = parents;
  m.n = n;
  return launch(pages_fork_kernel, (unsigned)sm_count() * 4, (unsigned)kMoveThreads, stream, "pages_fork_kernel", m);
}

int launch_pages_free(const ia_page_cache& c, const int32_t* rows, int n, cudaStream_t stream) {
  State st;
  if (int s = state_of(c, &st)) return s;
  return launch(pages_free_kernel, (unsigned)n, 512u, stream, "pages_free_kernel", FreeParams{st, scratch_of(c).guard, rows});
}

int launch_pages_compact(const ia_page_cache& c, cudaStream_t stream) {
  State st;
  if (int s = state_of(c, &st)) return s;
  const Scratch sc = scratch_of(c);
  const CompactParams p{st, sc};
  const int s = c.n_pages <= kSmallCompact
                    ? launch(pages_compact_plan_kernel<1>, 1u, (unsigned)kPlanThreads, stream, "pages_compact_plan_kernel", p)
                    : launch(pages_compact_plan_kernel<kPlanCtas>, (unsigned)kPlanCtas, (unsigned)kPlanThreads, stream,
                             "pages_compact_plan_kernel", p, kPlanCtas);
  if (s) return s;
  return launch(pages_compact_kernel, (unsigned)sm_count() * 4, (unsigned)kMoveThreads, stream, "pages_compact_kernel",
                moves_of(c, st, sc));
}

int launch_pages_write(const ia_page_cache& c, const int32_t* rows, const int32_t* starts, int n, const PagesWrite& w,
                       cudaStream_t stream) {
  State st;
  if (int s = state_of(c, &st)) return s;
  const int size = c.dtype == IA_BF16 ? 2 : 4;
  const int64_t warps = w.n_tokens, ctas = (warps + kMoveThreads / 32 - 1) / (kMoveThreads / 32);
  return launch(pages_write_kernel, (unsigned)std::min<int64_t>(ctas, sm_count() * 8), (unsigned)kMoveThreads, stream,
                "pages_write_kernel",
                WriteParams{st, scratch_of(c).guard, rows, starts, n, w.n_tokens, (const char*)w.k, (const char*)w.v, (char*)w.k_pool, (char*)w.v_pool,
                            w.k_tok_stride * size, w.k_head_stride * size, w.v_tok_stride * size, w.v_head_stride * size,
                            c.page_stride * size, c.head_stride * size, c.n_kv_heads, c.head_dim * size / 16});
}

}  // namespace ia
