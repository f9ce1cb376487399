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
// Measured: moving 1.14 GB of pages 182 us (0.97 of the copy peak), a plan over 18,400 pages 10 us, 64 forks of 8k tokens 19 us with
// the free before them (the host's 18 us); the plan is a chain of dependent loads and barriers.
#include <algorithm>

#include "dense_attention.cuh"
#include "page_cache.cuh"

namespace ia {
namespace {

constexpr int kPage = 16;
constexpr int kPlanCtas = 8, kPlanThreads = 1024;  // of the large plan; the small one is one CTA
constexpr int kSmallList = 256, kSmallPool = 65536;
constexpr int kMoveThreads = 256;

// scratch: counters, then per entry of a list the inclusive sum of the pages wanted and what was granted, then the moves
struct Scratch {
  int* n_moves;      // [4]: moves, live pages, unused
  int* owner;        // [n_rows] first entry of the list that names the row
  int* upto;         // [n_entries] inclusive sums
  int* kept;         // [n_entries] pages of the row before, or taken over from the parent; -1: the entry was refused
  int* new_len;      // [n_entries]
  int2* moves;       // [n_pages] (from, to)
  int* remap;        // [n_pages]
};
int64_t scratch_layout(char* base, int64_t n_rows, int64_t n_pages, Scratch* s) {
  int64_t off = 0;
  auto take = [&](int64_t bytes) {
    char* r = base ? base + off : nullptr;
    off += (bytes + 255) / 256 * 256;
    return r;
  };
  char* a[7] = {take(16),         take(n_rows * 4),  take(n_rows * 4), take(n_rows * 4),
                take(n_rows * 4), take(n_pages * 8), take(n_pages * 4)};  // no list is longer than the table
  if (s) *s = Scratch{(int*)a[0], (int*)a[1], (int*)a[2], (int*)a[3], (int*)a[4], (int2*)a[5], (int*)a[6]};
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

// how many of the pages [p0, p1) are free; four counts at a time where the array allows it
__device__ __forceinline__ int count_free(const int* refs, int p0, int p1) {
  int n = 0, g = p0;
  if ((reinterpret_cast<uintptr_t>(refs + p0) & 15) == 0) {
#pragma unroll 4
    for (; g + 4 <= p1; g += 4) {
      const int4 r = *reinterpret_cast<const int4*>(refs + g);
      n += (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0);
    }
  }
  for (; g < p1; ++g) n += refs[g] == 0;
  return n;
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
  __shared__ int named[CTAS == 1 ? kSmallList : 1];
  constexpr int kAll = CTAS * kPlanThreads;
  const State& st = p.st;
  const int me = cta_rank<CTAS>() * kPlanThreads + threadIdx.x;
  const int per = (p.n + kAll - 1) / kAll, i0 = min(p.n, me * per), i1 = min(p.n, i0 + per);
  if constexpr (CTAS > 1) sync_all<CTAS>();  // the whole cluster runs before anyone reads a peer's shared memory
  grid_dependency_wait();
  if (p.fork) grid_launch_dependents();  // the copies follow; what follows an extend is not known here
  // free pages; a thread counts a run of them
  const int run = ((st.n_pages + kAll - 1) / kAll + 3) & ~3, p0 = min(st.n_pages, me * run), p1 = min(st.n_pages, p0 + run);
  const int n_free = count_free(st.refs, p0, p1);
  // a row that the list names twice belongs to its first entry
  bool again = false;
  if constexpr (CTAS == 1) {
    if (me < p.n) named[me] = p.rows[me];
    __syncthreads();
    if (me < p.n)
      for (int i = 0; i < me; ++i) again |= named[i] == named[me];
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
  int wanted = 0;
  for (int i = i0; i < i1; ++i) {
    const int row = p.rows[i], other = p.other[i];
    int kept = -1, need = 0;
    if constexpr (CTAS > 1)
      if ((unsigned)row < (unsigned)st.n_rows) again = __ldcg(p.sc.owner + row) != i;
    if ((unsigned)row < (unsigned)st.n_rows && !again) {
      const int len = len_of(st, row);
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
    if (!fits && p.sc.kept[i] >= 0) {
      p.sc.kept[i] = -1;
      report(st, IA_DEV_STATUS_NO_PAGES);
    }
    if (fits) granted += need;
  }
  __threadfence();
  const Sums grants = scan<CTAS>(granted, warp_sums, &cta_sum);  // also: the sums above are visible to all
  // new lengths; all lengths were read before the barriers above
  for (int i = i0; i < i1; ++i)
    if (p.sc.kept[i] >= 0) st.lens[p.rows[i]] = p.sc.new_len[i];
  // the free page of rank r goes to the entry whose sums enclose r
  int rank = free_pages.before;
  for (int g = p0; g < p1 && rank < grants.total; ++g) {
    if (st.refs[g] != 0) continue;
    int lo = 0, hi = p.n - 1;  // first entry with upto > rank
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldcg(p.sc.upto + mid) > rank) hi = mid;
      else lo = mid + 1;
    }
    const int before = lo > 0 ? __ldcg(p.sc.upto + lo - 1) : 0, at = __ldcg(p.sc.kept + lo) + rank - before;
    st.table[(int64_t)p.rows[lo] * st.max_pages + at] = g;
    st.refs[g] = 1;
    if (p.fork) p.sc.moves[rank] = make_int2(st.table[(int64_t)p.other[lo] * st.max_pages + at], g);
    ++rank;
  }
  if (me == 0) p.sc.n_moves[0] = p.fork ? grants.total : 0;
}

// Live pages at or past the number of live pages move into the holes below it, in order.
struct CompactParams { State st; Scratch sc; };
template <int CTAS> __global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(const CompactParams p) {
  __shared__ int warp_sums[32];
  __shared__ int cta_sum;
  constexpr int kAll = CTAS * kPlanThreads;
  const State& st = p.st;
  const Scratch& sc = p.sc;
  const int me = cta_rank<CTAS>() * kPlanThreads + threadIdx.x;
  if constexpr (CTAS > 1) sync_all<CTAS>();
  grid_dependency_wait();
  grid_launch_dependents();
  const int run = ((st.n_pages + kAll - 1) / kAll + 3) & ~3, p0 = min(st.n_pages, me * run), p1 = min(st.n_pages, p0 + run);
  const Sums all = scan<CTAS>(p1 - p0 - count_free(st.refs, p0, p1), warp_sums, &cta_sum);
  const int n_live = all.total;
  // live pages before n_live: the sum up to the boundary; holes below it and movers above it pair off by rank
  int hole = p0 - all.before;
  const int upto = max(p0, min(p1, n_live));
  const Sums low = scan<CTAS>(upto - p0 - count_free(st.refs, p0, upto), warp_sums, &cta_sum);
  int mover = all.before - min(all.before, low.total);
  if (p0 < n_live && p1 > n_live) mover = 0;
  for (int g = p0; g < p1; ++g) {
    const bool is_live = st.refs[g] != 0;
    if (g < n_live && !is_live) sc.moves[hole++].y = g;
    if (g >= n_live && is_live) {
      sc.remap[g] = mover;  // the move that takes this page
      sc.moves[mover++].x = g;
    }
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
struct FreeParams { State st; const int* rows; };
__global__ void __launch_bounds__(512) pages_free_kernel(const FreeParams p) {
  __shared__ int len_s;
  const State& st = p.st;
  grid_dependency_wait();
  const int row = p.rows[blockIdx.x];
  if ((unsigned)row >= (unsigned)st.n_rows) {
    if (threadIdx.x == 0) report(st, DEV_STATUS_BAD_INDEX);
    return;
  }
  if (threadIdx.x == 0) len_s = max(0, min(atomicExch(st.lens + row, 0), st.max_pages * kPage));
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
  int entry = -1, row = 0, start = 0, end = 0, first = 0;  // the entry at hand: tokens [start, end), positions from `first`
  bool good = false;
  for (int t = me; t < p.n_tokens; t += warps) {
    if (entry < 0 || t < start || t >= end) {
      int lo = 0, hi = p.n - 1;  // last entry with starts[entry] <= t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.starts[mid] <= t) lo = mid;
        else hi = mid - 1;
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
      bool again = false;
      for (int i = lane; good && i < lo; i += 32) again |= p.rows[i] == row;
      good = good && !__any_sync(0xffffffffu, again);  // a row named twice: the first entry counts
      if (good) {
        first = len_of(st, row) - (end - start);
        good = first >= 0;
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
  return launch(pages_free_kernel, (unsigned)n, 512u, stream, "pages_free_kernel", FreeParams{st, rows});
}

int launch_pages_compact(const ia_page_cache& c, cudaStream_t stream) {
  State st;
  if (int s = state_of(c, &st)) return s;
  const Scratch sc = scratch_of(c);
  const CompactParams p{st, sc};
  const int s = c.n_pages <= kSmallPool
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
                WriteParams{st, rows, starts, n, w.n_tokens, (const char*)w.k, (const char*)w.v, (char*)w.k_pool, (char*)w.v_pool,
                            w.k_tok_stride * size, w.k_head_stride * size, w.v_tok_stride * size, w.v_head_stride * size,
                            c.page_stride * size, c.head_stride * size, c.n_kv_heads, c.head_dim * size / 16});
}

}  // namespace ia
