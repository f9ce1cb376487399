// Dense attention on the CUDA cores, the merge of the shared-prefix decode step, and the host side of the prompt's plan.
//
//   o_r = sum_{j < limit_r} softmax_j(q_r . k_j / sqrt(D)) v_j
//
// One pass over the keys in tiles of 64 with the running maximum m and sum l of each row: a tile's logits go from
// registers through shared memory into the second product, the accumulator is rescaled by exp(m_old - m_new) when the
// maximum moves.  All of it in fp32.  A thread owns RPT rows x 4 keys of the logits and RPT rows x D / 16 output columns;
// 16 neighbouring lanes share a row, so the row's statistics are four shuffles.  Rows of 132 floats keep the key reads of
// 8 lanes on 32 banks.  A 4096-token prompt at 32 / 8 heads of 128: 38 TFLOP/s, bound by latency: two warps a scheduler, which wait
// for operands from shared memory, with the FMA pipe busy for 57 % of the cycles and shared memory for 49 %.  Decode steps of up to kFewRows rows are bound by reading the cache and have a form of their own.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <functional>
#include <queue>
#include <utility>
#include <vector>

#include "dense_attention.cuh"

namespace ia {
namespace {

constexpr int kThreads = 256, kKeys = 64, kPLd = kKeys + 4, kFewRows = 16;

// K and V of the next tile replace each as soon as it has been used.
template <int D, int RPT> struct Smem {
  static constexpr int rows = 16 * RPT, ld = D + 4;
  static constexpr int q = 0, k = q + rows * ld, v = k + kKeys * ld, p = v + kKeys * D, floats = p + rows * kPLd;
  static constexpr size_t bytes = (size_t)floats * 4 + rows * 8;  // + limits and flags
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // 0: sixteen zero bytes, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
               "r"(n)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// rows of a [kKeys, D] tile from key j0 on; rows at or past `hi`, and rows without an address, are zero
template <bool VALUES, int D, int LD, typename Key>
__device__ __forceinline__ void load_tile(float* dst, const float* any, int j0, int hi, const Key& key) {
#pragma unroll 4
  for (int i = threadIdx.x; i < kKeys * D / 4; i += kThreads) {
    const int row = i / (D / 4), c = i % (D / 4) * 4;
    const float *k = any, *v = any;
    const bool ok = j0 + row < hi && key(j0 + row, k, v);
    cp_async16(dst + row * LD + c, (VALUES ? v : k) + (ok ? c : 0), ok);
  }
}

// Rows [0, n_rows) of one piece over the keys [lo, hi).  q_row(r): the row's query; limit(r): the keys below it are seen;
// sink.row(r) -> where its outputs go.
template <int D, int RPT, typename Key, typename QRow, typename Limit, typename Sink>
__device__ void attend(float* sm, int n_rows, int lo, int hi, float scale_log2, const Key& key, const QRow& q_row,
                       const Limit& limit, const Sink& sink) {
  using S = Smem<D, RPT>;
  constexpr int ROWS = S::rows, LD = S::ld, NO = D / 64;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  float *qs = sm + S::q, *ks = sm + S::k, *vs = sm + S::v, *ps = sm + S::p;
  int* lim = reinterpret_cast<int*>(sm + S::floats);
  int* bad = lim + ROWS;
  const float* any = q_row(0);
  __syncthreads();  // the piece before is done with the shared memory
  for (int i = tid; i < ROWS * D / 4; i += kThreads) {
    const int row = i / (D / 4), c = i % (D / 4) * 4;
    cp_async16(qs + row * LD + c, row < n_rows ? q_row(row) + c : any, row < n_rows);
  }
  load_tile<false, D, LD>(ks, any, lo, hi, key);
  cp_commit();
  load_tile<true, D, D>(vs, any, lo, hi, key);
  cp_commit();
  if (tid < ROWS) {
    lim[tid] = tid < n_rows ? limit(tid) : 0;
    bad[tid] = 0;
  }
  float o[RPT][NO][4], m[RPT], l[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int a = 0; a < NO; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) o[i][a][b] = 0.f;
  }
  for (int j0 = lo; j0 < hi; j0 += kKeys) {
    const int ahead = j0 + kKeys;
    cp_wait<1>();
    __syncthreads();
    float s[RPT][4];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[i][c] = 0.f;
#pragma unroll 2
    for (int d = 0; d < D; d += 4) {
      float4 kv[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) kv[c] = *reinterpret_cast<const float4*>(ks + (tx + 16 * c) * LD + d);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float4 qv = *reinterpret_cast<const float4*>(qs + (ty * RPT + i) * LD + d);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[i][c] += qv.x * kv[c].x;
          s[i][c] += qv.y * kv[c].y;
          s[i][c] += qv.z * kv[c].z;
          s[i][c] += qv.w * kv[c].w;
        }
      }
    }
    __syncthreads();
    if (ahead < hi) load_tile<false, D, LD>(ks, any, ahead, hi, key);
    cp_commit();
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int end = lim[ty * RPT + i] - j0;
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[i][c] = tx + 16 * c < end ? s[i][c] * scale_log2 : -INFINITY;
        top = fmaxf(top, s[i][c]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float m_new = fmaxf(m[i], top), base = m_new == -INFINITY ? 0.f : m_new;
      const float keep = exp2f(m[i] - base);
      m[i] = m_new;
      l[i] *= keep;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float w = exp2f(s[i][c] - base);
        l[i] += w;
        ps[(ty * RPT + i) * kPLd + tx + 16 * c] = w;
      }
#pragma unroll
      for (int a = 0; a < NO; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) o[i][a][b] *= keep;
    }
    cp_wait<1>();
    __syncthreads();  // also: the row's weights are written
#pragma unroll 2
    for (int n = 0; n < kKeys; n += 4) {
      float4 w[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) w[i] = *reinterpret_cast<const float4*>(ps + (ty * RPT + i) * kPLd + n);
#pragma unroll
      for (int k4 = 0; k4 < 4; ++k4) {
#pragma unroll
        for (int a = 0; a < NO; ++a) {
          const float4 vv = *reinterpret_cast<const float4*>(vs + (n + k4) * D + tx * 4 + 64 * a);
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float wi = k4 == 0 ? w[i].x : k4 == 1 ? w[i].y : k4 == 2 ? w[i].z : w[i].w;
            o[i][a][0] += wi * vv.x;
            o[i][a][1] += wi * vv.y;
            o[i][a][2] += wi * vv.z;
            o[i][a][3] += wi * vv.w;
          }
        }
      }
    }
    __syncthreads();
    if (ahead < hi) load_tile<true, D, D>(vs, any, ahead, hi, key);
    cp_commit();
  }
  cp_wait<0>();
  __syncthreads();  // lim is written also where there was no tile
  bool some_bad = false;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int row = ty * RPT + i;
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
    if (row >= n_rows) continue;
    const bool empty = lim[row] <= lo;
    const float inv = empty ? 0.f : 1.f / l[i];
    bool finite = true;
#pragma unroll
    for (int a = 0; a < NO; ++a) {
      float e[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        e[b] = empty ? 0.f : o[i][a][b] * inv;
        finite &= fabsf(e[b]) <= 3.4028235e38f;
      }
      store_vec<4>(sink.row(row) + tx * 4 + 64 * a, e);
    }
    if (tx == 0 && sink.lse(row) != nullptr)
      *sink.lse(row) = empty ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
    if (!finite) bad[row] = 1;
    some_bad |= !finite;
  }
  if (!__syncthreads_or(some_bad)) return;
  for (int row = tid >> 5; row < n_rows; row += kThreads / 32) {
    if (!bad[row] || last_not_finite<float, D>(max(lo, lim[row]), hi, key) < 0) continue;
    float x[D / 32], mx, lx;
    exact_row<float, D, 2>(q_row(row), lo, lim[row], scale_log2, key, x, mx, lx);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) sink.row(row)[(tid & 31) + 32 * i] = x[i] / lx;
  }
}

struct RowSink {  // rows r = token * group + g of one kv head
  float *o, *l;
  int64_t o_tok, o_g, l_tok;
  int group;
  __device__ __forceinline__ float* row(int r) const { return o + r / group * o_tok + r % group * o_g; }
  __device__ __forceinline__ float* lse(int r) const { return l == nullptr ? nullptr : l + r / group * l_tok + r % group; }
};

// The decode step of a few rows (at most RP), where reading K and V is what takes the time: each warp has a ring of its own of
// 8-key batches and takes every eighth batch, D / 32 dims a lane.  32 / RP keys make 32 dot products, whose partial sums 31
// shuffles bring together so that lane k * RP + r ends up with the logit of key k and row r; weights go back the same way.
// The warps' outputs meet in shared memory at the end.  What a row does not see is never multiplied with it.
// 16 x 16000 shared keys at 8 kv heads of 128, 1 / 2 / 4 sequences of 4 rows each: 3.0 / 3.6 / 3.0 TB/s (the tiled form with
// 16 rows, three tiles under way: 1.2 TB/s for any of them; 16 rows here whatever there are: 1.9 TB/s).  Bound by the
// latency of a batch's chain - products, shuffles, exponential - with 8 warps an SM, and by the start of each segment.
// The batch loop is not unrolled: unrolled over a page, fetching the instructions took 50 us of a small step's 70 us.
constexpr int kWarps = kThreads / 32, kFewKeys = 8, kFewRing = 3 * 2 * kFewKeys * 128;  // floats of a warp's ring

template <int D, int RP, typename QRow, typename Limit>
__device__ void attend_few(float* sm, int n_rows, int lo, int hi, float scale_log2, const PagedKeys<float>& key, const QRow& q_row,
                           const Limit& limit, const RowSink& sink) {
  constexpr int V = D / 32, KB = 32 / RP, kBatch = 2 * kFewKeys * D, kStages = kFewRing / kBatch, kChunks = kFewKeys * D / 128;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, my_row = lane % RP, my_key = lane / RP;
  float* ring = sm + warp * kFewRing;
  __syncthreads();  // the piece before is done with the shared memory
  const auto page_of = [&](int j) {  // the page that holds key j, -1 where there is none
    if (j >= hi || (j >> 4) >= key.max_pages) return -1;
    const int page = key.table[j >> 4];
    return key.n_pages > 0 && page >= key.n_pages ? -1 : page;
  };
  const auto issue = [&](int j, int page, float* to) {  // a batch's K, then its V; zeros where there is no key
    const int64_t at = (int64_t)max(page, 0) * key.page_stride + (int64_t)(j & 15) * D;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = (i * 32 + lane) * 4;
      const bool ok = page >= 0 && j + c / D < hi;
      cp_async16(to + c, key.k + (ok ? at + c : 0), ok);
      cp_async16(to + kFewKeys * D + c, key.v + (ok ? at + c : 0), ok);
    }
  };
  constexpr int kStep = kWarps * kFewKeys;
  int j0 = lo + warp * kFewKeys, put = 0, get = 0;
#pragma unroll 1
  for (int i = 0; i < kStages - 1; ++i) {
    issue(j0 + i * kStep, page_of(j0 + i * kStep), ring + i * kBatch);
    cp_commit();
  }
  put = kStages - 1;
  int next = page_of(j0 + (kStages - 1) * kStep);
  float q[RP][V], acc[RP][V], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int r = 0; r < RP; ++r) {
    if (r < n_rows) load_vec<V>(q_row(r) + lane * V, q[r]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      q[r][i] = r < n_rows ? q[r][i] * scale_log2 : 0.f;
      acc[r][i] = 0.f;
    }
  }
  const int my_limit = my_row < n_rows ? limit(my_row) : 0;
#pragma unroll 1
  for (; j0 < hi; j0 += kStep) {
    __syncwarp();  // all lanes are done with the batch whose place is filled now
    issue(j0 + (kStages - 1) * kStep, next, ring + put * kBatch);
    cp_commit();
    if (++put == kStages) put = 0;
    next = page_of(j0 + kStages * kStep);
    cp_wait<kStages - 1>();
    __syncwarp();
    const float *ks = ring + get * kBatch + lane * V, *vs = ks + kFewKeys * D;
    if (++get == kStages) get = 0;
#pragma unroll 1
    for (int k0 = 0; k0 < kFewKeys; k0 += KB, ks += KB * D, vs += KB * D) {
      float s[32];
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        float x[V];
        load_vec<V>(ks + i * D, x);
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          s[i * RP + r] = q[r][0] * x[0];
#pragma unroll
          for (int d = 1; d < V; ++d) s[i * RP + r] += q[r][d] * x[d];
        }
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1)  // w values are left, in either half of the lanes the half that belongs there
#pragma unroll
        for (int i = 0; i < w; ++i) {
          const bool upper = lane & w;
          const float give = upper ? s[i] : s[i + w], keep = upper ? s[i + w] : s[i];
          s[i] = keep + __shfl_xor_sync(0xffffffffu, give, w);
        }
      const bool sees = j0 + k0 + my_key < my_limit;
      const unsigned seen = __ballot_sync(0xffffffffu, sees);
      const float t = sees ? s[0] : -INFINITY;
      float top = t;
#pragma unroll
      for (int w = RP; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.f : m_new;
      const float keep = exp2f(m - base), weight = exp2f(t - base);
      if (__any_sync(0xffffffffu, m_new != m)) {
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          const float kr = __shfl_sync(0xffffffffu, keep, r);
#pragma unroll
          for (int d = 0; d < V; ++d) acc[r][d] *= kr;
        }
        l *= keep;
      }
      m = m_new;
      l += weight;
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        float x[V];
        load_vec<V>(vs + i * D, x);
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          const float w = __shfl_sync(0xffffffffu, weight, i * RP + r);
          if (seen >> (i * RP + r) & 1) {
#pragma unroll
            for (int d = 0; d < V; ++d) acc[r][d] += w * x[d];
          }
        }
      }
    }
  }
#pragma unroll
  for (int w = RP; w < 32; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
  cp_wait<0>();
  __syncthreads();  // every ring is done with
  float *o = sm, *stats = sm + kWarps * RP * D;  // [warp][row][D], [warp][row](m, l)
#pragma unroll
  for (int r = 0; r < RP; ++r) store_vec<V>(o + (warp * RP + r) * D + lane * V, acc[r]);
  if (lane < RP) {
    stats[(warp * RP + lane) * 2] = m;
    stats[(warp * RP + lane) * 2 + 1] = l;
  }
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < n_rows * D; i += kThreads) {
    const int r = i / D, d = i % D;
    float M = -INFINITY, L = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, stats[(w * RP + r) * 2]);
    const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(stats[(w * RP + r) * 2] - base);
      L += stats[(w * RP + r) * 2 + 1] * f;
      x += o[(w * RP + r) * D + d] * f;
    }
    const bool empty = limit(r) <= lo;
    sink.row(r)[d] = empty ? 0.f : x / L;
    if (d == 0) *sink.lse(r) = empty ? -INFINITY : (M + log2f(L)) * kLn2;
  }
}

template <int D, int RPT>
__global__ void __launch_bounds__(kThreads) prompt_attention_kernel(const PromptTensors t, const PromptItem* items) {
  extern __shared__ __align__(16) float sm[];
  grid_dependency_wait();
  grid_launch_dependents();
  const PromptItem it = items[blockIdx.x];
  const int G = t.group, hq = t.n_kv_heads * G;
  const PackedKeys<float> key{(const float*)t.k + it.kv_tok * t.k_tok_stride + it.head * t.k_head_stride,
                              (const float*)t.v + it.kv_tok * t.v_tok_stride + it.head * t.v_head_stride, t.k_tok_stride,
                              t.v_tok_stride, it.kv_len};
  const float* q = (const float*)t.q + it.q_tok * t.q_tok_stride + (int64_t)it.head * G * t.q_head_stride;
  const auto q_row = [&](int r) { return q + r / G * t.q_tok_stride + r % G * t.q_head_stride; };
  const auto limit = [&](int r) { return max(0, min(it.limit0 + r / G, it.kv_len)); };
  const RowSink whole{(float*)t.out + ((int64_t)it.q_tok * hq + it.head * G) * D,
                      t.lse == nullptr ? nullptr : t.lse + (int64_t)it.q_tok * hq + it.head * G, (int64_t)hq * D, D, hq, G};
  const int64_t row0 = (int64_t)it.slot * kPartRows;
  const RowSink sink = t.part_o == nullptr ? whole : RowSink{t.part_o + row0 * D, t.part_lse + row0, (int64_t)G * D, D, G, G};
  attend<D, RPT>(sm, it.n_tok * G, 0, limit(it.n_tok * G - 1), kLog2e * rsqrtf((float)D), key, q_row, limit, sink);
}

// The decode step: this CTA's share of all units, segment by segment.
template <int D>
__global__ void __launch_bounds__(kThreads) shared_attention_kernel(const SharedParams p) {
  extern __shared__ __align__(16) float sm[];
  __shared__ unsigned long long scratch[kThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int G = p.group, hq = p.n_kv_heads * G, cta = blockIdx.x;
  SharedCursor c = find_share<0, kThreads>(p, cta, gridDim.x, scratch);
  while (c.left > 0) {
    const SharedEntity ent = load_entity(p, c.e);
    int lo, hi;
    entity_keys(p, c.e, ent, lo, hi);
    const int n = (int)min((int64_t)(c.units - c.k), c.left);
    const int2 lead = entity_lead(p, ent, hi);
    const int32_t* table = p.block_table + (int64_t)lead.x * p.max_pages;
    const int from = lo + c.k * ent.unit, to = max(from, min(lead.y, from + n * ent.unit));
    const bool own = c.e >= p.n_shared;
    const int64_t row0 = c.k == 0 ? item_rows(p, own, ent.first_seq, ent.n_seqs, c.h) : cta_rows(p, cta);
    const PagedKeys<float> key{(const float*)p.k_pool + c.h * p.head_stride, (const float*)p.v_pool + c.h * p.head_stride,
                               table, p.page_stride, D, p.n_pool_pages, p.max_pages};
    const float* q = (const float*)p.q + ((int64_t)ent.first_seq * hq + c.h * G) * D;
    const auto q_row = [&](int r) { return q + (int64_t)(r / G) * hq * D + r % G * D; };
    const auto limit = [&](int r) { return min(to, shared_seq_len(p, ent.first_seq + r / G)); };
    const RowSink sink{p.o + row0 * D, p.lse + row0, (int64_t)G * D, D, G, G};
    for (int j = (from >> 4) + threadIdx.x; j < (to + 15) >> 4; j += kThreads) {
      const int page = table[j];
      if (page < 0 || (p.n_pool_pages > 0 && page >= p.n_pool_pages)) atomicOr(p.status, DEV_STATUS_BAD_INDEX);
    }
    // Few rows: see attend_few.  More: the tile with the fewest empty rows; 16 groups of 8 / 16 sequences of 4 rows over
    // 4000 keys 0.59 / 0.74 ms, with tiles of 128 rows 1.13 / 1.21 ms.
    const int n_rows = ent.n_seqs * G;
    const float scale = kLog2e * rsqrtf((float)D);
    if (n_rows <= 4) attend_few<D, 4>(sm, n_rows, from, to, scale, key, q_row, limit, sink);
    else if (n_rows <= 8) attend_few<D, 8>(sm, n_rows, from, to, scale, key, q_row, limit, sink);
    else if (n_rows <= kFewRows) attend_few<D, kFewRows>(sm, n_rows, from, to, scale, key, q_row, limit, sink);
    else if (n_rows <= 32) attend<D, 2>(sm, n_rows, from, to, scale, key, q_row, limit, sink);
    else if (n_rows <= 64) attend<D, 4>(sm, n_rows, from, to, scale, key, q_row, limit, sink);
    else attend<D, 8>(sm, n_rows, from, to, scale, key, q_row, limit, sink);
    c.left -= n;
    c.k = 0;
    if (++c.h == p.n_kv_heads) {
      c.h = 0;
      if (c.left > 0)  // some entity behind this one has units: they were counted
        do c.units = entity_units<0>(p, ++c.e);
        while (c.units == 0);
    }
  }
}

// out[row] = sum_s o_s 2^(lse_s - M) / sum_s 2^(lse_s - M) over partial rows, a warp per output row.  Lane i fetches the i-th
// log-sum-exp, so the weights are there before the first partial row, whose loads then do not depend on one another.
// A part with a log-sum-exp of -infinity is one that the row sees nothing of, and zeros, or one whose logits are all -infinity, and
// NaN.  Neither weighs anything, so its row is not multiplied but left out; only where every part is of this kind does
// a NaN among them count: infinity minus infinity, as if the keys had not been cut.
template <int D> struct Merged {
  float acc[D / 32], M = -INFINITY, L = 0.f, weightless = 0.f;
  __device__ __forceinline__ Merged() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  }
  // `count` more, lane i's in row `row`
  __device__ __forceinline__ void add(const float* o, const float* lses, int64_t row, int count) {
    const int lane = threadIdx.x & 31;
    const float lse = lane < count ? __ldcg(lses + row) * kLog2e : -INFINITY;
    const float* src = o + row * D;
    const float m = fmaxf(M, warp_max(lse)), base = m == -INFINITY ? 0.f : m;
    const float keep = exp2f(M - base), w = exp2f(lse - base);
    const unsigned none = __ballot_sync(0xffffffffu, lane < count && lse == -INFINITY);
    L = L * keep + warp_sum(w);
    M = m;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] *= keep;
    if (none == 0) {
#pragma unroll 8
      for (int s = 0; s < count; ++s) add_row(src, w, s, false);
    } else {  // apart: the usual case keeps its short loop
#pragma unroll 1
      for (int s = 0; s < count; ++s) add_row(src, w, s, none >> s & 1);
    }
  }
  // lane s's row by its weight
  __device__ __forceinline__ void add_row(const float* src, float w, int s, bool none) {
    constexpr int V = D / 32;
    const float ws = __shfl_sync(0xffffffffu, w, s);
    const float* from = (const float*)__shfl_sync(0xffffffffu, (unsigned long long)src, s) + (threadIdx.x & 31) * V;
    float x[V];
    if constexpr (D == 128) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(from));
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(from));
      x[0] = v.x; x[1] = v.y;
    }
    if (none) weightless += x[0];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += ws * (none ? 0.f : x[i]);
  }
  template <typename T> __device__ __forceinline__ void store(T* to) {
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = L == 0.f ? weightless : acc[i] * inv;  // no keys: zeros
    store_vec<D / 32>(to + (threadIdx.x & 31) * (D / 32), acc);
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(256) prompt_merge_kernel(const PromptTensors t, const PromptPiece* pieces, int blocks) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.x % blocks * 8 + warp;
  const PromptPiece piece = pieces[blockIdx.x / blocks];
  grid_dependency_wait();
  grid_launch_dependents();
  const int G = t.group, hq = t.n_kv_heads * G;
  if (r >= piece.n_tok * G) return;
  Merged<D> merged;
  for (int s = 0; s < piece.parts; s += 32)
    merged.add(t.part_o, t.part_lse, (int64_t)(piece.slot + s + lane) * kPartRows + r, min(32, piece.parts - s));
  const int64_t row = (int64_t)(piece.q_tok + r / G) * hq + piece.head * G + r % G;
  if (t.lse != nullptr && lane == 0) t.lse[row] = merged.L == 0.f ? -INFINITY : (merged.M + log2f(merged.L)) * kLn2;
  merged.store((T*)t.out + row * D);
}

// The segments of a row's shared and own item.
template <typename T, int D>
__global__ void __launch_bounds__(256) shared_merge_kernel(const SharedParams p, const int2* seq_info, int ctas, T* out) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = p.group, hq = p.n_kv_heads * G;
  const int per_seq = (hq + 7) / 8, seq = blockIdx.x / per_seq, head = blockIdx.x % per_seq * 8 + warp;
  const int2 info = seq_info[seq];  // shared entity, the sequence's place in it
  const int own_e = p.n_shared + seq;
  grid_dependency_wait();
  grid_launch_dependents();
  if (head >= hq) return;
  const long long total = __ldcg(p.unit_begin + p.n_shared + p.batch);
  const long long begin[2] = {__ldcg(p.unit_begin + info.x), __ldcg(p.unit_begin + own_e)};
  const long long end[2] = {__ldcg(p.unit_begin + info.x + 1), __ldcg(p.unit_begin + own_e + 1)};
  ctas = shares_of(total, ctas);
  const int h = head / G, g = head % G;
  int n[2], c0[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const long long units = (end[i] - begin[i]) / p.n_kv_heads, u0 = begin[i] + h * units;
    c0[i] = units > 0 ? share_owner(u0, total, ctas) : 0;
    n[i] = units > 0 ? share_owner(u0 + units - 1, total, ctas) - c0[i] + 1 : 0;
  }
  const SharedEntity ent = load_entity(p, info.x);
  const int at[2] = {info.y * G + g, g};  // the row in its item
  const int64_t first[2] = {item_rows(p, false, ent.first_seq, ent.n_seqs, h) + at[0], item_rows(p, true, seq, 1, h) + at[1]};
  Merged<D> merged;
  for (int s0 = 0; s0 < n[0] + n[1]; s0 += 32) {
    const int mine = s0 + lane;
    const bool own = mine >= n[0];
    const int segment = own ? mine - n[0] : mine;
    const int64_t row = segment == 0 ? first[own] : cta_rows(p, c0[own] + segment) + at[own];
    merged.add(p.o, p.lse, row, min(32, n[0] + n[1] - s0));
  }
  merged.store(out + ((int64_t)seq * hq + head) * D);
}

template <typename... Args, typename... Given>
int launch(void (*kern)(Args...), unsigned grid, size_t smem, cudaStream_t stream, const char* what, Given... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = overlapped_launch_enabled() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  return e == cudaSuccess ? check_launch(what) : fail(IA_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
}

template <int D, int RPT>
int launch_prompt(const PromptTensors& t, const PromptItem* items, int n_items, cudaStream_t stream) {
  auto kern = prompt_attention_kernel<D, RPT>;
  static SmemOnce once;
  if (int s = once.allow((const void*)kern, Smem<D, RPT>::bytes, "prompt_attention_kernel")) return s;
  return launch(kern, (unsigned)n_items, Smem<D, RPT>::bytes, stream, "prompt_attention_kernel", t, items);
}
template <int D> int launch_shared(const SharedParams& p, int ctas, cudaStream_t stream) {
  auto kern = shared_attention_kernel<D>;
  static SmemOnce once;
  constexpr size_t bytes = std::max(Smem<D, 8>::bytes, (size_t)kWarps * kFewRing * 4);
  if (int s = once.allow((const void*)kern, bytes, "shared_attention_kernel")) return s;
  return launch(kern, (unsigned)ctas, bytes, stream, "shared_attention_kernel", p);
}
template <typename T, int D>
int launch_parts(const PromptTensors& t, const PromptPiece* pieces, int n_pieces, bool few_rows, cudaStream_t stream) {
  const int blocks = (std::is_same_v<T, float> && few_rows ? 32 : kPartRows) / 8;
  return launch(prompt_merge_kernel<T, D>, (unsigned)(n_pieces * blocks), 0, stream, "prompt_merge_kernel", t, pieces, blocks);
}
template <typename T, int D>
int launch_merge(const SharedParams& p, const int2* seq_info, int ctas, T* out, cudaStream_t stream) {
  const int per_seq = (p.n_kv_heads * p.group + 7) / 8;
  return launch(shared_merge_kernel<T, D>, (unsigned)(p.batch * per_seq), 0, stream, "shared_merge_kernel", p, seq_info,
                ctas, out);
}

}  // namespace

int SmemOnce::allow(const void* kern, size_t bytes, const char* what) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(IA_ERR_LAUNCH, "%s: no current device", what);
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return IA_OK;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return fail(IA_ERR_LAUNCH, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
  if (dev < 64) done.fetch_or(bit, std::memory_order_release);
  return IA_OK;
}

int sm_count() {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> cached[kMaxDevices];
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 148;
  if (int n = cached[dev].load(std::memory_order_relaxed)) return n;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return 148;
  cached[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

int launch_prompt_f32(const PromptTensors& t, int head_dim, const PromptItem* items, int n_items, bool few_rows, cudaStream_t stream) {
  if (head_dim == 128) return few_rows ? launch_prompt<128, 2>(t, items, n_items, stream) : launch_prompt<128, 8>(t, items, n_items, stream);
  return few_rows ? launch_prompt<64, 2>(t, items, n_items, stream) : launch_prompt<64, 8>(t, items, n_items, stream);
}

int launch_prompt_merge(const PromptTensors& t, int head_dim, int dtype, const PromptPiece* pieces, int n_pieces, bool few_rows,
                        cudaStream_t stream) {
  if (dtype == IA_F32)
    return head_dim == 128 ? launch_parts<float, 128>(t, pieces, n_pieces, few_rows, stream)
                           : launch_parts<float, 64>(t, pieces, n_pieces, few_rows, stream);
  return head_dim == 128 ? launch_parts<__nv_bfloat16, 128>(t, pieces, n_pieces, few_rows, stream)
                         : launch_parts<__nv_bfloat16, 64>(t, pieces, n_pieces, few_rows, stream);
}

int launch_shared_f32(const SharedParams& p, int head_dim, int ctas, cudaStream_t stream) {
  return head_dim == 128 ? launch_shared<128>(p, ctas, stream) : launch_shared<64>(p, ctas, stream);
}

int launch_shared_merge(const SharedParams& p, const int32_t* seq_info, int head_dim, int dtype, int ctas, void* out,
                        cudaStream_t stream) {
  const int2* info = reinterpret_cast<const int2*>(seq_info);
  if (dtype == IA_F32)
    return head_dim == 128 ? launch_merge<float, 128>(p, info, ctas, (float*)out, stream)
                           : launch_merge<float, 64>(p, info, ctas, (float*)out, stream);
  return head_dim == 128 ? launch_merge<__nv_bfloat16, 128>(p, info, ctas, (__nv_bfloat16*)out, stream)
                         : launch_merge<__nv_bfloat16, 64>(p, info, ctas, (__nv_bfloat16*)out, stream);
}

// ---- the prompt's plan ----------------------------------------------------------------------------------------------
// Words: a header of 8, where each CTA's items begin (ctas + 1 words, padded to whole items), the items, and the pieces where
// they are cut.
namespace {
constexpr int kRowsFew = 32, kRowsFull = 128, kMostParts = 32;  // parts an SM, at most
struct PlanShape {
  int n_items, ctas, item_tokens;
  bool few_rows;
  int chunk = 0, n_pieces = 0;  // keys of a part, 0: not cut
  int64_t first() const { return 8 + (int64_t)(ctas + 1 + 7) / 8 * 8; }
  int64_t ints() const { return first() + ((int64_t)n_items + n_pieces) * 8; }
};
struct PlanInput {
  const int32_t *q_lens, *kv_lens;
  int n_seqs, n_kv_heads, group, dtype;
};
int piece_keys(const PromptItem& it) { return std::max(0, std::min(it.limit0 + it.n_tok - 1, it.kv_len)); }
// the pieces, the longest first, so that what is started last is short
std::vector<PromptItem> make_pieces(const PlanInput& in, const PlanShape& s, int64_t* n_q, int64_t* n_kv) {
  std::vector<PromptItem> items;
  items.reserve(s.n_items);
  int64_t q0 = 0, k0 = 0;
  for (int i = 0; i < in.n_seqs; ++i) {
    for (int t = 0; t < in.q_lens[i]; t += s.item_tokens)
      for (int h = 0; h < in.n_kv_heads; ++h)
        items.push_back(PromptItem{(int)(q0 + t), std::min(s.item_tokens, in.q_lens[i] - t), (int)k0,
                                   in.kv_lens[i] - in.q_lens[i] + t + 1, in.kv_lens[i], h, 0, 0});
    q0 += in.q_lens[i];
    k0 += in.kv_lens[i];
  }
  std::stable_sort(items.begin(), items.end(),
                   [](const PromptItem& a, const PromptItem& b) { return piece_keys(a) > piece_keys(b); });
  *n_q = q0;
  *n_kv = k0;
  return items;
}
// The parts of the pieces, the longest first, and which piece they make up.
std::vector<PromptItem> cut_pieces(const std::vector<PromptItem>& whole, int chunk, std::vector<PromptPiece>* pieces) {
  std::vector<PromptItem> parts;
  for (const PromptItem& it : whole) {
    const int n = std::max(1, (piece_keys(it) + chunk - 1) / chunk);
    if (pieces) pieces->push_back(PromptPiece{it.q_tok, it.n_tok, it.head, (int)parts.size(), n, {0, 0, 0}});
    for (int i = 0; i < n; ++i) {
      const int lo = i * chunk;
      parts.push_back(PromptItem{it.q_tok, it.n_tok, it.kv_tok + lo, it.limit0 - lo, std::min(it.kv_len - lo, chunk), it.head, (int)parts.size(), 0});
    }
  }
  std::stable_sort(parts.begin(), parts.end(),
                   [](const PromptItem& a, const PromptItem& b) { return piece_keys(a) > piece_keys(b); });
  return parts;
}
// What a piece costs, in quarters of what a key costs a large piece.  Starting and ending one takes as long as 256 keys
// (tensor cores; a small one 192) or 32 (fp32; 16); a key of a small piece, half or a quarter of the rows, 1 / 2 or 3 / 8.
int64_t piece_cost(const PromptItem& it, int dtype, bool few_rows) {
  const int64_t n = piece_keys(it);
  if (dtype == IA_F32) return few_rows ? n + n / 2 + 4 * 16 : 4 * n + 4 * 32;
  return few_rows ? 2 * n + 4 * 192 : 4 * n + 4 * 256;
}
// The next longest piece goes to the SM with the least to do so far; returns what the busiest has to do.
int64_t spread(const std::vector<PromptItem>& items, int ctas, int dtype, bool few_rows, std::vector<int>* cta_of) {
  using Load = std::pair<int64_t, int>;
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> loads;
  for (int c = 0; c < ctas; ++c) loads.push({0, c});
  int64_t most = 0;
  for (const PromptItem& it : items) {
    const Load at = loads.top();
    loads.pop();
    if (cta_of != nullptr) cta_of->push_back(at.second);
    const int64_t load = at.first + piece_cost(it, dtype, few_rows);
    most = std::max(most, load);
    loads.push({load, at.second});
  }
  return most;
}
struct PlanTotals { int64_t cost, longest; };  // of all pieces, and of the costliest
PlanTotals totals_of(const PlanInput& in, const PlanShape& s) {
  PlanTotals t{0, 0};
  for (int i = 0; i < in.n_seqs; ++i)
    for (int64_t at = 0; at < in.q_lens[i]; at += s.item_tokens) {
      const int n = (int)std::min<int64_t>(s.item_tokens, in.q_lens[i] - at);
      const int64_t cost = piece_cost(PromptItem{0, n, 0, (int)(in.kv_lens[i] - in.q_lens[i] + at + 1), in.kv_lens[i], 0, 0, 0}, in.dtype, s.few_rows);
      t.cost += cost * in.n_kv_heads;
      t.longest = std::max(t.longest, cost);
    }
  return t;
}
PlanShape shape_of(const PlanInput& in, bool few_rows, bool* fits) {
  const int rows = kRowsFull / in.group;
  PlanShape s;
  s.few_rows = few_rows;
  s.item_tokens = in.dtype == IA_F32 ? (few_rows ? kRowsFew / in.group : rows) : (few_rows ? rows : 2 * rows);
  int64_t n = 0;
  for (int i = 0; i < in.n_seqs; ++i) n += ((int64_t)in.q_lens[i] + s.item_tokens - 1) / s.item_tokens;
  n *= in.n_kv_heads;
  *fits = n <= 0x7fffffff / 64;
  s.n_items = (int)n;
  s.ctas = in.dtype == IA_F32 ? (int)n : (int)std::min<int64_t>(n, sm_count());
  return s;
}
// What merging parts costs: as much as starting a large piece or two, and past two parts an SM the traffic of their rows through
// memory, out and back, at an SM's share of the copy peak.
int64_t merge_cost(const std::vector<PromptItem>& parts, int sms, const PlanInput& in) {
  int64_t rows = 0;
  for (const PromptItem& it : parts) rows += (int64_t)it.n_tok * in.group;
  const int64_t more = std::max<int64_t>(0, rows / sms - 2 * kPartRows);
  return in.dtype == IA_F32 ? 2 * 4 * 32 + more / 3 : 4 * 256 + 5 * more;
}
// Large pieces (128 rows in fp32, two tiles of 128 on the tensor cores) use what they read better, small ones (32, one tile)
// spread a short batch over more SMs: the plan is made for both and the one whose busiest SM ends first is taken.  32 / 8
// heads of 128, small and large pieces, us: fp32 one prompt of 600: 139 and 166, of 900: 301 and 242, 150, 30, 10, 400, 5 and
// 77: 90 and 119, four of 300: 156 and 131; bf16 one of 600: 18.5 and 23.5, of 1700: 45 and 44, four of 300: 22.7 and 19.5,
// three of 700: 37 and 31, 3000 and 2300: 148 and 138.
// Keys whole and cut, us: one token behind 16000: fp32 1742 and 111, bf16 146 and 30; 100 behind 8000: 893 and 476, 80 and 38;
// eight times 4 behind 3000: 334 and 179, 43 and 36; one fp32 prompt of 600: 137 and 114.
//
// With four large pieces an SM or more either kind keeps the SMs busy, so the one whose pieces cost less in all is taken: the large
// ones unless most are nearly empty.  On the tensor cores the small ones have to save an eighth: what they read twice counts
// then.  That is all there is to decide where the costliest piece is at most a third of an SM's work (handing out the longest
// first, the busiest SM then has at most a third too much), or where there are so many pieces that parts of all of them would take
// more than 0.3 GB of workspace; else the search goes on as with few.  Large and whole against what is taken, us, one token each
// behind 500 keys: 74 sequences fp32 516 and 193 (small), bf16 39.6 and 39.9 (small); one of them behind 16000: 3903 and 409 (cut),
// 147 and 67 (cut).  bf16: 100 pieces of 64 behind 200, one behind 30000: 524 and 170 (cut); 512 behind 16000 beside 11 behind
// 188: 317 and 220 (small); a prompt of 2000 and 100 of 30: 56.7 and, small, 59.2 (large is taken).
bool plan_shape(const PlanInput& in, PlanShape* s) {
  bool fits, fits_few;
  *s = shape_of(in, false, &fits);
  const bool many = s->n_items >= 4 * sm_count();
  const auto must_save = [&](int64_t cost) { return many && in.dtype != IA_F32 ? cost / 8 : 0; };
  const PlanShape shapes[2] = {*s, shape_of(in, true, &fits_few)};
  const int sms = sm_count();
  if (!fits || !fits_few) return fits;
  if (many) {
    const PlanTotals totals[2] = {totals_of(in, shapes[0]), totals_of(in, shapes[1])};
    const int few = totals[1].cost < totals[0].cost - must_save(totals[0].cost);
    *s = shapes[few];
    if (3 * sms * totals[few].longest <= totals[few].cost || shapes[0].n_items > kMostParts * sms) return true;
  }
  int64_t q, kv, best = 0, ideal[2] = {0, 0}, keys[2] = {0, 0};
  std::vector<PromptItem> whole[2];
  for (int few = 0; few < 2; ++few) {
    whole[few] = make_pieces(in, shapes[few], &q, &kv);
    for (const PromptItem& it : whole[few]) {
      keys[few] += piece_keys(it);
      ideal[few] += piece_cost(it, in.dtype, few != 0);
    }
    const int64_t cost = spread(whole[few], sms, in.dtype, few != 0, nullptr);
    if (few != 0 && cost >= best - must_save(best)) continue;
    best = cost;
    *s = shapes[few];
  }
  // Few rows and many keys: the keys are cut, for one or two parts an SM.  A slot of the workspace holds one row tile, so on the
  // tensor cores only small pieces are cut.
  for (int few = in.dtype == IA_F32 ? 0 : 1; few < 2; ++few) {
    if (whole[few].empty() || best * sms < ideal[few] + ideal[few] / 3) continue;
    for (int waves = 1; waves <= 2; ++waves) {
      const int chunk = (int)(std::min<int64_t>(keys[few] / (sms * waves) + 128, 1 << 30) / 128 * 128);
      if (chunk >= piece_keys(whole[few][0])) continue;
      const std::vector<PromptItem> parts = cut_pieces(whole[few], chunk, nullptr);
      if ((int64_t)parts.size() > (int64_t)kMostParts * sms) continue;
      const int64_t cost = spread(parts, sms, in.dtype, few != 0, nullptr) + merge_cost(parts, sms, in);
      if (cost >= best) continue;
      best = cost;
      *s = shapes[few];
      s->chunk = chunk;
      s->n_pieces = (int)whole[few].size();
      s->n_items = (int)parts.size();
      s->ctas = in.dtype == IA_F32 ? s->n_items : std::min(s->n_items, sms);
    }
  }
  return true;
}
}  // namespace

int64_t prompt_plan_ints(const int32_t* q_lens, const int32_t* kv_lens, int n_seqs, int n_kv_heads, int group, int dtype) {
  PlanShape s;
  return plan_shape(PlanInput{q_lens, kv_lens, n_seqs, n_kv_heads, group, dtype}, &s) ? s.ints() : -1;
}

int make_prompt_plan(const int32_t* q_lens, const int32_t* kv_lens, int n_seqs, int n_kv_heads, int group, int head_dim, int dtype,
                     int32_t* plan, int64_t plan_ints) {
  const PlanInput in{q_lens, kv_lens, n_seqs, n_kv_heads, group, dtype};
  PlanShape s;
  if (!plan_shape(in, &s) || plan_ints < s.ints()) return fail(IA_ERR_BAD_ARG, "prompt_plan: %lld words", (long long)plan_ints);
  int64_t q0, k0;
  std::vector<PromptItem> items = make_pieces(in, s, &q0, &k0);
  std::vector<PromptPiece> pieces;
  if (s.chunk > 0) items = cut_pieces(items, s.chunk, &pieces);
  std::vector<int> order(s.n_items), begin(s.ctas + 1, 0);
  if (dtype == IA_F32) {  // a CTA each, in this order
    for (int i = 0; i < s.n_items; ++i) order[i] = begin[i] = i;
    begin[s.ctas] = s.n_items;
  } else {  // a list for each SM
    std::vector<int> cta_of;
    spread(items, s.ctas, dtype, s.few_rows, &cta_of);
    for (const int c : cta_of) ++begin[c + 1];
    for (int c = 0; c < s.ctas; ++c) begin[c + 1] += begin[c];
    std::vector<int> next(begin.begin(), begin.end() - 1);
    for (int i = 0; i < s.n_items; ++i) order[next[cta_of[i]]++] = i;
  }
  const int64_t first = s.first();
  const int32_t head[8] = {s.n_items, s.ctas, (s.chunk > 0 ? 2 * s.n_pieces : 0) + s.few_rows, (int32_t)first, group * 1000 + head_dim,
                           n_kv_heads * 16 + dtype, (int32_t)q0, (int32_t)k0};
  std::copy(head, head + 8, plan);
  for (int64_t i = 8; i < first; ++i) plan[i] = begin[std::min<int64_t>(i - 8, s.ctas)];
  for (int i = 0; i < s.n_items; ++i) std::memcpy(plan + first + 8 * (int64_t)i, &items[order[i]], sizeof(PromptItem));
  if (!pieces.empty()) std::memcpy(plan + first + 8 * (int64_t)s.n_items, pieces.data(), pieces.size() * sizeof(PromptPiece));
  return IA_OK;
}

// ---- the plan of the shared-prefix step: a header of 8 words, the entities, then (shared entity, place in it) per sequence
int shared_row_block(int dtype) { return dtype == IA_F32 ? kRowsFull : 2 * kRowsFull; }
static int shared_members(int dtype, int group) { return shared_row_block(dtype) / kRowsFull * (kRowsFull / group); }
int shared_ctas() { return sm_count(); }
int64_t shared_parts(const int32_t* group_sizes, int n_groups, int group, int dtype) {
  const int per = shared_members(dtype, group);
  int64_t n = 0;
  for (int i = 0; i < n_groups; ++i) n += ((int64_t)group_sizes[i] + per - 1) / per;
  return n;
}
void make_shared_plan(const int32_t* group_sizes, int n_groups, int batch, int group, int dtype, int32_t* plan) {
  const int per = shared_members(dtype, group);
  const int n_shared = (int)shared_parts(group_sizes, n_groups, group, dtype);
  SharedEntity* ent = reinterpret_cast<SharedEntity*>(plan + 8);
  int32_t* info = plan + 8 + 8 * ((int64_t)n_shared + batch);
  std::fill(plan, plan + 8, 0);
  plan[0] = n_shared;
  // A unit of many rows takes several times as long as one of few, and shares are equal in units: where there are entities
  // of many rows, those of few get longer units.  16 groups of 8 / 16 / 32 sequences of 4 rows over 4000 keys with 1 to 256
  // own ones: 0.59 / 0.74 / 1.47 ms, with 64 keys throughout 0.62 / 0.95 / 2.14 ms.  Without such entities 64 keys
  // spread a short step over the most SMs.  The tensor-core kernel's unit is its key tile whatever the rows, so there shares are not
  // equal in time where entities of two row tiles stand beside own parts (64 sequences of 8 rows over 128k keys).
  bool wide = false;
  for (int g = 0; g < n_groups; ++g) wide |= std::min(per, group_sizes[g]) * group > kFewRows;
  const auto entity = [&](int first, int n, int group_first, int group_n, int g) {
    const int rows = n * group;
    const int unit = dtype != IA_F32 ? kTensorUnit : !wide ? kKeys : rows <= kFewRows ? 8 * kKeys : rows <= 32 ? 2 * kKeys : kKeys;
    return SharedEntity{first, n, group_first, group_n, g, unit, {0, 0}};
  };
  int seq = 0, e = 0;
  for (int g = 0; g < n_groups; ++g) {
    const int lead = seq;
    for (int m = 0; m < group_sizes[g]; m += per, ++e) {
      const int n = std::min(per, group_sizes[g] - m);
      ent[e] = entity(lead + m, n, lead, group_sizes[g], g);
      for (int i = 0; i < n; ++i) {
        info[2 * (lead + m + i)] = e;
        info[2 * (lead + m + i) + 1] = i;
        ent[n_shared + lead + m + i] = entity(lead + m + i, 1, lead + m + i, 1, g);
      }
    }
    seq += group_sizes[g];
  }
}

}  // namespace ia
