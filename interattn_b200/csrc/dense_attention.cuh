// Dense attention over all keys: the prompt (packed sequences, causal) and the decode step of sequences that share a
// prefix.  What the fp32 kernel (dense_attention.cu) and the tensor-core kernel (dense_attention_tc.cu) have in common:
// the pieces of work, how the decode step is cut into equal shares, and the exact form of a single row.
#pragma once

#include <atomic>

#include "ia_common.cuh"

namespace ia {

// One piece of a prompt: n_tok consecutive query tokens of one sequence and one kv head (n_tok * G query rows).
// Query token t of the piece sees the first clamp(limit0 + t, 0, kv_len) keys of its sequence.
struct PromptItem {
  int32_t q_tok;    // first query token, an index into the packed queries
  int32_t n_tok;
  int32_t kv_tok;   // first key token of the sequence, an index into the packed keys
  int32_t limit0;   // visible keys of the first query token; may be <= 0
  int32_t kv_len;
  int32_t head;     // kv head
  int32_t slot;     // a part of the keys: which kPartRows rows of the workspace it fills
  int32_t reserved;
};
static_assert(sizeof(PromptItem) == 32, "read as two 16-byte words");
// Few query rows and many keys: the keys of a piece are cut into parts of about equal length, items whose sequence is the
// part, and the parts' outputs and log-sum-exps are merged.
struct PromptPiece {
  int32_t q_tok, n_tok, head;
  int32_t slot, parts;  // its parts fill the slots [slot, slot + parts)
  int32_t reserved[3];
};
static_assert(sizeof(PromptPiece) == 32, "eight words of the plan");
constexpr int kPartRows = 128;

// Tensors of a prompt call; strides in elements, the D elements of one (token, head) contiguous.
struct PromptTensors {
  const void *q, *k, *v;
  void* out;        // [q tokens, n_q_heads, D] contiguous
  float* lse;       // [q tokens, n_q_heads], may be null
  int64_t q_tok_stride, q_head_stride, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride;
  int32_t n_q_tok, n_kv_tok, n_kv_heads, group;
  float *part_o, *part_lse;  // [slots, kPartRows, D] and [slots, kPartRows]; null: pieces are not cut
};

// ---- the decode step of sequences that share a prefix ---------------------------------------------------------------
// Entities: first the shared parts (consecutive members of a group, at most as many as fill a row block), then one own
// part per sequence.  A shared part covers the keys [0, split) of its group, split = shared_len rounded down to whole
// pages, read through the table row of the longest member (the first that holds the whole prefix, where one does: any
// member may have left); an own part covers [split, seq_len) of its sequence.
// An item is an (entity, kv head), its keys are cut into units (the tensor-core kernel: kUnit keys; fp32: as many as the
// plan says for the entity, so that units of many and of few rows take about as long), and CTA c of P takes the units
// [T c / P, T (c + 1) / P) of all T units laid end to end: equal shares whatever the lengths are, one run of keys per
// CTA and item.  Each (item, CTA) leaves a normalised partial output and its log-sum-exp: the segment that begins the item in
// the item's own rows, another in rows of the CTA - only the first segment of a CTA can begin inside an item.
constexpr int kTensorUnit = 128;
struct SharedEntity {
  int32_t first_seq, n_seqs;    // whose query rows
  int32_t group_first, group_n; // whose table rows may be read
  int32_t group;
  int32_t unit;                 // keys of a unit
  int32_t reserved[2];
};
static_assert(sizeof(SharedEntity) == 32, "eight words of the plan");
struct SharedParams {
  const void *q, *k_pool, *v_pool;
  const int32_t *block_table, *seq_lens, *shared_lens;
  const SharedEntity* entities;  // [n_shared + batch]
  float *o, *lse;                // partial rows: of the shared items, of the own items, row_block for every CTA
  long long* unit_begin;         // [n_shared + batch + 1] where the entities' units begin; written for the merge
  int* status;
  int64_t page_stride, head_stride;  // elements
  int32_t n_shared, batch, n_kv_heads, group, max_pages, n_pool_pages, row_block;
};

// where the partial rows of an item begin
__device__ __forceinline__ int64_t item_rows(const SharedParams& p, bool own, int first_seq, int n_seqs, int head) {
  const int64_t all = (int64_t)p.batch * p.n_kv_heads * p.group;
  return own ? all + ((int64_t)first_seq * p.n_kv_heads + head) * p.group
             : ((int64_t)first_seq * p.n_kv_heads + (int64_t)head * n_seqs) * p.group;
}
__device__ __forceinline__ int64_t cta_rows(const SharedParams& p, int cta) {
  return 2 * (int64_t)p.batch * p.n_kv_heads * p.group + (int64_t)cta * p.row_block;
}
__device__ __forceinline__ int shared_split(const SharedParams& p, int group) {
  return max(0, min(p.shared_lens[group], p.max_pages * 16)) & ~15;
}
__device__ __forceinline__ int shared_seq_len(const SharedParams& p, int seq) {
  return max(0, min(p.seq_lens[seq], p.max_pages * 16));
}
// the keys [lo, hi) of an entity
__device__ __forceinline__ void entity_keys(const SharedParams& p, int e, const SharedEntity& ent, int& lo, int& hi) {
  const int split = shared_split(p, ent.group);
  if (e < p.n_shared) {
    lo = 0;
    hi = split;
  } else {
    lo = split;
    hi = max(split, shared_seq_len(p, ent.first_seq));
  }
}
// The sequence whose table row an entity is read through, and how many of the keys [0, hi) that row holds.  By whole warps.
__device__ __forceinline__ int2 entity_lead(const SharedParams& p, const SharedEntity& ent, int hi) {
  int best = -1, who = 0;
  for (int i = threadIdx.x & 31; i < ent.group_n; i += 32) {
    const int len = min(hi, shared_seq_len(p, ent.group_first + i));
    if (len > best) {
      best = len;
      who = i;
    }
  }
  const int top = __reduce_max_sync(0xffffffffu, best);
  who = __reduce_min_sync(0xffffffffu, best == top ? who : 0x7fffffff);
  return make_int2(ent.group_first + who, top);
}
__device__ __forceinline__ SharedEntity load_entity(const SharedParams& p, int e) {  // two 16-byte loads
  union {
    int4 v[2];
    SharedEntity e;
  } u;
  u.v[0] = reinterpret_cast<const int4*>(p.entities + e)[0];
  u.v[1] = reinterpret_cast<const int4*>(p.entities + e)[1];
  return u.e;
}
template <int kUnit> __device__ __forceinline__ int entity_units(const SharedParams& p, int e) {  // kUnit 0: the plan's
  const SharedEntity ent = load_entity(p, e);
  int lo, hi;
  entity_keys(p, e, ent, lo, hi);
  const int unit = kUnit > 0 ? kUnit : ent.unit;
  return (hi - lo + unit - 1) / unit;
}
// no share is empty: between the first and the last CTA of an item every slot is written
__device__ __forceinline__ int shares_of(int64_t total, int ctas) { return total < ctas ? (int)total : ctas; }
__device__ __forceinline__ int64_t share_begin(int64_t total, int c, int ctas) { return total * c / ctas; }
// the CTA whose share holds unit x
__device__ __forceinline__ int share_owner(int64_t x, int64_t total, int ctas) {
  return (int)(((x + 1) * ctas + total - 1) / total) - 1;
}

// Where a CTA's share starts: entity, kv head, unit inside the item.
struct SharedCursor {
  int e, h, k, units;   // units of this item
  int64_t left;         // units of the share that are left
};

// Called by all kThreads threads of the CTA; `scratch`: kThreads / 32 64-bit words of shared memory, at least 3.
template <int kUnit, int kThreads>
__device__ __forceinline__ SharedCursor find_share(const SharedParams& p, int cta, int ctas, unsigned long long* scratch) {
  const int tid = threadIdx.x, lane = tid & 31;
  const int n = p.n_shared + p.batch, per = (n + kThreads - 1) / kThreads;
  const int e0 = min(n, tid * per), e1 = min(n, e0 + per);
  long long sum = 0;
  for (int e = e0; e < e1; ++e) sum += (long long)entity_units<kUnit>(p, e) * p.n_kv_heads;
  long long upto = sum;  // inclusive within the warp
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, w);
    if (lane >= w) upto += x;
  }
  if (lane == 31) scratch[tid >> 5] = (unsigned long long)upto;
  __syncthreads();
  long long before = upto - sum, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const long long x = (long long)scratch[w];
    if (w < (tid >> 5)) before += x;
    total += x;
  }
  __syncthreads();
  if (cta == 0) {
    long long at = before;
    for (int e = e0; e < e1; ++e) {
      p.unit_begin[e] = at;
      at += (long long)entity_units<kUnit>(p, e) * p.n_kv_heads;
    }
    if (tid == 0) p.unit_begin[n] = total;
  }
  ctas = shares_of(total, ctas);
  const long long u0 = cta < ctas ? share_begin(total, cta, ctas) : 0, u1 = cta < ctas ? share_begin(total, cta + 1, ctas) : 0;
  SharedCursor* found = reinterpret_cast<SharedCursor*>(scratch);
  if (u0 < u1 && u0 >= before && u0 < before + sum) {
    long long at = before;
    for (int e = e0; e < e1; ++e) {
      const int units = entity_units<kUnit>(p, e);
      const long long span = (long long)units * p.n_kv_heads;
      if (u0 < at + span) {
        const long long off = u0 - at;
        *found = SharedCursor{e, (int)(off / units), (int)(off % units), units, u1 - u0};
        break;
      }
      at += span;
    }
  }
  if (tid == 0 && u0 >= u1) *found = SharedCursor{0, 0, 0, 0, 0};
  __syncthreads();
  const SharedCursor c = *found;
  __syncthreads();
  return c;
}

// ---- one row, exactly as the formula has it -------------------------------------------------------------------------
// The tiled kernels multiply masked places by a weight of zero, and zero times an infinity or a NaN is a NaN.  A row whose
// result is not finite is therefore looked at again: if a value row that the row's tiles held but the row does not see is
// not finite, the row is redone here from the keys it sees.  Key(j) gives the addresses of key and value row j.
template <typename T, int D> __device__ __forceinline__ bool row_not_finite(const T* v) {  // by one thread
  bool bad = false;
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    float x[4];
    load_vec<4>(v + d, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) bad |= !(fabsf(x[e]) <= 3.4028235e38f);
  }
  return bad;
}
// The last key in [lo, hi) whose value row is not finite, or -1, by a whole warp, a lane a key.  Where several warps share the search,
// this one takes the 32 keys from lo + first on and every `step` after.
template <typename T, int D, typename Key> __device__ __forceinline__ int last_not_finite(int lo, int hi, const Key& key, int first = 0, int step = 32) {
  int last = -1;
  for (int64_t j = (int64_t)lo + first + (threadIdx.x & 31); j < hi; j += step) {
    const T *k, *v;
    if (key((int)j, k, v) && row_not_finite<T, D>(v)) last = (int)j;
  }
#pragma unroll  // not one instruction: with it here the assembler finds no registers for the fp32 kernel
  for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
  return last;
}
template <int N> __device__ __forceinline__ void unpack16(const uint4& w, float (&x)[N]) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (N == 8) {
      x[2 * i] = bf16lo(r[i]);
      x[2 * i + 1] = bf16hi(r[i]);
    } else {
      x[i] = __uint_as_float(r[i]);
    }
  }
}
// softmax(q . k_j * scale) v_j over [lo, hi) by a whole warp: a lane takes every 32nd key's logit, then the dims l, l + 32, ... of the
// values.  Bound by the latency of its loads: kAhead of them are on their way together, as many as the kernel has registers for.  A
// row whose every dim is NaN stays so: it ends there, with m and l of the keys so far.  (The log-sum-exp needs no second look:
// what a row does not see never got into its logits.)
template <typename T, int D, int kAhead, typename Key>
__device__ __forceinline__ void exact_row(const T* q, int lo, int hi, float scale_log2, const Key& key, float (&o)[D / 32], float& m,
                          float& l) {
  constexpr int kVec = 16 / sizeof(T), kLoads = D / kVec < kAhead ? D / kVec : kAhead;
  const int lane = threadIdx.x & 31;
  float qv[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    qv[i] = to_f32(q[lane + 32 * i]) * scale_log2;
    o[i] = 0.f;
  }
  m = -INFINITY;
  l = 0.f;
#pragma unroll 1
  for (int64_t j0 = lo; j0 < hi; j0 += 32) {
    const T *k = q, *v = q;
    const bool seen = j0 + lane < hi && key((int)j0 + lane, k, v);
    float s = 0.f;
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += kLoads * kVec) {
      uint4 raw[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) raw[i] = seen ? *reinterpret_cast<const uint4*>(k + d0 + i * kVec) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        float x[kVec];
        unpack16(raw[i], x);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const int d = d0 + i * kVec + e;
          s += __shfl_sync(0xffffffffu, qv[d / 32], d % 32) * x[e];
        }
      }
    }
    if (!seen) s = -INFINITY;
    const float m_new = fmaxf(m, warp_max(s));
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float keep = exp2f(m - base), w = exp2f(s - base);
    l = l * keep + (seen ? w : 0.f);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] *= keep;
    const unsigned which = __ballot_sync(0xffffffffu, seen);
#pragma unroll 1
    for (int s0 = 0; s0 < 32; s0 += kAhead) {
      T x[kAhead][D / 32];
#pragma unroll
      for (int s1 = 0; s1 < kAhead; ++s1) {
        const T* from = (const T*)__shfl_sync(0xffffffffu, (unsigned long long)v, s0 + s1);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) x[s1][i] = from[lane + 32 * i];  // of a key that is not seen: the query, unused
      }
#pragma unroll
      for (int s1 = 0; s1 < kAhead; ++s1) {
        const float ws = __shfl_sync(0xffffffffu, w, s0 + s1);
        if (which >> (s0 + s1) & 1) {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) o[i] += ws * to_f32(x[s1][i]);
        }
      }
    }
    m = m_new;
    bool lost = true;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) lost &= o[i] != o[i];
    if (__all_sync(0xffffffffu, lost)) break;
  }
  l = warp_sum(l);
}

template <typename T> struct PackedKeys {  // the keys of one sequence and kv head
  const T *k, *v;
  int64_t k_stride, v_stride;
  int n;
  __device__ __forceinline__ bool operator()(int j, const T*& kr, const T*& vr) const {
    if (j >= n) return false;
    kr = k + j * k_stride;
    vr = v + j * v_stride;
    return true;
  }
};
template <typename T> struct PagedKeys {
  const T *k, *v;          // pools at the kv head
  const int32_t* table;    // the sequence's row
  int64_t page_stride;
  int head_dim, n_pages, max_pages;  // n_pages 0: unknown, entries are trusted
  __device__ __forceinline__ bool operator()(int j, const T*& kr, const T*& vr) const {
    if ((j >> 4) >= max_pages) return false;
    const int page = table[j >> 4];
    if (page < 0 || (n_pages > 0 && page >= n_pages)) return false;
    const int64_t at = page * page_stride + (int64_t)(j & 15) * head_dim;
    kr = k + at;
    vr = v + at;
    return true;
  }
};

// ---- launchers ------------------------------------------------------------------------------------------------------
int sm_count();
struct SmemOnce {  // a kernel's shared memory, allowed once per device
  std::atomic<uint64_t> done{0};
  int allow(const void* kern, size_t bytes, const char* what);
};
int64_t prompt_plan_ints(const int32_t* q_lens, const int32_t* kv_lens, int n_seqs, int n_kv_heads, int group,
                         int dtype);  // -1: too large
int make_prompt_plan(const int32_t* q_lens, const int32_t* kv_lens, int n_seqs, int n_kv_heads, int group, int head_dim, int dtype,
                     int32_t* plan, int64_t plan_ints);
int shared_row_block(int dtype);  // query rows of a shared part, at most
int shared_ctas();
int64_t shared_parts(const int32_t* group_sizes, int n_groups, int group, int dtype);
void make_shared_plan(const int32_t* group_sizes, int n_groups, int batch, int group, int dtype, int32_t* plan);

int launch_prompt_f32(const PromptTensors& t, int head_dim, const PromptItem* items, int n_items, bool few_rows,
                      cudaStream_t stream);
int launch_prompt_merge(const PromptTensors& t, int head_dim, int dtype, const PromptPiece* pieces, int n_pieces, bool few_rows,
                        cudaStream_t stream);
int launch_shared_f32(const SharedParams& p, int head_dim, int ctas, cudaStream_t stream);
int launch_prompt_tc(const PromptTensors& t, int head_dim, const PromptItem* items, const int32_t* cta_begin, int ctas,
                     cudaStream_t stream);
int launch_shared_tc(const SharedParams& p, int head_dim, int ctas, cudaStream_t stream);
int launch_shared_merge(const SharedParams& p, const int32_t* seq_info, int head_dim, int dtype, int ctas, void* out,
                        cudaStream_t stream);

}  // namespace ia
