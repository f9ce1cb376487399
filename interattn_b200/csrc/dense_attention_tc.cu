// Dense attention on the 5th-generation tensor cores, bf16: whole prompts and the shared-prefix decode step, one kernel.
//
// A CTA holds two tiles of 128 query rows and streams keys and values in tiles of 128 past both:
//   S_w = Q_w K_j^T     (tcgen05.mma, both operands in shared memory, fp32 result in tensor memory)
//   P_w = exp2(S_w c - m c), l += row sums   (four warps per tile, a thread per row; P is written over S as bf16)
//   O_w += P_w V_j      (tcgen05.mma, P from tensor memory, V from shared memory, O stays in tensor memory)
// A query row is a (token, query head of the kv head): the G heads of a token share its keys, so a tile of 128 / G tokens
// needs K and V once for all of them, and a decode step over a shared prefix is the same computation with sequences in
// the place of tokens.
// The two tiles take turns: while the tensor core works on one tile's products the other's warps take exponentials.
// The running maximum follows the true one only when it has moved by more than 2^8 (weights then stay below 256, exact in
// the sums' fp32 and the same relative rounding in bf16): O is rescaled then, by the warps that own it, which is rare after
// the first tiles.  The weights are rounded to bf16 for the second product, half a step = 2^-8 relative each; their
// sum is taken before the rounding in fp32.
//
// Warps 0-3 and 4-7: softmax, rescaling and output of tile 0 and 1.  Warp 8: copies - it alone knows where work comes from
// (a list for prompts, an equal share of all units for the decode step) and hands the others descriptors through a small
// ring.  Warp 9: one thread issues every MMA.  Tensor memory: S_0, S_1, O_0, O_1 of 128 columns each.
#include <cuda.h>  // CUtensorMap (types only; the encoder is fetched through the runtime)

#include "dense_attention.cuh"

namespace ia {
namespace {

constexpr int kThreads = 320, kRows = 128, kKeys = 128, kWorkSlots = 4;
constexpr int kCopyWarp = 8, kMmaWarp = 9;

template <int D> struct Tc {
  static constexpr int halves = D / 64;                 // 128-byte wide column blocks
  static constexpr int block = kRows * 128;             // bytes of one [128 rows][128 bytes] block
  static constexpr int tile = halves * block;           // a Q, K or V tile
  static constexpr int stages = D == 128 ? 5 : 10;      // ring of K and V tiles
  static constexpr size_t smem = (size_t)(2 + stages) * tile + 1024;
};

// one piece of work, as the copy warp hands it to the others
struct Work {
  int q_tok, n_tok;   // query tokens (prompt) or sequences (decode step)
  int head;
  int tiles[2];       // key tiles for each row tile; 0: none
  int key0;           // first key: an index into the packed keys, or the position in the sequence
  int limit0;         // prompt: keys that the first query token sees
  int n_keys;         // keys from key0 on that anyone sees
  int own;            // decode step: own part (slots of G rows)
  int row;            // decode step: table row
  int64_t slot;
  int last;           // nothing follows
};

struct TcParams {
  CUtensorMap tm_q, tm_k, tm_v;
  PromptTensors t;           // prompt
  const PromptItem* items;
  const int32_t* cta_begin;  // CTA c takes the items [cta_begin[c], cta_begin[c + 1])
  SharedParams s;            // decode step
  int* status;
  int group;
};

// ---- barriers: every wait is bounded ----------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long global_timer_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
constexpr unsigned long long kWaitNs = 2000000000ull;
__device__ __noinline__ bool mbar_wait_slow(uint64_t* bar, uint32_t parity) {
  const unsigned long long start = global_timer_ns();
  do {
    if (mbar_try(bar, parity)) return true;
  } while (global_timer_ns() - start < kWaitNs);
  return false;
}
// false: the phase did not complete in time
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
  return mbar_try(bar, parity) || mbar_try(bar, parity) || mbar_wait_slow(bar, parity);
}

// ---- copies -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, int v, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(smem_u32(bar))
      : "memory");
}

// ---- tensor core ------------------------------------------------------------------------------------------------------
// shared-memory operand of 128-byte rows, 128-byte swizzle, groups of 8 rows 1024 bytes apart (bits 32-45).  Where the
// columns are the contiguous direction of the product (V: keys x dims, read as dims), bits 16-29 hold the distance to
// the next 64 columns.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t next_columns) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(next_columns >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// kind::f16: fp32 accumulate (bit 4), bf16 operands (bits 7, 10), B with its columns contiguous (bit 16), N >> 3 at bit 17,
// M >> 4 at bit 24
template <int N, bool BCols>
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((BCols ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
                            ((uint32_t)(kRows >> 4) << 24);
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// one arrival when every MMA issued so far by this thread has completed
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// lane l of the warp: row (lane of the address) + l; r[i]: column i
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
               "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               :
                 "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                 "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
                 "=r"(r[30]), "=r"(r[31])
               : "r"(taddr));
}
// After the wait the registers of the loads before it may be read.  Naming them ties every use to this point.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               :
                 "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
               "%12, %13, %14, %15, %16};"
               :
               :
                 "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
               "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, "
               "%31, %32};"
               :
               :
                 "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                 "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                 "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
               : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t w;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  return w;
}

struct Bars {
  uint64_t full[10], empty[10], q_full, q_empty, s_full[2], p_full[2], o_full[2], work_full[kWorkSlots], work_empty[kWorkSlots],
      drain;
};

// keys that the row's token sees, counted from the piece's first key
template <bool PAGED> __device__ __forceinline__ int row_limit(const TcParams& p, const Work& wk, int tok) {
  if constexpr (PAGED) return max(0, min(shared_seq_len(p.s, wk.q_tok + tok) - wk.key0, wk.n_keys));
  return max(0, min(wk.limit0 + tok, wk.n_keys));
}

// ---- copy warp: finds the work, fetches Q, K and V --------------------------------------------------------------------
template <int D, bool PAGED>
__device__ __forceinline__ void copy_role(const TcParams& p, Bars* bars, Work* ring, unsigned char* base, SharedCursor cur) {
  using C = Tc<D>;
  const int lane = threadIdx.x & 31, G = p.group, tpm = kRows / G;
  unsigned char* stage0 = base + 2 * C::tile;
  uint32_t it = 0, q_it = 0, w_it = 0;
  bool alive = true;
  int next_item = 0, end_item = 0;
  if constexpr (!PAGED) {
    next_item = p.cta_begin[blockIdx.x];
    end_item = p.cta_begin[blockIdx.x + 1];
  }
  const auto give_up = [&] {
    alive = false;
    if (lane == 0) atomicOr(p.status, IA_DEV_STATUS_ATTEND_WAIT);
  };
  while (alive) {
    Work wk{};
    if constexpr (PAGED) {
      wk.last = cur.left <= 0;
      if (!wk.last) {
        const SharedParams& s = p.s;
        const SharedEntity ent = s.entities[cur.e];
        int lo, hi;
        entity_keys(s, cur.e, ent, lo, hi);
        const int n = (int)min((int64_t)(cur.units - cur.k), cur.left);
        const int2 lead = entity_lead(s, ent, hi);
        wk.q_tok = ent.first_seq;
        wk.n_tok = ent.n_seqs;
        wk.head = cur.h;
        wk.key0 = lo + cur.k * kKeys;
        wk.n_keys = max(0, min(lead.y, wk.key0 + n * kKeys) - wk.key0);
        wk.own = cur.e >= s.n_shared;
        wk.row = lead.x;
        wk.slot = (int64_t)(wk.own ? cur.e - s.n_shared : cur.e) * s.n_kv_heads + cur.h + blockIdx.x;
        wk.tiles[0] = (wk.n_keys + kKeys - 1) / kKeys;
        wk.tiles[1] = ent.n_seqs > tpm ? wk.tiles[0] : 0;
        cur.left -= n;
        cur.k = 0;
        if (++cur.h == s.n_kv_heads) {
          cur.h = 0;
          if (cur.left > 0)  // some entity behind this one has units: they were counted
            do cur.units = entity_units<kKeys>(s, ++cur.e);
            while (cur.units == 0);
        }
      }
    } else {
      wk.last = next_item >= end_item;
      if (!wk.last) {
        const PromptItem item = p.items[next_item++];
        wk.q_tok = item.q_tok;
        wk.n_tok = item.n_tok;
        wk.head = item.head;
        wk.key0 = item.kv_tok;
        wk.limit0 = item.limit0;
        wk.n_keys = item.kv_len;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int toks = min(item.n_tok - w * tpm, tpm);
          if (toks > 0) wk.tiles[w] = (row_limit<false>(p, wk, w * tpm + toks - 1) + kKeys - 1) / kKeys;
        }
      }
    }
    const int slot = w_it % kWorkSlots;
    if (!mbar_wait(&bars->work_empty[slot], ((w_it / kWorkSlots) & 1) ^ 1)) {
      give_up();
      break;
    }
    if (lane == 0) {
      ring[slot] = wk;
      mbar_arrive(&bars->work_full[slot]);
    }
    ++w_it;
    if (wk.last) break;
    const int tiles = max(wk.tiles[0], wk.tiles[1]);
    for (int j = 0; j < tiles; ++j) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {  // K, then V
        if (which == 1 && j == 0) {              // Q behind the first K tile: the ring may be ahead of the last piece's end
          if (!mbar_wait(&bars->q_empty, (q_it & 1) ^ 1)) {
            give_up();
            break;
          }
          if (lane == 0) {
            const int active = (wk.tiles[0] > 0) + (wk.tiles[1] > 0);
            mbar_arrive_expect_tx(&bars->q_full, (uint32_t)(active * C::halves * tpm * G * 128));
#pragma unroll
            for (int w = 0; w < 2; ++w)
              for (int h = 0; wk.tiles[w] > 0 && h < C::halves; ++h)
                tma_load_5d(smem_u32(base + w * C::tile + h * C::block), &p.tm_q, 0, 0, wk.q_tok + w * tpm, h, wk.head,
                            &bars->q_full);
          }
          ++q_it;
        }
        const uint32_t st = it % C::stages;
        unsigned char* dst = stage0 + (size_t)st * C::tile;
        if (!mbar_wait(&bars->empty[st], ((it / C::stages) & 1) ^ 1)) {
          give_up();
          break;
        }
        ++it;
        uint64_t* full = &bars->full[st];
        if constexpr (!PAGED) {
          if (lane == 0) {
            mbar_arrive_expect_tx(full, C::tile);
            tma_load_4d(smem_u32(dst), which == 0 ? &p.tm_k : &p.tm_v, 0, wk.key0 + j * kKeys, 0, wk.head, full);
          }
        } else {
          const int valid = min(kKeys, wk.n_keys - j * kKeys);
          const int pages = which == 0 ? (valid + 15) >> 4 : valid >> 4;
          const int32_t* table = p.s.block_table + (int64_t)wk.row * p.s.max_pages + ((wk.key0 + j * kKeys) >> 4);
          const int page = lane < (valid + 15) >> 4 ? table[lane] : 0;
          const bool bad = page < 0 || (p.s.n_pool_pages > 0 && page >= p.s.n_pool_pages);
          if (bad) atomicOr(p.status, DEV_STATUS_BAD_INDEX);
          if (which == 1 && valid < kKeys) {
            // The last tile of a sequence: behind its last token the page may hold anything, and the tile's other pages
            // whatever the stage held before.  Zero times that must be zero, so the rows are written here.
            const int tail = __shfl_sync(0xffffffffu, bad ? -1 : page, pages & 7);
            const __nv_bfloat16* src = (const __nv_bfloat16*)p.s.v_pool + (int64_t)tail * p.s.page_stride + wk.head * p.s.head_stride;
            for (int i = lane; i < (kKeys - pages * 16) * (D / 8); i += 32) {
              const int row = i / (D / 8), c = i % (D / 8);
              uint4 x = make_uint4(0, 0, 0, 0);
              if (pages * 16 + row < valid && tail >= 0) x = *reinterpret_cast<const uint4*>(src + row * D + c * 8);
              const int pg = pages + (row >> 4), t = row & 15;
              *reinterpret_cast<uint4*>(dst + pg * (C::halves * 2048) + (c >> 3) * 2048 + t * 128 + (((c & 7) ^ (t & 7)) << 4)) = x;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)pages * (C::halves * 2048));
          __syncwarp();
          if (lane < pages) {
            if (which == 0) {  // [128 keys][128 bytes] per half
#pragma unroll
              for (int h = 0; h < C::halves; ++h)
                tma_load_5d(smem_u32(dst + h * C::block + lane * 2048), &p.tm_k, 0, 0, h, wk.head, page, full);
            } else {           // page by page: a k step of the second product is one page
              tma_load_5d(smem_u32(dst + lane * (C::halves * 2048)), &p.tm_v, 0, 0, 0, wk.head, page, full);
            }
          }
          __syncwarp();
        }
      }
      if (!alive) break;
    }
  }
  if (!alive) {  // no copy may be in flight when the CTA ends
    for (uint32_t i = it > C::stages ? it - C::stages : 0; i < it; ++i)
      mbar_wait(&bars->full[i % C::stages], (i / C::stages) & 1);
    if (q_it > 0) mbar_wait(&bars->q_full, (q_it - 1) & 1);
  }
}

// ---- MMA thread -------------------------------------------------------------------------------------------------------
template <int D, bool PAGED>
__device__ __forceinline__ void mma_role(const TcParams& p, Bars* bars, const Work* ring, unsigned char* base, uint32_t tmem) {
  using C = Tc<D>;
  const uint32_t q0 = smem_u32(base), stage0 = q0 + 2 * C::tile;
  constexpr uint32_t kNextCols = PAGED ? 2048 : C::block, kStepBytes = PAGED ? C::halves * 2048 : 2048;
  uint32_t it = 0, q_it = 0, w_it = 0, p_it[2] = {0, 0};
  bool alive = true;
  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (alive && !mbar_wait(bar, parity)) {
      alive = false;
      atomicOr(p.status, IA_DEV_STATUS_ATTEND_WAIT);
    }
    return alive;
  };
  const auto issue_s = [&](int w, uint32_t k) {
    const uint64_t a = umma_desc(q0 + w * C::tile, 0), b = umma_desc(k, 0);
#pragma unroll
    for (int h = 0; h < C::halves; ++h)
#pragma unroll
      for (int s = 0; s < 4; ++s)  // 16 dims = 32 bytes further inside the swizzled row
        umma_ss(tmem + w * 128, a + (h * C::block + s * 32) / 16, b + (h * C::block + s * 32) / 16, kIdesc<kKeys, false>, h + s > 0);
    umma_commit(&bars->s_full[w]);
  };
  while (alive) {
    const int slot = w_it % kWorkSlots;
    if (!wait(&bars->work_full[slot], (w_it / kWorkSlots) & 1)) break;
    const int n0 = ring[slot].tiles[0], n1 = ring[slot].tiles[1], last = ring[slot].last;
    mbar_arrive(&bars->work_empty[slot]);
    ++w_it;
    if (last) break;
    const int tiles = max(n0, n1);
    if (tiles == 0) continue;
    uint32_t st = it % C::stages;
    if (!wait(&bars->full[st], (it / C::stages) & 1) || !wait(&bars->q_full, q_it & 1)) break;
    ++q_it;
    ++it;
    tc_fence_after();
    if (n0 > 0) issue_s(0, stage0 + st * C::tile);
    if (n1 > 0) issue_s(1, stage0 + st * C::tile);
    umma_commit(&bars->empty[st]);
    if (tiles == 1) umma_commit(&bars->q_empty);
    for (int j = 0; j < tiles && alive; ++j) {
      const uint32_t vs = it % C::stages, ks = (it + 1) % C::stages;
      const bool more = j + 1 < tiles;
      if (!wait(&bars->full[vs], (it / C::stages) & 1)) break;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int n = w == 0 ? n0 : n1;
        if (j >= n) continue;
        if (!wait(&bars->p_full[w], p_it[w] & 1)) break;
        ++p_it[w];
        tc_fence_after();
        const uint64_t b = umma_desc(stage0 + vs * C::tile, kNextCols);
#pragma unroll
        for (int s = 0; s < kKeys / 16; ++s)  // 16 keys: 8 columns of packed weights, 16 rows of V
          umma_ts(tmem + 256 + w * 128, tmem + w * 128 + s * 8, b + s * kStepBytes / 16, kIdesc<D, true>, j + s > 0);
        if (j + 1 == n) umma_commit(&bars->o_full[w]);
        if (j + 1 < n) {
          if (!wait(&bars->full[ks], ((it + 1) / C::stages) & 1)) break;
          tc_fence_after();
          issue_s(w, stage0 + ks * C::tile);
        }
      }
      if (!alive) break;
      umma_commit(&bars->empty[vs]);
      if (more) {
        umma_commit(&bars->empty[ks]);
        if (j + 2 == tiles) umma_commit(&bars->q_empty);
      }
      it += more ? 2 : 1;
    }
  }
  umma_commit(&bars->drain);  // no MMA, and no arrival of one, may be in flight when the CTA ends
  if (!mbar_wait(&bars->drain, 0)) atomicOr(p.status, IA_DEV_STATUS_ATTEND_WAIT);
}

// ---- softmax warps ----------------------------------------------------------------------------------------------------
template <int D, bool PAGED>
__device__ __forceinline__ void softmax_role(const TcParams& p, Bars* bars, const Work* ring, uint32_t tmem) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = warp >> 2, row = (warp & 3) * 32 + lane;
  const int G = p.group, tpm = kRows / G, tok = w * tpm + row / G, g = row % G;
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const uint32_t s_addr = tmem + lanes + w * 128, o_addr = tmem + lanes + 256 + w * 128;
  const float c = kLog2e * rsqrtf((float)D);
  uint32_t s_it = 0, o_it = 0;
  const auto wait = [&](uint64_t* bar, uint32_t parity) {  // the whole warp goes on or none of it
    const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity));
    if (!ok && lane == 0) atomicOr(p.status, IA_DEV_STATUS_ATTEND_WAIT);
    return ok;
  };
  for (uint32_t w_it = 0;; ++w_it) {
    const int slot = w_it % kWorkSlots;
    if (!wait(&bars->work_full[slot], (w_it / kWorkSlots) & 1)) return;
    const Work wk = ring[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->work_empty[slot]);
    if (wk.last) return;
    const int n = wk.tiles[w];
    const bool valid = row < tpm * G && tok < wk.n_tok;
    const bool busy = __any_sync(0xffffffffu, valid);
    const int limit = valid ? row_limit<PAGED>(p, wk, tok) : 0;
    const int least = __reduce_min_sync(0xffffffffu, limit);  // below it nothing is masked for the warp
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < n; ++j) {
      if (!wait(&bars->s_full[w], s_it & 1)) return;
      ++s_it;
      if (busy) {
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld(s_addr + 32 * i, s[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_wait_ld(s[i]);
        const int seen = limit - j * kKeys;
        if (least < (j + 1) * kKeys) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (32 * i + k >= seen) s[i][k] = 0xff800000u;  // -inf
        }
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          top[i] = __uint_as_float(s[i][0]);
#pragma unroll
          for (int k = 1; k < 31; k += 2) top[i] = fmaxf(fmaxf(top[i], __uint_as_float(s[i][k])), __uint_as_float(s[i][k + 1]));
          top[i] = fmaxf(top[i], __uint_as_float(s[i][31]));
        }
        const float t = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if (j == 0) {
          m = t;
        } else {
          const bool far = (t - m) * c > 8.f;  // also where m is still -inf
          if (__any_sync(0xffffffffu, far)) {
            const float keep = far ? exp2_fast((m - t) * c) : 1.f;
            if (far) {
              m = t;
              l *= keep;
            }
            uint32_t o[32];
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {  // the products of the tile before are complete: S of this one came after them
              tmem_ld(o_addr + 32 * i, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
              tmem_st(o_addr + 32 * i, o);
            }
          }
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t packed[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float a = exp2_fast(fmaf(__uint_as_float(s[i][k]), c, -mc)), b = exp2_fast(fmaf(__uint_as_float(s[i][k + 1]), c, -mc));
            sum[(k >> 1) & 3] += a + b;
            packed[k >> 1] = pack_bf16(a, b);
          }
          tmem_st(s_addr + 16 * i, packed);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_full[w]);
    }
    if (n > 0) {
      if (!wait(&bars->o_full[w], o_it & 1)) return;
      ++o_it;
      tc_fence_after();
    }
    if (!busy) continue;
    // ---- output ----
    const int hq = p.group * (PAGED ? p.s.n_kv_heads : p.t.n_kv_heads);
    const bool empty = limit <= 0;
    const float inv = empty ? 0.f : 1.f / l;
    const float lse = empty ? -INFINITY : (m * c + __log2f(l)) * kLn2;
    __nv_bfloat16* out = nullptr;
    float* part = nullptr;
    float* lse_out = nullptr;
    if constexpr (PAGED) {
      const int64_t at = wk.slot * (wk.own ? G : p.s.row_block) + tok * G + g;
      part = (wk.own ? p.s.o_own : p.s.o_shared) + at * D;
      lse_out = (wk.own ? p.s.lse_own : p.s.lse_shared) + at;
    } else {
      const int64_t at = (int64_t)(wk.q_tok + tok) * hq + wk.head * G + g;
      out = (__nv_bfloat16*)p.t.out + at * D;
      lse_out = p.t.lse == nullptr ? nullptr : p.t.lse + at;
    }
    bool finite = true;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      uint32_t o[32];
      if (n > 0) {
        tmem_ld(o_addr + 32 * i, o);
        tmem_wait_ld(o);
      }
      float x[32];
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        x[k] = empty ? 0.f : __uint_as_float(o[k]) * inv;
        finite &= fabsf(x[k]) <= 3.4028235e38f;
      }
      if (valid) {
        if constexpr (PAGED) {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            *reinterpret_cast<float4*>(part + 32 * i + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
        } else {
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            *reinterpret_cast<uint4*>(out + 32 * i + k) = make_uint4(pack_bf16(x[k], x[k + 1]), pack_bf16(x[k + 2], x[k + 3]),
                                                                     pack_bf16(x[k + 4], x[k + 5]), pack_bf16(x[k + 6], x[k + 7]));
        }
      }
    }
    if (valid && lse_out != nullptr) *lse_out = lse;
    const unsigned bad = __ballot_sync(0xffffffffu, valid && !finite);
    if (bad != 0) {  // see exact_row
      const auto redo = [&](const auto& key, const __nv_bfloat16* q) {
        const int end = PAGED ? wk.n_keys : n * kKeys;
        const int last = last_not_finite<__nv_bfloat16, D>(least, end, key);
        for (int r = 0; r < 32; ++r) {
          const int lim = __shfl_sync(0xffffffffu, limit, r);
          if (!((bad >> r) & 1) || last < lim) continue;
          const uint64_t q_row = __shfl_sync(0xffffffffu, (unsigned long long)q, r);
          float x[D / 32], mx, lx;
          exact_row<__nv_bfloat16, D>((const __nv_bfloat16*)q_row, 0, lim, c, key, x, mx, lx);
          const uint64_t to = __shfl_sync(0xffffffffu, PAGED ? (unsigned long long)part : (unsigned long long)out, r);
          float* lse_to = (float*)__shfl_sync(0xffffffffu, (unsigned long long)lse_out, r);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            if constexpr (PAGED) ((float*)to)[lane + 32 * i] = x[i] / lx;
            else ((__nv_bfloat16*)to)[lane + 32 * i] = __float2bfloat16_rn(x[i] / lx);
          }
          if (lane == 0 && lse_to != nullptr) *lse_to = (mx + __log2f(lx)) * kLn2;
        }
      };
      __syncwarp();
      using T = __nv_bfloat16;
      if constexpr (PAGED) {
        const PagedKeys<T> key{(const T*)p.s.k_pool + wk.head * p.s.head_stride, (const T*)p.s.v_pool + wk.head * p.s.head_stride,
                               p.s.block_table + (int64_t)wk.row * p.s.max_pages + (wk.key0 >> 4), p.s.page_stride, D,
                               p.s.n_pool_pages, p.s.max_pages - (wk.key0 >> 4)};
        redo(key, (const T*)p.s.q + ((int64_t)(wk.q_tok + tok) * hq + wk.head * G + g) * D);
      } else {
        const PackedKeys<T> key{(const T*)p.t.k + wk.key0 * p.t.k_tok_stride + wk.head * p.t.k_head_stride,
                                (const T*)p.t.v + wk.key0 * p.t.v_tok_stride + wk.head * p.t.v_head_stride, p.t.k_tok_stride,
                                p.t.v_tok_stride, p.t.n_kv_tok - wk.key0};
        redo(key, (const T*)p.t.q + (int64_t)(wk.q_tok + tok) * p.t.q_tok_stride + (int64_t)(wk.head * G + g) * p.t.q_head_stride);
      }
    }
  }
}

template <int D, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1) attend_tc_kernel(const __grid_constant__ TcParams p) {
  using C = Tc<D>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Bars bars;
  __shared__ Work ring[kWorkSlots];
  __shared__ uint32_t tmem_s;
  __shared__ unsigned long long scratch[kThreads / 32];
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::stages; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&bars.s_full[w], 1);
      mbar_init(&bars.p_full[w], 4);  // a lane of each warp
      mbar_init(&bars.o_full[w], 1);
    }
    for (int i = 0; i < kWorkSlots; ++i) {
      mbar_init(&bars.work_full[i], 1);
      mbar_init(&bars.work_empty[i], 9);  // eight softmax warps and the MMA thread
    }
    mbar_init(&bars.drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  grid_dependency_wait();
  grid_launch_dependents();
  SharedCursor cur{};
  if constexpr (PAGED) cur = find_share<kKeys, kThreads>(p.s, blockIdx.x, gridDim.x, scratch);
  if (warp == kCopyWarp) {
    copy_role<D, PAGED>(p, &bars, ring, base, cur);
  } else if (warp == kMmaWarp) {
    if ((threadIdx.x & 31) == 0) mma_role<D, PAGED>(p, &bars, ring, base, tmem);
  } else {
    softmax_role<D, PAGED>(p, &bars, ring, tmem);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ---- host -------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static EncodeFn fn = nullptr;  // every thread would store the same pointer
  if (fn == nullptr) {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &found) == cudaSuccess &&
        found == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(sym);
  }
  return fn;
}
// strides in elements, of the dimensions behind the first; the first is 64 elements, the width of a swizzled row
template <int N>
int encode(CUtensorMap* tm, const void* base, const int64_t (&dims)[N], const int64_t (&strides)[N - 1], const int (&box)[N]) {
  EncodeFn enc = encoder();
  if (enc == nullptr) return fail(IA_ERR_LAUNCH, "dense attention: cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t d[N], s[N - 1];
  cuuint32_t b[N], one[N];
  for (int i = 0; i < N; ++i) {
    d[i] = (cuuint64_t)dims[i];
    b[i] = (cuuint32_t)box[i];
    one[i] = 1;
    if (i > 0) s[i - 1] = (cuuint64_t)strides[i - 1] * 2;
  }
  const CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, N, const_cast<void*>(base), d, s, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? IA_OK : fail(IA_ERR_LAUNCH, "dense attention: cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
}
int encode_q(CUtensorMap* tm, const void* q, int head_dim, int group, int n_kv_heads, int64_t tokens, int64_t tok_stride,
             int64_t head_stride) {
  return encode<5>(tm, q, {64, group, tokens, head_dim / 64, n_kv_heads}, {head_stride, tok_stride, 64, group * head_stride},
                   {64, group, kRows / group, 1, 1});
}

template <int D, bool PAGED> int launch_tc(const TcParams& p, int grid, cudaStream_t stream) {
  auto kern = attend_tc_kernel<D, PAGED>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Tc<D>::smem);
  if (e != cudaSuccess) return fail(IA_ERR_LAUNCH, "dense attention: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  e = launch_overlapped(kern, (unsigned)grid, (unsigned)kThreads, Tc<D>::smem, stream, p);
  return e == cudaSuccess ? check_launch("attend_tc_kernel") : fail(IA_ERR_LAUNCH, "attend_tc_kernel: %s", cudaGetErrorString(e));
}

}  // namespace

int launch_prompt_tc(const PromptTensors& t, int head_dim, const PromptItem* items, const int32_t* cta_begin, int ctas,
                     cudaStream_t stream) {
  TcParams p{};
  p.t = t;
  p.items = items;
  p.cta_begin = cta_begin;
  p.group = t.group;
  p.status = device_status_address();
  if (p.status == nullptr) return IA_ERR_LAUNCH;
  if (int s = encode_q(&p.tm_q, t.q, head_dim, t.group, t.n_kv_heads, t.n_q_tok, t.q_tok_stride, t.q_head_stride)) return s;
  if (t.n_kv_tok > 0) {
    const int64_t dims[4] = {64, t.n_kv_tok, head_dim / 64, t.n_kv_heads};
    const int box[4] = {64, kKeys, head_dim / 64, 1};
    const int64_t ks[3] = {t.k_tok_stride, 64, t.k_head_stride}, vs[3] = {t.v_tok_stride, 64, t.v_head_stride};
    if (int s = encode<4>(&p.tm_k, t.k, dims, ks, box)) return s;
    if (int s = encode<4>(&p.tm_v, t.v, dims, vs, box)) return s;
  }
  return head_dim == 128 ? launch_tc<128, false>(p, ctas, stream) : launch_tc<64, false>(p, ctas, stream);
}

int launch_shared_tc(const SharedParams& s, int head_dim, int ctas, cudaStream_t stream) {
  TcParams p{};
  p.s = s;
  p.group = s.group;
  p.status = s.status;
  const int64_t hq = (int64_t)s.n_kv_heads * s.group;
  if (int r = encode_q(&p.tm_q, s.q, head_dim, s.group, s.n_kv_heads, s.batch, hq * head_dim, head_dim)) return r;
  const int64_t dims[5] = {64, 16, head_dim / 64, s.n_kv_heads, s.n_pool_pages > 0 ? s.n_pool_pages : 0x7fffffff};
  const int64_t strides[4] = {head_dim, 64, s.head_stride, s.page_stride};
  const int k_box[5] = {64, 16, 1, 1, 1}, v_box[5] = {64, 16, head_dim / 64, 1, 1};
  if (int r = encode<5>(&p.tm_k, s.k_pool, dims, strides, k_box)) return r;
  if (int r = encode<5>(&p.tm_v, s.v_pool, dims, strides, v_box)) return r;
  return head_dim == 128 ? launch_tc<128, true>(p, ctas, stream) : launch_tc<64, true>(p, ctas, stream);
}

}  // namespace ia
