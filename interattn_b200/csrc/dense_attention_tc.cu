// Dense attention on the 5th-generation tensor cores, bf16: whole prompts and the shared-prefix decode step, one kernel.
//
// A CTA holds two tiles of 128 query rows and streams keys and values in tiles of 128 past both:
//   S_w = Q_w K_j^T     (tcgen05.mma, both operands in shared memory, fp32 result in tensor memory)
//   P_w = exp2(S_w c - m c), l += row sums   (four warps per tile, a thread per row; P is written over S as bf16)
//   O_w += P_w V_j      (tcgen05.mma, P from tensor memory, V from shared memory, O stays in tensor memory)
// A query row is a (token, query head of the kv head): the G heads of a token share its keys, so a tile of 128 / G tokens
// needs K and V once for all of them, and a decode step over a shared prefix is the same computation with sequences in
// the place of tokens.
// The two sets of softmax warps take turns with the tensor core: while it works on one's products the other takes
// exponentials.  Where a piece fills both row tiles each set has a tile and both see every key tile; where it fills only one
// (a decode step of few rows, a short prompt) the key tiles alternate between the sets, each with its own running maximum,
// sum and O, which are merged at the end: row and lane are the same in both, so either set reads the other's O from
// tensor memory.  In both cases the key tiles' steps run 0, 1, 0, 1, ... over the sets and across pieces, so the next
// piece's first products start while the last one's outputs are written.
// The running maximum follows the true one only when it has moved by more than 2^8 (weights then stay below 256, exact in
// the sums' fp32 and the same relative rounding in bf16): O is rescaled then, by the warps that own it, which is rare after
// the first tiles.  The weights are rounded to bf16 for the second product, half a step = 2^-8 relative each; their
// sum is taken before the rounding in fp32.
//
// Warps 0-3 and 4-7: softmax, rescaling and output of tile 0 and 1.  Warp 8: copies - it alone knows where work comes from
// (a list for prompts, an equal share of all units for the decode step) and hands the others descriptors through a small
// ring.  Warps 9 and 10 issue the MMAs of set 0 and 1, a set's second product and its next first product together: issuing
// holds a warp until the tensor core takes the instruction, so what one decides and waits for between them is hidden behind
// the other's.  Tensor memory: S_0, S_1, O_0, O_1 of 128 columns each.
//
// Measured at the Llama-3-8B heads, in a queue of passes: one 32k prompt 9.0 ms (0.97 PFLOP/s, 0.57 of the measured GEMM peak as a burst
// and 0.69 of the sustained one; the power cap holds the clock), one of 8k 0.57 ms, bound by a tile's chain of products and
// exponentials; a decode step of 64 sequences in eight groups, 955 MB, 234 us in this kernel (0.63 of the copy peak), a key
// tile taking 1.6 us an SM once the ring runs.
#include <type_traits>

#include <cuda.h>  // CUtensorMap (types only; the encoder is fetched through the runtime)

#include "dense_attention.cuh"

namespace ia {
namespace {

constexpr int kThreads = 352, kRows = 128, kKeys = kTensorUnit, kWorkSlots = 8;
constexpr int kCopyWarp = 8, kMmaWarp = 9;  // and 10

template <int D> struct Tc {
  static constexpr int halves = D / 64;                 // 128-byte wide column blocks
  static constexpr int block = kRows * 128;             // bytes of one [128 rows][128 bytes] block
  static constexpr int tile = halves * block;           // a Q tile
  static constexpr int kv_block = kKeys * 128, kv_tile = halves * kv_block;
  static constexpr int stages = D == 128 ? 4 : 8;      // ring of K and V tiles
  static constexpr int out_warp = 4096;                 // a warp's 32 rows of 128 bytes on their way out
  static constexpr size_t ring = 2 * (size_t)tile, tiles = ring + (size_t)stages * kv_tile, control = tiles + 8 * out_warp, smem = control + 3 * 1024;
};

// The key tiles of a piece and who takes them.  Split: one row tile, key tile j goes to set (first + j) % 2 of softmax warps.
// Else: row tile r goes to set (first + r) % 2, with all its key tiles.  Tile j's K is fetch ring + 2 j, its V the one behind.
struct Order {
  int split;
  int keys[2];        // keys that each row tile sees, at least 1; the second sees no fewer
  int first;
  uint32_t ring, q;   // uses of the K and V ring and of the Q tiles before this piece
  __device__ __forceinline__ int keys_of(int rt) const { return rt ? keys[1] : keys[0]; }
  __device__ __forceinline__ int tiles(int rt) const { return (keys_of(rt) + kKeys - 1) / kKeys; }
};

// one piece of work, as the copy warp hands it to the others
struct Work {
  int q_tok, n_tok;   // query tokens (prompt) or sequences (decode step)
  int head;
  Order order;
  int key0;           // first key: an index into the packed keys, or the position in the sequence
  int limit0;         // prompt: keys that the first query token sees
  int n_keys;         // keys from key0 on that anyone sees
  int row;            // decode step: table row
  int last;           // nothing follows
  int64_t out_row;    // where the partial rows begin, if there are any
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
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {  // without waiting
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
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
__device__ __forceinline__ bool mbar_wait_slow(uint64_t* bar, uint32_t parity) {
  const unsigned long long start = global_timer_ns();
  do {
    if (mbar_try(bar, parity)) return true;
  } while (global_timer_ns() - start < kWaitNs);
  return false;
}
// false: the phase did not complete in time
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
  return mbar_try(bar, parity) || mbar_wait_slow(bar, parity);
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
// true in one lane of a whole warp
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
// the same value in all lanes, and the compiler knows
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

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
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               :
                 "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
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
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               :
                 "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
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

// two fp32 numbers in a register pair
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// the larger of three, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

// 32 columns of a row
__device__ __forceinline__ void mask_row(uint32_t (&s)[32], int seen) {
#pragma unroll
  for (int k = 0; k < 32; ++k)
    if (k >= seen) s[k] = 0xff800000u;  // -inf
}
__device__ __forceinline__ void max_row(const uint32_t (&s)[32], float (&top)[4]) {
#pragma unroll
  for (int k = 0; k < 32; k += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) top[i] = max3(top[i], __uint_as_float(s[k + 2 * i]), __uint_as_float(s[k + 2 * i + 1]));
}
// exp2(s c - mc), added up, and as bf16 pairs to 16 columns of tensor memory
__device__ __forceinline__ void weights(const uint32_t (&s)[32], uint64_t c, uint64_t minus_mc, uint64_t (&sum)[2], uint32_t to) {
  uint32_t packed[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const uint64_t x = fma2(pair(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), c, minus_mc);
    float a, b;
    unpair(x, a, b);
    a = exp2_fast(a);
    b = exp2_fast(b);
    sum[k & 1] = add2(sum[k & 1], pair(a, b));
    packed[k] = pack_bf16(a, b);
  }
  tmem_st(to, packed);
}

struct Bars {
  uint64_t full[8], empty[8], q_full[2], q_empty[2], s_full[2], p_half[2], p_full[2], o_full[2], stats, read, work_full[kWorkSlots],
      work_empty[kWorkSlots], drain;
};

// keys that the row's token sees, counted from the piece's first key
template <bool PAGED> __device__ __forceinline__ int row_limit(const TcParams& p, const Work& wk, int tok) {
  if constexpr (PAGED) return max(0, min(shared_seq_len(p.s, wk.q_tok + tok) - wk.key0, wk.n_keys));
  return max(0, min(wk.limit0 + tok, wk.n_keys));
}

// ---- copy warp: finds the work, fetches Q, K and V --------------------------------------------------------------------
// The code that a tile takes is kept short in all three roles that run beside the softmax: their warps do little else than
// fetch instructions, past which the softmax warps stream their own.
template <int D, bool PAGED> struct CopyRole {
  using C = Tc<D>;
  const TcParams& p;
  Bars* bars;
  Work* ring;
  unsigned char* base;
  SharedCursor cur;
  int next_item, end_item;
  uint32_t it = 0, q_it = 0, w_it = 0;  // ring stages, Q tiles, pieces so far
  uint32_t parity = 0;
  Work wk, next;
  bool alive = true;
  // Decode step.  Lane l knows the entity window + l; page numbers are fetched a tile ahead, and the next piece is found
  // while the last one's tiles are under way: a chain of loads per piece would be longer than the piece.
  int window = -1, w_first, w_n, w_lo, w_hi, w_units, lead_of = -1;
  int2 lead;
  int ids, next_ids;                    // lane l: page l of the next tile, of the next piece's first

  __device__ __forceinline__ CopyRole(const TcParams& p_, Bars* b, Work* r, unsigned char* base_, const SharedCursor& c)
      : p(p_), bars(b), ring(r), base(base_), cur(c) {
    next_item = PAGED ? 0 : p.cta_begin[blockIdx.x];
    end_item = PAGED ? 0 : p.cta_begin[blockIdx.x + 1];
  }
  __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity_) {
    if (alive && !__all_sync(0xffffffffu, mbar_wait(bar, parity_))) {
      alive = false;
      if ((threadIdx.x & 31) == 0) atomicOr(p.status, IA_DEV_STATUS_ATTEND_WAIT);
    }
    return alive;
  }
  __device__ __forceinline__ void see(int e) {  // the window holds entity e
    if (window >= 0 && e >= window && e < window + 32) return;
    window = e;
    const int mine = e + (threadIdx.x & 31);
    w_first = w_n = w_lo = w_hi = w_units = 0;
    if (mine < p.s.n_shared + p.s.batch) {
      const SharedEntity ent = load_entity(p.s, mine);
      entity_keys(p.s, mine, ent, w_lo, w_hi);
      w_first = ent.first_seq;
      w_n = ent.n_seqs;
      w_units = (w_hi - w_lo + kKeys - 1) / kKeys;
    }
  }
  // this lane's page of key tile j
  __device__ __forceinline__ int page_of(const Work& k, int j) {
    const int lane = threadIdx.x & 31, held = (min(kKeys, k.n_keys - j * kKeys) + 15) >> 4;
    return lane < held ? p.s.block_table[(int64_t)k.row * p.s.max_pages + ((k.key0 + j * kKeys) >> 4) + lane] : 0;
  }
  __device__ __forceinline__ void look_ahead() {
    next = Work{};
    find(next);
    if constexpr (PAGED)
      if (!next.last) next_ids = page_of(next, 0);
  }
  __device__ __forceinline__ void find(Work& wk) {
    const int tpm = kRows / p.group;
    if constexpr (PAGED) {
      wk.last = cur.left <= 0;
      if (wk.last) return;
      const SharedParams& s = p.s;
      see(cur.e);
      const int at = cur.e - window, lo = __shfl_sync(0xffffffffu, w_lo, at), hi = __shfl_sync(0xffffffffu, w_hi, at);
      const int units = __shfl_sync(0xffffffffu, w_units, at), n = (int)min((int64_t)(units - cur.k), cur.left);
      wk.q_tok = __shfl_sync(0xffffffffu, w_first, at);
      wk.n_tok = __shfl_sync(0xffffffffu, w_n, at);
      const bool own = cur.e >= s.n_shared;
      if (!own && lead_of != cur.e) {
        lead_of = cur.e;
        lead = entity_lead(s, load_entity(s, cur.e), hi);
      }
      wk.row = own ? wk.q_tok : lead.x;
      wk.head = cur.h;
      wk.key0 = lo + cur.k * kKeys;
      wk.n_keys = max(0, min(own ? hi : lead.y, wk.key0 + n * kKeys) - wk.key0);
      wk.out_row = cur.k == 0 ? item_rows(s, own, wk.q_tok, wk.n_tok, cur.h) : cta_rows(s, blockIdx.x);
      wk.order.split = wk.n_tok <= tpm;
      wk.order.keys[0] = wk.order.keys[1] = max(1, wk.n_keys);  // a tile of keys that nobody sees, where there are none
      cur.left -= n;
      cur.k = 0;
      if (++cur.h == s.n_kv_heads) {
        cur.h = 0;
        ++cur.e;
        while (cur.left > 0) {  // some entity behind this one has units: they were counted
          see(cur.e);
          const unsigned some = __ballot_sync(0xffffffffu, w_units > 0) & ~((1u << (cur.e - window)) - 1u);
          if (some != 0) {
            cur.e = window + __ffs(some) - 1;
            break;
          }
          cur.e = window + 32;
        }
      }
    } else {
      wk.last = next_item >= end_item;
      if (wk.last) return;
      const PromptItem item = p.items[next_item++];
      wk.q_tok = item.q_tok;
      wk.n_tok = item.n_tok;
      wk.head = item.head;
      wk.key0 = item.kv_tok;
      wk.limit0 = item.limit0;
      wk.n_keys = item.kv_len;
      wk.out_row = (int64_t)item.slot * kPartRows;
      wk.order.split = item.n_tok <= tpm;
      wk.order.keys[0] = max(1, row_limit<false>(p, wk, min(item.n_tok, tpm) - 1));
      wk.order.keys[1] = max(1, row_limit<false>(p, wk, item.n_tok - 1));
    }
  }
  // K (which = 0) or V of key tile j into the next stage
  __device__ __forceinline__ void fetch(int j, int which, int page) {
    const int lane = threadIdx.x & 31;
    const uint32_t st = it % C::stages;
    uint64_t* full = &bars->full[st];
    unsigned char* dst = base + C::ring + (size_t)st * C::kv_tile;
    if (!wait(&bars->empty[st], ((it / C::stages) & 1) ^ 1)) return;
    ++it;
    // in the place of the set that does not read the tile
    if ((wk.order.split || j * kKeys >= wk.order.keys[0]) && lane == 0) mbar_arrive(&bars->empty[st]);
    if constexpr (!PAGED) {
      if (lane == 0) {
        mbar_arrive_expect_tx(full, C::kv_tile);
        tma_load_4d(smem_u32(dst), which == 0 ? &p.tm_k : &p.tm_v, 0, wk.key0 + j * kKeys, 0, wk.head, full);
      }
    } else {
      const int valid = min(kKeys, wk.n_keys - j * kKeys);
      const int pages = which == 0 ? (valid + 15) >> 4 : valid >> 4;
      if (which == 1 && (valid & 15 || valid == 0)) {
        // The last page of a sequence: behind its last token it may hold anything, and zero times that must be zero, so its
        // rows are written here.  What the second product does not read is left as it is.
        const int tail = __shfl_sync(0xffffffffu, page, pages & (kKeys / 16 - 1));
        const bool good = tail >= 0 && (p.s.n_pool_pages == 0 || tail < p.s.n_pool_pages);
        const __nv_bfloat16* src = (const __nv_bfloat16*)p.s.v_pool + (int64_t)tail * p.s.page_stride + wk.head * p.s.head_stride;
        const int c = lane % (D / 8);
        unsigned char* to = dst + pages * (C::halves * 2048) + (c >> 3) * 2048;
        uint4 x[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int row = i * (256 / D) + lane / (D / 8);
          x[i] = make_uint4(0, 0, 0, 0);
          if (pages * 16 + row < valid && good) x[i] = *reinterpret_cast<const uint4*>(src + row * D + c * 8);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int row = i * (256 / D) + lane / (D / 8);
          *reinterpret_cast<uint4*>(to + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = x[i];
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
            tma_load_5d(smem_u32(dst + h * C::kv_block + lane * 2048), &p.tm_k, 0, 0, h, wk.head, page, full);
        } else {           // page by page: a k step of the second product is one page
          tma_load_5d(smem_u32(dst + lane * (C::halves * 2048)), &p.tm_v, 0, 0, 0, wk.head, page, full);
        }
      }
      __syncwarp();
    }
  }
  __device__ __forceinline__ void fetch_q(int rt) {
    const uint32_t buf = q_it & 1;
    const int tpm = kRows / p.group;
    if (!wait(&bars->q_empty[buf], ((q_it >> 1) & 1) ^ 1)) return;
    ++q_it;
    if ((threadIdx.x & 31) == 0) {
      if (!wk.order.split || wk.order.keys[0] <= kKeys) mbar_arrive(&bars->q_empty[buf]);  // only one set reads it
      mbar_arrive_expect_tx(&bars->q_full[buf], (uint32_t)(C::halves * tpm * p.group * 128));
      for (int h = 0; h < C::halves; ++h)
        tma_load_5d(smem_u32(base + buf * C::tile + h * C::block), &p.tm_q, 0, 0, wk.q_tok + rt * tpm, h, wk.head,
                    &bars->q_full[buf]);
    }
  }
  __device__ __forceinline__ void run() {
    look_ahead();
    while (alive) {
      const int slot = w_it % kWorkSlots;
      if (!wait(&bars->work_empty[slot], ((w_it / kWorkSlots) & 1) ^ 1)) break;
      wk = next;
      ids = next_ids;
      wk.order.first = (int)parity;
      wk.order.ring = it;
      wk.order.q = q_it;
      const int tiles = wk.last ? 0 : wk.order.tiles(1);
      if (wk.order.split) parity ^= tiles & 1;  // the sets take turns across pieces too
      if ((threadIdx.x & 31) == 0) {
        ring[slot] = wk;
        mbar_arrive(&bars->work_full[slot]);
      }
      __syncwarp();
      ++w_it;
      if (wk.last) break;
#pragma unroll 1
      for (int j = 0; j < tiles && alive; ++j) {
        const int page = ids;
        if constexpr (PAGED) {
          if (page < 0 || (p.s.n_pool_pages > 0 && page >= p.s.n_pool_pages)) atomicOr(p.status, DEV_STATUS_BAD_INDEX);
          if ((j + 1) * kKeys < wk.n_keys) ids = page_of(wk, j + 1);
        }
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          fetch(j, which, page);
          if (j == 0 && which == 0) {  // Q behind the first K: the ring may be ahead of the end of the piece before
            fetch_q(0);
            if (!wk.order.split) fetch_q(1);
          }
        }
        if (j == min(2, tiles - 1)) look_ahead();  // not before the first tiles are under way
      }
    }
    if (!alive) {  // no copy may be in flight when the CTA ends
      for (uint32_t i = it > C::stages ? it - C::stages : 0; i < it; ++i) mbar_wait(&bars->full[i % C::stages], (i / C::stages) & 1);
      for (uint32_t i = q_it > 2 ? q_it - 2 : 0; i < q_it; ++i) mbar_wait(&bars->q_full[i & 1], (i >> 1) & 1);
    }
  }
};

// ---- MMA warps --------------------------------------------------------------------------------------------------------
template <int D, bool PAGED> struct MmaRole {
  using C = Tc<D>;
  static constexpr uint32_t kNextCols = PAGED ? 2048 : C::kv_block, kStepBytes = PAGED ? C::halves * 2048 : 2048;
  const TcParams& p;
  Bars* bars;
  const Work* ring;
  uint32_t q0, tmem;
  uint32_t me;  // the set
  uint32_t p_count = 0;
  bool alive = true;

  // the set's key tiles, piece after piece
  struct Cursor {
    uint32_t work = 0, use = 0, step = 0, q = 0;  // pieces opened; ring use of the tile, its step; Q tile
    int left = 0, keys = 0, width = 0;                       // tiles and keys from this one on, keys per step
    bool opens = false, shared_q = false;
  } s, v;

  __device__ __forceinline__ MmaRole(const TcParams& p_, Bars* b, const Work* r, uint32_t base, uint32_t t, uint32_t me_)
      : p(p_), bars(b), ring(r), q0(base), tmem(t), me(me_) {}
  __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
    if (alive && !__all_sync(0xffffffffu, mbar_wait(bar, parity))) {
      alive = false;
      if ((threadIdx.x & 31) == 0) atomicOr(p.status, IA_DEV_STATUS_ATTEND_WAIT);
    }
    return alive;
  }
  // On to the set's next tile; false: there is none.  The second product's cursor gives pieces back.
  __device__ __forceinline__ bool next(Cursor& c, bool give_back) {
    if (--c.left > 0) {
      c.use += c.step;
      c.keys -= c.width;
      c.opens = false;
      return true;
    }
    do {
      if (give_back && c.work > 0 && elect_one()) mbar_arrive(&bars->work_empty[(c.work - 1) % kWorkSlots]);
      const uint32_t slot = c.work % kWorkSlots;
      if (!wait(&bars->work_full[slot], (c.work / kWorkSlots) & 1) || ring[slot].last) {
        c.left = 1;  // and so it stays
        return false;
      }
      ++c.work;
      const Order o = ring[slot].order;
      const int i = (int)me ^ o.first;
      c.left = o.split ? (o.tiles(0) - i + 1) >> 1 : o.tiles(i);
      c.use = o.ring + (o.split ? 2 * i : 0);
      c.step = o.split ? 4 : 2;
      c.keys = o.split ? o.keys[0] - i * kKeys : o.keys_of(i);
      c.width = o.split ? 2 * kKeys : kKeys;
      c.q = o.q + (o.split ? 0 : i);
      c.opens = true;
    } while (c.left <= 0);
    return true;
  }
  // The values have to be known as the same in all lanes, or every operand of every MMA is moved to the uniform registers anew.
  struct First { uint64_t a, b; uint32_t ks, buf, closes, idesc; };
  __device__ __forceinline__ First first() const {
    First f;
    f.ks = uniform(s.use % C::stages);
    f.buf = uniform(s.q & 1);
    f.closes = uniform(s.left == 1);
    f.idesc = uniform(kIdesc<0, false> | ((uint32_t)min(kKeys / 16, (s.keys + 15) >> 4) << 18));  // N = 16 for each 16 keys
    f.a = umma_desc(q0 + f.buf * C::tile, 0);
    f.b = umma_desc(q0 + (uint32_t)C::ring + f.ks * C::kv_tile, 0);
    return f;
  }
  __device__ __forceinline__ bool first_ready() const {  // without waiting
    return __all_sync(0xffffffffu, (!s.opens || mbar_test(&bars->q_full[s.q & 1], (s.q >> 1) & 1)) &&
                                       mbar_test(&bars->full[s.use % C::stages], (s.use / C::stages) & 1));
  }
  __device__ __forceinline__ void issue_first(const First& f) const {
#pragma unroll
    for (int h = 0; h < C::halves; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)  // 16 dims = 32 bytes further inside the swizzled row
        umma_ss(tmem + me * 128, f.a + (h * C::block + i * 32) / 16, f.b + (h * C::kv_block + i * 32) / 16, f.idesc, h + i > 0);
    umma_commit(&bars->s_full[me]);
    umma_commit(&bars->empty[f.ks]);
    if (f.closes) umma_commit(&bars->q_empty[f.buf]);
  }
  __device__ __forceinline__ void run() {
    s.left = v.left = 1;  // the first call opens a piece
#pragma unroll 1
    for (bool start = true; (start || next(v, true)) && alive; start = false) {
      bool more = next(s, false);
      const First f = first();
      if (!start) {
        const uint32_t vs = uniform((v.use + 1) % C::stages), old = uniform(!v.opens),
                       k16 = uniform(min(kKeys / 16, (v.keys + 15) >> 4));
        const uint64_t b = umma_desc(q0 + (uint32_t)C::ring + vs * C::kv_tile, kNextCols);
        if (!wait(&bars->full[vs], ((v.use + 1) / C::stages) & 1) || !wait(&bars->p_half[me], p_count & 1)) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kKeys / 32; ++k)  // 16 keys: 8 columns of packed weights, 16 rows of V
            if (k < k16)
              umma_ts(tmem + 256 + me * 128, tmem + me * 128 + k * 8, b + k * kStepBytes / 16, kIdesc<D, true>, k > 0 ? 1u : old);
        }
        __syncwarp();
        const bool both = more && first_ready();
        if (!wait(&bars->p_full[me], p_count++ & 1)) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = kKeys / 32; k < kKeys / 16; ++k)
            if (k < k16)
              umma_ts(tmem + 256 + me * 128, tmem + me * 128 + k * 8, b + k * kStepBytes / 16, kIdesc<D, true>, 1u);
          umma_commit(&bars->o_full[me]);
          umma_commit(&bars->empty[vs]);
          if (both) issue_first(f);
        }
        __syncwarp();
        if (both) more = false;
      }
      if (more && alive) {
        if ((s.opens && !wait(&bars->q_full[s.q & 1], (s.q >> 1) & 1)) || !wait(&bars->full[s.use % C::stages], (s.use / C::stages) & 1)) break;
        tc_fence_after();
        if (elect_one()) issue_first(f);
        __syncwarp();
      }
    }
    if (elect_one()) umma_commit(&bars->drain);  // no MMA, and no arrival of one, may be in flight when the CTA ends
    __syncwarp();
    alive = true;
    wait(&bars->drain, 0);
  }
};

// ---- softmax warps ----------------------------------------------------------------------------------------------------
template <bool PAGED, bool PARTS> using OutOf = std::conditional_t<PAGED || PARTS, float, __nv_bfloat16>;

template <int D, bool PAGED, bool PARTS>
__device__ __forceinline__ void softmax_role(const TcParams& p, Bars* bars, const Work* ring, uint32_t tmem, unsigned char* out_base,
                                             float2 (*stats)[kRows], int* flagged) {
  using Out = OutOf<PAGED, PARTS>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = warp >> 2, row = (warp & 3) * 32 + lane;
  const int G = p.group, tpm = kRows / G, row_tok = row / G, g = row % G;
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const uint32_t s_addr = tmem + lanes + w * 128, o_addr = tmem + lanes + 256;
  const float c = kLog2e * rsqrtf((float)D);
  uint32_t s_it = 0, x_it = 0;
  const auto wait = [&](uint64_t* bar, uint32_t parity) {  // the whole warp goes on or none of it
    const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity));
    if (!ok && lane == 0) atomicOr(p.status, IA_DEV_STATUS_ATTEND_WAIT);
    return ok;
  };
  for (uint32_t w_it = 0;; ++w_it) {
    const int slot = w_it % kWorkSlots;
    if (!wait(&bars->work_full[slot], (w_it / kWorkSlots) & 1)) return;
    const Work& wk = ring[slot];  // read where it is needed: registers are scarce in the loop below
    if (wk.last) return;
    const auto done = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->work_empty[slot]);
    };
    const bool split = wk.order.split;
    const int me = w ^ wk.order.first;  // row tile, or place in the order of key tiles
    const int keys = wk.order.keys_of(split ? 0 : me), total = wk.order.tiles(split ? 0 : me), stride = split ? 2 : 1, begin = split ? me : 0;
    if (begin >= total) {  // the other set has the only key tile
      done();
      continue;
    }
    const int tok = (split ? 0 : me * tpm) + row_tok;
    const bool valid = row < tpm * G && tok < wk.n_tok;
    const bool busy = __any_sync(0xffffffffu, valid);
    const int limit = valid ? row_limit<PAGED>(p, wk, tok) : 0;
    const int least = __reduce_min_sync(0xffffffffu, valid ? limit : 0x7fffffff);  // below it nothing is masked
    float m = -INFINITY, l = 0.f;
    for (int j = begin; j < total; j += stride) {
      if (!wait(&bars->s_full[w], s_it & 1)) return;
      ++s_it;
      if (busy) {
        tc_fence_after();
        const int seen = limit - j * kKeys, all_seen = least - j * kKeys;
        uint32_t r[kKeys / 32][32];
#pragma unroll
        for (int i = 0; i < kKeys / 32; ++i) tmem_ld(s_addr + 32 * i, r[i]);
#pragma unroll
        for (int i = 0; i < kKeys / 32; ++i) tmem_wait_ld(r[i]);
        const int columns = keys - j * kKeys;  // behind them neither product reads or writes
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kKeys / 32; ++i) {
          if (i * 32 >= columns) break;
          if (all_seen < 32 * (i + 1)) mask_row(r[i], seen - 32 * i);
          max_row(r[i], top);
        }
        const float t = max3(top[0], top[1], max3(top[2], top[3], -INFINITY));
        if (j == begin) {
          m = t;
        } else {
          const bool far = !((t - m) * c <= 8.f) && t != -INFINITY;  // also where m is still -inf, or t is NaN
          if (__any_sync(0xffffffffu, far)) {
            const float keep = far ? exp2_fast((m - t) * c) : 1.f;
            if (far) {
              m = t;
              l *= keep;
            }
#pragma unroll 1
            for (int i = 0; i < D; i += 16) {  // the products of the tile before are complete: S of this one came after them
              uint32_t o[16];
              tmem_ld(o_addr + w * 128 + i, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
              tmem_st(o_addr + w * 128 + i, o);
            }
          }
        }
        float mc = m == -INFINITY ? 0.f : m * c;
        mc = fmaf(mc, 0.f, mc);  // infinite: NaN, as infinity - infinity in the weights
        const uint64_t c2 = pair(c, c), mc2 = pair(-mc, -mc);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < kKeys / 32; ++i) {
          if (i == kKeys / 64) {  // the second product begins with the first half of the keys
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->p_half[w]);
          }
          if (i * 32 < columns) weights(r[i], c2, mc2, sum, s_addr + 16 * i);
        }
        float la, lb;
        unpair(add2(sum[0], sum[1]), la, lb);
        l += la + lb;
        tmem_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) {
        if (!busy) mbar_arrive(&bars->p_half[w]);
        mbar_arrive(&bars->p_full[w]);
      }
    }
    if (!wait(&bars->o_full[w], (s_it - 1) & 1)) return;
    tc_fence_after();
    // ---- output: this set's O scaled, or over half of the columns both sets' ----
    float scale = 0.f, its_scale = 0.f, lse = -INFINITY;
    const bool merge = split && total > 1, empty = limit <= 0;
    if (merge) {
      stats[w][row] = make_float2(m, l);
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->stats);
      if (!wait(&bars->stats, x_it & 1)) return;
      tc_fence_after();
      const float2 other = stats[w ^ 1][row];
      const float top = fmaxf(m, other.x), at = top == -INFINITY ? 0.f : top;
      const float mine = exp2_fast((m - at) * c), its = exp2_fast((other.x - at) * c), sum = l * mine + other.y * its;
      if (!empty) {
        scale = mine / sum;
        its_scale = its / sum;
        lse = (top * c + __log2f(sum)) * kLn2;
      }
    } else if (!empty) {
      scale = 1.f / l;
      lse = (m * c + __log2f(l)) * kLn2;
    }
    const int64_t hq = (int64_t)G * (PAGED ? p.s.n_kv_heads : p.t.n_kv_heads);
    Out* out;          // of the piece's first row
    float* lse_out;    // of this row
    int at;            // this row, in elements from `out`; -1: none
    if constexpr (PAGED) {
      out = p.s.o + wk.out_row * D;
      at = (tok * G + g) * D;
      lse_out = p.s.lse + wk.out_row + tok * G + g;
    } else if constexpr (PARTS) {
      out = p.t.part_o + wk.out_row * D;
      at = (tok * G + g) * D;
      lse_out = p.t.part_lse + wk.out_row + tok * G + g;
    } else {
      const int64_t first = wk.q_tok * hq + wk.head * G;
      out = (Out*)p.t.out + first * D;
      at = (int)(tok * hq + g) * D;
      lse_out = p.t.lse == nullptr ? nullptr : p.t.lse + first + tok * hq + g;
    }
    if (!valid) at = -1;
    const int col0 = merge ? w * (D / 2) : 0, col1 = merge ? col0 + D / 2 : D;
    unsigned char* rows = out_base + warp * Tc<D>::out_warp;  // [32 rows][32 columns], 16-byte words swizzled
    constexpr int kWords = 32 * sizeof(Out) / 16;             // words of a row: 8 or 4
    uint64_t not_finite[2] = {0, 0};  // sums of zero times what is written
    if (busy) {
      int to[kWords];  // kWords neighbouring lanes write a row's run
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        to[i] = __shfl_sync(0xffffffffu, at, i * (32 / kWords) + lane / kWords);
        if (to[i] >= 0) to[i] += lane % kWords * (16 / (int)sizeof(Out));
      }
      const bool any_empty = __any_sync(0xffffffffu, empty);
      const uint64_t scale2 = pair(scale, scale), its2 = pair(its_scale, its_scale);
#pragma unroll 1
      for (int col = col0; col < col1; col += 32) {
        uint64_t x[16];
        {
          uint32_t o[32];
          tmem_ld(o_addr + w * 128 + col, o);
          tmem_wait_ld(o);
#pragma unroll
          for (int k = 0; k < 16; ++k) x[k] = mul2(pair(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1])), scale2);
          if (merge) {
            tmem_ld(o_addr + (w ^ 1) * 128 + col, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = fma2(pair(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1])), its2, x[k]);
          }
        }
        if (any_empty) {
#pragma unroll
          for (int k = 0; k < 16; ++k) x[k] = empty ? 0 : x[k];
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) not_finite[k & 1] = fma2(x[k], 0, not_finite[k & 1]);
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          uint32_t v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float lo, hi;
            if constexpr (PAGED || PARTS) {
              unpair(x[2 * k + i / 2], lo, hi);
              v[i] = __float_as_uint(i & 1 ? hi : lo);
            } else {
              unpair(x[4 * k + i], lo, hi);
              v[i] = pack_bf16(lo, hi);
            }
          }
          *reinterpret_cast<uint4*>(rows + lane * 128 + ((k ^ (lane & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        __syncwarp();
        uint4 v[kWords];  // all reads before the first write
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const int r = i * (32 / kWords) + lane / kWords, k = lane % kWords;
          v[i] = *reinterpret_cast<const uint4*>(rows + r * 128 + ((k ^ (r & 7)) << 4));
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i)
          if (to[i] >= 0) *reinterpret_cast<uint4*>(out + to[i] + col) = v[i];
        __syncwarp();
      }
      if (valid && lse_out != nullptr && (!merge || me == 0)) *lse_out = lse;
    }
    if (merge) {  // the other set has read O before the next piece's products may overwrite it
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->read);
      if (!wait(&bars->read, x_it & 1)) return;
      ++x_it;
    }
    float nan_lo, nan_hi;
    unpair(add2(not_finite[0], not_finite[1]), nan_lo, nan_hi);
    const unsigned bad = __ballot_sync(0xffffffffu, valid && !(nan_lo + nan_hi == 0.f));
    if (bad != 0 && lane == 0) *flagged = 1;  // see redo_rows
    done();
  }
}

struct Control {
  Bars bars;
  Work ring[kWorkSlots];
  float2 stats[2][kRows];  // (m, l) of either set, for the merge
  uint32_t tmem;
  int flagged;             // some row came out non-finite
};

// ---- rows that came out non-finite ------------------------------------------------------------------------------------
// See exact_row.  How long this takes grows with the rows times their keys, so it waits until the CTA's last piece is done and no
// role waits for another within a limit.  The pieces are gone through once more: which of their rows are not finite, which is
// the last bad value row that one of them held but does not see, and the rows that do not see it again, a warp each.  An 8192-token
// prompt of the Llama-3-8B heads whose last value is infinite: 18.7 ms instead of 0.57 (63 tokens of the last piece, eight SMs busy);
// with a NaN at every 1000th token 1.2 ms, at all of them 1.9 ms; 4 x 4800 tokens behind 150,000 each, the last of each
// infinite: 267 ms instead of 12.
struct Redo {
  unsigned rows[2 * kRows / 32];  // a bit a row
  int least, last;                // least limit of these rows; last bad key
};
template <int D, bool PAGED, bool PARTS, typename Key>
__device__ __forceinline__ void redo_piece(const TcParams& p, const Work& wk, int end, const Key& key, const __nv_bfloat16* q, int64_t q_tok_stride,
                           int64_t q_head_stride, OutOf<PAGED, PARTS>* out, int64_t out_tok_stride, Redo* redo) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = p.group, rows = wk.n_tok * G;
  constexpr int kWarps = kThreads / 32;
  __syncthreads();  // the piece before is done with the shared words
  if (threadIdx.x < 2 * kRows / 32) redo->rows[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    redo->least = 0x7fffffff;
    redo->last = -1;
  }
  __syncthreads();
  for (int r = warp; r < rows; r += kWarps) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) bad |= !(fabsf(to_f32(out[r / G * out_tok_stride + r % G * D + lane + 32 * i])) <= 3.4028235e38f);
    if (!__any_sync(0xffffffffu, bad) || lane != 0) continue;
    atomicOr(&redo->rows[r / 32], 1u << (r & 31));
    atomicMin(&redo->least, row_limit<PAGED>(p, wk, r / G));
  }
  __syncthreads();
  if (redo->least >= end) return;
  const int last = last_not_finite<__nv_bfloat16, D>(redo->least, end, key, warp * 32, kThreads);
  if (lane == 0) atomicMax(&redo->last, last);
  __syncthreads();
  for (int r = warp; r < rows; r += kWarps) {
    const int limit = row_limit<PAGED>(p, wk, r / G);
    if (!(redo->rows[r / 32] >> (r & 31) & 1) || redo->last < limit) continue;
    float x[D / 32], m, l;
    exact_row<__nv_bfloat16, D, 16>(q + r / G * q_tok_stride + r % G * q_head_stride, 0, limit, kLog2e * rsqrtf((float)D), key, x, m, l);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) from_f32(out[r / G * out_tok_stride + r % G * D + lane + 32 * i], x[i] / l);
  }
}
template <int D, bool PAGED, bool PARTS>
__device__ __noinline__ void redo_rows(const TcParams& p, unsigned long long* scratch, Redo* redo) {
  using T = __nv_bfloat16;
  const int G = p.group;
  Work wk{};
  if constexpr (PAGED) {
    const SharedParams& s = p.s;
    const int64_t hq = (int64_t)G * s.n_kv_heads;
    SharedCursor c = find_share<kKeys, kThreads>(s, blockIdx.x, gridDim.x, scratch);
    while (c.left > 0) {
      const SharedEntity ent = load_entity(s, c.e);
      int lo, hi;
      entity_keys(s, c.e, ent, lo, hi);
      const int n = (int)min((int64_t)(c.units - c.k), c.left);
      const bool own = c.e >= s.n_shared;
      const int2 lead = own ? make_int2(ent.first_seq, hi) : entity_lead(s, ent, hi);
      wk.q_tok = ent.first_seq;
      wk.n_tok = ent.n_seqs;
      wk.key0 = lo + c.k * kKeys;
      wk.n_keys = max(0, min(lead.y, wk.key0 + n * kKeys) - wk.key0);
      const int64_t row0 = c.k == 0 ? item_rows(s, own, ent.first_seq, ent.n_seqs, c.h) : cta_rows(s, blockIdx.x);
      const PagedKeys<T> key{(const T*)s.k_pool + c.h * s.head_stride, (const T*)s.v_pool + c.h * s.head_stride,
                             s.block_table + (int64_t)lead.x * s.max_pages + (wk.key0 >> 4), s.page_stride, D, s.n_pool_pages,
                             s.max_pages - (wk.key0 >> 4)};
      redo_piece<D, PAGED, PARTS>(p, wk, wk.n_keys, key, (const T*)s.q + (wk.q_tok * hq + c.h * G) * D, hq * D, D, s.o + row0 * D,
                                  (int64_t)G * D, redo);
      c.left -= n;
      c.k = 0;
      if (++c.h == s.n_kv_heads) {
        c.h = 0;
        if (c.left > 0)  // some entity behind this one has units: they were counted
          do c.units = entity_units<kKeys>(s, ++c.e);
          while (c.units == 0);
      }
    }
  } else {
    const PromptTensors& t = p.t;
    const int64_t hq = (int64_t)G * t.n_kv_heads;
    for (int i = p.cta_begin[blockIdx.x]; i < p.cta_begin[blockIdx.x + 1]; ++i) {
      const PromptItem item = p.items[i];
      wk.n_tok = item.n_tok;
      wk.limit0 = item.limit0;
      wk.n_keys = item.kv_len;
      const PackedKeys<T> key{(const T*)t.k + item.kv_tok * t.k_tok_stride + item.head * t.k_head_stride,
                              (const T*)t.v + item.kv_tok * t.v_tok_stride + item.head * t.v_head_stride, t.k_tok_stride,
                              t.v_tok_stride, t.n_kv_tok - item.kv_tok};
      const int end = (max(1, row_limit<false>(p, wk, item.n_tok - 1)) + kKeys - 1) / kKeys * kKeys;  // of the tiles that it held
      const T* q = (const T*)t.q + item.q_tok * t.q_tok_stride + (int64_t)item.head * G * t.q_head_stride;
      if constexpr (PARTS)
        redo_piece<D, PAGED, PARTS>(p, wk, end, key, q, t.q_tok_stride, t.q_head_stride, t.part_o + (int64_t)item.slot * kPartRows * D,
                                    (int64_t)G * D, redo);
      else
        redo_piece<D, PAGED, PARTS>(p, wk, end, key, q, t.q_tok_stride, t.q_head_stride,
                                    (T*)t.out + (item.q_tok * hq + item.head * G) * D, hq * D, redo);
    }
  }
}

template <int D, bool PAGED, bool PARTS>
__global__ void __launch_bounds__(kThreads, 1) attend_tc_kernel(const __grid_constant__ TcParams p) {
  using C = Tc<D>;
  extern __shared__ __align__(1024) unsigned char base[];
  static_assert(sizeof(Control) <= 3 * 1024, "the whole of an SM's shared memory is spoken for");
  Control& ctl = *reinterpret_cast<Control*>(base + C::control);
  Bars& bars = ctl.bars;
  const int warp = threadIdx.x >> 5;
  if ((smem_u32(base) & 1023u) != 0) {  // swizzled tiles start on 1024 bytes; there is no room to round up
    if (threadIdx.x == 0) atomicOr(p.status, IA_DEV_STATUS_ATTEND_WAIT);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::stages; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 2);  // both sets, or one and the copy warp
    }
    mbar_init(&bars.stats, 8);  // a lane of each softmax warp
    mbar_init(&bars.read, 8);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&bars.q_full[w], 1);
      mbar_init(&bars.q_empty[w], 2);
      mbar_init(&bars.s_full[w], 1);
      mbar_init(&bars.p_half[w], 4);  // a lane of each warp
      mbar_init(&bars.p_full[w], 4);
      mbar_init(&bars.o_full[w], 1);
    }
    for (int i = 0; i < kWorkSlots; ++i) {
      mbar_init(&bars.work_full[i], 1);
      mbar_init(&bars.work_empty[i], 10);  // eight softmax warps and two MMA threads
    }
    mbar_init(&bars.drain, 2);
    ctl.flagged = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem;
  grid_dependency_wait();
  grid_launch_dependents();
  SharedCursor cur{};
  if constexpr (PAGED) cur = find_share<kKeys, kThreads>(p.s, blockIdx.x, gridDim.x, reinterpret_cast<unsigned long long*>(ctl.stats));
  if (warp < kCopyWarp) {
    softmax_role<D, PAGED, PARTS>(p, &bars, ctl.ring, tmem, base + C::tiles, ctl.stats, &ctl.flagged);
  } else {
    if (warp == kCopyWarp) CopyRole<D, PAGED>(p, &bars, ctl.ring, base, cur).run();
    if (warp >= kMmaWarp) MmaRole<D, PAGED>(p, &bars, ctl.ring, smem_u32(base), uniform(tmem), uniform(warp - kMmaWarp)).run();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  if (ctl.flagged != 0)
    redo_rows<D, PAGED, PARTS>(p, reinterpret_cast<unsigned long long*>(ctl.stats), reinterpret_cast<Redo*>(base));
}

// ---- host -------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static std::atomic<EncodeFn> known{nullptr};  // any thread may be the first; all would store the same pointer
  EncodeFn fn = known.load(std::memory_order_relaxed);
  if (fn == nullptr) {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &found) == cudaSuccess &&
        found == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<EncodeFn>(sym);
      known.store(fn, std::memory_order_relaxed);
    }
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

template <int D, bool PAGED, bool PARTS = false> int launch_tc(const TcParams& p, int grid, cudaStream_t stream) {
  auto kern = attend_tc_kernel<D, PAGED, PARTS>;
  static SmemOnce once;
  if (int s = once.allow((const void*)kern, Tc<D>::smem, "attend_tc_kernel")) return s;
  const cudaError_t e = launch_overlapped(kern, (unsigned)grid, (unsigned)kThreads, Tc<D>::smem, stream, p);
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
  if (t.n_kv_tok == 0) {  // every row is empty, but still has a tile of keys that it does not see: let it be the queries
    p.t.k = p.t.v = t.q;
    const int64_t dims[4] = {64, t.n_q_tok, head_dim / 64, t.n_kv_heads}, strides[3] = {t.q_tok_stride, 64, t.q_head_stride};
    if (int s = encode<4>(&p.tm_k, t.q, dims, strides, {64, kKeys, head_dim / 64, 1})) return s;
    p.tm_v = p.tm_k;
  } else {
    const int64_t dims[4] = {64, t.n_kv_tok, head_dim / 64, t.n_kv_heads};
    const int box[4] = {64, kKeys, head_dim / 64, 1};
    const int64_t ks[3] = {t.k_tok_stride, 64, t.k_head_stride}, vs[3] = {t.v_tok_stride, 64, t.v_head_stride};
    if (int s = encode<4>(&p.tm_k, t.k, dims, ks, box)) return s;
    if (int s = encode<4>(&p.tm_v, t.v, dims, vs, box)) return s;
  }
  if (t.part_o != nullptr) return head_dim == 128 ? launch_tc<128, false, true>(p, ctas, stream) : launch_tc<64, false, true>(p, ctas, stream);
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
