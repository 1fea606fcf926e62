// hc_prompt_attn.cu -- causal attention of many query rows: whole prompts and
// chunks of them, on the fifth-generation tensor cores.
//
// The rows of one product are (new token, query head of the KV head's group)
// pairs in token order, 128 to a CTA, so a tile covers 128 / group tokens: a
// short prompt still fills tiles, a tile's causal border is narrow, and a key
// tile read once serves the whole group.  Per tile of 128 keys:
//   S = Q K^T      tcgen05.mma, both operands in shared memory, S f32 in
//                  tensor memory;
//   P = 2^(S c - m c), c = scale log2(e): one thread per row, so maximum and
//                  sum (f32, of the unrounded P) stay in registers; P is rounded
//                  to the value type and goes to tensor memory;
//   O += P V       tcgen05.mma with P read from tensor memory, O f32 there
//                  (head_dim columns).
// m is the row's running maximum, but moved only when it grew by more than 8
// (in log2 units): P then stays below 2^8, which no type here minds, and the pass
// over O in tensor memory that a new maximum needs becomes rare (the first
// few tiles).
//
// head_dim 128 and 256: two CTAs form a pair (cta_group::2, M = 256), each bringing
//   its 128 rows, half of the keys of K and half of the dims of V.  One CTA's
//   products of N = 128 read 128 bytes of shared memory per clock, all that there
//   is, and the arriving tiles come on top; in a pair the second operand is
//   shared, and K and V cross from L2 once for 256 rows.
// head_dim 64: one CTA; the exponentials bound it, not the products.
//
// Two warpgroups take the key tiles in turn, so that one's loads, maxima and
// barriers fall into the other's exponentials; they pass the row's m
// along in shared memory.  Tensor memory: O behind column 256, two S slots of 128
// columns; up to head_dim 128 P has two slots of 64 of its own, so an S slot is
// free as soon as its row is in registers and the next S does not wait for P.
// At head_dim 256 P takes the place of its S.
//
// The CTAs stay: each takes its next item (sequence, KV head, rows) from the
// launch by clusterlaunchcontrol shortly before the present one's last keys, the
// longest sums first, and loads its Q, K and V ahead.  Four warps store an
// item's rows while the softmax warps are at the next item's tiles.  Twelve
// prompts of 1 to 2048 tokens (1576 items of 6 tiles on average) take 233 us so;
// with the rows stored by the softmax warps, Q brought by threads and the next item
// taken one ahead it was 266 (8192 tokens at head_dim 256: 220 and 250).
//
// Few items over long keys (chunks of one long prompt) are cut along the keys:
// an item gets as many parts as its share of all tiles fills CTAs, each
// at least 8 tiles; parts leave their sums in the workspace and
// hc_prompt_join_kernel adds them up.  512 rows x 8 / 2 heads of 256 over 8192 keys:
// 93 us whole, 42 in parts.
//
// K and V arrive by TMA, page by page or straight from packed rows, 128-byte
// swizzled, which is the operand layout of both products (K rows are K-major; V is
// N-major as it lies).  Keys that a row does not see get -inf scores and add
// nothing: values behind the last key in use are zeroed before they are
// multiplied, and so is a value that only some rows of a tile see and that is not
// finite (0 * inf); it is added to the stored rows that see it afterwards.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "hc_paged.cuh"

namespace hc {
namespace {

constexpr int PR_KEYS = 128;     // keys per tile
constexpr int PR_ROWS = 128;     // rows per CTA
constexpr int PR_AHEAD = 3;      // tiles that are left to load of an item when the next is asked for
constexpr int PR_PART = 8;       // tiles in a part of an item's keys, at least
constexpr int PR_PLACES = 2;     // parts that a launch may have for each CTA (pair) of the machine
constexpr float PR_GROW = 8.0f;  // log2 units a maximum may grow before O is rescaled

template <int D>
struct PrCfg {
  static constexpr int CG = D == 64 ? 1 : 2;              // CTAs per MMA
  static constexpr bool kOwnP = D <= 128;                 // P beside S, not over it
  static constexpr uint32_t kTmemO = D == 256 ? 256 : 384;
  static constexpr int kThreads = 512;                    // 8 softmax warps; one each for K, V, S and O; 4 for items
  static constexpr int kQ = PR_ROWS * D * 2;              // bytes of Q
  static constexpr int kK = PR_KEYS / CG * D * 2;         // bytes of K and of V per stage in this CTA
  static constexpr int kStages = D == 256 ? 2 : 4;
  static constexpr int kRowBytes = D == 256 ? 64 : 128;   // output staging: of each of a warp's 32 rows
  static constexpr int kStage = 4 * 32 * kRowBytes;
  static constexpr int kQs = D == 256 ? 1 : 2;            // Q of the present item, and of the next where there is room
  static constexpr int kSmem = 1024 + kQs * kQ + 2 * kStages * kK + kStage;
  static constexpr int kKeys = PR_KEYS / CG;              // keys of K in this CTA
  static constexpr int kPieces = D / 64;                  // 128-byte pieces of a row
  static constexpr int kPiecesV = kPieces / CG;           // of them V pieces in this CTA
  __host__ __device__ static constexpr uint32_t p_col(uint32_t slot) { return kOwnP ? 256 + slot * 64 : slot * 128; }
};
// registers per thread: launched with 128, the two softmax warpgroups take 184
// (a row of 128 scores each) from the other two
constexpr int PR_REGS_SOFTMAX = 184, PR_REGS_OTHER = 72;
static_assert(2 * PR_REGS_SOFTMAX + 2 * PR_REGS_OTHER == 4 * 128, "the split is of what the block was launched with");

struct PrArgs {
  AttnArgs a;
  PagedBatch b;
  const void* v;       // read again where a value is not finite
  int64_t v_stride;
  int box_k, box_v;    // key rows per TMA copy, as powers of two
  int whole_k, whole_v;  // a copy brings the CTA's whole tile, every piece of it
  int64_t slots;
  int items;             // items of the launch at most
  int split;             // most parts that an item's keys are cut into
  int workers;           // CTAs (or pairs) that the machine runs at a time
  int q_copy;            // Q comes by TMA
  float* part_o;         // [place][32 rows][head_dim / 4][row] float4, not divided by the sum
  float2* part_ml;       // [place][SPAN rows]: maximum (in log2 units) and sum
  struct PrJoin* join;   // [item]
};

// ---- tcgen05 -----------------------------------------------------------------

// shared-memory operand descriptor: 128-byte swizzle, version 1
__device__ __forceinline__ uint64_t pr_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return uint64_t((saddr >> 4) & 0x3fff) | (uint64_t((lbo >> 4) & 0x3fff) << 16) | (uint64_t((sbo >> 4) & 0x3fff) << 32) |
         (1ull << 46) | (2ull << 61);
}

// instruction descriptor: f32 accumulator, both operands f16 (0) or bf16 (1)
constexpr uint32_t pr_idesc(uint32_t fmt, uint32_t m, uint32_t n, uint32_t b_n_major) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_n_major << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

template <int CG>
__device__ __forceinline__ void pr_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc))
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc))
        : "memory");
}
template <int CG>
__device__ __forceinline__ void pr_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc))
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc))
        : "memory");
}
// Arrives on `bar` (in both CTAs of a pair) when the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void pr_commit(uint64_t* bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(uint16_t(3))
        : "memory");
}
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

#define PR_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define PR_I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])

__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : PR_R8(r, 0), PR_R8(r, 8), PR_R8(r, 16), PR_R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tm_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : PR_R8(r, 0), PR_R8(r, 8)
      : "r"(addr));
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      PR_I8(r, 0), PR_I8(r, 8)
      : "memory");
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The larger of three; NaN if one is NaN.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// ---- barriers across a CTA pair -------------------------------------------------

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
template <int CG>
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  if constexpr (CG == 1) {
    mbar_arrive(bar);
  } else {
    asm volatile(
        "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, 0;\n\t"
        "mbarrier.arrive.shared::cluster.b64 _, [ra];\n\t}\n" ::"r"(smem_u32(bar))
        : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void sync_all() {
  if constexpr (CG == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}
__device__ __forceinline__ bool pr_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return ok != 0;
}
// The rest of a wait, bounded in time.  The hint lets the hardware suspend the
// warp until the phase is complete: without it the waiting warps of a block took a
// quarter of the issue slots.
constexpr uint32_t PR_SLEEP_NS = 1000000;
__device__ __forceinline__ bool pr_wait_on(uint64_t* bar, uint32_t parity, int* err) {
  unsigned long long t0 = 0;
  for (int it = 0;; ++it) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok)
                 : "r"(smem_u32(bar)), "r"(parity), "r"(PR_SLEEP_NS)
                 : "memory");
    if (ok) return true;
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    if (it == 0) {
      t0 = t;
    } else if (t - t0 > WAIT_LIMIT_NS) {
      if (err) atomicExch(err, DEVICE_ERR_TIMEOUT);
      return false;
    }
  }
}
// A bounded wait (as mbar_wait_parity) that costs one instruction's round trip
// where the phase is already complete.
__device__ __forceinline__ bool pr_wait(uint64_t* bar, uint32_t parity, int* err) {
  return pr_try(bar, parity) || pr_wait_on(bar, parity, err);
}
// Two barriers with their answers in flight together: the common case, both
// complete, costs one round trip instead of two.
__device__ __forceinline__ bool pr_wait2(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, int* err) {
  const bool x = pr_try(a, pa), y = pr_try(b, pb);
  return (x || pr_wait_on(a, pa, err)) && (y || pr_wait_on(b, pb, err));
}

// ---- the launch's next item (clusterlaunchcontrol) ------------------------------

// Asks for a cluster of this grid that has not started; the answer (16 bytes)
// arrives on `bar` in every CTA of the cluster.
template <int CG>
__device__ __forceinline__ void clc_ask(uint4* answer, uint64_t* bar) {
  if constexpr (CG == 1)
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(answer)),
                 "r"(smem_u32(bar))
                 : "memory");
  else
    asm volatile(
        "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.multicast::cluster::all.b128 "
        "[%0], [%1];" ::"r"(smem_u32(answer)),
        "r"(smem_u32(bar))
        : "memory");
}
// The first block of the cluster taken over, or -1 when none is left.
__device__ __forceinline__ int clc_answer(const uint4* answer) {
  uint32_t x, got;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t.reg .b32 y, z;\n\tld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %1, 1, 0, p;\n\t"
      "mov.u32 %0, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, _}, r;\n\t}\n"
      : "=&r"(x), "=&r"(got)
      : "r"(smem_u32(answer))
      : "memory");
  return got ? int(x) : -1;
}

template <int CG>
__device__ __forceinline__ void pr_tma(uint32_t dst, const CUtensorMap* map, int row, int piece, uint32_t bar) {
  if constexpr (CG == 1) {
    tma_load_3d(dst, map, 0, row, piece, bar);
  } else {
    // the barrier may be the other CTA's (its address without the pair bit)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
        "%4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(piece), "r"(bar)
        : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void pr_tma_q(uint32_t dst, const CUtensorMap* map, int piece, int head, int token, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(piece), "r"(head), "r"(token), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
        "%4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(piece), "r"(head), "r"(token), "r"(bar)
        : "memory");
}
constexpr uint32_t kLeaderMask = 0xfeffffffu;  // a shared::cluster address in the pair's even CTA

// ---- values that are not finite

template <class T>
__device__ __forceinline__ bool pr_not_finite(uint32_t v) {
  constexpr uint32_t e = sizeof(T) && HalfOps<T>::kMap == CU_TENSOR_MAP_DATA_TYPE_FLOAT16 ? 0x7c00u : 0x7f80u;
  return (v & e) == e || ((v >> 16) & e) == e;
}
// The two values of a word, 0 in the place of those that are not finite.
template <class T>
__device__ __forceinline__ uint32_t pr_finite(uint32_t v) {
  return (pr_not_finite<T>(v & 0xffffu) ? 0u : v & 0xffffu) | (pr_not_finite<T>(v >> 16) ? 0u : v & 0xffff0000u);
}
// x + v where v is not finite, else x.
template <class T>
__device__ __forceinline__ float2 pr_add_odd(float2 x, uint32_t v) {
  const float2 f = HalfOps<T>::unpack(v);
  return make_float2(pr_not_finite<T>(v & 0xffffu) ? x.x + f.x : x.x, pr_not_finite<T>(v >> 16) ? x.y + f.y : x.y);
}

// ---- the kernel ---------------------------------------------------------------------

// An item (or a part of one) as the scheduler hands it out; seq < 0: there is
// none left.
struct PrItem {
  int seq, head, tile;
  int place, part, parts;  // place: of the launch; parts of the item's keys
  SeqSpan span;
};

// What hc_prompt_join_kernel needs of an item.
struct PrJoin {
  int parts;  // below 2: the item wrote its rows itself
  int head, tile;
  int row0, n;
};

// What every role derives from an item.
struct PrGeom {
  int nrows, r0, pos0;  // rows of the sequence's product, the item's first, position of the first new token
  int key0, key_hi;     // first key of the first tile, one behind the last key that a row sees
  int units;            // key tiles
};
__device__ __forceinline__ PrGeom pr_geom(const PrItem& it, int group, int window, int rows_per_item) {
  PrGeom g;
  g.nrows = it.span.n * group;
  g.r0 = it.tile * rows_per_item;
  g.pos0 = it.span.len - it.span.n;
  const int p_first = g.pos0 + g.r0 / group, p_last = g.pos0 + (min(g.r0 + rows_per_item, g.nrows) - 1) / group;
  const int key_lo = first_key(p_first, window);
  g.key_hi = min(it.span.len, p_last + 1);
  g.key0 = key_lo / PR_KEYS * PR_KEYS;
  g.units = g.key_hi > key_lo ? (g.key_hi - g.key0 + PR_KEYS - 1) / PR_KEYS : 0;
  if (it.parts > 1) {
    const int per = (g.units + it.parts - 1) / it.parts, first = it.part * per;
    g.key0 += first * PR_KEYS;
    g.units = max(0, min(per, g.units - first));
    g.key_hi = min(g.key_hi, g.key0 + g.units * PR_KEYS);
  } else if (it.part > 0) {
    g.units = 0;
  }
  return g;
}

// Keys [all_lo, all_hi] are seen by every row of the item (in a pair each
// CTA looks after half of every value for both).
struct PrBorder {
  int all_lo, all_hi;
  __device__ __forceinline__ bool tile(int k0) const { return k0 + PR_KEYS - 1 > all_hi || k0 < all_lo; }
  // of a tile's keys the first that some row may not see
  __device__ __forceinline__ int seen(int k0) const { return k0 < all_lo ? 0 : max(0, all_hi + 1 - k0); }
};
__device__ __forceinline__ PrBorder pr_border(const PrItem& it, const PrGeom& g, int group, int window, int rows_per_item) {
  return {first_key(g.pos0 + (min(g.r0 + rows_per_item, g.nrows) - 1) / group, window),
          min(it.span.len - 1, g.pos0 + g.r0 / group)};
}

template <class T, int D>
__global__ void __launch_bounds__(PrCfg<D>::kThreads, 1)
    hc_prompt_attn_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                          const __grid_constant__ PrArgs p) {
  using Cfg = PrCfg<D>;
  constexpr int CG = Cfg::CG, ST = Cfg::kStages, SPAN = PR_ROWS * CG;
  constexpr uint32_t FMT = HalfOps<T>::kMap == CU_TENSOR_MAP_DATA_TYPE_FLOAT16 ? 0u : 1u;
  // the roles behind the softmax warps 0 .. 7; each is a warp of its own, since
  // what it does per tile is a chain of dependent steps
  constexpr int LOAD_K = 8, LOAD_V = 9, ISSUER = 10, ISSUER_O = 11, ITEMS = 12, ITEM_WARPS = 4;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(16) uint4 clc_resp;
  __shared__ __align__(8) uint64_t q_full[2], q_free[2], k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], v_peer[ST];
  __shared__ __align__(8) uint64_t s_full[2], s_free[2], p_ready[2], pv_done[2], o_free, m_pass[4], l_pass[4], l_free;
  __shared__ __align__(8) uint64_t pv_seen[2][4];
  __shared__ __align__(8) uint64_t item_full[2], item_empty[2], clc_full, clc_ready, near_end;
  __shared__ PrItem s_items[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_odd[4];              // item number + 1 of a tile with a value that is not finite
  __shared__ float s_m[PR_ROWS];        // the rows' m after the last tile decided
  __shared__ float2 s_l[2][PR_ROWS];    // (m, l) of each warpgroup at an item's end
  const int t = int(threadIdx.x), warp = t >> 5, lane = t & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sq = base, sk = base + Cfg::kQs * Cfg::kQ, sv = sk + ST * Cfg::kK, so = sv + ST * Cfg::kK;
  const int group = p.a.heads / p.a.kv_heads, window = p.a.window;
  int* const err = p.a.err;
  if (warp == ISSUER) {
    if constexpr (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  if (t == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&v_peer[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], p.q_copy ? 1 : ITEM_WARPS * CG);
      mbar_init(&q_free[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4 * CG);
      mbar_init(&p_ready[i], 4 * CG);
      mbar_init(&pv_done[i], 1);
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 15);  // every warp but the one that finds them
    }
    for (int w = 0; w < 4; ++w) {
      mbar_init(&m_pass[w], 1);
      for (int i = 0; i < 2; ++i) mbar_init(&pv_seen[i][w], 1);
      mbar_init(&l_pass[w], 2);
    }
    mbar_init(&o_free, ITEM_WARPS * CG);
    mbar_init(&l_free, ITEM_WARPS);
    mbar_init(&clc_full, 1);
    mbar_init(&clc_ready, 1);
    mbar_init(&near_end, 1);
    for (int i = 0; i < 4; ++i) s_odd[i] = 0;
  }
  tc_before();
  sync_all<CG>();
  tc_after();
  const uint32_t tmem = s_tmem;
  pdl_launch_next();  // the next launch sets itself up on the SMs that this one leaves free
  pdl_wait_prior();
  const float sc = fmaxf(fabsf(p.a.scale_log2), 1.2e-38f);
  bool ok = true;

  // Item i of this CTA, read by every warp from the ring.
  const auto next_item = [&](int i, PrItem* it) {
    ok = ok && pr_wait(&item_full[i & 1], uint32_t(i >> 1) & 1u, err);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) return false;
    *it = s_items[i & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[i & 1]);
    return it->seq >= 0;
  };
  // Rows of the CTA's tile: row rr is pair rem + rr counted from token tok0,
  // divided by a multiplication (exact for rem + rr < 2^21 / group; it is below
  // 1152).
  const uint32_t inv_group = ((1u << 21) + uint32_t(group) - 1u) / uint32_t(group);
  const auto row_at = [&](int tok0, int rem, int rr) {  // (token, head of the group)
    const int x = rem + rr, tok = int((uint32_t(x) * inv_group) >> 21);
    return make_int2(tok0 + tok, x - tok * group);
  };
  // The CTA's rows of an item into the swizzled operand layout by `n` threads,
  // where TMA cannot (a group that does not divide 128 rows, a negative
  // scale): 16 bytes at a time, neighbouring lanes neighbouring bytes of a row, all copies
  // in flight together.  A negative scale flips Q's sign (so that the maximum
  // is that of the scores).
  const auto load_q = [&](const PrItem& it, const PrGeom& g, uint32_t slot, int i0, int n) {
    const int rt = g.r0 + int(rank) * PR_ROWS;
    const int tok0 = rt / group, rem = rt - tok0 * group;
    const T* src = static_cast<const T*>(p.a.q) + int64_t(it.span.row0) * p.a.q_stride + it.head * group * D;
    const auto dst = [&](int i) {
      const int rr = i / (D / 8), c = i % (D / 8);
      return sq + slot * Cfg::kQ + (c >> 3) * (PR_ROWS * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4);
    };
#pragma unroll 4
    for (int i = i0; i < PR_ROWS * (D / 8); i += n) {
      const int rr = i / (D / 8), c = i % (D / 8);
      const bool in = rt + rr < g.nrows;
      const int2 w = row_at(tok0, rem, in ? rr : 0);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst(i)),
                   "l"(in ? src + int64_t(w.x) * p.a.q_stride + w.y * D + c * 8 : src), "r"(in ? 16 : 0)
                   : "memory");
    }
    cp_async_wait_all();
    if (p.a.scale_log2 < 0.0f)
      for (int i = i0; i < PR_ROWS * (D / 8); i += n) {
        uint32_t x, y, z, w;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x), "=r"(y), "=r"(z), "=r"(w) : "r"(dst(i)) : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst(i)), "r"(x ^ 0x80008000u), "r"(y ^ 0x80008000u),
                     "r"(z ^ 0x80008000u), "r"(w ^ 0x80008000u)
                     : "memory");
      }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (CG == 2) asm volatile("fence.acq_rel.cluster;" ::: "memory");
    __syncwarp();
  };

  if (warp >= LOAD_K) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PR_REGS_OTHER));
  if (warp == LOAD_K || warp == LOAD_V) {
    // ---- K or V tiles.  Lane i looks up the tile's i-th page; one lane issues
    // the copies, with operands that are uniform in the warp (see elect_one).
    // In a pair each CTA brings half: of K's keys, and of V's dims.
    const bool is_k = warp == LOAD_K;
    const int keys = is_k ? Cfg::kKeys : PR_KEYS, pieces = is_k ? Cfg::kPieces : Cfg::kPiecesV;
    const int shift = is_k ? p.box_k : p.box_v, box = 1 << shift;  // (divisions would cost as much as a tile's products)
    const bool whole = is_k ? p.whole_k : p.whole_v;
    const int off = is_k ? int(rank) * Cfg::kKeys : 0, piece0 = is_k ? 0 : int(rank) * Cfg::kPiecesV;
    const CUtensorMap* map = is_k ? &kmap : &vmap;
    const uint32_t stages = is_k ? sk : sv;
    uint64_t* full = is_k ? k_full : v_full;
    uint64_t* empty = is_k ? k_empty : v_empty;
    // K's halves both report to the pair's first CTA, whose thread uses them
    const bool mine = !is_k || rank == 0;
    PrItem it;
    int st = 0;
    uint32_t ph = 1;  // parity of the stage's last release; the first use waits for none
    uint32_t nq = 0;  // items with tiles so far
    for (int n_it = 0; next_item(n_it, &it); ++n_it) {
      const PrGeom g = pr_geom(it, group, window, SPAN);
      const auto row_of = [&](int key) {
        if (!p.b.table) return it.span.row0 + key;
        const int page = p.b.table[int64_t(it.seq) * p.b.width + (key >> p.b.page_shift)];
        const bool in = page >= 0 && page < p.b.pages;
        if (!in && err) atomicExch(err, DEVICE_ERR_PAGE);
        return in ? int((int64_t(page) << p.b.page_shift) + (key & ((1 << p.b.page_shift) - 1))) : int(p.slots);
      };
      const int first = it.head * Cfg::kPieces + piece0;
      if (!is_k && p.q_copy && g.units > 0) {
        // Q: 128 (token, head of the group) rows from a token on, per 64 columns.
        // Rows behind the sequence's last token are another's, or zeros;
        // nothing of theirs is stored.
        const uint32_t slot = nq % Cfg::kQs, use = nq / Cfg::kQs;
        if (use > 0) ok = ok && pr_wait(&q_free[slot], (use - 1) & 1u, err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (rank == 0 && elect_one()) mbar_expect_tx(&q_full[slot], Cfg::kQ * CG);
        __syncwarp();
        const int token = it.span.row0 + (g.r0 + int(rank) * PR_ROWS) / group;
        const uint32_t bar = smem_u32(&q_full[slot]) & (CG == 2 ? kLeaderMask : 0xffffffffu);
        if (elect_one())
          for (int c = 0; c < Cfg::kPieces; ++c)
            pr_tma_q<CG>(sq + slot * Cfg::kQ + c * (PR_ROWS * 128), &qmap, c, it.head * group, token, bar);
        __syncwarp();
        ++nq;
      }
      // the next item is asked for shortly before this one's last keys: earlier
      // it would wait here while other CTAs run dry
      const int ask = max(0, g.units - PR_AHEAD);
      if (is_k && g.units == 0 && lane == 0) mbar_arrive(&near_end);
      for (int k0 = g.key0, i = 0; i < g.units; ++i, k0 += PR_KEYS) {
        if (is_k && i == ask && lane == 0) mbar_arrive(&near_end);
        const int n = min(PR_KEYS, g.key_hi - k0);
        const auto copies = [&](int from) { return (min(keys, max(0, n - from)) + box - 1) >> shift; };
        const int c_n = copies(off);
        const int row = lane < c_n ? row_of(k0 + off + lane * box) : 0;
        ok = ok && pr_wait(&empty[st], ph, err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t bar = smem_u32(&full[st]) & (CG == 2 && is_k ? kLeaderMask : 0xffffffffu), to = stages + st * Cfg::kK;
        if (mine && elect_one())
          mbar_expect_tx(&full[st], uint32_t((is_k && CG == 2 ? c_n + copies(Cfg::kKeys) : c_n) * box * pieces * 128));
        __syncwarp();
        if (whole) {
          const int r = __shfl_sync(0xffffffffu, row, 0);
          if (c_n && elect_one()) pr_tma<CG>(to, map, r, first, bar);
          __syncwarp();
        } else {
          for (int c = 0; c < c_n; ++c) {
            const int r = __shfl_sync(0xffffffffu, row, c);
            if (elect_one())
              for (int piece = 0; piece < pieces; ++piece)
                pr_tma<CG>(to + piece * (keys * 128) + c * box * 128, map, r, first + piece, bar);
            __syncwarp();
          }
        }
        if (++st == ST) st = 0, ph ^= 1u;
      }
      if (!ok) break;
    }
    // after a timeout: the copies that nobody else waits for
    if (!ok && mine)
      for (int i = 0; i < ST; ++i) pr_wait(&full[i], ph, nullptr);
    if (!ok && !is_k && rank == 0 && p.q_copy && nq > 0) pr_wait(&q_full[(nq - 1) % Cfg::kQs], (nq - 1) / Cfg::kQs & 1u, nullptr);
  } else if (warp == ISSUER || warp == ISSUER_O) {
    // ---- the products, issued by one thread of the pair's first CTA.  What
    // an issuer does between a barrier and its product is on every tile's path
    // (all its waits and descriptors took over 1000 clocks a tile, as
    // long as the products of head_dim 128), so everything else is waited for first.
    constexpr uint32_t id_qk = pr_idesc(FMT, PR_ROWS * CG, PR_KEYS, 0), id_pv = pr_idesc(FMT, PR_ROWS * CG, D, 1);
    int k_st = 0, v_st = 0;
    uint32_t k_ph = 0, v_ph = 0, sn = 0, on = 0;  // stages of K and V, their parities; S and O products so far
    uint32_t nq = 0;                              // items with rows so far
    const auto issue_s = [&](bool last) {
      tc_after();
      if (elect_one()) {
        const uint64_t a = pr_desc(sq + nq % Cfg::kQs * Cfg::kQ, 16, 1024), b = pr_desc(sk + k_st * Cfg::kK, 16, 1024);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          pr_mma_ss<CG>(tmem + (sn & 1) * 128, a + ((k >> 2) * (PR_ROWS * 128) + (k & 3) * 32) / 16,
                        b + ((k >> 2) * (Cfg::kKeys * 128) + (k & 3) * 32) / 16, id_qk, k > 0);
        pr_commit<CG>(&s_full[sn & 1]);
        pr_commit<CG>(&k_empty[k_st]);
        if (last) pr_commit<CG>(&q_free[nq % Cfg::kQs]);
      }
      __syncwarp();
      ++sn;
      if (++k_st == ST) k_st = 0, k_ph ^= 1u;
    };
    const auto issue_o = [&](const PrGeom& g, int o) {
      // keys behind the last one in use are not multiplied, 16 at a time
      const int steps = (min(PR_KEYS, g.key_hi - g.key0 - o * PR_KEYS) + 15) / 16;
      tc_after();
      if (elect_one()) {
        const uint32_t a = tmem + Cfg::p_col(on & 1);
        const uint64_t b = pr_desc(sv + v_st * Cfg::kK, PR_KEYS * 128, 1024);
        pr_mma_ts<CG>(tmem + Cfg::kTmemO, a, b, id_pv, o > 0);
        if (steps == PR_KEYS / 16) {
#pragma unroll
          for (int k = 1; k < PR_KEYS / 16; ++k) pr_mma_ts<CG>(tmem + Cfg::kTmemO, a + k * 8, b + k * (2048 / 16), id_pv, true);
        } else {
          for (int k = 1; k < steps; ++k) pr_mma_ts<CG>(tmem + Cfg::kTmemO, a + k * 8, b + k * (2048 / 16), id_pv, true);
        }
        pr_commit<CG>(&pv_done[on & 1]);
        pr_commit<CG>(&v_empty[v_st]);
      }
      __syncwarp();
      ++on;
      if (++v_st == ST) v_st = 0, v_ph ^= 1u;
    };
    const auto wait_v = [&] {
      return CG == 2 ? pr_wait2(&v_full[v_st], v_ph, &v_peer[v_st], v_ph, err) : pr_wait(&v_full[v_st], v_ph, err);
    };
    PrItem it;
    for (int n_it = 0; next_item(n_it, &it); ++n_it) {
      const PrGeom g = pr_geom(it, group, window, SPAN);
      if (g.units == 0 || (warp == ISSUER_O && !Cfg::kOwnP)) continue;
      if (rank != 0) {  // the second CTA reports its half of every V tile
        if (warp == ISSUER)
          for (int i = 0; i < g.units; ++i) {
            ok = ok && pr_wait(&v_full[v_st], v_ph, err);
            __syncwarp();
            if (lane == 0 && ok) arrive_leader<CG>(&v_peer[v_st]);
            if (++v_st == ST) v_st = 0, v_ph ^= 1u;
          }
        continue;
      }
      if (warp == ISSUER) {
        ok = ok && pr_wait(&q_full[nq % Cfg::kQs], nq / Cfg::kQs & 1u, err);
      }
      if constexpr (Cfg::kOwnP) {
        // S and O each by a warp of their own: all that orders them are the slots
        if (warp == ISSUER) {
          for (int i = 0; i < g.units; ++i) {
            if (sn >= 2) ok = ok && pr_wait2(&k_full[k_st], k_ph, &s_free[sn & 1], ((sn >> 1) - 1) & 1u, err);
            else ok = ok && pr_wait(&k_full[k_st], k_ph, err);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            issue_s(i + 1 == g.units);
          }
        } else {
          if (nq > 0) ok = ok && pr_wait(&o_free, (nq - 1) & 1u, err);
          for (int o = 0; o < g.units; ++o) {
            ok = ok && wait_v() && pr_wait(&p_ready[on & 1], (on >> 1) & 1u, err);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            issue_o(g, o);
          }
        }
      } else {
        // P lies in its S slot, so S of tile o + 2 has to be issued behind O of
        // tile o, by the same thread
        ok = ok && pr_wait(&k_full[k_st], k_ph, err);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) issue_s(g.units == 1);
        if (ok && g.units > 1) {
          ok = pr_wait(&k_full[k_st], k_ph, err);
          ok = __all_sync(0xffffffffu, ok);
          if (ok) issue_s(g.units == 2);
        }
        if (nq > 0) ok = ok && pr_wait(&o_free, (nq - 1) & 1u, err);
        for (int o = 0; o < g.units && ok; ++o) {
          ok = wait_v();
          if (o + 2 < g.units) ok = ok && pr_wait2(&k_full[k_st], k_ph, &p_ready[on & 1], (on >> 1) & 1u, err);
          else ok = ok && pr_wait(&p_ready[on & 1], (on >> 1) & 1u, err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          issue_o(g, o);
          if (o + 2 < g.units) issue_s(o + 3 == g.units);
        }
      }
      if (!ok) break;
      ++nq;
    }
  } else {
    // ---- the items: which one is next, its Q, and the rows of the one before.
    // The sequences' tiles in order, each sequence's last rows (the longest sums)
    // first, the KV heads of a tile side by side.
    const int w4 = warp - ITEMS;
    const auto tiles = [&](const SeqSpan& q) { return (q.n * group + SPAN - 1) / SPAN * p.a.kv_heads; };
    int s0 = 0, before = 0;  // places of the sequences before s0
    SeqSpan own{};           // of the 32 sequences from `loaded` on, lane by lane
    int loaded = -1, mine = 0, incl = 0;
    // Key tiles of all items, about (every item of a sequence taken for its last),
    // for an item's share: parts are as long as what a CTA gets when all get
    // the same, so that few items over long keys fill the machine once.
    int64_t all_units = 0;
    if (p.split > 1) {
      for (int s = lane; s < p.b.seqs; s += 32) {
        bool bad;
        const SeqSpan q = seq_span(p.b, s, &bad);
        const int64_t keys = window > 0 ? min(int64_t(q.len), int64_t(window) + SPAN / group) : q.len;
        all_units += int64_t(tiles(q)) * ((keys + PR_KEYS - 1) / PR_KEYS);
      }
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) all_units += __shfl_xor_sync(0xffffffffu, all_units, d);
    }
    uint32_t nq = 0, v0 = 0, ends = 0;  // items with tiles whose Q was asked for; tiles and items with tiles that ended
    // The values that the softmax warps took out of an item's border tiles, added
    // to the warp's stored rows that see them.  A lane takes two values of every
    // 64, of one key after the other, so no two lanes meet in a row.
    const auto add_odd = [&](const PrItem& it, const PrGeom& g, int tok0, int rem, bool live) {
      const PrBorder border = pr_border(it, g, group, window, SPAN);
      const int pos = g.pos0 + row_at(tok0, rem, live ? w4 * 32 + lane : 0).x;
      const int lim = live ? min(pos, it.span.len - 1) : -1, low = first_key(pos, window);
#pragma unroll 1
      for (int u = 0; u < g.units; ++u) {
        const int k0 = g.key0 + u * PR_KEYS, end = min(k0 + PR_KEYS, g.key_hi);
        if (!border.tile(k0)) continue;
#pragma unroll 1
        for (int j = k0 + border.seen(k0); j < end; ++j) {
          int64_t row = it.span.row0 + int64_t(j);
          if (p.b.table) {
            const int page = p.b.table[int64_t(it.seq) * p.b.width + (j >> p.b.page_shift)];
            if (page < 0 || page >= p.b.pages) continue;  // (its values were taken as 0)
            row = (int64_t(page) << p.b.page_shift) + (j & ((1 << p.b.page_shift) - 1));
          }
          const T* const src = static_cast<const T*>(p.v) + row * p.v_stride + int64_t(it.head) * D + lane * 2;
          uint32_t v[D / 64];
          bool here = false;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            v[c] = *reinterpret_cast<const uint32_t*>(src + c * 64);
            here = here || pr_not_finite<T>(v[c]);
          }
          if (!__any_sync(0xffffffffu, here)) continue;
          for (unsigned rows = __ballot_sync(0xffffffffu, j <= lim && j >= low); rows; rows &= rows - 1) {
            const int r = __ffs(rows) - 1;
            const int2 own = row_at(tok0, rem, w4 * 32 + r);
            const int64_t at = (int64_t(it.span.row0 + own.x) * p.a.heads + it.head * group + own.y) * D;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              if (!pr_not_finite<T>(v[c])) continue;
              const int d = c * 64 + lane * 2;
              if (it.parts > 1 || p.a.out_f32) {
                float* const to = it.parts > 1 ? p.part_o + (int64_t(it.place) * SPAN + int(rank) * PR_ROWS + w4 * 32) * D +
                                                     (d >> 2) * 128 + r * 4 + (d & 2)
                                               : static_cast<float*>(p.a.out) + at + d;
                *reinterpret_cast<float2*>(to) = pr_add_odd<T>(*reinterpret_cast<const float2*>(to), v[c]);
              } else {
                uint32_t* const to = reinterpret_cast<uint32_t*>(static_cast<T*>(p.a.out) + at + d);
                const float2 x = pr_add_odd<T>(HalfOps<T>::unpack(*to), v[c]);
                *to = HalfOps<T>::pack(x.x, x.y);
              }
            }
          }
        }
      }
      __syncwarp();
    };
    // An item's rows, once its last product has landed: a lane has a row's sums.
    const auto put_rows = [&](const PrItem& it, int n) {
      const PrGeom g = pr_geom(it, group, window, SPAN);
      if (it.part >= it.parts) return;  // no keys are left for this part
      const int rt = g.r0 + int(rank) * PR_ROWS, tok0 = rt / group, rem = rt - tok0 * group, rr = w4 * 32 + lane;
      const bool live = rt + rr < g.nrows;
      float m = -INFINITY, l = 0.0f;
      bool odd = false;
      if (g.units > 0) {
        v0 += uint32_t(g.units);
        ok = ok && pr_wait(&l_pass[w4], ends & 1u, err);
        ok = ok && pr_wait(&pv_done[(v0 - 1) & 1], ((v0 - 1) >> 1) & 1u, err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        tc_after();
        ++ends;
        // the even tiles' sum first, whichever warpgroup had them
        const uint32_t even = (v0 - uint32_t(g.units)) & 1u;
        const float2 a = s_l[even][rr], b = s_l[even ^ 1u][rr];
        m = fmaxf(a.x, b.x);
        l = m == -INFINITY ? a.y + b.y : a.y * ex2((a.x - m) * sc) + b.y * ex2((b.x - m) * sc);
        odd = *static_cast<volatile int*>(&s_odd[n & 3]) == n + 1;
        __syncwarp();
        if (lane == 0) mbar_arrive(&l_free);
      }
      const uint32_t oa = tmem + (uint32_t(w4) * 32u << 16) + Cfg::kTmemO;
      const auto done_with_o = [&] {  // the next item's first product may overwrite O
        if (g.units == 0) return;
        tc_before();
        __syncwarp();
        if (lane == 0) arrive_leader<CG>(&o_free);
      };
      if (it.parts > 1) {
        // a part leaves its sums undivided: [warp's 32 rows][head_dim / 4][row] float4
        const int64_t rows = int64_t(it.place) * SPAN + int(rank) * PR_ROWS + w4 * 32;
        float* const to = p.part_o + rows * D + lane * 4;
        p.part_ml[rows + lane] = make_float2(m * sc, l);
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t o[16];
          tm_ld16(oa + c, o);
          tm_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<uint4*>(to + (c + e) * 32) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
        done_with_o();
      } else {
        const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
        const int64_t tok = int64_t(it.span.row0 + tok0) * p.a.heads + it.head * group;
        if (live && p.a.lse) {
          const int2 own = row_at(0, rem, rr);
          p.a.lse[tok + own.x * p.a.heads + own.y] = l == 0.0f ? -INFINITY : 0.6931471805599453f * (m * sc + log2f(l));
        }
        // RB bytes of each of the warp's 32 rows at a time through shared memory,
        // so that neighbouring lanes store neighbouring bytes: 16-byte chunk c of
        // row r lies at chunk c ^ key(r)
        constexpr int RB = Cfg::kRowBytes, CH = RB / 16, STEP = 32 / CH;  // rows of one pass of the stores
        const uint32_t stage = so + uint32_t(w4) * (32 * RB);
        const auto key = [](int r) { return CH == 4 ? (r >> 1) & 3 : r & 7; };
        const auto put = [&](int c, uint32_t a, uint32_t b, uint32_t d, uint32_t e) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * RB + ((c ^ key(lane)) << 4)), "r"(a),
                       "r"(b), "r"(d), "r"(e)
                       : "memory");
        };
        const int esz = p.a.out_f32 ? 4 : 2;
        uint8_t* const out = static_cast<uint8_t*>(p.a.out) + tok * D * esz + lane % CH * 16;
        const auto flush = [&](int bytes) {  // the staged bytes start there in a row
          __syncwarp();
#pragma unroll 4
          for (int i = 0; i < 32; i += STEP) {
            const int r = i + lane / CH;
            const int2 w = row_at(0, rem, w4 * 32 + r);
            uint4 x;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                         : "r"(stage + r * RB + ((lane % CH ^ key(r)) << 4))
                         : "memory");
            if (rt + w4 * 32 + r < g.nrows)
              *reinterpret_cast<uint4*>(out + int64_t((w.x * p.a.heads + w.y) * D * esz + bytes)) = x;
          }
          __syncwarp();
        };
        const int cols = RB / esz;  // of a pass: a multiple of 16
#pragma unroll 1
        for (int c = 0; c < D; c += cols) {
#pragma unroll 1
          for (int h = 0; h < cols; h += 16) {
            uint32_t o[16];
            if (g.units > 0) {
              tm_ld16(oa + c + h, o);
              tm_wait_ld();
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = 0;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
            if (p.a.out_f32) {
#pragma unroll
              for (int e = 0; e < 4; ++e) put(h / 4 + e, o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            } else {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  w[i] = HalfOps<T>::pack(__uint_as_float(o[8 * e + 2 * i]), __uint_as_float(o[8 * e + 2 * i + 1]));
                put(h / 8 + e, w[0], w[1], w[2], w[3]);
              }
            }
          }
          if (c + cols == D) done_with_o();
          flush(c * esz);
        }
      }
      __syncwarp();
      if (odd) add_odd(it, g, tok0, rem, live);
    };
    int x = int(blockIdx.x) / CG;
    PrItem prev;
    for (int n_it = 0; ok; ++n_it) {
      PrItem it;
      it.seq = -1;
      if (warp == ITEMS) {
        if (n_it > 0) {
          // a pair's first CTA asks for both, once the other has read the last answer
          if (lane == 0) {
            mbar_expect_tx(&clc_full, 16);
            if (CG == 2 && rank == 1) arrive_leader<CG>(&clc_ready);
            if (rank == 0) {
              ok = pr_wait(&near_end, uint32_t(n_it - 1) & 1u, err);
              if (CG == 2) ok = ok && pr_wait(&clc_ready, uint32_t(n_it - 1) & 1u, err);
              if (ok) clc_ask<CG>(&clc_resp, &clc_full);
            }
          }
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          ok = pr_wait(&clc_full, uint32_t(n_it - 1) & 1u, err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const int first = clc_answer(&clc_resp);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          x = first < 0 ? -1 : first / CG;
          __syncwarp();
        }
        // first parts first, so that whole items start at once
        const int part = p.split > 1 && x >= 0 ? x / p.items : 0, y = x - part * p.items;
        if (y < before) s0 = before = 0, loaded = -1;
        while (y >= 0 && s0 < p.b.seqs) {  // 32 sequences at a time
          if (loaded != s0) {
            loaded = s0;
            own = SeqSpan{};
            bool bad = false;
            if (s0 + lane < p.b.seqs) own = seq_span(p.b, s0 + lane, &bad);
            if (bad && err) atomicExch(err, DEVICE_ERR_PAGE);
            mine = incl = tiles(own);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
              const int v = __shfl_up_sync(0xffffffffu, incl, d);
              if (lane >= d) incl += v;
            }
          }
          const unsigned hit = __ballot_sync(0xffffffffu, y < before + incl);
          if (hit) {
            const int w = __ffs(hit) - 1;
            const int at = y - before - __shfl_sync(0xffffffffu, incl - mine, w), n = __shfl_sync(0xffffffffu, mine, w);
            it.span.row0 = __shfl_sync(0xffffffffu, own.row0, w);
            it.span.n = __shfl_sync(0xffffffffu, own.n, w);
            it.span.len = __shfl_sync(0xffffffffu, own.len, w);
            it.seq = s0 + w;
            it.place = x;
            it.part = part;
            it.parts = 1;
            it.tile = at / p.a.kv_heads;
            it.head = at - it.tile * p.a.kv_heads;
            it.tile = n / p.a.kv_heads - 1 - it.tile;
            if (p.split > 1) {
              PrItem whole = it;
              whole.part = 0;
              const int units = pr_geom(whole, group, window, SPAN).units;
              const int64_t share = all_units > 0 ? int64_t(units) * p.workers / all_units : 1;
              const int parts = int(min(share, int64_t(min(p.split, units / PR_PART))));
              if (parts > 1) {
                const int per = (units + parts - 1) / parts;
                it.parts = (units + per - 1) / per;
              }
            }
            break;
          }
          before += __shfl_sync(0xffffffffu, incl, 31);
          s0 += 32;
        }
        if (n_it >= 2) {
          ok = pr_wait(&item_empty[n_it & 1], uint32_t((n_it >> 1) - 1) & 1u, err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        if (lane == 0) {
          if (p.split > 1 && rank == 0 && part == 0 && y >= 0) {
            PrJoin j{};
            if (it.seq >= 0) j = {it.parts, it.head, it.tile, it.span.row0, it.span.n};
            p.join[y] = j;
          }
          s_items[n_it & 1] = it;
          mbar_arrive(&item_full[n_it & 1]);
        }
        __syncwarp();
      } else {
        next_item(n_it, &it);
      }
      if (!ok) break;
      if (!p.q_copy && it.seq >= 0) {
        const PrGeom g = pr_geom(it, group, window, SPAN);
        if (g.units > 0) {
          const uint32_t slot = nq % Cfg::kQs, use = nq / Cfg::kQs;
          if (use > 0) ok = pr_wait(&q_free[slot], (use - 1) & 1u, err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          load_q(it, g, slot, t - 32 * ITEMS, 32 * ITEM_WARPS);
          if (lane == 0) arrive_leader<CG>(&q_full[slot]);
          ++nq;
        }
      }
      if (n_it > 0) {
        put_rows(prev, n_it - 1);
        if (!ok) break;
      }
      if (it.seq < 0) break;
      prev = it;
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PR_REGS_SOFTMAX));
    // ---- softmax: thread = row; warpgroup wg takes the tiles whose number is
    // of its parity (over all items)
    const int wg = warp >> 2, w4 = warp & 3, lt = t & 127;
    const uint32_t lanes = uint32_t(w4) * 32u << 16;
    uint32_t v0 = 0;    // tiles before this item
    uint32_t ends = 0;  // items with tiles so far
    const uint32_t sa = tmem + lanes + uint32_t(wg) * 128, pa = tmem + lanes + Cfg::p_col(uint32_t(wg));
    const uint32_t oa = tmem + lanes + Cfg::kTmemO;
    PrItem it;
    for (int n_it = 0; next_item(n_it, &it); ++n_it) {
      const PrGeom g = pr_geom(it, group, window, SPAN);
      const int rt = g.r0 + int(rank) * PR_ROWS;  // the CTA's first row
      const int tok0 = rt / group, rem = rt - tok0 * group;
      const bool live = rt + lt < g.nrows;
      const int2 own = row_at(tok0, rem, live ? lt : 0);  // token, head of the group
      const int pos = g.pos0 + own.x;
      const int lim = live ? min(pos, it.span.len - 1) : -1, low = first_key(pos, window);
      float m = -INFINITY, l = 0.0f;
      const PrBorder border = pr_border(it, g, group, window, SPAN);
      for (int u = int((v0 ^ uint32_t(wg)) & 1u); u < g.units; u += 2) {
        const uint32_t v = v0 + uint32_t(u);
        const int k0 = g.key0 + u * PR_KEYS;
        ok = ok && pr_wait(&s_full[wg], (v >> 1) & 1u, err);
        __syncwarp();
        tc_after();
        uint32_t s[PR_KEYS];
#pragma unroll
        for (int c = 0; c < PR_KEYS; c += 32) tm_ld32(sa + c, s + c);
        // meanwhile: m as the other warpgroup left it at the tile before (an
        // item's first tile only waits its turn: s_m is the last item's until then)
        float prev = -INFINITY;
        if (v > 0) ok = ok && pr_wait(&m_pass[w4], (v - 1) & 1u, err);
        if (u > 0) prev = *static_cast<volatile float*>(&s_m[lt]);
        __syncwarp();
        tm_wait_ld();
        if constexpr (Cfg::kOwnP) {
          tc_before();
          __syncwarp();
          if (lane == 0 && ok) arrive_leader<CG>(&s_free[wg]);
        }
        const bool edge = border.tile(k0);
        if (edge) {
          const int hi = lim - k0, lo = low - k0;
#pragma unroll
          for (int c = 0; c < PR_KEYS; ++c)
            if (c > hi) s[c] = 0xff800000u;
          if (k0 < border.all_lo) {
#pragma unroll
            for (int c = 0; c < PR_KEYS; ++c)
              if (c < lo) s[c] = 0xff800000u;
          }
        }
        float mx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(__uint_as_float(s[e]), __uint_as_float(s[4 + e]), __uint_as_float(s[8 + e]));
#pragma unroll
        for (int c = 12; c + 8 <= PR_KEYS; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(s[c + e]), __uint_as_float(s[c + 4 + e]));
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(s[PR_KEYS - 4 + e]), mx[e]);
        float mt = max3(mx[0], mx[1], max3(mx[2], mx[3], mx[3]));
        // a score of +inf makes the row NaN (inf - inf), as a NaN does
        if (mt == INFINITY) mt = __int_as_float(0x7fffffff);
        // prev = -inf and NaN included; rows of no token may hold anything, and are not worth a pass over O
        const bool grew = lim >= 0 && !(mt <= prev) && !((mt - prev) * sc <= PR_GROW);
        const float now = grew ? mt : prev;
        s_m[lt] = now;
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&m_pass[w4]);
        if (__any_sync(0xffffffffu, now != m)) {  // rare: some row's m moved, here or there
          if (now != m) l *= ex2((m - now) * sc);  // (l is 0 as long as m is -inf)
          m = now;
        }
        if (__any_sync(0xffffffffu, grew) && u > 0) {
          const float f = grew ? ex2((prev - mt) * sc) : 1.0f;
          // O to the new m, once the product before has landed.  A parity tells a
          // phase from the next only: where values arrive late, the product of tile v - 3
          // may still be on its way when the scores of tile v are here, and its
          // barrier then reads as if that of tile v - 1 had landed.  The other
          // warpgroup waits for the former on its way to tile v - 1's P, so it says when
          // it has.  (Where P lies in its S slot, the scores of tiles v - 1 and v were issued
          // and committed behind that product, by the same thread, and have landed.)
          if constexpr (Cfg::kOwnP) ok = ok && pr_wait(&pv_seen[wg ^ 1][w4], ((v - 1) >> 1) & 1u, err);
          ok = ok && pr_wait(&pv_done[wg ^ 1], ((v - 1) >> 1) & 1u, err);
          __syncwarp();
          tc_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tm_ld16(oa + c, o);
            tm_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tm_st16(oa + c, o);
          }
        }
        const float ms = m == -INFINITY ? 0.0f : m * sc;
        const uint64_t sc2 = pack2(sc, sc), nm2 = pack2(-ms, -ms);
        uint64_t sum[2] = {pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
#pragma unroll
        for (int b = 0; b < PR_KEYS; b += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float e0, e1;
            unpack2(fma2(pack2(__uint_as_float(s[b + c]), __uint_as_float(s[b + c + 1])), sc2, nm2), e0, e1);
            e0 = ex2(e0), e1 = ex2(e1);
            sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], pack2(e0, e1));
            pk[c >> 1] = HalfOps<T>::pack(e0, e1);
          }
          if (Cfg::kOwnP && b == 0) {  // the P slot: the product that read it last
            if (v >= 2) ok = ok && pr_wait(&pv_done[wg], ((v >> 1) - 1) & 1u, err);
            __syncwarp();
            tc_after();
          }
          tm_st16(pa + b / 2, pk);
        }
        {
          float a, b;
          unpack2(add2(sum[0], sum[1]), a, b);
          l += a + b;
        }
        if (edge) {
          // values that only some rows see and that are not finite become 0 for
          // the product (0 * inf); the item warps add them to the rows that see
          // them.  Values behind the last key in use become 0 up to the next 16
          // (the product goes no further).
          constexpr int CH = Cfg::kPiecesV * 8;  // 16-byte chunks of a key's values in this CTA
          const uint32_t st = v % ST, vt = sv + st * Cfg::kK;
          const int used = min(PR_KEYS, g.key_hi - k0), seen = border.seen(k0);
          const auto chunk = [&](int i) {
            return vt + (i % CH >> 3) * (PR_KEYS * 128) + i / CH * 128 + ((i & 7) << 4);
          };
          ok = ok && pr_wait(&v_full[st], (v / ST) & 1u, err);
          ok = __all_sync(0xffffffffu, ok);
          bool odd = false;
          const auto load = [&](int i, uint32_t(&w)[4]) {
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(chunk(i))
                         : "memory");
          };
          if (ok) {
#pragma unroll 4
            for (int i = seen * CH + lt; i < used * CH; i += 128) {
              uint32_t w[4];
              load(i, w);
              odd = odd || pr_not_finite<T>(w[0]) || pr_not_finite<T>(w[1]) || pr_not_finite<T>(w[2]) || pr_not_finite<T>(w[3]);
            }
            if (used & 15) {
              for (int i = used * CH + lt; i < (used + 15 & ~15) * CH; i += 128)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(chunk(i)), "r"(0u) : "memory");
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
          }
          odd = __any_sync(0xffffffffu, odd);
          if (odd) {
#pragma unroll 1
            for (int i = seen * CH + lt; i < used * CH; i += 128) {
              uint32_t w[4];
              load(i, w);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk(i)), "r"(pr_finite<T>(w[0])),
                           "r"(pr_finite<T>(w[1])), "r"(pr_finite<T>(w[2])), "r"(pr_finite<T>(w[3]))
                           : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          if (odd && lane == 0) {
            // both CTAs' rows are the sums of both CTAs' dims
            for (int c = 0; c < CG; ++c) {
              if constexpr (CG == 1)
                atomicExch(&s_odd[n_it & 3], n_it + 1);
              else
                asm volatile(
                    "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %1;\n\tst.shared::cluster.u32 [ra], %2;\n\t}\n" ::"r"(
                        smem_u32(&s_odd[n_it & 3])),
                    "r"(c), "r"(n_it + 1)
                    : "memory");
            }
          }
          // what was written here is read by the pair's products, and its flag by the other CTA
          if (CG == 2 && (odd || (used & 15))) asm volatile("fence.acq_rel.cluster;" ::: "memory");
        }
        tm_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0 && ok) {
          arrive_leader<CG>(&p_ready[wg]);
          if constexpr (Cfg::kOwnP) mbar_arrive(&pv_seen[wg][w4]);  // the product of tile v - 2 has landed
        }
      }
      v0 += uint32_t(g.units);
      // ---- the item's sums of this warpgroup's tiles go to the item warps
      if (g.units > 0) {
        if (ends > 0) ok = ok && pr_wait(&l_free, (ends - 1) & 1u, err);
        s_l[wg][lt] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(&l_pass[w4]);
        ++ends;
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
    }
    // after a timeout the products in flight get one more bounded wait before
    // the tensor memory is freed
    if (!ok) {
      pr_wait(&s_full[0], 0, nullptr);
      pr_wait(&pv_done[0], 0, nullptr);
    }
  }
  __syncwarp();
  tc_before();
  sync_all<CG>();
  tc_after();
  if (warp == ISSUER) {
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Joins the parts of an item's keys: a warp takes 32 rows, a thread each, and
// 32 of their columns (a multiple of 32 for every head_dim): the maximum of
// all parts, then the sums against it in the parts' order.
constexpr int PJ_THREADS = 256;
template <class T, int D>
__global__ void __launch_bounds__(PJ_THREADS) hc_prompt_join_kernel(const __grid_constant__ PrArgs p) {
  constexpr int SPAN = PR_ROWS * PrCfg<D>::CG, COLS = 32;
  pdl_launch_next();
  pdl_wait_prior();
  const int lane = int(threadIdx.x) & 31, unit = int(blockIdx.y) * (PJ_THREADS / 32) + (int(threadIdx.x) >> 5);
  const PrJoin it = p.join[blockIdx.x];
  if (it.parts < 2) return;
  const int group = p.a.heads / p.a.kv_heads;
  const int r32 = unit / (D / COLS) * 32, col = unit % (D / COLS) * COLS;
  const int x = it.tile * SPAN + r32 + lane;
  if (x >= it.n * group) return;
  const int64_t rows = int64_t(blockIdx.x) * SPAN + r32, step = int64_t(p.items) * SPAN;
  const float2* ml = p.part_ml + rows + lane;
  const float* po = p.part_o + rows * D + col * 32 + lane * 4;
  float mx = -INFINITY;
  for (int i = 0; i < it.parts; ++i) mx = fmaxf(mx, ml[i * step].x);
  const float ms = mx == -INFINITY ? 0.0f : mx;
  float o[COLS], sum = 0.0f;
#pragma unroll
  for (int e = 0; e < COLS; ++e) o[e] = 0.0f;
  for (int i = 0; i < it.parts; ++i) {
    const float2 s = ml[i * step];
    const float f = ex2(s.x - ms);
    sum += f * s.y;
#pragma unroll
    for (int e = 0; e < COLS; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(po + i * step * D + e * 32);
      o[e] += f * v.x, o[e + 1] += f * v.y, o[e + 2] += f * v.z, o[e + 3] += f * v.w;
    }
  }
  const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
  const int64_t row = int64_t(it.row0 + x / group) * p.a.heads + it.head * group + x % group;
  if (p.a.out_f32) {
    float* to = static_cast<float*>(p.a.out) + row * D + col;
#pragma unroll
    for (int e = 0; e < COLS; e += 4)
      *reinterpret_cast<float4*>(to + e) = make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
  } else {
    T* to = static_cast<T*>(p.a.out) + row * D + col;
#pragma unroll
    for (int e = 0; e < COLS; e += 8)
      *reinterpret_cast<uint4*>(to + e) =
          make_uint4(HalfOps<T>::pack(o[e] * inv, o[e + 1] * inv), HalfOps<T>::pack(o[e + 2] * inv, o[e + 3] * inv),
                     HalfOps<T>::pack(o[e + 4] * inv, o[e + 5] * inv), HalfOps<T>::pack(o[e + 6] * inv, o[e + 7] * inv));
  }
  if (col == 0 && p.a.lse) p.a.lse[row] = sum == 0.0f ? -INFINITY : 0.6931471805599453f * (mx + log2f(sum));
}

constexpr int kPrMaxSms = 160;  // that the workspace allows for
constexpr size_t pr_places(int sms, int dim) { return size_t(sms / (dim == 64 ? 1 : 2) * PR_PLACES); }
constexpr size_t pr_span(int dim) { return dim == 64 ? PR_ROWS : 2 * PR_ROWS; }

template <class T, int D>
cudaError_t launch_prompt(PrArgs& p, const KvSource& kv, void* workspace, cudaStream_t st) {
  using Cfg = PrCfg<D>;
  auto kernel = hc_prompt_attn_kernel<T, D>;
  static std::atomic<uint64_t> attr{0};
  cudaError_t e = once_per_current_device(attr, [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  });
  if (e != cudaSuccess) return e;
  const int page = 1 << p.b.page_shift;
  const int bk = p.b.table ? std::min(Cfg::kKeys, page) : Cfg::kKeys, bv = p.b.table ? std::min(PR_KEYS, page) : PR_KEYS;
  p.box_k = __builtin_ctz(bk);
  p.whole_k = bk == Cfg::kKeys, p.whole_v = bv == PR_KEYS;
  p.box_v = __builtin_ctz(bv);
  p.slots = int64_t(kv.slots);
  const int group = p.a.heads / p.a.kv_heads;
  CUtensorMap qm{}, km, vm;
  e = encode_kv_map(&km, HalfOps<T>::kMap, kv.k, kv.slots, kv.k_stride, p.a.kv_heads, D, bk,
                             p.whole_k ? Cfg::kPieces : 1);
  if (e == cudaSuccess)
    e = encode_kv_map(&vm, HalfOps<T>::kMap, kv.v, kv.slots, kv.v_stride, p.a.kv_heads, D, bv, p.whole_v ? Cfg::kPiecesV : 1);
  if (e != cudaSuccess) return e;
  p.q_copy = PR_ROWS % group == 0 && p.a.scale_log2 >= 0.0f;
  if (p.q_copy) {
    const cuuint64_t dims[4] = {64, D / 64, cuuint64_t(p.a.heads), cuuint64_t(p.b.rows)};
    const cuuint64_t strides[3] = {128, D * 2, cuuint64_t(p.a.q_stride) * 2};
    const cuuint32_t box[4] = {64, 1, cuuint32_t(group), cuuint32_t(PR_ROWS / group)};
    e = encode_map(&qm, HalfOps<T>::kMap, 4, p.a.q, dims, strides, box);
    if (e != cudaSuccess) return e;
  }
  // every sequence adds at most one tile to those of the rows put together
  constexpr int SPAN = PR_ROWS * Cfg::CG;
  const int64_t items =
      (int64_t(p.b.rows) * group / SPAN + std::min(p.b.seqs, p.b.rows)) * p.a.kv_heads;
  if (items * Cfg::CG > INT32_MAX) return cudaErrorInvalidValue;
  p.items = int(items);
  // Few items over long keys are cut into parts, as far as the workspace goes
  p.workers = sm_count() / Cfg::CG;
  const size_t places = pr_places(std::min(kPrMaxSms, sm_count()), D);
  const int64_t keys = p.b.table ? int64_t(p.b.width) << p.b.page_shift : p.a.max_q;
  const int64_t seen = p.a.window > 0 ? std::min(keys, int64_t(p.a.window) + SPAN / group + PR_KEYS) : keys;
  p.split = int(std::max<int64_t>(1, std::min(int64_t(places) / items, (seen + PR_KEYS - 1) / PR_KEYS / PR_PART)));
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + places * SPAN * D);
  p.join = reinterpret_cast<PrJoin*>(p.part_ml + places * SPAN);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(items * p.split * Cfg::CG));
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = Cfg::CG;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, kernel, qm, km, vm, p);
  if (e != cudaSuccess || p.split == 1) return e;
  return launch_pdl(hc_prompt_join_kernel<T, D>, dim3(unsigned(items), SPAN / 32 * (D / 32) / (PJ_THREADS / 32)), dim3(PJ_THREADS), 0, st, p);
}

template <class T>
cudaError_t launch_prompt_t(PrArgs& p, const KvSource& kv, void* ws, cudaStream_t st) {
  switch (p.a.dim) {
    case 64: return launch_prompt<T, 64>(p, kv, ws, st);
    case 128: return launch_prompt<T, 128>(p, kv, ws, st);
    default: return launch_prompt<T, 256>(p, kv, ws, st);
  }
}

}  // namespace

size_t attn_prompt_workspace_bytes(int dim) {
  const size_t places = pr_places(kPrMaxSms, dim);
  return places * pr_span(dim) * (size_t(dim) * 4 + 8) + places / 2 * sizeof(PrJoin);
}

cudaError_t launch_attn_prompt(const AttnArgs& a, const PagedBatch& b, const KvSource& kv, void* workspace,
                               cudaStream_t st) {
  PrArgs p{};
  p.a = a;
  p.b = b;
  p.v = kv.v;
  p.v_stride = int64_t(kv.v_stride);
  return kv.dtype == HPC_DTYPE_F16 ? launch_prompt_t<__half>(p, kv, workspace, st)
                                   : launch_prompt_t<__nv_bfloat16>(p, kv, workspace, st);
}

}  // namespace hc
