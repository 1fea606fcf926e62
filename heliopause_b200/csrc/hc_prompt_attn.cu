// hc_prompt_attn.cu -- causal attention of many query rows: whole prompts and
// chunks of them, on the fifth-generation tensor cores.
//
// The rows of one product are (new token, query head of the KV head's group)
// pairs in token order, 128 to a tile, so a tile covers 128 / group tokens: a
// short prompt still fills tiles, a tile's causal border is narrow, and a key
// tile read once serves the whole group.  Per tile of 128 keys:
//   S = Q K^T      tcgen05.mma, both operands in shared memory, S f32 in
//                  tensor memory (128 columns, two buffers);
//   P = 2^(S c - m c), c = scale log2(e): one thread per row, so maximum and
//                  sum (f32, of the unrounded P) need no exchange; P is rounded to
//                  the value type and replaces S in tensor memory;
//   O += P V       tcgen05.mma with P read from tensor memory, O f32 there
//                  (dim columns).
// m is the row's running maximum, but moved only when it grew by more than 8
// (in log2 units): P then stays below 2^8, which no type here minds, and the pass
// over O in tensor memory that a new maximum needs becomes rare (the first
// few tiles).  The tensor core runs S of unit u + 1 before O of unit u, so the
// exponentials of one unit hide behind the products of another.
//
// head_dim 64 and 128: one CTA, two row tiles (256 rows) that take turns: per
//   key tile 4 products, each K and V byte is used by 256 rows.
// head_dim 256: O alone takes 256 of the 512 columns, so a CTA holds one row tile and
//   two CTAs form a pair (cta_group::2): M = 256, each CTA brings half of the
//   keys of K and half of the dims of V, so again each byte serves 256 rows --
//   with one tile per CTA the K and V traffic from L2 would be 64 bytes per clock
//   and SM, which it does not deliver -- and shared memory holds two stages of each.
//
// K and V arrive by TMA, page by page or straight from packed rows, 128-byte
// swizzled, which is the operand layout of both products (K rows are K-major; V is
// N-major as it lies).  Keys that a row does not see get -inf scores and add
// nothing: values behind the sequence's end are zeroed before they are
// multiplied, and if a value that only some rows of a tile see is not finite
// (0 * inf), the tile's rows are summed again by plain loops over what they see.
#include <algorithm>
#include <atomic>

#include "hc_paged.cuh"

namespace hc {
namespace {

constexpr int PR_KEYS = 128;  // keys per tile
constexpr int PR_ROWS = 128;  // rows per tile
constexpr float PR_GROW = 8.0f;  // log2 units a maximum may grow before O is rescaled

template <int D>
struct PrCfg {
  static constexpr int CG = D == 256 ? 2 : 1;             // CTAs per MMA
  static constexpr int NQ = D == 256 ? 1 : 2;             // row tiles per CTA
  static constexpr int kThreads = 256 * NQ + 64;          // softmax warps, producer, MMA issuer
  static constexpr int kQ = PR_ROWS * D * 2;              // bytes of a row tile
  static constexpr int kK = PR_KEYS / CG * D * 2;         // bytes of K and V per stage in this CTA
  static constexpr int kStages = D == 64 ? 4 : 2;
  static constexpr int kSmem = 1024 + NQ * kQ + 2 * kStages * kK;
  static constexpr int kBoxK = PR_KEYS / CG;              // most key rows per TMA copy of K
  static constexpr int kPieces = D / 64;                  // 128-byte pieces of a row
  static constexpr int kPiecesV = kPieces / CG;           // of them V pieces in this CTA
  static constexpr uint32_t kTmemO = 256;                 // column of O (S buffers at 0 and 128)
};

struct PrArgs {
  AttnArgs a;
  PagedBatch b;
  const void* k;       // for the plain loops
  const void* v;
  int64_t k_stride, v_stride;
  int box_k, box_v;    // key rows per TMA copy
  int64_t slots;
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
__device__ __forceinline__ void tm_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      PR_I8(r, 0), PR_I8(r, 8), PR_I8(r, 16), PR_I8(r, 24)
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
// mbar_wait_parity without a timer read where the phase is already complete.
__device__ __forceinline__ bool pr_wait(uint64_t* bar, uint32_t parity, int* err) {
  unsigned long long t0 = 0;
  for (int it = 0;; ++it) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok)
                 : "r"(smem_u32(bar)), "r"(parity)
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
constexpr uint32_t kLeaderMask = 0xfeffffffu;  // a shared::cluster address in the pair's even CTA

// ---- the tile's sums by plain loops -----------------------------------------------

// One row of a tile, from global memory: keys [lo, hi] of sequence `s`.  Only
// for tiles where a value that some rows do not see is not finite.
template <class T, int D>
__device__ __noinline__ void pr_plain_row(const PrArgs& p, int s, int row0, int kv_head, const T* q, int lo, int hi,
                                          T* out, float* out32, float* lse) {
  const auto at = [&](const void* base, int64_t stride, int j) {
    int64_t r = row0 + int64_t(j);
    if (p.b.table) {
      const int page = p.b.table[int64_t(s) * p.b.width + (j >> p.b.page_shift)];
      const bool in = page >= 0 && page < p.b.pages;
      r = ((in ? int64_t(page) : 0) << p.b.page_shift) + (j & ((1 << p.b.page_shift) - 1));
    }
    return static_cast<const T*>(base) + r * stride + int64_t(kv_head) * D;
  };
  const auto score = [&](int j) {
    const T* k = at(p.k, p.k_stride, j);
    float d = 0.0f;
    for (int i = 0; i < D; i += 2) {
      const float2 x = HalfOps<T>::unpack(*reinterpret_cast<const uint32_t*>(q + i));
      const float2 y = HalfOps<T>::unpack(*reinterpret_cast<const uint32_t*>(k + i));
      d = fmaf(x.x, y.x, d);
      d = fmaf(x.y, y.y, d);
    }
    return d * p.a.scale_log2;
  };
  float m = -INFINITY;
  for (int j = lo; j <= hi; ++j) m = fmaxf(m, score(j));
  const float ms = m == -INFINITY ? 0.0f : m;
  for (int c = 0; c < D; c += 32) {
    float o[32], l = 0.0f;
    for (int i = 0; i < 32; ++i) o[i] = 0.0f;
    for (int j = lo; j <= hi; ++j) {
      const float e = ex2(score(j) - ms);
      const T* v = at(p.v, p.v_stride, j) + c;
      l += e;
      for (int i = 0; i < 32; i += 2) {
        const float2 y = HalfOps<T>::unpack(*reinterpret_cast<const uint32_t*>(v + i));
        o[i] = fmaf(e, y.x, o[i]);
        o[i + 1] = fmaf(e, y.y, o[i + 1]);
      }
    }
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    for (int i = 0; i < 32; ++i) {
      if (out32) out32[c + i] = o[i] * inv;
      else out[c + i] = HalfOps<T>::from(o[i] * inv);
    }
    if (c == 0 && lse) *lse = l == 0.0f ? -INFINITY : 0.6931471805599453f * (m + log2f(l));
  }
}

template <class T>
__device__ __forceinline__ bool pr_not_finite(uint32_t v) {
  constexpr uint32_t e = sizeof(T) && HalfOps<T>::kMap == CU_TENSOR_MAP_DATA_TYPE_FLOAT16 ? 0x7c00u : 0x7f80u;
  return (v & e) == e || ((v >> 16) & e) == e;
}

// ---- the kernel ---------------------------------------------------------------------

template <class T, int D>
__global__ void __launch_bounds__(PrCfg<D>::kThreads, 1)
    hc_prompt_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                          const __grid_constant__ PrArgs p) {
  using Cfg = PrCfg<D>;
  constexpr int CG = Cfg::CG, NQ = Cfg::NQ, ST = Cfg::kStages, SPAN = PR_ROWS * NQ * CG;
  constexpr uint32_t FMT = HalfOps<T>::kMap == CU_TENSOR_MAP_DATA_TYPE_FLOAT16 ? 0u : 1u;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full, k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], s_full[2], p_ready[2], pv_done[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_item[3];  // sequence, KV head, tile
  __shared__ SeqSpan s_span;
  __shared__ int s_sum[Cfg::kThreads / 32];
  __shared__ int s_odd;
  __shared__ float s_half[2][2][NQ * PR_ROWS];  // [unit parity][column half][row]
  const int t = int(threadIdx.x), warp = t >> 5, lane = t & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sq = base, sk = base + NQ * Cfg::kQ, sv = sk + ST * Cfg::kK;
  const int group = p.a.heads / p.a.kv_heads, window = p.a.window;
  constexpr int PRODUCER = 8 * NQ, ISSUER = 8 * NQ + 1;
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
    mbar_init(&q_full, 8 * NQ * CG);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 8 * CG);
      mbar_init(&pv_done[i], 1);
    }
    s_item[0] = -1;
    s_odd = 0;
  }
  pdl_wait_prior();

  // ---- which item: the sequences' tiles in order, each sequence's last rows
  // (the longest sums) first, the KV heads of a tile side by side.  Thread t
  // counts sequences [t * per, ...); with up to one each, its span stays in
  // registers and the lengths are read once.
  {
    const int x = int(blockIdx.x) / CG;
    const int per = (p.b.seqs + Cfg::kThreads - 1) / Cfg::kThreads;
    const auto tiles = [&](const SeqSpan& q) { return (q.n * group + SPAN - 1) / SPAN * p.a.kv_heads; };
    int mine = 0;
    SeqSpan own{};
    bool any_bad = false;
    for (int i = 0; i < per; ++i) {
      const int s = t * per + i;
      if (s >= p.b.seqs) break;
      bool bad;
      own = seq_span(p.b, s, &bad);
      mine += tiles(own);
      any_bad = any_bad || bad;
    }
    if (any_bad && p.a.err) atomicExch(p.a.err, DEVICE_ERR_PAGE);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_sum[warp] = incl;
    tc_before();
    __syncthreads();
    for (int i = 0; i < warp; ++i) incl += s_sum[i];
    if (incl - mine <= x && x < incl) {
      int at = incl - mine;
      for (int s = t * per;; ++s) {
        bool bad;
        const SeqSpan q = per == 1 ? own : seq_span(p.b, s, &bad);
        const int n = tiles(q);
        if (x < at + n) {
          s_item[0] = s;
          s_item[1] = (x - at) % p.a.kv_heads;
          s_item[2] = n / p.a.kv_heads - 1 - (x - at) / p.a.kv_heads;
          s_span = q;
          break;
        }
        at += n;
      }
    }
  }
  sync_all<CG>();
  tc_after();
  const uint32_t tmem = s_tmem;
  const int seq = s_item[0], kv_head = s_item[1];
  if (seq >= 0) {
    const SeqSpan sp = s_span;
    const int nrows = sp.n * group, r0 = s_item[2] * SPAN, pos0 = sp.len - sp.n;
    const int p_first = pos0 + r0 / group, p_last = pos0 + (min(r0 + SPAN, nrows) - 1) / group;
    const int key_lo = window > 0 ? max(0, p_first - window + 1) : 0, key_hi = min(sp.len, p_last + 1);
    const int tile0 = key_lo / PR_KEYS;
    const int ntiles = key_hi > key_lo ? (key_hi + PR_KEYS - 1) / PR_KEYS - tile0 : 0;
    bool ok = true;

    if (warp == PRODUCER) {
      // ---- K and V tiles; lane i takes copies i, i + 32, ... of (page, piece)
      const auto row_of = [&](int key) {
        if (!p.b.table) return sp.row0 + key;
        const int page = p.b.table[int64_t(seq) * p.b.width + (key >> p.b.page_shift)];
        const bool in = page >= 0 && page < p.b.pages;
        if (!in && p.a.err) atomicExch(p.a.err, DEVICE_ERR_PAGE);
        return in ? int((int64_t(page) << p.b.page_shift) + (key & ((1 << p.b.page_shift) - 1))) : int(p.slots);
      };
      for (int j = 0; j < ntiles && ok; ++j) {
        const int st = j % ST, ph = j / ST, k0 = (tile0 + j) * PR_KEYS;
        const int n = min(PR_KEYS, sp.len - k0);
        // K: this CTA's keys [k0 + rank * 128 / CG, ...), every piece
        if (ph > 0) ok = pr_wait(&k_empty[st], uint32_t(ph - 1) & 1u, p.a.err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const auto copies_k = [&](int r) {
          return (min(Cfg::kBoxK, max(0, n - r * Cfg::kBoxK)) + p.box_k - 1) / p.box_k;
        };
        if (lane == 0 && rank == 0) {
          int c = 0;
          for (int r = 0; r < CG; ++r) c += copies_k(r);
          mbar_expect_tx(&k_full[st], uint32_t(c * p.box_k * D * 2));
        }
        __syncwarp();
        const int ck = copies_k(int(rank));
        for (int i = lane; i < ck * Cfg::kPieces; i += 32) {
          const int c = i / Cfg::kPieces, piece = i % Cfg::kPieces;
          const int row = row_of(k0 + int(rank) * Cfg::kBoxK + c * p.box_k);
          pr_tma<CG>(sk + st * Cfg::kK + piece * (Cfg::kBoxK * 128) + c * p.box_k * 128, &kmap, row,
                     kv_head * Cfg::kPieces + piece, smem_u32(&k_full[st]) & (CG == 2 ? kLeaderMask : 0xffffffffu));
        }
        // V: every key, this CTA's pieces
        if (ph > 0) ok = pr_wait(&v_empty[st], uint32_t(ph - 1) & 1u, p.a.err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int cv = (n + p.box_v - 1) / p.box_v;
        if (lane == 0) mbar_expect_tx(&v_full[st], uint32_t(cv * p.box_v * Cfg::kPiecesV * 128));
        __syncwarp();
        for (int i = lane; i < cv * Cfg::kPiecesV; i += 32) {
          const int c = i / Cfg::kPiecesV, piece = i % Cfg::kPiecesV;
          const int row = row_of(k0 + c * p.box_v);
          pr_tma<CG>(sv + st * Cfg::kK + piece * (PR_KEYS * 128) + c * p.box_v * 128, &vmap, row,
                     kv_head * Cfg::kPieces + int(rank) * Cfg::kPiecesV + piece, smem_u32(&v_full[st]));
        }
      }
      // the copies that nobody else waits for: after a timeout, all in flight
      if (!ok)
        for (int i = 0; i < ST; ++i) {
          if (rank == 0) mbar_wait_parity_sleep(&k_full[i], 0, p.a.err);
          mbar_wait_parity_sleep(&v_full[i], 0, p.a.err);
        }
    } else if (warp == ISSUER) {
      // ---- one thread of the pair's first CTA issues every product
      if (rank == 0 && lane == 0 && ntiles > 0) {
        constexpr uint32_t id_qk = pr_idesc(FMT, PR_ROWS * CG, PR_KEYS, 0), id_pv = pr_idesc(FMT, PR_ROWS * CG, D, 1);
        const int units = ntiles * NQ;
        const auto qk = [&](int u) {
          const int j = u / NQ, q = u % NQ, st = j % ST;
          if (q == 0) ok = ok && pr_wait(&k_full[st], uint32_t(j / ST) & 1u, p.a.err);
          if (!ok) return;
          tc_after();
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            pr_mma_ss<CG>(tmem + uint32_t(u & 1) * 128,
                          pr_desc(sq + q * Cfg::kQ + (k >> 2) * (PR_ROWS * 128) + (k & 3) * 32, 16, 1024),
                          pr_desc(sk + st * Cfg::kK + (k >> 2) * (Cfg::kBoxK * 128) + (k & 3) * 32, 16, 1024), id_qk, k > 0);
          pr_commit<CG>(&s_full[u & 1]);
          if (q == NQ - 1) pr_commit<CG>(&k_empty[st]);
        };
        ok = pr_wait(&q_full, 0, p.a.err);
        qk(0);
        for (int u = 0; u < units && ok; ++u) {
          if (u + 1 < units) qk(u + 1);
          const int j = u / NQ, q = u % NQ, st = j % ST;
          ok = ok && pr_wait(&p_ready[u & 1], uint32_t(u >> 1) & 1u, p.a.err);
          ok = ok && pr_wait(&v_full[st], uint32_t(j / ST) & 1u, p.a.err);
          if (!ok) break;
          tc_after();
#pragma unroll
          for (int k = 0; k < PR_KEYS / 16; ++k)
            pr_mma_ts<CG>(tmem + Cfg::kTmemO + q * D, tmem + uint32_t(u & 1) * 128 + k * 8,
                          pr_desc(sv + st * Cfg::kK + k * 2048, PR_KEYS * 128, 1024), id_pv, j > 0 || k > 0);
          pr_commit<CG>(&pv_done[u & 1]);
          if (q == NQ - 1) pr_commit<CG>(&v_empty[st]);
        }
      }
      __syncwarp();
    } else {
      // ---- softmax: thread = row of row tile q, half `half` of its columns
      const int q = warp >> 3, half = (warp >> 2) & 1, lt = t & 127, lt2 = t & 255;
      const uint32_t lanes = uint32_t(warp & 3) * 32u << 16;
      const int pair_bar = 1 + q * 4 + (warp & 3);  // the two warps that share 32 rows
      const int rt = r0 + (int(rank) * NQ + q) * PR_ROWS;  // the tile's first row
      const int r = rt + lt;
      const bool live = r < nrows;
      const int pos = pos0 + (live ? r : nrows - 1) / group;
      const int lim = live ? min(pos, sp.len - 1) : -1, low = window > 0 ? pos - window + 1 : 0;
      // keys [all_lo, all_hi] are seen by every row of the tile
      const int all_hi = min(sp.len - 1, pos0 + min(rt, nrows - 1) / group);
      const int all_lo = window > 0 ? pos0 + min(rt + PR_ROWS - 1, nrows - 1) / group - window + 1 : 0;
      const float sc = fmaxf(fabsf(p.a.scale_log2), 1.2e-38f);
      // Rows of the tile to (token, head of the group): row rr is pair
      // rem + rr counted from token tok0, divided by a multiplication (exact
      // below 2^21 / group, and rem + rr < 1152)
      const int tok0 = rt / group, rem = rt - tok0 * group;
      const uint32_t inv_group = ((1u << 21) + uint32_t(group) - 1u) / uint32_t(group);
      const auto row_at = [&](int rr) {  // element offset of the row's head in a [row][heads][D] tensor, less the token's
        const int x = rem + rr, tok = int((uint32_t(x) * inv_group) >> 21);
        return make_int2(sp.row0 + tok0 + tok, kv_head * group + x - tok * group);
      };
      // Q into the swizzled operand layout, 16 bytes at a time, neighbouring
      // lanes neighbouring bytes of a row, eight loads in flight per thread.
      // A negative scale flips Q's sign.
      {
        const uint32_t flip = p.a.scale_log2 < 0.0f ? 0x80008000u : 0u;
        constexpr int N = PR_ROWS * (D / 8) / 256, B = N < 8 ? N : 8;
#pragma unroll 1
        for (int i0 = 0; i0 < N; i0 += B) {
          uint4 v[B];
#pragma unroll
          for (int i = 0; i < B; ++i) {
            const int at = (i0 + i) * 256 + lt2, rr = at / (D / 8), c = at % (D / 8);
            v[i] = make_uint4(0, 0, 0, 0);
            if (rt + rr < nrows && ntiles > 0) {
              const int2 w = row_at(rr);
              v[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.a.q) + int64_t(w.x) * p.a.q_stride + w.y * D +
                                                     c * 8);
            }
          }
#pragma unroll
          for (int i = 0; i < B; ++i) {
            const int at = (i0 + i) * 256 + lt2, rr = at / (D / 8), c = at % (D / 8);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sq + q * Cfg::kQ + (c >> 3) * (PR_ROWS * 128) +
                                                                         rr * 128 + (((c & 7) ^ (rr & 7)) << 4)),
                         "r"(v[i].x ^ flip), "r"(v[i].y ^ flip), "r"(v[i].z ^ flip), "r"(v[i].w ^ flip)
                         : "memory");
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (CG == 2) asm volatile("fence.acq_rel.cluster;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive_leader<CG>(&q_full);
      }
      constexpr int HC = PR_KEYS / 2;  // columns of a half
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < ntiles; ++j) {
        const int u = j * NQ + q, buf = u & 1, st = j % ST, k0 = (tile0 + j) * PR_KEYS;
        ok = ok && pr_wait(&s_full[buf], uint32_t(u >> 1) & 1u, p.a.err);
        __syncwarp();
        tc_after();
        uint32_t s[HC];
        const uint32_t sa = tmem + lanes + uint32_t(buf) * 128;
#pragma unroll
        for (int c = 0; c < HC; c += 32) tm_ld32(sa + half * HC + c, s + c);
        tm_wait_ld();
        const bool edge = k0 + PR_KEYS - 1 > all_hi || k0 < all_lo;
        if (edge) {
          const int hi = lim - k0 - half * HC, lo = low - k0 - half * HC;
#pragma unroll
          for (int c = 0; c < HC; ++c)
            if (c > hi || c < lo) s[c] = 0xff800000u;
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[c] = __uint_as_float(s[c]);
#pragma unroll
        for (int c = 4; c + 4 < HC; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            mx[e] = fmaxf(mx[e], fmaxf(__uint_as_float(s[c + e]), __uint_as_float(s[c + 4 + e])));
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(s[HC - 4 + e]));
        float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        // the other half's maximum: one exchange between the two warps of the
        // rows (the slot alternates, so the next one need not wait for readers)
        s_half[j & 1][half][q * PR_ROWS + lt] = mt;
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        mt = fmaxf(mt, s_half[j & 1][half ^ 1][q * PR_ROWS + lt]);
        const bool grew = mt > m && !((mt - m) * sc <= PR_GROW);  // m = -inf included
        if (__any_sync(0xffffffffu, grew)) {
          const float f = grew ? ex2((m - mt) * sc) : 1.0f;
          if (grew) m = mt;
          l *= f;
          if (j > 0) {
            const int up = u - NQ;  // the tile's previous product must have landed
            ok = ok && pr_wait(&pv_done[up & 1], uint32_t(up >> 1) & 1u, p.a.err);
            __syncwarp();
            tc_after();
            const uint32_t oa = tmem + lanes + Cfg::kTmemO + uint32_t(q * D + half * (D / 2));
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
              uint32_t o[16];
              tm_ld16(oa + c, o);
              tm_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tm_st16(oa + c, o);
            }
          }
        }
        const float ms = m == -INFINITY ? 0.0f : m * sc;
        const uint64_t sc2 = pack2(sc, sc), nm2 = pack2(-ms, -ms);
        uint64_t sum[2] = {pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
        uint32_t pk[HC / 2];
#pragma unroll
        for (int c = 0; c < HC; c += 2) {
          const uint64_t x = fma2(pack2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sc2, nm2);
          float a, b;
          unpack2(x, a, b);
          a = ex2(a), b = ex2(b);
          sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], pack2(a, b));
          pk[c >> 1] = HalfOps<T>::pack(a, b);
        }
        // P takes the first half of S's columns: the other warp's scores are
        // read (the exchange above came after both loads)
        tm_st32(sa + half * (HC / 2), pk);
        {
          float a, b;
          unpack2(add2(sum[0], sum[1]), a, b);
          l += a + b;
        }
        if (edge) {
          // values of keys behind the end, and values that only some rows see
          ok = ok && pr_wait(&v_full[st], uint32_t(j / ST) & 1u, p.a.err);
          ok = __all_sync(0xffffffffu, ok);
          const uint32_t vt = sv + st * Cfg::kK;
          bool odd = false;
          if (ok)
            for (int i = lt2; i < PR_KEYS * Cfg::kPiecesV * 8; i += 256) {
              const int key = i / (Cfg::kPiecesV * 8), c = i % (Cfg::kPiecesV * 8);
              const uint32_t at = vt + (c >> 3) * (PR_KEYS * 128) + key * 128 + ((c & 7) << 4);
              if (k0 + key >= sp.len) {
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0u) : "memory");
              } else {
                uint32_t a, b, d, e;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(a), "=r"(b), "=r"(d), "=r"(e)
                             : "r"(at)
                             : "memory");
                odd = odd || pr_not_finite<T>(a) || pr_not_finite<T>(b) || pr_not_finite<T>(d) || pr_not_finite<T>(e);
              }
            }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          if (__any_sync(0xffffffffu, odd) && lane == 0) {
            // both CTAs' rows are the sums of both CTAs' dims
            if constexpr (CG == 1) {
              atomicExch(&s_odd, 1);
            } else {
              for (int c = 0; c < CG; ++c)
                asm volatile(
                    "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %1;\n\tst.shared::cluster.u32 [ra], %2;\n\t}\n" ::"r"(
                        smem_u32(&s_odd)),
                    "r"(c), "r"(1)
                    : "memory");
            }
          }
          // what was written here is read by the pair's products
          if (CG == 2) asm volatile("fence.acq_rel.cluster;" ::: "memory");
        } else if (CG == 2) {
          // the issuer sees only its own CTA's V barrier: a CTA's arrival on
          // p_ready also says that its half of V has landed
          ok = ok && pr_wait(&v_full[st], uint32_t(j / ST) & 1u, p.a.err);
          __syncwarp();
        }
        tm_wait_st();
        tc_before();
        // a warp whose wait gave up walks on without arriving, to meet the
        // other warp at the exchanges; nothing after it completes
        ok = __all_sync(0xffffffffu, ok);
        if (lane == 0 && ok) arrive_leader<CG>(&p_ready[buf]);
      }
      // ---- the rows' outputs
      if (ntiles > 0) {
        const int ul = (ntiles - 1) * NQ + q;
        ok = ok && pr_wait(&pv_done[ul & 1], uint32_t(ul >> 1) & 1u, p.a.err);
        ok = __all_sync(0xffffffffu, ok);
        tc_after();
      }
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");  // the last maxima are read
      s_half[0][half][q * PR_ROWS + lt] = l;
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      l = s_half[0][0][q * PR_ROWS + lt] + s_half[0][1][q * PR_ROWS + lt];
      if (ok) {
        const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
        const int2 own = row_at(live ? lt : 0);
        const int64_t row = int64_t(own.x) * p.a.heads + own.y;
        float* lse = p.a.lse ? p.a.lse + row : nullptr;
        if (ntiles > 0 && *static_cast<volatile int*>(&s_odd)) {
          if (live && half == 0)
            pr_plain_row<T, D>(p, seq, sp.row0, kv_head, static_cast<const T*>(p.a.q) + int64_t(own.x) * p.a.q_stride + own.y * D,
                               max(low, 0), lim, static_cast<T*>(p.a.out) + row * D,
                               p.a.out_f32 ? static_cast<float*>(p.a.out) + row * D : nullptr, lse);
        } else {
          // through shared memory (the operands are done with), so that a warp
          // stores whole rows: 16-byte chunk c of row rr at chunk c ^ (rr % 8)
          const int chunks = p.a.out_f32 ? D / 4 : D / 8;  // 16-byte chunks of a row
          const uint32_t stage = base + uint32_t(q * PR_ROWS) * chunks * 16;
#pragma unroll 1
          for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
            uint32_t o[32];
            if (ntiles > 0) {
              tm_ld32(tmem + lanes + Cfg::kTmemO + uint32_t(q) * D + c, o);
              tm_wait_ld();
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0;
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
            const auto put = [&](int chunk, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + (lt * chunks + (chunk ^ (lt & 7))) * 16), "r"(x),
                           "r"(y), "r"(z), "r"(w)
                           : "memory");
            };
            if (p.a.out_f32) {
#pragma unroll
              for (int e = 0; e < 32; e += 4) put((c + e) / 4, o[e], o[e + 1], o[e + 2], o[e + 3]);
            } else {
              uint32_t w[16];
#pragma unroll
              for (int e = 0; e < 16; ++e)
                w[e] = HalfOps<T>::pack(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
#pragma unroll
              for (int e = 0; e < 16; e += 4) put((c + 2 * e) / 8, w[e], w[e + 1], w[e + 2], w[e + 3]);
            }
          }
          if (live && lse && half == 0) *lse = l == 0.0f ? -INFINITY : 0.6931471805599453f * (m * sc + log2f(l));
        }
      }
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      if (ok && !(ntiles > 0 && *static_cast<volatile int*>(&s_odd))) {
        // the two warps of these 32 rows store 16 rows each
        const int chunks = p.a.out_f32 ? D / 4 : D / 8;
        const uint32_t stage = base + uint32_t(q * PR_ROWS) * chunks * 16;
        const int first = (warp & 3) * 32 + half * 16;
        const int shift = 31 - __clz(chunks);
#pragma unroll 4
        for (int i = lane; i < 16 * chunks; i += 32) {
          const int rr = first + (i >> shift), c = i & (chunks - 1);
          if (rt + rr >= nrows) break;
          uint4 v;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(stage + (rr * chunks + (c ^ (rr & 7))) * 16)
                       : "memory");
          const int2 w = row_at(rr);
          *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.a.out) + ((int64_t(w.x) * p.a.heads + w.y) * chunks + c) * 16) = v;
        }
      }
      // after a timeout the products in flight get one more bounded wait
      // before the tensor memory is freed
      if (!ok) {
        pr_wait(&s_full[0], 0, nullptr);
        pr_wait(&pv_done[0], 0, nullptr);
      }
      __syncwarp();
    }
  }
  tc_before();
  sync_all<CG>();
  tc_after();
  if (warp == ISSUER) {
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <class T, int D>
cudaError_t launch_prompt(PrArgs& p, const KvSource& kv, cudaStream_t st) {
  using Cfg = PrCfg<D>;
  auto kernel = hc_prompt_attn_kernel<T, D>;
  static std::atomic<uint64_t> attr{0};
  cudaError_t e = once_per_current_device(attr, [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  });
  if (e != cudaSuccess) return e;
  const int page = 1 << p.b.page_shift;
  p.box_k = p.b.table ? std::min(Cfg::kBoxK, page) : Cfg::kBoxK;
  p.box_v = p.b.table ? std::min(PR_KEYS, page) : PR_KEYS;
  p.slots = int64_t(kv.slots);
  CUtensorMap km, vm;
  e = encode_kv_map(&km, HalfOps<T>::kMap, kv.k, kv.slots, kv.k_stride, p.a.kv_heads, D, p.box_k, 1);
  if (e == cudaSuccess)
    e = encode_kv_map(&vm, HalfOps<T>::kMap, kv.v, kv.slots, kv.v_stride, p.a.kv_heads, D, p.box_v, 1);
  if (e != cudaSuccess) return e;
  // every sequence adds at most one tile to those of the rows put together
  constexpr int SPAN = PR_ROWS * Cfg::NQ * Cfg::CG;
  const int group = p.a.heads / p.a.kv_heads;
  const int64_t items =
      (int64_t(p.b.rows) * group / SPAN + std::min(p.b.seqs, p.b.rows)) * p.a.kv_heads;
  if (items * Cfg::CG > INT32_MAX) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(items * Cfg::CG));
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
  return cudaLaunchKernelEx(&cfg, kernel, km, vm, p);
}

template <class T>
cudaError_t launch_prompt_t(PrArgs& p, const KvSource& kv, cudaStream_t st) {
  switch (p.a.dim) {
    case 64: return launch_prompt<T, 64>(p, kv, st);
    case 128: return launch_prompt<T, 128>(p, kv, st);
    default: return launch_prompt<T, 256>(p, kv, st);
  }
}

}  // namespace

cudaError_t launch_attn_prompt(const AttnArgs& a, const PagedBatch& b, const KvSource& kv, cudaStream_t st) {
  PrArgs p{};
  p.a = a;
  p.b = b;
  p.k = kv.k;
  p.v = kv.v;
  p.k_stride = int64_t(kv.k_stride);
  p.v_stride = int64_t(kv.v_stride);
  return kv.dtype == HPC_DTYPE_F16 ? launch_prompt_t<__half>(p, kv, st) : launch_prompt_t<__nv_bfloat16>(p, kv, st);
}

}  // namespace hc
