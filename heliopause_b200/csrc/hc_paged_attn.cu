// hc_paged_attn.cu -- attention of few query rows over a long cache.
//
//   o = sum_j softmax_j(scale * q . k_j) v_j  over the keys j <= pos of the
// query's sequence (j > pos - window with a window), for the newest tokens of
// every sequence: one (decode), a pending token and its drafts (verify), or
// any number.  The query heads that share a KV head and the new tokens of the
// sequence are the rows of one product, so each key and value is read once
// for all of them: per element 2 rows multiply-adds for 2 bytes, which the
// memory bounds by far up to 24 rows.
//
// Work: an item is (sequence, KV head, block of 8, 16 or 24 rows); its keys are cut
// into tiles of 64, and the tiles of all items, in order, are dealt out
// evenly to a grid that fills the machine -- a CTA takes a run of tiles, so
// ragged batches balance to a tile and one long sequence spreads over every
// SM, with no plan made on the host.  A CTA that holds an item's every tile
// writes its output; items cut by a CTA boundary leave a partial (running
// maximum, sum, unnormalised output; at most two per CTA, in the workspace)
// which hc_attn_join_kernel joins in tile order.
//
// CTA: a producer warp keeps a ring of K and V tiles full by TMA (page by
// page, each piece of 64 elements 128-byte swizzled), so 100 KB and more are
// in flight per SM whatever the warps compute.  For every 8 rows (16 with heads
// of 64) four consumer warps take 16 keys each of every tile and share nothing
// until the item ends: S^T = K Q^T
// (m16n8k16: the 16 keys are the M side, so 8 rows cost 8 columns instead of
// a padded 16), the row maxima and sums in f32 over the warp's own keys, P
// rounded to the cache's type for the second product -- its relative 2^-8
// (2^-11 for f16) is that of the values it multiplies -- and O^T += V^T P^T in
// f32 registers.  The four partials of a row are added in shared memory at the end.
//
// A key that a row does not see adds nothing to it, whatever its value
// holds: values at or behind the sequence's end are zeroed in shared memory
// before they are multiplied (stale pages may hold NaN), and where a tile has
// keys that only some rows see, a value that is not finite sends the warp
// through scalar sums over the visible pairs.
//
// Measured: 32 sequences of 8192 to 32768 keys, 32 / 8 heads of 128 (2.72 GB)
// 398 to 410 us with the join, 6.7 TB/s -- a little above a plain copy's rate; 64 chats
// of 1 to 4096 keys, 8 / 2 heads of 256 (268 MB) 52.5 us, 5.1 TB/s: there each CTA
// has 29 tiles and pays some 12 us of starts, page look-ups, merge and join
// beside them, which is what one chat's token takes (10.3 to 10.8 us).
#include <algorithm>
#include <atomic>

#include "hc_paged.cuh"

namespace hc {
namespace {

constexpr int AR_TILE = 64;      // keys per tile
constexpr int AR_WARPS = 4;      // consumer warps of a row group, 16 keys of a tile each
constexpr float LN2 = 0.6931471805599453f;

// Rows of a block: RG groups of 8 NB, each with four consumer warps; the
// groups share the ring's tiles.
template <int D, int NB, int RG>
struct RowsCfg {
  static constexpr int kRows = 8 * NB * RG;
  static constexpr int kThreads = 32 * (AR_WARPS * RG + 1);
  static constexpr int kCtas = D == 256 || RG > 2 ? 1 : D == 128 || RG == 2 ? 2 : 3;  // per SM
  static constexpr int kSlot = AR_TILE * D * 2;                                      // one K or V tile
  static constexpr int kMergeRow = D + 4;                                            // floats; + 4: no bank conflicts
  static constexpr int kMergeWarps = RG == 1 ? AR_WARPS : 2;                         // whose rows of a group fit there
  static constexpr int kMerge = kMergeWarps * kRows * kMergeRow * 4;
  // fragments of Q^T in shared memory, where registers for them would spill
  static constexpr bool kQShared = RG > 1;
  static constexpr int kQ = kQShared ? kRows * D * 2 : 0;
  // as many tiles in flight as fit beside the merge buffer
  static constexpr int kFit = (227 * 1024 / kCtas - 2048 - 1024 - kMerge - kQ) / kSlot;
  static constexpr int kSlots = kFit < 16 ? kFit : 16;
  static constexpr int kSmem = 1024 + kSlots * kSlot + kMerge + kQ;                       // + alignment
};

// What the join kernel needs of an item cut by a CTA boundary.
struct JoinRec {
  int head, block;  // block < 0: nothing to join
  int row0, n;      // the sequence's rows
  int last;         // last CTA that may hold tiles of it
};

struct RowsWork {
  float* o;      // [2 * grid][rows of a block][D]
  float2* ml;    // [2 * grid][rows of a block]: maximum (in log2 units), sum
  JoinRec* rec;  // [grid]
};

struct RowsArgs {
  AttnArgs a;
  PagedBatch b;
  RowsWork w;
  int box_rows;  // rows of one TMA copy: min(page_size, 64), 64 without pages
  int64_t slots; // rows of the tensor maps (a coordinate there reads zeros)
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <class T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Tiles of one sequence's items: [first, first + count), the same for its
// heads and row blocks (a block skips those it does not see); at least one,
// so that rows that see nothing are written too.
struct SeqTiles {
  int first, count, blocks;
};
template <int R>
__device__ __forceinline__ SeqTiles seq_tiles(const SeqSpan& q, int group, int window) {
  SeqTiles t;
  t.first = first_key(q.len - q.n, window) / AR_TILE;
  t.count = max(1, (q.len + AR_TILE - 1) / AR_TILE - t.first);
  t.blocks = (q.n * group + R - 1) / R;
  return t;
}

__device__ __forceinline__ long long cta_begin(long long total, int c, int grid) { return total * c / grid; }

// The keys [lo, hi) that some row of an item's block sees.
struct BlockSpan {
  int rows, lo, hi, pos0;
};
template <int R>
__device__ __forceinline__ BlockSpan block_span(const SeqSpan& q, int block, int group, int window) {
  BlockSpan s;
  const int r0 = block * R;
  s.rows = min(R, q.n * group - r0);
  s.pos0 = q.len - q.n;  // position of the sequence's first new token
  const int p_first = s.pos0 + r0 / group, p_last = s.pos0 + (r0 + s.rows - 1) / group;
  s.lo = first_key(p_first, window);
  s.hi = min(q.len, p_last + 1);
  return s;
}

// A run of tiles [u, end) walked item by item.
struct Walk {
  int s, head, block, tile;  // tile: within the item, 0 ..
  long long u, end;
};

template <class T>
__device__ __forceinline__ bool not_finite2(uint32_t v);
template <>
__device__ __forceinline__ bool not_finite2<__half>(uint32_t v) {
  return (v & 0x7c00u) == 0x7c00u || (v & 0x7c000000u) == 0x7c000000u;
}
template <>
__device__ __forceinline__ bool not_finite2<__nv_bfloat16>(uint32_t v) {
  return (v & 0x7f80u) == 0x7f80u || (v & 0x7f800000u) == 0x7f800000u;
}

template <class T, int D, int NB, int RG>
__global__ void __launch_bounds__(RowsCfg<D, NB, RG>::kThreads, RowsCfg<D, NB, RG>::kCtas)
    hc_attn_rows_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                        const __grid_constant__ RowsArgs p) {
  using Cfg = RowsCfg<D, NB, RG>;
  constexpr int R = Cfg::kRows, GR = 8 * NB, KS = D / 16, WARPS = AR_WARPS * RG;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[Cfg::kSlots], empty[Cfg::kSlots];
  __shared__ long long s_sum[Cfg::kThreads / 32];
  __shared__ Walk s_walk;
  __shared__ float2 s_ml[WARPS][GR];
  const int t = int(threadIdx.x), warp = t >> 5, lane = t & 31;
  const int grid = int(gridDim.x), cta = int(blockIdx.x);
  const int group = p.a.heads / p.a.kv_heads, window = p.a.window;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* merge = reinterpret_cast<float*>(smem_raw + (base - smem_u32(smem_raw)) + Cfg::kSlots * Cfg::kSlot);
  if (t == 0) {
    for (int i = 0; i < Cfg::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], WARPS);
    }
  }
  pdl_launch_next();
  pdl_wait_prior();

  // ---- this CTA's run of tiles: thread t counts sequences [t * per, ...)
  const int per = (p.b.seqs + Cfg::kThreads - 1) / Cfg::kThreads;
  long long mine = 0;
  bool any_bad = false;
  for (int i = 0; i < per; ++i) {
    const int s = t * per + i;
    if (s >= p.b.seqs) break;
    bool bad;
    const SeqSpan q = seq_span(p.b, s, &bad);
    any_bad = any_bad || bad;
    const SeqTiles st = seq_tiles<R>(q, group, window);
    mine += (long long)p.a.kv_heads * st.blocks * st.count;
  }
  if (any_bad && p.a.err) atomicExch(p.a.err, DEVICE_ERR_PAGE);
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_sum[warp] = incl;
  if (t == 0) p.w.rec[cta].block = -1;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int i = 0; i < Cfg::kThreads / 32; ++i) {
    if (i < warp) incl += s_sum[i];
    total += s_sum[i];
  }
  const long long u0 = cta_begin(total, cta, grid), u1 = cta_begin(total, cta + 1, grid);
  if (u0 >= u1) {  // (fewer tiles than CTAs: the join reads an empty part here)
    if (t < R) p.w.ml[2 * cta * R + t] = make_float2(-INFINITY, 0.0f);
    return;
  }
  if (incl - mine <= u0 && u0 < incl) {
    long long at = incl - mine;
    for (int s = t * per;; ++s) {
      bool bad;
      const SeqTiles st = seq_tiles<R>(seq_span(p.b, s, &bad), group, window);
      const long long n = (long long)p.a.kv_heads * st.blocks * st.count;
      if (u0 < at + n) {
        const long long d = u0 - at;
        Walk w;
        w.s = s;
        w.tile = int(d % st.count);
        w.block = int(d / st.count % st.blocks);
        w.head = int(d / st.count / st.blocks);
        w.u = u0;
        w.end = u1;
        s_walk = w;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  Walk w = s_walk;

  int it = 0;  // K and V tiles so far: slot it % kSlots, phase it / kSlots
  bool ok = true;
  if (warp == WARPS) {
    // ---- producer: lane i looks up the tile's i-th page; one lane issues the
    // copies, with operands that are uniform in the warp (elect_one)
    const int box = p.box_rows, box_shift = __ffs(box) - 1, ppt = AR_TILE >> box_shift;
    while (w.u < w.end && ok) {
      bool bad;
      const SeqSpan q = seq_span(p.b, w.s, &bad);
      const SeqTiles st = seq_tiles<R>(q, group, window);
      for (; w.head < p.a.kv_heads && w.u < w.end && ok; ++w.head, w.block = 0) {
        for (; w.block < st.blocks && w.u < w.end && ok; ++w.block, w.tile = 0) {
          const BlockSpan sp = block_span<R>(q, w.block, group, window);
          for (; w.tile < st.count && w.u < w.end && ok; ++w.tile, ++w.u) {
            const int k0 = (st.first + w.tile) * AR_TILE;
            if (k0 + AR_TILE <= sp.lo || k0 >= sp.hi) continue;
            const int copies = (min(AR_TILE, q.len - k0) + box - 1) >> box_shift;
            int row = 0;
            if (lane < ppt && lane < copies) {
              if (p.b.table) {
                const int key = k0 + lane * box;
                const int page = p.b.table[int64_t(w.s) * p.b.width + (key >> p.b.page_shift)];
                const bool in = page >= 0 && page < p.b.pages;
                if (!in && p.a.err) atomicExch(p.a.err, DEVICE_ERR_PAGE);
                row = in ? int((int64_t(page) << p.b.page_shift) + (key & ((1 << p.b.page_shift) - 1))) : int(p.slots);
              } else {
                row = q.row0 + k0;
              }
            }
#pragma unroll
            for (int kv = 0; kv < 2; ++kv, ++it) {
              const int slot = it % Cfg::kSlots, ph = it / Cfg::kSlots;
              if (ph > 0 && !mbar_wait_parity_sleep(&empty[slot], uint32_t(ph - 1) & 1u, p.a.err)) ok = false;
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
              if (elect_one()) mbar_expect_tx(&full[slot], uint32_t(copies * box * D * 2));
              __syncwarp();
              for (int c = 0; c < copies; ++c) {
                const int r = __shfl_sync(0xffffffffu, row, c);
                if (elect_one())
                  tma_load_3d(base + slot * Cfg::kSlot + c * box * D * 2, kv ? &vmap : &kmap, 0, r, w.head * (D / 64),
                              smem_u32(&full[slot]));
                __syncwarp();
              }
            }
          }
        }
        if (w.block < st.blocks) break;
      }
      if (w.head < p.a.kv_heads) break;
      ++w.s, w.head = 0, w.block = 0, w.tile = 0;
    }
    // nothing of this CTA's is in flight when it ends: the consumers wait
    // for every copy; after a timeout the copies issued are waited for here
    if (!ok)
      for (int i = max(0, it - Cfg::kSlots); i < it; ++i)
        mbar_wait_parity_sleep(&full[i % Cfg::kSlots], uint32_t(i / Cfg::kSlots) & 1u, p.a.err);
    return;
  }

  // ---- consumers
  const int lr = lane >> 2, lc = lane & 3;
  const int rg = warp / AR_WARPS, kw = warp % AR_WARPS;  // row group, and the keys' quarter
  const int box_shift = __ffs(p.box_rows) - 1;
  // byte offset of key row j of a tile (its first 128-byte piece); pieces are box_rows * 128 apart
  const auto row_off = [&](int j) { return (j >> box_shift) * (p.box_rows * D * 2) + (j & (p.box_rows - 1)) * 128; };
  const int piece = p.box_rows * 128;
  const auto group_sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + rg), "n"(32 * AR_WARPS) : "memory"); };
  // this lane's ldmatrix rows (fixed within the tile) and 16-byte chunks
  const int kj = kw * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, kc = lane >> 4;
  const int vj = kw * 16 + (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;
  const uint32_t koff = uint32_t(row_off(kj)), voff = uint32_t(row_off(vj));
  while (w.u < w.end) {
    bool bad;
    const SeqSpan q = seq_span(p.b, w.s, &bad);
    const SeqTiles st = seq_tiles<R>(q, group, window);
    for (; w.head < p.a.kv_heads && w.u < w.end; ++w.head, w.block = 0) {
      for (; w.block < st.blocks && w.u < w.end; ++w.block, w.tile = 0) {
        const BlockSpan sp = block_span<R>(q, w.block, group, window);
        const int r0 = w.block * R + rg * GR;               // this group's first row
        const int rows = min(GR, sp.rows - rg * GR);        // none: below 1
        // B fragments of Q^T, straight from the rows
        uint32_t qf[Cfg::kQShared ? 1 : NB][KS][2];
        uint2* qs = reinterpret_cast<uint2*>(merge + Cfg::kMerge / 4) + rg * NB * KS * 32;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int r = r0 + nb * 8 + lr;
          const bool in = r - r0 < rows;
          const T* src = static_cast<const T*>(p.a.q) + int64_t(q.row0 + (in ? r / group : 0)) * p.a.q_stride +
                         (w.head * group + (in ? r % group : 0)) * D + lc * 2;
          if constexpr (Cfg::kQShared) {
#pragma unroll
            for (int k = kw; k < KS; k += AR_WARPS)
              qs[(k * NB + nb) * 32 + lane] = make_uint2(in ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u,
                                                         in ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u);
          } else {
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              qf[nb][k][0] = in ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
              qf[nb][k][1] = in ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
            }
          }
        }
        if constexpr (Cfg::kQShared) group_sync();
        // keys [low, lim] of this lane's two rows of every 8
        int lim[NB][2], low[NB][2];
        float m[NB][2], l[NB][2];
        float o[NB][KS][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = nb * 8 + lc * 2 + e;
            const int pos = sp.pos0 + (r0 + r) / group;
            lim[nb][e] = r < rows ? min(pos, q.len - 1) : -1;
            low[nb][e] = first_key(pos, window);
            m[nb][e] = -INFINITY;
            l[nb][e] = 0.0f;
          }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nb][k][e] = 0.0f;
        // every key of [all_lo, all_hi] is seen by every row of the group
        const int all_hi = min(q.len - 1, sp.pos0 + r0 / group);
        const int all_lo = first_key(sp.pos0 + (r0 + rows - 1) / group, window);
        const int tile0 = w.tile;
        for (; w.tile < st.count && w.u < w.end; ++w.tile, ++w.u) {
          const int k0 = (st.first + w.tile) * AR_TILE;
          // after a wait gave up the warp only walks on, to meet the others at the barriers
          if (!ok || k0 + AR_TILE <= sp.lo || k0 >= sp.hi) continue;
          const int j0 = k0 + kw * 16;  // this warp's keys
          const bool idle = rows < 1 || j0 >= sp.hi || j0 + 16 <= sp.lo;
          const int ks = it % Cfg::kSlots, kph = it / Cfg::kSlots;
          const int vs = (it + 1) % Cfg::kSlots, vph = (it + 1) / Cfg::kSlots;
          it += 2;
          uint32_t pb[NB][2];
          float pr[NB][4];
          ok = mbar_wait_parity(&full[ks], uint32_t(kph) & 1u, p.a.err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) continue;
          if (!idle) {
            float s[2][NB][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[h][nb][e] = 0.0f;
            const uint32_t kb = base + ks * Cfg::kSlot + koff;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              uint32_t af[4];
              ldsm4(af, kb + (k >> 2) * piece + ((((k & 3) * 2 + kc) ^ (kj & 7)) << 4));
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                if constexpr (Cfg::kQShared) {
                  const uint2 f = qs[(k * NB + nb) * 32 + lane];
                  mma16<T>(s[k & 1][nb], af, f.x, f.y);
                } else {
                  mma16<T>(s[k & 1][nb], af, qf[nb][k][0], qf[nb][k][1]);
                }
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[ks]);
            bool grew = false;
            float corr[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int ja = j0 + lr, jb = ja + 8;
                float a = (s[0][nb][e] + s[1][nb][e]) * p.a.scale_log2;
                float b = (s[0][nb][2 + e] + s[1][nb][2 + e]) * p.a.scale_log2;
                a = ja <= lim[nb][e] && ja >= low[nb][e] ? a : -INFINITY;
                b = jb <= lim[nb][e] && jb >= low[nb][e] ? b : -INFINITY;
                float mx = fmaxf(a, b);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float mn = fmaxf(m[nb][e], mx);
                const float ms = mn == -INFINITY ? 0.0f : mn;
                corr[nb][e] = ex2(m[nb][e] - ms);
                grew = grew || mn != m[nb][e];
                m[nb][e] = mn;
                pr[nb][e] = ex2(a - ms);
                pr[nb][2 + e] = ex2(b - ms);
                l[nb][e] = l[nb][e] * corr[nb][e] + (pr[nb][e] + pr[nb][2 + e]);
              }
              // [key][row] quarters -> [row][key], the B fragment of the second product
              pb[nb][0] = transpose8(HalfOps<T>::pack(pr[nb][0], pr[nb][1]));
              pb[nb][1] = transpose8(HalfOps<T>::pack(pr[nb][2], pr[nb][3]));
            }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[nb][k][e] *= corr[nb][e & 1];
            }
          } else {
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[ks]);
          }
          ok = mbar_wait_parity(&full[vs], uint32_t(vph) & 1u, p.a.err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) continue;
          if (!idle) {
            const uint32_t vt = base + vs * Cfg::kSlot;
            bool scalar = false;
            if (j0 + 15 > all_hi || j0 < all_lo) {  // some row does not see some of these keys
              bool odd = false;
              for (int i = lane; i < 16 * (D / 8); i += 32) {
                const int jj = i / (D / 8), c = i % (D / 8), j = kw * 16 + jj;
                const uint32_t at = vt + row_off(j) + (c >> 3) * piece + (((c & 7) ^ (j & 7)) << 4);
                if (j0 + jj >= q.len) {
                  asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(at), "r"(0u) : "memory");
                } else {
                  uint32_t v0, v1, v2, v3;
                  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                               : "=r"(v0), "=r"(v1), "=r"(v2), "=r"(v3)
                               : "r"(at)
                               : "memory");
                  odd = odd || not_finite2<T>(v0) || not_finite2<T>(v1) || not_finite2<T>(v2) || not_finite2<T>(v3);
                }
              }
              // the zeros are read by ldmatrix, and the slot's next copy
              // (the async proxy) must come after them
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              scalar = __any_sync(0xffffffffu, odd);
              __syncwarp();
            }
            if (!scalar) {
#pragma unroll
              for (int k = 0; k < KS; ++k) {
                uint32_t af[4];
                ldsm4_t(af, vt + voff + (k >> 2) * piece + ((((k & 3) * 2 + vc) ^ (vj & 7)) << 4));
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mma16<T>(o[nb][k], af, pb[nb][0], pb[nb][1]);
              }
            } else {
              for (int jj = 0; jj < 16; ++jj) {
                const int j = j0 + jj;
                if (j >= q.len) break;
                const int rj = kw * 16 + jj;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const float pe = __shfl_sync(0xffffffffu, jj < 8 ? pr[nb][e] : pr[nb][2 + e], (jj & 7) * 4 + lc);
                    if (j > lim[nb][e] || j < low[nb][e]) continue;
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                      for (int h = 0; h < 2; ++h) {
                        const int d = k * 16 + h * 8 + lr;
                        uint16_t bits;
                        asm volatile("ld.shared.u16 %0, [%1];"
                                     : "=h"(bits)
                                     : "r"(vt + row_off(rj) + (d >> 6) * piece + ((((d >> 3) & 7) ^ (rj & 7)) << 4) +
                                           (d & 7) * 2)
                                     : "memory");
                        const float v = HalfOps<T>::unpack(bits).x;
                        o[nb][k][h * 2 + e] = fmaf(pe, v, o[nb][k][h * 2 + e]);
                      }
                  }
                }
              }
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[vs]);
        }
        // ---- the item (or this CTA's part of it) is done: add the warps up
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = l[nb][e];
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            if (lr == 0) s_ml[warp][nb * 8 + lc * 2 + e] = make_float2(m[nb][e], v);
          }
        // one group: its four warps lay their sums out as rows and write the
        // rows' total.  More groups have room for two warps' rows each: two
        // warps hand their sums to the other two first, in the fragments' own
        // layout (one group with that step too: one chat's token 12.2 us instead
        // of 11.5, 32 long documents 414 instead of 402).
        constexpr int MW = Cfg::kMergeWarps;
        float* mb = merge + rg * MW * GR * Cfg::kMergeRow;
        if (MW == 2 && kw >= 2) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int k = 0; k < KS; ++k)
              *reinterpret_cast<float4*>(mb + (((kw - 2) * NB + nb) * KS + k) * 128 + lane * 4) =
                  make_float4(o[nb][k][0], o[nb][k][1], o[nb][k][2], o[nb][k][3]);
        }
        if constexpr (MW == 2) group_sync();
        const bool whole = tile0 == 0 && w.tile == st.count;
        const int part = tile0 > 0 ? 2 * cta : 2 * cta + 1;
        // a row's maximum, the warps' factors against it, and its sum
        const auto row_stats = [&](int r, float (&f)[AR_WARPS], float& mx) {
          mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < AR_WARPS; ++i) mx = fmaxf(mx, s_ml[rg * AR_WARPS + i][r].x);
          const float ms = mx == -INFINITY ? 0.0f : mx;
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < AR_WARPS; ++i) {
            const float2 v = s_ml[rg * AR_WARPS + i][r];
            f[i] = ex2(v.x - ms);
            sum += f[i] * v.y;
          }
          return sum;
        };
        if (MW == 2 && kw < 2) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float fa[2], fb[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float f[AR_WARPS], mx;
              row_stats(nb * 8 + lc * 2 + e, f, mx);
              fa[e] = kw ? f[1] : f[0], fb[e] = kw ? f[3] : f[2];
            }
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              const float4 x = *reinterpret_cast<const float4*>(mb + ((kw * NB + nb) * KS + k) * 128 + lane * 4);
              o[nb][k][0] = fa[0] * o[nb][k][0] + fb[0] * x.x, o[nb][k][1] = fa[1] * o[nb][k][1] + fb[1] * x.y;
              o[nb][k][2] = fa[0] * o[nb][k][2] + fb[0] * x.z, o[nb][k][3] = fa[1] * o[nb][k][3] + fb[1] * x.w;
            }
          }
        }
        if constexpr (MW == 2) group_sync();
        if (kw < MW) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                mb[(kw * GR + nb * 8 + lc * 2 + (e & 1)) * Cfg::kMergeRow + k * 16 + (e >> 1) * 8 + lr] = o[nb][k][e];
        }
        group_sync();
        constexpr int TPR = 32 * AR_WARPS / GR;  // threads per row
        {
          const int tg = kw * 32 + lane, r = tg / TPR, c = tg % TPR;
          if (r < rows) {
            float f[AR_WARPS], mx;
            const float sum = row_stats(r, f, mx);
            const int row = q.row0 + (r0 + r) / group, head = w.head * group + (r0 + r) % group;
            const int64_t prow = int64_t(part) * R + rg * GR + r;
            const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
            for (int d = c * 4; d < D; d += TPR * 4) {
              float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
              for (int i = 0; i < MW; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(mb + (i * GR + r) * Cfg::kMergeRow + d);
                const float g = MW == 2 ? 1.0f : f[i];
                v.x += g * x.x, v.y += g * x.y, v.z += g * x.z, v.w += g * x.w;
              }
              if (whole) {
                const int64_t at = (int64_t(row) * p.a.heads + head) * D + d;
                if (p.a.out_f32)
                  *reinterpret_cast<float4*>(static_cast<float*>(p.a.out) + at) =
                      make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                else
                  *reinterpret_cast<uint2*>(static_cast<T*>(p.a.out) + at) =
                      make_uint2(HalfOps<T>::pack(v.x * inv, v.y * inv), HalfOps<T>::pack(v.z * inv, v.w * inv));
              } else {
                *reinterpret_cast<float4*>(p.w.o + prow * D + d) = v;
              }
            }
            if (c == 0) {
              if (!whole) p.w.ml[prow] = make_float2(mx, sum);
              else if (p.a.lse) p.a.lse[int64_t(row) * p.a.heads + head] = sum == 0.0f ? -INFINITY : LN2 * (mx + log2f(sum));
            }
          }
        }
        if (t == 0 && !whole && tile0 == 0) {
          // this CTA holds the item's first tile: it records the join
          JoinRec r;
          r.head = w.head, r.block = w.block, r.row0 = q.row0, r.n = q.n;
          const long long last_tile = w.u - w.tile + st.count - 1;
          r.last = int(((last_tile + 1) * grid - 1) / total);
          p.w.rec[cta] = r;
        }
        group_sync();
      }
      if (w.block < st.blocks) break;
    }
    if (w.head < p.a.kv_heads) break;
    ++w.s, w.head = 0, w.block = 0, w.tile = 0;
  }
}

// Joins the partials of the item whose first tile CTA blockIdx.x held, one
// row per block: the maximum of all, then the sums, by groups of D / 4 threads
// that take every GROUPS-th partial each (one long sequence leaves a partial on
// every SM), added up in the groups' order.  What it waits for is a chain of
// loads: the record, the maxima, the sums; a CTA that held no tile left an empty
// partial, so nothing else has to be known.
constexpr int AJ_THREADS = 256, AJ_PARTS = 512;
template <class T, int D, int R>
__global__ void __launch_bounds__(AJ_THREADS) hc_attn_join_kernel(const __grid_constant__ RowsArgs p) {
  constexpr int LANES = D / 4, GROUPS = AJ_THREADS / LANES;
  __shared__ float2 s_ml[AJ_PARTS];
  __shared__ float s_max[AJ_THREADS / 32];
  __shared__ float4 s_o[GROUPS][LANES];
  __shared__ float s_sum[GROUPS];
  const int c0 = int(blockIdx.x), r = int(blockIdx.y), t = int(threadIdx.x);
  const int group = p.a.heads / p.a.kv_heads;
  pdl_launch_next();
  pdl_wait_prior();
  const JoinRec rec = p.w.rec[c0];
  if (rec.block < 0) return;
  const int r0 = rec.block * R;
  if (r >= min(R, rec.n * group - r0)) return;
  const int n = rec.last - c0 + 1;
  // the first CTA's part is its last item, the others' their first
  const auto slot = [&](int i) { return int64_t(i == 0 ? 2 * c0 + 1 : 2 * (c0 + i)) * R + r; };
  float mx = -INFINITY;
  for (int i = t; i < n; i += AJ_THREADS) {
    const float2 v = p.w.ml[slot(i)];
    s_ml[i] = v;
    mx = fmaxf(mx, v.x);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if ((t & 31) == 0) s_max[t >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < AJ_THREADS / 32; ++i) mx = fmaxf(mx, s_max[i]);
  const float ms = mx == -INFINITY ? 0.0f : mx;
  const int g = t / LANES, d = t % LANES * 4;
  float sum = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
  for (int i = g; i < n; i += GROUPS) {
    const float2 s = s_ml[i];
    // nothing seen there: perhaps nothing was written (and no branch, which would
    // put the loads behind one another)
    const bool has = s.x != -INFINITY;
    const float f = ex2(s.x - ms);
    float4 v = *reinterpret_cast<const float4*>(p.w.o + slot(has ? i : 0) * D + d);
    v.x = has ? v.x : 0.0f, v.y = has ? v.y : 0.0f, v.z = has ? v.z : 0.0f, v.w = has ? v.w : 0.0f;
    sum += f * s.y;
    o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
  }
  s_o[g][t % LANES] = o;
  if (t % LANES == 0) s_sum[g] = sum;
  __syncthreads();
  if (g != 0) return;
  sum = 0.0f;
  o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const float4 v = s_o[i][t];
    sum += s_sum[i];
    o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
  }
  const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
  const int64_t row = int64_t(rec.row0 + (r0 + r) / group) * p.a.heads + rec.head * group + (r0 + r) % group;
  if (p.a.out_f32)
    *reinterpret_cast<float4*>(static_cast<float*>(p.a.out) + row * D + d) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  else
    *reinterpret_cast<uint2*>(static_cast<T*>(p.a.out) + row * D + d) =
        make_uint2(HalfOps<T>::pack(o.x * inv, o.y * inv), HalfOps<T>::pack(o.z * inv, o.w * inv));
  if (t == 0 && p.a.lse) p.a.lse[row] = sum == 0.0f ? -INFINITY : LN2 * (mx + log2f(sum));
}

// CTAs per SM times the SMs, of which the workspace allows for 160.
constexpr int kMaxSms = 160;
size_t ws_bytes(int grid, int rows, int dim) {
  const auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
  return al(size_t(2 * grid) * rows * dim * 4) + al(size_t(2 * grid) * rows * 8) + al(size_t(grid) * sizeof(JoinRec));
}

template <int D, int NB, int RG>
size_t rows_ws() {
  return ws_bytes(kMaxSms * RowsCfg<D, NB, RG>::kCtas, RowsCfg<D, NB, RG>::kRows, D);
}

template <class T, int D, int NB, int RG>
cudaError_t launch_rows(RowsArgs& p, const KvSource& kv, void* workspace, cudaStream_t st) {
  using Cfg = RowsCfg<D, NB, RG>;
  auto kernel = hc_attn_rows_kernel<T, D, NB, RG>;
  static std::atomic<uint64_t> attr{0};
  cudaError_t e = once_per_current_device(attr, [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  });
  if (e != cudaSuccess) return e;
  const int grid = std::min(kMaxSms, sm_count()) * Cfg::kCtas;
  const auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.w.o = reinterpret_cast<float*>(ws);
  ws += al(size_t(2 * grid) * Cfg::kRows * D * 4);
  p.w.ml = reinterpret_cast<float2*>(ws);
  ws += al(size_t(2 * grid) * Cfg::kRows * 8);
  p.w.rec = reinterpret_cast<JoinRec*>(ws);
  p.box_rows = p.b.table ? std::min(AR_TILE, 1 << p.b.page_shift) : AR_TILE;
  p.slots = int64_t(kv.slots);
  CUtensorMap km, vm;
  e = encode_kv_map(&km, HalfOps<T>::kMap, kv.k, kv.slots, kv.k_stride, p.a.kv_heads, D, p.box_rows, D / 64);
  if (e == cudaSuccess)
    e = encode_kv_map(&vm, HalfOps<T>::kMap, kv.v, kv.slots, kv.v_stride, p.a.kv_heads, D, p.box_rows, D / 64);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kernel, dim3(grid), dim3(Cfg::kThreads), Cfg::kSmem, st, km, vm, p);
  if (e != cudaSuccess) return e;
  static_assert(3 * kMaxSms <= AJ_PARTS, "one partial per CTA at most");
  return launch_pdl(hc_attn_join_kernel<T, D, Cfg::kRows>, dim3(grid, Cfg::kRows), dim3(AJ_THREADS), 0, st, p);
}

template <class T, int D>
cudaError_t launch_rows_d(RowsArgs& p, const KvSource& kv, void* ws, cudaStream_t st) {
  // Up to 24 rows one block holds all of a KV head's queries and the keys are
  // read once: 20 rows of 16 sequences of 1000 to 4096 keys take 34 us at
  // head_dim 256, 87 at 32 / 8 heads of 128 and 2000 to 8000 keys; in two
  // blocks of 16 they took 45 and 110.  Heads of 64 read so little that more
  // CTAs with 16 rows in one group win there (20 rows: 74 us against 80).
  const int64_t rows = int64_t(p.a.max_q) * (p.a.heads / p.a.kv_heads);
  if (rows <= 8) return launch_rows<T, D, 1, 1>(p, kv, ws, st);
  if constexpr (D == 64) {
    return launch_rows<T, D, 2, 1>(p, kv, ws, st);
  } else {
    if (rows <= 16 || rows > 24) return launch_rows<T, D, 1, 2>(p, kv, ws, st);
    return launch_rows<T, D, 1, 3>(p, kv, ws, st);
  }
}

template <class T>
cudaError_t launch_rows_t(RowsArgs& p, const KvSource& kv, void* ws, cudaStream_t st) {
  switch (p.a.dim) {
    case 64: return launch_rows_d<T, 64>(p, kv, ws, st);
    case 128: return launch_rows_d<T, 128>(p, kv, ws, st);
    default: return launch_rows_d<T, 256>(p, kv, ws, st);
  }
}

}  // namespace

size_t attn_rows_workspace_bytes(int dim) {
  return dim == 64 ? std::max(rows_ws<64, 1, 1>(), rows_ws<64, 2, 1>())
         : dim == 128 ? std::max({rows_ws<128, 1, 1>(), rows_ws<128, 1, 2>(), rows_ws<128, 1, 3>()})
                      : std::max({rows_ws<256, 1, 1>(), rows_ws<256, 1, 2>(), rows_ws<256, 1, 3>()});
}

cudaError_t launch_attn_rows(const AttnArgs& a, const PagedBatch& b, const KvSource& kv, void* workspace,
                             cudaStream_t st) {
  RowsArgs p{};
  p.a = a;
  p.b = b;
  return kv.dtype == HPC_DTYPE_F16 ? launch_rows_t<__half>(p, kv, workspace, st)
                                   : launch_rows_t<__nv_bfloat16>(p, kv, workspace, st);
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (the
// library does not link the driver library itself).
cudaError_t encode_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
                       const cuuint64_t* strides, const cuuint32_t* box) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> cached{nullptr};
  Encode encode = cached.load();
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q{};
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    if (e != cudaSuccess) return e;
    if (q != cudaDriverEntryPointSuccess || !fn) return cudaErrorSymbolNotFound;
    encode = reinterpret_cast<Encode>(fn);
    cached.store(encode);
  }
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, type, cuuint32_t(rank), const_cast<void*>(base), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t encode_kv_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t slots,
                          uint64_t stride, int heads, int dim, int box_rows, int box_pieces) {
  const cuuint64_t dims[3] = {64, slots, cuuint64_t(heads) * (dim / 64)};
  const cuuint64_t strides[2] = {stride * 2, 128};
  const cuuint32_t box[3] = {64, cuuint32_t(box_rows), cuuint32_t(box_pieces)};
  return encode_map(map, type, 3, base, dims, strides, box);
}

}  // namespace hc

int hpc_paged_check(const char* what, size_t heads, size_t kv_heads, size_t head_dim, size_t rows, size_t seqs,
                    size_t pages, size_t page_size, size_t table_width) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return hpc_fail(HPC_ERR_SHAPE, "%s: head_dim %zu (64, 128 or 256)", what, head_dim);
  if (kv_heads < 1 || heads < 1 || heads % kv_heads || heads > 1024)
    return hpc_fail(HPC_ERR_HEADS, "%s: %zu heads over %zu KV heads", what, heads, kv_heads);
  if (rows > size_t(INT32_MAX) / heads || seqs > (1u << 20))
    return hpc_fail(HPC_ERR_SHAPE, "%s: %zu rows of %zu sequences", what, rows, seqs);
  if (page_size) {
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
      return hpc_fail(HPC_ERR_SHAPE, "%s: page_size %zu (a power of two from 16 to 1024)", what, page_size);
    // slots and positions are 32-bit numbers, and a tile's end may lie up to 128
    // behind the last of them
    const size_t most = (size_t(INT32_MAX) - 1024) / page_size;
    if (pages < 1 || pages > most || table_width < 1 || table_width > most)
      return hpc_fail(HPC_ERR_SHAPE, "%s: %zu pages, a table of %zu", what, pages, table_width);
  }
  return HPC_OK;
}

hc::PagedBatch hpc_paged_batch(const int32_t* starts, const int32_t* lens, const int32_t* table, size_t seqs,
                               size_t width, size_t rows, size_t pages, size_t page_size) {
  hc::PagedBatch b{};
  b.starts = starts;
  b.kv_lens = lens;
  b.table = table;
  b.seqs = int(seqs);
  b.width = int(width);
  b.rows = int(rows);
  while (page_size > 1) ++b.page_shift, page_size >>= 1;
  b.pages = int64_t(pages);
  return b;
}

namespace {

size_t workspace_need(size_t head_dim) {
  return std::max(hc::attn_rows_workspace_bytes(int(head_dim)), hc::attn_prompt_workspace_bytes(int(head_dim)));
}

int attention(const char* what, const void* d_q, size_t q_stride, const hc::KvSource& kv, hc::PagedBatch b,
              size_t heads, size_t kv_heads, size_t head_dim, size_t max_query_len, float scale, size_t window,
              void* d_workspace, size_t workspace_bytes, void* d_out, int out_dtype, float* d_lse, void* stream) {
  if (kv.dtype != HPC_DTYPE_F16 && kv.dtype != HPC_DTYPE_BF16)
    return hpc_fail(HPC_ERR_TYPE, "%s: keys and values of type %d", what, kv.dtype);
  if (out_dtype != HPC_DTYPE_F32 && out_dtype != kv.dtype)
    return hpc_fail(HPC_ERR_TYPE, "%s: output type %d", what, out_dtype);
  if (q_stride < heads * head_dim || q_stride % 8 || q_stride > size_t(INT32_MAX) || kv.k_stride < kv_heads * head_dim ||
      kv.k_stride % 8 || kv.v_stride < kv_heads * head_dim || kv.v_stride % 8 || kv.k_stride > size_t(INT32_MAX) ||
      kv.v_stride > size_t(INT32_MAX))
    return hpc_fail(HPC_ERR_SHAPE, "%s: row strides %zu, %zu, %zu (multiples of 8)", what, q_stride,
                    size_t(kv.k_stride), size_t(kv.v_stride));
  if (window > size_t(INT32_MAX) || !(scale == scale))
    return hpc_fail(HPC_ERR_SHAPE, "%s: window %zu, scale %g", what, window, double(scale));
  if (b.rows == 0 || b.seqs == 0) return HPC_OK;
  if (!d_q || !kv.k || !kv.v || !b.starts || !d_out || !d_workspace) return hpc_fail(HPC_ERR_ARG, "null pointer");
  const auto off = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
  if (off(d_q) || off(kv.k) || off(kv.v) || off(d_out) || off(d_workspace))
    return hpc_fail(HPC_ERR_ARG, "%s: tensors must be aligned to 16 bytes", what);
  const size_t need = workspace_need(head_dim);
  if (workspace_bytes < need)
    return hpc_fail(HPC_ERR_SHAPE, "%s: a workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  // Rows are written while keys, values and other rows' queries are still read.
  // Only a row's own query is behind it then, so `out` may be q itself.
  const auto bytes = [&](uint64_t rows, uint64_t stride, size_t row) { return ((rows - 1) * stride + row) * 2; };
  const auto meets = [&](const void* p, uint64_t n) {
    const uint64_t x = reinterpret_cast<uintptr_t>(p), o = reinterpret_cast<uintptr_t>(d_out);
    return x < o + uint64_t(b.rows) * heads * head_dim * (out_dtype == HPC_DTYPE_F32 ? 4 : 2) && o < x + n;
  };
  const bool in_place = d_out == d_q && out_dtype == kv.dtype && q_stride == heads * head_dim;
  if ((!in_place && meets(d_q, bytes(b.rows, q_stride, heads * head_dim))) ||
      meets(kv.k, bytes(kv.slots, kv.k_stride, kv_heads * head_dim)) ||
      meets(kv.v, bytes(kv.slots, kv.v_stride, kv_heads * head_dim)))
    return hpc_fail(HPC_ERR_ARG, "%s: the output lies over keys, values or other queries", what);
  hc::AttnArgs a{};
  a.q = d_q;
  a.q_stride = int64_t(q_stride);
  a.out = d_out;
  a.lse = d_lse;
  a.heads = int(heads), a.kv_heads = int(kv_heads), a.dim = int(head_dim);
  a.window = int(window);
  a.scale_log2 = float(double(scale) * 1.4426950408889634);
  a.out_f32 = out_dtype == HPC_DTYPE_F32;
  a.max_q = int(std::min(max_query_len, size_t(b.rows)));
  a.err = hc::device_status_word();
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Rows (new tokens x heads of a group) of a sequence: few go to the kernel
  // that the keys' bytes bound, more to tensor-core tiles of 128 rows.  16
  // sequences of 2000 to 8000 keys, 32 / 8 heads of 128: 20 rows 88 us there and 101
  // here, 32 rows 115 and 101, 64 rows 226 and 102; 1000 to 4096 keys, 8 / 2 heads
  // of 256: 20 rows 34 and 43, 32 rows 40 and 43, 48 rows 49 and 43.
  const bool few = int64_t(a.max_q) * (a.heads / a.kv_heads) <= (a.dim == 256 ? 32 : 24);
  HPC_CK(few ? hc::launch_attn_rows(a, b, kv, d_workspace, st) : hc::launch_attn_prompt(a, b, kv, d_workspace, st), what);
  return HPC_OK;
}

}  // namespace

extern "C" {

int hpc_attention_workspace_bytes(size_t heads, size_t kv_heads, size_t head_dim, size_t *out_bytes) {
  if (int rc = hpc_paged_check("attention workspace", heads, kv_heads, head_dim, 0, 0, 0, 0, 0)) return rc;
  if (!out_bytes) return hpc_fail(HPC_ERR_ARG, "null pointer");
  *out_bytes = workspace_need(head_dim);
  return HPC_OK;
}

int hpc_paged_attention(const void *d_q, size_t q_stride, const void *d_key_cache, const void *d_value_cache,
                        int cache_dtype, size_t pages, size_t page_size, const int32_t *d_page_table,
                        size_t table_width, const int32_t *d_query_starts, const int32_t *d_kv_lens, size_t seqs,
                        size_t rows, size_t heads, size_t kv_heads, size_t head_dim, size_t max_query_len, float scale,
                        size_t window, void *d_workspace, size_t workspace_bytes, void *d_out, int out_dtype,
                        float *d_lse, void *stream) {
  if (page_size == 0) return hpc_fail(HPC_ERR_SHAPE, "paged attention: page_size 0");
  if (int rc = hpc_paged_check("paged attention", heads, kv_heads, head_dim, rows, seqs, pages, page_size, table_width))
    return rc;
  if (rows && seqs && (!d_page_table || !d_kv_lens)) return hpc_fail(HPC_ERR_ARG, "null pointer");
  const uint64_t stride = uint64_t(kv_heads) * head_dim;
  const hc::KvSource kv{d_key_cache, d_value_cache, uint64_t(pages) * page_size, stride, stride, cache_dtype};
  return attention("paged attention", d_q, q_stride, kv,
                   hpc_paged_batch(d_query_starts, d_kv_lens, d_page_table, seqs, table_width, rows, pages, page_size),
                   heads, kv_heads, head_dim, max_query_len, scale, window, d_workspace, workspace_bytes, d_out,
                   out_dtype, d_lse, stream);
}

int hpc_prompt_attention(const void *d_q, size_t q_stride, const void *d_k, size_t k_stride, const void *d_v,
                         size_t v_stride, int dtype, const int32_t *d_query_starts, size_t seqs, size_t rows,
                         size_t heads, size_t kv_heads, size_t head_dim, size_t max_query_len, float scale,
                         size_t window, void *d_workspace, size_t workspace_bytes, void *d_out, int out_dtype,
                         float *d_lse, void *stream) {
  if (int rc = hpc_paged_check("prompt attention", heads, kv_heads, head_dim, rows, seqs, 0, 0, 0)) return rc;
  const hc::KvSource kv{d_k, d_v, rows, k_stride, v_stride, dtype};
  return attention("prompt attention", d_q, q_stride, kv,
                   hpc_paged_batch(d_query_starts, nullptr, nullptr, seqs, 0, rows, 0, 0), heads, kv_heads, head_dim,
                   max_query_len, scale, window, d_workspace, workspace_bytes, d_out, out_dtype, d_lse, stream);
}

}  // extern "C"
