// hc_logits.cu -- penalties, biases and a grammar mask on logits, and the k
// best tokens, in one pass over the logits.
//
// Per row and token i with logit l, in f64 and rounded once to f32:
//   seen in the history:       x = l > 0 ? l / repetition : l * repetition
//   c > 0 times in its output: x = x - frequency * c - presence
//   biases of i, added up in list order: x = x + sum
//   not allowed:               x = -inf
// A token whose value is -inf or NaN is no candidate; the others rank by
// value, then by the lower id -- the order of every top-k here
// (topK, runtime.ts:514-527) -- so the list feeds hpc_sample_candidates.
// Most tokens are touched by neither history nor bias and keep their f32 logit;
// the f64 arithmetic runs for the few that are.
//
// One read of the logits bounds it.  A CTA takes a chunk of a row (the chunk's
// logits in registers while it counts the history's tokens that fall
// into it, in shared memory; integer counts, so their order does not matter)
// and writes the chunk's k best; a second launch joins the chunks of each row.
// Neither sorts: the k-th largest of 128 group maxima is a floor that at least k
// tokens reach, and hardly any token of the other groups does, so the survivors
// (about 90 of 8192 for k = 64) are ranked by counting.  Keys are (ordered value,
// complement of the id): no two are equal, so the result does not depend on any
// order of execution.  Chunks are 8192 tokens, which spreads the floor's cost, or
// 2048 where those would leave SMs without work.
#include <algorithm>
#include <atomic>

#include "hc_paged.cuh"

namespace hc {
namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_GROUPS = LG_THREADS / 2;
constexpr int LG_MAX_K = 64;
constexpr uint32_t LG_SEEN = 0x80000000u, LG_BIASED = 0x40000000u, LG_COUNT = 0x3fffffffu;
constexpr int LG_BIASES = 1024;  // of a chunk, kept in shared memory
constexpr int LG_CAND = 2048;    // survivors of a chunk

struct LogitsArgs {
  const float* logits;
  int64_t stride;
  int vocab, k, chunks;
  const int32_t* hist;
  const int32_t* hist_starts;
  int64_t hist_len;
  const int32_t* prompt_lens;
  const float* rep;
  const float* freq;
  const float* pres;
  const int32_t* bias_ids;
  const float* bias_vals;
  const int32_t* bias_starts;
  int64_t bias_len;
  const uint32_t* allowed;
  int64_t allowed_stride;
  uint64_t* cand;  // [rows][chunks][k]
  int32_t* ids;
  float* vals;
};

// [a, b) of list `r` inside [0, len].
__device__ __forceinline__ void list_span(const int32_t* starts, int r, int64_t len, int64_t* a, int64_t* b) {
  *a = min(max(int64_t(starts[r]), int64_t(0)), len);
  *b = min(max(int64_t(starts[r + 1]), *a), len);
}

// The k largest of the block's keys (at(i), i < per, for each thread; 0 = none),
// largest first, to put(rank, key); fewer than k keys leave the last ranks 0.
// Distinct keys: no more than k groups reach the floor, so cand needs room for
// their 2 k per keys.
template <class At, class Put>
__device__ __forceinline__ void select_k(int per, int k, uint64_t* cand, At&& at, Put&& put) {
  __shared__ __align__(16) uint64_t s_max[LG_GROUPS];
  __shared__ uint64_t s_floor;
  __shared__ int s_n;
  const int t = int(threadIdx.x);
  uint64_t mx = 0;
  for (int i = 0; i < per; ++i) mx = max(mx, at(i));
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  if ((t & 1) == 0) s_max[t >> 1] = mx;
  if (t == 0) s_floor = 1, s_n = 0;  // fewer than k groups hold a key: all are candidates
  __syncthreads();
  if (t < LG_GROUPS) {
    const uint64_t own = s_max[t];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < LG_GROUPS; j += 2) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&s_max[j]);
      above += int(v.x > own) + int(v.y > own);
    }
    if (above == k - 1 && own != 0) s_floor = own;
  }
  __syncthreads();
  const uint64_t fl = s_floor;
  for (int i = 0; i < per; ++i) {
    const uint64_t x = at(i);
    if (x >= fl) cand[atomicAdd(&s_n, 1)] = x;
  }
  __syncthreads();
  const int n = s_n;
  for (int i = t; i < n; i += LG_THREADS) {
    const uint64_t own = cand[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += int(cand[j] > own);
    if (above < k) put(above, own);
  }
  for (int i = n + t; i < k; i += LG_THREADS) put(i, 0);
}

__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int EPT>
__global__ void __launch_bounds__(LG_THREADS) hc_logits_chunk_kernel(const __grid_constant__ LogitsArgs p) {
  constexpr int C = LG_THREADS * EPT;
  // counts of the chunk's tokens, then (the counts done with) the survivors
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t s_max[LG_GROUPS];
  __shared__ int b_id[LG_BIASES];
  __shared__ float b_val[LG_BIASES];
  __shared__ uint32_t s_floor;
  __shared__ int s_n, s_biases;
  __shared__ uint64_t s_best[LG_THREADS / 32];
  uint32_t* cnt = reinterpret_cast<uint32_t*>(smem);
  uint64_t* cand = reinterpret_cast<uint64_t*>(smem);
  const bool touched = p.hist != nullptr || p.bias_ids != nullptr;
  const int t = int(threadIdx.x), row = int(blockIdx.y), c0 = int(blockIdx.x) * C;
  const int n = min(C, p.vocab - c0);
  pdl_launch_next();
  if (touched)
    for (int i = t * 4; i < C; i += LG_THREADS * 4) *reinterpret_cast<uint4*>(cnt + i) = make_uint4(0, 0, 0, 0);
  if (t == 0) s_floor = 1, s_n = 0, s_biases = 0;
  pdl_wait_prior();
  // element i of this thread: four in a row by vector loads where the row
  // allows them, else one in 256
  const float* src = p.logits + int64_t(row) * p.stride + c0;
  const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  const auto index = [&](int i) { return vec ? (i >> 2) * (LG_THREADS * 4) + t * 4 + (i & 3) : i * LG_THREADS + t; };
  float x[EPT];
#pragma unroll
  for (int i = 0; i < EPT; i += 4) {
    const int at = index(i);
    if (vec && at + 4 <= n) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(src + at));
      x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int a = index(i + e);
        x[i + e] = a < n ? __ldcs(src + a) : -INFINITY;
      }
    }
  }
  __syncthreads();
  if (p.hist) {
    int64_t a, b;
    list_span(p.hist_starts, row, p.hist_len, &a, &b);
    const int64_t out0 = a + (p.prompt_lens ? max(p.prompt_lens[row], 0) : 0);
#pragma unroll 4
    for (int64_t h = a + t; h < b; h += LG_THREADS) {
      const uint32_t o = uint32_t(p.hist[h]) - uint32_t(c0);  // (a negative id wraps past every chunk)
      if (o < uint32_t(n)) {
        atomicOr(&cnt[o], LG_SEEN);
        if (h >= out0) atomicAdd(&cnt[o], 1u);
      }
    }
  }
  int64_t bias_a = 0, bias_b = 0;
  if (p.bias_ids) {
    list_span(p.bias_starts, row, p.bias_len, &bias_a, &bias_b);
    if (t < 32) {
      // one warp picks out the chunk's biases, in list order
      int kept = 0;
      for (int64_t h0 = bias_a; h0 < bias_b; h0 += 32) {
        const int64_t h = h0 + t;
        const uint32_t o = h < bias_b ? uint32_t(p.bias_ids[h]) - uint32_t(c0) : 0xffffffffu;
        const bool in = o < uint32_t(n);
        const unsigned m = __ballot_sync(0xffffffffu, in);
        const int at = kept + __popc(m & ((1u << t) - 1u));
        if (in) {
          atomicOr(&cnt[o], LG_BIASED);
          if (at < LG_BIASES) b_id[at] = int(o), b_val[at] = p.bias_vals[h];
        }
        kept += __popc(m);
      }
      if (t == 0) s_biases = kept;
    }
  }
  if (touched) __syncthreads();
  if (touched) {
    double rep = 1.0, freq = 0.0, pres = 0.0;
    if (p.hist) {
      if (p.rep) rep = p.rep[row];
      if (p.freq) freq = p.freq[row];
      if (p.pres) pres = p.pres[row];
    }
    const int biases = s_biases;
#pragma unroll
    for (int i = 0; i < EPT; i += 4) {
      uint32_t c[4];
      if (vec) {
        *reinterpret_cast<uint4*>(c) = *reinterpret_cast<const uint4*>(cnt + index(i));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = cnt[index(i + e)];
      }
      if (!(c[0] | c[1] | c[2] | c[3])) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!c[e]) continue;
        double v = x[i + e];
        if (c[e] & LG_SEEN) v = v > 0.0 ? v / rep : v * rep;
        if (c[e] & LG_COUNT) v = __dsub_rn(__dsub_rn(v, __dmul_rn(freq, double(c[e] & LG_COUNT))), pres);
        if (c[e] & LG_BIASED) {
          double sum = 0.0;  // the biases of one id add up first, in list order
          const int o = index(i + e);
          if (biases <= LG_BIASES) {
            for (int h = 0; h < biases; ++h)
              if (b_id[h] == o) sum += double(b_val[h]);
          } else {
            for (int64_t h = bias_a; h < bias_b; ++h)
              if (p.bias_ids[h] == c0 + o) sum += double(p.bias_vals[h]);
          }
          v += sum;
        }
        x[i + e] = float(v);
      }
    }
  }
  if (p.allowed) {
    const uint32_t* allow = p.allowed + int64_t(row) * p.allowed_stride;
#pragma unroll
    for (int i = 0; i < EPT; i += 4) {
      if (vec) {  // four tokens of one word (c0 and the index are multiples of 4)
        const int at = c0 + index(i);
        const uint32_t w = index(i) < n ? allow[at >> 5] >> (at & 31) : 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!((w >> e) & 1u)) x[i + e] = -INFINITY;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = index(i + e);
          if (at < n && !((allow[(c0 + at) >> 5] >> ((c0 + at) & 31)) & 1u)) x[i + e] = -INFINITY;
        }
      }
    }
  }
  // ordered values, 0 for what is no candidate (-inf, NaN); -0 ranks as 0
  uint32_t y[EPT], mx = 0;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    y[i] = x[i] > -INFINITY ? ordered(x[i] + 0.0f) : 0u;
    mx = max(mx, y[i]);
  }
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  // the low bits make the maxima distinct; the floor falls by 127 steps at most
  if ((t & 1) == 0) s_max[t >> 1] = mx ? (mx & ~127u) | uint32_t(t >> 1) : 0u;
  __syncthreads();
  if (t < LG_GROUPS) {
    const uint32_t own = s_max[t];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < LG_GROUPS; j += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(&s_max[j]);
      above += int(v.x > own) + int(v.y > own) + int(v.z > own) + int(v.w > own);
    }
    if (above == p.k - 1 && own != 0) s_floor = max(own & ~127u, 1u);
  }
  __syncthreads();
  const uint32_t fl = s_floor;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    if (y[i] >= fl) {
      const int at = atomicAdd(&s_n, 1);
      if (at < LG_CAND) cand[at] = (uint64_t(y[i]) << 32) | (0xffffffffu - uint32_t(c0 + index(i)));
    }
  }
  __syncthreads();
  const int m = s_n;
  uint64_t* out = p.cand + (int64_t(row) * p.chunks + blockIdx.x) * p.k;
  if (m <= LG_CAND) {
    for (int i = t; i < m; i += LG_THREADS) {
      const uint64_t own = cand[i];
      int above = 0;
#pragma unroll 4
      for (int j = 0; j < m; ++j) above += int(cand[j] > own);
      if (above < p.k) out[above] = own;
    }
    for (int i = m + t; i < p.k; i += LG_THREADS) out[i] = 0;
  } else {
    // many equal values at the floor: the largest key below the last, k times
    uint64_t last = ~uint64_t(0);
    for (int r = 0; r < p.k; ++r) {
      uint64_t best = 0;
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const uint64_t key = y[i] ? (uint64_t(y[i]) << 32) | (0xffffffffu - uint32_t(c0 + index(i))) : 0;
        if (key < last) best = max(best, key);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) best = max(best, uint64_t(__shfl_xor_sync(0xffffffffu, (unsigned long long)best, d)));
      __syncthreads();
      if ((t & 31) == 0) s_best[t >> 5] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < LG_THREADS / 32; ++w) best = max(best, s_best[w]);
      if (t == 0) out[r] = best;
      last = best;
    }
  }
}

// One row's chunk lists -> its ids and values.
__global__ void __launch_bounds__(LG_THREADS) hc_logits_join_kernel(const __grid_constant__ LogitsArgs p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int t = int(threadIdx.x), row = int(blockIdx.x);
  pdl_wait_prior();
  const int n = p.chunks * p.k, per = (n + LG_THREADS - 1) / LG_THREADS;
  const uint64_t* in = p.cand + int64_t(row) * n;
  select_k(
      per, p.k, reinterpret_cast<uint64_t*>(smem),
      [&](int i) { return t * per + i < n ? in[t * per + i] : uint64_t(0); },
      [&](int rank, uint64_t key) {
        const uint32_t o = uint32_t(key >> 32);
        const int64_t at = int64_t(row) * p.k + rank;
        p.ids[at] = key ? int32_t(0xffffffffu - uint32_t(key)) : -1;
        p.vals[at] = key ? __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o) : -INFINITY;
      });
}

constexpr int LG_LARGE = LG_THREADS * 32, LG_SMALL = LG_THREADS * 8;

// Tokens per chunk: large chunks where they give every SM two CTAs.
int chunk_of(size_t rows, size_t vocab) {
  return rows * ((vocab + LG_LARGE - 1) / LG_LARGE) >= 296 ? LG_LARGE : LG_SMALL;
}

template <int EPT>
cudaError_t launch_chunks(const LogitsArgs& p, unsigned rows, cudaStream_t st) {
  const bool touched = p.hist || p.bias_ids;
  const size_t smem = std::max(size_t(LG_CAND) * 8, touched ? size_t(LG_THREADS) * EPT * 4 : 0);
  return launch_pdl(hc_logits_chunk_kernel<EPT>, dim3(unsigned(p.chunks), rows), dim3(LG_THREADS), smem, st, p);
}

}  // namespace
}  // namespace hc

extern "C" {

int hpc_logits_topk_workspace_bytes(size_t rows, size_t vocab, size_t k, size_t *out_bytes) {
  if (rows > 65535 || vocab < 1 || vocab > HPC_LOGITS_MAX_VOCAB || k < 1 || k > size_t(hc::LG_MAX_K) || k > vocab)
    return hpc_fail(HPC_ERR_SHAPE, "logits: %zu rows of %zu, the best %zu (1..%d)", rows, vocab, k, hc::LG_MAX_K);
  if (!out_bytes) return hpc_fail(HPC_ERR_ARG, "null pointer");
  const size_t chunk = size_t(hc::chunk_of(rows, vocab));
  *out_bytes = rows * ((vocab + chunk - 1) / chunk) * k * 8;
  return HPC_OK;
}

int hpc_logits_topk(const float *d_logits, size_t row_stride, size_t rows, size_t vocab, size_t k,
                    const int32_t *d_history, size_t history_len, const int32_t *d_history_starts,
                    const int32_t *d_prompt_lens, const float *d_repetition, const float *d_frequency,
                    const float *d_presence, const int32_t *d_bias_ids, const float *d_bias_values, size_t bias_len,
                    const int32_t *d_bias_starts, const uint32_t *d_allowed, size_t allowed_stride, void *d_workspace,
                    size_t workspace_bytes, int32_t *d_ids, float *d_vals, void *stream) {
  size_t need = 0;
  if (int rc = hpc_logits_topk_workspace_bytes(rows, vocab, k, &need)) return rc;
  if (row_stride < vocab || (d_allowed && allowed_stride < (vocab + 31) / 32))
    return hpc_fail(HPC_ERR_SHAPE, "logits: row stride %zu, mask stride %zu of %zu tokens", row_stride, allowed_stride,
                    vocab);
  if (workspace_bytes < need)
    return hpc_fail(HPC_ERR_SHAPE, "logits: a workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (rows == 0) return HPC_OK;
  if (!d_logits || !d_workspace || !d_ids || !d_vals || (d_history && !d_history_starts) ||
      (d_bias_ids && (!d_bias_values || !d_bias_starts)))
    return hpc_fail(HPC_ERR_ARG, "null pointer");
  if (reinterpret_cast<uintptr_t>(d_workspace) % 8) return hpc_fail(HPC_ERR_ARG, "logits: workspace alignment");
  const size_t chunk = size_t(hc::chunk_of(rows, vocab));
  hc::LogitsArgs p{};
  p.logits = d_logits;
  p.stride = int64_t(row_stride);
  p.vocab = int(vocab), p.k = int(k), p.chunks = int((vocab + chunk - 1) / chunk);
  p.hist = d_history, p.hist_starts = d_history_starts, p.hist_len = int64_t(history_len);
  p.prompt_lens = d_prompt_lens;
  p.rep = d_repetition, p.freq = d_frequency, p.pres = d_presence;
  p.bias_ids = d_bias_ids, p.bias_vals = d_bias_values, p.bias_starts = d_bias_starts, p.bias_len = int64_t(bias_len);
  p.allowed = d_allowed, p.allowed_stride = int64_t(allowed_stride);
  p.cand = static_cast<uint64_t *>(d_workspace);
  p.ids = d_ids, p.vals = d_vals;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int per = (p.chunks * p.k + hc::LG_THREADS - 1) / hc::LG_THREADS;
  const size_t join = size_t(2) * p.k * per * 8;
  static std::atomic<uint64_t> attr{0};
  HPC_CK(hc::once_per_current_device(attr, [&] {
           // 512 lists of 64 at most: 2 * 64 * 128 keys
           return cudaFuncSetAttribute(hc::hc_logits_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 << 10);
         }),
         "logits attributes");
  HPC_CK(chunk == size_t(hc::LG_LARGE) ? hc::launch_chunks<32>(p, unsigned(rows), st)
                                       : hc::launch_chunks<8>(p, unsigned(rows), st),
         "logits launch");
  HPC_CK(hc::launch_pdl(hc::hc_logits_join_kernel, dim3(unsigned(rows)), dim3(hc::LG_THREADS), join, st, p),
         "logits join launch");
  return HPC_OK;
}

}  // extern "C"
