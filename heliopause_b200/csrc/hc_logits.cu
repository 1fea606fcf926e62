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
// One read of the logits bounds it.  A CTA streams a chunk of a row, 4096 tokens
// at a time with the next ones already on their way, and keeps the keys that
// can still be among its k best; a second launch joins the chunks of each row.
//   - The first 4096 give a floor without a sort: the k-th largest of 128 group
//     maxima is reached by at least k tokens and by few others.  It is raised
//     from the kept keys after two more steps, so that most later steps end
//     with one comparison per warp.
//   - Tokens of the history or with a bias (hundreds of a chunk's 32768) are left
//     out of the stream and taken from a list of their own, one thread each: in
//     the stream every warp that met one stood through its f64 division (the
//     64 x 262144 batch then took 77 us).
//   - The chunk's mask waits in shared memory: looked up in place, for the tokens
//     above the floor only, it held every warp up for two or three reads a step.
//   - The survivors get such a floor once more and are ranked by counting.
// Keys are (ordered value, complement of the id): no two are equal, so the
// result does not depend on any order of execution.  The chunk's part of the
// history is counted in shared memory, 16 bits a token (integer counts, so their
// order does not matter).  Chunks are as long as leaves every SM two CTAs, up to
// 32768 tokens: what a CTA does before and behind the stream, chains of
// dependent steps of some microseconds, is then paid once.
// Measured: 64 x 262144 with histories, biases and a mask 45.5 us (69 MB, 1.5
// TB/s; a chunk takes 19 us of such steps and 512 chunks are two rounds of the
// machine), one row of 262144 9.9 to 12 us, two such chains one behind the other.
#include <algorithm>
#include <atomic>

#include "hc_paged.cuh"

namespace hc {
namespace {

constexpr int LG_THREADS = 512;                // of a chunk's CTA
constexpr int LG_EPT = 8;                      // tokens per thread and step
constexpr int LG_STEP = LG_THREADS * LG_EPT;
constexpr int LG_MAX_STEPS = 8;
constexpr int LG_GROUPS = 128;
constexpr int LG_MAX_K = 64;
constexpr int LG_BIASES = 512;                 // of a chunk, kept in shared memory
constexpr int LG_RANKED = 256;                   // kept keys that are ranked as they are (a floor first costs 2 us)
constexpr int LG_CAND = 2560;                  // kept keys
constexpr int LG_FLAGS = 4096;                 // listed tokens with a history or a bias
// a token's 16 bits: seen in the history, has a bias, times in the output
constexpr uint32_t LG_SEEN = 0x8000u, LG_BIASED = 0x4000u, LG_COUNT = 0x3fffu;
constexpr int LG_JOIN_THREADS = 1024;
constexpr int LG_JOIN_GROUP = LG_JOIN_THREADS / LG_GROUPS;  // threads of a group
constexpr int LG_LISTS = 128;                  // most chunks of a row

struct LogitsArgs {
  const float* logits;
  int64_t stride;
  int vocab, k, chunks, steps;  // steps of LG_STEP tokens per chunk
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

__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The key of rank k - 1 among LG_GROUPS distinct group maxima in `mx` (0 = a
// group without keys) to *floor, which holds 1 before: where fewer than k groups
// have one, every key is above it.  Threads 0 .. LG_GROUPS - 1.
__device__ __forceinline__ void group_floor(const uint64_t* mx, int k, uint64_t* floor) {
  const uint64_t own = mx[threadIdx.x];
  int above = 0;
#pragma unroll 16
  for (int j = 0; j < LG_GROUPS; j += 2) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(mx + j);
    above += int(v.x > own) + int(v.y > own);
  }
  if (above == k - 1 && own != 0) *floor = own;
}

__device__ __forceinline__ float of_ordered(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

// The value of order o as a bound to be above; both zeros are above the value
// below zero.
__device__ __forceinline__ float just_below(uint32_t o) { return o == 0x7fffffffu ? -1.401298464e-45f : of_ordered(o); }

// Rank of cand[i] among n distinct keys: the larger ones.
__device__ __forceinline__ int rank_of(const uint64_t* cand, int n, uint64_t own) {
  int above = 0;
#pragma unroll 8
  for (int j = 0; j < n; ++j) above += int(cand[j] > own);
  return above;
}

// TOUCHED: with a history or biases; MASK: with a grammar; VEC: 16-byte loads.
template <bool TOUCHED, bool MASK, bool VEC>
__global__ void __launch_bounds__(LG_THREADS, 2) hc_logits_chunk_kernel(const __grid_constant__ LogitsArgs p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) uint64_t s_max[LG_GROUPS];
  __shared__ __align__(16) uint32_t s_top[LG_GROUPS];
  __shared__ uint16_t s_flag[TOUCHED ? LG_FLAGS : 1];
  __shared__ int b_id[TOUCHED ? LG_BIASES : 1];
  __shared__ float b_val[TOUCHED ? LG_BIASES : 1];
  __shared__ uint32_t s_allow[MASK ? LG_STEP * LG_MAX_STEPS / 32 : 1];
  __shared__ uint64_t s_floor, s_best[LG_THREADS / 32];
  __shared__ float s_over;
  __shared__ int s_n, s_flags, s_biases;
  uint64_t* cand = reinterpret_cast<uint64_t*>(smem);                        // LG_CAND keys
  uint32_t* cnt = reinterpret_cast<uint32_t*>(smem + size_t(LG_CAND) * 8);   // 16 bits per token of the chunk
  const int t = int(threadIdx.x), row = int(blockIdx.y), C = p.steps * LG_STEP, c0 = int(blockIdx.x) * C;
  const int n = min(C, p.vocab - c0);
  pdl_launch_next();
  if constexpr (TOUCHED)
    for (int i = t * 4; i < C / 2; i += LG_THREADS * 4) *reinterpret_cast<uint4*>(cnt + i) = make_uint4(0, 0, 0, 0);
  if (t == 0) s_n = 0, s_flags = 0, s_biases = 0, s_over = -INFINITY;
  pdl_wait_prior();
  // element i of this thread in a step: four in a row, or one in LG_THREADS
  const float* src = p.logits + int64_t(row) * p.stride + c0;
  const auto index = [&](int i) { return VEC ? (i >> 2) * (LG_THREADS * 4) + t * 4 + (i & 3) : i * LG_THREADS + t; };
  const auto load = [&](int step, float(&x)[LG_EPT]) {
    const float* s = src + step * LG_STEP;
    const int m = n - step * LG_STEP;
#pragma unroll
    for (int i = 0; i < LG_EPT; i += 4) {
      const int at = index(i);
      if (VEC && at + 4 <= m) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(s + at));
        x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int a = index(i + e);
          x[i + e] = a < m ? __ldcs(s + a) : -INFINITY;
        }
      }
    }
  };
  float x[LG_EPT];
  load(0, x);
  if constexpr (MASK) {
    const uint32_t* allow = p.allowed + int64_t(row) * p.allowed_stride + c0 / 32;
    for (int i = t; i < (n + 31) / 32; i += LG_THREADS) s_allow[i] = allow[i];
  }
  double rep = 1.0, freq = 0.0, pres = 0.0;
  int64_t hist_a = 0, hist_b = 0, out0 = 0, bias_a = 0, bias_b = 0;
  if (TOUCHED && p.hist) {
    list_span(p.hist_starts, row, p.hist_len, &hist_a, &hist_b);
    out0 = hist_a + (p.prompt_lens ? max(p.prompt_lens[row], 0) : 0);
    if (p.rep) rep = p.rep[row];
    if (p.freq) freq = p.freq[row];
    if (p.pres) pres = p.pres[row];
  }
  if (TOUCHED && p.bias_ids) list_span(p.bias_starts, row, p.bias_len, &bias_a, &bias_b);
  // Longer histories could overflow a count: there the counts are taken when a
  // seen token is valued.
  const bool counted = hist_b - hist_a <= int64_t(LG_COUNT);
  __syncthreads();
  if constexpr (TOUCHED) {
    // sets a token's bit; who finds none set lists the token
    const auto flag = [&](uint32_t o, uint32_t bit) {
      const uint32_t old = atomicOr(&cnt[o >> 1], bit << (16 * (o & 1))) >> (16 * (o & 1));
      if (!(old & (LG_SEEN | LG_BIASED))) {
        const int at = atomicAdd(&s_flags, 1);
        if (at < LG_FLAGS) s_flag[at] = uint16_t(o);
      }
    };
    // one warp picks out the chunk's biases, in list order; the others count the history
    const bool biased = bias_b > bias_a;
    const int lane = t & 31, counters = biased ? LG_THREADS - 32 : LG_THREADS;
#pragma unroll 4
    for (int64_t h = t < counters ? hist_a + t : hist_b; h < hist_b; h += counters) {
      const uint32_t o = uint32_t(p.hist[h]) - uint32_t(c0);  // (a negative id wraps past every chunk)
      if (o < uint32_t(n)) {
        flag(o, LG_SEEN);
        if (counted && h >= out0) atomicAdd(&cnt[o >> 1], 1u << (16 * (o & 1)));
      }
    }
    if (t >= counters) {
      int kept = 0;
      for (int64_t h0 = bias_a; h0 < bias_b; h0 += 32) {
        const int64_t h = h0 + lane;
        const uint32_t o = h < bias_b ? uint32_t(p.bias_ids[h]) - uint32_t(c0) : 0xffffffffu;
        const bool in = o < uint32_t(n);
        const unsigned m = __ballot_sync(0xffffffffu, in);
        const int at = kept + __popc(m & ((1u << lane) - 1u));
        if (in) {
          flag(o, LG_BIASED);
          if (at < LG_BIASES) b_id[at] = int(o), b_val[at] = p.bias_vals[h];
        }
        kept += __popc(m);
      }
      if (lane == 0) s_biases = kept;
    }
    __syncthreads();
  }
  const auto allowed = [&](int o) { return !MASK || ((s_allow[o >> 5] >> (o & 31)) & 1u); };
  const auto bits = [&](int o) { return TOUCHED ? (cnt[o >> 1] >> (16 * (o & 1))) & 0xffffu : 0u; };
  // token o's value from its logit and bits (the mask apart)
  const auto value = [&](float l, int o, uint32_t c) {
    double v = l;
    if (c & LG_SEEN) {
      v = v > 0.0 ? v / rep : v * rep;
      int64_t times = c & LG_COUNT;
      if (!counted)
        for (int64_t h = max(out0, hist_a); h < hist_b; ++h) times += p.hist[h] == c0 + o;
      if (times) v = __dsub_rn(__dsub_rn(v, __dmul_rn(freq, double(times))), pres);
    }
    if (c & LG_BIASED) {
      double sum = 0.0;  // the biases of one id add up first, in list order
      const int biases = s_biases;
      if (biases <= LG_BIASES) {
        for (int h = 0; h < biases; ++h)
          if (b_id[h] == o) sum += double(b_val[h]);
      } else {
        for (int64_t h = bias_a; h < bias_b; ++h)
          if (p.bias_ids[h] == c0 + o) sum += double(p.bias_vals[h]);
      }
      v += sum;
    }
    return float(v);
  };
  const auto key = [&](float v, int o) {  // -0 ranks as 0
    return (uint64_t(ordered(v + 0.0f)) << 32) | (0xffffffffu - uint32_t(c0 + o));
  };
  const auto keep = [&](float v, int o) {
    const int at = atomicAdd(&s_n, 1);
    if (at < LG_CAND) cand[at] = key(v, o);
  };

  // ---- the first step, and its floor (NaN fails every comparison)
  if (TOUCHED || MASK) {
#pragma unroll
    for (int i = 0; i < LG_EPT; i += 4) {
      if (VEC) {  // four tokens of one mask word and two count words
        const int at = index(i);
        uint32_t w = 0xfu;
        if (MASK) w = at < n ? s_allow[at >> 5] >> (at & 31) : 0u;
        uint2 c = make_uint2(0, 0);
        if (TOUCHED) c = *reinterpret_cast<const uint2*>(cnt + (at >> 1));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t ce = ((e < 2 ? c.x : c.y) >> (16 * (e & 1))) & (LG_SEEN | LG_BIASED);
          if (!((w >> e) & 1u) || ce) x[i + e] = -INFINITY;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int o = index(i + e);
          if (o < n && (!allowed(o) || bits(o))) x[i + e] = -INFINITY;
        }
      }
    }
  }
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < LG_EPT; ++i) mx = fmaxf(mx, x[i]);
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  // the low bits make the maxima distinct, so the floor falls by 127 steps of
  // the last place at most
  if ((t & 3) == 0) s_top[t >> 2] = mx > -INFINITY ? (ordered(mx) & ~127u) | uint32_t(t >> 2) : 0u;
  __syncthreads();
  if (t < LG_GROUPS) {
    const uint32_t own = s_top[t];
    int above = 0;
#pragma unroll 16
    for (int j = 0; j < LG_GROUPS; j += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(s_top + j);
      above += int(v.x > own) + int(v.y > own) + int(v.z > own) + int(v.w > own);
    }
    if (above == p.k - 1 && own != 0) {
      s_over = just_below((own & ~127u) - 1u);
    }
  }
  __syncthreads();
  float over = fmaxf(-INFINITY, s_over);  // (what follows -inf in that order is a NaN: no floor)
#pragma unroll
  for (int i = 0; i < LG_EPT; ++i)
    if (x[i] > over) keep(x[i], index(i));

  // ---- the listed tokens, one thread each
  if constexpr (TOUCHED) {
    const bool listed = s_flags <= LG_FLAGS;
    const int todo = listed ? s_flags : n;
    for (int i = t; i < todo; i += LG_THREADS) {
      const int o = listed ? int(s_flag[i]) : i;
      const uint32_t c = bits(o);
      if (!c || !allowed(o)) continue;
      const float v = value(src[o], o, c);
      if (v > over) keep(v, o);
    }
  }

  // ---- the stream, two steps on their way
  const int steps = min(p.steps, (n + LG_STEP - 1) / LG_STEP);
  const auto pass = [&](int step, const float(&y)[LG_EPT]) {
    float top = y[0];
#pragma unroll
    for (int i = 1; i < LG_EPT; ++i) top = fmaxf(top, y[i]);
    if (top > over) {
#pragma unroll
      for (int i = 0; i < LG_EPT; ++i) {
        const int o = step * LG_STEP + index(i);
        if (y[i] > over && allowed(o) && !(bits(o) & (LG_SEEN | LG_BIASED))) keep(y[i], o);
      }
    }
  };
  float y[LG_EPT];
  if (steps > 1) load(1, x);
  if (steps > 2) load(2, y);
  for (int step = 1; step < steps; step += 2) {
    pass(step, x);
    if (step + 2 < steps) load(step + 2, x);
    if (step + 1 < steps) pass(step + 1, y);
    if (step + 3 < steps) load(step + 3, y);
    if (step == 1 && steps > 5) {
      __syncthreads();
      const int have = min(s_n, LG_CAND);
      // all warps have read s_n before one of them keeps a key again: the
      // barriers below stand behind what was read
      __syncthreads();
      if (have > p.k) {
        if (t < LG_GROUPS) {
          uint64_t best = 0;
          for (int i = t; i < have; i += LG_GROUPS) best = max(best, cand[i]);
          s_max[t] = best;
        }
        if (t == 0) s_floor = 1;
        __syncthreads();
        if (t < LG_GROUPS) group_floor(s_max, p.k, &s_floor);
        __syncthreads();
        // a later token has to be above its value: an equal one has a higher id
        // than k that are kept -- unless listed tokens are among those
        const uint32_t f = uint32_t(s_floor >> 32);
        if (f) over = fmaxf(over, just_below(TOUCHED ? f - 1u : f));
      }
    }
  }
  __syncthreads();
  uint64_t* out = p.cand + (int64_t(row) * p.chunks + blockIdx.x) * p.k;
  const int have = s_n;
  if (have <= LG_CAND) {
    if (have > LG_RANKED) {  // the same floor once more before the ranking, pair by pair
      if (t < LG_GROUPS) {
        uint64_t best = 0;
        for (int i = t; i < have; i += LG_GROUPS) best = max(best, cand[i]);
        s_max[t] = best;
      }
      uint64_t own[LG_CAND / LG_THREADS];
#pragma unroll
      for (int i = 0; i < LG_CAND / LG_THREADS; ++i) own[i] = i * LG_THREADS + t < have ? cand[i * LG_THREADS + t] : 0;
      if (t == 0) s_floor = 1;
      __syncthreads();
      if (t == 0) s_n = 0;
      if (t < LG_GROUPS) group_floor(s_max, p.k, &s_floor);
      __syncthreads();
      const uint64_t floor = s_floor;
#pragma unroll
      for (int i = 0; i < LG_CAND / LG_THREADS; ++i)
        if (own[i] >= floor) cand[atomicAdd(&s_n, 1)] = own[i];
      __syncthreads();
    }
    const int m = s_n;
    for (int i = t; i < m; i += LG_THREADS) {
      const uint64_t own = cand[i];
      const int r = rank_of(cand, m, own);
      if (r < p.k) out[r] = own;
    }
    for (int i = m + t; i < p.k; i += LG_THREADS) out[i] = 0;
    return;
  }
  // more keys than there is room for (many equal values, or a row in ascending
  // order): the largest key below the last, k times over the whole chunk
  uint64_t last = ~uint64_t(0);
  for (int r = 0; r < p.k; ++r) {
    uint64_t best = 0;
    for (int o = t; o < n; o += LG_THREADS) {
      if (!allowed(o)) continue;
      const uint32_t c = bits(o);
      const float v = c ? value(src[o], o, c) : src[o];
      const uint64_t now = v > -INFINITY ? key(v, o) : 0;
      if (now < last) best = max(best, now);
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

// One row's chunk lists -> its ids and values, in the same way: the keys wait in
// shared memory.  A chunk's list falls with the rank, so a group takes
// other ranks of every list: of 64 lists of 64 some 90 keys are then above the
// floor (one row of 262144 takes 9.9 us so, 16.8 with runs of the lists as
// groups and a quarter of the threads).
__global__ void __launch_bounds__(LG_JOIN_THREADS) hc_logits_join_kernel(const __grid_constant__ LogitsArgs p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) uint64_t s_max[LG_GROUPS];
  __shared__ uint64_t s_floor;
  __shared__ int s_n;
  const int t = int(threadIdx.x), row = int(blockIdx.x);
  const int n = p.chunks * p.k, per = (n + LG_JOIN_THREADS - 1) / LG_JOIN_THREADS;
  uint64_t* keys = reinterpret_cast<uint64_t*>(smem);
  uint64_t* cand = keys + n;  // at most the keys of k groups reach the floor
  const uint64_t* in = p.cand + int64_t(row) * n;
  if (t == 0) s_floor = 1, s_n = 0;
  pdl_launch_next();
  pdl_wait_prior();
#pragma unroll 8
  for (int i = t; i < n; i += LG_JOIN_THREADS) keys[i] = in[i];
  __syncthreads();
  uint64_t mx = 0;
  for (int i = 0; i < per; ++i) {
    const int at = i * LG_JOIN_THREADS + ((33 * t + 37 * i) & (LG_JOIN_THREADS - 1));
    if (at < n) mx = max(mx, keys[at]);
  }
#pragma unroll
  for (int d = 1; d < LG_JOIN_GROUP; d <<= 1)
    mx = max(mx, uint64_t(__shfl_xor_sync(0xffffffffu, (unsigned long long)mx, d)));
  if (t % LG_JOIN_GROUP == 0) s_max[t / LG_JOIN_GROUP] = mx;
  __syncthreads();
  if (t < LG_GROUPS) group_floor(s_max, p.k, &s_floor);
  __syncthreads();
  const uint64_t floor = s_floor;
  for (int i = t; i < n; i += LG_JOIN_THREADS)
    if (keys[i] >= floor) cand[atomicAdd(&s_n, 1)] = keys[i];
  __syncthreads();
  const int m = s_n;
  const auto put = [&](int rank, uint64_t key) {
    const uint32_t o = uint32_t(key >> 32);
    const int64_t at = int64_t(row) * p.k + rank;
    p.ids[at] = key ? int32_t(0xffffffffu - uint32_t(key)) : -1;
    p.vals[at] = key ? of_ordered(o) : -INFINITY;
  };
  for (int i = t; i < m; i += LG_JOIN_THREADS) {
    const uint64_t own = cand[i];
    const int r = rank_of(cand, m, own);
    if (r < p.k) put(r, own);
  }
  for (int i = m + t; i < p.k; i += LG_JOIN_THREADS) put(i, 0);
}

static_assert(HPC_LOGITS_MAX_VOCAB <= LG_STEP * LG_MAX_STEPS * LG_LISTS, "lists of the largest vocabulary");

// Steps per chunk: the most that leave every SM two CTAs, and at most LG_LISTS
// chunks a row.
int chunk_steps(size_t rows, size_t vocab) {
  int steps = LG_MAX_STEPS;
  const auto chunks = [&](int n) { return (vocab + size_t(n) * LG_STEP - 1) / (size_t(n) * LG_STEP); };
  while (steps > 1 && rows * chunks(steps) < 296 && chunks(steps / 2) <= size_t(LG_LISTS)) steps /= 2;
  return steps;
}
using ChunkKernel = void (*)(LogitsArgs);
ChunkKernel chunk_kernel(bool touched, bool mask, bool vec) {
  if (vec)
    return touched ? mask ? hc_logits_chunk_kernel<true, true, true> : hc_logits_chunk_kernel<true, false, true>
           : mask  ? hc_logits_chunk_kernel<false, true, true>
                   : hc_logits_chunk_kernel<false, false, true>;
  return touched ? mask ? hc_logits_chunk_kernel<true, true, false> : hc_logits_chunk_kernel<true, false, false>
         : mask  ? hc_logits_chunk_kernel<false, true, false>
                 : hc_logits_chunk_kernel<false, false, false>;
}

size_t chunk_count(size_t rows, size_t vocab) {
  const size_t c = size_t(chunk_steps(rows, vocab)) * LG_STEP;
  return (vocab + c - 1) / c;
}

}  // namespace
}  // namespace hc

extern "C" {

int hpc_logits_topk_workspace_bytes(size_t rows, size_t vocab, size_t k, size_t *out_bytes) {
  if (rows > 65535 || vocab < 1 || vocab > HPC_LOGITS_MAX_VOCAB || k < 1 || k > size_t(hc::LG_MAX_K) || k > vocab)
    return hpc_fail(HPC_ERR_SHAPE, "logits: %zu rows of %zu, the best %zu (1..%d)", rows, vocab, k, hc::LG_MAX_K);
  if (!out_bytes) return hpc_fail(HPC_ERR_ARG, "null pointer");
  *out_bytes = rows * hc::chunk_count(rows, vocab) * k * 8;
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
  hc::LogitsArgs p{};
  p.logits = d_logits;
  p.stride = int64_t(row_stride);
  p.vocab = int(vocab), p.k = int(k), p.chunks = int(hc::chunk_count(rows, vocab));
  p.steps = hc::chunk_steps(rows, vocab);
  p.hist = d_history, p.hist_starts = d_history_starts, p.hist_len = int64_t(history_len);
  p.prompt_lens = d_prompt_lens;
  p.rep = d_repetition, p.freq = d_frequency, p.pres = d_presence;
  p.bias_ids = d_bias_ids, p.bias_vals = d_bias_values, p.bias_starts = d_bias_starts, p.bias_len = int64_t(bias_len);
  p.allowed = d_allowed, p.allowed_stride = int64_t(allowed_stride);
  p.cand = static_cast<uint64_t *>(d_workspace);
  p.ids = d_ids, p.vals = d_vals;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int per = (p.chunks * p.k + hc::LG_JOIN_THREADS - 1) / hc::LG_JOIN_THREADS;
  const size_t join = (size_t(p.chunks) * p.k + size_t(hc::LG_JOIN_GROUP) * p.k * per) * 8;
  const size_t cand = size_t(hc::LG_CAND) * 8;
  const size_t smem = cand + (d_history || d_bias_ids ? size_t(p.steps) * hc::LG_STEP * 2 : 0);
  static std::atomic<uint64_t> attr{0};
  HPC_CK(hc::once_per_current_device(attr, [&] {
           cudaError_t e = cudaSuccess;
           const int most = int(cand + hc::LG_MAX_STEPS * hc::LG_STEP * 2);
           for (int i = 0; i < 8 && e == cudaSuccess; ++i)
             e = cudaFuncSetAttribute(hc::chunk_kernel(i & 1, i & 2, i & 4), cudaFuncAttributeMaxDynamicSharedMemorySize, most);
           // 128 lists of 64 and the survivors, half of them at most
           if (e == cudaSuccess)
             e = cudaFuncSetAttribute(hc::hc_logits_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 << 10);
           return e;
         }),
         "logits attributes");
  const bool vec = reinterpret_cast<uintptr_t>(d_logits) % 16 == 0 && row_stride % 4 == 0;
  HPC_CK(hc::launch_pdl(hc::chunk_kernel(d_history || d_bias_ids, d_allowed, vec), dim3(unsigned(p.chunks), unsigned(rows)),
                        dim3(hc::LG_THREADS), smem, st, p),
         "logits launch");
  HPC_CK(hc::launch_pdl(hc::hc_logits_join_kernel, dim3(unsigned(rows)), dim3(hc::LG_JOIN_THREADS), join, st, p),
         "logits join launch");
  return HPC_OK;
}

}  // extern "C"
