// hc_paged_append.cu -- new tokens into the paged KV cache.
//
// For every new token at position p (its sequence's kv_len - new + i) and
// every head:   k' = rope_p(rms(k) * w_k),  v' = rms(v) or v,
//               q' = rope_p(rms(q) * w_q),
// rms(x) = x / sqrt(mean(x^2) + eps), each part optional; k' and v' go to
// slot (table[s][p / page_size], p % page_size), q' to its packed row.  The
// order is the decode step's (wasm/layers.ts:161-247: head norm, NeoX RoPE,
// KV write; the values' norm has no weight).
// Rotation: elements i and i + R of the first 2 R, by the angle
// p * inv_freq[i].  The angle is reduced in f64 -- in turns, where dropping
// the whole ones is exact, so a position of 2^31 keeps its 2^-22 -- and the
// sine and cosine are f32's; sums and products are f32, each result is
// rounded once to its 16-bit type.
//
// The work is bytes: each input row is read once, each output row written
// once.  One block takes one token: its angles are computed once (R of them,
// by R threads) and shared by the heads, one warp per head at a time with 16
// (8, 4) bytes of the result per lane; a lane's partner element sits R / E lanes
// away.  The first head's row is loaded before the token's sequence is
// known (rows do not depend on it), and the sequence is found by a 32-way
// search over the starts, one load per level.
// Measured: 5044 tokens of 32 / 8 heads of 128 from f32 (186 MB) 41 us, 4.5
// TB/s, bounded by issue (64%) more than by memory; one token of 64 chats 4.5 us.
#include "hc_paged.cuh"

namespace hc {
namespace {

constexpr int AP_MAX_WARPS = 8;

struct AppendArgs {
  const void* src[3];     // q (or nullptr), k, v
  int64_t stride[3];
  int heads[3];           // q, k, v heads; 0 q heads: no queries
  const float* norm_w[3];
  int norm[3];            // 0: none, 1: rms, 2: rms * weight
  const double* inv_freq;
  int rot_half;
  float eps;
  void* q_out;
  void* cache[2];
  PagedBatch b;
  int* err;
};

template <class T, int E>
__device__ __forceinline__ void load_row(const T* p, float (&x)[E]) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (E >= 4) {
#pragma unroll
      for (int i = 0; i < E; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p + i);
        x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
      }
    } else {
      const float2 v = *reinterpret_cast<const float2*>(p);
      x[0] = v.x, x[1] = v.y;
    }
  } else {
    uint32_t w[E / 2];
    if constexpr (E == 8) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (E == 4) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 v = HalfOps<T>::unpack(w[i]);
      x[2 * i] = v.x, x[2 * i + 1] = v.y;
    }
  }
}

template <class T, int E>
__device__ __forceinline__ void store_row(T* p, const float (&x)[E]) {
  uint32_t w[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) w[i] = HalfOps<T>::pack(x[2 * i], x[2 * i + 1]);
  if constexpr (E == 8) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(w);
  else if constexpr (E == 4) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(w);
  else *reinterpret_cast<uint32_t*>(p) = w[0];
}

// The sequence whose rows hold packed row t: the last s with starts[s] <= t.
// One warp, 32 probes a level.
__device__ __forceinline__ int find_seq(const int32_t* starts, int seqs, int t, int lane) {
  int lo = 0, n = seqs;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int i = lo + lane * step;
    const bool le = lane * step < n && starts[i] <= t;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    const int last = m ? 31 - __clz(m) : 0;
    n = min(step, n - last * step);
    lo += last * step;
  }
  return lo;
}

template <class TIn, class T, int E, int PER>
__global__ void __launch_bounds__(32 * AP_MAX_WARPS) hc_paged_append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int D = 32 * E;
  __shared__ float2 turn[D / 2];  // (cos, sin)
  __shared__ int s_pos, s_page;
  const int t = int(blockIdx.x), lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
  const int warps = int(blockDim.x) >> 5;
  const int hq = a.heads[0], hk = a.heads[1], total = hq + 2 * hk;
  const auto row_of = [&](int h, int* part, int* hh) {
    *part = h < hq ? 0 : h < hq + hk ? 1 : 2;
    *hh = *part == 0 ? h : *part == 1 ? h - hq : h - hq - hk;
    return static_cast<const TIn*>(a.src[*part]) + int64_t(t) * a.stride[*part] + *hh * D + lane * E;
  };
  pdl_launch_next();
  pdl_wait_prior();
  int part, hh;
  float xs[PER][E];  // this warp's first PER heads
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (warp + i * warps < total) load_row<TIn, E>(row_of(warp + i * warps, &part, &hh), xs[i]);
  if (warp == 0) {
    const int s = find_seq(a.b.starts, a.b.seqs, t, lane);
    if (lane == 0) {
      bool bad;
      const SeqSpan q = seq_span(a.b, s, &bad);
      // rows before the first or behind the last sequence have no position
      int pos = t >= q.row0 && t < q.row0 + q.n ? q.len - q.n + (t - q.row0) : -1;
      int page = 0;
      if (pos >= 0) {
        page = a.b.table[int64_t(s) * a.b.width + (pos >> a.b.page_shift)];
        if (page < 0 || page >= a.b.pages) bad = true, pos = -1;
      }
      if (bad && a.err) atomicExch(a.err, DEVICE_ERR_PAGE);
      s_pos = pos;
      s_page = page;
    }
  }
  __syncthreads();
  const int pos = s_pos;
  if (pos < 0) return;
  if (a.inv_freq) {
    for (int i = int(threadIdx.x); i < a.rot_half; i += int(blockDim.x)) {
      const double turns = double(pos) * (a.inv_freq[i] * 0.15915494309189533577);
      float sn, cs;
      sincospif(float(2.0 * (turns - rint(turns))), &sn, &cs);
      turn[i] = make_float2(cs, sn);
    }
    __syncthreads();
  }
  const int64_t slot = (int64_t(s_page) << a.b.page_shift) + (pos & ((1 << a.b.page_shift) - 1));
  const auto head = [&](int h, float(&x)[E]) {
    row_of(h, &part, &hh);
    if (a.norm[part]) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float sc = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
      if (a.norm[part] == 2) {
        float w[E];
        load_row<float, E>(a.norm_w[part] + lane * E, w);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = x[i] * sc * w[i];
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] *= sc;
      }
    }
    if (a.inv_freq && part != 2) {
      const int lanes = a.rot_half / E;  // lanes of the first half
      const bool first = lane < lanes, second = lane >= lanes && lane < 2 * lanes;
      const int from = first ? lane + lanes : second ? lane - lanes : lane;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float y = __shfl_sync(0xffffffffu, x[i], from);
        if (first || second) {
          const float2 cs = turn[(first ? lane : lane - lanes) * E + i];
          x[i] = first ? fmaf(x[i], cs.x, -(y * cs.y)) : fmaf(x[i], cs.x, y * cs.y);
        }
      }
    }
    T* dst = part == 0 ? static_cast<T*>(a.q_out) + (int64_t(t) * hq + hh) * D
                       : static_cast<T*>(a.cache[part - 1]) + (slot * hk + hh) * D;
    store_row<T, E>(dst + lane * E, x);
  };
  // PER rows in flight: a row's successor is loaded before its partner is used
  for (int h = warp; h < total; h += PER * warps) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (h + i * warps >= total) break;
      float x[E];
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = xs[i][e];
      const int after = h + (PER + i) * warps;
      if (after < total) load_row<TIn, E>(row_of(after, &part, &hh), xs[i]);
      head(h + i * warps, x);
    }
  }
}

template <class TIn, class T, int E>
cudaError_t launch_append_e(const AppendArgs& a, cudaStream_t st) {
  const int total = a.heads[0] + 2 * a.heads[1];
  const int per = (total + AP_MAX_WARPS - 1) / AP_MAX_WARPS;  // heads a warp takes, evenly
  const dim3 grid(unsigned(a.b.rows)), block(unsigned(32 * ((total + per - 1) / per)));
  return per == 1 ? launch_pdl(hc_paged_append_kernel<TIn, T, E, 1>, grid, block, 0, st, a)
                  : launch_pdl(hc_paged_append_kernel<TIn, T, E, 2>, grid, block, 0, st, a);
}

template <class TIn, class T>
cudaError_t launch_append(const AppendArgs& a, int dim, cudaStream_t st) {
  return dim == 64 ? launch_append_e<TIn, T, 2>(a, st) : dim == 128 ? launch_append_e<TIn, T, 4>(a, st)
                                                                    : launch_append_e<TIn, T, 8>(a, st);
}

}  // namespace
}  // namespace hc

extern "C" {

int hpc_paged_kv_append(const void *d_k, size_t k_stride, const void *d_v, size_t v_stride, const void *d_q,
                        size_t q_stride, int in_dtype, size_t rows, size_t heads, size_t kv_heads, size_t head_dim,
                        const double *d_inv_freq, size_t rot_half, const float *d_q_norm, const float *d_k_norm,
                        int norm_v, double eps, void *d_key_cache, void *d_value_cache, int cache_dtype, size_t pages,
                        size_t page_size, const int32_t *d_page_table, size_t table_width,
                        const int32_t *d_query_starts, const int32_t *d_kv_lens, size_t seqs, void *d_q_out,
                        void *stream) {
  if (page_size == 0) return hpc_fail(HPC_ERR_SHAPE, "paged append: page_size 0");
  if (int rc = hpc_paged_check("paged append", heads, kv_heads, head_dim, rows, seqs, pages, page_size, table_width))
    return rc;
  if (cache_dtype != HPC_DTYPE_F16 && cache_dtype != HPC_DTYPE_BF16)
    return hpc_fail(HPC_ERR_TYPE, "paged append: cache type %d", cache_dtype);
  if (in_dtype != HPC_DTYPE_F32 && in_dtype != cache_dtype)
    return hpc_fail(HPC_ERR_TYPE, "paged append: input type %d with cache type %d", in_dtype, cache_dtype);
  const size_t e = head_dim / 32, esz = in_dtype == HPC_DTYPE_F32 ? 4 : 2;
  if (rot_half > head_dim / 2 || rot_half % e)
    return hpc_fail(HPC_ERR_SHAPE, "paged append: %zu rotated pairs of head_dim %zu (at most half of it, in steps of %zu)",
                    rot_half, head_dim, e);
  if (k_stride < kv_heads * head_dim || v_stride < kv_heads * head_dim || (d_q && q_stride < heads * head_dim) ||
      k_stride % e || v_stride % e || (d_q && q_stride % e) || k_stride > size_t(INT32_MAX) ||
      v_stride > size_t(INT32_MAX) || q_stride > size_t(INT32_MAX))
    return hpc_fail(HPC_ERR_SHAPE, "paged append: row strides %zu, %zu, %zu", q_stride, k_stride, v_stride);
  if (!(eps >= 0.0)) return hpc_fail(HPC_ERR_ARG, "paged append: eps %g", eps);
  if (rows == 0 || seqs == 0) return HPC_OK;
  if (!d_k || !d_v || !d_key_cache || !d_value_cache || !d_page_table || !d_query_starts || !d_kv_lens ||
      (d_q && !d_q_out) || (rot_half && !d_inv_freq))
    return hpc_fail(HPC_ERR_ARG, "null pointer");
  const auto off = [](const void *p, size_t n) { return p && reinterpret_cast<uintptr_t>(p) % n != 0; };
  const size_t in_al = e * esz < 16 ? e * esz : 16, out_al = e * 2, w_al = e * 4 < 16 ? e * 4 : 16;
  if (off(d_k, in_al) || off(d_v, in_al) || off(d_q, in_al) || off(d_key_cache, out_al) || off(d_value_cache, out_al) ||
      off(d_q_out, out_al) || off(d_q_norm, w_al) || off(d_k_norm, w_al))
    return hpc_fail(HPC_ERR_ARG, "paged append: rows must be aligned to 16 bytes (or one lane's share of a head)");
  hc::AppendArgs a{};
  a.src[0] = d_q, a.src[1] = d_k, a.src[2] = d_v;
  a.stride[0] = int64_t(q_stride), a.stride[1] = int64_t(k_stride), a.stride[2] = int64_t(v_stride);
  a.heads[0] = d_q ? int(heads) : 0, a.heads[1] = a.heads[2] = int(kv_heads);
  a.norm_w[0] = d_q_norm, a.norm_w[1] = d_k_norm;
  a.norm[0] = d_q_norm ? 2 : 0, a.norm[1] = d_k_norm ? 2 : 0, a.norm[2] = norm_v ? 1 : 0;
  a.inv_freq = rot_half ? d_inv_freq : nullptr;
  a.rot_half = int(rot_half);
  a.eps = float(eps);
  a.q_out = d_q_out;
  a.cache[0] = d_key_cache, a.cache[1] = d_value_cache;
  a.b = hpc_paged_batch(d_query_starts, d_kv_lens, d_page_table, seqs, table_width, rows, pages, page_size);
  a.err = hc::device_status_word();
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  if (cache_dtype == HPC_DTYPE_F16)
    err = in_dtype == HPC_DTYPE_F32 ? hc::launch_append<float, __half>(a, int(head_dim), st)
                                    : hc::launch_append<__half, __half>(a, int(head_dim), st);
  else
    err = in_dtype == HPC_DTYPE_F32 ? hc::launch_append<float, __nv_bfloat16>(a, int(head_dim), st)
                                    : hc::launch_append<__nv_bfloat16, __nv_bfloat16>(a, int(head_dim), st);
  HPC_CK(err, "paged append launch");
  return HPC_OK;
}

}  // extern "C"
