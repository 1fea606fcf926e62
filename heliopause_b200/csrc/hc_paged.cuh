// hc_paged.cuh -- shared pieces of the paged KV cache and its attention.
//
// Cache layout: keys and values are [pages][page_size][kv_heads][head_dim]
// in f16 or bf16, page_size a power of two, so that the element rows of one
// (slot, head) are contiguous and slot = page * page_size + offset is one
// coordinate of a tensor map.  Sequence s of a batch owns the packed rows
// query_starts[s] .. query_starts[s + 1] - 1; kv_lens[s] is its length with
// them counted in, so row i of it stands at position kv_lens[s] - new + i.
// Lengths and tables are read on the device only (a captured graph follows
// them from replay to replay), so every value is bounded there: a length
// beyond the table, a page outside the cache or starts outside the rows set
// DEVICE_ERR_PAGE in the device status word, and no access follows them.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/heliocuda.h"
#include "hc_bulk.cuh"
#include "hc_common.cuh"
#include "hc_internal.h"
#include "hc_kernels.cuh"

namespace hc {

constexpr int DEVICE_ERR_PAGE = 2;  // a paged batch's table, lengths or starts point outside their buffers

// One batch of sequences, as the entry points take it.
struct PagedBatch {
  const int32_t* starts;   // [seqs + 1]
  const int32_t* kv_lens;  // [seqs]; nullptr: every sequence is its own rows (whole prompts)
  const int32_t* table;    // [seqs][width]; nullptr: keys are the packed rows themselves
  int seqs;
  int width;
  int rows;                // rows of the packed tensors
  int page_shift;          // log2(page_size)
  int64_t pages;
};

struct SeqSpan {
  int row0;  // first packed row
  int n;     // new tokens
  int len;   // keys
};

// Sequence s of the batch, every field inside its buffer.
__device__ __forceinline__ SeqSpan seq_span(const PagedBatch& b, int s, bool* bad) {
  SeqSpan q;
  const int a = b.starts[s], e = b.starts[s + 1];
  q.row0 = min(max(a, 0), b.rows);
  const int end = min(max(e, q.row0), b.rows);
  q.n = end - q.row0;
  *bad = q.row0 != a || end != e;
  q.len = q.n;
  if (b.kv_lens) {
    const int l = b.kv_lens[s];
    const long long cap = b.table ? (long long)b.width << b.page_shift : 0x7fffffffLL;
    q.len = int(min((long long)max(l, 0), cap));
    *bad = *bad || q.len != l;
  }
  return q;
}

// The first key that a row at position `pos` sees (window 0: all of them).  A
// position is negative where kv_lens is below the new tokens, so it is compared
// before anything is taken from it: with a window near 2^31 the
// difference would not fit.
__device__ __forceinline__ int first_key(int pos, int window) {
  return window > 0 && pos >= window ? pos - window + 1 : 0;
}

template <class T>
struct HalfOps;
template <>
struct HalfOps<__half> {
  static constexpr CUtensorMapDataType kMap = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  __device__ static uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  __device__ static __half from(float v) { return __float2half_rn(v); }
};
template <>
struct HalfOps<__nv_bfloat16> {
  static constexpr CUtensorMapDataType kMap = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  __device__ static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static float2 unpack(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }
  __device__ static __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// 2^x by the special-function unit: 0 for -inf, relative error about 2^-22,
// well below the 16-bit rounding that every probability gets before the
// tensor core multiplies it.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One lane of the converged warp.  Code that issues TMA copies or MMAs runs in
// the whole warp, on values that are the same in every lane, and only the
// instruction itself stands behind this: inside a branch on the lane number
// the compiler passes each one's operands lane by lane (about 80 clocks per
// instruction).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ void pdl_wait_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_next() { asm volatile("griddepcontrol.launch_dependents;"); }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// K or V as a tensor of 128-byte pieces: coordinates (element of the piece,
// slot or row, piece of the token), box 64 x box_rows x box_pieces, written to
// shared memory with the 128-byte swizzle (16-byte chunk c of row r of a
// piece at chunk c ^ (r % 8)).  The innermost coordinate is always 0.
// stride: elements from one token to the next (a multiple of 8).
cudaError_t encode_kv_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t slots,
                          uint64_t stride, int heads, int dim, int box_rows, int box_pieces);

// The same for dimensions, strides (bytes) and box of one's own.
cudaError_t encode_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
                       const cuuint64_t* strides, const cuuint32_t* box);

template <class... KArgs, class... Args>
inline cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                              Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// What an attention launch reads besides the batch.
struct AttnArgs {
  const void* q;
  int64_t q_stride;      // elements from one packed row to the next
  void* out;             // [rows][heads][dim], contiguous
  float* lse;            // [rows][heads] or nullptr
  int heads, kv_heads, dim;
  int window;            // keys a query sees, itself included; 0: all
  float scale_log2;      // scale * log2(e)
  int out_f32;           // out is f32 instead of the cache's type
  int max_q;             // most new tokens of a sequence
  int* err;
};

// The K and V maps' sources.
struct KvSource {
  const void* k;
  const void* v;
  uint64_t slots;
  uint64_t k_stride, v_stride;
  int dtype;
};

size_t attn_rows_workspace_bytes(int dim);
cudaError_t launch_attn_rows(const AttnArgs& a, const PagedBatch& b, const KvSource& kv, void* workspace,
                             cudaStream_t st);

// Many query rows per sequence, on the tensor cores (hc_prompt_attn.cu).
size_t attn_prompt_workspace_bytes(int dim);
cudaError_t launch_attn_prompt(const AttnArgs& a, const PagedBatch& b, const KvSource& kv, void* workspace,
                               cudaStream_t st);

}  // namespace hc

// Argument checks and the batch struct the paged entry points share
// (hc_paged_attn.cu).  table_width 0 with pages 0: no page table.
int hpc_paged_check(const char* what, size_t heads, size_t kv_heads, size_t head_dim, size_t rows, size_t seqs,
                    size_t pages, size_t page_size, size_t table_width);
hc::PagedBatch hpc_paged_batch(const int32_t* starts, const int32_t* lens, const int32_t* table, size_t seqs,
                               size_t width, size_t rows, size_t pages, size_t page_size);
