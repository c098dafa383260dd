// Internal interface of the 4-bit paged key/value cache (kv4.cu: store and load, kv4_attn.cu: attention).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace xtg {

// ---- the cache's layout: pool [pages][kv_heads][72 D] bytes, head dim D 64, 128 or 256; every word 32 bits ----
// A page holds 64 positions of a head in one contiguous block, so that it arrives in one bulk copy:
//   K codes   [D / H][64 slots][4][H / 32] words, H = min(D, 128): nibble n of word [h][slot][a][b] is the code of
//             head dim H h + 32 b + 8 a + n
//   K params  [D / 64][64 slots] words: the scale s (bf16, high half) and the offset z (bf16, low half) of the slot's
//             group of 64 head dims
//   V codes   [2][D / 32][8][4][4] words: nibble n of word [h][c][g][a][t] is the code of head dim 32 c + 8 t + g at
//             slot 32 h + 8 (n % 4) + 2 a + n / 4
//   V params  as K's
// A code c stands for s (c - 8) + z. The orders are those of mma.m16n8k16's operand fragments: lane 4 g + a of the
// attention kernel reads its K codes of a slot and its V codes of 32 slots with 16-byte shared-memory loads, and
// the nibbles n and n + 4 of a word become the two halves of one operand register.
constexpr int kKv4Page = 64;    // positions per page
constexpr int kKv4Group = 64;   // head dims sharing a scale and an offset

__host__ __device__ constexpr int kv4_block_bytes(int D) { return 72 * D; }
__host__ __device__ constexpr int kv4_k_params(int D) { return 32 * D; }   // byte offsets within a block
__host__ __device__ constexpr int kv4_v_codes(int D) { return 36 * D; }
__host__ __device__ constexpr int kv4_v_params(int D) { return 68 * D; }

// Scales are at least 2^-100 (so that 1 / s is finite); a group holding a NaN or an infinity has this word (scale -NaN,
// below every other as a signed integer) and reads back as NaN.
constexpr float kKv4MinScale = 7.888609052210118e-31f;
constexpr uint32_t kKv4NanParam = 0xffc00000u;

enum Kv4Type { kKv4F32 = 0, kKv4Bf16 = 1, kKv4F16 = 2 };

// Where a call's rows stand: sequence s's rows cu_rows[s] .. cu_rows[s + 1] - 1 at positions pos[s], pos[s] + 1, ...;
// position p is slot p % 64 of page table[s][p / 64]. A negative page or position holds nothing.
struct Kv4Where {
  uint8_t* pool;
  int64_t pages;
  int kv_heads, head_dim;
  const int32_t* table;   // [seqs][max_pages]
  int max_pages, seqs;
  const int32_t* pos;       // [seqs]
  const int32_t* cu_rows;   // [seqs + 1]
  int64_t rows;
  int32_t* err;   // or null: set to 6 for a position past the table, 7 for a page past the pool (both hold nothing)
  bool zero_rest; // a load or attention writes zeros for rows that are no sequence's, else leaves them
};

struct Kv4Rows {   // k, v rows of a store (strides in elements) or a load (contiguous)
  void *k, *v;
  int dtype;
  int64_t k_row, k_head, v_row, v_head;
};

struct Kv4Attn {
  Kv4Where w;
  const void* q;   // [rows][heads][D], strides in elements
  void* out;       // [rows][heads][D] contiguous, q's type
  int dtype;
  int64_t q_row, q_head;
  int heads, group, window;   // group: q heads per KV head
  float scale;
  int rows_per_seq;   // about how many rows a sequence has: chooses the tiling, not the result
  float* part;        // workspace, kv4_workspace_bytes
  int part_cost;      // set at the launch, as
  uint32_t polls;     // of a barrier before a wait gives up
};

void launch_kv4_store(const Kv4Where& w, const Kv4Rows& r, cudaStream_t s);
void launch_kv4_load(const Kv4Where& w, const Kv4Rows& r, cudaStream_t s);
int64_t kv4_workspace_bytes(int head_dim, int group, int rows_per_seq, int sms);
int kv4_wait_polls(int polls);   // sets the attention's polls (below 0: leaves them); the former value
void launch_kv4_attention(const Kv4Attn& a, int sms, cudaStream_t s);

#ifdef __CUDACC__
// A launch that may overlap the end of the kernel before it on the stream: the kernel waits (pdl_wait) before it reads or
// writes memory. Each of these kernels lets the next one launch once its own wait is over.
template <class... P, class... A>
void launch_kv4(void (*f)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t s, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  XTG_CUDA(cudaLaunchKernelEx(&cfg, f, static_cast<P>(args)...));
}

// Sequence s's rows within the call's `rows` (a bad cu_rows shortens them, never reaches outside).
__device__ __forceinline__ int64_t kv4_row_bound(const Kv4Where& w, int s) {
  const int64_t c = w.cu_rows[s];
  return c < 0 ? 0 : c > w.rows ? w.rows : c;
}

// Zeros for the rows of out, and of out2 if given (row_bytes each, a multiple of 16), before the sequences' first and after
// their last: by the grid's blocks from `block0` on, which do nothing else. So the others need not know of such rows: in
// every block the check cost 5 % of a bulk load. Four blocks, since such rows are few: 16 took a load of 1000 rows, 102
// blocks, from 4.6 to 5.4 us.
__device__ __forceinline__ void kv4_zero_rest(const Kv4Where& w, void* out, void* out2, int64_t row_bytes,
                                              unsigned block0) {
  const int64_t first = kv4_row_bound(w, 0), last = kv4_row_bound(w, w.seqs);
  for (int64_t i = blockIdx.x - block0; i < first + (w.rows - last); i += gridDim.x - block0) {
    const int64_t at = (i < first ? i : last + (i - first)) * row_bytes;
    for (int64_t x = 16 * threadIdx.x; x < row_bytes; x += 16 * blockDim.x) {
      *reinterpret_cast<uint4*>(static_cast<char*>(out) + at + x) = make_uint4(0, 0, 0, 0);
      if (out2) *reinterpret_cast<uint4*>(static_cast<char*>(out2) + at + x) = make_uint4(0, 0, 0, 0);
    }
  }
}
inline unsigned kv4_rest_blocks(const Kv4Where& w) { return w.zero_rest ? 4 : 0; }

// The page of sequence s's page index i in the pool, -1 when nothing is there.
__device__ __forceinline__ int64_t kv4_page(const Kv4Where& w, int s, int64_t i) {
  if (i < 0) return -1;
  if (i >= w.max_pages) {
    if (w.err) atomicExch(w.err, 6);
    return -1;
  }
  const int64_t p = w.table[(int64_t)s * w.max_pages + i];
  if (p >= w.pages) {
    if (w.err) atomicExch(w.err, 7);
    return -1;
  }
  return p < 0 ? -1 : p;
}
#endif

}  // namespace xtg
