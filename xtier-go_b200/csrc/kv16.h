// Internal interface of the 16-bit paged caches (kv16.cu: append with rotation, kv16_attn.cuh: attention).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace xtg {

enum Kv16Type { kKv16F32 = 0, kKv16Bf16 = 1, kKv16F16 = 2 };

// A cache and where a call's rows stand in it: sequence s's rows cu_rows[s] .. cu_rows[s + 1] - 1 at positions pos[s],
// pos[s] + 1, ...; position p is slot p % page of page table[s][p / page]. A negative page or position holds nothing.
// Strides in elements, of 16 bytes each or a multiple. A latent cache has one KV head, and its v is k's first v_dim dims.
struct Kv16Cache {
  void *k, *v;
  int dtype;   // kKv16Bf16 or kKv16F16
  bool latent;
  int64_t pages;
  int page, kv_heads, head_dim, v_dim;   // page: positions per page, a power of two
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
  const int32_t* table;   // [seqs][max_pages]
  int max_pages, seqs;
  const int32_t* pos;       // [seqs]
  const int32_t* cu_rows;   // [seqs + 1]
  int64_t rows;
  int32_t* err;   // or null: set to 6 for a position past the table, 7 for a page past the pool (both hold nothing)
};

struct Kv16Append {
  const void *k, *v, *q;   // q or null; of a latent cache v is the latent vectors, k their rotated keys
  void* q_out;             // contiguous, the cache's type
  int dtype, heads;        // of k, v and q
  int64_t k_row, k_head, v_row, v_head, q_row, q_head;
  const float* freq;       // radians a position, [rotary / 2]
  int rotary, first;       // dims first .. first + rotary - 1 of k's and q's heads turn
  bool interleaved;        // dims 2 i and 2 i + 1 are a pair, else i and i + rotary / 2
};

struct Kv16Attn {
  const void *q, *q_rot;   // [rows][heads][..]; q_rot: a latent cache's queries of the rotated key
  void* out;               // [rows][heads][v_dim] contiguous
  int heads;
  int64_t q_row, q_head, r_row, r_head;
  float scale;
  int window, rows_per_seq;   // rows_per_seq: about how many rows a sequence has: chooses the tiling, not the result
  bool zero_rest;             // zeros for rows that are no sequence's
  void* work;
};

bool kv16_dims(bool latent, int head_dim, int v_dim);   // whether there is a kernel for them
void launch_kv16_append(const Kv16Cache& c, const Kv16Append& a, int sms, cudaStream_t s);
int64_t kv16_workspace_bytes(bool latent, int head_dim, int v_dim, int group, int rows_per_seq, int sms);
int kv16_wait_polls(int polls);   // sets the attention's polls (below 0: leaves them); the former value
void launch_kv16_attention(const Kv16Cache& c, const Kv16Attn& a, int sms, cudaStream_t s);

}  // namespace xtg
