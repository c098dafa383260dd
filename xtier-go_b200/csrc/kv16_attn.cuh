// Attention over the 16-bit paged caches: every row sees the cached positions up to its own (with a window only the last
// `window` of these), and
//
//   o[r] = sum_p P[r][p] V[p] / sum_p P[r][p],  P[r][p] = 2^(S[r][p] - m[r]),  S = log2(e) scale q[r] . K[p]
//
// Both products run on tcgen05.mma transposed, so that the cache is the wide operand whatever the number of rows:
// S^T = K Q^T has a chunk's positions as the instruction's M and the rows as its N (16 .. 128), o^T = V^T P^T the dims of V
// as M. K and V are used as TMA brings them (128-byte swizzle: K as a K-major, V as an MN-major operand), no thread touches
// them; of a latent cache one tile is both. S^T and o^T lie in tensor memory; a thread of the softmax warps has one position
// and the rows as columns, so that a chunk's sums need no exchange between threads before the part's end. P^T goes back to
// shared memory as 16-byte pieces (8 rows of a position), the unswizzled MN-major operand.
//
// m[r] is a reference: the row's largest score when it was set (less kHead). It moves, and o and the sums are scaled, when a
// score passes it by kMost, which later chunks seldom bring about. P is rounded to the cache's type, the second product's
// operand (half a step of it, 2^-8 or 2^-11, which stays below the output's own rounding over more than a few positions), and
// summed up as rounded, so that a row's largest weight loses nothing; S, the sums and o are f32, o in stretches (kFoldSteps).
//
// A CTA, or a team of them (Block), takes an equal share of all (sequence, row block, KV head, chunk) items in that order,
// whatever the sequences' lengths; a block that a share cuts goes to the workspace in f32 and a second kernel joins its parts
// in order. The warps of a CTA: one walks the share and issues the copies, one issues the products, the others are the
// softmax's. Every wait is bounded.
//
// What bounds it (B200, bf16, device time, bytes or flops that cannot be done without against 7.43 TB/s of reading and 1692
// TFLOP/s): with few rows the cache's bytes: 64 sequences of 16384 .. 32768 positions, 24 q / 6 KV heads of 128, 690 us,
// 7.0 TB/s; 8 rows each of 64 sequences of 4096 .. 8192 197 us, 6.3 TB/s. With one short sequence latency: 1 x 4096 in 12
// us, of which the start and the plan are 2, the first tile and its softmax 3, the others 2, the end 1.5 and the join 3.5.
// With 128 rows a chunk's chain of waits: scores from tensor memory, the vote, exponentials, P back, 1.75 us at heads of
// 128, of which shared memory needs 0.95 by reckoning (the products read 128 KB, the copies and P write 96 KB, at 128 bytes
// a cycle); the tensor pipe is busy 23 % of a prompt's time, issue slots 33 %: 8192 rows from position 0 with heads of 192
// / 128 485 us, 710 TFLOP/s. A latent cache's tile takes 72 KB and q 72 KB, so there are two slots and a slot's time is
// copy, first product, softmax, second product one after another: 64 sequences of 8192 .. 16384 positions with 16 heads in
// 163 to 184 us, up to 5.5 TB/s, with 64 in 211, with 128 in 349 us, 620 TFLOP/s (the products alone, at their measured
// rates, 170).
// Tried and not taken: four groups of softmax warps for 64 and 128 rows (within 5 %, mostly slower), blocks of 64 rows side by
// side in place of 128 (products of 64 rows read shared memory as often for half the work: 185 -> 233 us), tiles in pieces of
// 128 dims with barriers of their own (20 % slower for latent caches), warps of their own for q (4 % faster for prompts, 4 to
// 10 % slower for latent caches), two CTAs an SM for 32 rows (window of 1024 66 -> 60 us with pages of 16, 58 -> 63 with
// pages of 64, the others 2 to 17 % slower).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "fp4mma.cuh"
#include "kv16.h"

namespace xtg {

namespace kv16 {

constexpr int kSmem = 232448, kSmemHalf = 115200;   // shared memory of a CTA, of one of two
constexpr int kCtrl = 3 * 1024;    // of it for barriers and per-row values
constexpr int kMaxGrid = 320;      // CTAs
// A row's reference is kHead below its largest score when it is set and moves when a score passes kMost above it: P is at
// most 2^kMost. bf16 has f32's range. f16's normal numbers end at 2^16 and at 2^-14: the head keeps small probabilities
// among them.
template <class T>
constexpr float kHead = std::is_same<T, __half>::value ? 4.f : 0.f;
template <class T>
constexpr float kMost = std::is_same<T, __half>::value ? 15.f : 16.f;
constexpr float kFloor = -3.0e38f;   // the least reference of a row that has seen a position
constexpr float kLog2e = 1.4426950408889634f;
// Steps of 16 positions that the matrix unit adds up before its sum goes to f32 sums in the workspace. It cuts its sums off
// towards zero, about two units of their last place a step: values of one sign came out 7.9e-4 small over 8192 steps (131072
// positions), 1.6 times half a step of f16. So after 256 steps 2.5e-5, a twentieth of half a step of f16, after 1024 1e-4, a
// fortieth of half a step of bf16. What it costs: f16 prompts of 128 rows with heads of 256 over 30000 positions 1207 -> 1264 us
// (with 128 steps 10 % more), over 16383 190 -> 194; calls of many short parts 3 % (take_out), the others at most 1 %.
template <class T>
constexpr int kFoldSteps = std::is_same<T, __half>::value ? 256 : 1024;
// Registers of a thread of the 8 softmax warps and of the 4 others, where there are 12. The compiler works with the 168 of the
// launch for all: with 128 rows and chunks of 128 positions it spills 24 bytes.
constexpr int kSoftmaxRegs = 200, kOtherRegs = 104;

template <class T_, int DK_, int DV_, bool LATENT_, int N_>
struct Shape {
  using T = T_;
  static constexpr int DK = DK_, DV = DV_, N = N_;
  static constexpr bool LATENT = LATENT_;
  static constexpr int C = DK <= 192 ? 128 : 64;   // positions of a chunk: the first product's M
  static constexpr int WG = N >= 32 ? 2 : 1;       // groups of 4 softmax warps, each with NW of the rows
  static constexpr int NW = N / WG;
  // Of these a thread has NC: all, or, where the 64 positions of a chunk lie in 16 of a warp's 32 lanes, half of them
  static constexpr int NC = C == 128 ? NW : NW / 2;
  static constexpr int kThreads = WG == 1 ? 192 : WG * 128 + 128;   // with the copies' warp and the products', and two that idle
  static constexpr int kSlotBytes = (DK > DV ? DK : DV) * C * 2;
  static constexpr int kQBytes = N * DK * 2, kPBytes = N * C * 2;
  // Buffers of P: two, where that leaves tiles enough (64 rows: 2 % faster; 128 rows, with a tile less, 1 % slower)
  static constexpr int PB = N <= 32 || (N == 64 && !LATENT) ? 2 : 1;
  static constexpr int kRest = kCtrl + kQBytes + PB * kPBytes;
  // Two CTAs an SM for few rows where three tiles fit into half of the memory, so that one's softmax runs beside the other's
  // (64 sequences of 4096 .. 8192 positions, 8 heads of 64: 166 -> 145 us; 64 of 16384 .. 32768, 24 / 6 heads of 128:
  // 734 -> 705 us; heads of 256 the same)
  static constexpr int OCC = N == 16 && C == 128 && (kSmemHalf - kRest) / kSlotBytes >= 3 ? 2 : 1;
  static constexpr int kFit = ((OCC == 2 ? kSmemHalf : kSmem) - kRest) / kSlotBytes;
  static constexpr int R = kFit > 12 ? 12 : kFit;  // slots of the ring
  static constexpr int kSmemBytes = R * kSlotBytes + kQBytes + PB * kPBytes + kCtrl;
  static constexpr int MO = DV >= 128 ? 128 : 64, DT = DV / MO;   // the second product's M, and how many of them
  static constexpr int kFold = kFoldSteps<T> * 16 / C;   // chunks whose second products are added up in the matrix unit
  static constexpr int kO = 2 * N;                 // tensor memory: S^T twice, then o^T
  static constexpr int kUsed = 2 * N + DT * N;
  static constexpr int kCols = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
  static_assert(R >= (LATENT ? 2 : 3) && kUsed <= 512, "shape");
};

// ---- the walk over a share ----

struct Params {
  CUtensorMap kmap, vmap;
  const void *q, *q_rot;
  void* out;
  int64_t q_row, q_head, r_row, r_head;
  const uint8_t* v;   // for values that are not finite
  int64_t v_page, v_head, v_slot;
  const int32_t *table, *pos, *cu_rows;
  int64_t pages, rows;
  int max_pages, seqs, page_log2, heads, kv_heads, group, window;
  uint32_t group_inv;
  int team;   // CTAs beside each other, a divisor of the grid
  uint32_t team_inv;   // ceil(2^32 / team)
  bool by_item;   // how the cuts are counted
  int part_cost, least_share;   // in chunks: a part's start and end where shares are cut, a share at least
  int slots;   // (sequence, row block) numbers, some of them empty
  float scale;
  bool zero_rest;
  int32_t* err;
  float* work;
  uint32_t polls;
};

// sequence s's first row, within the call's rows (a bad cu_rows shortens sequences, never reaches outside)
__device__ __forceinline__ int64_t row_bound(const Params& a, int s) {
  const int64_t c = a.cu_rows[s];
  return c < 0 ? 0 : c > a.rows ? a.rows : c;
}

__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {   // not negative; most are small
  return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// A row block is N consecutive (row, q head of the KV head's group) pairs of a sequence, one a CTA; `team` CTAs take as many
// blocks beside each other through the same chunks, so that what the blocks share comes from memory once. Sequence s's
// blocks of a team have numbers from cu_rows[s] group / (N team) + s on: at least as many as it needs, found without a
// prefix sum over the sequences.
struct Block {
  int s, p0;         // sequence, the position of its first row
  int64_t row0, f0;  // the call's row of the sequence's first, and the block's first pair in the sequence
  int count;         // pairs, 0: none
  int c0, chunks;    // the first chunk that one of its rows sees, and how many
  int64_t first, last;   // positions of its first and last row
};

template <class S>
__device__ __forceinline__ int64_t block_start(const Params& a, int s) {
  const uint32_t blocks = (uint32_t)(row_bound(a, s) * a.group) / S::N;   // pairs are below 2^31
  return (a.team == 1 ? blocks : __umulhi(blocks, a.team_inv)) + s;        // blocks / team: below 2^27, team at most 8
}

template <class S>
__device__ __forceinline__ int find_sequence(const Params& a, int64_t number) {
  int lo = 0, hi = a.seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (block_start<S>(a, mid) <= number)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Sequence s's pairs f0 .. f0 + count - 1; p0: the position of its first row
template <class S>
__device__ __forceinline__ Block block_at(const Params& a, int s, int p0, int64_t row0, int64_t f0, int count) {
  Block b = {s, p0, row0, f0, count, 0, 0, 0, 0};
  if (count == 0) return b;
  b.first = (int64_t)p0 + (uint32_t)f0 / (uint32_t)a.group;   // pairs are below 2^31
  b.last = (int64_t)p0 + (uint32_t)(f0 + count - 1) / (uint32_t)a.group;
  const int64_t end = (int64_t)a.max_pages << a.page_log2;
  const int64_t lo = a.window > 0 && b.first - a.window + 1 > 0 ? b.first - a.window + 1 : 0;
  const int64_t hi = b.last + 1 < end ? b.last + 1 : end;
  if (lo < hi) {
    b.c0 = (int)(lo / S::C);
    b.chunks = (int)((hi + S::C - 1) / S::C) - b.c0;
  }
  return b;
}

// The blocks of a team with this number
template <class S>
__device__ __forceinline__ Block block_of(const Params& a, int s, int64_t number) {
  const int p0 = a.pos[s];   // all that it needs at once
  const int64_t row0 = row_bound(a, s), n = row_bound(a, s + 1) - row0, pairs = n > 0 ? n * a.group : 0;
  const int most = S::N * a.team;
  const int64_t f0 = (number - block_start<S>(a, s)) * most, left = pairs - f0;
  return block_at<S>(a, s, p0, row0, f0, f0 < 0 || left <= 0 ? 0 : left < most ? (int)left : most);
}

struct Part {
  Block b;
  int head, from, count;   // KV head, chunks c0 + from .. c0 + from + count - 1
  int slot;                // of the workspace, -1: the whole block
};

// x / group for x below group + 128, by a multiplication: group_inv = ceil(2^32 / group), group at most 2^15
__device__ __forceinline__ uint32_t by_group(const Params& a, uint32_t x) { return a.group == 1 ? x : __umulhi(x, a.group_inv); }

// What the joining kernel needs about the block that starts in a CTA's share and ends in another's
struct Cut {
  int64_t row0, f0;
  int head, count, first, last;   // count 0: there is none; the CTA that starts it, the team that ends it
};

template <class S>
struct Share {   // the part of all items that a team takes, in units of chunks
  int64_t from, to, each;
  int64_t number, base;   // where it starts: a block's number and the units before it
  Block block;
};

template <class S>
__host__ __device__ constexpr int64_t part_floats() {
  return (int64_t)S::N * (S::DV + 2);
}
// what a CTA's softmax threads have added up of o: 128 lanes of tensor memory x N columns for each of its DT tiles
template <class S>
__host__ __device__ constexpr int64_t fold_floats() {
  return (int64_t)S::DT * 128 * S::N;
}
// workspace: 2 parts a CTA (acc [DV][N], reference [N], sum [N]), then the cuts, by CTA or, where there are fewer, by
// (block number, KV head, CTA of the team), then the CTAs' sums of o
template <class S>
__host__ __device__ constexpr int64_t fold_offset(int grid) {   // in bytes
  return 2 * (int64_t)grid * part_floats<S>() * 4 + (int64_t)grid * (int64_t)sizeof(Cut);
}
template <class S>
__host__ __device__ constexpr int64_t work_bytes(int grid) {
  return fold_offset<S>(grid) + (int64_t)grid * fold_floats<S>() * 4;
}

template <class S>
struct Walk {
  const Params& a;
  Share<S> sh;
  Block b;
  int s;
  int64_t number, base;
  int head;
  bool have;

  __device__ Walk(const Params& a_, const Share<S>& sh_) : a(a_), sh(sh_), number(sh_.number), base(sh_.base), head(0) {
    have = sh.from < sh.to;
    b = sh.block;
    s = b.s;
  }

  // The next part of the share. The blocks that start in it are noted in `cuts` (if given) for the joining kernel.
  __device__ bool next(Part& p, Cut* cuts) {
    while (have && base < sh.to) {
      if (b.count > 0 && head < a.kv_heads) {
        const int64_t at = base + a.part_cost;   // the item's first chunk
        const int64_t from = sh.from - at, to = sh.to - at;
        const int h = head++;
        const int64_t here = base;
        base += a.part_cost + b.chunks;
        int i = 0, j = 0;
        if (b.chunks == 0) {
          if (here < sh.from) continue;
        } else {
          i = from < 0 ? 0 : from > b.chunks ? b.chunks : (int)from;
          j = to < 0 ? 0 : to > b.chunks ? b.chunks : (int)to;
          if (i >= j) continue;
        }
        const bool starts = i == 0, ends = j == b.chunks;
        p = {b, h, i, j - i, starts && ends ? -1 : starts ? 2 * (int)blockIdx.x + 1 : 2 * (int)blockIdx.x};
        const int member = (int)(blockIdx.x % a.team), before = member * S::N;
        if (a.team > 1) {   // this CTA's block of the team's; it may see fewer chunks, or none of the share's
          p.b = block_at<S>(a, s, b.p0, b.row0, b.f0 + before, max(min(b.count - before, S::N), 0));
          const int x = max(b.c0 + i, p.b.c0), y = min(b.c0 + j, p.b.c0 + p.b.chunks);
          p.from = x - p.b.c0;
          p.count = max(y - x, 0);
        }
        if (cuts && starts && (a.by_item || !ends))
          cuts[a.by_item ? (number * a.kv_heads + h) * a.team + member : blockIdx.x] = {
              p.b.row0, p.b.f0, h, ends ? 0 : p.b.count, (int)blockIdx.x, (int)divide(at + b.chunks - 1, sh.each)};
        if (p.b.count == 0) continue;
        return true;
      }
      head = 0;
      if (++number >= a.slots) return have = false;
      if (s + 1 < a.seqs && block_start<S>(a, s + 1) <= number) ++s;
      b = block_of<S>(a, s, number);
    }
    return false;
  }
};

// The positions that some rows of a part's block see, counted from its first chunk on. In the second product they are taken
// in steps of 16: those of a chunk from `from` to `to`.
struct Seen {
  int lo, hi;
  template <class S>
  __device__ int from(int chunk) const {
    return max(lo - chunk * S::C, 0) & ~15;
  }
  template <class S>
  __device__ int to(int chunk) const {
    return min((hi - chunk * S::C + 15) & ~15, S::C);
  }
};
template <class S>
__device__ __forceinline__ Seen seen_by(const Params& a, const Part& p) {
  const int64_t start = (int64_t)(p.b.c0 + p.from) * S::C, hi = p.b.last + 1 - start, most = (int64_t)p.count * S::C;
  // (a part starts less than a chunk before what its window sees)
  return {a.window > 0 ? (int)max(p.b.first - a.window + 1 - start, (int64_t)0) : 0, (int)(hi < most ? hi : most)};
}

// ---- waits ----

__device__ __forceinline__ void give_up(int* failed, int32_t* err) {
  atomicExch(failed, 1);
  if (err) atomicExch(err, 1);
}

// false: it gave up, after `polls` more looks than one (a look that finds nothing takes about 4 us), or after one once
// another wait of the CTA has
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, uint32_t polls, int* failed, int32_t* err) {
  uint32_t spins = 0;
  while (!mbar_try_wait(bar, parity)) {
    ++spins;
    if (spins > polls || *reinterpret_cast<volatile int*>(failed)) {
      give_up(failed, err);
      return false;
    }
  }
  return true;
}

// one look at a barrier, which does not wait; all lanes of the warp
__device__ __forceinline__ bool passed(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return __all_sync(0xffffffffu, ok != 0);
}

// One lane of the warp, known to be one: the operands of what it issues then stay in uniform registers. With `lane == 0` each
// instruction of the products took 49 cycles to issue, more than most of them take to run (32 to 48).
__device__ __forceinline__ bool elected() {
  uint32_t r;
  asm volatile("{ .reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p; }" : "=r"(r));
  return r != 0;
}

// whether any of the `threads` threads of named barrier `id` votes yes
__device__ __forceinline__ bool vote(int id, int threads, bool yes) {
  uint32_t r;
  asm volatile(
      "{ .reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbar.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q; }"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((uint32_t)yes)
      : "memory");
  return r != 0;
}

// ---- tensor memory and operands ----

constexpr uint64_t kSwizzle128 = 2ull << 61;
__device__ __forceinline__ uint64_t operand(uint32_t saddr, uint32_t lbo, uint32_t sbo, uint64_t swizzle) {
  return smem_desc(saddr, lbo, sbo) | swizzle;
}

// the instruction: f32 sums, A and B of type T, M x N; transposed operands are MN-major
template <class T>
__host__ __device__ constexpr uint32_t instruction(int m, int n, bool transposed) {
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1 : 0, tr = transposed ? 1 : 0;
  return (1u << 4) | (type << 7) | (type << 10) | (tr << 15) | (tr << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(
          d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

// M columns from `taddr` on, of this warp's 32 lanes; HALVES: columns 0 .. M - 1 of its first 16 lanes for lanes 0 .. 15 and
// columns M .. 2 M - 1 of the same for lanes 16 .. 31
template <bool HALVES, int M>
__device__ __forceinline__ void load_columns(uint32_t taddr, float (&v)[M]) {
  static_assert(M % 8 == 0 && (HALVES || M % 16 == 0), "columns");
  uint32_t r[16];
#pragma unroll
  for (int c = 0; c < M; c += 16) {
    if (!HALVES) {
      tmem_ld16(taddr + c, *reinterpret_cast<float(*)[16]>(&v[c]));
    } else if (M % 16 == 8) {
      asm volatile("tcgen05.ld.sync.aligned.16x32bx2.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8], %9;"
                   : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                   : "r"(taddr + c), "n"(M));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c + j] = __uint_as_float(r[j]);
    } else {
      asm volatile(
          "tcgen05.ld.sync.aligned.16x32bx2.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16], %17;"
          : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
            "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
          : "r"(taddr + c), "n"(M));
#pragma unroll
      for (int j = 0; j < 16; ++j) v[c + j] = __uint_as_float(r[j]);
    }
  }
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float (&v)[16]) {
  uint32_t r[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(v[j]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// a box of the cache: slots from y on of 64-dim slices from x on, of a KV head z and page w
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int y, int x, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(
          dst),
      "l"(map), "r"(smem_u32(bar)), "r"(0), "r"(y), "r"(x), "r"(z), "r"(w)
      : "memory");
}

// 16 bytes from global to shared memory, zeros where not `live`
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ---- values of the cache's type ----

__device__ __forceinline__ uint32_t pack(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __half) { return pack_f16x2(lo, hi); }
__device__ __forceinline__ float2 unpack(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ __nv_bfloat16 narrow(float x, __nv_bfloat16) { return __float2bfloat16_rn(x); }
__device__ __forceinline__ __half narrow(float x, __half) { return __float2half_rn(x); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// sum += a half of a packed pair, without an instruction to unpack it
__device__ __forceinline__ void add_halves(float& lo, float& hi, uint32_t w, __nv_bfloat16) {
  asm("{ .reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.bf16 %0, l, %0;\n\tadd.rn.f32.bf16 %1, h, %1; }"
      : "+f"(lo), "+f"(hi)
      : "r"(w));
}
__device__ __forceinline__ void add_halves(float& lo, float& hi, uint32_t w, __half) {
  asm("{ .reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.f16 %0, l, %0;\n\tadd.rn.f32.f16 %1, h, %1; }"
      : "+f"(lo), "+f"(hi)
      : "r"(w));
}
// floats as integers of the same order (NaN aside), for atomicMax
__device__ __forceinline__ int ordered(float x) {
  const int i = __float_as_int(x);
  return i >= 0 ? i : i ^ 0x7fffffff;
}
__device__ __forceinline__ float of_ordered(int i) { return __int_as_float(i >= 0 ? i : i ^ 0x7fffffff); }

// Over groups of LANES lanes (32, or 16: the halves of a warp), each of M values: halves of the set change places at lane
// distances LANES / 2, .. 1 until every lane has spread_left values, which lanes may share. Value j of a lane is then number
// spread_column(j) of the set.
template <int M, int LANES, class F>
__device__ __forceinline__ void spread(float (&v)[M], F f) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = LANES / 2, m = M; d > 0; d >>= 1) {
    if (m > 1) {
      m >>= 1;
      const bool up = lane & d;
#pragma unroll
      for (int j = 0; j < M / 2; ++j)
        if (j < m) {
          const float other = __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j + m], d);
          v[j] = f(up ? v[j + m] : v[j], other);
        }
    } else {
      v[0] = f(v[0], __shfl_xor_sync(0xffffffffu, v[0], d));
    }
  }
}
template <int M, int LANES>
constexpr int spread_left() {
  return M > LANES ? M / LANES : 1;
}
template <int M, int LANES>
__device__ __forceinline__ int spread_column(int j) {
  const int lane = threadIdx.x & 31;
  int c = j;
#pragma unroll
  for (int d = LANES / 2, m = M; d > 0; d >>= 1)
    if (m > 1) {
      m >>= 1;
      if (lane & d) c += m;
    }
  return c;
}

// Zeros for the infinities and NaN among 8 values
__device__ __forceinline__ void drop_unbounded(uint4& x, uint32_t exponent, uint32_t one) {
  uint32_t* w = &x.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t hit = ((w[i] & exponent) + one) & 0x80008000u;   // a full exponent carries into the sign's bit
    w[i] &= ~((hit >> 15) * 0xffffu);
  }
}
__device__ __forceinline__ void drop_unbounded(uint4& x, __nv_bfloat16) { drop_unbounded(x, 0x7f807f80u, 0x00800080u); }
__device__ __forceinline__ void drop_unbounded(uint4& x, __half) { drop_unbounded(x, 0x7c007c00u, 0x04000400u); }

// Adds V's infinities and NaN of dim d, which drop_unbounded has taken out of the part's chunks where some of the block's
// rows see a position, to the rows r0 .. r0 + 15 that do: a weight above zero times these is these. (Where all rows see them they
// stay in the product, and a weight that rounded to zero makes NaN of an infinity, as a part's weight of zero does in the join.)
template <class S>
__device__ __forceinline__ void add_unbounded(const Params& a, const Part& p, int d, int r0, uint32_t j0, float (&o)[16]) {
  using T = typename S::T;
  const int64_t from = (int64_t)(p.b.c0 + p.from) * S::C;
  const int64_t to = min(from + (int64_t)p.count * S::C, (int64_t)a.max_pages << a.page_log2);
  const int between = (int)(p.b.last - p.b.first);   // positions that some rows see: behind the first row's, and before
                                                     // what the last row's window starts with
  for (int i = 1; i <= 2 * between; ++i) {
    const int64_t pos = i <= between ? p.b.first + i : p.b.first - a.window + (i - between);
    if (i > between && (a.window == 0 || pos > p.b.first)) break;
    if (pos < from || pos >= to) continue;
    const int64_t page = a.table[(int64_t)p.b.s * a.max_pages + (pos >> a.page_log2)];
    if (page < 0 || page >= a.pages) continue;
    const int64_t slot = pos & ((1 << a.page_log2) - 1);
    const float v = static_cast<float>(
        reinterpret_cast<const T*>(a.v)[page * a.v_page + p.head * a.v_head + slot * a.v_slot + d]);
    if (fabsf(v) < INFINITY) continue;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int64_t t = p.b.first + by_group(a, j0 + r0 + j);
      if (pos <= t && (a.window == 0 || pos > t - a.window)) o[j] += v;
    }
  }
}

// A group's columns of o from tensor memory to its threads' f32 sums, 4 rows of a tile every 128 float4: (first ? 0 : these scaled
// to the rows' references) + o; unless `bad`. kept: the reference of row `own`'s sums; the new one. Functions of their own: within
// the kernel they made calls of many short parts 5 % slower (4096 x 1 token over 128 positions 345 -> 361 us, so 355), although none
// of these comes here.
template <class S>
__device__ __noinline__ float take_out(uint32_t taddr, float4* sums, const float* ref, float* scale, float kept, bool first,
                                       bool bad, int bar) {
  const int own = threadIdx.x & 127;
  named_bar_sync(bar, 128);   // what was in `scale` was read
  if (own < S::NW) {
    const float now = ref[own];
    scale[own] = kept == now ? 1.f : ex2_approx(kept - now);
    kept = now;
  }
  named_bar_sync(bar, 128);
  if (bad) return kept;
  tc_fence_after();
  constexpr int kAtOnce = S::NW < 32 ? S::NW : 32;   // rows whose sums are on the way at once
#pragma unroll 1
  for (int m = 0; m < S::DT; ++m)
#pragma unroll 1
    for (int r0 = 0; r0 < S::NW; r0 += kAtOnce) {
      float4 x[kAtOnce / 4];
      float4* const at = sums + (m * S::NW + r0) / 4 * 128;
#pragma unroll
      for (int j = 0; j < kAtOnce / 4; ++j) x[j] = first ? make_float4(0.f, 0.f, 0.f, 0.f) : at[j * 128];
#pragma unroll
      for (int r = 0; r < kAtOnce; r += 16) {
        float o[16];
        tmem_ld16(taddr + m * S::N + r0 + r, o);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(scale + r0 + r + j), old = x[(r + j) / 4];
          at[(r + j) / 4 * 128] = make_float4(fmaf(old.x, f.x, o[j]), fmaf(old.y, f.y, o[j + 1]), fmaf(old.z, f.z, o[j + 2]),
                                              fmaf(old.w, f.w, o[j + 3]));
        }
      }
    }
  return kept;
}
// and back: o + these x scale
template <class S>
__device__ __noinline__ void bring_back(uint32_t taddr, const float4* sums, const float* scale) {
#pragma unroll 1
  for (int m = 0; m < S::DT; ++m)
#pragma unroll 1
    for (int r = 0; r < S::NW; r += 16) {
      float o[16];
      tmem_ld16(taddr + m * S::N + r, o);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const float4 x = sums[(m * S::NW + r + j) / 4 * 128], f = *reinterpret_cast<const float4*>(scale + r + j);
        o[j] = fmaf(x.x, f.x, o[j]), o[j + 1] = fmaf(x.y, f.y, o[j + 1]);
        o[j + 2] = fmaf(x.z, f.z, o[j + 2]), o[j + 3] = fmaf(x.w, f.w, o[j + 3]);
      }
      tmem_st16(taddr + m * S::N + r, o);
    }
  tmem_st_wait();
}

// ---- the CTA's shared memory ----

constexpr int kInfo = 16, kQueue = 4;

template <class S>
struct __align__(16) Ctrl {
  uint64_t full[S::R], empty[S::R], sfull[2], sfree[2], pready[2], pdone[2], qready, done, queue_full[kQueue],
      queue_empty[kQueue];
  Part queue[kQueue];
  uint32_t info[kInfo];   // of chunks in turn: the pieces that are there
  int64_t scan[12];
  Share<S> share;
  uint32_t tmem;
  int failed;
  int unbounded[4];   // of every 4th part that has chunks: whether positions that some rows see have values that are not
                      // finite
};
template <class S>
struct __align__(16) Rows {
  float ref[S::N], alpha[S::N];
  int top[S::N];   // ordered()
  int place[S::N];   // the row's place in out
};

template <class S>
__global__ void __launch_bounds__(S::kThreads, S::OCC) attention_kernel(const __grid_constant__ Params a) {
  using T = typename S::T;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  uint8_t* qbuf = smem + S::R * S::kSlotBytes;
  uint8_t* pbuf = qbuf + S::kQBytes;
  Ctrl<S>& c = *reinterpret_cast<Ctrl<S>*>(pbuf + S::PB * S::kPBytes);
  Rows<S>& rows = *reinterpret_cast<Rows<S>*>(&c + 1);
  static_assert(sizeof(Ctrl<S>) % 16 == 0 && sizeof(Ctrl<S>) + sizeof(Rows<S>) <= kCtrl, "control block");
  constexpr int kSoftmaxWarps = 4 * S::WG, kProducer = kSoftmaxWarps, kIssuer = kSoftmaxWarps + 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

  if (warp == kIssuer) tmem_alloc(&c.tmem, S::kCols);
  if (tid == 0) {
    for (int i = 0; i < S::R; ++i) {
      mbar_init(&c.full[i], 1);
      mbar_init(&c.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c.sfull[i], 1);
      mbar_init(&c.sfree[i], kSoftmaxWarps);
      mbar_init(&c.pready[i], kSoftmaxWarps);
      mbar_init(&c.pdone[i], 1);
    }
    mbar_init(&c.qready, kSoftmaxWarps);
    for (int i = 0; i < 4; ++i) c.unbounded[i] = 0;
    mbar_init(&c.done, 1);
    for (int i = 0; i < kQueue; ++i) {
      mbar_init(&c.queue_full[i], 1);
      mbar_init(&c.queue_empty[i], kSoftmaxWarps + 1);
    }
    c.failed = 0;
    mbar_init_fence();
  }
  for (int i = tid; i < S::N; i += S::kThreads) rows.top[i] = ordered(-INFINITY);

  float* parts = a.work;
  Cut* cuts = reinterpret_cast<Cut*>(parts + 2 * (int64_t)gridDim.x * part_floats<S>());

  // ---- the share: the cost of every block, summed up over `threads` threads, of which this is number `index` ----
  auto cost = [&](const Block& b) { return b.count > 0 ? (int64_t)(b.chunks + a.part_cost) * a.kv_heads : (int64_t)0; };
  auto plan = [&](int index, int threads, auto&& sum_before) {
    const int each = (a.slots + threads - 1) / threads;
    const int first = min(index * each, a.slots), last = min(first + each, a.slots);
    Block kept;   // the only one, where each is 1
    auto over_blocks = [&](auto&& f) {
      if (first >= last) return;
      int s = find_sequence<S>(a, first);
      for (int i = first; i < last; ++i) {
        if (s + 1 < a.seqs && block_start<S>(a, s + 1) <= i) ++s;
        kept = block_of<S>(a, s, i);
        if (f(i, kept)) break;
      }
    };
    int64_t mine = 0, before, total;
    over_blocks([&](int i, const Block& b) {
      if (blockIdx.x == 0 && a.by_item && b.count == 0)   // no share has these
        for (int x = 0; x < a.kv_heads * a.team; ++x) cuts[(int64_t)i * a.kv_heads * a.team + x].count = 0;
      if (blockIdx.x == 0 && a.err && b.count > 0 && b.last >= (int64_t)a.max_pages << a.page_log2) atomicExch(a.err, 6);
      mine += cost(b);
      return false;
    });
    sum_before(mine, before, total);
    const uint32_t teams = gridDim.x / a.team;
    Share<S> sh;
    sh.each = max(divide(total + teams - 1, teams), (int64_t)(a.part_cost + a.least_share));
    sh.from = sh.each * (blockIdx.x / a.team);
    sh.to = sh.from + sh.each < total ? sh.from + sh.each : total;
    if (sh.from >= sh.to) {
      if (index == 0) c.share.from = c.share.to = 0;
    } else if (before <= sh.from && sh.from < before + mine) {
      int64_t at = before;
      auto start = [&](int i, const Block& b) {
        const int64_t x = cost(b);
        if (sh.from < at + x) {
          sh.number = i;
          sh.base = at;
          sh.block = b;
          c.share = sh;
          return true;
        }
        at += x;
        return false;
      };
      if (each == 1)
        start(first, kept);
      else
        over_blocks(start);
    }
  };
  auto over_warp = [&](int64_t mine, int64_t& upto) {
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
  };
  // Few blocks: the copies' warp alone, which is the one to wait for it (one sequence of 4096 positions 12.4 us, with all warps
  // 12.7). From some 100 on it is the longer way: 125 blocks 115.6 us and 110.5, 250 blocks 118.0 and 112.1, a prompt of 4096 rows
  // (129) 214.7 and 210.7.
  const bool small_plan = a.slots <= 64;
  if (!small_plan) {
    pdl_wait();
    plan(tid, S::kThreads, [&](int64_t mine, int64_t& before, int64_t& total) {
      int64_t upto;
      over_warp(mine, upto);
      if (lane == 31) c.scan[warp] = upto;
      __syncthreads();
      total = 0;
      before = upto - mine;
#pragma unroll
      for (int w = 0; w < S::kThreads / 32; ++w) {
        if (w < warp) before += c.scan[w];
        total += c.scan[w];
      }
    });
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = c.tmem;
  bool gave_up = false;
  auto bounded = [&](uint64_t* bar, uint32_t parity) { return wait(bar, parity, a.polls, &c.failed, a.err); };

  // 384 threads start with 168 registers each, which are shared out
  if (warp >= kSoftmaxWarps) {
    if (S::WG == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kProducer) {
      // ---- the walk and the copies: K of a chunk before V of the chunk before, as the products take them ----
      constexpr int kSlicesK = S::DK / 64, kSlicesV = S::DV / 64;
      const int box = min(1 << a.page_log2, S::C), pieces_log2 = __ffs(S::C / box) - 1, pieces = 1 << pieces_log2;
      bool ok = true;
      if (a.polls == 0) {   // without a look
        give_up(&c.failed, a.err);
        ok = false;
      }
      pdl_wait();
      pdl_launch_next();
      if (small_plan) {
        plan(lane, 32, [&](int64_t mine, int64_t& before, int64_t& total) {
          int64_t upto;
          over_warp(mine, upto);
          total = __shfl_sync(0xffffffffu, upto, 31);
          before = upto - mine;
        });
        __syncwarp();
      }
      uint32_t entry = 0, chunk = 0, queued = 0;
      Part p;
      Walk<S> walk(a, c.share);
      // a tile of K or V into the next slot: in one copy where a page holds the chunk, else page by page and 64 dims at a time
      auto copy = [&](bool v, int head, int slot0, int page, uint32_t there) {
        const int st = entry % S::R, slices = v ? kSlicesV : kSlicesK;
        const CUtensorMap* map = v ? &a.vmap : &a.kmap;
        const uint32_t turn = entry / S::R, to = smem_u32(ring) + st * S::kSlotBytes;
        if (turn > 0) ok = __all_sync(0xffffffffu, bounded(&c.empty[st], (turn - 1) & 1));
        if (!ok) return;
        if (lane == 0) mbar_expect_tx(&c.full[st], (uint32_t)(__popc(there) * slices * box * 128));
        __syncwarp();
        if (pieces == 1) {
          if (lane == 0 && there) load_box(to, map, slot0, 0, head, page, &c.full[st]);
        } else {
          const int x = lane & (pieces - 1), pg = __shfl_sync(0xffffffffu, page, x);   // at most 8 pieces, 9 slices
          for (int slice = lane >> pieces_log2; slice < slices; slice += 32 >> pieces_log2)
            if (there >> x & 1) load_box(to + slice * S::C * 128 + x * box * 128, map, slot0, slice, head, pg, &c.full[st]);
        }
        ++entry;
      };
      Cut* const note = lane == 0 ? cuts : nullptr;
      if (!a.by_item && lane == 0) cuts[blockIdx.x].count = 0;
      bool more = true;
      auto next = [&] {   // the next part into the queue, or its end
        more = walk.next(p, note);
        const int qi = queued % kQueue;
        if (ok && queued >= kQueue) ok = __all_sync(0xffffffffu, bounded(&c.queue_empty[qi], (queued / kQueue - 1) & 1));
        if (ok && lane == 0) {
          if (!more) p.head = -1;
          c.queue[qi] = p;
          mbar_arrive(&c.queue_full[qi]);
        }
        ++queued;
      };
      next();
      while (more) {
        const int head = p.head, count = p.count, chunk0 = p.b.c0 + p.from;
        const int32_t* table = a.table + (int64_t)p.b.s * a.max_pages;
        const int64_t hi = min(p.b.last + 1, (int64_t)a.max_pages << a.page_log2);
        const int64_t lo = a.window > 0 ? p.b.first - a.window + 1 : 0;
        // lane i has the page of piece i; of the next chunk's ahead
        auto page_of = [&](int i) {
          const int64_t at = (int64_t)(chunk0 + i) * S::C + lane * box;
          return i >= count || lane >= pieces || at >= hi || at + box <= lo ? -1 : table[at >> a.page_log2];
        };
        int page = page_of(0), old_page = -1;
        uint32_t old_there = 0;
        int old_slot0 = 0;
        bool stepped = false;
        for (int i = 0; i < count && ok; ++i, ++chunk) {
          const int next_page = page_of(i + 1);   // looked at in the next turn
          if (page >= a.pages) {
            if (a.err) atomicExch(a.err, 7);
            page = -1;
          }
          if (i == count - 1) {   // the softmax looks for the next part at this one's last chunk
            next();
            stepped = true;
          }
          const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
          const int slot0 = (int)(((int64_t)(chunk0 + i) * S::C) & ((1 << a.page_log2) - 1));
          if (lane == 0) c.info[chunk % kInfo] = there;
          if (ok) copy(false, head, slot0, page, there);
          if (!S::LATENT) {
            if (i > 0 && ok) copy(true, head, old_slot0, old_page, old_there);
            if (i == count - 1 && ok) copy(true, head, slot0, page, there);
          }
          old_page = page;
          old_there = there;
          old_slot0 = slot0;
          page = next_page;
        }
        if (!stepped) next();
      }
      // no copy is left in flight
      for (uint32_t e = entry > (uint32_t)S::R ? entry - S::R : 0; e < entry; ++e) {
        uint32_t spins = 0;
        while (!mbar_try_wait(&c.full[e % S::R], (e / S::R) & 1))
          if (++spins > (1u << 18)) break;
      }
      __syncwarp();
    } else if (warp == kIssuer) {
      // ---- the products: whichever of a chunk's second and the next one's first has its operands ----
      constexpr uint32_t kS = instruction<T>(S::C, S::N, false), kOi = instruction<T>(S::MO, S::N, true);
      const uint32_t ring0 = __shfl_sync(0xffffffffu, smem_u32(ring), 0), q0 = __shfl_sync(0xffffffffu, smem_u32(qbuf), 0),
                     pb0 = __shfl_sync(0xffffffffu, smem_u32(pbuf), 0), t = __shfl_sync(0xffffffffu, tmem, 0);
      if (small_plan) pdl_wait();   // no bounded wait begins before the kernels that this one depends on have ended
      uint32_t entry = 0, chunk = 0, filled = 0;
      bool ok = a.polls != 0;
      for (uint32_t part = 0; ok; ++part) {
        const int qi = part % kQueue;
        ok = __all_sync(0xffffffffu, bounded(&c.queue_full[qi], (part / kQueue) & 1));
        if (!ok) break;
        const Part& p = c.queue[qi];
        const int n = __shfl_sync(0xffffffffu, p.count, 0);
        const bool end = __shfl_sync(0xffffffffu, p.head, 0) < 0;
        Seen seen = seen_by<S>(a, p);
        seen.lo = __shfl_sync(0xffffffffu, seen.lo, 0);
        seen.hi = __shfl_sync(0xffffffffu, seen.hi, 0);
        if (lane == 0) mbar_arrive(&c.queue_empty[qi]);
        if (end) break;
        if (n == 0) continue;
        ok = __all_sync(0xffffffffu, bounded(&c.qready, filled & 1));
        ++filled;
        tc_fence_after();
        uint32_t spins = 0;
        for (int si = 0, vi = 0; vi < n && ok;) {   // chunks whose first and whose second product were issued
          bool issued = false;
          if (vi < si) {
            const uint32_t e = S::LATENT ? entry + vi : vi == n - 1 ? entry + 2 * n - 1 : entry + 2 * vi + 2;
            const uint32_t st = e % S::R, ch = chunk + vi, pb = ch % S::PB;
            // (of a latent cache the first product has waited for the tile)
            if (passed(&c.pready[pb], (ch / S::PB) & 1) && (S::LATENT || passed(&c.full[st], (e / S::R) & 1))) {
              tc_fence_after();
              const uint32_t v0 = ring0 + st * S::kSlotBytes, p0 = pb0 + pb * S::kPBytes;
              const int from = seen.from<S>(vi), to = seen.to<S>(vi);
              const bool fresh = vi % S::kFold == 0;   // the sum so far is in the workspace
              if (elected()) {
                auto product = [&](int m, int x, bool accumulate) {
                  mma(t + S::kO + m * S::N, operand(v0 + m * (S::MO / 64) * S::C * 128 + x * 128, S::C * 128, 1024, kSwizzle128),
                      operand(p0 + x * 16, 128, S::C * 16, 0), kOi, accumulate);
                };
                if (to - from == S::C) {
#pragma unroll
                  for (int m = 0; m < S::DT; ++m)
#pragma unroll
                    for (int x = 0; x < S::C; x += 16) product(m, x, !fresh || x > 0);
                } else {
#pragma unroll 1
                  for (int m = 0; m < S::DT; ++m)
#pragma unroll 1
                    for (int x = from; x < to; x += 16) product(m, x, !fresh || x > from);
                }
                tc_commit(&c.empty[st]);
                tc_commit(&c.pdone[pb]);
              }
              __syncwarp();
              ++vi;
              issued = true;
            }
          }
          if (si < n && si < vi + 2) {
            const uint32_t e = S::LATENT ? entry + si : si == 0 ? entry : entry + 2 * si - 1;
            const uint32_t st = e % S::R, ch = chunk + si, buf = ch & 1;
            if (passed(&c.full[st], (e / S::R) & 1) && (ch < 2 || passed(&c.sfree[buf], ((ch >> 1) - 1) & 1))) {
              tc_fence_after();
              const uint32_t k0 = ring0 + st * S::kSlotBytes;
              if (elected()) {
#pragma unroll
                for (int x = 0; x < S::DK; x += 16)
                  mma(t + buf * S::N, operand(k0 + x / 64 * S::C * 128 + x % 64 * 2, 16, 1024, kSwizzle128),
                      operand(q0 + x / 64 * S::N * 128 + x % 64 * 2, 16, 1024, kSwizzle128), kS, x > 0);
                tc_commit(&c.sfull[buf]);
                if (!S::LATENT) tc_commit(&c.empty[st]);
              }
              __syncwarp();
              ++si;
              issued = true;
            }
          }
          if (issued) {
            spins = 0;
          } else if (++spins > 32 * a.polls || (spins % 64 == 0 && *reinterpret_cast<volatile int*>(&c.failed))) {
            // these looks do not wait: some 0.1 us each
            give_up(&c.failed, a.err);
            ok = false;
          }
          ok = __all_sync(0xffffffffu, ok);
        }
        entry += S::LATENT ? n : 2 * n;
        chunk += n;
      }
      if (elected()) {
        tc_commit(&c.done);
        uint32_t spins = 0;   // every product has ended before the tensor memory goes back
        while (!mbar_try_wait(&c.done, 0))
          if (++spins > (1u << 18)) break;
      }
      __syncwarp();
    }
  } else {
    // ---- softmax ----
    if (S::WG == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int wg = warp >> 2, quarter = warp & 3, bar = 1 + wg;
    // this thread's position of a chunk and, from col0 on, its rows of the group's
    const int at = S::C == 128 ? 32 * quarter + lane : 16 * quarter + (lane & 15);
    const int col0 = S::C == 128 ? 0 : (lane >> 4) * S::NC;
    const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16);
    float* ref = rows.ref + wg * S::NW;
    float* alpha = rows.alpha + wg * S::NW;
    int* top = rows.top + wg * S::NW;
    int* place = rows.place + wg * S::NW;
    const int own = tid & 127;
    const float sc = a.scale * kLog2e;
    const uint32_t group = (uint32_t)a.group;
    // this thread's columns of o's tiles, 4 rows at a time, as far as they were taken from tensor memory
    float4* const fold = reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(a.work) + fold_offset<S>(gridDim.x)) +
                         (blockIdx.x * fold_floats<S>() + wg * (S::DT * 128 * S::NW)) / 4 + own;
    const int box = min(1 << a.page_log2, S::C);
    const uint32_t all_pieces = (1u << (S::C / box)) - 1;

    // q's rows into the first product's operand, zeros past the last
    auto load_q = [&](const Part& p) {
      constexpr int kUnits = S::DK / 8;   // 16-byte pieces of a row
      const uint32_t f0 = (uint32_t)p.b.f0, rt0 = f0 / group, j0 = f0 - rt0 * group;
      const int64_t row0 = p.b.row0 + rt0;
      const int count = p.b.count, head0 = p.head * a.group;
#pragma unroll 4
      for (int i = 0; i < (S::NW * kUnits + 127) / 128; ++i) {
        const int x = i * 128 + own, row = x / kUnits, u = x % kUnits, r = wg * S::NW + row;
        if (S::NW * kUnits % 128 == 0 || row < S::NW) {
          const uint32_t pair = j0 + r, rt = by_group(a, pair);
          const int64_t t = row0 + rt, h = head0 + (int)(pair - rt * group);
          const T* from = S::LATENT && u >= S::DV / 8
                              ? static_cast<const T*>(a.q_rot) + t * a.r_row + h * a.r_head + (8 * u - S::DV)
                              : static_cast<const T*>(a.q) + t * a.q_row + h * a.q_head + 8 * u;
          const bool live = r < count;
          copy16(smem_u32(qbuf) + u / 8 * S::N * 128 + r * 128 + ((u ^ r) & 7) * 16, live ? from : a.q, live);
        }
      }
    };
    auto finish_q = [&] {
      copy16_wait();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.qready);
    };

    if (small_plan) pdl_wait();
    uint32_t chunk = 0, entry = 0, filled = 0;   // filled: parts with chunks
    bool bad = false, known = false;   // known: the next part is in the queue and its q on the way
    for (uint32_t part = 0;; ++part) {
      const Part& p = c.queue[part % kQueue];
      if (!known) bad = !__all_sync(0xffffffffu, bounded(&c.queue_full[part % kQueue], (part / kQueue) & 1)) || bad;
      if (vote(bar, 128, bad)) {
        bad = true;
        break;
      }
      if (p.head < 0) break;
      const int count = p.count;
      if (!known && count > 0) {
        load_q(p);
        finish_q();
      }
      known = false;
      const uint32_t t0 = (uint32_t)p.b.f0 / group, j0 = (uint32_t)p.b.f0 - t0 * group;
      if (own < S::NW) {
        // the row of out, counted over rows and heads (below 2^31)
        const uint32_t r = j0 + wg * S::NW + own, rt = by_group(a, r);
        place[own] = (int)((p.b.row0 + t0 + rt) * a.heads + (int64_t)p.head * a.group + (r - rt * group));
        ref[own] = -INFINITY;
      }
      volatile int* const unbounded = &c.unbounded[filled % 4];
      if (count > 0) {
        // the other group is in this part or at the end of the one before: a chunk's second product waits for both
        if (wg == 0 && own == 0) c.unbounded[(filled + 2) % 4] = 0;
        ++filled;
      }
      named_bar_sync(bar, 128);
      const int64_t first_pos = p.b.first, last_pos = p.b.last;
      const int64_t start0 = (int64_t)(p.b.c0 + p.from) * S::C;
      const int pairs = p.b.count;
      const Seen part_seen = seen_by<S>(a, p);
      float l[S::NC];
#pragma unroll
      for (int r = 0; r < S::NC; ++r) l[r] = 0.f;

      float kept = -INFINITY;   // of row `own`: the reference of the sums in the workspace

      for (int i = 0; i < count; ++i, ++chunk) {
        const int buf = chunk & 1;
        bad = !__all_sync(0xffffffffu, bounded(&c.sfull[buf], (chunk >> 1) & 1)) || bad;
        tc_fence_after();
        float y[S::NC];
        auto load_scores = [&] {
          load_columns<S::C == 64>(lanes + buf * S::N + wg * S::NW, y);
          tmem_ld_wait();
        };
        load_scores();
        bool q_coming = false;
        if (i == count - 1) {   // the last product that reads q is done
          const uint32_t next = part + 1;
          bad = !__all_sync(0xffffffffu, bounded(&c.queue_full[next % kQueue], (next / kQueue) & 1)) || bad;
          if (!bad) {
            known = true;
            const Part& np = c.queue[next % kQueue];
            q_coming = np.head >= 0 && np.count > 0;
            if (q_coming) load_q(np);
          }
        }
        const int64_t start = start0 + (int64_t)i * S::C, pos = start + at;
        const uint32_t there = c.info[chunk % kInfo];
        const bool clean = there == all_pieces && start + S::C - 1 <= first_pos &&
                           (a.window == 0 || start > last_pos - a.window);
        // rows lo .. hi - 1 of the block see this thread's position: their positions t = first_pos + (j0 + r) / group, with
        // pos - window < t - window + 1 <= pos <= t
        int lo = 0, hi = S::N;
        if (!clean) {
          const int64_t rel = pos - first_pos;
          const int64_t x = rel * group - j0, z = a.window > 0 ? (rel + a.window) * group - j0 : S::N;
          lo = x < 0 ? 0 : x > S::N ? S::N : (int)x;
          hi = z < 0 ? 0 : z > S::N ? S::N : (int)z;
          if (!(there >> (at / box) & 1)) lo = S::N;
        }
        const int lo_own = lo - wg * S::NW - col0, hi_own = hi - wg * S::NW - col0;
        auto hide = [&] {
#pragma unroll
          for (int r = 0; r < S::NC; ++r)
            if (r < lo_own) y[r] = -INFINITY;
          if (a.window > 0)
#pragma unroll
            for (int r = 0; r < S::NC; ++r)
              if (r >= hi_own) y[r] = -INFINITY;
        };
        auto less_reference = [&] {   // scores less the reference; what a row does not see is -infinity
#pragma unroll
          for (int r = 0; r < S::NC; r += 4) {
            const float4 f = *reinterpret_cast<const float4*>(ref + col0 + r);
            y[r] = fmaf(y[r], sc, -f.x);
            y[r + 1] = fmaf(y[r + 1], sc, -f.y);
            y[r + 2] = fmaf(y[r + 2], sc, -f.z);
            y[r + 3] = fmaf(y[r + 3], sc, -f.w);
          }
          if (!clean) hide();
        };
        bool over = false;
        if (i > 0) {
          less_reference();
          float m[4] = {y[0], y[1], y[2], y[3]};
#pragma unroll
          for (int r = 4; r + 1 < S::NC; r += 2) m[r / 2 % 4] = max_nan(m[r / 2 % 4], y[r], y[r + 1]);
          over = !(max_nan(max_nan(m[0], m[1], m[2]), m[3]) <= kMost<T>);
        }
        if (i == 0 || vote(bar, 128, bad || over)) {
          // a new reference
          if (i > 0) load_scores();
#pragma unroll
          for (int r = 0; r < S::NC; ++r) y[r] = fmaxf(y[r] * sc, kFloor);
          if (!clean) hide();
          spread<S::NC, S::C / 4>(y, [](float u, float v) { return fmaxf(u, v); });
#pragma unroll
          for (int j = 0; j < spread_left<S::NC, S::C / 4>(); ++j)
            atomicMax(&top[col0 + spread_column<S::NC, S::C / 4>(j)], ordered(y[j]));
          if (vote(bar, 128, bad)) {
            bad = true;
            break;
          }
          if (own < S::NW) {
            const float old = ref[own], now = fmaxf(old, of_ordered(top[own]) - kHead<T>);
            alpha[own] = now == old ? 1.f : ex2_approx(old - now);
            ref[own] = now;
            top[own] = ordered(-INFINITY);
          }
          named_bar_sync(bar, 128);
          load_scores();
          less_reference();
          if (i > 0) {   // the sums so far
#pragma unroll
            for (int r = 0; r < S::NC; ++r) l[r] *= alpha[col0 + r];
            const uint32_t b = (chunk - 1) % S::PB;
            bad = !__all_sync(0xffffffffu, bounded(&c.pdone[b], ((chunk - 1) / S::PB) & 1));
            if (!bad) {
              tc_fence_after();
#pragma unroll 1
              for (int m = 0; m < S::DT; ++m)
#pragma unroll 1
                for (int r = 0; r < S::NW; r += 16) {
                  float o[16];
                  const uint32_t from = lanes + S::kO + m * S::N + wg * S::NW + r;
                  tmem_ld16(from, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int j = 0; j < 16; ++j) o[j] *= alpha[r + j];
                  tmem_st16(from, o);
                }
              tmem_st_wait();
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&c.sfree[buf]);
        if (!clean) {
          // V at positions that no row sees is whatever lay there, and 0 x NaN is no 0: zeros. Where some rows see a
          // position, what is not finite becomes zeros too and is added to those rows at the part's end. The groups take a
          // share of the dims each.
          const uint32_t e = S::LATENT ? entry + i : i == count - 1 ? entry + 2 * count - 1 : entry + 2 * i + 2;
          bad = !__all_sync(0xffffffffu, bounded(&c.full[e % S::R], (e / S::R) & 1)) || bad;
          const bool seen = lo < min(hi, pairs);
          if (!bad && (!seen || lo > 0 || hi < pairs) && at >= part_seen.from<S>(i) && at < part_seen.to<S>(i)) {
            uint8_t* v = ring + e % S::R * S::kSlotBytes + at * 128;
            constexpr int kUnits = S::DV / (S::C == 128 ? 8 : 16) / S::WG;   // two threads have a position where C is 64
            const int unit0 = (S::C == 128 ? wg : 2 * wg + (lane >> 4)) * kUnits;
            // neighbouring positions take different 16-byte columns of the 8 at a time (of kUnits, if fewer)
            auto unit = [&](int i) {
              const int u = unit0 + (i ^ (at & (kUnits < 8 ? kUnits - 1 : 7)));
              return reinterpret_cast<uint4*>(v + u / 8 * S::C * 128 + (u % 8) * 16);
            };
            bool found = false;
            if (!seen) {
#pragma unroll
              for (int i = 0; i < kUnits; ++i) *unit(i) = make_uint4(0, 0, 0, 0);
            } else {
              uint32_t most = 0;   // of the magnitudes, as 16-bit integers
#pragma unroll 4
              for (int i = 0; i < kUnits; ++i) {
                const uint4 x = *unit(i);
                most = __vmaxu2(__vmaxu2(most, __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu)),
                                __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
              }
              constexpr uint32_t kFull = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;   // an exponent of ones
              found = (most & 0xffffu) >= kFull || (most >> 16) >= kFull;
              if (found)
                for (int i = 0; i < kUnits; ++i) {
                  uint4 x = *unit(i);
                  drop_unbounded(x, T());
                  *unit(i) = x;
                }
            }
            if (found) *unbounded = 1;
          }
        }
        // P, rounded, and its sums
        const uint32_t pb = chunk % S::PB;
        if (chunk >= (uint32_t)S::PB)
          bad = !__all_sync(0xffffffffu, bounded(&c.pdone[pb], (chunk / S::PB - 1) & 1)) || bad;
        uint8_t* to = pbuf + pb * S::kPBytes + (wg * S::NW + col0) / 8 * S::C * 16 + at * 16;
#pragma unroll
        for (int r = 0; r < S::NC; r += 8) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w[j] = pack(ex2_approx(y[r + 2 * j]), ex2_approx(y[r + 2 * j + 1]), T());
            add_halves(l[r + 2 * j], l[r + 2 * j + 1], w[j], T());
          }
          *reinterpret_cast<uint4*>(to + r / 8 * S::C * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (i > 0 && i % S::kFold == 0) {   // the second product of this chunk starts a new sum, the last one goes to the others
          const uint32_t b = (chunk - 1) % S::PB;
          if (S::PB > 1) bad = !__all_sync(0xffffffffu, bounded(&c.pdone[b], ((chunk - 1) / S::PB) & 1)) || bad;
          kept = take_out<S>(lanes + S::kO + wg * S::NW, fold, ref, alpha, kept, i == S::kFold, bad, bar);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&c.pready[pb]);
        if (q_coming) finish_q();
      }
      entry += S::LATENT ? count : 2 * count;

      // ---- the part's end: the rows' sums over all positions, then o ----
      if (count > 0 && !bad) {
        const uint32_t b = (chunk - 1) % S::PB;
        bad = !__all_sync(0xffffffffu, bounded(&c.pdone[b], ((chunk - 1) / S::PB) & 1));
      }
      if (vote(bar, 128, bad)) {
        bad = true;
        break;
      }
      float* sums = reinterpret_cast<float*>(pbuf + wg * (S::NW / 8) * S::C * 16);   // the group's part of P's place
      spread<S::NC, S::C / 4>(l, [](float u, float v) { return u + v; });
#pragma unroll
      for (int j = 0; j < spread_left<S::NC, S::C / 4>(); ++j)
        sums[quarter * S::NW + col0 + spread_column<S::NC, S::C / 4>(j)] = l[j];
      named_bar_sync(bar, 128);
      const int slot = p.slot;
      float* acc = parts + (int64_t)slot * part_floats<S>();
      if (own < S::NW) {
        const float sum = (sums[own] + sums[S::NW + own]) + (sums[2 * S::NW + own] + sums[3 * S::NW + own]);
        alpha[own] = ref[own] == -INFINITY ? 0.f : 1.f / sum;
        if (slot >= 0) {
          float* ml = acc + S::N * S::DV + wg * S::NW + own;
          ml[0] = ref[own];
          ml[S::N] = sum;
        }
        // what the sums in the workspace are scaled by
        if (count > S::kFold) ref[own] = kept == ref[own] ? 1.f : ex2_approx(kept - ref[own]);
      }
      named_bar_sync(bar, 128);
      tc_fence_after();
      if (count > S::kFold) bring_back<S>(lanes + S::kO + wg * S::NW, fold, ref);
      const int mine_rows = min(S::NW, pairs - wg * S::NW);
      const bool has_dim = S::MO == 128 || lane < 16;
      const int dim0 = S::MO == 128 ? 32 * quarter + lane : 16 * quarter + (lane & 15);
      // out as pairs of dims: even lanes take one row of two, odd lanes the other
      T* out = static_cast<T*>(a.out) + (dim0 & ~1);
      const bool add = count > 0 && *unbounded != 0;
#pragma unroll 1
      for (int m = 0; m < S::DT; ++m)
#pragma unroll 1
        for (int r = 0; r < mine_rows; r += 16) {
          float o[16] = {};
          if (count > 0) {
            tmem_ld16(lanes + S::kO + m * S::N + wg * S::NW + r, o);
            tmem_ld_wait();
          }
          const int d = m * S::MO + dim0;
          if (add && has_dim) add_unbounded<S>(a, p, d, wg * S::NW + r, j0, o);
          if (slot >= 0) {
            if (has_dim) {
              float4* to = reinterpret_cast<float4*>(acc + d * S::N + wg * S::NW + r);
#pragma unroll
              for (int j = 0; j < 4; ++j) to[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            }
          } else {
            const bool odd = lane & 1;
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float2 f = *reinterpret_cast<const float2*>(alpha + r + j);
              const uint32_t w = pack(o[j] * f.x, o[j + 1] * f.y, T()), other = __shfl_xor_sync(0xffffffffu, w, 1);
              const int x = r + j + odd;
              if (has_dim && x < mine_rows)
                *reinterpret_cast<uint32_t*>(out + (int64_t)place[x] * S::DV + m * S::MO) =
                    __byte_perm(w, other, odd ? 0x3276 : 0x5410);
            }
          }
        }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.queue_empty[part % kQueue]);
    }
    gave_up = bad;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssuer) tmem_dealloc(tmem, S::kCols);
  if (gave_up) {   // a wait of this group gave up: NaN for its rows of the share
    const int wg = warp >> 2, own = tid & 127;
    float* const ml = parts + S::N * S::DV;
    Walk<S> walk(a, c.share);
    Part p;
    while (walk.next(p, nullptr)) {
      const uint32_t group = (uint32_t)a.group, t0 = (uint32_t)p.b.f0 / group, j0 = (uint32_t)p.b.f0 - t0 * group;
      for (int r = wg * S::NW; r < min((wg + 1) * S::NW, p.b.count); ++r) {
        if (p.slot >= 0) {
          if (own < 2) ml[(int64_t)p.slot * part_floats<S>() + own * S::N + r] = NAN;
        } else {
          const uint32_t rt = by_group(a, j0 + r);
          const int64_t row = (p.b.row0 + t0 + rt) * a.heads + (int64_t)p.head * a.group + (j0 + r - rt * group);
          for (int d = own; d < S::DV; d += 128) static_cast<T*>(a.out)[row * S::DV + d] = narrow(NAN, T());
        }
      }
    }
  }
}

// Joins the parts of the item that starts in CTA c's share and ends in another's: one block per (cut, 16 rows, 64 dims). A
// warp a row for the parts' weights, then a thread 4 rows of a dim, every kGroups-th part. The blocks past these write
// zeros for the rows that are no sequence's.
constexpr int kJoinRows = 16, kJoinDims = 64;
// GROUPS of 256 threads: 4 where the cuts are counted by item, which are few then and have many parts each, else one, and an
// SM holds several blocks. Four, with 64 registers a thread: held to 48 for a fifth the compiler spilled 40 bytes, and calls with
// many cuts were slower (64 sequences of 12 heads on one KV head 45.8 us, with four 43.8; window of 1024 64.0 and 61.7).
template <class S>
constexpr unsigned join_blocks(int cuts) {
  return (unsigned)cuts * (S::N / kJoinRows) * (S::DV / kJoinDims);
}
template <class S, int GROUPS>
__global__ void __launch_bounds__(256 * GROUPS, GROUPS == 4 ? 1 : 4)
    join_kernel(const __grid_constant__ Params a, int grid, unsigned blocks) {
  using T = typename S::T;
  constexpr int kGroups = GROUPS, kThreads = 256 * kGroups, kWarps = kThreads / 32;
  __shared__ __align__(16) float weight[kMaxGrid][kJoinRows];
  __shared__ float inv[kJoinRows];
  __shared__ float4 more[kGroups > 1 ? kGroups - 1 : 1][256];
  __shared__ __align__(16) T result[kJoinRows][kJoinDims];
  pdl_wait();
  pdl_launch_next();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (blockIdx.x >= blocks) {
    const int64_t first = row_bound(a, 0), last = row_bound(a, a.seqs), n = (int64_t)a.heads * S::DV / 8;
    for (int64_t i = blockIdx.x - blocks; i < first + (a.rows - last); i += gridDim.x - blocks) {
      uint4* to = reinterpret_cast<uint4*>(a.out) + (i < first ? i : last + (i - first)) * n;
      for (int64_t x = tid; x < n; x += kThreads) to[x] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const float* parts = a.work;
  constexpr int kRowTiles = S::N / kJoinRows, kTiles = kRowTiles * (S::DV / kJoinDims);
  const int which = blockIdx.x / kTiles, tile = blockIdx.x % kTiles, r0 = tile % kRowTiles * kJoinRows,
            d0 = tile / kRowTiles * kJoinDims;
  const Cut cut = reinterpret_cast<const Cut*>(parts + 2 * (int64_t)grid * part_floats<S>())[which];
  if (r0 >= cut.count) return;
  const int cta = cut.first, n = cut.last - cta / a.team + 1;
  auto part = [&](int i) { return parts + (int64_t)(i == 0 ? 2 * cta + 1 : 2 * (cta + i * a.team)) * part_floats<S>(); };
  const int group = tid / 256, dim = tid % 256 / 4, rows = tid % 4;
  const int at = (d0 + dim) * S::N + r0 + 4 * rows;
  constexpr int kAhead = kGroups == 4 ? 4 : 3;   // parts requested before their weights are known
  float4 ahead[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (group + k * kGroups < n) ahead[k] = *reinterpret_cast<const float4*>(part(group + k * kGroups) + at);
  // a row's weights; NaN where a wait gave up
  for (int row = warp; row < kJoinRows; row += kWarps) {
    float top = -INFINITY, sum0 = 0.f, total = 0.f;
    for (int i = lane; i < n; i += 32) {
      const float x = part(i)[S::N * S::DV + r0 + row];
      if (i < 32) sum0 = part(i)[S::N * (S::DV + 1) + r0 + row];
      weight[i][row] = x;
      top = max_nan(top, x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    for (int i = lane; i < n; i += 32) {
      const float x = weight[i][row], w = x == -INFINITY ? 0.f : x == top ? 1.f : ex2_approx(x - top);
      weight[i][row] = w;
      total = fmaf(w, i < 32 ? sum0 : part(i)[S::N * (S::DV + 1) + r0 + row], total);
    }
    total = warp_sum(total);
    if (lane == 0) inv[row] = top == -INFINITY ? 0.f : 1.f / total;
  }
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](int i, const float4& x) {
    const float4 w = *reinterpret_cast<const float4*>(&weight[i][4 * rows]);
    o.x = fmaf(w.x, x.x, o.x);
    o.y = fmaf(w.y, x.y, o.y);
    o.z = fmaf(w.z, x.z, o.z);
    o.w = fmaf(w.w, x.w, o.w);
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (group + k * kGroups < n) add(group + k * kGroups, ahead[k]);
#pragma unroll 8
  for (int i = group + kAhead * kGroups; i < n; i += kGroups) add(i, *reinterpret_cast<const float4*>(part(i) + at));
  if (group > 0) more[group - 1][tid % 256] = o;
  __syncthreads();
  if (group == 0) {
#pragma unroll
    for (int g = 1; g < kGroups; ++g) {
      const float4 x = more[g - 1][tid];
      o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
    }
    const float v[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float f = inv[4 * rows + j];
      result[4 * rows + j][dim] = narrow(f == 0.f ? 0.f : v[j] * f, T());
    }
  }
  __syncthreads();
  if (tid < kJoinRows * kJoinDims / 8) {
    const int r = tid / (kJoinDims / 8), u = tid % (kJoinDims / 8);
    if (r0 + r < cut.count) {
      const uint32_t pair = (uint32_t)cut.f0 + r0 + r;
      const int64_t t = cut.row0 + pair / (uint32_t)a.group, h = (int64_t)cut.head * a.group + pair % (uint32_t)a.group;
      *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (t * a.heads + h) * S::DV + d0 + 8 * u) =
          *reinterpret_cast<const uint4*>(&result[r][8 * u]);
    }
  }
}

}  // namespace kv16
}  // namespace xtg
