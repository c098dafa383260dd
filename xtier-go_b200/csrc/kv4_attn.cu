// Attention over the 4-bit paged cache (layout: kv4.h): every row sees the cached positions up to its own, the call's
// rows among them (they are stored first), and with a window only the last `window` of these.
//
//   o[r] = sum_p P[r][p] V[p] / sum_p P[r][p],  P[r][p] = 2^(S[r][p] - max_p S[r][p]),  S = log2(e) scale q[r] . K[p]
//
// with K and V as s (code - 8) + z per group of 64 head dims. Both products run on mma.m16n8k16 (f16 in, f32 out)
// straight from the codes, transposed, so that the few query rows are the instruction's 8 columns and no part of it is
// idle: S^T = K Q^T takes 16 slots x 16 dims of K, o^T = V^T P^T 16 dims x 16 slots of V. A lane then holds the scores
// of slots g, g + 8 and rows 2 a, 2 a + 1 (lane = 4 g + a); movmatrix turns the probabilities into the second
// product's operand. The scales and offsets enter in f32:
//   q . K[p] = sum_G s[p][G] (q . code)_G + (z[p][G] - 8 s[p][G]) (sum q)_G    (f32 rows: code - 8, and z alone)
//   o[r]     = sum_p (P[r][p] s[p][G]) (code - 8) + P[r][p] z[p][G]            (P s: the operand, by group G)
// K's codes enter as f16 subnormals, the nibble itself: code 2^-24 (bits 0-3) or code 2^-20 (bits 4-7), exact; q
// carries 1/16 where they lie at bits 4-7. V's are centred first (64 + c / 16 less 64.5): a sum of uncentred codes over
// positions would put an error of about 2^-20 of the group's range into components far smaller than it. So are K's for
// f32 rows, whose scores would lose about two bits to the part that cancels.
// Precision of the f16 operands: q of 16-bit rows is exact in one plane (a power of two brings the row's largest value
// to 2^14 .. 2^15); of f32 rows it is hi + lo, 22 bits. P s is brought below 2^16 by a power of two per group (the largest
// scale met) and always has two planes: one would put 2^-12 of the largest value into the result, which a small component
// beside large values of other positions shows even after bf16's rounding. The matrix unit's own sum loses about 2^-24 of
// itself per step to truncation, always towards zero. So f32 rows' P V is taken from zero for every half chunk and added
// to an f32 accumulator, and 16-bit rows' is added up in the unit for 128 steps at most (2^-18), then to f32 sums in
// shared memory. A row's maximum is followed loosely (kSlack): scaling the sums at every new maximum cost 10 % more
// instructions.
//
// One CTA per SM takes an equal share of all (sequence, KV head, row block, 64-position chunk) items in that order,
// whatever the sequences' lengths: shares start and end inside a sequence, whose parts a second kernel joins. Producer
// warps bring chunks (one bulk copy of a page's block of the head) into a ring of shared memory; the consumer warps take
// half chunks (32 positions) in turn, each with a running maximum of its own, so that no warp waits for another before
// the end of a sequence's part. A row block is 4, 8 or 16 rows held by every warp. 4 rows are 8 columns, the two planes
// of P s side by side, and half the work per lane; 16 rows share the unpacked codes. More rows read the chunks again,
// from L2 when the row blocks of a head run at the same time, which costs less than the products of 16 rows take, and
// larger blocks would cost more at every part's start and end (64 rows over 8192 positions: blocks of 128 rows 66 us,
// of 16 rows 52 us). A block's chunks are those that the sequence's rows see between them; those that its own rows do not
// see are brought and passed over. That is nothing for the rows of a step, half the chunks of a prompt from position 0
// (4096 rows 1.27 ms), and most of them for a prompt longer than its window (8192 rows, window 1024: 1.74 ms; in eight calls
// at most 1.14 ms).
//
// What bounds it (B200, head dim 128, bf16): with 4 rows about equally the cache's bytes and the instructions (1180 per
// chunk and head), 64 sequences of 16384 .. 32768 positions in 240 us, 5.6 TB/s, 86 % of a copy's rate (204 us without any
// computation), and in 280 us, 74 %, in runs of seconds, where the power limit lowers the clock; one sequence of 131072
// positions in 28 us, 4.1 TB/s, of which 10 us are the start, the end of the parts and the join. With 16 rows the
// instructions around the products: 64 rows over 8192 positions in 49 us, 132 TFLOP/s, tensor pipe 35 % and issue slots
// 55 % busy.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "kv4.h"

namespace xtg {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
// Looks at a barrier before a wait gives up. One that finds nothing takes 4 us (mbarrier.try_wait suspends the thread), so
// this is a second; no wait of the kernel begins before the kernels it depends on have ended.
constexpr uint32_t kKv4Polls = 1u << 18;
constexpr float kSlack = 6.f;   // how far, in powers of two, a row's probabilities may pass 1 before its sums are scaled
constexpr int kUnit = 32;                        // positions a warp takes at once: half a chunk
constexpr int kUnits = kKv4Page / kUnit, kSteps = kUnit / 16;
// Consumer warps and registers: a warpgroup of producers beside them, from which setmaxnreg moves registers to the
// consumers; the sum of both shares must not pass what the CTA started with (threads x kStart).
template <int D, int ROWS>
struct Kv4Shape {
  static constexpr int kWarps = ROWS <= 8 && D <= 128 ? 12 : 8;
  static constexpr int kThreads = 32 * (kWarps + 4);
  static constexpr int kStart = 65536 / kThreads / 8 * 8;
  static constexpr int kProducerRegs = 40;
  static constexpr int kConsumerRegs = (kThreads * kStart - 128 * kProducerRegs) / (32 * kWarps) / 8 * 8;
  static_assert(kWarps % 4 == 0, "setmaxnreg takes whole warpgroups");
  static_assert(32 * kWarps * kConsumerRegs + 128 * kProducerRegs <= kThreads * kStart, "more registers than launched");
  static constexpr int kBlock = kv4_block_bytes(D);
  // The ring: 110 to 166 KB. A stage's chunks are always brought by the same producer and its halves taken by the same
  // consumer warps. A wait tells the phases of a barrier apart by their parity only, so it must not start while the
  // phase before is open: a warp that waits for a stage's next chunk has itself seen the last one arrive.
  static constexpr int kStages = D == 256 ? 8 : D == 128 ? (ROWS == 16 ? 12 : 18) : 24;
  static constexpr int kProducers = kStages % 4 ? 3 : 4;
  static_assert(kUnits * kStages % kWarps == 0 && kStages % kProducers == 0, "a stage with several owners");
  static constexpr int kMergeStride = D + 4;   // floats of a row's accumulator being merged
};

template <int D, int ROWS>
struct Kv4Smem {
  using Shape = Kv4Shape<D, ROWS>;
  uint8_t stage[Shape::kStages][Shape::kBlock];
  float acc[Shape::kWarps][ROWS][Shape::kMergeStride];   // a part's end: the warps' accumulators
  // the part's rows as operands, [8-row tile][plane][32-dim block][lane] (held in registers they cost more in spills than
  // their loads do here: 1 x 8 f32 rows at 32768 37.0 -> 34.5 us, 16 x 8 f32 rows of head dim 256 148 -> 130 us)
  uint4 q[(ROWS == 16 ? 2 : 1) * 2 * (D / 32) * 32];
  float qsum[ROWS][D / kKv4Group], qfac[ROWS];   // what belongs to a row's scores
  int qpos[ROWS];
  float m[Shape::kWarps][ROWS], l[Shape::kWarps][ROWS];
  uint64_t full[Shape::kStages], empty[Shape::kStages];
  int present[Shape::kStages];   // 0: no page, nothing was copied
  uint64_t scan[Shape::kThreads / 32];
  uint64_t start_base;   // items before the sequence that the CTA's share starts in
  int start_seq;
  // A wait ran out. Its warp leaves the stage as it is (a copy may be on its way there) and takes no more; the producers,
  // who get no free stage, stop, and wait for the copies that they have issued before they end. The CTA's rows become NaN.
  int failed;
};

// A part of a sequence's items: row block b of KV head h, chunks c0 .. c0 + take - 1 of the sequence's cnt from page lo.
// Positions are below 2^31 (the table holds fewer).
struct Part {
  int seq, b, h, row0, n, pos, lo, cnt, c0, take;
  uint32_t blocks;   // of the sequence
};

// What the combine reads: the split (sequence, row block, head) that a CTA's share ends in, and the last CTA with a
// part of it.
struct Kv4Split {
  int row0, n, h, b, last;   // last < 0: none
};

__device__ __forceinline__ uint64_t divide(uint64_t a, uint32_t b) {
  return a >> 32 ? a / b : (uint32_t)a / b;
}

__device__ __forceinline__ uint64_t item_count(const Kv4Attn& a, const Part& p) {
  return (uint64_t)p.blocks * (uint32_t)a.w.kv_heads * (uint32_t)(p.cnt + a.part_cost);
}

// The items of sequence s: KV heads x row blocks x (part_cost + chunks). Sequences with rows have at least one chunk (it
// may hold nothing), so that every row is written.
template <int ROWS>
__device__ __forceinline__ uint64_t kv4_items(const Kv4Attn& a, int s, Part& p) {
  p.pos = a.w.pos[s];
  p.row0 = (int)kv4_row_bound(a.w, s);
  p.n = (int)kv4_row_bound(a.w, s + 1) - p.row0;
  if (p.n <= 0) return 0;
  p.seq = s;
  const int64_t held = (int64_t)a.w.max_pages * kKv4Page;
  int64_t end = (int64_t)p.pos + p.n;
  if (end > held) {   // rows past the table see what the table holds
    if (a.w.err) atomicExch(a.w.err, 6);
    end = held;
  }
  const int first = a.window > 0 && p.pos >= a.window ? p.pos - a.window + 1 : 0;
  p.lo = first / kKv4Page;
  p.cnt = max((int)((end + kKv4Page - 1) >> 6) - p.lo, 1);
  p.blocks = ((uint32_t)p.n * (uint32_t)a.group + ROWS - 1) / ROWS;
  return item_count(a, p);
}

// Walks a CTA's share of the items part by part.
struct Walk {
  int s;
  bool known;           // the Part given to the next step has sequence s's fields already
  uint64_t off, left;   // from sequence s's first item
};

template <int ROWS>
__device__ __forceinline__ bool kv4_next(const Kv4Attn& a, Walk& k, Part& p) {
  while (k.left > 0 && k.s < a.w.seqs) {
    const uint64_t items = k.known ? item_count(a, p) : kv4_items<ROWS>(a, k.s, p);
    k.known = false;
    if (k.off >= items) {
      k.off -= items;
      ++k.s;
      continue;
    }
    const uint64_t seg = divide(k.off, p.cnt + a.part_cost);
    const int at = (int)(k.off - seg * (uint32_t)(p.cnt + a.part_cost));
    const int skip = max(a.part_cost - at, 0);
    if (skip >= k.left) break;
    p.c0 = at + skip - a.part_cost;
    p.h = (int)divide(seg, p.blocks);
    p.b = (int)(seg - (uint64_t)p.h * p.blocks);
    k.left -= skip;
    p.take = (int)((uint64_t)(p.cnt - p.c0) < k.left ? (uint64_t)(p.cnt - p.c0) : k.left);
    k.off += skip + p.take;
    k.left -= p.take;
    return true;
  }
  return false;
}

// 8 neighbouring query values (16-byte aligned)
__device__ __forceinline__ void load_q8(const void* base, int64_t at, int dtype, float (&x)[8]) {
  if (dtype == kKv4F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 a = p[0], b = p[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    return;
  }
  const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == kKv4Bf16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// 4 neighbouring output values
__device__ __forceinline__ void store_out4(void* base, int64_t at, int dtype, float4 v) {
  if (dtype == kKv4F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = v;
  } else if (dtype == kKv4Bf16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) =
        make_uint2(pack_f16x2(v.x, v.y), pack_f16x2(v.z, v.w));
  }
}

// x = hi + lo in f16: two values' hi parts and lo parts, packed
__device__ __forceinline__ void split_f16x2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = pack_f16x2(x0, x1);
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  lo = pack_f16x2(x0 - h.x, x1 - h.y);
}

__device__ __forceinline__ uint32_t hfma2_u32(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hadd2_u32(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// (a & b) | c in one instruction: with two immediates the compiler takes two
template <uint32_t MASK>
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "n"(MASK), "r"(c));
  return r;
}

// The codes at bits 0-3 (low) or 4-7 (high) of a word's halves as (code - 8) 2^-4 in f16: 64 + c / 16 less 64.5, and
// (1024 + 16 c) / 256 less 4.5; exact. base: 64 (low) and 1024 (high) in both halves.
__device__ __forceinline__ uint32_t codes_low(uint32_t w, uint32_t base) {
  return hadd2_u32(and_or<0x000f000fu>(w, base), 0xd408d408u);
}
__device__ __forceinline__ uint32_t codes_high(uint32_t w, uint32_t base) {
  return hfma2_u32(and_or<0x00f000f0u>(w, base), 0x1c001c00u, 0xc480c480u);
}

// D = A B
__device__ __forceinline__ void mma_f16_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_f16(d, a[0], a[1], a[2], a[3], b0, b1);
}

// The transpose of an 8 x 8 matrix of 16-bit values (lane 4 g + a holds row g, columns 2 a and 2 a + 1)
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ float pow2_bits(int biased) { return __uint_as_float((uint32_t)biased << 23); }

__device__ __forceinline__ void kv4_give_up(int* failed, int32_t* err) {
  atomicExch(failed, 1);
  if (err) atomicExch(err, 1);
}

// mbarrier wait that gives up: after `polls` more looks than one, or after one once another wait of the CTA has. The lanes
// of a warp that wait together may come to different ends: a vote decides for all.
__device__ __forceinline__ bool kv4_wait(uint64_t* bar, uint32_t parity, uint32_t polls, int* failed, int32_t* err) {
  uint32_t spins = 0;
  while (!mbar_try_wait(bar, parity)) {
    ++spins;
    if (spins > polls || *reinterpret_cast<volatile int*>(failed)) {
      kv4_give_up(failed, err);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// floats of a part's row in the workspace: m, l, 2 pads, acc[D]
__host__ __device__ constexpr int part_row(int D) { return D + 4; }

// ROWS: of a row block, 4, 8 or 16; TYPE: q's and out's.
template <int D, int ROWS, int TYPE>
__global__ void __launch_bounds__(Kv4Shape<D, ROWS>::kThreads, 1)
    kv4_attention_kernel(const Kv4Attn a, float* part, Kv4Split* splits) {
  using Shape = Kv4Shape<D, ROWS>;
  constexpr int kStages = Shape::kStages, kWarps = Shape::kWarps, kThreads = Shape::kThreads;
  constexpr int kGroups = D / kKv4Group, kBlocks = D / 32, H = D < 128 ? D : 128;
  // 8-row tiles; with 4 rows a tile's columns are the two planes of a row (kPair), and a lane has one row of scores, not 2
  constexpr int RT = ROWS == 16 ? 2 : 1, kE = ROWS == 4 ? 1 : 2;
  constexpr bool kPair = ROWS == 4;
  constexpr int kQPlanes = TYPE == kKv4F32 && !kPair ? 2 : 1, kPPlanes = kPair ? 1 : 2;   // operands per tile
  constexpr bool kDirect = TYPE != kKv4F32;    // P V added up in the matrix unit, kFold half chunks at most
  constexpr int kFold = kPair ? 64 : 32;       // 128 products into a sum
  constexpr bool kCentred = TYPE == kKv4F32;   // K's codes less 8 before the product
  constexpr float kCode = kCentred ? 1.f / 16.f : 1.f / 16777216.f;   // the unit in which K's codes enter
  extern __shared__ __align__(128) unsigned char smem_raw[];
  Kv4Smem<D, ROWS>& sm = *reinterpret_cast<Kv4Smem<D, ROWS>*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, tq = lane & 3;

  if (threadIdx.x == 0) {
    for (int st = 0; st < kStages; ++st) {
      mbar_init(&sm.full[st], 1);
      mbar_init(&sm.empty[st], kUnits);
    }
    mbar_init_fence();
    sm.failed = 0;
    sm.start_seq = a.w.seqs;
    sm.start_base = 0;
  }
  pdl_wait();   // everything the call reads may come from the kernel before
  // ---- this CTA's share of the items: an equal part of their sum over the sequences ----
  // (a CTA's items fit 32 bits: 2^32 chunks would take it a quarter of an hour)
  uint64_t share = 0;
  uint32_t share_items = 0, most = 0, extra = 0;   // CTAs below `extra` have `most` + 1 items, the others `most`
  auto take_share = [&](uint64_t total) {
    // with fewer items than CTAs one each, so that no share between two others is empty
    const uint32_t ctas = total < gridDim.x ? (uint32_t)total : gridDim.x;
    if (blockIdx.x >= ctas) return;
    most = (uint32_t)divide(total, ctas);
    extra = (uint32_t)(total - (uint64_t)most * ctas);
    share = (uint64_t)most * blockIdx.x + min(blockIdx.x, extra);
    share_items = most + (blockIdx.x < extra);
  };
  auto warp_sum_to = [&](uint64_t x) {   // inclusive, over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  Walk walk = {};
  Part p;
  if (a.w.seqs <= 32) {   // every warp by itself, a sequence per lane
    const uint64_t mine = lane < a.w.seqs ? kv4_items<ROWS>(a, lane, p) : 0, x = warp_sum_to(mine);
    take_share(__shfl_sync(0xffffffffu, x, 31));
    // the lane whose sequence the share starts in (CTAs without items: any)
    const uint32_t at = __ballot_sync(0xffffffffu, x - mine <= share && share < x);
    const int from = at ? __ffs(at) - 1 : 0;
    walk = {from, true, share - __shfl_sync(0xffffffffu, x - mine, from), share_items};
    p.seq = from;
    p.row0 = __shfl_sync(0xffffffffu, p.row0, from);
    p.n = __shfl_sync(0xffffffffu, p.n, from);
    p.pos = __shfl_sync(0xffffffffu, p.pos, from);
    p.lo = __shfl_sync(0xffffffffu, p.lo, from);
    p.cnt = __shfl_sync(0xffffffffu, p.cnt, from);
    p.blocks = __shfl_sync(0xffffffffu, p.blocks, from);
    __syncthreads();
  } else {
    const bool one_pass = a.w.seqs <= kThreads;
    for (int pass = 0; pass < 2; ++pass) {   // the sum, then where the share starts
      uint64_t base = 0;
      for (int s0 = 0; s0 < a.w.seqs; s0 += kThreads) {
        const int s = s0 + threadIdx.x;
        const uint64_t mine = s < a.w.seqs ? kv4_items<ROWS>(a, s, p) : 0;
        uint64_t x = warp_sum_to(mine), sum = 0;
        if (lane == 31) sm.scan[warp] = x;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < kThreads / 32; ++v) {
          if (v < warp) x += sm.scan[v];
          sum += sm.scan[v];
        }
        if ((one_pass || pass == 0) && s0 + kThreads >= a.w.seqs) take_share(base + sum);
        if ((one_pass || pass == 1) && base + x - mine <= share && share < base + x) {
          sm.start_seq = s;
          sm.start_base = base + x - mine;
        }
        base += sum;
        __syncthreads();
      }
      if (one_pass) break;
    }
    walk = {sm.start_seq, false, share - sm.start_base, share_items};
  }

  if (warp >= kWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape::kProducerRegs));
    // ---- producers: chunk k of the parts in order is warp k % kProducers', a page's block of the head into stage
    // k % kStages; 32 chunks' pages are looked up at once ----
    constexpr int kProducers = Shape::kProducers;
    const int pw = warp - kWarps;
    if (pw >= kProducers) return;
    const uint64_t once = l2_evict_first();
    const int64_t page_bytes = (int64_t)a.w.kv_heads * Shape::kBlock;
    int st = pw, next = pw;   // this warp's next stage, and its next chunk of the part
    uint32_t turn = 0;
    bool ok = true;   // lane 0, which waits and copies: at once; the others: after 32 chunks
    while (ok && kv4_next<ROWS>(a, walk, p)) {
      const uint8_t* head = a.w.pool + (int64_t)p.h * Shape::kBlock;
      while (ok && next < p.take) {
        const int count = min((p.take - next + kProducers - 1) / kProducers, 32);
        const int64_t page = lane < count ? kv4_page(a.w, p.seq, p.lo + p.c0 + next + kProducers * lane) : -1;
        const uint64_t mine = page >= 0 ? reinterpret_cast<uint64_t>(head + page * page_bytes) : 0;
        for (int j = 0; j < count; ++j) {
          const void* from = reinterpret_cast<const void*>(__shfl_sync(0xffffffffu, mine, j));
          if (lane == 0 && turn > 0 && ok) ok = kv4_wait(&sm.empty[st], (turn - 1) & 1, a.polls, &sm.failed, a.w.err);
          if (lane == 0 && ok) {
            sm.present[st] = from != nullptr;
            if (!from) {
              mbar_arrive(&sm.full[st]);
            } else {
              mbar_expect_tx(&sm.full[st], Shape::kBlock);
              if (p.blocks == 1)   // read once: the first to leave L2
                bulk_g2s_hint(sm.stage[st], from, Shape::kBlock, &sm.full[st], once);
              else
                bulk_g2s(sm.stage[st], from, Shape::kBlock, &sm.full[st]);
            }
          }
          __syncwarp();
          if (ok) st += kProducers;
          if (st >= kStages) {
            st -= kStages;
            ++turn;
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        next += count * kProducers;
      }
      next -= p.take;
    }
    pdl_launch_next();
    // no copy may outlive the CTA: the consumers have seen all of them arrive, unless a wait ran out
    if (lane == 0)
      for (int s = pw; s < kStages; s += kProducers) {
        const uint32_t issued = turn + (s < st);   // into this stage
        uint32_t i = 0;
        while (issued > 0 && !mbar_try_wait(&sm.full[s], (issued - 1) & 1) && ++i < kKv4Polls) continue;
        if (i == kKv4Polls && a.w.err) atomicExch(a.w.err, 1);
      }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Shape::kConsumerRegs));
    const uint32_t group = a.group;
    uint32_t base_low, base_high;   // kept in registers (codes_low)
    asm volatile("mov.b32 %0, 0x54005400;" : "=r"(base_low));
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(base_high));
    // chunks of the parts before; once a wait of this warp gave up, from kGivenUp on: it no longer knows the ring's phases
    uint32_t it = 0;
    constexpr uint32_t kGivenUp = 1u << 31;
    bool split_after = false;   // the last part goes on in the next CTA
    int x = 0;                  // this warp's next half chunk of the part
    bool more = false;          // the part goes on, its sums so far are in shared memory
    while (more || kv4_next<ROWS>(a, walk, p)) {
      // ---- the rows: row r of the sequence and KV head is (row r / group of the sequence, q head r % group) ----
      const uint32_t qrows = (uint32_t)p.n * group, r0 = (uint32_t)p.b * ROWS;
      // the position of the sequence's row i (past 2^31 - 1 the table holds nothing more to see)
      auto position = [&](uint32_t i) { return (int)min((int64_t)p.pos + i, (int64_t)0x7fffffff); };
      // the block's first position (below 0 nothing is seen) and last
      const int tmin = max(position(r0 / group), -1), tmax = position((min(r0 + ROWS, qrows) - 1) / group);

      // ---- Q as the first product's operand for every row of the block, by all consumer warps: a thread takes 8
      // neighbouring dims, the word of K codes that lane 4 g + (dims / 8) % 4 multiplies: nibble pair i (dims i, i + 4)
      // is a register of step i / 2 ----
      constexpr int kPieces = D / 8;   // threads per row
      const int pieces = more ? 0 : ROWS * kPieces;
      for (int x = threadIdx.x; x < pieces; x += 32 * kWarps) {   // whole warps: ROWS x D / 8 >= 32
        const int row = x / kPieces, d8 = x % kPieces;
        const uint32_t r = r0 + row, i = r / group;
        const bool live = r < qrows;
        float v[8] = {};
        if (live)
          load_q8(a.q, ((int64_t)p.row0 + i) * a.q_row + (int64_t)(p.h * group + (r - i * group)) * a.q_head + 8 * d8, TYPE,
                  v);
        float mx = 0.f, sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(v[e]));
#pragma unroll
        for (int o = 1; o < kPieces; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const int e2 = min(max((int)(__float_as_uint(mx) >> 23), 16), 254);   // biased exponent of the largest value
        // the factor is not negative (a maximum of scores stays one): a negative scale turns q's sign
        const float up = a.scale < 0.f ? -pow2_bits(min(268 - e2, 254)) : pow2_bits(min(268 - e2, 254));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] *= up;
          sum += v[e];
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);   // the group's 8 threads
        uint32_t hi[4], lo[4] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = e % 2 && !kCentred ? 0.0625f : 1.f;   // codes at bits 4-7 stand for 16 times the others
          if constexpr (TYPE == kKv4F32)
            split_f16x2(v[e] * f, v[e + 4] * f, hi[e], lo[e]);
          else
            hi[e] = pack_f16x2(v[e] * f, v[e + 4] * f);
        }
        const int column = kPair ? 2 * row : row % 8;
        const int at = (row / 8 * kQPlanes * kBlocks + d8 / 4) * 32 + 4 * column + d8 % 4;
        sm.q[at] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if constexpr (kPair || kQPlanes == 2) sm.q[at + (kPair ? 4 : kBlocks * 32)] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if (d8 % 8 == 0) sm.qsum[row][d8 / 8] = sum * kCode;
        if (d8 == 0) {
          sm.qfac[row] = fmaxf(fabsf(a.scale) / fabsf(up) * (kLog2e / kCode), 1.1754944e-38f);
          sm.qpos[row] = live ? position(i) : -1;
        }
      }
      if (!more) named_bar_sync(1, 32 * kWarps);
      // what belongs to the rows of this lane's scores: 8 j + 2 tq + {0, 1}, or tq
      float qsum[RT][kE][kGroups], rf[RT][kE];   // (sum q)_G and the factor from the products' unit to base-2 scores
      int t[RT][kE];                             // the row's position; dead rows see nothing
#pragma unroll
      for (int j = 0; j < RT; ++j) {
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const int row = 8 * j + kE * tq + e;
          rf[j][e] = sm.qfac[row];
          t[j][e] = sm.qpos[row];
#pragma unroll
          for (int G = 0; G < kGroups; ++G) qsum[j][e][G] = sm.qsum[row][G];
        }
      }

      // dims 32 c + 16 m + g (+ 8: the last two) of columns 2 tq + {0, 1}, without the offsets' part
      float o[RT][kBlocks][2][4];
      float oz[RT][kE][kGroups];   // sum of P z over this lane's slots
      float ref[RT][kE], run_l[RT][kE];
      int unit_e[kGroups];   // P s 2^(136 - unit_e) is below 2^16
#pragma unroll
      for (int j = 0; j < RT; ++j) {
#pragma unroll
        for (int c = 0; c < kBlocks; ++c)
#pragma unroll
          for (int m = 0; m < 2; ++m) o[j][c][m][0] = o[j][c][m][1] = o[j][c][m][2] = o[j][c][m][3] = 0.f;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          ref[j][e] = more ? sm.m[warp][8 * j + kE * tq + e] : -INFINITY;
          run_l[j][e] = 0.f;
#pragma unroll
          for (int G = 0; G < kGroups; ++G) oz[j][e][G] = 0.f;
        }
      }
#pragma unroll
      for (int G = 0; G < kGroups; ++G) unit_e[G] = 27;

      // half chunk hh of a stage, its first position p0
      auto unit = [&](const uint8_t* stg, int hh, int p0, bool masked) {
        const uint32_t* kw = reinterpret_cast<const uint32_t*>(stg) + hh * kUnit * (H / 8);
        const uint32_t* kpar = reinterpret_cast<const uint32_t*>(stg + kv4_k_params(D)) + hh * kUnit;
        const uint32_t* vw = reinterpret_cast<const uint32_t*>(stg + kv4_v_codes(D)) + hh * kUnit * (D / 8);
        const uint32_t* vpar = reinterpret_cast<const uint32_t*>(stg + kv4_v_params(D)) + hh * kUnit;
        // ---- scores of 16 slots each: slot 16 u + g of the lane's kE rows, then slot 16 u + 8 + g ----
        float s[RT][kSteps][2 * kE];
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
          float c[RT][kGroups][4];
#pragma unroll
          for (int hf = 0; hf < D / H; ++hf) {
            uint32_t w[2][H / 32];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int slot = 16 * u + 8 * e + g;
              if constexpr (H == 128) {
                const uint4 v = *reinterpret_cast<const uint4*>(kw + ((hf * kKv4Page + slot) * 4 + tq) * 4);
                w[e][0] = v.x, w[e][1] = v.y, w[e][2] = v.z, w[e][3] = v.w;
              } else {
                const uint2 v = *reinterpret_cast<const uint2*>(kw + (slot * 4 + tq) * 2);
                w[e][0] = v.x, w[e][1] = v.y;
              }
            }
#pragma unroll
            for (int b = 0; b < H / 32; ++b) {
              const int blk = hf * (H / 32) + b, G = blk / 2;
              uint4 q[RT][kQPlanes];
#pragma unroll
              for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int pl = 0; pl < kQPlanes; ++pl) q[j][pl] = sm.q[((j * kQPlanes + pl) * kBlocks + blk) * 32 + lane];
#pragma unroll
              for (int st = 0; st < 2; ++st) {
                const uint32_t w0 = st ? w[0][b] >> 8 : w[0][b], w1 = st ? w[1][b] >> 8 : w[1][b];
                uint32_t ka[4] = {w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u};
                if constexpr (kCentred) {
                  ka[0] = codes_low(w0, base_low), ka[1] = codes_low(w1, base_low);
                  ka[2] = codes_high(w0, base_high), ka[3] = codes_high(w1, base_high);
                }
#pragma unroll
                for (int j = 0; j < RT; ++j) {
#pragma unroll
                  for (int pl = 0; pl < kQPlanes; ++pl) {
                    const uint32_t b0 = st ? q[j][pl].z : q[j][pl].x, b1 = st ? q[j][pl].w : q[j][pl].y;
                    if (blk % 2 == 0 && st == 0 && pl == 0)
                      mma_f16_new(c[j][G], ka, b0, b1);
                    else
                      mma_f16_add(c[j][G], ka, b0, b1);
                  }
                }
              }
            }
          }
#pragma unroll
          for (int G = 0; G < kGroups; ++G) {
            const uint32_t w0 = kpar[G * kKv4Page + 16 * u + g], w1 = kpar[G * kKv4Page + 16 * u + 8 + g];
            const float s0 = __uint_as_float(w0 & 0xffff0000u), s1 = __uint_as_float(w1 & 0xffff0000u);
            constexpr float kLess = kCentred ? 0.f : -8.f;
            const float z0 = fmaf(kLess, s0, __uint_as_float(w0 << 16)), z1 = fmaf(kLess, s1, __uint_as_float(w1 << 16));
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
              for (int e = 0; e < 2 * kE; ++e) {
                const float sc = e < kE ? s0 : s1, of = e < kE ? z0 : z1, q1 = qsum[j][e % kE][G];
                float dot = c[j][G][kPair ? 2 * e : e];
                if constexpr (kPair && TYPE == kKv4F32) dot += c[j][G][2 * e + 1];
                s[j][u][e] = fmaf(sc, dot, G == 0 ? of * q1 : fmaf(of, q1, s[j][u][e]));
              }
          }
        }
        // ---- V's parameters, slots 8 i + g ----
        uint32_t w[kGroups][2 * kSteps];
#pragma unroll
        for (int G = 0; G < kGroups; ++G)
#pragma unroll
          for (int i = 0; i < 2 * kSteps; ++i) w[G][i] = vpar[G * kKv4Page + 8 * i + g];
        if (masked) {
          // a row does not see every slot: -inf for its score; what no row sees may hold anything
#pragma unroll
          for (int i = 0; i < 2 * kSteps; ++i) {
            const int pp = p0 + 8 * i + g;
            const bool none = pp > tmax || (a.window > 0 && pp <= tmin - a.window);
            bool sees[RT][kE];
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
              for (int e = 0; e < kE; ++e) {
                sees[j][e] = pp <= t[j][e] && (a.window <= 0 || pp > t[j][e] - a.window);
                if (!sees[j][e]) s[j][i / 2][kE * (i % 2) + e] = -INFINITY;
              }
#pragma unroll
            for (int G = 0; G < kGroups; ++G) {
              if (none) w[G][i] = 0;
              if ((int)w[G][i] < 0) {   // a NaN scale must not meet a probability of 0: into the sums of those that see it
                w[G][i] = 0;
#pragma unroll
                for (int j = 0; j < RT; ++j)
#pragma unroll
                  for (int e = 0; e < kE; ++e)
                    if (sees[j][e]) oz[j][e][G] = __uint_as_float(0x7fc00000u);
              }
            }
          }
        }
        // the scales' largest exponent per group: positive f32 order is integer order, NaN's word is negative
        bool move = false;
        int next_e[kGroups];
#pragma unroll
        for (int G = 0; G < kGroups; ++G) {
          int top = 0;
#pragma unroll
          for (int i = 0; i < 2 * kSteps; ++i) top = max(top, (int)w[G][i]);
          next_e[G] = top >> 23;
          move |= next_e[G] > unit_e[G];
        }
        // ---- the rows' references: a row's probabilities are 2^(score - ref), at most 2^kSlack; a reference (and V's
        // exponent) moves up when a maximum passes it by more, and then the sums are scaled ----
        float mx[RT][kE];
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            float m = fmaxf(s[j][0][e], s[j][0][e + kE]);
#pragma unroll
            for (int u = 1; u < kSteps; ++u) m = fmaxf(m, fmaxf(s[j][u][e], s[j][u][e + kE]));
            mx[j][e] = m * rf[j][e];
            move |= mx[j][e] > ref[j][e] + kSlack;
          }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int G = 0; G < kGroups; ++G) {
            int e2 = min(max(next_e[G], unit_e[G]), 254);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) e2 = max(e2, __shfl_xor_sync(0xffffffffu, e2, x));
            next_e[G] = e2;
          }
#pragma unroll
          for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int e = 0; e < kE; ++e) {
              float m = fmaxf(mx[j][e], ref[j][e]);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
              const float alpha = m == ref[j][e] ? 1.f : ex2_approx(ref[j][e] - m);
              ref[j][e] = m;
              run_l[j][e] *= alpha;
#pragma unroll
              for (int G = 0; G < kGroups; ++G) {
                oz[j][e][G] *= alpha;
                const float f = kDirect ? alpha * ex2_approx((float)(unit_e[G] - next_e[G])) : alpha;
#pragma unroll
                for (int c = 2 * G; c < 2 * G + 2; ++c)
#pragma unroll
                  for (int m2 = 0; m2 < 2; ++m2)
#pragma unroll
                    for (int x = kPair ? 0 : e; x < 4; x += kPair ? 1 : 2) o[j][c][m2][x] *= f;
              }
            }
#pragma unroll
          for (int G = 0; G < kGroups; ++G) unit_e[G] = next_e[G];
        }
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const float r = ref[j][e] == -INFINITY ? 0.f : ref[j][e];
#pragma unroll
            for (int u = 0; u < kSteps; ++u) {
              s[j][u][e] = ex2_approx(fmaf(s[j][u][e], rf[j][e], -r));
              s[j][u][e + kE] = ex2_approx(fmaf(s[j][u][e + kE], rf[j][e], -r));
              run_l[j][e] += s[j][u][e] + s[j][u][e + kE];
            }
          }
        // ---- P V by group of 64 dims ----
#pragma unroll
        for (int G = 0; G < kGroups; ++G) {
          const float down = pow2_bits(136 + 127 - unit_e[G]), up = pow2_bits(unit_e[G] - 9) * 16.f;
          uint32_t pb[RT][kPPlanes][2 * kSteps];
#pragma unroll
          for (int i = 0; i < 2 * kSteps; ++i) {
            const float sc = __uint_as_float(w[G][i] & 0xffff0000u) * down;
            const float of = __uint_as_float(w[G][i] << 16);
#pragma unroll
            for (int j = 0; j < RT; ++j) {
              // hi: the leading 11 bits (cut, so that an AND gives them), lo: the next 11
              float hi[kE], lo[kE];
#pragma unroll
              for (int e = 0; e < kE; ++e) {
                const float pr = s[j][i / 2][kE * (i % 2) + e], x = pr * sc;
                hi[e] = __uint_as_float(__float_as_uint(x) & 0xffffe000u);
                lo[e] = x - hi[e];
                oz[j][e][G] = fmaf(pr, of, oz[j][e][G]);
              }
              if constexpr (kPair) {
                pb[j][0][i] = transpose8(pack_f16x2(hi[0], lo[0]));
              } else {
                pb[j][0][i] = transpose8(pack_f16x2(hi[0], hi[kE - 1]));
                pb[j][kPPlanes - 1][i] = transpose8(pack_f16x2(lo[0], lo[kE - 1]));
              }
            }
          }
#pragma unroll
          for (int c = 2 * G; c < 2 * G + 2; ++c) {
            float d[RT][2][4];
            const uint4 v = *reinterpret_cast<const uint4*>(vw + ((c * 8 + g) * 4 + tq) * 4);
            const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int st = 0; st < 2; ++st) {
                const uint32_t w0 = st ? word[2 * m] >> 8 : word[2 * m], w1 = st ? word[2 * m + 1] >> 8 : word[2 * m + 1];
                const uint32_t va[4] = {codes_low(w0, base_low), codes_low(w1, base_low), codes_high(w0, base_high),
                                        codes_high(w1, base_high)};
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                  float(&to)[4] = kDirect ? o[j][c][m] : d[j][m];
#pragma unroll
                  for (int pl = 0; pl < kPPlanes; ++pl) {
                    if (!kDirect && st == 0 && pl == 0)
                      mma_f16_new(to, va, pb[j][pl][0], pb[j][pl][1]);
                    else
                      mma_f16_add(to, va, pb[j][pl][2 * st], pb[j][pl][2 * st + 1]);
                  }
                }
              }
            if constexpr (!kDirect)
#pragma unroll
              for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[j][c][m][e] = fmaf(d[j][m][e], up, o[j][c][m][e]);
          }
        }
      };

      // ---- this warp's half chunks of the part: every kWarps-th of the CTA's ----
      // Half chunk x is chunk x / kUnits, in the ring's stage and turn after `it` chunks; kWarps is a multiple of kUnits, so
      // a warp's half of the chunks stays the same.
      static_assert(kWarps % kUnits == 0 && kWarps / kUnits <= kStages, "the ring goes round once between a warp's chunks at most");
      if (!more) x = (int)((warp + kWarps - kUnits * it % kWarps) % kWarps);
      if (a.polls == 0) kv4_give_up(&sm.failed, a.w.err);   // without a look, and with copies under way
      const int hh = x % kUnits;
      const uint32_t k0 = it + x / kUnits;
      uint32_t st = k0 % kStages, turn = k0 / kStages;
      // units from seen_from + 1 to tmax hold a position that some row sees, those from full_from + 1 to full_to only such
      // that every row sees
      const int seen_from = a.window > 0 ? tmin - a.window - (kUnit - 1) : -kUnit;
      const int full_from = a.window > 0 ? tmax - a.window : -kUnit, full_to = tmin - (kUnit - 1);
      const int units = it < kGivenUp ? kUnits * p.take : 0;
      const int stop = kDirect ? min(units, x + kFold * kWarps) : units;
      bool ok = true;
      for (int p0 = (p.lo + p.c0) * kKv4Page + kUnit * x; x < stop; x += kWarps, p0 += kUnit * kWarps) {
        // the first look apart: with one vote, behind the loop of looks, 8-row blocks took 3 % longer
        if (!__all_sync(0xffffffffu, mbar_try_wait(&sm.full[st], turn & 1))) {
          ok = __all_sync(0xffffffffu, kv4_wait(&sm.full[st], turn & 1, a.polls, &sm.failed, a.w.err));
          if (!ok) break;
        }
        if (sm.present[st] && p0 <= tmax && p0 > seen_from) unit(sm.stage[st], hh, p0, p0 > full_to || p0 <= full_from);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[st]);
        st += kWarps / kUnits;
        if (st >= kStages) {
          st -= kStages;
          ++turn;
        }
      }

      // ---- the warp's sums into shared memory, with those of its half chunks before, which a lane finds in its own places
      // (added apart from the last lines: there, even where it does not happen, it cost 3 %) ----
      float up[kGroups];
#pragma unroll
      for (int G = 0; G < kGroups; ++G) up[G] = kDirect ? pow2_bits(unit_e[G] - 9) * 16.f : 1.f;
      if (kDirect && more) {
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const int row = 8 * j + kE * tq + e;
            const float m = sm.m[warp][row], old = m == ref[j][e] ? 1.f : ex2_approx(m - ref[j][e]);
            if (g == 0) run_l[j][e] = fmaf(old, sm.l[warp][row], run_l[j][e]);
#pragma unroll
            for (int c = 0; c < kBlocks; ++c)
#pragma unroll
              for (int i = 0; i < 4; ++i) {   // dims 8 i + g of the block
                float* y = &o[j][c][i / 2][2 * (i % 2)];
                y[kPair ? 0 : e] =
                    fmaf(old, sm.acc[warp][row][32 * c + 8 * i + g], (kPair ? y[0] + y[1] : y[e]) * up[c / 2]);
                if (kPair) y[1] = 0.f;
              }
          }
#pragma unroll
        for (int G = 0; G < kGroups; ++G) up[G] = 1.f;
        __syncwarp();
      }
#pragma unroll
      for (int j = 0; j < RT; ++j)
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const int row = 8 * j + kE * tq + e;
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            run_l[j][e] += __shfl_xor_sync(0xffffffffu, run_l[j][e], x);
#pragma unroll
            for (int G = 0; G < kGroups; ++G) oz[j][e][G] += __shfl_xor_sync(0xffffffffu, oz[j][e][G], x);
          }
          if (g == 0) {
            sm.m[warp][row] = ref[j][e];
            sm.l[warp][row] = run_l[j][e];
          }
#pragma unroll
          for (int c = 0; c < kBlocks; ++c)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const float(&y)[4] = o[j][c][m];
              float* to = &sm.acc[warp][row][32 * c + 16 * m + g];
              to[0] = fmaf(kPair ? y[0] + y[1] : y[e], up[c / 2], oz[j][e][c / 2]);
              to[8] = fmaf(kPair ? y[2] + y[3] : y[e + 2], up[c / 2], oz[j][e][c / 2]);
            }
        }
      if (!ok) it = kGivenUp;
      more = kDirect && ok && x < units;
      if (more) {   // the same part and rows: no other warp is waited for
        __syncwarp();
        continue;
      }
      it += p.take;

      // ---- the part's warps meet, by their maxima ----
      // the next part's rows may now be staged; its accumulators are written after the barrier that follows them
      named_bar_sync(1, 32 * kWarps);
      const bool whole = p.c0 == 0 && p.take == p.cnt;
      const float none = *reinterpret_cast<volatile int*>(&sm.failed) ? __uint_as_float(0x7fc00000u) : 0.f;
      float* mine = part + (int64_t)(2 * blockIdx.x + (p.c0 == 0 ? 1 : 0)) * ROWS * part_row(D);
      constexpr int kQuads = D / 4;   // threads per row
      for (int x = threadIdx.x; x < ROWS * kQuads; x += 32 * kWarps) {
        const int row = x / kQuads, d0 = 4 * (x % kQuads);
        const uint32_t rr = r0 + row;
        if (rr >= qrows) break;
        float mv[kWarps], M = -INFINITY, l = none;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int v = 0; v < kWarps; ++v) {
          mv[v] = sm.m[v][row];
          M = fmaxf(M, mv[v]);
        }
#pragma unroll
        for (int v = 0; v < kWarps; ++v) {
          const float wt = mv[v] == M ? 1.f : ex2_approx(mv[v] - M);
          const float4 u = *reinterpret_cast<const float4*>(&sm.acc[v][row][d0]);
          l = fmaf(wt, sm.l[v][row], l);
          y.x = fmaf(wt, u.x, y.x);
          y.y = fmaf(wt, u.y, y.y);
          y.z = fmaf(wt, u.z, y.z);
          y.w = fmaf(wt, u.w, y.w);
        }
        if (whole) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          const uint32_t i = rr / group;
          store_out4(a.out, (((int64_t)p.row0 + i) * a.heads + p.h * group + (rr - i * group)) * D + d0, TYPE,
                     make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
        } else {
          float* to = mine + (int64_t)row * part_row(D);
          *reinterpret_cast<float4*>(to + 4 + d0) = y;
          if (d0 == 0) *reinterpret_cast<float2*>(to) = make_float2(M, l);
        }
      }
      split_after = p.c0 == 0 && !whole;
      if (split_after && threadIdx.x == 0) {
        // the last item of this (sequence, row block, head), and the CTA whose share holds it
        const uint64_t end = share + share_items - p.take + p.cnt - 1, longer = (uint64_t)extra * (most + 1);
        splits[blockIdx.x] = {p.row0, p.n, p.h, p.b,
                              (int)(end < longer ? divide(end, most + 1) : extra + divide(end - longer, most))};
      }
    }
    if (threadIdx.x == 0 && !split_after) splits[blockIdx.x].last = -1;
  }
  pdl_launch_next();
}

// Row blockIdx.x % ROWS of the split (sequence, row block, KV head), if any, that CTA blockIdx.x / ROWS's share ended
// in: the last part of that CTA and the first parts of the CTAs after it, joined by their maxima. D / 4 threads take 4
// dims each of every kSets-th part; the sets' results are joined in their order. Blocks from sms x ROWS on write the zeros
// of rows that are no sequence's.
constexpr int kCombineThreads = 256;

template <int D, int ROWS>
__global__ void __launch_bounds__(kCombineThreads)
    kv4_combine_kernel(const Kv4Attn a, const float* part, const Kv4Split* splits, int sms) {
  constexpr int kQuads = D / 4, kSets = kCombineThreads / kQuads;   // 4, 8 or 16 sets of threads
  __shared__ __align__(16) float acc[kSets][D];
  __shared__ float sm_m[kSets], sm_l[kSets];
  pdl_wait();
  pdl_launch_next();
  const int first = blockIdx.x / ROWS, row = blockIdx.x % ROWS;
  if (first >= sms) {
    kv4_zero_rest(a.w, a.out, nullptr, (int64_t)a.heads * D * (a.dtype == kKv4F32 ? 4 : 2), sms * ROWS);
    return;
  }
  const Kv4Split sp = splits[first];
  const uint32_t group = a.group, rr = (uint32_t)sp.b * ROWS + row;
  if (sp.last < 0 || rr >= (uint32_t)sp.n * group) return;
  const int set = threadIdx.x / kQuads, d0 = 4 * (threadIdx.x % kQuads), parts = sp.last - first + 1;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = -INFINITY, l = 0.f;
  auto join = [&](float m, float add_l, const float4& u) {
    const float top = fmaxf(M, m);
    const float old = M == top ? 1.f : ex2_approx(M - top), add = m == top ? 1.f : ex2_approx(m - top);
    M = top;
    l = fmaf(add, add_l, l * old);
    y.x = fmaf(add, u.x, y.x * old);
    y.y = fmaf(add, u.y, y.y * old);
    y.z = fmaf(add, u.z, y.z * old);
    y.w = fmaf(add, u.w, y.w * old);
  };
#pragma unroll 4
  for (int k = set; k < parts; k += kSets) {
    const float* from = part + ((int64_t)(2 * (first + k) + (k == 0 ? 1 : 0)) * ROWS + row) * part_row(D);
    const float2 ml = *reinterpret_cast<const float2*>(from);
    join(ml.x, ml.y, *reinterpret_cast<const float4*>(from + 4 + d0));
  }
  *reinterpret_cast<float4*>(&acc[set][d0]) = y;
  if (d0 == 0) {
    sm_m[set] = M;
    sm_l[set] = l;
  }
  __syncthreads();
  if (set != 0) return;
#pragma unroll
  for (int v = 1; v < kSets; ++v) join(sm_m[v], sm_l[v], *reinterpret_cast<const float4*>(&acc[v][d0]));
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const uint32_t i = rr / group;
  store_out4(a.out, (((int64_t)sp.row0 + i) * a.heads + sp.h * group + (rr - i * group)) * D + d0, a.dtype,
             make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
}

// Rows of a row block: as many as a sequence has, 4, 8 or 16 (head dim 256 has no registers for 16).
int block_rows(int head_dim, int group, int rows_per_seq) {
  const int64_t rows = (int64_t)group * rows_per_seq;
  return rows <= 4 ? 4 : rows <= 8 || head_dim == 256 ? 8 : 16;
}

template <int D, int ROWS, int TYPE>
void launch(const Kv4Attn& a, int sms, cudaStream_t s) {
  float* part = a.part;
  Kv4Split* splits = reinterpret_cast<Kv4Split*>(part + (int64_t)sms * 2 * ROWS * part_row(D));
  static std::atomic<uint64_t> optin;
  const int smem = (int)sizeof(Kv4Smem<D, ROWS>);
  ensure_smem_optin((const void*)kv4_attention_kernel<D, ROWS, TYPE>, smem, optin);
  // setmaxnreg would wait forever in a kernel that starts with fewer registers than its shares were worked out for
  static const bool enough = [] {
    cudaFuncAttributes f;
    XTG_CUDA(cudaFuncGetAttributes(&f, (const void*)kv4_attention_kernel<D, ROWS, TYPE>));
    return f.numRegs >= Kv4Shape<D, ROWS>::kStart;
  }();
  XTG_REQUIRE(enough, "kv4: the attention kernel was compiled to fewer registers than it shares out");
  launch_kv4(kv4_attention_kernel<D, ROWS, TYPE>, sms, Kv4Shape<D, ROWS>::kThreads, smem, s, a, part, splits);
  launch_kv4(kv4_combine_kernel<D, ROWS>, sms * ROWS + kv4_rest_blocks(a.w), kCombineThreads, 0, s, a, (const float*)part,
             (const Kv4Split*)splits, sms);
}

template <int D, int ROWS>
void launch_type(const Kv4Attn& a, int sms, cudaStream_t s) {
  if (a.dtype == kKv4F32)
    launch<D, ROWS, kKv4F32>(a, sms, s);
  else if (a.dtype == kKv4Bf16)
    launch<D, ROWS, kKv4Bf16>(a, sms, s);
  else
    launch<D, ROWS, kKv4F16>(a, sms, s);
}

template <int D>
void launch_rows(const Kv4Attn& a, int rows, int sms, cudaStream_t s) {
  if (rows == 4)
    launch_type<D, 4>(a, sms, s);
  else if (D == 256 || rows == 8)
    launch_type<D, 8>(a, sms, s);
  else
    launch_type<D, D == 256 ? 8 : 16>(a, sms, s);
}

}  // namespace

namespace {
std::atomic<uint32_t> wait_polls{kKv4Polls};
}

int kv4_wait_polls(int polls) {
  return (int)(polls < 0 ? wait_polls.load() : wait_polls.exchange(std::min((uint32_t)polls, 1u << 24)));
}

int64_t kv4_workspace_bytes(int head_dim, int group, int rows_per_seq, int sms) {
  return (int64_t)sms * (2 * block_rows(head_dim, group, rows_per_seq) * part_row(head_dim) * (int64_t)sizeof(float) +
                         (int64_t)sizeof(Kv4Split));
}

void launch_kv4_attention(const Kv4Attn& args, int sms, cudaStream_t s) {
  Kv4Attn a = args;
  const int rows = block_rows(a.w.head_dim, a.group, a.rows_per_seq);
  // What the start of another part costs a CTA (its rows, its sums), in chunks: counted as items before the part's first,
  // so that a CTA with several parts gets fewer chunks, and few sequences' parts go to CTAs of their own. Measured at 4,
  // 8, 12, 16: 4 rows: 1 x 131072 29.2, 28.5, 27.7, 27.9 us, 512 x 2048 188, 184, 182, 182, 64 x 4096 of head dim 64, 8 q
  // on 8 KV heads 42.8, 42.5, 41.1, 40.4; others: 64 rows x 8192 49.5, 49.2, 49.4, 50.5, 12 rows x 8192 of 64 sequences
  // 31.8, 30.9, 30.7, 31.6, 16 x 8191 at head dim 256 35.6, 34.9, 35.8, 36.3 us.
  a.polls = wait_polls.load(std::memory_order_relaxed);
  a.window = std::min(a.window, 0x7fffffff - 63);   // all positions, and no overflow of -1 - window - 31
  a.part_cost = rows == 4 && a.w.head_dim <= 128 ? 12 : 8;
  if (a.w.head_dim == 256)
    launch_rows<256>(a, rows, sms, s);
  else if (a.w.head_dim == 128)
    launch_rows<128>(a, rows, sms, s);
  else
    launch_rows<64>(a, rows, sms, s);
}

}  // namespace xtg
