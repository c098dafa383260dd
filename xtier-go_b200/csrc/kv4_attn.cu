// Attention over the 4-bit paged cache (layout: kv4.h): every row sees the cached positions up to its own, the call's
// rows among them (they are stored first), and with a window only the last `window` of these.
//
//   o[r] = sum_p P[r][p] V[p] / sum_p P[r][p],  P[r][p] = 2^(S[r][p] - max_p S[r][p]),  S = log2(e) scale q[r] . K[p]
//
// with K and V as s (code - 8) + z per group of 64 head dims. Both products run on mma.m16n8k16 (f16 in, f32 out)
// straight from the codes: a query row's 16-row tile is 8 rows in two f16 planes, x = hi + lo (22 bits), the hi parts
// in the tile's rows 0-7 and the lo parts in rows 8-15, so that one instruction multiplies both and a lane holds both
// sums of the same (row, column). The scales and offsets enter in f32:
//   q . K[p] = sum_G s[p][G] (q . code - 8 sum q)_G + z[p][G] (sum q)_G        (-8 sum q: the accumulator's start)
//   o[r]     = sum_p (P[r][p] s[p][G]) (code - 8) + P[r][p] z[p][G]            (P s: the A operand, by group G)
// K's codes enter as f16 subnormals, the nibble itself: code 2^-24 (bits 0-3) or code 2^-20 (bits 4-7), exact; the
// query planes of the dims at bits 4-7 carry the factor 1/16. V's become 1024 + code less 1032: there the sum runs
// over positions whose terms cancel, and an uncentred code would cost the bits that cancel.
// P s is brought below 2^15 by a power of two per chunk and group (its largest scale); a chunk's product starts from
// zero and is added to the row's f32 accumulator with that power, so the matrix unit sums at most 64 positions.
//
// What bounds it: the cache's bytes with few rows, the instructions around the matrix products with many. One CTA per
// SM takes an equal share of all (sequence, row block, KV head, 64-position chunk) items in that order, whatever the
// sequences' lengths: shares start and end inside a sequence, whose parts a second kernel joins. A producer warp
// brings chunks (one bulk copy of a page's block of the head) into a ring; 8 consumer warps take them: a row block is
// 1, 2, 4 or 8 tiles of 8 rows, one per warp, and the 8 / tiles warps of a tile take every other chunk, each with a
// running maximum of its own, so that no warp waits for another before the end of a sequence's part.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "kv4.h"

namespace xtg {

namespace {

constexpr int kWarps = 8;                         // consumer warps
constexpr int kThreads = 32 * (kWarps + 1);       // and the producer
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct Kv4Shape {
  static constexpr int kBlock = kv4_block_bytes(D);
  static constexpr int kStages = D == 256 ? 8 : D == 128 ? 16 : 24;   // a multiple of 8; about 110 or 147 KB
  static constexpr int kMergeStride = D + 8;                          // floats of a row's accumulator being merged
};

template <int D>
struct Kv4Smem {
  uint8_t stage[Kv4Shape<D>::kStages][Kv4Shape<D>::kBlock];
  float acc[kWarps][8][Kv4Shape<D>::kMergeStride];
  float m[kWarps][8], l[kWarps][8];
  uint64_t full[Kv4Shape<D>::kStages], empty[Kv4Shape<D>::kStages];
  int present[Kv4Shape<D>::kStages];   // 0: no page, nothing was copied
  int64_t scan[kThreads / 32];
  int64_t start_base;   // items before the sequence that the CTA's share starts in
  int start_seq;
  int failed;           // a wait ran out: the rest of the call waits only briefly and computes nothing
};

// A part of a sequence's items: row block b of KV head h, chunks c0 .. c0 + take - 1 of the sequence's cnt from page lo.
struct Part {
  int seq, b, h;
  int64_t row0, n, pos, lo, cnt, c0, take;
};

// What the combine reads: the split (sequence, row block, head) that a CTA's share ends in, and the last CTA with a
// part of it.
struct Kv4Split {
  int64_t row0;
  int n, h, b, last;   // last < 0: none
};

// The items of sequence s: row blocks x KV heads x chunks. Sequences with rows have at least one chunk (it may hold
// nothing), so that every row is written.
__device__ __forceinline__ int64_t kv4_items(const Kv4Attn& a, int s, int rows_per_block, Part& p) {
  p.row0 = kv4_row_bound(a.w, s);
  p.n = kv4_row_bound(a.w, s + 1) - p.row0;
  if (p.n <= 0) return 0;
  p.seq = s;
  p.pos = a.w.pos[s];
  const int64_t end = p.pos + p.n;
  const int64_t first = a.window > 0 ? p.pos - a.window + 1 : 0;
  p.lo = first > 0 ? first / kKv4Page : 0;
  p.cnt = end > 0 ? (end + kKv4Page - 1) / kKv4Page - p.lo : 1;
  const int64_t most = (int64_t)a.w.max_pages - p.lo;
  if (end > (int64_t)a.w.max_pages * kKv4Page) {   // rows past the table see what the table holds
    if (a.w.err && threadIdx.x == 0) atomicExch(a.w.err, 6);
    p.cnt = most;
  }
  if (p.cnt < 1) p.cnt = 1;
  const int64_t qrows = p.n * (a.heads / a.w.kv_heads);
  return (qrows + rows_per_block - 1) / rows_per_block * a.w.kv_heads * p.cnt;
}

// Walks a CTA's share [start, end) of the items part by part.
struct Walk {
  int s;
  int64_t off, left;
};

__device__ __forceinline__ bool kv4_next(const Kv4Attn& a, int rows_per_block, Walk& k, Part& p) {
  while (k.left > 0 && k.s < a.w.seqs) {
    const int64_t items = kv4_items(a, k.s, rows_per_block, p);
    if (k.off >= items) {
      k.off -= items;
      ++k.s;
      continue;
    }
    const int64_t seg = k.off / p.cnt;
    p.c0 = k.off - seg * p.cnt;
    p.h = (int)(seg % a.w.kv_heads);
    p.b = (int)(seg / a.w.kv_heads);
    p.take = p.cnt - p.c0 < k.left ? p.cnt - p.c0 : k.left;
    k.off += p.take;
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

// The codes of two slots at bits 0-3 (SHIFTED false) or 4-7 of each half, less 8, as f16: 1024 + c - 1032, and
// (1024 + 16 c) / 16 - 72; exact.
__device__ __forceinline__ uint32_t v_codes_low(uint32_t w) {
  return hadd2_u32((w & 0x000f000fu) | 0x64006400u, 0xe408e408u);
}
__device__ __forceinline__ uint32_t v_codes_high(uint32_t w) {
  return hfma2_u32((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u);
}

__device__ __forceinline__ float pow2_bits(int biased) { return __uint_as_float((uint32_t)biased << 23); }

// mbarrier wait that gives up: after the bound, or soon once another wait of the CTA has.
__device__ __forceinline__ bool kv4_wait(uint64_t* bar, uint32_t parity, int* failed, int32_t* err) {
  uint32_t spins = 0;
  while (!mbar_try_wait(bar, parity)) {
    ++spins;
    if (spins > kMaxSpins || (spins > 4096 && *reinterpret_cast<volatile int*>(failed))) {
      atomicExch(failed, 1);
      if (err) atomicExch(err, 1);
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

template <int D>
__global__ void __launch_bounds__(kThreads, 1) kv4_attention_kernel(const Kv4Attn a, const int tiles, float* part,
                                                                   Kv4Split* splits) {
  using Shape = Kv4Shape<D>;
  constexpr int kStages = Shape::kStages;
  constexpr int kGroups = D / kKv4Group, kBlocks = D / 32, H = D < 128 ? D : 128;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  Kv4Smem<D>& sm = *reinterpret_cast<Kv4Smem<D>*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, tq = lane & 3;
  const int group = a.heads / a.w.kv_heads, block_rows = 8 * tiles, lanes = kWarps / tiles;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], tiles);
    }
    mbar_init_fence();
    sm.failed = 0;
    sm.start_seq = a.w.seqs;
    sm.start_base = 0;
  }
  __syncthreads();

  // ---- this CTA's share of the items: an equal part of their sum over the sequences ----
  int64_t total = 0, share = 0, share_end = 0;
  int64_t ctas = gridDim.x;   // with fewer items than CTAs one each, so that no share between two others is empty
  for (int pass = 0; pass < 2; ++pass) {   // the sum, then where the share starts
    int64_t base = 0;
    for (int s0 = 0; s0 < a.w.seqs; s0 += kThreads) {
      const int s = s0 + threadIdx.x;
      Part p;
      const int64_t mine = s < a.w.seqs ? kv4_items(a, s, block_rows, p) : 0;
      int64_t x = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      __syncthreads();
      if (lane == 31) sm.scan[warp] = x;
      __syncthreads();
      int64_t sum = 0;
      for (int v = 0; v < kThreads / 32; ++v) {
        if (v < warp) x += sm.scan[v];
        sum += sm.scan[v];
      }
      if (pass == 1 && base + x - mine <= share && share < base + x) {
        sm.start_seq = s;
        sm.start_base = base + x - mine;
      }
      base += sum;
    }
    if (pass == 0) {
      total = base;
      if (total < ctas) ctas = total;
      if (blockIdx.x < ctas) {
        share = total * blockIdx.x / ctas;
        share_end = total * (blockIdx.x + 1) / ctas;
      }
    }
  }
  __syncthreads();
  Walk walk = {sm.start_seq, share - sm.start_base, share_end - share};
  Part p;

  if (warp == kWarps) {
    // ---- producer: the chunks of every part in order, a page's block of the head per stage ----
    int64_t it = 0;
    while (kv4_next(a, block_rows, walk, p)) {
      for (int64_t k0 = 0; k0 < p.take; k0 += 32) {
        const int64_t mine = k0 + lane < p.take ? kv4_page(a.w, p.seq, p.lo + p.c0 + k0 + lane) : -1;
        const int count = (int)(p.take - k0 < 32 ? p.take - k0 : 32);
        for (int j = 0; j < count; ++j, ++it) {
          const int64_t page = __shfl_sync(0xffffffffu, mine, j);
          if (lane == 0) {
            const int st = (int)(it % kStages);
            const int64_t turn = it / kStages;
            const bool free_ = turn == 0 || kv4_wait(&sm.empty[st], (uint32_t)((turn - 1) & 1), &sm.failed, a.w.err);
            if (free_) {
              sm.present[st] = page >= 0;
              if (page >= 0) {
                mbar_expect_tx(&sm.full[st], Shape::kBlock);
                bulk_g2s(sm.stage[st], a.w.pool + (page * a.w.kv_heads + p.h) * (int64_t)Shape::kBlock, Shape::kBlock,
                         &sm.full[st]);
              } else {
                mbar_arrive(&sm.full[st]);
              }
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0 && share_end <= share) splits[blockIdx.x].last = -1;
  } else {
    const int rt = warp % tiles, sl = warp / tiles;   // this warp's tile of the row block, its turn among the chunks
    int64_t it = 0;
    bool split_after = false;   // the last part goes on in the next CTA
    while (kv4_next(a, block_rows, walk, p)) {
      // ---- the tile's rows: row r of the sequence and KV head is (row r / group of the sequence, q head r % group) ----
      const int64_t qrows = p.n * group, r0 = (int64_t)p.b * block_rows + 8 * rt, r = r0 + g;
      const bool live = r < qrows, any = r0 < qrows;
      const int64_t i = live ? r / group : 0;
      const int64_t t = live ? p.pos + i : -1;   // the row's position; dead rows see nothing
      // the tile's first and last position
      const int64_t tmin = p.pos + r0 / group, tmax = p.pos + (r0 + 7 < qrows ? r0 + 7 : qrows - 1) / group;

      // Q in two f16 planes, scaled by the power of two that brings the row's largest value to 2^14 .. 2^15; a lane has
      // the 8 dims of one K word per block of 32: nibble pair i (dims i, i + 4) is a register of step i / 2
      uint32_t qa[kBlocks][2][4];
      float qsum[kGroups], rf;   // (sum q)_G and the factor from the products' unit to base-2 scores
      {
        float x[kBlocks][8];
        float mx = 0.f;
        const int64_t at = (p.row0 + i) * a.q_row + (p.h * group + (live ? r % group : 0)) * a.q_head;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          if (live)
            load_q8(a.q, at + 32 * b + 8 * tq, a.dtype, x[b]);
          else
#pragma unroll
            for (int e = 0; e < 8; ++e) x[b][e] = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[b][e]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int e2 = (int)(__float_as_uint(mx) >> 23);   // biased exponent of the largest value
        if (e2 < 16) e2 = 16;
        if (e2 > 254) e2 = 254;
        const float up = pow2_bits(127 + 14 + 127 - e2 > 254 ? 254 : 268 - e2);
        rf = a.scale * kLog2e * (16777216.f / up);   // 2^24: the codes' unit
#pragma unroll
        for (int G = 0; G < kGroups; ++G) qsum[G] = 0.f;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[b][e] *= up;
            qsum[b / 2] += x[b][e];
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            split_f16x2(x[b][2 * e], x[b][2 * e + 4], qa[b][e][0], qa[b][e][1]);
            split_f16x2(x[b][2 * e + 1] * 0.0625f, x[b][2 * e + 5] * 0.0625f, qa[b][e][2], qa[b][e][3]);
          }
        }
#pragma unroll
        for (int G = 0; G < kGroups; ++G) {
          qsum[G] += __shfl_xor_sync(0xffffffffu, qsum[G], 1);
          qsum[G] += __shfl_xor_sync(0xffffffffu, qsum[G], 2);
          qsum[G] *= 1.f / 16777216.f;
        }
      }

      float o[kBlocks][4][2];   // the row's dims 32 c + 8 t + 2 tq + {0, 1}, without the offsets' part
      float oz[kGroups];        // sum of P z over this lane's slots
      float run_m = -INFINITY, run_l = 0.f;
#pragma unroll
      for (int c = 0; c < kBlocks; ++c)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) o[c][tt][0] = o[c][tt][1] = 0.f;
#pragma unroll
      for (int G = 0; G < kGroups; ++G) oz[G] = 0.f;

      auto chunk = [&](const uint8_t* stg, int64_t p0, auto masked_) {
        constexpr bool kMasked = decltype(masked_)::value;
        const uint32_t* kw = reinterpret_cast<const uint32_t*>(stg);
        const uint32_t* kpar = reinterpret_cast<const uint32_t*>(stg + kv4_k_params(D));
        const uint32_t* vw = reinterpret_cast<const uint32_t*>(stg + kv4_v_codes(D));
        const uint32_t* vpar = reinterpret_cast<const uint32_t*>(stg + kv4_v_params(D));
        // ---- scores: 8 tiles of 8 slots; this lane: slots 8 j + 2 tq + {0, 1} of its row ----
        float s[8][2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int slot = 8 * j + g;
          float c[kGroups][4];
#pragma unroll
          for (int G = 0; G < kGroups; ++G) {
            c[G][0] = c[G][1] = -8.f * qsum[G];
            c[G][2] = c[G][3] = 0.f;
          }
#pragma unroll
          for (int hf = 0; hf < D / H; ++hf) {
            uint32_t w[H / 32];
            if constexpr (H == 128) {
              const uint4 v = *reinterpret_cast<const uint4*>(kw + ((hf * kKv4Page + slot) * 4 + tq) * 4);
              w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(kw + (slot * 4 + tq) * 2);
              w[0] = v.x, w[1] = v.y;
            }
#pragma unroll
            for (int b = 0; b < H / 32; ++b) {
              const int blk = hf * (H / 32) + b;
              const uint32_t w8 = w[b] >> 8;
              mma_f16(c[blk / 2], qa[blk][0][0], qa[blk][0][1], qa[blk][0][2], qa[blk][0][3], w[b] & 0x000f000fu,
                      w[b] & 0x00f000f0u);
              mma_f16(c[blk / 2], qa[blk][1][0], qa[blk][1][1], qa[blk][1][2], qa[blk][1][3], w8 & 0x000f000fu,
                      w8 & 0x00f000f0u);
            }
          }
          s[j][0] = s[j][1] = 0.f;
#pragma unroll
          for (int G = 0; G < kGroups; ++G) {
            const uint2 w = *reinterpret_cast<const uint2*>(kpar + G * kKv4Page + 8 * j + 2 * tq);
            s[j][0] = fmaf(__uint_as_float(w.x & 0xffff0000u), c[G][0] + c[G][2], s[j][0]);
            s[j][1] = fmaf(__uint_as_float(w.y & 0xffff0000u), c[G][1] + c[G][3], s[j][1]);
            s[j][0] = fmaf(__uint_as_float(w.x << 16), qsum[G], s[j][0]);
            s[j][1] = fmaf(__uint_as_float(w.y << 16), qsum[G], s[j][1]);
          }
          s[j][0] *= rf;
          s[j][1] *= rf;
          if constexpr (kMasked) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int64_t pp = p0 + 8 * j + 2 * tq + e;
              if (pp > t || (a.window > 0 && pp <= t - a.window)) s[j][e] = -INFINITY;
            }
          }
        }
        // ---- the running maximum and sum ----
        float mx = s[0][0];
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fmaxf(s[j][0], s[j][1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float new_m = fmaxf(run_m, mx), ref = new_m == -INFINITY ? 0.f : new_m;
        const float alpha = ex2_approx(run_m - ref);
        run_m = new_m;
        run_l *= alpha;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          s[j][0] = ex2_approx(s[j][0] - ref);
          s[j][1] = ex2_approx(s[j][1] - ref);
          run_l += s[j][0] + s[j][1];
        }
        // ---- P V by group of 64 dims ----
#pragma unroll
        for (int G = 0; G < kGroups; ++G) {
          uint2 w[8];
          int top = 0;   // the largest scale's word: positive f32 order is integer order, NaN's word is negative
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            w[j] = *reinterpret_cast<const uint2*>(vpar + G * kKv4Page + 8 * j + 2 * tq);
            if constexpr (kMasked) {   // what no row of the tile sees may hold anything
              const int64_t pp = p0 + 8 * j + 2 * tq;
              if (pp > tmax || (a.window > 0 && pp <= tmin - a.window)) w[j].x = 0;
              if (pp + 1 > tmax || (a.window > 0 && pp + 1 <= tmin - a.window)) w[j].y = 0;
            }
            top = max(top, max((int)w[j].x, (int)w[j].y));
          }
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          int e2 = top >> 23;
          if (e2 < 27) e2 = 27;
          if (e2 > 254) e2 = 254;
          const float down = pow2_bits(268 - e2), up = pow2_bits(e2 - 14);
          uint32_t pa[4][4];
          oz[G] *= alpha;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float s0 = __uint_as_float(w[j].x & 0xffff0000u), s1 = __uint_as_float(w[j].y & 0xffff0000u);
            float x0 = s[j][0] * (s0 * down), x1 = s[j][1] * (s1 * down);
            if constexpr (kMasked) {   // a masked NaN scale gives nothing
              x0 = s[j][0] == 0.f ? 0.f : x0;
              x1 = s[j][1] == 0.f ? 0.f : x1;
            }
            split_f16x2(x0, x1, pa[j / 2][2 * (j & 1)], pa[j / 2][2 * (j & 1) + 1]);
            oz[G] = fmaf(s[j][0], __uint_as_float(w[j].x << 16), oz[G]);
            oz[G] = fmaf(s[j][1], __uint_as_float(w[j].y << 16), oz[G]);
          }
#pragma unroll
          for (int c = 2 * G; c < 2 * G + 2; ++c) {
            float d[4][4];
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) d[tt][0] = d[tt][1] = d[tt][2] = d[tt][3] = 0.f;
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const uint4 v = *reinterpret_cast<const uint4*>(vw + (((hh * kBlocks + c) * 8 + g) * 4 + tq) * 4);
              const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int tt = 0; tt < 4; ++tt) {
                const uint32_t w8 = word[tt] >> 8;
                const uint32_t(&p0_)[4] = pa[2 * hh];
                const uint32_t(&p1_)[4] = pa[2 * hh + 1];
                mma_f16(d[tt], p0_[0], p0_[1], p0_[2], p0_[3], v_codes_low(word[tt]), v_codes_high(word[tt]));
                mma_f16(d[tt], p1_[0], p1_[1], p1_[2], p1_[3], v_codes_low(w8), v_codes_high(w8));
              }
            }
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
              o[c][tt][0] = fmaf(d[tt][0] + d[tt][2], up, o[c][tt][0] * alpha);
              o[c][tt][1] = fmaf(d[tt][1] + d[tt][3], up, o[c][tt][1] * alpha);
            }
          }
        }
      };

      // ---- this warp's chunks of the part ----
      for (int64_t k = (sl - it % lanes + lanes) % lanes; k < p.take; k += lanes) {
        const int st = (int)((it + k) % kStages);
        const bool ok = kv4_wait(&sm.full[st], (uint32_t)(((it + k) / kStages) & 1), &sm.failed, a.w.err);
        const int64_t p0 = (p.lo + p.c0 + k) * kKv4Page;
        const bool seen = ok && any && sm.present[st] && p0 <= tmax && (a.window <= 0 || p0 + 63 > tmin - a.window);
        if (seen) {
          if (p0 + 63 <= tmin && (a.window <= 0 || p0 > tmax - a.window))
            chunk(sm.stage[st], p0, std::false_type());
          else
            chunk(sm.stage[st], p0, std::true_type());
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[st]);
      }
      it += p.take;

      // ---- the part's warps meet: per row, the warps of its tile by their maxima ----
      run_l += __shfl_xor_sync(0xffffffffu, run_l, 1);
      run_l += __shfl_xor_sync(0xffffffffu, run_l, 2);
#pragma unroll
      for (int G = 0; G < kGroups; ++G) {
        oz[G] += __shfl_xor_sync(0xffffffffu, oz[G], 1);
        oz[G] += __shfl_xor_sync(0xffffffffu, oz[G], 2);
      }
      if (tq == 0) {
        sm.m[warp][g] = run_m;
        sm.l[warp][g] = run_l;
      }
#pragma unroll
      for (int c = 0; c < kBlocks; ++c)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
          *reinterpret_cast<float2*>(&sm.acc[warp][g][32 * c + 8 * tt + 2 * tq]) =
              make_float2(o[c][tt][0] + oz[c / 2], o[c][tt][1] + oz[c / 2]);
      named_bar_sync(1, 32 * kWarps);
      const bool whole = p.c0 == 0 && p.take == p.cnt;
      float* mine = part + (int64_t)(2 * blockIdx.x + (p.c0 == 0 ? 1 : 0)) * block_rows * part_row(D);
      for (int x = threadIdx.x; x < block_rows * (D / 4); x += 32 * kWarps) {
        const int row = x / (D / 4), d0 = 4 * (x % (D / 4)), tile = row / 8, gg = row % 8;
        const int64_t rr = (int64_t)p.b * block_rows + row;
        if (rr >= qrows) continue;
        float M = -INFINITY;
        for (int v = 0; v < lanes; ++v) M = fmaxf(M, sm.m[v * tiles + tile][gg]);
        float l = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int v = 0; v < lanes; ++v) {
          const int from = v * tiles + tile;
          const float mv = sm.m[from][gg], wt = mv == M ? 1.f : ex2_approx(mv - M);
          const float4 u = *reinterpret_cast<const float4*>(&sm.acc[from][gg][d0]);
          l = fmaf(wt, sm.l[from][gg], l);
          y.x = fmaf(wt, u.x, y.x);
          y.y = fmaf(wt, u.y, y.y);
          y.z = fmaf(wt, u.z, y.z);
          y.w = fmaf(wt, u.w, y.w);
        }
        if (whole) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          const int64_t at = ((p.row0 + rr / group) * a.heads + p.h * group + rr % group) * D + d0;
          store_out4(a.out, at, a.dtype, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
        } else {
          float* to = mine + (int64_t)row * part_row(D);
          *reinterpret_cast<float4*>(to + 4 + d0) = y;
          if (d0 == 0) *reinterpret_cast<float2*>(to) = make_float2(M, l);
        }
      }
      split_after = p.c0 == 0 && !whole;
      if (split_after && threadIdx.x == 0) {
        // the last item of this (sequence, row block, head), and the CTA whose share holds it
        const int64_t end = share_end - p.take + p.cnt - 1;
        Kv4Split sp;
        sp.row0 = p.row0;
        sp.n = (int)(p.n < 0x7fffffff ? p.n : 0x7fffffff);
        sp.h = p.h;
        sp.b = p.b;
        sp.last = (int)(((end + 1) * ctas - 1) / total);
        splits[blockIdx.x] = sp;
      }
      named_bar_sync(1, 32 * kWarps);   // before the next part's sums
    }
    if (threadIdx.x == 0 && !split_after && share_end > share) splits[blockIdx.x].last = -1;
  }
  pdl_launch_next();
}

// The parts of a split (sequence, row block, KV head): the last part of CTA blockIdx.x and the first parts of the CTAs
// after it, joined by their maxima in that order. blockIdx.y: rows y, y + 8, ... of the block; 4 warps take every
// fourth part.
template <int D>
__global__ void __launch_bounds__(128) kv4_combine_kernel(const Kv4Attn a, const int tiles, const float* part,
                                                        const Kv4Split* splits) {
  constexpr int kPer = D / 32;
  __shared__ float red[4];
  __shared__ float acc[4][D];
  __shared__ float sum[4];
  pdl_wait();
  const Kv4Split sp = splits[blockIdx.x];
  if (sp.last < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, block_rows = 8 * tiles;
  const int group = a.heads / a.w.kv_heads, first = blockIdx.x, count = sp.last - first + 1;
  for (int row = blockIdx.y; row < block_rows; row += gridDim.y) {
    const int64_t rr = (int64_t)sp.b * block_rows + row;
    if (rr >= (int64_t)sp.n * group) return;   // the same for the whole block
    auto at = [&](int k) {   // the k-th part's row
      return part + ((int64_t)(2 * (first + k) + (k == 0 ? 1 : 0)) * block_rows + row) * part_row(D);
    };
    float M = -INFINITY;
    for (int k = threadIdx.x; k < count; k += 128) M = fmaxf(M, at(k)[0]);
    M = warp_max(M);
    if (lane == 0) red[warp] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float y[kPer] = {}, l = 0.f;
    for (int k = warp; k < count; k += 4) {
      const float* from = at(k);
      const float mv = from[0], wt = mv == M ? 1.f : ex2_approx(mv - M);
      l = fmaf(wt, from[1], l);
#pragma unroll
      for (int e = 0; e < kPer; ++e) y[e] = fmaf(wt, from[4 + 32 * e + lane], y[e]);
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[warp][32 * e + lane] = y[e];
    if (lane == 0) sum[warp] = l;
    __syncthreads();
    l = sum[0] + sum[1] + sum[2] + sum[3];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t to = ((sp.row0 + rr / group) * a.heads + sp.h * group + rr % group) * D;
    for (int d0 = 4 * threadIdx.x; d0 < D; d0 += 512) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < 4; ++k) {
        const float4 u = *reinterpret_cast<const float4*>(&acc[k][d0]);
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
      }
      store_out4(a.out, to + d0, a.dtype, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    }
    __syncthreads();
  }
}

// Tiles of 8 query rows that a CTA takes at once: as many as a sequence's rows fill, up to one per warp.
int row_tiles(int group, int rows_per_seq) {
  const int64_t need = ((int64_t)group * std::max(1, rows_per_seq) + 7) / 8;
  return need >= 5 ? 8 : need >= 3 ? 4 : (int)need;
}

template <int D>
void launch(const Kv4Attn& a, int sms, cudaStream_t s) {
  const int tiles = row_tiles(a.heads / a.w.kv_heads, a.rows_per_seq);
  float* part = a.part;
  Kv4Split* splits = reinterpret_cast<Kv4Split*>(part + (int64_t)sms * 2 * 8 * tiles * part_row(D));
  static std::atomic<uint64_t> optin;
  const int smem = (int)sizeof(Kv4Smem<D>);
  ensure_smem_optin((const void*)kv4_attention_kernel<D>, smem, optin);
  kv4_attention_kernel<D><<<sms, kThreads, smem, s>>>(a, tiles, part, splits);
  XTG_CUDA(cudaGetLastError());
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms, 8);
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  XTG_CUDA(cudaLaunchKernelEx(&cfg, kv4_combine_kernel<D>, a, tiles, (const float*)part, (const Kv4Split*)splits));
}

}  // namespace

int64_t kv4_workspace_bytes(int head_dim, int group, int rows_per_seq, int sms) {
  return (int64_t)sms * (2 * 8 * row_tiles(group, rows_per_seq) * part_row(head_dim) * (int64_t)sizeof(float) +
                         (int64_t)sizeof(Kv4Split));
}

void launch_kv4_attention(const Kv4Attn& a, int sms, cudaStream_t s) {
  if (a.w.head_dim == 64)
    launch<64>(a, sms, s);
  else if (a.w.head_dim == 128)
    launch<128>(a, sms, s);
  else
    launch<256>(a, sms, s);
}

}  // namespace xtg
