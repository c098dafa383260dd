// The 4-bit paged key/value cache: rows quantised into its pages (store) and read back (load). Layout: kv4.h.
//
// Quantiser, per group of 64 head dims, each step in f32 rounded to nearest:
//   lo, hi = min, max;  s = up_bf16(max(2^-100, (hi - lo) (1 / 15)));  z = bf16(lo + 8 s)
//   code = clamp(rint((x - z) (1 / s)), -8, 7) + 8
// The 16 levels z - 8 s .. z + 7 s reach from lo to hi (s is rounded up); only z's own rounding, at most 2^-8 |z|, can
// cut an end. The offset sits at the middle of the levels and not at lo, so that sums of s (code - 8) over many
// positions stay as small as the values' own sums.
//
// One pass over the rows and the pages. A CTA takes one page of one KV head, the heads of a page by neighbouring CTAs,
// which share the rows' DRAM pages. The page is the unit because neighbouring positions share the bytes of V: a CTA that
// owns the page merges all the call's rows into it without atomics, whatever their number.
//
// Measured (B200; algorithmic bytes / time against a copy's 6545 GB/s): 64 x 4096 rows of 6 x 128 read back as bf16 in
// 113 us, 6.0 TB/s, 91 % (123 us, 84 %, in runs of seconds on changing data). 8 x 4096 rows of 4 x 256 f16 written and read
// back in 73 us, 4.7 TB/s, 72 %: the store is bound by its instructions (issue slots 75 % busy), which a thread's 16 values
// share (8 values a thread: 75 us). Small calls are a chain of dependent loads (row offsets and position, page table,
// rows): 2.5 us for one row. Every CTA looks through all sequences, so that calls of very many take long: one row of each
// of 512 written and read back 40 us, of 4096 840 us.
#include <cuda_bf16.h>

#include "common.cuh"
#include "kv4.h"

namespace xtg {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t min_nan2(uint32_t a, uint32_t b, __nv_bfloat16) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t min_nan2(uint32_t a, uint32_t b, __half) {
  uint32_t r;
  asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// 16 neighbouring values as they lie in memory (16-byte aligned)
template <class T>
struct Piece {
  uint4 w[sizeof(T)];
};
template <class T>
__device__ __forceinline__ void load(const T* p, Piece<T>& x) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) x.w[i] = reinterpret_cast<const uint4*>(p)[i];
}

__device__ __forceinline__ float2 halves(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 halves(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ void to_f32(const Piece<float>& p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[4 * i] = __uint_as_float(p.w[i].x);
    x[4 * i + 1] = __uint_as_float(p.w[i].y);
    x[4 * i + 2] = __uint_as_float(p.w[i].z);
    x[4 * i + 3] = __uint_as_float(p.w[i].w);
  }
}
template <class T>
__device__ __forceinline__ void to_f32(const Piece<T>& p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w[4] = {p.w[i].x, p.w[i].y, p.w[i].z, p.w[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = halves(w[e], T());
      x[8 * i + 2 * e] = f.x;
      x[8 * i + 2 * e + 1] = f.y;
    }
  }
}

// The least and the greatest value of a group, NaN if it holds one: over the 4 lanes that have a piece each. 16-bit
// values are compared in pairs, the greatest as the least of the negated.
__device__ __forceinline__ void range(const Piece<float>& p, float& lo, float& hi) {
  float x[16];
  to_f32(p, x);
  lo = x[0];
  hi = -x[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) {
    lo = min_nan(lo, x[e]);
    hi = min_nan(hi, -x[e]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = min_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  hi = -hi;
}
template <class T>
__device__ __forceinline__ void range(const Piece<T>& p, float& lo, float& hi) {
  constexpr uint32_t kSigns = 0x80008000u;
  const T t = T();
  const uint32_t w[8] = {p.w[0].x, p.w[0].y, p.w[0].z, p.w[0].w, p.w[1].x, p.w[1].y, p.w[1].z, p.w[1].w};
  uint32_t l = w[0], h = w[0] ^ kSigns;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    l = min_nan2(l, w[i], t);
    h = min_nan2(h, w[i] ^ kSigns, t);
  }
  uint32_t both = min_nan2(__byte_perm(l, h, 0x5410), __byte_perm(l, h, 0x7632), t);   // least, negated greatest
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) both = min_nan2(both, __shfl_xor_sync(0xffffffffu, both, o), t);
  const float2 f = halves(both, t);
  lo = f.x;
  hi = -f.y;
}

__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(__half* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]), pack_f16x2(x[4], x[5]), pack_f16x2(x[6], x[7]));
}

// The values of 8 codes (nibbles of word) with the parameters p: 16 + code as the f32 whose mantissa starts with the
// nibble, less 24, then s (code - 8) + z with one rounding
__device__ __forceinline__ void values8(uint32_t word, uint32_t p, float (&x)[8]) {
  const float s = __uint_as_float(p & 0xffff0000u), z = __uint_as_float(p << 16);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t at19 = e < 5 ? word << (19 - 4 * e) : word >> (4 * e - 19);
    x[e] = fmaf(__uint_as_float((at19 & 0x00780000u) | 0x41800000u) - 24.f, s, z);
  }
}

// The transpose of 8 words of 8 nibbles: nibble c of word r becomes nibble r of word c
__device__ __forceinline__ void transpose_nibbles(uint32_t (&w)[8]) {
  constexpr uint32_t kLow = 0x0f0f0f0fu;
#pragma unroll
  for (int r = 0; r < 8; r += 2) {
    const uint32_t a = w[r], b = w[r + 1];
    w[r] = (a & kLow) | ((b << 4) & ~kLow);
    w[r + 1] = ((a >> 4) & kLow) | (b & ~kLow);
  }
#pragma unroll
  for (int r = 0; r < 8; r += r % 4 == 1 ? 3 : 1) {   // 0, 1, 4, 5
    const uint32_t a = w[r], b = w[r + 2];
    w[r] = __byte_perm(a, b, 0x6240);
    w[r + 2] = __byte_perm(a, b, 0x7351);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint32_t a = w[r], b = w[r + 4];
    w[r] = __byte_perm(a, b, 0x5410);
    w[r + 4] = __byte_perm(a, b, 0x7632);
  }
}

// The (sequence, page) of task blockIdx.x / kv_heads. A sequence of n rows touches at most n / 64 + 2 pages, so task numbers
// start at cu_rows[s] / 64 + 2 s for sequence s: found without a prefix sum over the sequences' positions.
struct Task {
  int64_t row0;   // the call's row at the page's first touched slot
  int64_t page;   // -1: nothing there
  int slot0, count;
};

// The thread that finds the task's sequence works the rest out (its position is loaded with the search: these loads one
// after another are most of a small call's time). False: nothing to do.
__device__ __forceinline__ bool find_task(const Kv4Where& w, Task& shared, Task& t) {
  const int64_t task = blockIdx.x / (uint32_t)w.kv_heads;
  if (threadIdx.x == 0) shared.count = 0;
  pdl_wait();
  pdl_launch_next();
  __syncthreads();
  for (int s = threadIdx.x; s < w.seqs; s += kThreads) {
    const int64_t a = kv4_row_bound(w, s), b = kv4_row_bound(w, s + 1), pos = w.pos[s];
    const int64_t from = task - (a / kKv4Page + 2 * (int64_t)s);
    if (from < 0 || task >= b / kKv4Page + 2 * (int64_t)(s + 1)) continue;
    const int64_t index = (pos >> 6) + from;   // floor: positions may be negative
    const int64_t p = index * kKv4Page;        // the page's first position
    const int64_t i0 = p > pos ? p - pos : 0, i1 = p + kKv4Page - pos < b - a ? p + kKv4Page - pos : b - a;
    if (i0 < i1) shared = {a + i0, kv4_page(w, s, index), (int)(pos + i0 - p), (int)(i1 - i0)};
  }
  __syncthreads();
  t = shared;
  return t.count > 0;
}

// Quantises the 16 values that this lane has of a group: their codes as nibbles, the group's parameters.
template <class T>
__device__ __forceinline__ void quantise(const Piece<T>& p, uint32_t (&word)[2], uint32_t& par) {
  float x[16], lo, hi;
  range(p, lo, hi);
  to_f32(p, x);
  const float raw = __fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f);
  const float s = fmaxf(__uint_as_float((__float_as_uint(raw) + 0xffffu) & 0xffff0000u), kKv4MinScale);
  const float z = __bfloat162float(__float2bfloat16_rn(__fadd_rn(lo, __fmul_rn(8.f, s))));
  const bool fine = raw < INFINITY && fabsf(z) < INFINITY;   // false for NaN too
  const float inv = __frcp_rn(s);
  // adding 1.5 2^23 + 8 rounds to an integer, ties to even, in the low bits: the code. Codes outside 0 .. 15 come only
  // from z's rounding where |z| passes 2^7 s: the least and the greatest value, which bound the others, tell.
  constexpr float kRound = 12582920.f;
  constexpr uint32_t kBits = 0x4b400000u;   // of code 0
  auto level = [&](float v) { return __fmul_rn(__fsub_rn(v, z), inv); };
  auto code = [&](float v) { return __float_as_uint(__fadd_rn(level(v), kRound)); };
  word[0] = word[1] = 0;
  if (code(lo) >= kBits && code(hi) <= kBits + 15) {
    // sum of 16^e bits(e) less that of code 0's bits
#pragma unroll
    for (int e = 15; e >= 0; --e) word[e / 8] = 16u * word[e / 8] + code(x[e]);
    word[0] -= kBits * 0x11111111u;
    word[1] -= kBits * 0x11111111u;
  } else {
#pragma unroll
    for (int e = 15; e >= 0; --e) {   // clamped first: a level may lie past what the addition rounds
      const float t = fminf(fmaxf(level(x[e]), -8.f), 7.f);
      word[e / 8] = 16u * word[e / 8] + (__float_as_uint(__fadd_rn(t, kRound)) - kBits);
    }
  }
  if (!fine) word[0] = word[1] = 0;
  par = fine ? (__float_as_uint(s) & 0xffff0000u) | (__float_as_uint(z) >> 16) : kKv4NanParam;
}

template <class T, int D>
__global__ void __launch_bounds__(kThreads) kv4_store_kernel(const Kv4Where w, const Kv4Rows r) {
  constexpr int H = D < 128 ? D : 128, kPerRow = D / 16, kRowsAtOnce = kThreads / kPerRow;
  constexpr int kStride = D / 8 + 4;   // of a slot's words in shared memory: 4 slots x 8 words without bank conflicts
  __shared__ __align__(8) uint32_t codes[kKv4Page * kStride];
  __shared__ Task task;
  Task t;
  if (!find_task(w, task, t) || t.page < 0) return;
  const int h = blockIdx.x % (uint32_t)w.kv_heads;
  uint8_t* block = w.pool + (t.page * w.kv_heads + h) * (int64_t)kv4_block_bytes(D);
  uint32_t* kcodes = reinterpret_cast<uint32_t*>(block);
  uint32_t* kpar = reinterpret_cast<uint32_t*>(block + kv4_k_params(D));
  uint32_t* vcodes = reinterpret_cast<uint32_t*>(block + kv4_v_codes(D));
  uint32_t* vpar = reinterpret_cast<uint32_t*>(block + kv4_v_params(D));

  // V's words, of a head dim each and 8 slots: item i < D is 8 neighbouring dims'. The slots that this call does not write
  // keep their codes, requested before the rows.
  static_assert(D <= kThreads, "an item per thread");
  const int tt = threadIdx.x & 3, a = (threadIdx.x >> 2) & 3, c = (threadIdx.x >> 4) % (D / 32), hh = threadIdx.x / (D / 2);
  uint32_t* vto = vcodes + ((hh * (D / 32) + c) * 8 * 4 + a) * 4 + tt;
  uint32_t mask = 0, old[8] = {};
  if (threadIdx.x < D) {
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int slot = 32 * hh + 2 * a + 8 * (n % 4) + n / 4;
      if (slot >= t.slot0 && slot < t.slot0 + t.count) mask |= 15u << (4 * n);
    }
    if (mask != 0 && mask != 0xffffffffu)
#pragma unroll
      for (int g = 0; g < 8; ++g) old[g] = vto[16 * g];
  }

  // a thread has dims d0 .. d0 + 15 of every kRowsAtOnce-th row, 4 threads a group
  const int d0 = 16 * (threadIdx.x % kPerRow), first = threadIdx.x / kPerRow;
  const T* ksrc = static_cast<const T*>(r.k) + t.row0 * r.k_row + h * r.k_head + d0;
  const T* vsrc = static_cast<const T*>(r.v) + t.row0 * r.v_row + h * r.v_head + d0;
  for (int i0 = 0; i0 < t.count; i0 += kRowsAtOnce) {   // whole warps: the groups' threads exchange their minima
    const int i = i0 + first, slot = t.slot0 + i;
    Piece<T> k = {}, v = {};
    if (i < t.count) {
      load(ksrc + i * r.k_row, k);
      load(vsrc + i * r.v_row, v);
    }
    uint32_t kw[2], kp, vw[2], vp;
    quantise(k, kw, kp);
    quantise(v, vw, vp);
    if (i < t.count) {
      uint32_t* to = kcodes + ((d0 / H * kKv4Page + slot) * 4 + d0 % 32 / 8) * (H / 32) + d0 % H / 32;
      to[0] = kw[0];
      to[H / 32] = kw[1];
      *reinterpret_cast<uint2*>(codes + slot * kStride + d0 / 8) = make_uint2(vw[0], vw[1]);
      if (d0 % 64 == 0) {
        kpar[d0 / 64 * kKv4Page + slot] = kp;
        vpar[d0 / 64 * kKv4Page + slot] = vp;
      }
    }
  }
  __syncthreads();
  if (mask != 0) {
    uint32_t words[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) words[n] = codes[(32 * hh + 2 * a + 8 * (n % 4) + n / 4) * kStride + 4 * c + tt];
    transpose_nibbles(words);
#pragma unroll
    for (int g = 0; g < 8; ++g) vto[16 * g] = (old[g] & ~mask) | (words[g] & mask);
  }
}

template <class T, int D>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 8 : 6) kv4_load_kernel(const Kv4Where w, const Kv4Rows r, unsigned tasks) {
  constexpr int H = D < 128 ? D : 128, kPerRow = D / 8;
  __shared__ __align__(16) uint32_t par[2][D / 64][kKv4Page];   // K's, V's
  __shared__ Task task;
  Task t;
  if (blockIdx.x >= tasks) {
    pdl_wait();
    pdl_launch_next();
    kv4_zero_rest(w, r.k, r.v, r.k_row * sizeof(T), tasks);
    return;
  }
  if (!find_task(w, task, t)) return;
  const int h = blockIdx.x % (uint32_t)w.kv_heads;
  T* kout = static_cast<T*>(r.k) + t.row0 * r.k_row + h * r.k_head;
  T* vout = static_cast<T*>(r.v) + t.row0 * r.v_row + h * r.v_head;
  if (t.page < 0) {   // nothing there: zeros
    const float zero[8] = {};
    for (int u = threadIdx.x; u < t.count * kPerRow; u += kThreads) {
      store8(kout + (u / kPerRow) * r.k_row + 8 * (u % kPerRow), zero);
      store8(vout + (u / kPerRow) * r.v_row + 8 * (u % kPerRow), zero);
    }
    return;
  }
  const uint8_t* block = w.pool + (t.page * w.kv_heads + h) * (int64_t)kv4_block_bytes(D);
  auto written = [&](int slot) { return slot >= t.slot0 && slot < t.slot0 + t.count; };
  // 2 D items of 64 values, 8 words each, D of K and D of V: K's two uint4 (of one slot each), V's of 8 dims at 8 slots
  constexpr int kItems = (2 * D + kThreads - 1) / kThreads;
  uint32_t words[kItems][8];
#pragma unroll
  for (int x = 0; x < kItems; ++x) {
    const int item = x * kThreads + threadIdx.x;
    if (item < D) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {   // uint4 item + D e: coalesced
        const uint4 v = reinterpret_cast<const uint4*>(block)[item + D * e];
        words[x][4 * e] = v.x, words[x][4 * e + 1] = v.y, words[x][4 * e + 2] = v.z, words[x][4 * e + 3] = v.w;
      }
    } else if (item < 2 * D) {
      const int i = item - D, tt = i & 3, a = (i >> 2) & 3, c = (i >> 4) % (D / 32), hh = i / (D / 2);
      const uint32_t* from = reinterpret_cast<const uint32_t*>(block + kv4_v_codes(D)) +
                             ((hh * (D / 32) + c) * 8 * 4 + a) * 4 + tt;
#pragma unroll
      for (int g = 0; g < 8; ++g) words[x][g] = from[16 * g];
    }
  }
  for (int i = threadIdx.x; i < D / 2; i += kThreads) {   // D / 4 16-byte pieces each
    const bool isv = i >= D / 4;
    reinterpret_cast<uint4*>(par)[i] = reinterpret_cast<const uint4*>(
        block + (isv ? kv4_v_params(D) : kv4_k_params(D)))[isv ? i - D / 4 : i];
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < kItems; ++x) {
    const int item = x * kThreads + threadIdx.x;
    if (item < D) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {   // word [hh][slot][a][b]: dims H hh + 32 b + 8 a ..
        const int i = 4 * (item + D * (e / 4)) + e % 4;
        const int b = i % (H / 32), a = i / (H / 32) % 4, slot = i / (H / 8) % kKv4Page, hh = i / (8 * H);
        if (!written(slot)) continue;
        const int d0 = H * hh + 32 * b + 8 * a;
        float v[8];
        values8(words[x][e], par[0][d0 / 64][slot], v);
        store8(kout + (slot - t.slot0) * r.k_row + d0, v);
      }
    } else if (item < 2 * D) {
      const int i = item - D, tt = i & 3, a = (i >> 2) & 3, c = (i >> 4) % (D / 32), hh = i / (D / 2);
      const int d0 = 32 * c + 8 * tt;
      transpose_nibbles(words[x]);
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int slot = 32 * hh + 2 * a + 8 * (n % 4) + n / 4;
        if (!written(slot)) continue;
        float v[8];
        values8(words[x][n], par[1][d0 / 64][slot], v);
        store8(vout + (slot - t.slot0) * r.v_row + d0, v);
      }
    }
  }
}

template <class F>
void by_type_and_dim(int dtype, int head_dim, F&& f) {
  auto dim = [&](auto t) {
    if (head_dim == 64)
      f(t, std::integral_constant<int, 64>());
    else if (head_dim == 128)
      f(t, std::integral_constant<int, 128>());
    else
      f(t, std::integral_constant<int, 256>());
  };
  if (dtype == kKv4F32)
    dim(float());
  else if (dtype == kKv4Bf16)
    dim(__nv_bfloat16());
  else
    dim(__half());
}

unsigned task_grid(const Kv4Where& w) {
  const int64_t ctas = (w.rows / kKv4Page + 2 * (int64_t)w.seqs) * w.kv_heads;
  XTG_REQUIRE(ctas < (1ll << 31) - 4, "kv4: too many pages x KV heads in one call");
  return (unsigned)ctas;
}

}  // namespace

void launch_kv4_store(const Kv4Where& w, const Kv4Rows& r, cudaStream_t s) {
  by_type_and_dim(r.dtype, w.head_dim, [&](auto t, auto d) {
    launch_kv4(kv4_store_kernel<decltype(t), decltype(d)::value>, task_grid(w), kThreads, 0, s, w, r);
  });
}

void launch_kv4_load(const Kv4Where& w, const Kv4Rows& r, cudaStream_t s) {
  by_type_and_dim(r.dtype, w.head_dim, [&](auto t, auto d) {
    const unsigned tasks = task_grid(w);
    launch_kv4(kv4_load_kernel<decltype(t), decltype(d)::value>, tasks + kv4_rest_blocks(w), kThreads, 0, s, w, r, tasks);
  });
}

}  // namespace xtg
