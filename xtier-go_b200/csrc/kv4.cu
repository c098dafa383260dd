// The 4-bit paged key/value cache: rows quantised into its pages (store) and read back (load). Layout: kv4.h.
//
// Quantiser, per group of 64 head dims, each step in f32 rounded to nearest:
//   lo, hi = min, max;  s = up_bf16(max(2^-100, (hi - lo) (1 / 15)));  z = bf16(lo + 8 s)
//   code = clamp(rint((x - z) (1 / s)), -8, 7) + 8
// The 16 levels z - 8 s .. z + 7 s reach from lo to hi (s is rounded up); only z's own rounding, at most 2^-9 |z|, can
// cut an end. The offset sits at the middle of the levels and not at lo, so that sums of s (code - 8) over many
// positions stay as small as the values' own sums.
//
// Both kernels are bound by memory: one pass over the rows and the pages. A CTA takes one page of one KV head. The
// page is the unit because neighbouring positions share the bytes of V: a CTA that owns the page merges all the
// call's rows into it without atomics, whatever their number.
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
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 8 neighbouring values (16-byte aligned) to and from f32
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const __half* p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
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

// The (sequence, page) of task blockIdx.x. A sequence of n rows touches at most n / 64 + 2 pages, so task numbers
// start at cu_rows[s] / 64 + 2 s for sequence s: found without a prefix sum over the sequences' positions.
struct Task {
  int64_t row0;   // the call's row at the page's first touched slot
  int slot0, count;
  int64_t page;
};

__device__ __forceinline__ bool find_task(const Kv4Where& w, int* shared_seq, Task& t) {
  const int64_t task = blockIdx.x;
  if (threadIdx.x == 0) *shared_seq = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < w.seqs; s += kThreads) {
    const int64_t lo = kv4_row_bound(w, s) / kKv4Page + 2 * (int64_t)s;
    const int64_t hi = kv4_row_bound(w, s + 1) / kKv4Page + 2 * (int64_t)(s + 1);
    if (lo <= task && task < hi) *shared_seq = s;
  }
  __syncthreads();
  const int s = *shared_seq;
  if (s < 0) return false;
  const int64_t a = kv4_row_bound(w, s), n = kv4_row_bound(w, s + 1) - a;
  const int64_t pos = w.pos[s];
  const int64_t index = (pos >> 6) + task - (a / kKv4Page + 2 * (int64_t)s);   // floor: positions may be negative
  const int64_t p = index * kKv4Page;                                          // the page's first position
  const int64_t i0 = p > pos ? p - pos : 0, i1 = p + kKv4Page - pos < n ? p + kKv4Page - pos : n;
  if (i0 >= i1) return false;
  t.row0 = a + i0;
  t.slot0 = (int)(pos + i0 - p);
  t.count = (int)(i1 - i0);
  t.page = kv4_page(w, s, index);
  return true;
}

template <class T, int D>
__global__ void __launch_bounds__(kThreads) kv4_store_kernel(const Kv4Where w, const Kv4Rows r) {
  constexpr int H = D < 128 ? D : 128, kPerRow = D / 8;
  constexpr int kStride = D + 16;   // of a slot's codes in shared memory: 8 slots x 4 dims without bank conflicts
  __shared__ __align__(16) uint8_t codes[kKv4Page * kStride];
  __shared__ int seq;
  Task t;
  if (!find_task(w, &seq, t) || t.page < 0) return;
  const int h = blockIdx.y;
  uint8_t* block = w.pool + (t.page * w.kv_heads + h) * (int64_t)kv4_block_bytes(D);
  uint32_t* kcodes = reinterpret_cast<uint32_t*>(block);
  uint32_t* kpar = reinterpret_cast<uint32_t*>(block + kv4_k_params(D));
  uint32_t* vcodes = reinterpret_cast<uint32_t*>(block + kv4_v_codes(D));
  uint32_t* vpar = reinterpret_cast<uint32_t*>(block + kv4_v_params(D));

  // one lane: 8 neighbouring dims of one row of K or V; 8 lanes: a group
  const int per = t.count * kPerRow;
  for (int u0 = 0; u0 < 2 * per; u0 += kThreads) {
    const int u = u0 + threadIdx.x;
    const bool live = u < 2 * per, isv = u >= per;
    const int i = (isv ? u - per : u) / kPerRow, d0 = 8 * (u % kPerRow), slot = t.slot0 + i;   // per: whole rows
    float x[8] = {};
    if (live) {
      const T* src = isv ? static_cast<const T*>(r.v) + (t.row0 + i) * r.v_row + h * r.v_head
                         : static_cast<const T*>(r.k) + (t.row0 + i) * r.k_row + h * r.k_head;
      load8(src + d0, x);
    }
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      lo = min_nan(lo, x[e]);
      hi = max_nan(hi, x[e]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const float raw = __fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f);
    const float s = fmaxf(__uint_as_float((__float_as_uint(raw) + 0xffffu) & 0xffff0000u), kKv4MinScale);
    const float z = bf16_bits_to_f32(f32_to_bf16_bits(__fadd_rn(lo, __fmul_rn(8.f, s))));
    const bool fine = raw < INFINITY && fabsf(z) < INFINITY;   // false for NaN too
    const float inv = __frcp_rn(s);
    uint32_t word = 0;
    uint32_t bytes[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = fminf(fmaxf(__fmul_rn(__fsub_rn(x[e], z), inv), -8.f), 7.f);
      // + 1.5 2^23 rounds to an integer, ties to even; + 8 makes it the code (0 .. 15, the low bits)
      const uint32_t code = fine ? __float_as_uint(__fadd_rn(c, 12582920.f)) & 15u : 0u;
      word |= code << (4 * e);
      bytes[e / 4] |= code << (8 * (e % 4));
    }
    if (live) {
      uint32_t* par = isv ? vpar : kpar;
      if ((d0 & 63) == 0)
        par[(d0 / 64) * kKv4Page + slot] =
            fine ? (__float_as_uint(s) & 0xffff0000u) | (__float_as_uint(z) >> 16) : kKv4NanParam;
      if (isv)
        *reinterpret_cast<uint2*>(codes + slot * kStride + d0) = make_uint2(bytes[0], bytes[1]);
      else
        kcodes[((d0 / H * kKv4Page + slot) * 4 + d0 % 32 / 8) * (H / 32) + d0 % H / 32] = word;
    }
  }
  __syncthreads();
  // V's words: 8 slots of a head dim each; the slots that this call does not write keep their codes
  for (int i = threadIdx.x; i < 8 * D; i += kThreads) {
    const int tt = i & 3, a = (i >> 2) & 3, g = (i >> 4) & 7, c = (i >> 7) % (D / 32), hh = i / (4 * D);
    const int first = 32 * hh + 2 * a, dim = 32 * c + 8 * tt + g;
    uint32_t word = 0, mask = 0;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int slot = first + 8 * (n % 4) + n / 4;
      if (slot >= t.slot0 && slot < t.slot0 + t.count) {
        word |= (uint32_t)codes[slot * kStride + dim] << (4 * n);
        mask |= 15u << (4 * n);
      }
    }
    if (mask == 0xffffffffu)
      vcodes[i] = word;
    else if (mask)
      vcodes[i] = (vcodes[i] & ~mask) | word;
  }
}

template <class T, int D>
__global__ void __launch_bounds__(kThreads) kv4_load_kernel(const Kv4Where w, const Kv4Rows r) {
  constexpr int H = D < 128 ? D : 128, kPerRow = D / 8;
  __shared__ __align__(16) uint32_t par[2][D / 64][kKv4Page];   // K's, V's
  __shared__ __align__(16) uint32_t vcodes[8 * D];
  __shared__ int seq;
  Task t;
  if (!find_task(w, &seq, t)) return;
  const int h = blockIdx.y;
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
  for (int i = threadIdx.x; i < 2 * D; i += kThreads)
    reinterpret_cast<uint4*>(vcodes)[i] = reinterpret_cast<const uint4*>(block + kv4_v_codes(D))[i];
  for (int i = threadIdx.x; i < D / 2; i += kThreads) {   // D / 4 16-byte pieces each
    const bool isv = i >= D / 4;
    reinterpret_cast<uint4*>(par)[i] = reinterpret_cast<const uint4*>(
        block + (isv ? kv4_v_params(D) : kv4_k_params(D)))[isv ? i - D / 4 : i];
  }
  __syncthreads();
  const uint32_t* kcodes = reinterpret_cast<const uint32_t*>(block);
  for (int u = threadIdx.x; u < t.count * kPerRow; u += kThreads) {   // K: the words in their own order
    const int b = u % (H / 32), a = u / (H / 32) % 4, hh = u / (H / 8) % (D / H), i = u / kPerRow;
    const int slot = t.slot0 + i, d0 = H * hh + 32 * b + 8 * a;
    const uint32_t word = kcodes[((hh * kKv4Page + slot) * 4 + a) * (H / 32) + b], p = par[0][d0 / 64][slot];
    const float s = __uint_as_float(p & 0xffff0000u), z = __uint_as_float(p << 16);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((int)((word >> (4 * e)) & 15u) - 8), s, z);
    store8(kout + i * r.k_row + d0, x);
  }
  // V: a warp takes 8 neighbouring slots (2 a + j) x 4 pieces of 8 dims, 16 words of each shared-memory row
  const int lane = threadIdx.x & 31;
  for (int o = threadIdx.x >> 5; o < 8 * (D / 32); o += kThreads / 32) {
    const int octet = o / (D / 32), c = o % (D / 32), tt = lane & 3, slot = 8 * octet + (lane >> 2);
    if (slot < t.slot0 || slot >= t.slot0 + t.count) continue;
    const int d0 = 32 * c + 8 * tt, n = octet % 4 + 4 * (slot % 2);
    const uint32_t p = par[1][d0 / 64][slot];
    const float s = __uint_as_float(p & 0xffff0000u), z = __uint_as_float(p << 16);
    float x[8];
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      const uint32_t word = vcodes[(((octet / 4 * (D / 32) + c) * 8 + g) * 4 + slot % 8 / 2) * 4 + tt];
      x[g] = fmaf((float)((int)((word >> (4 * n)) & 15u) - 8), s, z);
    }
    store8(vout + (slot - t.slot0) * r.v_row + d0, x);
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

dim3 task_grid(const Kv4Where& w) {
  return dim3((unsigned)(w.rows / kKv4Page + 2 * (int64_t)w.seqs), (unsigned)w.kv_heads);
}

}  // namespace

void launch_kv4_store(const Kv4Where& w, const Kv4Rows& r, cudaStream_t s) {
  by_type_and_dim(r.dtype, w.head_dim, [&](auto t, auto d) {
    kv4_store_kernel<decltype(t), decltype(d)::value><<<task_grid(w), kThreads, 0, s>>>(w, r);
  });
  XTG_CUDA(cudaGetLastError());
}

void launch_kv4_load(const Kv4Where& w, const Kv4Rows& r, cudaStream_t s) {
  by_type_and_dim(r.dtype, w.head_dim, [&](auto t, auto d) {
    kv4_load_kernel<decltype(t), decltype(d)::value><<<task_grid(w), kThreads, 0, s>>>(w, r);
  });
  XTG_CUDA(cudaGetLastError());
}

}  // namespace xtg
