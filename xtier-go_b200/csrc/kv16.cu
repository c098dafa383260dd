// The 16-bit paged caches: rows appended with their rotation, and the host side of the attention (kv16_attn.cuh).
//
// A row's keys and queries turn by its position: pair i (dims i and i + rotary / 2 of the rotated dims, or 2 i and 2 i + 1)
// by the angle position x freq[i]. The angle is taken as turns in 64 bits, since 32 would leave a far position's angle
// 2^-24 of itself off, and only what is past the last whole turn goes to sinpi and cospi in 32 bits. The turned values
// are rounded once, to the cache's type.
//
// One pass: a CTA takes some rows with all their heads, so that a row's angles, its sequence, page and slot are worked out
// once. 8 dims a thread (two times 8, of a pair's two halves), 16-byte loads and stores.
//
// Measured (B200, device time): 8 prompts of 2048 .. 4096 rows with 16 q / 4 KV heads of 256 f16 in 117 us, 5.8 TB/s of what
// is read and written, 88 % of a copy's rate (125 to 129 us in runs on changing data), issue slots 71 % busy, interleaved in 124
// us; 4 x 4096 rows of a latent cache with 128 q heads, interleaved, in 110 us, 80 %; one row in 3.3 us: one launch, then the
// row's sequence, page and angles one after another.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "kv16_launch.cuh"

namespace xtg {

namespace {

constexpr int kThreads = 256;
// Rows of a CTA where there are many: they share its start, and a thread its place where it keeps it (interleaved)
constexpr int kMaxRowsPerCta = 8;
constexpr int rows_per_cta(bool interleaved) { return interleaved ? kMaxRowsPerCta : 4; }
constexpr int kMaxRotary = 256;

struct Stream {   // k's, v's or q's heads of a row
  const void* src;
  int64_t row, head;   // strides of src
  int heads, units, turned;   // units a head, the first `turned` of them rotated
  int dims, first, rotary;    // rotary 0: copied
  int64_t out_head;           // q: stride of the output's heads; else the pool's
};

struct AppendArgs {
  Stream st[3];   // q, k, v
  void *q_out, *k, *v;
  int64_t k_page, k_slot, v_page, v_slot;
  int k_dim0;   // where k's dims start in its pool's slot
  const int32_t *table, *pos, *cu_rows;
  const float* freq;
  int64_t pages, rows;
  int max_pages, seqs, page_log2, rows_per_cta, half;
  int32_t* err;
};

struct Turn {
  float c, s;
};

// 8 neighbouring values as they lie in memory
template <class X>
struct Raw {
  uint4 w[sizeof(X) / 2];
};
template <class X>
__device__ __forceinline__ Raw<X> load8(const X* p) {
  Raw<X> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(X) / 2; ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
__device__ __forceinline__ void to_f32(const Raw<float>& r, float (&x)[8]) {
  const uint4 a = r.w[0], b = r.w[1];
  x[0] = __uint_as_float(a.x), x[1] = __uint_as_float(a.y), x[2] = __uint_as_float(a.z), x[3] = __uint_as_float(a.w);
  x[4] = __uint_as_float(b.x), x[5] = __uint_as_float(b.y), x[6] = __uint_as_float(b.z), x[7] = __uint_as_float(b.w);
}
template <class X>
__device__ __forceinline__ void to_f32(const Raw<X>& r, float (&x)[8]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = kv16::unpack(w[i], X());
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = kv16::pack(x[2 * i], x[2 * i + 1], T());
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// The last i with cu_rows[i] <= row, by a warp: 32 entries at a time
__device__ __forceinline__ int sequence_of(const AppendArgs& a, int64_t row) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = a.seqs;   // cu_rows[lo] <= row or lo == 0, of n entries from lo on
  while (n > 1) {
    const int step = (n + 31) / 32, i = lo + lane * step;
    const bool below = i < lo + n && a.cu_rows[i] <= row;
    const uint32_t m = __ballot_sync(0xffffffffu, below) | 1u;
    const int k = 31 - __clz(m);
    n = min(step, n - k * step);
    lo += k * step;
  }
  return lo;
}

// X: the rows' type, T: the cache's. By halves 7 CTAs an SM, of 32 registers a thread: for f32 rows one is spilled.
template <class X, class T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, INTERLEAVED ? 5 : 7) append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ __align__(16) Turn turn[kMaxRowsPerCta][kMaxRotary / 2];
  __shared__ struct {
    int64_t page, slot;   // page -1: nowhere to write
    int64_t pos;
    bool live;
  } at[kMaxRowsPerCta];
  pdl_wait();
  pdl_launch_next();
  const int64_t row0 = (int64_t)blockIdx.x * a.rows_per_cta;
  const int rows = (int)min((int64_t)a.rows_per_cta, a.rows - row0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < rows) {
    const int64_t row = row0 + warp;
    const int s = sequence_of(a, row);
    const int64_t from = a.cu_rows[s], to = a.cu_rows[s + 1], p = a.pos[s] + (row - from);
    if (lane == 0) {
      const bool live = row >= from && row < to;
      int64_t page = -1;
      if (live && p >= 0) {
        const int64_t i = p >> a.page_log2;
        if (i >= a.max_pages) {
          if (a.err) atomicExch(a.err, 6);
        } else {
          page = a.table[(int64_t)s * a.max_pages + i];
          if (page >= a.pages) {
            if (a.err) atomicExch(a.err, 7);
            page = -1;
          }
        }
      }
      at[warp] = {page, p & ((1 << a.page_log2) - 1), p, live};
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * a.half; i += kThreads) {
    const int r = i / a.half, e = i - r * a.half;
    const double turns = (double)at[r].pos * ((double)a.freq[e] * 0.15915494309189533577);
    const float half_turns = (float)(2.0 * (turns - rint(turns)));
    Turn t;
    sincospif(half_turns, &t.s, &t.c);
    turn[r][e] = t;
  }
  __syncthreads();
  const int n0 = a.st[0].heads * a.st[0].units, n1 = n0 + a.st[1].heads * a.st[1].units,
            n = n1 + a.st[2].heads * a.st[2].units;
  struct Place {
    int which, h, u, d;   // q, k or v, head, unit, first dim
    bool turned;
  };
  auto place = [&](int u) {
    const int which = u < n0 ? 0 : u < n1 ? 1 : 2;
    const Stream& st = a.st[which];
    u -= which == 0 ? 0 : which == 1 ? n0 : n1;
    const int h = u / st.units;
    u -= h * st.units;
    int d = st.first + 8 * u;
    if (u >= st.turned) {   // the dims before and behind the rotated ones
      d = 8 * (u - st.turned);
      if (d >= st.first && st.rotary) d += st.rotary;
    }
    return Place{which, h, u, d, u < st.turned};
  };
  auto source = [&](const Place& p, int r) {
    const Stream& st = a.st[p.which];
    return static_cast<const X*>(st.src) + (row0 + r) * st.row + p.h * st.head + p.d;
  };
  auto target = [&](const Place& p, int r) {
    const Stream& st = a.st[p.which];
    if (p.which == 0) return static_cast<T*>(a.q_out) + ((row0 + r) * st.heads + p.h) * st.dims + p.d;
    return p.which == 1 ? static_cast<T*>(a.k) + at[r].page * a.k_page + p.h * st.out_head + at[r].slot * a.k_slot + a.k_dim0 + p.d
                        : static_cast<T*>(a.v) + at[r].page * a.v_page + p.h * st.out_head + at[r].slot * a.v_slot + p.d;
  };
  auto nowhere = [&](const Place& p, int r) { return p.which > 0 && at[r].page < 0; };
  if (INTERLEAVED) {
    // a thread takes the same part of a head in all rows, two at once
    constexpr int kAtOnce = sizeof(X) == 4 ? 1 : 2;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const Place p = place(i);
      for (int r0 = 0; r0 < rows; r0 += kAtOnce) {
        Raw<X> raw[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          if (r0 + k < rows) raw[k] = load8(source(p, r0 + k));
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int r = r0 + k;
          if (r >= rows) break;
          if (nowhere(p, r)) continue;
          float x[8];
          to_f32(raw[k], x);
          if (p.turned) {
            const Turn* t = turn[r] + 4 * p.u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const Turn w = t[e];
              const float f = x[2 * e], g = x[2 * e + 1];
              x[2 * e] = f * w.c - g * w.s;
              x[2 * e + 1] = g * w.c + f * w.s;
            }
          }
          if (!at[r].live)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.f;
          store8(target(p, r), x);
        }
      }
    }
  } else {
    // a thread has two pieces on the way as it is: all parts of all rows in turn, with few registers and so many threads (with
    // the loop above and 95 registers the largest case took 239 us, with 32 it takes 117)
    for (int i = threadIdx.x; i < rows * n; i += kThreads) {
      const int r = i / n;
      const Place p = place(i - r * n);
      if (nowhere(p, r)) continue;
      const X* from = source(p, r);
      T* to = target(p, r);
      const bool live = at[r].live;
      float x[8];
      if (p.turned) {
        float y[8];
        to_f32(load8(from), x);
        to_f32(load8(from + a.half), y);
        const Turn* t = turn[r] + 8 * p.u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Turn w = t[e];
          const float f = x[e], g = y[e];
          x[e] = live ? f * w.c - g * w.s : 0.f;
          y[e] = live ? g * w.c + f * w.s : 0.f;
        }
        store8(to, x);
        store8(to + a.half, y);
      } else {
        to_f32(load8(from), x);
        if (!live)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = 0.f;
        store8(to, x);
      }
    }
  }
}

int log2_of(int page) {
  int n = 0;
  while ((1 << n) < page) ++n;
  return n;
}

template <class X, class T>
void launch_append(const AppendArgs& args, bool interleaved, unsigned grid, cudaStream_t s) {
  if (interleaved)
    kv16::launch_dependent(append_kernel<X, T, true>, grid, kThreads, 0, s, args);
  else
    kv16::launch_dependent(append_kernel<X, T, false>, grid, kThreads, 0, s, args);
}

// A pool's map: boxes of `box` slots x 64 dims of a page and KV head, or of all dims where a box holds a chunk's positions:
// 64 dims after 64 dims, as the products' operands lie. Few large copies: with boxes of 16 slots (2 KB each) 64 sequences of
// 16384 .. 32768 positions took 900 us, with 64 slots 730 us.
CUtensorMap pool_map(const void* pool, int dtype, int dims, int page, int heads, int64_t pages, int64_t slot, int64_t head,
                     int64_t page_stride, int box, bool whole) {
  static std::mutex mu;
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!encode) {
      cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
      void* fn = nullptr;
      XTG_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
      XTG_REQUIRE(fn && q == cudaDriverEntryPointSuccess, "kv16: no cuTensorMapEncodeTiled in the driver");
      encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }
  }
  CUtensorMap map;
  const cuuint64_t size[5] = {64u, (cuuint64_t)page, (cuuint64_t)dims / 64, (cuuint64_t)heads, (cuuint64_t)pages};
  // a stride that nothing steps by may be any
  const cuuint64_t strides[4] = {(cuuint64_t)(slot * 2), 128u, (cuuint64_t)((heads > 1 ? head : dims) * 2),
                                 (cuuint64_t)((pages > 1 ? page_stride : dims) * 2)};
  const cuuint32_t boxes[5] = {64u, (cuuint32_t)box, whole ? (cuuint32_t)dims / 64 : 1u, 1u, 1u};
  const cuuint32_t steps[5] = {1u, 1u, 1u, 1u, 1u};
  const CUresult r = encode(&map, dtype == kKv16Bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                            const_cast<void*>(pool), size, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  XTG_REQUIRE(r == CUDA_SUCCESS, "kv16: cuTensorMapEncodeTiled failed");
  return map;
}

// Looks at a barrier before a wait gives up: about a second, no wait begins before the kernels it depends on have ended.
constexpr uint32_t kPolls = 1u << 18;
std::atomic<uint32_t> wait_polls{kPolls};

}  // namespace

bool kv16_dims(bool latent, int head_dim, int v_dim) {
  return kv16::by_shape<__nv_bfloat16>(latent, head_dim, v_dim, 16, [](auto) {});
}

void launch_kv16_append(const Kv16Cache& c, const Kv16Append& r, int sms, cudaStream_t s) {
  AppendArgs a = {};
  auto stream = [&](const void* src, int64_t row, int64_t head, int heads, int dims, bool turned, int64_t out_head) {
    Stream st = {src, row, head, src ? heads : 0, 0, 0, dims, 0, 0, out_head};
    if (turned && r.rotary) {
      st.first = r.first;
      st.rotary = r.rotary;
      st.turned = r.interleaved ? r.rotary / 8 : r.rotary / 16;
    }
    st.units = st.turned + (dims - st.rotary) / 8;
    return st;
  };
  const int turned_dims = c.latent ? c.head_dim - c.v_dim : c.head_dim;
  a.st[0] = stream(r.q, r.q_row, r.q_head, r.heads, turned_dims, true, 0);
  a.st[1] = stream(r.k, r.k_row, r.k_head, c.kv_heads, turned_dims, true, c.k_head);
  a.st[2] = stream(r.v, r.v_row, r.v_head, c.kv_heads, c.v_dim, false, c.latent ? c.k_head : c.v_head);
  a.q_out = r.q_out;
  a.k = c.k;
  a.v = c.latent ? c.k : c.v;
  a.k_page = c.k_page;
  a.k_slot = c.k_slot;
  a.v_page = c.latent ? c.k_page : c.v_page;
  a.v_slot = c.latent ? c.k_slot : c.v_slot;
  a.k_dim0 = c.latent ? c.v_dim : 0;
  a.table = c.table;
  a.pos = c.pos;
  a.cu_rows = c.cu_rows;
  a.freq = r.freq;
  a.pages = c.pages;
  a.rows = c.rows;
  a.max_pages = c.max_pages;
  a.seqs = c.seqs;
  a.page_log2 = log2_of(c.page);
  a.half = r.rotary / 2;
  a.err = c.err;
  // as many as leave 8 CTAs for every SM
  a.rows_per_cta = (int)std::max<int64_t>(1, std::min<int64_t>(c.rows / (8 * sms), rows_per_cta(r.interleaved)));
  const int64_t grid = (c.rows + a.rows_per_cta - 1) / a.rows_per_cta;
  auto by_cache = [&](auto x) {
    using X = decltype(x);
    if (c.dtype == kKv16Bf16)
      launch_append<X, __nv_bfloat16>(a, r.interleaved, (unsigned)grid, s);
    else
      launch_append<X, __half>(a, r.interleaved, (unsigned)grid, s);
  };
  if (r.dtype == kKv16F32)
    by_cache(float());
  else if (r.dtype == kKv16Bf16)
    by_cache(__nv_bfloat16());
  else
    by_cache(__half());
}

int64_t kv16_workspace_bytes(bool latent, int head_dim, int v_dim, int group, int rows_per_seq, int sms) {
  int64_t bytes = -1;
  kv16::by_shape<__nv_bfloat16>(latent, head_dim, v_dim, kv16::block_rows(latent, (int64_t)group * rows_per_seq),
                                [&](auto shape) {
                                  using S = decltype(shape);
                                  bytes = kv16::work_bytes<S>(std::min(sms, kv16::kMaxGrid / 2) * S::OCC);
                                });
  return bytes;
}

int kv16_wait_polls(int polls) {
  return (int)(polls < 0 ? wait_polls.load() : wait_polls.exchange(std::min((uint32_t)polls, 1u << 24)));
}

void launch_kv16_attention(const Kv16Cache& c, const Kv16Attn& r, int sms, cudaStream_t s) {
  kv16::Params p = {};
  const int group = r.heads / c.kv_heads;
  // chunks of 128 positions, of 64 where the keys are wide (Shape::C)
  const int chunk = c.head_dim <= 192 ? 128 : 64, box = std::min(c.page, chunk);
  p.kmap = pool_map(c.k, c.dtype, c.head_dim, c.page, c.kv_heads, c.pages, c.k_slot, c.k_head, c.k_page, box,
                    box == chunk);
  p.vmap = c.latent ? p.kmap
                    : pool_map(c.v, c.dtype, c.v_dim, c.page, c.kv_heads, c.pages, c.v_slot, c.v_head, c.v_page, box,
                               box == chunk);
  p.q = r.q;
  p.q_rot = r.q_rot;
  p.out = r.out;
  p.q_row = r.q_row;
  p.q_head = r.q_head;
  p.r_row = r.r_row;
  p.r_head = r.r_head;
  p.v = static_cast<const uint8_t*>(c.latent ? c.k : c.v);
  p.v_page = c.latent ? c.k_page : c.v_page;
  p.v_head = c.latent ? c.k_head : c.v_head;
  p.v_slot = c.latent ? c.k_slot : c.v_slot;
  p.table = c.table;
  p.pos = c.pos;
  p.cu_rows = c.cu_rows;
  p.pages = c.pages;
  p.rows = c.rows;
  p.max_pages = c.max_pages;
  p.seqs = c.seqs;
  p.page_log2 = log2_of(c.page);
  p.heads = r.heads;
  p.kv_heads = c.kv_heads;
  p.group = group;
  p.group_inv = group > 1 ? (uint32_t)(((1ull << 32) + group - 1) / group) : 0;
  p.window = r.window;
  p.scale = r.scale;
  p.zero_rest = r.zero_rest;
  p.err = c.err;
  p.work = static_cast<float*>(r.work);
  p.polls = wait_polls.load(std::memory_order_relaxed);
  const int rows = kv16::block_rows(c.latent, (int64_t)group * r.rows_per_seq);
  const int most = std::min(sms, kv16::kMaxGrid / 2);
  if (c.dtype == kKv16Bf16)
    kv16::launch<__nv_bfloat16>(p, c.latent, c.head_dim, c.v_dim, rows, r.rows_per_seq, most, s);
  else
    kv16::launch<__half>(p, c.latent, c.head_dim, c.v_dim, rows, r.rows_per_seq, most, s);
}

}  // namespace xtg
