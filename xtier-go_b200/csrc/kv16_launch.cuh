// Launches of the attention over the 16-bit paged caches, by shape (included once for each type of the cache).
#pragma once

#include "kv16_attn.cuh"

namespace xtg {
namespace kv16 {

// Rows of a block, from about how many (row, q head) pairs of a KV head a sequence has: the smallest that holds them.
// A latent cache's tiles leave room for 64.
inline int block_rows(bool latent, int64_t pairs) {
  if (pairs <= 16) return 16;
  if (pairs <= 32) return 32;
  return pairs <= 64 || latent ? 64 : 128;
}

// f(a Shape) for the call's dims; false: there is no kernel for them
template <class T, class F>
bool by_shape(bool latent, int head_dim, int v_dim, int rows, F&& f) {
  auto with = [&](auto dk, auto dv, auto is_latent) {
    constexpr int DK = decltype(dk)::value, DV = decltype(dv)::value;
    constexpr bool L = decltype(is_latent)::value;
    if (rows == 16)
      f(Shape<T, DK, DV, L, 16>());
    else if (rows == 32)
      f(Shape<T, DK, DV, L, 32>());
    else if (rows == 64 || L)
      f(Shape<T, DK, DV, L, 64>());
    else
      f(Shape<T, DK, DV, L, L ? 64 : 128>());
    return true;
  };
  auto is = [&](bool l, int dk, int dv) { return latent == l && head_dim == dk && v_dim == dv; };
  using std::integral_constant;
  using No = std::false_type;
  using Yes = std::true_type;
  if (is(false, 64, 64)) return with(integral_constant<int, 64>(), integral_constant<int, 64>(), No());
  if (is(false, 128, 128)) return with(integral_constant<int, 128>(), integral_constant<int, 128>(), No());
  if (is(false, 192, 128)) return with(integral_constant<int, 192>(), integral_constant<int, 128>(), No());
  if (is(false, 256, 256)) return with(integral_constant<int, 256>(), integral_constant<int, 256>(), No());
  if (is(true, 320, 256)) return with(integral_constant<int, 320>(), integral_constant<int, 256>(), Yes());
  if (is(true, 576, 512)) return with(integral_constant<int, 576>(), integral_constant<int, 512>(), Yes());
  return false;
}

// Sequences of at most so many row blocks have a team of CTAs, which read their chunks side by side; with more (prompts, whose
// keys stay in L2 meanwhile) the blocks go one after another. Without teams and with these: 8 sequences of 256 rows over 32768
// positions 1233 and 1215 us, 4 of 200 rows over 16384 with heads of 256 352 and 328, 16 of 4 rows over latent caches with 128
// heads 221 and 202. Teams of up to 16 are within 1 % of these, but for 8 rows of 128 latent heads (477 us and 448).
constexpr int kMostTeam = 8;

// defined in kv16_bf16.cu and kv16_f16.cu
template <class T>
void launch(const Params& p, bool latent, int head_dim, int v_dim, int rows, int rows_per_seq, int sms, cudaStream_t s);

// A launch that may overlap the end of the kernel before it on the stream; the kernel waits (pdl_wait).
template <class... P, class... A>
void launch_dependent(void (*f)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t s, A&&... args) {
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

#ifdef KV16_TYPE
template <class T>
void launch(const Params& p, bool latent, int head_dim, int v_dim, int rows, int rows_per_seq, int sms, cudaStream_t s) {
  by_shape<T>(latent, head_dim, v_dim, rows, [&](auto shape) {
    using S = decltype(shape);
    Params a = p;
    const int64_t blocks_per_seq = ((int64_t)a.group * rows_per_seq + S::N - 1) / S::N;
    a.team = blocks_per_seq <= kMostTeam ? (int)std::min<int64_t>(blocks_per_seq, sms) : 1;
    // What a part costs besides its chunks, in chunks: 2 for few rows (64 sequences of 8 rows with a window of 1024: 73 us,
    // with 1 77, with 4 75), 3 for more (128 rows, prompts of 2048: 108 us, with 2 124, with 4 110; 64 rows, 64 sequences of 16
    // rows: 78 us, with 1 80), 4 for latent caches (16 x 4 rows: 27.4 us, with 2 29.4; latent 256 with 32 heads, 128 sequences of
    // 1024 .. 2048: 48.6 us, with 2 51.6; with 16 heads 25.7, with 2 27.7).
    a.part_cost = S::LATENT ? 4 : S::N <= 32 ? 2 : 3;
    a.least_share = 1;
    a.team_inv = a.team > 1 ? (uint32_t)(((1ull << 32) + a.team - 1) / a.team) : 0;
    const int grid = sms * S::OCC / a.team * a.team;
    const int64_t slots = a.rows * a.group / (S::N * a.team) + a.seqs;
    XTG_REQUIRE(slots < (1ll << 31), "kv16: too many row blocks in one call");
    a.slots = (int)slots;
    const int64_t items = slots * a.kv_heads * a.team;
    // Few items have many parts each, and a join per item is spread over more threads (1 x 4096: 12.4 us, by CTA 14.5; 6 x 4096
    // with 6 KV heads 16.9 and 19.9); more have few parts (32 latent sequences of 8192: by CTA 77.9 us, by item 81.6).
    a.by_item = items <= grid / 4;
    static std::atomic<uint64_t> optin;
    const void* kernel = reinterpret_cast<const void*>(&attention_kernel<S>);
    ensure_smem_optin(kernel, S::kSmemBytes, optin);
    if (S::WG == 2) {
      // setmaxnreg would wait forever in a kernel that starts with fewer registers than its shares were worked out for
      static std::atomic<int> registers{0};
      if (registers.load(std::memory_order_relaxed) == 0) {
        cudaFuncAttributes attr;
        XTG_CUDA(cudaFuncGetAttributes(&attr, kernel));
        registers.store(attr.numRegs, std::memory_order_relaxed);
      }
      XTG_REQUIRE((registers.load(std::memory_order_relaxed) + 7) / 8 * 8 * S::kThreads >= kSoftmaxRegs * 256 + kOtherRegs * 128,
                  "kv16: the attention kernel was built with too few registers");
    }
    launch_dependent(attention_kernel<S>, (unsigned)grid, S::kThreads, S::kSmemBytes, s, a);
    const unsigned blocks = join_blocks<S>(a.by_item ? (int)items : grid), all = blocks + (a.zero_rest ? 4 : 0);
    if (a.by_item)
      launch_dependent(join_kernel<S, 4>, all, 1024, 0, s, a, grid, blocks);
    else
      launch_dependent(join_kernel<S, 1>, all, 256, 0, s, a, grid, blocks);
  });
}
template void launch<KV16_TYPE>(const Params&, bool, int, int, int, int, int, cudaStream_t);
#endif

}  // namespace kv16
}  // namespace xtg
