// Dispatch, sizing and the merging kernel of the chunk attention (the kernel itself: chunk_tcgen05.cuh, one translation unit
// per shape).
#include "common.cuh"
#include "launch.h"

namespace pal {

#define PAL_CHUNK_SHAPES(X) X(32, 16) X(32, 32) X(64, 16) X(64, 32) X(80, 16) X(80, 32) X(96, 16) X(96, 32) X(128, 16) X(128, 32) X(256, 16) X(256, 32)
#define PAL_CHUNK_DECLARE(DD, TT) int launch_chunk_d##DD##_t##TT(const ChunkArgs& a, cudaStream_t stream);
PAL_CHUNK_SHAPES(PAL_CHUNK_DECLARE)
#undef PAL_CHUNK_DECLARE

ChunkPlan chunk_plan(long long total_tokens, int num_q_heads, int num_kv_heads, int head_dim) {
  ChunkPlan c;
  const int group = num_q_heads / num_kv_heads;
  c.tile_heads = group < 128 ? group : 128;
  c.head_blocks = (group + c.tile_heads - 1) / c.tile_heads;
  c.tile_tokens = 128 / c.tile_heads;
  c.grid = cached_sm_count();
  long long rows = (long long)chunk_accumulators(head_dim) * c.tile_tokens;
  if (rows > total_tokens) rows = total_tokens;
  c.part_rows = (int)rows * c.tile_heads;
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  c.ml_offset = up((size_t)c.grid * sizeof(ChunkCut));
  c.acc_offset = c.ml_offset + up((size_t)2 * c.grid * c.part_rows * 2 * sizeof(float));
  c.bytes = c.acc_offset + (size_t)2 * c.grid * c.part_rows * head_dim * sizeof(float);
  return c;
}

namespace {

constexpr int kMergeWarps = 4;

// One block per (border of a share, slice of rows); a warp merges one row at a time, a lane holds 4 elements of each 128.
// Bound: latency.  What a row needs is asked for at once: lanes fetch the (m, l) of 32 parts, one each, and the rows of the
// first eight parts are on the way before the weights are known; few rows need a second trip.  (5 tokens over 1000, 32 / 8 heads of
// 128, eight parts an item: 16.6 us a call, of which 4 in this kernel; four rows a warp, each part asked for when its weight is
// known: 23.5.)
constexpr int kMergeParts = 8;
template <typename T, int NV>  // NV: pieces of 128 elements of a row
__global__ void __launch_bounds__(kMergeWarps * 32) chunk_merge_kernel(const ChunkCut* cuts, const float2* ml,
                                                                       const float* acc, void* out, int out_f32,
                                                                       int part_rows, int tile_heads, int num_q_heads, int head_dim,
                                                                       int rows_per_block) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the attention kernel runs: its results are complete from here
  const ChunkCut c = cuts[blockIdx.x];
  if (c.parts <= 1) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r_end = min((int)(blockIdx.y + 1) * rows_per_block, c.tokens * tile_heads);
  auto slot_of = [&](int k) { return k == 0 ? 2 * (int)blockIdx.x + 1 : 2 * ((int)blockIdx.x + k); };
  for (int r = blockIdx.y * rows_per_block + warp; r < r_end; r += kMergeWarps) {
    const int tok = r / tile_heads, head = r - tok * tile_heads;
    if (head >= c.heads) continue;
    float4 y[kMergeParts][NV];
    auto fetch = [&](int k0) {  // parts k0 .. of this row
#pragma unroll
      for (int u = 0; u < kMergeParts; ++u)
        if (k0 + u < c.parts)
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (i * 128 + lane * 4 < head_dim)
              y[u][i] = *reinterpret_cast<const float4*>(acc + ((size_t)slot_of(k0 + u) * part_rows + r) * head_dim + i * 128 + lane * 4);
    };
    auto stats = [&](int k) { return k < c.parts ? ml[(size_t)slot_of(k) * part_rows + r] : make_float2(-INFINITY, 0.f); };
    const float2 first = stats(lane);
    fetch(0);
    float m = first.x;
    for (int k = lane + 32; k < c.parts; k += 32) m = fmaxf(m, stats(k).x);
#pragma unroll
    for (int sh = 16; sh >= 1; sh >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, sh));
    float den = 0.f;
    float4 x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < c.parts; k0 += 32) {
      const float2 v = k0 == 0 ? first : stats(k0 + lane);
      const float w = v.x > -INFINITY ? fast_exp2(v.x - m) : 0.f;
      den += v.y * w;
      const int count = min(32, c.parts - k0);
      for (int j = 0; j < count; j += kMergeParts) {
        if (k0 + j > 0) fetch(k0 + j);
#pragma unroll
        for (int u = 0; u < kMergeParts; ++u) {
          const float wu = __shfl_sync(0xffffffffu, w, (j + u) & 31);
          if (j + u < count)  // (a part without keys holds zeros; one of no weight may hold an infinity)
#pragma unroll
            for (int i = 0; i < NV; ++i)
              if (i * 128 + lane * 4 < head_dim) {
                x[i].x = fmaf(y[u][i].x, wu, x[i].x);
                x[i].y = fmaf(y[u][i].y, wu, x[i].y);
                x[i].z = fmaf(y[u][i].z, wu, x[i].z);
                x[i].w = fmaf(y[u][i].w, wu, x[i].w);
              }
        }
      }
    }
#pragma unroll
    for (int sh = 16; sh >= 1; sh >>= 1) den += __shfl_xor_sync(0xffffffffu, den, sh);
    const float inv = den == 0.f ? 0.f : 1.f / den;
    const size_t o = ((size_t)(c.row0 + tok) * num_q_heads + c.head0 + head) * head_dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int d = i * 128 + lane * 4;
      if (d >= head_dim) continue;
      if (out_f32)
        *reinterpret_cast<float4*>(static_cast<float*>(out) + o + d) = make_float4(x[i].x * inv, x[i].y * inv, x[i].z * inv, x[i].w * inv);
      else
        *reinterpret_cast<uint2*>(static_cast<T*>(out) + o + d) =
            make_uint2(Mma16816<T>::pack(x[i].x * inv, x[i].y * inv), Mma16816<T>::pack(x[i].z * inv, x[i].w * inv));
    }
  }
}

}  // namespace

int launch_chunk_merge(const ChunkArgs& a, const ChunkPlan& plan, const ChunkCut* cuts, const float* part_ml, const float* part_acc,
                       cudaStream_t stream) {
  // a row a warp up to 64 rows, up to four rows a warp above: sixteen blocks of 128 threads for each SM run at once
  const int slices = min((plan.part_rows + kMergeWarps - 1) / kMergeWarps, 16);
  const int rows_per_block = (plan.part_rows + slices - 1) / slices;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(plan.grid, slices);
  config.blockDim = dim3(kMergeWarps * 32);
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  auto launch = [&](auto kernel) {
    return (int)cudaLaunchKernelEx(&config, kernel, cuts, reinterpret_cast<const float2*>(part_ml), part_acc, a.out, a.out_f32 ? 1 : 0, plan.part_rows,
                                   plan.tile_heads, a.num_q_heads, a.head_dim, rows_per_block);
  };
  if (a.head_dim <= 128) return a.dtype == 0 ? launch(chunk_merge_kernel<__half, 1>) : launch(chunk_merge_kernel<__nv_bfloat16, 1>);
  return a.dtype == 0 ? launch(chunk_merge_kernel<__half, 2>) : launch(chunk_merge_kernel<__nv_bfloat16, 2>);
}

int launch_chunk(const ChunkArgs& a, cudaStream_t stream) {
#define PAL_CHUNK_CALL(DD, TT) \
  if (a.head_dim == DD && a.tokens_per_page == TT) return launch_chunk_d##DD##_t##TT(a, stream);
  PAL_CHUNK_SHAPES(PAL_CHUNK_CALL)
#undef PAL_CHUNK_CALL
  set_error("paged_attention_chunk: no kernel for head_dim=%d tokens_per_page=%d (head_dim in {32,64,80,96,128,256}, tokens_per_page in {16,32})",
            a.head_dim, a.tokens_per_page);
  return -2;
}

}  // namespace pal
