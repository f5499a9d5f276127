// What the two tcgen05 attention kernels (attention_tc.cu over the bf16 cache,
// attention_kv8.cu over the 8-bit one) share: tile sizes, work items, the shape of a
// key-split plan and the kernel that merges the split partials.  Included after CKV_DEFINE_ERR_WORD.
#pragma once

#include "ckv_common.cuh"

namespace ckv {
namespace {

constexpr int BM = 128;  // rows per Q tile (packed token x head)
constexpr int NQ = 2;    // Q tiles per CTA
constexpr int BN = 128;  // keys per tile
constexpr uint32_t ATOM_BYTES = 128 * 128;  // one [128 rows][64 bf16] swizzle-128 atom
constexpr float kRescaleThreshold = 8.0f;   // log2 units

// all lanes wait; the warp agrees on the outcome so collective TMEM ops stay converged
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  const bool ok = mbar_wait(bar, parity, abort, &g_err_word);
  return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = global_ns();
  while (!mbar_try_wait(bar, parity))
    if (global_ns() - t0 > kWaitLimitNs) break;
}

__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Work items: (row block rb, KV head hk, key split z).  Slots come in groups of one
// per (head, row block), row blocks from the last (longest) one down; group gi holds
// split z = n_split - max_splits + gi of the block, so a block's last split, the only
// one shorter than tps key tiles, is in the last group, and the longest blocks' full
// splits come first: roughly longest first over the whole grid.  A slot with z < 0 (a
// block with fewer splits) is empty and skipped.
struct Item {
  int rb, hk, split, n_split, kt0, n_kt, pad0, pad1;  // rb < 0: no more work
};
constexpr int kItemSlots = 4;  // ring of items published by the producer warp
// Epilogue staging: per softmax warp 32 rows x 16 words, rows padded to 20 words (80 B)
// so that the 16-byte writes of eight consecutive lanes fall in distinct banks
constexpr int kStageStride = 20;
constexpr uint32_t kStageBytes = NQ * 4 * 32 * kStageStride * 4;

// Merge the key splits of the row blocks that were split: O = sum_s 2^(m_s - M) O_s /
// sum_s 2^(m_s - M) l_s with M = max_s m_s (all in the log2 domain of the kernel).
// A warp takes R packed rows; for each, lane s reads split s's (m, l), then each lane sums its
// four columns over the splits, the loads of all its rows in flight together.  Rows of
// unsplit blocks were written directly.
constexpr int kCombineWarps = 8;
template <int HD, int R>
__global__ void __launch_bounds__(kCombineWarps * 32, 4) attention_combine_kernel(
    const int32_t* __restrict__ positions, uint16_t* __restrict__ out, int M, int Hq, int Hk, int n_ctx,
    int tps, int max_splits, const float* __restrict__ part_o, const float2* __restrict__ part_ml) {
  pdl_wait();  // the partials come from the attention kernel just before (dependent launch)
  pdl_launch_next();
  const int G = Hq / Hk;
  const int T = BM / G;
  constexpr int kChunks = NQ * BM / (kCombineWarps * R);  // CTAs per (row block, KV head)
  const int rb = blockIdx.x / kChunks, chunk = blockIdx.x - rb * kChunks, hk = blockIdx.y;
  const int t0 = rb * NQ * T;
  const int n_tok = min(NQ * T, M - t0);
  __shared__ int s_max;
  if (threadIdx.x == 0) s_max = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n_tok; i += blockDim.x)
    atomicMax(&s_max, min(max(positions[t0 + i], 0), n_ctx - 1));
  __syncthreads();
  const int n_split = ((s_max + BN) / BN + tps - 1) / tps;
  if (n_split <= 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t stride = NQ * BM;
  const int64_t blk = int64_t((rb * Hk + hk) * max_splits);
  // lane v < HD / 4 takes columns 4v .. 4v + 3: 16-byte half (v & 1) of 8-column chunk
  // v >> 1, stored swapped with the other half when bit 2 of the row is set (the
  // kernel's column-chunk-major partial layout)
  const bool mine = lane < HD / 4;
  float wgt[R], inv[R];
  int off[R];
  int64_t orow[R];
  bool ok[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int pr = (chunk * kCombineWarps + warp) * R + i;
    const int w = pr / BM, r = pr - w * BM;
    const int tr = r / G, g = r - tr * G, tt = w * T + tr;
    ok[i] = r < T * G && tt < n_tok;  // the same for the whole warp
    const float2 ml =
        ok[i] && lane < n_split ? part_ml[blk * stride + pr + lane * stride] : make_float2(-INFINITY, 0.f);
    float mmax = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mmax = fmaxf(mmax, __shfl_xor_sync(0xffffffffu, mmax, o));
    // a split in which the row saw no key has m = -inf: weight 0, also when that is every split
    wgt[i] = ml.x > -INFINITY ? exp2f(ml.x - mmax) : 0.f;
    float L = wgt[i] * ml.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    inv[i] = L > 0.f ? 1.0f / L : 0.f;
    off[i] = w * (BM * HD) + (lane >> 1) * (BM * 8) + r * 8 + (((lane & 1) ^ ((r >> 2) & 1)) << 2);
    orow[i] = (int64_t(t0 + tt) * Hq + hk * G + g) * HD;
  }
  const float* po = part_o + blk * NQ * BM * HD;
  float4 acc[R];
#pragma unroll
  for (int i = 0; i < R; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll(R == 1 ? 4 : 2)
  for (int sp = 0; sp < n_split; ++sp) {
    const float* ps = po + int64_t(sp) * NQ * BM * HD;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float ws = __shfl_sync(0xffffffffu, wgt[i], sp);
      if (mine && ok[i]) {
        const float4 x = *reinterpret_cast<const float4*>(ps + off[i]);
        acc[i].x = fmaf(ws, x.x, acc[i].x);
        acc[i].y = fmaf(ws, x.y, acc[i].y);
        acc[i].z = fmaf(ws, x.z, acc[i].z);
        acc[i].w = fmaf(ws, x.w, acc[i].w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (mine && ok[i])
      *reinterpret_cast<uint2*>(out + orow[i] + 4 * lane) =
          make_uint2(pack_bf2(acc[i].x * inv[i], acc[i].y * inv[i]), pack_bf2(acc[i].z * inv[i], acc[i].w * inv[i]));
}

// One row per warp while the warps of four rows each would not fill the SMs four CTAs deep (7 heads
// over 4: 36 rows over 5371 keys 29.1 -> 22.5 us with the attention, 123 rows 37.9 -> 33, 300 rows
// 51.0 -> 47), then four (938 rows over 5248 keys: 76 us, one row per warp 78).
template <int HD>
void launch_combine(int blocks, const int32_t* positions, uint16_t* out, int M, int Hq, int Hk, int n_ctx, int tps, int max_splits,
                    const float* part_o, const float2* part_ml, cudaStream_t stream) {
  const int64_t ctas = int64_t(blocks) * Hk * (NQ * BM / (kCombineWarps * 4));
  if (ctas < 4 * num_sms())
    launch_pdl(attention_combine_kernel<HD, 1>, dim3(blocks * (NQ * BM / kCombineWarps), Hk), dim3(kCombineWarps * 32), 0, stream,
               positions, out, M, Hq, Hk, n_ctx, tps, max_splits, part_o, part_ml);
  else
    launch_pdl(attention_combine_kernel<HD, 4>, dim3(blocks * (NQ * BM / (kCombineWarps * 4)), Hk), dim3(kCombineWarps * 32), 0, stream,
               positions, out, M, Hq, Hk, n_ctx, tps, max_splits, part_o, part_ml);
}

// Key-split plan: split only when the unsplit grid leaves SMs idle.
struct SplitPlan {
  int tps, max_splits, blocks;
  int64_t bytes;  // partial O and (max, sum) of every split item
};
// The workspace starts with the scheduler's two words (next slot, CTAs done), padded to
// 256 bytes; the split partials follow.
constexpr int64_t kSchedBytes = 256;

}  // namespace
}  // namespace ckv
