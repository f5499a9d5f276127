// Block selection of the sparse attention: a cheap score for every (query token, KV head,
// block of 16 keys), then the `top` best blocks of each (token, KV head), ascending.
//
// With mx_d, mn_d the digest codes (int8) of block b's channel maxima and minima and s_b
// their scale, a_g = max_d |q_gd| and c_gd = rn(fp32(q_gd * fp32(127 / a_g))) the codes of
// query head g:
//   bound_g = sum_d max(c_gd * mx_d, c_gd * mn_d)        (whole number, below 2^21)
//   score_b = fp32( max_g fp32(bound_g * a_g) * s_b )    (the group's best head)
// which bounds q . k over the block from above, up to the 8-bit steps.  Since c * mx >=
// c * mn exactly when c >= 0, the bound is one dot product of length 2D:
// (max(c, 0), min(c, 0)) . (mx, mn), so it runs on the int8 tensor-core path (mma.sync
// m16n8k32: 16 blocks x the up to 8 heads of a group).  Everything that decides the order
// is a whole number or one rounded fp32 product, so a selection is reproducible bit for
// bit; equal scores go to the lower block.
//
// The contraction index may be permuted freely as long as both operands agree: lane quad
// member c takes bytes [c * 2D/4, (c + 1) * 2D/4) of a digest row, so its operands are
// plain 16-byte loads and nothing is shuffled or staged.
#include <algorithm>

#include "ckv_common.cuh"

CKV_DEFINE_ERR_WORD(block_select)

namespace ckv {
namespace {

constexpr int kBlk = CKV_PAGE_TOKENS;
constexpr int kScoreWarps = 8;
constexpr int kTok = 16;  // query tokens per score CTA (they share the digest rows it loads)
constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100
constexpr int kMaxBlocks = 32768;  // keys of one (token, head) held in a CTA's registers
constexpr int kMaxTop = 4096;

// keys of one (token, head): rows of whole 16-byte vectors
__host__ __device__ __forceinline__ int64_t key_stride(int n_blocks) { return (int64_t(n_blocks) + 3) & ~int64_t(3); }

// order-preserving map of an fp32 score to uint32 (-0 first made +0); never 0, which stands for
// no key
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f + 0.0f);
  return max((b & 0x80000000u) ? ~b : (b | 0x80000000u), 1u);
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// a token's position p, clamped to the context (recorded when past it); negative: no key
__device__ __forceinline__ int token_pos(int p, int n_ctx, bool report) {
  if (p >= n_ctx) {
    if (report) atomicOr(&g_err_word, CKV_DEV_ERR_POSITION_RANGE);
    return n_ctx - 1;
  }
  return p < 0 ? -1 : p;
}

// One query head's values, HD / 32 per lane of the warp (packed bf16; zeros for a null row).
template <int HD>
__device__ __forceinline__ void query_load(const uint16_t* src, int lane, uint32_t (&w)[HD / 64]) {
#pragma unroll
  for (int e = 0; e < HD / 64; ++e) w[e] = src == nullptr ? 0u : *reinterpret_cast<const uint32_t*>(src + lane * (HD / 32) + 2 * e);
}
// Their codes into the head's row of shared memory, the positive parts and, HD bytes on, the
// negative ones; returns the largest |q| (NaN left out).
template <int HD>
__device__ __forceinline__ float query_codes(const uint32_t (&w)[HD / 64], uint8_t* row, int lane) {
  constexpr int CH = 2 * HD / 4, CS = CH + 16, E = HD / 32;
  uint32_t pos = 0, neg = 0, mag = 0;
#pragma unroll
  for (int e = 0; e < E / 2; ++e) {
    const uint32_t a = w[e] & 0x7fffu, b = (w[e] >> 16) & 0x7fffu;
    mag = max(mag, max(a > 0x7f80u ? 0u : a, b > 0x7f80u ? 0u : b));
  }
  float amax = __uint_as_float(__reduce_max_sync(0xffffffffu, mag) << 16);
  if (amax < kTiny) amax = 0.f;
  const float inv = amax > 0.f ? __fdiv_rn(127.0f, amax) : 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float f = (e & 1) ? hi_bf(w[e / 2]) : lo_bf(w[e / 2]);
    const int c = max(-127, min(127, __float2int_rn(__fmul_rn(f, inv))));
    pos |= uint32_t(uint8_t(c > 0 ? c : 0)) << (8 * e);
    neg |= uint32_t(uint8_t(c < 0 ? c : 0)) << (8 * e);
  }
  const int i = lane * E, j = HD + lane * E;  // byte offsets in the 2D-long row
  if constexpr (E == 4) {
    *reinterpret_cast<uint32_t*>(row + (i / CH) * CS + i % CH) = pos;
    *reinterpret_cast<uint32_t*>(row + (j / CH) * CS + j % CH) = neg;
  } else {
    *reinterpret_cast<uint16_t*>(row + (i / CH) * CS + i % CH) = uint16_t(pos);
    *reinterpret_cast<uint16_t*>(row + (j / CH) * CS + j % CH) = uint16_t(neg);
  }
  return amax;
}

// CTA: up to kTok tokens of one KV head against a strided set of 16-block tiles.  The
// query codes are made once per CTA in shared memory; a warp then holds one tile's digest
// rows in registers and runs every token of the CTA over them.  Row and chunk strides of
// the codes keep the eight lanes of a 16-byte shared load in distinct banks.  938 rows over 32,896
// tokens, 28 heads over 4: 61 us, bound by issue slots (per 16 blocks and token 8 mma and, to
// reduce and order the result, about as many other instructions as those take).
template <int HD, int NT>
__global__ void __launch_bounds__(kScoreWarps * 32)
    block_score_kernel(const uint16_t* __restrict__ q, const int8_t* __restrict__ dig, const float* __restrict__ dig_scale,
                       const int32_t* __restrict__ positions, int m, int t_begin, int Hq, int Hk, int n_ctx, int n_blocks,
                       uint32_t* __restrict__ keys) {
  constexpr int CH = 2 * HD / 4;            // bytes of a digest row per quad member
  constexpr int CS = CH + 16;               // the same in shared memory
  constexpr int RS = 4 * CS;                // one query head's codes
  constexpr int WORDS = CH / 16;            // 16-byte loads per row and lane
  extern __shared__ __align__(16) uint8_t s_raw[];
  uint8_t* s_code = s_raw;                                               // [kTok][NT * 8][RS]
  float* s_amax = reinterpret_cast<float*>(s_raw + kTok * NT * 8 * RS);  // [kTok][NT * 8]
  __shared__ int s_nb[kTok];
  const int G = Hq / Hk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.y;
  // the last tokens first: they usually see the most blocks
  const int t0 = t_begin + int(gridDim.z - 1 - blockIdx.z) * kTok;
  const int n_tok = min(kTok, t_begin + m - t0);
  pdl_wait();
  pdl_launch_next();
  if (threadIdx.x < kTok)
    s_nb[threadIdx.x] = threadIdx.x < n_tok
                            ? (token_pos(positions[t0 + threadIdx.x], n_ctx, hk == 0 && blockIdx.x == 0) + kBlk) / kBlk
                            : 0;
  // query codes: a warp per (token, head) row, the loads of four rows in flight together
  constexpr int R = 4;
  for (int r0 = warp; r0 < n_tok * NT * 8; r0 += kScoreWarps * R) {
    uint32_t w[R][HD / 64];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int r = r0 + u * kScoreWarps, t = r / (NT * 8), g = r - t * (NT * 8);
      query_load<HD>(t < n_tok && g < G ? q + (int64_t(t0 + t) * Hq + hk * G + g) * HD : nullptr, lane, w[u]);
    }
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int r = r0 + u * kScoreWarps;
      if (r >= n_tok * NT * 8) break;
      const float amax = query_codes<HD>(w[u], s_code + r * RS, lane);
      if (lane == 0) s_amax[r] = amax;
    }
  }
  __syncthreads();
  int nb_max = 0;
#pragma unroll
  for (int t = 0; t < kTok; ++t) nb_max = max(nb_max, s_nb[t]);
  const int gr = lane >> 2, qd = lane & 3;
  const int tiles = (nb_max + 15) / 16;
  for (int tile = blockIdx.x * kScoreWarps + warp; tile < tiles; tile += gridDim.x * kScoreWarps) {
    const int b0 = tile * 16;
    uint4 a[2][WORDS];  // digest rows b0 + gr and b0 + gr + 8, this lane's chunk
    float sc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int b = min(b0 + gr + 8 * i, n_blocks - 1);
      const int64_t row = int64_t(hk) * n_blocks + b;
#pragma unroll
      for (int w = 0; w < WORDS; ++w) a[i][w] = __ldg(reinterpret_cast<const uint4*>(dig + row * 2 * HD + qd * CH) + w);
      sc[i] = __ldg(dig_scale + row);
    }
    // two tokens at a time: independent chains of mma and reductions
    for (int t = 0; t < n_tok; t += 2) {
      const bool see[2] = {b0 < s_nb[t], t + 1 < n_tok && b0 < s_nb[t + 1]};
      if (!see[0] && !see[1]) continue;  // nothing of this tile is visible to the tokens
      const int tt[2] = {t, min(t + 1, n_tok - 1)};
      float best[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) best[u][0] = best[u][1] = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        int c[2][4] = {};
#pragma unroll
        for (int w = 0; w < WORDS; ++w)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint4 b = *reinterpret_cast<const uint4*>(s_code + ((tt[u] * NT + nt) * 8 + gr) * RS + qd * CS + 16 * w);
            mma_s8(c[u], a[0][w].x, a[1][w].x, a[0][w].y, a[1][w].y, b.x, b.y);
            mma_s8(c[u], a[0][w].z, a[1][w].z, a[0][w].w, a[1][w].w, b.z, b.w);
          }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float* am = s_amax + (tt[u] * NT + nt) * 8 + 2 * qd;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (nt * 8 + 2 * qd + e < G) {
              best[u][0] = fmaxf(best[u][0], __fmul_rn(float(c[u][e]), am[e]));
              best[u][1] = fmaxf(best[u][1], __fmul_rn(float(c[u][2 + e]), am[e]));
            }
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) best[u][e] = fmaxf(best[u][e], __shfl_xor_sync(0xffffffffu, best[u][e], o));
      // lane qd = 2u + e writes token u's key of block b0 + gr + 8e
      const int u = qd >> 1, b = b0 + gr + 8 * (qd & 1);
      const float top = qd == 0 ? best[0][0] : qd == 1 ? best[0][1] : qd == 2 ? best[1][0] : best[1][1];
      if ((u ? see[1] : see[0]) && b < n_blocks)
        keys[(int64_t(t0 - t_begin + t + u) * Hk + hk) * key_stride(n_blocks) + b] =
            order_key(__fmul_rn(top, (qd & 1) ? sc[1] : sc[0]));
    }
  }
}

struct TopArgs {
  const uint32_t* keys;  // [m][Hk][key_stride(n_blocks)], tokens from t_begin on
  const int32_t* positions;
  int32_t* out;  // [..][Hk][top]
  int m, t_begin, Hk, n_ctx, n_blocks, top, sink, recent;
};

// Sums over the group (a warp, or the CTA: partial sums alternate between two shared rows, so
// one barrier per sum is enough).
template <int T>
__device__ __forceinline__ int2 group_sum(int2 v, int2 (*s_part)[32], int& flip) {
  v.x = __reduce_add_sync(0xffffffffu, v.x);
  v.y = __reduce_add_sync(0xffffffffu, v.y);
  if constexpr (T > 32) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2* row = s_part[flip];
    flip ^= 1;
    if (lane == 0) row[warp] = v;
    __syncthreads();
    v = lane < T / 32 ? row[lane] : make_int2(0, 0);
    v.x = __reduce_add_sync(0xffffffffu, v.x);
    v.y = __reduce_add_sync(0xffffffffu, v.y);
  }
  return v;
}

// What the group's threads before this one hold together, and the whole sum.
template <int T>
__device__ __forceinline__ int exclusive_scan(int n, int (*s_mm)[32], int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  total = __shfl_sync(0xffffffffu, x, 31);
  if constexpr (T > 32) {
    __syncthreads();  // s_mm was last read before
    if (lane == 31) s_mm[0][warp] = x;
    __syncthreads();
    const int v = lane < T / 32 ? s_mm[0][lane] : 0;
    x += __reduce_add_sync(0xffffffffu, lane < warp ? v : 0);
    total = __reduce_add_sync(0xffffffffu, v);
  }
  return x - n;
}

// The largest value that at least `need` of the group's values reach (0: absent; at least
// `need` are present), built two bits at a time from the first bit in which they differ, by
// counting the values at or above three trial values: no atomics, an order that never varies.
// Stops as soon as a trial value is reached by exactly `need` values (then true).
template <int T, int N>
__device__ __forceinline__ bool kth_largest(const uint32_t (&v)[N], int n, int need, uint32_t& thr, int2 (*s_part)[32],
                                            int (*s_mm)[32], int& flip) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t hi_v = 0, lo_v = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n && v[i] != 0) {
      hi_v = max(hi_v, v[i]);
      lo_v = min(lo_v, v[i]);
    }
  hi_v = __reduce_max_sync(0xffffffffu, hi_v);
  lo_v = __reduce_min_sync(0xffffffffu, lo_v);
  if constexpr (T > 32) {
    __syncthreads();
    if (lane == 0) {
      s_mm[0][warp] = int(hi_v);
      s_mm[1][warp] = int(lo_v);
    }
    __syncthreads();
    hi_v = __reduce_max_sync(0xffffffffu, lane < T / 32 ? uint32_t(s_mm[0][lane]) : 0u);
    lo_v = __reduce_min_sync(0xffffffffu, lane < T / 32 ? uint32_t(s_mm[1][lane]) : 0xffffffffu);
  }
  if (hi_v == lo_v) {
    thr = hi_v;
    return false;
  }
  const int low0 = (31 - __clz(hi_v ^ lo_v)) & ~1;  // the pair of bits that the first difference lies in
  thr = low0 == 30 ? 0u : (hi_v >> (low0 + 2)) << (low0 + 2);
  for (int low = low0; low >= 0; low -= 2) {
    const uint32_t t1 = thr | (1u << low), t2 = thr | (2u << low), t3 = thr | (3u << low);
    int c1 = 0, c2 = 0, c3 = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) {
        c1 += v[i] >= t1;
        c2 += v[i] >= t2;
        c3 += v[i] >= t3;
      }
    const int2 c = group_sum<T>(make_int2(c1 | (c2 << 16), c3), s_part, flip);
    c1 = c.x & 0xffff, c2 = int(uint32_t(c.x) >> 16), c3 = c.y;
    int reached = -1;
    if (c3 >= need) thr = t3, reached = c3;
    else if (c2 >= need) thr = t2, reached = c2;
    else if (c1 >= need) thr = t1, reached = c1;
    if (reached == need) return true;
  }
  return false;
}

// The `top` blocks of one (token, head): T threads, thread t holding the KPT consecutive
// keys from t * KPT on.  The K-th largest key is searched among few values: the K-th largest
// of the maxima of groups of four keys is a lower bound for it that few more than K keys
// reach; those are gathered and searched.  Only where that does not apply (fewer groups than
// K, or too many keys at or above the bound, which takes ties) every key is counted.
// `load(b)` gives the keys of blocks b .. b + 3.  The 3752 selections of 64 among up to 2056 blocks (938
// rows, 4 heads) take 39 us, a chain of counting rounds each; one selection in a CTA, 3 to 5 us.
template <int T, int KPT, typename Load>
__device__ __forceinline__ void select_top(const TopArgs& a, int nb, int32_t* out, Load load) {
  constexpr int kGroups = T > 32 ? 1 : 8;  // (token, head) pairs per CTA
  constexpr int kFew = T > 512 ? T : T > 32 ? 512 : 128;  // gathered keys at most
  constexpr int GM = KPT / 4;
  __shared__ int2 s_part[2][32];
  __shared__ int s_mm[2][32];
  __shared__ uint32_t s_few[kGroups][kFew];
  const int t = T > 32 ? int(threadIdx.x) : int(threadIdx.x & 31);
  const int grp = T > 32 ? 0 : int(threadIdx.x >> 5);
  auto group_barrier = [] {
    if constexpr (T > 32) __syncthreads();
    else __syncwarp();
  };
  if (nb <= a.top) {  // every visible block
    for (int i = t; i < a.top; i += T) out[i] = i < nb ? i : -1;
    return;
  }
  // candidates: blocks in [sink, nb - recent); the others are taken (below nb) or absent
  const int lo_b = a.sink, hi_b = nb - a.recent;
  const int need = a.top - a.sink - a.recent;
  const int first = t * KPT;
  uint32_t k[KPT];
#pragma unroll
  for (int i = 0; i < KPT; i += 4) {
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (first + i < hi_b) x = load(first + i);
    k[i] = x.x, k[i + 1] = x.y, k[i + 2] = x.z, k[i + 3] = x.w;
  }
#pragma unroll
  for (int i = 0; i < KPT; ++i)
    if (first + i < lo_b || first + i >= hi_b) k[i] = 0u;
  int flip = 0;
  uint32_t thr = 0xffffffffu;  // keys above it are taken, and the first `ties` equal to it
  int ties = 0;
  bool exact = false;  // every key at or above thr is taken
  if (need > 0) {
    bool found = false;
    if ((hi_b - lo_b) / 4 - 1 >= need) {  // at least `need` whole groups
      uint32_t gm[GM], bound;
#pragma unroll
      for (int i = 0; i < GM; ++i) gm[i] = max(max(k[4 * i], k[4 * i + 1]), max(k[4 * i + 2], k[4 * i + 3]));
      kth_largest<T, GM>(gm, GM, need, bound, s_part, s_mm, flip);
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < KPT; ++i)
        if (k[i] >= bound) m |= 1u << i;
      // places by a scan of the counts (atomics on one counter would queue up)
      int c, at = exclusive_scan<T>(__popc(m), s_mm, c);
#pragma unroll
      for (int i = 0; i < KPT; ++i)
        if ((m >> i) & 1) {
          if (at < kFew) s_few[grp][at] = k[i];
          ++at;
        }
      group_barrier();
      if (c <= kFew) {
        uint32_t few[kFew / T];
#pragma unroll
        for (int i = 0; i < kFew / T; ++i) few[i] = t + i * T < c ? s_few[grp][t + i * T] : 0u;
        exact = c == need;
        thr = bound;
        if (!exact) exact = kth_largest<T, kFew / T>(few, (c + T - 1) / T, need, thr, s_part, s_mm, flip);
        found = true;
      }
    }
    if (!found) exact = kth_largest<T, KPT>(k, KPT, need, thr, s_part, s_mm, flip);
  }
  // blocks taken for sure and blocks whose key equals thr, as bits of this thread's keys
  uint32_t sure_m = 0, tie_m = 0;
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    if (k[i] > thr) sure_m |= 1u << i;
    if (k[i] == thr) tie_m |= 1u << i;
  }
  if (need <= 0) sure_m = tie_m = 0;
  if (exact) sure_m |= tie_m, tie_m = 0;
  // the first `sink` blocks and the last `recent` visible ones (their keys are 0)
  auto below = [&](int end) -> uint32_t {  // bits of this thread's blocks below `end`
    const int n = max(0, min(KPT, end - first));
    return n >= 32 ? 0xffffffffu : (1u << n) - 1;
  };
  const uint32_t forced = below(lo_b) | (below(nb) & ~below(hi_b));
  sure_m = (sure_m & ~forced) | forced;
  tie_m &= ~forced;
  int above = 0;
  if (!exact && need > 0) {
    above = group_sum<T>(make_int2(__popc(sure_m & ~forced), 0), s_part, flip).x;
    ties = need - above;
  }
  int total;
  // both counts in one scan (at most 32768 each)
  const uint32_t before = uint32_t(exclusive_scan<T>(__popc(sure_m) | (__popc(tie_m) << 16), s_mm, total));
  int sure = before & 0xffff, tie = before >> 16;  // taken for sure, and ties, before this thread's blocks
  // ascending: a block's place is what was taken before it
  for (uint32_t both = sure_m | tie_m; both != 0; both &= both - 1) {
    const uint32_t bit = both & (0u - both);
    bool take = true;
    const int at = sure + min(tie, ties);
    if (tie_m & bit) {
      take = tie < ties;
      ++tie;
    } else {
      ++sure;
    }
    if (take && at < a.top) out[at] = first + 31 - __clz(bit);
  }
}

// A warp (T = 32) or a CTA per (token, head), its keys in the workspace.
template <int T, int KPT>
__global__ void __launch_bounds__(T > 32 ? T : 256) block_top_kernel(const __grid_constant__ TopArgs a) {
  pdl_wait();
  pdl_launch_next();
  const int64_t id = T > 32 ? int64_t(blockIdx.x) : int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (id >= int64_t(a.m) * a.Hk) return;  // the whole group
  const int tok = a.t_begin + int(id / a.Hk);
  const int nb = (token_pos(a.positions[tok], a.n_ctx, false) + kBlk) / kBlk;
  const uint32_t* keys = a.keys + id * key_stride(a.n_blocks);
  select_top<T, KPT>(a, nb, a.out + (int64_t(tok) * a.Hk + id % a.Hk) * a.top,
                     [&](int b) { return __ldcg(reinterpret_cast<const uint4*>(keys + b)); });
}

// Scores and selection of few (token, head) pairs in one launch: a cluster of kCluster CTAs
// scores the blocks of one pair, every key going straight into the first CTA's shared memory,
// and that CTA selects.
constexpr int kCluster = 8;
template <int HD, int NT, int KPT>
__global__ void __launch_bounds__(256)
    block_select_cluster_kernel(const uint16_t* __restrict__ q, const int8_t* __restrict__ dig, const float* __restrict__ dig_scale,
                                int Hq, const __grid_constant__ TopArgs a) {
  constexpr int CH = 2 * HD / 4, CS = CH + 16, RS = 4 * CS, WORDS = CH / 16;
  __shared__ __align__(16) uint8_t s_code[NT * 8 * RS];
  __shared__ float s_amax[NT * 8];
  __shared__ __align__(16) uint32_t s_keys[256 * KPT];
  const int G = Hq / a.Hk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x, tok = blockIdx.y, hk = blockIdx.z;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA has started
  pdl_wait();
  pdl_launch_next();
  // everything that does not wait for something else is requested first: the position, the
  // first tile's digest rows (visible or not) and q
  const int p = a.positions[tok];
  const int gr = lane >> 2, qd = lane & 3;
  uint4 nd[2][WORDS];  // digest rows b0 + gr and b0 + gr + 8 of the next tile, this lane's chunk
  float nsc[2];
  auto load = [&](int tile) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t row = int64_t(hk) * a.n_blocks + min(tile * 16 + gr + 8 * i, a.n_blocks - 1);
#pragma unroll
      for (int w = 0; w < WORDS; ++w) nd[i][w] = __ldg(reinterpret_cast<const uint4*>(dig + row * 2 * HD + qd * CH) + w);
      nsc[i] = __ldg(dig_scale + row);
    }
  };
  load(rank * 8 + warp);
  for (int g = warp; g < NT * 8; g += 8) {
    uint32_t w[HD / 64];
    query_load<HD>(g < G ? q + (int64_t(tok) * Hq + hk * G + g) * HD : nullptr, lane, w);
    const float amax = query_codes<HD>(w, s_code + g * RS, lane);
    if (lane == 0) s_amax[g] = amax;
  }
  const int nb = (token_pos(p, a.n_ctx, hk == 0 && rank == 0) + kBlk) / kBlk;
  const int tiles = (nb + 15) / 16;
  const bool all = nb <= a.top;  // no choice to make
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // and so has the first one
  const uint32_t keys0 = cluster_smem_addr(s_keys, 0);
  for (int tile = rank * 8 + warp; tile < tiles && !all; tile += kCluster * 8) {
    const int b0 = tile * 16;
    uint4 d[2][WORDS];
    float sc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int w = 0; w < WORDS; ++w) d[i][w] = nd[i][w];
      sc[i] = nsc[i];
    }
    if (tile + kCluster * 8 < tiles) load(tile + kCluster * 8);
    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      int c[4] = {}, c2[4] = {};  // two chains
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        const uint4 b = *reinterpret_cast<const uint4*>(s_code + (nt * 8 + gr) * RS + qd * CS + 16 * w);
        mma_s8(c, d[0][w].x, d[1][w].x, d[0][w].y, d[1][w].y, b.x, b.y);
        mma_s8(c2, d[0][w].z, d[1][w].z, d[0][w].w, d[1][w].w, b.z, b.w);
      }
      const float* am = s_amax + nt * 8 + 2 * qd;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (nt * 8 + 2 * qd + e < G) {
          best[0] = fmaxf(best[0], __fmul_rn(float(c[e] + c2[e]), am[e]));
          best[1] = fmaxf(best[1], __fmul_rn(float(c[2 + e] + c2[2 + e]), am[e]));
        }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      best[0] = fmaxf(best[0], __shfl_xor_sync(0xffffffffu, best[0], o));
      best[1] = fmaxf(best[1], __shfl_xor_sync(0xffffffffu, best[1], o));
    }
    if (qd < 2) {
      const int b = b0 + gr + 8 * qd;
      const uint32_t key = order_key(__fmul_rn(qd ? best[1] : best[0], qd ? sc[1] : sc[0]));
      if (b < a.n_blocks) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(keys0 + 4u * b), "r"(key) : "memory");
    }
  }
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  if (rank != 0) return;
  select_top<256, KPT>(a, nb, a.out + (int64_t(tok) * a.Hk + hk) * a.top,
                       [&](int b) { return *reinterpret_cast<const uint4*>(s_keys + b); });
}

template <int HD, int NT, int KPT>
int launch_cluster(const uint16_t* q, const int8_t* dig, const float* dig_scale, int Hq, const TopArgs& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCluster, a.m, a.Hk);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, block_select_cluster_kernel<HD, NT, KPT>, q, dig, dig_scale, Hq, a);
  CKV_LAUNCH_CHECK("ckv_block_select(cluster)");
  return CKV_OK;
}

template <int HD, int NT>
int launch_few(const uint16_t* q, const int8_t* dig, const float* dig_scale, int Hq, const TopArgs& a, cudaStream_t stream) {
  if (a.n_blocks <= 1024) return launch_cluster<HD, NT, 4>(q, dig, dig_scale, Hq, a, stream);
  return launch_cluster<HD, NT, 16>(q, dig, dig_scale, Hq, a, stream);
}

// Few pairs and contexts up to 65,536 tokens take one launch of clusters, and no workspace.  One row,
// 4 heads: 6.0 / 8.0 / 9.2 us over 16,384 / 32,896 / 65,536 tokens against 7.6 / 8.9 / 8.9 us and a
// launch more; over 131,072 tokens with 8 heads the clusters' 64 SMs take 20 us, two kernels 15.
bool use_cluster(int m, int Hk, int n_blocks) { return int64_t(m) * Hk <= 32 && n_blocks <= 4096; }

template <int HD, int NT>
int launch_score(const uint16_t* q, const int8_t* dig, const float* dig_scale, const int32_t* positions, int m, int t_begin,
                 int Hq, int Hk, int n_ctx, int n_blocks, uint32_t* keys, cudaStream_t stream) {
  constexpr int smem = kTok * NT * 8 * (4 * (2 * HD / 4 + 16) + 4);
  auto kern = block_score_kernel<HD, NT>;
  if (int rc = set_smem_limit(reinterpret_cast<const void*>(kern), smem)) return rc;
  const int groups = ceil_div(m, kTok);
  // about three CTAs per SM, no more than there are tiles: each makes its tokens' codes (938 rows over
  // 32,896 tokens: selection 96 us, with twelve 117; 100 rows over 131,072: 64, with two or six 77 and 67)
  const int tiles = ceil_div(n_blocks, 16);
  const int x = std::max(1, std::min(ceil_div(tiles, kScoreWarps), ceil_div(3 * num_sms(), int64_t(groups) * Hk)));
  launch_pdl(kern, dim3(x, Hk, groups), dim3(kScoreWarps * 32), smem, stream, q, dig, dig_scale, positions, m, t_begin, Hq,
             Hk, n_ctx, n_blocks, keys);
  CKV_LAUNCH_CHECK("ckv_block_select(score)");
  return CKV_OK;
}

template <int T, int KPT>
int launch_top(const TopArgs& a, cudaStream_t stream) {
  const int64_t ids = int64_t(a.m) * a.Hk;
  launch_pdl(block_top_kernel<T, KPT>, dim3(unsigned(T > 32 ? ids : (ids + 7) / 8)), dim3(T > 32 ? T : 256), 0, stream, a);
  CKV_LAUNCH_CHECK("ckv_block_select(top)");
  return CKV_OK;
}

// tokens whose keys the workspace holds at once: all of them, or as many as 256 MB take
int64_t chunk_tokens(int m, int Hk, int n_blocks) {
  const int64_t per = int64_t(Hk) * key_stride(n_blocks) * 4;
  return std::min<int64_t>(m, std::max<int64_t>(kTok, (int64_t(256) << 20) / per / kTok * kTok));
}

bool select_shape_ok(int m, int Hq, int Hk, int HD, int n_ctx) {
  return m >= 0 && Hk > 0 && Hk <= 65535 && Hq > 0 && Hq % Hk == 0 && Hq / Hk <= 16 && (HD == 64 || HD == 128) && n_ctx > 0 &&
         ceil_div(n_ctx, kBlk) <= kMaxBlocks;
}

}  // namespace
}  // namespace ckv

using namespace ckv;

extern "C" int64_t ckv_block_select_workspace_size(int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx) {
  if (!select_shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) return 0;
  const int nb = ceil_div(n_ctx, kBlk);
  if (m > 0 && use_cluster(m, n_kv_heads, nb)) return 0;
  return chunk_tokens(m, n_kv_heads, nb) * n_kv_heads * key_stride(nb) * 4;
}

extern "C" int ckv_block_select_launches(int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx) {
  if (m <= 0 || !select_shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) return 0;
  if (use_cluster(m, n_kv_heads, ceil_div(n_ctx, kBlk))) return 1;
  return 2 * ceil_div(m, chunk_tokens(m, n_kv_heads, ceil_div(n_ctx, kBlk)));
}

namespace ckv {
// Everything that ckv_block_select refuses, without a launch (also asked by ckv_attention_sparse(_kv8)
// before their first one).
int block_select_check(const uint16_t* q, const int8_t* dig_codes, const float* dig_scale, const int32_t* positions,
                       const int32_t* blocks, int m, int Hq, int Hk, int HD, int n_ctx, int top, int sink, int recent,
                       const void* workspace, int64_t workspace_bytes) {
  CKV_REQUIRE(m >= 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0 && n_ctx > 0, "ckv_block_select: bad sizes");
  CKV_REQUIRE(sink >= 0 && recent >= 1 && top >= 1 && int64_t(sink) + recent <= top && top <= kMaxTop,
              "ckv_block_select: top %d (1 to %d) must hold the %d first and %d last blocks (at least one last)", top,
              kMaxTop, sink, recent);
  if (!select_shape_ok(m, Hq, Hk, HD, n_ctx)) {
    set_error("ckv_block_select: head_dim %d (64 or 128), %d query heads per KV head (at most 16), context %d (at most %d)", HD,
              Hq / Hk, n_ctx, kMaxBlocks * kBlk);
    return CKV_ERR_UNSUPPORTED;
  }
  if (m == 0) return CKV_OK;
  const int nb = ceil_div(n_ctx, kBlk);
  const bool few = use_cluster(m, Hk, nb);
  CKV_REQUIRE(q && dig_codes && dig_scale && positions && blocks && (few || workspace), "ckv_block_select: null pointer");
  CKV_REQUIRE(aligned16(q) && aligned16(dig_codes) && (few || aligned16(workspace)),
              "ckv_block_select: tensors must be 16-byte aligned");
  if (few) return CKV_OK;
  const int64_t need = chunk_tokens(m, Hk, nb) * Hk * key_stride(nb) * 4;
  CKV_REQUIRE(workspace_bytes >= need, "ckv_block_select: workspace of %lld bytes, needs %lld",
              static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  CKV_REQUIRE(m <= 1000000 && int64_t(m) * Hk < (int64_t(1) << 31) - 8, "ckv_block_select: too many rows");
  return CKV_OK;
}
}  // namespace ckv

extern "C" int ckv_block_select(const uint16_t* q, const int8_t* dig_codes, const float* dig_scale,
                                const int32_t* positions, int32_t* blocks, int m, int n_q_heads, int n_kv_heads,
                                int head_dim, int n_ctx, int top, int sink, int recent, void* workspace,
                                int64_t workspace_bytes, ckv_stream_t stream) {
  if (int rc = block_select_check(q, dig_codes, dig_scale, positions, blocks, m, n_q_heads, n_kv_heads, head_dim, n_ctx, top, sink,
                                  recent, workspace, workspace_bytes))
    return rc;
  if (m == 0) return CKV_OK;
  const int nb = ceil_div(n_ctx, kBlk);
  const bool few = use_cluster(m, n_kv_heads, nb);
  if (few) {
    const TopArgs a{nullptr, positions, blocks, m, 0, n_kv_heads, n_ctx, nb, top, sink, recent};
    const cudaStream_t s = as_stream(stream);
    if (head_dim == 128)
      return n_q_heads / n_kv_heads > 8 ? launch_few<128, 2>(q, dig_codes, dig_scale, n_q_heads, a, s)
                                        : launch_few<128, 1>(q, dig_codes, dig_scale, n_q_heads, a, s);
    return n_q_heads / n_kv_heads > 8 ? launch_few<64, 2>(q, dig_codes, dig_scale, n_q_heads, a, s)
                                      : launch_few<64, 1>(q, dig_codes, dig_scale, n_q_heads, a, s);
  }
  const int64_t step = chunk_tokens(m, n_kv_heads, nb);
  const cudaStream_t s = as_stream(stream);
  uint32_t* keys = static_cast<uint32_t*>(workspace);
  for (int64_t t = 0; t < m; t += step) {
    const int n = int(std::min<int64_t>(step, m - t));
    const bool two = n_q_heads / n_kv_heads > 8;
    int rc;
    if (head_dim == 128)
      rc = two ? launch_score<128, 2>(q, dig_codes, dig_scale, positions, n, int(t), n_q_heads, n_kv_heads, n_ctx, nb, keys, s)
               : launch_score<128, 1>(q, dig_codes, dig_scale, positions, n, int(t), n_q_heads, n_kv_heads, n_ctx, nb, keys, s);
    else
      rc = two ? launch_score<64, 2>(q, dig_codes, dig_scale, positions, n, int(t), n_q_heads, n_kv_heads, n_ctx, nb, keys, s)
               : launch_score<64, 1>(q, dig_codes, dig_scale, positions, n, int(t), n_q_heads, n_kv_heads, n_ctx, nb, keys, s);
    if (rc) return rc;
    const TopArgs a{keys, positions, blocks, n, int(t), n_kv_heads, n_ctx, nb, top, sink, recent};
    // a warp per (token, head) while its keys fit the warp's registers, then 128 threads (938 rows
    // over 32,896 tokens: 39 us, with 256 threads 9 us more) and more
    if (nb <= 512) rc = launch_top<32, 16>(a, s);
    else if (nb <= 1024) rc = launch_top<32, 32>(a, s);
    else if (nb <= 4096) rc = launch_top<128, 32>(a, s);
    else if (nb <= 8192) rc = launch_top<256, 32>(a, s);
    else rc = launch_top<1024, 32>(a, s);
    if (rc) return rc;
  }
  return CKV_OK;
}
