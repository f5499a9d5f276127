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
constexpr int kMaxBlocks = 49152;  // keys of one (token, head) held in shared memory
constexpr int kMaxTop = 4096;

// order-preserving map of an fp32 score to uint32 (-0 first made +0)
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// position of a token, clamped to the context (recorded when past it); negative: no key
__device__ __forceinline__ int token_pos(const int32_t* positions, int t, int n_ctx, bool report) {
  const int p = positions[t];
  if (p >= n_ctx) {
    if (report) atomicOr(&g_err_word, CKV_DEV_ERR_POSITION_RANGE);
    return n_ctx - 1;
  }
  return p < 0 ? -1 : p;
}

// CTA: up to kTok tokens of one KV head against a strided set of 16-block tiles.  The
// query codes are made once per CTA in shared memory; a warp then holds one tile's digest
// rows in registers and runs every token of the CTA over them.  Row and chunk strides of
// the codes keep the eight lanes of a 16-byte shared load in distinct banks.
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
  const int hk = blockIdx.z;
  const int t0 = t_begin + blockIdx.y * kTok;
  const int n_tok = min(kTok, t_begin + m - t0);
  pdl_wait();
  pdl_launch_next();
  if (threadIdx.x < kTok)
    s_nb[threadIdx.x] = threadIdx.x < n_tok
                            ? (token_pos(positions, t0 + threadIdx.x, n_ctx, hk == 0 && blockIdx.x == 0) + kBlk) / kBlk
                            : 0;
  // query codes: a warp per (token, head) row, HD / 32 values per lane
  for (int r = warp; r < n_tok * NT * 8; r += kScoreWarps) {
    const int t = r / (NT * 8), g = r - t * (NT * 8);
    constexpr int E = HD / 32;
    uint32_t pos = 0, neg = 0;  // E codes, the positive and the negative part
    float amax = 0.f;
    if (g < G) {
      const uint16_t* src = q + (int64_t(t0 + t) * Hq + hk * G + g) * HD + lane * E;
      float f[E];
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(src + e);
        f[e] = lo_bf(w);
        f[e + 1] = hi_bf(w);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) amax = fmaxf(amax, fabsf(f[e]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (amax < kTiny) amax = 0.f;
      const float inv = amax > 0.f ? __fdiv_rn(127.0f, amax) : 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = max(-127, min(127, __float2int_rn(__fmul_rn(f[e], inv))));
        pos |= uint32_t(uint8_t(c > 0 ? c : 0)) << (8 * e);
        neg |= uint32_t(uint8_t(c < 0 ? c : 0)) << (8 * e);
      }
    }
    uint8_t* row = s_code + r * RS;
    const int i = lane * E, j = HD + lane * E;  // byte offsets in the 2D-long row
    if constexpr (E == 4) {
      *reinterpret_cast<uint32_t*>(row + (i / CH) * CS + i % CH) = pos;
      *reinterpret_cast<uint32_t*>(row + (j / CH) * CS + j % CH) = neg;
    } else {
      *reinterpret_cast<uint16_t*>(row + (i / CH) * CS + i % CH) = uint16_t(pos);
      *reinterpret_cast<uint16_t*>(row + (j / CH) * CS + j % CH) = uint16_t(neg);
    }
    if (lane == 0) s_amax[r] = amax;
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
    for (int t = 0; t < n_tok; ++t) {
      if (b0 >= s_nb[t]) continue;  // nothing of this tile is visible to the token
      float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        int c[4] = {0, 0, 0, 0};
        const uint8_t* row = s_code + ((t * NT + nt) * 8 + gr) * RS + qd * CS;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
          const uint4 b = *reinterpret_cast<const uint4*>(row + 16 * w);
          mma_s8(c, a[0][w].x, a[1][w].x, a[0][w].y, a[1][w].y, b.x, b.y);
          mma_s8(c, a[0][w].z, a[1][w].z, a[0][w].w, a[1][w].w, b.z, b.w);
        }
        const float* am = s_amax + (t * NT + nt) * 8 + 2 * qd;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (nt * 8 + 2 * qd + e < G) {
            best[0] = fmaxf(best[0], __fmul_rn(float(c[e]), am[e]));
            best[1] = fmaxf(best[1], __fmul_rn(float(c[2 + e]), am[e]));
          }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        best[0] = fmaxf(best[0], __shfl_xor_sync(0xffffffffu, best[0], o));
        best[1] = fmaxf(best[1], __shfl_xor_sync(0xffffffffu, best[1], o));
      }
      if (qd < 2) {
        const int b = b0 + gr + 8 * qd;
        if (b < n_blocks)
          keys[(int64_t(t0 - t_begin + t) * Hk + hk) * n_blocks + b] = order_key(__fmul_rn(best[qd], sc[qd]));
      }
    }
  }
}

struct TopArgs {
  const uint32_t* keys;  // [m][Hk][n_blocks], tokens from t_begin on
  const int32_t* positions;
  int32_t* out;  // [..][Hk][top]
  int m, t_begin, Hk, n_ctx, n_blocks, top, sink, recent;
};

// count over the group (a warp, or the CTA: partial sums alternate between two shared rows,
// so one barrier per count is enough)
template <int T>
__device__ __forceinline__ int group_sum(int v, int (*s_part)[32], int& flip) {
  v = __reduce_add_sync(0xffffffffu, v);
  if constexpr (T > 32) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int* row = s_part[flip];
    flip ^= 1;
    if (lane == 0) row[warp] = v;
    __syncthreads();
    v = __reduce_add_sync(0xffffffffu, lane < T / 32 ? row[lane] : 0);
  }
  return v;
}

// The `top` blocks of one (token, head): T threads, thread t holding the KPT consecutive
// keys from t * KPT on (KPT = 0: the keys stay in shared memory, any number of them).  The
// K-th largest key is built bit by bit from the top by counting the keys at or above a
// trial value: no atomics, an order that never varies, and it stops as soon as a trial value
// is reached by exactly K keys.
template <int T, int KPT>
__global__ void __launch_bounds__(T > 32 ? T : 256) block_top_kernel(const __grid_constant__ TopArgs a) {
  constexpr int kGroups = T > 32 ? 1 : 8;  // (token, head) pairs per CTA
  extern __shared__ uint32_t s_keys[];
  __shared__ int s_part[2][32];
  __shared__ int s_scan[32];
  __shared__ int s_scan2[32];
  const int t = T > 32 ? int(threadIdx.x) : int(threadIdx.x & 31);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t id = int64_t(blockIdx.x) * kGroups + (T > 32 ? 0 : warp);
  pdl_wait();
  pdl_launch_next();
  if (id >= int64_t(a.m) * a.Hk) return;
  const int tok = a.t_begin + int(id / a.Hk), hk = int(id % a.Hk);
  const int nb = (token_pos(a.positions, tok, a.n_ctx, false) + kBlk) / kBlk;
  int32_t* out = a.out + (int64_t(tok) * a.Hk + hk) * a.top;
  if (nb <= a.top) {  // every visible block
    for (int i = t; i < a.top; i += T) out[i] = i < nb ? i : -1;
    return;
  }
  // candidates: blocks in [sink, nb - recent); the others are taken (below nb) or absent
  const int lo_b = a.sink, hi_b = nb - a.recent;
  const int need = a.top - a.sink - a.recent;
  const uint32_t* keys = a.keys + id * a.n_blocks;
  constexpr int R = KPT > 0 ? KPT : 1;
  uint32_t k[R];
  const int per = KPT > 0 ? KPT : (nb + T - 1) / T;
  const int first = t * per;
  uint32_t kmax = 0, kmin = 0xffffffffu;
  if constexpr (KPT > 0) {
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const int b = first + i;
      const bool cand = b >= lo_b && b < hi_b;
      k[i] = cand ? __ldcg(keys + b) : 0u;
      if (cand) {
        kmax = max(kmax, k[i]);
        kmin = min(kmin, k[i]);
      }
    }
  } else {
    for (int b = t; b < nb; b += T) {
      const bool cand = b >= lo_b && b < hi_b;
      const uint32_t v = cand ? __ldcg(keys + b) : 0u;
      s_keys[b] = v;
      if (cand) {
        kmax = max(kmax, v);
        kmin = min(kmin, v);
      }
    }
    __syncthreads();
  }
  auto key_at = [&](int i) -> uint32_t {
    if constexpr (KPT > 0) return k[i];
    return first + i < nb ? s_keys[first + i] : 0u;
  };
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  kmin = __reduce_min_sync(0xffffffffu, kmin);
  if constexpr (T > 32) {
    if (lane == 0) {
      s_scan[warp] = int(kmax);
      s_scan2[warp] = int(kmin);
    }
    __syncthreads();
    kmax = __reduce_max_sync(0xffffffffu, lane < T / 32 ? uint32_t(s_scan[lane]) : 0u);
    kmin = __reduce_min_sync(0xffffffffu, lane < T / 32 ? uint32_t(s_scan2[lane]) : 0xffffffffu);
    __syncthreads();
  }
  int flip = 0;
  uint32_t thr;        // keys above it are taken, and the first `ties` equal to it
  int ties = 0;
  bool exact = false;  // every key at or above thr is taken
  if (need <= 0) {
    thr = 0xffffffffu;
  } else {
    const int top_bit = kmax == kmin ? -1 : 31 - __clz(kmax ^ kmin);
    thr = top_bit < 0 ? kmax : (top_bit == 31 ? 0u : (kmax >> (top_bit + 1)) << (top_bit + 1));
    for (int bit = top_bit; bit >= 0; --bit) {
      const uint32_t trial = thr | (1u << bit);
      int cnt = 0;
      if constexpr (KPT > 0) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) cnt += k[i] >= trial;
      } else {
        for (int i = 0; i < per; ++i) cnt += key_at(i) >= trial;
      }
      cnt = group_sum<T>(cnt, s_part, flip);
      if (cnt >= need) {
        thr = trial;
        if (cnt == need) {
          exact = true;
          break;
        }
      }
    }
    if (!exact) {
      int above = 0;
      if constexpr (KPT > 0) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) above += k[i] > thr;
      } else {
        for (int i = 0; i < per; ++i) above += key_at(i) > thr;
      }
      ties = need - group_sum<T>(above, s_part, flip);
    }
  }
  // ascending output: taken blocks before this thread's, and equal keys before them
  auto cand_at = [&](int i) { return first + i >= lo_b && first + i < hi_b; };
  int n_sure = 0, n_tie = 0;
  if constexpr (KPT > 0) {
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const int b = first + i;
      const bool c = cand_at(i);
      n_sure += b < nb && (!c || (need > 0 && (exact ? k[i] >= thr : k[i] > thr)));
      n_tie += c && !exact && need > 0 && k[i] == thr;
    }
  } else {
    for (int i = 0; i < per; ++i) {
      const int b = first + i;
      const bool c = cand_at(i);
      const uint32_t v = key_at(i);
      n_sure += b < nb && (!c || (need > 0 && (exact ? v >= thr : v > thr)));
      n_tie += c && !exact && need > 0 && v == thr;
    }
  }
  // exclusive scans of both counts over the threads
  int sure = n_sure, tie = n_tie;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, sure, o), y = __shfl_up_sync(0xffffffffu, tie, o);
    if (lane >= o) {
      sure += x;
      tie += y;
    }
  }
  int sure_base = 0, tie_base = 0;
  if constexpr (T > 32) {
    if (lane == 31) {
      s_scan[warp] = sure;
      s_scan2[warp] = tie;
    }
    __syncthreads();
    sure_base = __reduce_add_sync(0xffffffffu, lane < warp ? s_scan[lane] : 0);
    tie_base = __reduce_add_sync(0xffffffffu, lane < warp ? s_scan2[lane] : 0);
  }
  sure += sure_base - n_sure;  // taken for sure, before this thread's keys
  tie += tie_base - n_tie;     // ties before them
  auto emit = [&](int i, uint32_t v) {
    const int b = first + i;
    if (b >= nb) return;
    const bool c = cand_at(i);
    bool take = !c || (need > 0 && (exact ? v >= thr : v > thr));
    int at = sure + min(tie, ties);
    if (c && !exact && need > 0 && v == thr) {
      take = tie < ties;
      ++tie;
    } else if (take) {
      ++sure;
    }
    if (take && at < a.top) out[at] = b;
  };
  if constexpr (KPT > 0) {
#pragma unroll
    for (int i = 0; i < KPT; ++i) emit(i, k[i]);
  } else {
    for (int i = 0; i < per; ++i) emit(i, key_at(i));
  }
}

template <int HD, int NT>
int launch_score(const uint16_t* q, const int8_t* dig, const float* dig_scale, const int32_t* positions, int m, int t_begin,
                 int Hq, int Hk, int n_ctx, int n_blocks, uint32_t* keys, cudaStream_t stream) {
  constexpr int smem = kTok * NT * 8 * (4 * (2 * HD / 4 + 16) + 4);
  auto kern = block_score_kernel<HD, NT>;
  if (int rc = set_smem_limit(reinterpret_cast<const void*>(kern), smem)) return rc;
  const int groups = ceil_div(m, kTok);
  // enough CTAs for about two per SM, no more than there are tiles
  const int tiles = ceil_div(n_blocks, 16);
  const int x = std::max(1, std::min(ceil_div(tiles, kScoreWarps), ceil_div(2 * num_sms(), int64_t(groups) * Hk)));
  launch_pdl(kern, dim3(x, groups, Hk), dim3(kScoreWarps * 32), smem, stream, q, dig, dig_scale, positions, m, t_begin, Hq,
             Hk, n_ctx, n_blocks, keys);
  CKV_LAUNCH_CHECK("ckv_block_select(score)");
  return CKV_OK;
}

template <int T, int KPT>
int launch_top(const TopArgs& a, cudaStream_t stream) {
  const int64_t ids = int64_t(a.m) * a.Hk;
  const int smem = KPT > 0 ? 0 : a.n_blocks * 4;
  auto kern = block_top_kernel<T, KPT>;
  if (smem > 48 * 1024)
    if (int rc = set_smem_limit(reinterpret_cast<const void*>(kern), smem)) return rc;
  launch_pdl(kern, dim3(unsigned(T > 32 ? ids : (ids + 7) / 8)), dim3(T > 32 ? T : 256), size_t(smem), stream, a);
  CKV_LAUNCH_CHECK("ckv_block_select(top)");
  return CKV_OK;
}

// tokens whose keys the workspace holds at once: all of them, or as many as 256 MB take
int64_t chunk_tokens(int m, int Hk, int n_blocks) {
  const int64_t per = int64_t(Hk) * n_blocks * 4;
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
  return chunk_tokens(m, n_kv_heads, nb) * n_kv_heads * nb * 4;
}

extern "C" int ckv_block_select_launches(int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx) {
  if (m <= 0 || !select_shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) return 0;
  return 2 * ceil_div(m, chunk_tokens(m, n_kv_heads, ceil_div(n_ctx, kBlk)));
}

extern "C" int ckv_block_select(const uint16_t* q, const int8_t* dig_codes, const float* dig_scale,
                                const int32_t* positions, int32_t* blocks, int m, int n_q_heads, int n_kv_heads,
                                int head_dim, int n_ctx, int top, int sink, int recent, void* workspace,
                                int64_t workspace_bytes, ckv_stream_t stream) {
  CKV_REQUIRE(m >= 0 && n_kv_heads > 0 && n_q_heads > 0 && n_q_heads % n_kv_heads == 0 && n_ctx > 0,
              "ckv_block_select: bad sizes");
  CKV_REQUIRE(sink >= 0 && recent >= 1 && top >= 1 && int64_t(sink) + recent <= top && top <= kMaxTop,
              "ckv_block_select: top %d (1 to %d) must hold the %d first and %d last blocks (at least one last)", top,
              kMaxTop, sink, recent);
  if (!select_shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) {
    set_error("ckv_block_select: head_dim %d (64 or 128), %d query heads per KV head (at most 16), context %d (at most %d)",
              head_dim, n_q_heads / n_kv_heads, n_ctx, kMaxBlocks * kBlk);
    return CKV_ERR_UNSUPPORTED;
  }
  if (m == 0) return CKV_OK;
  CKV_REQUIRE(q && dig_codes && dig_scale && positions && blocks && workspace, "ckv_block_select: null pointer");
  CKV_REQUIRE(aligned16(q) && aligned16(dig_codes) && aligned16(workspace), "ckv_block_select: tensors must be 16-byte aligned");
  const int nb = ceil_div(n_ctx, kBlk);
  const int64_t step = chunk_tokens(m, n_kv_heads, nb);
  CKV_REQUIRE(workspace_bytes >= step * n_kv_heads * nb * 4, "ckv_block_select: workspace of %lld bytes, needs %lld",
              static_cast<long long>(workspace_bytes), static_cast<long long>(step * n_kv_heads * nb * 4));
  CKV_REQUIRE(m <= 1048560 && int64_t(m) * n_kv_heads < (int64_t(1) << 31) - 8, "ckv_block_select: too many rows");
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
    // a warp per (token, head) while its keys fit the warp's registers, a CTA beyond
    if (nb <= 512) rc = launch_top<32, 16>(a, s);
    else if (nb <= 2048) rc = launch_top<256, 8>(a, s);
    else if (nb <= 8192) rc = launch_top<1024, 8>(a, s);
    else rc = launch_top<1024, 0>(a, s);
    if (rc) return rc;
  }
  return CKV_OK;
}
