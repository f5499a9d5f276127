// Attention of few query rows over 16-key blocks streamed straight from HBM: one or a few
// tokens over a whole 8-bit cache (decode), and any number of tokens over the blocks listed
// for each of them (8-bit or bf16 cache).
//
// Such calls read every key for at most 16 query rows, so they are bound by the cache's
// bytes; a 128-row tcgen05 tile would be nearly empty.  The kernel keeps the bytes moving:
// a warp takes whole blocks (contiguous, 2 KiB of K and of V at head_dim 128 in 8 bits)
// through a ring of TMA bulk copies in shared memory and uses mma.sync m16n8k16 with the
// roles turned round: the 16 keys of a block are the M rows, the up to 8 query rows the N
// columns, so nothing is padded for groups of up to 8 heads.
//   S^T [16 keys x 8 rows]  = K Q^T        A = K, contraction over head_dim
//   O^T [dims x 8 rows]    += V^T P^T      A = V^T, contraction over the 16 keys
// The contraction over head_dim may be permuted if K and Q agree, so quad member c of a
// lane group holds the 16-byte pieces c, c + 4, .. of the rows of keys g and g + 8 (g = lane /
// 4): plain 16-byte loads, four lanes to 64 contiguous bytes (whole sectors: with D/4
// contiguous dims per lane every sector was fetched twice).  For V, lane (g, c) holds the
// pieces g, g + 8 of keys 2c, 2c+1, 2c+8, 2c+9; pairing two keys' bytes with one byte
// permutation gives the A operand, so V is transposed without shared memory.  P^T is turned
// into the B operand by movmatrix.
// 8-bit codes become fp16 exactly (e4m3 by cvt, int8 by adding 1024), so no value is
// rounded before the tensor core: scores are q (fp16, scaled by a power of two per row) .
// code, times the block's fp32 key scale; P is multiplied by the block's value scale
// relative to a running power-of-two reference and rounded to fp16 (2^-12), accumulators,
// maxima and sums are fp32.  With a bf16 cache P goes in as two bf16 parts (2^-17).
// The online maximum is lazy: O is rescaled when a row's maximum grew by more than 2^8.
//
// Measured: one row over 131,069 tokens (40 heads over 8, e4m3, 269 MB) 49 us, 5.5 TB/s; over 5248
// tokens (28 over 4) 9.2 us, most of it latency (300 tokens: 6.4); 8 rows over 32,896 tokens 36 us,
// four row tiles of compute; 938 rows of 64 listed blocks 255 us over a bf16 cache (1.97 GB out
// of L2, 7.7 TB/s) and 173 us over an 8-bit one (issue slots: widening and the softmax).
#include <algorithm>

#include "ckv_common.cuh"

CKV_DEFINE_ERR_WORD(attention_blocks)

namespace ckv {
// block_select.cu
int block_select_check(const uint16_t* q, const int8_t* dig_codes, const float* dig_scale, const int32_t* positions,
                       const int32_t* blocks, int m, int Hq, int Hk, int HD, int n_ctx, int top, int sink, int recent,
                       const void* workspace, int64_t workspace_bytes);
namespace {

constexpr int kBlk = CKV_PAGE_TOKENS;
constexpr int kCluster = 8;  // CTAs that share one row tile's blocks and join through shared memory
constexpr float kLazy = 8.0f;       // log2 units
constexpr float kPBias = 64.0f;     // P * value scale / reference is at most 2^8 * 2^6 in fp16
enum { kBf16 = 0, kInt8 = 1, kE4m3 = 2 };

struct Args {
  const uint16_t* q;  // [m][Hq][D]
  const uint8_t *k, *v;  // [H][rows][D], 1 or 2 bytes per value
  const float *ks, *vs;  // [H][n_blocks] (8 bits)
  const int32_t* positions;
  const int32_t* blocks;  // [m][H][top] (listed form), ascending, -1 past the end
  uint16_t* out;          // [m][Hq][D]
  float* part_o;          // [splits][tiles][H][8 NT][D]
  float2* part_ml;        // [splits][tiles][H][8 NT]
  int64_t head_rows;      // cache rows per head
  int m, Hq, Hk, n_ctx, n_blocks, top, items, splits, head_tiles;  // items: entries that a list can hold, min(top, n_blocks)
  float scale_log2;
  bool after_select;  // launched behind a kernel of the selection, which started when q and positions were complete
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int CT>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (CT == kBf16) mma_bf16(c, a0, a1, a2, a3, b0, b1);
  else mma_f16(c, a0, a1, a2, a3, b0, b1);
}
// four codes -> two pairs of fp16, exactly: (0, 1) and (2, 3)
template <int CT>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CT == kE4m3) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // 0x6400 + u is the fp16 number 1024 + u, u = code + 128: minus 1152 is the code
    const uint32_t u = w ^ 0x80808080u, magic = 0x64646464u;
    uint32_t a, b;
    a = __byte_perm(u, magic, 0x4140);
    b = __byte_perm(u, magic, 0x4342);
    asm("sub.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
  }
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float r;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r) : "r"(addr) : "memory");
  return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 r;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w) : "r"(addr) : "memory");
  return r;
}
// What a row's partial maxima are taken relative to when they are joined: their maximum m, or 0
// when there is none.  Scores of NaN never become a maximum, but they make the partial sum
// and O NaN, which a weight of 0 does not silence: the row comes out as NaN.  One that saw no
// key has sums of 0 everywhere and comes out as zeros.
__device__ __forceinline__ float join_base(float m) { return m == -INFINITY ? 0.f : m; }

// A stage holds NB blocks: their 16 rows of K each, then their 16 rows of V.  Over a whole cache of
// 8 bits a warp works on two together: two independent chains of mma and exponentials, one wait
// and one request (131,069 tokens, 8 heads: 50 us, one by one 53; 8 rows over 32,896 tokens 35 and
// 39).  One by one where lists give a warp few blocks (938 rows of 64 blocks: 173 us, in pairs 183; 60
// rows 21.6 and 22.9), and where a pair of stages would not fit twelve warps (bf16).
template <int HD, int CT, bool LISTED>
struct Block {
  static constexpr int ES = CT == kBf16 ? 2 : 1;
  static constexpr int ROW = HD * ES;         // bytes of a row
  static constexpr int KW = HD / 4 * ES / 4;  // 32-bit words of K per key and lane (a multiple of 4)
  static constexpr int VW = HD / 8 * ES / 4;  // of V (2 or a multiple of 4)
  static constexpr int HALF = kBlk * ROW;     // bytes of one block's K
  static constexpr int NB = !LISTED && 4 * HALF <= 8192 ? 2 : 1;
  static constexpr int STAGE = 2 * NB * HALF;

  // The warp: the rows that exist of blocks ids (a bf16 cache may end inside a block; -1: none).
  // Lane i < 2 NB copies K or V of one block.
  static __device__ __forceinline__ void request(const Args& a, uint8_t* stage, uint64_t* bar, int hk, const int (&ids)[NB],
                                                 int lane) {
    auto rows_of = [&](int id) { return id < 0 ? 0u : uint32_t(min(int64_t(kBlk), a.head_rows - int64_t(id) * kBlk)) * ROW; };
    const int id0 = ids[0], id1 = ids[NB - 1];
    const uint32_t n0 = rows_of(id0), n1 = NB == 2 ? rows_of(id1) : 0u;
    const uint32_t total = 2 * (n0 + n1);
    // by a mask: a choice between array elements would put the array in local memory
    const uint32_t odd = NB == 2 && (lane & 1) ? ~0u : 0u;
    const int b = int(uint32_t(id0) ^ ((uint32_t(id0) ^ uint32_t(id1)) & odd));
    const uint32_t bytes = n0 ^ ((n0 ^ n1) & odd);
    if (lane == 0) mbar_expect_tx(bar, total);
    if (lane < 2 * NB && b >= 0)
      bulk_load(stage + lane * HALF, (lane < NB ? a.k : a.v) + (int64_t(hk) * a.head_rows + int64_t(b) * kBlk) * ROW, bytes, bar);
  }
  // k: the lane's pieces of keys g, g + 8
  static __device__ __forceinline__ void fetch_k(const uint8_t* stage, int lane, uint32_t (&k)[2][KW]) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int w = 0; w < KW; w += 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(stage + (g + 8 * i) * ROW + 16 * (w + c));
        k[i][w] = x.x, k[i][w + 1] = x.y, k[i][w + 2] = x.z, k[i][w + 3] = x.w;
      }
  }
  // v: of keys 2c, 2c + 1, 2c + 8, 2c + 9; rows past `vis` as zeros (they may hold anything, and a
  // weight of 0 does not silence a NaN)
  static __device__ __forceinline__ void fetch_v(const uint8_t* stage, int lane, int vis, uint32_t (&v)[4][VW]) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* row = stage + (2 * c + (i & 1) + 8 * (i >> 1)) * ROW;
      if constexpr (VW >= 4) {
#pragma unroll
        for (int w = 0; w < VW; w += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(row + 16 * g + 32 * w);
          v[i][w] = x.x, v[i][w + 1] = x.y, v[i][w + 2] = x.z, v[i][w + 3] = x.w;
        }
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(row + 8 * g);
        v[i][0] = x.x, v[i][1] = x.y;
      }
    }
    if (vis < kBlk - 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (2 * c + (i & 1) + 8 * (i >> 1) > vis)
#pragma unroll
          for (int w = 0; w < VW; ++w) v[i][w] = 0u;
    }
  }
};

// Running state of a warp: for each of its 8 NT query rows a maximum and a sum, and O.
template <int HD, int CT, int NT, bool LISTED>
struct State {
  static constexpr int KSTEPS = HD / 16;
  uint32_t qf[NT][KSTEPS][2];
  float f[NT][2];      // per query row 2c, 2c + 1: score factor (log2 domain)
  int lim[NT][2];      // last visible key
  float mx[NT][2], l[NT][2];
  float ref;           // value-scale reference (power of two; 0 before the first block)
  float o[NT][KSTEPS][4];  // the lane's V dims 2t, 2t + 1 x rows 2c, 2c + 1

  // The blocks ids of a stage (-1: none) with their scales; `last`: the last key any row sees.
  __device__ __forceinline__ void step(const uint8_t* stage, const int (&ids)[Block<HD, CT, LISTED>::NB],
                                       const float (&ks)[Block<HD, CT, LISTED>::NB], const float (&vs)[Block<HD, CT, LISTED>::NB], int last,
                                       int lane) {
    using B = Block<HD, CT, LISTED>;
    constexpr int NB = B::NB;
    const int g = lane >> 2;
    float s[NB][NT][4], s2[NB][NT][4];  // even and odd steps of the contraction: half the length of the chain
    {
      uint32_t k[NB][2][B::KW];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        B::fetch_k(stage + i * B::HALF, lane, k[i]);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][n][e] = s2[i][n][e] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < KSTEPS; ++t) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          uint32_t a0, a1, a2, a3;
          if constexpr (CT == kBf16) {
            a0 = k[i][0][2 * t], a2 = k[i][0][2 * t + 1], a1 = k[i][1][2 * t], a3 = k[i][1][2 * t + 1];
          } else {
            widen<CT>(k[i][0][t], a0, a2);
            widen<CT>(k[i][1][t], a1, a3);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) mma<CT>(t & 1 ? s2[i][n] : s[i][n], a0, a1, a2, a3, qf[n][t][0], qf[n][t][1]);
        }
      }
    }
    // Scores; a row's maximum is renewed (and O rescaled) only when some score exceeds it by
    // more than 2^kLazy, so the usual step needs no reduction over the lanes.
    bool grow = false;
    float vtop = 0.f;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int key = ids[i] < 0 ? 0x7fffff00 : ids[i] * kBlk + g;
      if constexpr (CT != kBf16) vtop = fmaxf(vtop, vs[i]);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float fk = CT == kBf16 ? f[n][r] : f[n][r] * ks[i];
          s[i][n][r] = key <= lim[n][r] ? (s[i][n][r] + s2[i][n][r]) * fk : -INFINITY;
          s[i][n][2 + r] = key + 8 <= lim[n][r] ? (s[i][n][2 + r] + s2[i][n][2 + r]) * fk : -INFINITY;
          grow |= fmaxf(s[i][n][r], s[i][n][2 + r]) > mx[n][r] + kLazy;  // (mx = -inf: any score)
        }
    }
    if constexpr (CT != kBf16) grow |= vtop > ref;
    if (__any_sync(0xffffffffu, grow)) {
      float rs = 1.0f;
      if constexpr (CT != kBf16) {
        if (vtop > ref) {  // the same for the whole warp
          // the next power of two at or above it
          const float up = __uint_as_float((__float_as_uint(vtop) + 0x007fffffu) & 0x7f800000u);
          rs = ref / up;
          ref = up;
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = mx[n][r];
#pragma unroll
          for (int i = 0; i < NB; ++i) top = fmaxf(top, fmaxf(s[i][n][r], s[i][n][2 + r]));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          const float corr = mx[n][r] == -INFINITY ? 0.f : ex2_approx(mx[n][r] - top);
          l[n][r] *= corr;
          mx[n][r] = top;
#pragma unroll
          for (int t = 0; t < KSTEPS; ++t) {
            o[n][t][r] *= corr * rs;
            o[n][t][2 + r] *= corr * rs;
          }
        }
    }
    uint32_t ph[NB][NT][2];
    [[maybe_unused]] uint32_t pl[NB][NT][2];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const float vn = CT == kBf16 ? 1.0f : (ref > 0.f ? vs[i] * (kPBias / ref) : 0.f);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float base = mx[n][e & 1] == -INFINITY ? 0.f : mx[n][e & 1];  // no visible key yet: P = 0, not NaN
          p[e] = ex2_approx(s[i][n][e] - base);
          l[n][e & 1] += p[e];
        }
        if constexpr (CT == kBf16) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t hi = pack_bf2(p[2 * h], p[2 * h + 1]);
            ph[i][n][h] = transpose8(hi);
            pl[i][n][h] = transpose8(pack_bf2(p[2 * h] - lo_bf(hi), p[2 * h + 1] - hi_bf(hi)));
          }
        } else {
          ph[i][n][0] = transpose8(pack_h2(p[0] * vn, p[1] * vn));
          ph[i][n][1] = transpose8(pack_h2(p[2] * vn, p[3] * vn));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      uint32_t v[4][B::VW];
      B::fetch_v(stage + (NB + i) * B::HALF, lane, ids[i] < 0 ? -1 : last - ids[i] * kBlk, v);
      if constexpr (CT == kBf16) {
#pragma unroll
        for (int w = 0; w < KSTEPS; ++w) {
          const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5410), a1 = __byte_perm(v[0][w], v[1][w], 0x7632);
          const uint32_t a2 = __byte_perm(v[2][w], v[3][w], 0x5410), a3 = __byte_perm(v[2][w], v[3][w], 0x7632);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_bf16(o[n][w], a0, a1, a2, a3, ph[i][n][0], ph[i][n][1]);
            mma_bf16(o[n][w], a0, a1, a2, a3, pl[i][n][0], pl[i][n][1]);
          }
        }
      } else {
#pragma unroll
        for (int w = 0; w < KSTEPS / 2; ++w) {
          // keys 2c, 2c+1 (and 2c+8, 2c+9) of dims 4w .. 4w+3, two keys of a dim side by side
          uint32_t a0, a1, a2, a3;
          widen<CT>(__byte_perm(v[0][w], v[1][w], 0x5140), a0, a1);
          widen<CT>(__byte_perm(v[2][w], v[3][w], 0x5140), a2, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * w], a0, a1, a2, a3, ph[i][n][0], ph[i][n][1]);
          widen<CT>(__byte_perm(v[0][w], v[1][w], 0x7362), a0, a1);
          widen<CT>(__byte_perm(v[2][w], v[3][w], 0x7362), a2, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * w + 1], a0, a1, a2, a3, ph[i][n][0], ph[i][n][1]);
        }
      }
    }
  }
};

// Shared memory: W rings of stages; after the loop the same space takes the warps' states, and
// behind it the CTA's joined state (read by the cluster's other CTAs) and the barriers.
template <int HD, int CT, int NT, int W, bool LISTED>
struct Layout {
  static constexpr int ROWS = 8 * NT;
  // two stages where more CTAs (W = 4) or warps share the SM: at 938 rows of 64 listed blocks three
  // CTAs of two stages take 255 us (bf16) and 173 us (8 bits), of three 303 (two CTAs) and 176 us
  static constexpr int STAGES = W == 8 ? 3 : 2;
  static constexpr int RING = STAGES * Block<HD, CT, LISTED>::STAGE;
  static constexpr int STRIDE = HD + 4;  // floats of a state row
  static constexpr int STATES = W * ROWS * (STRIDE + 2) * 4;
  static constexpr int JOINED = (W * RING > STATES ? W * RING : STATES + 15) / 16 * 16;
  static constexpr int BARS = JOINED + ROWS * (STRIDE + 2) * 4;
  static constexpr int BYTES = BARS + W * STAGES * 8 + 8;
};

// grid: (splits, row tiles, KV heads).  Dense (LISTED = false): tile y holds the packed rows
// (token, head of the group) [8 NT y, 8 NT (y + 1)) of its KV head.  Listed: tile y is head
// tile y % head_tiles of token y / head_tiles, and the split takes its share of the list.
// Four CTAs of listed 8-bit blocks share an SM (128 registers: 938 rows of 64 blocks 174 us; three CTAs
// of 136 registers 199); over a bf16 cache three do, by shared memory.
// JOIN: the kCluster splits of a tile are one cluster and leave finished rows; otherwise more
// than one split leaves partials for attention_blocks_join_kernel.
template <int HD, int CT, int NT, bool LISTED, int W, bool JOIN>
__global__ void __launch_bounds__(W * 32, W > 4 ? 1 : NT == 2 ? 2 : CT == kBf16 ? 3 : 4)
    attention_blocks_kernel(const __grid_constant__ Args a) {
  using L = Layout<HD, CT, NT, W, LISTED>;
  using B = Block<HD, CT, LISTED>;
  constexpr int KSTEPS = HD / 16, ROWS = L::ROWS;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int G = a.Hq / a.Hk;
  const int hk = blockIdx.z, split = blockIdx.x;
  const int tile = blockIdx.y;
  const int tok0 = LISTED ? tile / a.head_tiles : 0;
  const int row0 = LISTED ? tok0 * G + (tile % a.head_tiles) * ROWS : tile * ROWS;  // packed row
  const int row_end = LISTED ? tok0 * G + G : a.m * G;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS) + warp * L::STAGES;
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::BARS + W * L::STAGES * 8);
  if (lane == 0) {
    for (int s = 0; s < L::STAGES; ++s) mbar_init(&bars[s], 1);
    fence_barrier_init();
  }
  if (threadIdx.x == 0) *abort = 0;
  __syncthreads();
  // Behind the selection only the lists (and the output) wait for the kernel before: every CTA of
  // it lets this kernel start after its own wait, so q and the positions, written before the selection
  // began, are in L2 by then.  They are read there (ld.cg): a line of them that L1 still held
  // from an earlier kernel would be older.  (Over a whole cache they come through L1: up to twelve warps
  // read the same rows, and past it one row over 5248 tokens took 9.5 us instead of 9.3.)  One row and
  // 64 of 2056 blocks take 13.1 us, with q and the positions behind the wait 13.6.
  if (!a.after_select) pdl_wait();
  // as an operand owner a lane has query rows 8n + g: q and their positions first
  uint32_t w[NT][HD / 8];  // the dims of this lane's pieces of K (16 / ES dims each)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int pr = row0 + 8 * n + g;
    const bool ok = pr < row_end;
    const int tok = ok ? pr / G : 0;
#pragma unroll
    for (int e = 0; e < HD / 8; e += 4) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (ok) {
        const uint4* at = reinterpret_cast<const uint4*>(a.q + (int64_t(tok) * a.Hq + hk * G + (pr - tok * G)) * HD) +
                          (B::ES == 2 ? e + c : 8 * (e / 8) + 2 * c + (e / 4) % 2);
        if constexpr (LISTED) x = __ldcg(at);
        else x = __ldg(at);
      }
      w[n][e] = x.x, w[n][e + 1] = x.y, w[n][e + 2] = x.z, w[n][e + 3] = x.w;
    }
  }
  int pos[NT];
  int last = -1;  // last key any row of the tile sees
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int pr = row0 + 8 * n + g;
    int p = -1;
    if (pr < row_end) {
      if constexpr (LISTED) p = __ldcg(a.positions + pr / G);
      else p = a.positions[pr / G];
      if (p >= a.n_ctx) {
        if (split == 0 && hk == 0) atomicOr(&g_err_word, CKV_DEV_ERR_POSITION_RANGE);
        p = a.n_ctx - 1;
      }
      p = max(p, -1);
    }
    pos[n] = p;
    last = max(last, __reduce_max_sync(0xffffffffu, p));
  }
  if (a.after_select) pdl_wait();
  pdl_launch_next();
  const int nb = (last + kBlk) / kBlk;  // visible blocks
  const int n_items = LISTED ? a.items : nb;
  const int per = (n_items + a.splits - 1) / a.splits;
  const int i1 = min(n_items, (split + 1) * per);
  const int32_t* list = LISTED ? a.blocks + (int64_t(tok0) * a.Hk + hk) * a.top : nullptr;
  // item i's block, or -1 when there is none (past the list's end, out of range, not ascending).  Every
  // entry is held against the one before it, so a list that lets a block through twice is recorded.
  auto block_of = [&](int i) -> int {
    if (i >= i1) return -1;
    if constexpr (!LISTED) return i;
    const int b = list[i];  // not by the read-only path: the selection may write it while this kernel runs
    if (b == -1) return -1;
    const int before = i > 0 ? list[i - 1] : -2;  // -2: nothing before it
    if (b < 0 || b >= a.n_blocks || before >= b || before == -1) {
      if (lane == 0) atomicOr(&g_err_word, CKV_DEV_ERR_POSITION_RANGE);
      return -1;
    }
    return b < nb ? b : -1;  // wholly past the row's position: nothing visible
  };
  uint8_t* ring = smem + warp * L::RING;
  constexpr int NB = B::NB;
  int ids[L::STAGES][NB];                           // blocks in the ring, -1: none
  float ks[L::STAGES][NB] = {}, vs[L::STAGES][NB] = {};  // their scales
  int i = split * per + warp * NB;
  auto fill = [&](int s, int at) {
#pragma unroll
    for (int e = 0; e < NB; ++e) ids[s][e] = block_of(at + e);
    bool any = ids[s][0] >= 0;
    if constexpr (NB == 2) any |= ids[s][1] >= 0;
    if (any) B::request(a, ring + s * B::STAGE, &bars[s], hk, ids[s], lane);
    if constexpr (CT != kBf16) {
#pragma unroll
      for (int e = 0; e < NB; ++e) {
        const int64_t b = int64_t(hk) * a.n_blocks + ids[s][e];
        ks[s][e] = ids[s][e] < 0 ? 0.f : __ldg(a.ks + b);
        vs[s][e] = ids[s][e] < 0 ? 0.f : __ldg(a.vs + b);
      }
    }
  };
#pragma unroll
  for (int s = 0; s < L::STAGES; ++s) fill(s, i + s * W * NB);

  State<HD, CT, NT, LISTED> st;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float factor = a.scale_log2;
    if constexpr (CT == kBf16) {
#pragma unroll
      for (int t = 0; t < KSTEPS; ++t) {
        st.qf[n][t][0] = w[n][2 * t];
        st.qf[n][t][1] = w[n][2 * t + 1];
      }
    } else {
      // to fp16 through a power of two that puts the row's largest value in [2^14, 2^15):
      // exact down to 2^-38 of it
      uint32_t mag = 0;
#pragma unroll
      for (int e = 0; e < HD / 8; ++e) mag = __vmaxu2(mag, w[n][e] & 0x7fff7fffu);
      uint32_t am = max(mag & 0xffffu, mag >> 16);
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
      const int sh = am == 0 ? 0 : max(-126, min(126, 14 + 127 - int(am >> 7)));  // multiply by 2^sh
      const float up = __uint_as_float(uint32_t(sh + 127) << 23);
      factor *= __uint_as_float(uint32_t(127 - sh) << 23);
#pragma unroll
      for (int t = 0; t < KSTEPS; ++t) {
        st.qf[n][t][0] = pack_h2(lo_bf(w[n][2 * t]) * up, hi_bf(w[n][2 * t]) * up);
        st.qf[n][t][1] = pack_h2(lo_bf(w[n][2 * t + 1]) * up, hi_bf(w[n][2 * t + 1]) * up);
      }
    }
    // as a column owner: rows 8n + 2c and 8n + 2c + 1
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      st.f[n][r] = __shfl_sync(0xffffffffu, factor, 4 * (2 * c + r));
      st.lim[n][r] = __shfl_sync(0xffffffffu, pos[n], 4 * (2 * c + r));
      st.mx[n][r] = -INFINITY;
      st.l[n][r] = 0.f;
    }
#pragma unroll
    for (int t = 0; t < KSTEPS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[n][t][e] = 0.f;
  }
  st.ref = 0.f;

  uint32_t phase = 0;  // bit s: parity of stage s's next arrival
  bool ok = true;
  auto filled = [&](int s) {
    bool any = ids[s][0] >= 0;
    if constexpr (NB == 2) any |= ids[s][1] >= 0;
    return any;
  };
  while (i < i1 && ok) {
#pragma unroll
    for (int s = 0; s < L::STAGES; ++s) {
      if (filled(s)) {
        ok = ok && mbar_wait(&bars[s], (phase >> s) & 1, abort, &g_err_word);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        phase ^= 1u << s;
        st.step(ring + s * B::STAGE, ids[s], ks[s], vs[s], last, lane);
        __syncwarp();  // every lane has read the stage: it may be filled again
      }
      fill(s, i + (s + L::STAGES) * W * NB);
    }
    i += L::STAGES * W * NB;
  }
  if (!ok) {  // a copy never came: let those still out land (bounded) before the ring is reused
    uint32_t out = 0;
#pragma unroll
    for (int s = 0; s < L::STAGES; ++s) out |= filled(s) ? 1u << s : 0u;
    const uint64_t t0 = global_ns();
#pragma unroll 1
    for (int s = 0; s < L::STAGES; ++s)
      while ((out >> s) & 1) {
        if (mbar_try_wait(&bars[s], (phase >> s) & 1) || global_ns() - t0 > kWaitLimitNs) break;
      }
  }
  __syncthreads();  // the rings are free: they become the warps' states

  float* s_o = reinterpret_cast<float*>(smem);  // [W][ROWS][STRIDE]
  float* s_m = s_o + W * ROWS * L::STRIDE;      // [W][ROWS]
  float* s_l = s_m + W * ROWS;
  const float oscale = CT == kBf16 ? 1.0f : st.ref / kPBias;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float l = st.l[n][r];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      const int row = 8 * n + 2 * c + r;
      if (g == 0) {
        s_m[warp * ROWS + row] = st.mx[n][r];
        s_l[warp * ROWS + row] = l;
      }
#pragma unroll
      for (int t = 0; t < KSTEPS; t += 2)
        // V dims 2t .. 2t + 3 of the lane: piece t / 4 (8 dims) of a bf16 row, else its only one
        *reinterpret_cast<float4*>(s_o + (warp * ROWS + row) * L::STRIDE +
                                   (CT == kBf16 ? 64 * (t / 4) + 8 * g + 2 * (t % 4) : g * (HD / 8) + 2 * t)) =
            make_float4(st.o[n][t][r] * oscale, st.o[n][t][2 + r] * oscale, st.o[n][t + 1][r] * oscale,
                        st.o[n][t + 1][2 + r] * oscale);
    }
  __syncthreads();
  constexpr int QV = HD / 4;  // float4 columns of a row
  auto store_row = [&](int pr, int col, const float4& o, float l) {
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    const int tok = pr / G;
    *reinterpret_cast<uint2*>(a.out + (int64_t(tok) * a.Hq + hk * G + (pr - tok * G)) * HD + col) =
        make_uint2(pack_bf2(o.x * inv, o.y * inv), pack_bf2(o.z * inv, o.w * inv));
  };
  float* j_o = reinterpret_cast<float*>(smem + L::JOINED);  // [ROWS][STRIDE], then m and l
  const int64_t prow0 = ((int64_t(split) * gridDim.y + tile) * a.Hk + hk) * ROWS;
  for (int j = threadIdx.x; j < ROWS * QV; j += W * 32) {
    const int row = j / QV, col = (j - row * QV) * 4;
    const int pr = row0 + row;
    if (pr >= row_end) continue;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, s_m[w * ROWS + row]);
    const float base = join_base(m);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float wt = ex2_approx(s_m[w * ROWS + row] - base);
      const float4 x = *reinterpret_cast<const float4*>(s_o + (w * ROWS + row) * L::STRIDE + col);
      l = fmaf(wt, s_l[w * ROWS + row], l);
      o.x = fmaf(wt, x.x, o.x);
      o.y = fmaf(wt, x.y, o.y);
      o.z = fmaf(wt, x.z, o.z);
      o.w = fmaf(wt, x.w, o.w);
    }
    if constexpr (JOIN) {
      *reinterpret_cast<float4*>(j_o + row * L::STRIDE + col) = o;
      if (col == 0) {
        j_o[ROWS * L::STRIDE + row] = m;
        j_o[ROWS * (L::STRIDE + 1) + row] = l;
      }
    } else if (a.splits > 1) {
      *reinterpret_cast<float4*>(a.part_o + (prow0 + row) * HD + col) = o;
      if (col == 0) a.part_ml[prow0 + row] = make_float2(m, l);
    } else {
      store_row(pr, col, o, l);
    }
  }
  if constexpr (JOIN) {
    // the cluster's CTAs each finish a share of the columns from everybody's joined states
    cluster_sync();
    const int rank = split;  // the cluster spans the splits
    const int n_cols = min(ROWS, row_end - row0) * QV;
    for (int j = rank * (W * 32) + threadIdx.x; j < n_cols; j += kCluster * W * 32) {
      const int row = j / QV, col = (j - row * QV) * 4;
      float mr[kCluster], m = -INFINITY;
#pragma unroll
      for (int r = 0; r < kCluster; ++r) {
        mr[r] = ld_cluster(cluster_smem_addr(j_o + ROWS * L::STRIDE + row, r));
        m = fmaxf(m, mr[r]);
      }
      const float base = join_base(m);
      float l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < kCluster; ++r) {
        const float wt = ex2_approx(mr[r] - base);
        const float4 x = ld_cluster4(cluster_smem_addr(j_o + row * L::STRIDE + col, r));
        l = fmaf(wt, ld_cluster(cluster_smem_addr(j_o + ROWS * (L::STRIDE + 1) + row, r)), l);
        o.x = fmaf(wt, x.x, o.x);
        o.y = fmaf(wt, x.y, o.y);
        o.z = fmaf(wt, x.z, o.z);
        o.w = fmaf(wt, x.w, o.w);
      }
      store_row(row0 + row, col, o, l);
    }
    cluster_sync();  // no CTA leaves while its shared memory is read
  }
  if constexpr (LISTED) {
    // An ascending list ends before its entry `items`, and no split takes those from there on: one that
    // is not -1 is recorded.  (Last, where it holds no registers: in front of the loop it cost a CTA
    // per SM at head_dim 64, 863 rows of 23 blocks 26.3 us against 24.4.)
    if (a.top > a.items && blockIdx.x == 0)
      for (int i = a.items + threadIdx.x; i < a.top; i += W * 32)
        if (a.blocks[(int64_t(blockIdx.y / a.head_tiles) * a.Hk + blockIdx.z) * a.top + i] != -1)
          atomicOr(&g_err_word, CKV_DEV_ERR_POSITION_RANGE);
  }
}

// Joins the splits: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.  A CTA takes one
// packed row of one KV head; HD / 4 lanes hold four columns each, the other lane groups take
// other splits, and the groups meet in shared memory.
template <int HD>
__global__ void __launch_bounds__(256) attention_blocks_join_kernel(const __grid_constant__ Args a, int tiles, int rows_per_tile,
                                                                    int listed) {
  constexpr int QV = HD / 4, GROUPS = 256 / QV;
  __shared__ float s_red[8];
  __shared__ float4 s_acc[GROUPS][QV];
  __shared__ float s_l[GROUPS];
  const int hk = blockIdx.y;
  const int G = a.Hq / a.Hk;
  int tile, row;
  const int pr = blockIdx.x;  // packed row: token * G + head of the group
  const int tok = pr / G;
  if (listed) {
    const int gi = pr - tok * G;
    tile = tok * a.head_tiles + gi / rows_per_tile;
    row = gi % rows_per_tile;
  } else {
    tile = pr / rows_per_tile;
    row = pr % rows_per_tile;
  }
  const int grp = threadIdx.x / QV, col = (threadIdx.x % QV) * 4;
  pdl_wait();
  pdl_launch_next();
  const int64_t stride = int64_t(tiles) * a.Hk * rows_per_tile;
  const int64_t at = (int64_t(tile) * a.Hk + hk) * rows_per_tile + row;
  float m = -INFINITY;
  for (int s = threadIdx.x; s < a.splits; s += 256) m = fmaxf(m, __ldcg(&a.part_ml[s * stride + at].x));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = s_red[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, s_red[i]);
  const float base = join_base(m);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = grp; s < a.splits; s += GROUPS) {
    const float2 ml = __ldcg(&a.part_ml[s * stride + at]);
    const float4 x = __ldcg(reinterpret_cast<const float4*>(a.part_o + (s * stride + at) * HD + col));
    const float wt = ex2_approx(ml.x - base);
    l = fmaf(wt, ml.y, l);
    o.x = fmaf(wt, x.x, o.x);
    o.y = fmaf(wt, x.y, o.y);
    o.z = fmaf(wt, x.z, o.z);
    o.w = fmaf(wt, x.w, o.w);
  }
  s_acc[grp][threadIdx.x % QV] = o;
  if (threadIdx.x % QV == 0) s_l[grp] = l;
  __syncthreads();
  if (threadIdx.x < QV) {
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) {
      const float4 x = s_acc[i][threadIdx.x];
      o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
      l += s_l[i];
    }
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    *reinterpret_cast<uint2*>(a.out + (int64_t(tok) * a.Hq + hk * G + (pr - tok * G)) * HD + col) =
        make_uint2(pack_bf2(o.x * inv, o.y * inv), pack_bf2(o.z * inv, o.w * inv));
  }
}

struct Plan {
  int nt, tiles, head_tiles, splits;
  bool join;  // the splits are one cluster
  int64_t bytes;
};

// Bytes of cache that one CTA of a cluster streams at most: beyond, the few SMs of the clusters
// are slower than all SMs with a second kernel for the join (one row of 4 KV heads, in clusters and split:
// 1024 tokens 6.4 and 6.9 us, 5248 9.1 and 8.5 and the host's 3 us for a second launch, 8192 10.8 and 8.7).
constexpr int64_t kClusterBytes = 192 * 1024;

// CTAs of clusters that surely run at once: eight to a GPC's SMs, one each (its shared memory is
// taken by the rings); with 16 clusters the last waits for the others (15 us instead of 9).
constexpr int kClusterCtas = 96;

// Rows of one KV head in tiles of 8 (or 16).  With too few tiles to fill the SMs the blocks are
// split: over the eight CTAs of a cluster while that moves few bytes per CTA (one launch, no
// workspace), else over enough CTAs for three per SM, no finer than one block per warp.
Plan plan(int m, int G, int Hk, int HD, int es, int items, bool listed) {
  Plan p;
  p.nt = (listed ? G : int64_t(m) * G) > 8 ? 2 : 1;
  p.head_tiles = listed ? ceil_div(G, 8 * p.nt) : 1;
  p.tiles = listed ? m * p.head_tiles : ceil_div(int64_t(m) * G, 8 * p.nt);
  const int64_t ctas = std::max<int64_t>(1, int64_t(p.tiles) * Hk);
  const int64_t cta_bytes = int64_t(items) * kBlk * HD * es * 2 / kCluster;
  p.splits = 1;
  p.join = false;
  if (items > 4 && ctas * kCluster <= kClusterCtas && cta_bytes <= kClusterBytes) {
    p.splits = kCluster;
    p.join = true;
  } else {
    p.splits = int(std::min<int64_t>(std::max<int64_t>(1, (listed ? 3 : 1) * num_sms() / ctas), ceil_div(items, listed ? 4 : 8)));
  }
  p.bytes = p.splits > 1 && !p.join ? int64_t(p.splits) * ctas * 8 * p.nt * (int64_t(HD) * 4 + 8) : 0;
  return p;
}

template <int HD, int CT, int NT, bool LISTED>
int launch(Args a, const Plan& p, void* workspace, cudaStream_t stream) {
  a.splits = p.splits;
  a.head_tiles = p.head_tiles;
  if (p.join) {
    // 12 warps where pairs of blocks halve the steps (5248 tokens: 9.2 us, with eight 9.6; 64 to 128 listed
    // blocks: 6.9 and 7.3); eight with three stages over a bf16 cache (32 blocks: 5.7 us, with twelve 5.9)
    constexpr int WJ = NT == 1 && CT != kBf16 ? 12 : 8;
    using L = Layout<HD, CT, NT, WJ, LISTED>;
    auto kern = attention_blocks_kernel<HD, CT, NT, LISTED, WJ, true>;
    if (int rc = set_smem_limit(reinterpret_cast<const void*>(kern), L::BYTES)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.splits, p.tiles, a.Hk);
    cfg.blockDim = dim3(WJ * 32);
    cfg.dynamicSmemBytes = L::BYTES;
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
    cudaLaunchKernelEx(&cfg, kern, a);
    CKV_LAUNCH_CHECK("ckv_attention_blocks(cluster)");
    return CKV_OK;
  }
  if (p.splits > 1) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + int64_t(p.splits) * p.tiles * a.Hk * 8 * NT * HD);
  }
  constexpr int W = LISTED ? 4 : NT == 2 ? 8 : 12;
  using L = Layout<HD, CT, NT, W, LISTED>;
  auto kern = attention_blocks_kernel<HD, CT, NT, LISTED, W, false>;
  if (int rc = set_smem_limit(reinterpret_cast<const void*>(kern), L::BYTES)) return rc;
  launch_pdl(kern, dim3(p.splits, p.tiles, a.Hk), dim3(W * 32), L::BYTES, stream, a);
  CKV_LAUNCH_CHECK("ckv_attention_blocks");
  if (p.splits > 1) {
    launch_pdl(attention_blocks_join_kernel<HD>, dim3(a.m * (a.Hq / a.Hk), a.Hk), dim3(256), 0, stream, a, p.tiles, 8 * NT,
               int(LISTED));
    CKV_LAUNCH_CHECK("ckv_attention_blocks(join)");
  }
  return CKV_OK;
}

template <int HD, int CT, bool LISTED>
int launch_nt(const Args& a, const Plan& p, void* workspace, cudaStream_t stream) {
  return p.nt == 1 ? launch<HD, CT, 1, LISTED>(a, p, workspace, stream) : launch<HD, CT, 2, LISTED>(a, p, workspace, stream);
}

// The entries of a list of `top` that can name a block of the context: work and partials are planned
// for these (128 entries over 300 tokens would leave six of a cluster's eight CTAs without any).
int list_items(int top, int n_ctx) { return std::min(top, ceil_div(n_ctx, kBlk)); }

// Tokens of a listed call per launch: a grid's second dimension is limited, so tokens go in runs of at
// most 32768 tiles (rows are independent, and a call this long is never split along its lists).
int run_tokens(const Plan& p) { return std::max(1, 32768 / p.head_tiles); }

int launches(const Plan& p) { return p.splits > 1 && !p.join ? 2 : 1; }

// query rows (token, head) of a call: tile and row numbers stay within 32 bits
constexpr int64_t kMaxRows = (int64_t(1) << 31) - (1 << 20);

bool shape_ok(int m, int Hq, int Hk, int HD, int n_ctx) {
  return m >= 0 && Hk > 0 && Hk <= 65535 && Hq > 0 && Hq % Hk == 0 && (HD == 64 || HD == 128) && n_ctx > 0 && n_ctx <= (1 << 30) &&
         int64_t(m) * Hq <= kMaxRows;
}

int check(const char* name, const Args& a, int HD, int64_t tiles) {
  CKV_REQUIRE(a.m >= 0 && a.Hk > 0 && a.Hk <= 65535 && a.Hq > 0 && a.Hq % a.Hk == 0, "%s: %d query heads over %d KV heads", name,
              a.Hq, a.Hk);
  CKV_REQUIRE(a.n_ctx > 0 && a.n_ctx <= (1 << 30), "%s: context of %d", name, a.n_ctx);
  CKV_REQUIRE(a.scale_log2 >= 0.f && a.scale_log2 <= 3.0e38f, "%s: scale %g (0 to 2e38)", name,
              double(a.scale_log2 / 1.4426950408889634f));
  CKV_REQUIRE(int64_t(a.m) * a.Hq <= kMaxRows, "%s: %d rows of %d heads in one call", name, a.m, a.Hq);
  if (HD != 64 && HD != 128) {
    set_error("%s: head_dim %d (64 or 128)", name, HD);
    return CKV_ERR_UNSUPPORTED;
  }
  if (a.m == 0) return CKV_OK;
  CKV_REQUIRE(a.q && a.k && a.v && a.positions && a.out, "%s: null pointer", name);
  CKV_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.out), "%s: tensors must be 16-byte aligned", name);
  if (tiles > 65535) {
    set_error("%s: %lld row tiles (at most 65535 in one call)", name, static_cast<long long>(tiles));
    return CKV_ERR_UNSUPPORTED;
  }
  return CKV_OK;
}

// What ckv_attention_sparse(_kv8) needs: the selection's keys and the attention's partials, one
// after the other in the same space, and behind them the digest when the call builds it.
struct SparseSpace {
  int64_t step, digest;
  int64_t total() const { return step + digest; }
};
SparseSpace sparse_space(int m, int Hq, int Hk, int HD, int es, int n_ctx, int top, bool build) {
  const int64_t sel = ckv_block_select_workspace_size(m, Hq, Hk, HD, n_ctx);
  const int64_t att = plan(m, Hq / Hk, Hk, HD, es, list_items(top, n_ctx), true).bytes;
  const int64_t nb = ceil_div(n_ctx, kBlk);
  SparseSpace x;
  x.step = (std::max(sel, att) + 15) / 16 * 16;
  x.digest = build ? int64_t(Hk) * nb * (2 * HD + 4) : 0;
  return x;
}

int check_space(const char* name, int m, int Hq, int Hk, int HD, int es, int n_ctx, int top, bool build, const void* workspace,
                int64_t ws_bytes) {
  CKV_REQUIRE(m >= 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0 && n_ctx > 0 && top > 0 && int64_t(m) * Hq <= kMaxRows,
              "%s: bad sizes", name);
  if (m == 0) return CKV_OK;
  const int64_t need = sparse_space(m, Hq, Hk, HD, es, n_ctx, top, build).total();
  CKV_REQUIRE(ws_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "%s: workspace of %lld bytes, needs %lld (16-byte aligned)", name, static_cast<long long>(ws_bytes),
              static_cast<long long>(need));
  return CKV_OK;
}

// The arguments of a listed call; `type` -1: a bf16 cache.
struct Call {
  Args a;
  int HD, type;
  void* workspace;
  int64_t ws_bytes;
  Plan plan() const { return ckv::plan(a.m, a.Hq / a.Hk, a.Hk, HD, type < 0 ? 2 : 1, a.items, true); }
};

Call bf16_call(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache, const int32_t* positions, const int32_t* blocks,
               uint16_t* out, int m, int Hq, int Hk, int HD, int n_ctx, int top, float scale, void* workspace, int64_t ws_bytes,
               bool after_select) {
  return {{q, reinterpret_cast<const uint8_t*>(k_cache), reinterpret_cast<const uint8_t*>(v_cache), nullptr, nullptr, positions, blocks,
           out, nullptr, nullptr, int64_t(n_ctx), m, Hq, Hk, n_ctx, ceil_div(n_ctx, kBlk), top, list_items(top, n_ctx), 1, 1,
           scale * 1.4426950408889634f, after_select},
          HD, -1, workspace, ws_bytes};
}

Call kv8_call(const uint16_t* q, const uint8_t* k8, const uint8_t* v8, const float* k_scale, const float* v_scale,
              const int32_t* positions, const int32_t* blocks, uint16_t* out, int m, int Hq, int Hk, int HD, int n_ctx, int top,
              float scale, int type, void* workspace, int64_t ws_bytes, bool after_select) {
  const int nb = ceil_div(n_ctx, kBlk);
  return {{q, k8, v8, k_scale, v_scale, positions, blocks, out, nullptr, nullptr, int64_t(nb) * kBlk, m, Hq, Hk, n_ctx, nb, top,
           list_items(top, n_ctx), 1, 1, scale * 1.4426950408889634f, after_select},
          HD, type, workspace, ws_bytes};
}

// Everything that a listed call refuses, without a launch.
int check_call(const char* name, const Call& c, bool eight) {
  const Args& a = c.a;
  if (eight) {
    CKV_REQUIRE(c.type == CKV_KV8_INT8 || c.type == CKV_KV8_E4M3, "%s: type %d", name, c.type);
    CKV_REQUIRE(a.m == 0 || (a.ks && a.vs), "%s: null scales", name);
  }
  CKV_REQUIRE(a.top > 0, "%s: lists of %d blocks", name, a.top);
  if (int rc = check(name, a, c.HD, 0)) return rc;
  if (a.m == 0) return CKV_OK;
  CKV_REQUIRE(a.blocks != nullptr, "%s: null block list", name);
  const int64_t need = c.plan().bytes;
  CKV_REQUIRE(c.ws_bytes >= need && (need == 0 || (c.workspace && aligned16(c.workspace))),
              "%s: workspace of %lld bytes, needs %lld (16-byte aligned)", name, static_cast<long long>(c.ws_bytes),
              static_cast<long long>(need));
  return CKV_OK;
}

int launch_call(const Call& c, cudaStream_t s) {
  const Args& a = c.a;
  const Plan p = c.plan();
  const int run = run_tokens(p);
  for (int t = 0; t < a.m; t += run) {
    Args b = a;
    Plan pb = p;
    b.m = std::min(run, a.m - t);
    pb.tiles = b.m * p.head_tiles;
    b.q += int64_t(t) * a.Hq * c.HD;
    b.out += int64_t(t) * a.Hq * c.HD;
    b.positions += t;
    b.blocks += int64_t(t) * a.Hk * a.top;
    int rc;
    if (c.HD == 128)
      rc = c.type < 0 ? launch_nt<128, kBf16, true>(b, pb, c.workspace, s)
           : c.type == CKV_KV8_E4M3 ? launch_nt<128, kE4m3, true>(b, pb, c.workspace, s)
                                    : launch_nt<128, kInt8, true>(b, pb, c.workspace, s);
    else
      rc = c.type < 0 ? launch_nt<64, kBf16, true>(b, pb, c.workspace, s)
           : c.type == CKV_KV8_E4M3 ? launch_nt<64, kE4m3, true>(b, pb, c.workspace, s)
                                    : launch_nt<64, kInt8, true>(b, pb, c.workspace, s);
    if (rc) return rc;
  }
  return CKV_OK;
}

int attention_blocks(const char* name, const Call& c, bool eight, ckv_stream_t stream) {
  if (int rc = check_call(name, c, eight)) return rc;
  return c.a.m == 0 ? CKV_OK : launch_call(c, as_stream(stream));
}

}  // namespace

// Few query rows over a whole 8-bit cache; used by ckv_attention_kv8 (attention_kv8.cu).
int64_t kv8_stream_workspace(int m, int Hq, int Hk, int HD, int n_ctx) {
  return plan(m, Hq / Hk, Hk, HD, 1, ceil_div(n_ctx, kBlk), false).bytes;
}
// Steps (of a warp, over a pair of blocks) that the call's CTAs make one after the other.
int64_t kv8_stream_steps(int m, int Hq, int Hk, int HD, int n_ctx) {
  const Plan p = plan(m, Hq / Hk, Hk, HD, 1, ceil_div(n_ctx, kBlk), false);
  const int64_t waves = ceil_div(int64_t(p.tiles) * Hk * p.splits, num_sms());
  return waves * ceil_div(ceil_div(n_ctx, kBlk), int64_t(p.splits) * 8 * Block<128, kInt8, false>::NB);
}
int kv8_stream_launches(int m, int Hq, int Hk, int HD, int n_ctx) {
  return launches(plan(m, Hq / Hk, Hk, HD, 1, ceil_div(n_ctx, kBlk), false));
}
int kv8_stream_attention(const uint16_t* q, const uint8_t* k8, const uint8_t* v8, const float* ks, const float* vs,
                         const int32_t* positions, uint16_t* out, int m, int Hq, int Hk, int HD, int n_ctx, float scale, int type,
                         void* workspace, cudaStream_t stream) {
  const int nb = ceil_div(n_ctx, kBlk);
  Args a{q, k8, v8, ks, vs, positions, nullptr, out, nullptr, nullptr, int64_t(nb) * kBlk, m, Hq, Hk, n_ctx, nb, 0, 0, 1, 1,
         scale * 1.4426950408889634f, false};
  const Plan p = plan(m, Hq / Hk, Hk, HD, 1, nb, false);
  if (int rc = check("ckv_attention_kv8", a, HD, p.tiles)) return rc;
  if (HD == 128)
    return type == CKV_KV8_E4M3 ? launch_nt<128, kE4m3, false>(a, p, workspace, stream)
                                : launch_nt<128, kInt8, false>(a, p, workspace, stream);
  return type == CKV_KV8_E4M3 ? launch_nt<64, kE4m3, false>(a, p, workspace, stream)
                              : launch_nt<64, kInt8, false>(a, p, workspace, stream);
}

}  // namespace ckv

using namespace ckv;

extern "C" int64_t ckv_attention_blocks_workspace_size(int m, int n_q_heads, int n_kv_heads, int head_dim, int top, int bits) {
  if (m <= 0 || top <= 0 || !shape_ok(m, n_q_heads, n_kv_heads, head_dim, 1)) return 0;
  return plan(m, n_q_heads / n_kv_heads, n_kv_heads, head_dim, bits / 8, top, true).bytes;
}

extern "C" int ckv_attention_blocks_launches(int m, int n_q_heads, int n_kv_heads, int head_dim, int top, int bits) {
  if (m <= 0 || top <= 0 || !shape_ok(m, n_q_heads, n_kv_heads, head_dim, 1)) return 0;
  const Plan p = plan(m, n_q_heads / n_kv_heads, n_kv_heads, head_dim, bits / 8, top, true);
  return launches(p) * ceil_div(m, run_tokens(p));
}

extern "C" int ckv_attention_blocks(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                    const int32_t* positions, const int32_t* blocks, uint16_t* out, int m, int n_q_heads,
                                    int n_kv_heads, int head_dim, int n_ctx, int top, float scale, void* workspace,
                                    int64_t workspace_bytes, ckv_stream_t stream) {
  return attention_blocks("ckv_attention_blocks",
                          bf16_call(q, k_cache, v_cache, positions, blocks, out, m, n_q_heads, n_kv_heads, head_dim, n_ctx, top, scale,
                                    workspace, workspace_bytes, false),
                          false, stream);
}

extern "C" int ckv_attention_blocks_kv8(const uint16_t* q, const uint8_t* k8, const uint8_t* v8, const float* k_scale,
                                        const float* v_scale, const int32_t* positions, const int32_t* blocks, uint16_t* out,
                                        int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx, int top, float scale,
                                        int type, void* workspace, int64_t workspace_bytes, ckv_stream_t stream) {
  return attention_blocks("ckv_attention_blocks_kv8",
                          kv8_call(q, k8, v8, k_scale, v_scale, positions, blocks, out, m, n_q_heads, n_kv_heads, head_dim, n_ctx, top,
                                   scale, type, workspace, workspace_bytes, false),
                          true, stream);
}

extern "C" int64_t ckv_attention_sparse_workspace_size(int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx, int top,
                                                       int cache_bits, int build_digest) {
  if (m <= 0 || top <= 0 || !shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) return 0;
  return sparse_space(m, n_q_heads, n_kv_heads, head_dim, cache_bits / 8, n_ctx, top, build_digest != 0).total();
}

extern "C" int ckv_attention_sparse(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                    const int8_t* dig_codes, const float* dig_scale, const int32_t* positions, int32_t* blocks,
                                    uint16_t* out, int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx, int top, int sink,
                                    int recent, float scale, void* workspace, int64_t workspace_bytes, ckv_stream_t stream) {
  const bool build = dig_codes == nullptr;
  CKV_REQUIRE(build == (dig_scale == nullptr), "ckv_attention_sparse: digest pointers");
  if (int rc = check_space("ckv_attention_sparse", m, n_q_heads, n_kv_heads, head_dim, 2, n_ctx, top, build, workspace,
                           workspace_bytes))
    return rc;
  if (m == 0) return CKV_OK;
  const SparseSpace x = sparse_space(m, n_q_heads, n_kv_heads, head_dim, 2, n_ctx, top, build);
  int8_t* built = nullptr;
  float* built_scale = nullptr;
  if (build) {
    dig_codes = built = reinterpret_cast<int8_t*>(static_cast<uint8_t*>(workspace) + x.step);
    dig_scale = built_scale = reinterpret_cast<float*>(built + int64_t(n_kv_heads) * ceil_div(n_ctx, kBlk) * 2 * head_dim);
  }
  // every step is checked before the first is launched
  const Call c = bf16_call(q, k_cache, v_cache, positions, blocks, out, m, n_q_heads, n_kv_heads, head_dim, n_ctx, top, scale, workspace,
                           x.step, true);
  if (int rc = check_call("ckv_attention_sparse", c, false)) return rc;
  if (int rc = block_select_check(q, dig_codes, dig_scale, positions, blocks, m, n_q_heads, n_kv_heads, head_dim, n_ctx, top, sink, recent,
                                  workspace, x.step))
    return rc;
  if (build)
    if (int rc = ckv_block_digest(k_cache, int64_t(n_ctx) * head_dim, head_dim, n_ctx, n_ctx, 0, nullptr, built, built_scale, n_kv_heads,
                                  head_dim, n_ctx, stream))
      return rc;
  if (int rc = ckv_block_select(q, dig_codes, dig_scale, positions, blocks, m, n_q_heads, n_kv_heads, head_dim, n_ctx, top, sink,
                                recent, workspace, x.step, stream))
    return rc;
  return launch_call(c, as_stream(stream));
}

extern "C" int ckv_attention_sparse_kv8(const uint16_t* q, const uint8_t* k8, const uint8_t* v8, const float* k_scale,
                                        const float* v_scale, const int8_t* dig_codes, const float* dig_scale,
                                        const int32_t* positions, int32_t* blocks, uint16_t* out, int m, int n_q_heads,
                                        int n_kv_heads, int head_dim, int n_ctx, int top, int sink, int recent, float scale, int type,
                                        void* workspace, int64_t workspace_bytes, ckv_stream_t stream) {
  if (int rc = check_space("ckv_attention_sparse_kv8", m, n_q_heads, n_kv_heads, head_dim, 1, n_ctx, top, false, workspace,
                           workspace_bytes))
    return rc;
  if (m == 0) return CKV_OK;
  const Call c = kv8_call(q, k8, v8, k_scale, v_scale, positions, blocks, out, m, n_q_heads, n_kv_heads, head_dim, n_ctx, top, scale, type,
                          workspace, workspace_bytes, true);
  if (int rc = check_call("ckv_attention_sparse_kv8", c, true)) return rc;
  if (int rc = ckv_block_select(q, dig_codes, dig_scale, positions, blocks, m, n_q_heads, n_kv_heads, head_dim, n_ctx, top, sink,
                                recent, workspace, workspace_bytes, stream))
    return rc;
  return launch_call(c, as_stream(stream));
}
