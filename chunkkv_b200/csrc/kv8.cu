// The K/V cache held in 8 bits: quantising write, read back, and the block digests that
// the sparse attention's score reads.
//
// A block is 16 consecutive tokens of one KV head.  For X in {K, V}, with a the largest
// |x| of the block's written rows and qmax = 127 (int8) or 448 (e4m3):
//   scale = fp32(a / qmax), inv = fp32(qmax / a), code = rn(fp32(x * inv))
// and code * scale is the value held.  Each of the three is one correctly rounded fp32
// operation, so the codes are the same whatever computes them.  A block whose a is below
// 2^-100 (where qmax / a leaves fp32) holds zeros with scale 0.  Non-finite inputs are
// stored saturated (NaN as 0), left out of a, and reported in the device error word by the
// write that brings them.
//
// A block that is still being filled is requantised from its bf16 rows at every write:
// the rows written so far are kept in the cache's `tail`, and the rows of the block before it in
// `prev`.  So the codes do not depend on how the rows were split over appending writes, nor
// on rows that were written and taken back, as far as the start of the block before the
// one in progress (16 tokens at least).  A write that goes back further (or once more into an
// earlier block, before the next one is full) finds its block's earlier rows only as codes,
// and those are rounded a second time.
#include "ckv_common.cuh"

CKV_DEFINE_ERR_WORD(kv8)

namespace ckv {
namespace {

constexpr int kRows = CKV_PAGE_TOKENS;  // tokens per block
constexpr int kWarps = 4;  // 131,069 tokens, 8 heads: 126 us (6.4 TB/s); when chosen 133, with 2, 8, 16 warps per CTA 147, 156, 173
constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100
enum { kNone = 0, kInt8 = 1, kE4m3 = 2 };

struct WriteArgs {
  const uint16_t* src[2];  // K, V rows
  int64_t head_stride[2], row_stride[2];
  int32_t by_position, m, start;
  const int32_t* start_dev;
  int64_t src_rows;
  uint8_t* codes[2];  // [H][n_blocks * 16][D]
  float* scale[2];    // [H][n_blocks]
  uint16_t* tail;     // [2][H][16][D]
  int32_t* tail_end;  // [2][H]: one past the last token whose row the tail holds
  uint16_t* prev;     // [2][H][16][D]: the whole block before the tail's (may be null)
  int32_t* prev_end;  // [2][H]: one past its last token (0: none)
  int8_t* dig_codes;  // [H][n_blocks][2][D]
  float* dig_scale;   // [H][n_blocks]
  int H, n_ctx, n_blocks, grid_blocks, sides;
};

__device__ __forceinline__ uint32_t code4_int8(float a, float b, float c, float d, float inv) {
  // adding 1.5 * 2^23 rounds to the nearest whole number (ties to even), whose two's
  // complement is then the low byte; the product is rounded before it (no contraction)
  const float big = 12582912.0f;
  const uint32_t x = __float_as_uint(__fadd_rn(__fmul_rn(a, inv), big));
  const uint32_t y = __float_as_uint(__fadd_rn(__fmul_rn(b, inv), big));
  const uint32_t z = __float_as_uint(__fadd_rn(__fmul_rn(c, inv), big));
  const uint32_t w = __float_as_uint(__fadd_rn(__fmul_rn(d, inv), big));
  return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t code4_e4m3(float a, float b, float c, float d, float inv) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(__fmul_rn(b, inv)), "f"(__fmul_rn(a, inv)));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(__fmul_rn(d, inv)), "f"(__fmul_rn(c, inv)));
  return uint32_t(lo) | (uint32_t(hi) << 16);
}
template <int CT>
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d, float inv) {
  if constexpr (CT == kE4m3) return code4_e4m3(a, b, c, d, inv);
  return code4_int8(a, b, c, d, inv);
}
// two codes -> their values times the block's scale, as packed bf16
template <int CT>
__device__ __forceinline__ uint32_t value2(uint32_t two, float scale) {
  float a, b;
  if constexpr (CT == kE4m3) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(two)));
    asm("{\n\t.reg .b16 l, u;\n\tmov.b32 {l, u}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, u;\n\t}"
        : "=f"(a), "=f"(b)
        : "r"(h));
  } else {
    a = float(int8_t(two & 0xff));
    b = float(int8_t((two >> 8) & 0xff));
  }
  return pack_bf2(__fmul_rn(a, scale), __fmul_rn(b, scale));
}
// 16 bytes from global to shared memory, past L1 and the registers; complete after cp_async_wait
__device__ __forceinline__ void cp_async16(uint4* dst, const uint16_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ uint32_t bmax2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t bmin2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// One warp per (block, K | V, head): the whole block sits in the warp's registers (16 bytes
// per lane and pass, 4 KiB at head_dim 128, all loads in flight together), so the rows are
// read once, and nothing goes through shared memory.  CT == kNone keeps only the digest.
// Bound by HBM: 131,069 tokens of 8 heads with K's digest (825 MB) 137 us, 6.0 TB/s; a prompt of 5248
// tokens, whose rows are in L2, 3.9 us, and one token 2.4 us in a graph, the latency of a launch and of
// the tail's rows.  Five CTAs per SM (96 registers): left to the compiler, or with six, 147 and 4.2 us.  (The digest
// alone and head_dim 64 fit more of them.)
template <int HD, int CT>
__global__ void __launch_bounds__(kWarps * 32, HD == 128 && CT != kNone ? 5 : 1) kv8_write_kernel(const __grid_constant__ WriteArgs a) {
  constexpr int LPR = HD / 8;            // lanes per row
  constexpr int RPP = 32 / LPR;          // rows per pass
  constexpr int PASSES = kRows / RPP;    // 8 at HD = 128, 4 at HD = 64
  const int warp = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int bi = warp % a.grid_blocks, side = (warp / a.grid_blocks) % a.sides, h = warp / (a.grid_blocks * a.sides);
  pdl_wait();
  pdl_launch_next();
  if (h >= a.H) return;
  const int start = a.start_dev != nullptr ? *a.start_dev : a.start;
  if (start < 0 || int64_t(start) + a.m > a.n_ctx || (a.by_position && int64_t(start) + a.m > a.src_rows)) {
    if (warp == 0 && lane == 0) atomicOr(&g_err_word, CKV_DEV_ERR_POSITION_RANGE);
    return;
  }
  const int end = start + a.m;
  const int b0 = start / kRows, b = b0 + bi;
  if (int64_t(b) * kRows >= end) return;
  const int rows = min(kRows, end - b * kRows);              // written rows of the block
  const int old = bi == 0 ? start - b * kRows : 0;           // of them, from before this write
  const int r0 = lane / LPR, col = (lane % LPR) * 8;
  const uint16_t* src = a.src[side] + h * a.head_stride[side];
  const int64_t blk = int64_t(h) * a.n_blocks + b;
  int te = 0, prev_end = 0;  // what the tail and the block before it hold
  if (CT != kNone && bi == 0) {
    const int64_t at = int64_t(side) * a.H + h;
    te = a.tail_end[at];
    if (a.prev != nullptr) prev_end = a.prev_end[at];
  }
  uint4 x[PASSES];
  const uint16_t* row0 = src + (int64_t(b) * kRows + r0 - (a.by_position ? 0 : start)) * a.row_stride[side] + col;
  if (CT == kNone || old == 0) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
      x[p] = p * RPP + r0 < rows ? __ldg(reinterpret_cast<const uint4*>(row0 + p * RPP * a.row_stride[side])) : make_uint4(0u, 0u, 0u, 0u);
  } else {
    // earlier rows from the tail, whether or not it holds this block: all loads are in flight together
    const uint16_t* tail0 = a.tail + ((int64_t(side) * a.H + h) * kRows + r0) * HD + col;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int r = p * RPP + r0;
      const uint16_t* from = r < old ? tail0 + p * RPP * HD : row0 + p * RPP * a.row_stride[side];
      x[p] = r < rows ? *reinterpret_cast<const uint4*>(from) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  if constexpr (CT != kNone) {
    const int held = te > 0 && te / kRows == b ? te % kRows : 0;
    if (held < old) {
      // a write that goes back: from the block before the tail's, or the values of the codes
      const bool whole = prev_end == (b + 1) * kRows && held == 0;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int r = p * RPP + r0;
        if (r < old && r >= held) {
          if (whole) {
            x[p] = *reinterpret_cast<const uint4*>(a.prev + ((int64_t(side) * a.H + h) * kRows + r) * HD + col);
          } else {
            const uint2 c = *reinterpret_cast<const uint2*>(a.codes[side] + (blk * kRows + r) * HD + col);
            const float sc = a.scale[side][blk];
            x[p] = make_uint4(value2<CT>(c.x, sc), value2<CT>(c.x >> 16, sc), value2<CT>(c.y, sc), value2<CT>(c.y >> 16, sc));
          }
        }
      }
    }
  }
  // The rows of the block in progress stay in the tail and those of the block before it in prev, as
  // they came: what stands for an infinity goes by the block's largest value, which later rows may
  // raise.  A write that begins a block reads neither, so each of the two blocks' warps keeps its
  // own rows; else the warp that reads them writes them, so that no other warp can see them half
  // replaced, and rows of later blocks come to it through shared memory under the rest of its work
  // (248 tokens from the middle of a block 4.4 us, loaded at the end 6.1).
  const int keep = end % kRows, bl = end / kRows;
  const bool passed_on = CT != kNone && bi == 0 && start % kRows != 0 && bl != b;
  [[maybe_unused]] uint4* stage = nullptr;
  if constexpr (CT != kNone) {
    __shared__ uint4 s_rows[kWarps][2][PASSES * 32];
    stage = s_rows[threadIdx.x >> 5][0];
    if (passed_on) {
#pragma unroll 1  // few instructions and registers, for a path that long writes take once per head
      for (int p = 0; p < PASSES; ++p) {
        const int r = p * RPP + r0;
        const uint16_t* row = src + (int64_t(bl) * kRows + r - (a.by_position ? 0 : start)) * a.row_stride[side] + col;
        if (r < keep) cp_async16(&stage[p * 32 + lane], row);
        if (a.prev != nullptr && bl - 1 != b) cp_async16(&stage[(PASSES + p) * 32 + lane], row - kRows * a.row_stride[side]);
      }
    }
  }
  // (called last, or before the repairs below: in front of the sums it would hold everything up)
  auto keep_rows = [&] {
    const int64_t at = int64_t(side) * a.H + h;
    uint16_t *tail = a.tail + at * kRows * HD, *prev = a.prev + at * kRows * HD;
    if ((b == bl || (b == bl - 1 && a.prev != nullptr)) && (start % kRows == 0 || bi == 0)) {
      uint16_t* slot = b == bl ? tail : prev;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int r = p * RPP + r0;
        if (r < rows) *reinterpret_cast<uint4*>(slot + r * HD + col) = x[p];
      }
    }
    if (passed_on) {
      cp_async_wait();  // a lane reads back what it copied itself
#pragma unroll 1
      for (int p = 0; p < PASSES; ++p) {
        const int r = p * RPP + r0;
        if (r < keep) *reinterpret_cast<uint4*>(tail + r * HD + col) = stage[p * 32 + lane];
        if (a.prev != nullptr && bl - 1 != b) *reinterpret_cast<uint4*>(prev + r * HD + col) = stage[(PASSES + p) * 32 + lane];
      }
    }
    if (bi == 0 && lane == 0) {
      a.tail_end[at] = keep > 0 ? end : 0;
      if (bl > b) prev_end = bl * kRows;             // block bl - 1 is whole now
      else if (prev_end != b * kRows) prev_end = 0;  // b was taken up again: the block before it is not known
      if (a.prev != nullptr) a.prev_end[at] = prev_end;
    }
  };
  uint32_t mag = 0;  // largest |x| as bf16 bits, two at a time
#pragma unroll
  for (int p = 0; p < PASSES; ++p)
    mag = __vmaxu2(mag, __vmaxu2(__vmaxu2(x[p].x & 0x7fff7fffu, x[p].y & 0x7fff7fffu),
                                 __vmaxu2(x[p].z & 0x7fff7fffu, x[p].w & 0x7fff7fffu)));
  uint32_t amag = max(mag & 0xffffu, mag >> 16);
  amag = __reduce_max_sync(0xffffffffu, amag);
  const bool odd = amag >= 0x7f80u;
  if (odd) {  // rare: a non-finite row
    if constexpr (CT != kNone) keep_rows();
    amag = 0;
    bool fresh = false;  // reported by the write that brings it, not by those after it
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      uint16_t* e = reinterpret_cast<uint16_t*>(&x[p]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t mg = e[i] & 0x7fffu;
        if (mg < 0x7f80u) amag = max(amag, mg);
        else fresh |= p * RPP + r0 >= old;
        if (mg > 0x7f80u) e[i] = 0;
      }
    }
    amag = __reduce_max_sync(0xffffffffu, amag);
    if (__any_sync(0xffffffffu, fresh) && lane == 0) atomicOr(&g_err_word, CKV_DEV_ERR_NONFINITE);
    // an infinity becomes the block's largest value (the largest code)
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      uint16_t* e = reinterpret_cast<uint16_t*>(&x[p]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((e[i] & 0x7fffu) == 0x7f80u) e[i] = uint16_t((e[i] & 0x8000u) | amag);
    }
  }
  const float amax = __uint_as_float(amag << 16);
  const bool live = amax >= kTiny;
  if constexpr (CT != kNone) {
    const float qmax = CT == kE4m3 ? 448.0f : 127.0f;
    const float inv = live ? __fdiv_rn(qmax, amax) : 0.0f;
    if (lane == 0) a.scale[side][blk] = live ? __fdiv_rn(amax, qmax) : 0.0f;
    uint8_t* dst = a.codes[side] + blk * kRows * HD;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const uint32_t w[4] = {x[p].x, x[p].y, x[p].z, x[p].w};
      uint2 c;
      c.x = code4<CT>(lo_bf(w[0]), hi_bf(w[0]), lo_bf(w[1]), hi_bf(w[1]), inv);
      c.y = code4<CT>(lo_bf(w[2]), hi_bf(w[2]), lo_bf(w[3]), hi_bf(w[3]), inv);
      *reinterpret_cast<uint2*>(dst + (p * RPP + r0) * HD + col) = c;  // rows not written yet: zeros
    }
  }
  if (a.dig_codes != nullptr && side == 0) {
    // channel maxima and minima of the written rows, in this lane's 8 columns
    const uint32_t lowest = 0xff7fff7fu, highest = 0x7f7f7f7fu;  // largest finite bf16, both signs
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi[i] = lowest;
      lo[i] = highest;
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      if (p * RPP + r0 < rows) {
        const uint32_t w[4] = {x[p].x, x[p].y, x[p].z, x[p].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hi[i] = bmax2(hi[i], w[i]);
          lo[i] = bmin2(lo[i], w[i]);
        }
      }
    }
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hi[i] = bmax2(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
        lo[i] = bmin2(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
      }
    const float inv = live ? __fdiv_rn(127.0f, amax) : 0.0f;
    if (lane == 0) a.dig_scale[blk] = live ? __fdiv_rn(amax, 127.0f) : 0.0f;
    if (r0 < 2) {  // the first row's lanes write the maxima, the second row's the minima
      const uint32_t* w = r0 == 0 ? hi : lo;
      uint2 c;
      c.x = code4_int8(lo_bf(w[0]), hi_bf(w[0]), lo_bf(w[1]), hi_bf(w[1]), inv);
      c.y = code4_int8(lo_bf(w[2]), hi_bf(w[2]), lo_bf(w[3]), hi_bf(w[3]), inv);
      *reinterpret_cast<uint2*>(a.dig_codes + (blk * 2 + r0) * HD + col) = c;
    }
  }
  if constexpr (CT != kNone)
    if (!odd) keep_rows();
}

// Values of tokens [start, start + m) as bf16 rows [H][m][D]: a thread per 16 codes, one 16-byte
// load and two stores, and enough of them in flight: 131,069 tokens of 8 heads 130 us, 6.2 TB/s.
template <int HD, int CT>
__global__ void __launch_bounds__(256) kv8_read_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                       const float* __restrict__ ks, const float* __restrict__ vs,
                                                       uint16_t* __restrict__ ko, uint16_t* __restrict__ vo, int H,
                                                       int n_blocks, int start, int m) {
  pdl_wait();
  pdl_launch_next();
  constexpr int VPR = HD / 16;  // 16-byte vectors of codes per row
  const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t per_side = int64_t(H) * m * VPR;
  if (i >= 2 * per_side) return;
  const bool is_v = i >= per_side;
  const int64_t j = is_v ? i - per_side : i;
  const int c = int(j % VPR);
  const int64_t row = j / VPR;
  const int h = int(row / m), t = int(row % m) + start;
  const float scale = (is_v ? vs : ks)[int64_t(h) * n_blocks + t / kRows];
  const uint4 x = __ldg(reinterpret_cast<const uint4*>((is_v ? vc : kc) + (int64_t(h) * n_blocks * kRows + t) * HD + c * 16));
  uint4* dst = reinterpret_cast<uint4*>((is_v ? vo : ko) + row * HD + c * 16);
  dst[0] = make_uint4(value2<CT>(x.x, scale), value2<CT>(x.x >> 16, scale), value2<CT>(x.y, scale),
                      value2<CT>(x.y >> 16, scale));
  dst[1] = make_uint4(value2<CT>(x.z, scale), value2<CT>(x.z >> 16, scale), value2<CT>(x.w, scale),
                      value2<CT>(x.w >> 16, scale));
}

template <int HD, int CT>
int launch_write(const WriteArgs& a, cudaStream_t stream) {
  const int64_t warps = int64_t(a.grid_blocks) * a.sides * a.H;
  launch_pdl(kv8_write_kernel<HD, CT>, dim3(ceil_div(warps, kWarps)), dim3(kWarps * 32), 0, stream, a);
  CKV_LAUNCH_CHECK("ckv_kv8_write");
  return CKV_OK;
}

int check_source(const char* name, const uint16_t* p, int64_t head_stride, int64_t row_stride, int HD) {
  CKV_REQUIRE(p && aligned16(p), "%s: rows must be non-null and 16-byte aligned", name);
  CKV_REQUIRE(row_stride >= HD && row_stride % 8 == 0 && head_stride % 8 == 0 && head_stride >= 0,
              "%s: strides must be multiples of 8 elements (row stride at least head_dim)", name);
  return CKV_OK;
}

int check_range(const char* name, int m, int start, const int32_t* start_dev, int by_position, int64_t src_rows,
                int n_kv_heads, int n_ctx) {
  CKV_REQUIRE(n_kv_heads > 0 && n_kv_heads <= 65535 && n_ctx > 0 && n_ctx <= (1 << 30) && m >= 0, "%s: bad sizes", name);
  CKV_REQUIRE(m <= n_ctx, "%s: %d rows for a context of %d", name, m, n_ctx);
  CKV_REQUIRE(src_rows >= m, "%s: %lld source rows, %d to write", name, static_cast<long long>(src_rows), m);
  if (start_dev == nullptr) {
    CKV_REQUIRE(start >= 0 && int64_t(start) + m <= n_ctx, "%s: tokens [%d, %lld) outside the context of %d", name, start,
                static_cast<long long>(start) + m, n_ctx);
    CKV_REQUIRE(!by_position || int64_t(start) + m <= src_rows, "%s: source has %lld rows, position %d asked for", name,
                static_cast<long long>(src_rows), start + m - 1);
  }
  return CKV_OK;
}

}  // namespace
}  // namespace ckv

using namespace ckv;

extern "C" int ckv_kv8_write(const uint16_t* k, const uint16_t* v, int64_t k_head_stride, int64_t k_row_stride,
                             int64_t v_head_stride, int64_t v_row_stride, int64_t src_rows, int by_position, int m,
                             int start, const int32_t* start_dev, uint8_t* k8, uint8_t* v8, float* k_scale,
                             float* v_scale, uint16_t* tail, int32_t* tail_end, uint16_t* prev, int32_t* prev_end,
                             int8_t* dig_codes, float* dig_scale, int n_kv_heads, int head_dim, int n_ctx, int type,
                             ckv_stream_t stream) {
  CKV_REQUIRE(k8 && v8 && k_scale && v_scale && tail && tail_end, "ckv_kv8_write: null pointer");
  CKV_REQUIRE(aligned16(k8) && aligned16(v8) && aligned16(tail) && aligned16(prev),
              "ckv_kv8_write: the cache must be 16-byte aligned");
  CKV_REQUIRE((prev == nullptr) == (prev_end == nullptr), "ckv_kv8_write: prev pointers");
  CKV_REQUIRE((dig_codes == nullptr) == (dig_scale == nullptr) && aligned16(dig_codes), "ckv_kv8_write: digest pointers");
  CKV_REQUIRE(type == CKV_KV8_INT8 || type == CKV_KV8_E4M3, "ckv_kv8_write: type %d", type);
  if (head_dim != 64 && head_dim != 128) {
    set_error("ckv_kv8_write: head_dim %d (64 or 128)", head_dim);
    return CKV_ERR_UNSUPPORTED;
  }
  if (int rc = check_range("ckv_kv8_write", m, start, start_dev, by_position, src_rows, n_kv_heads, n_ctx)) return rc;
  if (m == 0) return CKV_OK;
  if (int rc = check_source("ckv_kv8_write: k", k, k_head_stride, k_row_stride, head_dim)) return rc;
  if (int rc = check_source("ckv_kv8_write: v", v, v_head_stride, v_row_stride, head_dim)) return rc;
  const int n_blocks = ceil_div(n_ctx, kRows);
  const int off = start_dev != nullptr ? kRows - 1 : start % kRows;
  WriteArgs a{{k, v}, {k_head_stride, v_head_stride}, {k_row_stride, v_row_stride}, by_position, m, start, start_dev,
              src_rows, {k8, v8}, {k_scale, v_scale}, tail, tail_end, prev, prev_end, dig_codes, dig_scale, n_kv_heads, n_ctx, n_blocks,
              ceil_div(int64_t(off) + m, kRows), 2};
  CKV_REQUIRE(int64_t(a.grid_blocks) * 2 * n_kv_heads < (int64_t(1) << 31), "ckv_kv8_write: too many blocks");
  const cudaStream_t s = as_stream(stream);
  if (head_dim == 128)
    return type == CKV_KV8_E4M3 ? launch_write<128, kE4m3>(a, s) : launch_write<128, kInt8>(a, s);
  return type == CKV_KV8_E4M3 ? launch_write<64, kE4m3>(a, s) : launch_write<64, kInt8>(a, s);
}

extern "C" int ckv_block_digest(const uint16_t* k, int64_t head_stride, int64_t row_stride, int64_t src_rows, int m,
                                int start, const int32_t* start_dev, int8_t* dig_codes, float* dig_scale, int n_kv_heads,
                                int head_dim, int n_ctx, ckv_stream_t stream) {
  CKV_REQUIRE(dig_codes && dig_scale && aligned16(dig_codes), "ckv_block_digest: null or unaligned digest");
  if (head_dim != 64 && head_dim != 128) {
    set_error("ckv_block_digest: head_dim %d (64 or 128)", head_dim);
    return CKV_ERR_UNSUPPORTED;
  }
  if (int rc = check_range("ckv_block_digest", m, start, start_dev, 1, src_rows, n_kv_heads, n_ctx)) return rc;
  if (m == 0) return CKV_OK;
  if (int rc = check_source("ckv_block_digest: k", k, head_stride, row_stride, head_dim)) return rc;
  const int n_blocks = ceil_div(n_ctx, kRows);
  const int off = start_dev != nullptr ? kRows - 1 : start % kRows;
  WriteArgs a{{k, nullptr}, {head_stride, 0}, {row_stride, 0}, 1, m, start, start_dev, src_rows, {nullptr, nullptr},
              {nullptr, nullptr}, nullptr, nullptr, nullptr, nullptr, dig_codes, dig_scale, n_kv_heads, n_ctx, n_blocks,
              ceil_div(int64_t(off) + m, kRows), 1};
  CKV_REQUIRE(int64_t(a.grid_blocks) * n_kv_heads < (int64_t(1) << 31), "ckv_block_digest: too many blocks");
  const cudaStream_t s = as_stream(stream);
  return head_dim == 128 ? launch_write<128, kNone>(a, s) : launch_write<64, kNone>(a, s);
}

extern "C" int ckv_kv8_read(const uint8_t* k8, const uint8_t* v8, const float* k_scale, const float* v_scale,
                            uint16_t* k_out, uint16_t* v_out, int n_kv_heads, int head_dim, int n_ctx, int start, int m,
                            int type, ckv_stream_t stream) {
  CKV_REQUIRE(type == CKV_KV8_INT8 || type == CKV_KV8_E4M3, "ckv_kv8_read: type %d", type);
  CKV_REQUIRE(n_kv_heads > 0 && n_ctx > 0 && n_ctx <= (1 << 30) && m >= 0 && start >= 0 && int64_t(start) + m <= n_ctx,
              "ckv_kv8_read: tokens [%d, %lld) outside the context of %d", start, static_cast<long long>(start) + m, n_ctx);
  if (head_dim != 64 && head_dim != 128) {
    set_error("ckv_kv8_read: head_dim %d (64 or 128)", head_dim);
    return CKV_ERR_UNSUPPORTED;
  }
  if (m == 0) return CKV_OK;
  CKV_REQUIRE(k8 && v8 && k_scale && v_scale && k_out && v_out, "ckv_kv8_read: null pointer");
  CKV_REQUIRE(aligned16(k8) && aligned16(v8) && aligned16(k_out) && aligned16(v_out),
              "ckv_kv8_read: tensors must be 16-byte aligned");
  const int64_t threads = 2 * int64_t(n_kv_heads) * m * (head_dim / 16);
  CKV_REQUIRE(threads / 256 < (int64_t(1) << 31) - 1, "ckv_kv8_read: too many rows");
  const dim3 grid(unsigned((threads + 255) / 256));
  const int nb = ceil_div(n_ctx, kRows);
  const cudaStream_t s = as_stream(stream);
#define CKV_READ(HD, CT) \
  launch_pdl(kv8_read_kernel<HD, CT>, grid, dim3(256), 0, s, k8, v8, k_scale, v_scale, k_out, v_out, n_kv_heads, nb, start, m)
  if (head_dim == 128) {
    if (type == CKV_KV8_E4M3) CKV_READ(128, kE4m3);
    else CKV_READ(128, kInt8);
  } else {
    if (type == CKV_KV8_E4M3) CKV_READ(64, kE4m3);
    else CKV_READ(64, kInt8);
  }
#undef CKV_READ
  CKV_LAUNCH_CHECK("ckv_kv8_read");
  return CKV_OK;
}
