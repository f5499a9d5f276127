// Attention over the 8-bit K/V cache (one fp32 scale per KV head and block of 16 tokens).
//
// Few packed rows (token x head of a group), and more over short contexts, stream the cache
// through attention_blocks.cu; the others the tcgen05 kernel below takes in 128-row tiles.
//
// It is the bf16 kernel's scheme (attention_tc.cu: two Q tiles per CTA, S and P in TMEM,
// lazy rescale, persistent items, key splits) with the operands made on the SM: a warpgroup
// of converters reads the codes from global memory (16 bytes per lane and load, one tile
// ahead in registers) and writes them as fp16 into the 128B-swizzled operand tiles.  Both
// code types are exact in fp16, so is q scaled by a power of two per row, and the block
// scales never touch the tensor core:
//   S (row, key) = q . code            tcgen05.mma kind::f16
//   x            = S c_b,  c_b = row factor * K scale of the key's block (8 blocks a tile)
//   P'           = 2^(x - m + 7) * (V scale of the block / reference), rounded to fp16
//   O           += P' code             tcgen05.mma, A = P' from TMEM
// The scale of a whole 16-column group folds into constants the softmax uses anyway: the
// group's maximum is scaled once, the exponent's multiply-add takes c_b and
// log2(V scale / reference) - m, and the group's sum of P' is divided by the V scale once.
// So the softmax, which bounds the kernel (issue slots), costs per score what it costs over
// a bf16 cache.  The reference is the power of two at or above the item's largest V scale:
// P' stays below 2^15 (2^8 of lazy growth, 2^7 of bias) and keeps 11 bits down to 2^-21 of
// a row's largest weight.
// Warps: 0..3 and 4..7 softmax / epilogue of Q tiles 0 and 1, 8..11 converters, 12 item
// scheduler, 13 MMA issuer and TMEM owner, 14 and 15 idle.  The 512 threads start with 128
// registers each; setmaxnreg moves them to the softmax warps (168 + 104 + 72: 65,536 in all).
//
// Measured (28 query heads over 4, head_dim 128): 5248 causal rows 246 us, 0.80 PFLOP/s (over a
// bf16 cache 218 us); 938 rows spread over 5248 keys 77 us (78); 123 rows at the end of 5371 keys
// 32 us (39).  The tensor pipe and the exponentials are each 38 % busy: what bounds a tile is the
// chain S -> softmax -> P V of each Q tile, of which two overlap.
#include <algorithm>
#include <functional>
#include <mutex>
#include <type_traits>

#include "ckv_common.cuh"

CKV_DEFINE_ERR_WORD(attention_kv8)

#include "attention_split.cuh"

namespace ckv {
// attention_blocks.cu
int64_t kv8_stream_workspace(int m, int Hq, int Hk, int HD, int n_ctx);
int kv8_stream_launches(int m, int Hq, int Hk, int HD, int n_ctx);
int64_t kv8_stream_steps(int m, int Hq, int Hk, int HD, int n_ctx);
int kv8_stream_attention(const uint16_t* q, const uint8_t* k8, const uint8_t* v8, const float* ks, const float* vs,
                         const int32_t* positions, uint16_t* out, int m, int Hq, int Hk, int HD, int n_ctx, float scale, int type,
                         void* workspace, cudaStream_t stream);
namespace {

constexpr int kBlk = CKV_PAGE_TOKENS;
constexpr int KS = 2;  // K stages
constexpr int VS = 2;  // V stages
constexpr int GRP = BN / kBlk;  // scale blocks per key tile
constexpr int kScaleSlots = 4;  // tiles whose block scales are held at once
constexpr int kThreads = 512;
constexpr int kWarpConv = 8, kWarpSched = 12, kWarpMma = 13;
constexpr uint32_t TMEM_COLS = 512;  // S/P of tile w at [128w, 128w+128), O of tile w at 256+128w
constexpr uint32_t O_COL = 256;
constexpr float kPBits = 7.0f;  // P' is 2^7 times its weight
constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100
constexpr int kRegsSoftmax = 168, kRegsConv = 104, kRegsRest = 72;
static_assert(8 * kRegsSoftmax + 4 * kRegsConv + 4 * kRegsRest == 16 * 128, "the split is what the launch holds");

template <int HD>
struct Cfg {
  static constexpr uint32_t Q_BYTES = BM * HD * 2;
  static constexpr uint32_t KV_TILE = BN * HD * 2;
  static constexpr uint32_t SMEM_NEED = 1024 + NQ * Q_BYTES + (KS + VS) * KV_TILE +
                                        kItemSlots * (sizeof(Item) + NQ * BM * 4) + kStageBytes +
                                        kScaleSlots * GRP * 12 + 64 + 40 * 8 + 16;
  // at least 120 KiB so two CTAs never share an SM: each allocates all 512 TMEM columns
  static constexpr uint32_t SMEM = SMEM_NEED > 120 * 1024 ? SMEM_NEED : 120 * 1024;
  static constexpr uint32_t IDESC_S = (1u << 4) | (uint32_t(BN >> 3) << 17) | (uint32_t(BM >> 4) << 24);  // fp16 operands
  static constexpr uint32_t IDESC_PV = (1u << 4) | (uint32_t(HD >> 3) << 17) | (uint32_t(BM >> 4) << 24) | (1u << 16);
};

// four codes -> two pairs of fp16, exactly
template <bool E4M3>
__device__ __forceinline__ uint2 widen4(uint32_t w) {
  uint2 r;
  if constexpr (E4M3) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(r.x), "=r"(r.y)
        : "r"(w));
  } else {
    // 0x6400 + u is the fp16 number 1024 + u, u = code + 128: minus 1152 is the code
    const uint32_t u = w ^ 0x80808080u, magic = 0x64646464u;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(r.x) : "r"(__byte_perm(u, magic, 0x4140)), "r"(0x64806480u));
    asm("sub.f16x2 %0, %1, %2;" : "=r"(r.y) : "r"(__byte_perm(u, magic, 0x4342)), "r"(0x64806480u));
  }
  return r;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// two floats from shared memory, where the code says (a hoisted load would hold registers)
__device__ __forceinline__ float2 lds2(const float* p) {
  float2 r;
  asm volatile("ld.volatile.shared.v2.f32 {%0,%1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(smem_u32(p)));
  return r;
}
// 16 TMEM columns from registers; complete after tmem_st_wait
__device__ __forceinline__ void tmem_st16_issue(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// The MMA warp stays converged and its operands warp-uniform, so that descriptors live in
// uniform registers (values that vary come from warp reductions); `lead` (one lane)
// predicates the issue alone.  Issued from a one-lane branch, each tcgen05.mma waited for its
// operands to be moved there: a 5248-token prompt took 441 us instead of 374.
__device__ __forceinline__ uint32_t elect_lead() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p;
}
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void commit_lead(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}
__device__ __forceinline__ void conv_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// A warp's 32 rows (32 sub ..) of a Q tile as fp16, each times the power of two that puts its
// largest value in [2^14, 2^15): exact down to 2^-38 of it.  `base`: the tile's first token and
// head; n_tok tokens of it exist.  HD / 8 lanes read one row.  Returns the inverse of the power
// of this thread's row.  Not inlined: it runs once per item, and its registers stay out of the
// softmax loop's.
template <int HD>
__device__ __noinline__ float place_q_rows(const uint16_t* base, uint8_t* tile, int Hq, int G, int n_tok, int sub) {
  constexpr int LPR = HD / 8, RPP = 32 / LPR, PASSES = 32 / RPP;  // lanes per row, rows per pass
  const int lane = threadIdx.x & 31, ch = lane % LPR;
  const uint32_t inv_g = (65536 + G - 1) / G;  // r / G for r < 128
  constexpr int B = 4;  // passes whose loads are in flight together; the next ones under these
  uint32_t mine = 127;
  uint4 z[B], y[B];
  auto load = [&](int p0, uint4(&x)[B]) {
#pragma unroll
    for (int p = 0; p < B; ++p) {
      const int rr = sub * 32 + (p0 + p) * RPP + lane / LPR, tq = int((uint32_t(rr) * inv_g) >> 16);
      x[p] = p0 < PASSES && tq < n_tok
                 ? __ldg(reinterpret_cast<const uint4*>(base + (int64_t(tq) * Hq + (rr - tq * G)) * HD) + ch)
                 : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  load(0, z);
  // rolled: the code runs once per item, and most of it would be instruction fetches
#pragma unroll 1
  for (int p0 = 0; p0 < PASSES; p0 += B) {
    load(p0 + B, y);
#pragma unroll
    for (int p = 0; p < B; ++p) {
      const uint32_t mg = __vmaxu2(__vmaxu2(z[p].x & 0x7fff7fffu, z[p].y & 0x7fff7fffu),
                                   __vmaxu2(z[p].z & 0x7fff7fffu, z[p].w & 0x7fff7fffu));
      uint32_t am = max(mg & 0xffffu, mg >> 16);
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) am = max(am, __shfl_xor_sync(0xffffffffu, am, o));
      const int sh = am == 0 ? 0 : max(-126, min(126, 14 + 127 - int(am >> 7)));
      const float up = __uint_as_float(uint32_t(sh + 127) << 23);
      const int rr = sub * 32 + (p0 + p) * RPP + lane / LPR;
      *reinterpret_cast<uint4*>(tile + (ch >> 3) * ATOM_BYTES + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4)) =
          make_uint4(pack_h2(lo_bf(z[p].x) * up, hi_bf(z[p].x) * up), pack_h2(lo_bf(z[p].y) * up, hi_bf(z[p].y) * up),
                     pack_h2(lo_bf(z[p].z) * up, hi_bf(z[p].z) * up), pack_h2(lo_bf(z[p].w) * up, hi_bf(z[p].w) * up));
      // the exponent goes to the lane that owns the row
      const uint32_t e = __shfl_sync(0xffffffffu, uint32_t(127 - sh), (lane % RPP) * LPR);
      if (lane / RPP == p0 + p) mine = e;
    }
#pragma unroll
    for (int p = 0; p < B; ++p) z[p] = y[p];
  }
  return __uint_as_float(mine << 23);
}

struct Args {
  const uint16_t* q;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int32_t* positions;
  uint16_t* out;
  float* part_o;
  float2* part_ml;
  unsigned* sched;  // next slot, zero at launch (null: CTA c takes slots c, c + gridDim.x, ...)
  int M, Hq, Hk, n_ctx, n_blocks, tps, max_splits, blocks;
  float scale_log2;
};

// Item.pad0: last key that any of its rows sees (-1: none), pad1: Q tiles that hold rows.
// Slots as for Item, row blocks outermost within a group: longest first over all heads.
template <int HD, bool E4M3>
__global__ void __launch_bounds__(kThreads, 1) attention_kv8_kernel(const __grid_constant__ Args a) {
  using C = Cfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                      // [NQ][Q_BYTES]
  uint8_t* sK = sQ + NQ * C::Q_BYTES;      // [KS][KV_TILE]
  uint8_t* sV = sK + KS * C::KV_TILE;      // [VS][KV_TILE]
  Item* items = reinterpret_cast<Item*>(sV + VS * C::KV_TILE);                    // [kItemSlots]
  int* s_pos = reinterpret_cast<int*>(items + kItemSlots);                        // [kItemSlots][NQ * BM]
  uint32_t* s_stage = reinterpret_cast<uint32_t*>(s_pos + kItemSlots * NQ * BM);  // [8 warps][32][20]
  float* s_ks = reinterpret_cast<float*>(s_stage + kStageBytes / 4);              // [kScaleSlots][GRP] K scale
  float* s_lv = s_ks + kScaleSlots * GRP;                                         // log2(V scale / reference) + 7
  float* s_iv = s_lv + kScaleSlots * GRP;                                         // reference / V scale
  float* s_ref = s_iv + kScaleSlots * GRP;                                        // [4] V scale references, by item
  float* s_red = s_ref + 4;                                                       // [4]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(s_red + 12);
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;
  uint64_t* v_empty = v_full + VS;
  uint64_t* s_full = v_empty + VS;    // [NQ]
  uint64_t* p_full = s_full + NQ;     // [NQ]
  uint64_t* p_half = p_full + NQ;     // [NQ]: the first 64 keys' P is in place
  uint64_t* o_done = p_half + NQ;     // [NQ]
  uint64_t* q_ready = o_done + NQ;    // [NQ]: Q tile w of the next item is in place
  uint64_t* o_full = q_ready + NQ;    // [NQ]: the item's last P V of tile w is done
  uint64_t* item_full = o_full + NQ;  // [kItemSlots]
  uint64_t* item_empty = item_full + kItemSlots;  // [kItemSlots]
  uint64_t* claim = item_empty + kItemSlots;  // the converters have begun the item's last tile
  uint64_t* drain = claim + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  // from a warp reduction, so that the compiler knows it for warp-uniform
  const int warp = int(__reduce_max_sync(0xffffffffu, threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const int G = a.Hq / a.Hk;
  const int T = BM / G;  // tokens per Q tile
  const int n_slots = a.blocks * a.Hk * a.max_splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], 128);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&v_full[s], 128);
      mbar_init(&v_empty[s], 1);
    }
    for (int w = 0; w < NQ; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&p_full[w], 128);
      mbar_init(&p_half[w], 128);
      mbar_init(&o_done[w], 1);
      mbar_init(&q_ready[w], 128);
      mbar_init(&o_full[w], 1);
    }
    for (int s = 0; s < kItemSlots; ++s) {
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], 1 + NQ * 4 + 4);  // the MMA thread, each softmax and converter warp
    }
    mbar_init(claim, 1);
    mbar_init(drain, 1);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == kWarpMma) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __reduce_max_sync(0xffffffffu, *tmem_slot);
  // set-up done; q, the cache, the positions and the workspace belong to the kernels
  // before (dependent launch)
  pdl_wait();
  pdl_launch_next();

  if (warp >= kWarpSched) {
    regs_dec<kRegsRest>();
    if (warp == kWarpSched) {
      // ---------------------------------------------------------------- item scheduler
      int it = 0;
      int cursor = blockIdx.x;
      while (true) {
        Item rec{-1, 0, 0, 0, 0, 0, 0, 0};
        int pv[NQ * BM / 32];  // the item's token positions, lane + 32 j (clamped)
#pragma unroll
        for (int j = 0; j < NQ * BM / 32; ++j) pv[j] = -1;
        // one item ahead, no more: claimed when the converters begin the last tile of the item
        // before (an SM that claims as many as its ring holds keeps them from idle ones: 938
        // rows over 32,896 keys took 705 us instead of 373)
        if (it > 0) {
          const bool begun = warp_wait(claim, (it - 1) & 1, abort);
          if (!begun) break;
        }
        while (true) {
          // the first slot is the CTA's own; the counter hands out those behind
          int slot = cursor;
          if (a.sched != nullptr && cursor != int(blockIdx.x)) {
            if (lane == 0) slot = int(gridDim.x + atomicAdd(a.sched, 1u));
            slot = __shfl_sync(0xffffffffu, slot, 0);
          }
          cursor += gridDim.x;
          if (slot >= n_slots) break;
          const int gi = slot / (a.Hk * a.blocks);  // slot group
          const int rem = slot - gi * (a.Hk * a.blocks);
          const int hk = rem % a.Hk;
          const int rb = a.blocks - 1 - rem / a.Hk;
          const int t0 = rb * NQ * T;
          const int n_tok = min(NQ * T, a.M - t0);
          int mx = -1;
#pragma unroll
          for (int j = 0; j < NQ * BM / 32; ++j) {
            const int i = lane + 32 * j;
            int p = -1;
            if (i < n_tok) {
              p = a.positions[t0 + i];
              if (p >= a.n_ctx) {
                if (gi == 0 && hk == 0) atomicOr(&g_err_word, CKV_DEV_ERR_POSITION_RANGE);
                p = a.n_ctx - 1;
              }
              p = max(p, -1);
            }
            pv[j] = p;
            mx = max(mx, p);
          }
          mx = __reduce_max_sync(0xffffffffu, mx);
          const int kt_all = max(mx, 0) / BN + 1;  // key tiles 0 .. last visible key (one at least)
          const int n_split = (kt_all + a.tps - 1) / a.tps;
          const int z = n_split - a.max_splits + gi;  // see Item
          if (z >= 0) {
            rec = Item{rb, hk, z, n_split, z * a.tps, min(a.tps, kt_all - z * a.tps), mx, n_tok > T ? 2 : 1};
            break;
          }
        }
        const int s = it % kItemSlots;
        bool free_slot = true;
        if (lane == 0) free_slot = mbar_wait(&item_empty[s], ((it / kItemSlots) & 1) ^ 1, abort, &g_err_word);
        if (!__shfl_sync(0xffffffffu, free_slot ? 1 : 0, 0)) break;
#pragma unroll
        for (int j = 0; j < NQ * BM / 32; ++j) s_pos[s * NQ * BM + lane + 32 * j] = pv[j];
        __threadfence_block();
        __syncwarp();
        if (lane == 0) {
          items[s] = rec;
          mbar_arrive(&item_full[s]);
        }
        if (rec.rb < 0) break;
        ++it;
      }
    } else if (warp == kWarpMma) {
      // ---------------------------------------------------------------- MMA issuer
      const uint32_t lead = elect_lead();
      auto issue_s = [&](int w, int gt) {
        const uint32_t q0 = smem_u32(sQ + w * C::Q_BYTES);
        const uint32_t k0 = smem_u32(sK + (gt % KS) * C::KV_TILE);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = (kk >> 2) * ATOM_BYTES + (kk & 3) * 32;
          mma_ss(lead, tmem + w * BN, umma_desc_sw128(q0 + off), umma_desc_sw128(k0 + off), C::IDESC_S, kk > 0 ? 1u : 0u);
        }
        commit_lead(lead, &s_full[w]);
      };
      // half of P_w V (64 keys): P arrives in two halves, so the first runs under the
      // exponentials of the second
      auto issue_pv = [&](int w, int gt, int half, bool first) {
        const uint32_t v0 = smem_u32(sV + (gt % VS) * C::KV_TILE) + half * (BN / 2 * 128);
        const uint32_t pbuf = tmem + w * BN + half * (BN / 4);
#pragma unroll
        for (int kk = 0; kk < BN / 32; ++kk)
          mma_ts(lead, tmem + O_COL + w * 128, pbuf + kk * 8, umma_desc_sw128_mn(v0 + kk * 16 * 128, ATOM_BYTES), C::IDESC_PV,
                 (!first || kk > 0) ? 1u : 0u);
      };
      // Per Q tile (w = 0, 1) the parities of its key tiles and items so far, tile 1 in the high
      // half of each word.  The loops over w stay rolled: unrolled, their descriptors
      // do not fit this warpgroup's registers.
      bool ok = true;
      int g = 0;  // key tiles consumed (all items)
      uint32_t tiles_w = 0, items_w = 0;
      for (int it = 0; ok; ++it) {
        const int s = it % kItemSlots;
        if (!warp_wait(&item_full[s], (it / kItemSlots) & 1, abort)) {
          ok = false;
          break;
        }
        const int n_kt = __reduce_max_sync(0xffffffffu, items[s].rb < 0 ? -1 : items[s].n_kt);
        const int nq = __reduce_max_sync(0xffffffffu, items[s].pad1);
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[s]);
        if (n_kt < 0) break;
        if (!warp_wait(&k_full[g % KS], (g / KS) & 1, abort)) {
          ok = false;
          break;
        }
#pragma unroll 1
        for (int w = 0; w < nq; ++w) {
          if (!warp_wait(&q_ready[w], (items_w >> (16 * w)) & 1, abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          issue_s(w, g);
        }
        if (!ok) break;
        commit_lead(lead, &k_empty[g % KS]);
#pragma unroll 1
        for (int jw = 0; jw < n_kt * nq; ++jw) {
          const int j = nq == 2 ? jw >> 1 : jw, w = nq == 2 ? jw & 1 : 0;
          const int gt = g + j, nxt = gt + 1;
          if (!warp_wait(&p_half[w], ((tiles_w >> (16 * w)) + j) & 1, abort) ||
              (w == 0 && !warp_wait(&v_full[gt % VS], (gt / VS) & 1, abort))) {
            ok = false;
            break;
          }
          tc_fence_after();
          issue_pv(w, gt, 0, j == 0);
          if (!warp_wait(&p_full[w], ((tiles_w >> (16 * w)) + j) & 1, abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          issue_pv(w, gt, 1, false);
          commit_lead(lead, &o_done[w]);
          if (j + 1 == n_kt) commit_lead(lead, &o_full[w]);  // O of tile w is final
          if (w == nq - 1) commit_lead(lead, &v_empty[gt % VS]);
          if (j + 1 < n_kt) {
            if (w == 0 && !warp_wait(&k_full[nxt % KS], (nxt / KS) & 1, abort)) {
              ok = false;
              break;
            }
            tc_fence_after();
            issue_s(w, nxt);
            if (w == nq - 1) commit_lead(lead, &k_empty[nxt % KS]);
          }
        }
        g += n_kt;
        const uint32_t both = nq == 2 ? 0x00010001u : 0x00000001u;
        if (n_kt & 1) tiles_w ^= both;
        items_w ^= both;
      }
      if (!ok) {
        commit_lead(lead, drain);
        drain_wait(drain, 0);
      }
    }
  } else if (warp >= kWarpConv) {
    // ------------------------------------------------------------------- converters
    regs_dec<kRegsConv>();
    const int t = threadIdx.x - kWarpConv * 32;  // 0 .. 127
    constexpr int ATOMS = HD / 64;               // 64-column atoms of an operand tile
    constexpr int NCH = BN / 32 * ATOMS;         // 16-code chunks per thread and tile
    // chunk c4 of a 64-column atom in row r0 + 32 i: four lanes read 64 bytes of a row.  The
    // widened chunk is the 16-byte units 2 c4 and 2 c4 + 1 of the row, swizzled by row % 8:
    // the two rows of eight lanes differ in that bit, so a store's lanes hit distinct banks.
    const int r0 = t >> 2, c4 = t & 3;
    const uint32_t u0 = ((2u * c4) ^ (r0 & 7)) * 16u, u1 = u0 ^ 16u;
    auto load = [&](const uint8_t* src, int hk, int kt, int last, uint4(&x)[NCH]) {
      const uint8_t* p = src + (int64_t(hk) * a.n_blocks * kBlk + int64_t(kt) * BN + r0) * HD + c4 * 16;
      const int vis = last - kt * BN - r0;  // rows past it stay zero
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        x[i] = (i / ATOMS) * 32 <= vis ? __ldg(reinterpret_cast<const uint4*>(p + (i / ATOMS) * 32 * HD + (i % ATOMS) * 64))
                                       : make_uint4(0u, 0u, 0u, 0u);
    };
    auto store = [&](uint8_t* tile, const uint4(&x)[NCH]) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const uint2 p0 = widen4<E4M3>(x[i].x), p1 = widen4<E4M3>(x[i].y), p2 = widen4<E4M3>(x[i].z), p3 = widen4<E4M3>(x[i].w);
        uint8_t* row = tile + (i % ATOMS) * ATOM_BYTES + (r0 + (i / ATOMS) * 32) * 128;
        *reinterpret_cast<uint4*>(row + u0) = make_uint4(p0.x, p0.y, p1.x, p1.y);
        *reinterpret_cast<uint4*>(row + u1) = make_uint4(p2.x, p2.y, p3.x, p3.y);
      }
    };
    bool ok = true;
    int g = 0;  // key tiles converted (all items)
    for (int it = 0; ok; ++it) {
      const int s = it % kItemSlots;
      if (!warp_wait(&item_full[s], (it / kItemSlots) & 1, abort)) break;
      const Item rec = items[s];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[s]);
      if (rec.rb < 0) break;
      const int last = rec.pad0;
      uint4 x[NCH], y[NCH];
      load(a.k, rec.hk, rec.kt0, last, x);
      // the item's V scale reference: the power of two at or above its largest scale
      {
        const int b1 = min((rec.kt0 + rec.n_kt) * GRP, (last + kBlk) / kBlk);
        float mx = 0.f;
        for (int b = rec.kt0 * GRP + t; b < b1; b += 128) mx = fmaxf(mx, __ldg(a.vs + int64_t(rec.hk) * a.n_blocks + b));
        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(mx));
        if (lane == 0) s_red[warp - kWarpConv] = __uint_as_float((bits + 0x007fffffu) & 0x7f800000u);
        conv_barrier();
      }
      float ref = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
      ref = ref > 0.f ? ref : 1.0f;
      if (t == 0) s_ref[it & 3] = ref;
      conv_barrier();  // s_red may be rewritten for the next item
      for (int j = 0; j < rec.n_kt; ++j) {
        const int gt = g + j, kt = rec.kt0 + j;
        if (j + 1 == rec.n_kt && t == 0) mbar_arrive(claim);
        load(a.v, rec.hk, kt, last, y);
        float ks = 0.f, vs = 0.f;
        if (t < GRP && kt * BN + t * kBlk <= last) {
          const int64_t b = int64_t(rec.hk) * a.n_blocks + kt * GRP + t;
          ks = __ldg(a.ks + b);
          vs = __ldg(a.vs + b);
        }
        if (!warp_wait(&k_empty[gt % KS], ((gt / KS) & 1) ^ 1, abort)) {
          ok = false;
          break;
        }
        store(sK + (gt % KS) * C::KV_TILE, x);
        if (t < GRP) {
          // a block of zeros (scale 0) adds nothing whatever its weight: any scale will do
          const int sl = (gt % kScaleSlots) * GRP + t;
          s_ks[sl] = ks;
          // at least 2^-100 of the reference, so that the inverse is finite and the weights do not
          // underflow in the row's sum (their products round to 0 from 2^-31 on)
          const float rel = vs > 0.f ? fmaxf(vs / ref, kTiny) : 1.0f;
          s_lv[sl] = log2f(rel) + kPBits;
          s_iv[sl] = 1.0f / rel;
        }
        fence_async_smem();
        mbar_arrive(&k_full[gt % KS]);
        if (j + 1 < rec.n_kt) load(a.k, rec.hk, kt + 1, last, x);
        if (!warp_wait(&v_empty[gt % VS], ((gt / VS) & 1) ^ 1, abort)) {
          ok = false;
          break;
        }
        store(sV + (gt % VS) * C::KV_TILE, y);
        fence_async_smem();
        mbar_arrive(&v_full[gt % VS]);
      }
      g += rec.n_kt;
    }
  } else {
    // ------------------------------------------------- softmax / correction / epilogue
    regs_inc<kRegsSoftmax>();
    const int w = warp >> 2;         // Q tile of this warpgroup
    const int sub = warp & 3;        // TMEM sub-partition (lanes 32*sub .. +31)
    const int r = sub * 32 + lane;   // row in the Q tile == TMEM lane
    const int tr = r / G;            // token of the row in the Q tile
    const uint32_t lane_base = tmem + (uint32_t(sub * 32) << 16);
    const uint32_t sbuf = lane_base + w * BN;
    const uint32_t obuf = lane_base + O_COL + w * 128;

    // this thread's row of an item: whether it is real, and the last key it sees (padding rows
    // see every key: they never force the masked path on their warp)
    struct Row {
      bool valid;
      int pos;
    };
    auto take = [&](int it, Item& rec, Row& x) -> bool {
      const int s = it % kItemSlots;
      if (!warp_wait(&item_full[s], (it / kItemSlots) & 1, abort)) return false;
      rec = items[s];
      const int tt = w * T + tr;  // token index in the item
      x.valid = rec.rb >= 0 && r < T * G && tt < min(NQ * T, a.M - rec.rb * NQ * T);
      x.pos = x.valid ? s_pos[s * NQ * BM + tt] : a.n_ctx - 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[s]);
      return true;
    };
    auto place_q = [&](const Item& rec) -> float {
      const float f = place_q_rows<HD>(a.q + (int64_t(rec.rb * NQ * T + w * T) * a.Hq + rec.hk * G) * HD, sQ + w * C::Q_BYTES,
                                       a.Hq, G, min(T, min(NQ * T, a.M - rec.rb * NQ * T) - w * T), sub);
      fence_async_smem();
      mbar_arrive(&q_ready[w]);
      return a.scale_log2 * f;
    };

    int g = 0;   // key tiles seen (all items): the scale slots
    int gw = 0;  // of them, by this Q tile
    int iw = 0;  // items by this Q tile
    Item cur;
    Row row{false, 0};
    bool ok = take(0, cur, row);
    float factor = 0.f;
    if (ok && cur.rb >= 0 && w < cur.pad1) factor = place_q(cur);
    for (int it = 0; ok && cur.rb >= 0; ++it) {
      float m = -INFINITY, l = 0.f, ref = 1.0f;
      const bool mine = w < cur.pad1;  // the item has rows on this tile
      for (int j = 0; mine && j < cur.n_kt; ++j) {
        const int gt = g + j;
        if (!warp_wait(&s_full[w], (gw + j) & 1, abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (j == 0) ref = s_ref[it & 3];
        const int lim = row.pos - (cur.kt0 + j) * BN;  // keys at index > lim are masked
        const bool full = __all_sync(0xffffffffu, lim >= BN - 1);
        const float* ksl = s_ks + (gt % kScaleSlots) * GRP;
        const float* lvl = s_lv + (gt % kScaleSlots) * GRP;
        const float* ivl = s_iv + (gt % kScaleSlots) * GRP;
        // pass 1: row max; a 16-column group's raw maximum times its factor (>= 0).  S comes 32
        // columns at a time, the next 32 on their way while these are worked on (both passes).
        float mx = -INFINITY;
        uint32_t u[2][32];
        tmem_ld32_issue(sbuf, u[0]);
#pragma unroll
        for (int h = 0; h < BN / 32; ++h) {
          tmem_ld_wait(u[h & 1]);
          if (h + 1 < BN / 32) tmem_ld32_issue(sbuf + 32 * (h + 1), u[(h + 1) & 1]);
          uint32_t(&v)[32] = u[h & 1];
          if (!full) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * h + e > lim) v[e] = __float_as_uint(-INFINITY);
          }
          const float2 kq = lds2(ksl + 2 * h);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint32_t* x = v + 16 * b;
            float p = max3f(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]));
            float q2 = max3f(__uint_as_float(x[3]), __uint_as_float(x[4]), __uint_as_float(x[5]));
#pragma unroll
            for (int e = 6; e < 14; e += 4) {
              p = max3f(p, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
              q2 = max3f(q2, __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
            }
            p = max3f(p, __uint_as_float(x[14]), __uint_as_float(x[15]));
            mx = fmaxf(mx, fmaxf(p, q2) * ((b ? kq.y : kq.x) * factor));  // -inf * 0 is NaN, which fmaxf drops
          }
        }
        tmem_ld32_issue(sbuf, u[0]);  // pass 2's first columns, on their way during the rescale's test
        const float m_new = fmaxf(m, mx);
        const bool need = j > 0 && m_new > m + kRescaleThreshold;
        if (__any_sync(0xffffffffu, need)) {
          // O may be touched only after P(j-1) V(j-1) has landed
          if (!warp_wait(&o_done[w], (gw + j - 1) & 1, abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const float corr = need ? ex2_approx(m - m_new) : 1.0f;
          tmem_ld_wait(u[0]);
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            float o[32];
            tmem_ld32(obuf + c, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= corr;
            tmem_st32(obuf + c, o);
          }
          l *= corr;
        }
        if (j == 0 || need) m = m_new;
        // pass 2: P' = 2^(s c - m + log2(vs / ref) + 7), one packed multiply-add per pair, back
        // over S as fp16 pairs; masked keys give exactly 0.  A row that has seen no key yet
        // keeps m = -inf and takes 0 as its base.
        const float neg_m = m == -INFINITY ? 0.f : -m;
        auto pass2 = [&](auto all_visible) {
          constexpr bool kAll = decltype(all_visible)::value;
#pragma unroll
          for (int h = 0; h < BN / 32; ++h) {
            tmem_ld_wait(u[h & 1]);
            if (h + 1 < BN / 32) tmem_ld32_issue(sbuf + 32 * (h + 1), u[(h + 1) & 1]);
            uint32_t(&v)[32] = u[h & 1];
            const float2 kq = lds2(ksl + 2 * h), lv = lds2(lvl + 2 * h), iv = lds2(ivl + 2 * h);
            uint32_t out16[16];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const float cb = (b ? kq.y : kq.x) * factor, add = neg_m + (b ? lv.y : lv.x);
              const float2 sc2 = make_float2(cb, cb), nm2 = make_float2(add, add);
              float2 rs0 = make_float2(0.f, 0.f), rs1 = rs0;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int pr = 8 * b + e;
                const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[2 * pr]), __uint_as_float(v[2 * pr + 1])), sc2, nm2);
                float2 pv = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                if constexpr (!kAll) {
                  pv.x = 32 * h + 2 * pr <= lim ? pv.x : 0.f;
                  pv.y = 32 * h + 2 * pr + 1 <= lim ? pv.y : 0.f;
                }
                if (e & 1) rs1 = __fadd2_rn(rs1, pv);
                else rs0 = __fadd2_rn(rs0, pv);
                out16[pr] = pack_h2(pv.x, pv.y);
              }
              const float2 rs = __fadd2_rn(rs0, rs1);
              l = fmaf(rs.x + rs.y, b ? iv.y : iv.x, l);
            }
            // P of keys 32 h .. goes to columns 16 h .., whose scores were read before
            tmem_st16_issue(sbuf + 16 * h, out16);
            if (h == 1) {
              tmem_st_wait();
              tc_fence_before();
              mbar_arrive(&p_half[w]);
            }
          }
        };
        if (full) pass2(std::true_type{});
        else pass2(std::false_type{});
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[w]);
      }
      if (!ok) break;
      g += cur.n_kt;
      // the next item's Q tile, under this item's last P V
      Item nxt;
      Row nrow{false, 0};
      if (!take(it + 1, nxt, nrow)) {
        ok = false;
        break;
      }
      float nfactor = 0.f;
      if (nxt.rb >= 0 && w < nxt.pad1) nfactor = place_q(nxt);
      if (!mine) {
        cur = nxt, row = nrow, factor = nfactor;
        continue;
      }
      gw += cur.n_kt;
      if (!warp_wait(&o_full[w], iw & 1, abort)) {
        ok = false;
        break;
      }
      ++iw;
      tc_fence_after();
      uint32_t* stg = s_stage + warp * (32 * kStageStride);
      if (cur.n_split > 1) {
        // one slice of the keys: unnormalised O (times the reference) with its (max, sum), in the
        // column-chunk-major layout that the combine kernel reads, by 1 KiB bulk stores
        const int64_t blk = (int64_t((cur.rb * a.Hk + cur.hk) * a.max_splits + cur.split) * NQ + w) * BM * HD;
        float* gdst = a.part_o + blk + sub * 32 * 8;
        uint8_t* stg8 = reinterpret_cast<uint8_t*>(stg);
        const int swz = (lane >> 2) & 1;
        int chunk = 0;
        const bool rows_here = __any_sync(0xffffffffu, row.valid);  // a warp of padding rows stores nothing
#pragma unroll 1
        for (int c = 0; c < HD && rows_here; c += 32) {
          float o[32];
          tmem_ld32(obuf + c, o);
#pragma unroll
          for (int h = 0; h < 4; ++h, ++chunk) {
            uint8_t* buf = stg8 + (chunk & 1) * 1024;
            if (chunk >= 2) {  // the store that last read this buffer has read it
              if (lane == 0) bulk_wait_read<1>();
              __syncwarp();
            }
            float4* mine = reinterpret_cast<float4*>(buf + lane * 32);
            mine[swz] = make_float4(o[8 * h] * ref, o[8 * h + 1] * ref, o[8 * h + 2] * ref, o[8 * h + 3] * ref);
            mine[swz ^ 1] = make_float4(o[8 * h + 4] * ref, o[8 * h + 5] * ref, o[8 * h + 6] * ref, o[8 * h + 7] * ref);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              bulk_store(gdst + (c / 8 + h) * (BM * 8), buf, 1024);
              bulk_commit();
            }
          }
        }
        if (lane == 0) bulk_wait_read<0>();  // both buffers free for the next epilogue
        __syncwarp();
        if (row.valid) {
          const int64_t prow = int64_t((cur.rb * a.Hk + cur.hk) * a.max_splits + cur.split) * (NQ * BM) + w * BM + r;
          a.part_ml[prow] = make_float2(m, l);
        }
      } else {
        // 16 words of each row at a time through the warp's staging tile: four lanes per row,
        // eight rows per store instruction
        int64_t dst[4];
        {
          const int t0 = cur.rb * NQ * T;
          const int n_tok = min(NQ * T, a.M - t0);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int rq = sub * 32 + 8 * k + (lane >> 2);
            const int tq = rq / G, gq = rq - tq * G, ttq = w * T + tq;
            const bool vq = rq < T * G && ttq < n_tok;
            dst[k] = !vq ? -1 : (int64_t(t0 + ttq) * a.Hq + cur.hk * G + gq) * HD;
          }
        }
        const float inv = l > 0.f ? ref / l : 0.f;
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          float o[32];
          tmem_ld32(obuf + c, o);
          uint4* mine = reinterpret_cast<uint4*>(stg + lane * kStageStride);
#pragma unroll
          for (int qd = 0; qd < 4; ++qd)
            mine[qd] = make_uint4(pack_bf2(o[8 * qd] * inv, o[8 * qd + 1] * inv), pack_bf2(o[8 * qd + 2] * inv, o[8 * qd + 3] * inv),
                                  pack_bf2(o[8 * qd + 4] * inv, o[8 * qd + 5] * inv), pack_bf2(o[8 * qd + 6] * inv, o[8 * qd + 7] * inv));
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint4 x = reinterpret_cast<const uint4*>(stg + (8 * k + (lane >> 2)) * kStageStride)[lane & 3];
            if (dst[k] >= 0) *reinterpret_cast<uint4*>(a.out + dst[k] + c + (lane & 3) * 8) = x;
          }
          __syncwarp();
        }
      }
      // O has been read: the next item's first P V (which overwrites it) is issued only
      // after this warpgroup's next p_full
      tc_fence_before();
      cur = nxt, row = nrow, factor = nfactor;
    }
    // the split partials' bulk stores have written global memory before the CTA ends
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// attention_blocks.cu takes the call (16 packed rows of a KV head to a tile, each streaming the
// cache) with up to kStreamRows packed rows, and with more while its CTAs make few steps: a step
// takes 1.8 us, as much as 6 of them cost here what an item's start, epilogue and join do.  Streamed
// and in tiles, 28 heads over 4: 8 rows over 32,896 keys 35 and 40 us; 10 rows over 4096 / 8192 /
// 16,384 keys 13 / 17 / 26 (10 steps) and 19 / 22 / 26; 36 rows over 512 / 2048 / 4096 keys
// 11 / 17 / 24 (8 steps) and 20 / 19 / 22 us.
constexpr int kStreamRows = 64, kStreamSteps = 6;
bool use_tiles(int m, int Hq, int Hk, int HD, int n_ctx) {
  return int64_t(m) * (Hq / Hk) > kStreamRows && kv8_stream_steps(m, Hq, Hk, HD, n_ctx) > kStreamSteps;
}

// Costs in key-tile times (2.5 us at head_dim 128), fitted to the times of every split length at
// eight shapes of 36 to 938 rows over 2048 to 32,896 keys (within 5 % of the best choice at
// each): an item's start and epilogue, the same with fp32 partials, and the second launch that
// joins them, alone, per split (a row's splits are added one after the other) and per byte.
constexpr double kItemCost = 0.5, kSplitItemCost = 3.0, kJoinCost = 1.0, kJoinSplitCost = 0.1, kJoinBytes = 5e6;

constexpr int kMaxSms = 256;

// Time of a plan: the items' makespan when the SMs take them in slot order (longest first),
// followed exactly while they are few, for then it is the last wave that counts, and the join.
// Row block b is assumed to reach position (b + 1) / blocks * n_ctx (rows spread over the
// context) or n_ctx - m + (b + 1) * rows (the last m positions).
double plan_cost(int m, int blocks, int Hk, int G, int HD, int n_ctx, int tps, int sms, bool spread) {
  const int max_kt = ceil_div(n_ctx, BN);
  const bool split = tps < max_kt;
  const int max_splits = ceil_div(max_kt, tps);
  const double fixed = split ? kSplitItemCost : kItemCost;
  const int64_t rows = int64_t(NQ) * (BM / G);
  int64_t items = 0;
  double total = 0.0, makespan = 0.0;
  double heap[kMaxSms] = {};  // the SMs' finishing times, earliest first
  const bool follow = int64_t(blocks) * Hk * max_splits <= 6 * int64_t(sms);
  for (int gi = 0; gi < max_splits; ++gi)
    for (int b = blocks - 1; b >= 0; --b) {
      const int64_t reach = spread ? (int64_t(b) + 1) * n_ctx / blocks
                                   : std::max<int64_t>(1, n_ctx - m + std::min<int64_t>(m, (int64_t(b) + 1) * rows));
      const int kt = std::max(1, ceil_div(reach, BN));
      const int n_split = ceil_div(kt, tps);
      const int z = n_split - max_splits + gi;
      if (z < 0) continue;
      const double c = std::min(tps, kt - z * tps) + fixed;
      items += Hk;
      total += c * Hk;
      for (int h = 0; h < Hk && follow; ++h) {
        std::pop_heap(heap, heap + sms, std::greater<double>());
        heap[sms - 1] += c;
        makespan = std::max(makespan, heap[sms - 1]);
        std::push_heap(heap, heap + sms, std::greater<double>());
      }
    }
  if (!follow) makespan = total / sms + 0.5 * (std::min(tps, max_kt) + fixed);
  const double join =
      split ? kJoinCost + kJoinSplitCost * max_splits + double(items) * NQ * BM * (HD * 4 + 8) / kJoinBytes : 0.0;
  return makespan + join;
}

// The number of splits with the shortest time over both assumptions (no split included).  Kept
// per shape, the oldest forgotten (a plan takes up to 0.4 ms on the host).
SplitPlan tile_plan(int m, int Hq, int Hk, int HD, int n_ctx) {
  struct Entry {
    int m, Hq, Hk, HD, n_ctx, sms;
    SplitPlan plan;
  };
  constexpr int kKept = 256;
  static std::mutex mu;
  static Entry kept[kKept];
  static int n_kept = 0, oldest = 0;
  const int sms = std::min(num_sms(), kMaxSms);
  {
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < n_kept; ++i) {
      const Entry& e = kept[i];
      if (e.m == m && e.Hq == Hq && e.Hk == Hk && e.HD == HD && e.n_ctx == n_ctx && e.sms == sms) return e.plan;
    }
  }
  SplitPlan p;
  p.blocks = ceil_div(m, int64_t(NQ) * (BM / (Hq / Hk)));
  const int max_kt = ceil_div(n_ctx, BN);
  p.tps = max_kt;
  const int64_t whole = int64_t(p.blocks) * Hk;
  // splitting only pays while whole rows do not fill the SMs several times over; at most 32
  // splits (the combine gives each one lane)
  if (whole < 4 * int64_t(sms)) {
    auto cost = [&](int tps) {
      return plan_cost(m, p.blocks, Hk, Hq / Hk, HD, n_ctx, tps, sms, true) +
             plan_cost(m, p.blocks, Hk, Hq / Hk, HD, n_ctx, tps, sms, false);
    };
    double best = cost(max_kt);
    const int most = std::min(whole >= 2 * int64_t(sms) ? 4 : 32, max_kt / 2);
    for (int n = 2; n <= most; n = n < 16 ? n + 1 : (n < most ? std::min(most, n + n / 4) : most + 1)) {
      const int tps = ceil_div(max_kt, n);
      const double c = cost(tps);
      if (c < best) {
        best = c;
        p.tps = tps;
      }
    }
  }
  p.max_splits = ceil_div(max_kt, p.tps);
  p.bytes = p.max_splits > 1 ? int64_t(p.blocks) * Hk * p.max_splits * NQ * BM * (int64_t(HD) * 4 + 8) : 0;
  std::lock_guard<std::mutex> lock(mu);
  const int at = n_kept < kKept ? n_kept++ : (oldest = (oldest + 1) % kKept);
  kept[at] = {m, Hq, Hk, HD, n_ctx, sms, p};
  return p;
}

template <int HD, bool E4M3>
int launch_tiles(Args a, const SplitPlan& p, void* workspace, cudaStream_t stream) {
  auto kern = attention_kv8_kernel<HD, E4M3>;
  static int regs = 0;  // the register split needs what the kernel is launched with
  if (regs == 0) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess) {
      set_error("ckv_attention_kv8: cudaFuncGetAttributes: %s", cudaGetErrorString(cudaGetLastError()));
      return CKV_ERR_CUDA;
    }
    regs = fa.numRegs;
  }
  if (regs != 128) {
    set_error("ckv_attention_kv8: built with %d registers per thread, its register split needs 128", regs);
    return CKV_ERR_CUDA;
  }
  if (int rc = set_smem_limit(reinterpret_cast<const void*>(kern), Cfg<HD>::SMEM)) return rc;
  const int64_t n_slots = int64_t(p.blocks) * a.Hk * p.max_splits;
  CKV_REQUIRE(n_slots < (int64_t(1) << 31) - 4 * 1024 * 1024, "ckv_attention_kv8: too many work items");
  if (n_slots > num_sms()) {  // more than one item per CTA: they take them from a counter
    a.sched = static_cast<unsigned*>(workspace);
    if (cudaMemsetAsync(a.sched, 0, sizeof(unsigned), stream) != cudaSuccess) {
      set_error("ckv_attention_kv8: cudaMemsetAsync: %s", cudaGetErrorString(cudaGetLastError()));
      return CKV_ERR_CUDA;
    }
  }
  if (p.max_splits > 1) {
    a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kSchedBytes);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + int64_t(p.blocks) * a.Hk * p.max_splits * NQ * BM * HD);
  }
  a.tps = p.tps, a.max_splits = p.max_splits, a.blocks = p.blocks;
  launch_pdl(kern, dim3(int(std::min<int64_t>(n_slots, num_sms()))), dim3(kThreads), Cfg<HD>::SMEM, stream, a);
  CKV_LAUNCH_CHECK("ckv_attention_kv8");
  if (p.max_splits > 1) {
    launch_combine<HD>(p.blocks, a.positions, a.out, a.M, a.Hq, a.Hk, a.n_ctx, p.tps, p.max_splits, a.part_o, a.part_ml, stream);
    CKV_LAUNCH_CHECK("ckv_attention_kv8(combine)");
  }
  return CKV_OK;
}

bool shape_ok(int m, int Hq, int Hk, int HD, int n_ctx) {
  return m > 0 && Hk > 0 && Hk <= 65535 && Hq > 0 && Hq % Hk == 0 && Hq / Hk <= 128 && (HD == 64 || HD == 128) && n_ctx > 0 &&
         n_ctx <= (1 << 30) && int64_t(m) * Hq <= (int64_t(1) << 31) - (1 << 20);  // row numbers stay within 32 bits
}

}  // namespace
}  // namespace ckv

using namespace ckv;

extern "C" int64_t ckv_attention_kv8_workspace_size(int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx) {
  if (!shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) return 0;
  return use_tiles(m, n_q_heads, n_kv_heads, head_dim, n_ctx) ? kSchedBytes + tile_plan(m, n_q_heads, n_kv_heads, head_dim, n_ctx).bytes
                                             : kv8_stream_workspace(m, n_q_heads, n_kv_heads, head_dim, n_ctx);
}

extern "C" int ckv_attention_kv8_launches(int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx) {
  if (!shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) return 0;
  if (use_tiles(m, n_q_heads, n_kv_heads, head_dim, n_ctx))
    return tile_plan(m, n_q_heads, n_kv_heads, head_dim, n_ctx).max_splits > 1 ? 2 : 1;
  return kv8_stream_launches(m, n_q_heads, n_kv_heads, head_dim, n_ctx);
}

extern "C" int ckv_attention_kv8_splits(int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx) {
  if (!shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx) || !use_tiles(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) return 0;
  return tile_plan(m, n_q_heads, n_kv_heads, head_dim, n_ctx).max_splits;
}

extern "C" int ckv_attention_kv8(const uint16_t* q, const uint8_t* k8, const uint8_t* v8, const float* k_scale,
                                 const float* v_scale, const int32_t* positions, uint16_t* out, int m, int n_q_heads,
                                 int n_kv_heads, int head_dim, int n_ctx, float scale, int type, void* workspace,
                                 int64_t workspace_bytes, ckv_stream_t stream) {
  CKV_REQUIRE(type == CKV_KV8_INT8 || type == CKV_KV8_E4M3, "ckv_attention_kv8: type %d", type);
  CKV_REQUIRE(m >= 0 && n_kv_heads > 0 && n_q_heads > 0 && n_q_heads % n_kv_heads == 0 && n_ctx > 0,
              "ckv_attention_kv8: bad sizes (%d rows, %d query heads, %d KV heads, context %d)", m, n_q_heads, n_kv_heads, n_ctx);
  if (m == 0) return CKV_OK;
  if (!shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) {
    set_error("ckv_attention_kv8: head_dim %d (64 or 128), %d query heads per KV head (at most 128), context %d, %d rows", head_dim,
              n_q_heads / n_kv_heads, n_ctx, m);
    return CKV_ERR_UNSUPPORTED;
  }
  CKV_REQUIRE(scale >= 0.f && scale * 1.4426950408889634f <= 3.0e38f, "ckv_attention_kv8: scale %g (0 to 2e38)", double(scale));
  CKV_REQUIRE(q && k8 && v8 && k_scale && v_scale && positions && out, "ckv_attention_kv8: null pointer");
  CKV_REQUIRE(aligned16(q) && aligned16(k8) && aligned16(v8) && aligned16(out),
              "ckv_attention_kv8: tensors must be 16-byte aligned");
  const int64_t need = ckv_attention_kv8_workspace_size(m, n_q_heads, n_kv_heads, head_dim, n_ctx);
  CKV_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "ckv_attention_kv8: workspace of %lld bytes, needs %lld (16-byte aligned)", static_cast<long long>(workspace_bytes),
              static_cast<long long>(need));
  if (!use_tiles(m, n_q_heads, n_kv_heads, head_dim, n_ctx))
    return kv8_stream_attention(q, k8, v8, k_scale, v_scale, positions, out, m, n_q_heads, n_kv_heads, head_dim, n_ctx, scale, type,
                                workspace, as_stream(stream));
  const Args a{q, k8, v8, k_scale, v_scale, positions, out, nullptr, nullptr, nullptr, m, n_q_heads, n_kv_heads, n_ctx,
               ceil_div(n_ctx, kBlk), 0, 0, 0, scale * 1.4426950408889634f};
  const SplitPlan p = tile_plan(m, n_q_heads, n_kv_heads, head_dim, n_ctx);
  const cudaStream_t s = as_stream(stream);
  if (head_dim == 128)
    return type == CKV_KV8_E4M3 ? launch_tiles<128, true>(a, p, workspace, s) : launch_tiles<128, false>(a, p, workspace, s);
  return type == CKV_KV8_E4M3 ? launch_tiles<64, true>(a, p, workspace, s) : launch_tiles<64, false>(a, p, workspace, s);
}
