// Attention over the 8-bit cache.
#include "ckv_common.cuh"

namespace ckv {
// attention_blocks.cu
int64_t kv8_stream_workspace(int m, int Hq, int Hk, int HD, int n_ctx);
int kv8_stream_launches(int m, int Hq, int Hk, int HD, int n_ctx);
int kv8_stream_attention(const uint16_t* q, const uint8_t* k8, const uint8_t* v8, const float* ks, const float* vs,
                         const int32_t* positions, uint16_t* out, int m, int Hq, int Hk, int HD, int n_ctx, float scale, int type,
                         void* workspace, cudaStream_t stream);
namespace {

bool shape_ok(int m, int Hq, int Hk, int HD, int n_ctx) {
  return m > 0 && Hk > 0 && Hk <= 65535 && Hq > 0 && Hq % Hk == 0 && Hq / Hk <= 128 && (HD == 64 || HD == 128) && n_ctx > 0 &&
         n_ctx <= (1 << 30);
}

}  // namespace
}  // namespace ckv

using namespace ckv;

extern "C" int64_t ckv_attention_kv8_workspace_size(int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx) {
  if (!shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) return 0;
  return kv8_stream_workspace(m, n_q_heads, n_kv_heads, head_dim, n_ctx);
}

extern "C" int ckv_attention_kv8_launches(int m, int n_q_heads, int n_kv_heads, int head_dim, int n_ctx) {
  if (!shape_ok(m, n_q_heads, n_kv_heads, head_dim, n_ctx)) return 0;
  return kv8_stream_launches(m, n_q_heads, n_kv_heads, head_dim, n_ctx);
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
    set_error("ckv_attention_kv8: head_dim %d (64 or 128), %d query heads per KV head (at most 128), context %d", head_dim,
              n_q_heads / n_kv_heads, n_ctx);
    return CKV_ERR_UNSUPPORTED;
  }
  CKV_REQUIRE(k_scale && v_scale, "ckv_attention_kv8: null scales");
  const int64_t need = kv8_stream_workspace(m, n_q_heads, n_kv_heads, head_dim, n_ctx);
  CKV_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "ckv_attention_kv8: workspace of %lld bytes, needs %lld (16-byte aligned)", static_cast<long long>(workspace_bytes),
              static_cast<long long>(need));
  return kv8_stream_attention(q, k8, v8, k_scale, v_scale, positions, out, m, n_q_heads, n_kv_heads, head_dim, n_ctx, scale, type,
                              workspace, as_stream(stream));
}
