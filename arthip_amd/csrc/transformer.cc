// Argument checks of the transformer operators (arthip_rope_axes, arthip_attention,
// arthip_gated_norm) and the packing of rotary frequencies. Host code only: a call
// that would read or write out of range ends here, before any launch.
#include "transformer.h"

#include <cmath>

namespace arthip {

namespace {

constexpr int kMaxTokens = 1 << 30;

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

size_t size_of(int type) { return type == ARTHIP_TYPE_F32 ? 4 : 2; }

// Strides of dimensions with one entry are never used.
bool multiples(const int64_t* stride, const int32_t* count, int n, int of) {
  for (int i = 0; i < n; ++i)
    if (count[i] > 1 && stride[i] % of != 0) return false;
  return true;
}

// An output whose stride along a dimension of more than one entry is 0 would be
// written by several workgroups.
bool distinct(const int64_t* stride, const int32_t* count, int n) {
  for (int i = 0; i < n; ++i)
    if (count[i] > 1 && stride[i] == 0) return false;
  return true;
}

bool same(const int64_t* a, const int64_t* b, const int32_t* count, int n) {
  for (int i = 0; i < n; ++i)
    if (count[i] > 1 && a[i] != b[i]) return false;
  return true;
}

}  // namespace

std::string check_rope(const arthip_rope_args& a) {
  const std::string at = "arthip_rope_axes: ";
  if (a.dtype < ARTHIP_TYPE_F16 || a.dtype > ARTHIP_TYPE_F32) return at + "unknown type";
  if (a.batch < 0 || a.tokens < 0 || a.q_heads < 0 || a.k_heads < 0)
    return at + "negative dimension";
  if (a.tokens > kMaxTokens || static_cast<int64_t>(a.batch) * a.tokens >= INT32_MAX)
    return at + "too many tokens";
  if (static_cast<int64_t>(a.q_heads) + a.k_heads > 65536) return at + "too many heads";
  if (a.head_dim < 2 || a.head_dim > 512 || a.head_dim % 2 != 0)
    return at + "head_dim must be even, from 2 to 512";
  if (a.n_freq < 1 || 2 * a.n_freq > a.head_dim) return at + "2 * n_freq must be from 2 to head_dim";
  if ((a.pairs & ~1) != 0 || (a.inverse & ~1) != 0) return at + "pairs and inverse are 0 or 1";
  if (a.batch == 0 || a.tokens == 0) return "";
  if (a.q_heads > 0 && (a.q == nullptr || a.q_out == nullptr)) return at + "null query buffer";
  if (a.k_heads > 0 && (a.k == nullptr || a.k_out == nullptr)) return at + "null key buffer";
  if (a.pos == nullptr || a.packed == nullptr) return at + "null positions or frequencies";
  const size_t sz = size_of(a.dtype);
  if ((a.q_heads > 0 && (!aligned(a.q, sz) || !aligned(a.q_out, sz))) ||
      (a.k_heads > 0 && (!aligned(a.k, sz) || !aligned(a.k_out, sz))) || !aligned(a.pos, 4) ||
      !aligned(a.packed, 16))
    return at + "misaligned buffer";
  const int32_t nq[3] = {a.batch, a.tokens, a.q_heads}, nk[3] = {a.batch, a.tokens, a.k_heads};
  if (a.q_heads > 0 && !distinct(a.q_out_stride, nq, 3)) return at + "query output with a zero stride";
  if (a.k_heads > 0 && !distinct(a.k_out_stride, nk, 3)) return at + "key output with a zero stride";
  if (a.q_heads > 0 && a.q == a.q_out && !same(a.q_stride, a.q_out_stride, nq, 3))
    return at + "in place needs the input's strides";
  if (a.k_heads > 0 && a.k == a.k_out && !same(a.k_stride, a.k_out_stride, nk, 3))
    return at + "in place needs the input's strides";
  return "";
}

std::string check_attention_shape(const arthip_attention_args& a) {
  const std::string at = "arthip_attention: ";
  if (a.batch < 0 || a.q_tokens < 0 || a.k_tokens < 0 || a.q_heads < 0)
    return at + "negative dimension";
  if (a.k_heads < 1 || a.q_heads % a.k_heads != 0)
    return at + "q_heads must be a multiple of k_heads";
  if (a.head_dim < 8 || a.head_dim > 256 || a.head_dim % 8 != 0)
    return at + "head_dim must be a multiple of 8 up to 256";
  if (a.q_tokens > kMaxTokens || a.k_tokens > kMaxTokens ||
      static_cast<int64_t>(a.q_tokens) * (a.q_heads / a.k_heads) > kMaxTokens)
    return at + "too many tokens";
  // Items of 32 rows and up to 64 ranges of keys number the workgroups in 31 bits. (A quotient,
  // as the product can pass 64 bits.)
  const int64_t items = (static_cast<int64_t>(a.q_tokens) * (a.q_heads / a.k_heads) + 31) / 32;
  if (items > 0 && static_cast<int64_t>(a.batch) * a.k_heads > (int64_t{1} << 24) / items)
    return at + "batch times heads times tokens too large";
  return "";
}

std::string check_attention(const arthip_attention_args& a) {
  const std::string at = "arthip_attention: ";
  if (a.dtype != ARTHIP_TYPE_F16 && a.dtype != ARTHIP_TYPE_BF16) return at + "type must be fp16 or bf16";
  const std::string shape = check_attention_shape(a);
  if (!shape.empty()) return shape;
  if (!std::isfinite(a.scale)) return at + "scale is not finite";
  if (!std::isfinite(a.cap) || a.cap < 0) return at + "cap is negative or not finite";
  if (a.left < -1 || a.right < -1 || a.left > kMaxTokens || a.right > kMaxTokens)
    return at + "window out of range";
  if (a.table != nullptr && a.table_len < 1) return at + "table without entries";
  if (a.table != nullptr && (a.table_zero < -kMaxTokens || a.table_zero > kMaxTokens))
    return at + "table_zero out of range";
  if (a.batch == 0 || a.q_tokens == 0 || a.q_heads == 0) return "";
  // Arrays over no tokens may be NULL: pairs are asked for where both sides have tokens.
  if (a.k_tokens > 0 && (a.doc_q == nullptr) != (a.doc_k == nullptr)) return at + "doc_q and doc_k come together";
  if (a.k_tokens > 0 && (a.code_q == nullptr) != (a.code_k == nullptr)) return at + "code_q and code_k come together";
  if (a.q == nullptr || a.out == nullptr) return at + "null query or output buffer";
  if (a.k_tokens > 0 && (a.k == nullptr || a.v == nullptr)) return at + "null key or value buffer";
  if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.out, 16))
    return at + "q, k, v and out must be aligned to 16 bytes";
  const int32_t n[3] = {a.batch, a.q_tokens, a.q_heads}, nk[3] = {a.batch, a.k_tokens, a.k_heads};
  if (!multiples(a.q_stride, n, 3, 8) || !multiples(a.k_stride, nk, 3, 8) ||
      !multiples(a.v_stride, nk, 3, 8) || !multiples(a.out_stride, n, 3, 8))
    return at + "strides must be multiples of 8 elements";
  for (const void* p : {static_cast<const void*>(a.lse), static_cast<const void*>(a.q_start),
                        static_cast<const void*>(a.kv_len), static_cast<const void*>(a.prefix),
                        static_cast<const void*>(a.doc_q), static_cast<const void*>(a.doc_k),
                        static_cast<const void*>(a.code_q), static_cast<const void*>(a.code_k),
                        static_cast<const void*>(a.slopes), static_cast<const void*>(a.table)})
    if (!aligned(p, 4)) return at + "misaligned buffer";
  if (!distinct(a.out_stride, n, 3)) return at + "output with a zero stride";
  if (a.out == a.q || a.out == a.k || a.out == a.v)
    return at + "output must not overlap an input";
  const size_t need = attention_plan(a).workspace;
  if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need))
    return at + "workspace too small: " + std::to_string(need) + " bytes needed";
  if (need > 0 && !aligned(a.workspace, 16)) return at + "misaligned workspace";
  return "";
}

std::string check_norm(const arthip_norm_args& a) {
  const std::string at = "arthip_gated_norm: ";
  if (a.dtype < ARTHIP_TYPE_F16 || a.dtype > ARTHIP_TYPE_F32) return at + "unknown type";
  if (a.residual_dtype != a.dtype && a.residual_dtype != ARTHIP_TYPE_F32)
    return at + "residual type must be the other type or fp32";
  if (a.post < ARTHIP_NORM_NONE || a.post > ARTHIP_NORM_LAYER || a.pre < ARTHIP_NORM_NONE ||
      a.pre > ARTHIP_NORM_LAYER)
    return at + "unknown norm";
  if (a.gate_act < ARTHIP_GATE_NONE || a.gate_act > ARTHIP_GATE_SILU)
    return at + "unknown gate activation";
  if (a.batch < 0 || a.tokens < 0) return at + "negative dimension";
  if (static_cast<int64_t>(a.batch) * a.tokens >= INT32_MAX) return at + "too many tokens";
  if (a.channels < 1 || a.channels > 32768) return at + "channels must be from 1 to 32768";
  if (!std::isfinite(a.eps) || a.eps < 0) return at + "eps is negative or not finite";
  if (!std::isfinite(a.residual_scale) || !std::isfinite(a.branch_scale))
    return at + "scale is not finite";
  if (a.batch == 0 || a.tokens == 0) return "";
  if (a.residual == nullptr) return at + "null residual";
  if (a.residual_out == nullptr && a.h == nullptr) return at + "no output";
  if (a.y == nullptr && (a.gate != nullptr || a.post != ARTHIP_NORM_NONE))
    return at + "gate or post norm without y";
  if (a.h == nullptr &&
      (a.pre != ARTHIP_NORM_NONE || a.mod_scale != nullptr || a.mod_shift != nullptr))
    return at + "pre norm or modulation without h";
  const size_t sz = size_of(a.dtype), rsz = size_of(a.residual_dtype);
  if (!aligned(a.residual, rsz) || !aligned(a.residual_out, rsz)) return at + "misaligned buffer";
  for (const void* p : {a.y, static_cast<const void*>(a.h), a.gate, a.mod_scale, a.mod_shift})
    if (!aligned(p, sz)) return at + "misaligned buffer";
  for (const float* p : {a.post_weight, a.post_bias, a.pre_weight, a.pre_bias})
    if (!aligned(p, 4)) return at + "misaligned buffer";
  const int32_t n[2] = {a.batch, a.tokens};
  if (a.residual_out != nullptr && !distinct(a.residual_out_stride, n, 2))
    return at + "residual output with a zero stride";
  if (a.h != nullptr && !distinct(a.h_stride, n, 2)) return at + "h with a zero stride";
  if (a.residual_out == a.residual && !same(a.residual_stride, a.residual_out_stride, n, 2))
    return at + "in place needs the input's strides";
  if (a.h != nullptr && (a.h == a.residual || a.h == a.y || a.h == a.residual_out))
    return at + "h must not overlap another tensor";
  if (a.residual_out != nullptr && a.residual_out == a.y)
    return at + "residual output must not overlap y";
  return "";
}

}  // namespace arthip
