// Argument checks of the paged cache (arthip_cache_write, arthip_paged_attention,
// arthip_key_weights, arthip_cache_evict). Host code only: a call that would read or
// write out of range ends here, before any launch; what lies on the device (pages,
// lengths, offsets) is checked or clamped by the kernels.
#include "paged.h"

#include <cmath>
#include <tuple>

namespace arthip {

namespace {

constexpr int kMaxTokens = 1 << 30;
constexpr int64_t kMaxSlotStride = 1 << 24;

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

std::string check_pages(const std::string& at, const arthip_pages& p) {
  if (p.dtype != ARTHIP_TYPE_F16 && p.dtype != ARTHIP_TYPE_BF16) return at + "type must be fp16 or bf16";
  if (p.batch < 0 || p.tokens < 0 || p.max_pages < 0 || p.pool_pages < 0) return at + "negative dimension";
  if (p.batch > 65536) return at + "more than 65536 sequences";
  if (p.k_heads < 1 || p.k_heads > 65536) return at + "k_heads must be from 1 to 65536";
  if (p.head_dim < 8 || p.head_dim > 256 || p.head_dim % 8 != 0)
    return at + "head_dim must be a multiple of 8 up to 256";
  if (p.page_size < 16 || p.page_size % 16 != 0 || p.page_size > 65536)
    return at + "page_size must be a multiple of 16 up to 65536";
  if (p.tokens > kMaxTokens || static_cast<int64_t>(p.max_pages) * p.page_size > kMaxTokens)
    return at + "too many tokens";
  if (p.batch == 0) return "";
  if (p.kv_len == nullptr) return at + "null lengths";
  if (p.pages == nullptr && p.max_pages > 0) return at + "null pages";
  if (p.q_offsets == nullptr && p.tokens != p.batch) return at + "without q_offsets each sequence has one token";
  if (!aligned(p.pages, 4) || !aligned(p.kv_len, 4) || !aligned(p.q_offsets, 4)) return at + "misaligned buffer";
  return "";
}

bool multiples(const int64_t* stride, int n) {
  for (int i = 0; i < n; ++i)
    if (stride[i] % 8 != 0) return false;
  return true;
}

std::string check_pool(const std::string& at, const arthip_pages& p, const void* pool, const int64_t* stride,
                       const char* name) {
  if (pool == nullptr && p.pool_pages > 0 && p.max_pages > 0) return at + "null " + name;
  if (!aligned(pool, 16)) return at + name + " must be aligned to 16 bytes";
  if (!multiples(stride, 3)) return at + name + ": strides must be multiples of 8 elements";
  // Kernels address a page, and a slot in it, by 32 bits each.
  if (stride[0] < 0 || stride[0] > kMaxTokens) return at + name + ": a page's stride must be from 0 to 2^30";
  if (stride[1] < 0 || stride[1] > kMaxSlotStride || stride[1] * p.page_size > kMaxTokens)
    return at + name + ": a slot's stride must be from 0 to 2^24, and a page's slots within 2^30";
  return "";
}

// A pool that is written: no two rows may be one.
std::string check_written(const std::string& at, const arthip_pages& p, const int64_t* stride, const char* name) {
  if ((p.pool_pages > 1 && stride[0] == 0) || stride[1] == 0 || (p.k_heads > 1 && stride[2] == 0))
    return at + name + " with a zero stride";
  return "";
}

// Queries, and the heads and scores of paged attention and the key weights.
std::string check_heads(const std::string& at, const arthip_pages& p, int q_heads, int left, int causal) {
  if (q_heads < 0 || q_heads % p.k_heads != 0) return at + "q_heads must be a multiple of k_heads";
  if (q_heads / p.k_heads > 128) return at + "more than 128 query heads a key head";
  if (static_cast<int64_t>(p.tokens) * (q_heads / p.k_heads) > kMaxTokens) return at + "too many tokens";
  if (left < -1 || left > kMaxTokens) return at + "window out of range";
  if (causal != 0 && causal != 1) return at + "causal is 0 or 1";
  return "";
}

std::string check_scores(const std::string& at, float scale, float cap) {
  if (!std::isfinite(scale)) return at + "scale is not finite";
  if (!std::isfinite(cap) || cap < 0) return at + "cap is negative or not finite";
  return "";
}

}  // namespace

std::string check_cache_write(const arthip_cache_write_args& a) {
  const std::string at = "arthip_cache_write: ";
  const arthip_pages& p = a.p;
  std::string wrong = check_pages(at, p);
  if (!wrong.empty()) return wrong;
  if (a.slots < 0 || a.slots > kMaxTokens) return at + "slots out of range";
  if (p.batch == 0 || p.tokens == 0) return "";
  if (a.k == nullptr || a.v == nullptr) return at + "null key or value buffer";
  if (!aligned(a.k, 16) || !aligned(a.v, 16)) return at + "k and v must be aligned to 16 bytes";
  if (!multiples(a.k_stride, 2) || !multiples(a.v_stride, 2)) return at + "strides must be multiples of 8 elements";
  for (const auto& [pool, stride, name] :
       {std::tuple{a.k_cache, a.k_cache_stride, "k_cache"}, std::tuple{a.v_cache, a.v_cache_stride, "v_cache"}}) {
    wrong = check_pool(at, p, pool, stride, name);
    if (wrong.empty()) wrong = check_written(at, p, stride, name);
    if (!wrong.empty()) return wrong;
  }
  if (a.k_cache == a.v_cache && a.k_cache != nullptr) return at + "k_cache and v_cache must not overlap";
  for (const void* x : {a.k, a.v})
    if (x == a.k_cache || x == a.v_cache) return at + "k and v must not overlap the cache";
  if ((a.positions == nullptr) != (a.token_positions == nullptr) && a.slots > 0)
    return at + "positions and token_positions come together";
  if (!aligned(a.positions, 4) || !aligned(a.token_positions, 4)) return at + "misaligned buffer";
  if (a.positions != nullptr && ((p.batch > 1 && a.positions_stride[0] == 0) ||
                                 (p.k_heads > 1 && a.positions_stride[1] == 0)))
    return at + "positions with a zero stride";
  return "";
}

std::string check_paged_attention_shape(const arthip_paged_attention_args& a) {
  const std::string at = "arthip_paged_attention: ";
  const std::string wrong = check_pages(at, a.p);
  return wrong.empty() ? check_heads(at, a.p, a.q_heads, a.left, a.causal) : wrong;
}

std::string check_paged_attention(const arthip_paged_attention_args& a) {
  const std::string at = "arthip_paged_attention: ";
  const arthip_pages& p = a.p;
  std::string wrong = check_paged_attention_shape(a);
  if (wrong.empty()) wrong = check_scores(at, a.scale, a.cap);
  if (!wrong.empty()) return wrong;
  if (p.batch == 0 || p.tokens == 0 || a.q_heads == 0) return "";
  if (a.q == nullptr || a.out == nullptr) return at + "null query or output buffer";
  if (!aligned(a.q, 16) || !aligned(a.out, 16)) return at + "q and out must be aligned to 16 bytes";
  if (!multiples(a.q_stride, 2) || !multiples(a.out_stride, 2)) return at + "strides must be multiples of 8 elements";
  if ((p.tokens > 1 && a.out_stride[0] == 0) || (a.q_heads > 1 && a.out_stride[1] == 0))
    return at + "output with a zero stride";
  if (!aligned(a.lse, 4)) return at + "misaligned buffer";
  wrong = check_pool(at, p, a.k_cache, a.k_cache_stride, "k_cache");
  if (wrong.empty()) wrong = check_pool(at, p, a.v_cache, a.v_cache_stride, "v_cache");
  if (!wrong.empty()) return wrong;
  if (a.out == a.q || a.out == a.k_cache || a.out == a.v_cache) return at + "output must not overlap an input";
  const size_t need = paged_plan(a).workspace();
  if (a.workspace == nullptr || a.workspace_bytes < need)
    return at + "workspace too small: " + std::to_string(need) + " bytes needed";
  if (!aligned(a.workspace, 16)) return at + "misaligned workspace";
  return "";
}

std::string check_key_weights_shape(const arthip_key_weights_args& a) {
  const std::string at = "arthip_key_weights: ";
  std::string wrong = check_pages(at, a.p);
  if (wrong.empty()) wrong = check_heads(at, a.p, a.q_heads, a.left, a.causal);
  if (!wrong.empty()) return wrong;
  if (a.q_heads == 0) return at + "no query heads";
  if (a.slots < 0 || a.slots > kMaxTokens) return at + "slots out of range";
  // A workgroup of 256 threads takes 256 slots of a head, and splits come only to few workgroups: 2^23 times
  // 128 slots keep a launch's threads, and the workspace's entries of a split, below 2^31.
  const int64_t items = (static_cast<int64_t>(a.slots) + 127) / 128;
  if (items > 0 && static_cast<int64_t>(a.p.batch) * a.p.k_heads > (int64_t{1} << 23) / items)
    return at + "batch times heads times slots too large";
  return "";
}

std::string check_key_weights(const arthip_key_weights_args& a) {
  const std::string at = "arthip_key_weights: ";
  const arthip_pages& p = a.p;
  std::string wrong = check_key_weights_shape(a);
  if (wrong.empty()) wrong = check_scores(at, a.scale, a.cap);
  if (!wrong.empty()) return wrong;
  if (!std::isfinite(a.decay)) return at + "decay is not finite";
  if (p.batch == 0 || a.slots == 0) return "";
  if (a.out == nullptr) return at + "null output";
  if (a.weights == nullptr && a.decay != 0) return at + "null weights";
  if (!aligned(a.out, 4) || !aligned(a.weights, 4) || !aligned(a.lse, 4)) return at + "misaligned buffer";
  if ((p.batch > 1 && a.out_stride[0] == 0) || (p.k_heads > 1 && a.out_stride[1] == 0))
    return at + "output with a zero stride";
  if (a.out == a.weights && ((p.batch > 1 && a.out_stride[0] != a.weights_stride[0]) ||
                             (p.k_heads > 1 && a.out_stride[1] != a.weights_stride[1])))
    return at + "in place needs the input's strides";
  if (a.out == a.lse) return at + "output must not overlap an input";
  if (p.tokens > 0) {
    if (a.q == nullptr || a.lse == nullptr) return at + "null queries or lse";
    if (!aligned(a.q, 16)) return at + "q must be aligned to 16 bytes";
    if (!multiples(a.q_stride, 2)) return at + "strides must be multiples of 8 elements";
    for (int i = 0; i < 2; ++i)
      if (a.q_stride[i] < 0 || a.q_stride[i] > kMaxTokens) return at + "strides of q must be from 0 to 2^30";
    // A tile's queries, 64 rows of (token, head), lie within 31 bits of bytes of its first; one stride of
    // each kind is room for a buffer's beginning before the rows.
    const int64_t group = a.q_heads / p.k_heads;
    if ((64 / group + 2) * a.q_stride[0] + group * a.q_stride[1] >= int64_t{1} << 30)
      return at + "queries too far apart";
    wrong = check_pool(at, p, a.k_cache, a.k_cache_stride, "k_cache");
    if (!wrong.empty()) return wrong;
    if (a.out == a.q || a.out == a.k_cache) return at + "output must not overlap an input";
  }
  const size_t need = key_weights_plan(a).workspace;
  if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need))
    return at + "workspace too small: " + std::to_string(need) + " bytes needed";
  if (need > 0 && !aligned(a.workspace, 16)) return at + "misaligned workspace";
  return "";
}

std::string check_cache_evict(const arthip_cache_evict_args& a) {
  const std::string at = "arthip_cache_evict: ";
  arthip_pages p = a.p;
  p.tokens = p.batch;  // not used here
  p.q_offsets = nullptr;
  std::string wrong = check_pages(at, p);
  if (!wrong.empty()) return wrong;
  if (a.slots < 0 || a.slots > kMaxTokens) return at + "slots out of range";
  if (a.keep < 1 || a.keep > kMaxTokens) return at + "keep must be positive";
  if (a.recent < 0 || a.first < 0 || static_cast<int64_t>(a.recent) + a.first > a.keep)
    return at + "recent and first must be positive and add up to keep at most";
  if (p.batch == 0) return "";
  if (static_cast<int64_t>(p.batch) * p.k_heads > int64_t{1} << 21) return at + "batch times heads too large";
  if (a.weights == nullptr && a.slots > 0) return at + "null weights";
  if (a.kept == nullptr) return at + "null kept";
  if (a.positions_out != nullptr && a.positions == nullptr && a.slots > 0) return at + "positions_out without positions";
  for (const void* x : {static_cast<const void*>(a.weights), static_cast<const void*>(a.positions),
                        static_cast<const void*>(a.new_len), static_cast<const void*>(a.weights_out),
                        static_cast<const void*>(a.positions_out), static_cast<const void*>(a.kept)})
    if (!aligned(x, 4)) return at + "misaligned buffer";
  for (const auto& [pool, stride, name] :
       {std::tuple{a.k_cache, a.k_cache_stride, "k_cache"}, std::tuple{a.v_cache, a.v_cache_stride, "v_cache"}}) {
    wrong = check_pool(at, p, pool, stride, name);
    if (wrong.empty()) wrong = check_written(at, p, stride, name);
    if (!wrong.empty()) return wrong;
  }
  if (a.k_cache == a.v_cache && a.k_cache != nullptr) return at + "k_cache and v_cache must not overlap";
  const void* in[] = {a.weights, a.positions, p.kv_len, p.pages, a.k_cache, a.v_cache};
  const void* out[] = {a.new_len, a.weights_out, a.positions_out, a.kept};
  for (const void* o : out)
    for (const void* i : in)
      if (o != nullptr && o == i) return at + "results must not overlap inputs";
  return "";
}

}  // namespace arthip
