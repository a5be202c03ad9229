// fqkv_kv4_api.cu -- the extern "C" boundary of the paged 4-bit key/value cache
// (include/fused_rmsnorm_qkv.h).  Arguments are checked before any CUDA call; nothing is
// allocated or synchronised.
#include <cmath>
#include <cstdint>

#include "fqkv_kv4.cuh"

using namespace fqkv;

namespace {

// More query rows (heads that share a KV head, times queries) than this go to the prompt kernel:
// 16 requests of 500 to 6000 tokens, 8 KV heads: split 44, 62, 74, 87, 101 us at 16, 24, 32, 40, 48
// rows, prompt 85 us at any; one request of 4000 tokens, 24 rows: 21 against 34 us.
constexpr int64_t kPromptRows = 32;
constexpr float kLog2e = 1.4426950408889634f;

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

bool supported(int64_t D, int64_t group) {
  return (D == 64 || D == 128) && (group == 32 || group == 64 || group == 128) && group <= D;
}

int check_cache(const fqkv_kv4_cache* c, Kv4Cache* out) {
  if (!c || !c->data) return api_fail(FQKV_ERR_NULL, "the cache and its data must not be NULL");
  if (c->dtype != FQKV_F16 && c->dtype != FQKV_BF16)
    return api_fail(FQKV_ERR_DTYPE, "the cache's dtype must be FQKV_F16 or FQKV_BF16");
  if (!supported(c->head_dim, c->group_size))
    return api_fail(FQKV_ERR_SHAPE, "head_dim must be 64 or 128 and group_size 32, 64 or 128, at most head_dim");
  if (c->block_size <= 0 || c->block_size % kKv4Rec != 0)
    return api_fail(FQKV_ERR_SHAPE, "block_size must be a positive multiple of 16");
  if (c->n_blocks <= 0 || c->n_kv_heads <= 0 || c->n_kv_heads > 32767 ||
      c->n_blocks > INT32_MAX / (int64_t)c->block_size)
    return api_fail(FQKV_ERR_SHAPE, "n_blocks and n_kv_heads must be positive, slots below 2^31, heads below 2^15");
  if (!aligned(c->data, 128)) return api_fail(FQKV_ERR_ALIGN, "the cache must be 128-byte aligned");
  *out = Kv4Cache{static_cast<uint8_t*>(c->data), c->n_blocks, c->n_kv_heads, c->head_dim, c->block_size,
                  c->group_size};
  return 0;
}

int check_flags(int64_t flags, int64_t also = 0) {
  return flags & ~(FQKV_FLAG_PDL | also)
             ? api_fail(FQKV_ERR_SCHEDULE, "the cache's calls take FQKV_FLAG_PDL (attention: FQKV_FLAG_TEST_WITHHOLD)")
             : 0;
}

int done(cudaError_t e, const char* what) { return e == cudaSuccess ? 0 : api_cuda_fail(e, what); }

// n int32 words at p.  The plan's blocks of threads read lengths, free list and count while others
// write outputs and table entries, so none of what is written may overlap anything else.
struct Words {
  const int32_t* p;
  int64_t n;
};

bool overlap(const Words& a, const Words& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  return a.n > 0 && b.n > 0 && x < y + 4 * (uintptr_t)b.n && y < x + 4 * (uintptr_t)a.n;
}

// Whether `a` meets the first `width` words of one of `rows` rows, `stride` words apart.
bool overlap_rows(const Words& a, const int32_t* rows_at, int64_t rows, int64_t stride, int64_t width) {
  if (width <= 0 || !overlap(a, Words{rows_at, (rows - 1) * stride + width})) return false;
  const int64_t x = reinterpret_cast<intptr_t>(a.p) - reinterpret_cast<intptr_t>(rows_at);
  if (x < 0 || x % (4 * stride) < 4 * width) return true;
  return x / (4 * stride) + 1 < rows && x + 4 * a.n > (x / (4 * stride) + 1) * 4 * stride;
}

bool for_prompts(int64_t G, int64_t max_query_len) { return max_query_len > kPromptRows / G; }

}  // namespace

extern "C" FQKV_API int64_t fqkv_kv4_record_bytes(int64_t head_dim, int64_t group_size) {
  return supported(head_dim, group_size) ? kv4_record_bytes((int)head_dim, (int)(head_dim / group_size)) : 0;
}

extern "C" FQKV_API int fqkv_kv4_plan(const int32_t* context_lens, const int32_t* new_lens, int64_t n_requests,
                                      int32_t* block_tables, int64_t table_stride, int64_t table_width,
                                      const int32_t* free_blocks, int64_t free_capacity, const int32_t* n_free,
                                      int64_t block_size, int64_t n_tokens, int32_t* query_start, int32_t* positions,
                                      int32_t* slots, int32_t* seq_lens, int32_t* n_free_out, int32_t* refused,
                                      int64_t flags, void* stream) {
  if (!context_lens || !new_lens || !block_tables || !n_free || !query_start || !seq_lens || !n_free_out || !refused ||
      (free_capacity > 0 && !free_blocks) || (n_tokens > 0 && (!positions || !slots)))
    return api_fail(FQKV_ERR_NULL, "a required pointer is NULL");
  if (n_requests <= 0 || n_requests > INT32_MAX || n_tokens < 0 || n_tokens > INT32_MAX || free_capacity < 0)
    return api_fail(FQKV_ERR_SHAPE, "n_requests must be positive, n_tokens and free_capacity not negative, below 2^31");
  if (block_size <= 0 || block_size > INT32_MAX || block_size % kKv4Rec != 0)
    return api_fail(FQKV_ERR_SHAPE, "block_size must be a positive multiple of 16");
  if (table_width < 0 || table_width > INT32_MAX || table_stride < table_width)
    return api_fail(FQKV_ERR_SHAPE, "table_stride must be at least table_width, which is not negative");
  const Words words[] = {{query_start, n_requests + 1}, {positions, n_tokens},     {slots, n_tokens},
                         {seq_lens, n_requests},        {n_free_out, 1},           {refused, 1},  // six written
                         {context_lens, n_requests},    {new_lens, n_requests},    {free_blocks, free_capacity},
                         {n_free, 1}};
  for (int i = 0; i < 10; ++i) {
    if (overlap_rows(words[i], block_tables, n_requests, table_stride, table_width))
      return api_fail(FQKV_ERR_ALIAS, "block_tables, which the plan writes, overlaps another argument");
    for (int j = i < 6 ? i + 1 : 10; j < 10; ++j)
      if (overlap(words[i], words[j]))
        return api_fail(FQKV_ERR_ALIAS, "an output of the plan overlaps an input or another output: every CTA reads "
                                        "all lengths, the free list and n_free");
  }
  if (int rc = check_flags(flags)) return rc;
  int sms = 0;
  if (int rc = api_sm100(&sms)) return rc;
  const Kv4PlanParams p{context_lens, new_lens, n_requests, block_tables, table_stride, table_width, free_blocks,
                        free_capacity, n_free, (int)block_size, n_tokens, query_start, positions, slots, seq_lens,
                        n_free_out, refused};
  return done(launch_kv4_plan(p, flags & FQKV_FLAG_PDL, static_cast<cudaStream_t>(stream)), "plan launch");
}

extern "C" FQKV_API int fqkv_kv4_append(const fqkv_kv4_cache* cache, const void* k, const void* v, int64_t n_batch,
                                        int64_t n_seq, int64_t k_stride_b, int64_t k_stride_s, int64_t k_stride_h,
                                        int64_t v_stride_b, int64_t v_stride_s, int64_t v_stride_h,
                                        const int32_t* slots, int64_t flags, void* stream) {
  Kv4Cache c;
  if (int rc = check_cache(cache, &c)) return rc;
  if (!k || !v || !slots) return api_fail(FQKV_ERR_NULL, "k, v and slots must not be NULL");
  if (n_batch <= 0 || n_seq <= 0 || n_batch > INT32_MAX / n_seq)
    return api_fail(FQKV_ERR_SHAPE, "n_batch and n_seq must be positive and their product below 2^31");
  if (!aligned(k, 16) || !aligned(v, 16) ||
      ((k_stride_b | k_stride_s | k_stride_h | v_stride_b | v_stride_s | v_stride_h) & 7))
    return api_fail(FQKV_ERR_ALIGN, "k and v rows must be 16-byte aligned (strides multiples of 8 elements)");
  if (int rc = check_flags(flags)) return rc;
  int sms = 0;
  if (int rc = api_sm100(&sms)) return rc;
  const Kv4AppendParams p{c, static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), k_stride_b, k_stride_s,
                          k_stride_h, v_stride_b, v_stride_s, v_stride_h, n_batch * n_seq, n_seq, slots};
  return done(launch_kv4_append(p, cache->dtype == FQKV_BF16, flags & FQKV_FLAG_PDL, static_cast<cudaStream_t>(stream)),
              "append launch");
}

extern "C" FQKV_API int fqkv_kv4_gather(const fqkv_kv4_cache* cache, const int32_t* slots, int64_t n_tokens, void* k,
                                        void* v, int64_t flags, void* stream) {
  Kv4Cache c;
  if (int rc = check_cache(cache, &c)) return rc;
  if (!k || !v || !slots) return api_fail(FQKV_ERR_NULL, "k, v and slots must not be NULL");
  if (n_tokens <= 0 || n_tokens > INT32_MAX) return api_fail(FQKV_ERR_SHAPE, "n_tokens must be positive, below 2^31");
  if (!aligned(k, 16) || !aligned(v, 16)) return api_fail(FQKV_ERR_ALIGN, "k and v must be 16-byte aligned");
  if (int rc = check_flags(flags)) return rc;
  int sms = 0;
  if (int rc = api_sm100(&sms)) return rc;
  const Kv4GatherParams p{c, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v), n_tokens, slots};
  return done(launch_kv4_gather(p, cache->dtype == FQKV_BF16, flags & FQKV_FLAG_PDL, static_cast<cudaStream_t>(stream)),
              "gather launch");
}

extern "C" FQKV_API int64_t fqkv_kv4_workspace_bytes(int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                                                     int64_t max_query_len) {
  if (n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads || (head_dim != 64 && head_dim != 128) ||
      max_query_len < 0)
    return -FQKV_ERR_SHAPE;
  const int D = (int)head_dim;
  return kKv4CounterBytes + (for_prompts(n_q_heads / n_kv_heads, max_query_len) ? kv4_prompt_partial_bytes(D)
                                                                              : kv4_split_partial_bytes(D));
}

extern "C" FQKV_API int fqkv_kv4_attention(const fqkv_kv4_cache* cache, const void* q, int64_t q_stride_r,
                                           int64_t q_stride_t, int64_t q_stride_h, int64_t n_q_heads,
                                           const int32_t* query_start, int64_t n_tokens, int64_t n_seq,
                                           int64_t n_requests, int64_t max_query_len, const int32_t* block_tables,
                                           int64_t table_stride, int64_t table_width, const int32_t* seq_lens,
                                           int64_t window, float scale, void* out, int64_t out_stride_t,
                                           void* workspace, int64_t workspace_bytes, int64_t flags, void* stream) {
  Kv4Cache c;
  if (int rc = check_cache(cache, &c)) return rc;
  if (!q || !out || !block_tables || !seq_lens) return api_fail(FQKV_ERR_NULL, "a required pointer is NULL");
  if (n_tokens <= 0 || n_requests <= 0 || n_tokens > INT32_MAX || n_requests > INT32_MAX ||
      (!query_start && (n_seq <= 0 || n_seq != n_tokens / n_requests || n_tokens % n_requests)))
    return api_fail(FQKV_ERR_SHAPE, "n_tokens and n_requests must be positive, with n_tokens = n_requests * n_seq "
                                    "where query_start is NULL");
  if (n_q_heads <= 0 || n_q_heads % c.n_kv || n_q_heads > 65535 || n_tokens > INT32_MAX / n_q_heads)
    return api_fail(FQKV_ERR_SHAPE, "n_q_heads must be a positive multiple of n_kv_heads, tokens * heads below 2^31");
  if (max_query_len < 0 || window < 0 || window > INT32_MAX || table_width < 0 || table_stride < table_width ||
      table_width > INT32_MAX / c.P)
    return api_fail(FQKV_ERR_SHAPE, "max_query_len and window must not be negative, table_stride at least table_width, "
                                    "and a table's tokens below 2^31");
  if (!(fabsf(scale) > 0.0f && fabsf(scale) <= 1e30f))
    return api_fail(FQKV_ERR_SHAPE, "scale must be finite and not zero");
  if (out_stride_t < n_q_heads * c.D) return api_fail(FQKV_ERR_SHAPE, "out_stride_t is smaller than a token's row");
  if (!aligned(q, 16) || ((q_stride_r | q_stride_t | q_stride_h) & 7) || !aligned(out, 16) || (out_stride_t & 7))
    return api_fail(FQKV_ERR_ALIGN, "q and out rows must be 16-byte aligned (strides multiples of 8 elements)");
  if (q_stride_r < 0 || q_stride_t < 0 || q_stride_h < 0)
    return api_fail(FQKV_ERR_SHAPE, "q's strides must not be negative");
  const uintptr_t q0 = reinterpret_cast<uintptr_t>(q), o0 = reinterpret_cast<uintptr_t>(out);
  const uintptr_t q_bytes = 2 * (uintptr_t)((query_start ? (n_tokens - 1) * q_stride_t
                                                         : (n_requests - 1) * q_stride_r + (n_seq - 1) * q_stride_t) +
                                            (n_q_heads - 1) * q_stride_h + c.D);
  const uintptr_t o_bytes = 2 * (uintptr_t)((n_tokens - 1) * out_stride_t + n_q_heads * c.D);
  if (q0 < o0 + o_bytes && o0 < q0 + q_bytes) return api_fail(FQKV_ERR_ALIAS, "out overlaps q");
  const int64_t need = fqkv_kv4_workspace_bytes(n_q_heads, c.n_kv, c.D, max_query_len);
  if (!workspace || workspace_bytes < need) return api_fail(FQKV_ERR_WORKSPACE, "workspace missing or too small");
  if (!aligned(workspace, 256)) return api_fail(FQKV_ERR_ALIGN, "the workspace must be 256-byte aligned");
  if (int rc = check_flags(flags, FQKV_FLAG_TEST_WITHHOLD)) return rc;
  int sms = 0;
  if (int rc = api_sm100(&sms)) return rc;
  Kv4AttnParams p{};
  p.c = c;
  p.q = static_cast<const uint16_t*>(q);
  p.q_r = q_stride_r, p.q_t = q_stride_t, p.q_h = q_stride_h;
  p.query_start = query_start;
  p.T = n_tokens, p.S = n_seq;
  p.R = (int)n_requests, p.n_q = (int)n_q_heads, p.G = (int)(n_q_heads / c.n_kv);
  p.table = block_tables, p.table_stride = table_stride, p.width = (int)table_width;
  p.seq_lens = seq_lens;
  p.window = (int)window;
  p.scale_log2 = scale * kLog2e;
  p.out = static_cast<uint16_t*>(out), p.o_t = out_stride_t;
  p.counters = static_cast<int*>(workspace);
  p.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + kKv4CounterBytes);
  p.withhold = (flags & FQKV_FLAG_TEST_WITHHOLD) != 0;
  const bool pdl = flags & FQKV_FLAG_PDL, bf16 = cache->dtype == FQKV_BF16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return done(for_prompts(p.G, max_query_len) ? launch_kv4_attn_prompt(p, sms, bf16, pdl, st)
                                              : launch_kv4_attn_split(p, sms, bf16, pdl, st),
              "attention launch");
}
