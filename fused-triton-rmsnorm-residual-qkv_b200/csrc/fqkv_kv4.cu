// fqkv_kv4.cu -- the bookkeeping and storage kernels of the paged 4-bit key/value cache:
// block tables and slots planned from request lengths, keys and values quantised into their
// slots, and slots read back as numbers.
#include "fqkv_kv4.cuh"

namespace fqkv {
namespace {

// ---------------------------------------------------------------------------
// Plan.
//
// Three prefix sums over the requests decide everything: tokens before a request, blocks
// needed before it, and whether it is granted.  Each CTA scans all lengths itself (8 bytes a
// request, from L2) in chunks of kPlanThreads requests and writes the tokens of its own range,
// so the kernel is one launch without a dependency between CTAs.  A token finds its request by
// binary search in the chunk's ends (shared memory).  A new block's table entry is written by
// the block's first token, so the table needs no pass of its own; entries that are read (blocks
// a request already has) and entries that are written are disjoint.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 512;
constexpr int kPlanTokens = 2048;  // tokens per CTA

// Inclusive scan over the block; *total receives the sum.  One 64-bit value per thread.
__device__ __forceinline__ long long block_scan(long long v, long long* s_warp, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(~0u, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();  // s_warp may still be read from the previous scan
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    const long long u = s_warp[w];
    if (w < warp) before += u;
    all += u;
  }
  *total = all;
  return v + before;
}

__global__ void __launch_bounds__(kPlanThreads) kv4_plan_kernel(const Kv4PlanParams p) {
  __shared__ long long s_warp[kPlanThreads / 32];
  __shared__ int s_end[kPlanThreads], s_start[kPlanThreads], s_ctx[kPlanThreads], s_have[kPlanThreads];
  __shared__ int s_before[kPlanThreads];  // blocks taken before this request, -1: not granted
  pdl_wait();
  pdl_launch_dependents();
  const long long t_lo = (long long)blockIdx.x * kPlanTokens;
  const long long t_hi = min(t_lo + kPlanTokens, (long long)p.T);
  const bool writer = blockIdx.x == 0;
  long long n_free = p.n_free[0];
  n_free = n_free < 0 ? 0 : n_free > p.free_capacity ? p.free_capacity : n_free;
  if (writer && threadIdx.x == 0) {
    if (n_free != p.n_free[0]) record_status(FQKV_STATUS_BAD_INDEX);
    p.query_start[0] = 0;
  }
  long long tokens = 0, blocks = 0, used = 0, refused = 0;
  for (int64_t r0 = 0; r0 < p.R; r0 += kPlanThreads) {
    const int64_t r = r0 + threadIdx.x;
    const bool have_r = r < p.R;
    const int raw_c = have_r ? p.ctx[r] : 0, raw_n = have_r ? p.add[r] : 0;
    const bool sane = raw_c >= 0 && raw_n >= 0;
    const long long c = raw_c < 0 ? 0 : raw_c, n = raw_n < 0 ? 0 : raw_n;
    long long total;
    const long long end = tokens + block_scan(n, s_warp, &total);
    tokens += total;
    const long long have = (c + p.P - 1) / p.P, want = (c + n + p.P - 1) / p.P;
    const bool fits = have_r && sane && want <= p.width && end <= p.T && c + n <= INT32_MAX;
    const long long need = fits ? want - have : 0;
    const long long upto = blocks + block_scan(need, s_warp, &total);
    blocks += total;
    const bool granted = fits && (need == 0 || upto <= n_free);
    // Granted needs are a prefix of the needs, so what comes before a granted request is taken.
    s_start[threadIdx.x] = (int)min(end - n, (long long)INT32_MAX);
    s_end[threadIdx.x] = (int)min(end, (long long)INT32_MAX);
    s_ctx[threadIdx.x] = (int)c;
    s_have[threadIdx.x] = (int)have;
    s_before[threadIdx.x] = granted ? (int)(upto - need) : -1;
    if (writer) {
      if (have_r) {
        p.query_start[r + 1] = (int)min(end, (long long)p.T);
        p.seq_lens[r] = granted ? (int)(c + n) : 0;
      }
      block_scan(granted ? need : 0, s_warp, &total);
      used += total;
      refused += __syncthreads_count(have_r && !granted);
    }
    __syncthreads();
    // This CTA's tokens among the chunk's.
    const int in_chunk = (int)min((long long)kPlanThreads, (long long)(p.R - r0));
    const long long lo = max(t_lo, (long long)s_start[0]), hi = min(t_hi, (long long)s_end[in_chunk - 1]);
    for (long long t = lo + threadIdx.x; t < hi; t += kPlanThreads) {
      int a = 0, b = in_chunk - 1;  // the first request whose end is past t
      while (a < b) {
        const int m = (a + b) >> 1;
        if (s_end[m] > t) b = m;
        else a = m + 1;
      }
      const int pos = s_ctx[a] + (int)(t - s_start[a]);
      const int before = s_before[a];
      int slot = -1;
      if (before >= 0) {
        const int nth = pos / p.P, in_block = pos - nth * p.P;
        int* entry = p.table + (r0 + a) * p.table_stride + nth;
        int block;
        if (nth < s_have[a]) {
          block = *entry;
        } else {
          block = p.free_blocks[n_free - 1 - (before + (nth - s_have[a]))];
          if (in_block == 0) *entry = block;
        }
        slot = block * p.P + in_block;
      }
      p.positions[t] = pos;
      p.slots[t] = slot;
    }
    __syncthreads();
  }
  for (long long t = max(t_lo, tokens) + threadIdx.x; t < t_hi; t += kPlanThreads) {
    p.positions[t] = 0;
    p.slots[t] = -1;
  }
  if (writer && threadIdx.x == 0) {
    p.n_free_out[0] = (int)(n_free - used);
    p.refused[0] = (int)refused;
  }
}

// ---------------------------------------------------------------------------
// Append and gather: one thread per 8 dims of a token's key or value head; the D / 8 lanes of
// a head row are neighbours in a warp, so a group's minimum and maximum are shuffles.
// ---------------------------------------------------------------------------
constexpr int kStoreThreads = 256;

template <typename T>
__device__ __forceinline__ bool non_finite(uint16_t b);
template <>
__device__ __forceinline__ bool non_finite<__nv_bfloat16>(uint16_t b) {
  return (b & 0x7F80u) == 0x7F80u;
}
template <>
__device__ __forceinline__ bool non_finite<__half>(uint16_t b) {
  return (b & 0x7C00u) == 0x7C00u;
}

// Record base of (slot, head), or null when the slot holds nothing.
__device__ __forceinline__ uint8_t* slot_record(const Kv4Cache& c, int slot, int head, int rec_bytes) {
  if (slot < 0) return nullptr;
  const int block = slot / c.P, at = slot - block * c.P;
  if (block >= c.n_blocks) {
    record_status(FQKV_STATUS_BAD_INDEX);
    return nullptr;
  }
  return c.data + (((int64_t)block * c.n_kv + head) * (c.P / kKv4Rec) + at / kKv4Rec) * rec_bytes;
}

// 16-bit word of the values (h, g, c, i, b): token t = 8 h + 2 c + b, dims 32 i + 4 g .. + 3.
template <int D>
__device__ __forceinline__ int value_word(int t, int i, int g) {
  const int h = t >> 3, c = (t >> 1) & 3, b = t & 1;
  return D == 128 ? ((h * 32 + g * 4 + c) * 4 + i) * 2 + b : ((g * 4 + c) * 4 + h * 2 + i) * 2 + b;
}

template <typename T, int D, int NG>
__global__ void __launch_bounds__(kStoreThreads) kv4_append_kernel(const Kv4AppendParams p) {
  constexpr int LPR = D / 8, LPG = LPR / NG, REC = kv4_record_bytes(D, NG);
  pdl_wait();
  pdl_launch_dependents();
  const int kind = (int)blockIdx.y / p.c.n_kv, head = (int)blockIdx.y % p.c.n_kv;
  const int64_t token = (int64_t)blockIdx.x * (kStoreThreads / LPR) + threadIdx.x / LPR;
  const int seg = threadIdx.x % LPR;
  const bool live = token < p.T;
  const int slot = live ? p.slots[token] : -1;
  uint16_t x[8] = {};
  if (slot >= 0) {
    const int64_t b = token / p.S, s = token - b * p.S;
    const uint16_t* src = kind == 0 ? p.k + b * p.k_b + s * p.k_s + head * p.k_h
                                    : p.v + b * p.v_b + s * p.v_s + head * p.v_h;
    *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(src + seg * 8);
  }
  float f[8], lo, hi;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = Elem<T>::to_f(x[e]);
    bad |= non_finite<T>(x[e]);
    lo = e ? fminf(lo, f[e]) : f[e];
    hi = e ? fmaxf(hi, f[e]) : f[e];
  }
#pragma unroll
  for (int o = 1; o < LPG; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
  }
  // The minimum is one of the 16-bit inputs, so it is stored exactly; the scale is rounded once,
  // and the codes are formed with the rounded scale that a reader multiplies them by.
  const uint16_t scale16 = Elem<T>::from_f(__fmul_rn(hi - lo, 1.0f / 15.0f));
  const float scale = Elem<T>::to_f(scale16);
  bad |= non_finite<T>(scale16);
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) bad |= __shfl_xor_sync(~0u, (int)bad, o) != 0;
  uint32_t code[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = rintf(__fdiv_rn(f[e] - lo, scale));
    code[e] = scale > 0.0f && !bad ? (uint32_t)fminf(fmaxf(v, 0.0f), 15.0f) : 0u;
  }
  const uint32_t param = bad ? 0x7FFF7FFFu  // NaN in both types
                             : (uint32_t)scale16 | ((uint32_t)Elem<T>::from_f(lo) << 16);
  uint8_t* rec = slot_record(p.c, slot, head, REC);
  const int t = slot & (kKv4Rec - 1);
  if (kind == 0) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w |= (code[2 * j] << (4 * j)) | (code[2 * j + 1] << (16 + 4 * j));
    if (rec) {
      const int i = seg >> 2, c = seg & 3;
      *reinterpret_cast<uint32_t*>(rec + t * (D / 2) + c * (D / 8) + i * 4) = w;
    }
  } else {
    uint32_t half[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      half[0] |= code[j] << (4 * j);
      half[1] |= code[4 + j] << (4 * j);
    }
    // Tokens 2 c and 2 c + 1 share 32-bit words.  When the next (previous) row of the warp is
    // the other token of the pair, each of the two lanes writes one whole word.
    const int other_slot = __shfl_xor_sync(~0u, slot, LPR);
    const uint32_t o0 = __shfl_xor_sync(~0u, half[0], LPR), o1 = __shfl_xor_sync(~0u, half[1], LPR);
    if (rec) {
      uint16_t* words = reinterpret_cast<uint16_t*>(rec + 8 * D);
      const int i = seg >> 2, g = 2 * (seg & 3);
      if (other_slot == (slot ^ 1)) {
        if (t & 1)
          *reinterpret_cast<uint32_t*>(words + value_word<D>(t ^ 1, i, g + 1)) = o1 | (half[1] << 16);
        else
          *reinterpret_cast<uint32_t*>(words + value_word<D>(t, i, g)) = half[0] | (o0 << 16);
      } else {
        words[value_word<D>(t, i, g)] = (uint16_t)half[0];
        words[value_word<D>(t, i, g + 1)] = (uint16_t)half[1];
      }
    }
  }
  if (rec && seg % LPG == 0)
    *reinterpret_cast<uint32_t*>(rec + 16 * D + kind * 64 * NG + (t * NG + seg / LPG) * 4) = param;
}

template <typename T, int D, int NG>
__global__ void __launch_bounds__(kStoreThreads) kv4_gather_kernel(const Kv4GatherParams p) {
  constexpr int LPR = D / 8, LPG = LPR / NG, REC = kv4_record_bytes(D, NG);
  pdl_wait();
  pdl_launch_dependents();
  const int kind = (int)blockIdx.y / p.c.n_kv, head = (int)blockIdx.y % p.c.n_kv;
  const int64_t token = (int64_t)blockIdx.x * (kStoreThreads / LPR) + threadIdx.x / LPR;
  const int seg = threadIdx.x % LPR;
  if (token >= p.T) return;
  const int slot = p.slots[token];
  const uint8_t* rec = slot_record(p.c, slot, head, REC);
  uint32_t o[4] = {0, 0, 0, 0};
  if (rec) {
    const int t = slot & (kKv4Rec - 1), i = seg >> 2, c = seg & 3;
    const uint32_t param =
        *reinterpret_cast<const uint32_t*>(rec + 16 * D + kind * 64 * NG + (t * NG + seg / LPG) * 4);
    const float scale = Elem<T>::to_f((uint16_t)param), low = Elem<T>::to_f((uint16_t)(param >> 16));
    uint32_t code[8];
    if (kind == 0) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + t * (D / 2) + c * (D / 8) + i * 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) code[e] = (w >> (4 * (e >> 1) + 16 * (e & 1))) & 15u;
    } else {
      const uint16_t* words = reinterpret_cast<const uint16_t*>(rec + 8 * D);
      const uint32_t a = words[value_word<D>(t, i, 2 * c)], b = words[value_word<D>(t, i, 2 * c + 1)];
#pragma unroll
      for (int e = 0; e < 8; ++e) code[e] = ((e < 4 ? a : b) >> (4 * (e & 3))) & 15u;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = Elem<T>::from_f2(__fmaf_rn((float)code[2 * e], scale, low), __fmaf_rn((float)code[2 * e + 1], scale, low));
  }
  uint16_t* dst = (kind == 0 ? p.k : p.v) + (token * p.c.n_kv + head) * D + seg * 8;
  *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
}

template <typename F>
cudaError_t by_layout(const Kv4Cache& c, bool bf16, F f) {
  const int ng = c.D / c.group;
#define FQKV_KV4_CASE(D_, NG_) \
  if (c.D == D_ && ng == NG_)  \
    return bf16 ? f.template operator()<__nv_bfloat16, D_, NG_>() : f.template operator()<__half, D_, NG_>();
  FQKV_KV4_CASE(128, 1)
  FQKV_KV4_CASE(128, 2)
  FQKV_KV4_CASE(128, 4)
  FQKV_KV4_CASE(64, 1)
  FQKV_KV4_CASE(64, 2)
#undef FQKV_KV4_CASE
  return cudaErrorInvalidValue;
}

struct AppendLaunch {
  const Kv4AppendParams& p;
  bool pdl;
  cudaStream_t stream;
  template <typename T, int D, int NG>
  cudaError_t operator()() const {
    const dim3 grid((unsigned)((p.T * (D / 8) + kStoreThreads - 1) / kStoreThreads), (unsigned)(2 * p.c.n_kv));
    return kv4_launch(kv4_append_kernel<T, D, NG>, grid, kStoreThreads, 0, pdl, stream, p);
  }
};

struct GatherLaunch {
  const Kv4GatherParams& p;
  bool pdl;
  cudaStream_t stream;
  template <typename T, int D, int NG>
  cudaError_t operator()() const {
    const dim3 grid((unsigned)((p.T * (D / 8) + kStoreThreads - 1) / kStoreThreads), (unsigned)(2 * p.c.n_kv));
    return kv4_launch(kv4_gather_kernel<T, D, NG>, grid, kStoreThreads, 0, pdl, stream, p);
  }
};

}  // namespace

cudaError_t launch_kv4_plan(const Kv4PlanParams& p, bool pdl, cudaStream_t stream) {
  const int64_t ctas = p.T > 0 ? (p.T + kPlanTokens - 1) / kPlanTokens : 1;
  return kv4_launch(kv4_plan_kernel, dim3((unsigned)ctas), kPlanThreads, 0, pdl, stream, p);
}

cudaError_t launch_kv4_append(const Kv4AppendParams& p, bool bf16, bool pdl, cudaStream_t stream) {
  return by_layout(p.c, bf16, AppendLaunch{p, pdl, stream});
}

cudaError_t launch_kv4_gather(const Kv4GatherParams& p, bool bf16, bool pdl, cudaStream_t stream) {
  return by_layout(p.c, bf16, GatherLaunch{p, pdl, stream});
}

}  // namespace fqkv
