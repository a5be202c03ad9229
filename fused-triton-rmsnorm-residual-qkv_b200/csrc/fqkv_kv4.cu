// fqkv_kv4.cu -- the bookkeeping and storage kernels of the paged 4-bit key/value cache:
// block tables and slots planned from request lengths, keys and values quantised into their
// slots, and slots read back as numbers.
#include "fqkv_kv4_work.cuh"

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
        // An id without a slot (negative, or past what 31 bits name) stores nothing.
        const long long at = (long long)block * p.P + in_block;
        if (at < 0 || at > INT32_MAX) record_status(FQKV_STATUS_BAD_INDEX);
        else slot = (int)at;
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
// Append and gather: a thread takes the part of a token's head that is contiguous in the cache,
// so that codes move in 16-byte pieces (8 at D = 64): for keys the dims 32 i + 8 c .. + 7 of lane
// c of four, for values 32 i + 4 g .. + 3 of lane g of eight, for all i.  The lanes of a token are
// neighbours, so a group's minimum and maximum are shuffles.  Bound by the 16-bit numbers' bytes.
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

// Byte offset among the values' codes of the NW words (i = 0 .. NW - 1) of token t's pair, lane g.
template <int D>
__device__ __forceinline__ int value_words(int t, int g) {
  const int h = t >> 3, c = (t >> 1) & 3;
  return D == 128 ? (h * 32 + g * 4 + c) * 16 : (g * 4 + c) * 16 + h * 8;
}

template <int N>
__device__ __forceinline__ void store_words(uint8_t* p, const uint32_t* w) {
  if constexpr (N == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (N == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(p) = w[0];
}

// Minimum and maximum of packed 16-bit pairs; a NaN stays.
template <typename T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (Kv4Nib<T>::kFullRange) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (Kv4Nib<T>::kFullRange) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// One token's keys (KIND 0) or values (1) of one head: N = 8 or 4 dims per i, LANES lanes a token.
template <typename T, int D, int NG, int KIND>
__device__ __forceinline__ void append_rows(const Kv4AppendParams& p, int head) {
  constexpr int NW = D / 32, N = KIND ? 4 : 8, LANES = 32 / N, REC = kv4_record_bytes(D, NG), WPG = NW / NG;
  const int64_t token = (int64_t)blockIdx.x * (kStoreThreads / LANES) + threadIdx.x / LANES;
  const int part = threadIdx.x % LANES;
  const bool live = token < p.T;
  const int slot = live ? p.slots[token] : -1;
  uint32_t x[NW][N / 2] = {};
  if (live) {  // the numbers do not wait for the slot
    const int64_t b = p.S == p.T ? 0 : token / p.S, s = token - b * p.S;
    const uint16_t* src = KIND ? p.v + b * p.v_b + s * p.v_s + head * p.v_h : p.k + b * p.k_b + s * p.k_s + head * p.k_h;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if constexpr (N == 8) *reinterpret_cast<uint4*>(x[i]) = *reinterpret_cast<const uint4*>(src + 32 * i + 8 * part);
      else *reinterpret_cast<uint2*>(x[i]) = *reinterpret_cast<const uint2*>(src + 32 * i + 4 * part);
    }
  }
  uint32_t param[NG];
  float low[NG], scale[NG];
  bool bad = false;
#pragma unroll
  for (int grp = 0; grp < NG; ++grp) {
    uint32_t lo = x[grp * WPG][0], hi = lo;
#pragma unroll
    for (int i = grp * WPG; i < (grp + 1) * WPG; ++i)
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        lo = min2<T>(lo, x[i][e]);
        hi = max2<T>(hi, x[i][e]);
      }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
      lo = min2<T>(lo, __shfl_xor_sync(~0u, lo, o));
      hi = max2<T>(hi, __shfl_xor_sync(~0u, hi, o));
    }
    lo = min2<T>(lo, __byte_perm(lo, lo, 0x1032));
    hi = max2<T>(hi, __byte_perm(hi, hi, 0x1032));
    // The minimum is one of the 16-bit inputs, so it is stored exactly; the scale is rounded once,
    // and the codes are formed with the rounded scale that a reader multiplies them by.
    low[grp] = Elem<T>::to_f((uint16_t)lo);
    // At the end of the type's range the rounded scale may take code 15 past the largest number; one
    // step lower does not, so that finite rows are read back finite by whoever rounds to 16 bits.
    uint16_t scale16 = Elem<T>::from_f(__fmul_rn(Elem<T>::to_f((uint16_t)hi) - low[grp], 1.0f / 15.0f));
    if (non_finite<T>(Elem<T>::from_f(__fmaf_rn(15.0f, Elem<T>::to_f(scale16), low[grp]))) && !non_finite<T>(scale16))
      --scale16;
    scale[grp] = Elem<T>::to_f(scale16);
    bad |= non_finite<T>((uint16_t)lo) || non_finite<T>((uint16_t)hi) || non_finite<T>(scale16);
    param[grp] = (uint32_t)scale16 | (lo << 16);
  }
  // (the groups' extremes, and so `bad`, are the same in all lanes of the token)
  // Codes clamp(rint(d / s), 0, 15), d = x - minimum >= 0, with the quotient correctly rounded
  // first.  d times an approximate reciprocal is off by less than 4e-6, so only a quotient that
  // close to a half is divided out (16-bit numbers meet halves often enough that a whole thread's
  // codes are not done again for one).  Adding 1.5 * 2^23 rounds and leaves the code in the low
  // bits.  N codes per word: pairs of dims (2 j, 2 j + 1) at bits (4 j, 16 + 4 j) for keys, dim j
  // at bits 4 j for values.
  uint32_t w[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const float s = scale[i / WPG], lo = low[i / WPG];
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    // (nothing passes where the reciprocal is not normal)
    const float tight = s > 1e-37f && s < 1e37f ? 0.49999f : -1.0f;
    w[i] = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = Elem<T>::to_f((uint16_t)(e & 1 ? x[i][e / 2] >> 16 : x[i][e / 2])) - lo;
      const float q = fminf(d * inv, 15.0f);
      float r = __fadd_rn(q, 12582912.0f);
      if (!(fabsf(q - __fadd_rn(r, -12582912.0f)) < tight)) r = __fadd_rn(fminf(__fdiv_rn(d, s), 15.0f), 12582912.0f);
      w[i] |= (__float_as_uint(r) & 15u) << (KIND ? 4 * e : 4 * (e >> 1) + 16 * (e & 1));
    }
    if (!(s > 0.0f)) w[i] = 0;
  }
  if (bad) {
#pragma unroll
    for (int i = 0; i < NW; ++i) w[i] = 0;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) param[grp] = 0x7FFF7FFFu;  // NaN in both types
  }
  uint8_t* rec = slot_record(p.c, slot, head, REC);
  const int t = slot & (kKv4Rec - 1);
  if constexpr (KIND == 0) {
    if (rec) store_words<NW>(rec + t * (D / 2) + part * (D / 8), w);
  } else {
    // Tokens 2 c and 2 c + 1 share 32-bit words.  When the token before or after this one in the
    // call is the other of the pair and in this warp, each of the two writes half of the words.
    const int from = ((int)(threadIdx.x & 31) + (t & 1 ? -LANES : LANES)) & 31;
    const bool near = t & 1 ? (int)(threadIdx.x & 31) >= LANES : (int)(threadIdx.x & 31) < 32 - LANES;
    const int other_slot = __shfl_sync(~0u, slot, from);
    uint32_t o[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) o[i] = __shfl_sync(~0u, w[i], from);
    // The other token pairs with this one only if it chose this lane as its partner too.
    if (rec) {
      uint8_t* at = rec + 8 * D + value_words<D>(t, part);
      if (near && slot >= 0 && other_slot == (slot ^ 1)) {
        uint32_t both[NW];
#pragma unroll
        for (int i = 0; i < NW; ++i) both[i] = t & 1 ? o[i] | (w[i] << 16) : w[i] | (o[i] << 16);
        if (t & 1) store_words<NW / 2>(at + 2 * NW, both + NW / 2);
        else store_words<NW / 2>(at, both);
      } else {
#pragma unroll
        for (int i = 0; i < NW; ++i) *reinterpret_cast<uint16_t*>(at + 4 * i + 2 * (t & 1)) = (uint16_t)w[i];
      }
    }
  }
  if (rec && part == 0) store_words<NG>(rec + 16 * D + KIND * 64 * NG + t * NG * 4, param);
}

template <typename T, int D, int NG>
__global__ void __launch_bounds__(kStoreThreads) kv4_append_kernel(const Kv4AppendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int head = (int)blockIdx.y >> 1;
  if (blockIdx.y & 1) append_rows<T, D, NG, 1>(p, head);
  else if ((int64_t)blockIdx.x * (kStoreThreads / 4) < p.T) append_rows<T, D, NG, 0>(p, head);
}

template <typename T, int D, int NG, int KIND>
__device__ __forceinline__ void gather_rows(const Kv4GatherParams& p, int head) {
  constexpr int NW = D / 32, N = KIND ? 4 : 8, LANES = 32 / N, REC = kv4_record_bytes(D, NG), WPG = NW / NG;
  const int64_t token = (int64_t)blockIdx.x * (kStoreThreads / LANES) + threadIdx.x / LANES;
  const int part = threadIdx.x % LANES;
  if (token >= p.T) return;
  const int slot = p.slots[token];
  const uint8_t* rec = slot_record(p.c, slot, head, REC);
  uint32_t w[NW] = {}, param[NG] = {};
  if (rec) {
    const int t = slot & (kKv4Rec - 1);
    const uint8_t* at = KIND ? rec + 8 * D + value_words<D>(t, part) : rec + t * (D / 2) + part * (D / 8);
    if constexpr (NW == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(at);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(at);
      w[0] = v.x, w[1] = v.y;
    }
    if constexpr (KIND == 1) {
#pragma unroll
      for (int i = 0; i < NW; ++i) w[i] = t & 1 ? w[i] >> 16 : w[i];
    }
    const uint32_t* q = reinterpret_cast<const uint32_t*>(rec + 16 * D + KIND * 64 * NG) + t * NG;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) param[grp] = q[grp];
  }
  uint16_t* dst = (KIND ? p.v : p.k) + (token * p.c.n_kv + head) * D + N * part;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const float scale = Elem<T>::to_f((uint16_t)param[i / WPG]), low = Elem<T>::to_f((uint16_t)(param[i / WPG] >> 16));
    uint32_t o[N / 2];
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      const uint32_t a = KIND ? (w[i] >> (8 * e)) & 15u : (w[i] >> (4 * e)) & 15u;
      const uint32_t b = KIND ? (w[i] >> (8 * e + 4)) & 15u : (w[i] >> (4 * e + 16)) & 15u;
      o[e] = Elem<T>::from_f2(__fmaf_rn((float)a, scale, low), __fmaf_rn((float)b, scale, low));
    }
    store_words<N / 2>(reinterpret_cast<uint8_t*>(dst + 32 * i), o);
  }
}

template <typename T, int D, int NG>
__global__ void __launch_bounds__(kStoreThreads) kv4_gather_kernel(const Kv4GatherParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int head = (int)blockIdx.y >> 1;
  if (blockIdx.y & 1) gather_rows<T, D, NG, 1>(p, head);
  else if ((int64_t)blockIdx.x * (kStoreThreads / 4) < p.T) gather_rows<T, D, NG, 0>(p, head);
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
    const dim3 grid((unsigned)((p.T + kStoreThreads / 8 - 1) / (kStoreThreads / 8)), (unsigned)(2 * p.c.n_kv));
    return kv4_launch(kv4_append_kernel<T, D, NG>, grid, kStoreThreads, 0, pdl, stream, p);
  }
};

struct GatherLaunch {
  const Kv4GatherParams& p;
  bool pdl;
  cudaStream_t stream;
  template <typename T, int D, int NG>
  cudaError_t operator()() const {
    const dim3 grid((unsigned)((p.T + kStoreThreads / 8 - 1) / (kStoreThreads / 8)), (unsigned)(2 * p.c.n_kv));
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
