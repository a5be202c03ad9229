// fqkv_kv4_prompt.cu -- causal attention over the paged 4-bit cache for many query rows per KV
// head (prompts and chunks of prompts), on tcgen05.
//
// Mathematics.  S = Q K^T and O = P V with the online softmax: P = exp2(c S - c ref), where c is
// the score scale times log2(e) and ref a row maximum that is only moved (and O and the row sum
// rescaled) when the true maximum exceeds it by 8 in the exponent; P stays below 2^8 (in bf16, whose
// values may be as large as fp32's, below 2^-16) and the quotient O / sum does not depend on ref.
// Keys and values are formed once per CTA as round16(scale * code + minimum), one rounding to the
// cache's type (the operand type of the product), which keeps the range of the numbers and adds at
// most an eighth to what the 4 bits lost (0.034 against 0.29 steps, root mean square, in bf16); P is
// rounded to the same type, row sums, maxima and accumulators are fp32.
//
// Shape.  A CTA takes 256 query rows of one KV head (all heads that share it, so the keys are
// unpacked once for them) as two tiles of 128 and walks the keys 128 at a time:
//   warps 0-3, 4-7   softmax of the two tiles, one row per thread, S and O in TMEM; P goes back
//                    to TMEM over S and is the A operand of the second product
//   warps 8-11       4-bit codes from global memory to swizzled shared-memory operands, and the
//                    queries of the next item while the current one ends
//   warp 12          issues the products
// TMEM holds two O tiles and two S tiles, so a step's 128 keys are taken as two halves: while a
// tile's warps exponentiate one half, the tensor core forms the scores of the other (and works for
// the other tile).  S of a half follows P V of the same half, in issue order, into the same columns.
// The values are stored transposed (dims x keys, K-major) because the cache interleaves tokens
// in pairs: a thread's eight tokens of one dim are one 16-byte store without any permutation.
//
// Bound: per 128 keys the products take 2048 tensor cycles at full rate (2560 in halves: the first
// product is then bound by the reads of its shared-memory operands), the softmax 32768 exponentials
// (2048 cycles of the special function unit) and the unpacking about 500 issue slots of every
// scheduler.  Measured (B200, bf16, 32 / 8 heads, a prompt of 4096 tokens): 191 us, 720 TFLOP/s of
// the causal half; a step takes about 4500 cycles, in which no unit is busy more than two thirds:
// the products of the four (tile, half) pairs, their softmax and the unpacking wait for each other.
// Beginning and ending an item costs about three steps.  A quarter of the exponentials as a
// polynomial on the FMA pipe changed nothing, and was left out.
#include "fqkv_kv4_work.cuh"

namespace fqkv {
namespace {

constexpr int kPThreads = 416;
constexpr int kPRows = 256;
constexpr int kPTile = 128;  // keys per step
constexpr int kPMinTiles = 4;

// What beginning and ending an item costs, in steps (measured on a prompt of 4096 tokens, whose
// CTAs have between 2 and 14 items: 291, 247, 220, 201 us with 0, 1, 2, 3).
constexpr int kPLead = 3;
// P is held this many powers of two lower in bf16: 2^16 products with the largest number fit O.
constexpr float kPLower = 24.0f;
using Work = Kv4Work<kPRows, kPTile, kPThreads, 1, kPLead>;

// D[tmem] (+)= A[tmem] * B[smem desc]^T, kind::f16.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Register lists of 8.
#define FQKV_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), \
                      "=r"(a[i + 6]), "=r"(a[i + 7])
#define FQKV_W8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), \
                      "r"(a[i + 6]), "r"(a[i + 7])

// 32 consecutive columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : FQKV_R8(r, 0), FQKV_R8(r, 8), FQKV_R8(r, 16), FQKV_R8(r, 24)
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      FQKV_W8(r, 0), FQKV_W8(r, 8)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ------------------------------------------------------------------ packed fp32 pairs
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack64(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float max3_nan(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// Scores of keys outside [lo, hi) of a chunk become -inf.
__device__ __forceinline__ void hide32(uint32_t* r, int lo, int hi) {
#pragma unroll
  for (int k = 0; k < 32; ++k)
    if (k < lo || k >= hi) r[k] = 0xFF800000u;
}
// P = exp2(c S - off) of 32 keys to 16 columns at `dst`, added to `sum` in fp32.
template <typename T>
__device__ __forceinline__ void exp32(const uint32_t* r, uint64_t c, uint64_t off, uint32_t dst, uint64_t (&sum)[2]) {
  uint32_t pk[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const uint64_t x = fma2(pack2(__uint_as_float(r[2 * k]), __uint_as_float(r[2 * k + 1])), c, off);
    float a, b;
    unpack64(x, a, b);
    a = kv4_exp2(a);
    b = kv4_exp2(b);
    sum[k & 1] = add2(sum[k & 1], pack2(a, b));
    pk[k] = Elem<T>::from_f2(a, b);
  }
  tmem_st16(dst, pk);
}

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void bulk_prefetch_l2(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}
// Asynchronous 16-byte copy global -> shared; zeros where `in` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
// One arrival for a warp whose lanes have all got here.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

struct Bars {
  uint64_t k_full[2], v_full[2];    // operands of a step written: one arrival per unpacking warp
  uint64_t k_empty[2], v_empty[2];  // and read by all products
  uint64_t q_full;                  // the queries of an item
  uint64_t s_full[2][2], p_full[2][2];  // [tile][half]: scores formed; probabilities written
  uint64_t o_done[2][2];                // [tile][half]: an item's last step added to O
  uint64_t drained;                     // every product that was issued has completed
};

// Whether a scale or a minimum (packed pair) is a NaN or an infinity.
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint32_t par) {
  constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
  return (par & e) == e || (par & (e << 16)) == e << 16;
}

template <int D>
constexpr int operand_bytes() {
  return 128 * D * 2;  // one operand tile: 128 x D or D x 128, 16-bit
}
template <int D>
constexpr int prompt_smem() {
  return 6 * operand_bytes<D>() + 1024;  // Q0, Q1, K x 2, V x 2; 1024-byte alignment
}
constexpr int slot_floats(int D) { return kPRows * (D + 2); }

template <typename T, int D, int NG>
__global__ void __launch_bounds__(kPThreads, 1) kv4_prompt_kernel(const Kv4AttnParams p) {
  constexpr int OP = operand_bytes<D>();
  constexpr int REC = kv4_record_bytes(D, NG);
  constexpr int NW = D / 32;
  constexpr bool kBf16 = Kv4Nib<T>::kFullRange;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ Work::Shared s_work;
  __shared__ uint32_t s_tmem;
  __shared__ int s_last;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0);

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.k_full[i], 4);
      mbar_init(&bars.v_full[i], 4);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_empty[i], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bars.s_full[i][h], 1);
        mbar_init(&bars.o_done[i][h], 1);
        mbar_init(&bars.p_full[i][h], 4);
      }
    }
    mbar_init(&bars.q_full, 4);
    mbar_init(&bars.drained, 1);
    fence_mbarrier_init_cluster();
  }
  pdl_wait();
  pdl_launch_dependents();
  Work w;
  if (!w.locate(p, s_work, gridDim.x, kPMinTiles)) return;
  if (warp == 8) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  if (warp < 8) {
    // ================================================================ softmax
    const int t = warp >> 2, row = tid & 127;  // tile, row of the tile = TMEM lane
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_tm = tmem + t * 128 + lane_base, o_tm = tmem + 256 + t * 128 + lane_base;  // S (P over it), O
    const float c = fabsf(p.scale_log2);
    const uint64_t c2 = pack2(c, c);
    uint32_t s_phase = 0, o_phase = 0;
    bool ok = true;  // after a wait that ran out nothing is waited for, and every barrier is still reached
    const auto wait = [&](uint64_t* bar, uint32_t phase) { ok = __all_sync(~0u, ok && mbar_wait(bar, phase & 1u)); };
    for (long long u = w.u0; u < w.u1;) {
      const long long ue = min(w.u1, w.item + w.n_tiles);
      int first, last;
      w.part_tiles(u, ue, first, last);
      const int rows = w.req.n * p.G - w.rb * kPRows;  // live rows of the block
      const int grow = w.rb * kPRows + t * 128 + row;  // row of the request
      const int j = (int)((uint32_t)grow / (uint32_t)p.G);
      const bool live = j < w.req.n;
      const bool tile_used = rows > t * 128;
      uint16_t* out = p.out + (int64_t)(w.req.start + j) * p.o_t + (int64_t)(w.kvh * p.G + grow - j * p.G) * D;
      float ref = -INFINITY, sum = 0.0f;
      if (tile_used) {
        const int pos = kv4_position(w.req, j);
        const int see_hi = live ? min(pos + 1, w.req.len) : w.req.len;      // keys [see_lo, see_hi)
        const int see_lo = live && p.window > 0 ? max(0, pos - p.window + 1) : 0;
        const bool warp_live = rows > t * 128 + (warp & 3) * 32;
        uint64_t sum2[2] = {0, 0};
        for (int tile = first; tile < last; ++tile) {
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            wait(&bars.s_full[t][half], s_phase);
            tc_fence_after();
            if (warp_live) {
              uint32_t s[64];
              const uint32_t at = s_tm + half * 64;
              tmem_ld32(at, s);
              tmem_ld32(at + 32, s + 32);
              tmem_wait_ld();
              const int key0 = tile * kPTile + half * 64, lo = see_lo - key0, hi = see_hi - key0;
              if (__any_sync(~0u, lo > 0 || hi < 64)) {
                hide32(s, lo, hi);
                hide32(s + 32, lo - 32, hi - 32);
              }
              float m[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) m[k] = max_nan(__uint_as_float(s[k]), __uint_as_float(s[k + 4]));
#pragma unroll
              for (int k = 8; k < 64; k += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  m[e] = max3_nan(m[e], __uint_as_float(s[k + e]), __uint_as_float(s[k + 4 + e]));
              const float top = max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3]));
              // ---- move the reference, and rescale O and the sum, when the maximum outgrew it
              if (__any_sync(~0u, top > ref && (top - ref) * c > 8.0f)) {
                const float to = fmaxf(top, ref);
                const float f = to == -INFINITY ? 1.0f : kv4_exp2((ref - to) * c);
                ref = to;
                sum2[0] = fma2(sum2[0], pack2(f, f), 0ull);
                sum2[1] = fma2(sum2[1], pack2(f, f), 0ull);
                if (tile > first || half) {
                  // The other half's product came before the scores that took that half's columns.
                  if (half && tile + 1 == last) wait(&bars.o_done[t][0], o_phase);
                  else wait(&bars.s_full[t][half ^ 1], half ? s_phase ^ 1u : s_phase);
                  tc_fence_after();
#pragma unroll 1
                  for (int k = 0; k < D / 16; ++k) {
                    uint32_t o[16];
                    tmem_ld16(o_tm + k * 16, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tmem_st16(o_tm + k * 16, o);
                  }
                  tmem_wait_st();
                }
              }
              // A NaN or an infinite score makes the whole row NaN.
              const float off = top != top || ref == INFINITY ? NAN
                                : ref == -INFINITY            ? 0.0f
                                                              : fmaf(-ref, c, kBf16 ? -kPLower : 0.0f);
              const uint64_t off2 = pack2(off, off);
              exp32<T>(s, c2, off2, at, sum2);  // P (16-bit pairs) over the half's first 32 columns
              exp32<T>(s + 32, c2, off2, at + 16, sum2);
              tmem_wait_st();
            }
            tc_fence_before();
            warp_arrive(&bars.p_full[t][half]);
          }
          s_phase ^= 1u;
        }
        float x, y;
        sum2[0] = add2(sum2[0], sum2[1]);
        unpack64(sum2[0], x, y);
        sum = x + y;
      }

      const bool nothing = first == last;  // the run ended before the item's keys
      const bool complete = u - w.item <= kPLead && ue == w.item + w.n_tiles;
      const int fc = complete ? 0 : w.first_cta(), lc = complete ? 0 : w.last_cta();
      const int side = w.u0 - w.item > kPLead ? 0 : 1;
      const bool more = ue < w.u1 && w.next(p);
      if (nothing) break;
      if (tile_used) {
        wait(&bars.o_done[t][0], o_phase);
        wait(&bars.o_done[t][1], o_phase);
        o_phase ^= 1u;
        tc_fence_after();
        if (!ok) sum = NAN;
      }
      if (complete) {
        if (tile_used) {
          const float inv = sum > 0.0f ? 1.0f / sum : sum;  // nothing seen: zeros; NaN stays
#pragma unroll 1
          for (int k = 0; k < D / 64; ++k) {
            uint32_t o[64];
            tmem_ld32(o_tm + k * 64, o);
            tmem_ld32(o_tm + k * 64 + 32, o + 32);
            tmem_wait_ld();
            if (live) {
#pragma unroll
              for (int e = 0; e < 64; e += 8) {
                uint4 v;
                v.x = Elem<T>::from_f2(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
                v.y = Elem<T>::from_f2(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
                v.z = Elem<T>::from_f2(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
                v.w = Elem<T>::from_f2(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
                *reinterpret_cast<uint4*>(out + k * 64 + e) = v;
              }
            }
          }
        }
      } else {
        // Part: reference and sum per row, then O as [dims / 4][rows] groups of four.
        const int me = (int)blockIdx.x, brow = t * 128 + row;
        float* part = p.partial + (int64_t)(2 * me + side) * slot_floats(D);
        if (tile_used) {
          part[brow] = ref;
          part[kPRows + brow] = sum;
#pragma unroll 1
          for (int k = 0; k < D / 64; ++k) {
            uint32_t o[64];
            tmem_ld32(o_tm + k * 64, o);
            tmem_ld32(o_tm + k * 64 + 32, o + 32);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 64; e += 4)
              *reinterpret_cast<uint4*>(part + 2 * kPRows + ((k * 16 + e / 4) * kPRows + brow) * 4) =
                  make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        __threadfence();
        named_bar_sync(1, 256);
        if (tid == 0) {
          const int arrived = atomicAdd(p.counters + fc, 1);
          s_last = arrived == lc - fc;
          if (s_last) p.counters[fc] = 0;
        }
        named_bar_sync(1, 256);
        if (s_last && tile_used) {
          __threadfence();
          const auto slot = [&](int x) { return p.partial + (int64_t)(2 * x + (x == fc ? 1 : 0)) * slot_floats(D); };
          // Four parts at a time, so that their loads are in flight together; two are the rule.
          float top = -INFINITY, l = 0.0f;
          for (int x0 = fc; x0 <= lc; x0 += 4) {
            float m[4], z[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const float* src = slot(min(x0 + y, lc)) + brow;
              m[y] = __ldcg(src);
              z[y] = x0 + y <= lc ? __ldcg(src + kPRows) : 0.0f;
            }
            const float to = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), top);
            const float at = to == -INFINITY ? 0.0f : to;
            l *= kv4_exp2((top - at) * c);
#pragma unroll
            for (int y = 0; y < 4; ++y) l = fmaf(z[y], kv4_exp2((m[y] - at) * c), l);
            top = to;
          }
          const float to = top == -INFINITY ? 0.0f : top;
          const float inv = l > 0.0f ? 1.0f / l : l;
          if (live) {
#pragma unroll 1
            for (int k = 0; k < D / 32; ++k) {
              float v[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = 0.0f;
#pragma unroll 2
              for (int x = fc; x <= lc; ++x) {
                const float f = kv4_exp2((__ldcg(slot(x) + brow) - to) * c);
                const float* src = slot(x) + 2 * kPRows + (k * 8 * kPRows + brow) * 4;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const float4 o = __ldcg(reinterpret_cast<const float4*>(src + e * kPRows * 4));
                  v[4 * e] += o.x * f, v[4 * e + 1] += o.y * f, v[4 * e + 2] += o.z * f, v[4 * e + 3] += o.w * f;
                }
              }
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                uint4 o;
                o.x = Elem<T>::from_f2(v[e] * inv, v[e + 1] * inv);
                o.y = Elem<T>::from_f2(v[e + 2] * inv, v[e + 3] * inv);
                o.z = Elem<T>::from_f2(v[e + 4] * inv, v[e + 5] * inv);
                o.w = Elem<T>::from_f2(v[e + 6] * inv, v[e + 7] * inv);
                *reinterpret_cast<uint4*>(out + k * 32 + e) = o;
              }
            }
          }
        }
        named_bar_sync(1, 256);  // s_last is written again by the next piece
      }
      tc_fence_before();
      u = ue;
      if (!more) break;
    }
  } else if (warp < 12) {
    // ================================================================ codes to operands
    const int dw = warp - 8, key = tid - 256;
    const int vr = (lane >> 1) & 1, vh = lane & 1, vg = lane >> 2;  // values: record, token half, dim group
    const int rpb = p.c.P / kKv4Rec;
    const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;  // a negative scale negates the keys
    const uint32_t magic = kv4_opaque(Kv4Nib<T>::kOffset2, p.n_q);
    uint32_t it = 0;
    bool ok = true;  // the same in all lanes, which meet at every tile
    const auto wait = [&](uint64_t* bar, uint32_t phase) { ok = __all_sync(~0u, ok && mbar_wait(bar, phase & 1u)); };
    uint32_t kc[4 * NW], kp[NG], vq[NG], vc[4 * NW], vp[8 * NG];
    for (long long u = w.u0; u < w.u1 && ok;) {
      const long long ue = min(w.u1, w.item + w.n_tiles);
      int first, last;
      w.part_tiles(u, ue, first, last);
      if (first == last) break;
      const int* table = p.table + (int64_t)w.r * p.table_stride;
      const int n_rec = (w.req.len + kKv4Rec - 1) / kKv4Rec;
      // This warp's two records of a tile: (nth, off) are the block's place in the table and the
      // record's in the block, stepped without a division.  Blocks are looked up one tile before
      // their codes are loaded, which is one tile before they are unpacked.
      const int step_n = 8 / rpb, step_o = 8 % rpb;
      int nth[2], off[2], ahead = first * 8 + 2 * dw, next[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        nth[k] = (int)((uint32_t)(ahead + k) / (uint32_t)rpb);
        off[k] = ahead + k - nth[k] * rpb;
        next[k] = ahead + k < n_rec ? __ldg(table + nth[k]) : -1;
      }
      const uint8_t *ra, *rb;
      const auto advance = [&]() {  // ra, rb: the records of the tile `ahead`; then the next tile's blocks
        const uint8_t* at[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          at[k] = nullptr;
          if (ahead + k < n_rec) {
            if (next[k] < 0 || next[k] >= p.c.n_blocks) {
              record_status(FQKV_STATUS_BAD_INDEX);
              next[k] = 0;
            }
            at[k] = p.c.data + (((int64_t)next[k] * p.c.n_kv + w.kvh) * rpb + off[k]) * REC;
          }
          nth[k] += step_n;
          off[k] += step_o;
          if (off[k] >= rpb) off[k] -= rpb, ++nth[k];
          next[k] = ahead + 8 + k < n_rec ? __ldg(table + nth[k]) : -1;
        }
        ra = at[0], rb = at[1];
        ahead += 8;
      };
      advance();
      // Codes and parameters of this thread's key; a key past the last one gets zeros.
      const auto load_k = [&](int tile) {
        const uint8_t* rec = lane < 16 ? ra : rb;
        const bool in = rec != nullptr && tile * kPTile + key < w.req.len;
#pragma unroll
        for (int k = 0; k < NW; ++k) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) v = __ldg(reinterpret_cast<const uint4*>(rec + (lane & 15) * (D / 2)) + k);
          kc[4 * k] = v.x, kc[4 * k + 1] = v.y, kc[4 * k + 2] = v.z, kc[4 * k + 3] = v.w;
        }
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          kp[k] = in ? __ldg(reinterpret_cast<const uint32_t*>(rec + 16 * D) + (lane & 15) * NG + k) : 0u;
          vq[k] = in ? __ldg(reinterpret_cast<const uint32_t*>(rec + 16 * D + 64 * NG) + (lane & 15) * NG + k) : 0u;
        }
      };
      // Codes of eight tokens (half vh of record vr) and 4 NW dims, and the tokens' parameters.
      const auto load_v = [&](int tile) {
        const uint8_t* rec = vr ? rb : ra;
        const bool in = rec != nullptr;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (D == 128) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (in) v = __ldg(reinterpret_cast<const uint4*>(rec + 8 * D + (vh * 8 + vg) * 64) + k);
            vc[4 * k] = v.x, vc[4 * k + 1] = v.y, vc[4 * k + 2] = v.z, vc[4 * k + 3] = v.w;
          } else {
            uint2 v = make_uint2(0, 0);
            if (in) v = __ldg(reinterpret_cast<const uint2*>(rec + 8 * D + vg * 64 + k * 16 + vh * 8));
            vc[2 * k] = v.x, vc[2 * k + 1] = v.y;
          }
        }
        const int t0 = tile * kPTile + (2 * dw + vr) * kKv4Rec + 8 * vh;
#pragma unroll
        for (int k = 0; k < 8 * NG; ++k)
          vp[k] = in && t0 + k / NG < w.req.len
                      ? __ldg(reinterpret_cast<const uint32_t*>(rec + 16 * D + 64 * NG) + 8 * NG * vh + k)
                      : 0u;
      };
      load_k(first);
      load_v(first);
      // The queries of the request's next row block to L2, a token's heads at a time.
      if (p.q_h == D && w.rb + 1 < w.blocks) {
        const int j0 = (int)((uint32_t)((w.rb + 1) * kPRows) / (uint32_t)p.G);
        const int j1 = min((int)((uint32_t)((w.rb + 2) * kPRows - 1) / (uint32_t)p.G), w.req.n - 1);
        const uint16_t* q0 = p.q + (p.query_start ? (int64_t)w.req.start * p.q_t : w.r * p.q_r) +
                             (int64_t)(w.kvh * p.G) * p.q_h;
        for (int j = j0 + key; j <= j1; j += 128) bulk_prefetch_l2(q0 + j * p.q_t, (uint32_t)(p.G * D * 2));
      }
      // The item's queries, once the previous item's last scores have been formed.
      const auto copy_q = [&]() {
        constexpr int CH = D / 8, STEP = 128 / CH;  // 16-byte chunks of a row; rows copied at a time
        if (it > 0) wait(&bars.k_empty[(it - 1) & 1], (it - 1) >> 1);
        const int ch = key % CH, dj = STEP / p.G, dh = STEP % p.G;
        int row = key / CH, j = (int)((uint32_t)(w.rb * kPRows + row) / (uint32_t)p.G);
        int h = w.rb * kPRows + row - j * p.G;
        const uint16_t* q0 = p.q + (p.query_start ? (int64_t)w.req.start * p.q_t : w.r * p.q_r) +
                             (int64_t)(w.kvh * p.G) * p.q_h + ch * 8;
#pragma unroll 4
        for (; row < kPRows; row += STEP) {
          const bool in = j < w.req.n;
          const uint16_t* src = in ? q0 + j * p.q_t + h * p.q_h : p.q;
          copy16(smem_u32(smem) + (row / 128) * OP + (ch / 8) * 128 * 128 + sw128_offset(row % 128, ch % 8), src, in);
          j += dj;
          h += dh;
          if (h >= p.G) h -= p.G, ++j;
        }
      };
      for (int tile = first; tile < last && ok; ++tile, ++it) {
        const int stage = it & 1;
        const uint32_t phase = (it >> 1) & 1u;
        uint8_t* k_tile = smem + (2 + stage) * OP;
        uint8_t* v_tile = smem + (4 + stage) * OP;
        if (it >= 2) wait(&bars.k_empty[stage], phase ^ 1u);
        // ---- keys: a word is eight dims, one 16-byte chunk of the key's row
        uint32_t hide = flip;  // a key whose value row is NaN scores NaN, so whoever sees it becomes NaN
#pragma unroll
        for (int k = 0; k < NG; ++k)
          if (not_finite<kBf16>(vq[k])) hide = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const uint32_t par = hide == 0xFFFFFFFFu ? hide : kp[i * NG / NW] ^ hide;
          const uint32_t s2 = __byte_perm(par, par, 0x1010), m2 = __byte_perm(par, par, 0x3232);
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            const uint32_t x = kc[cc * NW + i];  // dims 32 i + 8 cc ..
            using N = Kv4Nib<T>;
            uint4 v;
            v.x = N::fma2(N::sub2(N::template pair<0>(x, magic), magic), s2, m2);
            v.y = N::fma2(N::sub2(N::template pair<1>(x, magic), magic), s2, m2);
            v.z = N::fma2(N::sub2(N::template pair<2>(x, magic), magic), s2, m2);
            v.w = N::fma2(N::sub2(N::template pair<3>(x, magic), magic), s2, m2);
            const int chunk = 4 * i + cc;
            *reinterpret_cast<uint4*>(k_tile + (chunk / 8) * 128 * 128 + sw128_offset(key, chunk % 8)) = v;
          }
        }
        fence_proxy_async_smem();
        if (!(p.withhold && it == 0 && dw == 0 && blockIdx.x == 0)) warp_arrive(&bars.k_full[stage]);
        if (tile == first) copy_q();
        if (tile + 1 < last) {
          advance();
          load_k(tile + 1);
        }
        if (tile == first) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_proxy_async_smem();
          warp_arrive(&bars.q_full);
        }
        if (it >= 2) wait(&bars.v_empty[stage], phase ^ 1u);
        // ---- values: rows are dims, a chunk is eight tokens
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          uint32_t s2[4], m2[4];  // token pairs
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t a = vp[2 * cc * NG + grp], b = vp[(2 * cc + 1) * NG + grp];
            // NaN parameters: zeros here, the key's scores carry the NaN
            if (not_finite<kBf16>(a)) a = 0;
            if (not_finite<kBf16>(b)) b = 0;
            s2[cc] = __byte_perm(a, b, 0x5410);
            m2[cc] = __byte_perm(a, b, 0x7632);
          }
#pragma unroll
          for (int i = grp * NW / NG; i < (grp + 1) * NW / NG; ++i) {
            using N = Kv4Nib<T>;
            uint32_t o[4][4];
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) {
              const uint32_t x = vc[cc * NW + i];
              o[0][cc] = N::fma2(N::sub2(N::template pair<0>(x, magic), magic), s2[cc], m2[cc]);
              o[1][cc] = N::fma2(N::sub2(N::template pair<1>(x, magic), magic), s2[cc], m2[cc]);
              o[2][cc] = N::fma2(N::sub2(N::template pair<2>(x, magic), magic), s2[cc], m2[cc]);
              o[3][cc] = N::fma2(N::sub2(N::template pair<3>(x, magic), magic), s2[cc], m2[cc]);
            }
            const int chunk = (2 * dw + vr) * 2 + vh;  // of 16 chunks of eight keys
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              const int d = 32 * i + 4 * vg + jj;
              *reinterpret_cast<uint4*>(v_tile + (chunk / 8) * D * 128 + sw128_offset(d, chunk % 8)) =
                  make_uint4(o[jj][0], o[jj][1], o[jj][2], o[jj][3]);
            }
          }
        }
        fence_proxy_async_smem();
        warp_arrive(&bars.v_full[stage]);
        if (tile + 1 < last) load_v(tile + 1);
      }
      u = ue;
      if (u >= w.u1 || !w.next(p)) break;
    }
  } else {
    // ================================================================ products
    constexpr uint32_t idesc_s = make_idesc_f16(128, 64, kBf16), idesc_o = make_idesc_f16(128, D, kBf16);
    // The whole warp walks the loop, so that descriptors and addresses stay warp-uniform, and one
    // elected lane issues: a lane that walks alone takes half as long again for a step.
    const uint64_t base = make_sw128_desc(smem_u32(smem));
    uint32_t it = 0, q_phase = 0, p_phase[2] = {0, 0};
    bool ok = true;
    const auto wait = [&](uint64_t* bar, uint32_t phase) { ok = __all_sync(~0u, ok && mbar_wait(bar, phase & 1u)); };
    const auto issue_s = [&](int t, int h, uint32_t x) {
      const uint64_t a = base + (uint64_t)(t * (OP >> 4)),
                     b = base + (uint64_t)((2 + (x & 1)) * (OP >> 4) + h * (64 * 128 >> 4));
      const uint32_t d = tmem + t * 128 + h * 64;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint64_t off = ((k / 4) * 128 * 128 + (k % 4) * 32) >> 4;
        umma_f16(d, a + off, b + off, idesc_s, k > 0);
      }
      umma_commit(&bars.s_full[t][h]);
    };
    const auto issue_o = [&](int t, int h, uint32_t x, bool accumulate) {
      const uint64_t b = base + (uint64_t)((4 + (x & 1)) * (OP >> 4) + h * (D * 128 >> 4));
      const uint32_t a = tmem + t * 128 + h * 64, d = tmem + 256 + t * 128;
#pragma unroll
      for (int k = 0; k < 4; ++k) umma_f16_ts(d, a + k * 8, b + (k * 32 >> 4), idesc_o, k > 0 || accumulate);
    };
    for (long long u = w.u0; u < w.u1 && ok;) {
      const long long ue = min(w.u1, w.item + w.n_tiles);
      int first, last;
      w.part_tiles(u, ue, first, last);
      const int n = __shfl_sync(~0u, last - first, 0);
      const int tiles = __shfl_sync(~0u, w.req.n * p.G - w.rb * kPRows > 128 ? 2 : 1, 0);
      if (n == 0) break;
      wait(&bars.k_full[it & 1], it >> 1);
      wait(&bars.q_full, q_phase);
      q_phase ^= 1u;
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (t < tiles) issue_s(t, h, it);
        umma_commit(&bars.k_empty[it & 1]);
      }
      __syncwarp();
#pragma unroll 1
      for (int x = 0; x < n && ok; ++x, ++it) {
        const bool ahead = x + 1 < n;
        wait(&bars.v_full[it & 1], it >> 1);
        if (ahead) wait(&bars.k_full[(it + 1) & 1], (it + 1) >> 1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (t < tiles) {
              wait(&bars.p_full[t][h], p_phase[t]);
              tc_fence_after();
              if (ok && elect_one()) {
                issue_o(t, h, it, x > 0 || h > 0);
                if (ahead) issue_s(t, h, it + 1);
                else umma_commit(&bars.o_done[t][h]);
                if (h == 1 && t == tiles - 1) {
                  umma_commit(&bars.v_empty[it & 1]);
                  if (ahead) umma_commit(&bars.k_empty[(it + 1) & 1]);
                }
              }
              __syncwarp();
            }
        p_phase[0] ^= 1u;
        if (tiles == 2) p_phase[1] ^= 1u;
      }
      u = ue;
      if (u >= w.u1 || !w.next(p)) break;
    }
    // No product may be in flight when TMEM is freed and the block ends, also after a wait that ran out.
    if (elect_one()) umma_commit(&bars.drained);
    __syncwarp();
    mbar_wait(&bars.drained, 0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

template <typename T, int D, int NG>
cudaError_t launch_one(const Kv4AttnParams& p, int sms, bool pdl, cudaStream_t stream) {
  const auto kernel = kv4_prompt_kernel<T, D, NG>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), prompt_smem<D>());
  if (e != cudaSuccess) return e;
  const int grid = sms < kKv4PromptMaxGrid ? sms : kKv4PromptMaxGrid;
  return kv4_launch(kernel, dim3((unsigned)grid), kPThreads, prompt_smem<D>(), pdl, stream, p);
}

template <typename T>
cudaError_t launch_t(const Kv4AttnParams& p, int sms, bool pdl, cudaStream_t stream) {
  const int ng = p.c.D / p.c.group;
  if (p.c.D == 128) {
    if (ng == 1) return launch_one<T, 128, 1>(p, sms, pdl, stream);
    if (ng == 2) return launch_one<T, 128, 2>(p, sms, pdl, stream);
    return launch_one<T, 128, 4>(p, sms, pdl, stream);
  }
  if (ng == 1) return launch_one<T, 64, 1>(p, sms, pdl, stream);
  return launch_one<T, 64, 2>(p, sms, pdl, stream);
}

}  // namespace

int64_t kv4_prompt_partial_bytes(int D) { return (int64_t)2 * kKv4PromptMaxGrid * slot_floats(D) * 4; }

cudaError_t launch_kv4_attn_prompt(const Kv4AttnParams& p, int sms, bool bf16, bool pdl, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, sms, pdl, stream) : launch_t<__half>(p, sms, pdl, stream);
}

}  // namespace fqkv
