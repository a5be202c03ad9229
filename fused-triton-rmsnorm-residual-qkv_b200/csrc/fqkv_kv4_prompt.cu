// fqkv_kv4_prompt.cu -- causal attention over the paged 4-bit cache for many query rows per KV
// head (prompts and chunks of prompts), on tcgen05.
//
// Mathematics.  S = Q K^T and O = P V with the online softmax: P = exp2(c S - c ref), where c is
// the score scale times log2(e) and ref a row maximum that is only moved (and O and the row sum
// rescaled) when the true maximum exceeds it by 8 in the exponent; P stays below 2^8 and the
// quotient O / sum does not depend on ref.  Keys and values are formed once per CTA as
// round16(scale * code + minimum), one rounding to the cache's type (the operand type of the
// product); P is rounded to the same type, row sums, maxima and accumulators are fp32.
//
// Shape.  A CTA takes 256 query rows of one KV head (all heads that share it, so the keys are
// unpacked once for them) as two tiles of 128 and walks the keys 128 at a time:
//   warps 0-3, 4-7   softmax of the two tiles, one row per thread, S and O in TMEM; P goes back
//                    to TMEM over S and is the A operand of the second product
//   warps 8-11       4-bit codes from global memory to swizzled shared-memory operands
//   warp 12          issues the products: S0(j+1) follows P0 V(j), S1(j+1) follows P1 V(j), so
//                    one tile's softmax runs under the other tile's products
// The values are stored transposed (dims x keys, K-major) because the cache interleaves tokens
// in pairs: a thread's eight tokens of one dim are one 16-byte store without any permutation.
//
// Bound: per 128 keys the four products take 2048 tensor cycles, the softmax 32768 exponentials
// (2048 cycles of the special function unit) and the unpacking about 500 issue cycles.
#include "fqkv_kv4_work.cuh"

namespace fqkv {
namespace {

constexpr int kPThreads = 416;  // 13 warps: 128 registers a thread
constexpr int kPRows = 256;
constexpr int kPTile = 128;  // keys per step
constexpr int kPMinTiles = 4;

using Work = Kv4Work<kPRows, kPTile, kPThreads, 1>;

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
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      FQKV_W8(r, 0), FQKV_W8(r, 8), FQKV_W8(r, 16), FQKV_W8(r, 24)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      FQKV_W8(r, 0), FQKV_W8(r, 8)
      : "memory");
}

// Scores of keys outside [lo, hi) of this chunk become -inf.
__device__ __forceinline__ void hide32(uint32_t (&r)[32], int lo, int hi) {
#pragma unroll
  for (int k = 0; k < 32; ++k)
    if (k < lo || k >= hi) r[k] = 0xFF800000u;
}
__device__ __forceinline__ float max32(const uint32_t (&r)[32]) {
  float m[4];
#pragma unroll
  for (int k = 0; k < 32; ++k) m[k & 3] = k < 4 ? __uint_as_float(r[k]) : fmaxf(m[k & 3], __uint_as_float(r[k]));
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// P = exp2(c S - off) of 32 keys to 16 columns at `dst`; returns their fp32 sum.
template <typename T>
__device__ __forceinline__ float exp32(const uint32_t (&r)[32], float c, float off, uint32_t dst) {
  uint32_t pk[16];
  float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float x = kv4_exp2(fmaf(__uint_as_float(r[2 * k]), c, -off));
    const float y = kv4_exp2(fmaf(__uint_as_float(r[2 * k + 1]), c, -off));
    a[2 * (k & 1)] += x, a[2 * (k & 1) + 1] += y;
    pk[k] = Elem<T>::from_f2(x, y);
  }
  tmem_st16(dst, pk);
  return (a[0] + a[1]) + (a[2] + a[3]);
}

struct Bars {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t q_full[2], s_full[2], p_full[2], o_done[2];
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
  constexpr bool kBf16 = sizeof(T) == 2 && Kv4Nib<T>::kOffset == 128.0f;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ Work::Shared s_work;
  __shared__ uint32_t s_tmem;
  __shared__ int s_last;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.k_full[i], 128);
      mbar_init(&bars.v_full[i], 128);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_empty[i], 1);
      mbar_init(&bars.q_full[i], 128);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 128);
      mbar_init(&bars.o_done[i], 1);
    }
    fence_mbarrier_init_cluster();
  }
  pdl_wait();
  pdl_launch_dependents();
  Work w;
  if (!w.locate(p, s_work, gridDim.x, kPMinTiles)) return;
  if (warp == 12) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const auto s_col = [&](int t) { return tmem + t * 128; };        // S, and P over it
  const auto o_col = [&](int t) { return tmem + 256 + t * 128; };  // O

  if (warp < 8) {
    // ================================================================ softmax
    const int t = warp >> 2, row = tid & 127;  // tile, row of the tile = TMEM lane
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const float c = fabsf(p.scale_log2);
    const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;  // a negative scale goes into Q
    uint32_t s_phase = 0, o_phase = 0;
    bool ok = true;  // after a wait that ran out nothing is waited for, and every barrier is still reached
    for (long long u = w.u0; u < w.u1;) {
      const long long ue = min(w.u1, w.item + w.n_tiles);
      const int first = w.tile_lo + (int)(u - w.item), last = first + (int)(ue - u);
      const int rows = w.req.n * p.G - w.rb * kPRows;  // live rows of the block
      const int grow = w.rb * kPRows + t * 128 + row;  // row of the request
      const int j = grow / p.G, h = grow - j * p.G;
      const bool live = j < w.req.n;
      const int pos = w.req.len - w.req.n + j;
      const bool tile_used = rows > t * 128;
      float ref = -INFINITY, sum = 0.0f;
      if (tile_used) {
        // ---- this row of Q into the tile's operand
        uint8_t* q_tile = smem + t * OP;
        const uint16_t* q = p.q + (p.query_start ? (int64_t)(w.req.start + j) * p.q_t : w.r * p.q_r + j * p.q_t) +
                            (int64_t)(w.kvh * p.G + h) * p.q_h;
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (live) v = *reinterpret_cast<const uint4*>(q + k * 8);
          v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
          *reinterpret_cast<uint4*>(q_tile + (k / 8) * 128 * 128 + sw128_offset(row, k % 8)) = v;
        }
        fence_proxy_async_smem();
        mbar_arrive(&bars.q_full[t]);

        const int see_hi = live ? min(pos + 1, w.req.len) : w.req.len;      // keys [see_lo, see_hi)
        const int see_lo = live && p.window > 0 ? max(0, pos - p.window + 1) : 0;
        const bool warp_live = rows > t * 128 + (warp & 3) * 32;
        for (int tile = first; tile < last; ++tile) {
          ok = __all_sync(~0u, ok && mbar_wait(&bars.s_full[t], s_phase & 1u));
          s_phase ^= 1u;
          tc_fence_after();
          if (warp_live) {
            // The row's 128 scores are read twice, for the maximum and for the exponentials, 64 at a
            // time: a thread stays within the 128 registers that 13 warps leave it.
            uint32_t r0[32], r1[32];
            const int lo = see_lo - tile * kPTile, hi = see_hi - tile * kPTile;
            const bool edge = __any_sync(~0u, lo > 0 || hi < kPTile);
            tmem_ld32(s_col(t) + lane_base, r0);
            tmem_ld32(s_col(t) + lane_base + 32, r1);
            tmem_wait_ld();
            if (edge) hide32(r0, lo, hi), hide32(r1, lo - 32, hi - 32);
            float top = fmaxf(max32(r0), max32(r1));
            tmem_ld32(s_col(t) + lane_base + 64, r0);
            tmem_ld32(s_col(t) + lane_base + 96, r1);
            tmem_wait_ld();
            if (edge) hide32(r0, lo - 64, hi - 64), hide32(r1, lo - 96, hi - 96);
            top = fmaxf(top, fmaxf(max32(r0), max32(r1)));
            // ---- move the reference, and rescale O and the sum, when the maximum outgrew it
            if (__any_sync(~0u, top > ref && (top - ref) * c > 8.0f)) {
              const float to = fmaxf(top, ref);
              const float f = to == -INFINITY ? 1.0f : kv4_exp2((ref - to) * c);
              ref = to;
              sum *= f;
              if (tile > first) {
                ok = __all_sync(~0u, ok && mbar_wait(&bars.o_done[t], (o_phase ^ 1u) & 1u));
                tc_fence_after();
#pragma unroll 1
                for (int k = 0; k < D / 32; ++k) {
                  uint32_t o[32];
                  tmem_ld32(o_col(t) + lane_base + k * 32, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                  tmem_st32(o_col(t) + lane_base + k * 32, o);
                }
                tmem_wait_st();
              }
            }
            const float off = ref == -INFINITY ? 0.0f : ref * c;
            // P (16-bit pairs) over the scores that have been read: columns 0-63 of the tile's S.
            tmem_ld32(s_col(t) + lane_base, r0);
            tmem_ld32(s_col(t) + lane_base + 32, r1);
            tmem_wait_ld();
            if (edge) hide32(r0, lo, hi), hide32(r1, lo - 32, hi - 32);
            sum += exp32<T>(r0, c, off, s_col(t) + lane_base);
            tmem_ld32(s_col(t) + lane_base + 64, r0);
            sum += exp32<T>(r1, c, off, s_col(t) + lane_base + 16);
            tmem_ld32(s_col(t) + lane_base + 96, r1);
            tmem_wait_ld();
            if (edge) hide32(r0, lo - 64, hi - 64), hide32(r1, lo - 96, hi - 96);
            sum += exp32<T>(r0, c, off, s_col(t) + lane_base + 32);
            sum += exp32<T>(r1, c, off, s_col(t) + lane_base + 48);
            tmem_wait_st();
          }
          o_phase ^= 1u;  // the product of this tile completes phase o_phase ^ 1 of o_done
          tc_fence_before();
          mbar_arrive(&bars.p_full[t]);
        }
        // ---- O of the piece is complete
        ok = __all_sync(~0u, ok && mbar_wait(&bars.o_done[t], (o_phase ^ 1u) & 1u));
        tc_fence_after();
      }

      const bool complete = u == w.item && ue == w.item + w.n_tiles;
      uint16_t* out = p.out + (int64_t)(w.req.start + j) * p.o_t + (int64_t)(w.kvh * p.G + h) * D;
      if (complete) {
        if (tile_used) {
          const float inv = sum > 0.0f ? 1.0f / sum : sum;  // nothing seen: zeros; NaN stays
#pragma unroll 1
          for (int k = 0; k < D / 32; ++k) {
            uint32_t o[32];
            tmem_ld32(o_col(t) + lane_base + k * 32, o);
            tmem_wait_ld();
            if (live) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                uint4 v;
                v.x = Elem<T>::from_f2(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
                v.y = Elem<T>::from_f2(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
                v.z = Elem<T>::from_f2(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
                v.w = Elem<T>::from_f2(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
                *reinterpret_cast<uint4*>(out + k * 32 + e) = v;
              }
            }
          }
        }
      } else {
        // Part: reference and sum per row, then O as [dims / 4][rows] groups of four.
        const int fc = w.first_cta(), lc = w.last_cta(), me = (int)blockIdx.x;
        const int brow = t * 128 + row;
        float* part = p.partial + (int64_t)(2 * me + (w.item < w.u0 ? 0 : 1)) * slot_floats(D);
        if (tile_used) {
          part[brow] = ref;
          part[kPRows + brow] = sum;
#pragma unroll 1
          for (int k = 0; k < D / 32; ++k) {
            uint32_t o[32];
            tmem_ld32(o_col(t) + lane_base + k * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(part + 2 * kPRows + ((k * 8 + e / 4) * kPRows + brow) * 4) =
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
          float top = -INFINITY, l = 0.0f;
          for (int x = fc; x <= lc; ++x) top = fmaxf(top, __ldcg(slot(x) + brow));
          const float to = top == -INFINITY ? 0.0f : top;
          for (int x = fc; x <= lc; ++x)
            l += __ldcg(slot(x) + kPRows + brow) * kv4_exp2((__ldcg(slot(x) + brow) - to) * c);
          const float inv = l > 0.0f ? 1.0f / l : l;
          if (live) {
#pragma unroll 1
            for (int k = 0; k < D / 32; ++k) {
              float v[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = 0.0f;
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
      if (u >= w.u1 || !w.next(p)) break;
    }
  } else if (warp < 12) {
    // ================================================================ codes to operands
    const int dw = warp - 8, key = tid - 256;
    const int vr = (lane >> 1) & 1, vh = lane & 1, vg = lane >> 2;  // values: record, token half, dim group
    const int rpb = p.c.P / kKv4Rec;
    uint32_t it = 0;
    bool ok = true;
    uint32_t kc[4 * NW], kp[NG], vq[NG], vc[4 * NW], vp[8 * NG];
    const uint8_t *ra, *rb;  // this warp's two records of a tile
    for (long long u = w.u0; u < w.u1 && ok;) {
      const long long ue = min(w.u1, w.item + w.n_tiles);
      const int first = w.tile_lo + (int)(u - w.item), last = first + (int)(ue - u);
      const int* table = p.table + (int64_t)w.r * p.table_stride;
      const int n_rec = (w.req.len + kKv4Rec - 1) / kKv4Rec;
      const auto records = [&](int tile) {
        ra = kv4_record(p, table, tile * 8 + 2 * dw, n_rec, rpb, w.kvh, REC);
        rb = kv4_record(p, table, tile * 8 + 2 * dw + 1, n_rec, rpb, w.kvh, REC);
      };
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
      records(first);
      load_k(first);
      load_v(first);
      for (int tile = first; tile < last && ok; ++tile, ++it) {
        const int stage = it & 1;
        const uint32_t phase = (it >> 1) & 1u;
        uint8_t* k_tile = smem + (2 + stage) * OP;
        uint8_t* v_tile = smem + (4 + stage) * OP;
        if (it >= 2) ok = mbar_wait(&bars.k_empty[stage], phase ^ 1u);
        // ---- keys: a word is eight dims, one 16-byte chunk of the key's row
        uint32_t hide = 0;  // a key whose value row is NaN scores NaN, so whoever sees it becomes NaN
#pragma unroll
        for (int k = 0; k < NG; ++k)
          if (not_finite<kBf16>(vq[k])) hide = 0x7FFF7FFFu;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const uint32_t par = kp[i * NG / NW];
          const uint32_t s2 = __byte_perm(par, par, 0x1010), m2 = __byte_perm(par, par, 0x3232);
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            const uint32_t x = kc[cc * NW + i];  // dims 32 i + 8 cc ..
            using N = Kv4Nib<T>;
            uint4 v;
            v.x = N::fma2(N::sub2(N::template pair<0>(x), N::kOffset2), s2, m2) | hide;
            v.y = N::fma2(N::sub2(N::template pair<1>(x), N::kOffset2), s2, m2) | hide;
            v.z = N::fma2(N::sub2(N::template pair<2>(x), N::kOffset2), s2, m2) | hide;
            v.w = N::fma2(N::sub2(N::template pair<3>(x), N::kOffset2), s2, m2) | hide;
            const int chunk = 4 * i + cc;
            *reinterpret_cast<uint4*>(k_tile + (chunk / 8) * 128 * 128 + sw128_offset(key, chunk % 8)) = v;
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(&bars.k_full[stage]);
        if (tile + 1 < last) {
          records(tile + 1);
          load_k(tile + 1);
        }
        if (it >= 2) ok = ok && mbar_wait(&bars.v_empty[stage], phase ^ 1u);
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
              o[0][cc] = N::fma2(N::sub2(N::template pair<0>(x), N::kOffset2), s2[cc], m2[cc]);
              o[1][cc] = N::fma2(N::sub2(N::template pair<1>(x), N::kOffset2), s2[cc], m2[cc]);
              o[2][cc] = N::fma2(N::sub2(N::template pair<2>(x), N::kOffset2), s2[cc], m2[cc]);
              o[3][cc] = N::fma2(N::sub2(N::template pair<3>(x), N::kOffset2), s2[cc], m2[cc]);
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
        mbar_arrive(&bars.v_full[stage]);
        if (tile + 1 < last) load_v(tile + 1);
      }
      u = ue;
      if (u >= w.u1 || !w.next(p)) break;
    }
  } else {
    if (lane == 0) {
      // ============================================================== products
      constexpr uint32_t idesc_s = make_idesc_f16(128, 128, kBf16), idesc_o = make_idesc_f16(128, D, kBf16);
      const uint32_t base = smem_u32(smem);
      uint32_t it = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
      bool ok = true;
      const auto issue_s = [&](int t, int stage) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k / 4) * 128 * 128 + (k % 4) * 32;
          umma_f16(s_col(t), make_sw128_desc(base + t * OP + off), make_sw128_desc(base + (2 + stage) * OP + off),
                   idesc_s, k > 0);
        }
        umma_commit(&bars.s_full[t]);
      };
      const auto issue_o = [&](int t, int stage, bool accumulate) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_f16_ts(o_col(t), s_col(t) + k * 8,
                      make_sw128_desc(base + (4 + stage) * OP + (k / 4) * D * 128 + (k % 4) * 32), idesc_o,
                      accumulate || k > 0);
        umma_commit(&bars.o_done[t]);
      };
      for (long long u = w.u0; u < w.u1 && ok;) {
        const long long ue = min(w.u1, w.item + w.n_tiles);
        const int n = (int)(ue - u);
        const int tiles = w.req.n * p.G - w.rb * kPRows > 128 ? 2 : 1;
        for (int x = 0; x <= n && ok; ++x) {
          // Step x: the second products of tile x - 1, then the first products of tile x.
          const uint32_t a = it + x, b = it + x - 1;
          if (x < n) ok = ok && mbar_wait(&bars.k_full[a & 1], (a >> 1) & 1u);
          if (x > 0) ok = ok && mbar_wait(&bars.v_full[b & 1], (b >> 1) & 1u);
          for (int t = 0; t < tiles && ok; ++t) {
            if (x == 0) {
              ok = ok && mbar_wait(&bars.q_full[t], q_phase[t]);
              q_phase[t] ^= 1u;
            } else {
              ok = ok && mbar_wait(&bars.p_full[t], p_phase[t]);
              p_phase[t] ^= 1u;
            }
            tc_fence_after();
            if (!ok) break;
            if (x > 0) issue_o(t, b & 1, x > 1);
            if (x < n) issue_s(t, a & 1);
          }
          if (x < n) umma_commit(&bars.k_empty[a & 1]);
          if (x > 0) umma_commit(&bars.v_empty[b & 1]);
        }
        it += n;
        u = ue;
        if (u >= w.u1 || !w.next(p)) break;
      }
      // Everything issued has completed before TMEM is freed.
      mbar_wait(&bars.k_empty[(it - 1) & 1], ((it - 1) >> 1) & 1u);
      mbar_wait(&bars.v_empty[(it - 1) & 1], ((it - 1) >> 1) & 1u);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
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
