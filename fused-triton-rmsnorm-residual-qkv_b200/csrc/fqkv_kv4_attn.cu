// fqkv_kv4_attn.cu -- causal attention over the paged 4-bit cache for few query rows per KV
// head (single tokens, drafts): split over the key axis, one pass over the codes.
//
// Mathematics.  A code c stands for s c + m, with s and m per token and group of dims, so
//   q . k_t = sum_groups ( s_tg * (q_g . c_tg) + m_tg * sum(q_g) )
//   sum_t p_t v_t = sum_t (p_t s_tg) (c_tg - 8) + sum_t p_t (m_tg + 8 s_tg).
// The tensor cores multiply the small integers, exact in fp16, and the parameters meet the scores
// and the probabilities in fp32: no dequantised tile is ever formed.  Four bits become an fp16
// number by placing them in the mantissa of a constant (1024 + c or 64 + c): a word's eight codes
// cost one shift and four three-input logic operations.  For the keys the constants are taken back
// by the value the accumulator starts with; for the values they are subtracted and the codes
// centred, so that the sum over a long context does not cancel a large offset.  bf16 queries are
// divided by a power of two per row and group, exactly but for numbers 2^-14 below their group's
// largest.  p s is rounded to 16 bits for the product (the one rounding to fewer than 32 bits besides
// the output); maxima, sums and outputs are fp32.  The reference exponent holds the largest p s at
// 2^15, near the end of fp16's range, so that a weight keeps its eleven bits down to 2^-29 of the
// largest and is dropped below 2^-40 of it (2^20 such weights are 2^-20 of it).  Where a head has
// several groups, s is in the group's own unit, so that "the largest" is the group's own up to what
// its scales differ from key to key.
//
// Shape.  Both products are transposed (keys x queries and dims x queries, m16n8k16), so the
// query heads that share a KV head fill the 8-wide side and 1 to 8 query rows cost the same.
// A record's bytes are stored in fragment order: a warp's 16-byte shared loads are conflict
// free and need no transposition (the values' tokens are interleaved in pairs).
//
// Bound: the codes' bytes over HBM, 2176 per 16 tokens and KV head at D = 128 with one group, about
// 90 cycles of an SM's share of the bandwidth.  Measured (B200, bf16, 64 requests of 1 to 8000
// tokens, 32 / 8 heads, 288 MB): 87 us, 3.3 TB/s; copies alone 58 us, everything but the products
// and their unpacking 64 us.  The rest is issue: about 350 instructions a record, of which the
// logic pipe (one per two cycles and scheduler) takes about half.
//
// Split.  The items (request, KV head, block of query rows) are laid end to end as tiles of 32
// tokens and cut into equal runs, one per CTA and within it one per warp, whatever the lengths.  A
// warp streams its run through a ring of its own, filled by bulk copies of whole records, without
// a barrier between items; a CTA's warps join their parts once, at the end.  An item cut between
// CTAs is joined by the CTA that arrives last, which adds the parts in the order of the CTAs, so
// the result does not depend on the arrival order.
#include "fqkv_kv4_work.cuh"

namespace fqkv {
namespace {

constexpr int kTile = 32;    // tokens per ring stage (two records)
constexpr float kRoom = 15.0f;  // log2 of the largest weight p s
// Several groups in a head have a unit each, a power of two between 2^-60 and 2^60 that keeps the
// largest of the group's scales so far below 1; it is taken with a factor of four to spare, so that it
// hardly moves.
constexpr int kMostUnit = 60, kUnitRoom = 2;

// Untiled bulk copy global -> shared, counted on a local mbarrier.  Addresses and size are
// multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight codes of a word as four fp16 pairs (nibbles j and j + 4): 1024 + code for j = 0, 2, where
// the four bits are the mantissa's lowest, 64 + code for j = 1, 3, where they are bits 4-7.
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t low, uint32_t high, uint32_t& p0, uint32_t& p1,
                                           uint32_t& p2, uint32_t& p3) {
  const uint32_t v = w >> 8;
  p0 = kv4_place<0x000F000Fu>(w, low);
  p1 = kv4_place<0x00F000F0u>(w, high);
  p2 = kv4_place<0x000F000Fu>(v, low);
  p3 = kv4_place<0x00F000F0u>(v, high);
}
constexpr uint32_t kMagicLow = 0x64006400u;    // 1024
constexpr uint32_t kMagicHigh = 0x54005400u;   // 64
constexpr uint32_t kCentreLow = 0x64086408u;   // 1032 = 1024 + 8
constexpr uint32_t kCentreHigh = 0x54805480u;  // 72 = 64 + 8

__device__ __forceinline__ uint32_t sub_f16x2(uint32_t x, uint32_t y) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  lo = Elem<T>::to_f((uint16_t)w);
  hi = Elem<T>::to_f((uint16_t)(w >> 16));
}
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t w, float& lo, float& hi) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xFFFF0000u);
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

__device__ __forceinline__ float reciprocal_of_power(float x) {
  return __uint_as_float((254u << 23) - __float_as_uint(x));
}

// a / b by an approximate reciprocal and one step of refinement; exact where the quotient is a
// small integer.  Not meaningful for b = 0 or subnormal.
__device__ __forceinline__ float quotient(float a, float b) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(b));
  const float q = a * r;
  return fmaf(fmaf(-q, b, a), r, q);
}

__device__ __forceinline__ float log2_approx(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// Query rows of an item.  Sixteen rows unpack the codes half as often, but leave a warp
// its accumulators only at twelve warps an SM: 54 us against 44 us for two items of eight (16
// requests of 500 to 6000 tokens, 16 rows on 8 KV heads), 84 against 62 us at 24 rows.
constexpr int kRows = 8;
// Warps of a CTA, two CTAs on an SM; fewer where eight rings of larger records leave no room (seven
// of two groups fit, but have 128 registers a thread, as eight have, which spill: 64 requests with
// groups of 64 take 117.7 us with seven and 113.5 with six).
template <int D, int NG>
constexpr int warps() {
  return D == 128 ? (NG == 1 ? 8 : 6) : 8;
}
// Ring stages of a warp, about 9 KB.
template <int D>
constexpr int stages() {
  return D == 128 ? 2 : 4;
}
template <int D, int NG>
constexpr int ring_bytes() {
  return stages<D>() * 2 * kv4_record_bytes(D, NG);
}
// A warp's part of an item as floats: its outputs by column, padded by four floats so that the
// float4 stores of a quarter-warp (four columns, two dim groups) meet eight different bank groups.
template <int D>
constexpr int part_floats() {
  return kRows * (D + 4);
}
// A stage's parameters as the lanes use them, per token and group: the values' {s, r, z, log2 of
// the token's largest s less kRoom}, s and z in the group's unit, then the keys' {s, m}.
template <int NG>
constexpr int param_bytes() {
  return kTile * NG * 24;
}
template <int D, int NG>
constexpr int smem_bytes() {
  return warps<D, NG>() * (ring_bytes<D, NG>() + part_floats<D>() * 4 + param_bytes<NG>());
}

// What the join needs to know of a warp's part of an item.
struct PartInfo {
  long long item;  // first tile of the item in the batch; -1: no part
  int n_tiles, row0, start, n, head0;
};

template <typename T, int D, int NG>
__global__ void __launch_bounds__(warps<D, NG>() * 32, 2)
    kv4_attn_split_kernel(const Kv4AttnParams p) {
  constexpr int WARPS = warps<D, NG>(), THREADS = WARPS * 32;
  constexpr int ROWS = kRows;            // query rows of an item
  constexpr int REC = kv4_record_bytes(D, NG), kStages = stages<D>();
  constexpr int NW = D / 32;             // 32-dim blocks: words per lane and key row
  constexpr int WPG = NW / NG;           // words of one scale group
  constexpr int PART = part_floats<D>();
  static_assert(PART * 4 <= ring_bytes<D, NG>(), "a part fits the ring");
  using Work = Kv4Work<ROWS, kTile, THREADS, WARPS, 0>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_bar[WARPS][kStages];
  __shared__ typename Work::Shared s_work;
  __shared__ Work s_item[WARPS], s_ahead[WARPS];  // each warp's item, and the item its copies have reached
  __shared__ PartInfo s_info[WARPS][2];
  __shared__ float s_max[WARPS][2][ROWS], s_sum[WARPS][2][ROWS];
  __shared__ __align__(16) float s_unit[WARPS][NG];  // powers of two that a warp's groups' scales are multiplied by
  __shared__ int s_last[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const uint32_t magic_low = kv4_opaque(kMagicLow, p.n_q), magic_high = kv4_opaque(kMagicHigh, p.n_q);
  uint8_t* ring = smem + warp * ring_bytes<D, NG>();
  float* parts = reinterpret_cast<float*>(smem + WARPS * ring_bytes<D, NG>());
  float4* pv = reinterpret_cast<float4*>(smem + WARPS * (ring_bytes<D, NG>() + PART * 4) + warp * param_bytes<NG>());
  float2* pk = reinterpret_cast<float2*>(pv + kTile * NG);
  // Slot 0: a part that the warp finished before its run ended.  Slot 1: its last part, in the
  // ring, which is idle by then.
  const auto part_at = [&](int w, int slot) -> float* {
    return slot ? reinterpret_cast<float*>(smem + w * ring_bytes<D, NG>()) : parts + w * PART;
  };
  if (tid < WARPS * kStages) {
    mbar_init(&s_bar[tid / kStages][tid % kStages], 2);  // a tile's two records
    fence_mbarrier_init_cluster();
  }
  pdl_wait();
  pdl_launch_dependents();
  {
    Work first;
    if (!first.locate(p, s_work, gridDim.x, WARPS)) return;  // its barriers publish the mbarriers
    if (lane == 0) {
      s_item[warp] = s_ahead[warp] = first;
      s_info[warp][0].item = s_info[warp][1].item = -1;
    }
    __syncwarp();
  }
  // The warp's items live in shared memory: a few loads now and then instead of registers that the
  // inner loop needs.
  const Work& w = s_item[warp];
  const long long run_end = w.b;

  // ---- copies: the warp's run of tiles, in order, across its items
  const uint8_t *src = nullptr, *src_next = nullptr;  // records 2 src_tile + lane, and the 32 after them
  int src_tile = 0, ahead_tile, ahead_end;  // next tile to copy, end of this item's part of the run
  int stage_in = 0;
  int to_copy = (int)(run_end - w.a);
  const auto address = [&](int rec) {
    const Work& x = s_ahead[warp];
    return kv4_record(p, p.table + (int64_t)x.r * p.table_stride, rec, (x.req.len + kKv4Rec - 1) / kKv4Rec,
                      p.c.P / kKv4Rec, x.kvh, REC);
  };
  const auto enter = [&]() {
    const Work& x = s_ahead[warp];
    const long long at = run_end - to_copy;
    ahead_tile = x.tile_lo + (int)(at - x.item);
    ahead_end = x.tile_lo + (int)(min(run_end, x.item + x.n_tiles) - x.item);
    src_tile = ahead_tile;
    src = address(2 * ahead_tile + lane);
    src_next = 2 * ahead_end > 2 * ahead_tile + 32 ? address(2 * ahead_tile + 32 + lane) : nullptr;
  };
  const auto copy_next = [&](bool withhold) {
    if (to_copy <= 0) return;
    if (ahead_tile == ahead_end) {
      Work x = s_ahead[warp];
      __syncwarp();
      x.next(p);
      if (lane == 0) s_ahead[warp] = x;
      __syncwarp();
      enter();
    }
    if (ahead_tile - src_tile >= 16) {
      src = src_next;
      src_tile += 16;
      if (ahead_end > src_tile + 16) src_next = address(2 * (src_tile + 16) + lane);
    }
    const uint32_t k = (uint32_t)(lane - 2 * (ahead_tile - src_tile));
    if (k < 2 && !withhold) {  // the lanes of this tile's records; past the last record there is nothing to wait for
      if (src) {
        mbar_arrive_expect_tx(&s_bar[warp][stage_in], REC);
        bulk_load(smem_u32(ring + (stage_in * 2 + k) * REC), src, REC, &s_bar[warp][stage_in]);
      } else {
        mbar_arrive(&s_bar[warp][stage_in]);
      }
    }
    stage_in = stage_in + 1 == kStages ? 0 : stage_in + 1;
    ++ahead_tile;
    --to_copy;
  };
  if (to_copy > 0) enter();
#pragma unroll
  for (int s = 0; s < kStages; ++s) copy_next(s == 0 && p.withhold && blockIdx.x == 0 && warp == 0);

  int stage = 0;
  uint32_t parity = 0;  // bit s: phase of ring stage s
  bool ok = true;       // after a wait that ran out nothing is copied or waited for, and rows become NaN
  for (long long u = w.a; u < run_end;) {
    // ---- a piece: tiles [u, ue) of item w
    const long long ue = min(run_end, w.item + w.n_tiles);
    const int wt = w.tile_lo + (int)(u - w.item), we = wt + (int)(ue - u);
    const int len = w.req.len;
    // Queries: this lane's fragments (row g) in fp16, bf16 ones divided by the power of two of the
    // largest of their row and group, which is exact but for numbers 2^-14 below it.
    constexpr int NU = Kv4Nib<T>::kFullRange ? NG : 1, WPU = NW / NU;
    uint32_t qf[NW][4];
    float qs[NG][2], qo[NG][2];  // this lane's columns: sums of the queries, and minus the sums
                                 // weighted with the codes' offsets
    float cf[NU][2];             // score scale, in units of log2, times the groups' powers of two
    int col_pos[2];
    {
      const int row = w.rb * ROWS + g;
      const int j = (int)((uint32_t)row / (uint32_t)p.G), h = row - j * p.G;
      const uint16_t* qrow = p.q + (p.query_start ? (int64_t)(w.req.start + j) * p.q_t : w.r * p.q_r + j * p.q_t) +
                             (int64_t)(w.kvh * p.G + h) * p.q_h;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (j < w.req.n) v = *reinterpret_cast<const uint4*>(qrow + 8 * (4 * i + c));
        qf[i][0] = v.x, qf[i][1] = v.y, qf[i][2] = v.z, qf[i][3] = v.w;
      }
      float unit[NU];
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        unit[u] = 1.0f;
        if (Kv4Nib<T>::kFullRange) {
          float big = 0.0f;
#pragma unroll
          for (int i = u * WPU; i < (u + 1) * WPU; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float a, b;
              unpack2<T>(qf[i][e], a, b);
              big = fmaxf(big, fmaxf(fabsf(a), fabsf(b)));
            }
          big = fmaxf(big, __shfl_xor_sync(~0u, big, 1));
          big = fmaxf(big, __shfl_xor_sync(~0u, big, 2));
          // the power of two at or below `big`, within 2^+-120; an infinite or NaN row stays what it is
          const int ex = min(max((int)(__float_as_uint(big) >> 23) - 127, -120), 120);
          unit[u] = power_of_two(ex);
#pragma unroll
          for (int i = u * WPU; i < (u + 1) * WPU; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float a, b;
              unpack2<T>(qf[i][e], a, b);
              qf[i][e] = Elem<__half>::from_f2(a * power_of_two(-ex), b * power_of_two(-ex));
            }
        }
      }
      float sum[NG] = {}, off[NG] = {};
#pragma unroll
      for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float a, b;
          unpack2<__half>(qf[i][e], a, b);
          sum[i / WPG] += a + b;
          off[i / WPG] -= (e & 1 ? 64.0f : 1024.0f) * (a + b);
        }
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        sum[k] += __shfl_xor_sync(~0u, sum[k], 1);
        sum[k] += __shfl_xor_sync(~0u, sum[k], 2);
        off[k] += __shfl_xor_sync(~0u, off[k], 1);
        off[k] += __shfl_xor_sync(~0u, off[k], 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qs[k][e] = __shfl_sync(~0u, sum[k], 8 * c + 4 * e);
          qo[k][e] = __shfl_sync(~0u, off[k], 8 * c + 4 * e);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int u = 0; u < NU; ++u) cf[u][e] = p.scale_log2 * __shfl_sync(~0u, unit[u], 8 * c + 4 * e);
        col_pos[e] = kv4_position(w.req, (int)((uint32_t)(w.rb * ROWS + 2 * c + e) / (uint32_t)p.G));
      }
    }
    // Tiles in [full_lo, full_hi) are visible to every row of the block.
    const int last_j = min((int)((uint32_t)(w.rb * ROWS + ROWS - 1) / (uint32_t)p.G), w.req.n - 1);
    const int full_hi = (kv4_position(w.req, (int)((uint32_t)(w.rb * ROWS) / (uint32_t)p.G)) + 1) / kTile;
    const int full_lo = p.window > 0 ? (max(0, kv4_position(w.req, last_j) - p.window + 1) + kTile - 1) / kTile : 0;

    float out[NW][2][4];
    float top[2], sum[2], bias[NG][2];
#pragma unroll
    for (int i = 0; i < NW; ++i)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[i][m][e] = 0.0f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = -INFINITY;
      sum[e] = 0.0f;
#pragma unroll
      for (int k = 0; k < NG; ++k) bias[k][e] = 0.0f;
    }

    if (NG > 1) {
      __syncwarp();
      if (lane < NG) s_unit[warp][lane] = power_of_two(kMostUnit);
      __syncwarp();
    }
    for (int tile = ok ? wt : we; tile < we; ++tile) {
      if (!__all_sync(~0u, mbar_wait(&s_bar[warp][stage], (parity >> stage) & 1u))) {
        // Nothing may be in flight into the ring when it is used for parts and when the block ends.
        int at = stage;
        do {
          mbar_wait(&s_bar[warp][at], (parity >> at) & 1u);
          at = at + 1 == kStages ? 0 : at + 1;
        } while (at != stage_in);
        __syncwarp();
        to_copy = 0;
        ok = false;
        break;
      }
      parity ^= 1u << stage;
      const uint8_t* rec = ring + stage * 2 * REC;
      // ---- parameters: each lane prepares one token's
      {
        const uint8_t* at = rec + (lane >> 4) * REC + 16 * D + (lane & 15) * NG * 4;
        uint32_t wk[NG], wv[NG];
        lds_words<NG>(at, wk);
        lds_words<NG>(at + 64 * NG, wv);
        float sv[NG], mv[NG], unit[NG], widest = 0.0f;
        const auto scaled = [&](int grp, float u) {
          unpack2<T>(wv[grp], sv[grp], mv[grp]);
          // A scale of zero goes with codes of zero; any scale then stands for the same numbers.
          if (sv[grp] == 0.0f) sv[grp] = fmaxf(fabsf(mv[grp]), 1e-20f);
          if (NG > 1) sv[grp] *= u, mv[grp] *= u;
        };
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          unit[grp] = NG > 1 ? s_unit[warp][grp] : 1.0f;
          scaled(grp, unit[grp]);
          widest = fmaxf(widest, sv[grp]);
        }
        if constexpr (NG > 1) {
          if (__any_sync(~0u, widest > 1.0f)) {  // what was added up is brought to the new units
            const Work& x = s_item[warp];
            const int t = tile * kTile + lane;
            const int j0 = (int)((uint32_t)(x.rb * ROWS) / (uint32_t)p.G);
            const int j1 = min((int)((uint32_t)(x.rb * ROWS + ROWS - 1) / (uint32_t)p.G), x.req.n - 1);
            // (what no row of the block sees may be anything)
            const bool visible = t < x.req.len && t <= kv4_position(x.req, j1) &&
                                 (p.window <= 0 || t > kv4_position(x.req, j0) - p.window);
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
              const float old = unit[grp];
              scaled(grp, 1.0f);
              // (positive floats are ordered as integers)
              const bool counts = visible && sv[grp] < INFINITY;
              const uint32_t most = __reduce_max_sync(~0u, counts ? __float_as_uint(sv[grp]) : 0u);
              const int up = max(-kMostUnit, min(kMostUnit, 126 - kUnitRoom - (int)(most >> 23)));
              unit[grp] = fminf(old, power_of_two(up));
              const float f = unit[grp] * reciprocal_of_power(old);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                bias[grp][e] *= f;
#pragma unroll
                for (int i = grp * WPG; i < (grp + 1) * WPG; ++i)
#pragma unroll
                  for (int m = 0; m < 2; ++m) out[i][m][e] *= f, out[i][m][e + 2] *= f;
              }
            }
            widest = 0.0f;
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
              scaled(grp, unit[grp]);
              widest = fmaxf(widest, sv[grp]);
            }
            __syncwarp();
            if (lane == 0)
#pragma unroll
              for (int grp = 0; grp < NG; ++grp) s_unit[warp][grp] = unit[grp];
          }
        }
        // Below 2^-60 a token counts as 2^-60, so that its probability and their sum stay in fp32's range.
        float lg = fmaxf(log2_approx(widest), -60.0f) - kRoom;
        if (!(lg < 1e9f)) lg = 0.0f;
        // A value row that is not finite makes its key's scores NaN, so that whoever sees the key becomes
        // NaN, also where the weight would have been zero.
        float bad = 0.0f;
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) bad = fmaf(0.0f, sv[grp], fmaf(0.0f, mv[grp], bad));
        __syncwarp();                 // the previous tile's have been read
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          // The offset part p (m + 8 s) is formed from the rounded weight x = p s as x (m / s + 8),
          // so that both parts of p v carry the same rounding and a value near zero keeps a small
          // error; where the offset is far larger than the scale, from p itself, so that a weight
          // too small for fp16 loses nothing of it.
          const float q = quotient(mv[grp], sv[grp]) + 8.0f;
          const bool small = fabsf(q) <= 16.0f;
          float sk, mk;
          unpack2<T>(wk[grp], sk, mk);
          pv[lane * NG + grp] =
              make_float4(sv[grp], small ? q : 0.0f, small ? 0.0f : fmaf(8.0f, sv[grp], mv[grp]), lg);
          pk[lane * NG + grp] = make_float2(grp ? sk : sk + bad, mk);
        }
        __syncwarp();
      }
      // ---- scores, in units of log2: s[record][key g: cols, key g + 8: cols]
      float s[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint8_t* k = rec + m * REC;
        uint32_t wa[NW], wb[NW];
        lds_words<NW>(k + g * (D / 2) + c * (D / 8), wa);
        lds_words<NW>(k + (g + 8) * (D / 2) + c * (D / 8), wb);
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          float acc[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = qo[grp][e & 1];
#pragma unroll
          for (int i = grp * WPG; i < (grp + 1) * WPG; ++i) {
            uint32_t a0[4], a1[4];
            code_pairs(wa[i], magic_low, magic_high, a0[0], a0[2], a1[0], a1[2]);
            code_pairs(wb[i], magic_low, magic_high, a0[1], a0[3], a1[1], a1[3]);
            mma16816(acc, a0, qf[i][0], qf[i][1]);
            mma16816(acc, a1, qf[i][2], qf[i][3]);
          }
          const float2 ka = pk[(m * kKv4Rec + g) * NG + grp], kb = pk[(m * kKv4Rec + g + 8) * NG + grp];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = fmaf(e < 2 ? ka.x : kb.x, acc[e], (e < 2 ? ka.y : kb.y) * qs[grp][e & 1]);
            const float f = cf[grp * NU / NG][e & 1];
            s[m][e] = grp ? fmaf(v, f, s[m][e]) : v * f;
          }
        }
      }
      const bool whole = tile >= full_lo && tile < full_hi;
      if (!whole) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = tile * kTile + m * kKv4Rec + g + (e < 2 ? 0 : 8), pos = col_pos[e & 1];
            const bool seen = t <= pos && t < len && (p.window <= 0 || t > pos - p.window);
            if (!seen) s[m][e] = -INFINITY;
          }
      }
      // ---- the reference exponent is that of p s, so that the weights p s are at most 2^kRoom
      float lg[2][2];  // record, key g or g + 8
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int y = 0; y < 2; ++y) lg[m][y] = pv[(m * kKv4Rec + g + 8 * y) * NG].w;
      // ---- running reference and rescale
      bool grew = false;
      float now[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float m = fmaxf(fmaxf(s[0][e] + lg[0][0], s[0][e + 2] + lg[0][1]),
                        fmaxf(s[1][e] + lg[1][0], s[1][e + 2] + lg[1][1]));
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
        now[e] = fmaxf(m, top[e]);
        grew |= m > top[e];
      }
      if (__any_sync(~0u, grew)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = kv4_exp2(top[e] - (now[e] == -INFINITY ? 0.0f : now[e]));
          top[e] = now[e];
          sum[e] *= f;
#pragma unroll
          for (int k = 0; k < NG; ++k) bias[k][e] *= f;
#pragma unroll
          for (int i = 0; i < NW; ++i)
#pragma unroll
            for (int m = 0; m < 2; ++m) out[i][m][e] *= f, out[i][m][e + 2] *= f;
        }
      }
      float ref[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) ref[e] = top[e] == -INFINITY ? 0.0f : top[e];
      // ---- probabilities, and the products with the values
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint8_t* k = rec + m * REC;
        uint32_t va[NW], vb[NW];  // tokens 0..7 and 8..15 of the record
        if constexpr (D == 128) {
          lds_words<4>(k + 8 * D + lane * 16, va);
          lds_words<4>(k + 8 * D + 512 + lane * 16, vb);
        } else {
          uint32_t v4[4];
          lds_words<4>(k + 8 * D + lane * 16, v4);
          va[0] = v4[0], va[1] = v4[1], vb[0] = v4[2], vb[1] = v4[3];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[m][e] = kv4_exp2(s[m][e] - ref[e & 1]);
          sum[e & 1] += s[m][e];
        }
        uint32_t pf[NG][2];
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          const float4 va4 = pv[(m * kKv4Rec + g) * NG + grp], vb4 = pv[(m * kKv4Rec + g + 8) * NG + grp];
          const float r[2] = {va4.y, vb4.y}, z[2] = {va4.z, vb4.z};
          float x[4], b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = s[m][e] * (e < 2 ? va4.x : vb4.x);
          if (!whole) {  // a key that is not seen may carry NaN parameters
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (s[m][e] == 0.0f) x[e] = 0.0f;
          }
          const uint32_t w01 = Elem<__half>::from_f2(x[0], x[1]), w23 = Elem<__half>::from_f2(x[2], x[3]);
          unpack2<__half>(w01, b[0], b[1]);
          unpack2<__half>(w23, b[2], b[3]);
          if (whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              bias[grp][e & 1] = fmaf(b[e], r[e >> 1], fmaf(s[m][e], z[e >> 1], bias[grp][e & 1]));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (s[m][e] != 0.0f)
                bias[grp][e & 1] = fmaf(b[e], r[e >> 1], fmaf(s[m][e], z[e >> 1], bias[grp][e & 1]));
          }
          pf[grp][0] = movmatrix_trans(w01);
          pf[grp][1] = movmatrix_trans(w23);
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          uint32_t a0[4], a1[4];
          code_pairs(va[i], magic_low, magic_high, a0[0], a0[1], a1[0], a1[1]);
          code_pairs(vb[i], magic_low, magic_high, a0[2], a0[3], a1[2], a1[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a0[e] = sub_f16x2(a0[e], e & 1 ? kCentreHigh : kCentreLow);
            a1[e] = sub_f16x2(a1[e], e & 1 ? kCentreHigh : kCentreLow);
          }
          mma16816(out[i][0], a0, pf[i / WPG][0], pf[i / WPG][1]);
          mma16816(out[i][1], a1, pf[i / WPG][0], pf[i / WPG][1]);
        }
      }
      __syncwarp();  // every lane has read this stage
      copy_next(false);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }

    if (!ok) sum[0] = sum[1] = NAN;
    // ---- the piece's sums over the keys
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        sum[e] += __shfl_xor_sync(~0u, sum[e], o);
#pragma unroll
        for (int k = 0; k < NG; ++k) bias[k][e] += __shfl_xor_sync(~0u, bias[k][e], o);
      }
    float back[NG];  // from the groups' units
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) back[grp] = NG > 1 ? reciprocal_of_power(s_unit[warp][grp]) : 1.0f;
    const bool complete = u == w.item && ue == w.item + w.n_tiles;
    const int slot = ue == run_end;
    float* part = part_at(warp, slot);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = 2 * c + e;
      if (complete) {
        const int row = w.rb * ROWS + col, j = (int)((uint32_t)row / (uint32_t)p.G), h = row - j * p.G;
        const float inv = sum[e] > 0.0f ? 1.0f / sum[e] : sum[e];  // nothing seen: zeros; NaN stays
        uint16_t* o = p.out + (int64_t)(w.req.start + j) * p.o_t + (int64_t)(w.kvh * p.G + h) * D + 4 * g;
        if (j < w.req.n) {
#pragma unroll
          for (int i = 0; i < NW; ++i) {
            const float b = bias[i / WPG][e], f = inv * back[i / WPG];
            uint2 v;
            v.x = Elem<T>::from_f2((out[i][0][e] + b) * f, (out[i][0][e + 2] + b) * f);
            v.y = Elem<T>::from_f2((out[i][1][e] + b) * f, (out[i][1][e + 2] + b) * f);
            *reinterpret_cast<uint2*>(o + 32 * i) = v;
          }
        }
      } else {
        if (g == 0) {
          s_max[warp][slot][col] = top[e];
          s_sum[warp][slot][col] = sum[e];
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const float b = bias[i / WPG][e], f = back[i / WPG];
          *reinterpret_cast<float4*>(part + col * (D + 4) + 32 * i + 4 * g) =
              make_float4((out[i][0][e] + b) * f, (out[i][0][e + 2] + b) * f, (out[i][1][e] + b) * f,
                          (out[i][1][e + 2] + b) * f);
        }
      }
    }
    if (!complete && lane == 0)
      s_info[warp][slot] = PartInfo{w.item, w.n_tiles, w.rb * ROWS, w.req.start, w.req.n, w.kvh * p.G};
    u = ue;
    if (u < run_end) {
      Work x = w;
      __syncwarp();
      x.next(p);  // (where lengths changed under the kernel and none is left, the tiles copied are still consumed)
      if (lane == 0) s_item[warp] = x;
      __syncwarp();
    }
  }

  // ---- join the warps' parts, item by item: four dims of one column per thread
  __syncthreads();
  const Work& any = s_item[0];
  constexpr int SLOT = ROWS * (D + 2);
  const auto store = [&](const PartInfo& x, int col, int dim, float4 v, float l) {
    const int row = x.row0 + col, j = (int)((uint32_t)row / (uint32_t)p.G), h = row - j * p.G;
    if (j >= x.n) return;
    const float inv = l > 0.0f ? 1.0f / l : l;
    uint2 o;
    o.x = Elem<T>::from_f2(v.x * inv, v.y * inv);
    o.y = Elem<T>::from_f2(v.z * inv, v.w * inv);
    *reinterpret_cast<uint2*>(p.out + (int64_t)(x.start + j) * p.o_t + (int64_t)(x.head0 + h) * D + dim) = o;
  };
  // Lane e looks after entry e = warp * 2 + slot; the entries of one item are one ballot.
  const long long entry = lane < 2 * WARPS ? s_info[lane >> 1][lane & 1].item : -1;
  int shared_at[2] = {-1, -1};  // an entry of each item shared with other CTAs
  for (uint32_t left = __ballot_sync(~0u, entry >= 0); left;) {
    const int x = __ffs(left) - 1;
    const uint32_t mine = __ballot_sync(~0u, entry == __shfl_sync(~0u, entry, x)) & left;
    left &= ~mine;
    const PartInfo& info = s_info[x >> 1][x & 1];
    const bool here = info.item >= any.u0 && info.item + info.n_tiles <= any.u1;
    const int side = info.item < any.u0 ? 0 : 1;
    if (!here) shared_at[side] = x;
    float* part = p.partial + (int64_t)(2 * (int)blockIdx.x + side) * SLOT;
    for (int k = tid; k < ROWS * D / 4; k += THREADS) {
      const int col = k / (D / 4), dim = k % (D / 4) * 4;
      float m = -INFINITY, l = 0.0f;
      for (uint32_t z = mine; z; z &= z - 1) {
        const int e = __ffs(z) - 1;
        m = fmaxf(m, s_max[e >> 1][e & 1][col]);
      }
      const float to = m == -INFINITY ? 0.0f : m;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (uint32_t z = mine; z; z &= z - 1) {
        const int e = __ffs(z) - 1;
        const float f = kv4_exp2(s_max[e >> 1][e & 1][col] - to);
        const float4 o = *reinterpret_cast<const float4*>(part_at(e >> 1, e & 1) + col * (D + 4) + dim);
        l = fmaf(s_sum[e >> 1][e & 1][col], f, l);
        v.x = fmaf(o.x, f, v.x), v.y = fmaf(o.y, f, v.y), v.z = fmaf(o.z, f, v.z), v.w = fmaf(o.w, f, v.w);
      }
      if (here) {
        store(info, col, dim, v, l);
      } else {
        if (dim == 0) {
          part[col] = m;
          part[ROWS + col] = l;
        }
        *reinterpret_cast<float4*>(part + 2 * ROWS + col * D + dim) = v;
      }
    }
  }
  if (shared_at[0] < 0 && shared_at[1] < 0) return;

  // ---- items shared with other CTAs: the last to arrive adds the parts, in the order of the CTAs
  __threadfence();
  __syncthreads();
  if (tid < 2 && shared_at[tid] >= 0) {
    const PartInfo& info = s_info[shared_at[tid] >> 1][shared_at[tid] & 1];
    const int fc = any.owner(info.item), lc = any.owner(info.item + info.n_tiles - 1);
    const bool last = atomicAdd(p.counters + fc, 1) == lc - fc;
    if (last) p.counters[fc] = 0;
    s_last[tid] = last;
  }
  __syncthreads();
  for (int side = 0; side < 2; ++side) {
    if (shared_at[side] < 0 || !s_last[side]) continue;
    __threadfence();
    const PartInfo& info = s_info[shared_at[side] >> 1][shared_at[side] & 1];
    const int fc = any.owner(info.item), lc = any.owner(info.item + info.n_tiles - 1);
    const auto slot = [&](int x) { return p.partial + (int64_t)(2 * x + (x == fc ? 1 : 0)) * SLOT; };
    for (int k = tid; k < ROWS * D / 4; k += THREADS) {
      const int col = k / (D / 4), dim = k % (D / 4) * 4;
      float m = -INFINITY, l = 0.0f;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      // Eight parts at a time: their loads are in flight together.
      for (int x0 = fc; x0 <= lc; x0 += 8) {
        float pm[8], pl[8];
        float4 po[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const float* q = slot(min(x0 + y, lc));
          pm[y] = x0 + y <= lc ? __ldcg(q + col) : -INFINITY;
          pl[y] = __ldcg(q + ROWS + col);
          po[y] = __ldcg(reinterpret_cast<const float4*>(q + 2 * ROWS + col * D + dim));
        }
        float to = m;
#pragma unroll
        for (int y = 0; y < 8; ++y) to = fmaxf(to, pm[y]);
        const float at = to == -INFINITY ? 0.0f : to;
        const float old = kv4_exp2(m - at);
        l *= old, v.x *= old, v.y *= old, v.z *= old, v.w *= old;
        m = to;
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const float f = kv4_exp2(pm[y] - at);
          if (x0 + y > lc) continue;
          l = fmaf(pl[y], f, l);
          v.x = fmaf(po[y].x, f, v.x), v.y = fmaf(po[y].y, f, v.y);
          v.z = fmaf(po[y].z, f, v.z), v.w = fmaf(po[y].w, f, v.w);
        }
      }
      store(info, col, dim, v, l);
    }
  }
}

template <typename T, int D, int NG>
cudaError_t launch_one(const Kv4AttnParams& p, int sms, bool pdl, cudaStream_t stream) {
  constexpr int smem = smem_bytes<D, NG>();
  const auto kernel = kv4_attn_split_kernel<T, D, NG>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  const int grid = 2 * sms < kKv4MaxGrid ? 2 * sms : kKv4MaxGrid;
  return kv4_launch(kernel, dim3((unsigned)grid), warps<D, NG>() * 32, smem, pdl, stream, p);
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

int64_t kv4_split_partial_bytes(int D) { return (int64_t)2 * kKv4MaxGrid * kRows * (D + 2) * 4; }

cudaError_t launch_kv4_attn_split(const Kv4AttnParams& p, int sms, bool bf16, bool pdl, cudaStream_t stream) {
  return bf16 ? launch_t<__nv_bfloat16>(p, sms, pdl, stream) : launch_t<__half>(p, sms, pdl, stream);
}

}  // namespace fqkv
