// fqkv_kv4_attn.cu -- causal attention over the paged 4-bit cache for few query rows per KV
// head (single tokens, drafts): split over the key axis, one pass over the codes.
//
// Mathematics.  A code c stands for s c + m, with s and m per token and group of dims, so
//   q . k_t = sum_groups ( s_tg * (q_g . c_tg) + m_tg * sum(q_g) )
//   sum_t p_t v_t = sum_t (p_t s_tg) (c_tg - 8) + sum_t p_t (m_tg + 8 s_tg).
// The tensor cores multiply the small integers, exact in 16 bits, and the parameters meet the
// scores and the probabilities in fp32: no dequantised tile is ever formed.  An integer becomes
// a 16-bit float by placing its four bits in the mantissa of a constant (128 + c in bf16,
// 64 + c in fp16): one shift and one three-input logic operation per two codes.  For the keys
// the constant is taken back by starting the accumulator at -constant * sum(q_g); for the values
// it is subtracted, and the codes centred, with one packed subtraction, so that the sum over a
// long context does not cancel a large offset.  p s is rounded to 16 bits for the product (the
// one rounding to fewer than 32 bits besides the output); maxima, sums and outputs are fp32.
//
// Shape.  Both products are transposed (keys x queries and dims x queries, m16n8k16), so the
// query heads that share a KV head fill the 8-wide side and 1 to 8 query rows cost the same.
// A record's bytes are stored in fragment order: a warp's 16-byte shared loads are conflict
// free and need no transposition (the values' tokens are interleaved in pairs).
//
// Bound: the codes' bytes over HBM.  Per 16 tokens and KV head that is 2176 bytes at D = 128
// (one group), about 90 cycles of an SM's share of the bandwidth, against about 50 cycles of
// issue slots for the unpacking, the products and the softmax.
//
// Split.  The items (request, KV head, block of query rows) are laid end to end as tiles of 32
// tokens and cut into equal runs, one per CTA, whatever the lengths; inside a CTA each warp
// takes a contiguous part of a piece with a ring of its own, filled by bulk copies of whole
// records.  An item cut between CTAs is joined by the CTA that arrives last, which adds the
// parts in the order of the CTAs, so the result does not depend on the arrival order.
#include "fqkv_kv4.cuh"

namespace fqkv {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;    // tokens per ring stage (two records)
constexpr int kStages = 2;
constexpr int kMinTiles = 8;  // a CTA gets at least one tile per warp before the work is cut finer

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

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Nibbles j and j + 4 of w (bits 4 j and 16 + 4 j) as a pair of 16-bit floats offset() + code.
template <typename T>
struct Nib;
template <>
struct Nib<__nv_bfloat16> {
  static constexpr float kOffset = 128.0f;  // 0x4300: four mantissa bits of weight 1..8
  static constexpr float kMinNormal = 1e-30f;
  static constexpr uint32_t kCentre = 0x43084308u;  // 136 = offset + 8
  template <int j>
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    return ((w >> (4 * j)) & 0x000F000Fu) | 0x43004300u;
  }
  static __device__ __forceinline__ uint32_t centred(uint32_t x) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(kCentre));
    return r;
  }
};
template <>
struct Nib<__half> {
  static constexpr float kOffset = 64.0f;  // 0x5400: mantissa bits 4..7 have weight 1..8
  static constexpr float kMinNormal = 6.2e-5f;
  static constexpr uint32_t kCentre = 0x54805480u;  // 72 = offset + 8
  template <int j>
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    const uint32_t x = j == 0 ? w << 4 : w >> (4 * (j > 0 ? j - 1 : 0));
    return (x & 0x00F000F0u) | 0x54005400u;
  }
  static __device__ __forceinline__ uint32_t centred(uint32_t x) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(kCentre));
    return r;
  }
};

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  lo = Elem<T>::to_f((uint16_t)w);
  hi = Elem<T>::to_f((uint16_t)(w >> 16));
}

// a / b by an approximate reciprocal and one step of refinement; exact where the quotient is a
// small integer.  Not meaningful for b = 0 or subnormal.
__device__ __forceinline__ float quotient(float a, float b) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(b));
  const float q = a * r;
  return fmaf(fmaf(-q, b, a), r, q);
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

// One request as the kernel sees it: lengths clamped to what the tables and q hold.
struct Request {
  int start, n, len;  // first token, queries, keys
};

__device__ __forceinline__ Request load_request(const Kv4AttnParams& p, int r) {
  Request q;
  int64_t a, b;
  if (p.query_start) {
    a = p.query_start[r];
    b = p.query_start[r + 1];
  } else {
    a = (int64_t)r * p.S;
    b = a + p.S;
  }
  const int64_t a0 = a, b0 = b;
  a = a < 0 ? 0 : a > p.T ? p.T : a;
  b = b < a ? a : b > p.T ? p.T : b;
  const int len0 = p.seq_lens[r];
  const int64_t cap = (int64_t)p.width * p.c.P;
  q.len = len0 < 0 ? 0 : len0 > cap ? (int)cap : len0;
  q.start = (int)a;
  q.n = (int)(b - a);
  if (a != a0 || b != b0 || q.len != len0) record_status(FQKV_STATUS_BAD_INDEX);
  return q;
}

// Row block rb of a request: query rows [rb * ROWS, ...) of n * G rows (row = j * G + head).
template <int ROWS>
__device__ __forceinline__ void block_tiles(const Kv4AttnParams& p, const Request& q, int rb, int& tile_lo,
                                            int& n_tiles) {
  const int j0 = rb * ROWS / p.G, j1 = min((rb * ROWS + ROWS - 1) / p.G, q.n - 1);
  const int hi = max(0, min(q.len, q.len - q.n + j1 + 1));
  const int lo = p.window > 0 ? max(0, q.len - q.n + j0 - p.window + 1) : 0;
  tile_lo = lo / kTile;
  n_tiles = max(1, (hi + kTile - 1) / kTile - tile_lo);
}

template <int ROWS>
__device__ __forceinline__ long long request_tiles(const Kv4AttnParams& p, const Request& q) {
  const int blocks = (q.n * p.G + ROWS - 1) / ROWS;
  long long sum = 0;
  for (int rb = 0; rb < blocks; ++rb) {
    int lo, n;
    block_tiles<ROWS>(p, q, rb, lo, n);
    sum += n;
  }
  return sum * p.c.n_kv;
}

template <int D, int NG, int NT>
constexpr int ring_bytes() {
  return kWarps * kStages * 2 * kv4_record_bytes(D, NG);
}
// Per-column maxima and sums of the warps, and half of the warps' outputs for the tree sum.
template <int D, int NG, int NT>
constexpr int smem_bytes() {
  return ring_bytes<D, NG, NT>() + kWarps / 2 * 8 * NT * D * 4;
}

template <typename T, int D, int NG, int NT>
__global__ void __launch_bounds__(kThreads, 2) kv4_attn_split_kernel(const Kv4AttnParams p) {
  constexpr int ROWS = 8 * NT;           // query rows of an item
  constexpr int REC = kv4_record_bytes(D, NG);
  constexpr int NW = D / 32;             // 32-dim blocks: words per lane and key row
  constexpr int WPG = NW / NG;           // words of one scale group
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_bar[kWarps][kStages];
  __shared__ long long s_scan[kWarps];
  __shared__ long long s_found;
  __shared__ int s_r, s_last;
  __shared__ float s_max[kWarps][ROWS], s_sum[kWarps][ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * kStages * 2 * REC;
  float* s_out = reinterpret_cast<float*>(smem + ring_bytes<D, NG, NT>());
  if (tid < kWarps * kStages) mbar_init(&s_bar[tid / kStages][tid % kStages], 1);
  if (tid == 0) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  // ---- total work, and this CTA's run of tiles [u0, u1)
  long long mine = 0;
  for (int r = tid; r < p.R; r += kThreads) mine += request_tiles<ROWS>(p, load_request(p, r));
  long long total = mine;
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
  if (lane == 0) s_scan[warp] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += s_scan[w];
  const long long ctas = max(1ll, min((long long)gridDim.x, total / kMinTiles));
  const long long cta = blockIdx.x;
  if (cta >= ctas || total == 0) return;
  const long long u0 = cta * total / ctas, u1 = (cta + 1) * total / ctas;

  // ---- the request that holds tile u0
  long long base = 0;
  for (int r0 = 0; r0 < p.R; r0 += kThreads) {
    const int r = r0 + tid;
    const long long n = r0 == 0 && p.R <= kThreads ? mine
                        : r < p.R                  ? request_tiles<ROWS>(p, load_request(p, r))
                                                   : 0;
    long long v = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(~0u, v, o);
      if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = v;
    __syncthreads();
    long long before = base;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_scan[w];
      base += s_scan[w];
    }
    if (before + v - n <= u0 && u0 < before + v) {
      s_r = r;
      s_found = before + v - n;
    }
    if (base > u0) break;
  }
  __syncthreads();

  int r = s_r;
  Request req = load_request(p, r);
  int blocks = (req.n * p.G + ROWS - 1) / ROWS;
  int kvh = 0, rb = 0, tile_lo = 0, n_tiles = 0;
  long long item = s_found;  // first tile of the current item
  {
    const long long per_head = request_tiles<ROWS>(p, req) / p.c.n_kv;
    kvh = (int)((u0 - item) / per_head);
    item += kvh * per_head;
    for (;; ++rb) {
      block_tiles<ROWS>(p, req, rb, tile_lo, n_tiles);
      if (u0 < item + n_tiles) break;
      item += n_tiles;
    }
  }

  uint32_t parity = 0;  // bit s: phase of ring stage s
  for (long long u = u0; u < u1;) {
    // ---- one piece: tiles [u, ue) of item (r, kvh, rb); this warp's part [wt, we) of its tiles
    const long long ue = min(u1, item + n_tiles);
    const int piece = (int)(ue - u);
    const int wt = tile_lo + (int)(u - item) + (int)((long long)piece * warp / kWarps);
    const int we = tile_lo + (int)(u - item) + (int)((long long)piece * (warp + 1) / kWarps);
    const int pos0 = req.len - req.n;  // position of query 0

    // Record addresses: lane L holds record 2 * wt_base + L of the warp's tiles, 16 tiles at a time.
    const int* table = p.table + (int64_t)r * p.table_stride;
    const int n_rec = (req.len + kKv4Rec - 1) / kKv4Rec;
    const int rpb = p.c.P / kKv4Rec;
    const auto address = [&](int rec) -> const uint8_t* {
      if (rec >= n_rec) return nullptr;
      const int nth = rec / rpb;
      int block = table[nth];
      if (block < 0 || block >= p.c.n_blocks) {
        record_status(FQKV_STATUS_BAD_INDEX);
        block = 0;
      }
      return p.c.data + (((int64_t)block * p.c.n_kv + kvh) * rpb + (rec - nth * rpb)) * REC;
    };
    const uint8_t* src = address(2 * wt + lane);
    const uint8_t* src_next = address(2 * wt + 32 + lane);
    int src_tile = wt;  // src covers tiles [src_tile, src_tile + 16)
    const auto issue = [&](int tile, int stage) {
      if (tile - src_tile >= 16) {
        src = src_next;
        src_tile += 16;
        src_next = address(2 * (src_tile + 16) + lane);
      }
      const int k = lane - 2 * (tile - src_tile);  // 0, 1: the lanes that hold this tile's records
      const bool mine_rec = (k == 0 || k == 1) && src != nullptr;
      const uint32_t have = __popc(__ballot_sync(~0u, mine_rec));
      if (lane == 0) mbar_arrive_expect_tx(&s_bar[warp][stage], have * REC);
      __syncwarp();
      if (mine_rec) bulk_load(smem_u32(ring + (stage * 2 + k) * REC), src, REC, &s_bar[warp][stage]);
    };
#pragma unroll
    for (int s = 0; s < kStages; ++s)
      if (wt + s < we) issue(wt + s, s);

    // ---- queries: this lane's fragments (row g of each 8) and the sums of its columns' rows
    uint32_t qf[NT][NW][4];
    float qs[NT][NG][2];
    int col_pos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = rb * ROWS + nt * 8 + g;
      const int j = row / p.G, h = row - j * p.G;
      const bool live = j < req.n;
      const uint16_t* qrow = p.q + (p.query_start ? (int64_t)(req.start + j) * p.q_t : r * p.q_r + j * p.q_t) +
                             (int64_t)(kvh * p.G + h) * p.q_h;
      float sum[NG] = {};
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (live) v = *reinterpret_cast<const uint4*>(qrow + 8 * (4 * i + c));
        qf[nt][i][0] = v.x, qf[nt][i][1] = v.y, qf[nt][i][2] = v.z, qf[nt][i][3] = v.w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float a, b;
          unpack2<T>(qf[nt][i][e], a, b);
          sum[i / WPG] += a + b;
        }
      }
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        sum[k] += __shfl_xor_sync(~0u, sum[k], 1);
        sum[k] += __shfl_xor_sync(~0u, sum[k], 2);
        qs[nt][k][0] = __shfl_sync(~0u, sum[k], 8 * c);
        qs[nt][k][1] = __shfl_sync(~0u, sum[k], 8 * c + 4);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) col_pos[nt][e] = pos0 + (rb * ROWS + nt * 8 + 2 * c + e) / p.G;
    }
    // Tiles in [full_lo, full_hi) are visible to every row of the block.
    const int last_j = min((rb * ROWS + ROWS - 1) / p.G, req.n - 1);
    const int full_hi = (max(0, pos0 + rb * ROWS / p.G + 1)) / kTile;
    const int full_lo = p.window > 0 ? (max(0, pos0 + last_j - p.window + 1) + kTile - 1) / kTile : 0;

    float out[NW][2][NT][4];
    float top[NT][2], sum[NT][2], bias[NT][NG][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) out[i][m][nt][e] = 0.0f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[nt][e] = -INFINITY;
        sum[nt][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < NG; ++k) bias[nt][k][e] = 0.0f;
      }
    }

    int stage = 0;
    for (int tile = wt; tile < we; ++tile) {
      mbar_wait(&s_bar[warp][stage], (parity >> stage) & 1u);
      parity ^= 1u << stage;
      const uint8_t* rec = ring + stage * 2 * REC;
      // ---- scores, in units of log2: s[record][nt][key g: cols, key g + 8: cols]
      float s[2][NT][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint8_t* k = rec + m * REC;
        uint32_t wa[NW], wb[NW], pa[NG], pb[NG];
        lds_words<NW>(k + g * (D / 2) + c * (D / 8), wa);
        lds_words<NW>(k + (g + 8) * (D / 2) + c * (D / 8), wb);
        lds_words<NG>(k + 16 * D + g * NG * 4, pa);
        lds_words<NG>(k + 16 * D + (g + 8) * NG * 4, pb);
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][e] = -Nib<T>::kOffset * qs[nt][grp][e & 1];
#pragma unroll
          for (int i = grp * WPG; i < (grp + 1) * WPG; ++i) {
            const uint32_t a0[4] = {Nib<T>::template pair<0>(wa[i]), Nib<T>::template pair<0>(wb[i]),
                                    Nib<T>::template pair<1>(wa[i]), Nib<T>::template pair<1>(wb[i])};
            const uint32_t a1[4] = {Nib<T>::template pair<2>(wa[i]), Nib<T>::template pair<2>(wb[i]),
                                    Nib<T>::template pair<3>(wa[i]), Nib<T>::template pair<3>(wb[i])};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<T>(acc[nt], a0, qf[nt][i][0], qf[nt][i][1]);
              mma16816<T>(acc[nt], a1, qf[nt][i][2], qf[nt][i][3]);
            }
          }
          float sa, ma, sb, mb;
          unpack2<T>(pa[grp], sa, ma);
          unpack2<T>(pb[grp], sb, mb);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = fmaf(e < 2 ? sa : sb, acc[nt][e], (e < 2 ? ma : mb) * qs[nt][grp][e & 1]);
              s[m][nt][e] = grp ? s[m][nt][e] + v : v;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][nt][e] *= p.scale_log2;
      }
      const bool whole = tile >= full_lo && tile < full_hi;
      if (!whole) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = tile * kTile + m * kKv4Rec + g + (e < 2 ? 0 : 8), pos = col_pos[nt][e & 1];
              const bool seen = t <= pos && t < req.len && (p.window <= 0 || t > pos - p.window);
              if (!seen) s[m][nt][e] = -INFINITY;
            }
      }
      // ---- running maximum and rescale
      float scale_old[NT][2], ref[NT][2];
      bool grew = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
          m = fmaxf(m, top[nt][e]);
          grew |= m > top[nt][e];
          ref[nt][e] = m == -INFINITY ? 0.0f : m;
          scale_old[nt][e] = exp2f(top[nt][e] - ref[nt][e]);
          top[nt][e] = m;
        }
      if (__any_sync(~0u, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sum[nt][e] *= scale_old[nt][e];
#pragma unroll
            for (int k = 0; k < NG; ++k) bias[nt][k][e] *= scale_old[nt][e];
          }
#pragma unroll
          for (int i = 0; i < NW; ++i)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int e = 0; e < 4; ++e) out[i][m][nt][e] *= scale_old[nt][e & 1];
        }
      }
      // ---- probabilities, and the products with the values
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint8_t* k = rec + m * REC;
        uint32_t pa[NG], pb[NG];
        lds_words<NG>(k + 16 * D + 64 * NG + g * NG * 4, pa);
        lds_words<NG>(k + 16 * D + 64 * NG + (g + 8) * NG * 4, pb);
        uint32_t va[NW], vb[NW];  // tokens 0..7 and 8..15 of the record
        if constexpr (D == 128) {
          lds_words<4>(k + 8 * D + lane * 16, va);
          lds_words<4>(k + 8 * D + 512 + lane * 16, vb);
        } else {
          uint32_t v4[4];
          lds_words<4>(k + 8 * D + lane * 16, v4);
          va[0] = v4[0], va[1] = v4[1], vb[0] = v4[2], vb[1] = v4[3];
        }
        uint32_t pf[NT][NG][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pr[e] = exp2f(s[m][nt][e] - ref[nt][e & 1]);
            sum[nt][e & 1] += pr[e];
          }
#pragma unroll
          for (int grp = 0; grp < NG; ++grp) {
            float sa, ma, sb, mb;
            unpack2<T>(pa[grp], sa, ma);
            unpack2<T>(pb[grp], sb, mb);
            // (m + 8 s) / s: the offset part is formed from the rounded weight, so that both
            // parts of p v carry the same rounding and a value near zero keeps a small error.
            // A weight below the type's normal range (or a scale of zero) says nothing about p.
            const float ra = quotient(ma, sa) + 8.0f, rb = quotient(mb, sb) + 8.0f;
            const float ca = fmaf(8.0f, sa, ma), cb = fmaf(8.0f, sb, mb);
            float w[4], b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = pr[e] * (e < 2 ? sa : sb);
              // A key that is not seen may carry a NaN or an infinity as its parameters.
              if (!whole && s[m][nt][e] == -INFINITY) w[e] = 0.0f;
            }
            const uint32_t w01 = Elem<T>::from_f2(w[0], w[1]), w23 = Elem<T>::from_f2(w[2], w[3]);
            unpack2<T>(w01, b[0], b[1]);
            unpack2<T>(w23, b[2], b[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              b[e] = w[e] < Nib<T>::kMinNormal ? pr[e] * (e < 2 ? ca : cb) : b[e] * (e < 2 ? ra : rb);
              if (!whole && s[m][nt][e] == -INFINITY) b[e] = 0.0f;
            }
            bias[nt][grp][0] += b[0] + b[2];
            bias[nt][grp][1] += b[1] + b[3];
            pf[nt][grp][0] = movmatrix_trans(w01);
            pf[nt][grp][1] = movmatrix_trans(w23);
          }
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const uint32_t a0[4] = {Nib<T>::centred(Nib<T>::template pair<0>(va[i])),
                                  Nib<T>::centred(Nib<T>::template pair<1>(va[i])),
                                  Nib<T>::centred(Nib<T>::template pair<0>(vb[i])),
                                  Nib<T>::centred(Nib<T>::template pair<1>(vb[i]))};
          const uint32_t a1[4] = {Nib<T>::centred(Nib<T>::template pair<2>(va[i])),
                                  Nib<T>::centred(Nib<T>::template pair<3>(va[i])),
                                  Nib<T>::centred(Nib<T>::template pair<2>(vb[i])),
                                  Nib<T>::centred(Nib<T>::template pair<3>(vb[i]))};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816<T>(out[i][0][nt], a0, pf[nt][i / WPG][0], pf[nt][i / WPG][1]);
            mma16816<T>(out[i][1][nt], a1, pf[nt][i / WPG][0], pf[nt][i / WPG][1]);
          }
        }
      }
      __syncwarp();  // every lane has read this stage
      if (tile + kStages < we) issue(tile + kStages, stage);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }

    // ---- join the warps: maxima and sums through shared memory, outputs by a tree
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          sum[nt][e] += __shfl_xor_sync(~0u, sum[nt][e], o);
#pragma unroll
          for (int k = 0; k < NG; ++k) bias[nt][k][e] += __shfl_xor_sync(~0u, bias[nt][k][e], o);
        }
        if (g == 0) {
          s_max[warp][nt * 8 + 2 * c + e] = top[nt][e];
          s_sum[warp][nt * 8 + 2 * c + e] = sum[nt][e];
        }
      }
    __syncthreads();
    float all_top[NT][2], all_sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = nt * 8 + 2 * c + e;
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_max[w][col]);
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) l += s_sum[w][col] * exp2f(s_max[w][col] - ref);
        all_top[nt][e] = m;
        all_sum[nt][e] = l;
        const float f = exp2f(top[nt][e] - ref);
#pragma unroll
        for (int i = 0; i < NW; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            out[i][x][nt][e] = (out[i][x][nt][e] + bias[nt][i / WPG][e]) * f;
            out[i][x][nt][e + 2] = (out[i][x][nt][e + 2] + bias[nt][i / WPG][e]) * f;
          }
      }
    constexpr int PER = NW * 2 * NT * 4;  // outputs per lane
    float* flat = &out[0][0][0][0];
#pragma unroll
    for (int half = kWarps / 2; half >= 1; half >>= 1) {
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int k = 0; k < PER; ++k) s_out[((warp - half) * PER + k) * 32 + lane] = flat[k];
      }
      __syncthreads();
      if (warp < half) {
#pragma unroll
        for (int k = 0; k < PER; ++k) flat[k] += s_out[(warp * PER + k) * 32 + lane];
      }
      __syncthreads();
    }

    // ---- write the item, or this CTA's part of it
    const auto store = [&](int row, int dim, const float (&v)[4], float l) {
      const int j = row / p.G, h = row - j * p.G;
      if (j >= req.n) return;
      const float inv = l > 0.0f ? 1.0f / l : l;  // nothing seen: zeros; NaN stays
      uint2 o;
      o.x = Elem<T>::from_f2(v[0] * inv, v[1] * inv);
      o.y = Elem<T>::from_f2(v[2] * inv, v[3] * inv);
      *reinterpret_cast<uint2*>(p.out + (int64_t)(req.start + j) * p.o_t + (int64_t)(kvh * p.G + h) * D + dim) = o;
    };
    const bool complete = u == item && ue == item + n_tiles;
    if (complete) {
      if (warp == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < NW; ++i) {
              const float v[4] = {out[i][0][nt][e], out[i][0][nt][e + 2], out[i][1][nt][e], out[i][1][nt][e + 2]};
              store(rb * ROWS + nt * 8 + 2 * c + e, 32 * i + 4 * g, v, all_sum[nt][e]);
            }
      }
    } else {
      constexpr int SLOT = ROWS * (D + 2);
      const long long first = ((item + 1) * ctas - 1) / total;
      const long long last = ((item + n_tiles) * ctas - 1) / total;
      float* part = p.partial + (2 * cta + (item < u0 ? 0 : 1)) * SLOT;
      if (warp == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int col = nt * 8 + 2 * c + e;
            if (g == 0) {
              part[col] = all_top[nt][e];
              part[ROWS + col] = all_sum[nt][e];
            }
#pragma unroll
            for (int i = 0; i < NW; ++i)
              *reinterpret_cast<float4*>(part + 2 * ROWS + col * D + 32 * i + 4 * g) =
                  make_float4(out[i][0][nt][e], out[i][0][nt][e + 2], out[i][1][nt][e], out[i][1][nt][e + 2]);
          }
        __threadfence();
        __syncwarp();
        if (lane == 0) s_last = atomicAdd(p.counters + first, 1) == (int)(last - first);
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        // Four dims of one column per thread; the parts in the order of the CTAs.
        for (int k = tid; k < ROWS * D / 4; k += kThreads) {
          const int col = k / (D / 4), dim = (k % (D / 4)) * 4;
          float m = -INFINITY, l = 0.0f;
          for (long long x = first; x <= last; ++x)
            m = fmaxf(m, __ldcg(p.partial + (2 * x + (x == first ? 1 : 0)) * SLOT + col));
          const float ref = m == -INFINITY ? 0.0f : m;
          float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
          for (long long x = first; x <= last; ++x) {
            const float* q = p.partial + (2 * x + (x == first ? 1 : 0)) * SLOT;
            const float f = exp2f(__ldcg(q + col) - ref);
            l += __ldcg(q + ROWS + col) * f;
            const float4 o = __ldcg(reinterpret_cast<const float4*>(q + 2 * ROWS + col * D + dim));
            v[0] += o.x * f, v[1] += o.y * f, v[2] += o.z * f, v[3] += o.w * f;
          }
          store(rb * ROWS + col, dim, v, l);
        }
        if (tid == 0) p.counters[first] = 0;
      }
      __syncthreads();  // s_last is written again by the next piece
    }

    // ---- next item
    u = ue;
    if (u >= u1) break;
    item += n_tiles;
    if (++rb == blocks) {
      rb = 0;
      if (++kvh == p.c.n_kv) {
        kvh = 0;
        blocks = 0;
        while (blocks == 0 && ++r < p.R) {
          req = load_request(p, r);
          blocks = (req.n * p.G + ROWS - 1) / ROWS;
        }
        if (blocks == 0) break;  // lengths that changed under the kernel
      }
    }
    block_tiles<ROWS>(p, req, rb, tile_lo, n_tiles);
  }
}

template <typename T, int D, int NG, int NT>
cudaError_t launch_one(const Kv4AttnParams& p, int sms, bool pdl, cudaStream_t stream) {
  constexpr int smem = smem_bytes<D, NG, NT>();
  const auto kernel = kv4_attn_split_kernel<T, D, NG, NT>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  const int grid = sms * 2 < kKv4MaxGrid ? sms * 2 : kKv4MaxGrid;
  return kv4_launch(kernel, dim3((unsigned)grid), kThreads, smem, pdl, stream, p);
}

template <typename T, int NT>
cudaError_t launch_nt(const Kv4AttnParams& p, int sms, bool pdl, cudaStream_t stream) {
  const int ng = p.c.D / p.c.group;
  if (p.c.D == 128) {
    if (ng == 1) return launch_one<T, 128, 1, NT>(p, sms, pdl, stream);
    if (ng == 2) return launch_one<T, 128, 2, NT>(p, sms, pdl, stream);
    return launch_one<T, 128, 4, NT>(p, sms, pdl, stream);
  }
  if (ng == 1) return launch_one<T, 64, 1, NT>(p, sms, pdl, stream);
  return launch_one<T, 64, 2, NT>(p, sms, pdl, stream);
}

}  // namespace

cudaError_t launch_kv4_attn_split(const Kv4AttnParams& p, int row_blocks8, int sms, bool bf16, bool pdl,
                                  cudaStream_t stream) {
  if (row_blocks8 == 1)
    return bf16 ? launch_nt<__nv_bfloat16, 1>(p, sms, pdl, stream) : launch_nt<__half, 1>(p, sms, pdl, stream);
  return bf16 ? launch_nt<__nv_bfloat16, 2>(p, sms, pdl, stream) : launch_nt<__half, 2>(p, sms, pdl, stream);
}

}  // namespace fqkv
