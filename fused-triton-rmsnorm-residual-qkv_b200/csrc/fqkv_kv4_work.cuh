// fqkv_kv4_work.cuh -- how the attention kernels of the 4-bit cache cut a ragged batch into
// equal runs.  Items (request, KV head, block of ROWS query rows) are laid end to end as tiles
// of TILE tokens and cut into one contiguous run per CTA, whatever the lengths.  A CTA's part of
// an item is a piece; items cut between CTAs are joined through the workspace by the CTA that
// arrives last, in the order of the CTAs.
#pragma once

#include "fqkv_kv4.cuh"

namespace fqkv {

// One request as the kernels see it: lengths clamped to what the tables and q hold.
struct Kv4Request {
  int start, n, len;  // first token, queries, keys
};

__device__ __forceinline__ Kv4Request kv4_load_request(const Kv4AttnParams& p, int r) {
  Kv4Request q;
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

template <int ROWS, int TILE, int THREADS>
struct Kv4Work {
  struct Shared {
    long long scan[THREADS / 32];
    long long found;
    int r;
  };

  long long total, ctas, u0, u1;  // all tiles, CTAs that have work, this CTA's run
  // The current item: request r, KV head, row block; its tiles [tile_lo, tile_lo + n_tiles), the
  // first of which is tile `item` of the batch; row blocks of the request.
  Kv4Request req;
  long long item;
  int r, kvh, rb, blocks, tile_lo, n_tiles;

  // Tiles that row block rb of a request reads (at least one, so that every item is visited).
  // Rows are (query j, head) with row = j * G + head.
  static __device__ __forceinline__ void block_tiles(const Kv4AttnParams& p, const Kv4Request& q, int rb, int& tile_lo,
                                                     int& n_tiles) {
    const int j0 = rb * ROWS / p.G, j1 = min((rb * ROWS + ROWS - 1) / p.G, q.n - 1);
    const int hi = max(0, min(q.len, q.len - q.n + j1 + 1));
    const int lo = p.window > 0 ? max(0, q.len - q.n + j0 - p.window + 1) : 0;
    tile_lo = lo / TILE;
    n_tiles = max(1, (hi + TILE - 1) / TILE - tile_lo);
  }

  static __device__ __forceinline__ int row_blocks(const Kv4AttnParams& p, const Kv4Request& q) {
    return (q.n * p.G + ROWS - 1) / ROWS;
  }

  static __device__ __forceinline__ long long head_tiles(const Kv4AttnParams& p, const Kv4Request& q) {
    const int n = row_blocks(p, q);
    long long sum = 0;
    for (int rb = 0; rb < n; ++rb) {
      int lo, tiles;
      block_tiles(p, q, rb, lo, tiles);
      sum += tiles;
    }
    return sum;
  }

  // Called by the whole block.  False: this CTA has no work.
  __device__ __forceinline__ bool locate(const Kv4AttnParams& p, Shared& s, int max_ctas, int min_tiles) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long mine = 0, sum = 0;
    for (int k = tid; k < p.R; k += THREADS) {
      mine = head_tiles(p, kv4_load_request(p, k)) * p.c.n_kv;
      sum += mine;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) s.scan[warp] = sum;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) total += s.scan[w];
    ctas = max(1ll, min((long long)max_ctas, total / min_tiles));
    const long long cta = blockIdx.x;
    if (cta >= ctas || total == 0) return false;
    u0 = cta * total / ctas;
    u1 = (cta + 1) * total / ctas;
    long long base = 0;
    for (int k0 = 0; k0 < p.R; k0 += THREADS) {
      const int k = k0 + tid;
      const long long n = p.R <= THREADS ? mine : k < p.R ? head_tiles(p, kv4_load_request(p, k)) * p.c.n_kv : 0;
      long long v = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += u;
      }
      __syncthreads();
      if (lane == 31) s.scan[warp] = v;
      __syncthreads();
      long long before = base;
      for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += s.scan[w];
        base += s.scan[w];
      }
      if (before + v - n <= u0 && u0 < before + v) {
        s.r = k;
        s.found = before + v - n;
      }
      if (base > u0) break;
    }
    __syncthreads();
    r = s.r;
    item = s.found;
    req = kv4_load_request(p, r);
    blocks = row_blocks(p, req);
    const long long per_head = head_tiles(p, req);
    kvh = (int)((u0 - item) / per_head);
    item += kvh * per_head;
    for (rb = 0;; ++rb) {
      block_tiles(p, req, rb, tile_lo, n_tiles);
      if (u0 < item + n_tiles) break;
      item += n_tiles;
    }
    return true;
  }

  // The item after the current one.  False: none (lengths that changed under the kernel).
  __device__ __forceinline__ bool next(const Kv4AttnParams& p) {
    item += n_tiles;
    if (++rb == blocks) {
      rb = 0;
      if (++kvh == p.c.n_kv) {
        kvh = 0;
        blocks = 0;
        while (blocks == 0 && ++r < p.R) {
          req = kv4_load_request(p, r);
          blocks = row_blocks(p, req);
        }
        if (blocks == 0) return false;
      }
    }
    block_tiles(p, req, rb, tile_lo, n_tiles);
    return true;
  }

  // First and last CTA that have a part of the current item; a CTA's part goes to workspace slot
  // 2 * cta (the item began before its run) or 2 * cta + 1.
  __device__ __forceinline__ int first_cta() const { return (int)(((item + 1) * ctas - 1) / total); }
  __device__ __forceinline__ int last_cta() const { return (int)(((item + n_tiles) * ctas - 1) / total); }
};

// Address of record `rec` (16 tokens) of a request for one KV head; null past its last key.
__device__ __forceinline__ const uint8_t* kv4_record(const Kv4AttnParams& p, const int* table, int rec, int n_rec,
                                                     int rpb, int kvh, int rec_bytes) {
  if (rec >= n_rec) return nullptr;
  const int nth = rec / rpb;
  int block = table[nth];
  if (block < 0 || block >= p.c.n_blocks) {
    record_status(FQKV_STATUS_BAD_INDEX);
    block = 0;
  }
  return p.c.data + (((int64_t)block * p.c.n_kv + kvh) * rpb + (rec - nth * rpb)) * rec_bytes;
}

// Four-bit codes as 16-bit floats: nibbles j and j + 4 of w (bits 4 j and 16 + 4 j) as the pair
// kOffset + code, by placing the four bits in the mantissa of a constant.
template <typename T>
struct Kv4Nib;
template <>
struct Kv4Nib<__nv_bfloat16> {
  static constexpr float kOffset = 128.0f;  // 0x4300: four mantissa bits of weight 1..8
  static constexpr uint32_t kOffset2 = 0x43004300u;
  static constexpr uint32_t kCentre2 = 0x43084308u;  // 136 = offset + 8
  static constexpr float kMinNormal = 1e-30f;
  template <int j>
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    return ((w >> (4 * j)) & 0x000F000Fu) | kOffset2;
  }
  static __device__ __forceinline__ uint32_t sub2(uint32_t x, uint32_t y) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
  }
  static __device__ __forceinline__ uint32_t fma2(uint32_t x, uint32_t y, uint32_t z) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(z));
    return r;
  }
};
template <>
struct Kv4Nib<__half> {
  static constexpr float kOffset = 64.0f;  // 0x5400: mantissa bits 4..7 have weight 1..8
  static constexpr uint32_t kOffset2 = 0x54005400u;
  static constexpr uint32_t kCentre2 = 0x54805480u;  // 72 = offset + 8
  static constexpr float kMinNormal = 6.2e-5f;
  template <int j>
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    const uint32_t x = j == 0 ? w << 4 : w >> (4 * (j > 0 ? j - 1 : 0));
    return (x & 0x00F000F0u) | kOffset2;
  }
  static __device__ __forceinline__ uint32_t sub2(uint32_t x, uint32_t y) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
  }
  static __device__ __forceinline__ uint32_t fma2(uint32_t x, uint32_t y, uint32_t z) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(z));
    return r;
  }
};

__device__ __forceinline__ float kv4_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

}  // namespace fqkv
