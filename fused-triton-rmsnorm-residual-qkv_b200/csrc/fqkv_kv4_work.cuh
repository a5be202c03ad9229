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

// Position of query j: -1 for those before the first token, which see nothing, so that a window of
// any size can be taken off it.
__device__ __forceinline__ int kv4_position(const Kv4Request& q, int j) { return max(-1, q.len - q.n + j); }

// x * y / z for the cutting points: 32-bit arithmetic where the product allows it (a 64-bit
// division costs about 0.3 us of a CTA's start).
__device__ __forceinline__ long long kv4_muldiv(long long x, long long y, long long z, bool small) {
  return small ? (long long)((uint32_t)x * (uint32_t)y / (uint32_t)z) : x * y / z;
}

// POINTS: 1, or the block's warps; the run of the CTA or of each of its warps starts there.
// LEAD: an item counts as LEAD tiles more than it reads, in front of them, for what it costs to
// begin and to end one; a run that starts or ends among them starts or ends with the item.
template <int ROWS, int TILE, int THREADS, int POINTS, int LEAD>
struct Kv4Work {
  struct Shared {
    long long scan[THREADS / 32];
    long long found[POINTS], per_head[POINTS];
    Kv4Request req[POINTS];
    int r[POINTS];
    int rows[2];  // tokens of the batch that belong to a request: [rows[0], rows[1])
  };

  long long total, u0, u1;  // all tiles, this CTA's run
  long long a, b;           // this warp's part of it (POINTS > 1)
  // The current item: request r, KV head, row block; tiles [item, item + n_tiles) of the batch, of
  // which the first LEAD stand for nothing and the others for the keys' tiles from tile_lo on; row
  // blocks of the request.
  long long item;
  Kv4Request req;
  int ctas;   // CTAs that have work
  bool small;  // total * ctas is below 2^32
  int r, kvh, rb, blocks, tile_lo, n_tiles;

  // Tiles that row block rb of a request reads (at least one, so that every item is visited).
  // Rows are (query j, head) with row = j * G + head.
  static __device__ __forceinline__ void block_tiles(const Kv4AttnParams& p, const Kv4Request& q, int rb, int& tile_lo,
                                                     int& n_tiles) {
    const int j1 = min((int)((uint32_t)(rb * ROWS + ROWS - 1) / (uint32_t)p.G), q.n - 1);
    const int hi = max(0, min(q.len, q.len - q.n + j1 + 1));
    int lo = 0;
    if (p.window > 0) lo = max(0, kv4_position(q, (int)((uint32_t)(rb * ROWS) / (uint32_t)p.G)) - p.window + 1);
    tile_lo = lo / TILE;
    n_tiles = max(1, (hi + TILE - 1) / TILE - tile_lo) + LEAD;
  }

  // The keys' tiles [first, last) of the part [u, ue) of the current item.
  __device__ __forceinline__ void part_tiles(long long u, long long ue, int& first, int& last) const {
    first = tile_lo + max(0, (int)(u - item) - LEAD);
    last = tile_lo + max(0, (int)(ue - item) - LEAD);
  }

  static __device__ __forceinline__ int row_blocks(const Kv4AttnParams& p, const Kv4Request& q) {
    return (q.n * p.G + ROWS - 1) / ROWS;
  }

  // Tiles of one KV head of the lane's request (0 for q.n == 0).  Requests of more than two row
  // blocks are summed by the whole warp, one after the other.  Called by whole warps.
  static __device__ __forceinline__ long long head_tiles(const Kv4AttnParams& p, const Kv4Request& q) {
    const int lane = threadIdx.x & 31, n = row_blocks(p, q);
    long long sum = 0;
    int lo, tiles;
    if (n > 0 && n <= 2) {
      block_tiles(p, q, 0, lo, tiles);
      sum = tiles;
      if (n == 2) {
        block_tiles(p, q, 1, lo, tiles);
        sum += tiles;
      }
    }
    for (uint32_t big = __ballot_sync(~0u, n > 2); big; big &= big - 1) {
      const int owner = __ffs(big) - 1;
      Kv4Request o;
      o.start = 0;
      o.n = __shfl_sync(~0u, q.n, owner);
      o.len = __shfl_sync(~0u, q.len, owner);
      const int on = row_blocks(p, o);
      long long part = 0;
      for (int rb = lane; rb < on; rb += 32) {
        block_tiles(p, o, rb, lo, tiles);
        part += tiles;
      }
#pragma unroll
      for (int k = 16; k; k >>= 1) part += __shfl_xor_sync(~0u, part, k);
      if (lane == owner) sum = part;
    }
    return sum;
  }

  // Zeros for tokens [lo, hi) of out, which no item holds.
  static __device__ __forceinline__ void zero_rows(const Kv4AttnParams& p, int64_t lo, int64_t hi) {
    for (int64_t t = lo + blockIdx.x; t < hi; t += gridDim.x)
      for (int e = threadIdx.x; e < p.n_q * p.c.D / 8; e += THREADS)
        reinterpret_cast<uint4*>(p.out + t * p.o_t)[e] = make_uint4(0, 0, 0, 0);
  }

  // First tile of the run of point k.
  __device__ __forceinline__ long long point(int k) const {
    return POINTS == 1 ? u0 : u0 + kv4_muldiv(k, u1 - u0, POINTS, small);
  }

  // Called by the whole block.  False: this CTA has no work.  Tokens of no request (a plan's upper
  // bound of the tokens leaves some past the last request's) are written here, without any work too.
  __device__ __forceinline__ bool locate(const Kv4AttnParams& p, Shared& s, int max_ctas, int min_tiles) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Kv4Request none{0, 0, 0};
    // Pass 0 sums; the pass that finds the run's request is the same one when all requests fit the
    // block, a second walk over the chunks otherwise.
    const bool one = p.R <= THREADS;
    Kv4Request q = none;
    long long heads = 0, before = 0;
    total = 0;
    for (int k0 = 0; k0 < p.R; k0 += THREADS) {
      const int k = k0 + tid;
      q = k < p.R ? kv4_load_request(p, k) : none;
      if (k == 0) s.rows[0] = q.start;
      if (k == p.R - 1) s.rows[1] = q.start + q.n;
      heads = head_tiles(p, q);
      long long v = heads * p.c.n_kv;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += u;
      }
      if (lane == 31) s.scan[warp] = v;
      __syncthreads();
      before = total + v - heads * p.c.n_kv;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += s.scan[w];
        total += s.scan[w];
      }
      if (!one) __syncthreads();
    }
    if (__builtin_expect(s.rows[0] > 0 || s.rows[1] < p.T, 0)) {
      zero_rows(p, 0, s.rows[0]);
      zero_rows(p, s.rows[1], p.T);
    }
    ctas = (int)max(1ll, min((long long)max_ctas, total / min_tiles));
    small = total < (1ll << 32) / 1024;
    const int cta = blockIdx.x;
    if (cta >= ctas || total == 0) return false;
    u0 = kv4_muldiv(cta, total, ctas, small);
    u1 = kv4_muldiv(cta + 1, total, ctas, small);
    if (one) {
      publish(s, q, tid, before, heads, p.c.n_kv);
    } else {
      long long base = 0;
      for (int k0 = 0; k0 < p.R && base < u1; k0 += THREADS) {
        const int k = k0 + tid;
        q = k < p.R ? kv4_load_request(p, k) : none;
        heads = head_tiles(p, q);
        long long v = heads * p.c.n_kv;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long u = __shfl_up_sync(~0u, v, o);
          if (lane >= o) v += u;
        }
        __syncthreads();
        if (lane == 31) s.scan[warp] = v;
        __syncthreads();
        before = base + v - heads * p.c.n_kv;
        for (int w = 0; w < THREADS / 32; ++w) {
          if (w < warp) before += s.scan[w];
          base += s.scan[w];
        }
        publish(s, q, k, before, heads, p.c.n_kv);
      }
    }
    __syncthreads();
    const int at_point = POINTS == 1 ? 0 : warp;
    a = point(at_point);
    b = POINTS == 1 ? u1 : point(at_point + 1);
    r = s.r[at_point];
    req = s.req[at_point];
    item = s.found[at_point];
    blocks = row_blocks(p, req);
    const long long per_head = s.per_head[at_point];
    kvh = 0;
    while (a - item >= per_head) {  // fewer steps than KV heads, and no division
      item += per_head;
      ++kvh;
    }
    // The row block: each lane sums its own share of 32 blocks at a time.
    for (rb = 0;; rb += 32) {
      int lo, tiles = 0;
      if (rb + lane < blocks) block_tiles(p, req, rb + lane, lo, tiles);
      int v = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += u;
      }
      const uint32_t past = __ballot_sync(~0u, a < item + v);
      if (past) {
        const int at = __ffs(past) - 1;
        item += __shfl_sync(~0u, v - tiles, at);
        rb += at;
        break;
      }
      item += __shfl_sync(~0u, v, 31);
    }
    block_tiles(p, req, rb, tile_lo, n_tiles);
    return true;
  }

  __device__ __forceinline__ void publish(Shared& s, const Kv4Request& q, int k, long long before, long long heads,
                                          int n_kv) const {
    const long long after = before + heads * n_kv;
    if (after <= u0 || before >= u1) return;
#pragma unroll
    for (int x = 0; x < POINTS; ++x) {
      const long long u = point(x);
      if (before <= u && u < after) {
        s.r[x] = k;
        s.found[x] = before;
        s.per_head[x] = heads;
        s.req[x] = q;
      }
    }
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
        if (blocks == 0) {
          r = p.R - 1;
          req = Kv4Request{0, 0, 0};
          return false;
        }
      }
    }
    block_tiles(p, req, rb, tile_lo, n_tiles);
    return true;
  }

  // First and last CTA that have keys of the current item; a CTA's part goes to workspace slot
  // 2 * cta (the item began before its run) or 2 * cta + 1.
  __device__ __forceinline__ int owner(long long tile) const {
    return small ? (int)(((uint32_t)(tile + 1) * (uint32_t)ctas - 1) / (uint32_t)total)
                 : (int)(((tile + 1) * ctas - 1) / total);
  }
  __device__ __forceinline__ int first_cta() const { return owner(item + LEAD); }
  __device__ __forceinline__ int last_cta() const { return owner(item + n_tiles - 1); }
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

// (x & MASK) | magic in one instruction.  `magic` is a register whose value the compiler cannot
// see (kv4_opaque): two immediates would make it two instructions, and this is the kernels' most
// frequent one.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t kv4_place(uint32_t x, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "n"(MASK), "r"(magic));
  return r;
}
// `value`, from a number that is never negative.
__device__ __forceinline__ uint32_t kv4_opaque(uint32_t value, int not_negative) {
  return value ^ ((uint32_t)not_negative >> 31);
}

// Four-bit codes as 16-bit floats: nibbles j and j + 4 of w (bits 4 j and 16 + 4 j) as the pair
// offset + code, by placing the four bits in the mantissa of a constant (kOffset2, opaque).
template <typename T>
struct Kv4Nib;
template <>
struct Kv4Nib<__nv_bfloat16> {
  static constexpr uint32_t kOffset2 = 0x43004300u;  // 128: four mantissa bits of weight 1..8
  static constexpr bool kFullRange = true;  // of fp32
  template <int j>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, uint32_t magic) {
    return kv4_place<0x000F000Fu>(w >> (4 * j), magic);
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
  static constexpr uint32_t kOffset2 = 0x54005400u;  // 64: mantissa bits 4..7 have weight 1..8
  static constexpr bool kFullRange = false;
  template <int j>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, uint32_t magic) {
    return kv4_place<0x00F000F0u>(j == 0 ? w << 4 : w >> (4 * (j > 0 ? j - 1 : 0)), magic);
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
