// Attention of one new token per sequence over a paged key/value cache.
//
// For query head h of row b, with the tokens V that its window leaves visible,
//   o = sum_V e^(s_j - m) v_j / sum_V e^(s_j - m),  s_j = scale q.k_j,  m = max s_j.
// A row's cache is a list of 32-token tiles (those with a visible token), cut
// into pieces of piece_tiles() tiles.  One block takes one piece of one row for
// the query heads that share a KV head (each key and value is read once for
// all of them) and leaves the piece's maximum, sum and unnormalised output in
// fp32; a second kernel joins the pieces in their order.  A row that fits in
// one piece is finished by the first kernel.  Tiles and pieces depend on the
// row's own length and window alone, so its bits do not depend on the batch.
// Scores are kept in units of log2 (the scale carries log2(e)).
//
// Not in the reference, which keeps no cache between calls.
#include <algorithm>
#include <mutex>
#include <numeric>

#include "bio_tile.cuh"

namespace bio {

struct PagedParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  int64_t q_sb, q_sh, k_sp, k_sh, k_st, v_sp, v_sh, v_st, o_sb, o_sh;
  int64_t heads, pages, table_rows, table_width, t_sr;
  int kv_heads, group, page_size, d, dv;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* rows;
  int window, sinks;   // window 0: everything is visible
  int max_len;         // tokens that a row may have: its columns', below 2^31 by two tiles
  int box_rows;        // tokens of a TMA box: gcd(page size, tile)
  int group_shift;     // log2 of the boxes along a tile
  FixedDiv by_page;    // position -> column of the table
  float scale_log2;
  int64_t max_pieces;  // most pieces that any row can have
  int least;           // tiles of a piece at least: 1, or kSimtTiles
  int dvp;             // floats between partial outputs
  float* acc;          // [batch * heads][max_pieces][dvp]
  float2* ml;          // [batch * heads][max_pieces]: maximum, sum (-1: refused)
  int* status;
};

constexpr int kTile = 32;  // tokens of a tile

// Tiles of a piece of a row of n tiles.  Short pieces spread one sequence over
// the SMs; long rows take longer ones, since every piece costs a write and a
// read of its fp32 output.  `least` is what the kernel's way of working asks for.
// Measured (bf16, D 128), one row, 8 heads on 1: 1024 tokens 15 us, 2048 17, 2080
// 23, 8192 26, 8224 and up to 65536 36: a warp walks its piece's tiles in series.
// 128 rows, 8 KV heads, groups of 4 / 8 / 16: 1024 tokens 169 / 189 / 300 us (82
// for the bytes), 2048 230 / 253 / 396 (163), 2080 230 / 236 / 278 (166): with a
// piece per tile or two, wide groups write and read back as much as the cache holds.
__host__ __device__ __forceinline__ int piece_tiles(int n, int least) {
  const int c = n <= 32 ? 1 : n <= 64 ? 2 : n <= 256 ? 8 : 16;
  return c > least ? c : least;
}

__host__ __device__ __forceinline__ int pieces_of(int tiles, int least) {
  const int c = piece_tiles(tiles, least);
  return (tiles + c - 1) / c;
}

// What a row sees: token j with j < len and (j < sinks or j >= start).  Tile t
// of the row is the tile t < head ? t : t + jump of its tokens.  Positions fit
// in 32 bits, those of a last tile's hidden tokens too: max_len leaves room.
struct Visible {
  int row;  // row of the table, -1 if refused
  int len, sinks, start;
  int head, jump, tiles;
  __device__ __forceinline__ int base(int t) const { return (t < head ? t : t + jump) * kTile; }
  __device__ __forceinline__ bool sees(int j) const {
    return j < len && (j < sinks || j >= start);
  }
};

// The row of query b and its length; (-1, 0) if one of them is out of range.
__device__ __forceinline__ int2 row_of(const PagedParams& p, int64_t b) {
  const int row = p.rows != nullptr ? p.rows[b] : static_cast<int>(b);
  if (row < 0 || row >= p.table_rows) return make_int2(-1, 0);
  const int len = p.lens[row];
  return len < 0 || len > p.max_len ? make_int2(-1, 0) : make_int2(row, len);
}

__device__ __forceinline__ Visible visible_of(const PagedParams& p, int2 row_len) {
  Visible z;
  z.row = row_len.x;
  z.len = row_len.y;
  z.start = p.window > 0 && p.window < z.len ? z.len - p.window : 0;
  z.sinks = min(p.sinks, z.start);
  z.head = z.sinks / kTile + (z.sinks % kTile != 0);
  z.jump = max(0, z.start / kTile - z.head);
  z.tiles = z.len / kTile + (z.len % kTile != 0) - z.jump;
  return z;
}

// ---------------------------------------------------------------------------
// CUDA-core kernel: fp32, and 16-bit pages whose rows are not 16-byte aligned.
// LPK lanes share one key (16 dims each), so a warp handles 32 / LPK keys at
// once for HB query heads; q waits in shared memory.
// HBM bounds it with one query head per KV head (fp32, 32 rows of 4000 tokens, 8
// heads of 128: 166 us, 6.3 TB/s), the instructions per key and head with more (32
// heads on 8: 252 us, 4.2 TB/s; without the loads ahead and with each head's chain
// by itself 289 us; 16 heads of 256 on one, 4 rows of 30000: 294 -> 208 us).  A
// block's start and its warps' join cost as much as some hundred keys, so a piece
// has kSimtTiles tiles at least, and 64 columns take 4 lanes, not 8 (128 heads on
// 8, 20 rows of 1108: 275 -> 153 us).
// ---------------------------------------------------------------------------
constexpr int kSimtWarps = 4;
constexpr int kSimtTiles = 4;  // a tile for each warp of a piece's block at least
constexpr int kLaneDims = 16;

// Dim of element e of lane li: four-float groups (VEC) or single elements.
template <int LPK, bool VEC>
__device__ __forceinline__ int lane_dim(int li, int e) {
  return VEC ? ((e >> 2) * LPK + li) * 4 + (e & 3) : li + LPK * e;
}

template <typename T, int LPK, bool VEC>
__device__ __forceinline__ void load_dims(const T* row, int li, int d, bool on,
                                          float (&x)[kLaneDims]) {
#pragma unroll
  for (int e = 0; e < kLaneDims; ++e) x[e] = 0.f;
  if (!on) return;
  if constexpr (VEC) {
    static_assert(sizeof(T) == 4, "four-float groups");
#pragma unroll
    for (int e = 0; e < kLaneDims; e += 4) {
      const int c = lane_dim<LPK, VEC>(li, e);
      if (c < d) {
        const float4 w = *reinterpret_cast<const float4*>(row + c);
        x[e] = w.x; x[e + 1] = w.y; x[e + 2] = w.z; x[e + 3] = w.w;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kLaneDims; ++e) {
      const int c = lane_dim<LPK, VEC>(li, e);
      if (c < d) x[e] = to_f32(row[c]);
    }
  }
}

template <typename T, int HB, int LPK, bool VEC>
__global__ void __launch_bounds__(kSimtWarps * 32) paged_simt_kernel(const PagedParams p) {
  constexpr int kKeys = 32 / LPK;          // keys of a warp at once
  constexpr int kDims = LPK * kLaneDims;   // padded head dim
  __shared__ float qs[HB][kDims];
  __shared__ float part[kSimtWarps][HB][kDims];
  __shared__ float2 part_ml[kSimtWarps][HB];

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int li = lane % LPK, sub = lane / LPK;
  const int blocks_per_group = (p.group + HB - 1) / HB;
  int64_t x = blockIdx.x;
  const int64_t piece = x % p.max_pieces;
  x /= p.max_pieces;
  const int hb = static_cast<int>(x % blocks_per_group);
  x /= blocks_per_group;
  const int hk = static_cast<int>(x % p.kv_heads);
  const int64_t b = x / p.kv_heads;
  const int h0 = hk * p.group + hb * HB;              // first query head
  const int nh = min(HB, p.group - hb * HB);

  const Visible z = visible_of(p, row_of(p, b));
  const int c = piece_tiles(z.tiles, p.least), pieces = pieces_of(z.tiles, p.least);
  if (piece > 0 && piece >= pieces) return;
  int bad = z.row < 0;

  for (int i = threadIdx.x; i < HB * kDims; i += blockDim.x) {
    const int h = i / kDims, e = i % kDims;
    qs[h][e] = h < nh && e < p.d
                   ? to_f32(static_cast<const T*>(p.q)[b * p.q_sb + (h0 + h) * p.q_sh + e]) *
                         p.scale_log2
                   : 0.f;
  }
  __syncthreads();

  float m[HB], l[HB], o[HB][kLaneDims];
#pragma unroll
  for (int h = 0; h < HB; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int e = 0; e < kLaneDims; ++e) o[h][e] = 0.f;
  }
  const T* kb = static_cast<const T*>(p.k) + hk * p.k_sh;
  const T* vb = static_cast<const T*>(p.v) + hk * p.v_sh;
  const int t0 = static_cast<int>(piece) * c, left = min(c, z.tiles - t0) * kTile;
  // Two keys ahead: the page of key i + 2 and the key and value of i + 1 are on
  // their way while key i is worked on.
  constexpr int kStep = kSimtWarps * kKeys;
  struct Place {
    int page, slot;
    bool on;
  };
  auto place_of = [&](int x0) {
    Place w{0, 0, false};
    if (x0 >= left) return w;
    const int x1 = x0 + sub;  // kKeys divides the tile: all of them lie in one
    const int pos = z.base(t0 + x1 / kTile) + x1 % kTile;
    const int col = p.by_page.quotient(pos);
    w.on = z.sees(pos);
    if (w.on) w.page = p.table[z.row * p.t_sr + col];
    w.slot = pos - col * p.page_size;
    return w;
  };
  auto load = [&](Place w, float (&kx)[kLaneDims], float (&vx)[kLaneDims]) {
    if (w.on && (w.page < 0 || w.page >= p.pages)) {
      bad = 1;
      w.on = false;
    }
    load_dims<T, LPK, VEC>(kb + w.page * p.k_sp + w.slot * p.k_st, li, p.d, w.on, kx);
    load_dims<T, LPK, VEC>(vb + w.page * p.v_sp + w.slot * p.v_st, li, p.dv, w.on, vx);
    return w.on;
  };
  auto take = [&](const float (&kx)[kLaneDims], const float (&vx)[kLaneDims], bool on) {
    float s[HB];
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      float a = 0.f, b = 0.f;  // two chains
#pragma unroll
      for (int e = 0; e < kLaneDims; e += 2) {
        a = fmaf(qs[h][lane_dim<LPK, VEC>(li, e)], kx[e], a);
        b = fmaf(qs[h][lane_dim<LPK, VEC>(li, e + 1)], kx[e + 1], b);
      }
      s[h] = a + b;
    }
#pragma unroll
    for (int w = LPK / 2; w > 0; w >>= 1)
#pragma unroll
      for (int h = 0; h < HB; ++h) s[h] += __shfl_xor_sync(0xffffffffu, s[h], w);
    bool up = false;
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      if (!on) s[h] = -INFINITY;
      up |= s[h] > m[h];
    }
    if (__any_sync(0xffffffffu, up)) {  // a factor of 1 changes nothing
#pragma unroll
      for (int h = 0; h < HB; ++h) {
        const float top = fmaxf(m[h], s[h]);
        const float f = top > m[h] ? exp2f(m[h] - top) : 1.f;
        l[h] *= f;
#pragma unroll
        for (int e = 0; e < kLaneDims; ++e) o[h][e] *= f;
        m[h] = top;
      }
    }
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      const float w = s[h] == -INFINITY ? 0.f : exp2f(s[h] - m[h]);
      l[h] += w;
      // the values of a key out of sight were loaded as zeros
#pragma unroll
      for (int e = 0; e < kLaneDims; ++e) o[h][e] = fmaf(w, vx[e], o[h][e]);
    }
  };
  float kx[2][kLaneDims], vx[2][kLaneDims];
  bool on[2];
  int x0 = warp * kKeys;
  on[0] = load(place_of(x0), kx[0], vx[0]);
  Place then = place_of(x0 + kStep);
  for (; x0 < left; x0 += 2 * kStep) {
    on[1] = load(then, kx[1], vx[1]);
    then = place_of(x0 + 2 * kStep);
    take(kx[0], vx[0], on[0]);
    if (x0 + kStep >= left) break;
    on[0] = load(then, kx[0], vx[0]);
    then = place_of(x0 + 3 * kStep);
    take(kx[1], vx[1], on[1]);
  }

  // join the warp's key lanes (a fixed tree), then the warps in order
#pragma unroll
  for (int h = 0; h < HB; ++h) {
#pragma unroll
    for (int w = LPK; w < 32; w <<= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m[h], w);
      const float l2 = __shfl_xor_sync(0xffffffffu, l[h], w);
      const float top = fmaxf(m[h], m2);
      const float f1 = m[h] == -INFINITY ? 0.f : exp2f(m[h] - top);
      const float f2 = m2 == -INFINITY ? 0.f : exp2f(m2 - top);
      l[h] = l[h] * f1 + l2 * f2;
#pragma unroll
      for (int e = 0; e < kLaneDims; ++e) {
        const float o2 = __shfl_xor_sync(0xffffffffu, o[h][e], w);
        o[h][e] = o[h][e] * f1 + o2 * f2;
      }
      m[h] = top;
    }
    if (sub == 0) {
#pragma unroll
      for (int e = 0; e < kLaneDims; ++e)
        part[warp][h][lane_dim<LPK, VEC>(li, e)] = o[h][e];
      if (li == 0) part_ml[warp][h] = make_float2(m[h], l[h]);
    }
  }
  bad = __syncthreads_or(bad);
  if (bad && threadIdx.x == 0) raise_status(p.status, BIO_DEV_INDEX);
  for (int i = threadIdx.x; i < nh * p.dv; i += blockDim.x) {
    const int h = i / p.dv, e = i - h * p.dv;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSimtWarps; ++w) top = fmaxf(top, part_ml[w][h].x);
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kSimtWarps; ++w) {
      const float2 t = part_ml[w][h];
      const float f = t.x == -INFINITY ? 0.f : exp2f(t.x - top);
      sum = fmaf(t.y, f, sum);
      acc = fmaf(part[w][h][e], f, acc);
    }
    const int64_t bh = b * p.heads + h0 + h;
    if (pieces <= 1) {
      const float y = bad || sum == 0.f ? 0.f : acc / sum;
      static_cast<T*>(p.o)[b * p.o_sb + (h0 + h) * p.o_sh + e] = from_f32<T>(y);
    } else {
      p.acc[(bh * p.max_pieces + piece) * p.dvp + e] = acc;
      if (e == 0) p.ml[bh * p.max_pieces + piece] = make_float2(top, bad ? -1.f : sum);
    }
  }
}

// ---------------------------------------------------------------------------
// 16-bit kernel: TMA into swizzled shared memory, m16n8k16 products.
//
// One warp owns one item: a piece of one row for 8 * NH query heads of one KV
// head.  It walks the piece's tiles through its own ring of S stages, each a
// tile's keys, values and the item's queries, and refills a stage as soon as
// it has used it, across item borders, so that loads never wait for the
// arithmetic and warps never wait for each other.  A tile is fetched in boxes
// of 64 columns by R tokens, R = gcd(page size, 32), so a box never leaves its
// page.  Per tile, in two halves of 16 tokens:
//   S^T [16 keys x 8 heads] = K [16 x d] Q^T     A: ldmatrix, B: ldmatrix of Q
//   p = 2^(s - m) in the accumulator layout, rounded to T; movmatrix turns its
//   8 x 8 quarters into the B operand of
//   O^T [d x 8 heads] += V^T [d x 16] P^T        A: ldmatrix.trans
// P is rounded because the product takes operands of V's type; l sums the rounded
// weights, so that the ones that the values got add up to 1.
// Keys are the 16-row side, so a group of 8 heads fills the 8-column side
// exactly and m, l and the rescale factors of a head pair sit in the lane that
// holds that pair of O.  The cache is read once at a few flops per byte: what
// bounds it is HBM, not the products (m16n8k16 covers 2048 products per
// instruction; the tcgen05 tile of 128 rows would be 15/16 padding here).
// Measured on 128 rows of 1..8192 tokens (32 heads on 8, d 128, 2.15 GB): lanes
// copying 16-token tiles by cp.async 636 us, TMA 614 us, both with four warps
// on an item joining through shared memory; a warp per item 450 us, then bound
// by the serial chain of one warp's instructions, which 32-token tiles halve:
// 413 us.  No divisions and two sums per product chain: 398 us.  This kernel now
// runs 354 us of the 379..392 (6.1 TB/s read).  No gain from three stages and four
// warps (437 us) or from keys and values in slots of their own and eight warps
// (401 us, two waits a tile instead of one).
// ---------------------------------------------------------------------------
constexpr int kListRows = 512;   // rows whose piece counts fit in shared memory

template <int DP, int NH>
struct PagedSmem {
  static constexpr int kBlocks = DP / 64;                   // 64-column blocks
  static constexpr int kKv = kTile * 128 * kBlocks;         // keys (or values) of a tile
  static constexpr int kQ = 8 * NH * 128 * kBlocks;
  static constexpr int kStage = 2 * kKv + kQ;
  static constexpr int kMaxWarps = 12;
  static constexpr int kMisc = kMaxWarps * 8 * 2 + 72 * 4 + (3 * kListRows + 4) * 4;
  // one CTA per SM, as many warps as find room with two stages each
  static constexpr int kStages = 2;
  static constexpr int kFit = (226 * 1024 - kMisc) / (kStages * kStage);
  static constexpr int kWarps = kFit > kMaxWarps ? kMaxWarps : kFit;
  static constexpr int kBytes = 1024 + kMisc + kWarps * kStages * kStage;
  static_assert(kWarps >= 1 && kBytes <= 227 * 1024, "no room");
  static_assert(kStage % 1024 == 0, "the swizzle counts from 1024-byte borders");
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t mov_trans(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4],
                                                 uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two probabilities rounded to T, and their rounded values for the sum.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b, float& ra, float& rb);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b, float& ra, float& rb) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  ra = __low2float(v);
  rb = __high2float(v);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b, float& ra, float& rb) {
  const __half2 v = __floats2half2_rn(a, b);
  ra = __low2float(v);
  rb = __high2float(v);
  return *reinterpret_cast<const uint32_t*>(&v);
}

struct PagedItem {
  Visible z;
  int b;           // query
  int hk, h0, nh;  // KV head, first query head, number of them
  int piece, pieces;
  int t0, tiles;   // of the piece
};

template <typename T, int DP, int NH>
__global__ void __launch_bounds__(PagedSmem<DP, NH>::kWarps * 32, 1)
    paged_mma_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const PagedParams p, int items,
                     int batch, int list) {
  using L = PagedSmem<DP, NH>;
  constexpr int S = L::kStages, W = L::kWarps, HB = 8 * NH;
  extern __shared__ uint8_t smem[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + W * S * L::kStage);  // [W][S]
  int* misc = reinterpret_cast<int*>(bars + W * S);  // [W][S]: a stage's refused pages
  int* scan = misc + 48;                             // list: sums of the warps
  volatile int* abort_flag = misc + 64;
  int2* rows = reinterpret_cast<int2*>(misc + 72);   // list: table row and length of query b
  int* first = misc + 72 + 2 * kListRows;            // list: items before query b, [batch + 1]
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hblocks = (p.group + HB - 1) / HB;
  const int hgs = p.kv_heads * hblocks;

  if (threadIdx.x == 0) {
    for (int i = 0; i < W * S; ++i) mbar_init(&bars[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // The products run over all DP columns.  The boxes fill up to the next 64
  // with zeros; blocks that no box covers (d and dv differ) are zeroed here.
  if (p.d <= DP - 64 || p.dv <= DP - 64) {
    uint4* z = reinterpret_cast<uint4*>(ring);
    for (int i = threadIdx.x; i < W * S * L::kStage / 16; i += blockDim.x)
      z[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  // an empty or refused row has one item, which writes zeros
  int total = items;
  if (list) {
    // items of every row, as a running sum in shared memory
    int carry = 0;
    for (int b0 = 0; b0 < batch; b0 += blockDim.x) {
      const int b = b0 + threadIdx.x;
      int mine = 0;
      if (b < batch) {
        rows[b] = row_of(p, b);
        mine = max(1, pieces_of(visible_of(p, rows[b]).tiles, 1)) * hgs;
      }
      int inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      if (lane == 31) scan[warp] = inc;
      __syncthreads();
      int base = carry, sum = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (w < warp) base += scan[w];
        sum += scan[w];
      }
      if (b < batch) first[b] = base + inc - mine;
      carry += sum;
      __syncthreads();
    }
    if (threadIdx.x == 0) first[batch] = carry;
    total = carry;
  }
  __syncthreads();

  // item number -> what to do (without a list: nothing, for a piece that the row lacks)
  auto decode = [&](int item, PagedItem& it) {
    unsigned rest, hg;
    int2 row;
    if (list) {
      int lo = 0, hi = batch;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= item) lo = mid; else hi = mid;
      }
      it.b = lo;
      rest = item - first[lo];
      it.piece = rest / hgs;
      hg = rest - it.piece * hgs;
      row = rows[lo];
    } else {
      rest = static_cast<unsigned>(item) / static_cast<unsigned>(p.max_pieces);
      it.piece = item - rest * static_cast<unsigned>(p.max_pieces);
      it.b = rest / hgs;
      hg = rest - it.b * hgs;
      row = row_of(p, it.b);
    }
    it.hk = hblocks == 1 ? hg : hg / hblocks;
    const int before = (hg - it.hk * hblocks) * HB;  // heads of the group in earlier blocks
    it.h0 = it.hk * p.group + before;
    it.nh = min(HB, p.group - before);
    it.z = visible_of(p, row);
    const int c = piece_tiles(it.z.tiles, 1);
    it.pieces = max(1, pieces_of(it.z.tiles, 1));
    it.t0 = it.piece * c;
    it.tiles = max(0, min(c, it.z.tiles - it.t0));
  };

  // ------------------------------------------------------------- producer side
  // the next tile to fetch: its item, its number, and its groups' pages
  uint8_t* my_ring = ring + warp * (S * L::kStage);
  uint64_t* my_bars = bars + warp * S;
  const int step = gridDim.x * W;
  int in_item = blockIdx.x + gridDim.x * warp, in_tile = 0;
  bool in_done = in_item >= total;
  if (in_done) return;  // no barrier of the block follows
  PagedItem in;
  decode(in_item, in);
  const int groups = 1 << p.group_shift, group_mask = groups - 1;
  int in_page = 0, in_slot = 0;  // of group `lane` of the tile (lanes below groups)
  bool in_held = false;          // the group has a visible token
  auto look_up = [&]() {
    while (!in_done && in_tile >= in.tiles) {
      in_item += step;
      in_tile = 0;
      in_done = in_item >= total;
      if (!in_done) decode(in_item, in);
    }
    in_held = false;
    if (!in_done && lane < groups) {
      const int pos = in.z.base(in.t0 + in_tile) + lane * p.box_rows;
      // visible in [pos, pos + box_rows): before the sinks' end, or from start to the length
      in_held = pos < in.z.sinks || (pos < in.z.len && pos + p.box_rows > in.z.start);
      if (in_held) {
        const int col = p.by_page.quotient(pos);
        in_slot = pos - col * p.page_size;
        // not looked at before the next fetch, so that nobody waits for it here
        in_page = p.table[in.z.row * p.t_sr + col];
      }
    }
  };
  const int kc = (p.d + 63) / 64, vc = (p.dv + 63) / 64;  // 64-column boxes of a row
  // box x of a tile: group x % groups, column block x / groups (the keys', then the values')
  const int boxes = groups * (kc + vc), tile_bytes = (kc + vc) * p.box_rows * 128;
  const uint32_t my_ring32 = smem_u32(my_ring), my_bars32 = smem_u32(my_bars);
  int issued = 0;  // tiles fetched so far
  auto fetch = [&](int stage) {
    if (in_done) return;
    ++issued;
    const bool refused = in_held && (in_page < 0 || in_page >= p.pages);
    const int page = in_held && !refused ? in_page : -1;
    const int held = __popc(__ballot_sync(0xffffffffu, page >= 0));
    const int lost = __any_sync(0xffffffffu, refused);
    const uint32_t dst = my_ring32 + stage * L::kStage, bar = my_bars32 + stage * 8;
    if (lane == 0) {
      const bool query = in_tile == 0;  // the item's queries travel with its first tile
      misc[warp * S + stage] = lost;
      expect_bytes(bar, held * tile_bytes + (query ? kc * HB * 128 : 0));
      if (query)
        for (int c = 0; c < kc; ++c)
          load_box(dst + 2 * L::kKv + c * HB * 128, &tmQ, bar, c * 64, in.h0, in.b, 0);
    }
    __syncwarp();
    for (int x0 = 0; x0 < boxes; x0 += 32) {
      const int x = x0 + lane, g = x & group_mask, c = x >> p.group_shift;
      const int pg = __shfl_sync(0xffffffffu, page, g);
      const int slot = __shfl_sync(0xffffffffu, in_slot, g);
      if (x < boxes && pg >= 0) {
        const uint32_t to = dst + g * p.box_rows * 128;
        if (c < kc)
          load_box(to + c * (kTile * 128), &tmK, bar, c * 64, slot, in.hk, pg);
        else
          load_box(to + L::kKv + (c - kc) * (kTile * 128), &tmV, bar, (c - kc) * 64, slot, in.hk,
                   pg);
      }
    }
    ++in_tile;
    look_up();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(s);

  // ------------------------------------------------------------- consumer side
  int stage = 0, used = 0;
  uint32_t phase = 0;
  bool ok = true;
  // A tile lies in 64-column blocks of 128-byte rows whose 16-byte chunks are
  // xor-ed with the row: chunk 2 t + c of row r is at (r * 128 + ((c ^ r) * 16))
  // ^ (t % 4 * 32) of block t / 4, so only an xor is left per k-step.
  const int qrow = lane & 7, krow = lane & 15, vrow = (lane & 7) + ((lane >> 4) << 3);
  const uint32_t qoff = qrow * 128 + (((lane >> 3) ^ qrow) << 4);
  const uint32_t koff = krow * 128 + (((lane >> 4) ^ (krow & 7)) << 4);
  const uint32_t voff = vrow * 128 + ((((lane >> 3) & 1) ^ (vrow & 7)) << 4);
  for (int item = blockIdx.x + gridDim.x * warp; item < total; item += step) {
    PagedItem it;
    decode(item, it);
    if (it.piece >= it.pieces) continue;
    int bad = it.z.row < 0;
    float m[NH][2], l[NH][2], o[DP / 16][NH][4];
    uint32_t qf[DP / 16][NH][2];
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][n][e] = 0.f;
    }
    for (int tile = 0; tile < it.tiles; ++tile) {
      if (ok) ok = parked_wait(my_bars32 + stage * 8, phase, abort_flag, p.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {  // a wait ran out: no more loads, zeros for what is left
        bad = 1;
        break;
      }
      const uint32_t sk = my_ring32 + stage * L::kStage, sv = sk + L::kKv, sq = sv + L::kKv;
      bad |= misc[warp * S + stage];
      const int pos = it.z.base(it.t0 + tile);
      const bool edge =
          !(pos + kTile <= it.z.len && (pos >= it.z.start || pos + kTile <= it.z.sinks));
      if (edge) {
        // tokens out of sight have weight 0, but 0 * NaN is not 0
        uint8_t* v = my_ring + stage * L::kStage + L::kKv;
        for (int r = 0; r < kTile; ++r)
          if (!it.z.sees(pos + r))
            for (int c = lane; c < vc * 8; c += 32)
              *reinterpret_cast<uint4*>(v + (c >> 3) * (kTile * 128) + r * 128 +
                                        (((c & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();  // the next load of this stage comes after these writes
        __syncwarp();
      }
      if (tile == 0) {
        // B operand: heads in rows of 8, four 8-dim chunks per ldmatrix
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int t = 0; t < DP / 16; t += 2) {
            uint32_t r[4];
            ldsm_x4(((sq + n * 1024 + qoff) ^ ((t & 2) << 5)) + (t >> 2) * (HB * 128), r);
            qf[t][n][0] = r[0];
            qf[t][n][1] = r[1];
            qf[t + 1][n][0] = r[2];
            qf[t + 1][n][1] = r[3];
          }
      }
      // s[half][n]: rows: keys lane / 4 and lane / 4 + 8; columns: heads 2 (lane % 4) + {0, 1}.
      // Even and odd k-steps have sums of their own: a product waits for the one before it.
      float s[2][NH][4], s2[2][NH][4];
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][n][e] = s[1][n][e] = s2[0][n][e] = s2[1][n][e] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) {
        const uint32_t at = ((sk + koff) ^ ((t & 3) << 5)) + (t >> 2) * (kTile * 128);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t a[4];
          ldsm_x4(at + x * 2048, a);
#pragma unroll
          for (int n = 0; n < NH; ++n)
            mma16816<T>(t & 1 ? s2[x][n] : s[x][n], a, qf[t][n][0], qf[t][n][1]);
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[x][n][e] = (s[x][n][e] + s2[x][n][e]) * p.scale_log2;
      if (edge) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (it.z.sees(pos + x * 8 + (lane >> 2))) continue;
#pragma unroll
          for (int n = 0; n < NH; ++n)
            s[x >> 1][n][(x & 1) * 2] = s[x >> 1][n][(x & 1) * 2 + 1] = -INFINITY;
        }
      }
      uint32_t pf[2][NH][2];
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e]));
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          top = fmaxf(top, m[n][e]);
          // scores of -inf alone have no maximum to subtract: their weight is 0
          const float ref = top == -INFINITY ? 0.f : top;
          f[e] = pow2(m[n][e] - ref);
          m[n][e] = top;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            s[x][n][e] = pow2(s[x][n][e] - ref);
            s[x][n][2 + e] = pow2(s[x][n][2 + e] - ref);
          }
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float r00, r01, r10, r11;
          pf[x][n][0] = mov_trans(pack2<T>(s[x][n][0], s[x][n][1], r00, r01));
          pf[x][n][1] = mov_trans(pack2<T>(s[x][n][2], s[x][n][3], r10, r11));
          sum[0] += r00 + r10;
          sum[1] += r01 + r11;
        }
        l[n][0] = l[n][0] * f[0] + sum[0];
        l[n][1] = l[n][1] * f[1] + sum[1];
        if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) {
            o[t][n][0] *= f[0];
            o[t][n][1] *= f[1];
            o[t][n][2] *= f[0];
            o[t][n][3] *= f[1];
          }
        }
      }
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) {
        const uint32_t at = ((sv + voff) ^ ((t & 3) << 5)) + (t >> 2) * (kTile * 128);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t a[4];
          ldsm_x4_t(at + x * 2048, a);
#pragma unroll
          for (int n = 0; n < NH; ++n) mma16816<T>(o[t][n], a, pf[x][n][0], pf[x][n][1]);
        }
      }
      __syncwarp();
      fetch(stage);
      ++used;
      if (++stage == S) {
        stage = 0;
        phase ^= 1;
      }
    }
    // ------------------------------------------------------- the item's result
    if (bad && lane == 0) raise_status(p.status, BIO_DEV_INDEX);
#pragma unroll
    for (int n = 0; n < NH; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], w);
        const int h = n * 8 + 2 * (lane & 3) + e;
        if (h >= it.nh) continue;
        if (it.pieces == 1) {
          const bool none = bad || l[n][e] == 0.f;
          const float inv = 1.f / l[n][e];
          T* out = static_cast<T*>(p.o) + it.b * p.o_sb + (it.h0 + h) * p.o_sh;
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int c = t * 16 + u * 8 + (lane >> 2);
              if (c < p.dv) out[c] = from_f32<T>(none ? 0.f : o[t][n][2 * u + e] * inv);
            }
          }
        } else {
          const int64_t at = (static_cast<int64_t>(it.b) * p.heads + it.h0 + h) * p.max_pieces +
                             it.piece;
          float* acc = p.acc + at * p.dvp;
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int c = t * 16 + u * 8 + (lane >> 2);
              if (c < p.dv) acc[c] = o[t][n][2 * u + e];
            }
          }
          if (lane < 4) p.ml[at] = make_float2(m[n][e], bad ? -1.f : l[n][e]);
        }
      }
    }
  }
  // after a wait that ran out, copies may still be in flight
  for (; used < issued; ++used)
    if (!mbar_wait_drain(&my_bars[used % S], (used / S) & 1)) raise_status(p.status, BIO_DEV_TIMEOUT);
}

// ---------------------------------------------------------------------------
// Joins the pieces of every (row, head): weights e^(m_i - max m); pieces i = j,
// j + 8, ... make sum j, and the eight sums are added in order.  With SPREAD, the
// eight warps of a block make the sums of one head; without, a warp makes all of
// them, eight loads in flight, and a block joins eight heads.  Bits are the same.
// Latency bounds it: up to 32 pieces of 4096 heads (67 MB) took 25 us with a block
// per head and take 16 with a warp; 256 pieces of 64 heads want the block, since 64
// warps would leave most of the SMs idle.
// ---------------------------------------------------------------------------
constexpr int kJoinWarps = 8;
constexpr int kSpreadPieces = 64;  // more pieces than this: a block per head

__device__ __forceinline__ void add_scaled(float4& y, const float4& a, float f) {
  y.x = fmaf(a.x, f, y.x);
  y.y = fmaf(a.y, f, y.y);
  y.z = fmaf(a.z, f, y.z);
  y.w = fmaf(a.w, f, y.w);
}

// G: 128-column groups of an output row
template <typename T, int G, bool SPREAD>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const PagedParams p,
                                                                     int64_t outputs) {
  constexpr int U = kJoinWarps;
  __shared__ float4 part[SPREAD ? kJoinWarps : 1][32 * G];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t bh = SPREAD ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * kJoinWarps + warp;
  const int64_t b = min(bh, outputs - 1) / p.heads, h = bh - b * p.heads;
  // lengths were there before the kernel that this one waits for began
  const int pieces = pieces_of(visible_of(p, row_of(p, b)).tiles, p.least);
  // Every thread waits, also where nothing is left to join: what comes next on the
  // stream waits for this grid alone, and rows of one piece are written by the other.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (bh >= outputs || pieces <= 1) return;  // bh: only without SPREAD
  const float2* ml = p.ml + bh * p.max_pieces;
  const int groups = p.dvp / 4;  // four-float groups of an output row
  const float4* acc = reinterpret_cast<const float4*>(p.acc + bh * p.max_pieces * p.dvp);
  // round r, load u: piece 8 r + u of all sums, or piece 8 (8 r + u) + warp of the warp's
  auto piece_of = [&](int r, int u) { return SPREAD ? (r * U + u) * kJoinWarps + warp : r * U + u; };
  float4 a[U][G];
  auto load = [&](int r) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int i = piece_of(r, u);
        a[u][g] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < pieces && lane + 32 * g < groups)
          a[u][g] = acc[static_cast<int64_t>(i) * groups + lane + 32 * g];
      }
  };
  load(0);
  float top = -INFINITY;
  bool bad = false;
  for (int i = lane; i < pieces; i += 32) {
    top = fmaxf(top, ml[i].x);
    bad |= ml[i].y == -1.f;
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  bad = __any_sync(0xffffffffu, bad);
  float sum = 0.f;
  for (int i = lane; i < pieces; i += 32)
    sum = fmaf(ml[i].y, ml[i].x == -INFINITY ? 0.f : exp2f(ml[i].x - top), sum);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);

  constexpr int Y = SPREAD ? 1 : U;
  float4 y[Y][G];
#pragma unroll
  for (int j = 0; j < Y; ++j)
#pragma unroll
    for (int g = 0; g < G; ++g) y[j][g] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int r = 0; piece_of(r, 0) < pieces; ++r) {
    if (r > 0) load(r);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = piece_of(r, u);
      if (i >= pieces) break;
      const float f = ml[i].x == -INFINITY ? 0.f : exp2f(ml[i].x - top);
#pragma unroll
      for (int g = 0; g < G; ++g) add_scaled(y[SPREAD ? 0 : u][g], a[u][g], f);
    }
  }
  T* out = static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh;
  const bool none = bad || sum == 0.f;
  if constexpr (SPREAD) {
#pragma unroll
    for (int g = 0; g < G; ++g) part[warp][lane + 32 * g] = y[0][g];
    __syncthreads();
    const float* flat = reinterpret_cast<const float*>(part);
    for (int e = threadIdx.x; e < p.dv; e += blockDim.x) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) x += flat[w * 128 * G + e];
      out[e] = from_f32<T>(none ? 0.f : x / sum);
    }
  } else {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < Y; ++j) {
        x[0] += y[j][g].x;
        x[1] += y[j][g].y;
        x[2] += y[j][g].z;
        x[3] += y[j][g].w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = (lane + 32 * g) * 4 + e;
        if (c < p.dv) out[c] = from_f32<T>(none ? 0.f : x[e] / sum);
      }
    }
  }
}

}  // namespace bio

namespace {

constexpr int64_t kMaxGrid = 2147483647;
// Items are counted in 32 bits, up to one step (a warp of every SM) past the last.
constexpr int64_t kMaxItems = kMaxGrid - 65536;
// The kernels count positions in 32 bits, up to the end of a row's last tile and
// of the tile after it.
constexpr int64_t kMaxTokens = kMaxGrid - 2 * bio::kTile;

// Most pieces that a row of up to `most` tiles can have.
int64_t most_pieces(int64_t most, int least) {
  int64_t pieces = 1;
  for (int64_t top : {static_cast<int64_t>(32), static_cast<int64_t>(64),
                      static_cast<int64_t>(256), most}) {
    const int64_t k = bio::pieces_of(static_cast<int>(top < most ? top : most), least);
    if (k > pieces) pieces = k;
  }
  return pieces;
}

struct Split {
  int64_t most;    // tiles that any row can have
  int64_t pieces;
  int dvp;
  int64_t acc_bytes, bytes;
};

int split_of(const bio_paged_attn_args* a, Split* s) {
  if (a == nullptr) return BIO_ERR_ARG;
  if (a->batch < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads ||
      a->heads > 65536 || a->d < 1 || a->d > 256 || a->dv < 1 || a->dv > 256 || a->page_size < 1 ||
      a->page_size > 65536 || a->pages < 0 || a->pages > kMaxGrid || a->table_rows < 0 ||
      a->table_rows > kMaxGrid || a->table_width < 0 || a->table_width > kMaxGrid / a->page_size)
    return BIO_ERR_SHAPE;
  if (a->window < 0 || a->window > kMaxGrid || a->sinks < 0 || a->sinks > kMaxGrid)
    return BIO_ERR_ARG;
  const int64_t T = bio::kTile;
  int64_t most = (a->table_width * a->page_size + T - 1) / T;
  if (a->window > 0)  // the window's tiles, one more where it starts inside one, the sinks'
    most = std::min(most, (a->window + T - 1) / T + 1 + (a->sinks + T - 1) / T);
  s->most = most;
  s->pieces = most_pieces(most, 1);  // longer pieces need less
  s->dvp = (a->dv + 3) / 4 * 4;
  if (a->batch > kMaxGrid / a->heads || a->batch * a->heads > kMaxItems / s->pieces)
    return BIO_ERR_SHAPE;
  const int64_t parts = s->pieces > 1 ? a->batch * a->heads * s->pieces : 0;
  s->acc_bytes = parts * s->dvp * 4;
  s->bytes = s->acc_bytes + parts * 8;
  return BIO_OK;
}

template <typename T, int HB, int LPK, bool VEC>
int launch_simt(const bio::PagedParams& p, int64_t batch, cudaStream_t s) {
  const int64_t grid = batch * p.kv_heads * ((p.group + HB - 1) / HB) * p.max_pieces;
  bio::paged_simt_kernel<T, HB, LPK, VEC>
      <<<static_cast<unsigned>(grid), bio::kSimtWarps * 32, 0, s>>>(p);
  return bio_host::launch_status(cudaGetLastError());
}

template <typename T, int LPK, bool VEC>
int dispatch_simt(const bio::PagedParams& p, int64_t batch, cudaStream_t s) {
  if (p.group >= 3) return launch_simt<T, 4, LPK, VEC>(p, batch, s);
  if (p.group == 2) return launch_simt<T, 2, LPK, VEC>(p, batch, s);
  return launch_simt<T, 1, LPK, VEC>(p, batch, s);
}

// As many lanes per key as its columns fill.
template <typename T, bool VEC>
int run_simt(bio::PagedParams* p, int64_t batch, int64_t most, cudaStream_t s) {
  p->least = bio::kSimtTiles;
  p->max_pieces = most_pieces(most, p->least);
  const int dim = std::max(p->d, p->dv);
  return dim > 128  ? dispatch_simt<T, 16, VEC>(*p, batch, s)
         : dim > 64 ? dispatch_simt<T, 8, VEC>(*p, batch, s)
                    : dispatch_simt<T, 4, VEC>(*p, batch, s);
}

template <typename T, int DP, int NH>
int launch_mma(const bio::PagedParams& p, int64_t batch, cudaStream_t s) {
  using L = bio::PagedSmem<DP, NH>;
  static std::once_flag once[bio_host::kMaxDevices];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= bio_host::kMaxDevices)
    return BIO_ERR_LAUNCH;
  cudaError_t set = cudaSuccess;
  std::call_once(once[device], [&] {
    set = cudaFuncSetAttribute(bio::paged_mma_kernel<T, DP, NH>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  });
  if (set != cudaSuccess) return BIO_ERR_LAUNCH;
  CUtensorMap q, k, v;
  // a pool without pages is never read: any aligned address will do for its maps
  const int64_t pages = std::max<int64_t>(p.pages, 1);
  if (!bio_host::map_of<T>(&q, p.q, p.d, p.heads, batch, 1, p.q_sh, p.q_sb, 0, 8 * NH) ||
      !bio_host::map_of<T>(&k, p.pages > 0 ? p.k : p.q, p.d, p.page_size, p.kv_heads, pages, p.k_st, p.k_sh,
                 p.k_sp, p.box_rows) ||
      !bio_host::map_of<T>(&v, p.pages > 0 ? p.v : p.q, p.dv, p.page_size, p.kv_heads, pages, p.v_st, p.v_sh,
                 p.v_sp, p.box_rows))
    return BIO_ERR_ALIGN;
  const int64_t sms = bio_host::sm_count(device);
  const int64_t items =
      batch * p.kv_heads * ((p.group + 8 * NH - 1) / (8 * NH)) * p.max_pieces;
  if (sms <= 0) return BIO_ERR_LAUNCH;
  // A few possible items per warp are walked as they are (an item of a piece
  // that the row does not have costs a look at its length).  Beyond, every
  // block first builds the list of the items that exist.
  const bool list = items > 2 * sms * L::kWarps && batch <= bio::kListRows;
  // one block per item, until the SMs are full; then a block's warps take items too
  const int64_t grid = std::min(items, sms);
  bio::paged_mma_kernel<T, DP, NH>
      <<<static_cast<unsigned>(grid), L::kWarps * 32, L::kBytes, s>>>(
          q, k, v, p, static_cast<int>(items), static_cast<int>(batch), list ? 1 : 0);
  return bio_host::launch_status(cudaGetLastError());
}

template <typename T>
int dispatch_mma(const bio::PagedParams& p, int64_t batch, cudaStream_t s) {
  const int dim = p.d > p.dv ? p.d : p.dv;
  // 16 heads at once halve the cache traffic of wide groups; at 256 columns
  // their partial results would not leave room for the ring
  if (dim > 128) return launch_mma<T, 256, 1>(p, batch, s);
  if (dim > 64)
    return p.group > 8 ? launch_mma<T, 128, 2>(p, batch, s) : launch_mma<T, 128, 1>(p, batch, s);
  return p.group > 8 ? launch_mma<T, 64, 2>(p, batch, s) : launch_mma<T, 64, 1>(p, batch, s);
}

template <typename T>
int run(bio::PagedParams p, int64_t batch, int64_t most, cudaStream_t s) {
  int st;
  p.least = 1;
  if constexpr (sizeof(T) == 4) {
    const uint64_t bits = reinterpret_cast<uint64_t>(p.k) | reinterpret_cast<uint64_t>(p.v) |
                          4 * static_cast<uint64_t>(p.k_sp | p.k_sh | p.k_st | p.v_sp | p.v_sh |
                                                    p.v_st | p.d | p.dv);
    st = bits % 16 == 0 ? run_simt<T, true>(&p, batch, most, s)
                        : run_simt<T, false>(&p, batch, most, s);
  } else {
    const uint64_t bits = reinterpret_cast<uint64_t>(p.q) | reinterpret_cast<uint64_t>(p.k) |
                          reinterpret_cast<uint64_t>(p.v) |
                          2 * static_cast<uint64_t>(p.q_sb | p.q_sh | p.k_sp | p.k_sh | p.k_st |
                                                    p.v_sp | p.v_sh | p.v_st | p.d | p.dv);
    st = bits % 16 == 0 ? dispatch_mma<T>(p, batch, s) : BIO_ERR_ALIGN;
    // rows off a 16-byte boundary, or strides that no tensor map takes
    if (st == BIO_ERR_ALIGN) st = run_simt<T, false>(&p, batch, most, s);
  }
  if (st != BIO_OK || p.max_pieces == 1) return st;
  const bool spread = p.max_pieces > bio::kSpreadPieces, wide = p.dvp > 128;
  const int64_t outputs = batch * p.heads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(
      spread ? outputs : (outputs + bio::kJoinWarps - 1) / bio::kJoinWarps));
  cfg.blockDim = dim3(bio::kJoinWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  auto join = spread ? (wide ? bio::paged_join_kernel<T, 2, true> : bio::paged_join_kernel<T, 1, true>)
                     : (wide ? bio::paged_join_kernel<T, 2, false>
                             : bio::paged_join_kernel<T, 1, false>);
  return bio_host::launch_status(cudaLaunchKernelEx(&cfg, join, p, outputs));
}

}  // namespace

extern "C" {

int64_t bio_paged_attention_workspace(const bio_paged_attn_args* args) {
  Split s;
  return split_of(args, &s) == BIO_OK ? s.bytes : 0;
}

int bio_paged_attention(const bio_paged_attn_args* a, void* workspace, int64_t workspace_bytes,
                        void* stream) {
  Split s;
  int st = split_of(a, &s);
  if (st != BIO_OK) return st;
  if (a->batch == 0) return BIO_OK;
  if (a->q == nullptr || a->o == nullptr || a->seq_lens == nullptr ||
      (a->table_width > 0 && a->page_table == nullptr) ||
      (a->pages > 0 && (a->k == nullptr || a->v == nullptr)))
    return BIO_ERR_ARG;
  if (s.bytes > 0 && (workspace == nullptr || workspace_bytes < s.bytes))
    return BIO_ERR_SCRATCH;
  if (s.bytes > 0 && reinterpret_cast<uintptr_t>(workspace) % 16) return BIO_ERR_ALIGN;
  st = bio_host::ensure_device(a->device);
  if (st != BIO_OK) return st;
  bio::PagedParams p;
  p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o;
  p.q_sb = a->q_sb; p.q_sh = a->q_sh;
  p.k_sp = a->k_sp; p.k_sh = a->k_sh; p.k_st = a->k_st;
  p.v_sp = a->v_sp; p.v_sh = a->v_sh; p.v_st = a->v_st;
  p.o_sb = a->o_sb; p.o_sh = a->o_sh;
  p.heads = a->heads; p.pages = a->pages;
  p.table_rows = a->table_rows; p.table_width = a->table_width; p.t_sr = a->t_sr;
  p.kv_heads = static_cast<int>(a->kv_heads);
  p.group = static_cast<int>(a->heads / a->kv_heads);
  p.page_size = static_cast<int>(a->page_size);
  p.d = a->d; p.dv = a->dv;
  p.table = a->page_table; p.lens = a->seq_lens; p.rows = a->rows;
  p.window = static_cast<int>(a->window);
  p.sinks = static_cast<int>(a->sinks);
  p.max_len = static_cast<int>(std::min(a->table_width * a->page_size, kMaxTokens));
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.box_rows = std::gcd(p.page_size, bio::kTile);
  p.group_shift = 0;
  while ((p.box_rows << p.group_shift) < bio::kTile) ++p.group_shift;
  p.by_page = bio::fixed_div(p.page_size);
  p.max_pieces = s.pieces;
  p.dvp = s.dvp;
  p.acc = static_cast<float*>(workspace);
  p.ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + s.acc_bytes);
  p.status = bio_host::status_word(a->device);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case BIO_F32: return run<float>(p, a->batch, s.most, cs);
    case BIO_F16: return run<__half>(p, a->batch, s.most, cs);
    case BIO_BF16: return run<__nv_bfloat16>(p, a->batch, s.most, cs);
    default: return BIO_ERR_DTYPE;
  }
}

}  // extern "C"
