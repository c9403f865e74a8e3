// Attention of one new token per sequence over a paged key/value cache.
//
// For query head h of row b, with the n tokens that its window leaves visible,
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q.k_j,  m = max s_j.
// The visible tokens are cut into pieces of piece_tokens(n) tokens.  One block
// takes one piece of one row for the query heads that share a KV head (each
// key and value is read once for all of them) and leaves the piece's maximum,
// sum and unnormalised output in fp32; a second kernel joins the pieces in
// their order.  A row that fits in one piece is finished by the first kernel.
// The piece size depends on n alone, so a row's bits do not depend on the
// batch.  Scores are kept in units of log2 (scale * log2(e) goes into q).
//
// Not in the reference, which keeps no cache between calls.
#include <mutex>

#include "bio_common.cuh"

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
  int64_t window, sinks;
  float scale_log2;
  int64_t max_pieces;  // most pieces that any row can have
  int dvp;             // floats between partial outputs
  float* acc;          // [batch * heads][max_pieces][dvp]
  float2* ml;          // [batch * heads][max_pieces]: maximum, sum (-1: refused)
  int* status;
};

// Tokens of a piece of a row that sees n tokens.  Short pieces spread one
// sequence over the SMs; long rows take longer ones, since every piece costs a
// write and a read of its fp32 output.
__host__ __device__ __forceinline__ int piece_tokens(int64_t n) {
  return n <= 1024 ? 64 : n <= 8192 ? 128 : n <= 32768 ? 256 : 512;
}

// What row b sees: tokens u = 0..n-1, token u at position u < sinks ? u : u + skip.
struct Visible {
  int64_t row;  // row of the table, -1 if refused
  int64_t n, sinks, skip;
};

__device__ __forceinline__ Visible visible_of(const PagedParams& p, int64_t b) {
  Visible z;
  z.row = p.rows != nullptr ? p.rows[b] : b;
  z.n = z.sinks = z.skip = 0;
  if (z.row < 0 || z.row >= p.table_rows) {
    z.row = -1;
    return z;
  }
  const int64_t len = p.lens[z.row];
  if (len < 0 || len > p.table_width * p.page_size) {
    z.row = -1;
    return z;
  }
  z.n = len;
  if (p.window > 0 && p.window < len) {
    z.sinks = min(p.sinks, len - p.window);
    z.skip = len - p.window - z.sinks;
    z.n = p.window + z.sinks;
  }
  return z;
}

// ---------------------------------------------------------------------------
// CUDA-core kernel: fp32, and 16-bit pages whose rows are not 16-byte aligned.
// LPK lanes share one key (16 dims each), so a warp handles 32 / LPK keys at
// once for HB query heads; q waits in shared memory.
// ---------------------------------------------------------------------------
constexpr int kSimtWarps = 4;
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

  const Visible z = visible_of(p, b);
  const int c = piece_tokens(z.n);
  const int64_t pieces = (z.n + c - 1) / c;
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
  const int64_t u1 = min(z.n, (piece + 1) * c);
  for (int64_t u0 = piece * c + warp * kKeys; u0 < u1; u0 += kSimtWarps * kKeys) {
    const int64_t u = u0 + sub;
    const int64_t pos = u < z.sinks ? u : u + z.skip;
    const int64_t col = pos / p.page_size;
    bool on = u < u1;
    const int page = on ? p.table[z.row * p.t_sr + col] : 0;
    if (page < 0 || page >= p.pages) {
      bad = 1;
      on = false;
    }
    const int64_t slot = pos - col * p.page_size;
    float kx[kLaneDims], vx[kLaneDims];
    load_dims<T, LPK, VEC>(kb + page * p.k_sp + slot * p.k_st, li, p.d, on, kx);
    load_dims<T, LPK, VEC>(vb + page * p.v_sp + slot * p.v_st, li, p.dv, on, vx);
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < kLaneDims; ++e) s = fmaf(qs[h][lane_dim<LPK, VEC>(li, e)], kx[e], s);
#pragma unroll
      for (int w = LPK / 2; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      if (!on) s = -INFINITY;
      const float top = fmaxf(m[h], s);
      if (top > m[h]) {
        const float f = exp2f(m[h] - top);
        l[h] *= f;
#pragma unroll
        for (int e = 0; e < kLaneDims; ++e) o[h][e] *= f;
        m[h] = top;
      }
      const float w = s == -INFINITY ? 0.f : exp2f(s - top);
      l[h] += w;
      if (on) {
#pragma unroll
        for (int e = 0; e < kLaneDims; ++e) o[h][e] = fmaf(w, vx[e], o[h][e]);
      }
    }
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
// 16-bit kernel: cp.async into swizzled shared memory, m16n8k16 products.
//
// Four warps share an item (one piece of one row for 8 * NH query heads of one
// KV head); warp w takes the 16-token tiles w, w + 4, ....  Every warp has its
// own ring of S stages, each a tile's keys, values and the item's queries, and
// refills a stage as soon as it has used it, across item borders, so the loads
// never wait for the arithmetic.  Per tile:
//   S^T [16 keys x 8 heads] = K [16 x d] Q^T     A: ldmatrix, B: ldmatrix of Q
//   p = 2^(s - m) in the accumulator layout, rounded to T; movmatrix turns its
//   8 x 8 halves into the B operand of
//   O^T [d x 8 heads] += V^T [d x 16] P^T        A: ldmatrix.trans
// Keys are the 16-row side, so a group of 8 heads fills the 8-column side
// exactly and m, l and the rescale factors of a head pair sit in the lane that
// holds that pair of O.  The cache is read once at a few flops per byte: what
// bounds it is HBM, not the products (m16n8k16 covers 2048 products per
// instruction; the tcgen05 tile of 128 rows would be 15/16 padding here).
// ---------------------------------------------------------------------------
constexpr int kMmaWarps = 4;
constexpr int kTile = 16;         // tokens of a tile
constexpr int kListRows = 1024;   // rows whose piece counts fit in shared memory

template <int DP, int NH>
struct PagedSmem {
  static constexpr int kRow = DP * 2;                       // bytes of a token's row
  static constexpr int kStage = 2 * kTile * kRow + 8 * NH * kRow;
  static constexpr int kPitch = DP + 4;                     // floats, spreads the banks
  static constexpr int kPart = kMmaWarps * 8 * NH * kPitch * 4;
  static constexpr int kList = (kListRows + 4) * 4;
  static constexpr int kMisc = kMmaWarps * 8 * NH * 8 + 64 * 4 + kList;
  // two CTAs per SM where two stages fit, else one with as many as fit
  static constexpr int kTwo = (113 * 1024 - kPart - kMisc) / (kMmaWarps * kStage);
  static constexpr int kOne = (226 * 1024 - kPart - kMisc) / (kMmaWarps * kStage);
  static constexpr int kCtas = kTwo >= 2 ? 2 : 1;
  static constexpr int kStages = kTwo >= 2 ? (kTwo > 4 ? 4 : kTwo) : (kOne > 6 ? 6 : kOne);
  static constexpr int kBytes = kPart + kMisc + kMmaWarps * kStages * kStage;
  static_assert(kStages >= 2, "a ring needs two stages");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
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
  int64_t b;       // query
  Visible z;
  int hg;          // KV head * blocks of heads + block
  int64_t piece, pieces;
  int64_t u0;      // first token of the piece
  int tokens;
};

template <typename T, int DP, int NH>
__global__ void __launch_bounds__(kMmaWarps * 32, PagedSmem<DP, NH>::kCtas)
    paged_mma_kernel(const PagedParams p, int64_t batch, int list) {
  using L = PagedSmem<DP, NH>;
  constexpr int S = L::kStages, HB = 8 * NH;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  float* part = reinterpret_cast<float*>(ring + kMmaWarps * S * L::kStage);
  float2* part_ml = reinterpret_cast<float2*>(part + L::kPart / 4);
  int* misc = reinterpret_cast<int*>(part_ml + kMmaWarps * HB);  // [0..31] stage flags, [32..] bad
  int* first = misc + 64;          // list: items before row b, [batch + 1]
  int* scan = misc + 40;           // list: sums of the four warps
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hblocks = (p.group + HB - 1) / HB;
  const int hgs = p.kv_heads * hblocks;

  // columns past d / dv are never written by the copies: zero the ring once
  if (p.d < DP || p.dv < DP) {
    uint4* z = reinterpret_cast<uint4*>(ring);
    for (int i = threadIdx.x; i < kMmaWarps * S * L::kStage / 16; i += blockDim.x)
      z[i] = make_uint4(0, 0, 0, 0);
  }
  auto pieces_of = [&](const Visible& z) -> int64_t {
    const int c = piece_tokens(z.n);
    const int64_t k = (z.n + c - 1) / c;
    return k > 1 ? k : 1;  // an empty or refused row has one item, which writes zeros
  };
  int64_t total = 1;
  if (list) {
    // items of every row, as a running sum in shared memory
    int carry = 0;
    for (int64_t b0 = 0; b0 < batch; b0 += blockDim.x) {
      const int64_t b = b0 + threadIdx.x;
      const int mine = b < batch ? static_cast<int>(pieces_of(visible_of(p, b))) * hgs : 0;
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
      for (int w = 0; w < kMmaWarps; ++w) {
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

  // item number -> what to do; without a list the block has one item
  auto decode = [&](int64_t item, PagedItem& it) {
    int64_t rest;
    if (list) {
      int lo = 0, hi = static_cast<int>(batch);
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= item) lo = mid; else hi = mid;
      }
      it.b = lo;
      rest = item - first[lo];
      it.hg = static_cast<int>(rest % hgs);
      it.piece = rest / hgs;
    } else {
      rest = blockIdx.x;
      it.piece = rest % p.max_pieces;
      rest /= p.max_pieces;
      it.hg = static_cast<int>(rest % hgs);
      it.b = rest / hgs;
    }
    it.z = visible_of(p, it.b);
    const int c = piece_tokens(it.z.n);
    it.pieces = pieces_of(it.z);
    it.u0 = it.piece * c;
    it.tokens = static_cast<int>(max(static_cast<int64_t>(0),
                                     min(static_cast<int64_t>(c), it.z.n - it.u0)));
  };

  // ------------------------------------------------------------- producer side
  // the next tile to fetch: its item, its number, and its tokens' pages
  const uint32_t my_ring = smem_u32(ring) + warp * (S * L::kStage);
  int64_t in_item = list ? blockIdx.x : 0;
  PagedItem in;
  decode(in_item, in);
  const bool dead = !list && in.piece >= in.pieces;
  if (dead) return;
  int in_tile = warp;
  bool in_done = in_item >= total;
  int in_page = -1, in_slot = 0;  // of token `lane` of the tile (lanes 0..15)
  auto look_up = [&]() {
    while (!in_done && in_tile * kTile >= in.tokens) {
      in_item += gridDim.x;
      if (!list || in_item >= total) {
        in_done = true;
      } else {
        decode(in_item, in);
        in_tile = warp;
      }
    }
    in_page = -1;
    if (!in_done && lane < kTile && in_tile * kTile + lane < in.tokens) {
      const int64_t u = in.u0 + in_tile * kTile + lane;
      const int64_t pos = u < in.z.sinks ? u : u + in.z.skip;
      const int col = static_cast<int>(pos / p.page_size);
      in_slot = static_cast<int>(pos - static_cast<int64_t>(col) * p.page_size);
      in_page = p.table[in.z.row * p.t_sr + col];
      if (in_page < 0 || in_page >= p.pages) in_page = -2;  // refused
    }
  };
  const unsigned kc = p.d / 8, vc = p.dv / 8;  // 16-byte chunks of a row
  auto fetch = [&](int stage) {
    if (!in_done) {
      const uint32_t dst = my_ring + stage * L::kStage;
      const int hk = in.hg / hblocks;
      const char* kb = static_cast<const char*>(p.k) + hk * p.k_sh * 2;
      const char* vb = static_cast<const char*>(p.v) + hk * p.v_sh * 2;
      const int lost = __any_sync(0xffffffffu, in_page == -2);
      if (lane == 0) misc[warp * 8 + stage] = lost;
      // DP / 8 chunks per row: a warp covers `rows` rows per step
      constexpr int kChunks = DP / 8;
      constexpr int kRows = kChunks >= 32 ? 1 : 32 / kChunks;
      const unsigned ch = lane % kChunks;
#pragma unroll
      for (int r0 = 0; r0 < kTile; r0 += kRows) {
        const int r = r0 + lane / kChunks;
        const int page = __shfl_sync(0xffffffffu, in_page, r);
        const int slot = __shfl_sync(0xffffffffu, in_slot, r);
        const bool on = page >= 0;
        const uint32_t d = dst + r * L::kRow + ((ch ^ (r & 7)) << 4);
        const char* ks = on ? kb + (page * p.k_sp + slot * p.k_st) * 2 + ch * 16 : kb;
        const char* vs = on ? vb + (page * p.v_sp + slot * p.v_st) * 2 + ch * 16 : vb;
        if (ch < kc) cp_async16(d, ks, on);
        if (ch < vc) cp_async16(d + kTile * L::kRow, vs, on);
      }
      if (in_tile == warp) {  // the item's queries travel with its first tile
        const int h0 = hk * p.group + (in.hg - hk * hblocks) * HB;
        const int nh = min(HB, p.group - (in.hg - hk * hblocks) * HB);
        const char* qb = static_cast<const char*>(p.q) + (in.b * p.q_sb + h0 * p.q_sh) * 2;
#pragma unroll
        for (int r0 = 0; r0 < HB; r0 += kRows) {
          const int r = r0 + lane / kChunks;
          const uint32_t d = dst + 2 * kTile * L::kRow + r * L::kRow + ((ch ^ (r & 7)) << 4);
          if (ch < kc) cp_async16(d, r < nh ? qb + r * p.q_sh * 2 + ch * 16 : qb, r < nh);
        }
      }
      in_tile += kMmaWarps;
      look_up();
    }
    cp_async_commit();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(s);

  // ------------------------------------------------------------- consumer side
  const int ksteps = (p.d + 15) / 16, vsteps = (p.dv + 15) / 16;
  int stage = 0;
  for (int64_t item = list ? blockIdx.x : 0; item < total; item += gridDim.x) {
    PagedItem it;
    decode(item, it);
    const int hk = it.hg / hblocks, hb = it.hg - hk * hblocks;
    const int h0 = hk * p.group + hb * HB, nh = min(HB, p.group - hb * HB);
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
    for (int tile = warp; tile * kTile < it.tokens; tile += kMmaWarps) {
      cp_async_wait<S - 1>();
      __syncwarp();
      const uint32_t sk = my_ring + stage * L::kStage;
      const uint32_t sv = sk + kTile * L::kRow, sq = sv + kTile * L::kRow;
      bad |= misc[warp * 8 + stage];
      if (tile == warp) {
        // B operand: heads in rows of 8, four 8-dim chunks per ldmatrix
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int t = 0; t < DP / 16; t += 2) {
            uint32_t r[4];
            const int row = n * 8 + (lane & 7), ch = t * 2 + (lane >> 3);
            ldsm_x4(sq + row * L::kRow + ((ch ^ (row & 7)) << 4), r);
            qf[t][n][0] = r[0];
            qf[t][n][1] = r[1];
            qf[t + 1][n][0] = r[2];
            qf[t + 1][n][1] = r[3];
          }
      }
      float s[NH][4];
#pragma unroll
      for (int n = 0; n < NH; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) {
        if (t < ksteps) {
          uint32_t a[4];
          const int row = lane & 15, ch = t * 2 + (lane >> 4);
          ldsm_x4(sk + row * L::kRow + ((ch ^ (row & 7)) << 4), a);
#pragma unroll
          for (int n = 0; n < NH; ++n) mma16816<T>(s[n], a, qf[t][n][0], qf[t][n][1]);
        }
      }
      // rows of s: keys lane / 4 and lane / 4 + 8; columns: heads 2 (lane % 4) + {0, 1}
      const int left = it.tokens - tile * kTile;
      const bool on0 = (lane >> 2) < left, on1 = (lane >> 2) + 8 < left;
      uint32_t pf[NH][2];
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float s0 = on0 ? s[n][e] * p.scale_log2 : -INFINITY;
          const float s1 = on1 ? s[n][2 + e] * p.scale_log2 : -INFINITY;
          float top = fmaxf(s0, s1);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          top = fmaxf(top, m[n][e]);
          f[e] = m[n][e] == -INFINITY ? 0.f : exp2f(m[n][e] - top);
          m[n][e] = top;
          s[n][e] = s0 == -INFINITY ? 0.f : exp2f(s0 - top);
          s[n][2 + e] = s1 == -INFINITY ? 0.f : exp2f(s1 - top);
        }
        float r00, r01, r10, r11;
        pf[n][0] = mov_trans(pack2<T>(s[n][0], s[n][1], r00, r01));
        pf[n][1] = mov_trans(pack2<T>(s[n][2], s[n][3], r10, r11));
        l[n][0] = l[n][0] * f[0] + (r00 + r10);
        l[n][1] = l[n][1] * f[1] + (r01 + r11);
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
        if (t < vsteps) {
          uint32_t a[4];
          const int i = lane >> 3, row = (lane & 7) + (i & 2) * 4, ch = t * 2 + (i & 1);
          ldsm_x4_t(sv + row * L::kRow + ((ch ^ (row & 7)) << 4), a);
#pragma unroll
          for (int n = 0; n < NH; ++n) mma16816<T>(o[t][n], a, pf[n][0], pf[n][1]);
        }
      }
      __syncwarp();
      fetch(stage);
      stage = stage + 1 == S ? 0 : stage + 1;
    }
    // ------------------------------------------------------- the item's result
#pragma unroll
    for (int n = 0; n < NH; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], w);
        const int h = n * 8 + 2 * (lane & 3) + e;
        if (lane < 4) part_ml[warp * HB + h] = make_float2(m[n][e], l[n][e]);
        float* row = part + (warp * HB + h) * L::kPitch + (lane >> 2);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
          if (t < vsteps) {
            row[t * 16] = o[t][n][e];
            row[t * 16 + 8] = o[t][n][2 + e];
          }
        }
      }
    }
    bad = __syncthreads_or(bad);
    if (bad && threadIdx.x == 0) raise_status(p.status, BIO_DEV_INDEX);
    const int quads = p.dv / 4;
    for (int i = threadIdx.x; i < nh * quads; i += blockDim.x) {
      const int h = i / quads, e = (i - h * quads) * 4;
      float top = -INFINITY, w[kMmaWarps], sum = 0.f;
#pragma unroll
      for (int x = 0; x < kMmaWarps; ++x) top = fmaxf(top, part_ml[x * HB + h].x);
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < kMmaWarps; ++x) {
        const float2 ml = part_ml[x * HB + h];
        w[x] = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
        sum = fmaf(ml.y, w[x], sum);
        const float4 a =
            *reinterpret_cast<const float4*>(part + (x * HB + h) * L::kPitch + e);
        y.x = fmaf(a.x, w[x], y.x);
        y.y = fmaf(a.y, w[x], y.y);
        y.z = fmaf(a.z, w[x], y.z);
        y.w = fmaf(a.w, w[x], y.w);
      }
      const int64_t bh = it.b * p.heads + h0 + h;
      if (it.pieces == 1) {
        const bool none = bad || sum == 0.f;
        T* out = static_cast<T*>(p.o) + it.b * p.o_sb + (h0 + h) * p.o_sh + e;
        out[0] = from_f32<T>(none ? 0.f : y.x / sum);
        out[1] = from_f32<T>(none ? 0.f : y.y / sum);
        out[2] = from_f32<T>(none ? 0.f : y.z / sum);
        out[3] = from_f32<T>(none ? 0.f : y.w / sum);
      } else {
        *reinterpret_cast<float4*>(p.acc + (bh * p.max_pieces + it.piece) * p.dvp + e) = y;
        if (e == 0) p.ml[bh * p.max_pieces + it.piece] = make_float2(top, bad ? -1.f : sum);
      }
    }
    __syncthreads();  // the partial results are free for the next item
  }
  cp_async_wait<0>();
}

// ---------------------------------------------------------------------------
// Joins the pieces of one (row, head): weights e^(m_i - max m), eight warps
// take the pieces i = warp, warp + 8, ... and are added in order.
// ---------------------------------------------------------------------------
constexpr int kJoinWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const PagedParams p) {
  __shared__ float4 part[kJoinWarps][64];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t bh = blockIdx.x, b = bh / p.heads, h = bh - b * p.heads;
  const Visible z = visible_of(p, b);
  const int c = piece_tokens(z.n);
  const int pieces = static_cast<int>((z.n + c - 1) / c);
  if (pieces <= 1) return;
  const float2* ml = p.ml + bh * p.max_pieces;
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

  const int groups = p.dvp / 4;  // four-float groups of an output row, <= 64
  const float4* acc = reinterpret_cast<const float4*>(p.acc + bh * p.max_pieces * p.dvp);
  float4 y[2];
  y[0] = y[1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = warp; i < pieces; i += kJoinWarps) {
    const float f = ml[i].x == -INFINITY ? 0.f : exp2f(ml[i].x - top);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if (lane + 32 * g >= groups) continue;
      const float4 a = acc[static_cast<int64_t>(i) * groups + lane + 32 * g];
      y[g].x = fmaf(a.x, f, y[g].x);
      y[g].y = fmaf(a.y, f, y[g].y);
      y[g].z = fmaf(a.z, f, y[g].z);
      y[g].w = fmaf(a.w, f, y[g].w);
    }
  }
#pragma unroll
  for (int g = 0; g < 2; ++g)
    if (lane + 32 * g < groups) part[warp][lane + 32 * g] = y[g];
  __syncthreads();
  T* out = static_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh;
  const float* flat = reinterpret_cast<const float*>(part);
  for (int e = threadIdx.x; e < p.dv; e += blockDim.x) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) a += flat[w * 256 + e];
    out[e] = from_f32<T>(bad || sum == 0.f ? 0.f : a / sum);
  }
}

}  // namespace bio

namespace {

constexpr int64_t kMaxGrid = 2147483647;

// Most pieces that a row can have when it sees up to `most` tokens.
int64_t most_pieces(int64_t most) {
  int64_t pieces = 1;
  for (int64_t top : {static_cast<int64_t>(1024), static_cast<int64_t>(8192),
                      static_cast<int64_t>(32768), most}) {
    const int64_t n = top < most ? top : most;
    const int c = bio::piece_tokens(n);
    const int64_t k = (n + c - 1) / c;
    if (k > pieces) pieces = k;
  }
  return pieces;
}

struct Split {
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
  int64_t most = a->table_width * a->page_size;
  if (a->window > 0 && a->window + a->sinks < most) most = a->window + a->sinks;
  s->pieces = most_pieces(most);
  s->dvp = (a->dv + 3) / 4 * 4;
  if (a->batch > kMaxGrid / a->heads || a->batch * a->heads > kMaxGrid / s->pieces)
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

template <typename T, bool VEC>
int dispatch_simt(const bio::PagedParams& p, int64_t batch, cudaStream_t s) {
  const bool wide = p.d > 128 || p.dv > 128;
  if (p.group >= 3)
    return wide ? launch_simt<T, 4, 16, VEC>(p, batch, s) : launch_simt<T, 4, 8, VEC>(p, batch, s);
  if (p.group == 2)
    return wide ? launch_simt<T, 2, 16, VEC>(p, batch, s) : launch_simt<T, 2, 8, VEC>(p, batch, s);
  return wide ? launch_simt<T, 1, 16, VEC>(p, batch, s) : launch_simt<T, 1, 8, VEC>(p, batch, s);
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
  const int64_t slots = static_cast<int64_t>(bio_host::sm_count(device)) * L::kCtas;
  const int64_t items =
      batch * p.kv_heads * ((p.group + 8 * NH - 1) / (8 * NH)) * p.max_pieces;
  // A block per possible item when they run in a few rounds: blocks of pieces
  // that a row does not have end at once.  Beyond, every block builds the list
  // of the items that exist and walks it.
  const bool list = items > 4 * slots && batch <= bio::kListRows;
  const int64_t grid = list ? slots : items;
  if (slots <= 0) return BIO_ERR_LAUNCH;
  bio::paged_mma_kernel<T, DP, NH>
      <<<static_cast<unsigned>(grid), bio::kMmaWarps * 32, L::kBytes, s>>>(p, batch, list ? 1 : 0);
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
int run(const bio::PagedParams& p, int64_t batch, cudaStream_t s) {
  int st;
  if constexpr (sizeof(T) == 4) {
    const uint64_t bits = reinterpret_cast<uint64_t>(p.k) | reinterpret_cast<uint64_t>(p.v) |
                          4 * static_cast<uint64_t>(p.k_sp | p.k_sh | p.k_st | p.v_sp | p.v_sh |
                                                    p.v_st | p.d | p.dv);
    st = bits % 16 == 0 ? dispatch_simt<T, true>(p, batch, s)
                        : dispatch_simt<T, false>(p, batch, s);
  } else {
    const uint64_t bits = reinterpret_cast<uint64_t>(p.q) | reinterpret_cast<uint64_t>(p.k) |
                          reinterpret_cast<uint64_t>(p.v) |
                          2 * static_cast<uint64_t>(p.q_sb | p.q_sh | p.k_sp | p.k_sh | p.k_st |
                                                    p.v_sp | p.v_sh | p.v_st | p.d | p.dv);
    st = bits % 16 == 0 ? dispatch_mma<T>(p, batch, s) : dispatch_simt<T, false>(p, batch, s);
  }
  if (st != BIO_OK || p.max_pieces == 1) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * p.heads));
  cfg.blockDim = dim3(bio::kJoinWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return bio_host::launch_status(cudaLaunchKernelEx(&cfg, bio::paged_join_kernel<T>, p));
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
  p.window = a->window; p.sinks = a->sinks;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.max_pieces = s.pieces;
  p.dvp = s.dvp;
  p.acc = static_cast<float*>(workspace);
  p.ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + s.acc_bytes);
  p.status = bio_host::status_word(a->device);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case BIO_F32: return run<float>(p, a->batch, cs);
    case BIO_F16: return run<__half>(p, a->batch, cs);
    case BIO_BF16: return run<__nv_bfloat16>(p, a->batch, cs);
    default: return BIO_ERR_DTYPE;
  }
}

}  // extern "C"
