// Prefill attention with a sliding window and sink tokens (dense and packed).
//
// Query i sits at position p = i + (lk - lq) and sees key j iff j <= p and
// (j > p - window or j < sinks):
//   o_i = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q_i.k_j.
// A row that sees no key (p < 0) gives zeros.
//
// 16-bit operands run on tcgen05 (window_tc_kernel), fp32 on the CUDA cores
// (window_row_kernel).
//
// Not in the reference, whose SDPA (batch_invariant_ops.py:1148-1213) would
// need the mask as a tensor and visits every key.
#include <algorithm>
#include <mutex>

#include "bio_tile.cuh"

namespace bio {

struct WindowParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st, o_sb, o_sh, o_st;
  int64_t batch, heads, group, lq, lk;  // packed: total query / key tokens
  int d, dv;
  float scale;
  int64_t window, sinks;
  const void* cu_q;
  const void* cu_k;
  int cu_is64;
  int64_t nseq;
  int* status;
};

__device__ __forceinline__ int64_t win_off(const void* p, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i]
              : static_cast<int64_t>(static_cast<const int*>(p)[i]);
}

constexpr int kWinWarps = 8;
constexpr int kWinDims = 256;

// One warp computes one row.  It walks the row's visible keys in order, 32 at a
// time: lane j computes the score of key j, the maximum and the sum of
// exponentials use a fixed xor-shuffle tree, and lane t accumulates output
// columns t, t + 32, ....  Keys that the row does not see are never read.
// `pos` is the query's position; kb and vb point at key 0 of its sequence.
template <typename T>
__device__ __noinline__ void window_row(const T* qrow, const T* kb, const T* vb, T* out,
                                        int64_t k_st, int64_t v_st, int d, int dv, float scale,
                                        int64_t window, int64_t sinks, int64_t pos) {
  const int lane = threadIdx.x & 31;
  // visible keys u = 0..n-1: key u < few ? u : u + skip
  const int64_t lo = max(static_cast<int64_t>(0), pos - window + 1);
  const int64_t few = min(sinks, lo), skip = lo - few;
  const int64_t n = max(static_cast<int64_t>(0), pos + 1 - skip);
  float m = -INFINITY, l = 0.f, o[kWinDims / 32];
#pragma unroll
  for (int e = 0; e < kWinDims / 32; ++e) o[e] = 0.f;
  for (int64_t u0 = 0; u0 < n; u0 += 32) {
    const int64_t u = u0 + lane;
    float s = -INFINITY;
    if (u < n) {
      const T* krow = kb + (u < few ? u : u + skip) * k_st;
      float a = 0.f;
      for (int c = 0; c < d; ++c) a = fmaf(to_f32(qrow[c]), to_f32(krow[c]), a);
      s = a * scale;
    }
    float top = s;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    top = fmaxf(top, m);
    const float f = m == -INFINITY ? 0.f : expf(m - top);
    const float w = s == -INFINITY ? 0.f : expf(s - top);
    float sum = w;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * f + sum;
    m = top;
#pragma unroll
    for (int e = 0; e < kWinDims / 32; ++e) o[e] *= f;
    const int keys = static_cast<int>(min(static_cast<int64_t>(32), n - u0));
    for (int j = 0; j < keys; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const int64_t uj = u0 + j;
      const T* vrow = vb + (uj < few ? uj : uj + skip) * v_st;
#pragma unroll
      for (int e = 0; e < kWinDims / 32; ++e) {
        const int c = lane + 32 * e;
        if (c < dv) o[e] = fmaf(wj, to_f32(vrow[c]), o[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < kWinDims / 32; ++e) {
    const int c = lane + 32 * e;
    if (c < dv) out[c] = from_f32<T>(l == 0.f ? 0.f : o[e] / l);
  }
}

template <typename T, bool PACKED>
__global__ void __launch_bounds__(kWinWarps * 32) window_row_kernel(const WindowParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWinWarps + warp;
  if (row >= (PACKED ? 1 : p.batch) * p.heads * p.lq) return;
  const int64_t t = row % p.lq, bh = row / p.lq, h = bh % p.heads, b = bh / p.heads;
  int64_t pos = t + p.lk - p.lq, k0 = 0;  // position of the query, first key token
  if constexpr (PACKED) {
    int64_t lo = 0, hi = p.nseq;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (win_off(p.cu_q, p.cu_is64, mid) <= t) lo = mid; else hi = mid;
    }
    if (p.nseq < 1) return;
    const int64_t q0 = win_off(p.cu_q, p.cu_is64, lo), q1 = win_off(p.cu_q, p.cu_is64, lo + 1);
    k0 = win_off(p.cu_k, p.cu_is64, lo);
    const int64_t k1 = win_off(p.cu_k, p.cu_is64, lo + 1);
    if (t >= win_off(p.cu_q, p.cu_is64, p.nseq)) return;  // outside every sequence
    if (q0 > t || q1 <= t || q1 > p.lq || k0 < 0 || k1 < k0 || k1 > p.lk ||
        win_off(p.cu_q, p.cu_is64, 0) != 0 || win_off(p.cu_k, p.cu_is64, 0) != 0) {
      if (lane == 0) raise_status(p.status, BIO_DEV_INDEX);
      return;
    }
    pos = (t - q0) + (k1 - k0) - (q1 - q0);
  }
  const int64_t bq = PACKED ? 0 : b;
  window_row<T>(static_cast<const T*>(p.q) + bq * p.q_sb + h * p.q_sh + t * p.q_st,
                static_cast<const T*>(p.k) + bq * p.k_sb + h / p.group * p.k_sh + k0 * p.k_st,
                static_cast<const T*>(p.v) + bq * p.v_sb + h / p.group * p.v_sh + k0 * p.v_st,
                static_cast<T*>(p.o) + bq * p.o_sb + h * p.o_sh + t * p.o_st, p.k_st, p.v_st, p.d,
                p.dv, p.scale, p.window, p.sinks, pos);
}

// ---------------------------------------------------------------------------
// tcgen05 kernel.
//
// A job is a tile of 128 query rows that share a KV head: `gh` query heads of
// the group with `tok` = 128 / gh consecutive tokens each (row r: head r / tok,
// token r % tok), so the keys that a tile visits are its window plus tok - 1, not
// plus 127, and a key block is loaded once for all those heads.  Jobs are dealt
// out round robin to one persistent CTA per SM:
//   warp 0      TMA: Q, then K and V blocks of BN keys through one ring.
//   warp 1      MMA: S = Q K^T into one of three buffers, O += P V, fp32 in TMEM;
//               P (16 bits) lies over the S that it came from.
//   warps 4-11  softmax: two groups of 128 threads, a thread per query row, take
//               the blocks in turn.
// S of block i + 2 is issued before PV of block i, so each group finds its next
// scores ready while the other one and the tensor cores are at work, and nobody
// waits for one chain.  The groups hand the rows' running reference m to each
// other right after a block's maximum; each keeps its own sum l.  The ring, S and
// O run on across jobs: a job's first blocks start while the last rows of the
// one before are still being stored.
//
// What was measured on the way (32768 tokens, 32 heads on 8, d 128, window 1024):
// two tiles with one S buffer each 842 us, bound by the chain softmax -> PV -> S of
// a tile (4900 clocks a round, 3200 of them products: an M = 128, K = 16 product
// takes about 100 clocks at N = 64 as at N = 128); two threads per row 838 us (the
// two tiles' exponentials then run at the same time, and the special-function
// unit is what both want); 64-key blocks with two buffers per tile 977 us (twice
// the products).
//
// Blocks are cut on the absolute grid of BN keys and trimmed to the 32-key
// columns that some row of the tile sees: a window costs about window + tok + 32
// columns per row, four sink tokens one 32-key column.  Masked scores weigh
// exactly 0 and untrimmed columns add exactly 0, so a row's bits depend on its
// own query, keys and position only.
//
// Scores, maxima and sums are fp32 in registers.  The reference m of the
// exponentials moves only when a block's maximum exceeds it by more than 8
// (log2), so O is rarely rescaled and P stays below 2^8; P is rounded to the
// operand type, as the product needs, l sums it unrounded.
//
// A hidden key in a visited block has weight 0, but 0 * Inf or 0 * NaN in V
// would still reach the row: a row whose output is not finite is computed once
// more, by its warp, from its visible keys alone (window_row).  Keys of a
// neighbouring packed sequence are zeroed in shared memory instead, so that
// they cannot even change a row's bits.
// ---------------------------------------------------------------------------
struct WindowJobs {
  int gh, tok, hblocks;  // heads and tokens of a tile, tiles across a group
  int qblocks;           // dense: blocks of tok tokens per sequence; packed: at most
  int jobs;
  int window, sinks;     // at most 2^30
  float scale_log2;      // > 0
  int negate;            // the scale was negative: scores change sign
  int vec_out;           // output rows take 16-byte stores
};

template <int DP>
struct WinSmem {
  static constexpr int BN = DP == 256 ? 64 : 128;  // keys of a block
  static constexpr uint32_t kQ = 128 * DP * 2;
  static constexpr uint32_t kSlot = BN * DP * 2;   // K or V of a block
  static constexpr uint32_t kSwap = 4 * 128 * 4;   // m of two groups, l of two jobs
  static constexpr int kFit = (227 * 1024 - 1024 - 512 - static_cast<int>(kSwap + kQ)) /
                              static_cast<int>(kSlot);
  static constexpr int kSlots = kFit > 12 ? 12 : kFit;
  static constexpr uint32_t kBytes = 1024 + kQ + kSlots * kSlot + 512 + kSwap;
  static constexpr int kThreads = 384;
  static constexpr uint32_t kO = DP == 256 ? 256 : 384;  // TMEM columns of O; S buffers x at x * BN
  static_assert(kSlots >= 4, "K of three blocks and a V");
};

struct WinJob {
  int b, hk, h0, nh;        // sequence of the batch, KV head, query heads
  int q0, lq, lk;           // first query of the tile, lengths of its sequence
  int qt, kt;               // tokens of the operands at which the sequence starts
  int pf, n;                // position of the tile's first token, number of tokens
  int lo, hi, sx;           // keys: [lo, hi) for the windows of its rows, [0, sx) sinks before
  int head, jump, blocks;   // block i of the job is block i < head ? i : i + jump of the keys
};

template <int BN>
__device__ __forceinline__ void window_plan(const WindowJobs& w, WinJob& j) {
  j.n = max(0, min(w.tok, j.lq - j.q0));
  j.pf = j.q0 + j.lk - j.lq;
  j.hi = j.n > 0 ? max(0, j.pf + j.n) : 0;
  j.lo = j.hi > 0 ? max(0, j.pf - w.window + 1) : 0;
  j.sx = min(w.sinks, j.lo);
  j.head = (j.sx + BN - 1) / BN;
  j.jump = max(0, j.lo / BN - j.head);
  j.blocks = j.hi == 0 ? 0 : (j.hi - 1) / BN + 1 - j.jump;
}

// Columns [x, y) of the job's block i that some row sees, on the 32-column grid.
template <int BN>
__device__ __forceinline__ int2 window_span(const WinJob& j, int i) {
  const int base = (i < j.head ? i : i + j.jump) * BN;
  int x = max(j.lo - base, 0), y = min(j.hi - base, BN);
  if (x >= y) x = y = 0;
  const int s = min(j.sx - base, BN);
  if (s > 0) {
    x = 0;
    y = max(y, s);
  }
  return make_int2(x & ~31, (y + 31) & ~31);
}

// Blocks x <= i < y of the job: every row sees every key by its window, and all
// 128 rows exist (or are padding of the tile's shape).
template <int BN>
__device__ __forceinline__ int2 window_whole(const WindowJobs& w, const WinJob& j) {
  if (w.negate || j.n < w.tok || j.nh < w.gh || j.pf < 0) return make_int2(0, 0);
  const int x = (max(0, j.pf + j.n - w.window) + BN - 1) / BN;  // first inside the last window
  const int y = (j.pf + 1) / BN;                                // first past the first row
  // only what lies behind the sinks' blocks keeps its distance
  return make_int2(max(x, j.head + j.jump) - j.jump, y - j.jump);
}

// Job number -> job.  All lanes of the warp call it; false: no such job.
template <int BN, bool PACKED>
__device__ __forceinline__ bool window_job(const WindowParams& p, const WindowJobs& w, int number,
                                           WinJob& j) {
  const int lane = threadIdx.x & 31;
  const int tiles = static_cast<int>(p.heads / p.group) * w.hblocks;
  int qb, hx;
  if constexpr (!PACKED) {
    const int rest = number / w.qblocks;
    qb = number - rest * w.qblocks;
    j.b = rest / tiles;
    hx = rest - j.b * tiles;
    j.lq = static_cast<int>(p.lq);
    j.lk = static_cast<int>(p.lk);
    j.qt = j.kt = 0;
  } else {
    qb = number / tiles;
    hx = number - qb * tiles;
    j.b = 0;
    if (win_off(p.cu_q, p.cu_is64, 0) != 0 || win_off(p.cu_k, p.cu_is64, 0) != 0) {
      raise_status(p.status, BIO_DEV_INDEX);
      return false;
    }
    // 32 sequences at a time: the one whose blocks hold block qb
    const int span = w.tok;
    bool found = false;
    for (int64_t s0 = 0; s0 < p.nseq && !found; s0 += 32) {
      const int64_t s = s0 + lane;
      int64_t qa = 0, qz = 0, ka = 0, kz = 0;
      int n = 0;
      if (s < p.nseq) {
        qa = win_off(p.cu_q, p.cu_is64, s);
        qz = win_off(p.cu_q, p.cu_is64, s + 1);
        ka = win_off(p.cu_k, p.cu_is64, s);
        kz = win_off(p.cu_k, p.cu_is64, s + 1);
        if (qa < 0 || qz < qa || qz > p.lq || ka < 0 || kz < ka || kz > p.lk)
          raise_status(p.status, BIO_DEV_INDEX);
        else
          n = static_cast<int>((qz - qa + span - 1) / span);
      }
      int inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const unsigned past = __ballot_sync(0xffffffffu, inc > qb);
      if (past == 0) {
        qb -= __shfl_sync(0xffffffffu, inc, 31);
        continue;
      }
      const int f = __ffs(past) - 1;
      qb -= __shfl_sync(0xffffffffu, inc - n, f);
      j.lq = __shfl_sync(0xffffffffu, static_cast<int>(qz - qa), f);
      j.lk = __shfl_sync(0xffffffffu, static_cast<int>(kz - ka), f);
      j.qt = __shfl_sync(0xffffffffu, static_cast<int>(qa), f);
      j.kt = __shfl_sync(0xffffffffu, static_cast<int>(ka), f);
      found = true;
    }
    if (!found) return false;
  }
  j.q0 = qb * w.tok;
  j.hk = hx / w.hblocks;
  const int before = (hx - j.hk * w.hblocks) * w.gh;
  j.h0 = j.hk * static_cast<int>(p.group) + before;
  j.nh = min(w.gh, static_cast<int>(p.group) - before);
  window_plan<BN>(w, j);
  return true;
}

__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// The MMA warp runs in step and one elected thread issues the tcgen05
// instructions, so that waits, spans and descriptors stay uniform.
__device__ __forceinline__ bool elect_leader() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is != 0;
}
__device__ __forceinline__ void commit_to(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}

__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void split_pair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_two(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_two<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack_two<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Bits [x, y) of a 32-bit word, x and y anywhere.
__device__ __forceinline__ uint32_t bits_between(int x, int y) {
  const int a = min(max(x, 0), 32), b = min(max(y, 0), 32);
  const uint64_t below_b = (1ull << b) - 1, below_a = (1ull << a) - 1;
  return static_cast<uint32_t>(below_b & ~below_a);
}

// 32 lanes x 8 columns of TMEM, the load waited for.
__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}

// Shared-space addresses of the barriers (8 bytes each).
struct WinBars {
  uint32_t base;
  __device__ uint32_t full(int s) const { return base + s * 8; }
  __device__ uint32_t empty(int s) const { return base + 96 + s * 8; }
  __device__ uint32_t s_full(int x) const { return base + 192 + x * 8; }
  __device__ uint32_t p_ready(int x) const { return base + 216 + x * 8; }
  __device__ uint32_t pv_done(int x) const { return base + 400 + x * 8; }
  __device__ uint32_t l_ready(int x) const { return base + 256 + x * 8; }
  __device__ uint32_t q_full() const { return base + 272; }
  __device__ uint32_t q_empty() const { return base + 280; }
  __device__ uint32_t o_done() const { return base + 288; }
  __device__ uint32_t o_free() const { return base + 296; }
  __device__ uint32_t all_done(int x) const { return base + 304 + x * 8; }
  __device__ uint32_t m_ready(int group, int quarter) const {
    return base + 320 + group * 32 + quarter * 8;
  }
};

// The ring of a job of n blocks carries K0 K1 K2 V0 K3 V1 ..., the order in which
// the products need them: the places of K and V of block i.
__device__ __forceinline__ int ring_of_k(int i) { return i < 3 ? i : 2 * i - 2; }
__device__ __forceinline__ int ring_of_v(int i, int n) { return min(i + 3, n) + i; }

template <typename T, int DP, bool PACKED>
__global__ void __launch_bounds__(WinSmem<DP>::kThreads, 1)
    window_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const WindowParams p,
                     const WindowJobs w) {
  using L = WinSmem<DP>;
  constexpr int BN = L::BN, NS = L::kSlots, NC = BN / 32;
  constexpr uint32_t kFmt = std::is_same<T, __half>::value ? 0u : 1u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* ring = smem + L::kQ;
  uint8_t* tail = ring + NS * L::kSlot;
  const uint32_t q32 = smem_u32(smem), ring32 = smem_u32(ring);
  const WinBars bar{smem_u32(tail)};
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 384);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 388);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kc = (p.d + 63) / 64, vc = (p.dv + 63) / 64;

  if (threadIdx.x == 0) {
    uint64_t* b = reinterpret_cast<uint64_t*>(tail);
    // p_ready, l_ready and o_free: four warps arrive
    for (int i = 0; i < 53; ++i) {
      if (i == 48 || i == 49) continue;  // the TMEM address and the abort flag
      mbar_init(b + i, (i >= 27 && i < 30) || i == 32 || i == 33 || i == 37 ? 4 : 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // All 512 columns of TMEM start at address 0, which as a constant costs the MMA
  // warp no move to a uniform register.
  constexpr uint32_t tmem = 0;
  if (*tmem_slot != tmem) {  // the same for every thread
    if (threadIdx.x == 0) raise_status(p.status, BIO_DEV_TIMEOUT);
    if (warp == 1) tmem_dealloc(*tmem_slot, 512);
    return;
  }
  auto wait = [&](uint32_t b, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, parked_wait(b, parity & 1u, abort_flag, p.status));
  };

  // 384 threads start with 168 registers each, 128 of them go on with 56 and
  // 256 with 216: 62464 of the 64512
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // -------------------------------------------------------------- producer
      int slot = 0, count = 0, q_used = 0;  // ring position; blocks, queries loaded so far
      uint32_t turn = 0;
      bool ok = true;
      for (int number = blockIdx.x; ok && number < w.jobs; number += gridDim.x) {
        WinJob j;
        if (!window_job<BN, PACKED>(p, w, number, j)) continue;
        auto load = [&](bool key, int i) {
          const int2 s = window_span<BN>(j, i);
          const int chunks = key ? kc : vc, boxes = chunks * ((s.y - s.x) / 32);
          ok = wait(bar.empty(slot), turn ^ 1u);
          if (!ok) return;
          if (lane == 0) expect_bytes(bar.full(slot), boxes * 32 * 128);
          __syncwarp();
          if (lane < boxes) {
            const int c = lane % chunks, r = s.x + lane / chunks * 32;
            load_box(ring32 + slot * L::kSlot + c * (BN * 128) + r * 128, key ? &tmK : &tmV,
                     bar.full(slot), c * 64, j.kt + (i < j.head ? i : i + j.jump) * BN + r, j.hk,
                     j.b);
          }
          ++count;
          if (++slot == NS) {
            slot = 0;
            turn ^= 1u;
          }
        };
        const int n = j.blocks;
        if (n == 0) continue;
        load(true, 0);
        if (ok) ok = wait(bar.q_empty(), q_used ^ 1);
        if (!ok) break;
        if (lane == 0) {
          expect_bytes(bar.q_full(), kc * w.gh * w.tok * 128);
          for (int c = 0; c < kc; ++c)
            load_box(q32 + c * 16384, &tmQ, bar.q_full(), c * 64, j.qt + j.q0, j.h0, j.b);
        }
        ++q_used;
        if (n > 1) load(true, 1);
        for (int i = 0; ok && i < n; ++i) {
          if (i + 2 < n) load(true, i + 2);
          if (ok) load(false, i);
        }
      }
      // every copy has to land before the block's shared memory goes
      if (lane == 0) {
        for (int i = max(0, count - NS); i < count; ++i)
          if (!mbar_wait_drain(reinterpret_cast<uint64_t*>(tail) + i % NS, (i / NS) & 1))
            raise_status(p.status, BIO_DEV_TIMEOUT);
        if (q_used > 0 &&
            !mbar_wait_drain(reinterpret_cast<uint64_t*>(tail) + 34, (q_used - 1) & 1))
          raise_status(p.status, BIO_DEV_TIMEOUT);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------- S products
      int before = 0, jobs_done = 0;        // blocks and jobs so far
      bool ok = true;
      for (int number = blockIdx.x; ok && number < w.jobs; number += gridDim.x) {
        WinJob j;
        if (!window_job<BN, PACKED>(p, w, number, j)) continue;
        const int n = j.blocks;
        if (n == 0) continue;
        const int2 open = window_whole<BN>(w, j);
        ok = wait(bar.q_full(), jobs_done);
        for (int i = 0; ok && i < n; ++i) {
          const int g = before + i, x = g % 3, pos = 2 * before + ring_of_k(i), slot = pos % NS;
          const int2 s = i >= open.x && i < open.y ? make_int2(0, BN) : window_span<BN>(j, i);
          const uint32_t idesc = idesc_f16(kFmt, 128, s.y - s.x, false, false);
          const uint64_t qd = smem_desc_sw128(q32, 16, 1024);
          const uint64_t kd = smem_desc_sw128(ring32 + slot * L::kSlot + s.x * 128, 16, 1024);
          const uint32_t to = tmem + x * BN + s.x;
          ok = wait(bar.full(slot), pos / NS);
          // the P before in this buffer has been used
          if (ok && g >= 3) ok = wait(bar.pv_done(x), g / 3 - 1);
          if (!ok) break;
          tc_fence_after();
          if (elect_leader()) {
            // 16 columns are 32 bytes, 2 units of a descriptor; 64 columns a chunk
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
              if (DP == 64 || (k >> 2) < kc)
                umma_f16(to, qd + (k >> 2) * 1024 + (k & 3) * 2,
                         kd + (k >> 2) * (BN * 8) + (k & 3) * 2, idesc, k > 0 ? 1u : 0u);
            commit_to(bar.s_full(x));
            commit_to(bar.empty(slot));  // the keys are free once the products are done
            if (i == n - 1) commit_to(bar.q_empty());
          }
          __syncwarp();
        }
        before += n;
        ++jobs_done;
      }
      if (elect_leader()) commit_to(bar.all_done(0));
      if (!mbar_wait_drain(reinterpret_cast<uint64_t*>(tail) + 38, 0))
        raise_status(p.status, BIO_DEV_TIMEOUT);
    } else if (warp == 2) {
      // ------------------------------------------------------------ PV products
      int before = 0, jobs_done = 0;
      bool ok = true;
      for (int number = blockIdx.x; ok && number < w.jobs; number += gridDim.x) {
        WinJob j;
        if (!window_job<BN, PACKED>(p, w, number, j)) continue;
        const int n = j.blocks;
        if (n == 0) continue;
        const int2 open = window_whole<BN>(w, j);
        for (int i = 0; ok && i < n; ++i) {
          const int g = before + i, x = g % 3, pos = 2 * before + ring_of_v(i, n), slot = pos % NS;
          const int2 s = i >= open.x && i < open.y ? make_int2(0, BN) : window_span<BN>(j, i);
          // 16 keys are 2048 bytes of V and 8 columns of P
          const uint64_t vd = smem_desc_sw128(ring32 + slot * L::kSlot, BN * 128, 1024);
          const uint32_t pa = tmem + x * BN;
          const uint32_t idesc = idesc_f16(kFmt, 128, vc * 64, false, true);
          ok = wait(bar.full(slot), pos / NS);
          // the rows of the job before have left O
          if (ok && i == 0 && jobs_done > 0) ok = wait(bar.o_free(), jobs_done - 1);
          if (ok) ok = wait(bar.p_ready(x), g / 3);
          if (!ok) break;
          tc_fence_after();
          if (elect_leader()) {
#pragma unroll
            for (int k = 0; k < BN / 16; ++k)
              if (k * 16 >= s.x && k * 16 < s.y)
                umma_f16_ts(tmem + L::kO, pa + k * 8, vd + k * 128, idesc,
                            i > 0 || k * 16 > s.x ? 1u : 0u);
            commit_to(bar.pv_done(x));
            commit_to(bar.empty(slot));
            if (i == n - 1) commit_to(bar.o_done());
          }
          __syncwarp();
        }
        before += n;
        ++jobs_done;
      }
      if (elect_leader()) commit_to(bar.all_done(1));
      if (!mbar_wait_drain(reinterpret_cast<uint64_t*>(tail) + 39, 0))
        raise_status(p.status, BIO_DEV_TIMEOUT);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ----------------------------------------------------------------- softmax
    const int group = (warp - 4) >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the tile: the warp's quarter of the lanes
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // (quarter * 32) << 16
    const uint32_t o_at = tmem + lanes + L::kO;
    const int rh = r / w.tok, rt = r - rh * w.tok;
    const uint64_t scale2 = pair_of(w.scale_log2, w.scale_log2);
    float* m_of = reinterpret_cast<float*>(tail + 512);  // [group][row]
    float* l_of = m_of + 256;                            // [job & 1][row]
    // m goes from warp to warp: of a quarter of the rows, from group to group
    const uint32_t give = bar.m_ready(group, warp & 3), take = bar.m_ready(group ^ 1, warp & 3);
    uint32_t taken = 0;                        // times that this warp took m
    int blocks_before = 0, jobs_done = 0, sums_left = 0;
    // After a wait that ran out the rest goes through without waiting for anything.
    bool ok = true;
    auto hold = [&](uint32_t b, uint32_t parity) {
      if (ok) ok = wait(b, parity);
    };
    for (int number = blockIdx.x; number < w.jobs; number += gridDim.x) {
      WinJob j;
      if (!window_job<BN, PACKED>(p, w, number, j)) continue;
      const bool valid = rh < j.nh && rt < j.n;
      const int at = j.pf + rt;                     // position of the row
      const int2 open = window_whole<BN>(w, j);
      float m = -INFINITY, l = 0.f, m_before = -INFINITY;
      // global block number g = blocks_before + i: group g & 1, buffer g % 3
      for (int i = (blocks_before & 1) ^ group; i < j.blocks; i += 2) {
        const int g = blocks_before + i, x = g % 3;
        const bool whole = i >= open.x && i < open.y;
        int2 s = make_int2(0, BN);
        if (!whole) s = window_span<BN>(j, i);
        hold(bar.s_full(x), g / 3);
        tc_fence_after();
        const uint32_t s_at = tmem + lanes + x * BN;
        uint32_t f[NC][32];
        float top;
        if (whole) {
#pragma unroll
          for (int c = 0; c < NC; ++c) tmem_ld_32x32b_x32(s_at + c * 32, f[c]);
#pragma unroll
          for (int c = 0; c < NC; ++c) tmem_ld_wait_tied(f[c]);
        } else {
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            if (c * 32 < s.x || c * 32 >= s.y) {  // trimmed: as if hidden
#pragma unroll
              for (int e = 0; e < 32; ++e) f[c][e] = 0xff800000u;
              continue;
            }
            tmem_ld_32x32b_x32(s_at + c * 32, f[c]);
            tmem_ld_wait_tied(f[c]);
            if (w.negate) {
#pragma unroll
              for (int e = 0; e < 32; ++e) f[c][e] ^= 0x80000000u;
            }
            const int a = (i < j.head ? i : i + j.jump) * BN + c * 32;
            const uint32_t sees = valid ? bits_between(at - w.window + 1 - a, at + 1 - a) |
                                              bits_between(0, min(w.sinks, at + 1) - a)
                                        : 0u;
            if (!__all_sync(0xffffffffu, sees == 0xffffffffu)) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(sees & (1u << e))) f[c][e] = 0xff800000u;  // -inf
            }
          }
        }
        {
          float a0 = -INFINITY, a1 = -INFINITY, a2 = -INFINITY, a3 = -INFINITY;
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              a0 = max3(a0, __uint_as_float(f[c][e]), __uint_as_float(f[c][e + 1]));
              a1 = max3(a1, __uint_as_float(f[c][e + 2]), __uint_as_float(f[c][e + 3]));
              a2 = max3(a2, __uint_as_float(f[c][e + 4]), __uint_as_float(f[c][e + 5]));
              a3 = max3(a3, __uint_as_float(f[c][e + 6]), __uint_as_float(f[c][e + 7]));
            }
          top = fmaxf(fmaxf(a0, a1), fmaxf(a2, a3));
        }
        const float scaled = top == -INFINITY ? top : top * w.scale_log2;
        // The reference as the block before left it.  Taking it in every block, a
        // job's first one too, is also what keeps a group from leaving the next one
        // over a value that the other has not read yet.
        if (g > 0) hold(take, taken++);
        if (i > 0) {
          m_before = m_of[(group ^ 1) * 128 + r];
        }
        const float was = m;  // the reference of this group's l
        m = scaled > m_before + 8.f ? scaled : m_before;
        m_of[group * 128 + r] = m;
        __syncwarp();
        if (lane == 0) arrive(give);
        l *= was == m ? 1.f : pow2(was - m);
        const bool moved = m != m_before;
        if (i > 0 && __any_sync(0xffffffffu, moved)) {
          // O holds the blocks before this one, by the old reference
          hold(bar.pv_done((g - 1) % 3), (g - 1) / 3);
          tc_fence_after();
          const float alpha = moved ? pow2(m_before - m) : 1.f;
#pragma unroll 1
          for (int c = 0; c < vc * 8; ++c) {  // 8 columns at a time: few registers
            uint32_t v[8];
            tmem_ld_x8(o_at + c * 8, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
            tmem_st_x8(o_at + c * 8, v);
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const uint64_t ref2 = pair_of(-ref, -ref);
        uint64_t sum2 = 0, sum3 = 0;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (!whole && (c * 32 < s.x || c * 32 >= s.y)) continue;
          uint32_t packed[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float a, bb;
            split_pair(fma_pair(pair_of(__uint_as_float(f[c][2 * e]),
                                        __uint_as_float(f[c][2 * e + 1])),
                                scale2, ref2),
                       a, bb);
            a = pow2(a);
            bb = pow2(bb);
            packed[e] = pack_two<T>(a, bb);
            if (e & 1)
              sum3 = add_pair(sum3, pair_of(a, bb));
            else
              sum2 = add_pair(sum2, pair_of(a, bb));
          }
          tmem_st_32x32b_x16(s_at + c * 16, packed);
        }
        float s0, s1;
        split_pair(add_pair(sum2, sum3), s0, s1);
        l += s0 + s1;
        if (PACKED) {
          const int first = (i < j.head ? i : i + j.jump) * BN;
          if (first + s.y > j.lk) {
            // the block's last columns may be another sequence's tokens
            // (the ring took two places for each of the blocks before)
            const int pos = 2 * blocks_before + ring_of_v(i, j.blocks);
            hold(bar.full(pos % NS), pos / NS);
            uint8_t* v = ring + pos % NS * L::kSlot;
            for (int row = max(0, j.lk - first); row < s.y; ++row)
              for (int c = r; c < vc * 8; c += 128)
                *reinterpret_cast<uint4*>(v + (c >> 3) * (BN * 128) + row * 128 + (c & 7) * 16) =
                    make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive(bar.p_ready(x));
      }
      // The group of the last block stores the rows; the other one leaves its sum.
      const bool store = ((blocks_before + j.blocks - 1) & 1) == group;
      blocks_before += j.blocks;
      const int left = sums_left & 1, left_turn = sums_left >> 1;
      if (j.blocks > 1) ++sums_left;
      if (j.blocks > 0) ++jobs_done;
      if (!store) {
        if (j.blocks > 1) {
          l_of[left * 128 + r] = l;
          __syncwarp();
          if (lane == 0) arrive(bar.l_ready(left));
        }
        continue;
      }
      // ------------------------------------------------------------- the output
      if (j.blocks > 1) {
        hold(bar.l_ready(left), left_turn);
        // the other group's sum goes by the reference of the block before the last
        const float theirs = l_of[left * 128 + r];
        l += m_before == m ? theirs : theirs * pow2(m_before - m);
      }
      const int tok = j.qt + j.q0 + rt;
      T* out = valid ? static_cast<T*>(p.o) + j.b * p.o_sb + (j.h0 + rh) * p.o_sh + tok * p.o_st
                     : nullptr;
      if (j.blocks > 0) {
        hold(bar.o_done(), jobs_done - 1);
        tc_fence_after();
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      float odd = 0.f;  // becomes NaN with the first output that is not finite
#pragma unroll 1
      for (int c = 0; c < vc * 2; ++c) {
        uint32_t v[32];
        if (j.blocks > 0) {
          tmem_ld_32x32b_x32(o_at + c * 32, v);
          tmem_ld_wait_tied(v);
          if (c == vc * 2 - 1) {  // O is free for the next job
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive(bar.o_free());
          }
        }
        if (l == 0.f || j.blocks == 0) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0;
        }
        if (!valid) continue;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float y = __uint_as_float(v[e]) * inv;
          odd = fmaf(y, 0.f, odd);
          v[e] = __float_as_uint(y);
        }
        if (w.vec_out) {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            if (c * 32 + e < p.dv)
              *reinterpret_cast<uint4*>(out + c * 32 + e) = make_uint4(
                  pack_two<T>(__uint_as_float(v[e]), __uint_as_float(v[e + 1])),
                  pack_two<T>(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])),
                  pack_two<T>(__uint_as_float(v[e + 4]), __uint_as_float(v[e + 5])),
                  pack_two<T>(__uint_as_float(v[e + 6]), __uint_as_float(v[e + 7])));
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c * 32 + e < p.dv) out[c * 32 + e] = from_f32<T>(__uint_as_float(v[e]));
        }
      }
      __syncwarp();
      unsigned again = __ballot_sync(0xffffffffu, valid && !(odd == 0.f));
      while (again != 0) {
        const int x = __ffs(again) - 1;
        again &= again - 1;
        const int xh = j.h0 + __shfl_sync(0xffffffffu, rh, x);
        const int xt = __shfl_sync(0xffffffffu, rt, x);
        const int64_t xtok = j.qt + j.q0 + xt;
        window_row<T>(
            static_cast<const T*>(p.q) + j.b * p.q_sb + xh * p.q_sh + xtok * p.q_st,
            static_cast<const T*>(p.k) + j.b * p.k_sb + j.hk * p.k_sh + j.kt * p.k_st,
            static_cast<const T*>(p.v) + j.b * p.v_sb + j.hk * p.v_sh + j.kt * p.v_st,
            static_cast<T*>(p.o) + j.b * p.o_sb + xh * p.o_sh + xtok * p.o_st, p.k_st, p.v_st, p.d,
            p.dv, p.scale, p.window, p.sinks, j.pf + xt);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

}  // namespace bio

namespace {

constexpr int64_t kMaxGrid = 2147483647;

template <typename T>
int launch_rows(const bio::WindowParams& p, bool packed, cudaStream_t s) {
  const int64_t rows = (packed ? 1 : p.batch) * p.heads * p.lq;
  const int64_t blocks = (rows + bio::kWinWarps - 1) / bio::kWinWarps;
  if (blocks > kMaxGrid) return BIO_ERR_SHAPE;
  if (packed)
    bio::window_row_kernel<T, true><<<static_cast<unsigned>(blocks), bio::kWinWarps * 32, 0, s>>>(p);
  else
    bio::window_row_kernel<T, false><<<static_cast<unsigned>(blocks), bio::kWinWarps * 32, 0, s>>>(p);
  return bio_host::launch_status(cudaGetLastError());
}

template <typename T, int DP, bool PACKED>
int launch_tc(const bio::WindowParams& p, const bio_attn_args* a, cudaStream_t s) {
  constexpr bool packed = PACKED;
  using L = bio::WinSmem<DP>;
  static std::once_flag once[bio_host::kMaxDevices];
  cudaError_t set = cudaSuccess;
  std::call_once(once[a->device], [&] {
    set = cudaFuncSetAttribute(bio::window_tc_kernel<T, DP, PACKED>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  });
  if (set != cudaSuccess) return BIO_ERR_LAUNCH;
  const int sms = bio_host::sm_count(a->device);
  if (sms <= 0) return BIO_ERR_LAUNCH;
  bio::WindowJobs w;
  const int64_t group = p.group;
  w.hblocks = static_cast<int>((group + 15) / 16);  // up to 16 heads of a group in a tile
  w.gh = static_cast<int>((group + w.hblocks - 1) / w.hblocks);
  w.tok = 128 / w.gh;
  const int64_t span = w.tok, tiles = a->kv_heads * w.hblocks;
  const int64_t qblocks = (p.lq + span - 1) / span + (packed ? p.nseq : 0);
  const int64_t jobs = qblocks * tiles * (packed ? 1 : p.batch);
  if (qblocks > kMaxGrid || jobs > kMaxGrid) return BIO_ERR_SHAPE;
  w.qblocks = static_cast<int>(qblocks);
  w.jobs = static_cast<int>(jobs);
  w.window = static_cast<int>(std::min<int64_t>(p.window, 1 << 30));
  w.sinks = static_cast<int>(std::min<int64_t>(p.sinks, 1 << 30));
  w.negate = p.scale < 0.f;
  // a scale of 0 weighs every visible key alike; hidden ones stay at -inf
  const float scale = (w.negate ? -p.scale : p.scale) * 1.4426950408889634f;
  w.scale_log2 = scale == 0.f ? 1.17549435e-38f : scale;
  w.vec_out = reinterpret_cast<uintptr_t>(p.o) % 16 == 0 &&
              (p.o_sb | p.o_sh | p.o_st | p.dv) % 8 == 0;
  CUtensorMap q, k, v;
  const int64_t batch = packed ? 1 : p.batch;
  // without keys nothing is read through K and V: any operand will do for their maps
  const bool none = p.lk == 0;
  if (!bio_host::map_of<T>(&q, p.q, p.d, p.lq, p.heads, batch, p.q_st, p.q_sh, p.q_sb, w.tok,
                           w.gh) ||
      !bio_host::map_of<T>(&k, none ? p.q : p.k, p.d, none ? 1 : p.lk, a->kv_heads, batch, p.k_st,
                           p.k_sh, p.k_sb, 32) ||
      !bio_host::map_of<T>(&v, none ? p.q : p.v, p.dv, none ? 1 : p.lk, a->kv_heads, batch, p.v_st,
                           p.v_sh, p.v_sb, 32))
    return BIO_ERR_ALIGN;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(jobs, sms));
  bio::window_tc_kernel<T, DP, PACKED><<<grid, L::kThreads, L::kBytes, s>>>(q, k, v, p, w);
  return bio_host::launch_status(cudaGetLastError());
}

template <typename T>
int launch_half(const bio::WindowParams& p, const bio_attn_args* a, bool packed, cudaStream_t s) {
  const uint64_t bits = reinterpret_cast<uint64_t>(p.q) | reinterpret_cast<uint64_t>(p.k) |
                        reinterpret_cast<uint64_t>(p.v) |
                        2 * static_cast<uint64_t>(p.q_sb | p.q_sh | p.q_st | p.k_sb | p.k_sh |
                                                  p.k_st | p.v_sb | p.v_sh | p.v_st);
  if (bits % 16 != 0) return BIO_ERR_ALIGN;
  const int dim = std::max(p.d, p.dv);
  if (packed)
    return dim <= 64    ? launch_tc<T, 64, true>(p, a, s)
           : dim <= 128 ? launch_tc<T, 128, true>(p, a, s)
                        : launch_tc<T, 256, true>(p, a, s);
  return dim <= 64    ? launch_tc<T, 64, false>(p, a, s)
         : dim <= 128 ? launch_tc<T, 128, false>(p, a, s)
                      : launch_tc<T, 256, false>(p, a, s);
}

int run_window(const bio_attn_args* a, int64_t window, int64_t sinks, bool packed, void* stream) {
  if (a == nullptr) return BIO_ERR_ARG;
  if (a->d < 1 || a->dv < 1 || a->d > bio::kWinDims || a->dv > bio::kWinDims)
    return BIO_ERR_SHAPE;
  if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->heads > 65536 ||
      a->batch < 0 || a->lq < 0 || a->lk < 0 || a->lq > (1 << 30) || a->lk > (1 << 30))
    return BIO_ERR_SHAPE;
  if (window < 1 || window > kMaxGrid || sinks < 0 || sinks > kMaxGrid || a->causal != 0 ||
      a->mask_kind != BIO_MASK_NONE)
    return BIO_ERR_ARG;
  if (packed && (a->cu_q == nullptr || a->cu_k == nullptr || a->nseq < 0)) return BIO_ERR_ARG;
  const int64_t batch = packed ? 1 : a->batch;
  if (batch == 0 || a->lq == 0) return BIO_OK;
  if (batch > kMaxGrid / a->heads || batch * a->heads > (static_cast<int64_t>(1) << 50) / a->lq)
    return BIO_ERR_SHAPE;
  if (a->q == nullptr || a->o == nullptr || (a->lk > 0 && (a->k == nullptr || a->v == nullptr)))
    return BIO_ERR_ARG;
  int st = bio_host::ensure_device(a->device);
  if (st != BIO_OK) return st;
  bio::WindowParams p;
  p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o;
  p.q_sb = a->q_sb; p.q_sh = a->q_sh; p.q_st = a->q_st;
  p.k_sb = a->k_sb; p.k_sh = a->k_sh; p.k_st = a->k_st;
  p.v_sb = a->v_sb; p.v_sh = a->v_sh; p.v_st = a->v_st;
  p.o_sb = a->o_sb; p.o_sh = a->o_sh; p.o_st = a->o_st;
  p.batch = a->batch; p.heads = a->heads; p.group = a->heads / a->kv_heads;
  p.lq = a->lq; p.lk = a->lk; p.d = a->d; p.dv = a->dv;
  p.scale = a->scale;
  p.window = window; p.sinks = sinks;
  p.cu_q = a->cu_q; p.cu_k = a->cu_k; p.cu_is64 = a->cu_is64; p.nseq = a->nseq;
  p.status = bio_host::status_word(a->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case BIO_F32: return launch_rows<float>(p, packed, s);
    case BIO_F16: return launch_half<__half>(p, a, packed, s);
    case BIO_BF16: return launch_half<__nv_bfloat16>(p, a, packed, s);
    default: return BIO_ERR_DTYPE;
  }
}

}  // namespace

extern "C" {

int bio_attention_window(const bio_attn_args* args, int64_t window, int64_t sinks, void* stream) {
  return run_window(args, window, sinks, false, stream);
}

int bio_attention_window_varlen(const bio_attn_args* args, int64_t window, int64_t sinks,
                                void* stream) {
  return run_window(args, window, sinks, true, stream);
}

}  // extern "C"
