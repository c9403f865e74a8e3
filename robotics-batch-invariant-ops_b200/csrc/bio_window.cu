// Prefill attention with a sliding window and sink tokens (dense and packed).
//
// Query i sits at position p = i + (lk - lq) and sees key j iff j <= p and
// (j > p - window or j < sinks):
//   o_i = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q_i.k_j.
// A row that sees no key (p < 0) gives zeros.
//
// 16-bit operands run on tcgen05 (window_tc_kernel), fp32 on the CUDA cores
// (window_f32_kernel).
//
// Not in the reference, whose SDPA (batch_invariant_ops.py:1148-1213) would
// need the mask as a tensor and visits every key.
#include <algorithm>
#include <mutex>
#include <type_traits>

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

// ---------------------------------------------------------------------------
// tcgen05 kernel.
//
// A job is NT tiles of 128 query rows that share a KV head.  A tile packs `gh`
// query heads of the group with `tok` = 128 / gh consecutive tokens each (row r:
// head r / tok, token r % tok), so the keys that a tile visits are its window
// plus tok - 1, not plus 127, and a key block is loaded once for the whole
// group.  Jobs are dealt out round robin to one persistent CTA per SM:
//   warp 0      TMA: Q tiles, then K and V blocks of BN keys through one ring.
//   warp 1      MMA: S_t = Q_t K^T, O_t += P_t V, fp32 in TMEM; P (16 bits) lies
//               over the S that it came from.
//   warps 4..   softmax: one thread per query row; the 128 rows of tile t belong
//               to warps 4 + 4 t .. 7 + 4 t, which take over registers of the
//               first four warps.
// The ring, S and O run on across jobs: a job's first products start while the
// last rows of the one before are still being stored.  With two tiles (D <= 128)
// the tensor cores work on one tile while the other is in its softmax; with one
// (D <= 256) S has two buffers, and S of block i is issued before P of block
// i - 1 is waited for.
//
// What bounds it is the chain softmax -> PV -> S of a tile and the instructions of
// the single warps along it, not the products (an M = 128, N = 128, K = 16 product
// runs for 64 clocks): a look at a barrier costs 125 clocks and more even when
// nobody has to wait, so barriers that are due together are looked at together
// (one per lane), and a TMA box about 50, so blocks are loaded whole.
//
// Measured, 32768 tokens, 32 heads on 8, D 128, window 1024: 770 us, 705 TFLOP/s
// of visible products; window 16384 runs at 1050, so the two blocks that a window
// cuts, the sinks' block, refill and output cost a job about 10 of its 28 us.
// Steps: one thread issuing everything in a divergent branch 1073 us, an elected
// thread of a uniform warp 842, polled instead of suspended waits and outputs in
// 32-byte stores 775.  Slower and gone: a share of the exponentials on the FMA
// pipe (872), two threads per row (838 beside 842, twice the barriers), 64-key
// blocks with two S buffers (977), three S buffers shared by two softmax groups
// (840, a second issuing warp).
//
// Blocks are cut on the absolute grid of BN keys; products are trimmed, per tile,
// to the 32-key columns that some row of the tile sees.  Masked scores weigh
// exactly 0 and untrimmed columns add exactly 0, so a row's bits depend on its
// own query, keys and position only.
//
// Scores, maxima and sums are fp32 in registers (128 scores a thread).  The
// reference m of the exponentials moves only when a block's maximum exceeds it
// by more than 8 (log2), so O is rarely rescaled and P stays below 2^8.  In fp16 P
// is kept 2^7 times larger (below 2^15): weights under 2^-25 of the largest would be
// rounded to nothing, and some 100000 of them are worth more than a rounding.  P is
// rounded to the operand type, as the product needs; l sums it unrounded, since the
// rounded values would have to be unpacked again: 95 instead of 86 us (512 tokens
// behind 4096, D 64) and 827 instead of 771 us (the case above), for an error that
// is 1 % smaller (bf16, 1500 tokens, window 1024: 2.05e-3 instead of 2.07e-3 of the
// output's norm, 1.61e-3 of it the rounding of the output).
//
// A hidden key in a visited block has weight 0, but 0 * Inf or 0 * NaN in V
// would still reach the row.  A block whose rows all came out finite is done.  One
// that wrote anything else goes through its jobs once more, with the values of
// every key that holds an Inf or NaN zeroed in shared memory: rows that do not see
// such a key get the bits that they have beside finite values, since it adds
// exactly 0 either way.  Rows that see one, or are not finite for another reason,
// are computed by their warp from their visible keys alone (window_row) after the
// last job, since a long row can take longer than the waits of the other warps.
// Keys of a neighbouring packed sequence are zeroed in shared memory at once.
// ---------------------------------------------------------------------------
struct WindowJobs {
  int gh, tok, hblocks;  // heads and tokens of a tile, tiles across a group
  int qblocks;           // dense: blocks of NT * tok tokens per sequence; packed: at most
  int jobs;
  int window, sinks;     // at most 2^30
  float scale_log2;      // > 0
  int negate;            // the scale was negative: scores change sign
  int vec_out;           // output rows take 32-byte (2) or 16-byte (1) stores
  FixedDiv by_qblocks, by_tiles, by_hblocks;
};

template <int DP>
struct WinSmem {
  static constexpr int NT = DP == 256 ? 1 : 2;     // tiles of a job
  static constexpr int BN = DP == 256 ? 64 : 128;  // keys of a block
  static constexpr uint32_t kQ = 128 * DP * 2;
  static constexpr uint32_t kSlot = BN * DP * 2;   // K or V of a block
  static constexpr int kFit = (227 * 1024 - 1024 - 512 - NT * static_cast<int>(kQ)) /
                              static_cast<int>(kSlot);
  static constexpr int kSlots = kFit > 8 ? 8 : kFit;
  static constexpr uint32_t kBytes = 1024 + NT * kQ + kSlots * kSlot + 512;
  static constexpr int kThreads = 128 + 128 * NT;
  static_assert(kSlots >= 4, "K and V of two blocks");
};

// Keys of a tile: [lo, hi) for the windows of its rows, [0, sx) sinks before it.
struct WinTile {
  int pf, n;   // position of its first token, number of tokens
  int lo, hi, sx;
  int last;    // the tile's last block of the job, -1: it sees no key
};

struct WinJob {
  int b, hk, h0, nh;        // sequence of the batch, KV head, query heads
  int q0, lq, lk;           // first query of the job, lengths of its sequence
  int qt, kt;               // tokens of the operands at which the sequence starts
  int head, jump, blocks;   // block i of the job is block i < head ? i : i + jump of the keys
  WinTile tile[2];
};

template <int NT, int BN>
__device__ __forceinline__ void window_plan(const WindowJobs& w, WinJob& j) {
  int first = 0x7fffffff, last = -1;
  j.head = 0;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    WinTile& x = j.tile[t];
    const int q = j.q0 + t * w.tok;
    x.n = max(0, min(w.tok, j.lq - q));
    x.pf = q + j.lk - j.lq;
    x.hi = x.n > 0 ? max(0, x.pf + x.n) : 0;
    x.lo = x.hi > 0 ? max(0, x.pf - w.window + 1) : 0;
    x.sx = min(w.sinks, x.lo);
    if (x.hi > 0) {
      j.head = max(j.head, (x.sx + BN - 1) / BN);
      first = min(first, x.lo / BN);
      last = max(last, (x.hi - 1) / BN);
    }
  }
  j.jump = last < 0 ? 0 : max(0, first - j.head);
  j.blocks = last < 0 ? 0 : last + 1 - j.jump;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int b = (j.tile[t].hi - 1) / BN;
    j.tile[t].last = j.tile[t].hi == 0 ? -1 : b < j.head ? b : b - j.jump;
  }
}

// Columns [x, y) of the job's block i that some row of the tile sees, on the
// 32-column grid; empty: x == y.
template <int BN>
__device__ __forceinline__ int2 window_span(const WinJob& j, const WinTile& t, int i) {
  const int base = (i < j.head ? i : i + j.jump) * BN;
  int x = max(t.lo - base, 0), y = min(t.hi - base, BN);
  if (x >= y) x = y = 0;
  const int s = min(t.sx - base, BN);
  if (s > 0) {
    x = 0;
    y = max(y, s);
  }
  return make_int2(x & ~31, (y + 31) & ~31);
}

// Blocks x <= i < y of the job: every row of the tile sees every key by its
// window, and all 128 rows exist (or are padding of the tile's shape).
template <int BN>
__device__ __forceinline__ int2 window_whole(const WindowJobs& w, const WinJob& j,
                                             const WinTile& t) {
  if (w.negate || t.n < w.tok || j.nh < w.gh || t.pf < 0) return make_int2(0, 0);
  const int x = (max(0, t.pf + t.n - w.window) + BN - 1) / BN;  // first inside the last window
  const int y = (t.pf + 1) / BN;                                // first past the first row
  // only what lies behind the sinks' blocks keeps its distance
  return make_int2(max(x, j.head + j.jump) - j.jump, y - j.jump);
}

// Job number -> job.  All lanes of the warp call it; false: no such job.
template <int NT, int BN, bool PACKED>
__device__ __forceinline__ bool window_job(const WindowParams& p, const WindowJobs& w, int number,
                                           WinJob& j) {
  const int lane = threadIdx.x & 31;
  const int tiles = static_cast<int>(w.by_tiles.n);
  int qb, hx;
  if constexpr (!PACKED) {
    const int rest = w.by_qblocks.quotient(number);
    qb = number - rest * w.qblocks;
    j.b = w.by_tiles.quotient(rest);
    hx = rest - j.b * tiles;
    j.lq = static_cast<int>(p.lq);
    j.lk = static_cast<int>(p.lk);
    j.qt = j.kt = 0;
  } else {
    qb = w.by_tiles.quotient(number);
    hx = number - qb * tiles;
    j.b = 0;
    if (win_off(p.cu_q, p.cu_is64, 0) != 0 || win_off(p.cu_k, p.cu_is64, 0) != 0) {
      raise_status(p.status, BIO_DEV_INDEX);
      return false;
    }
    // 32 sequences at a time: the one whose blocks hold block qb
    const int span = NT * w.tok;
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
  j.q0 = qb * NT * w.tok;
  j.hk = w.by_hblocks.quotient(hx);
  const int before = (hx - j.hk * w.hblocks) * w.gh;
  j.h0 = j.hk * static_cast<int>(p.group) + before;
  j.nh = min(w.gh, static_cast<int>(p.group) - before);
  window_plan<NT, BN>(w, j);
  return true;
}

__device__ __forceinline__ void prefetch_box(const CUtensorMap* map, int c0, int c1, int c2,
                                             int c3) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
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

// Two values of type T in a word: a + 0 * y, which is NaN from the first y that is
// not finite on.
template <typename T>
__device__ __forceinline__ uint32_t note_odd(uint32_t a, uint32_t y);
template <>
__device__ __forceinline__ uint32_t note_odd<__nv_bfloat16>(uint32_t a, uint32_t y) {
  const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&y),
                                   __floats2bfloat162_rn(0.f, 0.f),
                                   *reinterpret_cast<const __nv_bfloat162*>(&a));
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t note_odd<__half>(uint32_t a, uint32_t y) {
  const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&y), __floats2half2_rn(0.f, 0.f),
                            *reinterpret_cast<const __half2*>(&a));
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Bits of a value of type T that are all set in infinities and NaN.
template <typename T>
constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;

// The lowest x bits of a word, x anywhere.
__device__ __forceinline__ uint32_t low_bits(int x) {
  return __funnelshift_lc(0xffffffffu, 0u, max(x, 0));
}

// Which of the keys a .. a + 31 a query at position `at` sees.
__device__ __forceinline__ uint32_t window_sees(const WindowJobs& w, int at, int a) {
  return (low_bits(at + 1 - a) & ~low_bits(at - w.window + 1 - a)) |
         low_bits(min(w.sinks, at + 1) - a);
}

// Zeroes the values of the keys of a block (BN rows of 128 bytes per 64 columns)
// that are not finite and says which keys these are.  Every warp that is going to
// use the block calls it: each finds such a key itself or, where another warp was
// faster, finds its bit in `shared`, which is set before the zeros are written.
template <typename T, int BN>
__device__ __noinline__ void clean_values(uint8_t* v, uint32_t* shared, int chunks,
                                          uint32_t (&bad)[BN / 32]) {
  constexpr uint32_t e = kExponent<T>;
  const int lane = threadIdx.x & 31;
  auto odd = [](uint32_t x) { return (x & e) == e || (x >> 16 & e) == e; };
  for (int n = lane; n < BN; n += 32) {
    bool found = false;
    for (int x = 0; x < chunks * 8; ++x) {
      const uint4 y = *reinterpret_cast<const uint4*>(v + (x >> 3) * (BN * 128) + n * 128 +
                                                      (((x ^ n) & 7) << 4));
      found |= odd(y.x) || odd(y.y) || odd(y.z) || odd(y.w);
    }
    if (!found) continue;
    atomicOr(shared + (n >> 5), 1u << (n & 31));
    __threadfence_block();
    for (int x = 0; x < chunks * 8; ++x)
      *reinterpret_cast<uint4*>(v + (x >> 3) * (BN * 128) + n * 128 + ((x & 7) << 4)) =
          make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();  // the products read what is left
  __syncwarp();
#pragma unroll
  for (int c = 0; c < BN / 32; ++c) bad[c] = *const_cast<volatile uint32_t*>(shared + c);
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
  __device__ uint32_t empty(int s) const { return base + 64 + s * 8; }
  __device__ uint32_t q_full(int t) const { return base + 128 + t * 8; }
  __device__ uint32_t q_empty(int t) const { return base + 144 + t * 8; }
  __device__ uint32_t s_full(int x) const { return base + 160 + x * 8; }
  __device__ uint32_t p_ready(int x) const { return base + 176 + x * 8; }
  __device__ uint32_t o_done(int t) const { return base + 192 + t * 8; }
  __device__ uint32_t pv_done() const { return base + 208; }
  __device__ uint32_t all_done() const { return base + 216; }
};

// The ring of a job of n blocks carries K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1): the
// place of V of block i.
__device__ __forceinline__ int ring_of_v(int i, int n) { return i < n - 1 ? 2 * i + 2 : 2 * n - 1; }

template <typename T, int DP, bool PACKED>
__global__ void __launch_bounds__(WinSmem<DP>::kThreads, 1)
    window_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const WindowParams p,
                     const WindowJobs w) {
  using L = WinSmem<DP>;
  constexpr int NT = L::NT, BN = L::BN, NS = L::kSlots, NC = BN / 32;
  constexpr uint32_t kFmt = std::is_same<T, __half>::value ? 0u : 1u;
  constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;  // log2
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* ring = smem + NT * L::kQ;
  uint8_t* tail = ring + NS * L::kSlot;
  const uint32_t q32 = smem_u32(smem), ring32 = smem_u32(ring);
  const WinBars bar{smem_u32(tail)};
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 256);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 260);
  volatile int* odd_rows = reinterpret_cast<volatile int*>(tail + 264);
  uint32_t* bad_keys = reinterpret_cast<uint32_t*>(tail + 272);  // [NS][4], clean turn only
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kc = (p.d + 63) / 64, vc = (p.dv + 63) / 64;

  if (threadIdx.x == 0) {
    uint64_t* b = reinterpret_cast<uint64_t*>(tail);
    for (int i = 0; i < 28; ++i) mbar_init(b + i, i == 22 || i == 23 ? 4 : 1);  // p_ready: 4 warps
    *abort_flag = 0;
    *odd_rows = 0;
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
  // warp no move to a uniform register.  S at column 0 and 128, O_t at 256 + 128 t.
  constexpr uint32_t tmem = 0;
  if (*tmem_slot != tmem) {  // the same for every thread
    if (threadIdx.x == 0) raise_status(p.status, BIO_DEV_TIMEOUT);
    if (warp == 1) tmem_dealloc(*tmem_slot, 512);
    return;
  }
  auto wait = [&](uint32_t b, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, spin_wait(b, parity & 1u, abort_flag, p.status));
  };
  // Three barriers at once, one per lane.
  auto wait_all = [&](uint32_t a, uint32_t pa, uint32_t b, uint32_t pb, uint32_t c,
                      uint32_t pc) -> bool {
    const uint32_t at = lane == 0 ? a : lane == 1 ? b : c;
    const uint32_t parity = lane == 0 ? pa : lane == 1 ? pb : pc;
    return __all_sync(0xffffffffu, spin_wait(at, parity & 1u, abort_flag, p.status));
  };

  // Every warp of the block comes here once, after its last job or after a wait that
  // ran out: whether a row was not finite, so that all jobs are done again, clean.
  auto clean_turn = [&]() -> bool {
    __syncwarp();
    asm volatile("bar.sync 1, %0;" ::"n"(L::kThreads) : "memory");
    return *odd_rows != 0 && *abort_flag == 0;
  };

  // 384 threads start with 168 registers each, 128 of them go on with 72 and
  // 256 with 216: the same 64512
  constexpr bool kShift = NT == 2;
  if (warp < 4) {
    if (kShift) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // -------------------------------------------------------------- producer
      int slot = 0, count = 0;              // ring position, blocks loaded so far
      uint32_t turn = 0;
      int q_used[2] = {0, 0};
      bool ok = true;
      for (int again = 0; again < 2 && (again == 0 || clean_turn()); ++again) {
        for (int number = blockIdx.x; ok && number < w.jobs; number += gridDim.x) {
          WinJob j;
          if (!window_job<NT, BN, PACKED>(p, w, number, j)) continue;
          const int n = j.blocks;
          if (n == 0) continue;
          auto load = [&](const CUtensorMap* map, int chunks, int i) {
            if (lane == 0) {
              // whoever looked at the slot's last block has done so: it was empty
              if (again) *reinterpret_cast<uint4*>(bad_keys + slot * 4) = make_uint4(0, 0, 0, 0);
              const int row = j.kt + (i < j.head ? i : i + j.jump) * BN;
              expect_bytes(bar.full(slot), chunks * (BN * 128));
              for (int c = 0; c < chunks; ++c)
                load_box(ring32 + slot * L::kSlot + c * (BN * 128), map, bar.full(slot), c * 64,
                         row, j.hk, j.b);
            }
            ++count;
            if (++slot == NS) {
              slot = 0;
              turn ^= 1u;
            }
          };
          ok = wait(bar.empty(slot), turn ^ 1u);
          if (!ok) break;
          load(&tmK, kc, 0);
          {  // the next job's queries on their way into L2, behind this job's first keys
            WinJob then;
            const int at = number + static_cast<int>(gridDim.x);
            if (at < w.jobs && window_job<NT, BN, PACKED>(p, w, at, then) && lane < NT * kc) {
              const int t = lane / kc;
              prefetch_box(&tmQ, (lane - t * kc) * 64, then.qt + then.q0 + t * w.tok, then.h0,
                           then.b);
            }
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (j.tile[t].last < 0 || !ok) continue;
            ok = wait(bar.q_empty(t), q_used[t] ^ 1);
            if (!ok) break;
            if (lane == 0) {
              expect_bytes(bar.q_full(t), kc * w.gh * w.tok * 128);
              for (int c = 0; c < kc; ++c)
                load_box(q32 + t * L::kQ + c * 16384, &tmQ, bar.q_full(t), c * 64,
                         j.qt + j.q0 + t * w.tok, j.h0, j.b);
            }
            ++q_used[t];
          }
          for (int i = 1; ok && i <= n; ++i) {
            const bool key = i < n;           // K of block i, then V of block i - 1
            const int slot2 = slot + 1 == NS ? 0 : slot + 1;
            const uint32_t turn2 = slot + 1 == NS ? turn ^ 1u : turn;
            const uint32_t e1 = bar.empty(slot), e2 = key ? bar.empty(slot2) : e1;
            ok = wait_all(e1, turn ^ 1u, e2, (key ? turn2 : turn) ^ 1u, e1, turn ^ 1u);
            if (!ok) break;
            if (key) load(&tmK, kc, i);
            load(&tmV, vc, i - 1);
          }
        }
        // every copy has to land before the block's shared memory goes
        if (lane == 0) {
          for (int i = max(0, count - NS); i < count; ++i)
            if (!mbar_wait_drain(reinterpret_cast<uint64_t*>(tail) + i % NS, (i / NS) & 1))
              raise_status(p.status, BIO_DEV_TIMEOUT);
          for (int t = 0; t < NT; ++t)
            if (q_used[t] > 0 &&
                !mbar_wait_drain(reinterpret_cast<uint64_t*>(tail) + 16 + t, (q_used[t] - 1) & 1))
              raise_status(p.status, BIO_DEV_TIMEOUT);
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------- MMA
      int slot = 0;                         // ring position of what comes next
      uint32_t turn = 0;
      int s_used[NT], p_used[NT], q_used[NT];  // S, PV and jobs of tile t
#pragma unroll
      for (int t = 0; t < NT; ++t) s_used[t] = p_used[t] = q_used[t] = 0;
      bool ok = true;
      auto next = [&]() {
        if (++slot == NS) {
          slot = 0;
          turn ^= 1u;
        }
      };
      for (int again = 0; again < 2 && (again == 0 || clean_turn()); ++again) {
        for (int number = blockIdx.x; ok && number < w.jobs; number += gridDim.x) {
          WinJob j;
          if (!window_job<NT, BN, PACKED>(p, w, number, j)) continue;
          const int n = j.blocks;
          if (n == 0) continue;
          int2 open[NT], held[NT];            // whole blocks; columns of the P that waits
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            open[t] = window_whole<BN>(w, j, j.tile[t]);
            held[t] = make_int2(0, 0);
          }
          uint32_t begun = 0;                 // bit t: O_t holds something
          // S of block i, whose keys are at ring position `at`
          auto products_s = [&](int t, int i, int at, int2 s) {
            tc_fence_after();
            const int x = NT == 2 ? t : s_used[t] & 1;
            const uint32_t idesc = idesc_f16(kFmt, 128, s.y - s.x, false, false);
            const uint64_t qd = smem_desc_sw128(q32 + t * L::kQ, 16, 1024);
            const uint64_t kd = smem_desc_sw128(ring32 + at * L::kSlot + s.x * 128, 16, 1024);
            const uint32_t to = tmem + x * 128 + s.x;
            if (elect_leader()) {
              // 16 columns are 32 bytes, 2 units of a descriptor; 64 columns a chunk
#pragma unroll
              for (int k = 0; k < DP / 16; ++k)
                if (DP == 64 || (k >> 2) < kc)
                  umma_f16(to, qd + (k >> 2) * 1024 + (k & 3) * 2,
                           kd + (k >> 2) * (BN * 8) + (k & 3) * 2, idesc, k > 0 ? 1u : 0u);
              commit_to(bar.s_full(x));
              if (i == j.tile[t].last) commit_to(bar.q_empty(t));
            }
            __syncwarp();
            ++s_used[t];
            if (i == j.tile[t].last) ++q_used[t];
          };
          // PV of block i, whose values are at ring position `at`
          auto products_pv = [&](int t, int i, int at) {
            tc_fence_after();
            const int x = NT == 2 ? t : p_used[t] & 1;
            const uint32_t idesc = idesc_f16(kFmt, 128, vc * 64, false, true);
            // 16 keys are 2048 bytes of V and 8 columns of P
            const uint64_t vd = smem_desc_sw128(ring32 + at * L::kSlot, BN * 128, 1024);
            const uint32_t pa = tmem + x * 128, to = tmem + 256 + t * 128;
            const bool on = (begun >> t) & 1u;
            if (elect_leader()) {
#pragma unroll
              for (int k = 0; k < BN / 16; ++k)
                if (k * 16 >= held[t].x && k * 16 < held[t].y)
                  umma_f16_ts(to, pa + k * 8, vd + k * 128, idesc,
                              on || k * 16 > held[t].x ? 1u : 0u);
              if (NT == 1) commit_to(bar.pv_done());
              if (i == j.tile[t].last) commit_to(bar.o_done(t));
            }
            __syncwarp();
            begun |= 1u << t;
            ++p_used[t];
          };
          auto p_bar = [&](int t) { return bar.p_ready(NT == 2 ? t : p_used[t] & 1); };
          auto p_turn = [&](int t) {
            return static_cast<uint32_t>(NT == 2 ? p_used[t] : p_used[t] >> 1);
          };
          for (int i = 0; ok && i <= n; ++i) {
            const bool key = i < n, value = i > 0;
            const int k_at = slot;
            const uint32_t k_turn = turn;
            if (key) next();
            const int v_at = slot;
            const uint32_t v_turn = turn;
            if (value) next();
            int2 now[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              now[t] = make_int2(0, 0);
              if (key)
                now[t] = i >= open[t].x && i < open[t].y ? make_int2(0, BN)
                                                         : window_span<BN>(j, j.tile[t], i);
            }
            const bool p0 = held[0].x < held[0].y;
            // the block's keys, the values of the one before, and with two tiles the
            // first tile's P; queries with a job's first keys
            const uint32_t b0 = key ? bar.full(k_at) : bar.full(v_at), t0 = key ? k_turn : v_turn;
            uint32_t b2 = b0, t2 = t0;
            if (NT == 2 && p0) {
              b2 = p_bar(0);
              t2 = p_turn(0);
            }
            ok = wait_all(b0, t0, value ? bar.full(v_at) : b0, value ? v_turn : t0, b2, t2);
#pragma unroll
            for (int t = 0; t < NT; ++t)
              if (ok && i == 0 && j.tile[t].last >= 0) ok = wait(bar.q_full(t), q_used[t]);
            if (!ok) break;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const bool s_on = now[t].x < now[t].y, p_on = held[t].x < held[t].y;
              if (NT == 1 && s_on) products_s(t, i, k_at, now[t]);
              if (p_on && ok) {
                if (NT == 1 || t > 0) ok = wait(p_bar(t), p_turn(t));
                if (ok) products_pv(t, i - 1, v_at);
              }
              if (NT == 2 && s_on && ok) products_s(t, i, k_at, now[t]);
              held[t] = now[t];
            }
            // what the products issued so far have read is free once they are done
            if (ok && elect_leader()) {
              if (key) commit_to(bar.empty(k_at));
              if (value) commit_to(bar.empty(v_at));
            }
            __syncwarp();
          }
        }
        if (elect_leader()) commit_to(bar.all_done());
        if (!mbar_wait_drain(reinterpret_cast<uint64_t*>(tail) + 27, again))
          raise_status(p.status, BIO_DEV_TIMEOUT);
      }
    } else {
      clean_turn();
    }
  } else {
    if (kShift) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ----------------------------------------------------------------- softmax
    const int t = NT == 2 ? (warp - 4) >> 2 : 0;
    const int r = (warp & 3) * 32 + lane;  // row of the tile: the warp's quarter of the lanes
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // (quarter * 32) << 16
    const uint32_t o_at = tmem + lanes + 256 + t * 128;
    const int rh = r / w.tok, rt = r - rh * w.tok;
    const uint64_t scale2 = pair_of(w.scale_log2, w.scale_log2);
    int base = 0, s_used = 0, jobs_done = 0;  // ring position of the job's first K
    bool ok = true, odd = false;              // odd: an output of the warp is not finite
    // a copy for each turn, so that the first does not pay for the other
    auto all_jobs = [&](auto turn) {
      constexpr bool kClean = decltype(turn)::value;
      for (int number = blockIdx.x; ok && number < w.jobs; number += gridDim.x) {
        WinJob j;
        if (!window_job<NT, BN, PACKED>(p, w, number, j)) continue;
        WinTile tile = j.tile[0];
        if (NT == 2 && t == 1) tile = j.tile[NT - 1];
        const bool valid = rh < j.nh && rt < tile.n;
        const int at = tile.pf + rt;                     // position of the row
        const int2 open = window_whole<BN>(w, j, tile);
        float m = -INFINITY, l = 0.f;
        bool first = true, dirty = false;  // dirty: the row sees a key that was cleaned
        for (int i = 0; i <= tile.last; ++i) {
          const bool whole = i >= open.x && i < open.y;
          int2 s = make_int2(0, BN);
          if (!whole) s = window_span<BN>(j, tile, i);
          if (s.x >= s.y) continue;
          const int x = NT == 2 ? t : s_used & 1;
          ok = wait(bar.s_full(x), NT == 2 ? s_used : s_used >> 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t s_at = tmem + lanes + x * 128;
          uint32_t f[NC][32];
#pragma unroll
          for (int c = 0; c < NC; ++c) tmem_ld_32x32b_x32(s_at + c * 32, f[c]);
#pragma unroll
          for (int c = 0; c < NC; ++c) tmem_ld_wait_tied(f[c]);
          if (!whole) {
            const uint32_t flip = w.negate ? 0x80000000u : 0u;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              // keys a + e: inside the window, or one of the sinks; trimmed columns hold
              // what was there before
              const int a = (i < j.head ? i : i + j.jump) * BN + c * 32;
              uint32_t sees = window_sees(w, at, a);
              if (!valid || c * 32 < s.x || c * 32 >= s.y) sees = 0u;
              if (flip != 0u || !__all_sync(0xffffffffu, sees == 0xffffffffu)) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  f[c][e] = sees & (1u << e) ? f[c][e] ^ flip : 0xff800000u;  // -inf
              }
            }
          }
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
          const float top = fmaxf(fmaxf(a0, a1), fmaxf(a2, a3));
          const float scaled = top == -INFINITY ? top : top * w.scale_log2;
          const bool move = scaled > m + 8.f;
          const float alpha = move ? pow2(m - scaled) : 1.f;
          if (move) m = scaled;
          l *= alpha;
          if (!first && __any_sync(0xffffffffu, alpha != 1.f)) {
            // S of this block was issued after the PV before it (two tiles), or that
            // one has to be waited for (one tile)
            if (NT == 1) {
              ok = wait(bar.pv_done(), s_used - 1);
              if (!ok) break;
              tc_fence_after();
            }
#pragma unroll 1
            for (int c = 0; c < vc * 8; ++c) {  // 8 columns at a time: few registers
              uint32_t v[8];
              tmem_ld_x8(o_at + c * 8, v);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
              tmem_st_x8(o_at + c * 8, v);
            }
          }
          first = false;
          const float ref = m == -INFINITY ? 0.f : m - kLift;
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
          if constexpr (kClean) {
            const int pos = base + ring_of_v(i, j.blocks);
            ok = wait(bar.full(pos % NS), pos / NS);
            if (!ok) break;
            uint32_t bad[NC];
            clean_values<T, BN>(ring + pos % NS * L::kSlot, bad_keys + pos % NS * 4, vc, bad);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              const int a = (i < j.head ? i : i + j.jump) * BN + c * 32;
              dirty |= (bad[c] & window_sees(w, at, a)) != 0u;
            }
          }
          if (PACKED) {
            const int from = (i < j.head ? i : i + j.jump) * BN;
            if (from + s.y > j.lk) {
              // the block's last columns may be another sequence's tokens
              const int pos = base + ring_of_v(i, j.blocks);
              ok = wait(bar.full(pos % NS), pos / NS);
              if (!ok) break;
              uint8_t* v = ring + pos % NS * L::kSlot;
              for (int row = max(0, j.lk - from); row < s.y; ++row)
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
          ++s_used;
        }
        base += 2 * j.blocks;
        if (!ok) continue;
        // ------------------------------------------------------------- the output
        const int tok = j.qt + j.q0 + t * w.tok + rt;
        T* out = valid ? static_cast<T*>(p.o) + j.b * p.o_sb + (j.h0 + rh) * p.o_sh + tok * p.o_st
                       : nullptr;
        if (tile.last >= 0) {
          ok = wait(bar.o_done(t), jobs_done);
          if (!ok) continue;
          ++jobs_done;
          tc_fence_after();
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const uint64_t inv2 = pair_of(inv, inv);
        uint32_t odd2 = 0;
#pragma unroll 1
        for (int c = 0; c < vc * 2; ++c) {
          uint32_t v[32];
          if (tile.last >= 0) {
            tmem_ld_32x32b_x32(o_at + c * 32, v);
            tmem_ld_wait_tied(v);
          }
          if (l == 0.f || tile.last < 0) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0;
          }
          if (!valid) continue;
          uint32_t y[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t o2 = fma_pair(
                pair_of(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), inv2, 0);
            float lo, hi;
            split_pair(o2, lo, hi);
            y[e] = kClean && dirty ? 0x7fff7fffu : pack_two<T>(lo, hi);  // NaN: again below
            odd2 = note_odd<T>(odd2, y[e]);
          }
          if (w.vec_out == 2) {  // whole 32-byte sectors
#pragma unroll
            for (int e = 0; e < 16; e += 8)
              if (c * 32 + 2 * e < p.dv)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(
                                 out + c * 32 + 2 * e),
                             "r"(y[e]), "r"(y[e + 1]), "r"(y[e + 2]), "r"(y[e + 3]), "r"(y[e + 4]),
                             "r"(y[e + 5]), "r"(y[e + 6]), "r"(y[e + 7])
                             : "memory");
          } else if (w.vec_out == 1) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              if (c * 32 + 2 * e < p.dv)
                *reinterpret_cast<uint4*>(out + c * 32 + 2 * e) =
                    make_uint4(y[e], y[e + 1], y[e + 2], y[e + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e < p.dv)
                reinterpret_cast<uint16_t*>(out)[c * 32 + e] =
                    static_cast<uint16_t>(y[e >> 1] >> (16 * (e & 1)));
          }
        }
        tc_fence_before();  // the next job's PV overwrites O after this row's next P
        if (__any_sync(0xffffffffu, (odd2 & 0x7fff7fffu) != 0u)) {  // zeros keep their sign
          odd = true;
          if (lane == 0) *odd_rows = 1;
        }
      }
    };
    all_jobs(std::false_type{});
    if (clean_turn()) all_jobs(std::true_type{});
    // Rows that are not finite, from their visible keys alone: a warp's job is one
    // row, and nobody waits for this one any more.  The output tells which they are.
    for (int number = blockIdx.x; ok && odd && number < w.jobs; number += gridDim.x) {
      WinJob j;
      if (!window_job<NT, BN, PACKED>(p, w, number, j)) continue;
      WinTile tile = j.tile[0];
      if (NT == 2 && t == 1) tile = j.tile[NT - 1];
      const int64_t first = j.qt + j.q0 + t * w.tok;  // the tile's first token
      T* out = static_cast<T*>(p.o) + j.b * p.o_sb + j.h0 * p.o_sh + first * p.o_st;
      bool bad = false;
      if (rh < j.nh && rt < tile.n) {
        const uint16_t* row = reinterpret_cast<const uint16_t*>(out + rh * p.o_sh + rt * p.o_st);
        for (int c = 0; c < p.dv; ++c) bad |= (row[c] & kExponent<T>) == kExponent<T>;
      }
      for (unsigned again = __ballot_sync(0xffffffffu, bad); again != 0; again &= again - 1) {
        const int y = __ffs(again) - 1;
        const int xh = __shfl_sync(0xffffffffu, rh, y), xt = __shfl_sync(0xffffffffu, rt, y);
        window_row<T>(
            static_cast<const T*>(p.q) + j.b * p.q_sb + (j.h0 + xh) * p.q_sh +
                (first + xt) * p.q_st,
            static_cast<const T*>(p.k) + j.b * p.k_sb + j.hk * p.k_sh + j.kt * p.k_st,
            static_cast<const T*>(p.v) + j.b * p.v_sb + j.hk * p.v_sh + j.kt * p.v_st,
            out + xh * p.o_sh + xt * p.o_st, p.k_st, p.v_st, p.d, p.dv, p.scale, p.window, p.sinks,
            tile.pf + xt);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------
// fp32 kernel: one CTA per tile of 64 query rows (packed like the tiles above,
// tok = 64 / gh tokens of gh heads), key blocks of BN keys in shared memory.
// Thread (ty, tx) computes scores of rows 4 ty .. 4 ty + 3 and keys tx + 16 c,
// the 16 threads of a row share its maximum and sum by shuffles, the weights go
// through shared memory, and it accumulates 4 rows x 4 columns per 64 columns of
// O.  V of a block and K of the next one are copied (cp.async) while the
// products before them run.  FFMA and the shared loads that feed it bound it: 64
// products per 8 loads of 16 bytes in S, 128 per 12 in PV.  Columns that no row of
// the tile sees are skipped 32 at a time.  A tile with a row that is not finite is
// gone through once more with such values zeroed, as above.
// Measured: 99 us for 1024 queries, 8 heads over 2 of 128, window 512 (16 TFLOP/s;
// one warp per row, with K read from L2 for every row, ran at 1).  A window of 31
// keys (4 x 10198 queries, 8 heads of 128) wastes most of its blocks: 1074 us, and
// 1609 with whole blocks and with queries and outputs moved by words.
// ---------------------------------------------------------------------------
// what lies on 16-byte borders
constexpr int kVecKv = 1, kVecQ = 2, kVecO = 4;

template <int DP>
struct WinF32 {
  static constexpr int BN = DP == 256 ? 32 : 64;
  static constexpr int kPitch = DP + 4;  // floats: 16-byte loads of 8 rows hit all banks
  static constexpr int kP = BN + 4;
  static constexpr int kBytes = 4 * (64 * kPitch + 2 * BN * kPitch + 64 * kP) + 64;
};

__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int bytes, bool on) {
  // bytes 16 or 4; nothing but zeros arrives for `on` false
  if (bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(on ? 16 : 0)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
                 "r"(on ? 4 : 0)
                 : "memory");
}

// Rows [r0, r1) of `src` (row stride in elements, cols floats) into dst [..][pitch];
// rows from `have` on and columns from cols to DP are zeros.
template <int DP>
__device__ __forceinline__ void copy_tile(float* dst, int pitch, int r0, int r1, const float* src,
                                          int64_t stride, int have, int cols, bool vec) {
  const uint32_t d = smem_u32(dst);
  if (vec) {
    for (int x = threadIdx.x; x < (r1 - r0) * (DP / 4); x += 256) {
      const int r = r0 + x / (DP / 4), c = x % (DP / 4) * 4;
      const bool on = r < have && c < cols;
      copy_async(d + (r * pitch + c) * 4, on ? src + r * stride + c : src, 16, on);
    }
  } else {
    for (int x = threadIdx.x; x < (r1 - r0) * DP; x += 256) {
      const int r = r0 + x / DP, c = x % DP;
      const bool on = r < have && c < cols;
      copy_async(d + (r * pitch + c) * 4, on ? src + r * stride + c : src, 4, on);
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

template <int DP, bool PACKED>
__global__ void __launch_bounds__(256) window_f32_kernel(const WindowParams p, const WindowJobs w,
                                                         int vec) {
  using L = WinF32<DP>;
  constexpr int BN = L::BN, NC = BN / 16, NO = DP / 64;
  extern __shared__ float4 smem_f4[];
  float* sq = reinterpret_cast<float*>(smem_f4);
  float* sk = sq + 64 * L::kPitch;
  float* sv = sk + BN * L::kPitch;
  float* sp = sv + BN * L::kPitch;
  uint32_t* redo = reinterpret_cast<uint32_t*>(sp + 64 * L::kP);  // [2] rows that are not finite
  uint32_t* bad_keys = redo + 2;                                  // [2] keys of a block
  WinJob j;
  if (!window_job<1, BN, PACKED>(p, w, blockIdx.x, j)) return;  // the same for every warp
  const WinTile tile = j.tile[0];
  const float* q = static_cast<const float*>(p.q) + j.b * p.q_sb + j.h0 * p.q_sh +
                   static_cast<int64_t>(j.qt + j.q0) * p.q_st;
  const float* k = static_cast<const float*>(p.k) + j.b * p.k_sb + j.hk * p.k_sh + j.kt * p.k_st;
  const float* v = static_cast<const float*>(p.v) + j.b * p.v_sb + j.hk * p.v_sh + j.kt * p.v_st;
  float* o = static_cast<float*>(p.o) + j.b * p.o_sb + j.h0 * p.o_sh +
             static_cast<int64_t>(j.qt + j.q0) * p.o_st;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  if (threadIdx.x < 4) redo[threadIdx.x] = 0;  // bad_keys too

  // queries: row r is head r / tok, token r % tok
  const int wide_q = vec & kVecQ ? 4 : 1;
  for (int x = threadIdx.x; x < 64 * DP / wide_q; x += 256) {
    const int r = x * wide_q / DP, c = x * wide_q % DP, h = r / w.tok, t = r - h * w.tok;
    const bool on = h < j.nh && t < tile.n && c < p.d;
    copy_async(smem_u32(sq + r * L::kPitch + c), on ? q + h * p.q_sh + t * p.q_st + c : q,
               4 * wide_q, on);
  }
  auto first_of = [&](int i) { return (i < j.head ? i : i + j.jump) * BN; };
  auto load = [&](float* dst, const float* src, int64_t stride, int i, int cols) {
    const int at = first_of(i);
    const int2 span = window_span<BN>(j, tile, i);
    copy_tile<DP>(dst, L::kPitch, span.x, span.y, src + at * stride, stride, min(BN, j.lk - at),
                  cols, (vec & kVecKv) != 0);
  };
  auto whole_tile = [&](auto turn) {
    constexpr bool kClean = decltype(turn)::value;
    float m[4], l[4], acc[4][NO][4];
    uint32_t dirty = 0;  // bit a: row a of the thread sees a key that was cleaned
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      m[a] = -INFINITY;
      l[a] = 0.f;
#pragma unroll
      for (int c = 0; c < NO; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[a][c][e] = 0.f;
    }
    if (j.blocks > 0) load(sk, k, p.k_st, 0, p.d);
    for (int i = 0; i < j.blocks; ++i) {
      load(sv, v, p.v_st, i, p.dv);
      asm volatile("cp.async.wait_group 1;" ::: "memory");  // the keys
      __syncthreads();
      float s[4][NC];
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int c = 0; c < NC; ++c) s[a][c] = 0.f;
      // the 32-key columns that some row sees
      const int2 span = window_span<BN>(j, tile, i);
      auto scores = [&](auto from, auto to) {
        constexpr int C0 = decltype(from)::value, C1 = decltype(to)::value;
#pragma unroll 4
        for (int d = 0; d < DP; d += 4) {
          float4 x[4], y[NC];
#pragma unroll
          for (int a = 0; a < 4; ++a)
            x[a] = *reinterpret_cast<const float4*>(sq + (ty * 4 + a) * L::kPitch + d);
#pragma unroll
          for (int c = C0; c < C1; ++c)
            y[c] = *reinterpret_cast<const float4*>(sk + (tx + 16 * c) * L::kPitch + d);
#pragma unroll
          for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int c = C0; c < C1; ++c) {
              s[a][c] = fmaf(x[a].x, y[c].x, s[a][c]);
              s[a][c] = fmaf(x[a].y, y[c].y, s[a][c]);
              s[a][c] = fmaf(x[a].z, y[c].z, s[a][c]);
              s[a][c] = fmaf(x[a].w, y[c].w, s[a][c]);
            }
        }
      };
      using std::integral_constant;
      if (BN == 32 || span.y - span.x > 32)
        scores(integral_constant<int, 0>{}, integral_constant<int, NC>{});
      else if (span.x == 0)
        scores(integral_constant<int, 0>{}, integral_constant<int, 2>{});
      else
        scores(integral_constant<int, NC - 2>{}, integral_constant<int, NC>{});
      const int key0 = first_of(i);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int r = ty * 4 + a, h = r / w.tok, t = r - h * w.tok, at = tile.pf + t;
        const bool valid = h < j.nh && t < tile.n;
        float top = m[a];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int key = key0 + tx + 16 * c;
          const bool sees = valid && key <= at && (key > at - w.window || key < w.sinks);
          s[a][c] = sees ? s[a][c] * p.scale : -INFINITY;
          top = fmaxf(top, s[a][c]);
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float ref = top == -INFINITY ? 0.f : top;
        const float f = expf(m[a] - ref);
        m[a] = top;
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float e = expf(s[a][c] - ref);
          sum += e;
          sp[r * L::kP + tx + 16 * c] = e;
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        l[a] = l[a] * f + sum;
#pragma unroll
        for (int c = 0; c < NO; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[a][c][e] *= f;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");  // the values
      __syncthreads();                                       // and nobody needs the keys any more
      if constexpr (kClean) {
        // the clean turn, as above: keys whose values are not finite, which rows see them,
        // and zeros in their place
        constexpr int kParts = 256 / BN;
        const int n = threadIdx.x / kParts, part = threadIdx.x % kParts;
        const bool on = n >= span.x && n < span.y;
        bool found = false;
        for (int c = part; on && c < DP; c += kParts) found |= !isfinite(sv[n * L::kPitch + c]);
        if (found) atomicOr(&bad_keys[n >> 5], 1u << (n & 31));
        __syncthreads();
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const int r = ty * 4 + a, at = tile.pf + r % w.tok;
#pragma unroll
          for (int c = 0; c < BN / 32; ++c)
            if (bad_keys[c] & window_sees(w, at, key0 + c * 32)) dirty |= 1u << a;
        }
        for (int c = part; on && ((bad_keys[n >> 5] >> (n & 31)) & 1u) && c < DP; c += kParts)
          sv[n * L::kPitch + c] = 0.f;
        __syncthreads();
        if (threadIdx.x < 2) bad_keys[threadIdx.x] = 0;
      }
      if (i + 1 < j.blocks) load(sk, k, p.k_st, i + 1, p.d);
#pragma unroll 2
      for (int n = span.x; n < span.y; n += 4) {
        float4 x[4];
#pragma unroll
        for (int a = 0; a < 4; ++a)
          x[a] = *reinterpret_cast<const float4*>(sp + (ty * 4 + a) * L::kP + n);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
          for (int c = 0; c < NO; ++c) {
            const float4 y =
                *reinterpret_cast<const float4*>(sv + (n + u) * L::kPitch + c * 64 + tx * 4);
#pragma unroll
            for (int a = 0; a < 4; ++a) {
              const float e = u == 0 ? x[a].x : u == 1 ? x[a].y : u == 2 ? x[a].z : x[a].w;
              acc[a][c][0] = fmaf(e, y.x, acc[a][c][0]);
              acc[a][c][1] = fmaf(e, y.y, acc[a][c][1]);
              acc[a][c][2] = fmaf(e, y.z, acc[a][c][2]);
              acc[a][c][3] = fmaf(e, y.w, acc[a][c][3]);
            }
          }
        }
      }
      __syncthreads();  // the values and the weights may be overwritten
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // a job without keys, too
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int r = ty * 4 + a, h = r / w.tok, t = r - h * w.tok;
      if (h >= j.nh || t >= tile.n) continue;
      float odd = 0.f;
      float* row = o + h * p.o_sh + t * p.o_st;
#pragma unroll
      for (int c = 0; c < NO; ++c) {
        const int col = c * 64 + tx * 4;
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] = l[a] == 0.f ? 0.f : acc[a][c][e] / l[a];
          odd = fmaf(y[e], 0.f, odd);
        }
        if ((vec & kVecO) != 0 && col < p.dv) {
          *reinterpret_cast<float4*>(row + col) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < p.dv) row[col + e] = y[e];
        }
      }
      if (!(odd == 0.f) || ((dirty >> a) & 1u)) atomicOr(&redo[r >> 5], 1u << (r & 31));
    }
    __syncthreads();
  };
  whole_tile(std::false_type{});
  if ((redo[0] | redo[1]) == 0u) return;
  __syncthreads();
  if (threadIdx.x < 2) redo[threadIdx.x] = 0;
  whole_tile(std::true_type{});
  for (int r = threadIdx.x >> 5; r < 64; r += 8) {
    if (!((redo[r >> 5] >> (r & 31)) & 1u)) continue;
    const int h = r / w.tok, t = r - h * w.tok;
    window_row<float>(q + h * p.q_sh + t * p.q_st, k, v, o + h * p.o_sh + t * p.o_st, p.k_st,
                      p.v_st, p.d, p.dv, p.scale, p.window, p.sinks, tile.pf + t);
  }
}

}  // namespace bio

namespace {

constexpr int64_t kMaxGrid = 2147483647;

// Tiles of `rows` query rows, `tiles_per_job` of them in a job.
int plan_jobs(const bio::WindowParams& p, const bio_attn_args* a, bool packed, int rows,
              int tiles_per_job, bio::WindowJobs* w) {
  const int64_t group = p.group;
  w->hblocks = static_cast<int>((group + 15) / 16);  // up to 16 heads of a group in a tile
  w->gh = static_cast<int>((group + w->hblocks - 1) / w->hblocks);
  w->tok = rows / w->gh;
  const int64_t span = static_cast<int64_t>(tiles_per_job) * w->tok;
  const int64_t tiles = a->kv_heads * w->hblocks;
  const int64_t qblocks = (p.lq + span - 1) / span + (packed ? p.nseq : 0);
  const int64_t jobs = qblocks * tiles * (packed ? 1 : p.batch);
  if (qblocks > kMaxGrid || jobs > (1 << 30)) return BIO_ERR_SHAPE;
  w->qblocks = static_cast<int>(qblocks);
  w->jobs = static_cast<int>(jobs);
  w->by_qblocks = bio::fixed_div(qblocks);
  w->by_tiles = bio::fixed_div(tiles);
  w->by_hblocks = bio::fixed_div(w->hblocks);
  w->window = static_cast<int>(std::min<int64_t>(p.window, 1 << 30));
  w->sinks = static_cast<int>(std::min<int64_t>(p.sinks, 1 << 30));
  w->negate = p.scale < 0.f;
  // a scale of 0 weighs every visible key alike; hidden ones stay at -inf
  const float scale = (w->negate ? -p.scale : p.scale) * 1.4426950408889634f;
  w->scale_log2 = scale == 0.f ? 1.17549435e-38f : scale;
  w->vec_out = 0;
  return BIO_OK;
}

template <int DP, bool PACKED>
int launch_f32(const bio::WindowParams& p, const bio_attn_args* a, cudaStream_t s) {
  using L = bio::WinF32<DP>;
  static std::once_flag once[bio_host::kMaxDevices];
  cudaError_t set = cudaSuccess;
  std::call_once(once[a->device], [&] {
    set = cudaFuncSetAttribute(bio::window_f32_kernel<DP, PACKED>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  });
  if (set != cudaSuccess) return BIO_ERR_LAUNCH;
  bio::WindowJobs w;
  const int st = plan_jobs(p, a, PACKED, 64, 1, &w);
  if (st != BIO_OK) return st;
  auto on16 = [](const void* x, int64_t strides) {
    return (reinterpret_cast<uint64_t>(x) | 4 * static_cast<uint64_t>(strides)) % 16 == 0;
  };
  int vec = 0;
  if (on16(p.k, p.k_sb | p.k_sh | p.k_st | p.d) && on16(p.v, p.v_sb | p.v_sh | p.v_st | p.dv))
    vec |= bio::kVecKv;
  if (on16(p.q, p.q_sb | p.q_sh | p.q_st | p.d)) vec |= bio::kVecQ;
  if (on16(p.o, p.o_sb | p.o_sh | p.o_st | p.dv)) vec |= bio::kVecO;
  bio::window_f32_kernel<DP, PACKED><<<static_cast<unsigned>(w.jobs), 256, L::kBytes, s>>>(p, w,
                                                                                           vec);
  return bio_host::launch_status(cudaGetLastError());
}

int launch_float(const bio::WindowParams& p, const bio_attn_args* a, bool packed, cudaStream_t s) {
  const int dim = std::max(p.d, p.dv);
  if (packed)
    return dim <= 64    ? launch_f32<64, true>(p, a, s)
           : dim <= 128 ? launch_f32<128, true>(p, a, s)
                        : launch_f32<256, true>(p, a, s);
  return dim <= 64    ? launch_f32<64, false>(p, a, s)
         : dim <= 128 ? launch_f32<128, false>(p, a, s)
                      : launch_f32<256, false>(p, a, s);
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
  const int st = plan_jobs(p, a, PACKED, 128, L::NT, &w);
  if (st != BIO_OK) return st;
  const uint64_t out_bits = reinterpret_cast<uint64_t>(p.o) |
                            2 * static_cast<uint64_t>(p.o_sb | p.o_sh | p.o_st | p.dv);
  w.vec_out = out_bits % 32 == 0 ? 2 : out_bits % 16 == 0 ? 1 : 0;
  CUtensorMap q, k, v;
  const int64_t batch = packed ? 1 : p.batch;
  // without keys nothing is read through K and V: any operand will do for their maps
  auto keys_map = [&](CUtensorMap* map, const void* x, int64_t cols, int64_t st, int64_t sh,
                      int64_t sb) {
    return p.lk == 0 ? bio_host::map_of<T>(map, p.q, p.d, 1, 1, 1, 0, 0, 0, L::BN)
                     : bio_host::map_of<T>(map, x, cols, p.lk, a->kv_heads, batch, st, sh, sb,
                                           L::BN);
  };
  if (!bio_host::map_of<T>(&q, p.q, p.d, p.lq, p.heads, batch, p.q_st, p.q_sh, p.q_sb, w.tok,
                           w.gh) ||
      !keys_map(&k, p.k, p.d, p.k_st, p.k_sh, p.k_sb) ||
      !keys_map(&v, p.v, p.dv, p.v_st, p.v_sh, p.v_sb))
    return BIO_ERR_ALIGN;
  const unsigned grid = static_cast<unsigned>(std::min(w.jobs, sms));
  bio::window_tc_kernel<T, DP, PACKED><<<grid, L::kThreads, L::kBytes, s>>>(q, k, v, p, w);
  return bio_host::launch_status(cudaGetLastError());
}

template <typename T>
int launch_half(const bio::WindowParams& p, const bio_attn_args* a, bool packed, cudaStream_t s) {
  // the stride of a dimension of one element is never used
  const int64_t batch = packed ? 1 : p.batch;
  auto used = [](int64_t n, int64_t stride) {
    return 2 * static_cast<uint64_t>(n > 1 ? stride : 0);
  };
  uint64_t bits = reinterpret_cast<uint64_t>(p.q) | used(batch, p.q_sb) | used(p.heads, p.q_sh) |
                  used(p.lq, p.q_st);
  if (p.lk > 0)
    bits |= reinterpret_cast<uint64_t>(p.k) | reinterpret_cast<uint64_t>(p.v) |
            used(batch, p.k_sb | p.v_sb) | used(a->kv_heads, p.k_sh | p.v_sh) |
            used(p.lk, p.k_st | p.v_st);
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
    case BIO_F32: return launch_float(p, a, packed, s);
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
