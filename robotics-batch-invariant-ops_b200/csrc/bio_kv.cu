// Pages of a key/value cache: writing new tokens, growing, freeing and
// branching sequences, and moving the pages in use into another pool.
//
// All of it is data movement and integer bookkeeping on the device (page
// table, lengths, reference counts), with no host synchronisation.  Page
// numbers never depend on the order in which threads run: reference counts
// change by integer atomics, which commute, and free pages are handed out in
// the order of their numbers by one block that scans the counts.
//
// Not in the reference, which keeps no cache between calls.
#include <algorithm>

#include "bio_tile.cuh"

namespace bio {

struct KvPool {
  char* k;
  char* v;
  int64_t layers, pages;
  int heads, page_size;
  int64_t k_sl, k_sp, k_sh, k_st;  // bytes
  int64_t v_sl, v_sp, v_sh, v_st;
  int k_row, v_row;                // bytes of one token of one head
};

struct KvTable {
  int32_t* table;
  int64_t t_sr;
  int64_t rows, width;
  int32_t* lens;
  int32_t* refs;
  int64_t pages;
  int page_size;
  int* status;
};

// A later kernel of a chain starts while the one before it drains, and waits
// here until that one's writes are visible.
__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void chain_start_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ bool in_pool(int page, int64_t pages) {
  return page >= 0 && page < pages;
}

// ---------------------------------------------------------------------------
// append: one warp per token, V-wide loads, the token's keys then its values.
// DRAM bounds it (32752 tokens of 8 heads of 128, 268 MB moved: 48 us, 5.6 TB/s;
// eight loads in flight per lane instead of four cost registers: 54 us); for one
// token of each of 64 rows the call itself does (11 us, 3 us of it on the device).
// ---------------------------------------------------------------------------
constexpr int kAppendWarps = 4;

template <typename V>
__global__ void __launch_bounds__(kAppendWarps * 32)
    kv_append_kernel(const KvPool pool, const KvTable tb, const char* __restrict__ k, int64_t k_st,
                     int64_t k_sh, const char* __restrict__ v, int64_t v_st, int64_t v_sh,
                     const int32_t* __restrict__ rows, const int32_t* __restrict__ positions,
                     int64_t tokens, const FixedDiv by_vk, const FixedDiv by_vv) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kAppendWarps + (threadIdx.x >> 5);
  if (t >= tokens) return;
  const int row = rows[t], pos = positions[t];
  if (pos < 0) return;
  const int col = pos / pool.page_size, slot = pos - col * pool.page_size;
  const bool in = row >= 0 && row < tb.rows && col < tb.width;
  const int page = in ? tb.table[row * tb.t_sr + col] : -1;
  if (!in_pool(page, pool.pages)) {
    if (lane == 0) raise_status(tb.status, BIO_DEV_INDEX);
    return;
  }
  const unsigned vk = by_vk.n, vv = by_vv.n;  // vectors of one head
  const unsigned nk = vk * pool.heads, n = nk + vv * pool.heads;
  const char* ks = k + t * k_st;
  const char* vs = v + t * v_st;
  char* kd = pool.k + page * pool.k_sp + slot * pool.k_st;
  char* vd = pool.v + page * pool.v_sp + slot * pool.v_st;
  constexpr int U = 4;  // loads in flight per lane
  for (unsigned i0 = lane; i0 < n; i0 += 32 * U) {
    V val[U];
    char* to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned i = i0 + 32 * u;
      to[u] = nullptr;
      if (i >= n) continue;
      const bool key = i < nk;
      const unsigned j = key ? i : i - nk, w = key ? vk : vv;
      const unsigned h = key ? by_vk.quotient(j) : by_vv.quotient(j), c = (j - h * w) * sizeof(V);
      val[u] = *reinterpret_cast<const V*>((key ? ks + h * k_sh : vs + h * v_sh) + c);
      to[u] = (key ? kd + h * pool.k_sh : vd + h * pool.v_sh) + c;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (to[u] != nullptr) *reinterpret_cast<V*>(to[u]) = val[u];
  }
}

// ---------------------------------------------------------------------------
// free and evict: one block per listed row
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;

// Whether row rows[i] appears earlier in the list (block-wide answer).
__device__ __forceinline__ bool seen_before(const int32_t* rows, int64_t i) {
  const int r = rows[i];
  int hit = 0;
  for (int64_t j = threadIdx.x; j < i; j += blockDim.x) hit |= rows[j] == r;
  return __syncthreads_or(hit) != 0;
}

// window < 0: release everything and set the length to 0.
__global__ void __launch_bounds__(kRowThreads)
    kv_release_kernel(const KvTable tb, const int32_t* __restrict__ rows, int64_t window,
                      int64_t sinks) {
  const int64_t i = blockIdx.x;
  const int r = rows[i];
  const bool bad = r < 0 || r >= tb.rows;
  if (seen_before(rows, i) || bad) {
    if (threadIdx.x == 0) raise_status(tb.status, BIO_DEV_INDEX);
    return;
  }
  int64_t lo = 0, hi = tb.width;  // columns [lo, hi) go
  if (window >= 0) {
    const int64_t p = tb.page_size, gone = static_cast<int64_t>(tb.lens[r]) - window;
    lo = (sinks + p - 1) / p;
    hi = gone > 0 ? min(tb.width, gone / p) : 0;
  }
  for (int64_t c = lo + threadIdx.x; c < hi; c += blockDim.x) {
    int32_t* e = tb.table + r * tb.t_sr + c;
    if (in_pool(*e, tb.pages)) atomicSub(&tb.refs[*e], 1);
    *e = -1;
  }
  if (window < 0 && threadIdx.x == 0) tb.lens[r] = 0;
}

// ---------------------------------------------------------------------------
// fork, first kernel: one block per branch.  Releases and shares change
// different rows' entries, and the counts by atomics, so all branches run at
// once.  want[i]: 1 page for a partial last page, 0 none, -1 skipped.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kRowThreads)
    kv_fork_table_kernel(const KvTable tb, const int32_t* __restrict__ src,
                         const int32_t* __restrict__ dst, int64_t n, int32_t* __restrict__ want) {
  chain_start_next();
  const int64_t i = blockIdx.x;
  const int s = src[i], d = dst[i];
  int bad = s < 0 || s >= tb.rows || d < 0 || d >= tb.rows;
  for (int64_t j = threadIdx.x; j < n; j += blockDim.x)
    bad |= src[j] == d || (j != i && dst[j] == d);
  const int64_t len = bad ? 0 : tb.lens[s];
  bad |= len < 0 || len > tb.width * tb.page_size;
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) {
      want[i] = -1;
      raise_status(tb.status, BIO_DEV_INDEX);
    }
    return;
  }
  const int64_t full = len / tb.page_size;
  for (int64_t c = threadIdx.x; c < tb.width; c += blockDim.x) {
    int32_t* e = tb.table + d * tb.t_sr + c;
    const int old = *e;
    int now = c < full ? tb.table[s * tb.t_sr + c] : -1;
    if (now >= tb.pages) {
      raise_status(tb.status, BIO_DEV_INDEX);
      now = -1;
    }
    if (in_pool(old, tb.pages)) atomicSub(&tb.refs[old], 1);
    if (now >= 0) atomicAdd(&tb.refs[now], 1);
    *e = now < 0 ? -1 : now;
  }
  if (threadIdx.x == 0) {
    const bool part = len % tb.page_size != 0;
    const bool held = part && in_pool(tb.table[s * tb.t_sr + full], tb.pages);
    if (part && !held) raise_status(tb.status, BIO_DEV_INDEX);
    want[i] = held ? 1 : 0;
  }
}

// ---------------------------------------------------------------------------
// One block hands out the lowest free pages: request i's columns first(i) ..
// first(i) + want[i] of its row take the next ones in order.  The block scans
// the counts 4096 at a time and stops when every request is served.
// ---------------------------------------------------------------------------
constexpr int kScanThreads = 1024;

// Exclusive sum over the block; *total gets the sum.  Two barriers.
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  const int ws = lane < kScanThreads / 32 ? warp_sums[lane] : 0;
  int wi = ws;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, wi, o);
    if (lane >= o) wi += y;
  }
  *total = __shfl_sync(0xffffffffu, wi, 31);
  const int base = __shfl_sync(0xffffffffu, wi - ws, warp);
  __syncthreads();
  return base + inc - x;
}

template <bool FORK>
__global__ void __launch_bounds__(kScanThreads)
    kv_assign_kernel(const KvTable tb, const int32_t* __restrict__ src,
                     const int32_t* __restrict__ rows, const int32_t* __restrict__ new_lens,
                     int64_t n, int32_t* __restrict__ want, int32_t* __restrict__ first_of) {
  // rows: the rows that grow (dst of a fork).  want[i], then the running sum
  // before request i in first_of[i]; first_of[n] is the number of pages asked.
  __shared__ int sums[32];
  if (FORK) {
    chain_start_next();
    chain_wait();
  }
  const int64_t P = tb.page_size;
  int asked = 0;
  for (int64_t i0 = 0; i0 < n; i0 += kScanThreads) {
    const int64_t i = i0 + threadIdx.x;
    int w = 0;
    if (i < n) {
      if (FORK) {
        w = want[i];
      } else {
        const int r = rows[i], want_len = new_lens[i];
        bool bad = r < 0 || r >= tb.rows || want_len < 0 || want_len > tb.width * P;
        for (int64_t j = 0; j < i; ++j) bad |= rows[j] == r;
        const int64_t len = bad ? 0 : tb.lens[r];
        bad |= len < 0 || len > tb.width * P;
        if (bad) raise_status(tb.status, BIO_DEV_INDEX);
        w = bad ? -1 : static_cast<int>(max(static_cast<int64_t>(0),
                                            (want_len + P - 1) / P - (len + P - 1) / P));
        want[i] = w;
      }
      w = max(w, 0);
    }
    int total;
    const int before = block_scan(w, sums, &total);
    if (i < n) first_of[i] = asked + before;
    asked += total;
  }
  if (threadIdx.x == 0) first_of[n] = asked;
  __syncthreads();
  auto first_column = [&](int64_t i) -> int64_t {
    return FORK ? tb.lens[src[i]] / P : (tb.lens[rows[i]] + P - 1) / P;
  };
  int found = 0;
  for (int64_t p0 = 0; p0 < tb.pages && found < asked; p0 += 4 * kScanThreads) {
    const int64_t p = p0 + 4 * threadIdx.x;
    bool free_page[4];
    int mine = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      free_page[u] = p + u < tb.pages && tb.refs[p + u] == 0;
      mine += free_page[u];
    }
    int total;
    int rank = found + block_scan(mine, sums, &total);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (!free_page[u]) continue;
      if (rank < asked) {
        int64_t lo = 0, hi = n;  // the last request that starts at or before rank
        while (hi - lo > 1) {
          const int64_t mid = (lo + hi) >> 1;
          if (first_of[mid] <= rank) lo = mid; else hi = mid;
        }
        tb.table[rows[lo] * tb.t_sr + first_column(lo) + rank - first_of[lo]] =
            static_cast<int32_t>(p + u);
        tb.refs[p + u] = 1;
      }
      ++rank;
    }
    found += total;
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < n; i += kScanThreads) {
    const int w = want[i];
    if (w < 0) continue;
    const int got = max(0, min(w, found - first_of[i]));
    const int64_t room = (first_column(i) + got) * P;
    if (got < w) raise_status(tb.status, BIO_DEV_PAGES);
    const int r = rows[i];
    const int64_t len = FORK ? tb.lens[src[i]] : new_lens[i];
    const int64_t now = min(len, room);
    if (FORK) {
      tb.lens[r] = static_cast<int32_t>(now);
    } else if (now > tb.lens[r]) {
      tb.lens[r] = static_cast<int32_t>(now);
    }
  }
}

// fork, last kernel: the tokens of the partial page.  Block (i, x) copies them
// for branch i in K or V of a layer (unit u = x, x + parts, ... of 2 * layers), so
// that the chain of loads that finds the pages is walked once for all its units.
// 128 branches in 32 layers (240 MB moved): 46 us with both kernels before it, which
// wait on memory latency; eight branches in 18 layers 17 us, 9 us on the device.
template <typename V>
__global__ void __launch_bounds__(kRowThreads)
    kv_fork_copy_kernel(const KvPool pool, const KvTable tb, const int32_t* __restrict__ src,
                        const int32_t* __restrict__ dst, const int32_t* __restrict__ want,
                        unsigned parts, const FixedDiv by_vk, const FixedDiv by_vv) {
  chain_wait();
  const unsigned i = blockIdx.x / parts;
  if (want[i] <= 0) return;
  const int s = src[i], d = dst[i];
  const int len = tb.lens[s], part = len % pool.page_size;
  if (tb.lens[d] != len) return;  // the pool had no page left
  const int64_t full = len / pool.page_size;
  const int64_t from = tb.table[s * tb.t_sr + full], to = tb.table[d * tb.t_sr + full];
  constexpr int U = 4;
  for (int64_t u0 = blockIdx.x - i * parts; u0 < 2 * pool.layers; u0 += parts) {
    const bool key = (u0 & 1) == 0;
    const int64_t sh = key ? pool.k_sh : pool.v_sh, st = key ? pool.k_st : pool.v_st;
    char* base = key ? pool.k + (u0 >> 1) * pool.k_sl : pool.v + (u0 >> 1) * pool.v_sl;
    const char* read = base + from * (key ? pool.k_sp : pool.v_sp);
    char* write = base + to * (key ? pool.k_sp : pool.v_sp);
    const FixedDiv by_w = key ? by_vk : by_vv;  // vectors of a token of a head
    const unsigned n = by_w.n * part * pool.heads;
    for (unsigned i0 = threadIdx.x; i0 < n; i0 += kRowThreads * U) {
      V val[U];
      int64_t off[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const unsigned x = i0 + kRowThreads * u;
        off[u] = -1;
        if (x >= n) continue;
        const int row = by_w.quotient(x), h = static_cast<unsigned>(row) / static_cast<unsigned>(part);
        off[u] = h * sh + (row - h * part) * st + (x - row * by_w.n) * sizeof(V);
        val[u] = *reinterpret_cast<const V*>(read + off[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (off[u] >= 0) *reinterpret_cast<V*>(write + off[u]) = val[u];
    }
  }
}

// ---------------------------------------------------------------------------
// compact, first kernel: new number of every page in use (its rank), the list
// of pages in use, and the new counts.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kScanThreads)
    kv_rank_kernel(const int32_t* __restrict__ refs, int64_t pages, int32_t* __restrict__ out_refs,
                   int64_t out_pages, int32_t* __restrict__ rank_of, int32_t* __restrict__ in_use,
                   int* status) {
  // rank_of[pages], in_use[1 + pages]: in_use[0] the number of pages that move
  __shared__ int sums[32];
  chain_start_next();
  int64_t found = 0;
  for (int64_t p0 = 0; p0 < pages; p0 += 4 * kScanThreads) {
    const int64_t p = p0 + 4 * threadIdx.x;
    int ref[4], mine = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      ref[u] = p + u < pages ? refs[p + u] : 0;
      mine += ref[u] > 0;
    }
    int total;
    int64_t rank = found + block_scan(mine, sums, &total);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (p + u >= pages) continue;
      const bool moves = ref[u] > 0 && rank < out_pages;
      rank_of[p + u] = moves ? static_cast<int32_t>(rank) : -1;
      if (moves) {
        in_use[1 + rank] = static_cast<int32_t>(p + u);
        out_refs[rank] = ref[u];
      }
      rank += ref[u] > 0;
    }
    found += total;
  }
  if (found > out_pages && threadIdx.x == 0) raise_status(status, BIO_DEV_PAGES);
  const int64_t moved = min(found, out_pages);
  if (threadIdx.x == 0) in_use[0] = static_cast<int32_t>(moved);
  for (int64_t p = moved + threadIdx.x; p < out_pages; p += kScanThreads) out_refs[p] = 0;
}

// compact, second kernel: the table, then the pages.  Block (x, y, z) copies
// pieces z, z + gridDim.z, ... of U * kRowThreads vectors of pages x, x +
// gridDim.x, ... of one layer's K or V (y, y + gridDim.y, ...): no division to
// find a page, and none inside it where its bytes lie together (FLAT).  DRAM
// bounds it: 2500 pages of 16 layers (5.2 GB moved) 840 us, 6.2 TB/s.  With
// divisions per vector the issue of instructions did: 1476 us.
struct KvCopySide {
  const char* from;
  char* to;
  int64_t from_sl, from_sp, from_s1, from_s2, to_sl, to_sp, to_s1, to_s2;  // bytes
  unsigned per;               // vectors of a page: runs of by_run.n vectors in groups of by_n2.n
  FixedDiv by_run, by_n2;
};

__device__ __forceinline__ uint4 load_once(const uint4* p) { return __ldcs(p); }
__device__ __forceinline__ uint2 load_once(const uint2* p) { return __ldcs(p); }
__device__ __forceinline__ unsigned load_once(const unsigned* p) { return __ldcs(p); }
__device__ __forceinline__ unsigned short load_once(const unsigned short* p) { return __ldcs(p); }

template <typename V, bool FLAT>
__global__ void __launch_bounds__(kRowThreads, 4)
    kv_compact_kernel(const KvCopySide ks, const KvCopySide vs, int64_t layers, const KvTable tb,
                      const KvTable out, const int32_t* __restrict__ rank_of,
                      const int32_t* __restrict__ in_use) {
  chain_wait();
  const int64_t block = (static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x +
                        blockIdx.x;
  const int64_t threads = static_cast<int64_t>(gridDim.x) * gridDim.y * gridDim.z * kRowThreads;
  for (int64_t x = block * kRowThreads + threadIdx.x; x < tb.rows * tb.width; x += threads) {
    const int64_t r = x / tb.width, c = x - r * tb.width;
    const int page = tb.table[r * tb.t_sr + c];
    if (page >= tb.pages) raise_status(tb.status, BIO_DEV_INDEX);
    out.table[r * out.t_sr + c] = in_pool(page, tb.pages) ? rank_of[page] : -1;
  }
  constexpr int U = 8;
  constexpr unsigned kPiece = U * kRowThreads;
  const int moved = in_use[0];
  for (int64_t y = blockIdx.y; y < 2 * layers; y += gridDim.y) {
    const KvCopySide& c = (y & 1) == 0 ? ks : vs;
    const unsigned per = c.per;
    auto offset = [&](unsigned v, int64_t s1, int64_t s2) -> int64_t {
      if (FLAT) return static_cast<int64_t>(v) * sizeof(V);
      const int r = c.by_run.quotient(v), i1 = c.by_n2.quotient(r);
      return i1 * s1 + (r - i1 * static_cast<int>(c.by_n2.n)) * s2 +
             static_cast<int64_t>(v - r * c.by_run.n) * sizeof(V);
    };
    for (int64_t rank = blockIdx.x; rank < moved; rank += gridDim.x) {
      const char* from = c.from + (y >> 1) * c.from_sl + in_use[1 + rank] * c.from_sp;
      char* to = c.to + (y >> 1) * c.to_sl + rank * c.to_sp;
      for (unsigned at = blockIdx.z * kPiece; at < per; at += gridDim.z * kPiece) {
        V val[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const unsigned v = at + u * kRowThreads + threadIdx.x;
          if (v < per)
            val[u] = load_once(reinterpret_cast<const V*>(from + offset(v, c.from_s1, c.from_s2)));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const unsigned v = at + u * kRowThreads + threadIdx.x;
          if (v < per) __stcs(reinterpret_cast<V*>(to + offset(v, c.to_s1, c.to_s2)), val[u]);
        }
      }
    }
  }
}

}  // namespace bio

namespace {

int elem_bytes(int32_t dtype) {
  return dtype == BIO_F32 ? 4 : (dtype == BIO_F16 || dtype == BIO_BF16) ? 2 : 0;
}

constexpr int64_t kMaxInt = 2147483647;

int check_pool(const bio_kv_pool* p) {
  if (p == nullptr) return BIO_ERR_ARG;
  if (elem_bytes(p->dtype) == 0) return BIO_ERR_DTYPE;
  if (p->layers < 0 || p->pages < 0 || p->pages > kMaxInt || p->kv_heads < 1 ||
      p->kv_heads > 65536 || p->page_size < 1 || p->page_size > 65536 || p->d < 1 ||
      p->d > 65536 || p->dv < 1 || p->dv > 65536)
    return BIO_ERR_SHAPE;
  // vectors of a page are counted in 32 bits
  if (p->kv_heads * p->page_size > (1 << 28) / (p->d > p->dv ? p->d : p->dv)) return BIO_ERR_SHAPE;
  if (p->layers > 0 && p->pages > 0 && (p->k == nullptr || p->v == nullptr)) return BIO_ERR_ARG;
  return BIO_OK;
}

int check_table(const bio_kv_table* t, bool lens, bool refs) {
  if (t == nullptr) return BIO_ERR_ARG;
  if (t->rows < 0 || t->rows > kMaxInt || t->width < 0 || t->width > kMaxInt || t->pages < 0 ||
      t->pages > kMaxInt || t->page_size < 1 || t->page_size > 65536)
    return BIO_ERR_SHAPE;
  if (t->rows > 0 && t->width > 0 && t->page_table == nullptr) return BIO_ERR_ARG;
  if (lens && t->rows > 0 && t->seq_lens == nullptr) return BIO_ERR_ARG;
  if (refs && t->pages > 0 && t->ref_counts == nullptr) return BIO_ERR_ARG;
  return BIO_OK;
}

bio::KvPool pool_view(const bio_kv_pool* p) {
  const int64_t e = elem_bytes(p->dtype);
  bio::KvPool v;
  v.k = static_cast<char*>(p->k);
  v.v = static_cast<char*>(p->v);
  v.layers = p->layers;
  v.pages = p->pages;
  v.heads = static_cast<int>(p->kv_heads);
  v.page_size = static_cast<int>(p->page_size);
  v.k_sl = p->k_sl * e; v.k_sp = p->k_sp * e; v.k_sh = p->k_sh * e; v.k_st = p->k_st * e;
  v.v_sl = p->v_sl * e; v.v_sp = p->v_sp * e; v.v_sh = p->v_sh * e; v.v_st = p->v_st * e;
  v.k_row = static_cast<int>(p->d * e);
  v.v_row = static_cast<int>(p->dv * e);
  return v;
}

bio::KvTable table_view(const bio_kv_table* t) {
  bio::KvTable v;
  v.table = t->page_table;
  v.t_sr = t->t_sr;
  v.rows = t->rows;
  v.width = t->width;
  v.lens = t->seq_lens;
  v.refs = t->ref_counts;
  v.pages = t->pages;
  v.page_size = static_cast<int>(t->page_size);
  v.status = bio_host::status_word(t->device);
  return v;
}

// Widest vector (16, 8, 4 or 2 bytes) that every one of these byte offsets is a multiple of.
struct Width {
  uint64_t bits = 16;
  void add(const void* p) { bits |= reinterpret_cast<uint64_t>(p); }
  void add(int64_t n) { bits |= static_cast<uint64_t>(n); }
  void add(const bio::KvPool& p) {
    add(p.k); add(p.v);
    add(p.k_sl); add(p.k_sp); add(p.k_sh); add(p.k_st); add(p.k_row);
    add(p.v_sl); add(p.v_sp); add(p.v_sh); add(p.v_st); add(p.v_row);
  }
  int bytes() const { return static_cast<int>(bits & (~bits + 1)); }
};

// Launch that may overlap the end of the kernel before it on the stream; the
// kernel waits for that one itself (chain_wait).
template <typename... P, typename... A>
int launch_chained(void (*kernel)(P...), dim3 grid, unsigned block, cudaStream_t s,
                   A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return bio_host::launch_status(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
}

template <typename F>
int with_width(int bytes, F f) {
  switch (bytes) {
    case 16: return f(uint4{});
    case 8: return f(uint2{});
    case 4: return f(uint32_t{});
    case 2: return f(uint16_t{});
    default: return BIO_ERR_ALIGN;  // a pointer that no element can have
  }
}

}  // namespace

extern "C" {

int bio_kv_append(const bio_kv_pool* pool, const bio_kv_table* table, const void* k, int64_t k_st,
                  int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, const int32_t* rows,
                  const int32_t* positions, int64_t tokens, void* stream) {
  int st = check_pool(pool);
  if (st == BIO_OK) st = check_table(table, false, false);
  if (st != BIO_OK) return st;
  if (pool->layers != 1 || table->page_size != pool->page_size || tokens < 0) return BIO_ERR_SHAPE;
  if (tokens == 0) return BIO_OK;
  if (k == nullptr || v == nullptr || rows == nullptr || positions == nullptr) return BIO_ERR_ARG;
  const int64_t blocks = (tokens + bio::kAppendWarps - 1) / bio::kAppendWarps;
  if (blocks > kMaxInt) return BIO_ERR_SHAPE;
  st = bio_host::ensure_device(pool->device);
  if (st != BIO_OK) return st;
  const bio::KvPool p = pool_view(pool);
  const bio::KvTable t = table_view(table);
  const int64_t e = elem_bytes(pool->dtype);
  Width w;
  w.add(p);
  w.add(k); w.add(v);
  w.add(k_st * e); w.add(k_sh * e); w.add(v_st * e); w.add(v_sh * e);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return with_width(w.bytes(), [&](auto vec) {
    using V = decltype(vec);
    bio::kv_append_kernel<V><<<static_cast<unsigned>(blocks), bio::kAppendWarps * 32, 0, s>>>(
        p, t, static_cast<const char*>(k), k_st * e, k_sh * e, static_cast<const char*>(v),
        v_st * e, v_sh * e, rows, positions, tokens, bio::fixed_div(p.k_row / sizeof(V)),
        bio::fixed_div(p.v_row / sizeof(V)));
    return bio_host::launch_status(cudaGetLastError());
  });
}

int64_t bio_kv_workspace(int64_t n, int64_t pages) {
  if (n < 0 || pages < 0 || n > kMaxInt || pages > kMaxInt) return 0;
  const int64_t rows = 2 * n + 1, moved = 2 * pages + 1;
  return 4 * (rows > moved ? rows : moved);
}

int bio_kv_extend(const bio_kv_table* table, const int32_t* rows, const int32_t* new_lens,
                  int64_t n, void* workspace, int64_t workspace_bytes, void* stream) {
  int st = check_table(table, true, true);
  if (st != BIO_OK) return st;
  if (n < 0 || n > kMaxInt) return BIO_ERR_SHAPE;
  if (n == 0) return BIO_OK;
  if (rows == nullptr || new_lens == nullptr || workspace == nullptr) return BIO_ERR_ARG;
  if (workspace_bytes < 4 * (2 * n + 1)) return BIO_ERR_SCRATCH;
  st = bio_host::ensure_device(table->device);
  if (st != BIO_OK) return st;
  int32_t* ws = static_cast<int32_t*>(workspace);
  bio::kv_assign_kernel<false><<<1, bio::kScanThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      table_view(table), nullptr, rows, new_lens, n, ws, ws + n);
  return bio_host::launch_status(cudaGetLastError());
}

static int release(const bio_kv_table* table, const int32_t* rows, int64_t n, int64_t window,
                   int64_t sinks, void* stream) {
  int st = check_table(table, true, true);
  if (st != BIO_OK) return st;
  if (n < 0 || n > kMaxInt) return BIO_ERR_SHAPE;
  if (n == 0) return BIO_OK;
  if (rows == nullptr) return BIO_ERR_ARG;
  st = bio_host::ensure_device(table->device);
  if (st != BIO_OK) return st;
  bio::kv_release_kernel<<<static_cast<unsigned>(n), bio::kRowThreads, 0,
                           static_cast<cudaStream_t>(stream)>>>(table_view(table), rows, window,
                                                                sinks);
  return bio_host::launch_status(cudaGetLastError());
}

int bio_kv_free(const bio_kv_table* table, const int32_t* rows, int64_t n, void* stream) {
  return release(table, rows, n, -1, 0, stream);
}

int bio_kv_evict(const bio_kv_table* table, const int32_t* rows, int64_t n, int64_t window,
                 int64_t sinks, void* stream) {
  if (window < 1 || window > kMaxInt || sinks < 0 || sinks > kMaxInt) return BIO_ERR_ARG;
  return release(table, rows, n, window, sinks, stream);
}

int bio_kv_fork(const bio_kv_pool* pool, const bio_kv_table* table, const int32_t* src,
                const int32_t* dst, int64_t n, void* workspace, int64_t workspace_bytes,
                void* stream) {
  int st = check_pool(pool);
  if (st == BIO_OK) st = check_table(table, true, true);
  if (st != BIO_OK) return st;
  if (table->page_size != pool->page_size || table->pages != pool->pages || n < 0)
    return BIO_ERR_SHAPE;
  if (n == 0) return BIO_OK;
  if (src == nullptr || dst == nullptr || workspace == nullptr) return BIO_ERR_ARG;
  if (n > kMaxInt / 2 || pool->layers > kMaxInt / 2 / n) return BIO_ERR_SHAPE;
  if (workspace_bytes < 4 * (2 * n + 1)) return BIO_ERR_SCRATCH;
  st = bio_host::ensure_device(pool->device);
  if (st != BIO_OK) return st;
  const int sms = bio_host::sm_count(pool->device);
  if (sms <= 0) return BIO_ERR_LAUNCH;
  const bio::KvPool p = pool_view(pool);
  const bio::KvTable t = table_view(table);
  int32_t* ws = static_cast<int32_t*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  bio::kv_fork_table_kernel<<<static_cast<unsigned>(n), bio::kRowThreads, 0, s>>>(t, src, dst, n,
                                                                                  ws);
  st = bio_host::launch_status(cudaGetLastError());
  if (st != BIO_OK) return st;
  st = launch_chained(bio::kv_assign_kernel<true>, 1, bio::kScanThreads, s, t, src, dst,
                      static_cast<const int32_t*>(nullptr), n, ws, ws + n);
  if (st != BIO_OK || pool->layers == 0) return st;
  Width w;
  w.add(p);
  return with_width(w.bytes(), [&](auto vec) {
    using V = decltype(vec);
    // as many blocks as run at once, and a unit for each at least
    const int64_t parts =
        std::max<int64_t>(1, std::min(2 * p.layers, (static_cast<int64_t>(sms) * 8 + n - 1) / n));
    return launch_chained(bio::kv_fork_copy_kernel<V>, static_cast<unsigned>(n * parts),
                          bio::kRowThreads, s, p, t, src, dst, ws, static_cast<unsigned>(parts),
                          bio::fixed_div(p.k_row / sizeof(V)), bio::fixed_div(p.v_row / sizeof(V)));
  });
}

int bio_kv_compact(const bio_kv_pool* pool, const bio_kv_table* table, const bio_kv_pool* out_pool,
                   const bio_kv_table* out_table, void* workspace, int64_t workspace_bytes,
                   void* stream) {
  int st = check_pool(pool);
  if (st == BIO_OK) st = check_pool(out_pool);
  if (st == BIO_OK) st = check_table(table, false, true);
  if (st == BIO_OK) st = check_table(out_table, false, true);
  if (st != BIO_OK) return st;
  if (pool->dtype != out_pool->dtype) return BIO_ERR_DTYPE;
  if (pool->layers != out_pool->layers || pool->kv_heads != out_pool->kv_heads ||
      pool->page_size != out_pool->page_size || pool->d != out_pool->d ||
      pool->dv != out_pool->dv || table->rows != out_table->rows ||
      table->width != out_table->width || table->pages != pool->pages ||
      out_table->pages != out_pool->pages || pool->device != out_pool->device)
    return BIO_ERR_SHAPE;
  if (workspace == nullptr) return BIO_ERR_ARG;
  if (workspace_bytes < 4 * (2 * pool->pages + 1)) return BIO_ERR_SCRATCH;
  st = bio_host::ensure_device(pool->device);
  if (st != BIO_OK) return st;
  const int sms = bio_host::sm_count(pool->device);
  if (sms <= 0) return BIO_ERR_LAUNCH;
  const bio::KvPool p = pool_view(pool), q = pool_view(out_pool);
  const bio::KvTable t = table_view(table), o = table_view(out_table);
  int32_t* rank_of = static_cast<int32_t*>(workspace);
  int32_t* in_use = rank_of + pool->pages;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  bio::kv_rank_kernel<<<1, bio::kScanThreads, 0, s>>>(t.refs, t.pages, o.refs, o.pages, rank_of,
                                                      in_use, t.status);
  st = bio_host::launch_status(cudaGetLastError());
  if (st != BIO_OK) return st;
  Width w;
  w.add(p);
  w.add(q);
  return with_width(w.bytes(), [&](auto vec) {
    using V = decltype(vec);
    auto side = [&](bool key) {
      bio::KvCopySide c;
      c.from = key ? p.k : p.v;
      c.to = key ? q.k : q.v;
      c.from_sl = key ? p.k_sl : p.v_sl; c.to_sl = key ? q.k_sl : q.v_sl;
      c.from_sp = key ? p.k_sp : p.v_sp; c.to_sp = key ? q.k_sp : q.v_sp;
      c.from_s1 = key ? p.k_sh : p.v_sh; c.to_s1 = key ? q.k_sh : q.v_sh;
      c.from_s2 = key ? p.k_st : p.v_st; c.to_s2 = key ? q.k_st : q.v_st;
      const int64_t row = key ? p.k_row : p.v_row;
      int64_t n1 = p.heads, n2 = p.page_size, run = row / sizeof(V);
      if (c.from_s2 == row && c.to_s2 == row) {  // a head's tokens lie together
        run *= n2;
        n2 = 1;
        if (c.from_s1 == row * p.page_size && c.to_s1 == c.from_s1) {  // and the heads do
          run *= n1;
          n1 = 1;
        }
      }
      c.per = static_cast<unsigned>(n1 * n2 * run);
      c.by_run = bio::fixed_div(run);
      c.by_n2 = bio::fixed_div(n2);
      return c;
    };
    const bio::KvCopySide key = side(true), value = side(false);
    constexpr unsigned kPiece = 8 * bio::kRowThreads;
    const unsigned most = std::max(key.per, value.per);
    dim3 grid;
    grid.y = static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(2 * p.layers, 1), 65535));
    grid.z = std::min((most + kPiece - 1) / kPiece, 64u);
    const int64_t wide = (static_cast<int64_t>(sms) * 8 + grid.y * grid.z - 1) / (grid.y * grid.z);
    grid.x = static_cast<unsigned>(std::max<int64_t>(std::min(wide, q.pages), 1));
    const bool flat = key.by_run.n == key.per && value.by_run.n == value.per;
    auto kernel = flat ? bio::kv_compact_kernel<V, true> : bio::kv_compact_kernel<V, false>;
    return launch_chained(kernel, grid, bio::kRowThreads, s, key, value, p.layers, t, o,
                          static_cast<const int32_t*>(rank_of),
                          static_cast<const int32_t*>(in_use));
  });
}

}  // extern "C"
