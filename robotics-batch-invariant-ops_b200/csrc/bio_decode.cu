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
    st = dispatch_simt<T, false>(p, batch, s);
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
