// Prefill attention with a sliding window and sink tokens (dense and packed).
//
// Query i sits at position p = i + (lk - lq) and sees key j iff j <= p and
// (j > p - window or j < sinks):
//   o_i = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q_i.k_j.
// A row that sees no key (p < 0) gives zeros.
//
// One warp owns one query row.  It walks the row's visible keys in order, 32
// at a time: lane j computes the score of key j, the maximum and the sum of
// exponentials use a fixed xor-shuffle tree, and lane t accumulates output
// columns t, t + 32, ....  Keys that the row does not see are never read, and
// nothing depends on the other rows of the launch.
//
// Not in the reference, whose SDPA (batch_invariant_ops.py:1148-1213) would
// need the mask as a tensor and visits every key.
#include "bio_common.cuh"

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

template <typename T, bool PACKED>
__global__ void __launch_bounds__(kWinWarps * 32) window_row_kernel(const WindowParams p) {
  __shared__ float qs[kWinWarps][kWinDims];
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
  T* out = static_cast<T*>(p.o) + bq * p.o_sb + h * p.o_sh + t * p.o_st;
  const T* qrow = static_cast<const T*>(p.q) + bq * p.q_sb + h * p.q_sh + t * p.q_st;
  const T* kb = static_cast<const T*>(p.k) + bq * p.k_sb + h / p.group * p.k_sh + k0 * p.k_st;
  const T* vb = static_cast<const T*>(p.v) + bq * p.v_sb + h / p.group * p.v_sh + k0 * p.v_st;
  for (int c = lane; c < p.d; c += 32) qs[warp][c] = to_f32(qrow[c]);
  __syncwarp();

  // visible keys u = 0..n-1: key u < few ? u : u + skip
  const int64_t lo = max(static_cast<int64_t>(0), pos - p.window + 1);
  const int64_t few = min(p.sinks, lo), skip = lo - few;
  const int64_t n = max(static_cast<int64_t>(0), pos + 1 - skip);
  float m = -INFINITY, l = 0.f, o[kWinDims / 32];
#pragma unroll
  for (int e = 0; e < kWinDims / 32; ++e) o[e] = 0.f;
  for (int64_t u0 = 0; u0 < n; u0 += 32) {
    const int64_t u = u0 + lane;
    float s = -INFINITY;
    if (u < n) {
      const T* krow = kb + (u < few ? u : u + skip) * p.k_st;
      float a = 0.f;
      for (int c = 0; c < p.d; ++c) a = fmaf(qs[warp][c], to_f32(krow[c]), a);
      s = a * p.scale;
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
      const T* vrow = vb + (uj < few ? uj : uj + skip) * p.v_st;
#pragma unroll
      for (int e = 0; e < kWinDims / 32; ++e) {
        const int c = lane + 32 * e;
        if (c < p.dv) o[e] = fmaf(wj, to_f32(vrow[c]), o[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < kWinDims / 32; ++e) {
    const int c = lane + 32 * e;
    if (c < p.dv) out[c] = from_f32<T>(l == 0.f ? 0.f : o[e] / l);
  }
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

int run_window(const bio_attn_args* a, int64_t window, int64_t sinks, bool packed, void* stream) {
  if (a == nullptr) return BIO_ERR_ARG;
  if (a->d < 1 || a->dv < 1 || a->d > bio::kWinDims || a->dv > bio::kWinDims)
    return BIO_ERR_SHAPE;
  if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->heads > 65536 ||
      a->batch < 0 || a->lq < 0 || a->lk < 0 || a->lq > kMaxGrid || a->lk > kMaxGrid)
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
    case BIO_F16: return launch_rows<__half>(p, packed, s);
    case BIO_BF16: return launch_rows<__nv_bfloat16>(p, packed, s);
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
