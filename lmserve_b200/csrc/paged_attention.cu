// Attention of a batch over its pages of one layer's paged cache, with or without prefixes that
// several requests share, for sm_100a.
//
// Row r = (token t, query head h) of request b reads the keys of its group's prefix (all of them)
// and the request's own keys j <= len - n + i, where n new tokens of the request are its last n
// keys and t is the i-th of them (causal; every key otherwise):
//   s_j = scale * q_r . k_j,  m = max s_j,  l = sum exp(s_j - m),  out_r = sum exp(s_j - m) v_j / l
//   lse_r = m + log l;  a row without any key: out = 0, lse = -inf.
// Scores, m, l and the accumulator are fp32; out is rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.cuh"

namespace lms {

namespace {

template <bool BF16>
__device__ __forceinline__ float2 up2(uint32_t w) {
  if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t down2(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Largest i in [0, n) with a[i] <= x, or -1 (a ascending).
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
  int lo = -1, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int list_keys(const PageList& l, int i, int block_size) {
  const int n = l.indptr[i + 1] - l.indptr[i];
  if (n <= 0) return 0;
  const int last = min(max(l.last[i], 0), block_size);
  return (n - 1) * block_size + last;
}

// Byte offset of key `key` of list i in either plane, or -1 where the page number or its place in
// the table is out of range (the key is then read as zeros; reported by the debug checks).
__device__ __forceinline__ long long key_offset(const AttentionParams& p, const PageList& l, int first, int key) {
  const int pg = key / p.block_size;
  const long long at = (long long)first + pg;
  if (at < 0 || at >= l.num_indices) return -1;
  const int page = l.indices[at];
  if (page < 0 || page >= p.num_blocks) {
    if (p.checks) report(p.err, kErrBadPage, kWhereAttention, at, page);
    return -1;
  }
  return (long long)page * p.block_stride + (long long)(key - pg * p.block_size) * p.slot_stride;
}

// One warp a row; a lane owns the element pairs lane, lane + 32, ... of the head.
constexpr int kMaxPairs = 4;

template <bool BF16>
__global__ void __launch_bounds__(128) attention_rows_kernel(const AttentionParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(row / p.num_heads), h = (int)(row - (long long)t * p.num_heads);
  if (t >= p.num_tokens) return;
  int b = t, n_new = 1, i = 0;
  if (p.qo_indptr != nullptr) {
    b = last_not_above(p.qo_indptr, p.num_requests + 1, t);
    if (b < 0 || b >= p.num_requests) return;  // behind the last request: left as it is
    n_new = p.qo_indptr[b + 1] - p.qo_indptr[b];
    i = t - p.qo_indptr[b];
  }
  const int pairs = p.head_dim / 2;
  const int kv_head_bytes = (h / (p.num_heads / p.num_kv_heads)) * p.head_dim * 2;
  const uint32_t* q = reinterpret_cast<const uint32_t*>(p.q + (long long)t * p.q_tok + (long long)h * p.head_dim * 2);
  float2 qv[kMaxPairs], acc[kMaxPairs];
#pragma unroll
  for (int e = 0; e < kMaxPairs; ++e) {
    const int at = lane + 32 * e;
    qv[e] = at < pairs ? up2<BF16>(q[at]) : make_float2(0.f, 0.f);
    acc[e] = make_float2(0.f, 0.f);
  }
  float m = -INFINITY, l = 0.f;
  for (int part = 0; part < 2; ++part) {
    const PageList& list = part == 0 ? p.prefix : p.own;
    if (list.indptr == nullptr) continue;
    int which = b;
    if (part == 0) {
      which = p.group_indptr != nullptr ? last_not_above(p.group_indptr, p.num_groups + 1, b) : 0;
      if (which < 0 || which >= p.num_groups) continue;
    }
    const int len = list_keys(list, which, p.block_size);
    const int end = part == 1 && p.causal ? min(len, len - n_new + i + 1) : len;
    const int first = list.indptr[which];
    for (int key = 0; key < end; ++key) {
      const long long off = key_offset(p, list, first, key);
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(p.kcache + off + kv_head_bytes);
      const uint32_t* vp = reinterpret_cast<const uint32_t*>(p.vcache + off + kv_head_bytes);
      float s = 0.f;
      float2 v[kMaxPairs];
#pragma unroll
      for (int e = 0; e < kMaxPairs; ++e) {
        const int at = lane + 32 * e;
        float2 k = make_float2(0.f, 0.f);
        v[e] = k;
        if (at < pairs && off >= 0) {
          k = up2<BF16>(kp[at]);
          v[e] = up2<BF16>(vp[at]);
        }
        s = fmaf(qv[e].x, k.x, fmaf(qv[e].y, k.y, s));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      s *= p.scale;
      const float top = fmaxf(m, s);
      const float keep = m == -INFINITY ? 0.f : __expf(m - top);
      const float w = s == -INFINITY ? 0.f : __expf(s - top);
      m = top;
      l = l * keep + w;
#pragma unroll
      for (int e = 0; e < kMaxPairs; ++e) {
        acc[e].x = fmaf(w, v[e].x, acc[e].x * keep);
        acc[e].y = fmaf(w, v[e].y, acc[e].y * keep);
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint32_t* o = reinterpret_cast<uint32_t*>(p.out + (long long)t * p.o_tok + (long long)h * p.head_dim * 2);
#pragma unroll
  for (int e = 0; e < kMaxPairs; ++e)
    if (lane + 32 * e < pairs) o[lane + 32 * e] = down2<BF16>(acc[e].x * inv, acc[e].y * inv);
  if (p.lse != nullptr && lane == 0) p.lse[row] = l > 0.f ? m + __logf(l) : -INFINITY;
}

}  // namespace

long long attention_workspace_bytes(const AttentionParams&, int) { return 0; }

cudaError_t launch_attention(const AttentionParams& p, int, bool pdl, int* launches, cudaStream_t stream) {
  const long long ctas = ((long long)p.num_tokens * p.num_heads + 3) / 4;
  if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  *launches = 1;
  return p.is_bf16 ? cudaLaunchKernelEx(&cfg, attention_rows_kernel<true>, p)
                   : cudaLaunchKernelEx(&cfg, attention_rows_kernel<false>, p);
}

}  // namespace lms
