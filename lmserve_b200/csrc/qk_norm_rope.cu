// Norm of every query and key head, rotary position embedding and paged cache write in one
// pass over a layer's projections, for sm_100a.
//
// For a head x of D elements (the norm is taken before the rotation):
//   n = x * w / sqrt(mean(x^2) + eps)
//   out[i]       = n[i]       * cos[i]       - n[D/2 + i] * sin[i]
//   out[D/2 + i] = n[D/2 + i] * cos[D/2 + i] + n[i]       * sin[D/2 + i],   i < D/2
// with the weight row w shared by all query (or all key) heads and cos / sin the two halves of
// the position's row, as in rope_cache.cu.  Squares, their sum, the norm and the rotation are
// held in fp32; the one rounding to the element type is the store.
//
// One lane owns 8 consecutive elements of the first half and the 8 matching ones of the second
// (two 16-byte loads), D/16 lanes own a head - padded to the next power of two, so that the sum
// of squares is a butterfly over aligned lanes - and HPT heads of the token follow each other in
// a lane: their loads are in flight together and the cos / sin row is fetched once for all of
// them.  Heads are numbered [0, NH) = Q, [NH, NH+NKV) = K, [NH+NKV, NH+2*NKV) = V (copied).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.cuh"

namespace lms {

namespace {

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& r, float* f) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 v;
    if (BF16) {
      v.x = __uint_as_float(w[i] << 16);
      v.y = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (BF16) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 ldv(const char* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void stv(char* p, const uint4& v) { *reinterpret_cast<uint4*>(p) = v; }

// Bound by HBM for many tokens (q, k, v read and written once): 8192 tokens of 32 + 2 * 8 heads of 128,
// 206 MB, in 36.8 us, 5.6 TB/s; four heads a lane (1: 53 us, 2: 42, 6: 65), CTAs of 128 threads, 8 on an SM
// (64 registers; 256 threads at 80 registers: 40 us).
template <bool BF16, int HPT, int THREADS>
__global__ void __launch_bounds__(THREADS, 8)
qk_norm_rope_kernel(const QkNormRopeParams p, const int lane_shift, const int head_groups,
                    const long long n_items) {
  // item = (t * head_groups + hg) << lane_shift | j
  const long long item = (long long)blockIdx.x * THREADS + threadIdx.x;
  const int lanes = 1 << lane_shift;
  const int j = (int)(item & (lanes - 1));
  const long long q = item >> lane_shift;
  const bool live = item < n_items;
  int t, hg;
  if (n_items <= 0x7fffffffll) {
    t = (int)((unsigned)q / (unsigned)head_groups);
    hg = (int)((unsigned)q - (unsigned)t * (unsigned)head_groups);
  } else {
    t = (int)(q / head_groups);
    hg = (int)(q - (long long)t * head_groups);
  }
  const int half_bytes = p.head_dim;
  const int head_bytes = 2 * p.head_dim;
  const int vec = j * 16;
  const bool owns = live && vec < half_bytes;  // lanes past the head only take part in the shuffles
  const int heads_total = p.num_heads + p.num_kv_heads * (p.kcache != nullptr ? 2 : 1);

  const char* src[HPT];
  int head[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = hg + i * head_groups;
    head[i] = owns && h < heads_total ? h : -1;
    src[i] = h < p.num_heads ? p.q + (long long)t * p.q_tok + (long long)h * head_bytes
             : h < p.num_heads + p.num_kv_heads
                 ? p.k + (long long)t * p.k_tok + (long long)(h - p.num_heads) * head_bytes
                 : p.v + (long long)t * p.v_tok +
                       (long long)(h - p.num_heads - p.num_kv_heads) * head_bytes;
    if (head[i] >= 0 && (vec & 127) == 0) {  // hints only, as in rope_cache.cu
      prefetch_l2(src[i] + vec);
      prefetch_l2(src[i] + half_bytes + vec);
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  uint4 xr[HPT], yr[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    xr[i] = yr[i] = make_uint4(0, 0, 0, 0);
    if (head[i] >= 0) {
      xr[i] = ldv(src[i] + vec);
      yr[i] = ldv(src[i] + half_bytes + vec);
    }
  }
  long long pos = -1, slot = -1;
  if (owns) {
    pos = p.pos64 ? reinterpret_cast<const long long*>(p.positions)[t]
                  : (long long)reinterpret_cast<const int*>(p.positions)[t];
    if (p.kcache != nullptr) slot = p.slots[t];
  }
  // An index outside the table or the cache is never used: the token's rotated heads (or its
  // cache rows) stay unwritten, and the debug checks report it.
  const bool turn = owns && pos >= 0 && pos < p.max_pos;
  if (p.checks && owns && !turn && hg == 0 && j == 0) report(p.err, kErrBadPosition, kWhereQkNorm, t, pos);
  long long cache_off = -1;
  if (slot >= p.num_slots) {
    if (p.checks && hg == 0 && j == 0) report(p.err, kErrBadSlot, kWhereQkNorm, t, slot);
  } else if (slot >= 0) {
    long long blk, in;
    if (p.block_shift >= 0) {
      blk = slot >> p.block_shift;
      in = slot & ((1ll << p.block_shift) - 1);
    } else {
      blk = slot / p.block_size;
      in = slot - blk * p.block_size;
    }
    cache_off = blk * p.block_stride + in * p.slot_stride;
  }
  uint4 cs[4];
  cs[0] = cs[1] = cs[2] = cs[3] = make_uint4(0, 0, 0, 0);
  if (turn) {
    const char* row = p.cos_sin + pos * p.cs_row;
    cs[0] = ldv(row + vec);
    cs[1] = ldv(row + half_bytes + vec);
    cs[2] = ldv(row + head_bytes + vec);
    cs[3] = ldv(row + head_bytes + half_bytes + vec);
  }

  float inv[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {  // whole warps: lanes without a head add zeros
    float x[8], y[8];
    unpack8<BF16>(xr[i], x);
    unpack8<BF16>(yr[i], y);
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], fmaf(y[e], y[e], sum));
    for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    inv[i] = rsqrtf(sum * p.inv_dim + p.eps);
  }

#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = head[i];
    if (h < 0) continue;
    const bool is_q = h < p.num_heads;
    if (h >= p.num_heads + p.num_kv_heads) {  // V: plain copy into the cache
      if (cache_off >= 0) {
        char* d = p.vcache + cache_off + (long long)(h - p.num_heads - p.num_kv_heads) * head_bytes;
        stv(d + vec, xr[i]);
        stv(d + half_bytes + vec, yr[i]);
      }
      continue;
    }
    if (!turn) continue;
    const char* weight = is_q ? p.q_weight : p.k_weight;
    float x[8], y[8], w[8], c[8], s[8], ox[8], oy[8];
    unpack8<BF16>(xr[i], x);
    unpack8<BF16>(yr[i], y);
    unpack8<BF16>(ldv(weight + vec), w);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * inv[i] * w[e];
    unpack8<BF16>(ldv(weight + half_bytes + vec), w);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = y[e] * inv[i] * w[e];
    unpack8<BF16>(cs[0], c);
    unpack8<BF16>(cs[2], s);
#pragma unroll
    for (int e = 0; e < 8; ++e) ox[e] = fmaf(x[e], c[e], -(y[e] * s[e]));
    unpack8<BF16>(cs[1], c);
    unpack8<BF16>(cs[3], s);
#pragma unroll
    for (int e = 0; e < 8; ++e) oy[e] = fmaf(y[e], c[e], x[e] * s[e]);
    const uint4 a = pack8<BF16>(ox), b = pack8<BF16>(oy);
    if (is_q) {
      char* d = p.q_out + (long long)t * p.qo_tok + (long long)h * head_bytes;
      stv(d + vec, a);
      stv(d + half_bytes + vec, b);
      continue;
    }
    const long long kvh = (long long)(h - p.num_heads) * head_bytes;
    if (p.k_out != nullptr) {
      char* d = p.k_out + (long long)t * p.ko_tok + kvh;
      stv(d + vec, a);
      stv(d + half_bytes + vec, b);
    }
    if (cache_off >= 0) {
      stv(p.kcache + cache_off + kvh + vec, a);
      stv(p.kcache + cache_off + kvh + half_bytes + vec, b);
    }
  }
}

template <bool BF16, int HPT>
cudaError_t launch(const QkNormRopeParams& p, int lane_shift, int heads_total, bool pdl,
                   cudaStream_t stream) {
  constexpr int THREADS = 128;
  const int head_groups = (heads_total + HPT - 1) / HPT;
  const long long n_items = ((long long)p.num_tokens * head_groups) << lane_shift;
  const long long ctas = (n_items + THREADS - 1) / THREADS;
  if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<BF16, HPT, THREADS>, p, lane_shift,
                            head_groups, n_items);
}

}  // namespace

cudaError_t launch_qk_norm_rope(const QkNormRopeParams& p_in, int sms, bool pdl, cudaStream_t stream) {
  QkNormRopeParams p = p_in;
  p.block_shift = -1;
  if (p.block_size > 0 && (p.block_size & (p.block_size - 1)) == 0) {
    p.block_shift = 0;
    while ((1 << p.block_shift) < p.block_size) ++p.block_shift;
  }
  p.inv_dim = 1.0f / (float)p.head_dim;
  int lane_shift = 0;
  while ((16 << lane_shift) < p.head_dim) ++lane_shift;
  const int heads_total = p.num_heads + p.num_kv_heads * (p.kcache != nullptr ? 2 : 1);
  // One head a lane while the launch fits the GPU at once: the chain of a lane is what such a
  // call waits for.
  const long long lanes = ((long long)p.num_tokens * heads_total) << lane_shift;
  const bool one = lanes <= 2048ll * sms;
  if (p.is_bf16)
    return one ? launch<true, 1>(p, lane_shift, heads_total, pdl, stream)
               : launch<true, 4>(p, lane_shift, heads_total, pdl, stream);
  return one ? launch<false, 1>(p, lane_shift, heads_total, pdl, stream)
             : launch<false, 4>(p, lane_shift, heads_total, pdl, stream);
}

}  // namespace lms
