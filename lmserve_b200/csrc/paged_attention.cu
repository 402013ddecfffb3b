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


// ---------------------------------------------------------------- shared pieces of the matrix kernels
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void cp_async16(uint32_t smem, const void* gmem, bool valid) {
  const int bytes = valid ? 16 : 0;  // the rest of the 16 bytes is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A part of a row's softmax that another launch joins: out / l and lse in base 2.
struct Partials {
  float* lse;  // [slots][num_heads]
  float* out;  // [slots][num_heads][head_dim]
};

// ---------------------------------------------------------------- one token a request
// Bound by HBM: every K / V row is read once for the G = num_heads / num_kv_heads rows that share
// it.  The pages of all requests form one axis (kv_indptr's own), cut into 16-key units; CTA x of
// a head block takes the x-th equal run of units, whatever requests it meets, so the load is even
// for any mix of lengths and nothing is planned on the host.  A request inside one run is
// finished there; one cut by a border leaves a partial in each run (slot 2x if it began in an
// earlier run, else 2x + 1) for the join kernel.
//
// Inside a CTA a warp works alone: head hs = w % HB of the block, every KS-th 16-key tile of the
// run (KS = 8 / HB), its own ring of cp.async stages, no block-wide barrier in the loop.  Q (16
// rows, G of them used) stays in registers as the A operand of m16n8k16; K and V tiles are read
// with ldmatrix from rows swizzled by 16-byte chunk ^ (row & 7).  The KS warps of a head join
// their (m, l, out) through shared memory when a request ends.
constexpr int kDecodeWarps = 8;
constexpr int kTile = 16;  // keys

struct DecodeParams {
  AttentionParams a;
  Partials part;
  int n_ranges;        // equal runs of the page axis
  int hb_shift;        // log2 of the heads a CTA works on
  int units_per_page;  // 16-key units of a page
  int whole_slot;      // first slot of whole requests when a join follows for every row, else -1
};

struct TileMeta {
  int request;
  int keys;   // keys of the tile that exist
  int flags;  // 1: first tile of the request in this warp, 2: last
  int slot;   // where the result goes: -1 = the output row
};

template <int D, int NST>
struct DecodeSmem {
  static constexpr int kRow = D * 2;
  static constexpr int kStage = 2 * kTile * kRow;
  static constexpr int kRing = kDecodeWarps * NST * kStage;
  static constexpr int kMeta = kDecodeWarps * NST * (int)sizeof(TileMeta);
  static int bytes(int G, int hb) {
    const int join = hb < kDecodeWarps ? kDecodeWarps * G * (D + 2) * 4 : 0;
    return kRing + kMeta + join;
  }
};

template <bool BF16, int D, int NST>
__global__ void __launch_bounds__(kDecodeWarps * 32, 1) attention_decode_kernel(const DecodeParams p) {
  using S = DecodeSmem<D, NST>;
  extern __shared__ __align__(128) char smem[];
  constexpr int kSteps = D / 16, kChunks = D / 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int HB = 1 << p.hb_shift, KS = kDecodeWarps >> p.hb_shift;
  const int hs = warp & (HB - 1), ks = warp >> p.hb_shift;
  const int kvh = blockIdx.y * HB + hs;
  const AttentionParams& a = p.a;
  const int G = a.num_heads / a.num_kv_heads;
  const int UPP = p.units_per_page, BS = a.block_size;
  const uint32_t ring = smem_u32(smem) + warp * NST * S::kStage;
  TileMeta* meta = reinterpret_cast<TileMeta*>(smem + S::kRing) + warp * NST;
  float* joins = reinterpret_cast<float*>(smem + S::kRing + S::kMeta);

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (kvh >= a.num_kv_heads) return;  // all KS warps of such a head slot leave together

  // this CTA's run of units, [u_begin, u_end) of the page axis
  const int* indptr = a.own.indptr;
  const int B = a.num_requests;
  const long long axis0 = indptr[0];
  const long long units = ((long long)indptr[B] - axis0) * UPP;
  const long long chunk = (units + p.n_ranges - 1) / p.n_ranges;
  const long long u_begin = chunk * blockIdx.x, u_end = min(u_begin + chunk, units);
  if (u_begin >= u_end) return;

  // the request of the first unit: the last b with indptr[b] <= its page, 32 probes a round
  int b0 = 0;
  {
    const long long page = axis0 + u_begin / UPP;
    int lo = 0, n = B;  // the answer is in [lo, lo + n)
    while (n > 1) {
      const int step = (n + 31) / 32;
      const int at = lo + lane * step;
      const bool below = lane * step < n && indptr[at] <= page;
      const int last = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
      n = min(step, n - last * step);
      lo += last * step;
    }
    b0 = lo;
  }

  // Producer: walks the requests of the run, 32 of them loaded at a time (one a lane).
  int batch = b0, in_batch = -1;      // in_batch: index of the current request, -1 before the first
  long long my_first = 0, my_end = 0; // lane's request: its pages on the axis
  int my_last = 0;
  auto load_batch = [&]() {
    const int b = batch + lane;
    my_first = my_end = 0;
    my_last = 0;
    if (b < B) {
      my_first = indptr[b];
      my_end = indptr[b + 1];
      my_last = min(max(a.own.last[b], 0), BS);
    }
  };
  load_batch();
  int key = 0, key_end = 0, first_page = 0;  // of the current request: next tile of this warp, end
  int request = -1, slot = -1;
  bool fresh = false, done = false;          // fresh: no tile of the request issued yet

  auto key_of = [&](long long unit) { return (long long)(unit / UPP) * BS + (unit % UPP) * kTile; };
  auto next_request = [&]() {
    for (;;) {
      if (++in_batch == 32) {
        batch += 32;
        in_batch = 0;
        if (batch >= B) { done = true; return; }
        load_batch();
      }
      const long long first = __shfl_sync(0xffffffffu, my_first, in_batch);
      const long long end = __shfl_sync(0xffffffffu, my_end, in_batch);
      const int last = __shfl_sync(0xffffffffu, my_last, in_batch);
      request = batch + in_batch;
      if (request >= B) { done = true; return; }
      const long long s0 = (first - axis0) * UPP, s1 = (end - axis0) * UPP;  // its units
      if (s0 >= u_end) { done = true; return; }
      if (end <= first || s1 <= u_begin) continue;
      const long long len = (end - first - 1) * BS + last;
      const long long k0 = s0 < u_begin ? key_of(u_begin - s0) : 0;
      const long long k1 = s1 > u_end ? min(key_of(u_end - s0), len) : len;
      key = (int)min(k0, len) + ks * kTile;
      key_end = (int)k1;
      first_page = (int)first;
      const bool whole = s0 >= u_begin && s1 <= u_end;
      slot = whole ? (p.whole_slot < 0 ? -1 : p.whole_slot + request)
                   : 2 * (int)blockIdx.x + (s0 < u_begin ? 0 : 1);
      fresh = true;
      return;
    }
  };

  // Page numbers of the tile after the one being issued are fetched one tile ahead.
  const long long head_off = (long long)kvh * S::kRow;
  int row_page = 0;       // lane r < 16: page number of row r of the pending tile, -1 = none
  int pend_key = 0, pend_flags = 0, pend_keys = 0, pend_request = 0, pend_slot = 0;
  bool pending = false;
  auto fetch = [&]() {  // describe the next tile and start loading its page numbers
    pending = false;
    if (done) return;
    if (request < 0 || (!fresh && key >= key_end)) next_request();
    if (done) return;
    pend_flags = fresh ? 1 : 0;
    pend_request = request;
    pend_slot = slot;
    pend_key = key;
    pend_keys = max(0, min(kTile, key_end - key));
    key += KS * kTile;
    if (key >= key_end) pend_flags |= 2;
    fresh = false;
    pending = true;
    row_page = -1;
    if (lane < pend_keys) {
      const long long at = (long long)first_page + (pend_key + lane) / BS;
      if (at >= 0 && at < a.own.num_indices) {
        row_page = a.own.indices[at];
        if (row_page < 0 || row_page >= a.num_blocks) {
          if (a.checks) report(a.err, kErrBadPage, kWhereAttention, at, row_page);
          row_page = -1;
        }
      }
    }
  };
  auto issue = [&](int stage) {  // start the pending tile's copies; always one commit
    if (lane == 0) {
      TileMeta m;
      m.request = pending ? pend_request : -1;
      m.keys = pend_keys;
      m.flags = pend_flags;
      m.slot = pend_slot;
      meta[stage] = m;
    }
    if (pending) {
      long long off = -1;
      if (row_page >= 0)
        off = (long long)row_page * a.block_stride + (long long)((pend_key + lane) % BS) * a.slot_stride + head_off;
      const uint32_t base = ring + stage * S::kStage;
      constexpr int kRowsAtOnce = 32 / kChunks;
#pragma unroll
      for (int i = 0; i < kTile / kRowsAtOnce; ++i) {
        const int row = i * kRowsAtOnce + lane / kChunks, c = lane % kChunks;
        const long long o = __shfl_sync(0xffffffffu, off, row);
        const uint32_t dst = base + row * S::kRow + ((c ^ (row & 7)) << 4);
        const bool ok = o >= 0;
        cp_async16(dst, ok ? a.kcache + o + c * 16 : a.kcache, ok);
        cp_async16(dst + kTile * S::kRow, ok ? a.vcache + o + c * 16 : a.vcache, ok);
      }
    }
    cp_async_commit();
  };

  fetch();
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) {
    issue(s);
    if (pending) fetch();
  }

  // Consumer
  uint32_t q[kSteps][4];
  float o[D / 8][4];
  float m[2], l[2];
  const float scale2 = a.scale * kLog2e;
  const int r0 = lane >> 2, c0 = (lane & 3) * 2;
  for (int it = 0;; ++it) {
    const int stage = it % NST;
    cp_async_wait<NST - 2>();
    __syncwarp();
    const TileMeta t = meta[stage];
    if (t.request < 0) break;
    issue((it + NST - 1) % NST);
    if (pending) fetch();

    if (t.flags & 1) {
      const char* rows = a.q + (long long)t.request * a.q_tok + (long long)kvh * G * S::kRow + c0 * 2;
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = r0 + (e & 1) * 8;
          q[k][e] = r < G ? *reinterpret_cast<const uint32_t*>(rows + r * S::kRow + k * 32 + (e >> 1) * 16) : 0u;
        }
#pragma unroll
      for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
    }

    if (t.keys > 0) {
      const uint32_t kbase = ring + stage * S::kStage, vbase = kbase + kTile * S::kRow;
      float s[2][4] = {};
      {
        // matrices 0..3 of an ldmatrix: (keys 0-7, d lo) (keys 0-7, d hi) (keys 8-15, d lo) (keys 8-15, d hi)
        const int row = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t b[4];
          ldsm4(b, kbase + row * S::kRow + (((2 * k + half) ^ (row & 7)) << 4));
          mma16816<BF16>(s[0], q[k], b[0], b[1]);
          mma16816<BF16>(s[1], q[k], b[2], b[3]);
        }
      }
      float top[2] = {m[0], m[1]};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool live = n * 8 + c0 + (e & 1) < t.keys;
          s[n][e] = live ? s[n][e] * scale2 : -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      }
      if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float keep = m[i] == top[i] ? 1.f : exp2_fast(m[i] - top[i]);
          m[i] = top[i];
          l[i] *= keep;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][2 * i] *= keep;
            o[n][2 * i + 1] *= keep;
          }
        }
      }
      // The weights enter the second product in the element type, as a rounded part and the
      // rounded rest: two products, error 2^-16 instead of 2^-8, on pipes that HBM leaves idle.
      const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float w0 = exp2_fast(s[n][2 * i] - base[i]), w1 = exp2_fast(s[n][2 * i + 1] - base[i]);
          l[i] += w0 + w1;
          hi[2 * n + i] = down2<BF16>(w0, w1);
          const float2 h = up2<BF16>(hi[2 * n + i]);
          lo[2 * n + i] = down2<BF16>(w0 - h.x, w1 - h.y);
        }
      {
        // (keys 0-7, d n) (keys 8-15, d n) (keys 0-7, d n+1) (keys 8-15, d n+1), transposed
        const int row = lane & 15, half = lane >> 4;
#pragma unroll
        for (int n = 0; n < D / 8; n += 2) {
          uint32_t b[4];
          ldsm4_t(b, vbase + row * S::kRow + (((n + half) ^ (row & 7)) << 4));
          mma16816<BF16>(o[n], hi, b[0], b[1]);
          mma16816<BF16>(o[n + 1], hi, b[2], b[3]);
          mma16816<BF16>(o[n], lo, b[0], b[1]);
          mma16816<BF16>(o[n + 1], lo, b[2], b[3]);
        }
      }
    }

    if (t.flags & 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      }
      const int head0 = kvh * G;
      char* out = a.out + (long long)t.request * a.o_tok + (long long)head0 * S::kRow;
      float* lse = t.slot >= 0 ? p.part.lse + (long long)t.slot * a.num_heads + head0
                   : a.lse != nullptr ? a.lse + (long long)t.request * a.num_heads + head0 : nullptr;
      float* po = p.part.out + ((long long)max(t.slot, 0) * a.num_heads + head0) * D;
      const float unit = t.slot >= 0 ? 1.f : kLn2;  // partials keep base 2
      if (KS == 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = r0 + 8 * i;
          if (r >= G) continue;
          const float inv = l[i] > 0.f ? 1.f / l[i] : 0.f;
          if (lse != nullptr && c0 == 0) lse[r] = l[i] > 0.f ? (m[i] + log2f(l[i])) * unit : -INFINITY;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            const float x = o[n][2 * i] * inv, y = o[n][2 * i + 1] * inv;
            if (t.slot >= 0) *reinterpret_cast<float2*>(po + r * D + n * 8 + c0) = make_float2(x, y);
            else *reinterpret_cast<uint32_t*>(out + r * S::kRow + (n * 8 + c0) * 2) = down2<BF16>(x, y);
          }
        }
      } else {
        // [warp][G][D] accumulators, then [warp][G] maxima and sums
        float* jm = joins + kDecodeWarps * G * D;
        float* jl = jm + kDecodeWarps * G;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = r0 + 8 * i;
          if (r >= G) continue;
          if (c0 == 0) {
            jm[warp * G + r] = m[i];
            jl[warp * G + r] = l[i];
          }
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(joins + (warp * G + r) * D + n * 8 + c0) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + hs), "r"(KS * 32) : "memory");
        for (int e = ks * 32 + lane; e < G * (D / 2); e += KS * 32) {
          const int r = e / (D / 2), d = (e - r * (D / 2)) * 2;
          float mm = -INFINITY;
          for (int k = 0; k < KS; ++k) mm = fmaxf(mm, jm[(hs + k * HB) * G + r]);
          float ll = 0.f, x = 0.f, y = 0.f;
          if (mm != -INFINITY)
            for (int k = 0; k < KS; ++k) {
              const int w = (hs + k * HB) * G + r;
              const float f = exp2_fast(jm[w] - mm);
              const float2 v = *reinterpret_cast<const float2*>(joins + w * D + d);
              ll = fmaf(f, jl[w], ll);
              x = fmaf(f, v.x, x);
              y = fmaf(f, v.y, y);
            }
          const float inv = ll > 0.f ? 1.f / ll : 0.f;
          if (t.slot >= 0) *reinterpret_cast<float2*>(po + r * D + d) = make_float2(x * inv, y * inv);
          else *reinterpret_cast<uint32_t*>(out + r * S::kRow + d * 2) = down2<BF16>(x * inv, y * inv);
          if (d == 0 && lse != nullptr) lse[r] = ll > 0.f ? (mm + log2f(ll)) * unit : -INFINITY;
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + hs), "r"(KS * 32) : "memory");
      }
    }
  }
  cp_async_wait<0>();
}

// ---------------------------------------------------------------- join
// One warp a row: the row's partials, weighted by 2^(lse - max lse).  A row of a request that one
// run held whole is finished already; a request without any key gets its zeros here.
struct JoinParams {
  AttentionParams a;
  Partials part;
  int n_ranges, units_per_page;
};

template <bool BF16, int D>
__global__ void __launch_bounds__(128) attention_join_kernel(const JoinParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const AttentionParams& a = p.a;
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(row / a.num_heads), h = (int)(row - (long long)t * a.num_heads);
  if (t >= a.num_tokens) return;
  const int* indptr = a.own.indptr;
  const long long axis0 = indptr[0];
  const long long units = ((long long)indptr[a.num_requests] - axis0) * p.units_per_page;
  const long long chunk = (units + p.n_ranges - 1) / p.n_ranges;
  const long long s0 = (indptr[t] - axis0) * p.units_per_page, s1 = (indptr[t + 1] - axis0) * p.units_per_page;
  int x0 = 0, x1 = -1;  // the runs that hold a part of the request
  if (s1 > s0 && chunk > 0) {
    x0 = (int)min(max(s0 / chunk, 0ll), p.n_ranges - 1ll);
    x1 = (int)min(max((s1 - 1) / chunk, 0ll), p.n_ranges - 1ll);
    if (x0 == x1) return;
  }
  constexpr int E = D / 32;
  float acc[E] = {}, m = -INFINITY, l = 0.f;
  for (int x = x0; x <= x1; ++x) {
    const long long at = (long long)(2 * x + (x == x0 ? 1 : 0)) * a.num_heads + h;
    const float s = p.part.lse[at];
    if (s == -INFINITY) continue;
    const float top = fmaxf(m, s), keep = exp2_fast(m - top), w = exp2_fast(s - top);
    m = top;
    l = l * keep + w;
    const float* v = p.part.out + at * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(w, v[e], acc[e] * keep);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint32_t* out = reinterpret_cast<uint32_t*>(a.out + (long long)t * a.o_tok + ((long long)h * D + lane * E) * 2);
#pragma unroll
  for (int e = 0; e < E; e += 2) out[e / 2] = down2<BF16>(acc[e] * inv, acc[e + 1] * inv);
  if (a.lse != nullptr && lane == 0) a.lse[row] = l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
}

// ---------------------------------------------------------------- launch rules
// What a call launches, from its counts alone.
struct Plan {
  bool decode;         // one token a request, no shared prefix
  int n_ranges, hb_shift, units_per_page;
  long long slots;     // partials
};

Plan plan_of(const AttentionParams& p, int sms) {
  Plan r{};
  const int G = p.num_heads / p.num_kv_heads;
  r.units_per_page = (p.block_size + kTile - 1) / kTile;
  r.decode = p.qo_indptr == nullptr && p.own.indptr != nullptr && p.prefix.indptr == nullptr && G <= 16 &&
             (p.head_dim == 64 || p.head_dim == 128);
  if (r.decode) {
    // One CTA an SM.  The more heads a CTA takes, the fewer warps meet when a request ends, but
    // the shorter the runs: a run should hold 16 units at least for each request that it cuts.
    const long long units = (p.own.num_indices + 1) * r.units_per_page;
    int shift = 3;
    while (shift > 0 && (1 << (shift - 1)) >= p.num_kv_heads) --shift;
    auto blocks = [&](int s) { return (p.num_kv_heads + (1 << s) - 1) >> s; };
    while (shift > 0 && units * blocks(shift) < 16ll * sms) --shift;
    r.hb_shift = shift;
    r.n_ranges = sms / blocks(shift);
    if (r.n_ranges < 1) r.n_ranges = 1;
    r.slots = 2ll * r.n_ranges;
  }
  return r;
}

long long align256(long long x) { return (x + 255) & ~255ll; }

Partials partials_at(const AttentionParams& p, const Plan& plan) {
  Partials r;
  r.lse = reinterpret_cast<float*>(p.workspace);
  r.out = reinterpret_cast<float*>(p.workspace + align256(plan.slots * p.num_heads * 4));
  return r;
}

struct Launch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  Launch(dim3 grid, int threads, size_t smem, bool pdl, cudaStream_t stream) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
  }
};

template <bool BF16, int D, int NST>
cudaError_t launch_decode(const AttentionParams& p, const Plan& plan, bool pdl, int* launches, cudaStream_t stream) {
  DecodeParams d{};
  d.a = p;
  d.part = partials_at(p, plan);
  d.n_ranges = plan.n_ranges;
  d.hb_shift = plan.hb_shift;
  d.units_per_page = plan.units_per_page;
  d.whole_slot = -1;
  const int G = p.num_heads / p.num_kv_heads, HB = 1 << plan.hb_shift;
  auto kernel = attention_decode_kernel<BF16, D, NST>;
  const int smem = DecodeSmem<D, NST>::bytes(G, HB);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  Launch go(dim3(plan.n_ranges, (p.num_kv_heads + HB - 1) / HB), kDecodeWarps * 32, smem, pdl, stream);
  e = cudaLaunchKernelEx(&go.cfg, kernel, d);
  if (e != cudaSuccess) return e;
  JoinParams j{};
  j.a = p;
  j.part = d.part;
  j.n_ranges = plan.n_ranges;
  j.units_per_page = plan.units_per_page;
  const long long ctas = ((long long)p.num_tokens * p.num_heads + 3) / 4;
  if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  Launch join(dim3((unsigned)ctas), 128, 0, pdl, stream);
  *launches = 2;
  return cudaLaunchKernelEx(&join.cfg, attention_join_kernel<BF16, D>, j);
}

template <bool BF16>
cudaError_t launch_rows(const AttentionParams& p, bool pdl, int* launches, cudaStream_t stream) {
  const long long ctas = ((long long)p.num_tokens * p.num_heads + 3) / 4;
  if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  Launch go(dim3((unsigned)ctas), 128, 0, pdl, stream);
  *launches = 1;
  return cudaLaunchKernelEx(&go.cfg, attention_rows_kernel<BF16>, p);
}

template <bool BF16>
cudaError_t launch_typed(const AttentionParams& p, const Plan& plan, bool pdl, int* launches, cudaStream_t stream) {
  if (plan.decode) {
    const bool few = p.num_heads / p.num_kv_heads <= 8;
    if (p.head_dim == 64) return launch_decode<BF16, 64, 5>(p, plan, pdl, launches, stream);
    return few ? launch_decode<BF16, 128, 3>(p, plan, pdl, launches, stream)
               : launch_decode<BF16, 128, 2>(p, plan, pdl, launches, stream);
  }
  return launch_rows<BF16>(p, pdl, launches, stream);
}

}  // namespace

long long attention_workspace_bytes(const AttentionParams& p, int sms) {
  const Plan plan = plan_of(p, sms);
  if (plan.slots == 0) return 0;
  return align256(plan.slots * p.num_heads * 4) + plan.slots * p.num_heads * p.head_dim * 4;
}

cudaError_t launch_attention(const AttentionParams& p, int sms, bool pdl, int* launches, cudaStream_t stream) {
  const Plan plan = plan_of(p, sms);
  return p.is_bf16 ? launch_typed<true>(p, plan, pdl, launches, stream)
                   : launch_typed<false>(p, plan, pdl, launches, stream);
}

}  // namespace lms
