// Attention of a batch over its pages of one layer's paged cache, with or without prefixes that
// several requests share, for sm_100a.
//
// Row r = (token t, query head h) of request b reads the keys of its group's prefix (all of them)
// and the request's own keys j <= len - n + i, where n new tokens of the request are its last n
// keys and t is the i-th of them (causal; every key otherwise):
//   s_j = scale * q_r . k_j,  m = max s_j,  l = sum exp(s_j - m),  out_r = sum exp(s_j - m) v_j / l
//   lse_r = m + log l;  a row without any key: out = 0, lse = -inf.
// Scores, m, l and the accumulator are fp32; out is rounded once.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

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

// Towards zero.
template <bool BF16>
__device__ __forceinline__ uint32_t down2_rz(float a, float b) {
  uint32_t r;
  if (BF16) asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
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

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// One warp, one row: a lane owns the element pairs lane, lane + 32, ... of the head, up to PAIRS of
// them.  Scores in base 2.  Keys that are not walked are not touched.
template <bool BF16>
struct RowWalk {
  static constexpr int PAIRS = 4;
  float2 q[PAIRS], acc[PAIRS];
  float m = -INFINITY, l = 0.f;

  __device__ __forceinline__ RowWalk(const char* row, int head_dim, int lane) {
#pragma unroll
    for (int e = 0; e < PAIRS; ++e) {
      const int at = lane + 32 * e;
      q[e] = at < head_dim / 2 ? up2<BF16>(reinterpret_cast<const uint32_t*>(row)[at]) : make_float2(0.f, 0.f);
      acc[e] = make_float2(0.f, 0.f);
    }
  }
  __device__ __forceinline__ void walk(const AttentionParams& p, const PageList& list, int first_page, int kvh,
                                       int key, int end, int lane) {
    const int head = kvh * p.head_dim * 2;
    for (; key < end; ++key) {
      const long long off = key_offset(p, list, first_page, key);
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(p.kcache + off + head);
      const uint32_t* vp = reinterpret_cast<const uint32_t*>(p.vcache + off + head);
      float s = 0.f;
      float2 v[PAIRS];
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) {
        const int at = lane + 32 * e;
        float2 k = make_float2(0.f, 0.f);
        v[e] = k;
        if (at < p.head_dim / 2 && off >= 0) {
          k = up2<BF16>(kp[at]);
          v[e] = up2<BF16>(vp[at]);
        }
        s = fmaf(q[e].x, k.x, fmaf(q[e].y, k.y, s));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      s *= p.scale * kLog2e;
      const float top = fmaxf(m, s);
      const float keep = m == -INFINITY ? 0.f : exp2_fast(m - top);
      const float w = s == -INFINITY ? 0.f : exp2_fast(s - top);
      m = top;
      l = l * keep + w;
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) {
        acc[e].x = fmaf(w, v[e].x, acc[e].x * keep);
        acc[e].y = fmaf(w, v[e].y, acc[e].y * keep);
      }
    }
  }
  __device__ __forceinline__ float inverse() const { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }  // NaN stays
  __device__ __forceinline__ float lse2() const { return l == 0.f ? -INFINITY : m + log2f(l); }
  __device__ __forceinline__ void store(char* out, int head_dim, int lane) const {
    const float inv = inverse();
#pragma unroll
    for (int e = 0; e < PAIRS; ++e)
      if (lane + 32 * e < head_dim / 2)
        reinterpret_cast<uint32_t*>(out)[lane + 32 * e] = down2<BF16>(acc[e].x * inv, acc[e].y * inv);
  }
};

// Any head dim: one warp a row, on the CUDA cores.
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
  const int kvh = h / (p.num_heads / p.num_kv_heads);
  RowWalk<BF16> w(p.q + (long long)t * p.q_tok + (long long)h * p.head_dim * 2, p.head_dim, lane);
  if (p.prefix.indptr != nullptr) {
    const int g = p.group_indptr != nullptr ? last_not_above(p.group_indptr, p.num_groups + 1, b) : 0;
    if (g >= 0 && g < p.num_groups)
      w.walk(p, p.prefix, p.prefix.indptr[g], kvh, 0, list_keys(p.prefix, g, p.block_size), lane);
  }
  const int len = list_keys(p.own, b, p.block_size);
  w.walk(p, p.own, p.own.indptr[b], kvh, 0, p.causal ? min(len, len - n_new + i + 1) : len, lane);
  w.store(p.out + (long long)t * p.o_tok + (long long)h * p.head_dim * 2, p.head_dim, lane);
  if (p.lse != nullptr && lane == 0) p.lse[row] = w.lse2() * kLn2;
}

// ---------------------------------------------------------------- shared pieces of the matrix kernels
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

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void prefetch_tensormap(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void tma_load4(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// Weights of the matrix kernels are 2^(s - m) with m at least kBelow under the largest score so far;
// m moves when a score passes it by more than kReach.  bf16 has the exponents of fp32: m may lag 8
// behind.  fp16 has 2^15 for its largest power and 2^-25 for half its smallest step, so it takes weights
// between 2^9 and 2^15: what a weight loses is 2^-34 of the largest, a million keys together 2^-14 of it
// (weights of at most one would lose 2^-25 each, and sums over many keys count on them).  Lags of
// 8, 6 and 4 (what is left of 15) take 101, 103 and 111 us for 32 requests of 1 ... 64 new tokens behind 4096
// keys, 100 before the weights were raised: each move rescales O.
template <bool BF16>
struct WeightRange {
  static constexpr float kBelow = BF16 ? 0.f : 9.f, kReach = BF16 ? 8.f : 15.f;
};

// A part of a row's softmax that another launch joins: out / l and lse in base 2.
struct Partials {
  float* lse;  // [slots][num_heads]
  float* out;  // [slots][num_heads][head_dim]
};

// ---------------------------------------------------------------- one token a request
// Bound by HBM: every K / V row is read once for the G = num_heads / num_kv_heads rows that share
// it.  The pages of all requests form one axis (kv_indptr's own), cut into 16-key units, with one
// unit more a request for what its end costs; CTA x of a head block takes the x-th equal run of
// units, whatever requests it meets, so the load is even for any mix of lengths and nothing is
// planned on the host.  A request inside one run is
// finished there; one cut by a border leaves a partial in each run (slot 2x if it began in an
// earlier run, else 2x + 1) for the join kernel.
//
// Inside a CTA a warp works alone: head hs = w % HB of the block, the ks-th of KS = 8 / HB equal parts
// of the run, its own ring of stages filled by TMA (a box a page, 128-byte swizzled) or, for many
// bytes and for page sizes a 16-key box does not fit, by cp.async rows; no barrier in the loop.  Both
// products are taken transposed, S^T = K Q^T and O^T += V^T P^T (m16n8k16), so that the 16-wide
// side is full of keys or head elements and the 8-wide side holds the G rows: half the products and
// registers of the other way round for G <= 8.  S^T turns into the second product's operand with
// movmatrix.  Measured (HBM copy rate 6.55 TB/s): 256 requests of up to 4000 keys, 8 key heads of 128,
// 2.1 GB in 308 to 314 us one call behind the other, 310 to 328 among other work; 512 requests of up to 1500 keys on one
// key head, 225 MB in 50 us, 4.5 TB/s: the first tiles are there after 4 to 5 us, the SMs' shares of the bandwidth differ by 15 %, and the
// slowest of the equal runs decides.  What the borders between the KS parts cut is joined through shared
// memory at the end (one barrier a CTA; a barrier a request, with the tiles dealt out in turn, cost 2 to 4 us each).
constexpr int kDecodeWarps = 8;
constexpr int kTile = 16;  // keys

struct DecodeParams {
  CUtensorMap kmap, vmap;
  AttentionParams a;
  Partials part;
  int n_ranges;        // equal runs of the page axis
  int hb_shift;        // log2 of the heads a CTA works on
  int units_per_page;  // 16-key units of a page
  int box;             // keys of a TMA box
  long long slot0;     // first slot of the runs
  bool join_all;       // whole requests too go to a slot (behind the runs' own): the prefix is joined
};

// Programmatic launches.  A kernel normally waits for the one before it (and lets the one behind it
// get ready).  Of the two kernels of a shared prefix and of the own keys, the second needs nothing
// that the first writes, only what that one has itself waited for before it let this one start: it
// runs beside it, on the SMs that are free, and waits behind its work instead, so that what follows
// (the join) still finds both done.
__device__ __forceinline__ void wait_before(bool beside) {
  if (!beside) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_behind(bool beside) {
  if (beside) asm volatile("griddepcontrol.wait;" ::: "memory");
}

struct __align__(16) TileMeta {
  int request;  // -1: behind the last tile
  int keys;     // keys of the tile that exist
  int flags;    // 1: first tile of the request in this warp, 2: last, kHead / kTail, kBefore / kBehind
  int slot;     // where the result goes: -1 = the output row (a slot is num_heads rows)
};
enum {
  kHead = 4,    // began in an earlier part of the run (or before it): joined at the end
  kTail = 8,    // began here and goes on in a later part
  kBefore = 16, // began before the CTA's run
  kBehind = 32  // goes on behind the CTA's run
};
struct Piece {  // what a warp leaves for the join: its head and its tail
  int request, flags;
};

template <int D, int NST>
struct DecodeSmem {
  static constexpr int kHalf = kTile * 128;             // 16 keys x 64 elements
  static constexpr int kPlane = D / 64 * kHalf;
  static constexpr int kStage = 2 * kPlane;
  static constexpr int kRing = kDecodeWarps * NST * kStage;
  static constexpr int kMeta = kDecodeWarps * (NST * (int)(sizeof(TileMeta) + sizeof(uint64_t)) + 2 * (int)sizeof(Piece));
  static int bytes(int G, int hb) {
    const int join = hb < kDecodeWarps ? kDecodeWarps * G * (D + 4) * 4 : 0;
    return 1024 + kRing + kMeta + join;
  }
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <bool BF16, int D, int NT, int NST, bool TMA>
__global__ void __launch_bounds__(kDecodeWarps * 32, 1) attention_decode_kernel(const __grid_constant__ DecodeParams p) {
  using S = DecodeSmem<D, NST>;
  extern __shared__ __align__(1024) char smem_raw[];
  constexpr int kSteps = D / 16, kRowBytes = D * 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int HB = 1 << p.hb_shift, KS = kDecodeWarps >> p.hb_shift;
  const int hs = warp & (HB - 1), ks = warp >> p.hb_shift;
  const int kvh = blockIdx.y * HB + hs;
  const AttentionParams& a = p.a;
  const int G = a.num_heads / a.num_kv_heads;
  const unsigned UPP = p.units_per_page, BS = a.block_size;
  char* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t ring = smem_u32(smem) + warp * NST * S::kStage;
  TileMeta* const meta = reinterpret_cast<TileMeta*>(smem + S::kRing) + warp * NST;
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + S::kRing + kDecodeWarps * NST * sizeof(TileMeta)) + warp * NST;
  Piece* const pieces = reinterpret_cast<Piece*>(smem + S::kRing + kDecodeWarps * NST * (sizeof(TileMeta) + sizeof(uint64_t)));
  // [warp][G][D] heads, then [warp][G] their maxima and sums; a tail takes the warp's own ring
  float* const heads = reinterpret_cast<float*>(smem + S::kRing + S::kMeta);

  if (TMA && threadIdx.x < 2) prefetch_tensormap(threadIdx.x == 0 ? &p.kmap : &p.vmap);
  if (TMA && lane < NST) mbar_init(&full[lane], 1);  // the warp's own
  if (lane < 2) pieces[warp * 2 + lane] = Piece{-1, 0};
  if (TMA) mbar_fence_init();
  __syncwarp();
  wait_before(false);
  if (kvh >= a.num_kv_heads) return;  // all KS warps of such a head slot leave together

  // This CTA's run of units, [u_begin, u_end) of the page axis, this warp's part of it, and the
  // request of its first unit: the last b with indptr[b] <= its page, 32 probes a round.
  const int* const indptr = a.own.indptr;
  const int B = a.num_requests;
  unsigned u_begin, u_end, w_begin, w_end;
  int axis0, b0;
  auto place = [&](int first, int b) { return (unsigned)(first - axis0) * UPP + (unsigned)b; };  // of request b on the axis
  {
    int lo = 0, n = B, step = (n + 31) / 32;  // the answer is in [lo, lo + n)
    int probe = lane * step < n ? indptr[lane * step] : 0;
    axis0 = indptr[0];
    const unsigned units = place(max(indptr[B], axis0), B);
    const unsigned chunk = (units + p.n_ranges - 1) / p.n_ranges;
    u_begin = chunk * blockIdx.x;
    u_end = min(u_begin + chunk, units);
    if (u_begin >= u_end) return;
    const unsigned part = (u_end - u_begin + KS - 1) / KS;
    w_begin = min(u_begin + part * ks, u_end);
    w_end = min(w_begin + part, u_end);
    while (n > 1) {
      const bool below = lane * step < n && place(probe, lo + lane * step) <= w_begin;
      const int last = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
      n = min(step, n - last * step);
      lo += last * step;
      step = (n + 31) / 32;
      probe = lane * step < n ? indptr[lo + lane * step] : 0;
    }
    b0 = lo;
  }

  // Producer: walks the requests of the run, 32 of them loaded at a time (one a lane).
  int batch = b0, in_batch = -1;  // in_batch: index of the current request, -1 before the first
  int my_first = 0, my_end = 0, my_last = 0;
  auto load_batch = [&]() {
    const int b = batch + lane;
    my_first = my_end = my_last = 0;
    if (b < B) {
      my_first = indptr[b];
      my_end = indptr[b + 1];
      my_last = min(max(a.own.last[b], 0), (int)BS);
    }
  };
  load_batch();
  int key = 0, key_end = 0, first_page = 0;  // of the current request: next tile of this warp, end
  int request = -1, slot = -1, cut = 0;
  bool fresh = false, done = w_begin >= w_end;  // fresh: no tile of the request issued yet

  auto key_of = [&](unsigned unit) { return (int)(unit / UPP * BS + unit % UPP * kTile); };
  auto next_request = [&]() {
    for (;;) {
      if (++in_batch == 32) {
        batch += 32;
        in_batch = 0;
        if (batch < B) load_batch();
      }
      const int first = __shfl_sync(0xffffffffu, my_first, in_batch);
      const int end = __shfl_sync(0xffffffffu, my_end, in_batch);
      const int last = __shfl_sync(0xffffffffu, my_last, in_batch);
      request = batch + in_batch;
      const unsigned s0 = place(first, request), s1 = s0 + (unsigned)(end - first) * UPP;  // its units
      if (request >= B || s0 >= w_end) { done = true; return; }
      if (end <= first || s1 <= w_begin) continue;
      const int len = (end - first - 1) * (int)BS + last;
      key = s0 < w_begin ? min(key_of(w_begin - s0), len) : 0;
      key_end = s1 > w_end ? min(key_of(w_end - s0), len) : len;
      first_page = first;
      cut = 0;
      slot = p.join_all ? (int)p.slot0 + 2 * p.n_ranges + request : -1;
      if (s0 < w_begin || s1 > w_end) {
        if (KS > 1) cut = (s0 < w_begin ? kHead : kTail) | (s0 < u_begin ? kBefore : 0) | (s1 > u_end ? kBehind : 0);
        else slot = (int)p.slot0 + 2 * (int)blockIdx.x + (s0 < u_begin ? 0 : 1);
      }
      fresh = true;
      return;
    }
  };

  // The next tile's description; its page numbers are on their way one tile before they are used.
  int row_page = -1, row_entry = 0;  // lane r < 16: page and entry of row r as the table has it, -1 = no row
  int row_at = -1;                   // its place in the table
  TileMeta next = {-1, 0, 0, 0};
  auto fetch = [&]() {
    next.request = -1;
    if (!done && (request < 0 || (!fresh && key >= key_end))) next_request();
    if (done) return;
    next.request = request;
    next.keys = max(0, min(kTile, key_end - key));
    next.slot = slot;
    next.flags = (fresh ? 1 : 0) | (key + kTile >= key_end ? 2 | cut : 0);
    fresh = false;
    row_at = row_page = -1;
    if (lane < next.keys) {
      const unsigned pg = (unsigned)(key + lane) / BS;
      row_entry = key + lane - (int)(pg * BS);
      const long long at = (long long)first_page + pg;
      if (at >= 0 && at < a.own.num_indices) {
        row_at = (int)at;
        row_page = a.own.indices[at];
      }
    }
    key += kTile;
  };
  // Q of a request, fetched when its first tile is issued, if the last one fetched is in use already
  uint32_t q_next[kSteps][NT][2];
  int q_next_at = -1;  // the tile (in order) it belongs to
  const int r0 = (lane & 3) * 2, e0 = lane >> 2;
  auto load_q = [&](uint32_t (*dst)[NT][2], int b) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool row = n * 8 + e0 < G;
      const char* src = a.q + (long long)b * a.q_tok + (long long)(kvh * G + n * 8 + e0) * kRowBytes + r0 * 2;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        dst[k][n][0] = row ? *reinterpret_cast<const uint32_t*>(src + k * 32) : 0u;
        dst[k][n][1] = row ? *reinterpret_cast<const uint32_t*>(src + k * 32 + 16) : 0u;
      }
    }
  };
  auto issue = [&](int stage) {  // starts the copies of the tile described by `next`
    if (lane == 0) meta[stage] = next;
    const uint32_t base = ring + stage * S::kStage;
    if (row_at >= 0 && (unsigned)row_page >= (unsigned)a.num_blocks) {
      if (a.checks) report(a.err, kErrBadPage, kWhereAttention, row_at, row_page);
      row_page = -1;  // zeros
    }
    if (TMA) {
      if (next.request >= 0) {
        const bool any = next.keys > 0;
        if (lane == 0) {
          if (any) mbar_expect_tx(&full[stage], S::kStage);
          else mbar_arrive(&full[stage]);
        }
        __syncwarp();
        constexpr int kBoxes = 2 * (D / 64);  // of one page: K and V, 64 elements each
        const int piece = lane / kBoxes, plane = lane / (D / 64) & 1, half = lane % (D / 64);
        const int src = piece * p.box;
        const int page = __shfl_sync(0xffffffffu, row_page, src & 15);
        const int entry = __shfl_sync(0xffffffffu, row_entry, src & 15);
        if (any && src < kTile)
          tma_load4(base + plane * S::kPlane + half * S::kHalf + src * 128, plane ? &p.vmap : &p.kmap, &full[stage],
                    half * 64, page < 0 ? 0 : entry, kvh, page);
      }
    } else {
      if (next.request >= 0) {
        long long off = -1;
        if (row_page >= 0)
          off = (long long)row_page * a.block_stride + (long long)row_entry * a.slot_stride + (long long)kvh * kRowBytes;
        constexpr int kChunks = D / 8, kRowsAtOnce = 32 / kChunks;
        const int c = lane % kChunks;
#pragma unroll
        for (int i = 0; i < kTile / kRowsAtOnce; ++i) {
          const int row = i * kRowsAtOnce + lane / kChunks;
          const long long o = __shfl_sync(0xffffffffu, off, row);
          const uint32_t dst = base + (c >> 3) * S::kHalf + row * 128 + (((c & 7) ^ (row & 7)) << 4);
          const bool ok = o >= 0;
          cp_async16(dst, ok ? a.kcache + o + c * 16 : a.kcache, ok);
          cp_async16(dst + S::kPlane, ok ? a.vcache + o + c * 16 : a.vcache, ok);
        }
      }
      cp_async_commit();
    }
  };

  int issued = 0;  // tiles
  auto advance = [&]() {
    issue(issued % NST);
    if (next.request >= 0) {
      if ((next.flags & 1) && q_next_at < 0) {
        load_q(q_next, next.request);
        q_next_at = issued;
      }
      ++issued;
      fetch();
    } else {
      ++issued;
    }
  };
  fetch();
#pragma unroll 1
  for (int s = 0; s < NST - 1; ++s) advance();

  // Consumer.  A lane holds, of S^T, keys lane / 4 and lane / 4 + 8 of rows 2 (lane % 4) and the next;
  // of O^T, elements 16 m + lane / 4 and + 8 of the same rows.
  uint32_t q[kSteps][NT][2];
  float o[kSteps][NT][4], m[NT][2], l[NT][2];
  const float scale2 = a.scale * kLog2e;
  // ldmatrix addresses inside a plane: row, then the lane's chunk of step 0; step k flips bits 5, 6
  const uint32_t k_addr = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_addr = ((lane & 7) + ((lane >> 4) << 3)) * 128 + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
  bool dead = false;
  int it = 0;
  for (;; ++it) {
    const int stage = it % NST;
    if (!TMA) cp_async_wait<NST - 2>();
    __syncwarp();
    const TileMeta t = meta[stage];
    if (t.request < 0) break;
    advance();
    if (TMA && !dead && !mbar_wait_bounded(&full[stage], (it / NST) & 1)) {
      report(a.err, kErrWaitTimeout, kWhereAttention, blockIdx.x, it);
      dead = true;  // goes on without waiting: the head's other warps meet it at the join's barrier
    }

    if (t.flags & 1) {
      if (q_next_at == it) {
        q_next_at = -1;
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            q[k][n][0] = q_next[k][n][0];
            q[k][n][1] = q_next[k][n][1];
          }
      } else {
        load_q(q, t.request);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) o[k][n][0] = o[k][n][1] = o[k][n][2] = o[k][n][3] = 0.f;
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
      }
    }

    if (t.keys > 0) {
      const uint32_t kbase = ring + stage * S::kStage, vbase = kbase + S::kPlane;
      if (t.keys < kTile && TMA) {
        // what lies behind the last key may be anything, and 0 * NaN is not 0
#pragma unroll
        for (int c = lane; c < kTile * D / 8; c += 32) {
          const int row = c / (D / 8), half = (c % (D / 8)) >> 3;
          if (row >= t.keys)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vbase + half * S::kHalf + row * 128 + (c & 7) * 16), "r"(0) : "memory");
        }
        fence_proxy_async();  // before the stage is filled again
        __syncwarp();
      }
      float s[NT][4] = {};
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        uint32_t x[4];
        ldsm4(x, kbase + (k >> 2) * S::kHalf + (k_addr ^ ((k & 3) << 5)));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<BF16>(s[n], x, q[k][n][0], q[k][n][1]);
      }
      uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] *= scale2;
        if (t.keys < kTile) {
          if (e0 >= t.keys) s[n][0] = s[n][1] = -INFINITY;
          if (e0 + 8 >= t.keys) s[n][2] = s[n][3] = -INFINITY;
        }
        float keep[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = fmaxf(s[n][i], s[n][2 + i]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          keep[i] = 1.f;
          if (top > m[n][i] + WeightRange<BF16>::kReach) {
            const float base = top - WeightRange<BF16>::kBelow;
            keep[i] = exp2_fast(m[n][i] - base);
            m[n][i] = base;
          }
        }
        if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            o[k][n][0] *= keep[0];
            o[k][n][1] *= keep[1];
            o[k][n][2] *= keep[0];
            o[k][n][3] *= keep[1];
          }
          l[n][0] *= keep[0];
          l[n][1] *= keep[1];
        }
        // The weights enter the second product in the element type, as a part and the rounded rest: two
        // products, error 2^-15 (bf16; fp16 2^-21, and 2^-34 of the largest) instead of 2^-8, on pipes that
        // HBM leaves idle.  The part is taken towards zero from a little less than the weight, so that
        // the rest is positive: both products of an infinity in V have its sign, and neither is 0 * infinity.
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float w0 = exp2_fast(s[n][2 * i] - (m[n][0] == -INFINITY ? 0.f : m[n][0]));
          const float w1 = exp2_fast(s[n][2 * i + 1] - (m[n][1] == -INFINITY ? 0.f : m[n][1]));
          l[n][0] += w0;
          l[n][1] += w1;
          const uint32_t h = down2_rz<BF16>(w0 * (1.f - 0x1p-12f), w1 * (1.f - 0x1p-12f));
          const float2 f = up2<BF16>(h);
          hi[n][i] = transpose8x8(h);
          lo[n][i] = transpose8x8(down2<BF16>(w0 - f.x, w1 - f.y));
        }
      }
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        uint32_t x[4];
        ldsm4_t(x, vbase + (k >> 2) * S::kHalf + (v_addr ^ ((k & 3) << 5)));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816<BF16>(o[k][n], x, hi[n][0], hi[n][1]);
          mma16816<BF16>(o[k][n], x, lo[n][0], lo[n][1]);
        }
      }
    }

    if (t.flags & 2) {
      const int head0 = kvh * G;
      char* const out = a.out + (long long)t.request * a.o_tok + (long long)head0 * kRowBytes;
      float* const lse = t.slot >= 0 ? p.part.lse + (long long)t.slot * a.num_heads + head0
                         : a.lse != nullptr ? a.lse + (long long)t.request * a.num_heads + head0 : nullptr;
      float* const po = p.part.out + ((long long)max(t.slot, 0) * a.num_heads + head0) * D;
      const float unit = t.slot >= 0 ? 1.f : kLn2;  // partials keep base 2
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 4);
          l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 8);
          l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 16);
        }
      if ((t.flags & (kHead | kTail)) == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float inv[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = n * 8 + r0 + i;
            inv[i] = l[n][i] > 0.f ? 1.f / l[n][i] : (l[n][i] == 0.f ? 0.f : l[n][i]);
            if (lse != nullptr && e0 == 0 && r < G) lse[r] = l[n][i] == 0.f ? -INFINITY : (m[n][i] + log2f(l[n][i])) * unit;
          }
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float x = o[k][n][2 * h] * inv[0], y = o[k][n][2 * h + 1] * inv[1];
              const int d = 16 * k + 8 * h;
              if (t.slot >= 0) {
                const int r = n * 8 + r0;
                if (r < G) po[r * D + d + e0] = x;
                if (r + 1 < G) po[(r + 1) * D + d + e0] = y;
              } else {
                const uint32_t v = transpose8x8(down2<BF16>(x, y));  // row lane / 4, two elements
                if (n * 8 + e0 < G) *reinterpret_cast<uint32_t*>(out + (n * 8 + e0) * kRowBytes + (d + r0) * 2) = v;
              }
            }
        }
      } else {
        // left for the join: a tail is the warp's last piece, its ring holds nothing any more
        const int tail = t.flags & kTail ? 1 : 0;
        float* const dst = tail ? reinterpret_cast<float*>(smem + warp * NST * S::kStage) : heads + warp * G * D;
        float* const stat = heads + kDecodeWarps * G * D + (warp * 2 + tail) * 2 * G;
        __syncwarp();
        if (lane == 0) pieces[warp * 2 + tail] = Piece{t.request, t.flags};
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = n * 8 + r0 + i;
            if (r >= G) continue;
            if (e0 == 0) {
              stat[r] = m[n][i];
              stat[G + r] = l[n][i];
            }
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
              dst[r * D + 16 * k + e0] = o[k][n][i];
              dst[r * D + 16 * k + 8 + e0] = o[k][n][2 + i];
            }
          }
      }
    }
  }
  if (KS > 1) {
    // Join what the borders between this head's warps cut: pieces in order, a chain is a run of
    // pieces of one request.  Every wait above was on a copy that is done, so the rings are free.
    asm volatile("bar.sync %0, %1;" ::"r"(1 + hs), "r"(KS * 32) : "memory");
    const int head0 = kvh * G;
    // lane i < 2 KS: the i-th piece; a chain starts where a piece's request is not the last one's
    const Piece mine = lane < 2 * KS ? pieces[(hs + (lane >> 1) * HB) * 2 + (lane & 1)] : Piece{-1, 0};
    const unsigned valid = __ballot_sync(0xffffffffu, mine.request >= 0);
    const unsigned before = valid & ((1u << lane) - 1u);
    const int previous = __shfl_sync(0xffffffffu, mine.request, before != 0 ? 31 - __clz(before) : lane);
    unsigned starts = __ballot_sync(0xffffffffu, mine.request >= 0 && (before == 0 || previous != mine.request));
    while (starts != 0) {
      const int first = __ffs(starts) - 1;
      starts &= starts - 1;
      const unsigned chain = valid & (starts != 0 ? (1u << (__ffs(starts) - 1)) - 1u : 0xffffffffu) & ~((1u << first) - 1u);
      const bool in_chain = chain >> lane & 1;
      const int which = __shfl_sync(0xffffffffu, mine.request, first);
      const bool from_before = __any_sync(0xffffffffu, in_chain && (mine.flags & kBefore));
      const bool goes_on = __any_sync(0xffffffffu, in_chain && (mine.flags & kBehind));
      const int slot = from_before  ? (int)p.slot0 + 2 * (int)blockIdx.x
                       : goes_on    ? (int)p.slot0 + 2 * (int)blockIdx.x + 1
                       : p.join_all ? (int)p.slot0 + 2 * p.n_ranges + which
                                    : -1;
      char* const out = a.out + (long long)which * a.o_tok + (long long)head0 * kRowBytes;
      float* const lse = slot >= 0 ? p.part.lse + (long long)slot * a.num_heads + head0
                         : a.lse != nullptr ? a.lse + (long long)which * a.num_heads + head0 : nullptr;
      float* const po = p.part.out + ((long long)max(slot, 0) * a.num_heads + head0) * D;
      for (int e = ks * 32 + lane; e < G * (D / 4); e += KS * 32) {
        const int r = e / (D / 4), d = (e - r * (D / 4)) * 4;
        float mm = -INFINITY, ll = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (unsigned left = chain; left != 0; left &= left - 1) {
          const int i = __ffs(left) - 1, w = hs + (i >> 1) * HB;
          const float* stat = heads + kDecodeWarps * G * D + (w * 2 + (i & 1)) * 2 * G;
          const float* src = i & 1 ? reinterpret_cast<const float*>(smem + w * NST * S::kStage) : heads + w * G * D;
          const float4 v = *reinterpret_cast<const float4*>(src + r * D + d);
          const float pm = stat[r], pl = stat[G + r];
          // A piece without a key has the sum 0.  Its maximum says less: NaN scores do not move it, and
          // their sum, NaN, has to reach the row.
          if (pl == 0.f) continue;
          const float top = fmaxf(mm, pm), keep = exp2_fast(mm - top), f = exp2_fast(pm - top);
          mm = top;
          ll = fmaf(ll, keep, f * pl);
          acc.x = fmaf(acc.x, keep, f * v.x);
          acc.y = fmaf(acc.y, keep, f * v.y);
          acc.z = fmaf(acc.z, keep, f * v.z);
          acc.w = fmaf(acc.w, keep, f * v.w);
        }
        const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);
        if (slot >= 0)
          *reinterpret_cast<float4*>(po + r * D + d) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        else
          *reinterpret_cast<uint2*>(out + r * kRowBytes + d * 2) = make_uint2(down2<BF16>(acc.x * inv, acc.y * inv), down2<BF16>(acc.z * inv, acc.w * inv));
        if (d == 0 && lse != nullptr) lse[r] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * (slot >= 0 ? 1.f : kLn2);
      }
      __syncwarp();
    }
  }
  if (!TMA) cp_async_wait<0>();
  // Every tile issued was also waited for, unless a wait ran out: then once more, so that no copy
  // is in flight when the CTA leaves.
  if (TMA && dead)
    for (int i = max(0, it - NST); i < it; ++i) mbar_wait_bounded(&full[i % NST], (i / NST) & 1);
}

// ---------------------------------------------------------------- tiles of rows
// Many rows share their keys: the tokens of one request (or of all requests of a prefix group)
// times the G heads of a key head.  Two row tiles of 128 (row = token * G + head) and one stream
// of 128-key tiles per CTA; S = Q K^T and O += P V run on the tensor cores (tcgen05, M = 128) with
// S, P and O in tensor memory.
//
//   warps 0-3, 4-7   softmax of row tile 0 / 1, one thread a row: S from tensor memory, running
//                    maximum and sum, P = 2^(S - m) in the element type over S's own columns
//   warp 8, 9        K / V tiles into two-or-more-stage rings
//   warp 11          describes the pieces of work (persistent CTAs, a two-deep ring), so that the look-up
//                    of the next one, and its first K and V tiles, run beside the end of the last
//   warp 10          issues the MMAs: PV of a tile, then the next QK of the same row tile, so that
//                    one row tile's softmax runs beside the other's products
//
// Measured: four prompts of 1000 to 3000 tokens, 28 query on 4 key heads of 128, causal, 226 GFLOP in 240 to
// 248 us (0.91 to 0.94 PFLOP/s of 1.66 measured for a large product).  A pair of 128-key tiles takes 3000 cycles where its four products
// take 2048: the softmax of a row tile (2100) and its products (900 behind its last P) follow one another,
// and two row tiles, all that tensor memory holds, overlap them to two thirds.  The tensor pipe is active
// for 42 % of the active cycles in the 16-tile pieces of a prefix (start, Q, first S and O's way out).
//
// The maximum is only moved (and O rescaled in tensor memory, by the softmax threads) when it
// grows by more than 8 in base 2 (6 in fp16, see WeightRange): fp32 sums and 16-bit P hold the factor.
// S of the next tile overwrites P: it is issued behind the PV that reads it, and the commit behind
// it tells the softmax warps that this PV, too, is complete.  P is rounded to the element type
// (half a step: 2^-8 in bf16; in fp16 2^-11, and 2^-34 of the largest for small weights): the rest, as a
// second operand, would double the products of PV, which bound this kernel.  l sums the weights before
// they are rounded.
//
// Pages of 8 to 128 keys (powers of two) and of multiples of 128 are loaded by TMA, one box a page
// and 64-element half row, 128-byte swizzled; a tile that reaches past the last key, and other page
// sizes, by cp.async rows with zeros behind the last key (what lies there may be anything, and 0 * NaN
// is not 0).
constexpr int kRows = 128;       // rows of a tile
constexpr int kKeys = 128;       // keys of a tile
constexpr int kTileThreads = 384;

struct TileParams {
  CUtensorMap kmap, vmap;
  AttentionParams a;
  PageList list;      // pages of each sequence (a request's own, or a group's prefix)
  Partials part;
  int shared;         // 1: sequences are prefix groups, 0: requests
  int n_seq, n_slots, n_splits;
  int slot0;          // first of n_splits sets of partials ([num_tokens] slots each), -1: final
  int causal;
  int box;            // keys of a TMA box, 0 = no TMA
  bool beside;        // see wait_before
};

template <int D>
struct TileSmem {
  static constexpr int kStages = D == 64 ? 4 : 2;
  static constexpr int kStage = kKeys * D * 2;
  static constexpr int kV = 0, kK = kStages * kStage, kQ = 2 * kStages * kStage;
  static constexpr int kBytes = kQ + 2 * kRows * D * 2;
};

struct TileBars {
  uint64_t kfull[4], kempty[4], vfull[4], vempty[4];
  uint64_t wfull[2], wempty[2], qfull[2], sfull[2], pfull[2][2], ofull[2], vraw, want, grant, done;
  uint32_t tmem;
  int cleaned[4];  // of the it-th piece, at it % 4: 1 + the first tile of V that lost an element to clean_tile, or 0
};

// Two row tiles of one key head against a run of key tiles.
struct TileWork {
  int t_begin, n_new;     // tokens of the sequence
  int row0, rows;         // rows of the pair, counted in the sequence; rows == 0: no more work
  int len, first_page;    // keys of the sequence, place of its first page in the list
  int tile0, n_kv;        // key tiles
  int kvh, split;

  // The first key that a row of the pair does not read although another may: causal rows read up to
  // their own token, and the first row's is the earliest.
  __device__ __forceinline__ int first_hidden(bool causal, int G) const {
    return causal ? min(len, max(0, len - n_new + row0 / G + 1)) : len;
  }
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 consecutive columns of the thread's own tensor memory lane.
__device__ __forceinline__ void tc_ld32(uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
// Two fp32 lanes in one instruction.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void tc_ld16(uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Shared memory operand of an MMA: rows (or K groups) of 128 bytes, 128-byte swizzle, 8-row groups
// 1024 bytes apart.  The low word holds the address and, for an operand whose rows run along K, the
// distance of its 64-element chunks (lbo); a step along K adds to the low word alone.
__device__ __forceinline__ uint32_t umma_low(uint32_t addr, uint32_t lbo) { return ((addr & 0x3ffffu) >> 4) | ((lbo >> 4) << 16); }
constexpr uint32_t kUmmaHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
// kind::f16, fp32 accumulators: element type (0 fp16, 1 bf16), M = 128, N, B along K or along N.
__device__ __forceinline__ constexpr uint32_t umma_idesc(bool bf16, int n, bool b_along_n) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_along_n ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// One thread of the warp, the same each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
template <uint32_t IDESC>
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.u32 p, %3, 0;\n\tmov.b64 x, {%1, %4};\n\tmov.b64 y, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(add), "n"(kUmmaHigh), "n"(IDESC)
      : "memory");
}
template <uint32_t IDESC>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.u32 p, %3, 0;\n\tmov.b64 y, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %5, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(add), "n"(kUmmaHigh), "n"(IDESC)
      : "memory");
}

// First token of sequence i (i <= n_seq).
__device__ __forceinline__ int token_of(const TileParams& p, int i) {
  if (p.shared) i = p.a.group_indptr != nullptr ? min(max(p.a.group_indptr[i], 0), p.a.num_requests)
                                                : (i > 0 ? p.a.num_requests : 0);
  return p.a.qo_indptr != nullptr ? p.a.qo_indptr[i] : i;
}

// Loads 128 keys of one plane into a stage.  One warp.
template <int D>
__device__ __forceinline__ void load_tile(const TileParams& p, const CUtensorMap* map, const char* cache, int kvh,
                                          int first_page, int len, int tile, uint32_t dst, uint64_t* full, int lane) {
  const AttentionParams& a = p.a;
  constexpr int kHalves = D / 64, kHalf = kKeys * 128;
  const int key0 = tile * kKeys;
  if (p.box > 0 && key0 + kKeys <= len) {
    if (lane == 0) mbar_expect_tx(full, kKeys * D * 2);
    __syncwarp();
    const int pieces = kKeys / p.box * kHalves;
    if (lane < pieces) {
      const int piece = lane / kHalves, half = lane - piece * kHalves;
      const int key = key0 + piece * p.box;
      const int pg = key / a.block_size;
      const long long at = (long long)first_page + pg;
      int page = -1;  // outside the map: the box is filled with zeros
      if (at >= 0 && at < p.list.num_indices) {
        page = p.list.indices[at];
        if (page < 0 || page >= a.num_blocks) {
          if (a.checks) report(a.err, kErrBadPage, kWhereAttention, at, page);
          page = -1;
        }
      }
      tma_load4(dst + half * kHalf + piece * p.box * 128, map, full, half * 64, key - pg * a.block_size, kvh, page);
    }
    return;
  }
  const char* head = cache + (long long)kvh * D * 2;
  constexpr int kChunks = D / 8, kRowsAtOnce = 32 / kChunks;
#pragma unroll 1
  for (int base = 0; base < kKeys; base += 32) {
    long long off = -1;
    const int key = key0 + base + lane;
    if (key < len) off = key_offset(a, p.list, first_page, key);
#pragma unroll 4
    for (int i = 0; i < 32 / kRowsAtOnce; ++i) {
      const int src = i * kRowsAtOnce + lane / kChunks, row = base + src, c = lane % kChunks;
      const long long o = __shfl_sync(0xffffffffu, off, src);
      cp_async16(dst + (c >> 3) * kHalf + row * 128 + (((c & 7) ^ (row & 7)) << 4), o >= 0 ? head + o + c * 16 : cache, o >= 0);
    }
  }
  cp_async_commit();
  cp_async_wait<0>();
  fence_proxy_async();  // generic-proxy writes, read by the tensor cores
  __syncwarp();
  if (lane == 0) mbar_arrive(full);
}

// Sets what is infinite or NaN in a stage of V to 0; true if there was anything.  One warp.
template <bool BF16, int D>
__device__ __forceinline__ bool clean_tile(uint32_t tile, int lane) {
  // an exponent of ones carries into bit 15 of its half word
  constexpr uint32_t kExp = BF16 ? 0x7f807f80u : 0x7c007c00u, kOne = BF16 ? 0x00800080u : 0x04000400u;
  constexpr int kBatch = 4;
  auto load = [&](int c, uint32_t* v) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(tile + c * 16) : "memory");
  };
  uint32_t found = 0;
#pragma unroll 1
  for (int c = lane; c < kKeys * D / 8; c += 32 * kBatch) {
    uint32_t v[kBatch][4];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) load(c + 32 * i, v[i]);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) found |= (v[i][w] & kExp) + kOne;
  }
  if (!__any_sync(0xffffffffu, (found & 0x80008000u) != 0)) return false;
#pragma unroll 1
  for (int c = lane; c < kKeys * D / 8; c += 32) {
    uint32_t v[4];
    load(c, v);
#pragma unroll
    for (int w = 0; w < 4; ++w) v[w] &= ~(((((v[w] & kExp) + kOne) & 0x80008000u) >> 15) * 0xffffu);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tile + c * 16), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
  }
  return true;
}

template <bool BF16, int D>
__global__ void __launch_bounds__(kTileThreads, 1) attention_tile_kernel(const __grid_constant__ TileParams p) {
  using S = TileSmem<D>;
  constexpr int ST = S::kStages, kHalf = kKeys * 128;
  extern __shared__ __align__(1024) char smem_raw[];
  __shared__ TileBars bars;
  __shared__ TileWork work[2];
  __shared__ __align__(16) uint4 granted;  // the launch control's answer
  const AttentionParams& a = p.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // known to be uniform
  const int G = a.num_heads / a.num_kv_heads;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&bars.kfull[s], 1);
      mbar_init(&bars.kempty[s], 1);
      mbar_init(&bars.vfull[s], 1);
      mbar_init(&bars.vempty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.wfull[i], 1);
      mbar_init(&bars.wempty[i], 11);
      mbar_init(&bars.qfull[i], 4);
      mbar_init(&bars.sfull[i], 1);
      mbar_init(&bars.pfull[i][0], 4);
      mbar_init(&bars.pfull[i][1], 4);
      mbar_init(&bars.ofull[i], 1);
    }
    mbar_init(&bars.vraw, 1);
    mbar_init(&bars.want, 1);
    mbar_init(&bars.grant, 1);
    mbar_init(&bars.done, 1);
    mbar_fence_init();
  }
  if (p.box > 0 && warp == 9 && lane < 2) prefetch_tensormap(lane == 0 ? &p.kmap : &p.vmap);
  if (warp == 10) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bars.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  wait_before(p.beside);

  const uint32_t sm_q = smem + S::kQ, sm_k = smem + S::kK, sm_v = smem + S::kV;
  // The sign of the scale goes into Q; a scale of 0 must still leave masked scores at -infinity.
  const float scale2 = fmaxf(fabsf(a.scale) * kLog2e, 1.1754944e-38f);

  // A wait that runs out ends the role; the others run out in turn, and the CTA leaves in order.
  auto wait = [&](uint64_t* bar, unsigned parity) -> bool {
    const bool ok = mbar_wait_bounded(bar, parity);
    if (!ok) report(a.err, kErrWaitTimeout, kWhereAttention, blockIdx.x, bar - bars.kfull);
    return __all_sync(0xffffffffu, ok);  // a warp goes on or leaves as one
  };
  // The it-th piece of work, once the scheduler has described it; rows == 0 behind the last one.
  auto next_work = [&](int it) -> TileWork {
    TileWork k;
    k.rows = 0;
    if (wait(&bars.wfull[it & 1], (it >> 1) & 1)) k = work[it & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.wempty[it & 1]);
    return k;
  };

  // Registers move from the warpgroup of the copies and the MMAs to the two of the softmax, whose
  // threads hold a row of S: (2 * 216 + 72) * 128 = 384 * 168, what the block was launched with.
  // (Without it the row spills: 270 instead of 220 us for the four prompts.)
  if (warp < 8) {
    // ------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int i = warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);  // lane 32 * (warp % 4) in bits 16..
    const uint32_t t_s = lanes + i * 128, t_o = lanes + 256 + i * 128;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    const int r = threadIdx.x;  // row of the tile pair
    int tiles = 0, pieces = 0;  // S tiles and pieces of work seen by this row tile
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const TileWork k = next_work(it);
      if (k.rows == 0) break;
      const bool has_row = r < k.rows;
      const int tok = (k.row0 + r) / G, g = k.row0 + r - tok * G;
      const long long out_row = (long long)(k.t_begin + tok) * a.num_heads + k.kvh * G + g;  // [token][head]
      const long long part_row = ((long long)(p.slot0 + k.split) * a.num_tokens) * a.num_heads + out_row;
      if (k.n_kv == 0) {  // nothing to read: an empty part, or rows of zeros
        if (has_row) {
          if (p.slot0 >= 0) {
            p.part.lse[part_row] = -INFINITY;
          } else {
            char* o = a.out + (long long)(k.t_begin + tok) * a.o_tok + (long long)(k.kvh * G + g) * D * 2;
            for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(o + c * 16) = make_uint4(0, 0, 0, 0);
            if (a.lse != nullptr) a.lse[out_row] = -INFINITY;
          }
        }
        continue;
      }
      if (i * kRows >= k.rows) continue;  // one row tile only
      {
        // The warp's 32 rows of Q, whole lines an instruction, all of them on their way before the
        // first is stored; rows that do not exist are zeros.
        constexpr int kChunks = D / 8, kAtOnce = 32 / kChunks;
        const char* const mine = a.q + (long long)(k.t_begin + tok) * a.q_tok + (long long)(k.kvh * G + g) * D * 2;
        const int c = lane % kChunks;
        uint4 qv[32 / kAtOnce];
#pragma unroll
        for (int x = 0; x < 32 / kAtOnce; ++x) {
          const int row = x * kAtOnce + lane / kChunks;
          const char* src = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), row));
          qv[x] = make_uint4(0, 0, 0, 0);
          if ((r & ~31) + row < k.rows) qv[x] = *reinterpret_cast<const uint4*>(src + c * 16);
        }
        const uint32_t dst = sm_q + i * kRows * D * 2 + (c >> 3) * (kRows * 128) + (warp & 3) * 32 * 128;
#pragma unroll
        for (int x = 0; x < 32 / kAtOnce; ++x) {
          const int row = x * kAtOnce + lane / kChunks;
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + row * 128 + (((c & 7) ^ (row & 7)) << 4)),
                       "r"(qv[x].x ^ flip), "r"(qv[x].y ^ flip), "r"(qv[x].z ^ flip), "r"(qv[x].w ^ flip) : "memory");
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.qfull[i]);
      }
      const bool live = (r & ~31) < k.rows;  // the warp has a row
      const int limit = p.causal ? min(k.len, k.len - k.n_new + tok + 1) : k.len;  // keys below it are read
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < k.n_kv; ++j, ++tiles) {
        if (!(ok = wait(&bars.sfull[i], tiles & 1))) break;
        tc_fence_after();
        if (live) {
          float s[kKeys];
          uint32_t* raw = reinterpret_cast<uint32_t*>(s);
#pragma unroll
          for (int c = 0; c < kKeys; c += 32) tc_ld32(raw + c, t_s + c);
          tc_wait_ld();
          const int seen = limit - (k.tile0 + j) * kKeys;
          if (!__all_sync(0xffffffffu, seen >= kKeys)) {
#pragma unroll
            for (int c = 0; c < kKeys; ++c)
              if (c >= seen) s[c] = -INFINITY;
          }
          // P goes out in two parts, so that the products of the first (3/4) run beside the second's
          // exponentials, all of which take the special-function unit (a quarter of them as a polynomial
          // on the FMA pipe changed nothing).  The first 64 keys' exponentials start from the maximum as it was, beside
          // the search for the tile's own; only where that is too far above (the first tile, and few
          // others) are they done again from the new one, after O has been rescaled.
          uint32_t w[kKeys / 2];
          uint64_t sums[2];
          const uint64_t scale_2 = pack2(scale2, scale2);
          auto weights = [&](int from, int to) {  // of the pairs [from, to)
            const float base = m == -INFINITY ? 0.f : m;
            const uint64_t base_2 = pack2(-base, -base);
#pragma unroll
            for (int c = 0; c < kKeys / 2; ++c) {
              if (c < from || c >= to) continue;
              const float2 x = unpack2(fma2(pack2(s[2 * c], s[2 * c + 1]), scale_2, base_2));
              const float x0 = exp2_fast(x.x), x1 = exp2_fast(x.y);
              sums[c & 1] = c < 2 ? pack2(x0, x1) : add2(sums[c & 1], pack2(x0, x1));
              w[c] = down2<BF16>(x0, x1);
            }
          };
          auto publish = [&](int part) {
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.pfull[i][part]);
          };
          weights(0, 32);
          float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int c = 4; c + 8 <= kKeys; c += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) tops[e] = max3(tops[e], s[c + e], s[c + 4 + e]);
#pragma unroll
          for (int e = 0; e < 4; ++e) tops[e] = max3(tops[e], s[kKeys - 4 + e], tops[0]);
          float top = max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]);
          top = top == -INFINITY ? top : top * scale2;
          constexpr float kBelow = WeightRange<BF16>::kBelow, kReach = WeightRange<BF16>::kReach;
          if (__any_sync(0xffffffffu, !(top <= m + kReach))) {
            float keep = 1.f;
            if (!(top <= m + kReach)) {  // a NaN score, too, moves it: the row is NaN from here on
              keep = exp2_fast(m - (top - kBelow));
              m = top - kBelow;
            }
            l *= keep;
            if (j > 0) {
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
                tc_ld16(o, t_o + c);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tc_st16(t_o + c, o);
              }
            }
            weights(0, 32);
          }
          tc_st32(t_s, w);
          weights(32, 48);
          tc_st16(t_s + 32, w + 32);
          publish(0);
          weights(48, 64);
          tc_st16(t_s + 48, w + 48);
          publish(1);
          const float2 sum = unpack2(add2(sums[0], sums[1]));
          l += sum.x + sum.y;
        } else if (lane == 0) {
          mbar_arrive(&bars.pfull[i][0]);
          mbar_arrive(&bars.pfull[i][1]);
        }
      }
      if (ok) ok = wait(&bars.ofull[i], pieces & 1);
      ++pieces;
      if (ok && live) {
        tc_fence_after();
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays
        // O leaves through the shared memory of the warp's own Q rows, which nothing reads any more: a
        // thread has a row, a store instruction should have whole 128-byte lines.
        const unsigned have = __ballot_sync(0xffffffffu, has_row);
        const uint32_t stage = sm_q + i * kRows * D * 2 + (warp & 3) * 32 * 128;
        auto emit = [&](auto part) {
          constexpr bool PART = decltype(part)::value;
          constexpr int kCols = PART ? D / 2 : D;  // of one pass
          constexpr int kPassBytes = D * 2;        // of one row: what a row of Q took
          constexpr int kChunks = kPassBytes / 16, kAtOnce = 32 / kChunks;
          char* const mine = PART ? reinterpret_cast<char*>(p.part.out + part_row * D)
                                  : a.out + (long long)(k.t_begin + tok) * a.o_tok + (long long)(k.kvh * G + g) * D * 2;
#pragma unroll 1
          for (int pass = 0; pass < D / kCols; ++pass) {
            uint32_t o[kCols];
#pragma unroll
            for (int c = 0; c < kCols; c += 32) tc_ld32(o + c, t_o + pass * kCols + c);
            tc_wait_ld();
#pragma unroll
            for (int c = 0; c < kCols; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * inv);
            constexpr int kPer = PART ? 4 : 8;  // values of a 16-byte chunk
#pragma unroll
            for (int e = 0; e < kCols; e += kPer) {
              uint32_t v[4];
#pragma unroll
              for (int x = 0; x < 4; ++x)
                v[x] = PART ? o[e + x] : down2<BF16>(__uint_as_float(o[(e + 2 * x) % kCols]), __uint_as_float(o[(e + 2 * x + 1) % kCols]));
              const int chunk = e / kPer;
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + (chunk >> 3) * (kRows * 128) + lane * 128 + (((chunk & 7) ^ (lane & 7)) << 4)),
                           "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
            }
            __syncwarp();
            const int chunk = lane % kChunks;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint4 v[16 / kAtOnce];
#pragma unroll
              for (int x = 0; x < 16 / kAtOnce; ++x) {
                const int row = half * 16 + x * kAtOnce + lane / kChunks;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[x].x), "=r"(v[x].y), "=r"(v[x].z), "=r"(v[x].w)
                             : "r"(stage + (chunk >> 3) * (kRows * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) : "memory");
              }
#pragma unroll
              for (int x = 0; x < 16 / kAtOnce; ++x) {
                const int row = half * 16 + x * kAtOnce + lane / kChunks;
                char* const dst = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), row));
                if (have >> row & 1) *reinterpret_cast<uint4*>(dst + pass * kPassBytes + chunk * 16) = v[x];
              }
            }
            __syncwarp();
          }
        };
        if (p.slot0 >= 0) emit(std::true_type{});
        else emit(std::false_type{});
        if (has_row) {
          const float lse2 = l == 0.f ? -INFINITY : m + log2f(l);
          if (p.slot0 >= 0) p.part.lse[part_row] = lse2;
          else if (a.lse != nullptr) a.lse[out_row] = lse2 * kLn2;
        }
        // What clean_tile took out of V reaches the rows that read its key: infinity or NaN, whatever
        // the weight.  Limits rise from row to row, so one walk over the tiles with keys that are hidden from
        // some row (those of 256 / G tokens, and the tile they begin in) serves the warp.
        if (const int from = bars.cleaned[it & 3]) {
          __syncwarp();
          float2 odd[D / 64] = {};
          int key = (from - 1) * kKeys;
          for (int who = 0; who < 32 && (have >> who & 1); ++who) {
            const int end = min(__shfl_sync(0xffffffffu, limit, who), (k.tile0 + k.n_kv) * kKeys);
            const long long w_part = __shfl_sync(0xffffffffu, part_row, who);
            const int w_tok = __shfl_sync(0xffffffffu, tok, who), w_g = __shfl_sync(0xffffffffu, g, who);
            for (; key < end; ++key) {
              const long long off = key_offset(a, p.list, k.first_page, key);
              if (off < 0) continue;
              const uint32_t* v = reinterpret_cast<const uint32_t*>(a.vcache + off + (long long)k.kvh * D * 2);
#pragma unroll
              for (int e = 0; e < D / 64; ++e) {
                const float2 f = up2<BF16>(v[lane + 32 * e]);
                if (!(fabsf(f.x) < INFINITY)) odd[e].x += f.x;
                if (!(fabsf(f.y) < INFINITY)) odd[e].y += f.y;
              }
            }
            if (__shfl_sync(0xffffffffu, l, who) == 0.f) continue;  // it reads no key
#pragma unroll
            for (int e = 0; e < D / 64; ++e) {
              if (odd[e].x == 0.f && odd[e].y == 0.f) continue;
              if (p.slot0 >= 0) {
                float2* const o = reinterpret_cast<float2*>(p.part.out + w_part * D) + lane + 32 * e;
                *o = make_float2(o->x + odd[e].x, o->y + odd[e].y);
              } else {
                uint32_t* const o = reinterpret_cast<uint32_t*>(a.out + (long long)(k.t_begin + w_tok) * a.o_tok + (long long)(k.kvh * G + w_g) * D * 2) + lane + 32 * e;
                const float2 f = up2<BF16>(*o);
                *o = down2<BF16>(f.x + odd[e].x, f.y + odd[e].y);
              }
            }
          }
        }
        tc_fence_before();
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  }
  if (warp == 8 || warp == 9) {
    // ------------------------------------------------ K (warp 8) and V (warp 9)
    const bool is_k = warp == 8;
    uint64_t* full = is_k ? bars.kfull : bars.vfull;
    uint64_t* empty = is_k ? bars.kempty : bars.vempty;
    int n = 0;  // tiles loaded so far
    int held = 0;  // of them, those looked through
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const TileWork k = next_work(it);
      if (k.rows == 0) break;
      // A key that is hidden from a row takes part in its PV with weight 0, and 0 * infinity is NaN: the
      // tiles of V with such keys are looked through before the MMAs get them.
      const int hidden = is_k ? k.len : k.first_hidden(p.causal, G);
      if (!is_k && lane == 0) bars.cleaned[it & 3] = 0;  // whoever reads that of piece it - 4 is past it
      for (int j = 0; j < k.n_kv; ++j, ++n) {
        const int s = n % ST, use = n / ST;
        if (use > 0 && !(ok = wait(&empty[s], (use - 1) & 1))) break;
        const bool hold = hidden < k.len && (k.tile0 + j + 1) * kKeys > hidden;
        const uint32_t dst = (is_k ? sm_k : sm_v) + s * S::kStage;
        load_tile<D>(p, is_k ? &p.kmap : &p.vmap, is_k ? a.kcache : a.vcache, k.kvh, k.first_page, k.len, k.tile0 + j,
                     dst, hold ? &bars.vraw : &full[s], lane);
        if (hold) {
          if (!(ok = wait(&bars.vraw, held++ & 1))) break;
          if (clean_tile<BF16, D>(dst, lane)) {
            fence_proxy_async();
            if (lane == 0 && bars.cleaned[it & 3] == 0) bars.cleaned[it & 3] = k.tile0 + j + 1;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
        }
      }
      if (is_k && lane == 0) mbar_arrive(&bars.want);  // time to look for more
    }
    // no copy may be in flight when the CTA leaves, whatever the others did
    if (!ok && held > 0) wait(&bars.vraw, (held - 1) & 1);
    for (int d = max(0, n - ST); d < n; ++d) wait(&full[d % ST], (d / ST) & 1);
  } else if (warp == 10) {
    // ------------------------------------------------ MMAs
    constexpr uint32_t id_s = umma_idesc(BF16, kKeys, false), id_o = umma_idesc(BF16, D, true);
    const bool one = elect_one();
    const uint32_t q_low = umma_low(sm_q, 16), k_low = umma_low(sm_k, 16), v_low = umma_low(sm_v, kHalf);
    auto qk = [&](int i, int s) {
      if (one) {
        const uint32_t a_low = q_low + i * (kRows * D * 2 >> 4), b_low = k_low + s * (S::kStage >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k >> 2) * (kRows * 128) + (k & 3) * 32) >> 4;
          umma_ss<id_s>(tmem + i * 128, a_low + off, b_low + off, k > 0);
        }
        tc_commit(&bars.sfull[i]);
      }
      __syncwarp();
    };
    int n = 0;                          // tiles so far, both rings
    int pieces[2] = {0, 0}, tiles[2] = {0, 0};  // of each row tile
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const TileWork k = next_work(it);
      if (k.rows == 0) break;
      if (k.n_kv == 0) continue;
      const int n_tiles = k.rows > kRows ? 2 : 1;
      ok = wait(&bars.kfull[n % ST], (n / ST) & 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i >= n_tiles || !ok) continue;
        // a row tile's Q also says that its last S and O have been read
        ok = wait(&bars.qfull[i], pieces[i]++ & 1);
        tc_fence_after();
        if (ok) qk(i, n % ST);
      }
      if (ok && one) tc_commit(&bars.kempty[n % ST]);
      for (int j = 0; ok && j < k.n_kv; ++j, ++n) {
        const int s = n % ST, next = (n + 1) % ST;
        if (!(ok = wait(&bars.vfull[s], (n / ST) & 1))) break;
        if (j + 1 < k.n_kv && !(ok = wait(&bars.kfull[next], ((n + 1) / ST) & 1))) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i >= n_tiles || !ok) continue;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            ok = ok && wait(&bars.pfull[i][half], tiles[i] & 1);
            tc_fence_after();
            if (ok && one) {
              const uint32_t b_low = v_low + s * (S::kStage >> 4);
#pragma unroll
              for (int c = half * (kKeys / 64 * 3); c < (half ? kKeys / 16 : kKeys / 64 * 3); ++c)
                umma_ts<id_o>(tmem + 256 + i * 128, tmem + i * 128 + c * 8, b_low + c * (2048 >> 4), c > 0 ? 1u : (uint32_t)j);
            }
            __syncwarp();
          }
          ++tiles[i];
          if (ok && one) {
            if (j + 1 == k.n_kv) tc_commit(&bars.ofull[i]);
            if (i + 1 == n_tiles) tc_commit(&bars.vempty[s]);
          }
          __syncwarp();
          if (ok && j + 1 < k.n_kv) qk(i, next);
        }
        if (ok && j + 1 < k.n_kv && one) tc_commit(&bars.kempty[next]);
      }
    }
    if (one) tc_commit(&bars.done);
    __syncwarp();
    wait(&bars.done, 0);
  } else if (warp == 11) {
    // ------------------------------------------------ what to do
    // The grid has a block for every piece of work.  A resident CTA does its own and then takes over
    // blocks that have not started (cluster launch control), when the last tile of a piece is on its
    // way: no counter in memory, and pieces of any length spread evenly.
    const int token0 = token_of(p, 0);
    int it = 0;
    bool ok = true;
    auto tell = [&](const TileWork& k) {
      if (it >= 2) ok = wait(&bars.wempty[it & 1], ((it >> 1) - 1) & 1);
      if (ok && lane == 0) {
        work[it & 1] = k;
        mbar_arrive(&bars.wfull[it & 1]);
      }
      __syncwarp();
      ++it;
    };
    const int per_slot = a.num_kv_heads * p.n_splits;
    unsigned e = blockIdx.x;
    for (int asked = 0; ok; ++asked) {
      if (asked > 0) {
        if (lane == 0) {
          mbar_expect_tx(&bars.grant, 16);
          asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(&granted)),
                       "r"(smem_u32(&bars.grant)) : "memory");
        }
        if (!(ok = wait(&bars.grant, (asked - 1) & 1))) break;
        unsigned given;
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b128 x;\n\tld.shared.b128 x, [%2];\n\t"
            "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, x;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
            "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, x;\n\t}" : "=r"(given), "=r"(e) : "r"(smem_u32(&granted)) : "memory");
        fence_proxy_async();  // read before the next answer is written there
        __syncwarp();
        if (given == 0) break;  // every block has been started by now
      }
      // The sequence of a slot: sequence i has the slots from rows(i) / 256 + i on, which leaves it
      // enough of them without a scan; some stay empty.  Late slots, with the longest causal rows, first.
      const int slot = p.n_slots - 1 - (int)(e / (unsigned)per_slot), in_slot = (int)(e % (unsigned)per_slot);
      int seq = 0;
      for (int n = p.n_seq; n > 1;) {
        const int step = (n + 31) / 32, at = seq + lane * step;
        const bool below = lane * step < n && (int)((unsigned)((token_of(p, at) - token0) * G) / (2u * kRows)) + at <= slot;
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
        n = min(step, n - last * step);
        seq += last * step;
      }
      TileWork k;
      k.first_page = p.list.indptr[seq];
      k.len = list_keys(p.list, seq, a.block_size);
      k.t_begin = token_of(p, seq);
      k.n_new = min(token_of(p, seq + 1), a.num_tokens) - k.t_begin;
      k.row0 = (slot - (int)((unsigned)((k.t_begin - token0) * G) / (2u * kRows)) - seq) * (2 * kRows);
      if (k.t_begin < 0 || k.row0 < 0 || k.row0 >= k.n_new * G) continue;
      k.rows = min(k.n_new * G - k.row0, 2 * kRows);
      k.kvh = in_slot % a.num_kv_heads;
      k.split = in_slot / a.num_kv_heads;
      // keys: to the last one that the last row reads
      int k_end = k.len;
      if (p.causal) k_end = min(k.len, max(0, k.len - k.n_new + (k.row0 + k.rows - 1) / G + 1));
      const long long kv_tiles = (k_end + kKeys - 1) / kKeys;
      k.tile0 = (int)(kv_tiles * k.split / p.n_splits);
      k.n_kv = (int)(kv_tiles * (k.split + 1) / p.n_splits) - k.tile0;
      if (k.n_kv > 0)  // its rows of Q, on their way into L2 before the softmax warps ask for them
        for (int x = lane; x < k.rows; x += 32) {
          const int tok = (k.row0 + x) / G, g = k.row0 + x - tok * G;
          const char* src = a.q + (long long)(k.t_begin + tok) * a.q_tok + (long long)(k.kvh * G + g) * D * 2;
          prefetch_l2(src);
          if (D > 64) prefetch_l2(src + 128);
        }
      tell(k);
      if (ok) ok = wait(&bars.want, (it - 1) & 1);
    }
    TileWork end = {};
    if (ok) tell(end);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 10) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  wait_behind(p.beside);
}

// ---------------------------------------------------------------- join
// One warp a row: the row's partials, weighted by 2^(lse - max lse).  Sets [0, n_shared) come from
// the prefix, [n_shared, n_sets) from the own keys, one slot a token each; behind them the slots of
// the decode kernel's runs.  A lane looks up the lse of one part, so the parts' weights are known
// before the first of them is read and their loads do not wait for one another.
struct JoinParams {
  AttentionParams a;
  Partials part;
  int n_shared, n_sets;
  bool runs;        // the own keys were read by the decode kernel
  bool all;         // its whole requests, too, lie in slots
  int n_ranges, units_per_page;
};
constexpr int kJoinWarps = 8;

// HPW rows (heads of one token) a warp: one where there are few rows, so that their parts are the
// parallel loads, four where there are many.
template <bool BF16, int D, int HPW>
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_kernel(const JoinParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const AttentionParams& a = p.a;
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x, h0 = (blockIdx.y * kJoinWarps + (threadIdx.x >> 5)) * HPW;
  if (h0 >= a.num_heads) return;
  int first = 0;  // parts of a row: sets [first, n_sets), then n_runs slots of the runs
  int x0 = 0, n_runs = 0;
  const bool grouped = p.n_shared > 0 && a.group_indptr != nullptr;
  const int q_first = a.qo_indptr != nullptr ? a.qo_indptr[0] : 0;
  const int q_last = a.qo_indptr != nullptr ? a.qo_indptr[a.num_requests] : a.num_tokens;
  const int b0 = grouped ? min(max(a.group_indptr[0], 0), a.num_requests) : 0;
  const int b1 = grouped ? min(max(a.group_indptr[a.num_groups], 0), a.num_requests) : 0;
  if (p.runs) {
    const int* indptr = a.own.indptr;
    const int axis0 = indptr[0], begin = indptr[t], end = indptr[t + 1];
    const unsigned units = (unsigned)max(indptr[a.num_requests] - axis0, 0) * p.units_per_page + a.num_requests;
    const unsigned chunk = (units + p.n_ranges - 1) / p.n_ranges;
    if (end > begin) {  // the runs that hold a part of the request
      const unsigned s0 = (unsigned)(begin - axis0) * p.units_per_page + t;
      x0 = (int)min(s0 / chunk, p.n_ranges - 1u);
      n_runs = max((int)min((s0 + (unsigned)(end - begin) * p.units_per_page - 1) / chunk, p.n_ranges - 1u) - x0 + 1, 0);
      if (n_runs == 1 && !p.all) return;  // finished by its run
    }
  }
  if (t < q_first || t >= q_last) return;  // left as it is
  if (grouped) {
    // a request outside every group has no set from the prefix
    const int t0 = a.qo_indptr != nullptr ? a.qo_indptr[b0] : b0, t1 = a.qo_indptr != nullptr ? a.qo_indptr[b1] : b1;
    if (t < t0 || t >= t1) first = p.n_shared;
  }
  const long long slot0 = (long long)p.n_sets * a.num_tokens;
  const int n_set = p.n_sets - first, n = n_set + n_runs;
  auto slot_of = [&](int i) -> long long {
    if (i < n_set) return (long long)(first + i) * a.num_tokens + t;
    if (n_runs == 1) return slot0 + 2 * p.n_ranges + t;  // whole
    const int x = i - n_set;
    return slot0 + 2 * (x0 + x) + (x == 0 ? 1 : 0);
  };
  constexpr int E = D / 32, kLook = 32 / HPW, kBatch = 8 / HPW;  // parts looked up / loaded at once
  float acc[HPW][E] = {}, m = -INFINITY, l = 0.f;  // m, l: of the head this lane looks up
  const int hh = lane / kLook;
  for (int base = 0; base < n; base += kLook) {
    const int count = min(kLook, n - base);
    long long at = 0;
    float s = -INFINITY;
    if (lane % kLook < count) {
      at = slot_of(base + lane % kLook) * a.num_heads;
      if (h0 + hh < a.num_heads) s = p.part.lse[at + h0 + hh];
    }
    float top = fmaxf(s, m);
#pragma unroll
    for (int o = kLook / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // NaN counts as a part (its row is NaN); a part without a key was not written
    const float w = s == -INFINITY ? 0.f : exp2_fast(s - top);
    const float keep = m == -INFINITY ? 0.f : exp2_fast(m - top);
    float sum = w;
#pragma unroll
    for (int o = kLook / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = fmaf(l, keep, sum);
    m = top;
#pragma unroll
    for (int x = 0; x < HPW; ++x) {
      const float k = __shfl_sync(0xffffffffu, keep, x * kLook);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[x][e] *= k;
    }
    for (int i = 0; i < count; i += kBatch) {
      float v[kBatch][HPW][E];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const long long slot = __shfl_sync(0xffffffffu, at, min(i + u, count - 1));
#pragma unroll
        for (int x = 0; x < HPW; ++x) {
          const float* src = p.part.out + (slot + min(h0 + x, a.num_heads - 1)) * D + lane * E;
          if constexpr (E == 4) {
            const float4 f = *reinterpret_cast<const float4*>(src);
            v[u][x][0] = f.x; v[u][x][1] = f.y; v[u][x][2] = f.z; v[u][x][3] = f.w;
          } else {
            const float2 f = *reinterpret_cast<const float2*>(src);
            v[u][x][0] = f.x; v[u][x][1] = f.y;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
#pragma unroll
        for (int x = 0; x < HPW; ++x) {
          const float wi = i + u < count ? __shfl_sync(0xffffffffu, w, x * kLook + min(i + u, count - 1)) : 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[x][e] = fmaf(wi, wi == 0.f ? 0.f : v[u][x][e], acc[x][e]);
        }
    }
  }
#pragma unroll
  for (int x = 0; x < HPW; ++x) {
    const float total = __shfl_sync(0xffffffffu, l, x * kLook), most = __shfl_sync(0xffffffffu, m, x * kLook);
    if (h0 + x >= a.num_heads) continue;
    const float inv = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);
    uint32_t* out = reinterpret_cast<uint32_t*>(a.out + (long long)t * a.o_tok + ((long long)(h0 + x) * D + lane * E) * 2);
    uint32_t r[E / 2];
#pragma unroll
    for (int e = 0; e < E; e += 2) r[e / 2] = down2<BF16>(acc[x][e] * inv, acc[x][e + 1] * inv);
    if constexpr (E == 4) *reinterpret_cast<uint2*>(out) = make_uint2(r[0], r[1]);
    else out[0] = r[0];
    if (a.lse != nullptr && lane == 0)
      a.lse[(long long)t * a.num_heads + h0 + x] = total == 0.f ? -INFINITY : (most + log2f(total)) * kLn2;
  }
}

// ---------------------------------------------------------------- launch rules
// Pairs of row tiles of a key head: every sequence has one at least.
long long row_tiles(long long tokens, long long seqs, const AttentionParams& p) {
  const long long tiles = (tokens * (p.num_heads / p.num_kv_heads) + 2 * kRows - 1) / (2 * kRows);
  return tiles < seqs ? seqs : tiles;
}

// Splits of the keys so that the row tiles fill the GPU, a tile of keys each at least.  One count for all
// sequences, from the mean of their keys by the length of the table.  (Twice or three times the pieces:
// 256 requests behind 8192 keys, prefix and own keys one behind the other, 108 and 114 us instead of 104.)
int splits_of(long long tokens, long long seqs, long long pages, const AttentionParams& p, int sms) {
  const long long keys = pages * p.block_size / (seqs > 0 ? seqs : 1);
  const long long tiles = row_tiles(tokens, seqs, p);
  long long n = sms / ((tiles > 0 ? tiles : 1) * p.num_kv_heads);
  if (n > keys / kKeys) n = keys / kKeys;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}

AttentionPlan plan_of(const AttentionParams& p, int sms) {
  AttentionPlan r{};
  const int G = p.num_heads / p.num_kv_heads;
  const bool shared = p.prefix.indptr != nullptr;
  r.units_per_page = (p.block_size + kTile - 1) / kTile;
  r.rows = p.head_dim != 64 && p.head_dim != 128;
  if (r.rows) return r;
  r.runs = p.qo_indptr == nullptr && G <= 16;
  if (shared) r.shared_splits = splits_of(p.num_tokens, p.num_groups, p.prefix.num_indices, p, sms);
  if (r.runs) {
    // One CTA an SM.  The more heads a CTA takes, the fewer warps meet when a request ends, but
    // the shorter the runs: a run should hold 16 units at least for each request that it cuts.
    const long long units = (p.own.num_indices + 1) * r.units_per_page;
    int shift = 3;
    while (shift > 0 && (1 << (shift - 1)) >= p.num_kv_heads) --shift;
    auto blocks = [&](int s) { return (p.num_kv_heads + (1 << s) - 1) >> s; };
    while (shift > 0 && units * blocks(shift) < 16ll * sms) --shift;
    r.hb_shift = shift;
    int run_sms = sms;
    if (shared) {
      // Beside the tiles of a prefix the runs take some of the SMs, and the prefix's pieces go over the
      // others in whole rounds: the pair of shares and splits that ends first, by what either takes on
      // an SM - 0.19 us a 16-key unit of a head of 128 (43 GB/s), 1.7 us a key tile and 8 us a piece,
      // taken for other head dims too - and what the join reads.  (256 requests behind 8192 keys: 104 us one behind the other, 100 with
      // half the SMs each, 114 where the pieces leave a third round; 8 groups: 58 to 48 us.)
      const double own = (double)units * p.num_kv_heads * p.head_dim * (0.19 / 128);
      const double tiles = (double)row_tiles(p.num_tokens, p.num_groups, p) * p.num_kv_heads;
      const long long keys = p.prefix.num_indices * p.block_size / (p.num_groups > 0 ? p.num_groups : 1);
      const double key_tiles = (double)((keys + kKeys - 1) / kKeys);
      const double part = (double)p.num_tokens * p.num_heads * p.head_dim * 8 / 6e6;
      // several prefixes: the counts give their mean, the longest may be twice that
      const double longest = p.num_groups > 1 ? 1 : 0;
      auto piece = [&](double splits) { return key_tiles / splits * 1.7 + 8; };
      auto tiles_end = [&](double rounds, double splits) { return rounds * piece(splits) + longest * key_tiles / splits * 1.7; };
      const double all = r.shared_splits;  // one behind the other, each on all SMs
      double best = own / sms + 6 + tiles_end((double)(((long long)(tiles * all) + sms - 1) / sms), all) + all * part;
      const int most = key_tiles < 12 ? (int)key_tiles : 12;
      for (int splits = 1; splits <= most; ++splits)
        for (int rounds = 1; rounds <= 3; ++rounds) {
          const long long left = ((long long)tiles * splits + rounds - 1) / rounds;
          const long long mine = sms - left;
          if (mine < 2 * sms / 5) continue;
          const double ends = own / mine + 6, t = tiles_end(rounds, splits);
          const double total = (t > ends ? t : ends) + splits * part;
          if (total < best) {
            best = total;
            run_sms = (int)mine;
            r.shared_splits = splits;
          }
        }
    }
    r.n_ranges = run_sms / blocks(shift);
    if (r.n_ranges < 1) r.n_ranges = 1;
    r.slots = 2ll * r.n_ranges + (shared ? p.num_requests : 0);
    r.join = true;
  } else {
    r.own_splits = splits_of(p.num_tokens, p.num_requests, p.own.num_indices, p, sms);
    r.join = shared || r.own_splits > 1;
  }
  if (r.join) r.slots += (long long)(r.shared_splits + r.own_splits) * p.num_tokens;
  return r;
}

long long align256(long long x) { return (x + 255) & ~255ll; }

Partials partials_at(const AttentionParams& p, const AttentionPlan& plan) {
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

// The driver's encoder, through the runtime (the library links no libcuda).
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    cudaGetLastError();
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// [page][head][entry][element] of one plane; false where TMA cannot address it.
bool encode_plane(const AttentionParams& p, const char* base, int box, CUtensorMap* map) {
  const EncodeTiled fn = encoder();
  if (fn == nullptr || p.num_blocks < 1) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)p.head_dim, (cuuint64_t)p.block_size, (cuuint64_t)p.num_kv_heads, (cuuint64_t)p.num_blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)p.slot_stride, (cuuint64_t)p.head_dim * 2, (cuuint64_t)p.block_stride};
  const cuuint32_t box_dims[4] = {64, (cuuint32_t)box, 1, 1}, ones[4] = {1, 1, 1, 1};
  return fn(map, p.is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<char*>(base),
            dims, strides, box_dims, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Shared memory beyond the default has to be asked for, once per kernel and device.
template <class K>
cudaError_t allow_smem(K kernel, int most, std::atomic<unsigned long long>* asked) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (asked->load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess) asked->fetch_or(bit, std::memory_order_release);
  return e;
}

template <bool BF16, int D, int NT, int NST>
cudaError_t launch_decode(const AttentionParams& p, const AttentionPlan& plan, bool pdl, cudaStream_t stream) {
  DecodeParams d{};
  d.a = p;
  d.part = partials_at(p, plan);
  d.n_ranges = plan.n_ranges;
  d.hb_shift = plan.hb_shift;
  d.units_per_page = plan.units_per_page;
  d.slot0 = (long long)(plan.shared_splits + plan.own_splits) * p.num_tokens;
  d.join_all = plan.shared_splits > 0;
  const int G = p.num_heads / p.num_kv_heads, HB = 1 << plan.hb_shift;
  // Below 512 MB of pages the boxes are as fast as rows or faster, since they cost fewer instructions
  // (256 requests of up to 512 keys, 8 key heads of 128, beside an 8192-key prefix: 91 us, by rows 92; 300 of
  // up to 200 keys, 37.6 and 39.0; 8 prefixes of up to 4000, 49.1 and 50.4).  Above it HBM alone counts, and
  // the rows' 16-byte requests keep it busier (256 requests of up to 4000 keys 330 us, by rows 314; with
  // pages of 32 keys 334 and 310; 64 of up to 16000, 4 heads of 64, 138 and 135).  At 524 MB they are equal.
  // Among other kernels that leave the L2 cache full of written lines both take 324 us for the first of these.
  const double bytes = 4.0 * p.own.num_indices * p.block_size * p.num_kv_heads * D;
  const bool rows = bytes > 512.0 * (1 << 20);
  d.box = rows ? 0 : p.block_size % kTile == 0 ? kTile : p.block_size == 8 ? 8 : 0;
  const bool tma = d.box > 0 && encode_plane(p, p.kcache, d.box, &d.kmap) && encode_plane(p, p.vcache, d.box, &d.vmap);
  auto kernel = tma ? attention_decode_kernel<BF16, D, NT, NST, true> : attention_decode_kernel<BF16, D, NT, NST, false>;
  const int smem = DecodeSmem<D, NST>::bytes(G, HB);
  static std::atomic<unsigned long long> asked[2];
  cudaError_t e = allow_smem(kernel, DecodeSmem<D, NST>::bytes(8 * NT, 1), &asked[tma]);
  if (e != cudaSuccess) return e;
  Launch go(dim3(plan.n_ranges, (p.num_kv_heads + HB - 1) / HB), kDecodeWarps * 32, smem, pdl, stream);
  return cudaLaunchKernelEx(&go.cfg, kernel, d);
}

template <bool BF16, int D>
cudaError_t launch_tile(const AttentionParams& p, const AttentionPlan& plan, bool shared, bool beside, bool pdl, cudaStream_t stream) {
  TileParams t{};
  t.a = p;
  t.list = shared ? p.prefix : p.own;
  t.part = partials_at(p, plan);
  t.shared = shared;
  t.n_seq = shared ? p.num_groups : p.num_requests;
  const int G = p.num_heads / p.num_kv_heads;
  const long long slots = (long long)p.num_tokens * G / (2 * kRows) + t.n_seq;
  t.n_splits = shared ? plan.shared_splits : plan.own_splits;
  if (slots > 0x7fffffffll || p.num_kv_heads > 65535) return cudaErrorInvalidConfiguration;
  t.n_slots = (int)slots;
  t.slot0 = plan.join ? (shared ? 0 : plan.shared_splits) : -1;
  t.causal = !shared && p.causal;
  t.beside = beside;
  const int bs = p.block_size;
  if (bs % kKeys == 0) t.box = kKeys;
  else if (bs >= 8 && bs < kKeys && kKeys % bs == 0) t.box = bs;
  if (t.box > 0 && !(encode_plane(p, p.kcache, t.box, &t.kmap) && encode_plane(p, p.vcache, t.box, &t.vmap))) t.box = 0;
  auto kernel = attention_tile_kernel<BF16, D>;
  const int smem = TileSmem<D>::kBytes + 1024;  // rounded up to the swizzle's 1024-byte pattern
  static std::atomic<unsigned long long> asked;
  cudaError_t e = allow_smem(kernel, smem, &asked);
  if (e != cudaSuccess) return e;
  const long long pieces = slots * p.num_kv_heads * t.n_splits;
  if (pieces > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  Launch go(dim3((unsigned)pieces), kTileThreads, smem, pdl, stream);
  return cudaLaunchKernelEx(&go.cfg, kernel, t);
}

template <bool BF16, int D>
cudaError_t launch_join(const AttentionParams& p, const AttentionPlan& plan, int sms, bool pdl, cudaStream_t stream) {
  JoinParams j{};
  j.a = p;
  j.part = partials_at(p, plan);
  j.n_shared = plan.shared_splits;
  j.n_sets = plan.shared_splits + plan.own_splits;
  j.runs = plan.runs;
  j.all = plan.shared_splits > 0;
  j.n_ranges = plan.n_ranges;
  j.units_per_page = plan.units_per_page;
  // four rows a warp once one a warp would not fit the GPU at once (64 warps an SM)
  const bool many = (long long)p.num_tokens * p.num_heads > 64ll * sms;
  const int heads = kJoinWarps * (many ? 4 : 1);
  Launch go(dim3(p.num_tokens, (p.num_heads + heads - 1) / heads), kJoinWarps * 32, 0, pdl, stream);
  return cudaLaunchKernelEx(&go.cfg, many ? attention_join_kernel<BF16, D, 4> : attention_join_kernel<BF16, D, 1>, j);
}

template <bool BF16>
cudaError_t launch_rows(const AttentionParams& p, bool pdl, cudaStream_t stream) {
  const long long ctas = ((long long)p.num_tokens * p.num_heads + 3) / 4;
  if (ctas > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  Launch go(dim3((unsigned)ctas), 128, 0, pdl, stream);
  return cudaLaunchKernelEx(&go.cfg, attention_rows_kernel<BF16>, p);
}

template <bool BF16, int D>
cudaError_t launch_matrix(const AttentionParams& p, const AttentionPlan& plan, int sms, bool pdl, int* launches, cudaStream_t stream) {
  const bool shared = plan.shared_splits > 0;
  cudaError_t e = cudaSuccess;
  if (plan.runs) {
    // the runs take their share of the SMs (plan_of) and leave the others to the prefix
    const bool few = p.num_heads / p.num_kv_heads <= 8;
    constexpr int kDeep = D == 64 ? 6 : 3;
    e = few ? launch_decode<BF16, D, 1, kDeep>(p, plan, pdl, stream) : launch_decode<BF16, D, 2, D == 64 ? 5 : 2>(p, plan, pdl, stream);
    *launches += e == cudaSuccess;
    if (e == cudaSuccess && shared) {
      e = launch_tile<BF16, D>(p, plan, true, true, pdl, stream);
      *launches += e == cudaSuccess;
    }
  } else {
    // few long pieces first, the short ones of the own keys on the SMs that they leave
    if (shared) {
      e = launch_tile<BF16, D>(p, plan, true, false, pdl, stream);
      *launches += e == cudaSuccess;
    }
    if (e == cudaSuccess) {
      e = launch_tile<BF16, D>(p, plan, false, shared, pdl, stream);
      *launches += e == cudaSuccess;
    }
  }
  if (e == cudaSuccess && plan.join) {
    e = launch_join<BF16, D>(p, plan, sms, pdl, stream);
    *launches += e == cudaSuccess;
  }
  return e;
}

template <bool BF16>
cudaError_t launch_typed(const AttentionParams& p, const AttentionPlan& plan, int sms, bool pdl, int* launches, cudaStream_t stream) {
  if (plan.rows) {
    *launches = 1;
    return launch_rows<BF16>(p, pdl, stream);
  }
  return p.head_dim == 64 ? launch_matrix<BF16, 64>(p, plan, sms, pdl, launches, stream)
                          : launch_matrix<BF16, 128>(p, plan, sms, pdl, launches, stream);
}

}  // namespace

AttentionPlan attention_plan(const AttentionParams& p, int sms) { return plan_of(p, sms); }

long long attention_workspace_bytes(const AttentionParams& p, const AttentionPlan& plan) {
  if (plan.slots == 0) return 0;
  return align256(plan.slots * p.num_heads * 4) + align256(plan.slots * p.num_heads * p.head_dim * 4);
}

cudaError_t launch_attention(const AttentionParams& p, const AttentionPlan& plan, int sms, bool pdl, int* launches, cudaStream_t stream) {
  *launches = 0;
  return p.is_bf16 ? launch_typed<true>(p, plan, sms, pdl, launches, stream)
                   : launch_typed<false>(p, plan, sms, pdl, launches, stream);
}

}  // namespace lms
