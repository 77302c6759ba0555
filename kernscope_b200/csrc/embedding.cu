// embedding.cu -- token embedding with scaling, and the table's gradient by
// sorted tokens.
//
//   out[i] = scale * table[token[i]]
//   dtable[v] = scale * sum over { i : token[i] = v } of dout[i]
//
// Both are bound by memory.  The gradient sums each table row in a fixed
// order, the order of the positions, whatever the timing: a stable radix sort
// of the tokens brings equal ones together, then CTAs walk the sorted
// positions over one segment of columns each, adding in fp32 and writing a row
// when its token ends.  A token whose positions lie in several chunks (of
// `chunk` positions) leaves an fp32 partial sum per chunk, and the CTA that
// finishes last adds those in order.  No floating-point atomics.
#include <algorithm>
#include <cuda_fp16.h>

#include "ks_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// 16 bytes (VEC) or lane-strided single elements of a row, as fp32
// ---------------------------------------------------------------------------
template <int DT>
struct Elem;
template <>
struct Elem<KS_BF16> {
  using T = uint16_t;
  static constexpr int kPer = 8;
  KS_DEV static float get(uint16_t v) { return ks_bf16_to_f32(v); }
  KS_DEV static uint16_t put(float v) { return ks_f32_to_bf16(v); }
};
template <>
struct Elem<KS_F16> {
  using T = uint16_t;
  static constexpr int kPer = 8;
  KS_DEV static float get(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  KS_DEV static uint16_t put(float v) { return __half_as_ushort(__float2half_rn(v)); }
};
template <>
struct Elem<KS_F32> {
  using T = float;
  static constexpr int kPer = 4;
  KS_DEV static float get(float v) { return v; }
  KS_DEV static float put(float v) { return v; }
};

// A lane's share of a row's segment, still as stored: 16 bytes (VEC), or as many
// single elements 32 columns apart, for rows that are not 16-byte aligned.
template <int DT, bool VEC>
struct Raw {
  using T = typename Elem<DT>::T;
  static constexpr int W = Elem<DT>::kPer;
  alignas(16) T v[W];
  // p: the row at the segment's first column; c: that column; lanes past `dim` hold zeros
  KS_DEV void load(const T *p, int64_t c, int64_t dim, int lane) {
    if constexpr (VEC) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (c + lane * W < dim) x = __ldg(reinterpret_cast<const uint4 *>(p + lane * W));
      *reinterpret_cast<uint4 *>(v) = x;
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = c + lane + j * 32 < dim ? __ldg(p + lane + j * 32) : T(0);
    }
  }
  KS_DEV void store(T *p, int64_t c, int64_t dim, int lane, bool stream) const {
    if constexpr (VEC) {
      if (c + lane * W < dim) {
        auto q = reinterpret_cast<uint4 *>(p + lane * W);
        if (stream) __stcs(q, *reinterpret_cast<const uint4 *>(v));
        else *q = *reinterpret_cast<const uint4 *>(v);
      }
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (c + lane + j * 32 < dim) p[lane + j * 32] = v[j];
    }
  }
};

// ---------------------------------------------------------------------------
// Forward: a warp per (row, four segments of 512 bytes), their loads in flight.
// A token outside [0, vocab) gives a row of zeros.  Outputs that do not fit the L2
// are stored as streams (65536 x 4096 bf16: 122.5 -> 119.4 us), smaller ones stay
// for their reader.  Bound by memory: 65536 x 4096 from 32000 rows, 710 MB, at 5.9
// TB/s; 64 x 2048 by the call, 9 us, whose kernel takes 4.
// ---------------------------------------------------------------------------
template <int DT, bool VEC>
__global__ void __launch_bounds__(256)
    emb_lookup_kernel(const int64_t *__restrict__ tokens, int64_t n, const typename Elem<DT>::T *__restrict__ table,
                      int64_t table_stride, typename Elem<DT>::T *__restrict__ out, int64_t out_stride, int64_t vocab,
                      int64_t dim, float scale, int stream) {
  using E = Elem<DT>;
  constexpr int W = E::kPer, kSeg = 32 * W, U = 4;
  const int lane = threadIdx.x & 31;
  const int64_t segs = (dim + kSeg - 1) / kSeg, groups = (segs + U - 1) / U;
  const int64_t i = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (i >= n * groups) return;
  const int64_t row = i / groups, c0 = (i - row * groups) * U * kSeg;
  const int64_t t = __ldg(tokens + row);
  const bool in = t >= 0 && t < vocab;
  Raw<DT, VEC> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    x[u].load(table + (in ? t : 0) * table_stride + c0 + u * kSeg, c0 + u * kSeg, in ? dim : 0, lane);
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int j = 0; j < W; ++j) x[u].v[j] = in ? E::put(E::get(x[u].v[j]) * scale) : 0;  // outside: not 0 * inf
    x[u].store(out + row * out_stride + c0 + u * kSeg, c0 + u * kSeg, dim, lane, stream != 0);
  }
}

KS_DEV uint32_t token_key(int64_t t, int64_t vocab, int64_t padding) {
  return t < 0 || t >= vocab || t == padding ? uint32_t(vocab) : uint32_t(t);  // the excluded ones sort last
}

// ---------------------------------------------------------------------------
// Stable sort of (token, position), and the zeros of the dense gradient.
//
// Up to kRankMax positions: each position's place is the number of smaller
// (token, position) pairs, counted directly, 16 threads a position, every CTA
// with all keys in shared memory.  (Whole calls with the limit at 8192 and as it is:
// 6208 x 72 into 3351 rows 21.0 and 20.5 us, 8192 x 256 into 32768 34.0 and 22.5:
// the comparisons keep the SMs from writing zeros.)
//
// More: radix, below.
// One cluster of 8 CTAs sorts: least-significant-digit radix passes of up to
// 10 bits, the digit counts exchanged through distributed shared memory (no
// counters in global memory, no spinning).  Each warp owns a contiguous part
// of the input and ranks 32 elements at a time with a match over the warp, so
// equal digits keep their order.  The other clusters of the grid write the
// zeros meanwhile, up to 512 KB a CTA: the sort is latency-bound and uses no bandwidth
// to speak of.  (With one zeroing CTA per SM the clusters that found no room at
// first made a second round of it: 134 MB in 36 us, 537 MB in 134, where it is 29
// and 94 now.  8192 tokens alone sort in 14 us, 131072 in 61.)
// ---------------------------------------------------------------------------
constexpr int kCluster = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kBatch = 8;  // loads in flight per lane

// What the other CTAs of the sorting kernels zero: rows `stride` apart and
// `bytes` long (even, as are their addresses), `share` bytes per CTA.
struct Zeros {
  char *p;
  int64_t rows, bytes, stride, share;
};

KS_DEV void zero_rows(const Zeros &z, int64_t cta) {
  const int64_t rows = z.rows, bytes = z.bytes, stride = z.stride, first = cta * z.share;
  char *p = z.p;
  const int64_t end = min(first + z.share, rows * bytes);
  for (int64_t at = first; at < end;) {
    const int64_t r = at / bytes, c = at - r * bytes;
    const int64_t len = min(bytes - c, end - at);
    char *q = p + r * stride + c;
    const int64_t head = min(len, int64_t((16 - (reinterpret_cast<uintptr_t>(q) & 15)) & 15));
    const int64_t vecs = (len - head) / 16, tail = len - head - vecs * 16;
    uint4 *v = reinterpret_cast<uint4 *>(q + head);
    for (int64_t i = threadIdx.x; i < vecs; i += kSortThreads) v[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x < head / 2) reinterpret_cast<uint16_t *>(q)[threadIdx.x] = 0;
    if (threadIdx.x < tail / 2) reinterpret_cast<uint16_t *>(q + len - tail)[threadIdx.x] = 0;
    at += len;
  }
}

constexpr int kRankMax = 4096;
constexpr int kRankBits = 12;
constexpr int kRankRows = kSortThreads / 16;  // positions per CTA

// FITS: token and position fit one 32-bit key (vocab < 2^20, position < 2^12).
template <bool FITS>
__global__ void __launch_bounds__(kSortThreads)
    emb_rank_kernel(const int64_t *__restrict__ tokens, int n, int64_t vocab, int64_t padding, uint2 *__restrict__ out,
                    uint32_t *counters, int64_t counters_n, const __grid_constant__ Zeros zeros) {
  __shared__ __align__(16) uint32_t keys[kRankMax];
  const int tid = threadIdx.x, ctas = (n + kRankRows - 1) / kRankRows;
  if (tid == 0) ks_pdl_release();
  if (int(blockIdx.x) >= ctas) {
    zero_rows(zeros, int64_t(blockIdx.x) - ctas);
    return;
  }
  for (int64_t i = int64_t(blockIdx.x) * kSortThreads + tid; i < counters_n; i += int64_t(ctas) * kSortThreads)
    counters[i] = 0;
  const int padded = (n + 63) / 64 * 64;
#pragma unroll 4
  for (int i = tid; i < padded; i += kSortThreads) {
    uint32_t k = 0xffffffffu;  // sorts behind everything
    if (i < n) {
      k = token_key(tokens[i], vocab, padding);
      if (FITS) k = k << kRankBits | uint32_t(i);
    }
    keys[i] = k;
  }
  __syncthreads();
  const int i = blockIdx.x * kRankRows + tid / 16;
  const uint32_t mine = i < n ? keys[i] : 0;
  int below = 0;
  for (int j = tid % 16 * 4; j < padded; j += 64) {
    const uint4 k = *reinterpret_cast<const uint4 *>(keys + j);
    if (FITS) {
      below += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
    } else {
      below += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
      below += (k.x == mine && j < i) + (k.y == mine && j + 1 < i) + (k.z == mine && j + 2 < i) +
               (k.w == mine && j + 3 < i);
    }
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
  if (tid % 16 == 0 && i < n) out[below] = make_uint2(FITS ? mine >> kRankBits : mine, uint32_t(i));
}

__global__ void __launch_bounds__(kSortThreads, 1)
    emb_sort_kernel(const int64_t *__restrict__ tokens, int64_t n, int64_t vocab, int64_t padding, int passes, int bits,
                    uint2 *buf0, uint2 *buf1, uint32_t *counters, int64_t counters_n,
                    const __grid_constant__ Zeros zeros) {
  extern __shared__ uint32_t sh[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) ks_pdl_release();
  if (blockIdx.x >= kCluster) {
    zero_rows(zeros, int64_t(blockIdx.x) - kCluster);
    return;
  }
  for (int64_t i = int64_t(blockIdx.x) * kSortThreads + tid; i < counters_n; i += kCluster * kSortThreads) counters[i] = 0;
  const int bins = 1 << bits;
  uint32_t *count = sh;                     // [warp][bin]: counts, then this warp's first rank in the CTA
  uint32_t *cta_count = sh + kSortWarps * bins;  // [bin], read by the whole cluster
  uint32_t *base = cta_count + bins;        // [bin]: where this CTA's elements of a digit begin
  __shared__ uint32_t wsum[kSortWarps];
  const uint32_t rank = ks_cluster_ctarank();
  const int64_t per_cta = ((n + kCluster - 1) / kCluster + kSortThreads - 1) / kSortThreads * kSortThreads;
  const int64_t per_warp = per_cta / kSortWarps;
  const int64_t lo = rank * per_cta + warp * per_warp, hi = min(lo + per_warp, n);
  for (int pass = 0; pass < passes; ++pass) {
    const uint2 *in = pass & 1 ? buf0 : buf1;  // pass 0 reads the tokens
    uint2 *out = pass & 1 ? buf1 : buf0;
    const int shift = pass * bits;
    auto fetch = [&](int64_t i) {
      if (pass > 0) return __ldcg(in + i);
      const int64_t t = __ldg(tokens + i);
      return make_uint2(token_key(t, vocab, padding), uint32_t(i));
    };
    for (int i = tid; i < kSortWarps * bins; i += kSortThreads) count[i] = 0;
    __syncthreads();
    uint32_t *mine = count + warp * bins;
    uint2 kv[kBatch];
    for (int64_t i = lo + lane; i < hi; i += 32 * kBatch) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i + u * 32 < hi) kv[u] = fetch(i + u * 32);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i + u * 32 < hi) atomicAdd(mine + ((kv[u].x >> shift) & (bins - 1)), 1u);
    }
    __syncthreads();
    if (tid < bins) {
      uint32_t s = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = count[w * bins + tid];
        count[w * bins + tid] = s;
        s += c;
      }
      cta_count[tid] = s;
    }
    ks_cluster_sync();
    uint32_t total = 0, before = 0;
    if (tid < bins) {
      const uint32_t at = ks_smem_u32(cta_count + tid);
#pragma unroll
      for (uint32_t r = 0; r < kCluster; ++r) {
        uint32_t c;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c) : "r"(ks_mapa(at, r)) : "memory");
        total += c;
        if (r < rank) before += c;
      }
    }
    // exclusive scan of the digits' totals
    uint32_t incl = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      uint32_t v = wsum[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      wsum[lane] = v;
    }
    __syncthreads();
    if (tid < bins) base[tid] = before + incl - total + (warp ? wsum[warp - 1] : 0u);
    __syncthreads();
    for (int64_t i0 = lo + lane; i0 - lane < hi; i0 += 32 * kBatch) {
      if (per_warp > 32 * kBatch) {  // otherwise they are still in kv
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (i0 + u * 32 < hi) kv[u] = fetch(i0 + u * 32);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (i0 - lane + u * 32 >= hi) break;
        const bool have = i0 + u * 32 < hi;
        const uint32_t d = have ? (kv[u].x >> shift) & (bins - 1) : uint32_t(bins);
        const uint32_t peers = __match_any_sync(0xffffffffu, d);
        const uint32_t below = __popc(peers & ((1u << lane) - 1u));
        if (have) out[base[d] + mine[d] + below] = kv[u];
        __syncwarp();
        if (have && below == 0) mine[d] += __popc(peers);
        __syncwarp();
      }
    }
    ks_cluster_sync();  // out is complete; cta_count may be rewritten
  }
}

// ---------------------------------------------------------------------------
// Sums over the sorted positions.  A CTA takes one chunk of them and one
// segment of columns (16 bytes a thread); every CTA has the same number of
// rows to read, whatever the tokens are.  The rows come through a ring of
// shared memory, kStages stages of kRows rows, filled by bulk copies (one per
// row, of up to 4 KB), so that about 100 KB a CTA are in flight while the
// threads add; reading them into registers instead (warps over short windows,
// 4 to 8 rows in flight each) reached 3.4 TB/s at 131072 x 1024 fp32.  Of rows that
// are not 16-byte aligned the ring takes the 16-byte granules they lie in, and the
// threads read single values at the row's offset.  (20000 x 510 bf16 into 50000 rows
// 36.8 us a call; with plain loads, four rows at a time, 56.7.)
// Measured: 131072 x 1024 fp32 into as many rows 123 us, 5.2 TB/s; 8192 x 2048 bf16
// 19 us, where the chain of start, sorted keys, first rows and joins (3 us) bounds
// it and not its 60 MB.
// part: [chunk][2][ld] fp32, slot 0 for a token that began in an earlier chunk,
// slot 1 for one that goes on into the next.
// ---------------------------------------------------------------------------
constexpr int kRows = 8;
constexpr int kStages = 3;
constexpr int kMaxChunk = 1024;
constexpr int kSegThreads = 256;  // at most: 4 KB of a row

// What every CTA of a launch shares.
template <int DT, int ODT>
struct GradArgs {
  const uint2 *sorted;
  int64_t n;
  int chunk;
  uint32_t segs;
  const typename Elem<DT>::T *dout;
  int64_t dout_stride;
  typename Elem<ODT>::T *dtable;
  int64_t dtable_stride, vocab, dim;
  float scale;
  int accumulate;
  float *part;
  int64_t ld;
  uint32_t *arrived;  // [chunk][2][segment] CTAs of a group that left their partials, [chunk][segment] groups
  int64_t chunks;
};

// A thread's sums: 16 bytes' worth of columns, adjacent (VEC) or blockDim apart.
// The methods take addresses at the segment's first column; `left`: columns from
// there to the row's end.
template <int DT, int ODT, bool VEC>
struct Sum {
  using E = Elem<DT>;
  using O = Elem<ODT>;
  static constexpr int W = E::kPer;
  float a[W];
  KS_DEV static int cols() { return blockDim.x * W; }
  KS_DEV static int col(int j) { return VEC ? threadIdx.x * W + j : threadIdx.x + j * blockDim.x; }
  KS_DEV void clear() {
#pragma unroll
    for (int j = 0; j < W; ++j) a[j] = 0.f;
  }
  KS_DEV void put_part(float *p, int left) const {
#pragma unroll
    for (int j = 0; j < W; j += VEC ? 4 : 1) {
      if (col(j) >= left) continue;
      if constexpr (VEC)
        *reinterpret_cast<float4 *>(p + col(j)) = make_float4(a[j], a[j + 1], a[j + 2], a[j + 3]);
      else
        p[col(j)] = a[j];
    }
  }
  KS_DEV void add_part(const float *p, int left) {
#pragma unroll
    for (int j = 0; j < W; j += VEC ? 4 : 1) {
      if (col(j) >= left) continue;
      if constexpr (VEC) {
        const float4 v = __ldcg(reinterpret_cast<const float4 *>(p + col(j)));
        a[j] += v.x;
        a[j + 1] += v.y;
        a[j + 2] += v.z;
        a[j + 3] += v.w;
      } else {
        a[j] += __ldcg(p + col(j));
      }
    }
  }
  KS_DEV void finish(typename O::T *row, int left, float scale, bool accumulate) const {
    constexpr int step = VEC ? W < O::kPer ? W : O::kPer : 1;  // values per 16-byte store
    static_assert(!VEC || step * sizeof(typename O::T) == 16, "whole vectors");
#pragma unroll
    for (int j = 0; j < W; j += step) {
      if (col(j) >= left) continue;
      typename O::T *p = row + col(j);
      alignas(16) typename O::T o[step];
      if (accumulate) {
        if constexpr (VEC)
          *reinterpret_cast<uint4 *>(o) = *reinterpret_cast<const uint4 *>(p);
        else
          o[0] = *p;
      }
#pragma unroll
      for (int k = 0; k < step; ++k) o[k] = O::put(accumulate ? fmaf(a[j + k], scale, O::get(o[k])) : a[j + k] * scale);
      if constexpr (VEC)
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(o);
      else
        *p = o[0];
    }
  }
};

constexpr int64_t kGroup = 32;  // chunks whose partials one CTA adds up

// A token that lies in chunks a to b, of which this CTA has left a partial sum.
// The last of the CTAs that hold a part of it, within each group of 32 chunks,
// adds the group's partials in order; the last group adds the groups'.  So the
// order of the sum is that of the chunks, whoever comes last, and a token that
// fills the whole batch is joined in two short chains.  (A kernel of its own
// for the joins cost 4 us more at 777 x 1001 and 12 at 131072 x 1024.)
struct Part {
  uint32_t key;
  int64_t a, b;
};

// What a CTA (chunk ch, segment seg) waits for in `arrived`, and whether it is last.
template <int DT, int ODT>
KS_DEV bool arrive_group(const GradArgs<DT, ODT> &g, const Part &t, int64_t ch, int64_t seg) {
  const int64_t first = max(t.a, ch / kGroup * kGroup), last = min(t.b, ch / kGroup * kGroup + kGroup - 1);
  uint32_t *counter = g.arrived + (first * 2 + (first == t.a ? 1 : 0)) * g.segs + seg;
  return int64_t(atomicAdd(counter, 1u)) == last - first;
}

template <int DT, int ODT, bool VEC>
KS_DEV void join(const GradArgs<DT, ODT> &g, const Part &t, int64_t ch, int64_t seg) {
  using S = Sum<DT, ODT, VEC>;
  __shared__ bool last_group;
  const int64_t c = seg * S::cols(), a = t.a, b = t.b;
  const int left = int(min(int64_t(S::cols()), g.dim - c));
  auto slot = [&](int64_t chunk) { return g.part + (chunk * 2 + (chunk == a ? 1 : 0)) * g.ld + c; };
  const int64_t first = max(a, ch / kGroup * kGroup), last = min(b, ch / kGroup * kGroup + kGroup - 1);
  S sum;
  sum.clear();
#pragma unroll 8
  for (int64_t j = first; j <= last; ++j) sum.add_part(slot(j), left);
  const int64_t ga = a / kGroup, gb = b / kGroup;
  if (ga != gb) {
    sum.put_part(slot(first), left);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0)
      last_group = int64_t(atomicAdd(g.arrived + g.chunks * 2 * g.segs + a * g.segs + seg, 1u)) == gb - ga;
    __syncthreads();
    if (!last_group) return;
    __threadfence();
    sum.clear();
#pragma unroll 8
    for (int64_t j = ga; j <= gb; ++j) sum.add_part(slot(max(a, j * kGroup)), left);
  }
  sum.finish(g.dtable + int64_t(t.key) * g.dtable_stride + c, left, g.scale, g.accumulate != 0);
}

template <int DT, int ODT, bool VEC>
__global__ void __launch_bounds__(kSegThreads)
    emb_grad_kernel(const __grid_constant__ GradArgs<DT, ODT> g, KsWait wait) {
  using S = Sum<DT, ODT, VEC>;
  using E = Elem<DT>;
  using T = typename E::T;
  extern __shared__ __align__(128) uint8_t ring[];  // [kStages][kRows][pitch]
  __shared__ uint2 kv[kMaxChunk];
  __shared__ uint64_t full[kStages];
  __shared__ int gave_up;
  const int tid = threadIdx.x;
  const int64_t ch = blockIdx.x / g.segs, seg = blockIdx.x - ch * g.segs, c = seg * S::cols();
  const int64_t lo = ch * g.chunk;
  const int held = int(min(int64_t(g.chunk), g.n - lo));
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) ks_mbar_init(full + s, 1);
    gave_up = 0;
    ks_fence_mbar_init();
  }
  ks_pdl_wait();
  for (int i = tid; i < held; i += blockDim.x) kv[i] = __ldcg(g.sorted + lo + i);
  constexpr uint32_t none = 0xffffffffu;  // no token: vocab < 2^31
  const uint32_t prev = lo > 0 ? __ldcg(&g.sorted[lo - 1].x) : none;
  uint32_t next = lo + held < g.n ? __ldcg(&g.sorted[lo + held].x) : none;
  __syncthreads();
  int cnt = held;  // the excluded tokens come last
  if (kv[held - 1].x >= g.vocab) {
    int a = 0, b = held - 1;  // the first of them
    while (a < b) {
      const int m = (a + b) / 2;
      if (kv[m].x >= g.vocab) b = m;
      else a = m + 1;
    }
    cnt = a;
    next = none;
  }
  if (cnt == 0) return;
  const int stages = (cnt + kRows - 1) / kRows;
  const int left = int(min(int64_t(S::cols()), g.dim - c));
  const uint32_t row_bytes = uint32_t(left) * sizeof(T);
  const uint32_t pitch = blockDim.x * 16 + (VEC ? 0 : 16);
  // where a row lies in its 16-byte granules
  const uint32_t first_byte = uint32_t(reinterpret_cast<uintptr_t>(g.dout + c)), step = uint32_t(g.dout_stride * sizeof(T));
  auto offset = [&](uint32_t pos) { return VEC ? 0u : (first_byte + pos * step) & 15u; };
  // rows of stage st into slot s of the ring, one copy per lane; !VEC: the whole
  // granules that hold the row (a granule with a byte of it is mapped memory)
  auto fill = [&](int st, int s) {
    if (st >= stages || tid >= 32) return;
    const int rows = min(kRows, cnt - st * kRows);
    const uint32_t pos = kv[st * kRows + min(tid, rows - 1)].y, off = offset(pos);
    uint32_t bytes = VEC ? row_bytes : (off + row_bytes + 15) & ~15u, all = rows * row_bytes;
    if constexpr (!VEC) all = __reduce_add_sync(0xffffffffu, tid < rows ? bytes : 0u);
    if (tid == 0) ks_mbar_arrive_expect_tx(full + s, all);
    __syncwarp();
    if (tid < rows)
      ks_bulk_load(ring + (s * kRows + tid) * pitch,
                   reinterpret_cast<const char *>(g.dout + int64_t(pos) * g.dout_stride + c) - off, bytes, full + s);
  };
  for (int s = 0; s < kStages; ++s) fill(s, s);
  // chunks that the first and the last token reach to, searched for while the
  // first rows are on their way: 32 chunk edges at a time, by every warp for itself
  int64_t first_chunk = ch, last_chunk = ch;
  bool from_before = prev == kv[0].x;
  if (from_before) {
    for (int64_t j = ch - 1;; j -= 32) {  // lane l: does the token begin before chunk j - l?
      const int64_t at = (j - (tid & 31)) * g.chunk;
      const uint32_t stop = __ballot_sync(0xffffffffu, !(at > 0 && __ldcg(&g.sorted[at - 1].x) == prev));
      if (stop) {
        first_chunk = j - (__ffs(stop) - 1);
        break;
      }
    }
  }
  if (next == kv[cnt - 1].x) {
    for (int64_t j = ch + 1;; j += 32) {  // lane l: does it go on past chunk j + l?
      const int64_t end = (j + (tid & 31) + 1) * g.chunk;
      const uint32_t stop = __ballot_sync(0xffffffffu, !(end < g.n && __ldcg(&g.sorted[end].x) == next));
      if (stop) {
        last_chunk = j + (__ffs(stop) - 1);
        break;
      }
    }
  }
  uint32_t head = none, tail = none;  // tokens of which this CTA leaves a partial sum
  bool head_goes_on = false;
  S sum;
  sum.clear();
  int slot = 0;
  uint32_t phase = 0;
  constexpr int R = kRows / 2;  // rows taken into registers at once
  for (int st = 0; st < stages; ++st) {
    const int i0 = st * kRows, rows = min(kRows, cnt - i0);
    // bit r: the token of row r ends there, or the chunk does
    const int k = min(i0 + (tid & (kRows - 1)), cnt - 1);
    const uint32_t ends = __ballot_sync(0xffffffffu, k == cnt - 1 || kv[k + 1].x != kv[k].x);
    if (!ks_mbar_wait(full + slot, phase, &gave_up, wait)) {
      for (int n = st; n < min(st + kStages, stages); ++n) {  // copies still on their way into this CTA's memory
        ks_mbar_wait(full + slot, phase, nullptr, wait);
        if (++slot == kStages) slot = 0, phase ^= 1;
      }
      return;
    }
#pragma unroll
    for (int r0 = 0; r0 < kRows; r0 += R) {
      if (r0 >= rows) break;
      T x[R][S::W];
#pragma unroll
      for (int r = 0; r < R; ++r) {  // rows past `rows` are read and not used
        const uint8_t *at = ring + (slot * kRows + r0 + r) * pitch;
        if constexpr (VEC) {
          const uint4 v = *reinterpret_cast<const uint4 *>(at + tid * 16);
          *reinterpret_cast<uint4 *>(x[r]) = v;
        } else {
          at += offset(kv[min(i0 + r0 + r, cnt - 1)].y);
#pragma unroll
          for (int j = 0; j < S::W; ++j) x[r][j] = reinterpret_cast<const T *>(at)[S::col(j)];
        }
      }
      if (r0 + R >= rows) {
        __syncthreads();  // the slot has been read
        fill(st + kStages, slot);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r0 + r >= rows) break;
#pragma unroll
        for (int j = 0; j < S::W; ++j) sum.a[j] += E::get(x[r][j]);
        if (!(ends >> (r0 + r) & 1)) continue;
        const int i = i0 + r0 + r;
        const uint32_t key = kv[i].x;
        const bool goes_on = i == cnt - 1 && next == key;
        if (from_before) {
          sum.put_part(g.part + ch * 2 * g.ld + c, left);
          head = key;
          head_goes_on = goes_on;
        } else if (goes_on) {
          sum.put_part(g.part + (ch * 2 + 1) * g.ld + c, left);
          tail = key;
        } else {
          sum.finish(g.dtable + int64_t(key) * g.dtable_stride + c, left, g.scale, g.accumulate != 0);
        }
        sum.clear();
        from_before = false;
      }
    }
    if (++slot == kStages) slot = 0, phase ^= 1;
  }
  if (head == none && tail == none) return;
  // both arrivals at once: a fence and an atomic take about a microsecond each
  __shared__ bool last[2];
  const Part h{head, first_chunk, head_goes_on ? last_chunk : ch}, t{tail, ch, last_chunk};
  __threadfence();
  __syncthreads();
  if (tid == 0) last[0] = head != none && arrive_group(g, h, ch, seg);
  if (tid == blockDim.x - 1) last[1] = tail != none && arrive_group(g, t, ch, seg);
  __syncthreads();
  const bool join_head = last[0], join_tail = last[1];
  __threadfence();
  if (join_head) join<DT, ODT, VEC>(g, h, ch, seg);
  if (join_tail) join<DT, ODT, VEC>(g, t, ch, seg);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int elem_size(int dt) { return dt == KS_F32 ? 4 : 2; }
bool dtype_ok(int dt) { return dt == KS_BF16 || dt == KS_F16 || dt == KS_F32; }
bool aligned16(const void *p, int64_t stride, int64_t dim, int esz) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * esz % 16 == 0 && dim * esz % 16 == 0;
}
bool off(const void *p, int esz) { return reinterpret_cast<uintptr_t>(p) % esz != 0; }

int check_sizes(const char *what, int64_t n, int64_t vocab, int64_t dim, int dt, char *reason, size_t len) {
  if (!dtype_ok(dt)) {
    ks::set_reason(reason, len, "%s: dtype must be bf16, fp16 or fp32", what);
    return KS_ERR_INVALID_CONFIG;
  }
  if (n <= 0 || vocab <= 0 || dim <= 0 || n >= (int64_t(1) << 31) || vocab >= (int64_t(1) << 31) ||
      dim >= (int64_t(1) << 31)) {
    ks::set_reason(reason, len, "%s: tokens, vocab and dim must be positive and below 2^31 (got %lld, %lld, %lld)", what,
                   (long long)n, (long long)vocab, (long long)dim);
    return KS_ERR_INVALID_ARGS;
  }
  return KS_OK;
}

struct GradPlan {
  int chunk;
  bool vec;
  int threads;           // of a CTA of emb_grad_kernel
  int64_t segs;          // segments of columns
  size_t shm;            // its ring
  int64_t chunks, ld;
  int bits, passes;
  int64_t counters;
  size_t o_buf0, o_buf1, o_count, o_part, bytes;
};

int grad_check(const ks_embedding_grad_config &c, const ks_embedding_grad_args &a, char *reason, size_t len) {
  int s = check_sizes("embedding_grad", a.tokens_count, a.vocab, a.dim, a.dtype, reason, len);
  if (s != KS_OK) return s;
  if (c.chunk < 0 || c.chunk > kMaxChunk) {
    ks::set_reason(reason, len, "embedding_grad: chunk must be 0 (chosen) or 1..%d", kMaxChunk);
    return KS_ERR_INVALID_CONFIG;
  }
  if (a.out_dtype != a.dtype && a.out_dtype != KS_F32) {
    ks::set_reason(reason, len, "embedding_grad: the gradient has the type of dout or fp32");
    return KS_ERR_INVALID_CONFIG;
  }
  if (a.dout_stride < a.dim || a.dtable_stride < a.dim) {
    ks::set_reason(reason, len, "embedding_grad: a row stride is smaller than dim");
    return KS_ERR_INVALID_ARGS;
  }
  ks::set_reason(reason, len, "");
  return KS_OK;
}

GradPlan grad_plan(const ks_embedding_grad_config &c, const ks_embedding_grad_args &a) {
  GradPlan p;
  const int64_t n = a.tokens_count;
  const int esz = elem_size(a.dtype);
  p.ld = (a.dim + 63) / 64 * 64;
  int64_t most_chunks = 0, most_counters = 0;  // of both kinds of rows: the workspace's size goes by the sizes alone
  const bool vec = aligned16(a.dout, a.dout_stride, a.dim, esz) &&
                   aligned16(a.dtable, a.dtable_stride, a.dim, elem_size(a.out_dtype)) && a.dim % (16 / esz) == 0;
  for (const bool v : {!vec, vec}) {
    p.vec = v;
    const int64_t want = (a.dim * esz + 15) / 16;  // threads for a whole row
    p.segs = (want + kSegThreads - 1) / kSegThreads;
    p.threads = int(((want + p.segs - 1) / p.segs + 31) / 32 * 32);
    p.segs = (want + p.threads - 1) / p.threads;
    p.shm = size_t(kStages) * kRows * (p.threads * 16 + (v ? 0 : 16));
    // one round of CTAs, as many as the SMs hold; two where chunks stay long
    // (131072 x 1024 fp32: 242 us in one round of 448 positions, 222 in two)
    const int64_t per_sm = std::min<int64_t>({int64_t(227 * 1024 / (p.shm + 9 * 1024 + 512)), 1024 / p.threads, 16});
    int64_t even = (n * p.segs + per_sm * ks::sm_count() - 1) / (per_sm * ks::sm_count());
    if (even >= 256) even = (even + 1) / 2;
    // at least 8 positions; 16 from 4096 on, where a frequent token would lie in many
    // chunks (5178 x 104 into 529 rows: 21.2 us in chunks of 8, 17.7 in 16; 4142 x 408
    // unaligned 28.7 and 23.1; 777 x 1001 13.8 and 15.6)
    const int64_t least = std::min<int64_t>(16, std::max<int64_t>(kRows, n / 256));
    p.chunk = c.chunk ? c.chunk : int(std::min<int64_t>(kMaxChunk, std::max<int64_t>(even, least)));
    p.chunks = (n + p.chunk - 1) / p.chunk;
    p.counters = p.chunks * 3 * p.segs;
    most_chunks = std::max(most_chunks, p.chunks);
    most_counters = std::max(most_counters, p.counters);
  }
  int b = 1;
  while ((int64_t(1) << b) <= a.vocab) ++b;  // keys 0..vocab
  p.passes = (b + 9) / 10;
  p.bits = (b + p.passes - 1) / p.passes;
  if (n <= kRankMax) p.passes = 1;  // one pass of comparisons instead
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += (bytes + 255) / 256 * 256;
    return at;
  };
  p.o_buf0 = take(size_t(n) * 8);
  p.o_buf1 = take(p.passes > 1 ? size_t(n) * 8 : 0);
  p.o_count = take(size_t(most_counters) * 4);
  p.o_part = take(size_t(most_chunks) * 2 * p.ld * 4);
  p.bytes = o;
  return p;
}

int sort_launch(const ks_embedding_grad_args &a, const GradPlan &p, uint2 *buf0, uint2 *buf1, uint32_t *counters,
                const Zeros &zeros, unsigned zero_ctas, cudaStream_t st) {
  const size_t shm = (size_t(kSortWarps) + 2) * (size_t(1) << p.bits) * 4;
  const int s = ks::allow_shared(reinterpret_cast<const void *>(emb_sort_kernel), shm);
  if (s != KS_OK) return s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(kCluster + (zero_ctas + kCluster - 1) / kCluster * kCluster);
  lc.blockDim = dim3(kSortThreads);
  lc.dynamicSmemBytes = shm;
  lc.stream = st;
  lc.attrs = attr;
  lc.numAttrs = 1;
  return ks::map_cuda(cudaLaunchKernelEx(&lc, emb_sort_kernel, a.tokens, a.tokens_count, a.vocab, a.padding_idx, p.passes,
                                         p.bits, buf0, buf1, counters, p.counters, zeros));
}

template <int DT, int ODT, bool VEC>
int grad_launch(const ks_embedding_grad_args &a, const GradPlan &p, cudaStream_t st) {
  using T = typename Elem<DT>::T;
  using O = typename Elem<ODT>::T;
  char *ws = static_cast<char *>(a.workspace);
  const GradArgs<DT, ODT> g = {reinterpret_cast<const uint2 *>(ws + (p.passes & 1 ? p.o_buf0 : p.o_buf1)),
                               a.tokens_count,
                               p.chunk,
                               uint32_t(p.segs),
                               static_cast<const T *>(a.dout),
                               a.dout_stride,
                               static_cast<O *>(a.dtable),
                               a.dtable_stride,
                               a.vocab,
                               a.dim,
                               a.scale,
                               a.accumulate,
                               reinterpret_cast<float *>(ws + p.o_part),
                               p.ld,
                               reinterpret_cast<uint32_t *>(ws + p.o_count),
                               p.chunks};
  if (p.chunks * p.segs > 0x7fffffff) return KS_ERR_INVALID_ARGS;
  auto kern = emb_grad_kernel<DT, ODT, VEC>;
  if (p.shm > 32 * 1024) {
    const int s = ks::allow_shared(reinterpret_cast<const void *>(kern), p.shm);
    if (s != KS_OK) return s;
  }
  return ks::launch_kernel(true, kern, dim3(unsigned(p.chunks * p.segs)), dim3(p.threads), p.shm, st, g, ks::wait_ctx());
}

template <int DT, int ODT>
int grad_launch_vec(const ks_embedding_grad_args &a, const GradPlan &p, cudaStream_t st) {
  return p.vec ? grad_launch<DT, ODT, true>(a, p, st) : grad_launch<DT, ODT, false>(a, p, st);
}

template <int DT>
int lookup_launch(const ks_embedding_args &a, cudaStream_t st) {
  using T = typename Elem<DT>::T;
  const int esz = elem_size(DT);
  const bool vec = aligned16(a.table, a.table_stride, a.dim, esz) && aligned16(a.out, a.out_stride, a.dim, esz);
  const int64_t groups = ((a.dim * esz + 511) / 512 + 3) / 4, total = a.tokens_count * groups;
  if ((total + 7) / 8 > 0x7fffffff) return KS_ERR_INVALID_ARGS;
  const unsigned grid = unsigned((total + 7) / 8);
  auto t = static_cast<const T *>(a.table);
  auto o = static_cast<T *>(a.out);
  return ks::launch_kernel(false, vec ? emb_lookup_kernel<DT, true> : emb_lookup_kernel<DT, false>, dim3(grid), dim3(256), 0, st,
                         a.tokens, a.tokens_count, t, a.table_stride, o, a.out_stride, a.vocab, a.dim, a.scale,
                           int(a.tokens_count * a.dim * esz > 96 << 20));
}

}  // namespace

extern "C" {

int ks_embedding_validate(const ks_embedding_args *a, char *reason, size_t len) {
  if (!a) return KS_ERR_INVALID_ARGS;
  int s = check_sizes("embedding", a->tokens_count, a->vocab, a->dim, a->dtype, reason, len);
  if (s != KS_OK) return s;
  if (a->table_stride < a->dim || a->out_stride < a->dim) {
    ks::set_reason(reason, len, "embedding: a row stride is smaller than dim");
    return KS_ERR_INVALID_ARGS;
  }
  ks::set_reason(reason, len, "");
  return KS_OK;
}

int ks_embedding_launch(const ks_embedding_args *a, void *stream) {
  if (!a || !a->tokens || !a->table || !a->out) return KS_ERR_INVALID_ARGS;
  int s = ks_embedding_validate(a, nullptr, 0);
  if (s != KS_OK) return s;
  const int esz = elem_size(a->dtype);
  if (off(a->tokens, 8) || off(a->table, esz) || off(a->out, esz)) return KS_ERR_INVALID_ARGS;
  const ks::Rows mem[] = {{a->out, a->tokens_count, a->dim * esz, a->out_stride * esz},
                          {a->table, a->vocab, a->dim * esz, a->table_stride * esz},
                          {a->tokens, 1, a->tokens_count * 8, 0}};
  if (ks::outputs_overlap(mem, 1, 3)) return KS_ERR_INVALID_ARGS;
  if ((s = ks::check_arch_sm100()) != KS_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case KS_BF16: return lookup_launch<KS_BF16>(*a, st);
    case KS_F16: return lookup_launch<KS_F16>(*a, st);
    default: return lookup_launch<KS_F32>(*a, st);
  }
}

int ks_embedding_grad_validate(const ks_embedding_grad_config *cfg, const ks_embedding_grad_args *a, char *reason,
                               size_t len) {
  if (!cfg || !a) return KS_ERR_INVALID_ARGS;
  return grad_check(*cfg, *a, reason, len);
}

int ks_embedding_grad_workspace_bytes(const ks_embedding_grad_config *cfg, const ks_embedding_grad_args *a,
                                      size_t *bytes) {
  if (!cfg || !a || !bytes) return KS_ERR_INVALID_ARGS;
  const int s = grad_check(*cfg, *a, nullptr, 0);
  if (s != KS_OK) return s;
  *bytes = grad_plan(*cfg, *a).bytes;
  return KS_OK;
}

int ks_embedding_grad_launch(const ks_embedding_grad_config *cfg, const ks_embedding_grad_args *a, void *stream) {
  if (!cfg || !a || !a->tokens || !a->dout || !a->dtable) return KS_ERR_INVALID_ARGS;
  int s = grad_check(*cfg, *a, nullptr, 0);
  if (s != KS_OK) return s;
  const int esz = elem_size(a->dtype), osz = elem_size(a->out_dtype);
  if (off(a->tokens, 8) || off(a->dout, esz) || off(a->dtable, osz)) return KS_ERR_INVALID_ARGS;
  const GradPlan p = grad_plan(*cfg, *a);
  if (!a->workspace || off(a->workspace, 256) || a->workspace_bytes < p.bytes) return KS_ERR_WORKSPACE;
  // the table's zeros are written before dout is read
  const ks::Rows mem[] = {{a->dtable, a->vocab, a->dim * osz, a->dtable_stride * osz},
                          {a->workspace, 1, int64_t(p.bytes), 0},
                          {a->dout, a->tokens_count, a->dim * esz, a->dout_stride * esz},
                          {a->tokens, 1, a->tokens_count * 8, 0}};
  if (ks::outputs_overlap(mem, 2, 4)) return KS_ERR_INVALID_ARGS;
  if ((s = ks::check_arch_sm100()) != KS_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char *ws = static_cast<char *>(a->workspace);

  Zeros zeros = {};
  unsigned zero_ctas = 0;
  if (!a->accumulate) {
    // a dense table is one long row
    const int64_t rows = a->dtable_stride == a->dim ? 1 : a->vocab;
    const int64_t bytes = (rows == 1 ? a->vocab : 1) * a->dim * osz;
    // two CTAs for every SM, 512 KB each at most: more rounds of CTAs even out
    const int64_t share = std::min<int64_t>(512 * 1024, std::max<int64_t>(16 * 1024, rows * bytes / (2 * ks::sm_count())));
    zeros = Zeros{static_cast<char *>(a->dtable), rows, bytes, a->dtable_stride * osz, (share + 15) / 16 * 16};
    const int64_t ctas = (rows * bytes + zeros.share - 1) / zeros.share;
    if (ctas > (1 << 30)) return KS_ERR_INVALID_ARGS;
    zero_ctas = unsigned(ctas);
  }
  auto counters = reinterpret_cast<uint32_t *>(ws + p.o_count);
  auto buf0 = reinterpret_cast<uint2 *>(ws + p.o_buf0), buf1 = reinterpret_cast<uint2 *>(ws + p.o_buf1);
  if (a->tokens_count <= kRankMax) {
    const unsigned grid = unsigned((a->tokens_count + kRankRows - 1) / kRankRows) + zero_ctas;
    s = ks::launch_kernel(false, a->vocab < (1 << (32 - kRankBits)) ? emb_rank_kernel<true> : emb_rank_kernel<false>, dim3(grid),
                          dim3(kSortThreads), 0, st, a->tokens, int(a->tokens_count), a->vocab, a->padding_idx, buf0,
                          counters, p.counters, zeros);
  } else {
    s = sort_launch(*a, p, buf0, buf1, counters, zeros, zero_ctas, st);
  }
  if (s != KS_OK) return s;
  if (a->dtype == KS_BF16)
    return a->out_dtype == KS_F32 ? grad_launch_vec<KS_BF16, KS_F32>(*a, p, st)
                                  : grad_launch_vec<KS_BF16, KS_BF16>(*a, p, st);
  if (a->dtype == KS_F16)
    return a->out_dtype == KS_F32 ? grad_launch_vec<KS_F16, KS_F32>(*a, p, st)
                                  : grad_launch_vec<KS_F16, KS_F16>(*a, p, st);
  return grad_launch_vec<KS_F32, KS_F32>(*a, p, st);
}

}  // extern "C"
