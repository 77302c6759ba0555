// embedding.cu -- token embedding with scaling, and the table's gradient by
// sorted tokens.
//
//   out[i] = scale * table[token[i]]
//   dtable[v] = scale * sum over { i : token[i] = v } of dout[i]
//
// Both are bound by memory.  The gradient sums each table row in a fixed
// order, the order of the positions, whatever the timing: a stable radix sort
// of the tokens brings equal ones together, then each warp walks `chunk`
// consecutive sorted positions over one segment of columns, adding in fp32
// and writing a row when its token ends.  A token whose positions lie in
// several chunks leaves an fp32 partial sum per chunk, and the warp that
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

// W values of a lane, still as stored.  VEC: 16-byte pieces at consecutive
// columns; otherwise columns lane, lane + 32, ...
template <int DT, int W, bool VEC>
struct Raw {
  using T = typename Elem<DT>::T;
  alignas(16) T v[W];
  // p: the row at the segment's first column; c: that column; lanes past `dim` hold zeros
  KS_DEV void load(const T *p, int64_t c, int64_t dim, int lane) {
    if constexpr (VEC) {
      constexpr int per = Elem<DT>::kPer;
#pragma unroll
      for (int j = 0; j < W / per; ++j) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (c + lane * W + j * per < dim) x = __ldg(reinterpret_cast<const uint4 *>(p + lane * W + j * per));
        *reinterpret_cast<uint4 *>(v + j * per) = x;
      }
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = c + lane + j * 32 < dim ? __ldg(p + lane + j * 32) : T(0);
    }
  }
  KS_DEV void store(T *p, int64_t c, int64_t dim, int lane) const {
    if constexpr (VEC) {
      constexpr int per = Elem<DT>::kPer;
#pragma unroll
      for (int j = 0; j < W / per; ++j)
        if (c + lane * W + j * per < dim)
          *reinterpret_cast<uint4 *>(p + lane * W + j * per) = *reinterpret_cast<const uint4 *>(v + j * per);
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (c + lane + j * 32 < dim) p[lane + j * 32] = v[j];
    }
  }
};

// ---------------------------------------------------------------------------
// Forward: a warp per (row, four segments of 512 bytes), their loads in flight.
// A token outside [0, vocab) gives a row of zeros.
// ---------------------------------------------------------------------------
template <int DT, bool VEC>
__global__ void __launch_bounds__(256)
    emb_lookup_kernel(const int64_t *__restrict__ tokens, int64_t n, const typename Elem<DT>::T *__restrict__ table,
                      int64_t table_stride, typename Elem<DT>::T *__restrict__ out, int64_t out_stride, int64_t vocab,
                      int64_t dim, float scale) {
  using E = Elem<DT>;
  constexpr int W = E::kPer, kSeg = 32 * W, U = 4;
  const int lane = threadIdx.x & 31;
  const int64_t segs = (dim + kSeg - 1) / kSeg, groups = (segs + U - 1) / U;
  const int64_t total = n * groups, step = int64_t(gridDim.x) * 8;
  for (int64_t i = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); i < total; i += step) {
    const int64_t row = i / groups, c0 = (i - row * groups) * U * kSeg;
    const int64_t t = __ldg(tokens + row);
    const bool in = t >= 0 && t < vocab;
    Raw<DT, W, VEC> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u].load(table + (in ? t : 0) * table_stride + c0 + u * kSeg, c0 + u * kSeg, in ? dim : 0, lane);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < W; ++j) x[u].v[j] = E::put(E::get(x[u].v[j]) * scale);
      if (!in) {
#pragma unroll
        for (int j = 0; j < W; ++j) x[u].v[j] = 0;  // not 0 * inf
      }
      x[u].store(out + row * out_stride + c0 + u * kSeg, c0 + u * kSeg, dim, lane);
    }
  }
}

// ---------------------------------------------------------------------------
// Stable sort of (token, position), and the zeros of the dense gradient.
//
// One cluster of 8 CTAs sorts: least-significant-digit radix passes of up to
// 10 bits, the digit counts exchanged through distributed shared memory (no
// counters in global memory, no spinning).  Each warp owns a contiguous part
// of the input and ranks 32 elements at a time with a match over the warp, so
// equal digits keep their order.  The other clusters of the grid write the
// zeros meanwhile: the sort is latency-bound and uses no bandwidth to speak of.
// ---------------------------------------------------------------------------
constexpr int kCluster = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;

constexpr int kZeroBytes = 32 * 1024;  // one bulk store of zeros

KS_DEV void bulk_store(void *dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(reinterpret_cast<uint64_t>(dst)),
               "r"(ks_smem_u32(src)), "r"(bytes)
               : "memory");
}

// Zeros over [p, p + bytes) (p and bytes even), the pieces of kZeroBytes dealt
// out over `ctas` CTAs; the even bytes before and after whole 16-byte words by
// the first of them.
KS_DEV void zero_span(char *p, int64_t bytes, const void *zeros, int64_t cta, int64_t ctas) {
  const int64_t head = min(bytes, int64_t((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15));
  const int64_t body = (bytes - head) / 16 * 16, tail = bytes - head - body;
  if (threadIdx.x == 0)
    for (int64_t at = cta * kZeroBytes; at < body; at += ctas * kZeroBytes)
      bulk_store(p + head + at, zeros, uint32_t(min(body - at, int64_t(kZeroBytes))));
  if (cta == 0 && threadIdx.x < head / 2) reinterpret_cast<uint16_t *>(p)[threadIdx.x] = 0;
  if (cta == 0 && threadIdx.x < tail / 2) reinterpret_cast<uint16_t *>(p + bytes - tail)[threadIdx.x] = 0;
}

__global__ void __launch_bounds__(kSortThreads, 1)
    emb_sort_kernel(const int64_t *__restrict__ tokens, int64_t n, int64_t vocab, int64_t padding, int passes, int bits,
                    uint2 *buf0, uint2 *buf1, uint32_t *counters, int64_t counters_n, char *zero, int64_t zero_rows,
                    int64_t zero_bytes, int64_t zero_stride) {
  extern __shared__ __align__(16) uint32_t sh[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) ks_pdl_release();
  if (blockIdx.x >= kCluster) {
    const int64_t ctas = gridDim.x - kCluster, cta = blockIdx.x - kCluster;
    for (int i = tid; i < kZeroBytes / 16; i += kSortThreads) reinterpret_cast<uint4 *>(sh)[i] = make_uint4(0, 0, 0, 0);
    ks_fence_proxy_async();
    __syncthreads();
    if (zero_rows == 1)
      zero_span(zero, zero_bytes, sh, cta, ctas);
    else
      for (int64_t r = cta; r < zero_rows; r += ctas) zero_span(zero + r * zero_stride, zero_bytes, sh, 0, 1);
    if (tid == 0) {
      ks_bulk_commit_group();
      ks_bulk_wait_all();
    }
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
      return make_uint2(t < 0 || t >= vocab || t == padding ? uint32_t(vocab) : uint32_t(t), uint32_t(i));
    };
    for (int i = tid; i < kSortWarps * bins; i += kSortThreads) count[i] = 0;
    __syncthreads();
    uint32_t *mine = count + warp * bins;
    for (int64_t i = lo + lane; i < hi; i += 32) atomicAdd(mine + ((fetch(i).x >> shift) & (bins - 1)), 1u);
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
    for (int64_t i0 = lo; i0 < hi; i0 += 32) {
      const int64_t i = i0 + lane;
      const bool have = i < hi;
      uint2 kv = make_uint2(0, 0);
      if (have) kv = fetch(i);
      const uint32_t d = have ? (kv.x >> shift) & (bins - 1) : uint32_t(bins);
      const uint32_t peers = __match_any_sync(0xffffffffu, d);
      const uint32_t below = __popc(peers & ((1u << lane) - 1u));
      if (have) out[base[d] + mine[d] + below] = kv;
      __syncwarp();
      if (have && below == 0) mine[d] += __popc(peers);
      __syncwarp();
    }
    ks_cluster_sync();  // out is complete; cta_count may be rewritten
  }
}

// ---------------------------------------------------------------------------
// Sums over the sorted positions.  A warp takes `chunk` (at most 32) of them
// and kSeg columns; U rows' loads are in flight.  part: [chunk][2][ld] fp32,
// slot 0 for a token that began in an earlier chunk, slot 1 for one that goes
// on into the next.
// ---------------------------------------------------------------------------
template <int DT, int ODT, bool VEC>
struct Sum {
  using E = Elem<DT>;
  using O = Elem<ODT>;
  static constexpr int W = E::kPer, kSeg = 32 * W;
  float a[W];
  KS_DEV void clear() {
#pragma unroll
    for (int j = 0; j < W; ++j) a[j] = 0.f;
  }
  KS_DEV static int64_t col(int j, int lane) { return VEC ? lane * W + j : lane + j * 32; }
  KS_DEV void put_part(float *p, int64_t c, int64_t dim, int lane) const {
    if constexpr (VEC) {
      if (c + lane * W < dim) {
#pragma unroll
        for (int j = 0; j < W; j += 4)
          *reinterpret_cast<float4 *>(p + c + lane * W + j) = make_float4(a[j], a[j + 1], a[j + 2], a[j + 3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (c + col(j, lane) < dim) p[c + col(j, lane)] = a[j];
    }
  }
  KS_DEV void add_part(const float *p, int64_t c, int64_t dim, int lane) {
    if constexpr (VEC) {
      if (c + lane * W < dim) {
#pragma unroll
        for (int j = 0; j < W; j += 4) {
          const float4 v = __ldcg(reinterpret_cast<const float4 *>(p + c + lane * W + j));
          a[j] += v.x;
          a[j + 1] += v.y;
          a[j + 2] += v.z;
          a[j + 3] += v.w;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (c + col(j, lane) < dim) a[j] += __ldcg(p + c + col(j, lane));
    }
  }
  KS_DEV void finish(typename O::T *row, int64_t c, int64_t dim, int lane, float scale, bool accumulate) {
    Raw<ODT, W, VEC> o;
    if (accumulate) o.load(row + c, c, dim, lane);
#pragma unroll
    for (int j = 0; j < W; ++j) o.v[j] = O::put(accumulate ? fmaf(a[j], scale, O::get(o.v[j])) : a[j] * scale);
    o.store(row + c, c, dim, lane);
  }
};

// What every warp of a launch shares.
template <int DT, int ODT>
struct GradArgs {
  const uint2 *sorted;
  int64_t n;
  int chunk;
  const typename Elem<DT>::T *dout;
  int64_t dout_stride;
  typename Elem<ODT>::T *dtable;
  int64_t dtable_stride, vocab, dim;
  float scale;
  int accumulate;
  float *part;
  int64_t ld;
  uint32_t *arrived;  // [chunk][2][segment] warps of a group that left their partials, [chunk][segment] groups
  int64_t chunks;
};

constexpr int64_t kGroup = 64;  // chunks whose partials one warp adds up

// A token of which this warp (chunk ch, segment seg) has just left a partial
// sum, in slot 1 if it begins here, goes on elsewhere.  The last of the warps
// that hold a part of it, within each group of 64 chunks, adds the group's
// partials in order; the last group adds the groups'.  So the order of the sum
// is that of the chunks, whoever comes last, and a token that fills the whole
// batch (131072 positions: 4096 partials) is joined in two short chains.
template <int DT, int ODT, bool VEC>
KS_DEV void join(const GradArgs<DT, ODT> &g, uint32_t key, int64_t ch, int64_t seg, int64_t segs, bool begins, bool goes_on,
                 int lane) {
  using S = Sum<DT, ODT, VEC>;
  const int64_t c = seg * S::kSeg;
  int64_t a = ch, b = ch;  // the token's first and last chunk
  if (!begins) {
    for (int64_t j = ch - 1;; j -= 32) {  // lane l: does it begin before chunk j - l?
      const int64_t at = (j - lane) * g.chunk;
      const bool on = at > 0 && __ldcg(&g.sorted[at - 1].x) == key;
      const uint32_t stop = __ballot_sync(0xffffffffu, !on);
      if (stop) {
        a = j - (__ffs(stop) - 1);
        break;
      }
    }
  }
  if (goes_on) {
    for (int64_t j = ch + 1;; j += 32) {  // lane l: does it go on past chunk j + l?
      const int64_t end = (j + lane + 1) * g.chunk;
      const bool on = end < g.n && __ldcg(&g.sorted[end].x) == key;
      const uint32_t stop = __ballot_sync(0xffffffffu, !on);
      if (stop) {
        b = j + (__ffs(stop) - 1);
        break;
      }
    }
  }
  auto slot = [&](int64_t chunk) { return g.part + (chunk * 2 + (chunk == a ? 1 : 0)) * g.ld; };
  auto last_of = [&](uint32_t *counter, int64_t expected) {
    __threadfence();
    __syncwarp();
    uint32_t before = 0;
    if (lane == 0) before = atomicAdd(counter, 1u);
    before = __shfl_sync(0xffffffffu, before, 0);
    __threadfence();
    return int64_t(before) == expected - 1;
  };
  const int64_t first = max(a, ch / kGroup * kGroup), last = min(b, ch / kGroup * kGroup + kGroup - 1);
  if (!last_of(g.arrived + (first * 2 + (first == a ? 1 : 0)) * segs + seg, last - first + 1)) return;
  S sum;
  sum.clear();
#pragma unroll 4
  for (int64_t j = first; j <= last; ++j) sum.add_part(slot(j), c, g.dim, lane);
  const int64_t ga = a / kGroup, gb = b / kGroup;
  if (ga != gb) {
    sum.put_part(slot(first), c, g.dim, lane);
    if (!last_of(g.arrived + g.chunks * 2 * segs + a * segs + seg, gb - ga + 1)) return;
    sum.clear();
#pragma unroll 4
    for (int64_t j = ga; j <= gb; ++j) sum.add_part(slot(max(a, j * kGroup)), c, g.dim, lane);
  }
  sum.finish(g.dtable + int64_t(key) * g.dtable_stride, c, g.dim, lane, g.scale, g.accumulate != 0);
}

template <int DT, int ODT, bool VEC>
__global__ void __launch_bounds__(256) emb_grad_kernel(const __grid_constant__ GradArgs<DT, ODT> g) {
  using S = Sum<DT, ODT, VEC>;
  constexpr int U = 8;
  ks_pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t segs = (g.dim + S::kSeg - 1) / S::kSeg;
  const int64_t id = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t ch = id / segs, seg = id - ch * segs, c = seg * S::kSeg;
  const int64_t lo = ch * g.chunk;
  if (lo >= g.n) return;
  const int cnt = int(min(int64_t(g.chunk), g.n - lo));
  uint2 kv = make_uint2(0, 0);
  if (lane < cnt) kv = __ldcg(g.sorted + lo + lane);
  const uint32_t none = 0xffffffffu;  // no token: vocab < 2^31
  const uint32_t prev = lo > 0 ? __ldcg(&g.sorted[lo - 1].x) : none;
  const uint32_t next = lo + cnt < g.n ? __ldcg(&g.sorted[lo + cnt].x) : none;
  bool from_before = prev == __shfl_sync(0xffffffffu, kv.x, 0);
  float *slots = g.part + ch * 2 * g.ld;
  S sum;
  sum.clear();
  for (int i0 = 0; i0 < cnt; i0 += U) {
    Raw<DT, S::W, VEC> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t key = __shfl_sync(0xffffffffu, kv.x, (i0 + u) & 31);
      const int64_t pos = __shfl_sync(0xffffffffu, kv.y, (i0 + u) & 31);
      const bool take = i0 + u < cnt && key < g.vocab;
      x[u].load(g.dout + (take ? pos * g.dout_stride : 0) + c, c, take ? g.dim : 0, lane);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i >= cnt) break;
      const uint32_t key = __shfl_sync(0xffffffffu, kv.x, i);
      if (key >= g.vocab) return;  // the excluded tokens come last
      const uint32_t after = i + 1 < cnt ? __shfl_sync(0xffffffffu, kv.x, (i + 1) & 31) : next;
#pragma unroll
      for (int j = 0; j < S::W; ++j) sum.a[j] += S::E::get(x[u].v[j]);
      if (after != key || i + 1 == cnt) {
        if (from_before || after == key) {
          sum.put_part(from_before ? slots : slots + g.ld, c, g.dim, lane);
          join<DT, ODT, VEC>(g, key, ch, seg, segs, !from_before, after == key, lane);
        } else {
          sum.finish(g.dtable + int64_t(key) * g.dtable_stride, c, g.dim, lane, g.scale, g.accumulate != 0);
        }
        sum.clear();
        from_before = false;
      }
    }
  }
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
  int64_t chunks, ld;
  int bits, passes;
  int64_t counters;
  size_t o_buf0, o_buf1, o_count, o_part, bytes;
};

int grad_check(const ks_embedding_grad_config &c, const ks_embedding_grad_args &a, char *reason, size_t len) {
  int s = check_sizes("embedding_grad", a.tokens_count, a.vocab, a.dim, a.dtype, reason, len);
  if (s != KS_OK) return s;
  if (c.chunk < 0 || c.chunk > 32) {
    ks::set_reason(reason, len, "embedding_grad: chunk must be 0 (chosen) or 1..32");
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
  const int64_t segs = (a.dim * elem_size(a.dtype) + 511) / 512;
  // 32 positions a warp where that leaves 16 warps for every SM, fewer positions otherwise
  p.chunk = c.chunk;
  if (p.chunk == 0) {
    p.chunk = 32;
    while (p.chunk > 4 && (n + p.chunk - 1) / p.chunk * segs < 16LL * ks::sm_count()) p.chunk /= 2;
  }
  p.chunks = (n + p.chunk - 1) / p.chunk;
  p.ld = (a.dim + 63) / 64 * 64;
  int b = 1;
  while ((int64_t(1) << b) <= a.vocab) ++b;  // keys 0..vocab
  p.passes = (b + 9) / 10;
  p.bits = (b + p.passes - 1) / p.passes;
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += (bytes + 255) / 256 * 256;
    return at;
  };
  p.o_buf0 = take(size_t(n) * 8);
  p.o_buf1 = take(p.passes > 1 ? size_t(n) * 8 : 0);
  // (segments of the narrower lane-strided path are as many: 512 bytes or 32 x per elements alike)
  p.counters = p.chunks * 3 * segs;
  p.o_count = take(size_t(p.counters) * 4);
  p.o_part = take(size_t(p.chunks) * 2 * p.ld * 4);
  p.bytes = o;
  return p;
}

template <int DT, int ODT, bool VEC>
int grad_launch(const ks_embedding_grad_args &a, const GradPlan &p, cudaStream_t st) {
  using S = Sum<DT, ODT, VEC>;
  using T = typename Elem<DT>::T;
  using O = typename Elem<ODT>::T;
  char *ws = static_cast<char *>(a.workspace);
  const GradArgs<DT, ODT> g = {reinterpret_cast<const uint2 *>(ws + (p.passes & 1 ? p.o_buf0 : p.o_buf1)),
                               a.tokens_count,
                               p.chunk,
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
  const int64_t segs = (a.dim + S::kSeg - 1) / S::kSeg, blocks = (p.chunks * segs + 7) / 8;
  if (blocks > 0x7fffffff) return KS_ERR_INVALID_ARGS;
  return ks::launch_kernel(true, emb_grad_kernel<DT, ODT, VEC>, dim3(unsigned(blocks)), dim3(256), 0, st, g);
}

template <int DT, int ODT>
int grad_launch_vec(const ks_embedding_grad_args &a, const GradPlan &p, cudaStream_t st) {
  const bool vec = aligned16(a.dout, a.dout_stride, a.dim, elem_size(DT)) &&
                   aligned16(a.dtable, a.dtable_stride, a.dim, elem_size(ODT)) && a.dim % Elem<DT>::kPer == 0;
  return vec ? grad_launch<DT, ODT, true>(a, p, st) : grad_launch<DT, ODT, false>(a, p, st);
}

template <int DT>
int lookup_launch(const ks_embedding_args &a, cudaStream_t st) {
  using T = typename Elem<DT>::T;
  const int esz = elem_size(DT);
  const bool vec = aligned16(a.table, a.table_stride, a.dim, esz) && aligned16(a.out, a.out_stride, a.dim, esz);
  const int64_t groups = ((a.dim * esz + 511) / 512 + 3) / 4, total = a.tokens_count * groups;
  const int grid = int(std::min<int64_t>((total + 7) / 8, int64_t(ks::sm_count()) * 64));
  auto t = static_cast<const T *>(a.table);
  auto o = static_cast<T *>(a.out);
  return ks::launch_kernel(false, vec ? emb_lookup_kernel<DT, true> : emb_lookup_kernel<DT, false>, dim3(grid), dim3(256), 0, st,
                         a.tokens, a.tokens_count, t, a.table_stride, o, a.out_stride, a.vocab, a.dim, a.scale);
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
  if ((s = ks::check_arch_sm100()) != KS_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char *ws = static_cast<char *>(a->workspace);

  int64_t zrows = 0, zbytes = 0;
  unsigned zero_ctas = 0;
  if (!a->accumulate) {
    zrows = a->dtable_stride == a->dim ? 1 : a->vocab;
    zbytes = (zrows == 1 ? a->vocab : 1) * a->dim * osz;
    const int64_t want = (a->vocab * a->dim * osz + 65535) / 65536;  // 64 KB a CTA at least
    zero_ctas = unsigned(std::min<int64_t>(want, ks::sm_count() - kCluster));
    zero_ctas = std::max(1u, zero_ctas / kCluster) * kCluster;
  }
  const size_t shm = std::max<size_t>((size_t(kSortWarps) + 2) * (size_t(1) << p.bits) * 4, kZeroBytes);
  cudaError_t e = cudaFuncSetAttribute(emb_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shm));
  if (e != cudaSuccess) return ks::map_cuda(e);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(kCluster + zero_ctas);
  lc.blockDim = dim3(kSortThreads);
  lc.dynamicSmemBytes = shm;
  lc.stream = st;
  lc.attrs = attr;
  lc.numAttrs = 1;
  e = cudaLaunchKernelEx(&lc, emb_sort_kernel, a->tokens, a->tokens_count, a->vocab, a->padding_idx, p.passes, p.bits,
                         reinterpret_cast<uint2 *>(ws + p.o_buf0), reinterpret_cast<uint2 *>(ws + p.o_buf1),
                         reinterpret_cast<uint32_t *>(ws + p.o_count), p.counters, static_cast<char *>(a->dtable), zrows, zbytes, a->dtable_stride * osz);
  if (e != cudaSuccess) return ks::map_cuda(e);
  if (a->dtype == KS_BF16)
    return a->out_dtype == KS_F32 ? grad_launch_vec<KS_BF16, KS_F32>(*a, p, st)
                                  : grad_launch_vec<KS_BF16, KS_BF16>(*a, p, st);
  if (a->dtype == KS_F16)
    return a->out_dtype == KS_F32 ? grad_launch_vec<KS_F16, KS_F32>(*a, p, st)
                                  : grad_launch_vec<KS_F16, KS_F16>(*a, p, st);
  return grad_launch_vec<KS_F32, KS_F32>(*a, p, st);
}

}  // extern "C"
