// grad_clip.cu -- global norm of many gradients, and the gradients scaled to it.
//
//   norm = sqrt(sum over all tensors of g^2),  c = min(1, max_norm / (norm + eps)),  out = c g
//
// Two passes over memory, both over one list of 32 KB chunks that the caller
// plans once for a set of tensors (pointers, lengths, types).  The first is
// persistent and leaves an fp64 partial per CTA.  The second has a CTA per
// chunk (a copy with 32 KB CTAs in launch order moved 6.8 TB/s on B200, the
// same loop in persistent CTAs 5.9) and walks the chunks backwards: what the
// first read last is still in the 126 MB L2.  Its CTAs add the partials up
// themselves, all in the same order, where there are few CTAs; with many, one
// block does it between the passes.  No atomics: the same bits every time.
// Bound by memory: 2^30 values, mostly bf16, 2.6 GB read twice and written once in
// 1166 us (the norm 357, 7.3 TB/s; the scaling 755, 6.8 TB/s); 48 tensors of 600 011
// values in all by the call, 8.7 us.
#include <algorithm>
#include <cuda_fp16.h>

#include "ks_common.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kCtasPerSm = 4;
constexpr int64_t kChunkBytes = 32 * 1024;
constexpr int kMaxCtas = 4096;

struct Chunk {
  const void *grad;
  void *out;
  int32_t count;
  int32_t dtype;
  int64_t pad;
};
static_assert(sizeof(Chunk) == 32, "one 32-byte sector");

template <int DT>
KS_DEV void unpack(uint4 x, float (&v)[8]) {
  if constexpr (DT == KS_F32) {
    v[0] = __uint_as_float(x.x);
    v[1] = __uint_as_float(x.y);
    v[2] = __uint_as_float(x.z);
    v[3] = __uint_as_float(x.w);
    v[4] = v[5] = v[6] = v[7] = 0.f;
  } else {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == KS_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = ks_bf16_lo(w[i]);
        v[2 * i + 1] = ks_bf16_hi(w[i]);
      }
    }
  }
}

template <int DT>
struct Type {
  using T = uint16_t;
  static constexpr int per = 8;
  KS_DEV static float get(T v) {
    if constexpr (DT == KS_F16) return __half2float(__ushort_as_half(v));
    return ks_bf16_to_f32(v);
  }
  KS_DEV static T put(float v) {
    if constexpr (DT == KS_F16) return __half_as_ushort(__float2half_rn(v));
    return ks_f32_to_bf16(v);
  }
};
template <>
struct Type<KS_F32> {
  using T = float;
  static constexpr int per = 4;
  KS_DEV static float get(float v) { return v; }
  KS_DEV static float put(float v) { return v; }
};

// Elements before the first 16-byte boundary of p.
template <int DT>
KS_DEV int head_of(const void *p, int count) {
  const int h = int((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / int(sizeof(typename Type<DT>::T));
  return min(h, count);
}

template <int DT>
KS_DEV float square_chunk(const Chunk &c) {
  using Y = Type<DT>;
  auto g = static_cast<const typename Y::T *>(c.grad);
  const int head = head_of<DT>(g, c.count), vecs = (c.count - head) / Y::per, tail = c.count - head - vecs * Y::per;
  auto v = reinterpret_cast<const uint4 *>(g + head);
  float s[2] = {0.f, 0.f};
#pragma unroll 4
  for (int i = threadIdx.x; i < vecs; i += kThreads) {
    float f[8];
    unpack<DT>(__ldg(v + i), f);
#pragma unroll
    for (int j = 0; j < Y::per; ++j) s[j & 1] = fmaf(f[j], f[j], s[j & 1]);
  }
  if (int(threadIdx.x) < head) {
    const float f = Y::get(g[threadIdx.x]);
    s[0] = fmaf(f, f, s[0]);
  }
  if (int(threadIdx.x) < tail) {
    const float f = Y::get(g[c.count - tail + threadIdx.x]);
    s[1] = fmaf(f, f, s[1]);
  }
  return s[0] + s[1];
}

template <int DT>
KS_DEV void scale_chunk(const Chunk &c, float k) {
  using Y = Type<DT>;
  auto g = static_cast<const typename Y::T *>(c.grad);
  auto o = static_cast<typename Y::T *>(c.out);
  const int head = head_of<DT>(g, c.count), vecs = (c.count - head) / Y::per, tail = c.count - head - vecs * Y::per;
  auto v = reinterpret_cast<const uint4 *>(g + head);
  const bool same = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(o)) & 15) == 0;
  constexpr int U = 4;  // loads in flight: a store to `out` keeps the compiler from moving loads past it
  for (int i0 = threadIdx.x; i0 < vecs; i0 += U * kThreads) {
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * kThreads < vecs) x[u] = v[i0 + u * kThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kThreads;
      if (i >= vecs) break;
      float f[8];
      unpack<DT>(x[u], f);
      alignas(16) typename Y::T y[Y::per];
#pragma unroll
      for (int j = 0; j < Y::per; ++j) y[j] = Y::put(f[j] * k);
      if (same) {
        *reinterpret_cast<uint4 *>(o + head + i * Y::per) = *reinterpret_cast<const uint4 *>(y);
      } else {
#pragma unroll
        for (int j = 0; j < Y::per; ++j) o[head + i * Y::per + j] = y[j];
      }
    }
  }
  if (int(threadIdx.x) < head) o[threadIdx.x] = Y::put(Y::get(g[threadIdx.x]) * k);
  if (int(threadIdx.x) < tail) o[c.count - tail + threadIdx.x] = Y::put(Y::get(g[c.count - tail + threadIdx.x]) * k);
}

KS_DEV double block_sum(double v, double *sh) {
  v = ks_warp_sum_f64(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    double t = threadIdx.x < kThreads / 32 ? sh[threadIdx.x] : 0.0;
    t = ks_warp_sum_f64(t);
    if (threadIdx.x == 0) sh[0] = t;
  }
  __syncthreads();
  return sh[0];
}

// Squares: fp32 within a chunk's share of a thread (at most 34 values: 32 of whole
// vectors, one before and one after them), fp64 across.  Squares in fp32 bound the values:
// above 1.8e19 they are infinite, below 2.6e-23 zero.
__global__ void __launch_bounds__(kThreads) clip_norm_kernel(const Chunk *__restrict__ table, int64_t chunks,
                                                             double *__restrict__ partial) {
  __shared__ double sh[32];
  ks_pdl_release();
  double acc = 0.0;
  for (int64_t i = blockIdx.x; i < chunks; i += gridDim.x) {
    const Chunk c = table[i];
    acc += double(c.dtype == KS_F32   ? square_chunk<KS_F32>(c)
                  : c.dtype == KS_F16 ? square_chunk<KS_F16>(c)
                                      : square_chunk<KS_BF16>(c));
  }
  const double t = block_sum(acc, sh);
  if (threadIdx.x == 0) partial[blockIdx.x] = t;
}

__global__ void __launch_bounds__(kThreads)
    clip_scale_kernel(const Chunk *__restrict__ table, int64_t chunks, const double *__restrict__ partial, int partials,
                      float max_norm, float eps, float *__restrict__ norm_out) {
  __shared__ double sh[32];
  Chunk c = {};
  if (chunks > 0) c = table[chunks - 1 - blockIdx.x];
  ks_pdl_wait();
  double total;
  if (partials == 1) {
    total = __ldcg(partial);
  } else {
    double acc = 0.0;
    for (int i = threadIdx.x; i < partials; i += kThreads) acc += __ldcg(partial + i);
    total = block_sum(acc, sh);
  }
  const float norm = float(sqrt(total));
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  const float r = max_norm / (norm + eps);
  const float k = r > 1.f ? 1.f : r;  // NaN stays NaN
  if (chunks == 0 || (k == 1.f && c.out == c.grad)) return;
  if (c.dtype == KS_F32)
    scale_chunk<KS_F32>(c, k);
  else if (c.dtype == KS_F16)
    scale_chunk<KS_F16>(c, k);
  else
    scale_chunk<KS_BF16>(c, k);
}

__global__ void __launch_bounds__(kThreads) clip_sum_kernel(const double *__restrict__ partial, int partials,
                                                            double *__restrict__ total) {
  __shared__ double sh[32];
  ks_pdl_release();
  ks_pdl_wait();
  double acc = 0.0;
  for (int i = threadIdx.x; i < partials; i += kThreads) acc += __ldcg(partial + i);
  const double t = block_sum(acc, sh);
  if (threadIdx.x == 0) *total = t;
}

}  // namespace

extern "C" {

int ks_grad_clip_plan(const ks_grad_tensor *t, int64_t count, void *table, size_t table_bytes, size_t *bytes,
                      int64_t *chunks) {
  if (count < 0 || (count > 0 && !t) || !bytes || !chunks) return KS_ERR_INVALID_ARGS;
  int64_t n = 0;
  auto *out = static_cast<Chunk *>(table);
  const int64_t room = table ? int64_t(table_bytes / sizeof(Chunk)) : 0;
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].dtype != KS_BF16 && t[i].dtype != KS_F16 && t[i].dtype != KS_F32) return KS_ERR_INVALID_CONFIG;
    const int esz = t[i].dtype == KS_F32 ? 4 : 2;
    if (t[i].numel < 0) return KS_ERR_INVALID_ARGS;
    if (t[i].numel == 0) continue;
    auto g = reinterpret_cast<uintptr_t>(t[i].grad), o = reinterpret_cast<uintptr_t>(t[i].out ? t[i].out : t[i].grad);
    if (!g || g % esz || o % esz) return KS_ERR_INVALID_ARGS;
    const int64_t per = kChunkBytes / esz;
    // the first chunk ends on a 16-byte boundary, so that the others begin on one
    int64_t first = per - int64_t(g & 15) / esz;
    for (int64_t at = 0; at < t[i].numel; ++n) {
      const int64_t c = std::min(at == 0 ? first : per, t[i].numel - at);
      if (table) {
        if (n >= room) return KS_ERR_WORKSPACE;
        out[n] = Chunk{reinterpret_cast<const void *>(g + at * esz), reinterpret_cast<void *>(o + at * esz), int32_t(c),
                       t[i].dtype, 0};
      }
      at += c;
    }
  }
  *bytes = size_t(n) * sizeof(Chunk);
  *chunks = n;
  return KS_OK;
}

int ks_grad_clip_workspace_bytes(int64_t chunks, size_t *bytes) {
  if (!bytes || chunks < 0) return KS_ERR_INVALID_ARGS;
  *bytes = size_t(std::max<int64_t>(1, std::min<int64_t>(chunks, kMaxCtas)) + 1) * sizeof(double);
  return KS_OK;
}

int ks_grad_clip_launch(const ks_grad_clip_args *a, void *stream) {
  if (!a || !a->norm || a->chunks < 0 || (a->chunks > 0 && !a->table)) return KS_ERR_INVALID_ARGS;
  auto odd = [](const void *p, uintptr_t m) { return (reinterpret_cast<uintptr_t>(p) & (m - 1)) != 0; };
  if (!(a->max_norm >= 0.f) || !(a->eps >= 0.f) || odd(a->norm, 4) || odd(a->table, 32)) return KS_ERR_INVALID_ARGS;
  size_t need = 0;
  int s = ks_grad_clip_workspace_bytes(a->chunks, &need);
  if (s != KS_OK) return s;
  if (!a->workspace || a->workspace_bytes < need || odd(a->workspace, 8)) return KS_ERR_WORKSPACE;
  if ((s = ks::check_arch_sm100()) != KS_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t most = std::min<int64_t>(int64_t(ks::sm_count()) * kCtasPerSm, kMaxCtas);
  const int grid = int(std::max<int64_t>(1, std::min(a->chunks, most)));
  if (a->chunks > 0x7fffffff) return KS_ERR_INVALID_ARGS;
  auto table = static_cast<const Chunk *>(a->table);
  auto partial = static_cast<double *>(a->workspace);
  s = ks::launch_kernel(false, clip_norm_kernel, dim3(grid), dim3(kThreads), 0, st, table, a->chunks, partial);
  if (s != KS_OK) return s;
  const double *sums = partial;
  int n = grid;
  if (a->chunks > grid) {  // more CTAs than partials
    s = ks::launch_kernel(true, clip_sum_kernel, dim3(1), dim3(kThreads), 0, st, partial, grid, partial + grid);
    if (s != KS_OK) return s;
    sums = partial + grid;
    n = 1;
  }
  return ks::launch_kernel(true, clip_scale_kernel, dim3(unsigned(std::max<int64_t>(1, a->chunks))), dim3(kThreads), 0, st,
                           table, a->chunks, sums, n, a->max_norm, a->eps, a->norm);
}

}  // extern "C"
