// linear_ce.cu -- softmax cross entropy of a linear layer over a large
// vocabulary, with its gradient, on the sm_100a tensor cores.
//
//   l = h w^T;  lse[r] = log sum_v exp l[r,v];  loss[r] = lse[r] - l[r,t[r]]
//   d[r,v] = f[r] (exp(l[r,v] - lse[r]) - [v == t[r]])
//   dh = d w;  dw = d^T h
//
// A loss alone writes nothing of the logits' size.  A gradient needs d as an
// operand, 2 bytes for every (token, column) of a piece of the vocabulary; the
// workspace says how large the pieces are.  Where it holds d whole, as many bytes as
// 16-bit logits (0.27 GB at 4096 x 32768, 2.1 GB at 8192 x 131072, up to 4 GiB by
// default in the torch front end), loss and gradient in one call take the logits once
// and write exponentials and then d there.  Four GEMM-shaped passes share one
// persistent kernel (TMA producer warp, one MMA-issuing thread, eight
// epilogue warps; tcgen05.mma kind::f16, fp32 accumulators in TMEM):
//   STATS  l = h w^T; the epilogue reduces each tile's row to (max, sum of
//          exponentials) and picks the target's logit out of the accumulator;
//   STORE  STATS that also writes exp(l - tile maximum) in 16 bits, for a call
//          that takes loss and gradient together and whose workspace holds 16
//          bits for every (token, column); a memory-bound pass then turns it
//          into d in place, and the logits are taken once: 6 instead of 8
//          tokens x vocab x dim operations;
//   PROB   l = h w^T again for one piece of the vocabulary; the epilogue
//          writes d in 16 bits to the workspace (every other gradient call);
//   GRADS  dh (+)= d w over the piece's columns (split over K when there are
//          few tiles; fp32 slabs, added up in a fixed order) and the piece's
//          rows of dw = d^T h, complete after one pass over the tokens, so each
//          is rounded and written once.  Both products in one launch: their
//          tiles are dealt out so that every SM has the same K-blocks to do,
//          where dh alone (128 tiles of 256 x 256 at 4096 x 2048) leaves 20 of
//          148 SMs idle.
// Operand layouts: h and w K-major in the logits' passes; for dh d K-major and w
// MN-major, for dw d MN-major (M = the vocabulary) and h MN-major -- all straight
// from the row-major tensors, no transpose pass.
//
// Rounding: products and sums are fp32; d is rounded to the inputs' type
// because the tensor cores take 16-bit operands (relative 2^-8 per value in
// bf16, 2^-11 in fp16, the size of the outputs' own rounding); the common factor
// grad_scale / count is left out of d and applied to the fp32 accumulator, so
// that a target's d, near -1, is near a power of two.  fp16 d is stored times
// 1024, so that probabilities down to 6e-8 stay normal numbers.  STORE rounds
// the exponential too, a second rounding of p (not of the target's d, which is
// formed from its logit).  The roundings of the many small values of d average out;
// that of a target's d, the largest of its row, is a factor on the whole term, and
// shows wherever a row of dw or dh is mostly that term, whatever the number of
// tokens.  Relative error in the 2-norm against 64 bits, n x 512 x 8192 and a target
// of its own for each token, beside that of products of a 32-bit d: bf16 0.0017 to
// 0.0019 and 0.0015 to 0.0017 at 65 to 2048 tokens, fp16 0.00025 and 0.00021.  Up to kFew tokens,
// one K-block, d is kept in two 16-bit parts at the cost of one more K-block (dw takes
// the second part, dh the residual of its row's target), and the two errors are equal;
// with more tokens it would cost a second product as large as dw's.  The target's logit is taken a second time, as a
// plain fp32 dot product: the tensor cores' accumulators truncate, which the sum
// over the vocabulary averages out but a loss of one large logit shows (4096 x
// 2048 x 65536: losses off by 2.3e-6 without it, 3.3e-7 with it, against 64 bits).
//
// What bounds it: many tokens, the tensor pipe and then the power cap (4096 x
// 2048 x 32768 bf16, loss and gradients 1341 us: STORE 363, 1.51 PFLOP/s; the
// pass over d 96, memory; GRADS 680, 1.62 PFLOP/s; scores of 4096 x 2048 x 65536
// in 847, beside 846 of the library's plain product under the same cap).  Few
// tokens, the read of w and two launches (scores of 16 x 1024 x 32000: 22.6 us a
// call, 20.7 in a replayed graph; STATS by itself 15 to 16, 66 MB at 4.2 TB/s on 125
// of the SMs, the combine kernel 5).  Taking the logits again instead of keeping
// exponentials: 4096 x 2048 x 32768 with 198 MB of workspace 1.80 ms, with 62 MB 2.17.
//
// Every mbarrier wait is bounded (KsWait), as in matmul.cu.
#include <algorithm>
#include <cuda_fp16.h>

#include "ks_common.cuh"

namespace {

constexpr int kBM = 128;
constexpr int kBK = 64;                        // one 128-byte swizzle row of 16-bit values
constexpr int kUmmaK = 16;
constexpr int kEpiWarps = 8;                    // two per TMEM lane quadrant, each with half of the columns
constexpr int kThreads = 64 + kEpiWarps * 32;  // producer, MMA, epilogue
constexpr uint32_t kABox = kBM * kBK * 2;      // 128 rows x 64 K (or two boxes of 64 K x 64 columns): 16 KB
constexpr uint32_t kBBox = kBK * 64 * 2;       // 64 K-rows x 64 columns: 8 KB
constexpr uint32_t kCStage = 32 * 128;         // an epilogue warp's staging: 32 rows x 64 columns of 16 bits, or x 32 of 32
constexpr int kFew = 64;                        // tokens up to which targets' residuals are carried
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kF16Range = 1024.f;            // factor on fp16 d
constexpr float kF16Exp = 32768.f;             // factor on STORE's fp16 exponentials, which are at most 1

enum Mode { STATS, STORE, PROB, GRADS };

// Scalars between the kernels of one call, in the workspace.
struct CeScalars {
  float fscale;  // on every row's f: the range factor of d
  float escale;  // on the accumulators of GRADS
  unsigned int counter;
  unsigned int foul;  // there is a row in `foul` (below)
};

// One product: output M x N over kb_total K-blocks of 64.
struct CeSide {
  int M, N;
  int kb_total, splits, kb_split;  // K-splits and K-blocks per split (dh)
  int band;                        // raster: N-tiles per band
  int b3d;                         // MN-major B map is (64 columns, K, blocks)
};

struct CeMaps {
  CUtensorMap a[2], b[2], c[2];
  CUtensorMap a_lo;  // dw of few tokens: the second part of d
};

struct CeGemm {
  CeSide side[2];         // GRADS: dh, dw; otherwise the first
  int n1, s1, s2;         // GRADS: the first n1 CTAs share dw tiles [s2, s2 + s1), the others [0, s2)
  int f16;
  // STATS / PROB
  int64_t tokens, vocab;
  int64_t v0;             // first vocabulary column of the piece (PROB)
  const int64_t *targets;
  int64_t ignore;
  float2 *part;           // [tokens][half tiles] (max, sum)
  int parts;              // half tiles
  float *tlogit;          // [rows_p] the target's logit, from the accumulator
  const uint16_t *h, *w;  // for the target's dot product
  int64_t h_stride, w_stride, dim;
  float *tdot;            // [rows_p] that dot product
  int64_t rows_p;
  const float *lse;
  const float *dloss;     // per token, or nullptr
  int few;                // tokens <= kFew
  float *lo;              // [kFew] d of the target less its 16-bit value
  uint16_t *d_lo;         // [tokens][d_ld] what the rounding of d left, rounded
  const uint8_t *foul;    // [rows_p] 1: a row of h without gradient that is not finite
  int64_t d_ld;
  CeScalars *sc;
  int out_f32, accumulate;  // dh goes to fp32 slabs, is added to them
  int release;            // another kernel of the call follows
};

template <int BN, int STAGES, int ACC, int MH>
struct Layout {
  static constexpr uint32_t a_bytes = MH * kABox;
  static constexpr uint32_t b_bytes = kBK * BN * 2;
  static constexpr uint32_t a_off = 0;
  static constexpr uint32_t b_off = a_off + STAGES * a_bytes;
  static constexpr uint32_t c_off = b_off + STAGES * b_bytes;
  static constexpr uint32_t bar_off = c_off + kEpiWarps * kCStage;
  static constexpr uint32_t n_bars = 2 * STAGES + ACC + ACC * MH + 1;
  static constexpr uint32_t misc_off = bar_off + n_bars * 8;
  static constexpr uint32_t bytes = misc_off + 16;
  static constexpr uint32_t request = bytes + 1024;  // slack to align the base to 1024
  static constexpr uint32_t tmem_cols = ACC * BN * MH;
  static_assert(tmem_cols == 128 || tmem_cols == 256 || tmem_cols == 512, "a power of two of TMEM columns");
  static_assert(request <= 227 * 1024, "shared memory");
};

KS_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

KS_DEV uint32_t pack2(float lo, float hi, bool f16) {
  if (f16) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&v);
  }
  return ks_pack_bf16x2(lo, hi);
}

KS_DEV float round16(float v, bool f16) {
  return f16 ? __half2float(__float2half_rn(v)) : ks_bf16_to_f32(ks_f32_to_bf16(v));
}

KS_DEV float value16(uint16_t v, bool f16) {
  return f16 ? __half2float(__ushort_as_half(v)) : ks_bf16_to_f32(v);
}

KS_DEV void tma_reduce_add_2d(const CUtensorMap *m, const void *src, int c0, int c1) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(ks_smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
}

// Work item t of a product -> output tile and K-split; splits outermost, tiles in
// bands of N-tiles, N fastest within a band's rows.
KS_DEV void work_coords(int t, int num_m, int num_n, int band, int &tm, int &tn, int &split) {
  const int tiles = num_m * num_n, size = band * num_m;
  split = t / tiles;
  t -= split * tiles;
  const int b = t / size, first = b * band, bn = min(num_n - first, band), r = t - b * size;
  tn = first + r % bn;
  tm = r / bn;
}

// A CTA's work: items of the first product dealt round robin, then (GRADS) tiles
// of the second, dealt round robin within each of the two classes of CTAs, so
// that the tiles in work at one time lie side by side and share operands in L2
// (runs of neighbouring tiles per CTA read d from DRAM once per column tile:
// 745 instead of 674 us for the two products of 4096 x 2048 x 32768).
template <bool TWO, int TM, int TN>
struct Work {
  int count, first;  // items in all, of the first product
  int second, step;  // tiles of the second: second, second + step, ...
  KS_DEV explicit Work(const CeGemm &p) {
    const CeSide &d = p.side[0];
    const int items = ((d.M + TM - 1) / TM) * ((d.N + TN - 1) / TN) * d.splits;
    const int cta = blockIdx.x, ctas = gridDim.x;
    first = cta < items ? (items - 1 - cta) / ctas + 1 : 0;
    count = first;
    second = step = 0;
    if (TWO) {
      const bool more = cta < p.n1;
      const int j = more ? cta : cta - p.n1, s = more ? p.s1 : p.s2;
      step = more ? p.n1 : ctas - p.n1;
      second = (more ? p.s2 : 0) + j;
      if (j < s) count += (s - 1 - j) / step + 1;
    }
  }
};

struct Item {
  int side, tm, tn, split, kb0, kb1;
};

template <bool TWO, int TM, int TN>
KS_DEV Item item_at(const CeGemm &p, const Work<TWO, TM, TN> &w, int i) {
  Item x;
  x.side = TWO && i >= w.first;
  const CeSide &d = p.side[TWO ? x.side : 0];
  const int t = x.side ? w.second + (i - w.first) * w.step : int(blockIdx.x) + i * int(gridDim.x);
  work_coords(t, (d.M + TM - 1) / TM, (d.N + TN - 1) / TN, d.band, x.tm, x.tn, x.split);
  x.kb0 = x.split * d.kb_split;
  x.kb1 = min(x.kb0 + d.kb_split, d.kb_total);
  return x;
}

KS_DEV float max32(const uint32_t (&r)[32]) {
  float m[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) m[j] = __uint_as_float(r[j]);
#pragma unroll
  for (int j = 4; j < 32; ++j) m[j & 3] = fmaxf(m[j & 3], __uint_as_float(r[j]));
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// tcgen05.wait::ld that the loaded registers depend on, so that their uses
// cannot move ahead of it.
KS_DEV void wait_loaded(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}

// <h[row], w[t]> in fp32 by one warp.
KS_DEV float target_dot(const uint16_t *h, const uint16_t *w, int64_t dim, bool f16, int lane) {
  auto val = [&](uint32_t v, int hi) {
    if (f16) {
      const __half2 x = *reinterpret_cast<const __half2 *>(&v);
      return hi ? __high2float(x) : __low2float(x);
    }
    return hi ? ks_bf16_hi(v) : ks_bf16_lo(v);
  };
  float a0 = 0.f, a1 = 0.f;
  int64_t k = 0;
  if (((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(w)) & 15) == 0) {
#pragma unroll 4
    for (int64_t at = lane * 8; at + 8 <= dim; at += 256) {
      const uint4 x = __ldcg(reinterpret_cast<const uint4 *>(h + at)), y = __ldcg(reinterpret_cast<const uint4 *>(w + at));
      a0 = fmaf(val(x.x, 0), val(y.x, 0), a0);
      a1 = fmaf(val(x.x, 1), val(y.x, 1), a1);
      a0 = fmaf(val(x.y, 0), val(y.y, 0), a0);
      a1 = fmaf(val(x.y, 1), val(y.y, 1), a1);
      a0 = fmaf(val(x.z, 0), val(y.z, 0), a0);
      a1 = fmaf(val(x.z, 1), val(y.z, 1), a1);
      a0 = fmaf(val(x.w, 0), val(y.w, 0), a0);
      a1 = fmaf(val(x.w, 1), val(y.w, 1), a1);
    }
    k = dim / 8 * 8;
  }
  for (k += lane; k < dim; k += 32) a0 = fmaf(val(__ldcg(h + k), 0), val(__ldcg(w + k), 0), a0);
  return ks_warp_sum(a0 + a1);
}

template <int MODE, int BN, int STAGES, int ACC, int MH>
__global__ void __launch_bounds__(kThreads, 1)
    ce_gemm_kernel(const __grid_constant__ CeMaps maps, const __grid_constant__ CeGemm p, KsWait wait) {
  using L = Layout<BN, STAGES, ACC, MH>;
  constexpr bool kGrads = MODE == GRADS;  // two products; B is MN-major, and A in the second
  constexpr int kTM = kBM * MH;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ks_smem_u32(smem_raw);
  uint8_t *smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::bar_off);
  uint64_t *full = bars, *empty = bars + STAGES, *tfull = bars + 2 * STAGES;
  uint64_t *tempty = bars + 2 * STAGES + ACC;  // [acc * MH + half]
  uint64_t *drain = bars + 2 * STAGES + ACC + ACC * MH;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::misc_off);
  volatile int *abort = reinterpret_cast<volatile int *>(smem + L::misc_off + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Work<kGrads, kTM, BN> work(p);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ks_mbar_init(full + s, 1);
      ks_mbar_init(empty + s, 1);
    }
    for (int a = 0; a < ACC; ++a) ks_mbar_init(tfull + a, 1);
    for (int a = 0; a < ACC * MH; ++a) ks_mbar_init(tempty + a, kEpiWarps);
    ks_mbar_init(drain, 1);
    *abort = 0;
    ks_fence_mbar_init();
    for (int d = 0; d < (kGrads ? 2 : 1); ++d) {
      ks_prefetch_tmap(&maps.a[d]);
      ks_prefetch_tmap(&maps.b[d]);
      if (MODE != STATS) ks_prefetch_tmap(&maps.c[d]);
    }
    if (p.release) ks_pdl_release();
  }
  if (warp == 1) {
    ks_tmem_alloc(tmem_slot, L::tmem_cols);
    ks_tmem_relinquish();
  }
  ks_tc_fence_before();
  __syncthreads();
  ks_tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  ks_pdl_wait();
  if ((MODE == STATS || MODE == STORE) && blockIdx.x == 0 && threadIdx.x == 0)
    p.sc->counter = p.sc->foul = 0;  // for the combine kernel that follows

  if (warp == 0 && lane == 0) {
    // ------------------------------------------------------------ producer
    int stage = 0;
    uint32_t phase = 0, armed = 0, armed_parity = 0;
    bool ok = true;
    for (int i = 0; i < work.count && ok; ++i) {
      const Item x = item_at(p, work, i);
      const CUtensorMap *ma = &maps.a[x.side], *mb = &maps.b[x.side];
      const int b3d = p.side[kGrads ? x.side : 0].b3d;
      for (int kb = x.kb0; kb < x.kb1; ++kb) {
        if (!ks_mbar_wait(empty + stage, phase ^ 1u, abort, wait)) {
          ok = false;
          break;
        }
        uint8_t *a_dst = smem + L::a_off + stage * L::a_bytes;
        uint8_t *b_dst = smem + L::b_off + stage * L::b_bytes;
        ks_mbar_arrive_expect_tx(full + stage, L::a_bytes + L::b_bytes);
        const bool second = kGrads && x.side && p.few && kb > 0;  // few tokens: one K-block of d, one of its second part
        if (kGrads && x.side)  // boxes of 64 K-rows x 64 columns, one copy for all of them
          ks_tma_load_3d(a_dst, second ? &maps.a_lo : ma, full + stage, 0, second ? 0 : kb * kBK, x.tm * (kTM / 64));
        else
          ks_tma_load_2d(a_dst, ma, full + stage, kb * kBK, x.tm * kTM);
        if (!kGrads) {
          ks_tma_load_2d(b_dst, mb, full + stage, kb * kBK, x.tn * BN);
        } else if (b3d) {
          ks_tma_load_3d(b_dst, mb, full + stage, 0, second ? 0 : kb * kBK, x.tn * (BN / 64));
        } else {
#pragma unroll
          for (int j = 0; j < BN / 64; ++j)
            ks_tma_load_2d(b_dst + j * kBBox, mb, full + stage, x.tn * BN + j * 64, second ? 0 : kb * kBK);
        }
        armed |= 1u << stage;
        armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // teardown: every load this thread issued must have landed before exit
    for (int s = 0; s < STAGES; ++s)
      if (armed & (1u << s)) ks_mbar_wait(full + s, (armed_parity >> s) & 1u, nullptr, wait);
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t fmt = p.f16 ? (7u << 7) | (7u << 10) : 0;  // f16 operands: format 0
    const bool foul = kGrads && __ldcg(&p.sc->foul) != 0;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto issue = [&](bool a_mn, int st, bool first_kb, uint32_t d_tmem, int h0, int h1) {
      const uint32_t idesc = (a_mn ? ks_idesc_bf16_f32(kBM, BN, true, kGrads) : ks_idesc_bf16_f32(kBM, BN, false, kGrads)) & ~fmt;
      const uint32_t a_addr = ks_smem_u32(smem + L::a_off + st * L::a_bytes);
      const uint32_t b_addr = ks_smem_u32(smem + L::b_off + st * L::b_bytes);
#pragma unroll
      for (int k = 0; k < kBK / kUmmaK; ++k) {
        // K-major: 128-byte rows, 8-row groups 1024 bytes apart, 32 bytes per K=16.
        // MN-major: 64-column boxes kBBox apart (LBO), 8 K-rows 1024 bytes apart (SBO), 2048 bytes per K=16.
        const uint64_t bdesc = kGrads ? ks_umma_desc_sw128(b_addr + k * 2048, kBBox, 1024)
                                      : ks_umma_desc_sw128(b_addr + k * 32, 16, 1024);
#pragma unroll
        for (int h = 0; h < MH; ++h) {
          if (h < h0 || h >= h1) continue;
          const uint64_t adesc = a_mn ? ks_umma_desc_sw128(a_addr + h * kABox + k * 2048, kBBox, 1024)
                                      : ks_umma_desc_sw128(a_addr + h * kABox + k * 32, 16, 1024);
          ks_umma_ss(d_tmem + h * BN, adesc, bdesc, idesc, !first_kb || k != 0);
        }
      }
    };
    // dw = d^T h: d of a token without gradient is 0, and 0 * NaN would reach every
    // row of dw.  Where there are such rows of h, the whole warp zeroes them in the
    // stage before the first MMA reads it (a K-row of a box is 128 bytes, whatever the
    // swizzle does within them; rows past the tokens are zeros already).  Without
    // them one thread is at work, as below.  (4096 x 2048 x 32768 with 5 / 30 % of the
    // rows NaN 1.41 / 1.68 ms a call, 1.34 / 1.28 with finite values in their place.)
    for (int i = 0; foul && i < work.count && ok; ++i) {
      const Item x = item_at(p, work, i);
      const int acc = i % ACC;
      for (int h = 0; h < MH && ok; ++h)
        ok = __all_sync(0xffffffffu, ks_mbar_wait(tempty + acc * MH + h, ((i / ACC) & 1) ^ 1u, abort, wait));
      ks_tc_fence_after();
      // lane l: the marks of rows 2 l and 2 l + 1 of a K-block, fetched one ahead
      auto marks = [&](int kb) {
        return __ldcg(reinterpret_cast<const uint16_t *>(p.foul + int64_t(p.few ? 0 : min(kb, x.kb1 - 1)) * kBK) + lane);
      };
      uint32_t next = x.side ? marks(x.kb0) : 0;
      for (int kb = x.kb0; kb < x.kb1 && ok; ++kb) {
        const uint32_t mark = next;
        if (x.side) next = marks(kb + 1);
        ok = __all_sync(0xffffffffu, ks_mbar_wait(full + stage, phase, abort, wait));
        if (!ok) break;
        if (x.side) {
          uint8_t *b = smem + L::b_off + stage * L::b_bytes;
#pragma unroll
          for (int r = 0; r < 2; ++r)
            for (uint32_t m = __ballot_sync(0xffffffffu, mark >> (8 * r) & 0xff); m; m &= m - 1)
              if (lane < BN / 8)
                *reinterpret_cast<uint4 *>(b + lane / 8 * kBBox + ((__ffs(m) - 1) * 2 + r) * 128 + lane % 8 * 16) =
                    make_uint4(0, 0, 0, 0);
          ks_fence_proxy_async();
        }
        __syncwarp();
        if (lane == 0) {
          ks_tc_fence_after();
          issue(x.side != 0, stage, kb == x.kb0, tmem_base + acc * BN * MH, 0, MH);
          ks_umma_commit(empty + stage);
        }
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok && lane == 0) ks_umma_commit(tfull + acc);
    }
    for (int i = 0; !foul && lane == 0 && i < work.count && ok; ++i) {
      const Item x = item_at(p, work, i);
      const bool a_mn = kGrads && x.side;
      const int acc = i % ACC;
      const uint32_t acc_phase = (i / ACC) & 1;
      // The epilogue frees the accumulator one 128-row half at a time: half
      // 0's MMAs start at once, the other half's are deferred over at most
      // STAGES - 1 K-blocks until it is drained too.
      if (!ks_mbar_wait(tempty + acc * MH, acc_phase ^ 1u, abort, wait)) break;
      ks_tc_fence_after();
      const uint32_t d_tmem = tmem_base + acc * BN * MH;
      bool rest_free = MH == 1;
      int pend = 0;
      for (int kb = x.kb0; kb < x.kb1; ++kb) {
        if (!ks_mbar_wait(full + stage, phase, abort, wait)) {
          ok = false;
          break;
        }
        ks_tc_fence_after();
        issue(a_mn, stage, kb == x.kb0, d_tmem, 0, 1);
        if (!rest_free) {
          if (pend + 1 < STAGES && kb + 1 < x.kb1 &&
              !ks_mbar_test_wait(ks_smem_u32(tempty + acc * MH + 1), acc_phase ^ 1u)) {
            ++pend;
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
            continue;
          }
          for (int h = 1; h < MH && ok; ++h) ok = ks_mbar_wait(tempty + acc * MH + h, acc_phase ^ 1u, abort, wait);
          if (!ok) break;
          ks_tc_fence_after();
          rest_free = true;
          for (int q = pend; q > 0; --q) {
            const int sp = (stage + STAGES - q) % STAGES;
            issue(a_mn, sp, kb - q == x.kb0, d_tmem, 1, MH);
            ks_umma_commit(empty + sp);
          }
          pend = 0;
        }
        issue(a_mn, stage, kb == x.kb0, d_tmem, 1, MH);
        ks_umma_commit(empty + stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) ks_umma_commit(tfull + acc);
    }
    // teardown: all MMAs issued by this thread complete before TMEM is freed
    if (lane == 0) {
      ks_umma_commit(drain);
      ks_mbar_wait(drain, 0, nullptr, wait);
    }
  } else if (warp >= 2) {
    // ------------------------------------------------------------ epilogue
    constexpr int kCols = BN / 2;        // columns of a tile that one warp drains, of each 128-row half
    constexpr int kBlocks = kCols / 32;  // 32-column blocks in them
    const int q = warp & 3;              // TMEM lane quadrant this warp may access
    const int cg = (warp - 2) / 4 * kCols;  // its first column
    uint8_t *stg = smem + L::c_off + (warp - 2) * kCStage;
    const bool f16 = p.f16 != 0;
    float scale = 1.f, fscale = 1.f;
    if (kGrads) scale = __ldcg(&p.sc->escale);
    if (MODE == PROB) fscale = __ldcg(&p.sc->fscale);
    if (MODE == STATS || MODE == STORE) {
      // these warps have nothing else to do until the first tile is complete
      for (int64_t row = int64_t(blockIdx.x) * kEpiWarps + warp - 2; row < p.tokens; row += int64_t(gridDim.x) * kEpiWarps) {
        const int64_t t = p.targets[row];
        if (t == p.ignore || t < 0 || t >= p.vocab) continue;
        const float v = target_dot(p.h + row * p.h_stride, p.w + t * p.w_stride, p.dim, f16, lane);
        if (lane == 0) p.tdot[row] = v;
      }
    }
    for (int i = 0; i < work.count; ++i) {
      const int acc = i % ACC;
      const uint32_t acc_phase = (i / ACC) & 1;
      const Item x = item_at(p, work, i);
      const int tm = x.tm, tn = x.tn;
      const bool wide = kGrads && !x.side && p.out_f32;        // 32-bit blocks, not scaled yet
      const bool add = kGrads && !x.side && p.accumulate;
      const float escale = wide ? 1.f : scale;
      const int out_m = p.side[kGrads ? x.side : 0].M, out_n = p.side[kGrads ? x.side : 0].N;
      const int64_t slab = kGrads && !x.side ? x.split * p.rows_p : 0;  // first row of the split's slab
      // what this lane's rows need, loaded while the MMAs still run
      int tcol[MH];       // target column relative to the tile, or one outside it
      float lse2[MH], f[MH];
      if (MODE == STATS || MODE == STORE || MODE == PROB) {
#pragma unroll
        for (int h = 0; h < MH; ++h) {
          const int64_t row = int64_t(tm) * kTM + h * kBM + q * 32 + lane;
          tcol[h] = -1;
          lse2[h] = 0.f;
          f[h] = 0.f;
          if (row < p.tokens) {
            const int64_t target = p.targets[row];
            const bool valid = target != p.ignore && target >= 0 && target < p.vocab;
            if (valid) {
              const int64_t c = target - p.v0 - int64_t(tn) * BN;
              if (c >= 0 && c < BN) tcol[h] = int(c);
              if (MODE == PROB) f[h] = p.dloss ? p.dloss[row] * fscale : fscale;
            }
            if (MODE == PROB) lse2[h] = __ldcg(p.lse + row) * kLog2e;
          }
        }
      }
      if (!ks_mbar_wait(tfull + acc, acc_phase, abort, wait)) break;
      ks_tc_fence_after();
      const uint32_t t_addr = tmem_base + (uint32_t(q * 32) << 16) + acc * BN * MH + cg;
      const int64_t col0 = p.v0 + int64_t(tn) * BN;  // first vocabulary column of the tile (STATS, STORE, PROB)
      if constexpr (MODE == STATS || MODE == STORE) {
        // A half's columns go into registers at once and the accumulator is free:
        // the next tile's MMAs run while the exponentials are taken (256 x 256 tiles
        // of 4096 x 2048 x 32768: the tensor pipe was 72 % busy when each 32-column
        // block was loaded as it was worked on, and the maximum read them twice).
#pragma unroll 1
        for (int h = 0; h < MH; ++h) {
          uint32_t r[kBlocks][32];
#pragma unroll
          for (int k = 0; k < kBlocks; ++k) ks_tmem_ld32(t_addr + h * BN + k * 32, r[k]);
#pragma unroll
          for (int k = 0; k < kBlocks; ++k) wait_loaded(r[k]);
          ks_tc_fence_before();
          __syncwarp();
          if (lane == 0) ks_mbar_arrive(tempty + acc * MH + h);
          const int64_t row = int64_t(tm) * kTM + h * kBM + q * 32 + lane;
          const int tc = (h == 0 ? tcol[0] : tcol[MH - 1]) - cg;  // the target inside this warp's columns
          if (__any_sync(0xffffffffu, tc >= 0 && tc < kCols)) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < kBlocks; ++k)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (k * 32 + j == tc) v = __uint_as_float(r[k][j]);
            if (tc >= 0 && tc < kCols) p.tlogit[row] = v;
          }
          const int64_t left = p.vocab - (col0 + cg);  // columns inside the vocabulary
          if (left < kCols) {
#pragma unroll
            for (int k = 0; k < kBlocks; ++k)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (k * 32 + j >= left) r[k][j] = __float_as_uint(-INFINITY);
          }
          float m = max32(r[0]);
#pragma unroll
          for (int k = 1; k < kBlocks; ++k) m = fmaxf(m, max32(r[k]));
          // an all -inf row: exponentials against 0 are 0, not NaN
          const float base = m == -INFINITY || m != m ? 0.f : m * kLog2e;
          float a4[4] = {0.f, 0.f, 0.f, 0.f};
          uint8_t *line = stg + lane * 128;
          const int64_t r0 = int64_t(tm) * kTM + h * kBM + q * 32;
#pragma unroll
          for (int k = 0; k < kBlocks; ++k) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float x = ex2(fmaf(__uint_as_float(r[k][j]), kLog2e, -base));
              a4[j & 3] += x;
              if (MODE == STORE) r[k][j] = __float_as_uint(f16 ? x * kF16Exp : x);
            }
            if constexpr (MODE == STORE) {
              // two blocks side by side fill the staging's 128-byte rows (row =
              // lane, 128-byte swizzle: 16-byte chunk v at position v ^ (lane & 7))
              if (k % 2 == 0) {
                if (lane == 0) ks_bulk_wait_read<0>();  // the last store has read the staging
                __syncwarp();
              }
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                uint4 y;
                y.x = pack2(__uint_as_float(r[k][v * 8 + 0]), __uint_as_float(r[k][v * 8 + 1]), f16);
                y.y = pack2(__uint_as_float(r[k][v * 8 + 2]), __uint_as_float(r[k][v * 8 + 3]), f16);
                y.z = pack2(__uint_as_float(r[k][v * 8 + 4]), __uint_as_float(r[k][v * 8 + 5]), f16);
                y.w = pack2(__uint_as_float(r[k][v * 8 + 6]), __uint_as_float(r[k][v * 8 + 7]), f16);
                *reinterpret_cast<uint4 *>(line + (((v + k % 2 * 4) ^ (lane & 7)) * 16)) = y;
              }
              if (k % 2 == 1) {
                const int c0 = tn * BN + cg + (k - 1) * 32;
                ks_fence_proxy_async();
                __syncwarp();
                if (lane == 0 && c0 < out_n && r0 < out_m) {  // blocks past the edge hold nothing
                  ks_tma_store_2d(&maps.c[0], stg, c0, int(r0));
                  ks_bulk_commit_group();
                }
              }
            }
          }
          if (row < p.tokens)
            p.part[row * p.parts + tn * 2 + cg / kCols] = make_float2(m, (a4[0] + a4[1]) + (a4[2] + a4[3]));
        }
        continue;
      }
      // block k: half k / kBlocks, columns cg + k % kBlocks * 32.  `next` is loaded while `r` is worked on.
      auto step = [&](int k, uint32_t (&r)[32], uint32_t (&next)[32]) {
        const int h = k / kBlocks, cb = cg + k % kBlocks * 32;
        wait_loaded(r);
        if (k + 1 < MH * kBlocks) ks_tmem_ld32(t_addr + (k + 1) / kBlocks * BN + (k + 1) % kBlocks * 32, next);
        if ((k + 1) % kBlocks == 0) {  // this warp's part of the half is in registers
          ks_tc_fence_before();
          __syncwarp();
          if (lane == 0) ks_mbar_arrive(tempty + acc * MH + h);
        }
        const int64_t row = int64_t(tm) * kTM + h * kBM + q * 32 + lane;
        const int tc = (h == 0 ? tcol[0] : tcol[MH - 1]) - cb;  // the target inside the block
        const int64_t left = p.vocab - (col0 + cb);             // columns of the block inside the vocabulary
        if constexpr (MODE == PROB) {
          const float fr = h == 0 ? f[0] : f[MH - 1];
          const float l2 = h == 0 ? lse2[0] : lse2[MH - 1];
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(fr * ex2(fmaf(__uint_as_float(r[j]), kLog2e, -l2)));
          if (__any_sync(0xffffffffu, tc >= 0 && tc < 32)) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j == tc) {
                const float d = __uint_as_float(r[j]) - fr;
                if (p.few) p.lo[row] = fr == 0.f ? 0.f : d - round16(d, f16);
                r[j] = __float_as_uint(d);
              }
          }
          if (left < 32 || fr == 0.f) {  // columns past the vocabulary, rows without gradient: zeros, whatever the logits
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j >= left || fr == 0.f) r[j] = 0u;
          }
          if (p.few && row < p.tokens && tn * BN + cb < out_n) {
            // the second part, 64 bytes a lane straight to memory
            uint4 *line = reinterpret_cast<uint4 *>(p.d_lo + row * p.d_ld + tn * BN + cb);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t y[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float a = __uint_as_float(r[v * 8 + e * 2]), b = __uint_as_float(r[v * 8 + e * 2 + 1]);
                y[e] = pack2(a - round16(a, f16), b - round16(b, f16), f16);
              }
              line[v] = make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
        } else if constexpr (kGrads) {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * escale);
        }
        {
          // 16 bits: two blocks side by side fill the staging's 128-byte rows, the
          // second one stores both.  (32-column stores, 64 bytes a row, wrote dw of
          // 16 tokens x 1024 x 32000 at 3 TB/s.)
          const bool second = !wide && (k & 1);
          const int c0 = tn * BN + cb - (second ? 32 : 0);
          const int64_t r0 = int64_t(tm) * kTM + h * kBM + q * 32;
          if (c0 >= out_n || r0 >= out_m) return;  // blocks past the edge hold nothing
          if (!second) {
            if (lane == 0) ks_bulk_wait_read<0>();  // the last store has read the staging
            __syncwarp();
          }
          // row = lane, 128-byte swizzle: 16-byte chunk v at position v ^ (lane & 7)
          uint8_t *line = stg + lane * 128;
          if (wide) {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              *reinterpret_cast<uint4 *>(line + ((v ^ (lane & 7)) * 16)) =
                  make_uint4(r[v * 4], r[v * 4 + 1], r[v * 4 + 2], r[v * 4 + 3]);
          } else {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint4 w;
              w.x = pack2(__uint_as_float(r[v * 8 + 0]), __uint_as_float(r[v * 8 + 1]), f16);
              w.y = pack2(__uint_as_float(r[v * 8 + 2]), __uint_as_float(r[v * 8 + 3]), f16);
              w.z = pack2(__uint_as_float(r[v * 8 + 4]), __uint_as_float(r[v * 8 + 5]), f16);
              w.w = pack2(__uint_as_float(r[v * 8 + 6]), __uint_as_float(r[v * 8 + 7]), f16);
              *reinterpret_cast<uint4 *>(line + (((v + (second ? 4 : 0)) ^ (lane & 7)) * 16)) = w;
            }
            if (!second) return;
          }
          ks_fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            if (add)
              tma_reduce_add_2d(&maps.c[x.side], stg, c0, int(slab + r0));
            else
              ks_tma_store_2d(&maps.c[x.side], stg, c0, int(slab + r0));
            ks_bulk_commit_group();
          }
        }
      };
      uint32_t ra[32], rb[32];
      ks_tmem_ld32(t_addr, ra);
#pragma unroll 1
      for (int k = 0; k < MH * kBlocks; k += 2) {
        step(k, ra, rb);
        step(k + 1, rb, ra);
      }
    }
    if (MODE != STATS && lane == 0) ks_bulk_wait_all();
  }

  ks_tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ks_tc_fence_after();
    ks_tmem_dealloc(tmem_base, L::tmem_cols);
  }
}

// ---------------------------------------------------------------------------
// lse and loss of every row from the tiles' (max, sum); the last block adds up
// the loss over the rows, in a fixed order, and leaves the gradient's scalars.
// ---------------------------------------------------------------------------
constexpr int kCombRows = 8;

struct Combine {
  const float2 *part;  // [tokens][tiles]
  int tiles;
  const float *tlogit, *tdot;
  const int64_t *targets;
  int64_t tokens, vocab, ignore;
  int reduction;
  float grad_scale;
  const float *dloss;
  float range;
  float *loss, *lse;
  double2 *sums;  // per block (loss, tokens that count)
  CeScalars *sc;
  uint8_t *foul;  // [tokens] for the gradient, or nullptr
};

struct RowStats {
  int64_t target;
  bool valid;  // a target in the vocabulary
  float tdot, lse;
  float loss;
  bool counts;
};

// One row by one warp; every lane has the result.
KS_DEV RowStats row_stats(const Combine &a, int64_t row, int lane) {
  RowStats r;
  // the row's own values, loaded beside the partial sums
  r.target = a.targets[row];
  r.tdot = __ldcg(a.tdot + row);
  const float old = __ldcg(a.tlogit + row);
  float m = -INFINITY, s = 0.f;
  auto add = [&](float m2, float s2) {  // (m, s) (+) (m2, s2); a side with no finite maximum adds its sum as it is
    const float mn = fmaxf(m, m2);
    if (mn == -INFINITY) {
      s += s2;  // zeros, or the NaN of a row that has one
    } else {
      s = s * ex2((m - mn) * kLog2e) + s2 * ex2((m2 - mn) * kLog2e);
    }
    m = mn;
  };
#pragma unroll 4
  for (int i = lane; i < a.tiles; i += 32) {
    const float2 v = __ldcg(a.part + row * a.tiles + i);
    add(v.x, v.y);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    add(m2, s2);
  }
  r.valid = r.target != a.ignore && r.target >= 0 && r.target < a.vocab;
  // the target's logit as the dot product, in the sum too
  if (r.valid && isfinite(r.tdot) && isfinite(old)) s += ex2((r.tdot - m) * kLog2e) - ex2((old - m) * kLog2e);
  r.lse = m + logf(s);  // -inf + log 0: a row of -inf logits
  r.counts = r.target != a.ignore;
  r.loss = !r.counts ? 0.f : r.valid ? r.lse - r.tdot : __int_as_float(0x7fc00000);
  return r;
}

// What one thread leaves of a row.  A value of h that is not finite makes every
// logit of its row infinite or NaN, and so the lse: no look at h is needed.
KS_DEV void put_row(const Combine &a, int64_t row, const RowStats &r) {
  a.lse[row] = r.lse;
  if (a.foul) {
    const bool foul = !r.valid && !isfinite(r.lse);
    a.foul[row] = foul;
    if (foul) a.sc->foul = 1;
  }
}

// Block `block` of `blocks` (256 threads) has the sums (l, n), known to thread 0;
// the last to arrive adds them all up.
KS_DEV void reduce_loss(const Combine &a, double l, double n, unsigned block, unsigned blocks) {
  __shared__ bool is_last;
  __shared__ double wl[8], wn[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    a.sums[block] = make_double2(l, n);
    __threadfence();
    is_last = blocks == 1 || atomicAdd(&a.sc->counter, 1u) == blocks - 1;
  }
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  l = n = 0.0;
  for (unsigned j = tid; j < blocks; j += 256) {
    const double2 v = __ldcg(a.sums + j);
    l += v.x;
    n += v.y;
  }
  l = ks_warp_sum_f64(l);
  n = ks_warp_sum_f64(n);
  if (lane == 0) {
    wl[warp] = l;
    wn[warp] = n;
  }
  __syncthreads();
  if (tid == 0) {
    l = n = 0.0;
    for (int j = 0; j < 8; ++j) {
      l += wl[j];
      n += wn[j];
    }
    const double c = a.reduction == KS_CE_MEAN ? (n > 0.0 ? n : 1.0) : 1.0;
    if (a.loss) a.loss[0] = float(l / c);
    a.sc->fscale = a.range;
    a.sc->escale = float(double(a.grad_scale) * (a.dloss ? double(a.dloss[0]) : 1.0) / c / double(a.range));
  }
}

// A warp per row, eight rows per block.  Reads 8 bytes for every half tile of a
// row: 10 us for 4096 rows of 32768 columns, behind its launch and chain of loads.
__global__ void __launch_bounds__(256) ce_combine_kernel(const __grid_constant__ Combine a, int release) {
  __shared__ double shl[kCombRows], shn[kCombRows];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (release) ks_pdl_release();
  ks_pdl_wait();
  const int64_t row = int64_t(blockIdx.x) * kCombRows + warp;
  double l = 0.0, n = 0.0;
  if (row < a.tokens) {
    const RowStats r = row_stats(a, row, lane);
    if (lane == 0) {
      put_row(a, row, r);
      if (a.reduction == KS_CE_NONE && a.loss) a.loss[row] = r.loss;
    }
    l = r.loss;
    n = r.counts;
  }
  if (lane == 0) {
    shl[warp] = l;
    shn[warp] = n;
  }
  if (a.reduction == KS_CE_NONE) return;
  __syncthreads();
  l = n = 0.0;
  if (tid == 0)
    for (int j = 0; j < kCombRows; ++j) {
      l += shl[j];
      n += shn[j];
    }
  reduce_loss(a, l, n, blockIdx.x, gridDim.x);
}

// STORE's exponentials e -> d in place: d = f (e exp(tile maximum - lse) -
// [target]).  A CTA takes 8192 columns of one row, 16 KB, a warp 1024 of them,
// four 16-byte loads a lane in flight.  Reads and writes 2 bytes a value: 537 MB
// for 4096 x 32768 in 91 to 97 us, 5.5 to 5.9 TB/s, the rate of a copy.
// COMBINE: every warp takes its row's lse from the tiles itself, and the combine
// kernel is left out.  That reads a row's (max, sum) pairs once per warp, so it is
// a matter of the bytes read again: up to kCombineBytes, and kCombineRows tokens.
// Whole calls without / with it, us, by those MB: 16 x 1024 x 32000 (1) 67.5 / 65.4,
// 333 x 1000 x 10007 (3) 54.6 / 52.8, 512 x 512 x 10007 (5) 42.8 / 42.8, 128 x 512 x
// 32000 (8) 40.1 / 39.5, 333 x 512 x 32768 (22) 62.7 / 60.8, 512 x 512 x 32768 (34)
// 74.6 / 76.5, 256 x 512 x 65536 (67) 85.6 / 88.2, 128 x 512 x 131072 (134) 114.5 /
// 119.8, 512 x 512 x 131072 (537) 252 / 298; 64 x 256 x 131072 (67) 80.5 / 78.8 is
// the one of these on the wrong side.
constexpr int kCombineRows = 512;
constexpr int64_t kCombineBytes = 24 << 20;
constexpr int kScaleCols = 8192;  // columns of a CTA: eight warps

template <bool COMBINE>
__global__ void __launch_bounds__(256)
    ce_scale_kernel(const __grid_constant__ Combine a, uint16_t *__restrict__ d, int64_t ld, int tile_log2, int f16,
                    float *lo, uint16_t *d_lo) {
  const int lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  ks_pdl_release();
  ks_pdl_wait();
  const int64_t vocab = a.vocab;
  int64_t t;
  bool valid;
  float l2, tdot;
  if (COMBINE) {
    const RowStats r = row_stats(a, row, lane);
    t = r.target;
    valid = r.valid;
    l2 = r.lse * kLog2e;
    tdot = r.tdot;
    if (blockIdx.y == 0) {
      if (threadIdx.x == 0) put_row(a, row, r);
      reduce_loss(a, r.loss, r.counts, unsigned(row), gridDim.x);
    }
  } else {
    t = a.targets[row];
    valid = t != a.ignore && t >= 0 && t < vocab;
    l2 = __ldcg(a.lse + row) * kLog2e;
    tdot = __ldcg(a.tdot + row);
  }
  const float f = valid ? a.range : 0.f, fe = f16 ? f / kF16Exp : f;
  uint16_t *dr = d + row * ld;
  const float dt = valid ? f * ex2(fmaf(tdot, kLog2e, -l2)) - f : 0.f;
  constexpr int step = 256;
  // the last columns first: STORE wrote them last, so they are still in L2, and the
  // first columns, where the products begin, are left there
  const int64_t blocks = (ld + 32 * step - 1) / (32 * step);
  for (int64_t y = blocks - 1 - blockIdx.y; y >= 0; y -= gridDim.y) {
    const int64_t c0 = (y * 8 + (threadIdx.x >> 5)) * (4 * step) + lane * 8;
    uint4 v[4];
    float k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = c0 + j * step;
      k[j] = 0.f;
      if (c < ld && valid) {
        v[j] = __ldcg(reinterpret_cast<const uint4 *>(dr + c));
        if (c < vocab) k[j] = __ldcg(&a.part[row * a.tiles + (c >> tile_log2)].x);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = c0 + j * step;
      if (c >= ld) continue;
      uint4 o = make_uint4(0, 0, 0, 0), rest = o;
      if (valid) {
        const float g = k[j] == -INFINITY ? 0.f : fe * ex2(fmaf(k[j], kLog2e, -l2));  // a tile of -inf logits holds zeros
        const uint32_t x[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (f16) {
            const __half2 z = *reinterpret_cast<const __half2 *>(&x[i]);
            y[2 * i] = __low2float(z) * g;
            y[2 * i + 1] = __high2float(z) * g;
          } else {
            y[2 * i] = ks_bf16_lo(x[i]) * g;
            y[2 * i + 1] = ks_bf16_hi(x[i]) * g;
          }
        }
        const int64_t at = t - c;
        if (at >= 0 && at < 8) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i == at) y[i] = dt;
          if (lo) lo[row] = dt - round16(dt, f16 != 0);
        }
        if (c + 8 > vocab) {  // columns past the vocabulary
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i >= vocab) y[i] = 0.f;
        }
        o = make_uint4(pack2(y[0], y[1], f16 != 0), pack2(y[2], y[3], f16 != 0), pack2(y[4], y[5], f16 != 0),
                       pack2(y[6], y[7], f16 != 0));
        if (d_lo) {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] -= round16(y[i], f16 != 0);
          rest = make_uint4(pack2(y[0], y[1], f16 != 0), pack2(y[2], y[3], f16 != 0), pack2(y[4], y[5], f16 != 0),
                            pack2(y[6], y[7], f16 != 0));
        }
      }
      *reinterpret_cast<uint4 *>(dr + c) = o;
      if (d_lo) *reinterpret_cast<uint4 *>(d_lo + row * ld + c) = rest;
    }
  }
}

// Gradient scalars of a backward call: mean and sum count the tokens; with a
// dloss per token its largest magnitude is taken out of d by a power of two,
// so that fp16 d keeps its range (one block: a few microseconds at 8192 tokens).
// Rows without gradient whose lse is not finite are noted, as put_row does.
__global__ void __launch_bounds__(1024)
    ce_scalars_kernel(const int64_t *__restrict__ targets, int64_t tokens, int64_t vocab, int64_t ignore, int reduction,
                      float grad_scale, const float *__restrict__ dloss, const float *__restrict__ lse, float range,
                      CeScalars *sc, uint8_t *foul) {
  __shared__ float shm[32];
  __shared__ double shn[32];
  ks_pdl_release();
  ks_pdl_wait();
  float mx = 0.f;
  double n = 0.0;
  bool any = false;
  for (int64_t r = threadIdx.x; r < tokens; r += 1024) {
    const int64_t t = targets[r];
    const bool valid = t != ignore && t >= 0 && t < vocab;
    const float g = valid && reduction == KS_CE_NONE && dloss ? dloss[r] : float(valid);
    const bool bad = g == 0.f && !isfinite(lse[r]);
    foul[r] = bad;
    any |= bad;
    if (t != ignore) n += 1.0;
    if (reduction == KS_CE_NONE && dloss) mx = fmaxf(mx, fabsf(g));
  }
  any = __syncthreads_or(any);
  mx = ks_warp_max(mx);
  n = ks_warp_sum_f64(n);
  if ((threadIdx.x & 31) == 0) {
    shm[threadIdx.x >> 5] = mx;
    shn[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  n = 0.0;
  mx = 0.f;
  for (int j = 0; j < 32; ++j) {
    n += shn[j];
    mx = fmaxf(mx, shm[j]);
  }
  double f = range, g = grad_scale;
  if (reduction == KS_CE_NONE) {
    if (dloss && mx > 0.f && mx < INFINITY) {
      int e;
      frexpf(mx, &e);
      f = ldexp(double(range), max(-100, min(100, -e)));
    }
  } else {
    if (dloss) g *= double(dloss[0]);
    if (reduction == KS_CE_MEAN) g /= n > 0.0 ? n : 1.0;
  }
  sc->fscale = float(f);
  sc->escale = float(g / f);
  sc->foul = any;
}

// dh = T(escale * sum of the fp32 slabs), slabs added in order; with few tokens
// the residual of the target's d is added.
__global__ void __launch_bounds__(256)
    ce_dh_finish_kernel(const float *__restrict__ slabs, int count, int64_t slab_elems, int64_t ld, int64_t rows,
                        int64_t cols, const CeScalars *sc, uint16_t *__restrict__ out, int64_t out_stride, int f16,
                        int vec, const float *lo, const int64_t *targets, int64_t vocab, int64_t ignore,
                        const uint16_t *w, int64_t w_stride) {
  ks_pdl_wait();
  const float e = __ldcg(&sc->escale);
  const int64_t cv = (cols + 3) / 4, total = rows * cv;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int64_t r = i / cv, c = (i - r * cv) * 4;
    float4 a = __ldcg(reinterpret_cast<const float4 *>(slabs + r * ld + c));
#pragma unroll 8
    for (int k = 1; k < count; ++k) {
      const float4 b = __ldcg(reinterpret_cast<const float4 *>(slabs + k * slab_elems + r * ld + c));
      a.x += b.x;
      a.y += b.y;
      a.z += b.z;
      a.w += b.w;
    }
    if (lo) {  // few tokens: the target's residual
      const int64_t t = targets[r];
      if (t != ignore && t >= 0 && t < vocab) {
        const float f = __ldcg(lo + r);
        const uint16_t *wr = w + t * w_stride + c;
        float v[4];
        for (int j = 0; j < 4; ++j) v[j] = c + j < cols ? value16(__ldcg(wr + j), f16 != 0) : 0.f;
        a.x = fmaf(f, v[0], a.x);
        a.y = fmaf(f, v[1], a.y);
        a.z = fmaf(f, v[2], a.z);
        a.w = fmaf(f, v[3], a.w);
      }
    }
    const uint32_t y0 = pack2(a.x * e, a.y * e, f16 != 0), y1 = pack2(a.z * e, a.w * e, f16 != 0);
    uint16_t *o = out + r * out_stride + c;
    if (vec && c + 4 <= cols) {
      *reinterpret_cast<uint2 *>(o) = make_uint2(y0, y1);
    } else {
      const uint16_t v[4] = {uint16_t(y0), uint16_t(y0 >> 16), uint16_t(y1), uint16_t(y1 >> 16)};
      for (int j = 0; j < 4 && c + j < cols; ++j) o[j] = v[j];
    }
  }
}

// 2-D copy of 16-bit values between row strides, one side of which TMA cannot
// address (odd strides or unaligned bases).  A warp takes 256 consecutive
// columns of a row at a time, 32 loads of 2 bytes per lane-strided step, so
// that both sides move in full 64-byte pieces whatever their alignment.
__global__ void __launch_bounds__(256)
    ce_copy2d_kernel(const uint16_t *__restrict__ src, int64_t src_stride, uint16_t *__restrict__ dst,
                     int64_t dst_stride, int64_t rows, int64_t cols, int release) {
  if (release) ks_pdl_release();
  ks_pdl_wait();
  const int64_t chunks = (cols + 255) / 256, total = rows * chunks;
  const int lane = threadIdx.x & 31;
  for (int64_t i = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); i < total; i += int64_t(gridDim.x) * 8) {
    const int64_t r = i / chunks, c = (i - r * chunks) * 256;
    const uint16_t *s = src + r * src_stride + c;
    uint16_t *d = dst + r * dst_stride + c;
    const int n = int(min(int64_t(256), cols - c));
    uint16_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * 32 + lane < n) v[j] = __ldcg(s + j * 32 + lane);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * 32 + lane < n) d[j * 32 + lane] = v[j];
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

bool tma_ok(const void *p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % 8 == 0; }

// One GEMM's tile: 256 x 256 (one CTA, two M=128 MMAs per B tile, one
// accumulator drained by halves), 128 x 256 or 128 x 128 (two accumulators).
struct Tile {
  int tm, tn;
  int64_t tiles(int64_t m, int64_t n) const { return ((m + tm - 1) / tm) * ((n + tn - 1) / tn); }
};

// What a tile costs, microseconds, measured under the power cap: one K-block on
// one SM, and what a tile's epilogue adds where the MMAs cannot run beside it.
// The logits' epilogue (exponentials) is the long one: scores of 8192 x 512 x
// 65536 take 529 us in 256 x 256 tiles and 479 in 128 x 256; at dim 1024 the two
// are equal, and from dim 2048 the large tile's smaller operand traffic wins (4096
// x 2048 x 65536: 848 against 890 us, beside 846 of the library's plain product).
struct Cost {
  Tile tile;
  double kb, tail;
};
constexpr Cost kLogitCosts[] = {{{256, 256}, 0.80, 2.0}, {{128, 256}, 0.46, 0.2}, {{128, 128}, 0.36, 0.5}};
constexpr Cost kProductCosts[] = {{{256, 256}, 0.74, 1.5}, {{128, 256}, 0.41, 0.5}, {{128, 128}, 0.29, 0.4}};
constexpr double kSlabBytesPerUs = 5e6;  // an fp32 slab is written once and read once

struct Choice {
  Tile tile;
  int64_t splits, kb_split;
  double item, other;  // GRADS: time of an item of dh, of a tile of dw
};

bool allowed(const Cost &c, const ks_linear_ce_config &cfg) {
  return (!cfg.tile_m || cfg.tile_m == c.tile.tm) && (!cfg.tile_n || cfg.tile_n == c.tile.tn);
}

// Tile of the logits' passes with the least estimated time: rounds of tiles over
// the SMs x K-blocks.
Tile pick_logits(const ks_linear_ce_config &cfg, int64_t m, int64_t n, int64_t kbs, int sms) {
  const Cost *best = nullptr;
  double least = 0;
  for (const Cost &c : kLogitCosts) {
    if (!allowed(c, cfg)) continue;
    const double us = double((c.tile.tiles(m, n) + sms - 1) / sms) * (double(kbs) * c.kb + c.tail);
    if (!best || us < least) {
      least = us;
      best = &c;
    }
  }
  return best->tile;
}

// Tile and K-splits of dh [m, n] over kbs K-blocks beside dw [vocab, n] over
// kb2: all work evenly over the SMs, but no less than the longest item, plus
// the slabs' traffic where K is split (at least 8 K-blocks a split; 4 or 16 make
// no difference).  Loss and gradients, bf16, as chosen and without a split: 333 x
// 1000 x 10007 56 and 81 us, 128 x 4096 x 32000 167 and 231, 64 x 2048 x 32768
// 109 and 201; where there are tiles enough the two are one.
Choice pick_grads(const ks_linear_ce_config &cfg, int64_t m, int64_t n, int64_t kbs, int64_t vocab, int64_t kb2, int sms) {
  Choice best = {};
  double least = 0;
  for (const Cost &c : kProductCosts) {
    if (!allowed(c, cfg)) continue;
    const int64_t tiles = c.tile.tiles(m, n);
    const double other = double(kb2) * c.kb + c.tail, dw = double(c.tile.tiles(vocab, n)) * other;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(2 * sms / tiles, kbs / 8));
    for (int64_t s = 1; s <= most; ++s) {
      const int64_t per = (kbs + s - 1) / s, used = (kbs + per - 1) / per;
      const double item = double(per) * c.kb + c.tail;
      double us = std::max(item, (double(tiles * used) * item + dw) / sms);
      if (used > 1) us += 4 + double(used) * double(m) * double(n) * 8 / kSlabBytesPerUs;
      if (best.splits == 0 || us < least) {
        least = us;
        best = Choice{c.tile, used, per, item, other};
      }
    }
  }
  return best;
}

// GRADS on `ctas` CTAs: those with one item of dh more than the others (the
// first n1) take fewer tiles of dw, s1 in all against s2.
void share(const Choice &c, int64_t items, int64_t tiles, int ctas, CeGemm &g) {
  const int64_t n1 = items % ctas, n2 = ctas - n1;
  const double hi = double(items / ctas + 1) * c.item, lo = double(items / ctas) * c.item;
  // level t: n1 (t - hi)+ + n2 (t - lo)+ = the tiles' time
  const double all = double(tiles) * c.other;
  double t = lo + all / double(n2);
  if (t > hi && n1) t = (all + double(n1) * hi + double(n2) * lo) / double(ctas);
  int64_t s1 = n1 ? int64_t(std::max(0.0, double(n1) * (t - hi) / c.other) + 0.5) : 0;
  s1 = std::min(s1, tiles);
  g.n1 = int(n1);
  g.s1 = int(s1);
  g.s2 = int(tiles - s1);
}

struct Plan {
  Tile g1;               // tiles of the logits' passes
  Choice grads;
  bool pack_h, pack_w, pad_dh, pad_dw;
  int64_t ld;            // row stride of packed h / w / padded outputs
  int64_t rows_p;        // tokens rounded up to 256
  int64_t n_tiles;       // vocabulary half tiles of STATS or STORE
  int64_t piece, pieces; // vocabulary columns per piece, pieces
  bool slabs;            // dh goes through fp32 slabs
  bool store;            // one piece, from STORE's exponentials
  int64_t slab_ld, slab_elems;
  size_t o_d_lo;         // few tokens: the second part of d
  size_t o_foul;         // [rows_p] rows of h without gradient that are not finite
  size_t o_sc, o_sums, o_part, o_tlogit, o_tdot, o_lo, o_lse, o_h, o_w, o_dh, o_slab, o_dw, o_d;
  size_t fixed, bytes;   // bytes: fixed + the piece's d (and padded dw)
};

int check(const ks_linear_ce_config &c, const ks_linear_ce_args &a, char *reason, size_t len) {
  if (!((c.tile_m == 0 && c.tile_n == 0) || (c.tile_m == 128 && (c.tile_n == 128 || c.tile_n == 256)) ||
        (c.tile_m == 256 && c.tile_n == 256))) {
    ks::set_reason(reason, len, "linear_ce: tile_m x tile_n must be 0 x 0 (chosen), 128 x 128, 128 x 256 or 256 x 256");
    return KS_ERR_INVALID_CONFIG;
  }
  if (c.piece < 0 || c.piece % 256 != 0) {
    ks::set_reason(reason, len, "linear_ce: piece must be 0 (chosen) or a multiple of 256");
    return KS_ERR_INVALID_CONFIG;
  }
  if (a.dtype != KS_BF16 && a.dtype != KS_F16) {
    ks::set_reason(reason, len, "linear_ce: dtype must be bf16 or fp16");
    return KS_ERR_INVALID_CONFIG;
  }
  if (a.pass < KS_CE_FORWARD || a.pass > KS_CE_GRAD || a.reduction < KS_CE_NONE || a.reduction > KS_CE_SUM) {
    ks::set_reason(reason, len, "linear_ce: pass or reduction out of range");
    return KS_ERR_INVALID_CONFIG;
  }
  if (a.pass == KS_CE_GRAD && a.reduction == KS_CE_NONE) {
    ks::set_reason(reason, len, "linear_ce: loss and gradient in one call need reduction mean or sum");
    return KS_ERR_INVALID_CONFIG;
  }
  const int64_t lim = (int64_t(1) << 31) - 512;
  if (a.tokens <= 0 || a.dim <= 0 || a.vocab <= 0 || a.tokens > lim || a.dim > lim || a.vocab > lim) {
    ks::set_reason(reason, len, "linear_ce: tokens, dim and vocab must be positive and below 2^31 - 512 (got %lld, %lld, %lld)",
                   (long long)a.tokens, (long long)a.dim, (long long)a.vocab);
    return KS_ERR_INVALID_ARGS;
  }
  if (a.h_stride < a.dim || a.w_stride < a.dim ||
      (a.pass != KS_CE_FORWARD && (a.dh_stride < a.dim || a.dw_stride < a.dim))) {
    ks::set_reason(reason, len, "linear_ce: a row stride is smaller than dim");
    return KS_ERR_INVALID_ARGS;
  }
  ks::set_reason(reason, len, "");
  return KS_OK;
}

// `avail`: workspace bytes; 0 asks for the least plan.
void make_plan(const ks_linear_ce_config &c, const ks_linear_ce_args &a, size_t avail, Plan &p) {
  const int sms = ks::sm_count();
  const bool fwd = a.pass != KS_CE_BACKWARD, bwd = a.pass != KS_CE_FORWARD;
  p.g1 = pick_logits(c, a.tokens, a.vocab, (a.dim + kBK - 1) / kBK, sms);
  p.pack_h = !tma_ok(a.h, a.h_stride);
  p.pack_w = !tma_ok(a.w, a.w_stride);
  p.pad_dh = bwd && !tma_ok(a.dh, a.dh_stride);
  p.pad_dw = bwd && !tma_ok(a.dw, a.dw_stride);
  p.ld = up(a.dim, 8);
  p.rows_p = up(a.tokens, 256);
  const int half = p.g1.tn / 2;               // columns that share a maximum
  p.n_tiles = up(a.vocab, 256) / half;        // of STORE, which runs over whole 256-column blocks
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += (bytes + 1023) / 1024 * 1024;
    return at;
  };
  p.o_sc = take(sizeof(CeScalars));
  p.o_sums = take(fwd ? size_t(std::max<int64_t>((a.tokens + kCombRows - 1) / kCombRows, std::min<int64_t>(a.tokens, kCombineRows))) * 16 : 0);
  p.o_part = take(fwd ? size_t(p.n_tiles) * a.tokens * 8 : 0);
  p.o_tlogit = take(fwd ? size_t(p.rows_p) * 4 : 0);
  p.o_tdot = take(fwd ? size_t(p.rows_p) * 4 : 0);
  p.o_lo = take(bwd ? kFew * 4 : 0);
  p.o_foul = take(bwd ? size_t(p.rows_p) : 0);
  p.o_lse = take(fwd ? size_t(p.rows_p) * 4 : 0);
  p.o_h = take(p.pack_h ? size_t(a.tokens) * p.ld * 2 : 0);
  p.o_w = take(p.pack_w ? size_t(a.vocab) * p.ld * 2 : 0);
  p.slabs = p.store = false;
  p.piece = p.pieces = 0;
  p.o_dh = p.o_slab = p.o_dw = p.o_d = p.o_d_lo = o;
  if (bwd) {
    const int64_t whole = up(a.vocab, 256);
    const bool few = a.tokens <= kFew;
    const size_t per_col = size_t(a.tokens) * (few ? 4 : 2) + (p.pad_dw ? size_t(p.ld) * 2 : 0);
    auto lay = [&](int64_t piece, size_t from) {
      o = from;
      p.piece = piece;
      p.pieces = (a.vocab + piece - 1) / piece;
      const int64_t cols = std::min(piece, a.vocab);
      p.grads = pick_grads(c, a.tokens, a.dim, (cols + kBK - 1) / kBK, cols, (a.tokens + kBK - 1) / kBK, sms);
      p.slabs = p.grads.splits > 1 || p.pieces > 1 || a.tokens <= kFew;
      p.slab_ld = up(a.dim, 32);
      p.slab_elems = p.rows_p * p.slab_ld;
      p.o_dh = take(p.pad_dh && !p.slabs ? size_t(a.tokens) * p.ld * 2 : 0);
      p.o_slab = take(p.slabs ? size_t(p.grads.splits) * p.slab_elems * 4 : 0);
      p.fixed = o;
      p.o_dw = take(p.pad_dw ? size_t(std::min(piece, a.vocab)) * p.ld * 2 : 0);
      p.o_d = take(size_t(a.tokens) * piece * 2);
      p.o_d_lo = take(few ? size_t(a.tokens) * piece * 2 : 0);
      p.bytes = o;
    };
    const size_t from = o;
    int64_t piece = c.piece ? std::min(c.piece, whole) : whole;
    lay(piece, from);
    while (!c.piece && p.bytes > avail && piece > 256) {
      // once it is not whole the slabs come in; from there on bytes fall with the piece
      const int64_t n = avail > p.fixed ? int64_t((avail - p.fixed) / per_col) / 256 * 256 : 256;
      piece = std::max<int64_t>(256, std::min<int64_t>(piece - 256, n));
      lay(piece, from);
    }
    p.store = a.pass == KS_CE_GRAD && p.pieces == 1;
  } else {
    p.fixed = p.bytes = o;
  }
  if (!p.store) p.n_tiles = up(a.vocab, p.g1.tn) / half;
}

template <int MODE, int BN, int STAGES, int ACC, int MH>
int launch(bool next, const CeMaps &maps, CeGemm &g, const Choice *c, cudaStream_t st) {
  using L = Layout<BN, STAGES, ACC, MH>;
  auto kern = ce_gemm_kernel<MODE, BN, STAGES, ACC, MH>;
  const int s = ks::allow_shared(reinterpret_cast<const void *>(kern), L::request);
  if (s != KS_OK) return s;
  const Tile t{kBM * MH, BN};
  const int64_t items = t.tiles(g.side[0].M, g.side[0].N) * g.side[0].splits;
  const int64_t tiles = MODE == GRADS ? t.tiles(g.side[1].M, g.side[1].N) : 0;
  if (items > (int64_t(1) << 30) || tiles > (int64_t(1) << 30)) return KS_ERR_INVALID_ARGS;
  const int ctas = int(std::min<int64_t>(items + tiles, ks::sm_count()));
  if (MODE == GRADS) share(*c, items, tiles, ctas, g);
  return ks::launch_kernel(next, kern, dim3(unsigned(ctas)), dim3(kThreads), L::request, st, maps, g, ks::wait_ctx());
}

template <int MODE>
int launch_tile(bool next, Tile t, const CeMaps &maps, CeGemm &g, const Choice *c, cudaStream_t st) {
  if (t.tm == 256) return launch<MODE, 256, 3, 1, 2>(next, maps, g, c, st);
  return t.tn == 256 ? launch<MODE, 256, 4, 2, 1>(next, maps, g, c, st)
                     : launch<MODE, 128, 5, 2, 1>(next, maps, g, c, st);
}

CUtensorMapDataType tm_type(int dtype) {
  return dtype == KS_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// K-major operand [rows, cols]: boxes of 64 columns (K) x `box` rows.
int map_k(CUtensorMap *m, int dtype, const void *p, int64_t rows, int64_t cols, int64_t stride, int box) {
  return ks::encode_tmap_2d(m, tm_type(dtype), p, uint64_t(cols), uint64_t(rows), uint64_t(stride) * 2, kBK, box,
                            CU_TENSOR_MAP_SWIZZLE_128B);
}

// MN-major operand [K rows, cols]: boxes of 64 columns x 64 K-rows; all of a
// tile's boxes in one copy when the columns are whole blocks of 64.
int map_mn(CUtensorMap *m, int dtype, const void *p, int64_t rows, int64_t cols, int64_t stride, int tile, int *b3d) {
  if (cols % 64 == 0 && ks::encode_tmap_3d(m, tm_type(dtype), p, 64, uint64_t(rows), uint64_t(cols / 64),
                                           uint64_t(stride) * 2, 128, 64, kBK, tile / 64,
                                           CU_TENSOR_MAP_SWIZZLE_128B) == KS_OK) {
    *b3d = 1;
    return KS_OK;
  }
  *b3d = 0;
  return ks::encode_tmap_2d(m, tm_type(dtype), p, uint64_t(cols), uint64_t(rows), uint64_t(stride) * 2, 64, kBK,
                            CU_TENSOR_MAP_SWIZZLE_128B);
}

// Output [rows, cols] of 16-bit values: blocks of 32 rows x 64 columns, 128-byte swizzle.
int map_out(CUtensorMap *m, int dtype, void *p, int64_t rows, int64_t cols, int64_t stride) {
  return ks::encode_tmap_2d(m, tm_type(dtype), p, uint64_t(cols), uint64_t(rows), uint64_t(stride) * 2, 64, 32,
                            CU_TENSOR_MAP_SWIZZLE_128B);
}

int copy2d(bool next, bool release, const void *src, int64_t ss, void *dst, int64_t ds, int64_t rows, int64_t cols,
           cudaStream_t st) {
  const int64_t items = rows * ((cols + 255) / 256);
  const int grid = int(std::min<int64_t>((items + 7) / 8, int64_t(ks::sm_count()) * 8));
  return ks::launch_kernel(next, ce_copy2d_kernel, dim3(grid), dim3(256), 0, st, static_cast<const uint16_t *>(src), ss,
                           static_cast<uint16_t *>(dst), ds, rows, cols, int(release));
}

int run(const ks_linear_ce_args &a, const Plan &p, cudaStream_t st) {
  char *ws = static_cast<char *>(a.workspace);
  const bool fwd = a.pass != KS_CE_BACKWARD, bwd = a.pass != KS_CE_FORWARD;
  auto sc = reinterpret_cast<CeScalars *>(ws + p.o_sc);
  const float range = a.dtype == KS_F16 ? kF16Range : 1.f;
  int s;
  bool next = false;  // a kernel of this call has been launched
  const void *h = a.h, *w = a.w;
  int64_t hs = a.h_stride, wst = a.w_stride;
  if (p.pack_h) {
    if ((s = copy2d(next, true, a.h, a.h_stride, ws + p.o_h, p.ld, a.tokens, a.dim, st)) != KS_OK) return s;
    next = true;
    h = ws + p.o_h;
    hs = p.ld;
  }
  if (p.pack_w) {
    if ((s = copy2d(next, true, a.w, a.w_stride, ws + p.o_w, p.ld, a.vocab, a.dim, st)) != KS_OK) return s;
    next = true;
    w = ws + p.o_w;
    wst = p.ld;
  }
  CeGemm g = {};
  g.f16 = a.dtype == KS_F16;
  g.tokens = a.tokens;
  g.vocab = a.vocab;
  g.targets = a.targets;
  g.ignore = a.ignore_index;
  g.rows_p = p.rows_p;
  g.sc = sc;
  g.release = 1;
  g.h = static_cast<const uint16_t *>(h);
  g.w = static_cast<const uint16_t *>(w);
  g.h_stride = hs;
  g.w_stride = wst;
  g.dim = a.dim;
  g.few = a.tokens <= kFew;
  g.lo = reinterpret_cast<float *>(ws + p.o_lo);
  auto foul = bwd ? reinterpret_cast<uint8_t *>(ws + p.o_foul) : nullptr;
  g.foul = foul;
  const int kd = int((a.dim + kBK - 1) / kBK);
  CeMaps maps = {};
  if ((s = map_k(&maps.a[0], a.dtype, h, a.tokens, a.dim, hs, p.g1.tm)) != KS_OK) return s;
  float *lse = a.lse;
  Combine comb = {};
  const int64_t again = (up(a.vocab, 256) + kScaleCols - 1) / kScaleCols * 8 * a.tokens * p.n_tiles * sizeof(float2);
  const bool combine_in_scale = p.store && a.tokens <= kCombineRows && again <= kCombineBytes;
  if (fwd) {
    if (!lse) lse = reinterpret_cast<float *>(ws + p.o_lse);
    if ((s = map_k(&maps.b[0], a.dtype, w, a.vocab, a.dim, wst, p.g1.tn)) != KS_OK) return s;
    g.part = reinterpret_cast<float2 *>(ws + p.o_part);
    g.parts = int(p.n_tiles);
    g.tlogit = reinterpret_cast<float *>(ws + p.o_tlogit);
    g.tdot = reinterpret_cast<float *>(ws + p.o_tdot);
    // STORE: [tokens, whole tiles], the columns past the vocabulary are -inf logits, zeros
    const int64_t wide = up(a.vocab, 256);
    g.side[0] = CeSide{int(a.tokens), int(p.store ? wide : a.vocab), kd, 1, kd, 8, 0};
    if (p.store) {
      if ((s = map_out(&maps.c[0], a.dtype, ws + p.o_d, a.tokens, wide, wide)) != KS_OK) return s;
      s = launch_tile<STORE>(next, p.g1, maps, g, nullptr, st);
    } else {
      s = launch_tile<STATS>(next, p.g1, maps, g, nullptr, st);
    }
    if (s != KS_OK) return s;
    comb = Combine{g.part, g.parts, g.tlogit, g.tdot, a.targets, a.tokens, a.vocab, a.ignore_index, a.reduction,
                   a.grad_scale, a.dloss, range, a.loss, lse, reinterpret_cast<double2 *>(ws + p.o_sums), sc, foul};
    if (!combine_in_scale) {
      const unsigned blocks = unsigned((a.tokens + kCombRows - 1) / kCombRows);
      s = ks::launch_kernel(true, ce_combine_kernel, dim3(blocks), dim3(256), 0, st, comb, int(bwd));
      if (s != KS_OK) return s;
    }
  }
  if (!bwd) return KS_OK;
  if (!fwd) {
    s = ks::launch_kernel(next, ce_scalars_kernel, dim3(1), dim3(1024), 0, st, a.targets, a.tokens, a.vocab, a.ignore_index,
                        a.reduction, a.grad_scale, a.dloss, lse, range, sc, foul);
    if (s != KS_OK) return s;
  }
  char *d = ws + p.o_d;
  float *slabs = reinterpret_cast<float *>(ws + p.o_slab);
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, vp = std::min(p.piece, a.vocab - v0), vpad = up(vp, 256);
    const char *wp = static_cast<const char *>(w) + v0 * wst * 2;
    g.v0 = v0;
    g.d_lo = reinterpret_cast<uint16_t *>(ws + p.o_d_lo);
    g.d_ld = vpad;
    // d of the piece: [tokens, vpad], columns past the vocabulary zero
    if (p.store) {
      const unsigned cols = unsigned(std::min<int64_t>((vpad + kScaleCols - 1) / kScaleCols, 65535));
      s = ks::launch_kernel(true, combine_in_scale ? ce_scale_kernel<true> : ce_scale_kernel<false>,
                            dim3(unsigned(a.tokens), cols), dim3(256), 0, st, comb, reinterpret_cast<uint16_t *>(d), vpad,
                            p.g1.tn == 256 ? 7 : 6, g.f16, g.few ? g.lo : nullptr, g.few ? g.d_lo : nullptr);
    } else {
      g.side[0] = CeSide{int(a.tokens), int(vpad), kd, 1, kd, 8, 0};
      g.lse = lse;
      g.dloss = a.reduction == KS_CE_NONE ? a.dloss : nullptr;
      if ((s = map_k(&maps.b[0], a.dtype, wp, vp, a.dim, wst, p.g1.tn)) != KS_OK) return s;
      if ((s = map_out(&maps.c[0], a.dtype, d, a.tokens, vpad, vpad)) != KS_OK) return s;
      s = launch_tile<PROB>(true, p.g1, maps, g, nullptr, st);
    }
    if (s != KS_OK) return s;
    // dh (+)= d w, and the piece's rows of dw = d^T h
    const Tile t = p.grads.tile;
    CeMaps mg = {};
    const int kv = int((vp + kBK - 1) / kBK), kt = int((a.tokens + kBK - 1) / kBK), per = int(p.grads.kb_split);
    g.side[0] = CeSide{int(a.tokens), int(a.dim), kv, (kv + per - 1) / per, per, 16, 0};
    // dw: the column tiles of a block of rows side by side, so that whole rows are written at about one time
    const int kd2 = g.few ? 2 : kt;  // few tokens: d and its second part, a K-block each
    g.side[1] = CeSide{int(vp), int(a.dim), kd2, 1, kd2, 16, 0};
    static_assert(kFew <= kBK, "few tokens are one K-block");
    if ((s = map_k(&mg.a[0], a.dtype, d, a.tokens, vp, vpad, t.tm)) != KS_OK) return s;
    if ((s = map_mn(&mg.b[0], a.dtype, wp, vp, a.dim, wst, t.tn, &g.side[0].b3d)) != KS_OK) return s;
    if (p.slabs)
      s = ks::encode_tmap_2d(&mg.c[0], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, slabs, uint64_t(p.slab_ld),
                             uint64_t(p.grads.splits) * p.rows_p, uint64_t(p.slab_ld) * 4, 32, 32,
                             CU_TENSOR_MAP_SWIZZLE_128B);
    else
      s = map_out(&mg.c[0], a.dtype, p.pad_dh ? ws + p.o_dh : a.dh, a.tokens, a.dim, p.pad_dh ? p.ld : a.dh_stride);
    if (s != KS_OK) return s;
    int a3d = 0;
    if ((s = map_mn(&mg.a[1], a.dtype, d, a.tokens, vpad, vpad, t.tm, &a3d)) != KS_OK) return s;
    if (!a3d) return KS_ERR_OTHER;
    if (g.few && (s = map_mn(&mg.a_lo, a.dtype, g.d_lo, a.tokens, vpad, vpad, t.tm, &a3d)) != KS_OK) return s;
    if ((s = map_mn(&mg.b[1], a.dtype, h, a.tokens, a.dim, hs, t.tn, &g.side[1].b3d)) != KS_OK) return s;
    char *dwp = static_cast<char *>(a.dw) + v0 * a.dw_stride * 2;
    if ((s = map_out(&mg.c[1], a.dtype, p.pad_dw ? ws + p.o_dw : dwp, vp, a.dim, p.pad_dw ? p.ld : a.dw_stride)) != KS_OK)
      return s;
    g.out_f32 = p.slabs;
    g.accumulate = p.slabs && i > 0;
    const bool last = i + 1 == p.pieces && !p.slabs && !p.pad_dh;
    g.release = !last || p.pad_dw;
    if ((s = launch_tile<GRADS>(true, t, mg, g, &p.grads, st)) != KS_OK) return s;
    g.release = 1;
    if (p.pad_dw && (s = copy2d(true, !last, ws + p.o_dw, p.ld, dwp, a.dw_stride, vp, a.dim, st)) != KS_OK) return s;
  }
  if (p.slabs) {
    const int64_t items = a.tokens * ((a.dim + 3) / 4);
    const int grid = int(std::min<int64_t>((items + 255) / 256, int64_t(ks::sm_count()) * 8));
    const int vec = reinterpret_cast<uintptr_t>(a.dh) % 8 == 0 && a.dh_stride % 4 == 0;
    return ks::launch_kernel(true, ce_dh_finish_kernel, dim3(grid), dim3(256), 0, st, slabs, int(p.grads.splits), p.slab_elems, p.slab_ld,
                           a.tokens, a.dim, sc, static_cast<uint16_t *>(a.dh), a.dh_stride, int(a.dtype == KS_F16), vec, g.few ? g.lo : nullptr,
                             a.targets, a.vocab, a.ignore_index, static_cast<const uint16_t *>(w), wst);
  }
  if (p.pad_dh) return copy2d(true, false, ws + p.o_dh, p.ld, a.dh, a.dh_stride, a.tokens, a.dim, st);
  return KS_OK;
}

}  // namespace

extern "C" {

int ks_linear_ce_validate(const ks_linear_ce_config *cfg, const ks_linear_ce_args *a, char *reason, size_t len) {
  if (!cfg || !a) return KS_ERR_INVALID_ARGS;
  return check(*cfg, *a, reason, len);
}

int ks_linear_ce_workspace_bytes(const ks_linear_ce_config *cfg, const ks_linear_ce_args *a, size_t limit,
                                 size_t *least, size_t *bytes) {
  if (!cfg || !a || !least || !bytes) return KS_ERR_INVALID_ARGS;
  const int s = check(*cfg, *a, nullptr, 0);
  if (s != KS_OK) return s;
  Plan p;
  make_plan(*cfg, *a, 0, p);
  *least = p.bytes;
  // the whole vocabulary in one piece can take less than its pieces, which need
  // fp32 slabs of dh (8192 x 4096 x 512: 8.8 against 139 MB)
  make_plan(*cfg, *a, size_t(-1), p);
  *least = std::min(*least, p.bytes);
  make_plan(*cfg, *a, std::max(limit, *least), p);
  *bytes = p.bytes;
  return KS_OK;
}

int ks_linear_ce_launch(const ks_linear_ce_config *cfg, const ks_linear_ce_args *a, void *stream) {
  if (!cfg || !a || !a->h || !a->w || !a->targets) return KS_ERR_INVALID_ARGS;
  int s = check(*cfg, *a, nullptr, 0);
  if (s != KS_OK) return s;
  if (a->pass != KS_CE_BACKWARD && !a->loss) return KS_ERR_INVALID_ARGS;
  if (a->pass == KS_CE_BACKWARD && !a->lse) return KS_ERR_INVALID_ARGS;
  if (a->pass != KS_CE_FORWARD && (!a->dh || !a->dw)) return KS_ERR_INVALID_ARGS;
  auto odd = [](const void *p, uintptr_t m) { return (reinterpret_cast<uintptr_t>(p) & (m - 1)) != 0; };
  if (odd(a->h, 2) || odd(a->w, 2) || odd(a->targets, 8) || odd(a->dloss, 4) || odd(a->loss, 4) || odd(a->lse, 4) ||
      odd(a->dh, 2) || odd(a->dw, 2))
    return KS_ERR_INVALID_ARGS;
  Plan p;
  make_plan(*cfg, *a, a->workspace_bytes, p);
  if (!a->workspace || p.bytes > a->workspace_bytes || odd(a->workspace, 256)) return KS_ERR_WORKSPACE;
  // dw is written while other tiles of the launch still read h and w, and dh too
  const bool fwd = a->pass != KS_CE_BACKWARD, bwd = a->pass != KS_CE_FORWARD;
  const int64_t n = a->tokens, row = a->dim * 2, one = a->reduction == KS_CE_NONE ? n * 4 : 4;
  const ks::Rows mem[] = {{a->workspace, 1, int64_t(p.bytes), 0},
                          {bwd ? a->dh : nullptr, n, row, a->dh_stride * 2},
                          {bwd ? a->dw : nullptr, a->vocab, row, a->dw_stride * 2},
                          {fwd ? a->loss : nullptr, 1, one, 0},
                          {a->lse, 1, n * 4, 0},
                          {a->h, n, row, a->h_stride * 2},
                          {a->w, a->vocab, row, a->w_stride * 2},
                          {a->targets, 1, n * 8, 0},
                          {bwd ? a->dloss : nullptr, 1, one, 0}};
  if (ks::outputs_overlap(mem, 5, 9)) return KS_ERR_INVALID_ARGS;
  if ((s = ks::check_arch_sm100()) != KS_OK) return s;
  return run(*a, p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
