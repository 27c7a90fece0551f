// Paged cascade attention for few query rows: decode, speculative or query
// tokens over cached chunks, short prompts.  Serves the calls that the kernels
// of attention.cu do not: a 4-bit cache (kv4.cuh) and a sliding window with
// sinks, over either cache.  Same segments, positions and differential RoPE as
// there; key n at position kn is visible to a query at position p iff kn <= p
// and, with a window W > 0, p - kn < W or kn < sinks.
//
// One producer warp walks the plan and streams tiles of K, V and scales by TMA
// into a shared-memory ring; four consumer warps take a quarter (16 or 32 keys)
// of every tile, each with its own online softmax, so consumers meet only at the
// end and hold no plan.  K is the A operand of
// S^T = K Q^T and V^T that of O^T += V^T P^T (mma.sync m16n8k16), so keys and
// head dims fill the 16 MMA rows and a tile of 8 query rows (token, head of the
// KV group) is one 8-wide B operand: a decode step's 4 or 8 heads of a KV head
// take one pass with little padding.
//
// 4-bit codes never become scaled values.  A code masked out of its word is an
// fp16 subnormal, c 2^-24 (c 2^-20 at bit 4), exact in the MMA, and
//   sum_d q_d (s c_d + z) = s sum_d q_d c_d + z sum_d q_d
// per group of 64: K runs through the MMA as codes, s touches only the 16 x 8
// scores and z sum q comes from one more MMA (z is bf16; the sums of the rounded
// queries are held as three bf16 terms).  For V, s is folded into P and a step's
// products start from one MMA per group with -8 in place of the codes, so that
// they sum s (c - 8): the MMA truncates its fp32 sums, and a mean of 7.5 carried
// through a long context would bias them.  Steps are added in fp32.  The value
// of code 8, sum_n p_n (8 s_n + z_n), is kept as one fp32 scalar per group and
// row, from the unrounded p, so the rounding of P s meets only the deviation.
// Rounding: queries are held in fp16 after scaling each row by a power of two
// to [2^10, 2^11) (elements 2^-25 below the row's largest are lost), P s in
// fp16 scaled by a power of two common to the warp, that of the largest step it
// has met (elements 2^-25 below that are lost); scores, softmax sums and outputs
// are fp32.  This holds for rotated query elements up to 2^100, steps of V from
// 2^-60 and constant groups of V (step 0) up to 2^50; above that, sums may
// overflow, below that, bits are lost.  With a bf16 cache the rotated query is
// split into two bf16 terms (hi + lo, 16 bits) and P is rounded to bf16 once.
//
// Measured on a B200 (GPU time, head_dim 128): a 4-bit cache is read at 4.0-4.3
// TB/s with every CTA slot busy.  Neither DRAM nor a pipe is full there (ALU pipe
// 45%, where the codes are taken apart, issue 51%): chains of dependent
// instructions on 2 to 3.5 warps a scheduler bound it, and registers the warps.
// A bf16 cache (32 windowed requests) is read at 6.2 TB/s.  A call's fixed time
// is about 6.5 us: four dependent reads of the plan, the first tile, one step,
// the join.
//
// The keys that a tile can see (the sink part and the window part of every
// segment) are split over the CTAs of a thread-block cluster, whose partial
// results are joined through distributed shared memory: no workspace, no
// counters, nothing that two launches could share.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "attention_rows.cuh"
#include "attention_types.cuh"
#include "common.cuh"
#include "kv4.cuh"
#include "launch.cuh"
#include "tmap.h"

namespace braid {

constexpr int ROWS_WARPS = 4;                       // consumer warps
constexpr int ROWS_THREADS = 32 * (ROWS_WARPS + 1);  // and the producer
constexpr int ROWS_END = INT_MIN;                   // description of the tile after the last
constexpr float ROWS_EV0 = -50.f;  // first exponent that the weights over a 4-bit cache are held times
constexpr float ROWS_M0 = -1e37f;  // running maximum before any visible key (finite: differences stay defined)

// D (+)= A (16 x 16) B (16 x 8), fp32 accumulation, fp16 or bf16 operands.  Plain (not volatile) asm: the compiler
// may order and schedule them freely.
#define BRAID_MMA(NAME, TYPE)                                                                                       \
  BRAID_DEVICE void NAME(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {                                   \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "        \
        "{%0,%1,%2,%3};"                                                                                            \
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                            \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));                                            \
  }                                                                                                                 \
  BRAID_DEVICE void NAME##_0(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {                               \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "        \
        "{%10,%10,%10,%10};"                                                                                        \
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                            \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));                                  \
  }
BRAID_MMA(mma_f16, "f16")
// D = A B + C, fp16 operands
BRAID_DEVICE void mma_f16_c(float* d, const float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
BRAID_MMA(mma_bf16, "bf16")
#undef BRAID_MMA
// Transpose of an 8 x 8 matrix of 16-bit elements held across the warp.
BRAID_DEVICE uint32_t movmatrix_t(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
BRAID_DEVICE uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Codes at bits 0..3 (times 2^-24 as fp16) and 4..7 (times 2^-20) of each half.
BRAID_DEVICE uint32_t nib_lo(uint32_t w) { return w & 0x000F000Fu; }
BRAID_DEVICE uint32_t nib_hi(uint32_t w) { return w & 0x00F000F0u; }
constexpr uint32_t NIB_LO_M8 = 0x80088008u, NIB_HI_M8 = 0x80808080u;  // -8 in the same units
BRAID_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Untiled bulk copy global -> shared (16-byte aligned, a multiple of 16 bytes), completion on `bar`.
BRAID_DEVICE void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
BRAID_DEVICE uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
BRAID_DEVICE uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
BRAID_DEVICE uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

// Compile-time shape of one instance.
template <int D_, int BITS_, int NT_>
struct RowsShape {
  static constexpr int D = D_, BITS = BITS_, NT = NT_;
  static constexpr int ROWS = 8 * NT;
  static constexpr bool Q4 = BITS == 4;
  // 16-key MMA tiles of a step: two independent ones keep a warp's pipes busier (steady decode from a 4-bit cache 3.94
  // -> 4.28 TB/s); with more row tiles the registers do not allow it
  static constexpr int MB = Q4 && NT == 1 ? 2 : 1;
  static constexpr int KB = 16 * MB;                  // keys of a step
  static constexpr int SUB = ((Q4 || D == 64) ? 2 : 1) / MB; // steps per consumer and tile
  static constexpr int TILE = ROWS_WARPS * SUB * KB;  // keys per tile
  static constexpr int STAGES = Q4 && NT == 1 ? 2 : 3;                    // tiles in the ring
  static constexpr bool QREG = NT == 1;               // one query tile: its fragments live in registers
  static constexpr int GR = Q4 ? D / KV4_GROUP : 1;   // scale groups of a row
  static constexpr int ROW_BYTES = Q4 ? D / 2 : 2 * D;
  static constexpr int KS = D / 16;                   // MMA steps along D
  static constexpr int LD = D + 4;
  // ring stage: K rows, V rows, K scales, V scales
  static constexpr int V_AT = TILE * ROW_BYTES, KS_AT = 2 * V_AT, VS_AT = KS_AT + (Q4 ? TILE * GR * 4 : 0);
  static constexpr int STAGE = VS_AT + (Q4 ? TILE * GR * 4 : 0);
  static constexpr int RING = STAGES * STAGE;
  // query fragments of a warp: 4 registers per lane and unit; a unit is an 8-element word of a K row (4-bit) or an MMA
  // step (bf16: two registers of hi, two of lo).
  static constexpr int QU = Q4 ? D / 32 : KS;
  static constexpr int QF = QREG ? 0 : NT * QU * 32 * 16;
  static constexpr int META_AT = RING + ROWS_WARPS * QF;  // tile descriptions (8 ints each), then the barriers
  static constexpr int BAR_AT = META_AT + STAGES * 32;
  static constexpr int LOOP = BAR_AT + STAGES * 16;
  static constexpr int MERGE = ROWS_WARPS * ROWS * LD * 4;  // partial results, in the same space afterwards
  static constexpr int BODY = LOOP > MERGE ? LOOP : MERGE;
  // what the other CTAs of the cluster send: this CTA's share of the elements from each of them, at most
  // ROWS * D floats and 4 per part of rounding up, and every part's (m, l) rows
  static constexpr int RECV = ROWS * D * 4 + 16 * 16;
  static constexpr int SMEM = BODY + RECV + 1024;
  // 4-bit: first element of word k of a K row / V row of a thread (t = lane % 4, g = lane / 4)
  BRAID_DEVICE static int k_dim(int k, int t) { return 8 * (t * (QU / 2) + (k >> 1)) + (k & 1) * (D / 2); }
  BRAID_DEVICE static int v_dim(int k, int g) {
    const int w = (D / 64) * g + k;
    return 8 * (w >> 1) + (w & 1) * (D / 2);
  }
  BRAID_DEVICE static constexpr int group(int k) { return GR == 2 ? (k & 1) : 0; }
  // bf16: byte offset of 16-byte chunk c of row r in a K or V tile (64-column halves, 128-byte swizzle)
  BRAID_DEVICE static uint32_t chunk(int r, int c) {
    return (uint32_t)((c >> 3) * (TILE * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
  }
};

// The producer's walk over the CTA's tiles: intervals of visible keys (two per
// segment: sinks, window), each in tiles of aligned cache slots.
struct RowsWalk {
  int v, vend;       // interval 2 * segment + part (segments counted from the sequence's first)
  int start;         // visible keys before interval v
  int r0, r1;        // this CTA's range of the visible keys
  int lo, hi;        // keys of the interval within the range, segment-local
  int off, sl;       // slot of key 0, first slot of the tile
  int pos0, delta;
  const int* pages;
  int npages;
};

struct RowsVisible {
  int min_pos, max_pos, window, sinks;
};

// The sequence's segments as the walk reads them: the first ROWS_SEGS in shared
// memory (one round trip for all of them), any further ones from the plan.
constexpr int ROWS_SEGS = 64;
struct RowsSegs {
  int len[ROWS_SEGS], pos0[ROWS_SEGS], off[ROWS_SEGS], delta[ROWS_SEGS], page0[ROWS_SEGS + 1];
};

// Keys [a, b) of part `part` of segment s (counted from the sequence's first) that some row of the tile sees.
BRAID_DEVICE void rows_interval(const RowsParams& p, const RowsSegs& sg, int sg0, const RowsVisible& vis, int s, int part,
                                int& a, int& b) {
  const int len = s < ROWS_SEGS ? sg.len[s] : p.seg_len[sg0 + s], pos0 = s < ROWS_SEGS ? sg.pos0[s] : p.seg_pos0[sg0 + s];
  const int hi = min(max(vis.max_pos - pos0 + 1, 0), len);
  int wlo = 0, slo = 0;
  if (vis.window > 0) {
    wlo = min(max(vis.min_pos - vis.window + 1 - pos0, 0), hi);
    slo = min(max(vis.sinks - pos0, 0), hi);
    if (slo >= wlo) wlo = slo = 0;  // they meet: one interval
  }
  a = part == 0 ? 0 : wlo;
  b = part == 0 ? slo : hi;
}

template <int KB>
BRAID_DEVICE bool rows_settle(const RowsParams& p, const RowsSegs& sg, int sg0, const RowsVisible& vis, RowsWalk& w) {
  for (; w.v < w.vend && w.start < w.r1; ++w.v) {
    const int s = w.v >> 1;
    int a, b;
    rows_interval(p, sg, sg0, vis, s, w.v & 1, a, b);
    const int n = max(b - a, 0);
    w.lo = a + max(w.r0 - w.start, 0);
    w.hi = n <= w.r1 - w.start ? b : a + (w.r1 - w.start);
    if (w.lo < w.hi) {
      const bool here = s < ROWS_SEGS;
      const int pg = here ? sg.page0[s] : p.seg_page_indptr[sg0 + s];
      w.off = here ? sg.off[s] : p.seg_offset[sg0 + s];
      w.pos0 = here ? sg.pos0[s] : p.seg_pos0[sg0 + s];
      w.delta = here ? sg.delta[s] : p.seg_delta[sg0 + s];
      w.pages = p.page_ids + pg;
      w.npages = (here ? sg.page0[s + 1] : p.seg_page_indptr[sg0 + s + 1]) - pg;
      w.sl = (w.off + w.lo) & ~(KB - 1);
      return true;
    }
    w.start += n;
  }
  return false;
}

template <int KB>
BRAID_DEVICE bool rows_next(const RowsParams& p, const RowsSegs& sg, int sg0, const RowsVisible& vis, RowsWalk& w) {
  w.sl += KB;
  if (w.sl < w.off + w.hi) return true;
  int a, b;
  rows_interval(p, sg, sg0, vis, w.v >> 1, w.v & 1, a, b);
  w.start += max(b - a, 0);
  ++w.v;
  return rows_settle<KB>(p, sg, sg0, vis, w);
}

// A lane's piece of the walk's tile: rows [at, at + n) of the tile (n 0: none)
// and the page id they are in, loaded one tile ahead of its use.  A tile in one
// page (PS a multiple of TILE) is one piece, else pieces are 16 rows.  Only rows
// of 16-slot groups that hold keys of the interval are copied: what the others
// hold is masked, whatever it is.
struct RowsPiece {
  int at, n, page, ofs;
};
template <int TILE>
BRAID_DEVICE RowsPiece rows_piece(const RowsParams& p, const RowsWalk& w, int lane) {
  const int a = max(w.off + w.lo - w.sl, 0) & ~15, b = min((w.off + w.hi - w.sl + 15) & ~15, TILE);
  RowsPiece x{0, 0, 0, 0};
  if (p.whole) {
    x.at = a;
    x.n = lane == 0 ? b - a : 0;
  } else {
    x.at = 16 * lane;
    x.n = x.at >= a && x.at < b ? 16 : 0;
  }
  if (x.n > 0) {
    const int idx = max(min((w.sl + x.at) / p.PS, w.npages - 1), 0);
    x.ofs = (w.sl + x.at) % p.PS;
    x.page = w.pages[idx];
  }
  return x;
}

// Start the copies of a tile into a ring stage and describe it there.  An id
// outside the pool reads page 0 or the last one.
template <typename Sh>
BRAID_DEVICE void rows_issue(const RowsParams& p, const CUtensorMap* tm, const RowsWalk& w, const RowsPiece& x, int kh,
                             int lane, uint32_t stage, uint64_t* bar, int* meta) {
  const int rows = __reduce_add_sync(0xffffffffu, x.n);
  if (lane == 0) {
    *reinterpret_cast<int4*>(meta) = make_int4(w.sl - w.off, w.lo, w.hi, w.pos0 + w.sl - w.off);
    meta[4] = w.delta;
    mbar_arrive_expect_tx(bar, rows * 2 * (Sh::ROW_BYTES + (Sh::Q4 ? Sh::GR * 4 : 0)));  // releases the description
  }
  __syncwarp();
  if (x.n > 0) {
    (void)BRAID_IN_BOUNDS(x.page >= 0 && x.page < p.num_pages, 4, x.page);
    const int page = min(max(x.page, 0), p.num_pages - 1);
    const int64_t row = ((int64_t)page * 2 * p.Hkv + kh) * p.PS + x.ofs;
    if constexpr (Sh::Q4) {
      const int64_t vrow = row + (int64_t)p.Hkv * p.PS;
      bulk_load(stage + x.at * Sh::ROW_BYTES, p.kv + row * Sh::ROW_BYTES, x.n * Sh::ROW_BYTES, bar);
      bulk_load(stage + Sh::KS_AT + x.at * 4 * Sh::GR, p.scales + row * Sh::GR, x.n * Sh::GR * 4, bar);
      bulk_load(stage + Sh::V_AT + x.at * Sh::ROW_BYTES, p.kv + vrow * Sh::ROW_BYTES, x.n * Sh::ROW_BYTES, bar);
      bulk_load(stage + Sh::VS_AT + x.at * 4 * Sh::GR, p.scales + vrow * Sh::GR, x.n * Sh::GR * 4, bar);
    } else {
      for (int u = 0; u < x.n; u += 16) {
#pragma unroll
        for (int h = 0; h < Sh::D / 64; ++h) {
          const uint32_t at = stage + h * (Sh::TILE * 128) + (x.at + u) * 128;
          tma_load_2d_u32(at, tm, bar, h * 64, (int)row + u);
          tma_load_2d_u32(at + Sh::V_AT, tm, bar, h * 64, (int)row + u + p.Hkv * p.PS);
        }
      }
    }
  }
}

// One row tile of queries, as loaded (bf16 pairs) and its rotation factors.
template <typename Sh>
struct RowsQ {
  static constexpr int E = Sh::Q4 ? 8 : 4;  // elements of a unit per thread
  uint32_t w[Sh::QU][E / 2];
  float cs[Sh::QU / 2][E], sn[Sh::QU / 2][E];
};

template <typename Sh>
BRAID_DEVICE void rows_load_q(const RowsParams& p, RowsQ<Sh>& x, int t0, int row0, int nrows, int kh, int nt, int lane) {
  const int g = lane >> 2, t = lane & 3, r = nt * 8 + g;
  const int rr = row0 + (r < nrows ? r : 0);
  const __nv_bfloat16* qp = p.q + (int64_t)(t0 + rr / p.G) * p.q_stride + (int64_t)(kh * p.G + rr % p.G) * Sh::D;
#pragma unroll
  for (int k = 0; k < Sh::QU; ++k) {
    if constexpr (Sh::Q4) {
      const uint4 u = r < nrows ? __ldcg(reinterpret_cast<const uint4*>(qp + Sh::k_dim(k, t))) : make_uint4(0, 0, 0, 0);
      x.w[k][0] = u.x; x.w[k][1] = u.y; x.w[k][2] = u.z; x.w[k][3] = u.w;
    } else {  // elements 16 k + 2 t, + 1, + 8, + 9
      x.w[k][0] = r < nrows ? __ldcg(reinterpret_cast<const unsigned*>(qp + 16 * k + 2 * t)) : 0u;
      x.w[k][1] = r < nrows ? __ldcg(reinterpret_cast<const unsigned*>(qp + 16 * k + 2 * t + 8)) : 0u;
    }
  }
}

// cos and sin of position `pos` for this thread's elements; units i and its partner share them.
template <typename Sh>
BRAID_DEVICE void rows_load_rope(const RowsParams& p, RowsQ<Sh>& x, int pos, int lane) {
  const int t = lane & 3;
  pos = pos < 0 ? 0 : (pos >= p.rope_len ? p.rope_len - 1 : pos);
  const float* cp = p.cos + (int64_t)pos * (Sh::D / 2);
  const float* sp = p.sin + (int64_t)pos * (Sh::D / 2);
#pragma unroll
  for (int i = 0; i < Sh::QU / 2; ++i) {
    if constexpr (Sh::Q4) {
      const int at = Sh::k_dim(2 * i, t);
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        *reinterpret_cast<float4*>(x.cs[i] + j) = *reinterpret_cast<const float4*>(cp + at + j);
        *reinterpret_cast<float4*>(x.sn[i] + j) = *reinterpret_cast<const float4*>(sp + at + j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const int at = 16 * i + 2 * t + 4 * j;
        *reinterpret_cast<float2*>(x.cs[i] + j) = *reinterpret_cast<const float2*>(cp + at);
        *reinterpret_cast<float2*>(x.sn[i] + j) = *reinterpret_cast<const float2*>(sp + at);
      }
    }
  }
}

// B fragments of a loaded tile.  4-bit: also this thread's word zq of the row's
// query sums (term t of row g) and hm, the row scales of columns 2t, 2t + 1.
template <typename Sh>
BRAID_DEVICE void rows_frag_q(const RowsParams& p, const RowsQ<Sh>& in, int lane, uint4* frag, uint32_t& zq, float* hm) {
  constexpr int QU = Sh::QU, E = RowsQ<Sh>::E;
  const int t = lane & 3;
  float x[QU][E];
#pragma unroll
  for (int k = 0; k < QU; ++k)
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      x[k][2 * j] = __uint_as_float(in.w[k][j] << 16) * p.q_sign;
      x[k][2 * j + 1] = __uint_as_float(in.w[k][j] & 0xFFFF0000u) * p.q_sign;
    }
  if (p.use_rope) {
#pragma unroll
    for (int i = 0; i < QU / 2; ++i) {
      // units ka (first half of the row) and kb hold rotary partners
      const int ka = Sh::Q4 ? 2 * i : i, kb = Sh::Q4 ? 2 * i + 1 : i + QU / 2;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float a = x[ka][j], b = x[kb][j];
        x[ka][j] = a * in.cs[i][j] - b * in.sn[i][j];
        x[kb][j] = b * in.cs[i][j] + a * in.sn[i][j];
      }
    }
  }
  if constexpr (Sh::Q4) {
    float mx = 0.f;
#pragma unroll
    for (int k = 0; k < QU; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(x[k][j]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // row scale 2^(10 - e) for a largest element in [2^e, 2^(e+1)); e held to [-60, 100]
    const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -60), 100);
    const float f = __int_as_float((10 - e + 127) << 23);
    const float h = __int_as_float((e - 10 + 127) << 23) * p.scale_log2 * 0x1p24f;
    float sq[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < QU; ++k) {
      uint32_t r4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // register i: elements (i, i + 4) of the word; odd i meet codes at bit 4, times 16
        const float up = (i & 1) ? 16.f : 1.f, dn = (i & 1) ? f * 0.0625f : f;
        r4[i] = pack_f16(x[k][i] * dn, x[k][i + 4] * dn);
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r4[i]));
        sq[Sh::group(k)] = fmaf(b.x + b.y, up, sq[Sh::group(k)]);
      }
      frag[k] = make_uint4(r4[0], r4[1], r4[2], r4[3]);
    }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1)
#pragma unroll
      for (int u = 0; u < Sh::GR; ++u) sq[u] += __shfl_xor_sync(0xffffffffu, sq[u], o);
    // sum q per group, in the units of q c (codes count 2^-24), as three bf16 terms: term i of both groups at k = 2i, 2i + 1
    float a = sq[0] * 0x1p-24f, b = sq[1] * 0x1p-24f;
    zq = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const uint32_t term = pack_bf16(a, b);
      if (t == i) zq = term;
      a -= __uint_as_float(term << 16);
      b -= __uint_as_float(term & 0xFFFF0000u);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) hm[c] = __shfl_sync(0xffffffffu, h, (2 * t + c) * 4);
  } else {
#pragma unroll
    for (int k = 0; k < QU; ++k) {
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float a = x[k][2 * i], b = x[k][2 * i + 1];
        hi[i] = pack_bf16(a, b);
        lo[i] = pack_bf16(a - __uint_as_float(hi[i] << 16), b - __uint_as_float(hi[i] & 0xFFFF0000u));
      }
      frag[k] = make_uint4(hi[0], hi[1], lo[0], lo[1]);
    }
    hm[0] = hm[1] = p.scale_log2;
    zq = 0;
  }
}

BRAID_DEVICE void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
BRAID_DEVICE void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
BRAID_DEVICE void dsmem_st_f4(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
BRAID_DEVICE void dsmem_st_f2(uint32_t addr, float a, float b) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1,%2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}

// One CTA: a tile of 8 NT rows of one sequence and KV head, one part of its visible keys.
template <int D, int BITS, int NT, int OCC>
__global__ void __launch_bounds__(ROWS_THREADS, OCC) attn_rows_kernel(const __grid_constant__ CUtensorMap tm,
                                                                         const RowsParams p) {
  using Sh = RowsShape<D, BITS, NT>;
  constexpr int GR = Sh::GR, MT = D / 16, MB = Sh::MB, KB = Sh::KB, QU = Sh::QU;
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~uintptr_t(1023));
  __shared__ float s_m[ROWS_WARPS][Sh::ROWS], s_l[ROWS_WARPS][Sh::ROWS];
  __shared__ float2 s_part[16][Sh::ROWS];  // (m, l) of every CTA of the cluster
  __shared__ RowsSegs segs;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int S = p.splits;
  const int kh = blockIdx.z / S, split = blockIdx.z % S, b = blockIdx.y;
  const uint32_t ring = smem_u32(sm), qf = ring + Sh::RING + warp * Sh::QF;
  int* meta = reinterpret_cast<int*>(sm + Sh::META_AT);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sm + Sh::BAR_AT);
  uint64_t* empty_bar = full_bar + Sh::STAGES;
  if (threadIdx.x == 0) {
    span_start(p.span);
    if constexpr (!Sh::Q4) tma_prefetch_desc(&tm);
    for (int i = 0; i < Sh::STAGES; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], ROWS_WARPS);
    }
    fence_barrier_init();
  }
  if (S > 1) cluster_arrive();  // met before the first remote store: every CTA of the cluster has started
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) span_waited(p.span);
  const int t0 = p.qo_indptr[b], t1 = p.qo_indptr[b + 1], sg0 = p.seg_indptr[b], nseg = p.seg_indptr[b + 1] - sg0;
  const int rows = (t1 - t0) * p.G, row0 = blockIdx.x * Sh::ROWS;
  if (row0 >= rows) {  // every CTA of the cluster alike
    if (S > 1) cluster_wait();
    return;
  }
  const int nrows = min(Sh::ROWS, rows - row0);
  for (int i = threadIdx.x; i < min(nseg, ROWS_SEGS); i += ROWS_THREADS) {
    segs.len[i] = p.seg_len[sg0 + i];
    segs.pos0[i] = p.seg_pos0[sg0 + i];
    segs.off[i] = p.seg_offset[sg0 + i];
    segs.delta[i] = p.seg_delta[sg0 + i];
    segs.page0[i] = p.seg_page_indptr[sg0 + i];
    segs.page0[i + 1] = p.seg_page_indptr[sg0 + i + 1];  // also written by its own thread, with the same value
  }
  int rpos[NT][2];  // positions of this thread's two rows (columns 2t, 2t + 1) of each tile; -1 past the last row
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = nt * 8 + 2 * t + c;
      rpos[nt][c] = r < nrows ? p.positions[t0 + (row0 + r) / p.G] : -1;
    }
  RowsVisible vis{INT_MAX, -1, p.window, p.sinks};
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      vis.max_pos = max(vis.max_pos, rpos[nt][c]);
      if (rpos[nt][c] >= 0) vis.min_pos = min(vis.min_pos, rpos[nt][c]);
    }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    vis.max_pos = max(vis.max_pos, __shfl_xor_sync(0xffffffffu, vis.max_pos, o));
    vis.min_pos = min(vis.min_pos, __shfl_xor_sync(0xffffffffu, vis.min_pos, o));
  }
  RowsQ<Sh> xq;  // one tile: loaded along with the plan
  int qpos = 0;  // position of row g
  if constexpr (Sh::QREG) {
    if (warp < ROWS_WARPS) {
      rows_load_q<Sh>(p, xq, t0, row0, nrows, kh, 0, lane);
      qpos = p.positions[t0 + (row0 + min(g, nrows - 1)) / p.G];
    }
  }
  __syncthreads();

  if (warp == ROWS_WARPS) {
    // ------------------------------------------------------------ producer
    RowsWalk w{};
    w.vend = 2 * nseg;
    w.r1 = INT_MAX;
    if (S > 1) {
      int total = 0;
      for (int v = 0; v < 2 * nseg; ++v) {
        int a, e;
        rows_interval(p, segs, sg0, vis, v >> 1, v & 1, a, e);
        total += max(e - a, 0);
      }
      const int per = ((total + S - 1) / S + Sh::TILE - 1) / Sh::TILE * Sh::TILE;
      w.r0 = min(total, split * per);
      w.r1 = min(total, w.r0 + per);
    }
    bool more = rows_settle<Sh::TILE>(p, segs, sg0, vis, w), ok = true;
    RowsPiece x{};
    if (more) x = rows_piece<Sh::TILE>(p, w, lane);
    int i = 0, st = 0, ph = 1;
    for (;; ++i) {
      if (i >= Sh::STAGES && !mbar_wait(&empty_bar[st], ph)) {
        ok = false;
        break;
      }
      if (!more) {
        if (lane == 0) {
          meta[8 * st] = ROWS_END;
          mbar_arrive(&full_bar[st]);
        }
        break;
      }
      rows_issue<Sh>(p, &tm, w, x, kh, lane, ring + st * Sh::STAGE, &full_bar[st], meta + 8 * st);
      more = rows_next<Sh::TILE>(p, segs, sg0, vis, w);
      if (more) x = rows_piece<Sh::TILE>(p, w, lane);
      if (++st == Sh::STAGES) {
        st = 0;
        ph ^= 1;
      }
    }
    // Tiles [0, i) were issued.  No copy may outlive the CTA or land in the space of the partial results, also where this
    // warp or a consumer gave up, so those not known to have landed are waited for.  Tile i - STAGES is known where the
    // loop ended regularly: the consumers released its stage to the end mark, whose arrival is that barrier's next phase.
    for (int j = max(0, i - Sh::STAGES + (ok ? 1 : 0)); j < i; ++j)
      (void)mbar_wait(&full_bar[j % Sh::STAGES], (j / Sh::STAGES) & 1);
  }
  // ---------------------------------------------------------------- consumers
  float acc[NT][MT][4];
  float m[NT][2], l[NT][2], rest[NT][GR][2];  // rest: sum of p (8 s + z) per V group (4-bit)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[nt][c] = ROWS_M0;
      l[nt][c] = 0.f;
#pragma unroll
      for (int h = 0; h < GR; ++h) rest[nt][h][c] = 0.f;
    }
  }
  // 4-bit: every p of this warp is held times 2^-ev, so that P s stays within fp16 whatever the steps; from -50 on, so
  // that sums of p (8 s + z) stay within fp32 where no step moves it (constant groups have step 0)
  float ev = ROWS_EV0, lim = 0x1p-46f;  // lim: 2^(ev + 4)

  uint4 qr[Sh::QREG ? QU : 1];
  uint32_t zq[NT];             // 4-bit: B fragment (k = 2t, 2t + 1) of z sum q: term t of row g's sums, 0 for t = 3
  float hm[NT][2];             // score units to base 2 of columns 2t, 2t + 1
  float th[NT][2], mb[NT][2];  // score above which the maximum moves; maximum in base 2 (+ ev)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      th[nt][c] = ROWS_M0;
      mb[nt][c] = 0.f;
    }
  // fragments of every tile for RoPE delta `delta`; the bounds in score units follow the rows' scales
  const auto build = [&](int delta, RowsQ<Sh>& xq) {
    if constexpr (Sh::QREG) {
      if (p.use_rope) rows_load_rope<Sh>(p, xq, qpos - delta, lane);
      rows_frag_q<Sh>(p, xq, lane, qr, zq[0], hm[0]);
    } else {
      __syncwarp();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        RowsQ<Sh> x;
        uint4 f[QU];
        rows_load_q<Sh>(p, x, t0, row0, nrows, kh, nt, lane);
        if (p.use_rope)
          rows_load_rope<Sh>(p, x, p.positions[t0 + (row0 + min(nt * 8 + g, nrows - 1)) / p.G] - delta, lane);
        rows_frag_q<Sh>(p, x, lane, f, zq[nt], hm[nt]);
#pragma unroll
        for (int k = 0; k < QU; ++k)
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(qf + ((nt * QU + k) * 32 + lane) * 16), "r"(f[k].x),
                       "r"(f[k].y), "r"(f[k].z), "r"(f[k].w)
                       : "memory");
      }
      __syncwarp();
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) th[nt][c] = m[nt][c] == ROWS_M0 ? ROWS_M0 : (m[nt][c] + 8.f) / hm[nt][c];
  };
  uint32_t m8[4];  // opaque, or the compiler would rebuild them for every use
  asm volatile("mov.b32 %0, %2; mov.b32 %1, %3;" : "=r"(m8[0]), "=r"(m8[1]) : "n"(NIB_LO_M8), "n"(NIB_HI_M8));
  m8[2] = m8[0];
  m8[3] = m8[1];
  bool ok = true;
  // the first segment's delta (most plans have one for all) while the first copies are under way
  int built = nseg > 0 ? segs.delta[0] : 0;
  if (warp < ROWS_WARPS) build(built, xq);
  int st = 0, ph = 0;
#pragma unroll 1
  while (warp < ROWS_WARPS) {
    if (!mbar_wait(&full_bar[st], ph)) {
      ok = false;
      break;
    }
    const int4 md = *reinterpret_cast<const int4*>(meta + 8 * st);
    if (md.x == ROWS_END) break;
    const int delta = meta[8 * st + 4];
    const uint32_t kt = ring + st * Sh::STAGE;
    const int lo = md.y, hi = md.z;
    uint64_t* const done = &empty_bar[st];
    if (++st == Sh::STAGES) {
      st = 0;
      ph ^= 1;
    }
    if (built != delta) {
      RowsQ<Sh> x;
      if constexpr (Sh::QREG) rows_load_q<Sh>(p, x, t0, row0, nrows, kh, 0, lane);
      build(delta, x);
      built = delta;
    }

    // every key of the tile visible to every row: nothing to mask
    const bool tile_inner = md.x >= lo && md.x + Sh::TILE <= hi && md.w + Sh::TILE - 1 <= vis.min_pos &&
                            (p.window == 0 || md.w > vis.max_pos - p.window || md.w + Sh::TILE <= p.sinks);
#pragma unroll 1
    for (int sub = 0; sub < Sh::SUB; ++sub) {
      const int key0 = (warp * Sh::SUB + sub) * KB, j0 = md.x + key0, kp0 = md.w + key0;  // this step's keys
      if (!tile_inner && (j0 >= hi || j0 + KB <= lo)) continue;

      // ---- scores S^T (times hm: base 2): rows g, g + 8 of each 16-key tile, columns 2t, 2t + 1
      float s[MB][NT][4];
      if constexpr (Sh::Q4) {
#pragma unroll
        for (int u = 0; u < MB; ++u) {
          uint32_t kw[2][QU], kz[2][GR];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int key = key0 + 16 * u + g + 8 * r;
            if constexpr (D == 128) {
              const uint4 v = lds128(kt + key * 64 + t * 16);
              kw[r][0] = v.x; kw[r][1] = v.y; kw[r][2] = v.z; kw[r][3] = v.w;
              const uint2 z = lds64(kt + Sh::KS_AT + key * 8);
              kz[r][0] = z.x; kz[r][1] = z.y;
            } else {
              const uint2 v = lds64(kt + key * 32 + t * 8);
              kw[r][0] = v.x; kw[r][1] = v.y;
              kz[r][0] = lds32(kt + Sh::KS_AT + key * 4);
            }
          }
          float sa[NT][GR][4];
#pragma unroll
          for (int k = 0; k < QU; ++k) {
            const uint32_t wa = kw[0][k], wb = kw[1][k];
            const uint32_t a0[4] = {nib_lo(wa), nib_lo(wb), nib_hi(wa), nib_hi(wb)};
            const uint32_t wa8 = wa >> 8, wb8 = wb >> 8;
            const uint32_t a1[4] = {nib_lo(wa8), nib_lo(wb8), nib_hi(wa8), nib_hi(wb8)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint4 q;
              if constexpr (Sh::QREG) q = qr[k];
              else q = lds128(qf + ((nt * QU + k) * 32 + lane) * 16);
              if (k < GR) mma_f16_0(sa[nt][Sh::group(k)], a0, q.x, q.y);
              else mma_f16(sa[nt][Sh::group(k)], a0, q.x, q.y);
              mma_f16(sa[nt][Sh::group(k)], a1, q.z, q.w);
            }
          }
          // z of both groups, at k = 2t, 2t + 1 of the rows g and g + 8 (zero at k >= 8 and, through zq, at k 6 and 7)
          const uint32_t az[4] = {GR == 2 ? __byte_perm(kz[0][0], kz[0][GR - 1], 0x7632) : kz[0][0] >> 16,
                                  GR == 2 ? __byte_perm(kz[1][0], kz[1][GR - 1], 0x7632) : kz[1][0] >> 16, 0u, 0u};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_bf16_0(s[u][nt], az, zq[nt], 0u);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int h = 0; h < GR; ++h) s[u][nt][e] = fmaf(kv4_scale(kz[e >> 1][h]), sa[nt][h][e], s[u][nt][e]);
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < MB; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = 0.f;
#pragma unroll
        for (int k = 0; k < QU; ++k)
#pragma unroll
          for (int u = 0; u < MB; ++u) {
            uint32_t a[4];
            ldsm_x4(kt + Sh::chunk(key0 + 16 * u + (lane & 7) + ((lane >> 3) & 1) * 8, 2 * k + (lane >> 4)), a[0], a[1], a[2], a[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint4 q;
              if constexpr (Sh::QREG) q = qr[k];
              else q = lds128(qf + ((nt * QU + k) * 32 + lane) * 16);
              mma_bf16(s[u][nt], a, q.z, q.w);
              mma_bf16(s[u][nt], a, q.x, q.y);
            }
          }
      }

      // ---- masks: only blocks at the ends of an interval or across a row's position or window need them
      const bool inner = tile_inner || (j0 >= lo && j0 + KB <= hi && kp0 + KB - 1 <= vis.min_pos &&
                                        (p.window == 0 || kp0 > vis.max_pos - p.window || kp0 + KB <= p.sinks));
      if (!inner) {
#pragma unroll
        for (int u = 0; u < MB; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d = 16 * u + g + 8 * (e >> 1);
              const int j = j0 + d, kp = kp0 + d, rp = rpos[nt][e & 1];
              const bool see = j >= lo && j < hi && kp <= rp && (p.window == 0 || rp - kp < p.window || kp < p.sinks);
              if (!see) s[u][nt][e] = -INFINITY;
            }
      }

      // ---- 4-bit: (s, z) words of V's keys; keys outside the interval may hold anything
      [[maybe_unused]] uint32_t vz[MB][2][GR];
      float big = 0.f;  // largest V step
      if constexpr (Sh::Q4) {
#pragma unroll
        for (int u = 0; u < MB; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int key = key0 + 16 * u + g + 8 * r;
            if constexpr (GR == 2) {
              const uint2 z2 = lds64(kt + Sh::VS_AT + key * 8);
              vz[u][r][0] = z2.x;
              vz[u][r][GR - 1] = z2.y;
            } else {
              vz[u][r][0] = lds32(kt + Sh::VS_AT + key * 4);
            }
          }
        if (!inner) {
#pragma unroll
          for (int u = 0; u < MB; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int j = j0 + 16 * u + g + 8 * r;
#pragma unroll
              for (int h = 0; h < GR; ++h) vz[u][r][h] = j >= lo && j < hi ? vz[u][r][h] : 0u;
            }
        }
        __nv_bfloat162 top = __float2bfloat162_rn(0.f);  // packed maximum of the (s, z) words; its s half counts
#pragma unroll
        for (int u = 0; u < MB; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int h = 0; h < GR; ++h) top = __hmax2(top, *reinterpret_cast<const __nv_bfloat162*>(&vz[u][r][h]));
        big = __low2float(top);
      }

      // ---- running maxima move only when a score passes one by 2^8 (P then stays below 2^8 in its 16-bit type), the
      // power of two of P s only when a step passes 2^4 times what it was set for
      bool over = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(s[0][nt][c], s[0][nt][2 + c]);
          if constexpr (MB == 2) mx = fmaxf(mx, fmaxf(s[1][nt][c], s[1][nt][2 + c]));
          over |= mx > th[nt][c];
        }
      if constexpr (Sh::Q4) over |= big > lim;
      if (__any_sync(0xffffffffu, over)) {
        float f = 1.f;
        if constexpr (Sh::Q4) {
          const float wb = warp_max(big);
          if (wb > lim) {
            const int ne = min((int)(__float_as_uint(wb) >> 23) - 127, 120);  // above ROWS_EV0 + 3
            f = ex2(ev - (float)ne);
            ev = (float)ne;
            lim = __int_as_float((ne + 4 + 127) << 23);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(s[0][nt][c], s[0][nt][2 + c]);
            if constexpr (MB == 2) mx = fmaxf(mx, fmaxf(s[1][nt][c], s[1][nt][2 + c]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = mx == -INFINITY ? m[nt][c] : fmaxf(m[nt][c], mx * hm[nt][c]);
            const float corr = ex2(m[nt][c] - mx) * f;
            m[nt][c] = mx;
            mb[nt][c] = (mx == ROWS_M0 ? 0.f : mx) + (Sh::Q4 ? ev : 0.f);
            th[nt][c] = mx == ROWS_M0 ? ROWS_M0 : (mx + 8.f) / hm[nt][c];
            l[nt][c] *= corr;
#pragma unroll
            for (int h = 0; h < GR; ++h) rest[nt][h][c] *= corr;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              acc[nt][i][c] *= corr;
              acc[nt][i][2 + c] *= corr;
            }
          }
      }

      // ---- P and O^T += V^T P^T
      const auto weigh = [&](auto masked) {
        constexpr bool MASK = decltype(masked)::value;
        uint32_t pq[MB][NT][GR][2];
#pragma unroll
        for (int u = 0; u < MB; ++u) {
          auto& pb = pq[u];
          [[maybe_unused]] float sv[2][GR], zv[2][GR];  // V's steps and the values of code 8
          if constexpr (Sh::Q4) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
              for (int h = 0; h < GR; ++h) {
                sv[r][h] = kv4_scale(vz[u][r][h]);
                zv[r][h] = fmaf(8.f, sv[r][h], kv4_offset(vz[u][r][h]));
              }
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float pr[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              pr[e] = ex2(fmaf(s[u][nt][e], hm[nt][e & 1], -mb[nt][e & 1]));
              l[nt][e & 1] += pr[e];
            }
            if constexpr (Sh::Q4) {
#pragma unroll
              for (int h = 0; h < GR; ++h) {
                float ps[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float sc = sv[e >> 1][h], zc = zv[e >> 1][h];
                  // a masked score has weight 0, and 0 times NaN would not be 0
                  const bool skip = MASK && s[u][nt][e] == -INFINITY;
                  ps[e] = skip ? 0.f : pr[e] * sc;
                  rest[nt][h][e & 1] = fmaf(pr[e], skip ? 0.f : zc, rest[nt][h][e & 1]);
                }
                pb[nt][h][0] = movmatrix_t(pack_f16(ps[0], ps[1]));
                pb[nt][h][1] = movmatrix_t(pack_f16(ps[2], ps[3]));
              }
            } else {
              pb[nt][0][0] = movmatrix_t(pack_bf16(pr[0], pr[1]));
              pb[nt][0][1] = movmatrix_t(pack_bf16(pr[2], pr[3]));
            }
          }
          if constexpr (!Sh::Q4) {
            uint32_t keep[2] = {~0u, ~0u};  // keys 2t, 2t + 1 and 2t + 8, 2t + 9: those outside the interval read as 0
            if constexpr (MASK) {
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int j = j0 + 16 * u + 2 * t + (r & 1) + 8 * (r >> 1);
                if (j < lo || j >= hi) keep[r >> 1] &= (r & 1) ? 0x0000FFFFu : 0xFFFF0000u;
              }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              uint32_t a[4];
              ldsm_x4_t(kt + Sh::V_AT + Sh::chunk(key0 + 16 * u + (lane & 7) + (lane >> 4) * 8, 2 * i + ((lane >> 3) & 1)), a[0],
                        a[1], a[2], a[3]);
              if constexpr (MASK) {
                a[0] &= keep[0];
                a[1] &= keep[0];
                a[2] &= keep[1];
                a[3] &= keep[1];
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_bf16(acc[nt][i], a, pb[nt][0][0], pb[nt][0][1]);
            }
          }
        }
        if constexpr (Sh::Q4) {
          constexpr int NV = D / 64;
          float low[NT][GR][4];  // -8 P of the step: what every MMA tile of a group starts from
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < GR; ++h) {
              mma_f16_0(low[nt][h], m8, pq[0][nt][h][0], pq[0][nt][h][1]);
              if constexpr (MB == 2) mma_f16(low[nt][h], m8, pq[MB - 1][nt][h][0], pq[MB - 1][nt][h][1]);
            }
          uint32_t vw[MB][4][NV];  // keys 2t, 2t + 1, 2t + 8, 2t + 9 of each 16
#pragma unroll
          for (int u = 0; u < MB; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int key = key0 + 16 * u + 2 * t + (r & 1) + 8 * (r >> 1);
              if constexpr (D == 128) {
                const uint2 v = lds64(kt + Sh::V_AT + key * 64 + g * 8);
                vw[u][r][0] = v.x; vw[u][r][1] = v.y;
              } else {
                vw[u][r][0] = lds32(kt + Sh::V_AT + key * 32 + g * 4);
              }
            }
#pragma unroll
          for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {  // halves of the words: MMA tiles 2 hf, 2 hf + 1
              uint32_t x[MB][2];
#pragma unroll
              for (int u = 0; u < MB; ++u) {
                x[u][0] = __byte_perm(vw[u][0][k], vw[u][1][k], hf ? 0x7632 : 0x5410);
                x[u][1] = __byte_perm(vw[u][2][k], vw[u][3][k], hf ? 0x7632 : 0x5410);
              }
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  float d[4];
#pragma unroll
                  for (int u = 0; u < MB; ++u) {
                    const uint32_t y0 = i ? x[u][0] >> 8 : x[u][0], y1 = i ? x[u][1] >> 8 : x[u][1];
                    const uint32_t av[4] = {nib_lo(y0), nib_hi(y0), nib_lo(y1), nib_hi(y1)};
                    if (u == 0) mma_f16_c(d, low[nt][Sh::group(k)], av, pq[u][nt][Sh::group(k)][0], pq[u][nt][Sh::group(k)][1]);
                    else mma_f16(d, av, pq[u][nt][Sh::group(k)][0], pq[u][nt][Sh::group(k)][1]);
                  }
#pragma unroll
                  for (int e = 0; e < 4; ++e) acc[nt][k * 4 + hf * 2 + i][e] += d[e];
                }
            }
        }
      };
      if (inner)
        weigh(std::false_type{});
      else
        weigh(std::true_type{});

    }
    // ---- every lane is done with the stage
    __syncwarp();
    if (lane == 0) mbar_arrive(done);
  }
  if (!ok) {  // a copy did not land in time: the rows become NaN
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt][0] = l[nt][1] = __int_as_float(0x7fc00000);
      m[nt][0] = m[nt][1] = 0.f;
    }
  }

  // ---- join the warps of the CTA, then the CTAs of the cluster
  __syncthreads();  // the ring's space becomes [warp][row][LD] partial outputs
  float* aw = reinterpret_cast<float*>(sm);
  const float up = Sh::Q4 ? ex2(ev) : 1.f;
  if (warp < ROWS_WARPS) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[nt][c];
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if constexpr (Sh::Q4) {
#pragma unroll
          for (int h = 0; h < GR; ++h)
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) rest[nt][h][c] += __shfl_xor_sync(0xffffffffu, rest[nt][h][c], o);
        }
        const int r = nt * 8 + 2 * t + c;
        if (g == 0) {
          // a sum that is NaN counts even if no score of the warp was a number, which leaves the maximum where it was
          s_m[warp][r] = sum != sum && m[nt][c] == ROWS_M0 ? 0.f : m[nt][c];
          s_l[warp][r] = sum * up;
        }
        float* dst = aw + (warp * Sh::ROWS + r) * Sh::LD;
        if constexpr (Sh::Q4) {
#pragma unroll
          for (int k = 0; k < D / 64; ++k) {
            float o8[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              o8[2 * i] = fmaf(acc[nt][k * 4 + i][c], 0x1p24f, rest[nt][Sh::group(k)][c]) * up;
              o8[2 * i + 1] = fmaf(acc[nt][k * 4 + i][2 + c], 0x1p20f, rest[nt][Sh::group(k)][c]) * up;
            }
            *reinterpret_cast<float4*>(dst + Sh::v_dim(k, g)) = make_float4(o8[0], o8[1], o8[2], o8[3]);
            *reinterpret_cast<float4*>(dst + Sh::v_dim(k, g) + 4) = make_float4(o8[4], o8[5], o8[6], o8[7]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            dst[16 * i + g] = acc[nt][i][c];
            dst[16 * i + g + 8] = acc[nt][i][2 + c];
          }
        }
      }
  }
  __syncthreads();
  constexpr int C4 = D / 4;
  // Remote stores into the receive space, which nothing else uses: the first cluster barrier (arrived at the start) says
  // that its CTA runs, the second that all parts are there, and then no CTA touches another's memory again.
  const uint32_t recv = smem_u32(sm + Sh::BODY);
  const int share = (nrows * C4 + S - 1) / S;  // float4 elements of a part that one CTA joins
  if (S > 1) cluster_wait();
  const auto store = [&](int r, int d, float4 o, float inv) {
    const int rr = row0 + r;
    __nv_bfloat16* dst = p.out + ((int64_t)(t0 + rr / p.G) * p.Hq + kh * p.G + rr % p.G) * D + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
  };
  for (int i = threadIdx.x; i < nrows * C4; i += ROWS_THREADS) {
    const int r = i / C4, d = (i % C4) * 4;
    float M = ROWS_M0;
#pragma unroll
    for (int q = 0; q < ROWS_WARPS; ++q) M = fmaxf(M, s_m[q][r]);
    float L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 0; q < ROWS_WARPS; ++q) {
      if (s_m[q][r] == ROWS_M0) continue;
      const float e = ex2(s_m[q][r] - M);
      L += s_l[q][r] * e;
      const float4 a = *reinterpret_cast<const float4*>(aw + (q * Sh::ROWS + r) * Sh::LD + d);
      o.x += a.x * e;
      o.y += a.y * e;
      o.z += a.z * e;
      o.w += a.w * e;
    }
    if (S == 1) {
      store(r, d, o, M == ROWS_M0 ? 0.f : 1.f / L);
    } else {
      const int q = i / share;  // the CTA that joins element i
      dsmem_st_f4(dsmem_map(recv + (split * share + i - q * share) * 16, q), o);
      if (d == 0)
        for (int u = 0; u < S; ++u) dsmem_st_f2(dsmem_map(smem_u32(&s_part[split][r]), u), M, L);
    }
  }
  if (S > 1) {
    cluster_arrive();
    cluster_wait();
    const float4* got = reinterpret_cast<const float4*>(sm + Sh::BODY);
    for (int n = threadIdx.x; n < min(share, nrows * C4 - split * share); n += ROWS_THREADS) {
      const int i = split * share + n, r = i / C4, d = (i % C4) * 4;
      float M = ROWS_M0, L = 0.f;
      for (int q = 0; q < S; ++q) M = fmaxf(M, s_part[q][r].x);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = 0; q < S; ++q) {
        const float2 ml = s_part[q][r];
        if (ml.x == ROWS_M0) continue;
        const float e = ex2(ml.x - M);
        const float4 v = got[q * share + n];
        L += ml.y * e;
        o.x += v.x * e;
        o.y += v.y * e;
        o.z += v.z * e;
        o.w += v.w * e;
      }
      store(r, d, o, M == ROWS_M0 ? 0.f : 1.f / L);
    }
  }
  if (threadIdx.x == 0) span_end(p.span);
}

// ------------------------------------------------------------------ host
int gemm_num_sms();
unsigned long long* next_span(const char* name);
void kv4_check_layer(const torch::Tensor& codes, const torch::Tensor& scales, const char* who);

// Key parts per row tile, and about how long the call then takes.
struct RowsPlan {
  int splits;
  int64_t ns;
};

// A power of two up to the 16 CTAs of a cluster, each part of at least one tile: the fewest waves of resident CTAs times
// (its keys' time + the fixed time of a CTA: plan, queries, first tile, joining).  Fitted on a B200 (head_dim 128): with
// every slot busy a CTA takes 17 ns a key from a 4-bit cache, from a bf16 one 24 ns with three CTAs an SM (one row tile)
// and 14 with one, and 8 us apart from its keys.  64 requests of 10000 keys: 288, 254, 259, 302 us at 1, 2, 4, 8 parts;
// 8 requests of 2100: 28, 22, 17, 24 us; one request of 600 on 8 KV heads: 10.7, 9.5, 8.2, 7.2 us.  `work`: row tiles of
// all sequences and KV heads.
template <int D, int BITS, int NT, int OCC>
static RowsPlan rows_plan(int64_t work, int64_t max_keys) {
  using Sh = RowsShape<D, BITS, NT>;
  const int64_t slots = (int64_t)std::min(OCC, (int)(227 * 1024 / (Sh::SMEM + 4096))) * gemm_num_sms();
  const int64_t per_key = (Sh::Q4 ? 17 : NT == 1 ? 24 : 14) * D / 128;  // ns
  RowsPlan best{1, INT64_MAX};
  for (int n = 1; n <= 16 && (n == 1 || max_keys >= (int64_t)n * Sh::TILE / 2); n *= 2) {
    const int64_t est = (work * n + slots - 1) / slots * (max_keys / n * per_key + 8000);
    if (est < best.ns) best = {n, est};
  }
  return best;
}

template <int D, int BITS, int NT, int OCC>
static void launch_rows(RowsParams& p, int64_t pool_rows, int64_t num_seqs, int64_t max_q, int64_t max_keys, cudaStream_t st) {
  using Sh = RowsShape<D, BITS, NT>;
  const auto k = attn_rows_kernel<D, BITS, NT, OCC>;
  static bool ready[64] = {};  // attributes are per device
  int dev;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (!ready[dev & 63]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
    C10_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    ready[dev & 63] = true;
  }
  const int64_t tiles = (max_q * p.G + Sh::ROWS - 1) / Sh::ROWS;
  const int S = rows_plan<D, BITS, NT, OCC>(tiles * num_seqs * p.Hkv, max_keys).splits;
  p.splits = S;
  p.whole = Sh::Q4 && p.PS % Sh::TILE == 0;
  TORCH_CHECK(tiles < (1ll << 31) && num_seqs <= 65535 && (int64_t)p.Hkv * S <= 65535, "attention: launch grid too large");
  CUtensorMap tm{};
  if (!Sh::Q4) tm = make_tmap(p.kv, pool_rows, D, D, 16);  // the layer pool as rows of D elements, boxes of 16 x 64
  launch_pdl_cluster(k, dim3((unsigned)tiles, (unsigned)num_seqs, (unsigned)(p.Hkv * S)), dim3(ROWS_THREADS),
                     Sh::SMEM, st, dim3(1, 1, (unsigned)S), tm, p);
}

// Calls of many rows a sequence (head_dim 128): the tcgen05 prefill kernel of attention_tc.cu with the window.  A 4-bit
// cache is first read into a bf16 workspace, page by page as the plan lists them: one more rounding of K and V to bf16,
// and 2 + 0.56 bytes an element once per call, against the whole prompt's products (4000 tokens of Llama-3-8B heads: 8 of
// 196 us).
int attn_prefill_tc_mode();
int attn_prefill_tc_rows();
int attn_prefill_tc_min_rows();
void launch_attn_prefill_tc(const AttnParams& p, int num_seqs, int max_q_len, int64_t P, cudaStream_t st);
void kv4_unpack_pages(torch::Tensor out, const torch::Tensor& codes, const torch::Tensor& scales, const RowsParams& p,
                      int64_t num_seqs, cudaStream_t st);

// Query rows per CTA as for the calls without a window: 128 where CTAs of 256 would fill less than half of the SMs.
static int prompt_cta_rows(int64_t max_rows, int64_t num_seqs, int64_t Hkv) {
  const int64_t units = (max_rows + attn_prefill_tc_rows() - 1) / attn_prefill_tc_rows() * num_seqs * Hkv;
  return units * 2 <= gemm_num_sms() ? attn_prefill_tc_min_rows() : attn_prefill_tc_rows();
}

// Key splits of that kernel, where its row tiles (`units`, of all sequences and KV heads) leave SMs idle, and about how
// long the call then takes in units of a 128-key tile: waves of (tiles and about two of prologue), and the join.
struct PromptPlan {
  int splits;
  int64_t tiles;
};
static PromptPlan prompt_plan(int64_t units, int64_t keys) {
  const int64_t sms = gemm_num_sms(), kvt = std::max<int64_t>(1, (keys + 127) / 128);
  PromptPlan best{1, (units + sms - 1) / sms * (kvt + 2)};
  for (int n = 2; n <= 32 && n <= kvt && units < sms; ++n) {
    const int64_t est = (units * n + sms - 1) / sms * ((kvt + n - 1) / n + 2) + n;
    if (est < best.tiles) best = {n, est};
  }
  return best;
}

// The largest workspace that a call over a 4-bit cache takes; one that would need more goes by rows.  64 requests over a
// shared chunk of 8192 tokens, 256 queries each (32 heads on 8), list 2.2 GB of it: 17.1 ms by rows, 3.0 so.
constexpr int64_t PROMPT_WORKSPACE = 4ll << 30;
int64_t attn_kv4_workspace_limit() { return PROMPT_WORKSPACE; }

// Whether a call of several queries takes the tcgen05 kernel.  By rows of the sequences, not of the batch: a sequence's
// rows are taken 16 at a time by the row kernel and up to 256 at a time by that one, whose tile costs the same however
// few they are, and from a 4-bit cache every listed page is written and read once more first.  The shorter of the two
// estimates decides: rows_plan() and a tile of 2.3 us, 8 us of prologue and output, and from a 4-bit cache 6 us and
// 0.14 ns a key and KV head (what a B200 measured with 4 heads on each of 8 KV heads).  By rows and by tcgen05, us:
//   queries x sequences over keys    4-bit cache        bf16 cache
//    64 x 1 over  3200                41    56           55    46
//   128 x 1 over  3200                67    60          108    44
//     2 x 64 over 3200                87   450          135   230
//    16 x 16 over 3200               131   120          223    61
//    64 x 16 over 3200               453   133          748    73
//    32 x 1 over 12000                70    88           99    63
// Sequences of unequal length count by their rows together, a tile more for each.
// A prompt of 512 rows takes the tcgen05 kernel also where that is up to 20 us slower (512 rows over 600 keys in 4 bits:
// 21 and 30), so that prompts round alike whatever their length.
static bool prompt_pays(bool q4, int64_t T, int64_t num_seqs, int64_t max_q_len, int64_t G, int64_t Hkv, int64_t PS,
                        int64_t keys, int64_t num_page_ids) {
  const int64_t max_rows = max_q_len * G, slots = num_page_ids * PS * Hkv;
  if (q4 && slots * 2 * 128 * 2 > PROMPT_WORKSPACE) return false;
  if (attn_prefill_tc_mode() >= 0) return attn_prefill_tc_mode() == 1;
  if (max_rows <= 8) return false;  // one row tile
  const auto tiles = [&](int64_t rows) {
    return std::min((max_rows + rows - 1) / rows * num_seqs, T * G / rows + num_seqs) * Hkv;
  };
  const int64_t by_rows = q4 ? rows_plan<128, 4, 2, 2>(tiles(16), keys).ns : rows_plan<128, 16, 2, 2>(tiles(16), keys).ns;
  const int64_t units = tiles(prompt_cta_rows(max_rows, num_seqs, Hkv));
  const int64_t here = 8000 + prompt_plan(units, keys).tiles * 2300 + (q4 ? 6000 + slots * 14 / 100 : 0);
  return here < by_rows + (max_rows >= 512 ? 20000 : 0);
}

static void attention_prompt(const RowsParams& r, const torch::Tensor* pool, const torch::Tensor& kv,
                             const c10::optional<torch::Tensor>& scales, int64_t T, int64_t num_seqs, int64_t max_q_len,
                             int64_t keys, int64_t num_page_ids, cudaStream_t st) {
  AttnParams p{};
  torch::Tensor work = pool != nullptr ? *pool : torch::empty({std::max<int64_t>(1, num_page_ids), 2, r.Hkv, r.PS, 128},
                                                              scales->options());
  if (pool == nullptr) kv4_unpack_pages(work, kv, *scales, r, num_seqs, st);
  p.page_identity = pool == nullptr ? 1 : 0;
  p.q = r.q;
  p.q_stride = r.q_stride;
  p.kv = reinterpret_cast<const __nv_bfloat16*>(work.data_ptr());
  p.out = r.out;
  p.qo_indptr = r.qo_indptr;
  p.positions = r.positions;
  p.seg_indptr = r.seg_indptr;
  p.seg_page_indptr = r.seg_page_indptr;
  p.seg_offset = r.seg_offset;
  p.seg_len = r.seg_len;
  p.seg_pos0 = r.seg_pos0;
  p.seg_delta = r.seg_delta;
  p.page_ids = r.page_ids;
  p.cos = r.cos;
  p.sin = r.sin;
  p.rope_len = r.rope_len;
  p.use_rope = r.use_rope;
  p.scale_log2 = r.scale_log2;
  p.q_flip = r.q_sign < 0.f ? 0x80008000u : 0u;
  p.Hq = r.Hq;
  p.Hkv = r.Hkv;
  p.G = r.G;
  p.PS = r.PS;
  p.num_pages = (int)work.size(0);
  p.window = r.window > 0 ? r.window : 1 << 30;
  p.sinks = r.window > 0 ? r.sinks : 0;
  p.span = r.span;
  p.cta_rows = prompt_cta_rows(max_q_len * r.G, num_seqs, r.Hkv);
  const int64_t work_units = (max_q_len * r.G + p.cta_rows - 1) / p.cta_rows * num_seqs * r.Hkv;
  p.num_splits = prompt_plan(work_units, keys).splits;
  TORCH_CHECK(num_seqs <= 65535 && (int64_t)r.Hkv * p.num_splits <= 65535, "attention: launch grid too large");
  torch::Tensor po, pl, ctr;  // the join's counters belong to this call alone
  if (p.num_splits > 1) {
    const auto f32 = work.options().dtype(at::kFloat);
    po = torch::empty({T * r.Hq * p.num_splits * 128}, f32);
    pl = torch::empty({T * r.Hq * p.num_splits}, f32);
    ctr = torch::zeros({work_units}, work.options().dtype(at::kInt));
    p.part_o = po.data_ptr<float>();
    p.part_lse = pl.data_ptr<float>();
    p.counters = ctr.data_ptr<int>();
  }
  launch_attn_prefill_tc(p, (int)num_seqs, (int)max_q_len, work.size(0), st);
}

// Attention of few rows over a bf16 layer pool (`kv`, `scales` undefined) or a
// 4-bit layer (`kv` = codes), with an optional window; into `out` if given.
torch::Tensor attention_rows(const c10::optional<torch::Tensor>& out_arg, const torch::Tensor& q, const torch::Tensor& kv,
                    const c10::optional<torch::Tensor>& scales, const torch::Tensor& qo_indptr,
                    const torch::Tensor& positions, const torch::Tensor& seg_indptr,
                    const torch::Tensor& seg_page_indptr, const torch::Tensor& seg_offset, const torch::Tensor& seg_len,
                    const torch::Tensor& seg_pos0, const torch::Tensor& seg_delta, const torch::Tensor& page_ids,
                    const torch::Tensor& cos, const torch::Tensor& sin, double scale, bool use_rope, int64_t num_seqs, int64_t max_q_len,
                    int64_t max_kv_len, int64_t window, int64_t sinks) {
  const bool q4 = scales.has_value() && scales->defined();
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 3, "attention: q must be bf16 [T, Hq, D]");
  const auto dev = q.device();
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  TORCH_CHECK(D == 64 || D == 128, "attention: head_dim must be 64 or 128");
  TORCH_CHECK(q.stride(2) == 1 && q.stride(1) == D && q.stride(0) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              "attention: the heads of a q row must be contiguous and rows 16-byte aligned");
  if (q4) {
    kv4_check_layer(kv, *scales, "attention");
  } else {
    TORCH_CHECK(kv.is_cuda() && kv.scalar_type() == at::kBFloat16 && kv.dim() == 5 && kv.is_contiguous() &&
                    kv.size(1) == 2 && reinterpret_cast<uintptr_t>(kv.data_ptr()) % 16 == 0,
                "attention: cache must be a contiguous bf16 tensor [P, 2, Hkv, page, D]");
    TORCH_CHECK(kv.numel() / D < (1ll << 31), "attention: a bf16 cache of more than 2^31 rows");
  }
  const at::cuda::CUDAGuard guard(dev);
  const bool given = out_arg.has_value() && out_arg->defined();
  const torch::Tensor out = given ? *out_arg : at::empty({T, Hq * D}, q.options());
  TORCH_CHECK(kv.device() == dev && out.device() == dev, "attention: q, cache and out on different devices");
  const int64_t Hkv = kv.size(2), PS = kv.size(3);
  TORCH_CHECK(kv.size(4) == (q4 ? D / 2 : D) && Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "attention: head layout mismatch");
  TORCH_CHECK(PS > 0 && PS % 16 == 0 && kv.size(0) > 0, "attention: page size must be a multiple of 16, the pool not empty");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.is_contiguous() && out.numel() == T * Hq * D &&
                  reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0,
              "attention: out must be a contiguous, 16-byte aligned bf16 [T, Hq * D]");
  TORCH_CHECK(window >= 0 && window < (1ll << 30) && sinks >= 0 && sinks < (1ll << 30),
              "attention: window and sinks must be in [0, 2^30)");
  TORCH_CHECK(num_seqs >= 0 && max_q_len >= 0 && max_q_len <= T, "attention: max_q_len must be in [0, T]");
  if (T == 0 || num_seqs == 0 || max_q_len == 0) return out;
  const auto i32 = [&](const torch::Tensor& t, int64_t n, const char* name) {
    TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous() && t.device() == dev && t.numel() >= n, "attention: ",
                name, " must be a contiguous int32 tensor of at least ", std::to_string(n), " elements on the device of the cache");
    return t.data_ptr<int>();
  };
  RowsParams p{};
  p.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  p.q_stride = q.stride(0);
  p.kv = reinterpret_cast<const uint8_t*>(kv.data_ptr());
  p.scales = q4 ? reinterpret_cast<const uint32_t*>(scales->data_ptr()) : nullptr;
  p.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  p.qo_indptr = i32(qo_indptr, num_seqs + 1, "qo_indptr");
  p.positions = i32(positions, T, "positions");
  p.seg_indptr = i32(seg_indptr, num_seqs + 1, "seg_indptr");
  const int64_t ns = seg_len.numel();
  p.seg_len = i32(seg_len, 0, "seg_len");
  p.seg_page_indptr = i32(seg_page_indptr, ns + 1, "seg_page_indptr");
  p.seg_offset = i32(seg_offset, ns, "seg_offset");
  p.seg_pos0 = i32(seg_pos0, ns, "seg_pos0");
  p.seg_delta = i32(seg_delta, ns, "seg_delta");
  p.page_ids = i32(page_ids, 0, "page_ids");
  if (use_rope) {
    TORCH_CHECK(cos.device() == dev && sin.device() == dev && cos.scalar_type() == at::kFloat &&
                    sin.scalar_type() == at::kFloat && cos.is_contiguous() && sin.is_contiguous() && cos.dim() == 2 &&
                    cos.size(1) == D / 2 && cos.size(0) >= 1 && sin.sizes() == cos.sizes() &&
                    reinterpret_cast<uintptr_t>(cos.data_ptr()) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(sin.data_ptr()) % 16 == 0,
                "attention: cos and sin must be contiguous, 16-byte aligned fp32 [positions, D/2] tables on the device of the cache");
    p.cos = cos.data_ptr<float>();
    p.sin = sin.data_ptr<float>();
    p.rope_len = (int)cos.size(0);
  }
  p.use_rope = use_rope ? 1 : 0;
  p.scale_log2 = std::max(std::fabs((float)scale) * LOG2E, 1e-20f);
  p.q_sign = scale < 0 ? -1.f : 1.f;
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.G = (int)(Hq / Hkv);
  p.PS = (int)PS;
  p.num_pages = (int)kv.size(0);
  p.window = (int)window;
  p.sinks = (int)sinks;
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  p.span = next_span("attn_rows");
  int64_t keys = std::max<int64_t>(1, max_kv_len);
  if (window > 0) keys = std::min(keys, window + sinks + max_q_len);
  const int64_t rows = max_q_len * p.G;
  if (D == 128 && max_q_len > 1 && prompt_pays(q4, T, num_seqs, max_q_len, p.G, Hkv, PS, keys, page_ids.numel())) {
    attention_prompt(p, q4 ? nullptr : &kv, kv, scales, T, num_seqs, max_q_len, keys, page_ids.numel(), st);
    return out;
  }
  const auto pick = [&](auto d, auto bits) {
    constexpr int DD = decltype(d)::value, BB = decltype(bits)::value;
    // One tile over a 4-bit cache: with work for every slot of three CTAs an SM their eight more warps pay (64 requests
    // of 4001-16001 tokens: 234 us, with two CTAs 246); with less, the two CTAs' registers do (8 requests of 2100: 12.1
    // us, with three 16.0; 16 windowed ones 52 and 78).
    if constexpr (BB == 4) {
      if (rows <= 8 && num_seqs * Hkv < 3 * gemm_num_sms()) {
        launch_rows<DD, BB, 1, 2>(p, kv.size(0) * 2 * Hkv * PS, num_seqs, max_q_len, keys, st);
        return;
      }
    }
    if (rows <= 8)
      launch_rows<DD, BB, 1, 3>(p, kv.size(0) * 2 * Hkv * PS, num_seqs, max_q_len, keys, st);
    else  // tiles of 16 rows: 32 spill and, of short queries, leave SMs idle (64 queries over 3136 keys, D 64: 27 us, with
          // 32 rows 36; a 2000-token prompt 213 and 216)
      launch_rows<DD, BB, 2, 2>(p, kv.size(0) * 2 * Hkv * PS, num_seqs, max_q_len, keys, st);
  };
  using std::integral_constant;
  if (D == 128 && q4)
    pick(integral_constant<int, 128>{}, integral_constant<int, 4>{});
  else if (D == 128)
    pick(integral_constant<int, 128>{}, integral_constant<int, 16>{});
  else if (q4)
    pick(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else
    pick(integral_constant<int, 64>{}, integral_constant<int, 16>{});
  return out;
}

BRAID_BOUNDS_READER(bounds_status_attention_rows)

}  // namespace braid
