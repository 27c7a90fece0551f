// Paged cascade attention for few query rows: decode, speculative or query
// tokens over cached chunks, short prompts.  Serves the calls that the kernels
// of attention.cu do not: a 4-bit cache (kv4.cuh) and a sliding window with
// sinks, over either cache.  Same segments, positions and differential RoPE as
// there; key n at position kn is visible to a query at position p iff kn <= p
// and, with a window W > 0, p - kn < W or kn < sinks.
//
// Every warp works alone on blocks of 16 keys: it loads K, V and the scales of
// a block straight into the registers that mma.sync takes them from, and keeps
// its own online softmax.  K is the A operand of S^T = K Q^T and V^T that of
// O^T += V^T P^T, so keys and head dims fill the 16 MMA rows and a tile of 8
// query rows (token, head of the KV group) is one 8-wide B operand: a decode
// step's 4 or 8 heads of a KV head take one pass with little padding.
//
// 4-bit codes never become scaled values.  fp16 1024 + c is one LOP3 away from
// a code word (c in the low mantissa bits), and
//   sum_d q_d (s c_d + z) = s (sum_d q_d (1024 + c_d) - 1024 sum_d q_d) + z sum_d q_d
// per group of 64: K runs through the MMA as 1024 + c with the accumulator
// starting at -1024 sum q, and s, z touch only the 16 x 8 scores.  V enters as
// c - 8 (one HFMA2 more: a bias of 1024 would drown long sums), s folded into P
// and sum_n p_n (8 s_n + z_n) kept as one fp32 scalar per group and row, from
// the unrounded p: the rounding of P s then meets only the deviation s (c - 8).
// Rounding: queries are held in fp16 after scaling each row by a power of two
// to [2^10, 2^11) (elements 2^-25 below the row's largest are lost), P s in
// fp16 scaled by a power of two common to the warp; scores, softmax sums and
// outputs are fp32.  With a bf16 cache the rotated query is split into two bf16
// terms (hi + lo, 16 bits) and P is rounded to bf16 once.
//
// The keys that a tile can see (the sink part and the window part of every
// segment) are split over the CTAs of a thread-block cluster, whose partial
// results are joined through distributed shared memory: no workspace, no
// counters, nothing that two launches could share.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "attention_types.cuh"
#include "common.cuh"
#include "kv4.cuh"
#include "launch.cuh"

namespace braid {

struct RowsParams {
  const __nv_bfloat16* q;   // rows of [Hq, D], q_stride elements apart
  int64_t q_stride;
  const uint8_t* kv;        // bf16 pool [P, 2, Hkv, PS, D] or the 4-bit codes
  const uint32_t* scales;   // 4-bit (s, z) pairs
  __nv_bfloat16* out;       // [T, Hq, D]
  const int* qo_indptr;
  const int* positions;
  const int* seg_indptr;
  const int* seg_page_indptr;
  const int* seg_offset;
  const int* seg_len;
  const int* seg_pos0;
  const int* seg_delta;
  const int* page_ids;
  const float* cos;
  const float* sin;
  float scale_log2;
  int use_rope, rope_len;
  int Hq, Hkv, G, PS, num_pages;
  int window, sinks;        // window 0: every earlier key
  int splits;               // CTAs per cluster
  unsigned long long* span;
};

constexpr int ROWS_WARPS = 4;
constexpr int ROWS_BLK = 16;  // keys per block

BRAID_DEVICE void mma16816_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Transpose of an 8 x 8 matrix of 16-bit elements held across the warp.
BRAID_DEVICE uint32_t movmatrix_t(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
BRAID_DEVICE uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
BRAID_DEVICE uint32_t f16_sub(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
BRAID_DEVICE uint32_t f16_fma(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// 1024 + (the nibble of each half at bit 0 / 16 times it at bit 4)
BRAID_DEVICE uint32_t nib_lo(uint32_t w) { return (w & 0x000F000Fu) | 0x64006400u; }
BRAID_DEVICE uint32_t nib_hi(uint32_t w) { return (w & 0x00F000F0u) | 0x64006400u; }
// the same as c - 8, exact in fp16
BRAID_DEVICE uint32_t nib_lo8(uint32_t w) { return f16_sub(nib_lo(w), 0x64086408u); }                   // - 1032
BRAID_DEVICE uint32_t nib_hi8(uint32_t w) { return f16_fma(nib_hi(w), 0x2C002C00u, 0xD480D480u); }      // / 16 - 72
BRAID_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Compile-time shape of one instance.
template <int D_, int BITS_, int NT_>
struct RowsShape {
  static constexpr int D = D_, BITS = BITS_, NT = NT_;
  static constexpr int ROWS = 8 * NT;
  static constexpr bool Q4 = BITS == 4;
  static constexpr int NW = D / 32;              // 8-element words of a K row per thread
  static constexpr int NV = D / 64;              // 8-element words of a V row per thread
  static constexpr int GR = Q4 ? D / KV4_GROUP : 1;  // scale groups of a row
  static constexpr int QREGS = Q4 ? 4 : 8;       // B registers per K word and query tile (bf16: hi and lo)
  static constexpr int KR = Q4 ? 2 * NW : 8 * NW;    // registers of a K block (rows g, g + 8)
  static constexpr int VR = Q4 ? 4 * NV : 16 * NV;   // registers of a V block (keys 2t, 2t+1, 2t+8, 2t+9)
  static constexpr int ROW_BYTES = Q4 ? D / 2 : 2 * D;
  static constexpr int LD = D + 4;
  // shared memory: per warp the query fragments and (4-bit) their sums; the same space holds the partial results later
  static constexpr int QF_WARP = NT * NW * 32 * QREGS * 4;
  static constexpr int INFO_WARP = NT * 8 * 8 * 4;
  static constexpr int BUILD = ROWS_WARPS * (QF_WARP + INFO_WARP);
  static constexpr int MERGE = ROWS_WARPS * ROWS * LD * 4;
  static constexpr int SMEM = BUILD > MERGE ? BUILD : MERGE;
  // first element of K word k / V word k of a thread (t = lane % 4, g = lane / 4)
  BRAID_DEVICE static int k_dim(int k, int t) {
    return Q4 ? 8 * (t * (NW / 2) + (k >> 1)) + (k & 1) * (D / 2) : 32 * k + 8 * t;
  }
  BRAID_DEVICE static int v_dim(int k, int g) {
    if (!Q4) return 64 * k + 8 * g;
    const int w = NV * g + k;
    return 8 * (w >> 1) + (w & 1) * (D / 2);
  }
  BRAID_DEVICE static constexpr int group(int k) { return GR == 2 ? (k & 1) : 0; }
  // the K word of the same thread that holds the rotary partners of word k
  BRAID_DEVICE static constexpr int partner(int k) { return Q4 ? (k ^ 1) : (k ^ (NW / 2)); }
  BRAID_DEVICE static constexpr bool first_half(int k) { return Q4 ? (k & 1) == 0 : k < NW / 2; }
};

// Walk of one warp over its blocks: intervals of visible keys (two per
// segment: sinks, window), each in blocks of 16 aligned cache slots dealt to
// the warps in turn.
struct RowsWalk {
  int v, vend;       // interval 2 * segment + part
  int start;         // visible keys before interval v
  int dealt;         // blocks before it
  int r0, r1;        // this CTA's range of the visible keys
  int lo, hi;        // keys of the interval within the range, segment-local
  int off, sl;       // slot of key 0, first slot of the block
  int pos0, delta;
  const int* pages;
  int pidx, pofs;    // page index and offset of sl
};

struct RowsVisible {
  int min_pos, max_pos, window, sinks;
};

// Keys [a, b) of part `part` of segment s that some row of the tile sees.
BRAID_DEVICE void rows_interval(const RowsParams& p, const RowsVisible& vis, int s, int part, int& a, int& b) {
  const int len = p.seg_len[s], pos0 = p.seg_pos0[s];
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

BRAID_DEVICE bool rows_settle(const RowsParams& p, const RowsVisible& vis, RowsWalk& w, int warp) {
  for (; w.v < w.vend && w.start < w.r1; ++w.v) {
    const int s = w.v >> 1;
    int a, b;
    rows_interval(p, vis, s, w.v & 1, a, b);
    const int n = max(b - a, 0);
    w.lo = a + max(w.r0 - w.start, 0);
    w.hi = n <= w.r1 - w.start ? b : a + (w.r1 - w.start);
    if (w.lo < w.hi) {
      w.off = p.seg_offset[s];
      const int first = (w.off + w.lo) & ~(ROWS_BLK - 1);
      const int blocks = (w.off + w.hi - first + ROWS_BLK - 1) / ROWS_BLK;
      const int mine = (warp - w.dealt) & (ROWS_WARPS - 1);
      if (mine < blocks) {
        w.pos0 = p.seg_pos0[s];
        w.delta = p.seg_delta[s];
        w.pages = p.page_ids + p.seg_page_indptr[s];
        w.sl = first + mine * ROWS_BLK;
        w.pidx = w.sl / p.PS;
        w.pofs = w.sl - w.pidx * p.PS;
        return true;
      }
      w.dealt += blocks;
    }
    w.start += n;
  }
  return false;
}

BRAID_DEVICE bool rows_next(const RowsParams& p, const RowsVisible& vis, RowsWalk& w, int warp) {
  w.sl += ROWS_BLK * ROWS_WARPS;
  if (w.sl < w.off + w.hi) {
    w.pofs += ROWS_BLK * ROWS_WARPS;
    while (w.pofs >= p.PS) {
      w.pofs -= p.PS;
      ++w.pidx;
    }
    return true;
  }
  const int first = (w.off + w.lo) & ~(ROWS_BLK - 1);
  w.dealt += (w.off + w.hi - first + ROWS_BLK - 1) / ROWS_BLK;
  int a, b;
  rows_interval(p, vis, w.v >> 1, w.v & 1, a, b);
  w.start += max(b - a, 0);
  ++w.v;
  return rows_settle(p, vis, w, warp);
}

// First row (slot) of the block in the layer's [page, K/V, head, slot] order; -1 for a page outside the pool.
BRAID_DEVICE int64_t rows_block_row(const RowsParams& p, const RowsWalk& w, int kh) {
  const int page = w.pages[w.pidx];
  if (!BRAID_IN_BOUNDS(page >= 0 && page < p.num_pages, 4, page) || (unsigned)page >= (unsigned)p.num_pages) return -1;
  return ((int64_t)page * 2 * p.Hkv + kh) * p.PS + w.pofs;
}

template <typename Sh>
BRAID_DEVICE void rows_load_k(const RowsParams& p, int64_t row, int g, int t, uint32_t* kr, uint32_t* ksz) {
  constexpr int D = Sh::D;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint8_t* src = p.kv + (row + g + 8 * r) * Sh::ROW_BYTES;
    if constexpr (Sh::Q4) {
      if constexpr (D == 128) {
        const uint4 u = __ldcg(reinterpret_cast<const uint4*>(src) + t);
        kr[r * 4] = u.x; kr[r * 4 + 1] = u.y; kr[r * 4 + 2] = u.z; kr[r * 4 + 3] = u.w;
        const uint2 z = __ldcg(reinterpret_cast<const uint2*>(p.scales) + row + g + 8 * r);
        ksz[r * 2] = z.x; ksz[r * 2 + 1] = z.y;
      } else {
        const uint2 u = __ldcg(reinterpret_cast<const uint2*>(src) + t);
        kr[r * 2] = u.x; kr[r * 2 + 1] = u.y;
        ksz[r] = __ldcg(p.scales + row + g + 8 * r);
      }
    } else {
#pragma unroll
      for (int k = 0; k < Sh::NW; ++k) {
        const uint4 u = __ldcg(reinterpret_cast<const uint4*>(src + 64 * k) + t);
        uint32_t* d = kr + (r * Sh::NW + k) * 4;
        d[0] = u.x; d[1] = u.y; d[2] = u.z; d[3] = u.w;
      }
    }
  }
}

template <typename Sh>
BRAID_DEVICE void rows_load_v(const RowsParams& p, int64_t row, int g, int t, uint32_t* vr, uint32_t* vsz) {
  constexpr int D = Sh::D;
#pragma unroll
  for (int r = 0; r < 4; ++r) {  // keys 2t, 2t+1, 2t+8, 2t+9
    const int key = 2 * t + (r & 1) + 8 * (r >> 1);
    const uint8_t* src = p.kv + (row + key) * Sh::ROW_BYTES;
    if constexpr (Sh::Q4) {
      if constexpr (D == 128) {
        const uint2 u = __ldcg(reinterpret_cast<const uint2*>(src) + g);
        vr[r * 2] = u.x; vr[r * 2 + 1] = u.y;
      } else {
        vr[r] = __ldcg(reinterpret_cast<const uint32_t*>(src) + g);
      }
    } else {
#pragma unroll
      for (int k = 0; k < Sh::NV; ++k) {
        const uint4 u = __ldcg(reinterpret_cast<const uint4*>(src + 128 * k) + g);
        uint32_t* d = vr + (r * Sh::NV + k) * 4;
        d[0] = u.x; d[1] = u.y; d[2] = u.z; d[3] = u.w;
      }
    }
  }
  if constexpr (Sh::Q4) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (D == 128) {
        const uint2 z = __ldcg(reinterpret_cast<const uint2*>(p.scales) + row + g + 8 * r);
        vsz[r * 2] = z.x; vsz[r * 2 + 1] = z.y;
      } else {
        vsz[r] = __ldcg(p.scales + row + g + 8 * r);
      }
    }
  }
}

// This warp's query tile rotated for a segment with RoPE delta `delta`, as B
// fragments in shared memory; 4-bit: also, per row, the group sums of the
// rounded query and of what 1024 of the codes' bias adds, and the row's scale.
template <typename Sh>
BRAID_DEVICE void rows_build_q(const RowsParams& p, uint32_t* qf, float* info, int t0, int row0, int nrows, int kh,
                               int delta, int lane) {
  constexpr int D = Sh::D, NW = Sh::NW, H2 = D / 2;
  const int g = lane >> 2, t = lane & 3;
#pragma unroll 1
  for (int nt = 0; nt < Sh::NT; ++nt) {
    const int r = nt * 8 + g;
    const bool live = r < nrows;
    const int rr = row0 + (live ? r : 0);
    const int tok = t0 + rr / p.G;
    const __nv_bfloat16* qp = p.q + (int64_t)tok * p.q_stride + (int64_t)(kh * p.G + rr % p.G) * D;
    float x[NW][8];
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (live) u = __ldcg(reinterpret_cast<const uint4*>(qp + Sh::k_dim(k, t)));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[k][2 * j] = __uint_as_float(w[j] << 16);
        x[k][2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
    if (p.use_rope) {
      int pos = p.positions[tok] - delta;
      pos = pos < 0 ? 0 : (pos >= p.rope_len ? p.rope_len - 1 : pos);
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        if (!Sh::first_half(k)) continue;
        const int kb = Sh::partner(k);
        const float* cp = p.cos + (int64_t)pos * H2 + Sh::k_dim(k, t);
        const float* sp = p.sin + (int64_t)pos * H2 + Sh::k_dim(k, t);
        float cs[8], sn[8];
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          *reinterpret_cast<float4*>(cs + j) = __ldcg(reinterpret_cast<const float4*>(cp + j));
          *reinterpret_cast<float4*>(sn + j) = __ldcg(reinterpret_cast<const float4*>(sp + j));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a = x[k][j], b = x[kb][j];
          x[k][j] = a * cs[j] - b * sn[j];
          x[kb][j] = b * cs[j] + a * sn[j];
        }
      }
    }
    if constexpr (Sh::Q4) {
      float mx = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(x[k][j]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // row scale 2^(10 - e) for a largest element in [2^e, 2^(e+1)); e held to [-100, 126]
      const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 126);
      const float f = __int_as_float((10 - e + 127) << 23), hm = __int_as_float((e - 10 + 127) << 23) * p.scale_log2;
      float sq[2] = {0.f, 0.f}, bias[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        uint32_t r4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // register i: elements (i, i + 4) of the word; odd i meet codes at bit 4, times 16
          const float up = (i & 1) ? 16.f : 1.f, dn = (i & 1) ? f * 0.0625f : f;
          const __half2 h = __floats2half2_rn(x[k][i] * dn, x[k][i + 4] * dn);
          r4[i] = *reinterpret_cast<const uint32_t*>(&h);
          const float2 b = __half22float2(h);
          sq[Sh::group(k)] += (b.x + b.y) * up;
          bias[Sh::group(k)] += (b.x + b.y) * 1024.f;
        }
        *reinterpret_cast<uint4*>(qf + ((nt * NW + k) * 32 + lane) * 4) = make_uint4(r4[0], r4[1], r4[2], r4[3]);
      }
#pragma unroll
      for (int o = 1; o <= 2; o <<= 1)
#pragma unroll
        for (int h = 0; h < Sh::GR; ++h) {
          sq[h] += __shfl_xor_sync(0xffffffffu, sq[h], o);
          bias[h] += __shfl_xor_sync(0xffffffffu, bias[h], o);
        }
      if (t == 0) {
        float* d = info + (nt * 8 + g) * 8;
        *reinterpret_cast<float4*>(d) = make_float4(-bias[0], sq[0], -bias[1], sq[1]);
        d[4] = hm;
      }
    } else {
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hi[i] = pack_bf16(x[k][2 * i], x[k][2 * i + 1]);
          lo[i] = pack_bf16(x[k][2 * i] - __uint_as_float(hi[i] << 16),
                            x[k][2 * i + 1] - __uint_as_float(hi[i] & 0xFFFF0000u));
        }
        uint32_t* d = qf + ((nt * NW + k) * 32 + lane) * 8;
        *reinterpret_cast<uint4*>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(d + 4) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
  }
  __syncwarp();
}

// Scores S^T (16 keys x 8 rows per query tile, base-2 units) of a K block.
template <typename Sh>
BRAID_DEVICE void rows_scores(const RowsParams& p, const uint32_t* kr, const uint32_t* ksz, const uint32_t* qf,
                              const float* info, int lane, float (*s)[4]) {
  constexpr int NW = Sh::NW, NT = Sh::NT;
  if constexpr (Sh::Q4) {
    const int t = lane & 3;
    float acc[NT][Sh::GR][4];
    float4 in[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      in[nt][0] = *reinterpret_cast<const float4*>(info + (nt * 8 + 2 * t) * 8);
      in[nt][1] = *reinterpret_cast<const float4*>(info + (nt * 8 + 2 * t + 1) * 8);
      acc[nt][0][0] = acc[nt][0][2] = in[nt][0].x;
      acc[nt][0][1] = acc[nt][0][3] = in[nt][1].x;
      if constexpr (Sh::GR == 2) {
        acc[nt][1][0] = acc[nt][1][2] = in[nt][0].z;
        acc[nt][1][1] = acc[nt][1][3] = in[nt][1].z;
      }
    }
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const uint32_t wa = kr[k], wb = kr[NW + k];
      const uint32_t a0[4] = {nib_lo(wa), nib_lo(wb), nib_hi(wa), nib_hi(wb)};
      const uint32_t wa8 = wa >> 8, wb8 = wb >> 8;
      const uint32_t a1[4] = {nib_lo(wa8), nib_lo(wb8), nib_hi(wa8), nib_hi(wb8)};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint4 b = *reinterpret_cast<const uint4*>(qf + ((nt * NW + k) * 32 + lane) * 4);
        mma16816_f16(acc[nt][Sh::group(k)], a0, b.x, b.y);
        mma16816_f16(acc[nt][Sh::group(k)], a1, b.z, b.w);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float hm0 = info[(nt * 8 + 2 * t) * 8 + 4], hm1 = info[(nt * 8 + 2 * t + 1) * 8 + 4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = e >> 1, c = e & 1;
        const uint32_t z0 = ksz[r * Sh::GR];
        float v = fmaf(kv4_scale(z0), acc[nt][0][e], kv4_offset(z0) * in[nt][c].y);
        if constexpr (Sh::GR == 2) {
          const uint32_t z1 = ksz[r * 2 + 1];
          v = fmaf(kv4_scale(z1), acc[nt][1][e], fmaf(kv4_offset(z1), in[nt][c].w, v));
        }
        s[nt][e] = v * (c ? hm1 : hm0);
      }
    }
  } else {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const uint32_t* wa = kr + k * 4;
      const uint32_t* wb = kr + (NW + k) * 4;
      const uint32_t a0[4] = {wa[0], wb[0], wa[1], wb[1]};
      const uint32_t a1[4] = {wa[2], wb[2], wa[3], wb[3]};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint32_t* d = qf + ((nt * NW + k) * 32 + lane) * 8;
        const uint4 b = *reinterpret_cast<const uint4*>(d), l = *reinterpret_cast<const uint4*>(d + 4);
        mma16816(s[nt], a0, l.x, l.y);
        mma16816(s[nt], a1, l.z, l.w);
        mma16816(s[nt], a0, b.x, b.y);
        mma16816(s[nt], a1, b.z, b.w);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] *= p.scale_log2;
  }
}

// One CTA: a tile of 8 NT rows of one sequence and KV head, one part of its visible keys.
template <int D, int BITS, int NT, int OCC>
__global__ void __launch_bounds__(32 * ROWS_WARPS, OCC) attn_rows_kernel(const RowsParams p) {
  using Sh = RowsShape<D, BITS, NT>;
  constexpr int GR = Sh::GR, MT = D / 16;
  extern __shared__ __align__(16) uint8_t sm_raw[];
  __shared__ float s_m[ROWS_WARPS][Sh::ROWS], s_l[ROWS_WARPS][Sh::ROWS];
  __shared__ float s_M[Sh::ROWS], s_L[Sh::ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int S = p.splits;
  const int kh = blockIdx.z / S, split = blockIdx.z % S, b = blockIdx.y;
  if (threadIdx.x == 0) span_start(p.span);
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) span_waited(p.span);
  const int t0 = p.qo_indptr[b], rows = (p.qo_indptr[b + 1] - t0) * p.G;
  const int row0 = blockIdx.x * Sh::ROWS;
  if (row0 >= rows) return;  // every CTA of the cluster alike
  const int nrows = min(Sh::ROWS, rows - row0);

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
  const int sg0 = p.seg_indptr[b], sg1 = p.seg_indptr[b + 1];
  RowsWalk w{};
  w.v = 2 * sg0;
  w.vend = 2 * sg1;
  w.r0 = 0;
  w.r1 = INT_MAX;
  if (S > 1) {
    int total = 0;
    for (int v = 2 * sg0; v < 2 * sg1; ++v) {
      int a, e;
      rows_interval(p, vis, v >> 1, v & 1, a, e);
      total += max(e - a, 0);
    }
    const int step = ROWS_BLK * ROWS_WARPS;
    const int per = ((total + S - 1) / S + step - 1) / step * step;
    w.r0 = min(total, split * per);
    w.r1 = min(total, w.r0 + per);
  }

  uint32_t* qf = reinterpret_cast<uint32_t*>(sm_raw + warp * (Sh::QF_WARP + Sh::INFO_WARP));
  float* info = reinterpret_cast<float*>(sm_raw + warp * (Sh::QF_WARP + Sh::INFO_WARP) + Sh::QF_WARP);
  float acc[NT][MT][4];
  float m[NT][2], l[NT][2], rest[NT][GR][2];  // rest: sum of p (8 s + z) per V group (4-bit)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[nt][c] = -INFINITY;
      l[nt][c] = 0.f;
#pragma unroll
      for (int h = 0; h < GR; ++h) rest[nt][h][c] = 0.f;
    }
  }
  float vdown = __int_as_float((100 + 127) << 23);  // 4-bit: P s and p z are held times this power of two

  uint32_t kr[Sh::KR], vr[Sh::VR], ksz[2 * GR], vsz[2 * GR];
  bool more = rows_settle(p, vis, w, warp);
  int64_t row = -1;
  int built = 0;
  bool have_q = false;
  if (more) {
    row = rows_block_row(p, w, kh);
    if (row >= 0) {
      rows_load_k<Sh>(p, row, g, t, kr, ksz);
      rows_load_v<Sh>(p, row + (int64_t)p.Hkv * p.PS, g, t, vr, vsz);
    }
  }
  while (more) {
    if (!have_q || built != w.delta) {
      __syncwarp();
      rows_build_q<Sh>(p, qf, info, t0, row0, nrows, kh, w.delta, lane);
      built = w.delta;
      have_q = true;
    }
    const int j0 = w.sl - w.off, lo = w.lo, hi = w.hi, kp0 = w.pos0 + j0;
    const bool loaded = row >= 0;
    float s[NT][4];
    if (loaded) rows_scores<Sh>(p, kr, ksz, qf, info, lane, s);
    // the next block's K comes in behind this block's softmax and P V
    more = rows_next(p, vis, w, warp);
    int64_t nrow = -1;
    if (more) {
      nrow = rows_block_row(p, w, kh);
      if (nrow >= 0) rows_load_k<Sh>(p, nrow, g, t, kr, ksz);
    }
    if (loaded) {
      const bool full = j0 >= lo && j0 + ROWS_BLK <= hi && kp0 + ROWS_BLK - 1 <= vis.min_pos &&
                        (p.window == 0 || kp0 > vis.max_pos - p.window || kp0 + ROWS_BLK <= p.sinks);
      uint32_t seen = ~0u;  // bit 4 nt + e: score e of tile nt
      if (!full) {
        seen = 0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + g + 8 * (e >> 1), kp = kp0 + g + 8 * (e >> 1), rp = rpos[nt][e & 1];
            const bool ok = j >= lo && j < hi && kp <= rp && (p.window == 0 || rp - kp < p.window || kp < p.sinks);
            if (!ok) s[nt][e] = -INFINITY;
            seen |= (ok ? 1u : 0u) << (4 * nt + e);
          }
        // keys no row sees (slots outside the segment among them) may hold anything
        if constexpr (Sh::Q4) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int j = j0 + g + 8 * r;
            if (j < lo || j >= hi) {
#pragma unroll
              for (int h = 0; h < GR; ++h) vsz[r * GR + h] = 0u;
            }
          }
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = j0 + 2 * t + (r & 1) + 8 * (r >> 1);
            if (j < lo || j >= hi) {
#pragma unroll
              for (int k = 0; k < 4 * Sh::NV; ++k) vr[r * 4 * Sh::NV + k] = 0u;
            }
          }
        }
      }
      // running maxima move only when a score passes one by 2^8 (then P stays below 2^8 in its 16-bit type)
      bool over = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) over |= fmaxf(s[nt][c], s[nt][2 + c]) > m[nt][c] + 8.f;
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(m[nt][c], fmaxf(s[nt][c], s[nt][2 + c]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float corr = mx == -INFINITY ? 1.f : ex2(m[nt][c] - mx);
            m[nt][c] = mx;
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
      uint32_t pb[NT][GR][2];
      if constexpr (Sh::Q4) {
        float sv[2][GR], zv[2][GR];
        float big = 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int h = 0; h < GR; ++h) {
            sv[r][h] = kv4_scale(vsz[r * GR + h]);
            zv[r][h] = fmaf(8.f, sv[r][h], kv4_offset(vsz[r * GR + h]));  // the value of code 8
            big = fmaxf(big, fmaxf(sv[r][h], fabsf(zv[r][h])));
          }
        if (__any_sync(0xffffffffu, big * vdown > 16.f)) {
          big = warp_max(big);
          const int e = min((int)(__float_as_uint(big) >> 23) - 127, 120);
          const float nd = __int_as_float((127 - e) << 23), f = nd / vdown;
          vdown = nd;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int e4 = 0; e4 < 4; ++e4) acc[nt][i][e4] *= f;
#pragma unroll
            for (int h = 0; h < GR; ++h) {
              rest[nt][h][0] *= f;
              rest[nt][h][1] *= f;
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int h = 0; h < GR; ++h) {
            sv[r][h] *= vdown;
            zv[r][h] *= vdown;
          }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float base = m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1];
            pr[e] = ex2(s[nt][e] - base);
            l[nt][e & 1] += pr[e];
          }
#pragma unroll
          for (int h = 0; h < GR; ++h) {
            float ps[4], pz[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              ps[e] = pr[e] * sv[e >> 1][h];
              pz[e] = pr[e] * zv[e >> 1][h];
            }
            if (!full) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!((seen >> (4 * nt + e)) & 1)) ps[e] = pz[e] = 0.f;  // 0 times NaN would not be 0
            }
            rest[nt][h][0] += pz[0] + pz[2];
            rest[nt][h][1] += pz[1] + pz[3];
            const uint32_t q0 = pack_f16(ps[0], ps[1]), q1 = pack_f16(ps[2], ps[3]);
            pb[nt][h][0] = movmatrix_t(q0);
            pb[nt][h][1] = movmatrix_t(q1);
          }
        }
#pragma unroll
        for (int k = 0; k < Sh::NV; ++k) {
          const uint32_t x0 = __byte_perm(vr[k], vr[Sh::NV + k], 0x5410);
          const uint32_t y0 = __byte_perm(vr[k], vr[Sh::NV + k], 0x7632);
          const uint32_t x1 = __byte_perm(vr[2 * Sh::NV + k], vr[3 * Sh::NV + k], 0x5410);
          const uint32_t y1 = __byte_perm(vr[2 * Sh::NV + k], vr[3 * Sh::NV + k], 0x7632);
          const uint32_t u[4] = {x0, x0 >> 8, y0, y0 >> 8}, v[4] = {x1, x1 >> 8, y1, y1 >> 8};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a[4] = {nib_lo8(u[i]), nib_hi8(u[i]), nib_lo8(v[i]), nib_hi8(v[i])};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816_f16(acc[nt][k * 4 + i], a, pb[nt][Sh::group(k)][0], pb[nt][Sh::group(k)][1]);
          }
        }
      } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float base = m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1];
            pr[e] = ex2(s[nt][e] - base);
            l[nt][e & 1] += pr[e];
          }
          pb[nt][0][0] = movmatrix_t(pack_bf16(pr[0], pr[1]));
          pb[nt][0][1] = movmatrix_t(pack_bf16(pr[2], pr[3]));
        }
#pragma unroll
        for (int k = 0; k < Sh::NV; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w0 = vr[k * 4 + i], w1 = vr[(Sh::NV + k) * 4 + i];
            const uint32_t w2 = vr[(2 * Sh::NV + k) * 4 + i], w3 = vr[(3 * Sh::NV + k) * 4 + i];
            const uint32_t a[4] = {__byte_perm(w0, w1, 0x5410), __byte_perm(w0, w1, 0x7632),
                                   __byte_perm(w2, w3, 0x5410), __byte_perm(w2, w3, 0x7632)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(acc[nt][k * 4 + i], a, pb[nt][0][0], pb[nt][0][1]);
          }
      }
    }
    row = nrow;
    if (more && row >= 0) rows_load_v<Sh>(p, row + (int64_t)p.Hkv * p.PS, g, t, vr, vsz);
  }

  // ---- join the warps of the CTA, then the CTAs of the cluster
  __syncthreads();  // the query fragments' space becomes [warp][row][LD] partial outputs
  float* aw = reinterpret_cast<float*>(sm_raw);
  const float up = 1.f / vdown;
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
        s_m[warp][r] = m[nt][c];
        s_l[warp][r] = sum;
      }
      float* dst = aw + (warp * Sh::ROWS + r) * Sh::LD;
#pragma unroll
      for (int k = 0; k < Sh::NV; ++k) {
        float o8[8];
        constexpr int one = GR - 1;  // group of V word k: k with two groups, 0 with one
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o8[2 * i] = acc[nt][k * 4 + i][c];
          o8[2 * i + 1] = acc[nt][k * 4 + i][2 + c];
        }
        if constexpr (Sh::Q4) {
#pragma unroll
          for (int i = 0; i < 8; ++i) o8[i] = (o8[i] + rest[nt][k & one][c]) * up;
        }
        *reinterpret_cast<float4*>(dst + Sh::v_dim(k, g)) = make_float4(o8[0], o8[1], o8[2], o8[3]);
        *reinterpret_cast<float4*>(dst + Sh::v_dim(k, g) + 4) = make_float4(o8[4], o8[5], o8[6], o8[7]);
      }
    }
  __syncthreads();
  constexpr int C4 = D / 4;
  const auto store = [&](int r, int d, float4 o, float inv) {
    const int rr = row0 + r;
    __nv_bfloat16* dst = p.out + ((int64_t)(t0 + rr / p.G) * p.Hq + kh * p.G + rr % p.G) * D + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
  };
  for (int i = threadIdx.x; i < nrows * C4; i += 32 * ROWS_WARPS) {
    const int r = i / C4, d = (i % C4) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int q = 0; q < ROWS_WARPS; ++q) M = fmaxf(M, s_m[q][r]);
    float L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 0; q < ROWS_WARPS; ++q) {
      if (s_m[q][r] == -INFINITY) continue;
      const float e = ex2(s_m[q][r] - M);
      L += s_l[q][r] * e;
      const float4 a = *reinterpret_cast<const float4*>(aw + (q * Sh::ROWS + r) * Sh::LD + d);
      o.x += a.x * e;
      o.y += a.y * e;
      o.z += a.z * e;
      o.w += a.w * e;
    }
    if (S == 1) {
      store(r, d, o, M == -INFINITY ? 0.f : 1.f / L);
    } else {
      *reinterpret_cast<float4*>(aw + r * Sh::LD + d) = o;  // slab 0: each element is read and written by this thread alone
      if (d == 0) {
        s_M[r] = M;
        s_L[r] = L;
      }
    }
  }
  if (S > 1) {
    cluster_sync_all();
    const uint32_t aw32 = smem_u32(aw), m32 = smem_u32(s_M), l32 = smem_u32(s_L);
    const auto ldf = [](uint32_t a) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
      return v;
    };
    for (int i = threadIdx.x + 32 * ROWS_WARPS * split; i < nrows * C4; i += 32 * ROWS_WARPS * S) {
      const int r = i / C4, d = (i % C4) * 4;
      float M = -INFINITY, L = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q0 = 0; q0 < S; q0 += 8) {  // the cluster's parts, eight in flight
        float mq[8], lq[8];
        float4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int q = min(q0 + u, S - 1);
          mq[u] = ldf(dsmem_map(m32 + 4 * r, q));
          lq[u] = ldf(dsmem_map(l32 + 4 * r, q));
          v[u] = dsmem_ld_f4(dsmem_map(aw32 + 4 * (r * Sh::LD + d), q));
          if (q0 + u >= S) mq[u] = -INFINITY;
        }
        float mx = M;
#pragma unroll
        for (int u = 0; u < 8; ++u) mx = fmaxf(mx, mq[u]);
        if (mx == -INFINITY) continue;
        const float f = ex2(M - mx);
        M = mx;
        L *= f;
        o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          if (mq[u] == -INFINITY) continue;
          const float e = ex2(mq[u] - mx);
          L += lq[u] * e;
          o.x += v[u].x * e;
          o.y += v[u].y * e;
          o.z += v[u].z * e;
          o.w += v[u].w * e;
        }
      }
      store(r, d, o, M == -INFINITY ? 0.f : 1.f / L);
    }
    cluster_sync_all();  // no CTA leaves while another reads its shared memory
  }
  if (threadIdx.x == 0) span_end(p.span);
}

// ------------------------------------------------------------------ host
int gemm_num_sms();
unsigned long long* next_span(const char* name);
void kv4_check_layer(const torch::Tensor& codes, const torch::Tensor& scales, const char* who);

template <int D, int BITS, int NT, int OCC>
static void launch_rows(RowsParams& p, int64_t num_seqs, int64_t max_q, int64_t max_keys, cudaStream_t st) {
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
  const int64_t work = tiles * num_seqs * p.Hkv;
  // Key parts per tile: enough CTAs for four per SM and resident slot, each
  // with at least 128 keys; a power of two up to the 16 CTAs of a cluster.
  int S = 1;
  while (S < 16 && work * S < (int64_t)OCC * gemm_num_sms() * 2 && max_keys >= (int64_t)S * 2 * 128) S *= 2;
  p.splits = S;
  TORCH_CHECK(tiles < (1ll << 31) && num_seqs <= 65535 && (int64_t)p.Hkv * S <= 65535, "attention: launch grid too large");
  launch_pdl_cluster(k, dim3((unsigned)tiles, (unsigned)num_seqs, (unsigned)(p.Hkv * S)), dim3(32 * ROWS_WARPS),
                     Sh::SMEM, st, dim3(1, 1, (unsigned)S), p);
}

// Attention of few rows over a bf16 layer pool (`kv`, `scales` undefined) or a
// 4-bit layer (`kv` = codes), with an optional window.
void attention_rows(torch::Tensor out, torch::Tensor q, torch::Tensor kv, c10::optional<torch::Tensor> scales,
                    torch::Tensor qo_indptr, torch::Tensor positions, torch::Tensor seg_indptr,
                    torch::Tensor seg_page_indptr, torch::Tensor seg_offset, torch::Tensor seg_len,
                    torch::Tensor seg_pos0, torch::Tensor seg_delta, torch::Tensor page_ids, torch::Tensor cos,
                    torch::Tensor sin, double scale, bool use_rope, int64_t num_seqs, int64_t max_q_len,
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
  }
  TORCH_CHECK(kv.device() == dev && out.device() == dev, "attention: q, cache and out on different devices");
  const int64_t Hkv = kv.size(2), PS = kv.size(3);
  TORCH_CHECK(kv.size(4) == (q4 ? D / 2 : D) && Hkv > 0 && Hq % Hkv == 0, "attention: head layout mismatch");
  TORCH_CHECK(PS > 0 && PS % 16 == 0, "attention: page size must be a multiple of 16");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.is_contiguous() && out.numel() == T * Hq * D,
              "attention: out must be a contiguous bf16 [T, Hq * D]");
  TORCH_CHECK(window >= 0 && window < (1ll << 30) && sinks >= 0 && sinks < (1ll << 30),
              "attention: window and sinks must be in [0, 2^30)");
  TORCH_CHECK(num_seqs >= 0 && max_q_len >= 0 && max_q_len <= T, "attention: max_q_len must be in [0, T]");
  if (T == 0 || num_seqs == 0 || max_q_len == 0) return;
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
                    cos.size(1) == D / 2 && cos.size(0) >= 1 && sin.sizes() == cos.sizes(),
                "attention: cos and sin must be contiguous fp32 [positions, D/2] tables on the device of the cache");
    p.cos = cos.data_ptr<float>();
    p.sin = sin.data_ptr<float>();
    p.rope_len = (int)cos.size(0);
  }
  p.use_rope = use_rope ? 1 : 0;
  p.scale_log2 = (float)scale * LOG2E;
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.G = (int)(Hq / Hkv);
  p.PS = (int)PS;
  p.num_pages = (int)kv.size(0);
  p.window = (int)window;
  p.sinks = (int)sinks;
  const at::cuda::CUDAGuard guard(dev);
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  p.span = next_span("attn_rows");
  int64_t keys = std::max<int64_t>(1, max_kv_len);
  if (window > 0) keys = std::min(keys, window + sinks + max_q_len);
  const int64_t rows = max_q_len * p.G;
  const auto pick = [&](auto d, auto bits) {
    constexpr int DD = decltype(d)::value, BB = decltype(bits)::value;
    if (rows <= 8)
      launch_rows<DD, BB, 1, BB == 4 ? 4 : 3>(p, num_seqs, max_q_len, keys, st);
    else if (rows <= 16 || (DD == 128 && BB == 16))
      launch_rows<DD, BB, 2, BB == 4 ? 3 : 2>(p, num_seqs, max_q_len, keys, st);
    else if constexpr (DD == 64 || BB == 4)
      launch_rows<DD, BB, 4, 2>(p, num_seqs, max_q_len, keys, st);
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
}

BRAID_BOUNDS_READER(bounds_status_attention_rows)

}  // namespace braid
