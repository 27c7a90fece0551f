// Append to and read-back from the 4-bit paged KV cache (layout in kv4.cuh).
//
// qkv_prepare_kv4: one pass over a step's QKV rows: per-head q/k RMSNorm,
// RoPE(k), per-group minimum and maximum, codes and scales stored at the
// token's slot.  Everything from the bf16 input to the code is fp32; the only
// roundings are those the format defines and, for a normalised q, one to bf16.
// Measured on a B200: 8191 tokens of 16 query and 8 KV heads of 128 with norms
// 40 us (110 MB: 2.7 TB/s; bound by issue, 76% of cycles: norm, rotation and
// quantisation), read-back of the same tokens 12 us.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "attention_rows.cuh"
#include "common.cuh"
#include "kv4.cuh"
#include "launch.cuh"

namespace braid {

unsigned long long* next_span(const char* name);
int gemm_num_sms();

// n / d of 0 <= n < 2^31 by a multiplication: m = ceil(2^(31 + k) / d) with 2^k >= d.
struct FastDiv {
  unsigned d, m, shift;
  explicit FastDiv(unsigned div = 1) : d(div), m(0), shift(0) {
    unsigned k = 0;
    while ((1ull << k) < div) ++k;
    m = (unsigned)(((1ull << (31 + k)) + div - 1) / div);
    shift = k;
  }
  BRAID_DEVICE unsigned div(unsigned n) const { return (unsigned)(((uint64_t)n * m) >> 31) >> shift; }
};

struct Kv4AppendParams {
  const __nv_bfloat16* qkv;  // [T, ld] rows of (Hq + 2 Hkv) heads
  __nv_bfloat16* q_out;      // [T, Hq, D], written only with a q norm
  uint32_t* codes;           // layer codes as words
  uint32_t* scales;          // layer (s, z) pairs
  const int* positions;
  const int* slots;
  const __nv_bfloat16* qn;   // nullptr: no norm
  const __nv_bfloat16* kn;
  const float* cos;
  const float* sin;
  float eps;
  int64_t ld;
  unsigned items;            // T * heads handled
  FastDiv heads;             // handled per token: 2 Hkv, or Hq + 2 Hkv with a q norm
  FastDiv page;              // slots of a page
  int Hq, Hkv, use_rope, num_slots, rope_len;
  unsigned long long* span;
};

BRAID_DEVICE void unpack8(uint4 u, float* v) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
  }
}
BRAID_DEVICE uint4 pack8(const float* v) {
  return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

// Eight codes round((v - z) / s), ties to even, clamped to 0..15.  bf16 inputs
// put many quotients exactly on a tie, so a product with 1 / s alone would often
// fall to the wrong side.  It gives a candidate c within one of the answer; its
// residual d - c s (c s has 12 bits and is exact) then decides as the exact
// quotient would: beyond half a step, or on it with c odd, c moves by one.
BRAID_DEVICE uint32_t kv4_codes(const float* v, float s, float z) {
  const float r = __fdividef(1.f, s);
  float c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float d = __fsub_rn(v[j], z);
    const float t = fmaf(d, r, 12582912.f);  // the integer lands in the low bits of the sum
    c[j] = t - 12582912.f;
    const float e = fmaf(-c[j], s, d), h = fabsf(e + e);
    if (h > s || (h == s && (__float_as_uint(t) & 1u))) c[j] += e > 0.f ? 1.f : -1.f;
    c[j] = fminf(fmaxf(c[j], 0.f), 15.f);
  }
  const float lo = fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]);
  const float hi = fmaf(fmaf(fmaf(c[7], 16.f, c[6]), 16.f, c[5]), 16.f, c[4]);
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// D / 8 lanes per (token, head), 8 elements (one 16-byte load, one code word)
// per lane; the rotary partner of a lane's elements is D / 16 lanes away, and
// 8 neighbouring lanes hold one group of 64.  U items per thread, all loads of
// them issued first.  Lanes past the last item stay for the shuffles and touch
// no memory.
template <int D, int U>
__global__ void __launch_bounds__(256) qkv_prepare_kv4_kernel(const Kv4AppendParams p) {
  constexpr int LPH = D / 8, IPB = 256 / LPH;
  if (threadIdx.x == 0) span_start(p.span);
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) span_waited(p.span);
  const int l = threadIdx.x % LPH;
  const unsigned first = blockIdx.x * (IPB * U) + threadIdx.x / LPH;
  unsigned tok[U];
  int head[U], slot[U], pos[U];
  uint4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned item = first + u * IPB;
    const bool live = item < p.items;
    tok[u] = live ? p.heads.div(item) : 0u;
    head[u] = live ? (int)(item - tok[u] * p.heads.d) + (p.Hq + 2 * p.Hkv - (int)p.heads.d) : -1;  // within the QKV row
    raw[u] = make_uint4(0, 0, 0, 0);
    slot[u] = -1;
    pos[u] = 0;
    if (live) {
      raw[u] = *reinterpret_cast<const uint4*>(p.qkv + (int64_t)tok[u] * p.ld + (int64_t)head[u] * D + l * 8);
      if (head[u] >= p.Hq) {
        slot[u] = p.slots[tok[u]];
        if (p.use_rope) pos[u] = p.positions[tok[u]];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool live = head[u] >= 0, is_q = live && head[u] < p.Hq, is_k = head[u] >= p.Hq && head[u] < p.Hq + p.Hkv;
    float v[8];
    unpack8(raw[u], v);
    const __nv_bfloat16* nw = is_q ? p.qn : (is_k ? p.kn : nullptr);
    if (__any_sync(0xffffffffu, nw != nullptr)) {
      // Squares rounded, then summed by halves: of the fours of neighbours (D 128) or of the elements (D 64), the upper
      // half onto the lower until one is left, the order of a plain strided reduction; the last steps are in the lane.
      float sq[8], ss;
#pragma unroll
      for (int j = 0; j < 8; ++j) sq[j] = __fmul_rn(v[j], v[j]);
      if constexpr (D == 128) {
        float a = ((sq[0] + sq[1]) + sq[2]) + sq[3], b = ((sq[4] + sq[5]) + sq[6]) + sq[7];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) {
          a += __shfl_xor_sync(0xffffffffu, a, o);
          b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        ss = a + b;
      } else {
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1)
#pragma unroll
          for (int j = 0; j < 8; ++j) sq[j] += __shfl_xor_sync(0xffffffffu, sq[j], o);
        ss = ((sq[0] + sq[4]) + (sq[2] + sq[6])) + ((sq[1] + sq[5]) + (sq[3] + sq[7]));
      }
      if (nw != nullptr) {
        const float rstd = rsqrtf(ss / D + p.eps);
        float wt[8];
        unpack8(*reinterpret_cast<const uint4*>(nw + l * 8), wt);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(__fmul_rn(v[j], rstd), wt[j]);
      }
    }
    if (is_q) *reinterpret_cast<uint4*>(p.q_out + ((int64_t)tok[u] * p.Hq + head[u]) * D + l * 8) = pack8(v);
    if (__all_sync(0xffffffffu, head[u] < p.Hq)) continue;  // nothing of this warp goes into the cache
    if (p.use_rope && __any_sync(0xffffffffu, is_k)) {
      float partner[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) partner[j] = __shfl_xor_sync(0xffffffffu, v[j], LPH / 2);
      if (is_k) {
        (void)BRAID_IN_BOUNDS(pos[u] >= 0 && pos[u] < p.rope_len, 2, pos[u]);
        const int64_t at = (int64_t)min(max(pos[u], 0), p.rope_len - 1) * (D / 2) + (l % (LPH / 2)) * 8;
        const unsigned flip = l < LPH / 2 ? 0x80000000u : 0u;  // the first half subtracts
        float cs[8], sn[8];
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          *reinterpret_cast<float4*>(cs + j) = *reinterpret_cast<const float4*>(p.cos + at + j);
          *reinterpret_cast<float4*>(sn + j) = *reinterpret_cast<const float4*>(p.sin + at + j);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)  // each product and the sum rounded on its own: codes at a border fall as in any fp32 form
          v[j] = __fadd_rn(__fmul_rn(v[j], cs[j]),
                           __uint_as_float(__float_as_uint(__fmul_rn(partner[j], sn[j])) ^ flip));
      }
    }
    float mn = v[0], mx = v[0], bad = v[0] * 0.f;  // bad: 0, or NaN once an element is not finite
#pragma unroll
    for (int j = 1; j < 8; ++j) {
      mn = fminf(mn, v[j]);
      mx = fmaxf(mx, v[j]);
      bad = fmaf(v[j], 0.f, bad);
    }
    if (bad != 0.f) mx = INFINITY;  // the group's range is then infinite
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    if (live && !is_q && BRAID_IN_BOUNDS(slot[u] >= 0 && slot[u] < p.num_slots, 1, slot[u]) && slot[u] >= 0 &&
        slot[u] < p.num_slots) {
      // mx - mn passes the fp32 range only for values of magnitude above 1.7e38; such a group counts as not finite
      const float range = mx - mn;
      const bool fine = range <= 3.4e38f;
      const __nv_bfloat16 sb = f2bf(fine ? __fmul_rn(range, 1.f / 15.f) : __int_as_float(0x7fc00000));
      const __nv_bfloat16 zb = f2bf(fine ? mn : __int_as_float(0x7fc00000));
      const float s = bf2f(sb), z = bf2f(zb);
      uint32_t word = 0;
      if (fine && s > 0.f) word = kv4_codes(v, s, z);
      const unsigned page = p.page.div((unsigned)slot[u]), off = (unsigned)slot[u] - page * p.page.d;
      const int kvh = head[u] - p.Hq;  // K heads, then V heads: the cache's order
      const int64_t row = (int64_t)(page * 2 * p.Hkv + kvh) * p.page.d + off;  // page * heads: below 2^31 rows
      p.codes[row * (D / 8) + kv4_word<D>(l)] = word;
      if (l % 8 == 0)
        p.scales[row * (D / KV4_GROUP) + l / 8] =
            (uint32_t)__bfloat16_as_ushort(sb) | ((uint32_t)__bfloat16_as_ushort(zb) << 16);
    }
  }
  if (threadIdx.x == 0) span_end(p.span);
}

// Values 8 l .. 8 l + 7 of a cache row from its code word and group pair, as bf16.
BRAID_DEVICE uint4 kv4_values(uint32_t w, uint32_t sz) {
  const float s = kv4_scale(sz), z = kv4_offset(sz);
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)  // 2^23 + c by its bits, then c exactly (a conversion would take the slow unit)
    v[j] = fmaf(s, __uint_as_float(((w >> (4 * j)) & 15u) | 0x4B000000u) - 8388608.f, z);
  return pack8(v);
}

// out[t, kv, head, :] = the values held at slots[t]; zeros for a slot outside the cache.
template <int D, int U>
__global__ void __launch_bounds__(256) kv4_read_kernel(__nv_bfloat16* out, const uint32_t* codes,
                                                       const uint32_t* scales, const int* slots, unsigned items,
                                                       FastDiv heads, FastDiv page_div,
                                                       int num_slots) {
  constexpr int LPH = D / 8, IPB = 256 / LPH;
  pdl_trigger();
  pdl_wait();
  const int l = threadIdx.x % LPH;
  const unsigned first = blockIdx.x * (IPB * U) + threadIdx.x / LPH;
  uint32_t w[U], sz[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned item = first + u * IPB;
    w[u] = sz[u] = 0u;  // stands for zeros
    if (item < items) {
      const unsigned t = heads.div(item);
      const int slot = slots[t];
      if (BRAID_IN_BOUNDS(slot >= 0 && slot < num_slots, 1, slot) && slot >= 0 && slot < num_slots) {
        const unsigned page = page_div.div((unsigned)slot), off = (unsigned)slot - page * page_div.d;
        const int64_t row = (int64_t)(page * heads.d + (item - t * heads.d)) * page_div.d + off;
        w[u] = codes[row * (D / 8) + kv4_word<D>(l)];
        sz[u] = scales[row * (D / KV4_GROUP) + l / 8];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned item = first + u * IPB;
    if (item < items) *reinterpret_cast<uint4*>(out + (int64_t)item * D + l * 8) = kv4_values(w[u], sz[u]);
  }
}

// Page i of the plan's list as bf16 page i of `out` [NP, 2, Hkv, PS, D], for the long-prompt attention: the slots of its
// segment that some query of the sequence sees (the others, which may hold anything, become 0).  Pages that no query
// sees are skipped: the attention does not read them.  One block per (page, K/V and head).
template <int D>
__global__ void __launch_bounds__(256) kv4_unpack_pages_kernel(__nv_bfloat16* out, const RowsParams p,
                                                               int num_seqs) {
  constexpr int LPR = D / 8;
  __shared__ int s_seg, s_seq, s_min, s_max;
  const int i = blockIdx.x;
  if (threadIdx.x == 0) {
    s_seg = s_seq = -1;
    s_min = INT_MAX;
    s_max = -1;
  }
  pdl_trigger();
  pdl_wait();
  __syncthreads();
  const int segs = p.seg_indptr[num_seqs];
  for (int s = threadIdx.x; s < segs; s += 256)
    if (p.seg_page_indptr[s] <= i && i < p.seg_page_indptr[s + 1]) s_seg = s;
  __syncthreads();
  const int s = s_seg;
  if (s < 0) return;
  for (int b = threadIdx.x; b < num_seqs; b += 256)
    if (p.seg_indptr[b] <= s && s < p.seg_indptr[b + 1]) s_seq = b;
  __syncthreads();
  if (s_seq < 0) return;
  int mn = INT_MAX, mx = -1;
  for (int t = p.qo_indptr[s_seq] + threadIdx.x; t < p.qo_indptr[s_seq + 1]; t += 256) {
    mn = min(mn, p.positions[t]);
    mx = max(mx, p.positions[t]);
  }
  mn = __reduce_min_sync(0xffffffffu, mn);
  mx = __reduce_max_sync(0xffffffffu, mx);
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&s_min, mn);
    atomicMax(&s_max, mx);
  }
  __syncthreads();
  const int off = p.seg_offset[s], len = p.seg_len[s], pos0 = p.seg_pos0[s];
  const int slot0 = (i - p.seg_page_indptr[s]) * p.PS;  // of the segment's pages
  // keys of this page, and those of them that lie in front of every query's window and behind the sinks or after them all
  const int a = max(slot0 - off, 0), b = min(slot0 + p.PS - off, len);
  if (a >= b || pos0 + a > s_max) return;
  if (p.window > 0 && pos0 + b - 1 <= s_min - p.window && pos0 + a >= p.sinks) return;
  const int page = min(max(p.page_ids[i], 0), p.num_pages - 1);
  (void)BRAID_IN_BOUNDS(p.page_ids[i] >= 0 && p.page_ids[i] < p.num_pages, 4, p.page_ids[i]);
  const int kvh = blockIdx.y;
  const int64_t src = ((int64_t)page * 2 * p.Hkv + kvh) * p.PS, dst = ((int64_t)i * 2 * p.Hkv + kvh) * p.PS;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(p.kv);
  for (int e = threadIdx.x; e < p.PS * LPR; e += 256) {
    const int r = e / LPR, l = e % LPR;
    uint4 o = make_uint4(0, 0, 0, 0);
    if (slot0 + r - off >= a && slot0 + r - off < b) o = kv4_values(codes[(src + r) * (D / 8) + kv4_word<D>(l)], p.scales[(src + r) * (D / KV4_GROUP) + l / 8]);
    *reinterpret_cast<uint4*>(out + (dst + r) * D + l * 8) = o;
  }
}

// ------------------------------------------------------------------ host
void kv4_unpack_pages(torch::Tensor out, const torch::Tensor& codes, const torch::Tensor& scales, const RowsParams& p,
                      int64_t num_seqs, cudaStream_t st) {
  TORCH_CHECK(codes.size(4) == 64 && out.is_contiguous() && out.scalar_type() == at::kBFloat16, "attention: unpack");
  launch_pdl(kv4_unpack_pages_kernel<128>, dim3((unsigned)out.size(0), (unsigned)(2 * p.Hkv)), dim3(256), 0, st,
             reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), p, (int)num_seqs);
}

void kv4_check_layer(const torch::Tensor& codes, const torch::Tensor& scales, const char* who) {
  TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == at::kByte && codes.dim() == 5 && codes.is_contiguous(), who,
              ": 4-bit cache codes must be a contiguous CUDA uint8 tensor [P, 2, Hkv, page, D/2]");
  TORCH_CHECK(scales.is_cuda() && scales.scalar_type() == at::kBFloat16 && scales.dim() == 6 && scales.is_contiguous(),
              who, ": 4-bit cache scales must be a contiguous CUDA bf16 tensor [P, 2, Hkv, page, D/64, 2]");
  TORCH_CHECK(scales.device() == codes.device(), who, ": codes and scales on different devices");
  const int64_t D = codes.size(4) * 2;
  TORCH_CHECK(D == 64 || D == 128, who, ": 4-bit cache head_dim must be 64 or 128");
  TORCH_CHECK(codes.size(2) > 0, who, ": 4-bit cache without KV heads");
  TORCH_CHECK(codes.size(1) == 2 && scales.size(0) == codes.size(0) && scales.size(1) == 2 &&
                  scales.size(2) == codes.size(2) && scales.size(3) == codes.size(3) &&
                  scales.size(4) == D / KV4_GROUP && scales.size(5) == 2,
              who, ": 4-bit cache codes and scales do not match");
  TORCH_CHECK(codes.size(3) > 0 && codes.size(0) * codes.size(3) < (1ll << 31) &&
                  codes.size(0) * 2 * codes.size(2) < (1ll << 31),
              who, ": more than 2^31 slots or (page, head) slabs");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(scales.data_ptr()) % 16 == 0,
              who, ": 4-bit cache tensors must be 16-byte aligned");
}

static void check_i32(const torch::Tensor& t, int64_t n, const torch::Device& dev, const char* who, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous() && t.device() == dev && t.numel() >= n, who, ": ", name,
              " must be a contiguous int32 tensor of at least ", std::to_string(n), " elements on the device of the cache");
}

// Returns q [T, Hq, D]: the normalised queries, or without a q norm their columns of qkv.
torch::Tensor qkv_prepare_kv4(const torch::Tensor& qkv, const torch::Tensor& positions, const torch::Tensor& slots,
                              const torch::Tensor& codes, const torch::Tensor& scales,
                              const c10::optional<torch::Tensor>& q_norm, const c10::optional<torch::Tensor>& k_norm,
                              double eps, const torch::Tensor& cos, const torch::Tensor& sin, int64_t Hq, int64_t Hkv,
                              int64_t D, bool use_rope) {
  const char* who = "qkv_prepare";
  kv4_check_layer(codes, scales, who);
  const auto dev = codes.device();
  TORCH_CHECK(qkv.is_cuda() && qkv.device() == dev && qkv.scalar_type() == at::kBFloat16 && qkv.dim() == 2 &&
                  qkv.size(1) == (Hq + 2 * Hkv) * D && qkv.stride(1) == 1 && qkv.stride(0) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0,
              who, ": qkv must be a bf16 [T, (Hq + 2 Hkv) D] tensor with 16-byte aligned rows on the device of the cache");
  TORCH_CHECK(Hq >= 0 && codes.size(2) == Hkv && codes.size(4) * 2 == D, who, ": cache layout mismatch");
  const int64_t T = qkv.size(0);
  const bool has_qn = q_norm.has_value() && q_norm->defined(), has_kn = k_norm.has_value() && k_norm->defined();
  const at::cuda::CUDAGuard g(dev);
  const torch::Tensor q_out =
      has_qn ? at::empty({T, Hq, D}, qkv.options()) : qkv.as_strided({T, Hq, D}, {qkv.stride(0), D, 1});
  if (T == 0) return q_out;
  check_i32(positions, T, dev, who, "positions");
  check_i32(slots, T, dev, who, "slots");
  for (const auto* w : {has_qn ? &*q_norm : nullptr, has_kn ? &*k_norm : nullptr})
    if (w != nullptr)
      TORCH_CHECK(w->device() == dev && w->scalar_type() == at::kBFloat16 && w->numel() == D && w->is_contiguous() &&
                      reinterpret_cast<uintptr_t>(w->data_ptr()) % 16 == 0,
                  who, ": norm weights must be contiguous, 16-byte aligned bf16 [D] on the device of the cache");
  if (use_rope)
    TORCH_CHECK(cos.device() == dev && sin.device() == dev && cos.scalar_type() == at::kFloat &&
                    sin.scalar_type() == at::kFloat && cos.is_contiguous() && sin.is_contiguous() && cos.dim() == 2 &&
                    cos.size(1) == D / 2 && cos.size(0) >= 1 && sin.sizes() == cos.sizes() &&
                    reinterpret_cast<uintptr_t>(cos.data_ptr()) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(sin.data_ptr()) % 16 == 0,
                who, ": cos and sin must be contiguous, 16-byte aligned fp32 [positions, D/2] tables on the device of the cache");
  Kv4AppendParams p{};
  p.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv.data_ptr());
  p.q_out = has_qn ? reinterpret_cast<__nv_bfloat16*>(q_out.data_ptr()) : nullptr;
  p.codes = reinterpret_cast<uint32_t*>(codes.data_ptr());
  p.scales = reinterpret_cast<uint32_t*>(scales.data_ptr());
  p.positions = positions.data_ptr<int>();
  p.slots = slots.data_ptr<int>();
  p.qn = has_qn ? reinterpret_cast<const __nv_bfloat16*>(q_norm->data_ptr()) : nullptr;
  p.kn = has_kn ? reinterpret_cast<const __nv_bfloat16*>(k_norm->data_ptr()) : nullptr;
  p.cos = use_rope ? cos.data_ptr<float>() : nullptr;
  p.sin = use_rope ? sin.data_ptr<float>() : nullptr;
  p.eps = (float)eps;
  p.ld = qkv.stride(0);
  p.heads = FastDiv((unsigned)(2 * Hkv + (has_qn ? Hq : 0)));
  p.page = FastDiv((unsigned)codes.size(3));
  TORCH_CHECK(T * p.heads.d < (1ll << 31), who, ": more than 2^31 (token, head) rows");
  p.items = (unsigned)(T * p.heads.d);
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.use_rope = use_rope ? 1 : 0;
  p.num_slots = (int)(codes.size(0) * codes.size(3));
  p.rope_len = use_rope ? (int)cos.size(0) : 1;
  p.span = next_span("qkv_prepare_kv4");
  auto st = at::cuda::getCurrentCUDAStream();
  const auto go = [&](auto k, unsigned per_block) {
    launch_pdl(k, dim3((p.items + per_block - 1) / per_block), dim3(256), 0, st, p);
  };
  // several items a thread once one each fills the SMs' resident blocks (8 of 256 threads) twice
  const unsigned ipb = (unsigned)(256 / (D / 8));
  const bool many = p.items >= ipb * 16 * (unsigned)gemm_num_sms();
  if (D == 128)
    many ? go(qkv_prepare_kv4_kernel<128, 4>, 4 * ipb) : go(qkv_prepare_kv4_kernel<128, 1>, ipb);
  else
    many ? go(qkv_prepare_kv4_kernel<64, 4>, 4 * ipb) : go(qkv_prepare_kv4_kernel<64, 1>, ipb);
  return q_out;
}

// bf16 [T, 2, Hkv, D] of what the cache holds at `slots`.
torch::Tensor kv4_read(const torch::Tensor& codes, const torch::Tensor& scales, const torch::Tensor& slots) {
  const char* who = "kv4_read";
  kv4_check_layer(codes, scales, who);
  const int64_t T = slots.numel(), Hkv = codes.size(2), PS = codes.size(3), D = codes.size(4) * 2;
  const at::cuda::CUDAGuard g(codes.device());
  const torch::Tensor out = at::empty({T, 2, Hkv, D}, scales.options());
  if (T == 0) return out;
  check_i32(slots, T, codes.device(), who, "slots");
  TORCH_CHECK(T * 2 * Hkv < (1ll << 31), who, ": more than 2^31 (slot, head) rows");
  const unsigned items = (unsigned)(T * 2 * Hkv), ipb = (unsigned)(256 / (D / 8));
  auto st = at::cuda::getCurrentCUDAStream();
  const auto go = [&](auto k, unsigned per_block) {
    launch_pdl(k, dim3((items + per_block - 1) / per_block), dim3(256), 0, st,
               reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), reinterpret_cast<const uint32_t*>(codes.data_ptr()),
               reinterpret_cast<const uint32_t*>(scales.data_ptr()), (const int*)slots.data_ptr<int>(), items,
               FastDiv((unsigned)(2 * Hkv)), FastDiv((unsigned)PS), (int)(codes.size(0) * PS));
  };
  const bool many = items >= ipb * 16 * (unsigned)gemm_num_sms();
  if (D == 128)
    many ? go(kv4_read_kernel<128, 4>, 4 * ipb) : go(kv4_read_kernel<128, 1>, ipb);
  else
    many ? go(kv4_read_kernel<64, 4>, 4 * ipb) : go(kv4_read_kernel<64, 1>, ipb);
  return out;
}

BRAID_BOUNDS_READER(bounds_status_kv4)

}  // namespace braid
