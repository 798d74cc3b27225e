// tq_norm_write.hip -- the rows of a layer's fused projection to what its
// attention takes, in one pass: q and k heads normed and rotated, K and V
// quantised into the packed cache.
//
// A row of qkv holds Hq q heads, H k heads and H v heads of hd elements.  Per q
// and k head x (fp32 throughout):
//   n = x / sqrt(mean(x^2) + eps) * w          (no weights: n = x)
//   y_i        = n_i        c_i - n_{i+half} s_i
//   y_{i+half} = n_{i+half} c_i + n_i        s_i      0 <= i < half
//   y_d        = n_d                                  d >= 2 half
// with (c_i, s_i) = (cos, sin)[pos[axis(i)], i]: positions of several axes (time,
// height, width) share the pairs out in sections, one after the other.  y is
// rounded once, to the row's type; q and k rows leave as they are rounded, and
// the cache takes the rounded k and the v as they come, so its bytes are those
// of tq_quantize_write_kv_cache over these rows (tq_quant.h, the same kernel).
//
// A workgroup takes vectors of one kind.  K and V: 64 vectors (32 at pd 256), 32 dims per lane, chunks of 8 as
// the write has them; where half a rotation is a whole number of chunk rows (the
// whole head at every padded size, half of it at 128 and 256) a pair stands in
// one lane, else the partner chunk is read again (from L1).
// q: a wave takes heads of one token, one chunk of 8 dims per lane, so that every
// load and store is 1 KB of consecutive bytes and the token's angles and the
// weight are loaded once for 4 x (64 / lanes of a head) heads; the pair's partner
// comes from lane ^ (half / 8) by DPP where half / 8 is a power of two.
//
// Bound by memory at large counts: 8192 tokens, 32 / 8 heads of 128 (193 MB) 51 us,
// 3.8 TB/s against 5.1 of a large copy: q alone runs at 4.2, and K and V, whose
// VALU work the plain write does in 13 us, take 20.  In front of the present form:
// q heads in the write's layout and K and V first 54; two loads a q wave for four 54;
// angles of all of a lane's pairs at once (105 registers) 52.  One decode step of 8
// tokens 6.5 us, a chain of position, angles, norm and bucketize.
#include <algorithm>

#include "tq_quant.h"

namespace tq {
namespace {

constexpr int kMaxAxes = 4;

struct NormWriteParams {
  const uint16_t* qkv;
  int64_t row;  // elements from row to row
  const uint16_t* qw;
  const uint16_t* kw;
  float eps, inv_hd;
  const float* cos_t;
  const float* sin_t;
  int64_t trows;
  int half, axes;
  int ends[kMaxAxes];  // the first pair behind each axis' section
  const void* pos;
  int pos64;
  int64_t pos_st;  // entries from axis to axis
  uint8_t* ks;
  uint8_t* vs;
  const float* signs;
  const int32_t* slots;
  uint32_t tokens, mk, mg;  // ceil(2^32 / kv heads), ceil(2^32 / q groups)
  int qgroups;              // waves that share a token's q heads
  int hq, hkv, hd, ebs;
  int64_t nslots;
  float scale;
  uint16_t* q;
  uint16_t* k;
  uint32_t kblocks, share;  // K workgroups; ceil(2^32 * groups of K and V / all)
};

template <int DT>
__device__ __forceinline__ float elem(const u32x4& v, int c) {
  if constexpr (DT == TQ_BF16)
    return __uint_as_float(c & 1 ? v[c / 2] & 0xffff0000u : v[c / 2] << 16);
  return c & 1 ? hi_half_f(v[c / 2]) : lo_half_f(v[c / 2]);
}

// eight floats rounded to DT (to nearest even)
template <int DT>
__device__ __forceinline__ u32x4 round8(const float* y) {
  typedef float f8 __attribute__((ext_vector_type(8)));
  const f8 v = {y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]};
  if constexpr (DT == TQ_BF16) {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(u32x4, __builtin_convertvector(v, b8));
  } else {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(u32x4, __builtin_convertvector(v, h8));
  }
}

__device__ __forceinline__ void load8(const float* src, float* x) {
  const float4 a = *reinterpret_cast<const float4*>(src);
  const float4 b = *reinterpret_cast<const float4*>(src + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// (cos, sin) of pairs i .. i + 7 of token t; inside: cleared where a position
// has no table row (its reads go to row 0)
__device__ __forceinline__ void angles(const NormWriteParams& p, uint32_t t, int i, float* c,
                                       float* s, bool& inside) {
  auto row_of = [&](int axis) -> int64_t {
    const int64_t at = (int64_t)axis * p.pos_st + t;
    const int64_t r = p.pos64 ? static_cast<const int64_t*>(p.pos)[at]
                              : static_cast<const int32_t*>(p.pos)[at];
    const bool ok = r >= 0 && r < p.trows;
    inside = inside && ok;
    return ok ? r : 0;
  };
  auto axis_of = [&](int pair) -> int {
    int a = 0;
    for (int x = 0; x + 1 < p.axes; x++) a += pair >= p.ends[x] ? 1 : 0;
    return a;
  };
  const int first = axis_of(i);
  if (p.axes == 1 || first == axis_of(i + 7)) {
    const int64_t at = row_of(first) * p.half + i;
    load8(p.cos_t + at, c);
    load8(p.sin_t + at, s);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; e++) {  // a section ends inside the chunk
    const int64_t at = row_of(axis_of(i + e)) * p.half + i + e;
    c[e] = p.cos_t[at];
    s[e] = p.sin_t[at];
  }
}

// 1 / sqrt(mean of squares + eps) of a vector, sum_squares(f) the sum of its
// squares times f^2 on every lane of it
template <int DT, class Sum>
__device__ __forceinline__ float norm_scale(const NormWriteParams& p, Sum sum_squares) {
  const float ss = sum_squares(1.0f);
  float r = rsqrtf(__builtin_fmaf(ss, p.inv_hd, p.eps));
  if (DT == TQ_BF16 && __builtin_amdgcn_ballot_w64(ss == INFINITY) != 0) {
    // squares beyond fp32 of values within it: those of the row times 2^-70
    // (eps is nothing beside them)
    const float down = 0x1p-70f, s2 = sum_squares(down);
    if (ss == INFINITY) r = rsqrtf(s2 * p.inv_hd) * down;
  }
  return r;
}

constexpr int kQRounds = 4;  // heads of a q wave: so many loads of 64 lanes

// q heads of one token.  X: half a rotation in chunks where that is a power of
// two, 0: any.
template <int PD, int DT, int X>
__device__ __forceinline__ void q_rows(const NormWriteParams& p, uint32_t blk) {
  constexpr int L = PD / 8, R = 64 / L;  // lanes per head, heads per load
  const int lane = threadIdx.x & 63;
  const uint32_t wid = blk * 4u + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wid >= p.tokens * (uint32_t)p.qgroups) return;
  const uint32_t t = p.qgroups == 1 ? wid : __umulhi(wid, p.mg);
  const int c = lane % L, d = 8 * c;
  const int first = (int)(wid - t * (uint32_t)p.qgroups) * (R * kQRounds);  // (uniform)
  const int h0 = first + lane / L;
  u32x4 raw[kQRounds];
#pragma unroll
  for (int i = 0; i < kQRounds; i++) {
    raw[i] = u32x4{0u, 0u, 0u, 0u};
    if (d < p.hd && h0 + i * R < p.hq)
      raw[i] = *reinterpret_cast<const u32x4*>(p.qkv + (int64_t)t * p.row +
                                               (int64_t)(h0 + i * R) * p.hd + d);
  }
  u32x4 w = {};
  if (p.qw && d < p.hd) w = *reinterpret_cast<const u32x4*>(p.qw + d);
  const int hb = X ? X : p.half / 8;  // chunks of half a rotation
  const bool low = c < hb, turned = c < 2 * hb;
  float cs[8], sn[8];
  bool inside = true;
  if (turned) angles(p, t, low ? d : d - p.half, cs, sn, inside);
  // (NaN rows where any lane's pairs lack a table row)
  const bool all_in = __builtin_amdgcn_ballot_w64(!inside) == 0;
#pragma unroll
  for (int i = 0; i < kQRounds; i++) {
    if (first + i * R >= p.hq) return;
    float r = 1.0f;
    if (p.qw) {  // uniform
      auto sum_squares = [&](float f) -> float {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float x = elem<DT>(raw[i], e) * f;
          ss = __builtin_fmaf(x, x, ss);
        }
        ss += xor_lane<1>(ss);
        ss += xor_lane<2>(ss);
        ss += xor_lane<4>(ss);
        if constexpr (L >= 16) ss += xor_lane<8>(ss);
        if constexpr (L >= 32) ss += xor_lane<16>(ss);
        return ss;
      };
      r = norm_scale<DT>(p, sum_squares);
    }
    if (!all_in) r = __builtin_nanf("");
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      y[e] = elem<DT>(raw[i], e) * r;
      if (p.qw) y[e] *= elem<DT>(w, e);
    }
    float b[8];
    if constexpr (X > 0) {
#pragma unroll
      for (int e = 0; e < 8; e++) b[e] = xor_lane<X>(y[e]);
    } else {
      const int from = turned ? (low ? lane + hb : lane - hb) : lane;
#pragma unroll
      for (int e = 0; e < 8; e++) b[e] = __shfl(y[e], from);
    }
    if (turned) {
#pragma unroll
      for (int e = 0; e < 8; e++)
        y[e] = __builtin_fmaf(y[e], cs[e], low ? -(b[e] * sn[e]) : b[e] * sn[e]);
    }
    if (d < p.hd && h0 + i * R < p.hq)
      *reinterpret_cast<u32x4*>(p.q + ((int64_t)t * p.hq + h0 + i * R) * p.hd + d) =
          round8<DT>(y);
  }
}

// X: half a rotation in chunks of 8 dims where that is a power of two, 0: any
template <int X>
struct NormRows {
  NormWriteParams p;
  template <int PD, int DT>
  __device__ __forceinline__ bool rows(u32x4* raw, bool& live, int& kv, uint32_t& t, int& h) const;
};

template <int X>
template <int PD, int DT>
__device__ __forceinline__ bool NormRows<X>::rows(u32x4* raw, bool& live, int& kv, uint32_t& t,
                                                  int& head) const {
  using FG = FastGeom<PD>;
  constexpr int P = FG::P, CPL = FG::CPL;
  // chunk rows from a pair's first half to its second where the pair stands in
  // one lane (0: it does not)
  constexpr int M = X % P == 0 && X / P <= CPL / 2 ? X / P : 0;
  const int lane = threadIdx.x & 63;
  const int pl = lane % P;
  // Groups of eight workgroups (one per XCD) of K and V, whose time is VALU work,
  // stand evenly among those of q, whose time is memory: group g is the next of
  // them where g * share / 2^32 passes a whole number (uniform).
  const uint32_t grp = blockIdx.x >> 3, ahead = __umulhi(grp, p.share);
  if ((uint32_t)(((uint64_t)(grp + 1) * p.share) >> 32) == ahead) {
    q_rows<PD, DT, X>(p, 8 * (grp - ahead) + (blockIdx.x & 7));
    return false;
  }
  uint32_t blk = 8 * ahead + (blockIdx.x & 7);
  if (blk >= 2 * p.kblocks) return false;
  const bool isv = blk >= p.kblocks;
  blk -= isv ? p.kblocks : 0u;
  const uint32_t H = (uint32_t)p.hkv;
  uint32_t g = blk * (uint32_t)FG::VPB + (threadIdx.x >> 6) * FG::VPW + lane / P;
  live = g < p.tokens * H;
  g = live ? g : 0u;  // lanes past the end work on the first vector and store nothing
  t = H == 1 ? g : __umulhi(g, p.mk);
  const uint32_t h = g - t * H;
  const uint16_t* const src =
      p.qkv + (int64_t)t * p.row + (int64_t)(p.hq + (isv ? p.hkv : 0) + h) * p.hd;
  kv = isv ? 1 : 0;
  head = (int)h;
#pragma unroll
  for (int i = 0; i < CPL; i++) {
    raw[i] = u32x4{0u, 0u, 0u, 0u};
    if (8 * (pl + P * i) < p.hd) raw[i] = *reinterpret_cast<const u32x4*>(src + 8 * (pl + P * i));
  }
  if (!isv) {
    const uint16_t* const wt = p.kw;
    bool inside = true;
    // the angles of the first pairs ahead of the norm
    float cs[8], sn[8];
    if (M > 0 || 8 * pl < 2 * p.half)
      angles(p, t, M > 0 || 8 * pl < p.half ? 8 * pl : 8 * pl - p.half, cs, sn, inside);
    float r = 1.0f;
    if (wt) {  // uniform
      auto sum_squares = [&](float f) -> float {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < CPL; i++)
#pragma unroll
          for (int c = 0; c < 8; c++) {
            const float x = elem<DT>(raw[i], c) * f;
            ss = __builtin_fmaf(x, x, ss);
          }
        ss += xor_lane<1>(ss);
        ss += xor_lane<2>(ss);
        if constexpr (P == 8) ss += xor_lane<4>(ss);
        return ss;
      };
      r = norm_scale<DT>(p, sum_squares);
    }
    auto normed = [&](const u32x4& x, int d, float* n) {
      u32x4 w = {};
      if (wt) w = *reinterpret_cast<const u32x4*>(wt + d);
#pragma unroll
      for (int c = 0; c < 8; c++) {
        n[c] = elem<DT>(x, c) * r;
        if (wt) n[c] *= elem<DT>(w, c);
      }
    };
    // Chunk rows (pairs of them) one after the other, each rounded back into raw
    // before the next one's loads: the registers of all angles at once would halve
    // the waves that fit a SIMD.
    if constexpr (M > 0) {
#pragma unroll
      for (int i = 0; i < CPL; i++) {
        if (i >= M && i < 2 * M) continue;
        const int d = 8 * (pl + P * i);
        if (d >= p.hd) continue;  // (never of a pair)
        if (i > 0) {
          __builtin_amdgcn_sched_barrier(0);
          if (i < M) angles(p, t, d, cs, sn, inside);
        }
        float a[8];
        normed(raw[i], d, a);
        if (i < M) {
          float b[8], y[8];
          normed(raw[i + M], d + p.half, b);
#pragma unroll
          for (int c = 0; c < 8; c++) {
            y[c] = __builtin_fmaf(a[c], cs[c], -(b[c] * sn[c]));
            b[c] = __builtin_fmaf(b[c], cs[c], a[c] * sn[c]);
          }
          raw[i] = round8<DT>(y);
          raw[i + M] = round8<DT>(b);
        } else {
          raw[i] = round8<DT>(a);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < CPL; i++) {
        const int d = 8 * (pl + P * i);
        if (i > 0) __builtin_amdgcn_sched_barrier(0);
        if (d >= p.hd) continue;
        const bool low = d < p.half;
        if (i > 0 && d < 2 * p.half) angles(p, t, low ? d : d - p.half, cs, sn, inside);
        float a[8];
        normed(raw[i], d, a);
        if (d < 2 * p.half) {
          const int o = low ? d + p.half : d - p.half;
          float b[8];
          normed(*reinterpret_cast<const u32x4*>(src + o), o, b);
#pragma unroll
          for (int c = 0; c < 8; c++) {
            const float turn = b[c] * sn[c];
            a[c] = __builtin_fmaf(a[c], cs[c], low ? -turn : turn);
          }
        }
        raw[i] = round8<DT>(a);
      }
    }
    // a lane sees the positions of its own pairs only: a vector is NaN if any of
    // its lanes lacks a table row
    float miss = inside ? 0.0f : 1.0f;
    miss += xor_lane<1>(miss);
    miss += xor_lane<2>(miss);
    if constexpr (P == 8) miss += xor_lane<4>(miss);
    uint16_t* const out = p.k;
#pragma unroll
    for (int i = 0; i < CPL; i++) {
      const int d = 8 * (pl + P * i);
      if (d >= p.hd) continue;
      if (miss != 0.0f) raw[i] = u32x4{0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};
      if (live && out) *reinterpret_cast<u32x4*>(out + ((int64_t)t * H + h) * p.hd + d) = raw[i];
    }
  }
  return true;
}

template <int PD, int DT>
hipError_t launch_norm_write(const NormWriteParams& p, dim3 grid, hipStream_t st) {
#define TQ_NW(X)                                                                               \
  hipLaunchKernelGGL((write_fast_kernel<PD, DT, NormRows<X>>), grid, dim3(256), 0, st, p.ks, p.vs, \
                     nullptr, nullptr, 0, 0, 0, 0, p.signs, p.slots, 0u, p.hkv, 0u, p.hd, p.ebs,   \
                     p.nslots, p.scale, NormRows<X>{p})
  const int x = p.half / 8;  // (at most PD / 16)
  if (x == 1) TQ_NW(1);
  else if (x == 2) TQ_NW(2);
  else if (x == 4) TQ_NW(4);
  else if (PD >= 128 && x == 8) TQ_NW((PD >= 128 ? 8 : 0));
  else if (PD >= 256 && x == 16) TQ_NW((PD >= 256 ? 16 : 0));
  else TQ_NW(0);
#undef TQ_NW
  return hipGetLastError();
}

// whether [a, a + n) and [b, b + m) share a byte
bool overlap(const void* a, int64_t n, const void* b, int64_t m) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && x < y + (uintptr_t)m && y < x + (uintptr_t)n;
}

}  // namespace
}  // namespace tq

extern "C" int tq_norm_rope_write(
    const void* qkv, int64_t qkv_row_stride, int32_t dtype, const void* q_weight,
    const void* k_weight, float eps, const float* cos_table, const float* sin_table,
    int64_t table_rows, int32_t rotated, const void* positions, int32_t position_bytes,
    int64_t position_stride, const int32_t* sections, int32_t axes, void* k_slab, void* v_slab,
    const float* signs, const int32_t* slot_mapping, int64_t num_tokens, int32_t num_qo_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t padded_dim, int32_t block_size, int32_t ebs,
    int64_t num_blocks, void* q_out, void* k_out, tq_stream_t stream) {
  using namespace tq;
  const char* who = "norm_rope_write";
  const int pd = padded_dim;
  if (pd != 64 && pd != 128 && pd != 256) {
    set_error("%s: padded_dim must be 64, 128 or 256, got %d", who, pd);
    return kEinval;
  }
  if (head_dim <= 0 || head_dim > pd || (pd > 64 && 2 * head_dim <= pd) || head_dim % 8 != 0) {
    set_error("%s: head_dim %d must be a multiple of 8 that pads to %d", who, head_dim, pd);
    return kEinval;
  }
  if (rotated <= 0 || rotated > head_dim || rotated % 16 != 0) {
    set_error("%s: %d rotated dims must be a multiple of 16 up to head_dim", who, rotated);
    return kEinval;
  }
  if (dtype != TQ_F16 && dtype != TQ_BF16) {
    set_error("%s: rows must be fp16 or bf16", who);
    return kEinval;
  }
  if (ebs % 16 != 0 || ebs < pd / 2 + 2 * (pd / 64)) {
    set_error("%s: ebs %d must be a multiple of 16 and >= %d", who, ebs, pd / 2 + 2 * (pd / 64));
    return kEinval;
  }
  if (num_qo_heads <= 0 || num_kv_heads <= 0 || num_qo_heads > 4096 || num_kv_heads > 4096 ||
      block_size <= 0 || num_tokens < 0 || num_blocks < 0 || table_rows < 0) {
    set_error("%s: bad sizes", who);
    return kEinval;
  }
  if ((position_bytes != 4 && position_bytes != 8) || axes < 1 || axes > kMaxAxes || !sections ||
      position_stride < 0) {
    set_error("%s: positions must be 32 or 64 bits wide, of 1 to %d axes with a section each", who,
              kMaxAxes);
    return kEinval;
  }
  int64_t pairs = 0;
  for (int a = 0; a < axes; a++) {
    if (sections[a] < 0) pairs = -1;
    if (pairs >= 0) pairs += sections[a];
  }
  if (pairs != rotated / 2) {
    set_error("%s: the sections must add up to the %d rotated pairs", who, rotated / 2);
    return kEinval;
  }
  if ((q_weight == nullptr) != (k_weight == nullptr)) {
    set_error("%s: both weights must be given, or none", who);
    return kEinval;
  }
  // (below, the squares of small bf16 rows would be lost beside it)
  if (q_weight && !(eps >= 0x1p-126f && eps < INFINITY)) {
    set_error("%s: eps must be a positive, normal fp32 number", who);
    return kEinval;
  }
  if (num_tokens == 0) return 0;
  if (table_rows == 0 || !qkv || !cos_table || !sin_table || !positions || !k_slab || !v_slab ||
      !signs || !slot_mapping || !q_out) {
    set_error("%s: null pointer or empty tables", who);
    return kEinval;
  }
  const int64_t width = (int64_t)(num_qo_heads + 2 * num_kv_heads) * head_dim;
  if (qkv_row_stride < width || qkv_row_stride % 8 != 0) {
    set_error("%s: the row stride %lld must be a multiple of 8 of at least %lld elements", who,
              (long long)qkv_row_stride, (long long)width);
    return kEinval;
  }
  const uintptr_t al = (uintptr_t)qkv | (uintptr_t)q_weight | (uintptr_t)k_weight |
                       (uintptr_t)cos_table | (uintptr_t)sin_table | (uintptr_t)signs |
                       (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)k_slab |
                       (uintptr_t)v_slab;
  if ((al & 15) != 0 || (uintptr_t)positions % position_bytes != 0) {
    set_error("%s: tensors must be 16-byte aligned", who);
    return kEinval;
  }
  const int64_t in_bytes = 2 * ((num_tokens - 1) * qkv_row_stride + width);
  const int64_t q_bytes = 2 * num_tokens * num_qo_heads * head_dim;
  const int64_t k_bytes = 2 * num_tokens * num_kv_heads * head_dim;
  if (overlap(qkv, in_bytes, q_out, q_bytes) || overlap(qkv, in_bytes, k_out, k_bytes) ||
      overlap(q_out, q_bytes, k_out, k_bytes)) {
    set_error("%s: q, k and the projection's rows must not overlap", who);
    return kEinval;
  }
  NormWriteParams p = {};
  p.row = qkv_row_stride;
  p.qw = static_cast<const uint16_t*>(q_weight);
  p.kw = static_cast<const uint16_t*>(k_weight);
  p.eps = eps;
  p.inv_hd = 1.0f / (float)head_dim;
  p.cos_t = cos_table;
  p.sin_t = sin_table;
  p.trows = table_rows;
  p.half = rotated / 2;
  p.axes = axes;
  for (int a = 0, end = 0; a < axes; a++) p.ends[a] = end += sections[a];
  p.pos64 = position_bytes == 8;
  p.pos_st = position_stride;
  p.ks = static_cast<uint8_t*>(k_slab);
  p.vs = static_cast<uint8_t*>(v_slab);
  p.signs = signs;
  p.hq = num_qo_heads;
  p.hkv = num_kv_heads;
  auto recip = [](int h) -> uint32_t {
    return h == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + h - 1) / h);
  };
  const int wave_heads = kQRounds * 64 / (pd / 8);  // of a q wave
  p.qgroups = (num_qo_heads + wave_heads - 1) / wave_heads;
  p.mg = recip(p.qgroups);
  p.mk = recip(num_kv_heads);
  p.hd = head_dim;
  p.ebs = ebs;
  p.nslots = num_blocks * (int64_t)block_size;
  p.scale = 1.0f / sqrtf((float)pd);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int vpb = pd == 64 ? FastGeom<64>::VPB : pd == 128 ? FastGeom<128>::VPB
                                                           : FastGeom<256>::VPB;
  // vector / heads by multiply-high is exact below 2^32 / heads: so many tokens
  // a launch
  const int64_t heads = std::max(num_qo_heads, num_kv_heads);
  const int64_t most = std::min<int64_t>(((int64_t)1 << 31) / (heads * heads), (int64_t)1 << 24);
  for (int64_t a = 0; a < num_tokens; a += most) {
    p.tokens = (uint32_t)std::min(most, num_tokens - a);
    p.qkv = static_cast<const uint16_t*>(qkv) + a * qkv_row_stride;
    p.pos = static_cast<const uint8_t*>(positions) + a * position_bytes;
    p.slots = slot_mapping + a;
    p.q = static_cast<uint16_t*>(q_out) + a * num_qo_heads * head_dim;
    p.k = k_out ? static_cast<uint16_t*>(k_out) + a * num_kv_heads * head_dim : nullptr;
    p.kblocks = (uint32_t)(((int64_t)p.tokens * num_kv_heads + vpb - 1) / vpb);
    const int64_t qblocks = ((int64_t)p.tokens * p.qgroups + 3) / 4;
    const int64_t kgroups = (2 * (int64_t)p.kblocks + 7) / 8, groups = kgroups + (qblocks + 7) / 8;
    p.share = (uint32_t)((((uint64_t)kgroups << 32) + groups - 1) / groups);
    const dim3 grid((unsigned)(8 * groups));
    hipError_t e;
#define TQ_NW(PD)                                                       \
  (dtype == TQ_F16 ? launch_norm_write<PD, TQ_F16>(p, grid, st)         \
                   : launch_norm_write<PD, TQ_BF16>(p, grid, st))
    e = pd == 64 ? TQ_NW(64) : pd == 128 ? TQ_NW(128) : TQ_NW(256);
#undef TQ_NW
    if (e != hipSuccess) {
      set_error("%s: launch failed: %s", who, hipGetErrorString(e));
      return (int)e;
    }
  }
  return 0;
}
