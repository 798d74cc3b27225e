// tq_write.hip -- quantize-and-scatter of K/V rows into the packed paged cache.
//
// Same numbers as the reference scatter kernel
// (csrc/include/turboquant/quantize_write_kernel.cuh:332-431), which gives
// every vector 32 lanes of VEC = pd/32 consecutive dims: the fp32 sum of
// squares, its reduction tree, sqrt, reciprocal, sign flip, FWHT butterflies
// and the 1/sqrt(pd) scale happen in the same order and give the same bits.
// MI355X layout: 16 lanes per vector, each holding the dims of two of the
// reference's lanes (p and p + 16), so a wave64 carries four vectors and the
// per-vector work (index math, reduction, sqrt, divide, norm store) is
// shared by twice the dims; a 256-thread workgroup writes 16 consecutive
// (token, head) entries, i.e. whole cache rows.  One launch covers K and V.
#include <stdarg.h>
#include <stdio.h>

#include <atomic>

#include "tq_quant.h"

namespace tq {

namespace {

// Load VEC consecutive input elements as fp32 (exact for fp16/bf16).  vec_ok:
// rows aligned to VEC elements and head_dim a multiple of VEC, so a run lies
// inside the row or past its end.
template <int VEC>
__device__ __forceinline__ void load_row(const void* base, int64_t off, int dtype,
                                         int d0, int head_dim, bool vec_ok, float* x) {
  if (vec_ok) {
#pragma unroll
    for (int i = 0; i < VEC; i++) x[i] = 0.0f;
    if (d0 >= head_dim) return;
    if (dtype == TQ_F32) {
      typedef float fv __attribute__((ext_vector_type(VEC)));
      const fv v = *reinterpret_cast<const fv*>(static_cast<const float*>(base) + off + d0);
#pragma unroll
      for (int i = 0; i < VEC; i++) x[i] = v[i];
      return;
    }
    typedef _Float16 hv __attribute__((ext_vector_type(VEC)));
    const hv v = *reinterpret_cast<const hv*>(static_cast<const _Float16*>(base) + off + d0);
#pragma unroll
    for (int i = 0; i < VEC; i++)
      x[i] = dtype == TQ_F16
                 ? (float)v[i]
                 : __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[i]) << 16);
    return;
  }
  if (dtype == TQ_F16) {
    const _Float16* p = reinterpret_cast<const _Float16*>(base) + off + d0;
#pragma unroll
    for (int i = 0; i < VEC; i++) x[i] = (d0 + i < head_dim) ? (float)p[i] : 0.0f;
  } else if (dtype == TQ_BF16) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + off + d0;
#pragma unroll
    for (int i = 0; i < VEC; i++)
      x[i] = (d0 + i < head_dim) ? __uint_as_float((uint32_t)p[i] << 16) : 0.0f;
  } else {
    const float* p = reinterpret_cast<const float*>(base) + off + d0;
#pragma unroll
    for (int i = 0; i < VEC; i++) x[i] = (d0 + i < head_dim) ? p[i] : 0.0f;
  }
}

// code = #{j : v >= b_j} over the 15 boundaries b_j = boundary_j * scale.
// The boundaries are symmetric with b_7 = 0, so for v >= 0 (this includes
// -0.0, as in the reference's `val >= b[mid]`) the code is 8 + #{k : v >= B_k},
// and for v < 0 or NaN it is 7 - #{k : |v| > B_k}, B_k = b_{7+k}.  On positive
// floats "a > B" is "bits(a) - 1 >= bits(B)" as integers, so one integer
// compare chain serves both sides.  Same result as the binary search of
// quantize_write_kernel.cuh:34-46 for every fp32 input.
__device__ __forceinline__ uint32_t bucketize(float v, const int32_t* bbits) {
  const bool pos = v >= 0.0f;
  int32_t a = (int32_t)(__float_as_uint(v) & 0x7fffffffu) - (pos ? 0 : 1);
  uint32_t k = 0;
#pragma unroll
  for (int j = 0; j < 7; j++) k += (a >= bbits[j]) ? 1u : 0u;
  return pos ? 8u + k : 7u - k;
}

// Quantize-and-scatter: 16 lanes per vector, 4 vectors per wave64, 16
// consecutive vectors (kv, token, head; head fastest, so the entries of one
// token's heads are written together) per 256-thread workgroup.  Physical
// lane p of a vector holds the dims of two lanes of the reference's 32-lane
// layout (quantize_write_kernel.cuh:332-431): lane p (dims VEC p .. +VEC) in
// x0 and lane p + 16 in x1.  The arithmetic is the reference's, in its
// order: per-lane FMA sums, the shfl_down tree 16, 8, 4, 2, 1 (its first
// level pairs x0 and x1 of one physical lane), IEEE sqrt and reciprocal,
// sign flip, FWHT stages h = 1 .. pd/2 in ascending order (the last one,
// between lanes p and p + 16, again inside one physical lane), 1/sqrt(pd),
// bucketize, pack.
//
// With 16 lanes per vector a small launch has four times the waves of the
// fast kernel below and a quarter of the work in each: K and V of 8 tokens x 8
// heads x 128 take 3.5 us against 4.0 us, 512 tokens 4.1 against 4.25, 1024
// tokens 5.15 against 4.5 (graph replays; so up to kSmallWrite vectors).  Above that it serves
// the rows that the fast kernel cannot load.
//
// sign_first: the signs are flipped before the squares, which leaves a NaN
// norm the sign that the fast kernel gives it (every other bit is the same).
template <int PD, bool VEC_OK>
__global__ __launch_bounds__(256) void write_kernel(
    uint8_t* __restrict__ k_slab, uint8_t* __restrict__ v_slab,
    const void* __restrict__ key, const void* __restrict__ value, int dtype,
    int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
    const float* __restrict__ signs, const int32_t* __restrict__ slots,
    uint32_t per_kv, int H, uint32_t hmul, int head_dim, int ebs, int64_t nslots,
    float scale, bool sign_first) {
#pragma clang fp contract(off)
  constexpr int VEC = PD / 32;
  const int lane = threadIdx.x & 15;
  const uint32_t g = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (g >= 2 * per_kv) return;  // a whole 16-lane group (one DPP row) leaves
  const int kv = g >= per_kv ? 1 : 0;
  const uint32_t rem = g - (kv ? per_kv : 0u);
  // t = rem / H by multiply-high (hmul = ceil(2^32 / H), exact for rem < 2^32 / H)
  const uint32_t t = H == 1 ? rem : __umulhi(rem, hmul);
  const int h = (int)(rem - t * (uint32_t)H);

  float x0[VEC], x1[VEC];
  const int da = lane * VEC, db = (lane + 16) * VEC;
  if (kv == 0) {
    load_row<VEC>(key, (int64_t)t * k_st + h * k_sh, dtype, da, head_dim, VEC_OK, x0);
    load_row<VEC>(key, (int64_t)t * k_st + h * k_sh, dtype, db, head_dim, VEC_OK, x1);
  } else {
    load_row<VEC>(value, (int64_t)t * v_st + h * v_sh, dtype, da, head_dim, VEC_OK, x0);
    load_row<VEC>(value, (int64_t)t * v_st + h * v_sh, dtype, db, head_dim, VEC_OK, x1);
  }
  const int32_t slot = slots[t];
  if (slot < 0 || (int64_t)slot >= nslots) return;  // whole 16-lane group together

  float g0[VEC], g1[VEC];
#pragma unroll
  for (int i = 0; i < VEC; i++) {
    g0[i] = signs[da + i];
    g1[i] = signs[db + i];
  }
  auto flip = [](float v, float s) {  // v * s for s = +-1, a NaN's sign too
    return __uint_as_float(__float_as_uint(v) ^ (__float_as_uint(s) & 0x80000000u));
  };
  if (sign_first) {  // uniform
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      x0[i] = flip(x0[i], g0[i]);
      x1[i] = flip(x1[i], g1[i]);
    }
  }
  // 1. per-lane sums of squares, FMA-accumulated in dim order
  float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
  for (int i = 0; i < VEC; i++) {
    s0 = __builtin_fmaf(x0[i], x0[i], s0);
    s1 = __builtin_fmaf(x1[i], x1[i], s1);
  }
  // 2. the tree: level 16 in-lane, then 8, 4, 2, 1 across the 16 lanes;
  //    every lane ends with the bits the reference's lane 0 holds
  float ss = s0 + s1;
  ss = ss + xor_lane<8>(ss);
  ss = ss + xor_lane<4>(ss);
  ss = ss + xor_lane<2>(ss);
  ss = ss + xor_lane<1>(ss);
  // 3. IEEE sqrt and reciprocal
  const float l2 = __builtin_sqrtf(ss);
  const float inv = (l2 > 1e-8f) ? (1.0f / l2) : 0.0f;
  // 4. normalise, flip signs
#pragma unroll
  for (int i = 0; i < VEC; i++) {
    x0[i] = x0[i] * inv;
    x1[i] = x1[i] * inv;
  }
  if (!sign_first) {
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      x0[i] = x0[i] * g0[i];
      x1[i] = x1[i] * g1[i];
    }
  }
  // 5. FWHT: in-lane stages h < VEC, cross-lane stages (lane xor 1..8), then
  //    the stage between lanes p and p + 16
#pragma unroll
  for (int hh = 1; hh < VEC; hh <<= 1) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2 * hh) {
#pragma unroll
      for (int k = 0; k < hh; k++) {
        float a = x0[i + k], b = x0[i + k + hh];
        x0[i + k] = a + b;
        x0[i + k + hh] = a - b;
        a = x1[i + k];
        b = x1[i + k + hh];
        x1[i + k] = a + b;
        x1[i + k + hh] = a - b;
      }
    }
  }
  // butterfly partner + sign * own value: fma(+-1, v, p) rounds once, to the
  // same bits as v + p (lower lane) or p - v (upper lane)
  auto cross = [&](auto dist) {
    constexpr int D = decltype(dist)::value;
    const float sg = (lane & D) ? -1.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      x0[i] = __builtin_fmaf(sg, x0[i], xor_lane<D>(x0[i]));
      x1[i] = __builtin_fmaf(sg, x1[i], xor_lane<D>(x1[i]));
    }
  };
  cross(std::integral_constant<int, 1>{});
  cross(std::integral_constant<int, 2>{});
  cross(std::integral_constant<int, 4>{});
  cross(std::integral_constant<int, 8>{});
#pragma unroll
  for (int i = 0; i < VEC; i++) {
    const float a = x0[i], b = x1[i];
    x0[i] = (a + b) * scale;
    x1[i] = (a - b) * scale;
  }

  // 6. bucketize against b_j * scale (fp32 products, as the reference forms them)
  int32_t bbits[7];
#pragma unroll
  for (int j = 0; j < 7; j++) bbits[j] = (int32_t)__float_as_uint(boundary_pos(j + 1) * scale);

  uint8_t* entry = (kv == 0 ? k_slab : v_slab) +
                   ((int64_t)slot * H + h) * (int64_t)ebs;  // slot*H == (block*bs+entry)*H
  // 7. pack: byte k = code[2k] << 4 | code[2k+1]
  uint32_t p0 = 0, p1 = 0;
#pragma unroll
  for (int i = 0; i < VEC; i += 2) {
    p0 |= ((bucketize(x0[i], bbits) << 4) | bucketize(x0[i + 1], bbits)) << (4 * i);
    p1 |= ((bucketize(x1[i], bbits) << 4) | bucketize(x1[i + 1], bbits)) << (4 * i);
  }
  uint8_t* d0p = entry + lane * (VEC / 2);
  uint8_t* d1p = entry + (lane + 16) * (VEC / 2);
  if constexpr (VEC == 2) {
    *d0p = (uint8_t)p0;
    *d1p = (uint8_t)p1;
  } else if constexpr (VEC == 4) {
    *reinterpret_cast<uint16_t*>(d0p) = (uint16_t)p0;
    *reinterpret_cast<uint16_t*>(d1p) = (uint16_t)p1;
  } else {
    *reinterpret_cast<uint32_t*>(d0p) = p0;
    *reinterpret_cast<uint32_t*>(d1p) = p1;
  }
  // 8. fp16(l2), round to nearest even, repeated pd/64 times after the codes
  if (lane == 0) {
    _Float16 nh = (_Float16)l2;
    uint32_t nb = (uint32_t)__builtin_bit_cast(uint16_t, nh);
    uint8_t* np = entry + PD / 2;
    if constexpr (PD == 64) {
      *reinterpret_cast<uint16_t*>(np) = (uint16_t)nb;
    } else if constexpr (PD == 128) {
      *reinterpret_cast<uint32_t*>(np) = nb | (nb << 16);
    } else {
      uint2 w;
      w.x = nb | (nb << 16);
      w.y = w.x;
      *reinterpret_cast<uint2*>(np) = w;
    }
  }
}

template <int PD>
hipError_t launch_write(bool vec_ok, dim3 grid, hipStream_t stream, uint8_t* ks, uint8_t* vs,
                        const void* key, const void* value, int dtype, int64_t k_st,
                        int64_t k_sh, int64_t v_st, int64_t v_sh, const float* signs,
                        const int32_t* slots, uint32_t per_kv, int H, uint32_t hmul, int hd,
                        int ebs, int64_t nslots, float scale, bool sign_first) {
  if (vec_ok)
    hipLaunchKernelGGL((write_kernel<PD, true>), grid, dim3(256), 0, stream, ks, vs, key, value,
                       dtype, k_st, k_sh, v_st, v_sh, signs, slots, per_kv, H, hmul, hd, ebs,
                       nslots, scale, sign_first);
  else
    hipLaunchKernelGGL((write_kernel<PD, false>), grid, dim3(256), 0, stream, ks, vs, key, value,
                       dtype, k_st, k_sh, v_st, v_sh, signs, slots, per_kv, H, hmul, hd, ebs,
                       nslots, scale, sign_first);
  return hipGetLastError();
}

template <int PD>
hipError_t launch_write_fast(hipStream_t stream, uint8_t* ks, uint8_t* vs, const void* key,
                             const void* value, int dtype, int64_t k_st, int64_t k_sh,
                             int64_t v_st, int64_t v_sh, const float* signs, const int32_t* slots,
                             uint32_t per_kv, int H, uint32_t hmul, int hd, int ebs,
                             int64_t nslots, float scale) {
  const int64_t blocks = (2 * (int64_t)per_kv + FastGeom<PD>::VPB - 1) / FastGeom<PD>::VPB;
  const dim3 grid((unsigned)blocks);
#define TQ_FAST(DT)                                                                              \
  hipLaunchKernelGGL((write_fast_kernel<PD, DT>), grid, dim3(256), 0, stream, ks, vs, key, value, \
                     k_st, k_sh, v_st, v_sh, signs, slots, per_kv, H, hmul, hd, ebs, nslots, scale,   \
                     PlainRows{})
  if (dtype == TQ_F16) TQ_FAST(TQ_F16);
  else if (dtype == TQ_BF16) TQ_FAST(TQ_BF16);
  else TQ_FAST(TQ_F32);
#undef TQ_FAST
  return hipGetLastError();
}

}  // namespace

thread_local char g_err[512];

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}

int device_cus() {
  constexpr int kMaxDev = 64;
  static std::atomic<int> cache[kMaxDev];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDev) return 0;
  int c = cache[dev].load(std::memory_order_relaxed);
  if (c == 0 && hipDeviceGetAttribute(&c, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess)
    cache[dev].store(c, std::memory_order_relaxed);
  return c;
}

}  // namespace tq

extern "C" const char* tq_last_error(void) { return tq::g_err; }
extern "C" int32_t tq_abi_version(void) { return TQ_ABI_VERSION; }

extern "C" int tq_quantize_write_kv_cache(void* k_slab, void* v_slab, const void* key,
                                          const void* value, int32_t in_dtype,
                                          int64_t k_stride_tok, int64_t k_stride_head,
                                          int64_t v_stride_tok, int64_t v_stride_head,
                                          const float* signs, const int32_t* slot_mapping,
                                          int64_t num_tokens, int32_t num_kv_heads,
                                          int32_t head_dim, int32_t padded_dim,
                                          int32_t block_size, int32_t ebs, int64_t num_blocks,
                                          tq_stream_t stream) {
  using namespace tq;
  const int pd = padded_dim;
  if (pd != 64 && pd != 128 && pd != 256) {
    set_error("quantize_write: padded_dim must be 64, 128 or 256, got %d", pd);
    return kEinval;
  }
  if (head_dim <= 0 || head_dim > pd || (pd > 64 && 2 * head_dim <= pd)) {
    set_error("quantize_write: head_dim %d does not pad to %d", head_dim, pd);
    return kEinval;
  }
  if (ebs % 16 != 0 || ebs < pd / 2 + 2 * (pd / 64)) {
    set_error("quantize_write: ebs %d must be a multiple of 16 and >= %d", ebs,
              pd / 2 + 2 * (pd / 64));
    return kEinval;
  }
  if (in_dtype != TQ_F32 && in_dtype != TQ_F16 && in_dtype != TQ_BF16) {
    set_error("quantize_write: unsupported input dtype %d", in_dtype);
    return kEinval;
  }
  if (num_kv_heads <= 0 || block_size <= 0 || num_tokens < 0 || num_blocks < 0) {
    set_error("quantize_write: bad sizes");
    return kEinval;
  }
  if (num_tokens == 0) return 0;
  if (!k_slab || !v_slab || !key || !value || !signs || !slot_mapping) {
    set_error("quantize_write: null pointer");
    return kEinval;
  }
  const int vec = pd / 32;
  const int esz = in_dtype == TQ_F32 ? 4 : 2;
  // vector loads: rows in whole runs of VEC elements, every row start aligned to them
  const bool vec_ok = head_dim % vec == 0 && (k_stride_tok % vec == 0) &&
                      (k_stride_head % vec == 0) && (v_stride_tok % vec == 0) &&
                      (v_stride_head % vec == 0) && ((uintptr_t)key % (vec * esz) == 0) &&
                      ((uintptr_t)value % (vec * esz) == 0);
  // 16 vectors per workgroup; token = rem / H by multiply-high, exact while
  // num_tokens * H < 2^32 / H
  const int64_t per_kv = num_tokens * (int64_t)num_kv_heads;
  if (per_kv * num_kv_heads >= (int64_t)1 << 32 || 2 * per_kv >= (int64_t)1 << 32) {
    set_error("quantize_write: too many tokens (%lld x %d heads)", (long long)num_tokens,
              num_kv_heads);
    return kEinval;
  }
  const uint32_t hmul =
      num_kv_heads == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + num_kv_heads - 1) / num_kv_heads);
  const int64_t blocks = (2 * per_kv + 15) / 16;
  const float scale = 1.0f / sqrtf((float)pd);
  const int64_t nslots = num_blocks * (int64_t)block_size;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  dim3 grid((unsigned)blocks);
  uint8_t* ks = static_cast<uint8_t*>(k_slab);
  uint8_t* vs = static_cast<uint8_t*>(v_slab);
  hipError_t e;
  // rows in whole 16-byte aligned pieces take the fast kernel
  const int al = 16 / esz;
  const bool fast_ok = head_dim % 8 == 0 && k_stride_tok % al == 0 && k_stride_head % al == 0 &&
                       v_stride_tok % al == 0 && v_stride_head % al == 0 &&
                       (uintptr_t)key % 16 == 0 && (uintptr_t)value % 16 == 0 &&
                       (uintptr_t)signs % 16 == 0;
  // small launches of padded size 64 or 128 take the general kernel (see there;
  // at 256 the fast one is as fast from one token on)
  constexpr int64_t kSmallWrite = 8192;
  const bool small = pd <= 128 && 2 * per_kv <= kSmallWrite;
  const bool sign_first = fast_ok && in_dtype == TQ_F16 && head_dim == pd;
  if (fast_ok && !small) {
#define TQ_FAST_PD(PD)                                                                            \
  launch_write_fast<PD>(s, ks, vs, key, value, in_dtype, k_stride_tok, k_stride_head,             \
                        v_stride_tok, v_stride_head, signs, slot_mapping, (uint32_t)per_kv,       \
                        num_kv_heads, hmul, head_dim, ebs, nslots, scale)
    e = pd == 64 ? TQ_FAST_PD(64) : pd == 128 ? TQ_FAST_PD(128) : TQ_FAST_PD(256);
#undef TQ_FAST_PD
    if (e != hipSuccess) {
      set_error("quantize_write: launch failed: %s", hipGetErrorString(e));
      return (int)e;
    }
    return 0;
  }
  switch (pd) {
    case 64:
      e = launch_write<64>(vec_ok, grid, s, ks, vs, key, value, in_dtype, k_stride_tok,
                           k_stride_head, v_stride_tok, v_stride_head, signs, slot_mapping,
                           (uint32_t)per_kv, num_kv_heads, hmul, head_dim, ebs, nslots, scale,
                           sign_first);
      break;
    case 128:
      e = launch_write<128>(vec_ok, grid, s, ks, vs, key, value, in_dtype, k_stride_tok,
                            k_stride_head, v_stride_tok, v_stride_head, signs, slot_mapping,
                            (uint32_t)per_kv, num_kv_heads, hmul, head_dim, ebs, nslots, scale,
                           sign_first);
      break;
    default:
      e = launch_write<256>(vec_ok, grid, s, ks, vs, key, value, in_dtype, k_stride_tok,
                            k_stride_head, v_stride_tok, v_stride_head, signs, slot_mapping,
                            (uint32_t)per_kv, num_kv_heads, hmul, head_dim, ebs, nslots, scale,
                            sign_first);
  }
  if (e != hipSuccess) {
    set_error("quantize_write: launch failed: %s", hipGetErrorString(e));
    return (int)e;
  }
  return 0;
}
