// tq_plan.h -- what the kernels that stream a paged cache share: lane
// exchanges without LDS, the balanced split plan, table addresses, the packed
// scores of two tiles, occupancy facts.
#pragma once

#include <math.h>

#include <mutex>

#include "tq_common.h"

namespace tq {

namespace {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// broadcast lane r of each quad (DPP quad_perm, no LDS)
template <int R>
__device__ __forceinline__ uint32_t quad_bcast(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, R * 0x55, 0xf, 0xf, false);
}

// Float max without NaN quieting: in IEEE mode fmaxf first canonicalizes
// both operands (two more VALU instructions); the scores are never
// signaling NaNs, so the plain instruction gives the same result.
__device__ __forceinline__ float vmax(float a, float b) {
#if defined(__HIP_DEVICE_COMPILE__)
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
#else
  return fmaxf(a, b);
#endif
}
__device__ __forceinline__ float vmax3(float a, float b, float c) {
#if defined(__HIP_DEVICE_COMPILE__)
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
#else
  return fmaxf(fmaxf(a, b), c);
#endif
}
// largest magnitude of three
__device__ __forceinline__ float vmax3_abs(float a, float b, float c) {
#if defined(__HIP_DEVICE_COMPILE__)
  float r;
  asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
#else
  return fmaxf(fmaxf(fabsf(a), fabsf(b)), fabsf(c));
#endif
}
// max(x, x of lane l ror 8 within its row): one DPP max (the s_nop covers
// the wait states of a DPP read after a VALU write of its source)
__device__ __forceinline__ float max_ror8(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  float r;
  asm("s_nop 1\n\tv_max_f32_dpp %0, %1, %1 row_ror:8 row_mask:0xf bank_mask:0xf"
      : "=v"(r)
      : "v"(x));
  return r;
#else
  return fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xf, 0xf,
                                                          false)));
#endif
}
// score * K norm, the norm an fp16 value in the low half of nr: one
// v_fma_mix (fp16 operand, fp32 math; +0 addend, which only differs from
// the product for a -0 score, and that feeds the same max and exp2)
__device__ __forceinline__ float mul_lo_half(float sc, uint32_t nr) {
#if defined(__HIP_DEVICE_COMPILE__)
  float r;
  asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(nr), "v"(sc));
  return r;
#else
  return sc * (float)__builtin_bit_cast(_Float16, (uint16_t)(nr & 0xffffu));
#endif
}
__device__ __forceinline__ float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return vmax(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return vmax(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor16_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float xor32_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// rotate by 8 lanes inside each 16-lane row (DPP row_ror:8)
__device__ __forceinline__ float ror8(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xf, 0xf, false));
}
// value of lane l ^ m (m = 1, 2, 4, 8 without LDS: DPP quad_perm, row
// half-mirror then quad reversal, row rotate by 8)
__device__ __forceinline__ float xor_lane(float x, int m) {
  const int v = __float_as_int(x);
  switch (m) {
    case 1: return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, false));
    case 2: return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, false));
    case 4: {
      const int t = __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, false);
      return __int_as_float(__builtin_amdgcn_mov_dpp(t, 0x1B, 0xf, 0xf, false));
    }
    case 8: return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, false));
    default: return __shfl_xor(x, m);
  }
}
// LDS byte address of a pointer into __shared__ memory.
__device__ __forceinline__ uint32_t lds_addr(const void* ptr) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)ptr;
}
// fp16 value held in the low / high half of a dword
__device__ __forceinline__ float lo_half(uint32_t v) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(v & 0xffffu));
}
__device__ __forceinline__ float hi_half(uint32_t v) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(v >> 16));
}

// ---- balanced split plan ------------------------------------------------
constexpr int kPlanAlign = 2 * kTile;   // unit sizes are whole steps
constexpr int kPlanMost = 1024;         // sequences a balanced plan takes

__device__ __forceinline__ int xor_lane_i(int v, int m) {
  return __float_as_int(xor_lane(__int_as_float(v), m));
}
__device__ __forceinline__ int permlane_xor16_i(int v) {
  const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  return (int)r[0] == v ? (int)r[1] : (int)r[0];
}
// sum / max over the 64 lanes (every lane gets the result): DPP lane xors
// inside rows of 16, then the 16- and 32-lane swaps
__device__ __forceinline__ int wave_sum_i(int v) {
  v += xor_lane_i(v, 1);
  v += xor_lane_i(v, 2);
  v += xor_lane_i(v, 4);
  v += xor_lane_i(v, 8);
  auto r = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = (int)(r[0] + r[1]);
  r = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return (int)(r[0] + r[1]);
}
__device__ __forceinline__ int wave_max_i(int v) {
  v = max(v, xor_lane_i(v, 1));
  v = max(v, xor_lane_i(v, 2));
  v = max(v, xor_lane_i(v, 4));
  v = max(v, xor_lane_i(v, 8));
  auto r = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = max((int)r[0], (int)r[1]);
  r = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return max((int)r[0], (int)r[1]);
}
// ceil(a / d) for a >= 0, d > 0, a + d < 2^31: below 2^24 a float estimate
// (off by at most one there) corrected both ways in integers; from 2^24 on
// (a sequence of 16M tokens or more) an integer division
__device__ __forceinline__ int ceil_div_est(int a, int d, float rd) {
  const int x = a + d - 1;
  if (x >= (1 << 24)) return x / d;
  int f = (int)((float)x * rd);
  f -= (f * d > x) ? 1 : 0;
  f += ((f + 1) * d <= x) ? 1 : 0;
  return f;
}

// The unit of a balanced plan a workgroup serves: sequence b (-1: none, the
// grid has more units than the plan uses), unit j of that sequence, its
// length L, page-table start ip, the sequence's first unit Pb and the unit
// size U in tokens.
struct PlanSlot {
  int b, j, L, Pb, U, ip;
};

// The plan from the sequence lengths, which `lens(i, lane)` returns for
// sequence 64 i + lane (0 past the batch) and `starts` likewise for the
// page-table starts; nreg = ceil(B / 64).  Every lane of a wave runs it and
// every field of the result is wave-uniform.  writer: this wave also stores
// the row table (rows = rowmul * units) and U.  U is a multiple of A tokens.
template <int A = kPlanAlign, typename LensFn, typename StartsFn>
__device__ __forceinline__ PlanSlot plan_slot(LensFn lens, StartsFn starts, int B, int nreg,
                                              int units, int u, int rowmul, int32_t* split_out,
                                              bool writer) {
  const int lane = threadIdx.x & 63;
  int tsum = 0, mx = 0, nz = 0;
  for (int i = 0; i < nreg; i++) {
    const int l = lens(i);
    tsum += l;
    mx = max(mx, l);
    nz += l > 0 ? 1 : 0;
  }
  tsum = __builtin_amdgcn_readfirstlane(wave_sum_i(tsum));
  mx = __builtin_amdgcn_readfirstlane(wave_max_i(mx));
  nz = __builtin_amdgcn_readfirstlane(wave_sum_i(nz));
  if (nreg == 1 && nz == B && (int64_t)mx * B == (int64_t)tsum) {
    // every sequence has the same length L: sum_b ceil(L / U) <= units is
    // ceil(L / U) <= k = floor(units / B), i.e. U >= L / k, so the plan has
    // a closed form (no search, no scan before the first page-id loads)
    const int k = units / B;
    const int U = ((mx + k - 1) / k + A - 1) / A * A;
    const int c = (mx + U - 1) / U;  // units per sequence
    PlanSlot r = {-1, 0, 0, 0, U, 0};
    if (u < B * c) {
      r.b = u / c;
      r.j = u - r.b * c;
      r.Pb = r.b * c;
      r.L = mx;
      r.ip = __builtin_amdgcn_readlane(starts(0), r.b);
    }
    if (writer) {
      if (lane < B) split_out[lane] = lane * c * rowmul;
      if (lane == 0) {
        split_out[B] = B * c * rowmul;
        split_out[B + 1] = U;
      }
    }
    r.b = __builtin_amdgcn_readfirstlane(r.b);
    r.j = __builtin_amdgcn_readfirstlane(r.j);
    r.L = __builtin_amdgcn_readfirstlane(r.L);
    r.Pb = __builtin_amdgcn_readfirstlane(r.Pb);
    r.ip = __builtin_amdgcn_readfirstlane(r.ip);
    return r;
  }
  auto units_for = [&](int k) -> int {
    const int d = k * A;
    const float rd = 1.0f / (float)d;
    int c = 0;
    for (int i = 0; i < nreg; i++) c += ceil_div_est(lens(i), d, rd);
    return __builtin_amdgcn_readfirstlane(wave_sum_i(c));
  };
  // smallest feasible k in (lo, hi]: every k below tsum / (units * A) needs
  // more than `units` units; k = ceil(max_len / A) needs nz <= units, and so
  // does any k >= tsum / ((units - nz) * A) (at most one partial unit per
  // sequence)
  int hi = max(1, (mx + A - 1) / A);
  if (units > nz) hi = min(hi, max(1, (tsum + (units - nz) * A - 1) / ((units - nz) * A)));
  int lo = (tsum + units * A - 1) / (units * A) - 1;
  lo = max(0, min(lo, hi - 1));
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (units_for(mid) <= units) hi = mid; else lo = mid;
  }
  const int U = hi * A;
  const float rdU = 1.0f / (float)U;
  PlanSlot r = {-1, 0, 0, 0, U, 0};
  int carry = 0;
  for (int i = 0; i < nreg; i++) {
    const int l = lens(i);
    const int c = ceil_div_est(l, U, rdU);
    int incl = c;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(incl, off);
      if (lane >= off) incl += y;
    }
    incl += carry;
    const int excl = incl - c;
    const int bb = 64 * i + lane;
    if (writer && bb < B) split_out[bb] = excl * rowmul;
    const uint64_t hit = __ballot(c > 0 && excl <= u && u < incl);
    if (hit) {
      const int l0 = __builtin_ctzll(hit);
      r.b = 64 * i + l0;
      r.Pb = __builtin_amdgcn_readlane(excl, l0);
      r.j = u - r.Pb;
      r.L = __builtin_amdgcn_readlane(l, l0);
      r.ip = __builtin_amdgcn_readlane(starts(i), l0);
    }
    carry = __builtin_amdgcn_readlane(incl, 63);
  }
  if (writer && lane == 0) {
    split_out[B] = carry * rowmul;
    split_out[B + 1] = U;
  }
  // every field is wave-uniform; saying so keeps the addresses built from
  // them in scalar registers (buffer descriptors need them there)
  r.b = __builtin_amdgcn_readfirstlane(r.b);
  r.j = __builtin_amdgcn_readfirstlane(r.j);
  r.L = __builtin_amdgcn_readfirstlane(r.L);
  r.Pb = __builtin_amdgcn_readfirstlane(r.Pb);
  r.U = __builtin_amdgcn_readfirstlane(r.U);
  r.ip = __builtin_amdgcn_readfirstlane(r.ip);
  return r;
}

// s_waitcnt immediate that waits until at most n vector-memory operations
// are outstanding (gfx9 encoding: vmcnt[3:0] | expcnt[6:4] | lgkmcnt[11:8] |
// vmcnt[5:4] in [15:14]; expcnt and lgkmcnt left at their maximum).
__host__ __device__ constexpr int vmcnt_imm(int n) {
  return (n & 15) | (7 << 4) | (15 << 8) | ((n >> 4) << 14);
}

// Table addresses from code bytes spread into 16-bit halves: lut_spread
// puts bytes 2i and 2i + 1 of w into the low and high halves of one register
// (v_perm), and lut_mad forms half * 2^SH + lanec in one v_mad_u32_u16
// (op_sel picks the half), so a pair of lookups costs three instructions
// instead of four.  lut_mad<SH, HI>(lut_spread(w, i), lanec) equals
// lut_addr<SH>(w, 2 * i + HI, lanec).
__device__ __forceinline__ uint32_t lut_spread(uint32_t w, int i) {
  return __builtin_amdgcn_perm(0u, w, i ? 0x0c030c02u : 0x0c010c00u);
}
template <int SH, int HI>
__device__ __forceinline__ uint32_t lut_mad(uint32_t h, uint32_t lanec) {
  uint32_t a;
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (HI)
    asm("v_mad_u32_u16 %0, %1, %2, %3 op_sel:[1,0,0,0]" : "=v"(a) : "v"(h), "s"(1u << SH), "v"(lanec));
  else
    asm("v_mad_u32_u16 %0, %1, %2, %3" : "=v"(a) : "v"(h), "s"(1u << SH), "v"(lanec));
#else
  a = ((HI ? h >> 16 : h & 0xffffu) << SH) + lanec;
#endif
  return a;
}

// PACK 2 scores of two tiles from their unmerged QC accumulators: lanes n < 8
// of each row get tile 0's hi + lo sums (lane n + 8 holds the lo part), lanes
// n >= 8 tile 1's (lane n - 8 holds the hi part): two DPP adds per value
// whose bank masks write one half of each row each.  The leading s_nops
// cover the wait states between the MFMAs that wrote a0 / a1 and their DPP
// read (inline assembly, so the compiler does not count them).
__device__ __forceinline__ float4_t pack_merge(float4_t a0, float4_t a1) {
  float4_t d;
#if defined(__HIP_DEVICE_COMPILE__)
  float d0, d1, d2, d3;
  asm volatile("s_nop 7\n\ts_nop 7\n\t"
               "v_add_f32_dpp %0, %4, %4 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
               "v_add_f32_dpp %0, %8, %8 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
               "v_add_f32_dpp %1, %5, %5 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
               "v_add_f32_dpp %1, %9, %9 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
               "v_add_f32_dpp %2, %6, %6 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
               "v_add_f32_dpp %2, %10, %10 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
               "v_add_f32_dpp %3, %7, %7 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
               "v_add_f32_dpp %3, %11, %11 row_ror:8 row_mask:0xf bank_mask:0xc"
               : "=&v"(d0), "=&v"(d1), "=&v"(d2), "=&v"(d3)
               : "v"(a0[0]), "v"(a0[1]), "v"(a0[2]), "v"(a0[3]), "v"(a1[0]), "v"(a1[1]),
                 "v"(a1[2]), "v"(a1[3]));
  d = float4_t{d0, d1, d2, d3};
#else
  d = a0 + a1;
#endif
  return d;
}

// Occupancy facts of one kernel on the current device: CUs and resident
// workgroups per CU.  Queried once per (device, kernel) and cached, so a
// decode launch costs no device queries after the first.
struct Occupancy {
  int cus, per_cu;
};
Occupancy occupancy(const void* kernel, int threads) {
  struct Entry {
    int dev;
    const void* kernel;
    int threads;
    Occupancy occ;
  };
  // a fixed table (no allocation on any call): a few kernels per device
  constexpr int kEntries = 256;
  static std::mutex mu;
  static Entry cache[kEntries];
  static int used = 0;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return {0, 0};
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < used; i++)
    if (cache[i].dev == dev && cache[i].kernel == kernel && cache[i].threads == threads)
      return cache[i].occ;
  Occupancy o = {0, 0};
  if (hipDeviceGetAttribute(&o.cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
      hipOccupancyMaxActiveBlocksPerMultiprocessor(&o.per_cu, kernel, threads, 0) != hipSuccess)
    return {0, 0};
  if (used < kEntries) cache[used++] = {dev, kernel, threads, o};
  return o;
}

}  // namespace

}  // namespace tq
