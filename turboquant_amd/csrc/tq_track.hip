// tq_track.hip -- attention that records what each cached token receives.
//
// Beside the packed paged cache stand two arrays, weights fp32 and positions
// int32 [num_blocks, num_kv_heads, block_size]: the attention weight that an
// entry has received so far, summed over the q heads of its kv head, and the
// position in its sequence that it came from.  Two calls add to them:
//
//  * tq_decode_paged_tracked: one new token per sequence.
//      s_ht = sm_scale q'_h . K^_t        q' = FWHT(s q)/sqrt(pd)
//      p_ht = exp(s_ht - lse_h)           K^ = codebook[code] norm/sqrt(pd)
//      o_h  = s FWHT(sum_t p_ht V^_t)/sqrt(pd)
//      weights[t] += sum of p_ht over the heads h of the group
//    A weight needs its head's normaliser, which is known only after every
//    key has been read, and a sum over heads cannot be corrected afterwards by
//    one factor.  So the keys are read in one kernel that leaves the scores
//    (fp32) and the splits' maxima and sums, and the values in a second one
//    that reads the scores back: normalised probabilities come out of one
//    exp2, go into the product with V and into the weights, and the splits of
//    a sequence join by plain sums.  The cache is read once; the scores cost
//    4 bytes per (token, q head) each way, against entry bytes (80 at head
//    size 128) per (token, kv head).
//  * tq_track_window: the last queries of a prompt chunk.  Their scores would
//    be far larger than the keys, so the keys are read twice instead: once
//    for the normalisers, once for the sums over the queries.
//
// Accuracy: the weights are fp32 sums that a long sequence is cut by, so the
// scores keep fp32 accuracy: q' and the codebook both enter the MFMAs as
// fp16 hi + lo pairs (22 bits), each scaled by a power of two that keeps the
// lo parts normal numbers.
#include <math.h>

#include <type_traits>

#include "tq_plan.h"

namespace tq {

namespace {

constexpr int kThreads = 512;  // 8 waves
constexpr int kWaves = 8;
constexpr float kNone = -0x1.fffffep127f;  // maximum of no scores (finite: no inf - inf)
constexpr float kLevelScale = 64.0f;

// ---- cached rows in LDS ----------------------------------------------------
// A workgroup serves a unit of one sequence's tokens for G kv heads, whose
// entries of one token are adjacent in the cache.  It streams them tile by
// tile (16 tokens) with direct-to-LDS copies of 1 KB; a step is TPS tiles, so
// that each of the 8 waves has NTW (tile, head) pairs a step whatever G is.
// Rows stand in LDS at an odd stride in 16-byte chunks (no bank conflicts
// between the 16 rows of a tile).
template <int PD, int G>
struct Rows {
  static constexpr int EBS = PD == 64 ? 48 : (PD == 128 ? 80 : 144);  // entry bytes
  static constexpr int CPT = G * EBS / 16;                   // chunks of a token row
  static constexpr int RCH = CPT | 1;                        // row stride in chunks
  static constexpr int ROWB = RCH * 16;
  static constexpr int NI = (kTile * RCH + 63) / 64;         // copies per tile
  static constexpr int TILEB = NI * 1024;
  static constexpr int NTW = PD == 256 || (PD == 128 && G == 1) ? 1 : 2;
  static constexpr int SUB = kWaves / G;                     // waves per head
  static constexpr int TPS = NTW * SUB;                      // tiles per step
  static constexpr int NJOB = TPS * NI;                      // copies per step
  static constexpr int NJ = (NJOB + kWaves - 1) / kWaves;    // copies per wave
  static constexpr int SLOT = TPS * TILEB;
  static constexpr int SPARE = NJOB % kWaves ? 1024 : 0;     // where unused copies go
  static constexpr int RING = 2 * SLOT + SPARE;
};

struct TrackParams {
  const uint8_t* slab;  // the K or V slab
  const int32_t* indices;
  const int32_t* indptr;
  const int32_t* seq_lens;
  int64_t entries;  // of the page table
  int num_blocks, B, Hq, Hkv, ratio, rp, block_size, HG, units;
  int pair;       // see share_of
  int rows;       // parts of the plan at most: units, or twice as many
  const void* q;
  int64_t q_sb, q_sh;
  int q_bf16, hd;
  const float* signs;
  float csc;  // score constant (log2 units)
  float osc;  // output constant
  // scores, log2 units: [tile of the table][Hkv][ratio][16], or by_page, where the
  // cache has fewer pages than the table entries, [page][Hkv][tile][ratio][16]
  float* s;
  int by_page;
  float2* stats;  // (max, sum) [Hkv][rows][rp]
  int32_t* split;
  float* po;  // partial outputs [rows][Hq][PD]
  float* weights;
  int32_t* positions;
  const int32_t* ends;
};

// The unit that workgroup `u` serves (plan_slot of tq_plan.h), `per` parts a
// unit; st: at least 8 KB of LDS, free again afterwards.
template <int A, typename Params>
__device__ __forceinline__ PlanSlot unit_of(const Params& p, int* st, int u, int per,
                                            bool writer) {
  const int lane = threadIdx.x & 63;
  if (p.B <= 64) {
    const bool in = lane < p.B;
    const int len = in ? max(p.seq_lens[lane], 0) : 0;
    const int ip = in ? p.indptr[lane] : 0;
    return plan_slot<A>([&](int) { return len; }, [&](int) { return ip; }, p.B, 1, p.units, u, per,
                        p.split, writer);
  }
  for (int i = threadIdx.x; i < kPlanMost; i += blockDim.x) {
    st[i] = i < p.B ? max(p.seq_lens[i], 0) : 0;
    st[kPlanMost + i] = i < p.B ? p.indptr[i] : 0;
  }
  __syncthreads();
  const PlanSlot r =
      plan_slot<A>([&](int i) { return st[64 * i + lane]; },
                   [&](int i) { return st[kPlanMost + 64 * i + lane]; }, p.B, (p.B + 63) >> 6,
                   p.units, u, per, p.split, writer);
  __syncthreads();
  return r;
}

// What a workgroup of the two streaming kernels serves: tokens [c0, c1) of the
// unit's sequence, for head group hg, as part `row` of the plan's.
//
// pair > 0: the grid is two workgroups a CU, and blocks u and u + grid / 2 share a
// unit: the one that came first gets `pair` percent of its tokens (rounded up to a
// tile).  Alone on the card the two were seen on one CU; the older one's waves win
// the arbitration there, so of two equal shares the second finished 10 of 42 us
// later at 8 x 32768 tokens.  Nothing but the time rests on where they run: beside
// other streams the shares are just uneven.
struct Share {
  PlanSlot ps;
  int c0, c1, hg, row;
};
__device__ __forceinline__ Share share_of(const TrackParams& p, int* st, bool writer) {
  const int half = gridDim.x >> 1;
  const int second = p.pair > 0 && (int)blockIdx.x >= half;
  const int bid = blockIdx.x - second * half, per = p.pair > 0 ? 2 : 1;
  Share s;
  s.hg = bid % p.HG;
  s.ps = unit_of<kPlanAlign>(p, st, bid / p.HG, per, writer);
  s.c0 = s.ps.j * s.ps.U;
  s.c1 = s.c0 + s.ps.U;
  if (p.pair > 0) {
    // (64 bits: a sequence may have up to 2^30 tokens)
    const int first = (int)(((int64_t)s.ps.U * p.pair / 100 + 15) & ~(int64_t)15);
    const int cut = s.c0 + min(first, s.ps.U);
    s.c0 = second ? cut : s.c0;
    s.c1 = second ? s.c1 : cut;
  }
  s.c0 = min(s.c0, s.ps.L);
  s.c1 = min(s.c1, s.ps.L);
  s.row = per * (s.ps.Pb + s.ps.j) + second;
  return s;
}

// A unit's tiles: where each lies, and the copies of a step.  Lane i of a
// window holds what concerns tile 64 k + i: `at` its place in the cache in
// tiles (page * tiles per page + place in the page; -1 outside the unit, the
// table or the cache) and `wt` its place in the weights of kv head 0 (or -1).  Two
// windows cover any three steps in a row, and tiles are looked up by readlane:
// a load here would make the compiler wait for the copies in flight.
template <int PD, int G>
struct Stream {
  using R = Rows<PD, G>;
  const TrackParams& p;
  int tile0, tiles;  // first tile of the sequence, tiles of the unit
  int ip, tpp;       // first table entry of the sequence, tiles per page
  int row0;          // the unit's first tile in the table
  int w;
  int base, at0, at1, wt0, wt1;  // windows base and base + 1
  uint32_t goff[R::NJ];  // source offsets of this lane's copies inside a tile

  __device__ __forceinline__ Stream(const TrackParams& pp, const PlanSlot& ps, int c0, int c1,
                                    int wave, int hg)
      : p(pp), tile0(c0 / kTile), tiles((c1 - c0 + kTile - 1) / kTile), ip(ps.ip),
        tpp(pp.block_size / kTile), row0((int)((uint32_t)ps.ip * (uint32_t)tpp) + tile0), w(wave), base(0) {
    const int lane = threadIdx.x & 63;
    const int stride = p.Hkv * R::EBS;
    window(0, at0, wt0);
    window(1, at1, wt1);
#pragma unroll
    for (int i = 0; i < R::NJ; i++) {
      // lanes past the rows reload the last chunk (into the tile's slack), the
      // pad chunk of a row the row's last
      const int pos = min((w + kWaves * i) % R::NI * 64 + lane, kTile * R::RCH - 1);
      goff[i] = (uint32_t)(pos / R::RCH * stride + hg * G * R::EBS +
                           min(pos % R::RCH, R::CPT - 1) * 16);
    }
  }
  __device__ __forceinline__ void window(int k, int& at, int& wt) const {
    const int t = 64 * k + (threadIdx.x & 63), g = tile0 + t;
    at = -1;
    wt = -1;
    const int64_t e = (int64_t)ip + g / tpp;
    if (t < tiles && e >= 0 && e < p.entries) {
      const int pg = p.indices[e];
      if (pg >= 0 && pg < p.num_blocks) {
        at = pg * tpp + g % tpp;
        wt = pg * p.Hkv * tpp + g % tpp;
      }
    }
  }
  // moves the windows on when step s starts behind the first one
  __device__ __forceinline__ void advance(int s) {
    if (s * R::TPS < 64 * (base + 1)) return;
    base++;
    at0 = at1;
    wt0 = wt1;
    window(base + 1, at1, wt1);
#if defined(__HIP_DEVICE_COMPILE__)
    // the loads end here, not at the first use on every path
    asm volatile("s_waitcnt vmcnt(0)" : "+v"(at1), "+v"(wt1));
#endif
  }
  // place of tile t in the cache, -1: none
  __device__ __forceinline__ int place(int t) const {
    return __builtin_amdgcn_readlane(t < 64 * (base + 1) ? at0 : at1, t & 63);
  }
  // the tile's place in kv head kvh's weights, in tiles, -1: none
  __device__ __forceinline__ int weight_tile(int t, int kvh) const {
    const int x = __builtin_amdgcn_readlane(t < 64 * (base + 1) ? wt0 : wt1, t & 63);
    return x < 0 ? -1 : x + kvh * tpp;
  }
  // ... of its scores, of a tile at weight_tile() w (the first one's if there is
  // none).  Pages stand once in the tables, so that the scores of a table that is
  // wider than the cache (rows padded to the longest context) take no more room than
  // the cache's tokens.
  __device__ __forceinline__ uint32_t score_tile(int t, int w, int kvh) const {
    const uint32_t row = ((uint32_t)row0 + t) * p.Hkv + kvh;
    return w < 0 ? 0u : p.by_page ? (uint32_t)w : row;
  }
  // the copies of step s into the slot at `dst` (spare: where a wave's copy
  // beyond the step's goes); every wave issues NJ of them, whatever they read:
  // the waits count them
  __device__ __forceinline__ void issue(int s, uint8_t* dst, uint8_t* spare) const {
#if defined(__HIP_DEVICE_COMPILE__)
    const int64_t stride = (int64_t)p.Hkv * R::EBS;
#pragma unroll
    for (int i = 0; i < R::NJ; i++) {
      const int j = w + kWaves * i;
      const bool in = R::SPARE == 0 || j < R::NJOB;
      const int at = in ? place(s * R::TPS + j / R::NI) : -1;
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(p.slab + (int64_t)max(at, 0) * (kTile * stride)), (short)0,
          at >= 0 ? (int)(kTile * stride) : 0, 0x00020000);
      uint8_t* to = in ? dst + j / R::NI * R::TILEB + j % R::NI * 1024 : spare;
      // non-temporal: every line is read once
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (void*)to, 16, goff[i], 0, 0, 2);
    }
#else
    (void)s; (void)dst; (void)spare;
#endif
  }
};

// a barrier without the wait for the copies in flight that __syncthreads adds
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}
// this wave's LDS writes are done (before a barrier())
__device__ __forceinline__ void lds_written() {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#endif
}

// 4-bit level of nibble n
__device__ __forceinline__ float level(int n) {
  const int m = n >= 8 ? n - 8 : 7 - n;
  float v = codebook(8);
#pragma unroll
  for (int i = 1; i < 8; i++) v = m == i ? codebook(8 + i) : v;
  return n >= 8 ? v : -v;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, half2_t{(_Float16)a, (_Float16)b});
}

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }
// x times the fp16 value in the low half of n.  Not the assembly of
// mul_lo_half: its operands here come straight from an MFMA or an exp2, whose
// wait states the compiler counts for its own instructions only.
__device__ __forceinline__ float by_half(float x, uint32_t n) {
  return __builtin_fmaf(x, lo_half(n), 0.f);
}

// The key table: code byte -> fp16 hi parts of its two levels (high nibble
// first, as the dims go) in the low dword, their lo parts in the high one,
// times kLevelScale; 2^LOG copies, lane l reads copy l mod 2^LOG.  Two entries are a
// whole MFMA operand (hi, lo, hi, lo of two dims each) against q' with every
// pair of dims twice: with hi and lo parts in operands of their own each entry
// would cost two moves.
template <int LOG>  // log2 of the copies
__device__ __forceinline__ void init_key_table(uint64_t* lut) {
  // a byte's copies are shared by blockDim.x / 256 threads, two copies a store
  const int per = (256 << LOG) / blockDim.x, byte = threadIdx.x * 256 / blockDim.x;
  const float a = level(byte >> 4) * kLevelScale, b = level(byte & 15) * kLevelScale;
  const float ah = (float)(_Float16)a, bh = (float)(_Float16)b;
  const uint32_t hi = pack_half(ah, bh), lo = pack_half(a - ah, b - bh);
  u32x4* const to = reinterpret_cast<u32x4*>(lut + threadIdx.x * per);
#pragma unroll
  for (int i = 0; i < 1 << LOG; i += 2)
    if (i < per) to[i / 2] = u32x4{hi, lo, hi, lo};
}
// the two operands of 8 codes; lanec = 8 * (lane mod the copies)
template <int LOG>
__device__ __forceinline__ void key_operands(uint32_t c, const uint64_t* lut, uint32_t lanec,
                                             half8_t& k0, half8_t& k1) {
  uint64_t e[4];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t h = lut_spread(c, i);
    const uint8_t* const t = reinterpret_cast<const uint8_t*>(lut);
    e[2 * i] = *reinterpret_cast<const uint64_t*>(t + lut_mad<LOG + 3, 0>(h, lanec));
    e[2 * i + 1] = *reinterpret_cast<const uint64_t*>(t + lut_mad<LOG + 3, 1>(h, lanec));
  }
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  k0 = __builtin_bit_cast(half8_t, u64x2{e[0], e[1]});
  k1 = __builtin_bit_cast(half8_t, u64x2{e[2], e[3]});
}
// q' of 8 dims with every pair of dims twice
__device__ __forceinline__ void twice(half8_t q, half8_t& q0, half8_t& q1) {
  const u32x4 v = __builtin_bit_cast(u32x4, q);
  q0 = __builtin_bit_cast(half8_t, u32x4{v[0], v[0], v[1], v[1]});
  q1 = __builtin_bit_cast(half8_t, u32x4{v[2], v[2], v[3], v[3]});
}

// the codes of a tile (or of two) and a norm, from LDS: one block that ends
// with its own wait, as the compiler does not see these reads
template <int PD>
__device__ __forceinline__ void read_keys(uint32_t row, uint32_t nrm, uint32_t* c, uint32_t& n) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (PD == 64) {
    u32x2 a;
    asm volatile("ds_read_b64 %0, %2\n\tds_read_u16 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(a), "=&v"(n) : "v"(row), "v"(nrm) : "memory");
    c[0] = a[0]; c[1] = a[1];
  } else if constexpr (PD == 128) {
    u32x4 a;
    asm volatile("ds_read_b128 %0, %2\n\tds_read_u16 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(a), "=&v"(n) : "v"(row), "v"(nrm) : "memory");
    c[0] = a[0]; c[1] = a[1]; c[2] = a[2]; c[3] = a[3];
  } else {
    u32x4 a, b;
    asm volatile("ds_read_b128 %0, %3\n\tds_read_b128 %1, %3 offset:16\n\tds_read_u16 %2, %4\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(a), "=&v"(b), "=&v"(n) : "v"(row), "v"(nrm) : "memory");
    c[0] = a[0]; c[1] = a[1]; c[2] = a[2]; c[3] = a[3];
    c[4] = b[0]; c[5] = b[1]; c[6] = b[2]; c[7] = b[3];
  }
#else
  (void)row; (void)nrm; (void)c; n = 0;
#endif
}
template <int PD>  // 64 or 128
__device__ __forceinline__ void read_key_pair(uint32_t row0, uint32_t row1, uint32_t nrm,
                                              uint32_t (*c)[PD / 32], uint32_t& n) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef typename std::conditional<PD == 128, u32x4, u32x2>::type KT;
  KT a, b;
  if constexpr (PD == 128)
    asm volatile("ds_read_b128 %0, %3\n\tds_read_b128 %1, %4\n\tds_read_u16 %2, %5\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(a), "=&v"(b), "=&v"(n) : "v"(row0), "v"(row1), "v"(nrm) : "memory");
  else
    asm volatile("ds_read_b64 %0, %3\n\tds_read_b64 %1, %4\n\tds_read_u16 %2, %5\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(a), "=&v"(b), "=&v"(n) : "v"(row0), "v"(row1), "v"(nrm) : "memory");
#pragma unroll
  for (int k = 0; k < PD / 32; k++) {
    c[0][k] = a[k];
    c[1][k] = b[k];
  }
#else
  (void)row0; (void)row1; (void)nrm; (void)c; n = 0;
#endif
}

// the norms of tokens 4 * (l/16) .. + 3, each lane holding that of l % 4
__device__ __forceinline__ void spread_norms(uint32_t n, uint32_t* v) {
  v[0] = quad_bcast<0>(n);
  v[1] = quad_bcast<1>(n);
  v[2] = quad_bcast<2>(n);
  v[3] = quad_bcast<3>(n);
}

// running maximum and sum of exp2 over four more scores
__device__ __forceinline__ void add_scores(const float4_t& x, float& m, float& l) {
#pragma clang fp contract(off)  // (scores that are stored rounded)
  const float mx = vmax3(vmax3(m, x[0], x[1]), x[2], x[3]);
  float e = 0.f;
#pragma unroll
  for (int r = 0; r < 4; r++) e += exp2_raw(x[r] - mx);
  l = l * exp2_raw(m - mx) + e;
  m = mx;
}
// two (maximum, sum) pairs
__device__ __forceinline__ void join_stats(float om, float ol, float& m, float& l) {
  const float mx = vmax(m, om);
  l = l * exp2_raw(m - mx) + ol * exp2_raw(om - mx);
  m = mx;
}

// FWHT over the 64 lanes' PD / 64 elements each (element lane * E + k)
template <int E>
__device__ __forceinline__ void fwht_wave(float* x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int h = 1; h < E; h <<= 1)
#pragma unroll
    for (int k = 0; k < E; k++)
      if (!(k & h)) {
        const float a = x[k], b = x[k + h];
        x[k] = a + b;
        x[k + h] = a - b;
      }
#pragma unroll
  for (int h = 1; h < 64; h <<= 1)
#pragma unroll
    for (int k = 0; k < E; k++) {
      const float o = xor_lane(x[k], h);
      x[k] = lane & h ? o - x[k] : x[k] + o;
    }
}

// A row of hd elements (fp16 or bf16): lane l holds dims l * E .. + E - 1, zero
// past hd
template <int E>
__device__ __forceinline__ void load_row(const void* q, int64_t off, bool bf16, int hd, float* x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < E; k++) {
    const int d = lane * E + k;
    const int64_t at = off + min(d, hd - 1);
    const uint16_t v = static_cast<const uint16_t*>(q)[at];
    const float f = bf16 ? __uint_as_float((uint32_t)v << 16)
                         : (float)__builtin_bit_cast(_Float16, v);
    x[k] = d < hd ? f : 0.f;
  }
}
// this lane's rotation signs (1 without them)
template <int E>
__device__ __forceinline__ void load_signs(const float* signs, float* s) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < E; k++) s[k] = signs ? signs[lane * E + k] : 1.f;
}
// ... and rotated: FWHT(s x)/sqrt(pd); without signs (rotate false) as it is
template <int E>
__device__ __forceinline__ void rotate_row(bool rotate, const float* s, float* x) {
  if (!rotate) return;
#pragma unroll
  for (int k = 0; k < E; k++) x[k] *= s[k];
  fwht_wave<E>(x);
  const float isq = 1.0f / sqrtf((float)(64 * E));
#pragma unroll
  for (int k = 0; k < E; k++) x[k] *= isq;
}
// The power of two that brings a row's largest magnitude into [128, 256), as an
// exponent: x * 2^e = hi + lo to 22 bits, the lo parts of the large elements
// normal numbers (and not below 2^-100: what it is taken out by stays one too).
__device__ __forceinline__ int row_exponent(float mx) {
  return mx > 0.f && mx < INFINITY ? min(100, 7 - ilogbf(mx)) : 0;
}

// ---- the keys: scores, and the splits' maxima and sums ----------------------
// MFMA 16x16x32: A = a tile's keys (row = token), B = q' (column = q head).
// QC (at most 8 q heads per kv head): columns 0-7 hold the hi parts of q',
// 8-15 the lo parts, so the products with the hi and the lo parts of the keys
// add up all four terms in one accumulator.  PACK (then, where a wave has two
// tiles a step): lanes n < 8 take on the scores of the first tile and n >= 8
// those of the second, which halves the work per score.
//
// Bound by memory.  8 x 32768 tokens, 32 q / 8 kv heads of 128: 44.4 us for 169
// MB read and 34 MB of scores written; 5.4 TB/s while it streams, and 6-8 us are
// the prologue (plan, q', table) in front of the first step.  At head sizes 64 and
// 256 (28.4 and 29.7 us for 103 and 86 MB) the prologue is a quarter of it and VALU
// instructions are issued in 58 and 64% of the busy cycles.  Measured and
// not kept, for the sum of a call's three kernels (114 us in that run): the next
// two or four steps touched in L2 during the prologue, no gain and 3% slower;
// one workgroup of 16 waves a CU instead of two of 8, 2% slower there and 11 to
// 27% on shorter calls.
template <int PD, int G, bool QC>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(PD == 256 && !QC ? 2 : 4)))
void track_scores_kernel(TrackParams p) {
  using R = Rows<PD, G>;
  constexpr int KB = PD / 32;
  constexpr bool PACK = QC && PD <= 128 && R::NTW == 2;
  constexpr int NS = PACK ? 1 : R::NTW;  // score sets
  struct __attribute__((aligned(16))) Lds {
    uint64_t lut[4096];
    uint8_t ring[R::RING];
  };
  __shared__ Lds sm;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q4 = lane >> 4, n = lane & 15;
  const Share sh = share_of(p, reinterpret_cast<int*>(sm.lut), blockIdx.x == 0 && w == 0);
  const PlanSlot& ps = sh.ps;
  if (ps.b < 0) return;
  const int c0 = sh.c0, c1 = sh.c1, hg = sh.hg;
  const int kvh = hg * G + w % G, sub = w / G;
  if (c0 >= c1) {  // a short unit's second share (uniform)
    if (sub == 0 && lane < p.rp)
      p.stats[((int64_t)kvh * p.rows + sh.row) * p.rp + lane] = make_float2(kNone, 0.f);
    return;
  }
  Stream<PD, G> st(p, ps, c0, c1, w, hg);
  const int steps = (st.tiles + R::TPS - 1) / R::TPS;
  const int head = QC ? n & 7 : n;
  // q' of the workgroup's heads: each wave rotates every eighth row into LDS
  // (where the table goes later), fp32 with the 16-byte pieces of a row in an
  // order of its own (no bank conflicts between rows); then each lane takes its
  // column's dims, scales them by the row's power of two and splits them.
  constexpr int E = PD / 64, NB = 4;  // rows loaded at a time
  const int rows = G * p.ratio;
  float* const rot = reinterpret_cast<float*>(sm.lut);
  const int64_t q_at = (int64_t)ps.b * p.q_sb + (int64_t)hg * rows * p.q_sh;
  // (every load of the prologue goes out in front of the copies: a later one
  // would wait for them)
  float x0[NB][E], sg[E];
  load_signs<E>(p.signs, sg);
#pragma unroll
  for (int i = 0; i < NB; i++)
    load_row<E>(p.q, q_at + min(w + kWaves * i, rows - 1) * p.q_sh, p.q_bf16, p.hd, x0[i]);
  uint8_t* const spare = sm.ring + 2 * R::SLOT;
  st.issue(0, sm.ring, spare);
  st.issue(1, sm.ring + R::SLOT, spare);
  for (int r0 = w; r0 < rows; r0 += NB * kWaves) {
    if (r0 != w)
#pragma unroll
      for (int i = 0; i < NB; i++)
        load_row<E>(p.q, q_at + min(r0 + kWaves * i, rows - 1) * p.q_sh, p.q_bf16, p.hd, x0[i]);
#pragma unroll
    for (int i = 0; i < NB; i++) {
      const int r = r0 + kWaves * i;
      if (r >= rows) break;
      rotate_row<E>(p.signs != nullptr, sg, x0[i]);
#pragma unroll
      for (int k = 0; k < E; k++) {
        const int d = lane * E + k;
        rot[r * PD + (((d >> 2) ^ (r & 7)) << 2) + (d & 3)] = x0[i][k];
      }
    }
  }
  lds_written();
  barrier();
  half8_t qa[2 * KB], qb[QC ? 1 : 2 * KB];
  float csc = 0.f;
  {
    const int r = w % G * p.ratio + min(head, p.ratio - 1);
    float x[8 * KB], mx = 0.f;
#pragma unroll
    for (int k = 0; k < 2 * KB; k++) {
      const int piece = (PD / 16) * q4 + k;
      const float4_t v =
          *reinterpret_cast<const float4_t*>(rot + r * PD + ((piece ^ (r & 7)) << 2));
#pragma unroll
      for (int j = 0; j < 4; j++) {
        x[4 * k + j] = v[j];
        mx = fmaxf(mx, fabsf(v[j]));
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const int ex = row_exponent(mx);
    const bool real = head < p.ratio;
    csc = real ? ldexpf(p.csc, -ex) : 0.f;
#pragma unroll
    for (int k = 0; k < KB; k++) {
      half8_t hi, lo;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float v = real ? ldexpf(x[8 * k + j], ex) : 0.f;
        hi[j] = (_Float16)v;
        lo[j] = (_Float16)(v - (float)hi[j]);
      }
      if constexpr (QC) {
        twice(n < 8 ? hi : lo, qa[2 * k], qa[2 * k + 1]);
      } else {
        twice(hi, qa[2 * k], qa[2 * k + 1]);
        twice(lo, qb[2 * k], qb[2 * k + 1]);
      }
    }
  }
  lds_written();
  barrier();  // every wave has its q'
  init_key_table<4>(sm.lut);
  lds_written();

  const int mine = PACK && n >= 8 ? R::SUB : 0;  // this lane's tile behind the wave's first
  const uint32_t ring = lds_addr(sm.ring);
  const uint32_t o_row = sub * R::TILEB + n * R::ROWB + w % G * R::EBS + q4 * (PD / 8);
  const uint32_t o_nrm = (sub + mine) * R::TILEB + (4 * q4 + (lane & 3)) * R::ROWB +
                         w % G * R::EBS + PD / 2;
  const uint32_t lanec = 8 * n;
  // this lane's scores inside a tile's
  float* const s_at = p.s + head * kTile + 4 * q4;
  const uint32_t tile_floats = p.ratio * kTile;
  float m = kNone, l = 0.f;
  float4_t sc[NS];
  float* to[NS];  // where they go
  bool keep[NS];

  auto store = [&] {  // the scores of a step
#pragma unroll
    for (int i = 0; i < NS; i++)
      if (keep[i]) *reinterpret_cast<float4_t*>(to[i]) = sc[i];
  };
  const bool store_lane = head < p.ratio && (PACK || n < p.ratio);

  for (int s = 0; s < steps; s++) {
    st.advance(s);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(R::NJ));
    barrier();  // the copies of step s have landed (and the table is there)
    uint32_t c[R::NTW][PD / 32], nr[NS];
    const uint32_t at = ring + (s & 1) * R::SLOT;
    if constexpr (PACK) {
      read_key_pair<PD>(at + o_row, at + o_row + R::SUB * R::TILEB, at + o_nrm, c, nr[0]);
    } else {
#pragma unroll
      for (int i = 0; i < R::NTW; i++)
        read_keys<PD>(at + o_row + R::SUB * R::TILEB * i, at + o_nrm + R::SUB * R::TILEB * i, c[i],
                      nr[i]);
    }
    if (s) store();
    barrier();  // every wave has read the slot
    st.issue(s + 2, sm.ring + (s & 1) * R::SLOT, spare);
    float4_t acc[R::NTW];
#pragma unroll
    for (int i = 0; i < R::NTW; i++) {
      acc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KB; k++) {
        half8_t k0, k1;
        key_operands<4>(c[i][k], sm.lut, lanec, k0, k1);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qa[2 * k], acc[i], 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qa[2 * k + 1], acc[i], 0, 0, 0);
        if constexpr (!QC) {
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qb[2 * k], acc[i], 0, 0, 0);
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qb[2 * k + 1], acc[i], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NS; i++) {
      const int t0 = s * R::TPS + sub + R::SUB * i;
      float4_t x;
      if constexpr (PACK) {
        x = pack_merge(acc[0], acc[R::NTW - 1]);
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = QC ? acc[i][r] + ror8(acc[i][r]) : acc[i][r];
      }
      uint32_t nv[4];
      spread_norms(nr[i], nv);
#pragma unroll
      for (int r = 0; r < 4; r++) x[r] = by_half(x[r], nv[r]) * csc;
      // all tokens of the tiles are there (uniform); else masks
      const int tl = PACK ? t0 + R::SUB : t0;  // the last tile
      const int p0 = st.weight_tile(t0, kvh), p1 = PACK ? st.weight_tile(tl, kvh) : p0;
      const uint32_t a0 = st.score_tile(t0, p0, kvh);
      to[i] = s_at + (uint64_t)(mine ? st.score_tile(tl, p1, kvh) : a0) * tile_floats;
      keep[i] = store_lane;
      if (p0 < 0 || p1 < 0 || (st.tile0 + tl + 1) * kTile > c1) {
        const bool there = (mine ? p1 : p0) >= 0;
        keep[i] = keep[i] && there;
        const int left = c1 - (st.tile0 + t0 + mine) * kTile - 4 * q4;
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = there && r < left ? x[r] : -INFINITY;
      }
      sc[i] = x;
      add_scores(x, m, l);
    }
  }
  store();
  // no copy may land after the workgroup's LDS is given away
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  // a head's lanes meet: its other tile's, then the token groups
  if constexpr (PACK) join_stats(ror8(m), ror8(l), m, l);
  join_stats(__shfl_xor(m, 16), __shfl_xor(l, 16), m, l);
  join_stats(__shfl_xor(m, 32), __shfl_xor(l, 32), m, l);
  if constexpr (R::SUB > 1) {  // the waves of a head, in LDS that nobody reads any more
    float2* const all = reinterpret_cast<float2*>(sm.ring);
    barrier();
    if (lane < 16) all[w * 16 + lane] = make_float2(m, l);
    lds_written();
    barrier();
    if (sub == 0)
#pragma unroll
      for (int i = 1; i < R::SUB; i++) {
        const float2 o = all[(w + i * G) * 16 + (lane & 15)];
        join_stats(o.x, o.y, m, l);
      }
  }
  if (sub == 0 && lane < p.rp)
    p.stats[((int64_t)kvh * p.rows + sh.row) * p.rp + lane] =
        lane < p.ratio ? make_float2(m, l) : make_float2(kNone, 0.f);
}

// V codes of tokens 4 * (l/16) .. + 3 (PD / 32 bytes each) of NT tiles and one
// norm
template <int PD, int G, int NT>
__device__ __forceinline__ void read_values(uint32_t row0, uint32_t row1, uint32_t nrm,
                                            uint32_t (*c)[PD == 256 ? 2 : 1][4], uint32_t& n) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int S = Rows<PD, G>::ROWB;
#define TQ_V8(OP)                                                                               \
  OP " %0, %9\n\t" OP " %1, %9 offset:%12\n\t" OP " %2, %9 offset:%13\n\t"                     \
  OP " %3, %9 offset:%14\n\t" OP " %4, %10\n\t" OP " %5, %10 offset:%12\n\t"                   \
  OP " %6, %10 offset:%13\n\t" OP " %7, %10 offset:%14\n\tds_read_u16 %8, %11\n\t"             \
     "s_waitcnt lgkmcnt(0)"
#define TQ_V4(OP)                                                                              \
  OP " %0, %5\n\t" OP " %1, %5 offset:%7\n\t" OP " %2, %5 offset:%8\n\t"                       \
  OP " %3, %5 offset:%9\n\tds_read_u16 %4, %6\n\ts_waitcnt lgkmcnt(0)"
  if constexpr (PD == 256) {
    static_assert(NT == 1, "one tile at a time");
    u32x2 a[4];
    asm volatile(TQ_V4("ds_read_b64")
                 : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(n)
                 : "v"(row0), "v"(nrm), "i"(S), "i"(2 * S), "i"(3 * S) : "memory");
#pragma unroll
    for (int j = 0; j < 4; j++) {
      c[0][0][j] = a[j][0];
      c[0][1][j] = a[j][1];
    }
  } else if constexpr (NT == 2) {
#define TQ_PAIR(OP)                                                                              \
  asm volatile(TQ_V8(OP)                                                                         \
               : "=&v"(c[0][0][0]), "=&v"(c[0][0][1]), "=&v"(c[0][0][2]), "=&v"(c[0][0][3]),     \
                 "=&v"(c[1][0][0]), "=&v"(c[1][0][1]), "=&v"(c[1][0][2]), "=&v"(c[1][0][3]),     \
                 "=&v"(n)                                                                        \
               : "v"(row0), "v"(row1), "v"(nrm), "i"(S), "i"(2 * S), "i"(3 * S) : "memory")
    if constexpr (PD == 64) TQ_PAIR("ds_read_u16");
    else TQ_PAIR("ds_read_b32");
#undef TQ_PAIR
  } else {
#define TQ_ONE(OP)                                                                               \
  asm volatile(TQ_V4(OP)                                                                         \
               : "=&v"(c[0][0][0]), "=&v"(c[0][0][1]), "=&v"(c[0][0][2]), "=&v"(c[0][0][3]),     \
                 "=&v"(n)                                                                        \
               : "v"(row0), "v"(nrm), "i"(S), "i"(2 * S), "i"(3 * S) : "memory")
    if constexpr (PD == 64) TQ_ONE("ds_read_u16");
    else TQ_ONE("ds_read_b32");
#undef TQ_ONE
  }
#undef TQ_V8
#undef TQ_V4
#else
  (void)row0; (void)row1; (void)nrm; (void)c; n = 0;
#endif
}

// The V levels are one fp16 each (a second one would double the table reads that
// feed the products): times this they lie within 8.7e-5 of fp16 grid points.
constexpr float kValueScale = 1.4809800386428833f;
// A wave scales the products probability x norm so that the largest one it has met
// stays below 2^kTop; where one passes that, below 2^kFresh.
constexpr int kTop = 15, kFresh = 11;
// Before the first product; a wave without any keeps it, and sums of up to 2^35 of
// others' products, taken to that scale, stay finite.
constexpr float kUnscaled = 0x1p60f;

// fp16 pair, towards zero (a hi part: the lo part takes up the rest)
__device__ __forceinline__ uint32_t pack_rtz(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
// nibble pairs of two tokens' code dwords: byte k indexes the levels (first
// token's nibble low) of dim 2k (even) and 2k + 1 (odd)
__device__ __forceinline__ void nibble_pairs(uint32_t a, uint32_t b, uint32_t& even,
                                             uint32_t& odd) {
  const uint32_t m4 = 0x0f0f0f0fu;
  odd = (a & m4) | ((b << 4) & ~m4);
  even = ((a >> 4) & m4) | (b & ~m4);
}

// ---- the values: output partials and the weights ----------------------------
// MFMA with A = V^T (row = dim slot), B = the probabilities in the layout of
// the scores' tile (16x16x16), or of a pair of tiles (PACK: 16x16x32, whose 8
// k-values of a lane are tokens 4 * (l/16) .. + 3 of either tile).  Dim of (row
// r, product i) is r * (PD/16) + i.  QC: columns 0-7 hold the hi parts of p *
// norm, 8-15 the lo parts; else p * norm is one fp16 (2^-12 relative, to nearest:
// a second operand would cost a product more for each).  Probabilities are
// relative to the sequence's maximum in the product and normalised at the end.
//
// p * norm has the range of fp32: V norms go down to 6e-8, and the tail of a
// long sequence holds most of its weight in small pieces.  So the norms are
// scaled by a power of two, which follows the largest p * norm that the wave has
// met: what hi and lo parts lose is below 2^-34 of that one.  Unscaled, rows of
// norm 0.01 lost up to a thousandth of such a tail and rows of norm 0.001 some
// percent.  The scale changes rarely (a uniform branch), the products so far
// with it; check and first change cost 0.5 to 1 us.
//
// Bound by memory: 44.8 us for 211 MB read (entries, scores, weights) and 17 MB
// written, sizes as above (32.5 and 29.5 us for 118 and 97 MB at head sizes 64 and
// 256, VALU issue in 65% of the busy cycles).  One kernel for keys and values and a
// small one for
// the weights would move the same bytes and save one prologue, at most 6%.
template <int PD, int G, bool QC>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4)))
void track_values_kernel(TrackParams p) {
  using R = Rows<PD, G>;
  constexpr int NO = PD / 16;           // products per tile
  constexpr int VW = PD == 256 ? 2 : 1;  // code dwords per token and lane
  constexpr bool PACK = QC && PD <= 128 && R::NTW == 2;
  constexpr int NS = PACK ? 1 : R::NTW;  // score sets
  constexpr int NT = PACK ? 2 : 1;       // tiles of a set
  struct __attribute__((aligned(16))) Lds {
    uint32_t lut[8192];  // code byte -> levels of its low and high nibble, 32 copies
    uint8_t ring[R::RING];
  };
  __shared__ Lds sm;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q4 = lane >> 4, n = lane & 15;
  const Share sh = share_of(p, reinterpret_cast<int*>(sm.lut), false);
  const PlanSlot& ps = sh.ps;
  if (ps.b < 0) return;
  const int c0 = sh.c0, c1 = sh.c1, hg = sh.hg;
  const int kvh = hg * G + w % G, sub = w / G;
  if (c0 >= c1) {  // (as above: a row of zeros)
    float* const row = p.po + ((int64_t)sh.row * p.Hq + hg * G * p.ratio) * PD;
    for (int i = threadIdx.x; i < G * p.ratio * PD; i += kThreads) row[i] = 0.f;
    return;
  }
  Stream<PD, G> st(p, ps, c0, c1, w, hg);
  const int steps = (st.tiles + R::TPS - 1) / R::TPS;
  const int head = QC ? n & 7 : n;
  const bool real = head < p.ratio;

  // the maximum and the sum of this lane's head over the sequence (the loads go
  // out in front of the copies, up to NP of them: a later one waits for the
  // copies)
  constexpr int NP = 8;
  float M = kNone, den = 0.f;
  const int per = p.pair > 0 ? 2 : 1;
  const int parts = (ps.L + ps.U - 1) / ps.U * per * p.rp;
  const float2* const src = p.stats + ((int64_t)kvh * p.rows + per * ps.Pb) * p.rp;
  float2 part[NP];
#pragma unroll
  for (int i = 0; i < NP; i++) part[i] = src[min(lane + 64 * i, parts - 1)];
  uint8_t* const spare = sm.ring + 2 * R::SLOT;
  st.issue(0, sm.ring, spare);
  st.issue(1, sm.ring + R::SLOT, spare);
#pragma unroll
  for (int i = 0; i < NP; i++)
    if (lane + 64 * i < parts) join_stats(part[i].x, part[i].y, M, den);
  for (int i = lane + 64 * NP; i < parts; i += 64) join_stats(src[i].x, src[i].y, M, den);
  for (int d = p.rp; d < 64; d <<= 1) join_stats(__shfl_xor(M, d), __shfl_xor(den, d), M, den);
  const float inv = real && den != 0.f ? 1.0f / den : 0.f;
  if (!real) M = INFINITY;  // lanes of no head: probabilities of zero
  {
    const int byte = threadIdx.x >> 1;  // two threads a byte, four copies a store
    const uint32_t e =
        pack_half(level(byte & 15) * kValueScale, level(byte >> 4) * kValueScale);
    u32x4* const to = reinterpret_cast<u32x4*>(sm.lut + threadIdx.x * 16);
#pragma unroll
    for (int i = 0; i < 4; i++) to[i] = u32x4{e, e, e, e};
  }
  lds_written();

  const int mine = PACK && n >= 8 ? R::SUB : 0;  // this lane's tile behind the wave's first
  const uint32_t ring = lds_addr(sm.ring);
  const uint32_t o_row = sub * R::TILEB + 4 * q4 * R::ROWB + w % G * R::EBS + n * (PD / 32);
  const uint32_t o_nrm = (sub + mine) * R::TILEB + (4 * q4 + (lane & 3)) * R::ROWB +
                         w % G * R::EBS + PD / 2;
  const uint32_t lanec = 4 * (lane & 31);
  const float* const s_at = p.s + min(head, p.ratio - 1) * kTile + 4 * q4;
  float* const w_at = p.weights + 4 * q4;
  const uint32_t tile_floats = p.ratio * kTile;
  float4_t O[NO];
#pragma unroll
  for (int i = 0; i < NO; i++) O[i] = float4_t{0.f, 0.f, 0.f, 0.f};
  float scale = kUnscaled;  // (uniform)

  // scores and weights of step s, loaded one step ahead of their use; lanes
  // whose tile is outside the unit or the cache read the arrays' start and are
  // masked
  struct Ahead {
    float4_t sc[NS], wt[NS];
    int at[NS];     // tiles of the weights, -1: none
    bool there[NS];  // all of a set's tiles are (uniform)
  } nx, cu;
  auto load = [&](int s, Ahead& a) {
#pragma unroll
    for (int i = 0; i < NS; i++) {
      const int t0 = s * R::TPS + sub + R::SUB * i;
      const int w0 = st.weight_tile(t0, kvh);
      const uint32_t s0 = st.score_tile(t0, w0, kvh);
      int at = w0;
      uint32_t of = s0;
      a.there[i] = w0 >= 0;
      if constexpr (PACK) {
        const int w1 = st.weight_tile(t0 + R::SUB, kvh);
        const uint32_t s1 = st.score_tile(t0 + R::SUB, w1, kvh);
        at = mine ? w1 : w0;
        of = mine ? s1 : s0;
        a.there[i] = w0 >= 0 && w1 >= 0;
      }
      a.at[i] = at;
      a.sc[i] = *reinterpret_cast<const float4_t*>(s_at + (uint64_t)of * tile_floats);
      a.wt[i] =
          *reinterpret_cast<const float4_t*>(w_at + (uint64_t)(uint32_t)max(at, 0) * kTile);
    }
  };
  const bool store_lane = PACK ? (n & 7) == 0 : n == 0;
  auto store = [&](const Ahead& a) {  // the weights of a step
#pragma unroll
    for (int i = 0; i < NS; i++)
      if (a.at[i] >= 0 && store_lane)
        *reinterpret_cast<float4_t*>(w_at + (uint64_t)(uint32_t)a.at[i] * kTile) = a.wt[i];
  };
  load(0, cu);

  for (int s = 0; s < steps; s++) {
    st.advance(s);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(R::NJ));
    barrier();
    uint32_t c[R::NTW][VW][4], nr[NS];
    const uint32_t at = ring + (s & 1) * R::SLOT;
#pragma unroll
    for (int i = 0; i < NS; i++)
      read_values<PD, G, NT>(at + o_row + R::SUB * R::TILEB * i,
                             at + o_row + R::SUB * R::TILEB * (i + 1),
                             at + o_nrm + R::SUB * R::TILEB * i, c + i, nr[i]);
    if (s) {
      store(cu);
      cu = nx;
    }
    load(s + 1, nx);
    barrier();
    st.issue(s + 2, sm.ring + (s & 1) * R::SLOT, spare);
#pragma unroll
    for (int i = 0; i < NS; i++) {
      const int t0 = s * R::TPS + sub + R::SUB * i, tl = PACK ? t0 + R::SUB : t0;
      uint32_t nv[4];
      spread_norms(__float_as_uint(lo_half(nr[i]) * scale), nv);
      float rel[4], g[4], x[4];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        rel[r] = exp2_raw(cu.sc[i][r] - M);
        x[r] = rel[r] * __uint_as_float(nv[r]);
      }
      // tiles with tokens that are not there, or with the newest one (uniform)
      const int first = (st.tile0 + t0 + mine) * kTile + 4 * q4;
      const bool whole = cu.there[i] && (st.tile0 + tl + 1) * kTile < ps.L;
      if (!whole) {
        const int left = cu.at[i] >= 0 ? c1 - first : 0;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          rel[r] = r < left ? rel[r] : 0.f;
          x[r] = r < left ? x[r] : 0.f;
        }
      }
      // this head's weights, summed over the group's heads
#pragma unroll
      for (int r = 0; r < 4; r++) {
        g[r] = rel[r] * inv;
        g[r] += xor_lane(g[r], 1);
        g[r] += xor_lane(g[r], 2);
        // (row_half_mirror: the other four of eight lanes, alike by now)
        g[r] += __int_as_float(
            __builtin_amdgcn_mov_dpp(__float_as_int(g[r]), 0x141, 0xf, 0xf, false));
        if constexpr (!QC) g[r] += ror8(g[r]);
      }
      if (whole) {
#pragma unroll
        for (int r = 0; r < 4; r++) cu.wt[i][r] += g[r];
      } else {
        const int left = c1 - first, last = ps.L - 1 - first;
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (r < left) cu.wt[i][r] = r == last ? g[r] : cu.wt[i][r] + g[r];
      }
      // B operand
      const float big = vmax3_abs(vmax3_abs(x[0], x[1], x[2]), x[3], 0.f);
      if (__any(big > (float)(1 << kTop))) {
        float mx = max_ror8(big);
        mx = vmax(mx, xor_lane(mx, 1));
        mx = vmax(mx, xor_lane(mx, 2));
        mx = vmax(mx, xor_lane(mx, 4));
        mx = xor32_max(xor16_max(mx));
        // (an infinite norm's outputs are no numbers whatever the scale)
        const float by = ldexpf(1.0f, kFresh - __builtin_amdgcn_frexp_expf(mx));
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] *= by;
        if (s || i)  // (else they are zero)
#pragma unroll
          for (int k = 0; k < NO; k++) O[k] *= by;
        scale = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(scale * by)));
      }
      uint32_t pb[4];
      if constexpr (QC) {
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          hi[j] = pack_rtz(x[2 * j], x[2 * j + 1]);
          lo[j] = pack_rtz(x[2 * j] - lo_half(hi[j]), x[2 * j + 1] - hi_half(hi[j]));
        }
        if constexpr (PACK) {
          // lanes n < 8 hold the first tile's, n >= 8 the second's: swap lo
          // parts against hi parts
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const uint32_t in = (uint32_t)__builtin_amdgcn_mov_dpp(
                (int)(mine ? hi[j] : lo[j]), 0x128, 0xf, 0xf, false);
            pb[j] = mine ? in : hi[j];
            pb[2 + j] = mine ? lo[j] : in;
          }
        } else {
          pb[0] = n < 8 ? hi[0] : lo[0];
          pb[1] = n < 8 ? hi[1] : lo[1];
        }
      } else {
        pb[0] = pack_half(x[0], x[1]);
        pb[1] = pack_half(x[2], x[3]);
      }
#pragma unroll
      for (int v = 0; v < VW; v++) {
        uint32_t ev[NT][2], od[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
          nibble_pairs(c[i + t][v][0], c[i + t][v][1], ev[t][0], od[t][0]);
          nibble_pairs(c[i + t][v][2], c[i + t][v][3], ev[t][1], od[t][1]);
        }
        constexpr int BY = PD == 64 ? 2 : 4;
        const uint8_t* const lut = reinterpret_cast<const uint8_t*>(sm.lut);
        auto entry = [&](uint32_t a) { return *reinterpret_cast<const uint32_t*>(lut + a); };
#pragma unroll
        for (int k = 0; k < BY; k += 2) {
          uint32_t a[4][2 * NT];  // dims 2k, 2k + 1, 2k + 2, 2k + 3
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const uint32_t he = lut_spread(ev[t][j], k / 2), ho = lut_spread(od[t][j], k / 2);
              a[0][2 * t + j] = entry(lut_mad<7, 0>(he, lanec));
              a[1][2 * t + j] = entry(lut_mad<7, 0>(ho, lanec));
              a[2][2 * t + j] = entry(lut_mad<7, 1>(he, lanec));
              a[3][2 * t + j] = entry(lut_mad<7, 1>(ho, lanec));
            }
#pragma unroll
          for (int d = 0; d < 4; d++) {
            float4_t& acc = O[8 * v + 2 * k + d];
            if constexpr (PACK)
              acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  __builtin_bit_cast(half8_t, u32x4{a[d][0], a[d][1], a[d][2 * NT - 2],
                                                    a[d][2 * NT - 1]}),
                  __builtin_bit_cast(half8_t, u32x4{pb[0], pb[1], pb[2], pb[3]}), acc, 0, 0, 0);
            else
              acc = __builtin_amdgcn_mfma_f32_16x16x16f16(
                  __builtin_bit_cast(half4_t, u32x2{a[d][0], a[d][1]}),
                  __builtin_bit_cast(half4_t, u32x2{pb[0], pb[1]}), acc, 0, 0, 0);
          }
        }
      }
    }
  }
  store(cu);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // (as above)
  if (p.positions && c1 == ps.L && sub == 0 && lane == 0) {  // the newest token's
    const int t = c1 - 1;
    const int64_t e = (int64_t)ps.ip + t / p.block_size;
    const int pg = e >= 0 && e < p.entries ? p.indices[e] : -1;
    if (pg >= 0 && pg < p.num_blocks)
      p.positions[((int64_t)pg * p.Hkv + kvh) * p.block_size + t % p.block_size] =
          p.ends[ps.b] - 1;
  }
  if constexpr (QC) {  // hi and lo columns
#pragma unroll
    for (int i = 0; i < NO; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) O[i][r] += ror8(O[i][r]);
  }
  // the waves of a head meet in LDS, halving their number each time; a sum has the
  // scale of the wave that goes on
#pragma unroll
  for (int half = R::SUB / 2; half > 0; half /= 2) {
    float4_t* const buf = reinterpret_cast<float4_t*>(&sm) + lane;
    float* const scales = reinterpret_cast<float*>(&sm + 1) - kWaves;
    static_assert(kWaves / 2 * NO * 1024 + kWaves * 4 <= sizeof(Lds),
                  "half the waves' outputs and their scales fit");
    barrier();
    if (sub >= half && sub < 2 * half) {
      scales[w - half * G] = scale;
#pragma unroll
      for (int i = 0; i < NO; i++) buf[((w - half * G) * NO + i) * 64] = O[i];
    }
    lds_written();
    barrier();
    if (sub < half) {
      const float by = scale / scales[w];
#pragma unroll
      for (int i = 0; i < NO; i++) O[i] += buf[(w * NO + i) * 64] * by;
    }
    lds_written();
  }
  if (sub == 0 && n < p.ratio) {
    float* const row = p.po + ((int64_t)sh.row * p.Hq + kvh * p.ratio + n) * PD;
    const float osc = inv * p.osc / scale;
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int i = 0; i < NO; i += 4)
        *reinterpret_cast<float4_t*>(row + (4 * q4 + r) * NO + i) =
            float4_t{O[i][r], O[i + 1][r], O[i + 2][r], O[i + 3][r]} * osc;
  }
}

// One row of hd elements rotated, scaled and split: x * scale = hi + lo.
// Returns 1 / scale.
template <int PD>
__device__ __forceinline__ float split_row(const void* q, int64_t off, bool bf16, int hd,
                                           const float* signs, _Float16* hi, _Float16* lo) {
  constexpr int E = PD / 64;
  float x[E], sg[E];
  load_row<E>(q, off, bf16, hd, x);
  load_signs<E>(signs, sg);
  rotate_row<E>(signs != nullptr, sg, x);
  float mx = 0.f;
#pragma unroll
  for (int k = 0; k < E; k++) mx = fmaxf(mx, fabsf(x[k]));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, xor_lane(mx, d));
  const int ex = row_exponent(mx);
#pragma unroll
  for (int k = 0; k < E; k++) {
    const float v = ldexpf(x[k], ex);
    hi[k] = (_Float16)v;
    lo[k] = (_Float16)(v - (float)hi[k]);
  }
  return ldexpf(1.0f, -ex);
}

// o = s FWHT(sum of the partial rows)/sqrt(pd): one workgroup per (sequence,
// q head), its four waves sharing the partial rows.  A launch and two dependent
// loads: 2.9 us for one sequence, 4.9 for 8 of 64 rows each.
template <int PD>
__global__ __launch_bounds__(256) void track_join_kernel(const float* __restrict__ po,
                                                         const int32_t* __restrict__ split,
                                                         int Hq, int hd, int bf16,
                                                         const float* __restrict__ signs,
                                                         void* __restrict__ o) {
  constexpr int E = PD / 64;
  __shared__ float part[3][PD];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int b = blockIdx.x / Hq, h = blockIdx.x % Hq;
  const int r0 = split[b], r1 = split[b + 1];
  float x[E];
#pragma unroll
  for (int k = 0; k < E; k++) x[k] = 0.f;
  const float* src = po + (int64_t)h * PD + lane * E;
#pragma unroll 4
  for (int r = r0 + wv; r < r1; r += 4) {
    const float* at = src + (int64_t)r * Hq * PD;
#pragma unroll
    for (int k = 0; k < E; k++) x[k] += at[k];
  }
  if (wv)
#pragma unroll
    for (int k = 0; k < E; k++) part[wv - 1][lane * E + k] = x[k];
  __syncthreads();
  if (wv) return;
#pragma unroll
  for (int i = 0; i < 3; i++)
#pragma unroll
    for (int k = 0; k < E; k++) x[k] += part[i][lane * E + k];
  if (signs) {
    fwht_wave<E>(x);
    const float isq = 1.0f / sqrtf((float)PD);
#pragma unroll
    for (int k = 0; k < E; k++) x[k] *= isq * signs[lane * E + k];
  }
  const int64_t at = ((int64_t)b * Hq + h) * hd;
#pragma unroll
  for (int k = 0; k < E; k++) {
    const int d = lane * E + k;
    if (d >= hd) break;
    if (bf16)
      static_cast<__bf16*>(o)[at + d] = (__bf16)x[k];
    else
      static_cast<_Float16*>(o)[at + d] = (_Float16)x[k];
  }
}

// ---- windows ---------------------------------------------------------------
// Rows of a (sequence, kv head): row i * ratio + h is q head h of the i-th of
// the last `window` queries (aligned to the end: the first ones are missing
// where the chunk is shorter), padded to whole tiles of 32.  MFMA 32x32x16:
// A = 32 keys (row = token), B = 32 rows of q'.  A wave keeps its keys'
// operands in registers and walks the rows, whose operands the rotation kernel
// has laid out in MFMA order.
struct WindowParams {
  const uint8_t* slab;  // K
  const int32_t* indices;
  const int32_t* indptr;
  const int32_t* seq_lens;
  const int32_t* q_start;  // [B + 1] rows of q
  int64_t entries;
  int num_blocks, B, Hkv, ratio, block_size, units, window, tiles;  // row tiles
  const half8_t* qf;  // [B][Hkv][tiles][PD/16][hi, lo][64 lanes]
  const float* qs;    // [B][Hkv][32 tiles]
  float csc;
  float2* stats;  // [Hkv][units of the first pass][32 tiles]
  float* lse;     // [B][Hkv][32 tiles] from window_lse_kernel; null: none ran
  int32_t* split;
  float* weights;
  int32_t* positions;
  const int32_t* ends;
};

// The rotated rows: hi and lo parts in the MFMA's order, and their scales; a wave
// a row (5 us for 2048 rows of 128: latency).
template <int PD>
__global__ __launch_bounds__(256) void rotate_window_kernel(
    const void* __restrict__ q, int64_t q_rows, int64_t q_sb, int64_t q_sh, int bf16, int hd,
    WindowParams p, const float* __restrict__ signs, _Float16* __restrict__ qf,
    float* __restrict__ qs) {
  constexpr int E = PD / 64;
  const int lane = threadIdx.x & 63;
  const uint32_t bt = blockIdx.x / 8;  // eight workgroups a tile, a row per wave
  const int tile = (int)(bt % (uint32_t)p.tiles), in = blockIdx.x % 8 * 4 + (threadIdx.x >> 6);
  const uint32_t bh = bt / (uint32_t)p.tiles;
  const int kvh = (int)(bh % (uint32_t)p.Hkv), b = (int)(bh / (uint32_t)p.Hkv);
  const int rho = tile * 32 + in;
  const int i = rho / p.ratio, h = rho % p.ratio;
  const int q0 = p.q_start[b], q1 = p.q_start[b + 1];
  const int64_t at = (int64_t)q1 - p.window + i;
  _Float16 hi[E] = {}, lo[E] = {};
  float inv = 0.f;
  if (i < p.window && at >= max(q0, 0) && at < q_rows)
    inv = split_row<PD>(q, at * q_sb + (int64_t)(kvh * p.ratio + h) * q_sh, bf16, hd, signs, hi,
                        lo);
  // dim d is element d % 8 of step (d % (PD / 2)) / 8 in lane half d / (PD / 2);
  // two dims a store, at head size 64 from two lanes (one stores hi, one lo)
  const int d = E == 1 ? lane & ~1 : lane * E;
  _Float16* const to = qf + (int64_t)bt * (PD / 16) * 1024 + d % (PD / 2) / 8 * 1024 +
                       (d / (PD / 2) * 32 + in) * 8 + d % 8;
  if constexpr (E == 1) {
    const uint32_t h16 = __builtin_bit_cast(uint16_t, hi[0]);
    const uint32_t l16 = __builtin_bit_cast(uint16_t, lo[0]);
    const bool odd = lane & 1;
    const uint32_t mine = odd ? l16 : h16, other = __shfl_xor(odd ? h16 : l16, 1);
    *reinterpret_cast<uint32_t*>(to + (odd ? 512 : 0)) =
        odd ? mine << 16 | other : other << 16 | mine;
  } else {
    typedef _Float16 row_t __attribute__((ext_vector_type(E)));
    row_t a, c;
#pragma unroll
    for (int k = 0; k < E; k++) a[k] = hi[k], c[k] = lo[k];
    *reinterpret_cast<row_t*>(to) = a;
    *reinterpret_cast<row_t*>(to + 512) = c;
  }
  if (lane == 0) qs[(int64_t)bt * 32 + in] = inv;
}

// hi and lo operands of 8 codes, in registers of their own
template <int LOG>
__device__ __forceinline__ void key_parts(uint32_t c, const uint64_t* lut, uint32_t lanec,
                                          half8_t& hi, half8_t& lo) {
  half8_t k0, k1;
  key_operands<LOG>(c, lut, lanec, k0, k1);
  const u32x4 a = __builtin_bit_cast(u32x4, k0), b = __builtin_bit_cast(u32x4, k1);
  hi = __builtin_bit_cast(half8_t, u32x4{a[0], a[2], b[0], b[2]});
  lo = __builtin_bit_cast(half8_t, u32x4{a[1], a[3], b[1], b[3]});
}

// A row's normaliser in log2 units from its maximum and sum.  Rows past the
// window or before the chunk's first query (scale 0) add nothing: +inf.
__device__ __forceinline__ float lse_of(float2 x, float scale) {
  return scale != 0.f && x.y != 0.f ? x.x + log2f(x.y) : INFINITY;
}
// (max, sum) of a row over units g, g + step, ... of n, `src` at the first one's
__device__ __forceinline__ float2 join_units(const float2* src, int stride, int g, int n,
                                             int step) {
  float2 a = make_float2(kNone, 0.f);
#pragma unroll 8
  for (int u = g; u < n; u += step) {
    const float2 x = src[(int64_t)u * stride];
    join_stats(x.x, x.y, a.x, a.y);
  }
  return a;
}

// The normalisers of a sequence's rows from its units' maxima and sums: a
// workgroup takes 32 rows, thread (r, g) their units g, g + 8, ...
__global__ __launch_bounds__(256) void window_lse_kernel(WindowParams p) {
  __shared__ float2 part[8][32];
  const int R = p.tiles * 32, r = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int tile = blockIdx.x % p.tiles;
  const int64_t bh = blockIdx.x / p.tiles;
  const int kvh = (int)(bh % p.Hkv), b = (int)(bh / p.Hkv);
  const int row = tile * 32 + r;
  const int u0 = p.split[b], u1 = p.split[b + 1];
  float2 a = join_units(p.stats + ((int64_t)kvh * p.units + u0) * R + row, R, g, u1 - u0, 8);
  part[g][r] = a;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int k = 1; k < 8; k++) join_stats(part[k][r].x, part[k][r].y, a.x, a.y);
  const int64_t at = bh * R + row;
  p.lse[at] = lse_of(a, p.qs[at]);
}

// All rows' normalisers into LDS (256 threads): window_lse_kernel's, or without
// it from the sequence's n units at u0 here, where half a wave takes a tile and,
// with fewer than 8 tiles, groups of them share its units.  (A barrier follows.)
__device__ __forceinline__ void row_lse(const WindowParams& p, int kvh, int64_t bh, int u0, int n,
                                        float2 (*part)[4][32], float* lse) {
  const int R = p.tiles * 32, r = threadIdx.x & 31, w = threadIdx.x >> 5;
  const float* const qs = p.qs + bh * R;
  if (p.lse) {
    for (int i = threadIdx.x; i < R; i += 256) lse[i] = p.lse[bh * R + i];
    return;
  }
  const float2* const src = p.stats + ((int64_t)kvh * p.units + u0) * R + r;
  if (p.tiles >= 8) {
    for (int t = w; t < p.tiles; t += 8) {
      const int row = t * 32 + r;
      lse[row] = lse_of(join_units(src + t * 32, R, 0, n, 1), qs[row]);
    }
    return;
  }
  const int groups = 8 / p.tiles, t = w % p.tiles, g = w / p.tiles;
  float2 a = make_float2(kNone, 0.f);
  if (g < groups) a = join_units(src + t * 32, R, g, n, groups);
  part[w >> 2][w & 3][r] = a;
  __syncthreads();
  if (g) return;
  for (int k = 1; k < groups; k++) {
    const int v = t + k * p.tiles;
    const float2 b = part[v >> 2][v & 3][r];
    join_stats(b.x, b.y, a.x, a.y);
  }
  lse[t * 32 + r] = lse_of(a, qs[t * 32 + r]);
}

// One pass of the keys over the rows.  SUM false: each row's maximum and sum
// over the unit's tokens; true: each token's sum of weights over the rows,
// added to (or, for the chunk's own tokens, set as) its weight.
//
// A workgroup's four waves hold 32 MT keys each as operands and walk the row
// tiles together: a tile's operands (PD * 128 bytes) come into LDS one ahead
// of their use, by direct-to-LDS copies that the four waves share.  The copies go
// out behind the products: in front of them, the compiler would wait for the
// copies before it reads the other buffer.
//
// Bound by the matrix products, three for one (hi hi, lo hi, hi lo), and the LDS
// reads that feed them.  A prompt of 32768 tokens, 256 rows, 8 kv heads of 128:
// 58 us for the statistics and 60 for the weights, 0.89 and 0.86 PFLOP/s of
// products issued (a large library product: 1.16).  A higher wave priority around
// the products, reads one to three steps ahead by hand and pages looked up a
// chunk ahead changed nothing.
template <int PD, int MT, bool SUM>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PD == 256 || MT == 2 ? 2 : 3)))
void window_kernel(WindowParams p) {
  // A score is a rounded product in both passes: one fused with what is subtracted
  // from it could pass the row's maximum by more than exp2 takes.
#pragma clang fp contract(off)
  constexpr int KS = PD / 16;
  constexpr int EBS = Rows<PD, 1>::EBS;
  constexpr int QT = PD * 128;  // bytes of a row tile's operands
  constexpr int TOK = 4 * 32 * MT;
  // (log2 of) the table's copies: what the LDS holds beside the rows' operands, so
  // that the table stays for all chunks.  16 copies in the operands' place, made
  // anew for each chunk: 150 us instead of 143 at 32768 tokens, 37.4 instead of
  // 29.2 for 3 chunks over 4000-16000 tokens at head size 64.
  constexpr int COPIES = PD == 64 ? 3 : (PD == 128 ? 2 : 1);
  typedef float float16_t __attribute__((ext_vector_type(16)));
  struct __attribute__((aligned(16))) Lds {
    uint64_t lut[256 << COPIES];
    uint8_t q[2][QT];
    float2 wave[2][4][32];        // a row tile's (max, sum) of each wave
    float2 rows[SUM ? 1 : 1024];  // running (max, sum) of the unit
    float lse[SUM ? 1024 : 1];    // the rows' normalisers
  };
  __shared__ Lds sm;
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.x / p.units, u = blockIdx.x % p.units;
  const PlanSlot ps = unit_of<TOK>(p, reinterpret_cast<int*>(sm.q), u, 1,
                                   !SUM && blockIdx.x == 0 && w == 0);
  if (ps.b < 0) return;
  const int q_len = p.q_start[ps.b + 1] - p.q_start[ps.b];
  if (SUM && q_len <= 0) return;  // no queries: the weights stay
  const int c0 = ps.j * ps.U, c1 = min(c0 + ps.U, ps.L);
  const int64_t bh = (int64_t)ps.b * p.Hkv + kvh;
  const uint8_t* const qf =
      reinterpret_cast<const uint8_t*>(p.qf) + bh * p.tiles * (int64_t)QT;
  const float* const qs = p.qs + bh * p.tiles * 32;
  if constexpr (SUM) row_lse(p, kvh, bh, u - ps.j, (ps.L + ps.U - 1) / ps.U, sm.wave, sm.lse);
  if constexpr (!SUM)
    for (int i = threadIdx.x; i < p.tiles * 32; i += 256) sm.rows[i] = make_float2(kNone, 0.f);
  const uint32_t lanec = 8 * (lane & ((1 << COPIES) - 1));
  init_key_table<COPIES>(sm.lut);
  __syncthreads();

  // copies of row tile rt into buffer rt & 1
  auto issue = [&](int rt) {
#if defined(__HIP_DEVICE_COMPILE__)
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(qf + (int64_t)rt * QT), (short)0, QT, 0x00020000);
#pragma unroll
    for (int j = 0; j < QT / 4096; j++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (void*)(sm.q[rt & 1] + (4 * j + w) * 1024), 16,
                                               (uint32_t)((4 * j + w) * 1024 + lane * 16), 0, 0, 0);
#else
    (void)rt;
#endif
  };

  for (int cb = c0; cb < c1; cb += TOK) {
    const int t0 = cb + w * 32 * MT;
    // the keys of tokens t0 + 32 m + col, as operands; their norms (fp16) by row
    // of the product's layout: row 8 * (i / 4) + 4 * half + i % 4
    half8_t kh[MT][KS], kl[MT][KS];
    uint32_t kn[MT][8];
    uint32_t okm[MT];
    int64_t place[MT];  // index of this lane's token in weights, -1: none
    float old[MT];      // and its weight
#pragma unroll
    for (int m = 0; m < MT; m++) {
      const int t = t0 + 32 * m + col;
      place[m] = -1;
      int64_t at = 0;
      if (t < c1) {
        const int64_t e = (int64_t)ps.ip + t / p.block_size;
        const int pg = e >= 0 && e < p.entries ? p.indices[e] : -1;
        if (pg >= 0 && pg < p.num_blocks) {
          const int in = t % p.block_size;
          place[m] = ((int64_t)pg * p.Hkv + kvh) * p.block_size + in;
          at = (((int64_t)pg * p.block_size + in) * p.Hkv + kvh) * EBS;
        }
      }
      okm[m] = (uint32_t)__ballot(place[m] >= 0);
      if constexpr (SUM) old[m] = p.weights[max(place[m], (int64_t)0)];
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.slab + at + half * (PD / 4));
      const uint32_t norm = *reinterpret_cast<const uint32_t*>(p.slab + at + PD / 2) & 0xffffu;
      uint32_t c[KS];
#pragma unroll
      for (int k = 0; k < KS; k += 4) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(src + k);
        c[k] = v[0]; c[k + 1] = v[1]; c[k + 2] = v[2]; c[k + 3] = v[3];
      }
#pragma unroll
      for (int k = 0; k < KS; k++) key_parts<COPIES>(c[k], sm.lut, lanec, kh[m][k], kl[m][k]);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int r = 8 * (i / 2) + 4 * half + 2 * (i % 2);
        kn[m][i] = (uint32_t)__shfl((int)norm, r) | (uint32_t)__shfl((int)norm, r + 1) << 16;
      }
    }
    float got[SUM ? MT : 1][16];
    if constexpr (SUM) {
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 16; i++) got[m][i] = 0.f;
    }
    bool all = t0 + 32 * MT <= c1;  // every token of the wave is there
#pragma unroll
    for (int m = 0; m < MT; m++) all = all && okm[m] == 0xffffffffu;
    __syncthreads();  // the last chunk's operands are no longer read
    // a row tile's scale, one tile ahead and in front of the copies
    float next_q = qs[col];
    issue(0);
    // the waves' statistics of tile rt, joined by one of them; tile rt + 1 has
    // buffers of its own, so the barrier of each tile is enough
    auto join_tile = [&](int rt) {
      if (w == (rt & 3) && half == 0) {
        float2 a = sm.rows[rt * 32 + col];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float2 b = sm.wave[rt & 1][k][col];
          join_stats(b.x, b.y, a.x, a.y);
        }
        sm.rows[rt * 32 + col] = a;
      }
    };

    for (int rt = 0; rt < p.tiles; rt++) {
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      barrier();  // tile rt is there, and nobody reads the other buffer
      const int row = rt * 32 + col;
      const float cq = next_q * p.csc, ls = SUM ? sm.lse[row] : 0.f;
      if (rt + 1 < p.tiles) {
        next_q = qs[row + 32];
      }
      if constexpr (!SUM)
        if (rt) join_tile(rt - 1);
      float16_t acc[MT];
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[m][i] = 0.f;
      const half8_t* const f = reinterpret_cast<const half8_t*>(sm.q[rt & 1]) + lane;
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const half8_t fh = f[k * 128], fl = f[k * 128 + 64];
#pragma unroll
        for (int m = 0; m < MT; m++) {
          acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[m][k], fh, acc[m], 0, 0, 0);
          acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl[m][k], fh, acc[m], 0, 0, 0);
          acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[m][k], fl, acc[m], 0, 0, 0);
        }
      }
#if defined(__HIP_DEVICE_COMPILE__)
      // reads ahead of the products (head size 256, two waves a SIMD: a call of 78 us
      // instead of 83, 16384 tokens, 64 queries of 16 q / 2 kv heads)
      __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
      for (int k = 0; k < KS - 3; k++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 9, 0);
#endif
      if (rt + 1 < p.tiles) issue(rt + 1);
      // Tokens that this row's query sees: the tile's first row sees least, and a row
      // that gives no weights nothing (its products may be no numbers, where a norm is
      // not finite; the first pass need not know, its statistics of such rows are not
      // used).  Bit c of
      // seen(m): the token of accumulator row c (+ 4 in the upper half) is there and
      // seen; made anew for each tile, as masks kept over the loop spill.
      const bool none = SUM && ls == INFINITY;
      const bool clear =
          all && t0 + 32 * MT - 1 <= ps.L - p.window + rt * 32 / p.ratio && !__any(none);
      auto seen = [&](int m) {
        uint32_t ok = okm[m];
#if defined(__HIP_DEVICE_COMPILE__)
        asm volatile("" : "+s"(ok));
#endif
        const int last = none ? -1 : ps.L - p.window + row / p.ratio - (t0 + 32 * m);
        return (ok & (last < 0 ? 0u : 0xffffffffu >> (31 - min(last, 31)))) >> (4 * half);
      };
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          acc[m][i] = by_half(acc[m][i], kn[m][i / 2]);
          acc[m][i + 1] = by_half(acc[m][i + 1], kn[m][i / 2] >> 16);
        }
      if constexpr (SUM) {
        if (!clear) {
#pragma unroll
          for (int m = 0; m < MT; m++) {
            const uint32_t bits = seen(m);
#pragma unroll
            for (int i = 0; i < 16; i++)
              acc[m][i] = bits & (1u << (8 * (i / 4) + i % 4)) ? acc[m][i] * cq - ls
                                                              : -INFINITY;
          }
        } else {
#pragma unroll
          for (int m = 0; m < MT; m++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[m][i] = acc[m][i] * cq - ls;
        }
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 16; i++) got[m][i] += exp2_raw(acc[m][i]);
      } else {
        float mx = kNone, l = 0.f;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 16; i++) acc[m][i] *= cq;
        if (!clear) {
#pragma unroll
          for (int m = 0; m < MT; m++) {
            const uint32_t bits = seen(m);
#pragma unroll
            for (int i = 0; i < 16; i++)
              acc[m][i] = bits & (1u << (8 * (i / 4) + i % 4)) ? acc[m][i] : -INFINITY;
          }
        }
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 16; i += 2) mx = vmax3(mx, acc[m][i], acc[m][i + 1]);
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 16; i++) l += exp2_raw(acc[m][i] - mx);
        join_stats(__shfl_xor(mx, 32), __shfl_xor(l, 32), mx, l);
        if (half == 0) sm.wave[rt & 1][w][col] = make_float2(mx, l);
        lds_written();
      }
    }
    if constexpr (!SUM) {
      barrier();
      join_tile(p.tiles - 1);
    }
    if constexpr (SUM) {
#pragma unroll
      for (int m = 0; m < MT; m++) {
        // Each step adds over one bit of the column and halves the values that a
        // lane holds: lane (col, half) ends with accumulator row col % 16's sum.
#pragma unroll
        for (int step = 0; step < 4; step++) {
          const bool bit = col >> step & 1;
#pragma unroll
          for (int i = 0; i < 8 >> step; i++) {
            const float keep = bit ? got[m][2 * i + 1] : got[m][2 * i];
            const float give = bit ? got[m][2 * i] : got[m][2 * i + 1];
            got[m][i] = keep + (step == 3 ? ror8(give) : xor_lane(give, 1 << step));
          }
        }
        // token col's row is 4 (col / 8) + col % 4 of half col / 4 % 2
        const float mine =
            __shfl(xor16_sum(got[m][0]), (col & 4) * 8 + (col >> 3) * 4 + (col & 3));
        if (half == 0 && place[m] >= 0) {
          const int t = t0 + 32 * m + col;
          if (t < ps.L - q_len) {
            p.weights[place[m]] = old[m] + mine;
          } else {
            p.weights[place[m]] = mine;
            if (p.positions) p.positions[place[m]] = p.ends[ps.b] - ps.L + t;
          }
        }
      }
    }
  }
  if constexpr (!SUM) {
    __syncthreads();
    float2* const out = p.stats + ((int64_t)kvh * p.units + u) * p.tiles * 32;
    for (int i = threadIdx.x; i < p.tiles * 32; i += 256) out[i] = sm.rows[i];
  }
}

// ---- host ------------------------------------------------------------------

// Kv heads of a workgroup: the largest of 8, 4, 2, 1 (at most 4 at head size
// 256) that divides their number and whose q' fit the 32 KB of the table.
int group_of(int pd, int hkv, int ratio) {
  int g = pd == 256 ? 4 : 8;
  while (hkv % g || g * ratio * pd * 4 > 32768) g >>= 1;
  return g;
}
size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

int check_track(const char* who, int batch, int64_t entries, int hq, int hkv, int pd, int bs) {
  if (pd != 64 && pd != 128 && pd != 256) {
    set_error("%s: padded_dim must be 64, 128 or 256, got %d", who, pd);
    return kEinval;
  }
  if (hkv <= 0 || hq <= 0 || hq % hkv != 0 || hq / hkv > 16) {
    set_error("%s: num_qo_heads %d / num_kv_heads %d must be an integer <= 16", who, hq, hkv);
    return kEinval;
  }
  if (hkv > 4096) {
    set_error("%s: num_kv_heads %d out of range", who, hkv);
    return kEinval;
  }
  if (bs <= 0 || bs % kTile != 0) {
    set_error("%s: block_size %d must be a positive multiple of 16", who, bs);
    return kEinval;
  }
  if (batch < 0 || batch > kPlanMost) {
    set_error("%s: batch %d out of range (0 .. %d)", who, batch, kPlanMost);
    return kEinval;
  }
  if (entries < 0 || entries > 0x7fffffffLL) {
    set_error("%s: %lld page-table entries out of range", who, (long long)entries);
    return kEinval;
  }
  return 0;
}

typedef void (*TrackFn)(TrackParams);
template <bool VALUES>
TrackFn track_fn(int pd, int g, bool qc) {
#define TQ_ONE(P, GG, Q) \
  (VALUES ? &track_values_kernel<P, GG, Q> : &track_scores_kernel<P, GG, Q>)
#define TQ_G(P, Q)                        \
  switch (g) {                            \
    case 8: return TQ_ONE(P, (P == 256 ? 4 : 8), Q); \
    case 4: return TQ_ONE(P, 4, Q);       \
    case 2: return TQ_ONE(P, 2, Q);       \
    default: return TQ_ONE(P, 1, Q);      \
  }
  if (pd == 64) {
    if (qc) { TQ_G(64, true) } else { TQ_G(64, false) }
  }
  if (pd == 128) {
    if (qc) { TQ_G(128, true) } else { TQ_G(128, false) }
  }
  if (qc) { TQ_G(256, true) } else { TQ_G(256, false) }
#undef TQ_G
#undef TQ_ONE
}

// Work units of a tracked decode: the workgroups that the scores kernel keeps
// resident, at least one per sequence; in pairs where that is two a CU.
struct TrackPlan {
  int units, pair, rows;
  int64_t blocks;
};
constexpr int kPairShare = 62;
TrackPlan track_plan(int batch, int pd, int g, int hg, bool qc) {
  const Occupancy occ =
      occupancy(reinterpret_cast<const void*>(track_fn<false>(pd, g, qc)), kThreads);
  TrackPlan t = {0, 0, 0, 0};
  if (occ.cus <= 0 || occ.per_cu <= 0) return t;
  t.units = max(batch, occ.cus * occ.per_cu / hg);
  t.rows = t.units;
  // Calls with pairs / with as many single units: 8 x 32768 tokens 93.9 / 95.3 us,
  // 32 x 8192 93.2 / 94.5, 32 x 16384 of 8 q / 1 kv heads 42.2 / 43.5, head size 256
  // 24 ragged sequences 60.1 / 63.0 and 8 x 32768 60.5 / 63.3; where a call is short
  // the uneven shares cost: 8 x 4096 36.4 / 34.9, 1 x 32768 51.3 / 49.9, at head size
  // 256 59.9 / 58.4.  Pairs in halves: 95.7, 95.0, 43.5, 62.4, 62.9, 35.1, 50.1, 58.5.
  // (Not at head size 64, where the shares finish together: 32.1 + 26.6 us
  // unpaired, 32.6 + 27.6 paired, 48 ragged sequences.)
  if (pd > 64 && occ.per_cu == 2 && occ.cus % hg == 0 && occ.cus / hg >= batch) {
    t.units = occ.cus / hg;
    t.pair = kPairShare;
    t.rows = 2 * t.units;
  }
  t.blocks = (int64_t)t.rows * hg;
  return t;
}

// A tracked decode's workspace, for scores of `pages` pages
struct TrackWs {
  size_t stats, split, s, po, total;
};
TrackWs track_ws(int batch, int64_t pages, int hq, int hkv, int pd, int bs, int parts) {
  const int ratio = hq / hkv;
  int rp = 1;
  while (rp < ratio) rp <<= 1;
  TrackWs w;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += up256(n);
    return r;
  };
  w.stats = take((size_t)hkv * parts * rp * 8);
  w.split = take((size_t)(batch + 2) * 4);
  // (a tile at least: tiles outside the table read the first one)
  w.s = take((size_t)max(pages, (int64_t)1) * bs * hq * 4);
  w.po = take((size_t)parts * hq * pd * 4);
  w.total = at;
  return w;
}

int launch(const char* who, const void* fn, int64_t blocks, int threads, void** args,
           tq_stream_t stream) {
  if (blocks > 0x7fffffffLL) {
    set_error("%s: grid too large", who);
    return kEinval;
  }
  hipError_t e = hipLaunchKernel(fn, dim3((unsigned)blocks), dim3(threads), args, 0,
                                 reinterpret_cast<hipStream_t>(stream));
  if (e == hipSuccess) e = hipGetLastError();
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", who, hipGetErrorString(e));
    return (int)e;
  }
  return 0;
}

int check_rows(const char* who, const void* q, int64_t sb, int64_t sh, int q_dtype, int hd,
               int pd) {
  if (hd <= 0 || hd > pd) {
    set_error("%s: head_dim %d out of range for padded_dim %d", who, hd, pd);
    return kEinval;
  }
  if (q_dtype != TQ_F16 && q_dtype != TQ_BF16) {
    set_error("%s: q must be fp16 or bf16", who);
    return kEinval;
  }
  (void)sb;
  if (!q || (uintptr_t)q % 2 || sh < 0) {
    set_error("%s: bad q", who);
    return kEinval;
  }
  return 0;
}

int check_state(const char* who, const uint8_t* k, const uint8_t* v, const int32_t* indices,
                const int32_t* indptr, const int32_t* seq_lens, int64_t entries, int ebs, int pd,
                int64_t num_blocks, int bs, int hkv, float* weights, int32_t* positions,
                const int32_t* ends) {
  const int want = pd == 64 ? 48 : (pd == 128 ? 80 : 144);
  if (ebs != want) {
    set_error("%s: ebs %d does not match padded_dim %d (expected %d)", who, ebs, pd, want);
    return kEinval;
  }
  if (num_blocks <= 0 || num_blocks > 0x7fffffffLL ||
      num_blocks * bs * (int64_t)hkv > 0x7fffffffLL * kTile ||
      num_blocks * (int64_t)bs > 0x7fffffffLL) {
    set_error("%s: %lld blocks of %d tokens, %d heads out of range", who, (long long)num_blocks,
              bs, hkv);
    return kEinval;
  }
  if (!k || !v || (!indices && entries) || !indptr || !seq_lens || !weights ||
      (positions && !ends)) {
    set_error("%s: null pointer", who);
    return kEinval;
  }
  if ((uintptr_t)k % 16 || (uintptr_t)v % 16 || (uintptr_t)weights % 16) {
    set_error("%s: cache slabs and weights must be 16-byte aligned", who);
    return kEinval;
  }
  return 0;
}

}  // namespace
}  // namespace tq

extern "C" int64_t tq_decode_tracked_workspace_bytes(int32_t batch, int64_t pages,
                                                     int32_t num_qo_heads, int32_t num_kv_heads,
                                                     int32_t padded_dim, int32_t block_size) {
  using namespace tq;
  const int rc = check_track("decode_tracked", batch, pages, num_qo_heads, num_kv_heads,
                             padded_dim, block_size);
  if (rc) return rc;
  if (batch == 0) return 0;
  const int ratio = num_qo_heads / num_kv_heads, g = group_of(padded_dim, num_kv_heads, ratio);
  const TrackPlan plan = track_plan(batch, padded_dim, g, num_kv_heads / g, ratio <= 8);
  if (plan.units <= 0) {
    set_error("decode_tracked: occupancy query failed");
    return kEinval;
  }
  return (int64_t)track_ws(batch, pages, num_qo_heads, num_kv_heads, padded_dim, block_size,
                           plan.rows)
      .total;
}

extern "C" int tq_decode_paged_tracked(
    const void* q, int64_t q_stride_b, int64_t q_stride_h, int32_t q_dtype, const uint8_t* k_slab,
    const uint8_t* v_slab, const int32_t* indices, int64_t num_indices, const int32_t* indptr,
    const int32_t* seq_lens, int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t padded_dim, int32_t block_size, int32_t ebs, int64_t num_blocks,
    float sm_scale, const float* signs, void* o, int32_t o_dtype, float* weights,
    int32_t* positions, const int32_t* ends, void* workspace, int64_t workspace_bytes,
    tq_stream_t stream) {
  using namespace tq;
  const char* who = "decode_tracked";
  int rc = check_track(who, batch, num_indices, num_qo_heads, num_kv_heads, padded_dim, block_size);
  if (rc || batch == 0) return rc;
  rc = check_rows(who, q, q_stride_b, q_stride_h, q_dtype, head_dim, padded_dim);
  if (rc) return rc;
  rc = check_state(who, k_slab, v_slab, indices, indptr, seq_lens, num_indices, ebs, padded_dim,
                   num_blocks, block_size, num_kv_heads, weights, positions, ends);
  if (rc) return rc;
  if (!o || (o_dtype != TQ_F16 && o_dtype != TQ_BF16)) {
    set_error("%s: o must be fp16 or bf16", who);
    return kEinval;
  }
  const int pd = padded_dim, ratio = num_qo_heads / num_kv_heads;
  const int g = group_of(pd, num_kv_heads, ratio);
  const bool qc = ratio <= 8;
  const TrackPlan plan = track_plan(batch, pd, g, num_kv_heads / g, qc);
  if (plan.units <= 0) {
    set_error("%s: occupancy query failed", who);
    return kEinval;
  }
  const TrackWs ws =
      track_ws(batch, min(num_indices, num_blocks), num_qo_heads, num_kv_heads, pd, block_size,
               plan.rows);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < (int64_t)ws.total) {
    set_error("%s: the workspace must be 16-byte aligned and hold %lld bytes, got %lld", who,
              (long long)ws.total, (long long)workspace_bytes);
    return kEinval;
  }
  uint8_t* const base = static_cast<uint8_t*>(workspace);
  TrackParams p = {};
  p.slab = k_slab;
  p.indices = indices;
  p.indptr = indptr;
  p.seq_lens = seq_lens;
  p.entries = num_indices;
  p.num_blocks = (int)num_blocks;
  p.B = batch;
  p.Hq = num_qo_heads;
  p.Hkv = num_kv_heads;
  p.ratio = ratio;
  p.rp = 1;
  while (p.rp < ratio) p.rp <<= 1;
  p.block_size = block_size;
  p.HG = num_kv_heads / g;
  p.units = plan.units;
  p.pair = plan.pair;
  p.rows = plan.rows;
  p.q = q;
  p.q_sb = q_stride_b;
  p.q_sh = q_stride_h;
  p.q_bf16 = q_dtype == TQ_BF16;
  p.hd = head_dim;
  p.signs = signs;
  const float isq = 1.0f / sqrtf((float)pd);
  p.csc = sm_scale * 1.4426950408889634f * isq / kLevelScale;
  p.osc = isq / kValueScale;
  p.s = reinterpret_cast<float*>(base + ws.s);
  p.by_page = num_indices > num_blocks;
  p.stats = reinterpret_cast<float2*>(base + ws.stats);
  p.split = reinterpret_cast<int32_t*>(base + ws.split);
  p.po = reinterpret_cast<float*>(base + ws.po);
  p.weights = weights;
  p.positions = positions;
  p.ends = ends;
  int hq = num_qo_heads, hd = head_dim;
  void* targs[] = {&p};
  rc = launch(who, reinterpret_cast<const void*>(track_fn<false>(pd, g, qc)),
              plan.blocks, kThreads, targs, stream);
  if (rc) return rc;
  p.slab = v_slab;
  rc = launch(who, reinterpret_cast<const void*>(track_fn<true>(pd, g, qc)),
              plan.blocks, kThreads, targs, stream);
  if (rc) return rc;
  {
    int ob = o_dtype == TQ_BF16;
    const float* po = p.po;
    const int32_t* split = p.split;
    void* args[] = {&po, &split, &hq, &hd, &ob, &signs, &o};
    const void* fn = pd == 64    ? reinterpret_cast<const void*>(&track_join_kernel<64>)
                     : pd == 128 ? reinterpret_cast<const void*>(&track_join_kernel<128>)
                                 : reinterpret_cast<const void*>(&track_join_kernel<256>);
    return launch(who, fn, (int64_t)batch * hq, 256, args, stream);
  }
}

namespace tq {
namespace {

struct WindowWs {
  size_t qf, qs, stats, lse, split, total;
  int tiles, units;
};
// units of a window call: three workgroups a CU over the kv heads, at least one
// per sequence (with 4 or 6 a CU 32768 tokens took 132.5 us as with 3, 4 prompts
// of up to 1500 34.2 and 38.5 for 29.4)
WindowWs window_ws(int batch, int window, int ratio, int hkv, int pd, int cus) {
  WindowWs w;
  w.tiles = (window * ratio + 31) / 32;
  w.units = max(batch, 3 * cus / hkv);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += up256(n);
    return r;
  };
  const size_t rows = (size_t)w.tiles * 32;
  w.qf = take((size_t)batch * hkv * rows * pd * 4);
  w.qs = take((size_t)batch * hkv * rows * 4);
  w.stats = take((size_t)hkv * w.units * rows * 8);
  w.lse = take((size_t)batch * hkv * rows * 4);
  w.split = take((size_t)(batch + 2) * 4);
  w.total = at;
  return w;
}
// Whether the second pass joins the units' statistics itself, in each workgroup
// again: where a thread would read at most 16 of them for a sequence of average
// length (its units x row tiles, over 8 half waves).  A launch less, measured with
// 12 reads (4 prompts of up to 1500 tokens, 128 rows) 30.4 -> 28.4 us and with 8
// (head size 64, 32 rows) 29.7 -> 28.8; with 86 (32768 tokens, 256 rows) it
// would be 130 -> 153.  Lengths are on the GPU, so a skewed batch is judged by its
// average too, and the threads of a long sequence's workgroups read more (units x
// row tiles / 8 at most): one prompt of 32768 tokens among 16, 64 queries, takes
// 148.8 us like this and 147.0 with the launch, one of 8192 among 4 39.1 and 38.2.
bool join_here(const WindowWs& w, int batch) {
  return (int64_t)w.units * w.tiles <= (int64_t)128 * batch;
}
int check_window(int window, int ratio) {
  if (window < 1 || window * (int64_t)ratio > 1024) {
    set_error("track_window: window %d x %d q heads per kv head out of range (1 .. 1024 rows)",
              window, ratio);
    return kEinval;
  }
  return 0;
}

}  // namespace
}  // namespace tq

extern "C" int64_t tq_track_window_workspace_bytes(int32_t batch, int32_t window,
                                                   int32_t num_qo_heads, int32_t num_kv_heads,
                                                   int32_t padded_dim) {
  using namespace tq;
  int rc = check_track("track_window", batch, 0, num_qo_heads, num_kv_heads, padded_dim, kTile);
  if (!rc) rc = check_window(window, num_qo_heads / num_kv_heads);
  if (rc) return rc;
  if (batch == 0) return 0;
  const int cus = device_cus();
  if (cus <= 0) {
    set_error("track_window: device query failed");
    return kEinval;
  }
  return (int64_t)window_ws(batch, window, num_qo_heads / num_kv_heads, num_kv_heads, padded_dim,
                            cus)
      .total;
}

extern "C" int tq_track_window(
    const void* q, int64_t num_rows, int64_t q_stride_tok, int64_t q_stride_h, int32_t q_dtype,
    const int32_t* query_start_loc, int32_t window, const uint8_t* k_slab, const int32_t* indices,
    int64_t num_indices, const int32_t* indptr, const int32_t* seq_lens, int32_t batch,
    int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, int32_t padded_dim,
    int32_t block_size, int32_t ebs, int64_t num_blocks, float sm_scale, const float* signs,
    float* weights, int32_t* positions, const int32_t* ends, void* workspace,
    int64_t workspace_bytes, tq_stream_t stream) {
  using namespace tq;
  const char* who = "track_window";
  int rc = check_track(who, batch, num_indices, num_qo_heads, num_kv_heads, padded_dim, block_size);
  if (!rc) rc = check_window(window, num_qo_heads / num_kv_heads);
  if (rc || batch == 0) return rc;
  rc = check_rows(who, q, q_stride_tok, q_stride_h, q_dtype, head_dim, padded_dim);
  if (rc) return rc;
  rc = check_state(who, k_slab, k_slab, indices, indptr, seq_lens, num_indices, ebs, padded_dim,
                   num_blocks, block_size, num_kv_heads, weights, positions, ends);
  if (rc) return rc;
  if (!query_start_loc || num_rows < 0) {
    set_error("%s: null pointer or negative row count", who);
    return kEinval;
  }
  const int cus = device_cus();
  if (cus <= 0) {
    set_error("%s: device query failed", who);
    return kEinval;
  }
  const int pd = padded_dim, ratio = num_qo_heads / num_kv_heads;
  const WindowWs ws = window_ws(batch, window, ratio, num_kv_heads, pd, cus);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < (int64_t)ws.total) {
    set_error("%s: the workspace must be 16-byte aligned and hold %lld bytes, got %lld", who,
              (long long)ws.total, (long long)workspace_bytes);
    return kEinval;
  }
  uint8_t* const base = static_cast<uint8_t*>(workspace);
  WindowParams p = {};
  p.slab = k_slab;
  p.indices = indices;
  p.indptr = indptr;
  p.seq_lens = seq_lens;
  p.q_start = query_start_loc;
  p.entries = num_indices;
  p.num_blocks = (int)num_blocks;
  p.B = batch;
  p.Hkv = num_kv_heads;
  p.ratio = ratio;
  p.block_size = block_size;
  p.units = ws.units;
  p.window = window;
  p.tiles = ws.tiles;
  p.qf = reinterpret_cast<half8_t*>(base + ws.qf);
  p.qs = reinterpret_cast<float*>(base + ws.qs);
  p.csc = sm_scale * 1.4426950408889634f / (sqrtf((float)pd) * kLevelScale);
  p.stats = reinterpret_cast<float2*>(base + ws.stats);
  p.lse = join_here(ws, batch) ? nullptr : reinterpret_cast<float*>(base + ws.lse);
  p.split = reinterpret_cast<int32_t*>(base + ws.split);
  p.weights = weights;
  p.positions = positions;
  p.ends = ends;
  const int64_t rows = (int64_t)batch * num_kv_heads * ws.tiles * 32;
  int bf = q_dtype == TQ_BF16, hd = head_dim;
  _Float16* qf = reinterpret_cast<_Float16*>(base + ws.qf);
  float* qs = reinterpret_cast<float*>(base + ws.qs);
  const void *fr, *f0, *f1;
  if (pd == 64) {
    fr = reinterpret_cast<const void*>(&rotate_window_kernel<64>);
    f0 = reinterpret_cast<const void*>(&window_kernel<64, 1, false>);
    f1 = reinterpret_cast<const void*>(&window_kernel<64, 1, true>);
  } else if (pd == 128) {
    fr = reinterpret_cast<const void*>(&rotate_window_kernel<128>);
    f0 = reinterpret_cast<const void*>(&window_kernel<128, 1, false>);
    f1 = reinterpret_cast<const void*>(&window_kernel<128, 1, true>);
  } else {
    fr = reinterpret_cast<const void*>(&rotate_window_kernel<256>);
    f0 = reinterpret_cast<const void*>(&window_kernel<256, 1, false>);
    f1 = reinterpret_cast<const void*>(&window_kernel<256, 1, true>);
  }
  void* rargs[] = {&q, &num_rows, &q_stride_tok, &q_stride_h, &bf, &hd, &p, &signs, &qf, &qs};
  rc = launch(who, fr, rows / 4, 256, rargs, stream);
  if (rc) return rc;
  void* args[] = {&p};
  // The first pass with two key tiles a wave, two workgroups a CU: half the LDS
  // reads a product.  At head size 128 and where the table has two chunks of 256
  // tokens a unit: 57.8 us instead of 64.8 at 32768 tokens, but 16.0 instead of
  // 11.7 for 4 prompts of up to 1500.  (The second pass spills with two; so do
  // both at head size 64.)
  const int wide = max(batch, 2 * cus / num_kv_heads);
  if (pd == 128 && p.lse && num_indices * block_size >= (int64_t)512 * wide) {
    p.units = wide;
    f0 = reinterpret_cast<const void*>(&window_kernel<128, 2, false>);
  }
  rc = launch(who, f0, (int64_t)p.units * num_kv_heads, 256, args, stream);
  if (rc) return rc;
  if (p.lse) {
    rc = launch(who, reinterpret_cast<const void*>(&window_lse_kernel), rows / 32, 256, args,
                stream);
    if (rc) return rc;
    p.units = ws.units;
  }
  return launch(who, f1, (int64_t)ws.units * num_kv_heads, 256, args, stream);
}
