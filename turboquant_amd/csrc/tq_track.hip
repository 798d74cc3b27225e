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
constexpr float kNone = -1e30f;  // maximum of no scores (finite: no inf - inf)
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
  const _Float16* qh;  // q' hi and lo parts [rows][PD], and 1 / their scale
  const _Float16* ql;
  const float* qs;
  float csc;  // score constant (log2 units)
  float osc;  // output constant
  float* s;   // scores, log2 units [table tile][Hkv][ratio][16]
  float2* stats;  // (max, sum) [Hkv][stat_rows][rp]
  int64_t stat_rows;
  int32_t* split;
  float* po;  // partial outputs [unit * SUB + sub][Hq][PD]
  float* weights;
  int32_t* positions;
  const int32_t* ends;
};

// The unit that workgroup `u` serves (plan_slot of tq_plan.h); st: at least
// 8 KB of LDS, free again afterwards.
__device__ __forceinline__ PlanSlot unit_of(const TrackParams& p, int* st, int u, bool writer) {
  const int lane = threadIdx.x & 63;
  if (p.B <= 64) {
    const bool in = lane < p.B;
    const int len = in ? max(p.seq_lens[lane], 0) : 0;
    const int ip = in ? p.indptr[lane] : 0;
    return plan_slot([&](int) { return len; }, [&](int) { return ip; }, p.B, 1, p.units, u, 1,
                     p.split, writer);
  }
  for (int i = threadIdx.x; i < kPlanMost; i += blockDim.x) {
    st[i] = i < p.B ? max(p.seq_lens[i], 0) : 0;
    st[kPlanMost + i] = i < p.B ? p.indptr[i] : 0;
  }
  __syncthreads();
  const PlanSlot r =
      plan_slot([&](int i) { return st[64 * i + lane]; },
                [&](int i) { return st[kPlanMost + 64 * i + lane]; }, p.B, (p.B + 63) >> 6,
                p.units, u, 1, p.split, writer);
  __syncthreads();
  return r;
}

// A unit's tiles: where each lies, and the copies of a step.  Lane i of a
// window holds what concerns tile 64 k + i: `at` its place in the cache in
// tiles (page * tiles per page + place in the page; -1 outside the unit, the
// table or the cache) and `wt` its place in the weights of kv head 0.  Two
// windows cover any three steps in a row, and tiles are looked up by readlane:
// a load here would make the compiler wait for the copies in flight.
template <int PD, int G>
struct Stream {
  using R = Rows<PD, G>;
  const TrackParams& p;
  int tile0, tiles;  // first tile of the sequence, tiles of the unit
  int ip, tpp;       // first table entry of the sequence, tiles per page
  int w;
  int base, at0, at1, wt0, wt1;  // windows base and base + 1
  uint32_t goff[R::NJ];  // source offsets of this lane's copies inside a tile

  __device__ __forceinline__ Stream(const TrackParams& pp, const PlanSlot& ps, int c0, int c1,
                                    int wave, int hg)
      : p(pp), tile0(c0 / kTile), tiles((c1 - c0 + kTile - 1) / kTile), ip(ps.ip),
        tpp(pp.block_size / kTile), w(wave), base(0) {
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
    wt = 0;
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
  // place of tile t in the cache (-1: none) and in the weights
  __device__ __forceinline__ int place(int t) const {
    return __builtin_amdgcn_readlane(t < 64 * (base + 1) ? at0 : at1, t & 63);
  }
  __device__ __forceinline__ int64_t weight_at(int t, int kvh) const {
    const int x = __builtin_amdgcn_readlane(t < 64 * (base + 1) ? wt0 : wt1, t & 63);
    return ((int64_t)x + (int64_t)kvh * tpp) * kTile;
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

// The key tables: code byte -> fp16 hi parts of its two levels (high nibble
// first, as the dims go), and their lo parts, times kLevelScale; 16 copies of
// each, lane l reads copy l mod 16.  Two tables of dwords: as pairs in one
// table, each operand register would cost a move.
__device__ __forceinline__ void init_key_table(uint32_t* hi, uint32_t* lo) {
  for (int e = threadIdx.x; e < 4096; e += blockDim.x) {
    const int byte = e >> 4;
    const float a = level(byte >> 4) * kLevelScale, b = level(byte & 15) * kLevelScale;
    const float ah = (float)(_Float16)a, bh = (float)(_Float16)b;
    hi[e] = pack_half(ah, bh);
    lo[e] = pack_half(a - ah, b - bh);
  }
}
// the operands of 8 codes
__device__ __forceinline__ void key_operands(uint32_t c, const uint32_t* hi, const uint32_t* lo,
                                             half8_t& kh, half8_t& kl) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int y = 0; y < 4; y++) {
    const uint32_t at = ((c >> (8 * y)) & 0xffu) << 4;
    h[y] = hi[at];
    l[y] = lo[at];
  }
  kh = __builtin_bit_cast(half8_t, u32x4{h[0], h[1], h[2], h[3]});
  kl = __builtin_bit_cast(half8_t, u32x4{l[0], l[1], l[2], l[3]});
}

// the codes of one tile and the norm of token 4 * (l/16) + l%4, from LDS: one
// block that ends with its own wait, as the compiler does not see these reads
template <int PD, int G>
__device__ __forceinline__ void read_key_tile(uint32_t row, uint32_t nrm, uint32_t* c,
                                              uint32_t& n) {
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

// ---- the keys: scores, and the splits' maxima and sums ----------------------
// MFMA 16x16x32: A = a tile's keys (row = token), B = q' (column = q head).
// QC (at most 8 q heads per kv head): columns 0-7 hold the hi parts of q',
// 8-15 the lo parts, so the products with the hi and the lo parts of the keys
// add up all four terms in one accumulator.
template <int PD, int G, bool QC>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4)))
void track_scores_kernel(TrackParams p) {
  using R = Rows<PD, G>;
  constexpr int KB = PD / 32;
  struct __attribute__((aligned(16))) Lds {
    uint32_t hi[4096], lo[4096];  // the key tables
    uint8_t ring[R::RING];
  };
  __shared__ Lds sm;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q4 = lane >> 4, n = lane & 15;
  const int hg = blockIdx.x % p.HG;
  const PlanSlot ps = unit_of(p, reinterpret_cast<int*>(sm.hi), blockIdx.x / p.HG,
                              blockIdx.x == 0 && w == 0);
  if (ps.b < 0) return;
  const int c0 = ps.j * ps.U, c1 = min(c0 + ps.U, ps.L);
  Stream<PD, G> st(p, ps, c0, c1, w, hg);
  const int steps = (st.tiles + R::TPS - 1) / R::TPS;

  const int kvh = hg * G + w % G, sub = w / G;
  const int head = QC ? n & 7 : n;
  half8_t qa[KB], qb[QC ? 1 : KB];
  float csc = 0.f;
  {
    const int64_t row = (int64_t)ps.b * p.Hq + kvh * p.ratio + min(head, p.ratio - 1);
    const bool real = head < p.ratio;
    const _Float16* src = (QC && n >= 8 ? p.ql : p.qh) + row * PD + (PD / 4) * q4;
#pragma unroll
    for (int k = 0; k < KB; k++) {
      const half8_t v = *reinterpret_cast<const half8_t*>(src + 8 * k);
      qa[k] = real ? v : half8_t{};
    }
    if constexpr (!QC) {
      const _Float16* lo = p.ql + row * PD + (PD / 4) * q4;
#pragma unroll
      for (int k = 0; k < KB; k++) {
        const half8_t v = *reinterpret_cast<const half8_t*>(lo + 8 * k);
        qb[k] = real ? v : half8_t{};
      }
    }
    csc = real ? p.csc * p.qs[row] : 0.f;
  }
  uint8_t* const spare = sm.ring + 2 * R::SLOT;
  st.issue(0, sm.ring, spare);
  st.issue(1, sm.ring + R::SLOT, spare);
  init_key_table(sm.hi, sm.lo);
  lds_written();
  // q' ends here, not at its first use inside the loop
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * R::NJ));

  const uint32_t ring = lds_addr(sm.ring);
  const uint32_t o_row = n * R::ROWB + w % G * R::EBS + q4 * (PD / 8);
  const uint32_t o_nrm = (4 * q4 + (lane & 3)) * R::ROWB + w % G * R::EBS + PD / 2;
  const uint32_t *const hi_t = sm.hi + n, *const lo_t = sm.lo + n;
  const int64_t tile_base = (int64_t)ps.ip * st.tpp + st.tile0;  // of the unit, in the table
  const int64_t max_tile = p.entries * st.tpp;
  float m = kNone, l = 0.f;
  float4_t sc[R::NTW];

  auto store = [&](int s) {  // the scores of step s
#pragma unroll
    for (int i = 0; i < R::NTW; i++) {
      const int t = s * R::TPS + sub + R::SUB * i;
      const int64_t gt = tile_base + t;
      if (t < st.tiles && gt >= 0 && gt < max_tile && n < p.ratio)
        *reinterpret_cast<float4_t*>(p.s + ((gt * p.Hkv + kvh) * p.ratio + n) * kTile + 4 * q4) =
            sc[i];
    }
  };

  for (int s = 0; s < steps; s++) {
    st.advance(s);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(R::NJ));
    barrier();  // the copies of step s have landed (and the table is there)
    uint32_t c[R::NTW][PD / 32], nr[R::NTW];
#pragma unroll
    for (int i = 0; i < R::NTW; i++) {
      const uint32_t at = ring + (s & 1) * R::SLOT + (sub + R::SUB * i) * R::TILEB;
      read_key_tile<PD, G>(at + o_row, at + o_nrm, c[i], nr[i]);
    }
    if (s) store(s - 1);
    barrier();  // every wave has read the slot
    st.issue(s + 2, sm.ring + (s & 1) * R::SLOT, spare);
#pragma unroll
    for (int i = 0; i < R::NTW; i++) {
      float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KB; k++) {
        half8_t hi, lo;
        key_operands(c[i][k], hi_t, lo_t, hi, lo);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, qa[k], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, qa[k], acc, 0, 0, 0);
        if constexpr (!QC) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, qb[k], acc, 0, 0, 0);
      }
      const int t = s * R::TPS + sub + R::SUB * i;
      const bool ok = st.place(t) >= 0;
      const int left = c1 - (st.tile0 + t) * kTile - 4 * q4;  // tokens of this lane's four
      const uint32_t nv[4] = {quad_bcast<0>(nr[i]), quad_bcast<1>(nr[i]), quad_bcast<2>(nr[i]),
                              quad_bcast<3>(nr[i])};
      float mx = m;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        float x = acc[r];
        if constexpr (QC) x += ror8(x);
        x = x * lo_half(nv[r]) * csc;
        sc[i][r] = ok && r < left ? x : -INFINITY;
        mx = fmaxf(mx, sc[i][r]);
      }
      l *= exp2f(m - mx);
      m = mx;
#pragma unroll
      for (int r = 0; r < 4; r++) l += exp2f(sc[i][r] - m);
    }
  }
  store(steps - 1);
  // no copy may land after the workgroup's LDS is given away
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  // a head's lanes n, n + 16, n + 32, n + 48 meet
  const float mx = fmaxf(fmaxf(m, __shfl_xor(m, 16)),
                         fmaxf(__shfl_xor(m, 32), __shfl_xor(m, 48)));
  l *= exp2f(m - mx);
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (lane < p.rp)
    p.stats[((int64_t)kvh * p.stat_rows + (int64_t)(ps.Pb + ps.j) * R::SUB + sub) * p.rp + lane] =
        lane < p.ratio ? make_float2(mx, l) : make_float2(kNone, 0.f);
}

// V codes of tokens 4 * (l/16) .. + 3 (PD / 32 bytes each) and one norm
template <int PD, int G>
__device__ __forceinline__ void read_value_tile(uint32_t row, uint32_t nrm, uint32_t (*c)[4],
                                                uint32_t& n) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int S = Rows<PD, G>::ROWB;
#define TQ_V4(OP)                                                                              \
  OP " %0, %5\n\t" OP " %1, %5 offset:%7\n\t" OP " %2, %5 offset:%8\n\t" OP " %3, %5 offset:%9\n\t" \
     "ds_read_u16 %4, %6\n\ts_waitcnt lgkmcnt(0)"
  if constexpr (PD == 64) {
    asm volatile(TQ_V4("ds_read_u16")
                 : "=&v"(c[0][0]), "=&v"(c[0][1]), "=&v"(c[0][2]), "=&v"(c[0][3]), "=&v"(n)
                 : "v"(row), "v"(nrm), "i"(S), "i"(2 * S), "i"(3 * S) : "memory");
  } else if constexpr (PD == 128) {
    asm volatile(TQ_V4("ds_read_b32")
                 : "=&v"(c[0][0]), "=&v"(c[0][1]), "=&v"(c[0][2]), "=&v"(c[0][3]), "=&v"(n)
                 : "v"(row), "v"(nrm), "i"(S), "i"(2 * S), "i"(3 * S) : "memory");
  } else {
    u32x2 a[4];
    asm volatile(TQ_V4("ds_read_b64")
                 : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(n)
                 : "v"(row), "v"(nrm), "i"(S), "i"(2 * S), "i"(3 * S) : "memory");
#pragma unroll
    for (int j = 0; j < 4; j++) {
      c[0][j] = a[j][0];
      c[1][j] = a[j][1];
    }
  }
#undef TQ_V4
#else
  (void)row; (void)nrm; (void)c; n = 0;
#endif
}

constexpr float kValueScale = 1.4809800386428833f;  // levels near fp16 grid points (8.7e-5)

// ---- the values: output partials and the weights ----------------------------
// MFMA 16x16x16: A = V^T (row = dim slot, k = tokens 4 * (l/16) ..), B = the
// probabilities, whose layout is that of the scores' tile.  Dim of (row r,
// product i) is r * (PD/16) + i.  QC: columns 0-7 hold the hi parts of
// p * norm, 8-15 the lo parts.
template <int PD, int G, bool QC>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(PD == 256 ? 2 : 4)))
void track_values_kernel(TrackParams p) {
  using R = Rows<PD, G>;
  constexpr int NO = PD / 16;           // products per tile
  constexpr int VW = PD == 256 ? 2 : 1;  // code dwords per token and lane
  struct __attribute__((aligned(16))) Lds {
    uint32_t lut[8192];  // code byte -> levels of its low and high nibble, 32 copies
    uint8_t ring[R::RING];
  };
  __shared__ Lds sm;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q4 = lane >> 4, n = lane & 15;
  const int hg = blockIdx.x % p.HG;
  const PlanSlot ps = unit_of(p, reinterpret_cast<int*>(sm.lut), blockIdx.x / p.HG, false);
  if (ps.b < 0) return;
  const int c0 = ps.j * ps.U, c1 = min(c0 + ps.U, ps.L);
  Stream<PD, G> st(p, ps, c0, c1, w, hg);
  const int steps = (st.tiles + R::TPS - 1) / R::TPS;
  uint8_t* const spare = sm.ring + 2 * R::SLOT;
  st.issue(0, sm.ring, spare);
  st.issue(1, sm.ring + R::SLOT, spare);
  const int kvh = hg * G + w % G, sub = w / G;
  const int head = QC ? n & 7 : n;

  // the maximum and the sum of this lane's head over the sequence
  float M = kNone, den = 0.f;
  {
    const int64_t rows = (int64_t)((ps.L + ps.U - 1) / ps.U) * R::SUB;
    const float2* src = p.stats + ((int64_t)kvh * p.stat_rows + (int64_t)ps.Pb * R::SUB) * p.rp;
    for (int64_t i = lane; i < rows * p.rp; i += 64) {
      const float2 x = src[i];
      const float mx = fmaxf(M, x.x);
      den = den * exp2f(M - mx) + x.y * exp2f(x.x - mx);
      M = mx;
    }
    for (int d = p.rp; d < 64; d <<= 1) {
      const float om = __shfl_xor(M, d), od = __shfl_xor(den, d);
      const float mx = fmaxf(M, om);
      den = den * exp2f(M - mx) + od * exp2f(om - mx);
      M = mx;
    }
  }
  const float inv = head < p.ratio && den != 0.f ? 1.0f / den : 0.f;
  {
    for (int e = threadIdx.x; e < 8192; e += kThreads) {
      const int byte = e >> 5;
      sm.lut[e] = pack_half(level(byte & 15) * kValueScale, level(byte >> 4) * kValueScale);
    }
    lds_written();
  }

  const uint32_t ring = lds_addr(sm.ring);
  const uint32_t o_row = 4 * q4 * R::ROWB + w % G * R::EBS + n * (PD / 32);
  const uint32_t o_nrm = (4 * q4 + (lane & 3)) * R::ROWB + w % G * R::EBS + PD / 2;
  const uint32_t* const lut = sm.lut + (lane & 31);
  const int64_t tile_base = (int64_t)ps.ip * st.tpp + st.tile0;
  float4_t O[NO];
#pragma unroll
  for (int i = 0; i < NO; i++) O[i] = float4_t{0.f, 0.f, 0.f, 0.f};

  // scores and weights of step s, loaded one step ahead of their use; tiles
  // outside the unit or the cache read an address inside the arrays and are
  // masked
  struct Ahead {
    float4_t sc[R::NTW], wt[R::NTW];
    int64_t at[R::NTW];  // of the weights, -1: none
  } nx, cu;
  auto load = [&](int s, Ahead& a) {
#pragma unroll
    for (int i = 0; i < R::NTW; i++) {
      const int t = s * R::TPS + sub + R::SUB * i;
      const bool ok = st.place(t) >= 0;
      const int64_t gt = ok ? tile_base + t : 0;
      a.at[i] = ok ? st.weight_at(t, kvh) : -1;
      a.sc[i] = *reinterpret_cast<const float4_t*>(
          p.s + ((gt * p.Hkv + kvh) * p.ratio + min(head, p.ratio - 1)) * kTile + 4 * q4);
      a.wt[i] = *reinterpret_cast<const float4_t*>(p.weights + max(a.at[i], (int64_t)0) + 4 * q4);
    }
  };
  auto store = [&](const Ahead& a) {  // the weights of a step
#pragma unroll
    for (int i = 0; i < R::NTW; i++)
      if (a.at[i] >= 0 && n == 0)
        *reinterpret_cast<float4_t*>(p.weights + a.at[i] + 4 * q4) = a.wt[i];
  };
  load(0, cu);

  for (int s = 0; s < steps; s++) {
    st.advance(s);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(R::NJ));
    barrier();
    uint32_t c[R::NTW][VW][4], nr[R::NTW];
#pragma unroll
    for (int i = 0; i < R::NTW; i++) {
      const uint32_t at = ring + (s & 1) * R::SLOT + (sub + R::SUB * i) * R::TILEB;
      read_value_tile<PD, G>(at + o_row, at + o_nrm, c[i], nr[i]);
    }
    if (s) {
      store(cu);
      cu = nx;
    }
    load(s + 1, nx);
    barrier();
    st.issue(s + 2, sm.ring + (s & 1) * R::SLOT, spare);
#pragma unroll
    for (int i = 0; i < R::NTW; i++) {
      const int t = s * R::TPS + sub + R::SUB * i;
      const int left = cu.at[i] >= 0 ? c1 - (st.tile0 + t) * kTile - 4 * q4 : 0;
      const int last = ps.L - 1 - (st.tile0 + t) * kTile - 4 * q4;
      const uint32_t nv[4] = {quad_bcast<0>(nr[i]), quad_bcast<1>(nr[i]), quad_bcast<2>(nr[i]),
                              quad_bcast<3>(nr[i])};
      float x[4];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float rel = r < left && head < p.ratio ? exp2f(cu.sc[i][r] - M) : 0.f;
        float g = rel * inv;  // this head's weight; summed over the group's heads
        g += xor_lane(g, 1);
        g += xor_lane(g, 2);
        g += xor_lane(g, 4);
        if constexpr (!QC) g += xor_lane(g, 8);
        if (r < left) cu.wt[i][r] = r == last ? g : cu.wt[i][r] + g;
        x[r] = r < left ? rel * lo_half(nv[r]) : 0.f;
        if constexpr (QC) {
          const float h = (float)(_Float16)x[r];
          x[r] = n < 8 ? h : x[r] - h;
        }
      }
      const half4_t pb = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
      // nibble pairs of tokens (0, 1) and (2, 3): byte k of ev / od indexes the
      // levels of dims 2k + 1 / 2k
#pragma unroll
      for (int v = 0; v < VW; v++) {
        const uint32_t m4 = 0x0f0f0f0fu;
        const uint32_t* cc = c[i][v];
        const uint32_t lo01 = (cc[0] & m4) | ((cc[1] & m4) << 4);
        const uint32_t hi01 = ((cc[0] >> 4) & m4) | (cc[1] & ~m4);
        const uint32_t lo23 = (cc[2] & m4) | ((cc[3] & m4) << 4);
        const uint32_t hi23 = ((cc[2] >> 4) & m4) | (cc[3] & ~m4);
        constexpr int BY = PD == 64 ? 2 : 4;
#pragma unroll
        for (int k = 0; k < BY; k++) {
          const uint32_t a0 = lut[((hi01 >> (8 * k)) & 0xffu) << 5];
          const uint32_t a1 = lut[((hi23 >> (8 * k)) & 0xffu) << 5];
          const uint32_t b0 = lut[((lo01 >> (8 * k)) & 0xffu) << 5];
          const uint32_t b1 = lut[((lo23 >> (8 * k)) & 0xffu) << 5];
          const int d = 8 * v + 2 * k;
          O[d] = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(half4_t, u32x2{a0, a1}),
                                                       pb, O[d], 0, 0, 0);
          O[d + 1] = __builtin_amdgcn_mfma_f32_16x16x16f16(
              __builtin_bit_cast(half4_t, u32x2{b0, b1}), pb, O[d + 1], 0, 0, 0);
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
  float* const row =
      p.po + (((int64_t)(ps.Pb + ps.j) * R::SUB + sub) * p.Hq + kvh * p.ratio + n) * PD;
  const float osc = inv * p.osc;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    float y[NO];
#pragma unroll
    for (int i = 0; i < NO; i++) {
      y[i] = O[i][r];
      if constexpr (QC) y[i] += ror8(y[i]);
      y[i] *= osc;
    }
    if (n < p.ratio)
#pragma unroll
      for (int i = 0; i < NO; i += 4)
        *reinterpret_cast<float4_t*>(row + (4 * q4 + r) * NO + i) =
            float4_t{y[i], y[i + 1], y[i + 2], y[i + 3]};
  }
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

// One row of hd elements (fp16 or bf16) rotated, scaled by a power of two to
// a maximum in [128, 256) and split: x * scale = hi + lo to 22 bits, lo parts
// of the large elements normal numbers.  Returns 1 / scale.
template <int PD>
__device__ __forceinline__ float split_row(const void* q, int64_t off, bool bf16, int hd,
                                           const float* signs, _Float16* hi, _Float16* lo) {
  constexpr int E = PD / 64;
  const int lane = threadIdx.x & 63;
  float x[E];
#pragma unroll
  for (int k = 0; k < E; k++) {
    const int d = lane * E + k;
    x[k] = 0.f;
    if (d < hd)
      x[k] = bf16 ? (float)static_cast<const __bf16*>(q)[off + d]
                  : (float)static_cast<const _Float16*>(q)[off + d];
    if (signs) x[k] *= signs[d];
  }
  if (signs) {
    fwht_wave<E>(x);
    const float isq = 1.0f / sqrtf((float)PD);
#pragma unroll
    for (int k = 0; k < E; k++) x[k] *= isq;
  }
  float mx = 0.f;
#pragma unroll
  for (int k = 0; k < E; k++) mx = fmaxf(mx, fabsf(x[k]));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, xor_lane(mx, d));
  int ex = 0;
  if (mx > 0.f && mx < INFINITY) ex = max(-100, min(100, 8 - (ilogbf(mx) + 1)));
  const float sc = ldexpf(1.0f, ex);
#pragma unroll
  for (int k = 0; k < E; k++) {
    const float v = x[k] * sc;
    hi[k] = (_Float16)v;
    lo[k] = (_Float16)(v - (float)hi[k]);
  }
  return ldexpf(1.0f, -ex);
}

template <int PD>
__global__ __launch_bounds__(256) void rotate_q_kernel(const void* __restrict__ q, int64_t q_sb,
                                                       int64_t q_sh, int bf16, int hd, int Hq,
                                                       int rows, const float* __restrict__ signs,
                                                       _Float16* __restrict__ qh,
                                                       _Float16* __restrict__ ql,
                                                       float* __restrict__ qs) {
  constexpr int E = PD / 64;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  _Float16 hi[E], lo[E];
  const float inv = split_row<PD>(q, row / Hq * q_sb + row % Hq * q_sh, bf16, hd, signs, hi, lo);
#pragma unroll
  for (int k = 0; k < E; k++) {
    qh[(int64_t)row * PD + lane * E + k] = hi[k];
    ql[(int64_t)row * PD + lane * E + k] = lo[k];
  }
  if (lane == 0) qs[row] = inv;
}

// o = s FWHT(sum of the partial rows)/sqrt(pd): one workgroup per (sequence,
// q head), its four waves sharing the partial rows
template <int PD>
__global__ __launch_bounds__(256) void track_join_kernel(const float* __restrict__ po,
                                                         const int32_t* __restrict__ split,
                                                         int sub, int Hq, int hd, int bf16,
                                                         const float* __restrict__ signs,
                                                         void* __restrict__ o) {
  constexpr int E = PD / 64;
  __shared__ float part[3][PD];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int b = blockIdx.x / Hq, h = blockIdx.x % Hq;
  const int r0 = split[b] * sub, r1 = split[b + 1] * sub;
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
  float2* stats;  // [Hkv][units][32 tiles]
  float* lse;     // [B][Hkv][32 tiles], log2 units, +inf: adds nothing
  int32_t* split;
  float* weights;
  int32_t* positions;
  const int32_t* ends;
};

template <int PD>
__global__ __launch_bounds__(256) void rotate_window_kernel(
    const void* __restrict__ q, int64_t q_rows, int64_t q_sb, int64_t q_sh, int bf16, int hd,
    WindowParams p, const float* __restrict__ signs, _Float16* __restrict__ qf, float* __restrict__ qs) {
  constexpr int E = PD / 64;
  const int64_t rows = (int64_t)p.B * p.Hkv * p.tiles * 32;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= rows) return;
  const int rho = (int)(row % (p.tiles * 32));
  const int64_t bh = row / (p.tiles * 32);
  const int kvh = (int)(bh % p.Hkv), b = (int)(bh / p.Hkv);
  const int i = rho / p.ratio, h = rho % p.ratio;
  const int q0 = p.q_start[b], q1 = p.q_start[b + 1];
  const int64_t at = (int64_t)q1 - p.window + i;
  _Float16 hi[E] = {}, lo[E] = {};
  float inv = 0.f;
  if (i < p.window && at >= max(q0, 0) && at < q_rows)
    inv = split_row<PD>(q, at * q_sb + (int64_t)(kvh * p.ratio + h) * q_sh, bf16, hd, signs, hi,
                        lo);
  // dim d is element d % 8 of half (d / 8) % ... : lane half d / (PD/2), step
  // (d % (PD/2)) / 8
  _Float16* const tile = qf + (bh * p.tiles + rho / 32) * (int64_t)(PD / 16) * 2 * 512;
#pragma unroll
  for (int k = 0; k < E; k++) {
    const int d = lane * E + k, half = d / (PD / 2), ks = d % (PD / 2) / 8;
    _Float16* const to = tile + ks * 1024 + (half * 32 + rho % 32) * 8 + d % 8;
    to[0] = hi[k];
    to[512] = lo[k];
  }
  if (lane == 0) qs[row] = inv;
}

// One pass of the keys over the rows.  SUM false: each row's maximum and sum
// over the unit's tokens; true: each token's sum of weights over the rows,
// added to (or, for the chunk's own tokens, set as) its weight.
template <int PD, int MT, bool SUM>
__global__ __launch_bounds__(256) void window_kernel(WindowParams p) {
  constexpr int KS = PD / 16;
  constexpr int EBS = Rows<PD, 1>::EBS;
  struct __attribute__((aligned(16))) Lds {
    uint32_t hi[4096], lo[4096];
    float2 st[SUM ? 1 : 4][SUM ? 1 : 1024];  // per wave: a row's running (max, sum)
  };
  __shared__ Lds sm;
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.x / p.units, u = blockIdx.x % p.units;
  TrackParams tp = {};
  tp.B = p.B;
  tp.units = p.units;
  tp.seq_lens = p.seq_lens;
  tp.indptr = p.indptr;
  tp.split = p.split;
  const PlanSlot ps = unit_of(tp, reinterpret_cast<int*>(sm.hi), u,
                              !SUM && blockIdx.x == 0 && w == 0);
  if (ps.b < 0) return;
  const int q_len = p.q_start[ps.b + 1] - p.q_start[ps.b];
  if (SUM && q_len <= 0) return;  // no queries: the weights stay
  init_key_table(sm.hi, sm.lo);
  const int c0 = ps.j * ps.U, c1 = min(c0 + ps.U, ps.L);
  const int64_t bh = (int64_t)ps.b * p.Hkv + kvh;
  const half8_t* const qf = p.qf + bh * p.tiles * KS * 2 * 64;
  const float* const qs = p.qs + bh * p.tiles * 32;
  const float* const lse = SUM ? p.lse + bh * p.tiles * 32 : nullptr;
  if constexpr (!SUM)
    for (int i = lane; i < p.tiles * 32; i += 64) sm.st[w][i] = make_float2(kNone, 0.f);
  __syncthreads();
  const uint32_t *const hi_t = sm.hi + (lane & 15), *const lo_t = sm.lo + (lane & 15);

  for (int t0 = c0 + w * 32 * MT; t0 < c1; t0 += 4 * 32 * MT) {
    // the keys of tokens t0 + 32 m + col, as operands; their norms by row of
    // the product's layout (row 8 * (i / 4) + 4 * half + i % 4)
    half8_t kh[MT][KS], kl[MT][KS];
    float kn[MT][16];
    uint32_t okm[MT];
    int64_t place[MT];  // index of this lane's token in weights, -1: none
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
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.slab + at + half * (PD / 4));
      const float norm = lo_half(*reinterpret_cast<const uint32_t*>(p.slab + at + PD / 2));
      uint32_t c[KS];
#pragma unroll
      for (int k = 0; k < KS; k += 4) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(src + k);
        c[k] = v[0]; c[k + 1] = v[1]; c[k + 2] = v[2]; c[k + 3] = v[3];
      }
#pragma unroll
      for (int k = 0; k < KS; k++) key_operands(c[k], hi_t, lo_t, kh[m][k], kl[m][k]);
#pragma unroll
      for (int i = 0; i < 16; i++) kn[m][i] = __shfl(norm, 8 * (i / 4) + 4 * half + i % 4);
    }
    float got[MT][16];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int i = 0; i < 16; i++) got[m][i] = 0.f;

    for (int rt = 0; rt < p.tiles; rt++) {
      typedef float float16_t __attribute__((ext_vector_type(16)));
      float16_t acc[MT];
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[m][i] = 0.f;
      const half8_t* f = qf + (int64_t)rt * KS * 2 * 64 + lane;
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const half8_t bh8 = f[k * 128], bl8 = f[k * 128 + 64];
#pragma unroll
        for (int m = 0; m < MT; m++) {
          acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[m][k], bh8, acc[m], 0, 0, 0);
          acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl[m][k], bh8, acc[m], 0, 0, 0);
          acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[m][k], bl8, acc[m], 0, 0, 0);
        }
      }
      const int row = rt * 32 + col;
      const float cq = qs[row] * p.csc;
      // the last token that this row's query sees
      const int see = ps.L - p.window + row / p.ratio;
      if constexpr (SUM) {
        const float ls = lse[row];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int tr = 8 * (i / 4) + 4 * half + i % 4;
            const float x = exp2f(acc[m][i] * kn[m][i] * cq - ls);
            got[m][i] += t0 + 32 * m + tr <= see ? x : 0.f;
          }
      } else {
        float mx = kNone, l = 0.f;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int tr = 8 * (i / 4) + 4 * half + i % 4;
            const bool ok = ((okm[m] >> tr) & 1) && t0 + 32 * m + tr <= see;
            acc[m][i] = ok ? acc[m][i] * kn[m][i] * cq : -INFINITY;
            mx = fmaxf(mx, acc[m][i]);
          }
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 16; i++) l += exp2f(acc[m][i] - mx);
        const float om = __shfl_xor(mx, 32), ol = __shfl_xor(l, 32);
        const float2 old = sm.st[w][row];
        const float top = fmaxf(fmaxf(mx, om), old.x);
        l = l * exp2f(mx - top) + ol * exp2f(om - top) + old.y * exp2f(old.x - top);
        if (half == 0) sm.st[w][row] = make_float2(top, l);
      }
    }
    if constexpr (SUM) {
#pragma unroll
      for (int m = 0; m < MT; m++) {
        float mine = 0.f;  // the sum of this lane's token, in lanes 0 .. 31
#pragma unroll
        for (int i = 0; i < 16; i++) {
          float g = got[m][i];
          g += xor_lane(g, 1);
          g += xor_lane(g, 2);
          g += xor_lane(g, 4);
          g += xor_lane(g, 8);
          g += __shfl_xor(g, 16);
          const float other = __shfl_xor(g, 32);
          const int r0 = 8 * (i / 4) + i % 4;  // half 0's row; half 1's is 4 further
          if (col == r0) mine = half ? other : g;
          if (col == r0 + 4) mine = half ? g : other;
        }
        if (half == 0 && place[m] >= 0) {
          const int t = t0 + 32 * m + col;
          if (t < ps.L - q_len) {
            p.weights[place[m]] += mine;
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
    for (int i = threadIdx.x; i < p.tiles * 32; i += 256) {
      float2 a = sm.st[0][i];
#pragma unroll
      for (int k = 1; k < 4; k++) {
        const float2 b = sm.st[k][i];
        const float top = fmaxf(a.x, b.x);
        a = make_float2(top, a.y * exp2f(a.x - top) + b.y * exp2f(b.x - top));
      }
      out[i] = a;
    }
  }
}

// the normalisers of a sequence's rows from its units' maxima and sums
__global__ __launch_bounds__(256) void window_lse_kernel(WindowParams p) {
  const int R = p.tiles * 32;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)p.B * p.Hkv * R) return;
  const int row = (int)(at % R);
  const int64_t bh = at / R;
  const int kvh = (int)(bh % p.Hkv), b = (int)(bh / p.Hkv);
  float m = kNone, l = 0.f;
#pragma unroll 4
  for (int u = p.split[b]; u < p.split[b + 1]; u++) {
    const float2 x = p.stats[((int64_t)kvh * p.units + u) * R + row];
    const float top = fmaxf(m, x.x);
    l = l * exp2f(m - top) + x.y * exp2f(x.x - top);
    m = top;
  }
  // rows past the window or before the chunk's first query add nothing
  p.lse[at] = p.qs[at] != 0.f && l != 0.f ? m + log2f(l) : INFINITY;
}

// ---- host ------------------------------------------------------------------

int group_of(int pd, int hkv) {
  int g = pd == 256 ? 4 : 8;
  while (hkv % g) g >>= 1;
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

// work units of a tracked decode: the workgroups that the scores kernel keeps
// resident, at least one per sequence
int track_units(int batch, int pd, int g, int hg, bool qc) {
  const Occupancy occ =
      occupancy(reinterpret_cast<const void*>(track_fn<false>(pd, g, qc)), kThreads);
  if (occ.cus <= 0 || occ.per_cu <= 0) return 0;
  return max(batch, occ.cus * occ.per_cu / hg);
}

// A tracked decode's workspace
struct TrackWs {
  size_t qh, ql, qs, stats, split, s, po, total;
};
TrackWs track_ws(int batch, int64_t entries, int hq, int hkv, int pd, int bs, int units, int sub) {
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
  const size_t rows = (size_t)batch * hq;
  w.qh = take(rows * pd * 2);
  w.ql = take(rows * pd * 2);
  w.qs = take(rows * 4);
  w.stats = take((size_t)hkv * units * sub * rp * 8);
  w.split = take((size_t)(batch + 2) * 4);
  // (a tile at least: tiles outside the table read the first one)
  w.s = take((size_t)max(entries, (int64_t)1) * bs * hq * 4);
  w.po = take((size_t)units * sub * hq * pd * 4);
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
  if (!k || !v || (!indices && entries) || !indptr || !seq_lens || !weights || (positions && !ends)) {
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

extern "C" int64_t tq_decode_tracked_workspace_bytes(int32_t batch, int64_t num_indices,
                                                     int32_t num_qo_heads, int32_t num_kv_heads,
                                                     int32_t padded_dim, int32_t block_size) {
  using namespace tq;
  const int rc = check_track("decode_tracked", batch, num_indices, num_qo_heads, num_kv_heads,
                             padded_dim, block_size);
  if (rc) return rc;
  if (batch == 0) return 0;
  const int g = group_of(padded_dim, num_kv_heads);
  const int units =
      track_units(batch, padded_dim, g, num_kv_heads / g, num_qo_heads / num_kv_heads <= 8);
  if (units <= 0) {
    set_error("decode_tracked: occupancy query failed");
    return kEinval;
  }
  return (int64_t)track_ws(batch, num_indices, num_qo_heads, num_kv_heads, padded_dim, block_size,
                           units, kWaves / g)
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
  rc = check_state(who, k_slab, v_slab, indices, indptr, seq_lens, num_indices, ebs, padded_dim, num_blocks,
                   block_size, num_kv_heads, weights, positions, ends);
  if (rc) return rc;
  if (!o || (o_dtype != TQ_F16 && o_dtype != TQ_BF16)) {
    set_error("%s: o must be fp16 or bf16", who);
    return kEinval;
  }
  const int pd = padded_dim, g = group_of(pd, num_kv_heads), sub = kWaves / g;
  const int ratio = num_qo_heads / num_kv_heads;
  const bool qc = ratio <= 8;
  const int units = track_units(batch, pd, g, num_kv_heads / g, qc);
  if (units <= 0) {
    set_error("%s: occupancy query failed", who);
    return kEinval;
  }
  const TrackWs ws =
      track_ws(batch, num_indices, num_qo_heads, num_kv_heads, pd, block_size, units, sub);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < (int64_t)ws.total) {
    set_error("%s: the workspace must be 16-byte aligned and hold %lld bytes, got %lld", who,
              (long long)ws.total, (long long)workspace_bytes);
    return kEinval;
  }
  uint8_t* const base = static_cast<uint8_t*>(workspace);
  _Float16* qh = reinterpret_cast<_Float16*>(base + ws.qh);
  _Float16* ql = reinterpret_cast<_Float16*>(base + ws.ql);
  float* qs = reinterpret_cast<float*>(base + ws.qs);
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
  p.units = units;
  p.qh = qh;
  p.ql = ql;
  p.qs = qs;
  const float isq = 1.0f / sqrtf((float)pd);
  p.csc = sm_scale * 1.4426950408889634f * isq / kLevelScale;
  p.osc = isq / kValueScale;
  p.s = reinterpret_cast<float*>(base + ws.s);
  p.stats = reinterpret_cast<float2*>(base + ws.stats);
  p.stat_rows = (int64_t)units * sub;
  p.split = reinterpret_cast<int32_t*>(base + ws.split);
  p.po = reinterpret_cast<float*>(base + ws.po);
  p.weights = weights;
  p.positions = positions;
  p.ends = ends;
  const int rows = batch * num_qo_heads;
  int bf = q_dtype == TQ_BF16, hq = num_qo_heads, hd = head_dim;
  {
    void* args[] = {&q, &q_stride_b, &q_stride_h, &bf, &hd, &hq, (void*)&rows, &signs, &qh, &ql,
                    &qs};
    const void* fn = pd == 64    ? reinterpret_cast<const void*>(&rotate_q_kernel<64>)
                     : pd == 128 ? reinterpret_cast<const void*>(&rotate_q_kernel<128>)
                                 : reinterpret_cast<const void*>(&rotate_q_kernel<256>);
    rc = launch(who, fn, (rows + 3) / 4, 256, args, stream);
    if (rc) return rc;
  }
  void* targs[] = {&p};
  rc = launch(who, reinterpret_cast<const void*>(track_fn<false>(pd, g, qc)),
              (int64_t)units * p.HG, kThreads, targs, stream);
  if (rc) return rc;
  p.slab = v_slab;
  rc = launch(who, reinterpret_cast<const void*>(track_fn<true>(pd, g, qc)),
              (int64_t)units * p.HG, kThreads, targs, stream);
  if (rc) return rc;
  {
    int ob = o_dtype == TQ_BF16, sb = sub;
    const float* po = p.po;
    const int32_t* split = p.split;
    void* args[] = {&po, &split, &sb, &hq, &hd, &ob, &signs, &o};
    const void* fn = pd == 64    ? reinterpret_cast<const void*>(&track_join_kernel<64>)
                     : pd == 128 ? reinterpret_cast<const void*>(&track_join_kernel<128>)
                                 : reinterpret_cast<const void*>(&track_join_kernel<256>);
    return launch(who, fn, rows, 256, args, stream);
  }
}

namespace tq {
namespace {

struct WindowWs {
  size_t qf, qs, stats, lse, split, total;
  int tiles, units;
};
// units of a window call: what the first pass keeps resident per kv head, at
// least one per sequence
WindowWs window_ws(int batch, int window, int ratio, int hkv, int pd, int cus) {
  WindowWs w;
  w.tiles = (window * ratio + 31) / 32;
  w.units = max(batch, 4 * cus / hkv);
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

extern "C" int tq_track_window(const void* q, int64_t num_rows, int64_t q_stride_tok, int64_t q_stride_h,
                               int32_t q_dtype, const int32_t* query_start_loc, int32_t window,
                               const uint8_t* k_slab, const int32_t* indices, int64_t num_indices,
                               const int32_t* indptr, const int32_t* seq_lens, int32_t batch,
                               int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                               int32_t padded_dim, int32_t block_size, int32_t ebs,
                               int64_t num_blocks, float sm_scale, const float* signs,
                               float* weights, int32_t* positions, const int32_t* ends,
                               void* workspace, int64_t workspace_bytes, tq_stream_t stream) {
  using namespace tq;
  const char* who = "track_window";
  int rc = check_track(who, batch, num_indices, num_qo_heads, num_kv_heads, padded_dim, block_size);
  if (!rc) rc = check_window(window, num_qo_heads / num_kv_heads);
  if (rc || batch == 0) return rc;
  rc = check_rows(who, q, q_stride_tok, q_stride_h, q_dtype, head_dim, padded_dim);
  if (rc) return rc;
  rc = check_state(who, k_slab, k_slab, indices, indptr, seq_lens, num_indices, ebs, padded_dim, num_blocks,
                   block_size, num_kv_heads, weights, positions, ends);
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
  p.lse = reinterpret_cast<float*>(base + ws.lse);
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
    f0 = reinterpret_cast<const void*>(&window_kernel<64, 2, false>);
    f1 = reinterpret_cast<const void*>(&window_kernel<64, 2, true>);
  } else if (pd == 128) {
    fr = reinterpret_cast<const void*>(&rotate_window_kernel<128>);
    f0 = reinterpret_cast<const void*>(&window_kernel<128, 2, false>);
    f1 = reinterpret_cast<const void*>(&window_kernel<128, 2, true>);
  } else {
    fr = reinterpret_cast<const void*>(&rotate_window_kernel<256>);
    f0 = reinterpret_cast<const void*>(&window_kernel<256, 1, false>);
    f1 = reinterpret_cast<const void*>(&window_kernel<256, 1, true>);
  }
  void* rargs[] = {&q, &num_rows, &q_stride_tok, &q_stride_h, &bf, &hd, &p, &signs, &qf, &qs};
  rc = launch(who, fr, (rows + 3) / 4, 256, rargs, stream);
  if (rc) return rc;
  void* args[] = {&p};
  rc = launch(who, f0, (int64_t)ws.units * num_kv_heads, 256, args, stream);
  if (rc) return rc;
  rc = launch(who, reinterpret_cast<const void*>(&window_lse_kernel), (rows + 255) / 256, 256,
              args, stream);
  if (rc) return rc;
  return launch(who, f1, (int64_t)ws.units * num_kv_heads, 256, args, stream);
}
