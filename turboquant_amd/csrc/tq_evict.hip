// tq_evict.hip -- eviction from the paged cache by accumulated weight.
//
// Per (sequence, kv head) with n > budget entries the `budget` entries with
// the largest key are kept: protected ones first (position < sink or >= end -
// recent), then by weight, equal ones by the lowest index.  Attention does not
// care where an entry stands (keys carry their rotary position), so kept
// entries in front of the budget stay, and the i-th kept entry behind it moves
// to the i-th place in front that is not kept: at most min(budget, n - budget)
// entries move, sources and destinations never meet, and a sequence that is a
// few tokens over its budget costs a few moves, where closing ranks would
// rewrite the whole cache.
//
// select_kernel: one workgroup per (sequence, kv head) reads weights and
// positions once into keys (32 bits that order like the rule above), which stay
// in LDS up to 32768 tokens, finds the budget-th largest by three radix passes
// (12 + 10 + 10 bits) and lists sources and destinations in index order by
// ballots.  move_kernel copies the listed entries, all sequences at once.
#include "tq_common.h"

namespace tq {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kQuads = 8;  // quads of tokens of a thread and chunk
constexpr int kChunk = 4 * kQuads * kSelThreads;  // tokens whose keys LDS holds
// 12 bits first: weights crowd into a few binades, and bins of 1/8 binade keep
// the lanes of a wave from meeting in one LDS counter
constexpr int kBins = 4096;
constexpr uint32_t kList = kBins - 1024;  // keys of one such bin kept aside

struct EvictParams {
  const int32_t* indices;
  const int32_t* indptr;
  const int32_t* seq_lens;
  const int32_t* ends;
  int64_t entries;
  int num_blocks, B, Hkv, block_size, shift;  // shift: log2 block_size or -1
  int budget, recent, sink;
  int64_t cap;  // moves per (sequence, head) at most
  int64_t half;  // lists by table place: their length per head; 0: a row's own lists
  float* weights;
  int32_t* positions;
  uint32_t* keys;  // [Hkv][entries * block_size], for sequences longer than kChunk
  // entry slots (page * block_size + place, -1: none), [B * Hkv][cap] or
  // [Hkv][half], see lists_of
  int32_t* dst;
  int32_t* src;
  int32_t* moves;  // [B * Hkv]
  uint8_t* ks;
  uint8_t* vs;
  int32_t* new_lens;
};

// slot of token i of a sequence whose table starts at ip, -1 outside the cache
__device__ __forceinline__ int slot_of(const EvictParams& p, int ip, int i) {
  const int pi = p.shift >= 0 ? i >> p.shift : i / p.block_size;
  const int64_t e = (int64_t)ip + pi;
  if (e < 0 || e >= p.entries) return -1;
  const int pg = p.indices[e];
  return pg >= 0 && pg < p.num_blocks ? pg * p.block_size + (i - pi * p.block_size) : -1;
}
// index of (slot, head) in weights and positions
__device__ __forceinline__ int64_t state_at(const EvictParams& p, int slot, int h) {
  const int pg = p.shift >= 0 ? slot >> p.shift : slot / p.block_size;
  return ((int64_t)pg * p.Hkv + h) * p.block_size + (slot - pg * p.block_size);
}

// Where a (sequence, head)'s lists start, and the moves that they have room for.
// n tokens make at most n / 2 moves, so by table place the lists of a sequence
// whose table starts at ip take half of what its tokens would.
struct Lists {
  int64_t at, room;
};
__device__ __forceinline__ Lists lists_of(const EvictParams& p, int bh, int h, int ip) {
  if (!p.half) return {bh * p.cap, p.cap};
  const int64_t first = (int64_t)ip * p.block_size / 2;
  return {h * p.half + first, p.half - first};
}

// Larger key, kept sooner: 0 no entry (set elsewhere), 1 NaN, then the weights
// in order (-0 as 0: kZero), all ones: protected, at a position outside [sink,
// sink + span).
constexpr uint32_t kZero = 0x80000000u, kHeld = 0xffffffffu;
__device__ __forceinline__ uint32_t key_of(float w, int pos, int sink, uint32_t span) {
  const uint32_t u = __float_as_uint(w + 0.f);  // (-0 + 0 = 0)
  const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return (uint32_t)pos - (uint32_t)sink >= span ? kHeld : (w != w ? 1u : k);
}

// inclusive sums over the 64 lanes, by DPP: shifts inside rows of 16, then the
// rows' totals
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
#define TQ_STEP(CTRL, ROWS) \
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false)
  TQ_STEP(0x111, 0xf);  // row_shr:1, 2, 4, 8
  TQ_STEP(0x112, 0xf);
  TQ_STEP(0x114, 0xf);
  TQ_STEP(0x118, 0xf);
  TQ_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
  TQ_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef TQ_STEP
  return v;
}

// base + the lanes before this one in mask
__device__ __forceinline__ uint32_t lanes_below(uint64_t mask, uint32_t base) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, base));
}

// Bound by the latencies of one workgroup's phases: 35 us at 32768 tokens (tile
// slots 2, loads with the first counts 11, the bin's list 4, other passes 1,
// ranks 3, source and destination lists 6.5) and 12 at 2050, on one CU a row.
// Loops over a chunk's quads stay loops: unrolled, with the keys in registers, the
// kernel was 42 KB of code, and fetching it cost a small call more than its work;
// eight quads in flight instead of four cost 1.7 and 1.2 us.
__global__ __launch_bounds__(kSelThreads) void select_kernel(EvictParams p) {
  __shared__ uint4 keys[kQuads * kSelThreads];
  __shared__ __attribute__((aligned(16))) uint32_t hist[kBins];
  uint32_t* const list = hist + 1024;  // (the second and third passes have 1024 bins)
  __shared__ int tiles[kChunk / kTile];  // entry slots of a chunk's tiles, -1: none
  __shared__ uint32_t tot[2][kQuads * kSelWaves];
  __shared__ uint32_t part[kSelWaves];
  __shared__ uint32_t found[3];  // bin, still needed inside it, its count
  __shared__ uint32_t many[3];   // protected ones, zeros, keys listed
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  const int ip = p.indptr[b];
  const int64_t room = p.entries * p.block_size, first = (int64_t)ip * p.block_size;
  // tokens behind the table have no entry: what they would change, a shorter
  // sequence does not
  const int n = ip < 0 ? 0 : (int)min((int64_t)p.seq_lens[b], max((int64_t)0, room - first));
  if (n <= p.budget) {
    if (tid == 0) p.moves[blockIdx.x] = 0;
    return;
  }
  // free: positions in [sink, ends - recent); none without positions
  const int sink = p.positions ? p.sink : 0;
  const int64_t free_to = p.positions ? (int64_t)p.ends[b] - p.recent : 0;
  const uint32_t span = p.positions ? (uint32_t)max(free_to - sink, (int64_t)0) : 1u;
  const int chunks = (n + kChunk - 1) / kChunk;  // (n < 2^31 - 2^16: the table's room is)
  uint4* const far = reinterpret_cast<uint4*>(p.keys + (int64_t)h * room + first);

  // Quad j of thread t is tokens 4 * (t + 1024 j) .. + 3 of a chunk (a quad lies in
  // one page).  Tokens behind the sequence get key 0, like those without an
  // entry: they stand behind every other one of that key and are never needed.
  // run(ch, j): first token of this wave's 256; runs behind the sequence are
  // left out everywhere.
  const auto run = [&](int ch, int j) { return ch * kChunk + 4 * (j * kSelThreads + 64 * w); };
  // a quad's keys, from LDS or, where there are more chunks than one, from the
  // workspace (a thread reads back what it wrote itself)
  const auto get = [&](int ch, int j) -> uint4 {
    if (chunks == 1) return keys[j * kSelThreads + tid];
    return run(ch, j) + 4 * lane < n ? far[(run(ch, j) >> 2) + lane] : make_uint4(0, 0, 0, 0);
  };
  const auto put = [&](int ch, int j, uint4 k) {
    if (chunks == 1)
      keys[j * kSelThreads + tid] = k;
    else if (run(ch, j) + 4 * lane < n)
      far[(run(ch, j) >> 2) + lane] = k;
  };
  // the chunk's tile slots into LDS, one round trip for all of them; slot(): of a
  // quad's first token
  const auto load_tiles = [&](int ch) {
    __syncthreads();
    for (int t = tid; t < kChunk / kTile && ch * kChunk + t * kTile < n; t += kSelThreads)
      tiles[t] = slot_of(p, ip, ch * kChunk + t * kTile);
    __syncthreads();
  };
  const auto slot_in = [&](int j) {
    const int q = j * kSelThreads + tid, s = tiles[q >> 2];
    return s < 0 ? -1 : s + 4 * (q & 3);
  };
  // The keys, and the first pass over them while they come: their upper 12 bits
  // counted.  Protected ones and zeros are many: counted in registers, not in one
  // LDS counter each.
  if (tid < 3) many[tid] = 0;
  for (int i = tid; i < kBins / 4; i += kSelThreads)
    reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
  uint32_t held = 0, zeros = 0;
#pragma unroll 1
  for (int ch = 0; ch < chunks; ch++) {
    constexpr int H = 4;  // quads in flight
    load_tiles(ch);
#pragma unroll 1
    for (int j0 = 0; j0 < kQuads && run(ch, j0) < n; j0 += H) {
      int slot[H];
      float4 wt[H];
      int4 ps[H];
#pragma unroll
      for (int j = 0; j < H; j++) {
        const int i = run(ch, j0 + j) + 4 * lane;
        slot[j] = i < n ? slot_in(j0 + j) : -1;
      }
#pragma unroll
      for (int j = 0; j < H; j++) {
        const int64_t at = state_at(p, max(slot[j], 0), h);
        wt[j] = *reinterpret_cast<const float4*>(p.weights + at);
        ps[j] = p.positions ? *reinterpret_cast<const int4*>(p.positions + at)
                            : make_int4(0, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < H; j++) {
        const int left = slot[j] >= 0 ? n - run(ch, j0 + j) - 4 * lane : 0;
        put(ch, j0 + j,
            make_uint4(0 < left ? key_of(wt[j].x, ps[j].x, sink, span) : 0u,
                       1 < left ? key_of(wt[j].y, ps[j].y, sink, span) : 0u,
                       2 < left ? key_of(wt[j].z, ps[j].z, sink, span) : 0u,
                       3 < left ? key_of(wt[j].w, ps[j].w, sink, span) : 0u));
      }
#pragma unroll 1
      for (int j = j0; j < j0 + H && run(ch, j) < n; j++) {
        const uint4 q = get(ch, j);
        const uint32_t k[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          held += k[e] == kHeld;
          zeros += k[e] == kZero;
          if (k[e] != kHeld && k[e] != kZero) atomicAdd(&hist[k[e] >> 20], 1u);
        }
      }
    }
  }
  held = wave_scan(held);
  zeros = wave_scan(zeros);
  if (lane == 63 && held + zeros) {
    atomicAdd(&hist[kHeld >> 20], held);
    atomicAdd(&hist[kZero >> 20], zeros);
    atomicAdd(&many[0], held);
    atomicAdd(&many[1], zeros);
  }

  // The budget-th largest key, 12 + 10 + 10 bits at a time.
  uint32_t need = (uint32_t)p.budget, prefix = 0, equal = 0;
  uint32_t listed = 0;  // keys of the first pass's bin in `list`, 0: not listed
#pragma unroll 1
  for (int pass = 0; pass < 3; pass++) {
    const int bits = pass == 0 ? 12 : 10, shift = 20 - 10 * pass;
    const int bins = 1 << bits;
    if (pass) {
      for (int i = tid; i < bins / 4; i += kSelThreads)
        reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      if (listed) {
        for (uint32_t i = tid; i < listed; i += kSelThreads) {
          const uint32_t k = list[i];
          if (k >> (shift + 10) == prefix) atomicAdd(&hist[k >> shift & 1023], 1u);
        }
      } else {
#pragma unroll 1
        for (int ch = 0; ch < chunks; ch++)
#pragma unroll 1
          for (int j = 0; j < kQuads && run(ch, j) < n; j++) {
            const uint4 q = get(ch, j);
            const uint32_t k[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (k[e] >> (shift + 10) == prefix) atomicAdd(&hist[k[e] >> shift & 1023], 1u);
          }
      }
    }
    __syncthreads();
    // bins from the top, four a thread: the one where the count reaches need
    const bool mine = tid < bins / 4;
    const int top = bins - 4 - 4 * tid;  // the lowest of this thread's bins
    const uint4 hv = *reinterpret_cast<const uint4*>(hist + (mine ? top : 0));
    const uint32_t c[4] = {mine ? hv.w : 0u, mine ? hv.z : 0u, mine ? hv.y : 0u,
                           mine ? hv.x : 0u};
    const uint32_t own = c[0] + c[1] + c[2] + c[3];
    const uint32_t incl = wave_scan(own);
    if (lane == 63) part[w] = incl;
    __syncthreads();
    uint32_t before = incl - own;
#pragma unroll
    for (int k = 0; k < kSelWaves; k++) before += k < w ? part[k] : 0;
    if (before < need && need <= before + own) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (before < need && need <= before + c[i]) {
          found[0] = top + 3 - i;
          found[1] = need - before;
          found[2] = c[i];
        }
        before += c[i];
      }
    }
    __syncthreads();
    prefix = (prefix << bits) | found[0];
    need = found[1];
    equal = found[2];
    if (pass == 0) {
      // the cut is a protected key, or zero with no other key in its bin
      if (prefix == kHeld >> 20 && need <= many[0]) {
        prefix = kHeld;
        equal = many[0];
        break;
      }
      if (prefix == kZero >> 20 && equal == many[1]) {
        prefix = kZero;
        break;
      }
      // the bin's keys, if they fit the list, so that the other passes need not
      // look at all of them (in any order: they are only counted)
      if (equal <= kList) {
#pragma unroll 1
        for (int ch = 0; ch < chunks; ch++)
#pragma unroll 1
          for (int j = 0; j < kQuads && run(ch, j) < n; j++) {
            const uint4 q = get(ch, j);
            const uint32_t k[4] = {q.x, q.y, q.z, q.w};
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) m += k[e] >> 20 == prefix;
            if (!__any(m)) continue;
            const uint32_t sum = wave_scan(m);
            uint32_t at = 0;
            if (lane == 63) at = atomicAdd(&many[2], sum);
            at = __builtin_amdgcn_readlane(at, 63) + sum - m;
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (k[e] >> 20 == prefix && at < kList) list[at++] = k[e];
          }
        listed = equal;
      }
    }
  }
  const uint32_t cut = prefix;

  // Kept: keys from the cut on; of those equal to it only the first `need`,
  // which are made larger than the cut, and the others smaller, if need is not
  // all of them.  Ranks are counts of the (chunk, j, wave) runs before, and of
  // the tokens before in the run.
  // exclusive sums of v[0 .. kQuads * kSelWaves) on top of `base`, by wave 0;
  // returns the total
  const auto scan = [&](uint32_t* v, uint32_t base) -> uint32_t {
    __syncthreads();
    if (w == 0) {
      const uint32_t a0 = v[2 * lane], a1 = v[2 * lane + 1];
      const uint32_t incl = wave_scan(a0 + a1);
      v[2 * lane] = base + incl - a0 - a1;
      v[2 * lane + 1] = base + incl - a1;
      if (lane == 63) part[0] = base + incl;
    }
    __syncthreads();
    return part[0];
  };
  static_assert(kQuads * kSelWaves == 128, "scan() takes two counts a lane");
  const Lists lists = lists_of(p, blockIdx.x, h, ip);
  int32_t* const dst = p.dst + lists.at;
  int32_t* const src = p.src + lists.at;
  const uint32_t cap = (uint32_t)min(lists.room, (int64_t)(p.half ? n / 2 : p.budget));
  const bool ties = equal != need;
  const uint32_t from = ties && cut != kHeld ? cut + 1 : cut;  // kept: keys >= from
  uint32_t eq_base = 0, hole_base = 0, more_base = 0;
#pragma unroll 1
  for (int ch = 0; ch < chunks; ch++) {
    if (ties) {
#pragma unroll 1
      for (int j = 0; j < kQuads; j++) {
        uint32_t c = 0;
        if (run(ch, j) < n) {
          const uint4 q = get(ch, j);
          const uint32_t k[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int e = 0; e < 4; e++) c += __popcll(__ballot(k[e] == cut));
        }
        if (lane == 0) tot[0][j * kSelWaves + w] = c;
      }
      const uint32_t next = scan(tot[0], eq_base);
#pragma unroll 1
      for (int j = 0; j < kQuads && run(ch, j) < n; j++) {
        const uint4 q = get(ch, j);
        uint32_t k[4] = {q.x, q.y, q.z, q.w};
        uint32_t rank = tot[0][j * kSelWaves + w];
#pragma unroll
        for (int e = 0; e < 4; e++) rank = lanes_below(__ballot(k[e] == cut), rank);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const bool same = k[e] == cut;
          k[e] = same ? (rank < need ? kHeld : 0u) : k[e];
          rank += same;
        }
        put(ch, j, make_uint4(k[0], k[1], k[2], k[3]));
      }
      eq_base = next;
      __syncthreads();  // tot[0] is read
    }
    // holes in front of the budget, kept ones behind it
#pragma unroll 1
    for (int j = 0; j < kQuads; j++) {
      const int i0 = run(ch, j), i = i0 + 4 * lane;
      uint32_t a = 0, c = 0;
      if (i0 < n) {
        const uint4 q = get(ch, j);
        const uint32_t k[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint64_t in = __ballot(k[e] >= from), front = __ballot(i + e < p.budget);
          a += __popcll(~in & front);
          c += __popcll(in & ~front);
        }
      }
      if (lane == 0) {
        tot[0][j * kSelWaves + w] = a;
        tot[1][j * kSelWaves + w] = c;
      }
    }
    const uint32_t hole_next = scan(tot[0], hole_base);
    const uint32_t more_next = scan(tot[1], more_base);
    if (chunks > 1) load_tiles(ch);  // (no loads below: they would wait for the stores)
#pragma unroll 1
    for (int j = 0; j < kQuads && run(ch, j) < n; j++) {
      const int i = run(ch, j) + 4 * lane, slot = i < n ? slot_in(j) : -1;
      const uint4 q = get(ch, j);
      const uint32_t k[4] = {q.x, q.y, q.z, q.w};
      // (both sides only in the run that the budget falls into)
#pragma unroll 1
      for (int back = 0; back < 2; back++) {
        if (back ? run(ch, j) + 256 <= p.budget : run(ch, j) >= p.budget) continue;  // (uniform)
        int32_t* const to = back ? src : dst;
        uint32_t rank = tot[back][j * kSelWaves + w];
        bool mark[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          mark[e] = (k[e] >= from) == (bool)back && (i + e >= p.budget) == (bool)back;
          rank = lanes_below(__ballot(mark[e]), rank);
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (mark[e] && rank < cap) to[rank++] = slot < 0 ? -1 : slot + e;
      }
    }
    hole_base = hole_next;
    more_base = more_next;
    __syncthreads();  // tot is read
  }
  // exactly budget entries are kept, so there are as many holes as sources
  // (the bounds by cap and kList hold by themselves; they are for page tables whose
  // ranges overlap, where another sequence's keys may stand in the workspace)
  if (tid == 0) p.moves[blockIdx.x] = (int32_t)min(more_base, cap);
}

// Entry moves: a move takes 2 EBS / 16 lanes for the codes and norms of K and V
// and one for weight and position.  A round is a run of move numbers for up to
// eight heads of a sequence: the i-th holes of the heads lie close together, and
// so do the pieces of cache lines that they share.  The rounds of up to 64
// (sequence, head group)s are numbered through, so that a few long sequences
// keep every workgroup busy, and rounds that follow one another go to one XCD
// (workgroups x mod 8), whose L2 holds the lines they share: 50.5 us for 8 x 32768
// tokens cut to 8192, 63.2 with rounds dealt out one by one.
constexpr int kMoveHeads = 8, kMoveRows = 64, kXcds = 8;
template <int EBS>
__global__ __launch_bounds__(256) void move_kernel(EvictParams p) {
  constexpr int E = EBS / 16, C = 2 * E + 1, NI = 4, PAIRS = 256 * NI / C;
  static_assert(PAIRS <= 256, "a move a thread");
  __shared__ int to_s[PAIRS], of_s[PAIRS];
  const int lane = threadIdx.x & 63;
  const int groups = (p.Hkv + kMoveHeads - 1) / kMoveHeads;
  // lane i of every wave: (sequence, head group) i of the grid row, its rounds
  // and those before
  const int row = blockIdx.y * kMoveRows + lane;
  const int lb = row / groups, lh = row - lb * groups, lh0 = lh * kMoveHeads;
  int lrounds = 0, lip = 0;
  if (lb < p.B) {
    if (p.half) lip = p.indptr[lb];
    const int heads = min(kMoveHeads, p.Hkv - lh0);
    int most = 0;
#pragma unroll
    for (int i = 0; i < kMoveHeads; i++)
      most = max(most, p.moves[lb * p.Hkv + lh0 + min(i, heads - 1)]);
    const int per = PAIRS / heads;
    lrounds = (int)(((uint32_t)most + per - 1) / per);
    if (lh == 0 && blockIdx.x == 0 && threadIdx.x < 64)
      p.new_lens[lb] = min(p.seq_lens[lb], p.budget);
  }
  const uint32_t lend = wave_scan((uint32_t)lrounds);
  const uint32_t rounds = __builtin_amdgcn_readlane(lend, 63);
  // 2^run rounds of every 2^(run + 3) in a row are one XCD's
  const uint32_t x = blockIdx.x;
  int run = min(5, 31 - __builtin_clz(gridDim.x / kXcds));
  while (run > 0 && (uint32_t)kXcds << run > rounds) run--;
  const uint32_t in = x & ((kXcds << run) - 1);
  uint32_t r = x - in + (in % kXcds << run) + in / kXcds;

  // this thread's move of a round (pairs <= 256), loaded a round ahead
  int to = -1, of = -1, nh = 1, nh0 = 0, npairs = 0;  // of the loaded round
  const auto load = [&](uint32_t round) {
    to = -1;
    if (round >= rounds) return;
    const int k = __popcll(__ballot(lend <= round));
    const int b = __builtin_amdgcn_readlane(lb, k);
    nh0 = __builtin_amdgcn_readlane(lh0, k);
    nh = min(kMoveHeads, p.Hkv - nh0);
    const int per = PAIRS / nh;
    npairs = per * nh;
    const int im = (int)threadIdx.x / nh, hm = (int)threadIdx.x - im * nh;
    const int64_t m =
        (int64_t)(round - (k ? __builtin_amdgcn_readlane(lend, max(k - 1, 0)) : 0)) * per + im;
    const int bh = b * p.Hkv + nh0 + hm;
    const Lists lists = lists_of(p, bh, nh0 + hm, __builtin_amdgcn_readlane(lip, k));
    if ((int)threadIdx.x < npairs && m < lists.room) {
      const int n = p.moves[bh];
      const int d = p.dst[lists.at + m], s = p.src[lists.at + m];
      to = m < n && s >= 0 ? d : -1;  // (-1: none, or on no page of the cache)
      of = s;
    }
  };
  load(r);
  for (; r < rounds; r += gridDim.x) {
    const int heads = nh, h0 = nh0, pairs = npairs;
    __syncthreads();
    if ((int)threadIdx.x < pairs) {
      to_s[threadIdx.x] = to;
      of_s[threadIdx.x] = of;
    }
    __syncthreads();
    load(r + gridDim.x);
    uint4 v[NI];
    int64_t at[NI];
    int c[NI];
#pragma unroll
    for (int j = 0; j < NI; j++) {
      const int f = threadIdx.x + 256 * j, i = f / C;
      c[j] = f - i * C;
      const int to = i < pairs ? to_s[i] : -1;
      if (to < 0) {
        c[j] = C;
        continue;
      }
      const int of = of_s[i], h = h0 + i % heads;
      if (c[j] < 2 * E) {
        const int o = (c[j] < E ? c[j] : c[j] - E) * 16;
        const uint8_t* const slab = c[j] < E ? p.ks : p.vs;
        at[j] = ((int64_t)to * p.Hkv + h) * EBS + o;
        v[j] = *reinterpret_cast<const uint4*>(slab + ((int64_t)of * p.Hkv + h) * EBS + o);
      } else {
        const int64_t z = state_at(p, of, h);
        at[j] = state_at(p, to, h);
        v[j].x = __float_as_uint(p.weights[z]);
        v[j].y = p.positions ? (uint32_t)p.positions[z] : 0u;
      }
    }
#pragma unroll
    for (int j = 0; j < NI; j++) {
      if (c[j] < 2 * E) {
        *reinterpret_cast<uint4*>((c[j] < E ? p.ks : p.vs) + at[j]) = v[j];
      } else if (c[j] == 2 * E) {
        p.weights[at[j]] = __uint_as_float(v[j].x);
        if (p.positions) p.positions[at[j]] = (int32_t)v[j].y;
      }
    }
  }
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// Lists of their own for every row, up to this many bytes of them; beyond, by
// table place, where they take 4 bytes per token of the table and head and no batch
// multiplies a budget that few sequences, or none, can exceed.
constexpr int64_t kOwnLists = 64 << 20;

struct EvictWs {
  size_t dst, src, moves, keys, total;
  int64_t cap, half;
};
EvictWs evict_ws(int batch, int hkv, int64_t entries, int bs, int budget) {
  EvictWs w;
  const int64_t room = entries * bs;
  w.cap = budget < room ? budget : room;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += up256(n);
    return r;
  };
  const int64_t rows = batch * hkv * w.cap, tables = hkv * (room / 2);
  w.half = rows * 8 > kOwnLists && tables < rows ? room / 2 : 0;
  w.dst = take((size_t)(w.half ? tables : rows) * 4);
  w.src = take((size_t)(w.half ? tables : rows) * 4);
  w.moves = take((size_t)batch * hkv * 4);
  w.keys = take(room > kChunk ? (size_t)room * hkv * 4 : 0);
  w.total = at;
  return w;
}

int check_evict(int batch, int hkv, int64_t entries, int bs, int budget) {
  if (batch < 0 || hkv <= 0 || hkv > 4096 || (int64_t)batch * hkv > 65535) {
    set_error("evict: batch %d x %d kv heads out of range", batch, hkv);
    return kEinval;
  }
  if (bs <= 0 || bs % kTile != 0) {
    set_error("evict: block_size %d must be a positive multiple of 16", bs);
    return kEinval;
  }
  if (entries < 0 || entries > 0x7fffffffLL || entries * bs > 0x7fff0000LL) {
    set_error("evict: %lld page-table entries of %d tokens out of range", (long long)entries, bs);
    return kEinval;
  }
  if (budget < 1) {
    set_error("evict: budget %d must be positive", budget);
    return kEinval;
  }
  return 0;
}

}  // namespace
}  // namespace tq

extern "C" int64_t tq_evict_workspace_bytes(int32_t batch, int32_t num_kv_heads,
                                            int64_t num_indices, int32_t block_size,
                                            int32_t budget) {
  using namespace tq;
  const int rc = check_evict(batch, num_kv_heads, num_indices, block_size, budget);
  if (rc) return rc;
  return (int64_t)evict_ws(batch, num_kv_heads, num_indices, block_size, budget).total;
}

extern "C" int tq_evict_paged(uint8_t* k_slab, uint8_t* v_slab, float* weights, int32_t* positions,
                              const int32_t* indices, int64_t num_indices, const int32_t* indptr,
                              const int32_t* seq_lens, const int32_t* ends, int32_t batch,
                              int32_t num_kv_heads, int32_t padded_dim, int32_t block_size,
                              int32_t ebs, int64_t num_blocks, int32_t budget, int32_t recent,
                              int32_t sink, int32_t* new_lens, void* workspace,
                              int64_t workspace_bytes, tq_stream_t stream) {
  using namespace tq;
  int rc = check_evict(batch, num_kv_heads, num_indices, block_size, budget);
  if (rc || batch == 0) return rc;
  if (padded_dim != 64 && padded_dim != 128 && padded_dim != 256) {
    set_error("evict: padded_dim must be 64, 128 or 256, got %d", padded_dim);
    return kEinval;
  }
  const int want = padded_dim == 64 ? 48 : (padded_dim == 128 ? 80 : 144);
  if (ebs != want) {
    set_error("evict: ebs %d does not match padded_dim %d (expected %d)", ebs, padded_dim, want);
    return kEinval;
  }
  if (recent < 0 || sink < 0 || (int64_t)recent + sink > budget) {
    set_error("evict: recent %d + sink %d must be non-negative and at most the budget %d", recent,
              sink, budget);
    return kEinval;
  }
  if (num_blocks <= 0 || num_blocks > 0x7fffffffLL ||
      num_blocks * (int64_t)block_size > 0x7fffffffLL) {
    set_error("evict: %lld blocks of %d tokens out of range", (long long)num_blocks, block_size);
    return kEinval;
  }
  if (!k_slab || !v_slab || !weights || (!indices && num_indices) || !indptr || !seq_lens ||
      !new_lens ||
      ((recent || sink) && !positions) || (positions && !ends)) {
    set_error("evict: null pointer");
    return kEinval;
  }
  if ((uintptr_t)k_slab % 16 || (uintptr_t)v_slab % 16 || (uintptr_t)weights % 16 ||
      (uintptr_t)positions % 16) {
    set_error("evict: cache slabs, weights and positions must be 16-byte aligned");
    return kEinval;
  }
  const EvictWs ws = evict_ws(batch, num_kv_heads, num_indices, block_size, budget);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < (int64_t)ws.total) {
    set_error("evict: the workspace must be 16-byte aligned and hold %lld bytes, got %lld",
              (long long)ws.total, (long long)workspace_bytes);
    return kEinval;
  }
  uint8_t* const base = static_cast<uint8_t*>(workspace);
  EvictParams p = {};
  p.indices = indices;
  p.indptr = indptr;
  p.seq_lens = seq_lens;
  p.ends = ends;
  p.entries = num_indices;
  p.num_blocks = (int)num_blocks;
  p.B = batch;
  p.Hkv = num_kv_heads;
  p.block_size = block_size;
  p.shift = block_size & (block_size - 1) ? -1 : __builtin_ctz(block_size);
  p.budget = budget;
  p.recent = recent;
  p.sink = sink;
  p.cap = ws.cap;
  p.half = ws.half;
  p.weights = weights;
  p.positions = positions;
  p.keys = num_indices * block_size > kChunk ? reinterpret_cast<uint32_t*>(base + ws.keys)
                                               : nullptr;
  p.dst = reinterpret_cast<int32_t*>(base + ws.dst);
  p.src = reinterpret_cast<int32_t*>(base + ws.src);
  p.moves = reinterpret_cast<int32_t*>(base + ws.moves);
  p.ks = k_slab;
  p.vs = v_slab;
  p.new_lens = new_lens;
  const int bh = batch * num_kv_heads;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(select_kernel, dim3((unsigned)bh), dim3(kSelThreads), 0, st, p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) {
    // Four workgroups a CU (64 at least for a grid row): with more at once fewer of
    // the lines that rounds have in common are shared, and those without work cost
    // their launch.  8 x 32768 tokens / 48 ragged sequences at head size 64 / 32
    // barely over their budget: 50.5 / 21.2 / 6.4 us, with 512 in all 57.9 / 22.0 /
    // 5.5, with 2048 56.7 / 22.2 / 7.3.
    const int64_t y = (int64_t)batch * ((num_kv_heads + kMoveHeads - 1) / kMoveHeads);
    const int64_t rows = (y + kMoveRows - 1) / kMoveRows;
    int64_t gx = 1024;
    while (gx > 64 && gx * rows > 1024) gx /= 2;
    const dim3 grid((unsigned)gx, (unsigned)rows);
    if (ebs == 48)
      hipLaunchKernelGGL(move_kernel<48>, grid, dim3(256), 0, st, p);
    else if (ebs == 80)
      hipLaunchKernelGGL(move_kernel<80>, grid, dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL(move_kernel<144>, grid, dim3(256), 0, st, p);
    e = hipGetLastError();
  }
  if (e != hipSuccess) {
    set_error("evict: launch failed: %s", hipGetErrorString(e));
    return (int)e;
  }
  return 0;
}
