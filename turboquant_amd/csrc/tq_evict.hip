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
// positions once into keys in LDS (32 bits that order like the rule above),
// finds the budget-th largest by three radix passes (11 + 11 + 10 bits) and
// lists sources and destinations in index order by ballots.  move_kernel
// copies the listed entries, all (sequence, head) pairs at once.
#include "tq_common.h"

namespace tq {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kLdsKeys = 32768;
constexpr int kBins = 2048;

struct EvictParams {
  const int32_t* indices;
  const int32_t* indptr;
  const int32_t* seq_lens;
  const int32_t* ends;
  int64_t entries;
  int num_blocks, B, Hkv, block_size, shift;  // shift: log2 block_size or -1
  int budget, recent, sink;
  int64_t cap;  // moves per (sequence, head) at most
  float* weights;
  int32_t* positions;
  uint32_t* keys;  // [Hkv][entries * block_size], for sequences longer than kLdsKeys
  int32_t* dst;    // [B * Hkv][cap] entry slots (page * block_size + place, -1: none)
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

// Larger key, kept sooner: 0 no entry, 1 NaN, then the weights in order
// (-0 as 0), all ones: protected.
__device__ __forceinline__ uint32_t key_of(const EvictParams& p, int ip, int i, int h,
                                           int64_t from) {
  const int slot = slot_of(p, ip, i);
  if (slot < 0) return 0;
  const int64_t at = state_at(p, slot, h);
  const float w = p.weights[at];
  if (p.positions) {
    const int pos = p.positions[at];
    if (pos < p.sink || pos >= from) return 0xffffffffu;
  }
  if (w != w) return 1;
  const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kSelThreads) void select_kernel(EvictParams p) {
  __shared__ uint32_t lds_keys[kLdsKeys];
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t tot[2][kSelWaves];
  __shared__ uint32_t found[3];  // bin, still needed inside it, its count
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
  const bool in_lds = n <= kLdsKeys;
  uint32_t* const far = p.keys + (int64_t)h * room + first;
  auto key = [&](int i) -> uint32_t { return in_lds ? lds_keys[i] : far[i]; };
  const int64_t from =
      p.positions && p.ends ? (int64_t)p.ends[b] - p.recent : (int64_t)0x7fffffffffffffff;
  for (int i = tid; i < n; i += kSelThreads) {  // (n < 2^31 - 2^10: room is)
    const uint32_t k = key_of(p, ip, i, h, from);
    if (in_lds)
      lds_keys[i] = k;
    else
      far[i] = k;
  }

  // the budget-th largest key, 11 + 11 + 10 bits at a time
  uint32_t need = (uint32_t)p.budget, prefix = 0, equal = 0;
  int shift = 21;
#pragma unroll
  for (int pass = 0; pass < 3; pass++) {
    const int bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSelThreads) {
      const uint32_t k = key(i);
      if (pass == 0 || (k >> (shift + bits)) == prefix)
        atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // bins from the top, two per thread: the one where the count reaches need
    const uint32_t c0 = hist[kBins - 1 - 2 * tid], c1 = hist[kBins - 2 - 2 * tid];
    uint32_t incl = c0 + c1;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t y = __shfl_up(incl, d);
      if (lane >= d) incl += y;
    }
    if (lane == 63) tot[0][w] = incl;
    __syncthreads();
    uint32_t before = incl - c0 - c1;
#pragma unroll
    for (int k = 0; k < kSelWaves; k++) before += k < w ? tot[0][k] : 0;
    if (before < need && need <= before + c0) {
      found[0] = kBins - 1 - 2 * tid;
      found[1] = need - before;
      found[2] = c0;
    } else if (before + c0 < need && need <= before + c0 + c1) {
      found[0] = kBins - 2 - 2 * tid;
      found[1] = need - before - c0;
      found[2] = c1;
    }
    __syncthreads();
    prefix = (prefix << bits) | found[0];
    need = found[1];
    equal = found[2];
    shift -= pass == 1 ? 10 : 11;
    __syncthreads();
  }
  const uint32_t cut = prefix;

  // each wave takes a run of indices, so that ranks are counts of the waves
  // before plus counts of the lanes below
  const int seg = ((n + kSelThreads - 1) / kSelThreads) * 64;
  const int i0 = min(w * seg, n), i1 = min(i0 + seg, n);
  const uint64_t below = lane ? ~0ull >> (64 - lane) : 0ull;
  uint32_t eq0 = 0;  // keys equal to the cut before this wave's run
  if (equal != need) {
    uint32_t c = 0;
    for (int i = i0; i < i1; i += 64)
      c += __popcll(__ballot(i + lane < i1 && key(min(i + lane, n - 1)) == cut));
    if (lane == 0) tot[0][w] = c;
    __syncthreads();
    for (int k = 0; k < w; k++) eq0 += tot[0][k];
    __syncthreads();
  }
  // kept: above the cut, or one of the first `need` equal to it
  auto kept = [&](int i, uint32_t& eq) -> bool {
    const bool in = i + lane < i1;
    const uint32_t k = in ? key(i + lane) : 0u;
    bool keep = in && k > cut;
    const uint64_t same = __ballot(in && k == cut);
    if (in && k == cut) keep = eq + __popcll(same & below) < need;
    eq += __popcll(same);
    return keep;
  };
  uint32_t holes = 0, more = 0, eq = eq0;
  for (int i = i0; i < i1; i += 64) {
    const bool keep = kept(i, eq), in = i + lane < i1, front = i + lane < p.budget;
    holes += __popcll(__ballot(in && !keep && front));
    more += __popcll(__ballot(in && keep && !front));
  }
  if (lane == 0) {
    tot[0][w] = holes;
    tot[1][w] = more;
  }
  __syncthreads();
  uint32_t hole0 = 0, more0 = 0;
  for (int k = 0; k < w; k++) {
    hole0 += tot[0][k];
    more0 += tot[1][k];
  }
  int32_t* const dst = p.dst + (int64_t)blockIdx.x * p.cap;
  int32_t* const src = p.src + (int64_t)blockIdx.x * p.cap;
  eq = eq0;
  for (int i = i0; i < i1; i += 64) {
    const bool keep = kept(i, eq), in = i + lane < i1, front = i + lane < p.budget;
    const uint64_t hm = __ballot(in && !keep && front), mm = __ballot(in && keep && !front);
    if (in && !keep && front) dst[hole0 + __popcll(hm & below)] = slot_of(p, ip, i + lane);
    if (in && keep && !front) src[more0 + __popcll(mm & below)] = slot_of(p, ip, i + lane);
    hole0 += __popcll(hm);
    more0 += __popcll(mm);
  }
  // exactly budget entries are kept, so there are as many holes as sources
  if (w == kSelWaves - 1 && lane == 0) p.moves[blockIdx.x] = (int32_t)more0;
}

// Entry moves: each takes 2 EBS / 16 lanes for the codes and norms of K and V
// and one for weight and position.
template <int EBS>
__global__ __launch_bounds__(256) void move_kernel(EvictParams p) {
  constexpr int E = EBS / 16, C = 2 * E + 1;
  const int bh = blockIdx.y, h = bh % p.Hkv;
  if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0) {
    const int b = bh / p.Hkv;
    p.new_lens[b] = min(p.seq_lens[b], p.budget);
  }
  const int64_t items = (int64_t)p.moves[bh] * C;
  const int32_t* const dst = p.dst + bh * p.cap;
  const int32_t* const src = p.src + bh * p.cap;
  for (int64_t f = (int64_t)blockIdx.x * 256 + threadIdx.x; f < items;
       f += (int64_t)gridDim.x * 256) {
    const int64_t m = f / C;
    const int c = (int)(f - m * C);
    const int to = dst[m], of = src[m];
    if (to < 0 || of < 0) continue;  // on no page of the cache
    if (c < 2 * E) {
      uint8_t* const slab = c < E ? p.ks : p.vs;
      const int o = (c < E ? c : c - E) * 16;
      *reinterpret_cast<uint4*>(slab + ((int64_t)to * p.Hkv + h) * EBS + o) =
          *reinterpret_cast<const uint4*>(slab + ((int64_t)of * p.Hkv + h) * EBS + o);
    } else {
      const int64_t a = state_at(p, to, h), z = state_at(p, of, h);
      p.weights[a] = p.weights[z];
      if (p.positions) p.positions[a] = p.positions[z];
    }
  }
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

struct EvictWs {
  size_t dst, src, moves, keys, total;
  int64_t cap;
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
  w.dst = take((size_t)batch * hkv * w.cap * 4);
  w.src = take((size_t)batch * hkv * w.cap * 4);
  w.moves = take((size_t)batch * hkv * 4);
  w.keys = take(room > kLdsKeys ? (size_t)room * hkv * 4 : 0);
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
  if (!k_slab || !v_slab || !weights || (!indices && num_indices) || !indptr || !seq_lens || !new_lens ||
      ((recent || sink) && !positions) || (positions && !ends)) {
    set_error("evict: null pointer");
    return kEinval;
  }
  if ((uintptr_t)k_slab % 16 || (uintptr_t)v_slab % 16) {
    set_error("evict: cache slabs must be 16-byte aligned");
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
  p.weights = weights;
  p.positions = positions;
  p.keys = num_indices * block_size > kLdsKeys ? reinterpret_cast<uint32_t*>(base + ws.keys)
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
    // up to four items a thread, and no more workgroups than keep the GPU busy
    const int64_t c = 2 * ebs / 16 + 1;
    int64_t gx = (ws.cap * c + 1023) / 1024;
    gx = gx < 1 ? 1 : gx;
    const int64_t most = 4096 / bh > 1 ? 4096 / bh : 1;
    gx = gx < most ? gx : most;
    const dim3 grid((unsigned)gx, (unsigned)bh);
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
