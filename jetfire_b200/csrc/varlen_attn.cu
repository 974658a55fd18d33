// Attention of packed prompts over their own keys and values (forward), on the fifth-generation tensor cores.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(f(scale q_i.k_j) - slope |i - j|) where i sees j
//
// One pass over the keys per row with a running reference m_i and sum l_i; nothing of size rows x keys leaves the chip.
// A work item is two tiles of 128 query rows that share every tile of 128 keys brought into shared memory: the same rows of two
// query heads of one KV head, or, where a KV head has a single query head, 256 rows of it.  S = Q K^T (fp32) stands in tensor memory, 128 columns per row tile; a thread owns a row: it
// reads its 128 scores, turns them into weights and writes them back, 16 bits each, over the scores, where they
// are the first operand of O += P V.  While one row tile's weights are computed the tensor core works on the other's products.
//
//   warps 0-3, 4-7   scores -> weights of row tile 0, 1; the rescaling of O when a reference moves; the result
//   warp 8           TMA loads: Q of an item, then K and V tiles through a ring of five 32 KB buffers
//   warp 9           issues the matrix products
//   warp 10          finds this block's work items (longest rows of all sequences first) ahead of the others
//   warp 11          clears values that are no numbers out of V tiles with masked entries
//
// The reference of a row lags its maximum by up to 2^kLag, so that O is rescaled rarely (both factors are exact
// powers in the exponent; the sum uses the same ones).  A masked entry's weight is 0, but 0 * inf in the product
// would not be: warp 11 looks at every V tile that has masked entries and zeroes infinities and NaN in it; rows that do see
// them get them back at the end (never, with finite inputs).
//
// The weights that meet V are rounded to the operands' type (half a step: bf16 2^-8 of themselves at most, fp16 2^-11); their sum, the scores and
// the output are fp32.
//
// Bound: per 128 x 128 scores the two products take 1024 cycles of the tensor core, the exponentials 1024 of the special function units (16
// a cycle).  One prompt of 8192 tokens, 64 / 8 heads, bf16, takes 883 to 902 us by itself = 1.22 to 1.25 PFLOP/s, 0.74 to 0.76 of what cuBLAS reaches, and
// 1010 among other calls, with the card near its power cap.  A
// step of both row tiles is 3500 cycles; with the weights left out it is 2950 (shared-memory reads of the operands and the hand-overs),
// and a row tile by itself goes through 1750 from its scores to its weights and waits 1020 for the next ones.

#include <cuda.h>

#include <algorithm>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "decode_common.cuh"
#include "tensor_common.cuh"

namespace jf {
namespace {

constexpr int kRows = 128, kKeys = 128;               // of a tile
constexpr int kKvStages = 5;
constexpr int kItems = 2;                             // work items looked up ahead
constexpr int kClean = 4;
constexpr int kThreads = 384;
// Registers: the warpgroups of rows take kRowRegs a thread, the other one is left kRoleRegs; together no more than the
// block is launched with (launch() checks that of the compiled kernel).
constexpr int kRowRegs = 208, kRoleRegs = 80;
constexpr float kLag = 8.0f;                          // log2
// schedule() goes through all sequences once a level, 0.27 us for 32 of them, and a block's items are up to 148 levels apart: so many
// keep who waits for one below 0.4 s.  An item of a sequence of so many rows goes through 2^17 key tiles, 9000 cycles each where scores
// lie beyond a cap: 0.9 s, for which schedule() waits.
constexpr int kMaxSeqs = 1 << 18, kMaxRows = 1 << 24;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
  const int32_t *cu, *prefix;
  const float* slopes;
  const uint16_t* v;
  uint16_t* out;
  float* lse;
  int32_t* status;
  int64_t v_stride_t, v_stride_h;
  int32_t T, n_seqs, H_q, H_kv, window;
  int32_t span, apart;    // rows of a sequence that an item covers; rows between its two tiles (0: same rows, two heads)
  int32_t G, units;       // query heads of a KV head; items per span of rows
  float scale, softcap;
  bool causal;
};

// row0: first row of the sequence (len < 0: no more items); q0: first row of the item in it; head: of its first tile; two: there is
// a second tile
struct Item { int row0, len, q0, head, prefix, two; };

struct Shared {
  uint64_t q_full, q_empty, products_done, kv_full[kKvStages], kv_empty[kKvStages], s_full[2], p_full[2][2], half_done[2], o_full[2], item_full[kItems], item_empty[kItems],
      cleaned[kClean];
  Item item[kItems];
  int bad[kItems];       // V tiles of the item held values that are no numbers
  uint32_t tmem;
};
constexpr int kSmemBytes = 2 * kTileBytes + kKvStages * kTileBytes + 1024;

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int head, int row, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(head), "r"(row), "r"(smem_u32(bar))
      : "memory");
}
// ---- which keys a row sees ----------------------------------------------------------------
__device__ __forceinline__ int first_key(const Params& P, int row) { return P.window > 0 ? max(0, row - P.window + 1) : 0; }
__device__ __forceinline__ int end_key(const Params& P, const Item& it, int row) {
  if (P.causal) return row + 1;
  return P.window > 0 ? static_cast<int>(min(static_cast<int64_t>(it.len), static_cast<int64_t>(row) + P.window)) : it.len;
}
__device__ __forceinline__ bool sees(const Params& P, const Item& it, int row, int j) {
  return j < it.len && (j < it.prefix || (j >= first_key(P, row) && j < end_key(P, it, row)));
}
// Key tiles of a row tile: some row sees some of tile t if t < some_p or lo <= t < hi; every row sees all of it if
// t < all_p or all_lo <= t < all_hi.
struct Tiles {
  int some_p, lo, hi, all_p, all_lo, all_hi;
  __device__ __forceinline__ bool uses(int t) const { return t < some_p || (t >= lo && t < hi); }
  __device__ __forceinline__ bool masked(int t) const { return t >= all_p && (t < all_lo || t >= all_hi); }
  __device__ __forceinline__ bool partly(int t) const { return uses(t) && masked(t); }
};
__device__ __forceinline__ Tiles tiles_of(const Params& P, const Item& it, int t) {
  if (t == 1 && !it.two) return Tiles{0, 0, 0, 0, 0, 0};
  const int q0 = it.q0 + t * P.apart;
  const int r1 = min(q0 + kRows, it.len) - 1;
  return Tiles{(it.prefix + kKeys - 1) / kKeys,
               first_key(P, q0) / kKeys,
               (end_key(P, it, r1) + kKeys - 1) / kKeys,
               it.prefix / kKeys,
               (first_key(P, r1) + kKeys - 1) / kKeys,
               min(end_key(P, it, q0), it.len) / kKeys};
}
// The key tiles of an item, the last first: count - a tiles down to `first`, then the prefix's a - 1 .. 0.  Each is used by one
// of its row tiles.  (From the row's own position backwards: where nearer keys weigh more, references settle early.)
struct Keys { int a, first, count; };
__device__ __forceinline__ Keys keys_of(const Params& P, const Item& it) {
  const int r0 = it.q0, r1 = min(r0 + P.span, it.len) - 1;
  const int np = (it.prefix + kKeys - 1) / kKeys, from = first_key(P, r0) / kKeys, to = (end_key(P, it, r1) + kKeys - 1) / kKeys;
  Keys k;
  k.a = min(np, from);
  k.first = from;
  k.count = k.a + max(to, np) - from;
  return k;
}
__device__ __forceinline__ int tile_of(const Keys& k, int i) {
  const int j = k.count - 1 - i;
  return j < k.a ? j : k.first + j - k.a;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {   // of two unsigned halves
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

template <int DT> __device__ __forceinline__ bool no_number(uint32_t half) {
  constexpr uint32_t inf = DT == JF_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
  return (half & inf) == inf;
}

// ---- the roles ------------------------------------------------------------------------------

// Work items of this block: level by level (the l-th span of rows of every sequence that has it, from the last), heads
// fastest, so that long rows come first and heads that share keys run at the same time; every gridDim.x-th is this block's.
__device__ __forceinline__ bool schedule(const Params& P, Shared& S) {
  const int lane = threadIdx.x & 31;
  int slot = 0, uses_of_slot = 0;
  auto emit = [&](int row0, int len, int q0, int unit, int prefix) {
    bool ok = true;
    if (uses_of_slot > 0) ok = wait_warp(&S.item_empty[slot], (uses_of_slot - 1) & 1);
    if (!ok) return false;
    if (lane == 0) {
      const int pairs = (P.G + 1) / 2, first = P.apart ? unit : unit / pairs * P.G + unit % pairs * 2;
      S.item[slot] = Item{row0, len, q0, first, prefix, P.apart ? q0 + P.apart < len : unit % pairs * 2 + 1 < P.G};
      S.bad[slot] = 0;
      mbar_arrive(&S.item_full[slot]);
    }
    __syncwarp();
    if (++slot == kItems) { slot = 0; ++uses_of_slot; }
    return true;
  };
  auto bounds = [&](int s, int& row0, int& len) {
    row0 = len = 0;
    if (s < P.n_seqs) {
      row0 = min(max(P.cu[s], 0), P.T);
      len = min(max(P.cu[s + 1], row0), P.T) - row0;
    }
  };
  int row0, len, most = 0;
  for (int c = 0; c < P.n_seqs; c += 32) {
    bounds(c + lane, row0, len);
    most = max(most, static_cast<int>(__reduce_max_sync(0xFFFFFFFFu, static_cast<unsigned>(len))));
  }
  int64_t want = blockIdx.x, before = 0;
  for (int level = (most + P.span - 1) / P.span - 1; level >= 0; --level)
    for (int c = 0; c < P.n_seqs; c += 32) {
      if (P.n_seqs > 32) bounds(c + lane, row0, len);
      const unsigned has = __ballot_sync(0xFFFFFFFFu, len > level * P.span);
      const int64_t n = static_cast<int64_t>(__popc(has)) * P.units;
      while (want < before + n) {
        const int at = static_cast<int>(want - before), src = __fns(has, 0, at / P.units + 1);
        const int r = __shfl_sync(0xFFFFFFFFu, row0, src), l = __shfl_sync(0xFFFFFFFFu, len, src);
        const int prefix = P.prefix ? min(max(P.prefix[c + src], 0), l) : 0;
        if (!emit(r, l, level * P.span, at % P.units, prefix)) return false;
        want += gridDim.x;
      }
      before += n;
    }
  return emit(0, -1, 0, 0, 0);
}

struct ItemReader {
  int slot = 0, round = 0;
  __device__ __forceinline__ bool next(Shared& S, Item& it) {
    if (!wait_warp(&S.item_full[slot], round & 1)) return false;
    it = S.item[slot];
    return true;
  }
  __device__ __forceinline__ void release_warp(Shared& S) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&S.item_empty[slot]);
    if (++slot == kItems) { slot = 0; ++round; }
  }
};
struct Ring {   // position in the ring of K and V tiles
  int stage = 0, round = 0;
  __device__ __forceinline__ void step(int n = 1) {
    stage += n;
    if (stage >= kKvStages) { stage -= kKvStages; ++round; }
  }
  __device__ __forceinline__ void back() {
    if (--stage < 0) { stage = kKvStages - 1; --round; }
  }
};

// `loaded`: Q tiles asked for; `ring`: one past the last K or V tile asked for.
__device__ __forceinline__ bool load(const Params& P, Shared& S, uint32_t q_smem, uint32_t kv_smem, const CUtensorMap* qm, const CUtensorMap* km,
                                     const CUtensorMap* vm, int& loaded, Ring& ring) {
  ItemReader items;
  Item it;
  for (int& n = loaded;;) {
    if (!items.next(S, it)) return false;
    if (it.len < 0) return true;
    const Keys keys = keys_of(P, it);
    const int kvh = it.head / P.G, tiles = it.two ? 2 : 1;
    if (n > 0 && !wait_warp(&S.q_empty, (n - 1) & 1)) return false;
    if (elect_one()) {
      mbar_expect_tx(&S.q_full, tiles * kTileBytes);
      for (int t = 0; t < tiles; ++t)
        for (int slab = 0; slab < 2; ++slab)
          tma_load(q_smem + t * kTileBytes + slab * kSlabBytes, qm, slab * 64, it.head + (P.apart ? 0 : t), it.row0 + it.q0 + t * P.apart, &S.q_full);
    }
    __syncwarp();
    ++n;
    for (int i = 0; i < keys.count; ++i) {
      const int row = it.row0 + tile_of(keys, i) * kKeys;
      for (int side = 0; side < 2; ++side) {
        if (ring.round > 0 && !wait_warp(&S.kv_empty[ring.stage], (ring.round - 1) & 1)) return false;
        if (elect_one()) {
          mbar_expect_tx(&S.kv_full[ring.stage], kTileBytes);
          for (int slab = 0; slab < 2; ++slab)
            tma_load(kv_smem + ring.stage * kTileBytes + slab * kSlabBytes, side ? vm : km, slab * 64, kvh, row, &S.kv_full[ring.stage]);
        }
        __syncwarp();
        ring.step();
      }
    }
    items.release_warp(S);
  }
}

// The copies that may be in flight: the block's shared memory stays until they are there, or a wait for one runs out.
__device__ __forceinline__ bool arrived(Shared& S, int loaded, Ring ring) {
  if (loaded > 0 && !wait_warp(&S.q_full, (loaded - 1) & 1)) return false;
  for (int i = 0; i < kKvStages && (ring.round > 0 || ring.stage > 0); ++i) {
    ring.back();
    if (!wait_warp(&S.kv_full[ring.stage], ring.round & 1)) return false;
  }
  return true;
}

template <int DT> __device__ __forceinline__ bool multiply(const Params& P, Shared& S, uint32_t q_smem, uint32_t kv_smem, uint32_t tmem) {
  constexpr uint32_t qk = instruction<DT>(false), pv = instruction<DT>(true);
  const uint64_t q_op = operand(q_smem, 16), k_op = operand(kv_smem, 16), v_op = operand(kv_smem, kSlabBytes);
  ItemReader items;
  Item it;
  Ring ring;
  int p_count[2] = {0, 0}, clean = 0;
  for (int n = 0;; ++n) {
    if (!items.next(S, it)) return false;
    if (it.len < 0) return true;
    const Keys keys = keys_of(P, it);
    const Tiles tiles[2] = {tiles_of(P, it, 0), tiles_of(P, it, 1)};
    int last[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      last[t] = keys.count - 1;
      while (last[t] >= 0 && !tiles[t].uses(tile_of(keys, last[t]))) --last[t];
    }
    if (!wait_warp(&S.q_full, n & 1)) return false;
    bool started[2] = {false, false};
    bool now[2] = {false, false};   // row tile t uses key tile i
    for (int i = -1; i < keys.count; ++i) {
      // products with V of tile i and scores of tile i + 1, row tile by row tile
      Ring v_ring = ring, k_ring = ring;
      if (i >= 0) k_ring.step();
      const int tile = i >= 0 ? tile_of(keys, i) : 0, then = tile_of(keys, i + 1);
      const bool more = i + 1 < keys.count, look = i >= 0 && (tiles[0].partly(tile) || tiles[1].partly(tile));
      const bool next[2] = {more && tiles[0].uses(then), more && tiles[1].uses(then)};
      bool v_here = false, k_here = false;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (now[t]) {
          if (!v_here) {
            if (!wait_warp(&S.kv_full[v_ring.stage], v_ring.round & 1)) return false;
            if (look) {
              if (!wait_warp(&S.cleaned[clean % kClean], clean / kClean & 1)) return false;
              ++clean;
            }
            v_here = true;
          }
          const uint64_t b = v_op + v_ring.stage * (kTileBytes >> 4);
#pragma unroll
          for (int h = 0; h < 2; ++h) {   // the weights come in two halves
            if (!wait_warp(&S.p_full[t][h], p_count[t] & 1)) return false;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k = h * 4; k < h * 4 + 4; ++k)
                mma_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, b + k * (2048 >> 4), pv, started[t] || k > 0);
              if (h == 0) tc_commit(&S.half_done[t]);
              else if (i == last[t]) tc_commit(&S.o_full[t]);
            }
            __syncwarp();
          }
          ++p_count[t];
          started[t] = true;
        }
        if (next[t]) {
          if (!k_here) {
            if (!wait_warp(&S.kv_full[k_ring.stage], k_ring.round & 1)) return false;
            k_here = true;
          }
          tc_fence_after();
          const uint64_t a = q_op + t * (kTileBytes >> 4), b = k_op + k_ring.stage * (kTileBytes >> 4);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t off = ((k >> 2) * kSlabBytes + (k & 3) * 32) >> 4;
              mma_ss(tmem + t * 128, a + off, b + off, qk, k > 0);
            }
            tc_commit(&S.s_full[t]);
          }
          __syncwarp();
        }
        now[t] = next[t];
      }
      if (elect_one()) {
        if (i >= 0) tc_commit(&S.kv_empty[v_ring.stage]);
        if (more) tc_commit(&S.kv_empty[k_ring.stage]);
        if (i + 2 == keys.count) tc_commit(&S.q_empty);
      }
      __syncwarp();
      ring = k_ring;
      ring.step();
    }
    // (the last step moved past a K tile that does not exist)
    ring.back();
    items.release_warp(S);
  }
}

template <int DT> __device__ __forceinline__ bool clean_values(const Params& P, Shared& S, unsigned char* kv) {
  constexpr uint32_t inf = DT == JF_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
  const int lane = threadIdx.x & 31;
  ItemReader items;
  Item it;
  Ring ring;
  int clean = 0;
  for (;;) {
    if (!items.next(S, it)) return false;
    if (it.len < 0) return true;
    const Keys keys = keys_of(P, it);
    const Tiles upper = tiles_of(P, it, 0), lower = tiles_of(P, it, 1);
    for (int i = 0; i < keys.count; ++i) {
      // every buffer is waited for and passed on, so that none is filled twice in between
      if (!wait_warp(&S.kv_full[ring.stage], ring.round & 1)) return false;
      if (lane == 0) mbar_arrive(&S.kv_empty[ring.stage]);
      ring.step();
      if (!wait_warp(&S.kv_full[ring.stage], ring.round & 1)) return false;
      const int t = tile_of(keys, i);
      if (upper.partly(t) || lower.partly(t)) {
        uint4* tile = reinterpret_cast<uint4*>(kv + ring.stage * kTileBytes);
        uint32_t top = 0;
#pragma unroll 8
        for (int n = lane; n < kTileBytes / 16; n += 32) {
          const uint4 x = tile[n];
          top = max2(max2(top, max2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu)), max2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
        }
        if (__any_sync(0xFFFFFFFFu, max(top & 0xFFFFu, top >> 16) >= inf)) {
          bool own = false;   // among the sequence's own rows
          for (int n = lane; n < kTileBytes / 4; n += 32) {
            uint32_t* w = reinterpret_cast<uint32_t*>(tile) + n;
            const uint32_t x = *w, y = (no_number<DT>(x) ? 0u : x & 0xFFFFu) | (no_number<DT>(x >> 16) ? 0u : x & 0xFFFF0000u);
            if (x != y) {
              *w = y;
              own |= t * kKeys + (n * 4 % kSlabBytes) / 128 < it.len;
            }
          }
          fence_proxy_async();
          if (__any_sync(0xFFFFFFFFu, own) && lane == 0) S.bad[items.slot] = 1;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.cleaned[clean % kClean]);
        ++clean;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.kv_empty[ring.stage]);
      ring.step();
    }
    items.release_warp(S);
  }
}

// 64 scores -> softened and biased ones, in units of log2.  `apart`: the row's position minus the first key's; `lin`: 1 if
// every key stands before every row of the tile, -1 if behind, 0 if neither.
template <bool CAP> __device__ __forceinline__ void reshape(float* s, const Params& P, float slope2, int apart, int lin) {
  const float sl2 = P.scale * kLog2e;
  if (CAP) {
    const float in = P.scale / P.softcap, cap2 = P.softcap * kLog2e;
    float most = 0.0f;
#pragma unroll
    for (int c = 0; c < 64; ++c) most = fmaxf(most, fabsf(s[c]));
    if (__all_sync(0xFFFFFFFFu, most * fabsf(in) <= 1.0f)) {
      // tanh z = z (1 + w q(w)), w = z^2 <= 1, q fitted here for the least relative error of the whole: 6.6e-7
      const uint64_t in2 = pair(in, in), c2 = pair(cap2, cap2);
#pragma unroll
      for (int c = 0; c < 64; c += 2) {
        const uint64_t z = mul2(pair(s[c], s[c + 1]), in2), w = mul2(z, z);
        uint64_t q = fma2(w, pair(-0.00312657771f, -0.00312657771f), pair(0.0169064086f, 0.0169064086f));
        q = fma2(q, w, pair(-0.0517682843f, -0.0517682843f));
        q = fma2(q, w, pair(0.132884905f, 0.132884905f));
        q = fma2(q, w, pair(-0.333302796f, -0.333302796f));
        q = fma2(q, w, pair(1.0f, 1.0f));
        split(mul2(mul2(z, c2), q), s[c], s[c + 1]);
      }
    } else {   // cap tanh z = cap - 2 cap / (e^(2z) + 1); a NaN stays one
      const float to_e = 2.0f * in * kLog2e;
#pragma unroll
      for (int c = 0; c < 64; ++c) s[c] = cap2 - __fdividef(2.0f * cap2, ex2(min_or_nan(s[c] * to_e, 126.0f)) + 1.0f);
    }
  }
  const float mul = CAP ? 1.0f : sl2;
  if (lin != 0) {
    // -slope |i - j| = lin * slope * (j - i) = k (c - apart) for the c-th key: four pairs that go on by 8 k, so that no
    // constants have to be brought up (what eight additions round is 2^-21 of the bias)
    const float k = lin * slope2;
    const uint64_t on = pair(8.0f * k, 8.0f * k), m2 = pair(mul, mul);
    uint64_t bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = pair(k * static_cast<float>(2 * e - apart), k * static_cast<float>(2 * e + 1 - apart));
#pragma unroll
    for (int c = 0; c < 64; c += 2) {
      uint64_t& b = bias[c / 2 & 3];
      const uint64_t x = pair(s[c], s[c + 1]);
      split(CAP ? add2(x, b) : fma2(x, m2, b), s[c], s[c + 1]);
      b = add2(b, on);
    }
  } else {
    const float a = static_cast<float>(apart);
#pragma unroll
    for (int c = 0; c < 64; ++c) s[c] = fmaf(fabsf(a - static_cast<float>(c)), -slope2, CAP ? s[c] : s[c] * mul);
  }
}

// Weights of 64 scores, 16 bits each, and their sum (added to `sum`).  A polynomial on the multiply-add units for a
// quarter of the exponentials gained nothing here (8192 tokens 949 -> 977 us).
template <int DT, bool SCALED> __device__ __forceinline__ void weigh(const float* s, uint32_t* p, uint64_t* sum, float sl2, float ref) {
  const uint64_t m2 = pair(sl2, sl2), r2 = pair(-ref, -ref);
#pragma unroll
  for (int c = 0; c < 64; c += 2) {
    float a, b;
    split(SCALED ? add2(pair(s[c], s[c + 1]), r2) : fma2(pair(s[c], s[c + 1]), m2, r2), a, b);
    a = ex2(a);
    b = ex2(b);
    sum[c / 2 & 1] = add2(sum[c / 2 & 1], pair(a, b));
    p[c / 2] = round2<DT>(a, b);
  }
}

// The same for scores under a cap whose magnitude stays below it: x = f(s) - ref with f(s) = s (c0 + w q(w)), w = s^2.
template <int DT, int TERMS> __device__ __forceinline__ void weigh_capped(const float* s, uint32_t* p, uint64_t* sum, const float (&co)[TERMS], float ref) {
  const uint64_t r2 = pair(-ref, -ref);
#pragma unroll
  for (int c = 0; c < 64; c += 2) {
    const uint64_t x = pair(s[c], s[c + 1]), w = mul2(x, x);
    uint64_t q = fma2(w, pair(co[TERMS - 1], co[TERMS - 1]), pair(co[TERMS - 2], co[TERMS - 2]));
#pragma unroll
    for (int k = TERMS - 3; k >= 0; --k) q = fma2(q, w, pair(co[k], co[k]));
    float a, b;
    split(fma2(x, q, r2), a, b);
    a = ex2(a);
    b = ex2(b);
    sum[c / 2 & 1] = add2(sum[c / 2 & 1], pair(a, b));
    p[c / 2] = round2<DT>(a, b);
  }
}

// Smallest of 64 scores, NaN left out of account.
__device__ __forceinline__ float smallest(const float* s) {
  float x[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int c = 4; c < 64; c += 4)
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = fminf(x[k], s[c + k]);
  return fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
}

// Largest of N scores; a NaN if there is one.
template <int N> __device__ __forceinline__ float largest(const float* s) {
  float x[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = s[k];
#pragma unroll
  for (int c = 4; c < N - 4; c += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = max3(x[k], s[c + k], s[c + 4 + k]);
  return max3(max3(x[0], x[1], s[N - 4]), max3(x[2], x[3], s[N - 3]), max3(s[N - 2], s[N - 1], s[N - 1]));
}

// Adds to a row of the result what the cleaned tiles' infinities and NaN do to it.
template <int DT> __device__ __noinline__ void give_back(const Params& P, const Item it, int row, uint16_t* out) {
  const Keys keys = keys_of(P, it);
  const Tiles upper = tiles_of(P, it, 0), lower = tiles_of(P, it, 1);
  for (int i = 0; i < keys.count; ++i) {
    const int tile = tile_of(keys, i);
    if (!upper.partly(tile) && !lower.partly(tile)) continue;
    for (int j = tile * kKeys; j < min((tile + 1) * kKeys, it.len); ++j) {
      if (!sees(P, it, row, j)) continue;
      const uint16_t* v = P.v + (static_cast<int64_t>(it.row0) + j) * P.v_stride_t + it.head / P.G * P.v_stride_h;
      for (int k = 0; k < JF_HEAD_DIM; ++k)
        if (no_number<DT>(v[k])) out[k] = Elem<DT>::from_f32(Elem<DT>::to_f32(out[k]) + Elem<DT>::to_f32(v[k]));
    }
  }
}

// FEAT: 0 plain, 1 bias (and scores that are scaled before their maximum is taken), 2 cap, with or without bias
template <int DT, int FEAT> __device__ __forceinline__ bool soften(const Params& P, Shared& S, uint32_t tmem, int t) {
  constexpr float kLift = DT == JF_DTYPE_FP16 ? 7.0f : 0.0f;   // fp16 weights use the range up to 2^15
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5 & 3, r = warp * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
  const uint32_t s_at = tmem + lanes + t * 128, o_at = tmem + lanes + 256 + t * 128;
  const float sl2 = P.scale * kLog2e;
  // log2(e) cap tanh(scale s / cap) = s (co[0] + co[1] s^2 + ...) while |s| <= cap_in (the fit of reshape(), in s); up to half of that two
  // terms fewer are as close (fitted the same way: 6.5e-7): packed documents 338 -> 327 us
  float co[6], few[4], cap_in = 0.0f;
  if (FEAT == 2) {
    constexpr float fit[6] = {1.0f, -0.333302796f, 0.132884905f, -0.0517682843f, 0.0169064086f, -0.00312657771f};
    constexpr float near[4] = {1.0f, -0.33328161f, 0.1320536f, -0.04475063f};
    const float in = P.scale / P.softcap, in2 = in * in;
    cap_in = in2 < 1e6f ? fabsf(P.softcap / P.scale) : -1.0f;   // (beyond, powers of in2 leave fp32's range)
    float power = sl2;
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      co[k] = fit[k] * power;
      if (k < 4) few[k] = near[k] * power;
      power *= in2;
    }
  }
  ItemReader items;
  Item it;
  int s_count = 0, o_count = 0;
  for (;;) {
    if (!items.next(S, it)) return false;
    if (it.len < 0) return true;
    const Keys keys = keys_of(P, it);
    const int q0 = it.q0 + t * P.apart, row = q0 + r, head = min(it.head + (P.apart ? 0 : t), P.H_q - 1);
    const Tiles tiles = tiles_of(P, it, t);
    const float slope2 = FEAT && P.slopes ? P.slopes[head] * kLog2e : 0.0f;
    float m = -INFINITY, l = 0.0f;
    bool have = false;
    for (int i = 0; i < keys.count; ++i) {
      const int tile = tile_of(keys, i), k0 = tile * kKeys;
      if (!tiles.uses(tile)) continue;
      const bool masked = tiles.masked(tile);
      if (!wait_warp(&S.s_full[t], s_count++ & 1)) return false;
      tc_fence_after();
      uint64_t sum[2] = {0, 0};
      // KEYS keys of the tile from key `from` on, a step of the online softmax: maximum, reference, weights
      auto step = [&](auto keys_tag, int from) {
        constexpr int N = decltype(keys_tag)::value;
        uint32_t u[N], p[32];
        float* s = reinterpret_cast<float*>(u);
#pragma unroll
        for (int c = 0; c < N; c += 32) tmem_ld32(s_at + from + c, u + c);
        tc_wait_ld();
        auto move_to = [&](float top) {
          // (the output holds this tile's first half only when its product is through)
          if (from > 0 && !wait_warp(&S.half_done[t], (s_count - 1) & 1)) return false;
          if (from > 0) tc_fence_after();
          if (top != top) l = top;   // a NaN among the scores is all that is left of the row
          const float to = fmaxf(m, top), f = to == m ? 1.0f : ex2(m - to);
          m = to;
          l *= f;
          sum[0] = mul2(sum[0], pair(f, f));
          sum[1] = mul2(sum[1], pair(f, f));
          if (have || from > 0) rescale(o_at, f);
          return true;
        };
        auto publish = [&](int h) {
          tmem_st32(s_at + h * 32, p);
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&S.p_full[t][h]);
        };
        if (FEAT == 2 && !masked && slope2 == 0.0f) {
          // the cap keeps the order of scores: the largest is taken before it, and the reference leaves with the last step of f
          const float high = largest<64>(s), low = smallest(s);
          const float most = fmaxf(fabsf(high), fabsf(low));
          if (__all_sync(0xFFFFFFFFu, most <= cap_in)) {
            const float w = high * high;
            float q = fmaf(w, co[5], co[4]);
#pragma unroll
            for (int k = 3; k >= 0; --k) q = fmaf(q, w, co[k]);
            // (a negative scale turns the order round)
            const float lw = low * low;
            float lq = fmaf(lw, co[5], co[4]);
#pragma unroll
            for (int k = 3; k >= 0; --k) lq = fmaf(lq, lw, co[k]);
            const float top = fmaxf(high * q, low * lq);
            if (__any_sync(0xFFFFFFFFu, top > m + kLag) && !move_to(top)) return false;
            if (__all_sync(0xFFFFFFFFu, most <= 0.5f * cap_in)) weigh_capped<DT, 4>(s, p, sum, few, m - kLift);
            else weigh_capped<DT, 6>(s, p, sum, co, m - kLift);
            publish(from / 64);
            return true;
          }
        }
#pragma unroll
        for (int c = 0; c < N; c += 64) {
          const int k1 = k0 + from + c;
          if (FEAT) reshape<FEAT == 2>(s + c, P, slope2, row - k1, k0 + kKeys <= q0 + 1 ? 1 : k0 >= q0 + kRows - 1 ? -1 : 0);
          if (masked) {
            const int a = first_key(P, row) - k1, b = min(end_key(P, it, row), it.len) - k1, e = it.prefix - k1;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const uint32_t bits = (below(b - 32 * w) & ~below(a - 32 * w)) | below(e - 32 * w);
#pragma unroll
              for (int k = 0; k < 32; ++k) s[c + w * 32 + k] = bits >> k & 1u ? s[c + w * 32 + k] : -INFINITY;
            }
          }
        }
        const float top = largest<N>(s) * (FEAT ? 1.0f : sl2);
        if (__any_sync(0xFFFFFFFFu, !(top <= m + kLag)) && !move_to(top)) return false;
        const float ref = m == -INFINITY ? 0.0f : m - kLift;
#pragma unroll
        for (int c = 0; c < N; c += 64) {
          weigh<DT, FEAT != 0>(s + c, p, sum, sl2, ref);
          publish(from / 64 + c / 64);
        }
        return true;
      };
      if (FEAT == 2) {   // half a tile at a time: what the cap takes of registers and code
#pragma unroll 1
        for (int h = 0; h < 2; ++h)
          if (!step(std::integral_constant<int, 64>(), h * 64)) return false;
      } else {
        if (!step(std::integral_constant<int, 128>(), 0)) return false;
      }
      have = true;
      float a, b, c, d;
      split(sum[0], a, b);
      split(sum[1], c, d);
      l += (a + b) + (c + d);
    }
    if (have) {
      if (!wait_warp(&S.o_full[t], o_count++ & 1)) return false;
      tc_fence_after();
      const int64_t at = (static_cast<int64_t>(it.row0) + row) * P.H_q + head;
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      // Two lanes write 64 bytes of a row at a time, 32 each where that is aligned: one prompt of 8192 tokens 971 us with 16 bytes of 32 rows an
      // instruction, 954 with 32 bytes of 32 rows, 924 so.  The loop is not unrolled: an item's end runs once, so its code comes from far.
      const bool wide = (reinterpret_cast<uint64_t>(P.out) & 31) == 0;   // (rows are 256 bytes)
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        tmem_ld32(o_at + c * 32, o);
        tc_wait_ld();
        // two lanes write 64 bytes of the even one's row, then of the odd one's
        uint32_t w[2][8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t a = round2<DT>(__uint_as_float(o[k * 2]) * inv, __uint_as_float(o[k * 2 + 1]) * inv);
          const uint32_t b = round2<DT>(__uint_as_float(o[k * 2 + 16]) * inv, __uint_as_float(o[k * 2 + 17]) * inv);
          const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, lane & 1 ? a : b, 1);
          w[0][k] = lane & 1 ? other : a;
          w[1][k] = lane & 1 ? b : other;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if ((row & ~1) + e >= it.len) continue;
          uint4* out = reinterpret_cast<uint4*>(P.out + (at + (e - (lane & 1)) * P.H_q) * JF_HEAD_DIM + c * 32 + (lane & 1) * 16);
          if (wide) {
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), JF_W8(w[e], 0) : "memory");
          } else {
            out[0] = make_uint4(w[e][0], w[e][1], w[e][2], w[e][3]);
            out[1] = make_uint4(w[e][4], w[e][5], w[e][6], w[e][7]);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      if (S.bad[items.slot] && row < it.len) give_back<DT>(P, it, row, P.out + at * JF_HEAD_DIM);
      __syncwarp();
      if (row < it.len && P.lse) P.lse[at] = l > 0.0f || l != l ? (m - kLift + __log2f(l)) * kLn2 : -INFINITY;
    }
    items.release_warp(S);
  }
}

template <int DT, int FEAT>
__global__ void __launch_bounds__(kThreads, 1)
varlen_attn_kernel(const __grid_constant__ Params P, const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap km,
                   const __grid_constant__ CUtensorMap vm) {
  extern __shared__ unsigned char raw[];
  __shared__ Shared S;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);   // (known to be the same for all lanes)
  unsigned char* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t q_smem = smem_u32(smem), kv_smem = q_smem + 2 * kTileBytes;
  if (threadIdx.x == 0) {
    mbar_init(&S.q_full, 1);
    mbar_init(&S.q_empty, 1);
    mbar_init(&S.products_done, 1);
    for (int i = 0; i < kKvStages; ++i) { mbar_init(&S.kv_full[i], 1); mbar_init(&S.kv_empty[i], 2); }   // empty: products done, looked over
    for (int t = 0; t < 2; ++t) { mbar_init(&S.s_full[t], 1); mbar_init(&S.p_full[t][0], 4); mbar_init(&S.p_full[t][1], 4); mbar_init(&S.half_done[t], 1); mbar_init(&S.o_full[t], 1); }
    for (int i = 0; i < kItems; ++i) { mbar_init(&S.item_full[i], 1); mbar_init(&S.item_empty[i], 11); }   // 8 + loads, products, cleaning
    for (int i = 0; i < kClean; ++i) mbar_init(&S.cleaned[i], 1);
    fence_barrier_init();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&S.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  pdl_wait();
  pdl_trigger();
  // every role ends by itself, a wait that ran out included, loads and products when theirs are through; the error is recorded by whoever
  // meets it
  bool ok = true;
  if (warp >= 8) {
    regs_dec<kRoleRegs>();
    if (warp == 8) {
      int loaded = 0;
      Ring ring;
      ok = load(P, S, q_smem, kv_smem, &qm, &km, &vm, loaded, ring);
      ok &= arrived(S, loaded, ring);
    } else if (warp == 9) {
      ok = multiply<DT>(P, S, q_smem, kv_smem, tmem);
      if (elect_one()) tc_commit(&S.products_done);
      __syncwarp();
      ok &= wait_warp(&S.products_done, 0);
    } else if (warp == 10) {
      ok = schedule(P, S);
    } else {
      ok = clean_values<DT>(P, S, smem + 2 * kTileBytes);
    }
  } else {
    regs_inc<kRowRegs>();
    ok = soften<DT, FEAT>(P, S, tmem, warp >> 2);
  }
  if (!ok) report_status(P.status, JF_ERR_TIMEOUT);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---- host -----------------------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qr) != cudaSuccess || qr != cudaDriverEntryPointSuccess)
      sym = nullptr;
    return reinterpret_cast<EncodeFn>(sym);
  }();
  return fn;
}

// (rows, heads, 128) as boxes of 128 rows of one head, 64 channels wide; rows past the end read as zeros.
jf_status_t rows_map(const void* base, int dtype, int64_t T, int32_t H, int64_t stride_t, int64_t stride_h, CUtensorMap* out) {
  EncodeFn fn = encode_fn();
  if (!fn) return JF_ERR_CUDA;
  const cuuint64_t dims[3] = {JF_HEAD_DIM, static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(T)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(H > 1 ? stride_h : JF_HEAD_DIM) * 2,
                                 static_cast<cuuint64_t>(T > 1 ? stride_t : JF_HEAD_DIM) * 2};
  const cuuint32_t box[3] = {64, 1, 128}, estr[3] = {1, 1, 1};
  const CUresult r = fn(out, dtype == JF_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { g_last_cuda_error = static_cast<int32_t>(r); return JF_ERR_CUDA; }
  return JF_OK;
}

template <int DT, int FEAT>
jf_status_t launch(const Params& P, int grid, cudaStream_t s, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v) {
  auto* kernel = varlen_attn_kernel<DT, FEAT>;
  static const int regs = [] {
    cudaFuncAttributes f{};
    return cudaFuncGetAttributes(&f, varlen_attn_kernel<DT, FEAT>) == cudaSuccess ? f.numRegs : 0;
  }();
  // (a warpgroup that asks for more than the block has waits for good)
  if (regs * kThreads < 256 * kRowRegs + 128 * kRoleRegs) return JF_ERR_UNSUPPORTED;
  JF_ENSURE_SMEM(kernel, kSmemBytes);
  JF_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(kThreads), kSmemBytes, s, P, q, k, v));
  return JF_OK;
}

// Where the calls that bring no record of their own note a wait that ran out, one a device: host memory that the kernel writes, so that
// looking at it takes no copy and no wait.  Never freed: captured graphs hold its address.
struct Record { void *host, *device; };
constexpr int kDevices = 64;
std::mutex g_record_mu;
Record g_records[kDevices];

jf_status_t record_of(int device, bool make, Record& r) {
  if (device < 0 || device >= kDevices) return JF_ERR_ARG;
  std::lock_guard<std::mutex> lock(g_record_mu);
  if (!g_records[device].host && make) {
    // (a capture that is under way, on any stream, does not mind: nothing of it depends on this)
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    JF_CUDA_TRY(cudaThreadExchangeStreamCaptureMode(&mode));
    Record made{};
    const jf_status_t st = jf_alloc_mapped(256, &made.host, &made.device);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (st != JF_OK) return st;
    memset(made.host, 0, 256);
    g_records[device] = made;
  }
  r = g_records[device];
  return JF_OK;
}
// An error that is there is taken: it is reported once.
jf_status_t taken(const Record& r) {
  if (!r.host) return JF_OK;
  const jf_status_t st = jf_decode_status_of_copy(r.host);
  if (st != JF_OK) memset(r.host, 0, JF_STATUS_RECORD_BYTES);
  return st;
}

}  // namespace

jf_status_t wait_record(cudaStream_t s, int32_t** device) {
  int index = 0;
  JF_CUDA_TRY(cudaGetDevice(&index));
  Record own{};
  jf_status_t e = record_of(index, true, own);
  if (e != JF_OK) return e;
  *device = static_cast<int32_t*>(own.device);
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  JF_CUDA_TRY(cudaStreamIsCapturing(s, &capture));
  return capture == cudaStreamCaptureStatusNone ? taken(own) : JF_OK;
}

}  // namespace jf

extern "C" jf_status_t jf_varlen_record(int32_t device, void** host) {
  using namespace jf;
  if (!host) return JF_ERR_ARG;
  Record r{};
  const jf_status_t st = record_of(device, true, r);
  *host = r.host;
  return st;
}

extern "C" jf_status_t jf_varlen_status(int32_t device) {
  using namespace jf;
  Record r{};
  const jf_status_t st = record_of(device, false, r);
  return st == JF_OK ? taken(r) : st;
}

extern "C" jf_status_t jf_varlen_attn(const jf_varlen_attn_args* a, jf_stream_t stream) {
  using namespace jf;
  if (!a) return JF_ERR_ARG;
  if (a->dtype != JF_DTYPE_BF16 && a->dtype != JF_DTYPE_FP16) return JF_ERR_ARG;
  if (a->T < 0 || a->n_seqs < 0 || a->H_q <= 0 || a->H_kv <= 0 || a->H_q % a->H_kv != 0 || a->window < 0) return JF_ERR_ARG;
  if (a->softcap != 0.0f && !(a->softcap >= 1.0e-30f && a->softcap <= 1.0e30f)) return JF_ERR_ARG;
  if (a->T > kMaxRows || a->n_seqs > kMaxSeqs) return JF_ERR_UNSUPPORTED;
  if (a->T == 0 || a->n_seqs == 0) return JF_OK;
  if (!a->q || !a->k || !a->v || !a->cu_seqlens || !a->out) return JF_ERR_ARG;
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->out, 16) || !aligned(a->status_record, 8)) return JF_ERR_ARG;
  auto stride_ok = [](int64_t size, int64_t stride) { return size == 1 || (stride > 0 && stride % 8 == 0 && stride < (1ll << 38)); };
  if (!stride_ok(a->T, a->q_stride_t) || !stride_ok(a->H_q, a->q_stride_h) || !stride_ok(a->T, a->k_stride_t) || !stride_ok(a->H_kv, a->k_stride_h) ||
      !stride_ok(a->T, a->v_stride_t) || !stride_ok(a->H_kv, a->v_stride_h))
    return JF_ERR_ARG;
  const auto s = static_cast<cudaStream_t>(stream);
  auto* status = static_cast<int32_t*>(a->status_record);
  if (!status) {
    const jf_status_t e = wait_record(s, &status);
    if (e != JF_OK) return e;
  }
  CUtensorMap q, k, v;
  jf_status_t st = rows_map(a->q, a->dtype, a->T, a->H_q, a->q_stride_t, a->q_stride_h, &q);
  if (st == JF_OK) st = rows_map(a->k, a->dtype, a->T, a->H_kv, a->k_stride_t, a->k_stride_h, &k);
  if (st == JF_OK) st = rows_map(a->v, a->dtype, a->T, a->H_kv, a->v_stride_t, a->v_stride_h, &v);
  if (st != JF_OK) return st;
  Params P{};
  P.cu = a->cu_seqlens;
  P.prefix = a->prefix_lens;
  P.slopes = a->alibi_slopes;
  P.v = static_cast<const uint16_t*>(a->v);
  P.out = static_cast<uint16_t*>(a->out);
  P.lse = a->lse;
  P.status = status;
  P.v_stride_t = a->v_stride_t;
  P.v_stride_h = a->v_stride_h;
  P.T = static_cast<int32_t>(a->T);
  P.n_seqs = a->n_seqs;
  P.H_q = a->H_q;
  // Two heads with the same keys rather than 256 rows of one: the two tiles of an item then have the same keys to go through, and a
  // sequence that ends within 128 rows of its last item leaves neither without work.
  P.G = a->H_q / a->H_kv;
  P.apart = P.G > 1 ? 0 : kRows;
  P.span = kRows + P.apart;
  P.units = P.G > 1 ? a->H_kv * ((P.G + 1) / 2) : a->H_q;
  P.H_kv = a->H_kv;
  P.window = a->window;
  P.scale = a->attn_scale;
  P.softcap = a->softcap;
  P.causal = a->causal != 0;
  const int64_t most = (a->T / P.span + std::min<int64_t>(a->n_seqs, a->T)) * P.units;   // work items
  const int grid = static_cast<int>(std::min<int64_t>(num_sms(), most));
  // (the plain form takes the maximum before it scales, so it needs a positive scale)
  const int feat = a->softcap > 0.0f ? 2 : a->alibi_slopes || !(a->attn_scale > 0.0f) ? 1 : 0;
  if (a->dtype == JF_DTYPE_BF16)
    return feat == 0 ? launch<JF_DTYPE_BF16, 0>(P, grid, s, q, k, v) : feat == 1 ? launch<JF_DTYPE_BF16, 1>(P, grid, s, q, k, v)
                                                                            : launch<JF_DTYPE_BF16, 2>(P, grid, s, q, k, v);
  return feat == 0 ? launch<JF_DTYPE_FP16, 0>(P, grid, s, q, k, v) : feat == 1 ? launch<JF_DTYPE_FP16, 1>(P, grid, s, q, k, v)
                                                                          : launch<JF_DTYPE_FP16, 2>(P, grid, s, q, k, v);
}
