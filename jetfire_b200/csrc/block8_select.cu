// Which blocks of the 8-bit cache a query attends to: the best by a cheap score, and the first and last of the sequence.
//
//   score_j = max_h qs_h * sum_c (min(q8_hc, 0) lo_jc + max(q8_hc, 0) hi_jc) * unit_j,   q8_h = rint(q_h / qs_h), qs_h = amax|q_h| / 127
//
// is an upper bound of q.k over block j, but for the query's rounding: lo and hi are the lowest and highest code of channel c in the
// block (block bounds, kept by the append), unit_j what a code of 1 stands for, h runs through the query heads of
// the KV head.  The sum is one integer product of 256 channels, exact, on the tensor cores (mma.s8: 16 blocks x 8
// heads); it and the two factors that follow, in fp32, have one value whatever the order, so the choice is the same on every run
// and in every plain form.  Ties go to the lower block.
//
// One kernel scores, 16 blocks a warp at a time, and leaves the scores as integers ordered like them; a second one, a block a row, brings a row's
// integers to shared memory and finds the limit above which blocks are chosen: histograms of 2048 bins over the range it must lie in, until one
// value is left or all that are left are taken.  A warp goes through a stretch of the row, so the list comes out in rising order by
// counting votes, and what reads it adds up in the same order always.
//
// Bound: the scores by memory (260 bytes a block and KV head, 256 of them in one piece): 4 x 4096 blocks, 8 KV heads, 34 MB, 11.9 us from cold caches =
// 2.9 TB/s, three dependent trips and two or four tiles a warp.  The choice by latency: a row of 4096 scores 4 us with warm caches (loads 0.7, the limit 1.7,
// the list 1.9).  With the attention over 128 of 4096 blocks of four sequences the call takes 25 us back to back, over all of them
// jf_block8_attn takes 101.  (Both in one kernel, a cluster a row with histograms over distributed shared memory: 31.)
#include "block8.cuh"

#include <algorithm>
#include <type_traits>

namespace jf {
namespace {

constexpr int kScoreWarps = 8, kTile = 16;        // blocks of a warp's tile
constexpr int kWarps = 16, kThreads = kWarps * 32; // of the choosing kernel
// Scoring blocks of a multiprocessor: warps take more tiles rather than that there are several waves.  (Four sequences of 4096 blocks, the whole call: 2 26 us, 3
// 25, 4, which leaves 64 registers, 30; a tile a warp and four waves 27.)
constexpr int kScoreBlocks = 3;
constexpr int kBins = 2048;
constexpr int kMaxBlocks = 1 << 18;
constexpr int kMaxKeys = 49152;                   // of a row in shared memory; longer rows are read from where they are
constexpr uint32_t kForced = 0xFFFFFFFFu;         // first and last blocks
constexpr uint32_t kNothing = 0x007FFFFFu;        // the key of -inf
constexpr float kSmallest = 0x1p-100f;

struct SelectParams {
  const uint16_t* q;
  const float* k_scales;
  const int8_t* bounds;
  const void* table;
  const int32_t* seq_lens;
  uint32_t* keys;                                 // (B, H_kv, row_keys)
  int32_t* chosen;
  int64_t num_blocks, bt_stride, row_keys;
  int32_t H_q, H_kv, G, max_len, top, first, last, tiles;   // tiles: of a scoring warp (0: nothing is scored)
  float unit;
  bool bt_i32;
};

struct Queries {
  alignas(16) int8_t q8[8][272];                  // min(q, 0), max(q, 0); rows on different banks
  float step[8];
};

// Four elements of the warp's query head, of eight heads from h0 on.
__device__ __forceinline__ uint2 load_query(const SelectParams& P, int64_t row0, int h0) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp >= 8 || h0 + warp >= P.G) return make_uint2(0, 0);
  return *reinterpret_cast<const uint2*>(P.q + (row0 + h0 + warp) * JF_HEAD_DIM + lane * 4);
}
// They in 8 bits.  A head with an element that is no number scores nothing, as one beyond the group.
template <int DT> __device__ __forceinline__ void round_queries(const SelectParams& P, Queries& S, uint2 w, int h0) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, amax = 0.0f;
  bool odd = h0 + warp >= P.G;
  if (!odd) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = Elem<DT>::to_f32(static_cast<uint16_t>((k < 2 ? w.x : w.y) >> 16 * (k & 1)));
      odd |= !(fabsf(x[k]) < __int_as_float(0x7F800000));
      amax = fmaxf(amax, fabsf(x[k]));
    }
  }
  amax = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(amax)));
  odd = __any_sync(0xFFFFFFFFu, odd);
  const float step = __fdiv_rn(fmaxf(amax, kSmallest), 127.0f);
  uint32_t neg = 0, pos = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int v = odd ? 0 : __float2int_rn(__fdiv_rn(x[k], step));
    neg |= (static_cast<uint32_t>(min(v, 0)) & 255u) << 8 * k;
    pos |= (static_cast<uint32_t>(max(v, 0)) & 255u) << 8 * k;
  }
  *reinterpret_cast<uint32_t*>(&S.q8[warp][lane * 4]) = neg;
  *reinterpret_cast<uint32_t*>(&S.q8[warp][128 + lane * 4]) = pos;
  if (lane == 0) S.step[warp] = odd ? __int_as_float(0x7FC00000) : step;
}

template <int DT>
__global__ void __launch_bounds__(kScoreWarps * 32, kScoreBlocks) block8_score_kernel(const __grid_constant__ SelectParams P) {
  __shared__ Queries S;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, b = blockIdx.z;
  pdl_wait();
  pdl_trigger();
  const int64_t row0 = static_cast<int64_t>(b) * P.H_q + kvh * P.G;
  uint2 query = load_query(P, row0, 0);   // (on its way beside the length)
  const int len = max(0, min(P.seq_lens[b], P.max_len)), n = (len + JF_BLOCK_SIZE - 1) / JF_BLOCK_SIZE;
  const int begin = static_cast<int>(blockIdx.x) * (kScoreWarps * kTile) * P.tiles;
  if (n <= P.top || begin >= n) return;
  const int end = min(begin + kScoreWarps * kTile * P.tiles, n);
  uint32_t* keys = P.keys + (static_cast<int64_t>(b) * P.H_kv + kvh) * P.row_keys;
  const int64_t head_row = static_cast<int64_t>(kvh) * P.num_blocks, table_row = static_cast<int64_t>(b) * P.bt_stride;
  // blocks' ids are looked up a tile ahead
  int64_t ids[2];
  auto look_up = [&](int at) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int j = at + g + 8 * r;
      ids[r] = -1;
      if (j < end) ids[r] = P.bt_i32 ? static_cast<const int32_t*>(P.table)[table_row + j] : static_cast<const int64_t*>(P.table)[table_row + j];
    }
  };
  for (int h0 = 0; h0 < P.G; h0 += 8) {
    look_up(begin + warp * kTile);
    if (h0 > 0) {
      query = load_query(P, row0, h0);
      __syncthreads();
    }
    round_queries<DT>(P, S, query, h0);
    __syncthreads();
    uint4 q[4];       // head g, 16 of its 256 products' channels t * 16 .., 64 + t * 16 .., ...
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const uint4*>(&S.q8[g][(t + 4 * i) * 16]);
    const float step0 = S.step[2 * t], step1 = S.step[2 * t + 1];
    for (int at = begin + warp * kTile; at < end; at += kScoreWarps * kTile) {
      uint4 x[2][4];
      float unit[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int64_t id = ids[r];
        const bool is = id >= 0 && id < P.num_blocks;
        unit[r] = is ? P.k_scales[head_row + id] : __int_as_float(0x7FC00000);
        const uint4* from = reinterpret_cast<const uint4*>(P.bounds + (head_row + (is ? id : 0)) * (2 * JF_HEAD_DIM)) + t;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[r][i] = is ? __ldg(from + 4 * i) : make_uint4(0, 0, 0, 0);
      }
      look_up(at + kScoreWarps * kTile);
      int d[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mma_s8_16832(d, x[0][i].x, x[1][i].x, x[0][i].y, x[1][i].y, q[i].x, q[i].y);
        mma_s8_16832(d, x[0][i].z, x[1][i].z, x[0][i].w, x[1][i].w, q[i].z, q[i].w);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        // (the largest number: what is none does not count)
        float best = fmaxf(fmaxf(-INFINITY, __fmul_rn(static_cast<float>(d[2 * r]), step0)), __fmul_rn(static_cast<float>(d[2 * r + 1]), step1));
        best = fmaxf(best, __shfl_xor_sync(0xFFFFFFFFu, best, 1));
        best = fmaxf(best, __shfl_xor_sync(0xFFFFFFFFu, best, 2));
        const float score = __fmul_rn(best, __fmul_rn(unit[r], P.unit));
        const int j = at + g + 8 * r;
        if (t == 0 && j < end) {
          uint32_t key = score != score ? kNothing : float_order_key(score);
          if (h0 > 0) key = max(key, keys[j]);
          keys[j] = j < P.first || j >= n - P.last ? kForced : key;
        }
      }
    }
  }
}

struct Choice {
  uint32_t count[kBins];
  uint32_t lo, hi;
  int scan[kWarps], scan2[kWarps], bin, over, in;
};

// Staged: the row's keys stand in shared memory.
template <bool STAGED>
__global__ void __launch_bounds__(kThreads) block8_choose_kernel(const __grid_constant__ SelectParams P) {
  extern __shared__ __align__(16) uint32_t staged[];
  __shared__ Choice S;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.y) * P.H_kv + blockIdx.x;
  if (threadIdx.x == 0) { S.lo = 0xFFFFFFFFu; S.hi = 0; }
  // (behind the scoring kernel, which has waited for whatever wrote the lengths, they are read ahead of the wait)
  if (P.tiles == 0) pdl_wait();
  const int len = max(0, min(P.seq_lens[blockIdx.y], P.max_len)), n = (len + JF_BLOCK_SIZE - 1) / JF_BLOCK_SIZE;
  if (P.tiles > 0) pdl_wait();
  pdl_trigger();
  int32_t* chosen = P.chosen + row * P.top;
  if (n <= P.top) {   // all of them
    for (int i = threadIdx.x; i < P.top; i += kThreads) chosen[i] = i < n ? i : -1;
    return;
  }
  const uint32_t* global = P.keys + row * P.row_keys;
  const uint32_t* keys = STAGED ? staged : global;
  __syncthreads();
  uint32_t lo = 0xFFFFFFFFu, hi = 0;   // least and largest key but the forced ones and -inf
  auto look_at = [&](uint32_t k) {
    if (k == kForced || k <= kNothing) return;
    lo = min(lo, k);
    hi = max(hi, k);
  };
  // (rows begin on multiples of 16 bytes)
#pragma unroll 2
  for (int i = threadIdx.x; i < n / 4; i += kThreads) {
    const uint4 k = *reinterpret_cast<const uint4*>(global + i * 4);
    if (STAGED) *reinterpret_cast<uint4*>(staged + i * 4) = k;
    look_at(k.x); look_at(k.y); look_at(k.z); look_at(k.w);
  }
  if (threadIdx.x < n % 4) {
    const uint32_t k = global[n / 4 * 4 + threadIdx.x];
    if (STAGED) staged[n / 4 * 4 + threadIdx.x] = k;
    look_at(k);
  }
  lo = __reduce_min_sync(0xFFFFFFFFu, lo);
  hi = __reduce_max_sync(0xFFFFFFFFu, hi);
  if (lane == 0 && lo <= hi) {
    atomicMin(&S.lo, lo);
    atomicMax(&S.hi, hi);
  }
  __syncthreads();
  lo = S.lo;
  hi = S.hi;
  // ---- the limit: of the keys in [from, above] the highest `need` are taken, those beyond `above` too
  int need = P.top - P.first - P.last;
  uint32_t from = lo, above = hi;
  auto none_left = [&] { from = above = kNothing; };   // what scores nothing, the first of it
  if (need == 0) from = above = kForced - 1;           // (no key is that)
  else if (lo > hi) none_left();
  else
    for (;;) {
      int shift = 0;
      while ((above - from) >> shift >= kBins) ++shift;
      constexpr int kEach = kBins / kThreads;
#pragma unroll
      for (int i = 0; i < kEach; ++i) S.count[threadIdx.x + i * kThreads] = 0;
      if (threadIdx.x == 0) S.bin = -1;
      __syncthreads();
#pragma unroll 4
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t k = keys[i];
        if (k >= from && k <= above) atomicAdd(&S.count[(k - from) >> shift], 1u);
      }
      __syncthreads();
      // a thread's bins, the highest of all first
      int c[kEach], sum = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        c[i] = static_cast<int>(S.count[kBins - 1 - (threadIdx.x * kEach + i)]);
        sum += c[i];
      }
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) S.scan[warp] = upto;
      __syncthreads();
      int total = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int v = S.scan[w];
        if (w < warp) upto += v;
        total += v;
      }
      int before = upto - sum;
      if (before < need && upto >= need) {   // one thread: the bin is among its own
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (before < need && before + c[i] >= need) {
            S.bin = kBins - 1 - static_cast<int>(threadIdx.x * kEach + i);
            S.over = before;
            S.in = c[i];
          }
          before += c[i];
        }
      }
      __syncthreads();
      if (S.bin < 0) {   // fewer scores than are needed (in the first round only): they are taken, and of the rest the first
        need -= total;
        none_left();
        break;
      }
      need -= S.over;
      from += static_cast<uint32_t>(S.bin) << shift;
      above = min(above, from + ((1u << shift) - 1u));
      if (S.in == need || shift == 0) break;
      __syncthreads();   // everybody has read the bin
    }
  // ---- the list: keys beyond `above`, and the first `need` of those in [from, above] (all of them, or of one value).  A warp has a stretch of the row.
  const int stretch = (n + kWarps * 32 - 1) / (kWarps * 32) * 32, k0 = min(warp * stretch, n), k1 = min(k0 + stretch, n);
  int over = 0, ties = 0;
#pragma unroll 4
  for (int i = k0; i < k1; i += 32) {
    const uint32_t k = i + lane < k1 ? keys[i + lane] : 0u;
    over += __popc(__ballot_sync(0xFFFFFFFFu, k > above));
    ties += __popc(__ballot_sync(0xFFFFFFFFu, k >= from && k <= above));
  }
  __syncthreads();
  if (lane == 0) { S.scan[warp] = over; S.scan2[warp] = ties; }
  __syncthreads();
  int at = 0, number = 0;   // places of the list, candidates before this warp's
#pragma unroll
  for (int w = 0; w < kWarps; ++w)
    if (w < warp) {
      at += S.scan[w];
      number += S.scan2[w];
    }
  at += min(number, need);
  const uint32_t below = (1u << lane) - 1u;
#pragma unroll 4
  for (int i = k0; i < k1; i += 32) {
    const uint32_t k = i + lane < k1 ? keys[i + lane] : 0u;
    const bool tie = k >= from && k <= above;
    const unsigned tied = __ballot_sync(0xFFFFFFFFu, tie);
    const bool take = k > above || (tie && number + __popc(tied & below) < need);
    const unsigned taken = __ballot_sync(0xFFFFFFFFu, take);
    if (take) chosen[at + __popc(taken & below)] = i + lane;
    at += __popc(taken);
    number += __popc(tied);
  }
}

int64_t row_keys_of(int64_t longest) { return (longest + JF_BLOCK_SIZE * 4 - 1) / (JF_BLOCK_SIZE * 4) * 4; }
uint64_t attn_part(int B, int H_q, int H_kv, int max_S, int top) {
  return (block8_attn_workspace(B, H_q, H_kv, static_cast<int>(std::min<int64_t>(max_S, int64_t{top} * JF_BLOCK_SIZE))) + 255) / 256 * 256;
}

}  // namespace
}  // namespace jf

extern "C" uint64_t jf_block8_sparse_workspace_bytes(int32_t B, int32_t H_q, int32_t H_kv, int32_t max_S, int32_t top_blocks) {
  if (top_blocks <= 0) return 0;
  const uint64_t attn = jf::attn_part(B, H_q, H_kv, max_S, top_blocks);
  return attn ? attn + static_cast<uint64_t>(B) * H_kv * jf::row_keys_of(max_S) * sizeof(uint32_t) : 0;
}

extern "C" jf_status_t jf_block8_sparse_attn(const jf_block8_sparse_args* a, jf_stream_t stream) {
  using namespace jf;
  if (!a) return JF_ERR_ARG;
  const jf_block8_attn_args& at = a->attn;
  if (a->top_blocks <= 0 || a->first_blocks < 0 || a->last_blocks < 1 || int64_t{a->first_blocks} + a->last_blocks > a->top_blocks) return JF_ERR_ARG;
  if (at.window != 0 || at.prefix_lens || at.alibi_slopes || !(at.attn_scale > 0.0f)) return JF_ERR_ARG;
  if (at.B > 0 && (!a->chosen || !aligned(a->chosen, 4) || !aligned(a->bounds, 16) || (at.num_blocks > 0 && !a->bounds))) return JF_ERR_ARG;
  Block8Source from;
  from.chosen = a->chosen;
  from.top = a->top_blocks;
  const jf_status_t checked = block8_attend(&at, from, stream, false);
  if (checked != JF_OK || at.B == 0) return checked;
  const int64_t longest = std::min<int64_t>(at.max_S, int64_t{at.max_blocks} * JF_BLOCK_SIZE), blocks = (longest + JF_BLOCK_SIZE - 1) / JF_BLOCK_SIZE;
  if (blocks > kMaxBlocks) return JF_ERR_UNSUPPORTED;
  if (at.workspace_bytes < jf_block8_sparse_workspace_bytes(at.B, at.H_q, at.H_kv, at.max_S, a->top_blocks)) return JF_ERR_WORKSPACE;
  SelectParams P{};
  P.q = static_cast<const uint16_t*>(at.q);
  P.k_scales = at.k_scales;
  P.bounds = a->bounds;
  P.table = at.block_table;
  P.seq_lens = at.seq_lens;
  P.keys = reinterpret_cast<uint32_t*>(static_cast<char*>(at.workspace) + attn_part(at.B, at.H_q, at.H_kv, at.max_S, a->top_blocks));
  P.chosen = a->chosen;
  P.num_blocks = at.num_blocks;
  P.bt_stride = at.bt_stride;
  P.row_keys = row_keys_of(at.max_S);
  P.H_q = at.H_q; P.H_kv = at.H_kv; P.G = at.H_q / at.H_kv;
  P.max_len = static_cast<int32_t>(longest);
  P.top = a->top_blocks; P.first = a->first_blocks; P.last = a->last_blocks;
  P.unit = at.codes == JF_CODES_INT8 ? 1.0f : 448.0f / 127.0f;
  P.bt_i32 = at.bt_is_i32 != 0;
  const auto s = static_cast<cudaStream_t>(stream);
  if (blocks > a->top_blocks) {   // (else there is nothing to choose)
    const int64_t tiles = (blocks + kScoreWarps * kTile - 1) / (kScoreWarps * kTile) * at.B * at.H_kv;
    P.tiles = static_cast<int>(std::min<int64_t>((tiles + kScoreBlocks * num_sms() - 1) / (kScoreBlocks * num_sms()), 16));
    const int each = kScoreWarps * kTile * P.tiles;
    const dim3 grid(static_cast<unsigned>((blocks + each - 1) / each), at.H_kv, at.B), block(kScoreWarps * 32);
    JF_CUDA_TRY(at.q_dtype == JF_DTYPE_BF16 ? launch_pdl(block8_score_kernel<JF_DTYPE_BF16>, grid, block, 0, s, P)
                                            : launch_pdl(block8_score_kernel<JF_DTYPE_FP16>, grid, block, 0, s, P));
  }
  const dim3 rows(at.H_kv, at.B), block(kThreads);
  if (blocks <= kMaxKeys) {
    auto* kernel = block8_choose_kernel<true>;
    JF_ENSURE_SMEM(kernel, kMaxKeys * 4);
    JF_CUDA_TRY(launch_pdl(kernel, rows, block, blocks > a->top_blocks ? static_cast<size_t>(blocks + 3) / 4 * 16 : 0, s, P));
  } else {
    JF_CUDA_TRY(launch_pdl(block8_choose_kernel<false>, rows, block, 0, s, P));
  }
  return block8_attend(&at, from, stream, true);
}
