// Decode attention over the cache of 8-bit codes with one scale per block of 16 positions and KV head.
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(f(attn_scale * q.k_j) + bias_j)
//
// Both products run on the tensor cores, the scales stay outside of them, in fp32.  int8 scores are exact integer sums: q of a
// head is a number of 22 bits below a power of two, cut into three signed bytes, and each meets the codes as they lie
// in memory (no conversion; what the 22 bits round is 2^-22 of the head's largest element).  e4m3 codes are converted to fp16, which
// holds them exactly, and meet q as fp16 numbers under a power of two per head that brings its largest element to [2^13,
// 2^14): what that rounds is 2^-38 of it.  V's codes become fp16 in either case.  The tile of a product is one block: scores as K (16
// positions) x q^T (8 heads of the group, NT times), outputs as V^T (8 x 16 channels) x p^T.  Channels and positions are
// contracted in whatever order the lanes hold them, so each lane takes 16-byte pieces of the rows as they lie in memory
// and turns them into operands in its own registers: no transposition.
//
// A warp goes through its blocks with a running reference m for every head, the sum of its weights and the output
// unnormalised.  The V scale of a block joins the exponent: w = exp2(s + log2(vs) - m) is what meets the codes, in
// fp16 (rounded to 11 bits: relative 2^-11 per weight at most, unbiased), and exp2(s - m) in fp32 what the sum gets (w / vs would
// be 1 to 2 % faster, but where scales are far apart w is 0 for positions that count).  m may lag the
// maximum by up to kLag, so that most blocks need one vote and no reduction.
//
// Work: the blocks of every sequence are cut into pieces of one length for the whole batch, chosen on the device from the lengths
// so that the pieces of a KV head fill about one wave; the pieces' partial results meet in a second kernel.  A
// sequence of one piece is written by the first kernel itself.  Short sequences are cut into as many pieces as a cluster has blocks,
// whose results meet in its shared memory.
//
// Bound: memory, 256 bytes per (position, KV head).  Four sequences of 65536 positions, 64 / 8 heads, int8: 101 us = 5.3 TB/s (copies of the
// same blocks without arithmetic, in an earlier cut of the work, 102; a plain copy runs at 6.5 TB/s); short ones by their dependent trips to memory: 6.2 us.
#include "block8.cuh"

#include <algorithm>
#include <type_traits>

namespace jf {
namespace {

constexpr int kWarps = 8;
constexpr int kStages = 3;                    // blocks of K and V in flight per warp
constexpr int kStageBytes = 2 * JF_BLOCK_SIZE * JF_HEAD_DIM;
// The reference of the fp16 weights lies 2^kLift below the maximum it was taken from and may lag the present one by
// 2^kLag: weights stay below 2^15, and what fp16 flushes to zero is below 2^-33 of the largest (a long row's many small weights add up;
// 2^-17 where the sum has moved the reference, see kFull).
constexpr float kLift = 9.0f, kLag = 6.0f;
constexpr float kNone = -3.0e38f;             // the reference of a row that has seen nothing (finite: differences are numbers)
// The sum counts in units of the weights, the reference follows weights times V scales: over blocks of zeros, whose scale is 2^-107 or
// 2^-108, a position adds 2^116.  A lane's sum beyond kFull moves the reference up by kDrop, so little that fp16 still holds the
// weights (two moves last a warp for 2^17 blocks); a warp's sum leaves below kLeave, so that those of all warps and pieces add up.
constexpr float kFull = 0x1p118f, kDrop = 8.0f, kLeave = 0x1p100f, kDown = 64.0f;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  const void* q;
  const uint8_t *k_data, *v_data;
  const float *k_scales, *v_scales;
  const void* table;
  const int32_t *seq_lens, *prefix_lens;
  const float* slopes;
  void* out;
  float* lse;
  float *part_o, *part_ml;      // [piece][kv head, group of heads][8 * NT][128] and [..][2]
  int64_t num_blocks, bt_stride;
  int32_t B, H_q, H_kv, G, groups, max_S, max_blocks, window, target, min_piece, pieces;
  float scale, softcap;
  int32_t cluster;              // blocks that share a sequence, 1 where pieces are looked for
  const int32_t* chosen;        // the blocks to be scanned, (B, H_kv, top), or null: all
  const void* shared;           // the table of the first shared_blocks blocks of every sequence; the sequence's own follow (max_blocks counts both)
  int32_t top, shared_blocks;
  int32_t behind;               // positions before those of the table, whose partial results are elsewhere
  bool bt_i32, one_wave, shared_i32, partial;   // partial: no piece is written out by itself
};

// The root of the factor that takes an output to a reference d above its own; a sum is multiplied by it twice.  (V scales up to 2^226 apart put d
// beyond what one factor in fp32 can be, while the sum, in units of the weights, is as large as others.)
__device__ __forceinline__ float half_step(float d) { return ex2(-0.5f * d); }

// What of a sequence is scanned: its first `head` blocks and the `count - head` blocks that end with its last position.
struct Span { int len, prefix, lo, head, first, count; };
template <bool PLAIN> __device__ __forceinline__ Span span_of(const AttnParams& P, int length, int prefix) {
  Span s;
  const int behind = PLAIN ? 0 : P.behind;
  s.len = min(max(min(length, P.max_S), behind) - behind, P.max_blocks * JF_BLOCK_SIZE);   // (a length may be any number)
  const int blocks = (s.len + JF_BLOCK_SIZE - 1) / JF_BLOCK_SIZE;
  s.prefix = s.lo = s.head = s.first = 0;
  s.count = !PLAIN && P.chosen ? min(blocks, P.top) : blocks;
  if (P.window > 0 && P.window < s.len) {
    s.lo = s.len - P.window;
    s.prefix = max(0, min(prefix, s.lo));
    s.first = s.lo / JF_BLOCK_SIZE;
    s.head = min((s.prefix + JF_BLOCK_SIZE - 1) / JF_BLOCK_SIZE, s.first);
    s.count = s.head + blocks - s.first;
  }
  return s;
}
__device__ __forceinline__ int prefix_of(const AttnParams& P, int b) { return P.window > 0 && P.prefix_lens ? P.prefix_lens[b] : 0; }
__device__ __forceinline__ int blocks_of(const AttnParams& P, int b) { return span_of<false>(P, P.seq_lens[b], prefix_of(P, b)).count; }
// Whose piece `x` is: n pieces of `piece` blocks (the last may be shorter) make up sequence b, the index-th is x.  The first
// piece of a sequence is the sum of those before it.
struct Cut { int piece, b, index, n, length, prefix; };
// Blocks per piece.  ceil(total / target) always leaves few enough pieces; a batch of at most 32 sequences (a lane holds the blocks of
// one) that is to fill one wave looks for the shortest pieces that still fit the grid: 32 sequences of very different length took
// 232 of 296 places before, and 1.4 us more.
__device__ __forceinline__ int piece_length(const AttnParams& P, int total, int mine) {
  int hi = max(P.min_piece, (total + P.target - 1) / P.target);
  if (P.one_wave) {
    const bool is = static_cast<int>(threadIdx.x & 31) < P.B;
    int lo = max(P.min_piece, (total + P.pieces - 1) / P.pieces);
    if ((hi - lo) * 8 < hi) return hi;
    while (lo < hi) {   // (more blocks a piece never make more pieces)
      const int mid = (lo + hi) / 2;
      if (__reduce_add_sync(0xFFFFFFFFu, is ? max(1, (mine + mid - 1) / mid) : 0) <= P.pieces) hi = mid;
      else lo = mid + 1;
    }
  }
  return hi;
}
// All lanes of a warp; b = -1 if there is no such piece.
template <bool PLAIN> __device__ __forceinline__ Cut find_piece(const AttnParams& P, int x) {
  const int lane = threadIdx.x & 31;
  int total = 0, length = 0, prefix = 0, mine = 0;
  auto look_at = [&](int b) {
    const bool is = b < P.B;
    length = is ? P.seq_lens[b] : 0;
    prefix = is ? prefix_of(P, b) : 0;
    mine = is ? span_of<PLAIN>(P, length, prefix).count : 0;
  };
  for (int b0 = 0; b0 < P.B; b0 += 32) {
    look_at(b0 + lane);
    total += __reduce_add_sync(0xFFFFFFFFu, mine);
  }
  Cut c{piece_length(P, total, mine), -1, 0, 0, 0, 0};
  int before = 0;
  for (int b0 = 0; b0 < P.B; b0 += 32) {
    if (P.B > 32) look_at(b0 + lane);
    const int n = b0 + lane < P.B ? max(1, (mine + c.piece - 1) / c.piece) : 0;   // an empty sequence is written by a piece too
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      if (lane >= o) sum += v;
    }
    const unsigned past = __ballot_sync(0xFFFFFFFFu, before + sum > x);
    if (past) {
      const int l = __ffs(past) - 1;
      c.b = b0 + l;
      c.n = __shfl_sync(0xFFFFFFFFu, n, l);
      c.index = x - before - (__shfl_sync(0xFFFFFFFFu, sum, l) - c.n);
      c.piece = (__shfl_sync(0xFFFFFFFFu, mine, l) + c.n - 1) / c.n;   // as many blocks in each
      c.length = __shfl_sync(0xFFFFFFFFu, length, l);
      c.prefix = __shfl_sync(0xFFFFFFFFu, prefix, l);
      return c;
    }
    before += __shfl_sync(0xFFFFFFFFu, sum, 31);
  }
  return c;
}

__device__ __forceinline__ int64_t block_id(const AttnParams& P, int64_t at) {
  return P.bt_i32 ? static_cast<const int32_t*>(P.table)[at] : static_cast<const int64_t*>(P.table)[at];
}

__device__ __forceinline__ int64_t shared_id(const AttnParams& P, int at) {
  return P.shared_i32 ? static_cast<const int32_t*>(P.shared)[at] : static_cast<const int64_t*>(P.shared)[at];
}

// The lower or upper two of four codes as fp16.  int8: `w` has its sign bits turned over, 0x6400 + u is 1024 + u.
template <int CODES> __device__ __forceinline__ uint32_t bias(uint32_t w) { return CODES == JF_CODES_INT8 ? w ^ 0x80808080u : w; }
template <int CODES, bool HIGH> __device__ __forceinline__ uint32_t widen(uint32_t w) {
  uint32_t d;
  if (CODES == JF_CODES_INT8)
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(prmt(w, 0x64646464u, HIGH ? 0x4342u : 0x4140u)), "r"(0x64806480u));
  else if (HIGH)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(d) : "r"(w));
  else
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(d) : "r"(w));
  return d;
}
// cap * tanh(x / cap) of four scores, for the whole warp the same way: up to |x| = cap by a polynomial fitted for the least
// relative error (6.6e-7), beyond it as cap - 2 cap / (e^(2x / cap) + 1).  A score that is NaN stays one either way.
__device__ __forceinline__ void soften4(float (&x)[4], float cap, float inv_cap) {
  float most = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) most = fmaxf(most, fabsf(x[k]));
  if (__all_sync(0xFFFFFFFFu, most <= cap)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float z = x[k] * inv_cap, w = z * z;
      float q = fmaf(w, -0.00312657771f, 0.0169064086f);
      q = fmaf(q, w, -0.0517682843f);
      q = fmaf(q, w, 0.132884905f);
      q = fmaf(q, w, -0.333302796f);
      x[k] = x[k] * fmaf(q, w, 1.0f);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = cap - __fdividef(2.0f * cap, ex2(min_or_nan(x[k] * inv_cap * (2.0f * kLog2e), 126.0f)) + 1.0f);
  }
}

// The blocks of a cluster share a sequence's pieces: no piece has to be looked for, and the results meet in shared memory.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t of_rank(const void* p, uint32_t rank) {   // the same place in another block's shared memory
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float4 load4_from(uint32_t at) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ float2 load2_from(uint32_t at) {
  float2 x;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(at) : "memory");
  return x;
}

// PLAIN: all blocks of the sequences' own tables, and whole results.  (Chosen blocks, a shared table and partial results as choices at run time cost 1.5 %
// of a call: 64 sequences of 1000 positions, 64 / 8 heads, 35.2 and 35.7 us.)
template <int CODES, int DT, int NT, bool FEAT, bool CLUSTER, bool PLAIN>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 2 : 1) block8_attn_kernel(const __grid_constant__ AttnParams P) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float sm_m[kWarps][8 * NT], sm_l[kWarps][8 * NT];
  __shared__ float2 sm_ml[8 * NT];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y / P.groups, grp = blockIdx.y % P.groups;
  const int first_head = kvh * P.G + grp * 8 * NT, heads = min(8 * NT, P.G - grp * 8 * NT);
  // (Behind block8_shared.cu's kernel, which has waited for what is in front of it before it lets this one start, and whose results are not
  // read here: the wait comes at the end, so that blocks may start where that kernel's have left.)
  const bool partial = !PLAIN && P.partial;
  if (!partial) pdl_wait();
  pdl_trigger();
  Cut cut{0, static_cast<int>(blockIdx.x) / P.cluster, static_cast<int>(blockIdx.x) % P.cluster, P.cluster, 0, 0};
  if (CLUSTER) {
    cut.length = P.seq_lens[cut.b];
    cut.prefix = prefix_of(P, cut.b);
  } else {
    cut = find_piece<PLAIN>(P, blockIdx.x);
    if (cut.b < 0) {
      if (partial) pdl_wait();
      return;
    }
  }
  const int b = cut.b;
  const Span span = span_of<PLAIN>(P, cut.length, cut.prefix);
  if (CLUSTER) cut.piece = (span.count + cut.n - 1) / cut.n;
  const int begin = cut.index * cut.piece, end = min(begin + cut.piece, span.count);
  // q of the lane's head (column g of each tile), and the slopes of the heads of its score columns 2t and 2t + 1
  uint4 q_raw[NT][4];
  float slope[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      q_raw[n][i] = make_uint4(0, 0, 0, 0);
      if (n * 8 + g < heads)
        q_raw[n][i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.q) +
                                                           (static_cast<int64_t>(b) * P.H_q + first_head + n * 8 + g) * JF_HEAD_DIM +
                                                           (i >> 1) * 64 + t * 16 + (i & 1) * 8));
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) slope[n][c] = FEAT && P.slopes && n * 8 + 2 * t + c < heads ? P.slopes[first_head + n * 8 + 2 * t + c] * kLog2e : 0.0f;
  }


  float o[NT][8][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[n][i][k] = 0.0f;
    m[n][0] = m[n][1] = kNone;
    l[n][0] = l[n][1] = 0.0f;
  }

  // The warp's blocks: begin + warp, + kWarps, ...; 32 of them are looked up at a time, a lane each.
  const int mine = begin + warp < end ? (end - begin - warp + kWarps - 1) / kWarps : 0;
  const int64_t table_row = static_cast<int64_t>(b) * P.bt_stride, head_row = static_cast<int64_t>(kvh) * P.num_blocks;
  const int32_t* chosen = !PLAIN && P.chosen ? P.chosen + (static_cast<int64_t>(b) * P.H_kv + kvh) * P.top : nullptr;
  auto position_of = [&](int i) {   // first position of the warp's i-th block
    const int at = begin + warp + i * kWarps;
    if (chosen) return chosen[at] * JF_BLOCK_SIZE;
    return (at < span.head ? at : span.first + at - span.head) * JF_BLOCK_SIZE;
  };
  struct Look { int id, pos; float ks, vs; };   // pos: 1 more where some of the block's positions are not seen
  auto look_up = [&](int i0) {
    Look r{-1, 0, 0.0f, 0.0f};
    if (i0 + lane < mine) {
      r.pos = position_of(i0 + lane);
      const int blk = r.pos / JF_BLOCK_SIZE, own = PLAIN ? blk : blk - P.shared_blocks;
      const int64_t id = !PLAIN && own < 0 ? shared_id(P, blk) : block_id(P, table_row + own);
      r.id = id < 0 || id >= P.num_blocks ? -1 : static_cast<int>(id);
      if (r.id >= 0) {
        r.ks = P.k_scales[head_row + r.id];
        r.vs = P.v_scales[head_row + r.id];
      }
      if (!(r.pos + JF_BLOCK_SIZE <= span.len && (r.pos >= span.lo || r.pos + JF_BLOCK_SIZE <= span.prefix))) r.pos += 1;
    }
    return r;
  };
  // What was looked up of 64 blocks: id (-1: nothing there), K scale, log2 of the V scale (0 is taken for 2^-100: weightless, but
  // its positions count), position.
  int4* entries = reinterpret_cast<int4*>(smem + kWarps * kStages * kStageBytes) + warp * 64;
  auto note = [&](int i0, const Look& r) {
    float lg;
    asm("lg2.approx.f32 %0, %1;" : "=f"(lg) : "f"(r.vs == 0.0f ? 0x1p-100f : r.vs));
    entries[(i0 + lane) & 63] = make_int4(r.id, __float_as_int(r.ks), __float_as_int(lg), r.pos);
  };
  // Rings of K and V blocks, kStages each; K runs one block ahead, since the scores of a block are worked out beside the
  // outputs of the one before it.
  unsigned char* k_ring = smem + warp * kStages * kStageBytes;
  unsigned char* v_ring = k_ring + kStages * (kStageBytes / 2);
  // A copy moves 512 consecutive bytes, four rows (pieces of rows that the lanes need were 130 us where this takes 102:
  // four sequences of 65536 positions, 8 KV heads, copies alone).  In shared memory the 16-byte chunks of a row change places
  // so that eight lanes which read together meet no bank twice: K's by the row's parity, V's by its pair.
  const int row4 = lane >> 3, chunk = lane & 7;
  const uint8_t* k_base = P.k_data + head_row * (JF_BLOCK_SIZE * JF_HEAD_DIM) + lane * 16;
  const uint8_t* v_base = P.v_data + head_row * (JF_BLOCK_SIZE * JF_HEAD_DIM) + lane * 16;
  const int k_to = row4 * JF_HEAD_DIM + ((chunk ^ (row4 & 1) << 2) << 4), v_to = row4 * JF_HEAD_DIM + ((chunk ^ (row4 >> 1) << 1) << 4);
  const int k_at = g * JF_HEAD_DIM + ((t ^ (g & 1) << 2) << 4), v_at = 2 * t * JF_HEAD_DIM + ((g ^ t << 1) << 4);
  auto fetch_k = [&](int id, int slot) {
    if (id < 0) return;
    const uint8_t* k = k_base + static_cast<int64_t>(id) * (JF_BLOCK_SIZE * JF_HEAD_DIM);
#pragma unroll
    for (int i = 0; i < 4; ++i) cp_async_16(k_ring + slot * 2048 + i * 512 + k_to, k + i * 512);
  };
  auto fetch_v = [&](int id, int slot) {
    if (id < 0) return;
    const uint8_t* v = v_base + static_cast<int64_t>(id) * (JF_BLOCK_SIZE * JF_HEAD_DIM);
#pragma unroll
    for (int i = 0; i < 4; ++i) cp_async_16(v_ring + slot * 2048 + i * 512 + (v_to ^ (i & 1) << 6), v + i * 512);
  };
  const Look look = look_up(0);
  // (copies arrive in the order of their groups: K of block j is in group j, V of block j in group j + 1)
  const int id0 = __shfl_sync(0xFFFFFFFFu, look.id, 0), id1 = __shfl_sync(0xFFFFFFFFu, look.id, 1), id2 = __shfl_sync(0xFFFFFFFFu, look.id, 2);
  fetch_k(id0, 0);
  cp_async_commit();
  fetch_k(id1, 1);
  fetch_v(id0, 0);
  cp_async_commit();
  fetch_k(id2, 2);
  fetch_v(id1, 1);
  cp_async_commit();
  // q as operands: fp16 pairs, or the three bytes of four elements at a time
  constexpr bool INT = CODES == JF_CODES_INT8;
  uint32_t qf[NT][INT ? 24 : 16];
  float sfac[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float x[32], amax = 0.0f, odd = 0.0f;   // odd: NaN if an element is no number, else 0
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w[4] = {q_raw[n][i].x, q_raw[n][i].y, q_raw[n][i].z, q_raw[n][i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float y = Elem<DT>::to_f32(static_cast<uint16_t>(w[k] >> 16 * e));
          x[i * 8 + k * 2 + e] = y;
          amax = fmaxf(amax, fabsf(y));
          odd = fmaf(y, 0.0f, odd);
        }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
      odd += __shfl_xor_sync(0xFFFFFFFFu, odd, o);
    }
    // a power of two that brings the largest element to [2^TOP, 2^(TOP + 1)); 2^126 at most
    constexpr int TOP = INT ? 21 : 13;
    const int e = max(min(static_cast<int>(__float_as_uint(amax) >> 23) - 127, 127), TOP - 126);
    const float up = __uint_as_float(static_cast<uint32_t>(TOP - e + 127) << 23);
#pragma unroll
    for (int w = 0; w < 8; ++w) {   // word w of the lane's 32 channels
      if (INT) {
        uint32_t lo = 0, mid = 0, hi = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int v = __float2int_rn(x[w * 4 + k] * up), a = static_cast<int8_t>(v), r = (v - a) >> 8, c = static_cast<int8_t>(r);
          lo |= (static_cast<uint32_t>(a) & 255u) << 8 * k;
          mid |= (static_cast<uint32_t>(c) & 255u) << 8 * k;
          hi |= (static_cast<uint32_t>((r - c) >> 8) & 255u) << 8 * k;
        }
        qf[n][w] = lo;
        qf[n][8 + w] = mid;
        qf[n][16 + w] = hi;
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const __half2 h = __floats2half2_rn(x[w * 4 + k * 2] * up, x[w * 4 + k * 2 + 1] * up);
          qf[n][w * 2 + k] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
    }
    // what brings a sum of products back, for the heads of the lane's score columns 2t and 2t + 1
    const float down = __uint_as_float(static_cast<uint32_t>(e - TOP + 127) << 23) + odd;
#pragma unroll
    for (int c = 0; c < 2; ++c) sfac[n][c] = __shfl_sync(0xFFFFFFFFu, down, (2 * t + c) * 4) * P.scale * kLog2e;
  }

  const float cap2 = FEAT ? P.softcap * kLog2e : 0.0f, inv_cap = cap2 > 0.0f ? 1.0f / cap2 : 0.0f;   // (scores are in units of log2)
  note(0, look);
  // Scores of a block, in units of log2 and with log2 of its V scale on top; -inf where there is nothing to see.
  auto score = [&](float (&s)[NT][4], int4 entry, const unsigned char* at) {
    const float ks = __int_as_float(entry.y), lvs = __int_as_float(entry.z);
    const int pos = entry.w & ~1;
    if (entry.x < 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[n][k] = -INFINITY;
      return;
    }
    if (INT) {
      int d[NT][3][4] = {};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint4 a = *reinterpret_cast<const uint4*>(at + (k_at ^ half << 6)), c = *reinterpret_cast<const uint4*>(at + (k_at ^ half << 6) + 1024);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            mma_s8_16832(d[n][k], a.x, c.x, a.y, c.y, qf[n][k * 8 + half * 4], qf[n][k * 8 + half * 4 + 1]);
            mma_s8_16832(d[n][k], a.z, c.z, a.w, c.w, qf[n][k * 8 + half * 4 + 2], qf[n][k * 8 + half * 4 + 3]);
          }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k)   // (the upper two together stay below 2^29)
          s[n][k] = fmaf(static_cast<float>(d[n][2][k] * 256 + d[n][1][k]), 256.0f, static_cast<float>(d[n][0][k])) * (sfac[n][k & 1] * ks);
    } else {
      float c2[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[n][k] = c2[n][k] = 0.0f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint4 lo = *reinterpret_cast<const uint4*>(at + (k_at ^ half << 6)), hi = *reinterpret_cast<const uint4*>(at + (k_at ^ half << 6) + 1024);
        const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, c[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t a0 = widen<CODES, false>(a[w]), a1 = widen<CODES, false>(c[w]), a2 = widen<CODES, true>(a[w]), a3 = widen<CODES, true>(c[w]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16_16816(half ? c2[n] : s[n], a0, a1, a2, a3, qf[n][(half * 8 + w * 2) % 16], qf[n][(half * 8 + w * 2 + 1) % 16]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[n][k] = (s[n][k] + c2[n][k]) * (sfac[n][k & 1] * ks);
    }
    if (FEAT) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (cap2 > 0.0f) soften4(s[n], cap2, inv_cap);
        if (P.slopes) {
          const float apart = static_cast<float>(span.len - 1 - g - pos);   // of the lane's first position; its second is 8 nearer
#pragma unroll
          for (int k = 0; k < 4; ++k) s[n][k] = fmaf(-slope[n][k & 1], k < 2 ? apart : apart - 8.0f, s[n][k]);
        }
      }
    }
    if (entry.w & 1) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int p = pos + g + k * 8;
        const bool seen = p < span.len && (p >= span.lo || p < span.prefix);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          s[n][2 * k] = seen ? s[n][2 * k] : -INFINITY;
          s[n][2 * k + 1] = seen ? s[n][2 * k + 1] : -INFINITY;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[n][k] += lvs;
  };
  cp_async_wait_group<2>();
  __syncwarp();
  float s[NT][4];
  int4 now = entries[0];   // block i
  score(s, now, k_ring);
  int slot = 0;            // i % kStages
  for (int i = 0; i < mine; ++i) {
    if ((i & 31) == 0) note(i + 32, look_up(i + 32));
    __syncwarp();          // the slots that are filled now were read in the step before
    const int slot1 = slot + 1 == kStages ? 0 : slot + 1, slot2 = slot1 + 1 == kStages ? 0 : slot1 + 1;
    fetch_k(entries[(i + 3) & 63].x, slot);   // (K of block i was read in the step before)
    fetch_v(entries[(i + 2) & 63].x, slot2);
    cp_async_commit();
    cp_async_wait_group<2>();
    __syncwarp();
    const int4 then = entries[(i + 1) & 63];
    const float lvs = __int_as_float(now.z);
    float ahead[NT][4];
    score(ahead, then, k_ring + slot1 * 2048);
    const unsigned char* at = v_ring + slot * 2048;
    bool above = false, full = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int k = 0; k < 4; ++k) above |= s[n][k] > m[n][k & 1] + (kLift + kLag);
      full |= fmaxf(l[n][0], l[n][1]) > kFull;
    }
    if (__any_sync(0xFFFFFFFFu, above || full)) {
      full = __any_sync(0xFFFFFFFFu, full);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = fmaxf(s[n][c], s[n][2 + c]);
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
          float to = fmaxf(m[n][c], top - kLift);
          if (full) {
            float most = l[n][c];
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 4));
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 8));
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 16));
            if (most > kFull) to = fmaxf(to, m[n][c] + kDrop);
          }
          const float h = half_step(to - m[n][c]), f = h * h;
          m[n][c] = to;
          l[n][c] *= h;
          l[n][c] *= h;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            o[n][j][c] *= f;
            o[n][j][2 + c] *= f;
          }
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float e0 = s[n][0] - m[n][0], e1 = s[n][1] - m[n][1], e2 = s[n][2] - m[n][0], e3 = s[n][3] - m[n][1];
      l[n][0] += ex2(e0 - lvs) + ex2(e2 - lvs);
      l[n][1] += ex2(e1 - lvs) + ex2(e3 - lvs);
      const __half2 a = __floats2half2_rn(ex2(e0), ex2(e1)), c = __floats2half2_rn(ex2(e2), ex2(e3));
      pb[n][0] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&a));
      pb[n][1] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&c));
    }
    if (now.x >= 0) {
      uint32_t r[4][4];
#pragma unroll
      for (int i2 = 0; i2 < 4; ++i2) {
        const uint4 x = *reinterpret_cast<const uint4*>(at + v_at + (i2 & 1) * JF_HEAD_DIM + (i2 >> 1) * 1024);
        r[i2][0] = bias<CODES>(x.x); r[i2][1] = bias<CODES>(x.y); r[i2][2] = bias<CODES>(x.z); r[i2][3] = bias<CODES>(x.w);
        if (CODES == JF_CODES_E4M3 && now.w & 1) {   // a weight of 0 does not make up for a row of NaN codes
          const int p = (now.w & ~1) + 2 * t + (i2 & 1) + (i2 >> 1) * 8;
          if (p >= span.len || (p < span.lo && p >= span.prefix)) r[i2][0] = r[i2][1] = r[i2][2] = r[i2][3] = 0;
        }
      }
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int hl = 0; hl < 2; ++hl) {   // channels 16g + 4w + 2hl (row g of the tile) and the next (row g + 8)
          const uint32_t x = prmt(r[0][w], r[1][w], hl ? 0x7362u : 0x5140u), y = prmt(r[2][w], r[3][w], hl ? 0x7362u : 0x5140u);
          const uint32_t a0 = widen<CODES, false>(x), a1 = widen<CODES, true>(x), a2 = widen<CODES, false>(y), a3 = widen<CODES, true>(y);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16_16816(o[n][2 * w + hl], a0, a1, a2, a3, pb[n][0], pb[n][1]);
        }
    }
    now = then;
    slot = slot1;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[n][k] = ahead[n][k];
  }
  cp_async_wait_all();

  // The warps' results meet: references first, then the sums under the common one.
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float x = l[n][c];
      x += __shfl_xor_sync(0xFFFFFFFFu, x, 4);
      x += __shfl_xor_sync(0xFFFFFFFFu, x, 8);
      x += __shfl_xor_sync(0xFFFFFFFFu, x, 16);
      if (x > kLeave) {
        const float to = m[n][c] + kDown, f = ex2(m[n][c] - to);
        m[n][c] = to;
        x *= f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[n][j][c] *= f;
          o[n][j][2 + c] *= f;
        }
      }
      if (g == 0) {
        sm_m[warp][n * 8 + 2 * t + c] = m[n][c];
        sm_l[warp][n * 8 + 2 * t + c] = x;
      }
    }
  __syncthreads();   // (also: every warp is through with its ring)
  float* so = reinterpret_cast<float*>(smem);   // [warp][head][128]
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float f[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float top = kNone;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w][n * 8 + 2 * t + c]);
      f[c] = ex2(m[n][c] - top);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)   // tile j: channels 16g + 2j (registers 0, 1) and 16g + 2j + 1
#pragma unroll
      for (int c = 0; c < 2; ++c)
        *reinterpret_cast<float2*>(so + (warp * 8 * NT + n * 8 + 2 * t + c) * JF_HEAD_DIM + 16 * g + 2 * j) =
            make_float2(o[n][j][c] * f[c], o[n][j][2 + c] * f[c]);
  }
  if (threadIdx.x < 8 * NT) {
    float top = kNone, z = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w][threadIdx.x]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float h = half_step(top - sm_m[w][threadIdx.x]);
      z = fmaf(sm_l[w][threadIdx.x] * h, h, z);
    }
    sm_ml[threadIdx.x] = make_float2(top, z);
  }
  __syncthreads();
  auto write = [&](int head, int d, float4 sum, float2 ml) {
    const int64_t row = static_cast<int64_t>(b) * P.H_q + first_head + head;
    const bool none = ml.y == 0.0f;   // (nothing seen: any position that is leaves a weight, or a NaN)
    const float r[4] = {sum.x, sum.y, sum.z, sum.w};
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = Elem<DT>::from_f32(none ? 0.0f : r[k] / ml.y);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.out) + row * JF_HEAD_DIM + d) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    if (d == 0 && P.lse) P.lse[row] = none ? -INFINITY : (ml.x + __log2f(ml.y)) / kLog2e;
  };
  constexpr int kQuads = JF_HEAD_DIM / 4;
  for (int i = threadIdx.x; i < heads * kQuads; i += kWarps * 32) {
    const int head = i / kQuads, d = i % kQuads * 4;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(so + (w * 8 * NT + head) * JF_HEAD_DIM + d);
      sum = make_float4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
    }
    if (cut.n == 1 && !partial) {
      write(head, d, sum, sm_ml[head]);
    } else if (CLUSTER && !partial) {
      *reinterpret_cast<float4*>(so + head * JF_HEAD_DIM + d) = sum;   // (no other thread reads these four)
    } else {
      const int64_t row = (static_cast<int64_t>(blockIdx.x) * gridDim.y + blockIdx.y) * (8 * NT) + head;
      *reinterpret_cast<float4*>(P.part_o + row * JF_HEAD_DIM + d) = sum;
      if (d == 0) *reinterpret_cast<float2*>(P.part_ml + row * 2) = sm_ml[head];
    }
  }
  if (CLUSTER && cut.n > 1) {
    cluster_sync();
    // every block joins its share of the (head, four channels)
    const int share = (heads * kQuads + cut.n - 1) / cut.n;
    for (int i = cut.index * share + threadIdx.x; i < min((cut.index + 1) * share, heads * kQuads); i += kWarps * 32) {
      const int head = i / kQuads, d = i % kQuads * 4;
      float2 ml[8];
      float4 x[8];
      float top = kNone, z = 0.0f;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < cut.n) {
          ml[r] = load2_from(of_rank(&sm_ml[head], r));
          x[r] = load4_from(of_rank(so + head * JF_HEAD_DIM + d, r));
          top = fmaxf(top, ml[r].x);
        }
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < cut.n) {
          const float h = half_step(top - ml[r].x), f = h * h;
          z = fmaf(ml[r].y * h, h, z);
          sum = make_float4(fmaf(x[r].x, f, sum.x), fmaf(x[r].y, f, sum.y), fmaf(x[r].z, f, sum.z), fmaf(x[r].w, f, sum.w));
        }
      write(head, d, sum, make_float2(top, z));
    }
    cluster_sync();   // nobody leaves while its shared memory is read
  }
  if (partial) pdl_wait();
}

// The pieces of a sequence.  A block of WARPS warps per (head, sequence) and 32 * VEC channels; a warp takes every WARPS-th piece.
template <int DT, int VEC, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) block8_join_kernel(const __grid_constant__ AttnParams P, int width, int grid_y) {
  __shared__ float sm_w[WARPS * 32], sm_z[WARPS], sm_top[WARPS], sm_o[WARPS][32 * VEC];
  const int b = blockIdx.y, h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // The lengths are not written by the kernel in front of this one, whose blocks all wait for what is in front of them before
  // they let this one start: they may be read at once.  Every warp works out for itself which pieces are the sequence's.
  int total = 0, first = 0, n = 0;
  for (int i = lane; i < P.B; i += 32) total += blocks_of(P, i);
  const int piece = piece_length(P, __reduce_add_sync(0xFFFFFFFFu, total), total);   // (up to 32 sequences: a lane's total is its own)
  for (int i = lane; i <= b; i += 32) {
    const int k = max(1, (blocks_of(P, i) + piece - 1) / piece);
    if (i < b) first += k; else n = k;
  }
  first = __reduce_add_sync(0xFFFFFFFFu, first);
  n = __reduce_add_sync(0xFFFFFFFFu, n);
  pdl_wait();   // (also by blocks with nothing to do: who follows this kernel relies on the one before it)
  pdl_trigger();
  if (n == 1) return;
  const int kvh = h / P.G, in_group = h % P.G, y = kvh * P.groups + in_group / width;
  const int64_t row0 = (static_cast<int64_t>(first) * grid_y + y) * width + in_group % width, step = static_cast<int64_t>(grid_y) * width;
  float top = kNone;
  for (int i = threadIdx.x; i < n; i += WARPS * 32) top = fmaxf(top, P.part_ml[(row0 + i * step) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (lane == 0) sm_top[warp] = top;
  __syncthreads();
  top = sm_top[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm_top[w]);
  float sum[VEC] = {}, z = 0.0f;
  for (int i0 = 0; i0 < n; i0 += WARPS * 32) {
    const int m = min(WARPS * 32, n - i0);
    if (threadIdx.x < m) {
      const float2 ml = *reinterpret_cast<const float2*>(P.part_ml + (row0 + (i0 + threadIdx.x) * step) * 2);
      const float h = half_step(top - ml.x);
      sm_w[threadIdx.x] = h * h;
      z = fmaf(ml.y * h, h, z);
    }
    __syncthreads();
    const float* o = P.part_o + (row0 + i0 * step) * JF_HEAD_DIM + (blockIdx.z * 32 + lane) * VEC;
#pragma unroll 8
    for (int i = warp; i < m; i += WARPS) {
      const float w = sm_w[i];
      if (VEC == 4) {
        const float4 x = *reinterpret_cast<const float4*>(o + i * step * JF_HEAD_DIM);
        const float e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] = fmaf(e[k], w, sum[k]);
      } else {
        sum[0] = fmaf(o[i * step * JF_HEAD_DIM], w, sum[0]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xFFFFFFFFu, z, o);
#pragma unroll
  for (int k = 0; k < VEC; ++k) sm_o[warp][lane * VEC + k] = sum[k];
  if (lane == 0) sm_z[warp] = z;
  __syncthreads();
  for (int ch = threadIdx.x; ch < 32 * VEC; ch += WARPS * 32) {
    float x = 0.0f;
    z = 0.0f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      x += sm_o[k][ch];
      z += sm_z[k];
    }
    const int64_t row = static_cast<int64_t>(b) * P.H_q + h;
    static_cast<uint16_t*>(P.out)[row * JF_HEAD_DIM + blockIdx.z * 32 * VEC + ch] = Elem<DT>::from_f32(z == 0.0f ? 0.0f : x / z);
    if (ch == 0 && blockIdx.z == 0 && P.lse) P.lse[row] = z == 0.0f ? -INFINITY : (top + __log2f(z)) / kLog2e;
  }
}

// The pieces of a sequence and the partial results of the positions before them (part_o, part_ml of `from`): WARPS warps per (sequence,
// head), four channels a lane.  A result there has references of its own for its output and for its sum.
template <int DT, int WARPS>
__global__ void __launch_bounds__(256) block8_join_shared_kernel(const __grid_constant__ AttnParams P, const __grid_constant__ Block8Source from, int width,
                                                                 int grid_y) {
  constexpr int ROWS = 8 / WARPS;
  __shared__ float2 sm_top[8], sm_z[8];
  __shared__ float4 sm_o[WARPS > 1 ? 8 : 1][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % WARPS;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + warp / WARPS;
  const int b = static_cast<int>(row / P.H_q), h = static_cast<int>(row % P.H_q);
  pdl_wait();
  pdl_trigger();
  if (b >= P.B) return;   // (with several warps a row there is a row for every block)
  int total = 0, first = b, n = 1;   // pieces of the sequence: one where no piece had to be looked for
  if (P.cluster == 0) {
    first = n = 0;
    for (int i = lane; i < P.B; i += 32) total += blocks_of(P, i);
    const int piece = piece_length(P, __reduce_add_sync(0xFFFFFFFFu, total), total);
    for (int i = lane; i <= b; i += 32) {
      const int k = max(1, (blocks_of(P, i) + piece - 1) / piece);
      if (i < b) first += k; else n = k;
    }
    first = __reduce_add_sync(0xFFFFFFFFu, first);
    n = __reduce_add_sync(0xFFFFFFFFu, n);
  }
  const int kvh = h / P.G, in_group = h % P.G, y = kvh * P.groups + in_group / width;
  const int64_t own0 = (static_cast<int64_t>(first) * grid_y + y) * width + in_group % width, step = static_cast<int64_t>(grid_y) * width;
  // the results of the row's pair of row tiles: those of the thread blocks that hold some of its units, and where it is a single tile of both groups
  const int64_t in_head = static_cast<int64_t>(b) * P.G + in_group;
  const int tile = static_cast<int>(in_head / 128), r = static_cast<int>(in_head % 128), pair = tile / 2;
  const bool two = pair * 2 + 1 < from.row_tiles;
  const int64_t item = static_cast<int64_t>(kvh) * from.pairs + pair, u0 = item * from.tiles, u1 = u0 + from.tiles - 1;
  const int64_t c0 = ((u0 + 1) * from.grid - 1) / from.units, c1 = ((u1 + 1) * from.grid - 1) / from.units;
  const int per = two ? 1 : 2, m = static_cast<int>(c1 - c0 + 1) * per;
  auto result = [&](int i) {   // row of part_o and part_ml
    const int64_t c = c0 + i / per;
    return ((c + item) * 2 + (two ? tile & 1 : i % per)) * 128 + r;
  };
  // references
  float top_o = kNone, top_l = kNone;
  for (int i = part * 32 + lane; i < n + m; i += WARPS * 32) {
    if (i < n) {
      const float x = P.part_ml[(own0 + i * step) * 2];
      top_o = fmaxf(top_o, x);
      top_l = fmaxf(top_l, x);
    } else {
      const float4 x = from.part_ml[result(i - n)];
      top_o = fmaxf(top_o, x.x);
      top_l = fmaxf(top_l, x.y);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top_o = fmaxf(top_o, __shfl_xor_sync(0xFFFFFFFFu, top_o, o));
    top_l = fmaxf(top_l, __shfl_xor_sync(0xFFFFFFFFu, top_l, o));
  }
  if (WARPS > 1) {
    if (lane == 0) sm_top[warp] = make_float2(top_o, top_l);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      top_o = fmaxf(top_o, sm_top[k].x);
      top_l = fmaxf(top_l, sm_top[k].y);
    }
  }
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float z = 0.0f;
  // (results part, part + WARPS, ...: a lane looks at one, then all lanes take their channels of each)
  for (int i0 = 0; i0 * WARPS < n + m; i0 += 32) {
    const int i = (i0 + lane) * WARPS + part;
    float w = 0.0f;
    int64_t at = -1;
    if (i < n) {
      const float2 x = *reinterpret_cast<const float2*>(P.part_ml + (own0 + i * step) * 2);
      const float f = half_step(top_l - x.x), e = half_step(top_o - x.x);
      z = fmaf(x.y * f, f, z);
      w = e * e;
      if (x.y != 0.0f) at = own0 + i * step;
    } else if (i < n + m) {
      const int64_t where = result(i - n);
      const float4 x = from.part_ml[where];
      const float f = half_step(top_l - x.y), e = half_step(top_o - x.x);
      z = fmaf(x.z * f, f, z);
      w = e * e;
      if (x.z != 0.0f) at = where;     // (a group without tiles left no output)
    }
    const int some = min(32, (n + m - i0 * WARPS + WARPS - 1) / WARPS);
    for (int k0 = 0; k0 < some; k0 += 8) {   // eight results in flight
      float4 x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t where = __shfl_sync(0xFFFFFFFFu, at, k0 + k);
        x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (where >= 0) x[k] = *reinterpret_cast<const float4*>(((i0 + k0 + k) * WARPS + part < n ? P.part_o : from.part_o) + where * JF_HEAD_DIM + lane * 4);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = __shfl_sync(0xFFFFFFFFu, w, k0 + k);
        sum = make_float4(fmaf(x[k].x, f, sum.x), fmaf(x[k].y, f, sum.y), fmaf(x[k].z, f, sum.z), fmaf(x[k].w, f, sum.w));
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xFFFFFFFFu, z, o);
  if (WARPS > 1) {
    if (lane == 0) sm_z[warp].x = z;
    sm_o[warp][lane] = sum;
    __syncthreads();
    if (warp > 0) return;
    z = 0.0f;
    sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      z += sm_z[k].x;
      const float4 x = sm_o[k][lane];
      sum = make_float4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
    }
  }
  const bool none = z == 0.0f;
  const float f = half_step(top_l - top_o);
  const float e[4] = {sum.x, sum.y, sum.z, sum.w};
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = Elem<DT>::from_f32(none ? 0.0f : e[k] / z * f * f);
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.out) + row * JF_HEAD_DIM + lane * 4) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
  if (lane == 0 && P.lse) P.lse[row] = none ? -INFINITY : (top_l + __log2f(z)) / kLog2e;
}

struct Plan { int G, nt, groups, target, min_piece, pieces; uint64_t bytes; };
constexpr int kMinPiece = 8;   // blocks
// Pieces of a sequence on average: from kManyPieces on the join spreads a row over four blocks of 16 warps, below kFewPieces it gives it four
// warps.  Its blocks start late, when those of the first kernel have left their registers, so the fewer they take the sooner all of
// them run: 32 sequences of up to 8191 positions, four KV heads, 30.5 -> 26.6 us against eight warps a row; two of 46000, 25.9 -> 21.6
// against blocks of 32 warps (of eight: 22.1, but one of 20000 with one KV head 14.2 and not 11.2).
constexpr int kManyPieces = 32, kFewPieces = 16;

// Pieces per KV head: one wave of blocks where the batch leaves room for it, three where it does not.
bool make_plan(int B, int H_q, int H_kv, int max_S, Plan& p) {
  if (B <= 0 || H_q <= 0 || H_kv <= 0 || max_S <= 0 || H_q % H_kv != 0) return false;
  p.G = H_q / H_kv;
  p.nt = p.G <= 8 ? 1 : 2;
  p.groups = (p.G + 8 * p.nt - 1) / (8 * p.nt);
  const int64_t columns = static_cast<int64_t>(H_kv) * p.groups;
  const int64_t most = (static_cast<int64_t>(max_S) + JF_BLOCK_SIZE - 1) / JF_BLOCK_SIZE;       // blocks of a sequence
  if (columns > 65535 || H_q > 65535 || B > 65535 || most * B > INT32_MAX / 2) return false;
  const int64_t wave = std::max<int64_t>(1, static_cast<int64_t>(num_sms()) * (p.nt == 1 ? 2 : 1) / columns);
  p.target = static_cast<int>(2 * B <= wave ? wave - B : 3 * wave);
  p.target = std::max(p.target, 1);
  // A sequence is cut where that finds work for idle multiprocessors: down to a block per warp for one sequence, hardly at all where
  // the batch fills them (64 x 1000 positions, 8 KV heads: 61 -> 45 us; 8 x 500: 16 -> 12).
  p.min_piece = static_cast<int>(std::min<int64_t>(64, std::max<int64_t>(kMinPiece, B * columns / 2)));
  const int64_t each = (most + p.min_piece - 1) / p.min_piece;
  p.pieces = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(p.target) + B, each * B));
  p.bytes = static_cast<uint64_t>(p.pieces) * columns * 8 * p.nt * (JF_HEAD_DIM + 2) * sizeof(float);
  return true;
}

// Blocks of a cluster, 0 for pieces and a join.  As many as leave every warp a block, up to eight and while all of them are resident at
// once, where that is at most kRounds blocks a warp; kFewRounds where pieces could spread over eight times as many multiprocessors.
// One sequence of 500 positions, 8 KV heads: 7.7 -> 6.0 us (6.2 with what the sums have gained since), of 4000: 11.7 -> 9.1; 64 of 300: 19.6 -> 17.4; 8 of 2000: 14.9 -> 12.4.  With 2
// columns, 4000 positions take 9.2 us so and 8.6 in pieces.
constexpr int kRounds = 6, kFewRounds = 2;
// Blocks a warp up to which a sequence's part behind a shared prefix is one block's work, found without a search: 256 sequences of up to 509
// positions, 8 KV heads, 86 -> 63 us.
constexpr int kOwnRounds = 8;
constexpr int kManyResults = 16;   // of a row, see where it is used
int cluster_size(const Plan& p, int B, int H_kv, int64_t longest) {
  const int64_t blocks = (longest + JF_BLOCK_SIZE - 1) / JF_BLOCK_SIZE, columns = static_cast<int64_t>(H_kv) * p.groups * B;
  const int64_t places = static_cast<int64_t>(num_sms()) * (p.nt == 1 ? 2 : 1);
  int c = 1;
  while (c < 8 && c * kWarps < blocks && 2 * c * columns <= places) c *= 2;
  const int rounds = 8 * c * columns <= places ? kFewRounds : kRounds;
  return blocks <= static_cast<int64_t>(c) * kWarps * rounds ? c : 0;
}

template <int CODES, int DT, int NT, bool FEAT, bool PLAIN>
jf_status_t launch_attn(const AttnParams& P, dim3 grid, cudaStream_t s) {
  constexpr int smem = std::max(kWarps * (kStages * kStageBytes + 64 * 16), kWarps * 8 * NT * JF_HEAD_DIM * 4);
  if (P.cluster == 0) {
    AttnParams Q = P;
    Q.cluster = 1;
    auto* kernel = block8_attn_kernel<CODES, DT, NT, FEAT, false, PLAIN>;
    JF_ENSURE_SMEM(kernel, smem);
    JF_CUDA_TRY(launch_pdl(kernel, grid, dim3(kWarps * 32), smem, s, Q));
    return JF_OK;
  }
  auto* kernel = block8_attn_kernel<CODES, DT, NT, FEAT, true, PLAIN>;
  JF_ENSURE_SMEM(kernel, smem);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(P.cluster * P.B, grid.y);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = P.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  JF_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, P));
  return JF_OK;
}
template <int CODES, int DT, bool PLAIN> jf_status_t launch_attn(const AttnParams& P, int nt, bool feat, dim3 grid, cudaStream_t s) {
  if (nt == 1) return feat ? launch_attn<CODES, DT, 1, true, PLAIN>(P, grid, s) : launch_attn<CODES, DT, 1, false, PLAIN>(P, grid, s);
  return feat ? launch_attn<CODES, DT, 2, true, PLAIN>(P, grid, s) : launch_attn<CODES, DT, 2, false, PLAIN>(P, grid, s);
}
template <int CODES, int DT> jf_status_t launch_attn(const AttnParams& P, int nt, bool feat, dim3 grid, cudaStream_t s) {
  const bool plain = !P.chosen && P.shared_blocks == 0 && !P.partial;
  return plain ? launch_attn<CODES, DT, true>(P, nt, feat, grid, s) : launch_attn<CODES, DT, false>(P, nt, feat, grid, s);
}

}  // namespace

uint64_t block8_attn_workspace(int B, int H_q, int H_kv, int max_S) {
  Plan p;
  return make_plan(B, H_q, H_kv, max_S, p) ? p.bytes : 0;
}

jf_status_t block8_attend(const jf_block8_attn_args* a, const Block8Source& from, jf_stream_t stream, bool launch) {
  if ((a->q_dtype != JF_DTYPE_BF16 && a->q_dtype != JF_DTYPE_FP16) || (a->codes != JF_CODES_INT8 && a->codes != JF_CODES_E4M3)) return JF_ERR_ARG;
  if (a->B < 0 || a->max_blocks < 0 || a->num_blocks < 0 || a->window < 0) return JF_ERR_ARG;
  if (a->softcap != 0.0f && !(a->softcap >= 1.0e-30f && a->softcap <= 1.0e30f)) return JF_ERR_ARG;
  if (a->B == 0) return JF_OK;
  Plan p;
  const int max_S = from.chosen   ? static_cast<int>(std::min<int64_t>(a->max_S, int64_t{from.top} * JF_BLOCK_SIZE))   // scanned
                    : from.part_o ? std::max(a->max_S - from.behind * JF_BLOCK_SIZE, 1)
                                  : a->max_S;
  if (!make_plan(a->B, a->H_q, a->H_kv, max_S, p)) return JF_ERR_ARG;
  if (!a->q || !a->seq_lens || !a->out) return JF_ERR_ARG;
  // (a table without columns and a cache without blocks have no memory; nothing of them is read)
  if (a->max_blocks > 0 && !a->block_table) return JF_ERR_ARG;
  if (a->num_blocks > 0 && (!a->k_data || !a->v_data || !a->k_scales || !a->v_scales)) return JF_ERR_ARG;
  if (!aligned(a->q, 16) || !aligned(a->k_data, 16) || !aligned(a->v_data, 16) || !aligned(a->out, 8)) return JF_ERR_ARG;
  if (a->num_blocks > INT32_MAX) return JF_ERR_UNSUPPORTED;
  if (a->max_blocks > (INT32_MAX - JF_BLOCK_SIZE) / JF_BLOCK_SIZE - from.shared_blocks) return JF_ERR_UNSUPPORTED;
  if (!a->workspace || a->workspace_bytes < p.bytes || !aligned(a->workspace, 16)) return JF_ERR_WORKSPACE;
  if (!launch) return JF_OK;
  AttnParams P{};
  P.q = a->q;
  P.k_data = static_cast<const uint8_t*>(a->k_data);
  P.v_data = static_cast<const uint8_t*>(a->v_data);
  P.k_scales = a->k_scales;
  P.v_scales = a->v_scales;
  P.table = a->block_table;
  P.seq_lens = a->seq_lens;
  P.prefix_lens = a->prefix_lens;
  P.slopes = a->alibi_slopes;
  P.out = a->out;
  P.lse = a->lse;
  const int64_t rows = static_cast<int64_t>(p.pieces) * a->H_kv * p.groups * 8 * p.nt;
  P.part_o = static_cast<float*>(a->workspace);
  P.part_ml = P.part_o + rows * JF_HEAD_DIM;
  P.num_blocks = a->num_blocks;
  P.bt_stride = a->bt_stride;
  P.B = a->B; P.H_q = a->H_q; P.H_kv = a->H_kv; P.G = p.G; P.groups = p.groups;
  P.max_S = a->max_S; P.max_blocks = a->max_blocks + from.shared_blocks; P.window = a->window;
  P.target = p.target; P.min_piece = p.min_piece; P.pieces = p.pieces;
  // (only where a piece is several rounds of a block's warps: the search takes 0.2 us)
  const int64_t longest = a->window > 0 ? std::min(max_S, a->window) : max_S;
  P.one_wave = a->B > 1 && a->B <= 32 && 2 * a->B <= p.pieces && longest / JF_BLOCK_SIZE * a->B > 32ll * p.target;
  P.scale = a->attn_scale; P.softcap = a->softcap;
  P.bt_i32 = a->bt_is_i32 != 0;
  P.chosen = from.chosen; P.top = from.top;
  P.behind = from.behind * JF_BLOCK_SIZE;
  P.partial = from.part_o != nullptr;
  P.shared = from.shared; P.shared_blocks = from.shared_blocks; P.shared_i32 = from.shared_i32;
  // (partial results: a block for a sequence and KV head, where that is a few rounds of blocks a warp)
  const int64_t own_blocks = (static_cast<int64_t>(std::min<int64_t>(max_S, int64_t{a->max_blocks} * JF_BLOCK_SIZE)) + JF_BLOCK_SIZE - 1) / JF_BLOCK_SIZE;
  P.cluster = P.partial ? own_blocks <= kWarps * kOwnRounds : cluster_size(p, a->B, a->H_kv, a->prefix_lens ? a->max_S : longest);   // (a prefix may be as long as the sequence)
  const bool feat = a->softcap > 0.0f || a->alibi_slopes;
  const auto s = static_cast<cudaStream_t>(stream);
  const dim3 grid(p.pieces, a->H_kv * p.groups);   // (clusters: launch_attn)
  jf_status_t st;
  if (a->q_dtype == JF_DTYPE_BF16)
    st = a->codes == JF_CODES_INT8 ? launch_attn<JF_CODES_INT8, JF_DTYPE_BF16>(P, p.nt, feat, grid, s)
                                   : launch_attn<JF_CODES_E4M3, JF_DTYPE_BF16>(P, p.nt, feat, grid, s);
  else
    st = a->codes == JF_CODES_INT8 ? launch_attn<JF_CODES_INT8, JF_DTYPE_FP16>(P, p.nt, feat, grid, s)
                                   : launch_attn<JF_CODES_E4M3, JF_DTYPE_FP16>(P, p.nt, feat, grid, s);
  const int width = 8 * p.nt, grid_y = a->H_kv * p.groups;
  if (st == JF_OK && P.partial) {
    // Eight warps a row where a row has many results and the rows do not fill the multiprocessors: 8 / 1 heads, 16 sequences over 65536 shared
    // positions (128 rows of 297 results) 74 -> 32 us, 32 / 8 heads, 32 over 4096 (1024 of 37) 33 -> 30; 64 over 4096 would go from 36 to 42.
    const int64_t results = (from.grid + int64_t{a->H_kv} * from.pairs) / (int64_t{a->H_kv} * from.pairs) * (from.row_tiles & 1 ? 2 : 1);
    auto join = [&](auto dt, auto warps) {
      constexpr int D = decltype(dt)::value, W = decltype(warps)::value;
      const dim3 rows(static_cast<unsigned>((int64_t{a->B} * a->H_q * W + 7) / 8));
      return launch_pdl(block8_join_shared_kernel<D, W>, rows, dim3(256), 0, s, P, from, width, grid_y);
    };
    using One = std::integral_constant<int, 1>;
    using Eight = std::integral_constant<int, 8>;
    using Bf16 = std::integral_constant<int, JF_DTYPE_BF16>;
    using Fp16 = std::integral_constant<int, JF_DTYPE_FP16>;
    const bool many = results > kManyResults && int64_t{a->B} * a->H_q <= 8 * num_sms();
    if (a->q_dtype == JF_DTYPE_BF16) JF_CUDA_TRY(many ? join(Bf16(), Eight()) : join(Bf16(), One()));
    else JF_CUDA_TRY(many ? join(Fp16(), Eight()) : join(Fp16(), One()));
    return JF_OK;
  }
  if (st != JF_OK || P.cluster > 0 || p.pieces == a->B) return st;   // (one piece per sequence: nothing to join)
  auto join = [&](auto vec, auto warps, int z) {
    constexpr int V = decltype(vec)::value, W = decltype(warps)::value;
    const dim3 rows(a->H_q, a->B, z), block(W * 32);
    return a->q_dtype == JF_DTYPE_BF16 ? launch_pdl(block8_join_kernel<JF_DTYPE_BF16, V, W>, rows, block, 0, s, P, width, grid_y)
                                       : launch_pdl(block8_join_kernel<JF_DTYPE_FP16, V, W>, rows, block, 0, s, P, width, grid_y);
  };
  using std::integral_constant;
  const int each = p.pieces / a->B;
  JF_CUDA_TRY(each >= kManyPieces  ? join(integral_constant<int, 1>(), integral_constant<int, 16>(), 4)
              : each >= kFewPieces ? join(integral_constant<int, 4>(), integral_constant<int, 8>(), 1)
                                   : join(integral_constant<int, 4>(), integral_constant<int, 4>(), 1));
  return JF_OK;
}

}  // namespace jf

extern "C" uint64_t jf_block8_workspace_bytes(int32_t B, int32_t H_q, int32_t H_kv, int32_t max_S) {
  return jf::block8_attn_workspace(B, H_q, H_kv, max_S);
}

extern "C" jf_status_t jf_block8_attn(const jf_block8_attn_args* a, jf_stream_t stream) {
  return a ? jf::block8_attend(a, jf::Block8Source{}, stream, true) : JF_ERR_ARG;
}
