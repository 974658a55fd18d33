// Decode attention of sequences that share their first positions, over the 8-bit cache, on the fifth-generation tensor cores.
//
//   out_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp(f(scale q_r.k_j)),   r through the query heads of a KV head in all sequences
//
// The shared positions meet all rows of a KV head in one product, so that they are read, and turned into operands, once for
// 256 rows.  The codes become fp16, which holds them exactly, on their way through registers into the operands' shared-memory layout; a row's
// query is fp16 under a power of two that brings its largest element to [2^13, 2^14) (what that rounds is 2^-38 of it).  The
// scales stay out of the products, in fp32: a block's K scale multiplies its 16 scores, its V scale joins their exponent.
//
// A row keeps two references.  w = exp2(x + log2 vs - R) is the weight that meets V's codes (fp16: half a step is 2^-11 of it), x the
// score in units of log2; R lags the maximum of x + log2 vs by up to 2^kLag.  The sum of exp2(x - m) is formed block by block from the
// same exponentials, times exp2(R - log2 vs - m): one more of them for 16 positions.  Where V scales lie so far apart (beyond
// 2^kSpread) that a weight could vanish while its position counts, those tiles take an exponential more for every position.
//
//   warps 0-3, 4-7   scores -> weights of row tile 0, 1 (a thread a row); the rescaling of O; the partial result
//   warps 8, 9       codes -> fp16 operands: 128 positions of K, then of V, two buffers each
//   warp 10          issues the matrix products
//   warp 11          looks blocks up and copies their codes into shared memory, 2048 bytes at a time
// What is not on the common path is kept small (the code that all of these go through has to fit the instruction caches: at 123 KB a unit took
// 8300 cycles on the GPCs that have all their multiprocessors at work, 5000 on the others).
//
// Work is a line of units -- (KV head, pair of row tiles, 128 positions) -- cut into pieces of one length, one for each thread block, so that all
// multiprocessors end together; where a piece passes from one pair of row tiles to the next it leaves two partial results.  A single row
// tile (128 rows or fewer) is worked on by both groups of warps, in turn on its tiles of positions.  What the sequences have behind the shared positions goes
// through block8_attn.cu's kernel, whose partial results are joined with these ones.
//
// Bound: the tensor pipe and the exponentials in turn, and shared memory, which the operands, the codes and their conversion share.  A unit of 256 rows
// takes 4400 cycles (3900 without copies and conversion): 256 sequences over 65536 positions, 64 / 8 heads, int8, 530 us = 1.04 PFLOP/s, 0.63 of what
// cuBLAS reaches; the whole call 575 us against 4240 through block8_attn.cu.
#include "block8.cuh"
#include "decode_common.cuh"
#include "tensor_common.cuh"

#include <algorithm>
#include <type_traits>

namespace jf {
namespace {

constexpr int kRows = 128, kKeys = 128;                // of a tile
constexpr int kTileBlocks = kKeys / JF_BLOCK_SIZE;
constexpr int kCodeBytes = kKeys * JF_HEAD_DIM;        // of a tile as it lies in the cache
constexpr int kStaged = 2;                             // K or V tiles on their way from memory
constexpr int kNotes = 8;
constexpr int kThreads = 384;
// Registers a thread: the rows' warpgroups, the other one; together no more than the block is launched with (launch() checks that).
constexpr int kRowRegs = 208, kRoleRegs = 80;
constexpr float kLag = 8.0f, kLift = 7.0f;             // log2; weights stay below 2^15
constexpr float kSumLag = 24.0f, kSpread = 64.0f;
constexpr float kNone = -3.0e38f;                      // the reference of a row that has seen nothing (finite: differences are numbers)
constexpr float kLog2e = 1.4426950408889634f;
constexpr size_t kWorkspaceAlign = 32;                 // partial outputs are written 32 bytes at a time
constexpr int kSmemBytes = 227 * 1024;

struct SharedParams {
  const uint16_t* q;
  const uint8_t *k_data, *v_data;
  const float *k_scales, *v_scales;
  const void* table;
  const int32_t* seq_lens;
  float* part_o;          // [piece, row tile of the pair][128][128]
  float4* part_ml;        // R - lift, m, sum
  int32_t* status;
  int64_t num_blocks;
  int32_t units, H_q, G, rows, row_tiles, pairs, tiles, blocks, max_S;   // rows: of a KV head; blocks: shared ones; tiles: of positions
  float scale, softcap;
  bool i32;
};

// Bounded: 2^24 attempts, a second or so.  (No wait here is for more than the work on a few tiles.)
__device__ __forceinline__ bool await(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, 0;\n"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "add.u32 n, n, 1;\n\t"
      "setp.lt.u32 q, n, 16777216;\n\t"
      "@q bra AGAIN;\n"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return __all_sync(0xFFFFFFFFu, done != 0);
}

// What a tile's rows need to know of it: its blocks' K scales, log2 of their V scales.
struct alignas(16) Note {
  float ks[kTileBlocks], lvs[kTileBlocks];
  float lvs_lo, lvs_hi;
  uint32_t dead;          // a bit for each block that is not there
  uint32_t odd;           // a K scale that is not above zero
};
struct Shared {
  uint64_t code_full[kStaged], code_empty[kStaged], q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2][2],
      o_full[2], note_full[kNotes], products_done;
  Note note[kNotes];
  uint32_t tmem;
  int begin, end;         // units of this thread block
};

constexpr int kUsedBytes = 6 * kTileBytes + kStaged * kCodeBytes + static_cast<int>(sizeof(Shared));
static_assert(kUsedBytes + 1023 <= kSmemBytes, "the operands start on a multiple of 1024, wherever shared memory does");

// The units of a thread block, item by item (an item: a KV head and a pair of row tiles).
struct Segment { int u, end, item, first, n; };   // n tiles of positions from `first` on
__device__ __forceinline__ Segment units_of(const Shared& S) { return Segment{S.begin, S.end, 0, 0, 0}; }
__device__ __forceinline__ bool next_segment(const SharedParams& P, Segment& s) {
  s.u += s.n;
  if (s.u >= s.end) return false;
  s.item = s.u / P.tiles;
  s.first = s.u - s.item * P.tiles;
  s.n = min(P.tiles - s.first, s.end - s.u);
  return true;
}
__device__ __forceinline__ bool two_tiles(const SharedParams& P, const Segment& s) { return s.item % P.pairs * 2 + 1 < P.row_tiles; }
// Whether group t of rows has anything to do in a segment.
__device__ __forceinline__ bool has_jobs(const SharedParams& P, const Segment& s, int t) { return t < s.n || two_tiles(P, s); }

// ---- codes -> operands --------------------------------------------------------------------------
template <int CODES> __device__ __forceinline__ uint32_t flip(uint32_t w) { return CODES == JF_CODES_INT8 ? w ^ 0x80808080u : w; }
template <int CODES, bool HIGH> __device__ __forceinline__ uint32_t widen(uint32_t w) {   // two of four codes as fp16
  uint32_t d;
  if (CODES == JF_CODES_INT8)   // (sign bits turned over: 0x6400 + u is 1024 + u)
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(prmt(w, 0x64646464u, HIGH ? 0x4342u : 0x4140u)), "r"(0x64806480u));
  else if (HIGH)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(d) : "r"(w));
  else
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(d) : "r"(w));
  return d;
}

// Codes of the tiles in turn, K then V, and each tile's note.  `sent`: K and V tiles asked for.
__device__ __forceinline__ bool load(const SharedParams& P, Shared& S, unsigned char* staged, int& sent) {
  const int lane = threadIdx.x & 31;
  const Segment range = units_of(S);
  const int sides = 2 * (range.end - range.u);
  // four units' blocks are looked up at a time, a lane each, a round ahead
  struct Look { int id; float ks, vs; };
  auto look_up = [&](int u0) {
    Look r{-1, 0.0f, 0.0f};
    const int u = u0 + (lane >> 3);
    if (u < range.end) {
      const int item = u / P.tiles, block = (u - item * P.tiles) * kTileBlocks + (lane & 7);
      if (block < P.blocks) {
        const int64_t id = P.i32 ? static_cast<const int32_t*>(P.table)[block] : static_cast<const int64_t*>(P.table)[block];
        const int64_t row = static_cast<int64_t>(item / P.pairs) * P.num_blocks;
        if (id >= 0 && id < P.num_blocks) {
          r.id = static_cast<int>(id);
          r.ks = P.k_scales[row + id];
          r.vs = P.v_scales[row + id];
        }
      }
    }
    return r;
  };
  Look now = look_up(range.u), then = look_up(range.u + 4);
#pragma unroll 1
  for (int& n = sent; n < sides; ++n) {
    const int g = n >> 1, u = range.u + g;
    const int side = n & 1, slot = n % kStaged, off = (g & 3) * 8;
    if (side == 0 && g > 0 && off == 0) {
      now = then;
      then = look_up(u + 4);
    }
    if (n >= kStaged && !await(&S.code_empty[slot], static_cast<uint32_t>(n / kStaged - 1) & 1u)) return false;
    const int id = __shfl_sync(0xFFFFFFFFu, now.id, (off + lane) & 31);
    const bool mine = lane < kTileBlocks, is = mine && id >= 0;
    const unsigned there = __ballot_sync(0xFFFFFFFFu, is);
    if (side == 0) {
      const float ks = __shfl_sync(0xFFFFFFFFu, now.ks, (off + lane) & 31), vs = __shfl_sync(0xFFFFFFFFu, now.vs, (off + lane) & 31);
      float lg;
      asm("lg2.approx.f32 %0, %1;" : "=f"(lg) : "f"(vs == 0.0f ? 0x1p-100f : vs));   // (weightless, but its positions count)
      Note& note = S.note[g % kNotes];
      if (mine) {
        note.ks[lane] = is ? ks : 1.0f;
        note.lvs[lane] = is ? lg : 0.0f;
      }
      const unsigned odd = __ballot_sync(0xFFFFFFFFu, is && !(ks > 0.0f));
      float lo = is ? lg : 3.0e38f, hi = is ? lg : -3.0e38f;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
      }
      if (lane == 0) {
        note.lvs_lo = lo;
        note.lvs_hi = hi;
        note.dead = ~there & 255u;
        note.odd = odd;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.note_full[g % kNotes]);
    }
    if (lane == 0) mbar_expect_tx(&S.code_full[slot], __popc(there) * (JF_BLOCK_SIZE * JF_HEAD_DIM));
    __syncwarp();
    if (is) {
      const int head = u / P.tiles / P.pairs;
      bulk_g2s(staged + slot * kCodeBytes + lane * (JF_BLOCK_SIZE * JF_HEAD_DIM),
               (side ? P.v_data : P.k_data) + (static_cast<int64_t>(head) * P.num_blocks + id) * (JF_BLOCK_SIZE * JF_HEAD_DIM),
               JF_BLOCK_SIZE * JF_HEAD_DIM, &S.code_full[slot]);
    }
    __syncwarp();
  }
  return true;
}
// The copies that may be in flight: the block's shared memory stays until they are there, or a wait for one runs out.
__device__ __forceinline__ bool arrived(Shared& S, int sent) {
  for (int n = max(sent - kStaged, 0); n < sent; ++n)
    if (!await(&S.code_full[n % kStaged], static_cast<uint32_t>(n / kStaged) & 1u)) return false;
  return true;
}

template <int CODES> __device__ __forceinline__ bool convert(const SharedParams& P, Shared& S, unsigned char* kv, const unsigned char* staged) {
  const int lane = threadIdx.x & 31, tid = threadIdx.x & 63;
  const Segment range = units_of(S);
  const int sides = 2 * (range.end - range.u);
  // A thread has the same 16 channels of rows r and r + 8 of every block: two chunks of 16 bytes of the operand's row.  Eight threads that read or
  // write together have half of a row and the other half of the next one, which the swizzle puts on all banks.
  const int row = tid >> 4 << 1 | (tid >> 2 & 1), cc = ((tid >> 2 ^ tid >> 3) & 1) << 2 | (tid & 3), j0 = (cc & 3) * 2, sw = row & 7;
  const uint32_t base = (cc >> 2) * kSlabBytes + row * 128;
  const uint32_t lo_at = base + ((j0 ^ sw) << 4), hi_at = base + (((j0 + 1) ^ sw) << 4);
#pragma unroll 1
  for (int n = 0; n < sides; ++n) {
    const int g = n >> 1, side = n & 1, slot = g & 1, stage = n % kStaged;
    if (!await(&S.code_full[stage], static_cast<uint32_t>(n / kStaged) & 1u)) return false;
    if (g >= 2 && !await(side ? &S.v_empty[slot] : &S.k_empty[slot], static_cast<uint32_t>((g >> 1) - 1) & 1u)) return false;
    const uint32_t dead = S.note[g % kNotes].dead;
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      const unsigned char* from = staged + stage * kCodeBytes + h * (kCodeBytes / 2) + row * JF_HEAD_DIM + cc * 16;
      unsigned char* to = kv + (side * 2 + slot) * kTileBytes + h * (kSlabBytes / 2);
      uint4 x[kTileBlocks];
#pragma unroll
      for (int i = 0; i < kTileBlocks; ++i) x[i] = *reinterpret_cast<const uint4*>(from + i * 1024);
      if (dead) {
#pragma unroll
        for (int i = 0; i < kTileBlocks; ++i)
          if (dead >> (h * 4 + i / 2) & 1u) x[i] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kTileBlocks; ++i) {
        const uint32_t w[4] = {flip<CODES>(x[i].x), flip<CODES>(x[i].y), flip<CODES>(x[i].z), flip<CODES>(x[i].w)};
        *reinterpret_cast<uint4*>(to + i * 1024 + lo_at) =
            make_uint4(widen<CODES, false>(w[0]), widen<CODES, true>(w[0]), widen<CODES, false>(w[1]), widen<CODES, true>(w[1]));
        *reinterpret_cast<uint4*>(to + i * 1024 + hi_at) =
            make_uint4(widen<CODES, false>(w[2]), widen<CODES, true>(w[2]), widen<CODES, false>(w[3]), widen<CODES, true>(w[3]));
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&S.code_empty[stage]);
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(side ? &S.v_full[slot] : &S.k_full[slot]);
  }
  return true;
}

// ---- the products -------------------------------------------------------------------------------
// Jobs of a segment: with two row tiles (positions i, row tile 0), (i, 1), (i + 1, 0), ...; with one (i, group 0), (i + 1, group 1), ...
// The scores of job j + 2, which goes to the same group as job j, are asked for behind the products of its weights with V.
__device__ __forceinline__ bool multiply(const SharedParams& P, Shared& S, uint32_t q_smem, uint32_t kv_smem, uint32_t tmem) {
  constexpr uint32_t qk = instruction<JF_DTYPE_FP16>(false), pv = instruction<JF_DTYPE_FP16>(true);
  const uint64_t q_op = operand(q_smem, 16), k_op = operand(kv_smem, 16), v_op = operand(kv_smem + 2 * kTileBytes, kSlabBytes);
  Segment s = units_of(S);
  uint32_t base = 0, p_count0 = 0, p_count1 = 0, q_count0 = 0, q_count1 = 0;   // tiles of positions, weights, queries so far
  while (next_segment(P, s)) {
    const bool two = two_tiles(P, s);
    const int jobs = two ? 2 * s.n : s.n;
    if (!await(&S.q_full[0], q_count0++ & 1)) return false;
    if (jobs > 1 && !await(&S.q_full[1], q_count1++ & 1)) return false;
    // (the group as a constant: arrays and addresses that depend on it stay out of memory)
    auto scores = [&](auto t_tag, int j) {
      constexpr int t = decltype(t_tag)::value;
      const uint32_t g = base + (two ? j >> 1 : j), slot = g & 1;
      if ((!two || t == 0) && !await(&S.k_full[slot], g >> 1 & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = q_op + t * (kTileBytes >> 4), b = k_op + slot * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = ((k >> 2) * kSlabBytes + (k & 3) * 32) >> 4;
          mma_ss(tmem + t * 128, a + off, b + off, qk, k > 0);
        }
        tc_commit(&S.s_full[t]);
        if (!two || t == 1) tc_commit(&S.k_empty[slot]);
      }
      __syncwarp();
      return true;
    };
    auto job = [&](auto t_tag, int j, uint32_t parity) {
      constexpr int t = decltype(t_tag)::value;
      const uint32_t g = base + (two ? j >> 1 : j), slot = g & 1;
      if ((!two || t == 0) && !await(&S.v_full[slot], g >> 1 & 1)) return false;
      const uint64_t b = v_op + slot * (kTileBytes >> 4);
#pragma unroll
      for (int h = 0; h < 2; ++h) {   // the weights come in two halves
        if (!await(&S.p_full[t][h], parity)) return false;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = h * 4; k < h * 4 + 4; ++k)
            mma_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, b + k * (2048 >> 4), pv, j >= 2 || k > 0);
          if (h == 1 && (!two || t == 1)) tc_commit(&S.v_empty[slot]);
          if (h == 1 && j + 2 >= jobs) tc_commit(&S.o_full[t]);
        }
        __syncwarp();
      }
      return j + 2 >= jobs || scores(t_tag, j + 2);
    };
    using First = std::integral_constant<int, 0>;
    using Second = std::integral_constant<int, 1>;
    if (!scores(First(), 0) || (jobs > 1 && !scores(Second(), 1))) return false;
#pragma unroll 1
    for (int j = 0; j < jobs; j += 2) {
      if (!job(First(), j, p_count0++ & 1)) return false;
      if (j + 1 < jobs && !job(Second(), j + 1, p_count1++ & 1)) return false;
    }
    base += s.n;
  }
  return true;
}

// ---- scores -> weights ----------------------------------------------------------------------------
// The largest of 16 scores; a NaN if there is one.
__device__ __forceinline__ float largest16(const float* s) {
  float a = max3(s[0], s[1], s[2]), b = max3(s[3], s[4], s[5]);
  a = max3(a, s[6], s[7]);
  b = max3(b, s[8], s[9]);
  a = max3(a, s[10], s[11]);
  b = max3(b, s[12], s[13]);
  return max3(max3(a, b, s[14]), s[15], s[15]);
}
// cap * tanh(x / cap) of 32 scores, in units of log2 (cap2: the cap in these units), for the whole warp the same way: up to
// |x| = cap by a polynomial (relative error 6.6e-7), beyond it as cap - 2 cap / (e^(2x / cap) + 1).  A NaN stays one.
__device__ __forceinline__ void cap32(float* x, float cap2, float inv) {
  float most = 0.0f;
#pragma unroll
  for (int c = 0; c < 32; ++c) most = fmaxf(most, fabsf(x[c]));
  if (__all_sync(0xFFFFFFFFu, most <= cap2)) {
    const uint64_t i2 = pair(inv, inv);
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
      const uint64_t v = pair(x[c], x[c + 1]), z = mul2(v, i2), w = mul2(z, z);
      uint64_t q = fma2(w, pair(-0.00312657771f, -0.00312657771f), pair(0.0169064086f, 0.0169064086f));
      q = fma2(q, w, pair(-0.0517682843f, -0.0517682843f));
      q = fma2(q, w, pair(0.132884905f, 0.132884905f));
      q = fma2(q, w, pair(-0.333302796f, -0.333302796f));
      q = fma2(q, w, pair(1.0f, 1.0f));
      split(mul2(v, q), x[c], x[c + 1]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 32; ++c) x[c] = cap2 - __fdividef(2.0f * cap2, ex2(min_or_nan(x[c] * inv * (2.0f * kLog2e), 126.0f)) + 1.0f);
  }
}

template <int DT, bool CAP> __device__ __forceinline__ bool soften(const SharedParams& P, Shared& S, unsigned char* q_smem, uint32_t tmem, int t) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5 & 3, r = warp * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
  const uint32_t s_at = tmem + lanes + t * 128, o_at = tmem + lanes + 256 + t * 128;
  const float cap2 = CAP ? P.softcap * kLog2e : 0.0f, inv_cap = CAP ? 1.0f / cap2 : 0.0f;
  // The row's query as fp16 into the operand's place; what brings its products to scores in units of log2, and the positions that it sees.
  // (more than there are: all of them)
  struct Row { float f; int len; bool idle; };   // idle: no lane of the warp has a row
  auto load_query = [&](const Segment& s) {
    const int tile = s.item % P.pairs * 2 + (two_tiles(P, s) ? t : 0), row = tile * kRows + r;
    Row to{0.0f, INT32_MAX, tile * kRows + warp * 32 >= P.rows};
    if (!has_jobs(P, s, t)) return to;   // (its queries would not be waited for)
    const uint4* from = nullptr;
    if (row < P.rows) {
      const int b = row / P.G, head = s.item / P.pairs * P.G + row % P.G;
      from = reinterpret_cast<const uint4*>(P.q + (static_cast<int64_t>(b) * P.H_q + head) * JF_HEAD_DIM);
      const int len = max(min(P.seq_lens[b], P.max_S), 0);
      if (len < P.blocks * JF_BLOCK_SIZE) to.len = len;
    }
    float amax = 0.0f, odd = 0.0f;   // odd: NaN if an element is no number, else 0
    uint4 x[4];
    auto read = [&](int i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = from ? __ldg(from + i + k) : make_uint4(0, 0, 0, 0);
    };
    // (twice through the row, in loops: the code runs once a segment and comes from far)
#pragma unroll 1
    for (int i = 0; i < 16; i += 4) {
      read(i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float y = Elem<DT>::to_f32(static_cast<uint16_t>(w[k] >> 16 * e));
            amax = fmaxf(amax, fabsf(y));
            odd = fmaf(y, 0.0f, odd);
          }
      }
    }
    constexpr int TOP = 13;
    const int e = max(min(static_cast<int>(__float_as_uint(amax) >> 23) - 127, 127), TOP - 126);
    const float up = copysignf(__uint_as_float(static_cast<uint32_t>(TOP - e + 127) << 23), P.scale);
    to.f = __uint_as_float(static_cast<uint32_t>(e - TOP + 127) << 23) * fabsf(P.scale) * kLog2e + odd;
    unsigned char* out = q_smem + r * 128;
#pragma unroll 1
    for (int i = 0; i < 16; i += 4) {
      read(i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float lo = Elem<DT>::to_f32(static_cast<uint16_t>(w[k])) * up, hi = Elem<DT>::to_f32(static_cast<uint16_t>(w[k] >> 16)) * up;
          h[k] = odd == 0.0f ? round2<JF_DTYPE_FP16>(lo, hi) : 0u;
        }
        *reinterpret_cast<uint4*>(out + (i >> 3) * kSlabBytes + ((((i + j) & 7) ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(&S.q_full[t]);
    return to;
  };

  Segment s = units_of(S);
  uint32_t base = 0, tiles = 0, ends = 0;   // tiles of positions so far: of the block, of this group; segments with some
  Row row{0.0f, 0, true};
  for (bool more = true; more;) {   // (the first time round there is nothing but queries to be loaded)
    const bool two = two_tiles(P, s);
    float R = kNone, m = kNone, l = 0.0f, lvs_top = -3.0e38f;
    bool have = false;
#pragma unroll 1
    for (int i = two ? 0 : t; i < s.n; i += two ? 1 : 2) {
      const uint32_t g = base + i;
      const Note& note = S.note[g % kNotes];
      const int end = (s.first + i + 1) * kKeys;
      if (!await(&S.note_full[g % kNotes], g / kNotes & 1)) return false;
      lvs_top = fmaxf(lvs_top, note.lvs_hi);
      const uint32_t dead = note.dead;
      const bool wide = lvs_top - note.lvs_lo > kSpread;
      const bool masked = __any_sync(0xFFFFFFFFu, row.len < end) || dead != 0;
      const bool scaled = CAP || masked || wide || note.odd != 0;
      if (!await(&S.s_full[t], tiles++ & 1)) return false;
      tc_fence_after();
      if (row.idle) {   // (whatever the weights of rows that are none are)
        __syncwarp();
        if (lane < 2) mbar_arrive(&S.p_full[t][lane]);
        have = true;
        continue;
      }
      if (scaled) {   // scores are brought to units of log2 one by one, and written back
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t u[32];
          float* x = reinterpret_cast<float*>(u);
          tmem_ld32(s_at + c * 32, u);
          const float2 ks = *reinterpret_cast<const float2*>(&note.ks[c * 2]);
          const float f0 = ks.x * row.f, f1 = ks.y * row.f;
          tc_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; k += 2) split(mul2(pair(x[k], x[k + 1]), k < 16 ? pair(f0, f0) : pair(f1, f1)), x[k], x[k + 1]);
          if (CAP) cap32(x, cap2, inv_cap);
          if (masked) {
            const int left = row.len - (end - kKeys) - c * 32;
            const uint32_t gone = (dead >> (c * 2) & 1u ? 0xFFFFu : 0u) | (dead >> (c * 2 + 1) & 1u ? 0xFFFF0000u : 0u);
            const uint32_t seen = (left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u) & ~gone;
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = seen >> k & 1u ? x[k] : -INFINITY;
          }
          tmem_st32(s_at + c * 32, u);
        }
        tc_wait_st();
      }
      uint32_t u[128];
      float* x = reinterpret_cast<float*>(u);
#pragma unroll
      for (int c = 0; c < 128; c += 32) tmem_ld32(s_at + c, u + c);
      float f[kTileBlocks], lvs[kTileBlocks];
#pragma unroll
      for (int b = 0; b < kTileBlocks; b += 4) {
        *reinterpret_cast<float4*>(f + b) = *reinterpret_cast<const float4*>(&note.ks[b]);
        *reinterpret_cast<float4*>(lvs + b) = *reinterpret_cast<const float4*>(&note.lvs[b]);
      }
#pragma unroll
      for (int b = 0; b < kTileBlocks; ++b) f[b] = scaled ? 1.0f : f[b] * row.f;
      tc_wait_ld();
      float top_x = -INFINITY, top_w = -INFINITY;
#pragma unroll
      for (int b = 0; b < kTileBlocks; b += 2) {
        const float y0 = largest16(x + b * 16) * f[b], y1 = largest16(x + b * 16 + 16) * f[b + 1];
        top_x = max3(top_x, y0, y1);
        top_w = max3(top_w, y0 + lvs[b], y1 + lvs[b + 1]);
      }
      if (__any_sync(0xFFFFFFFFu, !(top_w <= R + kLag) || top_x > m + kSumLag)) {
        const float to = !(top_w <= R + kLag) ? fmaxf(R, top_w) : R, by = ex2(R - to);   // (what other rows do does not move a row)
        R = to;
        if (have && __any_sync(0xFFFFFFFFu, by != 1.0f)) rescale(o_at, by);
        const float sum_to = top_x > m + kSumLag ? top_x : m;
        l *= ex2(m - sum_to);
        m = sum_to;
      }
      const float ref = R - kLift;
      if (wide) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld32(s_at + c * 32, v);
          tc_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; ++k) l += ex2(__uint_as_float(v[k]) - m);
        }
      }
      float sums[kTileBlocks];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t p[32];
#pragma unroll
        for (int b = h * 4; b < h * 4 + 4; ++b) {
          const uint64_t f2 = pair(f[b], f[b]), c2 = pair(lvs[b] - ref, lvs[b] - ref);
          uint64_t sum = 0;
#pragma unroll
          for (int k = b * 16; k < b * 16 + 16; k += 2) {
            float a, d;
            split(fma2(pair(x[k], x[k + 1]), f2, c2), a, d);
            a = ex2(a);
            d = ex2(d);
            sum = add2(sum, pair(a, d));
            p[(k - h * 64) / 2] = round2<JF_DTYPE_FP16>(a, d);
          }
          float a, d;
          split(sum, a, d);
          sums[b] = a + d;
        }
        tmem_st32(s_at + h * 32, p);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.p_full[t][h]);
      }
      if (!wide) {
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b) l = fmaf(sums[b], ex2(ref - lvs[b] - m), l);
      }
      have = true;
    }
    // the next queries, then the partial result
    const int64_t piece = (static_cast<int64_t>(blockIdx.x) + s.item) * 2 + t;
    const bool any = s.n > 0, idle = row.idle;
    base += s.n;
    more = next_segment(P, s);
    if (more) row = load_query(s);
    if (have) {
      if (!await(&S.o_full[t], ends++ & 1)) return false;
      tc_fence_after();
      float* out = P.part_o + (piece * kRows + r) * JF_HEAD_DIM;
#pragma unroll 1
      for (int c = idle ? 4 : 0; c < 4; ++c) {
        uint32_t o[32];
        tmem_ld32(o_at + c * 32, o);
        tc_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; k += 8)
          asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + c * 32 + k), JF_W8(o, k) : "memory");
      }
      tc_fence_before();
    }
    if (any) P.part_ml[piece * kRows + r] = make_float4(R - kLift, m, l, 0.0f);
    __syncwarp();
  }
  return true;
}

template <int DT, int CODES, bool CAP>
__global__ void __launch_bounds__(kThreads, 1) block8_shared_kernel(const __grid_constant__ SharedParams P) {
  extern __shared__ unsigned char raw[];
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);   // (known to be the same for all lanes)
  const uint32_t up = (1024u - (smem_u32(raw) & 1023u)) & 1023u;
  unsigned char *smem = raw + up, *kv = smem + 2 * kTileBytes, *staged = kv + 4 * kTileBytes;
  Shared& S = *reinterpret_cast<Shared*>(staged + kStaged * kCodeBytes);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.q_full[i], 4);
      mbar_init(&S.k_full[i], 2);
      mbar_init(&S.v_full[i], 2);
      mbar_init(&S.k_empty[i], 1);
      mbar_init(&S.v_empty[i], 1);
      mbar_init(&S.s_full[i], 1);
      mbar_init(&S.p_full[i][0], 4);
      mbar_init(&S.p_full[i][1], 4);
      mbar_init(&S.o_full[i], 1);
    }
    for (int i = 0; i < kStaged; ++i) {
      mbar_init(&S.code_full[i], 1);
      mbar_init(&S.code_empty[i], 2);
    }
    for (int i = 0; i < kNotes; ++i) mbar_init(&S.note_full[i], 1);
    mbar_init(&S.products_done, 1);
    S.begin = static_cast<int>(static_cast<int64_t>(blockIdx.x) * P.units / gridDim.x);
    S.end = static_cast<int>((static_cast<int64_t>(blockIdx.x) + 1) * P.units / gridDim.x);
    fence_barrier_init();
  }
  if (warp == 10) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&S.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  pdl_wait();
  pdl_trigger();
  // every role ends by itself, a wait that ran out included; the error is recorded by whoever meets it
  bool ok = true;
  if (warp < 8) {
    regs_inc<kRowRegs>();
    ok = soften<DT, CAP>(P, S, smem + (warp >> 2) * kTileBytes, tmem, warp >> 2);
  } else {
    regs_dec<kRoleRegs>();
    if (warp < 10) {
      ok = convert<CODES>(P, S, kv, staged);
    } else if (warp == 10) {
      ok = multiply(P, S, smem_u32(smem), smem_u32(kv), tmem);
      if (elect_one()) tc_commit(&S.products_done);
      __syncwarp();
      ok &= await(&S.products_done, 0);
    } else {
      int sent = 0;
      ok = load(P, S, staged, sent);
      ok &= arrived(S, sent);
    }
  }
  if (!ok) report_status(P.status, JF_ERR_TIMEOUT);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 10) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---- host -----------------------------------------------------------------------------------------

struct Plan {
  int G, row_tiles, pairs, tiles, grid;
  int64_t items, units;
  uint64_t own, o_bytes, bytes;   // scratch of the own positions' part, of the outputs, of all
};
// Units of a thread block at least: 8 to 64 sequences over 2048 positions, 32 / 8 heads, take 29 to 42 us with one, 26 to 40 with two, 34 to 54 with six.
constexpr int kLeastUnits = 2;
// Whether the shared positions go through the tensor cores, or once for every sequence through block8_attn.cu's kernel.  That one takes 5.5e-4 us
// for a block of a KV head and a sequence (1.5 times that for every 16 query heads, where a KV head has more than 8).  This one takes what three such readings
// do for a block of a KV head, what 10 more do for a sequence's own positions and its part of the join, and 7 us of launches and loads.  Back to back, us,
// decode kernel / this one:
//   32 / 8 heads, 65536 positions: 1 sequence 34 / 67, 2 48 / 68, 3 65 / 68, 4 82 / 68, 8 168 / 69; 16384: 3 25 / 26, 4 29 / 26, 8 51 / 27;
//     4096: 4 14 / 16, 8 22 / 19, 16 33 / 23; 32 over 1024 27 / 26, over 2048 42 / 29; 64 over 512 23 / 28, over 1024 49 / 29; 128 over 512 39 / 41, 256 over 256 56 / 61
//   8 / 1: 4 over 131072 30 / 33, 8 over 32768 21 / 24, over 65536 30 / 27, 16 over 16384 21 / 22, over 32768 30 / 29; 64 over 2048 14 / 22, 256 over 1024 39 / 27
//   32 / 2: 1 over 131072 27 / 41, 2 41 / 43, 3 57 / 45; 3 over 65536 34 / 34, 4 41 / 34; 8 over 8192 20 / 22, over 16384 27 / 26; 16 over 4096 22 / 23, over 8192 30 / 24
//   40 / 1: 1 over 131072 34 / 37, 2 over 32768 23 / 26, over 65536 34 / 30, 4 over 16384 23 / 20, 16 over 4096 25 / 23
// From cold caches a call takes 7 to 9 us more by the decode kernel, 8 to 20 by this one.
constexpr int64_t kFewBlocks = 13500;

bool tensor_form(int B, int H_q, int H_kv, int max_S, int shared_blocks) {
  const int seen = std::min(shared_blocks, (max_S - 1) / JF_BLOCK_SIZE + 1), G = H_q / H_kv;
  const int64_t halves = int64_t{B} * (G <= 8 ? 2 : 3 * ((G + 15) / 16));   // of a reading
  return H_kv * ((halves - 6) * seen - 20ll * B) > 2 * kFewBlocks;
}

bool make_plan(int B, int H_q, int H_kv, int max_S, int shared_blocks, Plan& p) {
  if (B <= 0 || H_q <= 0 || H_kv <= 0 || max_S <= 0 || H_q % H_kv != 0 || shared_blocks < 0 || shared_blocks > INT32_MAX / JF_BLOCK_SIZE - 1) return false;
  p = Plan{};
  if (!tensor_form(B, H_q, H_kv, max_S, shared_blocks)) {
    p.bytes = block8_attn_workspace(B, H_q, H_kv, max_S);
    return p.bytes > 0;
  }
  p.G = H_q / H_kv;
  const int64_t rows = int64_t{B} * p.G;
  if (rows > INT32_MAX / 2 || H_q > 65535 || B > 65535) return false;
  p.row_tiles = static_cast<int>((rows + kRows - 1) / kRows);
  p.pairs = (p.row_tiles + 1) / 2;
  const int seen = std::min(shared_blocks, (max_S - 1) / JF_BLOCK_SIZE + 1);   // of the shared blocks
  p.tiles = (seen + kTileBlocks - 1) / kTileBlocks;
  p.items = int64_t{H_kv} * p.pairs;
  p.units = p.items * p.tiles;
  if (p.units > INT32_MAX / 2) return false;
  p.grid = static_cast<int>(std::min<int64_t>(num_sms(), (p.units + kLeastUnits - 1) / kLeastUnits));
  p.own = (block8_attn_workspace(B, H_q, H_kv, std::max(max_S - shared_blocks * JF_BLOCK_SIZE, 1)) + 255) / 256 * 256;
  if (p.own == 0) return false;
  const uint64_t part_rows = static_cast<uint64_t>(p.grid + p.items) * 2 * kRows;
  p.o_bytes = part_rows * JF_HEAD_DIM * sizeof(float);
  p.bytes = p.own + p.o_bytes + part_rows * sizeof(float4);
  return true;
}

template <int DT, int CODES, bool CAP> jf_status_t launch(const SharedParams& P, int grid, cudaStream_t s) {
  auto* kernel = block8_shared_kernel<DT, CODES, CAP>;
  static const int regs = [] {
    cudaFuncAttributes f{};
    return cudaFuncGetAttributes(&f, block8_shared_kernel<DT, CODES, CAP>) == cudaSuccess ? f.numRegs : 0;
  }();
  // (a warpgroup that asks for more than the block has waits for good)
  if (regs * kThreads < 128 * (2 * kRowRegs + kRoleRegs)) return JF_ERR_UNSUPPORTED;
  JF_ENSURE_SMEM(kernel, kSmemBytes);
  JF_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(kThreads), kSmemBytes, s, P));
  return JF_OK;
}
template <int DT, int CODES> jf_status_t launch(const SharedParams& P, int grid, cudaStream_t s) {
  return P.softcap > 0.0f ? launch<DT, CODES, true>(P, grid, s) : launch<DT, CODES, false>(P, grid, s);
}

}  // namespace
}  // namespace jf

extern "C" uint64_t jf_block8_shared_workspace_bytes(int32_t B, int32_t H_q, int32_t H_kv, int32_t max_S, int32_t shared_blocks) {
  jf::Plan p;
  return jf::make_plan(B, H_q, H_kv, max_S, shared_blocks, p) ? p.bytes : 0;
}

extern "C" jf_status_t jf_block8_shared_attn(const jf_block8_shared_args* a, jf_stream_t stream) {
  using namespace jf;
  if (!a) return JF_ERR_ARG;
  jf_block8_attn_args at = a->attn;
  if (a->shared_blocks < 0 || at.window != 0 || at.prefix_lens || at.alibi_slopes) return JF_ERR_ARG;
  if (a->shared_blocks > INT32_MAX / JF_BLOCK_SIZE - 1) return JF_ERR_UNSUPPORTED;
  if (at.B > 0 && a->shared_blocks > 0 && !a->shared_table) return JF_ERR_ARG;
  Block8Source from;
  from.shared = a->shared_table;
  from.shared_blocks = a->shared_blocks;
  from.shared_i32 = a->shared_is_i32 != 0;
  at.workspace_bytes = UINT64_MAX;   // (what is needed is another plan's)
  const jf_status_t checked = block8_attend(&at, from, stream, false);
  if (checked != JF_OK || at.B == 0) return checked;
  at.workspace_bytes = a->attn.workspace_bytes;
  Plan p;
  if (!make_plan(at.B, at.H_q, at.H_kv, at.max_S, a->shared_blocks, p)) return JF_ERR_ARG;
  if (at.workspace_bytes < p.bytes || !aligned(at.workspace, kWorkspaceAlign)) return JF_ERR_WORKSPACE;
  const auto s = static_cast<cudaStream_t>(stream);
  SharedParams P{};
  jf_status_t st = wait_record(s, &P.status);   // (an error of an earlier call is returned whichever way this one goes)
  if (st != JF_OK) return st;
  if (!tensor_form(at.B, at.H_q, at.H_kv, at.max_S, a->shared_blocks)) return block8_attend(&at, from, stream, true);
  P.q = static_cast<const uint16_t*>(at.q);
  P.k_data = static_cast<const uint8_t*>(at.k_data);
  P.v_data = static_cast<const uint8_t*>(at.v_data);
  P.k_scales = at.k_scales;
  P.v_scales = at.v_scales;
  P.table = a->shared_table;
  P.seq_lens = at.seq_lens;
  P.part_o = reinterpret_cast<float*>(static_cast<char*>(at.workspace) + p.own);
  P.part_ml = reinterpret_cast<float4*>(static_cast<char*>(at.workspace) + p.own + p.o_bytes);
  P.num_blocks = at.num_blocks;
  P.units = static_cast<int32_t>(p.units);
  P.H_q = at.H_q;
  P.G = p.G;
  P.rows = at.B * p.G;
  P.row_tiles = p.row_tiles;
  P.pairs = p.pairs;
  P.tiles = p.tiles;
  P.blocks = std::min(a->shared_blocks, p.tiles * kTileBlocks);
  P.max_S = at.max_S;
  P.scale = at.attn_scale;
  P.softcap = at.softcap;
  P.i32 = a->shared_is_i32 != 0;
  if (at.q_dtype == JF_DTYPE_BF16)
    st = at.codes == JF_CODES_INT8 ? launch<JF_DTYPE_BF16, JF_CODES_INT8>(P, p.grid, s) : launch<JF_DTYPE_BF16, JF_CODES_E4M3>(P, p.grid, s);
  else
    st = at.codes == JF_CODES_INT8 ? launch<JF_DTYPE_FP16, JF_CODES_INT8>(P, p.grid, s) : launch<JF_DTYPE_FP16, JF_CODES_E4M3>(P, p.grid, s);
  if (st != JF_OK) return st;
  from = Block8Source{};
  from.behind = a->shared_blocks;
  from.part_o = P.part_o;
  from.part_ml = P.part_ml;
  from.units = p.units;
  from.grid = p.grid;
  from.tiles = p.tiles;
  from.pairs = p.pairs;
  from.row_tiles = p.row_tiles;
  at.workspace_bytes = p.own;
  return block8_attend(&at, from, stream, true);
}
