// Quantise-on-append into the cache of 8-bit codes with one scale per block of 16 positions and KV head.
//
// With s the scale of a block, int8 rows hold rint(x / s) for s = amax / 127, e4m3 rows hold x / s rounded to
// e4m3 for s the smallest power of two with amax <= 448 s (a power of two costs a floating-point code nothing,
// and a scale that grows later only moves its exponent).  A block that already holds positions of its sequence
// keeps max(old, new) as its scale; where it grew, the old codes are rounded once more, to code * (old / new).
// The scale of a block therefore depends on every row that the call brings to it, so one warp owns a (block,
// head, side): it holds the block's rows in registers -- half a warp a row, 16 bytes a lane, eight rounds --
// takes the maximum over them, and writes codes and scale once.  Which rows those are follows from the
// sequences' bounds (a token leads its block when it is its sequence's first or stands on a multiple of 16), so
// there is one launch, no scratch and no order among the writers.
//
// With a rotation (jf_block8_append_rotary) a key's pair of channels (a, b) becomes (a cos - b sin, b cos + a sin) on the way, in fp32,
// products and sums rounded one by one, and is quantised from there: no rounding to 16 bits in between.  The same launch rotates
// the step's queries.  With block bounds the warp that owns a block of K leaves the lowest and highest code of every channel, over
// all rows the block then holds: rounding keeps the order, so they are found among the scaled numbers and rounded once.
//
// Rotated: 8192 tokens, 64 / 8 heads, bf16 -> int8 with bounds (324 MB) 96 us from cold caches = 3.4 TB/s: the queries' rows alone 58, K and V
// alone 53.  K's staged warps have 96 registers and spill 180 to 192 bytes a thread, and V's and the
// queries' run with the same 20 warps a multiprocessor: 44 % of the issue slots are used, it is latency that is left.  Four sequences of a token, 32 / 8 heads,
// 3.8 us back to back.  Bounds without a rotation go through the same kernels: 8192 tokens, 8 KV heads, 36 us from cold caches and 14.7 back to back (without
// bounds 18 and 8.3; e4m3 37 and 15.5), 64 single tokens 11.7 and 3.9 (9.5 and 3.1; e4m3 12.9 and 5.3).
//
// Bound: memory -- 2 bytes read and 1 written per element.  8192 tokens, 8 KV heads, bf16 -> int8 (50 MB): 13.6 us = 3.7 TB/s, 16384: 22.1 us = 4.6
// TB/s; a warp's start (bounds, length, block id, rows: four dependent trips) and 700 instructions a block are what is left.
#include "jf_common.cuh"
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

namespace jf {
namespace {

constexpr int kWarps = 4;
constexpr float kSmallest = 0x1p-100f;   // keeps 1 / scale finite

struct AppendSide {
  const uint16_t* x;
  int64_t stride_t, stride_h;
  uint8_t* data;
  float* scales;
};
struct Rotation {
  const void *positions, *cos_sin;   // cos_sin null: none
  int64_t rows;                      // of the table
  const uint16_t* q;
  int64_t q_stride_t, q_stride_h;
  uint16_t* q_out;
  int8_t* bounds;                    // null: none
  int32_t H_q, rot, q_rounds, k_blocks, append_blocks;   // k_blocks: thread blocks of K, V's come behind them, the queries' behind append_blocks
  bool pos_i32, interleaved, table_f32;
};
struct AppendParams {
  AppendSide side[2];
  const int32_t* start;       // n_seqs + 1
  const int32_t* seq_lens;
  const void* table;
  int64_t bt_stride, num_blocks;
  int32_t T, H, n_seqs, max_blocks, chunk;
  bool bt_i32;
};

// Larger magnitudes of two pairs; NaN wins, the signs are left over.
template <int DT> __device__ __forceinline__ uint32_t absmax2(uint32_t a, uint32_t b) {
  uint32_t d;
  if (DT == JF_DTYPE_BF16) asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <int DT> __device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if (DT == JF_DTYPE_BF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
}

__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void split(uint64_t x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }

// Four scaled values (two pairs) as codes; none of them leaves the range.  int8: adding 1.5 * 2^23 rounds to an integer, half to
// even, and leaves its two's complement in the low byte.
template <int CODES> __device__ __forceinline__ uint32_t encode4(uint64_t ab, uint64_t cd) {
  float a, b, c, d;
  if (CODES == JF_CODES_INT8) {
    const uint64_t magic = pair(12582912.0f, 12582912.0f);
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(ab) : "l"(magic));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(cd) : "l"(magic));
    split(ab, a, b);
    split(cd, c, d);
    return prmt(prmt(__float_as_uint(a), __float_as_uint(b), 0x0040u), prmt(__float_as_uint(c), __float_as_uint(d), 0x0040u), 0x5410u);
  }
  split(ab, a, b);
  split(cd, c, d);
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}
// NaN as 0, what lies beyond the largest code as that
template <int CODES> __device__ __forceinline__ float tame(float v) {
  constexpr float top = CODES == JF_CODES_INT8 ? 127.0f : 448.0f;
  return v != v ? 0.0f : fminf(fmaxf(v, -top), top);
}

template <int CODES> __device__ __forceinline__ float decode1(uint32_t byte) {
  if (CODES == JF_CODES_INT8) return static_cast<float>(static_cast<int8_t>(byte));
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

// The scale that rows of this largest magnitude ask for.
template <int CODES> __device__ __forceinline__ float scale_for(float amax) {
  amax = fmaxf(amax, kSmallest);
  if (CODES == JF_CODES_INT8) return __fdiv_rn(amax, 127.0f);
  // 448 = 1.75 * 2^8: a mantissa above 1.75 needs the next exponent
  return __uint_as_float((((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - 8u) << 23);
}

template <bool VEC> __device__ __forceinline__ uint4 load8(const uint16_t* p) {
  if constexpr (VEC) return __ldg(reinterpret_cast<const uint4*>(p));
  else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __ldg(p + 2 * i) | static_cast<uint32_t>(__ldg(p + 2 * i + 1)) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---- rotation ---------------------------------------------------------------------------------

// cos of the angles of a lane's eight channels, and sin with the sign of the other channel of the pair.
struct Turn { float c[8], s[8]; };
// N neighbouring numbers of the table (`at` counts them; a multiple of N)
template <int DT, int N> __device__ __forceinline__ void table_row(const Rotation& R, int64_t at, float* x) {
  if (R.table_f32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(R.cos_sin) + at + i));
      x[i] = f.x; x[i + 1] = f.y; x[i + 2] = f.z; x[i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(R.cos_sin) + at + i));
      unpack2<DT>(w.x, x[i], x[i + 1]);
      unpack2<DT>(w.y, x[i + 2], x[i + 3]);
    }
  }
}
// A token whose position is not in the table gets angles that are no numbers.
__device__ __forceinline__ int64_t position_of(const Rotation& R, int64_t token) {
  return R.pos_i32 ? static_cast<const int32_t*>(R.positions)[token] : static_cast<const int64_t*>(R.positions)[token];
}
template <int DT> __device__ __forceinline__ Turn turn_of(const Rotation& R, int64_t pos, int col) {
  Turn t;
  const bool is = pos >= 0 && pos < R.rows;
  const int half = R.rot / 2;
  if (!is || col >= R.rot) {
#pragma unroll
    for (int k = 0; k < 8; ++k) t.c[k] = t.s[k] = __int_as_float(0x7FC00000);
  } else if (R.interleaved) {
    float c[4], s[4];
    table_row<DT, 4>(R, pos * R.rot + col / 2, c);
    table_row<DT, 4>(R, pos * R.rot + half + col / 2, s);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      t.c[2 * k] = t.c[2 * k + 1] = c[k];
      t.s[2 * k] = -s[k];
      t.s[2 * k + 1] = s[k];
    }
  } else {
    const int at = col < half ? col : col - half;
    table_row<DT, 8>(R, pos * R.rot + at, t.c);
    table_row<DT, 8>(R, pos * R.rot + half + at, t.s);
#pragma unroll
    for (int k = 0; k < 8; ++k) t.s[k] = col < half ? -t.s[k] : t.s[k];
  }
  return t;
}
// The same of a token whose row of the table stands in shared memory, in fp32 (NaN where it is not in the table).
__device__ __forceinline__ Turn turn_of(const Rotation& R, const float* row, int col) {
  Turn t;
  const int half = R.rot / 2;
  if (col >= R.rot) {
#pragma unroll
    for (int k = 0; k < 8; ++k) t.c[k] = t.s[k] = 0.0f;
  } else if (R.interleaved) {
    const float4 c = *reinterpret_cast<const float4*>(row + col / 2), s = *reinterpret_cast<const float4*>(row + half + col / 2);
    const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      t.c[2 * k] = t.c[2 * k + 1] = cs[k];
      t.s[2 * k] = -sn[k];
      t.s[2 * k + 1] = sn[k];
    }
  } else {
    const int at = col < half ? col : col - half;
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      *reinterpret_cast<float4*>(t.c + k) = *reinterpret_cast<const float4*>(row + at + k);
      *reinterpret_cast<float4*>(t.s + k) = *reinterpret_cast<const float4*>(row + half + at + k);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) t.s[k] = col < half ? -t.s[k] : t.s[k];
  }
  return t;
}
// A lane's eight channels of a row, rotated; all lanes of the warp (a pair's halves lie in two lanes of the half warp).
template <int DT> __device__ __forceinline__ void rotate(const Rotation& R, const uint4& raw, const Turn& t, int col, float* v) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  const int lane = threadIdx.x & 31, over = R.rot >> 4;
  const int from = R.interleaved ? lane : (lane & 16) | ((lane & 15) < over ? ((lane & 15) + over) & 15 : ((lane & 15) - over) & 15);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float a, b, x, y;
    unpack2<DT>(w[k], a, b);
    unpack2<DT>(__shfl_sync(0xFFFFFFFFu, w[k], from), x, y);
    if (R.interleaved) { x = b; y = a; }
    v[2 * k] = col < R.rot ? __fadd_rn(__fmul_rn(a, t.c[2 * k]), __fmul_rn(x, t.s[2 * k])) : a;
    v[2 * k + 1] = col < R.rot ? __fadd_rn(__fmul_rn(b, t.c[2 * k + 1]), __fmul_rn(y, t.s[2 * k + 1])) : b;
  }
}

// The queries' rows: a warp per token and 2 * q_rounds heads, half a warp a row.
template <int DT, bool VEC> __device__ __forceinline__ void rotate_queries(const AppendParams& P, const Rotation& R, int64_t item) {
  const int lane = threadIdx.x & 31, col = (lane & 15) * 8, per = 2 * R.q_rounds, chunks = (R.H_q + per - 1) / per;
  const int64_t t = item / chunks;
  if (t >= P.T) return;
  const int last = P.start[P.n_seqs];
  const int h0 = static_cast<int>(item - t * chunks) * per + (lane >> 4);
  const uint16_t* from = R.q + t * R.q_stride_t + col;
  const int64_t pos = position_of(R, t);
  auto rows = [&](auto n_tag) {
    constexpr int N = decltype(n_tag)::value;
    uint4 raw[N], then[N];
    auto read = [&](uint4* to, int h) {
#pragma unroll
      for (int i = 0; i < N; ++i) to[i] = h + 2 * i < R.H_q ? load8<VEC>(from + (h + 2 * i) * R.q_stride_h) : make_uint4(0, 0, 0, 0);
    };
    read(raw, h0);      // (on their way while the angles are looked up)
    const Turn turn = turn_of<DT>(R, pos, col);
    if (t >= last) return;   // rows of no sequence
#pragma unroll 1
    for (int h = h0;;) {
      const bool more = N > 1 && h + 2 * N < h0 + per;
      if (more) read(then, h + 2 * N);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float v[8];
        rotate<DT>(R, raw[i], turn, col, v);
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (DT == JF_DTYPE_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(v[2 * k + 1]), "f"(v[2 * k]));
          else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(v[2 * k + 1]), "f"(v[2 * k]));
        }
        if (h + 2 * i < R.H_q) *reinterpret_cast<uint4*>(R.q_out + (t * R.H_q + h + 2 * i) * JF_HEAD_DIM + col) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      if (!more) break;
      h += 2 * N;
#pragma unroll
      for (int i = 0; i < N; ++i) raw[i] = then[i];
    }
  };
  if (R.q_rounds == 1) rows(std::integral_constant<int, 1>());
  else rows(std::integral_constant<int, 4>());
}

// ---- blocks -----------------------------------------------------------------------------------

template <int CODES> __device__ __forceinline__ void decode8(uint2 c, float* v) {
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = decode1<CODES>((k < 4 ? c.x : c.y) >> 8 * (k & 3) & 255u);
}
template <int CODES> __device__ __forceinline__ uint2 encode8(const float* v) {
  return make_uint2(encode4<CODES>(pair(v[0], v[1]), pair(v[2], v[3])), encode4<CODES>(pair(v[4], v[5]), pair(v[6], v[7])));
}

// What write_block does for a side that is rotated, or whose bounds are kept; `at`: the block's place in the table; the warp's lanes hold the
// positions of the tokens from `first` on, `turns` their angles where there are more than a few.  The block's rows, their angles, its id, and what it holds of earlier rows are all asked for before one of
// them is waited for.  Sixteen rows are rotated twice, once for their maximum and once to be stored (64 values a lane held in between
// left room for 16 warps on a multiprocessor); up to two, a token of a decode step, once.
template <int DT, int CODES, bool VEC>
__device__ __forceinline__ void write_block_rotated(const AppendParams& P, const Rotation& R, const AppendSide& S, int h, int t, int cnt, int r,
                                                    int64_t at, int first, int64_t pos, const float* turns) {
  const int lane = threadIdx.x & 31, half = lane >> 4, col = (lane & 15) * 8;
  const uint16_t* x = S.x + static_cast<int64_t>(t) * S.stride_t + h * S.stride_h + col;
  auto body = [&](auto rounds_tag) {
    constexpr int N = decltype(rounds_tag)::value;
    const int64_t id = P.bt_i32 ? static_cast<const int32_t*>(P.table)[at] : static_cast<const int64_t*>(P.table)[at];
    uint4 raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = 2 * i + half;
      raw[i] = row < cnt ? load8<VEC>(x + row * S.stride_t) : make_uint4(0, 0, 0, 0);
    }
    auto angles = [&](int i) {
      const int token = t - first + min(2 * i + half, cnt - 1);
      return turns ? turn_of(R, turns + token * R.rot, col) : turn_of<DT>(R, __shfl_sync(0xFFFFFFFFu, pos, token), col);
    };
    Turn turn;
    auto rotated = [&](int i, float* v) {
      if (R.cos_sin) {
        if (N > 1) turn = angles(i);
        rotate<DT>(R, raw[i], turn, col, v);
      } else {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) unpack2<DT>(w[k], v[2 * k], v[2 * k + 1]);
      }
    };
    if (N == 1 && R.cos_sin) turn = angles(0);
    if (id < 0 || id >= P.num_blocks) return;
    float* scale_at = S.scales + h * P.num_blocks + id;
    uint8_t* rows = S.data + ((h * P.num_blocks + id) * JF_BLOCK_SIZE) * JF_HEAD_DIM + col;
    float old = r > 0 ? *scale_at : 0.0f;
    uint2 was[8];      // earlier rows of the block (of a few tokens: of many, they are the exception and looked at when their turn comes)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (N == 1 && 2 * i + half < r) was[i] = *reinterpret_cast<const uint2*>(rows + (2 * i + half) * JF_HEAD_DIM);
    if (!(old > 0.0f && old < __int_as_float(0x7F800000))) old = 0.0f;   // never written: nothing to keep
    float top = 0.0f, v[8];
    bool wild = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      rotated(i, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) {   // infinities and NaN do not count
        const float a = 2 * i + half < cnt ? fabsf(v[k]) : 0.0f;
        const bool fine = a < __int_as_float(0x7F800000);
        wild |= !fine;
        top = fmaxf(top, fine ? a : 0.0f);
      }
    }
    wild = __any_sync(0xFFFFFFFFu, wild);
    top = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top)));   // (not negative: ordered as their bits are)
    const float s = fmaxf(old, scale_for<CODES>(top)), inv = __frcp_rn(s);
    float lo[8], hi[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      lo[k] = __int_as_float(0x7F800000);
      hi[k] = -lo[k];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = 2 * i + half;
      if (N > 1) rotated(i, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = __fmul_rn(v[k], inv);
      if (wild) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = tame<CODES>(v[k]);
      }
      if (row < cnt) {
        *reinterpret_cast<uint2*>(rows + (r + row) * JF_HEAD_DIM) = encode8<CODES>(v);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          lo[k] = fminf(lo[k], v[k]);
          hi[k] = fmaxf(hi[k], v[k]);
        }
      }
    }
    const bool grew = s != old;
    if (r > 0 && (grew || R.bounds)) {
      const float ratio = __fdiv_rn(old, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = 2 * i + half;
        if (row >= r) continue;
        float w[8];
        if (N > 1) was[i] = *reinterpret_cast<const uint2*>(rows + row * JF_HEAD_DIM);
        decode8<CODES>(was[i], w);
        if (grew) {
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = tame<CODES>(__fmul_rn(w[k], ratio));
          *reinterpret_cast<uint2*>(rows + row * JF_HEAD_DIM) = encode8<CODES>(w);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          lo[k] = fminf(lo[k], w[k]);
          hi[k] = fmaxf(hi[k], w[k]);
        }
      }
    }
    __syncwarp();
    if (R.bounds) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        lo[k] = fminf(lo[k], __shfl_xor_sync(0xFFFFFFFFu, lo[k], 16));
        hi[k] = fmaxf(hi[k], __shfl_xor_sync(0xFFFFFFFFu, hi[k], 16));
        if (half) lo[k] = hi[k];        // half a warp for each of the two
      }
      uint2 code = encode8<CODES>(lo);
      if (CODES == JF_CODES_E4M3) {     // in units of 448 / 127 scales, outwards
        float w[8];
        decode8<CODES>(code, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float u = __fdiv_rn(w[k] * 127.0f, 448.0f);
          w[k] = half ? ceilf(u) : floorf(u);
        }
        code = encode8<JF_CODES_INT8>(w);
      }
      *reinterpret_cast<uint2*>(R.bounds + ((h * P.num_blocks + id) * 2 + half) * JF_HEAD_DIM + col) = code;
    }
    __syncwarp();
    if (lane == 0 && grew) *scale_at = s;
  };
  if (cnt <= 2) body(std::integral_constant<int, 1>());
  else body(std::integral_constant<int, 8>());
}

// Rows t .. t + cnt of the call into rows r .. r + cnt of block `id`; r rows of its sequence are there already.
template <int DT, int CODES, bool VEC>
__device__ __forceinline__ void write_block(const AppendParams& P, const AppendSide& S, int h, int t, int cnt, int r, int64_t id) {
  const int lane = threadIdx.x & 31, half = lane >> 4, col = (lane & 15) * 8;
  const uint16_t* x = S.x + static_cast<int64_t>(t) * S.stride_t + h * S.stride_h + col;
  uint4 raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 2 * i + half;
    raw[i] = row < cnt ? load8<VEC>(x + row * S.stride_t) : make_uint4(0, 0, 0, 0);
  }
  float* scale_at = S.scales + h * P.num_blocks + id;
  float old = r > 0 ? *scale_at : 0.0f;
  if (!(old > 0.0f && old < __int_as_float(0x7F800000))) old = 0.0f;   // never written: nothing to keep
  constexpr uint32_t kInf = DT == JF_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = absmax2<DT>(m, absmax2<DT>(absmax2<DT>(raw[i].x, raw[i].y), absmax2<DT>(raw[i].z, raw[i].w)));
  m &= 0x7FFF7FFFu;
  uint32_t top = __reduce_max_sync(0xFFFFFFFFu, max(m & 0xFFFFu, m >> 16));
  const bool clean = top < kInf;
  if (!clean) {   // infinities and NaN do not count
    uint32_t f = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t a = w[k] & 0x7FFFu, b = w[k] >> 16 & 0x7FFFu;
        f = max(f, max(a < kInf ? a : 0u, b < kInf ? b : 0u));
      }
    }
    top = __reduce_max_sync(0xFFFFFFFFu, f);
  }
  const float s = fmaxf(old, scale_for<CODES>(Elem<DT>::to_f32(static_cast<uint16_t>(top))));
  const float inv = __frcp_rn(s);
  const uint64_t inv2 = pair(inv, inv);
  uint8_t* rows = S.data + ((h * P.num_blocks + id) * JF_BLOCK_SIZE) * JF_HEAD_DIM + col;
  // Finite values stay in range: |x| <= amax, and amax * fp32(1 / fp32(amax / 127)) is within 2^-22 of 127.  The products are
  // rounded to fp32 before the codes are (not fused with what follows).
  auto store = [&](auto wild) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = 2 * i + half;
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      uint64_t v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a, b;
        unpack2<DT>(w[k], a, b);
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v[k]) : "l"(pair(a, b)), "l"(inv2));
        if (decltype(wild)::value) {
          split(v[k], a, b);
          v[k] = pair(tame<CODES>(a), tame<CODES>(b));
        }
      }
      if (row < cnt) *reinterpret_cast<uint2*>(rows + (r + row) * JF_HEAD_DIM) = make_uint2(encode4<CODES>(v[0], v[1]), encode4<CODES>(v[2], v[3]));
    }
  };
  if (clean) store(std::false_type());
  else store(std::true_type());
  if (r > 0 && s != old) {
    const float ratio = __fdiv_rn(old, s);
    for (int row = half; row < r; row += 2) {
      uint2* p = reinterpret_cast<uint2*>(rows + row * JF_HEAD_DIM);
      const uint2 c = *p;
      uint64_t v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t two = (k < 2 ? c.x : c.y) >> 16 * (k & 1);
        v[k] = pair(tame<CODES>(__fmul_rn(decode1<CODES>(two & 255u), ratio)), tame<CODES>(__fmul_rn(decode1<CODES>(two >> 8 & 255u), ratio)));
      }
      *p = make_uint2(encode4<CODES>(v[0], v[1]), encode4<CODES>(v[2], v[3]));
    }
  }
  __syncwarp();
  if (lane == 0 && s != old) *scale_at = s;
}

// A warp per (chunk of tokens, head, side): it writes every block whose first token of the call stands in the chunk.  With a rotation the
// warps of a thread block take heads of K of one chunk, whose tokens' angles they bring to shared memory together (kStaged); of chunks of one
// token each warp finds its own, in a kernel whose registers are not held down for the sake of more blocks on a multiprocessor
// (four sequences of a token 9.8 us from cold caches and not 13.0, 8192 tokens 98 and not 102).
enum { kPlain, kDirect, kStaged };
constexpr int kTurns = 31;   // tokens: the chunk's and 15 more
template <int DT, int CODES, bool VEC, int ROTARY>   // VEC: rows may be read 16 bytes at a time
__global__ void __launch_bounds__(kWarps * 32, ROTARY == kStaged ? 5 : ROTARY == kDirect ? 1 : 0) block8_append_kernel(const __grid_constant__ AppendParams P, const __grid_constant__ Rotation R) {
  __shared__ __align__(16) float sm_turns[ROTARY == kStaged ? kTurns * JF_HEAD_DIM : 1];
  const float* turns = nullptr;
  const int lane = threadIdx.x & 31;
  int side, h, t;
  if constexpr (ROTARY) {
    if (static_cast<int>(blockIdx.x) >= R.append_blocks) {
      pdl_wait();
      pdl_trigger();
      rotate_queries<DT, VEC>(P, R, static_cast<int64_t>(blockIdx.x - R.append_blocks) * kWarps + (threadIdx.x >> 5));
      return;
    }
    int64_t from;
    if (static_cast<int>(blockIdx.x) < R.k_blocks) {
      const int per = (P.H + kWarps - 1) / kWarps;
      side = 0;
      h = static_cast<int>(blockIdx.x) % per * kWarps + (threadIdx.x >> 5);
      from = static_cast<int64_t>(static_cast<int>(blockIdx.x) / per) * P.chunk;
    } else {
      const int item = static_cast<int>(blockIdx.x - R.k_blocks) * kWarps + static_cast<int>(threadIdx.x >> 5);
      side = 1;
      h = item % P.H;
      from = static_cast<int64_t>(item / P.H) * P.chunk;
    }
    if (from >= P.T) { pdl_wait(); return; }
    t = static_cast<int>(from);
    pdl_wait();
    pdl_trigger();
    if (ROTARY == kStaged && side == 0 && R.cos_sin) {
      const int pieces = R.rot / 4, all = min(P.chunk + 15, P.T - t) * pieces;
#pragma unroll 4
      for (int i = threadIdx.x; i < all; i += kWarps * 32) {
        const int token = i / pieces, piece = (i - token * pieces) * 4;
        const int64_t pos = position_of(R, t + token);
        float x[4];
        if (pos >= 0 && pos < R.rows) table_row<DT, 4>(R, pos * R.rot + piece, x);
        else x[0] = x[1] = x[2] = x[3] = __int_as_float(0x7FC00000);
        *reinterpret_cast<float4*>(sm_turns + token * R.rot + piece) = make_float4(x[0], x[1], x[2], x[3]);
      }
      __syncthreads();
      turns = sm_turns;
    }
    if (h >= P.H) return;
  } else {
    const uint32_t item = blockIdx.x * kWarps + (threadIdx.x >> 5), rest = item >> 1;
    side = item & 1;
    h = static_cast<int>(rest % static_cast<uint32_t>(P.H));
    const int64_t from = static_cast<int64_t>(rest / static_cast<uint32_t>(P.H)) * P.chunk;
    if (from >= P.T) { pdl_wait(); return; }
    t = static_cast<int>(from);
    pdl_wait();
    pdl_trigger();
  }
  const int first = t, end = min(t + P.chunk, P.T);
  const AppendSide& S = P.side[side];
  // positions of the tokens that may be in the chunk's blocks: its own and 15 more
  int64_t pos_of_lane = 0;
  if constexpr (ROTARY)
    if (side == 0 && R.cos_sin && !turns) pos_of_lane = position_of(R, min(t + lane, P.T - 1));
  // sequences that end at or before t
  int s = 0;
  for (int i = lane; i < P.n_seqs; i += 32) s += P.start[i + 1] <= t;
  s = __reduce_add_sync(0xFFFFFFFFu, s);
  while (t < end) {
    while (s < P.n_seqs && P.start[s + 1] <= t) ++s;
    if (s >= P.n_seqs) return;
    const int a = P.start[s], b = min(P.start[s + 1], P.T);
    if (t < a) { t = a; continue; }                         // rows of no sequence
    const int len = P.seq_lens[s];
    int pos = len - (b - t);
    if (pos < 0) { t += min(b - t, -pos); continue; }       // rows before the sequence's start
    const int step = t == a ? 0 : (JF_BLOCK_SIZE - (pos & 15)) & 15;
    t += step;
    pos += step;
    if (t >= b) { t = b; continue; }                        // the rest of this sequence's rows belong to an earlier leader
    if (t >= end) break;
    const int r = pos & 15, cnt = min(JF_BLOCK_SIZE - r, b - t);
    const int64_t blk = pos >> 4;
    if (blk < P.max_blocks) {
      const int64_t at = s * P.bt_stride + blk;
      if (ROTARY && side == 0) {
        write_block_rotated<DT, CODES, VEC>(P, R, S, h, t, cnt, r, at, first, pos_of_lane, turns);
      } else {
        const int64_t id = P.bt_i32 ? static_cast<const int32_t*>(P.table)[at] : static_cast<const int64_t*>(P.table)[at];
        if (id >= 0 && id < P.num_blocks) write_block<DT, CODES, VEC>(P, S, h, t, cnt, r, id);
      }
    }
    t += cnt;
  }
}

// Launches what both entry points check; R null: neither rotation nor bounds.
jf_status_t launch_append(AppendParams& P, const Rotation* R, int dtype, int codes, cudaStream_t s) {
  const bool there = P.n_seqs > 0 && P.max_blocks > 0 && P.num_blocks > 0;
  bool vec = aligned(P.side[0].x, 16) && aligned(P.side[1].x, 16) &&
             (P.side[0].stride_t | P.side[0].stride_h | P.side[1].stride_t | P.side[1].stride_h) % 8 == 0;
  const int64_t mean = P.T / std::max(P.n_seqs, 1);
  // Tokens a warp looks through.  16 suit one prompt (8192 tokens, 8 KV heads: 13.7 us, with chunks of four 17.2), but sequences of one
  // token would wait for one another there (64 of them beside a prompt of 2048: 31.5 us, with chunks of four 10.9), and
  // which sequences are long is not known here.
  P.chunk = P.n_seqs < 4 ? 16 : mean >= 8 ? 4 : mean >= 2 ? 2 : 1;
  const int64_t items = there ? (P.T + int64_t{P.chunk} - 1) / P.chunk * P.H * 2 : 0;
  int64_t blocks = (items + kWarps - 1) / kWarps;
  if (items > INT32_MAX) return JF_ERR_UNSUPPORTED;
  Rotation rot{};
  if (R) {
    rot = *R;
    const int64_t chunks_of = there ? (P.T + int64_t{P.chunk} - 1) / P.chunk : 0, k = chunks_of * ((P.H + kWarps - 1) / kWarps);
    blocks = k + (chunks_of * P.H + kWarps - 1) / kWarps;
    if (blocks > INT32_MAX / 2) return JF_ERR_UNSUPPORTED;
    rot.k_blocks = static_cast<int32_t>(k);
    rot.append_blocks = static_cast<int32_t>(blocks);
    if (rot.q && P.n_seqs > 0) {
      vec &= aligned(rot.q, 16) && (rot.q_stride_t | rot.q_stride_h) % 8 == 0;
      // Pairs of rows that a warp goes through with the angles of their token: as many as leave warps enough (8192 tokens, 64 heads: 4 129 us, 16 114)
      const int64_t pairs = static_cast<int64_t>(P.T) * rot.H_q / 2, enough = 64ll * num_sms();
      rot.q_rounds = pairs >= 16 * enough ? 16 : pairs >= 4 * enough ? 4 : 1;
      const int64_t chunks = (rot.H_q + 2 * rot.q_rounds - 1) / (2 * rot.q_rounds);
      blocks += (P.T * chunks + kWarps - 1) / kWarps;
    }
  }
  if (blocks == 0) return JF_OK;
  if (blocks > INT32_MAX) return JF_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks)), block(kWarps * 32);
  auto launch = [&](auto dt, auto code) {
    constexpr int D = decltype(dt)::value, C = decltype(code)::value;
    if (R && P.chunk > 1)
      return vec ? launch_pdl(block8_append_kernel<D, C, true, kStaged>, grid, block, 0, s, P, rot)
                 : launch_pdl(block8_append_kernel<D, C, false, kStaged>, grid, block, 0, s, P, rot);
    if (R)
      return vec ? launch_pdl(block8_append_kernel<D, C, true, kDirect>, grid, block, 0, s, P, rot)
                 : launch_pdl(block8_append_kernel<D, C, false, kDirect>, grid, block, 0, s, P, rot);
    return vec ? launch_pdl(block8_append_kernel<D, C, true, kPlain>, grid, block, 0, s, P, rot)
               : launch_pdl(block8_append_kernel<D, C, false, kPlain>, grid, block, 0, s, P, rot);
  };
  using Bf16 = std::integral_constant<int, JF_DTYPE_BF16>;
  using Fp16 = std::integral_constant<int, JF_DTYPE_FP16>;
  using Int8 = std::integral_constant<int, JF_CODES_INT8>;
  using E4m3 = std::integral_constant<int, JF_CODES_E4M3>;
  if (dtype == JF_DTYPE_BF16)
    JF_CUDA_TRY(codes == JF_CODES_INT8 ? launch(Bf16(), Int8()) : launch(Bf16(), E4m3()));
  else
    JF_CUDA_TRY(codes == JF_CODES_INT8 ? launch(Fp16(), Int8()) : launch(Fp16(), E4m3()));
  return JF_OK;
}

}  // namespace
}  // namespace jf

extern "C" jf_status_t jf_block8_append(const void* key, const void* value, int32_t dtype, int64_t T, int32_t H_kv, int64_t k_stride_t,
                                        int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h, const int32_t* query_start_loc,
                                        const int32_t* seq_lens, int32_t n_seqs, const void* block_table, int32_t bt_is_i32,
                                        int64_t bt_stride, int32_t max_blocks, int32_t codes, void* k_data, float* k_scales, void* v_data,
                                        float* v_scales, int64_t num_blocks, jf_stream_t stream) {
  using namespace jf;
  if (T < 0 || H_kv <= 0 || n_seqs < 0 || max_blocks < 0 || num_blocks < 0 || T > INT32_MAX - 64) return JF_ERR_ARG;
  if ((dtype != JF_DTYPE_BF16 && dtype != JF_DTYPE_FP16) || (codes != JF_CODES_INT8 && codes != JF_CODES_E4M3)) return JF_ERR_ARG;
  if (T == 0 || n_seqs == 0 || max_blocks == 0 || num_blocks == 0) return JF_OK;
  if (!key || !value || !query_start_loc || !seq_lens || !block_table || !k_data || !v_data || !k_scales || !v_scales) return JF_ERR_ARG;
  if (!aligned(k_data, 8) || !aligned(v_data, 8) || !aligned(k_scales, 4) || !aligned(v_scales, 4)) return JF_ERR_ARG;
  AppendParams P{};
  P.side[0] = {static_cast<const uint16_t*>(key), k_stride_t, k_stride_h, static_cast<uint8_t*>(k_data), k_scales};
  P.side[1] = {static_cast<const uint16_t*>(value), v_stride_t, v_stride_h, static_cast<uint8_t*>(v_data), v_scales};
  P.start = query_start_loc;
  P.seq_lens = seq_lens;
  P.table = block_table;
  P.bt_stride = bt_stride;
  P.num_blocks = num_blocks;
  P.T = static_cast<int32_t>(T);
  P.H = H_kv;
  P.n_seqs = n_seqs;
  P.max_blocks = max_blocks;
  P.bt_i32 = bt_is_i32 != 0;
  return launch_append(P, nullptr, dtype, codes, static_cast<cudaStream_t>(stream));
}

extern "C" jf_status_t jf_block8_append_rotary(const jf_block8_rotary_args* a, jf_stream_t stream) {
  using namespace jf;
  if (!a) return JF_ERR_ARG;
  if (a->T < 0 || a->T > INT32_MAX - 64 || a->H_kv <= 0 || a->H_q < 0 || a->H_q > 65535 || a->n_seqs < 0 || a->max_blocks < 0 || a->num_blocks < 0)
    return JF_ERR_ARG;
  if ((a->dtype != JF_DTYPE_BF16 && a->dtype != JF_DTYPE_FP16) || (a->codes != JF_CODES_INT8 && a->codes != JF_CODES_E4M3)) return JF_ERR_ARG;
  if (a->H_q > 0 && !a->cos_sin) return JF_ERR_ARG;
  if (a->cos_sin && (a->rot < 16 || a->rot > JF_HEAD_DIM || a->rot % 16 != 0 || a->table_rows < 0 || a->table_rows > INT64_MAX / 1024 ||
                     !aligned(a->cos_sin, 16)))
    return JF_ERR_ARG;
  if (a->T == 0 || a->n_seqs == 0) return JF_OK;
  if (!a->query_start_loc || !a->seq_lens || (a->cos_sin && !a->positions)) return JF_ERR_ARG;
  if (a->H_q > 0 && (!a->query || !a->query_out || !aligned(a->query_out, 16))) return JF_ERR_ARG;
  if (a->max_blocks > 0 && a->num_blocks > 0) {
    if (!a->key || !a->value || !a->block_table || !a->k_data || !a->v_data || !a->k_scales || !a->v_scales) return JF_ERR_ARG;
    if (!aligned(a->k_data, 8) || !aligned(a->v_data, 8) || !aligned(a->k_scales, 4) || !aligned(a->v_scales, 4) || !aligned(a->bounds, 8))
      return JF_ERR_ARG;
  }
  AppendParams P{};
  P.side[0] = {static_cast<const uint16_t*>(a->key), a->k_stride_t, a->k_stride_h, static_cast<uint8_t*>(a->k_data), a->k_scales};
  P.side[1] = {static_cast<const uint16_t*>(a->value), a->v_stride_t, a->v_stride_h, static_cast<uint8_t*>(a->v_data), a->v_scales};
  P.start = a->query_start_loc;
  P.seq_lens = a->seq_lens;
  P.table = a->block_table;
  P.bt_stride = a->bt_stride;
  P.num_blocks = a->num_blocks;
  P.T = static_cast<int32_t>(a->T);
  P.H = a->H_kv;
  P.n_seqs = a->n_seqs;
  P.max_blocks = a->max_blocks;
  P.bt_i32 = a->bt_is_i32 != 0;
  Rotation R{};
  R.positions = a->positions;
  R.cos_sin = a->cos_sin;
  R.rows = a->table_rows;
  R.q = a->H_q > 0 ? static_cast<const uint16_t*>(a->query) : nullptr;
  R.q_stride_t = a->q_stride_t;
  R.q_stride_h = a->q_stride_h;
  R.q_out = static_cast<uint16_t*>(a->query_out);
  R.bounds = a->bounds;
  R.H_q = a->H_q;
  R.rot = a->rot;
  R.pos_i32 = a->positions_i32 != 0;
  R.interleaved = a->interleaved != 0;
  R.table_f32 = a->table_f32 != 0;
  return launch_append(P, a->cos_sin || a->bounds ? &R : nullptr, a->dtype, a->codes, static_cast<cudaStream_t>(stream));
}
