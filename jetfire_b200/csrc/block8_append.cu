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
// Bound: memory -- 2 bytes read and 1 written per element.  8192 tokens, 8 KV heads, bf16 -> int8 (50 MB): 13.6 us = 3.7 TB/s, 16384: 22.1 us = 4.6
// TB/s; a warp's start (bounds, length, block id, rows: four dependent trips) and 700 instructions a block are what is left.
#include "jf_common.cuh"
#include <cuda_fp8.h>

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

// A warp per (chunk of tokens, head, side): it writes every block whose first token of the call stands in the chunk.
template <int DT, int CODES, bool VEC>   // VEC: rows may be read 16 bytes at a time
__global__ void __launch_bounds__(kWarps * 32) block8_append_kernel(const __grid_constant__ AppendParams P) {
  const int lane = threadIdx.x & 31;
  const uint32_t item = blockIdx.x * kWarps + (threadIdx.x >> 5), rest = item >> 1;
  const int side = item & 1, h = static_cast<int>(rest % static_cast<uint32_t>(P.H));
  const int64_t from = static_cast<int64_t>(rest / static_cast<uint32_t>(P.H)) * P.chunk;
  if (from >= P.T) { pdl_wait(); return; }
  int t = static_cast<int>(from);
  const int end = min(t + P.chunk, P.T);
  const AppendSide& S = P.side[side];
  pdl_wait();
  pdl_trigger();
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
      const int64_t id = P.bt_i32 ? static_cast<const int32_t*>(P.table)[at] : static_cast<const int64_t*>(P.table)[at];
      if (id >= 0 && id < P.num_blocks) write_block<DT, CODES, VEC>(P, S, h, t, cnt, r, id);
    }
    t += cnt;
  }
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
  const bool vec = aligned(key, 16) && aligned(value, 16) && (k_stride_t | k_stride_h | v_stride_t | v_stride_h) % 8 == 0;
  const int64_t mean = T / n_seqs;
  // Tokens a warp looks through.  16 suit one prompt (8192 tokens, 8 KV heads: 13.7 us, with chunks of four 17.2), but sequences of one
  // token would wait for one another there (64 of them beside a prompt of 2048: 31.5 us, with chunks of four 10.9), and
  // which sequences are long is not known here.
  P.chunk = n_seqs < 4 ? 16 : mean >= 8 ? 4 : mean >= 2 ? 2 : 1;
  const int64_t items = (T + P.chunk - 1) / P.chunk * H_kv * 2, blocks = (items + kWarps - 1) / kWarps;
  if (items > INT32_MAX) return JF_ERR_UNSUPPORTED;
  const auto s = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks)), block(kWarps * 32);
  auto launch = [&](auto dt, auto code) {
    constexpr int D = decltype(dt)::value, C = decltype(code)::value;
    return vec ? launch_pdl(block8_append_kernel<D, C, true>, grid, block, 0, s, P) : launch_pdl(block8_append_kernel<D, C, false>, grid, block, 0, s, P);
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
