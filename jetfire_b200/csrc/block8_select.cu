// Which blocks of the 8-bit cache a query attends to: the best by a cheap score, and the first and last of the sequence.
//
//   score_j = max_h qs_h * sum_c (min(q8_hc, 0) lo_jc + max(q8_hc, 0) hi_jc) * unit_j,   q8_h = rint(q_h / qs_h), qs_h = amax|q_h| / 127
//
// is an upper bound of q.k over block j, but for the query's rounding: lo and hi are the lowest and highest code of channel c in the
// block (block bounds, kept by the append), unit_j what a code of 1 stands for, h runs through the query heads of
// the KV head.  The sum is one integer product of 256 channels, exact, on the tensor cores (mma.s8: 16 blocks x 8
// heads); it and the two factors that follow, in fp32, have one value whatever the order, so the choice is the same on every run and in every plain form.  Ties go to the lower block.
//
// A cluster shares a (sequence, KV head): each of its blocks scores its part of the row and keeps the scores, as integers ordered like
// them, in its shared memory.  The limit above which a block is chosen is found by histograms over the range that it
// must lie in, each thread block's counted from the top and added up by all from the others' shared memory; one
// pass of 512 bins leaves a handful of scores in the bin that holds the limit.  Those are passed to all and ranked against
// one another.  The list comes out in rising order, so that what reads it adds up in the same order always.
//
// Bound: latency.  260 bytes a (block, KV head) are read once, in a few dependent trips (length, table, bounds), then three
// meetings of the cluster.
#include "block8.cuh"

#include <algorithm>
#include <type_traits>

namespace jf {
namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kBins = kThreads;                   // a bin a thread
constexpr int kMaxCluster = 16;                   // (above 8 where the device takes it)
constexpr int kMaxKeys = 16384;                   // scores of a block, 64 KB
constexpr int kCandidates = 512;
constexpr uint32_t kForced = 0xFFFFFFFFu;         // first and last blocks
constexpr uint32_t kNothing = 0x007FFFFFu;        // the key of -inf
constexpr float kSmallest = 0x1p-100f;

struct SelectParams {
  const uint16_t* q;
  const float* k_scales;
  const int8_t* bounds;
  const void* table;
  const int32_t* seq_lens;
  int32_t* chosen;
  int64_t num_blocks, bt_stride;
  int32_t H_q, H_kv, G, max_len, top, first, last;
  float unit;
  bool bt_i32;
};

struct Shared {
  uint32_t count[kBins];                          // of this block, from the bin to the highest
  uint32_t lo, hi;                                // least and largest key of this block (forced ones and -inf left out)
  uint32_t candidates[kCandidates];
  int scan[kWarps];
  float step[8];
  alignas(16) int8_t q8[8][272];                  // min(q, 0), max(q, 0); rows on different banks
};

__device__ __forceinline__ uint32_t load1_from(uint32_t at) {
  uint32_t x;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ void store1_to(uint32_t at, uint32_t x) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(x) : "memory"); }

// Sum of `x` over the threads before this one, and over all (the whole block; `total` may be used as soon as this returns).
__device__ __forceinline__ int scan_block(Shared& S, int x, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += v;
  }
  __syncthreads();
  if (lane == 31) S.scan[warp] = sum;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const int v = S.scan[w];
    if (w < warp) before += v;
    total += v;
  }
  return before + sum - x;
}

// The queries of heads h0 .. h0 + 8 in 8 bits.  A head with an element that is no number scores nothing, as one beyond the group.
template <int DT> __device__ __forceinline__ void round_queries(const SelectParams& P, Shared& S, int64_t row0, int h0) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp >= 8) return;
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, amax = 0.0f;
  bool odd = h0 + warp >= P.G;
  if (!odd) {
    const uint2 w = *reinterpret_cast<const uint2*>(P.q + (row0 + h0 + warp) * JF_HEAD_DIM + lane * 4);
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
__global__ void __launch_bounds__(kThreads) block8_select_kernel(const __grid_constant__ SelectParams P) {
  extern __shared__ uint32_t keys[];
  __shared__ Shared S;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x, ranks = gridDim.x, kvh = blockIdx.y, b = blockIdx.z;
  pdl_wait();
  pdl_trigger();
  const int len = max(0, min(P.seq_lens[b], P.max_len)), n = (len + JF_BLOCK_SIZE - 1) / JF_BLOCK_SIZE;
  const int64_t row = static_cast<int64_t>(b) * P.H_kv + kvh;
  int32_t* chosen = P.chosen + row * P.top;
  if (n <= P.top) {   // all of them (the whole cluster)
    for (int i = rank * kThreads + threadIdx.x; i < P.top; i += ranks * kThreads) chosen[i] = i < n ? i : -1;
    return;
  }
  // ---- scores: this block's part of the row, 16 at a time by a warp
  const int part = ((n + ranks - 1) / ranks + 15) / 16 * 16, begin = min(rank * part, n), mine = min(begin + part, n) - begin;
  const int64_t head_row = static_cast<int64_t>(kvh) * P.num_blocks, table_row = static_cast<int64_t>(b) * P.bt_stride;
  const int64_t row0 = static_cast<int64_t>(b) * P.H_q + kvh * P.G;
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
  for (int h0 = 0; h0 < P.G; h0 += 8) {
    if (h0 > 0) __syncthreads();
    round_queries<DT>(P, S, row0, h0);
    __syncthreads();
    uint4 q[4];       // head g, 16 of its 256 products' channels t * 16 .., 64 + t * 16 .., ...
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const uint4*>(&S.q8[g][(t + 4 * i) * 16]);
    const float step0 = S.step[2 * t], step1 = S.step[2 * t + 1];
    for (int at = warp * 16; at < mine; at += kWarps * 16) {
      uint4 x[2][4];
      float unit[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int j = begin + at + g + 8 * r;
        int64_t id = -1;
        if (j < begin + mine) id = P.bt_i32 ? static_cast<const int32_t*>(P.table)[table_row + j] : static_cast<const int64_t*>(P.table)[table_row + j];
        const bool is = id >= 0 && id < P.num_blocks;
        unit[r] = is ? P.k_scales[head_row + id] : __int_as_float(0x7FC00000);
        const uint4* from = reinterpret_cast<const uint4*>(P.bounds + (head_row + (is ? id : 0)) * (2 * JF_HEAD_DIM)) + t;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[r][i] = is ? __ldg(from + 4 * i) : make_uint4(0, 0, 0, 0);
      }
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
        const int i = at + g + 8 * r, j = begin + i;
        if (t == 0 && i < mine) {
          uint32_t key = score != score ? kNothing : float_order_key(score);
          if (h0 > 0) key = max(key, keys[i]);
          if (j < P.first || j >= n - P.last) key = kForced;
          keys[i] = key;
          if (h0 + 8 >= P.G && key != kForced && key > kNothing) {
            lo = min(lo, key);
            hi = max(hi, key);
          }
        }
      }
    }
  }
  lo = __reduce_min_sync(0xFFFFFFFFu, lo);
  hi = __reduce_max_sync(0xFFFFFFFFu, hi);
  if (threadIdx.x == 0) { S.lo = 0xFFFFFFFFu; S.hi = 0; }
  __syncthreads();
  if (lane == 0 && lo <= hi) {
    atomicMin(&S.lo, lo);
    atomicMax(&S.hi, hi);
  }
  cluster_sync();
  // ---- the limit: of the keys in [from, above] the highest `need` are taken, those beyond `above` too
  lo = 0xFFFFFFFFu;
  hi = 0;
  for (int r = 0; r < ranks; ++r) {
    lo = min(lo, load1_from(of_rank(&S.lo, r)));
    hi = max(hi, load1_from(of_rank(&S.hi, r)));
  }
  const int each = (mine + kThreads - 1) / kThreads, k0 = min(static_cast<int>(threadIdx.x) * each, mine), k1 = min(k0 + each, mine);
  int need = P.top - P.first - P.last, in = 0, in_before = 0, total;
  uint32_t from = lo, above = hi;
  bool ranked = false;
  auto none_left = [&] { from = above = kNothing; };   // what scores nothing, the first of it
  if (need == 0) from = above = kForced - 1;           // (no key is that)
  else if (lo > hi) none_left();
  else
    for (;;) {
      int shift = 0;
      while ((above - from) >> shift >= kBins) ++shift;
      S.count[threadIdx.x] = 0;
      __syncthreads();
      for (int i = k0; i < k1; ++i) {
        const uint32_t k = keys[i];
        if (k >= from && k <= above) atomicAdd(&S.count[(k - from) >> shift], 1u);
      }
      __syncthreads();
      const int bin = kBins - 1 - static_cast<int>(threadIdx.x), here = static_cast<int>(S.count[bin]);   // the highest first
      S.count[bin] = static_cast<uint32_t>(scan_block(S, here, total) + here);
      cluster_sync();
      int sum = 0;
      for (int r = 0; r < ranks; ++r) sum += static_cast<int>(load1_from(of_rank(&S.count[threadIdx.x], r)));
      const int reached = __syncthreads_count(sum >= need);   // bins from which on upwards there are `need` and more
      int over = 0, at_least = 0;
      in_before = 0;
      for (int r = 0; r < ranks; ++r) {
        const int x = static_cast<int>(load1_from(of_rank(&S.count[max(reached - 1, 0)], r)));
        const int y = reached > 0 && reached < kBins ? static_cast<int>(load1_from(of_rank(&S.count[reached], r))) : 0;
        at_least += x;
        over += y;
        if (r < rank) in_before += x - y;
      }
      if (reached == 0) {   // (in the first round only)
        need -= at_least;
        none_left();
        break;
      }
      need -= over;
      in = at_least - over;
      from += static_cast<uint32_t>(reached - 1) << shift;
      above = min(above, from + ((1u << shift) - 1u));
      ranked = in > need && shift > 0;
      if (!ranked || in <= kCandidates) break;
      cluster_sync();   // everybody has read the counts
    }
  // ---- the list.  Candidates, the keys in [from, above], are numbered in the order of their blocks, through all ranks.
  int c = 0, o = 0, c_all, o_all;
  for (int i = k0; i < k1; ++i) {
    const uint32_t k = keys[i];
    c += k >= from && k <= above;
    o += k > above;
  }
  const int c_at = scan_block(S, c, c_all);
  scan_block(S, o, o_all);
  if (ranked) {
    int at = in_before + c_at;
    for (int i = k0; i < k1; ++i) {
      const uint32_t k = keys[i];
      if (k < from || k > above) continue;
      for (int r = 0; r < ranks; ++r) store1_to(of_rank(&S.candidates[at], r), k);
      ++at;
    }
  }
  if (threadIdx.x == 0) {
    S.lo = static_cast<uint32_t>(c_all);
    S.hi = static_cast<uint32_t>(o_all);
  }
  cluster_sync();
  int c_before = 0, o_before = 0;
  for (int r = 0; r < rank; ++r) {
    c_before += static_cast<int>(load1_from(of_rank(&S.lo, r)));
    o_before += static_cast<int>(load1_from(of_rank(&S.hi, r)));
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // nothing of the others is read any more
  int c_taken = min(c_before, need);
  if (ranked) {
    bool take = false;
    if (static_cast<int>(threadIdx.x) < in) {
      const uint32_t k = S.candidates[threadIdx.x];
      int better = 0;
      for (int i = 0; i < in; ++i) {
        const uint32_t x = S.candidates[i];
        better += x > k || (x == k && i < static_cast<int>(threadIdx.x));
      }
      take = better < need;
    }
    S.count[threadIdx.x] = take;
    c_taken = __syncthreads_count(take && static_cast<int>(threadIdx.x) < c_before);
  }
  auto takes = [&](uint32_t k, int& number) {   // number: of the next candidate
    if (k > above) return true;
    if (k < from) return false;
    const int a = number++;
    return ranked ? S.count[a] != 0 : a < need;
  };
  int number = c_before + c_at, taken = 0;
  for (int i = k0; i < k1; ++i) taken += takes(keys[i], number);
  int at = o_before + c_taken + scan_block(S, taken, total);
  number = c_before + c_at;
  for (int i = k0; i < k1; ++i)
    if (takes(keys[i], number)) chosen[at++] = begin + i;
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Thread blocks that share a row: as many as leave a warp 16 of its blocks, while two of them find room on every multiprocessor; more
// where the row's scores do not fit fewer.
int ranks_of(int64_t rows, int64_t blocks) {
  int c = 1;
  while (c < kMaxCluster && int64_t{c} * kWarps * 16 < blocks && (2 * c * rows <= 2 * num_sms() || blocks > int64_t{c} * kMaxKeys)) c *= 2;
  return c;
}

}  // namespace
}  // namespace jf

extern "C" uint64_t jf_block8_sparse_workspace_bytes(int32_t B, int32_t H_q, int32_t H_kv, int32_t max_S, int32_t top_blocks) {
  if (top_blocks <= 0) return 0;
  return jf::block8_attn_workspace(B, H_q, H_kv, static_cast<int>(std::min<int64_t>(max_S, int64_t{top_blocks} * JF_BLOCK_SIZE)));
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
  if (blocks > int64_t{kMaxCluster} * kMaxKeys) return JF_ERR_UNSUPPORTED;
  SelectParams P{};
  P.q = static_cast<const uint16_t*>(at.q);
  P.k_scales = at.k_scales;
  P.bounds = a->bounds;
  P.table = at.block_table;
  P.seq_lens = at.seq_lens;
  P.chosen = a->chosen;
  P.num_blocks = at.num_blocks;
  P.bt_stride = at.bt_stride;
  P.H_q = at.H_q; P.H_kv = at.H_kv; P.G = at.H_q / at.H_kv;
  P.max_len = static_cast<int32_t>(longest);
  P.top = a->top_blocks; P.first = a->first_blocks; P.last = a->last_blocks;
  P.unit = at.codes == JF_CODES_INT8 ? 1.0f : 448.0f / 127.0f;
  P.bt_i32 = at.bt_is_i32 != 0;
  const int ranks = blocks <= a->top_blocks ? 1 : ranks_of(int64_t{at.B} * at.H_kv, blocks);
  const int64_t keys = blocks <= a->top_blocks ? 0 : ((blocks + ranks - 1) / ranks + 15) / 16 * 16;
  auto launch = [&](auto dt) {
    auto* kernel = block8_select_kernel<decltype(dt)::value>;
    JF_ENSURE_SMEM(kernel, kMaxKeys * 4);
    if (ranks > 8) JF_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ranks, at.H_kv, at.B);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(keys) * 4;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    JF_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, P));
    return static_cast<jf_status_t>(JF_OK);
  };
  const jf_status_t st = at.q_dtype == JF_DTYPE_BF16 ? launch(std::integral_constant<int, JF_DTYPE_BF16>())
                                                     : launch(std::integral_constant<int, JF_DTYPE_FP16>());
  return st == JF_OK ? block8_attend(&at, from, stream, true) : st;
}
