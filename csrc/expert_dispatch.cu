// Token rows sorted by expert and back.
//
//   order    pairs (token t, choice j) -> rows sorted by expert, earlier pairs first: offsets [E + 1],
//            slots [T, k] (row of the pair, -1 for a pair of no expert of [base, base + E)),
//            pairs [T k] (pair of the row, -1 past the last row)
//   gather   rows[slots[t, j]] = x[t]; rows past the last one are zero
//   combine  out[t] = residual[t] + sum_j w[t, j] y[slots[t, j]]      (fp32, in choice order, one rounding)
//   combine gradient  dy[slots[t, j]] = w[t, j] dout[t], dw[t, j] = <dout[t], y[slots[t, j]]>
//
// The gradient of gather is combine without weights.  Every kernel walks tokens and scatters through slots,
// so each token row is read once and no two writers share a row: no atomics, and the same bits every time.
// All but order are bound by HBM: one pass over the rows.
#include <cooperative_groups.h>

#include "launchers.h"
#include "common/sm100.cuh"
#include "common/rows.cuh"

namespace {
namespace cg = cooperative_groups;

// ----------------------------------------------------------------------------- order
// A stable counting sort in one launch: the CTAs of one cluster (1 to 8) take consecutive ranges of pairs, the
// warps of a CTA consecutive ranges of its range.  Pass 1 counts per warp (lanes of equal expert found by
// match_any, one of them adds: no atomics), the counts become starting rows (over experts, then CTAs through
// distributed shared memory, then warps), pass 2 hands out rows in the same order.
template <typename Id>
__global__ void __launch_bounds__(1024) expert_order_kernel(const Id* __restrict__ ids, int64_t id_stride, int k,
                                                            int n, int64_t base, int E, int32_t* __restrict__ offsets,
                                                            int32_t* __restrict__ slots,
                                                            int32_t* __restrict__ pairs) {
  extern __shared__ int32_t sm[];
  __shared__ int32_t wsum[32];
  const int W = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  int32_t* cnt = sm;           // [W][E]: counts, then the next row of (warp, expert)
  int32_t* tot = sm + W * E;   // [E]: this CTA's counts
  int32_t* start = tot + E;    // [E]: the expert's first row in this CTA
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  for (int i = tid; i < W * E; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  const int per = (((n + C * W - 1) / (C * W)) + 31) / 32 * 32;  // pairs of a warp
  const int lo = min((int64_t)n, (int64_t)(rank * W + warp) * per), hi = min((int64_t)n, (int64_t)lo + per);
  auto expert = [&](int i) -> int {
    if (i >= hi) return -1;
    const int64_t e = (int64_t)ids[(int64_t)(i / k) * id_stride + i % k] - base;
    return e >= 0 && e < E ? (int)e : -1;
  };
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int e = expert(i0 + lane);
    const unsigned m = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && lane == __ffs(m) - 1) cnt[warp * E + e] += __popc(m);
    __syncwarp();
  }
  __syncthreads();
  for (int e = tid; e < E; e += blockDim.x) {
    int run = 0;
    for (int w = 0; w < W; ++w) {
      const int c = cnt[w * E + e];
      cnt[w * E + e] = run;
      run += c;
    }
    tot[e] = run;
  }
  cl.sync();
  // experts' first rows: exclusive sums over E of the clusters' counts, blockDim.x experts at a time
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += blockDim.x) {
    const int e = e0 + tid;
    int all = 0, before = 0;
    if (e < E)
      for (int c = 0; c < C; ++c) {
        const int v = C == 1 ? tot[e] : *cl.map_shared_rank(tot + e, c);
        all += v;
        if (c < rank) before += v;
      }
    int inc = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int wbase = 0, block_sum = 0;
    for (int w = 0; w < W; ++w) {
      if (w < warp) wbase += wsum[w];
      block_sum += wsum[w];
    }
    if (e < E) {
      const int first = carry + wbase + inc - all;
      start[e] = first + before;
      if (rank == 0) offsets[e] = first;
    }
    carry += block_sum;
    __syncthreads();
  }
  if (rank == 0 && tid == 0) offsets[E] = carry;
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane, e = expert(i);
    const unsigned m = __match_any_sync(0xffffffffu, e);
    int row = -1;
    if (e >= 0) row = start[e] + cnt[warp * E + e] + __popc(m & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == __ffs(m) - 1) cnt[warp * E + e] += __popc(m);
    __syncwarp();
    if (i < hi) slots[i] = row;
    if (row >= 0) pairs[row] = i;
  }
  for (int i = carry + rank * blockDim.x + tid; i < n; i += C * blockDim.x) pairs[i] = -1;
  cl.sync();  // the other CTAs have read this one's counts
}

// ----------------------------------------------------------------------------- gather
// A pair's row exists; a slot outside the n rows (a table that expert_order did not make) has none.
__device__ __forceinline__ bool has_row(int r, int64_t n) { return r >= 0 && r < n; }

struct Plane {
  const uint8_t* src;
  int64_t src_stride;  // bytes
  uint8_t* dst;        // rows of `bytes`, contiguous
  int64_t bytes;
};

template <typename V>
__device__ __forceinline__ void gather_plane(const Plane& p, int64_t t, const int32_t* slot, int k, int64_t n,
                                             int64_t first, int64_t step) {
  const int64_t nv = p.bytes / sizeof(V);
  const V* s = reinterpret_cast<const V*>(p.src + t * p.src_stride);
  for (int64_t c = first; c < nv; c += step) {
    const V v = s[c];
    for (int j = 0; j < k; ++j) {
      const int r = slot[j];
      if (has_row(r, n)) reinterpret_cast<V*>(p.dst + (int64_t)r * p.bytes)[c] = v;
    }
  }
}
template <typename V>
__device__ __forceinline__ void zero_plane(const Plane& p, int64_t from, int64_t to, int64_t first, int64_t step) {
  // rows are contiguous: the tail is one range
  V* d = reinterpret_cast<V*>(p.dst + from * p.bytes);
  const int64_t nv = (to - from) * p.bytes / (int64_t)sizeof(V);
  V zero;
  memset(&zero, 0, sizeof(V));
  for (int64_t i = first; i < nv; i += step) d[i] = zero;
}

// Block (token, column part).  V: widest access that every row of plane 0 (rows) allows; S: of plane 1
// (the MXFP8 scales of the rows; null where there are none).
template <typename V, typename S>
__global__ void __launch_bounds__(256) expert_gather_kernel(const Plane rows_p, const Plane scales_p,
                                                            const int32_t* __restrict__ slots, int k, int64_t n,
                                                            const int32_t* __restrict__ offsets, int E) {
  const int64_t t = blockIdx.x;
  const int64_t first = (int64_t)blockIdx.y * blockDim.x + threadIdx.x, step = (int64_t)gridDim.y * blockDim.x;
  const int32_t* slot = slots + t * k;
  gather_plane<V>(rows_p, t, slot, k, n, first, step);
  if (scales_p.src) gather_plane<S>(scales_p, t, slot, k, n, first, step);
  const int64_t total = max(offsets[E], 0);
  if (total < n) {
    const int64_t at = (t * gridDim.y + blockIdx.y) * blockDim.x + threadIdx.x;
    const int64_t all = (int64_t)gridDim.x * gridDim.y * blockDim.x;
    zero_plane<V>(rows_p, total, n, at, all);
    if (scales_p.src) zero_plane<S>(scales_p, total, n, at, all);
  }
}

// ----------------------------------------------------------------------------- combine
// NV consecutive elements per access.
template <typename T, int NV>
__device__ __forceinline__ void load_n(const T* p, float (&v)[NV]) {
  if constexpr (NV == 1) {
    v[0] = rows::to_f<T>(*p);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < NV; i += 4) {
      const float4 f = *reinterpret_cast<const float4*>(p + i);
      v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
    }
  } else {
    rows::load8<T>(p, v);
  }
}
template <typename T, int NV>
__device__ __forceinline__ void store_n(T* p, const float (&v)[NV]) {
  if constexpr (NV == 1) {
    *p = rows::from_f<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < NV; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
    *reinterpret_cast<uint4*>(p) = rows::pack8<T>(v);
  }
}

constexpr int kBatch = 8;  // choices whose rows are in flight together

// Block (token, column part): thread c of the part sums its NV columns over the token's choices.
template <typename T, typename O, int NV>
__global__ void __launch_bounds__(256) expert_combine_kernel(const CombineArgs a) {
  const int64_t t = blockIdx.x;
  const int nv = a.width / NV;
  const int32_t* slot = a.slots + t * a.k;
  const float* wt = a.weights ? a.weights + t * a.ws : nullptr;
  const T* y = static_cast<const T*>(a.y);
  for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < nv; c += gridDim.y * blockDim.x) {
    float acc[NV];
    if (a.residual)
      load_n<O, NV>(static_cast<const O*>(a.residual) + t * a.rs + (int64_t)c * NV, acc);
    else
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[i] = 0.f;
    for (int j0 = 0; j0 < a.k; j0 += kBatch) {
      float v[kBatch][NV];
      float w[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int r = j0 + j < a.k ? slot[j0 + j] : -1;
        const bool here = has_row(r, a.T * a.k);
        // a pair without a row adds nothing, whatever its weight holds
        w[j] = here ? (wt ? wt[j0 + j] : 1.f) : 0.f;
        if (here)
          load_n<T, NV>(y + (int64_t)r * a.ys + (int64_t)c * NV, v[j]);
        else
#pragma unroll
          for (int i = 0; i < NV; ++i) v[j][i] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] = fmaf(w[j], v[j][i], acc[i]);
    }
    store_n<O, NV>(static_cast<O*>(a.out) + t * (int64_t)a.width + (int64_t)c * NV, acc);
  }
}

// Block per token: dout's columns are read once, every choice's y row once; the k dot products end in one
// block reduction per batch of choices.
template <typename T, typename O, int NV>
__global__ void __launch_bounds__(256) expert_combine_bwd_kernel(const CombineBwdArgs a) {
  __shared__ float red[kBatch][8];
  const int64_t t = blockIdx.x;
  const int nv = a.width / NV, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int32_t* slot = a.slots + t * a.k;
  const float* wt = a.weights + t * a.ws;
  const O* g = static_cast<const O*>(a.dout) + t * a.gs;
  const T* y = static_cast<const T*>(a.y);
  T* dy = static_cast<T*>(a.dy);
  const int64_t n = a.T * a.k;
  for (int j0 = 0; j0 < a.k; j0 += kBatch) {
    int r[kBatch];
    float w[kBatch], dot[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      r[j] = j0 + j < a.k ? slot[j0 + j] : -1;
      if (!has_row(r[j], n)) r[j] = -1;
      w[j] = r[j] >= 0 ? wt[j0 + j] : 0.f;
      dot[j] = 0.f;
    }
    for (int c = threadIdx.x; c < nv; c += blockDim.x) {
      float d[NV];
      load_n<O, NV>(g + (int64_t)c * NV, d);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (r[j] < 0) continue;
        float v[NV];
        if (a.dw) {
          load_n<T, NV>(y + (int64_t)r[j] * a.ys + (int64_t)c * NV, v);
#pragma unroll
          for (int i = 0; i < NV; ++i) dot[j] = fmaf(d[i], v[i], dot[j]);
        }
        if (dy) {
#pragma unroll
          for (int i = 0; i < NV; ++i) v[i] = w[j] * d[i];
          store_n<T, NV>(dy + (int64_t)r[j] * a.width + (int64_t)c * NV, v);
        }
      }
    }
    if (a.dw) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
        if (lane == 0) red[j][warp] = dot[j];
      }
      __syncthreads();
      if (threadIdx.x < kBatch && j0 + threadIdx.x < a.k) {
        float s = 0.f;
        for (int i = 0; i < warps; ++i) s += red[threadIdx.x][i];
        a.dw[t * a.k + j0 + threadIdx.x] = s;  // 0 for a pair without a row
      }
      __syncthreads();
    }
  }
  const int64_t total = max(a.offsets[a.E], 0);
  if (dy && total < n) {
    Plane p{nullptr, 0, reinterpret_cast<uint8_t*>(dy), (int64_t)a.width * (int64_t)sizeof(T)};
    const int64_t at = t * blockDim.x + threadIdx.x, all = (int64_t)gridDim.x * blockDim.x;
    if constexpr (NV == 1)
      zero_plane<T>(p, total, n, at, all);
    else
      zero_plane<uint4>(p, total, n, at, all);
  }
}

// Column parts of a token so that small batches still fill the GPU (about four blocks on each SM).
unsigned column_parts(int64_t tokens, int64_t accesses, int threads, int num_sms) {
  const int64_t most = (accesses + threads - 1) / threads;
  const int64_t want = (4 * (int64_t)num_sms + tokens - 1) / tokens;
  return (unsigned)(want < 1 ? 1 : want < most ? want : (most < 1 ? 1 : most));
}

template <typename V>
void gather_scales(const Plane& r, const Plane& s, const GatherArgs& a, cudaStream_t stream) {
  const int threads = r.bytes / (int64_t)sizeof(V) >= 256 ? 256 : 128;
  const dim3 grid((unsigned)a.T, column_parts(a.T, r.bytes / sizeof(V), threads, a.num_sms));
  const int64_t align = s.bytes | s.src_stride | reinterpret_cast<intptr_t>(s.src);
  if (!s.src || align % 16 == 0)
    expert_gather_kernel<V, uint4><<<grid, threads, 0, stream>>>(r, s, a.slots, a.k, a.T * a.k, a.offsets, a.E);
  else if (align % 4 == 0)
    expert_gather_kernel<V, uint32_t><<<grid, threads, 0, stream>>>(r, s, a.slots, a.k, a.T * a.k, a.offsets, a.E);
  else
    expert_gather_kernel<V, uint8_t><<<grid, threads, 0, stream>>>(r, s, a.slots, a.k, a.T * a.k, a.offsets, a.E);
}

template <typename T, typename O>
void combine_typed(const CombineArgs& a, bool vec, cudaStream_t stream) {
  const int nv = vec ? a.width / 8 : a.width;
  const int threads = nv >= 256 ? 256 : 128;
  const dim3 grid((unsigned)a.T, column_parts(a.T, nv, threads, a.num_sms));
  if (vec)
    expert_combine_kernel<T, O, 8><<<grid, threads, 0, stream>>>(a);
  else
    expert_combine_kernel<T, O, 1><<<grid, threads, 0, stream>>>(a);
}
template <typename T, typename O>
void combine_bwd_typed(const CombineBwdArgs& a, bool vec, cudaStream_t stream) {
  if (vec)
    expert_combine_bwd_kernel<T, O, 8><<<(unsigned)a.T, 256, 0, stream>>>(a);
  else
    expert_combine_bwd_kernel<T, O, 1><<<(unsigned)a.T, 256, 0, stream>>>(a);
}

}  // namespace

int launch_expert_order(const void* ids, bool wide, int64_t id_stride, int64_t T, int k, int64_t base, int E,
                        int32_t* offsets, int32_t* slots, int32_t* pairs, cudaStream_t stream) {
  const int64_t n = T * k;
  // one CTA up to 4096 pairs; beyond, about 4096 pairs a CTA
  const int cluster = n <= 4096 ? 1 : n <= 8192 ? 2 : n <= 16384 ? 4 : 8;
  int warps = (int)((n + 32 * cluster - 1) / (32 * cluster));
  warps = warps < 4 ? 4 : warps > 32 ? 32 : warps;
  const int most = (200 * 1024 / 4 - 2 * E) / E;  // shared memory: (warps + 2) counters of every expert
  warps = warps > most ? most : warps;
  if (warps < 1) return -1;
  const size_t smem = (size_t)(warps + 2) * E * sizeof(int32_t);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(cluster);
  cfg.blockDim = dim3(warps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (wide) {
    cudaFuncSetAttribute(expert_order_kernel<int64_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    return (int)cudaLaunchKernelEx(&cfg, expert_order_kernel<int64_t>, static_cast<const int64_t*>(ids), id_stride, k,
                                   (int)n, base, E, offsets, slots, pairs);
  }
  cudaFuncSetAttribute(expert_order_kernel<int32_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  return (int)cudaLaunchKernelEx(&cfg, expert_order_kernel<int32_t>, static_cast<const int32_t*>(ids), id_stride, k,
                                 (int)n, base, E, offsets, slots, pairs);
}

void launch_expert_gather(const GatherArgs& a, cudaStream_t stream) {
  if (a.T == 0 || a.k == 0) return;
  const Plane r{static_cast<const uint8_t*>(a.src), a.src_stride, static_cast<uint8_t*>(a.dst), a.row_bytes};
  const Plane s{static_cast<const uint8_t*>(a.scales), a.scales_stride, static_cast<uint8_t*>(a.scales_dst),
                a.scale_bytes};
  const int64_t align = r.bytes | r.src_stride | reinterpret_cast<intptr_t>(r.src);
  if (align % 16 == 0)
    gather_scales<uint4>(r, s, a, stream);
  else if (align % 4 == 0)
    gather_scales<uint32_t>(r, s, a, stream);
  else if (align % 2 == 0)
    gather_scales<uint16_t>(r, s, a, stream);
  else
    gather_scales<uint8_t>(r, s, a, stream);
}

// Types: 0 = BF16, 1 = FP16, 2 = FP32 (rows); out_f32: FP32 output and residual, else the rows' type.
void launch_expert_combine(const CombineArgs& a, int type, bool out_f32, bool vec, cudaStream_t stream) {
  if (a.T == 0 || a.width == 0) return;
  if (type == 2)
    combine_typed<float, float>(a, vec, stream);
  else if (type == 1)
    out_f32 ? combine_typed<__half, float>(a, vec, stream) : combine_typed<__half, __half>(a, vec, stream);
  else
    out_f32 ? combine_typed<__nv_bfloat16, float>(a, vec, stream)
            : combine_typed<__nv_bfloat16, __nv_bfloat16>(a, vec, stream);
}

void launch_expert_combine_bwd(const CombineBwdArgs& a, int type, bool out_f32, bool vec, cudaStream_t stream) {
  if (a.T == 0 || a.k == 0) return;
  if (type == 2)
    combine_bwd_typed<float, float>(a, vec, stream);
  else if (type == 1)
    out_f32 ? combine_bwd_typed<__half, float>(a, vec, stream) : combine_bwd_typed<__half, __half>(a, vec, stream);
  else
    out_f32 ? combine_bwd_typed<__nv_bfloat16, float>(a, vec, stream)
            : combine_bwd_typed<__nv_bfloat16, __nv_bfloat16>(a, vec, stream);
}
