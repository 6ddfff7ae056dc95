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

#include <type_traits>

#include "launchers.h"
#include "common/sm100.cuh"
#include "common/rows.cuh"

namespace {
namespace cg = cooperative_groups;

// ----------------------------------------------------------------------------- order
// A stable counting sort in one launch: the CTAs of one cluster (1 to 16) take consecutive ranges of pairs, the
// warps of a CTA consecutive ranges of its range.  Pass 1 counts per warp (one lane of those with equal experts
// adds: no atomics), the counts become starting rows (over warps, then CTAs, then experts), pass 2 hands out
// rows in the same order.  Latency bound: a lane's first kHeld ids and its peers of equal expert stay in
// registers for both passes, the ids loaded together, and each CTA pushes its counts into the others' shared
// memory, so that after the cluster barrier all reads are local.
constexpr int kOrderSmem = 200 * 1024;  // counters of a CTA at most
constexpr int kHeld = 8;  // ids of a lane held in registers (8 x 32 lanes x 16 warps x 16 CTAs = 65536 pairs)

template <typename Id>
__global__ void __launch_bounds__(512) expert_order_kernel(const Id* __restrict__ ids, int n, int64_t base, int E,
                                                            int32_t* __restrict__ offsets, int32_t* __restrict__ slots,
                                                            int32_t* __restrict__ pairs) {
  extern __shared__ int32_t sm[];
  __shared__ int32_t wsum[32];
  const int W = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  pm::griddep_launch_dependents();  // gather's blocks may be placed now; they wait for this grid's end
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  cl.barrier_arrive();  // waited for before this CTA writes to the others: they have all started
  int32_t* cnt = sm;           // [W][E]: counts, then the next row of (warp, expert)
  int32_t* tot = sm + W * E;   // [C][E]: every CTA's counts
  const int per = (((n + C * W - 1) / (C * W)) + 31) / 32 * 32;  // pairs of a warp
  const int lo = (int)min((int64_t)n, (int64_t)(rank * W + warp) * per), hi = (int)min((int64_t)n, (int64_t)lo + per);
  auto expert = [&](int i) -> int {
    if (i >= hi) return -1;
    const int64_t e = (int64_t)ids[i] - base;
    return e >= 0 && e < E ? (int)e : -1;
  };
  int held[kHeld];
  unsigned peer[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) held[j] = expert(lo + 32 * j + lane);
  const int bits = 32 - __clz(E);  // of 0 .. E (E: no expert)
  auto peers = [&](int e) {  // lanes of the same expert
    const unsigned v = e >= 0 ? (unsigned)e : (unsigned)E;
    unsigned m = 0xffffffffu;
#pragma unroll
    for (int b = 0; b < 8; ++b)  // bits past the last are 0 in every lane: no change
      m &= __ballot_sync(0xffffffffu, (v >> b) & 1) ^ (((v >> b) & 1) - 1);
    for (int b = 8; b < bits; ++b) m &= __ballot_sync(0xffffffffu, (v >> b) & 1) ^ (((v >> b) & 1) - 1);
    return m;
  };
  for (int i = tid; i < W * E; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  int32_t* mine = cnt + warp * E;
  auto count = [&](int e, unsigned m) {
    if (e >= 0 && lane == __ffs(m) - 1) mine[e] += __popc(m);
    __syncwarp();
  };
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if (lo + 32 * j < hi) count(held[j], peer[j] = peers(held[j]));
  for (int i0 = lo + 32 * kHeld; i0 < hi; i0 += 32) {
    const int e = expert(i0 + lane);
    count(e, peers(e));
  }
  __syncthreads();
  cl.barrier_wait();
  for (int e = tid; e < E; e += blockDim.x) {
    int c[16], run = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) c[w] = w < W ? cnt[w * E + e] : 0;
#pragma unroll
    for (int w = 0; w < 16; ++w)
      if (w < W) {
        cnt[w * E + e] = run;
        run += c[w];
      }
    for (int r = 0; r < C; ++r) *cl.map_shared_rank(tot + rank * E + e, r) = run;
  }
  cl.sync();
  // experts' first rows: exclusive sums over E of the cluster's counts, blockDim.x experts at a time
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += blockDim.x) {
    const int e = e0 + tid;
    int all = 0, before = 0;
    if (e < E)
      for (int c = 0; c < C; ++c) {
        const int v = tot[c * E + e];
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
    int ws = lane < W ? wsum[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, ws, o);
      if (lane >= o) ws += u;
    }
    const int wbase = warp ? __shfl_sync(0xffffffffu, ws, warp - 1) : 0;
    const int first = carry + wbase + inc - all;
    if (e < E) {
      tot[e] = first + before;  // row 0 of the table: only this thread reads column e
      if (rank == 0) offsets[e] = first;
    }
    carry += __shfl_sync(0xffffffffu, ws, 31);
    __syncthreads();
  }
  if (rank == 0 && tid == 0) offsets[E] = carry;
  auto place = [&](int i, int e, unsigned m) {
    int row = -1;
    if (e >= 0) row = tot[e] + mine[e] + __popc(m & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == __ffs(m) - 1) mine[e] += __popc(m);
    __syncwarp();
    if (i < hi) slots[i] = row;
    if (row >= 0) pairs[row] = i;
  };
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if (lo + 32 * j < hi) place(lo + 32 * j + lane, held[j], peer[j]);
  for (int i0 = lo + 32 * kHeld; i0 < hi; i0 += 32) {
    const int e = expert(i0 + lane);
    place(i0 + lane, e, peers(e));
  }
  for (int i = carry + rank * blockDim.x + tid; i < n; i += C * blockDim.x) pairs[i] = -1;
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
  pm::griddep_wait();  // (nothing is read before the grids ahead have ended)
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

// NV consecutive elements as loaded: converted only where they are added, so that kBatch rows in flight cost
// 4 registers each (16-bit types) instead of 8.
template <typename T, int NV>
struct Raw {
  static constexpr int kWords = NV == 1 ? 1 : NV * (int)sizeof(T) / 16;
  using Word = std::conditional_t<NV == 1, T, uint4>;
  Word w[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const Word*>(p)[i];
  }
  __device__ __forceinline__ void get(float (&v)[NV]) const {
    if constexpr (NV == 1) {
      v[0] = rows::to_f<T>(w[0]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        v[4 * i] = __uint_as_float(w[i].x);
        v[4 * i + 1] = __uint_as_float(w[i].y);
        v[4 * i + 2] = __uint_as_float(w[i].z);
        v[4 * i + 3] = __uint_as_float(w[i].w);
      }
    } else {
      rows::unpack8<T>(w[0], v);
    }
  }
};

// Block (token, column part): thread c of the part sums its NV columns over the token's choices.  The token's slots
// and weights are fetched together first, so that no row load waits for its slot.
template <typename T, typename O, int NV>
__global__ void __launch_bounds__(128) expert_combine_kernel(const CombineArgs a) {
  extern __shared__ int32_t slots[];
  float* wt = reinterpret_cast<float*>(slots + a.k);
  const int64_t t = blockIdx.x;
  const int nv = a.width / NV, k = a.k;
  for (int i = threadIdx.x; i < k; i += blockDim.x) {
    const int r = a.slots[t * k + i];
    slots[i] = has_row(r, a.T * k) ? r : -1;
    wt[i] = a.weights ? a.weights[t * a.ws + i] : 1.f;
  }
  __syncthreads();
  const T* y = static_cast<const T*>(a.y);
  const int step = gridDim.y * blockDim.x;
  for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < nv; c += step) {
    const int64_t col = (int64_t)c * NV;
    float acc[NV];
    if (a.residual) {
      Raw<O, NV> res;
      res.load(static_cast<const O*>(a.residual) + t * a.rs + col);
      res.get(acc);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[i] = 0.f;
    }
    for (int j0 = 0; j0 < k; j0 += kBatch) {
      const int32_t* slot = slots + j0;
      const float* w = wt + j0;
      Raw<T, NV> v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (j0 + j < k && slot[j] >= 0) v[j].load(y + (int64_t)slot[j] * a.ys + col);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (j0 + j < k && slot[j] >= 0) {  // a pair without a row adds nothing, whatever its weight holds
          float f[NV];
          v[j].get(f);
#pragma unroll
          for (int i = 0; i < NV; ++i) acc[i] = fmaf(w[j], f[i], acc[i]);
        }
    }
    store_n<O, NV>(static_cast<O*>(a.out) + t * a.width + col, acc);
  }
}

// Block per token, the last token first: the rows that the forward pass read last may still be in L2.  dout's
// columns are read once, every choice's y row once; the k dot products end in one block reduction per batch of
// choices.  Loads of a batch of rows before the stores of another: 94.6 us for 4096 x 8 rows of 4096, 107 by turns.
template <typename T, typename O, int NV>
__global__ void __launch_bounds__(128) expert_combine_bwd_kernel(const CombineBwdArgs a) {
  __shared__ float red[kBatch][4];
  const int64_t t = (int64_t)gridDim.x - 1 - blockIdx.x;
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
      float d[NV], v[NV];
      Raw<T, NV> in[kBatch];  // all loaded before the first store, which no load may pass
      load_n<O, NV>(g + (int64_t)c * NV, d);
      if (a.dw) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (r[j] >= 0) in[j].load(y + (int64_t)r[j] * a.ys + (int64_t)c * NV);
      }
      if (dy) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (r[j] >= 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = w[j] * d[i];
            store_n<T, NV>(dy + (int64_t)r[j] * a.width + (int64_t)c * NV, v);
          }
      }
      if (a.dw) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (r[j] >= 0) {
            in[j].get(v);
#pragma unroll
            for (int i = 0; i < NV; ++i) dot[j] = fmaf(d[i], v[i], dot[j]);
          }
      }
    }
    if (a.dw) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (j0 + j < a.k) {
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
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)a.T, column_parts(a.T, r.bytes / sizeof(V), threads, a.num_sms));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};  // the sort that usually precedes lets this launch overlap its end
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const int64_t align = s.bytes | s.src_stride | reinterpret_cast<intptr_t>(s.src);
  auto* fn = !s.src || align % 16 == 0 ? expert_gather_kernel<V, uint4>
             : align % 4 == 0          ? expert_gather_kernel<V, uint32_t>
                                       : expert_gather_kernel<V, uint8_t>;
  cudaLaunchKernelEx(&cfg, fn, r, s, a.slots, a.k, a.T * a.k, a.offsets, a.E);
}

template <typename T, typename O>
void combine_typed(const CombineArgs& a, bool vec, cudaStream_t stream) {
  // 128 threads: 6001 x 6 rows of 2048 take 32.0 us (5.4 TB/s) against 35.4 with 256, 1024 x 8 of 4096 15.7 against
  // 16.7, 8192 x 8 of 4096 92.8 (6.5 TB/s) either way; blocks of several tokens gain nothing
  const int nv = vec ? a.width / 8 : a.width;
  const dim3 grid((unsigned)a.T, column_parts(a.T, nv, 128, a.num_sms));
  const size_t smem = (size_t)a.k * 8;
  if (vec)
    expert_combine_kernel<T, O, 8><<<grid, 128, smem, stream>>>(a);
  else
    expert_combine_kernel<T, O, 1><<<grid, 128, smem, stream>>>(a);
}
template <typename T, typename O>
void combine_bwd_typed(const CombineBwdArgs& a, bool vec, cudaStream_t stream) {
  // 64 threads: 6001 x 6 rows of 2048 take 57.8 us against 61.0 with 128, 1024 x 8 of 4096 27.2 against 29.1, 4096 x 8
  // of 4096 94.6 (6.0 TB/s) either way; 128 where few tokens leave the GPU idle (8 tokens: 8.7 us a call against 10.7)
  const int threads = a.T < 512 ? 128 : 64;
  if (vec)
    expert_combine_bwd_kernel<T, O, 8><<<(unsigned)a.T, threads, 0, stream>>>(a);
  else
    expert_combine_bwd_kernel<T, O, 1><<<(unsigned)a.T, threads, 0, stream>>>(a);
}

}  // namespace

int launch_expert_order(const void* ids, bool wide, int64_t n, int64_t base, int E, int32_t* offsets, int32_t* slots,
                        int32_t* pairs, cudaStream_t stream) {
  // CTAs of the cluster: about 512 pairs each (one chunk of 32 a warp), at most 16, as long as the counts of
  // eight warps fit shared memory.  32768 pairs, 256 experts: 7.4 us with 16 CTAs, 10.0 with 8, 19.4 with 4.
  int cluster = 1;
  while (cluster < 16 && (int64_t)cluster * 512 < n) cluster *= 2;
  int warps = (int)((n + 32 * cluster - 1) / (32 * cluster));
  warps = warps < 4 ? 4 : warps > 16 ? 16 : warps;
  const int counters = kOrderSmem / 4 / E;  // shared memory: (warps + CTAs) counters of every expert
  while (cluster > 1 && counters - cluster < 8) cluster /= 2;
  warps = warps > counters - cluster ? counters - cluster : warps;
  if (warps < 1) return -1;
  const size_t smem = (size_t)(warps + cluster) * E * sizeof(int32_t);
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
  auto go = [&](auto* fn, auto* p) {
    // the limit is the kernel's, not this launch's: always the largest, or a smaller launch of another host thread
    // could lower it before this one
    if (smem > 40 * 1024) cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kOrderSmem);
    if (cluster > 8) cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return (int)cudaLaunchKernelEx(&cfg, fn, p, (int)n, base, E, offsets, slots, pairs);
  };
  return wide ? go(expert_order_kernel<int64_t>, static_cast<const int64_t*>(ids))
              : go(expert_order_kernel<int32_t>, static_cast<const int32_t*>(ids));
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
