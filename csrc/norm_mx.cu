// Residual add + RMSNorm with MXFP8 output rows, and the gradient of the residual add + RMSNorm.
//
//   s = x + d + df, stored in x's type; r = (mean(s^2) + eps)^-1/2; h = s r w       (fp32)
//   per 32 columns: e = the least integer with 448 2^e >= max(amax |h|, 1e-4), codes = E4M3(h 2^-e),
//   scale byte e + 127; h itself, rounded to x's type, on request (the router reads it)
//
// The codes are rounded once, from the fp32 h: rounding h to BF16 first would put about one value in
// thirty on the wrong side of an E4M3 rounding boundary.  The norm is that of the stored (rounded) stream,
// so that a reader of the stream finds the h that was computed from it.
#include "launchers.h"
#include "common/sm100.cuh"
#include "common/rows.cuh"

namespace {

constexpr int kVpt = 2;        // 8-column vectors of a thread
constexpr int kMaxWarps = 16;  // warps of a row (n <= 8192)
constexpr int kMaxStages = 8;

// Sum of N values over the blockDim.x threads of this thread's row (a power of two below 32, or whole warps);
// the block's blockDim.y rows reduce side by side.  Every thread of the block calls it, and for rows of
// more than one warp it is a barrier of the block.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[kMaxWarps]) {
  const int tx = blockDim.x;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1)
      if (o < tx) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (tx <= 32) return;
  const int warps = tx >> 5, warp = threadIdx.x >> 5;  // rows of several warps: row y's sums at red[y N + i]
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) red[threadIdx.y * N + i][warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.f;
    for (int j = 0; j < warps; ++j) v[i] += red[threadIdx.y * N + i][j];
  }
}

// A ring of row groups in shared memory: the group of blockDim.y rows that the block works on next, and those
// after it, arrive by bulk copies while the current one is reduced and stored, so the loads in flight do
// not depend on registers or occupancy.  Tensors follow one another in a stage, rows contiguous.
struct RowSource {
  const uint8_t* base;
  int64_t stride;  // bytes between rows
  int bytes;       // of a row (a multiple of 16)
};
template <int N>
struct RowRing {
  RowSource src[N];
  uint8_t* smem;
  uint64_t* full;
  int64_t rows;
  int stage_bytes, stages, group;
  // stage s <- rows [row0, row0 + group) (fewer at the end; nothing past the last).  Called by warp 0.
  __device__ __forceinline__ void issue(int s, int64_t row0, int lane) const {
    const int64_t left = rows - row0;
    if (left <= 0) return;
    const int have = left < group ? (int)left : group;
    uint32_t total = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (src[i].base) total += src[i].bytes * have;
    if (lane == 0) pm::mbar_arrive_expect_tx(full + s, total);
    __syncwarp();
    uint8_t* dst = smem + s * stage_bytes;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!src[i].base) continue;
      const uint8_t* from = src[i].base + row0 * src[i].stride;
      if (src[i].stride == src[i].bytes) {
        if (lane == 0) pm::bulk_g2s(dst, from, src[i].bytes * have, full + s);
      } else {
        for (int r = lane; r < have; r += 32) pm::bulk_g2s(dst + r * src[i].bytes, from + r * src[i].stride, src[i].bytes, full + s);
      }
      dst += src[i].bytes * group;
    }
  }
};

// The threads of a block walk groups of blockDim.y rows: group g, g + gridDim.x, ...  `ring`: rows come through
// the ring, else straight from global memory.
template <int N>
__device__ __forceinline__ void ring_start(RowRing<N>& ring, int64_t first, int64_t step) {
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  if (tid == 0) {
    for (int i = 0; i < ring.stages; ++i) pm::mbar_init(ring.full + i, 1);
    pm::fence_mbar_init();
  }
  __syncthreads();
  if (tid < 32)
    for (int i = 0; i < ring.stages; ++i) ring.issue(i, first + i * step, tid);
}

// A wait ran out (the error word says so): let the copies in flight land before the block leaves.
template <int N>
__device__ __noinline__ void ring_give_up(const RowRing<N>& ring, int st, uint32_t ph) {
  for (int s = 0; s < ring.stages; ++s) pm::mbar_wait(ring.full + s, s >= st ? ph : ph ^ 1, nullptr, 0, 20000000ull);
}

// Thread t of a row owns the 8-column vectors t, t + blockDim.x, ... (VPT of them), so the 4 lanes that share a
// 32-column group are neighbours.  One group of blockDim.y rows per block: the many resident blocks hide the
// latency of each other's loads, reductions and stores.
template <typename T, int VPT>
__global__ void __launch_bounds__(512) add_rmsnorm_mx_kernel(const NormMxArgs a) {
  __shared__ float red[kMaxWarps][kMaxWarps];
  const int nv = a.n >> 3, tx = threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < a.rows;
  float v[VPT][8];
  float ss[1] = {0.f};
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = tx + j * blockDim.x;
    if (live && c < nv) {
      rows::load8<T>(static_cast<const T*>(a.x) + row * a.xs + c * 8, v[j]);
      if (a.d) {
        float t[8];
        rows::load8<T>(static_cast<const T*>(a.d) + row * a.ds + c * 8, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] += t[i];
      }
      if (a.df) {
        float t[8];
        rows::load8<float>(a.df + row * a.dfs + c * 8, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] += t[i];
      }
      if (a.x_out) {
        const uint4 p = rows::pack8<T>(v[j]);
        *reinterpret_cast<uint4*>(static_cast<T*>(a.x_out) + row * a.xos + c * 8) = p;
        rows::unpack8<T>(p, v[j]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss[0] += v[j][i] * v[j][i];
    }
  }
  row_sum<1>(ss, red);
  const float r = rsqrtf(ss[0] / a.n + a.eps);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = tx + j * blockDim.x;
    float amax = 0.f;
    if (live && c < nv) {
      float w[8];
      rows::load8<float>(a.w + c * 8, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] = v[j][i] * r * w[i];
        amax = fmaxf(amax, fabsf(v[j][i]));
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    if (live && c < nv) {
      if (a.h) *reinterpret_cast<uint4*>(static_cast<T*>(a.h) + row * a.n + c * 8) = rows::pack8<T>(v[j]);
      const int e = pm::ue8m0_exp(amax);
      const float s = pm::exp2i(-e);
      uint2 q;
      q.x = (uint32_t)pm::f32x2_to_e4m3x2(v[j][0] * s, v[j][1] * s) |
            ((uint32_t)pm::f32x2_to_e4m3x2(v[j][2] * s, v[j][3] * s) << 16);
      q.y = (uint32_t)pm::f32x2_to_e4m3x2(v[j][4] * s, v[j][5] * s) |
            ((uint32_t)pm::f32x2_to_e4m3x2(v[j][6] * s, v[j][7] * s) << 16);
      *reinterpret_cast<uint2*>(a.codes + row * a.n + c * 8) = q;
      if ((c & 3) == 0) a.scales[row * (a.n >> 5) + (c >> 2)] = (uint8_t)(e + 127);
    }
  }
}

// dx = r (g - s r^2 mean(g s)) + dres with g = dh w; dw = sum over rows of dh s r.
// Each thread row of the grid (blockIdx.x, threadIdx.y) keeps its columns' sums of dw over the rows it walks;
// part[blockIdx.x] receives the block's, and norm_dw_kernel adds the blocks in order (the result does not depend
// on timing).
// Rows come through a shared-memory ring and stay packed in registers between the two passes, w stays in shared
// memory: few registers, so that several blocks share an SM and cover each other's reductions.
template <typename T, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) rmsnorm_bwd_kernel(const NormBwdArgs a, int stages) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[2][2 * kMaxWarps][kMaxWarps];
  __shared__ uint64_t full[kMaxStages];
  const int nv = a.n >> 3, tx = threadIdx.x, ty = threadIdx.y, group = blockDim.y;
  const int tid = ty * blockDim.x + tx;
  const int64_t step = (int64_t)gridDim.x * group;
  const int b2 = a.n * 2;
  RowRing<3> ring;
  ring.src[0] = {static_cast<const uint8_t*>(a.x), a.xs * 2, b2};
  ring.src[1] = {static_cast<const uint8_t*>(a.dh), a.dhs * 2, b2};
  ring.src[2] = {static_cast<const uint8_t*>(a.dres), a.drs * 2, b2};
  ring.smem = smem + a.n * 4;
  ring.full = full;
  ring.rows = a.rows;
  ring.stage_bytes = group * b2 * (a.dres ? 3 : 2);
  ring.stages = stages;
  ring.group = group;
  ring_start(ring, (int64_t)blockIdx.x * group, step);
  float* w = reinterpret_cast<float*>(smem);
  for (int i = tid * 4; i < a.n; i += blockDim.x * group * 4)
    *reinterpret_cast<float4*>(w + i) = *reinterpret_cast<const float4*>(a.w + i);
  __syncthreads();
  float dw[kVpt][8];
#pragma unroll
  for (int j = 0; j < kVpt; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[j][i] = 0.f;
  const float inv_n = 1.f / a.n;
  int st = 0;
  uint32_t ph = 0;
  bool flip = false;
  for (int64_t row0 = (int64_t)blockIdx.x * group; row0 < a.rows; row0 += step) {
    const int64_t row = row0 + ty;
    const bool live = row < a.rows;
    const T* at = reinterpret_cast<const T*>(ring.smem + st * ring.stage_bytes) + ty * a.n;
    if (!pm::mbar_wait(full + st, ph, tid == 0 ? a.err : nullptr, 502)) return ring_give_up(ring, st, ph);
    uint4 sp[kVpt], gp[kVpt], res[kVpt];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kVpt; ++j) {
      const int c = tx + j * blockDim.x;
      res[j] = sp[j] = gp[j] = make_uint4(0, 0, 0, 0);
      if (live && c < nv) {
        sp[j] = *reinterpret_cast<const uint4*>(at + c * 8);
        gp[j] = *reinterpret_cast<const uint4*>(at + group * a.n + c * 8);
        if (a.dres) res[j] = *reinterpret_cast<const uint4*>(at + 2 * group * a.n + c * 8);
        float s[8], g[8], wv[8];
        rows::unpack8<T>(sp[j], s);
        rows::unpack8<T>(gp[j], g);
        rows::load8<float>(w + c * 8, wv);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum[0] += s[i] * s[i];
          sum[1] += g[i] * wv[i] * s[i];
        }
      }
    }
    row_sum<2>(sum, red[flip]);  // two buffers: a slow warp may still read the last group's sums
    flip = !flip;
    if (blockDim.x <= 32) __syncthreads();  // (row_sum was no barrier) every thread has read this stage
    if (tid < 32) ring.issue(st, row0 + stages * step, tid);
    if (++st == stages) { st = 0; ph ^= 1; }
    const float r = rsqrtf(sum[0] * inv_n + a.eps);
    const float k = sum[1] * inv_n * r * r;
#pragma unroll
    for (int j = 0; j < kVpt; ++j) {
      const int c = tx + j * blockDim.x;
      if (live && c < nv) {
        float s[8], g[8], wv[8], o[8];
        rows::unpack8<T>(sp[j], s);
        rows::unpack8<T>(gp[j], g);
        rows::load8<float>(w + c * 8, wv);
        rows::unpack8<T>(res[j], o);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dw[j][i] += g[i] * (s[i] * r);
          o[i] += r * (g[i] * wv[i] - s[i] * k);
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + row * a.n + c * 8) = rows::pack8<T>(o);
        if (a.dxf) rows::store8f(a.dxf + row * a.n + c * 8, o);
      }
    }
  }
  // the block's rows of sums become one, in row order (the ring is drained: its memory is free)
  float* sums = reinterpret_cast<float*>(ring.smem);
  __syncthreads();
  if (ty > 0) {
#pragma unroll
    for (int j = 0; j < kVpt; ++j) {
      const int c = tx + j * blockDim.x;
      if (c < nv) rows::store8f(sums + (ty - 1) * a.n + c * 8, dw[j]);
    }
  }
  __syncthreads();
  if (ty > 0) return;
#pragma unroll
  for (int j = 0; j < kVpt; ++j) {
    const int c = tx + j * blockDim.x;
    if (c >= nv) continue;
    for (int r = 1; r < group; ++r) {
      float o[8];
      rows::load8<float>(sums + (r - 1) * a.n + c * 8, o);
#pragma unroll
      for (int i = 0; i < 8; ++i) dw[j][i] += o[i];
    }
    rows::store8f(a.part + (int64_t)blockIdx.x * a.n + c * 8, dw[j]);
  }
}

// dw[c] = sum over slots (blocks) of part[slot][c], in slot order within each of 64 fixed strands, the strands in order.
// Block (4 columns of float4, 64 strands): many short strands, because the sums wait on L2 latency.
__global__ void __launch_bounds__(256) norm_dw_kernel(const float* __restrict__ part, int slots, int n,
                                                      float* __restrict__ dw) {
  __shared__ float4 red[64][4];
  const int c = (blockIdx.x * 4 + threadIdx.x) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < n) {
#pragma unroll 4
    for (int r = threadIdx.y; r < slots; r += 64) {
      const float4 v = *reinterpret_cast<const float4*>(part + (int64_t)r * n + c);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
  }
  red[threadIdx.y][threadIdx.x] = s;
  for (int h = 32; h >= 1; h >>= 1) {
    __syncthreads();
    if (threadIdx.y < h) {
      const float4 v = red[threadIdx.y + h][threadIdx.x];
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
      red[threadIdx.y][threadIdx.x] = s;
    }
  }
  if (threadIdx.y == 0 && c < n) *reinterpret_cast<float4*>(dw + c) = s;
}

// code x 2^(scale - 127) in BF16 (exact: an E4M3 value has four significant bits).  Thread per 16 codes; memory bound.
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint4* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, int64_t n16,
                                                            uint4* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n16) return;
  const uint4 c = codes[i];
  const float s = exp2f((float)scales[i >> 1] - 127.f);
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t o[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 lo = __half22float2(pm::e4m3x2_to_h2((uint16_t)w[j])), hi = __half22float2(pm::e4m3x2_to_h2((uint16_t)(w[j] >> 16)));
    o[2 * j] = rows::pack2<__nv_bfloat16>(lo.x * s, lo.y * s);
    o[2 * j + 1] = rows::pack2<__nv_bfloat16>(hi.x * s, hi.y * s);
  }
  out[2 * i] = make_uint4(o[0], o[1], o[2], o[3]);
  out[2 * i + 1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// Threads of a row for `vpt` vectors each (a power of two from 4 to 32, or whole warps), and the rows of a
// block of about 256 threads.
dim3 norm_block(int n, int vpt) {
  const int nv = n / 8;
  int tx = 4;
  while (tx < nv && tx < 32) tx *= 2;
  if (nv > 32 * vpt) tx = ((nv + vpt - 1) / vpt + 31) / 32 * 32;
  const int ty = tx >= 256 ? 1 : 256 / tx;
  return dim3(tx, ty);
}
// Ring of a gradient block: blocks of an SM by warps and registers (the kernel's launch bounds: 80 a thread with at
// most 256 threads, so 6 warps on each quarter of an SM, else 128), then as many stages as their shared
// memory holds, two at least.
struct RingPlan {
  int stages, smem, blocks_per_sm;
};
RingPlan ring_plan(int n, bool res, const dim3& block) {
  const int stage = (int)block.y * n * 2 * (res ? 3 : 2), w = n * 4, whole = 208 * 1024;
  RingPlan p;
  const int threads = block.x * block.y;
  p.blocks_per_sm = (threads <= 256 ? 24 : 16) * 32 / threads;
  while (p.blocks_per_sm > 1 && whole / p.blocks_per_sm - 5 * 1024 - w < 2 * stage) --p.blocks_per_sm;
  p.stages = (whole / p.blocks_per_sm - 5 * 1024 - w) / stage;
  p.stages = p.stages > kMaxStages ? kMaxStages : p.stages;
  p.smem = w + p.stages * stage;
  return p;
}

// Vectors of a thread by width: one up to 4096 columns (74 us for 8192 rows of 4096 against 77 with two, 2.8 us
// against 3.6 for 8 rows: half the serial work of a thread), two beyond (512 threads).
template <int VPT>
void launch_fwd(const NormMxArgs& a, cudaStream_t stream) {
  const dim3 block = norm_block(a.n, VPT);
  const unsigned grid = (unsigned)((a.rows + block.y - 1) / block.y);
  if (a.half)
    add_rmsnorm_mx_kernel<__half, VPT><<<grid, block, 0, stream>>>(a);
  else
    add_rmsnorm_mx_kernel<__nv_bfloat16, VPT><<<grid, block, 0, stream>>>(a);
}

}  // namespace

void launch_add_rmsnorm_mx(const NormMxArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return;
  if (a.n <= 4096)
    launch_fwd<1>(a, stream);
  else
    launch_fwd<2>(a, stream);
}

int rmsnorm_bwd_slots(int64_t rows, int n, bool res, int num_sms) {
  const dim3 block = norm_block(n, kVpt);
  const int64_t groups = (rows + block.y - 1) / block.y;
  const int64_t most = (int64_t)num_sms * ring_plan(n, res, block).blocks_per_sm;
  return (int)(groups < most ? groups : most);
}

void launch_rmsnorm_bwd(const NormBwdArgs& a, int slots, cudaStream_t stream) {
  const dim3 block = norm_block(a.n, kVpt);
  if (slots > 0) {
    const RingPlan p = ring_plan(a.n, a.dres != nullptr, block);
    auto* fn = block.x * block.y <= 256
                   ? (a.half ? rmsnorm_bwd_kernel<__half, 256, 3> : rmsnorm_bwd_kernel<__nv_bfloat16, 256, 3>)
                   : (a.half ? rmsnorm_bwd_kernel<__half, 512, 1> : rmsnorm_bwd_kernel<__nv_bfloat16, 512, 1>);
    cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem);
    fn<<<slots, block, p.smem, stream>>>(a, p.stages);
  }
  norm_dw_kernel<<<(a.n + 15) / 16, dim3(4, 64), 0, stream>>>(a.part, slots, a.n, a.dw);
}

void launch_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t n, void* out, cudaStream_t stream) {
  if (n == 0) return;
  mx_dequantize_kernel<<<(unsigned)((n / 16 + 255) / 256), 256, 0, stream>>>(reinterpret_cast<const uint4*>(codes), scales,
                                                                           n / 16, static_cast<uint4*>(out));
}
