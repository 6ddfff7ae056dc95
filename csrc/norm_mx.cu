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

constexpr int kMaxWarps = 16;  // warps of a row (n <= 8192)

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
  // every warp adds the (at most 16) partial sums by shuffles: a loop over them cost half of a row's instructions
  const int w = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = w < warps ? red[threadIdx.y * N + i][w] : 0.f;
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
}

// Thread t of a row owns the 8-column vectors t, t + blockDim.x, ... (VPT of them), so the 4 lanes that share a
// 32-column group are neighbours.  One group of blockDim.y rows per block: the many resident blocks hide the
// latency of each other's loads, reductions and stores.  Four blocks of 512 (32 registers, no spills): 4096 rows of
// 8192 take 76 us against 81 with the 38 registers of three.
template <typename T, int VPT>
__global__ void __launch_bounds__(512, 4) add_rmsnorm_mx_kernel(const NormMxArgs a) {
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
// Rows come through a ring in shared memory, kDepth - 1 ahead, by asynchronous copies: each thread copies the vectors
// that it reads itself (kVpt of each operand), so the ring needs no barrier, and both passes over a row read it there.
// Bound by HBM: 43 us for 8192 rows of 4096 with dres (6.2 TB/s), 48.3 with norm_dw_kernel (55.9 with the next row in
// registers instead of the ring, and norm_dw_kernel launched after this one).  One vector a thread is slower (twice
// the reductions), and so are three blocks of 256 threads an SM (80 registers).
constexpr int kVpt = 2;
constexpr int kDepth = 3;  // of the ring: two take 53.9 us (norm_dw_kernel after it), three 51.7, four 51.9
__device__ __forceinline__ void copy16(uint4* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(pm::smem_u32(to)), "l"(__cvta_generic_to_global(from)) : "memory");
}
template <typename T>
__global__ void __launch_bounds__(512, 1) rmsnorm_bwd_kernel(const NormBwdArgs a) {
  extern __shared__ __align__(16) uint4 ring[];
  float* sums = reinterpret_cast<float*>(ring);  // [group - 1][n], at the end
  __shared__ float red[2][2 * kMaxWarps][kMaxWarps];
  const int nv = a.n >> 3, tx = threadIdx.x, ty = threadIdx.y, group = blockDim.y;
  const int64_t step = (int64_t)gridDim.x * group;
  const int threads = blockDim.x * blockDim.y, tensors = a.dres ? 3 : 2;
  uint4* slot = ring + ty * blockDim.x + tx;
  pm::griddep_launch_dependents();  // norm_dw_kernel waits for this grid's end
  float w[kVpt][8], dw[kVpt][8];
#pragma unroll
  for (int j = 0; j < kVpt; ++j) {
    const int c = tx + j * blockDim.x;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[j][i] = dw[j][i] = 0.f;
    if (c < nv) rows::load8<float>(a.w + c * 8, w[j]);
  }
  int put = 0, take = 0;
  auto fetch = [&](int64_t row) {
    uint4* to = slot + put * (tensors * kVpt * threads);
#pragma unroll
    for (int j = 0; j < kVpt; ++j) {
      const int c = tx + j * blockDim.x;
      if (row < a.rows && c < nv) {
        copy16(to + j * threads, static_cast<const T*>(a.x) + row * a.xs + c * 8);
        copy16(to + (kVpt + j) * threads, static_cast<const T*>(a.dh) + row * a.dhs + c * 8);
        if (a.dres) copy16(to + (2 * kVpt + j) * threads, static_cast<const T*>(a.dres) + row * a.drs + c * 8);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    put = put + 1 == kDepth ? 0 : put + 1;
  };
  const float inv_n = 1.f / a.n;
  bool flip = false;
  int64_t row0 = (int64_t)blockIdx.x * group;
#pragma unroll
  for (int q = 0; q < kDepth - 1; ++q) fetch(row0 + ty + q * step);
  for (; row0 < a.rows; row0 += step) {
    const int64_t row = row0 + ty;
    float sum[2] = {0.f, 0.f};
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
    const uint4* from = slot + take * (tensors * kVpt * threads);
    take = take + 1 == kDepth ? 0 : take + 1;
#pragma unroll
    for (int j = 0; j < kVpt; ++j)
      if (tx + j * blockDim.x < nv) {
        float s[8], g[8];
        rows::unpack8<T>(from[j * threads], s);
        rows::unpack8<T>(from[(kVpt + j) * threads], g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum[0] = fmaf(s[i], s[i], sum[0]);
          sum[1] = fmaf(g[i] * w[j][i], s[i], sum[1]);
        }
      }
    fetch(row + (kDepth - 1) * step);
    row_sum<2>(sum, red[flip]);  // two buffers: a slow warp may still read the last group's sums
    flip = !flip;
    const float r = rsqrtf(sum[0] * inv_n + a.eps);
    const float k = sum[1] * inv_n * r * r * r;
#pragma unroll
    for (int j = 0; j < kVpt; ++j) {
      const int c = tx + j * blockDim.x;
      if (row < a.rows && c < nv) {
        float s[8], g[8], o[8];
        rows::unpack8<T>(from[j * threads], s);
        rows::unpack8<T>(from[(kVpt + j) * threads], g);
        rows::unpack8<T>(a.dres ? from[(2 * kVpt + j) * threads] : make_uint4(0, 0, 0, 0), o);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float t = r * g[i];
          dw[j][i] = fmaf(t, s[i], dw[j][i]);
          o[i] = fmaf(-k, s[i], fmaf(t, w[j][i], o[i]));
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + row * a.n + c * 8) = rows::pack8<T>(o);
        if (a.dxf) rows::store8f(a.dxf + row * a.n + c * 8, o);
      }
    }
  }
  // the block's rows of sums become one, in row order
  asm volatile("cp.async.wait_group 0;" ::: "memory");  // the ring's memory is free
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
    for (int q = 1; q < group; ++q) {
      float t[8];
      rows::load8<float>(sums + (q - 1) * a.n + c * 8, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) dw[j][i] += t[i];
    }
    rows::store8f(a.part + (int64_t)blockIdx.x * a.n + c * 8, dw[j]);
  }
}

// dw[c] = sum over slots (blocks) of part[slot][c], in slot order within each of 64 fixed strands, the strands in order.
// Block (4 columns of float4, 64 strands): many short strands, because the sums wait on L2 latency.
__global__ void __launch_bounds__(256) norm_dw_kernel(const float* __restrict__ part, int slots, int n,
                                                      float* __restrict__ dw) {
  __shared__ float4 red[64][4];
  pm::griddep_wait();  // (nothing is read or written before the grids ahead have ended)
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

// code x 2^(scale - 127) in BF16: exact for scale bytes 3 to 246 (an E4M3 value has four significant bits), one rounding
// beyond them, to zero, a subnormal or infinity; byte 255 is E8M0's NaN.  Thread per 16 codes; memory bound.
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint4* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, int64_t n16,
                                                            uint4* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n16) return;
  const uint4 c = codes[i];
  const int e = scales[i >> 1];
  const float s = e == 255 ? __int_as_float(0x7fffffff) : exp2f((float)(e - 127));
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
// Vectors of a thread by width, two past 4096 columns and one up to there: half the serial work of a thread (2.7 us for
// 8 rows of 4096 against 3.6 with two; 27.2 for 4999 rows of 2080 against 29.5).  Many rows of 4096 would take two 3 %
// better (8192: 74 us, 5.9 TB/s, against 72): the rule looks at the width alone.
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

int rmsnorm_bwd_slots(int64_t rows, int n, int num_sms) {
  const dim3 block = norm_block(n, kVpt);
  // resident blocks: 512 threads an SM (the kernel's 128 registers)
  const int64_t groups = (rows + block.y - 1) / block.y, most = (int64_t)num_sms * (512 / (int)(block.x * block.y));
  return (int)(groups < most ? groups : most);
}

void launch_rmsnorm_bwd(const NormBwdArgs& a, int slots, cudaStream_t stream) {
  const dim3 block = norm_block(a.n, kVpt);
  if (slots > 0) {
    auto* fn = a.half ? rmsnorm_bwd_kernel<__half> : rmsnorm_bwd_kernel<__nv_bfloat16>;
    const size_t ring = (size_t)kDepth * (a.dres ? 3 : 2) * kVpt * block.x * block.y * sizeof(uint4);
    const size_t sums = (block.y - 1) * a.n * sizeof(float), smem = ring > sums ? ring : sums;
    // the limit is the kernel's, not this launch's: always the largest (a ring of 512 threads and three operands), or a
    // smaller launch of another host thread could lower it before this one
    constexpr int most = kDepth * 3 * kVpt * 512 * (int)sizeof(uint4);
    if (smem > 40 * 1024) cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    fn<<<slots, block, smem, stream>>>(a);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((a.n + 15) / 16);
  cfg.blockDim = dim3(4, 64);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};  // launched while the rows are still walked (3 us less)
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, norm_dw_kernel, static_cast<const float*>(a.part), slots, a.n, a.dw);
}

void launch_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t n, void* out, cudaStream_t stream) {
  if (n == 0) return;
  mx_dequantize_kernel<<<(unsigned)((n / 16 + 255) / 256), 256, 0, stream>>>(reinterpret_cast<const uint4*>(codes), scales,
                                                                           n / 16, static_cast<uint4*>(out));
}
