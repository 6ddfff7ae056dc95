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

// Sum of N values over the blockDim.x threads (a multiple of 32, at most 512) of this thread's row;
// the block's blockDim.y rows reduce side by side.  Every thread of the block calls it.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[N][16]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) red[threadIdx.y][i][warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.f;
    for (int j = 0; j < warps; ++j) v[i] += red[threadIdx.y][i][j];
  }
}

// Block (threads of a row, rows): thread t of a row owns the 8-column vectors t, t + blockDim.x, ...
// (VPT of them), so the 4 lanes that share a 32-column group are neighbours.
template <typename T, int VPT>
__global__ void __launch_bounds__(512) add_rmsnorm_mx_kernel(const NormMxArgs a) {
  __shared__ float red[8][1][16];
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < a.rows;
  const int nv = a.n >> 3, tx = threadIdx.x;
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
// Each row slot of the grid walks rows slot, slot + slots, ... and keeps its columns' sums of dw in
// registers; part[slot] receives them, and norm_dw_kernel adds the slots in order (the result does not
// depend on timing).
template <typename T, int VPT>
__global__ void __launch_bounds__(512) rmsnorm_bwd_kernel(const NormBwdArgs a) {
  __shared__ float red[2][8][2][16];
  const int nv = a.n >> 3, tx = threadIdx.x;
  const int slots = gridDim.x * blockDim.y, slot = blockIdx.x * blockDim.y + threadIdx.y;
  float w[VPT][8], dw[VPT][8];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = tx + j * blockDim.x;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[j][i] = dw[j][i] = 0.f;
    if (c < nv) rows::load8<float>(a.w + c * 8, w[j]);
  }
  const int64_t turns = (a.rows + slots - 1) / slots;
  for (int64_t t = 0; t < turns; ++t) {  // the same count in every thread: row_sum synchronizes the block
    const int64_t row = t * slots + slot;
    const bool live = row < a.rows;
    float s[VPT][8], g[VPT][8];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = tx + j * blockDim.x;
      if (live && c < nv) {
        rows::load8<T>(static_cast<const T*>(a.x) + row * a.xs + c * 8, s[j]);
        rows::load8<T>(static_cast<const T*>(a.dh) + row * a.dhs + c * 8, g[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum[0] += s[j][i] * s[j][i];
          sum[1] += g[j][i] * w[j][i] * s[j][i];
        }
      }
    }
    row_sum<2>(sum, red[t & 1]);  // two buffers: a slow warp still reads the last row's sums
    const float r = rsqrtf(sum[0] / a.n + a.eps);
    const float k = sum[1] / a.n * r * r;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = tx + j * blockDim.x;
      if (live && c < nv) {
        float o[8];
        if (a.dres)
          rows::load8<T>(static_cast<const T*>(a.dres) + row * a.drs + c * 8, o);
        else
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dw[j][i] += g[j][i] * (s[j][i] * r);
          o[i] += r * (g[j][i] * w[j][i] - s[j][i] * k);
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + row * a.n + c * 8) = rows::pack8<T>(o);
        if (a.dxf) rows::store8f(a.dxf + row * a.n + c * 8, o);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = tx + j * blockDim.x;
    if (c < nv) rows::store8f(a.part + (int64_t)slot * a.n + c * 8, dw[j]);
  }
}

// dw[c] = sum over slots of part[slot][c], in slot order within each of 16 fixed strands.
// Block (16 columns of float4, 16 strands).
__global__ void __launch_bounds__(256) norm_dw_kernel(const float* __restrict__ part, int slots, int n,
                                                      float* __restrict__ dw) {
  __shared__ float4 red[16][16];
  const int c = (blockIdx.x * 16 + threadIdx.x) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < n)
    for (int r = threadIdx.y; r < slots; r += 16) {
      const float4 v = *reinterpret_cast<const float4*>(part + (int64_t)r * n + c);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < n) {
    for (int r = 1; r < 16; ++r) {
      const float4 v = red[r][threadIdx.x];
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    *reinterpret_cast<float4*>(dw + c) = s;
  }
}

// Threads of a row (multiple of 32) for VPT vectors each, and rows of a block of about 256 threads.
dim3 norm_block(int n, int vpt) {
  const int tx = ((n / 8 + vpt - 1) / vpt + 31) / 32 * 32;
  const int ty = tx >= 256 ? 1 : (256 / tx > 8 ? 8 : 256 / tx);
  return dim3(tx, ty);
}

}  // namespace

void launch_add_rmsnorm_mx(const NormMxArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return;
  const dim3 block = norm_block(a.n, 2);
  const unsigned grid = (unsigned)((a.rows + block.y - 1) / block.y);
  if (a.half)
    add_rmsnorm_mx_kernel<__half, 2><<<grid, block, 0, stream>>>(a);
  else
    add_rmsnorm_mx_kernel<__nv_bfloat16, 2><<<grid, block, 0, stream>>>(a);
}

int rmsnorm_bwd_slots(int64_t rows, int n, int num_sms) {
  const dim3 block = norm_block(n, 2);
  const int64_t want = (rows + block.y - 1) / block.y;
  const int64_t most = (int64_t)num_sms * (1024 / (block.x * block.y) > 0 ? 1024 / (block.x * block.y) : 1);
  return (int)((want < most ? want : most) * block.y);
}

void launch_rmsnorm_bwd(const NormBwdArgs& a, int slots, cudaStream_t stream) {
  const dim3 block = norm_block(a.n, 2);
  if (slots > 0) {
    if (a.half)
      rmsnorm_bwd_kernel<__half, 2><<<slots / block.y, block, 0, stream>>>(a);
    else
      rmsnorm_bwd_kernel<__nv_bfloat16, 2><<<slots / block.y, block, 0, stream>>>(a);
  }
  norm_dw_kernel<<<(a.n + 63) / 64, dim3(16, 16), 0, stream>>>(a.part, slots, a.n, a.dw);
}
