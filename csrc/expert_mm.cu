// Matrix products of every expert's rows in one launch (tcgen05, BF16 or FP16 operands, fp32 accumulators).
//
//   kForward   y_e  = act(x_e W_e^T)     rows of x sorted by expert, W [E, N, K]; act: none, or SwiGLU over
//                                        W's rows [gate I | up I]: y = silu(g) u
//   kGradX     dx_e = dz_e W_e
//   kGradW     dW_e = dz_e^T x_e         (zero for an expert without rows)
//
// Expert e owns rows offsets[e] .. offsets[e + 1]; the offsets are read on the device, so no call waits for
// the host.  Rows past offsets[E] give zero rows (kForward, kGradX) and are not read (kGradW).
//
// Tile: 128 x 256 outputs, 64 of the reduced dimension per stage, both operands by TMA with the 128-byte
// swizzle.  Rows (x, dz) are the M = 128 operand of kForward and kGradX: an expert's last tile reads into
// the next expert's rows, which only fills accumulator rows that nobody stores.  kGradX reads W, and kGradW
// reads both operands, along their other dimension through MN-major descriptors, so nothing is transposed in
// memory; kGradW reduces over rows, so the rows past the expert's last one in its last stage are zeroed in
// shared memory before the MMA.  One persistent CTA per SM: a TMA warp, an MMA warp and four epilogue warps,
// the accumulator double-buffered in TMEM (2 x 256 columns), so that a tile's epilogue overlaps the next
// tile's products.
#include <cuda.h>

#include "launchers.h"
#include "common/sm100.cuh"
#include "common/rows.cuh"

namespace {

constexpr int kThreads = 192;      // warp 0 TMA producer, warp 1 MMA issuer, warps 2-5 epilogue
constexpr int kTileM = 128, kTileN = 256, kTileK = 64;
constexpr uint32_t kBBytes = kTileN * kTileK * 2;
constexpr uint32_t kChunk = 64 * 128;  // MN-major operands: 64 reduced rows x 64 columns (128 B)
constexpr int kEpiWarpBytes = 32 * 128;  // staging of one epilogue warp: 32 rows x 64 outputs
constexpr int kBand = 8;           // row tiles that walk the column tiles together (L2 reuse of both operands)
constexpr int kMaxStages = 8;
enum Mode { kForward = 0, kGradX = 1, kGradW = 2 };

// AM: rows of the A operand that a stage loads (the MMA always takes 128; rows past AM read whatever the
// stage holds and fill accumulator rows that nobody stores).
template <int AM>
struct Cfg {
  static constexpr uint32_t kABytes = AM * kTileK * 2;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = AM == 128 ? 4 : 5;
  static constexpr uint32_t kEpiOff = kStages * kStageBytes;
  static constexpr uint32_t kBarOff = kEpiOff + 4 * kEpiWarpBytes;
  static constexpr uint32_t kFixed = kBarOff + 256 + 1024;  // barriers, alignment; then the tile table
  static_assert(kABytes % 1024 == 0 && 128 * kTileK * 2 <= kStageBytes && kStages <= kMaxStages, "stage layout");
};

struct Tile {
  int e, m, n;      // expert, row tile and column tile inside it
  int row0, rows;   // kForward / kGradX: first row and rows of the tile; kGradW: the expert's
  int nk;           // stages (0: the tile is zero)
};

// Walks this CTA's tiles in order; every role of the CTA keeps its own walker.
template <int MODE, int AM>
struct Walker {
  const ExpertMmArgs& a;
  const int32_t* start;  // shared: first tile of each expert, [E + 2] (expert E: the rows past the last one)
  const int32_t* off;    // shared: offsets [E + 1]
  int tn, tm_w, e, t;
  __device__ Walker(const ExpertMmArgs& args, const int32_t* s, const int32_t* o) : a(args), start(s), off(o) {
    e = 0;
    t = (int)blockIdx.x - (int)gridDim.x;
    tn = a.tiles_n;
    tm_w = a.tiles_m;
  }
  __device__ bool next(Tile& k) {
    t += gridDim.x;
    const int E = a.E;
    if (t >= start[MODE == kGradW ? E : E + 1]) return false;
    while (t >= start[e + 1]) ++e;
    const int rel = t - start[e];
    int tm;
    k.e = e;
    if (MODE == kGradW) {
      tm = tm_w;
      k.row0 = off[e];
      k.rows = off[e + 1] - off[e];
      k.nk = (k.rows + kTileK - 1) / kTileK;
    } else {
      const int first = off[e], last = e < E ? off[e + 1] : a.P;
      tm = (last - first + AM - 1) / AM;
      k.row0 = first;
      k.rows = last - first;
      k.nk = e < E ? a.nk : 0;
    }
    const int band = rel / (kBand * tn), in = rel - band * kBand * tn;
    const int h = min(kBand, tm - band * kBand);
    k.n = in / h;
    k.m = band * kBand + in - k.n * h;
    if (MODE != kGradW) {
      k.row0 += k.m * AM;
      k.rows = min(AM, k.rows - k.m * AM);
    }
    return true;
  }
};

__device__ __forceinline__ float silu(float g) { return g / (1.f + __expf(-g)); }

template <typename T, int MODE, bool GATED, int AM>
__global__ void __launch_bounds__(kThreads, 1) expert_mm_kernel(const __grid_constant__ CUtensorMap tmA,
                                                                const __grid_constant__ CUtensorMap tmB,
                                                                const ExpertMmArgs a) {
  using C = Cfg<AM>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (pm::smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty = full + kStages;
  uint64_t* d_full = empty + kStages;  // [2]
  uint64_t* d_empty = d_full + 2;      // [2]
  uint64_t* drain = d_empty + 2;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tslot + 1);
  int32_t* off = reinterpret_cast<int32_t*>(smem + C::kBarOff + 256);
  int32_t* start = off + a.E + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == 0) {
    pm::tmem_alloc(tslot, 512);
    pm::tmem_relinquish();
  }
  if (tid == 32) {
    for (int s = 0; s < kStages; ++s) {
      pm::mbar_init(full + s, 1);
      pm::mbar_init(empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      pm::mbar_init(d_full + s, 1);
      pm::mbar_init(d_empty + s, 4);
    }
    pm::mbar_init(drain, 1);
    *abort_flag = 0;
    pm::fence_mbar_init();
  }
  if (warp == 2) {
    // offsets, clamped to 0 = off[0] <= off[e] <= off[e + 1] <= P (a wrong table must not reach memory), and tiles
    int carry_off = 0, carry_t = 0;
    for (int e0 = 0; e0 <= a.E; e0 += 32) {
      const int e = e0 + lane;
      int o = e > 0 && e <= a.E ? min(max(a.offsets[e], 0), a.P) : 0;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, o, s);
        if (lane >= s) o = max(o, u);
      }
      o = max(o, carry_off);
      if (e <= a.E) off[e] = o;
      carry_off = __shfl_sync(0xffffffffu, o, 31);
    }
    __syncwarp();
    for (int e0 = 0; e0 <= a.E; e0 += 32) {
      const int e = e0 + lane;
      int c = 0;
      if (e <= a.E) {
        if (MODE == kGradW)
          c = e < a.E ? a.tiles_m * a.tiles_n : 0;
        else
          c = ((e < a.E ? off[e + 1] : a.P) - off[e] + AM - 1) / AM * a.tiles_n;
      }
      int inc = c;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, s);
        if (lane >= s) inc += u;
      }
      if (e <= a.E) start[e + 1] = carry_t + inc;
      carry_t += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) start[0] = 0;
  }
  pm::tc_fence_before();
  __syncthreads();
  pm::tc_fence_after();
  const uint32_t tmem = *tslot;
  Walker<MODE, AM> walk(a, start, off);
  Tile t;
  // For converged warps: the same answer in every lane (tcgen05 instructions are warp-collective).
  auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
    const bool ok = __all_sync(0xffffffffu, pm::mbar_wait(bar, parity, lane == 0 ? a.err : nullptr, site));
    if (!ok) *abort_flag = 1;
    return ok;
  };
  auto stopped = [&] { return __any_sync(0xffffffffu, *abort_flag != 0) != 0; };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int st = 0, issued = 0;
      uint32_t ph = 0, last_ph[kStages];
      while (!*abort_flag && walk.next(t)) {
        for (int i = 0; i < t.nk; ++i) {
          if (!pm::mbar_wait(empty + st, ph ^ 1, a.err, 401)) {
            *abort_flag = 1;
            break;
          }
          uint8_t* sa = smem + st * C::kStageBytes;
          uint8_t* sb = sa + C::kABytes;
          pm::mbar_arrive_expect_tx(full + st, C::kStageBytes);
          const int k0 = i * kTileK;
          if (MODE == kGradW) {
            const int r0 = t.row0 + k0;
#pragma unroll
            for (int c = 0; c < 2; ++c) pm::tma_load_2d(sa + c * kChunk, &tmA, t.m * kTileM + 64 * c, r0, full + st);
#pragma unroll
            for (int c = 0; c < 4; ++c) pm::tma_load_2d(sb + c * kChunk, &tmB, t.n * kTileN + 64 * c, r0, full + st);
          } else {
            pm::tma_load_2d(sa, &tmA, k0, t.row0, full + st);
            if (MODE == kForward && GATED)  // 128 gate rows, then the matching 128 up rows
              pm::tma_load_4d(sb, &tmB, k0, t.n * (kTileN / 2), 0, t.e, full + st);
            else if (MODE == kForward)
              pm::tma_load_4d(sb, &tmB, k0, t.n * kTileN, t.e, 0, full + st);
            else
#pragma unroll
              for (int c = 0; c < 4; ++c)
                pm::tma_load_4d(sb + c * kChunk, &tmB, t.n * kTileN + 64 * c, k0, t.e, 0, full + st);
          }
          last_ph[st] = ph;
          if (issued < kStages) ++issued;
          if (++st == kStages) { st = 0; ph ^= 1; }
        }
      }
      if (*abort_flag)  // let the copies in flight land before the CTA can exit
        for (int j = 1; j <= issued; ++j) {
          const int s = (st - j + kStages) % kStages;
          pm::mbar_wait(full + s, last_ph[s], nullptr, 0, 20000000ull);
        }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (converged warp)
    const uint32_t idesc = pm::make_idesc_f16(kTileM, kTileN, sizeof(T) == 2 && a.half == 0 ? 1 : 0,
                                              MODE == kGradW ? 1 : 0, MODE == kForward ? 0 : 1);
    int st = 0, buf = 0;
    uint32_t ph = 0, dph = 0;
    while (!stopped() && walk.next(t)) {
      if (t.nk == 0) continue;
      if (!wait(d_empty + buf, dph ^ 1, 402)) break;
      pm::tc_fence_after();
      const uint32_t d = tmem + buf * kTileN;
      bool ok = true;
      for (int i = 0; i < t.nk; ++i) {
        ok = wait(full + st, ph, 403);
        if (!ok) break;
        uint8_t* sp = smem + st * C::kStageBytes;
        int steps = 4;
        if (MODE == kGradW && t.rows - i * kTileK < kTileK) {
          // the expert's last stage: its steps of 16 rows, the last of them completed with zero rows
          const int have = t.rows - i * kTileK;
          steps = (have + 15) / 16;
          const int pad = steps * 16 - have;
          for (int j = lane; j < pad * 6 * 8; j += 32) {
            const int chunk = j / (pad * 8), in = j - chunk * pad * 8, r = have + in / 8;
            *reinterpret_cast<uint4*>(sp + chunk * kChunk + r * 128 + (in & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          pm::fence_proxy_async_smem();
          __syncwarp();
        }
        pm::tc_fence_after();
        const uint32_t sa = pm::smem_u32(sp), sb = sa + C::kABytes;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (MODE == kGradW && k >= steps) break;
          const uint64_t ad = MODE == kGradW ? pm::make_sdesc(sa + k * 2048, kChunk, 1024)
                                             : pm::make_sdesc(sa + 32 * k, 16, 1024);
          const uint64_t bd = MODE == kForward ? pm::make_sdesc(sb + 32 * k, 16, 1024)
                                               : pm::make_sdesc(sb + k * 2048, kChunk, 1024);
          pm::umma_f16_warp(d, ad, bd, idesc, (i | k) ? 1u : 0u);
        }
        pm::umma_commit_warp(empty + st);
        if (++st == kStages) { st = 0; ph ^= 1; }
      }
      if (!ok) break;
      pm::umma_commit_warp(d_full + buf);
      buf ^= 1;
      if (buf == 0) dph ^= 1;
    }
    pm::umma_commit_warp(drain);  // arrives once every MMA issued above has completed
    pm::mbar_wait(drain, 0, lane == 0 ? a.err : nullptr, 404);
  } else {
    // ------------------------------------------------------------------ epilogue (warps 2-5)
    const int q = warp & 3;
    uint8_t* stage = smem + C::kEpiOff + (warp - 2) * kEpiWarpBytes;
    int buf = 0;
    uint32_t dph = 0;
    // One output row is `ld` elements; columns [c0, c0 + 64) of it, as far as `cols` reaches
    auto emit = [&](T* out, int64_t ld, int rows_here, int c0, int cols, const uint4 (&v)[8]) {
#pragma unroll
      for (int u = 0; u < 8; ++u) *reinterpret_cast<uint4*>(stage + lane * 128 + ((u ^ (lane & 7)) << 4)) = v[u];
      __syncwarp();
      // 8 lanes write the 128 bytes of a row: whole lines, four rows an instruction
      const int u = lane & 7;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const int r = g * 4 + (lane >> 3);
        const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 128 + ((u ^ (r & 7)) << 4));
        if (r < rows_here && c0 + u * 8 < cols) *reinterpret_cast<uint4*>(out + r * ld + c0 + u * 8) = w;
      }
      __syncwarp();
    };
    auto pack = [&](const float* f, uint4 (&v)[8]) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = make_uint4(rows::pack2<T>(f[8 * u], f[8 * u + 1]), rows::pack2<T>(f[8 * u + 2], f[8 * u + 3]),
                          rows::pack2<T>(f[8 * u + 4], f[8 * u + 5]), rows::pack2<T>(f[8 * u + 6], f[8 * u + 7]));
    };
    while (!stopped() && walk.next(t)) {
      const bool zero = t.nk == 0;
      if (!zero) {
        if (!wait(d_full + buf, dph, 405)) break;
        pm::tc_fence_after();
      }
      const uint32_t td = tmem + buf * kTileN + ((uint32_t)(32 * q) << 16);
      const int lim = MODE == kGradW ? a.M - t.m * kTileM : t.rows;  // rows of the tile that exist
      const int here = min(32, lim - 32 * q);
      if (here > 0) {
        const int64_t row = (MODE == kGradW ? (int64_t)t.e * a.M + t.m * kTileM : (int64_t)t.row0) + 32 * q;
        uint4 v[8];
        if (GATED) {
          const int I = a.N / 2;
#pragma unroll 1
          for (int c = 0; c < kTileN / 2; c += 64) {
            const int c0 = t.n * (kTileN / 2) + c;
            float g[64], u[64];
            if (zero) {
#pragma unroll
              for (int i = 0; i < 64; ++i) g[i] = u[i] = 0.f;
            } else {
              pm::tmem_ld32(td + c, *reinterpret_cast<float(*)[32]>(g));
              pm::tmem_ld32(td + c + 32, *reinterpret_cast<float(*)[32]>(g + 32));
              pm::tmem_ld32(td + c + 128, *reinterpret_cast<float(*)[32]>(u));
              pm::tmem_ld32(td + c + 160, *reinterpret_cast<float(*)[32]>(u + 32));
            }
            if (a.pre) {  // the products themselves, for the backward pass
              T* pr = static_cast<T*>(a.pre) + row * a.N;
              pack(g, v);
              emit(pr, a.N, here, c0, I, v);
              pack(u, v);
              emit(pr + I, a.N, here, c0, I, v);
            }
#pragma unroll
            for (int i = 0; i < 64; ++i) g[i] = silu(g[i]) * u[i];
            pack(g, v);
            emit(static_cast<T*>(a.out) + row * I, I, here, c0, I, v);
          }
        } else {
          T* out = static_cast<T*>(a.out) + row * a.N;
#pragma unroll 1
          for (int c = 0; c < kTileN; c += 64) {
            float f[64];
            if (zero) {
#pragma unroll
              for (int i = 0; i < 64; ++i) f[i] = 0.f;
            } else {
              pm::tmem_ld32(td + c, *reinterpret_cast<float(*)[32]>(f));
              pm::tmem_ld32(td + c + 32, *reinterpret_cast<float(*)[32]>(f + 32));
            }
            pack(f, v);
            emit(out, a.N, here, t.n * kTileN + c, a.N, v);
          }
        }
      }
      if (!zero) {
        pm::tc_fence_before();
        __syncwarp();
        if (lane == 0) pm::mbar_arrive(d_empty + buf);
        buf ^= 1;
        if (buf == 0) dph ^= 1;
      }
    }
  }
  pm::tc_fence_before();
  __syncthreads();
  if (warp == 0) pm::tmem_dealloc(tmem, 512);
}

// ----------------------------------------------------------------------------- SwiGLU gradient
// da = gradient of silu(g) u; z = [g | u] rows: dg = da u s (1 + g (1 - s)), du = da g s with s = sigmoid(g).
// Rows past offsets[E] are zero.  Memory bound: 6 bytes read and 4 written per value of da.
template <typename T>
__global__ void __launch_bounds__(256) swiglu_bwd_kernel(const T* __restrict__ da, int64_t das,
                                                         const T* __restrict__ z, int64_t zs, T* __restrict__ dz,
                                                         int64_t P, int I, const int32_t* __restrict__ offsets, int E) {
  const int nv = I / 8;
  const int64_t total = offsets[E];
  for (int64_t row = blockIdx.x; row < P; row += gridDim.x) {
    for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < nv; c += gridDim.y * blockDim.x) {
      float d[8], g[8], u[8];
      if (row < total) {
        rows::load8<T>(da + row * das + c * 8, d);
        rows::load8<T>(z + row * zs + c * 8, g);
        rows::load8<T>(z + row * zs + I + c * 8, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float s = 1.f / (1.f + __expf(-g[i])), gs = g[i] * s;
          const float up = u[i];
          u[i] = d[i] * gs;
          g[i] = d[i] * up * (s + gs * (1.f - s));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = u[i] = 0.f;
      }
      *reinterpret_cast<uint4*>(dz + row * 2 * I + c * 8) = rows::pack8<T>(g);
      *reinterpret_cast<uint4*>(dz + row * 2 * I + I + c * 8) = rows::pack8<T>(u);
    }
  }
}

template <typename T, int MODE, bool GATED, int AM>
int launch_mm(const CUtensorMap& ta, const CUtensorMap& tb, const ExpertMmArgs& a, cudaStream_t stream) {
  const int smem = (int)(Cfg<AM>::kFixed + (2 * a.E + 3) * sizeof(int32_t));
  if (smem > 232448) return -2;
  auto* fn = expert_mm_kernel<T, MODE, GATED, AM>;
  cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  fn<<<a.num_sms, kThreads, smem, stream>>>(ta, tb, a);
  return 0;
}

template <typename T>
int launch_mode(int mode, bool gated, bool few, const CUtensorMap& ta, const CUtensorMap& tb, const ExpertMmArgs& a,
                cudaStream_t s) {
  if (mode == kGradW) return launch_mm<T, kGradW, false, 128>(ta, tb, a, s);
  if (mode == kGradX) return launch_mm<T, kGradX, false, 128>(ta, tb, a, s);
  if (gated) return few ? launch_mm<T, kForward, true, 32>(ta, tb, a, s) : launch_mm<T, kForward, true, 128>(ta, tb, a, s);
  return few ? launch_mm<T, kForward, false, 32>(ta, tb, a, s) : launch_mm<T, kForward, false, 128>(ta, tb, a, s);
}

}  // namespace

// mode 0: out [P, N or N/2] = rows [P, K] of `x` with w [E, N, K]; 1: out [P, K] = dz [P, N] with w;
// 2: out [E, N, K] = dz [P, N] with x [P, K].  Returns 0, or the tensor-map encoding's error.
int launch_expert_mm(int mode, const ExpertMmCall& c, cudaStream_t stream) {
  ExpertMmArgs a{};
  a.E = c.E;
  a.P = (int)c.P;
  a.offsets = c.offsets;
  a.out = c.out;
  a.pre = c.pre;
  a.half = c.half;
  a.num_sms = c.num_sms;
  a.err = c.err;
  const uint64_t K = c.K, N = c.N, E = c.E, P = c.P;
  const bool few = mode == kForward && c.P <= (int64_t)32 * c.E;
  CUtensorMap ta, tb;
  int rc;
  if (mode == kForward) {
    const uint64_t da[2] = {K, P}, sa[1] = {(uint64_t)c.xs * 2};
    const uint32_t ba[2] = {kTileK, few ? 32u : 128u};
    rc = make_tmap_16b_sw128(&ta, c.x, 2, da, sa, ba, c.half);
    if (c.gated) {
      const uint64_t db[4] = {K, N / 2, 2, E}, sb[3] = {K * 2, N / 2 * K * 2, N * K * 2};
      const uint32_t bb[4] = {kTileK, 128, 2, 1};
      if (!rc) rc = make_tmap_16b_sw128(&tb, c.w, 4, db, sb, bb, c.half);
    } else {
      const uint64_t db[4] = {K, N, E, 1}, sb[3] = {K * 2, N * K * 2, E * N * K * 2};
      const uint32_t bb[4] = {kTileK, 256, 1, 1};
      if (!rc) rc = make_tmap_16b_sw128(&tb, c.w, 4, db, sb, bb, c.half);
    }
    a.N = (int)N;
    a.nk = (int)((K + kTileK - 1) / kTileK);
    a.tiles_n = (int)(((c.gated ? N / 2 : N) + (c.gated ? 127 : 255)) / (c.gated ? 128 : 256));
  } else {
    const uint64_t da[2] = {N, P}, sa[1] = {(uint64_t)c.dzs * 2};
    const uint32_t ba[2] = {kTileK, mode == kGradX ? 128u : 64u};
    rc = make_tmap_16b_sw128(&ta, c.dz, 2, da, sa, ba, c.half);
    a.N = (int)K;
    a.tiles_n = (int)((K + kTileN - 1) / kTileN);
    if (mode == kGradX) {
      const uint64_t db[4] = {K, N, E, 1}, sb[3] = {K * 2, N * K * 2, E * N * K * 2};
      const uint32_t bb[4] = {64, kTileK, 1, 1};
      if (!rc) rc = make_tmap_16b_sw128(&tb, c.w, 4, db, sb, bb, c.half);
      a.nk = (int)((N + kTileK - 1) / kTileK);
    } else {
      const uint64_t db[2] = {K, P}, sb[1] = {(uint64_t)c.xs * 2};
      const uint32_t bb[2] = {64, kTileK};
      if (!rc) rc = make_tmap_16b_sw128(&tb, c.x, 2, db, sb, bb, c.half);
      a.M = (int)N;
      a.tiles_m = (int)((N + kTileM - 1) / kTileM);
    }
  }
  if (rc) return rc;
  return c.half ? launch_mode<__half>(mode, c.gated, few, ta, tb, a, stream)
                : launch_mode<__nv_bfloat16>(mode, c.gated, few, ta, tb, a, stream);
}

void launch_swiglu_bwd(const void* da, int64_t das, const void* z, int64_t zs, void* dz, int64_t P, int I,
                       const int32_t* offsets, int E, int half, int num_sms, cudaStream_t stream) {
  if (P == 0 || I == 0) return;
  const int nv = I / 8, threads = nv >= 256 ? 256 : (nv + 31) / 32 * 32;
  const int64_t most = (int64_t)num_sms * 32;
  const dim3 grid((unsigned)(P < most ? P : most), P < 4 * num_sms ? (nv + threads - 1) / threads : 1);
  if (half)
    swiglu_bwd_kernel<__half><<<grid, threads, 0, stream>>>(static_cast<const __half*>(da), das,
                                                            static_cast<const __half*>(z), zs,
                                                            static_cast<__half*>(dz), P, I, offsets, E);
  else
    swiglu_bwd_kernel<__nv_bfloat16><<<grid, threads, 0, stream>>>(
        static_cast<const __nv_bfloat16*>(da), das, static_cast<const __nv_bfloat16*>(z), zs,
        static_cast<__nv_bfloat16*>(dz), P, I, offsets, E);
}
