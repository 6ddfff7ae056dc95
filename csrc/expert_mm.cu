// Matrix products of every expert's rows in one launch (tcgen05, BF16 or FP16 operands, fp32 accumulators).
//
//   kForward   y_e  = act(x_e W_e^T)     rows of x sorted by expert, W [E, N, K]; act: none, or SwiGLU over
//                                        W's rows [gate I | up I]: y = silu(g) u
//   kGradX     dx_e = dz_e W_e
//   kGradW     dW_e = dz_e^T x_e         (zero for an expert without rows)
//
// Expert e owns rows offsets[e] .. offsets[e + 1]; the offsets are read on the device, so no call waits for
// the host.  Rows before offsets[0] (a table of some of a larger table's experts) and past offsets[E] give zero rows
// (kForward, kGradX) and are not read (kGradW).
#include <cuda.h>

#include "launchers.h"
#include "common/sm100.cuh"
#include "common/rows.cuh"

namespace {

constexpr int kTileK = 64;         // of the reduced dimension per stage: 128 bytes, one swizzle row
constexpr int kMaxStages = 8;
enum Mode { kForward = 0, kGradX = 1, kGradW = 2 };

// Fast division and exponential: the full ones' extra instructions lengthened the gated epilogue by half.  The division
// is within 2 units in the last place; the exponential's bound grows with |g| (2 + 1.17 |g| units), to 2^-16 of it where
// it leaves fp32: far below the outputs' rounding (2^-8 BF16, 2^-11 FP16).  A denominator beyond 2^126, infinity included, gives 0.
__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }
__device__ __forceinline__ float silu(float g) { return __fdividef(g, 1.f + __expf(-g)); }

// off[0 .. E]: the running maximum of the offsets, clamped to 0 .. P (a wrong table must not reach memory);
// start[0 .. E + 2]: first tile of each expert, for tiles(rows of e, e) tiles each; "expert" E is the rows past the
// last one and "expert" E + 1 those before the first.  Called by one warp.
__device__ __forceinline__ int first_row(const ExpertMmArgs& a, const int32_t* off, int e) { return e <= a.E ? off[e] : 0; }
__device__ __forceinline__ int row_count(const ExpertMmArgs& a, const int32_t* off, int e) {
  return e < a.E ? off[e + 1] - off[e] : e == a.E ? a.P - off[e] : off[0];
}
template <typename Tiles>
__device__ __forceinline__ void tile_table(const ExpertMmArgs& a, int32_t* off, int32_t* start, int lane, Tiles tiles) {
  int carry_off = 0, carry_t = 0;
  for (int e0 = 0; e0 <= a.E; e0 += 32) {
    const int e = e0 + lane;
    int o = e <= a.E ? min(max(a.offsets[e], 0), a.P) : 0;
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
  for (int e0 = 0; e0 <= a.E + 1; e0 += 32) {
    const int e = e0 + lane;
    int inc = e <= a.E + 1 ? tiles(row_count(a, off, e), e) : 0;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, s);
      if (lane >= s) inc += u;
    }
    if (e <= a.E + 1) start[e + 1] = carry_t + inc;
    carry_t += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) start[0] = 0;
}

// ----------------------------------------------------------------------------- CTA pairs
// A pair (a cluster of two CTAs) computes D [256 x N], N <= 256: CTA r holds rows 128 r .. of A and of D, and
// half of B's N rows, so that each operand byte crosses from L2 to shared memory once per pair.  That crossing
// is what bounds a single-CTA kernel: 128 x 256 tiles take 48 KB per 512 tensor cycles, 96 bytes a cycle of an
// SM, and ran at 76 % of the tensor pipe; 256 x 256 pairs take 64 and run at 94 %.  The accumulator is
// double-buffered in TMEM, so a tile's epilogue overlaps the next tile's products.  With few rows an expert (a
// decode step) the weights' stream from HBM is the bound: six stages of up to 32 KB in flight per SM.
//
//   kForward, kGradX: A is the weight (256 output features), B the rows (tokens): D is y^T.  An expert's rows
//     are cut into tiles of at most 256, and N is the tile's rows rounded up to 32 (the MMA's step), so a
//     ragged expert costs its rows and not a multiple of a fixed tile.  The epilogue turns D through shared
//     memory.  Gated: A takes gate and up rows by turns, 8 and 8, so that a feature's two products lie 8 TMEM
//     lanes apart and meet by one exchange within the warp.
//   kGradW: A is dz^T (256 of n), B x^T (256 of k), both MN-major, reduced over the expert's rows.  The last
//     stage reads into the next expert's rows, and 0 x NaN is NaN: a warp of each CTA zeroes those rows of both
//     its operands in shared memory, ahead of the MMA.
//   kGradX reads W along its other dimension by an MN-major descriptor: nothing is transposed in memory.
constexpr int kEpiWarps = 8;
constexpr int kTrimWarp = 2 + kEpiWarps;
// warp 0 TMA producer, 1 MMA issuer (leader), 2-9 epilogue, kGradW: 10 ragged rows
constexpr int pair_threads(int mode) { return 32 * (kTrimWarp + (mode == kGradW ? 1 : 0)); }
constexpr uint32_t kEpiWarpBytes = 32 * 64;  // staging of an epilogue warp: 32 rows x 32 columns
constexpr uint32_t kHalf = 128 * 128;    // 128 rows x 64 elements: one CTA's A rows, or its half of B
constexpr uint32_t kChunk = 64 * 128;    // MN-major operands: 64 reduced rows x 64 columns
constexpr int kBand = 8;                 // row tiles that walk the feature tiles together (L2 reuse of both)

struct Pair {
  static constexpr uint32_t kABytes = kHalf;
  static constexpr uint32_t kStageBytes = kABytes + kHalf;
  static constexpr int kStages = 6;
  static constexpr uint32_t kEpiOff = kStages * kStageBytes;
  static constexpr uint32_t kBarOff = kEpiOff + kEpiWarps * kEpiWarpBytes;
  static constexpr uint32_t kTableOff = kBarOff + 512;
  static constexpr uint32_t kFixed = kTableOff + 1024;  // and alignment; then the tile table
};

struct PairTile {
  int e, m, n;     // expert; feature tile (n of dW); row tile (k of dW)
  int row0, rows;  // kForward / kGradX: the tile's rows; kGradW: the expert's
  int cols;        // B rows of the MMA: a multiple of 32
  int nk;          // stages (0: the tile is zero)
};

template <int MODE>
struct PairWalker {
  const ExpertMmArgs& a;
  const int32_t *start, *off;
  int e, t;
  __device__ PairWalker(const ExpertMmArgs& args, const int32_t* s, const int32_t* o) : a(args), start(s), off(o) {
    e = 0;
    t = (int)(blockIdx.x >> 1) - (int)(gridDim.x >> 1);
  }
  __device__ bool next(PairTile& k) {
    t += gridDim.x >> 1;
    const int E = a.E;
    if (t >= start[E + 2]) return false;
    while (t >= start[e + 1]) ++e;
    const int rel = t - start[e], first = first_row(a, off, e), rows = row_count(a, off, e);
    const int tn = MODE == kGradW ? a.tiles_n : (rows + 255) / 256;
    const int band = rel / (kBand * a.tiles_m), in = rel - band * kBand * a.tiles_m, h = min(kBand, tn - band * kBand);
    k.e = e;
    k.m = in / h;
    k.n = band * kBand + in - k.m * h;
    if (MODE == kGradW) {
      k.row0 = first;
      k.rows = rows;
      k.nk = (rows + kTileK - 1) / kTileK;
      k.cols = min(256, (a.N - k.n * 256 + 31) / 32 * 32);
    } else {
      // whole tiles, but the last two share what is left evenly (in steps of 32): a short last tile would cost its
      // weights' loads, which take half the time of a whole tile
      const int left = rows - (tn - 2) * 256, q = tn < 2 ? rows : min(256, ((left + 1) / 2 + 31) / 32 * 32);
      const int at = tn < 2 || k.n < tn - 1 ? k.n * 256 : (tn - 2) * 256 + q;
      k.row0 = first + at;
      k.rows = k.n < tn - 2 ? 256 : k.n == tn - 1 ? rows - at : q;
      k.cols = (k.rows + 31) / 32 * 32;
      k.nk = e < E ? a.nk : 0;
    }
    return true;
  }
};

template <typename T, int MODE, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair_threads(MODE), 1)
    expert_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const __grid_constant__ CUtensorMap tmB64, const __grid_constant__ CUtensorMap tmB32,
                       const ExpertMmArgs a) {
  using C = Pair;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (pm::smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);  // leader's: both CTAs' loads of a stage
  uint64_t* empty = full + kMaxStages;       // each CTA's: the MMA has read its stage
  uint64_t* tail = empty + kMaxStages;       // kGradW, each CTA's: loads of an expert's ragged last stage
  uint64_t* trimmed = tail + kMaxStages;     // leader's: both CTAs have zeroed the rows past the expert's last
  uint64_t* d_full = trimmed + kMaxStages;   // [2], each CTA's
  uint64_t* d_empty = d_full + 2;            // [2], leader's: epilogue warps of both CTAs
  uint64_t* drain = d_empty + 2;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tslot + 1);
  int32_t* off = reinterpret_cast<int32_t*>(smem + C::kTableOff);
  int32_t* start = off + a.E + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)pm::cluster_ctarank();

  if (warp == 0) {
    pm::tmem_alloc2(tslot, 512);
    pm::tmem_relinquish2();
  }
  if (tid == 32) {
    for (int s = 0; s < kStages; ++s) {
      pm::mbar_init(full + s, 1);
      pm::mbar_init(empty + s, 1);
      pm::mbar_init(tail + s, 1);
      pm::mbar_init(trimmed + s, 2);
    }
    for (int s = 0; s < 2; ++s) {
      pm::mbar_init(d_full + s, 1);
      pm::mbar_init(d_empty + s, 2 * kEpiWarps);
    }
    pm::mbar_init(drain, 1);
    *abort_flag = 0;
    pm::fence_mbar_init();
  }
  if (warp == 2)
    tile_table(a, off, start, lane, [&](int rows, int e) {
      return MODE == kGradW ? (e < a.E ? a.tiles_m * a.tiles_n : 0) : (rows + 255) / 256 * a.tiles_m;
    });
  pm::tc_fence_before();
  __syncthreads();
  pm::cluster_sync();  // the peer's barriers exist
  pm::tc_fence_after();
  const uint32_t tmem = *tslot;
  PairWalker<MODE> walk(a, start, off);
  PairTile t;
  auto wait = [&](uint32_t bar, uint32_t parity, int site) {
    if (pm::mbar_wait_warp(bar, parity, a.err, site)) return true;
    *abort_flag = 1;
    return false;
  };
  auto wait_cluster = [&](uint32_t bar, uint32_t parity, int site) {
    if (pm::mbar_wait_warp<true>(bar, parity, a.err, site)) return true;
    *abort_flag = 1;
    return false;
  };
  auto stopped = [&] { return __any_sync(0xffffffffu, *abort_flag != 0) != 0; };
  const uint32_t base = pm::smem_u32(smem), full_at = pm::smem_u32(full), empty_at = pm::smem_u32(empty);

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (each CTA its own halves)
    const uint32_t full_leader = pm::dsmem_addr(full, 0);
    int st = 0, issued = 0;
    uint32_t ph = 0;
    while (!stopped() && walk.next(t)) {
      // B rows (kGradW: columns) of this CTA.  kForward, kGradX: at most two boxes, because each load costs the
      // producer as much as 16 rows cost the transfer: 112 and 128 rows come as 128, 80 and 96 as 64 + 32,
      // 48 and 64 as 64, less as 32.
      const int half = t.cols >> 1;
      const int parts = MODE == kGradW ? (half + 63) / 64 : half == 80 || half == 96 ? 2 : 1;
      const uint32_t bytes = C::kABytes + (MODE == kGradW ? parts * kChunk : half > 96 ? kHalf : half > 64 ? 96 * 128 : half > 32 ? 64 * 128 : 32 * 128);
      const CUtensorMap* mb = half > 96 ? &tmB : half > 32 ? &tmB64 : &tmB32;
      const int f0 = t.m * 256 + rank * 128, r0 = t.row0 + rank * half, c0 = t.n * 256 + rank * half;
      const bool simple = MODE == kForward || (a.a_chunks == 2 && (MODE == kGradX || (a.b_chunks == 2 && half == 128)));
      for (int i = 0; i < t.nk; ++i) {
        if (!wait(empty_at + 8 * st, ph ^ 1, 401)) break;
        const uint32_t sa = base + st * C::kStageBytes, sb = sa + C::kABytes;
        const int k0 = i * kTileK;
        uint32_t bar = full_leader + 8 * st;
        if (MODE == kGradW && t.rows - k0 < kTileK) {  // ragged rows: the loads of each CTA are its own
          if (rank == 0) pm::mbar_arrive_expect_tx_warp(full_at + 8 * st, 0);
          bar = pm::dsmem_addr(tail + st, rank);
          pm::mbar_arrive_expect_tx_warp(pm::smem_u32(tail + st), bytes);
        } else if (rank == 0) {
          pm::mbar_arrive_expect_tx_warp(full_at + 8 * st, 2 * bytes);
        }
        if (simple) {
          if (MODE == kGradW)
            pm::tma2_stage_55_warp(sa, &tmA, t.row0 + k0, f0 >> 6, sb, &tmB, c0 >> 6, bar);
          else if (MODE == kGradX)
            pm::tma2_stage_52_warp(sa, &tmA, 0, k0, f0 >> 6, t.e, 0, sb, mb, k0, r0, bar);
          else if (GATED)  // 8 groups of 8 gate rows and the matching 8 up rows
            pm::tma2_stage_52_warp(sa, &tmA, k0, 0, 0, f0 >> 4, t.e, sb, mb, k0, r0, bar);
          else
            pm::tma2_stage_52_warp(sa, &tmA, k0, f0, t.e, 0, 0, sb, mb, k0, r0, bar);
        } else {  // MN-major operands whose chunks are no dimension: a load for each
          const int y = MODE == kGradW ? t.row0 + k0 : k0, w = MODE == kGradW ? 0 : t.e;
          if (a.a_chunks == 2) {
            pm::tma2_load_5d_warp(sa, &tmA, 0, y, f0 >> 6, w, 0, bar);
          } else {
            pm::tma2_load_5d_warp(sa, &tmA, f0, y, 0, w, 0, bar);
            pm::tma2_load_5d_warp(sa + kChunk, &tmA, f0 + 64, y, 0, w, 0, bar);
          }
          if (MODE == kGradX) {
            pm::tma2_load_2d_warp(sb, mb, k0, r0, bar);
          } else {
            pm::tma2_load_2d_warp(sb, &tmB64, c0, y, bar);
            if (parts == 2) pm::tma2_load_2d_warp(sb + kChunk, &tmB64, c0 + 64, y, bar);
          }
        }
        if (MODE != kGradW && parts == 2) pm::tma2_load_2d_warp(sb + 64 * 128, &tmB32, k0, r0 + 64, bar);
        if (issued < kStages) ++issued;
        if (++st == kStages) { st = 0; ph ^= 1; }
      }
    }
    // Every load has landed once the MMA has read its stage: wait for the last ones, so that no copy into this
    // CTA is in flight when it leaves.
    const bool gone = stopped();
    for (int j = 1; j <= issued; ++j) {
      const int s = (st - j + kStages) % kStages;
      pm::mbar_wait_warp(empty_at + 8 * s, s < st ? ph : ph ^ 1, gone ? nullptr : a.err, 406, gone ? 20000000ull : 2000000000ull);
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------------ MMA issuer (leader)
    // stage 0's operands; 16 of the reduced dimension are 32 bytes of a K-major row, 16 rows of an MN-major chunk
    constexpr int kAStep = MODE == kForward ? 2 : 128, kBStep = MODE == kGradW ? 128 : 2;
    const uint64_t a0 = pm::make_sdesc(base, MODE == kForward ? 16 : kChunk, 1024);
    const uint64_t b0 = pm::make_sdesc(base + C::kABytes, MODE == kGradW ? kChunk : 16, 1024);
    int st = 0, buf = 0;
    uint32_t ph = 0, dph = 0, trim_ph = 0;
    while (!stopped() && walk.next(t)) {
      if (t.nk == 0) continue;
      if (!wait_cluster(pm::smem_u32(d_empty + buf), dph ^ 1, 402)) break;
      pm::tc_fence_after();
      const uint32_t idesc = pm::make_idesc_f16(256, t.cols, a.half ? 0 : 1, MODE == kForward ? 0 : 1, MODE == kGradW ? 1 : 0);
      const uint32_t d = tmem + buf * 256;
      bool ok = true;
      for (int i = 0; i < t.nk; ++i) {
        const uint64_t ad = a0 + st * (C::kStageBytes >> 4), bd = b0 + st * (C::kStageBytes >> 4);
        const int have = t.rows - i * kTileK;
        if (MODE == kGradW && have < kTileK) {  // the ragged stage is ready when both CTAs have zeroed its rows
          ok = wait_cluster(pm::smem_u32(trimmed + st), (trim_ph >> st) & 1, 403);
          if (!ok) break;
          trim_ph ^= 1u << st;
          pm::tc_fence_after();
          for (int k = 0; k < (have + 15) / 16; ++k)
            pm::umma2_f16_warp(d, ad + k * kAStep, bd + k * kBStep, idesc, (i | k) ? 1u : 0u);
          pm::umma2_commit_both_warp(empty + st);
        } else {
          ok = wait(full_at + 8 * st, ph, 404);
          if (!ok) break;
          pm::tc_fence_after();
          pm::umma2_f16_stage_warp<kAStep, kBStep>(d, ad, bd, idesc, i ? 1u : 0u, empty_at + 8 * st);
        }
        if (++st == kStages) { st = 0; ph ^= 1; }
      }
      if (!ok) break;
      pm::umma2_commit_both_warp(d_full + buf);
      buf ^= 1;
      if (buf == 0) dph ^= 1;
    }
    // every MMA issued above has completed; the peer, where nobody waits for this, gets no arrival: it may be leaving
    pm::umma2_commit_own_warp(drain);
    pm::mbar_wait_warp(pm::smem_u32(drain), 0, a.err, 407);
  } else if (MODE == kGradW && warp == kTrimWarp) {
    // ------------------------------------------------------------------ ragged rows (both CTAs)
    // The MMA takes steps of 16 rows: the last one of an expert is completed with zero rows in every column chunk
    // (4 chunks of 8 16-byte units: a lane each).
    const uint32_t trimmed_leader = pm::dsmem_addr(trimmed, 0);
    int st = 0;
    uint32_t ph = 0;
    while (!stopped() && walk.next(t)) {
      if (t.nk == 0) continue;
      st = (st + t.nk - 1) % kStages;
      const int have = t.rows - (t.nk - 1) * kTileK;
      if (have < kTileK) {
        if (!wait(pm::smem_u32(tail + st), (ph >> st) & 1, 408)) break;
        ph ^= 1u << st;
        if ((lane >> 3) < 2 + ((t.cols >> 1) + 63) / 64) {
          uint8_t* at = smem + st * C::kStageBytes + (lane >> 3) * kChunk + (lane & 7) * 16;
          for (int r = have; r & 15; ++r) *reinterpret_cast<uint4*>(at + r * 128) = make_uint4(0, 0, 0, 0);
        }
        pm::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) pm::mbar_arrive_cluster(trimmed_leader + 8 * st);
      }
      if (++st == kStages) st = 0;
    }
  } else if (warp >= 2 && warp < 2 + kEpiWarps) {
    // ------------------------------------------------------------------ epilogue (warps 2-9 of both CTAs)
    const int q = warp & 3, side = (warp - 2) >> 2;  // TMEM lane quadrant; half of the columns
    uint8_t* stage = smem + C::kEpiOff + (warp - 2) * kEpiWarpBytes;
    int buf = 0;
    uint32_t dph = 0;
    // y^T: lane = feature, v[i] = row i of 32.  Through shared memory [32 rows][32 features], then 64 bytes of a
    // row by 4 lanes: eight rows an instruction.  `out`: the first row's first feature of this warp.
    auto emit_t = [&](T* out, int64_t ld, int rows_here, int feats, const float (&v)[32]) {
#pragma unroll
      for (int i = 0; i < 32; ++i) *reinterpret_cast<T*>(stage + i * 64 + lane * 2) = rows::from_f<T>(v[i]);
      __syncwarp();
      const int u = lane & 3;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int r = g * 8 + (lane >> 2);
        const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 64 + u * 16);
        if (r < rows_here && u * 8 < feats) *reinterpret_cast<uint4*>(out + r * ld + u * 8) = w;
      }
      __syncwarp();
    };
    // The same for [gate | up] rows of ld elements: units of 8 lanes go to the gate and the up half by turns.
    auto emit_pre = [&](T* out, int64_t ld, int up_off, int rows_here, int feats, const float (&v)[32]) {
#pragma unroll
      for (int i = 0; i < 32; ++i) *reinterpret_cast<T*>(stage + i * 64 + lane * 2) = rows::from_f<T>(v[i]);
      __syncwarp();
      const int u = lane & 3;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int r = g * 8 + (lane >> 2);
        const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 64 + u * 16);
        if (r < rows_here && u * 8 < feats) *reinterpret_cast<uint4*>(out + r * ld + (u & 1) * up_off + (u >> 1) * 8) = w;
      }
      __syncwarp();
    };
    // silu(gate) up: 32 rows of 16 features; lane 16 j + f (gate) has rows 0-15 and lane 16 j + 8 + f rows 16-31 of
    // feature 8 j + f.
    auto emit_gated = [&](T* out, int64_t ld, int rows_here, int feats, const float (&o)[16]) {
      uint8_t* mine = stage + ((lane >> 3) & 1) * 16 * 32 + ((lane >> 4) * 8 + (lane & 7)) * 2;
#pragma unroll
      for (int i = 0; i < 16; ++i) *reinterpret_cast<T*>(mine + i * 32) = rows::from_f<T>(o[i]);
      __syncwarp();
      const int u = lane & 1;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int r = g * 16 + (lane >> 1);
        const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 32 + u * 16);
        if (r < rows_here && u * 8 < feats) *reinterpret_cast<uint4*>(out + r * ld + u * 8) = w;
      }
      __syncwarp();
    };
    while (!stopped() && walk.next(t)) {
      const bool zero = t.nk == 0;
      if (!zero) {
        if (!wait(pm::smem_u32(d_full + buf), dph, 405)) break;
        pm::tc_fence_after();
      }
      const uint32_t td = tmem + buf * 256 + ((uint32_t)(32 * q) << 16);
      if (MODE == kGradW) {
        // lane = n, columns = k: 32 columns a time, written as 64 bytes of a row by 4 lanes
        const int n0 = t.m * 256 + rank * 128 + 32 * q, here = min(32, a.M - n0);
        T* out = static_cast<T*>(a.out) + ((int64_t)t.e * a.M + n0) * a.N;
        if (here > 0) {
#pragma unroll 1
          for (int c = side * 128; c < side * 128 + 128 && c < t.cols; c += 32) {
            float f[32];
            if (zero) {
#pragma unroll
              for (int i = 0; i < 32; ++i) f[i] = 0.f;
            } else {
              pm::tmem_ld32(td + c, f);
            }
            // 16-byte units of a row permuted by row / 2: conflict-free both ways
#pragma unroll
            for (int u = 0; u < 4; ++u)
              *reinterpret_cast<uint4*>(stage + lane * 64 + ((u ^ ((lane >> 1) & 3)) << 4)) =
                  make_uint4(rows::pack2<T>(f[8 * u], f[8 * u + 1]), rows::pack2<T>(f[8 * u + 2], f[8 * u + 3]),
                             rows::pack2<T>(f[8 * u + 4], f[8 * u + 5]), rows::pack2<T>(f[8 * u + 6], f[8 * u + 7]));
            __syncwarp();
            const int u = lane & 3, col = t.n * 256 + c + u * 8;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int r = g * 8 + (lane >> 2);
              const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 64 + ((u ^ ((r >> 1) & 3)) << 4));
              if (r < here && col < a.N) *reinterpret_cast<uint4*>(out + (int64_t)r * a.N + col) = w;
            }
            __syncwarp();
          }
        }
      } else {
        const int f0 = t.m * 256 + rank * 128 + 32 * q, feats = a.N - f0;  // of W's rows; gated: 16 gates and 16 ups
        if (feats > 0) {
#pragma unroll 1
          for (int c = side * 32; c < t.rows; c += 64) {
            const int64_t row = (int64_t)t.row0 + c;
            const int here = t.rows - c;
            float v[32];
            if (zero) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.f;
            } else {
              pm::tmem_ld32(td + c, v);
            }
            if (!GATED) {
              emit_t(static_cast<T*>(a.out) + row * a.N + f0, a.N, here, feats, v);
              continue;
            }
            // the products themselves, for the backward pass: lanes 8 j .. 8 j + 7 are gates (j even) or ups
            const int I = a.N / 2, up = (lane >> 3) & 1;
            if (a.pre) emit_pre(static_cast<T*>(a.pre) + row * a.N + (f0 >> 1), a.N, I, here, feats, v);
            // lanes 8 apart trade halves: a gate lane then has rows 0-15 of both products, an up lane rows 16-31
            float o[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[16 + i], 8);
              o[i] = up ? silu(got) * v[16 + i] : silu(v[i]) * got;
            }
            emit_gated(static_cast<T*>(a.out) + row * I + (f0 >> 1), I, here, feats >> 1, o);
          }
        }
      }
      if (!zero) {
        pm::tc_fence_before();
        __syncwarp();
        // released: the leader's next products into these columns come after the warp's reads of them
        if (lane == 0) pm::mbar_arrive_cluster(pm::dsmem_addr(d_empty + buf, 0));
        buf ^= 1;
        if (buf == 0) dph ^= 1;
      }
    }
  }
  pm::tc_fence_before();
  __syncthreads();
  pm::cluster_sync();  // no CTA leaves while its peer may still signal it or read its operands
  pm::tc_fence_after();
  if (warp == 0) pm::tmem_dealloc2(tmem, 512);
}

// ----------------------------------------------------------------------------- SwiGLU gradient
// da = gradient of silu(g) u; z = [g | u] rows: dg = da u s (1 + g (1 - s)), du = da g s with s = sigmoid(g).
// dz is rounded to 16 bits because the products dx and dw take it as a tensor core operand, as z was when it was kept: the
// error of dx and dw is that of two roundings (0.0023 of their norm with BF16, 0.0017 with an fp32 dz).
// Rows before offsets[0] and past offsets[E] are zero.  Memory bound: 6 bytes read and 4 written per value of da; a block per row (58 us
// for 16384 x 2048, 5.8 TB/s; walking blocks 61 us).
template <typename T>
__global__ void __launch_bounds__(256) swiglu_bwd_kernel(const T* __restrict__ da, int64_t das,
                                                         const T* __restrict__ z, int64_t zs, T* __restrict__ dz,
                                                         int64_t P, int I, const int32_t* __restrict__ offsets, int E) {
  const int nv = I / 8;
  const int64_t row = blockIdx.x;
  const bool owned = row >= offsets[0] && row < offsets[E];
  for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < nv; c += gridDim.y * blockDim.x) {
    float d[8], g[8], u[8];
    if (owned) {
      rows::load8<T>(da + row * das + c * 8, d);
      rows::load8<T>(z + row * zs + c * 8, g);
      rows::load8<T>(z + row * zs + I + c * 8, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = sigmoid(g[i]), gs = g[i] * s;
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

constexpr int kMaxSmem = 232448;

template <typename T, int MODE, bool GATED>
int launch_pair(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb64, const CUtensorMap& tb32, const ExpertMmArgs& a,
                cudaStream_t stream) {
  const int smem = (int)(Pair::kFixed + (2 * a.E + 4) * sizeof(int32_t));
  if (smem > kMaxSmem) return -2;
  auto* fn = expert_pair_kernel<T, MODE, GATED>;
  // the limit is the kernel's, not this launch's: always the largest, or a launch of another host thread with fewer
  // experts could lower it before this one
  cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  fn<<<a.num_sms / 2 * 2, pair_threads(MODE), smem, stream>>>(ta, tb, tb64, tb32, a);
  return 0;
}
template <typename T>
int launch_mode(int mode, bool gated, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb64,
                const CUtensorMap& tb32, const ExpertMmArgs& a, cudaStream_t s) {
  if (mode == kGradW) return launch_pair<T, kGradW, false>(ta, tb, tb64, tb32, a, s);
  if (mode == kGradX) return launch_pair<T, kGradX, false>(ta, tb, tb64, tb32, a, s);
  return gated ? launch_pair<T, kForward, true>(ta, tb, tb64, tb32, a, s)
               : launch_pair<T, kForward, false>(ta, tb, tb64, tb32, a, s);
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

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
  const uint64_t K = c.K, N = c.N, E = c.E, P = c.P, I = N / 2;
  CUtensorMap ta, tb, tb64, tb32;  // A; B in boxes of 128, 64 and 32 rows (kGradW: two chunks, or one)
  const uint64_t dx[2] = {K, P}, sx[1] = {(uint64_t)c.xs * 2}, dd[2] = {N, P}, sd[1] = {(uint64_t)c.dzs * 2};
  const uint64_t dw[5] = {K, N, E, 1, 1}, sw[4] = {K * 2, N * K * 2, 16, 16};
  // gated weights: [E][I / 8][gate | up][8][K]
  const uint64_t dg[5] = {K, 8, 2, I / 8, E}, sg[4] = {K * 2, I * K * 2, 8 * K * 2, N * K * 2};
  int rc;
  // MN-major operands [stack][rows][width]: one box of 64 rows x 2 chunks of 64 columns, where the chunks of a row
  // can be a dimension of the tensor (64 divides the width); else a box for each chunk
  auto chunked = [&](CUtensorMap* m, const void* p, uint64_t width, uint64_t rows, uint64_t stride, uint64_t stack, int* n) {
    *n = width % 64 == 0 ? 2 : 1;
    const uint64_t wide = width / 64, whole = stack > 1 ? rows * stride : 16;
    const uint64_t d2[5] = {64, rows, wide, stack, 1}, s2[4] = {stride, 128, whole, 16};
    const uint64_t d1[5] = {width, rows, 1, stack, 1}, s1[4] = {stride, 16, whole, 16};
    const uint32_t b2[5] = {64, kTileK, 2, 1, 1}, b1[5] = {64, kTileK, 1, 1, 1};
    return *n == 2 ? make_tmap_16b_sw128(m, p, 5, d2, s2, b2, c.half) : make_tmap_16b_sw128(m, p, 5, d1, s1, b1, c.half);
  };
  if (mode == kGradW) {
    const uint32_t box[2] = {64, kTileK};
    rc = chunked(&ta, c.dz, N, P, (uint64_t)c.dzs * 2, 1, &a.a_chunks);
    if (!rc) rc = chunked(&tb, c.x, K, P, (uint64_t)c.xs * 2, 1, &a.b_chunks);
    if (!rc) rc = make_tmap_16b_sw128(&tb64, c.x, 2, dx, sx, box, c.half);
    tb32 = tb64;
    a.N = (int)K;
    a.M = (int)N;
    a.tiles_m = ceil_div(N, 256);
    a.tiles_n = ceil_div(K, 256);
  } else {
    const void* r = mode == kForward ? c.x : c.dz;
    const uint64_t *dr = mode == kForward ? dx : dd, *sr = mode == kForward ? sx : sd;
    const uint32_t box128[2] = {kTileK, 128}, box64[2] = {kTileK, 64}, box32[2] = {kTileK, 32};
    rc = make_tmap_16b_sw128(&tb, r, 2, dr, sr, box128, c.half);
    if (!rc) rc = make_tmap_16b_sw128(&tb64, r, 2, dr, sr, box64, c.half);
    if (!rc) rc = make_tmap_16b_sw128(&tb32, r, 2, dr, sr, box32, c.half);
    if (c.gated) {
      const uint32_t box[5] = {kTileK, 8, 2, 8, 1};
      if (!rc) rc = make_tmap_16b_sw128(&ta, c.w, 5, dg, sg, box, c.half);
    } else if (mode == kGradX) {
      if (!rc) rc = chunked(&ta, c.w, K, N, K * 2, E, &a.a_chunks);
    } else {
      const uint32_t box[5] = {kTileK, 128, 1, 1, 1};
      if (!rc) rc = make_tmap_16b_sw128(&ta, c.w, 5, dw, sw, box, c.half);
    }
    a.N = (int)(mode == kForward ? N : K);
    a.nk = ceil_div(mode == kForward ? K : N, kTileK);
    const int64_t features = mode == kGradX ? K : c.gated ? I : N;
    a.tiles_m = ceil_div(features, c.gated ? 128 : 256);
  }
  if (rc) return rc;
  return c.half ? launch_mode<__half>(mode, c.gated, ta, tb, tb64, tb32, a, stream)
                : launch_mode<__nv_bfloat16>(mode, c.gated, ta, tb, tb64, tb32, a, stream);
}

void launch_swiglu_bwd(const void* da, int64_t das, const void* z, int64_t zs, void* dz, int64_t P, int I,
                       const int32_t* offsets, int E, int half, int num_sms, cudaStream_t stream) {
  if (P == 0 || I == 0) return;
  const int nv = I / 8, threads = nv >= 256 ? 256 : (nv + 31) / 32 * 32;
  const dim3 grid((unsigned)P, P < 4 * num_sms ? (nv + threads - 1) / threads : 1);
  if (half)
    swiglu_bwd_kernel<__half><<<grid, threads, 0, stream>>>(static_cast<const __half*>(da), das,
                                                            static_cast<const __half*>(z), zs,
                                                            static_cast<__half*>(dz), P, I, offsets, E);
  else
    swiglu_bwd_kernel<__nv_bfloat16><<<grid, threads, 0, stream>>>(
        static_cast<const __nv_bfloat16*>(da), das, static_cast<const __nv_bfloat16*>(z), zs,
        static_cast<__nv_bfloat16*>(dz), P, I, offsets, E);
}
