// w8a8.hip — linears in 8-bit integers for gfx950: activations with a scale per token, weights with one per channel.
//
//   y[m, n] = (sum_k x[m, k] w[n, k]) ws[n] xs[m] (+ bias[n])
//   h[m, i] = silu(y[m, i]) y[m, I + i], unrounded y          (gate_up_silu; w has 2 I rows)
//
// The sums are exact in 32 bits (K < 2^17), and every route ends in the same fp32 steps: a row's outputs
// are the same bits whatever the other rows, tiles or K slices of the call.
// The MFMAs take the weights as their rows, so that a lane holds neighbouring outputs of one token.
//
// w8a8_rows, few rows: bound by the weights' bytes. 16 weight rows a workgroup, straight to registers.
// w8a8_gemm, above: tiles in LDS, loaded steps ahead (global_load_lds); K is split over workgroups where the tiles
// alone leave compute units idle, and w8a8_reduce adds the slices.
#include <type_traits>

#include "sd_common.h"

namespace {

using sd::u32x4;
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

struct Args {
  const int8_t* x;
  int64_t xs;
  const float* x_scale;
  const int8_t* w;
  int64_t ws;
  const void* scale;
  int32_t scale_dtype;
  const uint16_t* bias;
  uint16_t* y;
  int64_t ys;
  int64_t M, N;  // N: outputs (gated: half of the weight rows)
  int32_t K;
  int32_t* part;  // K slices: [slice][M][weight rows]
  int32_t tiles_m, tiles_n, slices;
  int32_t wide_y;  // 16-byte stores of y are aligned
};

__device__ __forceinline__ float scale_at(const Args& a, int64_t n) {
  if (a.scale_dtype == SD_F32) return static_cast<const float*>(a.scale)[n];
  const uint16_t b = static_cast<const uint16_t*>(a.scale)[n];
  return a.scale_dtype == SD_F16 ? sd::from_bits<_Float16>(b) : sd::from_bits<__bf16>(b);
}

// What every route makes of a sum: sum ws, rounded, then its product with xs and the bias (0 without one) in one step.
__device__ __forceinline__ float output(int32_t sum, float ws, float xs, float bias) {
  return __builtin_fmaf(static_cast<float>(sum) * ws, xs, bias);
}
// silu(gate) up on the transcendental unit: the exponent's rounding moves the exponential by |gate| 2^-24, v_exp_f32 and
// v_rcp_f32 by one unit each, far below the output's half step. Below gate = -87, where silu(gate) is less than 2^-119, 0.
// (With expf and a division the epilogue of a 256 x 256 tile took 9 us, a third of its time.)
__device__ __forceinline__ float silu_up(float gate, float up) {
#pragma clang fp contract(off)
  const float e = __builtin_amdgcn_exp2f(gate * -1.442695041f);
  return gate * __builtin_amdgcn_rcpf(1.f + e) * up;
}

__device__ __forceinline__ i32x4 mfma16(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ i32x16 mfma32(u32x4 a, u32x4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// Lanes r < 8 of 16 hold units u of row r and of row r + 8, lanes r >= 8 units u + 4 of row r - 8 and of row r: after the
// exchange each lane holds units u and u + 4 of its own row.
__device__ __forceinline__ void own_units(u32x4 (&v)[2]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int a = static_cast<int>(v[0][e]), b = static_cast<int>(v[1][e]);
    v[0][e] = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(a, b, 0x128, 0xF, 0xC, false));  // row_ror:8
    v[1][e] = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(b, a, 0x128, 0xF, 0x3, false));
  }
}

// Up to 16 XT rows. A workgroup takes 16 weight rows (GATED: the gate's and the up rows of 8 outputs), its waves the
// stages of 128 columns in turn, loaded straight to registers two stages ahead. A load takes whole lines, of 8 rows, and
// the lanes exchange halves (of 16 rows by 64 bytes: weights from HBM, 16 x 2560 x 9728 11.9 us and 13.1 so, 1 x 19456 x
// 2560 11.1 and 11.9; from the caches 1% to 3% the other way, 1 x 4096 x 1024 3.10 and 3.03). The activations come from
// the caches, as many bytes a lane as of weights, which is what bounds it for more rows or many weight rows: 16 x 19456
// x 2560 takes 14.3 us here, 11.4 in tiles, 1 x 19456 x 2560 10.4 and 11.0. Registers decide how many loads a compute
// unit has in flight: stages of 256 columns took 10.9 us there, three of them ahead 10.6, two tiles a wave 13.9;
// nontemporal loads of the weights 13.5. 12 or 16 waves: within 3% of 8.
constexpr int kStage = 128;

template <typename T, int XT, bool GATED>
__global__ __launch_bounds__(512) void w8a8_rows(Args a) {
  extern __shared__ __attribute__((aligned(16))) int32_t red[];  // [wave][token][16]
  constexpr int kCols = GATED ? 8 : 16;                          // outputs of a workgroup
  constexpr int kUnits = kStage / 64;
  const int W = blockDim.x >> 6, M = static_cast<int>(a.M);
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kCols;
  const int unit = 16 * (lg + 4 * (lr >> 3));
  const int8_t *wrow[2], *xrow[XT][2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t n = min(n0 + (GATED ? lr & 7 : 8 * j + (lr & 7)), a.N - 1) + (GATED && j ? a.N : 0);
    wrow[j] = a.w + n * a.ws + unit;
#pragma unroll
    for (int i = 0; i < XT; ++i) xrow[i][j] = a.x + min(16 * i + 8 * j + (lr & 7), M - 1) * a.xs + unit;
  }
  i32x4 acc[XT];
#pragma unroll
  for (int i = 0; i < XT; ++i) acc[i] = i32x4{0, 0, 0, 0};
  struct Stage {
    u32x4 w[kUnits], x[XT][kUnits];
  };
  const int stages = (a.K + kStage - 1) / kStage;
  auto load = [&](Stage& st, int s) {
    const int k = min(s * kStage, a.K - 16 - unit);  // past K: columns that count nothing
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      st.w[j] = sd::load16(wrow[j] + k);
#pragma unroll
      for (int i = 0; i < XT; ++i) st.x[i][j] = sd::load16(xrow[i][j] + k);
    }
  };
  auto compute = [&](Stage& st, int s) {
    own_units(st.w);
#pragma unroll
    for (int i = 0; i < XT; ++i) own_units(st.x[i]);
    if (s * kStage + kStage > a.K) {  // uniform
#pragma unroll
      for (int j = 0; j < kUnits; ++j)
        if (s * kStage + 64 * j + 16 * lg >= a.K) st.w[j] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j)
#pragma unroll
      for (int i = 0; i < XT; ++i) acc[i] = mfma16(st.w[j], st.x[i][j], acc[i]);
  };
  Stage one, two;
  int s = wave;
  if (s < stages) load(one, s);
  if (s + W < stages) load(two, s + W);
  for (; s < stages; s += 2 * W) {
    compute(one, s);
    if (s + 2 * W < stages) load(one, s + 2 * W);
    if (s + W < stages) {
      compute(two, s + W);
      if (s + 3 * W < stages) load(two, s + 3 * W);
    }
  }
  // ---- the waves' sums meet: lane (lr, lg) holds weight rows 4 lg .. 4 lg + 3 of token lr
#pragma unroll
  for (int i = 0; i < XT; ++i)
    *reinterpret_cast<i32x4*>(red + ((wave * XT + i) * 16 + lr) * 16 + 4 * lg) = acc[i];
  __syncthreads();
  const bool bias = a.bias != nullptr;
  for (int o = tid; o < kCols * M; o += W * 64) {
    const int m = o / kCols, c = o % kCols;
    const int64_t out = n0 + c;
    if (out >= a.N) continue;
    const float xs = a.x_scale[m];
    auto value = [&](int row, int64_t at) {
      int32_t v = 0;
      for (int u = 0; u < W; ++u) v += red[(u * XT * 16 + m) * 16 + row];
      return output(v, scale_at(a, at), xs, bias ? sd::from_bits<T>(a.bias[at]) : 0.f);
    };
    const float y = value(c, out);
    a.y[m * a.ys + out] = sd::to_bits<T>(GATED ? silu_up(y, value(8 + c, a.N + out)) : y);
  }
}

__device__ __forceinline__ void to_lds16(const void* base, uint32_t off, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               ::"s"(l), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_addr(const void* l) {
  return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)l)));
}

// WM x WN waves of MT x NT tiles of 32 tokens x 32 weight rows; S stages of 128 columns in LDS, loaded S steps ahead.
// A step is four MFMA depths of 32 columns, whose operands are read two or three depths ahead, since a small wave's
// MFMAs of one depth (64 cycles for two tiles) take less time than its reads. Within a step the workgroup meets: all
// have read this stage, whose place takes the stage S steps on, and the next stage has landed and is read from here
// on, so that no MFMA waits for the reads after a barrier. With three stages or more it meets after the first depth,
// three depths ahead (777 x 2560 x 9728 in tiles of 128 x 128 33.3 us, 38.1 with operands one depth ahead, 40.3 when it
// meets after the second); with two after the second, which leaves the one stage in flight more time (1300 x 8192 x
// 8192 in tiles of 256 x 256 87.9 us, 92.5 after the first). Tried at 777 x 2560 x 9728 in 128 x 128 and no better: the
// freed stage loaded a step later without a wait for this step's reads (36.2), K split between two groups of waves for a
// third fewer reads (36.2), four waves of 64 x 64 each (33.3).
// What bounds long K: of those 33.3 us the loads and meetings alone take 32, the MFMAs and meetings alone 26, the reads
// and meetings alone 25. In loads alone a compute unit gets 32 KB in 0.23 us where its XCD's L2 holds them and in 0.34 to
// 0.38 where it does not, with 64 KB in flight or 128 (six stages of 96 x 96, eight of 64 x 64 are no faster than three
// and four). Here three quarters hit the L2 and 24 KB still take 0.39 us in tiles of 96 x 96; what the hits wait for is
// open. A wave that reads the lines ahead into the L2 costs more than it gives (a quarter of them: 37 us by vector loads,
// 100 by scalar ones). So tiles are chosen to give each compute unit the same share.
// LDS: 16-byte unit u of a row stands at u ^ turn, so that 16 rows' operand reads hit 16 different places of 256 bytes
// (64 banks). MFMA row 8 a + 4 h + b reads weight row 16 h + 4 a + b of its tile: a lane (half h of the wave) then holds
// sums of 16 neighbouring rows. GATED: rows 0 .. 15 of a tile are the gate's of 16 outputs, 16 .. 31 the up rows.
constexpr int kBlock = 128;

template <typename T, int WM, int WN, int MT, int NT, int S, bool GATED>
__global__ __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu((WM * WN + 3) / 4))) void w8a8_gemm(Args a) {
  constexpr int NW = WM * WN, BM = 32 * MT * WM, BN = 32 * NT * WN;
  constexpr int BO = GATED ? BN / 2 : BN;            // outputs
  constexpr int CX = BM / 8 / NW, CW = BN / 8 / NW;  // 1 KB loads (8 rows) of a wave and step
  constexpr int kX = BM * kBlock, kBytes = (BM + BN) * kBlock;
  constexpr int kPitch = 2 * BO + 16;  // of the output tile
  constexpr int kTile = S * kBytes > BM * kPitch ? S * kBytes : BM * kPitch;
  constexpr int kLoads = CX + CW, kDepths = kBlock / 32;
  static_assert(CX * NW * 8 == BM && CW * NW * 8 == BN, "whole 1 KB loads");
  static_assert(S <= 4, "what meet_at counts");
  __shared__ __attribute__((aligned(1024))) uint8_t sm[kTile];
  __shared__ __attribute__((aligned(16))) float lws[BN], lbias[BN], lxs[BM];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, lh = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;

  // Workgroup -> (slice, tile): every eighth workgroup shares an XCD (one L2), so each XCD takes a
  // contiguous run: 8 activation tiles by all weight tiles, then the next 8.
  const int items = a.tiles_m * a.tiles_n * a.slices;
  int id = blockIdx.x;
  {
    const int per = items / 8, rem = items % 8, xcd = id % 8;
    id = xcd * per + min(xcd, rem) + id / 8;
  }
  const int band = 8 * a.tiles_n * a.slices, band_i = id / band, in_band = id - band_i * band;
  const int brows = min(8, a.tiles_m - 8 * band_i);
  const int m_tile = 8 * band_i + in_band % brows, rest = in_band / brows;
  const int slice = rest % a.slices, n_tile = rest / a.slices;
  const int64_t m0 = static_cast<int64_t>(m_tile) * BM, n0 = static_cast<int64_t>(n_tile) * BO;
  const int blocks = (a.K + kBlock - 1) / kBlock;
  const int b0 = static_cast<int>(static_cast<int64_t>(slice) * blocks / a.slices);
  const int b1 = static_cast<int>(static_cast<int64_t>(slice + 1) * blocks / a.slices);

  auto x_turn = [](int r) { return (r >> 1) & 7; };
  auto w_turn = [](int r) { return ((r >> 1) & 3) | ((r >> 4) & 1) << 2; };
  auto column = [](int r) { return GATED ? (r >> 5) * 16 + (r & 15) : r; };  // of the tile's weight row r
  auto is_up = [](int r) { return GATED && (r & 16) != 0; };

  // ---- loads: 8 rows an instruction, lane l 16 bytes of row l / 8; rows past M or N repeat the last
  const int8_t* const xbase = a.x + m0 * a.xs;
  const int8_t* const wbase = a.w + n0 * a.ws;
  const int64_t up = GATED ? a.N * a.ws : 0;
  auto x_unit = [&](int i) { return 16u * ((lane & 7) ^ x_turn((wave * CX + i) * 8 + (lane >> 3))); };
  auto w_unit = [&](int i) { return 16u * ((lane & 7) ^ w_turn((wave * CW + i) * 8 + (lane >> 3))); };
  uint32_t xoff[CX], woff[CW];
#pragma unroll
  for (int i = 0; i < CX; ++i) {
    const int r = (wave * CX + i) * 8 + (lane >> 3);
    xoff[i] = static_cast<uint32_t>(min(static_cast<int64_t>(r), a.M - 1 - m0)) * static_cast<uint32_t>(a.xs) + x_unit(i);
  }
#pragma unroll
  for (int i = 0; i < CW; ++i) {
    const int r = (wave * CW + i) * 8 + (lane >> 3);
    woff[i] = static_cast<uint32_t>(min(static_cast<int64_t>(column(r)), a.N - 1 - n0)) * static_cast<uint32_t>(a.ws) +
              w_unit(i);
  }
  const uint32_t sm_at = lds_addr(sm);
  // The wave's loads [from, to) of a stage; `whole`: none of its columns lies past K (otherwise the last unit of a row
  // again, columns that count nothing).
  auto load = [&](int blk, int buf, int from, int to, auto whole) {
    const uint32_t at = sm_at + buf * kBytes;
    const uint32_t last = static_cast<uint32_t>(a.K - 16 - blk * kBlock);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if (i < from || i >= to) continue;
      if (i < CX) {
        uint32_t off = xoff[i];
        if constexpr (!decltype(whole)::value) off += min(x_unit(i), last) - x_unit(i);
        to_lds16(xbase + blk * kBlock, off, at + (wave * CX + i) * 1024);
      } else {
        const int c = wave * CW + i - CX;
        uint32_t off = woff[i - CX];
        if constexpr (!decltype(whole)::value) off += min(w_unit(i - CX), last) - w_unit(i - CX);
        to_lds16(wbase + (is_up(c * 8) ? up : 0) + blk * kBlock, off, at + kX + c * 1024);
      }
    }
  };
  // the scales and the bias, in the order of the tile's weight rows
  for (int r = tid; r < BN; r += NW * 64) {
    const int64_t n = min(n0 + column(r), a.N - 1) + (is_up(r) ? a.N : 0);
    lws[r] = scale_at(a, n);
    lbias[r] = a.bias ? sd::from_bits<T>(a.bias[n]) : 0.f;
  }
  for (int r = tid; r < BM; r += NW * 64) lxs[r] = a.x_scale[min(m0 + r, a.M - 1)];
#pragma unroll
  for (int i = 0; i < S; ++i)
    if (b0 + i < b1) load(b0 + i, i, 0, kLoads, std::false_type{});

  i32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][t][e] = 0;
  uint32_t x_at[kDepths], w_at[kDepths];  // operand reads: unit 2 j + lh of a row
  const int wr = 16 * ((lr >> 2) & 1) + 4 * (lr >> 3) + (lr & 3);
#pragma unroll
  for (int j = 0; j < kDepths; ++j) {
    x_at[j] = wm * (MT * 32 * kBlock) + lr * kBlock + (((2 * j + lh) ^ x_turn(lr)) * 16);
    w_at[j] = kX + wn * (NT * 32 * kBlock) + wr * kBlock + (((2 * j + lh) ^ w_turn(wr)) * 16);
  }
  u32x4 xf[kDepths][MT], wf[kDepths][NT];
  // The workgroup meets: all but the newest `stages` stages have landed in every wave's view, and every LDS read so far
  // is done.
  auto meet_at = [&](int stages) {
#define SD_MEET(n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((n) * kLoads) : "memory")
    if (stages <= 0) SD_MEET(0);
    else if (stages == 1) SD_MEET(1);
    else if (stages == 2) SD_MEET(2);
    else SD_MEET(3);
#undef SD_MEET
  };
  constexpr int kMeet = S == 2 ? 2 : 1;  // the depth before which the workgroup meets
  constexpr int kFirst = kDepths - kMeet;  // depths read before the loop
  auto read = [&](const uint8_t* stage, int j, int i) {  // the operands of depth j: token tile i, and its share of the others
    xf[j][i] = sd::load16(stage + x_at[j] + i * (32 * kBlock));
#pragma unroll
    for (int t = i * NT / MT; t < (i + 1) * NT / MT; ++t) wf[j][t] = sd::load16(stage + w_at[j] + t * (32 * kBlock));
  };
  meet_at(min(S, b1 - b0) - 1);
#pragma unroll
  for (int j = 0; j < kFirst; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) read(sm, j, i);
  int buf = 0;
  auto step = [&](int blk, auto middle) {  // middle: the stage S on is a whole one
    constexpr bool kMiddle = decltype(middle)::value;
    constexpr int kParts = MT * (kDepths - kMeet);  // the loads are spread over what follows the meeting
    const int next = buf + 1 == S ? 0 : buf + 1;
    const int left = a.K - blk * kBlock;
#pragma unroll
    for (int j = 0; j < kDepths; ++j) {
      if (j == kMeet) meet_at(kMiddle ? S - 2 : min(S - 2, b1 - 2 - blk));
      if (!kMiddle && left < kBlock) {  // the last columns
        const bool none = 32 * j + 16 * lh >= left;
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (none) wf[j][t] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        // the rest of this stage with its first depth, so that the reads are old when the workgroup meets
        if (j == 0) {
#pragma unroll
          for (int d = kFirst; d < kDepths; ++d) read(sm + buf * kBytes, d, i);
        } else if (j >= kMeet) {
          read(sm + next * kBytes, j - kMeet, i);
        }
        if (j >= kMeet && (kMiddle || blk + S < b1)) {
          const int q = (j - kMeet) * MT + i;
          load(blk + S, buf, q * kLoads / kParts, (q + 1) * kLoads / kParts, middle);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = mfma32(wf[j][t], xf[j][i], acc[i][t]);
        // one row of tiles after another: with the loads and reads all moved ahead of the MFMAs these wait for them
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    buf = next;
  };
  const int whole = min(b1, a.K / kBlock);
  int blk = b0;
  for (; blk + S < whole; ++blk) step(blk, std::true_type{});
  for (; blk < b1; ++blk) step(blk, std::false_type{});
  const int rows = static_cast<int>(min(static_cast<int64_t>(BM), a.M - m0));
  const int cols = static_cast<int>(min(static_cast<int64_t>(BO), a.N - n0));
  if (a.slices > 1) {  // a lane's 16 sums of a tile
    const int64_t width = GATED ? 2 * a.N : a.N;
    int32_t* const part = a.part + slice * a.M * width;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int c0 = GATED ? (wn * NT + t) * 16 : (wn * NT + t) * 32 + 16 * lh;
      const int64_t n = n0 + c0 + (GATED && lh ? a.N : 0);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int r = (wm * MT + i) * 32 + lr;
        if (r >= rows) continue;
        int32_t* const p = part + (m0 + r) * width + n;
        if (a.N % 4 == 0) {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (c0 + e < cols)
              *reinterpret_cast<i32x4*>(p + e) = i32x4{acc[i][t][e], acc[i][t][e + 1], acc[i][t][e + 2], acc[i][t][e + 3]};
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (c0 + e < cols) p[e] = acc[i][t][e];
        }
      }
    }
    return;
  }
  // ---- a lane's neighbouring outputs of a token and tile, through LDS to whole lines
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = (wm * MT + i) * 32 + lr;
      const float xs = lxs[r];
      if constexpr (GATED) {
        // the halves of the wave exchange 8 gates for 8 ups: each has both of 8 outputs
        const int at_w = (wn * NT + t) * 32 + 8 * lh;
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float v[2];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const auto z = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(acc[i][t][e + q]),
                                                            static_cast<uint32_t>(acc[i][t][e + q + 8]), false, false);
            const float g = output(static_cast<int32_t>(z[0]), lws[at_w + e + q], xs, lbias[at_w + e + q]);
            const float u = output(static_cast<int32_t>(z[1]), lws[at_w + 16 + e + q], xs, lbias[at_w + 16 + e + q]);
            v[q] = silu_up(g, u);
          }
          o[e / 2] = sd::pack2<T>(v[0], v[1]);
        }
        sd::store16(sm + r * kPitch + ((wn * NT + t) * 16 + 8 * lh) * 2, u32x4{o[0], o[1], o[2], o[3]});
      } else {
        const int at_w = (wn * NT + t) * 32 + 16 * lh;
        uint32_t o[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2)
          o[e / 2] = sd::pack2<T>(output(acc[i][t][e], lws[at_w + e], xs, lbias[at_w + e]),
                                  output(acc[i][t][e + 1], lws[at_w + e + 1], xs, lbias[at_w + e + 1]));
        uint8_t* const p = sm + r * kPitch + at_w * 2;
        sd::store16(p, u32x4{o[0], o[1], o[2], o[3]});
        sd::store16(p + 16, u32x4{o[4], o[5], o[6], o[7]});
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __syncthreads();
  uint16_t* const y0 = a.y + m0 * a.ys + n0;
  constexpr int kUnits = BO / 8;
  if (a.wide_y && cols % 8 == 0) {
    for (int i = tid; i < rows * kUnits; i += NW * 64) {
      const int r = i / kUnits, u = i % kUnits;
      if (u * 8 < cols) sd::store16(y0 + r * a.ys + u * 8, sd::load16(sm + r * kPitch + u * 16));
    }
  } else {
    // rows that start anywhere: the aligned 16 bytes of memory from a row's dwords in LDS, moved by half of one where
    // the row starts inside a dword; single outputs at the ends (2-byte stores of everything took 7 us a tile)
    for (int i = tid; i < rows * (kUnits + 1); i += NW * 64) {
      const int r = i / (kUnits + 1), u = i % (kUnits + 1);
      uint16_t* const row = y0 + r * a.ys;
      const int first = 8 * u - static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) >> 1);
      if (first >= 0 && first + 8 <= cols) {
        const uint32_t* const d = reinterpret_cast<const uint32_t*>(sm + r * kPitch) + (first >> 1);
        const uint32_t shift = (first & 1) * 16;
        u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_alignbit(d[e + 1], d[e], shift);
        sd::store16(row + first, v);
      } else {
        for (int e = max(first, 0); e < min(first + 8, cols); ++e)
          row[e] = *reinterpret_cast<const uint16_t*>(sm + r * kPitch + e * 2);
      }
    }
  }
}

// Sums of the K slices and the outputs; a thread takes V neighbouring outputs of a row (V divides N).
template <typename T, bool GATED, int V> __global__ __launch_bounds__(256) void w8a8_reduce(Args a) {
  const int64_t width = GATED ? 2 * a.N : a.N, all = a.M * a.N / V, step = a.M * width;
  const bool has_bias = a.bias != nullptr;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
    const int64_t m = i * V / a.N, n = i * V - m * a.N;
    const float xs = a.x_scale[m];
    float out[2][V];
#pragma unroll
    for (int h = 0; h < (GATED ? 2 : 1); ++h) {
      const int64_t c = n + (h ? a.N : 0);
      const int32_t* p = a.part + m * width + c;
      int32_t sum[V] = {};
      for (int s = 0; s < a.slices; ++s, p += step) {
        if constexpr (V == 4) {
          const i32x4 v = *reinterpret_cast<const i32x4*>(p);
#pragma unroll
          for (int e = 0; e < V; ++e) sum[e] += v[e];
        } else {
          sum[0] += *p;
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e)
        out[h][e] = output(sum[e], scale_at(a, c + e), xs, has_bias ? sd::from_bits<T>(a.bias[c + e]) : 0.f);
    }
    uint16_t* const y = a.y + m * a.ys + n;
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = sd::to_bits<T>(GATED ? silu_up(out[0][e], out[1][e]) : out[0][e]);
  }
}

// The tiles there are: 64 x 64 for few tiles of long rows (384 x 2560 x 9728 20.0 us, 23.3 in the others), 96 x 96 where
// it fills the device and 128 x 128 does not (777 x 2560 x 9728 30.8 and 33.3), 64 x 128 to 256 x 256 by size. Each with
// what it was measured to take (us): a round of workgroups `start` + steps x `alone` where each has a compute unit to
// itself, `full` a step where `per_cu` share it; and, since the whole device multiplies only as fast as its power allows,
// a workgroup `power_start` + steps x `power` of the device. The figures, fitted to times with weights in the caches, were
// then moved (by up to a fifth) to where the choices below lose least, with weights from HBM as well.
struct Tile {
  int bm, bn, per_cu;
  double start, alone, full, power_start, power;
};
constexpr Tile kTiles[] = {
    {256, 256, 1, 7.3, 0.996, 0.996, 0.0350, 0.00580},  {192, 256, 1, 4.9, 0.893, 0.893, 0.0337, 0.00430},
    {128, 256, 1, 5.0, 0.526, 0.526, 0.0230, 0.00320},  {192, 128, 1, 3.9, 0.419, 0.419, 0.0180, 0.00260},
    {128, 128, 1, 3.3, 0.318, 0.318, 0.0140, 0.00171},  {96, 96, 1, 3.7, 0.215, 0.215, 0.0110, 0.00120},
    {64, 128, 2, 2.21, 0.270, 0.539, 0.0060, 0.00096},  {64, 64, 2, 2.75, 0.140, 0.337, 0.0050, 0.00030},
    {32, 64, 4, 2.4, 0.149, 0.440, 0.0000, 0.00040},
};

// What runs a shape: w8a8_rows<XT> of W waves (slices 0), or a tile and K slices; with XT > 0 the former where there is
// no workspace for the slices.
struct Plan {
  int XT, W;
  int tile, slices;
};
// Up to 4 rows of up to so many columns need no workspace (what a caller may know without asking).
constexpr int64_t kLongSum = 16384;
Plan make_plan(int64_t M, int64_t N, int64_t K, bool gated) {
  Plan pl{};
  const int64_t cus = sd::device_cus();
  const int64_t wrows = gated ? 2 * N : N, groups = (wrows + 15) / 16, stages = (K + kStage - 1) / kStage;
  // Few rows: up to 4; more where weight rows are few, since every workgroup loads the activations anew (8 x 9000
  // x 4096 11.7 us there, 11.2 in tiles of 32 x 64, 12 rows 12.9 and 11.2; 16 x 6144 x 2560 6.7 and 6.8, 16 x 2560 x
  // 4096 6.0 and 8.3; 8 x 19456 x 2560 12.1 and 11.2), past 16 rows where the columns are few too (32 x 2560 x 4096 7.8
  // and 8.5, 32 x 4096 x 1024 3.9 and 5.0; 32 x 6144 x 2560 9.0 and 6.8, 32 x 2560 x 9728 16 and 10.7). Weights in the
  // caches; from HBM the limits would lie somewhat higher (8 x 9000 x 4096 12.8 and 13.5, 16 x 19456 x 2560 15.7 and 14.8).
  const bool few = M <= 4 || (M <= 8 && groups <= 3 * cus) || (M <= 16 && 2 * groups <= 3 * cus) ||
                   (M <= 32 && groups <= cus && stages <= 32);
  // Long sums of few weight rows: a workgroup walks its stages alone, which takes 0.52 to 0.82 us for 8 of them, while other
  // compute units have nothing; tiles in K slices use them all (16 x 512 x 65536 58.2 us there, 18.4 in tiles, 16 x 2560
  // x 28672 27.6 and 18.8, 1 x 1024 x 65536 37.6 and 19.3, 16 x 5120 x 9728 20.0 and 14.7). The figures of the tiles, of
  // more rows, are too good for so few by half; the last microseconds are the gated sums' addition. Asked only where it
  // may matter: 10 rounds of 8 stages are 11 us in either (16 x 2560 x 9728 11.1 and 10.3, weights from HBM 11.8 and 13.2).
  // Over 1178 shapes of up to 16 rows and 131056 columns the choice takes 0.9% more than the faster of the two on average,
  // 30% at worst (from HBM 0.4% and 16%); the kernel for few rows alone 17% and 265%.
  const int64_t rounds = (stages + 7) / 8 * ((groups + cus - 1) / cus);
  const bool either = few && 2 * groups <= 3 * cus && rounds > 10 && M <= 16 && (M > 4 || K > kLongSum);
  if (few) {
    pl.XT = M <= 16 ? 1 : 2;
    // 8 waves, 4 for very many workgroups (1 x 151936 x 1024 24.5 us, 27.1 with 8)
    pl.W = groups > 16 * cus ? 4 : 8;
    if (pl.W > stages) pl.W = static_cast<int>(stages);
    if (!either) return pl;
  }
  // The tile and slices of the least time by the figures above. Over 336 shapes of 17 to 4096 rows its choice takes 0.6%
  // more than the fastest of them on average, 13% at worst, with weights in the caches, 1.6% and 20% with weights from
  // HBM. Slices cost a launch and their sums' way to memory and back.
  const int64_t blocks = (K + kBlock - 1) / kBlock;
  double least = 1e30;
  for (int i = 0; i < static_cast<int>(sizeof(kTiles) / sizeof(kTiles[0])); ++i) {
    const Tile& t = kTiles[i];
    const int64_t tiles = ((M + t.bm - 1) / t.bm) * ((wrows + t.bn - 1) / t.bn), slots = t.per_cu * cus;
    const double more = t.per_cu > 1 ? (t.full - t.alone) / (t.per_cu - 1) : 0;
    for (int64_t s = 1; s == 1 || (s <= 16 && 4 * s <= blocks && tiles * s <= slots); ++s) {
      const double steps = static_cast<double>((blocks + s - 1) / s);
      auto round = [&](int64_t items) {  // (the larger of its two bounds, near where they meet somewhat more than both)
        const double l = t.start + steps * (t.alone + more * static_cast<double>((items + cus - 1) / cus - 1));
        const double w = static_cast<double>(items) * (t.power_start + steps * t.power) * 256 / static_cast<double>(cus);
        return __builtin_sqrt(__builtin_sqrt(l * l * l * l + w * w * w * w));
      };
      double cost = static_cast<double>(tiles * s / slots) * round(slots);
      if (tiles * s % slots) cost += round(tiles * s % slots);
      if (s > 1) cost += 3.34 + 0.14 * s + 1.45e-6 * s * static_cast<double>(M) * wrows;
      if (cost < least) {
        least = cost;
        pl.tile = i;
        pl.slices = static_cast<int>(s);
      }
    }
  }
  if (either && 2.9 + static_cast<double>(rounds) * (0.52 + 0.019 * static_cast<double>(M)) <=
                    1.45 * least + (gated ? 2 : 0))
    pl.slices = 0;
  return pl;
}

template <typename T, bool GATED> void launch_tiles(const Args& a, int tile, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.tiles_m) * a.tiles_n * a.slices));
#define SD_TILES(i, wm, wn, mt, nt, s)                                                                           \
  case i:                                                                                                        \
    static_assert(kTiles[i].bm == 32 * wm * mt && kTiles[i].bn == 32 * wn * nt, "the table's tile");             \
    hipLaunchKernelGGL((w8a8_gemm<T, wm, wn, mt, nt, s, GATED>), grid, dim3(64 * wm * wn), 0, st, a);            \
    break
  switch (tile) {
    SD_TILES(0, 2, 4, 4, 2, 2);
    SD_TILES(1, 2, 4, 3, 2, 2);
    SD_TILES(2, 2, 4, 2, 2, 3);
    SD_TILES(3, 2, 4, 3, 1, 3);
    SD_TILES(4, 2, 4, 2, 1, 4);
    SD_TILES(5, 1, 3, 3, 1, 4);
    SD_TILES(6, 2, 4, 1, 1, 3);
    SD_TILES(7, 2, 2, 1, 1, 4);
    SD_TILES(8, 1, 2, 1, 1, 3);
  }
#undef SD_TILES
}

template <typename T, bool GATED> int launch(Args a, const Plan& pl, hipStream_t st) {
  if (pl.slices == 0 || (pl.XT && pl.slices > 1 && !a.part)) {
    const int cols = GATED ? 8 : 16;
    const dim3 grid(static_cast<unsigned>((a.N + cols - 1) / cols)), block(pl.W * 64);
    const size_t lds = static_cast<size_t>(pl.W) * pl.XT * 1024;
    if (pl.XT == 1) hipLaunchKernelGGL((w8a8_rows<T, 1, GATED>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((w8a8_rows<T, 2, GATED>), grid, block, lds, st, a);
    return sd::check_launch("w8a8");
  }
  const Tile& t = kTiles[pl.tile];
  const int bo = GATED ? t.bn / 2 : t.bn;
  a.slices = a.part ? pl.slices : 1;  // without its workspace: one slice
  a.tiles_m = static_cast<int32_t>((a.M + t.bm - 1) / t.bm);
  a.tiles_n = static_cast<int32_t>((a.N + bo - 1) / bo);
  launch_tiles<T, GATED>(a, pl.tile, st);
  const int rc = sd::check_launch("w8a8");
  if (rc != SD_OK || a.slices == 1) return rc;
  const int64_t v = a.N % 4 == 0 ? 4 : 1;
  int64_t wgs = (a.M * a.N / v + 255) / 256;
  if (wgs > 2048) wgs = 2048;
  const dim3 grid(static_cast<unsigned>(wgs)), block(256);
  if (v == 4) hipLaunchKernelGGL((w8a8_reduce<T, GATED, 4>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((w8a8_reduce<T, GATED, 1>), grid, block, 0, st, a);
  return sd::check_launch("w8a8");
}

// (a launch takes fewer than 2^32 threads; no tile has more than 512 for 64 x 128 weight rows)
bool sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M <= (1ll << 24) && N <= (1ll << 21) && K < (1ll << 17) &&
         ((M + 63) / 64) * ((N + 63) / 64) < (1ll << 22);
}

size_t workspace(const Plan& pl, int64_t M, int64_t N, bool gated) {
  return pl.slices > 1 ? static_cast<size_t>(pl.slices) * M * N * (gated ? 2 : 1) * sizeof(int32_t) : 0;
}

int run(const char* what, bool gated, Args a, int32_t dtype, void* workspace_p, size_t workspace_bytes, void* stream) {
  sd::clear_error();
  const int64_t M = a.M, N = a.N;
  if (M < 0 || N <= 0 || a.K <= 0) {
    sd::set_error("%s: invalid sizes (M=%lld N=%lld K=%d)", what, (long long)M, (long long)N, a.K);
    return SD_ERR_VALUE;
  }
  if (a.K % 16 != 0) {
    sd::set_error("%s: K must be a multiple of 16, got %d", what, a.K);
    return SD_ERR_UNSUPPORTED;
  }
  if ((dtype != SD_BF16 && dtype != SD_F16) ||
      (a.scale_dtype != SD_BF16 && a.scale_dtype != SD_F16 && a.scale_dtype != SD_F32)) {
    sd::set_error("%s: dtype must be bf16 or f16, the weight scales' bf16, f16 or f32", what);
    return SD_ERR_UNSUPPORTED;
  }
  if (!sizes_ok(M, N, a.K) || (M > 1 && a.xs > (1ll << 23)) || ((gated || N > 1) && a.ws > (1ll << 23))) {
    sd::set_error("%s: M=%lld N=%lld K=%d (strides %lld, %lld) too large", what, (long long)M, (long long)N, a.K,
                  (long long)a.xs, (long long)a.ws);
    return SD_ERR_UNSUPPORTED;
  }
  if (M == 0) return SD_OK;
  const int64_t wrows = gated ? 2 * N : N;  // (N at most 2^21)
  if (!a.x || !a.x_scale || !a.w || !a.scale || !a.y) {
    sd::set_error("%s: null pointer argument", what);
    return SD_ERR_VALUE;
  }
  if (!sd::strides_ok({a.xs, a.ws, a.ys}) || a.xs < 0 || a.ws < 0 || a.ys < 0) {
    sd::set_error("%s: strides must lie in [0, 2^40]", what);
    return SD_ERR_VALUE;
  }
  if (!sd::aligned16(a.x) || !sd::aligned16(a.w) || (M > 1 && a.xs % 16 != 0) || (wrows > 1 && a.ws % 16 != 0)) {
    sd::set_error("%s: x and weight rows must be 16-byte aligned", what);
    return SD_ERR_UNSUPPORTED;
  }
  if (M > 1 && a.ys < N) {
    sd::set_error("%s: rows of y overlap (stride %lld, %lld columns)", what, (long long)a.ys, (long long)N);
    return SD_ERR_VALUE;
  }
  const sd::Span y = sd::span_rows(a.y, M, 2 * a.ys, 2 * N);
  const int64_t scale_bytes = a.scale_dtype == SD_F32 ? 4 : 2;
  if (sd::span_rows(a.x, M, a.xs, a.K).overlaps(y) || sd::span_rows(a.x_scale, M, 4, 4).overlaps(y) ||
      sd::span_rows(a.w, wrows, a.ws, a.K).overlaps(y) || sd::span_rows(a.scale, wrows, scale_bytes, scale_bytes).overlaps(y) ||
      (a.bias && sd::span_rows(a.bias, wrows, 2, 2).overlaps(y))) {
    sd::set_error("%s: y shares memory with another argument", what);
    return SD_ERR_VALUE;
  }
  a.wide_y = sd::aligned16(a.y) && a.ys % 8 == 0;
  const Plan pl = make_plan(M, N, a.K, gated);
  const size_t need = workspace(pl, M, N, gated);
  const bool held = need && workspace_p && workspace_bytes >= need && sd::aligned16(workspace_p);
  a.part = held ? static_cast<int32_t*>(workspace_p) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (gated) return dtype == SD_BF16 ? launch<__bf16, true>(a, pl, st) : launch<_Float16, true>(a, pl, st);
  return dtype == SD_BF16 ? launch<__bf16, false>(a, pl, st) : launch<_Float16, false>(a, pl, st);
}

Args args_of(const int8_t* x, int64_t xs, const float* x_scale, const int8_t* w, int64_t ws, const void* scale,
             int32_t scale_dtype, const void* bias, void* y, int64_t ys, int64_t M, int64_t N, int64_t K) {
  Args a{};
  a.x = x;
  a.xs = xs;
  a.x_scale = x_scale;
  a.w = w;
  a.ws = ws;
  a.scale = scale;
  a.scale_dtype = scale_dtype;
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.ys = ys;
  a.M = M;
  a.N = N;
  a.K = K < 0 ? -1 : K > 0x7ffffff0 ? 0x7ffffff0 : static_cast<int32_t>(K);
  return a;
}

}  // namespace

extern "C" size_t sd_w8a8_workspace_size(int64_t M, int64_t N, int64_t K, int32_t gated) {
  if (M <= 0 || N <= 0 || K <= 0 || !sizes_ok(M, N, K)) return 0;
  return workspace(make_plan(M, N, K, gated != 0), M, N, gated != 0);
}

extern "C" int64_t sd_w8a8_plan(int64_t M, int64_t N, int64_t K, int32_t gated) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 16 != 0 || !sizes_ok(M, N, K)) return 0;
  const Plan pl = make_plan(M, N, K, gated != 0);
  if (pl.slices == 0) return pl.W | 16 << 8;
  const Tile& t = kTiles[pl.tile];
  return pl.slices | t.bn << 8 | static_cast<int64_t>(t.bm) << 20 | static_cast<int64_t>(t.per_cu) << 32;
}

extern "C" int sd_w8a8_linear(const int8_t* x, int64_t x_stride_m, const float* x_scale, const int8_t* w,
                              int64_t w_stride_n, const void* scale, int32_t scale_dtype, const void* bias, void* y,
                              int64_t y_stride_m, int64_t M, int64_t N, int64_t K, int32_t dtype, void* workspace,
                              size_t workspace_bytes, void* stream) {
  return run("w8a8_linear", false,
             args_of(x, x_stride_m, x_scale, w, w_stride_n, scale, scale_dtype, bias, y, y_stride_m, M, N, K), dtype,
             workspace, workspace_bytes, stream);
}

extern "C" int sd_w8a8_gate_up_silu(const int8_t* x, int64_t x_stride_m, const float* x_scale, const int8_t* w,
                                    int64_t w_stride_n, const void* scale, int32_t scale_dtype, const void* bias,
                                    void* y, int64_t y_stride_m, int64_t M, int64_t N, int64_t K, int32_t dtype,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  return run("w8a8_gate_up_silu", true,
             args_of(x, x_stride_m, x_scale, w, w_stride_n, scale, scale_dtype, bias, y, y_stride_m, M, N, K), dtype,
             workspace, workspace_bytes, stream);
}
