// w8a8.hip — linears in 8-bit integers for gfx950: activations with a scale per token, weights with one per channel.
//
//   y[m, n] = (sum_k x[m, k] w[n, k]) ws[n] xs[m] (+ bias[n])
//   h[m, i] = silu(y[m, i]) y[m, I + i], unrounded y          (gate_up_silu; w has 2 I rows)
//
// The sums are exact in 32 bits (K < 2^17), and every route ends in the same three fp32 products: a row's outputs
// are the same bits whatever the other rows, tiles or K slices of the call.
// The MFMAs take the weights as their rows, so that a lane holds neighbouring outputs of one token.
//
// w8a8_rows, few rows: bound by the weights' bytes. 16 weight rows a tile, straight to registers; the waves of a
// workgroup take the columns in turn and add their sums in LDS.
// w8a8_gemm, above: tiles in LDS, loaded steps ahead (global_load_lds); K is split over workgroups where the tiles
// alone leave compute units idle, and w8a8_reduce adds the slices.
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

// What every route makes of a sum.
__device__ __forceinline__ float output(int32_t sum, float ws, float xs, bool has_bias, float bias) {
#pragma clang fp contract(off)
  const float y = static_cast<float>(sum) * ws * xs;
  return has_bias ? y + bias : y;
}
__device__ __forceinline__ float silu_up(float gate, float up) {
#pragma clang fp contract(off)
  return gate / (1.f + expf(-gate)) * up;
}

__device__ __forceinline__ i32x4 mfma16(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ i32x16 mfma32(u32x4 a, u32x4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// Up to 16 XT rows; a workgroup takes NT tiles of 16 weight rows (GATED: the gate's and the up rows of 16 outputs),
// its waves the stages of 256 columns in turn.
constexpr int kStage = 256;

template <typename T, int XT, int NT, bool GATED>
__global__ __launch_bounds__(1024) void w8a8_rows(Args a) {
  extern __shared__ __attribute__((aligned(16))) int32_t red[];  // [wave][tile][token][16]
  constexpr int kCols = GATED ? 16 : 16 * NT;                    // outputs of a workgroup
  static_assert(!GATED || NT == 2, "a gate tile and an up tile");
  const int W = blockDim.x >> 6, M = static_cast<int>(a.M);
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kCols;
  const int8_t* wrow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = min(n0 + (GATED ? 0 : 16 * t) + lr, a.N - 1);
    wrow[t] = a.w + ((GATED && t == 1 ? a.N : 0) + n) * a.ws;
  }
  const int8_t* xrow[XT];
#pragma unroll
  for (int i = 0; i < XT; ++i) xrow[i] = a.x + min(16 * i + lr, M - 1) * a.xs;
  i32x4 acc[XT][NT];
#pragma unroll
  for (int i = 0; i < XT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = i32x4{0, 0, 0, 0};
  struct Stage {
    u32x4 w[NT][4], x[XT][4];
  };
  const int stages = (a.K + kStage - 1) / kStage;
  auto load = [&](Stage& st, int s) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = min(s * kStage + 64 * j + 16 * lg, a.K - 16);  // past K: columns that count nothing
#pragma unroll
      for (int t = 0; t < NT; ++t) st.w[t][j] = sd::load16_stream(wrow[t] + k);
#pragma unroll
      for (int i = 0; i < XT; ++i) st.x[i][j] = sd::load16(xrow[i] + k);
    }
  };
  auto compute = [&](Stage& st, int s) {
    if (s * kStage + kStage > a.K) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (s * kStage + 64 * j + 16 * lg >= a.K) {
#pragma unroll
          for (int i = 0; i < XT; ++i) st.x[i][j] = u32x4{0, 0, 0, 0};
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < XT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = mfma16(st.w[t][j], st.x[i][j], acc[i][t]);
  };
  Stage one, two;
  int s = wave;
  if (s < stages) load(one, s);
  for (; s < stages; s += 2 * W) {
    if (s + W < stages) load(two, s + W);
    compute(one, s);
    if (s + W < stages) {
      if (s + 2 * W < stages) load(one, s + 2 * W);
      compute(two, s + W);
    }
  }
  // ---- the waves' sums meet: lane (lr, lg) holds outputs 4 lg .. 4 lg + 3 of token lr
#pragma unroll
  for (int i = 0; i < XT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
      *reinterpret_cast<i32x4*>(red + (((wave * NT + t) * XT + i) * 16 + lr) * 16 + 4 * lg) = acc[i][t];
  __syncthreads();
  constexpr int kWave = NT * XT * 256;
  for (int o = tid; o < kCols * M; o += W * 64) {
    const int m = o / kCols, c = o % kCols;
    const int64_t n = n0 + c;
    if (n >= a.N) continue;
    const float xs = a.x_scale[m];
    auto sum = [&](int t) {
      const int32_t* r = red + (t * XT * 16 + m) * 16 + (c & 15);
      int32_t v = 0;
      for (int u = 0; u < W; ++u) v += r[u * kWave];
      return v;
    };
    float y;
    if constexpr (GATED) {
      const bool bias = a.bias != nullptr;
      const float g = output(sum(0), scale_at(a, n), xs, bias, bias ? sd::from_bits<T>(a.bias[n]) : 0.f);
      const float u = output(sum(1), scale_at(a, a.N + n), xs, bias, bias ? sd::from_bits<T>(a.bias[a.N + n]) : 0.f);
      y = silu_up(g, u);
    } else {
      const bool bias = a.bias != nullptr;
      y = output(sum(c >> 4), scale_at(a, n), xs, bias, bias ? sd::from_bits<T>(a.bias[n]) : 0.f);
    }
    a.y[m * a.ys + n] = sd::to_bits<T>(y);
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

// WM x WN waves of MT x NT tiles of 32 tokens x 32 weight rows; S stages of 128 columns in LDS, loaded S - 1 steps
// ahead. 16-byte unit u of LDS row r stands at u ^ (r % 8): 8 rows' operand reads hit 8 different units. The rows of
// a weight tile are laid so that a lane's 16 sums of it are neighbours: MFMA row 8 a + 4 h + b is row 16 h + 4 a + b.
// GATED: the first half of a wave's weight tiles are the gate's, the second the up rows of the same outputs.
constexpr int kBlock = 128;

template <typename T, int WM, int WN, int MT, int NT, int S, bool GATED>
__global__ __launch_bounds__(WM * WN * 64) void w8a8_gemm(Args a) {
  constexpr int NW = WM * WN, BM = 32 * MT * WM, BN = 32 * NT * WN;
  constexpr int BO = GATED ? BN / 2 : BN;  // outputs
  constexpr int CX = BM / 8 / NW, CW = BN / 8 / NW;  // 1 KB loads (8 rows) of a wave and step
  constexpr int kX = BM * kBlock, kBytes = (BM + BN) * kBlock;
  constexpr int kPitch = 2 * BO + 16;  // of the output tile
  constexpr int kTile = S * kBytes > BM * kPitch ? S * kBytes : BM * kPitch;
  static_assert(CX * NW * 8 == BM && CW * NW * 8 == BN, "whole 1 KB loads");
  static_assert(!GATED || NT % 2 == 0, "as many gate tiles as up tiles");
  __shared__ __attribute__((aligned(1024))) uint8_t sm[kTile];
  __shared__ __attribute__((aligned(16))) float lws[BN], lxs[BM], lbias[BN];
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

  // LDS weight row -> output column of the tile (and whether it is an up row)
  auto col_of = [](int r) {
    const int q = r % 32, c = 16 * ((q >> 2) & 1) + 4 * (q >> 3) + (q & 3);
    if constexpr (GATED) return r / (32 * NT) * (16 * NT) + r / 32 % (NT / 2) * 32 + c;
    else return r - q + c;
  };
  auto is_up = [](int r) { return GATED && r / 32 % NT >= NT / 2; };

  // ---- loads: 8 rows an instruction, lane l unit (l % 8) ^ (l / 8) of row l / 8; rows past M or N repeat the last
  const int8_t* const xbase = a.x + m0 * a.xs;
  const int8_t* const wbase = a.w + n0 * a.ws;
  const int64_t up = GATED ? a.N * a.ws : 0;
  const uint32_t unit = 16 * ((lane & 7) ^ (lane >> 3));
  uint32_t xoff[CX], woff[CW];
#pragma unroll
  for (int i = 0; i < CX; ++i)
    xoff[i] = static_cast<uint32_t>(min(static_cast<int64_t>((wave * CX + i) * 8 + (lane >> 3)), a.M - 1 - m0)) *
              static_cast<uint32_t>(a.xs);
#pragma unroll
  for (int i = 0; i < CW; ++i)
    woff[i] = static_cast<uint32_t>(min(static_cast<int64_t>(col_of((wave * CW + i) * 8 + (lane >> 3))), a.N - 1 - n0)) *
              static_cast<uint32_t>(a.ws);
  const uint32_t sm_at = lds_addr(sm);
  const int blast = max(b1 - 1, b0);  // past the slice: its last block again, so that every step loads as much
  auto load = [&](int blk, int buf) {
    blk = min(blk, blast);
    const uint32_t at = sm_at + buf * kBytes;
    const uint32_t u = min(unit, static_cast<uint32_t>(a.K - 16 - blk * kBlock));  // past K: columns that count nothing
    const int8_t* xb = xbase + blk * kBlock;
    const int8_t* wb = wbase + blk * kBlock;
#pragma unroll
    for (int i = 0; i < CX; ++i) to_lds16(xb, xoff[i] + u, at + (wave * CX + i) * 1024);
#pragma unroll
    for (int i = 0; i < CW; ++i)
      to_lds16(is_up((wave * CW + i) * 8) ? wb + up : wb, woff[i] + u, at + kX + (wave * CW + i) * 1024);
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) load(b0 + i, i);
  // the scales, by output column in the order of a wave's tiles
  for (int r = tid; r < BN; r += NW * 64) {
    // r: wave wn, tile, neighbour
    const int t = r / 32 % NT;
    int64_t n;
    if constexpr (GATED) n = n0 + r / (32 * NT) * (16 * NT) + t % (NT / 2) * 32 + r % 32;
    else n = n0 + r;
    n = min(n, a.N - 1) + (GATED && t >= NT / 2 ? a.N : 0);
    lws[r] = scale_at(a, n);
    lbias[r] = a.bias ? sd::from_bits<T>(a.bias[n]) : 0.f;
  }
  for (int r = tid; r < BM; r += NW * 64) lxs[r] = a.x_scale[min(m0 + r, a.M - 1)];

  i32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][t][e] = 0;
  // operand reads: unit 2 j + lh of row lr of a tile
  uint32_t at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) at[j] = lr * kBlock + (((2 * j + lh) ^ (lr & 7)) * 16);
  constexpr int kLoads = CX + CW;
  int buf = 0;
  for (int blk = b0; blk < b1; ++blk) {
    // all but the newest S - 2 steps' loads have landed in every wave's view, and the slot of the step before is read
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * kLoads) : "memory");
    load(blk + S - 1, buf == 0 ? S - 1 : buf - 1);
    const uint8_t* const lx = sm + buf * kBytes + wm * (MT * 32 * kBlock);
    const uint8_t* const lw = sm + buf * kBytes + kX + wn * (NT * 32 * kBlock);
    const int left = a.K - blk * kBlock;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32x4 xf[MT], wf[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) xf[i] = sd::load16(lx + i * (32 * kBlock) + at[j]);
#pragma unroll
      for (int t = 0; t < NT; ++t) wf[t] = sd::load16(lw + t * (32 * kBlock) + at[j]);
      if (left < kBlock) {  // uniform
        const bool none = 32 * j + 16 * lh >= left;
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (none) wf[t] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = mfma32(wf[t], xf[i], acc[i][t]);
    }
    buf = buf + 1 == S ? 0 : buf + 1;
  }
  // the loads that ran ahead land before the stages' LDS is written again, or is another's
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const int rows = static_cast<int>(min(static_cast<int64_t>(BM), a.M - m0));
  const int cols = static_cast<int>(min(static_cast<int64_t>(BO), a.N - n0));
  if (a.slices > 1) {  // a lane's 16 sums of a tile
    const int64_t width = GATED ? 2 * a.N : a.N;
    int32_t* const part = a.part + slice * a.M * width;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int c0 = (GATED ? wn * (16 * NT) + t % (NT / 2) * 32 : (wn * NT + t) * 32) + 16 * lh;
      const int64_t n = n0 + c0 + (GATED && t >= NT / 2 ? a.N : 0);
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
  // ---- a lane's 16 neighbouring outputs of a token and tile, through LDS to whole lines
  __syncthreads();
  constexpr int kOut = GATED ? NT / 2 : NT;
  const bool has_bias = a.bias != nullptr;
#pragma unroll
  for (int t = 0; t < kOut; ++t) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = (wm * MT + i) * 32 + lr;
      const float xs = lxs[r];
      const int at_w = (wn * NT + t) * 32 + 16 * lh;
      uint32_t o[8];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        float v[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          v[q] = output(acc[i][t][e + q], lws[at_w + e + q], xs, has_bias, lbias[at_w + e + q]);
          if constexpr (GATED) {
            const int up_w = at_w + kOut * 32 + e + q;
            v[q] = silu_up(v[q], output(acc[i][t + kOut][e + q], lws[up_w], xs, has_bias, lbias[up_w]));
          }
        }
        o[e / 2] = sd::pack2<T>(v[0], v[1]);
      }
      uint8_t* const p = sm + r * kPitch + ((wn * kOut + t) * 32 + 16 * lh) * 2;
      sd::store16(p, u32x4{o[0], o[1], o[2], o[3]});
      sd::store16(p + 16, u32x4{o[4], o[5], o[6], o[7]});
    }
  }
  __syncthreads();
  uint16_t* const y0 = a.y + m0 * a.ys + n0;
  if (a.wide_y && cols % 8 == 0) {
    for (int i = tid; i < rows * (BO / 8); i += NW * 64) {
      const int r = i / (BO / 8), u = i % (BO / 8);
      if (u * 8 < cols) sd::store16(y0 + r * a.ys + u * 8, sd::load16(sm + r * kPitch + u * 16));
    }
  } else {
    for (int i = tid; i < rows * BO; i += NW * 64) {
      const int r = i / BO, c = i % BO;
      if (c < cols) y0[r * a.ys + c] = *reinterpret_cast<const uint16_t*>(sm + r * kPitch + c * 2);
    }
  }
}

// Sums of the K slices and the outputs.
template <typename T, bool GATED> __global__ __launch_bounds__(256) void w8a8_reduce(Args a) {
  const int64_t all = a.M * a.N, width = GATED ? 2 * a.N : a.N;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
    const int64_t m = i / a.N, n = i - m * a.N;
    const float xs = a.x_scale[m];
    const bool bias = a.bias != nullptr;
    auto value = [&](int64_t c) {
      int32_t s = 0;
      for (int v = 0; v < a.slices; ++v) s += a.part[(v * a.M + m) * width + c];
      return output(s, scale_at(a, c), xs, bias, bias ? sd::from_bits<T>(a.bias[c]) : 0.f);
    };
    const float y = value(n);
    a.y[m * a.ys + n] = sd::to_bits<T>(GATED ? silu_up(y, value(a.N + n)) : y);
  }
}

// What runs a shape: w8a8_rows<XT, NT> of W waves (XT > 0), or tiles of bm x bn weight rows and K slices.
struct Plan {
  int XT, NT, W;
  int bm, bn, slices;
};
Plan make_plan(int64_t M, int64_t N, int64_t K, bool gated) {
  Plan pl{};
  const int64_t cus = sd::device_cus();
  const int64_t wrows = gated ? 2 * N : N, stages = (K + kStage - 1) / kStage;
  if (M <= 32) {
    pl.XT = M <= 16 ? 1 : 2;
    pl.NT = gated ? 2 : 1;
    const int64_t groups = (wrows + 16 * pl.NT - 1) / (16 * pl.NT);
    pl.W = 4;
    while (pl.W < 16 && groups * pl.W < 8 * cus && pl.W < stages) pl.W *= 2;
    return pl;
  }
  const int64_t blocks = (K + kBlock - 1) / kBlock;
  auto tiles = [&](int bm, int bn) { return ((M + bm - 1) / bm) * ((wrows + bn - 1) / bn); };
  pl.bm = pl.bn = 256;
  if (tiles(256, 256) < 2 * cus) pl.bm = pl.bn = 128;
  if (tiles(128, 128) < cus) pl.bm = pl.bn = 64;
  pl.slices = 1;
  if (tiles(64, 64) < cus) {
    int64_t s = cus / tiles(64, 64);
    if (s > blocks / 4) s = blocks / 4;
    pl.slices = s < 1 ? 1 : s > 16 ? 16 : static_cast<int>(s);
  }
  return pl;
}

template <typename T, bool GATED> int launch(Args a, hipStream_t st) {
  const Plan pl = make_plan(a.M, a.N, a.K, GATED);
  if (pl.XT) {
    const int cols = GATED ? 16 : 16 * pl.NT;
    const dim3 grid(static_cast<unsigned>((a.N + cols - 1) / cols)), block(pl.W * 64);
    const size_t lds = static_cast<size_t>(pl.W) * pl.NT * pl.XT * 1024;
    constexpr int NT = GATED ? 2 : 1;
    if (pl.XT == 1) hipLaunchKernelGGL((w8a8_rows<T, 1, NT, GATED>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((w8a8_rows<T, 2, NT, GATED>), grid, block, lds, st, a);
    return sd::check_launch("w8a8");
  }
  const int bo = GATED ? pl.bn / 2 : pl.bn;
  a.slices = a.part ? pl.slices : 1;  // without its workspace: one slice
  a.tiles_m = static_cast<int32_t>((a.M + pl.bm - 1) / pl.bm);
  a.tiles_n = static_cast<int32_t>((a.N + bo - 1) / bo);
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.tiles_m) * a.tiles_n * a.slices)), block(256);
  if (pl.bm == 256) hipLaunchKernelGGL((w8a8_gemm<T, 2, 2, 4, 4, 2, GATED>), grid, block, 0, st, a);
  else if (pl.bm == 128) hipLaunchKernelGGL((w8a8_gemm<T, 2, 2, 2, 2, 3, GATED>), grid, block, 0, st, a);
  else if constexpr (GATED) hipLaunchKernelGGL((w8a8_gemm<T, 2, 1, 1, 2, 4, GATED>), grid, dim3(128), 0, st, a);
  else hipLaunchKernelGGL((w8a8_gemm<T, 2, 2, 1, 1, 4, GATED>), grid, block, 0, st, a);
  const int rc = sd::check_launch("w8a8");
  if (rc != SD_OK || a.slices == 1) return rc;
  int64_t wgs = (a.M * a.N + 255) / 256;
  if (wgs > 2048) wgs = 2048;
  hipLaunchKernelGGL((w8a8_reduce<T, GATED>), dim3(static_cast<unsigned>(wgs)), dim3(256), 0, st, a);
  return sd::check_launch("w8a8");
}

// (a launch takes fewer than 2^32 threads: tiles of 64 x 64 and 256 threads while they are few, of 256 x 256 then)
bool sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M <= (1ll << 24) && N <= (1ll << 21) && K < (1ll << 17) &&
         ((M + 255) / 256) * ((N + 127) / 128) < (1ll << 22);
}

size_t workspace(int64_t M, int64_t N, int64_t K, bool gated) {
  if (M <= 0 || N <= 0 || K <= 0 || !sizes_ok(M, N, K)) return 0;
  const Plan pl = make_plan(M, N, K, gated);
  return pl.slices > 1 ? static_cast<size_t>(pl.slices) * M * N * (gated ? 2 : 1) * sizeof(int32_t) : 0;
}

// Bytes of a matrix; ends at the address space's end where strides lead past it.
sd::Span span(const void* p, int64_t rows, int64_t stride_bytes, int64_t width_bytes) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  const unsigned __int128 hi = static_cast<unsigned __int128>(rows - 1) * stride_bytes + width_bytes + lo;
  return sd::Span{lo, hi > UINTPTR_MAX ? UINTPTR_MAX : static_cast<uintptr_t>(hi)};
}

int run(const char* what, bool gated, Args a, int32_t dtype, void* workspace_p, size_t workspace_bytes, void* stream) {
  sd::clear_error();
  const int64_t M = a.M, N = a.N, wrows = gated ? 2 * N : N;
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
  if (!sizes_ok(M, N, a.K) || (M > 1 && a.xs > (1ll << 23)) || (wrows > 1 && a.ws > (1ll << 23))) {
    sd::set_error("%s: M=%lld N=%lld K=%d (strides %lld, %lld) too large", what, (long long)M, (long long)N, a.K,
                  (long long)a.xs, (long long)a.ws);
    return SD_ERR_UNSUPPORTED;
  }
  if (M == 0) return SD_OK;
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
  const sd::Span y = span(a.y, M, 2 * a.ys, 2 * N);
  if (span(a.x, M, a.xs, a.K).overlaps(y) || span(a.x_scale, M, 4, 4).overlaps(y) ||
      span(a.w, wrows, a.ws, a.K).overlaps(y)) {
    sd::set_error("%s: y shares memory with an input", what);
    return SD_ERR_VALUE;
  }
  a.wide_y = sd::aligned16(a.y) && a.ys % 8 == 0;
  const size_t need = workspace(M, N, a.K, gated);
  a.part = need && workspace_p && workspace_bytes >= need ? static_cast<int32_t*>(workspace_p) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (gated) return dtype == SD_BF16 ? launch<__bf16, true>(a, st) : launch<_Float16, true>(a, st);
  return dtype == SD_BF16 ? launch<__bf16, false>(a, st) : launch<_Float16, false>(a, st);
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
  return workspace(M, N, K, gated != 0);
}

extern "C" int64_t sd_w8a8_plan(int64_t M, int64_t N, int64_t K, int32_t gated) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 16 != 0 || !sizes_ok(M, N, K)) return 0;
  const Plan pl = make_plan(M, N, K, gated != 0);
  if (pl.XT) return pl.W | 16 * pl.NT << 8;
  return pl.slices | pl.bn << 8 | static_cast<int64_t>(pl.bm) << 20;
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
