// w4a16.hip — the linear with 4-bit weights, group scales and 16-bit activations for gfx950:
//
//   y[m, n] = sum_g scale[n, g] * sum_{k in g} x[m, k] (code[n, k] - 8)  (+ bias[n])
//
// code 0..15: byte j of a weight row holds columns 2 j (low half) and 2 j + 1; groups of G columns,
// G a multiple of 32 that divides K. The codes go to the matrix cores as 16 + code (int4.h); the
// accumulator of each group starts at -24 sum x over the group, so that it ends at the group's exact
// integer-weight sum, and is scaled in fp32. A lane's 16-byte load is 32 columns of one weight row;
// four permlane swaps turn the four lane groups' dwords so that one MFMA covers 32 neighbouring
// columns (one group at a time), and the order 0, 4, 1, 5, 2, 6, 3, 7 that unpack8 leaves is met
// by putting the activations in the same order.
//
// Up to 32 rows (w4a16_rows): bound by the weights' bytes, N K / 2. A workgroup takes tiles of 16 weight
// rows, its waves the columns in turn; their sums meet in LDS and are added in wave order.
// Activations read by every wave from the caches instead of from LDS kept the address units busy: 75 us
// at 1 x 151936 x 1024 against 23 (78 MB of weights: 3.4 TB/s).
// Above (w4a16_gemm): activations, weights and scales go straight to LDS for the workgroup's waves
// (global_load_lds, steps of 128 columns, two or three ahead); K is split over workgroups where the tiles
// alone leave compute units idle, and w4a16_reduce adds the slices in order. Bound by instruction issue:
// a step of 128 x 256 outputs takes 2.0 us, of which its MFMAs, a fifth of them for the -24 sum x, are 1.1
// (4096 x 19456 x 2560: 445 to 468 us from card to card, 872 to 916 TFLOP/s; 777 rows, in tiles of 192
// columns, 112 to 118 us).
#include <type_traits>

#include "int4.h"

namespace {

using sd::f32x4;
using sd::u32x4;

struct Args {
  const uint16_t* x;
  int64_t xs;
  const uint8_t* w;
  int64_t ws;  // bytes
  const void* scale;
  int32_t scale_f16, scale_f32;  // the scales' type (neither: bf16)
  int32_t groups;     // per weight row
  uint64_t inv32;     // ceil(2^32 / (columns per group / 32))
  const uint16_t* bias;
  uint16_t* y;
  int64_t ys;
  int64_t M, N;
  int32_t K;
  int32_t tiles;  // w4a16_rows: groups of weight tiles a workgroup
  float* part;    // K slices: [slices][M][N] sums
  int32_t tiles_m, tiles_n, slices;
  int32_t wide_y;  // 16-byte stores of y are aligned
};

// Group of column k: k / 32 is below 2^15 and a group below 2^20 columns, where the product with the
// rounded-up reciprocal is exact (the error stays below 2^15 * 2^15 / 2^32 of a group).
__device__ __forceinline__ int group_of(const Args& a, int k) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(k) >> 5) * a.inv32) >> 32);
}
// S32: 32-bit scales. Raw bits: the conversion waits for the load only where it is used.
template <bool S32> __device__ __forceinline__ uint32_t load_scale(const Args& a, int64_t at) {
  if constexpr (S32) return static_cast<const uint32_t*>(a.scale)[at];
  else return static_cast<const uint16_t*>(a.scale)[at];
}
template <typename ST> __device__ __forceinline__ float scale_of(uint32_t bits) {
  if constexpr (sizeof(ST) == 4) return __uint_as_float(bits);
  else return sd::from_bits<ST>(static_cast<uint16_t>(bits));
}
template <bool S32> __device__ __forceinline__ float scale_value(const Args& a, uint32_t bits) {
  if constexpr (S32) return __uint_as_float(bits);
  else return a.scale_f16 ? sd::from_bits<_Float16>(static_cast<uint16_t>(bits)) : __uint_as_float(bits << 16);
}

// Dword i of lane group lg becomes dword lg of lane group i.
__device__ __forceinline__ u32x4 turn(u32x4 d) {
  auto swap32 = [](uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  };
  auto swap16 = [](uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  };
  uint32_t a = d.x, b = d.y, c = d.z, e = d.w;
  swap32(a, c);
  swap32(b, e);
  swap16(a, b);
  swap16(c, e);
  return u32x4{a, b, c, e};
}

template <typename T> __device__ __forceinline__ uint32_t minus24() {  // two T of -24
  return __is_same(T, __bf16) ? 0xC1C0C1C0u : 0xCE00CE00u;
}

constexpr int kBlock = 128;  // columns of a step: 16 bytes of weights a lane

__device__ __forceinline__ void to_lds16(const void* base, uint32_t off, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               ::"s"(l), "v"(off), "s"(base) : "memory", "m0");
}
// 32 bits a lane: a 16-bit word lands zero-extended.
template <bool S32> __device__ __forceinline__ void scale_to_lds(const void* base, uint32_t off, uint32_t l) {
  if constexpr (S32)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 ::"s"(l), "v"(off), "s"(base) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, %2"
                 ::"s"(l), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_addr(const void* l) {
  return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)l)));
}

// The 8 codes of a dword as 8 T of 16 + u in their own order, which unpack8's order costs activations
// that go straight to LDS. A byte's two codes reach their halves' mantissas by one product: at bit
// p of each half the byte moved by p and by 16 + p - 4, which do not meet.
template <typename T> __device__ __forceinline__ u32x4 unpack8_in_order(uint32_t w, uint32_t base) {
  constexpr uint32_t kShift = __is_same(T, __bf16) ? 3 : 6;
  constexpr uint32_t kBoth = (1u << kShift) | (1u << (kShift + 12));
  u32x4 r;
#pragma unroll
  for (int b = 0; b < 4; ++b)
    r[b] = ((((w >> (8 * b)) & 0xffu) * kBoth) & sd::Magic<T>::kMask) | base;
  return r;
}

// Up to 2 XI rows. FOLD: MFMAs (32 columns each) between two scalings, 4, 2 or 1. A workgroup takes
// `tiles` groups of NT tiles of 16 weight rows, one after another; its waves take a group's stages of 256
// columns in turn. A stage's weights (whole 128-byte lines of each row) and activations go straight to
// the wave's own LDS, kAhead stages ahead and on into the next group, so that the waves meet only where
// their sums do. The scales of all rows lie in LDS in fp32. LDS decides how many workgroups a compute
// unit holds: with sums kept for 16 rows whatever their number, 1 x 19456 x 2560 in groups of 64 took
// 13.2 us against 9.8, as two held 54 KB each where three hold 47.
constexpr int kStage = 256;                   // columns of a stage
constexpr int kTileBytes = 16 * kStage / 2;   // of a tile's weights in a stage
constexpr int stage_bytes(int xi, int nt) { return nt * kTileBytes + xi * 1024; }
constexpr int rows_ahead(int xi, int nt) { return xi == 1 && nt == 1 ? 3 : 2; }

template <typename T, int FOLD, int XI, int NT>
__global__ __launch_bounds__(XI == 16 ? 512 : 1024) void w4a16_rows(Args a) {
  constexpr int NF = 4 / FOLD, MT = (XI + 7) / 8, R = 2 * XI;
  constexpr int kAhead = rows_ahead(XI, NT), kBytes = stage_bytes(XI, NT);
  extern __shared__ __attribute__((aligned(1024))) char sm[];
  const int W = blockDim.x >> 6;
  float* const red = reinterpret_cast<float*>(sm + W * kAhead * kBytes);  // [wave][tile][R][16]
  float* const lscale = red + W * NT * R * 16;                            // [row of a group][pitch]
  const int M = static_cast<int>(a.M), pitch = a.groups | 1;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int first = blockIdx.x * a.tiles;
  const int tiles = min(a.tiles, a.tiles_n - first);
  const int64_t n0 = static_cast<int64_t>(first) * (16 * NT);
  const int stages = (a.K + kStage - 1) / kStage;

  // ---- loads. Weights: 8 rows an instruction, lane l unit (l % 8) ^ (l / 8) of row l / 8. Activations: 2
  //      rows an instruction, lane l unit (l % 32) ^ (row % 16); rows past M repeat the last.
  const uint32_t ws = static_cast<uint32_t>(a.ws);
  const uint32_t unit = 16 * ((lane & 7) ^ (lane >> 3)), row0 = (lane >> 3) * ws;
  uint32_t x_off[XI];
#pragma unroll
  for (int i = 0; i < XI; ++i)
    x_off[i] = static_cast<uint32_t>(min(2 * i + (lane >> 5), M - 1)) * static_cast<uint32_t>(2 * a.xs);
  const char* const x0 = reinterpret_cast<const char*>(a.x);
  char* const mine = sm + wave * kAhead * kBytes;
  const uint32_t mine_at = lds_addr(mine);
  int load_tile = 0, load_stage = wave;
  auto load = [&](int slot) {  // past the last group: its last stage again, into a slot nobody reads
    const int t = min(load_tile, tiles - 1), s = min(load_stage, stages - 1);
    const int64_t n = n0 + static_cast<int64_t>(16 * NT) * t;
    const uint8_t* base = a.w + n * a.ws + s * (kStage / 2);
    const uint32_t most = static_cast<uint32_t>(min(a.N - 1 - n, static_cast<int64_t>(16 * NT - 1))) * ws;
    const uint32_t u = min(unit, static_cast<uint32_t>(a.K / 2 - 16 - s * (kStage / 2)));
    const uint32_t l = mine_at + slot * kBytes;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) to_lds16(base, min(row0 + 8 * i * ws, most) + u, l + 1024 * i);
    const uint32_t last = static_cast<uint32_t>(2 * a.K - 16 - s * (2 * kStage));
#pragma unroll
    for (int i = 0; i < XI; ++i)
      to_lds16(x0 + s * (2 * kStage), x_off[i] + min(16u * ((lane & 31) ^ ((2 * i + (lane >> 5)) & 15)), last),
               l + NT * kTileBytes + 1024 * i);
    load_stage += W;
    if (load_stage >= stages) {
      load_stage = wave;
      ++load_tile;
    }
  };
  if (wave < stages) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(i);
  }
  const int srows = static_cast<int>(min(static_cast<int64_t>(16 * NT) * tiles, a.N - n0));
  // 16 lanes take 16 neighbouring scales of a row, several such items at once
  const int parts = (a.groups + 15) / 16, items = srows * parts;
  auto copy_scales = [&](auto s32) {
    constexpr bool kS32 = decltype(s32)::value;
    constexpr int kOnce = 8;
    for (int i0 = 0; i0 < items; i0 += kOnce * W * 4) {
      uint32_t v[kOnce];
      int at[kOnce];
#pragma unroll
      for (int o = 0; o < kOnce; ++o) {
        at[o] = -1;
        if (o && i0 + o * W * 4 >= items) continue;  // uniform
        const int i = i0 + o * W * 4 + (tid >> 4), r = parts == 1 ? i : i / parts;
        const int g = (i - r * parts) * 16 + (tid & 15);
        const bool in = i < items && g < a.groups;
        at[o] = in ? r * pitch + g : -1;
        v[o] = load_scale<kS32>(a, n0 * a.groups + (in ? r * a.groups + g : 0));
      }
#pragma unroll
      for (int o = 0; o < kOnce; ++o)
        if (at[o] >= 0) lscale[at[o]] = scale_value<kS32>(a, v[o]);
    }
  };
  if (a.scale_f32) copy_scales(std::true_type{});
  else copy_scales(std::false_type{});
  __syncthreads();

  const uint32_t base = sd::code_base<T>();
  const u32x4 m24 = {minus24<T>(), minus24<T>(), minus24<T>(), minus24<T>()};
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint32_t w_at = lr * 128 + ((lg ^ (lr & 7)) * 16);  // unit lg of row lr; the next block's: ^ 64
  uint32_t x_row[MT];  // LDS row of this lane's operand row, and what its units are turned by
  uint32_t x_turn[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = min(16 * i + lr, 2 * XI - 1);
    x_row[i] = NT * kTileBytes + m * 512;
    x_turn[i] = m & 15;
  }
  auto compute = [&](const char* st, const float* scale, int k) {
#pragma unroll
    for (int c = 0; c < kStage / kBlock; ++c) {
      const int left = a.K - k - c * kBlock;  // columns of this block and after
      if (left <= 0) break;                   // uniform
      u32x4 w[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        w[t] = sd::load16(st + t * kTileBytes + (w_at ^ (64 * c)));
        // one group a block: any order of the columns will do, as long as the activations' is the same
        if constexpr (FOLD < 4) w[t] = turn(w[t]);
      }
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        if (FOLD < 4 && 32 * FOLD * f >= left) break;  // uniform
        const int g = group_of(a, k + c * kBlock + 32 * FOLD * f);
        u32x4 x[MT][FOLD];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < FOLD; ++j) {
            const uint32_t u = 16 * c + (FOLD == 4 ? 4 * lg + j : 4 * (f * FOLD + j) + lg);
            x[i][j] = sd::load16(st + x_row[i] + ((u ^ x_turn[i]) * 16));
          }
        f32x4 v[MT][NT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          f32x4 start = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < FOLD; ++j) start = sd::Elem<T>::mfma(x[i][j], m24, start);
#pragma unroll
          for (int t = 0; t < NT; ++t) v[i][t] = start;
        }
#pragma unroll
        for (int j = 0; j < FOLD; ++j)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const u32x4 wf = unpack8_in_order<T>(w[t][f * FOLD + j], base);
#pragma unroll
            for (int i = 0; i < MT; ++i) v[i][t] = sd::Elem<T>::mfma(x[i][j], wf, v[i][t]);
          }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float sv = scale[t * 16 * pitch + g];
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][t] += sv * v[i][t];
        }
      }
    }
  };

  int slot = 0;
  for (int t = 0; t < tiles; ++t) {
    // rows past N: scales of rows past the group's, never written (the buffer holds whole groups)
    const float* scale = lscale + (16 * NT * t + lr) * pitch;
    for (int s = wave; s < stages; s += W) {
      // the oldest stage has landed (loads issued after it only make this wait longer)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((2 * NT + XI) * (kAhead - 1)) : "memory");
      compute(mine + slot * kBytes, scale, s * kStage);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // its words are read
      load(slot);
      slot = slot + 1 == kAhead ? 0 : slot + 1;
    }
    // ---- the waves' sums meet in LDS
    float* mr = red + wave * (NT * R * 16);
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (16 * i + 4 * lg + e < R) mr[(u * R + 16 * i + 4 * lg + e) * 16 + lr] = acc[i][u][e];
          acc[i][u][e] = 0.f;
        }
    __syncthreads();
    for (int i = tid; i < 16 * NT * M; i += W * 64) {  // 16 NT neighbouring outputs of a row
      const int m = i / (16 * NT), u = i / 16 % NT, c = i % 16;
      const int64_t n = n0 + static_cast<int64_t>(16) * (NT * t + u) + c;
      if (n >= a.N) continue;
      const float* r = red + (u * R + m) * 16 + c;
      float s = 0.f;
      for (int v = 0; v < W; ++v) s += r[v * (NT * R * 16)];
      if (a.bias) s += sd::from_bits<T>(a.bias[n]);
      a.y[m * a.ys + n] = sd::to_bits<T>(s);
    }
    if (t + 1 < tiles) __syncthreads();
  }
  // the loads that ran ahead land before the workgroup's LDS is another's
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// WM x WN waves of MT x NT tiles of 16 x 16 outputs; S stages of activations, weights and scales in LDS,
// all of them loaded S - 1 steps ahead straight from memory. (Weights and scales loaded to registers
// instead: the compiler's waits for them were waits for the activations behind them as well, 559 us.)
// The MFMAs take the weights as their rows: a lane then holds neighbouring outputs of one row, and the
// tile leaves through LDS in whole lines (2-byte stores of the other order: 487 us; 8-byte ones 661).
// Where there are 8 waves, two share a SIMD: they take turns, one unpacks while the other multiplies
// (503 us without; these three at 4096 x 19456 x 2560, between the first form's 559 and 449 now).
template <typename T, typename ST, int FOLD, int WM, int WN, int MT, int NT, int S>
__global__ __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(2)))
void w4a16_gemm(Args a) {
  constexpr int NW = WM * WN, BM = 16 * MT * WM, BN = 16 * NT * WN, NF = 4 / FOLD;
  constexpr int kRow = 2 * kBlock;                // bytes of an activation row's step
  constexpr int CX = BM * kRow / 1024 / NW;       // 1 KB loads (4 rows) of a wave and step
  constexpr int CW = (WN * NT + NW - 1) / NW;     // 1 KB loads (a tile's 16 rows) of a wave and step
  constexpr int kX = BM * kRow, kW = CW * NW * 1024, kS = NF * 256, kBytes = kX + kW + NW * kS;
  static_assert(CX * NW * 1024 == kX, "whole 1 KB loads");
  static_assert(S * kBytes <= (160 << 10), "a compute unit's LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t sm[S * kBytes];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
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
  const int rows = min(8, a.tiles_m - 8 * band_i);
  const int m_tile = 8 * band_i + in_band % rows, rest = in_band / rows;
  const int slice = rest % a.slices, n_tile = rest / a.slices;
  const int64_t m0 = static_cast<int64_t>(m_tile) * BM, n0 = static_cast<int64_t>(n_tile) * BN;
  const int blocks = (a.K + kBlock - 1) / kBlock;
  const int b0 = static_cast<int>(static_cast<int64_t>(slice) * blocks / a.slices);
  const int b1 = static_cast<int>(static_cast<int64_t>(slice + 1) * blocks / a.slices);

  // ---- loads. Activations: 16-byte unit u of row r stands at unit u ^ (r % 16) of its LDS row, so that
  //      the 16 rows of an operand read hit 16 different units. Weights: a lane's unit as it reads it.
  //      With groups of whole blocks (FOLD == 4) no unit lies past K.
  const char* xbase = reinterpret_cast<const char*>(a.x + m0 * a.xs);
  uint32_t xoff[CX], woff[CW];
#pragma unroll
  for (int i = 0; i < CX; ++i) {
    const int r = (wave * CX + i) * 4 + lg;
    xoff[i] = static_cast<uint32_t>(min(static_cast<int64_t>(r), a.M - 1 - m0) * a.xs * 2);
    if constexpr (FOLD == 4) xoff[i] += 16 * (lr ^ (r & 15));
  }
  const uint8_t* const wbase = a.w + n0 * a.ws;
  const int64_t last_n = a.N - 1 - n0;
#pragma unroll
  for (int i = 0; i < CW; ++i) {
    const int q = wave * CW + i, t = q % NT;
    const int r = min(q / NT * (16 * NT) + 4 * NT * (lr >> 2) + 4 * t + (lr & 3), BN - 1);
    woff[i] = static_cast<uint32_t>(min(static_cast<int64_t>(r), last_n)) * static_cast<uint32_t>(a.ws);
    if constexpr (FOLD == 4) woff[i] += 16 * lg;
  }
  constexpr int kScale = sizeof(ST);
  const char* const sbase = static_cast<const char*>(a.scale) + n0 * a.groups * kScale;
  const uint32_t soff =
      static_cast<uint32_t>(min(static_cast<int64_t>(wn * NT * 16 + min(lane, NT * 16 - 1)), last_n)) * a.groups * kScale;
  const uint32_t sm_at = lds_addr(sm);
  const int blast = max(b1 - 1, b0);  // past the slice: its last block again, so that every step loads as much
  auto load = [&](int blk, int buf) {
    blk = min(blk, blast);
    const uint32_t at = sm_at + buf * kBytes;
    const char* xb = xbase + static_cast<int64_t>(blk) * kRow;
    const uint32_t last = 2 * (a.K - blk * kBlock) - 16;  // the last unit of a row, past it again
#pragma unroll
    for (int i = 0; i < CX; ++i) {
      uint32_t off = xoff[i];
      if constexpr (FOLD < 4) off += min(16u * (lr ^ (((wave * CX + i) * 4 + lg) & 15)), last);
      to_lds16(xb, off, at + (wave * CX + i) * 1024);
    }
    const uint8_t* wb = wbase + blk * (kBlock / 2);
#pragma unroll
    for (int i = 0; i < CW; ++i) {
      uint32_t off = woff[i];
      if constexpr (FOLD < 4) off += min(16u * lg, static_cast<uint32_t>(a.K / 2 - 16 - blk * (kBlock / 2)));
      to_lds16(wb, off, at + kX + (wave * CW + i) * 1024);
    }
#pragma unroll
    for (int f = 0; f < NF; ++f)
      scale_to_lds<kScale == 4>(sbase + group_of(a, min(blk * kBlock + 32 * FOLD * f, a.K - 32)) * kScale, soff,
                        at + kX + kW + wave * kS + f * 256);
  };

  const uint32_t base = sd::code_base<T>();
  const u32x4 m24 = {minus24<T>(), minus24<T>(), minus24<T>(), minus24<T>()};
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  uint32_t x_at[4];  // operand reads: unit 4 j + lg of row lr of a tile
#pragma unroll
  for (int j = 0; j < 4; ++j) x_at[j] = (wm * MT * 16 + lr) * kRow + (((4 * j + lg) ^ lr) * 16);

  constexpr int kLoads = CX + CW + NF;  // vector memory instructions of a step
#pragma unroll
  for (int i = 0; i < S - 1; ++i) load(b0 + i, i);
  int buf = 0;
  constexpr bool kTurns = NW == 8;  // waves w and w + 4 are on one SIMD
  const bool second = kTurns && wave >= 4;
  // All but the newest S - 2 steps' loads have landed in every wave's view, and every LDS read so far is
  // done: the slot of the step before is free. The second waves run half a step behind: while they
  // multiply step b the first unpack b + 1, so the first load b + S - 1 only after their middle meeting.
  auto meet = [&]() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * kLoads) : "memory");
  };
  if (second) meet();
  for (int blk = b0; blk < b1; ++blk) {
    meet();
    const uint8_t* const lx = sm + buf * kBytes;
    if (!kTurns || second) load(blk + S - 1, buf == 0 ? S - 1 : buf - 1);
    u32x4 wf[NT][4];
    f32x4 sv[NT][NF];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const u32x4 w = turn(sd::load16(lx + kX + (wn * NT + t) * 1024 + lane * 16));
#pragma unroll
      for (int i = 0; i < 4; ++i) wf[t][i] = unpack8_in_order<T>(w[i], base);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const u32x4 bits = sd::load16(lx + kX + kW + wave * kS + f * 256 + (4 * NT * lg + 4 * t) * 4);
        // past K the last columns again (never with whole blocks): they count nothing
        const bool none = f && blk * kBlock + 32 * FOLD * f >= a.K;
#pragma unroll
        for (int e = 0; e < 4; ++e) sv[t][f][e] = none ? 0.f : scale_of<ST>(bits[e]);
      }
    }
    if constexpr (kTurns) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(wf[t][i]));
#pragma unroll
        for (int f = 0; f < NF; ++f) asm volatile("" : "+v"(sv[t][f]));
      }
      __builtin_amdgcn_sched_barrier(0);
      meet();
      if (!second) load(blk + S - 1, buf == 0 ? S - 1 : buf - 1);
      __builtin_amdgcn_s_setprio(1);
    }
    u32x4 xs[2][4];  // operands of a tile and of the next
#pragma unroll
    for (int j = 0; j < 4; ++j) xs[0][j] = sd::load16(lx + x_at[j]);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      u32x4(&xf)[4] = xs[i & 1];
      if (i + 1 < MT) {
#pragma unroll
        for (int j = 0; j < 4; ++j) xs[(i + 1) & 1][j] = sd::load16(lx + x_at[j] + (i + 1) * 16 * kRow);
      }
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        f32x4 start = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < FOLD; ++j) start = sd::Elem<T>::mfma(m24, xf[f * FOLD + j], start);
        f32x4 d[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) d[t] = start;
#pragma unroll
        for (int j = 0; j < FOLD; ++j)
#pragma unroll
          for (int t = 0; t < NT; ++t)
            d[t] = sd::Elem<T>::mfma(wf[t][f * FOLD + j], xf[f * FOLD + j], d[t]);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] += sv[t][f] * d[t];
      }
      // one tile after another: with all tiles' operands hoisted the accumulators spill
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kTurns) __builtin_amdgcn_s_setprio(0);
    buf = buf + 1 == S ? 0 : buf + 1;
  }
  if (kTurns && !second) meet();
  // the loads that ran ahead land before the workgroup's LDS is another's
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  // ---- a lane's 4 NT neighbouring outputs of a row of every activation tile, through LDS to whole lines
  auto out = [&](auto one, auto* to, int64_t stride, bool wide) {
    using O = decltype(one);
    constexpr int kPitch = BN * sizeof(O) + 16, kUnit = 16 / sizeof(O), kUnits = BN / kUnit;
    static_assert(BM * kPitch <= S * kBytes, "the tile fits where the stages were");
    const int64_t n = n0 + wn * (16 * NT) + 4 * NT * lg;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      f32x4 bias = {0.f, 0.f, 0.f, 0.f};
      if (a.bias && a.slices == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          bias[e] = sd::from_bits<T>(a.bias[min(n + 4 * t + e, a.N - 1)]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        O* p = reinterpret_cast<O*>(sm + ((wm * MT + i) * 16 + lr) * kPitch) + wn * (16 * NT) + 4 * NT * lg + 4 * t;
        const f32x4 v = acc[i][t] + bias;
        if constexpr (sizeof(O) == 4) *reinterpret_cast<f32x4*>(p) = v;
        else {
          union { uint16_t h[4]; uint2 u; } o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o.h[e] = sd::to_bits<T>(v[e]);
          *reinterpret_cast<uint2*>(p) = o.u;
        }
      }
    }
    __syncthreads();
    const int rows = static_cast<int>(min(static_cast<int64_t>(BM), a.M - m0));
    const int cols = static_cast<int>(min(static_cast<int64_t>(BN), a.N - n0));
    O* const y0 = to + m0 * stride + n0;
    if (wide && cols % kUnit == 0) {
      for (int i = tid; i < rows * kUnits; i += NW * 64) {
        const int r = i / kUnits, u = i % kUnits;
        if (u * kUnit < cols) *reinterpret_cast<u32x4*>(y0 + r * stride + u * kUnit) = sd::load16(sm + r * kPitch + u * 16);
      }
    } else {
      for (int i = tid; i < rows * BN; i += NW * 64) {
        const int r = i / BN, c = i % BN;
        if (c < cols) y0[r * stride + c] = *reinterpret_cast<const O*>(sm + r * kPitch + c * sizeof(O));
      }
    }
  };
  if (a.slices > 1) out(0.f, a.part + slice * a.M * a.N, a.N, a.N % 4 == 0);
  else out(uint16_t{}, a.y, a.ys, a.wide_y != 0);
}

// Sum of the K slices, in slice order, bias, rounding.
template <typename T> __global__ __launch_bounds__(256) void w4a16_reduce(Args a) {
  const int64_t all = a.M * a.N;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
    const int64_t m = i / a.N, n = i - m * a.N;
    float s = 0.f;
    for (int v = 0; v < a.slices; ++v) s += a.part[v * all + i];
    if (a.bias) s += sd::from_bits<T>(a.bias[n]);
    a.y[m * a.ys + n] = sd::to_bits<T>(s);
  }
}

// What runs a shape: up to 32 rows w4a16_rows<XI, NT> of W waves and its groups a workgroup; above (and
// where a row has so many groups that a tile's scales leave LDS no room) tiles of bm x bn and K slices.
struct Plan {
  int XI, NT, W, tiles;  // XI == 0: w4a16_gemm
  size_t lds;
  int bm, bn, slices;
};
Plan make_plan(int64_t M, int64_t N, int64_t K, int64_t group) {
  Plan pl{};
  const int64_t cus = sd::device_cus(), blocks = (K + kBlock - 1) / kBlock;
  const int fold = group % 128 == 0 ? 4 : group % 64 == 0 ? 2 : 1;
  const int64_t all = (N + 15) / 16, stages = (K + kStage - 1) / kStage;  // weight tiles, their stages
  pl.XI = M <= 2 ? 1 : M <= 8 ? 4 : M <= 16 ? 8 : 16;
  // Every wave reads its own share of x: past 8 rows that is more than the weights. Tiles of w4a16_gemm
  // share it: 16 x 19456 x 2560 16 us there and 19 here, 16 x 2560 x 9728 34 and 10; past 16 rows (32 x
  // 2560 x 9728 14 and 20) only layers of few tiles and stages stay (32 x 4096 x 1024 7.5 and 5.5).
  if (M <= 8 || (M <= 16 && all < 4 * cus) || (M <= 32 && all <= cus && stages <= 8)) {
    // two tiles share what a wave reads of x where there are workgroups enough
    pl.NT = all < 4 * cus ? 1 : 2;
    const int64_t groups = (all + pl.NT - 1) / pl.NT;
    auto bytes = [&](int64_t tiles, int W) {
      return static_cast<size_t>(W) * (rows_ahead(pl.XI, pl.NT) * stage_bytes(pl.XI, pl.NT) +
                                       pl.NT * pl.XI * 128) +
             static_cast<size_t>(tiles) * pl.NT * 16 * ((K / group) | 1) * 4;
    };
    constexpr size_t kMost = 150 << 10;
    // waves: no more than there are stages, more where the tiles are too few for the device
    // (1 x 2560 x 9728: 9.0 us with 4, 7.2 with 8; 1 x 4096 x 1024 3.4 with 4, 3.6 with 8)
    pl.W = 4;
    while (pl.W < (pl.XI == 16 ? 8 : 16) && groups * pl.W < 4 * cus && pl.W < stages && bytes(1, 2 * pl.W) <= kMost)
      pl.W *= 2;
    while (pl.W > 1 && bytes(1, pl.W) > kMost) pl.W /= 2;
    // and as many as there is LDS for where not every compute unit has a workgroup (7 x 2560 x 9728 in groups
    // of 64: 8 waves 9.1 us, 11 8.8)
    if (pl.XI < 16 && groups < cus)
      while (pl.W < 12 && pl.W < stages && bytes(1, pl.W + 1) <= kMost) ++pl.W;
    // groups a workgroup: one up to four workgroups a compute unit (1 x 19456 x 2560, 608 groups: 8.8 us,
    // 12.0 with two), then their share (1 x 151936 x 1024, 4748 groups: 22.8 us with four, 26.9 with one)
    pl.tiles = static_cast<int>(groups / (4 * cus));
    if (pl.tiles < 1) pl.tiles = 1;
    while (pl.tiles > 1 && bytes(pl.tiles, pl.W) > bytes(1, pl.W) + (8 << 10)) --pl.tiles;
    pl.lds = bytes(pl.tiles, pl.W);
    if (pl.lds <= (160 << 10)) return pl;
  }
  pl.XI = 0;
  auto tiles_of = [&](int bn) { return ((M + pl.bm - 1) / pl.bm) * ((N + bn - 1) / bn); };
  const bool wide = (N + 127) / 128 * 4 >= 2 * cus;
  if (M <= 32 || (M <= 64 && wide)) {
    pl.bm = M <= 32 ? 32 : 64;
    pl.bn = wide ? 128 : 64;
    // two workgroups a compute unit, slices of two steps or more
    const int64_t tiles = tiles_of(pl.bn);
    int64_t s = tiles >= cus ? 1 : (2 * cus) / tiles;
    if (s > blocks / 2) s = blocks / 2;
    pl.slices = s < 1 ? 1 : s > 16 ? 16 : static_cast<int>(s);
    return pl;
  }
  // Tile and slices of the least time, by the ns that a step was measured to take: with 64 x 64 outputs 570,
  // 900 for two workgroups of a compute unit together; with 128 rows, one workgroup a compute unit, 1380
  // for 128 columns to 2200 for 256. Slices cost a launch and their sums' way to memory and back.
  // (128 x 4096 x 1024: 64 x 64 7.5 us, 128 x 128 13.9; 384 x 2560 x 2560: 15, 29, in 4 slices 23;
  // 128 x 2560 x 2560: 64 x 64 14.5, in 2 slices 12.3; 777 x 19456 x 2560: 128 columns 143, 192 114, 256
  // 132; 777 x 2560 x 9728: 104, 81, 71 in 1, 2 and 3 slices.)
  int64_t least = INT64_MAX;
  auto consider = [&](int bm, int bn) {
    const int64_t t = ((M + bm - 1) / bm) * ((N + bn - 1) / bn), slots = bm == 64 ? 2 * cus : cus;
    const int64_t most = t >= cus ? 1 : blocks / 2 < 16 ? blocks / 2 : 16;
    for (int64_t s = 1; s == 1 || (s <= most && t * s <= slots); ++s) {
      const int64_t rounds = t * s / slots, rest = t * s % slots;
      int64_t step;
      if (bm == 64) step = rounds * 900 + (rest > cus ? 900 : rest > 0 ? 570 : 0);
      else step = (rounds + (rest > 0 ? 1 : 0)) * (560 + 32 * bn / 5);
      const int64_t cost = step * ((blocks + s - 1) / s) + (s > 1 ? 2600 + s * M * N / 500 : 0);
      if (cost < least) {
        least = cost;
        pl.bm = bm;
        pl.bn = bn;
        pl.slices = static_cast<int>(s);
      }
    }
  };
  consider(64, 64);
  if (M > 64)
    for (int bn = 128; bn <= (fold == 1 ? 128 : 256); bn += 64) consider(128, bn);
  return pl;
}

template <typename T, int FOLD, int XI> void launch_rows(const Args& a, const Plan& pl, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((a.tiles_n + pl.tiles - 1) / pl.tiles)), block(pl.W * 64);
  if (pl.NT == 1) hipLaunchKernelGGL((w4a16_rows<T, FOLD, XI, 1>), grid, block, pl.lds, st, a);
  else if constexpr (XI < 8) hipLaunchKernelGGL((w4a16_rows<T, FOLD, XI, 2>), grid, block, pl.lds, st, a);
}

template <typename T, typename ST, int FOLD> void launch_gemm(const Args& a, const Plan& pl, dim3 grid, hipStream_t st) {
  const dim3 block(256);
  if (pl.bm == 128 && pl.bn == 128)
    hipLaunchKernelGGL((w4a16_gemm<T, ST, FOLD, 2, 4, 4, 2, 3>), grid, dim3(512), 0, st, a);
  else if (pl.bm == 128) {
    if constexpr (FOLD > 1) {
      if (pl.bn == 256) hipLaunchKernelGGL((w4a16_gemm<T, ST, FOLD, 2, 4, 4, 4, 3>), grid, dim3(512), 0, st, a);
      else hipLaunchKernelGGL((w4a16_gemm<T, ST, FOLD, 2, 4, 4, 3, 3>), grid, dim3(512), 0, st, a);
    }
  } else if (pl.bm == 64 && pl.bn == 128)
    hipLaunchKernelGGL((w4a16_gemm<T, ST, FOLD, 1, 4, 4, 2, 3>), grid, block, 0, st, a);
  else if (pl.bm == 64)
    hipLaunchKernelGGL((w4a16_gemm<T, ST, FOLD, 1, 4, 4, 1, 3>), grid, block, 0, st, a);
  else if (pl.bn == 128)
    hipLaunchKernelGGL((w4a16_gemm<T, ST, FOLD, 1, 4, 2, 2, 4>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((w4a16_gemm<T, ST, FOLD, 1, 4, 2, 1, 4>), grid, block, 0, st, a);
}

template <typename T, int FOLD> int launch(Args a, int64_t group, hipStream_t st) {
  const Plan pl = make_plan(a.M, a.N, a.K, group);
  if (pl.XI) {
    a.tiles = pl.tiles;
    a.tiles_n = static_cast<int32_t>((a.N + 16 * pl.NT - 1) / (16 * pl.NT));
    if (pl.XI == 1) launch_rows<T, FOLD, 1>(a, pl, st);
    else if (pl.XI == 4) launch_rows<T, FOLD, 4>(a, pl, st);
    else if (pl.XI == 8) launch_rows<T, FOLD, 8>(a, pl, st);
    else launch_rows<T, FOLD, 16>(a, pl, st);
    return sd::check_launch("w4a16_linear");
  }
  a.slices = a.part ? pl.slices : 1;  // without its workspace: one slice
  a.tiles_m = static_cast<int32_t>((a.M + pl.bm - 1) / pl.bm);
  a.tiles_n = static_cast<int32_t>((a.N + pl.bn - 1) / pl.bn);
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.tiles_m) * a.tiles_n * a.slices));
  if (a.scale_f32) launch_gemm<T, float, FOLD>(a, pl, grid, st);
  else if (a.scale_f16) launch_gemm<T, _Float16, FOLD>(a, pl, grid, st);
  else launch_gemm<T, __bf16, FOLD>(a, pl, grid, st);
  const int rc = sd::check_launch("w4a16_linear");
  if (rc != SD_OK || a.slices == 1) return rc;
  int64_t wgs = (a.M * a.N + 255) / 256;
  if (wgs > 2048) wgs = 2048;
  hipLaunchKernelGGL((w4a16_reduce<T>), dim3(static_cast<unsigned>(wgs)), dim3(256), 0, st, a);
  return sd::check_launch("w4a16_linear");
}

template <typename T> int launch(const Args& a, int group, hipStream_t st) {
  if (group % 128 == 0) return launch<T, 4>(a, group, st);
  if (group % 64 == 0) return launch<T, 2>(a, group, st);
  return launch<T, 1>(a, group, st);
}

// (a launch takes fewer than 2^32 threads: tiles of 128 x 128 or more and 512 threads, 16 slices while tiles are few)
bool sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M <= (1ll << 24) && N <= (1ll << 21) && K <= (1ll << 20) &&
         ((M + 127) / 128) * ((N + 127) / 128) < (1ll << 23);
}

}  // namespace

extern "C" size_t sd_w4a16_workspace_size(int64_t M, int64_t N, int64_t K, int32_t group_size) {
  if (M <= 0 || N <= 0 || K <= 0 || group_size <= 0 || !sizes_ok(M, N, K)) return 0;
  const Plan pl = make_plan(M, N, K, group_size);
  return pl.slices > 1 ? static_cast<size_t>(pl.slices) * M * N * sizeof(float) : 0;
}

extern "C" int64_t sd_w4a16_plan(int64_t M, int64_t N, int64_t K, int32_t group_size) {
  if (M <= 0 || N <= 0 || K <= 0 || group_size <= 0 || group_size % 32 != 0 || K % group_size != 0 || !sizes_ok(M, N, K))
    return 0;
  const Plan pl = make_plan(M, N, K, group_size);
  if (pl.XI) return pl.W | 16 * pl.NT << 8;
  return pl.slices | pl.bn << 8 | static_cast<int64_t>(pl.bm) << 20;
}

extern "C" int sd_w4a16_linear(const void* x, int64_t x_stride_m, const uint8_t* w, int64_t w_stride_n,
                               const void* scale, int32_t scale_dtype, int32_t group_size,
                               const void* bias, void* y, int64_t y_stride_m, int64_t M, int64_t N,
                               int64_t K, int32_t dtype, void* workspace, size_t workspace_bytes,
                               void* stream) {
  sd::clear_error();
  const char* what = "w4a16_linear";
  if (M < 0 || N <= 0 || K <= 0 || group_size <= 0) {
    sd::set_error("%s: invalid sizes (M=%lld N=%lld K=%lld group=%d)", what, (long long)M, (long long)N,
                  (long long)K, group_size);
    return SD_ERR_VALUE;
  }
  if (group_size % 32 != 0 || K % group_size != 0) {
    sd::set_error("%s: groups must be a multiple of 32 columns and divide K, got %d of %lld", what,
                  group_size, (long long)K);
    return SD_ERR_UNSUPPORTED;
  }
  if ((dtype != SD_BF16 && dtype != SD_F16) ||
      (scale_dtype != SD_BF16 && scale_dtype != SD_F16 && scale_dtype != SD_F32)) {
    sd::set_error("%s: dtype must be bf16 or f16, the scales' bf16, f16 or f32", what);
    return SD_ERR_UNSUPPORTED;
  }
  if (!sizes_ok(M, N, K) || (M > 1 && x_stride_m > (1ll << 24)) || (N > 1 && w_stride_n > (1ll << 24))) {
    sd::set_error("%s: M=%lld N=%lld K=%lld (strides %lld, %lld) too large", what, (long long)M, (long long)N,
                  (long long)K, (long long)x_stride_m, (long long)w_stride_n);
    return SD_ERR_UNSUPPORTED;
  }
  if (M == 0) return SD_OK;
  if (!x || !w || !scale || !y) {
    sd::set_error("%s: null pointer argument", what);
    return SD_ERR_VALUE;
  }
  if (!sd::strides_ok({x_stride_m, w_stride_n, y_stride_m}) || x_stride_m < 0 || w_stride_n < 0 ||
      y_stride_m < 0) {
    sd::set_error("%s: strides must lie in [0, 2^40]", what);
    return SD_ERR_VALUE;
  }
  if (!sd::aligned16(x) || !sd::aligned16(w) || (M > 1 && x_stride_m % 8 != 0) ||
      (N > 1 && w_stride_n % 16 != 0)) {
    sd::set_error("%s: x and weight rows must be 16-byte aligned", what);
    return SD_ERR_UNSUPPORTED;
  }
  if (M > 1 && y_stride_m < N) {
    sd::set_error("%s: rows of y overlap (stride %lld, %lld columns)", what, (long long)y_stride_m, (long long)N);
    return SD_ERR_VALUE;
  }
  if (sd::span16(x, M, x_stride_m, K).overlaps(sd::span16(y, M, y_stride_m, N))) {
    sd::set_error("%s: y shares memory with x", what);
    return SD_ERR_VALUE;
  }
  Args a;
  a.x = static_cast<const uint16_t*>(x);
  a.xs = x_stride_m;
  a.w = w;
  a.ws = w_stride_n;
  a.scale = scale;
  a.scale_f16 = scale_dtype == SD_F16;
  a.scale_f32 = scale_dtype == SD_F32;
  a.groups = static_cast<int32_t>(K / group_size);
  const uint64_t parts = static_cast<uint64_t>(group_size) / 32;
  a.inv32 = ((1ull << 32) + parts - 1) / parts;
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.ys = y_stride_m;
  a.wide_y = sd::aligned16(y) && y_stride_m % 8 == 0;
  a.M = M;
  a.N = N;
  a.K = static_cast<int32_t>(K);
  const size_t need = sd_w4a16_workspace_size(M, N, K, group_size);
  a.part = need && workspace && workspace_bytes >= need ? static_cast<float*>(workspace) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SD_BF16) return launch<__bf16>(a, group_size, st);
  return launch<_Float16>(a, group_size, st);
}
