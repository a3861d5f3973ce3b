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
// Up to 16 rows (w4a16_gemv): bound by the weights' bytes, N K / 2. A workgroup takes 16 weight rows,
// its waves the 128-column blocks in turn; their sums meet in LDS. Above (w4a16_gemm): a tile of
// activation rows goes to LDS once for the four waves, each with its own weight rows in registers.
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
  int32_t scale_dtype;
  int32_t groups;  // per weight row
  int32_t group;
  const uint16_t* bias;
  uint16_t* y;
  int64_t ys;
  int64_t M, N;
  int32_t K;
};

// Raw bits of one scale (its conversion waits for the load only where it is used).
__device__ __forceinline__ uint32_t load_scale(const Args& a, int64_t at) {
  return a.scale_dtype == SD_F32 ? static_cast<const uint32_t*>(a.scale)[at]
                                 : static_cast<const uint16_t*>(a.scale)[at];
}
__device__ __forceinline__ float scale_value(const Args& a, uint32_t bits) {
  if (a.scale_dtype == SD_F32) return __uint_as_float(bits);
  if (a.scale_dtype == SD_BF16) return __uint_as_float(bits << 16);
  return sd::from_bits<_Float16>(static_cast<uint16_t>(bits));
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

// 8 activations in the order 0, 4, 1, 5, 2, 6, 3, 7.
__device__ __forceinline__ u32x4 reorder(u32x4 v) {
  return u32x4{__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
               __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
}

template <typename T> __device__ __forceinline__ uint32_t minus24() {  // two T of -24
  return __is_same(T, __bf16) ? 0xC1C0C1C0u : 0xCE00CE00u;
}

constexpr int kBlock = 128;  // columns of a step: one 16-byte load of weights a lane

// FOLD: MFMAs (32 columns each) between two scalings, 4, 2 or 1.
template <typename T, int FOLD, int W>
__global__ __launch_bounds__(W * 64) void w4a16_gemv(Args a) {
  __shared__ float red[W][16][17];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int64_t n = min(n0 + lr, a.N - 1);
  const uint8_t* wrow = a.w + n * a.ws;
  const uint16_t* xrow = a.x + min(static_cast<int64_t>(lr), a.M - 1) * a.xs;
  const int blocks = (a.K + kBlock - 1) / kBlock;

  struct Block {
    u32x4 w, x[4];
    uint32_t s[4 / FOLD];
  };
  auto load = [&](Block& d, int blk) {
    const int kb = min(blk, blocks - 1) * kBlock;
    d.w = sd::load16_stream(wrow + min(kb + 32 * lg, a.K - 32) / 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) d.x[i] = sd::load16(xrow + min(kb + 32 * i + 8 * lg, a.K - 8));
#pragma unroll
    for (int f = 0; f < 4 / FOLD; ++f)
      d.s[f] = load_scale(a, n * a.groups + min(kb + 32 * FOLD * f, a.K - 32) / a.group);
  };
  const uint32_t base = sd::code_base<T>();
  const u32x4 m24 = {minus24<T>(), minus24<T>(), minus24<T>(), minus24<T>()};
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const Block& d, int blk) {
    const int kb = blk * kBlock;
    const u32x4 w = turn(d.w);
#pragma unroll
    for (int f = 0; f < 4 / FOLD; ++f) {
      f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < FOLD; ++j) {
        const int i = f * FOLD + j;
        u32x4 x = reorder(d.x[i]);
        if (kb + 32 * i >= a.K) x = u32x4{0u, 0u, 0u, 0u};  // past the last column
        t = sd::Elem<T>::mfma(x, m24, t);
        t = sd::Elem<T>::mfma(x, sd::unpack8<T>(w[i], base), t);
      }
      acc += scale_value(a, d.s[f]) * t;
    }
  };
  constexpr int kAhead = 2;
  Block ring[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(ring[i], wave + i * W);
  for (int blk = wave; blk < blocks; blk += kAhead * W) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (blk + i * W < blocks) compute(ring[i], blk + i * W);
      load(ring[i], blk + (i + kAhead) * W);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[wave][4 * lg + i][lr] = acc[i];
  __syncthreads();
  for (int i = tid; i < 256; i += W * 64) {
    const int m = i >> 4, c = i & 15;
    if (m >= a.M || n0 + c >= a.N) continue;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < W; ++v) s += red[v][m][c];
    if (a.bias) s += sd::from_bits<T>(a.bias[n0 + c]);
    a.y[m * a.ys + n0 + c] = sd::to_bits<T>(s);
  }
}

// BM = 16 MT activation rows by BN = 64 NT weight rows; wave v has weight rows 16 NT v .. + 16 NT.
template <typename T, int FOLD, int MT, int NT>
__global__ __launch_bounds__(256) void w4a16_gemm(Args a) {
  constexpr int BM = 16 * MT, BN = 64 * NT, NF = 4 / FOLD;
  __shared__ __attribute__((aligned(16))) u32x4 lx[2][BM * 16];     // rows of 16 units of 8 columns
  __shared__ __attribute__((aligned(16))) float lsum[2][NF][BM];    // -24 sum x of a fold's columns
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * BM, n0 = static_cast<int64_t>(blockIdx.y) * BN;
  const int blocks = (a.K + kBlock - 1) / kBlock;

  // ---- activations: unit u of row r by the 16 threads u of each row
  const int u = tid & 15, r0 = tid >> 4;
  u32x4 xr[MT];
  auto load_x = [&](int blk) {
    const int k = min(blk * kBlock + 8 * u, a.K - 8);
#pragma unroll
    for (int i = 0; i < MT; ++i)
      xr[i] = sd::load16(a.x + min(m0 + 16 * i + r0, a.M - 1) * a.xs + k);
  };
  auto put_x = [&](int blk, int buf) {
    const bool in = blk * kBlock + 8 * u < a.K;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const u32x4 v = in ? reorder(xr[i]) : u32x4{0u, 0u, 0u, 0u};
      const int r = 16 * i + r0;
      lx[buf][r * 16 + (u ^ (r & 15))] = v;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) s = sd::dot2<T>(v[e], minus24<T>(), s);
      s = sd::dpp_add<0xB1>(s);
      s = sd::dpp_add<0x4E>(s);
      if constexpr (FOLD >= 2) s = sd::dpp_add<0x141>(s);
      if constexpr (FOLD >= 4) s = sd::dpp_add<0x140>(s);
      if (u % (4 * FOLD) == 0) lsum[buf][u / (4 * FOLD)][r] = s;
    }
  };
  // ---- weights and scales of this wave's rows
  u32x4 wr[NT];
  uint32_t sr[NT][NF];
  int64_t nrow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) nrow[t] = min(n0 + (wave * NT + t) * 16 + lr, a.N - 1);
  auto load_w = [&](int blk) {
    const int kb = blk * kBlock;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      wr[t] = sd::load16(a.w + nrow[t] * a.ws + min(kb + 32 * lg, a.K - 32) / 2);
#pragma unroll
      for (int f = 0; f < NF; ++f)
        sr[t][f] = load_scale(a, nrow[t] * a.groups + min(kb + 32 * FOLD * f, a.K - 32) / a.group);
    }
  };

  const uint32_t base = sd::code_base<T>();
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  load_x(0);
  load_w(0);
  put_x(0, 0);
  __syncthreads();
  for (int blk = 0; blk < blocks; ++blk) {
    const int buf = blk & 1;
    u32x4 wf[NT][4];
    float sv[NT][NF];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const u32x4 w = turn(wr[t]);
#pragma unroll
      for (int i = 0; i < 4; ++i) wf[t][i] = sd::unpack8<T>(w[i], base);
#pragma unroll
      for (int f = 0; f < NF; ++f) sv[t][f] = scale_value(a, sr[t][f]);
    }
    const int next = min(blk + 1, blocks - 1);
    load_x(next);
    load_w(next);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      u32x4 xf[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) xf[j] = lx[buf][(16 * i + lr) * 16 + ((4 * j + lg) ^ lr)];
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const f32x4 start = __builtin_bit_cast(f32x4, sd::load16(&lsum[buf][f][16 * i + 4 * lg]));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          f32x4 d = start;
#pragma unroll
          for (int j = 0; j < FOLD; ++j) d = sd::Elem<T>::mfma(xf[f * FOLD + j], wf[t][f * FOLD + j], d);
          acc[i][t] += sv[t][f] * d;
        }
      }
    }
    if (blk + 1 < blocks) put_x(blk + 1, buf ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = n0 + (wave * NT + t) * 16 + lr;
    if (n >= a.N) continue;
    const float b = a.bias ? sd::from_bits<T>(a.bias[n]) : 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t m = m0 + 16 * i + 4 * lg + e;
        if (m < a.M) a.y[m * a.ys + n] = sd::to_bits<T>(acc[i][t][e] + b);
      }
  }
}

template <typename T, int FOLD> int launch(const Args& a, hipStream_t st) {
  if (a.M <= 16) {
    const dim3 grid(static_cast<unsigned>((a.N + 15) / 16));
    hipLaunchKernelGGL((w4a16_gemv<T, FOLD, 4>), grid, dim3(256), 0, st, a);
  } else {
    auto grid = [&](int bm, int bn) {
      return dim3(static_cast<unsigned>((a.M + bm - 1) / bm), static_cast<unsigned>((a.N + bn - 1) / bn));
    };
    if (a.M <= 32) hipLaunchKernelGGL((w4a16_gemm<T, FOLD, 2, 1>), grid(32, 64), dim3(256), 0, st, a);
    else if (a.M <= 256) hipLaunchKernelGGL((w4a16_gemm<T, FOLD, 4, 2>), grid(64, 128), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((w4a16_gemm<T, FOLD, 8, 4>), grid(128, 256), dim3(256), 0, st, a);
  }
  return sd::check_launch("w4a16_linear");
}

}  // namespace

extern "C" int sd_w4a16_linear(const void* x, int64_t x_stride_m, const uint8_t* w, int64_t w_stride_n,
                               const void* scale, int32_t scale_dtype, int32_t group_size,
                               const void* bias, void* y, int64_t y_stride_m, int64_t M, int64_t N,
                               int64_t K, int32_t dtype, void* stream) {
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
  if (M > (1ll << 24) || N > (1ll << 21) || K > (1ll << 24)) {
    sd::set_error("%s: M=%lld N=%lld K=%lld too large", what, (long long)M, (long long)N, (long long)K);
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
  a.scale_dtype = scale_dtype;
  a.groups = static_cast<int32_t>(K / group_size);
  a.group = group_size;
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.ys = y_stride_m;
  a.M = M;
  a.N = N;
  a.K = static_cast<int32_t>(K);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool bf = dtype == SD_BF16;
  if (group_size % 128 == 0) return bf ? launch<__bf16, 4>(a, st) : launch<_Float16, 4>(a, st);
  if (group_size % 64 == 0) return bf ? launch<__bf16, 2>(a, st) : launch<_Float16, 2>(a, st);
  return bf ? launch<__bf16, 1>(a, st) : launch<_Float16, 1>(a, st);
}
