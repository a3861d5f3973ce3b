// act_int8.hip — activations in 8 bits with a scale per row, for gfx950: what the linears of w8a8.hip read.
//
//   v = x                                    (quantize)
//   v = s w, s = x + residual in fp32        (RMSNorm; residual_out = s rounded once)
//   code = round_half_even(127 v / max |v|), scale = max |v| / 127 (times 1 / sqrt(mean(s^2) + eps))
//   value = code scale
//
// The root mean square cancels out of the codes: the sum of squares and max |v| are one reduction, between
// which and the codes the row stays in registers. A code is that of the fp32 quotient of the fp32 v and max |v|; the
// normalised value itself is never rounded. A row with a NaN or an infinity in s or w has scale NaN and codes 0, a row of
// zeros scale 0. Where only the product leaves fp32 (bf16 s and w) it is formed again 2^128 smaller.
// Bound by memory: 7 bytes an element with a residual, 3 without either (8192 x 2560 with a residual 24 us, 147 MB at
// 6.2 TB/s from and to the caches; 4001 x 4096 without 9.9, 49 MB at 5.0), with vector issue close behind (14 of those
// 24 us); few rows by their latency, 2.2 to 3 us.
#include <math.h>

#include <type_traits>

#include "sd_common.h"

namespace {

using sd::u32x4;

struct Params {
  const uint16_t* x;
  int64_t xs;
  const uint16_t* res;  // NULL: no residual
  int64_t rs;
  const uint16_t* w;
  int8_t* codes;
  int64_t cs;
  float* scale;
  uint16_t* res_out;
  int64_t ros;
  int64_t rows;
  int32_t K;
  float eps;
};

__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max_u32(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false)));
}
// Maximum over the wave, by the moves of sd::xor_sum_down<32>.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max_u32(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max_u32(b[0], b[1]);
  v = dpp_max<0x128>(v);  // row_ror:8
  v = dpp_max<0x124>(v);  // row_ror:4
  v = dpp_max<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  return dpp_max<0xB1>(v);  // quad_perm [1, 0, 3, 2]
}

__device__ __forceinline__ float element(const u32x4& v, int i, float (*to)(uint16_t)) {
  return to(static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1))));
}

// The codes of 8 values: the quotient 127 v / most, rounded to fp32, to the nearest whole number (half to even). The
// product with the rounded 127 / most is off by up to 2^-16; its remainder 127 v - q most, exact in two parts, brings it
// to the nearest fp32, so that a tie is one and stays one. SHORT: v and most are 16-bit values, whose products are exact
// in one. No branch: taken only next to a border, the correction cost 1.2 us of a launch of 2.4 (its code came late).
template <bool SHORT>
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float most, float inv, float inv1) {
#pragma clang fp contract(off)
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float q = v[i] * inv, rem;
    if constexpr (SHORT) {
      rem = fmaf(-q, most, 127.f * v[i]);
    } else {
      const float p = q * most;
      rem = fmaf(127.f, v[i], -p) - fmaf(q, most, -p);
    }
    q = fmaf(rem, inv1, q);
    b[i] = __float_as_uint(q + 0x1.8p23f);  // the whole number nearest to q, in the low byte
  }
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __builtin_amdgcn_perm(b[2 * i + 1], b[2 * i], 0x0c0c0400u);
  return uint2{h[0] | h[1] << 16, h[2] | h[3] << 16};
}

// Maximum over the threads of a row; `red` may be in use by the row's other waves.
template <int TPR> __device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* red, int t) {
  v = wave_max(v);
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((t & 63) == 0) red[t >> 6] = v;
    __syncthreads();
    v = wave_max(red[t % (TPR / 64)]);
  }
  return v;
}

// TPR threads a row (64: four rows a workgroup, no barrier); thread t holds the 8-element chunks t, t + TPR, ...
// The squares of 64 chunks are summed by a wave, then those sums in order, whichever TPR and C <= 2 the launch took: a
// row's scale is the same bits whatever the other rows.
template <typename T, bool NORM, bool RES, int TPR, int C>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rows_int8_kernel(Params p) {
#pragma clang fp contract(off)
  constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
  constexpr int kSums = C <= 2 ? C : 1;
  constexpr bool kWide = NORM && std::is_same<T, __bf16>::value;  // (fp16 products stay below 2^34)
  __shared__ float red_sum[kSums * (TPR / 64)];
  __shared__ uint32_t red_max[TPR / 64];
  const int t = static_cast<int>(threadIdx.x) % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows +
                      __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / TPR);
  if (kRows > 1 && row >= p.rows) return;
  const uint16_t* x = p.x + row * p.xs;
  const uint16_t* res = RES ? p.res + row * p.rs : nullptr;
  u32x4 xb[C], rb[C], wb[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (c * TPR * 8 >= p.K) break;  // uniform
    const int e = min((c * TPR + t) * 8, p.K - 8);
    xb[c] = sd::load16(x + e);
    if constexpr (RES) rb[c] = sd::load16(res + e);
    if constexpr (NORM) wb[c] = sd::load16(p.w + e);
  }
  float v[C][8], sums[kSums] = {};
  uint32_t most_bits = 0;
  // Chunk c's products 2^128 smaller. Exact where it counts: where s or w is below 2^-62 the product is far below half a
  // level of a row that left fp32.
  [[maybe_unused]] uint32_t smaller = 0;  // the chunks that are
  [[maybe_unused]] auto again = [&](int c, int e) {
    const u32x4 xa = RES ? xb[c] : sd::load16(x + e), wa = sd::load16(p.w + e);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float s = element(xa, i, sd::from_bits<T>);
      if constexpr (RES) s = s + element(rb[c], i, sd::from_bits<T>);
      v[c][i] = s * 0x1p-64f * (element(wa, i, sd::from_bits<T>) * 0x1p-64f);
    }
    smaller |= 1u << c;
  };
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int e = (c * TPR + t) * 8;
    if (e >= p.K) break;  // (whole waves, mostly)
    float s[8];
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = element(xb[c], i, sd::from_bits<T>);
      if constexpr (RES) s[i] = s[i] + element(rb[c], i, sd::from_bits<T>);
      v[c][i] = s[i];
      if constexpr (NORM) {
        sums[kSums == 1 ? 0 : c] = fmaf(s[i], s[i], sums[kSums == 1 ? 0 : c]);
        v[c][i] = s[i] * element(wb[c], i, sd::from_bits<T>);
      }
      bits = max_u32(bits, __float_as_uint(v[c][i]) & 0x7fffffffu);  // NaN above infinity above all else
    }
    most_bits = max_u32(most_bits, bits);
    if constexpr (RES)
      sd::store16(p.res_out + row * p.ros + e, u32x4{sd::pack2<T>(s[0], s[1]), sd::pack2<T>(s[2], s[3]),
                                                     sd::pack2<T>(s[4], s[5]), sd::pack2<T>(s[6], s[7])});
    if constexpr (kWide && RES && C > 2)
      if (bits == 0x7f800000u) again(c, e);
  }
  // With a residual, s has to be formed again from what was loaded: residual_out may have taken its place in memory. Of
  // four chunks each for itself, since keeping all of them to here takes registers (777 x 9728 12.0 us, 10.9 so).
  if constexpr (kWide && RES && C <= 2) {
    if (most_bits == 0x7f800000u) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if ((c * TPR + t) * 8 >= p.K) break;
        again(c, (c * TPR + t) * 8);
      }
    }
  }
  float sum = 0.f;
  if constexpr (NORM) {
#pragma unroll
    for (int c = 0; c < kSums; ++c) sums[c] = sd::xor_sum_down<32>(sums[c]);
  }
  most_bits = wave_max(most_bits);
  if constexpr (TPR > 64) {
    const int wave = t >> 6;
    if ((t & 63) == 0) {
#pragma unroll
      for (int c = 0; c < kSums; ++c) red_sum[c * (TPR / 64) + wave] = sums[c];
      red_max[wave] = most_bits;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSums * (TPR / 64); ++i) sum += red_sum[i];
    if constexpr (TPR == 1024) {
      most_bits = wave_max(red_max[t % 16]);  // (16 more registers would leave one row a compute unit instead of two)
    } else {
      most_bits = 0;
#pragma unroll
      for (int i = 0; i < TPR / 64; ++i) most_bits = max_u32(most_bits, red_max[i]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < kSums; ++c) sum += sums[c];
  }
  [[maybe_unused]] float up = 1.f;  // v is 1 / up^2 of the product
  if constexpr (kWide) {
    if (most_bits == 0x7f800000u) {  // uniform: of the row. All its products 2^128 smaller; an infinity of s or w stays one
      uint32_t bits = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = (c * TPR + t) * 8;
        if (e >= p.K) break;
        if constexpr (!RES) again(c, e);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!(smaller >> c & 1)) v[c][i] = v[c][i] * 0x1p-64f * 0x1p-64f;
          bits = max_u32(bits, __float_as_uint(v[c][i]) & 0x7fffffffu);
        }
      }
      most_bits = row_max<TPR>(bits, red_max, t);
      up = 0x1p64f;
    }
  }
  const bool none = most_bits >= 0x7f800000u || most_bits == 0;
  const float most = __uint_as_float(most_bits);
  if (t == 0) {
    float scale = most / 127.f;
    if constexpr (NORM) scale = scale * (1.f / sqrtf(sum / static_cast<float>(p.K) + p.eps)) * up * up;
    if (most_bits == 0) scale = 0.f;
    if (most_bits >= 0x7f800000u) scale = __uint_as_float(0x7fc00000u);
    p.scale[row] = scale;
  }
  // by a power of two into the range where 127 v and the quotient's inverse are finite and normal
  const float to = most < 0x1p-60f ? 0x1p64f : most > 0x1p60f ? 0x1p-64f : 1.f;
  const float scaled = most * to, inv = 127.f / scaled, inv1 = inv * (1.f / 127.f);
  if (to != 1.f) {  // uniform: of the row
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] *= to;
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int e = (c * TPR + t) * 8;
    if (e >= p.K) break;
    *reinterpret_cast<uint2*>(p.codes + row * p.cs + e) = none ? uint2{0, 0} : codes8<!NORM>(v[c], scaled, inv, inv1);
  }
}

// code scale in T: a wave takes 2048 columns of a row.
constexpr int kSpan = 2048;
struct BackParams {
  const int8_t* codes;
  int64_t cs;
  const float* scale;
  void* out;
  int64_t os;
  int64_t items;  // rows * spans
  int32_t spans;
  int32_t K;
};
template <typename T> __global__ __launch_bounds__(256) void rows_from_int8_kernel(BackParams p) {
  const int lane = threadIdx.x & 63;
  const uint32_t item = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= p.items) return;
  const uint32_t row = item / static_cast<uint32_t>(p.spans);
  const int first = static_cast<int>(item - row * p.spans) * kSpan + lane * 8;
  const int8_t* codes = p.codes + row * p.cs;
  const float scale = p.scale[row];
  uint2 b[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) b[c] = *reinterpret_cast<const uint2*>(codes + min(first + c * 512, p.K - 8));
  T* const out = static_cast<T*>(p.out) + row * p.os;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int e = first + c * 512;
    if (e >= p.K) break;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t word = i < 4 ? b[c].x : b[c].y;
      f[i] = static_cast<float>(static_cast<int8_t>(word >> (8 * (i % 4)))) * scale;
    }
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<sd::f32x4*>(out + e) = sd::f32x4{f[0], f[1], f[2], f[3]};
      *reinterpret_cast<sd::f32x4*>(out + e + 4) = sd::f32x4{f[4], f[5], f[6], f[7]};
    } else {
      sd::store16(out + e, u32x4{sd::pack2<T>(f[0], f[1]), sd::pack2<T>(f[2], f[3]), sd::pack2<T>(f[4], f[5]),
                                 sd::pack2<T>(f[6], f[7])});
    }
  }
}

template <typename T, bool NORM, bool RES> void launch(const Params& p, hipStream_t st) {
#define SD_ROWS_INT8(tpr, c)                                                                              \
  hipLaunchKernelGGL((rows_int8_kernel<T, NORM, RES, tpr, c>),                                            \
                     dim3(static_cast<unsigned>(tpr < 256 ? (p.rows + 256 / tpr - 1) / (256 / tpr) : p.rows)), \
                     dim3(tpr < 256 ? 256 : tpr), 0, st, p)
  // A wave a row saves the barrier where rows are short and many, a thread for 8 elements saves steps where they are few
  // (norm with residual, us): 1 x 1024 2.5 with 256 threads, 2.7 with 64, 4096 x 1024 6.9 and 6.1; 1 x 2560 2.6 with 512
  // threads, 2.8 with 256, 200 x 2560 3.2 and 3.4, 32768 x 2560 107 and 101. Past that 512 threads: 777 x 8192 8.8, 9.6
  // with 256, 9.8 with 1024; 777 x 9728 10.8, 11.2 with 1024.
  if (p.K <= 512) SD_ROWS_INT8(64, 1);
  else if (p.K <= 1024 && p.rows > 512) SD_ROWS_INT8(64, 2);
  else if (p.K <= 2048) SD_ROWS_INT8(256, 1);
  else if (p.K <= 4096 && p.rows <= 512) SD_ROWS_INT8(512, 1);
  else if (p.K <= 4096) SD_ROWS_INT8(256, 2);
  else if (p.K <= 8192) SD_ROWS_INT8(512, 2);
  else if (p.K <= 16384) SD_ROWS_INT8(512, 4);
  else SD_ROWS_INT8(1024, 4);
#undef SD_ROWS_INT8
}
template <typename T> void launch(const Params& p, hipStream_t st) {
  if (!p.w) launch<T, false, false>(p, st);
  else if (p.res) launch<T, true, true>(p, st);
  else launch<T, true, false>(p, st);
}

constexpr int kMostColumns = 32768;
// (a launch takes fewer than 2^32 threads)
constexpr int64_t most_rows(int32_t columns) { return columns > 4096 ? (1 << 22) - 1 : (1 << 24) - 1; }

// Whether rows of residual_out (stride `os` >= K) share a byte with other rows of `in`, or with their own shifted: a
// workgroup loads a row before it stores it, another's rows at any time. Exact, so that rows may lie between rows.
bool meets_rows(const uint16_t* out, int64_t os, const uint16_t* in, int64_t is, int64_t rows, int64_t K) {
  if (in == out && (rows == 1 || is == os)) return false;
  if (!sd::span_rows(out, rows, 2 * os, 2 * K).overlaps(sd::span_rows(in, rows, 2 * is, 2 * K))) return false;
  if (rows == 1) return true;
  const __int128 step = 2 * os, width = 2 * K;
  const __int128 first = static_cast<__int128>(reinterpret_cast<uintptr_t>(in)) - reinterpret_cast<uintptr_t>(out);
  auto near_row = [&](__int128 at, int64_t least) {  // bytes at .. at + width and one of the rows `least` .. rows - 1
    __int128 j = at / step - (at % step < 0);
    for (int i = 0; i < 2; ++i, ++j)
      if (j >= least && j < rows && at - j * step < width && j * step - at < width) return true;
    return false;
  };
  if (is == os) return near_row(first, 1 - rows);  // every row's place is that of the first
  for (int64_t i = 0; i < rows; ++i)
    if (near_row(first + static_cast<__int128>(i) * 2 * is, 0)) return true;
  return false;
}

// What both entries ask of their sizes and outputs; SD_OK or the refusal.
int check(const char* what, const Params& p, int32_t dtype, bool residual) {
  if (p.rows < 0 || p.K <= 0) {
    sd::set_error("%s: invalid sizes (%lld rows of %d columns)", what, (long long)p.rows, p.K);
    return SD_ERR_VALUE;
  }
  if (p.K % 16 != 0 || p.K > kMostColumns || p.rows > most_rows(p.K) || (dtype != SD_BF16 && dtype != SD_F16)) {
    sd::set_error("%s: columns must be a multiple of 16 up to %d, rows below 2^24 (2^22 past 4096 columns), dtype bf16 "
                  "or f16 (%lld rows of %d columns, dtype %d)", what, kMostColumns, (long long)p.rows, p.K, dtype);
    return SD_ERR_UNSUPPORTED;
  }
  if (p.rows == 0) return SD_OK;
  if (!p.x || !p.codes || !p.scale || (residual && !p.res_out)) {
    sd::set_error("%s: null pointer argument", what);
    return SD_ERR_VALUE;
  }
  if (!sd::strides_ok({p.xs, p.rs, p.cs, p.ros}) || (p.rows > 1 && (p.cs < p.K || (residual && p.ros < p.K)))) {
    sd::set_error("%s: strides must lie within 2^40, output rows may not overlap", what);
    return SD_ERR_VALUE;
  }
  const bool more = p.rows > 1;
  if (!sd::aligned16(p.x) || !sd::aligned16(p.codes) || (more && (p.xs % 8 || p.cs % 16)) ||
      (p.w && !sd::aligned16(p.w)) ||
      (residual && (!sd::aligned16(p.res) || !sd::aligned16(p.res_out) || (more && (p.rs % 8 || p.ros % 8))))) {
    sd::set_error("%s: rows must be 16-byte aligned", what);
    return SD_ERR_UNSUPPORTED;
  }
  const int64_t width = 2 * static_cast<int64_t>(p.K);
  const sd::Span codes = sd::span_rows(p.codes, p.rows, p.cs, p.K), scale = sd::span_rows(p.scale, p.rows, 4, 4);
  const sd::Span w = sd::span_rows(p.w, 1, 0, width), res_out = sd::span_rows(p.res_out, p.rows, 2 * p.ros, width);
  bool shared = codes.overlaps(scale) || res_out.overlaps(w);
  for (const sd::Span& o : {sd::span_rows(p.x, p.rows, 2 * p.xs, width), sd::span_rows(p.res, p.rows, 2 * p.rs, width),
                            w, res_out})
    shared |= codes.overlaps(o) || scale.overlaps(o);
  if (residual)
    shared |= meets_rows(p.res_out, p.ros, p.x, p.xs, p.rows, p.K) || meets_rows(p.res_out, p.ros, p.res, p.rs, p.rows, p.K);
  if (shared) {
    sd::set_error("%s: outputs share memory with another argument", what);
    return SD_ERR_VALUE;
  }
  return SD_OK;
}

int run(const char* what, const Params& p, int32_t dtype, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SD_BF16) launch<__bf16>(p, st);
  else launch<_Float16>(p, st);
  return sd::check_launch(what);
}

}  // namespace

extern "C" int sd_quantize_rows_int8(const void* x, int64_t x_stride, int8_t* codes, int64_t codes_stride,
                                     float* scale, int64_t rows, int32_t columns, int32_t dtype, void* stream) {
  sd::clear_error();
  const Params p{static_cast<const uint16_t*>(x), x_stride, nullptr, 0, nullptr, codes, codes_stride, scale,
                 nullptr, 0, rows, columns, 0.f};
  const int rc = check("quantize_rows_int8", p, dtype, false);
  return rc != SD_OK || rows == 0 ? rc : run("quantize_rows_int8", p, dtype, stream);
}

extern "C" int sd_rmsnorm_int8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                               const void* weight, int8_t* codes, int64_t codes_stride, float* scale,
                               void* residual_out, int64_t residual_out_stride, int64_t rows, int32_t hidden,
                               float eps, int32_t dtype, void* stream) {
  sd::clear_error();
  const Params p{static_cast<const uint16_t*>(x), x_stride, static_cast<const uint16_t*>(residual), residual_stride,
                 static_cast<const uint16_t*>(weight), codes, codes_stride, scale,
                 static_cast<uint16_t*>(residual_out), residual_out_stride, rows, hidden, eps};
  const int rc = check("rmsnorm_int8", p, dtype, residual != nullptr);
  if (rc != SD_OK || rows == 0) return rc;
  if (!weight) {
    sd::set_error("rmsnorm_int8: null pointer argument");
    return SD_ERR_VALUE;
  }
  return run("rmsnorm_int8", p, dtype, stream);
}

extern "C" int sd_dequantize_rows_int8(const int8_t* codes, int64_t codes_stride, const float* scale, void* out,
                                       int64_t out_stride, int64_t rows, int32_t columns, int32_t dtype,
                                       void* stream) {
  sd::clear_error();
  const char* what = "dequantize_rows_int8";
  if (rows < 0 || columns <= 0) {
    sd::set_error("%s: invalid sizes (%lld rows of %d columns)", what, (long long)rows, columns);
    return SD_ERR_VALUE;
  }
  BackParams p{codes, codes_stride, scale, out, out_stride, 0, (columns - 1) / kSpan + 1, columns};
  if (columns % 16 != 0 || rows >= (1ll << 26) / p.spans || (dtype != SD_BF16 && dtype != SD_F16 && dtype != SD_F32)) {
    sd::set_error("%s: columns must be a multiple of 16, rows below 2^26 for each 2048 of them, dtype bf16, f16 or f32 "
                  "(%lld rows of %d columns, dtype %d)", what, (long long)rows, columns, dtype);
    return SD_ERR_UNSUPPORTED;
  }
  if (rows == 0) return SD_OK;
  if (!codes || !scale || !out) {
    sd::set_error("%s: null pointer argument", what);
    return SD_ERR_VALUE;
  }
  if (!sd::strides_ok({codes_stride, out_stride}) || (rows > 1 && out_stride < columns)) {
    sd::set_error("%s: strides must lie within 2^40, output rows may not overlap", what);
    return SD_ERR_VALUE;
  }
  if (!sd::aligned16(codes) || !sd::aligned16(out) ||
      (rows > 1 && (codes_stride % 16 || out_stride % (dtype == SD_F32 ? 4 : 8)))) {
    sd::set_error("%s: rows must be 16-byte aligned", what);
    return SD_ERR_UNSUPPORTED;
  }
  const int64_t bytes = dtype == SD_F32 ? 4 : 2;
  const sd::Span o = sd::span_rows(out, rows, bytes * out_stride, bytes * columns);
  if (o.overlaps(sd::span_rows(codes, rows, codes_stride, columns)) || o.overlaps(sd::span_rows(scale, rows, 4, 4))) {
    sd::set_error("%s: out shares memory with an input", what);
    return SD_ERR_VALUE;
  }
  p.items = rows * p.spans;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>((p.items + 3) / 4)), block(256);
  if (dtype == SD_BF16) hipLaunchKernelGGL(rows_from_int8_kernel<__bf16>, grid, block, 0, st, p);
  else if (dtype == SD_F16) hipLaunchKernelGGL(rows_from_int8_kernel<_Float16>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(rows_from_int8_kernel<float>, grid, block, 0, st, p);
  return sd::check_launch(what);
}
