// int4_cache.hip — the 4-bit paged KV cache for gfx950: appending a step's keys and values
// (with the per-head RMSNorm and the rotation on the way, or as they are) and reading rows
// back in 16 bits.
//
// Row of one token and kv head (head_dim 128): 128 bytes of codes, the key's 64 first, and
// 4 NG scales of the activation type T (NG = 128 / G groups of G = 32, 64 or 128 dims):
// (scale, zero) of each key group, then of each value group.
//   lo = min x, hi = max x over the group;  zero = T(lo);  scale = T(max(hi - zero, 0) / 15)
//   code = clamp(round_half_even((x - zero) / scale), 0, 15)    (0 where scale is 0)
//   value = zero + scale * code
// Codes are taken against the rounded scale and zero, so a value is at most half a step from
// its own unless the rounded range falls short of hi. x is the fp32 value: a key is not rounded
// to T between its rotation and its code (its copy for the caller is). A group with a NaN or an
// infinity, or whose scale or zero leaves T's range, becomes NaN as a whole.
//
// The order of a row's half bytes is what the attention kernel's matrix operands read with
// whole-dword loads and no shuffles: key dword 4 g + i, nibble p holds dim 32 i + 8 g +
// 2 (p % 4) + p / 4; value dword r, nibble t holds dim 16 t + r.
//
// All three kernels are bound by bytes (a few operations an element): 16 lanes take one row of
// 128, four rows a wave. An appended key is loaded 16 bytes a lane (8 neighbouring dims, one code
// dword); a value in 2-byte loads of dims lr, 16 + lr, ..., which are one code dword as well.
#include <math.h>

#include "int4.h"

namespace {

using sd::u32x4;

constexpr int kD = 128;
constexpr int kThreads = 256;  // 16 rows of 16 lanes

struct Cache {
  uint8_t* codes;
  int64_t c_sblk, c_spos, c_shead;  // bytes
  uint16_t* scales;
  int64_t s_sblk, s_spos, s_shead;  // elements
  int64_t num_slots;
  int32_t block_size;
};

struct AppendParams {
  Cache c;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_stok, q_shead, k_stok, k_shead, v_stok, v_shead;
  uint16_t* qo;  // (T, Hq, 128) contiguous
  uint16_t* ko;  // (T, Hkv, 128) contiguous, or NULL
  const uint16_t* qw;
  const uint16_t* kw;
  float eps;
  const int64_t* pos;
  const float* cs;
  int64_t cs_stride, max_pos;
  const int32_t* slots;
  int64_t tokens;
  int32_t hq, hkv;
  int32_t units;  // 16-lane items per token
};

struct LoadParams {
  Cache c;
  const int32_t* slots;
  uint16_t* k;
  uint16_t* v;
  int64_t rows;
  int32_t hkv;
};

__device__ __forceinline__ bool slot_rows(const Cache& c, int32_t slot, int h, int64_t& code,
                                          int64_t& scale) {
  if (slot < 0 || slot >= c.num_slots) return false;
  const int blk = slot / c.block_size, off = slot - blk * c.block_size;
  code = blk * c.c_sblk + off * c.c_spos + h * c.c_shead;
  scale = blk * c.s_sblk + off * c.s_spos + h * c.s_shead;
  return true;
}

template <int CTRL> __device__ __forceinline__ float dpp_move(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                       0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
template <int CTRL> __device__ __forceinline__ double dpp_move64(double v) {
  const uint2 b = __builtin_bit_cast(uint2, v);
  return __builtin_bit_cast(
      double, make_uint2(__builtin_bit_cast(uint32_t, dpp_move<CTRL>(__uint_as_float(b.x))),
                         __builtin_bit_cast(uint32_t, dpp_move<CTRL>(__uint_as_float(b.y)))));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140, kRor8 = 0x128;

// Reduction over LANES = 4, 8 or 16 neighbouring lanes (aligned), the same in each of them.
template <int LANES, typename F> __device__ __forceinline__ float over(float v, F f) {
  v = f(v, dpp_move<kXor1>(v));
  v = f(v, dpp_move<kXor2>(v));
  if constexpr (LANES >= 8) v = f(v, dpp_move<kHalfMirror>(v));
  if constexpr (LANES >= 16) v = f(v, dpp_move<kMirror>(v));
  return v;
}

// Larger of two, NaN if either is (v_maximum3_f32).
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// What turns a group's values into codes: (x - z) f * inv = (x - z) / s.
struct Grid {
  float s, z, f, inv;
};
// From the minimum and the maximum (NaN if any value is): the grid, and its scale and zero as stored.
template <typename T> __device__ __forceinline__ Grid group_grid(float lo, float hi, uint32_t& sz) {
  Grid g;
  g.z = static_cast<float>(sd::round16<T>(lo));
  // (a NaN maximum: fmaxf would drop it)
  g.s = static_cast<float>(sd::round16<T>(max_nan(hi - g.z, 0.f) / 15.f));
  if (!(g.s * 0.f + g.z * 0.f == 0.f)) g.s = g.z = __builtin_nanf("");
  sz = sd::pack2<T>(g.s, g.z);
  // the reciprocal of a bf16 scale below 2^-126 would overflow: both sides times 2^64
  g.f = g.s < 0x1p-64f ? 0x1p64f : 1.f;
  g.inv = g.s > 0.f ? 1.f / (g.s * g.f) : 0.f;
  g.s *= g.f;
  return g;
}

// Code of a value. The quotient is the correctly rounded one (a product with the correctly rounded
// reciprocal and one correction from the exact remainder: P. Markstein, 1990): values exactly between two
// codes, which scales of 8 bits make common, stay exactly between them and go to the even one.
__device__ __forceinline__ uint32_t code_of(float x, const Grid& g) {
  const float t = (x - g.z) * g.f, q = t * g.inv;
  const float c = rintf(fmaf(fmaf(-q, g.s, t), g.inv, q));
  return static_cast<uint32_t>(__builtin_amdgcn_fmed3f(c, 0.f, 15.f));
}

template <typename T> __device__ __forceinline__ void widen(u32x4 a, float v[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = sd::from_bits<T>(static_cast<uint16_t>(a[e / 2] >> (16 * (e & 1))));
}
template <typename T> __device__ __forceinline__ void store8(uint16_t* p, const float v[8]) {
  sd::store16(p, u32x4{sd::pack2<T>(v[0], v[1]), sd::pack2<T>(v[2], v[3]),
                       sd::pack2<T>(v[4], v[5]), sd::pack2<T>(v[6], v[7])});
}

// Norm (weights w, if any) and rotation of a row: lane c holds dims 8 c .. 8 c + 7; dim d's partner d ^ 64
// is the same element of lane c ^ 8, and sinv carries the sign of its term.
template <typename T>
__device__ __forceinline__ void norm_rotate_query(u32x4 raw, float x[8], bool norm, const float w[8],
                                                  float eps, const float cosv[8], const float sinv[8],
                                                  bool turn) {
  widen<T>(raw, x);
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = sd::dot2<T>(raw[e], raw[e], ss);
    ss = over<16>(ss, [](float a, float b) { return a + b; });
    const float r = rsqrtf(ss / 128.f + eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * (r * w[e]);
  }
  if (turn) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(dpp_move<kRor8>(x[e]), sinv[e], x[e] * cosv[e]);
  }
}
// The same for a key, whose codes follow from values that may lie next to a border: the squares are
// summed in 64 bits and every product is rounded by itself, so that the norm adds no more than its
// formula's own roundings. (Queries in this form took append's 4001 tokens from 24.3 to 25.3 us.)
template <typename T>
__device__ __forceinline__ void norm_rotate_key(u32x4 raw, float x[8], bool norm, const float w[8],
                                                float eps, const float cosv[8], const float sinv[8],
                                                bool turn) {
#pragma clang fp contract(off)
  widen<T>(raw, x);
  if (norm) {
    double sq = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) sq += static_cast<double>(x[e]) * x[e];
    sq += dpp_move64<kXor1>(sq);
    sq += dpp_move64<kXor2>(sq);
    sq += dpp_move64<kHalfMirror>(sq);
    sq += dpp_move64<kMirror>(sq);
    const float r = rsqrtf(static_cast<float>(sq) / 128.f + eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
  }
  if (turn) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * cosv[e] + dpp_move<kRor8>(x[e]) * sinv[e];
  }
}

// Key row in registers (lane c: dims 8 c ..) -> codes and scales.
template <typename T, int NG>
__device__ __forceinline__ void write_key(const float x[8], uint8_t* codes, uint16_t* scales, int c) {
  constexpr int kLanes = 16 / NG;
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = fminf(lo, x[e]);
    hi = max_nan(hi, x[e]);
  }
  lo = over<kLanes>(lo, [](float a, float b) { return fminf(a, b); });
  hi = over<kLanes>(hi, max_nan);
  uint32_t sz, word = 0;
  const Grid g = group_grid<T>(lo, hi, sz);
#pragma unroll
  for (int e = 0; e < 8; ++e) word |= code_of(x[e], g) << (4 * (e / 2) + 16 * (e & 1));
  reinterpret_cast<uint32_t*>(codes)[4 * (c & 3) + (c >> 2)] = word;
  if (c % kLanes == 0) reinterpret_cast<uint32_t*>(scales)[c / kLanes] = sz;
}

// Value row (lane r: dims r, 16 + r, ..., 112 + r) -> codes and scales.
template <typename T, int NG>
__device__ __forceinline__ void write_value(const uint16_t* v, uint8_t* codes, uint16_t* scales, int r) {
  constexpr int kPer = 8 / NG;  // of a lane's dims in one group
  float x[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) x[t] = sd::from_bits<T>(v[16 * t + r]);
  uint32_t word = 0, mine = 0;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float lo = x[g * kPer], hi = lo;
#pragma unroll
    for (int t = g * kPer + 1; t < (g + 1) * kPer; ++t) {
      lo = fminf(lo, x[t]);
      hi = max_nan(hi, x[t]);
    }
    lo = over<16>(lo, [](float a, float b) { return fminf(a, b); });
    hi = over<16>(hi, max_nan);
    uint32_t sz;
    const Grid grid = group_grid<T>(lo, hi, sz);
    mine = r == g ? sz : mine;
#pragma unroll
    for (int t = g * kPer; t < (g + 1) * kPer; ++t) word |= code_of(x[t], grid) << (4 * t);
  }
  reinterpret_cast<uint32_t*>(codes + 64)[r] = word;
  if (r < NG) reinterpret_cast<uint32_t*>(scales)[NG + r] = mine;
}

// ROTATE: a token's query heads in items of QR (norm, rotation, copy out), then its kv heads, one an item;
// without, only the kv heads. An item's rows are loaded before the first is used, its token's cos and
// sin once.
template <typename T, int NG, bool ROTATE, int QR>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendParams p) {
  const int c = threadIdx.x & 15;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 4;
  const int64_t t = item / p.units;
  if (t >= p.tokens) return;
  const int u = static_cast<int>(item - t * p.units);
  const int q_items = p.units - p.hkv;
  float cosv[8], sinv[8], w[8];
  bool turn = false;
  u32x4 raw[QR];
  if (u < q_items) {
#pragma unroll
    for (int i = 0; i < QR; ++i)
      raw[i] = sd::load16(p.q + t * p.q_stok + min(QR * u + i, p.hq - 1) * p.q_shead + 8 * c);
  } else {
    raw[0] = sd::load16(p.k + t * p.k_stok + (u - q_items) * p.k_shead + 8 * c);
  }
  if constexpr (ROTATE) {
    const int64_t ps = p.pos[t];
    turn = ps >= 0 && ps < p.max_pos;
    const float* row = p.cs + (turn ? ps : 0) * p.cs_stride + 8 * (c & 7);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cosv[e] = row[e];
      sinv[e] = c < 8 ? -row[64 + e] : row[64 + e];
    }
    if (p.qw) widen<T>(sd::load16((u < q_items ? p.qw : p.kw) + 8 * c), w);
  }
  float x[8];
  if (u < q_items) {
    if constexpr (ROTATE) {
#pragma unroll
      for (int i = 0; i < QR; ++i) {
        const int r = QR * u + i;
        if (r >= p.hq) break;
        norm_rotate_query<T>(raw[i], x, p.qw, w, p.eps, cosv, sinv, turn);
        store8<T>(p.qo + (t * p.hq + r) * kD + 8 * c, x);
      }
    }
    return;
  }
  const int h = u - q_items;
  const int32_t slot = p.slots[t];
  if constexpr (!ROTATE) widen<T>(raw[0], x);
  if constexpr (ROTATE) {
    norm_rotate_key<T>(raw[0], x, p.kw, w, p.eps, cosv, sinv, turn);
    if (p.ko) store8<T>(p.ko + (t * p.hkv + h) * kD + 8 * c, x);
  }
  int64_t code, scale;
  if (!slot_rows(p.c, slot, h, code, scale)) return;
  write_value<T, NG>(p.v + t * p.v_stok + h * p.v_shead, p.c.codes + code, p.c.scales + scale, c);
  write_key<T, NG>(x, p.c.codes + code, p.c.scales + scale, c);
}

// Lane c of a row writes dims 8 c .. 8 c + 7 of its key and value.
template <typename T, int NG>
__global__ __launch_bounds__(kThreads) void load_kernel(LoadParams p) {
  const int c = threadIdx.x & 15;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 4;
  const int64_t i = item / p.hkv;
  if (i >= p.rows) return;
  const int h = static_cast<int>(item - i * p.hkv);
  float kv[8], vv[8];
  int64_t code, scale;
  if (slot_rows(p.c, p.slots[i], h, code, scale)) {
    const uint8_t* row = p.c.codes + code;
    const uint32_t* sc = reinterpret_cast<const uint32_t*>(p.c.scales + scale);
    const uint32_t kw = reinterpret_cast<const uint32_t*>(row)[4 * (c & 3) + (c >> 2)];
    const u32x4 v0 = sd::load16(row + 64 + 32 * (c & 1)), v1 = sd::load16(row + 80 + 32 * (c & 1));
    const int g = c * NG / 16;
    const uint32_t ks = sc[g], vs = sc[NG + g];
    const float k_s = sd::from_bits<T>(static_cast<uint16_t>(ks));
    const float k_z = sd::from_bits<T>(static_cast<uint16_t>(ks >> 16));
    const float v_s = sd::from_bits<T>(static_cast<uint16_t>(vs));
    const float v_z = sd::from_bits<T>(static_cast<uint16_t>(vs >> 16));
    const uint32_t vw[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      kv[e] = fmaf(static_cast<float>((kw >> (4 * (e / 2) + 16 * (e & 1))) & 15u), k_s, k_z);
      vv[e] = fmaf(static_cast<float>((vw[e] >> (4 * (c >> 1))) & 15u), v_s, v_z);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) kv[e] = vv[e] = 0.f;
  }
  const int64_t o = (i * p.hkv + h) * kD + 8 * c;
  store8<T>(p.k + o, kv);
  store8<T>(p.v + o, vv);
}

int set_cache(const char* what, Cache& c, void* codes, int64_t c_sblk, int64_t c_spos, int64_t c_shead,
              void* scales, int64_t s_sblk, int64_t s_spos, int64_t s_shead, int32_t group,
              int64_t num_blocks, int32_t block_size, int32_t hkv, int32_t head_dim, int32_t dtype) {
  if (hkv <= 0 || block_size <= 0 || num_blocks <= 0) {
    sd::set_error("%s: invalid sizes (heads=%d bs=%d blocks=%lld)", what, hkv, block_size,
                  (long long)num_blocks);
    return SD_ERR_VALUE;
  }
  if (head_dim != kD || (group != 32 && group != 64 && group != 128)) {
    sd::set_error("%s: head_dim 128 and groups of 32, 64 or 128 only, got %d and %d", what, head_dim,
                  group);
    return SD_ERR_UNSUPPORTED;
  }
  if (dtype != SD_BF16 && dtype != SD_F16) {
    sd::set_error("%s: dtype must be bf16 or f16", what);
    return SD_ERR_UNSUPPORTED;
  }
  if (hkv > (1 << 16) || block_size > (1 << 20) || num_blocks > (1ll << 31) - 1 ||
      num_blocks * block_size > (1ll << 31) - 1) {
    sd::set_error("%s: cache of %lld blocks x %d positions x %d heads too large", what,
                  (long long)num_blocks, block_size, hkv);
    return SD_ERR_UNSUPPORTED;
  }
  if (!sd::strides_ok({c_sblk, c_spos, c_shead, s_sblk, s_spos, s_shead})) {
    sd::set_error("%s: strides must lie in [-2^40, 2^40] elements", what);
    return SD_ERR_VALUE;
  }
  if (!codes || !scales) {
    sd::set_error("%s: null pointer argument", what);
    return SD_ERR_VALUE;
  }
  const int64_t unit = group == 128 ? 4 : 8;  // scales of a row, up to 16 bytes of them
  if (!sd::aligned16(codes) || reinterpret_cast<uintptr_t>(scales) % (2 * unit) || c_sblk % 16 ||
      c_spos % 16 || c_shead % 16 || s_sblk % unit || s_spos % unit || s_shead % unit) {
    sd::set_error("%s: code rows must be 16-byte aligned and scale rows aligned to %d bytes", what,
                  static_cast<int>(2 * unit));
    return SD_ERR_UNSUPPORTED;
  }
  c = Cache{static_cast<uint8_t*>(codes), c_sblk, c_spos, c_shead, static_cast<uint16_t*>(scales),
            s_sblk, s_spos, s_shead, num_blocks * block_size, block_size};
  return SD_OK;
}

template <typename T, bool ROTATE, int QR> void launch_append(AppendParams& p, int group, hipStream_t st) {
  p.units = p.hkv + (ROTATE ? (p.hq + QR - 1) / QR : 0);
  const int64_t items = p.tokens * p.units;
  const dim3 grid(static_cast<unsigned>((items + kThreads / 16 - 1) / (kThreads / 16)));
  if (group == 32)
    hipLaunchKernelGGL((append_kernel<T, 4, ROTATE, QR>), grid, dim3(kThreads), 0, st, p);
  else if (group == 64)
    hipLaunchKernelGGL((append_kernel<T, 2, ROTATE, QR>), grid, dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL((append_kernel<T, 1, ROTATE, QR>), grid, dim3(kThreads), 0, st, p);
}

// Query heads per 16-lane item: one while few tokens leave the device idle, then four, so that a token's
// cos and sin are loaded for four rows at a time.
template <typename T> void launch_rotate(AppendParams& p, int group, hipStream_t st) {
  if (p.tokens * (p.hq + p.hkv) > 16384) launch_append<T, true, 4>(p, group, st);
  else launch_append<T, true, 1>(p, group, st);
}

template <typename T> void launch_load(const LoadParams& p, int group, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((p.rows * p.hkv + kThreads / 16 - 1) / (kThreads / 16)));
  if (group == 32)
    hipLaunchKernelGGL((load_kernel<T, 4>), grid, dim3(kThreads), 0, st, p);
  else if (group == 64)
    hipLaunchKernelGGL((load_kernel<T, 2>), grid, dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL((load_kernel<T, 1>), grid, dim3(kThreads), 0, st, p);
}

constexpr int64_t kMaxRows = 1ll << 27;  // token rows x heads of one call (2^31 threads)

bool rows_aligned(const void* p, int64_t s_tok, int64_t s_head) {
  return sd::aligned16(p) && s_tok % 8 == 0 && s_head % 8 == 0;
}

}  // namespace

extern "C" int sd_store_kvcache_int4(const void* key, int64_t key_stride_tok, int64_t key_stride_head,
                                     const void* value, int64_t value_stride_tok,
                                     int64_t value_stride_head, void* codes,
                                     int64_t codes_stride_block, int64_t codes_stride_pos,
                                     int64_t codes_stride_head, void* scales,
                                     int64_t scales_stride_block, int64_t scales_stride_pos,
                                     int64_t scales_stride_head, int32_t group_size,
                                     const int32_t* slot_mapping, int64_t num_tokens,
                                     int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                     int64_t num_blocks, int32_t dtype, void* stream) {
  sd::clear_error();
  const char* what = "store_kvcache_int4";
  AppendParams p{};
  if (num_tokens < 0) {
    sd::set_error("%s: invalid sizes (tokens=%lld)", what, (long long)num_tokens);
    return SD_ERR_VALUE;
  }
  const int rc = set_cache(what, p.c, codes, codes_stride_block, codes_stride_pos, codes_stride_head,
                           scales, scales_stride_block, scales_stride_pos, scales_stride_head,
                           group_size, num_blocks, block_size, num_kv_heads, head_dim, dtype);
  if (rc != SD_OK) return rc;
  if (num_tokens == 0) return SD_OK;
  if (!key || !value || !slot_mapping) {
    sd::set_error("%s: null pointer argument", what);
    return SD_ERR_VALUE;
  }
  if (num_tokens > kMaxRows / num_kv_heads) {
    sd::set_error("%s: %lld tokens x %d heads too large", what, (long long)num_tokens, num_kv_heads);
    return SD_ERR_UNSUPPORTED;
  }
  if (!sd::strides_ok({key_stride_tok, key_stride_head, value_stride_tok, value_stride_head})) {
    sd::set_error("%s: strides must lie in [-2^40, 2^40] elements", what);
    return SD_ERR_VALUE;
  }
  if (!rows_aligned(key, key_stride_tok, key_stride_head) ||
      !rows_aligned(value, value_stride_tok, value_stride_head)) {
    sd::set_error("%s: key and value rows must be 16-byte aligned", what);
    return SD_ERR_UNSUPPORTED;
  }
  p.k = static_cast<const uint16_t*>(key);
  p.v = static_cast<const uint16_t*>(value);
  p.k_stok = key_stride_tok;
  p.k_shead = key_stride_head;
  p.v_stok = value_stride_tok;
  p.v_shead = value_stride_head;
  p.slots = slot_mapping;
  p.tokens = num_tokens;
  p.hkv = num_kv_heads;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SD_BF16) launch_append<__bf16, false, 1>(p, group_size, st);
  else launch_append<_Float16, false, 1>(p, group_size, st);
  return sd::check_launch(what);
}

extern "C" int sd_qk_norm_rope_store_int4(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k, int64_t k_stride_tok,
    int64_t k_stride_head, const void* v, int64_t v_stride_tok, int64_t v_stride_head,
    int64_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    const void* q_weight, const void* k_weight, float eps, const int64_t* positions,
    const float* cos_sin, int64_t cos_sin_stride, int64_t max_position, void* q_out, void* k_out,
    void* codes, int64_t codes_stride_block, int64_t codes_stride_pos, int64_t codes_stride_head,
    void* scales, int64_t scales_stride_block, int64_t scales_stride_pos, int64_t scales_stride_head,
    int32_t group_size, int64_t num_blocks, int32_t block_size, const int32_t* slot_mapping,
    int32_t dtype, void* stream) {
  sd::clear_error();
  const char* what = "qk_norm_rope_store_int4";
  AppendParams p{};
  if (num_tokens < 0 || num_q_heads <= 0 || max_position <= 0) {
    sd::set_error("%s: invalid sizes (tokens=%lld q heads=%d positions=%lld)", what,
                  (long long)num_tokens, num_q_heads, (long long)max_position);
    return SD_ERR_VALUE;
  }
  const int rc = set_cache(what, p.c, codes, codes_stride_block, codes_stride_pos, codes_stride_head,
                           scales, scales_stride_block, scales_stride_pos, scales_stride_head,
                           group_size, num_blocks, block_size, num_kv_heads, head_dim, dtype);
  if (rc != SD_OK) return rc;
  if (num_tokens == 0) return SD_OK;
  if (!q || !k || !v || !q_out || !positions || !cos_sin || !slot_mapping || (!q_weight != !k_weight)) {
    sd::set_error("%s: null pointer argument", what);
    return SD_ERR_VALUE;
  }
  if (num_q_heads > (1 << 16) || max_position > (1ll << 40) ||
      num_tokens > kMaxRows / (num_q_heads + num_kv_heads)) {
    sd::set_error("%s: %lld tokens x %d + %d heads too large", what, (long long)num_tokens, num_q_heads,
                  num_kv_heads);
    return SD_ERR_UNSUPPORTED;
  }
  if (!sd::strides_ok({q_stride_tok, q_stride_head, k_stride_tok, k_stride_head, v_stride_tok,
                       v_stride_head, cos_sin_stride}) ||
      cos_sin_stride < kD || cos_sin_stride > (1ll << 20)) {
    sd::set_error("%s: strides must lie in [-2^40, 2^40] elements, cos_sin's in [128, 2^20]", what);
    return SD_ERR_VALUE;
  }
  if (!rows_aligned(q, q_stride_tok, q_stride_head) || !rows_aligned(k, k_stride_tok, k_stride_head) ||
      !rows_aligned(v, v_stride_tok, v_stride_head) || !sd::aligned16(q_out) || !sd::aligned16(k_out) ||
      !sd::aligned16(q_weight) || !sd::aligned16(k_weight) || !sd::aligned16(cos_sin) ||
      cos_sin_stride % 4 != 0) {
    sd::set_error("%s: q, k, v, weight and cos_sin rows must be 16-byte aligned", what);
    return SD_ERR_UNSUPPORTED;
  }
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q_stok = q_stride_tok;
  p.q_shead = q_stride_head;
  p.k_stok = k_stride_tok;
  p.k_shead = k_stride_head;
  p.v_stok = v_stride_tok;
  p.v_shead = v_stride_head;
  p.qo = static_cast<uint16_t*>(q_out);
  p.ko = static_cast<uint16_t*>(k_out);
  p.qw = static_cast<const uint16_t*>(q_weight);
  p.kw = static_cast<const uint16_t*>(k_weight);
  p.eps = eps;
  p.pos = positions;
  p.cs = cos_sin;
  p.cs_stride = cos_sin_stride;
  p.max_pos = max_position;
  p.slots = slot_mapping;
  p.tokens = num_tokens;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SD_BF16) launch_rotate<__bf16>(p, group_size, st);
  else launch_rotate<_Float16>(p, group_size, st);
  return sd::check_launch(what);
}

extern "C" int sd_load_kvcache_int4(const void* codes, int64_t codes_stride_block,
                                    int64_t codes_stride_pos, int64_t codes_stride_head,
                                    const void* scales, int64_t scales_stride_block,
                                    int64_t scales_stride_pos, int64_t scales_stride_head,
                                    int32_t group_size, const int32_t* slot_mapping, int64_t num_rows,
                                    int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                    int64_t num_blocks, int32_t dtype, void* key, void* value,
                                    void* stream) {
  sd::clear_error();
  const char* what = "load_kvcache_int4";
  LoadParams p{};
  if (num_rows < 0) {
    sd::set_error("%s: invalid sizes (rows=%lld)", what, (long long)num_rows);
    return SD_ERR_VALUE;
  }
  const int rc = set_cache(what, p.c, const_cast<void*>(codes), codes_stride_block, codes_stride_pos,
                           codes_stride_head, const_cast<void*>(scales), scales_stride_block,
                           scales_stride_pos, scales_stride_head, group_size, num_blocks, block_size,
                           num_kv_heads, head_dim, dtype);
  if (rc != SD_OK) return rc;
  if (num_rows == 0) return SD_OK;
  if (!slot_mapping || !key || !value) {
    sd::set_error("%s: null pointer argument", what);
    return SD_ERR_VALUE;
  }
  if (num_rows > kMaxRows / num_kv_heads) {
    sd::set_error("%s: %lld rows x %d heads too large", what, (long long)num_rows, num_kv_heads);
    return SD_ERR_UNSUPPORTED;
  }
  if (!sd::aligned16(key) || !sd::aligned16(value)) {
    sd::set_error("%s: key and value must be 16-byte aligned", what);
    return SD_ERR_UNSUPPORTED;
  }
  p.slots = slot_mapping;
  p.k = static_cast<uint16_t*>(key);
  p.v = static_cast<uint16_t*>(value);
  p.rows = num_rows;
  p.hkv = num_kv_heads;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SD_BF16) launch_load<__bf16>(p, group_size, st);
  else launch_load<_Float16>(p, group_size, st);
  return sd::check_launch(what);
}
