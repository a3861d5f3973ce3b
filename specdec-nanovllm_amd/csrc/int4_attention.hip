// int4_attention.hip — paged decode / speculative-verify attention over the 4-bit KV cache
// (the row format of int4_cache.hip) for gfx950.
//
// Per sequence b, kv head h, query row r = qi * Gq + g (Gq = Hq / Hkv):
//   o[r] = softmax_j(scale q[r] . K[j]) V,  j in [0, L_b - n_b + qi]
// with K[j][d] = z + s c, V[j][d] = z' + s' c' per group of dims. The codes go to the matrix cores
// as 16 + c (int4.h), and scales and zeros never touch an element:
//   q . K[j] = sum_g s_jg (q_g . (16 + c)_g) + (z_jg - 16 s_jg) sum(q_g)
//   O[d in g] = sum_j (p_j s'_jg) (16 + c')_jd + sum_j p_j (z'_jg - 16 s'_jg)
// One MFMA 16x16x32 covers 32 dims of 16 keys, so a group's product is one to four of them; the
// per-key scales meet the 16-lane score tile (4 keys a lane), and p s' is split into two bf16
// parts (hi + lo, 2^-17 relative), since a single rounding would double the output's error.
//
// Work: a pair is one (sequence, kv head), a chunk 128 keys of one pair: 32 for each of the 4 waves
// of a workgroup. All chunks, laid end to end, are cut into equal runs, one a workgroup, whatever
// the length mix (context lengths are read on the device). When a pair or the run ends, the waves
// merge their softmax states in LDS; a pair that several runs share leaves partials in the workspace
// (two slots a run: the pair it starts in, the pair it ends in), which the combine kernel merges.
// Where the table admits few chunks a pair, a run is one whole pair and there is no second launch.
//
// Bound by the bytes of the cache: 128 + 8 NG per key and kv head. A wave keeps kAhead steps of
// loads in flight in registers (18 dwords a step at NG = 2).
#include <math.h>

#include "int4.h"

namespace {

using sd::f32x4;
using sd::u32x4;

constexpr int kD = 128;
constexpr int kWaves = 4;
constexpr int kStep = 32;               // keys of a wave's step
constexpr int kChunk = kWaves * kStep;  // keys of a workgroup's step
constexpr int kPitch = kD + 4;          // floats of a row's state in LDS: acc, then m and l
constexpr int kWholeChunks = 4;         // up to this many chunks a pair: no splitting of pairs

struct Params {
  const uint16_t* q;
  int64_t q_stok, q_shead;
  const uint8_t* codes;
  int64_t c_sblk, c_shead;  // bytes
  uint32_t c_spos;          // bytes
  const uint8_t* scales;
  int64_t s_sblk, s_shead;  // bytes
  uint32_t s_spos;          // bytes
  int32_t num_blocks, block_size;
  int32_t bs_shift;  // log2(block_size), -1 where it is no power of two
  int32_t max_ctx;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* ctx;
  const int32_t* cu_k;
  const int32_t* cu_q;
  int32_t max_qlen;
  int64_t total_q;
  int32_t num_seqs, gq, hkv;
  float scale_log2;
  uint16_t* out;
  int64_t o_stok, o_shead;
  float* ws;      // [2 runs][rmax][kPitch]
  int32_t runs;   // workgroups of the main kernel
  int32_t whole;  // a run is one whole pair
  int32_t rmax;
};

__device__ __forceinline__ int seq_keys(const Params& p, int b) {
  const int L = p.ctx ? p.ctx[b] : p.cu_k[b + 1] - p.cu_k[b];
  return min(max(L, 0), p.max_ctx);
}
__device__ __forceinline__ int seq_keys_uniform(const Params& p, int b) {
  const int L = p.ctx ? sd::load_scalar_i32(p.ctx + b)
                      : sd::load_scalar_i32(p.cu_k + b + 1) - sd::load_scalar_i32(p.cu_k + b);
  return min(max(L, 0), p.max_ctx);
}
__device__ __forceinline__ int chunks_of(int L) { return (L + kChunk - 1) / kChunk; }

// Chunks (of one head) of all sequences before `upto`, by a whole wave.
__device__ int chunks_before(const Params& p, int upto) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
  for (int c = lane; c < upto; c += 64) sum += chunks_of(seq_keys(p, c));
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
  return __builtin_amdgcn_readfirstlane(sum);
}

// The sequence that holds chunk s of the layout (b major, then head, then chunk), and the chunks of
// one head before it. s < hkv * all chunks.
__device__ void locate(const Params& p, int s, int& b, int& before) {
  const int lane = threadIdx.x & 63;
  int run = 0;
  for (int c = 0; c < p.num_seqs; c += 64) {
    const int n = c + lane < p.num_seqs ? chunks_of(seq_keys(p, c + lane)) : 0;
    const int incl = sd::wave_inclusive_sum(n);
    const int excl = run + incl - n;
    const unsigned long long hit =
        __ballot(n > 0 && excl * p.hkv <= s && s < (excl + n) * p.hkv);
    if (hit) {
      const int src = __ffsll(hit) - 1;
      b = c + src;
      before = __builtin_amdgcn_readlane(excl, src);
      return;
    }
    run += __builtin_amdgcn_readlane(incl, 63);
  }
  b = p.num_seqs - 1;
  before = run;
}

struct Rows {
  int64_t q0;
  int nq;
};
__device__ __forceinline__ Rows seq_rows(const Params& p, int b) {
  if (!p.cu_q) return Rows{b, 1};
  const int a = sd::load_scalar_i32(p.cu_q + b), e = sd::load_scalar_i32(p.cu_q + b + 1);
  return Rows{a, min(max(e - a, 0), p.max_qlen)};
}

template <typename T>
__device__ __forceinline__ void store_row4(const Params& p, const Rows& sr, int h, int row, int c,
                                           f32x4 v) {
  const int qi = row / p.gq, g = row - qi * p.gq;
  const int64_t qt = sr.q0 + qi;
  if (qt < 0 || qt >= p.total_q) return;
  uint2 w;
  w.x = sd::pack2<T>(v.x, v.y);
  w.y = sd::pack2<T>(v.z, v.w);
  *reinterpret_cast<uint2*>(p.out + qt * p.o_stok + static_cast<int64_t>(h * p.gq + g) * p.o_shead + 4 * c) = w;
}

// Position in the layout: chunk j of the n chunks of pair (b, h), whose sequence has L keys.
struct Pos {
  int b, h, j, n, L;
};
__device__ __forceinline__ void next_pair(const Params& p, Pos& a) {
  a.j = 0;
  if (a.h + 1 < p.hkv) {
    ++a.h;
    return;
  }
  a.h = 0;
  do {
    if (++a.b >= p.num_seqs) {
      a.n = 0;
      return;
    }
    a.L = seq_keys_uniform(p, a.b);
    a.n = chunks_of(a.L);
  } while (a.n == 0);
}

// One wave's step as loaded: lane (lr, lg) holds the key half bytes 32 lg .. 32 lg + 31 of keys lr
// and 16 + lr, dword lr of the values of keys 4 lg + j and 16 + 4 lg + j, and of key lane / 2 the
// scales of its keys (even lanes) or values.
template <int NG> struct Step {
  u32x4 k[2];
  uint32_t v[8];
  uint32_t s[NG];
};

template <typename T, int NG, int RT, bool ONE_PAGE>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(RT == 1 ? 2 : 1)))
void int4_attn_main(Params p) {
  constexpr int kAhead = 3;
  constexpr int kRow = 4 * NG;  // floats of a key's scales in LDS
  __shared__ __attribute__((aligned(16))) float lds_s[kWaves][kStep][kRow];
  __shared__ __attribute__((aligned(16))) float lds_m[kWaves][RT * 16][kPitch];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;

  // ---- this run's chunks [s0, s1) and where they begin
  Pos cur;
  int left;
  bool entered = false;  // the current pair began in an earlier run
  const int run = blockIdx.x;
  if (p.whole) {
    cur.b = run / p.hkv;
    cur.h = run - cur.b * p.hkv;
    cur.j = 0;
    cur.L = seq_keys_uniform(p, cur.b);
    cur.n = left = chunks_of(cur.L);
    if (left == 0) {
      const Rows sr = seq_rows(p, cur.b);
      for (int i = tid; i < p.gq * sr.nq * 32; i += kWaves * 64)
        store_row4<T>(p, sr, cur.h, i / 32, i % 32, f32x4{0.f, 0.f, 0.f, 0.f});
      return;
    }
  } else {
    const int total = chunks_before(p, p.num_seqs) * p.hkv;
    const int S = (total + p.runs - 1) / p.runs;
    const int s0 = run * S;
    if (s0 >= total) return;
    left = min(S, total - s0);
    int before = 0;
    locate(p, s0, cur.b, before);
    cur.b = __builtin_amdgcn_readfirstlane(cur.b);
    cur.L = seq_keys_uniform(p, cur.b);
    cur.n = chunks_of(cur.L);
    const int in = s0 - before * p.hkv;
    cur.h = in / cur.n;
    cur.j = in - cur.h * cur.n;
    entered = cur.j > 0;
  }
  Pos ahead = cur;  // what load_step loads next
  int ahead_left = left;
  bool first_pair = true;

  auto page_base = [&](int b, int tok) {
    int pg = p.bs_shift >= 0 ? tok >> p.bs_shift : tok / p.block_size;
    int blk = p.bt[b * p.bt_stride + pg];
    return min(max(blk, 0), p.num_blocks - 1);
  };
  auto in_page = [&](int tok) {
    return p.bs_shift >= 0 ? tok & (p.block_size - 1) : tok % p.block_size;
  };
  // Loads the next step (the same loads whatever the lengths: positions past the end read the last
  // key, past the run the last chunk again) and moves on.
  auto load_step = [&](Step<NG>& st) {
    const int last = ahead.L - 1;
    const int t0 = min(ahead.j * kChunk + wave * kStep, last);
    const int64_t hc = ahead.h * p.c_shead, hs = ahead.h * p.s_shead;
    const int kv = min(t0 + (lane >> 1), last);  // the key whose scales this lane loads
    if constexpr (ONE_PAGE) {
      int pg = p.bs_shift >= 0 ? t0 >> p.bs_shift : t0 / p.block_size;
      int blk = sd::load_scalar_i32(p.bt + ahead.b * p.bt_stride + pg);
      blk = min(max(blk, 0), p.num_blocks - 1);
      const int off = in_page(t0);
      const uint8_t* cp = p.codes + blk * p.c_sblk + hc + static_cast<int64_t>(off) * p.c_spos;
      const uint8_t* sp = p.scales + blk * p.s_sblk + hs + static_cast<int64_t>(off) * p.s_spos;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
        st.k[tt] = sd::load16_stream(cp + static_cast<uint32_t>(min(t0 + 16 * tt + lr, last) - t0) * p.c_spos + 16 * lg);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tok = min(t0 + (j < 4 ? 4 * lg + j : 12 + 4 * lg + j), last);
        st.v[j] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(
            cp + static_cast<uint32_t>(tok - t0) * p.c_spos + 64 + 4 * lr));
      }
      const uint32_t* s32 = reinterpret_cast<const uint32_t*>(
          sp + static_cast<uint32_t>(kv - t0) * p.s_spos) + NG * (lane & 1);
#pragma unroll
      for (int g = 0; g < NG; ++g) st.s[g] = s32[g];
    } else {
      auto code_row = [&](int tok) {
        return p.codes + page_base(ahead.b, tok) * p.c_sblk + hc + static_cast<int64_t>(in_page(tok)) * p.c_spos;
      };
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
        st.k[tt] = sd::load16_stream(code_row(min(t0 + 16 * tt + lr, last)) + 16 * lg);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tok = min(t0 + (j < 4 ? 4 * lg + j : 12 + 4 * lg + j), last);
        st.v[j] = *reinterpret_cast<const uint32_t*>(code_row(tok) + 64 + 4 * lr);
      }
      const uint32_t* s32 = reinterpret_cast<const uint32_t*>(
          p.scales + page_base(ahead.b, kv) * p.s_sblk + hs + static_cast<int64_t>(in_page(kv)) * p.s_spos) + NG * (lane & 1);
#pragma unroll
      for (int g = 0; g < NG; ++g) st.s[g] = s32[g];
    }
    if (ahead_left > 1) {
      --ahead_left;
      if (++ahead.j == ahead.n) next_pair(p, ahead);
    }
  };

  // ---- state of the current pair
  u32x4 qop[RT][4];
  float qsum[RT][NG];
  int lim[RT], causal = 0;
  float m_run[RT], l_run[RT], zsum[RT][NG];
  f32x4 acc[RT][8];
  Rows sr{0, 0};

  auto begin_pair = [&]() {
    sr = seq_rows(p, cur.b);
    causal = cur.L - sr.nq;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = rt * 16 + lr;
      const int qi = row / p.gq, g = row - qi * p.gq;
      const int64_t qt = sr.q0 + qi;
      const bool valid = qi < sr.nq && qt >= 0 && qt < p.total_q;
      lim[rt] = valid ? min(causal + qi, cur.L - 1) : -1;
      const uint16_t* qp = p.q + (valid ? qt * p.q_stok + static_cast<int64_t>(cur.h * p.gq + g) * p.q_shead : 0) + 8 * lg;
      float part[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qop[rt][i] = valid ? sd::load16(qp + 32 * i) : u32x4{0u, 0u, 0u, 0u};
        const uint32_t w[4] = {qop[rt][i].x, qop[rt][i].y, qop[rt][i].z, qop[rt][i].w};
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s += sd::from_bits<T>(static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1))));
        part[i] = s;
      }
#pragma unroll
      for (int g2 = 0; g2 < NG; ++g2) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i * NG / 4 == g2) s += part[i];
        qsum[rt][g2] = sd::sum_over_groups(s);
        zsum[rt][g2] = 0.f;
      }
      m_run[rt] = -INFINITY;
      l_run[rt] = 0.f;
#pragma unroll
      for (int t = 0; t < 8; ++t) acc[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };

  auto compute_step = [&](const Step<NG>& st) {
    const int tb = cur.j * kChunk + wave * kStep;
    if (tb >= cur.L) return;  // wave-uniform
    // ---- scales to LDS in fp32: key (s c, (z - 16 s) c) with c = softmax scale * log2(e), value
      //    (s, z - 16 s); lane 2 k (2 k + 1) holds key k's key (value) scales
    {
      float* d = &lds_s[wave][lane >> 1][2 * NG * (lane & 1)];
      const float f = lane & 1 ? 1.f : p.scale_log2;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float s = sd::from_bits<T>(static_cast<uint16_t>(st.s[g]));
        const float z = sd::from_bits<T>(static_cast<uint16_t>(st.s[g] >> 16));
        d[g] = s * f;
        d[NG + g] = (z - 16.f * s) * f;
      }
    }
    sd::wave_lds_sync();
    // ---- scores (log2 units): lane holds key tb + 16 tt + 4 lg + i of row lr
    float sc[RT][8];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      u32x4 ka[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ka[i] = sd::unpack8<T>(st.k[tt][i]);
      f32x4 dot[RT][NG];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i * NG / 4 == g) c = sd::Elem<T>::mfma(ka[i], qop[rt][i], c);
          dot[rt][g] = c;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* ks = lds_s[wave][16 * tt + 4 * lg + i];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float s = 0.f;
#pragma unroll
          for (int g = 0; g < NG; ++g) s = fmaf(ks[g], dot[rt][g][i], fmaf(ks[NG + g], qsum[rt][g], s));
          sc[rt][4 * tt + i] = s;
        }
      }
    }
    const bool full = tb + kStep - 1 <= min(causal, cur.L - 1);
    if (!full) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int tok = tb + (e < 4 ? 4 * lg + e : 12 + 4 * lg + e);
          sc[rt][e] = tok <= lim[rt] ? sc[rt][e] : -INFINITY;
        }
    }
    // ---- online softmax; the running maximum moves only when a score exceeds it by more than 8
    //      (log2 units): p <= 2^8 otherwise, well inside fp32 and the bf16 parts
    u32x4 hi[RT][NG], lo[RT][NG];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float mloc = sc[rt][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mloc = fmaxf(mloc, sc[rt][e]);
      if (__any(mloc > m_run[rt] + 8.f)) {
        const float mnew = fmaxf(m_run[rt], sd::max_over_groups(mloc));
        const float alpha = sd::fast_exp2(m_run[rt] - (mnew == -INFINITY ? 0.f : mnew));
        l_run[rt] *= alpha;
#pragma unroll
        for (int g = 0; g < NG; ++g) zsum[rt][g] *= alpha;
#pragma unroll
        for (int t = 0; t < 8; ++t) acc[rt][t] *= alpha;
        m_run[rt] = mnew;
      }
      const float mb = m_run[rt] == -INFINITY ? 0.f : m_run[rt];
      float pv[8], ps[NG][8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pv[e] = sd::fast_exp2(sc[rt][e] - mb);
        l_run[rt] += pv[e];
        const float* vs = &lds_s[wave][e < 4 ? 4 * lg + e : 12 + 4 * lg + e][2 * NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float s = vs[g], z = vs[NG + g];
          if (!full) {  // a key that this row does not see may hold anything
            const bool seen = tb + (e < 4 ? 4 * lg + e : 12 + 4 * lg + e) <= lim[rt];
            s = seen ? s : 0.f;
            z = seen ? z : 0.f;
          }
          ps[g][e] = pv[e] * s;
          zsum[rt][g] = fmaf(pv[e], z, zsum[rt][g]);
        }
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) sd::split_pack<__bf16>(ps[g][2 * e], ps[g][2 * e + 1], h[e], l[e]);
        hi[rt][g] = u32x4{h[0], h[1], h[2], h[3]};
        lo[rt][g] = u32x4{l[0], l[1], l[2], l[3]};
      }
    }
    // ---- O^T += V^T P^T: byte b of the 8 value dwords holds tiles 2 b (low half) and 2 b + 1
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      uint32_t even[4], odd[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // byte b of keys 2 e and 2 e + 1, each in the low byte of a half
        const uint32_t z = __builtin_amdgcn_perm(st.v[2 * e + 1], st.v[2 * e],
                                                 0x0c040c00u + 0x00010001u * b);
        even[e] = sd::code_pair<__bf16, 0>(z);
        odd[e] = sd::code_pair<__bf16, 4>(z);
      }
      const u32x4 va = {even[0], even[1], even[2], even[3]}, vb = {odd[0], odd[1], odd[2], odd[3]};
      const int g = b * NG / 4;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        acc[rt][2 * b] = sd::Elem<__bf16>::mfma(va, hi[rt][g], acc[rt][2 * b]);
        acc[rt][2 * b + 1] = sd::Elem<__bf16>::mfma(vb, hi[rt][g], acc[rt][2 * b + 1]);
        acc[rt][2 * b] = sd::Elem<__bf16>::mfma(va, lo[rt][g], acc[rt][2 * b]);
        acc[rt][2 * b + 1] = sd::Elem<__bf16>::mfma(vb, lo[rt][g], acc[rt][2 * b + 1]);
      }
    }
    sd::wave_lds_sync();  // every lane has read the scales before the next step writes its own
  };

  // Merges the waves' states of the current pair: rows of out where this run saw the whole pair, a
  // partial otherwise. Every wave comes here.
  auto flush = [&](bool whole_pair) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = rt * 16 + lr;
      const float l = sd::sum_over_groups(l_run[rt]);
      float* d = lds_m[wave][row];
#pragma unroll
      for (int g = 0; g < NG; ++g) zsum[rt][g] = sd::sum_over_groups(zsum[rt][g]);
#pragma unroll
      for (int t = 0; t < 8; ++t)
        sd::store16(d + 16 * t + 4 * lg, __builtin_bit_cast(u32x4, acc[rt][t] + zsum[rt][t * NG / 8]));
      if (lg == 0) {
        d[kD] = m_run[rt];
        d[kD + 1] = l;
      }
    }
    __syncthreads();
    const int rows = p.gq * sr.nq;
    float* slot = p.ws + (2 * static_cast<int64_t>(run) + (first_pair ? 0 : 1)) * p.rmax * kPitch;
    for (int i = tid; i < rows * 32; i += kWaves * 64) {
      const int row = i >> 5, c = i & 31;
      float M = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) M = fmaxf(M, lds_m[w][row][kD]);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float m = lds_m[w][row][kD];
        // no finite score: l is 0 (nothing seen), or NaN, which stays
        const float f = m == -INFINITY ? lds_m[w][row][kD + 1] : exp2f(m - M);
        l = fmaf(f, lds_m[w][row][kD + 1], l);
        o += f * __builtin_bit_cast(f32x4, sd::load16(&lds_m[w][row][4 * c]));
      }
      if (whole_pair) {
        // l is 0 only for a row that sees no key (NaN stays NaN)
        const float inv = l == 0.f ? 0.f : 1.f / l;
        store_row4<T>(p, sr, cur.h, row, c, o * inv);
      } else {
        float* d = slot + row * kPitch;
        sd::store16(d + 4 * c, __builtin_bit_cast(u32x4, o));
        if (c == 0) {
          d[kD] = M;
          d[kD + 1] = l;
        }
      }
    }
    __syncthreads();
  };

  Step<NG> ring[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load_step(ring[i]);
  begin_pair();
  while (true) {
    bool done = false;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      compute_step(ring[i]);
      load_step(ring[i]);
      ++cur.j;
      --left;
      const bool ends = cur.j == cur.n;
      if (ends || left == 0) {
        flush(ends && !entered);
        if (left == 0) {
          done = true;
          break;
        }
        entered = first_pair = false;
        next_pair(p, cur);
        begin_pair();
      }
    }
    if (done) break;
  }
}

// One workgroup a pair: rows of pairs that several runs share from their partials, zeros for
// sequences without keys; a pair that one run saw whole is written already.
template <typename T> __global__ __launch_bounds__(256) void int4_attn_combine(Params p) {
  const int b = blockIdx.x / p.hkv, h = blockIdx.x - b * p.hkv;
  const int n = chunks_of(seq_keys_uniform(p, b));
  const Rows sr = seq_rows(p, b);
  const int rows = p.gq * sr.nq;
  if (n == 0) {
    for (int i = threadIdx.x; i < rows * 32; i += 256)
      store_row4<T>(p, sr, h, i >> 5, i & 31, f32x4{0.f, 0.f, 0.f, 0.f});
    return;
  }
  const int S = (chunks_before(p, p.num_seqs) * p.hkv + p.runs - 1) / p.runs;
  const int first = chunks_before(p, b) * p.hkv + h * n;
  const int r0 = first / S, r1 = (first + n - 1) / S;
  if (r0 == r1) return;
  for (int i = threadIdx.x; i < rows * 32; i += 256) {
    const int row = i >> 5, c = i & 31;
    auto state = [&](int r) {
      return p.ws + ((2 * static_cast<int64_t>(r) + (first > r * S ? 1 : 0)) * p.rmax + row) * kPitch;
    };
    float M = -INFINITY, l = 0.f;
    for (int r = r0; r <= r1; ++r) M = fmaxf(M, state(r)[kD]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int r = r0; r <= r1; ++r) {
      const float* s = state(r);
      const float f = s[kD] == -INFINITY ? s[kD + 1] : exp2f(s[kD] - M);
      l = fmaf(f, s[kD + 1], l);
      o += f * __builtin_bit_cast(f32x4, sd::load16(s + 4 * c));
    }
    store_row4<T>(p, sr, h, row, c, o * (l == 0.f ? 0.f : 1.f / l));
  }
}

struct Plan {
  int64_t runs;
  bool whole;
  int rmax, RT;
};

Plan make_plan(int num_seqs, int max_qlen, int hq, int hkv, int64_t max_ctx, int num_splits) {
  Plan pl;
  pl.rmax = hq / hkv * max_qlen;
  pl.RT = pl.rmax <= 16 ? 1 : 2;
  const int64_t pairs = static_cast<int64_t>(num_seqs) * hkv;
  const int64_t most = (max_ctx + kChunk - 1) / kChunk;  // chunks of a pair
  pl.whole = num_splits == 0 && most <= kWholeChunks;
  if (pl.whole) {
    pl.runs = pairs;
  } else {
    // one resident set of workgroups: 4 waves each, RT == 1 two workgroups a compute unit
    pl.runs = num_splits > 0 ? pairs * num_splits : static_cast<int64_t>(sd::device_cus()) * (pl.RT == 1 ? 2 : 1);
    if (pl.runs > pairs * most) pl.runs = pairs * most;
  }
  return pl;
}

bool plan_fits(int num_seqs, int hkv, int64_t max_ctx, int num_splits) {
  const int64_t pairs = static_cast<int64_t>(num_seqs) * hkv;
  return max_ctx <= (1ll << 30) && pairs <= (1ll << 23) && num_splits <= (1 << 16) &&
         pairs * ((max_ctx + kChunk - 1) / kChunk) <= (1ll << 30) &&
         (num_splits == 0 || pairs * num_splits <= (1ll << 22));
}

size_t ws_bytes(const Plan& pl) {
  return pl.whole ? 0 : static_cast<size_t>(2 * pl.runs) * pl.rmax * kPitch * sizeof(float);
}

template <typename T, int NG, int RT> void launch_main(const Params& p, hipStream_t st) {
  if (p.block_size % kStep == 0)
    hipLaunchKernelGGL((int4_attn_main<T, NG, RT, true>), dim3(p.runs), dim3(kWaves * 64), 0, st, p);
  else
    hipLaunchKernelGGL((int4_attn_main<T, NG, RT, false>), dim3(p.runs), dim3(kWaves * 64), 0, st, p);
}

template <typename T> int launch(const Params& p, const Plan& pl, int group, hipStream_t st) {
  if (pl.RT == 1) {
    if (group == 32) launch_main<T, 4, 1>(p, st);
    else if (group == 64) launch_main<T, 2, 1>(p, st);
    else launch_main<T, 1, 1>(p, st);
  } else {
    if (group == 32) launch_main<T, 4, 2>(p, st);
    else if (group == 64) launch_main<T, 2, 2>(p, st);
    else launch_main<T, 1, 2>(p, st);
  }
  const int rc = sd::check_launch("paged_attention_int4 main");
  if (rc != SD_OK || pl.whole) return rc;
  hipLaunchKernelGGL((int4_attn_combine<T>), dim3(p.num_seqs * p.hkv), dim3(256), 0, st, p);
  return sd::check_launch("paged_attention_int4 combine");
}

}  // namespace

extern "C" size_t sd_paged_attention_int4_workspace_size(int32_t num_seqs, int32_t max_qlen,
                                                         int32_t num_q_heads, int32_t num_kv_heads,
                                                         int64_t max_ctx, int32_t num_splits) {
  if (num_seqs <= 0 || max_qlen <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || max_ctx <= 0 ||
      num_splits < 0 || num_q_heads % num_kv_heads != 0)
    return 0;
  if (static_cast<int64_t>(num_q_heads) / num_kv_heads * max_qlen > 32 ||
      !plan_fits(num_seqs, num_kv_heads, max_ctx, num_splits))
    return SIZE_MAX;
  return ws_bytes(make_plan(num_seqs, max_qlen, num_q_heads, num_kv_heads, max_ctx, num_splits));
}

extern "C" int sd_paged_attention_int4(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* codes,
    int64_t codes_stride_block, int64_t codes_stride_pos, int64_t codes_stride_head, const void* scales,
    int64_t scales_stride_block, int64_t scales_stride_pos, int64_t scales_stride_head,
    int32_t group_size, int64_t num_blocks, int32_t block_size, const int32_t* block_table,
    int64_t bt_stride, int32_t max_blocks_per_seq, const int32_t* context_lens,
    const int32_t* cu_seqlens_k, const int32_t* cu_seqlens_q, int32_t max_qlen, int64_t total_q,
    int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float scale,
    int32_t dtype, void* out, int64_t out_stride_tok, int64_t out_stride_head, void* workspace,
    size_t workspace_bytes, int32_t num_splits, void* stream) {
  sd::clear_error();
  const char* what = "paged_attention_int4";
  if (num_seqs < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || block_size <= 0 || num_blocks <= 0 ||
      max_blocks_per_seq <= 0 || max_qlen <= 0 || total_q < 0 || num_splits < 0) {
    sd::set_error("%s: invalid sizes (seqs=%d hq=%d hkv=%d bs=%d blocks=%lld maxblk=%d max_qlen=%d "
                  "total_q=%lld splits=%d)",
                  what, num_seqs, num_q_heads, num_kv_heads, block_size, (long long)num_blocks,
                  max_blocks_per_seq, max_qlen, (long long)total_q, num_splits);
    return SD_ERR_VALUE;
  }
  if (num_q_heads % num_kv_heads != 0) {
    sd::set_error("%s: GQA needs num_q_heads %% num_kv_heads == 0 (%d vs %d)", what, num_q_heads,
                  num_kv_heads);
    return SD_ERR_VALUE;
  }
  if (head_dim != kD || (group_size != 32 && group_size != 64 && group_size != 128)) {
    sd::set_error("%s: head_dim 128 and groups of 32, 64 or 128 only, got %d and %d", what, head_dim,
                  group_size);
    return SD_ERR_UNSUPPORTED;
  }
  if (dtype != SD_BF16 && dtype != SD_F16) {
    sd::set_error("%s: dtype must be bf16 or f16", what);
    return SD_ERR_UNSUPPORTED;
  }
  if (static_cast<int64_t>(num_q_heads) / num_kv_heads * max_qlen > 32) {
    sd::set_error("%s: (num_q_heads / num_kv_heads) * max_qlen = %lld exceeds 32", what,
                  (long long)num_q_heads / num_kv_heads * max_qlen);
    return SD_ERR_UNSUPPORTED;
  }
  if (!cu_seqlens_q && max_qlen != 1) {
    sd::set_error("%s: max_qlen must be 1 without cu_seqlens_q", what);
    return SD_ERR_VALUE;
  }
  if (num_seqs == 0 || total_q == 0) return SD_OK;
  if (!q || !codes || !scales || !block_table || !out || (!context_lens && !cu_seqlens_k)) {
    sd::set_error("%s: null pointer argument", what);
    return SD_ERR_VALUE;
  }
  const int64_t max_ctx = static_cast<int64_t>(max_blocks_per_seq) * block_size;
  if (num_blocks > (1ll << 31) - 1 || total_q > (1ll << 31) - 1 ||
      !plan_fits(num_seqs, num_kv_heads, max_ctx, num_splits)) {
    sd::set_error("%s: %d sequences x %d kv heads x %lld keys (%d splits) is too much work for one call",
                  what, num_seqs, num_kv_heads, (long long)max_ctx, num_splits);
    return SD_ERR_UNSUPPORTED;
  }
  if (!sd::strides_ok({q_stride_tok, q_stride_head, codes_stride_block, codes_stride_pos,
                       codes_stride_head, scales_stride_block, scales_stride_pos,
                       scales_stride_head, bt_stride, out_stride_tok, out_stride_head})) {
    sd::set_error("%s: strides must lie in [-2^40, 2^40] elements", what);
    return SD_ERR_VALUE;
  }
  const int64_t unit = group_size == 128 ? 4 : 8;
  if (!sd::aligned16(q) || !sd::aligned16(codes) || reinterpret_cast<uintptr_t>(scales) % (2 * unit) ||
      (reinterpret_cast<uintptr_t>(out) & 7u) != 0 || q_stride_tok % 8 || q_stride_head % 8 ||
      codes_stride_block % 16 || codes_stride_pos % 16 || codes_stride_head % 16 ||
      scales_stride_block % unit || scales_stride_pos % unit || scales_stride_head % unit ||
      out_stride_tok % 4 || out_stride_head % 4) {
    sd::set_error("%s: q and code rows must be 16-byte aligned, scale rows aligned to %d bytes, out "
                  "rows to 8", what, static_cast<int>(2 * unit));
    return SD_ERR_UNSUPPORTED;
  }
  if (codes_stride_pos < 0 || scales_stride_pos < 0 || codes_stride_pos > (1ll << 25) ||
      scales_stride_pos > (1ll << 25)) {
    sd::set_error("%s: position strides of the cache must lie in [0, 2^25]", what);
    return SD_ERR_UNSUPPORTED;
  }
  const Plan pl = make_plan(num_seqs, max_qlen, num_q_heads, num_kv_heads, max_ctx, num_splits);
  const size_t need = ws_bytes(pl);
  if (need && (!workspace || workspace_bytes < need || !sd::aligned16(workspace))) {
    sd::set_error("%s: workspace of %zu bytes (16-byte aligned) required, got %zu", what, need,
                  workspace ? workspace_bytes : (size_t)0);
    return SD_ERR_WORKSPACE;
  }
  Params p;
  p.q = static_cast<const uint16_t*>(q);
  p.q_stok = q_stride_tok;
  p.q_shead = q_stride_head;
  p.codes = static_cast<const uint8_t*>(codes);
  p.c_sblk = codes_stride_block;
  p.c_shead = codes_stride_head;
  p.c_spos = static_cast<uint32_t>(codes_stride_pos);
  p.scales = static_cast<const uint8_t*>(scales);
  p.s_sblk = 2 * scales_stride_block;
  p.s_shead = 2 * scales_stride_head;
  p.s_spos = static_cast<uint32_t>(2 * scales_stride_pos);
  p.num_blocks = static_cast<int32_t>(num_blocks);
  p.block_size = block_size;
  p.bs_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
  p.max_ctx = static_cast<int32_t>(max_ctx);
  p.bt = block_table;
  p.bt_stride = bt_stride;
  p.ctx = context_lens;
  p.cu_k = cu_seqlens_k;
  p.cu_q = cu_seqlens_q;
  p.max_qlen = max_qlen;
  p.total_q = total_q;
  p.num_seqs = num_seqs;
  p.gq = num_q_heads / num_kv_heads;
  p.hkv = num_kv_heads;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = static_cast<uint16_t*>(out);
  p.o_stok = out_stride_tok;
  p.o_shead = out_stride_head;
  p.ws = static_cast<float*>(workspace);
  p.runs = static_cast<int32_t>(pl.runs);
  p.whole = pl.whole;
  p.rmax = pl.rmax;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SD_BF16) return launch<__bf16>(p, pl, group_size, st);
  return launch<_Float16>(p, pl, group_size, st);
}
