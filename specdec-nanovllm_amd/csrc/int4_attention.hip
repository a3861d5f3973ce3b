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
// of a workgroup (64 keys where a pair has two 16-row tiles: two waves then take the same keys, one
// tile each, and share what they load in the caches; one wave with both tiles has no registers left
// for a second wave on its SIMD and measured 32 us instead of 22 us for 8 x 7 rows). All chunks, laid end
// to end, are cut into equal runs, one a workgroup, whatever the length mix (context lengths are read
// on the device). When a pair or the run ends, the waves
// merge their softmax states in LDS; a pair that several runs share leaves partials in the workspace
// (two slots a run: the pair it starts in, the pair it ends in), which the combine kernel merges.
// Where the table admits few chunks a pair, a run is one whole pair and there is no second launch.
//
// A step's rows go from memory to LDS without registers (global_load_lds, 5 instructions a step), up
// to kAhead steps ahead; the 16-byte units of a row are permuted by the lanes' global addresses so
// that the operand reads hit all banks. Scales pass once more through LDS as fp32.
//
// Bound by the bytes of the cache, 128 + 8 NG per key and kv head, and close behind by vector issue:
// unpacking costs 144 instructions a step of 32 keys (two a code pair), the softmax of a 16-row tile
// as much again. Where a pair has at most 4 rows (decode with up to 4 query heads a kv head), 12 of
// the tile's 16 columns are empty; there each lane takes 2 of the 8 scores that lanes 0 .. 3 of its
// row of 16 hold (moves within the row), which leaves a quarter of the softmax (R4 below).
#include <math.h>

#include <type_traits>

#include "int4.h"

namespace {

using sd::f32x4;
using sd::u32x4;

constexpr int kD = 128;
constexpr int kStep = 32;               // keys of a wave's step
constexpr int kPitch = kD + 4;          // floats of a row's state: acc, then m and l
constexpr int kMergeRows = 8;           // rows of a tile the waves merge at a time
// Tables of up to this many keys: no splitting of pairs, and past kShortKeys twice the waves. One launch
// of 8 steps' length at most against two (16 heads, 1 x 1000 keys: 10.9 us a call against 14.8; without
// the host, from a graph, 11.4 against 10.0: a call from the host is what a decode step of one pays).
constexpr int kShortKeys = 512, kWholeKeys = 1024;

struct Params {
  const uint16_t* q;
  int64_t q_stok, q_shead;
  const uint8_t* codes;
  uint32_t c_sblk, c_spos, c_shead;  // bytes
  const uint8_t* scales;
  uint32_t s_sblk, s_spos, s_shead;  // bytes
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
  int32_t chunk_shift;  // log2 of a chunk's keys
};

// `total` chunks over `runs` workgroups: runs of one length, the first `more` of them one longer. (All of
// the longer length, and fewer runs: 29.7 us against 28.2 for 8 x 7 rows, 44.1 against 41.9 for 32 x 1.)
struct Cut {
  int each, more;
  __device__ __forceinline__ Cut(int total, int runs) : each(total / runs), more(total - each * runs) {}
  __device__ __forceinline__ int start(int r) const { return r * each + min(r, more); }
  __device__ __forceinline__ int run_of(int chunk) const {
    const int in_long = more * (each + 1);
    return chunk < in_long ? chunk / (each + 1) : more + (chunk - in_long) / max(each, 1);
  }
};

typedef const __attribute__((address_space(4))) int32_t* ScalarPtr;
// Load through the scalar cache of a wave-uniform word that nothing writes while the kernel runs.
__device__ __forceinline__ int scalar_load(const int32_t* p) {
  return *(ScalarPtr)(reinterpret_cast<uintptr_t>(p));
}

__device__ __forceinline__ int chunks_of(const Params& p, int L) {
  return (L + (1 << p.chunk_shift) - 1) >> p.chunk_shift;
}

// A sequence: its keys, query rows and the first of these.
struct Seq {
  int L, nq, q0;
};
__device__ __forceinline__ Seq seq_of(const Params& p, int k0, int k1, int q0, int q1, int b) {
  Seq s;
  s.L = min(max(p.ctx ? k0 : k1 - k0, 0), p.max_ctx);
  s.nq = p.cu_q ? min(max(q1 - q0, 0), p.max_qlen) : 1;
  s.q0 = p.cu_q ? q0 : b;
  return s;
}
// Sequence b on each lane. All four words are loaded whatever the arrays: loads under branches would
// wait for each other.
__device__ __forceinline__ Seq lane_seq(const Params& p, int b) {
  const int32_t* kp = p.ctx ? p.ctx : p.cu_k;
  const int32_t* qp = p.cu_q ? p.cu_q : kp;
  const int kn = p.ctx ? 0 : 1, qn = p.cu_q ? 1 : 0;
  const int k0 = kp[b], k1 = kp[b + kn], q0 = qp[b], q1 = qp[b + qn];
  return seq_of(p, k0, k1, q0, q1, b);
}
__device__ __forceinline__ Seq uniform_seq(const Params& p, int b) {
  const int32_t* kp = p.ctx ? p.ctx : p.cu_k;
  const int32_t* qp = p.cu_q ? p.cu_q : kp;
  const int kn = p.ctx ? 0 : 1, qn = p.cu_q ? 1 : 0;
  return seq_of(p, scalar_load(kp + b), scalar_load(kp + b + kn), scalar_load(qp + b),
                scalar_load(qp + b + qn), b);
}
__device__ __forceinline__ Seq seq_from_lane(const Seq& s, int lane) {
  return Seq{__builtin_amdgcn_readlane(s.L, lane), __builtin_amdgcn_readlane(s.nq, lane),
             __builtin_amdgcn_readlane(s.q0, lane)};
}

template <typename T>
__device__ __forceinline__ void store_row4(const Params& p, const Seq& sq, int h, int row, int c,
                                           f32x4 v) {
  const int qi = row / p.gq, g = row - qi * p.gq;
  const int64_t qt = static_cast<int64_t>(sq.q0) + qi;
  if (qt < 0 || qt >= p.total_q) return;
  uint2 w;
  w.x = sd::pack2<T>(v.x, v.y);
  w.y = sd::pack2<T>(v.z, v.w);
  *reinterpret_cast<uint2*>(p.out + qt * p.o_stok + static_cast<int64_t>(h * p.gq + g) * p.o_shead + 4 * c) = w;
}

// 16 (4) bytes per lane to LDS byte 16 (4) * lane of the wave-uniform address l. In assembly for the
// scalar-base form and because the compiler makes LDS reads wait for every such load in flight; the
// loop waits for its own. No register is written.
__device__ __forceinline__ uint32_t lds_addr(const void* l) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)l));
}
__device__ __forceinline__ void to_lds16(const uint8_t* base, uint32_t off, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               ::"s"(l), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void to_lds16(const uint8_t* at, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               ::"s"(l), "v"(at) : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(const uint8_t* at, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               ::"s"(l), "v"(at) : "memory", "m0");
}

// CTRL's lane moves of a value; lanes outside BANKS (four lanes a bit) keep `old`.
template <int CTRL, int BANKS> __device__ __forceinline__ float merge_dpp(float old, float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                       __builtin_bit_cast(int, old), __builtin_bit_cast(int, v), CTRL,
                                       0xF, BANKS, false));
}
template <int CTRL> __device__ __forceinline__ uint32_t move_dpp(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, true));
}
constexpr int kShl4 = 0x104, kShl8 = 0x108, kShl12 = 0x10C, kShr4 = 0x114, kShr8 = 0x118, kShr12 = 0x11C;
constexpr int kRor4 = 0x124, kRor8 = 0x128;

// How pages meet a wave's 32 keys: they lie in one page, each half does, or anything.
enum Pages { kOnePage, kHalfPages, kAnyPages };

// Position in the layout: chunk j of the n chunks of pair (b, h); blk: the pages of the wave's keys.
struct Pos {
  int b, h, j, n, L;
  int blk[2];
};
// 32 x 32 -> 64 bits (two scalar multiplies)
__device__ __forceinline__ uint64_t wide(uint32_t a, uint32_t b) { return static_cast<uint64_t>(a) * b; }

// LDS of one wave: kAhead slots of a step (32 rows of 128 bytes, then their scales), fp32 scales.
template <int NG> constexpr int ahead() { return NG == 4 ? 2 : 3; }
template <int NG> constexpr int slot_bytes() { return kStep * (kD + 8 * NG); }
template <int NG> constexpr int wave_bytes() { return ahead<NG>() * slot_bytes<NG>() + kStep * 16 * NG; }

template <typename T, int NG, int TS, bool R4, Pages PAGES, int kWaves>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
void int4_attn_main(Params p) {
  static_assert(!R4 || TS == 1, "four rows fit one tile");
  constexpr int kChunk = kWaves / TS * kStep;
  constexpr int kAhead = ahead<NG>();
  constexpr int kLoads = 5;  // vector memory instructions of a step
  constexpr int NE = R4 ? 2 : 8;  // scores of a row tile on a lane
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kWaves][wave_bytes<NG>()];
  __shared__ __attribute__((aligned(16))) float lds_m[kWaves][kMergeRows][kPitch];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int ks = wave / TS, ts = wave % TS;  // this wave's keys of a chunk, its row tile

  // ---- this run's chunks and where they begin
  Pos cur;
  Seq seqs{0, 1, 0};  // up to 64 sequences: sequence `lane`
  Seq sq;
  const bool in_lanes = p.num_seqs <= 64;
  int left, s0 = 0;
  bool entered = false;  // the current pair began in an earlier run
  const int run = blockIdx.x;
  auto seq_at = [&](int b) { return in_lanes ? seq_from_lane(seqs, b) : uniform_seq(p, b); };
  if (in_lanes) seqs = lane_seq(p, min(lane, p.num_seqs - 1));
  if (p.whole) {
    cur.b = run / p.hkv;
    cur.h = run - cur.b * p.hkv;
    cur.j = 0;
    sq = seq_at(cur.b);
    cur.L = sq.L;
    cur.n = left = chunks_of(p, cur.L);
    if (left == 0) {
      for (int i = tid; i < p.gq * sq.nq * 32; i += kWaves * 64)
        store_row4<T>(p, sq, cur.h, i / 32, i % 32, f32x4{0.f, 0.f, 0.f, 0.f});
      return;
    }
  } else {
    int total = 0;  // chunks of one head
    int before = 0;
    cur.b = 0;
    if (in_lanes) {
      const int n = lane < p.num_seqs ? chunks_of(p, seqs.L) : 0;
      const int incl = sd::wave_inclusive_sum(n);
      total = __builtin_amdgcn_readlane(incl, 63);
      const Cut cut(total * p.hkv, p.runs);
      s0 = cut.start(run);
      left = cut.start(run + 1) - s0;
      if (left <= 0) return;
      const unsigned long long hit =
          __ballot(n > 0 && (incl - n) * p.hkv <= s0 && s0 < incl * p.hkv);
      cur.b = __ffsll(hit) - 1;
      before = __builtin_amdgcn_readlane(incl - n, cur.b);
    } else {
      for (int c = lane; c < p.num_seqs; c += 64) total += chunks_of(p, lane_seq(p, c).L);
      for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off);
      total = __builtin_amdgcn_readfirstlane(total);
      const Cut cut(total * p.hkv, p.runs);
      s0 = cut.start(run);
      left = cut.start(run + 1) - s0;
      if (left <= 0) return;
      for (int c = 0, sum = 0; c < p.num_seqs; c += 64) {
        const int n = c + lane < p.num_seqs ? chunks_of(p, lane_seq(p, c + lane).L) : 0;
        const int incl = sum + sd::wave_inclusive_sum(n);
        const unsigned long long hit =
            __ballot(n > 0 && (incl - n) * p.hkv <= s0 && s0 < incl * p.hkv);
        if (hit) {
          const int src = __ffsll(hit) - 1;
          cur.b = c + src;
          before = __builtin_amdgcn_readlane(incl - n, src);
          break;
        }
        sum = __builtin_amdgcn_readlane(incl, 63);
      }
    }
    cur.b = __builtin_amdgcn_readfirstlane(cur.b);
    sq = seq_at(cur.b);
    cur.L = sq.L;
    cur.n = chunks_of(p, cur.L);
    const int in = s0 - before * p.hkv;
    cur.h = in / cur.n;
    cur.j = in - cur.h * cur.n;
    entered = cur.j > 0;
  }

  auto next_pair = [&](Pos& a) {
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
      a.L = seq_at(a.b).L;
      a.n = chunks_of(p, a.L);
    } while (a.n == 0);
  };

  // ---- loads: a step's rows, 8 a instruction, lane l unit (l % 8) ^ (l / 8) of row l / 8; its scales
  uint8_t* const mine = lds[wave];
  const uint32_t mine_at = __builtin_amdgcn_readfirstlane(lds_addr(mine));
  const uint32_t unit = ((lane & 7) ^ (lane >> 3)) * 16;
  uint32_t row_off[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) row_off[r] = static_cast<uint32_t>(8 * r + (lane >> 3)) * p.c_spos + unit;
  // the key whose scales this lane loads and the byte of them (16 bytes a lane; NG = 1: 4)
  const int s_key = NG == 4 ? lane >> 1 : NG == 2 ? lane & 31 : lane >> 1;
  const uint32_t s_byte = NG == 4 ? 16 * (lane & 1) : NG == 2 ? 0 : 4 * (lane & 1);

  auto page_of = [&](int tok) { return p.bs_shift >= 0 ? tok >> p.bs_shift : tok / p.block_size; };
  auto in_page = [&](int tok) {
    return p.bs_shift >= 0 ? tok & (p.block_size - 1) : tok % p.block_size;
  };
  auto first_key = [&](const Pos& a) { return min(a.j * kChunk + ks * kStep, a.L - 1); };
  // Table lookups of a position's pages, a step ahead of their use.
  auto find_pages = [&](Pos& a) {
    if constexpr (PAGES != kAnyPages) {
      const int t0 = first_key(a);
      const int32_t* row = p.bt + a.b * p.bt_stride;
      a.blk[0] = scalar_load(row + page_of(t0));
      if constexpr (PAGES == kHalfPages) a.blk[1] = scalar_load(row + page_of(min(t0 + 16, a.L - 1)));
    }
  };
  Pos pos = cur;  // what load_step loads next
  int pos_left = left;
  find_pages(pos);
  // The same instructions whatever the lengths: rows past the end read the last key, steps past the
  // run its last chunk again.
  auto load_step = [&](int slot) {
    const uint32_t l = mine_at + slot * slot_bytes<NG>(), ls = l + kStep * kD;
    const int last = pos.L - 1, t0 = first_key(pos);
    const uint8_t* const hc = p.codes + wide(pos.h, p.c_shead);
    const uint8_t* const hs = p.scales + wide(pos.h, p.s_shead);
    const uint8_t* s_at;
    if constexpr (PAGES == kOnePage) {
      const int blk = min(max(pos.blk[0], 0), p.num_blocks - 1), off = in_page(t0);
      const uint8_t* cp = hc + wide(blk, p.c_sblk) + wide(off, p.c_spos);
      // (the step's keys, then the product: that of all keys left may pass 32 bits)
      const uint32_t most = static_cast<uint32_t>(min(last - t0, kStep - 1)) * p.c_spos + unit;
#pragma unroll
      for (int r = 0; r < 4; ++r) to_lds16(cp, min(row_off[r], most), l + 1024 * r);
      s_at = hs + wide(blk, p.s_sblk) + wide(off, p.s_spos) +
             (static_cast<uint32_t>(min(s_key, last - t0)) * p.s_spos + s_byte);
    } else if constexpr (PAGES == kHalfPages) {
      const uint8_t* sp[2];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int t = min(t0 + 16 * f, last);
        const int blk = min(max(pos.blk[f], 0), p.num_blocks - 1), off = in_page(t);
        const uint8_t* cp = hc + wide(blk, p.c_sblk) + wide(off, p.c_spos);
        const uint32_t most = static_cast<uint32_t>(min(last - t, kStep / 2 - 1)) * p.c_spos + unit;
#pragma unroll
        for (int r = 0; r < 2; ++r) to_lds16(cp, min(row_off[r], most), l + 2048 * f + 1024 * r);
        sp[f] = hs + wide(blk, p.s_sblk) + wide(off, p.s_spos) +
                (static_cast<uint32_t>(min(s_key & 15, last - t)) * p.s_spos + s_byte);
      }
      s_at = s_key < 16 ? sp[0] : sp[1];
    } else {
      const int32_t* table = p.bt + pos.b * p.bt_stride;
      auto block = [&](int tok) { return min(max(table[page_of(tok)], 0), p.num_blocks - 1); };
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int tok = min(t0 + 8 * r + (lane >> 3), last);
        to_lds16(hc + wide(block(tok), p.c_sblk) + wide(in_page(tok), p.c_spos) + unit, l + 1024 * r);
      }
      const int tok = min(t0 + s_key, last);
      s_at = hs + wide(block(tok), p.s_sblk) + wide(in_page(tok), p.s_spos) + s_byte;
    }
    if constexpr (NG == 1) to_lds4(s_at, ls);
    else if (NG == 4 || lane < 32) to_lds16(s_at, ls);
    if (pos_left > 1) {
      --pos_left;
      if (++pos.j == pos.n) next_pair(pos);
      find_pages(pos);
    }
  };

  // ---- state of the current pair. R4: a lane's scores are row lr % 4's, keys 16 (lr / 8) + 4 lg +
  //      2 (lr / 4 % 2) and the next; its accumulators still row lr's (rows 4 .. 15: nothing).
  u32x4 qop[4];
  float qsum[NG], zsum[NG], m_run, l_run;
  int lim, causal = 0;
  f32x4 acc[8];
  auto key_of = [&](int e) {  // of score e, within the step
    return R4 ? 16 * (lr >> 3) + 4 * lg + 2 * ((lr >> 2) & 1) + e : e < 4 ? 4 * lg + e : 12 + 4 * lg + e;
  };

  auto begin_pair = [&]() {
    causal = cur.L - sq.nq;
    // R4: the columns of rows 4 .. 15 repeat rows 0 .. 3 (their scores stay unread)
    const int row = R4 ? lr & 3 : ts * 16 + lr;
    const int qi = row / p.gq, gq = row - qi * p.gq;
    const int64_t qt = static_cast<int64_t>(sq.q0) + qi;
    const bool valid = qi < sq.nq && qt >= 0 && qt < p.total_q;
    lim = valid ? min(causal + qi, cur.L - 1) : -1;
    const uint16_t* qp = p.q + (valid ? qt * p.q_stok + static_cast<int64_t>(cur.h * p.gq + gq) * p.q_shead : 0) + 8 * lg;
    float part[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      qop[i] = valid ? sd::load16(qp + 32 * i) : u32x4{0u, 0u, 0u, 0u};
      const uint32_t one = __is_same(T, __bf16) ? 0x3F803F80u : 0x3C003C00u;
      part[i] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) part[i] = sd::dot2<T>(qop[i][e], one, part[i]);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i * NG / 4 == g) s += part[i];
      qsum[g] = sd::sum_over_groups(s);
      zsum[g] = 0.f;
    }
    m_run = -INFINITY;
    l_run = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  };

  // ---- LDS addresses of the operand reads (see the loads for the order of a row's units)
  const uint32_t k_at = lr * 128 + ((lg ^ (lr & 7)) * 16);
  uint32_t v_at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v_at[j] = (4 * lg + j) * 128 + (((lr >> 2) ^ j) + 4 * (1 ^ (lg & 1))) * 16 + 4 * (lr & 3);
  float* const sf = reinterpret_cast<float*>(mine + kAhead * slot_bytes<NG>());  // [key][4 NG]
  const uint32_t kbase = sd::code_base<T>(), vbase = sd::code_base<__bf16>();

  auto compute = [&](const u32x4 (&kw)[2], const uint32_t (&vw)[8], int tb, auto full_) {
    constexpr bool kFull = decltype(full_)::value;
    // ---- scores in log2 units, from the products with the codes: there a lane holds keys
    //      16 tt + 4 lg + i of row lr
    float sc[NE];
    f32x4 dot[NG][2];
    auto score = [&](int e, int tt, int i) {
      const float* s = sf + key_of(e) * 4 * NG;
      float v = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float d = dot[g][tt][i];
        if constexpr (R4) {
          d = merge_dpp<kShr4, 0x2>(d, dot[g][0][2 + e]);
          d = merge_dpp<kShr8, 0x4>(d, dot[g][1][e]);
          d = merge_dpp<kShr12, 0x8>(d, dot[g][1][2 + e]);
        }
        v = fmaf(s[g], d, fmaf(s[NG + g], qsum[g], v));
      }
      sc[e] = kFull || tb + key_of(e) <= lim ? v : -INFINITY;
    };
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i * NG / 4 == g) c = sd::Elem<T>::mfma(sd::unpack8<T>(kw[tt][i], kbase), qop[i], c);
        dot[g][tt] = c;
      }
      if constexpr (!R4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) score(4 * tt + i, tt, i);
      }
    }
    if constexpr (R4) {
#pragma unroll
      for (int e = 0; e < 2; ++e) score(e, 0, e);
    }
    // ---- online softmax; the running maximum moves only when a score exceeds it by more than 8
    //      (log2 units): p <= 2^8 otherwise, well inside fp32 and the bf16 parts
    float mloc = sc[0];
#pragma unroll
    for (int e = 1; e < NE; ++e) mloc = fmaxf(mloc, sc[e]);
    if (__any(mloc > m_run + 8.f)) {
      mloc = sd::max_over_groups(mloc);
      if constexpr (R4) {
        mloc = fmaxf(mloc, __uint_as_float(move_dpp<kRor4>(__float_as_uint(mloc))));
        mloc = fmaxf(mloc, __uint_as_float(move_dpp<kRor8>(__float_as_uint(mloc))));
      }
      const float mnew = fmaxf(m_run, mloc);
      const float alpha = sd::fast_exp2(m_run - (mnew == -INFINITY ? 0.f : mnew));
      l_run *= alpha;
#pragma unroll
      for (int g = 0; g < NG; ++g) zsum[g] *= alpha;
#pragma unroll
      for (int t = 0; t < 8; ++t) acc[t] *= alpha;
      m_run = mnew;
    }
    const float mb = m_run == -INFINITY ? 0.f : m_run;
    u32x4 hi[NG], lo[NG];
#pragma unroll
    for (int e2 = 0; e2 < NE / 2; ++e2) {
      float ps[2][NG];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int e = 2 * e2 + u;
        const float pv = sd::fast_exp2(sc[e] - mb);
        l_run += pv;
        const float* s = sf + key_of(e) * 4 * NG + 2 * NG;
        const bool seen = kFull || tb + key_of(e) <= lim;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          // a key that this row does not see may hold anything
          ps[u][g] = pv * (seen ? s[g] : 0.f);
          zsum[g] = fmaf(pv, seen ? s[NG + g] : 0.f, zsum[g]);
        }
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t h, l;
        sd::split_pack<__bf16>(ps[0][g], ps[1][g], h, l);
        if constexpr (R4) {
          hi[g] = u32x4{h, move_dpp<kShl4>(h), move_dpp<kShl8>(h), move_dpp<kShl12>(h)};
          lo[g] = u32x4{l, move_dpp<kShl4>(l), move_dpp<kShl8>(l), move_dpp<kShl12>(l)};
        } else {
          hi[g][e2] = h;
          lo[g][e2] = l;
        }
      }
    }
    // ---- O^T += V^T P^T: byte b of the 8 value dwords holds tiles 2 b (low half) and 2 b + 1
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      u32x4 va, vb;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // byte b of keys 2 e and 2 e + 1, each in the low byte of a half
        const uint32_t z = __builtin_amdgcn_perm(vw[2 * e + 1], vw[2 * e], 0x0c040c00u + 0x00010001u * b);
        va[e] = sd::code_pair<__bf16, 0>(z, vbase);
        vb[e] = sd::code_pair<__bf16, 4>(z, vbase);
      }
      const int g = b * NG / 4;
      acc[2 * b] = sd::Elem<__bf16>::mfma(va, hi[g], acc[2 * b]);
      acc[2 * b + 1] = sd::Elem<__bf16>::mfma(vb, hi[g], acc[2 * b + 1]);
      acc[2 * b] = sd::Elem<__bf16>::mfma(va, lo[g], acc[2 * b]);
      acc[2 * b + 1] = sd::Elem<__bf16>::mfma(vb, lo[g], acc[2 * b + 1]);
    }
  };

  bool first_pair = true;
  auto step = [&](int slot) {
    const int tb = cur.j * kChunk + ks * kStep;
    // the oldest step in flight has landed (anything issued after the newer ones only waits longer)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kAhead - 1) * kLoads) : "memory");
    const uint8_t* d = mine + slot * slot_bytes<NG>();
    uint32_t raw[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) raw[g] = reinterpret_cast<const uint32_t*>(d + kStep * kD)[lane * NG + g];
    u32x4 kw[2];
    uint32_t vw[8];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) kw[tt] = sd::load16(d + k_at + 2048 * tt);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      vw[j] = *reinterpret_cast<const uint32_t*>(d + v_at[j & 3] + 2048 * (j >> 2));
    // ---- scales to LDS in fp32: key (s c, (z - 16 s) c) with c = softmax scale * log2(e), value
    //      (s, z - 16 s); lane 2 k (2 k + 1) holds key k's key (value) scales
    {
      float* o = sf + lane * 2 * NG;
      const float f = lane & 1 ? 1.f : p.scale_log2;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float s = sd::from_bits<T>(static_cast<uint16_t>(raw[g]));
        const float z = sd::from_bits<T>(static_cast<uint16_t>(raw[g] >> 16));
        o[g] = s * f;
        o[NG + g] = fmaf(-16.f, s, z) * f;
      }
    }
    // the slot's words are in registers: its next step may land
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    load_step(slot);
    if (tb < cur.L) {  // wave-uniform
      sd::wave_lds_sync();
      if (tb + kStep - 1 <= min(causal, cur.L - 1)) compute(kw, vw, tb, std::true_type{});
      else compute(kw, vw, tb, std::false_type{});
    }
    sd::wave_lds_sync();  // every lane has read the scales before the next step writes its own
  };

  // Merges the waves' states of the current pair: rows of out where this run saw the whole pair, a
  // partial otherwise. Every wave comes here.
  auto flush = [&](bool whole_pair) {
    float* slot = p.ws + (2 * static_cast<int64_t>(run) + (first_pair ? 0 : 1)) * p.rmax * kPitch;
    const int rows = p.gq * sq.nq;
    float l = sd::sum_over_groups(l_run);
#pragma unroll
    for (int g = 0; g < NG; ++g) zsum[g] = sd::sum_over_groups(zsum[g]);
    if constexpr (R4) {  // the four lanes of a row that share its scores
      l = sd::dpp_add<kRor8>(sd::dpp_add<kRor4>(l));
#pragma unroll
      for (int g = 0; g < NG; ++g) zsum[g] = sd::dpp_add<kRor8>(sd::dpp_add<kRor4>(zsum[g]));
    }
    for (int r8 = 0; r8 < 16 / kMergeRows && r8 * kMergeRows < rows; ++r8) {
      if (lr / kMergeRows == r8) {
        float* d = lds_m[wave][lr % kMergeRows];
#pragma unroll
        for (int t = 0; t < 8; ++t)
          sd::store16(d + 16 * t + 4 * lg, __builtin_bit_cast(u32x4, acc[t] + zsum[t * NG / 8]));
        if (lg == 0) {
          d[kD] = m_run;
          d[kD + 1] = l;
        }
      }
      __syncthreads();
      // a thread takes 4 dims of a row of each tile (8 waves: of one tile; there may be only one)
      const int r = (tid >> 5) % kMergeRows, c = tid & 31;
      for (int t = kWaves == 4 ? 0 : tid / (kMergeRows * 32); t < TS; t += kWaves == 4 ? 1 : 2) {
        const int row = 16 * t + kMergeRows * r8 + r;
        if (row >= rows) continue;
        float M = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = t; w < kWaves; w += TS) M = fmaxf(M, lds_m[w][r][kD]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = t; w < kWaves; w += TS) {
          const float m = lds_m[w][r][kD], lw = lds_m[w][r][kD + 1];
          // no finite score: l is 0 (nothing seen), or NaN, which stays
          const float f = m == -INFINITY ? lw : exp2f(m - M);
          sum = fmaf(f, lw, sum);
          o += f * __builtin_bit_cast(f32x4, sd::load16(&lds_m[w][r][4 * c]));
        }
        if (whole_pair) {
          // the sum is 0 only for a row that sees no key (NaN stays NaN)
          store_row4<T>(p, sq, cur.h, row, c, o * (sum == 0.f ? 0.f : 1.f / sum));
        } else {
          float* d = slot + row * kPitch;
          sd::store16(d + 4 * c, __builtin_bit_cast(u32x4, o));
          if (c == 0) {
            d[kD] = M;
            d[kD + 1] = sum;
          }
        }
      }
      __syncthreads();
    }
  };

#pragma unroll
  for (int i = 0; i < kAhead; ++i) load_step(i);
  begin_pair();
  for (int slot = 0;; slot = slot + 1 == kAhead ? 0 : slot + 1) {
    step(slot);
    ++cur.j;
    --left;
    if (cur.j == cur.n || left == 0) {
      flush(cur.j == cur.n && !entered);
      if (left == 0) break;
      entered = first_pair = false;
      next_pair(cur);
      sq = seq_at(cur.b);
      begin_pair();
    }
  }
  // the loads that ran ahead land before the workgroup's LDS is another's
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Rows of pairs that several runs share from their partials, zeros for sequences without keys; a
// pair that one run saw whole is written already. 4 dims of a row a thread.
template <typename T> __global__ __launch_bounds__(256) void int4_attn_combine(Params p) {
  __shared__ __attribute__((aligned(16))) float part[8][kPitch];
  const int tid = threadIdx.x, lane = tid & 63;
  const int b = blockIdx.x / p.hkv, h = blockIdx.x - b * p.hkv;
  int total = 0, before = 0;
  Seq sq;
  if (p.num_seqs <= 64) {
    const Seq s = lane_seq(p, min(lane, p.num_seqs - 1));
    const int n = lane < p.num_seqs ? chunks_of(p, s.L) : 0;
    const int incl = sd::wave_inclusive_sum(n);
    total = __builtin_amdgcn_readlane(incl, 63);
    before = __builtin_amdgcn_readlane(incl - n, b);
    sq = seq_from_lane(s, b);
  } else {
    for (int c = lane; c < p.num_seqs; c += 64) {
      const int n = chunks_of(p, lane_seq(p, c).L);
      total += n;
      before += c < b ? n : 0;
    }
    for (int off = 32; off > 0; off >>= 1) {
      total += __shfl_xor(total, off);
      before += __shfl_xor(before, off);
    }
    sq = uniform_seq(p, b);
  }
  const int n = chunks_of(p, sq.L), rows = p.gq * sq.nq;
  const int half = tid >> 5, c = tid & 31;
  if (n == 0) {
    for (int row = blockIdx.y * 8 + half; row < rows; row += gridDim.y * 8)
      store_row4<T>(p, sq, h, row, c, f32x4{0.f, 0.f, 0.f, 0.f});
    return;
  }
  const Cut cut(total * p.hkv, p.runs);
  const int first = before * p.hkv + h * n;
  const int r0 = cut.run_of(first), r1 = cut.run_of(first + n - 1);
  if (r0 == r1) return;
  // few partials: a half wave takes a row, 8 loads in flight (sharing from 8 partials on took 1 us longer
  // at 8 x 7 rows, with 9 of them); many: the half waves share a row's
  const bool share = r1 - r0 >= 16;
  for (int row = share ? blockIdx.y : blockIdx.y * 8 + half; row < rows; row += share ? gridDim.y : gridDim.y * 8) {
    float M = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    auto state = [&](int r) {
      return p.ws + ((2 * static_cast<int64_t>(r) + (first > cut.start(r) ? 1 : 0)) * p.rmax + row) * kPitch;
    };
    auto add = [&](float m2, float l2, f32x4 o2) {
      const float m = fmaxf(M, m2);
      // no finite score: l is 0 (nothing seen), or NaN, which stays
      const float f = M == -INFINITY ? l : exp2f(M - m), f2 = m2 == -INFINITY ? l2 : exp2f(m2 - m);
      l = l * f + l2 * f2;
      o = o * f + o2 * f2;
      M = m;
    };
    constexpr int kOnce = 8;  // loads in flight
    const int by = share ? 8 : 1;
    for (int r = share ? r0 + half : r0; r <= r1; r += by * kOnce) {
      float2 ml[kOnce];
      f32x4 v[kOnce];
#pragma unroll
      for (int i = 0; i < kOnce; ++i) {
        const float* s = state(min(r + by * i, r1));
        ml[i] = *reinterpret_cast<const float2*>(s + kD);
        v[i] = __builtin_bit_cast(f32x4, sd::load16(s + 4 * c));
      }
#pragma unroll
      for (int i = 0; i < kOnce; ++i)
        if (r + by * i <= r1) add(ml[i].x, ml[i].y, v[i]);
    }
    if (!share) {
      store_row4<T>(p, sq, h, row, c, o * (l == 0.f ? 0.f : 1.f / l));
      continue;
    }
    sd::store16(&part[half][4 * c], __builtin_bit_cast(u32x4, o));
    if (c == 0) {
      part[half][kD] = M;
      part[half][kD + 1] = l;
    }
    __syncthreads();
    if (half == 0) {
#pragma unroll
      for (int i = 1; i < 8; ++i)
        add(part[i][kD], part[i][kD + 1], __builtin_bit_cast(f32x4, sd::load16(&part[i][4 * c])));
      store_row4<T>(p, sq, h, row, c, o * (l == 0.f ? 0.f : 1.f / l));
    }
    __syncthreads();
  }
}

// Keys of a chunk of 4 or 8 waves: fewer where two waves share them
int64_t chunk_keys(int64_t rows, int waves) { return kStep * waves / (rows <= 16 ? 1 : 2); }

struct Plan {
  int64_t runs;
  bool whole;
  int rmax;
};

Plan make_plan(int num_seqs, int max_qlen, int hq, int hkv, int64_t max_ctx, int num_splits) {
  Plan pl;
  pl.rmax = hq / hkv * max_qlen;
  const int64_t pairs = static_cast<int64_t>(num_seqs) * hkv;
  pl.whole = num_splits == 0 && max_ctx <= kWholeKeys;
  if (pl.whole) {
    pl.runs = pairs;
  } else {
    // one resident set of workgroups of 4 waves, two a compute unit
    const int64_t chunk = chunk_keys(pl.rmax, 4), most = pairs * ((max_ctx + chunk - 1) / chunk);
    pl.runs = num_splits > 0 ? pairs * num_splits : 2ll * sd::device_cus();
    if (pl.runs > most) pl.runs = most;
  }
  return pl;
}

bool plan_fits(int num_seqs, int hkv, int64_t max_ctx, int num_splits) {
  const int64_t pairs = static_cast<int64_t>(num_seqs) * hkv, chunk = kStep * 2;
  return max_ctx <= (1ll << 30) && pairs <= (1ll << 23) && num_splits <= (1 << 16) &&
         pairs * ((max_ctx + chunk - 1) / chunk) <= (1ll << 30) &&
         (num_splits == 0 || pairs * num_splits <= (1ll << 22));
}

size_t ws_bytes(const Plan& pl) {
  return pl.whole ? 0 : static_cast<size_t>(2 * pl.runs) * pl.rmax * kPitch * sizeof(float);
}

template <typename T, int NG, int TS, bool R4, Pages PAGES> void launch_waves(const Params& p, hipStream_t st) {
  if (p.whole && p.max_ctx > kShortKeys)
    hipLaunchKernelGGL((int4_attn_main<T, NG, TS, R4, PAGES, 8>), dim3(p.runs), dim3(512), 0, st, p);
  else
    hipLaunchKernelGGL((int4_attn_main<T, NG, TS, R4, PAGES, 4>), dim3(p.runs), dim3(256), 0, st, p);
}

template <typename T, int NG, int TS, bool R4> void launch_main(const Params& p, hipStream_t st) {
  if (p.block_size % kStep == 0) launch_waves<T, NG, TS, R4, kOnePage>(p, st);
  else if (p.block_size % (kStep / 2) == 0) launch_waves<T, NG, TS, R4, kHalfPages>(p, st);
  else launch_waves<T, NG, TS, R4, kAnyPages>(p, st);
}

template <typename T, int NG> void launch_rows(const Params& p, hipStream_t st) {
  if (p.rmax <= 4) launch_main<T, NG, 1, true>(p, st);
  else if (p.rmax <= 16) launch_main<T, NG, 1, false>(p, st);
  else launch_main<T, NG, 2, false>(p, st);
}

template <typename T> int launch(const Params& p, const Plan& pl, int group, hipStream_t st) {
  if (group == 32) launch_rows<T, 4>(p, st);
  else if (group == 64) launch_rows<T, 2>(p, st);
  else launch_rows<T, 1>(p, st);
  const int rc = sd::check_launch("paged_attention_int4 main");
  if (rc != SD_OK || pl.whole) return rc;
  const int pairs = p.num_seqs * p.hkv;
  const dim3 grid(pairs, pl.runs >= 16ll * pairs ? p.rmax : (p.rmax + 7) / 8);
  hipLaunchKernelGGL((int4_attn_combine<T>), grid, dim3(256), 0, st, p);
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
      scales_stride_pos > (1ll << 24) || codes_stride_block < 0 || codes_stride_head < 0 ||
      scales_stride_block < 0 || scales_stride_head < 0 || codes_stride_block >= (1ll << 32) ||
      codes_stride_head >= (1ll << 32) || scales_stride_block >= (1ll << 31) ||
      scales_stride_head >= (1ll << 31)) {
    sd::set_error("%s: position strides of the cache must lie in [0, 2^25] bytes, block and head "
                  "strides in [0, 2^32) bytes", what);
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
  p.c_sblk = static_cast<uint32_t>(codes_stride_block);
  p.c_shead = static_cast<uint32_t>(codes_stride_head);
  p.c_spos = static_cast<uint32_t>(codes_stride_pos);
  p.scales = static_cast<const uint8_t*>(scales);
  p.s_sblk = static_cast<uint32_t>(2 * scales_stride_block);
  p.s_shead = static_cast<uint32_t>(2 * scales_stride_head);
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
  p.chunk_shift = __builtin_ctzll(chunk_keys(pl.rmax, pl.whole && max_ctx > kShortKeys ? 8 : 4));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SD_BF16) return launch<__bf16>(p, pl, group_size, st);
  return launch<_Float16>(p, pl, group_size, st);
}
