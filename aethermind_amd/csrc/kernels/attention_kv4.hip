// Causal grouped-query attention over a 4-bit KV cache (AM_KV_MXFP4, am_kv4.h).
//
// A block owns one unit (up to 16 / G query positions of one sequence with the G query
// heads of one kv head: the 16 columns of an MFMA tile) and a contiguous piece of its
// keys; its NW waves take the 32-key steps of the piece in turn.  No cache byte passes
// through LDS: both products' operands are built in the registers of the lane that loaded
// the codes, and v_cvt_scalef32_pk_bf16_fp4 gives two exact bf16 values an instruction.
//   * Scores S^T = K Q^T on v_mfma_f32_16x16x32_bf16.  The order of the reduction over d is
//     free, so lane (j, h) of score tile tt takes D/4 neighbouring dimensions of key
//     16 tt + j, (D/4) h on: one 16-byte load (D = 128), a whole scale group, and its word kk
//     is the operand of MFMA kk.  Q's operand holds the same dimensions.  Lane (j, h) gets
//     the scores of column j for keys 16 tt + 4 h + r, so column j's softmax state lives in
//     the lanes with lane % 16 = j.
//   * O += P V on the same MFMA: k slot e of lane group h is key 16 (e >> 2) + 4 h + (e & 3),
//     the keys whose scores the lane holds, so P stays in its lane.  Lane n of output tile t
//     holds dimension (D/16) n + t: it loads its 8 keys' D/16 neighbouring codes, converts
//     them, and byte permutes gather tile t's column.
//   * bf16 q: the products of scores are exact in fp32 sums, P is split into two bf16 parts
//     (16 bits).  fp32 q: q and P are three parts each (24 bits).
//   * exp2 with scale * log2(e) in the exponent's fma.  Running maxima are rescaled only when
//     one grew.
// Pieces: every block derives the same plan from the contexts (kv4_plan): pieces of at most
// `per` steps, the shortest with which all units fit the grid's slots.  The pieces of a unit
// write records with device-coherent stores and take a ticket; the last one merges them in
// piece order, so results do not depend on the schedule.  (The ordering that this relies on,
// relaxed device-coherent accesses around a wait, is the one of attention.hip's merge.)

#include <algorithm>
#include <cmath>

#include "am_kv4.h"
#include "am_launch_timing.h"

namespace am {
namespace {

struct Attn4Args {
  const void* q;
  void* out;
  const uint8_t *kc, *ks, *vc, *vs;
  const int64_t* start;
  const int32_t* lens;
  float* part;
  unsigned* tickets;
  KvRows kv;
  int32_t batch, seq, hq, hkv, G, qt, tiles, units, cap;
  int32_t slots;  // planned grid; 0: one piece per unit
  int32_t min_steps;
  float scale;  // of the scores, times log2(e)
};

typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
constexpr int kCpolSc1 = 16;
constexpr int kRawBufferFlags = 0x00020000;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kStep = 32;              // keys of a step
constexpr int64_t kTicketBytes = 16384;
constexpr int64_t kMaxSlotHeads = kTicketBytes / 4;  // slots x kv heads of a planned grid

// Value held by lane (lane ^ OFF), OFF 16 or 32.
template <int OFF>
__device__ __forceinline__ float xor_lane(float v, int lane) {
  if constexpr (OFF == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(((lane >> 4) & 1) ? r[0] : r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(lane < 32 ? r[1] : r[0]);
  }
}

// Sum over the lanes up to and including this one.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_shift_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan_i(int v) {
  v = dpp_shift_add<0x111, 0xF>(v);
  v = dpp_shift_add<0x112, 0xF>(v);
  v = dpp_shift_add<0x114, 0xF>(v);
  v = dpp_shift_add<0x118, 0xF>(v);
  return dpp_shift_add<0x143, 0xC>(dpp_shift_add<0x142, 0xA>(v));
}
__device__ __forceinline__ int wave_total_i(int v) { return __builtin_amdgcn_readlane(wave_scan_i(v), 63); }

// Keys of the unit's last live row, in [0, cap]; rows: its live rows (may be 0).
__device__ __forceinline__ int32_t unit_keys(const Attn4Args& p, int u, int32_t& rows) {
  const int b = p.tiles == 1 ? u : u / p.tiles, s0 = (u - b * p.tiles) * p.qt;
  rows = min(live_rows(p.lens, b, p.seq) - s0, p.qt);
  if (rows <= 0) return 0;
  const int64_t n = seq_position(p.start[b], s0 + rows);
  return static_cast<int32_t>(min(max(n, int64_t{0}), static_cast<int64_t>(p.cap)));
}
__device__ __forceinline__ int unit_steps(const Attn4Args& p, int u) {
  int32_t rows;
  return u < p.units ? (unit_keys(p, u, rows) + kStep - 1) / kStep : 0;
}

// Which unit and piece the slot takes.  per: steps of a piece.  unit < 0: no work.
struct Piece {
  int unit, piece, pieces, first, per;  // first: slot of the unit's first piece
};
__device__ __forceinline__ Piece kv4_plan(const Attn4Args& p, int slot, int lane) {
  if (p.slots == 0) return {slot, 0, 1, slot, 1 << 26};
  // steps of a lane's units lane, lane + 64, ...: the first ones stay in a register
  const int st0 = unit_steps(p, lane);
  int total = wave_total_i(st0);
  for (int c = 64; c < p.units; c += 64) total += wave_total_i(unit_steps(p, c + lane));
  auto pieces_at = [&](int per) {
    const uint32_t d = static_cast<uint32_t>(per);
    int n = wave_total_i(lane < p.units ? max((st0 + d - 1) / d, 1u) : 0);
    for (int c = 64; c < p.units; c += 64)
      n += wave_total_i(c + lane < p.units ? max((unit_steps(p, c + lane) + d - 1) / d, 1u) : 0);
    return n;
  };
  // ceil(steps / per) summed over the units is at most total / per + units, so `hi` fits
  int lo = max((total + p.slots - 1) / p.slots, p.min_steps);
  int hi = max((total + p.slots - p.units - 1) / (p.slots - p.units), lo);
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (pieces_at(mid) <= p.slots) hi = mid;
    else lo = mid + 1;
  }
  const uint32_t per = static_cast<uint32_t>(hi);
  int at = slot;
  for (int c = 0; c < p.units; c += 64) {
    const int st = c == 0 ? st0 : unit_steps(p, c + lane);
    const int n = c + lane < p.units ? static_cast<int>(max((st + per - 1) / per, 1u)) : 0;
    const int upto = wave_scan_i(n), all = __builtin_amdgcn_readlane(upto, 63);
    if (at < all) {
      const int i = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= at));
      const int mine = __builtin_amdgcn_readlane(n, i), before = __builtin_amdgcn_readlane(upto, i) - mine;
      return {c + i, at - before, mine, slot - (at - before), hi};
    }
    at -= all;
  }
  return {-1, 0, 1, 0, 1};
}

// Parts of an fp32 value as bf16, largest first: 8 bits each.
template <int N>
__device__ __forceinline__ void bf16_parts(float v, __bf16 (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    out[i] = static_cast<__bf16>(v);
    v -= static_cast<float>(out[i]);
  }
}

template <int D, bool F32, int NW>
__global__ __launch_bounds__(NW * 64) void kv4_attention_kernel(Attn4Args p) {
  constexpr int KK = D / 32;            // MFMA k steps of a score tile
  constexpr int CW = D / 16;            // dimensions per lane of a V row = output tiles
  constexpr int GR = D / 32;            // scale groups of a row
  constexpr int QP = F32 ? 3 : 1, PP = F32 ? 3 : 2;  // bf16 parts of q and P
  constexpr int NT = NW * 64;
  constexpr int RH = D + 4;             // floats of a column in a record: m, l, 2 pad, o[D]
  extern __shared__ float smem[];       // per wave: o[columns][D], then m, l [columns]
  __shared__ bool last;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int j = lane & 15, h = lane >> 4;
  const int g = blockIdx.x % p.hkv;
  const Piece at = kv4_plan(p, static_cast<int>(blockIdx.x) / p.hkv, lane);
  if (at.unit < 0) return;
  const int unit = __builtin_amdgcn_readfirstlane(at.unit), piece = __builtin_amdgcn_readfirstlane(at.piece);
  const int pieces = __builtin_amdgcn_readfirstlane(at.pieces);
  const int b = unit / p.tiles, s0 = (unit - b * p.tiles) * p.qt;
  int32_t rows;
  const int32_t n_keys = unit_keys(p, unit, rows);
  if (rows <= 0) return;  // (a unit without live rows has one piece)
  const int cols = rows * p.G;
  const int nsteps = (n_keys + kStep - 1) / kStep;
  const int lo = piece * at.per, hi = min(lo + at.per, nsteps);
  const int my = hi - lo > wave ? (hi - lo - wave + NW - 1) / NW : 0;  // this wave's steps

  // column j: position s0 + j / G, head g G + j % G; columns past the last repeat column 0
  const int col = j < cols ? j : 0;
  const int qrow = b * p.seq + s0 + col / p.G;
  const int64_t qoff = (static_cast<int64_t>(qrow) * p.hq + g * p.G + col % p.G) * D + (D / 4) * h;
  const int32_t limit = static_cast<int32_t>(
      min(max(seq_position(p.start[b], s0 + col / p.G + 1), int64_t{0}), static_cast<int64_t>(p.cap)));  // keys of the column
  bf16x8_t qop[QP][KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    if constexpr (F32) {
      f32x4_t x[2];
      x[0] = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p.q) + qoff + 8 * kk);
      x[1] = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p.q) + qoff + 8 * kk + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        __bf16 t[QP];
        bf16_parts<QP>(x[e >> 2][e & 3], t);
#pragma unroll
        for (int i = 0; i < QP; ++i) qop[i][kk][e] = t[i];
      }
    } else {
      qop[0][kk] = *reinterpret_cast<const bf16x8_t*>(static_cast<const uint16_t*>(p.q) + qoff + 8 * kk);
    }
  }

  struct Buf {
    uint32_t k[2][KK];   // codes of the lane's D/4 dimensions of two keys
    uint32_t ks[2];      // their scale bytes
    uint32_t v[8];       // CW codes of 8 keys
    uint32_t vs[2][GR];  // all scale bytes of two runs of 4 keys
  };
  auto issue = [&](Buf& bf, int i) {
    const int64_t off = p.kv.Row(b, g, static_cast<int64_t>(kStep) * (lo + wave + i * NW));
    const uint8_t* kc = p.kc + off / 2;
    const uint8_t* vc = p.vc + off / 2;
    const uint8_t* ks = p.ks + off / 32;
    const uint8_t* vs = p.vs + off / 32;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      __builtin_memcpy(bf.k[tt], __builtin_assume_aligned(kc + (16 * tt + j) * (D / 2) + (D / 8) * h, D / 8), D / 8);
      bf.ks[tt] = ks[(16 * tt + j) * GR + h * GR / 4];
      __builtin_memcpy(bf.vs[tt], __builtin_assume_aligned(vs + (16 * tt + 4 * h) * GR, 4 * GR), 4 * GR);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint8_t* at_v = vc + (16 * (e >> 2) + 4 * h + (e & 3)) * (D / 2) + (CW / 2) * j;
      if constexpr (CW == 8) bf.v[e] = *reinterpret_cast<const uint32_t*>(at_v);
      else bf.v[e] = *reinterpret_cast<const uint16_t*>(at_v);
    }
  };

  float m_run = -INFINITY, l_run = 0.0f;
  int32_t nan_key = 0x7FFFFFFF;  // the first key with a NaN value in this lane's dimensions
  f32x4_t o[CW];  // O[column 4h + r][CW j + t]
#pragma unroll
  for (int t = 0; t < CW; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](const Buf& bf, int i) {
    const int32_t base = kStep * (lo + wave + i * NW) + 4 * h;  // key of score (0, 0)
    float sc[8];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
      const float s = e8m0_scale_or_nan(bf.ks[tt]);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        uint32_t w[4];
        fp4_to_bf16(bf.k[tt][kk], s, w);
        const bf16x8_t a = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int i2 = QP - 1; i2 >= 0; --i2) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qop[i2][kk], acc, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[4 * tt + r] = base + 16 * tt + r < limit ? acc[r] : -INFINITY;
    }
    float bm = sc[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) bm = fmaxf(bm, sc[e]);
    bm = fmaxf(bm, xor_lane<16>(bm, lane));
    bm = fmaxf(bm, xor_lane<32>(bm, lane));
    const float mn = fmaxf(m_run, bm * p.scale);
    if (__builtin_amdgcn_ballot_w64(mn > m_run) != 0) {
      const float cf = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - mn);
      l_run *= cf;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float cr = __shfl(cf, 16 * h + 4 * h + r);
#pragma unroll
        for (int t = 0; t < CW; ++t) o[t][r] *= cr;
      }
      m_run = mn;
    }
    // (a column without a live key subtracts 0: exp2(-inf) is 0)
    const float sub = m_run == -INFINITY ? 0.0f : -m_run;
    bf16x8_t pop[PP];
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], p.scale, sub));
      sum += v;
      __bf16 t[PP];
      bf16_parts<PP>(v, t);
#pragma unroll
      for (int i2 = 0; i2 < PP; ++i2) pop[i2][e] = t[i2];
    }
    l_run += sum;
    // V: a NaN value must not reach the product, where the probability 0 of a key behind some
    // column's last one would spread it: its group counts as zero and its key is noted.  Keys
    // at or past n_keys may hold anything.
    uint32_t sb[8], most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (GR == 4) sb[e] = (bf.vs[e >> 2][e & 3] >> (8 * (j >> 2))) & 0xFFu;
      else sb[e] = (bf.vs[e >> 2][(e & 3) >> 1] >> (16 * (e & 1) + 8 * (j >> 3))) & 0xFFu;
      most = max(most, sb[e]);
    }
    if (__builtin_amdgcn_ballot_w64(most >= kScaleNan) != 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int32_t key = base + 16 * (e >> 2) + (e & 3);
        if (sb[e] >= kScaleNan) {
          if (key < n_keys) nan_key = min(nan_key, key);
          sb[e] = 0;
        }
      }
    }
    uint32_t pr[8][CW / 2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float s = e8m0_scale(sb[e]);
      pr[e][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(bf.v[e], s, 0));
      pr[e][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(bf.v[e], s, 1));
      if constexpr (CW == 8) {
        pr[e][2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(bf.v[e], s, 2));
        pr[e][3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(bf.v[e], s, 3));
      }
    }
#pragma unroll
    for (int t = 0; t < CW; ++t) {
      uint32_t w[4];
#pragma unroll
      for (int e2 = 0; e2 < 4; ++e2) {
        const uint32_t a0 = pr[2 * e2][t >> 1], a1 = pr[2 * e2 + 1][t >> 1];
        w[e2] = (t & 1) ? ((a0 >> 16) | (a1 & 0xFFFF0000u)) : ((a0 & 0xFFFFu) | (a1 << 16));
      }
      const bf16x8_t vop = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
      for (int i2 = PP - 1; i2 >= 0; --i2) o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pop[i2], vop, o[t], 0, 0, 0);
    }
  };

  if (my > 0) {
    Buf ba, bb;
    issue(ba, 0);
    for (int i = 0; i < my; i += 2) {
      if (i + 1 < my) issue(bb, i + 1);
      compute(ba, i);
      if (i + 1 >= my) break;
      if (i + 2 < my) issue(ba, i + 2);
      compute(bb, i + 1);
    }
  }

  // NaN values: the columns that have the key, in its group's dimensions
  nan_key = min(nan_key, __shfl_xor(nan_key, 16));
  nan_key = min(nan_key, __shfl_xor(nan_key, 32));
  if (__builtin_amdgcn_ballot_w64(nan_key != 0x7FFFFFFF) != 0) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool bad = nan_key < __shfl(limit, 16 * h + 4 * h + r);
#pragma unroll
      for (int t = 0; t < CW; ++t) o[t][r] = bad ? __builtin_nanf("") : o[t][r];
    }
  }
  // the waves' states into LDS; column j's sum over its four lane groups
  l_run += xor_lane<16>(l_run, lane);
  l_run += xor_lane<32>(l_run, lane);
  const int ncol = p.qt * p.G;  // columns of a full unit
  float* so = smem + static_cast<int64_t>(wave) * ncol * D;
  float* sm = smem + static_cast<int64_t>(NW) * ncol * D + wave * 2 * 16;
  if (h == 0 && j < cols) {
    sm[j] = m_run;
    sm[16 + j] = l_run;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int c = 4 * h + r;
    if (c < cols) {
#pragma unroll
      for (int t = 0; t < CW; ++t) so[c * D + CW * j + t] = o[t][r];
    }
  }
  __syncthreads();
  const float* sm0 = smem + static_cast<int64_t>(NW) * ncol * D;
  // merge of the waves for 4 dimensions of a column
  auto wave_merge = [&](int c, int d0, float& mx, float& den, f32x4_t& acc) {
    mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sm0[w * 32 + c]);
    den = 0.0f;
    acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // (a NaN score leaves the maximum and makes its wave's sum NaN)
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float m = sm0[w * 32 + c], f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
      den = __builtin_fmaf(sm0[w * 32 + 16 + c], f, den);
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(smem + (static_cast<int64_t>(w) * ncol + c) * D + d0);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(v[e], f, acc[e]);
    }
  };
  auto write_out = [&](int c, int d0, float den, const f32x4_t& acc) {
    const int64_t to = (static_cast<int64_t>(b * p.seq + s0 + c / p.G) * p.hq + g * p.G + c % p.G) * D + d0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = den == 0.0f ? 0.0f : acc[e] / den;  // no keys: zeros; a NaN sum stays
      if constexpr (F32) static_cast<float*>(p.out)[to + e] = v;
      else static_cast<uint16_t*>(p.out)[to + e] = f32_to_bf16_bits(v);
    }
  };
  if (pieces == 1) {
    for (int t = threadIdx.x; t < cols * (D / 4); t += NT) {
      const int c = t / (D / 4), d0 = 4 * (t % (D / 4));
      float mx, den;
      f32x4_t acc;
      wave_merge(c, d0, mx, den, acc);
      write_out(c, d0, den, acc);
    }
    return;
  }
  const int rec_floats = ncol * RH;
  auto record = [&](int pc) {
    float* r = p.part + (static_cast<int64_t>(at.first + pc) * p.hkv + g) * rec_floats;
    return __builtin_amdgcn_make_buffer_rsrc(r, 0, rec_floats * 4, kRawBufferFlags);
  };
  {
    const __amdgpu_buffer_rsrc_t mine = record(piece);
    for (int t = threadIdx.x; t < cols * (D / 4); t += NT) {
      const int c = t / (D / 4), d0 = 4 * (t % (D / 4));
      float mx, den;
      f32x4_t acc;
      wave_merge(c, d0, mx, den, acc);
      if (d0 == 0)
        __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(mx), __float_as_uint(den)}, mine, c * RH * 4, 0, kCpolSc1);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, acc), mine, (c * RH + 4 + d0) * 4, 0, kCpolSc1);
    }
  }
  __builtin_amdgcn_s_waitcnt(0);  // acknowledged before the ticket
  __syncthreads();
  unsigned* ticket = p.tickets + at.first * p.hkv + g;
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<unsigned>(pieces - 1);
  __syncthreads();
  if (!last) return;
  // Merge in piece order, kBatch records in flight at a time.
  constexpr int kBatch = 8;
  for (int t = threadIdx.x; t < cols * (D / 4); t += NT) {
    const int c = t / (D / 4), d0 = 4 * (t % (D / 4));
    float mx = -INFINITY, den = 0.0f;
    f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int r0 = 0; r0 < pieces; r0 += kBatch) {
      u32x2_t ml[kBatch];
      u32x4_t ov[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const __amdgpu_buffer_rsrc_t rec = record(min(r0 + u, pieces - 1));
        ml[u] = __builtin_amdgcn_raw_buffer_load_b64(rec, c * RH * 4, 0, kCpolSc1);
        ov[u] = __builtin_amdgcn_raw_buffer_load_b128(rec, (c * RH + 4 + d0) * 4, 0, kCpolSc1);
      }
      float bm = mx;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) bm = fmaxf(bm, __uint_as_float(ml[u][0]));
      const float f0 = bm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mx - bm);
      den *= f0;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= f0;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (r0 + u >= pieces) break;
        const float f = bm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(__uint_as_float(ml[u][0]) - bm);
        den = __builtin_fmaf(__uint_as_float(ml[u][1]), f, den);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(__uint_as_float(ov[u][e]), f, acc[e]);
      }
      mx = bm;
    }
    write_out(c, d0, den, acc);
  }
  if (threadIdx.x == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr int kWaves = 4;
constexpr int kMinSteps = 4;  // fewest steps of a piece

// Slots of the planned grid (0: a block per unit and kv head without a plan).
int64_t Slots(int64_t units, int64_t hkv, int64_t capacity) {
  const int64_t target = 2 * DeviceCUs();
  if (units * hkv >= target || units * CeilDiv(capacity, kStep) >= (int64_t{1} << 30)) return 0;
  const int64_t slots = std::max(CeilDiv(target, hkv), 2 * units);
  return slots * hkv <= kMaxSlotHeads ? slots : 0;
}

int64_t WorkspaceBytes(int64_t units, int64_t qt, int64_t G, int64_t hkv, int64_t head_dim, int64_t capacity) {
  return kTicketBytes + Slots(units, hkv, capacity) * hkv * qt * G * (head_dim + 4) * 4;
}

template <int D, bool F32>
void Launch(const Attn4Args& p, hipStream_t s) {
  const int64_t grid = static_cast<int64_t>(p.slots > 0 ? p.slots : p.units) * p.hkv;
  const int lds = kWaves * (p.qt * p.G * D + 32) * 4;
  RecordLaunch(grid, kWaves * 64, lds, "kv4_attention<%s,d=%d,waves=%d,slots=%d>", F32 ? "f32" : "bf16", D, kWaves, p.slots);
  hipLaunchKernelGGL((kv4_attention_kernel<D, F32, kWaves>), dim3(static_cast<unsigned>(grid)), dim3(kWaves * 64), lds, s, p);
}

}  // namespace
}  // namespace am

using namespace am;

extern "C" int64_t am_gfx950_kv4_attention_workspace_bytes(int64_t batch, int64_t seq, int64_t hq, int64_t hkv,
                                                           int64_t head_dim, int64_t capacity) {
  if (batch <= 0 || seq <= 0 || hkv <= 0 || hq <= 0 || capacity <= 0 || hq % hkv != 0 || hq / hkv > 16) return kTicketBytes;
  const int64_t G = hq / hkv, qt = std::min<int64_t>(16 / G, seq);
  return WorkspaceBytes(batch * CeilDiv(seq, qt), qt, G, hkv, head_dim, capacity);
}

extern "C" am_status_code am_gfx950_kv4_attention(const am_gfx950_kv4_attention_args* a, void* stream) {
  AM_CHECK_ARG(a != nullptr, "kv4_attention: null args");
  AM_CHECK_ARG(a->dtype == AM_DT_F32 || a->dtype == AM_DT_BF16, "kv4_attention: dtype must be f32 or bf16");
  AM_CHECK_ARG(a->hq > 0 && a->hkv > 0 && a->hq % a->hkv == 0, "kv4_attention: q heads must be a multiple of kv heads");
  AM_CHECK_ARG(a->hq / a->hkv <= 16, "kv4_attention: at most 16 q heads per kv head");
  AM_CHECK_ARG(a->batch >= 0 && a->seq >= 0 && a->capacity > 0 && a->capacity < (int64_t{1} << 31) - 64, "kv4_attention: bad shape");
  AM_CHECK_ARG(a->batch <= 65535 && a->seq <= (1 << 24) && a->hkv <= 65536 && a->batch * a->seq <= (1 << 24) &&
                   a->batch * a->seq * a->hkv <= (1 << 24), "kv4_attention: too many query rows");
  AM_CHECK_ARG(std::isfinite(a->scale) && a->scale >= 0.0f, "kv4_attention: scale must be finite and not negative");
  if (a->batch == 0 || a->seq == 0) return AM_STATUS_OK;
  AM_CHECK_ARG(a->q && a->out && a->start_pos_dev, "kv4_attention: null pointer");
  AM_CHECK_ARG(Aligned16(a->q) && Aligned16(a->out), "kv4_attention: q and out must be 16-byte aligned");
  const int64_t cbs = a->batch > 1 ? a->cache_batch_stride : 0;
  if (auto st = CheckKv4Cache(a->k_codes, a->k_scales, a->v_codes, a->v_scales, a->batch, a->hkv, a->head_dim, a->capacity, cbs, a->pages);
      st != AM_STATUS_OK)
    return st;
  Attn4Args p{};
  if (auto st = MakeKvRows(a->pages, cbs, a->capacity, a->hkv, a->head_dim, &p.kv); st != AM_STATUS_OK) return st;
  if (auto st = CheckStreamDevice(AsStream(stream)); st != AM_STATUS_OK) return st;
  const int64_t G = a->hq / a->hkv, qt = std::min<int64_t>(16 / G, a->seq), tiles = CeilDiv(a->seq, qt), units = a->batch * tiles;
  AM_CHECK_ARG(a->workspace != nullptr && Aligned16(a->workspace) &&
                   a->workspace_bytes >= WorkspaceBytes(units, qt, G, a->hkv, a->head_dim, a->capacity),
               "kv4_attention: workspace missing, unaligned or too small");
  p.q = a->q, p.out = a->out;
  p.kc = a->k_codes, p.ks = a->k_scales, p.vc = a->v_codes, p.vs = a->v_scales;
  p.start = a->start_pos_dev, p.lens = a->seq_lens;
  p.tickets = static_cast<unsigned*>(a->workspace);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + kTicketBytes);
  p.batch = static_cast<int32_t>(a->batch), p.seq = static_cast<int32_t>(a->seq);
  p.hq = static_cast<int32_t>(a->hq), p.hkv = static_cast<int32_t>(a->hkv), p.G = static_cast<int32_t>(G);
  p.qt = static_cast<int32_t>(qt), p.tiles = static_cast<int32_t>(tiles), p.units = static_cast<int32_t>(units);
  p.cap = static_cast<int32_t>(a->capacity);
  p.slots = static_cast<int32_t>(Slots(units, a->hkv, a->capacity));
  p.min_steps = kMinSteps;
  p.scale = kLog2e * (a->scale > 0.0f ? a->scale : 1.0f / sqrtf(static_cast<float>(a->head_dim)));
  hipStream_t s = AsStream(stream);
  if (a->dtype == AM_DT_BF16) a->head_dim == 128 ? Launch<128, false>(p, s) : Launch<64, false>(p, s);
  else a->head_dim == 128 ? Launch<128, true>(p, s) : Launch<64, true>(p, s);
  AM_RETURN_IF_LAUNCH_FAILED("kv4_attention");
  return AM_STATUS_OK;
}
