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
//   * Up to eight columns (HALF): they stand twice in the tile, and each copy takes the softmax of one
//     of the step's two score tiles.
//   * exp2 with scale * log2(e) in the exponent's fma.  The running sums are rescaled only when a
//     score passed its column's reference by 2^4.
// Pieces: every block derives the same plan from the contexts (kv4_plan): pieces of at most
// `per` steps, the shortest with which all units fit the grid's slots.  The pieces of a unit
// write records with device-coherent stores and take a ticket; the last one merges them in
// piece order, so results do not depend on the schedule.  (The ordering that this relies on,
// relaxed device-coherent accesses around a wait, is the one of attention.hip's merge.)
//
// What bounds it (32 q / 8 kv heads, d = 128, bf16, us inside a graph): one token over 131072 keys (143 MB)
// 33.5, 4.3 TB/s; the same kernel without its arithmetic 32.2, without its loads 25.8.  A plain read of
// those bytes takes 24 with its launch (2), so the fixed part is the rest: the plan and the first load (2), the waves'
// merge, record and ticket (3), the last block's merge (3).  16 sequences at 4200-8320 keys,
// paged (111 MB) 28.8 (27, 24); one at 640 keys 6.5 (5.1, 6.4: a step's chain of conversion, product,
// softmax, product is its latency).

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
  int32_t few_slots, few_steps;  // slots for at most few_steps steps in all
  int32_t split;  // many rows: most pieces of a block's keys
  uint32_t tiles_inv;  // ceil(2^32 / tiles): unit / tiles by a multiplication (below 2^16 units)
  int32_t g_inv;  // ceil(2^16 / G): c / G = (c * g_inv) >> 16 for a column c < 32
  float scale;  // of the scores, times log2(e)
};

typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
constexpr int kCpolSc1 = 16;
constexpr int kRawBufferFlags = 0x00020000;
constexpr float kLog2e = 1.4426950408889634f;
// A column's reference m (a maximum that its scores passed by at most kSlack, in log2): P = 2^(s - m - kSlack)
// stays at most 1, and the accumulators are rescaled when a score passes m + kSlack, seldom after
// the first steps, instead of with every new maximum.
constexpr float kSlack = 4.0f;
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

// Value held by lane (lane ^ 8).
__device__ __forceinline__ float half_row(float v) {
  return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(__float_as_uint(v)), 0x128, 0xF, 0xF, false)));  // row_ror:8
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

__device__ __forceinline__ int unit_seq(const Attn4Args& p, int u) {
  return p.tiles == 1 ? u : static_cast<int>(__umulhi(static_cast<uint32_t>(u), p.tiles_inv));
}

// Keys of the unit's last live row, in [0, cap]; rows: its live rows (may be 0).
__device__ __forceinline__ int32_t unit_keys(const Attn4Args& p, int u, int32_t& rows) {
  const int b = unit_seq(p, u), s0 = (u - b * p.tiles) * p.qt;
  const int64_t start = p.start[b];  // (in flight beside the length)
  rows = min(live_rows(p.lens, b, p.seq) - s0, p.qt);
  if (rows <= 0) return 0;
  const int64_t n = seq_position(start, s0 + rows);
  return static_cast<int32_t>(min(max(n, int64_t{0}), static_cast<int64_t>(p.cap)));
}
__device__ __forceinline__ int unit_steps(const Attn4Args& p, int u) {
  int32_t rows;
  return u < p.units ? (unit_keys(p, u, rows) + kStep - 1) / kStep : 0;
}

// Contexts of up to kWholeSteps steps are one piece, others are cut into pieces of at least
// kMinSteps.
constexpr int kWholeSteps = 32;
constexpr int kMinSteps = 16;
constexpr int kFewSteps = 32;  // of a CU

// Which unit and piece the slot takes.  per: steps of a piece.  unit < 0: no work.
struct Piece {
  int unit, piece, pieces, first, per;  // first: slot of the unit's first piece
};
__device__ __forceinline__ Piece kv4_plan(const Attn4Args& p, int slot, int lane) {
  if (p.slots == 0) return {slot, 0, 1, slot, 1 << 26};
  // steps of a lane's units lane, lane + 64, ...: the first ones stay in a register
  const int st0 = unit_steps(p, lane);
  if (p.units == 1) {  // nothing to share out
    const uint32_t st = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(st0));
    const uint32_t per = st <= kWholeSteps ? kWholeSteps
                                           : max((st + p.slots - 1) / static_cast<uint32_t>(p.slots), static_cast<uint32_t>(p.min_steps));
    const int n = static_cast<int>(max((st + per - 1) / per, 1u));
    return {slot < n ? 0 : -1, slot, n, 0, static_cast<int>(per)};
  }
  int total = wave_total_i(st0);
  for (int c = 64; c < p.units; c += 64) total += wave_total_i(unit_steps(p, c + lane));
  // pieces of a unit of st steps: few steps stay whole (a merge costs more than they do)
  auto split = [&](int st, int per, int u) -> int {
    if (u >= p.units) return 0;
    return st <= kWholeSteps ? 1 : static_cast<int>((static_cast<uint32_t>(st) + per - 1) / static_cast<uint32_t>(per));
  };
  auto pieces_at = [&](int per) {
    int n = wave_total_i(split(st0, per, lane));
    for (int c = 64; c < p.units; c += 64) n += wave_total_i(split(unit_steps(p, c + lane), per, c + lane));
    return n;
  };
  // ceil(steps / per) summed over the units is at most total / per + units, so `hi` fits
  const int slots = total <= p.few_steps ? p.few_slots : p.slots;
  int lo = max((total + slots - 1) / slots, p.min_steps);
  int hi = max((total + slots - p.units - 1) / (slots - p.units), lo);
  for (int mid = lo; lo < hi; mid = (lo + hi) >> 1) {  // (equal contexts mostly fit at the first try)
    if (pieces_at(mid) <= slots) hi = mid;
    else lo = mid + 1;
  }
  int at = slot;
  for (int c = 0; c < p.units; c += 64) {
    const int st = c == 0 ? st0 : unit_steps(p, c + lane);
    const int n = split(st, hi, c + lane);
    const int upto = wave_scan_i(n), all = __builtin_amdgcn_readlane(upto, 63);
    if (at < all) {
      const int i = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= at));
      const int mine = __builtin_amdgcn_readlane(n, i), before = __builtin_amdgcn_readlane(upto, i) - mine;
      const int steps = __builtin_amdgcn_readlane(st, i);  // (in equal pieces of at most hi)
      return {c + i, at - before, mine, slot - (at - before), mine == 1 ? kWholeSteps + hi : (steps + mine - 1) / mine};
    }
    at -= all;
  }
  return {-1, 0, 1, 0, 1};
}

// A block barrier for LDS alone: global loads that nobody needs any more stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Row offsets, in elements, of the steps first, first + every, ... (up to last) of (b, g): KvRows::Row
// of a step's first key without a table read in front of its loads.  A lane holds the block-table
// entry of one of 64 visits; planes are one block without end.
struct StepWalk {
  const int32_t* table;
  int64_t block_elems, base;
  int32_t num_blocks, stride, shift, mask, step_elems, first, every, last, lane, loaded = -1, entry = 0;

  __device__ __forceinline__ StepWalk(const KvRows& kv, int64_t b, int64_t g, int lane_, int first_, int every_, int last_)
      : step_elems(kStep * kv.d), first(first_), every(every_), last(last_), lane(lane_) {
    if (kv.table == nullptr) {
      table = nullptr;
      block_elems = 0;
      base = kv.Row(b, g, 0);
      shift = 31;
      mask = 0x7FFFFFFF;
    } else {
      table = kv.table + b * kv.stride;
      block_elems = (static_cast<int64_t>(kv.hkv) << kv.shift) * kv.d;
      base = (g << kv.shift) * kv.d;
      shift = kv.shift - 5;
      mask = (1 << shift) - 1;
    }
    num_blocks = static_cast<int32_t>(min(kv.num_blocks, int64_t{0x7FFFFFFF}));
    stride = kv.stride;
  }
  __device__ __forceinline__ int step(int u) const { return min(first + u * every, last); }
  __device__ __forceinline__ int64_t operator()(int u) {
    const int t = step(u);
    if (table == nullptr) return base + static_cast<int64_t>(t) * step_elems;
    if ((u >> 6) != loaded) {  // (wave-uniform)
      loaded = u >> 6;
      const int32_t e = table[min(step((u & ~63) + lane) >> shift, stride - 1)];
      entry = min(max(e, 0), num_blocks - 1);  // entries outside the pool are clamped into it
    }
    return __builtin_amdgcn_readlane(entry, u & 63) * block_elems + base + static_cast<int64_t>(t & mask) * step_elems;
  }
};

// Parts of an fp32 value as bf16, largest first: 8 bits each.
template <int N>
__device__ __forceinline__ void bf16_parts(float v, __bf16 (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    out[i] = static_cast<__bf16>(v);
    v -= static_cast<float>(out[i]);
  }
}

// Two 8-wave blocks fit a CU (fp32 q: one): 128 registers a wave.
template <int D, bool F32, int NW, bool HALF>
__global__ __launch_bounds__(NW * 64, F32 ? 2 : 4) void kv4_attention_kernel(Attn4Args p) {
  constexpr int KK = D / 32;            // MFMA k steps of a score tile
  constexpr int CW = D / 16;            // dimensions per lane of a V row = output tiles
  constexpr int GR = D / 32;            // scale groups of a row
  constexpr int QP = F32 ? 3 : 1, PP = F32 ? 3 : 2;  // bf16 parts of q and P
  constexpr int SN = HALF ? 4 : 8;      // scores of a lane
  constexpr int NT = NW * 64;
  constexpr int RH = D + 4;             // floats of a column in a record: m, l, 2 pad, o[D]
  extern __shared__ float smem[];       // per wave: o[columns][D], then m, l [columns]
  __shared__ bool last;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int j = lane & 15, h = lane >> 4;
  const int g = blockIdx.x;
  const Piece at = kv4_plan(p, static_cast<int>(blockIdx.y), lane);
  if (at.unit < 0) return;
  const int unit = __builtin_amdgcn_readfirstlane(at.unit), piece = __builtin_amdgcn_readfirstlane(at.piece);
  const int pieces = __builtin_amdgcn_readfirstlane(at.pieces);
  const int b = unit_seq(p, unit), s0 = (unit - b * p.tiles) * p.qt;
  int32_t rows;
  const int32_t n_keys = unit_keys(p, unit, rows);
  if (rows <= 0) return;  // (a unit without live rows has one piece)
  const int cols = rows * p.G;
  const int nsteps = (n_keys + kStep - 1) / kStep;
  const int lo = piece * at.per, hi = min(lo + at.per, nsteps);
  const int my = hi - lo > wave ? (hi - lo - wave + NW - 1) / NW : 0;  // this wave's steps

  // column j: position s0 + j / G, head g G + j % G; columns past the last repeat column 0
  // (HALF: column j - 8 from the eighth on)
  const int jc = HALF ? j & 7 : j, col = jc < cols ? jc : 0, crow = (col * p.g_inv) >> 16;
  const int64_t qoff = (static_cast<int64_t>(b * p.seq + s0 + crow) * p.hq + g * p.G + col - crow * p.G) * D + (D / 4) * h;
  const int32_t limit = static_cast<int32_t>(
      min(max(seq_position(p.start[b], s0 + crow + 1), int64_t{0}), static_cast<int64_t>(p.cap)));  // keys of the column
  // the first column's: steps up to it need no mask
  const int32_t least = static_cast<int32_t>(
      min(max(seq_position(p.start[b], s0 + 1), int64_t{0}), static_cast<int64_t>(p.cap)));
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

  // One step's codes and scale bytes in registers.  K of the next step is loaded once this
  // step's scores are taken, V once its products are, so one of the two is always in flight
  // behind the other's work.  (A load past the wave's last step reads that step again: a branch
  // around it would make every wait count on the worse of its two sides.)
  uint32_t k_code[2][KK];   // the lane's D/4 dimensions of two keys
  uint32_t k_scale[2];      // their scale bytes
  uint32_t v_code[8];       // CW codes of 8 keys
  uint32_t v_scale[2][GR];  // all scale bytes of two runs of 4 keys
  StepWalk step_rows(p.kv, b, g, lane, lo + wave, NW, lo + wave + (my - 1) * NW);
  auto issue_k = [&](int64_t off) {
    const uint8_t* kc = p.kc + off / 2;
    const uint8_t* ks = p.ks + off / 32;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      __builtin_memcpy(k_code[tt], __builtin_assume_aligned(kc + (16 * tt + j) * (D / 2) + (D / 8) * h, D / 8), D / 8);
      k_scale[tt] = ks[(16 * tt + j) * GR + h * GR / 4];
    }
  };
  auto issue_v = [&](int64_t off) {
    const uint8_t* vc = p.vc + off / 2;
    const uint8_t* vs = p.vs + off / 32;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
      __builtin_memcpy(v_scale[tt], __builtin_assume_aligned(vs + (16 * tt + 4 * h) * GR, 4 * GR), 4 * GR);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint8_t* at_v = vc + (16 * (e >> 2) + 4 * h + (e & 3)) * (D / 2) + (CW / 2) * j;
      if constexpr (CW == 8) v_code[e] = *reinterpret_cast<const uint32_t*>(at_v);
      else v_code[e] = *reinterpret_cast<const uint16_t*>(at_v);
    }
  };

  float m_run = -INFINITY, l_run = 0.0f;
  int32_t nan_key = 0x7FFFFFFF;  // the first key with a NaN value in this lane's dimensions
  f32x4_t o[CW];  // O[column 4h + r][CW j + t]
#pragma unroll
  for (int t = 0; t < CW; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  if (my > 0) {
    const int64_t off = step_rows(0);
    issue_k(off);
    __builtin_amdgcn_sched_barrier(0);  // (in the loop's order: its waits count on the worse one)
    issue_v(off);
    __builtin_amdgcn_sched_barrier(0);
  }
  for (int i = 0; i < my; ++i) {
    const int64_t next = step_rows(i + 1);
    const int32_t first = kStep * (lo + wave + i * NW);  // key of the step
    const int32_t base = first + 4 * h;                  // of this lane's score (0, 0)
    f32x4_t acc[2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      acc[tt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      const float s = e8m0_scale_or_nan(k_scale[tt]);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        uint32_t w[4];
        fp4_to_bf16(k_code[tt][kk], s, w);
        const bf16x8_t a = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int i2 = QP - 1; i2 >= 0; --i2) acc[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qop[i2][kk], acc[tt], 0, 0, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    issue_k(next);
    __builtin_amdgcn_sched_barrier(0);
    float sc[SN];
#pragma unroll
    for (int e = 0; e < SN; ++e) sc[e] = HALF ? (j < 8 ? acc[0][e] : acc[1][e]) : acc[e >> 2][e & 3];
    if (first + kStep > least) {  // (wave-uniform) some column ends in this step
      int32_t key = base + (HALF ? 16 * (j >> 3) : 0);
      asm volatile("" : "+v"(key));  // (nothing of this in other steps)
#pragma unroll
      for (int e = 0; e < SN; ++e)
        if (key + 16 * (e >> 2) + (e & 3) >= limit) sc[e] = -INFINITY;
    }
    float bm = sc[0];
#pragma unroll
    for (int e = 1; e < SN; ++e) bm = fmaxf(bm, sc[e]);
    if constexpr (HALF) bm = fmaxf(bm, half_row(bm));
    bm = fmaxf(bm, xor_lane<16>(bm, lane));
    bm = fmaxf(bm, xor_lane<32>(bm, lane));
    const float mn = fmaxf(m_run, bm * p.scale);
    if (__builtin_amdgcn_ballot_w64(mn > m_run + kSlack) != 0) {
      if (__builtin_amdgcn_ballot_w64(m_run > -INFINITY) != 0) {  // (nothing to rescale before the first scores)
        const float cf = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - mn);
        l_run *= cf;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float cr = __shfl(cf, 16 * h + 4 * h + r);
#pragma unroll
          for (int t = 0; t < CW; ++t) o[t][r] *= cr;
        }
      }
      m_run = mn;
    }
    // (a column without a live key subtracts 0: exp2(-inf) is 0)
    const float sub = m_run == -INFINITY ? 0.0f : -kSlack - m_run;
    uint32_t pw[PP][4];
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < SN; e += 2) {
      float v0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], p.scale, sub));
      float v1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e + 1], p.scale, sub));
      sum += v0;
      sum += v1;
      if constexpr (!F32) {  // the first part cut off (a permute; the rounding conversion takes two issues), the second rounded
        const uint32_t u0 = __float_as_uint(v0), u1 = __float_as_uint(v1);
        pw[0][e / 2] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
        v0 -= __uint_as_float(u0 & 0xFFFF0000u);
        v1 -= __uint_as_float(u1 & 0xFFFF0000u);
      }
#pragma unroll
      for (int i2 = F32 ? 0 : 1; i2 < PP; ++i2) {
        const uint32_t w = __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<__bf16>(v0), static_cast<__bf16>(v1)});
        pw[i2][e / 2] = w;
        if (i2 + 1 < PP) {
          v0 -= __uint_as_float(w << 16);
          v1 -= __uint_as_float(w & 0xFFFF0000u);
        }
      }
    }
    if constexpr (HALF) {  // lanes of the first half take the other tile's from the second (whose operand rows are not used)
#pragma unroll
      for (int i2 = 0; i2 < PP; ++i2)
#pragma unroll
        for (int i = 0; i < 2; ++i) pw[i2][2 + i] = __float_as_uint(half_row(__uint_as_float(pw[i2][i])));
    }
    l_run += sum;
    // V: a NaN value must not reach the product, where the probability 0 of a key behind some
    // column's last one would spread it: its group counts as zero and its key is noted.  Keys
    // at or past n_keys may hold anything.
    uint32_t sb[8], most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (GR == 4) sb[e] = (v_scale[e >> 2][e & 3] >> (8 * (j >> 2))) & 0xFFu;
      else sb[e] = (v_scale[e >> 2][(e & 3) >> 1] >> (16 * (e & 1) + 8 * (j >> 3))) & 0xFFu;
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
    // two neighbouring dimensions (output tiles 2 t2, 2 t2 + 1) of the lane's 8 keys at a time
    auto tile_pair = [&]<int T2>() {
      uint32_t pr[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        pr[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v_code[e], e8m0_scale(sb[e]), T2));
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        uint32_t w[4];
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2)
          w[e2] = __builtin_amdgcn_perm(pr[2 * e2 + 1], pr[2 * e2], odd ? 0x07060302u : 0x05040100u);
        const bf16x8_t vop = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int i2 = PP - 1; i2 >= 0; --i2)
          o[2 * T2 + odd] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8_t, make_uint4(pw[i2][0], pw[i2][1], pw[i2][2], pw[i2][3])), vop, o[2 * T2 + odd], 0, 0, 0);
      }
    };
    tile_pair.template operator()<0>();
    tile_pair.template operator()<1>();
    if constexpr (CW == 8) {
      tile_pair.template operator()<2>();
      tile_pair.template operator()<3>();
    }
    __builtin_amdgcn_sched_barrier(0);
    issue_v(next);
    __builtin_amdgcn_sched_barrier(0);
  }

  // NaN values: the columns that have the key, in its group's dimensions
  if (__builtin_amdgcn_ballot_w64(nan_key != 0x7FFFFFFF) != 0) {
    nan_key = min(nan_key, __shfl_xor(nan_key, 16));
    nan_key = min(nan_key, __shfl_xor(nan_key, 32));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool bad = nan_key < __shfl(limit, 16 * h + 4 * h + r);
#pragma unroll
      for (int t = 0; t < CW; ++t) o[t][r] = bad ? __builtin_nanf("") : o[t][r];
    }
  }
  // the waves' states into LDS; column j's sum over its four lane groups
  if constexpr (HALF) l_run += half_row(l_run);
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
  lds_barrier();
  // From here on every instruction runs once per block, so the fetch of the code itself costs
  // more than its work: loops stay rolled where their latency allows it.
  const int items = cols * (D / 4);  // 4 dimensions of a column
  const float* sm0 = smem + NW * ncol * D;
  auto wave_merge = [&](int t, float& mx, float& den, f32x4_t& acc) {
    const int c = t / (D / 4);
    float m[NW], l[NW];
    f32x4_t v[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      m[w] = sm0[w * 32 + c];
      l[w] = sm0[w * 32 + 16 + c];
      v[w] = *reinterpret_cast<const f32x4_t*>(smem + w * ncol * D + 4 * t);
    }
    mx = m[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) mx = fmaxf(mx, m[w]);
    // (a NaN score leaves the maximum and makes its wave's sum NaN)
    const float top = mx == -INFINITY ? 0.0f : mx;
    den = 0.0f;
    acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(m[w] - top);
      den = __builtin_fmaf(l[w], f, den);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(v[w][e], f, acc[e]);
    }
  };
  auto write_out = [&](int t, float den, const f32x4_t& acc) {
    const int c = t / (D / 4), d0 = 4 * (t % (D / 4)), row = (c * p.g_inv) >> 16;
    const int64_t to = (static_cast<int64_t>(b * p.seq + s0 + row) * p.hq + g * p.G + c - row * p.G) * D + d0;
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;  // no keys: zeros; a NaN sum stays
    f32x4_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = acc[e] * inv;
    if constexpr (F32) {
      *reinterpret_cast<f32x4_t*>(static_cast<float*>(p.out) + to) = v;
    } else {
      const uint32_t w0 = f32_to_bf16_bits(v[0]) | (static_cast<uint32_t>(f32_to_bf16_bits(v[1])) << 16);
      const uint32_t w1 = f32_to_bf16_bits(v[2]) | (static_cast<uint32_t>(f32_to_bf16_bits(v[3])) << 16);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + to) = make_uint2(w0, w1);
    }
  };
  // the unit's records: piece_bytes apart (at most kMaxSlotHeads records in all: 35 MB)
  const int piece_bytes = p.hkv * ncol * RH * 4;
  const __amdgpu_buffer_rsrc_t all = __builtin_amdgcn_make_buffer_rsrc(
      p.part + (static_cast<int64_t>(at.first) * p.hkv + g) * (ncol * RH), 0, (pieces - 1) * piece_bytes + ncol * RH * 4, kRawBufferFlags);
  for (int t = threadIdx.x; t < items; t += NT) {
    float mx, den;
    f32x4_t acc;
    wave_merge(t, mx, den, acc);
    if (pieces == 1) {
      write_out(t, den, acc);
    } else {
      const int c = t / (D / 4), at_rec = piece * piece_bytes + c * RH * 4;
      if (t % (D / 4) == 0)
        __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(mx), __float_as_uint(den)}, all, at_rec, 0, kCpolSc1);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, acc), all, at_rec + 16 + 16 * (t % (D / 4)), 0, kCpolSc1);
    }
  }
  if (pieces == 1) return;
  __builtin_amdgcn_s_waitcnt(0);  // acknowledged before the ticket
  __syncthreads();
  unsigned* ticket = p.tickets + at.first * p.hkv + g;
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<unsigned>(pieces - 1);
  __syncthreads();
  if (!last) return;
  // Merge: the threads form teams of one thread per 4 dimensions of a column; team w takes
  // the pieces w, w + teams, ..., kBatch records in flight at a time, and the teams' sums meet
  // in LDS (NW / 2 teams fit where the waves' states were).  The order follows from the shape
  // alone.
  constexpr int kBatch = 4;
  const int teams = max(1, min(NT / items, NW / 2)), team = teams == 1 ? 0 : static_cast<int>(threadIdx.x) / items;
  float* state = smem;  // (the waves' states are consumed) per team and item: m, l, 2 pad, o[4]
  for (int t = threadIdx.x - team * items; t < items && team < teams; t += NT) {
    const int c = t / (D / 4);
    float mx = -INFINITY, den = 0.0f;
    f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
    int off = team * piece_bytes + c * RH * 4;  // (reads past the last record give zeros)
#pragma unroll 1
    for (int r0 = team; r0 < pieces; r0 += kBatch * teams) {
      u32x2_t ml[kBatch];
      u32x4_t ov[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        ml[u] = __builtin_amdgcn_raw_buffer_load_b64(all, off, 0, kCpolSc1);
        ov[u] = __builtin_amdgcn_raw_buffer_load_b128(all, off + 16 + 16 * (t % (D / 4)), 0, kCpolSc1);
        off += teams * piece_bytes;
      }
      float bm = mx, m[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        m[u] = r0 + u * teams < pieces ? __uint_as_float(ml[u][0]) : -INFINITY;
        bm = fmaxf(bm, m[u]);
      }
      const float top = bm == -INFINITY ? 0.0f : bm;  // (then every l and o is 0 or NaN, and its factor 0: NaN stays)
      const float f0 = __builtin_amdgcn_exp2f(mx - top);
      den *= f0;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= f0;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float f = __builtin_amdgcn_exp2f(m[u] - top);
        den = __builtin_fmaf(__uint_as_float(ml[u][1]), f, den);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(__uint_as_float(ov[u][e]), f, acc[e]);
      }
      mx = bm;
    }
    float* st = state + (team * items + t) * 8;
    *reinterpret_cast<f32x4_t*>(st) = f32x4_t{mx, den, 0.f, 0.f};
    *reinterpret_cast<f32x4_t*>(st + 4) = acc;
  }
  __syncthreads();
  for (int t = threadIdx.x; t < items; t += NT) {
    float mx = -INFINITY, den = 0.0f;
    f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int w = 0; w < teams; ++w) mx = fmaxf(mx, state[(w * items + t) * 8]);
    mx = mx == -INFINITY ? 0.0f : mx;
#pragma unroll 1
    for (int w = 0; w < teams; ++w) {
      const float* st = state + (w * items + t) * 8;
      const float f = __builtin_amdgcn_exp2f(st[0] - mx);
      den = __builtin_fmaf(st[1], f, den);
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(st + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(v[e], f, acc[e]);
    }
    write_out(t, den, acc);
  }
  if (threadIdx.x == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- many query rows ----
//
// A block owns 4 x 32 MFMA columns (32 / G query positions with their G heads per wave) of one
// kv head and walks the keys up to its last row's in tiles of 32, in two key groups of four
// waves that take every other tile and merge in LDS:
//   * A group's threads load the codes of a tile two intervals ahead, and convert them into one
//     of four LDS buffers, K and V row-major with padded rows, so that the operand reads meet no
//     bank twice.  A conversion serves all the group's columns.
//   * S^T = K Q^T on v_mfma_f32_32x32x16_bf16: lane (j, h) holds column j's scores of keys
//     8 (r >> 2) + 4 h + (r & 3), and these are the k slots of its P operand in
//     O^T = V^T P^T: P stays in its lane, and so does the softmax state of column j, whose
//     rescaling needs no exchange.  V^T's operand comes from the row-major tile through
//     ds_read_b64_tr_b16.
//   * bf16 q: P is f16, 11 bits where bf16 has 8 (its rounding is 1/8 of out's own), in one
//     product instead of the two of a bf16 split.  V is f16 as well: codes times 2^(e - E) with E
//     the largest scale of the group's 32 dimensions among the block's keys, less 13; the block
//     reads its keys' scale bytes once beforehand (1/17 of the cache).  P carries 2^15 so that its
//     small values stay normal (below 2^-25 of the largest they are held to 2^-36 of it).  Row sums are those of the
//     rounded P.  Where a group's scales differ by more than 2^16, a value that one row alone sees
//     could push another row's out of f16: such a block takes bf16 V and P in two bf16 parts (2048
//     rows at 6144 keys: 331 us for 261).
//   * fp32 q: three bf16 parts of q and P, bf16 V.
//   * Few row blocks share the CUs by pieces of their keys (planned on the device, as many as
//     leave each block a CU): records, ticket and merge as above.
//   * The same pass over the scales finds the first NaN value of each group; it enters the
//     products as zero and spoils the columns that see its key at the end.
// What bounds it: 2048 rows at 6144 keys take 261 us, 0.92 PFLOP/s; the matrix pipes are busy 36% of
// that, the VALU 45%, LDS 32%, and a wave waits a third of its time to issue or at barriers.  Without the
// staging (conversion and LDS writes) it takes 221, without the products with V 252, without the
// exponentials 253, without the operand reads 253.
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
constexpr int kWideWaves = 4;   // waves of columns of a block
// Tiles of a piece of a block's keys.  A merge costs about what 8 tiles do: 200 rows at 2000 keys
// (four pieces) 26 us, with at least 32 tiles (two) 33.
constexpr int kMinTiles = 16;
constexpr int64_t kMaxSplit = 16;
constexpr int kVTop = 140;      // exponent byte of the largest scale of V in f16: 6 * 2^13
constexpr int kNear = 17;        // f16: the largest scale byte of a group less (the smallest - 1)
constexpr float kPBias = 15.0f;  // log2 of the factor on P in f16

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}

__device__ __forceinline__ uint32_t min_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
// Lane 63: op over all lanes.
template <class F>
__device__ __forceinline__ uint32_t wave_last(uint32_t v, F op) {
  auto with = [&]<int CTRL, int ROWS>() {
    v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(v), static_cast<int>(v), CTRL, ROWS, 0xF, false)));
  };
  with.template operator()<0x111, 0xF>();
  with.template operator()<0x112, 0xF>();
  with.template operator()<0x114, 0xF>();
  with.template operator()<0x118, 0xF>();
  with.template operator()<0x142, 0xA>();
  with.template operator()<0x143, 0xC>();
  return v;
}
__device__ __forceinline__ uint32_t less_one_u16x2(uint32_t a) {
  return __builtin_bit_cast(uint32_t, static_cast<u16x2_t>(__builtin_bit_cast(u16x2_t, a) - u16x2_t{1, 1}));
}

template <int D, bool F32, bool SPLIT>
__global__ __launch_bounds__(512) void kv4_attention_wide_kernel(Attn4Args p) {
  constexpr int QW = kWideWaves, KS = 2;              // waves of a key group, key groups
  constexpr int GR = D / 32, SL = D / 8;              // scale groups and pieces (8 values) of a row
  constexpr int NT = QW * KS * 64, GT = QW * 64;      // threads of the block, of a key group
  constexpr int PC = kStep * SL;                      // pieces (8 values) of a tile of K, of V
  constexpr int NP = 2 * PC / GT;                     // pieces of a thread per tile
  constexpr int QP = F32 ? 3 : 1;                     // bf16 parts of q
  constexpr int DT = D / 32;
  constexpr int OW = DT * 16 + 2;                     // words of a lane's state
  static_assert(PC % GT == 0 && GT % SL == 0, "a thread's pieces are K or V by their number alone");
  // Rows are padded: the 16 keys of an operand read of K lie 16 bytes apart in the banks' 256, the
  // 4 keys of half a transposed read of V 64 bytes.  (Against 16-byte slots XORed by the key: one
  // address for all of a tile's reads, the rest is their immediate offset.)
  constexpr int KR = 2 * D + 16, VR = 2 * D + 64;     // bytes of a row of K, of V
  constexpr int kBufBytes = kStep * (KR + VR);
  constexpr int NB = 4;                               // buffers of a key group
  constexpr int kSmem = std::max(KS * NB * kBufBytes, (KS - 1) * QW * OW * 256);
  static_assert(NT == 512, "two waves per SIMD, one of each half");
  __shared__ __align__(16) uint8_t smem_w[kSmem];     // per key group and buffer: K, V
  __shared__ uint32_t s_top[GR], s_low[GR];           // largest and smallest scale of V
  __shared__ int32_t s_nan[GR];                       // first key with a NaN value
  __shared__ bool s_last;

  const int kg = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / GT);
  const int tid = static_cast<int>(threadIdx.x) - kg * GT, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 31, h = lane >> 5;
  // kv head fastest, then the row blocks of all sequences, last (longest) first
  const int g = blockIdx.x;
  const int unit = p.units - 1 - static_cast<int>(blockIdx.y), b = unit_seq(p, unit);
  const int s0 = (unit - b * p.tiles) * (QW * p.qt);
  const int live = min(live_rows(p.lens, b, p.seq) - s0, QW * p.qt);  // live rows of the block
  if (live <= 0) return;
  auto keys_of = [&](int row) {  // keys of row s0 + row
    return static_cast<int32_t>(min(max(seq_position(p.start[b], s0 + row + 1), int64_t{0}), static_cast<int64_t>(p.cap)));
  };
  // the block's piece: tiles [tlo, thi) of its last row's keys
  const int all_tiles = (keys_of(live - 1) + kStep - 1) / kStep;
  int pieces = 1, piece = 0, tlo = 0, thi = all_tiles;
  int32_t kend = keys_of(live - 1);
  if constexpr (SPLIT) {
    pieces = max(min(all_tiles / kMinTiles, p.split), 1);
    piece = static_cast<int>(blockIdx.z);
    if (piece >= pieces) return;
    const int per = ((all_tiles + pieces - 1) / pieces + KS - 1) / KS * KS;
    tlo = min(piece * per, all_tiles);
    thi = min(tlo + per, all_tiles);
    kend = min(kend, kStep * thi);  // (no key of another piece counts)
  }
  const int ntiles = thi - tlo;

  // column j: position s0 + wave qt + j / G, head g G + j % G; columns behind the live rows
  // repeat the last row
  const int wrow = wave * p.qt;
  const int jrow = min((j * p.g_inv) >> 16, p.qt - 1), jhead = min(j - jrow * p.G, p.G - 1);
  const int row = min(wrow + jrow, live - 1);
  const bool mine = j < p.qt * p.G && wrow + jrow < live;
  const int64_t qrow = (static_cast<int64_t>(b * p.seq + s0 + row) * p.hq + g * p.G + jhead) * D;
  const int32_t limit = min(keys_of(row), kend), least = min(keys_of(wrow), kend);
  bf16x8_t qop[QP][D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    if constexpr (F32) {
      const f32x4_t* qp = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p.q) + qrow + 16 * kk + 8 * h);
      const f32x4_t x[2] = {qp[0], qp[1]};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        __bf16 t[QP];
        bf16_parts<QP>(x[e >> 2][e & 3], t);
#pragma unroll
        for (int i = 0; i < QP; ++i) qop[i][kk][e] = t[i];
      }
    } else {
      qop[0][kk] = *reinterpret_cast<const bf16x8_t*>(static_cast<const uint16_t*>(p.q) + qrow + 16 * kk + 8 * h);
    }
  }

  if constexpr (F32) {  // (the parts stay in registers: the compiler would split q again in every tile)
#pragma unroll
    for (int i = 0; i < QP; ++i)
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) asm volatile("" : "+v"(qop[i][kk]));
  }

  // Piece c of the thread: K pieces first, then V, in steps of GT / SL keys; its slot is the
  // same in all.  The row offset of the tile after is looked up one load earlier (a
  // block-table entry arrives meanwhile).
  constexpr int NK = PC / GT;  // K pieces of a thread
  const int psl = tid % SL, pkey0 = tid / SL;
  auto piece_is_v = [&](int c) { return c >= NK; };
  auto piece_key = [&](int c) { return pkey0 + c % NK * (GT / SL); };
  // (scales as whole words, whose byte is taken at the store: a byte load is extended at once,
  // which waits for it)
  uint32_t code[NP], scale[NP];
  auto scale_byte = [&](int c) { return (scale[c] >> (8 * ((piece_key(c) * GR + psl / 4) & 3))) & 0xFFu; };
  StepWalk tile_off(p.kv, b, g, lane, tlo + kg, KS, thi - 1);
  const uint32_t code_at = static_cast<uint32_t>(pkey0 * (D / 2) + 4 * psl);
  const uint32_t scale_at = static_cast<uint32_t>((pkey0 * GR + psl / 4) & ~3);
  auto load_tile = [&](int64_t off) {
    // (descriptors of the tile: the address arithmetic is scalar)
    auto tile = [&](const uint8_t* base, int64_t at, int bytes) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base + at), 0, bytes, kRawBufferFlags);
    };
    const uint64_t uoff = static_cast<uint64_t>(off);
    const auto kc = tile(p.kc, uoff >> 1, kStep * D / 2), ks = tile(p.ks, uoff >> 5, kStep * GR);
    const auto vc = tile(p.vc, uoff >> 1, kStep * D / 2), vs = tile(p.vs, uoff >> 5, kStep * GR);
#pragma unroll
    for (int c = 0; c < NP; ++c) {
      const uint32_t keys = c % NK * (GT / SL);
      code[c] = __builtin_amdgcn_raw_buffer_load_b32(piece_is_v(c) ? vc : kc, code_at + keys * (D / 2), 0, 0);
      scale[c] = __builtin_amdgcn_raw_buffer_load_b32(piece_is_v(c) ? vs : ks, scale_at + keys * GR, 0, 0);
    }
  };
  // every key group goes through as many tiles as the first (those past the last key's hold
  // no live key), so that all threads meet at the same barriers
  const int nu = (ntiles + KS - 1) / KS;
  int64_t next_off = 0;
  if (nu > 0) {
    load_tile(tile_off(0));
    next_off = tile_off(1);
  }

  // the block's scales of V: the largest, the smallest (but for 0, the scale of zeros) and the first
  // NaN of each group
  if (threadIdx.x < GR) {
    s_top[threadIdx.x] = 0;
    s_low[threadIdx.x] = 0xFFFF;
    s_nan[threadIdx.x] = 0x7FFFFFFF;
  }
  __syncthreads();
  {
    constexpr int PS = 2 * GR;          // 16-byte pieces of a step's scales
    constexpr int KW = 4 / GR;          // keys of a word
    auto scan = [&](auto&& each) {      // each(word, its first key)
      for (int i = threadIdx.x; i < ntiles * PS; i += NT) {
        const int step = tlo + i / PS, part = i % PS;
        const uint4 v = *reinterpret_cast<const uint4*>(p.vs + p.kv.Row(b, g, static_cast<int64_t>(kStep) * step) / 32 + 16 * part);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = kStep * step + (4 * part + e) * KW;
          each(w[e] & (key >= kend ? 0u : (KW == 2 && key + 1 >= kend) ? 0xFFFFu : ~0u), key);
        }
      }
    };
    // two bytes of each word as 16-bit values; the smallest less one, so that 0 is no value
    uint32_t top[2] = {0, 0}, low[2] = {~0u, ~0u};
    scan([&](uint32_t w, int) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t x = (w >> (8 * i)) & 0x00FF00FFu;
        top[i] = max_u16x2(top[i], x);
        low[i] = min_u16x2(low[i], less_one_u16x2(x));
      }
    });
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = wave_last(top[i], [](uint32_t a, uint32_t b) { return max_u16x2(a, b); });
      low[i] = wave_last(low[i], [](uint32_t a, uint32_t b) { return min_u16x2(a, b); });
    }
    if (lane == 63) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        atomicMax(&s_top[e % GR], (top[e & 1] >> (8 * (e & 2))) & 0xFFFFu);
        atomicMin(&s_low[e % GR], (low[e & 1] >> (8 * (e & 2))) & 0xFFFFu);
      }
    }
    __syncthreads();
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < GR; ++e) any = max(any, s_top[e]);
    if (any >= kScaleNan) {  // the largest again, byte by byte (block-uniform)
      __syncthreads();
      if (threadIdx.x < GR) s_top[threadIdx.x] = 0;
      __syncthreads();
      scan([&](uint32_t w, int key) {
        for (int e = 0; e < 4; ++e) {
          const uint32_t x = (w >> (8 * e)) & 0xFFu;
          if (x >= kScaleNan) atomicMin(&s_nan[e % GR], key + e / GR);
          else atomicMax(&s_top[e % GR], x);
        }
      });
      __syncthreads();
    }
  }
  bool any_nan = false;
#pragma unroll
  for (int e = 0; e < GR; ++e) any_nan = any_nan || __builtin_amdgcn_readfirstlane(s_nan[e]) != 0x7FFFFFFF;
  bool near = true;  // (block-uniform) the groups' scales lie close enough for f16
#pragma unroll
  for (int e = 0; e < GR; ++e) near = near && static_cast<int>(s_top[e]) - static_cast<int>(s_low[e]) <= kNear;

  // The walk over the keys.  H: V and P in f16.
  auto run = [&]<bool H>() {
  constexpr int PP = H ? 1 : F32 ? 3 : 2;  // parts of P

  // (buffer of the group's u-th tile)
  auto tile_k = [&](int u) { return smem_w + (kg * NB + (u & (NB - 1))) * kBufBytes; };
  auto tile_v = [&](int u) { return tile_k(u) + kStep * KR; };
  const int v_add = kVTop - static_cast<int>(s_top[psl / 4]);  // to a V piece's scale byte
  // V pieces that count as zero: NaN values, and keys past the last
  auto clear_dead = [&](int u) {
    const int t = tlo + u * KS + kg;
    if (any_nan || kStep * t + kStep > kend) {  // (block-uniform)
#pragma unroll
      for (int c = NK; c < NP; ++c)
        if (scale_byte(c) >= kScaleNan || kStep * t + piece_key(c) >= kend) code[c] = scale[c] = 0;
    }
  };
  auto store_tile = [&](int u) {
#pragma unroll
    for (int c = 0; c < NP; ++c) {
      const int key = piece_key(c);
      const uint32_t sb = scale_byte(c);
      uint32_t w[4];
      if (!piece_is_v(c)) {
        fp4_to_bf16(code[c], e8m0_scale_or_nan(sb), w);
        *reinterpret_cast<uint4*>(tile_k(u) + key * KR + 16 * psl) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        int e = static_cast<int>(sb);
        if constexpr (H) e = max(e + v_add, 0);  // (a group of zeros may lie below)
        const float s = e8m0_scale(static_cast<uint32_t>(e));
        if constexpr (!H) {
          fp4_to_bf16(code[c], s, w);
        } else {
          w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code[c], s, 0));
          w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code[c], s, 1));
          w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code[c], s, 2));
          w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code[c], s, 3));
        }
        *reinterpret_cast<uint4*>(tile_v(u) + key * VR + 16 * psl) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  };

  float m_run = -INFINITY, l_run = 0.0f;
  f32x16_t o[DT];  // O^T[32 dt + 8 (r >> 2) + 4 h + (r & 3)][column j]
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;

  f32x16_t acc;                                  // scores
  uint32_t pw[PP][2][4];                         // P operand: parts, chunks of 16 keys
  auto softmax = [&](int u) {
    const int t = tlo + u * KS + kg;
    if (kStep * t + kStep > least) {  // some column of the wave ends in or before this tile
      asm volatile("");               // (a branch: not selects in every tile)
      const int32_t base = kStep * t + 4 * h;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (base + 8 * (r >> 2) + (r & 3) >= limit) acc[r] = -INFINITY;
    }
    float bm = acc[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) bm = fmaxf(bm, acc[r]);
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(bm), __float_as_uint(bm), false, false);
    bm = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
    const float mn = fmaxf(m_run, bm * p.scale);
    if (__builtin_amdgcn_ballot_w64(mn > m_run + kSlack) != 0) {
      const float cf = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - mn);
      l_run *= cf;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= cf;
      m_run = mn;
    }
    const float sub = (H ? kPBias : 0.0f) - kSlack - (m_run == -INFINITY ? 0.0f : m_run);
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      float v0 = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[r], p.scale, sub));
      float v1 = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[r + 1], p.scale, sub));
      if constexpr (!H) {
        l_run += v0;
        l_run += v1;
#pragma unroll
        for (int i = 0; i < PP; ++i) {
          const uint32_t w = __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<__bf16>(v0), static_cast<__bf16>(v1)});
          pw[i][r / 8][(r % 8) / 2] = w;
          v0 -= __uint_as_float(w << 16);
          v1 -= __uint_as_float(w & 0xFFFF0000u);
        }
      } else {
        const f16x2_t v = {static_cast<_Float16>(v0), static_cast<_Float16>(v1)};
        l_run = __builtin_amdgcn_fdot2(v, f16x2_t{static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)}, l_run, false);
        pw[0][r / 8][(r % 8) / 2] = __builtin_bit_cast(uint32_t, v);
      }
    }
  };
  // A operand of V^T: lane (row, h) of output tile dt and k slots of chunk c: keys 16 c + 8 q +
  // 4 h .. +4, which the 16 lanes of a transposed read bring as 4 keys x 16 dimensions
  const int tkey = 4 * h + ((lane & 15) >> 2), tdim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  auto read_v = [&](int u, int c, s16x4_t (&part)[DT][2]) {
    const uint8_t* vt = tile_v(u) + tkey * VR + 2 * tdim;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint8_t* at = vt + (16 * c + 8 * q) * VR + 64 * dt;
        part[dt][q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(at));
      }
  };
  auto products = [&](int c, const s16x4_t (&part)[DT][2]) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const auto a = __builtin_shufflevector(part[dt][0], part[dt][1], 0, 1, 2, 3, 4, 5, 6, 7);
      if constexpr (!H) {
#pragma unroll
        for (int i = PP - 1; i >= 0; --i)
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8_t, a),
              __builtin_bit_cast(bf16x8_t, make_uint4(pw[i][c][0], pw[i][c][1], pw[i][c][2], pw[i][c][3])), o[dt], 0, 0, 0);
      } else {
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
            __builtin_bit_cast(f16x8_t, a),
            __builtin_bit_cast(f16x8_t, make_uint4(pw[0][c][0], pw[0][c][1], pw[0][c][2], pw[0][c][3])), o[dt], 0, 0, 0);
      }
    }
  };
  auto read_k = [&](int u, int kk) {
    return *reinterpret_cast<const bf16x8_t*>(tile_k(u) + j * KR + 16 * h + 32 * kk);
  };
  auto score = [&](int kk, bf16x8_t k) {
#pragma unroll
    for (int i = QP - 1; i >= 0; --i) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, qop[i][kk], acc, 0, 0, 0);
  };
  // M of tile u: P V of tile u - 1 and K Q^T of tile u.  Its operands are read ahead, so that
  // the products do not wait for LDS (without H there are no registers for that: read_m does nothing).
  s16x4_t vop[H ? 2 : 1][DT][2];
  bf16x8_t kop[H ? D / 16 : 1];
  auto read_m = [&](int u, bool pv, bool qk) {
    if constexpr (H) {
      if (pv) {
        read_v(u - 1, 0, vop[0]);
        read_v(u - 1, 1, vop[1]);
      }
      if (qk) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) kop[kk] = read_k(u, kk);
      }
    }
  };
  auto multiply = [&](int u, bool pv, bool qk) {
    if (pv) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if constexpr (!H) read_v(u - 1, c, vop[0]);
        products(c, vop[H ? c : 0]);
      }
    }
    if (qk) {
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        if constexpr (H) score(kk, kop[kk]);
        else score(kk, read_k(u, kk));
      }
    }
  };

  // A wave alternates between vector work (V: the softmax of its group's tile u, and its share
  // of the staging) and products (M: P V of tile u, K Q^T of tile u + 1).  Between two barriers
  // the first group does V then M, and the second, which shares every SIMD with it, M (of the
  // tile before) then V: while one wave of a SIMD multiplies the other exponentiates.  In phase
  // (every wave V then M, a barrier a tile) 2048 rows at 6144 keys took 329 us, so 300 at the time.
  // Interval u stores tile u + 2.  K of tile x is read in interval x - 1 (ahead of x in the
  // second group), its V in x or x + 1: four buffers.
  // (kg as a lane value: as a scalar one the loops' registers spill)
  const bool second = threadIdx.x >= GT;
  auto interval_end = [&]() {  // (nothing moves over it: the scheduler would mix the intervals' arithmetic)
    __builtin_amdgcn_sched_barrier(0);
    lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  if (nu > 0) {
    // (Tiles past the last are the last one again, into buffers that are free: no branch, so that
    // the softmax and the staging mix.)
    auto load_next = [&](int u) {
      load_tile(next_off);
      next_off = tile_off(u + 1);
    };
    auto vector_work = [&](int u) {
      clear_dead(u + 2);
      softmax(u);
      store_tile(u + 2);
      load_next(u + 3);
    };
    clear_dead(0);
    store_tile(0);
    load_next(1);
    clear_dead(1);
    store_tile(1);
    load_next(2);
    interval_end();
    read_m(0, false, true);
    multiply(0, false, true);
    if (second) {
      vector_work(0);
      read_m(1, true, nu > 1);
      interval_end();
      for (int u = 1; u < nu; ++u) {
        multiply(u, true, true);
        __builtin_amdgcn_sched_barrier(0);
        vector_work(u);
        read_m(u + 1, true, true);  // (the last K is not used: a tile's buffer all the same)
        interval_end();
      }
    } else {
      for (int u = 0; u + 1 < nu; ++u) {
        read_m(u + 1, true, true);
        __builtin_amdgcn_sched_barrier(0);
        vector_work(u);
        __builtin_amdgcn_sched_barrier(0);
        multiply(u + 1, true, true);
        interval_end();
      }
      read_m(nu, true, false);
      vector_work(nu - 1);
      interval_end();
    }
    multiply(nu, true, false);
  }

  // column j's sum over its two lanes, and the key groups' states
  l_run += xor_lane<32>(l_run, lane);
  {
    lds_barrier();  // both groups are done with their tiles
    float* rec = reinterpret_cast<float*>(smem_w) + wave * OW * 64 + lane;
    if (kg > 0) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) rec[(dt * 16 + r) * 64] = o[dt][r];
      rec[DT * 16 * 64] = m_run;
      rec[(DT * 16 + 1) * 64] = l_run;
    }
    __syncthreads();
    if (kg > 0 && (!SPLIT || pieces == 1)) return;
    if (kg == 0) {
      const float m2 = rec[DT * 16 * 64], l2 = rec[(DT * 16 + 1) * 64];
      const float mn = fmaxf(m_run, m2), top = mn == -INFINITY ? 0.0f : mn;
      const float f1 = __builtin_amdgcn_exp2f(m_run - top), f2 = __builtin_amdgcn_exp2f(m2 - top);
      l_run = l_run * f1 + l2 * f2;
      m_run = mn;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = o[dt][r] * f1 + rec[(dt * 16 + r) * 64] * f2;
      }
    }
  }
  // V's units back, and the NaN values
  auto in_units = [&](int dt, float v) {
    if constexpr (H) v = __builtin_ldexpf(v, static_cast<int>(s_top[dt]) - kVTop);
    return s_nan[dt] < limit ? __builtin_nanf("") : v;
  };
  auto write_out = [&](int dt, int r4, const f32x4_t& v) {
    const int64_t to = qrow + 32 * dt + 8 * r4 + 4 * h;
    if constexpr (F32) {
      *reinterpret_cast<f32x4_t*>(static_cast<float*>(p.out) + to) = v;
    } else {
      const uint32_t w0 = f32_to_bf16_bits(v[0]) | (static_cast<uint32_t>(f32_to_bf16_bits(v[1])) << 16);
      const uint32_t w1 = f32_to_bf16_bits(v[2]) | (static_cast<uint32_t>(f32_to_bf16_bits(v[3])) << 16);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + to) = make_uint2(w0, w1);
    }
  };
  if (!SPLIT || pieces == 1) {
    if (!mine) return;
    const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        f32x4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = in_units(dt, o[dt][4 * r4 + e] * inv);
        write_out(dt, r4, v);
      }
    return;
  }
  // Pieces: records as the other kernel's, a lane's state in 16-byte parts, with the reference
  // that P = 2^(s - m) has; the last piece's block merges them in order, a key group half of the dimensions.
  if constexpr (SPLIT) {
    constexpr int kRecBytes = OW * 64 * 4 * QW;
    const int slot = unit * p.hkv + g;
    const __amdgpu_buffer_rsrc_t all = __builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<uint8_t*>(p.part) + static_cast<int64_t>(slot) * p.split * kRecBytes, 0, pieces * kRecBytes, kRawBufferFlags);
    const int mine_at = wave * OW * 64 * 4 + lane * 16, ml_at = wave * OW * 64 * 4 + DT * 16 * 64 * 4 + lane * 8;
    if (kg == 0) {
      const float ref = m_run + (kSlack - (H ? kPBias : 0.0f));
      __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(ref), __float_as_uint(l_run)}, all, piece * kRecBytes + ml_at, 0, kCpolSc1);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          f32x4_t v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = in_units(dt, o[dt][4 * r4 + e]);
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), all, piece * kRecBytes + mine_at + (dt * 4 + r4) * 1024, 0, kCpolSc1);
        }
    }
    __builtin_amdgcn_s_waitcnt(0);  // acknowledged before the ticket
    __syncthreads();
    if (threadIdx.x == 0)
      s_last = __hip_atomic_fetch_add(p.tickets + slot, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<unsigned>(pieces - 1);
    __syncthreads();
    if (!s_last) return;
    float top = -INFINITY;
#pragma unroll 4
    for (int q = 0; q < pieces; ++q)
      top = fmaxf(top, __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(all, q * kRecBytes + ml_at, 0, kCpolSc1)));
    top = top == -INFINITY ? 0.0f : top;
    constexpr int HD = DT / KS;  // output tiles of a key group
    f32x4_t acc2[HD * 4];
    float den = 0.0f;
#pragma unroll
    for (int i = 0; i < HD * 4; ++i) acc2[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int q = 0; q < pieces; ++q) {
      const u32x2_t ml = __builtin_amdgcn_raw_buffer_load_b64(all, q * kRecBytes + ml_at, 0, kCpolSc1);
      u32x4_t w[HD * 4];
#pragma unroll
      for (int i = 0; i < HD * 4; ++i) w[i] = __builtin_amdgcn_raw_buffer_load_b128(all, q * kRecBytes + mine_at + (kg * HD * 4 + i) * 1024, 0, kCpolSc1);
      const float f = __builtin_amdgcn_exp2f(__uint_as_float(ml[0]) - top);
      den = __builtin_fmaf(__uint_as_float(ml[1]), f, den);
#pragma unroll
      for (int i = 0; i < HD * 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc2[i][e] = __builtin_fmaf(__uint_as_float(w[i][e]), f, acc2[i][e]);
    }
    if (mine) {
      const float inv = den == 0.0f ? 0.0f : 1.0f / den;
#pragma unroll
      for (int i = 0; i < HD * 4; ++i) {
        f32x4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc2[i][e] * inv;
        write_out(kg * HD + i / 4, i % 4, v);
      }
    }
    if (threadIdx.x == 0) __hip_atomic_store(p.tickets + slot, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  };
  if constexpr (F32) {
    run.template operator()<false>();
  } else {
    if (near) run.template operator()<true>();
    else run.template operator()<false>();
  }
}

constexpr int kWaves = 8;
constexpr int64_t kMaxRows = 65535;  // query rows of a call

// Slots of the planned grid (0: a block per unit and kv head without a plan).
int64_t Slots(int64_t units, int64_t hkv, int64_t capacity) {
  const int64_t cus = DeviceCUs(), target = 4 * units * hkv < cus ? cus : 2 * cus;
  if (units * hkv >= target || units * CeilDiv(capacity, kStep) >= (int64_t{1} << 30)) return 0;
  const int64_t slots = std::max(CeilDiv(target, hkv), 2 * units);
  return slots * hkv <= kMaxSlotHeads ? slots : 0;
}

// The kernel for many rows: its blocks and the most pieces of a block's keys that leave a CU to each.
struct Wide {
  int64_t tiles, blocks, split;
};
Wide WidePlan(int64_t batch, int64_t seq, int64_t G, int64_t hkv) {
  const int64_t tiles = CeilDiv(seq, kWideWaves * (32 / G)), blocks = batch * tiles * hkv;
  return {tiles, blocks, std::min(std::max<int64_t>(DeviceCUs() / blocks, 1), kMaxSplit)};
}

// The kernel for many rows where a sequence fills at least one of its blocks and the blocks make
// up 3/16 of the CUs.  32 q / 8 kv heads, d = 128 (us, this kernel / the other): 256 blocks (1000 rows at
// 0) 27 / 39; 128 blocks (512 rows) at 0 18.5 / 19.6, at 6144 75 / 112; 56 blocks (200 rows) at 0
// 12.5 / 10.3, at 2000 26 / 36, at 5000 39 / 57; 32 blocks (100 rows) at 0 10.6 / 6.9.  fp32 q: 80 blocks
// (300 rows) at 2048 44 / 52.  16 sequences of one row at 4200-8320 keys (128 blocks of one live
// column group in eight) 273 / 31.
bool ManyRows(int64_t batch, int64_t seq, int64_t G, int64_t hkv) {
  return seq >= kWideWaves * (32 / G) && 16 * WidePlan(batch, seq, G, hkv).blocks >= 3 * DeviceCUs();
}

int64_t WorkspaceBytes(int64_t batch, int64_t seq, int64_t G, int64_t hkv, int64_t head_dim, int64_t capacity) {
  if (ManyRows(batch, seq, G, hkv)) {
    const Wide w = WidePlan(batch, seq, G, hkv);
    return kTicketBytes + (w.split > 1 ? w.blocks * w.split * kWideWaves * 64 * (head_dim / 2 + 2) * 4 : 0);
  }
  const int64_t qt = std::min<int64_t>(16 / G, seq);
  return kTicketBytes + Slots(batch * CeilDiv(seq, qt), hkv, capacity) * hkv * qt * G * (head_dim + 4) * 4;
}

template <int D, bool F32>
void LaunchWide(Attn4Args p, hipStream_t s) {
  const Wide w = WidePlan(p.batch, p.seq, p.G, p.hkv);
  p.qt = 32 / p.G;
  p.tiles = static_cast<int32_t>(w.tiles);
  p.split = static_cast<int32_t>(w.split);
  p.units = p.batch * p.tiles;
  p.tiles_inv = static_cast<uint32_t>(CeilDiv(int64_t{1} << 32, p.tiles));
  const dim3 grid(static_cast<unsigned>(p.hkv), static_cast<unsigned>(p.units), static_cast<unsigned>(p.split));
  RecordLaunch(static_cast<int64_t>(grid.x) * grid.y * grid.z, 512, 0, "kv4_attention_wide<%s,d=%d,splits=%d>", F32 ? "f32" : "bf16", D, p.split);
  if (p.split > 1) hipLaunchKernelGGL((kv4_attention_wide_kernel<D, F32, true>), grid, dim3(512), 0, s, p);
  else hipLaunchKernelGGL((kv4_attention_wide_kernel<D, F32, false>), grid, dim3(512), 0, s, p);
}

template <int D, bool F32>
void Launch(const Attn4Args& p, hipStream_t s) {
  if (ManyRows(p.batch, p.seq, p.G, p.hkv)) return LaunchWide<D, F32>(p, s);
  // kv head fastest: with 8 kv heads every block of a head runs on one XCD
  const dim3 grid(static_cast<unsigned>(p.hkv), static_cast<unsigned>(p.slots > 0 ? p.slots : p.units));
  constexpr int NW = kWaves;
  const int lds = NW * (p.qt * p.G * D + 32) * 4;
  RecordLaunch(static_cast<int64_t>(grid.x) * grid.y, NW * 64, lds, "kv4_attention<%s,d=%d,waves=%d,slots=%d>", F32 ? "f32" : "bf16", D, NW, p.slots);
  if (!F32 && p.qt * p.G <= 8) hipLaunchKernelGGL((kv4_attention_kernel<D, F32, NW, !F32>), grid, dim3(NW * 64), lds, s, p);
  else hipLaunchKernelGGL((kv4_attention_kernel<D, F32, NW, false>), grid, dim3(NW * 64), lds, s, p);
}

}  // namespace
}  // namespace am

using namespace am;

extern "C" int64_t am_gfx950_kv4_attention_workspace_bytes(int64_t batch, int64_t seq, int64_t hq, int64_t hkv,
                                                           int64_t head_dim, int64_t capacity) {
  if (batch <= 0 || seq <= 0 || hkv <= 0 || hq <= 0 || capacity <= 0 || hq % hkv != 0 || hq / hkv > 16 ||
      batch > kMaxRows || seq > kMaxRows || hkv > 65536 || capacity >= (int64_t{1} << 31))
    return kTicketBytes;  // no call takes these
  return WorkspaceBytes(batch, seq, hq / hkv, hkv, head_dim, capacity);
}

extern "C" am_status_code am_gfx950_kv4_attention(const am_gfx950_kv4_attention_args* a, void* stream) {
  AM_CHECK_ARG(a != nullptr, "kv4_attention: null args");
  AM_CHECK_ARG(a->dtype == AM_DT_F32 || a->dtype == AM_DT_BF16, "kv4_attention: dtype must be f32 or bf16");
  AM_CHECK_ARG(a->hq > 0 && a->hkv > 0 && a->hq % a->hkv == 0, "kv4_attention: q heads must be a multiple of kv heads");
  AM_CHECK_ARG(a->hq / a->hkv <= 16, "kv4_attention: at most 16 q heads per kv head");
  AM_CHECK_ARG(a->batch >= 0 && a->seq >= 0 && a->capacity > 0 && a->capacity < (int64_t{1} << 31) - 64, "kv4_attention: bad shape");
  AM_CHECK_ARG(a->hkv <= 65536 && a->batch <= kMaxRows && a->seq <= kMaxRows && a->batch * a->seq <= kMaxRows,
               "kv4_attention: too many query rows");
  AM_CHECK_ARG(std::isfinite(a->scale * kLog2e) && a->scale >= 0.0f, "kv4_attention: scale must be finite and not negative");
  if (a->batch == 0 || a->seq == 0) return AM_STATUS_OK;
  AM_CHECK_ARG(a->q && a->out && a->start_pos_dev, "kv4_attention: null pointer");
  AM_CHECK_ARG(Aligned16(a->q) && Aligned16(a->out), "kv4_attention: q and out must be 16-byte aligned");
  const int64_t cbs = a->batch > 1 ? a->cache_batch_stride : 0;
  if (auto st = CheckKv4Cache(a->k_codes, a->k_scales, a->v_codes, a->v_scales, a->batch, a->head_dim, a->capacity, cbs, a->pages);
      st != AM_STATUS_OK)
    return st;
  Attn4Args p{};
  if (auto st = MakeKvRows(a->pages, cbs, a->capacity, a->hkv, a->head_dim, &p.kv); st != AM_STATUS_OK) return st;
  if (auto st = CheckStreamDevice(AsStream(stream)); st != AM_STATUS_OK) return st;
  const int64_t G = a->hq / a->hkv, qt = std::min<int64_t>(16 / G, a->seq), tiles = CeilDiv(a->seq, qt), units = a->batch * tiles;
  AM_CHECK_ARG(a->workspace != nullptr && Aligned16(a->workspace) &&
                   a->workspace_bytes >= WorkspaceBytes(a->batch, a->seq, G, a->hkv, a->head_dim, a->capacity),
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
  // Little work runs in one block a CU: a second one's merges cost more than it takes over.
  // 8 sequences at 1500-3000 keys (17 steps a CU) 14.3 -> 12.5 us, at 2500-5000 (29) 15.3 -> 14.2, 16 at
  // 1500-3000 (35) the same either way.
  const int64_t cus = DeviceCUs(), few = CeilDiv(cus, a->hkv);
  p.few_slots = static_cast<int32_t>(few >= 2 * units ? std::min<int64_t>(few, p.slots) : p.slots);
  p.few_steps = static_cast<int32_t>(kFewSteps * cus / a->hkv);
  p.tiles_inv = static_cast<uint32_t>(CeilDiv(int64_t{1} << 32, tiles));
  p.g_inv = static_cast<int32_t>(CeilDiv(1 << 16, G));
  p.scale = kLog2e * (a->scale > 0.0f ? a->scale : 1.0f / sqrtf(static_cast<float>(a->head_dim)));
  hipStream_t s = AsStream(stream);
  if (a->dtype == AM_DT_BF16) a->head_dim == 128 ? Launch<128, false>(p, s) : Launch<64, false>(p, s);
  else a->head_dim == 128 ? Launch<128, true>(p, s) : Launch<64, true>(p, s);
  AM_RETURN_IF_LAUNCH_FAILED("kv4_attention");
  return AM_STATUS_OK;
}
