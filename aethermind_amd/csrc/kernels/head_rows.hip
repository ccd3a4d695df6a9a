// Kernels over the rows of single heads: per-head norm and rotation (qk_norm_rope), the
// same with the cache write (kv_append, plain and 4-bit caches), and the rows of a 4-bit
// cache as values (kv4_read).  All of them stream: every input and output byte moves once.

#include <algorithm>
#include <cmath>

#include "am_kv4.h"
#include "am_launch_timing.h"

namespace am {

am_status_code CheckStreamDevice(hipStream_t s) {
  if (s == nullptr) return AM_STATUS_OK;
  int cur = -1, sdev = -1;
  if (hipGetDevice(&cur) != hipSuccess || hipStreamGetDevice(s, &sdev) != hipSuccess) (void)hipGetLastError();  // (else the next launch's)
  if (cur < 0 || cur != sdev)
    return SetLastError(AM_STATUS_INVALID_ARGUMENT, "the stream's device is not the current device");
  return AM_STATUS_OK;
}

am_status_code CheckKv4Cache(const void* kc, const void* ks, const void* vc, const void* vs, int64_t batch,
                             int64_t head_dim, int64_t capacity, int64_t cbs, const am_gfx950_kv_pages* pages) {
  AM_CHECK_ARG(head_dim == 64 || head_dim == 128, "kv4 cache: head_dim must be 64 or 128");
  AM_CHECK_ARG(kc && ks && vc && vs, "kv4 cache: null code or scale cache");
  AM_CHECK_ARG(Aligned16(kc) && Aligned16(ks) && Aligned16(vc) && Aligned16(vs),
               "kv4 cache: code and scale caches must be 16-byte aligned");
  if (pages == nullptr) {
    AM_CHECK_ARG(capacity % 32 == 0, "kv4 cache: without pages the capacity must be a multiple of 32");
    if (batch > 1)
      AM_CHECK_ARG(cbs >= 0 && cbs % (32 * head_dim) == 0,
                   "kv4 cache: cache_batch_stride must be a multiple of 32 * head_dim values");
  }
  return AM_STATUS_OK;
}

namespace {

struct HeadRowArgs {
  const void *q, *k, *v;
  void *q_out, *k_out;
  const void *q_w, *k_w;
  const float *cos_tab, *sin_tab;
  const int64_t* pos;   // norm_rope: position of each row; append: first position of each sequence
  const int32_t* lens;  // append
  int64_t qs, ks, vs, qos, kos;  // row strides
  int64_t limit;        // positions below it are rotated (and written)
  void *kc, *vc;
  uint8_t *ksc, *vsc;
  int32_t* err;
  KvRows kv;
  uint32_t rows, seq, hq, hk, hv;  // hv: 0 for norm_rope
  int32_t d;
  float eps;
};

enum HeadRowMode { kNormRope = 0, kAppendPlain = 1, kAppendKv4 = 2 };

// 8 values of a row as they sit in memory (bf16: 16 bytes, f32: 32).
template <class A>
struct Raw8 {
  uint4 w[sizeof(typename A::T) / 2];
};
template <class A, bool VEC>
__device__ __forceinline__ Raw8<A> load_raw8(const typename A::T* p) {
  Raw8<A> r;
  if constexpr (VEC) {
#pragma unroll
    for (size_t i = 0; i < sizeof(r) / 16; ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    typename A::T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i];
    __builtin_memcpy(&r, e, sizeof(r));
  }
  return r;
}
template <class A, bool VEC>
__device__ __forceinline__ void store_raw8(typename A::T* p, const Raw8<A>& r) {
  if constexpr (VEC) {
#pragma unroll
    for (size_t i = 0; i < sizeof(r) / 16; ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
  } else {
    typename A::T e[8];
    __builtin_memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = e[i];
  }
}
template <class A>
__device__ __forceinline__ void unpack8(const Raw8<A>& r, float (&v)[8]) {
#pragma unroll
  for (size_t i = 0; i < sizeof(r) / 16; ++i) {
    const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (A::kDtype == AM_DT_BF16) {
        v[2 * e] = __uint_as_float(w[e] << 16);
        v[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
      } else {
        v[4 * i + e] = __uint_as_float(w[e]);
      }
    }
  }
}
// One rounding to the type.  bf16: the conversion of two values at once, which is
// f32_to_bf16_bits but for the pattern of a NaN; those take the branch.
template <class A>
__device__ __forceinline__ Raw8<A> pack8(const float (&v)[8]) {
  Raw8<A> r;
  if constexpr (A::kDtype == AM_DT_BF16) {
    float t = 0.0f;  // NaN where a value is NaN or infinite
#pragma unroll
    for (int e = 0; e < 8; ++e) t = __builtin_fmaf(v[e], 0.0f, t);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<__bf16>(v[2 * e]), static_cast<__bf16>(v[2 * e + 1])});
    if (__builtin_expect(t != t, 0)) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = f32_to_bf16_bits(v[2 * e]) | (static_cast<uint32_t>(f32_to_bf16_bits(v[2 * e + 1])) << 16);
    }
    r.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      r.w[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                          __float_as_uint(v[4 * i + 3]));
  }
  return r;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ double dpp_add_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint64_t o = dpp_u32<CTRL>(static_cast<uint32_t>(b)) | (static_cast<uint64_t>(dpp_u32<CTRL>(static_cast<uint32_t>(b >> 32))) << 32);
  return v + __builtin_bit_cast(double, o);
}
template <int CTRL>
__device__ __forceinline__ float dpp_add_f32(float v) {
  return v + __uint_as_float(dpp_u32<CTRL>(__float_as_uint(v)));
}
// Sum over aligned groups of LP lanes (4, 8 or 16); every lane receives it.
template <int LP>
__device__ __forceinline__ float lanes_sum(float v) {
  v = dpp_add_f32<0x4E>(dpp_add_f32<0xB1>(v));         // quad_perm [1,0,3,2], [2,3,0,1]
  if constexpr (LP >= 8) v = dpp_add_f32<0x141>(v);   // row_half_mirror
  if constexpr (LP >= 16) v = dpp_add_f32<0x140>(v);  // row_mirror
  return v;
}
template <int LP>
__device__ __forceinline__ double lanes_sum(double v) {
  v = dpp_add_f64<0x4E>(dpp_add_f64<0xB1>(v));
  if constexpr (LP >= 8) v = dpp_add_f64<0x141>(v);
  if constexpr (LP >= 16) v = dpp_add_f64<0x140>(v);
  return v;
}

// Norm (gain w, or none) and rotation of one head's row: lane `sub` of LP holds values
// 8 sub .. +8 of each half, so a pair's two values are in one lane.
template <class F, int D, class A>
__device__ __forceinline__ void norm_rotate(float (&lo)[8], float (&hi)[8], bool norm, const Raw8<A> (&gain)[2], float eps,
                                            const float (&c)[8], const float (&s)[8], bool turn) {
  constexpr int LP = D / 16;
  F x1[8], x2[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x1[i] = lo[i], x2[i] = hi[i];
  if (norm) {
    F ss = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fma(x1[i], x1[i], fma(x2[i], x2[i], ss));
    ss = lanes_sum<LP>(ss);
    const F inv = F(1) / sqrt(ss / F(D) + F(eps));
    float w1[8], w2[8];
    unpack8<A>(gain[0], w1);
    unpack8<A>(gain[1], w2);
#pragma unroll
    for (int i = 0; i < 8; ++i) x1[i] = x1[i] * inv * F(w1[i]), x2[i] = x2[i] * inv * F(w2[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float y1, y2;
    if constexpr (sizeof(F) == 8) {
      y1 = static_cast<float>(x1[i] * c[i] - x2[i] * s[i]);
      y2 = static_cast<float>(x2[i] * c[i] + x1[i] * s[i]);
    } else {
      rope_rotate(x1[i], x2[i], c[i], s[i], y1, y2);
    }
    lo[i] = turn ? y1 : static_cast<float>(x1[i]);
    hi[i] = turn ? y2 : static_cast<float>(x2[i]);
  }
}

// 8 values of a group of 32 that four lanes hold, into 4 bytes of codes and (lane 0 of the
// four) the scale byte.  max|x| as an integer: NaN and infinity compare above every finite
// value.  Adding 0x200000 carries a mantissa of 1.75 or more into the exponent, so the
// shifted exponent less 2 is the smallest e with max|x| < 7 * 2^e.
__device__ __forceinline__ void kv4_store8(const float (&v)[8], int sub, uint8_t* codes, uint8_t* scale) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  m = max(m, dpp_u32<0xB1>(m));
  m = max(m, dpp_u32<0x4E>(m));
  const bool fine = m < 0x7F800000u;
  const int e = min(max(static_cast<int>((m + 0x200000u) >> 23) - 2, 0), 252);
  const float s = e8m0_scale(static_cast<uint32_t>(e));
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
  *reinterpret_cast<uint32_t*>(codes) = fine ? w : 0u;
  if ((sub & 3) == 0) *scale = static_cast<uint8_t>(fine ? e : 255);
}

// The position of a row and whether it is one to rotate and write; false: no live row.
template <int MODE>
__device__ __forceinline__ bool row_position(const HeadRowArgs& p, uint32_t row, uint32_t& b, int64_t& at, bool& ok) {
  b = 0;
  if constexpr (MODE == kNormRope) {
    at = p.pos[row];
  } else {
    b = row / p.seq;
    const uint32_t s = row - b * p.seq;
    if (static_cast<int32_t>(s) >= live_rows(p.lens, b, static_cast<int32_t>(p.seq))) return false;
    at = seq_position(p.pos[b], s);
  }
  ok = at >= 0 && at < p.limit;
  return true;
}

// D in {64, 128, 256}: LP = D / 16 lanes own a row of a head, 8 values of each half per
// lane (two 16-byte loads of bf16), and every row of a head its own lanes: 2048 rows of 32 + 8
// heads of 128 (43 MB) take 8.9 us, 4.8 TB/s, a copy's rate; two heads per lane group, the
// table row read once, 9.9, four 11.0; one row 2.3, 2.9 and 3.8.
template <class A, int D, int MODE, bool VEC>
__global__ __launch_bounds__(256) void head_rows_kernel(HeadRowArgs p) {
  constexpr int LP = D / 16;
  using T = typename A::T;
  const uint32_t item = blockIdx.x * (256 / LP) + threadIdx.x / LP;
  const int sub = threadIdx.x % LP;
  const uint32_t heads = p.hq + p.hk + p.hv;
  const uint32_t row = item / heads, h = item - row * heads;
  if (row >= p.rows) return;
  uint32_t b;
  int64_t at;
  bool ok;
  if (!row_position<MODE>(p, row, b, at, ok)) return;
  const bool is_q = h < p.hq, is_k = !is_q && h < p.hq + p.hk;
  const uint32_t g = is_q ? h : is_k ? h - p.hq : h - p.hq - p.hk;
  const T* x = static_cast<const T*>(is_q ? p.q : is_k ? p.k : p.v) + row * (is_q ? p.qs : is_k ? p.ks : p.vs) + g * D + 8 * sub;
  Raw8<A> lo = load_raw8<A, VEC>(x), hi = load_raw8<A, VEC>(x + D / 2);
  const T* w = static_cast<const T*>(is_q ? p.q_w : is_k ? p.k_w : nullptr);
  Raw8<A> gain[2];
  if (w != nullptr) {
    gain[0] = load_raw8<A, VEC>(w + 8 * sub);
    gain[1] = load_raw8<A, VEC>(w + D / 2 + 8 * sub);
  }
  float c[8], s[8];
  if (MODE == kNormRope || is_q || is_k) {
    const int64_t t = (ok ? at : 0) * (D / 2) + 8 * sub;
    unpack8<ActF32>(load_raw8<ActF32, VEC>(p.cos_tab + t), c);
    unpack8<ActF32>(load_raw8<ActF32, VEC>(p.sin_tab + t), s);
  }
  float x1[8], x2[8];
  unpack8<A>(lo, x1);
  unpack8<A>(hi, x2);
  if (MODE == kNormRope || is_q) {
    norm_rotate<float, D, A>(x1, x2, w != nullptr, gain, p.eps, c, s, ok);
    T* out = (is_q ? static_cast<T*>(p.q_out) + row * p.qos : static_cast<T*>(p.k_out) + row * p.kos) + g * D + 8 * sub;
    store_raw8<A, VEC>(out, pack8<A>(x1));
    store_raw8<A, VEC>(out + D / 2, pack8<A>(x2));
  } else if constexpr (MODE != kNormRope) {
    if (!ok && p.err != nullptr) *p.err = 1;
    const int64_t dst = ok ? p.kv.WriteRow(b, g, at) : -1;
    if (dst < 0) return;
    if constexpr (MODE == kAppendPlain) {
      if (is_k) {
        norm_rotate<float, D, A>(x1, x2, w != nullptr, gain, p.eps, c, s, true);
        lo = pack8<A>(x1);
        hi = pack8<A>(x2);
      }
      T* out = static_cast<T*>(is_k ? p.kc : p.vc) + dst + 8 * sub;
      store_raw8<A, VEC>(out, lo);
      store_raw8<A, VEC>(out + D / 2, hi);
    } else {
      // 64 bits: a key next to a code's border takes the same code whatever the order of the
      // sums (fp32 errors of 2^-24 move about one code in 10^6)
      if (is_k) norm_rotate<double, D, A>(x1, x2, w != nullptr, gain, p.eps, c, s, true);
      uint8_t* codes = static_cast<uint8_t*>(is_k ? p.kc : p.vc) + dst / 2 + 4 * sub;
      uint8_t* scales = (is_k ? p.ksc : p.vsc) + dst / 32 + sub / 4;
      kv4_store8(x1, sub, codes, scales);
      kv4_store8(x2, sub, codes + D / 4, scales + D / 64);
    }
  }
}

// Any even head_dim: one wave per row of a head, value by value.
template <class A, int MODE>
__global__ __launch_bounds__(256) void head_rows_any_kernel(HeadRowArgs p) {
  using T = typename A::T;
  const int lane = threadIdx.x & 63;
  const uint32_t heads = p.hq + p.hk + p.hv;
  const uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t row = item / heads, h = item - row * heads;
  if (row >= p.rows) return;
  uint32_t b;
  int64_t at;
  bool ok;
  if (!row_position<MODE>(p, row, b, at, ok)) return;
  const bool is_q = h < p.hq, is_k = !is_q && h < p.hq + p.hk;
  const uint32_t g = is_q ? h : is_k ? h - p.hq : h - p.hq - p.hk;
  const T* x = static_cast<const T*>(is_q ? p.q : is_k ? p.k : p.v) + row * (is_q ? p.qs : is_k ? p.ks : p.vs) +
               static_cast<int64_t>(g) * p.d;
  T* out;
  if (is_q) {
    out = static_cast<T*>(p.q_out) + row * p.qos + static_cast<int64_t>(g) * p.d;
  } else if (MODE == kNormRope) {
    out = static_cast<T*>(p.k_out) + row * p.kos + static_cast<int64_t>(g) * p.d;
  } else {
    const int64_t dst = ok ? p.kv.WriteRow(b, g, at) : -1;
    if (dst < 0) {
      if (!ok && p.err != nullptr) *p.err = 1;
      return;
    }
    out = static_cast<T*>(is_k ? p.kc : p.vc) + dst;
  }
  if (!is_q && !is_k) {
    for (int i = lane; i < p.d; i += 64) out[i] = x[i];
    return;
  }
  const T* w = static_cast<const T*>(is_q ? p.q_w : p.k_w);
  const int half = p.d / 2;
  float inv = 1.0f;
  if (w != nullptr) {
    float ss = 0.0f;
    for (int i = lane; i < p.d; i += 64) {
      const float v = A::load(x, i);
      ss = fmaf(v, v, ss);
    }
    inv = 1.0f / sqrtf(wave_sum(ss) / static_cast<float>(p.d) + p.eps);
  }
  for (int i = lane; i < half; i += 64) {
    float x1 = A::load(x, i), x2 = A::load(x, i + half);
    if (w != nullptr) {
      x1 = x1 * inv * A::load(w, i);
      x2 = x2 * inv * A::load(w, i + half);
    }
    float y1 = x1, y2 = x2;
    if (ok) rope_rotate(x1, x2, p.cos_tab[at * half + i], p.sin_tab[at * half + i], y1, y2);
    A::store(out, i, y1);
    A::store(out, i + half, y2);
  }
}

constexpr int64_t kMaxItems = int64_t{1} << 25;  // head rows of a call (a grid has fewer than 2^32 threads)

const char* const kModeName[] = {"qk_norm_rope", "kv_append", "kv_append_kv4"};

template <class A, int MODE, int D>
void LaunchHeadRows(const HeadRowArgs& p, bool vec, hipStream_t s) {
  const int64_t grid = CeilDiv(static_cast<int64_t>(p.rows) * (p.hq + p.hk + p.hv), 256 / (D / 16));
  RecordLaunch(grid, 256, 0, "%s<%s,d=%d,vec=%d>", kModeName[MODE], A::kDtype == AM_DT_BF16 ? "bf16" : "f32", D, vec ? 1 : 0);
  const dim3 blocks(static_cast<unsigned>(grid));
  if (vec) hipLaunchKernelGGL((head_rows_kernel<A, D, MODE, true>), blocks, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((head_rows_kernel<A, D, MODE, false>), blocks, dim3(256), 0, s, p);
}

template <class A, int MODE>
am_status_code LaunchMode(const HeadRowArgs& p, bool vec, hipStream_t s) {
  const int64_t items = static_cast<int64_t>(p.rows) * (p.hq + p.hk + p.hv);
  if (items > kMaxItems) return SetLastError(AM_STATUS_INVALID_ARGUMENT, "head rows: too many rows");
  if (p.d == 64) {
    LaunchHeadRows<A, MODE, 64>(p, vec, s);
  } else if (p.d == 128) {
    LaunchHeadRows<A, MODE, 128>(p, vec, s);
  } else if constexpr (MODE != kAppendKv4) {
    if (p.d == 256) {
      LaunchHeadRows<A, MODE, 256>(p, vec, s);
    } else {
      const int64_t grid = CeilDiv(items, 4);
      RecordLaunch(grid, 256, 0, "%s_any<%s,d=%d>", kModeName[MODE], A::kDtype == AM_DT_BF16 ? "bf16" : "f32", p.d);
      hipLaunchKernelGGL((head_rows_any_kernel<A, MODE>), dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, p);
    }
  }
  AM_RETURN_IF_LAUNCH_FAILED("head rows");
  return AM_STATUS_OK;
}

// ---- 4-bit rows as values ----
struct ReadArgs {
  const uint8_t *codes[2], *scales[2];  // k, v
  void* out[2];
  const int64_t* start;
  const int32_t* lens;
  KvRows kv;
  int64_t cap;
  uint32_t seq, hkv, batch;
};

// A thread converts 8 values of kReadRows rows: 4 bytes of codes into 16 (bf16) or 32 (f32)
// bytes each.  A block's rows follow each other in one head's plane, so the codes are read
// contiguously, and the output is written in whole rows of a head.  grid.y: k, v.  Four
// sequences of 8192 rows (170 MB): 32.9 us, 5.2 TB/s, a copy's rate (one row a thread, its head
// found by divisions, 42.8; four rows 33.0, eight 34.8; 37 rows 2.6, 2.9 and 3.0).
constexpr int kReadRows = 2;
template <class O, int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(ReadArgs p) {
  constexpr uint32_t LP = D / 8, RB = 256 / LP;  // lanes of a row, rows of the block at a time
  const uint32_t chunks = (p.seq + RB * kReadRows - 1) / (RB * kReadRows);
  const uint32_t bg = blockIdx.x / chunks, first = (blockIdx.x - bg * chunks) * (RB * kReadRows) + threadIdx.x / LP;
  const uint32_t b = bg / p.hkv, g = bg - b * p.hkv;
  const int sub = threadIdx.x % LP;
  const uint32_t live = static_cast<uint32_t>(live_rows(p.lens, b, static_cast<int32_t>(p.seq)));
  const int64_t start = seq_position(p.start[b], 0);
  uint32_t w[kReadRows], e[kReadRows];
#pragma unroll
  for (int r = 0; r < kReadRows; ++r) {
    const uint32_t s = first + r * RB;
    const int64_t at = start + s;
    w[r] = e[r] = 0;
    if (s < live && at >= 0 && at < p.cap) {
      const int64_t row = p.kv.Row(b, g, at);
      w[r] = *reinterpret_cast<const uint32_t*>(p.codes[blockIdx.y] + row / 2 + 4 * sub);
      e[r] = p.scales[blockIdx.y][row / 32 + sub / 4];
    }
  }
#pragma unroll
  for (int r = 0; r < kReadRows; ++r) {
    const uint32_t s = first + r * RB;
    if (s >= live) return;
    uint32_t pair[4];
    fp4_to_bf16(w[r], e8m0_scale_or_nan(e[r]), pair);
    const int64_t at_out = ((static_cast<int64_t>(b) * p.seq + s) * p.hkv + g) * D + 8 * sub;
    if constexpr (O::kDtype == AM_DT_BF16) {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out[blockIdx.y]) + at_out) = make_uint4(pair[0], pair[1], pair[2], pair[3]);
    } else {
      float4* out = reinterpret_cast<float4*>(static_cast<float*>(p.out[blockIdx.y]) + at_out);
#pragma unroll
      for (int t = 0; t < 2; ++t)
        out[t] = make_float4(__uint_as_float(pair[2 * t] << 16), __uint_as_float(pair[2 * t] & 0xFFFF0000u),
                             __uint_as_float(pair[2 * t + 1] << 16), __uint_as_float(pair[2 * t + 1] & 0xFFFF0000u));
    }
  }
}

bool IsAct(int32_t dt) { return dt == AM_DT_F32 || dt == AM_DT_BF16; }

}  // namespace
}  // namespace am

using namespace am;

extern "C" am_status_code am_gfx950_qk_norm_rope(const am_gfx950_qk_norm_rope_args* a, void* stream) {
  AM_CHECK_ARG(a != nullptr, "qk_norm_rope: null args");
  AM_CHECK_ARG(IsAct(a->dtype), "qk_norm_rope: dtype must be f32 or bf16");
  AM_CHECK_ARG(a->rows >= 0 && a->hq >= 0 && a->hkv >= 0 && a->hq + a->hkv > 0 && a->hq <= 65536 && a->hkv <= 65536,
               "qk_norm_rope: bad shape");
  AM_CHECK_ARG(a->head_dim > 0 && a->head_dim % 2 == 0 && a->head_dim <= 1024,
               "qk_norm_rope: head_dim must be even and at most 1024");
  AM_CHECK_ARG(a->max_pos > 0, "qk_norm_rope: max_pos must be positive");
  AM_CHECK_ARG(a->rows < (int64_t{1} << 31), "qk_norm_rope: too many rows");
  const int64_t d = a->head_dim;
  AM_CHECK_ARG(a->hq == 0 || (a->q_stride >= a->hq * d && a->q_out_stride >= a->hq * d),
               "qk_norm_rope: q row stride smaller than its heads");
  AM_CHECK_ARG(a->hkv == 0 || (a->k_stride >= a->hkv * d && a->k_out_stride >= a->hkv * d),
               "qk_norm_rope: k row stride smaller than its heads");
  const bool gains = (a->hq > 0 && a->q_norm_w) || (a->hkv > 0 && a->k_norm_w);
  if (gains) AM_CHECK_ARG(a->eps > 0.0f && std::isfinite(a->eps), "qk_norm_rope: eps must be finite and positive");
  if (a->rows == 0) return AM_STATUS_OK;
  AM_CHECK_ARG(a->hq == 0 || (a->q && a->q_out), "qk_norm_rope: null pointer");
  AM_CHECK_ARG(a->hkv == 0 || (a->k && a->k_out), "qk_norm_rope: null pointer");
  AM_CHECK_ARG(a->pos && a->cos_tab && a->sin_tab, "qk_norm_rope: null pointer");
  if (auto st = CheckStreamDevice(AsStream(stream)); st != AM_STATUS_OK) return st;
  HeadRowArgs p{};
  p.q = a->q, p.k = a->k, p.q_out = a->q_out, p.k_out = a->k_out;
  p.q_w = a->q_norm_w, p.k_w = a->k_norm_w;
  p.cos_tab = a->cos_tab, p.sin_tab = a->sin_tab, p.pos = a->pos;
  p.qs = a->q_stride, p.ks = a->k_stride, p.qos = a->q_out_stride, p.kos = a->k_out_stride;
  p.limit = a->max_pos;
  p.rows = static_cast<uint32_t>(a->rows);
  p.hq = static_cast<uint32_t>(a->hq), p.hk = static_cast<uint32_t>(a->hkv);
  p.d = static_cast<int32_t>(d);
  p.eps = a->eps;
  const int64_t step = a->dtype == AM_DT_BF16 ? 8 : 4;  // values of 16 bytes
  bool vec = Aligned16(a->cos_tab) && Aligned16(a->sin_tab);
  if (a->hq > 0)
    vec = vec && Aligned16(a->q) && Aligned16(a->q_out) && Aligned16(a->q_norm_w) && a->q_stride % step == 0 && a->q_out_stride % step == 0;
  if (a->hkv > 0)
    vec = vec && Aligned16(a->k) && Aligned16(a->k_out) && Aligned16(a->k_norm_w) && a->k_stride % step == 0 && a->k_out_stride % step == 0;
  return a->dtype == AM_DT_BF16 ? LaunchMode<ActBF16, kNormRope>(p, vec, AsStream(stream))
                                : LaunchMode<ActF32, kNormRope>(p, vec, AsStream(stream));
}

extern "C" am_status_code am_gfx950_kv_append(const am_gfx950_kv_append_args* a, void* stream) {
  AM_CHECK_ARG(a != nullptr, "kv_append: null args");
  AM_CHECK_ARG(IsAct(a->dtype), "kv_append: dtype must be f32 or bf16");
  AM_CHECK_ARG(a->cache_format == AM_KV_PLAIN || a->cache_format == AM_KV_MXFP4, "kv_append: unknown cache format");
  AM_CHECK_ARG(a->batch >= 0 && a->seq >= 0 && a->hq >= 0 && a->hkv > 0 && a->hq <= 65536 && a->hkv <= 65536 && a->capacity > 0,
               "kv_append: bad shape");
  AM_CHECK_ARG(a->head_dim > 0 && a->head_dim % 2 == 0 && a->head_dim <= 1024,
               "kv_append: head_dim must be even and at most 1024");
  AM_CHECK_ARG(a->max_pos >= a->capacity, "kv_append: the rotation tables must cover the capacity");
  AM_CHECK_ARG(a->batch <= kMaxItems && a->seq <= kMaxItems && a->batch * a->seq <= kMaxItems, "kv_append: too many rows");
  AM_CHECK_ARG(a->capacity < (int64_t{1} << 31), "kv_append: capacity too large");
  const int64_t d = a->head_dim;
  AM_CHECK_ARG(a->hq == 0 || (a->q_stride >= a->hq * d && a->q_out_stride >= a->hq * d),
               "kv_append: q row stride smaller than its heads");
  AM_CHECK_ARG(a->k_stride >= a->hkv * d && a->v_stride >= a->hkv * d, "kv_append: k or v row stride smaller than its heads");
  const bool gains = (a->hq > 0 && a->q_norm_w) || a->k_norm_w;
  if (gains) AM_CHECK_ARG(a->eps > 0.0f && std::isfinite(a->eps), "kv_append: eps must be finite and positive");
  if (a->batch == 0 || a->seq == 0) return AM_STATUS_OK;
  AM_CHECK_ARG(a->hq == 0 || (a->q && a->q_out), "kv_append: null pointer");
  AM_CHECK_ARG(a->k && a->v && a->k_cache && a->v_cache && a->start_pos_dev && a->cos_tab && a->sin_tab,
               "kv_append: null pointer");
  if (a->pages == nullptr && a->batch > 1)
    AM_CHECK_ARG(a->cache_batch_stride >= a->hkv * a->capacity * d, "kv_append: sequences share cache rows");
  const bool four = a->cache_format == AM_KV_MXFP4;
  const int64_t cbs = a->batch > 1 ? a->cache_batch_stride : 0;
  if (four)
    if (auto st = CheckKv4Cache(a->k_cache, a->k_scales, a->v_cache, a->v_scales, a->batch, d, a->capacity, cbs, a->pages);
        st != AM_STATUS_OK)
      return st;
  HeadRowArgs p{};
  if (auto st = MakeKvRows(a->pages, cbs, a->capacity, a->hkv, d, &p.kv); st != AM_STATUS_OK) return st;
  if (p.kv.err == nullptr) p.kv.err = a->err_flag;
  if (auto st = CheckStreamDevice(AsStream(stream)); st != AM_STATUS_OK) return st;
  p.q = a->q, p.k = a->k, p.v = a->v, p.q_out = a->q_out;
  p.q_w = a->q_norm_w, p.k_w = a->k_norm_w;
  p.cos_tab = a->cos_tab, p.sin_tab = a->sin_tab, p.pos = a->start_pos_dev, p.lens = a->seq_lens;
  p.qs = a->q_stride, p.ks = a->k_stride, p.vs = a->v_stride, p.qos = a->q_out_stride;
  p.limit = a->capacity;
  p.kc = a->k_cache, p.vc = a->v_cache, p.ksc = a->k_scales, p.vsc = a->v_scales;
  p.err = a->err_flag;
  p.rows = static_cast<uint32_t>(a->batch * a->seq), p.seq = static_cast<uint32_t>(a->seq);
  p.hq = static_cast<uint32_t>(a->hq), p.hk = p.hv = static_cast<uint32_t>(a->hkv);
  p.d = static_cast<int32_t>(d);
  p.eps = a->eps;
  const int64_t step = a->dtype == AM_DT_BF16 ? 8 : 4;
  bool vec = Aligned16(a->cos_tab) && Aligned16(a->sin_tab) && Aligned16(a->k) && Aligned16(a->v) && Aligned16(a->k_norm_w) &&
             a->k_stride % step == 0 && a->v_stride % step == 0 && Aligned16(a->k_cache) && Aligned16(a->v_cache) && cbs % step == 0;
  if (a->hq > 0)
    vec = vec && Aligned16(a->q) && Aligned16(a->q_out) && Aligned16(a->q_norm_w) && a->q_stride % step == 0 && a->q_out_stride % step == 0;
  hipStream_t s = AsStream(stream);
  if (four) return a->dtype == AM_DT_BF16 ? LaunchMode<ActBF16, kAppendKv4>(p, vec, s) : LaunchMode<ActF32, kAppendKv4>(p, vec, s);
  return a->dtype == AM_DT_BF16 ? LaunchMode<ActBF16, kAppendPlain>(p, vec, s) : LaunchMode<ActF32, kAppendPlain>(p, vec, s);
}

extern "C" am_status_code am_gfx950_kv4_read(const am_gfx950_kv4_read_args* a, void* stream) {
  AM_CHECK_ARG(a != nullptr, "kv4_read: null args");
  AM_CHECK_ARG(IsAct(a->out_dtype), "kv4_read: out dtype must be f32 or bf16");
  AM_CHECK_ARG(a->batch >= 0 && a->seq >= 0 && a->hkv > 0 && a->hkv <= 65536 && a->capacity > 0, "kv4_read: bad shape");
  AM_CHECK_ARG(a->batch <= kMaxItems && a->seq <= kMaxItems && a->batch * a->seq <= kMaxItems && a->batch * a->seq * a->hkv <= kMaxItems,
               "kv4_read: too many rows");
  AM_CHECK_ARG(a->capacity < (int64_t{1} << 31), "kv4_read: capacity too large");
  if (a->batch == 0 || a->seq == 0) return AM_STATUS_OK;
  AM_CHECK_ARG(a->k_out && a->v_out && a->start_pos_dev, "kv4_read: null pointer");
  AM_CHECK_ARG(Aligned16(a->k_out) && Aligned16(a->v_out), "kv4_read: outputs must be 16-byte aligned");
  const int64_t cbs = a->batch > 1 ? a->cache_batch_stride : 0;
  if (auto st = CheckKv4Cache(a->k_codes, a->k_scales, a->v_codes, a->v_scales, a->batch, a->head_dim, a->capacity, cbs, a->pages);
      st != AM_STATUS_OK)
    return st;
  ReadArgs p{};
  if (auto st = MakeKvRows(a->pages, cbs, a->capacity, a->hkv, a->head_dim, &p.kv); st != AM_STATUS_OK) return st;
  if (auto st = CheckStreamDevice(AsStream(stream)); st != AM_STATUS_OK) return st;
  p.codes[0] = a->k_codes, p.codes[1] = a->v_codes, p.scales[0] = a->k_scales, p.scales[1] = a->v_scales;
  p.out[0] = a->k_out, p.out[1] = a->v_out;
  p.start = a->start_pos_dev, p.lens = a->seq_lens, p.cap = a->capacity;
  p.seq = static_cast<uint32_t>(a->seq), p.hkv = static_cast<uint32_t>(a->hkv), p.batch = static_cast<uint32_t>(a->batch);
  const int64_t lp = a->head_dim / 8;
  const int64_t blocks = a->batch * a->hkv * CeilDiv(a->seq, 256 / lp * kReadRows);
  AM_CHECK_ARG(blocks < (int64_t{1} << 23), "kv4_read: too many rows");
  const dim3 grid(static_cast<unsigned>(blocks), 2);
  const bool bf = a->out_dtype == AM_DT_BF16;
  RecordLaunch(2 * static_cast<int64_t>(grid.x), 256, 0, "kv4_read<%s,d=%d>", bf ? "bf16" : "f32", static_cast<int>(a->head_dim));
  hipStream_t s = AsStream(stream);
  if (a->head_dim == 128) {
    if (bf) hipLaunchKernelGGL((kv4_read_kernel<ActBF16, 128>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((kv4_read_kernel<ActF32, 128>), grid, dim3(256), 0, s, p);
  } else {
    if (bf) hipLaunchKernelGGL((kv4_read_kernel<ActBF16, 64>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((kv4_read_kernel<ActF32, 64>), grid, dim3(256), 0, s, p);
  }
  AM_RETURN_IF_LAUNCH_FAILED("kv4_read");
  return AM_STATUS_OK;
}
