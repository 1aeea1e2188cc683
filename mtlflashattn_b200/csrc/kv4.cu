// The paged 4-bit key/value cache (mfa_kv4_*, include/mfa.h): appending, reading back, and
// attention over it. Built without fast math: the group scale's division and the quotients that
// are rounded to 4 bits are IEEE fp32, so a value on the border of two codes goes where the
// definition says.
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cmath>

#include "../../include/mfa.h"
#include "common.cuh"
#include "host.cuh"
#include "ptx.cuh"

namespace mfa {
namespace {

struct Kv4Cache {
  uint8_t *k, *v, *ks, *vs;
  const int* table;
  int64_t table_stride;
  int num_pages, page_shift, Hkv, B, max_pages;
  float k_unit, v_unit;
  int* err;
};

__device__ __forceinline__ void kv4_report(const Kv4Cache& c) {
  if (c.err != nullptr) atomicExch(c.err, MFA_ERR_INVALID);
}

// Row of head 0 of token t of sequence b, counted in (page, head, slot) rows; the row of head h
// is h << page_shift further. -1 where the token has no page.
__device__ __forceinline__ int64_t kv4_row(const Kv4Cache& c, int b, int64_t t) {
  const int64_t p = t >> c.page_shift;
  if (t < 0 || p >= c.max_pages) return -1;
  const int page = c.table[(int64_t)b * c.table_stride + p];
  if (page < 0 || page >= c.num_pages) return -1;
  return (((int64_t)page * c.Hkv) << c.page_shift) + (t & ((1 << c.page_shift) - 1));
}

// ------------------------------------------------------------------ 4-bit and 8-bit conversions
// The code in the low 4 bits: as the top bits of an fp16 it stands for 2^-14 of its value.
__device__ __forceinline__ float e2m1_f32(uint32_t code) {
  return __half2float(__ushort_as_half((unsigned short)((code & 8u) << 12 | (code & 7u) << 9))) *
         16384.f;
}
// The codes of a word's four bytes, two each with the low half first, as fp16. The word
// must not come straight from an 8- or 16-bit load: with one, ptxas 12.9 took the wrong bytes.
__device__ __forceinline__ void e2m1x8_f16(uint32_t w, uint32_t* d) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(w));
}
// fp32 pair to a byte of two codes, nearest with ties to the even code, saturating.
__device__ __forceinline__ uint32_t f32_e2m1x2(float lo, float hi) {
  uint32_t d;
  asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n\t"
      "mov.b32 %0, {b, 0, 0, 0};\n\t}"
      : "=r"(d)
      : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x2_f16(uint32_t two_bytes) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
      : "=r"(d)
      : "r"(two_bytes));
  return d;
}
__device__ __forceinline__ float f16_lo(uint32_t h2) {
  return __low2float(*reinterpret_cast<const __half2*>(&h2));
}
__device__ __forceinline__ float f16_hi(uint32_t h2) {
  return __high2float(*reinterpret_cast<const __half2*>(&h2));
}

// ------------------------------------------------------------------ append
struct Kv4Rows {
  const void *k, *v;
  int64_t k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
  const int *start, *lens;
  int L;
};

// One lane holds 4 consecutive dims of a row, 4 lanes a group. blockIdx.y: 0 keys, 1 values.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_append_kernel(const Kv4Cache c, const Kv4Rows r) {
  constexpr int kLanes = D / 4, NG = D / 16;
  const int64_t row = ((int64_t)blockIdx.x * 128 + threadIdx.x) / kLanes;  // (b, j, head)
  const int lane = threadIdx.x % kLanes;
  const bool is_v = blockIdx.y != 0;
  const int h = (int)(row % c.Hkv);
  const int64_t bj = row / c.Hkv;
  const int b = (int)(bj / r.L), j = (int)(bj % r.L);
  int64_t dst = -1;
  bool wanted = b < c.B && (r.lens == nullptr || j < r.lens[b]);
  if (wanted) {
    dst = kv4_row(c, b, (int64_t)(r.start != nullptr ? r.start[b] : 0) + j);
    if (dst < 0 && lane == 0) kv4_report(c);
  }
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (dst >= 0) {
    dst += (int64_t)h << c.page_shift;
    const T* src = is_v ? reinterpret_cast<const T*>(r.v) + b * r.v_sb + j * r.v_ss + h * r.v_sh
                        : reinterpret_cast<const T*>(r.k) + b * r.k_sb + j * r.k_ss + h * r.k_sh;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32<T>(src[4 * lane + i]);
  }
  const float per_unit = 1.f / (is_v ? c.v_unit : c.k_unit);  // exact: a power of two
  float top = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] *= per_unit;
    top = fmaxf(top, fabsf(x[i]));
    nan = nan || x[i] != x[i];
  }
  if (nan) top = NAN;
#pragma unroll
  for (int s = 1; s < 4; s <<= 1) {  // fmaxf drops a NaN: pass it on by hand
    const float other = __shfl_xor_sync(kFull, top, s);
    top = top != top || other != other ? NAN : fmaxf(top, other);
  }
  const float want = top != top ? top : fminf(__fdiv_rn(top, 6.f), 448.f);
  const uint32_t sbyte = __nv_cvt_float_to_fp8(want, __NV_SATFINITE, __NV_E4M3);
  const float scale = f16_lo(e4m3x2_f16(sbyte));
  uint32_t codes[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = scale > 0.f ? __fdiv_rn(x[i], scale) : 0.f;
    codes[i] = f32_e2m1x2(y, 0.f) & 15u;
  }
  const int i16 = lane / 4, u = lane % 4;  // group, quarter of the group
  if (!is_v) {
    if (dst >= 0)
      *reinterpret_cast<uint16_t*>(c.k + dst * (D / 2) + u * (D / 8) + 2 * i16) =
          (uint16_t)(codes[0] | codes[1] << 4 | codes[2] << 8 | codes[3] << 12);
  } else {
    // a byte holds dims g and g + 8 of a group: the partner lane (quarter u ^ 2) has the others
    const uint32_t mine = codes[0] | codes[1] << 8 | codes[2] << 16 | codes[3] << 24;
    const uint32_t other = __shfl_xor_sync(kFull, mine, 2);
    if (dst >= 0 && u < 2) {
      const uint32_t both = mine | other << 4;
#pragma unroll
      for (int n = 0; n < 4; ++n)
        c.v[dst * (D / 2) + (4 * u + n) * NG + i16] = (uint8_t)(both >> (8 * n));
    }
  }
  if (dst >= 0 && u == 0) (is_v ? c.vs : c.ks)[dst * NG + i16] = (uint8_t)sbyte;
}

// ------------------------------------------------------------------ gather
template <typename T>
__device__ __forceinline__ T held_as(float x);
template <>
__device__ __forceinline__ float held_as<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half held_as<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 held_as<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// One lane makes 4 consecutive dims of a row. blockIdx.y: 0 keys, 1 values.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_gather_kernel(const Kv4Cache c, const Kv4Rows r) {
  constexpr int kLanes = D / 4, NG = D / 16;
  const int64_t row = ((int64_t)blockIdx.x * 128 + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool is_v = blockIdx.y != 0;
  const int h = (int)(row % c.Hkv);
  const int64_t bj = row / c.Hkv;
  const int b = (int)(bj / r.L), j = (int)(bj % r.L);
  if (b >= c.B) return;
  const int64_t t = (int64_t)(r.start != nullptr ? r.start[b] : 0) + j;
  int64_t src = -1;
  if (t < r.lens[b]) {
    src = kv4_row(c, b, t);
    if (src < 0 && lane == 0) kv4_report(c);
  }
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (src >= 0) {
    src += (int64_t)h << c.page_shift;
    const int i16 = lane / 4, u = lane % 4;
    const float scale = f16_lo(e4m3x2_f16((is_v ? c.vs : c.ks)[src * NG + i16])) *
                        (is_v ? c.v_unit : c.k_unit);
    if (!is_v) {
      const uint32_t w =
          *reinterpret_cast<const uint16_t*>(c.k + src * (D / 2) + u * (D / 8) + 2 * i16);
#pragma unroll
      for (int n = 0; n < 4; ++n) x[n] = e2m1_f32(w >> (4 * n));
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n)  // a byte holds dims g and g + 8 of the group
        x[n] = e2m1_f32(c.v[src * (D / 2) + (4 * (u & 1) + n) * NG + i16] >> (u < 2 ? 0 : 4));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= scale;
  }
  T* dst = is_v ? const_cast<T*>(reinterpret_cast<const T*>(r.v)) + b * r.v_sb + j * r.v_ss + h * r.v_sh
                : const_cast<T*>(reinterpret_cast<const T*>(r.k)) + b * r.k_sb + j * r.k_ss + h * r.k_sh;
#pragma unroll
  for (int i = 0; i < 4; ++i) dst[4 * lane + i] = held_as<T>(x[i]);
}

// ------------------------------------------------------------------ attention
// S^T = K Q^T and O^T = V^T P^T with m16n8k16 tensor instructions: 16 cached tokens, then 16 dims,
// are the rows of A, so a tile of 8 query rows (the heads of a KV group, times the new tokens)
// wastes nothing, and A comes straight from the 4-bit codes in registers. All operands are fp16:
// e2m1 codes are exact in it, query rows are scaled by a power of two so that their largest value
// is below 2^11 (what falls under fp16's range then is 2^-35 of the row's largest), and
// probabilities lie in [0, 2^7].
//   scores: the k index of an instruction is one scale group; its fp32 result times the token's
//           scale is added up, so the key scales cost no rounding.
//   values: the scale of (token, group) multiplies the probability, in fp16, before the
//           instruction of that group (its rounding, 2^-11 of each term, is that of fp16 P).
struct Kv4Args {
  Kv4Cache c;
  const void* q;
  void* o;
  int64_t q_sb, q_ss, q_sh, o_sb, o_ss, o_sh;
  const int* seqlens;
  int Lq, Hq, group, bf16;
  float scale_l2;  // scale * k_unit * log2(e) (softcap: scale * k_unit / softcap)
  float softcap;
  int causal, wl, wr, sink;
  const float* alibi;
  int row_blocks, splits;
  float* ws_o;    // [split][B * Lq * Hq][D], each normalised by its own sum
  float* ws_lse;  // [split][B * Lq * Hq], log2
};

constexpr int kAttnWarps = 4;
constexpr float kGrow = 7.f;   // a row's reference is renewed when a score passes it by 2^7
constexpr float kBelow = 3.f;  // and is then set 2^3 below the new maximum

struct Kv4Range {
  int lo, hi, sk;
};
// Keys that the row at position i sees: [lo, hi) and [0, sk).
__device__ __forceinline__ Kv4Range kv4_range(const Kv4Args& a, int len, int i) {
  const int64_t centre = (int64_t)i + len - a.Lq;
  int64_t lo = a.wl >= 0 ? centre - a.wl : 0, hi = len;
  if (a.causal) hi = min(hi, centre + 1);
  if (a.wr >= 0) hi = min(hi, centre + a.wr + 1);
  hi = max(hi, (int64_t)0);
  Kv4Range r;
  r.lo = (int)min(max(lo, (int64_t)0), (int64_t)len);
  r.hi = (int)hi;
  r.sk = (int)min((int64_t)a.sink, hi);
  return r;
}

// tanh from its exponential form; 2^inf and 2^-inf give 1 and -1, a NaN stays one.
__device__ __forceinline__ float tanh_any(float y) {
  return 1.f - 2.f * rcp(ex2(y * 2.8853900817779268f) + 1.f);  // 2 log2(e)
}

__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t h2mul(uint32_t a, uint32_t b) {
  const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// N bytes (4, 8 or 16) to words.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 16) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else if constexpr (N == 8) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x; w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// A lane's share of 16 tokens: keys of tokens g and g + 8, values of tokens 2t, 2t + 1, 2t + 8 and
// 2t + 9 (lane = 4 g + t).
template <int D>
struct Kv4Tile {
  uint32_t k[2][D / 32], v[4][D / 64], ks[2][D / 64], vs[4][D / 64];
  int token;  // first token
  bool ok;    // its page exists
};

template <int D>
__device__ __forceinline__ void load_tile(const Kv4Args& a, int b, int hk, int tile, int lane,
                                          Kv4Tile<D>& f) {
  const Kv4Cache& c = a.c;
  const int g = lane >> 2, t = lane & 3;
  f.token = tile * 16;
  const int64_t row = kv4_row(c, b, f.token);
  f.ok = row >= 0;
  if (!f.ok) {
    if (lane == 0) kv4_report(c);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      f.k[0][2 * i] = f.k[0][2 * i + 1] = f.k[1][2 * i] = f.k[1][2 * i + 1] = 0;
      f.ks[0][i] = f.ks[1][i] = 0;
#pragma unroll
      for (int n = 0; n < 4; ++n) f.v[n][i] = f.vs[n][i] = 0;
    }
    return;
  }
  const int64_t r0 = row + ((int64_t)hk << c.page_shift);
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int64_t r = r0 + g + 8 * n;
    load_words<D / 8>(c.k + r * (D / 2) + t * (D / 8), f.k[n]);
    load_words<D / 16>(c.ks + r * (D / 16), f.ks[n]);
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int64_t r = r0 + 2 * t + (n & 1) + 8 * (n >> 1);
    load_words<D / 16>(c.v + r * (D / 2) + g * (D / 16), f.v[n]);
    load_words<D / 16>(c.vs + r * (D / 16), f.vs[n]);
  }
}

// A CTA serves 8 NT query rows of one (sequence, KV head) and one share of its visible tokens; its
// warps take tiles of 16 tokens in turn, each with its own softmax reference, and join at the end.
template <int D, int NT>
__global__ void __launch_bounds__(32 * kAttnWarps) kv4_attn(const __grid_constant__ Kv4Args a) {
  constexpr int NG = D / 16, kRows = 8 * NT;
  __shared__ float s_o[kAttnWarps][kRows][D + 4];
  __shared__ float s_m[kAttnWarps][kRows], s_l[kAttnWarps][kRows];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Kv4Cache& c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  int idx = blockIdx.x;
  const int rb = idx % a.row_blocks;
  idx /= a.row_blocks;
  const int split = idx % a.splits;
  idx /= a.splits;
  const int hk = idx % c.Hkv, b = idx / c.Hkv;
  const int rows = a.Lq * a.group, r0 = rb * kRows;
  const int64_t room = (int64_t)c.max_pages << c.page_shift;
  int len = a.seqlens[b];
  if (len < 0 || len > room) {
    if (threadIdx.x == 0) kv4_report(c);
    len = len < 0 ? 0 : (int)room;
  }
  // tiles of 16 tokens: [0, s1) hold first keys, [w0, w0 + n - s1) the window
  const int i_last = (min(r0 + kRows, rows) - 1) / a.group;
  const Kv4Range first = kv4_range(a, len, r0 / a.group), last = kv4_range(a, len, i_last);
  const bool any = last.hi > first.lo;
  const int w0 = any ? first.lo / 16 : (first.lo + 15) / 16;
  const int w1 = any ? (last.hi + 15) / 16 : w0;
  const int s1 = min((last.sk + 15) / 16, w0);
  const int n = s1 + w1 - w0;
  const int per = (n + a.splits - 1) / a.splits;
  const int j0 = min(n, split * per), j1 = min(n, j0 + per);

  // query fragments: lane (g, t) has dims 16 i + 4 t .. + 3 of row g of each tile of 8 rows
  uint32_t qf[NT][NG][2];
  float inv_f[NT];  // what a row was multiplied by, inverted
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = r0 + nt * 8 + g;
    float x[NG][4];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
      if (r < rows) {
        const int64_t at = b * a.q_sb + (r / a.group) * a.q_ss +
                           (int64_t)(hk * a.group + r % a.group) * a.q_sh + 16 * i + 4 * t;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[i][e] = a.bf16 ? to_f32(reinterpret_cast<const __nv_bfloat16*>(a.q)[at + e])
                           : to_f32(reinterpret_cast<const __half*>(a.q)[at + e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[i][e]));
    }
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
    // exponent of the row's largest value; f = 2^(10 - e) brings it to [2^10, 2^11)
    int e = (int)((__float_as_uint(top) >> 23) & 255u) - 127;
    if (e > 127 || top == 0.f) e = 10;  // infinite, or a row of zeros: as it is
    e = max(e, -100);
    const float f = __uint_as_float((uint32_t)(127 + 10 - e) << 23);
    inv_f[nt] = __uint_as_float((uint32_t)(127 - 10 + e) << 23);
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      qf[nt][i][0] = h2(x[i][0] * f, x[i][1] * f);
      qf[nt][i][1] = h2(x[i][2] * f, x[i][3] * f);
    }
  }
  // this lane's score columns are rows 2t and 2t + 1 of each tile of 8
  float sc[NT][2], slope[NT][2], m[NT][2], l[NT][2];
  int centre[NT][2];
  Kv4Range seen[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      sc[nt][e] = a.scale_l2 * __shfl_sync(kFull, inv_f[nt], 4 * (2 * t + e));
      const int r = r0 + nt * 8 + 2 * t + e;
      seen[nt][e] = kv4_range(a, len, min(r, rows - 1) / a.group);
      centre[nt][e] = min(r, rows - 1) / a.group + len - a.Lq;
      slope[nt][e] = a.alibi != nullptr && r < rows
                         ? a.alibi[(int64_t)b * a.Hq + hk * a.group + r % a.group] *
                               1.4426950408889634f
                         : 0.f;
      m[nt][e] = -INFINITY;
      l[nt][e] = 0.f;
    }
  float o[NT][NG][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;

  auto tile_of = [&](int j) { return j < s1 ? j : w0 + j - s1; };
  Kv4Tile<D> f, next;
  if (j0 + warp < j1) load_tile<D>(a, b, hk, tile_of(j0 + warp), lane, f);
  for (int j = j0 + warp; j < j1; j += kAttnWarps) {
    if (j + kAttnWarps < j1) load_tile<D>(a, b, hk, tile_of(j + kAttnWarps), lane, next);
    // ---- scores of 16 tokens: s[nt][0, 1] token g, s[nt][2, 3] token g + 8
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
#pragma unroll
    for (int w = 0; w < NG / 2; ++w) {  // a word: two groups
      uint32_t ka[4], kb[4];
      e2m1x8_f16(f.k[0][w], ka);
      e2m1x8_f16(f.k[1][w], kb);
      const uint32_t sa = e4m3x2_f16(f.ks[0][w / 2] >> (16 * (w & 1)));
      const uint32_t sb = e4m3x2_f16(f.ks[1][w / 2] >> (16 * (w & 1)));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t frag[4] = {ka[2 * i], kb[2 * i], ka[2 * i + 1], kb[2 * i + 1]};
        const float fa = i ? f16_hi(sa) : f16_lo(sa), fb = i ? f16_hi(sb) : f16_lo(sb);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float x[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816(x, frag, qf[nt][2 * w + i][0], qf[nt][2 * w + i][1]);
          s[nt][0] = fmaf(fa, x[0], s[nt][0]);
          s[nt][1] = fmaf(fa, x[1], s[nt][1]);
          s[nt][2] = fmaf(fb, x[2], s[nt][2]);
          s[nt][3] = fmaf(fb, x[3], s[nt][3]);
        }
      }
    }
    // ---- logits in log2 units, masks, probabilities
    uint32_t pb[NT][2], pm[NT][2];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      bool vis[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int col = e & 1, key = f.token + g + 8 * (e >> 1);
        float x = s[nt][e] * sc[nt][col];
        if (a.softcap > 0.f) x = a.softcap * 1.4426950408889634f * tanh_any(x);
        if (a.alibi != nullptr) x -= slope[nt][col] * fabsf((float)(centre[nt][col] - key));
        const Kv4Range& r = seen[nt][col];
        vis[e] = f.ok && (key >= r.lo || key < r.sk) && key < r.hi;
        s[nt][e] = vis[e] ? x : -INFINITY;
        grow = grow || s[nt][e] > m[nt][col] + kGrow;
      }
      pm[nt][0] = transpose8x8((vis[0] ? 0xffffu : 0u) | (vis[1] ? 0xffff0000u : 0u));
      pm[nt][1] = transpose8x8((vis[2] ? 0xffffu : 0u) | (vis[3] ? 0xffff0000u : 0u));
    }
    if (__any_sync(kFull, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(s[nt][e], s[nt][e + 2]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
          if (top > m[nt][e] + kGrow) {
            const float fresh = top - kBelow;
            const float factor = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - fresh);
            m[nt][e] = fresh;
            l[nt][e] *= factor;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
              o[nt][i][e] *= factor;
              o[nt][i][e + 2] *= factor;
            }
          }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float ref = m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1];
        p[e] = ex2(s[nt][e] - ref);
        l[nt][e & 1] += p[e];
      }
      pb[nt][0] = transpose8x8(h2(p[0], p[1]));  // tokens 2t, 2t + 1 of row g
      pb[nt][1] = transpose8x8(h2(p[2], p[3]));  // tokens 2t + 8, 2t + 9
    }
    // ---- values: a byte of two tokens' codes of one dim makes one operand register
#pragma unroll
    for (int w = 0; w < NG / 4; ++w) {  // a word: four groups
      uint32_t va[4], vb[4], vc[4], vd[4];
      const uint32_t x0 = f.v[0][w], x1 = f.v[1][w], x2 = f.v[2][w], x3 = f.v[3][w];
      e2m1x8_f16((x0 & 0x0f0f0f0fu) | ((x1 << 4) & 0xf0f0f0f0u), va);  // dim g, tokens 2t, 2t + 1
      e2m1x8_f16(((x0 >> 4) & 0x0f0f0f0fu) | (x1 & 0xf0f0f0f0u), vb);  // dim g + 8
      e2m1x8_f16((x2 & 0x0f0f0f0fu) | ((x3 << 4) & 0xf0f0f0f0u), vc);  // tokens 2t + 8, 2t + 9
      e2m1x8_f16(((x2 >> 4) & 0x0f0f0f0fu) | (x3 & 0xf0f0f0f0u), vd);
      const uint32_t s01 = __byte_perm(f.vs[0][w], f.vs[1][w], 0x5140);  // groups 4w, 4w + 1
      const uint32_t s23 = __byte_perm(f.vs[0][w], f.vs[1][w], 0x7362);
      const uint32_t t01 = __byte_perm(f.vs[2][w], f.vs[3][w], 0x5140);
      const uint32_t t23 = __byte_perm(f.vs[2][w], f.vs[3][w], 0x7362);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t sp = e4m3x2_f16((i < 2 ? s01 : s23) >> (16 * (i & 1)));
        const uint32_t tp = e4m3x2_f16((i < 2 ? t01 : t23) >> (16 * (i & 1)));
        const uint32_t frag[4] = {va[i], vb[i], vc[i], vd[i]};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          // the mask again: a NaN scale of a token that a row does not see must not reach it
          mma16816(o[nt][4 * w + i], frag, h2mul(pb[nt][0], sp) & pm[nt][0],
                   h2mul(pb[nt][1], tp) & pm[nt][1]);
      }
    }
    f = next;
  }

  // ---- join the warps
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + 2 * t + e;
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(kFull, l[nt][e], d);
      if (g == 0) {
        s_m[warp][r] = m[nt][e];
        s_l[warp][r] = l[nt][e];
      }
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        s_o[warp][r][16 * i + g] = o[nt][i][e];
        s_o[warp][r][16 * i + 8 + g] = o[nt][i][e + 2];
      }
    }
  __syncthreads();
  for (int x = threadIdx.x; x < kRows * D; x += 32 * kAttnWarps) {
    const int rr = x / D, d = x % D, r = r0 + rr;
    if (r >= rows) break;
    float top = -INFINITY, sum = 0.f, val = 0.f;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, s_m[w][rr]);
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      const float f2 = s_m[w][rr] == -INFINITY ? 0.f : ex2(s_m[w][rr] - top);
      // a warp that saw only NaN scores has no maximum, but its NaN sum
      const float weight = s_l[w][rr] != s_l[w][rr] ? s_l[w][rr] : f2;
      sum += weight * s_l[w][rr];
      val += weight * s_o[w][rr][d];
    }
    const float out = sum == 0.f ? 0.f : val / sum;
    const int i = r / a.group, h = hk * a.group + r % a.group;
    if (a.splits == 1) {
      const int64_t at = b * a.o_sb + i * a.o_ss + (int64_t)h * a.o_sh + d;
      if (a.bf16) reinterpret_cast<__nv_bfloat16*>(a.o)[at] = __float2bfloat16_rn(out * c.v_unit);
      else reinterpret_cast<__half*>(a.o)[at] = __float2half_rn(out * c.v_unit);
    } else {
      const int64_t all = (int64_t)c.B * a.Lq * a.Hq;
      const int64_t at = split * all + ((int64_t)b * a.Lq + i) * a.Hq + h;
      a.ws_o[at * D + d] = out;
      if (d == 0) a.ws_lse[at] = sum == 0.f ? -INFINITY : top + log2f(sum);
    }
  }
}

// Joins the splits: one warp per output row, lanes over D.
template <int D>
__global__ void __launch_bounds__(128) kv4_join(const __grid_constant__ Kv4Args a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t all = (int64_t)a.c.B * a.Lq * a.Hq;
  const int64_t r = ((int64_t)blockIdx.x * 128 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (r >= all) return;
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) top = fmaxf(top, a.ws_lse[s * all + r]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
  float sum = 0.f, val[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) val[i] = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float lse = a.ws_lse[s * all + r];
    const float w = lse == -INFINITY ? 0.f : ex2(lse - (top == -INFINITY ? 0.f : top));
    sum += w;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      val[i] = fmaf(w, a.ws_o[(s * all + r) * D + lane + 32 * i], val[i]);
  }
  const int h = (int)(r % a.Hq);
  const int64_t bi = r / a.Hq;
  const int64_t at = bi / a.Lq * a.o_sb + bi % a.Lq * a.o_ss + h * a.o_sh;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const float out = (sum == 0.f ? 0.f : val[i] / sum) * a.c.v_unit;
    if (a.bf16) reinterpret_cast<__nv_bfloat16*>(a.o)[at + lane + 32 * i] = __float2bfloat16_rn(out);
    else reinterpret_cast<__half*>(a.o)[at + lane + 32 * i] = __float2half_rn(out);
  }
}

// ------------------------------------------------------------------ host
bool is_unit(float u) {
  int e = 0;
  return std::frexp(u, &e) == 0.5f && e >= -13 && e <= 5;  // 2^(e - 1)
}

int check_cache(const mfa_kv4_cache* c) {
  if (c == nullptr) return MFA_ERR_INVALID;
  if (c->D != 64 && c->D != 128) return MFA_ERR_UNSUPPORTED;
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)) != 0)
    return MFA_ERR_UNSUPPORTED;
  if (c->num_pages < 0 || c->Hkv < 1 || c->B < 0 || c->max_pages < 0) return MFA_ERR_INVALID;
  if ((int64_t)c->max_pages * c->page_size >= (1ll << 31)) return MFA_ERR_INVALID;
  if (!is_unit(c->k_unit) || !is_unit(c->v_unit)) return MFA_ERR_INVALID;
  if (c->B == 0) return MFA_OK;
  if (c->num_pages > 0 && (c->k == nullptr || c->v == nullptr || c->k_scale == nullptr ||
                           c->v_scale == nullptr))
    return MFA_ERR_INVALID;
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale))
    return MFA_ERR_INVALID;
  if (c->max_pages > 0 && c->block_table == nullptr) return MFA_ERR_INVALID;
  return MFA_OK;
}

Kv4Cache resolve_cache(const mfa_kv4_cache* c) {
  Kv4Cache r;
  r.k = static_cast<uint8_t*>(c->k);
  r.v = static_cast<uint8_t*>(c->v);
  r.ks = static_cast<uint8_t*>(c->k_scale);
  r.vs = static_cast<uint8_t*>(c->v_scale);
  r.table = c->block_table;
  r.table_stride = c->table_stride;
  r.num_pages = c->num_pages;
  r.page_shift = 0;
  while ((1 << r.page_shift) < c->page_size) ++r.page_shift;
  r.Hkv = c->Hkv;
  r.B = c->B;
  r.max_pages = c->max_pages;
  r.k_unit = c->k_unit;
  r.v_unit = c->v_unit;
  r.err = c->err;
  return r;
}

int check_rows(const mfa_kv4_cache* c, const mfa_kv4_rows* r, bool gather) {
  const int rc = check_cache(c);
  if (rc != MFA_OK) return rc;
  if (r == nullptr || r->L < 0) return MFA_ERR_INVALID;
  if (r->dtype != MFA_FP16 && r->dtype != MFA_BF16 && !(gather && r->dtype == MFA_FP32))
    return MFA_ERR_UNSUPPORTED;
  if (c->B == 0 || r->L == 0) return MFA_OK;
  if (r->k == nullptr || r->v == nullptr || (gather && r->lens == nullptr)) return MFA_ERR_INVALID;
  if (((int64_t)c->B * r->L * c->Hkv * (c->D / 4) + 127) / 128 >= (1ll << 31))
    return MFA_ERR_UNSUPPORTED;
  return MFA_OK;
}

Kv4Rows resolve_rows(const mfa_kv4_rows* r) {
  Kv4Rows x;
  x.k = r->k;
  x.v = r->v;
  x.k_sb = r->k_stride[0]; x.k_ss = r->k_stride[1]; x.k_sh = r->k_stride[2];
  x.v_sb = r->v_stride[0]; x.v_ss = r->v_stride[1]; x.v_sh = r->v_stride[2];
  x.start = r->start;
  x.lens = r->lens;
  x.L = r->L;
  return x;
}

template <typename T>
int launch_append(const Kv4Cache& c, const Kv4Rows& r, int D, cudaStream_t st) {
  const dim3 grid((unsigned)(((int64_t)c.B * r.L * c.Hkv * (D / 4) + 127) / 128), 2);
  if (D == 128) kv4_append_kernel<T, 128><<<grid, 128, 0, st>>>(c, r);
  else kv4_append_kernel<T, 64><<<grid, 128, 0, st>>>(c, r);
  return cudaGetLastError() == cudaSuccess ? MFA_OK : MFA_ERR_CUDA;
}
template <typename T>
int launch_gather(const Kv4Cache& c, const Kv4Rows& r, int D, cudaStream_t st) {
  const dim3 grid((unsigned)(((int64_t)c.B * r.L * c.Hkv * (D / 4) + 127) / 128), 2);
  if (D == 128) kv4_gather_kernel<T, 128><<<grid, 128, 0, st>>>(c, r);
  else kv4_gather_kernel<T, 64><<<grid, 128, 0, st>>>(c, r);
  return cudaGetLastError() == cudaSuccess ? MFA_OK : MFA_ERR_CUDA;
}

int check_fwd(const mfa_kv4_cache* c, const mfa_kv4_fwd_params* p) {
  const int rc = check_cache(c);
  if (rc != MFA_OK) return rc;
  if (p == nullptr) return MFA_ERR_INVALID;
  if (p->dtype != MFA_FP16 && p->dtype != MFA_BF16) return MFA_ERR_UNSUPPORTED;
  if (p->Lq < 0 || p->Hq < 1 || p->Hq % c->Hkv != 0 || !(p->softcap >= 0.f) || p->win_left < -1 ||
      p->win_right < -1 || p->sink < 0)
    return MFA_ERR_INVALID;
  if (c->B == 0 || p->Lq == 0) return MFA_OK;
  if (p->q == nullptr || p->o == nullptr || p->seqlens == nullptr) return MFA_ERR_INVALID;
  if ((int64_t)c->B * p->Lq * p->Hq >= (1ll << 31)) return MFA_ERR_UNSUPPORTED;
  return MFA_OK;
}

struct Kv4Plan {
  int nt, row_blocks, splits;
  size_t bytes;
};
// Tiles of 8 rows per CTA, and how many CTAs share the tokens of a (sequence, KV head): as many
// as fill the SMs once, four CTAs each, with at least 16 tiles of 16 tokens apiece.
Kv4Plan plan_fwd(const mfa_kv4_cache* c, const mfa_kv4_fwd_params* p, int sms) {
  Kv4Plan k;
  const int64_t rows = (int64_t)p->Lq * (p->Hq / c->Hkv);
  k.nt = rows > 8 ? 2 : 1;
  k.row_blocks = (int)((rows + 8 * k.nt - 1) / (8 * k.nt));
  int64_t keys = (int64_t)c->max_pages * c->page_size;
  if (p->win_left >= 0) {  // what a row block can see at most
    const int64_t right = p->causal ? 0 : p->win_right >= 0 ? p->win_right : keys;
    const int64_t window = (int64_t)p->win_left + 1 + right + 8 * k.nt + 16 + (int64_t)p->sink + 16;
    if (window < keys) keys = window;
  }
  const int64_t ctas = (int64_t)c->B * c->Hkv * k.row_blocks;
  int64_t s = 4ll * sms / ctas;
  const int64_t most = keys / 256;
  s = s < most ? s : most;
  k.splits = (int)(s < 1 ? 1 : s > 128 ? 128 : s);
  const int64_t out_rows = (int64_t)c->B * p->Lq * p->Hq;
  k.bytes = k.splits > 1 ? (size_t)k.splits * out_rows * (c->D + 1) * sizeof(float) : 0;
  return k;
}

template <int D>
int launch_fwd(const Kv4Args& a, int nt, cudaStream_t st) {
  const int64_t grid = (int64_t)a.c.B * a.c.Hkv * a.splits * a.row_blocks;
  if (grid >= (1ll << 31)) return MFA_ERR_UNSUPPORTED;
  if (nt == 1) kv4_attn<D, 1><<<(unsigned)grid, 32 * kAttnWarps, 0, st>>>(a);
  else kv4_attn<D, 2><<<(unsigned)grid, 32 * kAttnWarps, 0, st>>>(a);
  if (a.splits > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((int64_t)a.c.B * a.Lq * a.Hq + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kv4_join<D>, a) != cudaSuccess) return MFA_ERR_CUDA;
  }
  return cudaGetLastError() == cudaSuccess ? MFA_OK : MFA_ERR_CUDA;
}

}  // namespace
}  // namespace mfa

extern "C" {

int mfa_kv4_append(const mfa_kv4_cache* c, const mfa_kv4_rows* r, void* stream) {
  if (mfa::fault_injected("kv4")) return MFA_ERR_FAULT_INJECTED;
  mfa::NvtxRange range("mfa_kv4_append");
  const int rc = mfa::check_rows(c, r, false);
  if (rc != MFA_OK || c->B == 0 || r->L == 0) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  (void)cudaGetLastError();
  const mfa::Kv4Cache cc = mfa::resolve_cache(c);
  const mfa::Kv4Rows rr = mfa::resolve_rows(r);
  return r->dtype == MFA_BF16 ? mfa::launch_append<__nv_bfloat16>(cc, rr, c->D, st)
                              : mfa::launch_append<__half>(cc, rr, c->D, st);
}

int mfa_kv4_gather(const mfa_kv4_cache* c, const mfa_kv4_rows* r, void* stream) {
  if (mfa::fault_injected("kv4")) return MFA_ERR_FAULT_INJECTED;
  mfa::NvtxRange range("mfa_kv4_gather");
  const int rc = mfa::check_rows(c, r, true);
  if (rc != MFA_OK || c->B == 0 || r->L == 0) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  (void)cudaGetLastError();
  const mfa::Kv4Cache cc = mfa::resolve_cache(c);
  const mfa::Kv4Rows rr = mfa::resolve_rows(r);
  if (r->dtype == MFA_FP32) return mfa::launch_gather<float>(cc, rr, c->D, st);
  return r->dtype == MFA_BF16 ? mfa::launch_gather<__nv_bfloat16>(cc, rr, c->D, st)
                              : mfa::launch_gather<__half>(cc, rr, c->D, st);
}

size_t mfa_kv4_fwd_workspace_size(const mfa_kv4_cache* c, const mfa_kv4_fwd_params* p) {
  if (mfa::check_fwd(c, p) != MFA_OK || c->B == 0 || p->Lq == 0) return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  return mfa::plan_fwd(c, p, mfa::dev_info(dev).sms).bytes;
}

int mfa_kv4_fwd(const mfa_kv4_cache* c, const mfa_kv4_fwd_params* p, void* stream) {
  if (mfa::fault_injected("kv4")) return MFA_ERR_FAULT_INJECTED;
  mfa::NvtxRange range("mfa_kv4_fwd");
  const int rc = mfa::check_fwd(c, p);
  if (rc != MFA_OK || c->B == 0 || p->Lq == 0) return rc;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return MFA_ERR_NO_DEVICE;
  const mfa::Kv4Plan plan = mfa::plan_fwd(c, p, mfa::dev_info(dev).sms);
  if (plan.bytes > 0 && (p->workspace == nullptr || p->workspace_bytes < plan.bytes))
    return MFA_ERR_SCRATCH_TOO_SMALL;
  mfa::Kv4Args a;
  a.c = mfa::resolve_cache(c);
  a.q = p->q;
  a.o = p->o;
  a.q_sb = p->q_stride[0]; a.q_ss = p->q_stride[1]; a.q_sh = p->q_stride[2];
  a.o_sb = p->o_stride[0]; a.o_ss = p->o_stride[1]; a.o_sh = p->o_stride[2];
  a.seqlens = p->seqlens;
  a.Lq = p->Lq;
  a.Hq = p->Hq;
  a.group = p->Hq / c->Hkv;
  a.bf16 = p->dtype == MFA_BF16;
  a.softcap = p->softcap;
  a.scale_l2 = p->scale * c->k_unit *
               (p->softcap > 0.f ? 1.f / p->softcap : 1.4426950408889634f);
  a.causal = p->causal ? 1 : 0;
  a.wl = p->win_left;
  a.wr = p->win_right;
  a.sink = p->win_left >= 0 ? p->sink : 0;
  a.alibi = p->alibi;
  a.row_blocks = plan.row_blocks;
  a.splits = plan.splits;
  a.ws_o = static_cast<float*>(p->workspace);
  a.ws_lse = a.ws_o + (int64_t)plan.splits * c->B * p->Lq * p->Hq * c->D;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  (void)cudaGetLastError();
  return c->D == 128 ? mfa::launch_fwd<128>(a, plan.nt, st) : mfa::launch_fwd<64>(a, plan.nt, st);
}

}  // extern "C"
