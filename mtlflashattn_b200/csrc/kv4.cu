// The paged 4-bit key/value cache (mfa_kv4_*, include/mfa.h): appending, reading back, and
// attention over it. Built without fast math: the group scale's division and the quotients that
// are rounded to 4 bits are IEEE fp32, so a value on the border of two codes goes where the
// definition says.
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/mfa.h"
#include "common.cuh"
#include "host.cuh"
#include "ptx.cuh"

namespace mfa {
namespace {

template <bool B>
struct BoolC {
  static constexpr bool value = B;
};

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
// The scales in a word's four bytes as two pairs of fp16.
__device__ __forceinline__ void e4m3x4_f16(uint32_t w, uint32_t* d) {
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
      : "=r"(d[0]), "=r"(d[1])
      : "r"(w));
}
__device__ __forceinline__ float f16_lo(uint32_t h2) {
  return __low2float(*reinterpret_cast<const __half2*>(&h2));
}
__device__ __forceinline__ float f16_hi(uint32_t h2) {
  return __high2float(*reinterpret_cast<const __half2*>(&h2));
}

// x / d for 0 <= x < 2^31, with shift = ceil(log2(d)) and mul = floor(2^32 (2^shift - d) / d) + 1
// (divisor_of).
__device__ __forceinline__ int kv4_div(int x, uint32_t mul, uint32_t shift) {
  return (int)((__umulhi((uint32_t)x, mul) + (uint32_t)x) >> shift);
}

// ------------------------------------------------------------------ append and gather
// 16-bit rows on one side, 0.28 of their bytes on the other; the append is bound by issue (74 % of
// the slots taken), the gather (61 %) by nothing alone. B200, 2 x 8192 tokens, 8 heads,
// D = 128, bf16: append 20.6 us (4.2 TB/s), gather 15.4 us (5.6 TB/s). A CTA takes
// a tile of 4096 codes of one head (32 rows of D = 128, 64 of D = 64), keys or values, through
// shared memory, where the layout's permutation happens, so that every access to memory is 16
// bytes of a row; rows are (sequence, token) pairs in one line and look up their pages themselves.
struct Kv4Rows {
  void *k, *v;
  int64_t k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
  const int *start, *lens;
  int L;
  uint32_t L_mul, L_shift;  // row / L, as kv4_div
  // gather for the 16-bit forward: 1 = only the tokens that its blocks of 128 keys can touch, and
  // zeros for those of them that no row sees, which need not have a page
  int visible_only, Lq, wl, sink;
};
constexpr int kRowThreads = 128;

// Which row of the pool a (sequence, row) pair is: -1 without a page, -2 where there is none to do.
__device__ __forceinline__ int64_t kv4_find(const Kv4Cache& c, int b, int64_t t, int h, bool wanted) {
  if (!wanted) return -2;
  const int64_t row = kv4_row(c, b, t);
  return row < 0 ? -1 : row + ((int64_t)h << c.page_shift);
}

template <typename T>
struct Kv4Two;
template <>
struct Kv4Two<__half> {
  using type = __half2;
  static __device__ __forceinline__ float lo(type x) { return __low2float(x); }
  static __device__ __forceinline__ float hi(type x) { return __high2float(x); }
};
template <>
struct Kv4Two<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ float lo(type x) { return __low2float(x); }
  static __device__ __forceinline__ float hi(type x) { return __high2float(x); }
};

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) kv4_append_kernel(const Kv4Cache c, const Kv4Rows r) {
  constexpr int NG = D / 16, kTile = 8192 / D / 2, kItems = kTile * NG / kRowThreads;
  __shared__ alignas(16) uint8_t s_codes[kTile][D / 2];
  __shared__ int64_t s_dst[kTile];
  const bool is_v = blockIdx.z != 0;
  const int h = blockIdx.y;
  const int all = c.B * r.L, row0 = blockIdx.x * kTile;
  // a thread's groups of 16 dims of a row; all loads first
  uint4 raw[kItems][2];
#pragma unroll
  for (int n = 0; n < kItems; ++n) {
    const int x = (threadIdx.x + n * kRowThreads) / NG, i = threadIdx.x % NG;
    const int row = row0 + x, b = kv4_div(row, r.L_mul, r.L_shift), j = row - b * r.L;
    const T* src = is_v ? static_cast<const T*>(r.v) + b * r.v_sb + j * r.v_ss + h * r.v_sh
                        : static_cast<const T*>(r.k) + b * r.k_sb + j * r.k_ss + h * r.k_sh;
    raw[n][0] = raw[n][1] = make_uint4(0, 0, 0, 0);
    if (row < all) {
      raw[n][0] = reinterpret_cast<const uint4*>(src + 16 * i)[0];
      raw[n][1] = reinterpret_cast<const uint4*>(src + 16 * i)[1];
    }
  }
  for (int x = threadIdx.x; x < kTile; x += kRowThreads) {
    const int row = row0 + x, b = kv4_div(row, r.L_mul, r.L_shift), j = row - b * r.L;
    const bool wanted = row < all && (r.lens == nullptr || j < r.lens[b]);
    const int64_t dst =
        kv4_find(c, b, (int64_t)(wanted && r.start != nullptr ? r.start[b] : 0) + j, h, wanted);
    if (dst == -1) kv4_report(c);
    s_dst[x] = dst;
  }
  const float per_unit = 1.f / (is_v ? c.v_unit : c.k_unit);  // exact: a power of two
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kItems; ++n) {
    const int x = (threadIdx.x + n * kRowThreads) / NG, i = threadIdx.x % NG;
    const uint32_t w[8] = {raw[n][0].x, raw[n][0].y, raw[n][0].z, raw[n][0].w,
                           raw[n][1].x, raw[n][1].y, raw[n][1].z, raw[n][1].w};
    // the largest size; a NaN wins
    using T2 = typename Kv4Two<T>::type;
    T2 top2 = __habs2(*reinterpret_cast<const T2*>(&w[0]));
#pragma unroll
    for (int e = 1; e < 8; ++e)
      top2 = __hmax2_nan(top2, __habs2(*reinterpret_cast<const T2*>(&w[e])));
    const float ta = Kv4Two<T>::lo(top2), tb = Kv4Two<T>::hi(top2);
    const bool nan = ta != ta || tb != tb;
    const float want = nan ? NAN : fminf(__fdiv_rn(fmaxf(ta, tb) * per_unit, 6.f), 448.f);
    const uint32_t sbyte = __nv_cvt_float_to_fp8(want, __NV_SATFINITE, __NV_E4M3);
    const float scale = f16_lo(e4m3x2_f16(sbyte));
    // x / scale to the nearest code. With the rounded reciprocal the quotient is off by 2^-24 of
    // itself; a quotient of an 11-bit by a 4-bit number is either exactly half way between two
    // codes or at least 2^-11 of itself (2^-13 absolute) away from it, so rounding it to 2^-16 (by
    // adding and taking away 1.5 * 2^7) gives the right side and restores exact halves.
    const float inv = scale > 0.f ? __frcp_rn(scale) * per_unit : 0.f;
    // (with a NaN scale the codes do not matter)
    const uint64_t inv2 = f2pack(inv, inv), up = f2pack(192.f, 192.f), down = f2pack(-192.f, -192.f);
    float v[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const T2 x2 = *reinterpret_cast<const T2*>(&w[e]);
      const uint64_t y = ffma2(f2pack(Kv4Two<T>::lo(x2), Kv4Two<T>::hi(x2)), inv2, up);
      f2unpack(fadd2(y, down), v[2 * e], v[2 * e + 1]);
    }
    uint32_t code[8];
    if (!is_v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) code[e] = f32_e2m1x2(v[2 * e], v[2 * e + 1]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<uint16_t*>(&s_codes[x][u * (D / 8) + 2 * i]) =
            (uint16_t)(code[2 * u] | code[2 * u + 1] << 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) code[e] = f32_e2m1x2(v[e], v[e + 8]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s_codes[x][e * NG + i] = (uint8_t)code[e];
    }
    const int64_t dst = s_dst[x];
    if (dst >= 0) (is_v ? c.vs : c.ks)[dst * NG + i] = (uint8_t)sbyte;
  }
  __syncthreads();
  constexpr int kPieces = D / 32;  // 16-byte pieces of a row's codes
#pragma unroll
  for (int y = threadIdx.x; y < kTile * kPieces; y += kRowThreads) {
    const int x = y / kPieces, q = y % kPieces;
    const int64_t dst = s_dst[x];
    if (dst >= 0)
      reinterpret_cast<uint4*>((is_v ? c.v : c.k) + dst * (D / 2))[q] =
          reinterpret_cast<const uint4*>(s_codes[x])[q];
  }
}

// A pair of values as T, exact.
template <typename T>
struct Kv4Pair;
template <>
struct Kv4Pair<__half> {
  using type = uint32_t;
  static __device__ __forceinline__ type make(float a, float b) { return pack2<false>(a, b); }
};
template <>
struct Kv4Pair<__nv_bfloat16> {
  using type = uint32_t;
  static __device__ __forceinline__ type make(float a, float b) { return pack2<true>(a, b); }
};
template <>
struct Kv4Pair<float> {
  using type = float2;
  static __device__ __forceinline__ type make(float a, float b) { return make_float2(a, b); }
};

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) kv4_gather_kernel(const Kv4Cache c, const Kv4Rows r) {
  constexpr int NG = D / 16, kTile = 8192 / D / 2, kPieces = D / 32;  // 16-byte code pieces of a row
  constexpr int kPad = 16 / sizeof(T);
  using Pair = typename Kv4Pair<T>::type;
  __shared__ alignas(16) T s_out[kTile][D + kPad];
  __shared__ int64_t s_src[kTile], s_dst[kTile];
  const bool is_v = blockIdx.z != 0;
  const int h = blockIdx.y;
  const int all = c.B * r.L, row0 = blockIdx.x * kTile;
  int any = 0;
  for (int x = threadIdx.x; x < kTile; x += kRowThreads) {
    const int row = row0 + x;
    int64_t src = -3;  // a row that is not written
    if (row < all) {
      const int b = kv4_div(row, r.L_mul, r.L_shift), j = row - b * r.L;
      int len = r.lens[b];
      const int64_t t = (int64_t)(r.start != nullptr ? r.start[b] : 0) + j;
      bool touched = true, seen = true;
      if (r.visible_only) {
        if (j == 0 && (len < 0 || len > r.L) && h == 0 && !is_v) kv4_report(c);
        len = max(0, min(len, r.L));  // as the forward cuts it: the window hangs on it
        const int centre = len - r.Lq;  // of the first row
        const int lo = r.wl >= 0 && centre > r.wl ? centre - r.wl : 0;
        touched = t < ((int64_t)len + 127) / 128 * 128 &&
                  (t >= lo / 128 * 128 || t < ((int64_t)r.sink + 127) / 128 * 128);
        seen = t >= lo || t < r.sink;
      }
      if (touched) {
        src = kv4_find(c, b, t, h, seen && t < len);
        if (src == -1) kv4_report(c);
        any = 1;
      }
      s_dst[x] = is_v ? b * r.v_sb + j * r.v_ss + h * r.v_sh : b * r.k_sb + j * r.k_ss + h * r.k_sh;
    }
    s_src[x] = src;
  }
  if (!__syncthreads_or(any)) return;
  // kTile * kPieces = 128: one piece of one row per thread
  {
    const int x = threadIdx.x / kPieces, q = threadIdx.x % kPieces;
    const int64_t src = s_src[x];
    uint4 raw = make_uint4(0, 0, 0, 0);
    uint32_t sc[NG / 4];
#pragma unroll
    for (int i = 0; i < NG / 4; ++i) sc[i] = 0;
    if (src >= 0) {
      raw = reinterpret_cast<const uint4*>((is_v ? c.v : c.k) + src * (D / 2))[q];
#pragma unroll
      for (int i = 0; i < NG / 4; ++i)
        sc[i] = reinterpret_cast<const uint32_t*>((is_v ? c.vs : c.ks) + src * NG)[i];
    }
    float scale[NG];
#pragma unroll
    for (int i = 0; i < NG / 4; ++i) {
      uint32_t two[2];
      e4m3x4_f16(sc[i], two);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        scale[4 * i + 2 * e] = f16_lo(two[e]) * (is_v ? c.v_unit : c.k_unit);
        scale[4 * i + 2 * e + 1] = f16_hi(two[e]) * (is_v ? c.v_unit : c.k_unit);
      }
    }
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    auto put = [&](int d, uint32_t h2v, float f) {
      *reinterpret_cast<Pair*>(&s_out[x][d]) = Kv4Pair<T>::make(f16_lo(h2v) * f, f16_hi(h2v) * f);
    };
    if (!is_v) {
      // a word is two groups' 4 dims of one quarter u
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int u = (16 * q + 4 * n) / (D / 8), i = 4 * n % (D / 8) / 2;
        uint32_t two[4];
        e2m1x8_f16(w[n], two);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          put(16 * (i + e / 2) + 4 * u + 2 * (e & 1), two[e], scale[i + e / 2]);
      }
    } else {
      // NG bytes of dims g and g + 8; two neighbouring g make pairs
#pragma unroll
      for (int n = 0; n < 16 / NG; n += 2) {
        const int g = 16 * q / NG + n;
#pragma unroll
        for (int z = 0; z < NG / 4; ++z) {
          const uint32_t x0 = w[n * NG / 4 + z], x1 = w[(n + 1) * NG / 4 + z];
          uint32_t lo[4], hi[4];
          e2m1x8_f16((x0 & 0x0f0f0f0fu) | ((x1 << 4) & 0xf0f0f0f0u), lo);
          e2m1x8_f16(((x0 >> 4) & 0x0f0f0f0fu) | (x1 & 0xf0f0f0f0u), hi);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            put(16 * (4 * z + e) + g, lo[e], scale[4 * z + e]);
            put(16 * (4 * z + e) + 8 + g, hi[e], scale[4 * z + e]);
          }
        }
      }
    }
  }
  __syncthreads();
  constexpr int kVec = D * (int)sizeof(T) / 16;  // 16-byte pieces of an output row
#pragma unroll 4
  for (int y = threadIdx.x; y < kTile * kVec; y += kRowThreads) {
    const int x = y / kVec, q = y % kVec;
    if (s_src[x] == -3) continue;
    reinterpret_cast<uint4*>(static_cast<T*>(is_v ? r.v : r.k) + s_dst[x])[q] = reinterpret_cast<const uint4*>(s_out[x])[q];
  }
}

// ------------------------------------------------------------------ attention
// S^T = K Q^T and O^T = V^T P^T with m16n8k16 tensor instructions: 16 cached tokens, then 16 dims,
// are the rows of A, so a tile of 8 query rows (the heads of a KV group, times the new tokens)
// wastes nothing, and A comes straight from the 4-bit codes in registers. All operands are fp16:
// e2m1 codes are exact in it, query rows are scaled by a power of two so that their largest value
// is below 2^11 (what falls under fp16's range then is 2^-35 of the row's largest), and
// probabilities lie in [0, 2^15].
//   scores: the k index of an instruction is one scale group; its fp32 result times the token's
//           scale is added up, so the key scales cost no rounding.
//   values: the scale of (token, group) multiplies the codes. A code has 2 significant bits and a
//           scale 4, and their product lies in [2^-10, 2688], so it is exact in fp16.
// The one rounding to fewer bits than fp32 is that of a probability: 2^-11 of it down to 2^-25 of
// the largest that its warp has met (fp16's normal numbers), 2^-36 of that largest below. A product
// of probability and scale leaves fp16's range far sooner: with a first key of value 0 and 8192
// more of 2^-23 of its weight each, values 0.03 +- 0.02, the output was off by 5 to 7 %, now 0.2 %.
//
// A CTA is four consumer warps and a producer warp. The producer copies blocks of 128 tokens (codes
// and scales, one bulk copy each per page piece) into a ring; each consumer takes two tiles of 16 of
// the tokens, both at a time, so that one's conversions fill the other's waits.
// Work is shared out by blocks, not by sequences: the blocks of every (sequence, KV head, tile of
// query rows) that has visible keys stand in one line, which the CTAs of one wave cut into equal
// shares. A share that covers a whole unit writes its rows; one that does not leaves a partial
// result, and kv4_join adds those up. Lengths are read on the device.
//
// What bounds it is latency: no pipe is full (issue 57 %, ALU, which converts the codes, 46 %, tensor
// 22 %, memory 57 % of a copy's rate), and 13 warps per SM wait for each other's loads and results.
// B200, this kernel: 1 x 1 x 131072 tokens, 64/8 heads, D = 128: 39 us, 3.9 TB/s of codes and scales
// (60 % of a copy's rate); 32 x 1 x up to 8192, 32/8 heads: 42 us; 1 x 1 x 4096: 7.5 us. An earlier
// form's copies alone took 21 us for the first, from L2; with eight warps of one tile it took 51 us,
// not 43.
struct Kv4Args {
  Kv4Cache c;
  const void* q;
  void* o;
  int64_t q_sb, q_ss, q_sh, o_sb, o_ss, o_sh;
  const int* seqlens;
  int Lq, Hq, group, bf16;
  uint32_t group_mul, group_shift;  // row / group, as kv4_div
  float scale_l2;  // scale * k_unit * log2(e) (softcap: scale * k_unit / softcap)
  float softcap;
  int causal, wl, wr, sink;
  const float* alibi;
  int row_blocks;
  int ctas;  // that the line is cut for
  // workspace: partial sums of two units per CTA, [CTA][2][rows][D], and their references and sums
  // of weights [CTA][2][rows]
  float* ws_o;
  float2* ws_ml;
};

constexpr int kAttnWarps = 4;                  // consumer warps
constexpr int kAttnThreads = 32 * kAttnWarps + 32;
constexpr int kWarpTiles = 2;  // tiles of 16 tokens that a consumer takes of a block
constexpr int kBlockTokens = 16 * kWarpTiles * kAttnWarps;
constexpr int kBlockTiles = kBlockTokens / 16;
constexpr int kAttnStages = 3;
// Blocks per CTA at least: more leave SMs idle in short calls. 1 x 1 x 4096, 32/8 heads, a captured
// call with 2 / 4 / 8 blocks: 10.2 / 11.5 / 14.5 us; 1 x 1 x 16384: 14.5 / 15.1 / 17.7.
constexpr int kMinShare = 2;
// Beginning and ending a unit takes about as long as so many blocks. A captured call with 2 / 3 / 4:
// 32 x 1 x up to 8192 48.7 / 46.7 / 48.0 us, 8 x 1 x up to 26000 54.0 / 53.6 / 53.8, 4 x 8 x 8192 47.1 /
// 46.6 / 46.5, 1 x 8 x 32768 42.1 / 41.9 / 44.0 (32/8 heads): flat, within what the lengths make of it.
constexpr int kUnitCost = 2;
// CTAs per SM: what shared memory and 128 registers per thread allow; two tiles of rows at D = 128
// take more of both.
__host__ __device__ constexpr int kv4_ctas(int D, int nt) { return D == 128 && nt == 2 ? 2 : 3; }
constexpr float kGrow = 15.f;   // a row's reference is renewed when a score passes it by 2^15
constexpr float kBelow = 11.f;  // and is then set 2^11 below the new maximum

__device__ __forceinline__ int kv4_pos(const Kv4Args& a, int r) {  // r / group
  return kv4_div(r, a.group_mul, a.group_shift);
}

struct Kv4Range {
  int lo, hi, sk;
};
// Keys that the row at position i < Lq sees: [lo, hi) and [0, sk). Written so that nothing passes
// 32 bits: the row's centre i + len - Lq is below len.
__device__ __forceinline__ Kv4Range kv4_range(const Kv4Args& a, int len, int i) {
  const int centre = len - (a.Lq - i);
  Kv4Range r;
  r.lo = a.wl >= 0 && centre > a.wl ? centre - a.wl : 0;
  r.hi = a.causal ? centre + 1 : len;
  if (a.wr >= 0 && a.wr < len - 1 - centre) r.hi = min(r.hi, centre + a.wr + 1);
  r.hi = max(r.hi, 0);
  r.sk = min(a.sink, r.hi);
  return r;
}

__device__ __forceinline__ int kv4_length(const Kv4Args& a, int b) {
  const int room = a.c.max_pages << a.c.page_shift;  // below 2^31
  const int len = a.seqlens[b];
  return len < 0 ? 0 : min(len, room);
}

// The blocks that a tile of query rows sees: [0, s1) hold first keys, [w0, w0 + n - s1) the window.
struct Kv4Span {
  Kv4Range first, last;  // of the tile's first and last row
  int s1, w0, n;
  __device__ __forceinline__ int at(int j) const { return j < s1 ? j : w0 + j - s1; }
  // whether a row sees one of the tokens [t, t + n)
  __device__ __forceinline__ bool sees(int t, int n) const {
    return (t + n > first.lo && t < last.hi) || t < last.sk;
  }
};
template <int kRows>
__device__ __forceinline__ Kv4Span kv4_span(const Kv4Args& a, int len, int rb) {
  const int rows = a.Lq * a.group, r0 = rb * kRows;
  Kv4Span s;
  s.first = kv4_range(a, len, kv4_pos(a, r0));
  s.last = kv4_range(a, len, kv4_pos(a, min(r0 + kRows, rows) - 1));
  constexpr unsigned kT = kBlockTokens;
  const bool any = s.last.hi > s.first.lo;
  s.w0 = (unsigned)(any ? s.first.lo : s.first.lo + (int)kT - 1) / kT;
  const int w1 = any ? (int)((unsigned)(s.last.hi + (int)kT - 1) / kT) : s.w0;
  s.s1 = min((int)((unsigned)(s.last.sk + (int)kT - 1) / kT), s.w0);
  s.n = s.s1 + w1 - s.w0;
  return s;
}
// A unit's room in the line: its cost, then its blocks.
__device__ __forceinline__ int kv4_room(int n) { return n > 0 ? n + kUnitCost : 0; }
// Room of one KV head of a sequence.
template <int kRows>
__device__ __forceinline__ int kv4_head_room(const Kv4Args& a, int len) {
  int n = 0;
#pragma unroll 1
  for (int rb = 0; rb < a.row_blocks; ++rb) n += kv4_room(kv4_span<kRows>(a, len, rb).n);
  return n;
}

// What each CTA takes of a line of this length.
__device__ __forceinline__ int kv4_share(const Kv4Args& a, int total) {
  return max(kMinShare, (int)(((unsigned)total + a.ctas - 1) / a.ctas));
}

// Where a CTA stands in the line of blocks.
template <int kRows>
struct Kv4Walk {
  int b, hk, rb, j;  // unit, block within it (below 0: the unit's cost is not paid yet)
  int left;          // what is left of the share
  int len;
  Kv4Span span;
  int take;          // blocks of this unit that are this CTA's: [j, j + take)

  __device__ __forceinline__ void look(const Kv4Args& a) {
    len = kv4_length(a, b);
    span = kv4_span<kRows>(a, len, rb);
    take = 0;
    if (span.n > 0) {
      if (j < 0) {
        left += j;
        j = 0;
      }
      take = max(0, min(span.n - j, left));
    }
  }
  __device__ __forceinline__ void next(const Kv4Args& a) {
    left -= take;
    take = 0;
#pragma unroll 1
    while (left > 0 && take == 0) {
      j = -kUnitCost;
      if (++rb == a.row_blocks) {
        rb = 0;
        if (++hk == a.c.Hkv) {
          hk = 0;
          if (++b >= a.c.B) {
            left = 0;
            return;
          }
        }
      }
      look(a);
    }
  }
};

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
// All bits set in the halves that are NaN.
__device__ __forceinline__ uint32_t h2nan(uint32_t a) {
  const __half2 v = *reinterpret_cast<const __half2*>(&a);
  return __hneu2_mask(v, v);
}
// Untiled bulk copy (no multicast) of n bytes, completing on an mbarrier; both sides 16-byte
// aligned, n a multiple of 16.
__device__ __forceinline__ void bulk_load(uint8_t* dst, const uint8_t* src, uint32_t n,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(n), "r"(smem_u32(bar))
      : "memory");
}

// Whether one of four e4m3 bytes is NaN (0x7f, 0xff).
__device__ __forceinline__ bool has_nan_scale(uint32_t w) {
  return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
}

// N bytes (4, 8 or 16) of shared memory to words.
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

// Four columns of an output row from their weighted sums and the sum of the weights.
__device__ __forceinline__ void kv4_store(const Kv4Args& a, int64_t at, float4 val, float sum) {
  const float f = sum == 0.f ? 0.f : a.c.v_unit / sum;
  if (sum == 0.f) val = make_float4(0.f, 0.f, 0.f, 0.f);
  uint2 w;
  if (a.bf16) {
    w.x = pack2<true>(val.x * f, val.y * f);
    w.y = pack2<true>(val.z * f, val.w * f);
  } else {
    w.x = pack2<false>(val.x * f, val.y * f);
    w.y = pack2<false>(val.z * f, val.w * f);
  }
  *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.o) + at) = w;
}

// What the consumers have to know of a unit's part: blocks [j, j + take) of its span.
struct Kv4Unit {
  int b, hk, r0, len, j, take;  // take = 0: there are no more
  Kv4Span span;
};

template <int D, int NT>
struct Kv4Smem {
  static constexpr int kRows = 8 * NT;
  static constexpr uint32_t kCodes = kBlockTokens * D / 2, kScales = kBlockTokens * D / 16;
  static constexpr uint32_t kStage = 2 * kCodes + 2 * kScales;  // K, V, K scales, V scales
  alignas(128) uint8_t ring[kAttnStages][kStage];
  // a unit's query rows, as they are; the padding spreads 8 rows over the banks
  alignas(16) uint16_t q[kRows][D + 16];
  // the warps' sums, to be joined; until then, each warp's scales of a block
  alignas(16) float o[kAttnWarps][kRows][D + 4];
  float m[kAttnWarps][kRows], l[kAttnWarps][kRows];
  Kv4Unit unit[2];  // this one and, while its end is being written, the next one
  uint64_t full[kAttnStages], empty[kAttnStages], q_full, q_empty, met;
  unsigned bad[kAttnStages];  // bit i: tokens [16 i, 16 i + 16) of the block have no page
  int scan[kAttnThreads / 32];
  int b, hk, rb, j, share;
  int abort;
};

template <int D, int NT>
__global__ void __launch_bounds__(kAttnThreads, kv4_ctas(D, NT))
    kv4_attn(const __grid_constant__ Kv4Args a) {
  constexpr int NG = D / 16, kRows = 8 * NT;
  using Smem = Kv4Smem<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw + (((smem_u32(smem_raw) + 127u) & ~127u) -
                                                  smem_u32(smem_raw)));
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Kv4Cache& c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- where this CTA's share begins: sums over the sequences, each thread a run of them
  {
    const int run = (c.B + kAttnThreads - 1) / kAttnThreads;
    const int b0 = min(c.B, (int)threadIdx.x * run), b1 = min(c.B, b0 + run);
    int mine = 0;
    for (int b = b0; b < b1; ++b)
      mine += kv4_head_room<kRows>(a, kv4_length(a, b)) * c.Hkv;  // below 2^31 in all
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(kFull, upto, d);
      if (lane >= d) upto += x;
    }
    if (lane == 31) sm.scan[warp] = upto;
    if (threadIdx.x == 0) {
      sm.abort = 0;
      for (int i = 0; i < kAttnStages; ++i) {
        mbar_init(&sm.full[i], 1);
        mbar_init(&sm.empty[i], kAttnWarps);
      }
      mbar_init(&sm.q_full, 1);
      mbar_init(&sm.q_empty, kAttnWarps);
      mbar_init(&sm.met, kAttnWarps);
      fence_mbar_init();
    }
    __syncthreads();
    int total = 0, before = upto - mine;
#pragma unroll
    for (int w = 0; w < kAttnThreads / 32; ++w) {
      if (w < warp) before += sm.scan[w];
      total += sm.scan[w];
    }
    const int share = kv4_share(a, total);
    if (blockIdx.x == 0)
      for (int b = b0; b < b1; ++b)
        if (a.seqlens[b] != kv4_length(a, b)) kv4_report(c);
    const int64_t begin = (int64_t)share * blockIdx.x;
    if (begin >= total) return;  // all threads alike
    const int start = (int)begin;
    if (start >= before && start < before + mine) {
      int x = start - before, b = b0, len, head;
      while (true) {
        len = kv4_length(a, b);
        head = kv4_head_room<kRows>(a, len);
        if (x < head * c.Hkv) break;
        x -= head * c.Hkv;
        ++b;
      }
      sm.b = b;
      sm.hk = (int)((unsigned)x / (unsigned)head);
      x -= sm.hk * head;
      int rb = 0;
      for (int n; x >= (n = kv4_room(kv4_span<kRows>(a, len, rb).n)); ++rb) x -= n;
      sm.rb = rb;
      sm.j = x - kUnitCost;
      sm.share = min(share, total - start);
    }
    __syncthreads();
  }
  volatile int* abort_flag = &sm.abort;

  if (warp == kAttnWarps) {
    // ---------------------------------------------------------------- producer
    // A block is one piece, or as many as it has pages. The lanes look up the pages of the next 32
    // pieces at once, a batch ahead of the one whose copies are being issued.
    Kv4Walk<kRows> walk;
    walk.b = sm.b;
    walk.hk = sm.hk;
    walk.rb = sm.rb;
    walk.j = sm.j;
    walk.left = sm.share;
    walk.look(a);
    const int piece = min(kBlockTokens, 1 << c.page_shift);
    const int pshift = min(__ffs(kBlockTokens) - 1, c.page_shift);         // log2(piece)
    const int bshift = __ffs(kBlockTokens) - 1 - pshift, batch = 32 >> bshift;  // blocks
    auto page_of = [&](const Kv4Walk<kRows>& w) {  // of the batch that begins at w.j
      const int j = w.j + (lane >> bshift);
      const int t = w.span.at(j) * kBlockTokens + ((lane & ((1 << bshift) - 1)) << pshift);
      // -2: no row sees a token there, and there need not be a page
      const bool on = w.take > 0 && lane < w.take << bshift && w.span.sees(t, piece);
      return on ? c.table[(int64_t)w.b * c.table_stride + (t >> c.page_shift)] : -2;
    };
    auto skip = [&](Kv4Walk<kRows>& w) {  // to the next batch
      if (w.take > batch) {
        w.j += batch;
        w.left -= batch;
        w.take -= batch;
      } else {
        w.next(a);
      }
    };
    int it = 0, unit = 0;
    int pages = page_of(walk);
    Kv4Walk<kRows> ahead = walk;
    bool ok = true, fresh = true;  // fresh: a unit begins
    while (ok) {
      if (fresh) {  // its description, and its query rows, one per lane
        ok = __all_sync(kFull, mbar_wait(&sm.q_empty, (uint32_t)(unit & 1) ^ 1u, abort_flag));
        if (!ok) break;
        const int r0 = walk.rb * kRows, n = walk.take > 0 ? min(kRows, a.Lq * a.group - r0) : 0;
        if (lane == 0) {
          Kv4Unit& u = sm.unit[unit & 1];
          u.b = walk.b;
          u.hk = walk.hk;
          u.r0 = r0;
          u.len = walk.len;
          u.j = walk.j;
          u.take = walk.take;
          u.span = walk.span;
          mbar_expect_tx(&sm.q_full, (uint32_t)n * D * 2);
        }
        __syncwarp();
        if (lane < n) {
          const int i = kv4_pos(a, r0 + lane), h = walk.hk * a.group + r0 + lane - i * a.group;
          const int64_t at = walk.b * a.q_sb + i * a.q_ss + (int64_t)h * a.q_sh;
          bulk_load(reinterpret_cast<uint8_t*>(sm.q[lane]),
                    static_cast<const uint8_t*>(a.q) + 2 * at, D * 2, &sm.q_full);
        }
        ++unit;
        if (walk.take == 0) break;
      }
      fresh = walk.take <= batch;
      skip(ahead);
      const int pages_next = page_of(ahead);
      const int n = min(walk.take, batch);
      const int64_t base_row = (int64_t)walk.hk << c.page_shift;
#pragma unroll 1
      for (int x = 0; x < n; ++x, ++it) {
        const int slot = it % kAttnStages;
        const uint32_t phase = (uint32_t)(it / kAttnStages) & 1u;
        const int page = __shfl_sync(kFull, pages, (x << bshift) + (lane & ((1 << bshift) - 1)));
        ok = __all_sync(kFull, mbar_wait(&sm.empty[slot], phase ^ 1u, abort_flag));
        if (!ok) break;
        const bool good = lane < 1 << bshift && page >= 0 && page < c.num_pages;
        if (lane < 1 << bshift && page != -2 && !good) kv4_report(c);
        const unsigned have = __ballot_sync(kFull, good);
        if (lane == 0) {
          unsigned bad = 0;
#pragma unroll
          for (int i = 0; i < kBlockTiles; ++i)
            bad |= (have >> (16 * i >> pshift) & 1 ? 0u : 1u) << i;
          sm.bad[slot] = bad;
          mbar_expect_tx(&sm.full[slot], (uint32_t)(__popc(have) << pshift) * (D + D / 8));
        }
        __syncwarp();
        if (good) {
          const int y = lane << pshift;  // the piece's first token within the block
          const int t = walk.span.at(walk.j + x) * kBlockTokens + y;
          const int64_t row = (((int64_t)page * c.Hkv) << c.page_shift) + base_row +
                              (t & ((1 << c.page_shift) - 1));
          uint8_t* dst = sm.ring[slot];
          bulk_load(dst + y * (D / 2), c.k + row * (D / 2), piece * (D / 2), &sm.full[slot]);
          bulk_load(dst + Smem::kCodes + y * (D / 2), c.v + row * (D / 2), piece * (D / 2),
                    &sm.full[slot]);
          dst += 2 * Smem::kCodes;
          bulk_load(dst + y * (D / 16), c.ks + row * (D / 16), piece * (D / 16), &sm.full[slot]);
          bulk_load(dst + Smem::kScales + y * (D / 16), c.vs + row * (D / 16), piece * (D / 16),
                    &sm.full[slot]);
        }
      }
      walk = ahead;
      pages = pages_next;
    }
    // every copy has landed before the CTA's shared memory is given back
    for (int i = max(0, it - kAttnStages); i < it; ++i)
      mbar_wait_drain(&sm.full[i % kAttnStages], (uint32_t)(i / kAttnStages) & 1u);
    if (unit > 0) mbar_wait_drain(&sm.q_full, (uint32_t)(unit - 1) & 1u);
    if (lane == 0 && sm.abort && c.err != nullptr) atomicExch(c.err, MFA_ERR_TIMEOUT);
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int g = lane >> 2, t = lane & 3;
  // Row r of a tile's 16 is token r ^ ((r >> 1) & 1): the tokens whose values a lane reads at once
  // then lie in both halves of the banks.
  const int key_of = g ^ ((g >> 1) & 1);
  const int rows = a.Lq * a.group;
  const bool general = a.softcap > 0.f || a.alibi != nullptr;
  int it = 0;
  uint32_t meetings = 0;
  auto meet = [&] {  // the consumer warps, after what each wrote to shared memory
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.met);
    return __all_sync(kFull, mbar_wait(&sm.met, meetings++ & 1u, abort_flag)) != 0;
  };
  for (int unit = 0;; ++unit) {
    bool ok = __all_sync(kFull, mbar_wait(&sm.q_full, (uint32_t)unit & 1u, abort_flag));
    const Kv4Unit& u = sm.unit[unit & 1];
    if (!ok || u.take == 0) break;
    const int r0 = u.r0;
    // query fragments: lane (g, t) has dims 16 i + 4 t .. + 3 of row g of each tile of 8 rows
    uint32_t qf[NT][NG][2];
    float inv_f[NT];  // what a row was multiplied by, inverted
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[NG][4];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        uint2 raw = *reinterpret_cast<const uint2*>(&sm.q[nt * 8 + g][16 * i + 4 * t]);
        if (r0 + nt * 8 + g >= rows) raw = make_uint2(0, 0);
        if (a.bf16) {
          x[i][0] = __uint_as_float(raw.x << 16);
          x[i][1] = __uint_as_float(raw.x & 0xffff0000u);
          x[i][2] = __uint_as_float(raw.y << 16);
          x[i][3] = __uint_as_float(raw.y & 0xffff0000u);
        } else {
          x[i][0] = f16_lo(raw.x);
          x[i][1] = f16_hi(raw.x);
          x[i][2] = f16_lo(raw.y);
          x[i][3] = f16_hi(raw.y);
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
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.q_empty);
    // this lane's score columns are rows 2t and 2t + 1 of each tile of 8; m is the reference
    // and m_sub what is subtracted (0 while there is none)
    float sc[NT][2], m[NT][2], m_sub[NT][2], l[NT][2];
    float o[NT][NG][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sc[nt][e] = a.scale_l2 * __shfl_sync(kFull, inv_f[nt], 4 * (2 * t + e));
        m[nt][e] = -INFINITY;
        m_sub[nt][e] = l[nt][e] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
    }

    // blocks whose every token all rows see: [j_full, j_full + n_full) of the window
    const Kv4Span& see = u.span;
    const int j_full = see.s1 - see.w0 + (see.last.lo + kBlockTokens - 1) / kBlockTokens;
    const unsigned n_full = max(0, see.s1 - see.w0 + see.first.hi / kBlockTokens - j_full);

    const int j_end = u.j + u.take;
    for (int j = u.j; j < j_end; ++j, ++it) {
      const int slot = it % kAttnStages;
      ok = __all_sync(kFull, mbar_wait(&sm.full[slot], (uint32_t)(it / kAttnStages) & 1u,
                                       abort_flag));
      if (!ok) break;
      const unsigned bad = sm.bad[slot];
      const bool easy = (unsigned)(j - j_full) < n_full && bad == 0 && !general;
      const uint8_t* base = sm.ring[slot];
      // The warp converts the scales of its tiles once, not every lane those it needs: a key's as
      // fp32, a value's in pairs of the tile's rows 2p, 2p + 1 as fp16.
      const int tile0 = 16 * kWarpTiles * warp;  // this warp's tokens within the block
      float* k_scale = &sm.o[warp][0][0];                                  // [token][NG]
      uint32_t* v_scale = reinterpret_cast<uint32_t*>(k_scale + 32 * NG);  // [tile][pair][NG]
      bool clean = true;
      __syncwarp();  // the last block's have been read
      {
        const uint8_t* yp = base + 2 * Smem::kCodes + (tile0 + lane) * NG;
        uint32_t w[NG / 4], two[2];
        load_words<NG>(yp, w);
#pragma unroll
        for (int i = 0; i < NG / 4; ++i) {
          e4m3x4_f16(w[i], two);
          reinterpret_cast<float4*>(k_scale + lane * NG)[i] =
              make_float4(f16_lo(two[0]), f16_hi(two[0]), f16_lo(two[1]), f16_hi(two[1]));
        }
        // lane: tile, pair and (D = 128) half of the groups
        constexpr int kHalves = NG / 4;
        const int pair = lane / kHalves, half = lane % kHalves;  // pair: 8 tile + p
        if (pair < 8 * kWarpTiles) {
          const int first = 2 * pair + (pair & 1), second = 2 * pair + 1 - (pair & 1);
          const uint8_t* zp = base + 2 * Smem::kCodes + Smem::kScales + tile0 * NG + 4 * half;
          const uint32_t za = *reinterpret_cast<const uint32_t*>(zp + first * NG);
          const uint32_t zb = *reinterpret_cast<const uint32_t*>(zp + second * NG);
          uint4 out;
          e4m3x4_f16(__byte_perm(za, zb, 0x5140), two);
          out.x = two[0];
          out.y = two[1];
          e4m3x4_f16(__byte_perm(za, zb, 0x7362), two);
          out.z = two[0];
          out.w = two[1];
          reinterpret_cast<uint4*>(v_scale + pair * NG)[half] = out;
          // The NaN scale of a token must not reach a row that does not see it. Such tokens have
          // probability 0 there, so with finite scales nothing is left to do. (In an easy block
          // every row sees every token.)
          if (!easy) clean = !(has_nan_scale(za) || has_nan_scale(zb));
        }
        if (!easy) clean = __all_sync(kFull, clean);
      }
      __syncwarp();
      // this lane's codes: keys of rows g and g + 8 of each tile, values of rows 2t, 2t + 1, 2t + 8
      // and 2t + 9
      const int flip = t & 1, other = 1 - 2 * flip;  // rows from a token to its partner
      const uint8_t* kp = base + (tile0 + key_of) * (D / 2) + t * (D / 8);
      const uint8_t* vp = base + Smem::kCodes + (tile0 + 2 * t + flip) * (D / 2) + g * (D / 16);
      const int v_other = other * (D / 2);
      // ---- scores of the tiles: s[h][nt][0, 1] row g, s[h][nt][2, 3] row g + 8
      const bool careful = !easy;  // alike in all lanes
      float s[kWarpTiles][NT][4];
      uint32_t v[kWarpTiles][4][D / 64];
#pragma unroll
      for (int h = 0; h < kWarpTiles; ++h) {
        uint32_t k0[D / 32], k1[D / 32];
        load_words<D / 8>(kp + 16 * h * (D / 2), k0);
        load_words<D / 8>(kp + (16 * h + 8) * (D / 2), k1);
        load_words<D / 16>(vp + 16 * h * (D / 2), v[h][0]);
        load_words<D / 16>(vp + v_other + 16 * h * (D / 2), v[h][1]);
        load_words<D / 16>(vp + (16 * h + 8) * (D / 2), v[h][2]);
        load_words<D / 16>(vp + v_other + (16 * h + 8) * (D / 2), v[h][3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][nt][e] = 0.f;
        float fa[NG], fb[NG];
#pragma unroll
        for (int i = 0; i < NG; i += 4) {
          *reinterpret_cast<float4*>(fa + i) =
              *reinterpret_cast<const float4*>(k_scale + (16 * h + key_of) * NG + i);
          *reinterpret_cast<float4*>(fb + i) =
              *reinterpret_cast<const float4*>(k_scale + (16 * h + key_of + 8) * NG + i);
        }
#pragma unroll
        for (int w = 0; w < NG / 2; ++w) {  // a word: two groups
          uint32_t ka[4], kb[4];
          e2m1x8_f16(k0[w], ka);
          e2m1x8_f16(k1[w], kb);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t frag[4] = {ka[2 * i], kb[2 * i], ka[2 * i + 1], kb[2 * i + 1]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float x[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816(x, frag, qf[nt][2 * w + i][0], qf[nt][2 * w + i][1]);
              s[h][nt][0] = fmaf(fa[2 * w + i], x[0], s[h][nt][0]);
              s[h][nt][1] = fmaf(fa[2 * w + i], x[1], s[h][nt][1]);
              s[h][nt][2] = fmaf(fb[2 * w + i], x[2], s[h][nt][2]);
              s[h][nt][3] = fmaf(fb[2 * w + i], x[3], s[h][nt][3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[slot]);  // the slot is free again
      // ---- logits in log2 units, masks
#pragma unroll
      for (int h = 0; h < kWarpTiles; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][nt][e] *= sc[nt][e & 1];
      unsigned hidden[kWarpTiles] = {};  // bit 4 nt + e: the row does not see the token
      if (careful) {
#pragma unroll
        for (int h = 0; h < kWarpTiles; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = min(r0 + nt * 8 + 2 * t + (e & 1), rows - 1), i = kv4_pos(a, r);
              const int key = see.at(j) * kBlockTokens + tile0 + 16 * h + key_of + 8 * (e >> 1);
              float x = s[h][nt][e];
              if (a.softcap > 0.f) x = a.softcap * 1.4426950408889634f * tanh_any(x);
              if (a.alibi != nullptr)
                x -= a.alibi[(int64_t)u.b * a.Hq + u.hk * a.group + r - i * a.group] *
                     1.4426950408889634f * fabsf((float)(i + u.len - a.Lq - key));
              const Kv4Range seen = kv4_range(a, u.len, i);
              const bool vis = !(bad >> (kWarpTiles * warp + h) & 1) &&
                               (key >= seen.lo || key < seen.sk) && key < seen.hi;
              s[h][nt][e] = vis ? x : -INFINITY;
              hidden[h] |= (vis ? 0u : 1u) << (4 * nt + e);
            }
      }
      // ---- a row's reference, over the tiles
      float top[NT][2];
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = fmaxf(s[0][nt][e], s[0][nt][e + 2]);
#pragma unroll
          for (int h = 1; h < kWarpTiles; ++h)
            top[nt][e] = fmax3(top[nt][e], s[h][nt][e], s[h][nt][e + 2]);
          grow = grow || top[nt][e] > m[nt][e] + kGrow;
        }
      if (__any_sync(kFull, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = top[nt][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(kFull, x, d));
            if (x > m[nt][e] + kGrow) {
              const float fresh = x - kBelow;
              const float factor = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - fresh);
              m[nt][e] = m_sub[nt][e] = fresh;
              l[nt][e] *= factor;
#pragma unroll
              for (int i = 0; i < NG; ++i) {
                o[nt][i][e] *= factor;
                o[nt][i][e + 2] *= factor;
              }
            }
          }
      }
      // ---- probabilities
      uint32_t pb[kWarpTiles][NT][2];
#pragma unroll
      for (int h = 0; h < kWarpTiles; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = ex2(s[h][nt][e] - m_sub[nt][e & 1]);
          l[nt][0] += p[0] + p[2];
          l[nt][1] += p[1] + p[3];
          pb[h][nt][0] = transpose8x8(h2(p[0], p[1]));  // rows 2t, 2t + 1 of the tile for row g of q
          pb[h][nt][1] = transpose8x8(h2(p[2], p[3]));  // rows 2t + 8, 2t + 9
        }
      // ---- values: a byte of two tokens' codes of one dim makes one operand register
      auto values = [&](auto masked) {
#pragma unroll
        for (int h = 0; h < kWarpTiles; ++h) {
          uint32_t poison[NT][2];  // NaN where the row sees the token, else 0
          if constexpr (decltype(masked)::value) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                poison[nt][e] =
                    transpose8x8((hidden[h] >> (4 * nt + 2 * e) & 1 ? 0u : 0x7fffu) |
                                 (hidden[h] >> (4 * nt + 2 * e + 1) & 1 ? 0u : 0x7fff0000u));
          }
#pragma unroll
          for (int w = 0; w < NG / 4; ++w) {  // a word: four groups
            const uint32_t v0 = v[h][0][w], v1 = v[h][1][w], v2 = v[h][2][w], v3 = v[h][3][w];
            uint32_t va[4], vb[4], vc[4], vd[4];
            e2m1x8_f16((v0 & 0x0f0f0f0fu) | ((v1 << 4) & 0xf0f0f0f0u), va);  // dim g
            e2m1x8_f16(((v0 >> 4) & 0x0f0f0f0fu) | (v1 & 0xf0f0f0f0u), vb);  // dim g + 8
            e2m1x8_f16((v2 & 0x0f0f0f0fu) | ((v3 << 4) & 0xf0f0f0f0u), vc);
            e2m1x8_f16(((v2 >> 4) & 0x0f0f0f0fu) | (v3 & 0xf0f0f0f0u), vd);
            // pairs of tokens' scales, groups 4w .. 4w + 3
            const uint4 s4 = *reinterpret_cast<const uint4*>(v_scale + (8 * h + t) * NG + 4 * w);
            const uint4 t4 = *reinterpret_cast<const uint4*>(v_scale + (8 * h + t + 4) * NG + 4 * w);
            const uint32_t sp[4] = {s4.x, s4.y, s4.z, s4.w}, tp[4] = {t4.x, t4.y, t4.z, t4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t s0 = sp[i], s1 = tp[i];
              if constexpr (decltype(masked)::value) {
                // A NaN scale makes NaN of the rows that see its token: of those alone, as a
                // probability of 0 times a NaN value would be one in every row. It counts as 0
                // below, and codes (finite) times NaN or 0 are added here.
                const uint32_t n0 = h2nan(s0), n1 = h2nan(s1);
                const uint32_t codes[4] = {va[i], vb[i], vc[i], vd[i]};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma16816(o[nt][4 * w + i], codes, n0 & poison[nt][0], n1 & poison[nt][1]);
                s0 &= ~n0;
                s1 &= ~n1;
              }
              const uint32_t frag[4] = {h2mul(va[i], s0), h2mul(vb[i], s0), h2mul(vc[i], s1),
                                        h2mul(vd[i], s1)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816(o[nt][4 * w + i], frag, pb[h][nt][0], pb[h][nt][1]);
            }
          }
        }
      };
      if (clean) values(BoolC<false>{});
      else values(BoolC<true>{});
    }

    if (!ok) break;
    // ---- join the warps: a common reference per row, then their sums
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(kFull, l[nt][e], d);
        if (g == 0) sm.m[warp][nt * 8 + 2 * t + e] = m[nt][e];
      }
    if (!meet()) break;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = nt * 8 + 2 * t + e;
        float top = sm.m[0][r];
#pragma unroll
        for (int w = 1; w < kAttnWarps; ++w) top = fmaxf(top, sm.m[w][r]);
        // a warp that saw only NaN scores has no reference, but its NaN sum, which stays
        const float f = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - top);
        if (g == 0) sm.l[warp][r] = l[nt][e] * (l[nt][e] != l[nt][e] ? 1.f : f);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          sm.o[warp][r][16 * i + g] = o[nt][i][e] * f;
          sm.o[warp][r][16 * i + 8 + g] = o[nt][i][e + 2] * f;
        }
      }
    if (!meet()) break;
    const bool whole = u.take == u.span.n;
    const int64_t part = (2 * (int64_t)blockIdx.x + (u.j == 0)) * kRows;
    for (int x = threadIdx.x; x < kRows * (D / 4); x += 32 * kAttnWarps) {
      const int rr = x / (D / 4), d = x % (D / 4) * 4, r = r0 + rr;
      if (r >= rows) break;
      float sum = 0.f;
      float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(&sm.o[w][rr][d]);
        sum += sm.l[w][rr];
        val.x += y.x;
        val.y += y.y;
        val.z += y.z;
        val.w += y.w;
      }
      if (whole) {
        const int i = kv4_pos(a, r), h = u.hk * a.group + r - i * a.group;
        kv4_store(a, u.b * a.o_sb + i * a.o_ss + (int64_t)h * a.o_sh + d, val, sum);
      } else {
        *reinterpret_cast<float4*>(a.ws_o + (part + rr) * D + d) = val;
        if (d == 0) {
          float top = sm.m[0][rr];
#pragma unroll
          for (int w = 1; w < kAttnWarps; ++w) top = fmaxf(top, sm.m[w][rr]);
          a.ws_ml[part + rr] = make_float2(top, sum);
        }
      }
    }
    if (!meet()) break;
  }
}

// Adds up the partial results of a row: one block per output row. Rows that one CTA finished are
// left as they are; rows without visible keys become 0. The parts' weights are made first, all at
// once, so that the long loop only loads and adds. Launched while kv4_attn still runs, it finds its
// parts before the last CTAs end; 1 x 1 x 131072: a captured call takes 42.8 us, kv4_attn 39.2.
constexpr int kJoinThreads = 256;
constexpr int kJoinParts = 512;  // weights held at a time
template <int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) kv4_join(const __grid_constant__ Kv4Args a) {
  constexpr int kRows = 8 * NT, kLanes = D / 4, kAtOnce = kJoinThreads / kLanes;
  __shared__ float4 s_val[kAtOnce][kLanes];
  __shared__ float s_weight[kJoinParts], s_red[2][kJoinThreads / 32];
  __shared__ int s_line[2][kJoinThreads / 32];
  const int h = (int)(blockIdx.x % a.Hq);
  const int bi = blockIdx.x / a.Hq, b = bi / a.Lq, i = bi - b * a.Lq;
  const int hk = kv4_pos(a, h), r = i * a.group + h - hk * a.group, rb = r / kRows, rr = r % kRows;
  const int lane = threadIdx.x % kLanes, p = threadIdx.x / kLanes;
  const int warp = threadIdx.x / 32;
  // Where the row's unit stands in the line, while the last CTAs are still at work: what comes
  // before the sequence, and the whole.
  int before = 0, total = 0;
  for (int x = threadIdx.x; x < a.c.B; x += kJoinThreads) {
    const int n = kv4_head_room<kRows>(a, kv4_length(a, x)) * a.c.Hkv;
    total += n;
    if (x < b) before += n;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    before += __shfl_xor_sync(kFull, before, d);
    total += __shfl_xor_sync(kFull, total, d);
  }
  if (threadIdx.x % 32 == 0) {
    s_line[0][warp] = before;
    s_line[1][warp] = total;
  }
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) {
    before += s_line[0][w];
    total += s_line[1][w];
  }
  const int len = kv4_length(a, b);
  int head = 0, ahead = 0;  // room of the head's units, and of those before this one
  int n = 0;
#pragma unroll 1
  for (int x = 0; x < a.row_blocks; ++x) {
    const int y = kv4_span<kRows>(a, len, x).n;
    if (x < rb) ahead += kv4_room(y);
    if (x == rb) n = y;
    head += kv4_room(y);
  }
  const unsigned share = kv4_share(a, total), u0 = before + hk * head + ahead + kUnitCost;
  int c0 = 0, c1 = -1;
  if (n > 0) {
    c0 = u0 / share;
    c1 = (u0 + n - 1) / share;
  }
  // every block waits, also one with nothing to add: what follows this grid relies on it
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (n > 0 && c0 == c1) return;
  auto part = [&](int cta) { return (2 * (int64_t)cta + (cta == c0)) * kRows + rr; };
  const float2 none = make_float2(-INFINITY, 0.f);
  const float2 mine = c0 + (int)threadIdx.x <= c1 ? a.ws_ml[part(c0 + threadIdx.x)] : none;
  float top = mine.x;
  for (int x = c0 + threadIdx.x + kJoinThreads; x <= c1; x += kJoinThreads)
    top = fmaxf(top, a.ws_ml[part(x)].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
  if (threadIdx.x % 32 == 0) s_red[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) top = fmaxf(top, s_red[0][w]);
  float sum = 0.f;
  float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int from = c0; from <= c1; from += kJoinParts) {
    const int to = min(c1 + 1, from + kJoinParts);
    if (from > c0) __syncthreads();
    for (int x = from + threadIdx.x; x < to; x += kJoinThreads) {
      const float2 ml = x == c0 + (int)threadIdx.x ? mine : a.ws_ml[part(x)];
      const float f = ml.y != ml.y ? ml.y : ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
      s_weight[x - from] = f;
      sum = fmaf(f, ml.y, sum);
    }
    __syncthreads();
#pragma unroll 8
    for (int x = from + p; x < to; x += kAtOnce) {
      const float f = s_weight[x - from];
      const float4 y = reinterpret_cast<const float4*>(a.ws_o + part(x) * D)[lane];
      val.x = fmaf(f, y.x, val.x);
      val.y = fmaf(f, y.y, val.y);
      val.z = fmaf(f, y.z, val.z);
      val.w = fmaf(f, y.w, val.w);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
  if (threadIdx.x % 32 == 0) s_red[1][warp] = sum;
  s_val[p][lane] = val;
  __syncthreads();
  if (threadIdx.x >= kLanes) return;
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) sum += s_red[1][w];
  val = s_val[0][lane];
#pragma unroll
  for (int x = 1; x < kAtOnce; ++x) {
    const float4 y = s_val[x][lane];
    val.x += y.x;
    val.y += y.y;
    val.z += y.z;
    val.w += y.w;
  }
  kv4_store(a, b * a.o_sb + i * a.o_ss + (int64_t)h * a.o_sh + 4 * lane, val, sum);
}

// ------------------------------------------------------------------ host
void divisor_of(int d, uint32_t* mul, uint32_t* shift) {
  *shift = 0;
  while ((1ull << *shift) < (uint64_t)d) ++*shift;
  *mul = (uint32_t)((((1ull << *shift) - d) << 32) / d + 1);
}

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
  // token indices, and what is added to them for a block, stay within 32 bits
  if ((int64_t)c->max_pages * c->page_size > (1ll << 31) - 4096) return MFA_ERR_INVALID;
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
  // rows are read and written in 16-byte pieces
  const int es = r->dtype == MFA_FP32 ? 4 : 2;
  bool ok = aligned16(r->k) && aligned16(r->v);
  for (int i = 0; i < 3; ++i)
    ok = ok && r->k_stride[i] * es % 16 == 0 && r->v_stride[i] * es % 16 == 0;
  return ok ? MFA_OK : MFA_ERR_INVALID;
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
  divisor_of(x.L > 0 ? x.L : 1, &x.L_mul, &x.L_shift);
  x.visible_only = 0;
  return x;
}

template <typename T, int D, bool kGather>
int launch_rows(const Kv4Cache& c, const Kv4Rows& r, cudaStream_t st) {
  constexpr int kTile = 8192 / D / 2;
  const int64_t tiles = ((int64_t)c.B * r.L + kTile - 1) / kTile;
  if ((int64_t)c.B * r.L + kTile >= (1ll << 31) || c.Hkv > 65535) return MFA_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)tiles, c.Hkv, 2);
  if constexpr (kGather) kv4_gather_kernel<T, D><<<grid, kRowThreads, 0, st>>>(c, r);
  else kv4_append_kernel<T, D><<<grid, kRowThreads, 0, st>>>(c, r);
  return cudaGetLastError() == cudaSuccess ? MFA_OK : MFA_ERR_CUDA;
}
template <typename T, bool kGather>
int launch_rows(const Kv4Cache& c, const Kv4Rows& r, int D, cudaStream_t st) {
  return D == 128 ? launch_rows<T, 128, kGather>(c, r, st) : launch_rows<T, 64, kGather>(c, r, st);
}

// Query rows per KV head up to which the codes are read directly. Each 16 rows read and convert
// the codes again, while the other way converts them once, to memory, for the tensor-core forward.
// Measured on B200 (us a captured call, directly / not) at 32, 48, 64 and 96 rows: 4 x 8192 keys, 32/8
// heads, D = 128: 47/69, 65/72, 80/69, 117/70; 1 x 32768: 42/68, 56/68, 70/68, 102/72; and at 16 and
// 32 rows of D = 64, 16 x 2048 keys, 16/16 heads: 51/67, 87/67.
int64_t direct_rows(int D) { return D == 128 ? 48 : 16; }

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
  // the direct path's line is counted in 32 bits
  const int64_t rows = (int64_t)p->Lq * (p->Hq / c->Hkv);
  if (rows <= direct_rows(c->D) &&
      (double)c->B * c->Hkv * ((rows + 7) / 8) *
              ((double)c->max_pages * c->page_size / kBlockTokens + 10) >= 2147483648.0)
    return MFA_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(p->o) % 8 != 0) return MFA_ERR_INVALID;
  for (int i = 0; i < 3; ++i)
    if (p->o_stride[i] % 4 != 0 || p->q_stride[i] % 8 != 0) return MFA_ERR_INVALID;
  if (!aligned16(p->q)) return MFA_ERR_INVALID;
  return MFA_OK;
}

struct Kv4Plan {
  bool direct;
  // straight from the codes
  int nt, row_blocks, ctas;
  int64_t o;           // bytes of the partial sums
  // by way of 16-bit keys and values
  int seqs;            // sequences at a time
  int64_t kv;          // bytes of their keys, and of their values
  size_t bytes;
};

constexpr int64_t kStageBytes = 512ll << 20;  // keys and values of the sequences done at a time

// The forward of sequences [b0, b0 + n) over keys and values in 16 bits, [n, capacity, Hkv, D].
mfa_fwd_params staged_params(const mfa_kv4_cache* c, const mfa_kv4_fwd_params* p, int b0, int n,
                             void* k, void* v) {
  mfa_fwd_params f;
  std::memset(&f, 0, sizeof(f));
  const int64_t row = (int64_t)c->Hkv * c->D, room = (int64_t)c->max_pages * c->page_size;
  f.q = static_cast<const uint8_t*>(p->q) + 2 * b0 * p->q_stride[0];
  f.o = static_cast<uint8_t*>(p->o) + 2 * b0 * p->o_stride[0];
  f.k = k;
  f.v = v;
  for (int i = 0; i < 3; ++i) {
    f.q_stride[i] = p->q_stride[i];
    f.o_stride[i] = p->o_stride[i];
    f.k_stride[i] = f.v_stride[i] = i == 0 ? room * row : i == 1 ? row : c->D;
  }
  f.B = n;
  f.Hq = p->Hq;
  f.Hkv = c->Hkv;
  f.Lq = p->Lq;
  f.Lk = (int)room;
  f.D = c->D;
  f.scale = p->scale;
  f.softcap = p->softcap;
  f.causal = p->causal;
  f.win_left = p->win_left;
  f.win_right = p->win_right;
  f.sink = p->sink;
  f.alibi = p->alibi != nullptr ? p->alibi + (int64_t)b0 * p->Hq : nullptr;
  f.dtype = p->dtype;
  f.o_dtype = -1;
  f.err = c->err;
  return f;
}

Kv4Plan plan_fwd(const mfa_kv4_cache* c, const mfa_kv4_fwd_params* p, int sms) {
  Kv4Plan k;
  const int64_t rows = (int64_t)p->Lq * (p->Hq / c->Hkv);
  k.direct = rows <= direct_rows(c->D) || c->max_pages == 0;
  if (!k.direct) {
    const int64_t each = 2ll * c->max_pages * c->page_size * c->Hkv * c->D;
    k.seqs = (int)std::max<int64_t>(1, std::min<int64_t>(c->B, kStageBytes / 2 / each));
    k.kv = k.seqs * each;
    // the last group may be smaller and split its keys more
    size_t split = 0;
    for (int n : {k.seqs, c->B % k.seqs}) {
      if (n == 0) continue;
      // the plan asks for no address: any aligned one stands for the keys'
      void* any = const_cast<void*>(p->q);
      const mfa_fwd_params f = staged_params(c, p, 0, n, any, any);
      split = std::max(split, mfa_fwd_workspace_size(&f));
    }
    k.bytes = (size_t)(2 * k.kv) + split;
    return k;
  }
  // One wave of resident CTAs, whatever the lengths are.
  k.nt = rows > 8 ? 2 : 1;
  // (a table without pages may come with any number of rows: none of them has a place in the line)
  k.row_blocks = c->max_pages == 0 ? 0 : (int)((rows + 8 * k.nt - 1) / (8 * k.nt));
  k.ctas = sms * kv4_ctas(c->D, k.nt);
  const int64_t parts = 2ll * k.ctas * 8 * k.nt;
  k.o = parts * c->D * 4;
  k.bytes = (size_t)(k.o + parts * 8);
  return k;
}

// Keys and values to 16 bits, then the tensor-core forward, a group of sequences after another.
int run_staged_fwd(const mfa_kv4_cache* c, const mfa_kv4_fwd_params* p, const Kv4Plan& plan,
                   cudaStream_t st) {
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  for (int b0 = 0; b0 < c->B; b0 += plan.seqs) {
    const int n = std::min(plan.seqs, c->B - b0);
    mfa_fwd_params f = staged_params(c, p, b0, n, ws, ws + plan.kv);
    f.workspace = ws + 2 * plan.kv;
    f.workspace_bytes = p->workspace_bytes - 2 * plan.kv;
    Kv4Cache cc = resolve_cache(c);
    cc.B = n;
    cc.table += b0 * cc.table_stride;
    Kv4Rows r;
    r.k = ws;
    r.v = ws + plan.kv;
    r.k_sb = r.v_sb = f.k_stride[0];
    r.k_ss = r.v_ss = f.k_stride[1];
    r.k_sh = r.v_sh = f.k_stride[2];
    r.start = nullptr;
    r.lens = p->seqlens + b0;
    r.L = f.Lk;
    divisor_of(r.L, &r.L_mul, &r.L_shift);
    r.visible_only = 1;
    r.Lq = p->Lq;
    r.wl = p->win_left;
    r.sink = p->win_left >= 0 ? p->sink : 0;
    int rc = p->dtype == MFA_BF16 ? launch_rows<__nv_bfloat16, true>(cc, r, c->D, st)
                                  : launch_rows<__half, true>(cc, r, c->D, st);
    if (rc == MFA_OK) rc = forward_padded(&f, p->seqlens + b0, st);
    if (rc != MFA_OK) return rc;
  }
  return MFA_OK;
}

template <int D, int NT>
int launch_fwd(const Kv4Args& a, int ctas, int dev, cudaStream_t st) {
  constexpr int smem = (int)sizeof(Kv4Smem<D, NT>) + 128;
  if (ensure_smem(kv4_attn<D, NT>, dev, smem) != cudaSuccess) return MFA_ERR_CUDA;
  kv4_attn<D, NT><<<ctas, kAttnThreads, smem, st>>>(a);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.c.B * a.Lq * a.Hq));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kv4_join<D, NT>, a) != cudaSuccess) return MFA_ERR_CUDA;
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
  return r->dtype == MFA_BF16 ? mfa::launch_rows<__nv_bfloat16, false>(cc, rr, c->D, st)
                              : mfa::launch_rows<__half, false>(cc, rr, c->D, st);
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
  if (r->dtype == MFA_FP32) return mfa::launch_rows<float, true>(cc, rr, c->D, st);
  return r->dtype == MFA_BF16 ? mfa::launch_rows<__nv_bfloat16, true>(cc, rr, c->D, st)
                              : mfa::launch_rows<__half, true>(cc, rr, c->D, st);
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
  if (p->workspace == nullptr || p->workspace_bytes < plan.bytes) return MFA_ERR_SCRATCH_TOO_SMALL;
  if (!mfa::aligned16(p->workspace)) return MFA_ERR_INVALID;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  (void)cudaGetLastError();
  if (!plan.direct) return mfa::run_staged_fwd(c, p, plan, st);
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
  mfa::divisor_of(a.group, &a.group_mul, &a.group_shift);
  a.softcap = p->softcap;
  a.scale_l2 = p->scale * c->k_unit *
               (p->softcap > 0.f ? 1.f / p->softcap : 1.4426950408889634f);
  a.causal = p->causal ? 1 : 0;
  a.wl = p->win_left;
  a.wr = p->win_right;
  a.sink = p->win_left >= 0 ? p->sink : 0;
  a.alibi = p->alibi;
  a.row_blocks = plan.row_blocks;
  a.ctas = plan.ctas;
  a.ws_o = static_cast<float*>(p->workspace);
  a.ws_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(p->workspace) + plan.o);
  if (c->D == 128)
    return plan.nt == 1 ? mfa::launch_fwd<128, 1>(a, plan.ctas, dev, st)
                        : mfa::launch_fwd<128, 2>(a, plan.ctas, dev, st);
  return plan.nt == 1 ? mfa::launch_fwd<64, 1>(a, plan.ctas, dev, st)
                      : mfa::launch_fwd<64, 2>(a, plan.ctas, dev, st);
}

}  // extern "C"
