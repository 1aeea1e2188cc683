// Per-head RMS norm of queries and keys with the position rotation in the same pass
// (mfa_qk_norm_rope, include/mfa.h). For a head row x of D values, all in fp32:
//   y = x / sqrt(mean(x^2) + eps) * w
//   (a, b) -> (a cos - b sin, a sin + b cos) over the pairs (i, i + R/2) or (2i, 2i + 1), i < R/2
// and one rounding to the tensor's type at the end. 1 / sqrt is the hardware's, off by 2^-22 at
// most, the rest IEEE fp32 (built without fast math).
#include <cuda_runtime.h>

#include <type_traits>

#include "../../include/mfa.h"
#include "common.cuh"
#include "host.cuh"
#include "ptx.cuh"

namespace mfa {
namespace {

struct NormRopeArgs {
  const void *q, *k;
  void *q_out, *k_out;
  int64_t q_sb, q_ss, q_sh, k_sb, k_ss, k_sh;  // inputs; the outputs are contiguous [B, L, H, D]
  const void *q_weight, *k_weight, *cos, *sin;
  int64_t cos_row, sin_row;
  const void* positions;
  int64_t pos_sb, pos_ss;
  int B, L, Hq, Hkv, D, R, max_pos, pos64, w_fp32, rot_fp32, interleaved;
  int w_vec, rot_vec;  // weights and tables can be read 16 bytes at a time (vector kernel)
  int segments;  // warps that share one token's heads (vector kernel)
  float eps, inv_D;
  int* err;
};

// The token's row of the tables, or -1 where its position lies outside of them.
__device__ __forceinline__ int64_t table_row(const NormRopeArgs& a, int b, int l) {
  int64_t p = l;
  if (a.positions != nullptr) {
    const int64_t i = (int64_t)b * a.pos_sb + (int64_t)l * a.pos_ss;
    p = a.pos64 ? reinterpret_cast<const int64_t*>(a.positions)[i]
                : reinterpret_cast<const int*>(a.positions)[i];
  }
  return p >= 0 && p < a.max_pos ? p : -1;
}

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// One value of a table or weight that is fp32 or of the tensors' type.
template <typename T>
__device__ __forceinline__ float load_any(const void* p, int64_t i, int fp32) {
  return fp32 ? reinterpret_cast<const float*>(p)[i] : to_f32<T>(reinterpret_cast<const T*>(p)[i]);
}

// 8 consecutive values in 16-byte aligned memory, as they are and as fp32.
template <typename T>
struct Eight {
  uint4 raw[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
  }
  __device__ __forceinline__ void get(float* v) const {
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(e[i]);
  }
  __device__ __forceinline__ void set(const float* v) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(raw)[i] = v[i];
    } else {
      constexpr bool kBF16 = std::is_same_v<T, __nv_bfloat16>;
      raw[0] = make_uint4(pack2<kBF16>(v[0], v[1]), pack2<kBF16>(v[2], v[3]),
                          pack2<kBF16>(v[4], v[5]), pack2<kBF16>(v[6], v[7]));
    }
  }
};

// 8 consecutive values of a table or weight from index i on.
template <typename T>
__device__ __forceinline__ void load_eight(const void* p, int64_t i, int fp32, int vec, float* out) {
  if (vec && fp32) {
    Eight<float> e;
    e.load(static_cast<const float*>(p) + i);
    e.get(out);
  } else if (vec) {
    Eight<T> e;
    e.load(static_cast<const T*>(p) + i);
    e.get(out);
  } else {
#pragma unroll
    for (int n = 0; n < 8; ++n) out[n] = load_any<T>(p, i + n, fp32);
  }
}

// Any head dim, strides and rotation width: one warp per head row, one value per lane and step. Not
// made for speed: 16384 tokens, 32/8 heads, bf16, D = 128 in unaligned rows 365 us (0.94 TB/s),
// D = 80 with R = 40 in split halves 296 us (the vector kernel, interleaved: 57).
template <typename T>
__global__ void __launch_bounds__(128) norm_rope_any(const __grid_constant__ NormRopeArgs a) {
  const int H = a.Hq + a.Hkv;
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= (int64_t)a.B * a.L * H) return;
  const int hh = (int)(w % H);
  const int64_t token = w / H;
  const int b = (int)(token / a.L), l = (int)(token % a.L);
  const bool is_k = hh >= a.Hq;
  const int h = is_k ? hh - a.Hq : hh;
  const T* x = is_k ? reinterpret_cast<const T*>(a.k) + b * a.k_sb + l * a.k_ss + h * a.k_sh
                    : reinterpret_cast<const T*>(a.q) + b * a.q_sb + l * a.q_ss + h * a.q_sh;
  T* o = is_k ? reinterpret_cast<T*>(a.k_out) + (token * a.Hkv + h) * a.D
              : reinterpret_cast<T*>(a.q_out) + (token * a.Hq + h) * a.D;
  const void* weight = is_k ? a.k_weight : a.q_weight;
  int64_t row = 0;
  if (a.R > 0 && (row = table_row(a, b, l)) < 0) {
    for (int d = lane; d < a.D; d += 32) o[d] = from_f32<T>(0.f);
    if (lane == 0 && a.err != nullptr) atomicExch(a.err, MFA_ERR_INVALID);
    return;
  }
  float sum = 0.f;
  for (int d = lane; d < a.D; d += 32) {
    const float v = to_f32<T>(x[d]);
    sum = fmaf(v, v, sum);
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  const float inv = rsqrtf(fmaf(sum, a.inv_D, a.eps));
  auto y = [&](int d) {
    const float v = to_f32<T>(x[d]) * inv;
    return weight != nullptr ? v * load_any<T>(weight, d, a.w_fp32) : v;
  };
  const int half = a.R / 2;
  for (int d = lane; d < a.D; d += 32) {
    float v = y(d);
    if (d < a.R) {
      const int p = a.interleaved ? d >> 1 : d < half ? d : d - half;
      const bool second = a.interleaved ? (d & 1) : d >= half;
      const int partner = a.interleaved ? d ^ 1 : second ? d - half : d + half;
      const float c = load_any<T>(a.cos, row * a.cos_row + p, a.rot_fp32);
      const float s = load_any<T>(a.sin, row * a.sin_row + p, a.rot_fp32);
      const float u = y(partner);
      v = second ? u * s + v * c : v * c - u * s;
    }
    o[d] = from_f32<T>(v);
  }
}

// D % 16 == 0 and 16-byte aligned rows. A row is LP lanes (D / 16 of them at work), each with two
// chunks of 8 values: with split halves the chunks p and p + R/16 that rotate with each other
// (R % 16 == 0), interleaved any two (R % 8 == 0), so no value crosses lanes but the sum of
// squares. A warp takes groups of heads of one token, first of q and then of k, and keeps the
// token's cosines and sines in registers; the next group's rows are on their way while one is
// worked on. Per value there are few bytes and many instructions: the arithmetic is in
// packed pairs and the registers are kept at 80 for 16-bit rows (16384 tokens, 32/8 heads, D = 128,
// bf16: 65 us, 5.3 TB/s; with scalar arithmetic 77; 64 registers: 82; fp32 106 us, 6.4 TB/s).
// kAll: R = D, every dim rotates, so none has to be kept out of its pair's rotation (66.3 us for
// that case with three sets of inputs in turn; 67.9 without the distinction).
template <typename T, bool kInterleaved, bool kAll, int LP>
__global__ void __launch_bounds__(128, sizeof(T) == 2 ? 6 : 5)
    norm_rope_vec(const __grid_constant__ NormRopeArgs a) {
  constexpr int kRows = 32 / LP;  // heads a warp holds at once
  const int w = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, sub = lane % LP;
  const int token = w / a.segments, seg = w - token * a.segments;
  if (token >= a.B * a.L) return;
  const int b = token / a.L, l = token - b * a.L;
  const bool active = sub < a.D / 16;
  const int pairs = kInterleaved ? 0 : a.R / 16;  // leading lanes whose chunks rotate together
  const int c0 = 8 * (kInterleaved || sub >= pairs ? 2 * sub : sub);
  const int c1 = kInterleaved || sub >= pairs ? c0 + 8 : c0 + a.R / 2;
  const bool rot0 = kAll || (active && c0 < a.R), rot1 = kAll || (active && c1 < a.R);
  const int gq = (a.Hq + kRows - 1) / kRows, all = gq + (a.Hkv + kRows - 1) / kRows;
  const int per = (all + a.segments - 1) / a.segments;
  const int g_end = min(all, (seg + 1) * per);
  const T* q = static_cast<const T*>(a.q) + b * a.q_sb + l * a.q_ss;
  const T* k = static_cast<const T*>(a.k) + b * a.k_sb + l * a.k_ss;
  T* qo = static_cast<T*>(a.q_out) + (int64_t)token * a.Hq * a.D;
  T* ko = static_cast<T*>(a.k_out) + (int64_t)token * a.Hkv * a.D;
  Eight<T> lo, hi;
  auto fetch = [&](int g) {
    const bool is_k = g >= gq;
    const int h = (is_k ? g - gq : g) * kRows + lane / LP;
    if (!active || g >= g_end || h >= (is_k ? a.Hkv : a.Hq)) return;
    const T* src = is_k ? k + h * a.k_sh : q + h * a.q_sh;
    lo.load(src + c0);
    hi.load(src + c1);
  };
  fetch(seg * per);
  int64_t row = 0;
  const bool bad = a.R > 0 && (row = table_row(a, b, l)) < 0;
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
  }
  if (!bad) {
    // the angles of the lane's 8 pairs stand side by side; interleaved, the last lane that
    // rotates may have 4 of them
    const int p = kInterleaved ? c0 / 2 : c0;
    if (active && rot0 && (rot1 || !kInterleaved)) {
      load_eight<T>(a.cos, row * a.cos_row + p, a.rot_fp32, a.rot_vec, cs);
      load_eight<T>(a.sin, row * a.sin_row + p, a.rot_fp32, a.rot_vec, sn);
    } else if (active && rot0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cs[i] = load_any<T>(a.cos, row * a.cos_row + p + i, a.rot_fp32);
        sn[i] = load_any<T>(a.sin, row * a.sin_row + p + i, a.rot_fp32);
      }
    }
  } else if (lane == 0 && seg == 0 && a.err != nullptr) {
    atomicExch(a.err, MFA_ERR_INVALID);
  }
  uint64_t wt[8];  // weights, in pairs
  for (int g = seg * per; g < g_end; ++g) {
    const bool is_k = g >= gq;
    const int h = (is_k ? g - gq : g) * kRows + lane / LP;
    const bool on = active && h < (is_k ? a.Hkv : a.Hq);
    if (g == seg * per || g == gq) {  // whose weights change
      const void* weight = is_k ? a.k_weight : a.q_weight;
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 1.f;
      if (weight != nullptr && active) {
        load_eight<T>(weight, c0, a.w_fp32, a.w_vec, v);
        load_eight<T>(weight, c1, a.w_fp32, a.w_vec, v + 8);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) wt[i] = f2pack(v[2 * i], v[2 * i + 1]);
    }
    float v[16];
    lo.get(v);
    hi.get(v + 8);
    fetch(g + 1);
    uint64_t x[8], sum2 = f2pack(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = f2pack(v[2 * i], v[2 * i + 1]);
      sum2 = ffma2(x[i], x[i], sum2);
    }
    float sum, odd;
    f2unpack(sum2, sum, odd);
    sum = on ? sum + odd : 0.f;
#pragma unroll
    for (int s = LP / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    const float inv = rsqrtf(fmaf(sum, a.inv_D, a.eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmul2(fmul2(x[i], f2pack(inv, inv)), wt[i]);
    // Dims that do not rotate stay as they are: turned by an angle of 0, one that is not finite
    // would make NaN of the other of its pair.
    if (!kInterleaved) {  // pairs of pairs: (u0, u1) and (v0, v1) turn by two angles
      const uint64_t turns = rot0 ? ~0ull : 0ull;  // of the other, nothing is added
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t c = f2pack(cs[2 * i], cs[2 * i + 1]), s = f2pack(sn[2 * i], sn[2 * i + 1]);
        const uint64_t u = x[i], t = x[i + 4];
        x[i] = fsub2(fmul2(u, c), fmul2(t & turns, s));
        x[i + 4] = ffma2(u & turns, s, fmul2(t, c));
        f2unpack(x[i], v[2 * i], v[2 * i + 1]);
        f2unpack(x[i + 4], v[8 + 2 * i], v[8 + 2 * i + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float u, t;
        f2unpack(x[i], u, t);
        const bool turns = i < 4 ? rot0 : rot1;
        v[2 * i] = u * cs[i] - (turns ? t : 0.f) * sn[i];
        v[2 * i + 1] = (turns ? u : 0.f) * sn[i] + t * cs[i];
      }
    }
    if (bad)
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    if (on) {
      T* o = (is_k ? ko : qo) + h * a.D;
      Eight<T> out;
      out.set(v);
      out.store(o + c0);
      out.set(v + 8);
      out.store(o + c1);
    }
  }
}

template <typename T, bool kInterleaved, bool kAll>
void launch_vec(const NormRopeArgs& a, int64_t warps, cudaStream_t st) {
  const unsigned blocks = (unsigned)((warps + 3) / 4);
  if (a.D > 64) norm_rope_vec<T, kInterleaved, kAll, 8><<<blocks, 128, 0, st>>>(a);
  else if (a.D > 32) norm_rope_vec<T, kInterleaved, kAll, 4><<<blocks, 128, 0, st>>>(a);
  else norm_rope_vec<T, kInterleaved, kAll, 2><<<blocks, 128, 0, st>>>(a);
}

template <typename T>
int launch_norm_rope(NormRopeArgs a, bool vec, int sms, cudaStream_t st) {
  const int64_t tokens = (int64_t)a.B * a.L;
  const int H = a.Hq + a.Hkv;
  const int rows = a.D > 64 ? 4 : a.D > 32 ? 8 : 16;  // heads a warp holds at once
  // few tokens: spread each one's heads over warps until every SM has 16
  a.segments = 1;
  const int most = (a.Hq + rows - 1) / rows + (a.Hkv + rows - 1) / rows;
  while (a.segments < most && tokens * a.segments < 16 * sms) ++a.segments;
  const int64_t warps = vec ? tokens * a.segments : tokens * H;
  if (warps >= (1ll << 31)) return MFA_ERR_UNSUPPORTED;
  if (!vec) norm_rope_any<T><<<(unsigned)((warps + 3) / 4), 128, 0, st>>>(a);
  else if (a.R == a.D)
    (a.interleaved ? launch_vec<T, true, true> : launch_vec<T, false, true>)(a, warps, st);
  else
    (a.interleaved ? launch_vec<T, true, false> : launch_vec<T, false, false>)(a, warps, st);
  return cudaGetLastError() == cudaSuccess ? MFA_OK : MFA_ERR_CUDA;
}

}  // namespace
}  // namespace mfa

extern "C" int mfa_qk_norm_rope(const mfa_norm_rope_params* p, void* stream) {
  if (mfa::fault_injected("norm_rope")) return MFA_ERR_FAULT_INJECTED;
  mfa::NvtxRange range("mfa_qk_norm_rope");
  if (p == nullptr) return MFA_ERR_INVALID;
  if (p->dtype < 0 || p->dtype > 2) return MFA_ERR_UNSUPPORTED;
  if (p->D < 1 || p->D > 128) return MFA_ERR_UNSUPPORTED;
  if ((p->w_dtype != p->dtype && p->w_dtype != MFA_FP32) ||
      (p->rot_dtype != p->dtype && p->rot_dtype != MFA_FP32))
    return MFA_ERR_UNSUPPORTED;
  if (p->B < 0 || p->L < 0 || p->Hq < 1 || p->Hkv < 1 || p->R < 0 || p->R > p->D || p->R % 2 != 0 ||
      p->max_pos < 0 || !(p->eps >= 0.f))
    return MFA_ERR_INVALID;
  if (p->B == 0 || p->L == 0) return MFA_OK;
  if (p->q == nullptr || p->k == nullptr || p->q_out == nullptr || p->k_out == nullptr)
    return MFA_ERR_INVALID;
  if (p->R > 0 && (p->cos == nullptr || p->sin == nullptr)) return MFA_ERR_INVALID;
  mfa::NormRopeArgs a;
  a.q = p->q; a.k = p->k; a.q_out = p->q_out; a.k_out = p->k_out;
  a.q_sb = p->q_stride[0]; a.q_ss = p->q_stride[1]; a.q_sh = p->q_stride[2];
  a.k_sb = p->k_stride[0]; a.k_ss = p->k_stride[1]; a.k_sh = p->k_stride[2];
  a.q_weight = p->q_weight; a.k_weight = p->k_weight;
  a.cos = p->cos; a.sin = p->sin;
  a.cos_row = p->cos_stride; a.sin_row = p->sin_stride;
  a.positions = p->positions;
  a.pos_sb = p->pos_stride[0]; a.pos_ss = p->pos_stride[1];
  a.B = p->B; a.L = p->L; a.Hq = p->Hq; a.Hkv = p->Hkv; a.D = p->D; a.R = p->R;
  a.max_pos = p->max_pos;
  a.pos64 = p->pos64;
  a.w_fp32 = p->w_dtype == MFA_FP32;
  a.rot_fp32 = p->rot_dtype == MFA_FP32;
  a.interleaved = p->interleaved ? 1 : 0;
  a.segments = 1;
  a.eps = p->eps;
  a.inv_D = 1.f / (float)p->D;
  a.err = p->err;
  const int es = p->dtype == MFA_FP32 ? 4 : 2;
  bool vec = p->D % 16 == 0 && p->R % (p->interleaved ? 8 : 16) == 0 && mfa::aligned16(p->q) &&
             mfa::aligned16(p->k) && mfa::aligned16(p->q_out) && mfa::aligned16(p->k_out);
  for (int i = 0; i < 3; ++i)
    vec = vec && p->q_stride[i] * es % 16 == 0 && p->k_stride[i] * es % 16 == 0;
  const int rs = p->rot_dtype == MFA_FP32 ? 4 : 2;
  a.w_vec = mfa::aligned16(p->q_weight) && mfa::aligned16(p->k_weight);
  a.rot_vec = mfa::aligned16(p->cos) && mfa::aligned16(p->sin) && p->cos_stride * rs % 16 == 0 &&
              p->sin_stride * rs % 16 == 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return MFA_ERR_NO_DEVICE;
  const int sms = mfa::dev_info(dev).sms;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  (void)cudaGetLastError();
  if (p->dtype == MFA_FP32) return mfa::launch_norm_rope<float>(a, vec, sms, st);
  if (p->dtype == MFA_BF16) return mfa::launch_norm_rope<__nv_bfloat16>(a, vec, sms, st);
  return mfa::launch_norm_rope<__half>(a, vec, sms, st);
}
