// Per-head RMS norm of queries and keys with the position rotation in the same pass
// (mfa_qk_norm_rope, include/mfa.h). For a head row x of D values, all in fp32:
//   y = x / sqrt(mean(x^2) + eps) * w
//   (a, b) -> (a cos - b sin, a sin + b cos) over the pairs (i, i + R/2) or (2i, 2i + 1), i < R/2
// and one rounding to the tensor's type at the end. Built without fast math: the square root,
// the division and the mean are IEEE fp32.
#include <cuda_runtime.h>

#include "../../include/mfa.h"
#include "common.cuh"
#include "host.cuh"

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
  int segments;  // warps that share one token's heads (vector kernel)
  float eps;
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

// N consecutive values as fp32, from 16-byte aligned memory.
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float* out) {
  constexpr int kPer = 16 / (int)sizeof(T);
  static_assert(N % kPer == 0, "whole 16-byte loads");
#pragma unroll
  for (int c = 0; c < N / kPer; ++c) {
    const uint4 raw = reinterpret_cast<const uint4*>(p)[c];
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < kPer; ++i) out[c * kPer + i] = to_f32<T>(e[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  constexpr int kPer = 16 / (int)sizeof(T);
#pragma unroll
  for (int c = 0; c < N / kPer; ++c) {
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < kPer; ++i) e[i] = from_f32<T>(v[c * kPer + i]);
    reinterpret_cast<uint4*>(p)[c] = raw;
  }
}

// Any head dim, strides and rotation width: one warp per head row, one value per lane and step.
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
  const float inv = 1.f / sqrtf(sum / (float)a.D + a.eps);
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
// squares. A warp walks heads of one token and keeps its cosines, sines and weights in registers.
template <typename T, bool kInterleaved, int LP>
__global__ void __launch_bounds__(128) norm_rope_vec(const __grid_constant__ NormRopeArgs a) {
  constexpr int kRows = 32 / LP;  // heads a warp holds at once
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31, sub = lane % LP;
  const int64_t token = w / a.segments;
  const int seg = (int)(w % a.segments);
  if (token >= (int64_t)a.B * a.L) return;
  const int b = (int)(token / a.L), l = (int)(token % a.L);
  const bool active = sub < a.D / 16;
  const int pairs = kInterleaved ? 0 : a.R / 16;  // leading lanes whose chunks rotate together
  const int c0 = 8 * (kInterleaved || sub >= pairs ? 2 * sub : sub);
  const int c1 = kInterleaved || sub >= pairs ? c0 + 8 : c0 + a.R / 2;
  const bool rot0 = active && c0 < a.R, rot1 = active && c1 < a.R;
  int64_t row = 0;
  const bool bad = a.R > 0 && (row = table_row(a, b, l)) < 0;
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
  }
  if (!bad) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool rot = kInterleaved ? (i < 4 ? rot0 : rot1) : rot0;
      const int p = kInterleaved ? (i < 4 ? c0 : c1) / 2 + (i & 3) : c0 + i;
      if (rot) {
        cs[i] = load_any<T>(a.cos, row * a.cos_row + p, a.rot_fp32);
        sn[i] = load_any<T>(a.sin, row * a.sin_row + p, a.rot_fp32);
      }
    }
  } else if (lane == 0 && seg == 0 && a.err != nullptr) {
    atomicExch(a.err, MFA_ERR_INVALID);
  }
  const int H = a.Hq + a.Hkv;
  const int per = (H + a.segments * kRows - 1) / (a.segments * kRows) * kRows;
  const int h_end = min(H, (seg + 1) * per);
  float wt[16];
  int wt_of = -1;  // whose weights wt holds: 0 the queries', 1 the keys'
  for (int h0 = seg * per; h0 < h_end; h0 += kRows) {  // the warp's lanes stay together
    const int hh = h0 + lane / LP;
    const bool on = active && hh < h_end;
    const int is_k = hh >= a.Hq;
    const int h = is_k ? hh - a.Hq : hh;
    float x[16];
    float sum = 0.f;
    if (on) {
      const T* src = is_k ? reinterpret_cast<const T*>(a.k) + b * a.k_sb + l * a.k_ss + h * a.k_sh
                          : reinterpret_cast<const T*>(a.q) + b * a.q_sb + l * a.q_ss + h * a.q_sh;
      load_vec<T, 8>(src + c0, x);
      load_vec<T, 8>(src + c1, x + 8);
#pragma unroll
      for (int i = 0; i < 16; ++i) sum = fmaf(x[i], x[i], sum);
    }
#pragma unroll
    for (int s = LP / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    if (!on) continue;
    if (wt_of != is_k) {
      wt_of = is_k;
      const void* weight = is_k ? a.k_weight : a.q_weight;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        wt[i] = weight != nullptr ? load_any<T>(weight, (i < 8 ? c0 : c1 - 8) + i, a.w_fp32) : 1.f;
    }
    const float inv = 1.f / sqrtf(sum / (float)a.D + a.eps);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = bad ? 0.f : x[i] * inv * wt[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float& u = x[kInterleaved ? 2 * i : i];
      float& v = x[kInterleaved ? 2 * i + 1 : i + 8];
      const float y0 = u * cs[i] - v * sn[i], y1 = u * sn[i] + v * cs[i];
      u = y0;
      v = y1;
    }
    T* o = is_k ? reinterpret_cast<T*>(a.k_out) + (token * a.Hkv + h) * a.D
                : reinterpret_cast<T*>(a.q_out) + (token * a.Hq + h) * a.D;
    store_vec<T, 8>(o + c0, x);
    store_vec<T, 8>(o + c1, x + 8);
  }
}

template <typename T, bool kInterleaved>
void launch_vec(const NormRopeArgs& a, int64_t warps, cudaStream_t st) {
  const unsigned blocks = (unsigned)((warps + 3) / 4);
  if (a.D > 64) norm_rope_vec<T, kInterleaved, 8><<<blocks, 128, 0, st>>>(a);
  else if (a.D > 32) norm_rope_vec<T, kInterleaved, 4><<<blocks, 128, 0, st>>>(a);
  else norm_rope_vec<T, kInterleaved, 2><<<blocks, 128, 0, st>>>(a);
}

template <typename T>
int launch_norm_rope(NormRopeArgs a, bool vec, cudaStream_t st) {
  const int64_t tokens = (int64_t)a.B * a.L;
  const int H = a.Hq + a.Hkv;
  const int rows = a.D > 64 ? 4 : a.D > 32 ? 8 : 16;  // heads a warp holds at once
  // few tokens: spread each one's heads over warps until every SM has 16
  a.segments = 1;
  const int most = (H + rows - 1) / rows;
  while (a.segments < most && tokens * a.segments < 148 * 16) ++a.segments;
  const int64_t warps = vec ? tokens * a.segments : tokens * H;
  if ((warps + 3) / 4 >= (1ll << 31)) return MFA_ERR_UNSUPPORTED;
  if (!vec) norm_rope_any<T><<<(unsigned)((warps + 3) / 4), 128, 0, st>>>(a);
  else if (a.interleaved) launch_vec<T, true>(a, warps, st);
  else launch_vec<T, false>(a, warps, st);
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
  a.err = p->err;
  const int es = p->dtype == MFA_FP32 ? 4 : 2;
  bool vec = p->D % 16 == 0 && p->R % (p->interleaved ? 8 : 16) == 0 && mfa::aligned16(p->q) &&
             mfa::aligned16(p->k) && mfa::aligned16(p->q_out) && mfa::aligned16(p->k_out);
  for (int i = 0; i < 3; ++i)
    vec = vec && p->q_stride[i] * es % 16 == 0 && p->k_stride[i] * es % 16 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  (void)cudaGetLastError();
  if (p->dtype == MFA_FP32) return mfa::launch_norm_rope<float>(a, vec, st);
  if (p->dtype == MFA_BF16) return mfa::launch_norm_rope<__nv_bfloat16>(a, vec, st);
  return mfa::launch_norm_rope<__half>(a, vec, st);
}
