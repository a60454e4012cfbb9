// Residual add + RMS norm + int8 tokens with one scale per 128-k chunk.
//
//   h = x + r,  y = h * rsqrt(mean(h^2) + eps) * w,
//   s = max(max|y| over the chunk, 1e-6) * (1 / 127),  q = rint(y * (1 / s))
//
// One pass over the data: a CTA holds its row in registers between the sum of squares
// and the quantisation, so x and r are read once and h, q, s written once.  Half a warp
// holds a chunk (8 values a thread), so the chunk's maximum is four shuffles.  Bound by HBM:
// 2048 x 5120 fp32 in 23.4 us (5.8 TB/s, 0.89 of the measured copy rate), 8193 x 2048 fp16
// in 24.5 us (4.8 TB/s; twice the arithmetic a byte), 11 x 5120 in 2.9 us (latency).
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "tlx_internal.h"

namespace tlx {
namespace {

// max that keeps a NaN: a row with one gets NaN scales, not zeros that hide it
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

struct NormArgs {
  const void *x, *r;
  int64_t ldx, ldr;
  const float* w;
  float eps;
  int m, k;
  void* h;
  int64_t ldh;
  int8_t* xq;
  int64_t ldq;
  float* sx;
  int32_t* rs;
};

template <typename T>
__device__ __forceinline__ void get8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (std::is_same_v<T, __half>) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
        f[2 * j] = t.x;
        f[2 * j + 1] = t.y;
      } else {
        f[2 * j] = __uint_as_float(u[j] << 16);
        f[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void put8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (std::is_same_v<T, __half>) {
        u[j] = h2_bits(__floats2half2_rn(f[2 * j], f[2 * j + 1]));
      } else {
        const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// kVec: 8-value vectors a thread holds
template <typename TX, typename TR, int kVec>
__global__ void __launch_bounds__(1024) add_rms_norm_q8_kernel(const NormArgs a) {
  __shared__ float red[32];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  const int nv = a.k >> 3;
  const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
  const TR* r = a.r ? static_cast<const TR*>(a.r) + row * a.ldr : nullptr;
  TR* h = a.h ? static_cast<TR*>(a.h) + row * a.ldh : nullptr;
  float f[kVec][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nv) {
      get8(x + 8 * v, f[i]);
      if (r) {
        float g[8];
        get8(r + 8 * v, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] += g[j];
      }
      if (h) put8(h + 8 * v, f[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(f[i][j], f[i][j], ss);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) red[warp] = ss;
  __syncthreads();
  float total = 0.f;
  for (int w = 0; w < warps; ++w) total += red[w];
  const float rstd = rsqrtf(total / static_cast<float>(a.k) + a.eps);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    const bool ok = v < nv;   // a chunk's 16 threads agree: nv is a multiple of 16
    float y[8];
    float am = 0.f;
    if (ok) {
      float w[8];
      get8(a.w + 8 * v, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = f[i][j] * rstd * w[j];
        am = max_nan(am, fabsf(y[j]));
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) am = max_nan(am, __shfl_xor_sync(0xffffffffu, am, o));
    const float s = max_nan(am, 1e-6f) * (1.0f / 127.0f);
    // y times one reciprocal a chunk: |y / s| <= 127 needs no clamp, and a code differs from
    // the IEEE quotient's only where y / s is within 127 2^-22 of a half-integer.  Eight
    // divisions a thread made the 16-bit rows compute bound (28.0 -> 24.5 us at 8193 x 2048).
    const float to_code = __fdiv_rn(1.0f, s);
    int sum = 0;
    if (ok) {
      uint32_t p[2] = {0u, 0u};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int q = __float2int_rn(y[j] * to_code);
        p[j >> 2] |= (static_cast<uint32_t>(q) & 0xFFu) << (8 * (j & 3));
        sum += q;
      }
      *reinterpret_cast<uint2*>(a.xq + row * a.ldq + 8 * v) = make_uint2(p[0], p[1]);
      if ((lane & 15) == 0) a.sx[row * (a.k >> 7) + (v >> 4)] = s;
    }
    if (a.rs) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (ok && (lane & 15) == 0) a.rs[row * (a.k >> 7) + (v >> 4)] = sum;
    }
  }
}

template <typename TX, typename TR>
int launch_norm(const NormArgs& a, cudaStream_t s) {
  const int nv = a.k >> 3;
  // vectors a thread holds: one where it fits (a row ends soonest: 11 x 5120 in 3.1 us, with
  // two 3.7), two where many 16-bit rows keep the SMs full (twice the bytes in flight a
  // thread: 8193 x 2048 7 % faster, fp32 2048 x 5120 4 % slower)
  const bool two = sizeof(TX) + sizeof(TR) == 4 && a.m >= 1024;
  const int vec = nv <= 1024 && !two ? 1 : nv <= 2048 ? 2 : 4;
  const int threads = std::max(32, ((nv + vec - 1) / vec + 31) & ~31);
  if (vec == 1) add_rms_norm_q8_kernel<TX, TR, 1><<<a.m, threads, 0, s>>>(a);
  else if (vec == 2) add_rms_norm_q8_kernel<TX, TR, 2><<<a.m, threads, 0, s>>>(a);
  else add_rms_norm_q8_kernel<TX, TR, 4><<<a.m, threads, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? TLX_OK : TLX_ERR_LAUNCH;
}

template <typename TX>
int launch_norm_r(const NormArgs& a, int r_dtype, cudaStream_t s) {
  if (r_dtype == TLX_DT_F32) return launch_norm<TX, float>(a, s);
  if (r_dtype == TLX_DT_F16) return launch_norm<TX, __half>(a, s);
  return launch_norm<TX, __nv_bfloat16>(a, s);
}

bool al(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool known(int dt) { return dt == TLX_DT_F32 || dt == TLX_DT_F16 || dt == TLX_DT_BF16; }
int size_of(int dt) { return dt == TLX_DT_F32 ? 4 : 2; }

}  // namespace
}  // namespace tlx

using namespace tlx;

extern "C" int tlx_add_rms_norm_q8(const void* x, int x_dtype, int64_t ldx, const void* residual, int r_dtype,
                                   int64_t ldr, const float* weight, float eps, int m, int64_t k, void* h_out,
                                   int64_t ldh, int8_t* xq, int64_t ldq, float* sx, int32_t* rs, void* stream) {
  if (!x || !weight || !xq || !sx) return TLX_ERR_NULL;
  if (!known(x_dtype) || !known(r_dtype)) return TLX_ERR_DTYPE;
  if (m < 1 || m > (1 << 24) || k < 128 || k % 128 || k > 32768 || !(eps >= 0.f)) return TLX_ERR_SHAPE;
  if (ldx < k || ldq < k || (residual && ldr < k) || (h_out && ldh < k)) return TLX_ERR_SHAPE;
  if (!al(x, 16) || ldx * size_of(x_dtype) % 16 || !al(weight, 16) || !al(xq, 8) || ldq % 8) return TLX_ERR_ALIGN;
  if (residual && (!al(residual, 16) || ldr * size_of(r_dtype) % 16)) return TLX_ERR_ALIGN;
  if (h_out && (!al(h_out, 16) || ldh * size_of(r_dtype) % 16)) return TLX_ERR_ALIGN;
  const NormArgs a{x, residual, ldx, ldr, weight, eps, m, static_cast<int>(k), h_out, ldh, xq, ldq, sx, rs};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x_dtype == TLX_DT_F32) return launch_norm_r<float>(a, r_dtype, s);
  if (x_dtype == TLX_DT_F16) return launch_norm_r<__half>(a, r_dtype, s);
  return launch_norm_r<__nv_bfloat16>(a, r_dtype, s);
}
