// RMS norm (with the residual's addition in front) whose output is e4m3 with scales: what the e4m3 experts take.
//   r = bf16(x + residual)   (or x)          the residual stream as it is stored is what is normalised
//   y = r * rsqrt(mean(r^2) + eps) * weight   fp32, not rounded before it is quantised
//   s = max(max |y| over the group, 1e-10) / 448,   q = e4m3(y / s)      group = 128 columns or the whole token
//   (y times 1 / s, each rounded to fp32: 2^-23 of y / s at most, against the 2^-4 of e4m3)
//   normed = bf16(y)                          optional, for the router that reads the same activations
// ops.add_rms_norm rounds between the two products and before the weight (it follows the reference's bits); here each
// output is rounded once, from fp32.
//
// Bound: HBM. A token needs 2 (+ 2 residual in, + 2 residual out) bytes in and 1 (+ 2 normed) bytes out per column
// and is read once: one CTA per token keeps the rounded sum in registers (two 16-byte vectors a thread), so that the
// only exchange is the block's sum of squares, and the group's maximum is a shuffle over 16 lanes (8 columns each).
// T = 8192, H = 4096 with residual and bf16 output: 49 us, 6.1 TB/s, 0.94 of the copy rate
// (51 us and 0.91 as a call from Python); T = 64, H = 2048: 2.5 us.
#include <cuda_fp8.h>

#include "launch.cuh"
#include "moe_b200_internal.cuh"
#include "rms_norm_row.cuh"

namespace moe_b200 {

namespace {

constexpr float kFp8Max = 448.f;
constexpr float kScaleFloor = 1e-10f;

// Maximum that keeps a NaN, so that a group with one says so in its scale.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

template <int kVecs, bool kAdd, bool kPerToken>
__global__ void __launch_bounds__(1024)
rms_norm_quant_fp8_kernel(uint8_t* __restrict__ q, float* __restrict__ scales, __nv_bfloat16* normed,
                          __nv_bfloat16* residual_out, const __nv_bfloat16* residual, const __nv_bfloat16* input,
                          const __nv_bfloat16* __restrict__ weight, float eps, int H) {
  __shared__ float red[2][32];
  grid_dependency_launch();
  grid_dependency_wait();
  const int t = threadIdx.x;
  const int lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
  const size_t off = static_cast<size_t>(blockIdx.x) * H;
  Bf16x8 v[kVecs];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int c = 8 * (i * blockDim.x + t);
    v[i].u = make_uint4(0, 0, 0, 0);
    if (c < H) {
      v[i].u = *reinterpret_cast<const uint4*>(input + off + c);
      if (kAdd) {
        Bf16x8 r;
        r.u = *reinterpret_cast<const uint4*>(residual + off + c);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i].h[j] = __float2bfloat16_rn(__bfloat162float(v[i].h[j]) + __bfloat162float(r.h[j]));
        *reinterpret_cast<uint4*>(residual_out + off + c) = v[i].u;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = __bfloat162float(v[i].h[j]);
      sum = fmaf(x, x, sum);
    }
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if (lane == 0) red[0][warp] = sum;
  __syncthreads();
  float total = lane < warps ? red[0][lane] : 0.f;
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) total += __shfl_xor_sync(0xffffffffu, total, m);
  const float rstd = rsqrtf(total / H + eps);

  float token_max = 0.f;
  if (kPerToken) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int c = 8 * (i * blockDim.x + t);
      if (c < H) {
        Bf16x8 w;
        w.u = *reinterpret_cast<const uint4*>(weight + c);
#pragma unroll
        for (int j = 0; j < 8; ++j) token_max = max_nan(token_max, fabsf(__bfloat162float(v[i].h[j]) * rstd * __bfloat162float(w.h[j])));
      }
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) token_max = max_nan(token_max, __shfl_xor_sync(0xffffffffu, token_max, m));
    if (lane == 0) red[1][warp] = token_max;
    __syncthreads();
    token_max = lane < warps ? red[1][lane] : 0.f;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) token_max = max_nan(token_max, __shfl_xor_sync(0xffffffffu, token_max, m));
  }

#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int c = 8 * (i * blockDim.x + t);
    float y[8];
    float amax = 0.f;
    if (c < H) {
      Bf16x8 w;
      w.u = *reinterpret_cast<const uint4*>(weight + c);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = __bfloat162float(v[i].h[j]) * rstd * __bfloat162float(w.h[j]);
        amax = max_nan(amax, fabsf(y[j]));
      }
    }
    if (kPerToken) {
      amax = token_max;
    } else {
#pragma unroll
      for (int m = 8; m > 0; m >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, m));
    }
    if (c < H) {
      const float scale = max_nan(amax, kScaleFloor) / kFp8Max;
      const float inv = 1.f / scale;
      if (kPerToken) {
        if (t == 0 && i == 0) scales[blockIdx.x] = scale;
      } else if ((lane & 15) == 0) {
        scales[static_cast<size_t>(blockIdx.x) * (H >> 7) + (c >> 7)] = scale;
      }
      *reinterpret_cast<uint2*>(q + off + c) =
          make_uint2(e4m3x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv), e4m3x4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv));
      if (normed != nullptr) {
        Bf16x8 o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o.h[j] = __float2bfloat16_rn(y[j]);
        *reinterpret_cast<uint4*>(normed + off + c) = o.u;
      }
    }
  }
}

template <int kVecs>
cudaError_t launch_vecs(uint8_t* q, float* scales, __nv_bfloat16* normed, __nv_bfloat16* residual_out,
                        const __nv_bfloat16* residual, const __nv_bfloat16* input, const __nv_bfloat16* weight, float eps,
                        int T, int H, bool per_token, int threads, cudaStream_t stream) {
  auto kernel = residual != nullptr ? (per_token ? rms_norm_quant_fp8_kernel<kVecs, true, true> : rms_norm_quant_fp8_kernel<kVecs, true, false>)
                                    : (per_token ? rms_norm_quant_fp8_kernel<kVecs, false, true> : rms_norm_quant_fp8_kernel<kVecs, false, false>);
  return launch_pdl(kernel, dim3(T), dim3(threads), 0, stream, q, scales, normed, residual_out, residual, input, weight, eps, H);
}

}  // namespace

int launch_rms_norm_quant_fp8(uint8_t* q, float* scales, __nv_bfloat16* normed, __nv_bfloat16* residual_out,
                              const __nv_bfloat16* residual, const __nv_bfloat16* input, const __nv_bfloat16* weight,
                              float eps, int T, int H, bool per_token, cudaStream_t stream) {
  if (T == 0) return kStatusOk;
  const int vecs = H / 8;
  // Two vectors a thread up to 768 threads, then four, which leave the SM two tokens more at a time (H = 12288, T = 4096:
  // 78 us with two, 99 with four; H = 16384, T = 2048: 68 with two, 60 with four).
  const int per_thread = vecs <= 1536 ? 2 : 4;
  const int threads = ((vecs + per_thread - 1) / per_thread + 31) / 32 * 32;
  const cudaError_t e = per_thread == 2
                            ? launch_vecs<2>(q, scales, normed, residual_out, residual, input, weight, eps, T, H, per_token, threads, stream)
                            : launch_vecs<4>(q, scales, normed, residual_out, residual, input, weight, eps, T, H, per_token, threads, stream);
  if (int st = check_cuda(e, "rms_norm_quant_fp8 launch")) return st;
  count_launches(1);
  return check_launch("rms_norm_quant_fp8");
}

}  // namespace moe_b200
