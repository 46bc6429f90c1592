// Products with 4-bit weights and group scales, for few tokens: dense (w4_linear) and over the routed experts.
//   W[n, k] = (code[n, k] - zero[n, k / g]) * scale[n, k / g]     codes two a byte, low nibble first; zero = 8 if not given
//   dense    y[m, n] = bf16(sum_k W[n, k] x[m, k] + bias[n])
//   experts  h = act(W13_e x_t + b13_e);  out[t] = bf16(sum_j w_tj (W2_e h_tj + b2_e)),  e = topk_ids[t, j]
// Sums are fp32; the intermediate h and the slots' results stay fp32 until the one rounding of the output.
#include "launch.cuh"
#include "moe_b200_internal.cuh"
#include "ptx.cuh"

namespace moe_b200 {

namespace {

// sum_k W[n, k] x[k] over a warp; every lane takes 32 consecutive k (one 16-byte load, inside one group) at a time.
template <typename X>
__device__ __forceinline__ float w4_dot(const uint8_t* w, const __nv_bfloat16* scale, const uint8_t* zero, const X* x, int K,
                                        int group, int lane) {
  float total = 0.f;
  for (int k0 = lane * 32; k0 < K; k0 += 1024) {
    const uint4 raw = *reinterpret_cast<const uint4*>(w + k0 / 2);
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
    const int gi = k0 / group;
    const float z = zero != nullptr ? static_cast<float>(zero[gi] & 15) : 8.f;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      s = fmaf(static_cast<float>((words[i / 8] >> (4 * (i % 8))) & 15u) - z, static_cast<float>(x[k0 + i]), s);
    total = fmaf(s, __bfloat162float(scale[gi]), total);
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) total += __shfl_xor_sync(0xffffffffu, total, m);
  return total;
}

__global__ void __launch_bounds__(256)
w4_linear_kernel(__nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ x, long long x_ld, W4Matrix w, int M, int N, int K) {
  grid_dependency_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= N) return;
  const size_t g0 = static_cast<size_t>(n) * (K / w.group);
  for (int m = 0; m < M; ++m) {
    const float y = w4_dot(w.q + static_cast<size_t>(n) * (K / 2), w.scale + g0, w.zero != nullptr ? w.zero + g0 : nullptr, x + m * x_ld, K, w.group, lane);
    if (lane == 0) out[static_cast<size_t>(m) * N + n] = __float2bfloat16_rn(y + (w.bias != nullptr ? __bfloat162float(w.bias[n]) : 0.f));
  }
}

__device__ __forceinline__ float w4_act(float gate, float up, int activation) {
  if (activation == 0) return gate / (1.f + expf(-gate)) * up;
  const float g = fminf(gate, 7.f), u = fminf(fmaxf(up, -7.f), 7.f);
  return g / (1.f + expf(-1.702f * g)) * (u + 1.f);
}

__global__ void __launch_bounds__(256)
w4_gate_up_kernel(float* __restrict__ h, const __nv_bfloat16* __restrict__ x, const int* __restrict__ ids, W4Matrix w, int E,
                  int k, int H, int I, int activation) {
  grid_dependency_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int j = blockIdx.x * 8 + (threadIdx.x >> 5), slot = blockIdx.y;
  const int e = ids[slot];
  if (j >= I || e < 0 || e >= E) return;
  const int row[2] = {activation == 0 ? j : 2 * j, activation == 0 ? I + j : 2 * j + 1};
  float y[2];
  for (int i = 0; i < 2; ++i) {
    const size_t r = static_cast<size_t>(e) * 2 * I + row[i], g0 = r * (H / w.group);
    y[i] = w4_dot(w.q + r * (H / 2), w.scale + g0, w.zero != nullptr ? w.zero + g0 : nullptr, x + static_cast<size_t>(slot / k) * H, H, w.group, lane);
    if (w.bias != nullptr) y[i] += __bfloat162float(w.bias[r]);
  }
  if (lane == 0) h[static_cast<size_t>(slot) * I + j] = w4_act(y[0], y[1], activation);
}

__global__ void __launch_bounds__(256)
w4_down_kernel(__nv_bfloat16* __restrict__ out, const float* __restrict__ h, const float* __restrict__ tw, const int* __restrict__ ids,
               W4Matrix w, int E, int k, int H, int I) {
  grid_dependency_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5), t = blockIdx.y;
  if (n >= H) return;
  float sum = 0.f;
  for (int j = 0; j < k; ++j) {
    const size_t slot = static_cast<size_t>(t) * k + j;
    const int e = ids[slot];
    if (e < 0 || e >= E) continue;
    const size_t r = static_cast<size_t>(e) * H + n, g0 = r * (I / w.group);
    float y = w4_dot(w.q + r * (I / 2), w.scale + g0, w.zero != nullptr ? w.zero + g0 : nullptr, h + slot * I, I, w.group, lane);
    if (w.bias != nullptr) y += __bfloat162float(w.bias[r]);
    sum = fmaf(tw[slot], y, sum);
  }
  if (lane == 0) out[static_cast<size_t>(t) * H + n] = __float2bfloat16_rn(sum);
}

}  // namespace

int launch_w4_linear(__nv_bfloat16* out, const __nv_bfloat16* x, long long x_ld, const W4Matrix& w, int M, int N, int K, cudaStream_t stream) {
  if (M == 0) return kStatusOk;
  if (int st = check_cuda(launch_pdl(w4_linear_kernel, dim3((N + 7) / 8), dim3(256), 0, stream, out, x, x_ld, w, M, N, K), "w4_linear launch")) return st;
  count_launches(1);
  return check_launch("w4_linear");
}

size_t w4_experts_workspace_bytes(int T, int top_k, int H, int I) {
  (void)H;
  return static_cast<size_t>(T > 0 ? T : 1) * top_k * I * sizeof(float);
}

int launch_w4_experts(__nv_bfloat16* out, const __nv_bfloat16* x, const W4Matrix& w13, const W4Matrix& w2, const float* topk_w,
                      const int* topk_ids, int T, int E, int top_k, int H, int I, int activation, void* workspace,
                      cudaStream_t stream) {
  float* h = static_cast<float*>(workspace);
  if (int st = check_cuda(launch_pdl(w4_gate_up_kernel, dim3((I + 7) / 8, T * top_k), dim3(256), 0, stream, h, x, topk_ids, w13, E, top_k, H, I, activation), "w4 gate_up launch")) return st;
  if (int st = check_cuda(launch_pdl(w4_down_kernel, dim3((H + 7) / 8, T), dim3(256), 0, stream, out, h, topk_w, topk_ids, w2, E, top_k, H, I), "w4 down launch")) return st;
  count_launches(2);
  return check_launch("w4_experts");
}

}  // namespace moe_b200
