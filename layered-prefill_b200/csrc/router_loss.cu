// The router's training side: balance loss, z loss and per-expert counts from the logits and the chosen experts, and the
// gradient of these losses and of the routed weights with respect to the logits.
//   counted tokens: those whose mask byte is non-zero (all without a mask); n = their number (1 in the divisions if none)
//   p_t = softmax(l_t), lse_t = log sum exp(l_t), c_e = number of (t, j) with topk_ids[t, j] == e, P_e = sum_t p_te / n
//   balance = E * sum_e (c_e / n) * P_e            z = sum_t lse_t^2 / n
// Gradient, with g_b, g_z and dw the gradients of balance, z and of the routed weights w_j = p_{id_j} / S
// (S = sum of the picked p when renormalised, else 1), c being constant:
//   u_e  = g_b * E * c_e / n^2 + sum_{j: id_j = e} du_j,  du_j = (dw_j - sum_i dw_i w_i) / S  (dw_j without the renormalisation)
//   dl_e = p_e * (u_e - sum_i p_i u_i + g_z * 2 * lse / n)
// Both passes read the logits once and recompute the softmax in registers (one warp a token): writing p and reading it
// back would cost more than the exponentials. Sums over the tokens are fp32 over at most a few hundred terms a
// warp, then fixed-order sums over warps and CTAs (double in the last step), so that two runs give the same bits; counts are integers.
#include "launch.cuh"
#include "moe_b200_internal.cuh"

namespace moe_b200 {

namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxBlocks = 128;  // CTAs of the first pass = rows of the second pass's sum
constexpr float kLog2e = 1.4426950408889634f;

template <bool kBf16>
__device__ __forceinline__ float load_logit(const void* p, size_t i) {
  if constexpr (kBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  else return static_cast<const float*>(p)[i];
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// The lane's probabilities (experts lane, lane + 32, ...; 0 past E) and the row's lse.
template <int kVpl, bool kBf16>
__device__ __forceinline__ void softmax_row(const void* logits, size_t off, int E, int lane, float (&p)[kVpl], float& lse, float& row_max, float& inv_sum) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kVpl; ++i) {
    const int e = lane + 32 * i;
    p[i] = e < E ? load_logit<kBf16>(logits, off + e) : -INFINITY;
    m = (p[i] > m || p[i] != p[i]) ? p[i] : m;  // a NaN logit reaches the sum below in any case
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kVpl; ++i) {
    p[i] = lane + 32 * i < E ? exp2f((p[i] - m) * kLog2e) : 0.f;
    sum += p[i];
  }
  sum = warp_sum(sum);
  inv_sum = 1.f / sum;
#pragma unroll
  for (int i = 0; i < kVpl; ++i) p[i] *= inv_sum;
  row_max = m;
  lse = m + logf(sum);
}

struct LossOut {
  float* losses;
  int* counts;
  int* num_tokens;
  float* mean_probs;
};

// Workspace of the first pass: sums of p [blocks][E], counts [blocks][E], then z sums and token counts [blocks].
struct LossParts {
  float* p;
  int* c;
  float* z;
  int* n;
};

// Called by a whole CTA: the sums over `blocks` rows of parts, and the outputs.
__device__ void finish_losses(const LossParts& w, int blocks, int E, const LossOut& out) {
  __shared__ double red[32];
  __shared__ int s_n;
  __shared__ double s_z;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  if (warp == 0) {
    int n = 0;
    double z = 0;
    for (int b = lane; b < blocks; b += 32) {
      n += w.n[b];
      z += w.z[b];
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
      n += __shfl_xor_sync(0xffffffffu, n, m);
      z += __shfl_xor_sync(0xffffffffu, z, m);
    }
    if (lane == 0) {
      s_n = n;
      s_z = z;
    }
  }
  __syncthreads();
  const int n = s_n;
  const double inv_n = 1.0 / (n > 0 ? n : 1);
  double bal = 0;
  for (int e = t; e < E; e += blockDim.x) {
    double p = 0;
    int c = 0;
    for (int b = 0; b < blocks; ++b) {
      p += w.p[static_cast<size_t>(b) * E + e];
      c += w.c[static_cast<size_t>(b) * E + e];
    }
    p *= inv_n;
    out.mean_probs[e] = static_cast<float>(p);
    out.counts[e] = c;
    bal += p * c * inv_n;
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) bal += __shfl_xor_sync(0xffffffffu, bal, m);
  if (lane == 0) red[warp] = bal;
  __syncthreads();
  if (t == 0) {
    double s = 0;
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) s += red[i];
    out.losses[0] = static_cast<float>(s * E);
    out.losses[1] = static_cast<float>(s_z * inv_n);
    *out.num_tokens = n;
  }
}

template <int kVpl, bool kBf16>
__global__ void __launch_bounds__(512)
router_loss_kernel(const void* __restrict__ logits, const int* __restrict__ ids, const uint8_t* __restrict__ mask, int T, int E,
                   int k, LossParts w) {
  extern __shared__ float smem[];  // [warps][E] sums of p, then [E] counts
  __shared__ float s_z[16];
  __shared__ int s_n[16];
  grid_dependency_launch();
  grid_dependency_wait();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
  int* s_counts = reinterpret_cast<int*>(smem + static_cast<size_t>(warps) * E);
  for (int e = t; e < E; e += blockDim.x) s_counts[e] = 0;
  __syncthreads();
  float acc[kVpl];
#pragma unroll
  for (int i = 0; i < kVpl; ++i) acc[i] = 0.f;
  float z = 0.f;
  int n = 0;
  for (int tok = blockIdx.x * warps + warp; tok < T; tok += gridDim.x * warps) {
    if (mask != nullptr && mask[tok] == 0) continue;  // the same for the whole warp
    float p[kVpl], lse, m, inv;
    softmax_row<kVpl, kBf16>(logits, static_cast<size_t>(tok) * E, E, lane, p, lse, m, inv);
#pragma unroll
    for (int i = 0; i < kVpl; ++i) acc[i] += p[i];
    z = fmaf(lse, lse, z);
    ++n;
    for (int j = lane; j < k; j += 32) {
      const int id = ids[static_cast<size_t>(tok) * k + j];
      if (id >= 0 && id < E) atomicAdd(&s_counts[id], 1);
    }
  }
#pragma unroll
  for (int i = 0; i < kVpl; ++i)
    if (lane + 32 * i < E) smem[static_cast<size_t>(warp) * E + lane + 32 * i] = acc[i];
  if (lane == 0) {
    s_z[warp] = z;
    s_n[warp] = n;
  }
  __syncthreads();
  for (int e = t; e < E; e += blockDim.x) {
    float s = 0.f;
    for (int i = 0; i < warps; ++i) s += smem[static_cast<size_t>(i) * E + e];
    w.p[static_cast<size_t>(blockIdx.x) * E + e] = s;
    w.c[static_cast<size_t>(blockIdx.x) * E + e] = s_counts[e];
  }
  if (t == 0) {
    float zs = 0.f;
    int ns = 0;
    for (int i = 0; i < warps; ++i) {
      zs += s_z[i];
      ns += s_n[i];
    }
    w.z[blockIdx.x] = zs;
    w.n[blockIdx.x] = ns;
  }
}

__global__ void __launch_bounds__(1024) router_loss_finish_kernel(LossParts w, int blocks, int E, LossOut out) {
  grid_dependency_launch();
  grid_dependency_wait();
  finish_losses(w, blocks, E, out);
}

template <int kVpl, bool kBf16>
__global__ void __launch_bounds__(256)
router_backward_kernel(void* __restrict__ grad, const void* __restrict__ logits, const int* __restrict__ ids,
                       const int* __restrict__ counts, const int* __restrict__ num_tokens,
                       const float* __restrict__ grad_losses, const float* __restrict__ grad_w,
                       const uint8_t* __restrict__ mask, int T, int E, int k, int renormalize) {
  grid_dependency_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int tok = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (tok >= T) return;
  const size_t off = static_cast<size_t>(tok) * E;
  float g[kVpl];
  if (mask != nullptr && mask[tok] == 0) {
#pragma unroll
    for (int i = 0; i < kVpl; ++i) g[i] = 0.f;
  } else {
    float p[kVpl], lse, m, inv;
    softmax_row<kVpl, kBf16>(logits, off, E, lane, p, lse, m, inv);
    float u[kVpl];
    float g_z = 0.f;
#pragma unroll
    for (int i = 0; i < kVpl; ++i) u[i] = 0.f;
    if (grad_losses != nullptr) {
      const float n = static_cast<float>(max(*num_tokens, 1));
      const float coef = grad_losses[0] * E / n / n;
      g_z = grad_losses[1] * 2.f * lse / n;
#pragma unroll
      for (int i = 0; i < kVpl; ++i)
        if (lane + 32 * i < E) u[i] = coef * static_cast<float>(counts[lane + 32 * i]);
    }
    if (grad_w != nullptr) {
      // lane j holds slots j, j + 32, ...; S and the weighted sum first, then every slot's term goes to its expert's lane
      float s = 0.f, gs = 0.f;
      for (int j = lane; j < k; j += 32) {
        const int id = ids[static_cast<size_t>(tok) * k + j];
        if (id >= 0 && id < E) {
          const float pj = exp2f((load_logit<kBf16>(logits, off + id) - m) * kLog2e) * inv;
          s += pj;
          gs += pj * grad_w[static_cast<size_t>(tok) * k + j];
        }
      }
      s = warp_sum(s);
      gs = warp_sum(gs);
      const float inv_s = renormalize ? 1.f / s : 1.f;
      const float mean = renormalize ? gs * inv_s : 0.f;
      for (int j = 0; j < k; ++j) {
        const int id = ids[static_cast<size_t>(tok) * k + j];
        const float du = (grad_w[static_cast<size_t>(tok) * k + j] - mean) * inv_s;
#pragma unroll
        for (int i = 0; i < kVpl; ++i)
          if (id == lane + 32 * i) u[i] += du;
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < kVpl; ++i) dot = fmaf(p[i], u[i], dot);
    dot = warp_sum(dot);
#pragma unroll
    for (int i = 0; i < kVpl; ++i) g[i] = p[i] * (u[i] - dot + g_z);
  }
#pragma unroll
  for (int i = 0; i < kVpl; ++i) {
    const int e = lane + 32 * i;
    if (e < E) {
      if constexpr (kBf16) static_cast<__nv_bfloat16*>(grad)[off + e] = __float2bfloat16_rn(g[i]);
      else static_cast<float*>(grad)[off + e] = g[i];
    }
  }
}

int loss_blocks(int T, int warps) {
  const int want = (T + warps - 1) / warps;
  return want < 1 ? 1 : (want > kMaxBlocks ? kMaxBlocks : want);
}

constexpr int kLossWarps = 16;

// Calls f(integral_constant<kVpl>) with the smallest supported number of experts a lane.
template <typename F>
auto with_vpl(int E, F&& f) {
  const int need = (E + 31) / 32;
  if (need <= 1) return f(std::integral_constant<int, 1>{});
  if (need <= 2) return f(std::integral_constant<int, 2>{});
  if (need <= 4) return f(std::integral_constant<int, 4>{});
  if (need <= 8) return f(std::integral_constant<int, 8>{});
  if (need <= 16) return f(std::integral_constant<int, 16>{});
  return f(std::integral_constant<int, 32>{});
}

int check_router(const char* what, int T, int E, int k) {
  if (T < 0 || E <= 0 || k <= 0 || k > E) return set_error(kStatusInvalidArgument, "%s: need T >= 0 and 0 < k <= E (T=%d E=%d k=%d)", what, T, E, k);
  if (E > kMaxExperts) return set_error(kStatusInvalidArgument, "%s: more than %d experts", what, kMaxExperts);
  if (static_cast<long long>(T) * k > 0x7fffffffll) return set_error(kStatusInvalidArgument, "%s: T * k does not fit the int32 counts", what);
  return kStatusOk;
}

}  // namespace

size_t router_loss_workspace_bytes(int T, int E) {
  const size_t b = loss_blocks(T, kLossWarps);
  return b * E * 8 + b * 8;
}

int launch_router_loss(float* losses, int* counts, int* num_tokens, float* mean_probs, const void* gating, int gating_is_bf16,
                       const int* topk_ids, const uint8_t* token_mask, int T, int E, int k, void* workspace,
                       size_t workspace_bytes, cudaStream_t stream) {
  if (int st = check_router("router_loss", T, E, k)) return st;
  const size_t need = router_loss_workspace_bytes(T, E);
  if (workspace == nullptr || workspace_bytes < need)
    return set_error(kStatusWorkspaceTooSmall, "router_loss: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  const int blocks = loss_blocks(T, kLossWarps);
  LossParts w;
  w.p = static_cast<float*>(workspace);
  w.c = reinterpret_cast<int*>(w.p + static_cast<size_t>(blocks) * E);
  w.z = reinterpret_cast<float*>(w.c + static_cast<size_t>(blocks) * E);
  w.n = reinterpret_cast<int*>(w.z + blocks);
  const size_t smem = (static_cast<size_t>(kLossWarps) + 1) * E * sizeof(float);
  const cudaError_t e = with_vpl(E, [&](auto vpl) {
    constexpr int V = decltype(vpl)::value;
    auto kernel = gating_is_bf16 ? router_loss_kernel<V, true> : router_loss_kernel<V, false>;
    if (smem > 48 * 1024) {
      const cudaError_t a = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (a != cudaSuccess) return a;
    }
    return launch_pdl(kernel, dim3(blocks), dim3(kLossWarps * 32), smem, stream, gating, topk_ids, token_mask, T, E, k, w);
  });
  if (int st = check_cuda(e, "router_loss launch")) return st;
  LossOut out{losses, counts, num_tokens, mean_probs};
  if (int st = check_cuda(launch_pdl(router_loss_finish_kernel, dim3(1), dim3(1024), 0, stream, w, blocks, E, out), "router_loss finish launch")) return st;
  count_launches(2);
  return check_launch("router_loss");
}

int launch_router_backward(void* grad_logits, const void* gating, int gating_is_bf16, const int* topk_ids, const int* counts,
                           const int* num_tokens, const float* grad_losses, const float* grad_topk_weights,
                           const uint8_t* token_mask, int T, int E, int k, int renormalize, cudaStream_t stream) {
  if (int st = check_router("router_backward", T, E, k)) return st;
  if (T == 0) return kStatusOk;
  const cudaError_t e = with_vpl(E, [&](auto vpl) {
    constexpr int V = decltype(vpl)::value;
    auto kernel = gating_is_bf16 ? router_backward_kernel<V, true> : router_backward_kernel<V, false>;
    return launch_pdl(kernel, dim3((T + 7) / 8), dim3(256), 0, stream, grad_logits, gating, topk_ids, counts, num_tokens,
                      grad_losses, grad_topk_weights, token_mask, T, E, k, renormalize);
  });
  if (int st = check_cuda(e, "router_backward launch")) return st;
  count_launches(1);
  return check_launch("router_backward");
}

}  // namespace moe_b200
