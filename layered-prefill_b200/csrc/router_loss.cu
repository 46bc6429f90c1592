// The router's training side: balance loss, z loss and per-expert counts from the logits and the chosen experts, and the
// gradient of these losses and of the routed weights with respect to the logits.
//   counted tokens: those whose mask byte is non-zero (all without a mask); n = their number (1 in the divisions if none)
//   p_t = softmax(l_t), lse_t = log sum exp(l_t), c_e = number of (t, j) with topk_ids[t, j] == e, P_e = sum_t p_te / n
//   balance = E * sum_e (c_e / n) * P_e            z = sum_t lse_t^2 / n
// Gradient, with g_b, g_z and dw the gradients of balance, z and of the routed weights w_j = p_{id_j} / S
// (S = sum of the picked p when renormalised, else 1), c being constant:
//   u_e  = g_b * E * c_e / n^2 + sum_{j: id_j = e} du_j,  du_j = (dw_j - sum_i dw_i w_i) / S  (dw_j without the renormalisation)
//   dl_e = p_e * (u_e - sum_i p_i u_i + g_z * 2 * lse / n)
// Both passes read the logits once and recompute the softmax in registers: writing p and reading it back would cost
// more than the exponentials. Eight lanes take a token of up to 256 experts (32 lanes one of more), so that a warp works on four
// at once and a reduction costs three shuffles for all of them (with a warp a token the reductions were most of the work). Sums over the
// tokens are fp32 over short runs of a lane group (loss_run), then over its runs and over warps, then over CTAs (double), all in
// fixed orders, so that two runs give the same bits; counts are integers. Bound: HBM (logits in, gradient out) for large batches,
// launches for small ones: one CTA does the whole first pass of a small batch.
#include <type_traits>

#include "launch.cuh"
#include "moe_b200_internal.cuh"
#include "ptx.cuh"

namespace moe_b200 {

namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxBlocks = 296;  // CTAs of the first pass = rows of the second pass's sum
constexpr int kLossWarps = 16;
// Tokens, and logits, that one CTA of kOneWarps warps takes alone, without the second pass: both passes of 128 tokens with 128
// experts 8.9 us, against 9.4 with a second pass; with 384 experts 13.2 against 10.0.
constexpr int kOneCta = 128, kOneCtaLogits = 16384;
constexpr int kOneWarps = 32;
constexpr float kLog2e = 1.4426950408889634f;

// kL lanes a token, kN experts a lane in vectors of kW neighbours: vector v of lane l (of the kL) starts at expert (v * kL + l) * kW.
template <int kL, int kW>
__device__ __forceinline__ int expert_of(int i, int l) { return ((i / kW) * kL + l) * kW + i % kW; }

template <bool kBf16, int kL, int kW, int kN>
__device__ __forceinline__ void load_row(const void* logits, size_t off, int E, int l, float (&x)[kN]) {
#pragma unroll
  for (int v = 0; v < kN / kW; ++v) {
    const int e = (v * kL + l) * kW;
    if constexpr (kW == 4) {
      if (e < E) {
        if constexpr (kBf16) {
          const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(logits) + off + e);
          x[4 * v] = __uint_as_float(r.x << 16);
          x[4 * v + 1] = __uint_as_float(r.x & 0xffff0000u);
          x[4 * v + 2] = __uint_as_float(r.y << 16);
          x[4 * v + 3] = __uint_as_float(r.y & 0xffff0000u);
        } else {
          const float4 r = *reinterpret_cast<const float4*>(static_cast<const float*>(logits) + off + e);
          x[4 * v] = r.x; x[4 * v + 1] = r.y; x[4 * v + 2] = r.z; x[4 * v + 3] = r.w;
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) x[4 * v + q] = -INFINITY;
      }
    } else {
      if constexpr (kBf16) x[v] = e < E ? __bfloat162float(static_cast<const __nv_bfloat16*>(logits)[off + e]) : -INFINITY;
      else x[v] = e < E ? static_cast<const float*>(logits)[off + e] : -INFINITY;
    }
  }
}

template <int kL>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int m = kL / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

__device__ __forceinline__ float exp2_ftz(float x) {  // 2 ulp; what is below 2^-126 of the largest counts as nothing
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// x: logits in, exp(x - max) out (0 past E: those logits are -inf). A NaN reaches the sum whatever the maximum makes of it.
template <int kL, int kN>
__device__ __forceinline__ void exp_row(float (&x)[kN], float& row_max, float& sum) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i < kN; ++i) m = fmaxf(m, x[i]);
#pragma unroll
  for (int s = kL / 2; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    x[i] = exp2_ftz((x[i] - m) * kLog2e);
    sum += x[i];
  }
  row_max = m;
}

// The lane's experts in a row of shared memory (on 16 bytes for vectors of four).
template <int kL, int kW, int kN>
__device__ __forceinline__ void put_row(float* row, int E, int l, const float (&x)[kN]) {
#pragma unroll
  for (int v = 0; v < kN / kW; ++v) {
    const int e = (v * kL + l) * kW;
    if (e >= E) continue;
    if constexpr (kW == 4) *reinterpret_cast<float4*>(row + e) = make_float4(x[4 * v], x[4 * v + 1], x[4 * v + 2], x[4 * v + 3]);
    else row[e] = x[v];
  }
}
template <int kL, int kW, int kN>
__device__ __forceinline__ void get_row(const float* row, int E, int l, float (&x)[kN]) {  // 0 past E
#pragma unroll
  for (int v = 0; v < kN / kW; ++v) {
    const int e = (v * kL + l) * kW;
    if constexpr (kW == 4) {
      const float4 q = e < E ? *reinterpret_cast<const float4*>(row + e) : make_float4(0.f, 0.f, 0.f, 0.f);
      x[4 * v] = q.x; x[4 * v + 1] = q.y; x[4 * v + 2] = q.z; x[4 * v + 3] = q.w;
    } else {
      x[v] = e < E ? row[e] : 0.f;
    }
  }
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

constexpr int kFinishCtas = 8;

struct FinishShared {
  double red[32], s_p[1024], s_bal[kFinishCtas], s_z;
  int s_c[1024], s_n;
};

// The sums over `blocks` rows of parts, and the outputs. Called by all threads of a CTA (rank 0 of 1) or of a cluster of
// kFinishCtas, whose CTAs take E / ranks experts each; several threads share an expert's rows. Fixed orders throughout.
template <int kRanks>
__device__ void finish_losses(const LossParts& w, int blocks, int E, const LossOut& out, int rank) {
  __shared__ FinishShared sh;
  auto& [red, s_p, s_bal, s_z, s_c, s_n] = sh;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int per = (E + kRanks - 1) / kRanks, e0 = rank * per, mine = max(0, min(per, E - e0));
  const int parts = static_cast<int>(blockDim.x) / per;  // blockDim.x >= per
  if (t < parts * mine) {
    const int x = t % mine, part = t / mine;
    double p = 0;
    int c = 0;
#pragma unroll 8
    for (int b = part; b < blocks; b += parts) {
      p += w.p[static_cast<size_t>(b) * E + e0 + x];
      c += w.c[static_cast<size_t>(b) * E + e0 + x];
    }
    s_p[t] = p;
    s_c[t] = c;
  }
  if (warp == static_cast<int>(blockDim.x >> 5) - 1) {
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
  if (t < mine) {
    double p = 0;
    int c = 0;
    for (int i = 0; i < parts; ++i) {
      p += s_p[i * mine + t];
      c += s_c[i * mine + t];
    }
    p *= inv_n;
    out.mean_probs[e0 + t] = static_cast<float>(p);
    out.counts[e0 + t] = c;
    bal = p * c * inv_n;
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) bal += __shfl_xor_sync(0xffffffffu, bal, m);
  if (lane == 0) red[warp] = bal;
  __syncthreads();
  if (t == 0) {
    bal = 0;
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) bal += red[i];
    if (kRanks > 1) st_cluster_f64(&s_bal[rank], 0, bal);
  }
  if (kRanks > 1) cluster_sync_all();
  if (rank == 0 && t == 0) {
    if (kRanks > 1) {
      bal = 0;
      for (int i = 0; i < kRanks; ++i) bal += s_bal[i];
    }
    out.losses[0] = static_cast<float>(bal * E);
    out.losses[1] = static_cast<float>(s_z * inv_n);
    *out.num_tokens = n;
  }
}

template <bool kBf16, int kL, int kW, int kN>
__global__ void __launch_bounds__(kOneWarps * 32)
router_loss_kernel(const void* __restrict__ logits, const int* __restrict__ ids, const uint8_t* __restrict__ mask, int T, int E,
                   int k, int run, int alone, LossParts w, LossOut out) {
  extern __shared__ float smem[];  // [warps][E] sums of p, then [E] counts
  __shared__ float s_z[kOneWarps];
  __shared__ int s_n[kOneWarps];
  grid_dependency_wait();
  grid_dependency_launch();
  constexpr int kTokens = 32 / kL;  // of a warp at a time
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
  const int l = lane % kL;
  int* s_counts = reinterpret_cast<int*>(smem + static_cast<size_t>(warps) * E);
  for (int e = t; e < E; e += blockDim.x) s_counts[e] = 0;
  __syncthreads();
  float z_all = 0.f;
  int n = 0;
  const int stride = gridDim.x * warps * kTokens;
  int tok0 = (blockIdx.x * warps + warp) * kTokens;
  bool first = true;
  do {  // `run` tokens a lane group, then its sums join the warp's
    float acc[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) acc[i] = 0.f;
    float z = 0.f;
    for (int turn = 0; turn < run && tok0 < T; ++turn, tok0 += stride) {
      const int tok = tok0 + lane / kL;
      const bool live = tok < T && (mask == nullptr || mask[tok] != 0);
      float x[kN];
#pragma unroll
      for (int i = 0; i < kN; ++i) x[i] = 0.f;
      if (live) {
        load_row<kBf16, kL, kW>(logits, static_cast<size_t>(tok) * E, E, l, x);
        for (int j = l; j < k; j += kL) {
          const int id = ids[static_cast<size_t>(tok) * k + j];
          if (id >= 0 && id < E) atomicAdd(&s_counts[id], 1);
        }
      }
      float m, sum;
      exp_row<kL>(x, m, sum);
      sum = lanes_sum<kL>(sum);
      if (live) {
        const float inv = 1.f / sum, lse = m + logf(sum);
#pragma unroll
        for (int i = 0; i < kN; ++i) acc[i] = fmaf(x[i], inv, acc[i]);
        z = fmaf(lse, lse, z);
        ++n;
      }
    }
#pragma unroll
    for (int s = 16; s >= kL; s >>= 1) {  // the tokens of the warp
#pragma unroll
      for (int i = 0; i < kN; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], s);
      z += __shfl_xor_sync(0xffffffffu, z, s);
    }
    z_all += z;
    if (lane < kL) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int e = expert_of<kL, kW>(i, l);
        if (e >= E) continue;
        float& row = smem[static_cast<size_t>(warp) * E + e];
        row = first ? acc[i] : row + acc[i];
      }
    }
    first = false;
  } while (tok0 < T);
#pragma unroll
  for (int s = 16; s >= kL; s >>= 1) n += __shfl_xor_sync(0xffffffffu, n, s);
  if (lane == 0) {
    s_z[warp] = z_all;
    s_n[warp] = n;
  }
  __syncthreads();
  if (alone) w = LossParts{smem, s_counts, s_z, s_n};  // a CTA alone keeps its parts
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
  if (alone) {
    __syncthreads();
    finish_losses<1>(w, 1, E, out, 0);
  }
}

__global__ void __launch_bounds__(1024) router_loss_finish_kernel(LossParts w, int blocks, int E, LossOut out) {
  cluster_sync_all();  // every CTA has started: its shared memory may be written from now on
  grid_dependency_wait();
  grid_dependency_launch();
  finish_losses<kFinishCtas>(w, blocks, E, out, static_cast<int>(cluster_ctarank()));
}

// Every warp takes tokens a grid apart, the next ones' logits on their way meanwhile. The gradient of the losses is formed in
// registers; that of the routed weights touches k of the E experts, and is added in a row of shared memory through
// which the row leaves for the registers that store it.
template <bool kBf16, int kL, int kW, int kN>
__global__ void __launch_bounds__(256)
router_backward_kernel(void* __restrict__ grad, const void* __restrict__ logits, const int* __restrict__ ids,
                       const int* __restrict__ counts, const int* __restrict__ num_tokens,
                       const float* __restrict__ grad_losses, const float* __restrict__ grad_w,
                       const uint8_t* __restrict__ mask, int T, int E, int k, int renormalize) {
  extern __shared__ __align__(16) float smem[];  // [E] g_b * E * c_e / n^2, then a row a token
  grid_dependency_wait();
  grid_dependency_launch();
  constexpr int kTokens = 32 / kL;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane % kL, group = lane / kL;
  const int E4 = (E + 3) & ~3;
  const float* s_base = smem;
  float* row = smem + E4 + static_cast<size_t>(warp * kTokens + group) * E4;
  float g_z = 0.f;  // g_z * 2 / n (times lse)
  float g_b = 0.f;
  if (grad_losses != nullptr) {
    const float n = static_cast<float>(max(*num_tokens, 1));
    g_b = grad_losses[0] * E / n / n;
    g_z = grad_losses[1] * 2.f / n;
  }
  for (int e = threadIdx.x; e < E; e += blockDim.x) smem[e] = grad_losses != nullptr ? g_b * static_cast<float>(counts[e]) : 0.f;
  __syncthreads();
  const int stride = gridDim.x * (blockDim.x >> 5) * kTokens;
  float next[kN];
  bool next_live = false;
  int next_id = -1;  // of slot l
  float next_gw = 0.f;
  auto fetch = [&](int at) {
    next_live = at < T && (mask == nullptr || mask[at] != 0);
    next_id = -1;
    next_gw = 0.f;
#pragma unroll
    for (int i = 0; i < kN; ++i) next[i] = 0.f;
    if (next_live) {
      load_row<kBf16, kL, kW>(logits, static_cast<size_t>(at) * E, E, l, next);
      if (grad_w != nullptr && l < k) {
        next_id = ids[static_cast<size_t>(at) * k + l];
        next_gw = grad_w[static_cast<size_t>(at) * k + l];
      }
    }
  };
  int tok0 = (blockIdx.x * (blockDim.x >> 5) + warp) * kTokens;
  if (tok0 >= T) return;
  fetch(tok0 + group);
  for (; tok0 < T; tok0 += stride) {
    const int tok = tok0 + group;
    float x[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) x[i] = next[i];
    const bool live = next_live;
    int id = next_id;
    float gw = next_gw;
    fetch(tok + stride);
    float m, sum, dot = 0.f, u[kN];
    exp_row<kL>(x, m, sum);
    get_row<kL, kW>(s_base, E, l, u);
#pragma unroll
    for (int i = 0; i < kN; ++i) dot = fmaf(x[i], u[i], dot);
    sum = lanes_sum<kL>(sum);
    dot = lanes_sum<kL>(dot);
    const float inv = 1.f / sum;
    float add = g_z * (m + logf(sum)) - dot * inv;
    if (grad_w == nullptr) {
#pragma unroll
      for (int i = 0; i < kN; ++i) x[i] = x[i] * inv * (u[i] + add);
    } else {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kN; ++i) x[i] *= inv;
      put_row<kL, kW>(row, E, l, x);
      __syncwarp();
      // p of the picked experts, their sum and its product with the gradients; slots past the lanes in further turns
      float s = 0.f, gs = 0.f;
      if (id >= 0 && id < E) {
        s = row[id];
        gs = s * gw;
      }
      if (live) {
        for (int j = l + kL; j < k; j += kL) {
          const int o = ids[static_cast<size_t>(tok) * k + j];
          if (o >= 0 && o < E) {
            s += row[o];
            gs = fmaf(row[o], grad_w[static_cast<size_t>(tok) * k + j], gs);
          }
        }
      }
      s = lanes_sum<kL>(s);
      gs = lanes_sum<kL>(gs);
      const float inv_s = renormalize ? 1.f / s : 1.f;
      const float mean = renormalize ? gs * inv_s : 0.f;
      if (!renormalize) add -= gs;  // sum p du, which the renormalisation makes zero
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kN; ++i) u[i] += add;  // u - sum p u + g_z 2 lse / n
      put_row<kL, kW>(row, E, l, u);
      __syncwarp();
      for (int j0 = 0; j0 < k; j0 += kL) {
        if (j0 > 0) {
          const int j = j0 + l;
          const bool in = live && j < k;
          id = in ? ids[static_cast<size_t>(tok) * k + j] : -1;
          gw = in ? grad_w[static_cast<size_t>(tok) * k + j] : 0.f;
        }
        // slots of the same expert add up in slot order, by the first of them
        const bool ok = id >= 0 && id < E;
        const unsigned same = __match_any_sync(0xffffffffu, ok ? group * kMaxExperts + id : -1 - lane);
        float du = ok ? (gw - mean) * inv_s : 0.f;
        const bool lead = ok && __ffs(same) - 1 == lane;
        if (__any_sync(0xffffffffu, ok && !lead)) {
          const float own = du;
          du = 0.f;
          for (int j = 0; j < 32; ++j) {
            const float o = __shfl_sync(0xffffffffu, own, j);
            if (same >> j & 1) du += o;
          }
        }
        if (lead) row[id] += du;
        __syncwarp();
      }
      get_row<kL, kW>(row, E, l, u);
#pragma unroll
      for (int i = 0; i < kN; ++i) x[i] *= u[i];
    }
    if (tok >= T) continue;
    const size_t off = static_cast<size_t>(tok) * E;
#pragma unroll
    for (int v = 0; v < kN / kW; ++v) {
      const int e = (v * kL + l) * kW;
      if (e >= E) continue;
      if (!live) {
#pragma unroll
        for (int q = 0; q < kW; ++q) x[kW * v + q] = 0.f;
      }
      if constexpr (kW == 4) {
        if constexpr (kBf16) {
          __nv_bfloat162 a = __floats2bfloat162_rn(x[4 * v], x[4 * v + 1]), b = __floats2bfloat162_rn(x[4 * v + 2], x[4 * v + 3]);
          *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(grad) + off + e) =
              make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
        } else {
          *reinterpret_cast<float4*>(static_cast<float*>(grad) + off + e) = make_float4(x[4 * v], x[4 * v + 1], x[4 * v + 2], x[4 * v + 3]);
        }
      } else {
        if constexpr (kBf16) static_cast<__nv_bfloat16*>(grad)[off + e] = __float2bfloat16_rn(x[v]);
        else static_cast<float*>(grad)[off + e] = x[v];
      }
    }
  }
}

int lanes_of(int E) { return E <= 256 ? 8 : 32; }
bool one_cta(int T, int E) { return T <= kOneCta && T * E <= kOneCtaLogits; }
int loss_warps(int T, int E) { return one_cta(T, E) ? kOneWarps : kLossWarps; }

int loss_blocks(int T, int E) {
  if (one_cta(T, E)) return 1;
  const int per = kLossWarps * 32 / lanes_of(E), want = (T + per - 1) / per;
  return want > kMaxBlocks ? kMaxBlocks : want;
}

template <int N>
using Int = std::integral_constant<int, N>;

// Calls f(kL, kW, kN): vectors of four where they start on their own size, else single experts. Up to 256 experts in vectors, the
// usual form, a lane holds just as many vectors as E needs: what is past E would be empty work (both passes of 65519 tokens, fp32: E = 96 31.9
// us, and 36.3 in the width of 128; 192 40.7, and 56.4 in that of 256; 160 35.0, and 54.2). Elsewhere kN is the next of two to four
// widths. The first pass has 64 registers a thread, as one CTA of a small batch has 1024 threads: from 24 experts a lane on it spills, 64 to
// 240 bytes.
template <typename F>
cudaError_t with_lanes(int E, bool vectors, F&& f) {
  if (lanes_of(E) == 32) {
    if (vectors && E % 4 == 0) return E <= 512 ? f(Int<32>{}, Int<4>{}, Int<16>{}) : f(Int<32>{}, Int<4>{}, Int<32>{});
    return E <= 512 ? f(Int<32>{}, Int<1>{}, Int<16>{}) : f(Int<32>{}, Int<1>{}, Int<32>{});
  }
  if (vectors && E % 4 == 0) {
    switch ((E + 31) / 32) {
      case 1: return f(Int<8>{}, Int<4>{}, Int<4>{});
      case 2: return f(Int<8>{}, Int<4>{}, Int<8>{});
      case 3: return f(Int<8>{}, Int<4>{}, Int<12>{});
      case 4: return f(Int<8>{}, Int<4>{}, Int<16>{});
      case 5: return f(Int<8>{}, Int<4>{}, Int<20>{});
      case 6: return f(Int<8>{}, Int<4>{}, Int<24>{});
      case 7: return f(Int<8>{}, Int<4>{}, Int<28>{});
      default: return f(Int<8>{}, Int<4>{}, Int<32>{});
    }
  }
  const int n = (E + 7) / 8;
  if (n <= 2) return f(Int<8>{}, Int<1>{}, Int<2>{});
  if (n <= 8) return f(Int<8>{}, Int<1>{}, Int<8>{});
  if (n <= 16) return f(Int<8>{}, Int<1>{}, Int<16>{});
  return f(Int<8>{}, Int<1>{}, Int<32>{});
}

bool on_16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Tokens that a lane group adds up in a row before their sum joins the others', itself one addition of many: 64, or the root of
// their number where that is more, so that neither chain is longer than max(64, root) + 1 additions (up to 4096 tokens a group, that
// is 19 million tokens of many experts, a chain is off by at most 2^-17 in all; of 2^30 tokens 476 + 476 additions follow each other).
int loss_run(int T, int E, int blocks, int warps) {
  const long long at_once = static_cast<long long>(blocks) * warps * (32 / lanes_of(E)), turns = (T + at_once - 1) / at_once;
  int run = 64;
  while (static_cast<long long>(run) * run < turns) ++run;
  return run;
}

// What the kernel holds in fixed arrays counts against the 48 KB that it may have without asking, too. It asks for the most that
// any call needs, so that calls of two host threads ask for the same.
constexpr size_t kLossFixedSmem = sizeof(FinishShared) + kOneWarps * (sizeof(float) + sizeof(int));
constexpr size_t kLossMostSmem = (kOneWarps + 1) * kMaxExperts * sizeof(float);
template <typename K>
cudaError_t allow_loss_smem(K kernel, size_t dynamic) {
  if (dynamic + kLossFixedSmem <= 48 * 1024) return cudaSuccess;
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kLossMostSmem));
}

int check_router(const char* what, int T, int E, int k) {
  if (T < 0 || E <= 0 || k <= 0 || k > E) return set_error(kStatusInvalidArgument, "%s: need T >= 0 and 0 < k <= E (T=%d E=%d k=%d)", what, T, E, k);
  if (E > kMaxExperts) return set_error(kStatusInvalidArgument, "%s: more than %d experts", what, kMaxExperts);
  if (T > 1 << 30 || static_cast<long long>(T) * k > 0x7fffffffll) return set_error(kStatusInvalidArgument, "%s: T * k is too large for the int32 counts", what);
  return kStatusOk;
}

}  // namespace

size_t router_loss_workspace_bytes(int T, int E) {
  if (one_cta(T, E)) return 0;
  const size_t b = loss_blocks(T, E);
  return b * E * 8 + b * 8;
}

int launch_router_loss(float* losses, int* counts, int* num_tokens, float* mean_probs, const void* gating, int gating_is_bf16,
                       const int* topk_ids, const uint8_t* token_mask, int T, int E, int k, void* workspace,
                       size_t workspace_bytes, cudaStream_t stream) {
  if (int st = check_router("router_loss", T, E, k)) return st;
  const size_t need = router_loss_workspace_bytes(T, E);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4 != 0))
    return set_error(kStatusWorkspaceTooSmall, "router_loss: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  const int blocks = loss_blocks(T, E), warps = loss_warps(T, E);
  LossParts w;
  w.p = static_cast<float*>(workspace);
  w.c = reinterpret_cast<int*>(w.p + static_cast<size_t>(blocks) * E);
  w.z = reinterpret_cast<float*>(w.c + static_cast<size_t>(blocks) * E);
  w.n = reinterpret_cast<int*>(w.z + blocks);
  const LossOut out{losses, counts, num_tokens, mean_probs};
  const size_t smem = (static_cast<size_t>(warps) + 1) * E * sizeof(float);
  const cudaError_t e = with_lanes(E, on_16(gating), [&](auto lc, auto wc, auto nc) {
    constexpr int L = decltype(lc)::value, W = decltype(wc)::value, N = decltype(nc)::value;
    auto kernel = gating_is_bf16 ? router_loss_kernel<true, L, W, N> : router_loss_kernel<false, L, W, N>;
    const cudaError_t a = allow_loss_smem(kernel, smem);
    if (a != cudaSuccess) return a;
    return launch_pdl(kernel, dim3(blocks), dim3(warps * 32), smem, stream, gating, topk_ids, token_mask, T, E, k, loss_run(T, E, blocks, warps),
                      static_cast<int>(one_cta(T, E)), w, out);
  });
  if (int st = check_cuda(e, "router_loss launch")) return st;
  if (!one_cta(T, E)) {
    if (int st = check_cuda(launch_pdl_cluster(router_loss_finish_kernel, dim3(kFinishCtas), dim3(1024), 0, stream, kFinishCtas, w, blocks, E, out), "router_loss finish launch")) return st;
  }
  count_launches(one_cta(T, E) ? 1 : 2);
  return check_launch("router_loss");
}

int launch_router_backward(void* grad_logits, const void* gating, int gating_is_bf16, const int* topk_ids, const int* counts,
                           const int* num_tokens, const float* grad_losses, const float* grad_topk_weights,
                           const uint8_t* token_mask, int T, int E, int k, int renormalize, cudaStream_t stream) {
  if (int st = check_router("router_backward", T, E, k)) return st;
  if (T == 0) return kStatusOk;
  const int tokens = 8 * 32 / lanes_of(E);  // of a CTA at a time
  const size_t smem = (grad_topk_weights != nullptr ? tokens + 1ull : 1ull) * ((E + 3) & ~3) * sizeof(float);  // at most 36 KB, and no fixed arrays
  const cudaError_t e = with_lanes(E, on_16(gating) && on_16(grad_logits), [&](auto lc, auto wc, auto nc) {
    constexpr int L = decltype(lc)::value, W = decltype(wc)::value, N = decltype(nc)::value;
    auto kernel = gating_is_bf16 ? router_backward_kernel<true, L, W, N> : router_backward_kernel<false, L, W, N>;
    // as many CTAs as are resident, each with several tokens a lane group in turn, so that the counts are fetched once and
    // the next logits are on their way (T = 65519, E = 160: 38 us both passes; 42 us with four times the CTAs)
    const int most = device_sm_count() * 2;
    const int want = (T + tokens - 1) / tokens;
    return launch_pdl(kernel, dim3(want < most ? want : most), dim3(256), smem, stream, grad_logits, gating, topk_ids, counts,
                      num_tokens, grad_losses, grad_topk_weights, token_mask, T, E, k, renormalize);
  });
  if (int st = check_cuda(e, "router_backward launch")) return st;
  count_launches(1);
  return check_launch("router_backward");
}

}  // namespace moe_b200
