// Products with 4-bit weights and group scales, for few tokens: dense (w4_linear) and over the routed experts.
//   W[n, k] = (code[n, k] - zero[n, k / g]) * scale[n, k / g]     codes two a byte, low nibble first; zero = 8 if not given
//   dense    y[m, n] = bf16(sum_k W[n, k] x[m, k] + bias[n])
//   experts  h = act(W13_e x_t + b13_e);  out[t] = bf16(sum_j w_tj (W2_e h_tj + b2_e)),  e = topk_ids[t, j]
//
// Bound: the weight bytes. An SM has to turn 23 bytes = 46 codes a cycle into products to keep up with HBM, which plain
// fused multiply-adds cannot (one instruction a code and token), so the products run on the tensor cores with the WEIGHTS as the
// 16-row operand and 8 tokens as columns (mma m16n8k16; tcgen05 wants its operand in shared or tensor memory, i.e. the
// unpacked weights written out once more, four times the bytes that come in, for tiles that are 128 rows high). A code
// becomes bf16 in two instructions for two codes: (w >> 4i) & 0x000f000f | 0x43004300 is the pair (128 + code_i, 128 + code_{i+4}) of an
// eight-code word, minus (128 + zero) is exact. Products with x are exact in fp32; a group's sum is scaled in fp32.
// The pairing (i, i + 4) is undone on the activations' side (four byte permutes per eight tokens and eight words).
//
// Work: a worker is kWk warps that split K; it takes tiles of 16 * kRB weight rows x up to 8 * kTB tokens in turn. Every warp
// streams its 128-column chunks of codes and activations through a ring of its own with 16-byte cp.async, which runs on
// into the next tile, so the warps never wait for one another inside a tile; the warps' sums meet in shared memory at its end.
#include "launch.cuh"
#include "moe_b200_internal.cuh"
#include "ptx.cuh"

namespace moe_b200 {

namespace {

constexpr int kWarps = 8;
constexpr int kChunk = 128;         // columns of a step
constexpr int kListSlots = 1024;    // slots whose lists are built in shared memory
constexpr int kListExperts = 1024;

enum W4Mode { kDense = 0, kGateUp = 1, kDown = 2 };

struct W4Params {
  W4Matrix w;
  int rows;               // weight rows of one matrix (dense N, 2 I, H)
  int K;
  int wk_log2;            // log2 of the warps of a worker
  int row_tiles;
  const __nv_bfloat16* x;  // dense / gate_up: [tokens, K]; down: [slots][2][K], the high and the low part
  long long x_ld;
  int m;                  // dense: tokens; experts: slots
  const int* ids;
  int top_k;
  int E;
  int activation;
  const float* topk_w;
  void* out;              // dense bf16 [m][rows]; gate_up bf16 [slots][2][I]; down fp32 [slots][rows]
};

// Token blocks of the routed experts: slots in expert order and, per block, its expert and where its slots are.
struct SlotLists {
  uint16_t slots[kListSlots];
  uint16_t expert[kListSlots];
  uint16_t start[kListSlots];
  uint8_t count[kListSlots];
  int blocks;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Codes i and i + 4 of a word as bf16 minus the zero point; zz holds 128 + zero twice.
template <int i>
__device__ __forceinline__ uint32_t unpack(uint32_t w, uint32_t zz) {
  return sub_bf16x2(((w >> (4 * i)) & 0x000f000fu) | 0x43004300u, zz);
}

__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float w4_act(float gate, float up, int activation) {
  if (activation == 0) return gate / (1.f + __expf(-gate)) * up;
  const float g = fminf(gate, 7.f), u = fminf(fmaxf(up, -7.f), 7.f);
  return g / (1.f + __expf(-1.702f * g)) * (u + 1.f);
}

// Sorts the slots by expert, in ascending order inside an expert (every CTA of both passes has to find the same
// blocks), and cuts each expert's into blocks of `width`. A warp ranks its 128 slots 32 at a time with match.any over its own row
// of `table` [kWarps][E]; a prefix over the warps and one over the experts give every slot its place. Called by the whole CTA.
__device__ void build_lists(SlotLists& l, int* count, uint16_t* table, const int* __restrict__ ids, int numel, int E, int width) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  uint16_t* row = table + warp * E;
  for (int e = lane; e < E; e += 32) row[e] = 0;
  __syncwarp();
  constexpr int kPer = kListSlots / (32 * kWarps);
  int mine[kPer], pos[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = (warp * kPer + i) * 32 + lane;
    mine[i] = s < numel ? ids[s] : -1;
    if (mine[i] >= E || mine[i] < 0) mine[i] = -1;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const unsigned same = __match_any_sync(0xffffffffu, mine[i]);
    const int rank = __popc(same & ((1u << lane) - 1u));
    const int base = mine[i] >= 0 ? row[mine[i]] : 0;
    pos[i] = base + rank;
    __syncwarp();
    if (mine[i] >= 0 && rank == 0) row[mine[i]] = static_cast<uint16_t>(base + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  for (int e = t; e < E; e += blockDim.x) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int c = table[w * E + e];
      table[w * E + e] = static_cast<uint16_t>(sum);
      sum += c;
    }
    count[e] = sum;
  }
  __syncthreads();
  if (t < 32) {  // first slot and first block of every expert, packed into one word for the scan
    int base = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + t;
      const int c = e < E ? count[e] : 0;
      const int v = c | (((c + width - 1) / width) << 16);
      int s = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, s, d);
        if (t >= d) s += o;
      }
      const int first = base + s - v;
      if (e < E) count[e] = first & 0xffff;
      for (int b = 0; b * width < c; ++b) {
        const int at = (first >> 16) + b;
        l.expert[at] = static_cast<uint16_t>(e);
        l.start[at] = static_cast<uint16_t>((first & 0xffff) + b * width);
        l.count[at] = static_cast<uint8_t>(min(width, c - b * width));
      }
      base += __shfl_sync(0xffffffffu, s, 31);
    }
    if (t == 0) l.blocks = base >> 16;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (mine[i] >= 0) l.slots[count[mine[i]] + row[mine[i]] + pos[i]] = static_cast<uint16_t>((warp * kPer + i) * 32 + lane);
  __syncthreads();
}

template <int kMode, int kRB, int kTB>
struct W4Shape {
  static constexpr int kParts = kMode == kDown ? 2 : 1;  // high and low part of the activations
  static constexpr int kRows = 16 * kRB;
  static constexpr int kTokens = 8 * kTB;
  static constexpr int kA = kRows * 64;
  static constexpr int kX = kTokens * 256;
  static constexpr int kStage = kA + kParts * kX;
  static constexpr int kStages = (24 * 1024) / kStage < 6 ? ((24 * 1024) / kStage < 3 ? 3 : (24 * 1024) / kStage) : 6;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kRedLd = kRows + 4;  // floats between two tokens' sums: lanes (row g, tokens 2t) hit 32 banks
  static constexpr int kRed = kWarps * kTokens * kRedLd * 4;
  static constexpr int kLists = kMode == kDense ? 0 : static_cast<int>(sizeof(SlotLists)) + kListExperts * 4;
  static constexpr int kSmem = kRing + kRed + (kLists + 15) / 16 * 16;
};

// What a tile is: its token block's columns and the first weight row of each of its row blocks.
struct Tile {
  int n;        // tokens
  int base;     // dense: first token; experts: first entry of the slot list
  int row;      // first row of the tile (gate_up: first of its 8 * kRB intermediate columns)
  long long mat;  // first row of the expert's matrix
};

template <int kMode, int kRB, int kTB>
__global__ void __launch_bounds__(32 * kWarps, 1) w4_mma_kernel(const W4Params p) {
  using S = W4Shape<kMode, kRB, kTB>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wk = 1 << p.wk_log2;
  const int kw = warp & (wk - 1);                                        // this warp's share of K
  const int worker = (blockIdx.x * kWarps + warp) >> p.wk_log2;
  const int workers = (gridDim.x * kWarps) >> p.wk_log2;
  const uint32_t ring = smem_u32(smem) + warp * (S::kStages * S::kStage);
  float* red = reinterpret_cast<float*>(smem + S::kRing);
  SlotLists& lists = *reinterpret_cast<SlotLists*>(smem + S::kRing + S::kRed);

  grid_dependency_wait();
  grid_dependency_launch();

  int blocks;
  if (kMode == kDense) {
    blocks = (p.m + S::kTokens - 1) / S::kTokens;
  } else {
    static_assert(kMode == kDense || S::kRed >= kWarps * kListExperts * 2, "the table of the sort borrows the sums' place");
    build_lists(lists, reinterpret_cast<int*>(&lists + 1), reinterpret_cast<uint16_t*>(red), p.ids, p.m, p.E, S::kTokens);
    blocks = lists.blocks;
  }
  const int tiles = blocks * p.row_tiles;
  const int chunks = (p.K + kChunk - 1) / kChunk;
  const int steps = (chunks - kw + wk - 1) >> p.wk_log2;  // of this warp in a tile
  const int gpc_log2 = p.w.group == 128 ? 0 : (p.w.group == 64 ? 1 : 2);  // groups in a chunk
  const int groups = p.K / p.w.group;

  auto tile_at = [&](int i) {
    Tile r;
    if (kMode == kDense) {
      const int b = i % blocks;  // a row tile's token blocks follow each other: its weights come from L2 again
      r.row = i / blocks * S::kRows;
      r.base = b * S::kTokens;
      r.n = min(S::kTokens, p.m - r.base);
      r.mat = 0;
    } else {
      const int b = i / p.row_tiles;
      r.row = i % p.row_tiles * (kMode == kGateUp ? S::kRows / 2 : S::kRows);
      r.base = lists.start[b];
      r.n = lists.count[b];
      r.mat = static_cast<long long>(lists.expert[b]) * p.rows;
    }
    return r;
  };
  // weight row of row r (0 .. 15) of row block rb
  auto weight_row = [&](const Tile& tile, int rb, int r) -> int {
    if (kMode == kGateUp) {  // rows 0-7: gate of 8 columns of the intermediate, rows 8-15: up of the same columns
      const int j = tile.row + rb * 8 + (r & 7);
      return p.activation == 0 ? j + (r >> 3) * (p.rows >> 1) : 2 * j + (r >> 3);
    }
    return tile.row + rb * 16 + r;
  };
  auto x_row = [&](const Tile& tile, int n) -> const __nv_bfloat16* {
    if (kMode == kDense) return p.x + static_cast<long long>(tile.base + n) * p.x_ld;
    const int slot = lists.slots[tile.base + n];
    return p.x + static_cast<long long>(kMode == kGateUp ? slot / p.top_k : slot) * p.x_ld;
  };

  // ------------------------------------------------------------------ loads of one step into the ring
  int l_tile = worker, l_step = 0, l_slot = 0;
  Tile lt = {};
  const uint8_t* a_src[2 * kRB];
  bool a_ok[2 * kRB];
  const __nv_bfloat16* x_src[4 * kTB];
  auto open_tile = [&]() {
    if (l_tile >= tiles) return;
    lt = tile_at(l_tile);
#pragma unroll
    for (int i = 0; i < 2 * kRB; ++i) {
      const int row = weight_row(lt, i >> 1, (i & 1) * 8 + g);
      a_ok[i] = kMode == kGateUp || row < p.rows;
      a_src[i] = p.w.q + (lt.mat + (a_ok[i] ? row : 0)) * (p.K >> 1) + t * 16;
    }
#pragma unroll
    for (int i = 0; i < 4 * kTB; ++i) {
      const int n = i * 2 + (lane >> 4);
      x_src[i] = n < lt.n ? x_row(lt, n) + (lane & 15) * 8 : nullptr;
    }
  };
  auto load_step = [&]() {
    if (l_tile < tiles) {
      const int k0 = (kw + (l_step << p.wk_log2)) * kChunk;
      const uint32_t dst = ring + l_slot * S::kStage;
      const bool in_a = k0 + t * 32 < p.K;
#pragma unroll
      for (int i = 0; i < 2 * kRB; ++i) {
        const int r = i * 8 + g;
        cp_async_16(dst + r * 64 + ((t + (r >> 1)) & 3) * 16, in_a ? a_src[i] + (k0 >> 1) : p.w.q, in_a && a_ok[i] ? 16 : 0);
      }
      const bool in_x = k0 + (lane & 15) * 8 < p.K;
#pragma unroll
      for (int i = 0; i < 4 * kTB; ++i) {
        if (i * 2 < lt.n || i < 4) {
          const int n = i * 2 + (lane >> 4);
          const bool ok = in_x && x_src[i] != nullptr;
          const uint32_t at = dst + S::kA + n * 256 + (((lane & 15) ^ ((n & 1) * 4)) * 16);
#pragma unroll
          for (int part = 0; part < S::kParts; ++part)
            cp_async_16(at + part * S::kX, ok ? x_src[i] + k0 + part * p.K : p.x, ok ? 16 : 0);
        }
      }
      if (++l_step == steps) {
        l_step = 0;
        l_tile += workers;
        open_tile();
      }
    }
    cp_async_commit();
    if (++l_slot == S::kStages) l_slot = 0;
  };

  if (steps > 0) {
    open_tile();
#pragma unroll 1
    for (int i = 0; i < S::kStages - 1; ++i) load_step();
  }

  // ------------------------------------------------------------------ products
  int slot = 0;
  for (int tile_i = worker; tile_i < tiles; tile_i += workers) {
    const Tile tile = tile_at(tile_i);
    const int nb = kTB == 1 ? 1 : (tile.n + 7) >> 3;
    float tot[kRB][kTB][4];
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
      for (int tb = 0; tb < kTB; ++tb)
#pragma unroll
        for (int i = 0; i < 4; ++i) tot[rb][tb][i] = 0.f;
    // scales and zero points: lane t of a quad fetches those of group t of the chunk for its rows, one step ahead
    const __nv_bfloat16* s_src[2 * kRB];
    const uint8_t* z_src[2 * kRB];
#pragma unroll
    for (int i = 0; i < 2 * kRB; ++i) {
      const int row = weight_row(tile, i >> 1, (i & 1) * 8 + g);
      const long long at = (tile.mat + (kMode == kGateUp || row < p.rows ? row : 0)) * groups;
      s_src[i] = p.w.scale + at;
      z_src[i] = p.w.zero + at;
    }
    float s_next[2 * kRB];
    uint32_t z_next[2 * kRB];
    auto fetch_scales = [&](int step) {
      const int gi = ((kw + (step << p.wk_log2)) << gpc_log2) + (t & ((1 << gpc_log2) - 1));
      const bool ok = step < steps && gi < groups;
#pragma unroll
      for (int i = 0; i < 2 * kRB; ++i) {
        s_next[i] = ok ? __bfloat162float(s_src[i][gi]) : 0.f;
        z_next[i] = ok && p.w.zero != nullptr ? (z_src[i][gi] & 15u) * 0x00010001u + 0x43004300u : 0x43084308u;
      }
    };
    fetch_scales(0);
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      cp_async_wait<S::kStages - 2>();
      __syncwarp();
      load_step();  // into the slot that the previous step has left
      float s_cur[2 * kRB];
      uint32_t z_cur[2 * kRB];
#pragma unroll
      for (int i = 0; i < 2 * kRB; ++i) {
        s_cur[i] = s_next[i];
        z_cur[i] = z_next[i];
      }
      fetch_scales(step + 1);
      const uint32_t src = ring + slot * S::kStage;
      if (++slot == S::kStages) slot = 0;
      float acc[kRB][kTB][4];
      uint32_t zz[2 * kRB];
#pragma unroll
      for (int c = 0; c < 4; ++c) {  // 32 columns
        const int per = 4 >> gpc_log2;  // of these in a group
        if ((c & (per - 1)) == 0) {
          const int from = (lane & ~3) | (c >> (2 - gpc_log2));
#pragma unroll
          for (int i = 0; i < 2 * kRB; ++i) zz[i] = __shfl_sync(0xffffffffu, z_cur[i], from);
#pragma unroll
          for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
            for (int tb = 0; tb < kTB; ++tb)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[rb][tb][i] = 0.f;
        }
        uint32_t b[S::kParts][kTB][4];
#pragma unroll
        for (int tb = 0; tb < kTB; ++tb) {
          if (tb < nb) {
#pragma unroll
            for (int part = 0; part < S::kParts; ++part) {
              const uint4 v = ld_shared_v4(src + S::kA + part * S::kX + (tb * 8 + g) * 256 + (((c * 4 + t) ^ ((g & 1) * 4)) * 16));
              b[part][tb][0] = __byte_perm(v.x, v.z, 0x5410);  // (x0, x4)
              b[part][tb][1] = __byte_perm(v.x, v.z, 0x7632);  // (x1, x5)
              b[part][tb][2] = __byte_perm(v.y, v.w, 0x5410);  // (x2, x6)
              b[part][tb][3] = __byte_perm(v.y, v.w, 0x7632);  // (x3, x7)
            }
          }
        }
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb) {
          const uint32_t at = src + (rb * 16 + g) * 64 + ((c + (g >> 1)) & 3) * 16 + t * 4;
          const uint32_t lo = ld_shared_u32(at), hi = ld_shared_u32(at + 8 * 64);
          const uint32_t zl = zz[2 * rb], zh = zz[2 * rb + 1];
          const uint32_t a0 = unpack<0>(lo, zl), a1 = unpack<0>(hi, zh), a2 = unpack<1>(lo, zl), a3 = unpack<1>(hi, zh);
          const uint32_t a4 = unpack<2>(lo, zl), a5 = unpack<2>(hi, zh), a6 = unpack<3>(lo, zl), a7 = unpack<3>(hi, zh);
#pragma unroll
          for (int tb = 0; tb < kTB; ++tb) {
            if (tb < nb) {
#pragma unroll
              for (int part = 0; part < S::kParts; ++part) {
                mma_bf16(acc[rb][tb], a0, a1, a2, a3, b[part][tb][0], b[part][tb][1]);
                mma_bf16(acc[rb][tb], a4, a5, a6, a7, b[part][tb][2], b[part][tb][3]);
              }
            }
          }
        }
        if ((c & (per - 1)) == per - 1) {
          const int from = (lane & ~3) | (c >> (2 - gpc_log2));
#pragma unroll
          for (int rb = 0; rb < kRB; ++rb) {
            const float sl = __shfl_sync(0xffffffffu, s_cur[2 * rb], from), sh = __shfl_sync(0xffffffffu, s_cur[2 * rb + 1], from);
#pragma unroll
            for (int tb = 0; tb < kTB; ++tb) {
              tot[rb][tb][0] = fmaf(acc[rb][tb][0], sl, tot[rb][tb][0]);
              tot[rb][tb][1] = fmaf(acc[rb][tb][1], sl, tot[rb][tb][1]);
              tot[rb][tb][2] = fmaf(acc[rb][tb][2], sh, tot[rb][tb][2]);
              tot[rb][tb][3] = fmaf(acc[rb][tb][3], sh, tot[rb][tb][3]);
            }
          }
        }
      }
    }

    // ---------------------------------------------------------------- the worker's warps meet; epilogue
    auto worker_sync = [&]() {
      __syncwarp();
      if (wk > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + (warp >> p.wk_log2)), "r"(32 * wk) : "memory");
    };
    float* mine = red + warp * (S::kTokens * S::kRedLd);
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
      for (int tb = 0; tb < kTB; ++tb) {
        float* q = mine + (tb * 8 + 2 * t) * S::kRedLd + rb * 16 + g;
        q[0] = tot[rb][tb][0];
        q[S::kRedLd] = tot[rb][tb][1];
        q[8] = tot[rb][tb][2];
        q[S::kRedLd + 8] = tot[rb][tb][3];
      }
    worker_sync();
    const float* all = red + (warp - kw) * (S::kTokens * S::kRedLd);
    auto sum_at = [&](int n, int r) {
      float s = 0.f;
      for (int i = 0; i < wk; ++i) s += all[(i * S::kTokens + n) * S::kRedLd + r];
      return s;
    };
    const int th = kw * 32 + lane;
    if (kMode == kGateUp) {
      constexpr int kCols = S::kRows / 2;
      const int I = p.rows >> 1;
      __nv_bfloat16* h = static_cast<__nv_bfloat16*>(p.out);
      for (int i = th; i < tile.n * kCols; i += 32 * wk) {
        const int n = i / kCols, jj = i % kCols, j = tile.row + jj;
        if (j < I) {
          const int r = (jj >> 3) * 16 + (jj & 7);
          float gate = sum_at(n, r), up = sum_at(n, r + 8);
          if (p.w.bias != nullptr) {
            gate += __bfloat162float(p.w.bias[tile.mat + weight_row(tile, jj >> 3, jj & 7)]);
            up += __bfloat162float(p.w.bias[tile.mat + weight_row(tile, jj >> 3, 8 + (jj & 7))]);
          }
          const float v = w4_act(gate, up, p.activation);
          const __nv_bfloat16 v_hi = __float2bfloat16_rn(v);
          __nv_bfloat16* dst = h + static_cast<long long>(lists.slots[tile.base + n]) * 2 * I + j;
          dst[0] = v_hi;
          dst[I] = __float2bfloat16_rn(v - __bfloat162float(v_hi));
        }
      }
    } else {
      for (int i = th; i < tile.n * S::kRows; i += 32 * wk) {
        const int n = i / S::kRows, r = i % S::kRows, row = tile.row + r;
        if (row < p.rows) {
          float y = sum_at(n, r);
          if (p.w.bias != nullptr) y += __bfloat162float(p.w.bias[tile.mat + row]);
          if (kMode == kDense) {
            static_cast<__nv_bfloat16*>(p.out)[static_cast<long long>(tile.base + n) * p.rows + row] = __float2bfloat16_rn(y);
          } else {
            const int s = lists.slots[tile.base + n];
            static_cast<float*>(p.out)[static_cast<long long>(s) * p.rows + row] = y * p.topk_w[s];
          }
        }
      }
    }
    worker_sync();
  }
  cp_async_wait_all();
}

// out[t] = bf16(sum over the slots with an expert, in slot order)
__global__ void __launch_bounds__(256)
w4_sum_kernel(__nv_bfloat16* __restrict__ out, const float* __restrict__ c3, const int* __restrict__ ids, int E, int k, int H) {
  grid_dependency_wait();
  grid_dependency_launch();
  const int n = (blockIdx.x * blockDim.x + threadIdx.x) * 4;
  const int t = blockIdx.y;
  if (n >= H) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < k; ++j) {
    const long long slot = static_cast<long long>(t) * k + j;
    const int e = ids[slot];
    if (e < 0 || e >= E) continue;
    const float4 v = *reinterpret_cast<const float4*>(c3 + slot * H + n);
    s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
  }
  uint2 o;
  __nv_bfloat162 a = __floats2bfloat162_rn(s[0], s[1]), b = __floats2bfloat162_rn(s[2], s[3]);
  o.x = *reinterpret_cast<uint32_t*>(&a);
  o.y = *reinterpret_cast<uint32_t*>(&b);
  *reinterpret_cast<uint2*>(out + static_cast<long long>(t) * H + n) = o;
}

// Warps of a worker: all eight while the tiles are too few to keep as many workers busy, fewer when there are many.
int pick_wk_log2(long long tiles, int chunks, int sms) {
  int lg = 3;
  while (lg > 0 && ((1 << lg) > chunks || tiles >= static_cast<long long>(sms) * (kWarps >> lg) * 8)) --lg;
  return lg;
}

template <int kMode, int kRB, int kTB>
cudaError_t launch_shape(W4Params p, long long tiles, cudaStream_t stream) {
  using S = W4Shape<kMode, kRB, kTB>;
  static_assert(S::kSmem <= 227 * 1024, "ring, sums and lists have to fit an SM's shared memory");
  auto kernel = w4_mma_kernel<kMode, kRB, kTB>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  const int sms = device_sm_count();
  p.wk_log2 = pick_wk_log2(tiles, (p.K + kChunk - 1) / kChunk, sms);
  const long long ctas = (tiles * (1 << p.wk_log2) + kWarps - 1) / kWarps;
  return launch_pdl(kernel, dim3(static_cast<unsigned>(ctas < sms ? ctas : sms)), dim3(32 * kWarps), S::kSmem, stream, p);
}

}  // namespace

int launch_w4_linear(__nv_bfloat16* out, const __nv_bfloat16* x, long long x_ld, const W4Matrix& w, int M, int N, int K, cudaStream_t stream) {
  if (M == 0) return kStatusOk;
  W4Params p{};
  p.w = w; p.rows = N; p.K = K; p.x = x; p.x_ld = x_ld; p.m = M; p.out = out;
  const int rb = N <= 64 * device_sm_count() ? 2 : 4;
  p.row_tiles = (N + 16 * rb - 1) / (16 * rb);
  const int tb = M <= 8 ? 1 : 2;
  const long long tiles = static_cast<long long>(p.row_tiles) * ((M + 8 * tb - 1) / (8 * tb));
  if (tiles > 0x3fffffffll) return set_error(kStatusInvalidArgument, "w4_linear: M x N too large");
  cudaError_t e;
  if (rb == 2) e = tb == 1 ? launch_shape<kDense, 2, 1>(p, tiles, stream) : launch_shape<kDense, 2, 2>(p, tiles, stream);
  else e = tb == 1 ? launch_shape<kDense, 4, 1>(p, tiles, stream) : launch_shape<kDense, 4, 2>(p, tiles, stream);
  if (int st = check_cuda(e, "w4_linear launch")) return st;
  count_launches(1);
  return check_launch("w4_linear");
}

size_t w4_experts_workspace_bytes(int T, int top_k, int H, int I) {
  const int piece = top_k < kListSlots ? kListSlots / top_k : 1;
  const size_t slots = static_cast<size_t>(T < 1 ? 1 : (T < piece ? T : piece)) * top_k;
  return slots * (4 * static_cast<size_t>(I) + 4 * static_cast<size_t>(H));
}

int launch_w4_experts(__nv_bfloat16* out, const __nv_bfloat16* x, const W4Matrix& w13, const W4Matrix& w2, const float* topk_w,
                      const int* topk_ids, int T, int E, int top_k, int H, int I, int activation, void* workspace,
                      cudaStream_t stream) {
  if (E > kListExperts || top_k > kListSlots)
    return set_error(kStatusInvalidArgument, "fused_experts_w4: at most %d experts and %d slots a token", kListExperts, kListSlots);
  const int piece = kListSlots / top_k;  // tokens whose slots fit the lists in shared memory
  for (int t0 = 0; t0 < T; t0 += piece) {
    const int tt = T - t0 < piece ? T - t0 : piece;
    const int slots = tt * top_k;
    const int* ids = topk_ids + static_cast<long long>(t0) * top_k;
    __nv_bfloat16* h = static_cast<__nv_bfloat16*>(workspace);
    float* c3 = reinterpret_cast<float*>(h + static_cast<size_t>(slots) * 2 * I);
    const int active = slots < E ? slots : E;
    W4Params p{};
    p.w = w13; p.rows = 2 * I; p.K = H; p.x = x + static_cast<long long>(t0) * H; p.x_ld = H; p.m = slots; p.ids = ids; p.top_k = top_k;
    p.E = E; p.activation = activation; p.out = h;
    p.row_tiles = (I + 31) / 32;
    long long tiles = static_cast<long long>(active) * p.row_tiles;
    if (int st = check_cuda(launch_shape<kGateUp, 4, 1>(p, tiles, stream), "w4 gate_up launch")) return st;
    p.w = w2; p.rows = H; p.K = I; p.x = h; p.x_ld = 2 * I; p.topk_w = topk_w + static_cast<long long>(t0) * top_k; p.out = c3;
    p.row_tiles = (H + 63) / 64;
    tiles = static_cast<long long>(active) * p.row_tiles;
    if (int st = check_cuda(launch_shape<kDown, 4, 1>(p, tiles, stream), "w4 down launch")) return st;
    if (int st = check_cuda(launch_pdl(w4_sum_kernel, dim3((H / 4 + 255) / 256, tt), dim3(256), 0, stream,
                                       out + static_cast<long long>(t0) * H, c3, ids, E, top_k, H), "w4 sum launch"))
      return st;
    count_launches(3);
  }
  return check_launch("w4_experts");
}

}  // namespace moe_b200
