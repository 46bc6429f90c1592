// Products with 4-bit weights and group scales, for few tokens: dense (w4_linear) and over the routed experts.
//   W[n, k] = (code[n, k] - zero[n, k / g]) * scale[n, k / g]     codes two a byte, low nibble first; zero = 8 if not given
//   dense    y[m, n] = bf16(sum_k W[n, k] x[m, k] + bias[n])
//   experts  h = act(W13_e x_t + b13_e);  out[t] = bf16(sum_j w_tj (W2_e h_tj + b2_e)),  e = topk_ids[t, j]
//
// Bound: the weight bytes. An SM has to turn 23 bytes = 46 codes a cycle into products to keep up with HBM, which plain
// fused multiply-adds cannot (one instruction a code and token), so the products run on the tensor cores with the WEIGHTS as the
// 16-row operand and 8 tokens as columns. tcgen05 wants its operand in shared or tensor memory, i.e. the unpacked
// weights written out once more for tiles that are 128 rows high; mma.sync takes them from the registers in which they are unpacked.
// The integer form (m16n8k32, u8 codes) takes codes as they are: three instructions unpack eight of them (w & 0x0f0f0f0f and
// (w >> 4) & 0x0f0f0f0f), against seven to bf16 (shift, mask and a 128 that has to leave the sum again), and one instruction multiplies
// 32 columns instead of 16 at the same rate. Unpacking is what bounds the loop next to the loads.
//   The activations become 16-bit integers with a power of two f for every token and 128 columns:
//   x = f * (256 hi + lo), hi signed and lo unsigned bytes, two products a word; f puts the largest |x| of them between 2^14 and 2^15.
//   A bf16 value has 8 significant bits, so that all down to 2^-7 of the largest are exact and smaller ones are off by at most
//   2^-15 of the largest; the intermediate h of the experts (fp32) is off by that everywhere. Where a few columns stand out so far that this
//   would show in rows which have no weight for them (see kMarkBelow), what is cut off is added as 16 bits more: off by 2^-29 of the
//   largest then. Integer sums are exact; then
//   sum (code - zero) x = f * (256 sum code hi + sum code lo - zero * sum x) in fp32, times the group's scale, summed in fp32.
//   Where a value is not finite f is NaN, so that its token's results are NaN.
//   A CTA makes these integers itself where they are few; where many CTAs would make many of them (a batch, a long K) a kernel in
//   front does it once, while this one prepares its lists and its first codes.
// The sums start at 0x4b400000, which makes their bits the float 12582912 + sum: no conversion instruction.
//
// Work: a tile is 16 * kRB weight rows x one block of up to 8 * kTB tokens; a CTA takes consecutive tiles, so that it
// meets few token blocks. The activations of a window of them stay in shared memory as the integers above, in the
// order in which the codes come, next to their group sums. A worker is 1 to 16 warps that split a tile's columns. Every warp
// streams codes through a FIFO of its own (16-byte cp.async, four 128-column steps deep) that runs on into the next tile, so
// no warp waits for another inside a window. What bounds it now: the instructions of a step (about 200 for 32 rows, at two a cycle
// and SM, and the latency of its chain of codes, products and sums) and of a tile's end; the same loop without products reads at 5.2 to
// 5.7 TB/s, the cases below at 3.6 to 3.9. The sixteen warps and their rings leave 128 registers a thread, and two row blocks do not
// quite fit them: ptxas spills 44 to 100 bytes a thread there without zero points, 52 to 336 with them, 152 to 668 with two
// token blocks as well; one row block spills 0 to 48.
// Measured (graph replay): 64 tokens over 128 experts, H = 2048, I = 768: 84 us, 3.7 TB/s, against 205 us of the bf16 experts;
// 93 tokens, H = 4096, I = 1536, groups of 64: 335 us, 3.9 TB/s, as long as the card stays below its power limit, 368 us at 1.7 GHz
// when it has run into it (after 0.07 s of nothing else); N = 131075, K = 2048, groups of 32, five tokens: 42 us, 3.7 TB/s.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "launch.cuh"
#include "moe_b200_internal.cuh"
#include "ptx.cuh"

namespace moe_b200 {

namespace {

constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kChunk = 128;         // columns of a step
constexpr int kStages = 4;          // steps in a warp's FIFO
constexpr int kListSlots = 1024;    // slots whose lists are built in shared memory
constexpr int kListExperts = 1024;
constexpr size_t kPreparedChunks = 64;
constexpr int kMaxSmem = 227 * 1024 - 128;  // dynamic; the sort has a few words of its own

enum W4Mode { kDense = 0, kGateUp = 1, kDown = 2 };

struct W4Params {
  W4Matrix w;
  int rows;               // weight rows of one matrix (dense N, 2 I, H)
  int K;
  int span;               // columns whose activations are in shared memory at a time, a multiple of kChunk
  int cap;                // token rows whose activations fit
  int whole;              // K is a multiple of kChunk
  int scale_words;        // scales of a row can be read four (2), two (1) or one (0) at a time
  int wk_log2;            // log2 of the warps of a worker
  int row_tiles;
  const void* x;          // dense / gate_up: bf16 [tokens, K]; down: fp32 [slots, K]
  long long x_ld;
  int m;                  // dense: tokens; experts: slots
  const int* ids;
  int top_k;
  int E;
  int activation;
  const float* topk_w;
  const uint8_t* xq;      // integers made in front (quant_x_kernel), or null
  const float* xm;
  void* out;              // dense bf16 [m][rows]; gate_up fp32 [slots][I]; down fp32 [slots][rows]
};

// Token blocks of the routed experts: slots in expert order and, per block, its expert and where its slots are.
struct SlotLists {
  uint16_t slots[kListSlots];
  uint16_t expert[kListSlots];
  uint16_t start[kListSlots];
  uint8_t count[kListSlots];
  int blocks;
};

// d = c + codes (16 rows x 32 columns, u8) * x bytes (32 columns x 8 tokens), signed (the high bytes) or unsigned.
template <bool kSigned>
__device__ __forceinline__ void mma_codes(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
  if constexpr (kSigned)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}

// The same of signed bytes (what the zero point has left already).
template <bool kSigned>
__device__ __forceinline__ void mma_weights(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kSigned)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int kFloatBits = 0x4b400000;    // bits of 12582912.f, one more for every unit up to 2^22
constexpr float kFloatBias = 12582912.f;

// 16 bytes to shared memory (zeros for size 0), both at a constant distance behind an address.
template <int kDst, int kSrc>
__device__ __forceinline__ void cp_async_at(uint32_t dst, const uint8_t* src, uint32_t size) {
  asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16, %4;" ::"r"(dst), "l"(src), "n"(kDst), "n"(kSrc), "r"(size) : "memory");
}

// Reads of the FIFO, at a constant distance behind an address; volatile, for they must stay behind the wait for their copy.
template <int kOff>
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4+%5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr), "n"(kOff) : "memory");
  return v;
}
template <int kOff>
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2+%3];" : "=r"(v.x), "=r"(v.y) : "r"(addr), "n"(kOff) : "memory");
  return v;
}
template <int kOff>
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1+%2];" : "=r"(v) : "r"(addr), "n"(kOff) : "memory");
  return v;
}

__device__ __forceinline__ float w4_act(float gate, float up, int activation) {
  if (activation == 0) return __fdividef(gate, 1.f + __expf(-gate)) * up;
  // a NaN stays one: fminf and fmaxf would make a limit of it
  const float g = gate > 7.f ? 7.f : gate, u = up > 7.f ? 7.f : (up < -7.f ? -7.f : up);
  return __fdividef(g, 1.f + __expf(-1.702f * g)) * (u + 1.f);
}

// Sorts the slots by expert, in ascending order inside an expert (every CTA of both passes has to find the same
// blocks), and cuts each expert's into blocks of `width`. 32 slots rank themselves with match.any and leave their counts in a row of
// `table` [(numel + 31) / 32][E]; prefixes over the rows and over the experts give every slot its place. Called by the whole CTA.
__device__ void build_lists(SlotLists& l, int* first_of, uint16_t* table, const int* __restrict__ ids, int numel, int E, int width) {
  __shared__ int warp_total[kWarps];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  constexpr int kPer = kListSlots / kThreads;
  static_assert(kPer * kThreads == kListSlots);
  const int rows = (numel + 31) >> 5;
  int mine[kPer], rank[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = warp + i * kWarps;
    if (r >= rows) break;
    const int s = r * 32 + lane;
    mine[i] = s < numel ? ids[s] : -1;
    if (mine[i] >= E || mine[i] < 0) mine[i] = -1;
    for (int e = lane; e < E; e += 32) table[r * E + e] = 0;
    const unsigned same = __match_any_sync(0xffffffffu, mine[i]);
    rank[i] = __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (mine[i] >= 0 && rank[i] == 0) table[r * E + mine[i]] = static_cast<uint16_t>(__popc(same));
  }
  __syncthreads();
  int base = 0;  // slots so far, and blocks in the upper half
  for (int e0 = 0; e0 < E; e0 += kThreads) {
    const int e = e0 + t;
    int c = 0;
    if (e < E) {
      for (int r0 = 0; r0 < rows; r0 += 16) {
        int n[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) n[r] = r0 + r < rows ? table[(r0 + r) * E + e] : 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (r0 + r < rows) table[(r0 + r) * E + e] = static_cast<uint16_t>(c);
          c += n[r];
        }
      }
    }
    const int v = c | (((c + width - 1) / width) << 16);
    int s = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += o;
    }
    if (lane == 31) warp_total[warp] = s;
    __syncthreads();
    int before = base;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int n = warp_total[w];
      if (w < warp) before += n;
      base += n;
    }
    const int first = before + s - v;
    if (e < E) first_of[e] = first & 0xffff;
    for (int b = 0; b * width < c; ++b) {
      const int at = (first >> 16) + b;
      l.expert[at] = static_cast<uint16_t>(e);
      l.start[at] = static_cast<uint16_t>((first & 0xffff) + b * width);
      l.count[at] = static_cast<uint8_t>(min(width, c - b * width));
    }
    if (t == 0) l.blocks = base >> 16;
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = warp + i * kWarps;
    if (r >= rows) break;
    if (mine[i] >= 0) l.slots[first_of[mine[i]] + table[r * E + mine[i]] + rank[i]] = static_cast<uint16_t>(r * 32 + lane);
  }
  __syncthreads();
}

template <int kMode, int kRB, int kTB>
struct W4Shape {
  static constexpr int kRows = 16 * kRB;
  static constexpr int kTokens = 8 * kTB;
  static constexpr int kStage = kRows * 64;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kRed = kWarps * kRB * kTB * 4 * 32 * 4;
  static constexpr int kLists = kMode == kDense ? 0 : (static_cast<int>(sizeof(SlotLists)) + 15) / 16 * 16;
  // a token row of `span` columns: 64 bytes more than a multiple of 128, so that the two tokens of an eight-lane phase of a
  // 16-byte read use different banks
  __host__ __device__ static constexpr int x_ld(int span) { return span * 2 + 64; }
  __host__ __device__ static constexpr int x_row_bytes(int span, int gpc) { return x_ld(span) + (span / kChunk * (gpc + 1) | 1) * 4; }
  static constexpr int kFixed = kRing + kRed + kLists;
};

// kGpc: groups in a chunk; kZero: zero points are given. Lane (g, t) = (lane / 4, lane % 4) of a warp holds row g and g + 8 of a row block; its word j of a
// chunk of 128 columns starts at column col_of(j, t), so that the columns of a word index belong to one group.
template <int kGpc>
__device__ __forceinline__ int col_of(int j, int t) {
  return kGpc == 1 ? 32 * t + 8 * j : (kGpc == 2 ? 64 * (j >> 1) + 16 * t + 8 * (j & 1) : 32 * j + 8 * t);
}

// v: integers in their low 16 bits. Bytes 1 (high) of columns 0, 2, 4, 6 and of 1, 3, 5, 7, then bytes 0.
__device__ __forceinline__ uint4 pack_ints(const uint32_t (&v)[8]) {
  uint32_t o[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t a02 = __byte_perm(v[h], v[2 + h], 0x5410), a46 = __byte_perm(v[4 + h], v[6 + h], 0x5410);
    o[h] = __byte_perm(a02, a46, 0x7531);
    o[2 + h] = __byte_perm(a02, a46, 0x6420);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// The float whose low 16 bits are x / f rounded to nearest. An fp32 value may lie past 32767.5, a bf16 one does not.
template <bool kFp32>
__device__ __forceinline__ float int_of(float x, float to_int) {
  return kFp32 ? fminf(x * to_int, 32767.f) + kFloatBias : fmaf(x, to_int, kFloatBias);
}

// A chunk of a token whose integers cut off too much of it is marked in the last bit of its f (which moves its products by 2^-23, no
// more than one of the additions that follow), and what they cut off is added behind the loop. An integer is off by at most 1/2,
// all 128 together by at most 5.7 and as a rule by 3.3 (their norm). With every magnitude counted as 1024 at most (2^-4 to 2^-5 of the
// largest), a chunk below kMarkBelow, that is of a norm below 4096, is marked: in the others the columns left next to any eight
// have a norm of 2896, so that what is cut off stays below 2^-9 of them, a rounding of the output, also in rows whose weights for
// those eight are zero. Of normally distributed values none are marked, of those with a column of 100 times the rest all.
constexpr float kMarkCap = 1024.f, kMarkBelow = 16.f * kMarkCap * kMarkCap;
constexpr uint32_t kMark = 1;

// The integers of 128 columns of a token by sixteen neighbouring lanes, lane u holding the eight columns from col_of(u / 4, u % 4) on.
// ints: see pack_ints; sum: of its group; returns f, marked or not.
template <int kGpc, bool kFp32>
__device__ __forceinline__ float quant_x(const float (&x)[8], uint4& ints, int& sum) {
  uint32_t big = 0;  // the largest magnitude as bits, which order like the values, NaN last
#pragma unroll
  for (int k = 0; k < 8; ++k) big = max(big, __float_as_uint(x[k]) & 0x7fffffffu);
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, m));
  const bool finite = big < 0x7f800000u;
  const int e = min(max(static_cast<int>(big >> 23), 20), 254);  // biased exponent; 2^-107 and less count as that
  const float to_int = __uint_as_float(static_cast<uint32_t>(254 + 14 - e) << 23);  // 2^(14 - exponent)
  uint32_t v[8];
  sum = 0;
  float norm = 0.f;  // its square
  bool cut = false;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float i = int_of<kFp32>(x[k], to_int), scaled = x[k] * to_int;
    v[k] = __float_as_uint(i);
    sum += static_cast<int>(v[k]) - kFloatBits;
    const float m = fminf(fabsf(scaled), kMarkCap);
    norm = fmaf(m, m, norm);
    cut |= i - kFloatBias != scaled;
  }
  ints = pack_ints(v);
  if (!finite) sum = 0;
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  sum += __shfl_xor_sync(0xffffffffu, sum, 2);
  if (kGpc < 4) sum += __shfl_xor_sync(0xffffffffu, sum, 4);
  if (kGpc < 2) sum += __shfl_xor_sync(0xffffffffu, sum, 8);
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) norm += __shfl_xor_sync(0xffffffffu, norm, m);
  const uint32_t cuts = __ballot_sync(0xffffffffu, cut) >> (threadIdx.x & 16) & 0xffffu;
  if (!finite) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(static_cast<uint32_t>(e - 14) << 23 | (norm < kMarkBelow && cuts != 0 ? kMark : 0));
}

__device__ __forceinline__ void load_x8(const __nv_bfloat16* src, float (&x)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(src);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[2 * k] = __uint_as_float(w[k] << 16);
    x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load_x8(const float* src, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// xq [rows][chunks][256] and xm [rows][chunks][kGpc + 1] (the groups' sums, f) of bf16 rows.
template <int kGpc>
__global__ void __launch_bounds__(256)
quant_x_kernel(uint8_t* __restrict__ xq, float* __restrict__ xm, const __nv_bfloat16* __restrict__ x, long long x_ld, int rows, int K) {
  grid_dependency_wait();
  grid_dependency_launch();
  const int chunks = (K + kChunk - 1) / kChunk;
  const long long at = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 4;  // chunk of a row
  const int u = threadIdx.x & 15;
  const bool ok = at < static_cast<long long>(rows) * chunks;
  const int row = ok ? static_cast<int>(at / chunks) : 0, c = ok ? static_cast<int>(at % chunks) : 0;
  const int col = c * kChunk + col_of<kGpc>(u >> 2, u & 3);
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (col < K) load_x8(x + row * x_ld + col, v);
  uint4 ints;
  int sum;
  const float f = quant_x<kGpc, false>(v, ints, sum);
  if (!ok) return;
  *reinterpret_cast<uint4*>(xq + at * 256 + u * 16) = ints;
  constexpr int kUnits = 16 / kGpc;
  if (u % kUnits == 0) xm[at * (kGpc + 1) + u / kUnits] = static_cast<float>(sum);
  if (u == 0) xm[at * (kGpc + 1) + kGpc] = f;
}

template <int kMode, int kRB, int kTB, int kGpc, bool kZero>
__global__ void __launch_bounds__(kThreads, 1) w4_mma_kernel(const W4Params p) {
  using S = W4Shape<kMode, kRB, kTB>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wk = 1 << p.wk_log2;
  const int kw = warp & (wk - 1);             // this warp's share of the columns
  const int worker = warp >> p.wk_log2;
  const int workers = kWarps >> p.wk_log2;
  uint8_t* const fifo = smem + warp * (kStages * S::kStage);
  float* const red = reinterpret_cast<float*>(smem + S::kRing);
  SlotLists& lists = *reinterpret_cast<SlotLists*>(smem + S::kRing + S::kRed);
  uint8_t* const x_mem = smem + S::kRing + S::kRed + S::kLists;
  const int x_ld = S::x_ld(p.span);
  float* const x_sum = reinterpret_cast<float*>(x_mem + p.cap * x_ld);  // [cap][chunks][kGpc sums of the integers, f], rows of an odd length
  const int xs_ld = p.span / kChunk * (kGpc + 1) | 1;

  // The down pass follows the gate_up pass, and a pass with prepared integers the kernel that makes them, and both let this one
  // start only after their own wait: all but what they write is there already, so that the lists are made and the first codes
  // are under way before the wait.
  const bool early = kMode == kDown || p.xq != nullptr;
  if (!early) {
    grid_dependency_wait();
    grid_dependency_launch();
  }

  int blocks;
  if (kMode == kDense) {
    blocks = (p.m + S::kTokens - 1) / S::kTokens;
  } else {
    static_assert(kMode == kDense || S::kRing + S::kRed >= kListSlots / 32 * kListExperts * 2 + kListExperts * 4, "the sort borrows the place of FIFOs and sums");
    build_lists(lists, reinterpret_cast<int*>(smem), reinterpret_cast<uint16_t*>(smem + kListExperts * 4), p.ids, p.m, p.E, S::kTokens);
    blocks = lists.blocks;
  }
  // this CTA's tiles, token block by token block
  const long long total = static_cast<long long>(blocks) * p.row_tiles;
  const int first = static_cast<int>(total * blockIdx.x / gridDim.x), last = static_cast<int>(total * (blockIdx.x + 1) / gridDim.x);
  if (first == last) {
    if (early) grid_dependency_wait();
    return;
  }

  const int spans = (p.K + p.span - 1) / p.span;
  const int groups = p.K / p.w.group;
  const uint32_t row_bytes = static_cast<uint32_t>(p.K) >> 1;
  // Row r (0 .. 15) of row block rb lies rb * step_rb + (r / 8) * step_half + (r % 8) * step_row rows behind the tile's first.
  // gate_up: rows 0-7 of a block are the gate of 8 columns of the intermediate, rows 8-15 their up.
  const int step_row = kMode == kGateUp && p.activation != 0 ? 2 : 1;
  const int step_half = kMode != kGateUp ? 8 : (p.activation == 0 ? p.rows >> 1 : 1);
  const int step_rb = kMode == kGateUp ? 8 * step_row : 16;
  // Rows past the end (of a matrix with fewer than kRows) are read as the last one, and not written.
  const int row_lo = kMode == kGateUp ? g * step_row : min(g, p.rows - 1);
  uint32_t q_off[2 * kRB], s_off[2 * kRB];  // of this lane's rows in bytes of codes and in groups, from row_lo on
#pragma unroll
  for (int i = 0; i < 2 * kRB; ++i) {
    const int row = kMode == kGateUp ? (i >> 1) * step_rb + (i & 1) * step_half : min(8 * i + g, p.rows - 1) - row_lo;
    q_off[i] = static_cast<uint32_t>(row) * row_bytes;
    s_off[i] = static_cast<uint32_t>(row) * groups;
  }
  auto first_row = [&](int r) -> int {  // of row tile r
    // the last tile takes rows of the one before again rather than rows past the end
    return kMode == kGateUp ? r * (S::kRows / 2) : max(0, min(r * S::kRows, p.rows - S::kRows));
  };
  auto first_row_of_matrix = [&](int block) -> long long {
    return kMode == kDense ? 0 : static_cast<long long>(lists.expert[block]) * p.rows;
  };
  auto entries_of = [&](int block, int& base, int& n) {  // first entry (token, place in the slot list) and number of a block's
    base = kMode == kDense ? block * S::kTokens : lists.start[block];
    n = kMode == kDense ? min(S::kTokens, p.m - base) : lists.count[block];
  };
  // A place in this CTA's work: tile number, its token block and its row tile. Going on from one to the next takes no division.
  struct Place {
    int tile, block, r;
  };
  auto advance = [&](Place& at, int by) {
    at.tile += by;
    at.r += by;
    while (at.r >= p.row_tiles) {
      at.r -= p.row_tiles;
      ++at.block;
    }
  };
  const int first_block = first / p.row_tiles, last_block = (last - 1) / p.row_tiles;
  auto window_end = [&](int block) {  // the blocks from `block` on whose activations fit together, those of this CTA
    if (spans > 1) return block + 1;
    int base, at, n;
    entries_of(block, base, n);
    int b = block + 1;
    for (; b <= last_block; ++b) {
      entries_of(b, at, n);
      if (at + n - base > p.cap) break;
    }
    return b;
  };
  auto chunks_of = [&](int span_i, int& begin, int& n) {  // this warp's chunks of a span
    const int chunks = (min(p.span, p.K - span_i * p.span) + kChunk - 1) / kChunk;
    begin = (kw * chunks) >> p.wk_log2;
    n = (((kw + 1) * chunks) >> p.wk_log2) - begin;
  };

  // ------------------------------------------------------------------ codes: one step of this warp into its FIFO
  int l_end_block = window_end(first_block), l_end = min(last, l_end_block * p.row_tiles);  // of the window
  Place l_at{first, first_block, first - first_block * p.row_tiles};
  advance(l_at, worker);
  int l_span = 0, l_left = 0, l_col = 0;
  const uint8_t* l_src[2 * kRB];
  auto open = [&]() {  // (l_at, l_span); a worker's tiles are `workers` apart inside a window
    while (l_at.tile >= l_end) {
      if (l_end == last) {
        l_at.tile = last;
        return;
      }
      l_at = Place{l_end, l_end_block, 0};
      advance(l_at, worker);
      l_end_block = window_end(l_end_block);
      l_end = min(last, l_end_block * p.row_tiles);
    }
    int begin;
    chunks_of(l_span, begin, l_left);
    l_col = l_span * p.span + begin * kChunk + t * 32;
    const uint8_t* src = p.w.q + (first_row_of_matrix(l_at.block) + first_row(l_at.r) * step_row + row_lo) * row_bytes + (l_col >> 1);
#pragma unroll
    for (int i = 0; i < 2 * kRB; ++i) l_src[i] = src + q_off[i];
  };
  // 16-byte piece u of a row of 64 bytes is kept at u ^ swap: the reads below are free of bank conflicts at every width
  const int swap = (g & 2) | ((g >> 2) & 1);
  const uint32_t l_dst = smem_u32(fifo) + g * 64 + ((t ^ swap) * 16);
  // Chunk kSlot of four; a tile's chunks begin at slot 0, and what is missing to a multiple of four stays empty.
  auto load_chunk = [&](auto slot_c) {
    constexpr int kSlot = decltype(slot_c)::value;
    if (kSlot < l_left) {
      const uint32_t size = p.whole || l_col + kSlot * kChunk < p.K ? 16 : 0;  // zeros are written behind the last column
      cp_async_at<kSlot * S::kStage, kSlot * (kChunk / 2)>(l_dst, l_src[0], size);
      cp_async_at<kSlot * S::kStage + 512, kSlot * (kChunk / 2)>(l_dst, l_src[1], size);
      if constexpr (kRB > 1) {
        cp_async_at<kSlot * S::kStage + 1024, kSlot * (kChunk / 2)>(l_dst, l_src[2 % (2 * kRB)], size);
        cp_async_at<kSlot * S::kStage + 1536, kSlot * (kChunk / 2)>(l_dst, l_src[3 % (2 * kRB)], size);
      }
    }
    cp_async_commit();
    if (kSlot == kStages - 1) {
      l_left -= kStages;
      l_col += kStages * kChunk;
#pragma unroll
      for (int i = 0; i < 2 * kRB; ++i) l_src[i] += kStages * kChunk / 2;
      if (l_left <= 0 && l_at.tile < last) {
        if (++l_span == spans) {
          l_span = 0;
          advance(l_at, workers);
        }
        l_left = 0;
        open();
      }
    }
  };

  // ------------------------------------------------------------------ activations of entries and a span of columns
  using X = std::conditional_t<kMode == kDown, float, __nv_bfloat16>;
  auto source_row = [&](int entry) -> long long {
    if (kMode == kDense) return entry;
    return kMode == kGateUp ? lists.slots[entry] / p.top_k : lists.slots[entry];
  };
  auto load_x = [&](int base, int n, int span_i) -> bool {  // whether this thread has met a marked chunk
    const int c0 = span_i * p.span;
    const int chunks = (min(p.span, p.K - c0) + kChunk - 1) / kChunk;
    uint32_t marks = 0;
    // half a warp takes a chunk of a token
    int row = 0, c = warp * 2 + (lane >> 4);
    const int u = lane & 15;
    if (kMode != kDown && p.xq != nullptr) {
      // not by cp.async: its wait would be for the codes under way too
      const int all = (p.K + kChunk - 1) / kChunk;
      constexpr int kAhead = 4;
      for (int at = warp * 2; at < n * chunks; at += kAhead * 2 * kWarps) {
        uint4 v[kAhead];
        float s[kAhead];
        int to[kAhead], to_s[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          while (c >= chunks) {
            c -= chunks;
            ++row;
          }
          const int r = min(row, n - 1);  // behind the last chunk: one of the last token again
          const long long src = source_row(base + r) * all + c0 / kChunk + c;
          v[i] = *reinterpret_cast<const uint4*>(p.xq + src * 256 + u * 16);
          s[i] = u <= kGpc ? p.xm[src * (kGpc + 1) + u] : 0.f;
          to[i] = r * x_ld + c * 256 + u * 16;
          to_s[i] = r * xs_ld + c * (kGpc + 1) + u;
          if (u == kGpc) marks |= __float_as_uint(s[i]);
          c += 2 * kWarps;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          *reinterpret_cast<uint4*>(x_mem + to[i]) = v[i];
          if (u <= kGpc) x_sum[to_s[i]] = s[i];
        }
      }
      return (marks & kMark) != 0;
    }
    for (int at = warp * 2; at < n * chunks; at += 2 * kWarps) {
      while (c >= chunks) {
        c -= chunks;
        ++row;
      }
      const int r = min(row, n - 1);
      const int col = c0 + c * kChunk + col_of<kGpc>(u >> 2, u & 3);
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (col < p.K) load_x8(static_cast<const X*>(p.x) + source_row(base + r) * p.x_ld + col, v);
      uint4 ints;
      int sum;
      const float f = quant_x<kGpc, kMode == kDown>(v, ints, sum);
      *reinterpret_cast<uint4*>(x_mem + r * x_ld + c * 256 + u * 16) = ints;
      constexpr int kUnits = 16 / kGpc;
      if (u % kUnits == 0) x_sum[r * xs_ld + c * (kGpc + 1) + u / kUnits] = static_cast<float>(sum);
      if (u == 0) x_sum[r * xs_ld + c * (kGpc + 1) + kGpc] = f;
      marks |= __float_as_uint(f);
      c += 2 * kWarps;
    }
    return (marks & kMark) != 0;
  };

  // ------------------------------------------------------------------ scales and zero points of this lane's rows
  // Four scales of a row (kUnit chunks) are fetched at a time, where they start on their size with one load: an SM has more rows
  // under way than its first-level cache has lines, so that every further load of a row would go to the second level again. The
  // fetch is one unit ahead, that of a tile's first unit in front of the end of the tile before.
  constexpr int kUnit = 4 / kGpc;
  const __nv_bfloat16* s_src[2 * kRB];
  const uint8_t* z_src = nullptr;
  int gi = 0, words = 0;
  uint32_t s_next[2 * kRB][2], z_next[2 * kRB];
  bool fetched = false;
  auto open_scales = [&](const Place& at, int span_i) {
    int begin, n;
    chunks_of(span_i, begin, n);
    gi = (span_i * p.span / kChunk + begin) * kGpc;
    words = gi % 4 == 0 ? p.scale_words : (gi % 2 == 0 ? min(p.scale_words, 1) : 0);
    const long long s_at = (first_row_of_matrix(at.block) + first_row(at.r) * step_row + row_lo) * groups + gi;
#pragma unroll
    for (int i = 0; i < 2 * kRB; ++i) s_src[i] = p.w.scale + s_at + s_off[i];
    z_src = p.w.zero + s_at;
  };
  auto fetch_scales = [&](auto ahead_c) {  // of the unit so many chunks behind s_src
    constexpr int kAhead = decltype(ahead_c)::value * kGpc;
    if (words == 2) {
#pragma unroll
      for (int i = 0; i < 2 * kRB; ++i) {
        const uint2 v = *reinterpret_cast<const uint2*>(s_src[i] + kAhead);
        s_next[i][0] = v.x;
        s_next[i][1] = v.y;
        if (kZero) z_next[i] = *reinterpret_cast<const uint32_t*>(z_src + s_off[i] + kAhead);
      }
    } else if (words == 1) {
#pragma unroll
      for (int i = 0; i < 2 * kRB; ++i) {
        const bool more = gi + kAhead + 2 < groups;
        s_next[i][0] = *reinterpret_cast<const uint32_t*>(s_src[i] + kAhead);
        s_next[i][1] = more ? *reinterpret_cast<const uint32_t*>(s_src[i] + kAhead + 2) : 0;
        if (kZero) {
          z_next[i] = *reinterpret_cast<const uint16_t*>(z_src + s_off[i] + kAhead);
          if (more) z_next[i] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(z_src + s_off[i] + kAhead + 2)) << 16;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2 * kRB; ++i) {
        s_next[i][0] = s_next[i][1] = 0;
        if (kZero) z_next[i] = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (gi + kAhead + q < groups) {
            s_next[i][q / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(s_src[i] + kAhead + q)) << (16 * (q & 1));
            if (kZero) z_next[i] |= static_cast<uint32_t>(z_src[s_off[i] + kAhead + q]) << (8 * q);
          }
        }
      }
    }
  };

  open();
  load_chunk(std::integral_constant<int, 0>{});
  load_chunk(std::integral_constant<int, 1>{});
  load_chunk(std::integral_constant<int, 2>{});
  if (early) {
    grid_dependency_wait();
    grid_dependency_launch();
  }

  // ------------------------------------------------------------------ products
  const int start[4] = {kFloatBits, kFloatBits, kFloatBits, kFloatBits};
  const uint32_t fifo_lane = smem_u32(fifo) + g * 64;
  int marked = 0;  // whether a chunk of the activations in shared memory is
  for (int block0 = first_block; block0 <= last_block;) {
    const int block1 = window_end(block0);
    Place at{first, first_block, first - first_block * p.row_tiles};
    if (block0 > first_block) at = Place{block0 * p.row_tiles, block0, 0};
    const int win_last = min(last, block1 * p.row_tiles);
    const int rounds = (win_last - at.tile + workers - 1) >> (4 - p.wk_log2);
    advance(at, worker);
    int win_base, win_n, base, n_tokens;
    entries_of(block0, win_base, win_n);
    entries_of(block1 - 1, base, n_tokens);
    win_n = base + n_tokens - win_base;
    for (int round = 0; round < rounds; ++round) {
      const bool active = at.tile < win_last;
      const int block = active ? at.block : block0;
      entries_of(block, base, n_tokens);
      const int row0 = first_row(at.r);
      const long long mat = first_row_of_matrix(block);
      const Place here = at;
      advance(at, workers);
      // columns past the block's tokens are not written: they take the last one's activations
      const uint8_t* x_lane[kTB];
      const float* xs_lane[kTB][2];
#pragma unroll
      for (int tb = 0; tb < kTB; ++tb) {
        x_lane[tb] = x_mem + (base - win_base + min(tb * 8 + g, n_tokens - 1)) * x_ld + t * 16;
#pragma unroll
        for (int o = 0; o < 2; ++o)
          xs_lane[tb][o] = x_sum + (base - win_base + min(tb * 8 + 2 * t + o, n_tokens - 1)) * xs_ld;
      }
      float tot[kRB][kTB][4];
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
        for (int tb = 0; tb < kTB; ++tb)
#pragma unroll
          for (int i = 0; i < 4; ++i) tot[rb][tb][i] = 0.f;

      for (int span_i = 0; span_i < spans; ++span_i) {
        if (spans > 1 || round == 0) {
          __syncthreads();  // the last readers of the previous activations are done
          marked = __syncthreads_or(load_x(win_base, win_n, span_i));
        }
        if (!active) continue;
        int begin, left;
        chunks_of(span_i, begin, left);
        if (!fetched) {
          open_scales(here, span_i);
          fetch_scales(std::integral_constant<int, 0>{});
        }
        fetched = false;
        const uint8_t* x_at[kTB];
        const float* xs_at[kTB][2];
#pragma unroll
        for (int tb = 0; tb < kTB; ++tb) {
          x_at[tb] = x_lane[tb] + begin * 256;
          xs_at[tb][0] = xs_lane[tb][0] + begin * (kGpc + 1);
          xs_at[tb][1] = xs_lane[tb][1] + begin * (kGpc + 1);
        }
        uint32_t s_cur[2 * kRB][2], z_cur[2 * kRB];
        auto chunk = [&](auto slot_c) {  // the products of chunk kSlot of four
          constexpr int kSlot = decltype(slot_c)::value;
          cp_async_wait<kStages - 2>();
          if (kGpc > 1) __syncwarp();  // with one group in a chunk a lane reads what it has fetched itself
          if (kSlot >= left) {
            load_chunk(std::integral_constant<int, (kSlot + 3) % kStages>{});
            return;
          }
          uint32_t w[2 * kRB][4];
          auto read_row = [&](auto row_c) {
            constexpr int i = decltype(row_c)::value, kAt = kSlot * S::kStage + i * 512;
            if constexpr (kGpc == 1) {
              const uint4 v = lds128<kAt>(fifo_lane + (t ^ swap) * 16);
              w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
            } else if constexpr (kGpc == 2) {
              const uint2 u = lds64<kAt>(fifo_lane + ((t >> 1) ^ swap) * 16 + (t & 1) * 8);
              const uint2 v = lds64<kAt>(fifo_lane + ((2 + (t >> 1)) ^ swap) * 16 + (t & 1) * 8);
              w[i][0] = u.x; w[i][1] = u.y; w[i][2] = v.x; w[i][3] = v.y;
            } else {
              w[i][0] = lds32<kAt>(fifo_lane + swap * 16 + t * 4);
              w[i][1] = lds32<kAt>(fifo_lane + (1 ^ swap) * 16 + t * 4);
              w[i][2] = lds32<kAt>(fifo_lane + (2 ^ swap) * 16 + t * 4);
              w[i][3] = lds32<kAt>(fifo_lane + (3 ^ swap) * 16 + t * 4);
            }
          };
          read_row(std::integral_constant<int, 0>{});
          read_row(std::integral_constant<int, 1>{});
          if constexpr (kRB > 1) {
            read_row(std::integral_constant<int, 2 % (2 * kRB)>{});
            read_row(std::integral_constant<int, 3 % (2 * kRB)>{});
          }
          load_chunk(std::integral_constant<int, (kSlot + 3) % kStages>{});  // into the slot that the previous chunk has left
          if (kSlot % kUnit == 0) {
#pragma unroll
            for (int i = 0; i < 2 * kRB; ++i) {
              if (kZero) z_cur[i] = z_next[i];
              s_cur[i][0] = s_next[i][0];
              s_cur[i][1] = s_next[i][1];
            }
            if (left > kSlot + kUnit) fetch_scales(std::integral_constant<int, kSlot + kUnit>{});
          }
          int high[kRB][kTB][4], low[kRB][kTB][4];
          float part[kRB][kTB][4];  // of the chunk, in units of f
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            constexpr int kPer = 4 / kGpc;
            uint4 b[kTB];
#pragma unroll
            for (int tb = 0; tb < kTB; ++tb) b[tb] = *reinterpret_cast<const uint4*>(x_at[tb] + kSlot * 256 + j * 64);
#pragma unroll
            for (int rb = 0; rb < kRB; ++rb) {
              const uint32_t lo = w[2 * rb][j], hi = w[2 * rb + 1][j];  // rows g and g + 8
              const uint32_t a[4] = {lo & 0x0f0f0f0fu, hi & 0x0f0f0f0fu, (lo >> 4) & 0x0f0f0f0fu, (hi >> 4) & 0x0f0f0f0fu};
#pragma unroll
              for (int tb = 0; tb < kTB; ++tb) {
                if (j % kPer == 0) {
                  mma_codes<true>(high[rb][tb], a, b[tb].x, b[tb].y, start);
                  mma_codes<false>(low[rb][tb], a, b[tb].z, b[tb].w, start);
                } else {
                  mma_codes<true>(high[rb][tb], a, b[tb].x, b[tb].y, high[rb][tb]);
                  mma_codes<false>(low[rb][tb], a, b[tb].z, b[tb].w, low[rb][tb]);
                }
              }
            }
            if (j % kPer == kPer - 1) {
              constexpr int kLast = kPer - 1;
              const int q = (j - kLast) / kPer;
              float s[2 * kRB], z[2 * kRB];
#pragma unroll
              for (int i = 0; i < 2 * kRB; ++i) {
                const int at = kSlot % kUnit * kGpc + q;
                const uint32_t v = s_cur[i][at / 2];
                s[i] = __uint_as_float(at & 1 ? v & 0xffff0000u : v << 16);
                // -zero: 0xcb000000 are the bits of -8388608, one less for every unit
                if (kZero) z[i] = __uint_as_float(((z_cur[i] >> (8 * at)) & 15u) | 0xcb000000u) + 8388608.f;
              }
#pragma unroll
              for (int tb = 0; tb < kTB; ++tb)
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                  const float xs = xs_at[tb][o][kSlot * (kGpc + 1) + q];
#pragma unroll
                  for (int i = 0; i < 2 * kRB; ++i) {
                    // 256 times the high sum and the zero point's share meet first, with the low sum's bias taken off: where the
                    // weights cancel, what is left is below 2^24 and every step exact (weights of zero give zero)
                    const float high_sum = fmaf(__int_as_float(high[i >> 1][tb][2 * (i & 1) + o]), 256.f, -257.f * kFloatBias);
                    const float v = fmaf(kZero ? z[i] : -8.f, xs, high_sum) + __int_as_float(low[i >> 1][tb][2 * (i & 1) + o]);
                    float& acc = part[i >> 1][tb][2 * (i & 1) + o];
                    acc = q == 0 ? s[i] * v : fmaf(s[i], v, acc);
                  }
                }
            }
          }
#pragma unroll
          for (int tb = 0; tb < kTB; ++tb)
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const float f = xs_at[tb][o][kSlot * (kGpc + 1) + kGpc];
#pragma unroll
              for (int i = 0; i < 2 * kRB; ++i) {
                float& sum = tot[i >> 1][tb][2 * (i & 1) + o];
                sum = fmaf(f, part[i >> 1][tb][2 * (i & 1) + o], sum);
              }
            }
        };
#pragma unroll 1
        for (; left > 0; left -= kStages) {
          chunk(std::integral_constant<int, 0>{});
          chunk(std::integral_constant<int, 1>{});
          chunk(std::integral_constant<int, 2>{});
          chunk(std::integral_constant<int, 3>{});
#pragma unroll
          for (int tb = 0; tb < kTB; ++tb) {
            x_at[tb] += kStages * 256;
            xs_at[tb][0] += kStages * (kGpc + 1);
            xs_at[tb][1] += kStages * (kGpc + 1);
          }
#pragma unroll
          for (int i = 0; i < 2 * kRB; ++i) s_src[i] += kStages * kGpc;
          z_src += kStages * kGpc;
          gi += kStages * kGpc;
        }
        // What the integers of marked chunks cut off: once more through these chunks, with (x / f - integer) * 2^15 as integers against
        // code - zero. Behind the loop and in as few registers as it can be, because the loop above has none to spare; codes and
        // activations come from the second level cache. A marked chunk costs as much as two to five others: 64 tokens over 128
        // experts, H = 2048, I = 768: 85 us without one, 114 us with two of the 16 chunks of every token, 290 us with all.
        if (__builtin_expect(marked, 0)) {
          int entry0, tokens, window0, unused, chunks;  // found anew rather than kept over the loop
          entries_of(block, entry0, tokens);
          entries_of(block0, window0, unused);
          chunks_of(span_i, begin, chunks);
          const long long first = first_row_of_matrix(block) + first_row(here.r) * step_row + row_lo;
          const float* const f_at = x_sum + (entry0 - window0) * xs_ld + kGpc;
#pragma unroll 1
          for (int c = begin; c < begin + chunks; ++c) {
#pragma unroll
            for (int tb = 0; tb < kTB; ++tb) {
              const int mine = min(tb * 8 + g, tokens - 1);  // token whose activations this lane brings
              const uint32_t f_mine = __float_as_uint(f_at[mine * xs_ld + c * (kGpc + 1)]);
              if (!__any_sync(0xffffffffu, f_mine & kMark)) continue;
              const float to_int = __uint_as_float((254u << 23) - (f_mine & ~kMark));
              const int c0 = span_i * p.span + c * kChunk;
              const X* const x_at = static_cast<const X*>(p.x) + source_row(entry0 + mine) * p.x_ld;
#pragma unroll 1
              for (int q = 0; q < kGpc; ++q) {
                const int group = c0 / (kChunk / kGpc) + q;
                if (group >= groups) continue;
                int high[kRB][4] = {}, low[kRB][4] = {};
#pragma unroll 1
                for (int j = q * (4 / kGpc); j < (q + 1) * (4 / kGpc); ++j) {
                  const int col = c0 + col_of<kGpc>(j, t);
                  const bool in = col < p.K;
                  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                  if (in && (f_mine & kMark)) load_x8(x_at + col, x);
                  uint32_t v[8];
#pragma unroll
                  for (int k = 0; k < 8; ++k) {
                    const float cut = x[k] * to_int - (int_of<kMode == kDown>(x[k], to_int) - kFloatBias);  // exact, -1/2 to 1
                    v[k] = __float_as_uint(fminf(cut * 32768.f, 32767.f) + kFloatBias);
                  }
                  const uint4 b = pack_ints(v);
#pragma unroll
                  for (int rb = 0; rb < kRB; ++rb) {
                    uint32_t w[2], z[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                      w[h] = in ? *reinterpret_cast<const uint32_t*>(p.w.q + first * row_bytes + (col >> 1) + q_off[2 * rb + h]) : 0u;
                      z[h] = (kZero ? p.w.zero[first * groups + group + s_off[2 * rb + h]] & 15u : 8u) * 0x01010101u;
                    }
                    const uint32_t a[4] = {__vsub4(w[0] & 0x0f0f0f0fu, z[0]), __vsub4(w[1] & 0x0f0f0f0fu, z[1]),
                                           __vsub4((w[0] >> 4) & 0x0f0f0f0fu, z[0]), __vsub4((w[1] >> 4) & 0x0f0f0f0fu, z[1])};
                    mma_weights<true>(high[rb], a, b.x, b.y);
                    mma_weights<false>(low[rb], a, b.z, b.w);
                  }
                }
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                  const uint32_t f = __float_as_uint(f_at[min(tb * 8 + 2 * t + o, tokens - 1) * xs_ld + c * (kGpc + 1)]);
                  const float unit = __uint_as_float(f & ~kMark) * 0x1p-15f;
#pragma unroll
                  for (int i = 0; i < 2 * kRB; ++i) {
                    const float s = __bfloat162float(p.w.scale[first * groups + group + s_off[i]]);
                    const int r = 2 * (i & 1) + o;
                    float& sum = tot[i >> 1][tb][r];
                    sum = fmaf(unit * s, static_cast<float>(high[i >> 1][r] * 256 + low[i >> 1][r]), sum);
                  }
                }
              }
            }
          }
        }
      }

      if (active && at.tile < win_last) {
        open_scales(at, 0);
        fetch_scales(std::integral_constant<int, 0>{});
        fetched = true;
      }

      // -------------------------------------------------------------- the worker's warps meet
      if (wk > 1) {
        float* mine = red + warp * (kRB * kTB * 128) + lane;
        if (kw != 0 && active) {
#pragma unroll
          for (int i = 0; i < kRB * kTB * 4; ++i) mine[i * 32] = tot[i / (4 * kTB)][i / 4 % kTB][i & 3];
        }
        __syncwarp();
        asm volatile("bar.sync %0, %1;" ::"r"(1 + worker), "r"(32 * wk) : "memory");
        if (kw == 0 && active) {
          for (int k = 1; k < wk; ++k)
#pragma unroll
            for (int i = 0; i < kRB * kTB * 4; ++i) tot[i / (4 * kTB)][i / 4 % kTB][i & 3] += mine[k * (kRB * kTB * 128) + i * 32];
        }
        __syncwarp();
        asm volatile("bar.sync %0, %1;" ::"r"(1 + worker), "r"(32 * wk) : "memory");
      }
      if (kw != 0 || !active) continue;
      // -------------------------------------------------------------- epilogue: lane holds rows g, g + 8 of tokens 2t, 2t + 1
#pragma unroll
      for (int tb = 0; tb < kTB; ++tb)
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const int n = tb * 8 + 2 * t + o;
          if (n >= n_tokens) continue;
          if (kMode == kGateUp) {
            const int I = p.rows >> 1;
            float* dst = static_cast<float*>(p.out) + static_cast<long long>(lists.slots[base + n]) * I;
#pragma unroll
            for (int rb = 0; rb < kRB; ++rb) {
              const int j = row0 + rb * 8 + g;
              float gate = tot[rb][tb][o], up = tot[rb][tb][2 + o];
              if (p.w.bias != nullptr) {
                gate += __bfloat162float(p.w.bias[mat + j * step_row]);
                up += __bfloat162float(p.w.bias[mat + j * step_row + step_half]);
              }
              dst[j] = w4_act(gate, up, p.activation);
            }
          } else {
            const int s = kMode == kDense ? base + n : lists.slots[base + n];
            const float scale = kMode == kDense ? 1.f : p.topk_w[s];
#pragma unroll
            for (int i = 0; i < 2 * kRB; ++i) {
              const int row = row0 + i * 8 + g;
              if (row >= p.rows) continue;
              float y = tot[i >> 1][tb][2 * (i & 1) + o];
              if (p.w.bias != nullptr) y += __bfloat162float(p.w.bias[mat + row]);
              const long long at = static_cast<long long>(s) * p.rows + row;
              if (kMode == kDense) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
              else static_cast<float*>(p.out)[at] = y * scale;
            }
          }
        }
    }
    block0 = block1;
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

// Token blocks that evenly spread slots come to; a guess, for the split of the work only.
int expected_blocks(int slots, int E) {
  const double active = E * (1.0 - std::exp(-static_cast<double>(slots) / E));
  const double full = (slots - 4.0 * active) / 8.0;
  const int b = static_cast<int>(active + (full > 0 ? full : 0.0));
  return b < 1 ? 1 : b;
}

// How a launch is split, and a guess of its time in cycles; the shape with the least is taken. What it weighs: a chunk of a
// warp takes about 850 cycles for 16 rows with all warps at work (1450 for 32), more with small groups and two token blocks, a
// tile's end 2200, a window is a whole number of rounds and, where others follow, waits for its slowest worker, and activations
// come at 64 bytes a cycle behind a latency of 1500. It does not know what a shape spills and is off by tens of percent where shapes
// lie close. Measured with the row blocks forced (calls, us; what is taken first): N = 131075, K = 2048, groups of 32, M = 5 two 42.0, one
// 46.3; 64 tokens over 128 experts (H = 2048, I = 768) two 85.2, one 83; 93 tokens (H = 4096, I = 1536, groups of 64 with zero points) one in
// gate_up and two in down 357, two in both 375, one in both 356; M = 16, N = 4096, K = 8192, groups of 64 with zero points two
// 22.1, one 17.1: there it takes the slower.
struct W4Split {
  int span, cap, wk_log2, ctas;
  double cost;
};

template <int kMode, int kRB, int kTB, int kGpc>
W4Split split_of(const W4Params& p, long long blocks) {
  using S = W4Shape<kMode, kRB, kTB>;
  constexpr int kRoom = kMaxSmem - S::kFixed;
  static_assert(kRoom / S::x_row_bytes(4 * kChunk, kGpc) >= S::kTokens);
  W4Split r{};
  const int chunks = (p.K + kChunk - 1) / kChunk;
  int spans = 1;  // as few equal spans as leave room for a block's tokens
  const int entries = std::max(1, std::min(p.m, kMode == kDense ? p.m : kListSlots));
  while (kRoom / S::x_row_bytes((chunks + spans - 1) / spans * kChunk, kGpc) < std::min(S::kTokens, entries)) ++spans;
  const int span_chunks = (chunks + spans - 1) / spans;
  r.span = span_chunks * kChunk;
  r.cap = std::min(kRoom / S::x_row_bytes(r.span, kGpc), entries);
  const int row_tiles = ((kMode == kGateUp ? p.rows / 2 : p.rows) + S::kRows / (kMode == kGateUp ? 2 : 1) - 1) / (S::kRows / (kMode == kGateUp ? 2 : 1));
  const long long tiles = blocks * row_tiles;
  const int sms = device_sm_count();
  r.ctas = static_cast<int>(tiles < sms ? tiles : sms);
  const double per_cta = static_cast<double>(tiles) / r.ctas;
  const double tokens = std::max(1.0, std::min<double>(S::kTokens, static_cast<double>(entries) / blocks));  // of a block
  const double windows = spans > 1 ? 1 + per_cta / row_tiles : std::ceil(std::min<double>(entries, (per_cta / row_tiles + 1) * tokens) / r.cap);
  const double rows_a_window = std::min<double>(r.cap, std::max<double>(entries < S::kTokens ? entries : S::kTokens, static_cast<double>(entries) / r.ctas));
  const int last_chunks = chunks - (chunks - 1) / span_chunks * span_chunks;  // every warp has a step in every span
  r.cost = -1;
  for (int lg = 0; lg <= 4 && (1 << lg) <= std::min(last_chunks, span_chunks); ++lg) {
    const double rounds = windows * (std::ceil(per_cta / windows / (kWarps >> lg)) + 1.5 * std::min(1.0, windows - 1));
    const double steps = (spans - 1.0) * ((span_chunks + (1 << lg) - 1) >> lg) + ((last_chunks + (1 << lg) - 1) >> lg);
    const double x_loads = spans > 1 ? rounds * spans : windows;
    const double cost = rounds * (steps * (250 + 600 * kRB) * (1 + 0.2 * (kGpc - 1)) * (1 + 0.5 * (kTB - 1)) + 2200) +
                        x_loads * (1500 + rows_a_window * (kMode == kDown ? 4 : 2) * r.span / 64.0);
    if (r.cost < 0 || cost < r.cost) {
      r.cost = cost;
      r.wk_log2 = lg;
    }
  }
  return r;
}

template <int kMode, int kRB, int kTB, int kGpc, bool kZero>
cudaError_t launch_split(W4Params p, const W4Split& s, cudaStream_t stream) {
  using S = W4Shape<kMode, kRB, kTB>;
  auto kernel = w4_mma_kernel<kMode, kRB, kTB, kGpc, kZero>;
  static std::atomic<unsigned long long> done{0};  // devices on which the kernel may take all shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  p.row_tiles = ((kMode == kGateUp ? p.rows / 2 : p.rows) + S::kRows / (kMode == kGateUp ? 2 : 1) - 1) / (S::kRows / (kMode == kGateUp ? 2 : 1));
  p.span = s.span;
  p.cap = s.cap;
  p.wk_log2 = s.wk_log2;
  p.whole = p.K % kChunk == 0;
  const uintptr_t s_at = reinterpret_cast<uintptr_t>(p.w.scale), z_at = reinterpret_cast<uintptr_t>(p.w.zero);
  const int groups = p.K / p.w.group;
  p.scale_words = groups % 4 == 0 && s_at % 8 == 0 && z_at % 4 == 0 ? 2 : (groups % 2 == 0 && s_at % 4 == 0 && z_at % 2 == 0 ? 1 : 0);
  return launch_pdl(kernel, dim3(s.ctas), dim3(kThreads), S::kFixed + s.cap * S::x_row_bytes(s.span, kGpc), stream, p);
}

template <int kMode, int kTB, int kGpc>
double least_cost(const W4Params& p, long long blocks) {
  return std::min(split_of<kMode, 1, kTB, kGpc>(p, blocks).cost, split_of<kMode, 2, kTB, kGpc>(p, blocks).cost);
}

template <int kMode, int kTB, int kGpc>
cudaError_t launch_groups(W4Params p, long long blocks, int x_rows, void* xq, cudaStream_t stream) {
  // More than eight tokens: blocks of sixteen, unless a long K leaves no room for so many activations and the weights
  // are better read once more (M = 16, N = 4096, K = 8192: 26 us in one block of two halves of K, 24 us in two blocks).
  if constexpr (kTB == 2) {
    const long long more = (p.m + 7) / 8;
    if (least_cost<kMode, 1, kGpc>(p, more) < least_cost<kMode, 2, kGpc>(p, blocks)) return launch_groups<kMode, 1, kGpc>(p, more, x_rows, xq, stream);
  }
  if (xq != nullptr) {
    const long long chunks = static_cast<long long>(x_rows) * ((p.K + kChunk - 1) / kChunk);
    p.xq = static_cast<uint8_t*>(xq);
    p.xm = reinterpret_cast<float*>(static_cast<uint8_t*>(xq) + chunks * 256);
    const cudaError_t e = launch_pdl(quant_x_kernel<kGpc>, dim3(static_cast<unsigned>((chunks + 15) / 16)), dim3(256), 0, stream,
                                     static_cast<uint8_t*>(xq), const_cast<float*>(p.xm), static_cast<const __nv_bfloat16*>(p.x),
                                     p.x_ld, x_rows, p.K);
    if (e != cudaSuccess) return e;
    count_launches(1);
  }
  const W4Split one = split_of<kMode, 1, kTB, kGpc>(p, blocks), two = split_of<kMode, 2, kTB, kGpc>(p, blocks);
  if (one.cost < two.cost)
    return p.w.zero != nullptr ? launch_split<kMode, 1, kTB, kGpc, true>(p, one, stream) : launch_split<kMode, 1, kTB, kGpc, false>(p, one, stream);
  return p.w.zero != nullptr ? launch_split<kMode, 2, kTB, kGpc, true>(p, two, stream) : launch_split<kMode, 2, kTB, kGpc, false>(p, two, stream);
}

// x_rows, xq: rows of bf16 activations and room for their integers, or null
template <int kMode, int kTB>
cudaError_t launch_mode(const W4Params& p, long long blocks, int x_rows, void* xq, cudaStream_t stream) {
  if (p.w.group == 128) return launch_groups<kMode, kTB, 1>(p, blocks, x_rows, xq, stream);
  if (p.w.group == 64) return launch_groups<kMode, kTB, 2>(p, blocks, x_rows, xq, stream);
  return launch_groups<kMode, kTB, 4>(p, blocks, x_rows, xq, stream);
}

// Room for the integers of `rows` activations of K columns, 0 where the CTAs make them themselves: up to kPreparedChunks chunks
// of 128 columns, two turns of a CTA's warps, for which a launch in front takes longer than it saves (N = 4096: 80 chunks 6.8 us
// prepared and 7.2 without, 512 chunks 11.3 and 14.6; the experts of one token, 16 chunks, 16.9 and 15.9).
size_t prepared_bytes(int rows, int K, int group) {
  const size_t chunks = static_cast<size_t>(rows) * ((K + kChunk - 1) / kChunk);
  return chunks <= kPreparedChunks ? 0 : chunks * (256 + 4 * (kChunk / group + 1));
}

}  // namespace

size_t w4_linear_workspace_bytes(int M, int K, int group) { return prepared_bytes(M, K, group); }

int launch_w4_linear(__nv_bfloat16* out, const __nv_bfloat16* x, long long x_ld, const W4Matrix& w, int M, int N, int K,
                     void* workspace, cudaStream_t stream) {
  if (M == 0) return kStatusOk;
  W4Params p{};
  p.w = w; p.rows = N; p.K = K; p.x = x; p.x_ld = x_ld; p.m = M; p.out = out;
  const int tb = M <= 8 ? 1 : 2;
  const long long blocks = (M + 8 * tb - 1) / (8 * tb);
  if (blocks * ((N + 15) / 16) > 0x3fffffffll || K > 1 << 24) return set_error(kStatusInvalidArgument, "w4_linear: M x N or K too large");
  void* xq = prepared_bytes(M, K, w.group) > 0 ? workspace : nullptr;
  const cudaError_t e = tb == 1 ? launch_mode<kDense, 1>(p, blocks, M, xq, stream) : launch_mode<kDense, 2>(p, blocks, M, xq, stream);
  if (int st = check_cuda(e, "w4_linear launch")) return st;
  count_launches(1);
  return check_launch("w4_linear");
}

namespace {
size_t w4_aligned(size_t v) { return (v + 255) / 256 * 256; }
}  // namespace

size_t w4_experts_workspace_bytes(int T, int top_k, int H, int I) {
  const int piece = top_k < kListSlots ? kListSlots / top_k : 1;
  const int tt = T < 1 ? 1 : (T < piece ? T : piece);
  const size_t slots = static_cast<size_t>(tt) * top_k;
  return w4_aligned(slots * 4 * I) + w4_aligned(slots * 4 * H) + prepared_bytes(tt, H, 32);
}

int launch_w4_experts(__nv_bfloat16* out, const __nv_bfloat16* x, const W4Matrix& w13, const W4Matrix& w2, const float* topk_w,
                      const int* topk_ids, int T, int E, int top_k, int H, int I, int activation, void* workspace,
                      cudaStream_t stream) {
  if (E > kListExperts || top_k > kListSlots)
    return set_error(kStatusInvalidArgument, "fused_experts_w4: at most %d experts and %d slots a token", kListExperts, kListSlots);
  if (static_cast<long long>(I) * H >= 1ll << 32) return set_error(kStatusInvalidArgument, "fused_experts_w4: an expert's matrix is too large (H=%d I=%d)", H, I);
  const int piece = kListSlots / top_k;  // tokens whose slots fit the lists in shared memory
  for (int t0 = 0; t0 < T; t0 += piece) {
    const int tt = T - t0 < piece ? T - t0 : piece;
    const int slots = tt * top_k;
    const int* ids = topk_ids + static_cast<long long>(t0) * top_k;
    uint8_t* at = static_cast<uint8_t*>(workspace);
    float* h = reinterpret_cast<float*>(at);
    float* c3 = reinterpret_cast<float*>(at += w4_aligned(static_cast<size_t>(slots) * 4 * I));
    void* xq = prepared_bytes(tt, H, w13.group) > 0 ? at + w4_aligned(static_cast<size_t>(slots) * 4 * H) : nullptr;
    const int blocks = expected_blocks(slots, E);
    W4Params p{};
    p.w = w13; p.rows = 2 * I; p.K = H; p.x = x + static_cast<long long>(t0) * H; p.x_ld = H; p.m = slots; p.ids = ids; p.top_k = top_k;
    p.E = E; p.activation = activation; p.out = h;
    if (int st = check_cuda(launch_mode<kGateUp, 1>(p, blocks, tt, xq, stream), "w4 gate_up launch")) return st;
    p.w = w2; p.rows = H; p.K = I; p.x = h; p.x_ld = I; p.topk_w = topk_w + static_cast<long long>(t0) * top_k; p.out = c3;
    if (int st = check_cuda(launch_mode<kDown, 1>(p, blocks, 0, nullptr, stream), "w4 down launch")) return st;
    if (int st = check_cuda(launch_pdl(w4_sum_kernel, dim3((H / 4 + 255) / 256, tt), dim3(256), 0, stream,
                                       out + static_cast<long long>(t0) * H, c3, ids, E, top_k, H), "w4 sum launch"))
      return st;
    count_launches(3);
  }
  return check_launch("w4_experts");
}

}  // namespace moe_b200
