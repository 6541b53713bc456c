// Block-scaled FP8 (E4M3) products for checkpoints that hold their weights in
// 8 bits: activations with one fp32 scale per 128 columns of a row, weights
// with one fp32 scale per 128 x 128 block.
//
//   quantize   a = max(|x| of the block, 1e-12); q = e4m3(x * f32(448 / a)),
//              scale f32(a / 448): the product and both quotients rounded once
//   product    y[m, n] = sum_b sx[m, b] * sw[n / 128, b] * d_b,
//              d_b = sum over the 128 columns of block b of qx[m, c] * qw[n, c]
//   SwiGLU     h = g / (1 + exp(-g)) * u of the gate and up columns, in fp32,
//              quantized as above without a rounding in between
//
// The tensor cores give d_b (the products of E4M3 values are exact in fp32,
// the sum is held in fp32); the scales are arbitrary fp32 numbers, which the
// block-scaled MMA kinds cannot take (they take powers of two), so every
// d_b leaves tensor memory once and is added into registers with one FMA.
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace praxis {

constexpr int kFp8Block = 128;          // columns per activation scale, rows and columns per weight scale
constexpr float kE4m3Max = 448.0f;
constexpr float kFp8MinAmax = 1.0e-12f;

// Four floats -> four E4M3 codes (round to nearest even; NaN stays NaN).
__device__ __forceinline__ uint32_t cvt_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// ---------------------------------------------------------------------------
// Rows of the routed slots
// ---------------------------------------------------------------------------
// The experts' segments of rows, each padded to whole 128-row tiles, and a row
// of its expert's segment for every routed slot p: pcsr[e] + inverse[p] - csr[e]
// with csr = 0. Which row a slot gets within the segment depends on the order
// of the CTAs; nothing else does, since every row is computed by itself and
// read back through inverse. So one counting pass is enough (the dispatch of
// the NVFP4 path keeps the slots' order: count, scan, scatter; 1024 slots of 32
// experts 11 us there, 3.7 here, 65536 slots of 64 experts 32 and 14). A CTA takes
// 4096 slots; with several of them each claims its share of every segment from
// the counters, and the last one lays out the segments and their tiles.
constexpr int kFp8SlotThreads = 1024;  // and the most experts
constexpr int kFp8SlotItems = 4;

__global__ void __launch_bounds__(kFp8SlotThreads) fp8_slots_kernel(
    const int64_t* top_idx, int64_t positions, int experts, uint32_t* counters, int64_t* __restrict__ inverse,
    int32_t* __restrict__ csr, int32_t* __restrict__ pcsr, TileEntry* __restrict__ tiles, int max_tiles,
    int32_t* __restrict__ num_tiles) {
  pdl_wait();  // the previous kernel of the stream has completed
  pdl_trigger();
  __shared__ uint32_t s_count[kFp8SlotThreads];  // slots per expert, then where this CTA's begin
  __shared__ uint32_t s_warp[32];
  __shared__ bool s_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  s_count[tid] = 0;
  const int64_t p0 = (int64_t)blockIdx.x * (kFp8SlotThreads * kFp8SlotItems) + tid;
  int e[kFp8SlotItems];
  uint32_t rank[kFp8SlotItems];
#pragma unroll
  for (int i = 0; i < kFp8SlotItems; ++i) {
    const int64_t p = p0 + i * kFp8SlotThreads;
    e[i] = p < positions ? checked_expert(top_idx[p], experts) : -1;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kFp8SlotItems; ++i) {
    const uint32_t peers = __match_any_sync(0xffffffffu, e[i]);
    const int leader = __ffs(peers) - 1;
    uint32_t before = 0;
    if (lane == leader && e[i] >= 0) before = atomicAdd(&s_count[e[i]], (uint32_t)__popc(peers));
    rank[i] = __shfl_sync(0xffffffffu, before, leader) + __popc(peers & ((1u << lane) - 1u));
  }
  __syncthreads();
  const bool alone = gridDim.x == 1;
  uint32_t count = s_count[tid], begin = 0;
  if (!alone && count > 0) begin = atomicAdd(&counters[tid], count);
  __syncthreads();
  s_count[tid] = begin;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kFp8SlotItems; ++i)
    if (e[i] >= 0) inverse[p0 + i * kFp8SlotThreads] = s_count[e[i]] + rank[i];
  if (!alone) {
    __threadfence();
    __syncthreads();
    if (tid == 0) s_last = atomicAdd(&counters[experts], 1u) == gridDim.x - 1;
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    count = tid < experts ? __ldcg(&counters[tid]) : 0u;
  }
  // segments and tiles: an exclusive scan of the experts' tiles
  const uint32_t mine = (count + kTileRows - 1) / kTileRows;
  uint32_t sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) s_warp[warp] = sum;
  __syncthreads();
  uint32_t base = 0;
  for (int w = 0; w < warp; ++w) base += s_warp[w];
  const uint32_t end = base + sum, at = end - mine;
  if (tid < experts) {
    csr[tid] = 0;
    pcsr[tid] = (int32_t)at * kTileRows;
    if (tid == experts - 1) {
      csr[experts] = 0;
      pcsr[experts] = (int32_t)end * kTileRows;
      num_tiles[0] = (int32_t)end;
    }
    for (uint32_t j = 0; j < mine && at + j < (uint32_t)max_tiles; ++j) {
      TileEntry t;
      t.expert = tid;
      t.row0 = (int32_t)(at + j) * kTileRows;
      t.valid = (int32_t)min(count - j * kTileRows, (uint32_t)kTileRows);
      t.pad = 0;
      tiles[at + j] = t;
    }
  }
}

// ---------------------------------------------------------------------------
// Activation quantization
// ---------------------------------------------------------------------------
// A warp takes 1024 columns of a row, four 16-byte loads per lane in flight;
// sixteen lanes hold one block of 128 columns, whose largest magnitude is four
// shuffles. Scales are stored block-major, scale[b * scale_ld + row]: the GEMM
// epilogue reads one block's scales of 32 consecutive rows at once. With
// `top_idx` the row goes to the rows of the token's routed slots, quantized once.
// Six CTAs per SM hold the kernel at 40 registers (11 of them spilled).
struct Fp8Rows {
  const int64_t* top_idx;  // [rows, top_k]; nullptr: row r goes to row r
  const int64_t* inverse;
  const int32_t* csr;
  const int32_t* pcsr;
  int32_t top_k;  // 1 without top_idx
  int32_t experts;
};

constexpr Fp8Rows kFp8SameRows = {nullptr, nullptr, nullptr, nullptr, 1, 0};

constexpr int kFp8QuantWarps = 8;
constexpr int kFp8QuantCols = 1024;  // per warp

__global__ void __launch_bounds__(32 * kFp8QuantWarps, 6) fp8_quantize_kernel(
    const uint16_t* x, int64_t rows, int cols, int64_t ldx, Fp8Rows to, uint8_t* __restrict__ q,
    float* __restrict__ scale, int64_t scale_ld) {
  // routed, the previous kernel is fp8_slots_kernel, which writes no row of x
  if (to.top_idx == nullptr) {
    pdl_wait();
    pdl_trigger();
  }
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kFp8QuantWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int col0 = blockIdx.y * kFp8QuantCols + lane * 8;
  uint4 v[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    v[u] = make_uint4(0u, 0u, 0u, 0u);
    if (col0 + 256 * u < cols) v[u] = ldg_stream(reinterpret_cast<const uint4*>(x + row * ldx + col0 + 256 * u));
  }
  uint2 codes[4];
  float s[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float2 f[4] = {unpack_bf16x2(v[u].x), unpack_bf16x2(v[u].y), unpack_bf16x2(v[u].z), unpack_bf16x2(v[u].w)};
    float a = kFp8MinAmax;
#pragma unroll
    for (int j = 0; j < 4; ++j) a = fmaxf(a, fmaxf(fabsf(f[j].x), fabsf(f[j].y)));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    const float r = div_rn(kE4m3Max, a);
    s[u] = div_rn(a, kE4m3Max);
    codes[u] = make_uint2(cvt_e4m3x4(mul_rn(f[0].x, r), mul_rn(f[0].y, r), mul_rn(f[1].x, r), mul_rn(f[1].y, r)),
                          cvt_e4m3x4(mul_rn(f[2].x, r), mul_rn(f[2].y, r), mul_rn(f[3].x, r), mul_rn(f[3].y, r)));
  }
  int64_t dest = row;
  if (to.top_idx != nullptr) {
    pdl_wait();
    pdl_trigger();
    if (lane < to.top_k) {
      const int64_t p = row * to.top_k + lane;
      const int e = checked_expert(to.top_idx[p], to.experts);
      dest = (int64_t)to.pcsr[e] + to.inverse[p] - to.csr[e];
    }
  }
  for (int j = 0; j < to.top_k; ++j) {
    const int64_t d = (int64_t)__shfl_sync(0xffffffffu, (unsigned long long)dest, j);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int col = col0 + 256 * u;
      if (col < cols) {
        *reinterpret_cast<uint2*>(q + d * cols + col) = codes[u];
        if ((lane & 15) == 0) scale[(int64_t)(col / kFp8Block) * scale_ld + d] = s[u];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Weight packing: w [E, K, N] bf16 (input features first) -> q [E, N, K] E4M3
// and scale [E, ceil(N / 128), ceil(K / 128)], one CTA per 128 x 128 block:
// rows of w are read 256 bytes at a time, the codes are turned in shared
// memory and written 128 bytes per output row.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) fp8_pack_kernel(const uint16_t* __restrict__ w, int64_t k_dim, int64_t n_dim,
                                                       uint8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ uint8_t codes[kFp8Block][kFp8Block + 4];  // [n][k]
  __shared__ float s_max[8];
  const int kb = (int)((k_dim + kFp8Block - 1) / kFp8Block), nb = (int)((n_dim + kFp8Block - 1) / kFp8Block);
  const int b = (int)(blockIdx.x % kb), nblk = (int)(blockIdx.x / kb % nb);
  const int64_t e = blockIdx.x / kb / nb;
  const int64_t k0 = (int64_t)b * kFp8Block, n0 = (int64_t)nblk * kFp8Block;
  const int n = threadIdx.x & 127, kh = threadIdx.x >> 7;
  const uint16_t* src = w + e * k_dim * n_dim + k0 * n_dim + n0 + n;
  float a = kFp8MinAmax;
  if (n0 + n < n_dim)
    for (int k = kh; k < kFp8Block && k0 + k < k_dim; k += 2) a = fmaxf(a, fabsf(bf16_to_f32(src[(int64_t)k * n_dim])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = a;
  __syncthreads();
  a = s_max[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) a = fmaxf(a, s_max[i]);
  const float r = div_rn(kE4m3Max, a);
  if (n0 + n < n_dim)
    for (int k = kh; k < kFp8Block && k0 + k < k_dim; k += 2)
      codes[n][k] = (uint8_t)cvt_e4m3x4(mul_rn(bf16_to_f32(src[(int64_t)k * n_dim]), r), 0.0f, 0.0f, 0.0f);
  __syncthreads();
  for (int i = threadIdx.x; i < kFp8Block * 32; i += 256) {
    const int row = i >> 5, c = (i & 31) * 4;
    if (n0 + row < n_dim && k0 + c < k_dim)
      *reinterpret_cast<uint32_t*>(q + (e * n_dim + n0 + row) * k_dim + k0 + c) =
          *reinterpret_cast<const uint32_t*>(&codes[row][c]);
  }
  if (threadIdx.x == 0) scale[(e * nb + nblk) * kb + b] = div_rn(a, kE4m3Max);
}

// ---------------------------------------------------------------------------
// GEMM on tcgen05: 128 x 256 of the output per CTA (or 128 x 64, see below), one
// CTA per SM, persistent over the output tiles.
//
// warp 0      TMA producer: per k-block of 128 columns the A rows and the
//             weight rows (128-byte swizzle)
// warp 1      MMA issuer: per k-block one group of 4 MMAs into one of the
//             tensor-memory buffers (two of 256 columns, four of 64)
// warp 2      relay: waits for a group's commit and meets the epilogue warps at
//             a named barrier
// warp 3      relay: waits for a k-block's operands and meets the issuer and the
//             epilogue (which has read the buffer) at a named barrier
// warps 4..   epilogue: two warps per lane quadrant (one for 64 columns). Per
//             k-block a thread reads its row's columns 16 at a time, the next
//             load in flight while it adds the last, times sx * sw, to its
//             registers, and gives the buffer back as soon as it is read.
//
// A buffer's round trip (products 512 clocks, commit, sums 260, release, next
// issue) decides the rate, and what the warps wait on decides the round trip:
// with operands at rest a k-block takes 620 clocks where the epilogue and the
// issuer meet at named barriers, 805 where every epilogue warp waits on the
// commit's mbarrier and arrives on another (680 and 900 with 16 epilogue warps
// of 64 columns). An mbarrier wait or a second commit in the issuer's loop
// delays its next MMA by 100 to 200 clocks, hence the relays and one commit per
// k-block, which frees the stage and announces the sums at once.
//
// Bound: 128 x 256 x 128 products are 512 clocks of the tensor core, its operand
// reads and the TMA writes of a k-block 768 clocks of shared memory, the FMAs of
// the block sums 256 clocks of the fp32 lanes; 880 clocks are reached. CTA pairs
// (cta_group::2, 256 x 256) need 512 clocks of shared memory but two more hops
// across the cluster per buffer: 950 clocks, and 948 against 878 us for 16384
// tokens through 4 of 64 experts (C 2048, F 1536). In a row of calls both hold
// the card at its power limit (990 W, 1.6 GHz).
//
// 64-column tiles (four buffers, one epilogue warp per quadrant) are for
// outputs whose 256-column tiles leave most SMs idle.
// ---------------------------------------------------------------------------
enum Fp8Mode : int { FP8_PLAIN = 0, FP8_SWIGLU = 1 };

struct Fp8GemmParams {
  CUtensorMap tmap_a;    // activation codes [rows, K], boxes of 128 rows
  CUtensorMap tmap_a32;  // the same, boxes of 32 rows (FEW)
  CUtensorMap tmap_b;    // weight codes [E * N, K], boxes of 128 rows
  CUtensorMap tmap_out;  // bf16 output [rows, N], boxes of 32 rows x 64 columns (tma_out)
  const float* xs;       // activation scales, [K blocks][xs_ld]
  int64_t xs_ld;
  const float* ws;       // weight scales [E][N blocks][K blocks]
  const TileEntry* tiles;    // grouped: table of 128-row tiles; nullptr: dense rows
  const int32_t* num_tiles;
  int64_t rows;          // rows of the activations and of the output
  int32_t N;             // weight rows per expert (2F for FP8_SWIGLU)
  int32_t K;
  int32_t experts;
  uint16_t* out;         // FP8_PLAIN: [rows, N]
  int32_t tma_out;       // N % 8 == 0 and a 16-byte aligned output
  uint8_t* hq;           // FP8_SWIGLU: hidden codes [rows, N / 2]
  float* hs;             // FP8_SWIGLU: hidden scales, [N / 256][hs_ld]
  int64_t hs_ld;
};

// Named barriers (the last two kinds one per tensor-memory buffer).
constexpr uint32_t kFp8BarMax = 1;   // SwiGLU row maxima: the epilogue warps
constexpr uint32_t kFp8BarSums = 2;  // a buffer holds its block sums: relay -> epilogue
constexpr uint32_t kFp8BarGo = 6;    // a buffer is read and its next operands are there: epilogue, relay -> issuer

template <int BN>
struct Fp8Shape {
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BN * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 64 ? 8 : 4;
  static constexpr int BUFS = BN == 64 ? 4 : 2;  // tensor-memory buffers of BN columns
  static constexpr int OUT_BOX = 4096;           // 32 rows x 64 bf16 per epilogue warp
  static constexpr int EPI_WARPS = BN == 64 ? 4 : 8;
  static constexpr int COLS = 4 * BN / EPI_WARPS;  // columns per epilogue thread
  // Registers: 12 warps launch with 168 each (64512 in all); the first four
  // give some back, and the epilogue's 128 sums and two 16-column loads in
  // flight fit (ptxas spills 60 bytes of the plain instance's other values, 20 of
  // the SwiGLU one's; of those with few rows 104 and none). 8 warps (BN = 64)
  // have enough as they are.
  static constexpr int EPI_WARP0 = 4;
  static constexpr int THREADS = 32 * (EPI_WARP0 + EPI_WARPS);
  static constexpr bool SPLIT_REGS = EPI_WARPS == 8;
  static constexpr int LAUNCH_REGS = 168, FRONT_REGS = 40, EPI_REGS = 232;
  static_assert(!SPLIT_REGS ||
                    32 * EPI_WARP0 * FRONT_REGS + 32 * EPI_WARPS * EPI_REGS <= THREADS * LAUNCH_REGS,
                "register split");
  static constexpr size_t SMEM_BYTES = 1024 + (size_t)STAGES * STAGE_BYTES + EPI_WARPS * OUT_BOX + 256;
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
  static_assert(8 * (2 * STAGES + 1) <= 256 && BUFS <= 4, "barriers");
};

// E4M3 x E4M3 -> F32 (kind::f8f6f4), K-major operands, K = 32 per MMA.
__host__ __device__ constexpr uint32_t idesc_e4m3(uint32_t m, uint32_t n) {
  return (1u << 4)            // D format: F32
         | ((n >> 3) << 17)   // N / 8 (A and B format 0: E4M3)
         | ((m >> 4) << 24);  // M / 16
}

// The high word of a descriptor is the same for every operand here; the low
// word (the address) moves by 2 per 32 bytes.
template <int ACCUMULATE>
__device__ __forceinline__ void tc_mma_e4m3(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi,
                                            uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "n"(ACCUMULATE)
      : "memory");
}

// acc[0..15] += f * (the 16 columns in r). The statements are volatile, so they
// stay behind the wait for the loads of r.
__device__ __forceinline__ void fp8_add_block(float* acc, const uint32_t (&r)[16], float f) {
#pragma unroll
  for (int j = 0; j < 16; ++j)
    asm volatile("fma.rn.f32 %0, %1, %2, %0;" : "+f"(acc[j]) : "f"(__uint_as_float(r[j])), "f"(f));
}

// mbar_wait (common.cuh) for waits on the path of every MMA: each try may
// suspend the warp for up to 100 us of its own (polling warps take issue slots
// and shared-memory cycles from the others), and the clock is read every 64
// tries. An error that another kernel has left is no reason to give up: only
// the limit ends the wait.
__device__ __forceinline__ bool fp8_wait(uint64_t* bar, uint32_t parity, unsigned int code) {
  constexpr uint64_t limit_ns = 2000000000ull;
  const uint32_t addr = smem_u32(bar);
  uint64_t start = 0;
  for (uint32_t i = 1;; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity), "r"(100000u)
        : "memory");
    if (done) return true;
    if ((i & 63u) == 0u) {
      const uint64_t now = globaltimer_ns();
      if (start == 0) {
        start = now;
      } else if (now - start > limit_ns) {
        record_error(code);
        return false;
      }
    }
  }
}

template <int REGS>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// Row tile m of the launch: dense rows, or the table's entry.
__device__ __forceinline__ TileEntry fp8_tile(const Fp8GemmParams& p, int m) {
  if (p.tiles != nullptr) {
    return p.tiles[m];
  }
  TileEntry t;
  t.expert = 0;
  t.row0 = m * kTileRows;
  t.valid = (int32_t)min((int64_t)kTileRows, p.rows - t.row0);
  t.pad = 0;
  return t;
}

// A tile of up to 32 rows, loaded into all four quarters of the A operand: each
// quadrant of tensor memory holds the sums of all its rows, and the warps of a
// quadrant take a quarter of the columns instead of a quarter of the rows.
constexpr int kFp8FewRows = 32;

// g / (1 + exp(-g)) * u for two columns, in place of the gates. With
// s = exp(-|g|), which lies in 0..1 and never overflows, the sigmoid is
// 1 / (1 + s) for a gate above 0 and s / (1 + s) below, and one reciprocal
// serves both columns: 1 / (d0 d1) times the other denominator, 1 <= d <= 2.
// Relative error: about 2^-21 of the approximations and products plus |g| 2^-24
// of the rounded exponent (2^-18 for a gate of -40), against the 2^-4 of the
// rounding to E4M3 that follows. exp(-|g|) below 2^-126 is 0: a gate below
// -87.3 gives 0 in place of at most 1.1e-36 |u|. As the quotient has it, NaN
// stays NaN and a gate of -inf gives NaN.
__device__ __forceinline__ void swiglu_pair_f32(float& g0, float& g1, float u0, float u1) {
  float s0, s1, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(s0) : "f"(-1.4426950408889634f * fabsf(g0)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(s1) : "f"(-1.4426950408889634f * fabsf(g1)));
  const float d0 = 1.0f + s0, d1 = 1.0f + s1;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d0 * d1));
  g0 *= g0 < 0.0f ? s0 : 1.0f;
  g1 *= g1 < 0.0f ? s1 : 1.0f;
  g0 *= r * d1 * u0;
  g1 *= r * d0 * u1;
}

// Tensor-memory column of a thread's chunk c of 16 columns, from its first.
template <int MODE>
__device__ constexpr uint32_t chunk_col(int c) {
  return 16 * c + (MODE == FP8_SWIGLU && c >= 4 ? 64 : 0);
}

template <int BN, int MODE, bool FEW>
__global__ void __launch_bounds__(Fp8Shape<BN>::THREADS, 1)
    fp8_gemm_kernel(const __grid_constant__ Fp8GemmParams p) {
  using S = Fp8Shape<BN>;
  static_assert(!FEW || BN == 256, "the few rows' columns are split for 256");
  static_assert(MODE == FP8_PLAIN || BN == 256, "a SwiGLU tile is one block of 128 hidden columns");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + S::STAGES * S::A_BYTES;
  uint8_t* sOut = sB + S::STAGES * S::B_BYTES;
  float* s_max = reinterpret_cast<float*>(sOut);  // FP8_SWIGLU: row maxima [unit parity][half][row]
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + S::EPI_WARPS * S::OUT_BOX);
  uint64_t* done = full + S::STAGES;  // products of a stage complete: its sums are there, its memory is free
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + S::STAGES);

  const int warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[s], 1);
    }
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.tmap_a);
    tma_prefetch_desc(&p.tmap_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::BUFS * BN);
    tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int F = p.N / 2;
  const int n_tiles = MODE == FP8_SWIGLU ? F / 128 : (p.N + BN - 1) / BN;
  const int num_m =
      p.tiles != nullptr ? p.num_tiles[0] : (int)((p.rows + kTileRows - 1) / kTileRows);
  const int total = num_m * n_tiles;
  const int k_blocks = (p.K + kFp8Block - 1) / kFp8Block;
  const int first = blockIdx.x, step = gridDim.x;
  // k-blocks of this CTA: every role below takes exactly this many turns, on
  // every path, so that the named barriers stay matched (the issuer commits
  // each turn, so the waits for its commits end too)
  const int turns = first < total ? ((total - 1 - first) / step + 1) * k_blocks : 0;

  if (warp < S::EPI_WARP0) {
    if constexpr (S::SPLIT_REGS) regs_down<S::FRONT_REGS>();
    if (warp == 0) {
      // ---------------- TMA producer ----------------
      // one lane per copy: A, the weight rows, of 256 in two copies
      constexpr uint32_t kCopies = BN == 256 ? 3 : 2;
      // (lanes 3..5: the second to fourth copy of up to 32 rows)
      const bool b_lane = lane > 0 && lane < kCopies;
      uint8_t* const dst0 = b_lane ? sB + (lane - 1) * 16384 : sA + (lane == 0 ? 0 : lane - 2) * 4096;
      const uint32_t dst_step = b_lane ? S::B_BYTES : S::A_BYTES;
      const int part = lane == 2 ? 1 : 0;  // weight rows of columns 0..127, 128..255
      const CUtensorMap* map = &p.tmap_b;
      bool a_lane = false;
      auto first_row = [&](int u) {
        const int m = u / n_tiles, n = u - m * n_tiles;
        const TileEntry t = fp8_tile(p, m);
        const bool few = FEW && t.valid <= kFp8FewRows;
        a_lane = lane == 0 || (few && lane >= 3 && lane < 6);
        if (!b_lane) map = few ? &p.tmap_a32 : &p.tmap_a;
        return !b_lane ? t.row0
                       : t.expert * p.N + (MODE == FP8_SWIGLU ? n * 128 + part * F : n * BN + part * 128);
      };
      // The weights and the table were there before the previous kernel began
      // (see run_fp8_gemm): the first stages' weight rows come in while it ends,
      // their A rows after it (64 x 1024 x 1024 in a row of calls 7.8 -> 7.0 us,
      // 256 tokens through 4 of 64 experts 149 -> 145 us).
      const int early = min(turns, S::STAGES);
      int u = first, kb = 0, row = turns > 0 ? first_row(first) : 0;
      auto next = [&] {
        if (++kb == k_blocks) {
          kb = 0;
          u += step;
          if (u < total) row = first_row(u);
        }
      };
#pragma unroll 1
      for (int s = 0; s < early; ++s, next()) {
        if (lane == 0) mbar_arrive_expect_tx(&full[s], S::STAGE_BYTES);
        __syncwarp();
        if (b_lane) tma_load_2d(dst0 + s * dst_step, map, &full[s], kb * 128, row);
      }
      u = first;
      kb = 0;
      row = turns > 0 ? first_row(first) : 0;
      pdl_wait();
      pdl_trigger();
#pragma unroll 1
      for (int s = 0; s < early; ++s, next())
        if (a_lane) tma_load_2d(dst0 + s * dst_step, map, &full[s], kb * 128, row);
      __syncwarp();
      uint32_t stage = early % S::STAGES, phase = early / S::STAGES;
      int issued = early;
      bool ok = true;
      for (; u < total && ok; u += step, kb = 0) {
        row = first_row(u);
        for (; kb < k_blocks; ++kb) {
          ok = fp8_wait(&done[stage], phase ^ 1u, kErrTimeoutProducer);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&full[stage], S::STAGE_BYTES);
          __syncwarp();
          if (a_lane || b_lane) tma_load_2d(dst0 + stage * dst_step, map, &full[stage], kb * 128, row);
          ++issued;
          if (++stage == S::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // no copy is in flight when the block ends, on the way out after a timeout either
#pragma unroll 1
      for (int i = issued < S::STAGES ? 0 : issued - S::STAGES; i < issued; ++i)
        fp8_wait(&full[i % S::STAGES], (i / S::STAGES) & 1, kErrTimeoutProducer);
    } else if (warp == 1) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t idesc = idesc_e4m3(128, BN);
      const uint64_t a_desc = smem_desc(smem_u32(sA), 16, 1024, kLayoutSwizzle128B);
      const uint32_t desc_hi = (uint32_t)(a_desc >> 32), a_lo = (uint32_t)a_desc;
      const uint32_t b_lo = (uint32_t)smem_desc(smem_u32(sB), 16, 1024, kLayoutSwizzle128B);
      uint32_t stage = 0, buf = 0;
      for (int i = 0; i < turns; ++i) {
        named_sync(kFp8BarGo + buf, i < S::BUFS ? 64 : 32 * (S::EPI_WARPS + 2));
        tc_fence_after();
        if (lane == 0) {
          const uint32_t a = a_lo + stage * (S::A_BYTES >> 4), b = b_lo + stage * (S::B_BYTES >> 4);
          const uint32_t d = tmem + buf * BN;
          tc_mma_e4m3<0>(d, a, b, desc_hi, idesc);
          tc_mma_e4m3<1>(d, a + 2, b + 2, desc_hi, idesc);
          tc_mma_e4m3<1>(d, a + 4, b + 4, desc_hi, idesc);
          tc_mma_e4m3<1>(d, a + 6, b + 6, desc_hi, idesc);
          tc_commit(&done[stage]);
        }
        __syncwarp();
        if (++stage == S::STAGES) stage = 0;
        if (++buf == S::BUFS) buf = 0;
      }
      // the epilogue's releases of the last buffers
      for (int i = turns < S::BUFS ? 0 : turns - S::BUFS; i < turns; ++i)
        named_sync(kFp8BarGo + i % S::BUFS, 32 * (S::EPI_WARPS + 2));
    } else if (warp == 2) {
      // ---------------- relay: products complete -> epilogue ----------------
      uint32_t stage = 0, phase = 0;
      for (int i = 0; i < turns; ++i) {
        fp8_wait(&done[stage], phase, kErrTimeoutEpilogue);
        __syncwarp();
        named_sync(kFp8BarSums + i % S::BUFS, 32 * (S::EPI_WARPS + 1));
        if (++stage == S::STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    } else {
      // ---------------- relay: operands landed -> issuer ----------------
      // takes part in the go barrier for what would be a wait of the issuer
      uint32_t stage = 0, stage_phase = 0, buf = 0;
      bool ok = true;
      for (int i = 0; i < turns; ++i) {
        ok = ok && fp8_wait(&full[stage], stage_phase, kErrTimeoutMma);
        __syncwarp();
        named_sync(kFp8BarGo + buf, i < S::BUFS ? 64 : 32 * (S::EPI_WARPS + 2));
        if (++stage == S::STAGES) {
          stage = 0;
          stage_phase ^= 1u;
        }
        if (++buf == S::BUFS) buf = 0;
      }
      for (int i = turns < S::BUFS ? 0 : turns - S::BUFS; i < turns; ++i)
        named_sync(kFp8BarGo + i % S::BUFS, 32 * (S::EPI_WARPS + 2));
    }
  } else {
    if constexpr (S::SPLIT_REGS) regs_up<S::EPI_REGS>();
    // ---------------- epilogue ----------------
    pdl_wait();
    const uint32_t quad = (uint32_t)(warp & 3);
    const int h = (warp - S::EPI_WARP0) >> 2;  // columns COLS h .. (SwiGLU: gate 64 h .. and up 128 + 64 h ..)
    const int row_in_tile = (int)(quad * 32 + lane);
    const uint32_t taddr = tmem + ((quad * 32u) << 16) + (MODE == FP8_SWIGLU ? 64u : (uint32_t)S::COLS) * h;
    const int n_blocks = (p.N + kFp8Block - 1) / kFp8Block;
    // A unit's rows, columns and scale addresses, and the scales of its first
    // two k-blocks, are fetched while the previous unit is written out (the
    // activation scales are the previous kernel's: ordinary loads).
    const int64_t up = MODE == FP8_SWIGLU ? (int64_t)(F / 128) * k_blocks : 0;
    int n = 0, valid = 0;
    bool few = false;
    int64_t row = 0;
    const float *xs = nullptr, *ws = nullptr;
    float x0 = 0.0f, w00 = 0.0f, w01 = 0.0f, x1 = 0.0f, w10 = 0.0f, w11 = 0.0f;
    auto fetch = [&](int u) {
      const int m = u / n_tiles;
      const TileEntry t = fp8_tile(p, m);
      n = u - m * n_tiles;
      valid = t.valid;
      few = FEW && valid <= kFp8FewRows;
      row = (int64_t)t.row0 + (few ? (int)lane : row_in_tile);
      xs = p.xs + min(row, p.rows - 1);
      // the weight scales of this thread's columns: one row of blocks, or the
      // gate's and the up's
      const int nb0 = MODE == FP8_SWIGLU ? n : min((n * BN + h * S::COLS) / kFp8Block, n_blocks - 1);
      ws = p.ws + ((int64_t)t.expert * n_blocks + nb0) * k_blocks;
      x0 = *xs;
      w00 = __ldg(ws);
      if (MODE == FP8_SWIGLU) w01 = __ldg(ws + up);
      if (k_blocks > 1) {
        x1 = xs[p.xs_ld];
        w10 = __ldg(ws + 1);
        if (MODE == FP8_SWIGLU) w11 = __ldg(ws + 1 + up);
      }
    };
    uint32_t buf = 0, unit = 0;
    if (first < total) fetch(first);
    // the scales of k-block kb, and the loads of those two blocks on
    auto scales = [&](int kb, float& f0, float& f1) {
      f0 = x0 * w00;
      f1 = MODE == FP8_SWIGLU ? x0 * w01 : f0;
      x0 = x1;
      w00 = w10;
      w01 = w11;
      if (kb + 2 < k_blocks) {
        x1 = xs[(int64_t)(kb + 2) * p.xs_ld];
        w10 = __ldg(ws + kb + 2);
        if (MODE == FP8_SWIGLU) w11 = __ldg(ws + kb + 2 + up);
      }
    };
    for (int u = first; u < total; u += step, ++unit) {
      uint32_t ra[16], rb[16];
      if (FEW && few) {
        // 32 columns: 32 in a row, or 16 of the gate and the same 16 of the up
        float acc[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[j] = 0.0f;
        const uint32_t tf = tmem + ((quad * 32u) << 16) + (MODE == FP8_SWIGLU ? 64u * h + 16u * quad : 128u * h + 32u * quad);
        for (int kb = 0; kb < k_blocks; ++kb) {
          float f0, f1;
          scales(kb, f0, f1);
          named_sync(kFp8BarSums + buf, 32 * (S::EPI_WARPS + 1));
          tc_fence_after();
          tc_ld_32x32b_x16(tf + buf * BN, ra);
          tc_ld_32x32b_x16(tf + buf * BN + (MODE == FP8_SWIGLU ? 128 : 16), rb);
          tc_wait_ld();
          tc_fence_before();
          named_arrive(kFp8BarGo + buf, 32 * (S::EPI_WARPS + 2));
          fp8_add_block(acc, ra, f0);
          fp8_add_block(acc + 16, rb, f1);
          if (++buf == S::BUFS) buf = 0;
        }
        const int n_out = n;
        const int64_t row_out = row;
        const bool live = (int)lane < valid;
        if (u + step < total) fetch(u + step);
        if constexpr (MODE == FP8_SWIGLU) {
          float a = kFp8MinAmax;
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            swiglu_pair_f32(acc[j], acc[j + 1], acc[16 + j], acc[17 + j]);
            a = fmaxf(a, fmaxf(fabsf(acc[j]), fabsf(acc[j + 1])));
          }
          float* mx = s_max + (unit & 1u) * 256 + lane;
          mx[(2 * quad + h) * 32] = a;
          named_sync(kFp8BarMax, 32 * S::EPI_WARPS);
#pragma unroll
          for (int i = 0; i < 8; ++i) a = fmaxf(a, mx[i * 32]);
          if (live) {
            const float r = div_rn(kE4m3Max, a);
            uint32_t c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              c[i] = cvt_e4m3x4(mul_rn(acc[4 * i], r), mul_rn(acc[4 * i + 1], r), mul_rn(acc[4 * i + 2], r),
                                mul_rn(acc[4 * i + 3], r));
            *reinterpret_cast<uint4*>(p.hq + row_out * F + n_out * 128 + 64 * h + 16 * quad) =
                make_uint4(c[0], c[1], c[2], c[3]);
            if (h == 0 && quad == 0) p.hs[(int64_t)n_out * p.hs_ld + row_out] = div_rn(a, kE4m3Max);
          }
        } else {
          const int col = n_out * BN + 128 * h + 32 * (int)quad;
          if (live && col < p.N) {
            uint4* dst = reinterpret_cast<uint4*>(p.out + row_out * p.N + col);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float* v = acc + 8 * i;
              dst[i] = make_uint4(cvt_bf16x2(v[0], v[1]), cvt_bf16x2(v[2], v[3]), cvt_bf16x2(v[4], v[5]),
                                  cvt_bf16x2(v[6], v[7]));
            }
          }
        }
        __syncwarp();
        continue;
      }
      float acc[S::COLS];
#pragma unroll
      for (int j = 0; j < S::COLS; ++j) acc[j] = 0.0f;
      for (int kb = 0; kb < k_blocks; ++kb) {
        const uint32_t tb = taddr + buf * BN;
        float f0, f1;
        scales(kb, f0, f1);
        named_sync(kFp8BarSums + buf, 32 * (S::EPI_WARPS + 1));
        tc_fence_after();
        tc_ld_32x32b_x16(tb, ra);
#pragma unroll
        for (int c = 0; c < S::COLS / 16; c += 2) {
          tc_wait_ld();
          tc_ld_32x32b_x16(tb + chunk_col<MODE>(c + 1), rb);
          fp8_add_block(acc + 16 * c, ra, c < 4 ? f0 : f1);
          if (c + 2 == S::COLS / 16) break;
          tc_wait_ld();
          tc_ld_32x32b_x16(tb + chunk_col<MODE>(c + 2), ra);
          fp8_add_block(acc + 16 * (c + 1), rb, c < 4 ? f0 : f1);
        }
        tc_wait_ld();
        tc_fence_before();
        named_arrive(kFp8BarGo + buf, 32 * (S::EPI_WARPS + 2));
        fp8_add_block(acc + S::COLS - 16, rb, f1);
        if (++buf == S::BUFS) buf = 0;
      }
      const int n_out = n;
      const int64_t row_out = row;
      const int valid_out = valid;
      if (u + step < total) fetch(u + step);
      if constexpr (MODE == FP8_SWIGLU) {
        // 64 hidden columns 128 n_out + 64 h ..; the other half's warps hold the
        // rest of the row's block, so the row maxima meet in shared memory
        float a = kFp8MinAmax;
#pragma unroll
        for (int j = 0; j < 64; j += 2) {
          swiglu_pair_f32(acc[j], acc[j + 1], acc[64 + j], acc[65 + j]);
          a = fmaxf(a, fmaxf(fabsf(acc[j]), fabsf(acc[j + 1])));
        }
        float* mx = s_max + (unit & 1u) * 256 + row_in_tile;
        mx[h * 128] = a;
        named_sync(kFp8BarMax, 32 * S::EPI_WARPS);
        a = fmaxf(a, mx[(h ^ 1) * 128]);
        if (row_in_tile < valid_out) {
          const float r = div_rn(kE4m3Max, a);
          uint8_t* dst = p.hq + row_out * F + n_out * 128 + 64 * h;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float* v = acc + 32 * j + 4 * i;
              c[i] = cvt_e4m3x4(mul_rn(v[0], r), mul_rn(v[1], r), mul_rn(v[2], r), mul_rn(v[3], r));
            }
            st_global_v8(reinterpret_cast<uint16_t*>(dst + 32 * j), make_uint4(c[0], c[1], c[2], c[3]),
                         make_uint4(c[4], c[5], c[6], c[7]));
          }
          if (h == 0) p.hs[(int64_t)n_out * p.hs_ld + row_out] = div_rn(a, kE4m3Max);
        }
      } else {
        const int col0 = n_out * BN + S::COLS * h;
        // boxes of 32 rows x 64 columns in the TMA 128-byte swizzle
        uint8_t* box = sOut + (warp - S::EPI_WARP0) * S::OUT_BOX;
        const int box_rows = valid_out - 32 * (int)quad;  // rows of the box that exist
#pragma unroll
        for (int i = 0; i < S::COLS / 64; ++i) {
          const int col = col0 + 64 * i;
          if (p.tma_out && lane == 0) bulk_wait_group_read0();
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float* v = acc + 64 * i + 8 * c;
            *reinterpret_cast<uint4*>(box + lane * 128 + ((c ^ (lane & 7)) << 4)) =
                make_uint4(cvt_bf16x2(v[0], v[1]), cvt_bf16x2(v[2], v[3]), cvt_bf16x2(v[4], v[5]),
                           cvt_bf16x2(v[6], v[7]));
          }
          if (p.tma_out) {
            // of a table's tile the padding rows are written too (scratch),
            // never rows of the next tile
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0 && box_rows > 0 && col < p.N) {
              tma_store_2d(&p.tmap_out, box, col, (int32_t)row_out);
              bulk_commit_group();
            }
          } else {
            // rows that are no multiple of 16 bytes: a lane writes column lane
            // and lane + 32 of each row
            __syncwarp();
            const int64_t r0 = row_out - (int64_t)lane;
            for (int r = 0; r < min(box_rows, 32); ++r) {
              uint16_t* dst = p.out + (r0 + r) * p.N + col;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int c = (int)lane + 32 * j;
                if (col + c < p.N)
                  dst[c] = *reinterpret_cast<const uint16_t*>(box + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
              }
            }
          }
        }
      }
      __syncwarp();
    }
    if (MODE == FP8_PLAIN && lane == 0) bulk_wait_group0();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::BUFS * BN);
  }
}

// ---------------------------------------------------------------------------
// Few rows: the weight is streamed once through the registers.
//
// With at most 8 rows per weight the product is the time to read the weight,
// and a 128-row MMA tile leaves most SMs without a tile (4096 x 4096: 16 tiles).
// Here a CTA takes 16 weight rows and its warps share the k-blocks: a lane holds
// 2 rows x 2 x 16 bytes of a block, which are the A operand of four
// mma.m16n8k32 as they are (both operands use the same order of the 128
// columns, so no lane exchanges bytes). The CTA quantizes its activation rows
// into shared memory while the first weight loads are in flight; a consumed
// block's registers are loaded again at once.
//
// Up  (SwiGLU): gate and up rows together, h = swiglu kept in fp32.
// Down (routed): each warp takes one of the token's routed slots (or a share of
// its k-blocks) and the sum over the warps is the weighted combine.
// ---------------------------------------------------------------------------
enum Fp8Stream : int { FP8_STREAM_LINEAR = 0, FP8_STREAM_UP = 1, FP8_STREAM_DOWN = 2 };

struct Fp8StreamParams {
  const void* x;          // LINEAR, UP: bf16 rows, pitch ldx; DOWN: fp32 hidden rows [rows or rows * top_k, K]
  int64_t ldx;
  const uint8_t* wq;      // [E][N][K]
  const float* ws;        // [E][N blocks][K blocks]
  int32_t rows;           // rows of x (tokens)
  int32_t N, K;           // UP: N = 2F
  int32_t experts;
  int32_t top_k;          // 0: dense (all rows share the weight); else one row per routed slot
  const int64_t* top_idx;
  const uint16_t* gate;   // DOWN, routed
  float scaling;
  const uint16_t* shared;  // DOWN, routed: added after rounding, or nullptr
  float* hidden;          // UP: [rows or rows * top_k, F]
  uint16_t* out;          // LINEAR, DOWN: bf16 [rows, N]
};

// 16 warps per SM in any case: DOWN has two for each of up to 8 slots, UP takes
// four CTAs of four (one token through 8 of 64 experts: 24.3 us against 25.5
// with two of eight).
template <int OP>
__host__ __device__ constexpr int fp8_stream_warps() {
  return OP == FP8_STREAM_DOWN ? 16 : OP == FP8_STREAM_UP ? 4 : 8;
}

// Quantized activation rows in shared memory: row pitch (64 bytes more than a
// multiple of 128: the 8 rows of an operand load fall into different banks),
// then the scales [rows][K blocks].
__host__ __device__ constexpr int fp8_stream_pitch(int k) { return (k + kFp8Block - 1) / kFp8Block * kFp8Block + 64; }
__host__ __device__ constexpr size_t fp8_stream_smem(int rows, int k) {
  return (size_t)rows * (fp8_stream_pitch(k) + 4 * ((k + kFp8Block - 1) / kFp8Block));
}

// Eight activations of a row as floats (the previous kernel's results, or may be:
// ordinary loads).
__device__ __forceinline__ void load8(const uint16_t* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = unpack_bf16x2(w[j]);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 f = reinterpret_cast<const float4*>(p)[i];
    v[4 * i] = f.x;
    v[4 * i + 1] = f.y;
    v[4 * i + 2] = f.z;
    v[4 * i + 3] = f.w;
  }
}

// `rows` rows (pitch ldx) -> codes and scales in shared memory, half a warp per
// block of 128 columns and U blocks in flight. Columns past k are zero codes.
template <typename T, int THREADS, int U>
__device__ __forceinline__ void fp8_stream_quantize(const T* x, int64_t ldx, int rows, int k, uint8_t* codes,
                                                    float* scales) {
  const int k_blocks = (k + kFp8Block - 1) / kFp8Block, pitch = fp8_stream_pitch(k);
  const int total = rows * k_blocks, sub = threadIdx.x & 15;
  constexpr int GROUPS = THREADS / 16;
  for (int i0 = 0; i0 < total; i0 += U * GROUPS) {  // whole warps take every turn
    float v[U][8];
    int r[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * GROUPS + (int)(threadIdx.x >> 4);
      r[u] = i < total ? i / k_blocks : -1;
      b[u] = i - r[u] * k_blocks;
      const int col = b[u] * kFp8Block + 8 * sub;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[u][j] = 0.0f;
      if (r[u] >= 0 && col < k) load8(x + (int64_t)r[u] * ldx + col, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float m = kFp8MinAmax;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[u][j]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (r[u] >= 0) {
        const float q = div_rn(kE4m3Max, m);
        *reinterpret_cast<uint2*>(codes + r[u] * pitch + b[u] * kFp8Block + 8 * sub) = make_uint2(
            cvt_e4m3x4(mul_rn(v[u][0], q), mul_rn(v[u][1], q), mul_rn(v[u][2], q), mul_rn(v[u][3], q)),
            cvt_e4m3x4(mul_rn(v[u][4], q), mul_rn(v[u][5], q), mul_rn(v[u][6], q), mul_rn(v[u][7], q)));
        if (sub == 0) scales[r[u] * k_blocks + b[u]] = div_rn(m, kE4m3Max);
      }
    }
  }
}

// d += A (16 x 32 E4M3) * B (32 x 8 E4M3), fp32 sums
__device__ __forceinline__ void mma_e4m3_16x8x32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// blockIdx.x: 16 weight rows (UP: 16 hidden columns), and every gridDim.x-th 16
// after them; blockIdx.y: dense: 0; UP: the routed slot; DOWN: the token.
template <int OP>
__global__ void __launch_bounds__(32 * fp8_stream_warps<OP>(), 16 / fp8_stream_warps<OP>())
    fp8_stream_kernel(const __grid_constant__ Fp8StreamParams p) {
  // behind UP, which writes the hidden rows alone, DOWN loads its first weights
  // before it waits
  if (OP != FP8_STREAM_DOWN) {
    pdl_wait();
    pdl_trigger();
  }
  constexpr int WARPS = fp8_stream_warps<OP>();
  constexpr int SETS = OP == FP8_STREAM_UP ? 2 : 1;
  constexpr int AHEAD = 4 / SETS;  // k-blocks of a warp whose loads are in flight
  using T = typename std::conditional<OP == FP8_STREAM_DOWN, float, uint16_t>::type;
  extern __shared__ __align__(16) uint8_t s_codes[];
  __shared__ float s_sum[WARPS][SETS][16][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int cols = OP == FP8_STREAM_UP ? p.N / 2 : p.N;  // output columns
  const int k_blocks = (p.K + kFp8Block - 1) / kFp8Block, n_blocks = (p.N + kFp8Block - 1) / kFp8Block;
  const bool routed = p.top_k > 0;
  // this CTA's activation rows, and this warp's share: rows of one weight, from
  // k-block kb0 on
  int expert = 0, kb0 = warp, step = WARPS, row0 = 0, rows = p.rows;
  bool busy = true;
  float weight = 1.0f;
  const T* x = static_cast<const T*>(p.x);
  if (routed && OP == FP8_STREAM_DOWN) {
    const int per = WARPS / p.top_k, slot = warp / per;  // warps per slot
    rows = p.top_k;
    x += (int64_t)blockIdx.y * p.top_k * p.ldx;
    busy = slot < p.top_k;
    if (busy) {
      const int64_t r = (int64_t)blockIdx.y * p.top_k + slot;
      expert = checked_expert(p.top_idx[r], p.experts);
      weight = mul_rn(bf16_to_f32(p.gate[r]), p.scaling);
      kb0 = warp % per;
      step = per;
      row0 = slot;
    }
  } else if (routed) {
    rows = 1;
    x += (int64_t)(blockIdx.y / p.top_k) * p.ldx;
    expert = checked_expert(p.top_idx[blockIdx.y], p.experts);
  }
  const int my_rows = routed ? 1 : rows;  // rows that share this warp's weight
  const uint8_t* w = p.wq + ((int64_t)expert * p.N + g) * p.K + 16 * t;
  const float* ws = p.ws + (int64_t)expert * n_blocks * k_blocks;
  const int64_t set_off = (int64_t)cols * p.K, ws_off = (int64_t)(cols / kFp8Block) * k_blocks;
  uint4 a[AHEAD][SETS][2][2];  // [block][set][row g, g + 8][64-byte half]
  float sw[AHEAD][SETS];
  auto load = [&](int i, int n0, int kb) {
    const bool in = busy && kb < k_blocks;
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int col = kb * kFp8Block + 64 * j;
          a[i][s][r][j] = make_uint4(0u, 0u, 0u, 0u);
          if (in && col + 16 * t < p.K && n0 + g + 8 * r < cols)
            a[i][s][r][j] = ldg_stream(
                reinterpret_cast<const uint4*>(w + s * set_off + (int64_t)(n0 + 8 * r) * p.K + col));
        }
      sw[i][s] = in ? __ldg(ws + s * ws_off + (int64_t)(n0 / kFp8Block) * k_blocks + kb) : 0.0f;
    }
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(i, blockIdx.x * 16, kb0 + i * step);
  if (OP == FP8_STREAM_DOWN) {
    pdl_wait();
    pdl_trigger();
  }
  const int pitch = fp8_stream_pitch(p.K);
  float* scales = reinterpret_cast<float*>(s_codes + (size_t)rows * pitch);
  fp8_stream_quantize<T, 32 * WARPS, OP == FP8_STREAM_UP ? 2 : 4>(x, p.ldx, rows, p.K, s_codes, scales);
  __syncthreads();
  // rows past my_rows read row0's codes; their sums are not stored
  const uint8_t* b_row = s_codes + (size_t)(row0 + (g < my_rows ? g : 0)) * pitch + 16 * t;
  const float* sx0 = scales + (row0 + (2 * t < my_rows ? 2 * t : 0)) * k_blocks;
  const float* sx1 = scales + (row0 + (2 * t + 1 < my_rows ? 2 * t + 1 : 0)) * k_blocks;
  for (int n0 = blockIdx.x * 16; n0 < cols; n0 += gridDim.x * 16) {
    float acc[SETS][4] = {};
    for (int base = kb0; busy && base < k_blocks; base += AHEAD * step) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int kb = base + i * step;
        if (kb >= k_blocks) break;
        const uint4 b0 = *reinterpret_cast<const uint4*>(b_row + kb * kFp8Block);
        const uint4 b1 = *reinterpret_cast<const uint4*>(b_row + kb * kFp8Block + 64);
        const float s0 = sx0[kb], s1 = sx1[kb];
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
          float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma_e4m3_16x8x32(d, a[i][s][0][0].x, a[i][s][1][0].x, a[i][s][0][0].y, a[i][s][1][0].y, b0.x, b0.y);
          mma_e4m3_16x8x32(d, a[i][s][0][0].z, a[i][s][1][0].z, a[i][s][0][0].w, a[i][s][1][0].w, b0.z, b0.w);
          mma_e4m3_16x8x32(d, a[i][s][0][1].x, a[i][s][1][1].x, a[i][s][0][1].y, a[i][s][1][1].y, b1.x, b1.y);
          mma_e4m3_16x8x32(d, a[i][s][0][1].z, a[i][s][1][1].z, a[i][s][0][1].w, a[i][s][1][1].w, b1.z, b1.w);
          const float f0 = s0 * sw[i][s], f1 = s1 * sw[i][s];
          acc[s][0] = fmaf(d[0], f0, acc[s][0]);
          acc[s][1] = fmaf(d[1], f1, acc[s][1]);
          acc[s][2] = fmaf(d[2], f0, acc[s][2]);
          acc[s][3] = fmaf(d[3], f1, acc[s][3]);
        }
        if (kb + AHEAD * step < k_blocks) load(i, n0, kb + AHEAD * step);
      }
    }
    // the next 16 rows' first loads, under way during the reduction
    if (n0 + (int)gridDim.x * 16 < cols) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) load(i, n0 + gridDim.x * 16, kb0 + i * step);
    }
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      s_sum[warp][s][g][2 * t] = acc[s][0] * weight;
      s_sum[warp][s][g][2 * t + 1] = acc[s][1] * weight;
      s_sum[warp][s][g + 8][2 * t] = acc[s][2] * weight;
      s_sum[warp][s][g + 8][2 * t + 1] = acc[s][3] * weight;
    }
    __syncthreads();
    const int n = n0 + (threadIdx.x & 15), c = threadIdx.x >> 4;  // output column n of activation row c
    if (c < my_rows && n < cols) {
      float sum[SETS];
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        sum[s] = s_sum[0][s][n - n0][c];
#pragma unroll
        for (int i = 1; i < WARPS; ++i) sum[s] += s_sum[i][s][n - n0][c];
      }
      const int64_t row = routed ? blockIdx.y : c;
      if constexpr (OP == FP8_STREAM_UP) {
        float g0 = sum[0], g1 = 0.0f;
        swiglu_pair_f32(g0, g1, sum[1], 0.0f);
        p.hidden[row * cols + n] = g0;
      } else {
        uint16_t y = f32_to_bf16(sum[0]);
        if (OP == FP8_STREAM_DOWN && routed && p.shared != nullptr)
          y = f32_to_bf16(add_rn(bf16_to_f32(y), bf16_to_f32(p.shared[row * cols + n])));
        p.out[row * cols + n] = y;
      }
    }
    if (n0 + (int)gridDim.x * 16 < cols) __syncthreads();  // the sums are read
  }
}

// The dispatch of `rows` rows to themselves (one expert, gate 1), for the fused
// tail after a streamed feed-forward.
__global__ void fp8_identity_kernel(int rows, int64_t* inverse, int64_t* top_idx, uint16_t* gate, int32_t* csr,
                                    int32_t* pcsr) {
  pdl_wait();  // the previous kernel of the stream has completed
  pdl_trigger();
  for (int i = threadIdx.x; i < rows; i += blockDim.x) {
    inverse[i] = i;
    top_idx[i] = 0;
    gate[i] = 0x3F80;  // 1 in bf16
  }
  if (threadIdx.x < 2) csr[threadIdx.x] = pcsr[threadIdx.x] = threadIdx.x == 0 ? 0 : rows;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Rows of `cols` elements in boxes of 128 bytes x box_rows, 128-byte swizzle.
static int fp8_map(CUtensorMap* map, CUtensorMapDataType type, int elem, const void* base, int64_t rows, int64_t cols,
                   int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return set_error(PRAXIS_B200_ECUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t gdim[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t gstride[1] = {(cuuint64_t)cols * elem};
  cuuint32_t box[2] = {(cuuint32_t)(128 / elem), (cuuint32_t)box_rows};
  cuuint32_t estride[2] = {1u, 1u};
  CUresult r = fn(map, type, 2, const_cast<void*>(base), gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(PRAXIS_B200_ECUDA, "cuTensorMapEncodeTiled (fp8) failed (%d)", (int)r);
  return PRAXIS_B200_OK;
}

// Launches on at most one CTA per SM; `units` bounds the work.
template <int BN, int MODE, bool FEW>
static int fp8_launch(const Fp8GemmParams& p, int64_t units, cudaStream_t stream) {
  using S = Fp8Shape<BN>;
  auto kernel = fp8_gemm_kernel<BN, MODE, FEW>;
  static DeviceOnce attr;
  const int rc = device_once(attr, [&](int dev) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM_BYTES);
    if (e != cudaSuccess)
      return set_error(PRAXIS_B200_ECUDA, "fp8 gemm smem attribute (device %d): %s", dev, cudaGetErrorString(e));
    // setmaxnreg waits for registers that the launch does not have
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, kernel);
    if (e != cudaSuccess || (S::SPLIT_REGS && fa.numRegs < S::LAUNCH_REGS))
      return set_error(PRAXIS_B200_ECUDA, "fp8 gemm: built with %d registers a thread, needs %d", fa.numRegs,
                       S::LAUNCH_REGS);
    return (int)PRAXIS_B200_OK;
  });
  if (rc) return rc;
  const int grid = (int)(units < sm_count() ? units : sm_count());
  launch_pdl(kernel, dim3(grid), dim3(S::THREADS), S::SMEM_BYTES, stream, p);
  return check_launch("fp8_gemm");
}

static size_t fp8_slots_workspace(int experts) { return (size_t)(experts + 1) * 4; }

static int run_fp8_slots(const int64_t* top_idx, int64_t positions, int experts, void* workspace, int64_t* inverse,
                         int32_t* csr, int32_t* pcsr, TileEntry* tiles, int max_tiles, int32_t* num_tiles,
                         cudaStream_t stream) {
  constexpr int64_t kPerCta = kFp8SlotThreads * kFp8SlotItems;
  const int64_t ctas = (positions + kPerCta - 1) / kPerCta;
  if (ctas > 1) {
    const cudaError_t e = cudaMemsetAsync(workspace, 0, fp8_slots_workspace(experts), stream);
    if (e != cudaSuccess) return set_error(PRAXIS_B200_ECUDA, "fp8 slots: %s", cudaGetErrorString(e));
  }
  launch_pdl(fp8_slots_kernel, dim3((unsigned)ctas), dim3(kFp8SlotThreads), 0, stream, top_idx, positions, experts,
             static_cast<uint32_t*>(workspace), inverse, csr, pcsr, tiles, max_tiles, num_tiles);
  return check_launch("fp8_slots");
}

int run_fp8_quantize(const uint16_t* x, int64_t rows, int cols, int64_t ldx, const Fp8Rows& to, uint8_t* q,
                     float* scale, int64_t scale_ld, cudaStream_t stream) {
  if (rows == 0) return PRAXIS_B200_OK;
  const dim3 grid((unsigned)((rows + kFp8QuantWarps - 1) / kFp8QuantWarps),
                  (unsigned)((cols + kFp8QuantCols - 1) / kFp8QuantCols));
  launch_pdl(fp8_quantize_kernel, grid, dim3(32 * kFp8QuantWarps), 0, stream, x, rows, cols, ldx, to, q, scale,
             scale_ld);
  return check_launch("fp8_quantize");
}

int run_fp8_pack(const uint16_t* w, int64_t experts, int64_t k, int64_t n, uint8_t* q, float* scale,
                 cudaStream_t stream) {
  const int64_t blocks = experts * ((n + kFp8Block - 1) / kFp8Block) * ((k + kFp8Block - 1) / kFp8Block);
  if (blocks == 0) return PRAXIS_B200_OK;
  fp8_pack_kernel<<<(unsigned)blocks, 256, 0, stream>>>(w, k, n, q, scale);
  return check_launch("fp8_pack");
}

// One GEMM over quantized rows, launched behind the kernel that wrote them
// (the quantization or the gate/up GEMM, which write neither the weights nor
// the tile table and let this one start only when all before them is done).
// Dense (tiles == nullptr): `rows` rows against
// one weight. Grouped: fp8_slots_kernel's tables, rows = padded rows, max_tiles
// bounds the 128-row tiles. out (FP8_PLAIN) or hq / hs (FP8_SWIGLU) get the result.
struct Fp8Gemm {
  const uint8_t* q;
  const float* xs;
  int64_t xs_ld;
  const uint8_t* wq;
  const float* ws;
  int64_t rows;
  int32_t n, k, experts;
  const TileEntry* tiles;
  const int32_t* num_tiles;
  int32_t max_tiles;
  int64_t slots;  // routed rows without the padding
  uint16_t* out;
  uint8_t* hq;
  float* hs;
  int64_t hs_ld;
};

int run_fp8_gemm(const Fp8Gemm& g, cudaStream_t stream) {
  if (g.rows == 0) return PRAXIS_B200_OK;
  const bool swiglu = g.out == nullptr;
  const int64_t n_tiles = swiglu ? g.n / 256 : (g.n + 255) / 256;
  const int64_t m_tiles = g.tiles != nullptr ? g.max_tiles : (g.rows + 127) / 128;
  // 64-column tiles where they all fit the SMs at once (K = 4096, cold weights:
  // 32 tiles of 256 columns 21 us, the same in 64 columns 18; 64 tiles 23 against 28)
  const bool narrow = !swiglu && g.tiles == nullptr && 4 * m_tiles * n_tiles <= sm_count();
  Fp8GemmParams p;
  memset(&p, 0, sizeof(p));
  int rc = fp8_map(&p.tmap_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.q, g.rows, g.k, 128);
  if (rc) return rc;
  rc = fp8_map(&p.tmap_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.wq, (int64_t)g.experts * g.n, g.k, narrow ? 64 : 128);
  if (rc) return rc;
  if (!swiglu && g.n % 8 == 0 && ((uintptr_t)g.out & 15) == 0) {
    rc = fp8_map(&p.tmap_out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, g.out, g.rows, g.n, 32);
    if (rc) return rc;
    p.tma_out = 1;
  }
  // Few rows per tile on average: the kernel that splits such tiles by columns
  // (4 of 64 experts, C 2048, F 1536, 64 tokens 136 -> 125 us, 512 tokens, 32 rows
  // per expert, 139 -> 135; 1024 tokens 146 -> 149, so not beyond).
  const bool few = !narrow && (swiglu || (p.tma_out && g.n % 32 == 0)) &&
                   (g.tiles != nullptr ? g.slots <= (int64_t)kFp8FewRows * g.experts : g.rows <= kFp8FewRows);
  if (few) {
    rc = fp8_map(&p.tmap_a32, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.q, g.rows, g.k, kFp8FewRows);
    if (rc) return rc;
  }
  p.xs = g.xs;
  p.xs_ld = g.xs_ld;
  p.ws = g.ws;
  p.num_tiles = g.num_tiles;
  p.rows = g.rows;
  p.N = g.n;
  p.K = g.k;
  p.experts = g.experts;
  p.out = g.out;
  p.hq = g.hq;
  p.hs = g.hs;
  p.hs_ld = g.hs_ld;
  p.tiles = g.tiles;
  if (narrow) return fp8_launch<64, FP8_PLAIN, false>(p, m_tiles * ((g.n + 63) / 64), stream);
  const int64_t units = m_tiles * n_tiles;
  if (swiglu)
    return few ? fp8_launch<256, FP8_SWIGLU, true>(p, units, stream) : fp8_launch<256, FP8_SWIGLU, false>(p, units, stream);
  return few ? fp8_launch<256, FP8_PLAIN, true>(p, units, stream) : fp8_launch<256, FP8_PLAIN, false>(p, units, stream);
}

constexpr size_t kFp8StreamSmemMax = 160 * 1024;

template <int OP>
static int fp8_stream_launch(const Fp8StreamParams& p, int groups, cudaStream_t stream) {
  auto kernel = fp8_stream_kernel<OP>;
  static DeviceOnce attr;
  const int rc = device_once(attr, [&](int dev) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFp8StreamSmemMax);
    if (e != cudaSuccess)
      return set_error(PRAXIS_B200_ECUDA, "fp8 stream smem attribute (device %d): %s", dev, cudaGetErrorString(e));
    return (int)PRAXIS_B200_OK;
  });
  if (rc) return rc;
  const int cols = OP == FP8_STREAM_UP ? p.N / 2 : p.N;
  const int rows = p.top_k == 0 ? p.rows : OP == FP8_STREAM_DOWN ? p.top_k : 1;
  // with several activation rows a CTA quantizes them once for all its columns
  const int tiles = (cols + 15) / 16, most = sm_count() * (16 / fp8_stream_warps<OP>());
  launch_pdl(kernel, dim3((unsigned)(rows > 1 && groups == 1 && tiles > most ? most : tiles), (unsigned)groups),
             dim3(32 * fp8_stream_warps<OP>()), fp8_stream_smem(rows, p.K), stream, p);
  return check_launch("fp8_stream");
}

// Whether a product of `rows` rows goes through the streaming kernels: dense up
// to the 8 rows that share a weight; routed slots read their expert's weight
// each for itself, so as long as they are few, more of them where many experts
// leave the tiles few rows each (streamed / in tiles, cold weights, us: C 2048,
// F 1536, 64 experts, 16 slots 49 / 50, 24 slots 68 / 61; C 1024, F 2048, 8
// experts, 8 slots 21 / 27, 12 slots 29 / 28; 32 experts, 12 slots 30 / 33, 16
// slots 38 / 36). The quantized rows have to fit the shared memory (k_up:
// columns of the rows, k_down: of the hidden rows, 0 for a linear product).
static bool fp8_streams(int64_t rows, int top_k, int experts, int k_up, int k_down) {
  if (top_k == 0 ? rows > 8 : rows * top_k > 8 + experts / 8) return false;
  return fp8_stream_smem(top_k == 0 ? (int)rows : 1, k_up) <= kFp8StreamSmemMax &&
         fp8_stream_smem(top_k == 0 ? (int)rows : top_k, k_down) <= kFp8StreamSmemMax;
}

static int run_fp8_stream_linear(const Fp8StreamParams& p, cudaStream_t stream) {
  return fp8_stream_launch<FP8_STREAM_LINEAR>(p, 1, stream);
}

// The feed-forward: p.x bf16 rows, p.hidden fp32 scratch.
static int run_fp8_stream_ffn(Fp8StreamParams p, const uint8_t* down_q, const float* down_scale, int32_t dim,
                              int32_t hidden, cudaStream_t stream) {
  int rc = fp8_stream_launch<FP8_STREAM_UP>(p, p.top_k > 0 ? p.rows * p.top_k : 1, stream);
  if (rc) return rc;
  p.x = p.hidden;
  p.ldx = hidden;
  p.wq = down_q;
  p.ws = down_scale;
  p.N = dim;
  p.K = hidden;
  return fp8_stream_launch<FP8_STREAM_DOWN>(p, p.top_k > 0 ? p.rows : 1, stream);
}

static int run_fp8_identity(int rows, int64_t* inverse, int64_t* top_idx, uint16_t* gate, int32_t* csr, int32_t* pcsr,
                            cudaStream_t stream) {
  launch_pdl(fp8_identity_kernel, dim3(1), dim3(64), 0, stream, rows, inverse, top_idx, gate, csr, pcsr);
  return check_launch("fp8_identity");
}

}  // namespace praxis
