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
// Activation quantization
// ---------------------------------------------------------------------------
// Sixteen lanes take one block of 128 columns (8 columns, 16 bytes, each): the
// largest magnitude is four shuffles, and a warp reads 512 and writes 256
// contiguous bytes. Scales are stored block-major, scale[b * scale_ld + row]:
// the GEMM epilogue reads one block's scales of 32 consecutive rows at once.
// With `inverse` the block goes to the rows of the token's K routed slots
// (pcsr[e] + inverse - csr[e], as the dispatch laid them out), quantized once.
struct Fp8Rows {
  const int64_t* top_idx;  // [rows, top_k]; nullptr: row r goes to row r
  const int64_t* inverse;
  const int32_t* csr;
  const int32_t* pcsr;
  int32_t top_k;
  int32_t experts;
};

constexpr int kFp8QuantThreads = 256;

__global__ void __launch_bounds__(kFp8QuantThreads) fp8_quantize_kernel(
    const uint16_t* __restrict__ x, int64_t rows, int cols, int64_t ldx, Fp8Rows to, uint8_t* __restrict__ q,
    float* __restrict__ scale, int64_t scale_ld) {
  pdl_wait();  // the previous kernel of the stream has completed
  pdl_trigger();
  const int blocks = (cols + kFp8Block - 1) / kFp8Block;
  const int64_t total = rows * blocks;
  const int sub = threadIdx.x & 15;
  const int64_t step = (int64_t)gridDim.x * (kFp8QuantThreads / 16);
  // every lane of a warp makes the same number of turns (the shuffles below)
  const int64_t first = (int64_t)blockIdx.x * (kFp8QuantThreads / 16) + (threadIdx.x >> 4);
  const int64_t warp_first = (int64_t)blockIdx.x * (kFp8QuantThreads / 16) + (threadIdx.x >> 5) * 2;
  for (int64_t i = first, w = warp_first; w < total; i += step, w += step) {
    const bool live = i < total;
    const int64_t row = live ? i / blocks : 0;
    const int b = live ? (int)(i - row * blocks) : 0;
    const int col = b * kFp8Block + sub * 8;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (live && col < cols) v = ldg_stream(reinterpret_cast<const uint4*>(x + row * ldx + col));
    const float2 f[4] = {unpack_bf16x2(v.x), unpack_bf16x2(v.y), unpack_bf16x2(v.z), unpack_bf16x2(v.w)};
    float a = kFp8MinAmax;
#pragma unroll
    for (int j = 0; j < 4; ++j) a = fmaxf(a, fmaxf(fabsf(f[j].x), fabsf(f[j].y)));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    const float r = div_rn(kE4m3Max, a);
    const uint2 codes = make_uint2(cvt_e4m3x4(mul_rn(f[0].x, r), mul_rn(f[0].y, r), mul_rn(f[1].x, r), mul_rn(f[1].y, r)),
                                   cvt_e4m3x4(mul_rn(f[2].x, r), mul_rn(f[2].y, r), mul_rn(f[3].x, r), mul_rn(f[3].y, r)));
    if (!live) continue;
    const float s = div_rn(a, kE4m3Max);
    if (to.top_idx == nullptr) {
      if (col < cols) *reinterpret_cast<uint2*>(q + row * cols + col) = codes;
      if (sub == 0) scale[(int64_t)b * scale_ld + row] = s;
    } else {
      for (int j = 0; j < to.top_k; ++j) {
        const int64_t p = row * to.top_k + j;
        const int e = checked_expert(to.top_idx[p], to.experts);
        const int64_t dest = (int64_t)to.pcsr[e] + to.inverse[p] - to.csr[e];
        if (col < cols) *reinterpret_cast<uint2*>(q + dest * cols + col) = codes;
        if (sub == 0) scale[(int64_t)b * scale_ld + dest] = s;
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
// GEMM on tcgen05, 128 x 256 of the output per CTA (CTAS = 1) or 256 x 256 per
// CTA pair (CTAS = 2, cta_group::2: each CTA holds its 128 rows and half of
// the weight rows, so a k-block brings 32 KB per SM instead of 48).
//
// warp 0      TMA producer: per k-block of 128 columns the A rows and the
//             weight rows in boxes of 64 rows (128-byte swizzle)
// warp 1      MMA issuer (leader CTA): per k-block two MMA groups of 128
//             columns ("halves"), each into one of its two tensor-memory
//             buffers: 4 x 128 columns are all 512
// warps 4..11 epilogue: half h = (warp - 4) / 4 belongs to four warps, one per
//             lane quadrant. Per k-block a thread reads the 128 columns of its
//             row in four loads, the next in flight while it adds the last,
//             times sx * sw, to 128 registers. A buffer is free again as soon
//             as it is read, 3 MMA groups (768 clocks) before the issuer needs
//             it.
//
// Bound: 128 x 256 x 128 products are 512 clocks of one SM's tensor core; the
// FMAs of the 128 x 256 block sums are 256 clocks of its fp32 lanes.
// ---------------------------------------------------------------------------
enum Fp8Mode : int { FP8_PLAIN = 0, FP8_SWIGLU = 1 };

struct Fp8GemmParams {
  CUtensorMap tmap_a;    // activation codes [rows, K], boxes of 128 rows
  CUtensorMap tmap_b;    // weight codes [E * N, K], boxes of 128 rows
  CUtensorMap tmap_out;  // bf16 output [rows, N], boxes of 32 rows x 64 columns (FP8_PLAIN, N % 8 == 0)
  const float* xs;       // activation scales, [K blocks][xs_ld]
  int64_t xs_ld;
  const float* ws;       // weight scales [E][N blocks][K blocks]
  const TileEntry* tiles;    // grouped: table of 128-row tiles (CTAS = 1) or 256-row pairs; nullptr: dense rows
  const int32_t* num_tiles;
  int64_t rows;          // rows of the activations and of the output
  int32_t N;             // weight rows per expert (2F for FP8_SWIGLU)
  int32_t K;
  int32_t experts;
  uint16_t* out;         // FP8_PLAIN: [rows, N]
  int32_t tma_out;
  uint8_t* hq;           // FP8_SWIGLU: hidden codes [rows, N / 2]
  float* hs;             // FP8_SWIGLU: hidden scales, [N / 256][hs_ld]
  int64_t hs_ld;
};

template <int CTAS>
struct Fp8Shape {
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = 256 / CTAS * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = CTAS == 2 ? 6 : 4;
  static constexpr int EPI_WARPS = 8;
  static constexpr int OUT_BOX = 4096;  // 32 rows x 64 bf16 per epilogue warp
  // Registers: 12 warps launch with 168 each (64512 in all); the four warps
  // of the producer and the issuer give some back, and the epilogue's 128
  // sums and two 32-column loads in flight fit without spilling.
  static constexpr int EPI_WARP0 = 4;
  static constexpr int THREADS = 32 * (EPI_WARP0 + EPI_WARPS);
  static constexpr int LAUNCH_REGS = 168, FRONT_REGS = 40, EPI_REGS = 232;
  static_assert(32 * EPI_WARP0 * FRONT_REGS + 32 * EPI_WARPS * EPI_REGS <= THREADS * LAUNCH_REGS, "register split");
  static constexpr size_t SMEM_BYTES = 1024 + (size_t)STAGES * STAGE_BYTES + EPI_WARPS * OUT_BOX + 256;
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

// E4M3 x E4M3 -> F32 (kind::f8f6f4), K-major operands, K = 32 per MMA.
__host__ __device__ constexpr uint32_t idesc_e4m3(uint32_t m, uint32_t n) {
  return (1u << 4)            // D format: F32
         | ((n >> 3) << 17)   // N / 8 (A and B format 0: E4M3)
         | ((m >> 4) << 24);  // M / 16
}

// The high word of a descriptor is the same for every operand here; the low
// word (the address) moves by 2 per 32 bytes.
template <int CTAS, int ACCUMULATE>
__device__ __forceinline__ void tc_mma_e4m3(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi,
                                            uint32_t idesc) {
  if constexpr (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "n"(ACCUMULATE)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "n"(ACCUMULATE)
        : "memory");
}

template <int CTAS>
__device__ __forceinline__ void fp8_commit(uint64_t* bar) {
  if constexpr (CTAS == 1) tc_commit(bar);
  else tc_commit_pair(bar, 0x3);
}

// acc[0..7] += f * (the 16 columns in r), one FMA each. The statements are
// volatile, so they stay behind the wait for the loads of r.
__device__ __forceinline__ void fp8_add_block(uint64_t* acc, const uint32_t (&r)[16], float f) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    asm volatile(
        "{\n\t.reg .b64 d, s;\n\tmov.b64 d, {%1, %2};\n\tmov.b64 s, {%3, %3};\n\t"
        "fma.rn.f32x2 %0, d, s, %0;\n\t}"
        : "+l"(acc[j])
        : "r"(r[2 * j]), "r"(r[2 * j + 1]), "f"(f));
}
__device__ __forceinline__ float2 unpack_f32x2(uint64_t v) {
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// mbar_wait (common.cuh) that looks at the clock only every 64 tries: a wait
// per k-block and role is on the path of every MMA here, and the first read of
// %globaltimer alone costs about as much as a k-block's products.
__device__ __forceinline__ bool fp8_wait(uint64_t* bar, uint32_t parity, unsigned int code,
                                         uint64_t limit_ns = 2000000000ull, bool stop_on_error = true) {
  uint64_t start = 0;
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) == 0u) {
      if (stop_on_error && error_raised()) return false;
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
template <int CTAS>
__device__ __forceinline__ TileEntry fp8_tile(const Fp8GemmParams& p, int m) {
  if (p.tiles != nullptr) {
    TileEntry t = p.tiles[m];
    if (CTAS == 1) t.pad = kTileRows;  // rows that may be stored
    return t;
  }
  TileEntry t;
  t.expert = 0;
  t.row0 = m * CTAS * kTileRows;
  t.valid = (int32_t)min((int64_t)CTAS * kTileRows, p.rows - t.row0);
  t.pad = t.valid;
  return t;
}

// g / (1 + exp(-g)) * u
__device__ __forceinline__ float swiglu_f32(float g, float u) {
  return __fdividef(1.0f, 1.0f + __expf(-g)) * g * u;
}

// Tensor-memory column of a thread's chunk c of 16 columns, from its first.
template <int MODE>
__device__ constexpr uint32_t chunk_col(int c) {
  return 16 * c + (MODE == FP8_SWIGLU && c >= 4 ? 64 : 0);
}

template <int CTAS, int MODE>
__device__ __forceinline__ void fp8_gemm_body(const Fp8GemmParams& p) {
  pdl_wait();  // the previous kernel of the stream has completed
  pdl_trigger();
  using S = Fp8Shape<CTAS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + S::STAGES * S::A_BYTES;
  uint8_t* sOut = sB + S::STAGES * S::B_BYTES;  // output boxes; FP8_SWIGLU: row maxima [2 units][2 halves][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + S::EPI_WARPS * S::OUT_BOX);
  uint64_t* empty = full + S::STAGES;
  uint64_t* acc_full = empty + S::STAGES;  // per buffer
  uint64_t* acc_empty = acc_full + 2;      // per buffer, the leader's
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t rank = CTAS == 1 ? 0u : cluster_ctarank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], S::EPI_WARPS * CTAS);
    }
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.tmap_a);
    tma_prefetch_desc(&p.tmap_b);
  }
  if (warp == 1) {
    if constexpr (CTAS == 1) {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    } else {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    }
  }
  __syncwarp();
  tc_fence_before();
  if constexpr (CTAS == 1) __syncthreads();
  else cluster_sync();  // barriers of both CTAs initialised before any cross-CTA signal
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int F = p.N / 2;
  const int n_tiles = MODE == FP8_SWIGLU ? F / 128 : (p.N + 255) / 256;
  const int num_m =
      p.tiles != nullptr ? p.num_tiles[CTAS - 1] : (int)((p.rows + CTAS * kTileRows - 1) / (CTAS * kTileRows));
  const int total = num_m * n_tiles;
  const int k_blocks = (p.K + kFp8Block - 1) / kFp8Block;
  const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;

  if (warp < S::EPI_WARP0) {
    regs_down<S::FRONT_REGS>();
    if (warp == 0 && lane == 0) {
      // ---------------- TMA producer (every CTA) ----------------
      const uint32_t full_leader = CTAS == 1 ? 0u : mapa_shared(smem_u32(full), 0);
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int u = first; u < total && ok; u += step) {
        const int m = u / n_tiles, n = u - m * n_tiles;
        const TileEntry t = fp8_tile<CTAS>(p, m);
        const int a_row = t.row0 + 128 * (int)rank;
        // the weight rows of columns 0..127 (leader) and 128..255 (its peer)
        const int b_row = t.expert * p.N + (MODE == FP8_SWIGLU ? n * 128 : n * 256);
        const int b_up = MODE == FP8_SWIGLU ? F : 128;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!fp8_wait(&empty[stage], phase ^ 1u, kErrTimeoutProducer)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], CTAS * S::STAGE_BYTES);
          uint8_t* a = sA + stage * S::A_BYTES;
          uint8_t* b = sB + stage * S::B_BYTES;
          if constexpr (CTAS == 1) {
            tma_load_2d(a, &p.tmap_a, &full[stage], kb * 128, a_row);
            tma_load_2d(b, &p.tmap_b, &full[stage], kb * 128, b_row);
            tma_load_2d(b + 16384, &p.tmap_b, &full[stage], kb * 128, b_row + b_up);
          } else {
            const uint32_t fb = full_leader + stage * 8;
            tma_load_2d_pair(a, &p.tmap_a, fb, kb * 128, a_row);
            tma_load_2d_pair(b, &p.tmap_b, fb, kb * 128, b_row + (int)rank * b_up);
          }
          if (++stage == S::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // after an error the copies in flight still land before the CTA ends
      if (!ok && rank == 0)
        for (uint32_t s = 0; s < S::STAGES; ++s)
          fp8_wait(&full[s], s < stage ? phase : phase ^ 1u, kErrTimeoutProducer, 50000000ull, false);
    } else if (warp == 1 && lane == 0 && rank == 0) {
      // ---------------- MMA issuer (leader) ----------------
      constexpr uint32_t idesc = idesc_e4m3(128 * CTAS, 256);
      const uint64_t a_desc = smem_desc(smem_u32(sA), 16, 1024, kLayoutSwizzle128B);
      const uint32_t desc_hi = (uint32_t)(a_desc >> 32), a_lo = (uint32_t)a_desc;
      const uint32_t b_lo = (uint32_t)smem_desc(smem_u32(sB), 16, 1024, kLayoutSwizzle128B);
      uint32_t stage = 0, phase = 0, cnt = 0;
      bool ok = true;
      for (int u = first; u < total && ok; u += step) {
        for (int kb = 0; kb < k_blocks && ok; ++kb, ++cnt) {
          const uint32_t buf = cnt & 1u, buf_phase = (cnt >> 1) & 1u;
          ok = fp8_wait(&full[stage], phase, kErrTimeoutMma);
          if (!ok) break;
          const uint32_t a = a_lo + stage * (S::A_BYTES >> 4), b = b_lo + stage * (S::B_BYTES >> 4);
          ok = fp8_wait(&acc_empty[buf], buf_phase ^ 1u, kErrTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + buf * 256;
          tc_mma_e4m3<CTAS, 0>(d, a, b, desc_hi, idesc);
          tc_mma_e4m3<CTAS, 1>(d, a + 2, b + 2, desc_hi, idesc);
          tc_mma_e4m3<CTAS, 1>(d, a + 4, b + 4, desc_hi, idesc);
          tc_mma_e4m3<CTAS, 1>(d, a + 6, b + 6, desc_hi, idesc);
          fp8_commit<CTAS>(&acc_full[buf]);
          fp8_commit<CTAS>(&empty[stage]);
          if (++stage == S::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else {
    regs_up<S::EPI_REGS>();
    // ---------------- epilogue (warps 4..11, every CTA) ----------------
    // After a wait that gave up the warps go through the remaining units
    // without waiting or storing, so that the named barriers stay matched.
    const uint32_t quad = (uint32_t)(warp & 3);
    const int h = (warp - S::EPI_WARP0) >> 2;
    const int row_in_cta = (int)(quad * 32 + lane);
    const uint32_t acc_empty_leader = CTAS == 1 ? 0u : mapa_shared(smem_u32(acc_empty), 0);
    // SwiGLU: 64 gate columns and the up columns 128 further on; else 128 in a row
    const uint32_t taddr = tmem + ((quad * 32u) << 16) + (MODE == FP8_SWIGLU ? 64u : 128u) * h;
    uint8_t* box = sOut + (warp - S::EPI_WARP0) * S::OUT_BOX;
    const int n_blocks = (p.N + kFp8Block - 1) / kFp8Block;
    uint32_t cnt = 0, unit = 0;
    bool ok = true;
    for (int u = first; u < total; u += step, ++unit) {
      const int m = u / n_tiles, n = u - m * n_tiles;
      const TileEntry t = fp8_tile<CTAS>(p, m);
      const int row_in_tile = row_in_cta + 128 * (int)rank;
      const int64_t row = (int64_t)t.row0 + row_in_tile;
      const float* xs = p.xs + min(row, p.rows - 1);
      // the weight scales of this thread's columns: one row of blocks, or the
      // gate's (columns 0..63) and the up's (64..127)
      const int nb0 = MODE == FP8_SWIGLU ? n : min(2 * n + h, n_blocks - 1);
      const int nb1 = MODE == FP8_SWIGLU ? n + F / 128 : nb0;
      const float* ws0 = p.ws + ((int64_t)t.expert * n_blocks + nb0) * k_blocks;
      const float* ws1 = p.ws + ((int64_t)t.expert * n_blocks + nb1) * k_blocks;
      uint64_t acc[64];  // two neighbouring columns each
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0;
      float f0 = __ldg(xs) * __ldg(ws0), f1 = MODE == FP8_SWIGLU ? __ldg(xs) * __ldg(ws1) : f0;
      uint32_t ra[16], rb[16];
      ok = ok && fp8_wait(&acc_full[cnt & 1u], (cnt >> 1) & 1u, kErrTimeoutEpilogue);
      tc_fence_after();
      tc_ld_32x32b_x16(taddr + (cnt & 1u) * 256, ra);
      for (int kb = 0; kb < k_blocks; ++kb, ++cnt) {
        const uint32_t buf = cnt & 1u, tb = taddr + buf * 256;
        float sx = 0.0f, w0 = 0.0f, w1 = 0.0f;
        if (kb + 1 < k_blocks) {
          sx = __ldg(xs + (int64_t)(kb + 1) * p.xs_ld);
          w0 = __ldg(ws0 + kb + 1);
          if (MODE == FP8_SWIGLU) w1 = __ldg(ws1 + kb + 1);
        }
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
          const float f = c < 4 ? f0 : f1;
          tc_wait_ld();
          tc_ld_32x32b_x16(tb + chunk_col<MODE>(c + 1), rb);
          fp8_add_block(acc + 8 * c, ra, f);
          if (c == 6) break;
          tc_wait_ld();
          tc_ld_32x32b_x16(tb + chunk_col<MODE>(c + 2), ra);
          fp8_add_block(acc + 8 * (c + 1), rb, f);
        }
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CTAS == 1 || rank == 0) mbar_arrive(&acc_empty[buf]);
          else mbar_arrive_cluster(acc_empty_leader + buf * 8);
        }
        if (kb + 1 < k_blocks) {
          const uint32_t next = cnt + 1;
          ok = ok && fp8_wait(&acc_full[next & 1u], (next >> 1) & 1u, kErrTimeoutEpilogue);
          tc_fence_after();
          tc_ld_32x32b_x16(taddr + (next & 1u) * 256, ra);
        }
        fp8_add_block(acc + 56, rb, f1);
        f0 = sx * w0;
        f1 = MODE == FP8_SWIGLU ? sx * w1 : f0;
      }
      if constexpr (MODE == FP8_SWIGLU) {
        // 64 hidden columns 128 n + 64 h ..; the other half's warps hold the
        // rest of the row's block, so the row maxima meet in shared memory
        float a = kFp8MinAmax;
        float2 hid[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float2 g = unpack_f32x2(acc[j]), v = unpack_f32x2(acc[32 + j]);
          hid[j] = make_float2(swiglu_f32(g.x, v.x), swiglu_f32(g.y, v.y));
          a = fmaxf(a, fmaxf(fabsf(hid[j].x), fabsf(hid[j].y)));
        }
        float* s_max = reinterpret_cast<float*>(sOut) + (unit & 1u) * 256;
        s_max[h * 128 + row_in_cta] = a;
        named_sync(1, 32 * S::EPI_WARPS);
        a = fmaxf(a, s_max[(h ^ 1) * 128 + row_in_cta]);
        if (ok && row_in_tile < t.valid) {
          const float r = div_rn(kE4m3Max, a);
          uint4* dst = reinterpret_cast<uint4*>(p.hq + row * F + n * 128 + 64 * h);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 v0 = hid[8 * j + 2 * i], v1 = hid[8 * j + 2 * i + 1];
              c[i] = cvt_e4m3x4(mul_rn(v0.x, r), mul_rn(v0.y, r), mul_rn(v1.x, r), mul_rn(v1.y, r));
            }
            dst[j] = make_uint4(c[0], c[1], c[2], c[3]);
          }
          if (h == 0) p.hs[(int64_t)n * p.hs_ld + row] = div_rn(a, kE4m3Max);
        }
      } else {
        const int col0 = n * 256 + 128 * h;
        if (p.tma_out) {
          // two boxes of 32 rows x 64 columns in the TMA 128-byte swizzle; a
          // table's tile is stored whole (its padding rows are scratch)
          const int live = t.pad - 128 * (int)rank - 32 * (int)quad;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (lane == 0) bulk_wait_group_read0();
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 v = unpack_f32x2(acc[i * 32 + c * 4 + j]);
                w[j] = cvt_bf16x2(v.x, v.y);
              }
              *reinterpret_cast<uint4*>(box + lane * 128 + ((c ^ (lane & 7)) << 4)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0 && ok && live > 0 && col0 + 64 * i < p.N) {
              tma_store_2d(&p.tmap_out, box, col0 + 64 * i, t.row0 + 128 * (int)rank + 32 * (int)quad);
              bulk_commit_group();
            }
          }
        } else if (ok && row_in_tile < t.valid) {
          // rows of N bf16 that are not multiples of 16 bytes
          uint16_t* dst = p.out + row * p.N + col0;
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            const float2 v = unpack_f32x2(acc[j]);
            if (col0 + 2 * j < p.N) dst[2 * j] = f32_to_bf16(v.x);
            if (col0 + 2 * j + 1 < p.N) dst[2 * j + 1] = f32_to_bf16(v.y);
          }
        }
      }
    }
    if (MODE == FP8_PLAIN && lane == 0) bulk_wait_group0();
  }

  __syncwarp();
  tc_fence_before();
  if constexpr (CTAS == 1) __syncthreads();
  else cluster_sync();  // all tensor-memory reads and cross-CTA signals of the pair done
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CTAS == 1) tmem_dealloc(tmem, 512);
    else tmem_dealloc_pair(tmem, 512);
  }
}

template <int MODE>
__global__ void __launch_bounds__(Fp8Shape<1>::THREADS, 1) fp8_gemm_kernel(const __grid_constant__ Fp8GemmParams p) {
  fp8_gemm_body<1, MODE>(p);
}

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Fp8Shape<2>::THREADS, 1)
    fp8_gemm_pair_kernel(const __grid_constant__ Fp8GemmParams p) {
  fp8_gemm_body<2, MODE>(p);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static int fp8_map(CUtensorMap* map, CUtensorMapDataType type, int elem, const void* base, int64_t rows, int64_t cols,
                   int box_cols, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return set_error(PRAXIS_B200_ECUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t gdim[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t gstride[1] = {(cuuint64_t)cols * elem};
  cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  cuuint32_t estride[2] = {1u, 1u};
  CUresult r = fn(map, type, 2, const_cast<void*>(base), gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(PRAXIS_B200_ECUDA, "cuTensorMapEncodeTiled (fp8) failed (%d)", (int)r);
  return PRAXIS_B200_OK;
}

// Launches on at most one CTA (pair) per SM; `units` bounds the work.
template <int CTAS, int MODE>
static int fp8_launch(const Fp8GemmParams& p, int64_t units, cudaStream_t stream) {
  using S = Fp8Shape<CTAS>;
  auto kernel = [] {
    if constexpr (CTAS == 1) return fp8_gemm_kernel<MODE>;
    else return fp8_gemm_pair_kernel<MODE>;
  }();
  static DeviceOnce attr;
  static int max_groups[kMaxDevices] = {0};
  const int rc = device_once(attr, [&](int dev) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM_BYTES);
    if (e != cudaSuccess)
      return set_error(PRAXIS_B200_ECUDA, "fp8 gemm smem attribute (device %d): %s", dev, cudaGetErrorString(e));
    // setmaxnreg waits for registers that the launch does not have
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, kernel);
    if (e != cudaSuccess || fa.numRegs < S::LAUNCH_REGS)
      return set_error(PRAXIS_B200_ECUDA, "fp8 gemm: built with %d registers a thread, needs %d", fa.numRegs,
                       S::LAUNCH_REGS);
    int n = sm_count();
    if (CTAS == 2) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2 * (sm_count() / 2));
      cfg.blockDim = dim3(S::THREADS);
      cfg.dynamicSmemBytes = S::SMEM_BYTES;
      cudaLaunchAttribute a;
      a.id = cudaLaunchAttributeClusterDimension;
      a.val.clusterDim.x = 2;
      a.val.clusterDim.y = 1;
      a.val.clusterDim.z = 1;
      cfg.attrs = &a;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
      if (e != cudaSuccess || n <= 0) n = sm_count() / 2;
    }
    max_groups[dev] = n;
    return (int)PRAXIS_B200_OK;
  });
  if (rc) return rc;
  int dev = 0;
  cudaGetDevice(&dev);
  const int groups = (int)(units < max_groups[dev] ? units : max_groups[dev]);
  launch_pdl(kernel, dim3(CTAS * groups), dim3(S::THREADS), S::SMEM_BYTES, stream, p);
  return check_launch("fp8_gemm");
}

int run_fp8_quantize(const uint16_t* x, int64_t rows, int cols, int64_t ldx, const Fp8Rows& to, uint8_t* q,
                     float* scale, int64_t scale_ld, cudaStream_t stream) {
  if (rows == 0) return PRAXIS_B200_OK;
  const int64_t blocks = rows * ((cols + kFp8Block - 1) / kFp8Block);
  int64_t grid = (blocks + kFp8QuantThreads / 16 - 1) / (kFp8QuantThreads / 16);
  const int64_t most = (int64_t)sm_count() * 8;
  if (grid > most) grid = most;
  launch_pdl(fp8_quantize_kernel, dim3((unsigned)grid), dim3(kFp8QuantThreads), 0, stream, x, rows, cols, ldx, to, q,
             scale, scale_ld);
  return check_launch("fp8_quantize");
}

int run_fp8_pack(const uint16_t* w, int64_t experts, int64_t k, int64_t n, uint8_t* q, float* scale,
                 cudaStream_t stream) {
  const int64_t blocks = experts * ((n + kFp8Block - 1) / kFp8Block) * ((k + kFp8Block - 1) / kFp8Block);
  if (blocks == 0) return PRAXIS_B200_OK;
  fp8_pack_kernel<<<(unsigned)blocks, 256, 0, stream>>>(w, k, n, q, scale);
  return check_launch("fp8_pack");
}

// One GEMM over quantized rows. Dense (tiles == nullptr): `rows` rows against
// one weight. Grouped: the dispatch's tables, rows = padded rows, max_tiles
// bounds the 128-row tiles and mean_rows is the mean number of routed rows per
// expert. out (FP8_PLAIN) or hq / hs (FP8_SWIGLU) get the result.
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
  int64_t mean_rows;
  uint16_t* out;
  uint8_t* hq;
  float* hs;
  int64_t hs_ld;
};

int run_fp8_gemm(const Fp8Gemm& g, cudaStream_t stream) {
  if (g.rows == 0) return PRAXIS_B200_OK;
  Fp8GemmParams p;
  memset(&p, 0, sizeof(p));
  int rc = fp8_map(&p.tmap_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.q, g.rows, g.k, 128, 128);
  if (rc) return rc;
  rc = fp8_map(&p.tmap_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.wq, (int64_t)g.experts * g.n, g.k, 128, 128);
  if (rc) return rc;
  const bool swiglu = g.out == nullptr;
  if (!swiglu && g.n % 8 == 0 && ((uintptr_t)g.out & 15) == 0) {
    rc = fp8_map(&p.tmap_out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, g.out, g.rows, g.n, 64, 32);
    if (rc) return rc;
    p.tma_out = 1;
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
  const int64_t n_tiles = swiglu ? g.n / 256 : (g.n + 255) / 256;
  const bool pair = g.tiles != nullptr ? g.mean_rows >= 256 : (g.rows + 255) / 256 * n_tiles >= sm_count() / 2;
  p.tiles = g.tiles == nullptr ? nullptr : pair ? g.tiles + g.max_tiles : g.tiles;
  const int64_t m_tiles = g.tiles != nullptr ? g.max_tiles : (g.rows + (pair ? 255 : 127)) / (pair ? 256 : 128);
  const int64_t units = m_tiles * n_tiles;
  if (swiglu)
    return pair ? fp8_launch<2, FP8_SWIGLU>(p, units, stream) : fp8_launch<1, FP8_SWIGLU>(p, units, stream);
  return pair ? fp8_launch<2, FP8_PLAIN>(p, units, stream) : fp8_launch<1, FP8_PLAIN>(p, units, stream);
}

}  // namespace praxis
