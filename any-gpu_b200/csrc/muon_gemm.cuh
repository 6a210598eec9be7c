// The products of the Newton-Schulz iteration on tcgen05 (kind::f16), at
// fp32-level accuracy, for a group of matrices of any shapes in one launch.
//
// Split operands.  Every matrix of the iteration is kept as two fp16 planes,
// x 2^e = hi + lo 2^-11 with hi = fp16(x 2^e) and lo = fp16((x 2^e - hi) 2^11):
// 22 bits of each value in the 4 bytes a float takes.  The iteration bounds its
// values (|X| <= 1.21, |A| <= 1.46, |a I + b A + c A A| <= 3.45 in the 2-norm,
// so every entry too), and e is the power of two that brings this bound just
// below fp16's largest value; lo is as large as hi, so both leave fp16's normal
// range only for entries below 2^-28.  (With lo unscaled that began at 2^-18:
// rows 1e-5 of the others came out 2e-5 to 1e-4 off, where fp32 keeps 4e-6.)
// A product is three MMAs into one fp32 accumulator, (lo hi + hi lo) 2^-11 +
// hi hi, the shift being an operand of the MMA that follows the small terms (lo
// lo is below 2^-22), at the fp16 rate, twice tf32's: half the time of the
// 3xTF32 GEMM (umma2_x3_kernel.cuh), which also has to split its operands in a
// pass of its own.  Here the epilogue that produces a matrix writes it split,
// so operands go from global memory through TMA to the tensor core as they are.
//
// Segments.  The tensor core's fp32 sum truncates, an error that grows with
// the number of MMAs summed (a K loop of 1024 in the 3xTF32 GEMM's segments of
// 512 left 2.6e-5 after five steps, where fp32 FMAs leave 1e-6).  So an
// accumulator takes K = 64 kSeg, small terms first, and the epilogue warps add
// it, rounding to nearest, to a sum in registers while the tensor core fills
// the other one.
//
// Symmetry.  A X X^T and products of commuting symmetric matrices are
// symmetric: only 256 x 256 blocks on and below the diagonal are computed and
// stored.  Whoever reads such a matrix takes a block above the diagonal from its mirror
// image, as an MN-major operand instead of a K-major one (the descriptors and
// the instruction's major bits change, the shared memory's size does not), so
// nothing is stored twice.
//
// Tiles.  BN x BN outputs: 256 x 256 by a CTA pair (cta_group::2), or
// 128 x 128 by one CTA for products with few tiles.  Either way a stage holds, per
// CTA, both planes of 128 rows of A and 128 of B by 64 of K: 64 KB, three
// stages.
//
//   warp 0      TMA of the CTA's halves (no multicast)
//   warp 1      tensor memory; one lane of the leader CTA issues the MMAs
//   warps 4-11  epilogue: warp w owns 32 rows (w % 4) of half the columns, its
//               sums in registers (128 of the 232 it takes over from warps 0-3)
//
// Bound by the tensor core: three symmetric products of 4096^3 take 465 us, 1413
// TFLOP/s of MMAs, 0.85 of the measured fp16 rate; products with X (4096 x 45312
// together) 3.24 ms, 1408.  In a long run the power limit takes the clock to
// 1.3 GHz.  One wave of small tiles is bound by its ends: seven products of
// 1024^3 take 37 us, of which 20 are MMAs.  The shift of the small terms costs
// 0.5 to 2.5% of a product.
//
// Every wait is bounded as in umma2_kernel.cuh.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace agpu {
namespace muon {

constexpr int kBlock = 256;      // blocks of a symmetric matrix: whole ones are stored
constexpr int kBK = 64;          // fp16 elements of K per stage: one 128-byte row
constexpr int kSeg = 1;          // K-blocks summed by one accumulator
static_assert(kSeg == 1, "the small terms of an accumulator come before its hi hi");
constexpr int kStages = 3;
constexpr int kEpi = 8;          // epilogue warps
constexpr int kPlane = 128 * 128;          // bytes of one plane of an operand tile
constexpr int kOperand = 2 * kPlane;       // hi and lo
constexpr int kStage = 2 * kOperand;       // A and B
constexpr int kStaging = 4096;             // bytes per epilogue warp
constexpr int kSmem = 1024 + kStages * kStage + kEpi * kStaging + 256;
constexpr int kThreads = 128 + 32 * kEpi;
// Registers: 168 a thread at launch (384 threads), then 40 for warps 0-3 and
// 232 for the epilogue: 128 * 40 + 256 * 232 = 384 * 168.  Spills as
// ptxas reports them: 108 bytes of stores and 184 of loads with pair tiles, 20
// and 36 with single ones.
constexpr int kRegsLow = 40, kRegsHigh = 232;
// Matrices per launch.  They travel as kernel parameters, 640 bytes each;
// launches of at most kFewItems keep below 4 KB.
constexpr int kMaxItems = 24, kFewItems = 6;

// Coefficients of the quintic and the exponents of the split matrices.
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kXScale = 32768.0f;  // X and A = X X^T
constexpr float kMScale = 16384.0f;  // a I + b A + c A A
constexpr int kLoShift = 11;          // lo = fp16((x - hi) 2^11)
// What the tensor core's truncation takes from an accumulator on average: half
// a unit in the last place (0.72 2^-24 of the value) for each of the n MMAs of
// full size, at partial sums of half the final value: 0.36 n 2^-24, that is
// 0.7 2^-23 for the n = 4 of a segment (measured: 0.8 to 1.0e-7, alike in every
// product).  Alike in all elements, such an error is amplified by the
// iteration; rounded to a factor a float can hold it is put back.  It is the
// average for that n: one dominant term loses more the earlier it comes (0.72
// 2^-24 for each MMA behind it), and the on-chip kernel, whose accumulators take up to
// 16, uses the same factor.  What that leaves is 1e-7 of a product.
constexpr float kUntruncate = 1.0f + 0x1p-23f;

// Operands and result of a product, with P = scale * (A B):
enum class Mode {
  Gram,   // A = B = X: out = P, symmetric
  Poly,   // A = B symmetric: out = a I + b g + P, symmetric
  Mul,    // A, B symmetric and commuting: out = P, symmetric
  Step,   // A symmetric, B = X: out = P
  Update  // A symmetric, B = X: w = decay * w + gain * (A B), fp32
};

struct Item {
  // tiles of A and B with K along their rows, and across them (a block above
  // the diagonal of a symmetric operand; X as B of Step and Update)
  CUtensorMap a, at, b, bt;
  int m, n, k;             // out [m, n], contraction k
  int tiles_m, tiles_n, first;  // first: this item's first tile
  __half* out;             // hi plane; the others follow, `plane` elements apart
  const __half* g;         // split like out
  long long plane;         // of out and g
  int ld;                  // of out and g: a multiple of 64
  float scale;
  float* w;                // [m, n] or, if w_transposed, [n, m]
  float decay, gain;
  int w_transposed;
  int part;                // out is a part of a sum: floats, not split (as_halves)
};

template <int CAP>
struct Items {
  Item item[CAP];
  int count, tiles;
  Mode mode;
};

__host__ __device__ constexpr bool symmetric_out(Mode m) {
  return m == Mode::Gram || m == Mode::Poly || m == Mode::Mul;
}

struct Tile {
  int item, m0, n0;
};

template <int BN, int CAP>
__device__ __forceinline__ Tile tile_at(const Items<CAP>& g, int t) {
  Tile r;
  r.item = 0;
  while (r.item + 1 < g.count && t >= g.item[r.item + 1].first) ++r.item;
  const Item& it = g.item[r.item];
  const int q = t - it.first;
  if (symmetric_out(g.mode)) {  // blocks of the lower triangle by rows, (kBlock / BN)^2 tiles each
    constexpr int S = kBlock / BN;
    const int blk = q / (S * S), sub = q % (S * S);
    int i = (int)((sqrtf(8.0f * (float)blk + 1.0f) - 1.0f) * 0.5f);
    while (i * (i + 1) / 2 > blk) --i;
    while ((i + 1) * (i + 2) / 2 <= blk) ++i;
    r.m0 = i * kBlock + sub / S * BN;
    r.n0 = (blk - i * (i + 1) / 2) * kBlock + sub % S * BN;
  } else {  // groups of 16 row tiles, rows fastest: B's column block stays in L2
    constexpr int G = 16;
    const int span = G * it.tiles_n;
    const int first_m = (q / span) * G;
    const int size = min(it.tiles_m - first_m, G);
    r.m0 = (first_m + (q % span) % size) * BN;
    r.n0 = ((q % span) / size) * BN;
  }
  return r;
}

// K-blocks of a tile (none outside the matrix: a part of a diagonal block).
__device__ __forceinline__ int k_blocks(const Item& it, const Tile& t) {
  return t.m0 < it.m && t.n0 < it.n ? (it.k + kBK - 1) / kBK : 0;
}

// hi and lo of two scaled values, packed.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  float2 r;  // (x - hi) 2^11, exact, as x 2^11 - hi 2^11 on two floats at once
  asm("{\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 a, a, %6;\n\tfma.rn.f32x2 a, b, %7, a;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x), "f"(y), "f"(f.x), "f"(f.y), "l"(0x4500000045000000ull),
        "l"(0xc5000000c5000000ull));
  static_assert(kLoShift == 11, "the constants are 2048 and -2048, twice");
  const __half2 l = __floats2half2_rn(r.x, r.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Parts of a sum stay floats: the upper halves of two of them, and the lower
// halves, packed, in the two planes that hi and lo would take.
__device__ __forceinline__ void as_halves(float x, float y, uint32_t& upper, uint32_t& lower) {
  upper = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
  lower = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x5410);
}
__device__ __forceinline__ void from_halves(uint32_t upper, uint32_t lower, float& x, float& y) {
  x = __uint_as_float(__byte_perm(lower, upper, 0x5410));
  y = __uint_as_float(__byte_perm(lower, upper, 0x7632));
}

// The epilogue takes a warp's 32 rows in blocks of 64 columns, the next one
// always in v[0..63]: a loop, not code unrolled over all 128 columns, and one
// kernel for all modes.  A tile's 128 KB per CTA leave in 5,500 cycles when all
// CTAs store at once (3.4 KB a cycle, what L2 takes); with a kernel per mode and
// unrolled code the first tile of a launch took 13,000, waiting for
// instructions, and blocks of 32 columns (64-byte runs) 11,000.
//
// A plane of a block passes through 4 KB of shared memory per warp, a 128-byte
// line per row in 16-byte pieces, piece j of line r at j ^ (r % 8), so that
// neither rows nor lines conflict on banks.
__device__ __forceinline__ uint8_t* piece(uint8_t* stg, int line, int j) {
  return stg + line * 128 + ((j ^ (line & 7)) << 4);
}

// One plane of a block, a row per thread, to global memory by lines.
__device__ __forceinline__ void store_plane(const uint32_t (&h)[32], uint8_t* stg, int lane,
                                            __half* out, int ld, int rows) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<uint4*>(piece(stg, lane, j)) =
        make_uint4(h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]);
  __syncwarp();
  out += (long long)(lane >> 3) * ld + (lane & 7) * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int line = i * 4 + (lane >> 3);
    const uint4 d = *reinterpret_cast<uint4*>(piece(stg, line, lane & 7));
    if (line < rows) *reinterpret_cast<uint4*>(out + (long long)i * 4 * ld) = d;
  }
  __syncwarp();
}

// One plane of a block of g, loaded by lines ahead of its use (lines behind the
// last row repeat it: their sums are not stored).
struct Block {
  uint4 d[8];
};

__device__ __forceinline__ void load_block(Block& b, int lane, const __half* g, int ld,
                                           int rows) {
  g += (long long)(lane >> 3) * ld + (lane & 7) * 8;
  if (rows >= 32) {  // loads that no condition selects: all in flight at once
#pragma unroll
    for (int i = 0; i < 8; ++i)
      b.d[i] = *reinterpret_cast<const uint4*>(g + (long long)i * 4 * ld);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      b.d[i] = make_uint4(0, 0, 0, 0);
      if (i * 4 + (lane >> 3) < rows)
        b.d[i] = *reinterpret_cast<const uint4*>(g + (long long)i * 4 * ld);
    }
  }
}

__device__ __forceinline__ void put_block(const Block& b, uint8_t* stg, int lane) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<uint4*>(piece(stg, i * 4 + (lane >> 3), lane & 7)) = b.d[i];
  __syncwarp();
}

// v += f * the staged block.
__device__ __forceinline__ void add_block(float* v, float f, uint8_t* stg, int lane) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint4 d = *reinterpret_cast<const uint4*>(piece(stg, lane, j));
    const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[8 * j + 2 * i] = fmaf(f, x.x, v[8 * j + 2 * i]);
      v[8 * j + 2 * i + 1] = fmaf(f, x.y, v[8 * j + 2 * i + 1]);
    }
  }
  __syncwarp();
}

// w = decay w + gain v for 32 x 32 values, `rows` x `cols` of them inside the
// matrix, w at the first; through shared memory, so that global memory is
// accessed along its lines whether w is stored like v or transposed.
__device__ __forceinline__ void update_block(const float* v, uint8_t* stg, int lane, float* w,
                                             long long pitch, bool transposed, float decay,
                                             float gain, int rows, int cols) {
  const bool keep = decay != 0.0f;  // 0: w is only written
  if (transposed) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      *reinterpret_cast<float*>(piece(stg, j, lane >> 2) + (lane & 3) * 4) = v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<float4*>(piece(stg, lane, j)) =
          make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  }
  __syncwarp();
  const int lines = transposed ? cols : rows, len = transposed ? rows : cols;
  if (pitch % 4 == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0 && len >= 32) {
    const int l0 = lane >> 3, p = lane & 7;
    float4 old[8];
    if (keep && lines >= 32) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        old[i] = *reinterpret_cast<const float4*>(w + (i * 4 + l0) * pitch + p * 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        old[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (keep && i * 4 + l0 < lines)
          old[i] = *reinterpret_cast<const float4*>(w + (i * 4 + l0) * pitch + p * 4);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int l = i * 4 + l0;
      const float4 x = *reinterpret_cast<const float4*>(piece(stg, l, p));
      if (l < lines)
        *reinterpret_cast<float4*>(w + l * pitch + p * 4) =
            make_float4(fmaf(gain, x.x, decay * old[i].x), fmaf(gain, x.y, decay * old[i].y),
                        fmaf(gain, x.z, decay * old[i].z), fmaf(gain, x.w, decay * old[i].w));
    }
  } else {
    for (int l0 = 0; l0 < 32; l0 += 8) {
      float old[8];
#pragma unroll
      for (int l = 0; l < 8; ++l)
        old[l] = keep && l0 + l < lines && lane < len ? w[(l0 + l) * pitch + lane] : 0.f;
#pragma unroll
      for (int l = 0; l < 8; ++l) {
        const float x = *reinterpret_cast<float*>(piece(stg, l0 + l, lane >> 2) + (lane & 3) * 4);
        if (l0 + l < lines && lane < len)
          w[(l0 + l) * pitch + lane] = fmaf(gain, x, decay * old[l]);
      }
    }
  }
  __syncwarp();
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// a += b on two floats at once.
__device__ __forceinline__ void add2(float& a0, float& a1, uint32_t b0, uint32_t b1) {
  asm("{\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "r"(b0), "r"(b1));
}

template <bool PAIR, int CAP>
__global__ void __launch_bounds__(kThreads, 1)
    muon_gemm_kernel(const __grid_constant__ Items<CAP> g, unsigned int* status) {
  // one kernel for all modes: consecutive launches find its code in the caches
  const Mode mode = g.mode;
  const bool a_sym = mode != Mode::Gram;                       // A is a symmetric operand
  const bool b_sym = mode == Mode::Poly || mode == Mode::Mul;  // B likewise
  const bool b_rows = mode == Mode::Gram;                      // B has K along its rows
  constexpr int BN = PAIR ? 256 : 128;   // tile rows and columns
  constexpr int NC = BN / 2;             // columns of an epilogue warp
  constexpr int CTAS = PAIR ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = ring + kStages * kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + kEpi * kStaging);  // leader's is used
  uint64_t* empty = full + kStages;    // both CTAs
  uint64_t* tfull = empty + kStages;   // [2] both CTAs
  uint64_t* tempty = tfull + 2;        // [2] leader's is used
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = PAIR ? (int)ptx::cluster_rank() : 0;
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&tfull[i], 1);
      ptx::mbar_init(&tempty[i], CTAS * kEpi);  // one arrive per epilogue warp
    }
    ptx::mbar_init(drain, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    if (PAIR) {
      ptx::tmem_alloc_pair(tmem_slot, 2 * BN);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(tmem_slot, 2 * BN);
      ptx::tmem_relinquish();
    }
  }
  if (warp == 0 && lane == 0 && (int)(blockIdx.x / CTAS) < g.tiles) {
    const Item& it = g.item[tile_at<BN, CAP>(g, blockIdx.x / CTAS).item];
    if (!b_rows) {
      ptx::prefetch_tmap(&it.at);
      ptx::prefetch_tmap(&it.bt);
    }
    ptx::prefetch_tmap(&it.a);
    if (b_rows || b_sym) ptx::prefetch_tmap(&it.b);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (PAIR) ptx::cluster_sync();  // peer barriers initialised, tensor memory allocated
  ptx::tc_fence_after();
  ptx::griddep_wait();  // the previous kernel's outputs are visible from here on
  ptx::griddep_launch_dependents();
  const uint32_t tmem_base = *tmem_slot;
  const int cluster_id = blockIdx.x / CTAS, n_clusters = gridDim.x / CTAS;

  if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsHigh));
    const int q = warp & 3;                 // tensor-memory lanes 32 q ..
    const int cbase = (warp - 4) / 4 * NC;  // columns of the tile
    uint8_t* stg = staging + (warp - 4) * kStaging;
    int unit = 0;
    bool ok = true;
    for (int t = cluster_id; t < g.tiles && ok; t += n_clusters) {
      const Tile tile = tile_at<BN, CAP>(g, t);
      const Item& it = g.item[tile.item];
      // copies: parameters indexed at run time would be fetched at every use
      const int m = it.m, n = it.n, ld = it.ld;
      const int num_k = k_blocks(it, tile);
      const int row0 = tile.m0 + rank * 128 + q * 32, col0 = tile.n0 + cbase;
      const bool live = row0 < m && col0 < n;
      const long long plane = it.plane;
      const long long at = (long long)row0 * ld + col0;
      const int rows = m - row0;
      const __half* src = it.g + at;  // Poly
      float* w = it.w;                // Update
      const bool tr = it.w_transposed, part = it.part;
      const long long pitch = tr ? m : n;
      const float decay = it.decay;
      // what the epilogue reads, a line per lane, into L2 meanwhile
      if (mode == Mode::Poly && live) {
        if (lane < rows)
#pragma unroll
          for (int c = 0; c < NC; c += 64)
            if (col0 + c < n) {
              prefetch_l2(src + (long long)lane * ld + c);
              prefetch_l2(src + plane + (long long)lane * ld + c);
            }
      } else if (mode == Mode::Update && live) {
        w += tr ? col0 * pitch + row0 : row0 * pitch + (long long)col0;
#pragma unroll
        for (int c = 0; c < NC; c += 32)
          if (decay != 0.0f && (tr ? col0 + c + lane < n : lane < rows && col0 + c < n))
            prefetch_l2(w + (tr ? (c + lane) * pitch : lane * pitch + c));
      }
      float v[NC];
      Block next;  // of g; the first one before the last segment
#pragma unroll
      for (int i = 0; i < NC; ++i) v[i] = 0.f;
      for (int k0 = 0; k0 < num_k; k0 += kSeg, ++unit) {
        const int acc = unit & 1;
        if (mode == Mode::Poly && live && k0 + kSeg >= num_k)
          load_block(next, lane, src + plane, ld, rows);
        // warp-uniform: every lane takes the same exit
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(&tfull[acc], (unit >> 1) & 1, status, 0x605,
                                                    abort_flag))) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t from = tmem_base + ((uint32_t)(q * 32) << 16) + acc * BN + cbase;
#pragma unroll
        for (int c = 0; c < NC; c += 32) {
          uint32_t x[32];
          ptx::tmem_ld32(from + c, x);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; i += 2) add2(v[c + i], v[c + i + 1], x[i], x[i + 1]);
        }
        // the accumulator is free again; the handoff carries no generic-memory
        // data, so the peer's remote arrive is CTA-scope
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (leader) ptx::mbar_arrive(&tempty[acc]);
          else ptx::mbar_arrive_remote(ptx::mapa(ptx::smem_u32(&tempty[acc]), 0));
        }
      }
      if (!ok) break;
      if (!live) continue;
      const float scale = mode == Mode::Update ? it.gain : it.scale;
      __half* out = it.out + at;
#pragma unroll 1
      for (int c = 0; c < NC; c += 64) {
        if (col0 + c >= n) break;
        if (mode == Mode::Update) {
          float* y = w + (tr ? c * pitch : (long long)c);
          update_block(v, stg, lane, y, pitch, tr, decay, scale, rows, n - col0 - c);
          if (col0 + c + 32 < n)
            update_block(v + 32, stg, lane, y + (tr ? 32 * pitch : 32ll), pitch, tr, decay, scale,
                         rows, n - col0 - c - 32);
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] *= scale;
          if (mode == Mode::Poly) {  // small terms first
            constexpr float f = kB * (kMScale / kXScale), f_lo = f / (1 << kLoShift);
            put_block(next, stg, lane);
            load_block(next, lane, src + c, ld, rows);
            add_block(v, f_lo, stg, lane);
            put_block(next, stg, lane);
            if (c + 64 < NC && col0 + c + 64 < n)
              load_block(next, lane, src + plane + c + 64, ld, rows);
            add_block(v, f, stg, lane);
            const int diagonal = row0 - col0 - c;  // of the warp's first row
            if (diagonal > -32 && diagonal < 64) {
#pragma unroll
              for (int i = 0; i < 64; ++i) v[i] += i == diagonal + lane ? kA * kMScale : 0.f;
            }
          }
          uint32_t hi[32], lo[32];
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (part) as_halves(v[2 * i], v[2 * i + 1], hi[i], lo[i]);
            else split2(v[2 * i], v[2 * i + 1], hi[i], lo[i]);
          store_plane(hi, stg, lane, out + c, ld, rows);
          store_plane(lo, stg, lane, out + plane + c, ld, rows);
        }
#pragma unroll
        for (int i = 0; i < NC - 64; ++i) v[i] = v[i + 64];
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
    if (warp == 0) {
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        long long issued = 0;
        for (int t = cluster_id; t < g.tiles && ok; t += n_clusters) {
          const Tile tile = tile_at<BN, CAP>(g, t);
          const Item& it = g.item[tile.item];
          const int num_k = k_blocks(it, tile);
          const int am = tile.m0 + rank * 128, bn = tile.n0 + rank * 128;
          const int a_upper = (tile.m0 / kBlock + 1) * kBlock;
          const int b_upper = (tile.n0 / kBlock + 1) * kBlock;
          for (int kb = 0; kb < num_k; ++kb) {
            if (!ptx::mbar_wait(&empty[stage], phase ^ 1, status, 0x601, abort_flag)) {
              ok = false;
              break;
            }
            if (leader) ptx::mbar_arrive_expect_tx(&full[stage], CTAS * kStage);
            uint8_t* sa = ring + stage * kStage;
            uint8_t* sb = sa + kOperand;
            const int k = kb * kBK;
            const bool at = a_sym && k >= a_upper, bt = b_sym ? k >= b_upper : !b_rows;
            if (PAIR) {
              const uint32_t bar = ptx::mapa(ptx::smem_u32(&full[stage]), 0);
              if (at) ptx::tma_load_4d_pair(sa, &it.at, bar, 0, k, am / 64, 0);
              else ptx::tma_load_3d_pair(sa, &it.a, bar, k, am, 0);
              if (bt) ptx::tma_load_4d_pair(sb, &it.bt, bar, 0, k, bn / 64, 0);
              else ptx::tma_load_3d_pair(sb, &it.b, bar, k, bn, 0);
            } else {
              if (at) ptx::tma_load_4d(sa, &it.at, &full[stage], 0, k, am / 64, 0);
              else ptx::tma_load_3d(sa, &it.a, &full[stage], k, am, 0);
              if (bt) ptx::tma_load_4d(sb, &it.bt, &full[stage], 0, k, bn / 64, 0);
              else ptx::tma_load_3d(sb, &it.b, &full[stage], k, bn, 0);
            }
            ++issued;
            if (++stage == kStages) { stage = 0; phase ^= 1; }
          }
        }
        if (leader) {
          // wait (bounded) for the last round of each stage, so that no copy of
          // the CTAs is in flight when they exit
          for (int s = 0; s < kStages && s < issued; ++s) {
            const long long round = (issued - 1 - s) / kStages;
            ptx::mbar_wait(&full[s], (uint32_t)(round & 1), status, 0x607, nullptr);
          }
        }
      }
    } else if (warp == 1) {
      if (lane == 0 && leader) {
        int stage = 0;
        uint32_t phase = 0;
        int unit = 0;  // segments so far
        bool ok = true;
        for (int t = cluster_id; t < g.tiles && ok; t += n_clusters) {
          const Tile tile = tile_at<BN, CAP>(g, t);
          const int num_k = k_blocks(g.item[tile.item], tile);
          // K from which a symmetric operand's blocks lie above the diagonal
          const int a_upper = (tile.m0 / kBlock + 1) * kBlock;
          const int b_upper = (tile.n0 / kBlock + 1) * kBlock;
          for (int k0 = 0; k0 < num_k && ok; k0 += kSeg, ++unit) {
            const int acc = unit & 1;
            if (!ptx::mbar_wait<PAIR>(&tempty[acc], ((unit >> 1) & 1) ^ 1, status, 0x602,
                                      abort_flag)) {
              ok = false;
              break;
            }
            ptx::tc_fence_after();
            const uint32_t d = tmem_base + acc * BN;
            const int k1 = min(num_k, k0 + kSeg);
            for (int kb = k0; kb < k1; ++kb) {
              if (!ptx::mbar_wait(&full[stage], phase, status, 0x603, abort_flag)) {
                ok = false;
                break;
              }
              ptx::tc_fence_after();
              const uint32_t sa = ptx::smem_u32(ring + stage * kStage), sb = sa + kOperand;
              const bool at = a_sym && kb * kBK >= a_upper;
              const bool bt = b_sym ? kb * kBK >= b_upper : !b_rows;
              const uint32_t idesc =
                  ptx::make_idesc_f16(CTAS * 128, BN, false, false) | (at << 15) | (bt << 16);
              // K-major: 16 elements = 32 bytes along the swizzled row;
              // MN-major: 16 rows of 128 bytes, 64-column chunks 8 KB apart
              const uint64_t a0 = ptx::make_sdesc(sa, at ? 8192 : 16, 1024, 2);
              const uint64_t b0 = ptx::make_sdesc(sb, bt ? 8192 : 16, 1024, 2);
              const uint32_t a_step = at ? 2048 >> 4 : 32 >> 4, b_step = bt ? 2048 >> 4 : 32 >> 4;
              auto a_desc = [&](int kk, int plane) {
                return a0 + kk * a_step + plane * (kPlane >> 4);
              };
              auto b_desc = [&](int kk, int plane) {
                return b0 + kk * b_step + plane * (kPlane >> 4);
              };
              auto mma = [&](uint64_t a, uint64_t b, bool more) {
                if (PAIR) ptx::mma_f16_ss_pair(d, a, b, idesc, more);
                else ptx::mma_f16_ss(d, a, b, idesc, more);
              };
  #pragma unroll
              for (int kk = 0; kk < kBK / 16; ++kk) {
                mma(a_desc(kk, 1), b_desc(kk, 0), kb > k0 || kk > 0);
                mma(a_desc(kk, 0), b_desc(kk, 1), true);
              }
  #pragma unroll
              for (int kk = 0; kk < kBK / 16; ++kk) {
                if (kk > 0) mma(a_desc(kk, 0), b_desc(kk, 0), true);
                else if (PAIR)
                  ptx::mma_f16_ss_pair_shifted<kLoShift>(d, a_desc(0, 0), b_desc(0, 0), idesc);
                else
                  ptx::mma_f16_ss_shifted<kLoShift>(d, a_desc(0, 0), b_desc(0, 0), idesc);
              }
              if (PAIR) ptx::mma_commit_pair(&empty[stage], 0x3);
              else ptx::mma_commit(&empty[stage]);
              if (++stage == kStages) { stage = 0; phase ^= 1; }
            }
            if (!ok) break;
            if (PAIR) ptx::mma_commit_pair(&tfull[acc], 0x3);
            else ptx::mma_commit(&tfull[acc]);
          }
        }
        if (PAIR) ptx::mma_commit_pair(drain, 0x3);
        else ptx::mma_commit(drain);
        ptx::mbar_wait(drain, 0, status, 0x604, nullptr);
      }
    }
  }

  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if (PAIR) ptx::cluster_sync();  // the pair's MMAs are retired before either frees TMEM
  if (warp == 1) {
    ptx::tc_fence_after();
    if (PAIR) ptx::tmem_dealloc_pair(tmem_base, 2 * BN);
    else ptx::tmem_dealloc(tmem_base, 2 * BN);
  }
}

}  // namespace muon
}  // namespace agpu
