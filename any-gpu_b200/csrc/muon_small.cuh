// The whole Newton-Schulz iteration of a matrix of at most 128 rows (of its
// shorter side) in one kernel: a cluster of CTAs per matrix, each holding 256
// columns of X on chip for all steps.  Through the grouped products
// (muon_gemm.cuh) such a matrix costs 17 launches, 85 us for 32 x 32 and 100 for
// 64 x 256.
//
// Shared memory of a CTA: X split in two fp16 planes (128 KB: four chunks of 64
// columns, each a plane pair of 128 lines of 128 bytes, 128-byte swizzle) and a
// square S of two such chunks (64 KB), which holds A, then the polynomial b A +
// c A A.  The same image of X serves the tensor core as a K-major operand (A =
// X X^T) and as an MN-major one (times X).  Tensor memory: columns 0-255
// accumulate, 256-511 keep X in fp32 for the term a X, added outside the
// tensor core: the rounding of a small matrix shows more than that of a large
// one (|X|_F is at most sqrt(128)), and with a X inside the 22-bit products
// 64 x 256 was off by 2.2e-6, twice what fp32 arithmetic is.
//
// A step, all eight warps together, with the MMAs issued by one thread:
//   A = X X^T over this CTA's columns; the cluster's parts are summed through
//   distributed shared memory (each CTA sums 1/C of the elements of all and
//   stores them to all); S = A; A A; S = b A + c A A; times X; X = a X + that.
// Within an accumulator all small terms (lo hi, hi lo) come first, so only the
// hi hi products, at most 16, are truncated at full size.  Here lo = fp16(x 2^e -
// hi), without the grouped products' shift, which takes 64 x 256 from 57 us to
// 62: rows far smaller than the others are held by a X in fp32 (rows 1e-6 of
// the others: 2.2e-6 off at most).
//
// Diagonals.  As the singular values near 1, A and the polynomial near multiples
// of I, and 22 bits of a diagonal element scale its whole row.  So S holds them
// without their diagonals, which are applied in fp32 outside: with A = D + O,
//   (A A)_ij = (O O)_ij + (D_i + D_j) O_ij,  (A A)_ii = (O O)_ii + D_i^2,
//   X_i <- (a + (b A + c A A)_ii) X_i + (off-diagonal polynomial times X)_i.
//
// Bound by the latency of its phases: 64 x 256, five steps, take 53 us, of which
// the tensor core's products at its peak rate are under 1 us.  By the SM's
// clock a step is 12,000 cycles: issuing the 24 MMAs of A 3,200, reading A back
// 1,400, splitting it into S 1,000, A A 1,400, the polynomial into S 2,200,
// times X 1,900, the new X 1,000; the way in (loads, norm, first split) 11,000.
// 128 x 256: 66 us; 32 x 32: 35; 128 x 2048, a cluster of 8, 95, where summing
// A over the cluster takes 10,000 cycles a step.
//
// Every wait is bounded.  Behind one that expired a CTA issues no more MMAs and
// stores no result, but takes part in the cluster's barriers to the end; the
// status word says that the matrix is not valid.
#pragma once

#include "muon_gemm.cuh"

namespace agpu {
namespace muon {

constexpr int kSmallRows = 128, kSmallCols = 256, kSmallCluster = 16;
constexpr int kSmallThreads = 256;
constexpr int kChunkBytes = 2 * kPlane;                      // a plane pair of 64 columns
constexpr int kSmallX = kSmallCols / 64 * kChunkBytes;       // 128 KB
constexpr int kSmallS = kSmallRows / 64 * kChunkBytes;       // 64 KB
constexpr int kSmallSmem = 1024 + kSmallX + kSmallS + 256 + 2 * kSmallRows * 4;
constexpr int kSmallItems = 80;  // below 4 KB of kernel parameters

struct SmallItem {
  const float* grad;
  float* momentum;  // or null: the update is `grad`
  float* w;
  int m, n;         // shorter and longer side
  int tall;         // stored [n, m]
  float decay, gain;
};

struct SmallItems {
  SmallItem item[kSmallItems];
  float mu;
  int nesterov, steps;
};

__device__ __forceinline__ float update_of(float g, float m, float mu, bool nesterov) {
  return nesterov ? (1.0f - mu) * g + mu * m : m;
}
__device__ __forceinline__ float step_momentum(float g, float m, float mu) {
  return mu * m + (1.0f - mu) * g;
}
// |U|_F of a sum of squares, at least 1e-30; a NaN stays one, and fills X.
__device__ __forceinline__ double floored_norm(double squares) {
  const double norm = sqrt(squares);
  return norm < 1e-30 ? 1e-30 : norm;
}

// S as 128 x 128 floats, X as 128 x 256 floats: 16-byte piece p of row r.
__device__ __forceinline__ float4* square_piece(uint8_t* s, int r, int p) {
  return reinterpret_cast<float4*>(s + r * 512 + ((p ^ (r & 7)) << 4));
}
__device__ __forceinline__ float4* slice_piece(uint8_t* x, int r, int p) {
  return reinterpret_cast<float4*>(x + r * 1024 + ((p ^ (r & 7)) << 4));
}

// hi and lo of two scaled values, packed.
__device__ __forceinline__ void split_plain(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// 32 scaled values of a row (columns c0 .. c0 + 31 of a split image) to both planes.
__device__ __forceinline__ void put_row(uint8_t* image, int row, int c0, const float (&v)[32]) {
  uint8_t* line = image + (c0 >> 6) * kChunkBytes + row * 128;
  const int p0 = (c0 & 63) >> 3;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 hi, lo;
    split_plain(v[8 * j + 0], v[8 * j + 1], hi.x, lo.x);
    split_plain(v[8 * j + 2], v[8 * j + 3], hi.y, lo.y);
    split_plain(v[8 * j + 4], v[8 * j + 5], hi.z, lo.z);
    split_plain(v[8 * j + 6], v[8 * j + 7], hi.w, lo.w);
    const int at = ((p0 + j) ^ (row & 7)) << 4;
    *reinterpret_cast<uint4*>(line + at) = hi;
    *reinterpret_cast<uint4*>(line + kPlane + at) = lo;
  }
}

__global__ void __launch_bounds__(kSmallThreads, 1)
    muon_small_kernel(const __grid_constant__ SmallItems g, int cluster, unsigned int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* X = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                          ~uintptr_t(1023));
  uint8_t* S = X + kSmallX;
  double* red = reinterpret_cast<double*>(S + kSmallS);  // [8] warps, [8] the CTA's sum
  uint64_t* done = reinterpret_cast<uint64_t*>(red + 9);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint64_t* drain = done + 2;
  // [128] diagonal of A at scale kXScale; [128] a + the polynomial's
  float* diag = reinterpret_cast<float*>(red + 32);
  float* coef = diag + kSmallRows;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int rank = (int)blockIdx.x % cluster;
  const SmallItem& it = g.item[blockIdx.x / cluster];
  const int m = it.m, n = it.n;
  const bool tall = it.tall != 0;
  const float* grad = it.grad;
  float* momentum = it.momentum;
  const float mu = g.mu;
  const bool nesterov = g.nesterov != 0;
  const int c0 = rank * kSmallCols, w = max(0, min(kSmallCols, n - c0));  // this CTA's columns

  if (tid == 0) {
    ptx::mbar_init(done, 1);
    ptx::mbar_init(drain, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 0) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }

  // The update of this CTA's columns, into X as floats, and the sum of its
  // squares: by lines of memory (columns if tall, else rows), kLoads elements
  // per lane at a time, of one line or several short ones.
  const int pitch = tall ? m : n;
  const long long slice = tall ? (long long)c0 * m : (long long)c0;
  double s = 0.0;
  {
    constexpr int kLoads = 16;
    const int inner = tall ? m : w, lines = tall ? w : m;
    const int shift = inner > 128 ? 3 : inner > 64 ? 2 : inner > 32 ? 1 : 0;  // 32s of a line
    const int per = kLoads >> shift;                                         // lines at a time
    for (int l0 = warp * per; l0 < lines; l0 += kSmallThreads / 32 * per) {
      float x[kLoads], mo[kLoads];
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        const int line = l0 + (k >> shift), j = ((k & ((1 << shift) - 1)) << 5) + lane;
        const int at = min(line, lines - 1) * pitch + min(j, inner - 1);
        x[k] = ptx::load_now(grad + slice + at);
        if (momentum) mo[k] = ptx::load_now(momentum + slice + at);
      }
      if (momentum) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
          const int line = l0 + (k >> shift), j = ((k & ((1 << shift) - 1)) << 5) + lane;
          const float next = step_momentum(x[k], mo[k], mu);
          x[k] = update_of(x[k], next, mu, nesterov);
          if (line < lines && j < inner) momentum[slice + line * pitch + j] = next;
        }
      }
      // the squares over a power of two near the largest are summed in 32 bits,
      // what comes of them in 64: one conversion instead of kLoads
      float top = 0.f, sum = 0.f;
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        const int line = l0 + (k >> shift), j = ((k & ((1 << shift) - 1)) << 5) + lane;
        const bool in = line < lines && j < inner;
        const int r = tall ? j : line, c = tall ? line : j;
        ptx::store_shared_if(in, reinterpret_cast<float*>(slice_piece(X, r, c >> 2)) + (c & 3), x[k]);
        x[k] = in ? x[k] : 0.f;
        top = fmaxf(top, fabsf(x[k]));
      }
      const uint32_t power = min(max(__float_as_uint(top) & 0x7f800000u, 0x00800000u), 0x7e800000u);
      const float over = __uint_as_float(0x7f000000u - power);
#pragma unroll
      for (int k = 0; k < kLoads; ++k) sum = fmaf(x[k] * over, x[k] * over, sum);
      const double back = __uint_as_float(power);
      s = fma(back * back, (double)sum, s);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) red[warp] = s;
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (tid == 0) {
    s = 0.0;
    for (int i = 0; i < kSmallThreads / 32; ++i) s += red[i];
    red[8] = s;
  }
  if (cluster > 1) ptx::cluster_sync();
  else __syncthreads();
  s = 0.0;
  for (int p = 0; p < cluster; ++p) {
    double part;
    asm volatile("ld.shared::cluster.f64 %0, [%1];"
                 : "=d"(part)
                 : "r"(ptx::mapa(ptx::smem_u32(red + 8), p)));
    s += part;
  }
  const float inv = (float)(kXScale / floored_norm(s));

  // this thread's row, and half of the columns; its warp's tensor-memory lanes
  const int row = (warp & 3) * 32 + lane, half = warp >> 2;
  const bool live = (warp & 3) * 32 < m;  // warp-uniform: some of its rows exist
  const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);

  // X from the floats, scaled: to tensor memory, and when all have been read,
  // split into their place (whole chunks, so that K's last columns are zero)
  const int chunks = (w + 63) / 64;
  const int end = min(chunks * 64, half * 128 + 128);
  if (live) {
#pragma unroll 1
    for (int c = half * 128; c < end; c += 32) {
      float v[32];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 d = *slice_piece(X, row, (c >> 2) + j);
        v[4 * j] = d.x, v[4 * j + 1] = d.y, v[4 * j + 2] = d.z, v[4 * j + 3] = d.w;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = row < m && c + j < w ? v[j] * inv : 0.f;
      ptx::tmem_st32(lanes + 256 + c, reinterpret_cast<uint32_t(&)[32]>(v));
    }
    ptx::tmem_wait_st();
  }
  __syncthreads();
  if (live) {
#pragma unroll 1
    for (int c = half * 128; c < end; c += 32) {
      uint32_t v[32];
      ptx::tmem_ld32(lanes + 256 + c, v);
      ptx::tmem_wait_ld();
      put_row(X, row, c, reinterpret_cast<const float(&)[32]>(v));
    }
  }

  const int n_rows = (m + 15) / 16 * 16;       // columns of A computed
  const int accs = n_rows <= 64 ? 4 : 2, acc_cols = 256 / accs;  // of A
  const int mine = half * 64;                  // this thread's columns of A: 64
  const bool has_a = live && mine < n_rows;
  const uint32_t x_addr = ptx::smem_u32(X), s_addr = ptx::smem_u32(S);
  uint32_t phase = 0;
  bool ok = true;
  // what every thread wrote to shared memory is there for the tensor core, and
  // the accumulators have been read
  auto ready = [&] {
    ptx::fence_proxy_async_smem();
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
  };
  auto finish = [&] {  // all threads: wait for the issued MMAs
    ok = ok && ptx::mbar_wait(done, phase, status, 0x611, abort_flag);
    phase ^= 1;
    ptx::tc_fence_after();
  };
  auto kmajor = [&](uint32_t addr) { return ptx::make_sdesc(addr, 16, 1024, 2); };

#pragma unroll 1
  for (int step = 0; step < g.steps; ++step) {
    ready();
    if (tid == 0 && ok && !*abort_flag) {
      const uint32_t idesc = ptx::make_idesc_f16(128, n_rows, false, false);
      for (int pass = 0; pass < 2; ++pass)
        for (int c = 0; c < chunks; ++c) {
          const uint64_t hi = kmajor(x_addr + c * kChunkBytes), lo = hi + (kPlane >> 4);
          const uint32_t d = tmem + c % accs * acc_cols;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint64_t k = kk * (32 >> 4);
            if (pass == 0) {
              ptx::mma_f16_ss(d, lo + k, hi + k, idesc, c >= accs || kk > 0);
              ptx::mma_f16_ss(d, hi + k, lo + k, idesc, 1u);
            } else {
              ptx::mma_f16_ss(d, hi + k, hi + k, idesc, 1u);
            }
          }
        }
      ptx::mma_commit(done);
    }
    finish();
    float gv[64];  // A, at scale kXScale
#pragma unroll
    for (int i = 0; i < 64; ++i) gv[i] = 0.f;
    if (has_a) {
      for (int c = 0; c < min(chunks, accs); ++c) {
#pragma unroll
        for (int b = 0; b < 64; b += 32) {
          uint32_t x[32];
          ptx::tmem_ld32(lanes + c * acc_cols + mine + b, x);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; i += 2) add2(gv[b + i], gv[b + i + 1], x[i], x[i + 1]);
        }
      }
#pragma unroll
      for (int i = 0; i < 64; ++i) gv[i] *= kUntruncate / kXScale;
    }
    if (cluster > 1) {
      if (has_a) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          *square_piece(S, row, (mine >> 2) + j) =
              make_float4(gv[4 * j], gv[4 * j + 1], gv[4 * j + 2], gv[4 * j + 3]);
      }
      ptx::cluster_sync();
      // rows in groups of `cluster`: this CTA sums row r of each, to all
      for (int i = tid; i < (m + cluster - 1) / cluster * 32; i += kSmallThreads) {
        const int r = (i >> 5) * cluster + rank, p = i & 31;
        if (r >= m || p * 4 >= n_rows) continue;
        const uint32_t at = ptx::smem_u32(square_piece(S, r, p));
        constexpr int kParts = 8;  // in flight
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int q0 = 0; q0 < cluster; q0 += kParts) {
          float4 d[kParts];
#pragma unroll
          for (int q = 0; q < kParts; ++q)
            if (q0 + q < cluster)
              asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                           : "=f"(d[q].x), "=f"(d[q].y), "=f"(d[q].z), "=f"(d[q].w)
                           : "r"(ptx::mapa(at, q0 + q)));
#pragma unroll
          for (int q = 0; q < kParts; ++q)
            if (q0 + q < cluster)
              sum = make_float4(sum.x + d[q].x, sum.y + d[q].y, sum.z + d[q].z, sum.w + d[q].w);
        }
        for (int q = 0; q < cluster; ++q)
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(ptx::mapa(at, q)),
                       "f"(sum.x), "f"(sum.y), "f"(sum.z), "f"(sum.w)
                       : "memory");
      }
      ptx::cluster_sync();
      if (has_a) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float4 d = *square_piece(S, row, (mine >> 2) + j);
          gv[4 * j] = d.x, gv[4 * j + 1] = d.y, gv[4 * j + 2] = d.z, gv[4 * j + 3] = d.w;
        }
      }
      __syncthreads();  // before S is written as an operand
    }
    // S = gv, with zeros behind row and column m (accumulators hold anything
    // there); its diagonal element, if it is here, leaves through `d`
    const bool whole = (warp & 3) * 32 + 32 <= m && mine + 64 <= m;
    const bool has_diag = live && (row >> 6) == half;  // both the same in a warp
    auto put_square = [&](float& d) {
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (row >= m || mine + i >= m) gv[i] = 0.f;
      }
      if (has_diag) {
        d = 0.f;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          d = mine + i == row ? gv[i] : d;
          gv[i] = mine + i == row ? 0.f : gv[i];
        }
      }
      put_row(S, row, mine, reinterpret_cast<const float(&)[32]>(gv[0]));
      put_row(S, row, mine + 32, reinterpret_cast<const float(&)[32]>(gv[32]));
    };
    float d_row = 0.f;
    if (live) put_square(d_row);
    if (has_diag) diag[row] = d_row;
    ready();
    const int ks = (m + 15) / 16;  // K in 16s of the products with a square
    if (tid == 0 && ok && !*abort_flag) {
      const uint32_t idesc = ptx::make_idesc_f16(128, n_rows, false, false);
      for (int pass = 0; pass < 2; ++pass)
        for (int k = 0; k < ks; ++k) {
          const uint32_t a = s_addr + (k >> 2) * kChunkBytes + (k & 3) * 32;
          if (pass == 0) {
            ptx::mma_f16_ss(tmem, kmajor(a + kPlane), kmajor(a), idesc, k > 0);
            ptx::mma_f16_ss(tmem, kmajor(a), kmajor(a + kPlane), idesc, 1u);
          } else {
            ptx::mma_f16_ss(tmem, kmajor(a), kmajor(a), idesc, 1u);
          }
        }
      ptx::mma_commit(done);
    }
    finish();
    if (live) {
      // off the diagonal b A + c (O O + (D_i + D_j) A), on it b D + c (O O + D^2)
      constexpr float kOO = kC * kUntruncate * (kMScale / (kXScale * kXScale));
      constexpr float kDD = kC * (kMScale / (kXScale * kXScale));
      constexpr float kLinear = kB * (kMScale / kXScale);
      const float di = diag[row], lin_i = fmaf(kDD, di, kLinear);
      const float on_diag = lin_i * di;  // b D + c D^2
#pragma unroll
      for (int b = 0; b < 64; b += 32) {
        if (has_a) {
          uint32_t x[32];
          ptx::tmem_ld32(lanes + mine + b, x);
          ptx::tmem_wait_ld();
          float dj4[32];
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(dj4 + i) =
                reinterpret_cast<const float4*>(diag)[(mine + b + i) / 4];
#pragma unroll
          for (int i = 0; i < 32; ++i)
            gv[b + i] = fmaf(kOO, __uint_as_float(x[i]),
                             fmaf(kDD, dj4[i], lin_i) * gv[b + i]);
          if (has_diag) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (mine + b + i == row) gv[b + i] = fmaf(kOO, __uint_as_float(x[i]), on_diag);
          }
        }
      }
      put_square(d_row);
      if (has_diag) coef[row] = kA + d_row * (1.0f / kMScale);
    }
    ready();
    if (tid == 0 && ok && !*abort_flag) {
      // X as an MN-major operand: 64-column chunks kChunkBytes apart, 16 rows of K 2 KB
      const uint32_t idesc = ptx::make_idesc_f16(128, max(chunks, 1) * 64, false, true);
      auto rows_of = [&](uint32_t addr) { return ptx::make_sdesc(addr, kChunkBytes, 1024, 2); };
      for (int pass = 0; pass < 2; ++pass)
        for (int k = 0; k < ks; ++k) {
          const uint32_t a = s_addr + (k >> 2) * kChunkBytes + (k & 3) * 32;
          const uint32_t b = x_addr + k * 2048;
          if (pass == 0) {
            ptx::mma_f16_ss(tmem, kmajor(a + kPlane), rows_of(b), idesc, k > 0);
            ptx::mma_f16_ss(tmem, kmajor(a), rows_of(b + kPlane), idesc, 1u);
          } else {
            ptx::mma_f16_ss(tmem, kmajor(a), rows_of(b), idesc, 1u);
          }
        }
      ptx::mma_commit(done);
    }
    finish();
    const bool last = step + 1 == g.steps;
    if (live) {
      const float decay = it.decay, gain = it.gain / kXScale, ci = coef[row];
      uint8_t* stg = S + warp * kStaging;  // the last step's products with S are done
#pragma unroll 1
      for (int c = half * 128; c < min(w, half * 128 + 128); c += 32) {
        uint32_t x[32], y[32];
        ptx::tmem_ld32(lanes + 256 + c, x);
        ptx::tmem_ld32(lanes + c, y);
        ptx::tmem_wait_ld();
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i)
          v[i] = fmaf(ci, __uint_as_float(x[i]), __uint_as_float(y[i]) * (kUntruncate / kMScale));
        if (last) {
          if (!__all_sync(0xffffffffu, ok)) break;
          const int r0 = (warp & 3) * 32;
          update_block(v, stg, lane, it.w + slice + (tall ? c * pitch + r0 : r0 * pitch + c), pitch,
                       tall, decay, gain, m - r0, w - c);
        } else {
          ptx::tmem_st32(lanes + 256 + c, reinterpret_cast<uint32_t(&)[32]>(v));
          put_row(X, row, c, v);
        }
      }
      ptx::tmem_wait_st();
    }
  }
  if (tid == 0 && (!ok || *abort_flag)) {  // what was issued is behind it before tensor memory is given back
    ptx::mma_commit(drain);
    ptx::mbar_wait(drain, 0, status, 0x612, nullptr);
  }
  ptx::tc_fence_before();
  if (cluster > 1) ptx::cluster_sync();  // no CTA leaves while others may read its memory
  else __syncthreads();
  if (warp == 0) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

}  // namespace muon
}  // namespace agpu
