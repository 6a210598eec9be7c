// Orthogonalised updates: the quintic Newton-Schulz iteration and the
// optimiser step built on it.  No counterpart in the reference crate (its
// optimiser is AdamW, src/optim.rs); it stands beside agpu_adamw_step for the
// matrices of a model.  For a matrix W with gradient G and momentum M:
//   M <- mu M + (1 - mu) G,   U = (1 - mu) G + mu M (nesterov) or M
//   X = U / max(|U|_F, 1e-30), then `steps` times (rows <= cols; else on X^T)
//       A = X X^T,  X <- (a I + b A + c A A) X
//   W <- (1 - lr wd) W - lr 0.2 sqrt(max(rows, cols)) X
// which drives the singular values of X towards 1 (the iteration's coefficients:
// K. Jordan et al., 2024; the factor of the update: J. Liu et al., 2025).
//
// Matrices of at most 128 x 4096 go through the whole iteration on chip
// (muon_small.cuh), unless larger ones are in a call of few.  All others of a
// call go through it together, a group per launch: two kernels form the scaled
// split X, then three products a step (muon_gemm.cuh), the last of which updates
// W in its epilogue.  A of few long rows is summed from parts over their columns.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <exception>
#include <mutex>
#include <vector>

#include "agpu_internal.cuh"
#include "muon_gemm.cuh"
#include "muon_small.cuh"

namespace agpu {

namespace {

using muon::Item;
using muon::Mode;

constexpr int kThreads = 256;
constexpr int kMaxParts = 1024;  // CTAs (and partial sums) of one matrix's norm
constexpr size_t kGroupBytes = 8ull << 30;  // scratch of a group of several matrices
constexpr int kGramRows = 512;  // least rows for steps on the Gram matrix

// One matrix: what the call gives, and its scratch.
struct Source {
  const float* grad;
  float* momentum;  // or null: the update is `grad`
  __half* x;        // split X [m, n], two planes
  long long plane;
  int ld;           // of x: n rounded up to 64
  int rows, cols;
  int m, n;         // min, max
};

struct Sources {
  Source item[muon::kMaxItems];
  double* partial;  // [item][gridDim.x]
  float mu;
  int nesterov;
};

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  __syncthreads();
  if (lane == 0) red[w] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) s += red[i];
  return s;
}

using muon::step_momentum;
using muon::update_of;

__device__ __forceinline__ bool aligned16(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// blockIdx.y = matrix.  Steps its momentum and sums the squares of its update
// per CTA, in double: a gradient's squares leave the range of a float.
__global__ void __launch_bounds__(kThreads)
    muon_update_kernel(const __grid_constant__ Sources p) {
  __shared__ double red[kThreads / 32];
  const Source& it = p.item[blockIdx.y];
  const long long n = (long long)it.rows * it.cols;
  const bool vec = aligned16(it.grad) && aligned16(it.momentum);
  double s = 0.0;
  for (long long i = (blockIdx.x * (long long)kThreads + threadIdx.x) * 4; i < n;
       i += (long long)gridDim.x * kThreads * 4) {
    float g[4], m[4];
    const int cnt = (int)min(4ll, n - i);
    if (vec && cnt == 4) {
      *reinterpret_cast<float4*>(g) = *reinterpret_cast<const float4*>(it.grad + i);
      if (it.momentum)
        *reinterpret_cast<float4*>(m) = *reinterpret_cast<const float4*>(it.momentum + i);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        g[j] = j < cnt ? it.grad[i + j] : 0.f;
        m[j] = j < cnt && it.momentum ? it.momentum[i + j] : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float u = g[j];
      if (it.momentum) {
        m[j] = step_momentum(g[j], m[j], p.mu);
        u = update_of(g[j], m[j], p.mu, p.nesterov);
      }
      s += (double)u * u;
    }
    if (it.momentum) {
      if (vec && cnt == 4) {
        *reinterpret_cast<float4*>(it.momentum + i) = *reinterpret_cast<float4*>(m);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < cnt) it.momentum[i + j] = m[j];
      }
    }
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) p.partial[(long long)blockIdx.y * gridDim.x + blockIdx.x] = s;
}

// 8 scaled values to both planes, 16 bytes each.
__device__ __forceinline__ void store_split(const float (&v)[8], __half* out, long long plane) {
  uint4 hi, lo;
  muon::split2(v[0], v[1], hi.x, lo.x);
  muon::split2(v[2], v[3], hi.y, lo.y);
  muon::split2(v[4], v[5], hi.z, lo.z);
  muon::split2(v[6], v[7], hi.w, lo.w);
  *reinterpret_cast<uint4*>(out) = hi;
  *reinterpret_cast<uint4*>(out + plane) = lo;
}

// blockIdx.y = matrix.  X = its update over the norm, split, with rows along
// the longer side (a tall matrix is transposed in shared memory); columns n to
// ld are zero.
__global__ void __launch_bounds__(kThreads)
    muon_split_kernel(const __grid_constant__ Sources p) {
  __shared__ double red[kThreads / 32];
  __shared__ float tile[32][65];
  const Source& it = p.item[blockIdx.y];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  double s = 0.0;
  for (int i = threadIdx.x; i < gridDim.x; i += kThreads)
    s += p.partial[(long long)blockIdx.y * gridDim.x + i];
  const float inv = (float)(muon::kXScale / muon::floored_norm(block_sum(s, red)));
  auto value = [&](long long i) {
    const float g = it.grad[i];
    return it.momentum ? update_of(g, it.momentum[i], p.mu, p.nesterov) : g;
  };
  if (it.rows <= it.cols) {
    const int groups = it.ld / 8;
    const long long total = (long long)it.m * groups;
    const bool vec = it.cols % 4 == 0 && aligned16(it.grad) && aligned16(it.momentum);
    for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < total;
         i += (long long)gridDim.x * kThreads) {
      const long long r = i / groups;
      const int c = (int)(i - r * groups) * 8;
      const long long at = r * it.cols + c;
      float v[8];
      if (vec && c + 8 <= it.cols) {
        float m[8];
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
          *reinterpret_cast<float4*>(v + h) = *reinterpret_cast<const float4*>(it.grad + at + h);
          if (it.momentum)
            *reinterpret_cast<float4*>(m + h) =
                *reinterpret_cast<const float4*>(it.momentum + at + h);
        }
        if (it.momentum)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = update_of(v[j], m[j], p.mu, p.nesterov);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < it.cols ? value(at + j) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= inv;
      store_split(v, it.x + r * it.ld + c, it.plane);
    }
    return;
  }
  // tall: 64 source rows x 32 source columns -> 32 rows of 64
  const int tiles_r = it.ld / 64, tiles_c = (it.cols + 31) / 32;
  for (long long t = blockIdx.x; t < (long long)tiles_r * tiles_c; t += gridDim.x) {
    const int r0 = (int)(t / tiles_c) * 64, c0 = (int)(t % tiles_c) * 32;
    __syncthreads();
    float u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = r0 + warp + 8 * j, c = c0 + lane;
      u[j] = r < it.rows && c < it.cols ? value((long long)r * it.cols + c) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) tile[lane][warp + 8 * j] = u[j] * inv;
    __syncthreads();
    const int r = threadIdx.x / 8, c = (threadIdx.x % 8) * 8;
    if (c0 + r < it.m) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = tile[r][c + j];
      store_split(v, it.x + (long long)(c0 + r) * it.ld + r0 + c, it.plane);
    }
  }
}

// A = X X^T of matrices whose columns were dealt out over several items of a
// launch: the sum of the parts (floats in two planes of halves), in order, split.
// Blocks above the diagonal are not stored.
struct Part {
  const __half* part;  // the first one's planes; the others follow, 2 planes apart
  __half* out;
  long long plane;
  int m, ld, slices;
};

struct Parts {
  Part item[muon::kMaxItems];
  int blocks;  // CTAs per matrix
};

__global__ void __launch_bounds__(kThreads) muon_sum_kernel(const __grid_constant__ Parts p) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const Part& it = p.item[blockIdx.x / p.blocks];
  const __half* part = it.part;
  const long long plane = it.plane;
  const int groups = it.ld / 8, slices = it.slices, m = it.m;
  for (int i = blockIdx.x % p.blocks * kThreads + threadIdx.x; i < m * groups;
       i += p.blocks * kThreads) {
    const int r = i / groups, c = (i - r * groups) * 8;
    if (c / muon::kBlock > r / muon::kBlock) continue;
    const long long at = (long long)r * it.ld + c;
    float v[8] = {};
    for (int k = 0; k < slices; ++k) {
      const uint4 upper = *reinterpret_cast<const uint4*>(part + 2 * k * plane + at);
      const uint4 lower = *reinterpret_cast<const uint4*>(part + (2 * k + 1) * plane + at);
      const uint32_t h[4] = {upper.x, upper.y, upper.z, upper.w};
      const uint32_t l[4] = {lower.x, lower.y, lower.z, lower.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x, y;
        muon::from_halves(h[j], l[j], x, y);
        v[2 * j] += x;
        v[2 * j + 1] += y;
      }
    }
    store_split(v, it.out + at, plane);
  }
}

// ------------------------------------------------------ tensor-map encode --
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// A split matrix [rows, cols] of two planes.  k_major: tiles of 128 rows x 64
// columns (the contraction runs along the rows' columns); else 64 rows (the
// contraction) x 2 chunks of 64 columns.  A box holds both planes.
agpu_status make_map(CUtensorMap* map, const __half* base, int rows, int cols, int ld,
                     long long plane, bool k_major) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(AGPU_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t r = rows, c = cols, l = ld, pb = (cuuint64_t)plane * 2;
  const cuuint64_t dk[3] = {c, r, 2}, sk[2] = {l * 2, pb};
  const cuuint64_t dn[4] = {64, r, l / 64, 2}, sn[3] = {l * 2, 128, pb};
  const cuuint32_t bk[3] = {64, 128, 2}, bn[4] = {64, 64, 2, 2}, es[4] = {1, 1, 1, 1};
  const CUresult e =
      fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, k_major ? 3 : 4, const_cast<__half*>(base),
         k_major ? dk : dn, k_major ? sk : sn, k_major ? bk : bn, es,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (e != CUDA_SUCCESS)
    return fail(AGPU_ERR_CUDA, "orthogonalize: tensor map encode failed (%d)", (int)e);
  return AGPU_OK;
}

// ------------------------------------------------------------ the products --
using Group = muon::Items<muon::kMaxItems>;

template <bool PAIR, int CAP>
agpu_status launch_items(agpu_device* dev, const muon::Items<CAP>& g, cudaStream_t s) {
  auto kern = muon::muon_gemm_kernel<PAIR, CAP>;
  AGPU_CUDA((set_smem_once<muon::muon_gemm_kernel<PAIR, CAP>>(dev, muon::kSmem)));
  const int slots = PAIR ? std::max(1, dev->sm_count / 2) : dev->sm_count;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(std::min(g.tiles, slots) * (PAIR ? 2 : 1)), 1, 1);
  cfg.blockDim = dim3(muon::kThreads, 1, 1);
  cfg.dynamicSmemBytes = muon::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  AGPU_CUDA(cudaLaunchKernelEx(&cfg, kern, g, dev->d_status));
  return after_launch(dev, "muon_gemm_kernel");
}

// Tiles of one matrix's product with tiles of bn x bn.
long long count_tiles(Mode mode, long long m, long long n, long long bn) {
  const long long tm = (m + bn - 1) / bn, tn = (n + bn - 1) / bn;
  if (!muon::symmetric_out(mode)) return tm * tn;
  const long long blocks = (m + muon::kBlock - 1) / muon::kBlock, sub = muon::kBlock / bn;
  return blocks * (blocks + 1) / 2 * sub * sub;
}

template <bool PAIR>
agpu_status launch_product(agpu_device* dev, Group& g, cudaStream_t s) {
  constexpr int BN = PAIR ? 256 : 128;
  long long tiles = 0;
  for (int i = 0; i < g.count; ++i) {
    Item& it = g.item[i];
    it.tiles_m = (it.m + BN - 1) / BN;
    it.tiles_n = (it.n + BN - 1) / BN;
    it.first = (int)tiles;
    tiles += count_tiles(g.mode, it.m, it.n, BN);
    if (tiles > 0x3fffffff) return fail(AGPU_ERR_UNSUPPORTED, "orthogonalize: too large");
  }
  g.tiles = (int)tiles;
  if (g.count > muon::kFewItems)
    return launch_items<PAIR, muon::kMaxItems>(dev, g, s);
  muon::Items<muon::kFewItems> few;
  std::copy(g.item, g.item + g.count, few.item);
  few.count = g.count;
  few.tiles = g.tiles;
  few.mode = g.mode;
  return launch_items<PAIR, muon::kFewItems>(dev, few, s);
}

// Pair tiles (4 times the work on twice the SMs) once their waves are worth it:
// a wave of them took 20 us where one of single tiles took 15 (products with X of
// eight matrices around 1024 x 2816, K = 1024).
agpu_status product(agpu_device* dev, Mode mode, Group& g, cudaStream_t s) {
  g.mode = mode;
  long long pairs = 0, singles = 0;
  for (int i = 0; i < g.count; ++i) {
    pairs += count_tiles(mode, g.item[i].m, g.item[i].n, 256);
    singles += count_tiles(mode, g.item[i].m, g.item[i].n, 128);
  }
  const long long sms = dev->sm_count;
  const long long pair_waves = ceil_div(pairs, std::max(1ll, sms / 2));
  if (4 * pair_waves <= 3 * (long long)ceil_div(singles, sms))
    return launch_product<true>(dev, g, s);
  return launch_product<false>(dev, g, s);
}

// A symmetric [m, m] matrix, split; its tensor maps with K along the rows (k)
// and across them (n).
struct Square {
  __half* p;
  CUtensorMap k, n;
};

// One matrix through the iteration.
struct Work {
  Source src;
  float* w;
  float decay, gain;
  __half* x[2];  // split X, in turn
  CUtensorMap xk[2], xn[2];
  Square sq[5];
  int squares;       // of sq in use
  long long square;  // elements of a plane of one
  int ld_square;

  size_t halves() const { return 4 * (size_t)src.plane + 2 * (size_t)squares * square; }
};

// Steps taken on the Gram matrix between two products with X.  With M =
// a I + b A + c A A a step is X' = M X, so A' = X' X'^T = M A M: several steps
// need X only at their ends, X' = (M_3 M_2 M_1) X, and products of [m, m]
// matrices between, which commute and are symmetric.  In units of m^3 a step
// on X costs 3 n/m + 1, a segment of three steps 3 n/m + 9 and of two
// 3 n/m + 5: five steps as 3 + 2 take 6 n/m + 14 instead of 15 n/m + 5.
// Rounding in A is amplified until the next X X^T, by up to 3.45^2 a step: in
// fp32 arithmetic 3 + 2 stays within 1.5 times the error of single steps,
// 5 in one segment is 10 to 100 times worse.
constexpr int kMaxSegment = 3;

// Length of segment i when `steps` are split into `segments`, longest first.
int segment_length(int steps, int segments, int i) {
  return steps / segments + (i < steps % segments ? 1 : 0);
}

// K-blocks per item of A = X X^T.  A launch of fewer tiles than SMs takes as long
// as its longest contraction (256 x 8192, each launch by itself under ncu: A 103
// us, the other products of a step 14 each; dealt out, 16 and 12.5 for the sum of
// the parts), so its columns are dealt out over more items, as short as the SMs
// and a launch's items allow, but not below 512 columns.  Five steps on 256 x
// 8192, launches overlapping, take 217 us instead of 600, on 500 x 4000 231
// instead of 397, on 300 x 1500 174 instead of 223; below 16 K-blocks saved the
// launch takes what it gives (300 x 1024).
int slice_blocks(agpu_device* dev, const Work* w, int count) {
  constexpr int kLeast = 512 / muon::kBK;
  int most = 0;
  for (int i = 0; i < count; ++i) most = std::max(most, (w[i].src.n + muon::kBK - 1) / muon::kBK);
  for (int len = kLeast; len < most; len += kLeast) {
    long long tiles = 0, items = 0;
    for (int i = 0; i < count; ++i) {
      const int slices = ((w[i].src.n + muon::kBK - 1) / muon::kBK + len - 1) / len;
      items += slices;
      tiles += slices * count_tiles(Mode::Gram, w[i].src.m, w[i].src.m, 128);
    }
    if (items <= muon::kMaxItems && tiles <= dev->sm_count) return most - len >= 16 ? len : most;
  }
  return most;
}

// Matrices that share launches and scratch.
struct Batch {
  Work* w;
  int count;
  bool on_gram;
  int slice;       // K-blocks per item of A = X X^T
  int parts;       // CTAs per matrix that form X
  int summed = 0;  // matrices whose columns are dealt out
  Sources src = {};
  Parts sums = {};
  std::vector<CUtensorMap> parts_of[2];  // slices of X, in turn

  int slices(int i) const {
    return ((w[i].src.n + muon::kBK - 1) / muon::kBK + slice - 1) / slice;
  }
  size_t bytes() const {  // of scratch
    size_t halves = 0;
    for (int i = 0; i < count; ++i) {
      halves += w[i].halves();
      if (slices(i) > 1) halves += 2 * (size_t)slices(i) * w[i].square;  // parts of A
    }
    return halves * sizeof(__half) + (size_t)count * parts * sizeof(double);
  }
};

// Matrices of one kind as batches that fit a launch and the scratch limit.
void plan_batches(agpu_device* dev, std::vector<Work>& all, bool on_gram,
                  std::vector<Batch>& out) {
  const size_t limit = on_gram ? muon::kMaxItems / 2 : muon::kMaxItems;
  for (size_t first = 0; first < all.size();) {
    size_t halves = all[first].halves(), end = first + 1;
    while (end < all.size() && end - first < limit &&
           (halves + all[end].halves()) * sizeof(__half) <= kGroupBytes)
      halves += all[end++].halves();
    Batch b;
    b.w = &all[first];
    b.count = (int)(end - first);
    b.on_gram = on_gram;
    b.slice = slice_blocks(dev, b.w, b.count);
    // CTAs per matrix: two waves over all, at least 4096 elements each
    long long most = 0;
    for (int i = 0; i < b.count; ++i)
      most = std::max(most, (long long)b.w[i].src.rows * b.w[i].src.cols);
    const long long waves = 16ll * dev->sm_count / b.count;
    b.parts = (int)std::max<long long>(
        1, std::min<long long>({(long long)kMaxParts, waves, most / 4096}));
    out.push_back(std::move(b));
    first = end;
  }
}

// Lays a batch out in the scratch and encodes its tensor maps.
agpu_status prepare_batch(agpu_device* dev, Batch& b, void* scratch, float mu, bool nesterov) {
  Sources& src = b.src;
  src.mu = mu;
  src.nesterov = nesterov;
  __half* h = static_cast<__half*>(scratch);
  for (int i = 0; i < b.count; ++i) {
    Work& t = b.w[i];
    const int m = t.src.m, n = t.src.n;
    for (int k = 0; k < 2; ++k, h += 2 * t.src.plane) {
      t.x[k] = h;
      AGPU_TRY(make_map(&t.xk[k], h, m, n, t.src.ld, t.src.plane, true));
      AGPU_TRY(make_map(&t.xn[k], h, m, n, t.src.ld, t.src.plane, false));
    }
    for (int k = 0; k < t.squares; ++k, h += 2 * t.square) {
      t.sq[k].p = h;
      AGPU_TRY(make_map(&t.sq[k].k, h, m, m, t.ld_square, t.square, true));
      AGPU_TRY(make_map(&t.sq[k].n, h, m, m, t.ld_square, t.square, false));
    }
    t.src.x = t.x[0];
    src.item[i] = t.src;
    const int slices = b.slices(i), cols = b.slice * muon::kBK;
    if (slices == 1) continue;
    for (int k = 0; k < 2; ++k)
      for (int c = 0; c < n; c += cols) {
        b.parts_of[k].emplace_back();
        AGPU_TRY(make_map(&b.parts_of[k].back(), t.x[k] + c, m, std::min(cols, n - c), t.src.ld,
                          t.src.plane, true));
      }
    b.sums.item[b.summed++] = {h, t.sq[0].p, t.square, m, t.ld_square, slices};
    b.sums.blocks =
        std::max(b.sums.blocks, (int)ceil_div((uint64_t)m * t.ld_square / 8, kThreads));
    h += 2 * (size_t)slices * t.square;
  }
  b.sums.blocks = std::min(b.sums.blocks, 4 * dev->sm_count);
  src.partial = reinterpret_cast<double*>(h);
  return AGPU_OK;
}

// The launches of a prepared batch.
agpu_status run_batch(agpu_device* dev, const Batch& b, uint32_t steps, cudaStream_t s) {
  Work* w = b.w;
  const int count = b.count;
  constexpr float X = muon::kXScale, M = muon::kMScale, T = muon::kUntruncate;
  Group g = {};
  // dst = scale * (a b) of every matrix's squares, added to g
  auto add_mul = [&](int dst, int a, int c, float scale) {
    for (int i = 0; i < count; ++i) {
      Item& it = g.item[g.count++];
      it.a = w[i].sq[a].k;
      it.at = w[i].sq[a].n;
      it.b = w[i].sq[c].k;
      it.bt = w[i].sq[c].n;
      it.m = it.n = it.k = w[i].src.m;
      it.out = w[i].sq[dst].p;
      it.plane = w[i].square;
      it.ld = w[i].ld_square;
      it.scale = scale;
      it.part = 0;
    }
  };
  const dim3 grid((unsigned)b.parts, (unsigned)count);
  muon_update_kernel<<<grid, kThreads, 0, s>>>(b.src);
  AGPU_TRY(after_launch(dev, "muon_update_kernel"));
  muon_split_kernel<<<grid, kThreads, 0, s>>>(b.src);
  AGPU_TRY(after_launch(dev, "muon_split_kernel"));

  const int segments = b.on_gram ? ((int)steps + kMaxSegment - 1) / kMaxSegment : (int)steps;
  for (int seg = 0; seg < segments; ++seg) {
    const int len = segment_length((int)steps, segments, seg), cur = seg & 1;
    // squares: A, the product of the segment's polynomials (in turn), the
    // step's polynomial, and that times A
    constexpr int kGram = 0, kPoly = 3, kPolyGram = 4;
    int total = 1;
    float total_scale = M;
    g.count = 0;
    size_t part = 0;
    for (int i = 0, sum = 0; i < count; ++i) {  // A = X X^T
      const int slices = b.slices(i), n = w[i].src.n;
      for (int j = 0; j < slices; ++j) {
        Item& it = g.item[g.count++];
        it.a = it.b = slices > 1 ? b.parts_of[cur][part++] : w[i].xk[cur];
        it.m = it.n = w[i].src.m;
        it.k = slices > 1 ? std::min(b.slice * muon::kBK, n - j * b.slice * muon::kBK) : n;
        it.out = slices > 1 ? const_cast<__half*>(b.sums.item[sum].part) + 2 * j * w[i].square
                            : w[i].sq[kGram].p;
        it.plane = w[i].square;
        it.ld = w[i].ld_square;
        it.scale = T / X;
        it.part = slices > 1;
      }
      sum += slices > 1;
    }
    AGPU_TRY(product(dev, Mode::Gram, g, s));
    if (b.summed) {
      AGPU_CUDA(launch_after(muon_sum_kernel, (uint64_t)b.summed * b.sums.blocks, kThreads, 0, s,
                             b.sums));
      AGPU_TRY(after_launch(dev, "muon_sum_kernel"));
    }
    for (int j = 0; j < len; ++j) {
      const int poly = j ? kPoly : total;
      g.count = 0;
      add_mul(poly, kGram, kGram, muon::kC * T * (M / (X * X)));
      for (int i = 0; i < count; ++i) g.item[i].g = w[i].sq[kGram].p;
      AGPU_TRY(product(dev, Mode::Poly, g, s));
      g.count = 0;
      if (j + 1 < len) add_mul(kPolyGram, poly, kGram, T / M);
      if (j) {
        const float next = total_scale / 4;  // |polynomial| <= 3.45 a step
        add_mul(3 - total, poly, total, T * (next / (M * total_scale)));
        total = 3 - total;
        total_scale = next;
      }
      if (g.count) AGPU_TRY(product(dev, Mode::Mul, g, s));
      if (j + 1 < len) {  // A of the next step
        g.count = 0;
        add_mul(kGram, poly, kPolyGram, T / M);
        AGPU_TRY(product(dev, Mode::Mul, g, s));
      }
    }
    g.count = count;
    for (int i = 0; i < count; ++i) {  // times X
      Item& it = g.item[i];
      it.a = w[i].sq[total].k;
      it.at = w[i].sq[total].n;
      it.bt = w[i].xn[cur];
      it.m = it.k = w[i].src.m;
      it.n = w[i].src.n;
      it.out = w[i].x[1 - cur];
      it.plane = w[i].src.plane;
      it.ld = w[i].src.ld;
      it.scale = T / total_scale;
      it.part = 0;
      it.w = w[i].w;
      it.decay = w[i].decay;
      it.gain = T * (w[i].gain / (X * total_scale));
      it.w_transposed = w[i].src.rows > w[i].src.cols;
    }
    if (seg + 1 < segments) AGPU_TRY(product(dev, Mode::Step, g, s));
    else AGPU_TRY(product(dev, Mode::Update, g, s));
  }
  return AGPU_OK;
}

// Scratch of a call, given back when it returns.
struct Scratch {
  agpu_device* dev;
  cudaStream_t s;
  void* p = nullptr;
  ~Scratch() { pool_free(dev, p, s); }
};

// Matrices of at most 128 x 4096, each by a cluster of CTAs in one launch; the
// ones with equally many CTAs together.  Against the grouped products: one 64 x
// 256 takes 53 us instead of 100, one 128 x 2048 95 instead of 150, forty of
// them 287 instead of 625, 148 of 128 x 256 136 instead of 1290; clusters of 16:
// one 28 x 3050 68 instead of 138, one 128 x 4096 105 instead of 174, 24 of them
// 424 instead of 538.
void set_cluster(cudaLaunchConfig_t& cfg, cudaLaunchAttribute& attr, int count, int cluster,
                 cudaStream_t s) {
  cfg = {};
  cfg.gridDim = dim3((unsigned)(count * cluster), 1, 1);
  cfg.blockDim = dim3(muon::kSmallThreads, 1, 1);
  cfg.dynamicSmemBytes = muon::kSmallSmem;
  cfg.stream = s;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
}

// The largest cluster the device takes: above 8 CTAs that depends on how many
// SMs its groups have.  Asked once per device.
agpu_status largest_cluster(agpu_device* dev, int* most) {
  static std::atomic<int> known[64];
  std::atomic<int>& k = known[dev->ordinal & 63];
  *most = k.load(std::memory_order_acquire);
  if (*most) return AGPU_OK;
  AGPU_CUDA(cudaFuncSetAttribute(muon::muon_small_kernel,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, muon::kSmallSmem));
  AGPU_CUDA(cudaFuncSetAttribute(muon::muon_small_kernel,
                                 cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr;
  int clusters = 0;
  set_cluster(cfg, attr, 1, muon::kSmallCluster, nullptr);
  AGPU_CUDA(cudaOccupancyMaxActiveClusters(&clusters, muon::muon_small_kernel, &cfg));
  *most = clusters ? muon::kSmallCluster : 8;
  k.store(*most, std::memory_order_release);
  return AGPU_OK;
}

bool is_small(const Source& s, int cluster) {
  return s.m <= muon::kSmallRows && s.n <= muon::kSmallCols * cluster;
}

agpu_status run_small(agpu_device* dev, const std::vector<Work>& all, float mu, bool nesterov,
                      uint32_t steps, cudaStream_t s) {
  muon::SmallItems g = {};
  g.mu = mu;
  g.nesterov = nesterov;
  g.steps = (int)steps;
  for (int cluster = 1; cluster <= muon::kSmallCluster; ++cluster) {
    int count = 0;
    for (size_t i = 0; i <= all.size(); ++i) {
      if (count == muon::kSmallItems || (i == all.size() && count)) {
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr;
        set_cluster(cfg, attr, count, cluster, s);
        AGPU_CUDA(cudaLaunchKernelEx(&cfg, muon::muon_small_kernel, g, cluster, dev->d_status));
        AGPU_TRY(after_launch(dev, "muon_small_kernel"));
        count = 0;
      }
      if (i == all.size()) break;
      const Source& t = all[i].src;
      if ((t.n + muon::kSmallCols - 1) / muon::kSmallCols != cluster) continue;
      g.item[count++] = {t.grad, t.momentum, all[i].w, t.m, t.n, t.rows > t.cols, all[i].decay,
                         all[i].gain};
    }
  }
  return AGPU_OK;
}

// w = decay * w + gain * (orthogonalised update) of every matrix.  All that can
// run out (host memory, scratch) is taken before the first launch, as much
// scratch as the largest batch needs: a call that fails has stepped no matrix.
agpu_status run_all(agpu_device* dev, std::vector<Work>& all, float mu, bool nesterov,
                    uint32_t steps, cudaStream_t s) {
  for (Work& t : all) {
    Source& src = t.src;
    src.m = std::min(src.rows, src.cols);
    src.n = std::max(src.rows, src.cols);
    if (src.n > 0x7fffff00) return fail(AGPU_ERR_UNSUPPORTED, "orthogonalize: too large");
    src.ld = (src.n + 63) / 64 * 64;
    src.plane = (long long)src.m * src.ld;
    t.ld_square = (src.m + 63) / 64 * 64;
    t.square = (long long)src.m * t.ld_square;
    t.squares = 2;
  }
  // Small matrices on their own, unless they fit beside larger ones, whose
  // launches are made anyway: 1024 x 1024 takes 275 us, with four of 64 x 256
  // 277, and 335 if these go on their own (2048 x 2048 with 128 x 2048: 583, 673).
  std::vector<Work> small, large;
  int cluster = 0;
  AGPU_TRY(largest_cluster(dev, &cluster));
  for (const Work& t : all) (is_small(t.src, cluster) ? small : large).push_back(t);
  if (large.empty() || all.size() > (size_t)muon::kMaxItems) all.swap(large);
  else small.clear();
  // long contractions first, so that the last wave of a launch is short
  std::stable_sort(all.begin(), all.end(), [](const Work& a, const Work& b) {
    return a.src.m != b.src.m ? a.src.m > b.src.m : a.src.n > b.src.n;
  });
  // Steps on the Gram matrix for wide matrices, if there are enough of them
  // to fill the SMs by themselves.
  std::vector<Work> wide, rest;
  long long pairs = 0;
  for (const Work& t : all) {
    const bool is_wide = steps > 1 && t.src.m >= kGramRows && t.src.n >= (3ll * t.src.m) / 2;
    (is_wide ? wide : rest).push_back(t);
    if (is_wide) pairs += count_tiles(Mode::Gram, t.src.m, t.src.m, 256);
  }
  std::vector<Batch> batches;
  if (pairs < dev->sm_count / 2) {
    plan_batches(dev, all, false, batches);
  } else {
    for (Work& t : wide) t.squares = 5;
    plan_batches(dev, wide, true, batches);
    plan_batches(dev, rest, false, batches);
  }
  size_t bytes = 0;
  for (const Batch& b : batches) bytes = std::max(bytes, b.bytes());
  Scratch scratch = {dev, s};
  if (bytes) AGPU_TRY(pool_alloc(dev, bytes, &scratch.p, s));
  for (Batch& b : batches) AGPU_TRY(prepare_batch(dev, b, scratch.p, mu, nesterov));
  AGPU_TRY(run_small(dev, small, mu, nesterov, steps, s));
  for (const Batch& b : batches) AGPU_TRY(run_batch(dev, b, steps, s));
  return AGPU_OK;
}

}  // namespace

agpu_status launch_orthogonalize(agpu_device* dev, const float* x, float* out, uint32_t batch,
                                 uint32_t rows, uint32_t cols, uint32_t steps,
                                 cudaStream_t s) try {
  const size_t n = (size_t)rows * cols;
  if (n == 0) return AGPU_OK;
  std::vector<Work> all(batch);
  for (uint32_t i = 0; i < batch; ++i) {
    all[i].src = {x + i * n, nullptr, nullptr, 0, 0, (int)rows, (int)cols, 0, 0};
    all[i].w = out + i * n;
    all[i].decay = 0.0f;
    all[i].gain = 1.0f;
  }
  return run_all(dev, all, 0.0f, false, steps, s);
} catch (const std::exception&) {
  return fail(AGPU_ERR_OOM, "orthogonalize: out of host memory");
}

agpu_status launch_muon(agpu_device* dev, const agpu_muon_tensor* t, uint32_t count, float lr,
                        float momentum, bool nesterov, float weight_decay, uint32_t steps,
                        cudaStream_t s) try {
  std::vector<Work> all;
  all.reserve(count);
  for (uint32_t i = 0; i < count; ++i) {
    if ((uint64_t)t[i].rows * t[i].cols == 0) continue;
    Work w = {};
    w.src = {t[i].grad, t[i].momentum, nullptr, 0, 0, (int)t[i].rows, (int)t[i].cols, 0, 0};
    w.w = t[i].param;
    w.decay = 1.0f - lr * weight_decay;
    w.gain = -lr * 0.2f * std::sqrt((float)std::max(t[i].rows, t[i].cols));
    all.push_back(w);
  }
  return run_all(dev, all, momentum, nesterov, steps, s);
} catch (const std::exception&) {
  return fail(AGPU_ERR_OOM, "muon_step: out of host memory");
}

}  // namespace agpu
