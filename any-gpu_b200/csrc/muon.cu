// Orthogonalised updates: the quintic Newton-Schulz iteration and the
// optimiser step built on it.  No counterpart in the reference crate (its
// optimiser is AdamW, src/optim.rs); it stands beside agpu_adamw_step for the
// matrices of a model.  For a matrix W with gradient G and momentum M:
//   M <- mu M + (1 - mu) G,   U = (1 - mu) G + mu M (nesterov) or M
//   X = U / max(|U|_F, 1e-30), then `steps` times (rows <= cols; else on X^T)
//       A = X X^T,  X <- a X + (b A + c A A) X
//   W <- (1 - lr wd) W - lr 0.2 sqrt(max(rows, cols)) X
// which drives the singular values of X towards 1.
#include <algorithm>
#include <cmath>
#include <vector>

#include "agpu_internal.cuh"

namespace agpu {

namespace {

constexpr int kThreads = 256;
constexpr int kParts = 1024;  // CTAs (and partial sums) of a norm
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr double kNormFloor = 1e-30;

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

// u = the update (momentum applied when there is one), and its squares' sums
// per CTA, in double: a gradient's squares leave the range of a float.
__global__ void __launch_bounds__(kThreads)
    muon_update_kernel(const float* __restrict__ grad, float* __restrict__ momentum,
                       float* __restrict__ u, long long n, float mu, bool nesterov,
                       double* __restrict__ partial) {
  __shared__ double red[kThreads / 32];
  double s = 0.0;
  for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < n;
       i += (long long)gridDim.x * kThreads) {
    float v = grad[i];
    if (momentum) {
      const float m = mu * momentum[i] + (1.0f - mu) * v;
      momentum[i] = m;
      v = nesterov ? (1.0f - mu) * v + mu * m : m;
    }
    u[i] = v;
    s += (double)v * v;
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ void __launch_bounds__(kThreads)
    muon_normalise_kernel(float* __restrict__ u, long long n, const double* __restrict__ partial,
                          int parts) {
  __shared__ double red[kThreads / 32];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) s += partial[i];
  const float inv = (float)(1.0 / fmax(sqrt(block_sum(s, red)), kNormFloor));
  for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < n;
       i += (long long)gridDim.x * kThreads)
    u[i] *= inv;
}

// y = p x + q y; y is only written when q is 0
__global__ void __launch_bounds__(kThreads)
    muon_axpby_kernel(const float* __restrict__ x, float* __restrict__ y, long long n, float p,
                      float q) {
  for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < n;
       i += (long long)gridDim.x * kThreads)
    y[i] = q != 0.0f ? p * x[i] + q * y[i] : p * x[i];
}

unsigned grid_for(long long n) {
  return (unsigned)std::max<long long>(1, std::min<long long>((n + kThreads - 1) / kThreads,
                                                              kParts));
}

struct PrecisionScope {
  int saved;
  explicit PrecisionScope(int mode) : saved(g_thread_precision) { g_thread_precision = mode; }
  ~PrecisionScope() { g_thread_precision = saved; }
};

// X (scratch [rows, cols]) through the iteration; y, a, b are scratch.
agpu_status iterate(agpu_device* dev, float*& x, float*& y, float* a, float* b, uint32_t rows,
                    uint32_t cols, uint32_t steps, cudaStream_t s) {
  const bool tall = rows > cols;
  const uint32_t m = tall ? cols : rows, n = tall ? rows : cols;
  const long long mm = (long long)m * m, mn = (long long)m * n;
  PrecisionScope scope(AGPU_PREC_FFMA);
  for (uint32_t i = 0; i < steps; ++i) {
    AGPU_TRY(launch_gemm(dev, x, x, a, 1, m, m, n, tall, !tall, s));
    AGPU_TRY(launch_gemm(dev, a, a, b, 1, m, m, m, false, false, s));
    muon_axpby_kernel<<<grid_for(mm), kThreads, 0, s>>>(a, b, mm, kB, kC);
    AGPU_TRY(after_launch(dev, "muon_axpby_kernel"));
    if (tall) AGPU_TRY(launch_gemm(dev, x, b, y, 1, n, m, m, false, false, s));
    else AGPU_TRY(launch_gemm(dev, b, x, y, 1, m, n, m, false, false, s));
    muon_axpby_kernel<<<grid_for(mn), kThreads, 0, s>>>(x, y, mn, kA, 1.0f);
    AGPU_TRY(after_launch(dev, "muon_axpby_kernel"));
    std::swap(x, y);
  }
  return AGPU_OK;
}

// out = decay * out + gain * (orthogonalised update)
agpu_status update(agpu_device* dev, const float* grad, float* momentum, float* out, uint32_t rows,
                   uint32_t cols, float mu, bool nesterov, float decay, float gain,
                   uint32_t steps, cudaStream_t s) {
  const long long n = (long long)rows * cols;
  if (n == 0) return AGPU_OK;
  const long long m = std::min(rows, cols);
  void* scratch = nullptr;
  AGPU_TRY(pool_alloc(dev, kParts * sizeof(double) + (2 * n + 2 * m * m) * sizeof(float), &scratch,
                      s));
  double* partial = static_cast<double*>(scratch);
  float* x = reinterpret_cast<float*>(partial + kParts);
  float *a = x + n, *b = a + m * m, *y = b + m * m;
  auto run = [&]() -> agpu_status {
    const unsigned grid = grid_for(n);
    muon_update_kernel<<<grid, kThreads, 0, s>>>(grad, momentum, x, n, mu, nesterov, partial);
    AGPU_TRY(after_launch(dev, "muon_update_kernel"));
    muon_normalise_kernel<<<grid, kThreads, 0, s>>>(x, n, partial, (int)grid);
    AGPU_TRY(after_launch(dev, "muon_normalise_kernel"));
    AGPU_TRY(iterate(dev, x, y, a, b, rows, cols, steps, s));
    muon_axpby_kernel<<<grid, kThreads, 0, s>>>(x, out, n, gain, decay);
    return after_launch(dev, "muon_axpby_kernel");
  };
  const agpu_status st = run();
  pool_free(dev, scratch, s);
  return st;
}

}  // namespace

agpu_status launch_orthogonalize(agpu_device* dev, const float* x, float* out, uint32_t batch,
                                 uint32_t rows, uint32_t cols, uint32_t steps, cudaStream_t s) {
  const size_t n = (size_t)rows * cols;
  for (uint32_t i = 0; i < batch; ++i)
    AGPU_TRY(update(dev, x + i * n, nullptr, out + i * n, rows, cols, 0.f, false, 0.f, 1.f, steps,
                    s));
  return AGPU_OK;
}

agpu_status launch_muon(agpu_device* dev, const agpu_muon_tensor* t, uint32_t count, float lr,
                        float momentum, bool nesterov, float weight_decay, uint32_t steps,
                        cudaStream_t s) {
  for (uint32_t i = 0; i < count; ++i)
    AGPU_TRY(update(dev, t[i].grad, t[i].momentum, t[i].param, t[i].rows, t[i].cols, momentum,
                    nesterov, 1.0f - lr * weight_decay,
                    -lr * 0.2f * std::sqrt((float)std::max(t[i].rows, t[i].cols)), steps, s));
  return AGPU_OK;
}

}  // namespace agpu
