// Token embedding: the lookup and its gradient.  No counterpart in the
// reference crate (its tape starts from dense leaves).
//
//   lookup     out[t, :] = scale * table[ids[t], :]
//   gradient   d_table[v, :] (+)= scale * sum over { t : ids[t] = v } of grad_out[t, :]
//
// ids[t] = -1 is padding: a zero row in the lookup, no term in the gradient.
// Any other id outside [0, vocab) counts as padding too and records
// AGPU_BAD_TOKEN_CODE in the device status word.
//
// The gradient sums each table row's tokens in a fixed order (by position,
// in fixed chunks), so it is deterministic: the tokens are sorted by id first
// instead of being added with floating-point atomics.
#include <algorithm>

#include "agpu_internal.cuh"

namespace agpu {

namespace {

constexpr int kThreads = 256;
constexpr int kIndexWarps = 32;      // warps of an index CTA
constexpr int kMaxRowsPerCta = 1024; // table rows of an index CTA (one thread scans one)
constexpr int kChunk = 32;           // sorted positions summed by one CTA
constexpr int kInFlight = 8;         // gradient rows a thread has in flight

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

__device__ __forceinline__ float4 zero(float4) { return make_float4(0.f, 0.f, 0.f, 0.f); }
__device__ __forceinline__ float zero(float) { return 0.f; }
__device__ __forceinline__ float4 times(float4 a, float s) {
  return make_float4(a.x * s, a.y * s, a.z * s, a.w * s);
}
__device__ __forceinline__ float times(float a, float s) { return a * s; }
__device__ __forceinline__ float4 plus(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
__device__ __forceinline__ float plus(float a, float b) { return a + b; }

// ---------------------------------------------------------------- lookup --
// V = float4 (dim and pointers allow it) or float; `dv` = row length in V.
// A CTA covers J * 256 consecutive V of the output, so one 64-bit division
// finds its first row and the rest is 32-bit.
template <typename V, int J>
__global__ void __launch_bounds__(kThreads)
    embedding_kernel(const V* __restrict__ table, const int* __restrict__ ids,
                     V* __restrict__ out, long long total, unsigned dv, unsigned vocab,
                     float scale, unsigned int* status) {
  const long long base = (long long)blockIdx.x * (kThreads * J);
  const long long t0 = base / dv;
  const unsigned r0 = (unsigned)(base - t0 * dv);
  V v[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const unsigned off = j * kThreads + threadIdx.x;
    v[j] = zero(V());
    if (base + off < total) {
      const unsigned q = (r0 + off) / dv, c = (r0 + off) - q * dv;
      const int id = __ldg(ids + t0 + q);
      if ((unsigned)id < vocab) v[j] = __ldg(table + (long long)id * dv + c);
      else if (id != -1) atomicCAS(status, 0u, AGPU_BAD_TOKEN_CODE);
    }
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const unsigned off = j * kThreads + threadIdx.x;
    if (base + off < total) __stcs(out + base + off, times(v[j], scale));
  }
}

// -------------------------------------------------------------- gradient --
// Stable counting sort of the token positions by id.  Each CTA owns the
// table rows [lo, lo + rows) and reads all ids itself, twice: it counts its
// own rows' tokens per warp (a warp owns a contiguous range of positions, so
// warp order is position order) and the tokens of lower rows, which is where
// its output starts; then it places its tokens.  No CTA waits for another.
//   order[p] = token position, sorted[p] = its id, for p in sorted order
//   starts[v] = first p of row v, starts[vocab] = number of tokens with a row
__global__ void __launch_bounds__(kIndexWarps * 32)
    embedding_index_kernel(const int* __restrict__ ids, int tokens, int vocab, int rows,
                           int* __restrict__ order, int* __restrict__ sorted,
                           int* __restrict__ starts, unsigned int* status) {
  extern __shared__ int count[];  // [kIndexWarps][rows]
  __shared__ int red[kIndexWarps];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int lo = blockIdx.x * rows, hi = min(lo + rows, vocab);
  for (int i = tid; i < kIndexWarps * rows; i += blockDim.x) count[i] = 0;
  __syncthreads();

  const int per = ((tokens + kIndexWarps - 1) / kIndexWarps + 31) / 32 * 32;
  const long long p0 = (long long)warp * per;
  const int begin = (int)min((long long)tokens, p0), end = (int)min((long long)tokens, p0 + per);
  int* mine = count + warp * rows;
  int below = 0;
  for (int i = begin + lane; i < end; i += 32) {
    const int id = __ldg(ids + i);
    if (id >= lo && id < hi) atomicAdd(mine + (id - lo), 1);
    below += id >= 0 && id < lo;
    if (blockIdx.x == 0 && (id < -1 || id >= vocab)) atomicCAS(status, 0u, AGPU_BAD_TOKEN_CODE);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
  if (lane == 0) red[warp] = below;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kIndexWarps; ++w) base += red[w];
  __syncthreads();

  // thread r: row r's total, then an exclusive scan over the rows
  int total = 0;
  if (tid < rows)
    for (int w = 0; w < kIndexWarps; ++w) total += count[w * rows + tid];
  int scan = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += up;
  }
  if (lane == 31) red[warp] = scan;
  __syncthreads();
  for (int w = 0; w < warp; ++w) scan += red[w];
  int first = base + scan - total;
  if (tid < rows) {
    if (lo + tid < vocab) starts[lo + tid] = first;
    if (lo + tid == vocab - 1) starts[vocab] = first + total;
    for (int w = 0; w < kIndexWarps; ++w) {  // counts become output offsets
      const int n = count[w * rows + tid];
      count[w * rows + tid] = first;
      first += n;
    }
  }
  __syncthreads();

  for (int i0 = begin; i0 < end; i0 += 32) {
    const int i = i0 + lane;
    const int id = i < end ? __ldg(ids + i) : -1;
    const bool in = id >= lo && id < hi;
    if (__ballot_sync(0xffffffffu, in) == 0) continue;
    // lanes with the same row keep their order; other lanes match only themselves
    const unsigned same = __match_any_sync(0xffffffffu, in ? id : -1 - lane);
    const int rank = __popc(same & ((1u << lane) - 1));
    const int at = in ? mine[id - lo] : 0;
    __syncwarp();
    if (in) {
      order[at + rank] = i;
      sorted[at + rank] = id;
      if (rank == 0) mine[id - lo] = at + __popc(same);
    }
    __syncwarp();
  }
}

// CTA b < sum_blocks: chunk b / slices of the sorted positions, columns of
// slice b % slices (one V per thread).  Rows that lie inside the chunk are
// written; a row that crosses into or out of it leaves its part in
//   partial[2 * chunk]      the row that began in an earlier chunk
//   partial[2 * chunk + 1]  the row that begins here and goes on
// for embedding_join_kernel.  The other CTAs write zeros to the rows without
// tokens (none of them when accumulating).
template <typename V>
__global__ void __launch_bounds__(kThreads)
    embedding_sum_kernel(const V* __restrict__ grad, const int* __restrict__ order,
                         const int* __restrict__ sorted, const int* __restrict__ starts,
                         V* __restrict__ d_table, V* __restrict__ partial, int vocab, int dv,
                         int slices, long long sum_blocks, int zero_rows, bool accumulate,
                         float scale) {
  const int tid = threadIdx.x;
  if ((long long)blockIdx.x >= sum_blocks) {
    const long long v0 = (blockIdx.x - sum_blocks) * zero_rows;
    const int n = (int)min((long long)zero_rows, vocab - v0);
    for (int r = 0; r < n; ++r) {
      if (__ldg(starts + v0 + r) != __ldg(starts + v0 + r + 1)) continue;
      V* row = d_table + (v0 + r) * dv;
      for (int c = tid; c < dv; c += kThreads) __stcs(row + c, zero(V()));
    }
    return;
  }
  __shared__ int tok[kChunk], row[kChunk + 2];  // row[0] = the position before the chunk
  const long long chunk = blockIdx.x / slices;
  const int col = (int)(blockIdx.x % slices) * kThreads + tid;
  const int n = __ldg(starts + vocab);
  const long long p0 = chunk * kChunk;
  if (p0 >= n) return;
  const int len = (int)min((long long)kChunk, n - p0);
  if (tid < len) tok[tid] = order[p0 + tid];
  if (tid < len + 2) {
    const long long p = p0 - 1 + tid;
    row[tid] = p >= 0 && p < n ? sorted[p] : -1;
  }
  __syncthreads();
  if (col >= dv) return;

  bool head = row[0] == row[1];  // the first row began in an earlier chunk
  V acc = zero(V());
  for (int i0 = 0; i0 < len; i0 += kInFlight) {
    V g[kInFlight], d[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int i = i0 + u;
      if (i < len) {
        g[u] = __ldcs(grad + (long long)tok[i] * dv + col);
        if (accumulate && row[i + 1] != row[i + 2])
          d[u] = d_table[(long long)row[i + 1] * dv + col];
      }
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int i = i0 + u;
      if (i < len) {
        acc = plus(acc, g[u]);
        const bool ends = row[i + 1] != row[i + 2];
        if (ends && !head) {
          V y = times(acc, scale);
          if (accumulate) y = plus(d[u], y);
          __stcs(d_table + (long long)row[i + 1] * dv + col, y);
        } else if (ends || i == len - 1) {
          partial[(2 * chunk + (head ? 0 : 1)) * dv + col] = acc;
        }
        if (ends) {
          acc = zero(V());
          head = false;
        }
      }
    }
  }
}

// The rows that cross chunks: the CTAs of the chunk a row begins in add its
// parts in chunk order.
template <typename V>
__global__ void __launch_bounds__(kThreads)
    embedding_join_kernel(const int* __restrict__ sorted, const int* __restrict__ starts,
                          const V* __restrict__ partial, V* __restrict__ d_table, int vocab,
                          int dv, int slices, bool accumulate, float scale) {
  const long long chunk = blockIdx.x / slices;
  const int col = (int)(blockIdx.x % slices) * kThreads + threadIdx.x;
  const int n = __ldg(starts + vocab);
  const long long p1 = (chunk + 1) * kChunk;
  if (p1 >= n || col >= dv) return;
  const int row = __ldg(sorted + p1);
  const int first = __ldg(starts + row);
  if (first < chunk * kChunk || first >= p1) return;  // begins in another chunk
  const long long last = (__ldg(starts + row + 1) - 1) / kChunk;
  V acc = partial[(2 * chunk + 1) * dv + col];
  for (long long k = chunk + 1; k <= last; k += kInFlight) {
    V part[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (k + u <= last) part[u] = partial[2 * (k + u) * dv + col];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (k + u <= last) acc = plus(acc, part[u]);
  }
  V y = times(acc, scale);
  V* dst = d_table + (long long)row * dv + col;
  if (accumulate) y = plus(*dst, y);
  *dst = y;
}

template <typename V>
agpu_status lookup(agpu_device* dev, const float* table, const int32_t* ids, float* out,
                   uint64_t tokens, uint32_t vocab, uint32_t dv, float scale, cudaStream_t s) {
  const uint64_t total = tokens * dv;
  const uint64_t blocks4 = ceil_div(total, kThreads * 4);
  if (blocks4 > 0x7fffffffull) return fail(AGPU_ERR_UNSUPPORTED, "embedding: output too large");
  const V* tb = reinterpret_cast<const V*>(table);
  V* o = reinterpret_cast<V*>(out);
  // four V per thread once that still gives every SM eight CTAs; below it the
  // call is bound by latency and more CTAs with one load each finish sooner
  if (blocks4 >= 8ull * dev->sm_count)
    embedding_kernel<V, 4><<<(unsigned)blocks4, kThreads, 0, s>>>(
        tb, ids, o, (long long)total, dv, vocab, scale, dev->d_status);
  else
    embedding_kernel<V, 1><<<(unsigned)ceil_div(total, kThreads), kThreads, 0, s>>>(
        tb, ids, o, (long long)total, dv, vocab, scale, dev->d_status);
  return after_launch(dev, "embedding_kernel");
}

template <typename V>
agpu_status gradient(agpu_device* dev, const float* grad_out, const int32_t* ids, float* d_table,
                     int tokens, int vocab, uint32_t dv, float scale, bool accumulate,
                     cudaStream_t s) {
  const int rows = (int)std::min<uint64_t>(
      kMaxRowsPerCta, std::max<uint64_t>(32, ceil_div(vocab, dev->sm_count)));
  const uint64_t chunks = ceil_div(tokens, kChunk), slices = ceil_div(dv, kThreads);
  const uint64_t sum_blocks = chunks * slices;
  const int zero_rows = std::max<int>(1, 4096 / (int)dv);
  const uint64_t zero_blocks = accumulate ? 0 : ceil_div(vocab, zero_rows);
  if (sum_blocks + zero_blocks > 0x7fffffffull)
    return fail(AGPU_ERR_UNSUPPORTED, "embedding_backward: too large");
  const size_t ints = (2ull * tokens + vocab + 1 + 3) / 4 * 4;
  void* scratch = nullptr;
  AGPU_TRY(pool_alloc(dev, ints * 4 + 2 * chunks * dv * sizeof(V), &scratch, s));
  int* order = static_cast<int*>(scratch);
  int *sorted = order + tokens, *starts = sorted + tokens;
  V* partial = reinterpret_cast<V*>(order + ints);
  const int smem = kIndexWarps * rows * (int)sizeof(int);
  cudaError_t e =
      set_smem_once<embedding_index_kernel>(dev, kIndexWarps * kMaxRowsPerCta * sizeof(int));
  agpu_status st = e == cudaSuccess ? AGPU_OK : cuda_status(e, "embedding_backward");
  if (st == AGPU_OK) {
    embedding_index_kernel<<<(unsigned)ceil_div(vocab, rows), kIndexWarps * 32, smem, s>>>(
        ids, tokens, vocab, rows, order, sorted, starts, dev->d_status);
    st = after_launch(dev, "embedding_index_kernel");
  }
  const V* g = reinterpret_cast<const V*>(grad_out);
  V* d = reinterpret_cast<V*>(d_table);
  if (st == AGPU_OK) {
    embedding_sum_kernel<V><<<(unsigned)(sum_blocks + zero_blocks), kThreads, 0, s>>>(
        g, order, sorted, starts, d, partial, vocab, (int)dv, (int)slices, (long long)sum_blocks,
        zero_rows, accumulate, scale);
    st = after_launch(dev, "embedding_sum_kernel");
  }
  if (st == AGPU_OK && chunks > 1) {
    embedding_join_kernel<V><<<(unsigned)sum_blocks, kThreads, 0, s>>>(
        sorted, starts, partial, d, vocab, (int)dv, (int)slices, accumulate, scale);
    st = after_launch(dev, "embedding_join_kernel");
  }
  pool_free(dev, scratch, s);
  return st;
}

}  // namespace

agpu_status launch_embedding(agpu_device* dev, const float* table, const int32_t* ids, float* out,
                             uint64_t tokens, uint32_t vocab, uint32_t dim, float scale,
                             cudaStream_t s) {
  if (tokens == 0 || dim == 0) return AGPU_OK;
  if (dim % 4 == 0 && aligned16(table) && aligned16(out))
    return lookup<float4>(dev, table, ids, out, tokens, vocab, dim / 4, scale, s);
  return lookup<float>(dev, table, ids, out, tokens, vocab, dim, scale, s);
}

agpu_status launch_embedding_backward(agpu_device* dev, const float* grad_out, const int32_t* ids,
                                      float* d_table, uint64_t tokens, uint32_t vocab,
                                      uint32_t dim, float scale, bool accumulate,
                                      cudaStream_t s) {
  if (vocab == 0 || dim == 0) return AGPU_OK;
  if (tokens == 0) {
    if (!accumulate)
      AGPU_CUDA(cudaMemsetAsync(d_table, 0, (size_t)vocab * dim * sizeof(float), s));
    return AGPU_OK;
  }
  if (dim % 4 == 0 && aligned16(grad_out) && aligned16(d_table))
    return gradient<float4>(dev, grad_out, ids, d_table, (int)tokens, (int)vocab, dim / 4, scale,
                            accumulate, s);
  return gradient<float>(dev, grad_out, ids, d_table, (int)tokens, (int)vocab, dim, scale,
                         accumulate, s);
}

}  // namespace agpu
