// Token embedding: the lookup and its gradient.  No counterpart in the
// reference crate (its tape starts from dense leaves).
//
//   lookup     out[t, :] = scale * table[ids[t], :]
//   gradient   d_table[v, :] (+)= scale * sum over { t : ids[t] = v } of grad_out[t, :]
//
// ids[t] = -1 is padding: a zero row in the lookup, no term in the gradient.
// Any other id outside [0, vocab) counts as padding too and records
// AGPU_BAD_TOKEN_CODE in a device status word of its own.
//
// The gradient sums each table row's tokens in a fixed order (by position,
// in fixed chunks), so it is deterministic: the tokens are sorted by id first
// instead of being added with floating-point atomics.
#include <algorithm>
#include <type_traits>

#include "agpu_internal.cuh"
#include "ptx.cuh"

namespace agpu {

namespace {

constexpr int kThreads = 256;
constexpr int kIndexWarps = 32;      // warps of an index CTA
constexpr int kMaxRowsPerCta = 1024; // table rows of an index CTA (one thread scans one)
constexpr int kMinOwners = 128;      // index CTAs, a power of two
constexpr int kQueue = 64;           // tokens a warp of the index holds back
constexpr int kJoinGroups = 4;       // groups of a join CTA, each a part of a row's parts
constexpr int kMaxChunk = 64;        // sorted positions summed by one CTA, at most
constexpr int kInFlight = 8;         // gradient rows a thread has in flight
constexpr int kIdsAhead = 8;         // ids a thread of the index has in flight
static_assert(0x7fffff00ll + 32 * kIdsAhead <= 0x80000000ll, "an int holds every position");
constexpr int kFewCtas = 4;          // its CTAs on an SM
constexpr int kFewTokens = 256;      // tokens of the one-launch gradient, at most
constexpr int kFewRows = 16;         // table rows of one of its CTAs, at most

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

__device__ __forceinline__ float4 zero(float4) { return make_float4(0.f, 0.f, 0.f, 0.f); }
__device__ __forceinline__ float zero(float) { return 0.f; }
__device__ __forceinline__ float4 times(float4 a, float s) {
  return make_float4(a.x * s, a.y * s, a.z * s, a.w * s);
}
__device__ __forceinline__ float times(float a, float s) { return a * s; }
__device__ __forceinline__ float4 pick(bool c, float4 a) {
  return make_float4(c ? a.x : 0.f, c ? a.y : 0.f, c ? a.z : 0.f, c ? a.w : 0.f);
}
__device__ __forceinline__ float pick(bool c, float a) { return c ? a : 0.f; }
__device__ __forceinline__ float4 plus(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
__device__ __forceinline__ float plus(float a, float b) { return a + b; }

// ---------------------------------------------------------------- lookup --
// V = float4 (dim and pointers allow it) or float; `dv` = row length in V.
// Bound by HBM: 32768 tokens of 64000 x 2048 in 56 us, 0.95 of the copy rate.
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
// Few tokens and a table of a few MB: one launch, no scratch.  Each CTA owns
// `rows` table rows and 256 columns, orders the tokens of its rows by (row,
// position) in shared memory, and writes every element: its sum, or zero.
// Bound by latency: 37 tokens into 1001 x 99 take 4.7 us, sorting them 13; 200
// into 1000 x 512 7 and 14.  All 256 tokens on one row are its worst case, 21
// and 14.  In a table of more rows per CTA the zeros take longer than the
// sorting path's: 8 tokens into 32000 x 4096 88 and 76.
template <typename V>
__global__ void __launch_bounds__(kThreads, kFewCtas)
    embedding_few_kernel(const V* __restrict__ grad, const int* __restrict__ ids,
                         V* __restrict__ d_table, int tokens, int vocab, int dv, int rows,
                         int slices, bool accumulate, float scale, unsigned int* status) {
  constexpr int kPer = kFewTokens / kThreads;
  // the CTA's tokens by position: ids and positions; then their order
  __shared__ int id[kFewTokens], pos[kFewTokens], list[kFewTokens], first[kFewRows + 1];
  __shared__ int counts[kPer * kThreads / 32];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int lo = blockIdx.x / slices * rows, n = min(rows, vocab - lo);
  const int col = blockIdx.x % slices * kThreads + tid;
  int mine[kPer];
  unsigned in[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) mine[j] = ptx::load_now(ids + min(j * kThreads + tid, tokens - 1));
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const bool live = j * kThreads + tid < tokens;
    if (blockIdx.x == 0 && live && (mine[j] < -1 || mine[j] >= vocab))
      atomicCAS(status, 0u, AGPU_BAD_TOKEN_CODE);
    in[j] = __ballot_sync(0xffffffffu, live && mine[j] >= lo && mine[j] < lo + n);
    if (lane == 0) counts[j * kThreads / 32 + warp] = __popc(in[j]);
  }
  __syncthreads();
  int found = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w == warp && (in[j] >> lane & 1u)) {
        const int k = found + __popc(in[j] & ((1u << lane) - 1u));
        id[k] = mine[j];
        pos[k] = j * kThreads + tid;
      }
      found += counts[j * kThreads / 32 + w];
    }
  }
  __syncthreads();
  for (int k = tid; k < found; k += kThreads) {
    int rank = 0;
    for (int u = 0; u < found; ++u) rank += id[u] < id[k] || (id[u] == id[k] && u < k);
    list[rank] = pos[k];
  }
  if (tid <= n) {  // tokens of rows before row tid, 0..n <= kFewRows
    int before = 0;
    for (int u = 0; u < found; ++u) before += id[u] < lo + tid;
    first[tid] = before;
  }
  __syncthreads();
  if (col >= dv) return;
  V* dst = d_table + (long long)lo * dv + col;
  auto add = [&](auto most, V& acc, int p, int p1) {
    V g[most];
#pragma unroll
    for (int u = 0; u < most; ++u)
      g[u] = ptx::load_now(grad + (long long)list[min(p + u, p1 - 1)] * dv + col);
#pragma unroll
    for (int u = 0; u < most; ++u) acc = plus(acc, pick(p + u < p1, g[u]));
  };
  for (int r = 0; r < n; ++r, dst += dv) {
    const int p0 = first[r], p1 = first[r + 1];
    if (p0 == p1) {
      if (!accumulate) __stcs(dst, zero(V()));
      continue;
    }
    V acc = zero(V());
    int p = p0;
    for (; p1 - p > kInFlight; p += 2 * kInFlight) 
      add(std::integral_constant<int, 2 * kInFlight>(), acc, p, p1);
    if (p < p1) add(std::integral_constant<int, kInFlight>(), acc, p, p1);
    acc = times(acc, scale);
    if (accumulate) acc = plus(*dst, acc);
    __stcs(dst, acc);
  }
}

// Stable counting sort of the token positions by row.  Row v belongs to CTA
// v % owners (owners a power of two) as its row v / owners: neighbouring ids,
// which are the frequent ones in a text's vocabulary, go to different CTAs (with
// contiguous ranges one CTA had 57% of 65536 such tokens, and took 83 us).  The
// sorted order is by (v % owners, v / owners, position); only that equal ids
// are together matters.  Each CTA reads all ids itself, twice: it counts its own
// rows' tokens per warp (a warp has a contiguous range of positions, so warp
// order is position order) and the tokens of earlier CTAs' rows, which is where
// its output starts; then it places its tokens.  No CTA waits for another.
//   order[p] = token position, sorted[p] = its id, for p in sorted order
//   starts[slot] = first p of the slot of a row (slot_of_row), and behind the
//   last slot the number of tokens with a row
// Positions are ints that step up to 32 * kIdsAhead past the last token, and so
// `tokens` is at most 2^31 - 256 (the caller refuses more).
// Bound by instruction issue: 4096 tokens 9 us, 65536 28.
struct Owners {
  int shift, rows;  // owners = 1 << shift, rows of each
};

__device__ __forceinline__ int slot_of_row(Owners o, int row) {
  return (row & ((1 << o.shift) - 1)) * o.rows + (row >> o.shift);
}

__global__ void __launch_bounds__(kIndexWarps * 32)
    embedding_index_kernel(const int* __restrict__ ids, int tokens, int vocab, Owners own,
                           int* __restrict__ order, int* __restrict__ sorted,
                           int* __restrict__ starts, unsigned int* status) {
  extern __shared__ int count[];  // [kIndexWarps][rows]
  __shared__ int red[kIndexWarps];
  __shared__ int2 queue[kIndexWarps][kQueue];  // (position, id) of tokens to be placed
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int rows = own.rows, mask = (1 << own.shift) - 1, me = blockIdx.x;
  ptx::griddep_launch_dependents();
  for (int i = tid; i < kIndexWarps * rows; i += blockDim.x) count[i] = 0;
  __syncthreads();
  ptx::griddep_wait();

  const int per = ((tokens + kIndexWarps - 1) / kIndexWarps + 31) / 32 * 32;
  const long long p0 = (long long)warp * per;
  const int begin = (int)min((long long)tokens, p0), end = (int)min((long long)tokens, p0 + per);
  int* mine = count + warp * rows;
  int below = 0;
  for (int i0 = begin + lane; i0 < end; i0 += 32 * kIdsAhead) {
    int id[kIdsAhead];
#pragma unroll
    for (int u = 0; u < kIdsAhead; ++u) id[u] = ptx::load_now(ids + min(i0 + 32 * u, end - 1));
#pragma unroll
    for (int u = 0; u < kIdsAhead; ++u) {
      if (i0 + 32 * u >= end) id[u] = -1;
      const bool live = (unsigned)id[u] < (unsigned)vocab;
      const int owner = id[u] & mask;
      if (live && owner == me) atomicAdd(mine + (id[u] >> own.shift), 1);
      below += live && owner < me;
      if (me == 0 && !live && id[u] != -1) atomicCAS(status, 0u, AGPU_BAD_TOKEN_CODE);
    }
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
    starts[me * rows + tid] = first;
    if (me == mask && tid == rows - 1) starts[(mask + 1) * rows] = first + total;
    for (int w = 0; w < kIndexWarps; ++w) {  // counts become output offsets
      const int n = count[w * rows + tid];
      count[w * rows + tid] = first;
      first += n;
    }
  }
  __syncthreads();

  // A warp's tokens gather in its queue, in order, and are placed 32 at a time:
  // ranking equal ids among 32 lanes costs the same for one token as for 32.
  int held = 0;
  auto place = [&](int n) {
    const int2 t = lane < n ? queue[warp][lane] : make_int2(0, -1 - lane);
    const unsigned same = __match_any_sync(0xffffffffu, t.y);
    const int rank = __popc(same & ((1u << lane) - 1));
    const int at = lane < n ? mine[t.y >> own.shift] : 0;
    __syncwarp();
    if (lane < n) {
      order[at + rank] = t.x;
      sorted[at + rank] = t.y;
      if (rank == 0) mine[t.y >> own.shift] = at + __popc(same);
    }
    __syncwarp();
  };
  for (int i0 = begin; i0 < end; i0 += 32 * kIdsAhead) {
    int id[kIdsAhead];
#pragma unroll
    for (int u = 0; u < kIdsAhead; ++u) id[u] = ptx::load_now(ids + min(i0 + 32 * u + lane, end - 1));
#pragma unroll
    for (int u = 0; u < kIdsAhead; ++u) {
      if (i0 + 32 * u + lane >= end) id[u] = -1;
      const bool in = (unsigned)id[u] < (unsigned)vocab && (id[u] & mask) == me;
      const unsigned who = __ballot_sync(0xffffffffu, in);
      if (who == 0) continue;
      if (in)
        queue[warp][held + __popc(who & ((1u << lane) - 1))] =
            make_int2(i0 + 32 * u + lane, id[u]);
      __syncwarp();
      held += __popc(who);
      if (held >= 32) {
        place(32);
        held -= 32;
        const int2 rest = lane < held ? queue[warp][32 + lane] : make_int2(0, 0);
        __syncwarp();
        if (lane < held) queue[warp][lane] = rest;
        __syncwarp();
      }
    }
  }
  if (held) place(held);
}

// CTA b < sum_blocks: 256 / lanes neighbouring chunks of the sorted positions
// (one if a row has 256 V or more), columns of slice b % slices, one V per
// thread.  Rows that lie inside the chunk are
// written; a row that crosses into or out of it leaves its part in
//   partial[2 * chunk]      the row that began in an earlier chunk
//   partial[2 * chunk + 1]  the row that begins here and goes on
// for embedding_join_kernel.  The other CTAs write zeros to the rows without
// tokens (none of them when accumulating).  Bound by HBM: 4096 tokens into
// 32000 x 4096 82 us (524 MB of them the table), 65536 added to 100000 x 1024 65.
template <typename V, bool ACCUMULATE>
__global__ void __launch_bounds__(kThreads, 4)
    embedding_sum_kernel(const V* grad, const int* order, const int* sorted, const int* starts,
                         V* d_table, V* partial, int vocab,
                         Owners own, int dv, int slices, int lanes, int chunk_len,
                         long long sum_blocks, int zero_rows, float scale) {
  constexpr int U = ACCUMULATE ? kInFlight / 2 : kInFlight;
  __shared__ int toks[kThreads / 32][kMaxChunk], rows[kThreads / 32][kMaxChunk + 2];
  const int tid = threadIdx.x;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  if ((long long)blockIdx.x >= sum_blocks) {
    const long long v0 = (blockIdx.x - sum_blocks) * zero_rows;
    const int n = (int)min((long long)zero_rows, vocab - v0) * dv;
    V* base = d_table + v0 * dv;
#pragma unroll 4
    for (int i = tid; i < n; i += kThreads) {
      const int slot = slot_of_row(own, (int)v0 + i / dv);
      if (starts[slot] == starts[slot + 1]) __stcs(base + i, zero(V()));
    }
    return;
  }
  const int group = tid / lanes, lane = tid % lanes;
  const long long chunk = blockIdx.x / slices * (long long)(kThreads / lanes) + group;
  const int col = (int)(blockIdx.x % slices) * kThreads + lane;
  const int n = starts[own.rows << own.shift];
  const long long p0 = chunk * chunk_len;
  const int len = (int)max(0ll, min((long long)chunk_len, n - p0));
  int *tok = toks[group], *row = rows[group];  // row[0] = the position before the chunk
  for (int i = lane; i < len; i += lanes) tok[i] = order[p0 + i];
  if (len > 0)
    for (int i = lane; i < len + 2; i += lanes) {
      const long long p = p0 - 1 + i;
      row[i] = p >= 0 && p < n ? sorted[p] : -1;
    }
  __syncthreads();
  if (col >= dv || len == 0) return;

  bool head = row[0] == row[1];  // the first row began in an earlier chunk
  V acc = zero(V());
  for (int i0 = 0; i0 < len; i0 += U) {
    V g[U], d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i < len) {
        g[u] = __ldcs(grad + (long long)tok[i] * dv + col);
        if (ACCUMULATE && row[i + 1] != row[i + 2])
          d[u] = d_table[(long long)row[i + 1] * dv + col];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i < len) {
        acc = plus(acc, g[u]);
        const bool ends = row[i + 1] != row[i + 2];
        if (ends && !head) {
          V y = times(acc, scale);
          if (ACCUMULATE) y = plus(d[u], y);
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
// parts.  A frequent token's row has hundreds of them, so each of a CTA's
// groups adds a contiguous quarter in chunk order, and the quarters follow.
// Parts come from L2; 8 and 12 us for the sums above.
template <typename V>
__global__ void __launch_bounds__(kThreads)
    embedding_join_kernel(const int* sorted, const int* starts, const V* partial, V* d_table,
                          Owners own,
                          int dv, int slices, int chunk_len, bool accumulate, float scale) {
  constexpr int kCols = kThreads / kJoinGroups;
  __shared__ V sums[kJoinGroups][kCols];
  const long long chunk = blockIdx.x / slices;
  const int group = threadIdx.x / kCols, lane = threadIdx.x % kCols;
  const int col = (int)(blockIdx.x % slices) * kCols + lane;
  ptx::griddep_wait();
  const int n = starts[own.rows << own.shift];
  const long long p1 = (chunk + 1) * chunk_len;
  if (p1 >= n) return;
  const int row = sorted[p1];
  const int slot = slot_of_row(own, row), first = starts[slot];
  if (first < chunk * chunk_len || first >= p1) return;  // begins in another chunk
  // part 0 is the chunk's own, part k the head of chunk `chunk + k`
  const int parts = (int)((starts[slot + 1] - 1) / chunk_len - chunk) + 1;
  const int per = (parts + kJoinGroups - 1) / kJoinGroups;
  V acc = zero(V());
  if (col < dv) {
    const int end = min(parts, (group + 1) * per);
    for (int k = group * per; k < end; k += kInFlight) {
      V part[kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int j = min(k + u, end - 1);
        part[u] = ptx::load_now(partial + (2 * (chunk + j) + (j == 0)) * dv + col);
      }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) acc = plus(acc, pick(k + u < end, part[u]));
    }
  }
  sums[group][lane] = acc;
  __syncthreads();
  if (group != 0 || col >= dv) return;
#pragma unroll
  for (int g = 1; g < kJoinGroups; ++g) acc = plus(acc, sums[g][lane]);
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
        tb, ids, o, (long long)total, dv, vocab, scale, dev->d_status + kTokenStatus);
  else
    embedding_kernel<V, 1><<<(unsigned)ceil_div(total, kThreads), kThreads, 0, s>>>(
        tb, ids, o, (long long)total, dv, vocab, scale, dev->d_status + kTokenStatus);
  return after_launch(dev, "embedding_kernel");
}

template <typename V>
agpu_status gradient(agpu_device* dev, const float* grad_out, const int32_t* ids, float* d_table,
                     int tokens, int vocab, uint32_t dv, float scale, bool accumulate,
                     cudaStream_t s) {
  const uint64_t slices = ceil_div(dv, kThreads);
  const uint64_t per = ceil_div(vocab * slices, (uint64_t)kFewCtas * dev->sm_count);
  if (tokens <= kFewTokens && per <= kFewRows) {
    const uint64_t blocks = ceil_div(vocab, per) * slices;
    embedding_few_kernel<V><<<(unsigned)blocks, kThreads, 0, s>>>(
        reinterpret_cast<const V*>(grad_out), ids, reinterpret_cast<V*>(d_table), tokens, vocab,
        (int)dv, (int)per, (int)slices, accumulate, scale, dev->d_status + kTokenStatus);
    return after_launch(dev, "embedding_few_kernel");
  }
  Owners own = {0, 0};
  while ((1 << own.shift) < kMinOwners ||
         ceil_div(vocab, 1ull << own.shift) > (uint64_t)kMaxRowsPerCta)
    ++own.shift;
  own.rows = (int)ceil_div(vocab, 1ull << own.shift);
  const uint64_t slots = (uint64_t)own.rows << own.shift;
  // long chunks leave fewer parts to join, if there are enough of them
  const int chunk_len =
      ceil_div(tokens, kMaxChunk) * slices >= 4ull * dev->sm_count ? kMaxChunk : kMaxChunk / 2;
  const uint64_t chunks = ceil_div(tokens, chunk_len);
  int lanes = 32;
  while (lanes < (int)dv && lanes < kThreads) lanes *= 2;
  const uint64_t sum_blocks = ceil_div(chunks, kThreads / lanes) * slices;
  const uint64_t join_slices = ceil_div(dv, kThreads / kJoinGroups);
  const int zero_rows = std::max<int>(1, 4096 / (int)dv);
  const uint64_t zero_blocks = accumulate ? 0 : ceil_div(vocab, zero_rows);
  if (sum_blocks + zero_blocks > 0x7fffffffull || chunks * join_slices > 0x7fffffffull)
    return fail(AGPU_ERR_UNSUPPORTED, "embedding_backward: too large");
  const size_t ints = (2ull * tokens + slots + 1 + 3) / 4 * 4;
  void* scratch = nullptr;
  AGPU_TRY(pool_alloc(dev, ints * 4 + 2 * chunks * dv * sizeof(V), &scratch, s));
  int* order = static_cast<int*>(scratch);
  int *sorted = order + tokens, *starts = sorted + tokens;
  V* partial = reinterpret_cast<V*>(order + ints);
  const V* g = reinterpret_cast<const V*>(grad_out);
  V* d = reinterpret_cast<V*>(d_table);
  auto run = [&]() -> agpu_status {
    AGPU_CUDA(set_smem_once<embedding_index_kernel>(dev,
                                                    kIndexWarps * kMaxRowsPerCta * sizeof(int)));
    AGPU_CUDA(launch_after(embedding_index_kernel, 1ull << own.shift, kIndexWarps * 32,
                           kIndexWarps * own.rows * (int)sizeof(int), s, ids, tokens, vocab, own,
                           order, sorted, starts, dev->d_status + kTokenStatus));
    AGPU_TRY(after_launch(dev, "embedding_index_kernel"));
    auto sum = accumulate ? embedding_sum_kernel<V, true> : embedding_sum_kernel<V, false>;
    AGPU_CUDA(launch_after(sum, sum_blocks + zero_blocks, kThreads, 0, s, g, order, sorted, starts,
                           d, partial, vocab, own, (int)dv, (int)slices, lanes, chunk_len,
                           (long long)sum_blocks, zero_rows, scale));
    AGPU_TRY(after_launch(dev, "embedding_sum_kernel"));
    if (chunks == 1) return AGPU_OK;
    AGPU_CUDA(launch_after(embedding_join_kernel<V>, chunks * join_slices, kThreads, 0, s, sorted,
                           starts, partial, d, own, (int)dv, (int)join_slices, chunk_len,
                           accumulate, scale));
    return after_launch(dev, "embedding_join_kernel");
  };
  const agpu_status st = run();
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
