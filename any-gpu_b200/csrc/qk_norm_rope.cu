// RMS norm of every query and key head followed by the rotary embedding, in
// one pass, and its backward.  No counterpart in the reference crate; it is
// rmsnorm per head and rope (llama_ops.cu) without the store and reload
// between them.  For a head x of `dim` elements at position p, weight w:
//   r = 1 / sqrt(mean(x^2) + eps),  y_i = x_i r w_i,  then for i < rot/2
//   out_i         = y_i cos a_i - y_{i+rot/2} sin a_i
//   out_{i+rot/2} = y_{i+rot/2} cos a_i + y_i sin a_i,   a_i = p base^(-2i/rot)
// and out_i = y_i for i >= rot.  Backward, from g = d out:
//   g' = the rotation by -a of g,  h_i = g'_i w_i,
//   dx_i = r (h_i - x_i r^2 mean(h x)),  dw_i = sum over heads of g'_i x_i r.
//
// Both directions move each element once and are bound by memory bandwidth:
// 2 x 2048 tokens of 32 + 32 heads of 128 take 44 us (0.94 of the copy rate),
// the backward of 4 x 2048 tokens of 32 + 8 heads 87 (0.88); one token of 16
// sequences 6 us, the latency of a launch and of the angles.
#include <algorithm>
#include <cmath>

#include "agpu_internal.cuh"
#include "ptx.cuh"

namespace agpu {

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;

struct Strides {
  long long seq, head, batch;
};

// Operands indexed by 0 = queries, 1 = keys.
struct Args {
  const float* x[2];
  const float* g[2];  // backward: gradients of the outputs
  float* y[2];        // forward: outputs; backward: gradients of the inputs
  const float* w[2];  // weights or null (ones)
  Strides in[2], out[2];
  int heads[2];
  int batches[2];  // vector kernels: warp batches per token
  const int* positions;
  long long tokens;
  int seq, dim, rot;
  float eps;
  double log2_base;
  float* partial;  // backward: [CTA][2][dim] sums for the weights' gradients, or null
};

// cos and sin of p * inv_freq.  The product reaches p radians, so it and its
// reduction to [-pi, pi] are in double; what the float argument of sincosf
// loses is put back to first order.
__device__ __forceinline__ void turn(double inv_freq, int p, float& c, float& s) {
  const double a = (double)p * inv_freq;
  const double r = fma(-rint(a * 0.15915494309189535), 6.283185307179586, a);
  const float f = (float)r, lo = (float)(r - (double)f);
  float s0, c0;
  sincosf(f, &s0, &c0);
  c = c0 - s0 * lo;
  s = s0 + c0 * lo;
}

__device__ __forceinline__ double inv_freq_of(int i, int rot, double log2_base) {
  return exp2(-2.0 * (double)i / (double)rot * log2_base);
}

__device__ __forceinline__ int position_of(const Args& a, long long token) {
  return a.positions ? __ldg(a.positions + token) : (int)(token % a.seq);
}

__device__ __forceinline__ long long offset(const Strides& st, long long b, long long s, int h) {
  return b * st.batch + s * st.seq + h * st.head;
}

__device__ __forceinline__ float4 ldg4(const float* p) {
  return __ldcs(reinterpret_cast<const float4*>(p));
}
__device__ __forceinline__ void st4(float* p, float4 v) {
  __stcs(reinterpret_cast<float4*>(p), v);
}
__device__ __forceinline__ float dot4(float4 a, float4 b) {
  return (a.x * b.x + a.y * b.y) + (a.z * b.z + a.w * b.w);
}
__device__ __forceinline__ float4 mul4(float4 a, float4 b) {
  return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w);
}
__device__ __forceinline__ float4 mul4(float4 a, float b) {
  return make_float4(a.x * b, a.y * b, a.z * b, a.w * b);
}
// a + b * c
__device__ __forceinline__ float4 fma4(float4 b, float4 c, float4 a) {
  return make_float4(fmaf(b.x, c.x, a.x), fmaf(b.y, c.y, a.y), fmaf(b.z, c.z, a.z),
                     fmaf(b.w, c.w, a.w));
}
__device__ __forceinline__ float4 neg4(float4 a) { return make_float4(-a.x, -a.y, -a.z, -a.w); }

// Vector layout: a head is dim/8 slots of two float4, one slot per lane of a
// group of `lanes` (a power of two >= dim/8): slot j < rot/8 holds elements
// 4j.. and rot/2 + 4j.. (the pairs that rotate together), the others two
// neighbouring float4 behind the rotated part.
struct Slot {
  int a, b;   // element offsets of the two float4
  bool live, turns;
};

__device__ __forceinline__ Slot slot_of(int j, int dim, int rot) {
  Slot s;
  s.live = j < dim / 8;
  s.turns = j < rot / 8;
  s.a = s.turns ? 4 * j : rot + 8 * (j - rot / 8);
  s.b = s.turns ? rot / 2 + 4 * j : s.a + 4;
  if (!s.live) s.a = s.b = 0;
  return s;
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ void turns_of(const double (&f)[4], const Slot& sl, int p, float4& c,
                                         float4& s) {
  c = make_float4(1.f, 1.f, 1.f, 1.f);
  s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (sl.turns) {
    turn(f[0], p, c.x, s.x);
    turn(f[1], p, c.y, s.y);
    turn(f[2], p, c.z, s.z);
    turn(f[3], p, c.w, s.w);
  }
}

// Vector kernels: a batch is the next J * 32 / lanes query or key heads of a
// token, one head per group of lanes and j < J.  A warp takes a contiguous
// range of all batches (tokens in order, their queries first), so warps differ
// by one batch at most and neighbouring batches share their angles.  The
// operands of the next batch are on their way into shared memory (cp.async, 16
// bytes a lane, read by the lane that copied them: no barrier) while one is
// worked on: 8 KB in flight per warp without holding registers.  With the
// loads in registers the backward kernel needed 152 of them and reached 47% of
// the DRAM bandwidth.
constexpr int kPieces = 8;  // float4 per lane and batch
constexpr int kStages = 3;  // batches in shared memory: one worked on, the others on their way
constexpr int kCtas = 4;    // CTAs on an SM

struct Batch {
  long long token, b, s;
  int part;  // of the token: queries' batches, then keys'
  int k, h;  // queries or keys; this lane's first head
};

__device__ __forceinline__ void at_batch(const Args& a, Batch& t, long long i, int per_token) {
  t.token = i / per_token;
  t.part = (int)(i - t.token * per_token);
  t.b = t.token / a.seq;
  t.s = t.token - t.b * a.seq;
}

__device__ __forceinline__ void next_batch(const Args& a, Batch& t, int per_token) {
  if (++t.part < per_token) return;
  t.part = 0;
  ++t.token;
  if (++t.s == a.seq) {
    t.s = 0;
    ++t.b;
  }
}

__device__ __forceinline__ void copy16(float4* dst, const float* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src)
               : "memory");
}

// J heads per lane group and batch: 2 operands (x, and g backward) x 2 float4.
template <bool BACKWARD>
__global__ void __launch_bounds__(kThreads, kCtas) qk_vec_kernel(const __grid_constant__ Args a,
                                                             int lanes, int warps) {
  constexpr int J = BACKWARD ? 2 : 4;
  extern __shared__ float4 dyn[];  // [kStages][kPieces][kThreads]
  float4(*buf)[kPieces][kThreads] = reinterpret_cast<float4(*)[kPieces][kThreads]>(dyn);
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int group = lane / lanes, groups = 32 / lanes;
  const Slot sl = slot_of(lane % lanes, a.dim, a.rot);
  const float inv_dim = 1.0f / (float)a.dim;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f), one = make_float4(1.f, 1.f, 1.f, 1.f);
  const int per_token = a.batches[0] + a.batches[1];
  const long long all = a.tokens * per_token, w = blockIdx.x * (long long)kWarps + warp;
  long long i = w < warps ? w * all / warps : 0;
  const long long end = w < warps ? (w + 1) * all / warps : 0;

  // this lane's heads of a batch, and its copies into a stage
  auto heads_of = [&](Batch& t) {
    t.k = t.part >= a.batches[0];
    t.h = (t.k ? t.part - a.batches[0] : t.part) * groups * J + group;
  };
  auto fetch = [&](Batch& t, int stage) {
    heads_of(t);
    const float* x = a.x[t.k] + offset(a.in[t.k], t.b, t.s, t.h);
    const float* g = BACKWARD ? a.g[t.k] + offset(a.out[t.k], t.b, t.s, t.h) : nullptr;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (t.h + j * groups < a.heads[t.k] && sl.live) {
        copy16(&buf[stage][2 * j][tid], x + sl.a);
        copy16(&buf[stage][2 * j + 1][tid], x + sl.b);
        if (BACKWARD) {
          copy16(&buf[stage][2 * J + 2 * j][tid], g + sl.a);
          copy16(&buf[stage][2 * J + 2 * j + 1][tid], g + sl.b);
        }
      }
      x += groups * a.in[t.k].head;
      if (BACKWARD) g += groups * a.out[t.k].head;
    }
  };

  Batch cur = {}, ahead;
  if (i < end) at_batch(a, cur, i, per_token);
  ahead = cur;
#pragma unroll
  for (int p = 0; p < kStages - 1; ++p) {
    if (i + p < end) {
      fetch(ahead, p);
      next_batch(a, ahead, per_token);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  double f[4];
  for (int e = 0; e < 4; ++e) f[e] = sl.turns ? inv_freq_of(sl.a + e, a.rot, a.log2_base) : 0.0;
  float4 dw[2][2] = {{zero, zero}, {zero, zero}};  // weights' gradients: queries, keys
  float4 c, sn;           // cos and sin of a token
  long long turned = -1;  // which
  // forward: the weights' products with cos and sin, of queries or keys
  float4 ac, as, bc, bs;
  int folded = -1;
  for (int stage = 0; i < end; ++i) {
    if (i + kStages - 1 < end) {
      fetch(ahead, stage == 0 ? kStages - 1 : stage - 1);
      next_batch(a, ahead, per_token);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    heads_of(cur);
    if (turned != cur.token) {
      turned = cur.token;
      turns_of(f, sl, position_of(a, cur.token), c, sn);
      folded = -1;
    }
    const int k = cur.k;
    float4 wa = one, wb = one;
    if ((BACKWARD || folded != k) && a.w[k] && sl.live) {
      wa = __ldg(reinterpret_cast<const float4*>(a.w[k] + sl.a));
      wb = __ldg(reinterpret_cast<const float4*>(a.w[k] + sl.b));
    }
    if (!BACKWARD && folded != k) {
      folded = k;
      ac = mul4(wa, c);
      as = mul4(wa, sn);
      bc = mul4(wb, c);
      bs = neg4(mul4(wb, sn));
    }
    const Strides& to = BACKWARD ? a.in[k] : a.out[k];
    float* y = a.y[k] + offset(to, cur.b, cur.s, cur.h);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
#pragma unroll
    for (int j = 0; j < J; ++j, y += groups * to.head) {
      const bool in = cur.h + j * groups < a.heads[k] && sl.live;
      const float4 xa = in ? buf[stage][2 * j][tid] : zero;
      const float4 xb = in ? buf[stage][2 * j + 1][tid] : zero;
      float ss = dot4(xa, xa) + dot4(xb, xb);
      if (!BACKWARD) {
        const float r = rsqrtf(group_sum(ss, lanes) * inv_dim + a.eps);
        if (in) {
          st4(y + sl.a, mul4(fma4(xb, bs, mul4(xa, ac)), r));
          st4(y + sl.b, mul4(fma4(xa, as, mul4(xb, bc)), r));
        }
      } else {
        const float4 ga = in ? buf[stage][2 * J + 2 * j][tid] : zero;
        const float4 gb = in ? buf[stage][2 * J + 2 * j + 1][tid] : zero;
        const float4 ua = fma4(gb, sn, mul4(ga, c));  // rotated back
        const float4 ub = fma4(neg4(ga), sn, mul4(gb, c));
        const float4 ha = mul4(ua, wa), hb = mul4(ub, wb);
        float hx = dot4(ha, xa) + dot4(hb, xb);
        ss = group_sum(ss, lanes);
        hx = group_sum(hx, lanes);
        const float r = rsqrtf(ss * inv_dim + a.eps);
        const float4 na = mul4(xa, r), nb = mul4(xb, r);
        const float m = -(hx * r) * inv_dim;  // -mean(h x r)
        const float4 mm = make_float4(m, m, m, m);
        if (in) {
          st4(y + sl.a, mul4(fma4(na, mm, ha), r));
          st4(y + sl.b, mul4(fma4(nb, mm, hb), r));
          if (k) {
            dw[1][0] = fma4(ua, na, dw[1][0]);
            dw[1][1] = fma4(ub, nb, dw[1][1]);
          } else {
            dw[0][0] = fma4(ua, na, dw[0][0]);
            dw[0][1] = fma4(ub, nb, dw[0][1]);
          }
        }
      }
    }
    next_batch(a, cur, per_token);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (!BACKWARD || !a.partial) return;
  ptx::griddep_launch_dependents();  // qk_weight_grad_kernel, which waits for all of this one
  // the CTA's sums: groups and warps in order
  float4(*red)[32][4] = reinterpret_cast<float4(*)[32][4]>(dyn);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int h = 0; h < 2; ++h) red[warp][lane][2 * k + h] = dw[k][h];
  __syncthreads();
  if (warp < 2 && lane < lanes && sl.live) {  // warp = queries or keys, lane = slot
    float4 pa = zero, pb = zero;
    for (int v = 0; v < kWarps; ++v)
      for (int gr = 0; gr < groups; ++gr) {
        pa = fma4(one, red[v][gr * lanes + lane][2 * warp], pa);
        pb = fma4(one, red[v][gr * lanes + lane][2 * warp + 1], pb);
      }
    float* p = a.partial + (blockIdx.x * 2ll + warp) * a.dim;
    *reinterpret_cast<float4*>(p + sl.a) = pa;
    *reinterpret_cast<float4*>(p + sl.b) = pb;
  }
}

// Any head dim, stride and alignment: a CTA per token (grid stride), its
// cos / sin table in shared memory, a warp per head.  Element i belongs to
// lane i % 32 (i < rot/2: the pair i, i + rot/2).
template <bool BACKWARD>
__global__ void __launch_bounds__(kThreads) qk_any_kernel(const __grid_constant__ Args a) {
  extern __shared__ float sm[];  // cos, sin [rot/2 each]; backward: [kWarps][2][dim] weight sums
  const int half = a.rot / 2, dim = a.dim;
  float *cs = sm, *sn = sm + half;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float* acc = sm + a.rot + warp * 2 * dim;
  if (BACKWARD)
    for (int i = lane; i < 2 * dim; i += 32) acc[i] = 0.f;
  for (long long token = blockIdx.x; token < a.tokens; token += gridDim.x) {
    const int p = position_of(a, token);
    __syncthreads();
    for (int i = threadIdx.x; i < half; i += kThreads)
      turn(inv_freq_of(i, a.rot, a.log2_base), p, cs[i], sn[i]);
    __syncthreads();
    const long long b = token / a.seq, s = token - b * a.seq;
    for (int hh = warp; hh < a.heads[0] + a.heads[1]; hh += kWarps) {
      const int k = hh >= a.heads[0], h = k ? hh - a.heads[0] : hh;
      const float* x = a.x[k] + offset(a.in[k], b, s, h);
      const float* w = a.w[k];
      const float* g = BACKWARD ? a.g[k] + offset(a.out[k], b, s, h) : nullptr;
      float* y = a.y[k] + offset(BACKWARD ? a.in[k] : a.out[k], b, s, h);
      float ss = 0.f, hx = 0.f;
      for (int i = lane; i < dim; i += 32) ss += x[i] * x[i];
      if (BACKWARD) {
        for (int i = lane; i < half; i += 32) {
          const float ua = g[i] * cs[i] + g[i + half] * sn[i];
          const float ub = g[i + half] * cs[i] - g[i] * sn[i];
          hx += (w ? ua * w[i] : ua) * x[i] + (w ? ub * w[i + half] : ub) * x[i + half];
        }
        for (int i = a.rot + lane; i < dim; i += 32) hx += (w ? g[i] * w[i] : g[i]) * x[i];
        hx = group_sum(hx, 32);
      }
      ss = group_sum(ss, 32);
      const float r = 1.0f / sqrtf(ss / (float)dim + a.eps);
      const float m = hx * r / (float)dim;
      // one element: the normalised input and the gradient (rotated back)
      auto back = [&](int i, float u) {
        const float n = x[i] * r;
        y[i] = r * ((w ? u * w[i] : u) - n * m);
        acc[k * dim + i] += u * n;
      };
      for (int i = lane; i < half; i += 32) {
        if (BACKWARD) {
          const float ga = g[i], gb = g[i + half];
          back(i, ga * cs[i] + gb * sn[i]);
          back(i + half, gb * cs[i] - ga * sn[i]);
        } else {
          const float ya = x[i] * r * (w ? w[i] : 1.f);
          const float yb = x[i + half] * r * (w ? w[i + half] : 1.f);
          y[i] = ya * cs[i] - yb * sn[i];
          y[i + half] = yb * cs[i] + ya * sn[i];
        }
      }
      for (int i = a.rot + lane; i < dim; i += 32) {
        if (BACKWARD) back(i, g[i]);
        else y[i] = x[i] * r * (w ? w[i] : 1.f);
      }
    }
  }
  if (BACKWARD && a.partial) {
    ptx::griddep_launch_dependents();  // qk_weight_grad_kernel, which waits for all of this one
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * dim; i += kThreads) {
      float v = 0.f;
      for (int w = 0; w < kWarps; ++w) v += sm[a.rot + w * 2 * dim + i];
      a.partial[(long long)blockIdx.x * 2 * dim + i] = v;
    }
  }
}

// d_weight[k][i] = sum over the CTAs' partial sums, in a fixed order: lane =
// column, each of 32 warps sums every 32nd part, warp 0 adds the warps.
// Latency: 592 parts of 2 x 128 take 7 us, its launch overlaps the pass before.
__global__ void __launch_bounds__(1024) qk_weight_grad_kernel(const float* __restrict__ partial,
                                                              int parts, int dim, float* dq,
                                                              float* dk) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int col = blockIdx.x * 32 + lane;
  float v = 0.f;
  ptx::griddep_wait();
  if (col < 2 * dim) {
#pragma unroll 8
    for (int p = warp; p < parts; p += 32) v += partial[(long long)p * 2 * dim + col];
  }
  red[warp][lane] = v;
  __syncthreads();
  if (warp != 0 || col >= 2 * dim) return;
  v = 0.f;
  for (int w = 0; w < 32; ++w) v += red[w][lane];
  float* d = col < dim ? dq : dk;
  if (d) d[col < dim ? col : col - dim] = v;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

Strides strides_of(const agpu_attn_layout& l) {
  return {(long long)l.seq_stride, (long long)l.head_stride, (long long)l.batch_stride};
}

Args make_args(const agpu_qk_norm_rope& d, const float* q, const float* k, const float* qw,
               const float* kw, const int32_t* positions) {
  Args a = {};
  a.x[0] = q;
  a.x[1] = k;
  a.w[0] = qw;
  a.w[1] = kw;
  a.in[0] = strides_of(d.q_in);
  a.in[1] = strides_of(d.k_in);
  a.out[0] = strides_of(d.q_out);
  a.out[1] = strides_of(d.k_out);
  a.heads[0] = (int)d.q_heads;
  a.heads[1] = (int)d.k_heads;
  a.positions = positions;
  a.tokens = (long long)d.batch * d.seq;
  a.seq = (int)d.seq;
  a.dim = (int)d.dim;
  a.rot = (int)d.rot_dim;
  a.eps = d.eps;
  a.log2_base = std::log2((double)d.base);
  return a;
}

bool vector_ok(const Args& a) {
  if (a.dim % 8 || a.rot % 8 || a.dim > 256) return false;
  for (int k = 0; k < 2; ++k) {
    if (!a.heads[k]) continue;
    for (const Strides* s : {&a.in[k], &a.out[k]})
      if (s->seq % 4 || s->head % 4 || s->batch % 4) return false;
    if (!aligned16(a.x[k]) || !aligned16(a.g[k]) || !aligned16(a.y[k]) || !aligned16(a.w[k]))
      return false;
  }
  return true;
}

int lanes_for(int dim) {
  int lanes = 1;
  while (lanes < dim / 8) lanes *= 2;
  return lanes;
}

constexpr int kVecSmem = kStages * kPieces * kThreads * sizeof(float4);

// Batches per token, and the warps that share all of them.
int split_batches(Args& a, int lanes, int j, int sm_count) {
  const int heads = 32 / lanes * j;
  for (int k = 0; k < 2; ++k) a.batches[k] = (a.heads[k] + heads - 1) / heads;
  return (int)std::min<long long>(a.tokens * (a.batches[0] + a.batches[1]),
                                  (long long)kCtas * kWarps * sm_count);
}

agpu_status sum_weight_grads(agpu_device* dev, const Args& a, int parts, float* dq, float* dk,
                             cudaStream_t s) {
  AGPU_CUDA(launch_after(qk_weight_grad_kernel, (2 * a.dim + 31) / 32, 1024, 0, s, a.partial, parts,
                         a.dim, dq, dk));
  return after_launch(dev, "qk_weight_grad_kernel");
}

}  // namespace

agpu_status launch_qk_norm_rope(agpu_device* dev, const agpu_qk_norm_rope& d, const float* q,
                                const float* k, const float* q_weight, const float* k_weight,
                                const int32_t* positions, float* q_out, float* k_out,
                                cudaStream_t s) {
  Args a = make_args(d, q, k, q_weight, k_weight, positions);
  a.y[0] = q_out;
  a.y[1] = k_out;
  if (a.tokens == 0 || a.heads[0] + a.heads[1] == 0) return AGPU_OK;
  if (vector_ok(a)) {
    const int lanes = lanes_for(a.dim);
    const int warps = split_batches(a, lanes, 4, dev->sm_count);
    AGPU_CUDA(set_smem_once<qk_vec_kernel<false>>(dev, kVecSmem));
    qk_vec_kernel<false><<<(warps + kWarps - 1) / kWarps, kThreads, kVecSmem, s>>>(a, lanes, warps);
  } else {
    const unsigned grid = (unsigned)std::min<long long>(a.tokens, 16ll * dev->sm_count);
    qk_any_kernel<false><<<grid, kThreads, a.rot * sizeof(float), s>>>(a);
  }
  return after_launch(dev, "qk_norm_rope");
}

agpu_status launch_qk_norm_rope_backward(agpu_device* dev, const agpu_qk_norm_rope& d,
                                         const float* d_q_out, const float* d_k_out,
                                         const float* q, const float* k, const float* q_weight,
                                         const float* k_weight, const int32_t* positions,
                                         float* d_q, float* d_k, float* d_q_weight,
                                         float* d_k_weight, cudaStream_t s) {
  Args a = make_args(d, q, k, q_weight, k_weight, positions);
  a.g[0] = d_q_out;
  a.g[1] = d_k_out;
  a.y[0] = d_q;
  a.y[1] = d_k;
  if (a.tokens == 0 || a.heads[0] + a.heads[1] == 0) {
    for (float* w : {d_q_weight, d_k_weight})
      if (w) AGPU_CUDA(cudaMemsetAsync(w, 0, d.dim * sizeof(float), s));
    return AGPU_OK;
  }
  const bool vec = vector_ok(a);
  const int lanes = lanes_for(a.dim);
  unsigned grid;
  int warps = 0;
  if (vec) {
    warps = split_batches(a, lanes, 2, dev->sm_count);
    grid = (warps + kWarps - 1) / kWarps;
  } else {
    grid = (unsigned)std::min<long long>(a.tokens, 4ll * dev->sm_count);
  }
  if (vec) AGPU_CUDA(set_smem_once<qk_vec_kernel<true>>(dev, kVecSmem));
  void* scratch = nullptr;
  if (d_q_weight || d_k_weight) {
    AGPU_TRY(pool_alloc(dev, (size_t)grid * 2 * a.dim * sizeof(float), &scratch, s));
    a.partial = static_cast<float*>(scratch);
  }
  if (vec) {
    qk_vec_kernel<true><<<grid, kThreads, kVecSmem, s>>>(a, lanes, warps);
  } else {
    const size_t smem = (a.rot + kWarps * 2 * a.dim) * sizeof(float);
    qk_any_kernel<true><<<grid, kThreads, smem, s>>>(a);
  }
  agpu_status st = after_launch(dev, "qk_norm_rope_backward");
  if (st == AGPU_OK && scratch) {
    st = sum_weight_grads(dev, a, (int)grid, d_q_weight, d_k_weight, s);
  }
  pool_free(dev, scratch, s);
  return st;
}

}  // namespace agpu
