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
// Both directions move each element once and are bound by memory bandwidth.
#include <algorithm>
#include <cmath>

#include "agpu_internal.cuh"

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
  int units[2];   // vector kernels: warp units per token
  int per_unit;   // heads per warp unit
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

// A warp unit is one token's next `per_unit` query or key heads; a warp walks
// units with the grid's stride and keeps its slot's frequencies.
__global__ void __launch_bounds__(kThreads) qk_forward_vec_kernel(const __grid_constant__ Args a,
                                                                  int lanes) {
  constexpr int J = 4;
  const int lane = threadIdx.x % 32, group = lane / lanes, groups = 32 / lanes;
  const Slot sl = slot_of(lane % lanes, a.dim, a.rot);
  const float inv_dim = 1.0f / (float)a.dim;
  double f[4];
  for (int i = 0; i < 4; ++i) f[i] = sl.turns ? inv_freq_of(sl.a + i, a.rot, a.log2_base) : 0.0;
  const int per_token = a.units[0] + a.units[1];
  const long long units = a.tokens * per_token;
  for (long long u = blockIdx.x * (long long)kWarps + threadIdx.x / 32; u < units;
       u += (long long)gridDim.x * kWarps) {
    const long long token = u / per_token;
    const int part = (int)(u - token * per_token);
    const int k = part >= a.units[0];
    const int h0 = (k ? part - a.units[0] : part) * a.per_unit;
    const int h1 = min(h0 + a.per_unit, a.heads[k]);
    const long long b = token / a.seq, s = token - b * a.seq;
    const float* x = a.x[k] + offset(a.in[k], b, s, 0);
    float* y = a.y[k] + offset(a.out[k], b, s, 0);
    float4 c, sn;
    turns_of(f, sl, position_of(a, token), c, sn);
    float4 wa = make_float4(1.f, 1.f, 1.f, 1.f), wb = wa;
    if (a.w[k] && sl.live) {
      wa = __ldg(reinterpret_cast<const float4*>(a.w[k] + sl.a));
      wb = __ldg(reinterpret_cast<const float4*>(a.w[k] + sl.b));
    }
    for (int hb = h0; hb < h1; hb += groups * J) {
      float4 xa[J], xb[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int h = hb + j * groups + group;
        xa[j] = xb[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (h < h1 && sl.live) {
          xa[j] = ldg4(x + h * a.in[k].head + sl.a);
          xb[j] = ldg4(x + h * a.in[k].head + sl.b);
        }
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int h = hb + j * groups + group;
        const float ss = group_sum(dot4(xa[j], xa[j]) + dot4(xb[j], xb[j]), lanes);
        const float r = 1.0f / sqrtf(ss * inv_dim + a.eps);
        const float4 ya = mul4(mul4(xa[j], r), wa), yb = mul4(mul4(xb[j], r), wb);
        if (h < h1 && sl.live) {
          st4(y + h * a.out[k].head + sl.a, fma4(neg4(yb), sn, mul4(ya, c)));
          st4(y + h * a.out[k].head + sl.b, fma4(ya, sn, mul4(yb, c)));
        }
      }
    }
  }
}

// The same units; each lane also sums its slot's weight gradients over all
// units of its warp, and the CTA's warps add theirs in warp order.
__global__ void __launch_bounds__(kThreads) qk_backward_vec_kernel(const __grid_constant__ Args a,
                                                                   int lanes) {
  constexpr int J = 2;
  __shared__ float4 red[kWarps][32][2];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int group = lane / lanes, groups = 32 / lanes;
  const Slot sl = slot_of(lane % lanes, a.dim, a.rot);
  const float inv_dim = 1.0f / (float)a.dim;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  double f[4];
  for (int i = 0; i < 4; ++i) f[i] = sl.turns ? inv_freq_of(sl.a + i, a.rot, a.log2_base) : 0.0;
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    float4 dwa = zero, dwb = zero;
    const long long units = a.tokens * a.units[k];
    for (long long u = blockIdx.x * (long long)kWarps + warp; u < units;
         u += (long long)gridDim.x * kWarps) {
      const long long token = u / a.units[k];
      const int h0 = (int)(u - token * a.units[k]) * a.per_unit;
      const int h1 = min(h0 + a.per_unit, a.heads[k]);
      const long long b = token / a.seq, s = token - b * a.seq;
      const float* x = a.x[k] + offset(a.in[k], b, s, 0);
      const float* g = a.g[k] + offset(a.out[k], b, s, 0);
      float* y = a.y[k] + offset(a.in[k], b, s, 0);
      float4 c, sn;
      turns_of(f, sl, position_of(a, token), c, sn);
      float4 wa = make_float4(1.f, 1.f, 1.f, 1.f), wb = wa;
      if (a.w[k] && sl.live) {
        wa = __ldg(reinterpret_cast<const float4*>(a.w[k] + sl.a));
        wb = __ldg(reinterpret_cast<const float4*>(a.w[k] + sl.b));
      }
      for (int hb = h0; hb < h1; hb += groups * J) {
        float4 xa[J], xb[J], ga[J], gb[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int h = hb + j * groups + group;
          xa[j] = xb[j] = ga[j] = gb[j] = zero;
          if (h < h1 && sl.live) {
            xa[j] = ldg4(x + h * a.in[k].head + sl.a);
            xb[j] = ldg4(x + h * a.in[k].head + sl.b);
            ga[j] = ldg4(g + h * a.out[k].head + sl.a);
            gb[j] = ldg4(g + h * a.out[k].head + sl.b);
          }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int h = hb + j * groups + group;
          const float4 ua = fma4(gb[j], sn, mul4(ga[j], c));        // rotated back
          const float4 ub = fma4(neg4(ga[j]), sn, mul4(gb[j], c));
          const float4 ha = mul4(ua, wa), hbv = mul4(ub, wb);
          float ss = dot4(xa[j], xa[j]) + dot4(xb[j], xb[j]);
          float hx = dot4(ha, xa[j]) + dot4(hbv, xb[j]);
          ss = group_sum(ss, lanes);
          hx = group_sum(hx, lanes);
          const float r = 1.0f / sqrtf(ss * inv_dim + a.eps);
          const float4 na = mul4(xa[j], r), nb = mul4(xb[j], r);
          const float m = -(hx * r) * inv_dim;  // -mean(h x r)
          const float4 mm = make_float4(m, m, m, m);
          if (h < h1 && sl.live) {
            st4(y + h * a.in[k].head + sl.a, mul4(fma4(na, mm, ha), r));
            st4(y + h * a.in[k].head + sl.b, mul4(fma4(nb, mm, hbv), r));
            dwa = fma4(ua, na, dwa);
            dwb = fma4(ub, nb, dwb);
          }
        }
      }
    }
    if (!a.partial) continue;
    __syncthreads();
    red[warp][lane][0] = dwa;
    red[warp][lane][1] = dwb;
    __syncthreads();
    if (threadIdx.x < lanes && sl.live) {  // lane == slot: sum groups and warps in order
      dwa = dwb = zero;
      for (int w = 0; w < kWarps; ++w)
        for (int gr = 0; gr < groups; ++gr) {
          const float4 pa = red[w][gr * lanes + lane][0], pb = red[w][gr * lanes + lane][1];
          dwa = make_float4(dwa.x + pa.x, dwa.y + pa.y, dwa.z + pa.z, dwa.w + pa.w);
          dwb = make_float4(dwb.x + pb.x, dwb.y + pb.y, dwb.z + pb.z, dwb.w + pb.w);
        }
      float* p = a.partial + ((long long)blockIdx.x * 2 + k) * a.dim;
      *reinterpret_cast<float4*>(p + sl.a) = dwa;
      *reinterpret_cast<float4*>(p + sl.b) = dwb;
    }
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
__global__ void __launch_bounds__(1024) qk_weight_grad_kernel(const float* __restrict__ partial,
                                                              int parts, int dim, float* dq,
                                                              float* dk) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int col = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (col < 2 * dim)
    for (int p = warp; p < parts; p += 32) v += partial[(long long)p * 2 * dim + col];
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

// Heads per warp unit: as many as leave every SM 32 warps, so that a unit's
// angles serve several heads.
void split_units(Args& a, int lanes, int sm_count) {
  const int groups = 32 / lanes;
  a.per_unit = groups * 8;
  for (;;) {
    for (int k = 0; k < 2; ++k) a.units[k] = (a.heads[k] + a.per_unit - 1) / a.per_unit;
    if (a.per_unit <= groups || a.tokens * (a.units[0] + a.units[1]) >= 32ll * sm_count) return;
    a.per_unit /= 2;
  }
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
    split_units(a, lanes, dev->sm_count);
    const long long want = (a.tokens * (a.units[0] + a.units[1]) + kWarps - 1) / kWarps;
    const unsigned grid = (unsigned)std::min<long long>(want, 6ll * dev->sm_count);
    qk_forward_vec_kernel<<<grid, kThreads, 0, s>>>(a, lanes);
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
  if (vec) {
    split_units(a, lanes, dev->sm_count);
    const long long most = a.tokens * std::max(a.units[0], a.units[1]);
    grid = (unsigned)std::min<long long>((most + kWarps - 1) / kWarps, 6ll * dev->sm_count);
  } else {
    grid = (unsigned)std::min<long long>(a.tokens, 4ll * dev->sm_count);
  }
  void* scratch = nullptr;
  if (d_q_weight || d_k_weight) {
    AGPU_TRY(pool_alloc(dev, (size_t)grid * 2 * a.dim * sizeof(float), &scratch, s));
    a.partial = static_cast<float*>(scratch);
  }
  if (vec) {
    qk_backward_vec_kernel<<<grid, kThreads, 0, s>>>(a, lanes);
  } else {
    const size_t smem = (a.rot + kWarps * 2 * a.dim) * sizeof(float);
    qk_any_kernel<true><<<grid, kThreads, smem, s>>>(a);
  }
  agpu_status st = after_launch(dev, "qk_norm_rope_backward");
  if (st == AGPU_OK && scratch) {
    qk_weight_grad_kernel<<<(2 * a.dim + 31) / 32, 1024, 0, s>>>(a.partial, (int)grid, a.dim,
                                                                 d_q_weight, d_k_weight);
    st = after_launch(dev, "qk_weight_grad_kernel");
  }
  pool_free(dev, scratch, s);
  return st;
}

}  // namespace agpu
