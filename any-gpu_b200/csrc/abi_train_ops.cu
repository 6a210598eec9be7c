// C-ABI entry points of the ops for training on tokens: embedding, head norms
// with the rotary embedding, orthogonalised updates.  Arguments are checked
// before the device is touched, so a refused call has no effect.
#include <algorithm>
#include <cmath>
#include <exception>
#include <iterator>
#include <utility>
#include <vector>

#include "agpu_internal.cuh"

using namespace agpu;

namespace {

agpu_status use_device(agpu_device* dev, const char* fn) {
  if (!dev) return fail(AGPU_ERR_INVALID, "%s: NULL device", fn);
  if (cudaSetDevice(dev->ordinal) != cudaSuccess)
    return fail(AGPU_ERR_CUDA, "%s: cannot select device %d", fn, dev->ordinal);
  return AGPU_OK;
}

agpu_status check_len(const agpu_buffer* b, uint64_t want, const char* fn, const char* name,
                      bool i32 = false) {
  if (!b) return fail(AGPU_ERR_INVALID, "%s: %s is NULL", fn, name);
  if (b->i32 != i32)
    return fail(AGPU_ERR_INVALID, "%s: %s must be an %s buffer", fn, name,
                i32 ? "int32 (agpu_upload_i32)" : "f32");
  if (b->len != want)
    return fail(AGPU_ERR_SHAPE, "%s: %s has %llu elems, expected %llu", fn, name,
                (unsigned long long)b->len, (unsigned long long)want);
  return AGPU_OK;
}

agpu_status check_embedding(uint64_t tokens, uint32_t vocab, uint32_t dim, const char* fn) {
  if (tokens && vocab == 0) return fail(AGPU_ERR_INVALID, "%s: vocab is 0", fn);
  if (tokens > 0x7fffffffull) return fail(AGPU_ERR_UNSUPPORTED, "%s: too many tokens", fn);
  if (vocab > 0x3fffffffu || dim > 0x3fffffffu)
    return fail(AGPU_ERR_UNSUPPORTED, "%s: table too large", fn);
  return AGPU_OK;
}

// The gradient's positions are 32-bit, and its sorting kernel steps up to 256
// of them past the last token.
agpu_status check_embedding_backward(uint64_t tokens, uint32_t vocab, uint32_t dim,
                                     const char* fn) {
  if (tokens > 0x7fffff00ull) return fail(AGPU_ERR_UNSUPPORTED, "%s: too many tokens", fn);
  return check_embedding(tokens, vocab, dim, fn);
}

// Whether no two elements of [batch, seq, heads, dim] share an address: by
// increasing stride, each axis steps past everything the smaller ones cover.
bool distinct(const agpu_attn_layout& l, uint32_t batch, uint32_t seq, uint32_t heads,
              uint32_t dim) {
  struct Axis { uint64_t stride, count; } ax[3] = {
      {l.seq_stride, seq}, {l.head_stride, heads}, {l.batch_stride, batch}};
  uint64_t covered = dim;
  bool used[3] = {};
  for (int k = 0; k < 3; ++k) {
    int best = -1;
    for (int i = 0; i < 3; ++i)
      if (!used[i] && (best < 0 || ax[i].count <= 1 || (ax[best].count > 1 &&
                                                        ax[i].stride < ax[best].stride)))
        best = i;
    used[best] = true;
    if (ax[best].count <= 1) continue;
    if (ax[best].stride < covered || ax[best].stride > (1ull << 40)) return false;
    covered += (ax[best].count - 1) * ax[best].stride;
  }
  return true;
}

agpu_status check_qk(const agpu_qk_norm_rope& d, const char* fn) {
  if (d.dim == 0 || d.dim > 1024)
    return fail(AGPU_ERR_UNSUPPORTED, "%s: head dim %u outside [1, 1024]", fn, d.dim);
  if (d.rot_dim % 2 || d.rot_dim > d.dim)
    return fail(AGPU_ERR_SHAPE, "%s: rot_dim %u is odd or above the head dim %u", fn, d.rot_dim,
                d.dim);
  if (!(d.base > 0.f) || !std::isfinite(d.base))
    return fail(AGPU_ERR_INVALID, "%s: base must be positive", fn);
  if (!(d.eps >= 0.f) || !std::isfinite(d.eps))
    return fail(AGPU_ERR_INVALID, "%s: eps must not be negative", fn);
  if ((uint64_t)d.batch * d.seq > 0x7fffffffull || d.q_heads > 65535 || d.k_heads > 65535)
    return fail(AGPU_ERR_UNSUPPORTED, "%s: too many tokens or heads", fn);
  if ((d.q_heads && (!distinct(d.q_in, d.batch, d.seq, d.q_heads, d.dim) ||
                     !distinct(d.q_out, d.batch, d.seq, d.q_heads, d.dim))) ||
      (d.k_heads && (!distinct(d.k_in, d.batch, d.seq, d.k_heads, d.dim) ||
                     !distinct(d.k_out, d.batch, d.seq, d.k_heads, d.dim))))
    return fail(AGPU_ERR_SHAPE, "%s: a layout's strides make elements overlap", fn);
  return AGPU_OK;
}

// The buffer layer's geometry: contiguous [batch, seq, heads, dim] in, the
// same or [batch, heads, seq, dim] out.
agpu_qk_norm_rope contiguous(uint32_t batch, uint32_t seq, uint32_t q_heads, uint32_t k_heads,
                             uint32_t dim, uint32_t rot_dim, float eps, float base,
                             bool head_major) {
  const uint64_t n = seq, d = dim;
  auto in = [&](uint64_t h) { return agpu_attn_layout{h * d, d, n * h * d}; };
  auto out = [&](uint64_t h) {
    return head_major ? agpu_attn_layout{d, n * d, h * n * d} : in(h);
  };
  return {batch, seq, q_heads, k_heads, dim, rot_dim, eps, base,
          in(q_heads), in(k_heads), out(q_heads), out(k_heads)};
}

uint64_t elems(const agpu_qk_norm_rope& d, uint32_t heads) {
  return (uint64_t)d.batch * d.seq * heads * d.dim;
}

// A buffer that is freed unless released.
struct Owned {
  agpu_buffer* b = nullptr;
  ~Owned() { agpu_buffer_free(b); }
  float* ptr() const { return b ? b->dptr : nullptr; }
  void give(agpu_buffer** out) {
    if (out) *out = b;
    b = nullptr;
  }
};

agpu_status check_steps(uint32_t steps, const char* fn) {
  if (steps == 0 || steps > 64)
    return fail(AGPU_ERR_INVALID, "%s: steps %u outside [1, 64]", fn, steps);
  return AGPU_OK;
}

agpu_status check_muon(float lr, float momentum, float weight_decay, uint32_t steps,
                       const char* fn) {
  if (!std::isfinite(lr) || !std::isfinite(weight_decay))
    return fail(AGPU_ERR_INVALID, "%s: lr and weight_decay must be finite", fn);
  if (!(momentum >= 0.f && momentum < 1.f))
    return fail(AGPU_ERR_INVALID, "%s: momentum outside [0, 1)", fn);
  return check_steps(steps, fn);
}

// Written tensors (parameters and momenta) may share memory neither with each
// other nor with a gradient: the matrices of a step are updated side by side.
// Also checks each for NULL.
agpu_status check_muon_tensors(const agpu_muon_tensor* t, uint32_t count, const char* fn) try {
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  spans.reserve(2 * (size_t)count);
  for (uint32_t i = 0; i < count; ++i) {
    const uint64_t n = (uint64_t)t[i].rows * t[i].cols;
    if (n == 0) continue;
    if (!t[i].param || !t[i].grad || !t[i].momentum)
      return fail(AGPU_ERR_INVALID, "%s: tensor %u has a NULL pointer", fn, i);
    for (const float* p : {t[i].param, t[i].momentum}) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(p);
      spans.emplace_back(a, a + n * sizeof(float));
    }
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second)
      return fail(AGPU_ERR_INVALID, "%s: two parameters or momenta share memory", fn);
  for (uint32_t i = 0; i < count; ++i) {
    const uint64_t n = (uint64_t)t[i].rows * t[i].cols;
    if (n == 0) continue;
    const uintptr_t a = reinterpret_cast<uintptr_t>(t[i].grad), b = a + n * sizeof(float);
    // the last span that begins before the gradient's end
    auto it = std::lower_bound(spans.begin(), spans.end(), std::make_pair(b, (uintptr_t)0));
    if (it != spans.begin() && std::prev(it)->second > a)
      return fail(AGPU_ERR_INVALID, "%s: gradient %u shares memory with a parameter or momentum",
                  fn, i);
  }
  return AGPU_OK;
} catch (const std::exception&) {
  return fail(AGPU_ERR_OOM, "%s: out of host memory", fn);
}

// Elements stay below 2^40 (more than any device holds), so no product wraps.
agpu_status check_matrix(uint32_t rows, uint32_t cols, const char* fn, uint32_t batch = 1) {
  const uint64_t n = (uint64_t)rows * cols, most = 1ull << 40;
  if (rows > 0x7fffffffu || cols > 0x7fffffffu || n > most || (n && batch > most / n))
    return fail(AGPU_ERR_UNSUPPORTED, "%s: matrix too large", fn);
  return AGPU_OK;
}

}  // namespace

extern "C" {

// --------------------------------------------------------------- embedding --
agpu_status agpu_embedding(agpu_device* dev, const agpu_buffer* table, const agpu_buffer* ids,
                           uint64_t tokens, uint32_t vocab, uint32_t dim, float scale,
                           agpu_buffer** out) {
  if (!out) return fail(AGPU_ERR_INVALID, "embedding: out is NULL");
  *out = nullptr;
  AGPU_TRY(check_embedding(tokens, vocab, dim, "embedding"));
  AGPU_TRY(check_len(table, (uint64_t)vocab * dim, "embedding", "table"));
  AGPU_TRY(check_len(ids, tokens, "embedding", "ids", true));
  AGPU_TRY(use_device(dev, "embedding"));
  Owned o;
  AGPU_TRY(new_buffer(dev, tokens * dim, &o.b));
  AGPU_TRY(launch_embedding(dev, table->dptr, reinterpret_cast<const int32_t*>(ids->dptr),
                            o.ptr(), tokens, vocab, dim, scale, dev->stream));
  o.give(out);
  return AGPU_OK;
}

agpu_status agpu_embedding_backward(agpu_device* dev, const agpu_buffer* grad_out,
                                    const agpu_buffer* ids, uint64_t tokens, uint32_t vocab,
                                    uint32_t dim, float scale, agpu_buffer** d_table) {
  if (!d_table) return fail(AGPU_ERR_INVALID, "embedding_backward: d_table is NULL");
  *d_table = nullptr;
  AGPU_TRY(check_embedding_backward(tokens, vocab, dim, "embedding_backward"));
  AGPU_TRY(check_len(grad_out, tokens * dim, "embedding_backward", "grad_out"));
  AGPU_TRY(check_len(ids, tokens, "embedding_backward", "ids", true));
  AGPU_TRY(use_device(dev, "embedding_backward"));
  Owned o;
  AGPU_TRY(new_buffer(dev, (uint64_t)vocab * dim, &o.b));
  AGPU_TRY(launch_embedding_backward(dev, grad_out->dptr,
                                     reinterpret_cast<const int32_t*>(ids->dptr), o.ptr(), tokens,
                                     vocab, dim, scale, false, dev->stream));
  o.give(d_table);
  return AGPU_OK;
}

agpu_status agpu_launch_embedding(agpu_device* dev, const float* table, const int32_t* ids,
                                  float* out, uint64_t tokens, uint32_t vocab, uint32_t dim,
                                  float scale, void* stream) {
  AGPU_TRY(check_embedding(tokens, vocab, dim, "launch_embedding"));
  if ((!table || !ids || !out) && tokens * dim)
    return fail(AGPU_ERR_INVALID, "launch_embedding: NULL pointer");
  AGPU_TRY(use_device(dev, "launch_embedding"));
  return launch_embedding(dev, table, ids, out, tokens, vocab, dim, scale,
                          pick_stream(dev, stream));
}

agpu_status agpu_launch_embedding_backward(agpu_device* dev, const float* grad_out,
                                           const int32_t* ids, float* d_table, uint64_t tokens,
                                           uint32_t vocab, uint32_t dim, float scale,
                                           int accumulate, void* stream) {
  AGPU_TRY(check_embedding_backward(tokens, vocab, dim, "launch_embedding_backward"));
  if (((!grad_out || !ids) && tokens * dim) || (!d_table && (uint64_t)vocab * dim))
    return fail(AGPU_ERR_INVALID, "launch_embedding_backward: NULL pointer");
  AGPU_TRY(use_device(dev, "launch_embedding_backward"));
  return launch_embedding_backward(dev, grad_out, ids, d_table, tokens, vocab, dim, scale,
                                   accumulate != 0, pick_stream(dev, stream));
}

// ------------------------------------------------------- head norms + rope --
agpu_status agpu_qk_norm_rope_forward(agpu_device* dev, const agpu_buffer* q, const agpu_buffer* k,
                                      const agpu_buffer* q_weight, const agpu_buffer* k_weight,
                                      const agpu_buffer* positions, uint32_t batch, uint32_t seq,
                                      uint32_t q_heads, uint32_t k_heads, uint32_t dim,
                                      uint32_t rot_dim, float eps, float base, int head_major,
                                      agpu_buffer** q_out, agpu_buffer** k_out) {
  const char* fn = "qk_norm_rope";
  if ((!q_out && q_heads) || (!k_out && k_heads))
    return fail(AGPU_ERR_INVALID, "%s: an output is NULL", fn);
  if (q_out) *q_out = nullptr;
  if (k_out) *k_out = nullptr;
  const agpu_qk_norm_rope d =
      contiguous(batch, seq, q_heads, k_heads, dim, rot_dim, eps, base, head_major != 0);
  AGPU_TRY(check_qk(d, fn));
  if (q_heads) AGPU_TRY(check_len(q, elems(d, q_heads), fn, "q"));
  if (k_heads) AGPU_TRY(check_len(k, elems(d, k_heads), fn, "k"));
  if (q_weight) AGPU_TRY(check_len(q_weight, dim, fn, "q_weight"));
  if (k_weight) AGPU_TRY(check_len(k_weight, dim, fn, "k_weight"));
  if (positions) AGPU_TRY(check_len(positions, (uint64_t)batch * seq, fn, "positions", true));
  AGPU_TRY(use_device(dev, fn));
  Owned qo, ko;
  if (q_heads) AGPU_TRY(new_buffer(dev, elems(d, q_heads), &qo.b));
  if (k_heads) AGPU_TRY(new_buffer(dev, elems(d, k_heads), &ko.b));
  auto ptr = [](const agpu_buffer* b) { return b ? b->dptr : nullptr; };
  AGPU_TRY(launch_qk_norm_rope(dev, d, q_heads ? q->dptr : nullptr, k_heads ? k->dptr : nullptr,
                               ptr(q_weight), ptr(k_weight),
                               reinterpret_cast<const int32_t*>(ptr(positions)), qo.ptr(),
                               ko.ptr(), dev->stream));
  qo.give(q_out);
  ko.give(k_out);
  return AGPU_OK;
}

agpu_status agpu_qk_norm_rope_backward(
    agpu_device* dev, const agpu_buffer* d_q_out, const agpu_buffer* d_k_out,
    const agpu_buffer* q, const agpu_buffer* k, const agpu_buffer* q_weight,
    const agpu_buffer* k_weight, const agpu_buffer* positions, uint32_t batch, uint32_t seq,
    uint32_t q_heads, uint32_t k_heads, uint32_t dim, uint32_t rot_dim, float eps, float base,
    int head_major, agpu_buffer** d_q, agpu_buffer** d_k, agpu_buffer** d_q_weight,
    agpu_buffer** d_k_weight) {
  const char* fn = "qk_norm_rope_backward";
  if ((!d_q && q_heads) || (!d_k && k_heads))
    return fail(AGPU_ERR_INVALID, "%s: an output is NULL", fn);
  for (agpu_buffer** o : {d_q, d_k, d_q_weight, d_k_weight})
    if (o) *o = nullptr;
  const agpu_qk_norm_rope d =
      contiguous(batch, seq, q_heads, k_heads, dim, rot_dim, eps, base, head_major != 0);
  AGPU_TRY(check_qk(d, fn));
  if (q_heads) {
    AGPU_TRY(check_len(d_q_out, elems(d, q_heads), fn, "d_q_out"));
    AGPU_TRY(check_len(q, elems(d, q_heads), fn, "q"));
  }
  if (k_heads) {
    AGPU_TRY(check_len(d_k_out, elems(d, k_heads), fn, "d_k_out"));
    AGPU_TRY(check_len(k, elems(d, k_heads), fn, "k"));
  }
  if (q_weight) AGPU_TRY(check_len(q_weight, dim, fn, "q_weight"));
  if (k_weight) AGPU_TRY(check_len(k_weight, dim, fn, "k_weight"));
  if (positions) AGPU_TRY(check_len(positions, (uint64_t)batch * seq, fn, "positions", true));
  AGPU_TRY(use_device(dev, fn));
  Owned dq, dk, dqw, dkw;
  if (q_heads) AGPU_TRY(new_buffer(dev, elems(d, q_heads), &dq.b));
  if (k_heads) AGPU_TRY(new_buffer(dev, elems(d, k_heads), &dk.b));
  if (d_q_weight) AGPU_TRY(new_buffer(dev, dim, &dqw.b));
  if (d_k_weight) AGPU_TRY(new_buffer(dev, dim, &dkw.b));
  auto ptr = [](const agpu_buffer* b) { return b ? b->dptr : nullptr; };
  AGPU_TRY(launch_qk_norm_rope_backward(
      dev, d, q_heads ? d_q_out->dptr : nullptr, k_heads ? d_k_out->dptr : nullptr,
      q_heads ? q->dptr : nullptr, k_heads ? k->dptr : nullptr, ptr(q_weight), ptr(k_weight),
      reinterpret_cast<const int32_t*>(ptr(positions)), dq.ptr(), dk.ptr(), dqw.ptr(), dkw.ptr(),
      dev->stream));
  dq.give(d_q);
  dk.give(d_k);
  dqw.give(d_q_weight);
  dkw.give(d_k_weight);
  return AGPU_OK;
}

agpu_status agpu_launch_qk_norm_rope(agpu_device* dev, const agpu_qk_norm_rope* shape,
                                     const float* q, const float* k, const float* q_weight,
                                     const float* k_weight, const int32_t* positions,
                                     float* q_out, float* k_out, void* stream) {
  const char* fn = "launch_qk_norm_rope";
  if (!shape) return fail(AGPU_ERR_INVALID, "%s: NULL shape", fn);
  AGPU_TRY(check_qk(*shape, fn));
  const bool any = shape->batch && shape->seq;
  if (any && ((shape->q_heads && (!q || !q_out)) || (shape->k_heads && (!k || !k_out))))
    return fail(AGPU_ERR_INVALID, "%s: NULL pointer", fn);
  AGPU_TRY(use_device(dev, fn));
  return launch_qk_norm_rope(dev, *shape, q, k, q_weight, k_weight, positions, q_out, k_out,
                             pick_stream(dev, stream));
}

agpu_status agpu_launch_qk_norm_rope_backward(
    agpu_device* dev, const agpu_qk_norm_rope* shape, const float* d_q_out, const float* d_k_out,
    const float* q, const float* k, const float* q_weight, const float* k_weight,
    const int32_t* positions, float* d_q, float* d_k, float* d_q_weight, float* d_k_weight,
    void* stream) {
  const char* fn = "launch_qk_norm_rope_backward";
  if (!shape) return fail(AGPU_ERR_INVALID, "%s: NULL shape", fn);
  AGPU_TRY(check_qk(*shape, fn));
  const bool any = shape->batch && shape->seq;
  if (any && ((shape->q_heads && (!d_q_out || !q || !d_q)) ||
              (shape->k_heads && (!d_k_out || !k || !d_k))))
    return fail(AGPU_ERR_INVALID, "%s: NULL pointer", fn);
  AGPU_TRY(use_device(dev, fn));
  return launch_qk_norm_rope_backward(dev, *shape, d_q_out, d_k_out, q, k, q_weight, k_weight,
                                      positions, d_q, d_k, d_q_weight, d_k_weight,
                                      pick_stream(dev, stream));
}

// --------------------------------------------------- orthogonalised updates --
agpu_status agpu_orthogonalize(agpu_device* dev, const agpu_buffer* x, uint32_t batch,
                               uint32_t rows, uint32_t cols, uint32_t steps, agpu_buffer** out) {
  const char* fn = "orthogonalize";
  if (!out) return fail(AGPU_ERR_INVALID, "%s: out is NULL", fn);
  *out = nullptr;
  AGPU_TRY(check_steps(steps, fn));
  AGPU_TRY(check_matrix(rows, cols, fn, batch));
  AGPU_TRY(check_len(x, (uint64_t)batch * rows * cols, fn, "x"));
  AGPU_TRY(use_device(dev, fn));
  Owned o;
  AGPU_TRY(new_buffer(dev, x->len, &o.b));
  AGPU_TRY(launch_orthogonalize(dev, x->dptr, o.ptr(), batch, rows, cols, steps, dev->stream));
  o.give(out);
  return AGPU_OK;
}

agpu_status agpu_launch_orthogonalize(agpu_device* dev, const float* x, float* out, uint32_t batch,
                                      uint32_t rows, uint32_t cols, uint32_t steps,
                                      void* stream) {
  const char* fn = "launch_orthogonalize";
  AGPU_TRY(check_steps(steps, fn));
  AGPU_TRY(check_matrix(rows, cols, fn, batch));
  const uint64_t n = (uint64_t)batch * rows * cols;
  if ((!x || !out) && n) return fail(AGPU_ERR_INVALID, "%s: NULL pointer", fn);
  const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(out);
  if (a != b && (a < b ? b - a : a - b) < n * sizeof(float))
    return fail(AGPU_ERR_INVALID, "%s: out overlaps x", fn);
  AGPU_TRY(use_device(dev, fn));
  return launch_orthogonalize(dev, x, out, batch, rows, cols, steps, pick_stream(dev, stream));
}

agpu_status agpu_muon_step(agpu_device* dev, agpu_buffer* const* params,
                           const agpu_buffer* const* grads, agpu_buffer* const* momenta,
                           const uint32_t* rows, const uint32_t* cols, uint32_t count, float lr,
                           float momentum, int nesterov, float weight_decay,
                           uint32_t steps) try {
  const char* fn = "muon_step";
  AGPU_TRY(check_muon(lr, momentum, weight_decay, steps, fn));
  if (count && (!params || !grads || !momenta || !rows || !cols))
    return fail(AGPU_ERR_INVALID, "%s: NULL array", fn);
  std::vector<agpu_muon_tensor> t(count);
  for (uint32_t i = 0; i < count; ++i) {
    AGPU_TRY(check_matrix(rows[i], cols[i], fn));
    const uint64_t n = (uint64_t)rows[i] * cols[i];
    AGPU_TRY(check_len(params[i], n, fn, "a parameter"));
    AGPU_TRY(check_len(grads[i], n, fn, "a gradient"));
    AGPU_TRY(check_len(momenta[i], n, fn, "a momentum"));
    t[i] = {params[i]->dptr, grads[i]->dptr, momenta[i]->dptr, rows[i], cols[i]};
  }
  AGPU_TRY(check_muon_tensors(t.data(), count, fn));
  AGPU_TRY(use_device(dev, fn));
  return launch_muon(dev, t.data(), count, lr, momentum, nesterov != 0, weight_decay, steps,
                     dev->stream);
} catch (const std::exception&) {
  return fail(AGPU_ERR_OOM, "muon_step: out of host memory");
}

agpu_status agpu_launch_muon(agpu_device* dev, const agpu_muon_tensor* tensors, uint32_t count,
                             float lr, float momentum, int nesterov, float weight_decay,
                             uint32_t steps, void* stream) {
  const char* fn = "launch_muon";
  AGPU_TRY(check_muon(lr, momentum, weight_decay, steps, fn));
  if (count && !tensors) return fail(AGPU_ERR_INVALID, "%s: NULL tensor array", fn);
  for (uint32_t i = 0; i < count; ++i)
    AGPU_TRY(check_matrix(tensors[i].rows, tensors[i].cols, fn));
  AGPU_TRY(check_muon_tensors(tensors, count, fn));
  AGPU_TRY(use_device(dev, fn));
  return launch_muon(dev, tensors, count, lr, momentum, nesterov != 0, weight_decay, steps,
                     pick_stream(dev, stream));
}

}  // extern "C"
