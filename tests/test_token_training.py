"""The token ops together, as a user's training loop has them: embedding ->
projections -> head norms with the rotary embedding -> causal attention ->
output projection -> loss on the tape, then one step of both optimisers; and
the LLaMA-style layer with head norms.

On the CPU the same tape runs over numpy (float64 inside), which checks the
recording and the backward rules against differences; on the GPU its results
are compared with that."""
from __future__ import annotations

import numpy as np
import pytest

gpu = pytest.mark.gpu
B, S, H, D, V = 2, 12, 2, 64, 50
E = H * D


class _Buf:
    def __init__(self, data):
        self.data = np.asarray(data, np.float64).reshape(-1)
        self.len = self.data.size


class NumpyDevice:
    """The device methods this training step uses, in float64 (test infrastructure)."""

    def upload(self, x): return _Buf(x)
    def upload_i32(self, x): return np.asarray(x, np.int64).reshape(-1)
    def alloc(self, n): return _Buf(np.zeros(n))
    def read(self, b): return b.data.copy()
    def add(self, a, b): return _Buf(a.data + b.data)
    def sub(self, a, b): return _Buf(a.data - b.data)
    def scale(self, a, s): return _Buf(a.data * s)
    def mse_loss(self, p, t): return _Buf([((p.data - t.data) ** 2).mean()])

    def gemm(self, a, b, batch, m, n, k, trans_a=False, trans_b=False):
        x = a.data.reshape(k, m).T if trans_a else a.data.reshape(m, k)
        y = b.data.reshape(n, k).T if trans_b else b.data.reshape(k, n)
        return _Buf(x @ y)

    def gemm_ex(self, a, b, batch, m, n, k, bias=None, act=0):
        assert bias is None and act == 0
        return self.gemm(a, b, 1, m, n, k)

    def transpose(self, a, o, d0, d1, i):
        return _Buf(a.data.reshape(o, d0, d1, i).transpose(0, 2, 1, 3))

    def embedding(self, t, ids, tokens, vocab, dim, scale):
        rows = t.data.reshape(vocab, dim)[np.maximum(ids, 0)]
        return _Buf(np.where((ids >= 0)[:, None], rows, 0) * scale)

    def embedding_backward(self, g, ids, tokens, vocab, dim, scale):
        d = np.zeros((vocab, dim))
        np.add.at(d, ids[ids >= 0], g.data.reshape(tokens, dim)[ids >= 0] * scale)
        return _Buf(d)

    @staticmethod
    def _angles(pos, batch, seq, rot, base):
        p = np.arange(seq)[None].repeat(batch, 0) if pos is None else pos.reshape(batch, seq)
        a = p[..., None] * base ** (-np.arange(0, rot, 2) / rot)
        return np.cos(a)[:, :, None], np.sin(a)[:, :, None]

    def qk_norm_rope(self, q, k, qw, kw, pos, b, s, hq, hk, d, rot, eps, base, major):
        outs = []
        rot = d if rot is None else rot
        c, sn = self._angles(pos, b, s, rot, base)
        for x, w, h in ((q, qw, hq), (k, kw, hk)):
            x = x.data.reshape(b, s, h, d)
            y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.data
            u, v = y[..., :rot // 2], y[..., rot // 2:rot]
            y = np.concatenate([u * c - v * sn, v * c + u * sn, y[..., rot:]], -1)
            outs.append(_Buf(y.transpose(0, 2, 1, 3) if major else y))
        return tuple(outs)

    def qk_norm_rope_backward(self, gq, gk, q, k, qw, kw, pos, b, s, hq, hk, d, rot, eps, base,
                              major):
        dx, dws = [], []
        rot = d if rot is None else rot
        c, sn = self._angles(pos, b, s, rot, base)
        for g, x, w, h in ((gq, q, qw, hq), (gk, k, kw, hk)):
            x = x.data.reshape(b, s, h, d)
            g = (g.data.reshape(b, h, s, d).transpose(0, 2, 1, 3) if major
                 else g.data.reshape(b, s, h, d))
            u, v = g[..., :rot // 2], g[..., rot // 2:rot]
            g = np.concatenate([u * c + v * sn, v * c - u * sn, g[..., rot:]], -1)
            r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
            n, gw = x * r, g * w.data
            dx.append(_Buf(r * (gw - n * (gw * n).mean(-1, keepdims=True))))
            dws.append(_Buf((g * n).sum((0, 1, 2))))
        return (*dx, *dws)

    def _p(self, q, k, bh, s, d):
        sc = (q.data.reshape(bh, s, d) @ k.data.reshape(bh, s, d).transpose(0, 2, 1)) / np.sqrt(d)
        sc = np.where(np.tril(np.ones((s, s), bool)), sc, -np.inf)
        p = np.exp(sc - sc.max(-1, keepdims=True))
        return p / p.sum(-1, keepdims=True)

    def sdpa_causal(self, q, k, v, bh, s, d):
        return _Buf(self._p(q, k, bh, s, d) @ v.data.reshape(bh, s, d))

    def sdpa_backward(self, q, k, v, g, bh, s, d, causal):
        assert causal
        p = self._p(q, k, bh, s, d)
        g = g.data.reshape(bh, s, d)
        dp = g @ v.data.reshape(bh, s, d).transpose(0, 2, 1)
        ds = p * (dp - (p * dp).sum(-1, keepdims=True)) / np.sqrt(d)
        return (_Buf(ds @ k.data.reshape(bh, s, d)),
                _Buf(ds.transpose(0, 2, 1) @ q.data.reshape(bh, s, d)),
                _Buf(p.transpose(0, 2, 1) @ g))


def _params(r):
    f = lambda *s: (r.standard_normal(s) * 0.2).astype(np.float32)
    return {"table": f(V, E), "wq": f(E, E), "wk": f(E, E), "wv": f(E, E), "wo": f(E, E),
            "qn": 1 + f(D), "kn": 1 + f(D)}


def _batch(r):
    ids = r.integers(0, V, (B, S)).astype(np.int32)
    ids[:, 5] = ids[:, 0]      # the same token twice
    ids[1, -2:] = -1           # padding behind the shorter sequence
    return ids, r.standard_normal(B * S * E).astype(np.float32)


def _train_step(dev, params, ids, target, positions=None):
    """-> (loss, {name: gradient buffer}, tape)."""
    from any_gpu.autograd import Tape
    t = Tape(dev)
    p = {k: t.leaf(v) for k, v in params.items()}
    T = B * S
    pos = None if positions is None else dev.upload_i32(positions)
    x = t.embedding(p["table"], dev.upload_i32(ids), T, V, E, np.sqrt(E))
    q, k, v = (t.linear(x, p[n], None, T, E, E) for n in ("wq", "wk", "wv"))
    q, k = t.qk_norm_rope(q, k, p["qn"], p["kn"], pos, B, S, H, H, D, head_major=True)
    v = t.transpose(v, B, S, H, D)
    o = t.transpose(t.scaled_dot_product_attention(q, k, v, B * H, S, D, causal=True), B, H, S, D)
    y = t.add(x, t.linear(o, p["wo"], None, T, E, E))
    loss = t.mse_loss(y, t.leaf(target))
    t.backward(loss)
    return t.read(loss)[0], {n: t.grad(i) for n, i in p.items()}, t


@pytest.mark.parametrize("positions", [None, "given"])
def test_tape_gradients_against_differences(positions):
    """Central differences of the loss in float64 along random directions."""
    dev, r = NumpyDevice(), np.random.default_rng(0)
    params, (ids, target) = _params(r), _batch(r)
    pos = None if positions is None else r.integers(0, 99, (B, S))
    _, grads, _ = _train_step(dev, params, ids, target, pos)
    for name, value in params.items():
        d = r.standard_normal(value.shape)
        h = 1e-6
        lo, hi = (_train_step(dev, {**params, name: value + s * h * d}, ids, target, pos)[0]
                  for s in (-1, 1))
        want = float((grads[name].data * d.ravel()).sum())
        assert abs((hi - lo) / (2 * h) - want) <= 1e-6 * max(1.0, abs(want)), name


def test_output_that_nothing_uses():
    """Only the queries (or neither output) reach the loss."""
    from any_gpu.autograd import Tape
    dev, r = NumpyDevice(), np.random.default_rng(1)
    for used in ("q", "k", "none"):
        t = Tape(dev)
        q, k = t.leaf(r.standard_normal(24)), t.leaf(r.standard_normal(24))
        w = t.leaf(np.ones(4))
        qo, ko = t.qk_norm_rope(q, k, w, w, None, 1, 3, 2, 2, 4)
        y = {"q": qo, "k": ko, "none": t.leaf(np.ones(24))}[used]
        t.backward(t.mse_loss(y, t.leaf(np.zeros(24))))
        if used == "none":
            assert t.read_grad(q) is None and t.read_grad(w) is None
            continue
        live, dead = (q, k) if used == "q" else (k, q)
        assert np.abs(t.read_grad(live)).max() > 0
        assert np.abs(t.read_grad(dead)).max() == 0


@gpu
def test_training_step(dev):
    """The tape on the GPU in 3xTF32 (products within 1e-5 relative, six of
    them on the longest path: 1e-4 for a gradient), then a step of each optimiser."""
    from any_gpu import AdamW, Muon
    r = np.random.default_rng(0)
    params, (ids, target) = _params(r), _batch(r)
    want_loss, want, _ = _train_step(NumpyDevice(), params, ids, target)
    with dev.precision("tf32x3"):
        loss, grads, tape = _train_step(dev, params, ids, target)
    assert abs(loss - want_loss) <= 1e-5 * want_loss
    for n in params:
        g, w = dev.read(grads[n]).astype(np.float64), want[n].data
        assert np.linalg.norm(g - w) <= 1e-4 * np.linalg.norm(w), n
    matrices, rest = ["wq", "wk", "wv", "wo"], ["table", "qn", "kn"]
    bufs = {n: dev.upload(v) for n, v in params.items()}
    Muon(lr=1e-2).step(dev, [bufs[n] for n in matrices], [grads[n] for n in matrices],
                       [(E, E)] * 4)
    AdamW(lr=1e-2).step(dev, [bufs[n] for n in rest], [grads[n] for n in rest])
    for n in matrices:  # a step moves every matrix by lr 0.2 sqrt(E) times singular values near 1
        move = dev.read(bufs[n]) - params[n].ravel() * (1 - 1e-2 * 0.01)
        s = np.linalg.svd(move.reshape(E, E).astype(np.float64), compute_uv=False)
        assert s.max() <= 1e-2 * 0.2 * np.sqrt(E) * 1.25
    with dev.precision("tf32x3"):
        new = {n: dev.read(b).reshape(params[n].shape) for n, b in bufs.items()}
        _, again, _ = _train_step(dev, new, ids, target)
    assert all(np.isfinite(dev.read(g)).all() for g in again.values())


@gpu
def test_a_training_step_moves_every_matrix(dev):
    """The matrices after a step on the tape's gradients against the float64 step on the same
    gradients: |W error| <= 4 u (|W| + |move|) + 2e-5 |move|, as in the optimiser's tests."""
    from any_gpu import Muon
    from test_muon import TOL, U, _step
    r = np.random.default_rng(2)
    params, (ids, target) = _params(r), _batch(r)
    _, grads, tape = _train_step(dev, params, ids, target)
    names = ["wq", "wk", "wv", "wo"]
    bufs = {n: dev.upload(params[n]) for n in names}
    opt = Muon(lr=1e-2)
    opt.step(dev, [bufs[n] for n in names], [grads[n] for n in names], [(E, E)] * 4)
    for n in names:
        g = dev.read(grads[n]).reshape(E, E)
        want, _, move = _step(params[n], g, np.zeros((E, E)), 1e-2, 0.95, True, 0.01, 5)
        got = dev.read(bufs[n]).reshape(E, E)
        assert np.linalg.norm(got - want) <= 4 * U * (np.linalg.norm(want) + move) + TOL * move
        assert np.linalg.norm(got - params[n]) >= 0.5 * move > 0


@gpu
def test_llama_layer_with_head_norms(dev, orc):
    """The layer with qk_norm against the same layer composed in float64 on its
    attention inputs: the fused pass is the only difference to the layer without."""
    import torch
    from any_gpu.llama import LlamaDims, layer_forward
    dims = LlamaDims(batch=2, seq=40, d_model=256, heads=4, ffn=96, qk_norm=True)
    g = torch.Generator().manual_seed(0)
    f = lambda *s: (torch.randn(*s, generator=g) * 0.1).cuda()
    d, F, T = dims.d_model, dims.ffn, dims.tokens
    w = {"attn_norm": 1 + f(d), "ffn_norm": 1 + f(d), "wqkv": f(d, 3 * d), "wo": f(d, d),
         "wgu": f(d, 2 * F), "wd": f(F, d), "q_norm": 1 + f(64), "k_norm": 1 + f(64)}
    x = f(T, d) * 10
    ws = {k: torch.zeros(n, device="cuda") for k, n in dims.workspace_elems().items()}
    y = torch.zeros(T, d, device="cuda")
    torch.cuda.synchronize()
    with dev.precision("tf32x3"):
        layer_forward(dev, dims, x.data_ptr(), {k: v.data_ptr() for k, v in w.items()},
                      {k: v.data_ptr() for k, v in ws.items()}, y.data_ptr())
    dev.synchronize()
    w = {k: v.double() for k, v in w.items()}
    norm = lambda t, wt: t / (t.square().mean(-1, keepdim=True) + dims.eps).sqrt() * wt
    X = x.double()
    q, k, v = (norm(X, w["attn_norm"]) @ w["wqkv"]).view(2, 40, 3, 4, 64).unbind(2)
    a = torch.arange(40, device="cuda").double()[:, None] * 10000.0 ** (
        -torch.arange(0, 64, 2, device="cuda").double() / 64)
    c, s = a.cos()[None, :, None], a.sin()[None, :, None]

    def turn(t):
        return torch.cat([t[..., :32] * c - t[..., 32:] * s, t[..., 32:] * c + t[..., :32] * s], -1)
    q, k = turn(norm(q, w["q_norm"])), turn(norm(k, w["k_norm"]))
    p = (torch.einsum("bqhd,bkhd->bhqk", q, k) / 8).softmax(-1)
    o = torch.einsum("bhqk,bkhd->bqhd", p, v).reshape(T, d)
    x2 = X + o @ w["wo"]
    gu = (norm(x2, w["ffn_norm"]) @ w["wgu"]).view(T, F // 32, 2, 32)
    act = (torch.nn.functional.silu(gu[:, :, 0]) * gu[:, :, 1]).reshape(T, F)
    want = x2 + act @ w["wd"]
    assert (y.double() - want).norm() <= 1e-4 * want.norm()  # as the layer's other tests in 3xTF32


@gpu
def test_calls_on_two_streams_at_once(dev):
    """Calls that take scratch, side by side on two streams, give what they give alone."""
    import torch
    from any_gpu import QkNormRope, muon_tensors
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    tokens, vocab, dim, shape = 3000, 700, 256, QkNormRope(2, 400, 6, 2, 64)
    sides = []
    for _ in range(2):
        sides.append({"ids": torch.randint(-1, vocab, (tokens,), generator=g, device="cuda",
                                           dtype=torch.int32),
                      "grad": rand(tokens, dim), "gq": rand(2, 400, 6, 64),
                      "gk": rand(2, 400, 2, 64), "q": rand(2, 400, 6, 64),
                      "k": rand(2, 400, 2, 64), "w": rand(64), "mats": [rand(200, 300), rand(60, 90)]})

    def run(x, stream):
        """Enqueues one call of each; the outputs, filled beforehand."""
        h = stream.cuda_stream
        dev.launch_embedding_backward(x["grad"].data_ptr(), x["ids"].data_ptr(),
                                      x["o"][0].data_ptr(), tokens, vocab, dim, 1.0, stream=h)
        dev.launch_qk_norm_rope_backward(
            shape, x["gq"].data_ptr(), x["gk"].data_ptr(), x["q"].data_ptr(), x["k"].data_ptr(),
            x["w"].data_ptr(), x["w"].data_ptr(), 0, *[t.data_ptr() for t in x["o"][1:5]], h)
        dev.launch_muon(muon_tensors([(w.data_ptr(), u.data_ptr(), m.data_ptr(), *u.shape)
                                      for w, u, m in zip(x["o"][5:7], x["mats"], x["o"][7:9])]),
                        0.02, 0.9, True, 0.0, 5, h)

    def outputs():
        return [torch.zeros(s, device="cuda") for s in
                [(vocab, dim), (2, 400, 6, 64), (2, 400, 2, 64), (64,), (64,), (200, 300), (60, 90),
                 (200, 300), (60, 90)]]
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for together in (False, True):
        for x in sides:
            x["o"] = outputs()
        torch.cuda.synchronize()
        for _ in range(6):
            for x, stream in zip(sides, streams):
                run(x, stream)
                if not together:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        results.append([x["o"] for x in sides])
    for alone, beside in zip(*results):
        for a, b in zip(alone, beside):
            assert torch.equal(a, b)
    dev.synchronize()
