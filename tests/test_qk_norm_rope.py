"""Head norms with the rotary embedding, and their backward, against numpy in
float64.

Tolerances (u = 2^-24, D = head dim).  The sum of D squares is off by at most
D u relative (any order), so r = 1 / sqrt(.) by (D / 2 + 4) u; a cosine or sine
by 4 u absolute (one rounding of the reduced angle, put back, and two units of
sincosf) plus p 2^-51 for the angle itself in double.  An output is two
products of such factors and a sum: (D / 2 + 16) u + p 2^-51 times |y_a| + |y_b|.
A gradient element r (h - n mean(h n)) adds the mean's own sum of D terms:
see _backward_bound.  A weight's gradient sums N terms: (N + D / 2 + 16) u
times the sum of their magnitudes."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

U = 2.0 ** -24
gpu = pytest.mark.gpu


def _turn(pos, rot, base):
    a = pos[..., None].astype(np.float64) * base ** (-np.arange(0, rot, 2) / max(rot, 1))
    return np.cos(a)[:, :, None], np.sin(a)[:, :, None]


def _rotate(y, c, s, rot):
    a, b = y[..., :rot // 2], y[..., rot // 2:rot]
    return np.concatenate([a * c - b * s, b * c + a * s, y[..., rot:]], -1)


def _forward(x, w, pos, rot, eps, base):
    """x [B, S, H, D] -> (output, bound), float64."""
    x = x.astype(np.float64)
    d = x.shape[-1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    c, s = _turn(pos, rot, base)
    mag = np.abs(y)
    pair = _rotate(mag, np.ones_like(c), -np.ones_like(s), rot)
    pair[..., rot // 2:rot] = mag[..., :rot // 2] + mag[..., rot // 2:rot]
    return _rotate(y, c, s, rot), ((d / 2 + 16) * U + np.abs(pos).max() * 2.0 ** -51) * pair


def _backward(x, w, pos, rot, eps, base, g):
    """(dx, its bound, dw, its bound), float64."""
    x, g = x.astype(np.float64), g.astype(np.float64)
    d, far = x.shape[-1], np.abs(pos).max() * 2.0 ** -51
    c, s = _turn(pos, rot, base)
    u = _rotate(g, c, -s, rot)
    mag = np.abs(g)
    gu = mag.copy()
    gu[..., :rot // 2] += mag[..., rot // 2:rot]
    gu[..., rot // 2:rot] += mag[..., :rot // 2]       # bounds |u|
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n, h = x * r, u * w
    dx = r * (h - n * (h * n).mean(-1, keepdims=True))
    hn = (gu * np.abs(w) * np.abs(n)).mean(-1, keepdims=True)
    # h: 8 u; r twice, n three times in the second term; the mean's D terms
    bound = r * ((d / 2 + 16) * U + far) * gu * np.abs(w) \
        + r * np.abs(n) * ((2.5 * d + 32) * U + far) * hn
    count = x.shape[0] * x.shape[1] * x.shape[2]
    dw = (u * n).sum((0, 1, 2))
    wb = ((count + d / 2 + 16) * U + far) * (gu * np.abs(n)).sum((0, 1, 2))
    return dx, bound, dw, wb


# batch, seq, q heads, k heads, dim, rot, positions given
CASES = [(1, 1, 1, 1, 2, 2, False), (1, 1, 32, 8, 128, 128, True), (2, 5, 3, 1, 64, 64, False),
         (3, 7, 5, 5, 80, 40, True), (2, 33, 4, 2, 256, 256, True), (1, 9, 6, 3, 96, 32, False),
         (2, 4, 2, 1, 50, 24, True), (1, 3, 2, 2, 7, 6, False), (2, 3, 1, 4, 8, 0, True),
         (1, 2, 3, 2, 1024, 1024, True), (1, 1, 17, 3, 1, 0, False), (4, 130, 9, 3, 32, 16, True),
         (1, 6, 40, 40, 16, 8, False), (2, 3, 0, 4, 64, 64, True), (2, 3, 4, 0, 66, 64, True)]


def _inputs(case, seed=0):
    b, s, hq, hk, d, rot, given = case
    r = np.random.default_rng(seed + d + hq)
    f = lambda *sh: r.standard_normal(sh).astype(np.float32)
    pos = r.integers(-5, 200000, (b, s)) if given else np.broadcast_to(np.arange(s), (b, s))
    x = {"q": f(b, s, hq, d) * 3, "k": f(b, s, hk, d) * 0.1, "qw": 1 + f(d) * 0.2,
         "kw": 1 + f(d) * 0.2, "gq": f(b, s, hq, d), "gk": f(b, s, hk, d)}
    if hq > 1:
        x["q"][0, 0, 1] = 0  # a zero head: r = 1 / sqrt(eps)
    return x, pos.astype(np.int32)


def _major(a):
    return np.ascontiguousarray(a.transpose(0, 2, 1, 3))


@gpu
@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_backward(dev, case, head_major):
    b, s, hq, hk, d, rot, given = case
    x, pos = _inputs(case)
    eps, base = 1e-5, 10000.0
    geo = (b, s, hq, hk, d, rot, eps, base, head_major)
    up = lambda a: dev.upload(a) if a.size else None
    P = dev.upload_i32(pos) if given else None
    Q, K, QW, KW = up(x["q"]), up(x["k"]), up(x["qw"]), up(x["kw"])
    lay = _major if head_major else (lambda a: a)
    outs = dev.qk_norm_rope(Q, K, QW, KW, P, *geo)
    for out, n, heads in zip(outs, "qk", (hq, hk)):
        if not heads:
            assert out is None
            continue
        want, tol = _forward(x[n], x[n + "w"].astype(np.float64), pos, rot, eps, base)
        got = dev.read(out).reshape(lay(want).shape)
        assert (np.abs(got - lay(want)) <= lay(tol)).all()
    grads = dev.qk_norm_rope_backward(up(lay(x["gq"])), up(lay(x["gk"])), Q, K, QW, KW, P, *geo)
    for dx, dw, n, heads in zip(grads[:2], grads[2:], "qk", (hq, hk)):
        if not heads:
            assert dx is None
            np.testing.assert_array_equal(dev.read(dw), np.zeros(d))
            continue
        want, tol, want_w, tol_w = _backward(x[n], x[n + "w"].astype(np.float64), pos, rot, eps,
                                             base, x["g" + n])
        assert (np.abs(dev.read(dx).reshape(want.shape) - want) <= tol).all()
        assert (np.abs(dev.read(dw) - want_w) <= tol_w).all()


@gpu
def test_no_weights_and_no_weight_gradients(dev):
    case = (2, 3, 4, 2, 64, 64, False)
    b, s, hq, hk, d, rot, _ = case
    x, pos = _inputs(case)
    geo = (b, s, hq, hk, d, rot, 1e-6, 500.0, False)
    Q, K = dev.upload(x["q"]), dev.upload(x["k"])
    qo, ko = dev.qk_norm_rope(Q, K, None, None, None, *geo)
    want, tol = _forward(x["q"], np.ones(d), pos, rot, 1e-6, 500.0)
    assert (np.abs(dev.read(qo).reshape(want.shape) - want) <= tol).all()
    from any_gpu import QkNormRope
    dq, dk = dev.alloc(Q.len), dev.alloc(K.len)
    dev.launch_qk_norm_rope_backward(QkNormRope(b, s, hq, hk, d, rot, 1e-6, 500.0),
                                     dev.upload(x["gq"]).device_ptr,
                                     dev.upload(x["gk"]).device_ptr, Q.device_ptr, K.device_ptr,
                                     0, 0, 0, dq.device_ptr, dk.device_ptr)
    want, tol, _, _ = _backward(x["k"], np.ones(d), pos, rot, 1e-6, 500.0, x["gk"])
    assert (np.abs(dev.read(dk).reshape(want.shape) - want) <= tol).all()


@gpu
@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("dim", [128, 72])
def test_packed_strides_in_place_on_a_callers_stream(dev, dim, shift):
    """q and k inside a packed [B, S, H + 2 K, D] projection, rotated in place."""
    import torch
    from any_gpu import QkNormRope
    case = (2, 5, 4, 2, dim, dim, True)
    b, s, hq, hk, d, rot, _ = case
    x, pos = _inputs(case)
    r = np.random.default_rng(1)
    v = r.standard_normal((b, s, hk, d)).astype(np.float32)
    packed = np.concatenate([x["q"], x["k"], v], 2)
    buf = torch.cat([torch.full((shift,), 5.0), torch.from_numpy(packed).reshape(-1)]).cuda()
    P = torch.from_numpy(pos).cuda()
    QW, KW = torch.from_numpy(x["qw"]).cuda(), torch.from_numpy(x["kw"]).cuda()
    st = ((hq + 2 * hk) * d, d, s * (hq + 2 * hk) * d)
    shape = QkNormRope(b, s, hq, hk, d, rot, 1e-6, 10000.0, st, st, st, st)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    q = buf.data_ptr() + 4 * shift
    dev.launch_qk_norm_rope(shape, q, q + 4 * hq * d, QW.data_ptr(), KW.data_ptr(), P.data_ptr(),
                            q, q + 4 * hq * d, stream.cuda_stream)
    stream.synchronize()
    assert (buf[:shift] == 5).all()
    got = buf[shift:].cpu().numpy().reshape(packed.shape)
    for n, sl in (("q", slice(0, hq)), ("k", slice(hq, hq + hk))):
        want, tol = _forward(x[n], x[n + "w"].astype(np.float64), pos, rot, 1e-6, 10000.0)
        assert (np.abs(got[:, :, sl] - want) <= tol).all()
    np.testing.assert_array_equal(got[:, :, hq + hk:], v)


@gpu
@pytest.mark.parametrize("dim", [64, 50])
def test_strides_past_32_bits(dev, dim):
    """Two sequences 2^32 + 64 elements apart, rotated in place, and their gradients."""
    import torch
    from any_gpu import QkNormRope
    case = (2, 3, 2, 0, dim, dim, False)
    b, s, h, _, d, rot, _ = case
    x, pos = _inputs(case)
    far = 2 ** 32 + 64
    buf = torch.empty(far + s * h * d, device="cuda")
    views = [buf[i * far:i * far + s * h * d].view(s, h, d) for i in range(b)]
    near, wide = (h * d, d, s * h * d), (h * d, d, far)
    W = torch.from_numpy(x["qw"]).cuda()

    def fill(a):
        for v, y in zip(views, a):
            v.copy_(torch.from_numpy(y))
        torch.cuda.synchronize()

    def read():
        dev.synchronize()
        return np.stack([v.cpu().numpy() for v in views])
    zeros = (0, 0, 0)
    fill(x["q"])
    shape = QkNormRope(b, s, h, 0, d, rot, 1e-6, 10000.0, wide, zeros, wide, zeros)
    dev.launch_qk_norm_rope(shape, buf.data_ptr(), 0, W.data_ptr(), 0, 0, buf.data_ptr(), 0)
    want, tol = _forward(x["q"], x["qw"].astype(np.float64), pos, rot, 1e-6, 10000.0)
    assert (np.abs(read() - want) <= tol).all()
    fill(x["gq"])  # gradients far apart, the input near
    Q, dx = torch.from_numpy(x["q"]).cuda(), torch.empty(x["q"].shape, device="cuda")
    dw = torch.empty(d, device="cuda")
    torch.cuda.synchronize()
    shape = QkNormRope(b, s, h, 0, d, rot, 1e-6, 10000.0, near, zeros, wide, zeros)
    dev.launch_qk_norm_rope_backward(shape, buf.data_ptr(), 0, Q.data_ptr(), 0, W.data_ptr(), 0, 0,
                                     dx.data_ptr(), 0, dw.data_ptr(), 0)
    dev.synchronize()
    want, tol, want_w, tol_w = _backward(x["q"], x["qw"].astype(np.float64), pos, rot, 1e-6,
                                         10000.0, x["gq"])
    assert (np.abs(dx.cpu().numpy() - want) <= tol).all()
    assert (np.abs(dw.cpu().numpy() - want_w) <= tol_w).all()


@gpu
def test_matches_rmsnorm_then_rope(dev):
    """The fused pass against the two ops it fuses: both are within the bound of the formula."""
    b, s, h, d = 2, 17, 3, 128
    x, pos = _inputs((b, s, h, h, d, d, False))
    X, W = dev.upload(x["q"]), dev.upload(x["qw"])
    two = dev.read(dev.rope(dev.rmsnorm(X, W, b * s * h, d, 1e-6), b, s, h, d))
    one = dev.read(dev.qk_norm_rope(X, None, W, None, None, b, s, h, 0, d)[0])
    _, tol = _forward(x["q"], x["qw"].astype(np.float64), pos, d, 1e-6, 10000.0)
    assert (np.abs(one - two) <= 2 * tol.ravel()).all()


@gpu
def test_backward_is_deterministic_and_replays_in_a_graph(dev):
    import torch
    from any_gpu import QkNormRope
    b, s, hq, hk, d = 2, 300, 8, 2, 64
    x, _ = _inputs((b, s, hq, hk, d, d, False))
    t = {k: torch.from_numpy(v).cuda() for k, v in x.items()}
    shape = QkNormRope(b, s, hq, hk, d)
    outs = []
    for graphed in (False, True):
        o = [torch.zeros_like(t[k]) for k in ("q", "k", "qw", "kw")]
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        call = lambda: dev.launch_qk_norm_rope_backward(
            shape, t["gq"].data_ptr(), t["gk"].data_ptr(), t["q"].data_ptr(), t["k"].data_ptr(),
            t["qw"].data_ptr(), t["kw"].data_ptr(), 0, *[v.data_ptr() for v in o],
            stream.cuda_stream)
        if graphed:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                call()
            for _ in range(2):
                with torch.cuda.stream(stream):
                    graph.replay()
        else:
            call()
        torch.cuda.synchronize()
        outs.append(o)
    for a, c in zip(*outs):
        assert torch.equal(a, c)


@gpu
def test_empty_and_nonfinite(dev):
    empty = dev.upload(np.zeros(0))
    w = dev.upload(np.ones(8))
    q, k = dev.qk_norm_rope(empty, empty, w, w, None, 0, 5, 2, 1, 8)
    assert q.len == 0 and k.len == 0
    grads = dev.qk_norm_rope_backward(empty, empty, empty, empty, w, w, None, 0, 5, 2, 1, 8)
    np.testing.assert_array_equal(dev.read(grads[2]), np.zeros(8))
    x = np.ones((1, 3, 1, 8), np.float32)
    x[0, 1, 0, 3] = np.nan
    y = dev.read(dev.qk_norm_rope(dev.upload(x), None, w, None, None, 1, 3, 1, 0, 8)[0])
    y = y.reshape(3, 8)
    assert np.isnan(y[1]).all() and np.isfinite(y[[0, 2]]).all()


@gpu
def test_buffer_layer_refusals(dev):
    from any_gpu import AnyGpuError

    def status(*a, **k):
        with pytest.raises(AnyGpuError) as e:
            dev.qk_norm_rope(*a, **k)
        return e.value.status
    x, w, p = dev.upload(np.ones(48)), dev.upload(np.ones(8)), dev.upload_i32([0, 1, 2])
    assert status(x, None, w, None, p, 1, 3, 3, 0, 8) == 1          # q length
    assert status(x, None, dev.upload(np.ones(9)), None, p, 1, 3, 2, 0, 8) == 1
    assert status(x, None, w, None, dev.upload_i32([0]), 1, 3, 2, 0, 8) == 1
    assert status(x, None, w, None, dev.upload(np.ones(3)), 1, 3, 2, 0, 8) == 2  # f32 positions
    assert status(None, None, w, None, p, 1, 3, 2, 0, 8) == 2
    dev.synchronize()


def test_launch_layer_refusals():
    """Arguments are checked before the device: no GPU is needed to be refused."""
    from any_gpu import QkNormRope, _lib
    lib = _lib.load()
    p = C.c_void_p(256)

    def status(ptrs=(p,) * 7, **k):
        a = dict(batch=2, seq=3, q_heads=4, k_heads=2, dim=8)
        a.update(k)
        shape = QkNormRope(**a)
        s1 = lib.agpu_launch_qk_norm_rope(None, C.byref(shape), *ptrs, None)
        s2 = lib.agpu_launch_qk_norm_rope_backward(None, C.byref(shape), p, p, *ptrs, p, p, None)
        assert s1 == s2
        return s1
    assert status(dim=0) == 7 and status(dim=1025) == 7
    assert status(rot_dim=3) == 1 and status(rot_dim=10) == 1
    assert status(base=0.0) == 2 and status(base=float("inf")) == 2 and status(base=-1.0) == 2
    assert status(eps=-1.0) == 2 and status(eps=float("nan")) == 2
    assert status(batch=2**16, seq=2**16) == 7 and status(q_heads=65536) == 7
    assert status(q_in=(32, 7, 96)) == 1        # heads overlap
    assert status(k_out=(16, 8, 40)) == 1       # batches overlap
    assert status(q_out=(8, 0, 96)) == 1
    assert status(ptrs=(None, p, p, p, p, p, p)) == 2
    assert status(ptrs=(p, p, p, p, p, p, None)) == 2
    assert status() == 2 and b"NULL device" in lib.agpu_last_error_message()
    # legal layouts get as far as the device: head-major, and axes of one element
    for k in (dict(q_out=(8, 24, 96)), dict(batch=1, q_in=(32, 8, 0)), dict(seq=1, k_in=(0, 8, 16))):
        assert status(**k) == 2 and b"NULL device" in lib.agpu_last_error_message()
    assert lib.agpu_launch_qk_norm_rope(None, None, *([p] * 7), None) == 2


def test_formula_against_differences():
    """The gradients the GPU tests compare with, against central differences in
    float64 (step 1e-5: truncation ~1e-10, rounding ~1e-11 of losses ~1)."""
    r = np.random.default_rng(0)
    x, w, g = r.standard_normal((2, 2, 2, 6)), 1 + 0.3 * r.standard_normal(6), None
    g = r.standard_normal(x.shape)
    pos, rot = r.integers(0, 50, (2, 2)), 4
    loss = lambda x_, w_: float((_forward(x_, w_, pos, rot, 1e-3, 100.0)[0] * g).sum())
    dx, _, dw, _ = _backward(x, w, pos, rot, 1e-3, 100.0, g)
    h = 1e-5
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = h
        assert abs((loss(x + e, w) - loss(x - e, w)) / (2 * h) - dx[i]) <= 1e-7
    for i in range(6):
        e = np.zeros(6)
        e[i] = h
        assert abs((loss(x, w + e) - loss(x, w - e)) / (2 * h) - dw[i]) <= 1e-7
