"""Orthogonalised updates against numpy in float64.

Tolerances, relative in the Frobenius norm.

TOL = 2e-5, for matrices whose singular values are spread like a gradient's
(a few large ones on a floor of noise that the iteration lifts to 1 too).  One
step maps a singular value s to s (a + b l + c l^2), l = s^2 <= 1.46; a relative
error e of A = X X^T or of B = b A + c A^2 (against its largest eigenvalue)
moves the result by at most 1.21 (|b| + 2 c 1.46) 1.46 e < 20 e.  The products
keep 22 bits of each factor and sum in 32-bit accumulators: e <= 2^-20.  (A of a
long contraction may be a sum of parts P = X' X'^T over columns X' of X, each
rounded to 22 bits: |P_ij| <= sqrt(P_ii P_jj), and these sum to at most
sqrt(A_ii A_jj), so the roundings together are within one of that size.)

DEGENERATE = 1.1e-3, for matrices with singular values that stay 0 (rank 1, a
single entry).  What a step leaves in those directions is not moved towards 1
but multiplied by the slope at 0, a = 3.4445, in every later step: by a^5 =
485 from the initial rounding on.  Rounding X to 22 bits before each step:
2^-22 (a^5 + a^4 + a^3 + a^2 + a) = 2^-22 685 = 1.6e-4.  An error e of A turns
a large direction into a dead one, |b| e <= 4.775 2^-20 a step, and the steps
behind it multiply that by 1 + a + ... + a^4 = 198: 9.0e-4.

SEGMENTS = 3e-4, for groups of wide matrices, whose steps may be taken on A =
X X^T for up to three steps between two products with X (A' = M A M, M = a I +
b A + c A^2).  An error e <= 2^-20 of A grows there by at most a^2 = 11.9 a
step, in directions of small singular values, where M is near a: a segment of
three moves M by |b| / a (1 + 11.9 + 141) e = 214 e = 2.0e-4, one of two by
18 e = 1.7e-5.  Later steps do not enlarge a relative error of a small singular
value.  Of one segment of three and two of two, with TOL: 2.6e-4."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

U = 2.0 ** -24
TOL = 2e-5
DEGENERATE = 1.1e-3
SEGMENTS = 3e-4
A, B, CC = 3.4445, -4.7750, 2.0315
gpu = pytest.mark.gpu


def _orthogonalize(u, steps=5):
    u = u.astype(np.float64)
    x = u / max(np.linalg.norm(u), 1e-30)
    tall = u.shape[0] > u.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        g = x @ x.T
        x = A * x + (B * g + CC * (g @ g)) @ x
    return x.T if tall else x


def _rel(got, want):
    return np.linalg.norm(np.asarray(got, np.float64).ravel() - want.ravel()) / max(
        np.linalg.norm(want), 1e-300)


def _gradient(r, rows, cols):
    """A decaying spectrum on top of noise."""
    k = min(rows, cols, 16)
    x = (r.standard_normal((rows, k)) * 0.7 ** np.arange(k)) @ r.standard_normal((k, cols))
    return (x + 0.5 * r.standard_normal((rows, cols))).astype(np.float32)


SHAPES = [(1, 1), (1, 9), (9, 1), (7, 5), (32, 32), (33, 129), (64, 256), (128, 128), (127, 127),
          (130, 100), (129, 257), (256, 512), (200, 1000), (1000, 200), (255, 300), (513, 520),
          (640, 384), (1024, 1031), (100, 300), (128, 2048), (2000, 64), (40, 513), (1030, 16),
          (128, 2049), (128, 4096), (3900, 60), (19, 4097), (17, 767), (96, 1500), (65, 256),
          (200, 5000), (6000, 140), (300, 1500), (130, 8191), (50, 4200), (260, 1025), (2049, 257)]


@gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_orthogonalize(dev, rows, cols):
    r = np.random.default_rng(rows * cols)
    x = _gradient(r, rows, cols) * np.float32(1e-3)
    X = dev.upload(x)
    got = dev.read(dev.orthogonalize(X, 1, rows, cols))
    assert _rel(got, _orthogonalize(x)) <= TOL
    np.testing.assert_array_equal(dev.read(X).reshape(x.shape), x)  # the input is only read
    np.testing.assert_array_equal(got, dev.read(dev.orthogonalize(X, 1, rows, cols)))


@gpu
@pytest.mark.parametrize("batch,rows,cols,steps", [(3, 40, 72, 1), (2, 130, 64, 3), (5, 256, 256, 5),
                                                   (2, 300, 700, 8), (9, 16, 16, 5)])
def test_batches_and_steps(dev, batch, rows, cols, steps):
    r = np.random.default_rng(batch)
    # scales far apart: every matrix is normalised by itself
    x = np.stack([_gradient(r, rows, cols) * np.float32(10.0 ** (6 * i - 12)) for i in range(batch)])
    x[-1] = _gradient(r, rows, cols)
    got = dev.read(dev.orthogonalize(dev.upload(x), batch, rows, cols, steps)).reshape(x.shape)
    for g, m in zip(got, x):
        assert _rel(g, _orthogonalize(m, steps)) <= TOL


# Groups that fill the card: tiles of CTA pairs, steps on the Gram matrix (m >=
# 512, n >= 1.5 m), more matrices than a launch takes, of either kind.
@gpu
@pytest.mark.parametrize("batch,rows,cols,steps,tol", [
    (24, 600, 600, 2, TOL), (26, 520, 800, 5, SEGMENTS), (8, 1000, 1537, 4, SEGMENTS),
    (8, 1537, 1000, 7, SEGMENTS), (7, 1025, 1540, 3, SEGMENTS), (27, 140, 150, 5, TOL),
    (83, 40, 30, 5, TOL), (50, 20, 600, 3, TOL), (3, 150, 2100, 5, TOL), (9, 5000, 20, 5, TOL),
    (2, 700, 4000, 5, TOL)])
def test_large_groups(dev, batch, rows, cols, steps, tol):
    r = np.random.default_rng(rows)
    x = np.stack([_gradient(r, rows, cols) for i in range(batch)])
    X = dev.upload(x)
    got = dev.read(dev.orthogonalize(X, batch, rows, cols, steps))
    np.testing.assert_array_equal(got, dev.read(dev.orthogonalize(X, batch, rows, cols, steps)))
    got = got.reshape(x.shape)
    few = max(rows, cols) > 256
    for i in {0, 11, 12, 24, batch - 1} if few else range(batch):
        if i < batch:
            assert _rel(got[i], _orthogonalize(x[i], steps)) <= tol
    assert np.isfinite(got).all()


def _worst_line(got, want):
    """Largest relative error of a line along the longer side."""
    axis = 1 if want.shape[0] <= want.shape[1] else 0
    return (np.linalg.norm(got.reshape(want.shape) - want, axis=axis)
            / np.linalg.norm(want, axis=axis)).max()


@gpu
@pytest.mark.parametrize("batch,rows,cols,tol", [
    (1, 64, 256, TOL), (1, 256, 64, TOL), (1, 120, 1000, TOL), (1, 300, 700, TOL),
    (1, 700, 300, TOL), (1, 200, 5000, TOL), (8, 1000, 1537, SEGMENTS)])
@pytest.mark.parametrize("scale", [1e-4, 1e-6])
def test_lines_of_very_different_size(dev, batch, rows, cols, tol, scale):
    """Every fourth line (along the longer side) far smaller than the others: each is as
    accurate as the matrix.  With X = D Y, D the lines' scales, A = D Y Y^T D, and what
    is said above of X, A and M holds of row i relative to |Y_i| d_i, and of their entries
    (i, j) relative to d_i d_j, as long as an entry keeps its 22 bits: down to 2^-28, and
    these are above 2^-31 (three bits fewer, in one rounding of several)."""
    r = np.random.default_rng(rows)
    x = r.standard_normal((batch, rows, cols)).astype(np.float32)
    lines = x if rows <= cols else x.transpose(0, 2, 1)
    lines[:, ::4] *= np.float32(scale)
    lines[:, 5] *= np.float32(1e-3)
    got = dev.read(dev.orthogonalize(dev.upload(x), batch, rows, cols)).reshape(x.shape)
    for i in {0, batch - 1}:
        assert _worst_line(got[i], _orthogonalize(x[i])) <= tol


@gpu
def test_parts_of_a_long_contraction_are_summed_in_32_bits(dev):
    """A = X X^T of two rows of 8192, dealt out over slices of 512 columns, whose first
    two parts of A_10 are 8390662 and -8390661 units of the last place of a float of
    their size: what is left, one unit, is lost if a part keeps fewer bits.

    Every number up to A_10 is a whole one that a float holds: |x|^2 = 2^30, so the
    scaled X is x itself, sums stay below 2^24, and the factor 1 + 2^-23 moves both
    parts by one unit.  One step, in a column where row 1 is zero: out_1 = M_10 x_0,
    M_10 = A_10 (b + c (A_00 + A_11)), A_00 + A_11 = 1.  M_10 2^14 = 2.74 2^-16 is kept
    in steps of 2^-24, within 7.2e-4 of itself."""
    x = np.zeros((2, 8192))
    x[:, :511] = 128
    x[:, 511] = 42, 439
    x[0, 512:1023], x[1, 512:1023] = 128, -128
    x[:, 1023] = 103, -179
    assert [x[0, s:s + 512] @ x[1, s:s + 512] for s in (0, 512)] == [8390662, -8390661]
    x[0, 1024:3000] = 512
    free = iter(range(4096, 8192))
    rest = 2**30 - int((x * x).sum())
    while rest:  # the remaining squares, in columns where row 0 is zero
        v = min(512, int(np.sqrt(rest)))
        x[1, next(free)] = v
        rest -= v * v
    assert (x * x).sum() == 2**30 and x[0] @ x[1] == 1
    got = dev.read(dev.orthogonalize(dev.upload(x.astype(np.float32)), 1, 2, 8192, 1))
    want = (B + CC) * 2.0**-30 * 512 / 2**15
    assert (np.abs(got.reshape(2, 8192)[1, 1024:3000] - want) <= 1e-3 * abs(want)).all()


def _orthogonalize32(u, steps):
    """The iteration in float32 throughout."""
    f = np.float32
    x = u / f(np.linalg.norm(u.astype(np.float64)))
    tall = u.shape[0] > u.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        g = x @ x.T
        x = f(A) * x + (f(B) * g + f(CC) * (g @ g)) @ x
    assert x.dtype == f
    return x.T if tall else x


@gpu
@pytest.mark.parametrize("batch,rows,cols,steps", [
    (26, 520, 800, 5), (8, 1000, 1537, 4), (8, 1537, 1000, 7), (7, 1025, 1540, 3),
    (13, 600, 4000, 5), (1, 300, 700, 5), (1, 200, 5000, 5), (1, 1024, 1024, 5)])
def test_as_accurate_as_float32(dev, batch, rows, cols, steps):
    """Matrices without small singular values: ten times, at most, the error of the same
    iteration in float32.  What dominates a product here (the diagonal of M = a I + b A +
    c A A) is one term: float32 rounds it once, 2^-24.  The kernel rounds both operands to
    22 bits, 2^-23 each, and truncates the term in up to four MMAs, 2^-23 each, one of which
    the factor 1 + 2^-23 puts back: 5 2^-23 = 10 2^-24.  Both errors then take the same way
    through the steps.  (13 of 600 x 4000: twelve and one whose columns are dealt out, both
    in steps on the Gram matrix.)"""
    r = np.random.default_rng(rows + batch)
    x = r.standard_normal((batch, rows, cols)).astype(np.float32)
    got = dev.read(dev.orthogonalize(dev.upload(x), batch, rows, cols, steps)).reshape(x.shape)
    for i in {0, batch - 1}:
        want = _orthogonalize(x[i], steps)
        assert _rel(got[i], want) <= 10 * _rel(_orthogonalize32(x[i], steps), want)


@gpu
def test_degenerate_members_of_a_wide_group(dev):
    """On the Gram path, beside ordinary ones: a zero matrix, one of rank 1, one with a NaN,
    one with an infinity.

    Rank 1, as for DEGENERATE: rounding X before each step leaves 1.6e-4.  An error e <=
    2^-20 of A turns the large direction into a dead one, |b| e; in a segment the next A' =
    M A M multiplies it by at most 1.2 a = 4.1.  Steps of segments of 3 and 2 leave |b| e
    (a^4 + 5.1 a^3 + 22.1 a^2 + a + 5.1) = 4.775 621 e = 2.8e-3."""
    r = np.random.default_rng(4)
    x = np.stack([_gradient(r, 520, 800) for _ in range(26)])
    plain = dev.read(dev.orthogonalize(dev.upload(x), *x.shape)).reshape(x.shape)
    x[1] = 0
    x[3] = np.outer(np.linspace(-1, 1, 520), np.arange(1, 801))
    x[12, 519, 7] = np.nan
    x[25, 0, 799] = np.inf
    got = dev.read(dev.orthogonalize(dev.upload(x), *x.shape)).reshape(x.shape)
    assert not got[1].any()
    assert _rel(got[3], _orthogonalize(x[3])) <= 3e-3
    assert np.isnan(got[12]).all() and np.isnan(got[25]).all()
    rest = [i for i in range(26) if i not in (1, 3, 12, 25)]
    np.testing.assert_array_equal(got[rest], plain[rest])


@gpu
def test_singular_values_are_driven_to_one(dev):
    x = np.random.default_rng(5).standard_normal((96, 200)).astype(np.float32)
    s = np.linalg.svd(dev.read(dev.orthogonalize(dev.upload(x), 1, 96, 200)).reshape(96, 200),
                      compute_uv=False)
    assert 0.6 < s.min() and s.max() < 1.25  # the quintic's range around 1


@gpu
def test_degenerate_inputs(dev):
    run = lambda x: dev.read(dev.orthogonalize(dev.upload(x), 1, *x.shape)).reshape(x.shape)
    np.testing.assert_array_equal(run(np.zeros((40, 70), np.float32)), np.zeros((40, 70)))
    one = np.outer(np.arange(1, 41), np.linspace(-1, 1, 70)).astype(np.float32)  # rank 1
    assert _rel(run(one), _orthogonalize(one)) <= DEGENERATE
    tiny = np.random.default_rng(0).standard_normal((40, 70)).astype(np.float32) * np.float32(1e-30)
    assert _rel(run(tiny), _orthogonalize(tiny)) <= TOL
    big = np.random.default_rng(0).standard_normal((40, 70)).astype(np.float32) * np.float32(1e30)
    assert _rel(run(big), _orthogonalize(big)) <= TOL
    spike = np.zeros((70, 40), np.float32)
    spike[3, 5] = -2.0  # one entry of size 1 after scaling
    assert _rel(run(spike), _orthogonalize(spike)) <= DEGENERATE
    bad = np.ones((40, 70), np.float32)
    bad[1, 2] = np.nan
    assert np.isnan(run(bad)).all()
    assert dev.orthogonalize(dev.upload(np.zeros(0)), 0, 4, 4).len == 0
    assert dev.orthogonalize(dev.upload(np.zeros(0)), 2, 0, 4).len == 0


def _step(w, g, m, lr, mu, nesterov, wd, steps):
    w, g, m = (a.astype(np.float64) for a in (w, g, m))
    mu = float(np.float32(mu))
    m = mu * m + (1 - mu) * g
    u = (1 - mu) * g + mu * m if nesterov else m
    gain = lr * 0.2 * np.sqrt(max(w.shape))
    o = _orthogonalize(u, steps)
    return (1 - lr * wd) * w - gain * o, m, gain * np.linalg.norm(o)


@gpu
@pytest.mark.parametrize("rows,cols", [(40, 300), (300, 40), (200, 140)])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_nonfinite_matrix_stays_alone(dev, rows, cols, value):
    r = np.random.default_rng(9)
    x = np.stack([_gradient(r, rows, cols) for _ in range(3)])
    x[1, rows - 1, 3] = value
    got = dev.read(dev.orthogonalize(dev.upload(x), 3, rows, cols)).reshape(x.shape)
    assert np.isnan(got[1]).all()
    for i in (0, 2):
        assert _rel(got[i], _orthogonalize(x[i])) <= TOL


@gpu
@pytest.mark.parametrize("nesterov", [True, False])
def test_optimizer_steps(dev, nesterov):
    """Several steps over matrices of equal and different shapes in one call:
    |W error| <= 4 u (|W| + |update|) + TOL |update| a step, momentum 4 u a step."""
    from any_gpu import Muon
    r = np.random.default_rng(7)
    shapes = [(64, 96), (96, 64), (64, 96), (130, 33), (64, 64), (1, 50), (64, 96), (300, 260)]
    opt = Muon(lr=0.05, nesterov=nesterov, weight_decay=0.1)
    w = [r.standard_normal(s).astype(np.float32) for s in shapes]
    params = [dev.upload(a) for a in w]
    ref = [(a.astype(np.float64), np.zeros(a.shape)) for a in w]
    err = np.zeros(len(w))
    for step in range(3):
        g = [_gradient(r, *s) for s in shapes]
        opt.step(dev, params, [dev.upload(a) for a in g], shapes)
        for i, (wi, mi) in enumerate(ref):
            # each step from what the device holds, so errors do not add up
            base = w[i] if step == 0 else held[i][0]
            mom = mi if step == 0 else held[i][1]
            want, m, size = _step(base, g[i], mom, 0.05, 0.95, nesterov, 0.1, 5)
            got = dev.read(params[i]).reshape(want.shape)
            got_m = dev.read(opt.states[i]).reshape(want.shape)
            assert np.linalg.norm(got - want) <= (4 * U * (np.linalg.norm(want) + size)
                                                  + TOL * size)
            assert np.linalg.norm(got_m - m) <= 4 * U * (np.linalg.norm(m) + np.linalg.norm(g[i]))
        held = [(dev.read(p).reshape(s), dev.read(m).reshape(s))
                for p, m, s in zip(params, opt.states, shapes)]


@gpu
@pytest.mark.parametrize("small", [2, 40])
def test_optimizer_steps_over_all_kinds(dev, small):
    """Wide, square and small matrices in one call, and more small ones than fit
    beside the others."""
    from any_gpu import Muon
    r = np.random.default_rng(small)
    shapes = [(1024, 1600)] * 8 + [(300, 512), (513, 400)]
    tiny = [(48, 100), (100, 16), (120, 700)]
    shapes = (tiny * 20)[:small] + shapes
    w = [r.standard_normal(s).astype(np.float32) for s in shapes]
    g = [_gradient(r, *s) for s in shapes]
    params = [dev.upload(a) for a in w]
    Muon(lr=0.05).step(dev, params, [dev.upload(a) for a in g], shapes)
    for i in list(range(min(small, 6))) + [small - 1, small, small + 7, small + 8, small + 9]:
        want, _, size = _step(w[i], g[i], np.zeros(shapes[i]), 0.05, 0.95, True, 0.01, 5)
        bound = 4 * U * (np.linalg.norm(want) + size) + (SEGMENTS if i >= small else TOL) * size
        assert np.linalg.norm(dev.read(params[i]) - want.ravel()) <= bound


@gpu
@pytest.mark.parametrize("shapes", [[(50, 77), (128, 128)], [(200, 3001), (300, 260), (60, 70)],
                                    [(1024, 1540)] * 8])
def test_caller_memory_unaligned_stream_and_graph(dev, shapes):
    """Odd addresses, a caller's stream, and the same step replayed from two graphs."""
    import torch
    from any_gpu import muon_tensors
    r = np.random.default_rng(2)
    start = [[_gradient(r, *s) for s in shapes] for _ in range(3)]
    results = []
    for mode in ("eager", "graph"):
        hold = [[torch.cat([torch.zeros(1), torch.from_numpy(a).reshape(-1)]).cuda() for a in b]
                for b in start]
        ptr = lambda t: t.data_ptr() + 4
        tensors = muon_tensors([(ptr(p), ptr(g), ptr(m), *s)
                                for p, g, m, s in zip(*hold, shapes)])
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        call = lambda: dev.launch_muon(tensors, 0.02, 0.9, True, 0.0, 5, stream.cuda_stream)
        if mode == "eager":
            call()
            call()
        else:
            graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
            for graph in graphs:
                with torch.cuda.graph(graph, stream=stream):
                    call()
            with torch.cuda.stream(stream):
                for graph in graphs:
                    graph.replay()
        torch.cuda.synchronize()
        results.append(hold)
        assert all(t[0] == 0 for b in hold for t in b)
    for a, b in zip(*results):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    x = torch.from_numpy(start[0][0]).cuda()
    torch.cuda.synchronize()
    dev.launch_orthogonalize(x.data_ptr(), x.data_ptr(), 1, *shapes[0])  # in place
    dev.synchronize()
    assert _rel(x.cpu().numpy(), _orthogonalize(start[0][0])) <= TOL


@gpu
@pytest.mark.parametrize("shapes", [[(40, 30)] * 30, [(1024, 1600)] * 8])
def test_out_of_memory_steps_no_matrix(dev, shapes):
    """One matrix more, whose scratch (275 GB) no device has, in the batch behind the
    others': none of them is touched.  Its addresses are not memory; nothing reads them."""
    import torch
    from any_gpu import AnyGpuError, muon_tensors
    g = torch.Generator(device="cuda").manual_seed(1)
    p, u, m = ([torch.randn(s, generator=g, device="cuda") for s in shapes] for _ in range(3))
    held = [t.clone() for t in p + m]
    far = [(1 << 52, 1 << 53, 1 << 54, 2**17, 2**17)]
    own = [(a.data_ptr(), b.data_ptr(), c.data_ptr(), *a.shape) for a, b, c in zip(p, u, m)]
    torch.cuda.synchronize()
    with pytest.raises(AnyGpuError) as e:
        dev.launch_muon(muon_tensors(own + far), 0.02)
    assert e.value.status == 4
    dev.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(p + m, held))
    dev.launch_muon(muon_tensors(own), 0.02)
    dev.synchronize()
    assert not any(torch.equal(a, b) for a, b in zip(p + m, held))


@gpu
def test_batches_of_a_call_share_scratch(dev):
    """Small ones on chip, two batches in steps on the Gram matrix (one of them of a single
    matrix, columns dealt out) and two of the others, one after the other in the same
    scratch: eager, and from a graph replayed for the second step."""
    import torch
    from any_gpu import muon_tensors
    shapes = [(40, 70)] * 3 + [(512, 3000)] * 13 + [(300, 280)] * 25 + [(500, 40)]
    r = np.random.default_rng(6)
    start = [[_gradient(r, *s) for s in shapes] for _ in range(3)]
    results = []
    for graphed in (False, True):
        hold = [[torch.from_numpy(a).cuda() for a in b] for b in start]
        tensors = muon_tensors([(p.data_ptr(), g.data_ptr(), m.data_ptr(), *p.shape)
                                for p, g, m in zip(*hold)])
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        call = lambda: dev.launch_muon(tensors, 0.02, 0.9, True, 0.1, 5, stream.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        if graphed:
            with torch.cuda.graph(graph, stream=stream):
                call()
        for step in range(2):
            with torch.cuda.stream(stream):
                graph.replay() if graphed else call()
            torch.cuda.synchronize()
            if step == 0 and not graphed:
                for i in (0, 3, 15, 16, 39, 40, 41):
                    want, _, size = _step(start[0][i], start[1][i], start[2][i], 0.02, 0.9, True,
                                          0.1, 5)
                    bound = (4 * U * (np.linalg.norm(want) + size)
                             + (SEGMENTS if 3 <= i < 16 else TOL) * size)
                    assert np.linalg.norm(hold[0][i].cpu().numpy() - want) <= bound
        results.append(hold)
    for a, b in zip(*results):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@gpu
def test_precision_mode_does_not_matter(dev):
    x = dev.upload(_gradient(np.random.default_rng(0), 256, 384))
    want = dev.read(dev.orthogonalize(x, 1, 256, 384))
    for mode in ("tf32", "tf32x3", "ffma"):
        with dev.precision(mode):
            np.testing.assert_array_equal(dev.read(dev.orthogonalize(x, 1, 256, 384)), want)


@gpu
def test_buffer_layer_refusals(dev):
    from any_gpu import AnyGpuError, Muon

    def status(call):
        with pytest.raises(AnyGpuError) as e:
            call()
        return e.value.status
    x, y = dev.upload(np.ones(12)), dev.upload(np.ones(12))
    assert status(lambda: dev.orthogonalize(x, 1, 3, 5)) == 1
    assert status(lambda: dev.orthogonalize(x, 1, 3, 4, 0)) == 2
    assert status(lambda: dev.orthogonalize(dev.upload_i32(np.ones(12, int)), 1, 3, 4)) == 2
    assert status(lambda: Muon(0.1).step(dev, [x], [y], [(3, 5)])) == 1
    assert status(lambda: Muon(0.1).step(dev, [x, x], [y, y], [(3, 4), (3, 4)])) == 2  # twice
    assert status(lambda: Muon(0.1).step(dev, [x], [x], [(3, 4)])) == 2
    assert status(lambda: Muon(0.1).step(dev, [x], [y, y], [(3, 4)])) == 1
    np.testing.assert_array_equal(dev.read(x), np.ones(12))


def test_launch_layer_refusals():
    """Arguments are checked before the device: no GPU is needed to be refused."""
    from any_gpu import _lib, muon_tensors
    lib = _lib.load()
    f, p = C.c_float, C.c_void_p(1 << 20)

    def step(tensors=((1 << 20, 1 << 30, 1 << 24, 8, 8),), lr=0.1, mu=0.9, wd=0.0, steps=5):
        t = muon_tensors(list(tensors))
        return lib.agpu_launch_muon(None, C.addressof(t), len(t), f(lr), f(mu), 1, f(wd), steps,
                                    None)
    assert step(steps=0) == 2 and step(steps=65) == 2
    assert step(mu=1.0) == 2 and step(mu=-0.1) == 2 and step(mu=float("nan")) == 2
    assert step(lr=float("inf")) == 2 and step(wd=float("nan")) == 2
    assert step(tensors=[(0, 1 << 30, 1 << 24, 8, 8)]) == 2
    assert step(tensors=[(1 << 20, 0, 1 << 24, 8, 8)]) == 2
    assert step(tensors=[(1 << 20, 1 << 30, 1 << 24, 2**31, 8)]) == 7
    share = [(1 << 20, 1 << 30, 1 << 24, 8, 8), ((1 << 20) + 252, 1 << 30, 1 << 25, 8, 8)]
    assert step(tensors=share) == 2 and b"share memory" in lib.agpu_last_error_message()
    assert step(tensors=[(1 << 20, 1 << 30, 1 << 20, 8, 8)]) == 2  # momentum is the parameter
    for grad in (1 << 20, (1 << 20) + 252, (1 << 20) - 252, (1 << 24) + 8, (1 << 20) - 1024):
        pair = [(1 << 20, 1 << 30, 1 << 24, 8, 8), (1 << 21, grad, 1 << 25, 32, 32)]
        assert step(tensors=pair) == 2 and b"gradient 1 shares" in lib.agpu_last_error_message()
    free = [(1 << 20, 1 << 30, 1 << 24, 8, 8), (1 << 21, (1 << 20) + 256, 1 << 25, 8, 8)]
    assert step(tensors=free) == 2 and b"NULL device" in lib.agpu_last_error_message()
    assert step() == 2 and b"NULL device" in lib.agpu_last_error_message()
    orth = lambda *a: lib.agpu_launch_orthogonalize(None, *a, None)
    assert orth(p, p, 1, 8, 8, 0) == 2
    assert orth(None, p, 1, 8, 8, 5) == 2 and orth(p, None, 1, 8, 8, 5) == 2
    assert orth(p, p, 1, 2**31, 1, 5) == 7
    assert orth(p, p, 16, 2**30, 2**30, 5) == 7  # 2^64 elements
    assert orth(p, p, 2**31, 2**10, 1, 5) == 7
    assert orth(p, p, 1, 8, 8, 5) == 2 and b"NULL device" in lib.agpu_last_error_message()


def test_orthogonalize_refuses_an_output_across_its_input():
    """Matrices are worked on side by side: only the same place is safe."""
    from any_gpu import _lib
    lib = _lib.load()

    def status(x, out, batch=2):
        return lib.agpu_launch_orthogonalize(None, C.c_void_p(x), C.c_void_p(out), batch, 8, 8, 5,
                                             None)
    x, size = 1 << 20, 2 * 8 * 8 * 4
    for out in (x + 4, x - 4, x + size // 2, x + size - 4, x - size + 4):
        assert status(x, out) == 2 and b"overlaps" in lib.agpu_last_error_message()
    for out in (x, x + size, x - size):
        assert status(x, out) == 2 and b"NULL device" in lib.agpu_last_error_message()
    assert status(x, x + 4, 0) == 2 and b"NULL device" in lib.agpu_last_error_message()


def test_outcomes_of_bounded_waits_are_used():
    """No kernel goes on as if a wait had succeeded: a statement that drops the outcome of
    mbar_wait may only be a drain (no abort flag), and none that was collected is dropped.
    By the source, since no call makes a tensor core stop."""
    from pathlib import Path
    import re
    csrc = Path(__file__).resolve().parents[1] / "any-gpu_b200" / "csrc"
    text = (csrc / "muon_small.cuh").read_text() + (csrc / "muon_gemm.cuh").read_text()
    dropped = re.findall(r"[;{})]\s*ptx::mbar_wait\w*(?:<\w+>)?\(([^;]*)\);", text)
    assert dropped and all(d.split(",")[-1].strip() == "nullptr" for d in dropped), dropped
    assert "(void)ok" not in text
    assert re.search(r"if \(!__all_sync\(0xffffffffu, ok\)\) break;[^}]*update_block", text)


def test_iteration_of_the_reference():
    """The float64 iteration the GPU tests compare with, against its closed form on the
    singular values."""
    x = np.random.default_rng(1).standard_normal((6, 9))
    u, s, vt = np.linalg.svd(x / np.linalg.norm(x), full_matrices=False)
    for _ in range(5):
        s = A * s + B * s ** 3 + CC * s ** 5
    assert np.abs(_orthogonalize(x) - (u * s) @ vt).max() <= 1e-12
    assert np.abs(_orthogonalize(x.T) - ((u * s) @ vt).T).max() <= 1e-12
