"""Token embedding and its gradient against numpy in float64.

Tolerances.  The lookup is one product per element, so it equals float32
numpy exactly.  A gradient element is a sum of L float32 terms (any order:
at most (L - 1) u relative to the sum of magnitudes, u = 2^-24), a product
with the scale and, when accumulating, one more sum: (L + 2) u times the sum of
all magnitudes bounds it."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

U = 2.0 ** -24
gpu = pytest.mark.gpu


def _ids(r, tokens, vocab, kind):
    if kind == "same":
        return np.full(tokens, vocab // 2, np.int32)
    if kind == "padding":
        return np.full(tokens, -1, np.int32)
    if kind == "ends":
        return r.choice([0, vocab - 1, -1], tokens).astype(np.int32)
    ids = np.minimum((vocab ** r.random(tokens)).astype(np.int64) - 1, vocab - 1)  # like text
    ids[r.random(tokens) < 0.05] = -1
    return ids.astype(np.int32)


def _gradient(grad, ids, vocab, scale, start=None):
    """(float64 gradient, its elementwise error bound)."""
    dim = grad.shape[1]
    total, mag = np.zeros((vocab, dim)), np.zeros((vocab, dim))
    live = ids >= 0
    np.add.at(total, ids[live], grad[live].astype(np.float64))
    np.add.at(mag, ids[live], np.abs(grad[live]).astype(np.float64))
    count = np.bincount(ids[live], minlength=vocab)[:, None]
    total, mag = total * float(np.float32(scale)), mag * abs(scale)
    if start is not None:
        total, mag = total + start, mag + np.abs(start)
    return total, (count + 2) * U * mag


CASES = [(1, 1, 1), (1, 7, 4), (5, 33, 3), (31, 100, 64), (32, 100, 64), (33, 100, 65),
         (64, 31, 99), (65, 1001, 128), (300, 1000, 256), (1000, 777, 1028), (4097, 5000, 36),
         (20000, 300, 20), (20, 400000, 4), (128, 310000, 3), (129, 310000, 3),
         (256, 600, 512), (257, 600, 512), (255, 9400, 99)]


@gpu
@pytest.mark.parametrize("tokens,vocab,dim", CASES)
def test_lookup(dev, tokens, vocab, dim):
    r = np.random.default_rng(tokens + dim)
    table = r.standard_normal((vocab, dim)).astype(np.float32)
    ids = _ids(r, tokens, vocab, "text")
    for scale in (1.0, -3.7):
        got = dev.read(dev.embedding(dev.upload(table), dev.upload_i32(ids), tokens, vocab, dim,
                                     scale)).reshape(tokens, dim)
        want = np.where((ids >= 0)[:, None], table[np.maximum(ids, 0)], 0) * np.float32(scale)
        np.testing.assert_array_equal(got, want)


@gpu
@pytest.mark.parametrize("kind", ["text", "same", "padding", "ends"])
@pytest.mark.parametrize("tokens,vocab,dim", CASES)
def test_gradient(dev, tokens, vocab, dim, kind):
    r = np.random.default_rng(tokens + dim)
    grad = r.standard_normal((tokens, dim)).astype(np.float32)
    ids = _ids(r, tokens, vocab, kind)
    G, I = dev.upload(grad), dev.upload_i32(ids)
    got = dev.read(dev.embedding_backward(G, I, tokens, vocab, dim, 2.5))
    want, tol = _gradient(grad, ids, vocab, 2.5)
    assert (np.abs(got.reshape(vocab, dim) - want) <= tol).all()
    again = dev.read(dev.embedding_backward(G, I, tokens, vocab, dim, 2.5))
    np.testing.assert_array_equal(got, again)  # fixed order of every sum
    start = r.standard_normal((vocab, dim)).astype(np.float32)
    acc = dev.upload(start)
    dev.launch_embedding_backward(G.device_ptr, I.device_ptr, acc.device_ptr, tokens, vocab, dim,
                                  2.5, accumulate=True)
    want, tol = _gradient(grad, ids, vocab, 2.5, start)
    got = dev.read(acc).reshape(vocab, dim)
    assert (np.abs(got - want) <= tol).all()
    untouched = np.setdiff1d(np.arange(vocab), ids)
    np.testing.assert_array_equal(got[untouched], start[untouched])


@gpu
def test_gradient_long_rows(dev):
    """Rows whose tokens span many chunks, and a row that begins and ends at one's border."""
    r = np.random.default_rng(0)
    counts = [64, 32, 33, 31, 1, 4000, 0, 95, 1]
    ids = np.repeat(np.arange(len(counts)), counts).astype(np.int32)
    r.shuffle(ids)
    dim, vocab = 260, len(counts)
    grad = r.standard_normal((ids.size, dim)).astype(np.float32)
    got = dev.read(dev.embedding_backward(dev.upload(grad), dev.upload_i32(ids), ids.size, vocab,
                                          dim)).reshape(vocab, dim)
    want, tol = _gradient(grad, ids, vocab, 1.0)
    assert (np.abs(got - want) <= tol).all()


@gpu
def test_no_tokens_and_empty_sizes(dev):
    none = dev.upload_i32(np.zeros(0, np.int32))
    empty = dev.upload(np.zeros(0, np.float32))
    assert dev.embedding(dev.upload(np.ones(12)), none, 0, 3, 4).len == 0
    np.testing.assert_array_equal(dev.read(dev.embedding_backward(empty, none, 0, 3, 4)),
                                  np.zeros(12))
    acc = dev.upload(np.ones(12))
    dev.launch_embedding_backward(0, 0, acc.device_ptr, 0, 3, 4, accumulate=True)
    np.testing.assert_array_equal(dev.read(acc), np.ones(12))
    assert dev.embedding_backward(empty, none, 0, 0, 4).len == 0
    ids = dev.upload_i32([0, 1])
    assert dev.embedding(empty, ids, 2, 3, 0).len == 0


@gpu
def test_nonfinite_rows_stay_in_their_row(dev):
    table = np.ones((4, 8), np.float32)
    table[2] = np.nan
    table[3] = np.inf
    got = dev.read(dev.embedding(dev.upload(table), dev.upload_i32([0, -1, 2, 3]), 4, 4, 8))
    got = got.reshape(4, 8)
    assert (got[0] == 1).all() and (got[1] == 0).all()
    assert np.isnan(got[2]).all() and np.isposinf(got[3]).all()
    grad = np.ones((4, 8), np.float32)
    grad[1] = np.nan  # padding's gradient goes nowhere
    d = dev.read(dev.embedding_backward(dev.upload(grad), dev.upload_i32([0, -1, 2, 2]), 4, 4, 8))
    np.testing.assert_array_equal(d.reshape(4, 8)[:, 0], [1, 0, 2, 0])


@gpu
@pytest.mark.parametrize("bad", [5, -2, 2**31 - 1, -2**31])
def test_bad_id_is_reported_and_counts_as_padding(dev, bad):
    from any_gpu import AnyGpuError
    table, ids = dev.upload(np.ones(40)), dev.upload_i32([1, bad, 4])
    out = dev.embedding(table, ids, 3, 5, 8)
    with pytest.raises(AnyGpuError) as e:
        dev.synchronize()
    assert e.value.status == 2
    np.testing.assert_array_equal(dev.read(out).reshape(3, 8)[:, 0], [1, 0, 1])
    d = dev.embedding_backward(dev.upload(np.ones(24)), ids, 3, 5, 8)
    with pytest.raises(AnyGpuError) as e:
        dev.synchronize()
    assert e.value.status == 2
    np.testing.assert_array_equal(dev.read(d).reshape(5, 8)[:, 0], [0, 1, 0, 0, 1])


@gpu
@pytest.mark.parametrize("tokens", [3, 300])  # one launch, and sorted
def test_bad_id_does_not_hide_an_expired_wait(dev, tokens):
    """A bad id before a wait that runs out: both are reported, the wait first."""
    from any_gpu import AnyGpuError
    dev.synchronize()
    ids = dev.upload_i32([7] + [1] * (tokens - 1))
    dev.embedding(dev.upload(np.ones(40)), ids, tokens, 5, 8)
    dev.embedding_backward(dev.upload(np.ones(8 * tokens)), ids, tokens, 5, 8)
    dev.selftest_wait_timeout(300)
    for status, code in ((6, "0x7e57"), (2, "0x7091")):
        with pytest.raises(AnyGpuError) as e:
            dev.synchronize()
        assert e.value.status == status and code in str(e.value)
    dev.synchronize()


@gpu
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_unaligned_pointers_on_a_callers_stream(dev, shift):
    import torch
    tokens, vocab, dim = 70, 50, 64
    r = np.random.default_rng(shift)
    table = r.standard_normal((vocab, dim)).astype(np.float32)
    grad = r.standard_normal((tokens, dim)).astype(np.float32)
    ids = _ids(r, tokens, vocab, "text")
    at = lambda a: torch.cat([torch.zeros(shift), torch.from_numpy(a).reshape(-1)]).cuda()
    T, G, I = at(table), at(grad), torch.from_numpy(ids).cuda()
    out, d = torch.full((tokens * dim + shift,), 7.0).cuda(), torch.full((vocab * dim + shift,),
                                                                         7.0).cuda()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    ptr = lambda t: t.data_ptr() + 4 * shift
    dev.launch_embedding(ptr(T), I.data_ptr(), ptr(out), tokens, vocab, dim, 1.0,
                         stream.cuda_stream)
    dev.launch_embedding_backward(ptr(G), I.data_ptr(), ptr(d), tokens, vocab, dim, 1.0, False,
                                  stream.cuda_stream)
    stream.synchronize()
    assert (out[:shift] == 7).all() and (d[:shift] == 7).all()
    want = np.where((ids >= 0)[:, None], table[np.maximum(ids, 0)], 0)
    np.testing.assert_array_equal(out[shift:].cpu().numpy().reshape(tokens, dim), want)
    want, tol = _gradient(grad, ids, vocab, 1.0)
    assert (np.abs(d[shift:].cpu().numpy().reshape(vocab, dim) - want) <= tol).all()


@gpu
def test_captured_graphs_replay_with_new_ids(dev):
    """Two graphs of the same call, replayed in turn with other inputs."""
    import torch
    tokens, vocab, dim = 200, 90, 32
    r = np.random.default_rng(3)
    stream = torch.cuda.Stream()
    G = torch.zeros(tokens, dim, device="cuda")
    I = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    outs, graphs = [], []
    for _ in range(2):
        d = torch.zeros(vocab, dim, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            dev.launch_embedding_backward(G.data_ptr(), I.data_ptr(), d.data_ptr(), tokens, vocab,
                                          dim, 1.0, False, stream.cuda_stream)
        outs.append(d)
        graphs.append(graph)
    for _ in range(3):
        grad = r.standard_normal((tokens, dim)).astype(np.float32)
        ids = _ids(r, tokens, vocab, "text")
        G.copy_(torch.from_numpy(grad))
        I.copy_(torch.from_numpy(ids))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for graph in graphs:
                graph.replay()
        torch.cuda.synchronize()
        want, tol = _gradient(grad, ids, vocab, 1.0)
        for d in outs:
            assert (np.abs(d.cpu().numpy() - want) <= tol).all()


@gpu
def test_offsets_past_32_bits(dev):
    """A table of more than 2^32 elements: rows at its far end."""
    import torch
    vocab, dim, tokens = 1050000, 4100, 40
    if torch.cuda.mem_get_info()[0] < 24e9:
        pytest.skip("needs 24 GB")
    table = torch.empty(vocab, dim, device="cuda")
    table[-50:] = torch.arange(50.0, device="cuda")[:, None]
    ids = torch.randint(vocab - 50, vocab, (tokens,), dtype=torch.int32, device="cuda")
    out = torch.empty(tokens, dim, device="cuda")
    torch.cuda.synchronize()
    dev.launch_embedding(table.data_ptr(), ids.data_ptr(), out.data_ptr(), tokens, vocab, dim)
    dev.synchronize()
    assert (out == (ids - (vocab - 50)).float()[:, None]).all()
    dev.launch_embedding_backward(out.data_ptr(), ids.data_ptr(), table.data_ptr(), tokens, vocab,
                                  dim)
    dev.synchronize()
    want = torch.zeros(50, dim, device="cuda").index_add_(0, (ids - (vocab - 50)).long(), out)
    assert (table[-50:] == want).all()  # sums of small integers: exact in any order
    assert not table[:1000].any() and not table[vocab // 2:vocab // 2 + 1000].any()


@gpu
def test_buffer_layer_refusals(dev):
    from any_gpu import AnyGpuError

    def status(call):
        with pytest.raises(AnyGpuError) as e:
            call()
        return e.value.status
    table, ids, grad = dev.upload(np.ones(20)), dev.upload_i32([0, 1, 2]), dev.upload(np.ones(12))
    assert status(lambda: dev.embedding(table, ids, 3, 5, 5)) == 1     # table length
    assert status(lambda: dev.embedding(table, ids, 4, 5, 4)) == 1     # ids length
    assert status(lambda: dev.embedding(table, dev.upload(np.ones(3)), 3, 5, 4)) == 2  # f32 ids
    assert status(lambda: dev.embedding(dev.upload_i32(np.ones(20, int)), ids, 3, 5, 4)) == 2
    assert status(lambda: dev.embedding_backward(grad, ids, 3, 5, 5)) == 1
    assert status(lambda: dev.embedding_backward(grad, dev.upload(np.ones(3)), 3, 5, 4)) == 2
    dev.synchronize()


def test_launch_layer_refusals():
    """Arguments are checked before the device: no GPU is needed to be refused."""
    from any_gpu import _lib
    lib = _lib.load()
    f, p = C.c_float(1), C.c_void_p(256)
    look = lambda *a: lib.agpu_launch_embedding(None, *a, f, None)
    back = lambda *a: lib.agpu_launch_embedding_backward(None, *a, f, 0, None)
    for call in (look, back):
        assert call(p, p, p, 3, 0, 4) == 2          # tokens without a table
        assert call(p, p, p, 2**31, 5, 4) == 7
        assert call(p, p, p, 3, 2**32 - 1, 4) == 7
        assert call(p, p, p, 3, 5, 2**30) == 7
        assert call(None, p, p, 3, 5, 4) == 2
        assert call(p, None, p, 3, 5, 4) == 2
        assert call(p, p, None, 3, 5, 4) == 2
        assert call(p, p, p, 3, 5, 4) == 2 and b"NULL device" in lib.agpu_last_error_message()
    out = C.c_void_p()
    assert lib.agpu_embedding(None, None, None, 1, 1, 1, f, None) == 2
    assert lib.agpu_embedding(None, None, None, 1, 1, 1, f, C.byref(out)) == 2
    assert lib.agpu_embedding_backward(None, None, None, 1, 1, 1, f, C.byref(out)) == 2
    assert lib.agpu_upload_i32(None, None, 1, C.byref(out)) == 2


def test_most_tokens_of_the_gradient():
    """The gradient's 32-bit positions hold 2^31 - 256 tokens; the lookup's are 64-bit."""
    from any_gpu import _lib
    lib = _lib.load()
    f, p, out = C.c_float(1), C.c_void_p(256), C.c_void_p()
    look = lambda n: lib.agpu_launch_embedding(None, p, p, p, n, 5, 1, f, None)
    back = lambda n: lib.agpu_launch_embedding_backward(None, p, p, p, n, 5, 1, f, 0, None)
    most = 2**31 - 256
    assert back(most) == 2 and b"NULL device" in lib.agpu_last_error_message()
    assert back(most + 1) == 7 and back(2**31 - 32) == 7 and back(2**31 - 1) == 7
    assert lib.agpu_embedding_backward(None, None, None, most + 1, 5, 1, f, C.byref(out)) == 7
    assert look(2**31 - 1) == 2 and b"NULL device" in lib.agpu_last_error_message()


def test_positions_of_the_sort_stay_in_an_int():
    """The sorting kernel's position arithmetic in Python integers, for the most tokens
    the call takes: per warp, the last ids read by the last lane."""
    warps, ahead, most = 32, 8, 2**31 - 256
    for tokens in (most, most - 1, most - 31, most - 32 * ahead * warps):
        assert tokens + warps - 1 < 2**31
        per = ((tokens + warps - 1) // warps + 31) // 32 * 32
        end = 0
        for warp in range(warps):
            begin, last = end, min(tokens, (warp + 1) * per)
            assert begin == min(tokens, warp * per) and last >= begin
            end = last
            if end > begin:
                for i0 in (begin + lane + (end - 1 - begin - lane) // (32 * ahead) * 32 * ahead
                           for lane in range(32) if begin + lane < end):
                    assert i0 < end and i0 + 32 * ahead < 2**31  # the step behind the last one
        assert end == tokens


def test_formula_against_differences():
    """The gradient the GPU tests compare with, against differences of the lookup (linear)."""
    r = np.random.default_rng(0)
    ids = np.array([2, 0, -1, 2, 3], np.int32)
    grad, table = r.standard_normal((5, 3)), r.standard_normal((4, 3))
    loss = lambda t: float((np.where((ids >= 0)[:, None], t[np.maximum(ids, 0)], 0) * grad).sum())
    want, _ = _gradient(grad.astype(np.float32), ids, 4, 1.0)
    for v in range(4):
        for c in range(3):
            t = table.copy()
            t[v, c] += 1
            # linear: exact but for rounding of ~60 operations in float64 and grad's cast
            assert abs((loss(t) - loss(table)) - want[v, c]) <= 1e-6
