"""int32 buffers (token ids, positions) are no floats: every op on f32 data refuses
them, whichever operand they are."""
from __future__ import annotations

import ctypes as C
import re

import numpy as np
import pytest

from conftest import ROOT

COPIES = {"agpu_read", "agpu_write", "agpu_read_async", "agpu_write_async"}
# operands without elements here, or of either kind: refused in their own tests
OTHERS = {"agpu_embedding", "agpu_embedding_backward", "agpu_qk_norm_rope_forward",
          "agpu_qk_norm_rope_backward"}


def _ops():
    """{name: [(type, parameter)]} of the header's ops with a device and buffers."""
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "agpu.h").read_text(), flags=re.S)
    ops = {}
    for name, params in re.findall(r"AGPU_API\s+agpu_status\s+(agpu_\w+)\s*\(([^;]*?)\)\s*;", text):
        params = [p.strip().rsplit(None, 1) for p in " ".join(params.split()).split(",")]
        params = [(t.replace("const", "").strip(), n) for t, n in params]
        if ("agpu_device*", "dev") in params and any(t == "agpu_buffer*" for t, _ in params):
            ops[name] = params
    return {n: p for n, p in ops.items() if n not in COPIES | OTHERS}


CASES = [(n, i) for n, p in _ops().items() for i, (t, _) in enumerate(p) if t == "agpu_buffer*"]


def test_the_header_is_understood():
    ops = {n for n, _ in CASES}
    assert {"agpu_add", "agpu_gemm_ex", "agpu_conv2d", "agpu_mse_loss", "agpu_sdpa_backward",
            "agpu_group_norm_backward", "agpu_orthogonalize", "agpu_transpose"} <= ops
    assert len(ops) >= 40 and ("agpu_conv2d", 3) in CASES  # its bias


@pytest.mark.gpu
@pytest.mark.parametrize("name,at", CASES, ids=[f"{n}-{i}" for n, i in CASES])
def test_refused_as_floats(dev, name, at):
    """One element everywhere, no padding: only the kind of one operand is wrong."""
    from any_gpu import _lib
    lib = _lib.load()
    ids, x = dev.upload_i32([1]), dev.upload([1.0])
    outs, args = [], []
    for i, (kind, param) in enumerate(_ops()[name]):
        if kind == "agpu_device*":
            args.append(dev.handle)
        elif kind == "agpu_buffer*":
            args.append((ids if i == at else x).handle)
        elif kind == "agpu_buffer**":
            outs.append(C.c_void_p())
            args.append(C.byref(outs[-1]))
        elif kind == "float":
            args.append(C.c_float(1))
        elif kind == "int" or "pad" in param or param in ("ph", "pw", "slice_offset"):
            args.append(0)
        else:
            assert kind in ("uint32_t", "uint64_t"), (kind, param)
            args.append(1)
    assert getattr(lib, name)(*args) == 2, name
    assert b"f32 buffer" in lib.agpu_last_error_message()
    assert all(not o.value for o in outs)


@pytest.mark.gpu
def test_read_and_write_keep_the_values(dev):
    """New ids in an existing buffer, and ids read back: integers, not a float's bits."""
    table, ids = dev.upload(np.arange(12.0)), dev.upload_i32([2, 0])
    got = dev.read(ids)
    assert got.dtype == np.int32 and got.tolist() == [2, 0]
    dev.write(ids, [1, -1])
    assert dev.read(ids).tolist() == [1, -1]
    np.testing.assert_array_equal(dev.read(dev.embedding(table, ids, 2, 3, 4)),
                                  [4, 5, 6, 7, 0, 0, 0, 0])
    with pytest.raises(TypeError):
        dev.write(ids, [1.0, 2.0])
    with pytest.raises(OverflowError):
        dev.write(ids, [0, 2**31])
    assert dev.read(ids).tolist() == [1, -1]


@pytest.mark.gpu
def test_refused_by_the_optimisers(dev):
    from any_gpu import AdamW, AnyGpuError, Muon
    ids, x, y = dev.upload_i32([1, 2]), dev.upload([1, 2]), dev.upload([3, 4])
    for p, g in ((ids, x), (x, ids)):
        for step in (lambda: AdamW(0.1).step(dev, [p], [g]),
                     lambda: Muon(0.1).step(dev, [p], [g], [(1, 2)])):
            with pytest.raises(AnyGpuError) as e:
                step()
            assert e.value.status == 2
    np.testing.assert_array_equal(dev.read(x), [1, 2])
