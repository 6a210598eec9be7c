"""Operators for training a language model, as measured cases.

    embedding           out[t] = scale * table[ids[t]]; id -1 is padding (a zero row)
    embedding_grad      d_table[v] (+)= scale * sum of grad_out[t] over the tokens t with id v
    qk_norm_rope        RMS norm of every query and key head, then the rotary embedding
    qk_norm_rope_grad   its gradients: queries, keys and the two norm weights
    orthogonalize       Newton-Schulz iteration X <- aX + (bA + cA^2) X, A = X X^T
    muon_step           momentum, orthogonalised update, decoupled weight decay, in place

Each has a plain form in elementary torch operations (`own` false), the
framework's call (`own` true) and its definition in 64 bits (`exact`).
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

# coefficients of the quintic Newton-Schulz iteration
NS = (3.4445, -4.7750, 2.0315)
NORM_FLOOR = 1e-30


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # one decoding step of a batch of 8 sequences: latency
        {"name": "embedding_decode", "op": "embedding", "tokens": 8, "vocab": 32000, "dim": 4096,
         "scale": 1.0},
        # a training batch of 16 sequences of 2048
        {"name": "embedding_train", "op": "embedding", "tokens": 32768, "vocab": 64000,
         "dim": 2048, "scale": math.sqrt(2048.0)},
        # a short sequence into a small table, odd sizes
        {"name": "embedding_grad_short", "op": "embedding_grad", "tokens": 37, "vocab": 1001,
         "dim": 99, "scale": 1.0, "accumulate": False},
        # the layer benchmark's batch 2 x 2048, d_model 4096: a fresh gradient buffer
        {"name": "embedding_grad_layer", "op": "embedding_grad", "tokens": 4096, "vocab": 32000,
         "dim": 4096, "scale": 1.0, "accumulate": False},
        # a long micro-batch added to the gradient of the ones before it
        {"name": "embedding_grad_long", "op": "embedding_grad", "tokens": 65536, "vocab": 100000,
         "dim": 1024, "scale": 32.0, "accumulate": True},
        # one new token of 16 sequences far into their contexts, shared key heads
        {"name": "qk_decode", "op": "qk_norm_rope", "batch": 16, "seq": 1, "q_heads": 32,
         "k_heads": 8, "dim": 128, "rot_dim": 128, "base": 500000.0, "far": 100000,
         "given": True, "head_major": False},
        # the layer benchmark's batch 2 x 2048, packed projection, 32 heads of 128
        {"name": "qk_prefill", "op": "qk_norm_rope", "batch": 2, "seq": 2048, "q_heads": 32,
         "k_heads": 32, "dim": 128, "rot_dim": 128, "base": 10000.0, "far": 0,
         "given": False, "head_major": False},
        # ragged small training batch, half of each head rotated
        {"name": "qk_grad_odd", "op": "qk_norm_rope_grad", "batch": 3, "seq": 77, "q_heads": 6,
         "k_heads": 2, "dim": 80, "rot_dim": 40, "base": 10000.0, "far": 1000,
         "given": True, "head_major": True},
        # a training batch with shared key heads, outputs laid out for attention
        {"name": "qk_grad_train", "op": "qk_norm_rope_grad", "batch": 4, "seq": 2048,
         "q_heads": 32, "k_heads": 8, "dim": 128, "rot_dim": 128, "base": 10000.0, "far": 0,
         "given": False, "head_major": True},
        # one small matrix: latency
        {"name": "orthogonalize_small", "op": "orthogonalize", "batch": 1, "rows": 64,
         "cols": 256, "steps": 5},
        # the matrices of one small layer, one of them odd
        {"name": "muon_small_layer", "op": "muon_step",
         "shapes": "1024x1024,1024x1024,1024x1024,1024x1024,1024x2816,1024x2816,2816x1024,"
                   "1000x333", "steps": 5, "nesterov": True},
        # the layer benchmark's matrices: packed qkv, output, packed gate/up, down projections
        {"name": "muon_layer", "op": "muon_step",
         "shapes": "4096x12288,4096x4096,4096x22016,11008x4096", "steps": 5, "nesterov": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embedding", "embedding_grad", "qk_norm_rope", "qk_norm_rope_grad",
                     "orthogonalize", "muon_step"])
    if op in ("embedding", "embedding_grad"):
        vocab, dim = _log_int(rng, 300, 100000), _log_int(rng, 33, 4096)
        if rng.random() < 0.6:
            dim = max(32, dim // 64 * 64)
        tokens = _log_int(rng, 1, 65536)
        while tokens * dim > 65536 * 1024 or vocab * dim > 32000 * 4096:
            tokens, vocab = max(1, tokens // 2), max(300, vocab // 2)
        case = {"op": op, "tokens": tokens, "vocab": vocab, "dim": dim,
                "scale": rng.choice([1.0, round(math.sqrt(dim), 4)])}
        if op == "embedding_grad":
            case["accumulate"] = rng.random() < 0.3
        return case
    if op in ("qk_norm_rope", "qk_norm_rope_grad"):
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256, 50])
        k_heads = rng.choice([1, 2, 3, 4, 8])
        q_heads = k_heads * rng.choice([1, 1, 2, 4, 5, 8])
        while (q_heads + k_heads) * dim > 64 * 128:
            q_heads, k_heads = max(1, q_heads // 2), max(1, k_heads // 2)
        rows = _log_int(rng, 1, 4 * 2048)
        batch = rng.choice([1, 1, 2, 4, 7])
        case = {"op": op, "batch": batch, "seq": max(1, rows // batch), "q_heads": q_heads,
                "k_heads": k_heads, "dim": dim,
                "rot_dim": dim if rng.random() < 0.7 else dim // 4 * 2,
                "base": rng.choice([10000.0, 500000.0]), "far": rng.choice([0, 1000, 100000]),
                "given": False, "head_major": rng.random() < 0.5}
        case["given"] = case["far"] > 0 or rng.random() < 0.3
        return case
    steps = rng.choice([5, 5, 5, 3, 6])
    if op == "orthogonalize":
        rows, cols = _log_int(rng, 17, 4096), _log_int(rng, 17, 8192)
        batch = rng.choice([1, 1, 2, 3, 8])
        while batch > 1 and batch * rows * cols > 4096 * 8192:
            batch //= 2
        return {"op": op, "batch": batch, "rows": rows, "cols": cols, "steps": steps}
    shapes = []
    for _ in range(rng.randint(1, 5)):
        rows = _log_int(rng, 32, 4096)
        shapes.append((rows, max(32, int(rows * rng.choice([1, 1, 1, 1.5, 2.75, 0.25])))))
    if rng.random() < 0.5:
        shapes += [shapes[0]] * rng.randint(1, 3)
    return {"op": op, "shapes": ",".join("%dx%d" % s for s in shapes), "steps": steps,
            "nesterov": rng.random() < 0.7}


# ------------------------------------------------------------------ inputs --
def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ids(g, tokens, vocab):
    """Token ids with the frequencies of text: P(id) ~ 1 / (id + 1), the last 1/32 padding."""
    u = torch.rand(tokens, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab)) - 1).floor().clamp(0, vocab - 1).to(torch.int32)
    if tokens // 32:
        ids[-(tokens // 32):] = -1
    return ids


def _gradient(g, batch, rows, cols):
    """A matrix like a layer's gradient: a decaying spectrum on top of noise."""
    r = max(1, min(rows, cols, 32))
    scale = 0.8 ** torch.arange(r, device="cuda", dtype=torch.float32)
    x = (_randn(g, batch, rows, r) * scale) @ _randn(g, batch, r, cols)
    return (x + 0.5 * _randn(g, batch, rows, cols)).mul_(1e-3)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = {"case": dict(case)}
    if op in ("embedding", "embedding_grad"):
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        s["ids"] = _ids(g, t, v)
        if op == "embedding":
            s["table"] = _randn(g, v, d).mul_(0.02)
            s["out"] = torch.empty(t, d, device="cuda")
        else:
            s["grad_out"] = _randn(g, t, d).mul_(1e-2)
            s["d_table"] = (_randn(g, v, d).mul_(1e-2) if case["accumulate"]
                            else torch.empty(v, d, device="cuda"))
    elif op in ("qk_norm_rope", "qk_norm_rope_grad"):
        b, n, hq, hk, d = (case[k] for k in ("batch", "seq", "q_heads", "k_heads", "dim"))
        # a packed projection [batch, seq, (hq + 2 hk) * dim]: queries, keys, values
        s["qkv"] = _randn(g, b, n, hq + 2 * hk, d)
        s["q_weight"] = 1 + 0.1 * _randn(g, d)
        s["k_weight"] = 1 + 0.1 * _randn(g, d)
        s["positions"] = None
        if case["given"]:
            start = torch.randint(0, case["far"] + 1, (b, 1), generator=g, device="cuda")
            s["positions"] = (start + torch.arange(n, device="cuda")).to(torch.int32)
        shape = (lambda h: (b, h, n, d)) if case["head_major"] else (lambda h: (b, n, h, d))
        if op == "qk_norm_rope":
            s["q_out"] = torch.empty(*shape(hq), device="cuda")
            s["k_out"] = torch.empty(*shape(hk), device="cuda")
        else:
            s["dq_out"] = _randn(g, *shape(hq))
            s["dk_out"] = _randn(g, *shape(hk))
            s["d_qkv"] = torch.zeros_like(s["qkv"])
            s["d_q_weight"] = torch.empty(d, device="cuda")
            s["d_k_weight"] = torch.empty(d, device="cuda")
    elif op == "orthogonalize":
        s["x"] = _gradient(g, case["batch"], case["rows"], case["cols"])
        s["out"] = torch.empty_like(s["x"])
    else:
        s["grads"] = [_gradient(g, 1, *sh)[0] for sh in _shapes(case)]
        s["momenta"] = [_gradient(g, 1, *sh)[0] for sh in _shapes(case)]
        s["params"] = [_randn(g, *sh).mul_(0.02) for sh in _shapes(case)]
    return s


# --------------------------------------------------------------- the passes --
_LR, _MU, _DECAY = 0.02, 0.95, 0.01
_EPS = 1e-6


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _angles(case, positions):
    """cos and sin [batch or 1, seq, rot_dim / 2] of every position's angles."""
    rot = case["rot_dim"]
    if positions is None:
        positions = torch.arange(case["seq"], device="cuda")[None]
    freq = case["base"] ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    a = positions.double()[..., None] * freq
    return a.cos().float(), a.sin().float()


def _norm_rope(x, w, cos, sin, rot):
    """x [batch, seq, heads, dim] -> the same shape."""
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
    half = rot // 2
    a, b = y[..., :half], y[..., half:rot]
    c, s = cos[:, :, None], sin[:, :, None]
    return torch.cat((a * c - b * s, b * c + a * s, y[..., rot:]), -1)


def _norm_rope_grad(x, w, cos, sin, rot, g):
    half = rot // 2
    a, b = g[..., :half], g[..., half:rot]
    c, s = cos[:, :, None], sin[:, :, None]
    g = torch.cat((a * c + b * s, b * c - a * s, g[..., rot:]), -1)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    xn = x * r
    d_w = (g * xn).sum((0, 1, 2))
    g = g * w
    return r * (g - xn * (g * xn).mean(-1, keepdim=True)), d_w


def _orthogonalize(u, steps):
    """u [..., rows, cols] -> the Newton-Schulz iterate after `steps` steps."""
    a, b, c = NS
    x = u / (u * u).sum((-2, -1), keepdim=True).sqrt().clamp(min=NORM_FLOOR)
    wide = u.shape[-2] > u.shape[-1]
    if wide:
        x = x.mT
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.mT if wide else x).contiguous()


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "embedding":
        ids = s["ids"]
        rows = s["table"][ids.clamp(min=0)] * case["scale"]
        s["out"].copy_(rows * (ids >= 0)[:, None])
        return s["out"]
    if op == "embedding_grad":
        ids = s["ids"]
        g = s["grad_out"] * (ids >= 0)[:, None] * case["scale"]
        if not case["accumulate"]:
            s["d_table"].zero_()
        return s["d_table"].index_add_(0, ids.clamp(min=0), g)
    if op in ("qk_norm_rope", "qk_norm_rope_grad"):
        hq, hk, rot = case["q_heads"], case["k_heads"], case["rot_dim"]
        cos, sin = _angles(case, s["positions"])
        q, k = s["qkv"][:, :, :hq], s["qkv"][:, :, hq:hq + hk]
        major = (lambda t: t.transpose(1, 2)) if case["head_major"] else (lambda t: t)
        if op == "qk_norm_rope":
            s["q_out"].copy_(major(_norm_rope(q, s["q_weight"], cos, sin, rot)))
            s["k_out"].copy_(major(_norm_rope(k, s["k_weight"], cos, sin, rot)))
            return s["q_out"], s["k_out"]
        d_q, s["d_q_weight"] = _norm_rope_grad(q, s["q_weight"], cos, sin, rot,
                                               major(s["dq_out"]))
        d_k, s["d_k_weight"] = _norm_rope_grad(k, s["k_weight"], cos, sin, rot,
                                               major(s["dk_out"]))
        s["d_qkv"][:, :, :hq] = d_q
        s["d_qkv"][:, :, hq:hq + hk] = d_k
        return s["d_qkv"], s["d_q_weight"], s["d_k_weight"]
    if op == "orthogonalize":
        return s["out"].copy_(_orthogonalize(s["x"], case["steps"]))
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        m.mul_(_MU).add_(g, alpha=1 - _MU)
        u = g * (1 - _MU) + m * _MU if case["nesterov"] else m
        o = _orthogonalize(u, case["steps"])
        p.mul_(1 - _LR * _DECAY).sub_(o, alpha=_LR * 0.2 * math.sqrt(max(p.shape)))
    return s["params"], s["momenta"]


_DEV = None


def _device():
    global _DEV
    if _DEV is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "any-gpu_b200"))
        from any_gpu import GpuDevice
        _DEV = GpuDevice.gpu(torch.cuda.current_device())
    return _DEV


def _qk_shape(case):
    """The call's geometry, kept by a program like a plan."""
    from any_gpu import QkNormRope
    b, n, hq, hk, d = (case[k] for k in ("batch", "seq", "q_heads", "k_heads", "dim"))
    packed = ((hq + 2 * hk) * d, d, n * (hq + 2 * hk) * d)
    out = ((lambda h: (d, n * d, h * n * d)) if case["head_major"]
           else (lambda h: (h * d, d, n * h * d)))
    return QkNormRope(batch=b, seq=n, q_heads=hq, k_heads=hk, dim=d, rot_dim=case["rot_dim"],
                      eps=_EPS, base=case["base"], q_in=packed, k_in=packed, q_out=out(hq),
                      k_out=out(hk))


def _run_own(s):
    dev = _device()
    case = s["case"]
    op = case["op"]
    if op == "embedding":
        dev.launch_embedding(s["table"].data_ptr(), s["ids"].data_ptr(), s["out"].data_ptr(),
                             case["tokens"], case["vocab"], case["dim"], case["scale"])
        return s["out"]
    if op == "embedding_grad":
        dev.launch_embedding_backward(s["grad_out"].data_ptr(), s["ids"].data_ptr(),
                                      s["d_table"].data_ptr(), case["tokens"], case["vocab"],
                                      case["dim"], case["scale"], case["accumulate"])
        return s["d_table"]
    if op in ("qk_norm_rope", "qk_norm_rope_grad"):
        if "shape" not in s:
            s["shape"] = _qk_shape(case)
        q = s["qkv"].data_ptr()
        keys = case["q_heads"] * case["dim"] * 4
        pos = 0 if s["positions"] is None else s["positions"].data_ptr()
        if op == "qk_norm_rope":
            dev.launch_qk_norm_rope(s["shape"], q, q + keys, s["q_weight"].data_ptr(),
                                    s["k_weight"].data_ptr(), pos, s["q_out"].data_ptr(),
                                    s["k_out"].data_ptr())
            return s["q_out"], s["k_out"]
        d_q = s["d_qkv"].data_ptr()
        dev.launch_qk_norm_rope_backward(s["shape"], s["dq_out"].data_ptr(),
                                         s["dk_out"].data_ptr(), q, q + keys,
                                         s["q_weight"].data_ptr(), s["k_weight"].data_ptr(), pos,
                                         d_q, d_q + keys, s["d_q_weight"].data_ptr(),
                                         s["d_k_weight"].data_ptr())
        return s["d_qkv"], s["d_q_weight"], s["d_k_weight"]
    if op == "orthogonalize":
        dev.launch_orthogonalize(s["x"].data_ptr(), s["out"].data_ptr(), case["batch"],
                                 case["rows"], case["cols"], case["steps"])
        return s["out"]
    if "tensors" not in s:
        from any_gpu import muon_tensors
        s["tensors"] = muon_tensors(
            [(p.data_ptr(), g.data_ptr(), m.data_ptr(), *p.shape)
             for p, g, m in zip(s["params"], s["grads"], s["momenta"])])
    dev.launch_muon(s["tensors"], _LR, _MU, case["nesterov"], _DECAY, case["steps"])
    return s["params"], s["momenta"]


# -------------------------------------------------------------------- work --
def _distinct(case):
    """Expected number of distinct rows among the case's tokens."""
    t, v = case["tokens"], case["vocab"]
    p = np.diff(np.log(np.arange(1, v + 1, dtype=np.float64))) / math.log(v)
    return float((1 - (1 - p) ** (t - t // 32)).sum())


def work(case):
    op = case["op"]
    if op in ("embedding", "embedding_grad"):
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        live = t - t // 32
        rows = _distinct(case)
        if op == "embedding":
            return {"bytes": 4 * (rows * d + t * d + t), "flops": t * d}
        written = 2 * rows if case["accumulate"] else v
        return {"bytes": 4 * (live * d + written * d + t), "flops": 2 * live * d}
    if op in ("qk_norm_rope", "qk_norm_rope_grad"):
        rows = case["batch"] * case["seq"]
        n = rows * (case["q_heads"] + case["k_heads"]) * case["dim"]
        if op == "qk_norm_rope":
            return {"bytes": 8 * n + 4 * rows, "flops": 7 * n}
        return {"bytes": 12 * n + 4 * rows, "flops": 14 * n}
    shapes = ([(case["rows"], case["cols"])] * case["batch"] if op == "orthogonalize"
              else _shapes(case))
    flops = size = 0
    for r, c in shapes:
        m, n = min(r, c), max(r, c)
        # X X^T and A A are symmetric: half of each; then B X
        flops += case["steps"] * (m * m * n + m * m * m + 2 * m * m * n)
        size += r * c
    return {"bytes": 4 * size * (2 if op == "orthogonalize" else 5), "flops": flops}


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embedding":
        live = torch.nonzero(s["ids"] >= 0)[:, 0]
        out = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device="cuda")
        out[live] = torch.index_select(s["table"], 0, s["ids"][live]).double() * case["scale"]
        return out
    if op == "embedding_grad":
        d = (s["d_table"].double() if case["accumulate"] else
             torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda"))
        order = torch.argsort(s["ids"], stable=True)
        order = order[s["ids"][order] >= 0]
        if order.numel():
            ids, count = torch.unique_consecutive(s["ids"][order], return_counts=True)
            end = count.cumsum(0)
            total = torch.cat((torch.zeros(1, case["dim"], dtype=torch.float64, device="cuda"),
                               s["grad_out"][order].double().cumsum(0)))
            d[ids.long()] += (total[end] - total[end - count]) * case["scale"]
        return d
    if op in ("qk_norm_rope", "qk_norm_rope_grad"):
        hq, hk, rot = case["q_heads"], case["k_heads"], case["rot_dim"]
        pos = (torch.arange(case["seq"], device="cuda")[None] if s["positions"] is None
               else s["positions"]).double()
        inv = torch.exp(torch.arange(rot // 2, device="cuda", dtype=torch.float64)
                        * (-2.0 * math.log(case["base"]) / rot))
        turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"),
                           (pos[:, :, None] * inv)[:, :, None])

        def definition(x, w):
            y = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2
                               / case["dim"] + _EPS) * w
            z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * turn
            y = torch.cat((z.real, z.imag, y[..., rot:]), -1)
            return y.transpose(1, 2) if case["head_major"] else y

        qkv = s["qkv"].double()
        leaves = [qkv[:, :, :hq].clone(), qkv[:, :, hq:hq + hk].clone(),
                  s["q_weight"].double(), s["k_weight"].double()]
        if op == "qk_norm_rope":
            return (definition(leaves[0], leaves[2]).contiguous(),
                    definition(leaves[1], leaves[3]).contiguous())
        for x in leaves:
            x.requires_grad_(True)
        torch.autograd.backward([definition(leaves[0], leaves[2]),
                                 definition(leaves[1], leaves[3])],
                                [s["dq_out"].double(), s["dk_out"].double()])
        values = torch.zeros_like(qkv[:, :, hq + hk:])
        return (torch.cat((leaves[0].grad, leaves[1].grad, values), 2), leaves[2].grad,
                leaves[3].grad)

    def polynomial(u):
        """The iterate as one polynomial of the Gram matrix applied to the scaled matrix."""
        a, b, c = NS
        x = u / torch.linalg.vector_norm(u).clamp(min=NORM_FLOOR)
        tall = x.shape[0] > x.shape[1]
        gram = x.T @ x if tall else x @ x.T
        eye = torch.eye(gram.shape[0], dtype=torch.float64, device="cuda")
        total = eye
        for _ in range(case["steps"]):
            factor = a * eye + gram @ (b * eye + c * gram)
            total = factor @ total
            gram = factor @ gram @ factor
        return x @ total if tall else total @ x

    if op == "orthogonalize":
        return torch.stack([polynomial(x.double()) for x in s["x"]])
    params, momenta = [], []
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        g, m = g.double(), m.double()
        m = _MU * m + (1 - _MU) * g
        u = (1 - _MU) * g + _MU * m if case["nesterov"] else m
        momenta.append(m)
        params.append((1 - _LR * _DECAY) * p.double()
                      - _LR * 0.2 * math.sqrt(max(p.shape)) * polynomial(u))
    return params, momenta
