"""Operators of a training and serving step, measured: plain forms, the library's calls, exact values.

Three operators, each with its gradient:

* ``linear``   y = act(x W^T + b) + r, the product with its epilogue in one pass
* ``gated``    h = act(x Wg^T) * (x Wu^T), both projections and the product of the feed-forward block
* ``distill``  the loss against a teacher's top logits, per row
               sum_j p_j (log p_j - log q[id_j]),  p = softmax(t / T) over the kept slots,
               q = softmax(x / T) over the vocabulary

``run`` computes them from elementary operations in 32 bits, or, with ``own``, makes the library's calls.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MOST_FLOPS = 6 * 8192 * 2 * 14336 * 4096  # of the largest listed case
_MOST_LOGITS = 8192 * 128256


def listed():
    return [
        # one stream's next token through an attention output projection, the residual row added
        {"name": "linear_token", "op": "linear", "rows": 1, "n": 4096, "k": 4096, "dtype": "bf16", "act": "none",
         "bias": False, "residual": True, "train": False},
        # 64 rollout streams' next tokens through a feed-forward block's second product
        {"name": "linear_step64", "op": "linear", "rows": 64, "n": 4096, "k": 14336, "dtype": "bf16", "act": "none",
         "bias": False, "residual": True, "train": False},
        # a prompt chunk of odd length through a fused q|k|v projection with bias
        {"name": "linear_chunk_fp16", "op": "linear", "rows": 1999, "n": 6144, "k": 4096, "dtype": "fp16",
         "act": "none", "bias": True, "residual": False, "train": False},
        # a small head (value head, adapter) in training: odd rows and width, every epilogue part
        {"name": "linear_gelu_train", "op": "linear", "rows": 777, "n": 1001, "k": 520, "dtype": "bf16",
         "act": "gelu", "bias": True, "residual": True, "train": True},
        # an output projection over one replayed training batch, forward and backward
        {"name": "linear_train", "op": "linear", "rows": 8192, "n": 4096, "k": 4096, "dtype": "bf16", "act": "none",
         "bias": True, "residual": True, "train": True},
        # one stream's next token through the gated projections
        {"name": "gated_token", "op": "gated", "rows": 1, "d": 4096, "f": 14336, "dtype": "bf16", "act": "silu",
         "train": False},
        # 48 streams' next tokens
        {"name": "gated_step48_fp16", "op": "gated", "rows": 48, "d": 4096, "f": 14336, "dtype": "fp16",
         "act": "silu", "train": False},
        # prefill of a long prompt
        {"name": "gated_prefill", "op": "gated", "rows": 4096, "d": 4096, "f": 14336, "dtype": "bf16", "act": "silu",
         "train": False},
        # one replayed training batch, forward and backward
        {"name": "gated_train", "op": "gated", "rows": 8192, "d": 4096, "f": 14336, "dtype": "bf16", "act": "silu",
         "train": True},
        # loss of one chunk of a replayed batch against the teacher's 64 best logits a token
        {"name": "distill_loss", "op": "distill", "rows": 8192, "vocab": 128256, "top": 64, "dtype": "fp32",
         "grad_dtype": "fp32", "temperature": 1.0, "train": False},
        # loss and gradient, the gradient in the lm_head weight's type
        {"name": "distill_train", "op": "distill", "rows": 4096, "vocab": 128256, "top": 64, "dtype": "fp32",
         "grad_dtype": "bf16", "temperature": 1.0, "train": True},
        # a short turn, odd vocabulary, half-precision logits, softened targets
        {"name": "distill_small", "op": "distill", "rows": 333, "vocab": 32003, "top": 20, "dtype": "bf16",
         "grad_dtype": "bf16", "temperature": 2.0, "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "gated", "distill"])
    if op == "distill":
        rows, vocab = _log_int(rng, 1, 8192), _log_int(rng, 104, 128256)
        dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
        return {"op": op, "rows": min(rows, _MOST_LOGITS // vocab), "vocab": vocab,
                "top": min(vocab, _log_int(rng, 1, 128)), "dtype": dtype,
                "grad_dtype": rng.choice(["fp32", "bf16"]) if dtype == "fp32" else dtype,
                "temperature": rng.choice([1.0, 0.7, 2.0]), "train": rng.random() < 0.5}
    rows = _log_int(rng, 1, 8192)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    train = rng.random() < 0.4
    if op == "linear":
        n, k = _log_int(rng, 64, 14336), 8 * _log_int(rng, 8, 1792)
        while (6 if train else 2) * rows * n * k > _MOST_FLOPS:
            rows = max(1, rows // 2)
        return {"op": op, "rows": rows, "n": n, "k": k, "dtype": dtype,
                "act": rng.choice(["none", "none", "relu", "silu", "gelu"]), "bias": rng.random() < 0.5,
                "residual": rng.random() < 0.5, "train": train}
    f, d = _log_int(rng, 64, 14336), 8 * _log_int(rng, 8, 512)
    return {"op": op, "rows": rows, "d": d, "f": f, "dtype": dtype, "act": rng.choice(["silu", "silu", "gelu"]),
            "train": train}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype=None):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype or _DTYPES[case["dtype"]])

    s = dict(case)
    rows = case["rows"]
    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        s["x"], s["w"] = normal(rows, k), normal(n, k, scale=0.02)
        s["b"] = normal(n, scale=0.1) if case["bias"] else None
        s["r"] = normal(rows, n) if case["residual"] else None
        s["gy"] = normal(rows, n, scale=0.1) if case["train"] else None
    elif case["op"] == "gated":
        d, f = case["d"], case["f"]
        s["x"] = normal(rows, d)
        s["wg"], s["wu"] = normal(f, d, scale=0.02), normal(f, d, scale=0.02)
        s["gh"] = normal(rows, f, scale=0.1) if case["train"] else None
    else:
        vocab, top = case["vocab"], case["top"]
        s["x"] = normal(rows, vocab, scale=2.5)
        s["ids"] = torch.empty(rows, top, dtype=torch.long, device="cuda")
        s["t"] = torch.empty(rows, top, dtype=torch.float32, device="cuda")
        for a in range(0, rows, 512):  # a teacher near the student, a chunk of rows at a time
            part = s["x"][a:a + 512].float()
            part += normal(*part.shape, dtype=torch.float32)
            s["t"][a:a + 512], s["ids"][a:a + 512] = part.topk(top, dim=-1)
        # some rows keep fewer logits than there are slots, some (prompt tokens) none
        keep = torch.randint(1, top + 1, (rows, 1), generator=g, device="cuda")
        keep = torch.where(torch.rand(rows, 1, generator=g, device="cuda") < 0.8, top, keep)
        keep[::17] = 0 if rows > 1 else top
        free = torch.arange(top, device="cuda")[None, :] >= keep
        s["ids"][free] = -1
        s["t"][free] = -math.inf
        s["g"] = torch.rand(rows, generator=g, device="cuda") / rows if case["train"] else None
    return s


def _library():
    if "kvstreams" not in sys.modules:
        sys.path.insert(0, str(Path("faster-rl-training_b200").resolve()))
    from kvstreams import ops

    return ops


def run(state):
    return (_own if own else _plain)[state["op"]](state)


# ---------------------------------------------------------------------- plain forms
def _act(z, name):
    """act(z) and its derivative."""
    if name == "none":
        return z, None
    if name == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if name == "silu":
        e = 1.0 / (1.0 + torch.exp(-z))
        return z * e, e * (1.0 + z * (1.0 - e))
    cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_linear(s):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y, slope = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    y = y.to(dt)
    if not s["train"]:
        return {"y": y}
    dz = s["gy"].float()
    if slope is not None:
        dz = dz * slope
    out = {"y": y, "dx": (dz @ w).to(dt), "dw": (dz.t() @ x).to(dt)}
    if s["b"] is not None:
        out["db"] = dz.sum(0).to(dt)
    return out


def _plain_gated(s):
    dt = s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    u = x @ wu.t()
    a, slope = _act(x @ wg.t(), s["act"])
    h = (a * u).to(dt)
    if not s["train"]:
        return {"h": h}
    gh = s["gh"].float()
    dg, du = gh * u * slope, gh * a
    return {"h": h, "dx": (dg @ wg + du @ wu).to(dt), "dwg": (dg.t() @ x).to(dt), "dwu": (du.t() @ x).to(dt)}


def _plain_distill(s):
    x = s["x"].float() / s["temperature"]
    m = x.max(dim=-1, keepdim=True).values
    lse = m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    kept = (s["ids"] >= 0) & (s["t"] > -math.inf)
    t = torch.where(kept, s["t"] / s["temperature"], -math.inf)
    tm = t.max(dim=-1, keepdim=True).values
    tm = torch.where(tm > -math.inf, tm, 0.0)
    e = torch.where(kept, torch.exp(t - tm), 0.0)
    total = e.sum(-1, keepdim=True)
    some = total > 0
    total = torch.where(some, total, 1.0)
    p = e / total
    at = s["ids"].clamp(min=0)
    term = p * (torch.where(kept, t - tm, 0.0) - torch.log(total) - (x.gather(1, at) - lse))
    loss = torch.where(kept, term, 0.0).sum(-1)
    if not s["train"]:
        return {"loss": loss, "lse": lse[:, 0]}
    scale = torch.where(some[:, 0], s["g"] / s["temperature"], 0.0)[:, None]
    d = torch.exp(x - lse) * scale
    d.scatter_add_(1, at, -p * scale)
    return {"loss": loss, "lse": lse[:, 0], "dlogits": d.to(_DTYPES[s["grad_dtype"]])}


_plain = {"linear": _plain_linear, "gated": _plain_gated, "distill": _plain_distill}


# ---------------------------------------------------------------------- the library's calls
def _own_linear(s):
    ops, act = _library(), None if s["act"] == "none" else s["act"]
    if not s["train"]:
        return {"y": ops.linear(s["x"], s["w"], bias=s["b"], residual=s["r"], activation=act)}
    pre = ops.pre_buffer(s["x"], s["n"]) if act else None
    y = ops.linear(s["x"], s["w"], bias=s["b"], residual=s["r"], activation=act, pre=pre)
    dx, dw, db = ops.linear_backward(s["gy"], s["x"], s["w"], pre=pre, activation=act, bias_grad=s["b"] is not None)
    out = {"y": y, "dx": dx, "dw": dw}
    if db is not None:
        out["db"] = db
    return out


def _own_gated(s):
    ops = _library()
    if not s["train"]:
        return {"h": ops.gated_linear(s["x"], s["wg"], s["wu"], activation=s["act"])}
    pre = ops.pre_buffer(s["x"], 2 * s["f"])
    h = ops.gated_linear(s["x"], s["wg"], s["wu"], activation=s["act"], pre=pre)
    dx, dwg, dwu = ops.gated_linear_backward(s["gh"], s["x"], s["wg"], s["wu"], pre, activation=s["act"])
    return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu}


def _own_distill(s):
    ops = _library()
    loss, lse = ops.distill(s["x"], s["ids"], s["t"], s["temperature"])
    if not s["train"]:
        return {"loss": loss, "lse": lse}
    d = ops.distill_backward(s["x"], s["ids"], s["t"], lse, s["g"], s["temperature"],
                             out_dtype=_DTYPES[s["grad_dtype"]])
    return {"loss": loss, "lse": lse, "dlogits": d}


_own = {"linear": _own_linear, "gated": _own_gated, "distill": _own_distill}


# ---------------------------------------------------------------------- floors
def work(case):
    """Each input read once and each output written once; the products' multiply-adds."""
    size = 4 if case["dtype"] == "fp32" else 2
    rows, train = case["rows"], case["train"]
    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        values = rows * k + n * k + rows * n * (1 + case["residual"]) + n * case["bias"]
        total = size * values
        if train:
            total += size * (rows * n + rows * k + n * k + n * case["bias"])
        return {"bytes": total, "flops": (6 if train else 2) * rows * n * k}
    if case["op"] == "gated":
        d, f = case["d"], case["f"]
        total = size * (rows * d + 2 * f * d + rows * f)
        if train:
            total += size * (rows * f + rows * d + 2 * f * d)
        return {"bytes": total, "flops": (6 if train else 2) * rows * 2 * f * d}
    vocab, top = case["vocab"], case["top"]
    total = rows * (vocab * size + top * 12 + 8)
    if train:
        total += rows * (vocab * (4 if case["grad_dtype"] == "fp32" else 2) + 4)
    return {"bytes": total, "flops": (5 if train else 3) * rows * vocab}


# ---------------------------------------------------------------------- exact values
_EXACT_ACT = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu,
              "gelu": torch.nn.functional.gelu}


def exact(case, seed):
    """The definitions in 64 bits, gradients by differentiating them."""
    s = prepare(case, seed)
    if case["op"] == "distill":
        return _exact_distill(case, s)
    act = _EXACT_ACT[case["act"]]
    names = ["x", "w", "b"] if case["op"] == "linear" else ["x", "wg", "wu"]
    v = {k: s[k].double().requires_grad_(bool(case["train"])) for k in names if s.get(k) is not None}
    with torch.set_grad_enabled(bool(case["train"])):
        if case["op"] == "linear":
            y = act(torch.nn.functional.linear(v["x"], v["w"], v.get("b")))
            if s["r"] is not None:
                y = y + s["r"].double()
            out, up = {"y": y.detach()}, s["gy"]
        else:
            y = act(torch.nn.functional.linear(v["x"], v["wg"])) * torch.nn.functional.linear(v["x"], v["wu"])
            out, up = {"h": y.detach()}, s["gh"]
        if case["train"]:
            grads = torch.autograd.grad(y, list(v.values()), up.double())
            out.update({"d" + k: g for k, g in zip(v, grads)})
    return out


def _exact_distill(case, s):
    temp, parts = case["temperature"], []
    for a in range(0, case["rows"], 256):
        x = s["x"][a:a + 256].double().requires_grad_(bool(case["train"]))
        ids, t = s["ids"][a:a + 256], s["t"][a:a + 256].double()
        with torch.set_grad_enabled(bool(case["train"])):
            logq = torch.log_softmax(x / temp, dim=-1)
            kept = ids >= 0
            logp = torch.log_softmax(torch.where(kept, t / temp, -1e300), dim=-1)
            logp = torch.where(kept, logp, 0.0)
            p = torch.where(kept, logp.exp(), 0.0)
            loss = (p * (logp - logq.gather(1, ids.clamp(min=0)))).sum(-1)
            if case["train"]:
                (d,) = torch.autograd.grad(loss, [x], s["g"][a:a + 256].double())
                parts.append((loss.detach(), torch.logsumexp(x.detach() / temp, -1), d))
            else:
                parts.append((loss, torch.logsumexp(x / temp, -1)))
    cat = [torch.cat(p) for p in zip(*parts)]
    return dict(zip(["loss", "lse", "dlogits"], cat))
