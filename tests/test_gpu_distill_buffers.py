"""Where the distillation gradient may be written: in place also where several CTAs share a row, and not over
anything else that its kernels read."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(rows, vocab, top, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 2.5).to(dtype)
    ids = torch.randint(0, vocab, (rows, top), generator=g, device="cuda")
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    t = torch.randn(rows, top, generator=g, device="cuda").to(acc)
    return x, ids, t, torch.rand(rows, generator=g, device="cuda").to(acc)


def test_over_other_operands_is_refused():
    from kvstreams import ops

    x, ids, t, g = _case(4, 50, 3)
    _, lse = ops.distill(x, ids, t)
    want = ops.distill_backward(x, ids, t, lse, g)
    for which in ("lse", "grad", "teacher", "ids"):
        flat = torch.zeros(4 * 50, device="cuda")
        out = flat.view(4, 50)
        args = dict(ids=ids, teacher=t, lse=lse, grad=g)
        part = flat[100:100 + 4] if which in ("lse", "grad") else flat[60:72].view(4, 3) if which == "teacher" else \
            flat[60:84].view(torch.long).view(4, 3)
        part.copy_(args[which])
        args[which] = part
        with pytest.raises(ValueError, match="overlaps"):
            ops.distill_backward(x, **args, out=out)
        assert torch.equal(part, dict(ids=ids, teacher=t, lse=lse, grad=g)[which])  # nothing was written
    # beside them it may be
    flat = torch.zeros(4 + 200, device="cuda")
    flat[:4].copy_(lse)
    got = ops.distill_backward(x, ids, t, flat[:4], g, out=flat[4:].view(4, 50))
    assert torch.equal(got, want) and torch.equal(flat[:4], lse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("rows,vocab,top", [(1, 128256, 300), (3, 50001, 64), (5, 128256, 1024), (40, 32003, 20)])
def test_in_place_where_ctas_share_a_row(rows, vocab, top, dtype):
    """Bit for bit the gradient written elsewhere, ids that repeat and ids at the segments' ends among the slots."""
    from kvstreams import ops

    x, ids, t, g = _case(rows, vocab, top, dtype)
    for j, at in enumerate((0, vocab // 2 - 1, vocab // 2, vocab - 1, vocab // 8, vocab // 8, vocab - 1)):
        ids[:, j] = at
    _, lse = ops.distill(x, ids, t)
    want = ops.distill_backward(x, ids, t, lse, g)
    # the definition, each id's weights together
    p = torch.softmax(t.double(), -1)
    q = torch.softmax(x.double(), -1)
    exact = g.double()[:, None] * q.scatter_add(1, ids, -p)
    u, eps = (2.0**-46 if dtype == torch.float64 else 2.0**-18), torch.finfo(dtype).eps / 2
    mass = g.double()[:, None] * torch.zeros_like(q).scatter_add(1, ids, p).add_(q)
    assert ((want.double() - exact).abs() <= u * mass * (1 + lse.double().abs())[:, None] + exact.abs() * eps * 1.01 + 2.0**-25 * (dtype == torch.float16) + 1e-37).all()
    got = ops.distill_backward(x, ids, t, lse, g, out=x)
    assert got is x and torch.equal(x, want)
