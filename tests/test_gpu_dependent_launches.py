"""The products and the distillation kernels are launched so that each starts while the one before it still
runs, and waits for its end before the first read.  Chains in which every kernel reads what the one before
wrote, into the same buffers over and over with other values, equal the same calls one at a time."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _rand(g, *shape, scale=1.0, dtype=BF):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("rows,vocab", [(5, 1000), (3, 20000), (300, 1000)])
def test_every_kernel_sees_what_the_one_before_wrote(rows, vocab):
    from kvstreams import ops

    g = torch.Generator(device="cuda").manual_seed(rows)
    w1, wu, head = _rand(g, 512, 256, scale=0.1), _rand(g, 512, 256, scale=0.1), _rand(g, vocab, 512, scale=0.05)
    xs = [_rand(g, rows, 256) for _ in range(12)]
    ids = torch.randint(0, vocab, (rows, 7), generator=g, device="cuda")
    t = _rand(g, rows, 7, dtype=torch.float32)
    up = torch.rand(rows, generator=g, device="cuda")
    pre, h = torch.empty(rows, 1024, device="cuda"), torch.empty(rows, 512, dtype=BF, device="cuda")
    logits, dlog = (torch.empty(rows, vocab, dtype=BF, device="cuda") for _ in range(2))

    def step(x, pause):
        out = []
        for f in (lambda: ops.gated_linear(x, w1, wu, pre=pre, out=h), lambda: ops.linear(h, head, out=logits),
                  lambda: out.extend(ops.distill(logits, ids, t)),
                  lambda: ops.distill_backward(logits, ids, t, out[1], up, out=dlog),
                  lambda: out.extend(ops.linear_backward(dlog, h, head, bias_grad=True)),
                  lambda: out.extend(ops.gated_linear_backward(out[2], x, w1, wu, pre))):
            f()
            if pause:
                torch.cuda.synchronize()
        return out

    want = [[o.clone() for o in step(x, True)] for x in xs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = [step(x, False) for x in xs]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
