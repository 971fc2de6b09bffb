"""Calls of the products and of the distillation loss that callers may make: strided and misaligned
operands, outputs in place, captured graphs, other streams, threads, empty batches, sizes past 32-bit
offsets -- and what the wrappers refuse."""

import math
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _rand(seed, *shape, dtype=BF, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _off(t, shift=1):
    """A copy of ``t`` whose rows start ``shift`` elements into a wider, misaligned buffer."""
    wide = torch.full((t.shape[0], t.shape[1] + 13), 3.0, dtype=t.dtype, device=t.device)
    wide[:, shift:shift + t.shape[1]] = t
    return wide[:, shift:shift + t.shape[1]], wide


# both kernels: few rows (weights streamed) and many (pairs of CTAs); sizes that fill tiles and that do not
ROWS = [(5, 96, 128), (600, 320, 128), (600, 321, 128)]


@pytest.mark.parametrize("rows,n,k", ROWS)
def test_strides_and_alignment_do_not_change_results(rows, n, k):
    from kvstreams import ops

    x, w, u, b = _rand(1, rows, k), _rand(2, n, k), _rand(3, n, k), _rand(4, n)
    r, gy = _rand(5, rows, n), _rand(6, rows, n)
    pre = ops.pre_buffer(x, n)
    y = ops.linear(x, w, b, r, "silu", pre=pre)
    dx, dw, db = ops.linear_backward(gy, x, w, pre=pre, activation="silu", bias_grad=True)
    gpre = ops.pre_buffer(x, 2 * n)
    h = ops.gated_linear(x, w, u, pre=gpre)
    gx, gw, gu = ops.gated_linear_backward(gy, x, w, u, gpre)
    for shift in (1, 8):  # misaligned, and merely strided
        (xs, _), (ws, _), (us, _), (rs, _), (gs, _) = (_off(t, shift) for t in (x, w, u, r, gy))
        (ps, _), (hs, _) = _off(pre, shift), _off(gpre, shift)
        assert torch.equal(ops.linear(xs, ws, b, rs, "silu"), y)
        assert torch.equal(ops.gated_linear(xs, ws, us), h)
        got = ops.linear_backward(gs, xs, ws, pre=ps, activation="silu", bias_grad=True)
        assert all(torch.equal(p, q) for p, q in zip(got, (dx, dw, db)))
        got = ops.gated_linear_backward(gs, xs, ws, us, hs)
        assert all(torch.equal(p, q) for p, q in zip(got, (gx, gw, gu)))
        # outputs into strided buffers: what lies beside them stays
        (out, wide), (pout, pwide) = _off(torch.zeros_like(y), shift), _off(torch.zeros_like(pre), shift)
        assert ops.linear(x, w, b, r, "silu", pre=pout, out=out) is out
        assert torch.equal(out, y) and torch.equal(pout, pre)
        for t in (wide, pwide):
            assert (t[:, :shift] == 3).all() and (t[:, shift + n:] == 3).all()
        (gout, gwide) = _off(torch.zeros_like(gpre), shift)
        ops.gated_linear(x, w, u, pre=gout)
        assert torch.equal(gout, gpre) and (gwide[:, shift + 2 * n:] == 3).all() and (gwide[:, :shift] == 3).all()
    # transposed, expanded and higher-dimensional operands
    assert torch.equal(ops.linear(x.t().contiguous().t(), w.t().contiguous().t(), b, r, "silu"), y)
    assert torch.equal(ops.linear(x[:1].expand(rows, k), w)[rows - 1], ops.linear(x[:1], w)[0])
    assert torch.equal(ops.linear(x, w, residual=r[:1].expand(rows, n)), ops.linear(x, w, residual=r[:1].repeat(rows, 1)))
    cube = x.view(5, -1, k)
    assert torch.equal(ops.linear(cube, w, b, r.view(5, -1, n), "silu"), y.view(5, -1, n))
    assert torch.equal(ops.linear(cube.transpose(0, 1), w).transpose(0, 1).reshape(rows, n), ops.linear(x, w))
    assert ops.linear(x[0], w).shape == (n,)


@pytest.mark.parametrize("rows,n,k", ROWS)
def test_out_may_be_the_residual(rows, n, k):
    from kvstreams import ops

    x, w, r = _rand(1, rows, k), _rand(2, n, k), _rand(3, rows, n)
    want = ops.linear(x, w, residual=r)
    assert ops.linear(x, w, residual=r, out=r) is r
    assert torch.equal(r, want)


def test_no_rows():
    from kvstreams import functional as KF, ops

    x, w, u = torch.empty(0, 64, dtype=BF, device="cuda"), _rand(1, 40, 64), _rand(2, 40, 64)
    assert ops.linear(x, w, _rand(3, 40), activation="gelu").shape == (0, 40)
    assert ops.gated_linear(x.view(0, 3, 64), w, u).shape == (0, 3, 40)
    dx, dw, db = ops.linear_backward(torch.empty(0, 40, dtype=BF, device="cuda"), x, w, bias_grad=True)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()
    dx, dg, du = ops.gated_linear_backward(torch.empty(0, 40, dtype=BF, device="cuda"), x, w, u,
                                           ops.pre_buffer(x, 80))
    assert (dg == 0).all() and (du == 0).all()
    ws = w.clone().requires_grad_()
    KF.linear(x, ws).sum().backward()
    assert (ws.grad == 0).all()
    loss, lse = ops.distill(torch.empty(0, 9, device="cuda"), torch.empty(0, 2, dtype=torch.long, device="cuda"),
                            torch.empty(0, 2, device="cuda"))
    assert loss.shape == lse.shape == (0,)


def test_infinities_and_nan_stay_in_their_rows():
    """A row of x with inf / NaN changes its own output row only, through every tile and split."""
    from kvstreams import ops

    for rows in (3, 300):
        x, w = _rand(1, rows, 256), _rand(2, 200, 256)
        clean = ops.linear(x, w, activation="gelu")
        x[1, 5] = math.nan
        x[2, 7] = math.inf
        y = ops.linear(x, w, activation="gelu")
        assert y[1].isnan().all()
        assert not torch.isfinite(y[2]).any() or (y[2] == 0).any()  # +-inf, gelu(-inf) = nan or 0
        keep = [i for i in range(rows) if i not in (1, 2)]
        assert torch.equal(y[keep], clean[keep])
        assert ops.linear(x, w, activation="relu")[1].isnan().all()


@pytest.mark.parametrize("rows", [3, 200, 700])
def test_captured_and_replayed(rows):
    """Two graphs over the same operators, replayed in turn with new inputs in place."""
    from kvstreams import ops

    w, u, b = _rand(2, 264, 128), _rand(3, 264, 128), _rand(4, 264)
    ids = torch.randint(0, 264, (rows, 5), device="cuda")
    t = _rand(9, rows, 5, dtype=torch.float32)
    g1 = torch.rand(rows, device="cuda")

    def step(x, gy):
        pre, gpre = ops.pre_buffer(x, 264), ops.pre_buffer(x, 528)
        y = ops.linear(x, w, b, activation="gelu", pre=pre)
        h = ops.gated_linear(x, w, u, pre=gpre)
        outs = [y, h, *ops.linear_backward(gy, x, w, pre=pre, activation="gelu", bias_grad=True),
                *ops.gated_linear_backward(gy, x, w, u, gpre)]
        loss, lse = ops.distill(h, ids, t)
        return outs + [loss, lse, ops.distill_backward(h, ids, t, lse, g1)]

    graphs = []
    for seed in (1, 2):
        x, gy = _rand(10 + seed, rows, 128), _rand(20 + seed, rows, 264)
        step(x, gy)  # (first call of a kernel sets its attributes)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(x, gy)
        graphs.append((g, x, gy, outs))
    for round_ in range(2):
        for i, (g, x, gy, outs) in enumerate(graphs):
            x.copy_(_rand(100 + 10 * round_ + i, rows, 128))
            gy.copy_(_rand(200 + 10 * round_ + i, rows, 264))
        graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for g, x, gy, outs in graphs:
            assert all(torch.equal(p, q) for p, q in zip(outs, step(x, gy)))


def test_two_streams_and_threads():
    """Calls from two streams (two host threads) at once equal the same calls alone."""
    from kvstreams import ops

    cases = []
    for seed, rows in ((1, 4), (2, 300)):
        x, w, u = _rand(seed, rows, 512), _rand(seed + 5, 640, 512), _rand(seed + 6, 640, 512)
        gy = _rand(seed + 7, rows, 640)
        pre = ops.pre_buffer(x, 1280)

        def run(x=x, w=w, u=u, gy=gy, pre=pre):
            h = ops.gated_linear(x, w, u, pre=pre)
            return [h, ops.linear(x, w, activation="silu"), *ops.gated_linear_backward(gy, x, w, u, pre)]

        cases.append((run, [t.clone() for t in run()]))
    torch.cuda.synchronize()
    bad = []

    def work(run, want):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = run()
                s.synchronize()
                bad.extend(1 for p, q in zip(got, want) if not torch.equal(p, q))

    threads = [threading.Thread(target=work, args=c) for c in cases]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


CUT = (600, 1500, 14344)  # rows, n, k of a product whose tiles are cut among the pairs of CTAs


def test_cut_product_captured_and_replayed():
    """A cut product's flags are left clean: replays of two graphs in turn, with eager calls between,
    equal the eager results, and a row with a NaN stays alone."""
    from kvstreams import ops

    rows, n, k = CUT
    w, u = _rand(2, n, k, scale=0.05), _rand(3, n, k, scale=0.05)
    graphs = []
    for seed in (1, 2):
        x = _rand(10 + seed, rows, k)
        ops.linear(x, w)
        ops.gated_linear(x, w, u)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.linear(x, w, activation="silu")
            h = ops.gated_linear(x, w, u)
        graphs.append((g, x, y, h))
    for round_ in range(4):
        for i, (g, x, y, h) in enumerate(graphs):
            x.copy_(_rand(100 + 10 * round_ + i, rows, k))
            if round_ == 3:
                x[7, 3] = math.nan
        for g, *_ in graphs:
            g.replay()
        for g, x, y, h in graphs:
            assert torch.equal(y.nan_to_num(), ops.linear(x, w, activation="silu").nan_to_num())
            assert torch.equal(h.nan_to_num(), ops.gated_linear(x, w, u).nan_to_num())
            bad = y.isnan().any(1)
            assert bad.sum().item() == (1 if round_ == 3 else 0) and (round_ < 3 or y[7].isnan().all())


def test_cut_products_on_two_streams():
    from kvstreams import ops

    rows, n, k = CUT
    xs = [_rand(s, rows, k) for s in (1, 2)]
    ws = [_rand(s + 5, n, k, scale=0.05) for s in (1, 2)]
    want = [ops.linear(x, w) for x, w in zip(xs, ws)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.linear(xs[i], ws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_long_rows_captured():
    """Few long logits rows (a cluster per row) in a graph."""
    from kvstreams import ops

    x = _rand(1, 3, 50000, dtype=torch.float32)
    ids, t, g1 = torch.randint(0, 50000, (3, 9), device="cuda"), _rand(2, 3, 9, dtype=torch.float32), torch.rand(3, device="cuda")
    ops.distill_backward(x, ids, t, ops.distill(x, ids, t)[1], g1)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss, lse = ops.distill(x, ids, t)
        d = ops.distill_backward(x, ids, t, lse, g1)
    for seed in (3, 4):
        x.copy_(_rand(seed, 3, 50000, dtype=torch.float32))
        g.replay()
        l2, e2 = ops.distill(x, ids, t)
        assert torch.equal(loss, l2) and torch.equal(lse, e2)
        assert torch.equal(d, ops.distill_backward(x, ids, t, e2, g1))


def test_offsets_past_32_bits():
    """Results of more than 2^31 elements: the last rows and columns are where they belong."""
    from kvstreams import ops

    rows, n, k = 70000, 32768, 64  # 2.29e9 results
    x, w = _rand(1, rows, k), _rand(2, n, k)
    y = ops.linear(x, w)
    for r in (0, 65535, 65536, rows - 1):
        want = (x[r:r + 1].float() @ w.float().t())
        assert (y[r:r + 1].float() - want).abs().max().item() <= 2 ** -8 * want.abs().max().item() + 1e-3
    del y
    rows, vocab = 17000, 128256  # 2.18e9 logits
    lg = torch.zeros(rows, vocab, dtype=BF, device="cuda")
    lg[rows - 1, 77] = 4.0
    ids = torch.full((rows, 2), 77, dtype=torch.long, device="cuda")
    t = torch.zeros(rows, 2, device="cuda")
    loss, lse = ops.distill(lg, ids, t)
    lse_last = math.log(vocab - 1 + math.exp(4.0))
    assert abs(lse[rows - 1].item() - lse_last) <= 1e-4 and abs(lse[rows - 2].item() - math.log(vocab)) <= 1e-4
    d = ops.distill_backward(lg, ids, t, lse, torch.ones(rows, device="cuda"), out=lg)
    assert abs(d[rows - 1, 77].item() - (math.exp(4.0 - lse_last) - 1.0)) <= 2 ** -8
    assert abs(d[rows - 1, vocab - 1].item() * vocab - 1.0) <= 1e-2


def test_another_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    from kvstreams import ops

    x, w = _rand(1, 5, 64), _rand(2, 40, 64)
    want = ops.linear(x, w)
    assert torch.equal(ops.linear(x.to("cuda:1"), w.to("cuda:1")).to("cuda:0"), want)


def test_refusals():
    from kvstreams import ops

    x, w, u = _rand(1, 4, 64), _rand(2, 40, 64), _rand(3, 40, 64)
    gy, pre = _rand(4, 4, 40), ops.pre_buffer(x, 40)
    bad = ValueError
    for call in (
        lambda: ops.linear(x.float(), w.float()),
        lambda: ops.linear(x, w.half()),
        lambda: ops.linear(x, w[:, :32]),
        lambda: ops.linear(x[:, :60].contiguous(), w[:, :60].contiguous()),
        lambda: ops.linear(x, w[0]),
        lambda: ops.linear(x, w, activation="tanh"),
        lambda: ops.linear(x, w, bias=gy),
        lambda: ops.linear(x, w, bias=_rand(5, 40).float()),
        lambda: ops.linear(x, w, residual=gy[:3]),
        lambda: ops.linear(x, w, residual=gy[:1]),
        lambda: ops.linear(x, w, out=torch.empty(4, 41, dtype=BF, device="cuda")),
        lambda: ops.linear(x, w, out=torch.empty(40, 4, dtype=BF, device="cuda").t()),
        lambda: ops.linear(x, w, pre=ops.pre_buffer(x, 80)),
        lambda: ops.linear(x, w, pre=pre.half()),
        lambda: ops.gated_linear(x, w, u[:39]),
        lambda: ops.gated_linear(x, w, u, pre=pre),
        lambda: ops.linear_backward(gy[:3], x, w),
        lambda: ops.linear_backward(gy.float(), x, w),
        lambda: ops.linear_backward(gy, x, w, activation="silu"),
        lambda: ops.gated_linear_backward(gy, x, w, u, pre),
    ):
        with pytest.raises(bad):
            call()
    lg, ids, t = torch.zeros(4, 50, device="cuda"), torch.zeros(4, 3, dtype=torch.long, device="cuda"), torch.zeros(4, 3, device="cuda")
    g = torch.ones(4, device="cuda")
    loss, lse = ops.distill(lg, ids, t)
    for call in (
        lambda: ops.distill(lg.to(torch.int32), ids, t),
        lambda: ops.distill(lg[0], ids, t),
        lambda: ops.distill(lg.t(), ids, t),
        lambda: ops.distill(lg, ids[:3], t[:3]),
        lambda: ops.distill(lg, ids, t[:, :2]),
        lambda: ops.distill(lg, ids.float(), t),
        lambda: ops.distill(lg, ids[:, :0], t[:, :0]),
        lambda: ops.distill(lg[:, :0], ids, t),
        lambda: ops.distill_backward(lg, ids, t, lse[:3], g),
        lambda: ops.distill_backward(lg, ids, t, lse, g, out=torch.empty(4, 49, device="cuda")),
        lambda: ops.distill_backward(lg, ids, t, lse, g, out=torch.empty(50, 4, device="cuda").t()),
        lambda: ops.distill_backward(torch.zeros(5, 50, device="cuda")[:4], ids, t, lse, g, out_dtype=torch.int32),
    ):
        with pytest.raises(bad):
            call()
    # outputs over operands that are read meanwhile (k = n here, so the shapes fit)
    sq, wide = _rand(7, 64, 64), _rand(8, 6, 64)
    for call in (
        lambda: ops.linear(x, sq, out=x),
        lambda: ops.linear(sq, sq, out=sq),
        lambda: ops.linear(x, sq, residual=wide[:4], out=wide[1:5]),
        lambda: ops.gated_linear(x, sq, sq, out=x),
        lambda: ops.linear(x, sq, out=wide[:4], pre=wide[1:5]),
        lambda: ops.linear(x, sq, residual=wide[:4], pre=wide[:4]),
    ):
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert ops.linear(x, sq, out=wide[2:]).data_ptr() == wide[2:].data_ptr()
    big = torch.zeros(5, 50, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        ops.distill_backward(big[:4], ids, t, lse, g, out=big[1:])
    for T in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(RuntimeError, match="bad argument"):
            ops.distill(lg, ids, t, T)
    with pytest.raises(RuntimeError, match="unsupported"):
        ops.distill(lg, ids.repeat(1, 400), t.repeat(1, 400))
    with pytest.raises(RuntimeError, match="unsupported"):
        ops.distill_backward(lg.bfloat16(), ids, t, lse, g, out_dtype=torch.float32)
