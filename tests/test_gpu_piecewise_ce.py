"""Linear + cross entropy in pieces of the vocabulary against the formula in 64 bits.

Tolerances.  Products of 16-bit values are exact in fp32 and accumulate in fp32:
a logit is off by at most ``e_z = (d + 16) 2^-23 sum |h w|`` (a whole step for each
addition, whatever its rounding mode).  The log-sum-exp and the target logit are
then off by ``e_z`` each, plus a few fp32 roundings of values up to ``|lse| + ln V``.
Each element of dz is off by the change of the exponential (``2 e_z`` and the fp32
steps, relative) and half a step of its 16-bit type (``u``); sums over it add
``K 2^-23`` relative in fp32, and the result is rounded to the type once more."""

import math

import pytest
import torch


def _exact(h, w, t, ignore, reduction, g):
    """64-bit loss, dh, dw and elementwise error bounds of all three."""
    u16 = torch.finfo(h.dtype).eps / 2
    N, d = h.shape
    V = w.shape[0]
    h, w = h.double(), w.double()
    counted = (t != ignore) & (t >= 0) & (t < V)
    z = h @ w.t()
    ez = ((h.abs() @ w.abs().t()) * (d + 16) * 2.0 ** -23).amax(dim=1, keepdim=True)
    lse = torch.logsumexp(z, dim=1, keepdim=True)
    at = t.clamp(0, V - 1)[:, None]
    row = torch.where(counted, (lse - z.gather(1, at))[:, 0], torch.zeros((), dtype=torch.float64, device=h.device))
    erow = (2 * ez + 2.0 ** -21 * (lse.abs() + z.amax(1, keepdim=True).abs() + math.log(V) + 1))[:, 0] * counted
    n = counted.sum().clamp(min=1)
    if reduction == "none":
        loss, eloss, r = row, erow, g.double() * counted
    else:
        k = 1.0 if reduction == "sum" else 1.0 / n
        loss, eloss = row.sum() * k, erow.sum() * k + row.abs().sum() * k * 2.0 ** -23
        r = g.double() * k * counted
    p = torch.exp(z - lse)
    span = (z - lse).abs()  # the exponent's own rounding
    dz = p.clone().scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64)) * r[:, None]
    edz = (p * (3 * ez + 2.0 ** -21 * (span + lse.abs() + 2)) + dz.abs() / r.abs().clamp(min=1e-300)[:, None] * u16
           + 2.0 ** -22) * r.abs()[:, None]
    # fp16: dz is scaled so that the largest row weight is at least 2^13; its subnormals step by 2^-24
    top = r.abs().max()
    small = (top * 2.0 ** -13 * 2.0 ** -25) if u16 < 2.0 ** -9 else 0.0
    edz = edz + small * (r != 0)[:, None]
    K = 2.0 ** -23
    dh, dw = dz @ w, dz.t() @ h
    edh = (edz @ w.abs()) + (V + 64) * K * (dz.abs() @ w.abs())
    edw = (edz.t() @ h.abs()) + (N + 64) * K * (dz.abs().t() @ h.abs())
    tiny = torch.finfo(torch.float16).smallest_normal * 2.0 ** -11 if u16 < 2.0 ** -9 else 1e-38
    edh, edw = edh + (dh.abs() + edh) * u16 + tiny, edw + (dw.abs() + edw) * u16 + tiny
    return (loss, eloss + 1e-12), (dh, edh), (dw, edw)


def _inputs(N, V, d, dtype, seed, device="cuda", ignore=-100):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, d, generator=g) * (2.0 / math.sqrt(d))
    t = torch.randint(0, V, (N,), generator=g)
    h = torch.randn(N, d, generator=g) + w[t]
    t[torch.rand(N, generator=g) < 0.15] = ignore
    return [x.to(device) for x in (h.to(dtype), w.to(dtype), t)]


def _check(name, got, ref, err):
    bad = (got.double() - ref).abs() > err
    if got.dtype == torch.float16:  # a result from 65520 on rounds to infinity (the largest number is 65504, its step 32)
        bad &= ~(got.isinf() & (got.sign() == ref.sign()) & (ref.abs() + err >= 65520))
    assert not bad.any(), (name, int(bad.sum()), float(((got.double() - ref).abs() / err).max()))


def _run(h, w, t, reduction, g, ignore=-100, **kw):
    from llm_research_b200 import ops

    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ops.piecewise_linear_cross_entropy(h, w, t, ignore_index=ignore, reduction=reduction, **kw)
    dh, dw = torch.autograd.grad(loss, (h, w), g.to(loss.dtype))
    return loss.detach(), dh, dw


def _compare(h, w, t, reduction, g, ignore=-100, **kw):
    got = _run(h, w, t, reduction, g, ignore, **kw)
    for name, x, (ref, err) in zip(("loss", "dh", "dw"), got, _exact(h, w, t, ignore, reduction, g)):
        _check(name, x, ref, err)
    return got


# ------------------------------------------------------------------ CPU
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cpu_matches_torch(reduction):
    from llm_research_b200 import ops

    h, w, t = _inputs(20, 37, 6, torch.float64, 0, "cpu")
    h, w = h.requires_grad_(), w.requires_grad_()
    f = lambda a, b: ops.piecewise_linear_cross_entropy(a, b, t, reduction=reduction)  # noqa: E731
    ref = torch.nn.functional.cross_entropy(h @ w.t(), t, reduction=reduction)
    torch.testing.assert_close(f(h, w), ref)
    assert torch.autograd.gradcheck(f, (h, w))


def test_cpu_rows_that_do_not_count():
    from llm_research_b200 import ops

    h, w, _ = _inputs(4, 9, 8, torch.float32, 1, "cpu")
    t = torch.tensor([-1, 9, 3, 10 ** 12])
    rows = ops.piecewise_linear_cross_entropy(h, w, t, reduction="none")
    assert rows[[0, 1, 3]].eq(0).all() and rows[2] > 0
    assert ops.piecewise_linear_cross_entropy(h, w, t) == rows[2]
    assert ops.piecewise_linear_cross_entropy(h, w, t, ignore_index=3) == 0
    assert ops.piecewise_linear_cross_entropy(h.view(2, 2, 8), w, t.view(2, 2), reduction="none").shape == (2, 2)


def test_refusals():
    from llm_research_b200 import ops

    h, w, t = _inputs(4, 9, 8, torch.float32, 1, "cpu")
    with pytest.raises(ValueError, match="reduction"):
        ops.piecewise_linear_cross_entropy(h, w, t, reduction="max")
    with pytest.raises(ValueError, match="targets"):
        ops.piecewise_linear_cross_entropy(h, w, t[:3])
    with pytest.raises(ValueError, match="h \\(..., d\\)"):
        ops.piecewise_linear_cross_entropy(h[:, :4], w, t)
    with pytest.raises(TypeError, match="int64"):
        ops.piecewise_linear_cross_entropy(h, w, t.int())
    with pytest.raises(ValueError, match="piece"):
        ops.piecewise_linear_cross_entropy(h, w, t, piece=0)


# ------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V,d,piece", [(1, 1, 8, None), (1, 300, 64, None), (3, 257, 8, 256), (130, 1000, 72, 304),
                                         (257, 513, 264, 8), (512, 4096, 256, None), (700, 2503, 136, 1024),
                                         (64, 100287, 128, 20000), (1500, 3001, 1024, 768)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_against_64_bits(dtype, N, V, d, piece, reduction):
    h, w, t = _inputs(N, V, d, dtype, N + V)
    g = torch.randn(N, device="cuda") if reduction == "none" else torch.tensor(0.7, device="cuda")
    if N > 1 and reduction == "none":
        g[1] = 0.0
    if N == 1:
        t[0] = V - 1
    a = _compare(h, w, t, reduction, g, piece=piece)
    b = _run(h, w, t, reduction, g, piece=piece)
    for x, y in zip(a, b):
        assert torch.equal(x, y)  # fixed order of every sum


@pytest.mark.gpu
def test_sum_ignore_and_leading_shape():
    from llm_research_b200 import ops

    h, w, t = _inputs(6 * 11, 515, 48, torch.bfloat16, 5, ignore=7)
    _compare(h, w, t, "sum", torch.tensor(-2.0, device="cuda"), ignore=7)
    t[3], t[4], t[5] = -1, 515, 2 ** 40
    _compare(h, w, t, "mean", torch.tensor(1.0, device="cuda"), ignore=7)
    rows = ops.piecewise_linear_cross_entropy(h.view(6, 11, 48), w, t.view(6, 11), ignore_index=7, reduction="none")
    assert rows.shape == (6, 11) and rows.flatten()[[3, 4, 5]].eq(0).all()
    # strided hidden states (the positions but the last), a pitched and an unaligned table
    h3 = h.view(6, 11, 48)[:, :-1]
    want = ops.piecewise_linear_cross_entropy(h3.contiguous(), w, t.view(6, 11)[:, 1:].contiguous())
    assert want == ops.piecewise_linear_cross_entropy(h3, w, t.view(6, 11)[:, 1:])
    wide = torch.zeros(515, 60, device="cuda", dtype=torch.bfloat16)
    for off in (0, 3, 8):
        wide[:, off:off + 48] = w
        assert want == ops.piecewise_linear_cross_entropy(h3, wide[:, off:off + 48], t.view(6, 11)[:, 1:])


@pytest.mark.gpu
def test_no_row_counts_and_no_rows():
    h, w, t = _inputs(40, 300, 64, torch.float16, 6)
    t[:] = -100
    for red, g in (("mean", torch.tensor(1.0)), ("none", torch.ones(40))):
        loss, dh, dw = _run(h, w, t, red, g.cuda())
        assert loss.eq(0).all() and dh.eq(0).all() and dw.eq(0).all()
    loss, dh, dw = _run(h[:0], w, t[:0], "mean", torch.tensor(1.0).cuda())
    assert loss == 0 and dh.shape == (0, 64) and dw.eq(0).all()
    loss, dh, dw = _run(h[:0], w, t[:0], "none", torch.ones(0).cuda())
    assert loss.shape == (0,) and dw.shape == w.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1e-6, 1.0, 3e4])
def test_small_and_large_row_weights(dtype, scale):
    """fp16 keeps the small probabilities of dz whatever the size of the weights."""
    h, w, t = _inputs(200, 900, 64, dtype, 9)
    _compare(h, w, t, "none", torch.randn(200, device="cuda") * scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("weight", [0.7, -3e-5, 1e-35])
def test_one_weight_for_all_rows(dtype, weight):
    """Row losses with one upstream weight (``rows.mean()``) have the gradients of the sum
    with it, to the bit: the weight is not rounded into the 16-bit logits' gradient."""
    h, w, t = _inputs(200, 900, 64, dtype, 21)
    g = torch.full((200,), abs(weight), device="cuda")
    _, dh, dw = _run(h, w, t, "none", g)
    _, dh2, dw2 = _run(h, w, t, "sum", g[0])
    if weight > 1e-30 or weight < 0:
        assert torch.equal(dh, dh2) and torch.equal(dw, dw2)
    _compare(h, w, t, "none", weight * g / g[0])


@pytest.mark.gpu
def test_extreme_logits():
    """Peaked rows, and infinities in rows that count: the loss of the other rows stays."""
    from llm_research_b200 import ops

    h, w, t = _inputs(64, 700, 32, torch.bfloat16, 10)
    big = h.clone()
    big[:8] *= 200.0
    _compare(big, w, t, "none", torch.ones(64, device="cuda"))
    want = ops.piecewise_linear_cross_entropy(h, w, t, reduction="none")
    bad = h.clone()
    bad[5, 0], bad[6, 1] = float("nan"), float("inf")
    got = ops.piecewise_linear_cross_entropy(bad, w, t, reduction="none")
    keep = [i for i in range(64) if i not in (5, 6)]
    assert torch.equal(got[keep], want[keep])
    for i in (5, 6):
        assert (t[i] == -100 and got[i] == 0) or got[i].isnan()


@pytest.mark.gpu
def test_one_gradient_only_and_frozen():
    from llm_research_b200 import ops

    h, w, t = _inputs(300, 1200, 64, torch.bfloat16, 11)
    _, dh, dw = _run(h, w, t, "mean", torch.tensor(1.0).cuda(), piece=512)
    for need_h, need_w in ((True, False), (False, True)):
        a, b = h.detach().requires_grad_(need_h), w.detach().requires_grad_(need_w)
        loss = ops.piecewise_linear_cross_entropy(a, b, t, piece=512)
        loss.backward()
        assert torch.equal(a.grad, dh) if need_h else a.grad is None
        assert torch.equal(b.grad, dw) if need_w else b.grad is None
    with torch.no_grad():
        assert torch.equal(ops.piecewise_linear_cross_entropy(h, w, t), loss.detach())


@pytest.mark.gpu
def test_graph_replay_and_other_stream():
    h, w, t = _inputs(300, 1200, 64, torch.bfloat16, 12)
    g = torch.tensor(1.0, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = _run(h, w, t, "mean", g, piece=512)
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = _run(h, w, t, "mean", g, piece=512)
    gr.replay()
    for x, y in zip(out, first):
        assert torch.equal(x, y)
    h.copy_(h.roll(1, 0))
    gr.replay()
    for x, y in zip(out, _run(h, w, t, "mean", g, piece=512)):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_cuda_refusals():
    from llm_research_b200 import ops

    h, w, t = _inputs(4, 9, 12, torch.bfloat16, 1)
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.piecewise_linear_cross_entropy(h, w, t)
    h, w, t = _inputs(4, 9, 16, torch.bfloat16, 1)
    with pytest.raises(TypeError, match="both be bf16"):
        ops.piecewise_linear_cross_entropy(h, w.half(), t)
    with pytest.raises(TypeError, match="both be bf16"):
        ops.piecewise_linear_cross_entropy(h.float(), w.float(), t)
    with pytest.raises(RuntimeError, match="one CUDA device"):
        ops.piecewise_linear_cross_entropy(h, w, t.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("up", [float("inf"), float("-inf"), float("nan")])
def test_upstream_infinity_does_not_reach_rows_that_do_not_count(dtype, reduction, up):
    """As in ``F.cross_entropy``: the gradient of an ignored row is 0 whatever arrives."""
    h, w, t = _inputs(70, 300, 64, dtype, 13)
    skip = t == -100
    _, dh, dw = _run(h, w, t, reduction, torch.tensor(up, device="cuda"))
    assert skip.any() and dh[skip].eq(0).all()
    assert not dh[~skip].isfinite().any() and not dw.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_weight_without_a_value_stays_in_its_row(dtype, bad):
    """The other rows' dh has the bits that it has beside a finite weight."""
    h, w, t = _inputs(70, 300, 64, dtype, 14)
    t[:4] = torch.tensor([5, 6, 7, -100], device="cuda")
    g = torch.full((70,), 50.0, device="cuda")
    g[9:] += torch.rand(61, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    _, want, _ = _run(h, w, t, "none", g)
    g[0], g[3] = bad, bad
    _, dh, dw = _run(h, w, t, "none", g)
    assert torch.equal(dh[1:], want[1:]) and dh[3].eq(0).all()
    assert not dh[0].isfinite().any() and not dw.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_any_one_weight_for_all_rows(dtype):
    """``test_one_weight_for_all_rows`` at weights whose reciprocal times themselves is not
    1 in fp32 (1 / 41 and about one number in seven)."""
    h, w, t = _inputs(200, 900, 64, dtype, 21)
    for weight in (1 / 41, 1 / 47, 1 / 55, 0.83):
        g = torch.full((200,), weight, device="cuda")
        _, dh, dw = _run(h, w, t, "none", g)
        _, dh2, dw2 = _run(h, w, t, "sum", g[0])
        assert torch.equal(dh, dh2) and torch.equal(dw, dw2)


@pytest.mark.gpu
def test_contiguous_operands_that_start_anywhere():
    """Contiguous h and w off a 16-byte boundary (slices of a flat buffer)."""
    h, w, t = _inputs(33, 130, 24, torch.bfloat16, 15)
    g = torch.tensor(1.0, device="cuda")
    want = _run(h, w, t, "mean", g)

    def moved(x, off):
        flat = torch.empty(x.numel() + 8, device="cuda", dtype=x.dtype)
        return flat[off:off + x.numel()].view(x.shape).copy_(x)

    for off in (1, 4):
        for a, b in ((moved(h, off), w), (h, moved(w, off)), (moved(h, off), moved(w, off))):
            for x, y in zip(_run(a, b, t, "mean", g), want):
                assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("N,V", [(40000, 5003), (140000, 1500), (1, 100287), (3, 9)])
def test_default_pieces(N, V):
    """The default width where its buffer takes the vocabulary in two pieces, and in one."""
    h, w, t = _inputs(N, V, 16, torch.bfloat16, 16)
    _compare(h, w, t, "sum", torch.tensor(1.0, device="cuda"))
