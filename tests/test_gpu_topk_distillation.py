"""Distillation from a teacher's top logits against the formula in 64 bits.

Tolerances (``T`` the temperature).  The log-sum-exp of V fp32 terms is off by a few
fp32 steps of its parts (the maximum / T, ln of the sum) and 2^-21 for the
exponentials; the loss multiplies by ``T^2`` and sums K terms of weight p.  An
element of the gradient ``c (q - p)`` is off by the exponent's rounding,
``2^-22 (|x - m| / T + ln V + 4)`` relative to q, 2^-22 relative to p, and half a
step of its type."""

import math

import pytest
import torch

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _exact(x, teacher, ids, T, reduction, g):
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    V, K = x.shape[-1], ids.shape[-1]
    x, teacher, ids = x.reshape(-1, V).double(), teacher.reshape(-1, K).double(), ids.reshape(-1, K).long()
    kept = (ids >= 0) & (ids < V) & (teacher != -math.inf)
    some = kept.any(1)
    y = torch.where(kept, teacher / T, torch.full_like(teacher, -1e300))
    y = torch.where(some[:, None], y, torch.zeros_like(y))
    p = torch.softmax(y, 1) * kept
    at = ids.clamp(0, V - 1)
    logq = torch.log_softmax(x / T, 1)
    lq, zero = logq.gather(1, at), torch.zeros_like(p)
    lp = torch.log_softmax(y, 1)
    use = p > 0
    term = torch.where(use, p * (lp - lq), zero).sum(1)
    size = torch.where(use, p * (lp.abs() + lq.abs() + ((x.amax(1, keepdim=True) / T).abs())), zero).sum(1)
    rows, erows = T * T * term * some, T * T * (size + math.log(V) + 4) * 2.0 ** -20 * some
    n = some.sum().clamp(min=1)
    if reduction == "none":
        loss, eloss, r = rows, erows, g.double().reshape(-1) * some
    else:
        k = 1.0 if reduction == "sum" else 1.0 / n
        loss, eloss, r = rows.sum() * k, erows.sum() * k, g.double() * k * some
    q = torch.exp(logq)
    pd = torch.zeros_like(x).scatter_add_(1, at, p)
    dx = T * r[:, None] * (q - pd)
    span = (x - x.amax(1, keepdim=True)).abs() / T
    edx = T * r.abs()[:, None] * (torch.nan_to_num(q * (span + math.log(V) + 4), 0.0) * 2.0 ** -21 + (pd + q) * 2.0 ** -20)
    edx = edx + (dx.abs() + edx) * half + tiny
    return (loss, eloss + 1e-12), (dx, edx)


def _inputs(N, V, K, dtype, seed, ragged=True, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, V, generator=g) * 2
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)])
    teacher = (torch.randn(N, K, generator=g) * 2 + 5).sort(1, descending=True)[0]
    x.scatter_add_(1, ids, teacher * 0.7)
    if ragged:
        kept = torch.randint(0, K + 1, (N, 1), generator=g)
        kept[0] = K
        ids = torch.where(torch.arange(K) < kept, ids, -1)
    return [t.to(device) for t in (x.to(dtype), teacher.to(dtype), ids)]


def _run(x, teacher, ids, T, reduction, g):
    from llm_research_b200 import ops

    x = x.detach().requires_grad_()
    loss = ops.topk_distillation(x, teacher, ids, T, reduction)
    dx, = torch.autograd.grad(loss, x, g.to(loss.dtype))
    return loss.detach(), dx


def _check(name, got, ref, err):
    ref = ref.reshape(got.shape)
    bad = ~((got.double() - ref).abs() <= err.reshape(got.shape))
    assert not bad.any(), (name, int(bad.sum()), float(((got.double() - ref).abs() / err.reshape(got.shape)).max()))


def _compare(x, teacher, ids, T, reduction, g):
    loss, dx = _run(x, teacher, ids, T, reduction, g)
    (l, el), (d, ed) = _exact(x, teacher, ids, T, reduction, g)
    _check("loss", loss, l, el)
    _check("dx", dx, d, ed)
    assert dx.shape == x.shape and dx.dtype == x.dtype and loss.dtype == torch.float32
    return loss, dx


# ------------------------------------------------------------------ CPU
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cpu_formula_and_gradient(reduction):
    from llm_research_b200 import ops

    x, teacher, ids = _inputs(9, 31, 5, torch.float64, 0, device="cpu")
    x.requires_grad_()
    g = torch.randn(9, dtype=torch.float64) if reduction == "none" else torch.tensor(1.3, dtype=torch.float64)
    loss = ops.topk_distillation(x, teacher, ids, 2.0, reduction)
    dx, = torch.autograd.grad(loss, x, g)
    (l, _), (d, _) = _exact(x.detach(), teacher, ids, 2.0, reduction, g)
    torch.testing.assert_close(loss, l)
    torch.testing.assert_close(dx, d)
    assert torch.autograd.gradcheck(lambda t: ops.topk_distillation(t, teacher, ids, 2.0, reduction), (x,))


def test_cpu_is_the_full_distillation_when_all_tokens_are_listed():
    from genesis.verifier.distillation import VerificationDistillation
    from llm_research_b200 import ops

    g = torch.Generator().manual_seed(2)
    s, t = torch.randn(6, 13, generator=g), torch.randn(6, 13, generator=g)
    ids = torch.arange(13).expand(6, 13)
    full = VerificationDistillation(4, 4).temperature_scaled_loss(s, t, 3.0)
    torch.testing.assert_close(ops.topk_distillation(s, t, ids, 3.0), full)


def test_refusals():
    from llm_research_b200 import ops

    x, teacher, ids = _inputs(3, 9, 2, torch.float32, 0, device="cpu")
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            ops.topk_distillation(x, teacher, ids, bad)
    with pytest.raises(ValueError, match="reduction"):
        ops.topk_distillation(x, teacher, ids, 1.0, "batch")
    with pytest.raises(TypeError, match="int64 or int32"):
        ops.topk_distillation(x, teacher, ids.float())
    with pytest.raises(ValueError, match="leading shape"):
        ops.topk_distillation(x, teacher[:2], ids[:2])
    with pytest.raises(ValueError, match="leading shape"):
        ops.topk_distillation(x, teacher[:, :1], ids)
    with pytest.raises(ValueError, match="leading shape"):
        ops.topk_distillation(x, teacher[:, :0], ids[:, :0])


# ------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,K", [(1, 1, 1), (1, 100287, 32), (2, 5, 5), (3, 31, 7), (40, 512, 64), (33, 1001, 255),
                                   (17, 32000, 16), (700, 1023, 1), (5, 40000, 1024)])
@pytest.mark.parametrize("reduction,T", [("mean", 1.0), ("none", 2.5)])
def test_against_64_bits(dtype, N, V, K, reduction, T):
    x, teacher, ids = _inputs(N, V, K, dtype, N + V + K)
    g = torch.randn(N, device="cuda") if reduction == "none" else torch.tensor(0.6, device="cuda")
    a = _compare(x, teacher, ids, T, reduction, g)
    b = _run(x, teacher, ids.int(), T, reduction, g)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_views_leading_shapes_and_mixed_types():
    from llm_research_b200 import ops

    for V in (512, 501):  # aligned rows, and rows that start anywhere
        x, teacher, ids = _inputs(4 * 6, V, 9, torch.bfloat16, 4)
        x, teacher, ids = x.view(4, 6, V), teacher.float().view(4, 6, 9), ids.view(4, 6, 9)
        one = torch.ones((), device="cuda")
        _compare(x[:, :-1], teacher[:, 1:], ids[:, 1:], 2.0, "sum", one)
        _compare(x.transpose(0, 1), teacher.transpose(0, 1), ids.transpose(0, 1), 2.0, "mean", one)
        _compare(x[..., ::2], teacher, ids, 1.0, "mean", one)
        _compare(x[0, 0], teacher[0, 0], ids[0, 0], 1.0, "none", one)
        rows = ops.topk_distillation(x.view(2, 2, 6, V), teacher.view(2, 2, 6, 9), ids.view(2, 2, 6, 9), 1.0, "none")
        assert rows.shape == (2, 2, 6)
        loss = ops.topk_distillation(x.requires_grad_(), teacher, ids)  # a broadcast upstream gradient
        (loss.expand(3).sum()).backward()
        _check("dx", x.grad, *_exact(x.detach(), teacher, ids, 1.0, "mean", 3 * one)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_masks_and_extremes(dtype):
    x, teacher, ids = _inputs(12, 300, 6, dtype, 7, ragged=False)
    low = torch.finfo(dtype).min
    ids[0] = -1                                   # no teacher at all
    ids[1, 2], ids[1, 3] = 300, 2 ** 40           # tokens outside the vocabulary
    teacher[2, 1] = float("-inf")                 # listed, without weight
    teacher[3] = float("-inf")                    # all of them: an empty row
    ids[4, 1:], teacher[4, 1:] = -1, float("nan")  # what stands in padding is not looked at
    x[5, 100:200] = float("-inf")                 # masked vocabulary
    ids[5] = torch.arange(6, device="cuda")
    x[6, 10:] = low                               # masked by the lowest value
    ids[6] = torch.arange(6, device="cuda")
    x[7] = low                                    # a whole row of it: uniform
    x[0, 3], x[3, 4] = float("nan"), float("inf")  # rows without a teacher do not look at x
    ids[8] = ids[8, 0]                            # one token six times
    ids[9, 4] = ids[9, 1]
    g = torch.randn(12, device="cuda")
    loss, dx = _run(x, teacher, ids, 1.5, "none", g)
    clean = x.clone()
    clean[0, 3] = clean[3, 4] = 0
    (l, el), (d, ed) = _exact(clean, torch.where(teacher.isnan(), 0, teacher), ids, 1.5, "none", g)
    live = [i for i in range(12) if i != 7]
    _check("loss", loss[live], l[live], el[live])
    _check("dx", dx[live], d[live], ed[live])
    assert loss[[0, 3]].eq(0).all() and dx[[0, 3]].eq(0).all()
    # row 7: softmax is 1 / V, the loss sum p (ln p + ln V)
    _check("loss", loss[7:8], l[7:8], el[7:8].clamp(max=1e-3))
    _check("dx", dx[7:8], d[7:8], ed[7:8])


@pytest.mark.gpu
def test_nan_that_counts_and_minus_infinity_at_a_listed_token():
    x, teacher, ids = _inputs(4, 300, 6, torch.float32, 8, ragged=False)
    x[0, 5] = float("nan")
    teacher[1, 2] = float("nan")
    x[2, ids[2, 0]] = float("-inf")
    loss, dx = _run(x, teacher, ids, 1.0, "none", torch.ones(4, device="cuda"))
    assert loss[0].isnan() and loss[1].isnan() and loss[2] == float("inf") and loss[3].isfinite()
    assert dx[0].isnan().all() and dx[3].isfinite().all() and dx[2].isfinite().all()


@pytest.mark.gpu
def test_nothing_counts_and_no_rows():
    x, teacher, ids = _inputs(5, 64, 3, torch.bfloat16, 9)
    loss, dx = _run(x, teacher, torch.full_like(ids, -1), 1.0, "mean", torch.tensor(1.0, device="cuda"))
    assert loss == 0 and dx.eq(0).all()
    loss, dx = _run(x[:0], teacher[:0], ids[:0], 1.0, "mean", torch.tensor(1.0, device="cuda"))
    assert loss == 0 and dx.shape == (0, 64)
    loss, dx = _run(x[:0], teacher[:0], ids[:0], 1.0, "none", torch.ones(0, device="cuda"))
    assert loss.shape == (0,)


@pytest.mark.gpu
def test_graph_replay_and_other_stream():
    from llm_research_b200 import ops

    x, teacher, ids = _inputs(50, 2000, 8, torch.bfloat16, 10)
    g = torch.tensor(1.0, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = _run(x, teacher, ids, 2.0, "mean", g)
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = _run(x, teacher, ids, 2.0, "mean", g)
    gr.replay()
    assert torch.equal(out[0], first[0]) and torch.equal(out[1], first[1])
    with torch.no_grad():
        assert torch.equal(ops.topk_distillation(x, teacher, ids, 2.0), first[0])
    x.copy_(x.roll(1, 0))
    gr.replay()
    again = _run(x, teacher, ids, 2.0, "mean", g)
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


@pytest.mark.gpu
def test_cuda_refusals():
    from llm_research_b200 import ops

    x, teacher, ids = _inputs(3, 2000, 2, torch.float32, 0)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        ops.topk_distillation(x.double(), teacher, ids)
    with pytest.raises(ValueError, match="at most 1024"):
        ops.topk_distillation(x, teacher.repeat(1, 600), ids.repeat(1, 600))
    with pytest.raises(RuntimeError, match="one CUDA device"):
        ops.topk_distillation(x, teacher.cpu(), ids)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,K", [(2500, 301, 5), (1776, 1024, 128), (1777, 16384, 33), (1800, 515, 129)])
def test_many_rows(dtype, N, V, K):
    """Rows by warps (lists up to 128 entries, short rows) and by blocks; a list with repetitions."""
    x, teacher, ids = _inputs(N, V, K, dtype, N)
    ids[7] = ids[7, 0]
    ids[8, -1] = ids[8, 0]
    _compare(x, teacher, ids, 1.3, "none", torch.randn(N, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,K", [(3, 60000, 40), (40, 1000, 7), (1800, 600, 7)])
def test_masked_tokens_and_offsets_cost_no_precision(dtype, N, V, K):
    """Large negative logits at the first tokens (a mask), a whole eighth of the
    vocabulary or a listed token, and rows with a common offset."""
    x, teacher, ids = _inputs(N, V, K, dtype, N, ragged=False)
    mask = -6e4 if dtype == torch.float16 else -1e9
    ids.clamp_(min=V // 8)  # listed tokens are not masked (a few are listed twice now)
    x[:, 0] = mask
    x[1, :V // 8] = mask
    x[2] += 64.0
    x[2, :3] = mask
    _compare(x, teacher, ids, 1.7, "none", torch.randn(N, device="cuda"))


def _compare_rows(loss, dx, x, teacher, ids, T, g):
    """Row losses and their gradient against ``_exact``.  Its bound leaves out that the
    exponent (t - t_max) log2(e) / T of a probability p = e^(...) / S is rounded four times in
    fp32 (log2 e, its division by T, the difference, the product), each by up to 2^-24 of it:
    relative to p that is (t_max - t) / T 2^-22, 2^-18.5 for T = 0.5 and logits 6 apart.  And
    it leaves out that an exponential, or a product with it, below the smallest normal
    number 2^-126 is 0."""
    (l, el), (d, ed) = _exact(x, teacher, ids, T, "none", g)
    y = teacher.double() / T
    span = y.amax(1, keepdim=True) - y
    ep = T * g.double().abs()[:, None] * torch.softmax(y, 1) * span * 2.0 ** -22
    ed = ed + torch.zeros_like(ed).scatter_add_(1, ids, ep) + (T * g.double().abs()[:, None] + 1) * 2.0 ** -126
    _check("loss", loss, l, el)
    _check("dx", dx, d, ed)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,V,K", [(12, 60000, 40), (40, 1001, 7), (1800, 600, 7)])
@pytest.mark.parametrize("mask", [-1e10, -1e12, -1e20, -1e30, None])
@pytest.mark.parametrize("T", [0.5, 1.0, 2.0, 3.5])
def test_masks_of_any_size(dtype, N, V, K, mask, T):
    """Masks from -1e10 to the type's lowest value (None) at the first, the last and a
    listed token, over a stretch, and rows that hold nothing else.

    The loss and the gradient do not change with a row's offset.  The rows of large
    values are compared with the same rows less their largest value: the differences are
    exact (equal values, values within a factor of two, or a mask that takes the other
    one in whole), and the bounds are those of the small values."""
    x, teacher, ids = _inputs(N, V, K, dtype, N, ragged=False)
    low = torch.finfo(dtype).min if mask is None else mask
    ids.clamp_(min=V // 8, max=V - 2)  # the listed tokens are not masked
    x[0, 0] = low
    x[1, -1] = low
    x[2, ids[2, 0]] = max(low, -1e30)  # times T, the lowest value would leave fp32
    x[3, :V // 8] = low
    x[4, 0], x[4, -1], x[4, 1:9] = low, low, float("-inf")
    x[5] = low                         # uniform
    x[6] = low
    x[6, V // 2:] = low * (1 - 2.0 ** -6)  # uniform over a half, the rest adds nothing
    ids[6] = V // 2 + torch.arange(K, device="cuda")
    x[7] = abs(low)
    g = torch.randn(N, device="cuda")
    loss, dx = _run(x, teacher, ids, T, "none", g)
    near = x.clone()
    near[5:8] -= x[5:8].amax(1, keepdim=True)
    _compare_rows(loss, dx, near, teacher, ids, T, g)


@pytest.mark.gpu
@pytest.mark.parametrize("N,V", [(26, 40000), (26, 777), (1800, 300)])
@pytest.mark.parametrize("T", [0.01, 1.0, 3.5])
def test_large_offsets(N, V, T):
    """Rows around an offset of 2^14 to 2^26, either sign: each small difference is exact
    in fp32 there, and costs no precision."""
    x, teacher, ids = _inputs(N, V, 9, torch.float32, 5, ragged=False)
    step = torch.randint(0, 8, (N, V), device="cuda", generator=torch.Generator("cuda").manual_seed(2)).float()
    for r in range(26):
        offset = 2.0 ** (14 + r // 2)
        unit = max(1.0, offset * 2.0 ** -22)
        x[r] = (offset if r % 2 else -offset) + unit * step[r]
    g = torch.randn(N, device="cuda")
    loss, dx = _run(x, teacher, ids, T, "none", g)
    near = x - x.amax(1, keepdim=True)
    _compare_rows(loss, dx, near, teacher, ids, T, g)


def test_temperature_that_leaves_fp32_is_refused():
    """On CUDA the temperature and its square are fp32 numbers."""
    from llm_research_b200.ops.distill import check_cuda_temperature

    for T in (1e-18, 1e-3, 1.0, 1e18):
        check_cuda_temperature(T)
    for T in (1e-46, 1e-20, 1e20, 1e39):
        with pytest.raises(ValueError, match="temperature"):
            check_cuda_temperature(T)


@pytest.mark.gpu
def test_temperature_that_leaves_fp32_is_refused_on_cuda():
    from llm_research_b200 import ops

    x, teacher, ids = _inputs(3, 50, 2, torch.float32, 0)
    for T in (1e-46, 1e-20, 1e20, 1e39):
        with pytest.raises(ValueError, match="temperature"):
            ops.topk_distillation(x, teacher, ids, T)


def test_cpu_rows_without_a_teacher_do_not_look_at_the_logits():
    """Loss 0 and gradient 0 there, as on CUDA, whatever the logits hold."""
    from llm_research_b200 import ops

    x, teacher, ids = _inputs(4, 31, 5, torch.float32, 3, ragged=False, device="cpu")
    ids[1], teacher[2] = -1, float("-inf")
    x[1, 3], x[2, 4] = float("nan"), float("inf")
    x[3, 30] = float("-inf")
    ids[3].clamp_(max=29)
    for reduction in ("mean", "sum", "none"):
        y = x.clone().requires_grad_()
        loss = ops.topk_distillation(y, teacher, ids, 1.0, reduction)
        dx, = torch.autograd.grad(loss.sum(), y)
        assert loss.isfinite().all() and dx.isfinite().all() and dx[1:3].eq(0).all()


@pytest.mark.parametrize("T", [0.25, 1.0])
def test_cpu_row_of_the_lowest_value(T):
    """Uniform, also where the value over T leaves fp32."""
    from llm_research_b200 import ops

    x, teacher, ids = _inputs(2, 31, 5, torch.float32, 3, ragged=False, device="cpu")
    x[1] = 0.0
    want = ops.topk_distillation(x, teacher, ids, T, "none")
    x[1] = torch.finfo(torch.float32).min
    torch.testing.assert_close(ops.topk_distillation(x, teacher, ids, T, "none"), want)
