"""The vocabulary operators as they are used together: one training step from token
ids to the loss over a tied table (lookup, head loss in pieces, distillation), and
HLRT's loss in pieces.

The run is compared with the same step in 64 bits on the same 16-bit values.  Each
16-bit tensor on the way (embeddings, hidden states, logits, and every gradient)
adds half a step, relative 2^-9 for bf16, to what feeds on it; no path crosses more
than six of them, and independent roundings of many summands do not add up beyond
their largest, so 6 * 2^-9 of the 2-norm bounds each gradient."""

import pytest
import torch


def _step(ids, w, mix, targets, teacher, tids, embed, ce, kd):
    x = embed(ids, w)
    h = torch.tanh(x @ mix)
    logits = h @ w.t()
    return ce(h, w, targets) + 0.5 * kd(logits, teacher, tids)


def _plain_ce(h, w, t):
    return torch.nn.functional.cross_entropy(h @ w.t(), t, ignore_index=-100)


def _plain_kd(x, teacher, ids, T=2.0):
    kept = ids >= 0
    some = kept.any(1)
    y = (teacher / T).masked_fill(~kept, -float("inf"))
    y = torch.where(some[:, None], y, torch.zeros_like(y))
    p = torch.softmax(y, 1) * kept
    q = torch.log_softmax(x / T, 1).gather(1, ids.clamp(min=0))
    return T * T * (torch.special.xlogy(p, p) - p * q).masked_fill(~kept, 0).sum() / some.sum()


def _inputs(device, dtype, N=96, V=1003, d=64, K=7):
    g = torch.Generator().manual_seed(3)
    w = (0.3 * torch.randn(V, d, generator=g)).to(dtype)
    mix = (torch.randn(d, d, generator=g) / 8).to(dtype)
    ids = torch.randint(0, V, (N,), generator=g)
    ids[::5] = 17
    targets = torch.randint(0, V, (N,), generator=g)
    targets[::9] = -100
    tids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)])
    tids[3] = -1
    tids[5, 4:] = -1
    teacher = torch.randn(N, K, generator=g).to(dtype)
    return [t.to(device) for t in (ids, w, mix, targets, teacher, tids)]


def _grads(f, w, mix):
    w, mix = w.detach().clone().requires_grad_(), mix.detach().clone().requires_grad_()
    loss = f(w, mix)
    return (loss.detach(), *torch.autograd.grad(loss, (w, mix)))


def _both(device, dtype):
    from llm_research_b200 import ops

    ids, w, mix, targets, teacher, tids = _inputs(device, dtype)
    got = _grads(lambda a, b: _step(ids, a, b, targets, teacher, tids,
                                    lambda i, t: ops.embedding(i, t, scale=8.0),
                                    ops.piecewise_linear_cross_entropy,
                                    lambda x, t, i: ops.topk_distillation(x, t, i, 2.0)), w, mix)
    ref = _grads(lambda a, b: _step(ids, a, b, targets, teacher.double(), tids, lambda i, t: 8.0 * t[i],
                                    _plain_ce, _plain_kd), w.double(), mix.double())
    return got, ref


def test_step_cpu():
    got, ref = _both("cpu", torch.float64)
    for a, b in zip(got, ref):
        torch.testing.assert_close(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_step_gpu(dtype):
    got, ref = _both("cuda", dtype)
    tol = 6 * torch.finfo(dtype).eps / 2
    for a, b in zip(got, ref):
        assert (a.double() - b).norm() <= tol * b.norm()
    for a, b in zip(got, _both("cuda", dtype)[0]):  # the three operators are deterministic
        assert (a.double() - b.double()).norm() <= tol * b.double().norm()


@pytest.mark.gpu
def test_step_captured_and_replayed():
    """A whole step in a graph; replayed on other tokens it gives what the eager step gives."""
    from llm_research_b200 import ops

    ids, w, mix, targets, teacher, tids = _inputs("cuda", torch.bfloat16)
    w.requires_grad_()

    def step():
        x = ops.embedding(ids, w, scale=8.0)
        h = torch.tanh(x)
        loss = ops.piecewise_linear_cross_entropy(h, w, targets) + ops.topk_distillation(h @ w.t(), teacher, tids, 2.0)
        dw, = torch.autograd.grad(loss, w)
        return loss.detach(), dw

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for shift in (0, 5):
        ids.copy_(ids.roll(shift))
        targets.copy_(targets.roll(shift))
        graph.replay()
        want = step()
        torch.testing.assert_close(out[0], want[0])
        torch.testing.assert_close(out[1].float(), want[1].float(), rtol=2 ** -7, atol=1e-6)


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls in flight on two streams share no workspace: the results are those of one after the other."""
    from llm_research_b200 import ops

    def inputs(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        ids = torch.randint(0, 5000, (9000,), device="cuda", generator=g)
        w = (0.1 * torch.randn(5000, 128, device="cuda", generator=g)).bfloat16().requires_grad_()
        h = torch.randn(700, 128, device="cuda", generator=g).bfloat16().requires_grad_()
        x = torch.randn(700, 5000, device="cuda", generator=g).bfloat16().requires_grad_()
        t = torch.randint(0, 5000, (700,), device="cuda", generator=g)
        te = torch.randn(700, 20, device="cuda", generator=g)
        ti = torch.randint(0, 5000, (700, 20), device="cuda", generator=g)
        dy = torch.randn(9000, 128, device="cuda", generator=g).bfloat16()
        return ids, w, h, x, t, te, ti, dy

    def run(ids, w, h, x, t, te, ti, dy):
        one = torch.ones((), device="cuda")
        dw, = torch.autograd.grad(ops.embedding(ids, w, 2.0), w, dy)
        ce = torch.autograd.grad(ops.piecewise_linear_cross_entropy(h, w, t, piece=1024), (h, w), one)
        dx, = torch.autograd.grad(ops.topk_distillation(x, te, ti, 2.0), x, one)
        return dw, *ce, dx

    sets = [inputs(s) for s in (1, 2)]
    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k] = run(*sets[k])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for u, v in zip(a, b):
            assert torch.equal(u, v)


@pytest.mark.gpu
def test_gradients_of_these_gradients():
    """The lookup can be differentiated twice, the two losses say that they cannot."""
    from llm_research_b200 import ops

    ids, w, mix, targets, teacher, tids = _inputs("cuda", torch.float16)
    h = (0.1 * torch.randn(96, 64, device="cuda")).half().requires_grad_()
    for loss in (ops.piecewise_linear_cross_entropy(h, w, targets),
                 ops.topk_distillation(h @ w.t(), teacher, tids)):
        dh, = torch.autograd.grad(loss, h, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            (loss.sum() + dh.float().square().sum()).backward()


def test_hlrt_loss_in_pieces():
    from genesis.model.hlrt import HLRT
    from genesis.training.train_phase1_bootstrap import ntp_objective
    from llm_research_b200.models.presets import build_hlrt_config

    cfg = build_hlrt_config("toy")
    ids = torch.randint(0, cfg.vocab_size, (2, 48), generator=torch.Generator().manual_seed(1))
    res = []
    for how in (True, "pieces"):
        torch.manual_seed(0)
        m = HLRT(cfg)
        loss = ntp_objective({"hlrt": m}, None, {"input_ids": ids, "fused_lm_loss": how})
        loss.backward()
        res.append((loss.detach(), {n: p.grad for n, p in m.named_parameters() if p.grad is not None}))
    torch.testing.assert_close(res[0][0], res[1][0])
    for n, g in res[0][1].items():
        torch.testing.assert_close(res[1][1][n], g, atol=1e-5, rtol=1e-4, msg=n)
    m.eval()
    with torch.no_grad():
        labels = torch.cat([ids[:, 1:], torch.full((2, 1), -100)], 1)
        rows = m(ids, labels=labels, lm_loss="pieces", lm_reduction="none")["lm_loss"]
        logits = m(ids)["logits"]
    ref = torch.nn.functional.cross_entropy(logits.flatten(0, 1), labels.flatten(), reduction="none").view(2, 48)
    assert rows.shape == (2, 48)
    torch.testing.assert_close(rows, ref)
    with pytest.raises(ValueError, match="lm_loss"):
        m(ids, labels=labels, lm_loss="columns")
    with pytest.raises(ValueError, match="lm_reduction"):
        m(ids, labels=labels, lm_reduction="none")


@pytest.mark.gpu
def test_hlrt_trains_on_the_loss_in_pieces():
    """bf16 HLRT on the GPU: the piecewise loss against the row-chunked one (whose logits
    are rounded to bf16, relative 2^-9 of values below 8 here)."""
    from genesis.model.hlrt import HLRT
    from llm_research_b200.models.presets import build_hlrt_config

    cfg = build_hlrt_config("toy")
    torch.manual_seed(0)
    m = HLRT(cfg).to("cuda", torch.bfloat16)
    ids = torch.randint(0, cfg.vocab_size, (2, 64), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    labels = torch.cat([ids[:, 1:], ids.new_full((2, 1), -100)], 1)
    grads, losses = [], []
    for how in ("rows", "pieces"):
        m.zero_grad(set_to_none=True)
        out = m(ids, labels=labels, lm_loss=how)
        out["lm_loss"].backward()
        losses.append(float(out["lm_loss"].detach()))
        grads.append(m.embeddings.weight.grad.float())
    assert abs(losses[0] - losses[1]) <= 8 * 2 ** -9
    assert (grads[0] - grads[1]).norm() <= 0.05 * grads[0].norm()
    assert torch.isfinite(grads[1]).all()


@pytest.mark.gpu
def test_verifier_distillation_from_a_stored_list():
    from genesis.verifier.distillation import VerificationDistillation

    d = VerificationDistillation(8, 4).cuda()
    g = torch.Generator("cuda").manual_seed(4)
    student = torch.randn(3, 5, 300, device="cuda", generator=g).requires_grad_()
    teacher = torch.randn(3, 5, 300, device="cuda", generator=g)
    top, ids = teacher.topk(300, dim=-1)  # the whole vocabulary: the full-vocabulary loss
    full = d.temperature_scaled_loss(student.reshape(-1, 300), teacher.reshape(-1, 300), 2.0)
    loss = d.topk_loss(student, top, ids, 2.0)
    torch.testing.assert_close(loss, full, rtol=1e-5, atol=1e-6)
    a, b = torch.autograd.grad(loss, student)[0], torch.autograd.grad(full, student)[0]
    torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-7)


@pytest.mark.gpu
def test_losses_changed_in_place():
    """``loss /= steps`` before the backward, as accumulation loops do."""
    from llm_research_b200 import ops

    ids, w, mix, targets, teacher, tids = _inputs("cuda", torch.bfloat16)
    h = (0.1 * torch.randn(96, 64, device="cuda")).bfloat16().requires_grad_()
    x = (h @ w.t()).detach().requires_grad_()
    for leaf, f in ((h, lambda red: ops.piecewise_linear_cross_entropy(h, w, targets, reduction=red)),
                    (x, lambda red: ops.topk_distillation(x, teacher, tids, reduction=red))):
        for red in ("mean", "sum", "none"):
            up = torch.ones((), device="cuda") if red != "none" else torch.ones(96, device="cuda")
            want, = torch.autograd.grad(f(red), leaf, up / 4)
            loss = f(red)
            loss /= 4
            got, = torch.autograd.grad(loss, leaf, up)
            assert torch.equal(got, want)
    out = ops.embedding(ids.view(8, 12), w.requires_grad_())
    out *= 2
    dw, = torch.autograd.grad(out.float().sum(), w)
    assert dw[17, 0] == 2 * float((ids == 17).sum())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Tables, hidden states and logits of more than 2^31 elements."""
    from llm_research_b200 import ops

    V, d = 1100003, 2048
    g = torch.Generator("cuda").manual_seed(6)
    w = torch.empty(V, d, device="cuda", dtype=torch.bfloat16)
    for b in range(0, V, 1 << 17):
        w[b:b + (1 << 17)] = torch.randn(min(1 << 17, V - b), d, device="cuda", generator=g) / d ** 0.5
    w.requires_grad_()
    ids = torch.tensor([V - 1, 0, V - 1, 1048577, 5], device="cuda")
    out = ops.embedding(ids, w)
    assert torch.equal(out, w[ids])
    dy = torch.randn(5, d, device="cuda", generator=g).bfloat16()
    dw, = torch.autograd.grad(out, w, dy)
    assert torch.equal(dw[[0, 1048577, 5]], dy[[1, 3, 4]])
    assert torch.equal(dw[V - 1], (dy[0].float() + dy[2].float()).bfloat16())
    assert dw[6:1048577].any().item() is False and dw[1048578:V - 1].any().item() is False
    del dw

    h = torch.randn(4, d, device="cuda", generator=g).bfloat16().requires_grad_()
    t = torch.tensor([V - 1, 1, 1048577, -100], device="cuda")
    loss = ops.piecewise_linear_cross_entropy(h, w, t, reduction="none")
    z = torch.cat([h.detach().float() @ w.detach()[b:b + (1 << 17)].float().t() for b in range(0, V, 1 << 17)], 1)
    ref = torch.nn.functional.cross_entropy(z.double(), t, reduction="none", ignore_index=-100)
    assert (loss.double() - ref).abs().max() < 1e-4
    dh, dw = torch.autograd.grad(loss, (h, w), torch.ones(4, device="cuda"))
    p = torch.softmax(z.double(), 1)
    for j in (0, 1, 1048577, V - 2, V - 1):
        dz = (p[:, j] - (t == j).double()) * (t >= 0)
        row = dz @ h.detach().double()
        # dz and the result are rounded once each (2^-9), fp32 sums in between
        assert (dw[j].double() - row).abs().max() <= 2 ** -8 * 1.01 * (dz.abs()[:, None] * h.detach().double().abs()).sum(0).max()
    assert dh[3].eq(0).all()
    del dh, dw, w, z, p

    n, V = 70001, 32001
    x = torch.zeros(n, V, device="cuda", dtype=torch.bfloat16)
    x[-2:] = torch.randn(2, V, device="cuda", generator=g)
    tids = torch.full((n, 3), -1, device="cuda")
    tids[-2:] = torch.tensor([[7, V - 1, 2], [V - 2, 0, 1]], device="cuda")
    teacher = torch.randn(n, 3, device="cuda", generator=g)
    x.requires_grad_()
    rows = ops.topk_distillation(x, teacher, tids, reduction="none")
    dx, = torch.autograd.grad(rows, x, torch.ones(n, device="cuda"))
    tail = x.detach()[-2:].double().requires_grad_()
    want = _plain_kd(tail, teacher[-2:].double(), tids[-2:], 1.0) * 2
    torch.testing.assert_close(rows[-2:].sum().double(), want.detach(), rtol=1e-5, atol=1e-5)
    ref, = torch.autograd.grad(want, tail)
    assert (dx[-2:].double() - ref).abs().max() <= 2 ** -9 * ref.abs().max() + 1e-6
    assert rows[:-2].eq(0).all() and not dx[:-2].any()


@pytest.mark.gpu
def test_losses_refuse_forward_mode():
    import torch.autograd.forward_ad as fw

    from llm_research_b200 import ops

    ids, w, mix, targets, teacher, tids = _inputs("cuda", torch.bfloat16)
    h = (0.1 * torch.randn(96, 64, device="cuda")).bfloat16()
    x = h @ w.t()
    one = torch.ones((), device="cuda")
    for grad in (False, True):
        for f, leaf in ((lambda a: ops.piecewise_linear_cross_entropy(a, w, targets), h),
                        (lambda a: ops.piecewise_linear_cross_entropy(h, a, targets), w),
                        (lambda a: ops.topk_distillation(a, teacher, tids), x)):
            with fw.dual_level():
                a = leaf.clone().requires_grad_(grad)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(fw.make_dual(a, torch.ones_like(a)))
                if grad:
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        torch.autograd.grad(f(a), a, fw.make_dual(one, one))
    with fw.dual_level():  # the teacher is a constant in both modes
        loss = ops.topk_distillation(x, fw.make_dual(teacher, torch.ones_like(teacher)), tids)
        assert fw.unpack_dual(loss).tangent is None and torch.equal(loss, ops.topk_distillation(x, teacher, tids))


@pytest.mark.parametrize("how", ["piece", "chunks", ""])
def test_unknown_kind_of_fused_loss_is_refused(how):
    """A misspelt kind is an error; the empty string means off, as any false value does."""
    from genesis.model.hlrt import HLRT
    from genesis.training.train_phase1_bootstrap import ntp_objective
    from llm_research_b200.models.presets import build_hlrt_config

    cfg = build_hlrt_config("toy")
    torch.manual_seed(0)
    m = HLRT(cfg)
    ids = torch.randint(0, cfg.vocab_size, (1, 16), generator=torch.Generator().manual_seed(1))
    batch = {"input_ids": ids, "fused_lm_loss": how}
    if how == "":
        assert torch.isfinite(ntp_objective({"hlrt": m}, None, batch))
    else:
        with pytest.raises(ValueError, match="fused_lm_loss"):
            ntp_objective({"hlrt": m}, None, batch)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_each_operator_gives_the_same_bits_again(dtype):
    """Every sum has a fixed order.  (In the whole step autograd's own products come between.)"""
    from llm_research_b200 import ops

    ids, w, mix, targets, teacher, tids = _inputs("cuda", dtype, N=3000, V=5003)
    h = w[ids].clone()
    x = (h.float() @ w.float().t()).to(dtype)

    def run():
        a, b, c = (t.detach().clone().requires_grad_() for t in (w, h, x))
        out = ops.embedding(ids, a, 8.0)
        ce = ops.piecewise_linear_cross_entropy(b, a, targets, piece=1024)
        kd = ops.topk_distillation(c, teacher, tids, 2.0)
        return (out, ce, kd, *torch.autograd.grad(out, a, h), *torch.autograd.grad(ce, (b, a)),
                *torch.autograd.grad(kd, c))

    for u, v in zip(run(), run()):
        assert torch.equal(u, v)
