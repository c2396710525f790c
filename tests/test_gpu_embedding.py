"""Token embedding (lookup with scaling, gradient by sorted tokens) against the
formula in 64 bits.

Tolerances: the output is ``scale * w`` in fp32 (relative 2^-24) rounded once, so
half a step of the type, plus 2^-24.  A gradient row sums ``c`` terms in fp32; in
any order its error is below ``c * 2^-24 * sum |terms|``, then one rounding."""

import pytest
import torch

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _half_step(t):
    return torch.finfo(t).eps / 2


def _check_out(out, w, ids, scale):
    ref = w.double()[ids.long()] * scale
    # subnormal results (fp16) round to half of the smallest subnormal
    tiny = torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps / 2
    assert (out.double() - ref).abs().le(ref.abs() * (_half_step(out.dtype) + 2.0 ** -23) + tiny).all()


def _check_grad(dw, dy, ids, V, scale, padding=None):
    d = dy.shape[-1]
    dy, ids = dy.reshape(-1, d).double(), ids.reshape(-1).long()
    ok = (ids >= 0) & (ids < V)
    if padding is not None:
        ok &= ids != padding
    ref = torch.zeros(V, d, dtype=torch.float64, device=dy.device)
    mag, count = torch.zeros_like(ref), torch.zeros(V, 1, dtype=torch.float64, device=dy.device)
    ref.index_add_(0, ids[ok], dy[ok])
    mag.index_add_(0, ids[ok], dy[ok].abs())
    count.index_add_(0, ids[ok], torch.ones_like(dy[ok][:, :1]))
    ref, mag = ref * scale, mag * abs(scale)
    tiny = torch.finfo(dw.dtype).smallest_normal * torch.finfo(dw.dtype).eps / 2
    tol = ref.abs() * _half_step(dw.dtype) + (count + 2) * 2.0 ** -24 * mag * (1 + _half_step(dw.dtype)) + tiny
    assert (dw.double() - ref).abs().le(tol).all()


# ------------------------------------------------------------------ CPU
def test_cpu_matches_formula_and_gradient():
    from llm_research_b200 import ops

    g = torch.Generator().manual_seed(0)
    w = torch.randn(11, 5, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[1, 4, 4], [10, 0, 1]])
    out = ops.embedding(ids, w, scale=3.0, padding_idx=4)
    torch.testing.assert_close(out, 3.0 * w[ids])
    dy = torch.randn(2, 3, 5, generator=g, dtype=torch.float64)
    dw, = torch.autograd.grad(out, w, dy)
    _check_grad(dw, dy, ids, 11, 3.0, padding=4)
    assert (dw[4] == 0).all()
    assert torch.autograd.gradcheck(lambda t: ops.embedding(ids, t, scale=0.5), (w,))


def test_refusals():
    from llm_research_b200 import ops

    w = torch.zeros(7, 4)
    with pytest.raises(TypeError, match="int64 or int32"):
        ops.embedding(torch.zeros(3), w)
    with pytest.raises(ValueError, match="weight must be"):
        ops.embedding(torch.zeros(3, dtype=torch.long), torch.zeros(7))
    for bad in (7, -8):
        with pytest.raises(ValueError, match="padding_idx"):
            ops.embedding(torch.zeros(3, dtype=torch.long), w, padding_idx=bad)
    with pytest.raises(IndexError):
        ops.embedding(torch.tensor([7]), w)


# ------------------------------------------------------------------ GPU
def _tokens(n, V, g):
    """Few frequent tokens (several occurrence counts around the piece sizes), many rare ones."""
    ids = torch.randint(0, V, (n,), generator=g)
    hot = torch.rand(n, generator=g)
    ids[hot < 0.3] = V // 2
    ids[(hot >= 0.3) & (hot < 0.35)] = 0
    ids[(hot >= 0.35) & (hot < 0.37)] = V - 1
    return ids


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (1, 512, 128), (7, 33, 8), (64, 5, 24), (65, 3, 40), (300, 512, 1001),
                                   (4097, 32000, 256), (8193, 100287, 129), (20000, 1000, 2048), (70000, 50000, 72)])
def test_embedding_forward_backward(dtype, n, V, d):
    from llm_research_b200 import ops

    g = torch.Generator().manual_seed(n + V + d)
    ids = _tokens(n, V, g).cuda()
    w = torch.randn(V, d, generator=g).to(dtype).cuda().requires_grad_()
    dy = torch.randn(n, d, generator=g).to(dtype).cuda()
    pad = V // 2 if V > 2 else None
    out = ops.embedding(ids, w, scale=1.7, padding_idx=pad)
    dw, = torch.autograd.grad(out, w, dy)
    assert out.shape == (n, d) and out.dtype == dtype and dw.dtype == dtype
    _check_out(out, w.detach(), ids, 1.7)
    _check_grad(dw, dy, ids, V, 1.7, pad)
    # int32 ids and another run: the same bits
    out2 = ops.embedding(ids.int(), w, scale=1.7, padding_idx=pad)
    dw2, = torch.autograd.grad(out2, w, dy)
    assert torch.equal(out, out2) and torch.equal(dw, dw2)
    with torch.no_grad():
        assert torch.equal(out, ops.embedding(ids, w, scale=1.7))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [63, 64, 65, 4096, 4097, 5000, 16385, 65537])
def test_one_token_everywhere(n):
    """A single segment, split into pieces (or not), equals the 64-bit sum."""
    from llm_research_b200 import ops

    w = torch.zeros(9, 64, device="cuda", requires_grad=True)
    ids = torch.full((n,), 5, device="cuda")
    dy = torch.randn(n, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(n))
    dw, = torch.autograd.grad(ops.embedding(ids, w), w, dy)
    _check_grad(dw, dy, ids, 9, 1.0)
    assert (dw[:5] == 0).all() and (dw[6:] == 0).all()


@pytest.mark.gpu
def test_shapes_strides_and_empty():
    from llm_research_b200 import ops

    g = torch.Generator("cuda").manual_seed(3)
    base = torch.randn(50, 80, device="cuda", generator=g).to(torch.bfloat16)
    ids = torch.randint(0, 50, (6, 8), device="cuda", generator=g)
    for w in (base[:, :64], base[:, 3:67], base.t()[:50, :40], base[::2][:, 8:]):  # pitched, unaligned, transposed
        V = w.shape[0]
        w = w.detach().requires_grad_()
        i = ids.t()[1:, ::2] % V  # not contiguous
        out = ops.embedding(i, w, scale=0.25)
        assert out.shape == (*i.shape, w.shape[1])
        _check_out(out, w.detach(), i, 0.25)
        dy = torch.randn(w.shape[1], *i.shape, device="cuda", generator=g).to(torch.bfloat16).permute(1, 2, 0)
        dw, = torch.autograd.grad(out, w, dy)
        _check_grad(dw, dy, i, V, 0.25)
        # a broadcast gradient (stride 0)
        dw, = torch.autograd.grad(ops.embedding(i, w).float().sum(), w)
        _check_grad(dw, torch.ones(*i.shape, w.shape[1], device="cuda"), i, V, 1.0)
    w = base.requires_grad_()
    assert ops.embedding(torch.tensor(4, device="cuda"), w).shape == (80,)
    out = ops.embedding(torch.zeros(0, 3, dtype=torch.long, device="cuda"), w)
    dw, = torch.autograd.grad(out.sum(), w)
    assert out.shape == (0, 3, 80) and (dw == 0).all() and dw.shape == w.shape


@pytest.mark.gpu
def test_ids_outside_the_table_give_nan_and_no_gradient():
    from llm_research_b200 import ops

    w = torch.randn(10, 16, device="cuda", requires_grad=True)
    ids = torch.tensor([3, -1, 10, 2 ** 40, -2 ** 40, 9], device="cuda")
    out = ops.embedding(ids, w)
    assert out[1:5].isnan().all() and torch.equal(out[[0, 5]], w[[3, 9]])
    dy = torch.randn(6, 16, device="cuda")
    dw, = torch.autograd.grad(out, w, dy)
    _check_grad(dw, dy, ids, 10, 1.0)


@pytest.mark.gpu
def test_double_backward_is_the_lookup():
    from llm_research_b200 import ops

    w = torch.randn(10, 8, device="cuda", requires_grad=True)
    ids = torch.tensor([1, 1, 4, 7, 12], device="cuda")
    dy = torch.randn(5, 8, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(ops.embedding(ids, w, 2.0, padding_idx=4), w, dy, create_graph=True)
    v = torch.randn_like(dw)
    gdy, = torch.autograd.grad((dw * v).sum(), dy)
    ref = 2.0 * v[ids.clamp(max=9)]
    ref[2] = 0
    ref[4] = 0
    torch.testing.assert_close(gdy, ref, rtol=2 ** -23, atol=0)


@pytest.mark.gpu
def test_infinities_stay_in_their_rows():
    from llm_research_b200 import ops

    w = torch.randn(6, 32, device="cuda").to(torch.float16)
    w[2, 5], w[3, 6] = float("inf"), float("nan")
    w.requires_grad_()
    ids = torch.tensor([0, 2, 3, 1], device="cuda")
    out = ops.embedding(ids, w, 2.0)
    assert out[1, 5].isinf() and out[2, 6].isnan() and out[[0, 3]].isfinite().all()
    dy = torch.ones(4, 32, device="cuda", dtype=torch.float16)
    dy[3, 1], dy[0, 2] = float("nan"), float("-inf")
    dw, = torch.autograd.grad(out, w, dy)
    assert dw[1, 1].isnan() and dw[0, 2] == float("-inf") and dw[4:].eq(0).all() and dw[2:4].eq(2).all()


@pytest.mark.gpu
def test_other_stream_and_graph_replay():
    from llm_research_b200 import ops

    g = torch.Generator("cuda").manual_seed(8)
    w = torch.randn(300, 64, device="cuda", generator=g).to(torch.bfloat16).requires_grad_()
    ids = torch.randint(0, 300, (1000,), device="cuda", generator=g)
    dy = torch.randn(1000, 64, device="cuda", generator=g).to(torch.bfloat16)

    def step():
        out = ops.embedding(ids, w, 1.5)
        return out.detach(), torch.autograd.grad(out, w, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            out0, dw0 = step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step())
        graphs.append(gr)
    for new in range(2):
        ids.copy_(torch.randint(0, 300, (1000,), device="cuda", generator=g))
        for gr in graphs:
            gr.replay()
        for out, dw in outs:
            _check_out(out, w.detach(), ids, 1.5)
            _check_grad(dw, dy, ids, 300, 1.5)


@pytest.mark.gpu
def test_cuda_refusals():
    from llm_research_b200 import ops
    from llm_research_b200._ext import native

    ids = torch.zeros(3, dtype=torch.long, device="cuda")
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        ops.embedding(ids, torch.zeros(4, 4, device="cuda", dtype=torch.float64))
    with pytest.raises(RuntimeError, match="one CUDA device"):
        ops.embedding(ids.cpu(), torch.zeros(4, 4, device="cuda"))
    with pytest.raises(RuntimeError, match="dy"):
        native().embedding_bwd(torch.zeros(2, 4, device="cuda"), ids, 4, -1, 1.0)


@pytest.mark.gpu
def test_shared_embeddings_use_the_kernel_and_keep_their_results():
    from genesis.model.embeddings import SharedEmbeddings

    for dtype in (torch.bfloat16, torch.float32):
        m = SharedEmbeddings(400, 96, padding_idx=3).to("cuda", dtype)
        ids = torch.randint(0, 400, (4, 50), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
        ids[:, 40:] = 3
        out = m(ids)
        assert type(out.grad_fn).__name__ != "EmbeddingBackward0"
        ref = torch.nn.functional.embedding(ids, m.weight, 3)
        assert torch.equal(out, ref)
        dy = torch.randn_like(out)
        out.backward(dy)
        _check_grad(m.weight.grad, dy, ids, 400, 1.0, padding=3)
        assert (m.weight.grad[3] == 0).all()


@pytest.mark.gpu
def test_forward_mode_derivative_is_the_lookup_of_the_tangent():
    import torch.autograd.forward_ad as fw

    from llm_research_b200 import ops

    g = torch.Generator("cuda").manual_seed(9)
    w, t = (torch.randn(20, 24, device="cuda", generator=g) for _ in range(2))
    ids = torch.tensor([[3, 0, 3], [19, 7, 5]], device="cuda")
    dy, dyt = (torch.randn(2, 3, 24, device="cuda", generator=g) for _ in range(2))
    for grad in (False, True):
        with fw.dual_level():
            w1 = w.clone().requires_grad_(grad)
            out = fw.unpack_dual(ops.embedding(ids, fw.make_dual(w1, t), 1.5, padding_idx=3))
            assert torch.equal(out.primal, 1.5 * w[ids]) and torch.equal(out.tangent, 1.5 * t[ids])
            if grad:
                dw, = torch.autograd.grad(out.primal, w1, dy)
                _check_grad(dw, dy, ids, 20, 1.5, padding=3)
    w.requires_grad_()
    for create_graph in (False, True):  # the gradient is linear in dy as well
        with fw.dual_level():
            out = ops.embedding(ids, w, 1.5, padding_idx=3)
            dw = fw.unpack_dual(torch.autograd.grad(out, w, fw.make_dual(dy, dyt), create_graph=create_graph)[0])
            _check_grad(dw.primal, dy, ids, 20, 1.5, padding=3)
            _check_grad(dw.tangent, dyt, ids, 20, 1.5, padding=3)


# ------------------------------------------------------------------ SharedEmbeddings as a module
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _shared(device, **kw):
    from genesis.model.embeddings import SharedEmbeddings

    torch.manual_seed(2)
    m = SharedEmbeddings(40, 16, **kw).to(device)
    return m, torch.tensor([[1, 5, 5], [39, 0, 2]], device=device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [1.0, 4.0])
def test_hooks_and_replacements_of_the_inner_embedding_act(device, scale):
    """Hooks see the rows of the table; the scale comes behind them."""
    m, ids = _shared(device, scale=scale)
    want, rows, seen = m(ids), m.weight[ids], []
    pre = m.embedding.register_forward_pre_hook(lambda mod, args: seen.append("pre") or (args[0] * 0 + 5,))
    post = m.embedding.register_forward_hook(lambda mod, args, out: out + 1)
    assert torch.equal(m(ids), ((m.weight[5] + 1) * scale).expand(2, 3, 16)) and seen == ["pre"]
    pre.remove(), post.remove()
    back = m.embedding.register_full_backward_hook(lambda mod, gin, gout: seen.append(gout[0].clone()))
    m(ids).sum().backward()
    assert seen[1].eq(scale).all()
    back.remove()
    every = torch.nn.modules.module.register_module_forward_hook(
        lambda mod, args, out: seen.append(out) if mod is m.embedding else None)
    assert torch.equal(m(ids), want) and torch.equal(seen[2], rows)
    every.remove()
    assert torch.equal(m(ids), want) and len(seen) == 3
    other = torch.nn.Embedding(40, 16).to(device)
    inner, m.embedding = m.embedding, other
    assert torch.equal(m(ids), other(ids) * scale)

    class Shifted(torch.nn.Embedding):
        def forward(self, i):
            return super().forward(i) + 1

    m.embedding = Shifted(40, 16).to(device)
    assert torch.equal(m(ids), (m.weight[ids] + 1) * scale)
    m.embedding = inner
    inner.forward = lambda i: torch.ones(*i.shape, 16, device=device)
    assert m(ids).eq(scale).all() and m(ids).shape == (2, 3, 16)


@pytest.mark.parametrize("device", DEVICES)
def test_settings_of_the_inner_embedding_act(device):
    F = torch.nn.functional
    m, ids = _shared(device)
    dy = torch.randn(2, 3, 16, device=device)
    m.embedding.scale_grad_by_freq = True
    w = m.weight.detach().clone().requires_grad_()
    F.embedding(ids, w, scale_grad_by_freq=True).backward(dy)
    m(ids).backward(dy)
    torch.testing.assert_close(m.weight.grad, w.grad)
    m, ids = _shared(device)
    m.embedding.sparse = True
    m(ids).backward(dy)
    assert m.weight.grad.is_sparse
    m, ids = _shared(device)
    m.embedding.max_norm = 0.5
    out = m(ids)
    assert out.norm(dim=-1).le(0.5 * (1 + 1e-5)).all()
    assert m.weight[[1, 5, 39, 0, 2]].norm(dim=-1).le(0.5 * (1 + 1e-5)).all() and m.weight[3].norm() > 1


@pytest.mark.parametrize("device", DEVICES)
def test_shared_embeddings_under_function_transforms_and_tracing(device):
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch._subclasses import FakeTensorMode

    m, ids = _shared(device, scale=2.0)
    want = m(ids).detach()
    assert torch.equal(torch.vmap(m)(ids), want)
    params = dict(m.named_parameters())
    tangents = {k: torch.randn_like(p) for k, p in params.items()}

    def f(p):
        return torch.func.functional_call(m, p, (ids,))

    grads = torch.func.grad(lambda p: f(p).sum())(params)
    count = torch.bincount(ids.flatten(), minlength=40).to(want.dtype)
    assert torch.equal(grads["embedding.weight"], (2 * count)[:, None].expand(40, 16))
    out, tangent = torch.func.jvp(f, (params,), (tangents,))
    assert torch.equal(out, want) and torch.equal(tangent, 2 * tangents["embedding.weight"][ids])
    assert torch.equal(make_fx(m)(ids)(ids.flip(0)), want.flip(0))
    assert torch.equal(torch.jit.trace(m, ids)(ids.flip(0)), want.flip(0))
    assert torch.equal(torch.fx.symbolic_trace(m)(ids), want)
    assert torch.equal(torch.jit.script(m)(ids), want)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fake = m(mode.from_tensor(ids))
    assert fake.shape == (2, 3, 16) and fake.device.type == device


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,d", [(5000, 300000, 16), (40000, 300000, 8), (40000, 262145, 33)])
def test_sort_of_three_passes_over_several_blocks(dtype, n, V, d):
    from llm_research_b200 import ops

    g = torch.Generator().manual_seed(n + V)
    ids = _tokens(n, V, g)
    ids[::7] = ids[0] % 1000 + 511 * 512  # tokens that differ in the last digit alone
    ids, w = ids.cuda(), torch.zeros(V, d, device="cuda", dtype=dtype, requires_grad=True)
    dy = torch.randn(n, d, generator=g).to(dtype).cuda()
    dw, = torch.autograd.grad(ops.embedding(ids, w), w, dy)
    _check_grad(dw, dy, ids, V, 1.0)
    dw2, = torch.autograd.grad(ops.embedding(ids, w), w, dy)
    assert torch.equal(dw, dw2)
