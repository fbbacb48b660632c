"""The language-model operators through the host-side extension and through Python: the same bits, and which calls the extension
takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _calls():
    from flash_pop_b200 import layer_ops, token_ops
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s, t=BF: torch.randn(*s, generator=g, device="cuda").to(t)
    qk, w, ph = rnd(2, 9, 2, 4, 64), rnd(64, t=torch.float32), rnd(2, 9, 32, 2, t=torch.float32)
    x, res, seed = rnd(3, 70, 33), rnd(3, 70, 33), torch.tensor([7], device="cuda")
    table, ids = rnd(500, 96), torch.randint(0, 500, (3, 70), generator=g, device="cuda")
    z, t = rnd(6, 50, 1003), torch.randint(0, 1003, (6, 50), generator=g, device="cuda")
    return {
        "qk_norm_rotary": ((qk[:, :, 0], qk[:, :, 1], w, w + 1), lambda q, k, a, b: layer_ops.qk_norm_rotary(q, k, a, b, ph, 1e-5)),
        "dropout": ((x, res), lambda x, r: (layer_ops.dropout(x, 0.3, seed, r), layer_ops.dropout(x, 0.3, seed))),
        "embedding": ((table,), lambda w: (token_ops.embedding(ids, w, 3.0, -2),)),
        "token_scores": ((z,), lambda z: token_ops.token_scores(z, t, 7)),
    }


@pytest.mark.parametrize("name", ["qk_norm_rotary", "dropout", "embedding", "token_scores"])
def test_extension_and_python_path_give_the_same_bits(name, monkeypatch):
    from flash_pop_b200 import _lib
    inputs, call = _calls()[name]

    def run():
        with torch.no_grad():
            plain = [t.clone() for t in call(*inputs)]
        leaves = [t.detach().clone().requires_grad_(True) for t in inputs]
        out = [t for t in call(*leaves) if t is not None]
        ends = [t for t in out if t.is_floating_point()]
        return plain + [t.detach() for t in out] + list(torch.autograd.grad(ends, leaves, [torch.ones_like(t) for t in ends]))

    want = run()
    monkeypatch.setattr(_lib, "native", lambda: _lib._Declines())
    for a, b in zip(run(), want, strict=True):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_ordinary_calls_are_taken_and_others_left():
    from flash_pop_b200 import _lib
    n = _lib.native()
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s, t=BF: torch.randn(*s, generator=g, device="cuda").to(t)
    q, w, ph = rnd(2, 3, 4, 64), rnd(64, t=torch.float32), rnd(1, 3, 32, 2, t=torch.float32)
    assert n.qk_norm_rotary(q, q, w, None, ph, 1e-6) is not None
    for bad in ((q, q, w[:32], None, ph, 1e-6), (q, q.float(), w, None, ph, 1e-6), (q, q, w.to(BF), None, ph, 1e-6), (q, q, w, None, ph[:, :2], 1e-6),
                (q, q, w, None, ph, 1), (q.transpose(0, 1), q, w, None, ph, 1e-6), (q[..., :60], q[..., :60], None, None, None, 1e-6)):
        assert n.qk_norm_rotary(*bad) is None
    x, seed = rnd(5, 7), torch.tensor([1], device="cuda")
    assert n.dropout(x, x, 0.5, seed) is not None
    for bad in ((x, x[:4], 0.5, seed), (x, x.float(), 0.5, seed), (x, None, 1.5, seed), (x, None, 0.5, seed.int()), (x, None, 0.5, seed.cpu()),
                (x.t(), None, 0.5, seed), (x.half(), None, 0.5, seed), (x, None, float("nan"), seed)):
        assert n.dropout(*bad) is None
    t = torch.randint(0, 5, (4,), device="cuda")
    assert n.embedding(t, x, 1.0, -1) is not None
    for bad in ((t.int(), x, 1.0, -1), (t, x.t(), 1.0, -1), (t, x.half(), 1.0, -1), (t[:0], x, 1.0, -1), (t.cpu(), x, 1.0, -1), (t, x, 1, -1), (t, x, 1.0, None)):
        assert n.embedding(*bad) is None
    assert n.token_scores(x[:4], t, 3) is not None
    for bad in ((x, t, 3), (x[:4], t, 8), (x[:4], t, 33), (x[:4], t, -1), (x[:4].half(), t, 0), (x[:4], t.int(), 0), (rnd(4, 2, 7)[:, 0], t[:3], 0)):
        assert n.token_scores(*bad) is None


@pytest.mark.parametrize("name", ["qk_norm_rotary", "dropout", "embedding", "token_scores"])
@pytest.mark.parametrize("fast", [True, False])
def test_partial_gradients_strided_gradients_and_second_ones(name, fast, monkeypatch):
    from flash_pop_b200 import _lib
    if not fast:
        monkeypatch.setattr(_lib, "native", lambda: _lib._Declines())
    inputs, call = _calls()[name]
    leaves = [t.detach().clone().requires_grad_(True) for t in inputs]
    ends = [t for t in call(*leaves) if t is not None and t.is_floating_point()]
    want = torch.autograd.grad(ends, leaves, [torch.ones_like(t) for t in ends], retain_graph=True)
    for i, leaf in enumerate(leaves):                              # one input's alone: the others need none
        (got,) = torch.autograd.grad(ends, [leaf], [torch.ones_like(t) for t in ends], retain_graph=True)
        assert torch.equal(got, want[i])
    got = torch.autograd.grad(ends, leaves, [torch.ones(1, device="cuda", dtype=t.dtype).expand(t.shape) for t in ends], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))       # expanded gradients, which no kernel reads in place
    odd = [torch.ones(*t.shape[:-1], t.shape[-1] + 1, device="cuda", dtype=t.dtype)[..., 1:] for t in ends]
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(ends, leaves, odd, retain_graph=True), want))
    few = [t.detach().requires_grad_(i == 0) for i, t in enumerate(leaves)]
    out = [t for t in call(*few) if t is not None and t.is_floating_point()]
    assert torch.equal(torch.autograd.grad(out, few[:1], [torch.ones_like(t) for t in out])[0], want[0])
    gs = [torch.ones_like(t, requires_grad=True) for t in ends]
    once = torch.autograd.grad(ends, leaves, gs, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(once, want))
    with pytest.raises(RuntimeError, match="twice"):
        once[0].float().pow(2).sum().backward()


def test_saved_tensors_that_change_raise():
    from flash_pop_b200 import layer_ops
    x, seed = torch.randn(50, device="cuda", requires_grad=True), torch.tensor([3], device="cuda")
    y = layer_ops.dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), [x])


def test_forward_mode_gradients_are_not_dropped():
    from flash_pop_b200 import token_ops
    from torch.autograd import forward_ad as fw
    z, t = torch.randn(3, 50, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with fw.dual_level():
        with pytest.raises(RuntimeError):
            token_ops.token_scores(fw.make_dual(z, torch.ones_like(z)), t)


@pytest.mark.parametrize("name", ["qk_norm_rotary", "dropout", "embedding", "token_scores"])
@pytest.mark.parametrize("fast", [True, False])
def test_a_capture_beside_a_living_eager_graph_of_its_leaves_is_refused(name, fast, monkeypatch):
    """The engine would make the default stream wait within the capture, an error that ends the process: the operator's node raises
    before, and the same capture works once the eager outputs are gone."""
    from flash_pop_b200 import layer_ops, token_ops
    if not fast:                                                   # the operators' Python nodes, with the extension's check
        for module in (layer_ops, token_ops):
            for f in ("qk_norm_rotary", "dropout", "embedding", "token_scores"):
                if hasattr(module, f):
                    monkeypatch.setattr(module._lib.native(), f, lambda *a: None)
    inputs, call = _calls()[name]
    leaves = [t.detach().clone().requires_grad_(True) for t in inputs]

    def step():
        ends = [t for t in call(*leaves) if t is not None and t.is_floating_point()]
        return ends, lambda: torch.autograd.grad(ends, leaves, [torch.ones_like(t) for t in ends], retain_graph=True)

    eager, grads = step()
    want = grads()
    torch.cuda.synchronize()
    refused, graph, pool = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.graph_pool_handle()
    with torch.cuda.graph(refused, pool=pool):
        ends, again = step()
        with pytest.raises(RuntimeError, match="release the outputs of the eager calls"):
            again()
    del eager, grads, ends, again
    with torch.cuda.graph(graph, pool=pool):
        ends, again = step()
        got = again()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


@pytest.mark.parametrize("name", ["qk_norm_rotary", "dropout", "embedding", "token_scores"])
def test_traced_calls_compute_when_they_run(name):
    """A recorded graph of a call gives the call's results for other inputs."""
    inputs, call = _calls()[name]
    with torch.no_grad():
        traced = torch.jit.trace(lambda *a: tuple(t for t in call(*a) if t is not None), inputs, check_trace=False)
        others = [torch.randn_like(t) for t in inputs]
        for args in (inputs, others, inputs):
            got, want = traced(*args), [t for t in call(*args) if t is not None]
            assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_extension_leaves_traced_calls():
    from flash_pop_b200 import _lib
    n, seen = _lib.native(), []
    x, seed = torch.randn(5, 7, device="cuda"), torch.tensor([1], device="cuda")

    def f(x):
        seen.append((n.dropout(x, None, 0.5, seed), n.rotary(x.view(1, 5, 1, 7), None, x, False, x.dtype)))
        return x * 2

    torch.jit.trace(f, (x,), check_trace=False)
    assert seen == [(None, None)] and n.dropout(x, None, 0.5, seed) is not None
