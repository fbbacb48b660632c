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
    assert n.qk_norm_forward(q, q, w, None, ph, 1e-6) is not None and n.qk_norm_backward(q, q, w, None, ph, 1e-6, q, q, True, False)[3] is None
    for bad in ((q, q, w[:32], None, ph, 1e-6), (q, q.float(), w, None, ph, 1e-6), (q, q, w.to(BF), None, ph, 1e-6), (q, q, w, None, ph[:, :2], 1e-6),
                (q, q, w, None, ph, 1), (q.transpose(0, 1), q, w, None, ph, 1e-6), (q[..., :60], q[..., :60], None, None, None, 1e-6)):
        assert n.qk_norm_forward(*bad) is None
    x, seed = rnd(5, 7), torch.tensor([1], device="cuda")
    assert n.dropout(x, x, 0.5, seed) is not None
    for bad in ((x, x[:4], 0.5, seed), (x, x.float(), 0.5, seed), (x, None, 1.5, seed), (x, None, 0.5, seed.int()), (x, None, 0.5, seed.cpu()),
                (x.t(), None, 0.5, seed), (x.half(), None, 0.5, seed), (x, None, float("nan"), seed)):
        assert n.dropout(*bad) is None
    t = torch.randint(0, 5, (4,), device="cuda")
    assert n.embedding_forward(t, x, 1.0) is not None and n.embedding_backward(t, x[:4], 9, -1, 1.0) is not None
    for bad in ((t.int(), x, 1.0), (t, x.t(), 1.0), (t, x.half(), 1.0), (t[:0], x, 1.0), (t.cpu(), x, 1.0), (t, x, 1)):
        assert n.embedding_forward(*bad) is None
    assert n.embedding_backward(t, x, 9, -1, 1.0) is None and n.embedding_backward(t, x[:4].t().contiguous().t(), 9, -1, 1.0) is None
    assert n.scores_forward(x[:4], t, 3) is not None
    for bad in ((x, t, 3), (x[:4], t, 8), (x[:4], t, 33), (x[:4], t, -1), (x[:4].half(), t, 0), (x[:4], t.int(), 0), (rnd(4, 2, 7)[:, 0], t[:3], 0)):
        assert n.scores_forward(*bad) is None


def test_forward_mode_gradients_are_not_dropped():
    from flash_pop_b200 import token_ops
    from torch.autograd import forward_ad as fw
    z, t = torch.randn(3, 50, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with fw.dual_level():
        with pytest.raises(RuntimeError):
            token_ops.token_scores(fw.make_dual(z, torch.ones_like(z)), t)
