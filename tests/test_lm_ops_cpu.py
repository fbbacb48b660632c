"""Refusals of the language-model operators: argument checks of the C ABI that need no device, and of the Python entry points."""
import ctypes

import pytest
import torch

from flash_pop_b200 import _lib, layer_ops, token_ops

BF = torch.bfloat16


@pytest.fixture(scope="module")
def handle():
    _lib.build()
    return _lib.lib()


SEQ = _lib._Seq(None, 0, 0, 0)
SHAPE, NULL, DTYPE, STRIDE, LARGE, SPACE = 2, 1, 3, 4, 11, 12


def test_qk_norm_entry_points(handle):
    fwd = lambda B=1, T=4, Hq=2, Hk=2, d=16, dt=0, w=None, ph=None, step=0, q=SEQ: handle.fpb_qk_norm_rotary_fwd(
        B, T, Hq, Hk, d, dt, 1e-6, w, None, ph, step, q, SEQ, SEQ, SEQ, None)
    assert fwd(d=12) == fwd(d=264) == fwd(d=0) == fwd(B=-1) == SHAPE
    assert fwd(dt=7) == DTYPE and fwd() == NULL
    assert fwd(T=(1 << 31) - 100, Hq=1, Hk=1) == fwd(B=1 << 16, T=1 << 15) == fwd(Hq=1 << 15) == LARGE
    assert fwd(w=ctypes.c_void_p(4)) == fwd(ph=ctypes.c_void_p(8)) == fwd(ph=ctypes.c_void_p(16), step=1) == STRIDE
    assert fwd(q=_lib._Seq(0x1008, 128, 32, 16)) == STRIDE
    bwd = lambda scratch, q=SEQ, **kw: handle.fpb_qk_norm_rotary_bwd(0, 4, 2, 2, 16, 0, 1e-6, None, None, None, 0, q, q, q, q, q, q, None, None, scratch, None)
    assert bwd(None) == NULL and bwd(ctypes.c_void_p(8)) == SPACE


def test_dropout_entry_point(handle):
    call = lambda n=8, dt=0, p=0.5, seed=None, x=None: handle.fpb_dropout(n, dt, p, seed, x, None, None, None)
    assert call(n=-1) == call(p=-0.1) == call(p=1.5) == call(p=float("nan")) == SHAPE
    assert call(n=1 << 40) == LARGE and call(dt=2) == DTYPE and call() == NULL
    assert handle.fpb_dropout(8, 0, 0.5, 0x1004, 0x2000, None, 0x3000, None) == STRIDE
    assert handle.fpb_dropout(8, 1, 0.5, 0x1000, 0x2002, None, 0x3000, None) == STRIDE


def test_embedding_entry_points(handle):
    fwd = lambda N=4, V=8, D=16, dt=0, t=0x1000, w=0x2000, ws=16, y=0x3000: handle.fpb_embedding_fwd(N, V, D, dt, t, w, ws, 1.0, y, None)
    assert fwd(N=-1) == fwd(V=0) == fwd(D=0) == SHAPE
    assert fwd(N=1 << 31) == fwd(V=1 << 31) == LARGE and fwd(dt=5) == DTYPE
    assert fwd(t=None) == fwd(w=None) == fwd(y=None) == NULL
    assert fwd(ws=15) == fwd(t=0x1004) == fwd(w=0x2001) == STRIDE
    need = handle.fpb_embedding_workspace(4, 8, 16)
    assert need > 0 and handle.fpb_embedding_workspace(0, 8, 16) == handle.fpb_embedding_workspace(4, 0, 16) == 0
    assert handle.fpb_embedding_workspace(1 << 20, 32000, 1024) < 1 << 30
    bwd = lambda dy=0x2000, s=16, dw=0x3000, ws=0x4000, n=need: handle.fpb_embedding_bwd(4, 8, 16, 0, 0x1000, -1, 1.0, dy, s, dw, ws, n, None)
    assert bwd(dy=None) == bwd(dw=None) == NULL and bwd(s=15) == STRIDE
    assert bwd(ws=None) == bwd(ws=0x4008) == bwd(n=need - 1) == SPACE


def test_token_scores_entry_points(handle):
    fwd = lambda rows=2, V=100, dt=0, top=0, z=0x1000, s=100, t=0x2000, out=0x3000, stats=0x4000, tt=None: handle.fpb_token_scores_fwd(
        rows, V, dt, top, z, s, t, out, out, stats, tt, tt, None)
    assert fwd(rows=-1) == fwd(V=0) == fwd(top=33) == fwd(top=-1) == fwd(V=5, s=5, top=6) == SHAPE
    assert fwd(rows=1 << 31) == fwd(V=(1 << 30) + 1, s=1 << 31) == LARGE and fwd(dt=9) == DTYPE
    assert fwd(z=None) == fwd(t=None) == fwd(out=None) == fwd(stats=None) == fwd(top=3) == NULL
    assert fwd(s=99) == fwd(z=0x1001) == fwd(t=0x2004) == fwd(stats=0x4004) == STRIDE
    bwd = lambda top=0, ent=0x3000, d=0x5000, ds=100, gt=None: handle.fpb_token_scores_bwd(2, 100, 0, top, 0x1000, 100, 0x2000, ent, 0x4000, None, None, None,
                                                                                           gt, d, ds, None)
    assert bwd(ent=None) == bwd(d=None) == bwd(top=2, gt=0x6000) == NULL and bwd(ds=99) == STRIDE


def test_cpu_tensors_are_refused():
    x, ids = torch.randn(2, 3, 2, 16), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: layer_ops.qk_norm_rotary(x, x, None, None, None), lambda: layer_ops.dropout(x, 0.5, ids[:1]),
                 lambda: token_ops.embedding(ids, x[0, 0]), lambda: token_ops.token_scores(x[0, 0], ids)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.fixture
def anywhere(monkeypatch):
    """The checks behind the one for the device, which comes first."""
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)


def test_refused_arguments(anywhere):
    q, w, ph = torch.randn(2, 3, 4, 16), torch.ones(16), torch.zeros(1, 3, 8, 2)
    one = torch.zeros(1, dtype=torch.int64)
    ids, table, logits = torch.zeros(2, 5, dtype=torch.int64), torch.randn(7, 8), torch.randn(2, 5, 9)
    qk, drop, embed, score = layer_ops.qk_norm_rotary, layer_ops.dropout, token_ops.embedding, token_ops.token_scores
    for call in (
        lambda: qk(q[0], q[0], w, w, ph), lambda: qk(q, q[:1], w, w, ph), lambda: qk(q, q[..., :8], w, w, ph),
        lambda: qk(q[..., :12], q[..., :12], None, None, None), lambda: qk(q.repeat(1, 1, 1, 17), q.repeat(1, 1, 1, 17), None, None, None),
        lambda: qk(q, q.to(BF), w, w, ph), lambda: qk(q.half(), q.half(), w, w, ph), lambda: qk(q, q, w[:8], w, ph),
        lambda: qk(q, q, w, w.long(), ph), lambda: qk(q, q, w, w, ph.double()), lambda: qk(q, q, w, w, ph[:, :2]),
        lambda: qk(q, q, w, w, ph.expand(3, 3, 8, 2)), lambda: qk(q, q.to("meta"), w, w, ph), lambda: qk(q, q, w.to("meta"), w, ph),
        lambda: drop(q, -0.1, one), lambda: drop(q, 1.1, one), lambda: drop(q, float("nan"), one), lambda: drop(q.half(), 0.1, one),
        lambda: drop(q, 0.1, one.int()), lambda: drop(q, 0.1, ids), lambda: drop(q, 0.1, one.to("meta")), lambda: drop(q, 0.1, one, q[:1]),
        lambda: drop(q, 0.1, one, q.to(BF)), lambda: layer_ops.CounterDropout(1.5), lambda: layer_ops.CounterDropout(-0.5),
        lambda: embed(ids, table[0]), lambda: embed(ids, table[:0]), lambda: embed(ids, table.half()), lambda: embed(ids.float(), table),
        lambda: embed(ids.to("meta"), table), lambda: embed(ids, table, 1.0, 7), lambda: embed(ids, table, 1.0, -8),
        lambda: score(logits, ids[:1]), lambda: score(logits.half(), ids), lambda: score(logits, ids, 10), lambda: score(logits, ids, -1),
        lambda: score(torch.randn(1, 50), ids[0, :1], 33), lambda: score(logits, ids.float()), lambda: score(logits, ids.to("meta")),
        lambda: score(logits[..., :0], ids),
    ):
        with pytest.raises(ValueError):
            call()


def test_layers_take_the_options_and_refuse_what_the_norms_cannot():
    import flash_pop_b200 as fp
    cpu = dict(num_heads=2, head_dim_v=16, dim_feedforward=32, device="cpu", dtype=torch.float32)
    net = fp.RetNetDecoder(fp.RetNetDecoderLayer.Config(**cpu, qk_norm=True, counter_dropout=True), 1)
    names = {n for n in net.state_dict() if "norm_weight" in n}
    assert names == {"layers.0.retention.q_norm_weight", "layers.0.retention.k_norm_weight"}
    assert net.layers[0].retention.q_norm_weight.shape == (16,) and type(net.layers[0].dropout) is layer_ops.CounterDropout
    plain = fp.RetNetDecoder(fp.RetNetDecoderLayer.Config(**cpu), 1)
    assert not [n for n in plain.state_dict() if "norm_weight" in n] and type(plain.layers[0].dropout) is torch.nn.Dropout
    with pytest.raises(ValueError, match="multiple of 8"):
        fp.RetNetDecoder(fp.RetNetDecoderLayer.Config(**cpu, head_dim_qk=12, qk_norm=True), 1)


def test_counter_dropout_without_anything_to_drop_needs_no_device():
    x, r = torch.randn(3, 4), torch.randn(3, 4)
    m = layer_ops.CounterDropout(0.0)
    assert m(x) is x and torch.equal(m(x, r), r + x)
    m = layer_ops.CounterDropout(0.5).eval()
    assert m(x) is x and not m.active() and "p=0.5" in repr(m)


def test_eps_of_the_norms_is_checked(handle, anywhere):
    fwd = lambda eps: handle.fpb_qk_norm_rotary_fwd(1, 4, 2, 2, 16, 0, eps, None, None, None, 0, SEQ, SEQ, SEQ, SEQ, None)
    bwd = lambda eps: handle.fpb_qk_norm_rotary_bwd(1, 4, 2, 2, 16, 0, eps, None, None, None, 0, SEQ, SEQ, SEQ, SEQ, SEQ, SEQ, None, None, None, None)
    for eps in (-1e-6, float("nan"), -float("inf")):
        assert fwd(eps) == bwd(eps) == SHAPE
        q = torch.randn(2, 3, 4, 16)
        with pytest.raises(ValueError, match="eps"):
            layer_ops.qk_norm_rotary(q, q, None, None, None, eps)
        import flash_pop_b200 as fp
        with pytest.raises(ValueError, match="eps"):
            fp.RetNetDecoder(fp.RetNetDecoderLayer.Config(num_heads=2, head_dim_v=16, dim_feedforward=32, device="cpu", dtype=torch.float32, qk_norm=True,
                                                          qk_norm_eps=eps), 1)
    assert fwd(0.0) == NULL and bwd(0.0) == NULL


def test_counter_dropout_is_for_cuda_tensors_of_two_types(anywhere, monkeypatch):
    """What it cannot drop it refuses, with the same errors as the operator; in eval mode and at p = 0 it takes anything."""
    m, x = layer_ops.CounterDropout(0.5), torch.randn(3, 4)
    for t in (x.half(), x.double(), x.long()):
        with pytest.raises(ValueError, match="bfloat16 or float32"):
            m(t)
        with pytest.raises(ValueError, match="bfloat16 or float32"):
            m(t, t)
        assert m.eval()(t) is t and m.train().active()
    monkeypatch.undo()
    with pytest.raises(RuntimeError, match="no CPU path"):
        m(x)
