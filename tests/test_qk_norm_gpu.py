"""Norms of queries and keys with the rotation, against the formulas in 64 bits: values, gradients, layouts, refusals."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}          # one rounding of the result


def _phasors(rows, T, d, seed=0):
    start = torch.arange(rows, dtype=torch.float64)[:, None] * 37 + torch.arange(T, dtype=torch.float64)
    angle = start[..., None] * 10000.0 ** -torch.linspace(0, 1, d // 2, dtype=torch.float64)
    return torch.stack((angle.cos(), angle.sin()), -1).float().cuda()


def _formula(x, w, ph, eps):
    """y of doubles, elementary operations only."""
    n = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    n = n if w is None else n * w
    if ph is None:
        return n
    c, s = (ph[..., i].double().unsqueeze(2) for i in (0, 1))
    a, b = n[..., 0::2], n[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _row_max(t):
    return t.abs().amax(-1, keepdim=True)


def _check(q, k, wq, wk, ph, eps, dyq, dyk):
    from flash_pop_b200.layer_ops import qk_norm_rotary
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk) if t is not None]
    it = iter(leaves)
    a = [next(it) if t is not None else None for t in (q, k, wq, wk)]
    got = qk_norm_rotary(*a, ph, eps)
    grads = dict(zip([n for n, t in zip("q k wq wk".split(), (q, k, wq, wk)) if t is not None], torch.autograd.grad(got, leaves, (dyq, dyk))))
    half = HALF[q.dtype]
    for x, w, dy, y, gx, gw in ((q, wq, dyq, got[0], grads["q"], grads.get("wq")), (k, wk, dyk, got[1], grads["k"], grads.get("wk"))):
        xd = x.double().requires_grad_(True)
        wd = None if w is None else w.double().requires_grad_(True)
        ref = _formula(xd, wd, ph, eps)
        assert y.dtype == x.dtype and y.shape == x.shape and gx.shape == x.shape and gx.dtype == x.dtype
        # the result's rounding, and 16 operations in fp32 relative to the row's largest element
        assert bool(((y.double() - ref).abs() <= half * ref.abs() + 2.0 ** -20 * _row_max(ref) + 1e-30).all())
        gr = torch.autograd.grad(ref, [xd] if w is None else [xd, wd], dy.double())
        # terms that cancel: r g w and the projection on n, both at most r max |g| max |w| sqrt(d), of d products summed in fp32
        r = 1 / (x.double().pow(2).mean(-1, keepdim=True) + eps).sqrt()
        scale = r * _row_max(dy.double()) * 2 * (1.0 if w is None else float(w.double().abs().max()))
        assert bool(((gx.double() - gr[0]).abs() <= half * gr[0].abs() + 2.0 ** -18 * scale).all())
        if w is not None:
            # chains of at most 64 rows a thread and sums over threads and CTAs behind them: 128 roundings of all the terms' sizes
            n = x.double() * r
            g = dy.double() if ph is None else _formula_back(dy.double(), ph)
            assert gw.dtype == w.dtype
            bound = 128 * 2.0 ** -24 * (g * n).abs().sum((0, 1, 2)) + 1e-30 + (HALF[BF] * gr[1].abs() if w.dtype == BF else 0)
            assert bool(((gw.double() - gr[1]).abs() <= bound).all())


def _formula_back(g, ph):
    c, s = (ph[..., i].double().unsqueeze(2) for i in (0, 1))
    a, b = g[..., 0::2], g[..., 1::2]
    return torch.stack((a * c + b * s, b * c - a * s), -1).flatten(-2)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,Hq,Hk,d", [(1, 1, 1, 1, 8), (2, 3, 4, 4, 16), (1, 257, 3, 1, 24), (3, 65, 8, 2, 40), (2, 130, 5, 5, 64), (1, 33, 7, 9, 104),
                                         (2, 77, 8, 8, 128), (1, 19, 2, 16, 200), (2, 31, 3, 3, 256)])
def test_values_and_gradients(B, T, Hq, Hk, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(B * 1000 + T)
    rnd = lambda *s, t=dtype: torch.randn(*s, generator=g, device="cuda").to(t)
    q, k, dyq, dyk = rnd(B, T, Hq, d), rnd(B, T, Hk, d) * 3, rnd(B, T, Hq, d), rnd(B, T, Hk, d)
    _check(q, k, 1 + 0.2 * rnd(d, t=F32), 1 + 0.2 * rnd(d, t=F32), _phasors(1, T, d), 1e-6, dyq, dyk)


def test_tokens_beyond_one_round_of_the_launch():
    g = torch.Generator(device="cuda").manual_seed(1)
    for d, T in ((64, 21000), (256, 5000)):
        q, k, dyq, dyk = (torch.randn(1, T, h, d, generator=g, device="cuda").to(BF) for h in (2, 1, 2, 1))
        _check(q, k, torch.ones(d, device="cuda"), torch.ones(d, device="cuda"), _phasors(1, T, d), 1e-6, dyq, dyk)


def test_tables_weights_and_rows_of_zeros():
    g = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)
    B, T, H, d = 3, 9, 4, 64
    q, k, dyq, dyk = (rnd(B, T, H, d) for _ in range(4))
    _check(q, k, None, None, _phasors(B, T, d), 1e-5, dyq, dyk)                     # a table for each row, no weights
    _check(q, k, torch.rand(d, device="cuda"), None, None, 1e-6, dyq, dyk)           # one weight, no rotation
    _check(q, k, torch.rand(d, device="cuda").to(BF), torch.rand(d, device="cuda").to(BF), _phasors(1, T, d), 1e-6, dyq, dyk)
    q[0, 3], k[1, :, 2] = 0, 0
    q[2, 0] *= 1e-3
    _check(q, k, torch.ones(d, device="cuda"), torch.ones(d, device="cuda"), _phasors(1, T, d), 1e-6, dyq, dyk)


def test_layouts_give_the_bits_of_contiguous_tensors():
    from flash_pop_b200.layer_ops import qk_norm_rotary
    g = torch.Generator(device="cuda").manual_seed(3)
    B, T, H, d = 2, 37, 4, 64
    w, ph = torch.rand(d, device="cuda"), _phasors(1, T, d)
    packed = torch.randn(B, T, 3, H, d, generator=g, device="cuda").to(BF)
    views = [packed[:, :, 0], packed[:, :, 2]]
    odd = torch.randn(B, T, H, d + 1, generator=g, device="cuda").to(BF)
    for q, k in (views, [t.transpose(1, 2).contiguous().transpose(1, 2) for t in views], [odd[..., 1:], odd[..., :-1]],
                 [packed[:1, :, 0].expand(B, T, H, d), views[1]]):
        want = qk_norm_rotary(q.contiguous(), k.contiguous(), w, w, ph)
        got = qk_norm_rotary(q, k, w, w, ph)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # gradients that come expanded (a sum's) and through the packed leaf
    leaf = packed.detach().requires_grad_(True)
    yq, yk = qk_norm_rotary(leaf[:, :, 0], leaf[:, :, 2], w, w, ph)
    (gr,) = torch.autograd.grad(yq.sum() + yk.float().pow(2).sum(), [leaf])
    assert gr.shape == packed.shape and bool((gr[:, :, 1] == 0).all()) and bool(gr[:, :, 0].abs().sum() > 0)


def test_gradient_against_differences():
    from flash_pop_b200.layer_ops import qk_norm_rotary
    g = torch.Generator(device="cuda").manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    q, k, w, ph = rnd(1, 3, 2, 16), rnd(1, 3, 2, 16), 1 + 0.1 * rnd(16), _phasors(1, 3, 16)
    u, v = rnd(1, 3, 2, 16), rnd(1, 3, 2, 16)
    f = lambda q, w: float((qk_norm_rotary(q, k, w, w, ph)[0].double() * u.double()).sum() + (qk_norm_rotary(q, k, w, w, ph)[1].double() * v.double()).sum())
    ql, wl = q.clone().requires_grad_(True), w.clone().requires_grad_(True)
    yq, yk = qk_norm_rotary(ql, k, wl, wl, ph)
    gq, gw = torch.autograd.grad((yq, yk), [ql, wl], (u, v))
    dq, dw = rnd(*q.shape), rnd(16)
    # a step of 2^-7 along a direction: the difference is off by its third order (step^2) and by fp32 values of f over the step
    h = 2.0 ** -7
    for got, plus, minus in (((gq * dq).sum(), f(q + h * dq, w), f(q - h * dq, w)), ((gw * dw).sum(), f(q, w + h * dw), f(q, w - h * dw))):
        assert abs(float(got) - (plus - minus) / (2 * h)) <= 2e-2 * (1 + abs(float(got)))


def test_same_bits_twice_other_streams_and_graphs():
    from flash_pop_b200.layer_ops import qk_norm_rotary
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, dyq, dyk = (torch.randn(2, 500, 4, 64, generator=g, device="cuda").to(BF) for _ in range(4))
    w, ph = torch.rand(64, device="cuda").requires_grad_(True), _phasors(1, 500, 64)
    q.requires_grad_(True)

    def step():
        y = qk_norm_rotary(q, k, w, w, ph)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, [q, w], (dyq, dyk)))

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    for t in held:
        t.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_empty_calls():
    from flash_pop_b200.layer_ops import qk_norm_rotary
    w = torch.ones(16, device="cuda", requires_grad=True)
    for B, T, Hq, Hk in ((0, 4, 2, 2), (2, 0, 2, 2), (2, 3, 0, 2)):
        q, k = torch.ones(B, T, Hq, 16, device="cuda", requires_grad=True), torch.ones(B, T, Hk, 16, device="cuda")
        yq, yk = qk_norm_rotary(q, k, w, w, _phasors(1, T, 16))
        assert yq.shape == q.shape and yk.shape == k.shape
        gq, gw = torch.autograd.grad((yq, yk), [q, w], (torch.ones_like(yq), torch.ones_like(yk)))
        assert gq.shape == q.shape and gw.shape == w.shape and bool(torch.isfinite(gw).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,Hq,Hk,d", [(1, 3, 1, 1, 8), (2, 77, 5, 3, 40), (1, 33, 7, 1, 64), (1, 19, 3, 5, 200), (3, 21, 17, 16, 256)])
def test_without_eps(B, T, Hq, Hk, d, dtype):
    """eps = 0, or one that fp32 does not hold: rows that are not there (odd heads, the last stretch of tokens) leave nothing behind."""
    g = torch.Generator(device="cuda").manual_seed(T)
    rnd = lambda *s, t=dtype: torch.randn(*s, generator=g, device="cuda").to(t)
    q, k, dyq, dyk = rnd(B, T, Hq, d), rnd(B, T, Hk, d), rnd(B, T, Hq, d), rnd(B, T, Hk, d)
    for eps in (0.0, 1e-60):
        _check(q, k, 1 + 0.2 * rnd(d, t=F32), 1 + 0.2 * rnd(d, t=F32), _phasors(1, T, d), eps, dyq, dyk)


@pytest.mark.parametrize("fast", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_contiguous_tensors_that_are_not_aligned(dtype, fast, monkeypatch):
    from flash_pop_b200 import _lib
    from flash_pop_b200.layer_ops import qk_norm_rotary
    if not fast:
        monkeypatch.setattr(_lib, "native", lambda: _lib._Declines())
    g = torch.Generator(device="cuda").manual_seed(8)
    B, T, H, d = 2, 5, 3, 24
    n = B * T * H * d

    def offset(t, by=1):
        flat = torch.empty(n + by, device="cuda", dtype=t.dtype)
        flat[by:] = t.flatten()
        return flat[by:].view(t.shape)

    q, k, dyq, dyk = (torch.randn(B, T, H, d, generator=g, device="cuda").to(dtype) for _ in range(4))
    w, ph = torch.rand(d, device="cuda").requires_grad_(True), _phasors(1, T, d)
    moved = [offset(t) for t in (q, k, dyq, dyk)]
    assert all(t.is_contiguous() and t.data_ptr() % 16 for t in moved)

    def step(q, k, dyq, dyk):
        q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        y = qk_norm_rotary(q, k, w, w, ph)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, [q, k, w], (dyq, dyk)))

    want = step(q, k, dyq, dyk)
    for args in (moved, [moved[0], k, dyq, moved[3]], [q, k, moved[2], dyk]):
        assert all(torch.equal(a, b) for a, b in zip(step(*args), want, strict=True))
    ones = [torch.empty_strided((1, T, H, d), (7, H * d, d, 1), device="cuda", dtype=dtype).copy_(t[:1]) for t in (q, k, dyq, dyk)]
    assert all(t.is_contiguous() and t.stride(0) == 7 for t in ones)                     # an odd stride that no element uses
    assert all(torch.equal(a, b) for a, b in zip(step(*ones), step(q[:1], k[:1], dyq[:1], dyk[:1]), strict=True))


def _items(B, T, Hq, Hk, d):
    """How many pieces of work a tensor's launch is cut into, as the launch counts them: stretches of up to eight tokens a group of
    lanes, one row or two heads of it at a time, 256 threads."""
    lanes = 1
    while lanes * 8 < d:
        lanes *= 2
    groups, H = 256 // lanes, max(Hq, Hk)
    sets = (H + 1) // 2 if H > 1 else 1
    block, rounds = min(sets, groups), 8
    while True:
        stretch = groups // block * rounds
        items = B * -(-T // stretch) * -(-sets // block)
        if items >= 296 or rounds == 1:
            return items, rounds, -(-sets // block)
        rounds //= 2


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,Hq,Hk,d", [(8, 4096, 8, 8, 128), (6, 9001, 5, 2, 64), (8, 2503, 17, 40, 256), (1, 4001, 33, 1, 200), (31, 20011, 1, 1, 16)])
def test_launches_with_more_pieces_than_ctas(B, T, Hq, Hk, d, dtype):
    """More than 592 pieces: a CTA takes several, its sums of the weights' gradients carried over; more heads than a CTA holds at once."""
    from flash_pop_b200.layer_ops import qk_norm_rotary
    items, rounds, blocks = _items(B, T, Hq, Hk, d)
    assert items > 592 and rounds == 8 and (blocks > 1) == (d >= 200)
    g = torch.Generator(device="cuda").manual_seed(d)
    rnd = lambda *s, t=dtype: torch.randn(*s, generator=g, device="cuda").to(t)
    ph, half = _phasors(1, T, d), HALF[dtype]
    leaves = [rnd(B, T, Hq, d), rnd(B, T, Hk, d), 1 + 0.2 * rnd(d, t=F32), 1 + 0.2 * rnd(d, t=F32)]
    leaves = [t.requires_grad_(True) for t in leaves]
    y, dy = qk_norm_rotary(*leaves, ph, 1e-6), [rnd(B, T, Hq, d), rnd(B, T, Hk, d)]
    grads = torch.autograd.grad(y, leaves, dy)
    # additions behind one another in a weight's gradient: two heads of eight tokens a piece, a CTA's pieces, its groups of lanes, the CTAs'
    # sums by 32 warps and then the warps'; and four operations in each term
    chain = -(-items // 592) * 16 + 256 // min(d // 8, 32) + 592 // 32 + 1 + 32 + 4
    for i in (0, 1):
        x, w = leaves[i].detach().double(), leaves[2 + i].detach().double()
        ref = _formula(x, w, ph, 1e-6)
        # (as in _check)
        assert bool(((y[i].double() - ref).abs() <= half * ref.abs() + 2.0 ** -20 * _row_max(ref) + 1e-30).all())
        r = 1 / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        n, gr = x * r, _formula_back(dy[i].double(), ph)
        gw = gr * w
        ref = r * (gw - n * (gw * n).mean(-1, keepdim=True))
        scale = r * _row_max(dy[i].double()) * 2 * float(w.abs().max())
        assert bool(((grads[i].double() - ref).abs() <= half * ref.abs() + 2.0 ** -18 * scale).all())
        terms = gr * n
        assert bool(((grads[2 + i].double() - terms.sum((0, 1, 2))).abs() <= chain * 2.0 ** -24 * terms.abs().sum((0, 1, 2)) + 1e-30).all())
