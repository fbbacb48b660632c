"""Log probabilities, entropies, alternatives and their gradients, against 64 bits: masks, ties, infinities, odd rows."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}

# z - m and then - log s round a value of the result's size twice (2^-23 of it).  log s: every exponent is off by 2^-24 of itself
# (below 100 where it counts), the sums by 2^-24 for each addition of a chain: together below 512 roundings.  H below 128.
TOL = 512 * 2.0 ** -24


def _reference(z, tokens, top):
    """In doubles, row by row rules of the operator included."""
    z = z.double()
    V = z.size(1)
    empty = (z == -math.inf).all(1)
    bad = z.isnan().any(1) | (z == math.inf).any(1)
    m = z.nan_to_num(0).amax(1, keepdim=True)
    m = torch.where(empty[:, None] | bad[:, None], 0.0, z.amax(1, keepdim=True).nan_to_num(0))
    logp = (z - m) - (z - m).exp().sum(1, keepdim=True).log()
    logp = torch.where(empty[:, None], -math.inf, logp)
    logp = torch.where(bad[:, None], math.nan, logp)
    p = torch.where(empty[:, None], 0.0, logp.exp())
    entropy = -(p * torch.where(p == 0, 0.0, logp)).sum(1)
    inside = (tokens >= 0) & (tokens < V)
    given = torch.where(inside, logp.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0], 0.0)
    index = None
    if top:
        first = torch.where(z.isnan(), math.inf, z)                                       # NaN before all
        order = torch.sort(first, dim=1, descending=True, stable=True).indices
        nan_first = torch.sort(z.isnan().gather(1, order).int(), dim=1, descending=True, stable=True).indices
        index = order.gather(1, nan_first)[:, :top]
    return given, entropy, index, logp, p, inside, empty


def _gradient(ref, tokens, g1, g2, g3):
    given, H, index, logp, p, inside, empty = ref
    g1 = torch.where(inside, g1.double(), 0.0)
    total = g1 + (0 if index is None else g3.double().sum(1))
    d = -p * (total[:, None] + g2.double()[:, None] * (torch.where(p == 0, 0.0, logp) + H[:, None]))
    # (a p below 2^-126, fp32's smallest normal number, counts as 0: off by less than that, times its factor)
    size = torch.where(p == 0, 0.0, p + 2.0 ** -126 / (4 * TOL)) * (total.abs()[:, None] + (g2.double().abs()[:, None] * (torch.where(p == 0, 0.0, logp).abs() + H[:, None])))
    d.scatter_add_(1, tokens.clamp(0, d.size(1) - 1)[:, None], g1[:, None])
    size.scatter_add_(1, tokens.clamp(0, d.size(1) - 1)[:, None], g1.abs()[:, None])
    if index is not None:
        d.scatter_add_(1, index, g3.double())
        size.scatter_add_(1, index, g3.double().abs())
    return torch.where(empty[:, None], 0.0, d), size


def _check(z, tokens, top, grad=True):
    from flash_pop_b200.token_ops import token_scores
    leaf = z.detach().requires_grad_(grad)
    s = token_scores(leaf, tokens, top)
    ref = _reference(z, tokens, top)
    tol = TOL

    def near(a, b):
        return bool((torch.where(b.isfinite(), (a.double() - b).abs() <= tol + 2.0 ** -22 * b.abs(), (a.double() == b) | (a.isnan() & b.isnan()))).all())

    assert s.logprob.dtype == s.entropy.dtype == F32 and near(s.logprob, ref[0])
    assert near(s.entropy, ref[1])
    if top:
        assert torch.equal(s.top_tokens, ref[2])
        assert near(s.top_logprob, ref[3].gather(1, ref[2]))
    else:
        assert s.top_logprob is None and s.top_tokens is None
    if not grad:
        return s
    g = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *sh: torch.randn(*sh, generator=g, device="cuda")
    N = z.size(0)
    gs = [rnd(N), rnd(N)] + ([rnd(N, top)] if top else [])
    ends = [s.logprob, s.entropy] + ([s.top_logprob] if top else [])
    (d,) = torch.autograd.grad(ends, [leaf], gs)
    dref, size = _gradient(ref, tokens, gs[0], gs[1], gs[2] if top else None)
    assert d.shape == z.shape and d.dtype == z.dtype
    err = (d.double() - dref).abs()
    bound = HALF[z.dtype] * dref.abs() + size * 4 * tol + 2.0 ** -126          # (p as log p above; fp32's smallest normal number)
    assert bool(torch.where(dref.isnan(), d.isnan(), err <= bound).all())
    return s


def _logits(N, V, dtype, seed, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(N, V, generator=g, device="cuda") * scale).to(dtype), torch.randint(0, V, (N,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (2, 31, 5), (5, 32, 32), (4, 33, 32), (7, 255, 3), (3, 1000, 20), (2, 2047, 32), (1, 4099, 8),
                                     (300, 513, 4), (9, 16384, 20), (2, 16385, 1), (3, 32000, 20), (1, 50001, 32), (200, 32003, 5), (2, 70000, 32),
                                     (1, 131072, 8), (3, 262147, 20)])
def test_values_and_gradients(N, V, top, dtype):
    z, t = _logits(N, V, dtype, V)
    _check(z, t, top)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [100, 5000, 33000, 100001])
def test_masks_ties_and_extremes(V, dtype):
    z, t = _logits(12, V, dtype, V)
    low = torch.finfo(dtype).min
    z[0] = -math.inf                                             # nothing left
    z[1] = -math.inf
    z[1, V // 3] = 2.0                                           # one token left
    z[2, V // 2:] = -math.inf
    z[3, 10:] = low                                              # masked by the type's lowest value
    z[4] = low                                                    # that alone: all equal
    z[5] = 0                                                      # all equal
    z[6] = (torch.arange(V, device="cuda") % 3).to(dtype)        # a third of the row equal and largest
    z[7, V - 1] = 100.0                                          # sure of the last one
    z[8] = torch.arange(V, device="cuda").to(dtype)              # rising: every piece of the row beats the one before
    z[9, ::2] = -0.0
    z[9, 1::2] = 0.0                                              # both zeros are equal
    z[10] *= 1000
    z[11, 5:9] = z[11].max() + 1                                 # four equal largest
    t[1], t[2], t[3] = V // 3, V - 1, 50
    for top in (0, 1, 4, 32):
        _check(z, t, top)
    _check(z[:1], t[:1], 20)
    _check(z[4:7], t[4:7], 32)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V", [(2100, 9001), (1100, 20000), (2048, 257)])
def test_many_rows_with_masks_and_ties_among_them(N, V, dtype):
    """Rows by the thousand run with fewer threads each; masked, constant and rising ones among them take the longer ways."""
    z, t = _logits(N, V, dtype, N + V)
    z[::7] = -math.inf
    z[::14, V // 2:V // 2 + 9] = 1.0                              # nine tokens left, of one value
    z[1::50] = torch.finfo(dtype).min
    z[1::100, ::3] = -2.0
    z[2::60] = 0.5
    z[3::70] = torch.arange(V, device="cuda").to(dtype)
    z[4::90, 3] = math.nan
    z[5::80, V - 200:] = -math.inf                               # a masked end
    z[6::65, :V - 40] = -math.inf                                # the last forty left
    for top in (0, 8, 32):
        _check(z, t, top, grad=top == 8)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V", [(2048, 16003), (16, 16003), (200, 40010)])
def test_rows_where_the_choice_is_by_digits(N, V, dtype):
    """Rows where more elements reach the bound than there is room for: ties and neighbours at each digit, both signs, every split."""
    z, t = _logits(N, V, dtype, N + V + 1)
    i = torch.arange(V, device="cuda")
    unit = torch.finfo(dtype).eps
    special = [-(V - i) / 64.0,                                   # rising, negative
               torch.where(i % 29 == 5, 3.0, -1.0),               # a few hundred equal largest
               torch.where(i % 29 == 5, -3.0, -5.0) + (i == V - 7) * 1.0,      # negative ones, and one above them
               1.0 + unit * (i * 7 % 113 % 5),                    # neighbours of one another
               -1.0 - unit * (i * 7 % 113 % 5),
               torch.where(i > V // 2, i / 64.0, 0.0),            # rising from the middle on
               torch.where(i < 700, i / 8.0 - 50.0, -70.0),       # a rising start
               torch.where(i == V - 9, math.nan, i / 64.0),
               torch.where(i % 2 == 0, 2.0 ** -130, -(2.0 ** -130))]           # below the normal numbers
    for r, row in enumerate(special):
        z[r::len(special) + 2] = row.to(dtype)
    for top in (1, 8, 31):
        _check(z, t, top, grad=False)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_not_a_number_and_infinity_stay_in_their_rows(dtype):
    for V in (300, 40000):
        z, t = _logits(6, V, dtype, 1)
        z[1, 7], z[2, V - 2], z[3, 5], z[3, 9], z[4, 200:260] = math.nan, math.inf, math.inf, math.nan, math.nan
        s = _check(z, t, 20)
        assert s.logprob.isnan().tolist() == s.entropy.isnan().tolist() == [False, True, True, True, True, False]
        assert s.top_tokens[1, 0] == 7 and s.top_tokens[2, 0] == V - 2 and s.top_tokens[3, :2].tolist() == [9, 5]


def test_tokens_outside_the_vocabulary():
    z, t = _logits(6, 1000, BF, 2)
    t[1], t[2], t[3] = -100, 1000, 2 ** 40
    s = _check(z, t, 3)
    assert s.logprob[1:4].tolist() == [0, 0, 0] and bool((s.entropy > 0).all())


def test_agrees_with_cross_entropy_and_each_gradient_alone():
    from flash_pop_b200.layer_ops import cross_entropy
    from flash_pop_b200.token_ops import token_scores
    z, t = _logits(64, 32000, BF, 3)
    a, b = z.clone().requires_grad_(True), z.clone().requires_grad_(True)
    loss = -token_scores(a, t).logprob.mean()
    want = cross_entropy(b, t)
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5
    ga, gb = torch.autograd.grad(loss, [a])[0], torch.autograd.grad(want, [b])[0]
    assert bool(((ga.double() - gb.double()).abs() <= 2.0 ** -7 * gb.double().abs() + 1e-9).all())
    s = token_scores(a, t, 4)
    parts = [torch.autograd.grad(e.sum(), [a], retain_graph=True)[0].double() for e in (s.logprob, s.entropy, s.top_logprob)]
    whole = torch.autograd.grad(s.logprob.sum() + s.entropy.sum() + s.top_logprob.sum(), [a])[0].double()
    assert bool(((sum(parts) - whole).abs() <= 2.0 ** -7 * sum(p.abs() for p in parts) + 1e-9).all())
    assert not s.top_tokens.requires_grad


def test_gradient_against_differences():
    from flash_pop_b200.token_ops import token_scores
    z, t = _logits(4, 50, F32, 4, scale=1.0)
    g = torch.Generator(device="cuda").manual_seed(6)
    u, v, w, way = (torch.randn(*s, generator=g, device="cuda") for s in ((4,), (4,), (4, 3), (4, 50)))

    def f(z):
        s = token_scores(z, t, 3)
        return float((s.logprob.double() * u).sum() + (s.entropy.double() * v).sum() + (s.top_logprob.double() * w).sum())

    leaf = z.clone().requires_grad_(True)
    s = token_scores(leaf, t, 3)
    (d,) = torch.autograd.grad([s.logprob, s.entropy, s.top_logprob], [leaf], [u, v, w])
    h = 2.0 ** -9                                                 # (far below the gaps between the largest logits)
    assert abs(float((d * way).sum()) - (f(z + h * way) - f(z - h * way)) / (2 * h)) < 2e-2


def test_shapes_strides_and_rows_behind_the_last():
    from flash_pop_b200.token_ops import token_scores
    g = torch.Generator(device="cuda").manual_seed(7)
    for dtype in (BF, F32):
        z = torch.randn(3, 5, 1003, generator=g, device="cuda").to(dtype)
        t = torch.randint(0, 1003, (3, 5), generator=g, device="cuda")
        want = token_scores(z, t, 6)
        buf = torch.randn(3, 5, 1010, generator=g, device="cuda").to(dtype)
        buf[..., 3:1006] = z
        for view, ids in ((buf[..., 3:1006], t), (z, t.int()), (z.transpose(0, 1).contiguous().transpose(0, 1), t)):
            got = token_scores(view, ids, 6)
            # (rows that start elsewhere against 16 bytes may be summed in another order)
            assert torch.equal(got.top_tokens, want.top_tokens)
            assert all(bool(((a - b).abs() <= 512 * 2.0 ** -24).all()) for a, b in zip(got[:3], want[:3]))
        one = token_scores(z[1, 2], t[1, 2], 6)
        assert one.logprob.shape == () and one.top_tokens.shape == (6,)
        # the sums of a row do not depend on how many rows there are, up to the order of their additions
        assert torch.equal(one.top_tokens, want.top_tokens[1, 2]) and abs(float(one.logprob - want.logprob[1, 2])) < 1e-5
        none = token_scores(z[:0], t[:0], 2)
        assert none.logprob.shape == (0, 5) and none.top_tokens.shape == (0, 5, 2)
        leaf = z.clone().requires_grad_(True)
        (d,) = torch.autograd.grad(token_scores(leaf.transpose(0, 1), t.t()).logprob.sum(), [leaf])
        assert d.shape == z.shape
    row = torch.randn(1, 1003, device="cuda").expand(4, 1003)
    assert token_scores(row, t[0, :4], 2).top_tokens.unique(dim=0).size(0) == 1


def test_rows_beyond_32_bits():
    V = 32000
    N = (1 << 32) // V + 3
    z = torch.zeros(N, V, device="cuda", dtype=BF)
    z[-1, 31999] = 9.0
    t = torch.full((N,), 31999, device="cuda")
    from flash_pop_b200.token_ops import token_scores
    leaf = z.requires_grad_(True)
    s = token_scores(leaf, t, 2)
    assert s.top_tokens[-1].tolist() == [31999, 0] and s.top_tokens[-2].tolist() == [0, 1]
    assert abs(float(s.logprob[-2].detach()) + math.log(V)) < 1e-5
    (d,) = torch.autograd.grad(s.logprob.sum(), [leaf])
    p = math.exp(9) / (math.exp(9) + V - 1)
    assert abs(float(d[-1, 31999]) - (1 - p)) < 2.0 ** -8 and abs(float(d[-1, 0]) + p / math.exp(9)) < 1e-6


def test_same_bits_twice_and_in_a_graph():
    from flash_pop_b200.token_ops import token_scores
    for N in (3, 500):
        z, t = _logits(N, 32000, BF, 8)
        z.requires_grad_(True)

        def step():
            s = token_scores(z, t, 20)
            return [x.detach() for x in s] + list(torch.autograd.grad(s.logprob.sum() + s.entropy.sum(), [z]))

        want = step()
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                held = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


FILLS = [-1e5, -1e9, -5e9, -1e10, -1e12, -1e15, -1e20, -1e25]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [100, 5000, 33000, 100001])
def test_finite_masks_of_any_size(V, dtype):
    """A masked start, a masked end, all masked but a few, and all: whatever number stands for the mask."""
    z, t = _logits(4 * len(FILLS), V, dtype, V + 11)
    for i, fill in enumerate(FILLS):
        z[4 * i, :V // 2] = z[4 * i + 1, V // 2:] = z[4 * i + 3] = fill
        kept = z[4 * i + 2, V // 3:V // 3 + 4].clone()
        z[4 * i + 2] = fill
        z[4 * i + 2, V // 3:V // 3 + 4] = kept
    t[::4] = V - 1                                               # one given token that is not masked, of the others some are
    for top in (0, 3, 20, 32):
        _check(z, t, top)


def _large_rows(V, dtype):
    """Rows whose largest element is huge, or that pass from one size to another."""
    i = torch.arange(V, device="cuda", dtype=torch.float64)
    g = torch.Generator(device="cuda").manual_seed(V)
    noise = torch.randn(V, generator=g, device="cuda", dtype=torch.float64)
    rows = []
    for m in (3e9, 5e9, 1e10, 1e12, 1e20, 1e38):
        for sign in (1, -1):
            rows += [torch.full_like(i, sign * m),                                   # all equal
                     sign * m * (1 + torch.finfo(dtype).eps * (i % 3)),              # neighbours of one another
                     torch.where(i == V // 2, sign * m, 3 * noise if sign > 0 else 2 * sign * m)]      # one above the others
    for edge in (2.0 ** 18, 2.0 ** 20, 2.0 ** 24):                                  # up and down across sizes where fewer bits are left
        step = edge * torch.finfo(dtype).eps
        for sign in (1, -1):
            rows += [sign * edge + (i - V // 2) * step, sign * edge - (i - V // 2) * step, sign * edge + (i % 7 - 3) * step]
        rows.append(torch.where(i % 2 == 0, edge, -edge) + noise)
    rows += [noise - 5e9, torch.where(i < V // 2, -2.0 ** 19 - i, 2.0 ** 21), torch.where(i < V // 2, -2.0 ** 21 - i, 2.0 ** 19),
             torch.where(i < V // 2, -2.0 ** 21 - i, noise), torch.where(i < V // 2, -2.0 ** 20 + noise, -2.0 ** 20 - 1 + noise)]
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [7, 100, 5000, 33000, 100001])
def test_finite_rows_of_any_size(V, dtype):
    z = _large_rows(V, dtype)
    assert bool(z.isfinite().all())
    t = torch.randint(0, V, (z.size(0),), generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    t[::2] = z[::2].float().argmax(1)
    for top in (0, min(V, 5), min(V, 32)):
        _check(z, t, top)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_rows_of_any_size(dtype):
    V = 9001
    rows = _large_rows(V, dtype)
    z, t = _logits(2100, V, dtype, 12)
    z[:40 * rows.size(0)] = rows.repeat(40, 1)[:2100]
    z[-300::8, :V // 2] = -1e10
    z[-299::8, 9:] = -5e9
    for top in (0, 8):
        _check(z, t, top)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V", [(60, 40), (60, 511), (2100, 517), (60, 1023), (60, 1031), (2100, 4003), (60, 9001)])
def test_more_alternatives_than_half_of_the_parts(N, V, dtype):
    z, t = _logits(N, V, dtype, N + V + 2)
    z[::6] = -math.inf
    z[::12, V // 3:V // 3 + 18] = 1.0
    z[1::6] = torch.arange(V, device="cuda").to(dtype)
    z[2::6] = -0.5
    z[3::6, 20:] = torch.finfo(dtype).min
    z[4::18, 5] = math.nan
    for top in (15, 16, 17, 20, 21, 24, 31, 32):
        _check(z, t, top, grad=False)
