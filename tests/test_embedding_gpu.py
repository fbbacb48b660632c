"""Embedding lookup and the table's gradient, against 64 bits: sizes where tiles, digits and windows end, repeated and missing ids."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}


def _check(tokens, V, D, dtype, scale=1.0, padding=None, weight=None, dy=None):
    from flash_pop_b200.token_ops import embedding
    g = torch.Generator(device="cuda").manual_seed(V + D)
    w = torch.randn(V, D, generator=g, device="cuda").to(dtype) if weight is None else weight
    w = w.detach().requires_grad_(True)
    y = embedding(tokens, w, scale, padding)
    assert y.shape == (*tokens.shape, D) and y.dtype == dtype
    flat = tokens.flatten()
    inside = (flat >= 0) & (flat < V)
    safe = flat.clamp(0, V - 1).long()
    ref = torch.where(inside[:, None], w.detach().double()[safe] * scale, 0.0).view(y.shape)
    assert bool(((y.double() - ref).abs() <= (HALF[dtype] + 2.0 ** -23) * ref.abs()).all())       # rounded once, the scale in fp32
    dy = torch.randn(y.shape, generator=g, device="cuda").to(dtype) if dy is None else dy
    (got,) = torch.autograd.grad(y, [w], dy)
    used = inside if padding is None else inside & (flat != padding % V)
    terms = torch.where(used[:, None], dy.double().reshape(-1, D), 0.0)
    ref = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, safe, terms) * scale
    size = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, safe, terms.abs()) * abs(scale)
    n = torch.bincount(safe, minlength=V)[:, None].double()
    # one rounding of the result; each of the n - 1 additions and the scale round a partial sum below the sum of the sizes
    assert got.shape == (V, D) and got.dtype == dtype
    assert bool(((got.double() - ref).abs() <= HALF[dtype] * ref.abs() + (n + 1) * 2.0 ** -24 * size * 1.01).all())
    assert bool((got[(size == 0).all(1)] == 0).all())
    (again,) = torch.autograd.grad(embedding(tokens, w, scale, padding), [w], dy)
    assert torch.equal(got, again)
    return got


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 300, 8), (2, 3, 5), (31, 2, 64), (64, 64, 24), (65, 255, 100), (129, 256, 128), (1000, 257, 333),
                                   (4095, 4000, 40), (4096, 65535, 16), (4097, 65536, 8), (9001, 70000, 7), (20000, 33, 72), (3000, 1000, 1288),
                                   (777, 500, 2056)])
def test_values_and_gradients(N, V, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(N)
    _check(torch.randint(0, V, (N,), generator=g, device="cuda"), V, D, dtype, scale=1.5)


@pytest.mark.parametrize("D", [72, 333, 1024])
def test_repeated_missing_and_foreign_ids(D):
    g = torch.Generator(device="cuda").manual_seed(D)
    N, V = 9000, 5000
    same = torch.full((N,), 4321, device="cuda")
    _check(same, V, D, BF)
    _check(torch.zeros(N, dtype=torch.int64, device="cuda"), V, D, F32, scale=-0.5)
    _check(torch.full((300,), V - 1, device="cuda"), V, D, BF)
    _check(torch.arange(N, device="cuda") % 7 * 700, V, D, BF)
    _check(torch.arange(N, device="cuda") // 129, V, D, F32)                           # runs that end inside, at and over windows
    mixed = torch.randint(-5, V + 5, (N,), generator=g, device="cuda")
    mixed[::7], mixed[1::11], mixed[2::13] = -100, 2 ** 40, -2 ** 63
    _check(mixed, V, D, BF, padding=3)
    _check(torch.full((N,), -1, device="cuda"), V, D, BF)                              # no id inside: a table of zeros
    got = _check(same, V, D, BF, padding=4321)
    assert bool((got == 0).all())
    _check(mixed, V, D, F32, padding=-1)


def test_more_ids_than_the_sort_has_tiles_for():
    g = torch.Generator(device="cuda").manual_seed(3)
    for N, V in ((1_100_000, 3000), (2_200_003, 40), (1_048_577, 200_000)):
        _check(torch.randint(-1, V, (N,), generator=g, device="cuda"), V, 8, BF)


def test_shapes_types_and_strides():
    from flash_pop_b200.token_ops import embedding
    g = torch.Generator(device="cuda").manual_seed(0)
    V, D = 100, 64
    t = torch.randint(0, V, (4, 9), generator=g, device="cuda")
    _check(t, V, D, BF)
    _check(t.t(), V, D, BF)
    _check(t[:, ::2], V, D, F32)
    _check(t.int(), V, D, BF)
    _check(t[0, 0], V, D, BF)                                                            # a scalar id
    _check(t[:, :1].expand(4, 9), V, D, BF)
    wide = torch.randn(V, 2 * D + 8, generator=g, device="cuda").to(BF)
    _check(t, V, D, BF, weight=wide[:, 8:D + 8])                                       # rows of a wider matrix
    _check(t, V, D, BF, weight=wide[:, 1:D + 1])                                       # not aligned
    _check(t, V, D, BF, weight=torch.randn(D, V, device="cuda").to(BF).t())            # transposed
    _check(t, V, D, BF, dy=torch.randn(4, 1, D, generator=g, device="cuda").to(BF).expand(4, 9, D))
    _check(t, V, D, BF, dy=torch.randn(4, 9, 2 * D, generator=g, device="cuda").to(BF)[..., 1:D + 1])
    w = torch.randn(V, D, device="cuda", requires_grad=True)
    y = embedding(t[:0], w)
    assert y.shape == (0, 9, D) and bool((torch.autograd.grad(y.sum(), [w])[0] == 0).all())


def test_plain_lookup_equals_the_frameworks():
    g = torch.Generator(device="cuda").manual_seed(1)
    from flash_pop_b200.token_ops import embedding
    w = torch.randn(1000, 1024, generator=g, device="cuda").to(BF)
    t = torch.randint(0, 1000, (3, 500), generator=g, device="cuda")
    assert torch.equal(embedding(t, w), torch.nn.functional.embedding(t, w))


def test_rows_of_a_large_table_and_of_a_large_gradient():
    from flash_pop_b200.token_ops import embedding
    V, D = 1_100_000, 2048                                                             # 2.25e9 elements: offsets pass 32 bits
    w = torch.zeros(V, D, device="cuda", dtype=BF)
    w[-1], w[1_050_000] = 3, 5
    w.requires_grad_(True)
    t = torch.tensor([V - 1, 1_050_000, 0, V - 1], device="cuda")
    y = embedding(t, w)
    assert y[:, 0].tolist() == [3, 5, 0, 3] and bool((y == y[:, :1]).all())
    (g,) = torch.autograd.grad(y, [w], torch.ones_like(y))
    assert g[[V - 1, 1_050_000, 0, 1, V - 2], 7].tolist() == [2, 1, 1, 0, 0] and float(g[:, 2047].float().sum()) == 4


def test_two_captured_steps_and_another_stream():
    from flash_pop_b200.token_ops import embedding
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(3000, 256, generator=g, device="cuda").to(BF).requires_grad_(True)
    ids = [torch.randint(0, 3000, (n,), generator=g, device="cuda") for n in (700, 9000)]
    dys = [torch.randn(n, 256, generator=g, device="cuda").to(BF) for n in (700, 9000)]
    step = lambda i: torch.autograd.grad(embedding(ids[i], w, 2.0), [w], dys[i])[0]
    want = [step(0), step(1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, held, pool = [], [], torch.cuda.graph_pool_handle()
    with torch.cuda.stream(side):
        step(0), step(1)
        for i in range(2):                                                             # two graphs over one pool of memory
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=pool, stream=side):
                held.append(step(i))
            graphs.append(graph)
    for i in (1, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(held[i], want[i])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V,D", [(8191, 5000, 64), (8192, 8001, 65), (8193, 8001, 64), (8192, 1, 40), (5003, 8001, 333), (33, 200_003, 63), (7, 1 << 20, 72),
                                   (1000, 100, 1), (3000, 7, 1024), (8192, 24, 520), (257, 1500, 9608), (130, 90, 9601), (1, 5, 19_000)])
def test_gradients_of_a_few_ids(N, V, D, dtype):
    """Up to 8192 ids the gradient is one launch: tables of fewer rows than shares of it, tiles of 64 columns with a rest, more tiles than CTAs."""
    g = torch.Generator(device="cuda").manual_seed(N + D)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    _check(t, V, D, dtype, scale=0.75, padding=0)
    # as words fall: a few ids in every piece, most of them rare
    t = (V ** torch.rand(N, generator=g, device="cuda", dtype=torch.float64)).long() - 1
    t[N // 3:N // 3 + N // 10] = -100
    _check(t, V, D, dtype)


@pytest.mark.parametrize("D", [8, 333, 1024])
def test_runs_over_the_pieces_of_a_few_ids(D):
    N, V = 8192, 4000
    i = torch.arange(N, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(D)
    for n in (1, 2, 127, 128, 129, 1000, N):                       # one run: a piece each of one row or more
        _check(i[:n] * 0 + 3999, V, D, BF)
    for ids in (i % 2 * 1000, i // 64, i // 65, i // 63 * 9, i % 3 * 148, (i > 5) * 17, (i == N - 1) * 8, i // 4096 * 24,
                torch.where(i % 5 == 0, 11, i // 2 % V)):          # runs that end at, before and behind pieces' ends
        order = torch.randperm(N, generator=g, device="cuda")
        _check(ids, V, D, F32)
        _check(ids[order], V, D, BF)


def test_the_node_is_an_ordinary_one():
    """Saved tensors through hooks, freed or changed ones, an absent gradient, a second derivative, and a backward pass that is compiled."""
    from flash_pop_b200.token_ops import embedding
    w = torch.randn(50, 16, device="cuda", requires_grad=True)
    t = torch.randint(0, 50, (9,), device="cuda")
    (want,) = torch.autograd.grad(embedding(t, w, 2.0).sum(), [w])
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda x: packed.append(x.shape) or x.cpu(), lambda x: x.cuda()):
        y = embedding(t, w, 2.0)
    assert packed == [t.shape] and torch.equal(torch.autograd.grad(y.sum(), [w])[0], want)
    y = embedding(t, w, 2.0)
    y.sum().backward()
    assert torch.equal(w.grad, want) and y.grad_fn.name() == "EmbeddingBackward"
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    y = embedding(t, w, 2.0)
    t += 0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    (none,) = torch.autograd.grad(torch._C._functions.UndefinedGrad()(embedding(t, w)).sum(), [w], allow_unused=True)
    assert none is None
    with torch.autograd.detect_anomaly(check_nan=False):
        (got,) = torch.autograd.grad(embedding(t, w, 2.0).sum(), [w])
    assert torch.equal(got, want)
    import torch._dynamo.compiled_autograd as compiled
    for ids, table in ((t, w), (t, w), (torch.randint(0, 900, (3, 4000), device="cuda"), torch.randn(900, 8, device="cuda").to(BF).requires_grad_(True))):
        (want,) = torch.autograd.grad(embedding(ids, table, 0.5, 3).sum(), [table])
        table.grad = None
        with compiled._enable(torch.compile(backend="eager")):
            embedding(ids, table, 0.5, 3).sum().backward()
        assert torch.equal(table.grad, want)


@pytest.mark.parametrize("N,V,D,dtype", [(100, 131_072, 63, F32), (100, 131_073, 63, F32), (3000, 65_536, 100, BF), (3000, 65_537, 100, BF), (8192, 300_001, 5, BF),
                                         (500, 1 << 20, 8, BF), (500, (1 << 20) + 1, 8, F32), (1, 530_000, 72, BF), (8192, 200_000, 333, F32)])
def test_tables_on_both_sides_of_where_they_are_cleared_first(N, V, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(V + N)
    _check(torch.randint(0, V, (N,), generator=g, device="cuda"), V, D, dtype)
    _check(torch.full((N,), -1, device="cuda"), V, D, dtype)                           # nobody writes: zeros alone, whatever was there


def test_what_follows_a_gradient_waits_for_its_clearing():
    """A large table cleared by a launch of its own, and no id that anything waits for: what reads the result next sees zeros."""
    from flash_pop_b200.token_ops import embedding
    w = torch.zeros(3_000_000, 33, device="cuda", dtype=BF, requires_grad=True)
    t, dy = torch.full((5,), -1, device="cuda"), torch.ones(5, 33, device="cuda", dtype=BF)
    for _ in range(5):
        junk = torch.full((3_000_000, 33), 7.0, device="cuda", dtype=BF)                # (the memory that the gradient gets)
        del junk
        (got,) = torch.autograd.grad(embedding(t, w), [w], dy)
        assert float(got.abs().max()) == 0
        del got
