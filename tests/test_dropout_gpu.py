"""Dropout without a stored mask: the mask against the generator's published test vectors and its definition on the host, the sums,
the gradients, the module."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _philox(counter, key):
    """Philox4x32-10 in Python integers, from the paper's definition."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def _halves(n, seed, first=0):
    out = []
    for g in range(first // 8, (n + 7) // 8):
        for w in _philox([g & 0xFFFFFFFF, g >> 32, 0, 0], [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]):
            out += [w & 0xFFFF, w >> 16]
    return np.array(out[:n - first // 8 * 8])


def test_the_host_generator_gives_the_published_vectors():
    """Known answers that the generator's authors publish for philox4x32 with 10 rounds (all zeros, all ones, digits of pi)."""
    assert _philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert _philox([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert _philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def _seed(s):
    return torch.tensor([s], dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,p,seed", [(1, 0.5, 0), (7, 0.1, 1), (8, 0.9, -1), (9, 0.25, 2 ** 62 + 12345), (2049, 0.1, 77), (5000, 0.333, -(2 ** 63))])
def test_mask_values_and_gradients(n, p, seed, dtype):
    from flash_pop_b200.layer_ops import dropout
    g = torch.Generator(device="cuda").manual_seed(n)
    x, r, dy = (torch.randn(n, generator=g, device="cuda").to(dtype) for _ in range(3))
    threshold = round(p * 65536)
    keep = torch.from_numpy(_halves(n, seed & (2 ** 64 - 1)) >= threshold).cuda()
    factor = 65536 / (65536 - threshold)
    half = 2.0 ** -8 if dtype == BF else 2.0 ** -24
    for res in (None, r):
        leaf, rl = x.clone().requires_grad_(True), None if res is None else r.clone().requires_grad_(True)
        y = dropout(leaf, p, _seed(seed), rl)
        dropped = torch.where(keep, x.double() * factor, 0.0)
        ref = dropped if res is None else r.double() + dropped
        # the result's rounding; the factor's, the product's and the sum's in fp32
        assert bool(((y.double() - ref).abs() <= half * ref.abs() + 3 * 2.0 ** -24 * (dropped.abs() + ref.abs())).all())
        assert bool((y[~keep] == (0 if res is None else r[~keep])).all())
        grads = torch.autograd.grad(y, [leaf] if res is None else [leaf, rl], dy)
        ref = torch.where(keep, dy.double() * factor, 0.0)
        assert bool(((grads[0].double() - ref).abs() <= (half + 2 * 2.0 ** -24) * ref.abs()).all())
        assert res is None or torch.equal(grads[1], dy)


def test_places_beyond_32_bits_of_bytes_and_elements():
    from flash_pop_b200.layer_ops import dropout
    n = (1 << 32) + 19                              # 8.6 GB of bf16: the last elements lie behind the 2^32nd
    x = torch.ones(n, device="cuda", dtype=BF)
    y = dropout(x, 0.5, _seed(5))
    del x
    for first in (0, (1 << 31) - 8, (1 << 32) - 8):
        want = torch.from_numpy(_halves(min(first + 27, n), 5, first) >= 32768)
        assert torch.equal(y[first:first + want.numel()].cpu() == 2, want)
    assert abs(float(y[:1 << 28].float().mean()) - 1) < 5 * 2.0 ** -14          # five standard deviations of the mean


def test_edges_of_p_and_of_the_values():
    from flash_pop_b200.layer_ops import dropout
    x = torch.tensor([1.0, float("inf"), float("nan"), -2.0] * 500, device="cuda")
    x.requires_grad_(True)
    assert torch.equal(dropout(x, 0.0, _seed(1)).nan_to_num(), x.detach().nan_to_num())
    y = dropout(x, 1.0, _seed(1))
    assert bool((y == 0).all()) and bool((torch.autograd.grad(y.sum(), [x])[0] == 0).all())
    r = torch.full_like(x, 3.0).detach()
    assert torch.equal(dropout(x, 1.0, _seed(1), r), r)
    y = dropout(x, 0.5, _seed(1))
    gone = torch.from_numpy(_halves(2000, 1) < 32768).cuda()
    assert bool((y[gone] == 0).all()) and bool(torch.isnan(y[~gone][x[~gone].isnan()]).all())
    assert dropout(x[:0], 0.5, _seed(1)).shape == (0,)


def test_strides_alignment_and_shape_do_not_move_the_mask():
    from flash_pop_b200.layer_ops import dropout
    for dtype in (BF, F32):
        buf = torch.randn(3, 50, 71, device="cuda").to(dtype)
        want = dropout(buf, 0.3, _seed(9))
        flat = torch.cat((buf.new_zeros(1), buf.flatten()))[1:]                         # not 16-byte aligned
        assert torch.equal(dropout(flat, 0.3, _seed(9)), want.flatten())
        t = buf.transpose(0, 2).contiguous().transpose(0, 2)
        assert torch.equal(dropout(t, 0.3, _seed(9), t), dropout(buf, 0.3, _seed(9), buf))
        leaf = buf.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(dropout(leaf, 0.3, _seed(9)).sum(), [leaf])       # an expanded gradient
        assert torch.equal(g, dropout(torch.ones_like(buf), 0.3, _seed(9)))


def test_module_draws_from_torchs_generator():
    from flash_pop_b200.layer_ops import CounterDropout
    m, x, r = CounterDropout(0.4), torch.randn(64, 129, device="cuda").to(BF), torch.randn(64, 129, device="cuda").to(BF)
    torch.manual_seed(3)
    a, b = m(x, r), m(x, r)
    torch.manual_seed(3)
    assert torch.equal(m(x, r), a) and not torch.equal(a, b)
    torch.manual_seed(3)
    wide = m(x, r.float())                                       # a residual of another type is added as torch adds it
    torch.manual_seed(3)
    assert wide.dtype == F32 and torch.equal(wide, r.float() + m(x))
    m.eval()
    assert m(x) is x and torch.equal(m(x, r), r + x)
    m.train()
    # checkpointing brings the same masks back
    from torch.utils.checkpoint import checkpoint
    leaf = x.float().requires_grad_(True)
    torch.manual_seed(4)
    (want,) = torch.autograd.grad(m(leaf * 1).sum(), [leaf])
    torch.manual_seed(4)
    (got,) = torch.autograd.grad(checkpoint(lambda t: m(t * 1), leaf, use_reentrant=False).sum(), [leaf])
    assert torch.equal(got, want)


def test_a_captured_call_draws_anew_at_every_replay():
    from flash_pop_b200.layer_ops import CounterDropout
    m = CounterDropout(0.5)
    x = torch.ones(4096, device="cuda", requires_grad=True)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.autograd.grad(m(x).sum(), [x])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = m(x)
            (g,) = torch.autograd.grad(y.sum(), [x])
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, g)                     # of ones: value and gradient are both the scaled mask
        seen.append(y.detach().clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
