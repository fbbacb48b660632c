"""The language model with its embedding, query/key norms, dropout and token scores together, as a training, a scoring and a
decoding program use them."""
import math

import pytest
import torch

from oracle import retention_oracle as orc

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
OPTIONS = dict(embed_scale=math.sqrt(128), qk_norm=True, counter_dropout=True)


def _model(dropout=0.0, **kw):
    from flash_pop_b200.stack_lm import RetNetLM
    torch.manual_seed(0)
    m = RetNetLM(vocab_size=999, num_layers=2, num_heads=2, head_dim=64, dim_feedforward=192, dropout=dropout, **{**OPTIONS, **kw})
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "norm_weight" in n:
                p.mul_(torch.rand_like(p) + 0.5)
    return m


def _tokens(B=3, T=150, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, 999, (B, T), generator=g, device="cuda")


def _forward64(m, params, tokens):
    """The model in doubles on the host, from its formulas; `params`: names to doubles."""
    F = torch.nn.functional
    c = m.decoder.layer_config
    H, d = c.num_heads, c.head_dim_v
    x = params["embed.weight"][tokens] * m.embed_scale
    theta = 10000.0 ** -torch.linspace(0, 1, d // 2, dtype=torch.float64)
    angle = torch.arange(tokens.size(1), dtype=torch.float64)[:, None] * theta
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def normed(t, w):
        t = t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)

    for i in range(len(m.decoder.layers)):
        p = {k[len(f"decoder.layers.{i}."):]: v for k, v in params.items() if k.startswith(f"decoder.layers.{i}.")}
        lin = lambda n, t: F.linear(t, p[n + ".weight"], p[n + ".bias"])
        h = F.layer_norm(x, x.shape[-1:], p["norm1.weight"], p["norm1.bias"], 1e-6)
        q, k, v = (lin(f"retention.{n}_proj", h).unflatten(-1, (H, d)) for n in "qkv")
        q, k = normed(q, p["retention.q_norm_weight"]), normed(k, p["retention.k_norm_weight"])
        o, _ = orc.retention_chunkwise(q, k, v, torch.zeros(x.size(0), H, d, d, dtype=torch.float64),
                                       m.decoder.layers[i].retention.head_decays, 64)
        o = F.layer_norm(o, o.shape[-1:], None, None, 1e-6).flatten(-2)
        x = x + lin("retention.out_proj", o * F.silu(lin("retention.g_proj", h)))
        h = F.layer_norm(x, x.shape[-1:], p["norm2.weight"], p["norm2.bias"], 1e-6)
        x = x + lin("linear2", F.silu(lin("linear1", h)))
    return F.linear(F.layer_norm(x, x.shape[-1:], params["norm.weight"], params["norm.bias"], m.norm.eps), params["head.weight"])


def test_scores_and_gradients_against_64_bits():
    m, tokens = _model(), _tokens()
    s = m.score(tokens, top=5)
    assert s.logprob.shape == s.entropy.shape == (3, 149) and s.top_tokens.shape == (3, 149, 5)
    objective = s.logprob.mean() + 0.1 * s.entropy.mean() + 0.05 * s.top_logprob.mean()
    got = torch.autograd.grad(objective, list(m.parameters()))
    params = {n: p.detach().double().cpu().requires_grad_(True) for n, p in m.named_parameters()}
    logp = torch.log_softmax(_forward64(m, params, tokens[:, :-1].cpu()), -1)
    entropy = -(logp.exp() * logp).sum(-1)
    given = logp.gather(-1, tokens[:, 1:, None].cpu())[..., 0]
    # bf16 activations: some 20 roundings of 2^-9 of the logits (of size 4) on the way
    assert float((s.logprob.detach().cpu() - given).abs().max()) < 0.15 and float((s.entropy.cpu() - entropy).abs().max()) < 0.1
    chosen = logp.gather(-1, s.top_tokens.cpu())
    assert float((s.top_logprob.cpu() - chosen).abs().max()) < 0.15
    ref = torch.autograd.grad(given.mean() + 0.1 * entropy.mean() + 0.05 * chosen.mean(), list(params.values()))
    for n, a, b in zip(params, got, ref):
        # two layers of bf16 gradients: as a stack without these operators is off (1.1e-2), with room for small tensors
        assert float((a.double().cpu() - b).norm() / b.norm()) < 5e-2, n


def test_tokens_one_by_one_give_the_scores_of_the_whole():
    m, tokens = _model().eval(), _tokens(B=2, T=21)
    from flash_pop_b200.layer_ops import norm_in_fp32
    from flash_pop_b200.token_ops import embedding, token_scores
    with torch.no_grad():
        whole = m.score(tokens, top=3)
        state, steps = None, []
        for t in range(20):
            x = embedding(tokens[:, t], m.embed.weight, m.embed_scale)
            x, state = m.decoder.forward_recurrent(x, state)
            steps.append(token_scores(m.head(norm_in_fp32(m.norm, x)), tokens[:, t + 1], top=3))
    for i in (0, 1):
        assert float((torch.stack([s[i] for s in steps], 1) - whole[i]).abs().max()) < 0.15
    assert state.index == 20


def test_dropout_in_one_pass_with_the_residual_matches_two():
    m, tokens = _model(dropout=0.2), _tokens()
    results = []
    for fused in (True, False):
        if not fused:
            for layer in m.decoder.layers:
                layer._adds_dropout = lambda: False
        torch.manual_seed(11)
        loss = -m.score(tokens).logprob.mean()
        results.append([loss.detach(), *torch.autograd.grad(loss, list(m.parameters()))])
    for a, b in zip(*results):                                   # the same masks; one rounding less in the fused pass
        assert float((a.double() - b.double()).norm() / b.double().norm()) < 3e-2
    torch.manual_seed(12)
    assert float(-m.score(tokens).logprob.mean()) != float(results[1][0])
    m.eval()
    assert torch.equal(m.score(tokens).logprob, m.score(tokens).logprob)


def test_a_scoring_step_with_the_table_gradient_in_a_graph():
    m, tokens = _model(), _tokens(seed=3)
    table = m.embed.weight

    def step():
        s = m.score(tokens, top=2)
        return [s.logprob.detach(), s.top_tokens, *torch.autograd.grad(s.logprob.sum(), [table])]

    want = step()
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
    for a, b in zip(held, want):
        assert torch.equal(a, b)


def test_a_padded_batch_and_the_shortest_sequences():
    m, tokens = _model(), _tokens(B=3, T=40)
    table = m.embed.weight
    whole = m.score(tokens[:2, :25], top=4)
    want = torch.autograd.grad(whole.logprob.sum(), [table])[0]
    padded = tokens.clone()
    padded[:2, 25:] = -1                                         # no token: a zero row, the log probability 0, no gradient
    s = m.score(padded[:2], top=4)
    assert bool((s.logprob[:, 24:] == 0).all()) and bool(torch.isfinite(s.entropy).all())
    assert float((s.logprob[:, :24] - whole.logprob).detach().abs().max()) < 0.1          # (other lengths, other sums: bf16)
    got = torch.autograd.grad(s.logprob.sum(), [table])[0]
    assert float((got.double() - want.double()).norm() / want.double().norm()) < 5e-2
    for T in (0, 1):
        s = m.score(tokens[:, :T], top=2)
        assert s.logprob.shape == (3, 0) and s.top_tokens.shape == (3, 0, 2)
    assert m.score(tokens[:, :2]).logprob.shape == (3, 1)


def test_calls_on_two_streams_at_once():
    from flash_pop_b200 import layer_ops, token_ops
    g = torch.Generator(device="cuda").manual_seed(0)
    z, t = torch.randn(64, 20011, generator=g, device="cuda").to(BF).requires_grad_(True), torch.randint(0, 20011, (64,), generator=g, device="cuda")
    w, ids = torch.randn(3000, 320, generator=g, device="cuda").to(BF).requires_grad_(True), torch.randint(0, 3000, (20000,), generator=g, device="cuda")
    q = torch.randn(2, 300, 4, 64, generator=g, device="cuda").to(BF).requires_grad_(True)
    weight, seed = torch.rand(64, device="cuda", requires_grad=True), torch.tensor([9], device="cuda")

    def work():
        s = token_ops.token_scores(z, t, 20)
        y = layer_ops.dropout(token_ops.embedding(ids, w, 2.0), 0.1, seed)
        a, b = layer_ops.qk_norm_rotary(q, q, weight, None, None)
        return [s.logprob.detach(), s.top_tokens, *torch.autograd.grad([s.entropy.sum(), y.float().sum(), (a + b).float().sum()], [z, w, q, weight])]

    want = work()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(work())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_options_are_off_by_default_and_other_layers_take_them():
    import flash_pop_b200 as fp
    from flash_pop_b200.layer_ops import CounterDropout
    from flash_pop_b200.stack_lm import RetNetLM
    plain = RetNetLM(vocab_size=50, num_layers=1, num_heads=2, head_dim=16, dim_feedforward=32)
    assert plain.embed_scale is None and type(plain.decoder.layers[0].dropout) is torch.nn.Dropout
    assert not [n for n in plain.state_dict() if "norm_weight" in n]
    cfg = fp.POPDecoderLayer.Config(num_heads=2, head_dim_v=32, dim_feedforward=64, dropout=0.1, block_size=8, qk_norm=True, counter_dropout=True)
    pop = fp.POPRetNetDecoder(cfg, 1)
    x, sfx = torch.randn(2, 24, 64, device="cuda").to(BF), torch.randn(2, 3, 4, 64, device="cuda").to(BF)
    y, _, ys = pop.pop_forward(x, None, sfx)
    torch.autograd.grad(y.float().sum() + ys.float().sum(), list(pop.parameters()))
    assert type(pop.layers[0].dropout) is CounterDropout and y.shape == x.shape and ys.shape == sfx.shape
    lc = fp.DiffusionRetNetDecoderLayer.Config(num_heads=2, head_dim_v=32, dim_feedforward=64, dropout=0.1, qk_norm=True, counter_dropout=True)
    net = fp.DiffusionRetNetDecoder(fp.DiffusionRetNetDecoder.Config(layer_config=lc, num_layers=1))
    y, _ = net(x, torch.randn(2, 64, device="cuda").to(BF))
    y.float().sum().backward()
    assert bool(torch.isfinite(net.layers[0].retention.q_norm_weight.grad).all())


def test_one_token_launch_leaves_normed_layers_to_the_layer_path():
    from flash_pop_b200.retnet import MultiScaleRetention, RetNetDecoderLayer
    from flash_pop_b200.token_stack import decoder_token
    x = torch.randn(2, 128, device="cuda").to(BF)
    with torch.no_grad():
        assert decoder_token(_model().eval().decoder, x, None, RetNetDecoderLayer, MultiScaleRetention) is None
        assert decoder_token(_model(dropout=0.3, qk_norm=False).eval().decoder, x, None, RetNetDecoderLayer, MultiScaleRetention) is not None
        assert decoder_token(_model(dropout=0.3, qk_norm=False).decoder, x, None, RetNetDecoderLayer, MultiScaleRetention) is None


def _observe(module):
    """Counts of a module's forward hooks."""
    seen = {"pre": 0, "post": 0, "back": 0}
    module.register_forward_pre_hook(lambda m, a: seen.__setitem__("pre", seen["pre"] + 1))
    module.register_forward_hook(lambda m, a, y: seen.__setitem__("post", seen["post"] + 1))
    module.register_full_backward_hook(lambda m, gi, go: seen.__setitem__("back", seen["back"] + 1))
    return seen


def test_what_is_attached_to_the_embedding_is_kept():
    m, tokens = _model(), _tokens(T=30)
    table = m.embed.weight
    step = lambda t=tokens: torch.autograd.grad(m.score(t).logprob.sum(), [table])[0]
    want, want_padded = step(), None
    padded = tokens.clone()
    padded[:, 20:] = -1
    want_padded = step(padded)
    # the padding id's row gets no gradient, and the others what they had
    m.embed.padding_idx = int(tokens[0, 3])
    got = step()
    keep = torch.arange(999, device="cuda") != m.embed.padding_idx
    assert bool((got[~keep] == 0).all()) and bool((want[~keep] != 0).any()) and torch.equal(got[keep], want[keep])
    m.embed.padding_idx = None
    # hooks see the module's call; ids outside the table stay rows of zeros (the scale apart from the lookup: gradients of rows are rounded)
    seen = _observe(m.embed)
    for ids, ref in ((tokens, want), (padded, want_padded)):
        got = step(ids)
        assert float((got.double() - ref.double()).norm() / ref.double().norm()) < 3e-2
    assert seen == {"pre": 2, "post": 2, "back": 2}
    # a module in its place is called
    m = _model()

    class Twice(torch.nn.Embedding):
        def forward(self, ids):
            return 2 * super().forward(ids)

    twice = Twice(999, 128, device="cuda", dtype=BF)
    twice.load_state_dict(m.embed.state_dict())
    m.embed_scale /= 2
    plain = m(tokens)[0]
    m.embed = twice
    m.embed_scale /= 2
    assert torch.equal(m(tokens)[0], plain)                      # (powers of two)
