"""The operators at both ends of the language model and around its layers, as cases to time.

A case is a dict of plain values.  `listed()` gives the fixed ones, `draw(rng)` more of the same ranges; `prepare` makes
what a program holds before the call, `run` makes one pass (in plain torch, or with `own` through the package's entry
points), `work` says what the pass cannot do without, and `exact` gives the result in 64 bits.

Kinds of case:
  embed    rows of the embedding table for token ids, scaled, and the table's gradient      token_ops.embedding
  dropout  dropout by a counter-based generator, alone or added to a residual               layer_ops.dropout
  qknorm   RMS norm of queries and keys over each head, then the position rotation          layer_ops.qk_norm_rotary
  score    log probabilities of given tokens, entropy, the most likely alternatives         token_ops.token_scores
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"bf16": 2, "f32": 4}
EPS = 1e-6


def listed():
    return [
        # One decoding step of a serving batch: 16 rows of the table.  Nothing but latency.
        dict(name="embed_step", kind="embed", train=False, N=16, V=32000, D=1024, dtype="bf16", padding=False),
        # The embedding of a training step, 64 sequences of 4096 tokens: the largest; the gradient is a dense table.
        dict(name="embed_train", kind="embed", train=True, N=64 * 4096, V=32000, D=1024, dtype="bf16", padding=False),
        # A small ragged fp32 batch with padding, odd vocabulary and odd width.
        dict(name="embed_ragged_f32", kind="embed", train=True, N=5003, V=8001, D=333, dtype="f32", padding=True),
        # Dropout of a branch of a decoder layer added to the residual stream, and its gradient.
        dict(name="dropout_residual", kind="dropout", train=True, B=8, T=4096, D=1024, p=0.1, residual=True, dtype="bf16"),
        # Dropout inside the feed-forward of a small fp32 model, odd sizes.
        dict(name="dropout_ragged_f32", kind="dropout", train=True, B=3, T=777, D=1365, p=0.25, residual=False, dtype="f32"),
        # Queries and keys of one training layer, with the gradients of both and of the two weights.
        dict(name="qknorm_train", kind="qknorm", train=True, B=8, T=4096, H=8, d=128, dtype="bf16", packed=True),
        # One token of a serving batch.
        dict(name="qknorm_step", kind="qknorm", train=False, B=16, T=1, H=8, d=128, dtype="bf16", packed=False),
        # Small odd heads in fp32, ragged length.
        dict(name="qknorm_ragged_f32", kind="qknorm", train=True, B=3, T=1001, H=5, d=40, dtype="f32", packed=False),
        # A decoding step: scores and 20 alternatives of 16 rows, nearly all tokens masked in some of them (constrained decoding).
        dict(name="score_step", kind="score", train=False, N=16, V=32000, top=20, dtype="bf16", masked=0.25),
        # Policy-gradient or distillation step: log probabilities and entropies of two sequences, with the logits' gradient.
        dict(name="score_train", kind="score", train=True, N=8192, V=32000, top=0, dtype="bf16", masked=0.0),
        # Scoring a corpus with the 8 best alternatives of every position.
        dict(name="score_corpus", kind="score", train=False, N=16384, V=32000, top=8, dtype="bf16", masked=0.0),
        # fp32 logits over an odd vocabulary (rows start at any 4-byte boundary), alternatives and all gradients.
        dict(name="score_ragged_f32", kind="score", train=True, N=777, V=12347, top=5, dtype="f32", masked=0.1),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], evenly spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind, train, dtype = rng.choice(["embed", "dropout", "qknorm", "score"]), rng.random() < 0.6, rng.choice(["bf16", "bf16", "f32"])
    if kind == "embed":
        V, D = _log(rng, 300, 130000), rng.choice([64, 256, 333, 512, 1000, 1024, 1536, 2048])
        while V * D * SIZES[dtype] > 3e8:
            D //= 2
        most = min(64 * 4096, int(3e8 / (D * SIZES[dtype])))
        return dict(kind=kind, train=train, N=_log(rng, 1, most), V=V, D=D, dtype=dtype, padding=rng.random() < 0.5)
    if kind == "dropout":
        B, D = rng.randint(1, 8), _log(rng, 17, 4096)
        return dict(kind=kind, train=train, B=B, T=_log(rng, 1, max(1, (1 << 25) // (B * D))), D=D, p=rng.choice([0.05, 0.1, 0.2, 0.5]),
                    residual=rng.random() < 0.5, dtype=dtype)
    if kind == "qknorm":
        B, H, d = rng.randint(1, 16), rng.choice([1, 4, 5, 8, 16]), rng.choice([16, 40, 64, 96, 128, 256])
        return dict(kind=kind, train=train, B=B, T=_log(rng, 1, max(1, (1 << 25) // (B * H * d))), H=H, d=d, dtype=dtype,
                    packed=rng.random() < 0.5)
    V = _log(rng, 500, 130000)
    return dict(kind=kind, train=train, N=_log(rng, 1, int((5e8 if train else 1e9) / (V * SIZES[dtype]))), V=V, top=rng.choice([0, 0, 1, 5, 20, 32]),
                dtype=dtype, masked=rng.choice([0.0, 0.0, 0.1]))


def _words(n, V, gen):
    """n ranks below V, rank r as likely as 1 / (r + 3)."""
    cdf = (1.0 / (torch.arange(V, dtype=torch.float64) + 3.0)).cumsum(0)
    at = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * cdf[-1].item()
    return torch.searchsorted(cdf.cuda(), at).clamp_(max=V - 1)


def prepare(case, seed):
    c, gen = case, torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[c["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).to(dtype)

    st = dict(case=c)
    if c["kind"] == "embed":
        # ids fall off as words do (a few of them are in every sentence, most are rare), in an order of their own
        order = torch.randperm(c["V"], generator=gen, device="cuda")
        tokens = order[_words(c["N"], c["V"], gen)]
        st["padding_idx"] = None
        if c["padding"]:
            st["padding_idx"] = 0
            tokens[c["N"] - c["N"] // 10:] = 0
        st.update(tokens=tokens, weight=normal(c["V"], c["D"], scale=c["D"] ** -0.5), scale=math.sqrt(c["D"]))
        if c["train"]:
            st["weight"].requires_grad_(True)
            st["dy"] = normal(c["N"], c["D"], scale=0.01)
    elif c["kind"] == "dropout":
        shape = c["B"], c["T"], c["D"]
        st.update(x=normal(*shape), residual=normal(*shape) if c["residual"] else None,
                  seed=torch.randint(0, 2 ** 62, (1,), generator=gen, device="cuda"))
        if c["train"]:
            st["x"].requires_grad_(True)
            st["dy"] = normal(*shape, scale=0.01)
    elif c["kind"] == "qknorm":
        B, T, H, d = c["B"], c["T"], c["H"], c["d"]
        if c["packed"]:                       # views into one projection's output
            st["qk"] = normal(B, T, 2, H, d)
            st["q"], st["k"] = st["qk"][:, :, 0], st["qk"][:, :, 1]
        else:
            st["q"], st["k"] = normal(B, T, H, d), normal(B, T, H, d)
        st["wq"], st["wk"] = (1 + normal(d, scale=0.1, dtype=torch.float32) for _ in range(2))
        angle = (100 + torch.arange(T, device="cuda", dtype=torch.float64))[:, None] * 10000.0 ** -torch.linspace(0, 1, d // 2, device="cuda", dtype=torch.float64)
        st["phasors"] = torch.stack((angle.cos(), angle.sin()), -1).float().unsqueeze(0).contiguous()
        if c["train"]:
            st["leaves"] = [st[n].requires_grad_(True) for n in ("q", "k", "wq", "wk")] if not c["packed"] else \
                [st[n].detach().requires_grad_(True) for n in ("q", "k", "wq", "wk")]
            st["q"], st["k"], st["wq"], st["wk"] = st["leaves"]
            st["dyq"], st["dyk"] = normal(B, T, H, d, scale=0.01), normal(B, T, H, d, scale=0.01)
    else:
        N, V = c["N"], c["V"]
        logits = normal(N, V, scale=2.5)
        tokens = _words(N, V, gen)
        logits[torch.arange(N, device="cuda"), tokens] += 8.0          # a model that has learnt something
        if c["masked"]:
            rows = torch.rand(N, generator=gen, device="cuda") < c["masked"]
            allowed = torch.rand(V, generator=gen, device="cuda") < 40.0 / V
            hide = rows[:, None] & ~allowed[None]
            hide[torch.arange(N, device="cuda"), tokens] = False
            logits.masked_fill_(hide, -math.inf)
        st.update(logits=logits, tokens=tokens)
        if c["train"]:
            logits.requires_grad_(True)
            st["g"] = [normal(N, scale=1.0 / N, dtype=torch.float32), normal(N, scale=0.01 / N, dtype=torch.float32)]
            if c["top"]:
                st["g"].append(normal(N, c["top"], scale=0.1 / N, dtype=torch.float32))
    return st


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"embed": _embed, "dropout": _dropout, "qknorm": _qknorm, "score": _score}[state["case"]["kind"]](state)


def _run_own(st):
    from flash_pop_b200 import layer_ops, token_ops
    c = st["case"]
    with torch.set_grad_enabled(c["train"]):
        if c["kind"] == "embed":
            y = token_ops.embedding(st["tokens"], st["weight"], scale=st["scale"], padding_idx=st["padding_idx"])
            return [y.detach(), *torch.autograd.grad(y, [st["weight"]], st["dy"])] if c["train"] else [y]
        if c["kind"] == "dropout":
            y = layer_ops.dropout(st["x"], c["p"], st["seed"], residual=st["residual"])
            return [y.detach(), *torch.autograd.grad(y, [st["x"]], st["dy"])] if c["train"] else [y]
        if c["kind"] == "qknorm":
            q, k = layer_ops.qk_norm_rotary(st["q"], st["k"], st["wq"], st["wk"], st["phasors"], EPS)
            return [q.detach(), k.detach(), *torch.autograd.grad((q, k), st["leaves"], (st["dyq"], st["dyk"]))] if c["train"] else [q, k]
        s = token_ops.token_scores(st["logits"], st["tokens"], top=c["top"])
        out = [s.logprob.detach(), s.entropy.detach()]
        if c["top"]:
            out += [s.top_logprob.detach(), s.top_tokens]
        if c["train"]:
            ends = [s.logprob, s.entropy] + ([s.top_logprob] if c["top"] else [])
            out += torch.autograd.grad(ends, [st["logits"]], st["g"])
        return out


# ---- plain forms: elementary operations in 32 bits, rounded once at the end -----------------------------------------

def _embed(st):
    tokens, w, dtype = st["tokens"], st["weight"], st["weight"].dtype
    y = (w[tokens].float() * st["scale"]).to(dtype)
    if not st["case"]["train"]:
        return [y]
    dy = st["dy"].float() * st["scale"]
    if st["padding_idx"] is not None:
        dy = dy * (tokens != st["padding_idx"]).unsqueeze(1)
    return [y, torch.zeros(w.shape, device=w.device).index_add_(0, tokens, dy).to(dtype)]


def _philox(group, seed):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011) of the counters
    (group, 0) under the key `seed`, each word a 64-bit integer below 2^32."""
    low = 0xFFFFFFFF
    c0, c1, c2, c3 = group & low, group >> 32, torch.zeros_like(group), torch.zeros_like(group)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57            # (the product's 64 bits, whatever sign they are read with)
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def _keep(n, p, seed):
    """Which of n elements stay, and the factor: element i has half word i % 8 of the counter i / 8, and goes where that is
    below p in 16 bits."""
    threshold = int(round(p * 65536))
    words = _philox(torch.arange((n + 7) // 8, device=seed.device), seed)
    halves = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], 1).flatten()[:n]
    return halves >= threshold, 65536.0 / (65536 - threshold) if threshold < 65536 else 0.0


def _dropout(st):
    c, x, r = st["case"], st["x"], st["residual"]
    keep, factor = _keep(x.numel(), c["p"], st["seed"])
    keep = keep.view(x.shape)
    y = torch.where(keep, x.float() * factor, 0.0)
    out = [(y if r is None else y + r.float()).to(x.dtype)]
    if c["train"]:
        out.append(torch.where(keep, st["dy"].float() * factor, 0.0).to(x.dtype))
    return out


def _rotate(x, ph, sign):
    a, b, c, s = x[..., 0::2], x[..., 1::2], ph[..., 0].unsqueeze(2), ph[..., 1].unsqueeze(2) * sign
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _norm_rotate(x, w, ph, dy):
    xf = x.float()
    n = xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
    y = _rotate(n * w, ph, 1.0).to(x.dtype)
    if dy is None:
        return y, None, None
    g = _rotate(dy.float(), ph, -1.0)
    gw = g * w
    r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
    return y, (r * (gw - n * (gw * n).mean(-1, keepdim=True))).to(x.dtype), (g * n).sum((0, 1, 2))


def _qknorm(st):
    train = st["case"]["train"]
    q, dq, dwq = _norm_rotate(st["q"], st["wq"], st["phasors"], st["dyq"] if train else None)
    k, dk, dwk = _norm_rotate(st["k"], st["wk"], st["phasors"], st["dyk"] if train else None)
    return [q, k, dq, dk, dwq, dwk] if train else [q, k]


def _score(st):
    c, logits, tokens = st["case"], st["logits"], st["tokens"]
    z = logits.float()
    m = z.max(1, keepdim=True).values
    e = (z - m).exp()
    s = e.sum(1, keepdim=True)
    logp = (z - m) - s.log()
    p = e / s
    finite = torch.where(p > 0, logp, 0.0)
    entropy = -(p * finite).sum(1)
    out = [logp.gather(1, tokens[:, None])[:, 0], entropy]
    if c["top"]:
        # unique keys: the value's order in the upper half, earlier indices first in the lower
        bits = (z + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF) - 1, bits)
        key = order * (1 << 32) + (c["V"] - torch.arange(c["V"], device=z.device))
        index = torch.topk(key, c["top"], dim=1).indices
        out += [logp.gather(1, index), index]
    if c["train"]:
        g1, g2, g3 = st["g"][0], st["g"][1], st["g"][2] if c["top"] else None
        total = g1 if g3 is None else g1 + g3.sum(1)
        d = -p * (total[:, None] + g2[:, None] * (finite + entropy[:, None]))
        d.scatter_add_(1, tokens[:, None], g1[:, None])
        if g3 is not None:
            d.scatter_add_(1, index, g3)
        out.append(d.to(logits.dtype))
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    c, e = case, SIZES[case["dtype"]]
    if c["kind"] == "embed":
        rows, n = min(c["N"], c["V"]), c["N"] * c["D"]
        moved = 8 * c["N"] + e * (rows * c["D"] + n) + (8 * c["N"] + e * (n + c["V"] * c["D"]) if c["train"] else 0)
        return {"bytes": moved, "flops": n * (2 if c["train"] else 1)}
    if c["kind"] == "dropout":
        n = c["B"] * c["T"] * c["D"]
        return {"bytes": e * n * (2 + c["residual"] + (2 if c["train"] else 0)), "flops": n * (2 if c["train"] else 1)}
    if c["kind"] == "qknorm":
        n = 2 * c["B"] * c["T"] * c["H"] * c["d"]
        return {"bytes": e * n * (5 if c["train"] else 2) + 4 * c["T"] * c["d"], "flops": n * (20 if c["train"] else 8)}
    n = c["N"] * c["V"]
    return {"bytes": e * n * (3 if c["train"] else 1) + c["N"] * (16 + 12 * c["top"]), "flops": n * (12 if c["train"] else 5)}


# ---- the same passes in 64 bits -------------------------------------------------------------------------------------

def _mask64(n, p, seed):
    """The mask on the host: the generator's rounds on unsigned 64-bit words."""
    u = np.uint64
    low, seed = u(0xFFFFFFFF), int(seed)
    x = np.zeros((4, (n + 7) // 8), dtype=u)
    x[0] = np.arange((n + 7) // 8, dtype=u)
    x[1], x[0] = x[0] >> u(32), x[0] & low
    for r in range(10):
        key = [u((seed + r * 0x9E3779B9) & 0xFFFFFFFF), u(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)]
        first, second = x[0] * u(0xD2511F53), x[2] * u(0xCD9E8D57)
        x = np.stack((x[1] ^ (second >> u(32)) ^ key[0], second & low, x[3] ^ (first >> u(32)) ^ key[1], first & low))
    halves = np.ascontiguousarray(x.T.astype("<u4")).view("<u2").reshape(-1)[:n]
    return torch.from_numpy(halves.astype(np.int32) >= round(p * 65536)).cuda(), round(p * 65536) / 65536.0


def exact(case, seed):
    c, st = case, prepare(case, seed)
    wide = lambda t: t.detach().double()
    if c["kind"] == "embed":
        y = wide(st["weight"]).index_select(0, st["tokens"]).mul_(st["scale"])
        if not c["train"]:
            return [y]
        tokens, dy = st["tokens"], st["dy"]
        if st["padding_idx"] is not None:
            used = tokens != st["padding_idx"]
            tokens, dy = tokens[used], dy[used]
        grad = torch.zeros(c["V"], c["D"], dtype=torch.float64, device="cuda")
        for part, ids in zip(dy.split(1 << 16), tokens.split(1 << 16)):
            grad.index_add_(0, ids, part.double())
        return [y, grad.mul_(st["scale"])]
    if c["kind"] == "dropout":
        n = c["B"] * c["T"] * c["D"]
        keep, p = _mask64(n, c["p"], st["seed"].item())
        keep = keep.view(c["B"], c["T"], c["D"])
        y = wide(st["x"]) / (1 - p) * keep
        out = [y if st["residual"] is None else y + wide(st["residual"])]
        return out + [wide(st["dy"]) / (1 - p) * keep] if c["train"] else out
    if c["kind"] == "qknorm":
        leaves = [wide(st[n]).requires_grad_(c["train"]) for n in ("q", "k", "wq", "wk")]
        unit = torch.view_as_complex(wide(st["phasors"])).unsqueeze(2)

        def one(x, w):
            x = w * x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
            return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2))) * unit).flatten(-2)

        ends = [one(leaves[0], leaves[2]), one(leaves[1], leaves[3])]
        if not c["train"]:
            return ends
        return [t.detach() for t in ends] + list(torch.autograd.grad(ends, leaves, (wide(st["dyq"]), wide(st["dyk"]))))
    parts = []
    step = max(1, (1 << 26) // c["V"])
    for a in range(0, c["N"], step):
        b = slice(a, a + step)
        z = wide(st["logits"][b]).requires_grad_(c["train"])
        logp = torch.log_softmax(z, 1)
        entropy = torch.special.entr(logp.exp()).sum(1) if not c["train"] else -(logp.exp() * logp.masked_fill(z == -math.inf, 0.0)).sum(1)
        got = [logp.gather(1, st["tokens"][b, None])[:, 0], entropy]
        if c["top"]:
            index = torch.sort(z.detach(), dim=1, descending=True, stable=True).indices[:, :c["top"]]
            got += [logp.gather(1, index), index]
        if c["train"]:
            ends, weights = got[:3], [wide(g[b]) for g in st["g"]]
            (grad,) = torch.autograd.grad(ends, [z], weights)
            got = [t.detach() for t in got] + [grad]
        parts.append(got)
    return [torch.cat(ts) for ts in zip(*parts)]
