"""The layers at the entry of a transformer, as cases that can be timed and compared: what a user trains or serves them with.

A case is a dict of plain values.  `op` names the call:

  embedding       rows of a table by token id, scaled
  embedding_grad  the table's gradient from the gradient of the looked-up rows
  dropout         dropout from a counter-based generator (the backward is the same call on the gradient)
  rms_norm        residual addition (its branch optionally dropped) and root-mean-square norm, in 32, 16 or 8 bits
  rms_norm_grad   gradients of the norm's input, of the residual and of the weight

Where `own` is false the operators run in elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False  # set by whoever measures: False for the plain forms, True for the framework's kernels

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
FP8_MAX = 448.0


def _case(op, **given):
    """Every case says all choices of its operator."""
    choices = {"embedding": dict(tokens=1, vocab=1, dim=1, scale=1.0, dtype="bf16"),
               "embedding_grad": dict(tokens=1, vocab=1, dim=1, scale=1.0, dtype="bf16", out="bf16", padded=0.0, accumulate=False),
               "dropout": dict(rows=1, cols=1, p=0.1, dtype="bf16"),
               "rms_norm": dict(rows=1, cols=1, dtype="bf16", stream="bf16", out="bf16", residual=True, p=0.0, group=0),
               "rms_norm_grad": dict(rows=1, cols=1, dtype="bf16", stream="bf16", residual=True, p=0.0)}[op]
    return dict(choices, op=op, **given)


def listed():
    return [
        # one prompt of a text encoder: latency counts
        _case("embedding", name="lookup_prompt", tokens=77, vocab=49408, dim=768),
        # a training batch, rows scaled as they are looked up
        _case("embedding", name="lookup_batch", tokens=16384, vocab=32000, dim=4096, scale=64.0),
        # fine-tuning a text encoder on prompts: mostly untouched rows, gradients kept in 32 bits for the optimizer
        _case("embedding_grad", name="table_grad_prompts", tokens=616, vocab=49408, dim=768, out="f32", padded=0.5),
        # a further micro-batch onto the gradient that is there, odd sizes
        _case("embedding_grad", name="table_grad_accumulate", tokens=4095, vocab=10007, dim=1155, out="f32", padded=0.1, accumulate=True),
        # a large language model's table from a large batch
        _case("embedding_grad", name="table_grad_batch", tokens=32768, vocab=128000, dim=4096, scale=64.0),
        # an adapter's input
        _case("dropout", name="dropout_adapter", rows=1024, cols=1280, p=0.05),
        # the hidden layer of a wide feed-forward block
        _case("dropout", name="dropout_hidden", rows=16384, cols=8192, p=0.1),
        # one new token: latency counts
        _case("rms_norm", name="norm_one_token", rows=1, cols=4096),
        # a training batch with dropout of the branch that is added
        _case("rms_norm", name="norm_batch_dropout", rows=16384, cols=4096, p=0.1),
        # 8-bit activations for the products behind the norm, a scale for each 128 columns
        _case("rms_norm", name="norm_fp8_groups", rows=8192, cols=5120, out="fp8", group=128),
        # an odd width in 32 bits, as a small head has it
        _case("rms_norm_grad", name="norm_grad_odd_f32", rows=1025, cols=1281, dtype="f32", stream="f32"),
        # the backward pass of the training batch
        _case("rms_norm_grad", name="norm_grad_batch", rows=16384, cols=4096, p=0.1),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 1 if n == 3072 else n


def _width(rng, lo, hi):
    """A row's length: of the usual multiples, or any."""
    n = _log_int(rng, lo, hi)
    to = rng.choice([1, 8, 64, 128, 256])
    n = max(to, n // to * to)
    return n + to if n == 3072 else n


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["embedding", "embedding_grad", "embedding_grad", "dropout", "rms_norm", "rms_norm", "rms_norm_grad", "rms_norm_grad"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("embedding", "embedding_grad"):
        dim, vocab = _width(rng, 64, 4096), _log_int(rng, 500, 128000)
        tokens = min(_log_int(rng, 1, 32768), max(1, (1 << 27) // dim))
        scale = rng.choice([1.0, 1.0, float(round(math.sqrt(dim), 3))])
        if op == "embedding":
            return _case(op, tokens=tokens, vocab=vocab, dim=dim, scale=scale, dtype=dtype)
        out = rng.choice(["f32", dtype])
        while vocab * dim * (4 if out == "f32" else 2) > 1 << 30:
            vocab //= 2
        return _case(op, tokens=tokens, vocab=vocab, dim=dim, scale=scale, dtype=dtype, out=out,
                     padded=rng.choice([0.0, round(rng.uniform(0.01, 0.6), 2)]), accumulate=rng.random() < 0.3)
    cols = _width(rng, 64, 16384)
    rows = min(_log_int(rng, 1, 65536), (1 << (26 if dtype == "bf16" else 25)) // cols)
    p = rng.choice([0.0, round(rng.uniform(0.01, 0.5), 3)])
    if op == "dropout":
        return _case(op, rows=rows, cols=cols, p=max(p, 0.01), dtype=dtype)
    stream = rng.choice([dtype, "f32"])
    residual = rng.random() < 0.7
    if not residual:
        p, stream = 0.0, dtype
    if op == "rms_norm_grad":
        return _case(op, rows=rows, cols=cols, dtype=dtype, stream=stream, residual=residual, p=p)
    out = rng.choice(["bf16", dtype, "fp8"])
    return _case(op, rows=rows, cols=cols, dtype=dtype, stream=stream, out=out, residual=residual, p=p,
                 group=rng.choice([0, 128]) if out == "fp8" else 0)


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------

EPS = 1e-6
PAD = 0


def _tokens(case, g):
    """Token ids as text has them, a few of them very often: id k with probability log((k+2)/(k+1)) / log(vocab+1)."""
    u = torch.rand(case["tokens"], generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(case["vocab"] + 1)) - 1).long().clamp_(0, case["vocab"] - 1)
    if case.get("padded"):  # the ends of the sequences
        at = torch.arange(case["tokens"], device="cuda") % 256
        ids = torch.where(at >= 256 * (1 - case["padded"]), PAD, ids)
    return ids


def _padding(case):
    """The id that gets no gradient."""
    return PAD if case["padded"] else None


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype="bf16", std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(DTYPES[dtype])

    s = dict(case=case, seed=seed * 0x9E3779B9 + 12345, offset=seed % 1000)
    if case["op"] == "embedding":
        s.update(ids=_tokens(case, g), weight=normal(case["vocab"], case["dim"], dtype=case["dtype"], std=0.02))
    elif case["op"] == "embedding_grad":
        s.update(ids=_tokens(case, g), grad=normal(case["tokens"], case["dim"], dtype=case["dtype"], std=1e-3))
        s["out"] = normal(case["vocab"], case["dim"], dtype=case["out"], std=1e-3) if case["accumulate"] else None
    elif case["op"] == "dropout":
        s["x"] = normal(case["rows"], case["cols"], dtype=case["dtype"])
    else:
        shape = (case["rows"], case["cols"])
        s["weight"] = normal(case["cols"], dtype=case["dtype"], std=0.1, mean=1.0)
        if case["op"] == "rms_norm":
            s["x"] = normal(*shape, dtype=case["dtype"])
            s["residual"] = normal(*shape, dtype=case["stream"], std=2.0) if case["residual"] else None
        else:  # what the forward pass left, and the gradients that arrive
            s["h"] = normal(*shape, dtype=case["stream"], std=2.0)
            s["rstd"] = torch.rsqrt(s["h"].float().square().mean(1) + EPS)
            s["grad"] = normal(*shape, dtype=case["dtype"], std=1e-3)
            s["grad_h"] = normal(*shape, dtype=case["stream"], std=1e-3) if case["residual"] else None
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------

WORD = 0xFFFFFFFF


def _philox(group, seed, offset):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011), 32-bit words in int64."""
    c0, c1 = group & WORD, group >> 32
    c2, c3 = torch.full_like(group, offset & WORD), torch.full_like(group, offset >> 32)
    k0, k1 = seed & WORD, (seed >> 32) & WORD
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & WORD) ^ c1 ^ k0, b & WORD, ((a >> 32) & WORD) ^ c3 ^ k1, a & WORD
        k0, k1 = (k0 + 0x9E3779B9) & WORD, (k1 + 0xBB67AE85) & WORD
    return torch.stack((c0, c1, c2, c3), 1)


def _drop(x, p, seed, offset):
    """x in 32 bits, dropped: element i is kept where its 16 random bits are not below the threshold."""
    if p == 0:
        return x
    below = int(p * 65536 + 0.5)
    n = x.numel()
    words = _philox(torch.arange(-(-n // 8), device=x.device), seed, offset)
    bits = torch.stack((words & 0xFFFF, words >> 16), 2).view(-1)[:n].view(x.shape)
    return torch.where(bits >= below, x * (65536 / (65536 - below)), 0.0)


def _plain_embedding(s, case):
    return {"rows": (s["weight"][s["ids"]].float() * case["scale"]).to(DTYPES[case["dtype"]])}


def _plain_embedding_grad(s, case):
    ids, pad = s["ids"], _padding(case)
    rows = s["grad"].float()
    if pad is not None:
        rows = torch.where((ids == pad)[:, None], 0.0, rows)
    total = torch.zeros(case["vocab"], case["dim"], device="cuda").index_add_(0, ids, rows).mul_(case["scale"])
    if case["accumulate"]:
        return {"table": s["out"].copy_(total.add_(s["out"].float()))}
    return {"table": total.to(DTYPES[case["out"]])}


def _plain_dropout(s, case):
    return {"y": _drop(s["x"].float(), case["p"], s["seed"], s["offset"]).to(s["x"].dtype)}


def _plain_rms_norm(s, case):
    h = _drop(s["x"].float(), case["p"], s["seed"], s["offset"])
    if case["residual"]:
        h = h + s["residual"].float()
    rstd = torch.rsqrt(h.square().mean(1) + EPS)
    y = h * rstd[:, None] * s["weight"].float()
    out = {"rstd": rstd}
    if case["residual"]:
        out["h"] = h.to(DTYPES[case["stream"]])
    if case["out"] != "fp8":
        return dict(out, y=y.to(DTYPES[case["out"]]))
    wide = case["group"] or case["cols"]
    groups = -(-case["cols"] // wide)
    y = torch.nn.functional.pad(y, (0, groups * wide - case["cols"])).view(case["rows"], groups, wide)
    most = y.abs().amax(2, keepdim=True)
    codes = (y * torch.where(most > 0, FP8_MAX / most, 1.0)).to(torch.float8_e4m3fn)
    out["scales"] = torch.where(most > 0, most / FP8_MAX, 1.0).squeeze(2)
    return dict(out, y=codes.view(case["rows"], -1)[:, : case["cols"]].contiguous())


def _plain_rms_norm_grad(s, case):
    h, dy, rstd = s["h"].float(), s["grad"].float(), s["rstd"][:, None]
    dyw = dy * s["weight"].float()
    dh = dyw * rstd - h * (rstd.pow(3) * (dyw * h).sum(1, keepdim=True) / case["cols"])
    if case["residual"]:
        dh = dh + s["grad_h"].float()
    out = {"weight": (dy * h * rstd).sum(0).to(s["weight"].dtype), "x": _drop(dh, case["p"], s["seed"], s["offset"]).to(DTYPES[case["dtype"]])}
    return dict(out, residual=dh.to(DTYPES[case["stream"]])) if case["residual"] else out


PLAIN = {"embedding": _plain_embedding, "embedding_grad": _plain_embedding_grad, "dropout": _plain_dropout,
         "rms_norm": _plain_rms_norm, "rms_norm_grad": _plain_rms_norm_grad}


# ---------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------

def _own_embedding(layers, s, case):
    return {"rows": layers.embedding(s["ids"], s["weight"], case["scale"])}


def _own_embedding_grad(layers, s, case):
    return {"table": layers.embedding_grad(s["ids"], s["grad"], case["vocab"], case["scale"], padding_id=_padding(case),
                                           dtype=DTYPES[case["out"]], out=s["out"], accumulate=case["accumulate"])}


def _own_dropout(layers, s, case):
    return {"y": layers.dropout(s["x"], case["p"], s["seed"], s["offset"])}


def _own_rms_norm(layers, s, case):
    r = layers.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], p=case["p"], seed=s["seed"], offset=s["offset"],
                        dtype=DTYPES[case["out"]], scale_group=case["group"])
    out = {"y": r.y, "rstd": r.rstd}
    if case["residual"]:
        out["h"] = r.h
    return dict(out, scales=r.scales) if case["out"] == "fp8" else out


def _own_rms_norm_grad(layers, s, case):
    r = layers.rms_norm_grad(s["grad"], s["h"], s["rstd"], s["weight"], grad_h=s["grad_h"], p=case["p"], seed=s["seed"], offset=s["offset"],
                             dtype=DTYPES[case["dtype"]])
    out = {"weight": r.weight, "x": r.x}
    return dict(out, residual=r.residual) if case["residual"] else out


OWN = {"embedding": _own_embedding, "embedding_grad": _own_embedding_grad, "dropout": _own_dropout,
       "rms_norm": _own_rms_norm, "rms_norm_grad": _own_rms_norm_grad}


def run(state):
    case = state["case"]
    if own:
        from eridiffusion_amd import layers
        return OWN[case["op"]](layers, state, case)
    return PLAIN[case["op"]](state, case)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def _touched(case):
    """Rows of the table that the tokens are expected to name."""
    k = torch.arange(case["vocab"], dtype=torch.float64)
    chance = torch.log((k + 2) / (k + 1)) / math.log(case["vocab"] + 1)
    real = case["tokens"] * (1 - case.get("padded", 0.0))
    return max(1.0, float((1 - torch.exp(real * torch.log1p(-chance.clamp(max=1 - 1e-12)))).sum()))


def work(case):
    size = {"bf16": 2, "f32": 4, "fp8": 1}
    e = size[case["dtype"]]
    if case["op"] == "embedding":
        return {"bytes": case["tokens"] * (8 + case["dim"] * e) + _touched(case) * case["dim"] * e, "flops": case["tokens"] * case["dim"]}
    if case["op"] == "embedding_grad":
        real = case["tokens"] * (1 - case["padded"])
        rows = 2 * _touched(case) if case["accumulate"] else case["vocab"]
        return {"bytes": case["tokens"] * 8 + real * case["dim"] * e + rows * case["dim"] * size[case["out"]], "flops": real * case["dim"]}
    n = case["rows"] * case["cols"]
    if case["op"] == "dropout":
        return {"bytes": 2 * n * e, "flops": n}
    r = 2 * size[case["stream"]] if case["residual"] else 0
    if case["op"] == "rms_norm":
        groups = 0 if case["out"] != "fp8" else -(-case["cols"] // case["group"]) if case["group"] else 1
        return {"bytes": n * (e + r + size[case["out"]]) + case["rows"] * (4 + 4 * groups) + case["cols"] * e, "flops": 5 * n}
    return {"bytes": n * (2 * e + size[case["stream"]] + r) + case["rows"] * 4 + 2 * case["cols"] * e, "flops": 9 * n}


def _kept(n, p, seed, offset):
    """Which of n elements stay, by the generator's definition on 16-bit limbs."""
    def both(a, m):  # high and low word of the product of two 32-bit words
        p00, p01, p10, p11 = (a & 0xFFFF) * (m & 0xFFFF), (a & 0xFFFF) * (m >> 16), (a >> 16) * (m & 0xFFFF), (a >> 16) * (m >> 16)
        mid = (p00 >> 16) + (p01 & 0xFFFF) + (p10 & 0xFFFF)
        return p11 + (p01 >> 16) + (p10 >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (p00 & 0xFFFF)

    i = torch.arange(-(-n // 8), device="cuda")
    ctr = [i % 2**32, i // 2**32, torch.full_like(i, offset % 2**32), torch.full_like(i, offset // 2**32)]
    key = [seed % 2**32, seed // 2**32 % 2**32]
    for r in range(10):
        h0, l0 = both(ctr[0], 0xD2511F53)
        h1, l1 = both(ctr[2], 0xCD9E8D57)
        ctr = [h1 ^ ctr[1] ^ ((key[0] + r * 0x9E3779B9) % 2**32), l1, h0 ^ ctr[3] ^ ((key[1] + r * 0xBB67AE85) % 2**32), l0]
    keep = torch.empty(i.numel(), 8, dtype=torch.bool, device="cuda")
    for e in range(8):
        keep[:, e] = (ctr[e // 2] // 2 ** (16 * (e % 2))) % 65536 >= math.floor(p * 65536 + 0.5)
    return keep.reshape(-1)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    f = lambda name: s[name].double()  # noqa: E731
    if case["op"] == "embedding":
        return {"rows": f("weight").index_select(0, s["ids"]) * case["scale"]}
    if case["op"] == "embedding_grad":
        order = torch.argsort(s["ids"], stable=True)
        sums = torch.cat((torch.zeros(1, case["dim"], dtype=torch.float64, device="cuda"), f("grad")[order].cumsum(0)))
        ends = torch.searchsorted(s["ids"][order], torch.arange(case["vocab"] + 1, device="cuda"))
        table = (sums[ends[1:]] - sums[ends[:-1]]) * case["scale"]
        if _padding(case) is not None:
            table[_padding(case)] = 0
        return {"table": table + f("out") if case["accumulate"] else table}
    shape, p = (case["rows"], case["cols"]), case["p"]
    drop = lambda x: x if p == 0 else x * _kept(x.numel(), p, s["seed"], s["offset"]).view(shape) / (1 - math.floor(p * 65536 + 0.5) / 65536)  # noqa: E731
    if case["op"] == "dropout":
        return {"y": drop(f("x"))}
    w = f("weight")
    if case["op"] == "rms_norm":
        h = drop(f("x")) + (f("residual") if case["residual"] else 0)
        rstd = 1 / torch.sqrt((h * h).sum(1) / case["cols"] + EPS)
        y = torch.einsum("rc,r,c->rc", h, rstd, w)
        out = {"rstd": rstd, "h": h} if case["residual"] else {"rstd": rstd}
        if case["out"] != "fp8":
            return dict(out, y=y)
        parts = y.split(case["group"] or case["cols"], 1)
        out["scales"] = torch.stack([q.abs().max(1).values / FP8_MAX for q in parts], 1)
        return dict(out, y=torch.cat([q / out["scales"][:, k : k + 1] for k, q in enumerate(parts)], 1))
    rstd = f("rstd")[:, None]
    n = f("h") * rstd  # the normed rows; d(n_j)/d(h_k) = rstd * (1[j=k] - n_j n_k / cols)
    a = f("grad") * w
    dh = rstd * (a - n * (a * n).mean(1, keepdim=True)) + (f("grad_h") if case["residual"] else 0)
    out = {"weight": (f("grad") * n).sum(0), "x": drop(dh)}
    return dict(out, residual=dh) if case["residual"] else out
