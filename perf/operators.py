"""What the operators for several answers to one prompt are measured on.

Three operators of the kernel layer, each called as the engine calls it for one layer (the pages' copy: for all layers at once):

* ``copy``: pages of the cache copied inside their storage ``[layers, pages, planes, kv heads, 64, head size]``: the last,
  partly filled page of a prompt for each of its continuations; a whole sequence; pages moved to the lowest ids;
* ``shared``: a decoding step's attention (one new query a sequence) where groups of sequences hold the same pages for a
  prefix: keys ``j < len`` of sequence b, query head h on kv head h / G, scores ``scale q.k - slope_h (len - 1 - j)``, an entry
  without a value in the denominator (a stored number a head) and a gate on the result where a case has them;
* ``logprobs``: the log-probability of one token a row of float32 logits, ``x[t] - log sum exp x``.

Heads, head sizes, layers and vocabularies are those of the library's shapes.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 64
_DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---------------------------------------------------------------------------------------------- the cases
def _copy(name, layers, kv, dim, pairs, positions, planes=2, dtype="bfloat16"):
    """``positions``: filled positions of every page that is copied; 0: each page its own number."""
    return dict(name=name, kind="copy", layers=layers, kv=kv, dim=dim, pairs=pairs, positions=positions, planes=planes, dtype=dtype)


def _shared(name, groups, count, heads, kv, dim, prefix, suffix, alone=0, planes=2, extra="", dtype="bfloat16"):
    """``groups`` groups of ``count`` sequences over a prefix of ``prefix`` positions (whole pages), each with 1 to ``suffix`` positions of
    its own, and ``alone`` sequences that share nothing."""
    return dict(name=name, kind="shared", groups=groups, count=count, heads=heads, kv=kv, dim=dim, prefix=prefix, suffix=suffix, alone=alone,
                planes=planes, extra=extra, dtype=dtype)


def _logprobs(name, rows, vocab):
    return dict(name=name, kind="logprobs", rows=rows, vocab=vocab)


def listed():
    return [
        # one continuation of a short prompt on the smallest model writes into the page it shares: launch latency
        _copy("fork-0.5b", 24, 2, 64, 1, 21),
        # eight continuations of a prompt on the 7B shape: seven copies of its last page
        _copy("fork-7b", 28, 4, 128, 7, 37),
        # a sequence of 4,200 positions copied outright on the 32-bit path, its last page partly filled
        _copy("sequence-0.5b", 24, 2, 64, 66, 0, dtype="float32"),
        # a cache of half-empty storage compacted: full pages move
        _copy("compact-1.5b", 28, 2, 128, 333, 64),
        # two answers to one short question
        _shared("pair-0.5b", 1, 2, 14, 2, 64, 320, 40),
        # the benchmark's decode as eight answers to one prompt
        _shared("answers-7b", 1, 8, 28, 4, 128, 2048, 100),
        # many samples of one long document, full batch
        _shared("samples-7b", 1, 64, 28, 4, 128, 16384, 500),
        # several prompts with a few answers each, and requests that share nothing
        _shared("requests-1.5b", 4, 6, 12, 2, 128, 4032, 333, alone=3, extra="sink gate"),
        # four answers on the 32-bit path
        _shared("float32-0.5b", 1, 4, 14, 2, 64, 960, 130, dtype="float32"),
        # the score of one token of a step; of a batch's step; of a whole prompt's tokens
        _logprobs("step-0.5b", 1, 151936),
        _logprobs("batch-7b", 61, 152064),
        _logprobs("prompt-7b", 2000, 152064),
    ]


_SHAPES = [(24, 14, 2, 64), (28, 12, 2, 128), (36, 16, 2, 128), (28, 28, 4, 128), (48, 40, 8, 128)]     # layers, heads, kv heads, head size


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most and _plain_values(c) <= 5.6e8:
            return c


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def _plain_values(c):
    return (c["groups"] * c["count"] + c["alone"]) * (c["prefix"] + c["suffix"]) * c["kv"] * c["dim"] if c["kind"] == "shared" else 0


def _draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["copy", "shared", "shared", "logprobs"])
    layers, heads, kv, dim = rng.choice(_SHAPES)
    dtype = rng.choice(["bfloat16"] * 5 + ["float32"])
    if kind == "copy":
        return _drawn(_copy("", layers, kv, dim, log(1, 333), rng.choice([0, PAGE, rng.randint(1, PAGE)]), rng.choice([2, 2, 1]), dtype))
    if kind == "logprobs":
        return _drawn(_logprobs("", log(1, 2000), rng.choice([512, 1000, log(2000, 40000), 151936, 152064])))
    groups = rng.choice([1, 1, 2, log(2, 9)])
    planes = rng.choice([2, 2, 2, 1])
    if planes == 1:                                        # a latent that all heads read
        kv = 1
    if dtype == "float32":
        heads, kv, dim = 14, 2 if planes == 2 else 1, 64
    extra = rng.choice(["", "", "sink gate", "slopes"])
    return _drawn(_shared("", groups, log(2, 64), heads, kv, dim, PAGE * log(1, 256), log(1, 1500), rng.choice([0, 0, rng.randint(1, 9)]), planes, extra, dtype))


def _drawn(c):
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    return {"copy": _prepare_copy, "shared": _prepare_shared, "logprobs": _prepare_logprobs}[case["kind"]](case, seed)


def _prepare_copy(c, seed):
    gen, host = _generator(seed), torch.Generator().manual_seed(seed)
    n = c["pairs"]
    pages = 2 * n + 3
    storage = torch.randn(c["layers"], pages, c["planes"], c["kv"], PAGE, c["dim"], generator=gen, device="cuda", dtype=_DTYPES[c["dtype"]])
    order = torch.randperm(pages, generator=host)
    # one source for all where a prompt's last page goes to its continuations, else a page each; no page is both source and destination
    src = order[:n] if c["positions"] in (0, PAGE) else order[:1].expand(n)
    fill = torch.full((n,), c["positions"] or PAGE)
    if c["positions"] == 0:
        fill[-1] = int(torch.randint(1, PAGE + 1, (1,), generator=host))
    plan = torch.stack([src, order[n:2 * n], fill], 1).to(torch.int32)        # on the host, where the cache's bookkeeping is
    return {"case": c, "storage": storage, "plan": plan}


def _prepare_shared(c, seed):
    gen, host = _generator(seed), torch.Generator().manual_seed(seed)
    groups, count, dim, kv, heads, dtype = c["groups"], c["count"], c["dim"], c["kv"], c["heads"], _DTYPES[c["dtype"]]
    B, shared = groups * count + c["alone"], c["prefix"] // PAGE
    lens = c["prefix"] + torch.randint(1, c["suffix"] + 1, (B,), generator=host)
    width = -(-(c["prefix"] + c["suffix"]) // PAGE)
    own_pages = torch.full((B,), width - shared)
    own_pages[groups * count:] = width
    pages = groups * shared + int(own_pages.sum()) + 2
    ids = torch.randperm(pages, generator=host)
    table = torch.zeros(B, width, dtype=torch.int64)
    at = groups * shared
    table[:groups * count, :shared] = ids[:at].view(groups, 1, shared).expand(groups, count, shared).reshape(-1, shared)
    tail = groups * count * (width - shared)
    table[:groups * count, shared:] = ids[at:at + tail].view(-1, width - shared)
    if c["alone"]:
        table[groups * count:] = ids[at + tail:at + tail + c["alone"] * width].view(-1, width)
    storage = torch.randn(pages, c["planes"], kv, PAGE, dim, generator=gen, device="cuda", dtype=dtype)
    gate = "gate" in c["extra"]
    qkv = torch.randn(B, (heads * (2 if gate else 1) + 2 * kv) * dim, generator=gen, device="cuda", dtype=dtype)
    order = torch.arange(B)
    mine = torch.zeros(B, dtype=torch.int64)
    mine[:groups * count] = shared
    plan = torch.tensor([[g * count, count, shared] for g in range(groups)], dtype=torch.int32).view(-1, 3)
    dev = lambda t: t.to("cuda", torch.int32)                 # noqa: E731
    return {"case": c, "storage": storage, "qkv": qkv, "table": dev(table), "slot": dev(order), "len": dev(lens), "order": dev(order),
            "own_page": dev(mine), "groups": plan.cuda(), "max_len": int(lens.max()), "scale": dim ** -0.5,
            "sink": torch.randn(heads, generator=gen, device="cuda") if "sink" in c["extra"] else None,
            "slopes": 2.0 ** (-8.0 * (torch.arange(heads, device="cuda") + 1.0) / heads) if "slopes" in c["extra"] else None,
            "gate": (heads + 2 * kv) * dim if gate else 0, "out": torch.empty(B, heads * dim, device="cuda", dtype=dtype)}


def _prepare_logprobs(c, seed):
    gen = _generator(seed)
    logits = torch.randn(c["rows"], c["vocab"], generator=gen, device="cuda").mul_(2.5)
    drawn = torch.randint(0, c["vocab"], (c["rows"],), generator=gen, device="cuda")
    likely = torch.rand(c["rows"], generator=gen, device="cuda") < 0.7         # most tokens of a sequence are among the likely ones
    logits[torch.arange(c["rows"], device="cuda"), drawn] += likely * 12.0
    return {"case": c, "logits": logits, "tokens": drawn.to(torch.int32), "out": torch.empty(c["rows"], device="cuda")}


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"copy": _own_copy, "shared": _own_shared, "logprobs": _own_logprobs}[kind](state)
    return {"copy": _plain_copy, "shared": _plain_shared, "logprobs": _plain_logprobs}[kind](state)


def _plain_copy(s):
    plan = s["plan"].to("cuda", torch.int64)
    storage, src, dst = s["storage"], plan[:, 0], plan[:, 1]
    filled = (torch.arange(PAGE, device="cuda") < plan[:, 2, None]).view(1, -1, 1, 1, PAGE, 1)
    storage[:, dst] = torch.where(filled, storage[:, src], storage[:, dst])
    return storage


def _plain_shared(s):
    c, storage = s["case"], s["storage"]
    B, kv, dim, heads = s["qkv"].shape[0], c["kv"], c["dim"], c["heads"]
    pages = s["table"][s["slot"].long()].long()                                        # [B, width]
    span = pages.shape[1] * PAGE
    held = storage[pages]                                                              # [B, width, planes, kv, PAGE, dim]
    k = held[:, :, 0].transpose(1, 2).reshape(B, kv, span, dim).float()
    v = held[:, :, -1].transpose(1, 2).reshape(B, kv, span, dim).float()
    q = s["qkv"][:, :heads * dim].float().view(B, kv, heads // kv, dim)
    scores = (q @ k.transpose(2, 3) * s["scale"]).view(B, heads, span)
    back = (s["len"].view(-1, 1, 1) - 1 - torch.arange(span, device="cuda")).float()
    if s["slopes"] is not None:
        scores = scores - s["slopes"].view(1, -1, 1) * back
    scores = torch.where(back >= 0, scores, -math.inf)
    top = scores.amax(2, keepdim=True)
    p = torch.exp(scores - top)
    total = p.sum(2, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"].view(1, -1, 1) - top)
    out = (p.view(B, kv, heads // kv, span) @ v).view(B, heads, dim) / total
    if s["gate"]:
        out = out / (1 + torch.exp(-s["qkv"][:, s["gate"]:s["gate"] + heads * dim].float().view(B, heads, dim)))
    s["out"].copy_(out.view(B, heads * dim))
    return s["out"]


def _plain_logprobs(s):
    x = s["logits"]
    top = x.amax(1, keepdim=True)
    s["out"].copy_((x.gather(1, s["tokens"].long()[:, None]) - top - torch.log(torch.exp(x - top).sum(1, keepdim=True)))[:, 0])
    return s["out"]


_loaded = []


def _kernels():
    if not _loaded:
        from cima_b200.kernels import Kernels
        _loaded.append(Kernels(verbose=False))
    return _loaded[0]


def _own_copy(s):
    _kernels().copy_pages(s["storage"], s["plan"])
    return s["storage"]


def _own_shared(s):
    from cima_b200.cache.kv import LayerKV, SharedPrefixes
    c = s["case"]
    kv = LayerKV(s["storage"], s["table"], PAGE, 0, 0, 0, c["planes"])
    shared = SharedPrefixes(s["order"], s["own_page"], s["groups"], c["count"])
    _kernels().attention_shared(s["qkv"], kv, s["slot"], s["len"], shared, s["out"], c["heads"], c["kv"], c["dim"], s["scale"], s["max_len"],
                                head_sink=s["sink"], gate_col=s["gate"], slopes=s["slopes"])
    return s["out"]


def _own_logprobs(s):
    _kernels().token_logprobs(s["logits"], s["tokens"], s["out"])
    return s["out"]


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def _element(c):
    return 4 if c["dtype"] == "float32" else 2


def work(case):
    c = case
    if c["kind"] == "copy":
        positions = c["pairs"] * (c["positions"] or PAGE)
        read = positions if c["positions"] in (0, PAGE) else c["positions"]           # one page's filled positions serve every copy of it
        return {"bytes": (positions + read) * c["layers"] * c["planes"] * c["kv"] * c["dim"] * _element(c), "flops": 0}
    if c["kind"] == "logprobs":
        return {"bytes": c["rows"] * (c["vocab"] * 4 + 8), "flops": 3.0 * c["rows"] * c["vocab"]}
    B, suffix = c["groups"] * c["count"] + c["alone"], (c["suffix"] + 1) / 2
    keys = c["groups"] * c["prefix"] + B * suffix + c["alone"] * c["prefix"]
    rows = (3 if "gate" in c["extra"] else 2) * B * c["heads"] * c["dim"]
    return {"bytes": (keys * c["planes"] * c["kv"] * c["dim"] + rows) * _element(c),
            "flops": 4.0 * B * (c["prefix"] + suffix) * c["heads"] * c["dim"]}


# ---------------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    if case["kind"] == "copy":
        return None                                           # bits are moved, nothing is computed
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        rows = []
        for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
            rows.append(torch.log_softmax(x.double(), 1)[torch.arange(len(t), device="cuda"), t.long()])
        return torch.cat(rows)
    c, heads, kv, dim = case, case["heads"], case["kv"], case["dim"]
    out = []
    for b, n in enumerate(s["len"].tolist()):
        pages = s["table"][int(s["slot"][b]), :-(-n // PAGE)].long()
        held = s["storage"][pages].double()                   # [pages, planes, kv, PAGE, dim]
        k, v = (held[:, i].permute(1, 0, 2, 3).flatten(1, 2)[:, :n] for i in (0, c["planes"] - 1))
        q = s["qkv"][b, :heads * dim].double().view(kv, -1, dim)
        x = torch.einsum("kgd,knd->kgn", q, k).flatten(0, 1) * s["scale"]
        if s["slopes"] is not None:
            x = x - s["slopes"].double()[:, None] * torch.arange(n - 1, -1, -1, device="cuda")
        if s["sink"] is not None:
            x = torch.cat([x, s["sink"].double()[:, None]], 1)
        w = torch.softmax(x, 1)[:, :n].view(kv, -1, n)
        o = torch.einsum("kgn,knd->kgd", w, v).reshape(-1)
        if s["gate"]:
            o = o * torch.sigmoid(s["qkv"][b, s["gate"]:s["gate"] + heads * dim].double())
        out.append(o)
    return torch.stack(out)
