"""Inputs and 64-bit references of the operators for several answers to one prompt: attention over shared prefixes, copies of
pages, log-probabilities of tokens."""
import math
from types import SimpleNamespace

import torch

PAGE = 64
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}       # half a step of rounding, relative to the value


def shared_case(counts, prefix_pages, own, heads, kv, hd, dtype, *, planes=2, alone=(), gate=False, seed=0, device="cuda", spare=7, slots=None):
    """Groups of ``counts[i]`` sequences over ``prefix_pages[i]`` pages, each sequence with one of the positions in ``own`` (in turn) of its own, and
    sequences that share nothing of ``alone`` positions; in the batch the sequences stand in a shuffled order, and so do the pages in their
    storage.  Positions behind a sequence's end hold NaN, infinities and large numbers."""
    gen = torch.Generator().manual_seed(seed)
    seqs = []                                          # (group or -1, prefix pages, length)
    k = 0
    for g, (n, p) in enumerate(zip(counts, prefix_pages)):
        for _ in range(n):
            seqs.append((g, p, p * PAGE + own[k % len(own)]))
            k += 1
    seqs += [(-1, 0, n) for n in alone]
    B = len(seqs)
    place = torch.randperm(B, generator=gen).tolist()  # batch index of seqs[i]
    total = sum(prefix_pages) + sum(-(-n // PAGE) - p for _, p, n in seqs) + spare
    ids = torch.randperm(total, generator=gen).tolist()
    take = iter(ids)
    prefix_ids = [[next(take) for _ in range(p)] for p in prefix_pages]
    width = max(-(-n // PAGE) for *_, n in seqs) + 2
    slots = slots or B + 3
    slot_of = torch.randperm(slots, generator=gen)[:B].tolist()
    table = torch.full((slots, width), -1, dtype=torch.int32)
    storage = torch.randn(total, planes, kv, PAGE, hd, generator=gen).to(dtype)
    lens = [0] * B
    own_page = [0] * B
    slot = [0] * B
    for i, (g, p, n) in enumerate(seqs):
        b = place[i]
        pages = (prefix_ids[g] if g >= 0 else []) + [next(take) for _ in range(-(-n // PAGE) - p)]
        table[slot_of[i], :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        lens[b], own_page[b], slot[b] = n, p, slot_of[i]
        tail = n % PAGE
        if tail:
            junk = storage[pages[-1], :, :, tail:]
            junk[..., 0::3] = math.nan
            junk[..., 1::3] = math.inf
            junk[..., 2::3] = -3e38
    groups, at = [], 0
    for n, p in zip(counts, prefix_pages):
        groups.append([at, n, p])
        at += n
    cols = (heads * (2 if gate else 1) + 2 * kv) * hd
    qkv = torch.randn(B, cols, generator=gen).to(dtype)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)       # noqa: E731
    return SimpleNamespace(B=B, heads=heads, kv_heads=kv, hd=hd, planes=planes, dtype=dtype, storage=storage.to(device), table=table.to(device), qkv=qkv.to(device),
                           slot=i32(slot), len=i32(lens), order=i32(place), own_page=i32(own_page), groups=i32(groups or []).view(-1, 3), most=max(counts, default=0),
                           max_len=max(lens), scale=hd ** -0.5, gate_col=(heads + 2 * kv) * hd if gate else 0, lens=lens,
                           sink=torch.randn(heads, generator=gen).to(device), slopes=(2.0 ** (-8.0 * (torch.arange(heads) + 1.0) / heads)).to(device))


def shared_reference(c, *, head_sink=None, sink=0.0, slopes=None, gate_col=0):
    """(result, bound on a kernel's error), float64 [B, heads * hd].  The bound counts: the result's own rounding; for bfloat16 the rounding of
    each probability as an operand (half a step of its type relative to it, whatever its value's sign); the float32 score, whose error e
    (a sum of hd products, scaling and bias: hd + 8 roundings of the sum of their sizes) moves a probability by its e-fold; and the roundings of
    the float32 sums over n keys.  All relative to the sum of w |v|.  A gate's sigmoid (at most 1) takes another 8 float32 roundings."""
    nh, nkv, hd = c.heads, c.kv_heads, c.hd
    G = nh // nkv
    out, tol = [], []
    storage, qkv, table = c.storage.cpu(), c.qkv.cpu().double(), c.table.cpu()
    for b, n in enumerate(c.lens):
        pages = table[int(c.slot[b]), :-(-n // PAGE)].long()
        held = storage[pages].double()
        k, v = (held[:, i].permute(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :n].repeat_interleave(G, 0) for i in (0, c.planes - 1))
        q = qkv[b, :nh * hd].view(nh, 1, hd)
        s = (q * k).sum(2) * c.scale
        size = (q.abs() * k.abs()).sum(2) * abs(c.scale)
        back = torch.arange(n - 1, -1, -1, dtype=torch.float64)
        if slopes is not None:
            bias = slopes.cpu().double()[:, None] * back
            s, size = s - bias, size + bias
        extra = torch.full((nh,), -math.inf, dtype=torch.float64)
        if head_sink is not None:
            extra = head_sink.cpu().double()
        elif sink:
            extra = torch.full((nh,), math.log(sink), dtype=torch.float64)
        w = torch.softmax(torch.cat([s, extra[:, None]], 1), 1)[:, :n]
        o = torch.einsum("hn,hnd->hd", w, v)
        wv = torch.einsum("hn,hnd->hd", w, v.abs())
        e = (hd + 8) * 2.0 ** -24 * size.amax(1, keepdim=True)
        near = 2 * e + (n + 64) * 2.0 ** -24
        if c.dtype is torch.bfloat16:
            near = near + U[torch.bfloat16]
        t = near * wv
        if gate_col:
            gate = torch.sigmoid(qkv[b, gate_col:gate_col + nh * hd].view(nh, hd))
            o, t = o * gate, t * gate + 8 * 2.0 ** -24 * (wv * gate)
        out.append(o.reshape(-1))
        tol.append((t + U[c.dtype] * o.abs() + 1e-30).reshape(-1))
    return torch.stack(out), torch.stack(tol)


def logprob_reference(x, t):
    """(result, bound): x [n, V] float32, t [n].  Rounded in float32: x - m (relative 2^-24, 1.44 times that as an exponent of 2, so a term is off
    by its |x - m| times 2^-22), the exponential (4 steps), the sums (at most V / 4096 + 40 of them one after another), the logarithm (2 steps) and
    the two differences."""
    x = x.double()
    m = x.amax(1, keepdim=True)
    p = torch.softmax(x, 1)
    out = torch.log_softmax(x, 1).gather(1, t.long()[:, None])[:, 0]
    far = torch.where(p > 0, p * (m - x), 0.0).sum(1)
    lse = torch.logsumexp(x - m, 1)
    bound = far * 2.0 ** -22 + (x.shape[1] / 1024 + 48) * 2.0 ** -24 + lse.abs() * 2.0 ** -22 + out.abs() * 2.0 ** -23 + (m - x.gather(1, t.long()[:, None]))[:, 0] * 2.0 ** -24
    return out, bound
