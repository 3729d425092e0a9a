"""The operators of the paged 8-bit K/V cache and of beam search over it, as cases for a timing harness.

Five kinds, each through the package's public entry points (``vault_amd.paged`` and ``ops.beam_select``):

* ``append``   new keys rotated at their positions, K / V rounded to 8 bits with one scale per page and head and
               written into the pages of a page table, queries rotated on the way; a read brings the values back
* ``attend``   attention of one or many query tokens per sequence over its pages: causal, optionally with a sliding
               window and first tokens that stay visible
* ``read``     a range of every sequence's rows dequantized into a dense tensor
* ``select``   beam search's choice of the best continuations over beams and vocabulary
* ``reorder``  the page tables and the pages being filled after such a choice, the reordered tails read back

Cache layout: K codes [layers, pages, G, P, D], V codes [layers, pages, G, D, P], one fp32 scale per (layer, page,
head) each.  ``i8`` codes are stored with an offset of 128 (value = (u - 128) * scale), ``e4m3`` codes are float8_e4m3fn
bits.  The 1.54B configuration has 12 query / 2 KV heads of 128, a window of 1024, 512 sinks and 28 layers.
"""
import math
import random

import torch

own = False

QMAX = {"i8": 127.0, "e4m3": 448.0}
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
THETA = 1_000_000.0
F64 = torch.float64


def listed():
    return [
        # a decode step of 64 conversations at different lengths: one new token each
        dict(name="append_decode_64", kind="append", mix=1, seqs=64, new=1, length=4096, H=12, G=2, D=128, page=64,
             fmt="i8", dtype="fp32"),
        # prompts of four requests entering the cache together
        dict(name="append_prompt_4x4096", kind="append", mix=2, seqs=4, new=4096, length=5000, H=32, G=8, D=128,
             page=64, fmt="e4m3", dtype="bf16"),
        # one user's decode step over two windows of context: latency
        dict(name="attend_one_2112", kind="attend", mix=3, seqs=1, new=1, length=2112, H=12, G=2, D=128, page=64,
             fmt="i8", dtype="fp32", window=0, sinks=0),
        # a serving batch of 64 long conversations, one token each: the cache's bandwidth
        dict(name="attend_batch_64x16384", kind="attend", mix=4, seqs=64, new=1, length=16384, H=32, G=8, D=128,
             page=64, fmt="e4m3", dtype="bf16", window=0, sinks=0),
        # three drafted tokens per sequence checked at once, sliding window with pinned sinks, small pages
        dict(name="attend_window_32x3", kind="attend", mix=5, seqs=32, new=3, length=8192, H=12, G=2, D=128, page=16,
             fmt="i8", dtype="fp32", window=1024, sinks=512),
        # a chunk of a long prompt over the context before it
        dict(name="attend_chunk_1024", kind="attend", mix=6, seqs=1, new=1024, length=9216, H=12, G=2, D=128, page=64,
             fmt="i8", dtype="bf16", window=0, sinks=0),
        # one conversation brought back to the dense tensors of the streaming state
        dict(name="read_one_3584", kind="read", mix=7, layers=1, seqs=1, rows=3584, length=3600, G=2, D=128, page=64,
             fmt="i8", dtype="bf16"),
        # a batch of long contexts of one layer handed to dense attention
        dict(name="read_batch_16x8192", kind="read", mix=8, layers=1, seqs=16, rows=8191, length=8300, G=8, D=128,
             page=32, fmt="e4m3", dtype="fp32"),
        # beam search of four hypotheses for one request
        dict(name="select_1x4", kind="select", mix=9, groups=1, beams=4, vocab=32000, done=0),
        # sixteen requests of eight beams over the full vocabulary, some hypotheses finished
        dict(name="select_16x8", kind="select", mix=10, groups=16, beams=8, vocab=151665, done=1),
        # the reordering that follows, one request
        dict(name="reorder_1x4", kind="reorder", mix=11, layers=28, groups=1, beams=4, length=700, G=2, D=128, page=64,
             fmt="i8"),
        # and a batch of requests, large pages
        dict(name="reorder_16x8", kind="reorder", mix=12, layers=28, groups=16, beams=8, length=2100, G=2, D=128,
             page=128, fmt="e4m3"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "read", "select", "reorder"])
    c = dict(kind=kind, mix=rng.randrange(1 << 20))
    if kind == "select":
        c.update(groups=_log_uniform(rng, 1, 16), beams=_log_uniform(rng, 1, 16), vocab=_log_uniform(rng, 100, 151665),
                 done=rng.randrange(2))
        return c
    G = rng.choice([1, 2, 3, 4, 8])
    c.update(G=G, D=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), fmt=rng.choice(["i8", "e4m3"]))
    if kind == "reorder":
        c.update(layers=rng.randrange(1, 29), groups=_log_uniform(rng, 1, 16), beams=rng.randrange(1, 9),
                 length=_log_uniform(rng, 20, 2100), G=min(G, 2))
        return c
    c["dtype"] = rng.choice(["fp32", "bf16"])
    if kind == "read":
        c.update(layers=rng.randrange(1, 4), seqs=_log_uniform(rng, 1, 8), rows=_log_uniform(rng, 1, 4000))
        c["length"] = c["rows"] + rng.randrange(200)
        return c
    c["H"] = G * rng.choice([1, 2, 4, 5, 6, 8])
    if kind == "append":
        if rng.random() < 0.5:
            c.update(seqs=_log_uniform(rng, 1, 64), new=rng.randrange(1, 5), length=_log_uniform(rng, 10, 4096))
        else:
            c.update(seqs=rng.randrange(1, 5), new=_log_uniform(rng, 5, 3000), length=4000)
        return c
    if rng.random() < 0.6:
        c.update(seqs=_log_uniform(rng, 1, 64), new=rng.randrange(1, 5), length=_log_uniform(rng, 8, 8192))
    else:
        c.update(seqs=rng.randrange(1, 4), new=_log_uniform(rng, 5, 900), length=_log_uniform(rng, 1000, 6000))
    masked = rng.random() < 0.5
    c.update(window=_log_uniform(rng, 1, 2048) if masked else 0, sinks=rng.choice([0, 4, 33, 512]) if masked else 0)
    return c


# ---------------------------------------------------------------- inputs


def _dev():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=_dev())


def _sizes(c):
    """(tokens in the cache, new tokens) of every sequence: the first has the case's full sizes, the others less."""
    r = random.Random(c["mix"])
    lens, news = [c["length"]], [min(c["new"], c["length"])]
    for _ in range(c["seqs"] - 1):
        lens.append(r.randint(max(1, c["length"] // 4), c["length"]))
        n = c["new"] if c["new"] < 5 else r.randint(1, c["new"])
        news.append(min(n, lens[-1]))
    return lens, news


def _starts(n):
    out = [0]
    for v in n:
        out.append(out[-1] + v)
    return out


def _codes(shape, fmt, g):
    """Codes of normally distributed values, as a cache of trained activations holds them."""
    x = torch.randn(shape, generator=g, device=_dev())
    if fmt == "i8":
        return (x.mul_(40.0).round_().clamp_(-127, 127) + 128.0).to(torch.uint8)
    return x.mul_(110.0).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _cache(c, n_pages, g):
    L, G, D, P = c.get("layers", 1), c["G"], c["D"], c["page"]
    unit = 1.0 / 40.0 if c["fmt"] == "i8" else 1.0 / 110.0
    scale = lambda: (torch.rand(L, n_pages, G, generator=g, device=_dev()) + 0.5) * unit  # noqa: E731
    return dict(k=_codes((L, n_pages, G, P, D), c["fmt"], g), v=_codes((L, n_pages, G, D, P), c["fmt"], g),
                ks=scale(), vs=scale())


def _table(lens, page, spare, g):
    """A page table of `lens` tokens per sequence, pages scattered over the cache: [B, most pages], -1 where none."""
    n = [-(-v // page) for v in lens]
    ids = torch.randperm(sum(n) + spare, generator=g, device=_dev()).to(torch.int32)
    width = max(n)
    at = torch.full((len(n), width), -1, dtype=torch.int32, device=_dev())
    first = _starts(n)
    for b in range(len(n)):
        at[b, :n[b]] = ids[first[b]:first[b + 1]]
    return at, sum(n) + spare


def _rope(n, D):
    inv = THETA ** (-torch.arange(0, D, 2, dtype=F64, device=_dev()) / D)
    ang = torch.arange(n, dtype=F64, device=_dev())[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=_dev()).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=_dev())  # noqa: E731
    s = dict(c=c)
    if c["kind"] == "select":
        R = c["groups"] * c["beams"]
        s["logits"] = rand(R, c["vocab"]) * 3.0
        s["scores"] = -(rand(c["groups"], c["beams"]).abs() * 4.0).cumsum(1)
        s["eos"] = c["vocab"] // 2
        s["done"] = (torch.rand(c["groups"], c["beams"], generator=g, device=_dev()) < 0.2 * c["done"]).to(torch.uint8)
        return s
    if c["kind"] == "reorder":
        B, K = c["groups"], c["beams"]
        r = random.Random(c["mix"])
        lens = [v for v in [r.randint(max(1, c["length"] // 4), c["length"]) for _ in range(B)] for _ in range(K)]
        # every beam owns the page that its next token goes to
        s["table"], n_pages = _table([v + 1 for v in lens], c["page"], 3, g)
        s["lens"] = _ints(lens)
        s["tail"] = _ints([v // c["page"] * c["page"] for v in lens])
        s["parents"] = torch.randint(0, K, (B, K), generator=g, device=_dev(), dtype=torch.int32)
        s["table_out"], s["lens_out"] = torch.empty_like(s["table"]), torch.empty_like(s["lens"])
        s.update(_cache(c, n_pages, g))
        return s
    if c["kind"] == "read":
        r = random.Random(c["mix"])
        lens = [c["length"]] + [r.randint(max(1, c["length"] // 2), c["length"]) for _ in range(c["seqs"] - 1)]
        s["table"], n_pages = _table(lens, c["page"], 5, g)
        s["lens"] = _ints(lens)
        s["first"] = _ints([max(0, v - c["rows"]) for v in lens])
        s.update(_cache(c, n_pages, g))
        return s
    lens, news = _sizes(c)
    dt = DT[c["dtype"]]
    N = sum(news)
    s["table"], n_pages = _table(lens, c["page"], 5, g)
    s["lens"] = _ints(lens)
    s["q_start"] = None if max(news) == 1 else _ints(_starts(news))
    s["most"] = max(news)
    s.update(_cache(c, n_pages, g))
    s["q"] = (rand(N, c["H"], c["D"]) * 2.0).to(dt)
    if c["kind"] == "append":
        s["start"] = _ints([v - n for v, n in zip(lens, news)])
        s["newk"], s["newv"] = rand(N, c["G"], c["D"]).to(dt), rand(N, c["G"], c["D"]).to(dt)
        s["rope"] = _rope(max(lens), c["D"])
        # what is read back: from the start of the page that the first new token goes to
        s["first"] = s["start"] // c["page"] * c["page"]
        s["rows"] = max(v - (v - n) // c["page"] * c["page"] for v, n in zip(lens, news))
    return s


# ---------------------------------------------------------------- the package's own operators


def _handles(s):
    """The cache handle and the scratch that a program keeps beside its tensors."""
    if "kv" not in s:
        from vault_amd import ops, paged
        s["kv"] = paged.PagedKV(s["k"], s["v"], s["ks"], s["vs"], {"i8": paged.I8, "e4m3": paged.E4M3}[s["c"]["fmt"]])
        s["ws"] = ops.Workspace(s["k"].device)
    return s["kv"], s["ws"]


def _run_own(s):
    from vault_amd import ops, paged
    c = s["c"]
    if c["kind"] == "select":
        if "ws" not in s:
            s["ws"] = ops.Workspace(s["logits"].device)
        scores, parents, tokens, done = ops.beam_select(s["logits"], s["scores"], done=s["done"], eos=s["eos"],
                                                        ws=s["ws"])
        return dict(scores=scores, parents=parents, tokens=tokens, done=done)
    kv, ws = _handles(s)
    if c["kind"] == "append":
        q = paged.append(kv, 0, s["newk"], s["newv"], s["table"], s["start"], rope=s["rope"], q=s["q"],
                         q_start=s["q_start"], max_new=s["most"])
        k, v = paged.read(kv, s["table"], s["first"], s["rows"], s["lens"])
        return dict(q=q, k=k, v=v)
    if c["kind"] == "attend":
        return dict(out=paged.attend(kv, 0, s["q"], s["table"], s["lens"], q_start=s["q_start"], max_new=s["most"],
                                     window=c["window"], n_sink=c["sinks"], ws=ws))
    if c["kind"] == "read":
        k, v = paged.read(kv, s["table"], s["first"], c["rows"], s["lens"], dtype=DT[c["dtype"]])
        return dict(k=k, v=v)
    paged.reorder(kv, s["table"], s["lens"], s["parents"], s["table_out"], s["lens_out"])
    k, v = paged.read(kv, s["table_out"], s["tail"], c["page"], s["lens_out"])
    return dict(table=s["table_out"], lens=s["lens_out"], k=k, v=v)


# ---------------------------------------------------------------- plain forms


def _values(u, fmt):
    return u.float() - 128.0 if fmt == "i8" else u.view(torch.float8_e4m3fn).float()


def _round8(x, fmt):
    """fp32 quotients -> codes."""
    if fmt == "i8":
        return (x.round().clamp(-127, 127) + 128.0).to(torch.uint8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _gathered(s, layer, pages):
    """fp32 K, V [B, G, tokens, D] of the given table entries [B, n]."""
    c, at = s["c"], pages.clamp(min=0).long()
    B, n = pages.shape
    k = _values(s["k"][layer][at], c["fmt"]) * s["ks"][layer][at][..., None, None]        # [B, n, G, P, D]
    v = _values(s["v"][layer][at], c["fmt"]) * s["vs"][layer][at][..., None, None]        # [B, n, G, D, P]
    k = k.permute(0, 2, 1, 3, 4).reshape(B, c["G"], n * c["page"], c["D"])
    v = v.permute(0, 2, 1, 4, 3).reshape(B, c["G"], n * c["page"], c["D"])
    return k, v


def _plain_read(s, table, first, rows, lens, dtype):
    c = s["c"]
    L, P, B = s["k"].shape[0], c["page"], table.shape[0]
    pos = first[:, None] + torch.arange(rows, device=table.device)[None]                   # [B, rows]
    page = table.gather(1, (pos // P).clamp(max=table.shape[1] - 1).long())
    ok = (pos < lens[:, None]) & (page >= 0)
    at, off = page.clamp(min=0).long(), (pos % P).long()
    heads = torch.arange(c["G"], device=table.device)
    idx = (at[:, None, :], heads[None, :, None], off[:, None, :])                          # [B, G, rows]
    k = _values(s["k"][:, idx[0], idx[1], idx[2]], c["fmt"]) * s["ks"][:, idx[0], idx[1]][..., None]
    v = _values(s["v"].transpose(3, 4)[:, idx[0], idx[1], idx[2]], c["fmt"]) * s["vs"][:, idx[0], idx[1]][..., None]
    keep = ok[None, :, None, :, None]
    return (torch.where(keep, k, 0.0).to(dtype).view(L, B, c["G"], rows, c["D"]),
            torch.where(keep, v, 0.0).to(dtype).view(L, B, c["G"], rows, c["D"]))


def _owner(s, N):
    """The sequence of every row and its place in it."""
    dev = s["table"].device
    if s["q_start"] is None:
        return torch.arange(N, device=dev), torch.zeros(N, dtype=torch.long, device=dev)
    row = torch.arange(N, device=dev)
    seq = torch.searchsorted(s["q_start"].long(), row, right=True) - 1
    return seq, row - s["q_start"].long()[seq]


def _rotated(x, rope):
    """fp64 rotation of x [N, heads, D] by rope rows [N, D], rounded once to fp32."""
    h = x.shape[-1] // 2
    a, b = x[..., :h].double(), x[..., h:].double()
    cos, sin = rope[:, None, :h].double(), rope[:, None, h:].double()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).float()


def _plain_store(codes, scales, x, page, off, first_page, n_old, fmt):
    """Rows x [N, G, D] into codes [pages, G, P, D] at (page, off); the page that a sequence's first row goes to holds
    n_old older tokens."""
    n_pages, G = scales.shape
    a = torch.zeros(n_pages, G, device=x.device)
    a.scatter_reduce_(0, page[:, None].expand(-1, G), x.abs().amax(-1), "amax")
    touched = torch.zeros(n_pages, dtype=torch.bool, device=x.device)
    touched[page] = True
    older = torch.zeros(n_pages, dtype=torch.long, device=x.device)
    older[first_page] = n_old
    a = a / torch.full_like(a, QMAX[fmt])      # a division: by a plain number it would be a product with the inverse
    new = torch.where(older[:, None] > 0, torch.maximum(scales, a), a)
    new = torch.where(touched[:, None], new, scales)
    # older tokens of the pages that were partly filled, on the new scale
    grown = (older[first_page, None] > 0) & (new[first_page] > scales[first_page])        # [B, G]
    old = codes[first_page]                                                               # [B, G, P, D]
    q = _values(old, fmt).double() * scales[first_page].double()[..., None, None]
    again = _round8((q / new[first_page].double()[..., None, None]).float(), fmt)
    at = torch.arange(codes.shape[2], device=x.device)
    keep = grown[:, :, None] & (at[None, None] < n_old[:, None, None])
    codes[first_page] = torch.where(keep[..., None], again, old)
    div = torch.where(new > 0, new, 1.0)[page].double()[..., None]
    heads = torch.arange(G, device=x.device)[None]
    codes[page[:, None], heads, off[:, None]] = _round8((x.double() / div).float(), fmt)
    scales.copy_(new)


def _plain_append(s):
    c = s["c"]
    N = s["newk"].shape[0]
    seq, i = _owner(s, N)
    pos = s["start"].long()[seq] + i
    rope = s["rope"][pos]
    page = s["table"][seq, pos // c["page"]].long()
    first_page = s["table"].gather(1, (s["start"] // c["page"]).long()[:, None])[:, 0].long()
    n_old = (s["start"] % c["page"]).long()
    args = (page, pos % c["page"], first_page, n_old, c["fmt"])
    _plain_store(s["k"][0], s["ks"][0], _rotated(s["newk"], rope), *args)
    _plain_store(s["v"][0].transpose(2, 3), s["vs"][0], s["newv"].float(), *args)
    q = _rotated(s["q"], rope).to(s["q"].dtype)
    k, v = _plain_read(s, s["table"], s["first"], s["rows"], s["lens"], torch.float32)
    return dict(q=q, k=k, v=v)


def _plain_attend(s):
    c = s["c"]
    B, G, D, R = s["table"].shape[0], c["G"], c["D"], c["H"] // c["G"]
    k, v = _gathered(s, 0, s["table"])
    N, most, dev = s["q"].shape[0], s["most"], s["q"].device
    seq, i = _owner(s, N)
    q = torch.zeros(B, most, c["H"], D, device=dev)
    q[seq, i] = s["q"].float()
    n = torch.zeros(B, dtype=torch.long, device=dev).scatter_add_(0, seq, torch.ones_like(seq))
    q = q.view(B, most, G, R, D).permute(0, 2, 1, 3, 4).reshape(B, G, most * R, D)
    p = s["lens"].long()[:, None] - n[:, None] + torch.arange(most, device=dev)[None]      # [B, most]
    j = torch.arange(k.shape[2], device=dev)
    see = j[None, None] <= p[..., None]
    if c["window"]:
        see = see & ((j[None, None] > p[..., None] - c["window"]) | (j < c["sinks"]))
    see = see[:, None, :, None, :].expand(B, 1, most, R, j.numel()).reshape(B, 1, most * R, j.numel())
    a = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5
    a = a.masked_fill_(~see, -math.inf)
    m = a.amax(-1, keepdim=True).clamp(min=-3e38)
    a = a.sub_(m).exp_()
    o = torch.matmul(a, v) / a.sum(-1, keepdim=True)
    o = o.view(B, G, most, R, D).permute(0, 2, 1, 3, 4).reshape(B, most, c["H"], D)
    return dict(out=o[seq, i].to(s["q"].dtype))


def _plain_select(s):
    c = s["c"]
    B, K, V = c["groups"], c["beams"], c["vocab"]
    x = s["logits"].double()
    lse = torch.log((x - x.amax(1, keepdim=True)).exp().sum(1, keepdim=True)) + x.amax(1, keepdim=True)
    total = (s["scores"].double()[..., None] + (x - lse).view(B, K, V))
    ended = torch.full_like(total, -math.inf)
    ended[..., s["eos"]] = s["scores"].double()
    total = torch.where(s["done"][..., None] != 0, ended, total).view(B, K * V)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    if at.shape[1] < K:
        raise ValueError("fewer candidates than beams")
    parents, tokens = (at // V).to(torch.int32), at % V
    done = s["done"].gather(1, parents.long()) | (tokens == s["eos"]).to(torch.uint8)
    return dict(scores=best.float(), parents=parents, tokens=tokens, done=done)


def _plain_reorder(s):
    c = s["c"]
    B, K, P = c["groups"], c["beams"], c["page"]
    dev, T = s["table"].device, s["table"].shape[1]
    par = s["parents"].long()
    beam = torch.arange(K, device=dev).expand(B, K)
    takes = par[:, None, :] == beam[:, :, None]                                            # [B, parent, child]
    first = torch.where(takes, beam[:, None, :], K).amin(-1)                               # [B, parent]
    heir = first.gather(1, par) == beam                                                    # the child that takes over
    dead = ~takes.any(-1)
    rank = (~heir).long().cumsum(1) - 1                                                    # among the other children
    left = torch.argsort((~dead).long(), dim=1, stable=True)                               # dead beams first, in order
    giver = torch.where(heir, par, left.gather(1, rank.clamp(min=0)))
    row = (torch.arange(B, device=dev)[:, None] * K + par).view(-1)
    give = (torch.arange(B, device=dev)[:, None] * K + giver).view(-1)
    lens = s["lens"][row]
    at = (lens // P).long()[:, None]
    own_at = (s["lens"] // P).long()[:, None]
    tail = s["table"].gather(1, own_at)                                                    # [B K, 1]
    j = torch.arange(T, device=dev)[None]
    later = torch.where(j > own_at, s["table"], -1)
    table = torch.where(j < at, s["table"][row], torch.where(j == at, tail[give], later))
    src, dst = tail[row, 0].long(), tail[give, 0].long()
    for name in ("k", "v", "ks", "vs"):
        s[name][:, dst] = s[name][:, src]
    s["table_out"].copy_(table)
    s["lens_out"].copy_(lens)
    k, v = _plain_read(s, s["table_out"], s["tail"], P, s["lens_out"], torch.float32)
    return dict(table=s["table_out"], lens=s["lens_out"], k=k, v=v)


def run(s):
    if own:
        return _run_own(s)
    kind = s["c"]["kind"]
    if kind == "append":
        return _plain_append(s)
    if kind == "attend":
        return _plain_attend(s)
    if kind == "select":
        return _plain_select(s)
    if kind == "reorder":
        return _plain_reorder(s)
    k, v = _plain_read(s, s["table"], s["first"], s["c"]["rows"], s["lens"], DT[s["c"]["dtype"]])
    return dict(k=k, v=v)


# ---------------------------------------------------------------- what a pass cannot do without


def _visible(c):
    """(keys that some query of a sequence sees, (query, key) pairs), summed over the sequences."""
    keys = pairs = 0
    for n_kv, n_q in zip(*_sizes(c)):
        w, sink = c["window"], c["sinks"]
        seen = lambda p: p + 1 if not w else min(p + 1, w + min(sink, max(0, p + 1 - w)))  # noqa: E731
        pairs += sum(seen(n_kv - n_q + t) for t in range(n_q))
        lo = 0 if not w else max(0, n_kv - n_q - w + 1)
        keys += n_kv - lo + min(lo, sink)
    return keys, pairs


def work(case):
    c = case
    if c["kind"] == "select":
        n = c["groups"] * c["beams"]
        return dict(bytes=n * (c["vocab"] * 4 + 26), flops=n * c["vocab"] * 3)
    G, D, P = c["G"], c["D"], c["page"]
    if c["kind"] == "reorder":
        # on average K (1 - 1/K)^K beams lose their page to a copy; tails of K beams read back
        B, K, L = c["groups"], c["beams"], c["layers"]
        page = G * P * D * 2 + G * 8
        copies = B * K * (1.0 - 1.0 / K) ** K
        table = B * K * -(-(c["length"] + 1) // P) * 8
        return dict(bytes=L * (2 * copies * page + B * K * page * 5) + table, flops=L * B * K * G * P * D * 2)
    if c["kind"] == "read":
        n = c["layers"] * c["seqs"] * c["rows"] * G * D * 2
        return dict(bytes=n * (1 + DT[c["dtype"]].itemsize), flops=n)
    lens, news = _sizes(c)
    N, es = sum(news), DT[c["dtype"]].itemsize
    if c["kind"] == "append":
        back = sum(v - (v - n) // P * P for v, n in zip(lens, news))
        b = N * (2 * G * D * es + 2 * c["H"] * D * es + D * 4 + 2 * G * D) + back * G * D * 2 * 5
        return dict(bytes=b, flops=N * (2 * G + c["H"]) * D * 6)
    keys, pairs = _visible(c)
    return dict(bytes=keys * G * D * 2 + -(-keys // P) * G * 8 + 2 * N * c["H"] * D * es, flops=4 * pairs * c["H"] * D)


# ---------------------------------------------------------------- the definitions in 64 bits


def _code_values(fmt, dev):
    """What each of the 256 codes stands for, from the format's definition."""
    if fmt == "i8":
        return torch.arange(256, dtype=F64, device=dev) - 128.0
    out = []
    for u in range(256):
        e, m = (u >> 3) & 15, u & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        x = math.nan if (u & 127) == 127 else x
        out.append(-x if u & 128 else x)
    return torch.tensor(out, dtype=F64, device=dev)


def _to_code_values(x, fmt):
    """The nearest value that a code stands for (ties to even), x within the format's range."""
    if fmt == "i8":
        return torch.round(x).clamp(-127, 127)
    mag = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(mag.clamp(min=2.0 ** -6))) - 3.0)
    return torch.sign(x) * torch.round(mag / step) * step


def _exact_rows(s, name, layer, b, table, lo, hi):
    """fp64 rows [G, hi - lo, D] of sequence b."""
    c = s["c"]
    P = c["page"]
    val = _code_values(c["fmt"], s["k"].device)
    first, last = lo // P, -(-hi // P)
    pages = table[b, first:last].long()
    u = s[name][layer][pages]
    u = u if name == "k" else u.transpose(2, 3)
    x = val[u.long()] * s[name + "s"][layer][pages].double()[..., None, None]
    x = x.transpose(0, 1).reshape(c["G"], -1, c["D"])
    return x[:, lo - first * P:hi - first * P]


def _exact_read(s, table, first, rows, lens):
    c, L, B = s["c"], s["k"].shape[0], table.shape[0]
    out = {}
    for name in ("k", "v"):
        full = torch.zeros(L, B, c["G"], rows, c["D"], dtype=F64, device=table.device)
        for layer in range(L):
            for b in range(B):
                lo, hi = first[b], min(lens[b], first[b] + rows)
                if hi > lo:
                    full[layer, b, :, :hi - lo] = _exact_rows(s, name, layer, b, table, lo, hi)
        out[name] = full
    return out


def _exact_append(s):
    c = s["c"]
    lens, news = _sizes(c)
    P, G, D, h, fmt = c["page"], c["G"], c["D"], c["D"] // 2, c["fmt"]
    val, qs = _code_values(fmt, s["k"].device), _starts(news)
    rope = s["rope"].double()

    def turn(x, pos):
        x, cs, sn = x.double(), rope[pos, :h][:, None], rope[pos, h:][:, None]
        return torch.cat([x[..., :h] * cs - x[..., h:] * sn, x[..., h:] * cs + x[..., :h] * sn], -1)

    q, back = [], dict(k=torch.zeros(1, len(lens), G, s["rows"], D, dtype=F64, device=s["k"].device))
    back["v"] = torch.zeros_like(back["k"])
    for b, (hi, n) in enumerate(zip(lens, news)):
        lo = hi - n
        pos = torch.arange(lo, hi, device=s["k"].device)
        q.append(turn(s["q"][qs[b]:qs[b + 1]], pos))
        # the rotated key is held in fp32
        rows = dict(k=turn(s["newk"][qs[b]:qs[b + 1]], pos).float().double(), v=s["newv"][qs[b]:qs[b + 1]].double())
        base = lo // P * P
        for name, x in rows.items():
            for p0 in range(base, hi, P):
                a, z = max(p0, lo), min(p0 + P, hi)
                new = x[a - lo:z - lo].transpose(0, 1)                                     # [G, n, D]
                scale = (new.abs().amax((1, 2)) / QMAX[fmt]).float().double()
                if a > p0:
                    page = s["table"][b, p0 // P].long()
                    was = s[name + "s"][0, page].double()
                    scale = torch.maximum(scale, was)
                    u = s[name][0, page] if name == "k" else s[name][0, page].transpose(1, 2)
                    old = val[u[:, :a - p0].long()]
                    # quotients are rounded to fp32, then to 8 bits
                    again = _to_code_values((old * was[:, None, None] / scale[:, None, None]).float().double(), fmt)
                    old = torch.where((scale > was)[:, None, None], again, old)
                    back[name][0, b, :, p0 - base:a - base] = old * scale[:, None, None]
                code = _to_code_values((new / scale[:, None, None]).float().double(), fmt)
                back[name][0, b, :, a - base:z - base] = code * scale[:, None, None]
    return dict(q=torch.cat(q), k=back["k"], v=back["v"])


def _exact_attend(s):
    c = s["c"]
    lens, news = _sizes(c)
    G, D, R, qs, out = c["G"], c["D"], c["H"] // c["G"], _starts(news), []
    for b, (n_kv, n_q) in enumerate(zip(lens, news)):
        k, v = (_exact_rows(s, name, 0, b, s["table"], 0, n_kv) for name in ("k", "v"))
        q = s["q"][qs[b]:qs[b + 1]].double().view(n_q, G, R, D)
        j = torch.arange(n_kv, device=k.device)
        o = torch.empty_like(q)
        for g in range(G):
            for t0 in range(0, n_q, 128):
                p = n_kv - n_q + torch.arange(t0, min(n_q, t0 + 128), device=k.device)[:, None]
                see = j <= p
                if c["window"]:
                    see = see & ((j > p - c["window"]) | (j < c["sinks"]))
                a = (q[t0:t0 + 128, g] @ k[g].T) / math.sqrt(D)
                a = torch.where(see[:, None], a, -math.inf)
                o[t0:t0 + 128, g] = torch.softmax(a, -1) @ v[g]
        out.append(o.view(n_q, c["H"], D))
    return dict(out=torch.cat(out))


def _exact_select(s):
    c = s["c"]
    K, V, rows = c["beams"], c["vocab"], []
    for b in range(c["groups"]):
        cand = []
        for k in range(K):
            score = float(s["scores"][b, k])
            if int(s["done"][b, k]):
                cand.append((-score, k * V + s["eos"]))
                continue
            lp = torch.log_softmax(s["logits"][b * K + k].double(), 0)
            top = torch.topk(lp, min(V, K + 8))
            cand += [(-(score + t), k * V + i) for t, i in zip(top.values.tolist(), top.indices.tolist())]
        rows.append(sorted(cand)[:K])
    dev = s["logits"].device
    at = torch.tensor([[i for _, i in r] for r in rows], device=dev)
    parents, tokens = at // V, at % V
    done = s["done"].gather(1, parents) | (tokens == s["eos"]).to(torch.uint8)
    return dict(scores=torch.tensor([[-t for t, _ in r] for r in rows], dtype=F64, device=dev),
                parents=parents.to(torch.int32), tokens=tokens, done=done)


def _exact_reorder(s):
    c = s["c"]
    B, K, P = c["groups"], c["beams"], c["page"]
    table, lens, par = s["table"].tolist(), s["lens"].tolist(), s["parents"].tolist()
    new_table, new_lens, copies = [], [], []
    for b in range(B):
        tails = [table[b * K + k][lens[b * K + k] // P] for k in range(K)]
        free = [tails[k] for k in range(K) if k not in par[b]]
        taken = set()
        for k in range(K):
            p = par[b][k]
            at, n = lens[b * K + p] // P, lens[b * K + p]
            tail = tails[p]
            if p in taken:
                copies.append((tail, free[0]))
                tail = free.pop(0)
            taken.add(p)
            mine = lens[b * K + k] // P
            new_table.append([table[b * K + p][j] if j < at else tail if j == at else table[b * K + k][j] if j > mine
                              else -1 for j in range(len(table[0]))])
            new_lens.append(n)
    moved = {name: s[name].clone() for name in ("k", "v", "ks", "vs")}
    for src, dst in copies:
        for x in moved.values():
            x[:, dst] = x[:, src]
    t = dict(s, table=_ints(new_table), **moved)
    values = _exact_read(t, t["table"], s["tail"].tolist(), P, new_lens)
    return dict(table=t["table"], lens=_ints(new_lens), **values)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "append":
        return _exact_append(s)
    if kind == "attend":
        return _exact_attend(s)
    if kind == "select":
        return _exact_select(s)
    if kind == "reorder":
        return _exact_reorder(s)
    return _exact_read(s, s["table"], s["first"].tolist(), case["rows"], s["lens"].tolist())
