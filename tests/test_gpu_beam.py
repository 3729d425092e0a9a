"""Beam selection on the GPU against the float64 oracle, and a beam search over the paged cache as a user runs it.

Bars: parents, tokens and flags exactly; scores within the rounding of the result to fp32 and of the fp32 exponentials'
sum (2^-20 in its logarithm: 2^-22 each for exp2's argument and value, 2^-22 for the sum of a chunk in 32 steps per lane)."""
import numpy as np
import pytest
import torch

from oracle import paged as op
from vault_amd import ops, paged

pytestmark = pytest.mark.gpu


def _check(dev, x, s, done=None, eos=-1, ws=None):
    want = op.beam_select(x, s, done, eos)
    got = ops.beam_select(torch.from_numpy(x).to(dev), torch.from_numpy(s).to(dev),
                          done=None if done is None else torch.from_numpy(done).to(dev), eos=eos, ws=ws)
    sc, par, tok, dn = (t.cpu().numpy() for t in got)
    assert np.array_equal(par, want[1]) and np.array_equal(tok, want[2]), (par, want[1], tok, want[2])
    assert np.array_equal(dn, want[3])
    fin = np.isfinite(want[0])
    assert np.array_equal(fin, np.isfinite(sc))
    tol = 2.0 ** -24 * np.abs(want[0][fin]) + 2.0 ** -20
    assert (np.abs(sc[fin] - want[0][fin]) <= tol).all()
    return sc, par, tok, dn


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 5), (3, 4, 1000), (2, 8, 4096), (2, 8, 4097), (5, 3, 8191), (1, 64, 3000),
                                   (2, 33, 20000), (1, 5, 151665), (16, 8, 70001), (1, 64, 64), (1, 2, 1 << 19), (1, 33, 1 << 19)])
def test_select(dev, B, K, V):
    rng = np.random.default_rng(B * K + V)
    x = (rng.standard_normal((B * K, V)) * 3).astype(np.float32)
    s = -np.sort(rng.uniform(0, 5, (B, K))).astype(np.float32)
    _check(dev, x, s)
    done = (rng.random((B, K)) < 0.4).astype(np.uint8)
    _check(dev, x, s, done, eos=V - 1)


@pytest.mark.parametrize("K,V", [(4, 3000), (16, 9000), (64, 5000)])
def test_select_ties(dev, K, V):
    """Equal logits everywhere, few distinct values, sorted rows, equal beams: ties to the smaller beam, then token."""
    rng = np.random.default_rng(K)
    s = np.zeros((1, K), np.float32)
    _check(dev, np.zeros((K, V), np.float32), s)
    # one row's sum in any order of 32-bit additions is the same here: every exponential is 1 or 2^-k
    few = np.repeat(rng.integers(0, 2, (1, V)).astype(np.float32) * 64, K, 0)
    _check(dev, few, s)
    for row in (np.arange(V), np.arange(V)[::-1]):
        _check(dev, np.repeat((row * 1e-3).astype(np.float32)[None], K, 0), s)


def test_select_masks(dev):
    """-inf logits, the type's lowest value, NaN and +inf rows, inactive beams (-inf, -1e9, the lowest value), fewer
    candidates than beams, all finished."""
    rng = np.random.default_rng(3)
    K, V = 4, 6000
    x = rng.standard_normal((2 * K, V)).astype(np.float32)
    x[0, 10:] = -np.inf
    x[1, :] = -np.inf
    x[2, 5:] = np.finfo(np.float32).min
    x[3, 77] = np.nan
    x[5, 9] = np.inf
    x[6, 3000:] = -np.inf
    s = np.zeros((2, K), np.float32)
    _check(dev, x, s)
    for low in (-np.inf, np.float32(-1e9), np.finfo(np.float32).min):
        first = np.array([[0] + [low] * (K - 1)] * 2, np.float32)
        _check(dev, rng.standard_normal((2 * K, V)).astype(np.float32), first)
    few = np.full((K, V), -np.inf, np.float32)
    few[0, 5], few[2, 4000] = 1.0, 2.0
    sc, par, tok, dn = _check(dev, few, s[:1])
    assert list(tok[0][2:]) == [-1, -1] and list(par[0][2:]) == [2, 3] and list(dn[0][2:]) == [1, 1]
    _check(dev, x, s, np.ones((2, K), np.uint8), eos=0)
    _check(dev, x, np.full((2, K), -np.inf, np.float32))


def test_select_strided_in_graph(dev):
    """Logits as rows of a wider tensor; captured and replayed on new logits, eager work between, one workspace."""
    B, K, V = 3, 5, 30000
    rng = np.random.default_rng(6)
    wide = torch.zeros(B * K, V + 7, device=dev)
    x, s = wide[:, :V], torch.zeros(B, K, device=dev)
    ws = ops.Workspace(dev)
    ops.beam_select(x, s, ws=ws)
    graph = torch.cuda.CUDAGraph()
    st = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        out = ops.beam_select(x, s, ws=ws)
    for _ in range(4):
        x.copy_(torch.from_numpy(rng.standard_normal((B * K, V)).astype(np.float32)))
        s.copy_(torch.from_numpy(rng.standard_normal((B, K)).astype(np.float32)))
        graph.replay()
        want = op.beam_select(x.cpu().numpy(), s.cpu().numpy())
        assert np.array_equal(out[1].cpu().numpy(), want[1]) and np.array_equal(out[2].cpu().numpy(), want[2])
        again = ops.beam_select(x, s)
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_select_refusals(dev):
    x, s = torch.randn(6, 100, device=dev), torch.zeros(2, 3, device=dev)
    d = torch.zeros(2, 3, dtype=torch.uint8, device=dev)
    for f in (lambda: ops.beam_select(x.half(), s), lambda: ops.beam_select(x[:5], s), lambda: ops.beam_select(x.cpu(), s),
              lambda: ops.beam_select(x, s[0]), lambda: ops.beam_select(x, s, done=d), lambda: ops.beam_select(x.t(), s),
              lambda: ops.beam_select(x, s, done=d.bool(), eos=3), lambda: ops.beam_select(x, s.double())):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(Exception):
        ops.beam_select(x, s, done=d, eos=100)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_beam_search_over_the_cache(dev, fmt):
    """A toy model (one attention layer between random projections) searched with K beams, two prompts of different
    lengths: append, attend, the LM head, select, reorder, for more steps than two pages hold.  The oracle runs the same
    search in float64 on dense histories of its own cache; choices are equal at every step."""
    P, G, H, D, K, V, steps = 16, 1, 2, 64, 3, 200, 37
    rng = np.random.default_rng(21)
    emb = rng.standard_normal((V, (H + 2 * G) * D)).astype(np.float32)
    head = (rng.standard_normal((V, H * D)) * 2.0).astype(np.float32)
    prompts = [rng.integers(0, V, n) for n in (21, 5)]
    B = len(prompts)
    longest = max(len(q) for q in prompts) + steps + 1
    ang = np.arange(longest)[:, None] * (1e4 ** (-np.arange(0, D, 2) / D))
    rope = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    cols = -(-longest // P)
    table = np.arange(B * K * cols, dtype=np.int32).reshape(B * K, cols)
    table = rng.permutation(B * K * cols).astype(np.int32)[table]
    kv = paged.PagedKV.empty(1, B * K * cols, G, D, dev, page=P, fmt=paged.I8 if fmt == "i8" else paged.E4M3)
    cache = op.empty(B * K * cols, G, P, D, fmt)
    i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)  # noqa: E731
    d_emb, d_head, d_rope = (torch.from_numpy(a).to(dev) for a in (emb, head, rope))

    def split(x):
        x = x.reshape(-1, H + 2 * G, D)
        return x[:, :H], x[:, H:H + G], x[:, H + G:]

    # prompts into every beam's own pages (all but the last token)
    rows = np.concatenate([prompts[b][:-1] for b in range(B) for _ in range(K)])
    counts = [len(prompts[b]) - 1 for b in range(B) for _ in range(K)]
    q, k, v = split(emb[rows])
    op.append(cache, k, v, table, [0] * (B * K), counts, rope)
    dq, dk, dv = split(d_emb[torch.from_numpy(rows).to(dev)])
    d_table, d_next = i32(table), i32(table)
    lens = np.array(counts)
    d_lens, d_lens2 = i32(lens), i32(lens)
    qs = i32(np.concatenate([[0], np.cumsum(counts)]))
    paged.append(kv, 0, dk, dv, d_table, torch.zeros_like(d_lens), rope=d_rope, q_start=qs)

    scores = np.full((B, K), -np.inf, np.float32)
    scores[:, 0] = 0
    d_scores = torch.from_numpy(scores).to(dev)
    tokens = np.array([prompts[b][-1] for b in range(B) for _ in range(K)])
    d_tokens = torch.from_numpy(tokens).to(dev)
    ws = ops.Workspace(dev)
    for step in range(steps):
        q, k, v = split(emb[tokens])
        qr = op.append(cache, k, v, table, lens, [1] * (B * K), rope, q)
        o, _, _, _ = op.attend(cache, qr, table, lens + 1, [1] * (B * K))
        logits = o.reshape(B * K, -1) @ head.T.astype(np.float64)
        ts, tp, tt, _ = op.beam_select(logits, scores)

        dq, dk, dv = split(d_emb[d_tokens])
        dq = paged.append(kv, 0, dk, dv, d_table, d_lens, rope=d_rope, q=dq)
        do = paged.attend(kv, 0, dq, d_table, d_lens + 1, ws=ws)
        dl = do.reshape(B * K, -1) @ d_head.T
        assert np.abs(dl.double().cpu().numpy() - logits).max() < 1e-3
        d_scores, d_par, d_tok, _ = ops.beam_select(dl, d_scores, ws=ws)
        assert np.array_equal(d_par.cpu().numpy(), tp) and np.array_equal(d_tok.cpu().numpy(), tt), step
        scores, tokens, lens = ts.astype(np.float32), tt.reshape(-1), lens + 1
        d_lens += 1
        d_tokens = d_tok.reshape(-1)
        # each beam's open page is its own, also where the length has just reached a border
        paged.reorder(kv, d_table, d_lens, d_par, d_next, d_lens2)
        new, n2, copies = op.reorder(table.tolist(), lens, tp.tolist(), P)
        for src, dst in copies:
            for f in ("k", "v", "ks", "vs"):
                cache[f][dst] = cache[f][src]
        table, lens = np.array(new, np.int32), np.array(n2)
        d_table, d_next, d_lens, d_lens2 = d_next, d_table, d_lens2, d_lens
        assert np.array_equal(d_table.cpu().numpy(), table) and np.array_equal(d_lens.cpu().numpy(), lens)
