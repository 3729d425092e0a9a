"""The paged 8-bit K/V cache on the GPU against the float64 oracle (oracle/paged.py).

Bars: stored values and scales equal to the oracle's bit for bit (as the fp32 values that codes and scales stand for),
rotated queries within an fp32 rounding or two, attention within oracle.paged.attend_bound (derived there), reads the
product of code and scale rounded once, reordered tables and pages exactly."""
import numpy as np
import pytest
import torch

from oracle import paged as op
from vault_amd import _lib as L
from vault_amd import ops, paged

pytestmark = pytest.mark.gpu

FMT = {"i8": paged.I8, "e4m3": paged.E4M3}
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
HALF = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8}


def _rope(n, D, seed=0):
    ang = np.arange(n)[:, None] * (1e4 ** (-np.arange(0, D, 2) / D))
    return np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)


def _table(rng, lens, P, n_pages, cols=None):
    """Scattered pages for `lens` tokens per sequence; unused entries name no page."""
    need = [-(-int(n) // P) for n in lens]
    ids = rng.permutation(n_pages)[:sum(need)]
    cols = cols or max(max(need), 1)
    t = np.full((len(lens), cols), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = ids[at:at + n]
        at += n
    return t


def _garbage(rng, pages, G, P, D, fmt):
    """Random codes everywhere, every byte among them (the NaN codes too), scales NaN."""
    c = op.empty(pages, G, P, D, fmt)
    c["k"][:] = rng.integers(0, 256, c["k"].shape)
    c["v"][:] = rng.integers(0, 256, c["v"].shape)
    c["ks"][:], c["vs"][:] = np.nan, np.nan
    return c


def _fill(rng, c, table, lens, spread=0.0):
    """Codes that an append could have left at the sequences' tokens, with scales spread over 10^(+-spread)."""
    P, pages = c["k"].shape[2], c["k"].shape[0]
    fine = np.flatnonzero(np.isfinite(op.code_values(c["fmt"])) & (op.code_values(c["fmt"]) >= -127.5 if c["fmt"] == "i8"
                                                                     else True))
    for b, n in enumerate(lens):
        for pos in range(0, int(n), P):
            if pos // P >= table.shape[1]:
                break
            page = table[b, pos // P]
            if not 0 <= page < pages:
                continue
            m = min(P, int(n) - pos)
            G, D = c["k"].shape[1], c["k"].shape[3]
            c["k"][page, :, :m] = op.round8(rng.standard_normal((G, m, D)) * 40, c["fmt"])
            c["v"][page, :, :, :m] = op.round8(rng.standard_normal((G, D, m)) * 40, c["fmt"])
            c["ks"][page] = rng.uniform(0.5, 1.5, G) / 40
            c["vs"][page] = rng.uniform(0.5, 1.5, G) / 40 * 10.0 ** rng.uniform(-spread, spread, G)
    assert len(fine)


def _to(c, dev):
    """The oracle's cache on the device, as layer 1 of two."""
    two = lambda a: torch.from_numpy(np.stack([np.zeros_like(a), a])).to(dev)  # noqa: E731
    return paged.PagedKV(two(c["k"]), two(c["v"]), two(c["ks"]), two(c["vs"]), FMT[c["fmt"]])


def _i32(a, dev):
    return torch.from_numpy(np.asarray(a, dtype=np.int32)).to(dev)


def _starts(counts, dev):
    return _i32(np.concatenate([[0], np.cumsum(counts)]), dev)


def _held(kv, c, table, lens):
    """Codes and scales at the sequences' tokens: device against oracle, as values."""
    P = c["k"].shape[2]
    got = dict(k=kv.k[1].cpu().numpy(), v=kv.v[1].cpu().numpy(), ks=kv.k_scale[1].cpu().numpy(),
               vs=kv.v_scale[1].cpu().numpy(), fmt=c["fmt"])
    for b, n in enumerate(lens):
        n = min(int(n), table.shape[1] * P)
        gk, gv, ok = op.rows(got, table[b], 0, max(0, n))
        wk, wv, _ = op.rows(c, table[b], 0, max(0, n))
        assert np.array_equal(gk, wk, equal_nan=True), (b, "k")
        assert np.array_equal(gv, wv, equal_nan=True), (b, "v")
    return got


# ------------------------------------------------------------------ append

APPENDS = [  # D, page, G, H, starts, counts
    (128, 64, 2, 12, [0, 5, 63, 64, 130], [1, 1, 1, 1, 1]),
    (64, 16, 3, 3, [0, 1, 15, 16, 31], [1, 16, 17, 1, 40]),
    (128, 32, 1, 5, [0, 0, 7], [100, 0, 33]),
    (64, 128, 2, 4, [100, 300], [300, 1]),
    (128, 256, 2, 2, [250, 0], [20, 257]),
]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("shape", APPENDS, ids=lambda s: f"D{s[0]}P{s[1]}")
def test_append(dev, shape, fmt, dt):
    """Ragged runs into garbage pages, older tokens appended by the same operator first; scales grow in the second."""
    D, P, G, H, start, counts = shape
    rng = np.random.default_rng(D + P)
    lens = [s + n for s, n in zip(start, counts)]
    c = _garbage(rng, 60, G, P, D, fmt)
    kv = _to(c, dev)
    table = _table(rng, lens, P, 60)
    rope = _rope(max(lens) + 1, D)
    t, rt = _i32(table, dev), torch.from_numpy(rope).to(dev)
    for st, cn, amp in (([0] * len(start), start, 1.0), (start, counts, 1.7)):
        N = int(sum(cn))
        if N == 0:
            continue
        x = [torch.from_numpy(rng.standard_normal((N, h, D)).astype(np.float32) * amp).to(DT[dt]) for h in (G, G, H)]
        k, v, q = (y.float().numpy() for y in x)
        want = op.append(c, k, v, table, st, cn, rope, q)
        one = all(n == 1 for n in cn)
        got = paged.append(kv, 1, x[0].to(dev), x[1].to(dev), t, _i32(st, dev), rope=rt, q=x[2].to(dev),
                           q_start=None if one else _starts(cn, dev))
        # an fp32 product and an fma, then the rounding of the type
        tol = 3 * 2.0 ** -24 * (np.abs(q) + np.abs(np.roll(q, D // 2, -1))) + HALF[dt] * np.abs(want)
        assert got.dtype == DT[dt] and (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    _held(kv, c, table, lens)
    assert not kv.k[0].any() and not kv.k_scale[0].any()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_append_extremes(dev, fmt):
    """Zeros, ties at every half step, the smallest and largest magnitudes, infinities and NaN (which make their own page
    and head NaN and nothing else), without rotation."""
    D, P, G = 64, 16, 2
    rng = np.random.default_rng(9)
    c = _garbage(rng, 12, G, P, D, fmt)
    kv = _to(c, dev)
    table = _table(rng, [160], P, 12)
    x = rng.standard_normal((160, G, D)).astype(np.float32)
    x[0:16] = 0
    x[16:32] = np.round(x[16:32] * 40) + 0.5
    x[16, :, 0] = 127 if fmt == "i8" else 448
    x[32:48] *= 1e-38
    x[48:64] *= 3e37
    x[64:80] *= 1e-44
    x[83, 0, 5] = np.inf
    x[99, 1, 63] = -np.inf
    x[112, 0, 0] = np.nan
    x[128:144, 0] = 0
    x[128:144, 1] *= 10.0 ** rng.uniform(-9, 9, (16, D)).astype(np.float32)
    for at, n in ((0, 60), (60, 4), (64, 50), (114, 46)):
        op.append(c, x[at:at + n], x[at:at + n][:, ::-1], table, [at], [n])
        d = torch.from_numpy(x[at:at + n].copy()).to(dev)
        paged.append(kv, 1, d, d.flip(1), _i32(table, dev), _i32([at], dev), q_start=_starts([n], dev))
    got = _held(kv, c, table, [160])
    bad = np.isnan(got["ks"][table[0]])
    assert bad[5, 0] and bad[6, 1] and bad[7, 0] and bad.sum() == 3
    # a page that is started anew is clean again
    y = rng.standard_normal((16, G, D)).astype(np.float32)
    op.append(c, y, y, table, [80], [16])
    d = torch.from_numpy(y).to(dev)
    paged.append(kv, 1, d, d, _i32(table, dev), _i32([80], dev), q_start=_starts([16], dev))
    _held(kv, c, table, [160])
    assert np.isfinite(kv.k_scale[1].cpu().numpy()[table[0][5]]).all()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_append_skips_what_has_no_place(dev, fmt):
    """Positions below 0, past the table, pages that do not exist, rows behind the last sequence, positions without a
    rope row (NaN)."""
    D, P, G, H = 64, 16, 1, 2
    rng = np.random.default_rng(4)
    c = _garbage(rng, 20, G, P, D, fmt)
    kv = _to(c, dev)
    table = _table(rng, [64, 64, 64], P, 20)
    table[1, 1], table[2, 0] = -1, 20
    start, counts = [-3, 10, 5], [20, 60, 20]
    N = sum(counts) + 7
    k, v, q = (rng.standard_normal((N, h, D)).astype(np.float32) for h in (G, G, H))
    rope = _rope(40, D)
    want = op.append(c, k, v, table, start, counts, rope, q)
    out = torch.full((N, H, D), 77.0, device=dev)
    got = paged.append(kv, 1, *(torch.from_numpy(a).to(dev) for a in (k, v)), _i32(table, dev), _i32(start, dev),
                       rope=torch.from_numpy(rope).to(dev), q=torch.from_numpy(q).to(dev), q_out=out,
                       q_start=_starts(counts, dev))
    assert got is out
    g = out.cpu().numpy()
    assert (g[-7:] == 77).all() and (g[:3] == 77).all()
    assert np.allclose(g[3:-7], want[3:-7], atol=3e-6, equal_nan=True) and np.isnan(g[sum(counts[:2]) - 10]).all()
    for f in ("k", "v", "ks", "vs"):
        a = {"k": kv.k, "v": kv.v, "ks": kv.k_scale, "vs": kv.v_scale}[f][1].cpu().numpy()
        if f in ("ks", "vs"):
            assert np.array_equal(a, c[f], equal_nan=True)
        else:
            ok = np.isfinite(c["ks" if f == "k" else "vs"])     # codes of a NaN page mean nothing
            val = op.code_values(fmt)
            assert np.array_equal(val[a][ok], val[c[f]][ok], equal_nan=True)


def test_append_in_place_and_strided(dev):
    """q rotated in place; q, k, v as slices of one projection's rows."""
    D, P, G, H, N = 128, 64, 2, 4, 9
    rng = np.random.default_rng(5)
    c = op.empty(4, G, P, D, "i8")
    kv = _to(c, dev)
    qkv = torch.from_numpy(rng.standard_normal((N, H + 2 * G, D)).astype(np.float32)).to(dev)
    q, k, v = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    table, rope = np.array([[2]], np.int32), _rope(64, D)
    want = op.append(c, *(t.cpu().numpy() for t in (k, v)), table, [3], [N], rope, q.cpu().numpy())
    before = qkv[:, H:].clone()
    got = paged.append(kv, 1, k, v, _i32(table, dev), _i32([3], dev), rope=torch.from_numpy(rope).to(dev), q=q, q_out=q,
                       q_start=_starts([N], dev))
    assert got.data_ptr() == qkv.data_ptr() and torch.equal(qkv[:, H:], before)
    assert np.abs(q.double().cpu().numpy() - want).max() < 2e-6
    gk, gv, _ = op.rows(c, [2], 3, 3 + N)
    rk, rv = paged.read(kv, _i32(table, dev), _i32([3], dev), N, _i32([3 + N], dev))
    assert np.array_equal(rk[1, 0].double().cpu().numpy(), np.float32(gk)) and \
        np.array_equal(rv[1, 0].double().cpu().numpy(), np.float32(gv))


# ------------------------------------------------------------------ attention

def _attend(dev, c, table, lens, counts, H, dt, seed=0, qamp=2.0, tail=0, kv=None, **kw):
    rng = np.random.default_rng(seed)
    D = c["k"].shape[3]
    N = int(sum(counts))
    q = torch.from_numpy(rng.standard_normal((N + tail, H, D)).astype(np.float32) * qamp).to(DT[dt])
    out, size, reach, seen = op.attend(c, q[:N].float().numpy(), table, lens, counts, kw.get("window", 0),
                                       kw.get("n_sink", 0), kw.get("scale"))
    kv = kv or _to(c, dev)
    one = all(n == 1 for n in counts) and not tail
    dst = torch.full((N + tail, H, D), 55.0, dtype=DT[dt], device=dev)
    got = paged.attend(kv, 1, q.to(dev), _i32(table, dev), _i32(lens, dev), q_start=None if one else _starts(counts, dev),
                       out=dst, **kw)
    g = got.double().cpu().numpy()
    assert (g[N:] == 55).all()
    tol = op.attend_bound(out, size, reach, seen, D, dt == "bf16")
    bad = ~(np.abs(g[:N] - out) <= tol)
    bad &= ~(np.isnan(out) & np.isnan(g[:N]))
    assert not bad.any(), (np.argwhere(bad)[:5], np.nanmax(np.abs(g[:N] - out) / tol))
    return g[:N], out, tol


DECODE = [  # D, page, G, H, lens
    (128, 64, 2, 12, [1, 2, 63, 64, 65, 0, 700]),
    (64, 16, 1, 1, [1, 15, 16, 17, 300]),
    (128, 32, 3, 15, [33, 5, 1000]),
    (64, 256, 2, 34, [255, 257, 31]),
    (128, 128, 8, 32, [129, 400]),
    (64, 64, 1, 16, [5000]),
]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("shape", DECODE, ids=lambda s: f"D{s[0]}P{s[1]}H{s[3]}")
def test_attend_one_token(dev, shape, fmt, dt):
    D, P, G, H, lens = shape
    rng = np.random.default_rng(D + P)
    pages = sum(-(-n // P) for n in lens) + 3
    c = _garbage(rng, pages, G, P, D, fmt)
    table = _table(rng, lens, P, pages)
    _fill(rng, c, table, lens)
    got, out, _ = _attend(dev, c, table, lens, [1] * len(lens), H, dt)
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all()


MANY = [  # D, page, G, H, lens, counts, window, sinks
    (128, 64, 2, 12, [200, 64, 70], [100, 64, 1], 0, 0),
    (64, 16, 1, 3, [90, 33, 40, 5], [90, 0, 17, 8], 0, 0),          # more queries than tokens: rows that see nothing
    (128, 16, 2, 8, [400, 300], [3, 50], 64, 0),
    (64, 32, 2, 6, [500, 130], [70, 130], 33, 5),
    (128, 64, 1, 6, [1000, 20], [5, 20], 100, 70),
    (64, 128, 1, 20, [300], [40], 1, 0),
    (128, 32, 2, 4, [260], [2], 1, 300),
    (128, 64, 1, 7, [1500], [300], 0, 0),
]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("shape", MANY, ids=lambda s: f"D{s[0]}P{s[1]}H{s[3]}w{s[6]}")
def test_attend_many_tokens(dev, shape, fmt, dt):
    D, P, G, H, lens, counts, window, sinks = shape
    rng = np.random.default_rng(D + P + window)
    pages = sum(-(-n // P) for n in lens) + 3
    c = _garbage(rng, pages, G, P, D, fmt)
    table = _table(rng, lens, P, pages)
    _fill(rng, c, table, lens)
    _attend(dev, c, table, lens, counts, H, dt, tail=2, window=window, n_sink=sinks)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_attend_pages_left_behind(dev, fmt):
    """Pages between the sinks and the window given back (-1, or an id past the cache) and holding NaN: the same bits as
    with them; a hole inside the window is not visible."""
    D, P, G, H = 128, 16, 2, 6
    rng = np.random.default_rng(8)
    lens = [400, 170]
    c = _garbage(rng, 60, G, P, D, fmt)
    table = _table(rng, lens, P, 60)
    _fill(rng, c, table, lens)
    a, _, _ = _attend(dev, c, table, lens, [2, 1], H, "fp32", tail=1, window=50, n_sink=20)
    gone = table.copy()
    gone[0, 2:21], gone[1, 2:7] = -1, 60
    for page in table[0, 2:21]:
        c["ks"][page] = c["vs"][page] = np.nan
    b, _, _ = _attend(dev, c, gone, lens, [2, 1], H, "fp32", tail=1, window=50, n_sink=20)
    assert np.array_equal(a, b)
    gone[0, 23] = -7
    gone[1, :] = 1 << 30
    got, _, _ = _attend(dev, c, gone, lens, [2, 1], H, "fp32", tail=1, window=50, n_sink=20)
    assert (got[2] == 0).all() and (got[:2] != a[:2]).any()


def test_attend_past_the_table(dev):
    """Lengths past what the table's row can name: the tokens there are not visible."""
    rng = np.random.default_rng(8)
    c = _garbage(rng, 6, 1, 16, 64, "i8")
    table = _table(rng, [64, 64][:1], 16, 6)
    _fill(rng, c, table, [64])
    _attend(dev, c, table, [90], [30], 2, "fp32", tail=1)
    _attend(dev, c, table, [1 << 29], [1], 2, "fp32", window=1 << 29)
    _attend(dev, c, table, [-5], [1], 2, "fp32")


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_attend_scales_far_apart(dev, fmt, dt):
    """Page scales over 10 decades within one sequence, pages of zeros, and one page whose scale is 0."""
    D, P, G, H = 64, 16, 1, 4
    rng = np.random.default_rng(12)
    lens = [900, 64]
    c = _garbage(rng, 70, G, P, D, fmt)
    table = _table(rng, lens, P, 70)
    _fill(rng, c, table, lens, spread=5.0)
    z = table[0, 5]
    c["k"][z], c["v"][z], c["ks"][z], c["vs"][z] = (128, 128, 0, 0) if fmt == "i8" else (0, 0, 0, 0)
    # a page that takes nearly all the probability and holds zeros
    y = table[0, 7]
    c["v"][y], c["vs"][y] = 128 if fmt == "i8" else 0, 0
    c["ks"][y] *= 30
    for page in table[1, :4]:
        c["vs"][page] = 0
        c["v"][page] = 128 if fmt == "i8" else 0
    got, _, _ = _attend(dev, c, table, lens, [1, 1], H, dt)
    assert (got[1] == 0).all()


def test_attend_peaked_and_signed_scales(dev):
    """Scores up to some thousands (one key takes all), a negative scale, scale 0, zero queries."""
    rng = np.random.default_rng(13)
    D, P, G, H, lens = 128, 64, 2, 4, [300, 70]
    c = _garbage(rng, 9, G, P, D, "i8")
    table = _table(rng, lens, P, 9)
    _fill(rng, c, table, lens)
    for scale, amp in ((3.0, 20.0), (-0.1, 2.0), (0.0, 2.0), (0.1, 0.0), (0.1, 1e-30), (1e-30, 1e30)):
        # peaked softmaxes: the bound is of the scores' size, far from 1
        _attend(dev, c, table, lens, [1, 1], H, "fp32", qamp=amp, scale=scale)


def test_attend_nan_stays_where_it_is(dev):
    """A NaN block reaches the rows that see it and no others; non-finite queries reach their own rows."""
    rng = np.random.default_rng(14)
    D, P, G, H, lens = 64, 16, 2, 4, [100, 100]
    c = _garbage(rng, 20, G, P, D, "i8")
    table = _table(rng, lens, P, 20)
    _fill(rng, c, table, lens)
    c["vs"][table[0, 5], 0] = np.nan          # tokens 80 .. 95, heads 0 and 1
    c["ks"][table[1, 1], 1] = np.nan          # tokens 16 .. 31, heads 2 and 3
    kv = _to(c, dev)
    q = rng.standard_normal((60, H, D)).astype(np.float32)
    q[59, 0, 3], q[58, 3, 3] = np.inf, np.nan
    out = paged.attend(kv, 1, torch.from_numpy(q).to(dev), _i32(table, dev), _i32(lens, dev), q_start=_starts([30, 30], dev),
                       window=40).cpu().numpy()
    bad = np.isnan(out)
    want = np.zeros_like(bad)
    p = np.arange(70, 100)
    want[:30, :2] = (p >= 80)[:, None, None]
    want[30:, 2:] = (p - 40 < 31)[:, None, None]
    want[59, 0] = want[58, 3] = True
    assert np.array_equal(bad, want)


def test_attend_strides_and_hints(dev):
    """Rows of a wider tensor for q and out, table rows of a wider table, hints of any kind: the same values."""
    rng = np.random.default_rng(15)
    D, P, G, H, lens, counts = 128, 32, 2, 4, [700, 90, 300], [5, 9, 1]
    c = _garbage(rng, 50, G, P, D, "e4m3")
    table = _table(rng, lens, P, 50)
    _fill(rng, c, table, lens)
    kv = _to(c, dev)
    q = torch.from_numpy(rng.standard_normal((15, H, D)).astype(np.float32)).to(dev)
    wide = torch.zeros(15, H + 3, D, device=dev)
    wide[:, :H] = q
    tw = torch.full((3, table.shape[1] + 5), 3, dtype=torch.int32, device=dev)
    tw[:, :table.shape[1]] = _i32(table, dev)
    args = dict(q_start=_starts(counts, dev))
    a = paged.attend(kv, 1, q, _i32(table, dev), _i32(lens, dev), **args)
    out = torch.zeros(15, H + 1, D, device=dev)
    b = paged.attend(kv, 1, wide[:, :H], tw[:, :table.shape[1]], _i32(lens, dev), out=out[:, 1:], **args)
    assert torch.equal(a, b) and not out[:, 0].any()
    assert torch.equal(a, paged.attend(kv, 1, q, _i32(table, dev), _i32(lens, dev), **args))
    for mn, mk in ((1, 1), (15, 64), (9, 700), (0, 0)):
        d = paged.attend(kv, 1, q, _i32(table, dev), _i32(lens, dev), max_new=mn, max_keys=mk, **args)
        assert (d - a).abs().max() < 2e-6
    got = paged.attend(kv, 1, q[:3], _i32(table, dev), _i32(lens, dev))
    assert got.shape == (3, H, D)


def test_attend_offsets_past_32_bits(dev):
    """A cache whose codes and table entries lie past 4 GiB: the same bits as a small one."""
    D, P, G, H = 128, 256, 8, 8
    rng = np.random.default_rng(16)
    lens = [600]
    c = _garbage(rng, 3, G, P, D, "i8")
    table = np.array([[2, 0, 1]], np.int32)
    _fill(rng, c, table, lens)
    small = _to(c, dev)
    n = (1 << 32) // (G * P * D) + 40
    k = torch.zeros(1, n, G, P, D, dtype=torch.uint8, device=dev)
    v = torch.zeros(1, n, G, D, P, dtype=torch.uint8, device=dev)
    ks = torch.zeros(1, n, G, device=dev)
    vs = torch.zeros(1, n, G, device=dev)
    big = paged.PagedKV(k, v, ks, vs, paged.I8)
    far = [n - 1, n - 30, n - 7]
    for i, page in enumerate(table[0]):
        k[0, far[i]], v[0, far[i]] = small.k[1, page], small.v[1, page]
        ks[0, far[i]], vs[0, far[i]] = small.k_scale[1, page], small.v_scale[1, page]
    q = torch.randn(1, H, D, device=dev)
    a = paged.attend(small, 1, q, _i32(table, dev), _i32(lens, dev))
    b = paged.attend(big, 0, q, _i32([far], dev), _i32(lens, dev))
    assert torch.equal(a, b)
    x = torch.randn(100, G, D, device=dev)
    for kv, layer, t in ((small, 1, table), (big, 0, [far])):
        paged.append(kv, layer, x, x, _i32(t, dev), _i32([590], dev), q_start=_starts([100], dev))
    r = [paged.read(kv, _i32(t, dev), _i32([500], dev), 190, _i32([690], dev)) for kv, t in ((small, table), (big, [far]))]
    assert torch.equal(r[0][0][1], r[1][0][0]) and torch.equal(r[0][1][1], r[1][1][0])


# ------------------------------------------------------------------ read

@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("D,P,G", [(128, 64, 2), (64, 16, 3), (128, 256, 1), (64, 128, 1)])
def test_read(dev, fmt, dt, D, P, G):
    rng = np.random.default_rng(D + P)
    lens, first = [100, 0, 37, 300, 50], [-5, 0, 36, 200, 70]
    c = _garbage(rng, 60, G, P, D, fmt)
    table = _table(rng, lens, P, 60)
    _fill(rng, c, table, lens)
    if P == 16:
        table[3, 14] = -1
    kv = _to(c, dev)
    for n in (1, 17, 111, 0):
        k, v = paged.read(kv, _i32(table, dev), _i32(first, dev), n, _i32(lens, dev), DT[dt])
        assert k.shape == (2, 5, G, n, D) and k.dtype == DT[dt]
        for b in range(5):
            wk, wv, ok = op.rows(c, table[b], first[b], first[b] + n)
            there = ok & (np.arange(first[b], first[b] + n) < lens[b])
            for got, want in ((k, wk), (v, wv)):
                want = torch.from_numpy(np.where(there[None, :, None], want, 0)).float().to(DT[dt])   # code * scale in fp32
                assert torch.equal(got[1, b].cpu(), want)


# ------------------------------------------------------------------ reorder

@pytest.mark.parametrize("P", [16, 128])
@pytest.mark.parametrize("B,K", [(1, 1), (1, 4), (5, 7), (2, 64)])
def test_reorder(dev, B, K, P):
    """Tables, lengths, and every layer's pages and scales as the oracle says; pages that are no target keep their bytes.
    Lengths differ by group, some at a page's border; parents outside the group mean the beam itself."""
    rng = np.random.default_rng(B * K + P)
    layers, G, D, cols = 3, 2, 64, 6
    pages = B * K * cols
    kv = paged.PagedKV(*(torch.randint(0, 256, (layers, pages, G, *t), dtype=torch.uint8, device=dev)
                         for t in ((P, D), (D, P))),
                       *(torch.rand(layers, pages, G, device=dev) for _ in range(2)), paged.E4M3)
    for turn in range(4):
        lens = np.repeat(rng.integers(0, (cols - 1) * P, B), K)
        if turn == 1:
            lens[:] = 2 * P
        table = rng.permutation(pages).reshape(B * K, cols).astype(np.int32)
        par = rng.integers(0, K, (B, K)) if turn else np.full((B, K), K - 1)
        if turn == 3:
            par[0, 0], par[-1, -1] = -1, K
        was = [t.clone() for t in (kv.k, kv.v, kv.k_scale, kv.v_scale)]
        t, ln = _i32(table, dev), _i32(lens, dev)
        to, lo = torch.full_like(t, 99), torch.full_like(ln, 99)
        paged.reorder(kv, t, ln, _i32(par, dev), to, lo)
        wt, wl, copies = op.reorder(table.tolist(), lens, par.tolist(), P)
        assert to.tolist() == wt and lo.tolist() == wl
        for x, w in zip((kv.k, kv.v, kv.k_scale, kv.v_scale), was):
            for s, d in copies:
                w[:, d] = w[:, s]
            assert torch.equal(x, w)


def test_reorder_without_pages(dev):
    """Open pages that do not exist, or lie past the table, are not copied."""
    kv = paged.PagedKV.empty(1, 4, 1, 64, dev, page=16)
    kv.k.random_(0, 256)
    was = kv.k.clone()
    for lens, rows in (([16 * 2 + 3] * 2, [[0, 1], [2, 3]]), ([20, 20], [[0, -1], [2, 3]]), ([20, 20], [[0, 1], [2, 4]])):
        t, ln = _i32(rows, dev), _i32(lens, dev)
        to, lo = torch.empty_like(t), torch.empty_like(ln)
        paged.reorder(kv, t, ln, _i32([[0, 0]], dev), to, lo)
        assert to.tolist() == op.reorder(rows, lens, [[0, 0]], 16)[0] and torch.equal(kv.k, was)


# ------------------------------------------------------------------ refusals, streams, graphs

def test_refusals(dev):
    kv = paged.PagedKV.empty(1, 4, 2, 64, dev, page=16)
    t, n = _i32([[0, 1]], dev), _i32([5], dev)
    x, q = torch.randn(1, 2, 64, device=dev), torch.randn(1, 4, 64, device=dev)
    bad = [
        lambda: paged.PagedKV(kv.k, kv.k, kv.k_scale, kv.v_scale, paged.I8),
        lambda: paged.PagedKV(kv.k.cpu(), kv.v, kv.k_scale, kv.v_scale, paged.I8),
        lambda: paged.PagedKV(kv.k, kv.v, kv.k_scale.double(), kv.v_scale, paged.I8),
        lambda: paged.PagedKV(kv.k, kv.v, kv.k_scale, kv.v_scale, 8),
        lambda: paged.PagedKV.empty(1, 4, 2, 96, dev),
        lambda: paged.PagedKV.empty(1, 4, 2, 64, dev, page=8),
        lambda: paged.append(kv, 1, x, x, t, n),
        lambda: paged.append(kv, 0, x.half(), x.half(), t, n),
        lambda: paged.append(kv, 0, x, x.bfloat16(), t, n),
        lambda: paged.append(kv, 0, x.cpu(), x, t, n),
        lambda: paged.append(kv, 0, x, x, t.long(), n),
        lambda: paged.append(kv, 0, x, x, t, n.long()),
        lambda: paged.append(kv, 0, x.expand(3, 2, 64), x.expand(3, 2, 64), t, n),
        lambda: paged.append(kv, 0, x, x, t, n, q_start=_i32([0, 1, 2], dev)),
        lambda: paged.append(kv, 0, x, x, t, n, rope=torch.zeros(8, 32, device=dev)),
        lambda: paged.append(kv, 0, x, x, t, n, q=q.bfloat16()),
        lambda: paged.append(kv, 0, x, x, t, n, q_out=q),
        lambda: paged.append(kv, 0, x, x, t, n, q=q, q_out=q.transpose(1, 2)),
        lambda: paged.attend(kv, 0, q[:, :3], t, n),
        lambda: paged.attend(kv, 0, q.double(), t, n),
        lambda: paged.attend(kv, 0, q, t, n, window=-1),
        lambda: paged.attend(kv, 0, q, t, n, out=torch.empty(1, 4, 64)),
        lambda: paged.attend(kv, 0, q, t[0], n),
        lambda: paged.attend(kv, 0, q, t, n[:0]),
        lambda: paged.read(kv, t, n, -1, n),
        lambda: paged.read(kv, t, n, 3, n, torch.float16),
        lambda: paged.reorder(kv, t, n, _i32([[0]], dev), t, n.clone()),
        lambda: paged.reorder(kv, t, n, _i32([[0, 0]], dev), t.clone(), n.clone()),
        lambda: paged.reorder(kv, t, n, _i32([0], dev), t.clone(), n.clone()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError(i)
    with pytest.raises(L.VGXError):
        many = torch.zeros(1, 1 << 26, dtype=torch.int32, device=dev)
        paged.attend(kv, 0, q, many, n)
    e = torch.empty(0, 2, 64, device=dev)
    assert paged.attend(kv, 0, torch.empty(0, 4, 64, device=dev), t[:0], n[:0]).shape == (0, 4, 64)
    paged.append(kv, 0, e, e, t[:0], n[:0])


def _decode_step(kv, x, t, start, rope, ws):
    q = paged.append(kv, 0, x[1], x[2], t, start, rope=rope, q=x[0])
    return paged.attend(kv, 0, q, t, start + 1, ws=ws)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_captured_step_follows_the_device(dev, fmt):
    """One captured append + attend replayed while lengths, tables and inputs move on, with eager work between: every
    replay equals the eager step of another cache."""
    D, P, G, H, B = 128, 16, 2, 8, 5
    g = torch.Generator(device=dev).manual_seed(3)
    kv, ref = (paged.PagedKV.empty(1, 40, G, D, dev, page=P, fmt=FMT[fmt]) for _ in range(2))
    rope = torch.from_numpy(_rope(128, D)).to(dev)
    table = _i32(np.random.default_rng(1).permutation(40).reshape(B, 8), dev)
    start = _i32([0, 5, 14, 15, 31], dev)
    x = [torch.randn(B, h, D, generator=g, device=dev) for h in (H, G, G)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ws, ws2 = ops.Workspace(dev), ops.Workspace(dev)
    with torch.cuda.stream(s):
        _decode_step(kv, x, table, start, rope, ws)
    torch.cuda.current_stream().wait_stream(s)
    for t in (kv.k, kv.v, kv.k_scale, kv.v_scale):
        t.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = _decode_step(kv, x, table, start, rope, ws)
    for c in (ref.k, ref.v, ref.k_scale, ref.v_scale):
        c.zero_()
    for step in range(6):
        for y in x:
            y.normal_(generator=g)
        graph.replay()
        want = _decode_step(ref, x, table, start, rope, ws2)
        assert torch.equal(out, want), step
        assert torch.equal(kv.k, ref.k) and torch.equal(kv.v, ref.v) and torch.equal(kv.k_scale, ref.k_scale)
        start += 1
        torch.cuda.synchronize()


def test_two_streams(dev):
    """Two sequences' steps on two streams with a workspace each, and without one: the same bits as one after the other."""
    D, P, G, H = 128, 64, 2, 12
    rng = np.random.default_rng(2)
    kvs, tabs, lens, qs = [], [], [], []
    for i in range(2):
        c = _garbage(rng, 80, G, P, D, "i8")
        table = _table(rng, [4000], P, 80)
        _fill(rng, c, table, [4000])
        kvs.append(_to(c, dev))
        tabs.append(_i32(table, dev))
        lens.append(_i32([4000 - i], dev))
        qs.append(torch.randn(1, H, D, device=dev))
    want = [paged.attend(kvs[i], 1, qs[i], tabs[i], lens[i]) for i in range(2)]
    streams, spaces = [torch.cuda.Stream() for _ in range(2)], [ops.Workspace(dev), None]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged.attend(kvs[i], 1, qs[i], tabs[i], lens[i], ws=spaces[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_attend_joined_in_the_launch(dev, fmt, dt):
    """Splits joined by the last workgroup (a Workspace) give the bits of the joining launch (none); calls of several
    batches share the workspace, whose tickets are zero after each; beam selection may use it in between."""
    rng = np.random.default_rng(31)
    ws = ops.Workspace(dev)
    for lens, counts, H, D, P, G in (([3000], [1], 12, 128, 64, 2), ([2500, 70, 1], [1, 1, 1], 4, 64, 16, 4),
                                     ([1500, 900], [3, 4], 8, 128, 32, 2), ([5000] * 3, [1] * 3, 32, 128, 128, 1)):
        pages = sum(-(-n // P) for n in lens) + 2
        c = _garbage(rng, pages, G, P, D, fmt)
        table = _table(rng, lens, P, pages)
        _fill(rng, c, table, lens)
        kv = _to(c, dev)
        q = torch.from_numpy(rng.standard_normal((sum(counts), H, D)).astype(np.float32)).to(DT[dt]).to(dev)
        qs = None if set(counts) == {1} else _starts(counts, dev)
        args = (kv, 1, q, _i32(table, dev), _i32(lens, dev))
        kw = dict(q_start=qs, max_new=max(counts))
        want = paged.attend(*args, **kw)
        for _ in range(5):
            assert torch.equal(paged.attend(*args, ws=ws, **kw), want)
            assert not ws.tickets().any()
        ops.beam_select(torch.randn(6, 9000, device=dev), torch.zeros(2, 3, device=dev), ws=ws)
        out, size, reach, seen = op.attend(c, q.float().cpu().numpy(), table, lens, counts)
        tol = op.attend_bound(out, size, reach, seen, D, dt == "bf16")
        assert (np.abs(want.double().cpu().numpy() - out) <= tol).all()


def test_captured_splits(dev):
    """A captured call over several splits, replayed while the lengths grow and shrink, eager calls on the same workspace
    in between (never at the same time)."""
    rng = np.random.default_rng(32)
    D, P, G, H = 128, 64, 2, 12
    c = _garbage(rng, 80, G, P, D, "i8")
    table = _table(rng, [4000], P, 80)
    _fill(rng, c, table, [4000])
    kv, t, lens = _to(c, dev), _i32(table, dev), _i32([4000], dev)
    q, ws = torch.randn(1, H, D, device=dev), ops.Workspace(dev)
    paged.attend(kv, 1, q, t, lens, ws=ws)
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=s):
        out = paged.attend(kv, 1, q, t, lens, ws=ws)
    for n in (4000, 1, 0, 257, 64, 3999, 2000):
        lens.fill_(n)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, paged.attend(kv, 1, q, t, lens, ws=ws)) and torch.equal(got, paged.attend(kv, 1, q, t, lens))
        assert not ws.tickets().any() and (n > 0 or not got.any())


def test_workspace_first_used_in_a_capture(dev):
    """A workspace whose first user is a capture, then an eager call before any replay, then replays."""
    rng = np.random.default_rng(33)
    D, P, G, H = 64, 32, 2, 8
    c = _garbage(rng, 100, G, P, D, "i8")
    table = _table(rng, [3000], P, 100)
    _fill(rng, c, table, [3000])
    kv, t, lens = _to(c, dev), _i32(table, dev), _i32([3000], dev)
    q, ws = torch.randn(1, H, D, device=dev), ops.Workspace(dev)
    want = paged.attend(kv, 1, q, t, lens)
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=s):
        out = paged.attend(kv, 1, q, t, lens, ws=ws)
    assert torch.equal(paged.attend(kv, 1, q, t, lens, ws=ws), want)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(paged.attend(kv, 1, q, t, lens, ws=ws), want) and not ws.tickets().any()


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("lens,counts", [([2600], [1]), ([700, 5, 90], [9, 1, 30]), ([40], [40])])
def test_attend_in_place(dev, lens, counts, dt):
    """out is q: the same bits as into another tensor, split or not, with few rows and many."""
    rng = np.random.default_rng(34)
    D, P, G, H, N = 128, 32, 2, 12, sum(counts)
    c = _garbage(rng, 110, G, P, D, "e4m3")
    table = _table(rng, lens, P, 110)
    _fill(rng, c, table, lens)
    kv, t, n, ws = _to(c, dev), _i32(table, dev), _i32(lens, dev), ops.Workspace(dev)
    q = torch.from_numpy(rng.standard_normal((N, H, D)).astype(np.float32)).to(DT[dt]).to(dev)
    for most in (2, max(counts)):
        for w in (None, ws):
            kw = dict(q_start=_starts(counts, dev), max_new=most, ws=w)
            want, y = paged.attend(kv, 1, q, t, n, **kw), q.clone()
            assert paged.attend(kv, 1, y, t, n, out=y, **kw) is y and torch.equal(y, want)


def test_attend_lowest_lengths(dev):
    """Lengths below 0 down to the type's lowest: nothing is visible."""
    kv = paged.PagedKV.empty(1, 4, 1, 64, dev, page=16)
    for t in (kv.k, kv.v, kv.k_scale, kv.v_scale):
        t.fill_(7)
    table = _i32([[0, 1, 2, 3]] * 3, dev)
    for low in (-1, -(1 << 31) + 1, -(1 << 31)):
        for counts in ([1, 1, 1], [2, 0, 90]):
            got = paged.attend(kv, 0, torch.randn(sum(counts), 2, 64, device=dev), table, _i32([low] * 3, dev),
                               q_start=_starts(counts, dev))
            assert not got.any()


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("B", [64, 65, 515, 1100])
def test_many_sequences(dev, B, dt):
    """Batches past what a wave looks at at once, sequences without rows among them: append, attend and their rows."""
    rng = np.random.default_rng(B)
    D, P, G, H = 64, 16, 1, 3
    counts = rng.choice([0, 1, 2, 7], B, p=[0.3, 0.3, 0.3, 0.1])
    counts[-1] = 2
    held = rng.integers(0, 20, B)
    lens = held + counts
    N, cols = int(counts.sum()), 2
    table = rng.permutation(2 * B).reshape(B, cols)
    t, starts = _i32(table, dev), _starts(counts, dev)
    kv, one = (paged.PagedKV.empty(1, 2 * B, G, D, dev, page=P, fmt=FMT["i8"]) for _ in range(2))
    for c in (kv, one):
        for a in (c.k, c.v):
            a.copy_(torch.from_numpy(np.random.default_rng(1).integers(1, 256, tuple(a.shape), np.uint8)))
        c.k_scale.fill_(1e-9), c.v_scale.fill_(1e-9)
    k, v = (torch.from_numpy(rng.standard_normal((N, G, D)).astype(np.float32)).to(DT[dt]).to(dev) for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((N, H, D)).astype(np.float32)).to(DT[dt]).to(dev)
    paged.append(kv, 0, k, v, t, _i32(held, dev), q_start=starts)
    got = paged.attend(kv, 0, q, t, _i32(lens, dev), q_start=starts, max_new=7)
    at = np.concatenate([[0], np.cumsum(counts)])
    for b in [0, 1, B // 2, B - 1] + list(np.flatnonzero(counts)[::max(1, B // 40)]):
        lo, hi = at[b], at[b + 1]
        if lo == hi:
            continue
        only = _starts([int(counts[b])], dev)
        paged.append(one, 0, k[lo:hi], v[lo:hi], t[b:b + 1], _i32([held[b]], dev), q_start=only)
        for p in table[b]:
            assert torch.equal(kv.k[0, p], one.k[0, p]) and torch.equal(kv.v[0, p], one.v[0, p])
            assert torch.equal(kv.k_scale[0, p], one.k_scale[0, p])
        want = paged.attend(one, 0, q[lo:hi], t[b:b + 1], _i32([lens[b]], dev), q_start=only, max_new=7)
        assert torch.equal(got[lo:hi], want), b


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [
    # D, page, G, H, lens, counts, window, sinks: more than 96 query rows for a kv head
    (128, 64, 1, 8, [700, 64, 300], [100, 40, 3], 0, 0),
    (64, 16, 1, 3, [400, 33, 5, 1], [180, 20, 0, 1], 0, 0),
    (128, 32, 2, 24, [500, 90], [90, 9], 64, 5),
    (64, 128, 1, 20, [300, 7], [40, 7], 1, 0),
    (128, 16, 3, 21, [120, 1000, 8], [150, 30, 8], 200, 33),
    (128, 256, 1, 1, [1000], [500], 0, 0),
    (64, 64, 2, 10, [2500], [130], 0, 0),
])
def test_attend_blocks_of_rows(dev, shape, fmt, dt):
    D, P, G, H, lens, counts, window, sinks = shape
    rng = np.random.default_rng(35)
    pages = sum(-(-n // P) for n in lens) + 3
    c = _garbage(rng, pages, G, P, D, fmt)
    table = _table(rng, lens, P, pages)
    _fill(rng, c, table, lens)
    _attend(dev, c, table, lens, counts, H, dt, tail=2, window=window, n_sink=sinks)
