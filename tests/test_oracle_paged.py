"""The oracle of the paged 8-bit cache against independent facts (no GPU): the e4m3 rounding against torch's float8
conversion over every binade and tie, what an append may be off by, the attention against a dense softmax, the
reordering's ownership of pages, beam selection against a full sort; and the host-side refusals of the C entry points."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged as op
from vault_amd import _lib as L


def test_e4m3_codes_are_the_float8_ones():
    u = torch.arange(256, dtype=torch.uint8)
    want = u.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(op.code_values("e4m3"), want, equal_nan=True)
    val = np.sort(want[np.isfinite(want) & (want >= 0)])
    val = np.unique(val)
    mid = (val[1:] + val[:-1]) / 2                                   # every tie
    x = np.concatenate([val, mid, np.nextafter(mid.astype(np.float32), np.float32(0)).astype(np.float64),
                        np.nextafter(mid.astype(np.float32), np.float32(1e9)).astype(np.float64)])
    x = np.concatenate([x, -x]).astype(np.float32)
    got = op.round8(x, "e4m3")
    assert np.array_equal(got, torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_append_is_within_half_a_step(fmt):
    """A page filled in four runs: each value within half a step of its code plus, for every time its scale grew, half a
    step more."""
    rng = np.random.default_rng(1)
    c = op.empty(3, 2, 16, 64, fmt)
    x = rng.standard_normal((16, 2, 64)).astype(np.float32)
    x[8:] *= 3
    at, grown = 0, 0
    for n in (5, 3, 4, 4):
        before = c["ks"][1].copy()
        op.append(c, x[at:at + n], x[at:at + n], [[1]], [at], [n])
        grown += int((c["ks"][1] > before).any())
        at += n
    k, v, ok = op.rows(c, [1], 0, 16)
    assert ok.all() and np.array_equal(k, v)
    step = 0.5 / 127 if fmt == "i8" else 2.0 ** -4
    big = np.abs(x).max((0, 2))[:, None, None]
    tol = step * big if fmt == "i8" else step * np.abs(x.transpose(1, 0, 2)) + 2.0 ** -10 * big / 448
    assert (np.abs(k - x.transpose(1, 0, 2)) <= tol * grown * (1 + 1e-6)).all()


def test_attend_is_the_dense_softmax():
    rng = np.random.default_rng(2)
    c = op.empty(9, 2, 16, 64, "i8")
    n = 70
    x = rng.standard_normal((n, 2, 64)).astype(np.float32)
    y = rng.standard_normal((n, 2, 64)).astype(np.float32)
    table = [[4, 1, 7, 0, 8]]
    op.append(c, x, y, table, [0], [n])
    q = rng.standard_normal((3, 4, 64)).astype(np.float32)
    out, size, reach, seen = op.attend(c, q, table, [n], [3], window=20, n_sink=5)
    k, v, _ = op.rows(c, table[0], 0, n)
    qt = torch.from_numpy(q).double().transpose(0, 1)
    kt, vt = (torch.from_numpy(t).repeat_interleave(2, 0) for t in (k, v))
    p = torch.arange(n - 3, n)[:, None]
    j = torch.arange(n)[None]
    see = (j <= p) & ((j > p - 20) | (j < 5))
    a = (qt @ kt.transpose(1, 2)) / 8.0
    ref = torch.softmax(a.masked_fill(~see, -torch.inf), -1) @ vt
    assert np.abs(out - ref.transpose(0, 1).numpy()).max() < 1e-12
    assert list(seen) == [25, 25, 25]


def test_reorder_keeps_one_owner_of_every_open_page():
    rng = np.random.default_rng(3)
    for _ in range(50):
        B, K, P = rng.integers(1, 4), int(rng.integers(1, 9)), 16
        length = rng.integers(0, 100, B)
        lens = np.repeat(length, K)
        table = np.arange(B * K * 8).reshape(B * K, 8).tolist()
        par = rng.integers(0, K, (B, K)).tolist()
        t, n, copies = op.reorder(table, lens, par, P)
        tails = [t[r][n[r] // P] for r in range(B * K)]
        assert len(set(tails)) == B * K
        assert not {s for s, _ in copies} & {d for _, d in copies}
        for b in range(B):
            for i in range(K):
                p = par[b][i]
                at = n[b * K + i] // P
                assert t[b * K + i][:at] == table[b * K + p][:at] and t[b * K + i][at + 1:] == table[b * K + i][at + 1:]
                own = table[b * K + p][at]
                assert tails[b * K + i] == own or n[b * K + i] % P == 0 or (own, tails[b * K + i]) in copies


def test_beam_select_is_the_full_sort():
    rng = np.random.default_rng(4)
    x, s = rng.standard_normal((6, 50)).astype(np.float32), rng.standard_normal((2, 3)).astype(np.float32)
    done = np.array([[0, 1, 0], [0, 0, 0]])
    got = op.beam_select(x, s, done, eos=7)
    lp = torch.log_softmax(torch.from_numpy(x).double(), -1).numpy().reshape(2, 3, 50) + s[..., None]
    lp[0, 1] = -np.inf
    lp[0, 1, 7] = s[0, 1]
    for b in range(2):
        at = np.argsort(-lp[b].ravel(), kind="stable")[:3]
        assert np.array_equal(got[1][b], at // 50) and np.array_equal(got[2][b], at % 50)
        assert np.abs(got[0][b] - lp[b].ravel()[at]).max() < 1e-12


# ------------------------------------------------------------------ refusals (no HIP call is reached)

p = 1 << 20


def _kv(**kw):
    d = dict(fmt=L.I8, k=p, v=p, k_scale=p, v_scale=p, n_layers=2, n_pages=10, G=2, page=64, D=128,
             layer_stride=10 * 2 * 64 * 128, scale_layer_stride=20)
    d.update(kw)
    return L.PagedKV(*[d[f] for f, _ in L.PagedKV._fields_])


CACHE = [(dict(fmt=3), -5), (dict(k=None), -31), (dict(v_scale=None), -31), (dict(D=96), -7), (dict(page=48), -7),
         (dict(page=8), -7), (dict(G=0), -1), (dict(n_pages=0), -1), (dict(layer_stride=64), -1), (dict(k=p + 8), -11),
         (dict(layer_stride=10 * 2 * 64 * 128 + 8), -11), (dict(n_pages=1 << 31, layer_stride=1 << 60,
                                                                  scale_layer_stride=1 << 40), -10)]


@pytest.mark.parametrize("kw,code", CACHE)
def test_refused_caches(kw, code):
    lib, kv = L.load(), _kv(**kw)
    r = C.byref(kv)
    assert lib.vgx_paged_append(r, 0, L.F32, p, 256, p, 256, 1, p, 4, 4, p, None, 1, None, 0, 0, None, 0, None, 0, 0,
                                None) == code
    assert lib.vgx_paged_attn(r, 0, L.F32, p, 1536, p, 1536, 1, 12, p, 4, 4, p, None, 1, 1, 256, 0, 0, 1.0, p, 1 << 30,
                              None) == code
    assert lib.vgx_paged_read(r, L.F32, p, 4, 4, p, p, 1, 5, p, p, None) == code
    assert lib.vgx_paged_reorder(r, p, 4, 4, p, p, 1, 2, p + 64, 4, p + 64, None) == code


def test_refused_appends():
    lib, kv = L.load(), _kv()
    base = dict(layer=0, dtype=L.F32, k=p, ldk=256, v=p, ldv=256, N=3, table=p, ldt=4, cols=4, start=p, q_start=p, B=2,
                rope=p, rope_ld=128, rope_rows=9, q=p, ldq=1536, q_out=p, ldqo=1536, H=12)

    def rc(**kw):
        return lib.vgx_paged_append(C.byref(kv), *dict(base, **kw).values(), None)

    for kw, code in [(dict(layer=2), -1), (dict(layer=-1), -1), (dict(dtype=L.F16), -5), (dict(q_start=None), -1),
                     (dict(N=-1), -1), (dict(k=None), -31), (dict(table=None), -31), (dict(start=None), -31),
                     (dict(ldk=255), -1), (dict(ldk=257), -11), (dict(k=p + 4), -11), (dict(ldt=3), -1), (dict(cols=0), -1),
                     (dict(rope_ld=64), -1), (dict(rope=p + 4), -11), (dict(H=0), -1), (dict(q_out=None), -31),
                     (dict(ldq=1535), -1), (dict(N=1 << 31), -10)]:
        assert rc(**kw) == code, kw
    assert rc(N=0) == 0 and rc(B=0) == 0


def test_refused_attention():
    lib, kv = L.load(), _kv()
    base = dict(layer=0, dtype=L.F32, q=p, ldq=1536, out=p, ldo=1536, N=3, H=12, table=p, ldt=4, cols=4, lens=p, q_start=p,
                B=2, max_new=2, max_keys=256, window=0, n_sink=0, scale=1.0, ws=p, ws_bytes=1 << 30)

    def rc(**kw):
        return lib.vgx_paged_attn(C.byref(kv), *dict(base, **kw).values(), None)

    for kw, code in [(dict(layer=2), -1), (dict(dtype=L.Q8_0), -5), (dict(q_start=None), -1), (dict(q=None), -31),
                     (dict(out=None), -31), (dict(lens=None), -31), (dict(table=None), -31), (dict(H=13), -7),
                     (dict(H=0), -1), (dict(ldq=1535), -1), (dict(ldo=1537), -11), (dict(q=p + 4), -11), (dict(ldt=1), -1),
                     (dict(window=-1), -1), (dict(n_sink=-1), -1), (dict(max_keys=-1), -1), (dict(max_new=-1), -1),
                     (dict(cols=1 << 25, ldt=1 << 25), -10), (dict(N=1 << 31), -10)]:
        assert rc(**kw) == code, kw
    big = dict(max_keys=1 << 20, cols=1 << 14, ldt=1 << 14)
    assert rc(**big, ws=None) == -8 and rc(**big, ws_bytes=64) == -8 and rc(**big, ws=p + 4) == -8
    assert rc(N=0) == 0 and rc(B=0) == 0
    bytes_of = lib.vgx_paged_attn_workspace_bytes
    assert bytes_of(3, 2, 12, 2, 96, 2, 256, 0, 0) == -7 and bytes_of(3, 2, 12, 5, 64, 2, 256, 0, 0) == -7
    assert bytes_of(0, 0, 12, 2, 64, 0, 256, 0, 0) == 0


def test_refused_reads_and_reorders():
    lib, kv = L.load(), _kv()
    rd = dict(dtype=L.F32, table=p, ldt=4, cols=4, first=p, lens=p, B=1, n=5, k=p, v=p)
    for kw, code in [(dict(dtype=L.F16), -5), (dict(first=None), -31), (dict(k=None), -31), (dict(n=-1), -1),
                     (dict(v=p + 8), -11), (dict(B=40000), -10), (dict(ldt=3), -1)]:
        assert lib.vgx_paged_read(C.byref(kv), *dict(rd, **kw).values(), None) == code, kw
    assert lib.vgx_paged_read(C.byref(kv), *dict(rd, n=0).values(), None) == 0
    ro = dict(table=p, ldt=4, cols=4, lens=p, parents=p, groups=1, K=2, to=p + 64, ldo=4, lo=p + 64)
    for kw, code in [(dict(K=0), -1), (dict(K=65), -10), (dict(groups=-1), -1), (dict(parents=None), -31), (dict(to=p), -31),
                     (dict(lo=p), -31), (dict(ldo=3), -1), (dict(lens=None), -31)]:
        assert lib.vgx_paged_reorder(C.byref(kv), *dict(ro, **kw).values(), None) == code, kw
    assert lib.vgx_paged_reorder(C.byref(kv), *dict(ro, groups=0).values(), None) == 0


def test_refused_selections():
    lib = L.load()
    base = dict(logits=p, ld=100, groups=2, K=3, V=100, scores=p, done=p, eos=5, so=p, parents=p, tokens=p, do=p, ws=p,
                ws_bytes=1 << 20)
    for kw, code in [(dict(logits=None), -31), (dict(scores=None), -31), (dict(tokens=None), -31), (dict(ld=99), -1),
                     (dict(eos=100), -1), (dict(eos=-1), -31), (dict(K=0), -1), (dict(K=65), -10), (dict(V=(1 << 19) + 1), -10),
                     (dict(groups=-1), -1), (dict(groups=40000), -10), (dict(ws=None), -8), (dict(ws_bytes=8), -8),
                     (dict(ws=p + 8), -8)]:
        assert lib.vgx_beam_select(*dict(base, **kw).values(), None) == code, kw
    assert lib.vgx_beam_select(*dict(base, groups=0).values(), None) == 0
    assert lib.vgx_beam_select_workspace_bytes(1, 0, 5) == -1


def test_refused_tickets():
    lib, kv = L.load(), _kv()
    base = dict(layer=0, dtype=L.F32, q=p, ldq=1536, out=p, ldo=1536, N=3, H=12, table=p, ldt=4, cols=4, lens=p, q_start=p,
                B=2, max_new=2, max_keys=256, window=0, n_sink=0, scale=1.0, ws=p, ws_bytes=1 << 30, tickets=p, n=64)
    for kw, code in [(dict(n=-1), -1), (dict(tickets=p + 2), -11), (dict(out=None), -31), (dict(H=13), -7), (dict(ldq=1), -1)]:
        assert lib.vgx_paged_attn_tickets(C.byref(kv), *dict(base, **kw).values(), None) == code, kw
    assert lib.vgx_paged_attn_tickets(C.byref(kv), *dict(base, N=0).values(), None) == 0


def test_refused_sizes():
    """Launches of 2^32 threads and more, and rows whose number does not fit 32 bits."""
    lib, kv = L.load(), C.byref(_kv())
    n, wide = 1 << 29, 1 << 20
    bytes_of = lib.vgx_paged_attn_workspace_bytes
    assert bytes_of(n, 1, 8, 2, 64, n, 64, 0, 0) == -10 and bytes_of(n, 1, 4, 2, 64, n, 64, 0, 0) >= 0
    assert lib.vgx_paged_attn(kv, 0, L.BF16, p, 1536, p, 1536, 1 << 24, 12, p, 4, 4, p, None, 1 << 24, 1, 64, 0, 0, 1.0, p,
                              1 << 62, None) == -10
    assert lib.vgx_paged_append(kv, 0, L.F32, p, 256, p, 256, 1 << 24, p, 4, 4, p, None, 1 << 24, None, 0, 0, None, 0, None,
                                0, 0, None) == -10
    assert lib.vgx_paged_read(kv, L.F32, p, 4, 4, p, p, 1 << 62, 5, p, p, None) == -10
    small = C.byref(_kv(page=16))
    assert lib.vgx_paged_read(small, L.F32, p, 4, 4, p, p, 1, 1 << 28, p, p, None) == -10
    for groups in (wide, 1 << 24, 1 << 62):
        assert lib.vgx_paged_reorder(kv, p, 4, 4, p, p, groups, 64, p + 64, 4, p + 64, None) == -10
