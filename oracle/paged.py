"""Float64 restatement of the paged 8-bit K/V cache and of beam search over it (numpy, loops, no GPU).

A cache is a dict of numpy arrays of one layer: k codes uint8 [pages, G, P, D], v codes uint8 [pages, G, D, P], ks / vs
float32 [pages, G], and ``fmt`` ("i8": value (u - 128) * scale, "e4m3": float8 e4m3fn value * scale)."""
import numpy as np

QMAX = {"i8": 127.0, "e4m3": 448.0}


def code_values(fmt: str) -> np.ndarray:
    """What each of the 256 bytes stands for."""
    u = np.arange(256)
    if fmt == "i8":
        return u - 128.0
    e, m = (u >> 3) & 15, u & 7
    x = np.where(e == 0, m * 2.0 ** -9, (8.0 + m) * 2.0 ** (e - 10.0))
    x = np.where((u & 127) == 127, np.nan, x)
    return np.where(u & 128, -x, x)


def round8(x: np.ndarray, fmt: str) -> np.ndarray:
    """fp32 values -> bytes: the nearest code, ties to the even one, saturating."""
    x = np.asarray(x, dtype=np.float64)
    if fmt == "i8":
        return (np.clip(np.round(x), -127, 127) + 128).astype(np.uint8)
    mag = np.minimum(np.abs(x), 448.0)
    e = np.maximum(np.floor(np.log2(np.maximum(mag, 2.0 ** -20))), -6.0)
    q = np.round(mag / 2.0 ** (e - 3))                     # 0 .. 16 steps of the binade
    e, q = np.where(q == 16, e + 1, e), np.where(q == 16, 8, q)
    byte = np.where(q < 8, q, (e + 7) * 8 + (q - 8)).astype(np.int64)
    return (byte | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def empty(pages: int, G: int, P: int, D: int, fmt: str) -> dict:
    z = 128 if fmt == "i8" else 0
    return dict(k=np.full((pages, G, P, D), z, np.uint8), v=np.full((pages, G, D, P), z, np.uint8),
                ks=np.zeros((pages, G), np.float32), vs=np.zeros((pages, G), np.float32), fmt=fmt)


def rotate(x: np.ndarray, table_row: np.ndarray) -> np.ndarray:
    """x [heads, D] by one row [cos | sin], in float64."""
    h = x.shape[-1] // 2
    c, s = table_row[:h].astype(np.float64), table_row[h:].astype(np.float64)
    a, b = x[:, :h].astype(np.float64), x[:, h:].astype(np.float64)
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def _store(codes, scales, page, g, off, x, fmt):
    """Rows x [n, D] (float32) at tokens off .. of a page, whose tokens before off stay: codes [P, D] view."""
    with np.errstate(over="ignore", invalid="ignore"):
        a = np.float32(np.abs(x).max()) if np.isfinite(x).all() else np.float32(np.nan)
        new = np.float32(a / np.float32(QMAX[fmt]))
    was = scales[page, g]
    if off > 0:
        if np.isnan(was):
            new = np.float32(np.nan)
        elif new > was:
            val = code_values(fmt)[codes[:off]]
            codes[:off] = round8(np.float32(val * np.float64(was) / np.float64(new)), fmt)
        elif not np.isnan(new):
            new = was
    scales[page, g] = new
    if new > 0:
        codes[off:off + len(x)] = round8(np.float32(x.astype(np.float64) / np.float64(new)), fmt)
    else:
        codes[off:off + len(x)] = round8(np.zeros_like(x), fmt)


def append(cache: dict, k, v, table, start, counts, rope=None, q=None):
    """k, v [N, G, D] float32 rows packed by sequence; returns the rotated q (float64) or None.  Rows without a position
    at or above 0 or without a page are skipped."""
    P, G = cache["k"].shape[2], cache["k"].shape[1]
    pages = cache["k"].shape[0]
    qo = None if q is None else q.astype(np.float64).copy()
    row = 0
    for b, n in enumerate(counts):
        todo = {}
        for i in range(n):
            pos = int(start[b]) + i
            if pos < 0:
                continue
            bad = rope is not None and pos >= len(rope)
            kr = k[row + i].astype(np.float64)
            if rope is not None:
                kr = np.full_like(kr, np.nan) if bad else rotate(kr, rope[pos])
            if q is not None and rope is not None:
                qo[row + i] = np.nan if bad else rotate(q[row + i], rope[pos])
            col = pos // P
            page = table[b][col] if col < len(table[b]) else -1
            if 0 <= page < pages:
                todo.setdefault((page, col), []).append((pos % P, kr.astype(np.float32), v[row + i].astype(np.float32)))
        for (page, _), toks in todo.items():
            off = toks[0][0]
            for g in range(G):
                _store(cache["k"][page, g], cache["ks"], page, g, off, np.stack([t[1][g] for t in toks]), cache["fmt"])
                _store(cache["v"][page, g].T, cache["vs"], page, g, off, np.stack([t[2][g] for t in toks]), cache["fmt"])
        row += n
    return qo


def rows(cache: dict, table_row, lo: int, hi: int):
    """(k, v [G, hi - lo, D] float64, present [hi - lo])."""
    P, G, D = cache["k"].shape[2], cache["k"].shape[1], cache["k"].shape[3]
    val = code_values(cache["fmt"])
    k, v = np.zeros((G, hi - lo, D)), np.zeros((G, hi - lo, D))
    ok = np.zeros(hi - lo, bool)
    for i, pos in enumerate(range(lo, hi)):
        if pos < 0 or pos // P >= len(table_row):
            continue
        page = table_row[pos // P]
        if not 0 <= page < cache["k"].shape[0]:
            continue
        ok[i] = True
        k[:, i] = val[cache["k"][page, :, pos % P]] * cache["ks"][page][:, None].astype(np.float64)
        v[:, i] = val[cache["v"][page, :, :, pos % P]] * cache["vs"][page][:, None].astype(np.float64)
    return k, v, ok


def attend(cache: dict, q, table, lens, counts, window=0, n_sink=0, scale=None):
    """q [N, H, D] -> (out [N, H, D], size [N, H, D], reach [N, H], n [N]): size = sum p |v|, reach the largest
    |scale| sum |q||k| over the visible keys, n their number (what error bounds are made of)."""
    N, H, D = q.shape
    G = cache["k"].shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, size, reach, seen = np.zeros((N, H, D)), np.zeros((N, H, D)), np.zeros((N, H)), np.zeros(N, int)
    row = 0
    for b, n in enumerate(counts):
        k, v, ok = rows(cache, table[b], 0, max(0, int(lens[b])))
        j = np.arange(len(ok))
        for t in range(n):
            p = int(lens[b]) - n + t
            see = ok & (j <= p)
            if window > 0:
                see &= (j > p - window) | (j < n_sink)
            seen[row + t] = see.sum()
            if not see.any():
                continue
            for h in range(H):
                g = h // (H // G)
                kk, vv, qq = k[g][see], v[g][see], q[row + t, h].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    s = scale * (kk @ qq)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[row + t, h], size[row + t, h] = w @ vv, w @ np.abs(vv)
                    reach[row + t, h] = abs(scale) * (np.abs(kk) @ np.abs(qq)).max()
        row += n
    return out, size, reach, seen


def attend_bound(out, size, reach, seen, D: int, bf16: bool) -> np.ndarray:
    """What an attention with exact codes and fp32 sums may be off by.  Scores: D products summed in fp32 and a query held
    to 2^-22, so reach * (D + 4) 2^-24 each, twice in a quotient of sums; exp2 and the probability's pieces 2^-21; the
    sums over keys take a rounding per 16 keys and 64 more.  bf16 rows: probabilities rounded to fp16 (2^-11) and the
    result to bf16 (half a step, 2^-8)."""
    ds = reach[..., None] * (D + 4) * 2.0 ** -24
    tol = size * (2 * np.expm1(ds) + 2.0 ** -20 + (seen[:, None, None] / 16 + 64) * 2.0 ** -24)
    if bf16:
        tol = tol + 2.0 ** -11 * size + 2.0 ** -8 * np.abs(out)
    return tol + 1e-37


def reorder(table, lens, parents, P: int):
    """(table, lens, [(source page, target page)]) after beams of groups follow `parents` [B][K]; lists of lists."""
    new_table, new_lens, copies = [], [], []
    for b, par in enumerate(parents):
        K = len(par)
        par = [p if 0 <= p < K else i for i, p in enumerate(par)]
        row = lambda i: table[b * K + i]  # noqa: E731
        at = [max(0, int(lens[b * K + i])) // P for i in range(K)]
        tail = [row(i)[at[i]] if at[i] < len(row(i)) else -1 for i in range(K)]
        free, taken = [i for i in range(K) if i not in par], set()
        for i, p in enumerate(par):
            page = tail[p]
            if p in taken:
                page = tail[free.pop(0)]
                if int(lens[b * K + p]) % P:
                    copies.append((tail[p], page))
            taken.add(p)
            new_table.append([row(p)[j] if j < at[p] else page if j == at[p] else row(i)[j] if j > at[i] else -1
                              for j in range(len(row(i)))])
            new_lens.append(int(lens[b * K + p]))
    return new_table, new_lens, copies


def beam_select(logits, scores, done=None, eos=-1):
    """logits [B * K, V], scores [B, K] -> (scores, parents, tokens, done), float64 totals."""
    B, K = scores.shape
    V = logits.shape[1]
    out = [np.full((B, K), -np.inf), np.tile(np.arange(K), (B, 1)), np.full((B, K), -1), np.ones((B, K), int)]
    for b in range(B):
        cand = []
        for k in range(K):
            if done is not None and done[b, k]:
                total = np.full(V, -np.inf)
                total[eos] = scores[b, k]
            else:
                x = logits[b * K + k].astype(np.float64)
                with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
                    m = x.max()
                    total = scores[b, k] + (x - (np.log(np.exp(x - m).sum()) + m))
            ok = np.flatnonzero(total > -np.inf)
            ok = ok[np.argsort(-total[ok], kind="stable")][:K]
            cand += [(-total[i], k * V + i) for i in ok]
        for i, (t, f) in enumerate(sorted(cand)[:K]):
            out[0][b, i], out[1][b, i], out[2][b, i] = -t, f // V, f % V
            out[3][b, i] = int((done is not None and done[b, f // V] != 0) or f % V == eos)
    return out
