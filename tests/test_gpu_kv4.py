"""GPU parity of attention over 4-bit keys and values against plain 64-bit forms (kvref.py).

Bars, by the roundings that can meet (u = 2^-24, half an f32 step; h = 2^-8, half a bf16 step):
- norm + rotation: the f32 sum of squares of D <= 256 terms runs in chains of at most 24 and a
  tree of 5, halved by the root (15 u), then quotient, root, reciprocal and two products (5 u),
  the sine and cosine (2 u) and the turn (3 u): 25 u of the magnitudes that meet, 32 allowed;
  bf16 rounds once more (h of the value).
- cache contents: equal, codes and scales.
- attention: an exponent (log2 units) is off by at most D u of sum |q k| (D additions) and 2 u
  of itself, a probability by ln 2 of that and 2 u, in numerator and denominator; the sums of n
  products add (n + 64) u of sum P |v|.  bf16: probabilities as two terms (h^2 / 2 of sum P |v|)
  and the output's own h.
- attention of more than 16 rows of a kv head (maybe f16 operands, f = 2^-11 half an f16 step, eps / 2):
  bf16 calls round a probability (f), a key's int4 code times its scale (f: an exponent is off by
  f of sum |q k|), a value's int4 scale and its product with a code (2 f of sum P |v|); MXFP4 is
  exact.  f32 calls hold each rounded operand in two terms (f^2 = 4 u of it, twice a product)
  and leave out the product of the second two (f^2): 12 u of sum |q k| and of sum P |v|.  So do
  the exponents of calls that collect weights, whose own sums take exact products.  Below
  2^-14 an f16 holds steps of 2^-24: probabilities are carried so that the largest is 2^7 (bf16;
  2^14 f32) or more, so each of n is off by 2^-32 (2^-39) of the row's sum at least, and a value
  by 2^-25 of 2^14 for the largest of its tile: n 2^-31 (2^-38) of the largest |v| beside the rest.
- the 2-norm: errors of independent roundings grow as their root: exponents 4 u of the largest
  one, 16 u beside; f16 keys' f of the root of the sum of (q k)^2, twice for the denominator's
  share; f16 values and probabilities 3 f.
- eviction: indices, codes, scales and scores equal.
"""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import kvref

pytestmark = pytest.mark.gpu

U, H = 2.0 ** -24, 2.0 ** -8
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def host(t):
    return t.float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def dt(hip, name):
    return {"f32": hip.F32, "bf16": hip.BF16}[name]


def make_cache(rng, fmt, n_kv, D, page, n_pages, score=True):
    """A host cache of quantized normal keys (channels of unlike size) and values."""
    shape = (n_pages, n_kv, page, D)
    chan = np.exp(0.5 * rng.standard_normal((n_kv, 1, D)))
    k, ks = kvref.quantize(fmt, rng.standard_normal(shape) * chan)
    v, vs = kvref.quantize(fmt, rng.standard_normal(shape) * 0.5)
    w = np.exp(rng.standard_normal(shape[:3])).astype(np.float32) if score else None
    return dict(fmt=fmt, page=page, k=k, ks=ks, v=v, vs=vs, score=w)


def to_device(hip, c):
    arr = {n: dev(c[n]) for n in ("k", "ks", "v", "vs")}
    arr["score"] = None if c["score"] is None else dev(c["score"])
    n_kv, D = c["k"].shape[1], c["k"].shape[3] * 2
    return arr, hip.KV4(c["fmt"], n_kv, D, c["page"], arr["k"], arr["ks"], arr["v"], arr["vs"],
                        arr["score"])


def tables(rng, lens, page, n_pages, extra=1):
    per = max(-(-max(max(lens), 1) // page) + extra, 1)
    return rng.permutation(n_pages)[:len(lens) * per].reshape(len(lens), per).astype(np.int32)


def starts(news):
    return np.concatenate(([0], np.cumsum(news))).astype(np.int32)


# ---- norms and rotation --------------------------------------------------------------------


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,inter,dtype,far", [
    (1, 1, 1, 64, 64, False, "f32", 100), (3, 16, 16, 128, 128, False, "f32", 4096),
    (5, 7, 3, 128, 32, True, "bf16", 1 << 20), (2, 9, 1, 192, 192, False, "f32", 1 << 24),
    (4, 5, 2, 192, 48, False, "bf16", 1 << 20), (3, 6, 2, 192, 96, True, "f32", 1000),
    (7, 12, 4, 256, 256, False, "bf16", 1 << 18), (2, 3, 1, 256, 16, True, "f32", (1 << 31) - 1),
    (130, 24, 8, 64, 16, False, "bf16", 70000), (1, 64, 8, 128, 64, False, "f32", 5),
    (2, 0, 5, 128, 128, False, "f32", 9), (2, 5, 0, 64, 32, True, "f32", 9)])
def test_norm_rope(hip, T, Hq, Hkv, D, rot, inter, dtype, far):
    """Odd head counts, every head size, partial rotation, far positions, rows of a fused
    projection, queries or keys alone; columns beside the outputs stay as they are."""
    rng = np.random.default_rng(T + Hq + D + rot)
    heads = Hq + 2 * Hkv
    x = dev(rng.standard_normal((T, heads, D)).astype(np.float32) *
            np.exp(rng.standard_normal((T, heads, 1))).astype(np.float32), TYPES[dtype])
    w = [dev((1 + 0.3 * rng.standard_normal(D)).astype(np.float32)) for _ in range(2)]
    pos = rng.integers(0, far, T).astype(np.int32)
    pos[0] = far - 1
    freq = 10000.0 ** (-2.0 * np.arange(rot // 2) / rot)
    out = torch.full((T, Hq + Hkv + 1, D), 7.0, device="cuda", dtype=TYPES[dtype])
    row, orow = heads * D, (Hq + Hkv + 1) * D
    hip.qk_norm_rope_dev(dt(hip, dtype), T, D, x, row, Hq, out, orow, x[:, Hq:], row, Hkv,
                         out[:, Hq:], orow, w[0], w[1], 1e-6, dev(pos), dev(freq), rot, inter)
    torch.cuda.synchronize()
    got = host(out)
    assert (got[:, -1] == 7.0).all()
    for lo, n, wi in ((0, Hq, w[0]), (Hq, Hkv, w[1])):
        if n:
            y, size = kvref.norm_rope(host(x)[:, lo:lo + n], host(wi), 1e-6, pos, freq, rot, inter)
            tol = 32 * U * size + (H * np.abs(y) if dtype == "bf16" else 0)
            assert (np.abs(got[:, lo:lo + n] - y) <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_rope_in_place_without_weights_or_rotation(hip, dtype):
    rng = np.random.default_rng(5)
    x = dev(rng.standard_normal((9, 11, 128)).astype(np.float32), TYPES[dtype])
    y = x.clone()
    k = y[:, 8:]
    hip.qk_norm_rope_dev(dt(hip, dtype), 9, 128, y, 11 * 128, 8, y, 11 * 128, k, 11 * 128, 3, k,
                         11 * 128, None, None, 1e-5, None, None, 0)
    torch.cuda.synchronize()
    exp, size = kvref.norm_rope(host(x), None, 1e-5, None, None, 0, False)
    assert (np.abs(host(y) - exp) <= 32 * U * size + (H * np.abs(exp) if dtype == "bf16" else 0)).all()


# ---- append and read -----------------------------------------------------------------------


@pytest.mark.parametrize("fmt", [4, 7])
@pytest.mark.parametrize("dtype,n_kv,D,page,lens,news", [
    ("f32", 1, 64, 16, [1], [1]), ("bf16", 3, 128, 48, [5, 60, 97], [5, 1, 50]),
    ("f32", 16, 128, 64, [100, 1, 64, 65], [1, 1, 1, 1]), ("f32", 5, 192, 16, [33, 20], [33, 3]),
    ("bf16", 2, 256, 32, [70, 0, 31], [66, 0, 31]), ("f32", 2, 64, 16, [3, 2], [5, 2])])
def test_append_and_read(hip, fmt, dtype, n_kv, D, page, lens, news):
    """Codes and scales equal to the definition's, other slots untouched, scores cleared, strided
    rows, values of every size: zeros, ties, denormals, infinities, NaN; more rows than tokens."""
    rng = np.random.default_rng(fmt + D + page + len(lens))
    n_pages = 4 * len(lens) + sum(-(-n // page) for n in lens)
    c = make_cache(rng, fmt, n_kv, D, page, n_pages)
    arr, cache = to_device(hip, c)
    tab, qs, T = tables(rng, lens, page, n_pages), starts(news), sum(news)
    x = (rng.standard_normal((2, T + 2, n_kv + 1, D)) *
         np.exp(3 * rng.standard_normal((2, T + 2, n_kv + 1, 1)))).astype(np.float32)
    x[0, 0, 0, :64] = 0
    x[1, 0, 0, 3], x[1, 0, 0, 9] = np.inf, np.nan
    x[0, T - 1, 0, 1], x[1, T - 1, 0, 2] = -np.inf, 1e-42
    x[1, T - 1, 0, 32:64] = 1e-38
    x[0, T // 2, 0, :64] = np.float32(7 * 0.25) * np.repeat(np.arange(-8, 8), 4) / 8  # ties
    x[1, T // 2, 0, :64] = np.resize(np.array([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -5]), 64)
    xd = dev(x, TYPES[dtype])
    row = (n_kv + 1) * D
    hip.kv4_append_dev(cache, dt(hip, dtype), xd[0], row, xd[1], row, T + 2, dev(qs),
                       dev(np.array(lens, np.int32)), dev(tab), len(lens), tab.shape[1])
    torch.cuda.synchronize()
    xh = host(xd)
    exp = {n: c[n].copy() for n in ("k", "ks", "v", "vs", "score")}
    for r, b, t in kvref.rows_of(qs, lens):
        at = kvref.place(c, tab[b], t)
        if at:
            for i, n in enumerate("kv"):
                exp[n][at[0], :, at[1]], exp[n + "s"][at[0], :, at[1]] = \
                    kvref.quantize(fmt, xh[i, r, :n_kv])
            exp["score"][at[0], :, at[1]] = 0
    for n in exp:
        assert np.array_equal(host(arr[n]), exp[n]), n
    for out_type in ("f32", "bf16"):
        k, v = (torch.full((T + 2, n_kv, D), 3.0, device="cuda", dtype=TYPES[out_type])
                for _ in range(2))
        hip.kv4_read_dev(cache, dt(hip, out_type), k, v, T + 2, dev(qs),
                         dev(np.array(lens, np.int32)), dev(tab), len(lens), tab.shape[1])
        torch.cuda.synchronize()
        assert (host(k)[T:] == 3).all() and (host(v)[T:] == 3).all()
        for r, b, t in kvref.rows_of(qs, lens):
            at = kvref.place(c, tab[b], t)
            for got, n in ((k, "k"), (v, "v")):
                y = kvref.values(fmt, exp[n][at[0], :, at[1]], exp[n + "s"][at[0], :, at[1]]) \
                    if at else np.zeros((n_kv, D))
                y = torch.from_numpy(y).float().to(TYPES[out_type])
                assert torch.equal(got[r].cpu(), y)


@pytest.mark.parametrize("n_seq", [64, 65, 129, 5000])
def test_append_finds_its_sequence(hip, n_seq):
    """Many sequences, some with no new token, several or fewer tokens than rows; rows ahead of
    the first sequence and behind the last."""
    rng = np.random.default_rng(n_seq)
    news = rng.integers(0, 4, n_seq)
    news[[0, n_seq // 2, n_seq - 1]] = 0, 3, 1
    lens = news + rng.integers(-1, 3, n_seq).clip(-news)
    qs = (starts(news) + 2).astype(np.int32)
    T = int(qs[-1]) + 3
    c = make_cache(rng, 7, 1, 64, 16, n_seq)
    arr, cache = to_device(hip, c)
    tab = rng.permutation(n_seq).reshape(-1, 1).astype(np.int32)
    x = rng.standard_normal((2, T, 1, 64)).astype(np.float32)
    xd = dev(x)
    args = (T, dev(qs), dev(lens.astype(np.int32)), dev(tab), n_seq, 1)
    hip.kv4_append_dev(cache, hip.F32, xd[0], 64, xd[1], 64, *args)
    torch.cuda.synchronize()
    codes, scales = kvref.quantize(7, x)
    exp = {n: c[n].copy() for n in ("k", "ks", "v", "vs")}
    for r, b, t in kvref.rows_of(qs, lens):
        if t >= 0:
            for i, n in enumerate("kv"):
                exp[n][tab[b, 0], 0, t] = codes[i, r, 0]
                exp[n + "s"][tab[b, 0], 0, t] = scales[i, r, 0]
    for n in exp:
        assert np.array_equal(host(arr[n]), exp[n]), n


@pytest.mark.parametrize("fmt", [4, 7])
def test_append_rounds_exactly(hip, fmt):
    """Values on and next to every border of a code, at scales whose reciprocal rounds: each takes
    its own side, as the real quotient does."""
    rng = np.random.default_rng(fmt)
    T, D = 600, 64
    top = np.exp(rng.uniform(-60, 60, (T, 1))).astype(np.float32)
    s = top * np.float32(1 / 7) if fmt == 4 else np.float32(2.0) ** np.ceil(np.log2(top / 6))
    mids = np.arange(-6.5, 7) if fmt == 4 else \
        np.concatenate(((kvref.GRID[1:] + kvref.GRID[:-1]) / 2, -(kvref.GRID[1:] + kvref.GRID[:-1]) / 2))
    x = (np.resize(mids, (T, D)) * s.astype(np.float64)).astype(np.float32)
    x = np.nextafter(x, np.float32(np.inf) * rng.choice([-1, 1], x.shape), dtype=np.float32) \
        if fmt == 4 else np.where(rng.random(x.shape) < 0.5, x, np.nextafter(x, np.float32(0)))
    x = np.clip(x, -top, top).astype(np.float32)
    x[:, 0] = x[:, 33] = top[:, 0]
    c = make_cache(rng, fmt, 1, D, 16, 40)
    arr, cache = to_device(hip, c)
    tab = np.arange(38, dtype=np.int32)[None]
    xd = dev(x[:, None])
    hip.kv4_append_dev(cache, hip.F32, xd, D, xd, D, T, dev(starts([T])),
                       dev(np.array([T], np.int32)), dev(tab), 1, 38)
    torch.cuda.synchronize()
    codes, scales = kvref.quantize(fmt, x)
    assert np.array_equal(host(arr["k"])[:38, 0].reshape(-1, D // 2)[:T], codes)
    assert np.array_equal(host(arr["vs"])[:38, 0].reshape(608, -1)[:T], scales)
    if fmt == 7:  # the activation quantizer's codes
        cd, sd = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in (T * D // 2, T * D // 32))
        hip.quantize_mxfp4(xd, T, D, cd, sd)
        assert np.array_equal(host(cd).reshape(T, -1), codes)
        assert np.array_equal(host(sd).reshape(T, -1), scales)


# ---- attention -----------------------------------------------------------------------------


def run_attention(hip, cache, dtype, q, q_start, lens, tab, max_new, max_len, scale, window=0,
                  weights=0, fill=5.0, stream=None):
    """q: device [T, >= Hq, D] view; -> device out (rows of no sequence keep `fill`)."""
    T, Hq, D = q.shape
    n = hip.kv4_attention_work(cache.n_kv, D, Hq, T, len(lens), max_new, max_len, weights)
    work = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    out = torch.full((T, Hq, D), fill, device="cuda", dtype=TYPES[dtype])
    hip.kv4_attention_dev(cache, dt(hip, dtype), q, q.stride(0), Hq, T, q_start, lens, tab,
                          len(lens), tab.shape[1], max_new, max_len, scale, window, weights, out,
                          work, n, stream)
    torch.cuda.synchronize()
    return out


def check_attention(c, q, got, score, q_start, lens, tab, scale, window, weights, dtype,
                    fill=5.0, forced=False):
    D = q.shape[2]
    out, mag, (top, sums, root), exp_score = kvref.attention(c, q, q_start, lens, tab, scale,
                                                             window, weights)
    own = ~np.isnan(out).all((1, 2))
    assert (got[~own] == fill).all()
    prompt = int(np.max(np.diff(q_start))) * (q.shape[1] // c["k"].shape[1]) > 16 or forced
    f = 2.0 ** -11 if prompt else 0.0
    k_off = (f if c["fmt"] == 4 else 0) if dtype == "bf16" else 12 * U * prompt
    v_off = (3 * f if c["fmt"] == 4 else f) if dtype == "bf16" else 12 * U * prompt
    w_off = 12 * U * prompt
    if weights:
        k_off = w_off
    p_off = 2 * (np.log(2) * (U * (D * sums + 2 * top) + k_off * sums) + 2 * U)
    tol = mag * (p_off + v_off + (max(max(lens), 1) + 64) * U)
    if prompt:
        vs = c["vs"].astype(np.float64) if c["fmt"] == 4 else 2.0 ** (c["vs"] - 127.0)
        tol = tol + max(lens) * 2.0 ** (-31 if dtype == "bf16" else -38) * 8 * np.abs(vs).max()
    if dtype == "bf16":
        tol = tol + H * np.abs(out) + H * H / 2 * mag
    assert (np.abs(got - out)[own] <= tol[own] + 1e-37).all()
    norm = (4 * top + 16) * U + (H if dtype == "bf16" else 0) + 2 * k_off * root + v_off
    err = np.linalg.norm(got[own] - out[own]) / max(np.linalg.norm(out[own]), 1e-30)
    assert err <= norm or not out[own].any()
    if weights:
        most = np.maximum(np.abs(exp_score), 1.0)
        assert (np.abs(score - exp_score) <= most * (p_off + 300 * U)).all()
        assert np.linalg.norm(score - exp_score) <= (norm_of(top) + 2 * k_off * root) * np.linalg.norm(exp_score)
    return err


def norm_of(top):
    return (4 * top + 16) * U


ATTN = [
    # fmt, dtype, Hq, Hkv, D, page, lens, news, window, weights
    (4, "f32", 1, 1, 64, 16, [1], [1], 0, 2),                       # one token
    (7, "f32", 8, 8, 128, 16, [17, 2, 33], [1, 1, 1], 0, 1),        # decode, a head a group
    (4, "bf16", 8, 2, 128, 64, [300, 65, 1, 64], [1, 1, 1, 1], 0, 2),
    (7, "bf16", 40, 8, 64, 32, [700, 31], [1, 1], 0, 0),            # groups of 5
    (4, "f32", 6, 2, 192, 48, [130, 49], [3, 49], 0, 2),            # pages that end inside a tile
    (7, "f32", 3, 1, 192, 16, [50], [50], 20, 1),
    (4, "bf16", 4, 4, 256, 16, [90, 40], [33, 17], 0, 2),
    (7, "bf16", 16, 2, 256, 64, [257], [5], 0, 1),
    (7, "f32", 24, 1, 64, 16, [100, 5], [2, 5], 0, 2),              # 24 heads share a kv head
    (4, "bf16", 8, 2, 128, 64, [1500, 900], [70, 130], 0, 2),       # prompt chunks
    (7, "bf16", 4, 2, 64, 16, [800, 300], [200, 9], 64, 2),         # a window
    (4, "f32", 4, 1, 128, 64, [2500], [1], 0, 2),                   # split over the tokens
    (7, "f32", 2, 2, 128, 128, [3000, 10], [1, 1], 1000, 2),        # split, with a window
    (7, "bf16", 4, 2, 128, 16, [10, 0, 5], [12, 0, 5], 0, 2),       # more rows than tokens; none
]


@pytest.fixture(params=[0, 2], ids=["by size", "many rows"])
def rows_kernel(hip, request):
    """The kernel by the call's size, and that of many rows at every size."""
    assert hip.set_option("kv4_rows", request.param)
    yield request.param
    assert hip.set_option("kv4_rows", 0)


@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(map(str, c[:6])))
def test_attention(hip, rows_kernel, case):
    fmt, dtype, Hq, Hkv, D, page, lens, news, window, weights = case
    rng = np.random.default_rng(sum(lens) + D + Hq + fmt)
    n_pages = sum(-(-n // page) for n in lens) + len(lens) * (max(lens) // page + 3)
    c = make_cache(rng, fmt, Hkv, D, page, n_pages)
    arr, cache = to_device(hip, c)
    tab, qs, T = tables(rng, lens, page, n_pages), starts(news), sum(news)
    q = dev((2 * rng.standard_normal((T + 1, Hq + 1, D))).astype(np.float32), TYPES[dtype])[:, :Hq]
    ln = np.array(lens, np.int32)
    out = run_attention(hip, cache, dtype, q, dev(qs), dev(ln), dev(tab), max(news), max(lens),
                        D ** -0.5, window, weights)
    err = check_attention(c, host(q), host(out), host(arr["score"]), qs, ln, tab, D ** -0.5, window,
                          weights, dtype, forced=rows_kernel == 2)
    print("  err", err, flush=True)
    for n in ("k", "ks", "v", "vs"):
        assert np.array_equal(host(arr[n]), c[n])
    if not weights:
        assert np.array_equal(host(arr["score"]), c["score"])


@pytest.mark.parametrize("fmt", [4, 7])
@pytest.mark.parametrize("dtype,news,window", [("f32", [1, 1], 0), ("bf16", [20, 40], 0),
                                               ("f32", [1, 1], 30), ("bf16", [40, 20], 17)])
def test_attention_ignores_what_is_not_seen(hip, rows_kernel, fmt, dtype, news, window):
    """Non-finite scales behind a sequence's end, on its unseen pages, behind bad table entries and
    ahead of every window change nothing; bad entries are tokens that are not there."""
    rng = np.random.default_rng(fmt + len(dtype) + window)
    lens, page, Hq, Hkv, D = [100, 230], 16, 4, 2, 128
    c = make_cache(rng, fmt, Hkv, D, page, 60)
    tab, qs = tables(rng, lens, page, 60, extra=3), starts(news)
    tab[1, 3], tab[1, 8] = -1, 60
    tab[0, 9:] = -7
    arr, cache = to_device(hip, c)
    q = dev(rng.standard_normal((sum(news), Hq, D)).astype(np.float32), TYPES[dtype])
    ln = np.array(lens, np.int32)
    args = (dtype, q, dev(qs), dev(ln), dev(tab), max(news), max(lens), 0.2, window, 2)
    out = run_attention(hip, cache, *args)
    check_attention(c, host(q), host(out), host(arr["score"]), qs, ln, tab, 0.2, window, 2, dtype,
                    forced=rows_kernel == 2)
    used = np.zeros((60, page), bool)
    for b, n in enumerate(lens):
        first = max(0, n - news[b] - window + 1) if window else 0
        for t in range(first, n):
            p = kvref.place(c, tab[b], t)
            if p:
                used[p] = True
    for n in ("ks", "vs"):
        bad = np.nan if fmt == 4 else 255
        s = host(arr[n])
        s[np.broadcast_to(~used[:, None, :, None], s.shape)] = bad
        arr[n].copy_(dev(s))
    again = run_attention(hip, cache, *args)
    assert torch.equal(out, again)


@pytest.mark.parametrize("fmt,dtype", [(4, "f32"), (7, "bf16")])
def test_masked_future_tokens_may_be_anything(hip, rows_kernel, fmt, dtype):
    """New tokens whose scales are not finite are seen by the rows from them on, and by no row
    ahead of them."""
    rng = np.random.default_rng(fmt)
    c = make_cache(rng, fmt, 1, 64, 16, 4)
    tab, qs, ln = np.arange(4, dtype=np.int32)[None], starts([40]), np.array([50], np.int32)
    q = dev(rng.standard_normal((40, 2, 64)).astype(np.float32), TYPES[dtype])
    arr, cache = to_device(hip, c)
    args = (dtype, q, dev(qs), dev(ln), dev(tab), 40, 50, 0.2)
    clean = run_attention(hip, cache, *args)
    for n, s in (("ks", 35), ("vs", 35)):
        x = host(arr[n])
        x[s // 16, 0, s % 16] = np.nan if fmt == 4 else 255
        arr[n].copy_(dev(x))
    out = run_attention(hip, cache, *args)
    assert torch.equal(out[:25], clean[:25])  # row 25 is token 35
    assert torch.isnan(out[25:]).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_nonfinite_queries_stay_in_their_rows(hip, rows_kernel, dtype):
    rng = np.random.default_rng(9)
    c = make_cache(rng, 7, 2, 64, 16, 40)
    tab, qs = tables(rng, [200, 100], 16, 40), starts([30, 1])
    ln = np.array([200, 100], np.int32)
    x = rng.standard_normal((31, 4, 64)).astype(np.float32)
    arr, cache = to_device(hip, c)
    args = (dev(qs), dev(ln), dev(tab), 30, 200, 0.2)
    clean = run_attention(hip, cache, dtype, dev(x, TYPES[dtype]), *args)
    x[3, 1, 5], x[30, 2, 0] = np.nan, np.nan
    out = run_attention(hip, cache, dtype, dev(x, TYPES[dtype]), *args)
    bad = np.zeros((31, 4), bool)
    bad[3, 1] = bad[30, 2] = True
    assert torch.isnan(out[dev(bad)]).all()
    assert torch.equal(out[dev(~bad)], clean[dev(~bad)])


@pytest.mark.parametrize("max_new,max_len", [(1, 1), (3, 100), (200, 5000)])
def test_attention_sizes_are_hints(hip, rows_kernel, max_new, max_len):
    """Bounds below or above the real sizes change the launch, not what is computed."""
    rng = np.random.default_rng(3)
    c = make_cache(rng, 4, 2, 128, 32, 60)
    lens, news = [900, 40], [70, 40]
    tab, qs, ln = tables(rng, lens, 32, 60), starts(news), np.array(lens, np.int32)
    arr, cache = to_device(hip, c)
    q = dev(rng.standard_normal((110, 4, 128)).astype(np.float32))
    out = run_attention(hip, cache, "f32", q, dev(qs), dev(ln), dev(tab), max_new, max_len, 0.1, 0,
                        2)
    check_attention(c, host(q), host(out), host(arr["score"]), qs, ln, tab, 0.1, 0, 2, "f32",
                    forced=rows_kernel == 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_widest_window_and_rows_before_the_first_token(hip, rows_kernel, dtype):
    """More rows than tokens under the widest window a call takes: the rows ahead of the first
    token give zeros, and their positions take nothing from the rows they share a tile with."""
    rng = np.random.default_rng(11)
    c = make_cache(rng, 4, 2, 64, 32, 20)
    lens, news = [7, 90], [20, 33]
    tab, qs, ln = tables(rng, lens, 32, 20), starts(news), np.array(lens, np.int32)
    arr, cache = to_device(hip, c)
    q = torch.from_numpy(rng.standard_normal((53, 4, 64)).astype(np.float32)).cuda().to(TYPES[dtype])
    out = run_attention(hip, cache, dtype, q, dev(qs), dev(ln), dev(tab), 33, 90, 0.2, 2 ** 31 - 1, 2)
    check_attention(c, host(q), host(out), host(arr["score"]), qs, ln, tab, 0.2, 2 ** 31 - 1, 2, dtype,
                    forced=rows_kernel == 2)
    assert (host(out)[:13] == 0).all() and (host(out)[13:20] != 0).any()


def test_attention_scales(hip, rows_kernel):
    """Negative and zero scales, and logits past the exponents' range."""
    rng = np.random.default_rng(4)
    c = make_cache(rng, 4, 1, 64, 16, 20)
    tab, qs, ln = tables(rng, [200], 16, 20), starts([3]), np.array([200], np.int32)
    arr, cache = to_device(hip, c)
    q = dev(rng.standard_normal((3, 4, 64)).astype(np.float32))
    for scale in (0.0, -0.2, 30.0):
        out = run_attention(hip, cache, "f32", q, dev(qs), dev(ln), dev(tab), 3, 200, scale)
        check_attention(c, host(q), host(out), None, qs, ln, tab, scale, 0, 0, "f32",
                        forced=rows_kernel == 2)


def test_shared_pages_and_streams(hip):
    """Two sequences over one prefix's pages; calls on two streams at once, each with its own
    workspace and output, agree with the calls one after the other bit for bit."""
    rng = np.random.default_rng(8)
    c = make_cache(rng, 7, 4, 128, 32, 80)
    tab = tables(rng, [1000, 1000], 32, 80)
    tab[1, :20] = tab[0, :20]
    ln, qs = np.array([900, 1000], np.int32), starts([1, 4])
    arr, cache = to_device(hip, c)
    qs_d, ln_d, tab_d = dev(qs), dev(ln), dev(tab)
    q = [dev(rng.standard_normal((5, 16, 128)).astype(np.float32)) for _ in range(2)]
    n = hip.kv4_attention_work(4, 128, 16, 5, 2, 4, 1000)
    assert n > 0
    alone = [run_attention(hip, cache, "f32", x, qs_d, ln_d, tab_d, 4, 1000, 0.1) for x in q]
    check_attention(c, host(q[0]), host(alone[0]), None, qs, ln, tab, 0.1, 0, 0, "f32")
    st = [torch.cuda.Stream() for _ in q]
    work = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in q]
    out = [torch.empty_like(a) for a in alone]
    torch.cuda.synchronize()
    for _ in range(10):
        for i in range(2):
            hip.kv4_attention_dev(cache, hip.F32, q[i], 16 * 128, 16, 5, qs_d, ln_d, tab_d, 2,
                                  tab.shape[1], 4, 1000, 0.1, 0, 0, out[i], work[i], n, st[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, out))


@pytest.mark.parametrize("fmt", [4, 7])
def test_cache_past_32_bits(hip, fmt):
    """Pages whose codes lie more than 2^32 bytes into the pool."""
    rng = np.random.default_rng(fmt)
    n_kv, D, page = 8, 256, 128
    n_pages = (1 << 32) // (n_kv * page * D // 2) + 8
    small = make_cache(rng, fmt, n_kv, D, page, 8)
    big = {n: torch.empty((n_pages, *small[n].shape[1:]), device="cuda",
                          dtype=torch.float32 if small[n].dtype == np.float32 else torch.uint8)
           for n in ("k", "ks", "v", "vs", "score")}
    for n in big:
        big[n][-8:] = dev(small[n])
        big[n][:8] = dev(small[n])  # what a 32-bit offset would read instead
        big[n][:8].zero_()
    cache = hip.KV4(fmt, n_kv, D, page, big["k"], big["ks"], big["v"], big["vs"], big["score"])
    tab = rng.permutation(8)[:6].reshape(2, 3).astype(np.int32)
    ln, qs = np.array([300, 140], np.int32), starts([2, 9])
    far = dev(tab + n_pages - 8)
    kv = dev(rng.standard_normal((2, 11, n_kv, D)).astype(np.float32))
    hip.kv4_append_dev(cache, hip.F32, kv[0], n_kv * D, kv[1], n_kv * D, 11, dev(qs), dev(ln), far,
                       2, 3)
    for r, b, t in kvref.rows_of(qs, ln):
        p, s = kvref.place(small, tab[b], t)
        for i, n in enumerate("kv"):
            small[n][p, :, s], small[n + "s"][p, :, s] = kvref.quantize(fmt, host(kv)[i, r])
        small["score"][p, :, s] = 0
    q = dev(rng.standard_normal((11, n_kv, D)).astype(np.float32))
    out = run_attention(hip, cache, "f32", q, dev(qs), dev(ln), far, 9, 300, 0.1, 0, 1)
    check_attention(small, host(q), host(out), host(big["score"][-8:]), qs, ln, tab, 0.1, 0, 1, "f32")
    for n in ("k", "ks", "v", "vs"):
        assert np.array_equal(host(big[n][-8:]), small[n])


# ---- eviction ------------------------------------------------------------------------------


EVICT = [
    # fmt, n_kv, D, page, lens, keep, recent
    (4, 1, 64, 16, [40], 16, 0), (7, 3, 128, 48, [100, 20, 64, 65], 64, 10),
    (4, 2, 192, 16, [70, 1, 0], 33, 33), (7, 2, 256, 64, [500, 130], 129, 1),
    (4, 4, 128, 64, [3000, 2049], 1000, 100), (7, 1, 64, 16, [17], 16, 15), (7, 2, 64, 32, [90], 1, 0),
]


def moved(c, kept, new_lens, tab, dst):
    exp = {n: c[n].copy() for n in ("k", "ks", "v", "vs", "score")}
    for b in range(len(new_lens)):
        for j in range(new_lens[b]):
            to = kvref.place(c, dst[b], j)
            for h in range(kept.shape[1]):
                at = kvref.place(c, tab[b], int(kept[b, h, j]))
                if at and to:
                    for n in exp:
                        exp[n][to[0], h, to[1]] = c[n][at[0], h, at[1]]
    return exp


@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("scores", ["spread", "ties", "odd"])
def test_evict(hip, case, scores):
    fmt, n_kv, D, page, lens, keep, recent = case
    rng = np.random.default_rng(keep + sum(lens))
    need = -(-keep // page)
    n_pages = sum(-(-n // page) for n in lens) + len(lens) * (max(lens) // page + need + 3)
    c = make_cache(rng, fmt, n_kv, D, page, n_pages)
    if scores == "ties":
        c["score"] = rng.integers(0, 3, c["score"].shape).astype(np.float32)
    elif scores == "odd":  # negatives, signed zeros, infinities, NaN, denormals
        odd = np.array([-1, 0.0, -0.0, np.inf, -np.inf, np.nan, 1e-42, -1e-42, 3e38, 1], np.float32)
        c["score"] = rng.choice(odd, c["score"].shape)
    both = tables(rng, lens, page, n_pages, extra=1 + need)
    tab, dst = np.ascontiguousarray(both[:, :-need]), np.ascontiguousarray(both[:, -need:])
    arr, cache = to_device(hip, c)
    kept = torch.full((len(lens), n_kv, keep), -9, dtype=torch.int32, device="cuda")
    new = torch.full((len(lens),), -9, dtype=torch.int32, device="cuda")
    ln = np.array(lens, np.int32)
    hip.kv4_evict_dev(cache, dev(ln), dev(tab), len(lens), tab.shape[1], max(lens), keep, recent,
                      dev(dst), need, kept, new)
    torch.cuda.synchronize()
    ek, en = kvref.evict(c, ln, tab, keep, recent)
    assert np.array_equal(host(new), en)
    assert np.array_equal(host(kept), ek)
    exp = moved(c, ek, en, tab, dst)
    for n in exp:
        assert np.array_equal(host(arr[n]).view(np.uint8), exp[n].view(np.uint8)), n


@pytest.mark.parametrize("max_len", [1, 500, 60000])
def test_evict_long_and_bad_pages(hip, max_len):
    """Longer than the launch was sized for (and than the on-chip keys), tokens that are not
    there, pages that are not there to move to."""
    rng = np.random.default_rng(max_len)
    n, page, keep = 45000, 64, 300
    c = make_cache(rng, 7, 1, 64, page, 720)
    c["score"] = rng.integers(0, 500, c["score"].shape).astype(np.float32)
    perm = rng.permutation(720).astype(np.int32)
    tab, dst = perm[:704][None].copy(), perm[704:709][None].copy()
    tab[0, 5], tab[0, 600], tab[0, 702], dst[0, 2] = -1, 720, 9999, -1
    arr, cache = to_device(hip, c)
    kept = torch.empty((1, 1, keep), dtype=torch.int32, device="cuda")
    new = torch.empty(1, dtype=torch.int32, device="cuda")
    ln = np.array([n], np.int32)
    hip.kv4_evict_dev(cache, dev(ln), dev(tab), 1, 704, max_len, keep, 100, dev(dst), 5, kept, new)
    torch.cuda.synchronize()
    ek, en = kvref.evict(c, ln, tab, keep, 100)
    assert np.array_equal(host(kept), ek) and np.array_equal(host(new), en)
    exp = moved(c, ek, en, tab, dst)
    for a in exp:
        assert np.array_equal(host(arr[a]), exp[a]), a


# ---- together ------------------------------------------------------------------------------


def chain_step(hip, dtype, s, stream=None):
    """Norm and rotate, append, attend with weights: one decoding step of the attention layer."""
    T, Hq, Hkv, D, B = s["T"], s["Hq"], s["Hkv"], s["D"], s["B"]
    row = (Hq + 2 * Hkv) * D
    d = dt(hip, dtype)
    qkv = s["qkv"]
    hip.qk_norm_rope_dev(d, T, D, qkv, row, Hq, s["q"], Hq * D, qkv[:, Hq:], row, Hkv, s["k"],
                         Hkv * D, s["wq"], s["wk"], 1e-6, s["pos"], s["freq"], D, False, stream)
    hip.kv4_append_dev(s["cache"], d, s["k"], Hkv * D, qkv[:, Hq + Hkv:], row, T, s["q_start"],
                       s["lens"], s["tab"], B, s["tab"].shape[1], stream)
    hip.kv4_attention_dev(s["cache"], d, s["q"], Hq * D, Hq, T, s["q_start"], s["lens"], s["tab"], B,
                          s["tab"].shape[1], s["max_new"], s["max_len"], D ** -0.5, 0, 1, s["out"],
                          s["work"], s["work"].numel(), stream)


def chain_state(hip, rng, fmt, dtype, news, max_len=700, Hq=8, Hkv=2, D=128, page=32, pages=120):
    B, T = len(news), sum(news)
    c = make_cache(rng, fmt, Hkv, D, page, pages)
    c["score"][:] = 0
    arr, cache = to_device(hip, c)
    f = lambda *n: torch.empty(n, device="cuda", dtype=TYPES[dtype])  # noqa: E731
    n = hip.kv4_attention_work(Hkv, D, Hq, T, B, max(news), max_len, 1)
    return c, dict(T=T, Hq=Hq, Hkv=Hkv, D=D, B=B, cache=cache, arr=arr, max_new=max(news),
                   max_len=max_len, qkv=f(T, Hq + 2 * Hkv, D), q=f(T, Hq, D), k=f(T, Hkv, D),
                   out=f(T, Hq, D), work=torch.empty(n, dtype=torch.uint8, device="cuda"),
                   wq=dev(np.float32(1 + 0.1 * rng.standard_normal(D))),
                   wk=dev(np.float32(1 + 0.1 * rng.standard_normal(D))),
                   freq=dev(10000.0 ** (-2.0 * np.arange(D // 2) / D)), q_start=dev(starts(news)),
                   pos=torch.zeros(T, dtype=torch.int32, device="cuda"),
                   lens=torch.zeros(B, dtype=torch.int32, device="cuda"),
                   tab=dev(tables(rng, [max_len] * B, page, pages)))


@pytest.mark.parametrize("fmt,dtype", [(4, "f32"), (7, "bf16")])
def test_prompt_decode_evict_decode(hip, fmt, dtype):
    """A prompt in chunks, decoding, an eviction by the weights collected on the way, decoding
    on: each attention output against the plain form on the cache as it then is."""
    rng = np.random.default_rng(fmt)
    page = 32
    c, s = chain_state(hip, rng, fmt, dtype, [1, 1])
    _, p = chain_state(hip, np.random.default_rng(fmt + 1), fmt, dtype, [60, 41])
    p |= {n: s[n] for n in ("cache", "arr", "tab", "wq", "wk", "freq")}
    held, seen = np.zeros(2, np.int32), np.zeros(2, np.int32)
    score = np.zeros_like(c["score"], dtype=np.float64)

    def step(st, news):
        nonlocal held, seen, score
        x = rng.standard_normal(tuple(st["qkv"].shape)).astype(np.float32)
        st["qkv"].copy_(dev(x))
        held, seen = held + news, seen + news
        st["lens"].copy_(dev(held.astype(np.int32)))
        st["pos"].copy_(dev(np.concatenate([np.arange(e - n, e) for e, n in zip(seen, news)])
                            .astype(np.int32)))
        chain_step(hip, dtype, st)
        torch.cuda.synchronize()
        now = {n: host(st["arr"][n]) for n in ("k", "ks", "v", "vs")} | \
            dict(fmt=fmt, page=page, score=score)
        qs, tab = host(st["q_start"]), host(st["tab"])
        for r, b, t in kvref.rows_of(qs, held):
            pl = kvref.place(now, tab[b], t)
            score[pl[0], :, pl[1]] = 0
        out, mag, (top, _, root), score = kvref.attention(now, host(st["q"]), qs, held, tab,
                                                          128 ** -0.5, 0, 1)
        f, k_off = (2.0 ** -11, 12 * U) if st is p else (0.0, 0.0)  # many rows, maybe f16
        tol = (4 * top + 16) * U + (H if dtype == "bf16" else 0) + 2 * k_off * root + 3 * f
        assert np.linalg.norm(host(st["out"]) - out) <= tol * np.linalg.norm(out)
        assert np.linalg.norm(host(st["arr"]["score"]) - score) <= \
            ((4 * top + 64) * U + 2 * k_off * root) * np.linalg.norm(score)

    step(p, [60, 41])
    step(p, [60, 41])
    for _ in range(3):
        step(s, [1, 1])
    keep = 70
    dst = dev(np.setdiff1d(np.arange(120), host(s["tab"]))[:6].reshape(2, 3).astype(np.int32))
    kept = torch.empty((2, 2, keep), dtype=torch.int32, device="cuda")
    new = torch.empty(2, dtype=torch.int32, device="cuda")
    now = {n: host(s["arr"][n]) for n in ("k", "ks", "v", "vs", "score")} | dict(fmt=fmt, page=page)
    hip.kv4_evict_dev(s["cache"], s["lens"], s["tab"], 2, s["tab"].shape[1], 700, keep, 16, dst, 3,
                      kept, new)
    torch.cuda.synchronize()
    ek, en = kvref.evict(now, held, host(s["tab"]), keep, 16)
    assert np.array_equal(host(kept), ek) and np.array_equal(host(new), en)
    held = en.copy()
    fresh = torch.full_like(s["tab"], -1)
    fresh[:, :3] = dst
    fresh[:, 3:6] = s["tab"][:, :3]  # freed pages take the next tokens
    s["tab"].copy_(fresh)
    score = host(s["arr"]["score"]).astype(np.float64)
    for _ in range(30):
        step(s, [1, 1])


@pytest.mark.parametrize("fmt,dtype", [(7, "f32"), (4, "bf16")])
def test_captured_step_replays(hip, fmt, dtype):
    """A captured decoding step, replayed over growing sequences with eager steps between: every
    replay equals the eager step on a twin cache bit for bit."""
    rng = np.random.default_rng(fmt)
    _, a = chain_state(hip, np.random.default_rng(1), fmt, dtype, [1, 1, 1])
    _, b = chain_state(hip, np.random.default_rng(1), fmt, dtype, [1, 1, 1])
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        chain_step(hip, dtype, a, st)
    lens = np.array([5, 640, 31], np.int32)
    for i in range(8):
        lens = lens + 1
        x = dev(rng.standard_normal(tuple(a["qkv"].shape)).astype(np.float32))
        for s in (a, b):
            s["qkv"].copy_(x)
            s["lens"].copy_(dev(lens))
            s["pos"].copy_(dev(lens - 1))
        torch.cuda.synchronize()
        if i % 3 == 2:
            chain_step(hip, dtype, a)
        else:
            graph.replay()
        torch.cuda.synchronize()
        chain_step(hip, dtype, b)
        torch.cuda.synchronize()
        assert torch.equal(a["out"], b["out"])
        for n in ("k", "ks", "v", "vs", "score"):
            assert torch.equal(a["arr"][n], b["arr"][n]), n


def test_repeats_are_equal(hip, rows_kernel):
    """The same call again gives the same bits, weights included (no sum depends on an order)."""
    rng = np.random.default_rng(2)
    c = make_cache(rng, 4, 2, 128, 64, 120)
    arr, cache = to_device(hip, c)
    tab, ln = tables(rng, [3000, 1700], 64, 120), np.array([3000, 1700], np.int32)
    q = dev(rng.standard_normal((2, 16, 128)).astype(np.float32))
    args = ("f32", q, dev(starts([1, 1])), dev(ln), dev(tab), 1, 3000, 0.1, 0, 2)
    first, score = run_attention(hip, cache, *args), arr["score"].clone()
    for _ in range(5):
        assert torch.equal(run_attention(hip, cache, *args), first)
        assert torch.equal(arr["score"], score)


def test_stream_of_torch_and_null(hip):
    """NULL is the null stream; a torch stream orders the call behind its own work."""
    rng = np.random.default_rng(6)
    x = dev(rng.standard_normal((64, 8, 128)).astype(np.float32))
    y, z = torch.empty_like(x), torch.empty_like(x)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(5):
            big = big @ big * 1e-2
        w = x * 2
        hip.qk_norm_rope_dev(hip.F32, 64, 128, w, 1024, 8, y, 1024, None, 0, 0, None, 0, None, None,
                             0.0, None, None, 0, False, st)
    torch.cuda.synchronize()
    hip.qk_norm_rope_dev(hip.F32, 64, 128, x, 1024, 8, z, 1024, None, 0, 0, None, 0, None, None, 0.0,
                         None, None, 0)
    torch.cuda.synchronize()
    assert torch.equal(y, z)  # a power of two does not change the norm's roundings


FIRST = """
import numpy as np, torch
import mvllm_hip as h
h.init(0)
h.set_option("kv4_rows", 2)
z = lambda *s, dtype=torch.uint8: torch.zeros(s, dtype=dtype, device="cuda")
i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
c = h.KV4(4, 1, 64, 32, z(8, 1, 32, 32), z(8, 1, 32, 1, dtype=torch.float32), z(8, 1, 32, 32),
          z(8, 1, 32, 1, dtype=torch.float32), z(8, 1, 32, dtype=torch.float32))
q, out = torch.ones(40, 1, 64, device="cuda"), torch.ones(40, 1, 64, device="cuda")
kept, new, work = i32(*[7] * 16), i32(7), z(1 << 20)
qs, ln, tab, dst = i32(0, 40), i32(100), i32(0, 1, 2, 3), i32(4)
st = torch.cuda.Stream()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=st):
    h.kv4_attention_dev(c, h.F32, q, 64, 1, 40, qs, ln, tab, 1, 4, 40, 100, 1.0, 0, 2, out, work,
                        1 << 20, st)
    h.kv4_evict_dev(c, ln, tab, 1, 4, 100, 16, 4, dst, 1, kept, new, st)
for i in range(3):
    out.fill_(1)
    kept.fill_(7)
    g.replay()
    torch.cuda.synchronize()
    assert (out == 0).all() and int(new) == 16 and kept.tolist() == [*range(12), *range(96, 100)], kept
print("replayed")
"""


def test_first_call_of_a_process_is_captured():
    """The calls that set a kernel up on their first use may make it inside a capture."""
    p = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=100,
                       env=os.environ | {"PYTHONPATH": os.pathsep.join(sys.path)})
    assert p.returncode == 0 and "replayed" in p.stdout, p.stderr[-2000:]
