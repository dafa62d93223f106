"""Performance cases of the attention operators that keep keys and values in 4 bits, on one
MI355X: what a decoder layer runs in front of its routed experts.

  rope     mvllm_hip_qk_norm_rope_dev: RMSNorm of every query and key head and the position
           rotation, in one pass
  append   mvllm_hip_kv4_append_dev: new keys and values quantized into the paged cache
           (read back with mvllm_hip_kv4_read_dev, as the values it holds)
  attn     mvllm_hip_kv4_attention_dev: causal attention of new tokens over the cache, for
           decode and for prompt chunks, with or without the keys' accumulated weights
  evict    mvllm_hip_kv4_evict_dev: each head keeps its keys of most accumulated weight and its
           most recent ones, moved to fresh pages (read back as above)

The cache is paged: k / v codes [pages][kv heads][page][head dim / 2] (low nibble = even
element), scales [pages][kv heads][page][head dim / group].  fmt 4 is int4-g64 (value
(n - 8) * scale, f32 scales per 64 elements), fmt 7 MXFP4 (e2m1 codes, ue8m0 bytes per 32).
Sequence b's token t lies in page table[b][t / page]; its new tokens are rows
q_start[b]..q_start[b + 1] and the last of its lens[b] tokens.
"""
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

GROUP = {4: 64, 7: 32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HELD = 6.0 * 2.0 ** 125  # values beyond +-HELD are held as that
TINY = 2.0 ** -100       # int4 groups below are held as zeros


# ---- the cases -----------------------------------------------------------------------------


def _rope(name, **kw):
    return dict(name=name, kind="rope", **kw)


def _append(name, **kw):
    return dict(name=name, kind="append", **kw)


def _attn(name, **kw):
    return dict(name=name, kind="attn", **kw)


def _evict(name, **kw):
    return dict(name=name, kind="evict", **kw)


def listed():
    return [
        # 16 concurrent decode streams of a 2048-wide model with 16 heads of 128: launch latency
        _rope("rope_decode_T16", dtype="f32", T=16, Hq=16, Hkv=16, D=128, rot=128,
              interleaved=False, far=4096),
        # a prompt of 4096 tokens, grouped heads, half of each head rotated, far positions
        _rope("rope_prompt_T4096", dtype="bf16", T=4096, Hq=64, Hkv=8, D=128, rot=64,
              interleaved=True, far=1 << 20),
        # one new token of each of 16 streams enters the cache
        _append("append_decode_int4", dtype="f32", fmt=4, B=16, Hkv=16, D=128, page=64, lmin=100,
                lmax=2048, nmax=1),
        # prompt chunks of up to 2048 tokens of three sequences
        _append("append_prompt_mxfp4", dtype="bf16", fmt=7, B=3, Hkv=8, D=128, page=64,
                lmin=2048, lmax=8192, nmax=2048),
        # decode of one short conversation: the smallest attention call
        _attn("attn_decode_one_int4", dtype="f32", fmt=4, B=1, Hq=16, Hkv=16, D=128, page=64,
              lmin=777, lmax=777, nmax=1, window=0, weights=False),
        # 16 decode streams of the same model
        _attn("attn_decode_int4", dtype="f32", fmt=4, B=16, Hq=16, Hkv=16, D=128, page=64,
              lmin=100, lmax=4096, nmax=1, window=0, weights=False),
        # 32 long conversations of a grouped-head model: the cache is what is read
        _attn("attn_decode_long_mxfp4", dtype="bf16", fmt=7, B=32, Hq=64, Hkv=8, D=128, page=64,
              lmin=4096, lmax=16384, nmax=1, window=0, weights=False),
        # decode that collects every key's weight for the next eviction
        _attn("attn_decode_weights_mxfp4", dtype="f32", fmt=7, B=8, Hq=32, Hkv=8, D=128, page=32,
              lmin=1000, lmax=8192, nmax=1, window=0, weights=True),
        # prompt chunks over earlier context: the matrix products are what counts
        _attn("attn_prompt_int4", dtype="bf16", fmt=4, B=2, Hq=32, Hkv=8, D=128, page=64,
              lmin=6000, lmax=8192, nmax=1024, window=0, weights=False),
        # ragged short chunks (drafted tokens, prompt tails) within a window, narrow heads
        _attn("attn_ragged_window_mxfp4", dtype="bf16", fmt=7, B=7, Hq=24, Hkv=4, D=64, page=16,
              lmin=130, lmax=5001, nmax=97, window=1024, weights=True),
        # four short streams over their budget
        _evict("evict_int4", fmt=4, B=4, Hkv=4, D=128, page=16, lmin=520, lmax=1500, keep=500,
               recent=64),
        # long contexts cut to their half
        _evict("evict_long_mxfp4", fmt=7, B=4, Hkv=8, D=128, page=64, lmin=12000, lmax=32768,
               keep=8192, recent=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attn", "attn", "attn", "evict"])
    D = rng.choice([64, 128, 128, 192, 256])
    dtype, fmt = rng.choice(["f32", "bf16"]), rng.choice([4, 7])
    Hkv = rng.choice([1, 2, 3, 4, 8, 16])
    G = rng.choice([1, 2, 4, 5, 6, 8])
    page = rng.choice([16, 32, 48, 64, 128])
    if kind == "rope":
        return dict(kind=kind, dtype=dtype, T=_log(rng, 1, 4096), Hq=min(64, Hkv * G), Hkv=Hkv, D=D,
                    rot=rng.choice([16, 32, D // 2, D]), interleaved=rng.random() < 0.5,
                    far=_log(rng, 64, 1 << 20))
    if kind == "append":
        lmax = _log(rng, 20, 8192)
        return dict(kind=kind, dtype=dtype, fmt=fmt, B=_log(rng, 1, 16), Hkv=min(8, Hkv), D=D,
                    page=page, lmin=max(1, lmax // 3), lmax=lmax,
                    nmax=rng.choice([1, 1, _log(rng, 2, 700)]))
    if kind == "evict":
        lmax = _log(rng, 200, 16384)
        keep = max(8, int(lmax * rng.uniform(0.2, 0.8)))
        return dict(kind=kind, fmt=fmt, B=rng.randint(1, 6), Hkv=min(8, Hkv), D=min(D, 128),
                    page=page, lmin=max(1, lmax // 2), lmax=lmax, keep=keep,
                    recent=int(keep * rng.uniform(0.0, 0.5)))
    decode = rng.random() < 0.5
    lmax = _log(rng, 1, 12000) if decode else _log(rng, 64, 6000)
    return dict(kind=kind, dtype=dtype, fmt=fmt, B=_log(rng, 1, 16 if decode else 4),
                Hq=min(8, Hkv) * G, Hkv=min(8, Hkv), D=D, page=page, lmin=max(1, lmax // 4),
                lmax=lmax, nmax=rng.choice([1, 1, 2, 5]) if decode else _log(rng, 8, 600),
                window=rng.choice([0, 0, _log(rng, 16, 4096)]), weights=rng.random() < 0.4)


def _lens(c):
    """Tokens in the cache by sequence, the first one lmax, the others spread down to lmin."""
    return [c["lmax"] - int((c["lmax"] - c["lmin"]) * ((b * 0.6180339887) % 1.0))
            for b in range(c["B"])]


def _news(c):
    """New tokens by sequence (at most its length), the first one nmax."""
    return [max(1, min(n, c["nmax"] - int((c["nmax"] - 1) * ((b * 0.3819660113) % 1.0))))
            for b, n in enumerate(_lens(c))]


# ---- inputs --------------------------------------------------------------------------------


def _nibbles(codes):
    """[..., n / 2] bytes -> [..., n] nibbles, the low one first."""
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def _values(fmt, codes, scales):
    """What codes [..., D / 2] and scales [..., D / group] stand for, f32 [..., D]."""
    n = _nibbles(codes)
    if fmt == 4:
        v, s = n.float() - 8.0, scales
    else:
        v = torch.tensor(E2M1, device=codes.device)[n.int()]
        s = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    return (v.unflatten(-1, (-1, GROUP[fmt])) * s.unsqueeze(-1)).flatten(-2)


def _quantize(fmt, x):
    """[..., D] -> codes [..., D / 2], scales [..., D / group]."""
    x = x.float().nan_to_num(nan=0.0, posinf=HELD, neginf=-HELD).clamp(-HELD, HELD)
    x = x.unflatten(-1, (-1, GROUP[fmt]))
    top = x.abs().amax(-1)
    if fmt == 4:
        s = torch.where(top < TINY, torch.zeros_like(top), top / 7.0)
        wide = s.double().unsqueeze(-1)  # in 64 bits: a value next to a border takes its own side
        n = torch.where(wide > 0, (x.double() / wide).round(), torch.zeros_like(wide)).clamp(-7, 7)
        n, s = (n + 8).to(torch.uint8), s
    else:
        m, e = torch.frexp(top.clamp(min=6.0 * 2.0 ** -126) / 6.0)
        e = torch.where(m == 0.5, e - 1, e)  # the smallest e with top <= 6 * 2^e
        q = torch.ldexp(x, -e.unsqueeze(-1)).clamp(-6.0, 6.0)
        a = q.abs()
        n = sum((a > t).to(torch.uint8) for t in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0))
        n = torch.where((q < 0) & (n > 0), n | 8, n)
        s = (e + 127).to(torch.uint8)
    n = n.flatten(-2)
    return n[..., 0::2] | (n[..., 1::2] << 4), s


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _cache(c, g, lens, spare=0, scored=False):
    """A pool whose pages the sequences hold in random order, and their table; `spare` more pages
    a sequence in a second table."""
    per = -(-max(lens) // c["page"])
    pages = c["B"] * (per + spare)
    shape = (pages, c["Hkv"], c["page"], c["D"])
    chan = torch.exp(0.5 * _normal(g, c["Hkv"], 1, c["D"]))  # keys have channels of unlike size
    k, ks = _quantize(c["fmt"], _normal(g, *shape) * chan)
    v, vs = _quantize(c["fmt"], _normal(g, *shape) * 0.5)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s = dict(k=k, ks=ks, v=v, vs=vs, table=order[: c["B"] * per].reshape(c["B"], per).contiguous(),
             lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if spare:
        s["dst"] = order[c["B"] * per:].reshape(c["B"], spare).contiguous()
    if scored:
        # weights fall off steeply; many old keys of none at all tie
        w = torch.exp(2.0 * _normal(g, *shape[:3]))
        s["score"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.1, 0.0, w)
    return s


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": c}
    if c["kind"] == "rope":
        T, dt = c["T"], TYPES[c["dtype"]]
        # queries and keys are views of the projection's rows [queries | keys | values]
        s["qkv"] = _normal(g, T, c["Hq"] + 2 * c["Hkv"], c["D"]).to(dt)
        s["wq"], s["wk"] = (1.0 + 0.2 * _normal(g, c["D"]) for _ in range(2))
        s["pos"] = torch.randint(0, c["far"], (T,), generator=g, device="cuda", dtype=torch.int32)
        j = torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda")
        s["freq"] = 10000.0 ** (-2.0 * j / c["rot"])
        s["qo"] = torch.empty((T, c["Hq"], c["D"]), dtype=dt, device="cuda")
        s["ko"] = torch.empty((T, c["Hkv"], c["D"]), dtype=dt, device="cuda")
        return s
    lens = _lens(c)
    if c["kind"] == "evict":
        s |= _cache(c, g, lens, spare=-(-c["keep"] // c["page"]), scored=True)
        after = [min(n, c["keep"]) for n in lens]
        s["rows"] = sum(after)
        s["after"] = _starts(after)
        s["kept"] = torch.empty((c["B"], c["Hkv"], c["keep"]), dtype=torch.int32, device="cuda")
        s["new_lens"] = torch.empty(c["B"], dtype=torch.int32, device="cuda")
        s["kv_out"] = [torch.empty((s["rows"], c["Hkv"], c["D"]), device="cuda") for _ in range(2)]
        return s
    news, dt = _news(c), TYPES[c["dtype"]]
    T = sum(news)
    s["T"], s["q_start"] = T, _starts(news)
    s |= _cache(c, g, lens)
    if c["kind"] == "append":
        s["kn"], s["vn"] = (_normal(g, T, c["Hkv"], c["D"]).to(dt) for _ in range(2))
        s["kv_out"] = [torch.empty((T, c["Hkv"], c["D"]), device="cuda") for _ in range(2)]
        return s
    s["q"] = (2.0 * _normal(g, T, c["Hq"], c["D"])).to(dt)
    s["out"] = torch.empty((T, c["Hq"], c["D"]), dtype=dt, device="cuda")
    if c["weights"]:
        s["score"] = torch.zeros(s["k"].shape[:3], device="cuda")
    return s


def _starts(counts):
    return torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)


# ---- the plain forms -----------------------------------------------------------------------


def _plain_rope(s):
    c = s["case"]
    angle = s["pos"].double().unsqueeze(1) * s["freq"]  # far positions need the 64 bits
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)

    def one(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        r, rest = x[..., : c["rot"]], x[..., c["rot"]:]
        if c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = r.chunk(2, -1)
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((r, rest), -1).to(TYPES[c["dtype"]])

    q, k, _ = s["qkv"].split((c["Hq"], c["Hkv"], c["Hkv"]), 1)
    return {"q": one(q, s["wq"]), "k": one(k, s["wk"])}


def _places(s, starts, lens, rows):
    """(sequence, token) of each of the rows that q_start and lens describe."""
    r = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), r, right=True)
    return seq, lens[seq].long() - starts[seq + 1].long() + r


def _plain_append(s):
    c = s["case"]
    seq, tok = _places(s, s["q_start"], s["lens"], s["T"])
    page, slot = s["table"][seq, tok // c["page"]].long(), tok % c["page"]
    got = []
    for name, x in (("k", s["kn"]), ("v", s["vn"])):
        codes, scales = _quantize(c["fmt"], x)
        s[name][page, :, slot] = codes
        s[name + "s"][page, :, slot] = scales
        got.append(_values(c["fmt"], codes, scales))
    return {"k": got[0], "v": got[1]}


def _by_sequence(s, x):
    """A pool [pages, heads, page, n] as the sequences hold it: [B, heads, tokens, n]."""
    return x[s["table"].long()].transpose(1, 2).flatten(2, 3)


def _plain_attn(s):
    c = s["case"]
    B, G, n = c["B"], c["Hq"] // c["Hkv"], c["nmax"]
    k = _values(c["fmt"], _by_sequence(s, s["k"]), _by_sequence(s, s["ks"]))
    tokens = k.shape[2]
    seq, tok = _places(s, s["q_start"], s["lens"], s["T"])
    row = torch.arange(s["T"], device="cuda") - s["q_start"][seq].long()
    q = torch.zeros((B, n, c["Hq"], c["D"]), device="cuda")
    q[seq, row] = s["q"].float()
    at = torch.full((B, n), -1, device="cuda")  # the rows' positions; a row that is none sees nothing
    at[seq, row] = tok
    q = q.view(B, n, c["Hkv"], G, c["D"]).transpose(1, 2).reshape(B, c["Hkv"], n * G, c["D"])
    x = q @ k.transpose(2, 3).contiguous() * c["D"] ** -0.5
    del k
    t = torch.arange(tokens, device="cuda")
    seen = t <= at.unsqueeze(-1)
    if c["window"]:
        seen &= t > at.unsqueeze(-1) - c["window"]
    seen = seen.unsqueeze(1).repeat_interleave(G, 2)
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    v = _values(c["fmt"], _by_sequence(s, s["v"]), _by_sequence(s, s["vs"]))
    o = (p @ v).view(B, c["Hkv"], n, G, c["D"]).transpose(1, 2).reshape(B, n, c["Hq"], c["D"])
    r = {"out": o[seq, row].to(TYPES[c["dtype"]])}
    if c["weights"]:
        w = p.sum(2).unflatten(-1, (-1, c["page"])).transpose(1, 2)  # [B, pages, heads, page]
        held = (t < s["lens"].unsqueeze(1)).unflatten(-1, (-1, c["page"])).unsqueeze(2)
        old = s["score"][s["table"].long()]
        s["score"][s["table"].long()] = torch.where(held, w, old)
        r["score"] = s["score"]
    return r


def _plain_evict(s):
    c = s["case"]
    keep, recent = c["keep"], c["recent"]
    w = _by_sequence(s, s["score"].unsqueeze(-1)).squeeze(-1)  # [B, heads, tokens]
    t = torch.arange(w.shape[2], device="cuda")
    n = s["lens"].view(-1, 1, 1)
    w = torch.where(t >= n, -math.inf, torch.where(t >= n - recent, math.inf, w))
    if w.shape[2] < keep:
        w = torch.cat((w, w.new_full((*w.shape[:2], keep - w.shape[2]), -math.inf)), -1)
    best = w.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.where(best < n, best, 1 << 30).sort(-1).values
    kept = torch.where(kept < n, kept, -1)
    new_lens = s["lens"].clamp(max=keep)
    seq, tok = _places(s, s["after"], new_lens, s["rows"])
    src = kept[seq, :, tok]  # [rows, heads]
    head = torch.arange(c["Hkv"], device="cuda")
    page = torch.gather(s["table"][seq].long(), 1, src // c["page"])
    to = s["dst"][seq, tok // c["page"]].long().unsqueeze(1).expand(-1, c["Hkv"])
    heads = head.expand_as(src)
    got = {}
    for name in ("k", "ks", "v", "vs", "score"):
        got[name] = s[name][page, heads, src % c["page"]]
        s[name][to, heads, (tok % c["page"]).unsqueeze(1).expand_as(src)] = got[name]
    return {"kept": kept.to(torch.int32), "new_lens": new_lens, "score": s["score"],
            "k": _values(c["fmt"], got["k"], got["ks"]),
            "v": _values(c["fmt"], got["v"], got["vs"])}


# ---- the framework's operators -------------------------------------------------------------


def _library(s):
    """The binding, and the cache's handle as a program keeps it."""
    if "lib" not in s:
        path = os.path.join(ROOT, "micro-vllm_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import mvllm_hip
        mvllm_hip.init(0)
        s["lib"], c = mvllm_hip, s["case"]
        s["type"] = {"f32": mvllm_hip.F32, "bf16": mvllm_hip.BF16}[c.get("dtype", "f32")]
        if c["kind"] != "rope":
            s["cache"] = mvllm_hip.KV4(c["fmt"], c["Hkv"], c["D"], c["page"], s["k"], s["ks"],
                                       s["v"], s["vs"], s.get("score"))
        if c["kind"] == "attn":
            n = mvllm_hip.kv4_attention_work(c["Hkv"], c["D"], c["Hq"], s["T"], c["B"], c["nmax"],
                                             c["lmax"], c["weights"])
            s["work"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    return s["lib"]


def _own(s):
    c, L = s["case"], _library(s)
    st = torch.cuda.current_stream()
    if c["kind"] == "rope":
        row = s["qkv"].stride(0)
        k = s["qkv"][:, c["Hq"]:]
        L.qk_norm_rope_dev(s["type"], c["T"], c["D"], s["qkv"], row, c["Hq"], s["qo"],
                           c["Hq"] * c["D"], k, row, c["Hkv"], s["ko"], c["Hkv"] * c["D"],
                           s["wq"], s["wk"], 1e-6, s["pos"], s["freq"], c["rot"],
                           c["interleaved"], st)
        return {"q": s["qo"], "k": s["ko"]}
    if c["kind"] == "append":
        row = c["Hkv"] * c["D"]
        L.kv4_append_dev(s["cache"], s["type"], s["kn"], row, s["vn"], row, s["T"], s["q_start"],
                         s["lens"], s["table"], c["B"], s["table"].shape[1], st)
        k, v = s["kv_out"]
        L.kv4_read_dev(s["cache"], L.F32, k, v, s["T"], s["q_start"], s["lens"], s["table"],
                       c["B"], s["table"].shape[1], st)
        return {"k": k, "v": v}
    if c["kind"] == "attn":
        mode = L.WEIGHTS_STORE if c["weights"] else L.WEIGHTS_NONE
        L.kv4_attention_dev(s["cache"], s["type"], s["q"], c["Hq"] * c["D"], c["Hq"], s["T"],
                            s["q_start"], s["lens"], s["table"], c["B"], s["table"].shape[1],
                            c["nmax"], c["lmax"], c["D"] ** -0.5, c["window"], mode, s["out"],
                            s["work"], s["work"].numel(), st)
        return {"out": s["out"], "score": s["score"]} if c["weights"] else {"out": s["out"]}
    L.kv4_evict_dev(s["cache"], s["lens"], s["table"], c["B"], s["table"].shape[1], c["lmax"],
                    c["keep"], c["recent"], s["dst"], s["dst"].shape[1], s["kept"],
                    s["new_lens"], st)
    k, v = s["kv_out"]
    L.kv4_read_dev(s["cache"], L.F32, k, v, s["rows"], s["after"], s["new_lens"], s["dst"],
                   c["B"], s["dst"].shape[1], st)
    return {"kept": s["kept"], "new_lens": s["new_lens"], "score": s["score"], "k": k, "v": v}


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "append": _plain_append, "attn": _plain_attn,
            "evict": _plain_evict}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------


def _visible(c):
    """By sequence: (keys that some new token sees, (token, key) pairs)."""
    got = []
    for n, m in zip(_lens(c), _news(c)):
        span = c["window"] or n
        got.append((min(n, span + m - 1), sum(min(p + 1, span) for p in range(n - m, n))))
    return got


def work(case):
    c = case
    if c["kind"] == "rope":
        e = 4 if c["dtype"] == "f32" else 2
        rows = c["T"] * (c["Hq"] + c["Hkv"])
        return {"bytes": rows * c["D"] * 2 * e + 4 * c["T"], "flops": rows * c["D"] * 7}
    # codes and scales of one token's key (or value) of one head
    held = c["D"] // 2 + c["D"] // GROUP[c["fmt"]] * (4 if c["fmt"] == 4 else 1)
    if c["kind"] == "evict":
        after = sum(min(n, c["keep"]) for n in _lens(c))
        # weights read, kept tokens read and written, then read back as f32 values
        return {"bytes": c["Hkv"] * (4 * sum(_lens(c)) + after * (2 * (2 * held + 4) + 4 +
                                                                   2 * held + 8 * c["D"])),
                "flops": c["Hkv"] * after * 4 * c["D"]}
    e, T = (4 if c["dtype"] == "f32" else 2), sum(_news(c))
    if c["kind"] == "append":
        # rows read, codes written, then read back as f32 values
        return {"bytes": T * c["Hkv"] * 2 * (c["D"] * e + 2 * held + 4 * c["D"]),
                "flops": T * c["Hkv"] * c["D"] * 10}
    keys, pairs = (sum(x) for x in zip(*_visible(c)))
    b = keys * c["Hkv"] * 2 * held + 2 * T * c["Hq"] * c["D"] * e
    if c["weights"]:
        b += sum(_lens(c)) * c["Hkv"] * 4
    return {"bytes": b, "flops": 4 * pairs * c["Hq"] * c["D"]}


# ---- the definition in 64 bits -------------------------------------------------------------


def _hold(fmt, x):
    """The values that the cache holds of x [..., D], from the formats' definition."""
    g = GROUP[fmt]
    x = torch.nan_to_num(x.double(), nan=0.0, posinf=HELD, neginf=-HELD).clamp(-HELD, HELD)
    x = x.reshape(*x.shape[:-1], -1, g)
    top = x.abs().max(-1, keepdim=True).values
    if fmt == 4:
        s = (top.float() / 7.0).double()  # the scale is an f32
        s[top < TINY] = 1.0
        held = torch.round(x / s).clamp(-7, 7) * s
        return torch.where(top < TINY, 0.0, held).flatten(-2)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -126 * 6.0) / 6.0))
    e += (top > 6.0 * torch.exp2(e)).double()
    e -= (top <= 6.0 * torch.exp2(e - 1)).double() * (e > -126).double()
    s = torch.exp2(e)
    grid = torch.tensor(E2M1[:8], dtype=torch.float64, device=x.device)
    # the nearest magnitude; a tie goes to the smaller one
    mid = (grid[1:] + grid[:-1]) / 2
    near = grid[torch.bucketize((x / s).abs().contiguous(), mid)]
    return (near * x.sign() * s).flatten(-2)


def _wide(fmt, codes, scales):
    """Codes and scales as 64-bit values."""
    lut = torch.tensor(E2M1 if fmt == 7 else [n - 8.0 for n in range(16)], dtype=torch.float64,
                       device=codes.device)
    both = lut[torch.arange(256, device=codes.device).unsqueeze(1) >>
               torch.tensor([0, 4], device=codes.device) & 15]  # [256, 2]
    v = both[codes.int()].flatten(-2)
    s = scales.double() if fmt == 4 else torch.ldexp(torch.ones_like(scales, dtype=torch.float64),
                                                      scales.int() - 127)
    return v * s.repeat_interleave(GROUP[fmt], -1)


def _exact_rope(s):
    c = s["case"]
    r = {}
    for name, lo, h, w in (("q", 0, c["Hq"], s["wq"]), ("k", c["Hq"], c["Hkv"], s["wk"])):
        x = s["qkv"][:, lo:lo + h].double()
        x = x / ((x ** 2).sum(-1, keepdim=True) / c["D"] + 1e-6).sqrt() * w.double()
        j = torch.arange(c["rot"] // 2, device="cuda")
        a, b = (2 * j, 2 * j + 1) if c["interleaved"] else (j, j + c["rot"] // 2)
        z = torch.complex(x[..., a], x[..., b])
        z = z * torch.polar(torch.ones_like(s["freq"]), s["pos"].double()[:, None, None] * s["freq"])
        x[..., a], x[..., b] = z.real, z.imag
        r[name] = x
    return r


def _exact_attn(s):
    c = s["case"]
    G, P = c["Hq"] // c["Hkv"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    score = s["score"].double() if c["weights"] else None
    first = 0
    for b, (n, m) in enumerate(zip(_lens(c), _news(c))):
        at = torch.arange(n, device="cuda")
        page, slot = s["table"][b].long()[at // P], at % P
        for h in range(c["Hkv"]):
            k = _wide(c["fmt"], s["k"][page, h, slot], s["ks"][page, h, slot])
            v = _wide(c["fmt"], s["v"][page, h, slot], s["vs"][page, h, slot])
            q = s["q"][first:first + m, h * G:(h + 1) * G].double()
            x = q.reshape(m * G, -1) @ k.t().contiguous() / math.sqrt(c["D"])
            i = torch.arange(n - m, n, device="cuda").repeat_interleave(G).unsqueeze(1)
            hidden = at > i
            if c["window"]:
                hidden |= at <= i - c["window"]
            p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[first:first + m, h * G:(h + 1) * G] = (p @ v).view(m, G, -1)
            if c["weights"]:
                score[page, h, slot] = p.sum(0)
        first += m
    return {"out": out, "score": score} if c["weights"] else {"out": out}


def _exact_evict(s):
    c = s["case"]
    P = c["page"]
    kept = torch.full(s["kept"].shape, -1, dtype=torch.int32, device="cuda")
    score, k, v, new = s["score"].double(), [], [], []
    for b, n in enumerate(_lens(c)):
        m = min(n, c["keep"])
        new.append(m)
        at = torch.arange(n, device="cuda")
        page, slot = s["table"][b].long()[at // P], at % P
        old, ks, vs = max(0, n - c["recent"]), [], []
        for h in range(c["Hkv"]):
            w = s["score"][page, h, slot]
            by = torch.argsort(w[:old], descending=True, stable=True)[: m - (n - old)]
            i = torch.cat((by.sort().values, at[old:]))
            kept[b, h, :m] = i.int()
            ks.append(_wide(c["fmt"], s["k"][page[i], h, slot[i]], s["ks"][page[i], h, slot[i]]))
            vs.append(_wide(c["fmt"], s["v"][page[i], h, slot[i]], s["vs"][page[i], h, slot[i]]))
            j = torch.arange(m, device="cuda")
            score[s["dst"][b].long()[j // P], h, j % P] = w[i].double()
        k.append(torch.stack(ks, 1))
        v.append(torch.stack(vs, 1))
    return {"kept": kept, "new_lens": torch.tensor(new, dtype=torch.int32, device="cuda"),
            "score": score, "k": torch.cat(k), "v": torch.cat(v)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(s)
    if case["kind"] == "append":
        return {"k": _hold(case["fmt"], s["kn"]), "v": _hold(case["fmt"], s["vn"])}
    return _exact_attn(s) if case["kind"] == "attn" else _exact_evict(s)
