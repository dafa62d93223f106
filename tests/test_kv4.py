"""CPU checks of the 4-bit key/value cache's entry points: geometry, workspace sizes, and every
refusal (arguments are checked before the device is asked for; addresses are never read)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import mvllm_hip
from mvllm_hip import BF16, F32, HipError

A = 1 << 20  # a 16-byte aligned address that no call reads


def cache(fmt=4, n_kv=4, head_dim=128, page=64, n_pages=10, score=A, **kw):
    p = dict(k=A, ks=A, v=A, vs=A) | kw
    return mvllm_hip.KV4(fmt, n_kv, head_dim, page, p["k"], p["ks"], p["v"], p["vs"], score,
                         n_pages=n_pages)


@pytest.mark.parametrize("fmt,n_kv,D,page", [(4, 8, 128, 64), (7, 8, 128, 64), (4, 1, 192, 48),
                                             (7, 3, 64, 16), (7, 16, 256, 1024)])
def test_geometry(fmt, n_kv, D, page):
    total, b = mvllm_hip.kv4_geom(fmt, n_kv, D, page)
    rows = n_kv * page
    assert list(b) == [rows * D // 2, rows * (D // 64 * 4 if fmt == 4 else D // 32)] * 2
    assert total == b.sum()


@pytest.mark.parametrize("bad", [(5, 8, 128, 64), (4, 0, 128, 64), (4, 8, 96, 64), (4, 8, 128, 8),
                                 (4, 8, 128, 24), (7, 8, 128, 1040), (7, 1025, 128, 64)])
def test_geometry_refuses(bad):
    assert mvllm_hip.kv4_geom(*bad)[0] == -1


def test_workspace_sizes():
    f = mvllm_hip.kv4_attention_work
    assert f(8, 128, 32, 4, 4, 1, 100) >= 0
    assert f(8, 128, 32, 4, 4, 1, 100, True) >= 4 * 32 * 4
    assert f(1, 128, 8, 1, 1, 1, 100000) > 0  # one long sequence is split
    for bad in ((8, 128, 30, 4, 4, 1, 100), (8, 96, 32, 4, 4, 1, 100), (8, 128, 32, 0, 4, 1, 100),
                (8, 128, 32, 4, 0, 1, 100), (8, 128, 32, 4, 4, 0, 100), (8, 128, 32, 4, 4, 1, 0),
                (8, 128, 4, 4, 4, 1, 100), (1, 128, 65536, 4, 4, 1, 100),
                (1, 128, 1024, 1 << 21, 1, 1, 100)):
        with pytest.raises(HipError):
            f(*bad)


def refused(match, fn, *args):
    with pytest.raises(HipError, match=match):
        fn(*args)


BAD_CACHES = [dict(fmt=8), dict(n_kv=0), dict(head_dim=32), dict(head_dim=100), dict(page=20),
              dict(page=2048), dict(n_pages=0), dict(k=None), dict(ks=None), dict(v=None),
              dict(vs=None), dict(k=A + 8), dict(vs=A + 4)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches_are_refused(kw):
    c = cache(**kw)
    refused("bad cache", mvllm_hip.kv4_append_dev, c, F32, A, 512, A, 512, 4, A, A, A, 2, 4)
    refused("bad cache", mvllm_hip.kv4_read_dev, c, F32, A, 2 * A, 4, A, A, A, 2, 4)
    refused("bad cache", mvllm_hip.kv4_attention_dev, c, F32, A, 1024, 8, 4, A, A, A, 2, 4, 2, 100,
            0.1, 0, 0, 8 * A, A, 1 << 20)
    refused("bad cache", mvllm_hip.kv4_evict_dev, c, A, A, 2, 4, 200, 64, 8, 2 * A, 1, A, 3 * A)


# n_tok, q_start, lens, table, n_seq, max_pages
BAD_SEQS = [(0, A, A, A, 2, 4), (4, None, A, A, 2, 4), (4, A, None, A, 2, 4), (4, A, A, None, 2, 4),
            (4, A, A, A, 0, 4), (4, A, A, A, 65536, 4), (4, A, A, A, 2, 0), (4, A, A, A, 2, 1 << 25)]


@pytest.mark.parametrize("s", BAD_SEQS)
def test_bad_sequences_are_refused(s):
    c = cache()
    refused("bad sequences", mvllm_hip.kv4_append_dev, c, F32, A, 512, A, 512, *s)
    refused("bad sequences", mvllm_hip.kv4_read_dev, c, F32, A, 2 * A, *s)
    refused("bad sequences", mvllm_hip.kv4_attention_dev, c, F32, A, 1024, 8, *s, 2, 100, 0.1, 0, 0,
            8 * A, A, 1 << 20)


def test_append_and_read_refuse():
    c, s = cache(), (4, A, A, A, 2, 4)
    for dt, k, ks, v, vs in ((2, A, 512, A, 512), (F32, None, 512, A, 512), (F32, A, 512, None, 512),
                             (F32, A + 4, 512, A, 512), (F32, A, 510, A, 512), (BF16, A, 516, A, 512),
                             (F32, A, 512, A, -512)):
        refused("kv4_append_dev", mvllm_hip.kv4_append_dev, c, dt, k, ks, v, vs, *s)
    for dt, k, v in ((3, A, 2 * A), (F32, None, A), (F32, A, None), (F32, A + 2, 2 * A), (F32, A, A),
                     (F32, A, A + 4096)):
        refused("kv4_read_dev", mvllm_hip.kv4_read_dev, c, dt, k, v, *s)


def test_attention_refuses():
    ok = dict(dtype=F32, q=A, q_stride=1024, n_q=8, s=(4, A, A, A, 2, 4), max_new=2, max_len=100,
              scale=0.1, window=0, weights=0, out=8 * A, work=A, work_bytes=1 << 24)

    def call(c=None, **kw):
        a = ok | kw
        mvllm_hip.kv4_attention_dev(c or cache(), a["dtype"], a["q"], a["q_stride"], a["n_q"], *a["s"],
                                    a["max_new"], a["max_len"], a["scale"], a["window"], a["weights"],
                                    a["out"], a["work"], a["work_bytes"])
    for kw in (dict(dtype=2), dict(q=None), dict(q=A + 8), dict(q_stride=1023), dict(n_q=6),
               dict(n_q=2), dict(out=None), dict(out=8 * A + 4), dict(max_new=0), dict(max_len=0),
               dict(max_len=(1 << 30) + 1), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(window=-1), dict(out=A), dict(out=A + 1024), dict(dtype=BF16, q_stride=1028)):
        with pytest.raises(HipError, match="kv4_attention_dev: bad arguments"):
            call(**kw)
    for kw in (dict(weights=3), dict(weights=-1), dict(weights=1, c=cache(score=None))):
        with pytest.raises(HipError, match="weights"):
            call(**kw)
    for kw in (dict(work=None), dict(work_bytes=0), dict(work=A + 8)):
        with pytest.raises(HipError, match="workspace needs"):
            call(weights=1, **kw)


def test_evict_refuses():
    ok = dict(lens=A, table=A, n_seq=2, max_pages=4, max_len=200, keep=64, recent=8, dst=2 * A,
              dst_pages=1, kept=A, new=3 * A)

    def call(c=None, **kw):
        a = ok | kw
        mvllm_hip.kv4_evict_dev(c or cache(), a["lens"], a["table"], a["n_seq"], a["max_pages"],
                                a["max_len"], a["keep"], a["recent"], a["dst"], a["dst_pages"],
                                a["kept"], a["new"])
    for kw in (dict(lens=None), dict(table=None), dict(n_seq=0), dict(n_seq=70000), dict(max_pages=0),
               dict(max_len=0), dict(keep=0), dict(recent=-1), dict(recent=65), dict(dst=None),
               dict(dst=A), dict(dst=A + 16), dict(keep=65), dict(kept=None), dict(new=None),
               dict(new=A), dict(new=A + 4)):
        with pytest.raises(HipError, match="kv4_evict_dev: bad arguments"):
            call(**kw)
    with pytest.raises(HipError, match="score"):
        call(cache(score=None))


@pytest.mark.parametrize("n_kv,D,n_tok", [(1, 64, (1 << 23) + 1), (1024, 256, (1 << 16) + 1)])
def test_launches_past_32_bits_are_refused(n_kv, D, n_tok):
    """More tokens than a launch has threads for."""
    c, big = cache(n_kv=n_kv, head_dim=D), 1 << 50
    s = (n_tok, A, A, A, 2, 4)
    refused("bad sequences", mvllm_hip.kv4_append_dev, c, BF16, A, 0, A, 0, *s)
    refused("bad sequences", mvllm_hip.kv4_read_dev, c, BF16, A, big, *s)
    refused("bad sequences", mvllm_hip.kv4_attention_dev, c, BF16, A, 0, n_kv, *s, 1, 100, 0.1, 0, 0,
            big, A, 1 << 50)


def test_large_sizes_are_refused():
    c = cache()
    refused("bad arguments", mvllm_hip.qk_norm_rope_dev, F32, (1 << 23) + 1, 64, A, 64, 1, A, 64, None,
            0, 0, None, 0, None, None, 0.0, None, None, 0)
    refused("bad arguments", mvllm_hip.kv4_append_dev, c, F32, A, 1 << 40, A, 512, 4, A, A, A, 2, 4)
    refused("bad arguments", mvllm_hip.kv4_evict_dev, c, A, A, 2, 4, 200, (1 << 29) + 1, 8, 2 * A,
            1 << 24, A, 3 * A)
    with pytest.raises(HipError):
        mvllm_hip.kv4_attention_work(1, 64, 1, (1 << 23) + 1, 1, 1, 100)


def test_rope_refuses():
    ok = dict(dtype=F32, T=3, D=128, q=A, qs=1024, nq=8, qo=2 * A, qos=1024, k=A, ks=1024, nk=2,
              ko=3 * A, kos=256, wq=A, wk=A, eps=1e-6, pos=A, freq=A, rot=64)

    def call(**kw):
        a = ok | kw
        mvllm_hip.qk_norm_rope_dev(*a.values())
    for kw in (dict(dtype=2), dict(T=0), dict(D=96), dict(q=None), dict(qo=None), dict(k=None),
               dict(ko=None), dict(q=A + 4), dict(qs=1022), dict(dtype=BF16, qs=1028), dict(qos=960),
               dict(kos=128), dict(nq=-1), dict(nq=0, nk=0), dict(nq=65536), dict(wq=A + 4),
               dict(eps=-1.0), dict(eps=float("nan")), dict(pos=None), dict(rot=0), dict(rot=8),
               dict(rot=72), dict(rot=144)):
        with pytest.raises(HipError, match="qk_norm_rope_dev: bad arguments"):
            call(**kw)


def test_good_arguments_ask_for_the_device():
    """Without a device the same calls fail at the device, not at their arguments."""
    if mvllm_hip.lib().mvllm_hip_available():
        pytest.skip("already initialised in this process")
    c = cache()
    refused("mvllm_hip_init", mvllm_hip.kv4_append_dev, c, F32, A, 512, A, 512, 4, A, A, A, 2, 4)
    refused("mvllm_hip_init", mvllm_hip.kv4_evict_dev, c, A, A, 2, 4, 200, 64, 8, 2 * A, 1, A, 3 * A)
    refused("mvllm_hip_init", mvllm_hip.qk_norm_rope_dev, F32, 3, 128, None, 0, 0, None, 0, A, 1024, 2,
            2 * A, 1024, None, None, 0.0, None, None, 0)


def test_page_reciprocal(tmp_path):
    """The kernels' t / page (a multiplication) against the division, around every page border up
    to 2^30 tokens for all 64 page sizes."""
    src = tmp_path / "rcp.cpp"
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "micro-vllm_amd", "csrc", "kv4_common.h")).read()
    fn = text[text.index("inline uint32_t kv4_page_rcp"):]
    fn = fn[:fn.index("}") + 1]
    src.write_text("""#include <cstdint>
#include <cstdio>
%s
int main() {
    for (uint32_t page = 16; page <= 1024; page += 16) {
        const uint32_t m = kv4_page_rcp((int)page);
        for (uint64_t k = 0; k * page <= (1ull << 30); k += 1 + k / 997)
            for (int64_t d = -17; d <= 17; ++d) {
                const int64_t t = (int64_t)(k * page) + d;
                if (t < 0 || t >= (1 << 30)) continue;
                const uint32_t u = (uint32_t)t >> 4;
                const uint32_t q = m ? (uint32_t)(((uint64_t)u * m) >> 32) : u;
                if (q != (uint32_t)t / page) { printf("%%u %%lld\\n", page, (long long)t); return 1; }
            }
    }
    return 0;
}
""" % fn)
    exe = tmp_path / "rcp"
    subprocess.run(["g++", "-O2", "-o", str(exe), str(src)], check=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True)
    assert p.returncode == 0, p.stdout


def test_structure_matches_header():
    """The binding's structure has the header's size and field offsets."""
    d = mvllm_hip.KV4(7, 1, 2, 3, 4, 5, 6, 7, 8, n_pages=9).desc
    assert C.sizeof(d) == 5 * 8 + 5 * 4 + 4
    assert np.frombuffer(bytes(d), np.int32)[10:15].tolist() == [7, 1, 2, 3, 9]
