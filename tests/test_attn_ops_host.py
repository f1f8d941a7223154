"""The attention operators without a GPU: refusals, the rotary tables and the page-table arithmetic."""
import ctypes as C
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def cw():
    import cwen_b200
    from cwen_b200 import build
    build.build()
    cwen_b200.lib().cwen_cuda_shutdown()
    return cwen_b200


P = 1 << 20  # stands for a device pointer: nothing is read without an engine


def _kv(cw, **kw):
    d = dict(type=30, n_layer=2, n_pages=8, page_size=16, n_kv=4, head_dim=128, k=P, v=P)
    d.update(kw)
    return cw.Kv(*[d[n] for n, _ in cw.Kv._fields_])


def _rope(cw, n_rot=64, half=0, base=1e4, factor=1.0, ctx=0.0, fast=0.0, slow=0.0):
    r = cw.Rope()
    return cw.lib().cwen_rope_init(r, n_rot, half, base, factor, ctx, fast, slow), r


@pytest.mark.parametrize("kw", [dict(n_rot=0), dict(n_rot=-2), dict(n_rot=7), dict(n_rot=258), dict(base=0.0),
                                dict(base=-1.0), dict(base=math.nan), dict(base=math.inf), dict(factor=0.0),
                                dict(factor=math.nan), dict(factor=math.inf), dict(fast=1.0, slow=1.0, ctx=10.0),
                                dict(fast=32.0, slow=1.0, ctx=0.0), dict(fast=1.0, slow=32.0, ctx=10.0),
                                dict(fast=32.0, slow=-1.0, ctx=10.0), dict(fast=32.0, slow=1.0, ctx=10.0, factor=0.5),
                                dict(fast=math.nan, slow=1.0, ctx=10.0), dict(fast=32.0, slow=1.0, ctx=math.nan)])
def test_rope_init_refuses(cw, kw):
    rc, _ = _rope(cw, **kw)
    assert rc == -1 and b"cwen_rope_init" in cw.lib().cwen_cuda_last_error()
    assert cw.lib().cwen_rope_init(None, 64, 0, 1e4, 1.0, 0.0, 0.0, 0.0) == -1


@pytest.mark.parametrize("n_rot", [2, 64, 100, 256])
def test_rope_init_tables(cw, n_rot):
    """turn[] is base^(-2i/n) / 2 pi; linear scaling divides it; by parts, pairs that turn often keep their turn
    and slow ones are divided.  pow, the division and the blend round a few times each: 8 half steps of 64 bits."""
    i = np.arange(n_rot // 2)
    plain = 1e6 ** (-2.0 * i / n_rot) / (2 * math.pi)
    rc, r = _rope(cw, n_rot, 1, 1e6)
    assert rc == 0 and (r.n_rot, r.half, r.mscale) == (n_rot, 1, 1.0)
    np.testing.assert_allclose(r.turn[:n_rot // 2], plain, rtol=16 * 2 ** -53)
    assert not any(r.turn[n_rot // 2:])
    rc, r = _rope(cw, n_rot, 0, 1e6, factor=4.0)
    np.testing.assert_allclose(r.turn[:n_rot // 2], plain / 4, rtol=16 * 2 ** -53)
    rc, r = _rope(cw, n_rot, 0, 1e6, factor=8.0, ctx=4096.0, fast=32.0, slow=1.0)
    keep = np.clip((plain * 4096 - 1) / 31, 0, 1)
    np.testing.assert_allclose(r.turn[:n_rot // 2], plain * (keep + (1 - keep) / 8), rtol=64 * 2 ** -53)
    assert r.mscale == np.float32(0.1 * math.log(8) + 1)
    if n_rot >= 64:
        assert keep[0] == 1 and keep[-1] == 0 and ((keep > 0) & (keep < 1)).any()


KV_BAD = [dict(type=2), dict(type=8), dict(n_layer=0), dict(n_layer=1025), dict(n_pages=0), dict(page_size=0),
          dict(page_size=65537), dict(n_kv=0), dict(n_kv=257), dict(head_dim=4), dict(head_dim=130),
          dict(head_dim=520), dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 2)]


def _calls(cw, kv):
    """Each call with fit arguments: (function, list of arguments, place of each name)."""
    L, (_, r) = cw.lib(), _rope(cw)
    return {
        "rope": (L.cwen_cuda_rope, dict(r=r, type=30, n_rows=3, n_head=4, head_dim=128, x=P, xrow=512, xhead=128, pos=P,
                                        inverse=0, y=2 * P, yrow=512, yhead=128, stream=None)),
        "append": (L.cwen_cuda_kv_append, dict(c=kv, layer=1, table=P, table_stride=2, n_seq=3, type=30, n_rows=5, k=P,
                                               krow=512, khead=128, v=P, vrow=512, vhead=128, seq=P, slot=P, r=r,
                                               pos=None, stream=None)),
        "compact": (L.cwen_cuda_kv_compact, dict(c=kv, table=P, table_stride=2, n_seq=3, len=P, keep=P, len_out=2 * P,
                                                 stream=None)),
        "prompt": (L.cwen_cuda_attn_prompt, dict(type=30, n_seq=2, cu=P, n_rows=9, n_head=8, n_kv=4, head_dim=128,
                                                 scale=0.1, q=P, qrow=1024, qhead=128, k=P, krow=512, khead=128, v=P,
                                                 vrow=512, vhead=128, out=P, orow=1024, ohead=128, stream=None)),
        "tree": (L.cwen_cuda_attn_tree, dict(c=kv, layer=0, table=P, table_stride=4, n_seq=2, len=P, max_len=60, T=9,
                                             n_node=None, mask=None, n_head=8, scale=0.1, q=P, qrow=1024, qhead=128,
                                             out=P, orow=1024, ohead=128, ws=P, ws_bytes=1 << 40, stream=None)),
    }


def _rc(cw, name, kv=None, **kw):
    f, args = _calls(cw, kv or _kv(cw))[name]
    assert set(kw) <= set(args)
    args.update(kw)
    return f(*args.values())


@pytest.mark.parametrize("name", ["rope", "append", "compact", "prompt", "tree"])
def test_fit_arguments_need_an_engine(cw, name):
    assert _rc(cw, name) == -4
    assert cw.lib().cwen_cuda_attn_status(None) == -4


@pytest.mark.parametrize("name", ["append", "compact", "tree"])
@pytest.mark.parametrize("bad", KV_BAD, ids=lambda d: ",".join("%s=%s" % kv for kv in d.items()))
def test_cache_descriptions_refused(cw, name, bad):
    assert _rc(cw, name, _kv(cw, **bad)) == -1
    assert _rc(cw, name, None, c=None) == -1


@pytest.mark.parametrize("name,kw", [
    ("rope", dict(r=None)), ("rope", dict(type=2)), ("rope", dict(n_rows=-1)), ("rope", dict(n_head=0)),
    ("rope", dict(n_head=4097)), ("rope", dict(head_dim=32)), ("rope", dict(head_dim=514)), ("rope", dict(x=None)),
    ("rope", dict(y=None)), ("rope", dict(pos=None)), ("rope", dict(y=P, yrow=1024)), ("rope", dict(y=P, yhead=256)),
    ("append", dict(layer=2)), ("append", dict(layer=-1)), ("append", dict(table=None)),
    ("append", dict(table_stride=0)), ("append", dict(n_seq=0)), ("append", dict(type=1)), ("append", dict(n_rows=-1)),
    ("append", dict(k=None)), ("append", dict(v=None)), ("append", dict(seq=None)), ("append", dict(slot=None)),
    ("compact", dict(table=None)), ("compact", dict(table_stride=0)), ("compact", dict(n_seq=-1)),
    ("compact", dict(len=None)), ("compact", dict(keep=None)), ("compact", dict(len_out=P)),
    ("prompt", dict(type=8)), ("prompt", dict(n_seq=-1)), ("prompt", dict(n_seq=65536)), ("prompt", dict(n_rows=-1)),
    ("prompt", dict(n_head=9)), ("prompt", dict(n_head=2)), ("prompt", dict(n_kv=0)), ("prompt", dict(head_dim=80)),
    ("prompt", dict(head_dim=512)), ("prompt", dict(cu=None)), ("prompt", dict(q=None)), ("prompt", dict(k=None)),
    ("prompt", dict(v=None)), ("prompt", dict(out=None)),
    ("tree", dict(layer=2)), ("tree", dict(table=None)), ("tree", dict(table_stride=0)), ("tree", dict(n_seq=-1)),
    ("tree", dict(n_seq=65536)), ("tree", dict(len=None)), ("tree", dict(T=0)), ("tree", dict(T=65)),
    ("tree", dict(max_len=0)), ("tree", dict(max_len=65)), ("tree", dict(n_head=6)), ("tree", dict(q=None)),
    ("tree", dict(out=None)), ("tree", dict(ws=None)), ("tree", dict(ws=P + 4)), ("tree", dict(ws_bytes=0)),
], ids=str)
def test_arguments_refused(cw, name, kw):
    assert _rc(cw, name, **kw) == -1
    fn = {"rope": b"cwen_cuda_rope", "append": b"cwen_cuda_kv_append", "compact": b"cwen_cuda_kv_compact",
          "prompt": b"cwen_cuda_attn_prompt", "tree": b"cwen_cuda_attn_tree"}[name]
    assert cw.lib().cwen_cuda_last_error().startswith(fn)


def test_attention_head_dims(cw):
    """The cache keeps any head_dim that is a multiple of 8; attention takes 64, 128 and 256."""
    assert _rc(cw, "append", _kv(cw, head_dim=80)) == -4
    assert _rc(cw, "tree", _kv(cw, head_dim=80)) == -1
    _, r = _rope(cw, 96)
    assert _rc(cw, "append", _kv(cw, head_dim=80), r=r) == -1


PAGES = r"""
#include <stdio.h>
#include "kvpage.h"
int main(void) {
  int table[4] = {2, -1, 5, 1};
  long long slot;
  int stride, n_pages, page;
  while (scanf("%d %d %d %lld", &stride, &n_pages, &page, &slot) == 4)
    printf("%lld\n", (long long)cwp_row(table, stride, n_pages, page, slot));
  return 0;
}
"""


def test_page_lookup_never_leaves_the_pool(tmp_path):
    """Every lookup that the kernels make goes through cwp_row: bad slots and page ids give -1, good ones the row."""
    (tmp_path / "p.c").write_text(PAGES)
    subprocess.check_call(["gcc", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", "-I",
                           str(ROOT / "cwen_b200" / "csrc"), "-o", str(tmp_path / "p"), str(tmp_path / "p.c")])
    table, ask, want = [2, -1, 5, 1], [], []
    for stride in (1, 2, 4):
        for n_pages in (1, 2, 3, 5, 6):
            for page in (1, 5, 16, 65536):
                for slot in (-1, -2 ** 31, 0, page - 1, page, 2 * page - 1, 2 * page, 3 * page + page // 2, 4 * page - 1,
                             4 * page, 2 ** 31 - 1, 2 ** 31 + 63, 2 ** 40):
                    ask.append("%d %d %d %d" % (stride, n_pages, page, slot))
                    p = slot // page
                    ok = 0 <= slot and p < stride and 0 <= table[p] < n_pages
                    want.append(table[p] * page + slot % page if ok else -1)
    out = subprocess.run([str(tmp_path / "p")], input="\n".join(ask), capture_output=True, text=True, check=True).stdout
    assert [int(x) for x in out.split()] == want


def test_pool_rows_pass_32_bits(tmp_path):
    """A pool of more than 2^31 elements: the row number times its elements is computed in 64 bits."""
    (tmp_path / "q.c").write_text('#include <stdio.h>\n#include "kvpage.h"\nint main(void) { int t[1] = {2000000};'
                                  'printf("%lld", (long long)(cwp_row(t, 1, 2000001, 64, 63) * 4 * 256)); return 0; }')
    subprocess.check_call(["gcc", "-Wall", "-Werror", "-I", str(ROOT / "cwen_b200" / "csrc"), "-o", str(tmp_path / "q"),
                           str(tmp_path / "q.c")])
    assert int(subprocess.check_output([str(tmp_path / "q")])) == (2000000 * 64 + 63) * 1024


def test_struct_layout(cw, tmp_path):
    """The Python structs are the header's (checked with the C compiler)."""
    src = ('#include <stdio.h>\n#include <stddef.h>\n#include "cwen_cuda.h"\nint main(void) { printf("%zu %zu %zu %zu",'
           'sizeof(cwen_rope), offsetof(cwen_rope, turn), sizeof(cwen_kv), offsetof(cwen_kv, v)); return 0; }')
    r = subprocess.run(["gcc", "-x", "c", "-", "-I", str(ROOT / "include"), "-o", str(tmp_path / "layout")], input=src,
                       text=True, capture_output=True)
    assert r.returncode == 0, r.stderr
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "layout")]).split()]
    assert got == [C.sizeof(cw.Rope), cw.Rope.turn.offset, C.sizeof(cw.Kv), cw.Kv.v.offset]
