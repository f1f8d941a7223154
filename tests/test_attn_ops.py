"""The attention operators on the GPU against plain forms in 64 bits: types, layouts, odd and ragged sizes, strides,
masks that leave a row empty, non-finite values in masked places, bad page ids, streams and graphs, and the
operators one after another as a serving loop uses them."""
import math
import random

import pytest
import torch

from attn_ops_util import DT, U, Cache, attn_ref, close, ptr, rope_ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = 0, 1, 30


@pytest.fixture(scope="module")
def cw():
    import cwen_b200
    from cwen_b200 import build
    build.build()
    L = cwen_b200.lib()
    cwen_b200.check(L.cwen_cuda_init(0, 64, 16), "init")
    yield cwen_b200
    L.cwen_cuda_shutdown()


def stream():
    return torch.cuda.current_stream().cuda_stream or 1


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, t=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(DT[t])


def rows_of(g, n, heads, dim, t, row=None, head=None, offset=0, scale=1.0):
    """[n, heads, dim] values inside a larger NaN-filled buffer with the given strides: (view, row, head)."""
    head = head or dim
    row = row or heads * head
    buf = torch.full((offset + max(n, 1) * row + heads * head + dim,), math.nan, device="cuda", dtype=DT[t])
    x = torch.as_strided(buf, (n, heads, dim), (row, head, 1), offset)
    x.copy_(normal(g, n, heads, dim, t=t, scale=scale))
    return x, row, head


def status(cw):
    return cw.lib().cwen_cuda_attn_status(stream())


# ------------------------------------------------------------------ rope
def call_rope(cw, r, t, x, xs, pos, inverse, y, ys, st=None):
    cw.check(cw.lib().cwen_cuda_rope(r, t, x.shape[0], x.shape[1], x.shape[2], ptr(x), *xs, ptr(pos), inverse, ptr(y),
                                     *ys, st or stream()), "rope")


def rope_table(cw, n_rot, half=0, base=1e4, factor=1.0, ramp=False):
    r = cw.Rope()
    cw.check(cw.lib().cwen_rope_init(r, n_rot, half, base, factor, 4096.0, 32.0 * ramp, 1.0 * ramp))
    return r, torch.tensor(r.turn[:n_rot // 2], dtype=torch.float64, device="cuda")


def check_rope(got, x, pos, r, turn, sign, t):
    """cos and sin are off by at most 2^-23 + pi 2^-24 (a reduced turn's rounding to 32 bits, then two units of the
    function), the scale's product, the two products and the sum round once each: 2^-21 of |x0| + |x1|."""
    y, size = rope_ref(x.double(), pos, turn, r.mscale, r.half, sign)
    tol = size * 2.0 ** -21 + U[t] * 1.05 * y.abs() + (2.0 ** -25 if t == F16 else 0.0)
    assert ((got.double() - y).abs() <= tol).all(), float(((got.double() - y).abs() - tol).max())


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("rows,heads,dim,n_rot", [(1, 1, 2, 2), (9, 24, 256, 64), (37, 3, 128, 128), (5, 2, 80, 20),
                                                  (300, 5, 64, 32), (2, 7, 30, 14), (1, 64, 512, 256), (1000, 1, 8, 8)])
def test_rope(cw, t, half, rows, heads, dim, n_rot):
    g = gen(rows * 7 + dim)
    r, turn = rope_table(cw, n_rot, half)
    x = normal(g, rows, heads, dim, t=t)
    pos = torch.randint(0, 1 << 17, (rows,), generator=g, device="cuda", dtype=torch.int32)
    y = torch.full_like(x, math.nan)
    call_rope(cw, r, t, x, (heads * dim, dim), pos, 0, y, (heads * dim, dim))
    check_rope(y, x, pos, r, turn, 1.0, t)
    assert torch.equal(y[..., n_rot:], x[..., n_rot:])
    call_rope(cw, r, t, x, (heads * dim, dim), pos, 0, x, (heads * dim, dim))  # in place: the same bits
    assert torch.equal(x, y)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("row,head,offset", [(5000, 512, 0), (1031, 130, 3), (4096, 256, 1), (1, 700, 0)])
def test_rope_strides(cw, t, half, row, head, offset):
    """Rows inside wider rows (a projection's q and gate side by side), odd strides and bases, heads outside rows."""
    g = gen(3)
    n, heads, dim, n_rot = 6, 4, 128, 64
    if row == 1:  # head-major: [heads][rows][dim]
        row, head = dim, n * dim
    x, _, _ = rows_of(g, n, heads, dim, t, row, head, offset)
    keep = x.clone()
    out = torch.full((offset + n * 2048 + 5,), math.nan, device="cuda", dtype=DT[t])
    y = torch.as_strided(out, (n, heads, dim), (heads * 131, 131, 1), offset)
    r, turn = rope_table(cw, n_rot, half)
    pos = torch.arange(n, device="cuda", dtype=torch.int32) + 77
    call_rope(cw, r, t, x, (row, head), pos, 0, y, (heads * 131, 131))
    check_rope(y, keep, pos, r, turn, 1.0, t)
    touched = torch.zeros_like(out, dtype=torch.bool)
    torch.as_strided(touched, (n, heads, dim), (heads * 131, 131, 1), offset).fill_(True)
    assert out[~touched].isnan().all()


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("ramp,factor", [(False, 1.0), (False, 8.0), (True, 8.0), (True, 1.0)])
def test_rope_far_positions_and_scaling(cw, half, ramp, factor):
    g = gen(5)
    r, turn = rope_table(cw, 128, half, 1e6, factor, ramp)
    pos = torch.tensor([0, 1, -1, 65535, 1000003, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31], device="cuda", dtype=torch.int32)
    x = normal(g, len(pos), 3, 128)
    y = torch.empty_like(x)
    call_rope(cw, r, F32, x, (384, 128), pos, 0, y, (384, 128))
    check_rope(y, x, pos, r, turn, 1.0, F32)
    if not ramp:
        assert torch.equal(y[0], x[0])


@pytest.mark.parametrize("half", [0, 1])
def test_rope_inverse_is_the_gradient(cw, half):
    """The rotation is linear, so its gradient is its transpose: against autograd of the formula and differences."""
    g = gen(8)
    r, turn = rope_table(cw, 32, half, 1e4, 4.0, True)
    pos = torch.tensor([3, 900, 4095], device="cuda", dtype=torch.int32)
    x = normal(g, 3, 2, 64).double().requires_grad_()
    w = normal(g, 3, 2, 64)
    y, _ = rope_ref(x, pos, turn, r.mscale, half)
    (dx,) = torch.autograd.grad((y * w.double()).sum(), x)
    got = torch.empty_like(w)
    call_rope(cw, r, F32, w, (128, 64), pos, 1, got, (128, 64))
    check_rope(got, w, pos, r, turn, -1.0, F32)
    assert (got.double() - dx).abs().max() <= 2.0 ** -20 * w.abs().max() * 2
    # differences: L(x + h e) - L(x) = h dx for a linear map, through the operator itself
    xf, h = x.detach().float(), 0.25
    base, moved = torch.empty_like(xf), torch.empty_like(xf)
    call_rope(cw, r, F32, xf, (128, 64), pos, 0, base, (128, 64))
    for i in (0, 5, 17, 40):
        xe = xf.clone()
        xe[1, 1, i] += h
        call_rope(cw, r, F32, xe, (128, 64), pos, 0, moved, (128, 64))
        d = ((moved.double() - base.double()) * w.double()).sum() / h
        # each of the (at most) two differing results is off by 2^-20 of its size, over h
        assert abs(d - dx[1, 1, i]) <= 4 * 2.0 ** -20 * xe.abs().max() * w.abs().max() * 2 / h


def test_rope_nothing_to_do(cw):
    r, _ = rope_table(cw, 32)
    x = torch.zeros(4, device="cuda")
    assert cw.lib().cwen_cuda_rope(r, F32, 0, 1, 64, ptr(x), 64, 64, ptr(x), 0, ptr(x), 64, 64, stream()) == 0


def test_rope_keeps_non_finite_values_in_their_pair(cw):
    r, _ = rope_table(cw, 8, 1)
    x = torch.ones(1, 2, 64, device="cuda")
    x[0, 0, 1], x[0, 1, 20] = math.inf, math.nan
    pos = torch.tensor([3], device="cuda", dtype=torch.int32)
    y = torch.empty_like(x)
    call_rope(cw, r, F32, x, (128, 64), pos, 0, y, (128, 64))
    bad = ~y.isfinite()
    assert bad.nonzero().tolist() == [[0, 0, 1], [0, 0, 5], [0, 1, 20]]


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("src,t", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("page,n_kv,dim,n_rot,half", [(16, 4, 256, 64, 0), (1, 1, 64, 64, 1), (5, 3, 128, 20, 1),
                                                      (64, 2, 80, 0, 0), (24, 8, 128, 128, 0), (7, 2, 8, 6, 0)])
def test_append(cw, src, t, page, n_kv, dim, n_rot, half):
    """Every row lands in its place, rounded once; padding rows and every other place stay as they were."""
    g, rng = gen(page), random.Random(page)
    c = Cache(cw, t, 5, 70, page, n_kv, dim, layers=3, seed=page)
    where = [(s, j) for s in range(5) for j in range(70)]
    rng.shuffle(where)
    where = where[:93]
    seq, slot = ([p[i] for p in where] for i in (0, 1))
    for i in (4, 60):
        seq[i] = -1 - i
    k, krow, khead = rows_of(g, 93, n_kv, dim, src, n_kv * dim + 16, dim)
    v, vrow, vhead = rows_of(g, 93, n_kv, dim, src, n_kv * dim * 2 + 3 * (page == 5), dim)
    r, turn = rope_table(cw, n_rot, half) if n_rot else (None, None)
    ints = [torch.tensor(x, device="cuda", dtype=torch.int32) for x in (seq, slot, [9 + 3 * j for j in slot])]
    kc, vc = c.k.clone(), c.v.clone()
    cw.check(cw.lib().cwen_cuda_kv_append(c.desc, 1, ptr(c.table), c.stride, 5, src, 93, ptr(k), krow, khead, ptr(v), vrow,
                                          vhead, ptr(ints[0]), ptr(ints[1]), r, ptr(ints[2]) if n_rot else None, stream()))
    live = [i for i in range(93) if seq[i] >= 0]
    at = torch.stack([c.rows(seq[i], [slot[i]])[0] for i in live])
    got_k, got_v = c.flat("k", 1)[at], c.flat("v", 1)[at]
    assert torch.equal(got_v, v[live].float().to(DT[t]))
    if n_rot:
        check_rope(got_k, k[live], ints[2][live], r, turn, 1.0, t)
    else:
        assert torch.equal(got_k, k[live].float().to(DT[t]))
    for now, before in ((c.k, kc), (c.v, vc)):
        flat, old = now.view(3, -1, n_kv, dim), before.view(3, -1, n_kv, dim)
        rest = torch.ones(flat.shape[1], dtype=torch.bool, device="cuda")
        rest[at] = False
        assert flat[1][rest].isnan().all() and flat[0].isnan().all() and flat[2].isnan().all() and old.isnan().all()
    assert status(cw) == 0


def test_append_position_defaults_to_the_slot(cw):
    g = gen(1)
    r, turn = rope_table(cw, 64, 1)
    c = Cache(cw, F32, 1, 40, 16, 2, 64)
    k = normal(g, 40, 2, 64)
    seq, slot = torch.zeros(40, device="cuda", dtype=torch.int32), torch.arange(40, device="cuda", dtype=torch.int32)
    cw.check(cw.lib().cwen_cuda_kv_append(c.desc, 0, ptr(c.table), c.stride, 1, F32, 40, ptr(k), 128, 64, ptr(k), 128, 64,
                                          ptr(seq), ptr(slot), r, None, stream()))
    check_rope(c.flat("k")[c.rows(0, range(40))], k, slot, r, turn, 1.0, F32)


def test_append_out_of_range_is_left_out_and_reported(cw):
    g = gen(2)
    c = Cache(cw, BF16, 2, 32, 16, 2, 64)
    c.table[1, 1] = c.desc.n_pages  # one past the pool
    c.table[0, 1] = -1
    k = normal(g, 8, 2, 64, t=BF16)
    seq = torch.tensor([0, 2, 1, 0, 0, 1, 1, 1 << 30], device="cuda", dtype=torch.int32)
    slot = torch.tensor([3, 0, 17, 16, 32, -1, 2, 0], device="cuda", dtype=torch.int32)
    cw.check(cw.lib().cwen_cuda_kv_append(c.desc, 0, ptr(c.table), c.stride, 2, BF16, 8, ptr(k), 128, 64, ptr(k), 128, 64,
                                          ptr(seq), ptr(slot), None, None, stream()))
    assert status(cw) == -5 and b"out of range" in cw.lib().cwen_cuda_last_error()
    assert status(cw) == 0  # cleared
    good = torch.stack([c.rows(0, [3])[0], c.rows(1, [2])[0]])
    assert torch.equal(c.flat("k")[good], k[[0, 6]])
    assert int((~c.k.isnan()).sum()) == 2 * 2 * 64


# ------------------------------------------------------------------ compact
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("page,n_kv,dim,layers", [(1, 1, 8, 1), (16, 4, 256, 3), (5, 3, 80, 2), (64, 2, 64, 16)])
def test_compact(cw, t, page, n_kv, dim, layers):
    """Against moves made one after another; the other places keep their bits."""
    rng = random.Random(page * 100 + dim)
    keeps = [0, 1, 2, 1 << 63, (1 << 64) - 1, (1 << 64) - 2, 0b1011001, 0xaaaaaaaaaaaaaaaa,
             sum(1 << u for u in range(64) if rng.random() < 0.3), (1 << 63) | 1 << 31 | 1 << 32]
    n = len(keeps)
    c = Cache(cw, t, n, 100, page, n_kv, dim, layers, seed=dim)
    g = gen(dim)
    c.k.copy_(normal(g, *c.k.shape))
    c.v.copy_(normal(g, *c.v.shape))
    lens = [rng.randrange(0, 36) for _ in range(n)]
    want = {}
    for w in ("k", "v"):
        x = (c.k if w == "k" else c.v).clone().view(layers, -1, n_kv, dim)
        for s in range(n):
            for i, u in enumerate([u for u in range(64) if keeps[s] >> u & 1]):
                x[:, c.rows(s, [lens[s] + i])] = x[:, c.rows(s, [lens[s] + u])].clone()
        want[w] = x
    ln = torch.tensor(lens, device="cuda", dtype=torch.int32)
    kp = torch.tensor([m - (1 << 64) if m >> 63 else m for m in keeps], device="cuda")
    out = torch.full_like(ln, -7)
    cw.check(cw.lib().cwen_cuda_kv_compact(c.desc, ptr(c.table), c.stride, n, ptr(ln), ptr(kp), ptr(out), stream()))
    assert torch.equal(c.k.view_as(want["k"]), want["k"]) and torch.equal(c.v.view_as(want["v"]), want["v"])
    assert out.tolist() == [a + bin(m).count("1") for a, m in zip(lens, keeps)] and ln.tolist() == lens
    assert status(cw) == 0


def test_compact_bad_pages_are_left_out(cw):
    c = Cache(cw, F32, 3, 64, 16, 1, 8)
    g = gen(4)
    c.k.copy_(normal(g, *c.k.shape))
    c.v.copy_(c.k)
    before = c.k.clone()
    c.table[0, 1] = 10 ** 6
    c.table[1, 0] = -3
    ln = torch.tensor([10, 10, -4], device="cuda", dtype=torch.int32)
    kp = torch.tensor([1 << 10, 1 << 10, 1 << 10], device="cuda")  # 20 -> 10
    cw.check(cw.lib().cwen_cuda_kv_compact(c.desc, ptr(c.table), c.stride, 3, ptr(ln), ptr(kp), None, stream()))
    assert status(cw) == -5
    assert torch.equal(c.k, before) and torch.equal(c.v, before)


# ------------------------------------------------------------------ prompt attention
HEADS = [(24, 4, 256), (8, 8, 64), (14, 2, 64), (4, 1, 128), (6, 2, 128), (3, 1, 256)]


def run_prompt(cw, t, lens, nh, nkv, hd, scale=None, q=None, k=None, v=None, o=None, st=None, n_rows=None, cu=None):
    (q, qr, qh), (k, kr, kh), (v, vr, vh), (o, orow, oh) = q, k, v, o
    if cu is None:
        cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], device="cuda", dtype=torch.int32)
    cw.check(cw.lib().cwen_cuda_attn_prompt(t, len(lens), ptr(cu), n_rows if n_rows is not None else q.shape[0], nh, nkv, hd,
                                            scale if scale is not None else hd ** -0.5, ptr(q), qr, qh, ptr(k), kr, kh,
                                            ptr(v), vr, vh, ptr(o), orow, oh, st or stream()), "prompt")
    return o


def check_prompt(got, t, lens, nh, nkv, q, k, v, scale, first=0):
    at = first
    for n in lens:
        seen = torch.ones(n, n, device="cuda", dtype=torch.bool).tril()
        for h in range(nh):
            out, bound, av = attn_ref(q[at:at + n, h].double(), k[at:at + n, h // (nh // nkv)].double(),
                                      v[at:at + n, h // (nh // nkv)].double(), seen, scale)
            close(got[at:at + n, h], out, bound, av, t)
        at += n


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("lens", [[1], [2, 0, 3], [63, 1, 65, 64], [127, 129, 128], [0, 0, 300, 0], [517]], ids=str)
def test_prompt(cw, t, nh, nkv, hd, lens):
    g, n = gen(sum(lens) + hd), sum(lens)
    q, k, v = (rows_of(g, n, h, hd, t, scale=s) for h, s in ((nh, 2.0), (nkv, 1.0), (nkv, 1.0)))
    o = rows_of(g, n, nh, hd, t)
    o[0].fill_(math.nan)
    run_prompt(cw, t, lens, nh, nkv, hd, None, q, k, v, o)
    check_prompt(o[0], t, lens, nh, nkv, q[0], k[0], v[0], hd ** -0.5)
    assert status(cw) == 0


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("row,head,offset", [(8 * 512, 512, 0), (0, 0, 1), (0, 129, 0), (0, 136, 8), (-1, -1, 0)])
def test_prompt_strides(cw, t, row, head, offset):
    """q with its gate beside it, odd strides and bases (no 16-byte alignment), head-major rows."""
    g, lens, nh, nkv, hd = gen(12), [70, 133], 8, 2, 128
    n = sum(lens)
    bufs = []
    for h in (nh, nkv, nkv, nh):
        r, e = (row or None, head or None)
        if row == -1:
            r, e = hd, n * hd
        bufs.append(rows_of(g, n, h, hd, t, r if not (r and h == nkv and row > 0) else nkv * 512, e, offset))
    before = bufs[3][0].clone()
    assert before.isfinite().all()
    run_prompt(cw, t, lens, nh, nkv, hd, None, *bufs)
    check_prompt(bufs[3][0], t, lens, nh, nkv, bufs[0][0], bufs[1][0], bufs[2][0], hd ** -0.5)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 256])
def test_prompt_rows_outside_the_sequences_stay(cw, t, hd):
    g, lens, nh, nkv = gen(2), [20, 150], 4, 2
    n = 5 + sum(lens) + 9
    q, k, v, o = (rows_of(g, n, h, hd, t) for h in (nh, nkv, nkv, nh))
    for x in (q, k, v):
        x[0][:5], x[0][-9:] = math.nan, math.inf
    o[0].fill_(7.0)
    cu = torch.tensor([5, 25, 175], device="cuda", dtype=torch.int32)
    run_prompt(cw, t, lens, nh, nkv, hd, None, q, k, v, o, cu=cu)
    assert (o[0][:5] == 7).all() and (o[0][-9:] == 7).all()
    check_prompt(o[0], t, lens, nh, nkv, q[0], k[0], v[0], hd ** -0.5, first=5)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prompt_non_finite_values_reach_only_rows_that_see_them(cw, t, hd, what, bad):
    """Two sequences; place 40 of the first and place 100 of the second are poisoned: rows before do not change."""
    g, lens, nh, nkv = gen(9), [90, 200], 4, 2
    n = sum(lens)
    q, k, v, o = (rows_of(g, n, h, hd, t) for h in (nh, nkv, nkv, nh))
    run_prompt(cw, t, lens, nh, nkv, hd, None, q, k, v, o)
    clean = o[0].clone()
    x = k if what == "k" else v
    kc, vc = k[0].clone(), v[0].clone()
    x[0][40, 0, 3] = bad
    x[0][90 + 100, 1, hd - 1] = bad
    run_prompt(cw, t, lens, nh, nkv, hd, None, q, k, v, o)
    hit = torch.zeros(n, nh, hd, dtype=torch.bool, device="cuda")
    if what == "v":  # the poisoned dim only, and there always
        hit[40:90, :2, 3] = hit[190:, 2:, hd - 1] = True
        a = o[0][hit].float()
        assert a.isnan().all() if bad != bad else (a == bad).all()
    else:
        hit[40:90, :2] = hit[190:, 2:] = True
        if bad != bad:
            assert o[0][hit].isnan().all()
    # all else is what it is without the poison, within the operator's own bounds (the places in question are taken
    # from the clean run, which is held to the same bounds)
    check_prompt(clean, t, lens, nh, nkv, q[0], kc, vc, hd ** -0.5)
    check_prompt(torch.where(hit, clean, o[0]), t, lens, nh, nkv, q[0], kc, vc, hd ** -0.5)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 30.0])
def test_prompt_scales(cw, t, scale):
    """Equal weights, sharp and inverted softmax; keys whose scores grow along the row move the maximum each tile."""
    g, lens, nh, nkv, hd = gen(6), [400], 2, 1, 64
    q, k, v, o = (rows_of(g, 400, h, hd, t, scale=0.5) for h in (nh, nkv, nkv, nh))
    k[0].mul_(torch.linspace(0.02, 1.0, 400, device="cuda")[:, None, None].to(DT[t]))
    run_prompt(cw, t, lens, nh, nkv, hd, scale, q, k, v, o)
    check_prompt(o[0], t, lens, nh, nkv, q[0], k[0], v[0], scale)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_maximum_jumps(cw, t, hd):
    """The running maximum leaps late in the row (by far more than the weights' range): earlier sums vanish."""
    g, n = gen(7), 700
    q, k, v, o = (rows_of(g, n, 1, hd, t) for _ in range(4))
    q[0].fill_(1.0)
    k[0].mul_(0.01)
    for at, size in ((130, 1.0), (300, 4.0), (650, 12.0)):
        k[0][at] = size
    run_prompt(cw, t, [n], 1, 1, hd, 0.25, q, k, v, o)
    check_prompt(o[0], t, [n], 1, 1, q[0], k[0], v[0], 0.25)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("odd", [False, True])
def test_prompt_long(cw, t, hd, odd):
    """Rows of many tiles (for f32 of several windows, added up in the output), also in rows that no vector access fits."""
    g, lens, nh, nkv = gen(17), [2300, 1, 1153], 2, 1
    n = sum(lens)
    q, k, v, o = (rows_of(g, n, h, hd, t, None, hd + 3 if odd else None, 1 if odd else 0) for h in (nh, nkv, nkv, nh))
    k[0][2000] *= 3.0  # the maximum of many rows comes late
    o[0].fill_(math.nan)
    run_prompt(cw, t, lens, nh, nkv, hd, None, q, k, v, o)
    check_prompt(o[0], t, lens, nh, nkv, q[0], k[0], v[0], hd ** -0.5)


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("first,rest", [(0.0, 1e-4), (1.0, 1e6), (1e6, 1.0), (1e-20, 1e-20), (1e15, 1e15)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_prompt_f32_magnitudes(cw, hd, first, rest, what):
    """The f32 parts are scaled by what a window's first slots hold: zeros there, values that grow or shrink by a
    million behind them, tiny and huge ones.  K's stay within scores of a few units by q."""
    g, n = gen(15), 300
    q, k, v, o = (rows_of(g, n, 1, hd, F32) for _ in range(4))
    x = k if what == "k" else v
    x[0][:128] *= first
    x[0][128:] *= rest
    if what == "k":
        q[0].mul_(1.0 / max(first, rest))
    run_prompt(cw, F32, [n], 1, 1, hd, None, q, k, v, o)
    check_prompt(o[0], F32, [n], 1, 1, q[0], k[0], v[0], hd ** -0.5)


def test_prompt_malformed_offsets_stay_in_bounds(cw):
    """cu that decreases, is negative or passes n_rows is cut to the rows there are: finite neighbours stay right."""
    g, nh, nkv, hd, n = gen(3), 2, 1, 64, 100
    for t in (F32, BF16):
        q, k, v, o = (rows_of(g, n, h, hd, t) for h in (nh, nkv, nkv, nh))
        for cu in ([0, 50, 1000], [-20, 50, 100], [0, 60, 40, 100], [90, 10, 5], [2 ** 31 - 1, 2 ** 31 - 1]):
            c = torch.tensor(cu, device="cuda", dtype=torch.int32)
            run_prompt(cw, t, [0] * (len(cu) - 1), nh, nkv, hd, None, q, k, v, o, cu=c, n_rows=n)
        torch.cuda.synchronize()
    assert status(cw) == 0


def test_prompt_many_sequences(cw):
    """Hundreds of short sequences, most empty or one token long."""
    rng = random.Random(1)
    lens = [rng.choice([0, 0, 1, 1, 2, 5, 17]) for _ in range(700)]
    g, n, nh, nkv, hd = gen(1), sum(lens), 2, 1, 64
    for t in (F32, F16):
        q, k, v, o = (rows_of(g, n, h, hd, t) for h in (nh, nkv, nkv, nh))
        run_prompt(cw, t, lens, nh, nkv, hd, None, q, k, v, o)
        check_prompt(o[0], t, lens, nh, nkv, q[0], k[0], v[0], hd ** -0.5)


# ------------------------------------------------------------------ tree attention
def tree_masks(rng, n, T):
    out = []
    for _ in range(n):
        m = []
        for t in range(T):
            up = rng.randrange(-1, t) if t else -1
            m.append((m[up] if up >= 0 else 0) | 1 << t)
        out.append(m)
    return out


def signed(masks):
    return torch.tensor([[m - (1 << 64) if m >> 63 else m for m in row] for row in masks], device="cuda")


def run_tree(cw, c, lens, T, nh, q, o, mask=None, nodes=None, layer=0, scale=None, ws=None, st=None, max_len=None):
    nkv, hd = c.desc.n_kv, c.desc.head_dim
    (q, qr, qh), (o, orow, oh) = q, o
    ln = torch.tensor(lens, device="cuda", dtype=torch.int32) if not torch.is_tensor(lens) else lens
    nd = torch.tensor(nodes, device="cuda", dtype=torch.int32) if nodes is not None else None
    need = cw.lib().cwen_cuda_attn_tree_ws(c.desc, len(ln), T, nh)
    ws = ws if ws is not None else torch.full((need,), 255, device="cuda", dtype=torch.uint8)  # NaN bits
    assert ws.numel() >= need
    cw.check(cw.lib().cwen_cuda_attn_tree(c.desc, layer, ptr(c.table), c.stride, len(ln), ptr(ln),
                                          max_len or c.stride * c.page, T, ptr(nd), ptr(mask), nh,
                                          scale if scale is not None else hd ** -0.5, ptr(q), qr, qh, ptr(o), orow, oh,
                                          ptr(ws), ws.numel(), st or stream()), "tree")
    return o


def fill(c, lens, counts, g, layer=0):
    """Values in the slots of each sequence; everything else stays NaN."""
    for s, (n, m) in enumerate(zip(lens, counts)):
        at = c.rows(s, range(n + m))
        for w in ("k", "v"):
            c.flat(w, layer)[at] = normal(g, n + m, c.desc.n_kv, c.desc.head_dim, t=c.t)


def check_tree(c, got, q, lens, T, nh, masks, nodes, scale, layer=0):
    G = nh // c.desc.n_kv
    for s, n in enumerate(lens):
        m = nodes[s] if nodes is not None else T
        at = c.rows(s, range(n + m))
        seen = torch.ones(m, n + m, dtype=torch.bool)
        for t in range(m):
            bits = masks[s][t] if masks else (2 << t) - 1
            seen[t, n:] = torch.tensor([bool(bits >> u & 1) for u in range(m)])
        seen = seen.cuda()
        for h in range(nh):
            out, bound, av = attn_ref(q[s * T:s * T + m, h].double(), c.flat("k", layer)[at, h // G].double(),
                                      c.flat("v", layer)[at, h // G].double(), seen, scale)
            close(got[s * T:s * T + m, h], out, bound, av, c.t)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("T,page,lens", [(1, 16, [0, 1, 15, 16, 17, 200]), (9, 64, [500, 0, 63]), (64, 5, [33, 130]),
                                         (24, 1, [7]), (3, 100, [1000, 1]), (17, 24, [64, 65, 127])], ids=str)
def test_tree(cw, t, nh, nkv, hd, T, page, lens):
    """Trees over pages of any size, ragged lengths; unused places of the pages hold NaN."""
    g, rng = gen(T + hd), random.Random(T)
    c = Cache(cw, t, len(lens), max(lens) + T, page, nkv, hd, layers=2, seed=T)
    fill(c, lens, [T] * len(lens), g, layer=1)
    masks = tree_masks(rng, len(lens), T)
    q, o = rows_of(g, len(lens) * T, nh, hd, t, scale=2.0), rows_of(g, len(lens) * T, nh, hd, t)
    o[0].fill_(math.nan)
    run_tree(cw, c, lens, T, nh, q, o, signed(masks), layer=1)
    check_tree(c, o[0], q[0], lens, T, nh, masks, None, hd ** -0.5, 1)
    # a chain is the mask of all earlier nodes: the same bits
    chain = signed([[(2 << i) - 1 for i in range(T)]] * len(lens))
    a = run_tree(cw, c, lens, T, nh, q, o, chain, layer=1).clone()
    assert torch.equal(run_tree(cw, c, lens, T, nh, q, o, None, layer=1), a)
    check_tree(c, a, q[0], lens, T, nh, None, None, hd ** -0.5, 1)
    assert status(cw) == 0


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,hd", [(24, 4, 256), (32, 8, 128), (4, 4, 64)])
@pytest.mark.parametrize("T,lens", [(1, [40000]), (1, [3000, 12, 9000, 1]), (12, [20011]), (40, [5000, 4096])], ids=str)
def test_tree_long(cw, t, nh, nkv, hd, T, lens):
    """Long contexts, split over many CTAs and joined; two runs give the same bits."""
    g = gen(T)
    c = Cache(cw, t, len(lens), max(lens) + T, 64, nkv, hd, seed=T)
    fill(c, lens, [T] * len(lens), g)
    q, o = rows_of(g, len(lens) * T, nh, hd, t, scale=2.0), rows_of(g, len(lens) * T, nh, hd, t)
    a = run_tree(cw, c, lens, T, nh, q, o).clone()
    check_tree(c, a, q[0], lens, T, nh, None, None, hd ** -0.5)
    assert torch.equal(run_tree(cw, c, lens, T, nh, q, o), a)


@pytest.mark.parametrize("t", [F32, F16])
def test_tree_padded_batch(cw, t):
    """Sequences with fewer nodes than T: their rows stay, what lies behind the nodes is not read."""
    g, rng, T, nh, nkv, hd = gen(4), random.Random(4), 11, 6, 2, 128
    lens, nodes = [50, 0, 300, 7, 129], [11, 3, 0, 1, 10]
    c = Cache(cw, t, 5, 311, 16, nkv, hd)
    fill(c, lens, nodes, g)
    masks = [[m | (~0 << 11) & (2 ** 64 - 1) for m in row] for row in tree_masks(rng, 5, T)]  # bits past the nodes
    q, o = rows_of(g, 5 * T, nh, hd, t), rows_of(g, 5 * T, nh, hd, t)
    q[0].view(5, T, nh, hd)[1, 3:] = math.nan
    o[0].fill_(5.0)
    run_tree(cw, c, lens, T, nh, q, o, signed(masks), nodes)
    check_tree(c, o[0], q[0], lens, T, nh, masks, nodes, hd ** -0.5)
    rest = o[0].reshape(5, T, nh, hd)
    for s, m in enumerate(nodes):
        assert (rest[s, m:] == 5).all()
    # counts out of range are T or 0
    b = o[0].clone()
    run_tree(cw, c, [50, 0, 300, 7, 100], T, nh, q, o, signed(masks), [99, 3, -5, 1, 10])
    assert torch.equal(o[0][:11], b[:11]) and (o[0].view(5, T, nh, hd)[2] == 5).all()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_tree_rows_that_see_nothing(cw, t, hd):
    g, T, nh, nkv = gen(5), 5, 4, 2
    lens = [0, 20]
    c = Cache(cw, t, 2, 40, 16, nkv, hd)
    fill(c, lens, [T] * 2, g)
    masks = [[0, 2, 0, 1 << 3, 0], [0, 0, 1 << 4, 1, 31]]
    q, o = rows_of(g, 2 * T, nh, hd, t), rows_of(g, 2 * T, nh, hd, t)
    run_tree(cw, c, lens, T, nh, q, o, signed(masks))
    for i in (0, 2, 4):
        assert (o[0][i] == 0).all()
    check_tree(c, o[0], q[0], lens, T, nh, masks, None, hd ** -0.5)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_tree_non_finite_values_reach_only_rows_that_see_them(cw, t, hd, bad):
    """A poisoned node changes its descendants only; K and V."""
    g, T, nh, nkv = gen(6), 8, 4, 2
    lens = [100]
    masks = [[1, 3, 5, 9, 16, 48, 64, 128]]  # node 2 is seen by itself only; 4 by 4 and 5
    c = Cache(cw, t, 1, 120, 16, nkv, hd)
    fill(c, lens, [T], g)
    q, o = rows_of(g, T, nh, hd, t), rows_of(g, T, nh, hd, t)
    clean = run_tree(cw, c, lens, T, nh, q, o, signed(masks)).clone()
    for node, rows in ((2, [2]), (4, [4, 5])):
        for w in ("k", "v"):
            row = c.rows(0, [100 + node])
            keep = c.flat(w)[row].clone()
            c.flat(w)[row, :, 7] = bad
            got = run_tree(cw, c, lens, T, nh, q, o, signed(masks)).clone()
            c.flat(w)[row] = keep
            hit = torch.zeros_like(got, dtype=torch.bool)
            if w == "v":
                hit[rows, :, 7] = True
                x = got[hit].float()
                assert x.isnan().all() if bad != bad else (x == bad).all()
            else:
                hit[rows] = True
                if bad != bad:
                    assert got[hit].isnan().all()
            check_tree(c, torch.where(hit, clean, got), q[0], lens, T, nh, masks, None, hd ** -0.5)


def test_tree_out_of_range_is_left_out_and_reported(cw):
    """Bad page ids: the slots there take no part.  Lengths past max_len or below 0 are cut."""
    g, T, nh, nkv, hd = gen(7), 2, 4, 2, 64
    for t in (F32, BF16):
        lens = [60, 60, 60]
        c = Cache(cw, t, 3, 80, 16, nkv, hd)
        fill(c, lens, [T] * 3, g)
        q, o = rows_of(g, 3 * T, nh, hd, t), rows_of(g, 3 * T, nh, hd, t)
        good = run_tree(cw, c, lens, T, nh, q, o).clone()
        assert status(cw) == 0
        c.table[1, 1], c.table[1, 2] = -1, c.desc.n_pages
        run_tree(cw, c, lens, T, nh, q, o)
        assert status(cw) == -5 and status(cw) == 0
        assert torch.equal(o[0][:2], good[:2]) and torch.equal(o[0][4:], good[4:])
        at = torch.cat([c.rows(1, range(0, 16)), c.rows(1, range(48, 62))])
        seen = torch.ones(2, 30, dtype=torch.bool, device="cuda")
        seen[0, 29] = False
        for h in range(nh):
            out, bound, av = attn_ref(q[0][2:4, h].double(), c.flat("k")[at, h // 2].double(),
                                      c.flat("v")[at, h // 2].double(), seen, hd ** -0.5)
            close(o[0][2:4, h], out, bound, av, t)
        c.table.copy_(c.table_h)
        run_tree(cw, c, [60, -9, 60], T, nh, q, o)
        assert status(cw) == -5 and torch.equal(o[0][:2], good[:2])
        run_tree(cw, c, [60, 2 ** 31 - 1, 60], T, nh, q, o)
        assert status(cw) == -5 and torch.equal(o[0][:2], good[:2]) and torch.equal(o[0][4:], good[4:])
        run_tree(cw, c, [60, 30, 20], T, nh, q, o, max_len=62)
        assert status(cw) == 0 and torch.equal(o[0][:2], good[:2])


def test_tree_shared_pages_and_strided_rows(cw):
    """Two sequences that share the pages of a prefix; q with its gate beside it, odd bases."""
    g, T, nh, nkv, hd = gen(8), 4, 8, 2, 128
    for t, off in ((F32, 1), (F16, 3), (BF16, 0)):
        c = Cache(cw, t, 2, 200, 16, nkv, hd)
        c.table_h[1, :6] = c.table_h[0, :6]
        c.table.copy_(c.table_h)
        lens = [96 + 40, 96 + 3]
        fill(c, lens, [T] * 2, g)
        fill(c, [lens[0]], [T], g)
        q, o = rows_of(g, 2 * T, nh, hd, t, nh * 2 * hd + off, 2 * hd, off), rows_of(g, 2 * T, nh, hd, t, nh * 131, 131, off)
        masks = tree_masks(random.Random(1), 2, T)
        run_tree(cw, c, lens, T, nh, q, o, signed(masks))
        check_tree(c, o[0], q[0], lens, T, nh, masks, None, hd ** -0.5)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("n,T", [(40, 2), (130, 1), (300, 5)])
def test_tree_many_sequences(cw, t, n, T):
    """More sequences than a warp has lanes, some of them without nodes, lengths of none to a few tiles."""
    g, rng, nh, nkv, hd = gen(n), random.Random(n), 4, 2, 64
    lens = [rng.choice([0, 1, 5, 127, 128, 129, 400]) for _ in range(n)]
    nodes = [rng.choice([0, 1, T, T]) for _ in range(n)]
    c = Cache(cw, t, n, 400 + T, 16, nkv, hd)
    fill(c, lens, nodes, g)
    q, o = rows_of(g, n * T, nh, hd, t), rows_of(g, n * T, nh, hd, t)
    o[0].fill_(3.0)
    run_tree(cw, c, lens, T, nh, q, o, None, nodes)
    check_tree(c, o[0], q[0], lens, T, nh, None, nodes, hd ** -0.5)
    for s in range(n):
        assert (o[0][s * T + nodes[s]:(s + 1) * T] == 3).all()
    assert status(cw) == 0


@pytest.mark.parametrize("t", [F32, BF16])
def test_cache_of_more_than_2_31_elements(cw, t):
    """K and V pools of 2.1 G elements each: rows are written, read and moved on both sides of 2^31."""
    g, T, nh, nkv, hd = gen(19), 4, 8, 8, 256
    c = Cache(cw, t, 2, 700, 64, nkv, hd, spare=16500)
    n = c.desc.n_pages
    assert n * 64 * nkv * hd > 2 ** 31
    half = c.stride // 2
    c.table_h[0] = torch.arange(n - c.stride, n)  # the last pages, the first, and some of both
    c.table_h[1] = torch.cat([torch.arange(half), torch.arange(n - 2 * c.stride, n - 2 * c.stride + c.stride - half)])
    c.table.copy_(c.table_h)
    lens = [600, 690]
    rows = 600 + 690 + 2 * T
    k, v = (normal(g, rows, nkv, hd, t=t) for _ in range(2))
    seq = torch.tensor([0] * (600 + T) + [1] * (690 + T), device="cuda", dtype=torch.int32)
    slot = torch.cat([torch.arange(600 + T), torch.arange(690 + T)]).int().cuda()
    cw.check(cw.lib().cwen_cuda_kv_append(c.desc, 0, ptr(c.table), c.stride, 2, t, rows, ptr(k), nkv * hd, hd, ptr(v), nkv * hd,
                                          hd, ptr(seq), ptr(slot), None, None, stream()))
    at = torch.cat([c.rows(0, range(600 + T)), c.rows(1, range(690 + T))])
    assert torch.equal(c.flat("k")[at], k) and torch.equal(c.flat("v")[at], v)
    q, o = rows_of(g, 2 * T, nh, hd, t), rows_of(g, 2 * T, nh, hd, t)
    run_tree(cw, c, lens, T, nh, q, o)
    check_tree(c, o[0], q[0], lens, T, nh, None, None, hd ** -0.5)
    ln, kp = torch.tensor(lens, device="cuda", dtype=torch.int32), torch.tensor([0b1010, 0b1000], device="cuda")
    cw.check(cw.lib().cwen_cuda_kv_compact(c.desc, ptr(c.table), c.stride, 2, ptr(ln), ptr(kp), None, stream()))
    now = torch.cat([c.rows(0, [600, 601]), c.rows(1, [690])])
    assert torch.equal(c.flat("k")[now], k[[601, 603, 600 + T + 693]])
    assert torch.equal(c.flat("v")[now], v[[601, 603, 600 + T + 693]])
    assert status(cw) == 0


# ------------------------------------------------------------------ streams and graphs
def test_other_stream_and_graph_replay(cw):
    """On a side stream, then captured once and replayed with other lengths, pages and values in the same buffers; two
    graphs with a workspace each run at the same time."""
    g, T, nh, nkv, hd, n = gen(9), 3, 8, 2, 128, 4
    c = Cache(cw, BF16, n, 3000, 32, nkv, hd)
    lens = torch.tensor([2500, 10, 700, 0], device="cuda", dtype=torch.int32)
    fill(c, lens.tolist(), [T] * n, g)
    q, o = rows_of(g, n * T, nh, hd, BF16), rows_of(g, n * T, nh, hd, BF16)
    o2 = rows_of(g, n * T, nh, hd, BF16)
    need = cw.lib().cwen_cuda_attn_tree_ws(c.desc, n, T, nh)
    ws, ws2 = (torch.empty(need, device="cuda", dtype=torch.uint8) for _ in range(2))
    want = run_tree(cw, c, lens, T, nh, q, o, ws=ws).clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        o[0].zero_()
        run_tree(cw, c, lens, T, nh, q, o, ws=ws, st=side.cuda_stream)
    side.synchronize()
    assert torch.equal(o[0], want)
    graphs = []
    for out, w in ((o, ws), (o2, ws2)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            run_tree(cw, c, lens, T, nh, q, out, ws=w, st=torch.cuda.current_stream().cuda_stream)
        graphs.append(gr)
    for new in ([2500, 10, 700, 0], [3, 900, 0, 2000], [0, 0, 0, 1]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        fill(c, new, [T] * n, g)
        o[0].fill_(math.nan)
        o2[0].fill_(math.nan)
        torch.cuda.synchronize()
        for gr, s in zip(graphs, (side, torch.cuda.Stream())):
            with torch.cuda.stream(s):
                for _ in range(3):
                    gr.replay()
        torch.cuda.synchronize()
        check_tree(c, o[0], q[0], new, T, nh, None, None, hd ** -0.5)
        assert torch.equal(o[0], o2[0])
    assert status(cw) == 0


def test_prompt_graph_replay_with_other_lengths(cw):
    g, nh, nkv, hd, n = gen(10), 4, 2, 128, 400
    for t in (F32, BF16):
        q, k, v, o = (rows_of(g, n, h, hd, t) for h in (nh, nkv, nkv, nh))
        cu = torch.tensor([0, 400, 400, 400], device="cuda", dtype=torch.int32)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            run_prompt(cw, t, [0] * 3, nh, nkv, hd, None, q, k, v, o, cu=cu, st=torch.cuda.current_stream().cuda_stream)
        for lens in ([400, 0, 0], [1, 200, 199], [130, 140, 130]):
            cu.copy_(torch.tensor([0, lens[0], lens[0] + lens[1], 400], dtype=torch.int32))
            o[0].fill_(math.nan)
            gr.replay()
            torch.cuda.synchronize()
            check_prompt(o[0], t, lens, nh, nkv, q[0], k[0], v[0], hd ** -0.5)


def test_engine_stream_is_the_default(cw):
    """stream NULL is the engine's stream."""
    g = gen(2)
    r, turn = rope_table(cw, 64)
    x, pos = normal(g, 5, 2, 64), torch.arange(5, device="cuda", dtype=torch.int32)
    y = torch.zeros_like(x)
    torch.cuda.synchronize()
    cw.check(cw.lib().cwen_cuda_rope(r, F32, 5, 2, 64, ptr(x), 128, 64, ptr(pos), 0, ptr(y), 128, 64, None))
    assert cw.lib().cwen_cuda_attn_status(None) == 0  # synchronizes
    check_rope(y, x, pos, r, turn, 1.0, F32)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("nh,nkv,hd,n_rot,half", [(24, 4, 256, 64, 0), (8, 2, 128, 128, 1)])
def test_serving_loop(cw, t, nh, nkv, hd, n_rot, half):
    """Prompts, then drafted trees: rope, append, attention of the prompt from its rows and of trees from the pages,
    the accepted path compacted; every step equals attention over the tokens kept so far, in order."""
    g, rng = gen(11), random.Random(3)
    lens, T, steps, scale = [30, 1, 77], 6, 4, hd ** -0.5
    n, cap = len(lens), 77 + 6 * 7
    r, turn = rope_table(cw, n_rot, half)
    c = Cache(cw, t, n, cap, 16, nkv, hd, layers=2)
    L = cw.lib()

    def step(rows_seq, slots, posns):
        m = len(rows_seq)
        q, k, v = (rows_of(g, m, h, hd, t) for h in (nh, nkv, nkv))
        ints = [torch.tensor(x, device="cuda", dtype=torch.int32) for x in (rows_seq, slots, posns)]
        call_rope(cw, r, t, q[0], q[1:], ints[2], 0, q[0], q[1:])
        for layer in range(2):
            cw.check(L.cwen_cuda_kv_append(c.desc, layer, ptr(c.table), c.stride, n, t, m, ptr(k[0]), *k[1:], ptr(v[0]),
                                           *v[1:], ptr(ints[0]), ptr(ints[1]), r, ptr(ints[2]), stream()))
        return q, k, v, ints[2]

    seq = [s for s in range(n) for _ in range(lens[s])]
    slot = [i for m in lens for i in range(m)]
    q, k, v, pos = step(seq, slot, slot)
    kr = rows_of(g, len(seq), nkv, hd, t)
    call_rope(cw, r, t, k[0], k[1:], pos, 0, kr[0], kr[1:])
    at = torch.cat([c.rows(s, range(lens[s])) for s in range(n)])
    assert torch.equal(c.flat("k", 0)[at], kr[0]) and torch.equal(c.flat("v", 1)[at], v[0])
    o = rows_of(g, len(seq), nh, hd, t)
    run_prompt(cw, t, lens, nh, nkv, hd, scale, q, kr, v, o)
    check_prompt(o[0], t, lens, nh, nkv, q[0], kr[0], v[0], scale)
    kept = [(c.flat("k", 0)[c.rows(s, range(lens[s]))].clone(), c.flat("v", 0)[c.rows(s, range(lens[s]))].clone())
            for s in range(n)]
    ln = torch.tensor(lens, device="cuda", dtype=torch.int32)
    other = torch.empty_like(ln)
    for it in range(steps):
        now = ln.tolist()
        masks = tree_masks(rng, n, T)
        depth = [[bin(m).count("1") - 1 for m in row] for row in masks]
        q, k, v, pos = step([s for s in range(n) for _ in range(T)], [now[s] + i for s in range(n) for i in range(T)],
                            [now[s] + d for s in range(n) for d in depth[s]])
        o = rows_of(g, n * T, nh, hd, t)
        run_tree(cw, c, ln, T, nh, q, o, signed(masks), layer=it % 2)
        check_tree(c, o[0], q[0], now, T, nh, masks, None, scale, it % 2)
        tips = [rng.randrange(T) for _ in range(n)]
        paths = [[u for u in range(T) if masks[s][tips[s]] >> u & 1] for s in range(n)]
        for s in range(n):
            rows = c.rows(s, [now[s] + u for u in paths[s]])
            kept[s] = tuple(torch.cat([old, c.flat(w, 0)[rows]]) for old, w in zip(kept[s], "kv"))
        keep = signed([[masks[s][tips[s]]] for s in range(n)])
        cw.check(L.cwen_cuda_kv_compact(c.desc, ptr(c.table), c.stride, n, ptr(ln), ptr(keep), ptr(other), stream()))
        ln, other = other, ln
        for s in range(n):
            rows = c.rows(s, range(len(kept[s][0])))
            assert int(ln[s]) == len(kept[s][0])
            for layer in range(2):
                assert torch.equal(c.flat("k", layer)[rows], kept[s][0]) and torch.equal(c.flat("v", layer)[rows], kept[s][1])
    assert status(cw) == 0
