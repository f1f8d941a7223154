"""The attention operators on caller buffers as measured workloads.

Five operators, used one after another by a program that serves several
sequences from a paged cache: rotary positions on rows, writing K/V rows into
the pages, attention over whole prompts, attention of drafted trees (a single
token, a chain or a tree) over the pages, and compacting the accepted path.

`run` has two forms: the plain one in elementary torch operations, and with
`own` the calls of the C ABI (include/cwen_cuda.h) that a program makes.
"""
import functools
import math
import random

import numpy as np
import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GGML = {"f32": 0, "f16": 1, "bf16": 30}  # type numbers of the C ABI


# ---------------------------------------------------------------- the cases
def listed():
    # 24 query heads, 4 key/value heads of 256 with 64 rotated dims, 16
    # attention layers and a 32768-slot context are the engine's own geometry.
    return [
        # queries of one verify block (8 drafts and the pending token)
        dict(name="rope_block", op="rope", type="f32", rows=9, heads=24, dim=256, rot=64, half=False, factor=1.0,
             ramp=False, base=1e7, far=32759, inverse=False),
        # queries of a long prompt whose positions are scaled by parts, eight times past the trained context
        dict(name="rope_prompt", op="rope", type="bf16", rows=16384, heads=32, dim=128, rot=128, half=True, factor=8.0,
             ramp=True, base=1e6, far=245760, inverse=False),
        # K/V rows of four sequences' verify blocks, fp32 activations into an fp32 cache
        dict(name="append_block", op="append", type="f32", cache="f32", seqs=4, rows=36, kv=4, dim=256, rot=64,
             half=False, base=1e7, start=1500, page=64),
        # K/V rows of packed prompts, fp32 activations into a bf16 cache
        dict(name="append_prompt", op="append", type="f32", cache="bf16", seqs=7, rows=32768, kv=4, dim=256, rot=64,
             half=True, base=1e7, start=0, page=32),
        # one sequence's accepted path in a 16-layer fp32 cache
        dict(name="compact_one", op="compact", cache="f32", seqs=1, layers=16, kv=4, dim=256, nodes=16, start=700,
             page=64),
        # a batch of trees, long paths that cross pages of 16 slots
        dict(name="compact_batch", op="compact", cache="bf16", seqs=64, layers=16, kv=4, dim=256, nodes=60, start=90,
             page=16),
        # one short question, few small heads: latency
        dict(name="prompt_short", op="prompt", type="f16", seqs=1, rows=67, heads=14, kv=2, dim=64),
        # prompts of very different lengths packed into one call
        dict(name="prompt_packed", op="prompt", type="bf16", seqs=9, rows=16381, heads=24, kv=4, dim=256),
        # a prompt in the engine's own fp32
        dict(name="prompt_f32", op="prompt", type="f32", seqs=2, rows=4100, heads=24, kv=4, dim=256),
        # one token of one sequence, long context
        dict(name="tree_token", op="tree", type="bf16", seqs=1, nodes=1, tree="chain", len=32767, heads=24, kv=4,
             dim=256, page=64),
        # a verify block (chain of 9) over the engine's fp32 cache, long context
        dict(name="tree_chain_f32", op="tree", type="f32", seqs=1, nodes=9, tree="chain", len=32495, heads=24, kv=4,
             dim=256, page=64),
        # a serving batch: trees of up to 24 nodes over sequences of very different lengths
        dict(name="tree_batch", op="tree", type="f16", seqs=31, nodes=24, tree="tree", len=12000, heads=32, kv=8,
             dim=128, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "compact", "prompt", "prompt", "tree", "tree"])
    t = rng.choice(["f32", "f16", "bf16"])
    heads, kv, dim = rng.choice([(24, 4, 256), (32, 8, 128), (16, 16, 64), (14, 2, 64), (8, 1, 128), (5, 5, 128),
                                 (3, 1, 256)])
    page = rng.choice([8, 16, 24, 32, 64, 100])
    if op == "rope":
        ramp = rng.random() < 0.5
        return dict(op=op, type=t, rows=_log(rng, 1, 12000), heads=heads, dim=dim, rot=rng.choice([dim, dim // 2, dim // 4]),
                    half=rng.random() < 0.5, factor=rng.choice([2.0, 8.0, 32.0]) if ramp else rng.choice([1.0, 1.0, 4.0]),
                    ramp=ramp, base=rng.choice([1e4, 1e6, 1e7]), far=_log(rng, 1, 1000000), inverse=rng.random() < 0.25)
    if op == "append":
        seqs = _log(rng, 1, 40)
        return dict(op=op, type="f32" if rng.random() < 0.5 else t, cache=t, seqs=seqs, rows=seqs + _log(rng, 1, 24000),
                    kv=kv, dim=dim, rot=rng.choice([dim, dim // 2, dim // 4]), half=rng.random() < 0.5,
                    base=rng.choice([1e4, 1e6, 1e7]), start=rng.randrange(0, 3000), page=page)
    if op == "compact":
        return dict(op=op, cache=t, seqs=_log(rng, 1, 60), layers=rng.choice([1, 4, 16]), kv=min(kv, 8), dim=dim,
                    nodes=rng.randrange(2, 61), start=rng.randrange(0, 400), page=page)
    if op == "prompt":
        seqs = rng.choice([1, 1, 2, 3, 5, 8, 12])
        return dict(op=op, type=t, seqs=seqs, rows=seqs + _log(rng, 1, 4000 if t == "f32" else 12000), heads=heads, kv=kv,
                    dim=dim)
    seqs, nodes = _log(rng, 1, 32), rng.choice([1, 1, 2, 5, 9, 16, 24, 33, 64])
    top = 32000 if nodes == 1 else 16000
    return dict(op=op, type=t, seqs=seqs, nodes=nodes, tree="tree" if nodes > 1 and rng.random() < 0.6 else "chain",
                len=_log(rng, 1, max(60, top // seqs)), heads=heads, kv=kv, dim=dim, page=page)


def _shares(total, n):
    """n lengths >= 1 of very different sizes that add up to total (a fixed function of the two)."""
    if n == 1:
        return [total]
    w = [0.0] + [1.0 / (i + 1) ** 1.5 for i in range(n - 1)]  # the first is one token long
    left = total - n
    got = [1 + int(left * x / sum(w)) for x in w]
    got[1] += total - sum(got)
    return got


def _lens(case):
    """Committed slots and live nodes of a batch: the first sequence is the longest, the last (of several) is new."""
    n, top, t = case["seqs"], case["len"], case["nodes"]
    lens = [max(0, int(top * (1.0 - 0.97 * i / max(1, n - 1)))) for i in range(n)]
    if n > 2:
        lens[-1] = 0
    nodes = [t if i % 3 != 1 else max(1, t - 1 - (5 * i) % max(1, t)) for i in range(n)]
    return lens, nodes


def _paths(case):
    """keep masks of a compaction: an increasing path through each tree (a fixed function of the case)."""
    r = random.Random(case["seqs"] * 1009 + case["nodes"])
    out = []
    for s in range(case["seqs"]):
        p, u = [], r.randrange(0, 2)
        while u < case["nodes"]:
            p.append(u)
            u += 1 + (r.random() < 0.6) * r.randrange(1, 4)
        out.append(p)
    return out


# ---------------------------------------------------------------- inputs
def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, device="cuda", dtype=dtype)


def _table(g, slots, page, stride=None):
    """A page table whose sequences hold the given numbers of slots, pages in random order; spare pages too."""
    need = [-(-s // page) for s in slots]
    stride = stride or max(max(need), 1)
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").cpu().numpy()
    tab = np.full((len(slots), stride), -1, np.int32)
    at = 0
    for s, k in enumerate(need):
        tab[s, :k] = order[at:at + k]
        at += k
    return torch.from_numpy(tab).cuda(), total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    op, s = case["op"], dict(case)
    if op == "rope":
        s["x"] = _normal(g, case["rows"], case["heads"], case["dim"], dtype=DTYPE[case["type"]])
        s["y"] = torch.empty_like(s["x"])
        off = r.randrange(0, 17)
        s["pos"] = torch.arange(case["rows"], device="cuda", dtype=torch.int32) + (case["far"] + off)
        s["turn"], s["mscale"] = _turns(case)
    elif op == "append":
        n, rows = case["seqs"], _shares(case["rows"], case["seqs"])
        first = [case["start"] + r.randrange(0, 9) * (case["start"] > 0) for _ in range(n)]
        s["table"], s["pages"] = _table(g, [case["start"] + 9 + b for b in rows], case["page"])
        s["k"], s["v"] = (_normal(g, case["rows"], case["kv"], case["dim"], dtype=DTYPE[case["type"]]) for _ in range(2))
        s["seq"] = torch.repeat_interleave(torch.arange(n, device="cuda", dtype=torch.int32), _ints(rows, torch.int64))
        s["slot"] = torch.cat([torch.arange(a, a + b, device="cuda", dtype=torch.int32) for a, b in zip(first, rows)])
        s["pos"] = s["slot"] + 2
        s["kc"], s["vc"] = (torch.zeros(1, s["pages"], case["page"], case["kv"], case["dim"], device="cuda",
                                        dtype=DTYPE[case["cache"]]) for _ in range(2))
        s["turn"], s["mscale"] = _turns(case)
    elif op == "compact":
        lens = [max(0, case["start"] - r.randrange(0, 9)) for _ in range(case["seqs"])]
        s["table"], s["pages"] = _table(g, [case["start"] + case["nodes"]] * case["seqs"], case["page"])
        s["kc"], s["vc"] = (_normal(g, case["layers"], s["pages"], case["page"], case["kv"], case["dim"],
                                    dtype=DTYPE[case["cache"]]) for _ in range(2))
        s["len"] = _ints(lens)
        s["keep"] = _ints([sum(1 << u for u in p) for p in _paths(case)], torch.int64)
        s["len_out"] = torch.zeros_like(s["len"])
    elif op == "prompt":
        rows = _shares(case["rows"], case["seqs"])
        r.shuffle(rows)
        s["lens"] = rows
        s["cu"] = _ints([0] + list(np.cumsum(rows)))
        dt = DTYPE[case["type"]]
        s["q"] = _normal(g, case["rows"], case["heads"], case["dim"]).mul(1.5).to(dt)
        s["k"], s["v"] = (_normal(g, case["rows"], case["kv"], case["dim"], dtype=dt) for _ in range(2))
        s["o"] = torch.empty_like(s["q"])
    else:
        lens, nodes = _lens(case)
        T = case["nodes"]
        s["table"], s["pages"] = _table(g, [a + T for a in lens], case["page"])
        dt = DTYPE[case["type"]]
        s["kc"], s["vc"] = (_normal(g, 1, s["pages"], case["page"], case["kv"], case["dim"], dtype=dt) for _ in range(2))
        s["q"] = _normal(g, case["seqs"] * T, case["heads"], case["dim"]).mul(1.5).to(dt)
        s["o"] = torch.zeros_like(s["q"])
        s["len"], s["n_node"] = _ints(lens), _ints(nodes)
        s["max_len"] = max(lens) + T
        s["mask"] = None
        if case["tree"] == "tree":
            bits = []
            for _ in lens:
                m = []
                for t in range(T):
                    up = r.randrange(-1, t) if t else -1
                    m.append((m[up] if up >= 0 else 0) | 1 << t)
                bits.append([x - (1 << 64) if x >> 63 else x for x in m])
            s["mask"] = _ints(bits, torch.int64)
    return s


def _turns(case):
    """Turns per position of each pair, in 64 bits; scaled linearly or by parts (see the C header's cwen_rope_init)."""
    n, f = case["rot"], case.get("factor", 1.0)
    turn = case["base"] ** (-np.arange(0, n, 2, dtype=np.float64) / n) / (2 * math.pi)
    mscale = 1.0
    if case.get("ramp"):
        g = np.clip((turn * 32768 - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        turn = turn * (g + (1.0 - g) / f)
        mscale = 0.1 * math.log(f) + 1.0
    else:
        turn = turn / f
    return torch.from_numpy(turn).cuda(), mscale


# ---------------------------------------------------------------- one pass
def run(s):
    return (_own if own else _plain)[s["op"]](s)


def _turned(s, x, pos, sign=1.0):
    """x [rows, heads, dim] rotated, in 32 bits; angles in 64."""
    ang = 2 * math.pi * torch.frac(pos.double()[:, None] * s["turn"][None, :])
    c, i = (torch.cos(ang) * s["mscale"]).float()[:, None, :], (sign * torch.sin(ang) * s["mscale"]).float()[:, None, :]
    x, n = x.float(), s["rot"]
    y = x.clone()
    a, b = (slice(0, n // 2), slice(n // 2, n)) if s["half"] else (slice(0, n, 2), slice(1, n, 2))
    y[..., a] = x[..., a] * c - x[..., b] * i
    y[..., b] = x[..., a] * i + x[..., b] * c
    return y


def _plain_rope(s):
    return _turned(s, s["x"], s["pos"], -1.0 if s["inverse"] else 1.0).to(s["x"].dtype)


def _place(s, seq, slot):
    """(page, row in the page) of slots of sequences."""
    return s["table"][seq.long(), (slot // s["page"]).long()].long(), (slot % s["page"]).long()


def _plain_append(s):
    page, at = _place(s, s["seq"], s["slot"])
    s["kc"][0, page, at] = _turned(s, s["k"], s["pos"]).to(s["kc"].dtype)
    s["vc"][0, page, at] = s["v"].float().to(s["vc"].dtype)
    return {"k": s["kc"], "v": s["vc"]}


def _plain_compact(s):
    u = torch.arange(s["nodes"], device="cuda")
    bit = (s["keep"][:, None] >> u) & 1
    rank = torch.cumsum(bit, 1) - 1
    seq, node = torch.nonzero(bit, as_tuple=True)
    sp, sa = _place(s, seq, s["len"].long()[seq] + node)
    dp, da = _place(s, seq, s["len"].long()[seq] + rank[seq, node])
    s["kc"][:, dp, da] = s["kc"][:, sp, sa]
    s["vc"][:, dp, da] = s["vc"][:, sp, sa]
    return {"k": s["kc"], "v": s["vc"], "len": s["len"] + bit.sum(1).int()}


def _weights(scores, seen):
    """Softmax over the places that are seen; nothing seen gives zeros."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0)) * seen
    return p / p.sum(-1, keepdim=True).clamp_min(1e-37)


def _plain_prompt(s):
    o, h, kv, d = torch.zeros_like(s["q"]), s["heads"], s["kv"], s["dim"]
    at = 0
    for n in s["lens"]:  # one key/value head at a time: the scores of all would not fit
        i = torch.arange(n, device="cuda")
        seen = i[None, :] <= i[:, None]
        for j in range(kv):
            q = s["q"][at:at + n, j * (h // kv):(j + 1) * (h // kv)].float().transpose(0, 1)
            k, v = s["k"][at:at + n, j].float(), s["v"][at:at + n, j].float()
            p = _weights(q @ k.T * d ** -0.5, seen)
            o[at:at + n, j * (h // kv):(j + 1) * (h // kv)] = (p @ v).transpose(0, 1).to(o.dtype)
        at += n
    return o


def _plain_tree(s):
    n, T, h, kv, d = s["seqs"], s["nodes"], s["heads"], s["kv"], s["dim"]
    slot = torch.arange(s["max_len"], device="cuda")
    page = s["table"][:, slot // s["page"]].long().clamp_min(0)
    k, v = (c[0][page, (slot % s["page"])[None]].float().permute(0, 2, 1, 3) for c in (s["kc"], s["vc"]))
    q = s["q"].float().view(n, T, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, d)
    t, node = torch.arange(T, device="cuda"), slot[None, :] - s["len"].long()[:, None]
    inside = (node >= 0) & (node < s["n_node"][:, None])
    u = node.clamp(0, 63)
    if s["mask"] is None:
        bit = u[:, None, :] <= t[None, :, None]
    else:
        bit = ((s["mask"][:, :, None] >> u[:, None, :]) & 1).bool()
    seen = (node < 0)[:, None, :] | (inside[:, None, :] & bit)
    seen = seen[:, None, :, None, :].expand(n, kv, T, h // kv, -1).reshape(n, kv, T * (h // kv), -1)
    p = _weights(q @ k.transpose(2, 3) * d ** -0.5, seen)
    o = (p @ v).reshape(n, kv, T, h // kv, d).permute(0, 2, 1, 3, 4).reshape(n, T, h, d).to(s["q"].dtype)
    live = (t[None, :] < s["n_node"][:, None])[:, :, None, None]
    return torch.where(live, o, s["o"].view(n, T, h, d)).reshape(n * T, h, d)


_plain = {"rope": _plain_rope, "append": _plain_append, "compact": _plain_compact, "prompt": _plain_prompt,
          "tree": _plain_tree}


# ---------------------------------------------------------------- the calls that a program makes
@functools.cache
def _library():
    import cwen_b200 as cw
    if not cw.lib().cwen_cuda_ctx():
        cw.check(cw.lib().cwen_cuda_init(torch.cuda.current_device(), 32768, 16), "init")
    return cw, cw.lib()


@functools.cache
def _rope(rot, half, base, factor, ramp):
    cw, L = _library()
    r = cw.Rope()
    cw.check(L.cwen_rope_init(r, rot, int(half), base, factor, 32768.0, 32.0 if ramp else 0.0, 1.0 if ramp else 0.0), "rope")
    return r


def _rope_of(s):
    return _rope(s["rot"], s["half"], s["base"], s.get("factor", 1.0), s.get("ramp", False))


def _cache_of(cw, s, t):
    """The cache's description, as a program keeps it beside the buffers."""
    c = s.get("cache_desc")
    if c is None:
        L, pages, page, kv, d = s["kc"].shape
        c = s["cache_desc"] = cw.Kv(GGML[t], L, pages, page, kv, d, s["kc"].data_ptr(), s["vc"].data_ptr())
    return c


def _stream():
    return torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream (NULL means the engine's)


def _own_rope(s):
    cw, L = _library()
    x, y, h, d = s["x"], s["y"], s["heads"], s["dim"]
    rc = L.cwen_cuda_rope(_rope_of(s), GGML[s["type"]], s["rows"], h, d, x.data_ptr(), h * d, d, s["pos"].data_ptr(),
                          int(s["inverse"]), y.data_ptr(), h * d, d, _stream())
    if rc:
        cw.check(rc, "rope")
    return y


def _own_append(s):
    cw, L = _library()
    kv, d = s["kv"], s["dim"]
    rc = L.cwen_cuda_kv_append(_cache_of(cw, s, s["cache"]), 0, s["table"].data_ptr(), s["table"].shape[1], s["seqs"],
                               GGML[s["type"]], s["rows"], s["k"].data_ptr(), kv * d, d, s["v"].data_ptr(), kv * d, d,
                               s["seq"].data_ptr(), s["slot"].data_ptr(), _rope_of(s), s["pos"].data_ptr(), _stream())
    if rc:
        cw.check(rc, "append")
    return {"k": s["kc"], "v": s["vc"]}


def _own_compact(s):
    cw, L = _library()
    rc = L.cwen_cuda_kv_compact(_cache_of(cw, s, s["cache"]), s["table"].data_ptr(), s["table"].shape[1], s["seqs"],
                                s["len"].data_ptr(), s["keep"].data_ptr(), s["len_out"].data_ptr(), _stream())
    if rc:
        cw.check(rc, "compact")
    return {"k": s["kc"], "v": s["vc"], "len": s["len_out"]}


def _own_prompt(s):
    cw, L = _library()
    h, kv, d = s["heads"], s["kv"], s["dim"]
    rc = L.cwen_cuda_attn_prompt(GGML[s["type"]], s["seqs"], s["cu"].data_ptr(), s["rows"], h, kv, d, d ** -0.5,
                                 s["q"].data_ptr(), h * d, d, s["k"].data_ptr(), kv * d, d, s["v"].data_ptr(), kv * d, d,
                                 s["o"].data_ptr(), h * d, d, _stream())
    if rc:
        cw.check(rc, "prompt")
    return s["o"]


def _own_tree(s):
    cw, L = _library()
    h, d, T, c = s["heads"], s["dim"], s["nodes"], _cache_of(cw, s, s["type"])
    ws = s.get("ws")
    if ws is None:
        ws = s["ws"] = torch.empty(max(1, L.cwen_cuda_attn_tree_ws(c, s["seqs"], T, h)), dtype=torch.uint8, device="cuda")
    rc = L.cwen_cuda_attn_tree(c, 0, s["table"].data_ptr(), s["table"].shape[1], s["seqs"], s["len"].data_ptr(),
                               s["max_len"], T, s["n_node"].data_ptr(), s["mask"].data_ptr() if s["mask"] is not None else None,
                               h, d ** -0.5, s["q"].data_ptr(), h * d, d, s["o"].data_ptr(), h * d, d, ws.data_ptr(),
                               ws.numel(), _stream())
    if rc:
        cw.check(rc, "tree")
    return s["o"]


_own = {"rope": _own_rope, "append": _own_append, "compact": _own_compact, "prompt": _own_prompt, "tree": _own_tree}


# ---------------------------------------------------------------- what one pass cannot do without
def work(case):
    op = case["op"]
    if op == "rope":
        n = case["rows"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * SIZE[case["type"]] + 4 * case["rows"], "flops": 3 * n * case["rot"]}
    if op == "append":
        n = 2 * case["rows"] * case["kv"] * case["dim"]
        return {"bytes": n * (SIZE[case["type"]] + SIZE[case["cache"]]) + 12 * case["rows"],
                "flops": 3 * case["rows"] * case["kv"] * case["rot"]}
    if op == "compact":
        moved = sum(u != i for p in _paths(case) for i, u in enumerate(p))
        row = 2 * case["layers"] * case["kv"] * case["dim"] * SIZE[case["cache"]]
        return {"bytes": 2 * moved * row + 16 * case["seqs"], "flops": 0}
    if op == "prompt":
        lens = _shares(case["rows"], case["seqs"])
        return {"bytes": 2 * case["rows"] * (case["heads"] + case["kv"]) * case["dim"] * SIZE[case["type"]],
                "flops": 4 * case["heads"] * case["dim"] * sum(n * (n + 1) // 2 for n in lens)}
    lens, nodes = _lens(case)
    size = SIZE[case["type"]]
    flops = 4 * case["heads"] * case["dim"] * sum(t * (n + (t + 1) / 2) for n, t in zip(lens, nodes))
    rows = 2 * sum(n + t for n, t in zip(lens, nodes)) * case["kv"] + 2 * sum(nodes) * case["heads"]
    return {"bytes": rows * case["dim"] * size, "flops": flops}


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "rope":
        return _pairs64(case, s["x"], s["pos"], s["turn"] * (-1 if case["inverse"] else 1), s["mscale"])
    if op == "append":
        k, v = (torch.zeros(c.shape, device="cuda", dtype=torch.float64) for c in (s["kc"], s["vc"]))
        flat = s["table"].long()[s["seq"].long(), torch.div(s["slot"], case["page"], rounding_mode="floor").long()]
        flat = flat * case["page"] + s["slot"].long() % case["page"]
        k.view(-1, case["kv"], case["dim"]).index_copy_(0, flat, _pairs64(case, s["k"], s["pos"], s["turn"], s["mscale"]))
        v.view(-1, case["kv"], case["dim"]).index_copy_(0, flat, s["v"].double())
        return {"k": k, "v": v}
    if op == "compact":
        k, v = s["kc"].double().clone(), s["vc"].double().clone()
        lens, paths, table = s["len"].tolist(), _paths(case), s["table"].tolist()
        spot = lambda q, j: (table[q][j // case["page"]], j % case["page"])  # noqa: E731
        for q, path in enumerate(paths):
            for i, u in enumerate(path):  # in order: a source is never behind a destination
                (a, b), (x, y) = spot(q, lens[q] + u), spot(q, lens[q] + i)
                k[:, x, y], v[:, x, y] = k[:, a, b], v[:, a, b]
        return {"k": k, "v": v, "len": None}
    h, kv, d = case["heads"], case["kv"], case["dim"]
    if op == "prompt":
        o = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
        cu = s["cu"].tolist()
        for a, b in zip(cu, cu[1:]):
            for head in range(h):
                k, v = s["k"][a:b, head // (h // kv)].double(), s["v"][a:b, head // (h // kv)].double()
                for i in range(a, b, 2048):
                    e = min(b, i + 2048)
                    z = s["q"][i:e, head].double() @ k[:e - a].T / math.sqrt(d)
                    z = z + torch.full_like(z, -math.inf).triu(i - a + 1)
                    o[i:e, head] = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) @ v[:e - a]
        return o
    o, T = s["o"].double().clone(), case["nodes"]
    lens, nodes = _lens(case)
    for q in range(case["seqs"]):
        flat = torch.arange(lens[q] + nodes[q], device="cuda")
        flat = s["table"][q].long()[flat // case["page"]] * case["page"] + flat % case["page"]
        k, v = (c[0].reshape(-1, kv, d)[flat].double() for c in (s["kc"], s["vc"]))
        far = torch.zeros(nodes[q], lens[q] + nodes[q], device="cuda", dtype=torch.float64)
        bits = [2 ** (t + 1) - 1 for t in range(T)] if s["mask"] is None else s["mask"][q].tolist()
        hide = [[not bits[t] >> u & 1 for u in range(nodes[q])] for t in range(nodes[q])]
        far[:, lens[q]:][torch.tensor(hide, device="cuda")] = -math.inf
        for head in range(h):
            z = s["q"][q * T:q * T + nodes[q], head].double() @ k[:, head // (h // kv)].T / math.sqrt(d) + far
            o[q * T:q * T + nodes[q], head] = torch.softmax(z, 1) @ v[:, head // (h // kv)]
    return o


def _pairs64(case, x, pos, turn, mscale):
    """Rotation of the pairs as complex numbers, in 64 bits."""
    x, n = x.double(), case["rot"]
    w = torch.polar(torch.full((len(pos), n // 2), mscale, device="cuda", dtype=torch.float64),
                    2 * math.pi * torch.remainder(pos.double()[:, None] * turn, 1.0))
    z = x[..., :n].reshape(*x.shape[:2], *((2, n // 2) if case["half"] else (n // 2, 2)))
    z = torch.complex(z[..., 0, :], z[..., 1, :]) if case["half"] else torch.complex(z[..., 0], z[..., 1])
    z = torch.view_as_real(z * w[:, None, :])
    z = z.transpose(-1, -2) if case["half"] else z
    return torch.cat([z.reshape(*x.shape[:2], n), x[..., n:]], -1)
