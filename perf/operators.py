"""Timed cases of the paged cache's operators, in plain torch and through the library.

Operators
  append     keys and values of a step's new tokens into the pages of their sequences; RMS norm of every head of q and k and the rotation by one or
             several position axes on the way, the finished queries written beside
  attention  the step's queries (one token, a few drafted ones or a chunk of a prompt for each sequence, any mixture of them) over all positions
             that their sequences hold in their pages, causal, optionally over the last `window` positions only
  rope       rotation of the heads of a panel by positions with several axes (time, height, width), no cache

A step is described as a server has it on the device: first row and number of cached positions of every sequence, and a table of its pages.

Fields of a case: n_seq sequences with `mix` saying how many tokens each brings (one: 1 each; same: q each; ragged: 1 .. q; mixed: one sequence in eight
1 .. q, the others 1, with an idle slot and an empty one among them), past_min .. past positions in front of them, `pad` rows of the panel behind the last
sequence; heads / kv / hd the head layout, page the positions of a page, beside whether K and V of a page lie side by side in one pool; axes, rot, layout,
norm, f32 the rotation, the norms and the type that comes in; window and evicted (pages behind every window are gone from the table); shape_seed draws the lengths.
"""
import math
import random

import numpy as np
import torch

own = False
EPS = 1e-6
THETA = 1e6


def listed():
    a = dict(op="append", pad=0, beside=False, axes=1, rot=128, layout=1, norm=True, f32=False, hd=128)
    t = dict(op="attention", pad=0, beside=False, window=0, evicted=False, hd=128)
    return [
        # a decode step of a few users: the smallest call, all of it latency
        dict(a, name="append_decode", n_seq=8, mix="one", q=1, past_min=200, past=3000, heads=32, kv=8, page=16, shape_seed=1),
        # prompts and single tokens in one step far into long contexts, with rows of padding; pages of 32 with K and V side by side
        dict(a, name="append_mixed", n_seq=21, mix="mixed", q=150, past_min=1, past=200000, heads=64, kv=8, page=32, beside=True, pad=13, shape_seed=2),
        # image and text tokens of a prompt with three position axes, no norm, float projections
        dict(a, name="append_image", n_seq=3, mix="ragged", q=4000, past_min=0, past=500, heads=32, kv=8, page=64, axes=3, norm=False, f32=True, shape_seed=3),
        # a full step of prompt chunks on the widest block
        dict(a, name="append_panel", n_seq=4, mix="same", q=2048, past_min=0, past=2000, heads=64, kv=8, page=16, shape_seed=4),
        # one user, short context: latency
        dict(t, name="attn_one", n_seq=1, mix="one", q=1, past_min=1300, past=1300, heads=32, kv=8, page=16, shape_seed=5),
        # batched decoding over ragged contexts
        dict(t, name="attn_batch", n_seq=64, mix="one", q=1, past_min=400, past=4000, heads=64, kv=8, page=16, beside=True, shape_seed=6),
        # one user deep into a long context
        dict(t, name="attn_long", n_seq=1, mix="one", q=1, past_min=100000, past=100000, heads=64, kv=8, page=64, shape_seed=7),
        # a few drafted tokens per user to be verified, an odd page size
        dict(t, name="attn_draft", n_seq=16, mix="same", q=5, past_min=500, past=5000, heads=40, kv=8, page=24, shape_seed=8),
        # the next chunk of a long prompt
        dict(t, name="attn_chunk", n_seq=1, mix="same", q=2048, past_min=8192, past=8192, heads=32, kv=8, page=16, shape_seed=9),
        # chunks of prompts and decoding users in one step, small heads, the last 1000 positions only, older pages given back
        dict(t, name="attn_mixed", n_seq=24, mix="mixed", q=700, past_min=20, past=5000, heads=28, kv=4, page=32, window=1000, evicted=True, hd=64, pad=5, shape_seed=10),
        # patches of one small image in a vision encoder's float stream
        dict(op="rope", name="rope_patches", M=259, heads=16, hd=64, axes=2, rot=64, layout=0, f32=True, fused=False),
        # a video's tokens with (time, height, width), rotated where they lie in the rows of the fused projection
        dict(op="rope", name="rope_video", M=16001, heads=40, hd=128, axes=3, rot=128, layout=1, f32=False, fused=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "rope"])
    hd = rng.choice([64, 128, 128])
    if op == "rope":
        axes = rng.choice([1, 2, 3])
        rot = rng.choice([hd, hd, hd // 2, hd // 4 * 3])
        heads = rng.choice([2, 5, 8, 16, 28, 40])
        return dict(op=op, M=_log(rng, 1, 80000000 // (heads * hd)) if heads * hd > 4999 else _log(rng, 1, 16000), heads=heads, hd=hd, axes=axes, rot=rot,
                    layout=rng.choice([0, 1]), f32=rng.random() < 0.4, fused=rng.random() < 0.5)
    kv = rng.choice([1, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 7, 8])
    page = rng.choice([8, 16, 16, 24, 32, 48, 64, 128, 256])
    kind = rng.choice(["one", "one", "same", "ragged", "mixed"])
    n_seq = _log(rng, 1, 100) if kind != "same" else _log(rng, 1, 12)
    c = dict(op=op, n_seq=n_seq, mix=kind, heads=heads, kv=kv, hd=hd, page=page, beside=rng.random() < 0.5, pad=rng.choice([0, 0, 3, 40]), shape_seed=rng.randint(1, 10 ** 6))
    if op == "append":
        c.update(q=1 if kind == "one" else _log(rng, 2, 6000 // n_seq + 3), past_min=0, past=_log(rng, 1, 20000 // n_seq + 10), axes=rng.choice([1, 1, 3]),
                 rot=rng.choice([hd, hd, hd // 2]), layout=rng.choice([0, 1, 1]), norm=rng.random() < 0.6, f32=rng.random() < 0.3)
        return c
    c["q"] = 1 if kind == "one" else _log(rng, 2, max(8, 1500 // n_seq))
    c["past_min"] = rng.choice([0, 0, 10])
    c["past"] = _log(rng, 20, 90000 // n_seq if kind == "one" else 8000 // max(1, n_seq // 8))
    c["window"] = rng.choice([0, 0, 0, _log(rng, 16, 4000)])
    c["evicted"] = c["window"] > 0 and rng.random() < 0.6
    return c


def _shape(case):
    """Tokens and cached positions (these tokens included) of every sequence of a case, and the rows of the panel."""
    r, n, q = random.Random(case["shape_seed"]), case["n_seq"], case["q"]
    some = {"one": lambda i: 1, "same": lambda i: q, "ragged": lambda i: r.randint(1, q), "mixed": lambda i: r.randint(1, q) if i % 8 == 3 or n < 4 else 1}[case["mix"]]
    new = np.array([some(i) for i in range(n)])
    past = np.array([r.randint(case["past_min"], case["past"]) for i in range(n)])
    if case["mix"] == "mixed" and n >= 8:
        new[n // 2], new[5], past[5] = 0, 0, 0  # a slot without new tokens, and one without any
    return new, past + new, int(new.sum()) + case["pad"]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 71)
    return g


def _rotation(case, g, rows):
    """Frequencies in 64 bits, the axis of every pair (runs of pairs per axis), and the positions on every axis."""
    pairs, axes = case["rot"] // 2, case["axes"]
    s = dict(freq=THETA ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs))
    s["axis"] = (torch.arange(pairs, device="cuda") * axes // pairs).int()
    s["pos"] = torch.randint(0, 4000 if axes > 1 else 120000, (axes, rows), generator=g, device="cuda", dtype=torch.int32)
    return s


def prepare(case, seed):
    g = _gen(seed)
    rnd = lambda *shape, sigma=1.0: torch.randn(*shape, generator=g, device="cuda") * sigma  # noqa: E731
    s = dict(case)
    f = torch.float32 if case.get("f32") else torch.bfloat16
    if case["op"] == "rope":
        wide = case["heads"] * case["hd"] + (case["hd"] * 8 if case["fused"] else 0)
        s["panel"] = rnd(case["M"], wide).to(f)
        s["x"] = s["panel"][:, :case["heads"] * case["hd"]]
        s["out"] = torch.zeros(case["M"], case["heads"] * case["hd"], device="cuda", dtype=f)
        s.update(_rotation(case, g, case["M"]))
        return s
    heads, kv, hd, page = case["heads"], case["kv"], case["hd"], case["page"]
    new, length, rows = _shape(case)
    start = np.concatenate([[0], np.cumsum(new)])
    held = -(-length // page)
    n_pages = int(held.sum()) + 3 + int(held.sum()) // 10
    cols = int(held.max()) + 1
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    j = torch.arange(cols, device="cuda")
    held_d, first = torch.from_numpy(held).cuda(), torch.from_numpy(np.concatenate([[0], np.cumsum(held)[:-1]])).cuda()
    at = (first[:, None] + j).clamp(max=n_pages - 1)
    there = j < held_d[:, None]
    if case.get("evicted"):  # the first position that a new token still sees
        lo = torch.from_numpy(np.maximum(length - new - case["window"] + 1, 0)).cuda()
        there &= (j + 1) * page > lo[:, None]
    s["table"] = torch.where(there, order[at], -1).int()
    s["start"], s["len"] = torch.from_numpy(start).int().cuda(), torch.from_numpy(length).int().cuda()
    s["rows"], s["n_pages"], s["cols"], s["max_q"], s["max_len"], s["n_new"] = rows, n_pages, cols, int(new.max()), int(length.max()), int(start[-1])
    if case["beside"]:
        pool = rnd(n_pages, 2, page, kv, hd, sigma=1.2).bfloat16()
        s["k_pool"], s["v_pool"] = pool[:, 0], pool[:, 1]
    else:
        s["k_pool"], s["v_pool"] = rnd(n_pages, page, kv, hd, sigma=1.2).bfloat16(), rnd(n_pages, page, kv, hd, sigma=0.6).bfloat16()
    if case["op"] == "append":
        s["qkv"] = rnd(rows, (heads + 2 * kv) * hd).to(f)  # q, k and v of a token lie in one row of the fused projection
        s["q"], s["k"], s["v"] = s["qkv"][:, :heads * hd], s["qkv"][:, heads * hd:(heads + kv) * hd], s["qkv"][:, (heads + kv) * hd:]
        s.update(_rotation(case, g, rows))
        if case["axes"] == 1:
            s["pos"] = None  # text: the position in the cache
        s["q_norm"], s["k_norm"] = ((1.2 + rnd(hd, sigma=0.1)).bfloat16() for _ in "qk") if case["norm"] else (None, None)
    else:
        s["q"] = rnd(rows, heads * hd, sigma=1.2).bfloat16()
    s["out"] = rnd(rows, heads * hd).bfloat16()  # rows behind the last sequence stay as they are
    return s


# ---------------------------------------------------------------------------------------------------------------- the library's calls
class _At:
    """Device memory as the package's functions take it."""

    def __init__(self, t):
        self.ptr = t.data_ptr()


_CTX = {}  # by device and stream: a context's kernels go to the stream it was made for


def _handles(s, device, stream):
    """What a program keeps between its calls: the context, the descriptions of the cache and of the rotation, the addresses."""
    import koifish_b200 as kf
    if (device, stream) not in _CTX:
        _CTX[device, stream] = kf.Context(device, stream=stream or 1)  # 1: the handle of torch's default stream
    at = {n: _At(t) for n, t in s.items() if isinstance(t, torch.Tensor)}
    h = dict(kf=kf, ctx=_CTX[device, stream], at=at, stream=stream)
    if s["op"] != "attention":
        h["rot"] = kf.Rotation(at["freq"], s["rot"], layout=s["layout"], n_axes=s["axes"], pair_axis=at["axis"] if s["axes"] > 1 else None, pos=at.get("pos"))
    if s["op"] != "rope":
        h["kv"] = kf.PagedKV(at["k_pool"], at["v_pool"], s["n_pages"], s["page"], s["kv"], s["hd"], at["table"], s["cols"], s["n_seq"], at["start"], at["len"],
                             page_stride=s["k_pool"].stride(0))
    return h


def _own(s):
    h, device = s.get("handles"), s["out"].get_device()
    stream = torch._C._cuda_getCurrentRawStream(device)  # 0.1 us; torch.cuda.current_stream() makes an object, 3 us, as long as the whole call
    if h is None or h["stream"] != stream:
        h = s["handles"] = _handles(s, device, stream)
    kf, ctx, at = h["kf"], h["ctx"], h["at"]
    if s["op"] == "rope":
        kf.rope_axes(ctx, h["rot"], at["x"], s["M"], s["heads"], s["hd"], ldx=s["x"].stride(0), out=at["out"], f32=s["f32"])
    elif s["op"] == "append":
        ld = s["qkv"].stride(0)
        kf.paged_append(ctx, h["kv"], h["rot"], at["q"], at["k"], at["v"], s["rows"], s["heads"], q_norm=at.get("q_norm"), k_norm=at.get("k_norm"), eps=EPS,
                        ldq=ld, ldk=ld, ldv=ld, out=at["out"], src_f32=s["f32"])
        return s["out"], s["k_pool"], s["v_pool"]
    else:
        kf.paged_attention(ctx, h["kv"], at["q"], s["rows"], s["heads"], max_q=s["max_q"], window=s["window"], out=at["out"])
    return s["out"]


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _rotated(x, s, pos):
    """x [rows, heads, hd] float rotated by the angles of pos [axes, rows]"""
    angle = pos.double()[s["axis"].long()].T * s["freq"]  # [rows, pairs], 64 bits: far positions turn many times
    c, d = angle.cos().float()[:, None], angle.sin().float()[:, None]
    n = s["rot"] // 2
    if s["layout"]:
        a, b = x[..., :n], x[..., n:2 * n]
        return torch.cat([a * c - b * d, b * c + a * d, x[..., 2 * n:]], -1)
    a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
    return torch.cat([torch.stack([a * c - b * d, b * c + a * d], -1).flatten(-2), x[..., 2 * n:]], -1)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _plain_rope(s):
    x = s["x"].float().reshape(s["M"], s["heads"], s["hd"])
    s["out"].copy_(_rotated(x, s, s["pos"]).flatten(1))
    return s["out"]


def _owner(s):
    """Sequence and cached position of every new token."""
    row = torch.arange(s["n_new"], device="cuda")
    seq = torch.searchsorted(s["start"][1:].long(), row, right=True)
    return seq, s["len"][seq].long() - s["start"][seq + 1] + row


def _plain_append(s):
    n, heads, kv, hd, page = s["n_new"], s["heads"], s["kv"], s["hd"], s["page"]
    seq, place = _owner(s)
    pos = place.expand(s["axes"], n) if s["pos"] is None else s["pos"][:, :n]
    q, k = (_rotated(_normed(s[name][:n].float().reshape(n, h, hd), s[name + "_norm"]), s, pos) for name, h in (("q", heads), ("k", kv)))
    at, inside = s["table"][seq, place // page].long(), place % page
    s["k_pool"][at, inside] = k.bfloat16()
    s["v_pool"][at, inside] = s["v"][:n].reshape(n, kv, hd).bfloat16()
    s["out"][:n] = q.flatten(1).bfloat16()
    return s["out"], s["k_pool"], s["v_pool"]


def _plain_attention(s):
    heads, kv, hd, page, n = s["heads"], s["kv"], s["hd"], s["page"], s["n_new"]
    key = torch.arange(s["max_len"], device="cuda")
    at = s["table"][:, key // page].long()
    k, v = (s[name][at.clamp(min=0), key % page].float() for name in ("k_pool", "v_pool"))  # [seq, positions, kv, hd]
    new = (s["start"][1:] - s["start"][:-1]).long()
    i = torch.arange(s["max_q"], device="cuda")
    row = (s["start"][:-1, None].long() + i).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().reshape(s["n_seq"], s["max_q"], kv, heads // kv, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [seq, kv, group x tokens, hd]
    place = (s["len"].long() - new)[:, None] + i
    sees = (key <= place[..., None]) & (at >= 0)[:, None]
    sees = sees & (key > place[..., None] - s["window"]) if s["window"] else sees
    sees = sees[:, None].repeat(1, 1, heads // kv, 1)  # rows in the order of q's
    w = (q @ k.permute(0, 2, 3, 1)).mul_(hd ** -0.5).masked_fill_(~sees, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    o = (w @ v.permute(0, 2, 1, 3)) / torch.where(total == 0, 1, total)
    o = o.view(s["n_seq"], kv, heads // kv, s["max_q"], hd).permute(0, 3, 1, 2, 4).flatten(2)  # [seq, tokens, heads x hd]
    seq, at = _owner(s)
    s["out"][:n] = o[seq, at - (s["len"].long() - new)[seq]].bfloat16()
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "append": _plain_append, "attention": _plain_attention}[state["op"]](state)


# ---------------------------------------------------------------------------------------------------------------- cost, 64-bit results
def work(case):
    if case["op"] == "rope":
        x = case["M"] * case["heads"] * case["hd"]
        return dict(bytes=x * (8 if case["f32"] else 4) + case["M"] * case["axes"] * 4, flops=3.0 * x)
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    new, length, _ = _shape(case)
    if case["op"] == "append":
        x = int(new.sum()) * (heads + 2 * kv) * hd
        return dict(bytes=x * (6 if case["f32"] else 4) + int(new.sum()) * 4 * (case["axes"] + 1), flops=(7.0 if case["norm"] else 3.0) * x)
    far = case["window"] or 10 ** 9
    read, pairs = 0, 0
    for n, e in zip(new.tolist(), length.tolist()):
        last = np.arange(e - n, e)  # positions of the new tokens
        pairs += int(np.minimum(last + 1, far).sum())
        read += e - max(0, e - n - far + 1) if n else 0
    return dict(bytes=4.0 * read * kv * hd + 4.0 * int(new.sum()) * heads * hd, flops=4.0 * pairs * heads * hd)


def _turned(x, freq, axis, pos, layout):
    """Rows [.., hd] in 64 bits, their pairs taken as complex numbers and turned by e^(i angle)."""
    n = freq.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.stack([pos[a].double() * f for a, f in zip(axis.tolist(), freq)], -1))
    x = x.double().clone()
    a, b = (slice(0, n), slice(n, 2 * n)) if layout else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    z = torch.complex(x[..., a], x[..., b]) * turn[:, None, :]
    x[..., a], x[..., b] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    heads, hd = s["heads"], s["hd"]
    if s["op"] == "rope":
        return _turned(s["x"].reshape(s["M"], heads, hd), s["freq"], s["axis"], s["pos"], s["layout"]).reshape(s["M"], -1)
    kv, page, start, length, table = s["kv"], s["page"], s["start"].tolist(), s["len"].tolist(), s["table"].long()
    out = s["out"].double()
    if s["op"] == "append":
        k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
        for i in range(s["n_seq"]):
            a, b = start[i], start[i + 1]
            if a == b:
                continue
            place = torch.arange(length[i] - (b - a), length[i], device="cuda")
            pos = [place] * s["axes"] if s["pos"] is None else list(s["pos"][:, a:b])
            done = []
            for x, w, h in ((s["q"], s["q_norm"], heads), (s["k"], s["k_norm"], kv)):
                x = x[a:b].double().reshape(b - a, h, hd)
                if w is not None:
                    x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
                done.append(_turned(x, s["freq"], s["axis"], pos, s["layout"]))
            out[a:b] = done[0].reshape(b - a, -1)
            k_pool[table[i, place // page], place % page] = done[1]
            v_pool[table[i, place // page], place % page] = s["v"][a:b].double().reshape(b - a, kv, hd)
        return out, k_pool, v_pool
    for i in range(s["n_seq"]):
        a, b, e = start[i], start[i + 1], length[i]
        if a == b:
            continue
        pages = table[i, :-(-e // page)]
        held = (pages >= 0).repeat_interleave(page)[:e]
        k, v = (s[name][pages.clamp(min=0)].double().reshape(-1, kv, hd)[:e] for name in ("k_pool", "v_pool"))
        here = torch.arange(e, device="cuda")
        for h in range(heads):
            g = h // (heads // kv)
            for r in range(a, b, 1024):  # rows of the panel at a time
                n = min(b, r + 1024) - r
                at = torch.arange(e - (b - r), e - (b - r) + n, device="cuda")[:, None]
                hidden = (here > at) | ~held
                if s["window"]:
                    hidden = hidden | (here <= at - s["window"])
                p = torch.softmax((s["q"][r:r + n, h * hd:(h + 1) * hd].double() @ k[:, g].T / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1)
                out[r:r + n, h * hd:(h + 1) * hd] = torch.nan_to_num(p, nan=0.0) @ v[:, g]
    return out
