"""Timed cases of a paged cache held in 4 bits, in plain torch and through the library.

Operators
  append     keys and values of a step's new tokens, quantised into the pages of their sequences; RMS norm of every head of q and k and the rotation by one or several position
             axes on the way, the finished queries written beside.  The rows are read back behind it: what the cache stands for is what is compared
  read       the cached keys and values of ranges of positions back as rows of 16- or 32-bit numbers
  attention  the step's queries (one token, a few drafted ones or a chunk of a prompt for each sequence, any mixture of them) over the positions that their sequences hold, causal,
             optionally over the last `window` positions and the `first` ones only

Every 32 entries of a cached row are a group with a step and a zero in bf16: a code c of 0 .. 15 stands for step * (c - zero), with
  step = max((max - min) / 15, max |x| / 2048) rounded up to bf16,  zero = -min / step rounded to bf16,  c = x / step + zero rounded to a whole number and kept to 0 .. 15.
A page holds, for each kv head, units of 8 positions, one after the other: key codes, steps [8][groups] and zeros [8][groups] of the keys, value codes, steps [8][groups] and zeros
[groups][8] of the values.  Key codes: a row of head_dim / 2 bytes a position, its words [4][groups], word (t, j) the entries 32 j + 8 t ..+ 7 from the lowest 4 bits up.  Value
codes: words [8][4][2][groups / 2], word (g, p / 2, p % 2, w) of position p: entries 64 w + 4 g ..+ 3, then 64 w + 32 + 4 g ..+ 3.

A step is described as a server has it on the device: first row and number of cached positions of every sequence, and a table of its pages.

Fields of a case: n_seq sequences with `mix` saying how many tokens each brings (one: 1 each; same: q each; ragged: 1 .. q; mixed: one sequence in eight 1 .. q, the others 1, with
an idle slot and an empty one among them; all: every position, as a read of whole sequences wants), past_min .. past positions in front of them, `pad` rows of the panel behind the
last sequence; heads / kv / hd the head layout, page the positions of a page, layers: layers whose pages lie beside one another in the pool, of which the case has one; axes, rot,
layout, norm, f32 the rotation, the norms and the type of the rows; window, first and evicted (pages that no window nor the first positions need are gone from the table); shape_seed
draws the lengths.
"""
import math
import random

import numpy as np
import torch

own = False
EPS = 1e-6
THETA = 1e6
GROUP = 32


def listed():
    a = dict(op="append", pad=0, layers=1, axes=1, rot=128, layout=1, norm=True, f32=False, hd=128)
    r = dict(op="read", pad=0, layers=1, f32=False, hd=128)
    t = dict(op="attention", pad=0, layers=1, window=0, first=0, evicted=False, hd=128)
    return [
        # a decode step of a few users: the smallest call, all of it latency
        dict(a, name="append_decode", n_seq=8, mix="one", q=1, past_min=200, past=4000, heads=32, kv=8, page=16, shape_seed=1),
        # image and text tokens of prompts with three position axes, no norm, float projections
        dict(a, name="append_image", n_seq=3, mix="ragged", q=3000, past_min=0, past=500, heads=32, kv=8, page=64, axes=3, norm=False, f32=True, shape_seed=3),
        # a full step of prompt chunks on the widest block, two layers' pages beside one another
        dict(a, name="append_panel", n_seq=4, mix="same", q=2000, past_min=0, past=2000, heads=64, kv=8, page=16, layers=2, pad=7, shape_seed=4),
        # a short prefix of a few users, small heads, as floats
        dict(r, name="read_short", n_seq=5, mix="all", q=1, past_min=20, past=150, heads=8, kv=4, page=24, hd=64, f32=True, shape_seed=11),
        # the whole of a long conversation for a cache of another kind
        dict(r, name="read_long", n_seq=2, mix="all", q=1, past_min=20000, past=30000, heads=32, kv=8, page=32, shape_seed=12),
        # one user, short context: latency
        dict(t, name="attn_one", n_seq=1, mix="one", q=1, past_min=1300, past=1300, heads=32, kv=8, page=16, shape_seed=5),
        # batched decoding over ragged contexts
        dict(t, name="attn_batch", n_seq=64, mix="one", q=1, past_min=400, past=4000, heads=64, kv=8, page=16, layers=2, shape_seed=6),
        # one user deep into a long context
        dict(t, name="attn_long", n_seq=1, mix="one", q=1, past_min=100000, past=100000, heads=64, kv=8, page=64, shape_seed=7),
        # many users whose old pages were given back: the last 1000 positions and the first 4
        dict(t, name="attn_stream", n_seq=40, mix="one", q=1, past_min=500, past=30000, heads=40, kv=8, page=16, window=1000, first=4, evicted=True, shape_seed=13),
        # a few drafted tokens per user to be verified, an odd page size
        dict(t, name="attn_draft", n_seq=16, mix="same", q=5, past_min=500, past=5000, heads=40, kv=8, page=24, shape_seed=8),
        # the next chunk of a long prompt
        dict(t, name="attn_chunk", n_seq=1, mix="same", q=2048, past_min=8192, past=8192, heads=32, kv=8, page=16, shape_seed=9),
        # chunks of prompts and decoding users in one step, small heads, the last 1000 positions and the first 64, older pages given back
        dict(t, name="attn_mixed", n_seq=24, mix="mixed", q=700, past_min=20, past=5000, heads=28, kv=4, page=32, window=1000, first=64, evicted=True, hd=64, pad=5, shape_seed=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "attention", "attention", "attention", "attention"])
    hd = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 7, 8, 8, 12])
    page = rng.choice([8, 16, 16, 24, 32, 48, 64, 128, 256])
    kind = "all" if op == "read" else rng.choice(["one", "one", "same", "ragged", "mixed"])
    n_seq = _log(rng, 1, 100) if kind not in ("same", "all") else _log(rng, 1, 12)
    c = dict(op=op, n_seq=n_seq, mix=kind, heads=heads, kv=kv, hd=hd, page=page, layers=rng.choice([1, 1, 2, 3]), pad=rng.choice([0, 0, 3, 40]), shape_seed=rng.randint(1, 10 ** 6))
    if op == "read":
        c.update(q=1, past_min=0, past=_log(rng, 4, 50000 // n_seq), f32=rng.random() < 0.3)
        return c
    if op == "append":
        c.update(q=1 if kind == "one" else _log(rng, 2, 5000 // n_seq + 3), past_min=0, past=_log(rng, 1, 20000 // n_seq + 10), axes=rng.choice([1, 1, 3]),
                 rot=rng.choice([hd, hd, hd // 2]), layout=rng.choice([0, 1, 1]), norm=rng.random() < 0.6, f32=rng.random() < 0.3)
        return c
    c["q"] = 1 if kind == "one" else _log(rng, 2, max(8, 1500 // n_seq))
    c["past_min"] = rng.choice([0, 0, 10])
    c["past"] = _log(rng, 20, 90000 // n_seq if kind == "one" else 8000 // max(1, n_seq // 8))
    c["window"] = rng.choice([0, 0, 0, _log(rng, 16, 4000)])
    c["first"] = rng.choice([0, 1, 4, 40, 200]) if c["window"] else 0
    c["evicted"] = c["window"] > 0 and rng.random() < 0.6
    return c


def _shape(case):
    """Tokens and cached positions (these tokens included) of every sequence of a case, and the rows of the panel."""
    r, n, q = random.Random(case["shape_seed"]), case["n_seq"], case["q"]
    some = {"one": lambda i: 1, "same": lambda i: q, "ragged": lambda i: r.randint(1, q), "mixed": lambda i: r.randint(1, q) if i % 8 == 3 or n < 4 else 1, "all": lambda i: 1}[case["mix"]]
    new = np.array([some(i) for i in range(n)])
    past = np.array([r.randint(case["past_min"], case["past"]) for i in range(n)])
    if case["mix"] == "all":
        new, past = new + past, past * 0
    if case["mix"] == "mixed" and n >= 8:
        new[n // 2], new[5], past[5] = 0, 0, 0  # a slot without new tokens, and one without any
    return new, past + new, int(new.sum()) + case["pad"]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 97)
    return g


# ---------------------------------------------------------------------------------------------------------------- the format, in plain torch
def _unit(hd):
    """Bytes of 8 positions of a head."""
    return 8 * hd + 2 * hd


def _quantised(x):
    """x [..., hd] float -> whole-number codes [..., groups, 32], steps and zeros [..., groups] as floats that bf16 holds"""
    x = x.unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(-1), x.amax(-1)
    step = torch.maximum((hi - lo) / torch.full_like(lo, 15), torch.maximum(hi, -lo) / 2048)  # divided, not times the rounded 1 / 15
    step = ((step.view(torch.int32) + 0xffff) & -0x10000).view(torch.float32)  # up, to bf16
    some = torch.where(step > 0, step, 1.0)
    zero = torch.where(step > 0, -lo / some, 0.0).bfloat16().float()
    return (x / some[..., None] + zero[..., None]).round().clamp(0, 15), step, zero


def _views(s):
    """The parts of every (page, head, unit): key codes [8, bytes], key steps, key zeros, value codes [8, 4, 2, bytes], value steps, value zeros."""
    hd, ng = s["hd"], s["hd"] // GROUP
    u = s["pages"].unflatten(-1, (s["kv"], s["page"] // 8, _unit(hd)))
    at, out = 0, []
    for n, shape, what in ((4 * hd, (8, hd // 2), None), (16 * ng, (8, ng), 1), (16 * ng, (8, ng), 1), (4 * hd, (8, 4, 2, hd // 16), None), (16 * ng, (8, ng), 1), (16 * ng, (ng, 8), 1)):
        part = u[..., at:at + n]
        out.append((part.view(torch.bfloat16) if what else part).unflatten(-1, shape))
        at += n
    return out


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _bytes(c):
    c = c.to(torch.uint8).unflatten(-1, (-1, 2))
    return c[..., 0] | c[..., 1] << 4


def _store(s, page, row, k, v):
    """Keys and values [n, kv, hd] as floats into rows `row` of pages `page`."""
    kc, ks, kz, vc, vs, vz = _views(s)
    unit, p, ng = row // 8, row % 8, s["hd"] // GROUP
    c, step, zero = _quantised(k)
    kc[page, :, unit, p] = _bytes(c.unflatten(-1, (4, 8)).transpose(-3, -2).flatten(-3))
    ks[page, :, unit, p], kz[page, :, unit, p] = step.bfloat16(), zero.bfloat16()
    c, step, zero = _quantised(v)
    c = c.unflatten(-1, (8, 4)).unflatten(-3, (ng // 2, 2)).permute(0, 1, 4, 2, 3, 5).flatten(-3)  # [n, kv, 8, w | half | entry]
    vc[page, :, unit, :, p // 2, p % 2] = _bytes(c)
    vs[page, :, unit, p], vz[page, :, unit, :, p] = step.bfloat16(), zero.bfloat16()


def _load(s, page, row):
    """Keys and values [..., kv, hd] that rows `row` of pages `page` stand for, as floats."""
    kc, ks, kz, vc, vs, vz = _views(s)
    shape, page, row = page.shape, page.flatten(), row.flatten()
    unit, p, ng = row // 8, row % 8, s["hd"] // GROUP
    k = _nibbles(kc[page, :, unit, p]).unflatten(-1, (4, ng, 8)).transpose(-3, -2).flatten(-2).float()
    k = k.sub_(kz[page, :, unit, p].float()[..., None]).mul_(ks[page, :, unit, p].float()[..., None]).flatten(-2)
    v = _nibbles(vc[page, :, unit, :, p // 2, p % 2]).unflatten(-1, (ng // 2, 2, 4)).permute(0, 1, 3, 4, 2, 5).flatten(-2).flatten(-3, -2).float()
    v = v.sub_(vz[page, :, unit, :, p].float()[..., None]).mul_(vs[page, :, unit, p].float()[..., None]).flatten(-2)
    return k.unflatten(0, shape), v.unflatten(0, shape)


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = _gen(seed)
    rnd = lambda *shape, sigma=1.0: torch.randn(*shape, generator=g, device="cuda") * sigma  # noqa: E731
    s = dict(case)
    heads, kv, hd, page = case["heads"], case["kv"], case["hd"], case["page"]
    new, length, rows = _shape(case)
    start = np.concatenate([[0], np.cumsum(new)])
    held = -(-length // page)
    n_pages = int(held.sum()) + 3 + int(held.sum()) // 10
    cols = int(held.max()) + 1
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    j = torch.arange(cols, device="cuda")
    held_d, before = torch.from_numpy(held).cuda(), torch.from_numpy(np.concatenate([[0], np.cumsum(held)[:-1]])).cuda()
    at = (before[:, None] + j).clamp(max=n_pages - 1)
    there = j < held_d[:, None]
    if case.get("evicted"):  # the last positions that a new token still sees, and the first ones
        lo = torch.from_numpy(np.maximum(length - new - case["window"] + 1, 0)).cuda()
        there &= ((j + 1) * page > lo[:, None]) | (j * page < case["first"])
    s["table"] = torch.where(there, order[at], -1).int()
    s["start"], s["len"] = torch.from_numpy(start).int().cuda(), torch.from_numpy(length).int().cuda()
    s["rows"], s["n_pages"], s["cols"], s["max_q"], s["max_len"], s["n_new"] = rows, n_pages, cols, int(new.max()), int(length.max()), int(start[-1])
    bytes_ = page // 8 * kv * _unit(hd)
    s["pool"] = torch.empty(n_pages, case["layers"], bytes_, device="cuda", dtype=torch.uint8)
    s["pages"] = s["pool"][:, case["layers"] - 1]
    row = torch.arange(page, device="cuda")
    for a in range(0, n_pages, 1 + (1 << 25) // (page * kv * hd)):  # what lies in the pages was quantised before, a part of them at a time
        which = torch.arange(a, min(n_pages, a + 1 + (1 << 25) // (page * kv * hd)), device="cuda").repeat_interleave(page)
        _store(s, which, row.repeat(len(which) // page), rnd(len(which), kv, hd, sigma=1.2), rnd(len(which), kv, hd, sigma=0.6))
    f = torch.float32 if case.get("f32") else torch.bfloat16
    if case["op"] == "append":
        s["qkv"] = rnd(rows, (heads + 2 * kv) * hd)  # q, k and v of a token lie in one row of the fused projection
        s["qkv"][:, (heads + kv) * hd:] *= 2
        s["qkv"] = s["qkv"].to(f)
        s["q"], s["k"], s["v"] = s["qkv"][:, :heads * hd], s["qkv"][:, heads * hd:(heads + kv) * hd], s["qkv"][:, (heads + kv) * hd:]
        pairs, axes = case["rot"] // 2, case["axes"]
        s["freq"] = THETA ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
        s["axis"] = (torch.arange(pairs, device="cuda") * axes // pairs).int()  # runs of pairs per axis
        s["pos"] = torch.randint(0, 4000, (axes, rows), generator=g, device="cuda", dtype=torch.int32) if axes > 1 else None  # text: the position in the cache
        s["q_norm"], s["k_norm"] = ((0.9 + rnd(hd, sigma=0.1)).bfloat16() for _ in "qk") if case["norm"] else (None, None)
    elif case["op"] == "attention":
        s["q"] = rnd(rows, heads * hd, sigma=1.2).bfloat16()
    if case["op"] != "read":
        s["out"] = rnd(rows, heads * hd).bfloat16()  # rows behind the last sequence stay as they are
    if case["op"] != "attention":
        s["back"] = rnd(rows, 2 * kv * hd).to(torch.float32 if case["op"] == "read" and case["f32"] else torch.bfloat16)  # keys and values of a position beside one another
        s["back_k"], s["back_v"] = s["back"][:, :kv * hd], s["back"][:, kv * hd:]
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
    if s["op"] == "append":
        h["rot"] = kf.Rotation(at["freq"], s["rot"], layout=s["layout"], n_axes=s["axes"], pair_axis=at["axis"] if s["axes"] > 1 else None, pos=at.get("pos"))
    h["kv"] = kf.PagedQ4(at["pages"], s["n_pages"], s["page"], s["kv"], s["hd"], at["table"], s["cols"], s["n_seq"], at["start"], at["len"], page_stride=s["pages"].stride(0))
    return h


def _own(s):
    h, device = s.get("handles"), s["pages"].get_device()
    stream = torch._C._cuda_getCurrentRawStream(device)  # 0.1 us; torch.cuda.current_stream() makes an object, 3 us, as long as the whole call
    if h is None or h["stream"] != stream:
        h = s["handles"] = _handles(s, device, stream)
    kf, ctx, at = h["kf"], h["ctx"], h["at"]
    if s["op"] == "attention":
        kf.paged_attention_q4(ctx, h["kv"], at["q"], s["rows"], s["heads"], max_q=s["max_q"], window=s["window"], first=s["first"], out=at["out"])
        return s["out"]
    if s["op"] == "append":
        ld = s["qkv"].stride(0)
        kf.paged_append_q4(ctx, h["kv"], h["rot"], at["q"], at["k"], at["v"], s["rows"], s["heads"], q_norm=at.get("q_norm"), k_norm=at.get("k_norm"), eps=EPS,
                           ldq=ld, ldk=ld, ldv=ld, out=at["out"], src_f32=s["f32"])
    ld = s["back"].stride(0)
    kf.paged_read_q4(ctx, h["kv"], s["rows"], k_out=at["back_k"], v_out=at["back_v"], ldk=ld, ldv=ld, out_f32=s["back"].dtype == torch.float32)
    return (s["out"], s["back"]) if s["op"] == "append" else s["back"]


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


def _owner(s):
    """Sequence and cached position of every new token."""
    row = torch.arange(s["n_new"], device="cuda")
    seq = torch.searchsorted(s["start"][1:].long(), row, right=True)
    return seq, s["len"][seq].long() - s["start"][seq + 1] + row


def _plain_read(s):
    n, (seq, place) = s["n_new"], _owner(s)
    k, v = _load(s, s["table"][seq, place // s["page"]].long(), place % s["page"])
    s["back_k"][:n], s["back_v"][:n] = k.flatten(1), v.flatten(1)
    return s["back"]


def _plain_append(s):
    n, heads, kv, hd, page = s["n_new"], s["heads"], s["kv"], s["hd"], s["page"]
    seq, place = _owner(s)
    pos = place.expand(s["axes"], n) if s["pos"] is None else s["pos"][:, :n]
    q, k = (_rotated(_normed(s[name][:n].float().reshape(n, h, hd), s[name + "_norm"]), s, pos) for name, h in (("q", heads), ("k", kv)))
    _store(s, s["table"][seq, place // page].long(), place % page, k, s["v"][:n].float().reshape(n, kv, hd))
    s["out"][:n] = q.flatten(1).bfloat16()
    return s["out"], _plain_read(s)


def _plain_attention(s):
    heads, kv, hd, page, n = s["heads"], s["kv"], s["hd"], s["page"], s["n_new"]
    key = torch.arange(s["max_len"], device="cuda")
    at = s["table"][:, key // page].long()
    k, v = _load(s, at.clamp(min=0), (key % page).expand_as(at))  # [seq, positions, kv, hd]
    new = (s["start"][1:] - s["start"][:-1]).long()
    i = torch.arange(s["max_q"], device="cuda")
    row = (s["start"][:-1, None].long() + i).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().reshape(s["n_seq"], s["max_q"], kv, heads // kv, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [seq, kv, group x tokens, hd]
    place = (s["len"].long() - new)[:, None] + i
    sees = (key <= place[..., None]) & (at >= 0)[:, None]
    sees = sees & ((key > place[..., None] - s["window"]) | (key < s["first"])) if s["window"] else sees
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
    return {"read": _plain_read, "append": _plain_append, "attention": _plain_attention}[state["op"]](state)


# ---------------------------------------------------------------------------------------------------------------- cost, 64-bit results
def work(case):
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    new, length, _ = _shape(case)
    n, cached = int(new.sum()), _unit(hd) / 8 * kv  # bytes of a position's keys and values
    if case["op"] == "read":
        return dict(bytes=n * (cached + 2 * kv * hd * (4 if case["f32"] else 2)), flops=4.0 * n * kv * hd)
    if case["op"] == "append":
        src = 4 if case["f32"] else 2
        move = n * (heads * hd * (src + 2) + 2 * kv * hd * src + cached) + n * (cached + 4 * kv * hd)  # and read back
        return dict(bytes=move + n * 4.0 * (case["axes"] + 1), flops=n * hd * ((heads + kv) * (7.0 if case["norm"] else 3.0) + 12.0 * kv))
    far = case["window"] or 10 ** 9
    read, pairs = 0, 0
    for m, e in zip(new.tolist(), length.tolist()):
        lo = np.maximum(np.arange(e - m, e) - far + 1, 0)  # the first position inside the window of every new token
        pairs += int((np.arange(e - m, e) + 1 - lo + np.minimum(lo, case["first"])).sum())
        read += e - max(0, e - m - far + 1) + min(case["first"], max(0, e - m - far + 1)) if m else 0
    return dict(bytes=read * cached + 4.0 * n * heads * hd, flops=4.0 * pairs * heads * hd)


def _turned(x, freq, axis, pos, layout):
    """Rows [.., hd] in 64 bits, their pairs taken as complex numbers and turned by e^(i angle)."""
    n = freq.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.stack([pos[a].double() * f for a, f in zip(axis.tolist(), freq)], -1))
    x = x.double().clone()
    a, b = (slice(0, n), slice(n, 2 * n)) if layout else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    z = torch.complex(x[..., a], x[..., b]) * turn[:, None, :]
    x[..., a], x[..., b] = z.real, z.imag
    return x


def _to_bf16(x, up):
    """64-bit values at one of 8 bits of mantissa: the next one up, or the nearest."""
    m, e = torch.frexp(x)
    m = m * 256
    return torch.ldexp(torch.ceil(m) if up else torch.round(m), e - 8)


def _stands_for(x):
    """What the cache makes of rows [.., hd], in 64 bits."""
    done = torch.empty_like(x)
    for j in range(0, x.shape[-1], GROUP):
        y = x[..., j:j + GROUP]
        lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        step = _to_bf16(torch.maximum((hi - lo) / 15.0, torch.maximum(hi.abs(), lo.abs()) / 2048.0), True)
        zero = _to_bf16(-lo / step, False)
        done[..., j:j + GROUP] = step * (torch.clip(torch.round(y / step + zero), 0.0, 15.0) - zero)
    return torch.nan_to_num(done, nan=0.0)  # groups of zeros


def _held(s, i, value):
    """Keys or values of sequence i, [positions, kv, hd] in 64 bits, each entry looked up at its own place in the pool's bytes."""
    n, kv, hd, page, ng = int(s["len"][i]), s["kv"], s["hd"], s["page"], s["hd"] // GROUP
    p, h, d = (torch.arange(m, device="cuda") for m in (n, kv, hd))
    e = s["table"][i, p // page].long().clamp(min=0) * s["pool"][0].numel() + (s["layers"] - 1) * s["pages"].shape[1]
    unit = (e + p % page // 8 * _unit(hd))[:, None, None] + (h * (page // 8) * _unit(hd))[:, None]
    r = (p % 8)[:, None, None]
    flat, codes, table = s["pool"].view(-1), 4 * hd, 16 * ng
    if value:
        at = unit + codes + 2 * table
        byte = at + (d % 32 // 4) * (hd // 2) + r // 2 * (hd // 8) + r % 2 * (hd // 16) + d // 64 * 4 + d // 32 % 2 * 2 + d % 4 // 2
        step, zero = at + codes + 2 * (r * ng + d // 32), at + codes + table + 2 * (d // 32 * 8 + r)
    else:
        byte = unit + r * (hd // 2) + (d % 32 // 8) * (4 * ng) + d // 32 * 4 + d % 8 // 2
        step, zero = unit + codes + 2 * (r * ng + d // 32), unit + codes + table + 2 * (r * ng + d // 32)
    number = lambda a: ((flat[a].int() | flat[a + 1].int() << 8) << 16).view(torch.float32).double()  # noqa: E731
    code = torch.where(d % 2 == 1, flat[byte] >> 4, flat[byte] & 15).double()
    return number(step) * (code - number(zero))


def exact(case, seed):
    s = prepare(case, seed)
    heads, hd, kv, start, length = s["heads"], s["hd"], s["kv"], s["start"].tolist(), s["len"].tolist()
    if s["op"] == "read":
        back = s["back"].double()
        for i in range(s["n_seq"]):
            for value in (0, 1):
                back[start[i]:start[i + 1], value * kv * hd:(value + 1) * kv * hd] = _held(s, i, value)[length[i] - (start[i + 1] - start[i]):].flatten(1)
        return back
    out = s["out"].double()
    if s["op"] == "append":
        back = s["back"].double()
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
            back[a:b, :kv * hd] = _stands_for(done[1]).reshape(b - a, -1)
            back[a:b, kv * hd:] = _stands_for(s["v"][a:b].double().reshape(b - a, kv, hd)).reshape(b - a, -1)
        return out, back
    for i in range(s["n_seq"]):
        a, b, e = start[i], start[i + 1], length[i]
        if a == b:
            continue
        there = (s["table"][i, torch.arange(e, device="cuda") // s["page"]] >= 0)
        k, v = _held(s, i, 0), _held(s, i, 1)
        here = torch.arange(e, device="cuda")
        for h in range(heads):
            g = h // (heads // kv)
            for r in range(a, b, 1024):  # rows of the panel at a time
                n = min(b, r + 1024) - r
                at = torch.arange(e - (b - r), e - (b - r) + n, device="cuda")[:, None]
                hidden = (here > at) | ~there
                if s["window"]:
                    hidden = hidden | ((here <= at - s["window"]) & (here >= s["first"]))
                p = torch.softmax((s["q"][r:r + n, h * hd:(h + 1) * hd].double() @ k[:, g].T / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1)
                out[r:r + n, h * hd:(h + 1) * hd] = torch.nan_to_num(p, nan=0.0) @ v[:, g]
    return out
