"""GPU tests of the paged cache: append with norm and rotation, attention of a step's rows over the pages, rotation with several axes, and a run of them together.
Results are compared with the definitions in 64 bits."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import koifish_b200 as kf

pytestmark = pytest.mark.gpu
HALF16 = 2.0 ** -8  # half a step of bf16, relative


@pytest.fixture(scope="module")
def ctx():
    c = kf.Context(0, stream=torch.cuda.current_stream().cuda_stream or 1)
    yield c
    c.close()


class At:
    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


class Step:
    """A step of sequences with `new` tokens and `length` positions over pages in random order.  What belongs to no sequence is not a number: rows of pages that
    nobody has, rows behind a sequence's last position, and padding rows of the panel."""

    def __init__(self, new, length, heads, kv, hd, page, seed=0, beside=False, pad=0, drop=None, cols=0, extra=0):
        g = gen(seed)
        self.new, self.length, self.heads, self.kv, self.hd, self.page = list(new), list(length), heads, kv, hd, page
        held = [-(-n // page) for n in length]
        self.n_pages = sum(held) + 3
        self.cols = max(cols, max(held) + 1)
        order = torch.randperm(self.n_pages, generator=g, device="cuda").cpu().numpy()
        table, at = np.full((len(held), self.cols), 2 ** 31 - 1, dtype=np.int64), 0  # behind the last page: must not be followed
        for i, n in enumerate(held):
            table[i, :n] = order[at:at + n]
            at += n
        for i, j, e in drop or []:
            table[i, j] = e
        self.table = table
        self.rows = sum(new) + pad + extra
        start = np.concatenate([[0], np.cumsum(new)]) + extra
        stride = page * kv * hd
        if beside:
            pool = torch.full((self.n_pages, 2, page, kv, hd), float("nan"), device="cuda", dtype=torch.bfloat16)
            self.k, self.v, stride = pool[:, 0], pool[:, 1], 2 * stride
        else:
            self.k, self.v = (torch.full((self.n_pages, page, kv, hd), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in "kv")
        for i, n in enumerate(length):
            for j in range(held[i]):
                e, m = int(table[i, j]), min(page, n - j * page)
                if 0 <= e < self.n_pages:
                    self.k[e, :m] = (torch.randn(m, kv, hd, generator=g, device="cuda") * 1.3).bfloat16()
                    self.v[e, :m] = (torch.randn(m, kv, hd, generator=g, device="cuda") * 0.7 + 0.2).bfloat16()
        self.start = start.tolist()
        self.q = torch.full((self.rows, heads * hd), float("nan"), device="cuda", dtype=torch.bfloat16)
        a, b = self.start[0], self.start[-1]
        self.q[a:b] = (torch.randn(b - a, heads * hd, generator=g, device="cuda") * 1.3).bfloat16()
        self.d = [i32(np.where(table > 2 ** 31 - 1, 0, table)), i32(start), i32(length)]
        self.desc = kf.PagedKV(At(self.k), At(self.v), self.n_pages, page, kv, hd, At(self.d[0]), self.cols, len(held), At(self.d[1]), At(self.d[2]), page_stride=stride)

    def flat(self, i, pool):
        """rows of sequence i in 64 bits, and which of them are there"""
        n = self.length[i]
        pages = self.table[i, :-(-n // self.page)]
        ok = torch.tensor([0 <= int(e) < self.n_pages for e in pages for _ in range(self.page)], device="cuda", dtype=torch.bool)[:n]
        idx = torch.tensor([int(e) if 0 <= int(e) < self.n_pages else 0 for e in pages], device="cuda", dtype=torch.long)
        return pool[idx].reshape(-1, self.kv, self.hd)[:n].double(), ok

    def expect(self, scale, window, q=None):
        """(result, bound) of attention.  The bound counts: the result's rounding, at most half a step of it; the rounding of a weight to bf16, (1 + e) with |e| <= half a step
        -- where the sum of the weights is not rounded with them it changes the result by at most that much of the weighted mean of |v|, where it is, by sum w e (v - r), at most
        that much of mean |v| + |r|; fp32 errors of a score, hd + 2 roundings of sums whose terms add up to |q|.|k|, which change a weight by as much, and 2^-20 for
        exponentials and sums; each of them in numerator and denominator."""
        q = self.q if q is None else q
        out = torch.full((self.rows, self.heads * self.hd), float("nan"), device="cuda", dtype=torch.float64)
        tol = torch.zeros_like(out)
        group = self.heads // self.kv
        for i, n in enumerate(self.new):
            if n == 0:
                continue
            a, e, hd = self.start[i], self.length[i], self.hd
            k, ok = self.flat(i, self.k)
            v, _ = self.flat(i, self.v)
            p = torch.arange(e - n, e, device="cuda")[:, None]
            j = torch.arange(e, device="cuda")[None]
            sees = (j <= p) & ok[None]
            if window > 0:
                sees = sees & (j > p - window)
            v = torch.where(sees.any(0)[:, None, None], v, torch.zeros_like(v)) if e else v
            for h in range(self.heads):
                qh = q[a:a + n, h * hd:(h + 1) * hd].double()
                kh, vh = k[:, h // group], v[:, h // group]
                s = torch.where(sees, scale * (qh @ torch.where(sees.any(0)[:, None], kh, torch.zeros_like(kh)).T), torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
                size = scale * (qh.abs() @ torch.where(sees.any(0)[:, None], kh, torch.zeros_like(kh)).abs().T)
                top = s.amax(1, keepdim=True) if e else torch.full((n, 1), -math.inf, dtype=torch.float64, device="cuda")
                w = torch.where(sees, torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top)), torch.zeros_like(s))
                tot = w.sum(1, keepdim=True)
                w = w / torch.where(tot == 0, torch.ones_like(tot), tot)
                r = w @ vh
                mean = w @ vh.abs()
                delta = (hd + 2) * 2.0 ** -24 * (torch.where(sees, size, torch.zeros_like(size)).amax(1, keepdim=True) if e else 0) + 2.0 ** -20
                out[a:a + n, h * hd:(h + 1) * hd] = r
                tol[a:a + n, h * hd:(h + 1) * hd] = 1.01 * (2 * HALF16 * r.abs() + (HALF16 + 2 * delta) * mean) + 1e-30
        return out, tol

    def attend(self, ctx, scale, window=0, max_q=None, q=None, ldq=0, ldo=0, out=None):
        out = torch.full((self.rows, ldo or self.heads * self.hd), 7.0, device="cuda", dtype=torch.bfloat16) if out is None else out
        kf.paged_attention(ctx, self.desc, At(self.q if q is None else q), self.rows, self.heads, max_q=max(self.new) if max_q is None else max_q, scale=scale, window=window,
                           ldq=ldq, ldo=ldo, out=At(out))
        return out

    def check(self, ctx, window=0, scale=None, **kw):
        scale = self.hd ** -0.5 if scale is None else scale
        out = self.attend(ctx, scale, window, **kw)
        ctx.sync()
        ref, tol = self.expect(scale, window)
        a, b = self.start[0], self.start[-1]
        got = out[:, :self.heads * self.hd].double()
        assert torch.all(out[:a] == 7) and torch.all(out[b:] == 7) and torch.all(out[:, self.heads * self.hd:] == 7), "padding was written"
        bad = ~((got[a:b] - ref[a:b]).abs() <= tol[a:b])
        assert not bad.any(), "%d of %d off, worst %g" % (int(bad.sum()), bad.numel(), float(((got[a:b] - ref[a:b]).abs() / tol[a:b]).nan_to_num(1e9).max()))
        return out


# ---------------------------------------------------------------------------------------------------------------- attention, single tokens and few rows
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group,kv", [(1, 1), (4, 2), (5, 3), (8, 8), (16, 1)])
@pytest.mark.parametrize("page", [8, 24, 64, 160])
def test_single_tokens(ctx, hd, group, kv, page):
    """One token each: lengths of one, on and around page and tile ends, a sequence without new tokens, one without any position."""
    length = [1, 2, page - 1, page, page + 1, 63, 64, 65, 0, 129, 700, 1000]
    new = [1] * 12
    new[8], new[10] = 0, 0
    Step(new, length, group * kv, kv, hd, page, seed=page + hd, beside=page == 24, pad=3).check(ctx)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_seq,length", [(1, 5000), (1, 40000), (3, 9001), (40, 300), (300, 37)])
def test_single_tokens_runs(ctx, hd, n_seq, length):
    """Runs that end inside sequences, sequences over many runs, many sequences in a run, more than 32 of them."""
    r = np.random.RandomState(n_seq)
    lens = [length] if n_seq == 1 else r.randint(1, length, n_seq).tolist()
    Step([1] * n_seq, lens, 8, 2, hd, 16, seed=n_seq).check(ctx)


@pytest.mark.parametrize("window", [1, 7, 64, 100, 2 ** 31 - 1])
def test_single_tokens_window(ctx, window):
    """The first visible position inside a tile, inside a box, and at their ends; pages wholly behind the window given back, with entries of every kind."""
    length = [1, 64, 65, 128, 200, 333, 1024]
    drop = [(i, j, [-1, -7, 10 ** 6, 2 ** 31 - 1][j % 4]) for i, n in enumerate(length) for j in range(-(-n // 16)) if (j + 1) * 16 <= n - window]
    Step([1] * 7, length, 8, 2, 128, 16, seed=window % 1000, drop=drop).check(ctx, window=window)


def test_single_tokens_missing_pages(ctx):
    """Pages that are not there inside what a row would see, all of them in one sequence (zeros), the last one in another."""
    s = Step([1, 1, 1, 1], [100, 48, 300, 17], 8, 2, 64, 16, seed=5, drop=[(0, 2, -1), (0, 3, 99999), (1, 0, -1), (1, 1, -1), (1, 2, -1), (2, 18, -1), (3, 0, -5)])
    out = s.check(ctx)
    assert torch.all(out[1] == 0)


def test_single_tokens_scales(ctx):
    """Weights on one position, and on all alike."""
    for scale in (8.0, 1e-6):
        Step([1, 1], [500, 77], 8, 2, 128, 16, seed=3).check(ctx, scale=scale)


def test_rows_and_strides(ctx):
    """Queries inside wider rows, results in wider rows and at any element, rows in front of the first sequence, pages of more entries than the table says."""
    s = Step([1, 1, 1], [70, 5, 640], 8, 2, 128, 32, seed=8, extra=2, pad=1, cols=40)
    wide = torch.zeros(s.rows, 8 * 128 + 64, device="cuda", dtype=torch.bfloat16)
    wide[:, 64:] = s.q
    buf = torch.full((s.rows * (8 * 128 + 5) + 1,), 7.0, device="cuda", dtype=torch.bfloat16)
    out = buf[1:].view(s.rows, 8 * 128 + 5)
    s.check(ctx, q=wide[:, 64:], ldq=8 * 128 + 64, ldo=8 * 128 + 5, out=out)
    assert buf[0] == 7


def test_hidden_values(ctx):
    """Infinities and NaN in keys and values that no row sees -- behind the last position, and before the window inside its first box."""
    s = Step([1, 1], [90, 61], 8, 2, 128, 64, seed=9)
    for e, n in ((int(s.table[0, 0]), 90 - 50), (int(s.table[1, 0]), 61 - 50)):
        s.k[e, :n], s.v[e, :n] = float("inf"), float("nan")
    s.check(ctx, window=50)


def test_scores_of_minus_infinity(ctx):
    """Keys whose scores are -inf weigh nothing, wherever they stand; a row with no others gets zeros."""
    s = Step([1, 1], [200, 30], 4, 1, 64, 16, seed=10)
    s.q[:] = s.q.abs()
    for j in (0, 3, 12):
        s.k[int(s.table[0, j])] = float("-inf")
    for j in (0, 1):
        s.k[int(s.table[1, j])] = float("-inf")
    out = s.attend(ctx, 64 ** -0.5)
    ctx.sync()
    t = Step([1, 1], [200, 30], 4, 1, 64, 16, seed=10, drop=[(0, 0, -1), (0, 3, -1), (0, 12, -1), (1, 0, -1), (1, 1, -1)])
    t.k, t.v, t.q, t.table = s.k, s.v, s.q, np.where(t.table == -1, -1, s.table)
    ref, tol = t.expect(64 ** -0.5, 0)
    assert torch.all((out.double() - ref).abs() <= tol) and torch.all(out[1] == 0)


# ---------------------------------------------------------------------------------------------------------------- several tokens a sequence
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group,kv", [(1, 2), (4, 2), (5, 1), (7, 2), (8, 1), (64, 1)])
@pytest.mark.parametrize("new,past", [([2, 3, 1], [0, 62, 300]), ([5, 17, 0, 64], [1000, 3, 9, 0]), ([130, 1, 257], [0, 40, 511])])
def test_chunks(ctx, hd, group, kv, new, past):
    """Chunks on and around block and tile ends beside single tokens and an idle sequence."""
    Step(new, [a + b for a, b in zip(new, past)], group * kv, kv, hd, 16, seed=sum(new) + group, pad=2).check(ctx)


@pytest.mark.parametrize("max_q", [0, 1, 3, 100000])
def test_hint(ctx, max_q):
    """max_q is a hint: results hold whatever it says."""
    Step([1, 40, 3, 0, 200], [9, 50, 400, 5, 1000], 8, 2, 128, 16, seed=21).check(ctx, max_q=max_q)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [1, 33, 128, 500])
def test_chunks_window(ctx, hd, window):
    new, length = [3, 150, 1, 300, 40], [40, 150, 700, 900, 640]
    drop = [(i, j, -1) for i, n in enumerate(length) for j in range(-(-n // 8)) if (j + 1) * 8 <= n - new[i] + 1 - window]
    Step(new, length, 8, 2, hd, 8, seed=window, drop=drop, beside=True).check(ctx, window=window)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group,kv,window", [(7, 4, 0), (7, 4, 300), (4, 2, 0)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_mixed_runs(ctx, hd, group, kv, window, seed):
    """Steps with several blocks in a run: blocks of one row tile and of two, of one tile of positions and of many, in every order."""
    r = np.random.RandomState(seed)
    new = [1, 1, 1, 90, 1, 0, 30, 1, 40, 1] + [int(r.choice([1, 1, 2, 20, 75])) for _ in range(50)]
    length = [n + int(r.choice([0, 60, 200, r.randint(0, 900)])) for n in new]
    Step(new, length, group * kv, kv, hd, 16, seed=seed).check(ctx, window=window)


def test_chunks_before_the_first_position(ctx):
    """More new tokens than positions: the first rows stand before position 0 and see nothing."""
    s = Step([20, 40], [8, 33], 4, 1, 128, 8, seed=4)
    out = s.attend(ctx, 0.1)
    ctx.sync()
    assert torch.all(out[:12] == 0) and torch.all(out[20:27] == 0)
    t = Step([8, 33], [8, 33], 4, 1, 128, 8, seed=4)
    t.k, t.v, t.table = s.k, s.v, s.table
    ref, tol = t.expect(0.1, 0, q=torch.cat([s.q[12:20], s.q[27:60]]))
    got = torch.cat([out[12:20], out[27:60]]).double()
    assert torch.all((got - ref).abs() <= tol)


def test_chunks_missing_pages(ctx):
    s = Step([100, 9], [400, 9], 8, 2, 128, 24, seed=6, drop=[(0, 0, -1), (0, 7, -2), (0, 14, 5000), (1, 0, -1)])
    out = s.check(ctx)
    assert torch.all(out[100:109] == 0)


def test_beyond_the_table(ctx):
    """A length above what the table holds: the positions behind it are not there, those in front are seen."""
    s = Step([4, 1], [100, 64], 4, 2, 128, 16, seed=14)
    s.desc = kf.PagedKV(At(s.k), At(s.v), s.n_pages, 16, 2, 128, At(i32(s.table[:, :6])), 6, 2, At(s.d[1]), At(s.d[2]))
    s.table = s.table.copy()
    s.table[0, 6] = -1  # position 96 .. 99
    s.check(ctx)


def test_far_pages(ctx):
    """A pool of more than 2^32 elements with its pages far apart."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 20 GB")
    kv, hd, page, n_pages = 8, 128, 16, 40
    stride = (1 << 27) + 8  # elements; 40 pages: 5.4e9
    pool = torch.empty(n_pages * stride, device="cuda", dtype=torch.bfloat16)
    s = Step([1, 30], [300, 200], 32, kv, hd, page, seed=15)
    assert s.n_pages <= n_pages
    for name, off in (("k", 0), ("v", page * kv * hd)):
        far = pool[off:off + (s.n_pages - 1) * stride + page * kv * hd].as_strided((s.n_pages, page, kv, hd), (stride, kv * hd, hd, 1))
        far.copy_(getattr(s, name))
        setattr(s, name, far)
    s.desc = kf.PagedKV(At(s.k), At(s.v), s.n_pages, page, kv, hd, At(s.d[0]), s.cols, 2, At(s.d[1]), At(s.d[2]), page_stride=stride)
    s.check(ctx)


# ---------------------------------------------------------------------------------------------------------------- append and rotation
def turned(x, freq, axis, pos, layout, amp):
    """x [rows, heads, hd] in 64 bits"""
    n = freq.numel()
    t = torch.stack([pos[int(axis[j])].double() * freq[j] if 0 <= int(axis[j]) < len(pos) else torch.full((x.shape[0],), float("nan"), device="cuda", dtype=torch.float64)
                     for j in range(n)], 1)[:, None] if n else torch.zeros(x.shape[0], 1, 0, device="cuda", dtype=torch.float64)
    still = torch.isnan(t)
    c, s = torch.where(still, torch.ones_like(t), amp * torch.cos(t)), torch.where(still, torch.zeros_like(t), amp * torch.sin(t))
    a, b = (slice(0, n), slice(n, 2 * n)) if layout else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    y, size = x.clone(), x.abs()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def normed(x, w, eps):
    return x if w is None else x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()


# fp32 errors of a rotation, relative to |a| + |b|: the reduced angle / pi rounded to 24 bits (2^-25 pi), sine and cosine off by two units (2^-23), the factor, and
# two products and their sum (4 x 2^-24) -- together under 2^-21; with a norm 2^-20 more for the sum of squares, the root and two products
TURN, NORM = 2.0 ** -21, 2.0 ** -20


def append_and_check(ctx, src, hd, heads, kv, rot, layout, axes, norm, off, new, length):
    g = gen(hd + rot + axes)
    s = Step(new, length, heads, kv, hd, 24, seed=1, extra=1, pad=2, beside=off == 1)
    wide = (heads + 2 * kv) * hd + 8 + off
    panel = torch.randn(s.rows, wide, generator=g, device="cuda").to(src)
    q, k, v = (panel[:, off + a * hd:off + b * hd] for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    freq = 1e4 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) / max(1, rot // 2))
    axis = torch.arange(rot // 2, device="cuda", dtype=torch.int32) % axes
    if axes == 3 and rot:
        axis[rot // 4] = 5 - 8 * (rot // 4 % 2)  # an axis that does not exist: the pair does not turn
    pos = torch.randint(-3, 200000, (axes, s.rows + 3), generator=g, device="cuda", dtype=torch.int32) if axes > 1 else None
    wq, wk = ((1 + 0.3 * torch.randn(hd, generator=g, device="cuda")).bfloat16() for _ in "qk") if norm else (None, None)
    amp = 1.25 if axes == 2 else 1.0
    r = kf.Rotation(At(freq), rot, layout=layout, amp=amp, n_axes=axes, pair_axis=At(axis) if axes > 1 else None, pos=At(pos) if axes > 1 else None, pos_stride=s.rows + 3 if axes > 1 else 0)
    out = torch.full((s.rows, heads * hd + off), 7.0, device="cuda", dtype=torch.bfloat16)
    k0, v0 = s.k.clone(), s.v.clone()
    kf.paged_append(ctx, s.desc, r, At(q), At(k), At(v), s.rows, heads, q_norm=At(wq) if norm else None, k_norm=At(wk) if norm else None, eps=1e-5, ldq=wide, ldk=wide, ldv=wide,
                    out=At(out), ldo=heads * hd + off, src_f32=src == torch.float32)
    torch.cuda.synchronize()
    a, b = s.start[0], s.start[-1]
    assert torch.all(out[:a] == 7) and torch.all(out[b:] == 7) and torch.all(out[:, heads * hd:] == 7)
    for i, n in enumerate(new):
        lo, hi = s.start[i], s.start[i + 1]
        place = torch.arange(length[i] - n, length[i], device="cuda")
        p = [place] if pos is None else [pos[x, lo:hi] for x in range(axes)]
        for x, w, h, kind in ((q, wq, heads, "q"), (k, wk, kv, "k")):
            y, size = turned(normed(x[lo:hi].double().reshape(n, h, hd), w, 1e-5), freq, axis if axes > 1 else axis * 0, p, layout, amp)
            got = out[lo:hi, :heads * hd].reshape(n, h, hd) if kind == "q" else torch.stack([s.k[int(s.table[i, int(t) // 24]), int(t) % 24] for t in place]) if n else None
            if n:
                tol = 1.01 * (HALF16 * y.abs() + (TURN + NORM) * amp * size) + 1e-30
                assert torch.all((got.double() - y).abs() <= tol), (kind, i, float(((got.double() - y).abs() / tol).max()))
        for j, t in enumerate(place.tolist()):
            e, m = int(s.table[i, t // 24]), t % 24
            assert torch.equal(s.v[e, m], v[lo + j].reshape(kv, hd).bfloat16())
            k0[e, m], v0[e, m] = s.k[e, m], s.v[e, m]
    assert torch.equal(k0.contiguous().view(torch.int16), s.k.contiguous().view(torch.int16)) and torch.equal(v0.contiguous().view(torch.int16), s.v.contiguous().view(torch.int16))


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,heads,kv,rot,layout,axes,norm", [
    (128, 8, 2, 128, 1, 1, True), (128, 5, 5, 64, 1, 3, False), (128, 32, 8, 128, 0, 3, True), (64, 7, 1, 64, 1, 1, True), (64, 4, 2, 6, 0, 2, False),
    (128, 3, 1, 40, 1, 2, True), (64, 16, 4, 0, 1, 1, True)])
@pytest.mark.parametrize("off", [0, 1])
def test_append(ctx, src, hd, heads, kv, rot, layout, axes, norm, off):
    """Every layout and type, rows at 16 bytes and at any element (off), tokens on page ends, a sequence without new tokens, padding on both sides; every row of the pools
    that belongs to no new token stays as it was."""
    append_and_check(ctx, src, hd, heads, kv, rot, layout, axes, norm, off, [1, 40, 0, 7, 1], [1, 100, 30, 24, 300])


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,heads,kv,rot,layout,axes,norm", [(128, 3, 1, 128, 1, 3, True), (64, 20, 5, 32, 0, 1, False), (128, 65, 8, 128, 0, 1, True), (64, 2, 2, 64, 1, 2, False)])
@pytest.mark.parametrize("off", [0, 1])
def test_append_panels(ctx, src, hd, heads, kv, rot, layout, axes, norm, off):
    """Panels of so many tokens that a block takes four: sequences that end inside one, padding on both sides, heads that take one turn of a block and several."""
    append_and_check(ctx, src, hd, heads, kv, rot, layout, axes, norm, off, [1501, 1, 0, 1202, 3, 1], [1501, 700, 5, 1300, 24, 1])


def test_append_many_sequences(ctx):
    """Finding a token's sequence among up to 8192, most of them without new tokens."""
    r = np.random.RandomState(0)
    for n_seq in (33, 1025, 8192):
        new = (r.rand(n_seq) < 0.02).astype(int) * r.randint(1, 4, n_seq)
        new[-1], new[0] = 2, 1
        length = new + r.randint(0, 9, n_seq)
        s = Step(new, length, 1, 1, 64, 8, seed=n_seq)
        k = torch.randn(s.rows, 64, device="cuda").bfloat16()
        kf.paged_append(ctx, s.desc, None, At(s.q), At(k), At(k), s.rows, 1, out=At(s.q))
        torch.cuda.synchronize()
        for i in np.nonzero(new)[0]:
            for j in range(new[i]):
                t = int(length[i] - new[i] + j)
                assert torch.equal(s.k[int(s.table[i, t // 8]), t % 8, 0], k[s.start[i] + j])


def test_append_missing_pages(ctx):
    """Nothing is written for a token whose page is not there or that lies outside the table; its query is finished all the same."""
    s = Step([6, 3, 2], [30, 3, 2], 2, 1, 64, 8, seed=2, drop=[(0, 3, -1), (1, 0, 10 ** 8)])
    s.d[2][2] = 8 * s.cols + 1  # the last sequence's second token is behind the table
    before = s.k.clone(), s.v.clone()
    k = torch.randn(s.rows, 64, device="cuda").bfloat16()
    out = torch.zeros_like(s.q)
    kf.paged_append(ctx, s.desc, None, At(s.q), At(k), At(k), s.rows, 2, out=At(out))
    torch.cuda.synchronize()
    assert torch.equal(out, s.q)
    e = int(s.table[0, 3])
    same = [torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(before, (s.k, s.v))]
    assert e == -1 and all(same)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,heads,hd,rot,layout,axes", [(1, 1, 2, 2, 0, 1), (259, 16, 64, 64, 0, 2), (5, 3, 80, 80, 1, 3), (70, 2, 72, 36, 1, 2), (33, 4, 256, 256, 1, 3), (1000, 8, 128, 96, 1, 1),
                                                        (3, 200, 32, 32, 0, 2), (2, 5, 7, 4, 1, 1),
                                                        (2371, 3, 128, 128, 1, 3), (2500, 1, 64, 48, 0, 2), (4001, 35, 96, 96, 1, 2), (2369, 2, 72, 36, 1, 1)])
@pytest.mark.parametrize("inplace", [False, True])
def test_rope_axes(ctx, t, M, heads, hd, rot, layout, axes, inplace):
    g = gen(M + hd)
    x = torch.randn(M, heads * hd + 24, generator=g, device="cuda").to(t)
    freq = 1e6 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) / (rot // 2))
    axis = (torch.arange(rot // 2, device="cuda") * axes // (rot // 2)).int()
    pos = torch.randint(-100, 10 ** 7, (axes, M), generator=g, device="cuda", dtype=torch.int32)
    r = kf.Rotation(At(freq), rot, layout=layout, n_axes=axes, pair_axis=At(axis), pos=At(pos))
    want, size = turned(x[:, :heads * hd].double().reshape(M, heads, hd), freq, axis, list(pos), layout, 1.0)
    rest = x[:, heads * hd:].clone()
    if inplace:
        dev = At(x)
        kf.rope_axes(ctx, r, dev, M, heads, hd, ldx=x.stride(0), out=dev, f32=t == torch.float32)
        got = x[:, :heads * hd]
    else:
        out = torch.full((M + 1, heads * hd), 7.0, device="cuda", dtype=t)
        kf.rope_axes(ctx, r, At(x), M, heads, hd, ldx=x.stride(0), out=At(out), f32=t == torch.float32)
        got = out[:M]
        assert torch.all(out[M] == 7)
    torch.cuda.synchronize()
    assert torch.equal(rest, x[:, heads * hd:])
    half = HALF16 if t == torch.bfloat16 else 2.0 ** -24
    tol = 1.01 * (half * want.abs() + TURN * size) + 1e-30
    err = (got.double().reshape(M, heads, hd) - want).abs()
    assert torch.all(err <= tol), float((err / tol).max())


# ---------------------------------------------------------------------------------------------------------------- together
def serve(ctx, heads, kv, hd, page, chunks, seed=0, graph=False):
    """Sequences fed in steps of `chunks` (a list of steps, each a list of new tokens per sequence): append and attention, against attention over everything in 64 bits with the
    keys as the cache should hold them."""
    g = gen(seed)
    n_seq, total = len(chunks[0]), np.sum(chunks, 0)
    held = [-(-int(n) // page) for n in total]
    n_pages = sum(held) + 2
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.full((n_seq, max(held)), -1, device="cuda", dtype=torch.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    kp, vp = (torch.full((n_pages, page, kv, hd), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in "kv")
    freq = 1e4 ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) / (hd // 2))
    wq, wk = ((1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).bfloat16() for _ in "qk")
    wide = (heads + 2 * kv) * hd
    most = max(int(np.sum(c)) for c in chunks)
    panel, qbuf, out = (torch.zeros(most, w, device="cuda", dtype=torch.bfloat16) for w in (wide, heads * hd, heads * hd))
    start, lens = i32([0] * (n_seq + 1)), i32([0] * n_seq)
    desc = kf.PagedKV(At(kp), At(vp), n_pages, page, kv, hd, At(table), max(held), n_seq, At(start), At(lens))
    rot = kf.Rotation(At(freq), hd)

    def step():
        kf.paged_append(ctx, desc, rot, At(panel), At(panel[:, heads * hd:]), At(panel[:, (heads + kv) * hd:]), most, heads, At(wq), At(wk), ldq=wide, ldk=wide, ldv=wide, out=At(qbuf))
        kf.paged_attention(ctx, desc, At(qbuf), most, heads, max_q=max(max(c) for c in chunks), out=At(out))

    h = None
    if graph:
        step()
        h = C.c_void_p()
        ctx.check(ctx.lib.kf_graph_begin(ctx.h), "begin")
        step()
        ctx.check(ctx.lib.kf_graph_end(ctx.h, C.byref(h)), "end")
    past = np.zeros(n_seq, dtype=int)
    keys, vals = [[] for _ in range(n_seq)], [[] for _ in range(n_seq)]
    for c in chunks:
        n = int(np.sum(c))
        panel[:n] = torch.randn(n, wide, generator=g, device="cuda").bfloat16()
        start.copy_(i32(np.concatenate([[0], np.cumsum(c)])))
        lens.copy_(i32(past + c))
        out.fill_(7.0)
        torch.cuda.synchronize()
        if graph:
            ctx.check(ctx.lib.kf_graph_launch(ctx.h, h), "launch")
            ctx.sync()
        else:
            step()
            ctx.sync()
        assert torch.all(out[n:] == 7)
        row = 0
        for i in range(n_seq):
            m = int(c[i])
            if m == 0:
                continue
            x = panel[row:row + m].double()
            place = torch.arange(int(past[i]), int(past[i]) + m, device="cuda")
            q, _ = turned(normed(x[:, :heads * hd].reshape(m, heads, hd), wq, 1e-6), freq, torch.zeros(hd // 2, dtype=torch.int32), [place], 1, 1.0)
            k, _ = turned(normed(x[:, heads * hd:(heads + kv) * hd].reshape(m, kv, hd), wk, 1e-6), freq, torch.zeros(hd // 2, dtype=torch.int32), [place], 1, 1.0)
            keys[i].append(k), vals[i].append(x[:, (heads + kv) * hd:].reshape(m, kv, hd))
            kk, vv = torch.cat(keys[i]), torch.cat(vals[i])
            sees = torch.arange(len(kk), device="cuda")[None] <= place[:, None]
            for hh in range(heads):
                # the bound beside that of attention: q and k are rounded to bf16, which changes a score by at most half a step of each, |q|.|k| in size
                s = (q[:, hh] @ kk[:, hh // (heads // kv)].T) * hd ** -0.5
                size = (q[:, hh].abs() @ kk[:, hh // (heads // kv)].abs().T) * hd ** -0.5
                w = torch.softmax(s.masked_fill(~sees, -math.inf), 1)
                v = vv[:, hh // (heads // kv)]
                r, mean = w @ v, w @ v.abs()
                delta = torch.expm1((2.02 * HALF16 + (hd + 2) * 2.0 ** -24) * torch.where(sees, size, torch.zeros_like(size)).amax(1, keepdim=True)) + 2.0 ** -19
                err = (out[row:row + m, hh * hd:(hh + 1) * hd].double() - r).abs()
                assert torch.all(err <= 1.01 * (HALF16 * r.abs() + (HALF16 + 2 * delta) * mean)), (c, i, hh)
                # ... which is loose: the errors of many scores are independent, so the whole is far nearer
                assert float(err.norm() / r.norm()) < 0.02
            row += m
        past = past + np.asarray(c)
    if h:
        ctx.check(ctx.lib.kf_graph_destroy(h), "destroy")


@pytest.mark.parametrize("heads,kv,hd,page", [(8, 2, 128, 16), (4, 4, 64, 24)])
def test_serving(ctx, heads, kv, hd, page):
    """A prompt in chunks beside decoding sequences, drafts, idle slots."""
    serve(ctx, heads, kv, hd, page, [[70, 1, 5], [130, 1, 0], [1, 1, 300], [1, 0, 1], [4, 5, 3], [1, 1, 1]])


def test_serving_captured():
    """One captured step replayed over changing mixtures and lengths."""
    c = kf.Context(0)
    serve(c, 8, 2, 128, 16, [[9, 1, 40], [1, 1, 1], [0, 30, 2], [1, 1, 1], [20, 0, 17]], graph=True)
    c.close()


def test_two_captured_steps():
    """Two captured steps of one context, which share its workspace, replayed in turn and twice each; a context without a workspace refuses the capture and works afterwards."""
    c = kf.Context(0)
    a, b = Step([1, 1], [3000, 800], 8, 2, 128, 16, seed=60), Step([90, 1, 7], [700, 2000, 300], 8, 2, 64, 16, seed=61)
    outs = [torch.full((s.rows, s.heads * s.hd), 7.0, device="cuda", dtype=torch.bfloat16) for s in (a, b)]
    torch.cuda.synchronize()
    ctx_call = lambda s, o: kf.paged_attention(c, s.desc, At(s.q), s.rows, s.heads, max_q=max(s.new), scale=0.1, out=At(o))  # noqa: E731
    h = C.c_void_p()
    c.check(c.lib.kf_graph_begin(c.h), "begin")
    with pytest.raises(kf.KoifishError, match="before graph capture"):
        ctx_call(a, outs[0])
    c.check(c.lib.kf_graph_end(c.h, C.byref(h)), "end")
    c.check(c.lib.kf_graph_destroy(h), "destroy")
    for s, o in zip((b, a), reversed(outs)):
        ctx_call(s, o)
    graphs = []
    for s, o in zip((a, b), outs):
        h = C.c_void_p()
        c.check(c.lib.kf_graph_begin(c.h), "begin")
        ctx_call(s, o)
        c.check(c.lib.kf_graph_end(c.h, C.byref(h)), "end")
        graphs.append(h)
    c.sync()
    for o in outs:
        o.fill_(7.0)
    torch.cuda.synchronize()
    for h in graphs * 2 + graphs[::-1]:
        c.check(c.lib.kf_graph_launch(c.h, h), "launch")
    c.sync()
    for s, o in zip((a, b), outs):
        ref, tol = s.expect(0.1, 0)
        assert torch.all((o.double() - ref).abs() <= tol)
    for h in graphs:
        c.check(c.lib.kf_graph_destroy(h), "destroy")
    c.close()


def test_same_bits(ctx):
    """Pieces are merged in order: the same call gives the same bits."""
    s = Step([1, 1, 60, 5], [3000, 700, 900, 5000], 8, 2, 128, 16, seed=31)
    a = s.attend(ctx, 0.1)
    for _ in range(5):
        b = s.attend(ctx, 0.1)
        ctx.sync()
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("group,kv", [(5, 8), (7, 4), (12, 3), (17, 3)])
@pytest.mark.parametrize("hd", [64, 128])
def test_same_bits_whatever_ran_before(ctx, group, kv, hd):
    """Rows of a row tile that are nobody's hold what the call before left in shared memory, here queries fifty times as large: no result depends on them."""
    s = Step([138, 1, 77], [2231, 900, 1500], group * kv, kv, hd, 16, seed=group)
    other = Step([130] * 20, [400] * 20, 64, 1, hd, 16, seed=3)
    loud = other.q * 50
    a = s.attend(ctx, hd ** -0.5)
    for _ in range(6):
        other.attend(ctx, hd ** -0.5, q=loud)
        b = s.attend(ctx, hd ** -0.5)
        ctx.sync()
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_against_the_contiguous_cache(ctx):
    """One page per sequence is a contiguous cache: the same step through kf_attn_decode_gqa.  Both are within their bound of the 64-bit result, so within twice of each other."""
    s = Step([1] * 4, [512, 100, 33, 400], 16, 4, 128, 512, seed=40)
    ref, tol = s.expect(128 ** -0.5, 0)
    order = [int(s.table[i, 0]) for i in range(4)]
    k, v = s.k[order].contiguous(), s.v[order].contiguous()
    out = torch.zeros(4, 16 * 128, device="cuda", dtype=torch.bfloat16)
    pos = i32([n - 1 for n in s.length])
    ctx.check(ctx.lib.kf_attn_decode_gqa(ctx.h, out.data_ptr(), s.q.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), 4, 16, 4, 128, 512, 511, 512 * 4 * 128), "gqa")
    got = s.attend(ctx, 128 ** -0.5)
    ctx.sync()
    assert torch.all((out.double() - got.double()).abs() <= 2 * tol)


# ---------------------------------------------------------------------------------------------------------------- limits
def test_nothing_to_do(ctx):
    """No rows at all, and rows that all are padding."""
    s = Step([1], [5], 2, 1, 64, 8, seed=1)
    out = torch.full((4, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    kf.paged_attention(ctx, s.desc, At(s.q), 0, 2, max_q=1, out=At(out))
    kf.paged_append(ctx, s.desc, None, At(s.q), At(s.q), At(s.q), 0, 2, out=At(out))
    s.d[1][:] = 0
    q = torch.zeros(4, 128, device="cuda", dtype=torch.bfloat16)
    kf.paged_attention(ctx, s.desc, At(q), 4, 2, max_q=1, out=At(out))
    kf.paged_append(ctx, s.desc, None, At(q), At(q), At(q), 4, 2, out=At(out))
    torch.cuda.synchronize()
    assert torch.all(out == 7)


def test_wait_that_runs_out_is_reported():
    """A thread block that loads nothing: the call ends, the next synchronisation says so, and the context works afterwards."""
    for new in ([1, 1], [70, 1]):
        c = kf.Context(0, stream=torch.cuda.current_stream().cuda_stream or 1)
        s = Step(new, [400, 300], 8, 2, 128, 16, seed=50)
        s.check(c)
        c.set_int("attn_wait_us", 20000)
        c.set_int("attn_drop", 1)
        s.attend(c, 0.1)
        with pytest.raises(kf.KoifishError, match="wait ran out"):
            c.sync()
        c.set_int("attn_drop", 0)
        c.set_int("attn_wait_us", 0)
        c.sync()
        s.check(c)
        c.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cta", [0, 70])
@pytest.mark.parametrize("fresh", [False, True])
def test_wait_that_runs_out_among_many_pieces(hd, cta, fresh):
    """A thread block that loads nothing and whose run is longer than the queue of pieces, so that it never comes to the run's end: what the merge reads of it says so, whatever the
    workspace held -- nothing yet, or sums of the other head size over the records.  The error is told, rows of nobody stay as they are, and the next call is right."""
    c = kf.Context(0, stream=torch.cuda.current_stream().cuda_stream or 1)
    r = np.random.RandomState(hd)
    length = r.randint(20, 121, 200).tolist() + [400]
    s = Step([1] * 200 + [256], length, 32, 8, hd, 16, seed=hd, extra=2, pad=3)
    other = Step([130] * 20, [400] * 20, 64, 1, 192 - hd, 16, seed=3)
    # tiles: one for each of the 200 and kv head; the chunk's are fewer than 200 more a head, so a run of the first 70 thread blocks and more is pieces of one tile
    run = -(-8 * 200 // c.lib.kf_ctx_sm_count(c.h))
    assert run >= 6 and (cta + 1) * run < 8 * 200
    if not fresh:
        other.attend(c, 0.1)
        s.check(c)
        other.attend(c, 0.1, q=other.q * 50)
    c.sync()
    out = torch.full((s.rows, 32 * hd), 7.0, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    c.set_int("attn_wait_us", 20000), c.set_int("attn_drop", cta + 1)
    s.attend(c, 0.1, out=out)
    with pytest.raises(kf.KoifishError, match="wait ran out"):
        c.sync()
    c.set_int("attn_drop", 0), c.set_int("attn_wait_us", 0)
    assert torch.all(out[:2] == 7) and torch.all(out[-3:] == 7)
    c.sync()
    s.check(c)
    c.close()


@pytest.mark.parametrize("new", [[1, 1], [70, 1]])
def test_wait_that_runs_out_is_reported_as_this_kernel_s(new):
    """Named in the message and asked for by its own key, not by those of the other attention kernels."""
    c = kf.Context(0, stream=torch.cuda.current_stream().cuda_stream or 1)
    s = Step(new, [400, 300], 8, 2, 128, 16, seed=51)
    keys = ("attn_tc_error", "attn_gqa_error", "attn_paged_error")
    for told_by in ("sync", "call"):
        c.set_int("attn_wait_us", 20000), c.set_int("attn_drop", 1)
        s.attend(c, 0.1)
        c.set_int("attn_drop", 0), c.set_int("attn_wait_us", 0)
        assert [c.get_int(k) for k in keys] == [0, 0, 1]
        with pytest.raises(kf.KoifishError, match="wait ran out in the paged attention kernel"):
            c.sync() if told_by == "sync" else s.attend(c, 0.1)
        assert [c.get_int(k) for k in keys] == [0, 0, 0]
        c.sync()
        s.check(c)
    c.close()


def test_results_over_their_sources(ctx):
    """A result that lies over a part of what it is made of is refused; beside it in the same rows, or where the documentation has it in place, it is taken."""
    s = Step([1, 3, 1], [30, 20, 9], 4, 2, 64, 16, seed=70)
    wide, n = 4 * 64, s.rows
    buf = torch.zeros(n + 4, 3 * wide, device="cuda", dtype=torch.bfloat16)
    buf[1:n + 1, :wide] = s.q
    q, rows = buf[1:n + 1], buf.stride(0)
    bad = [(q, rows), (buf[2:], rows), (buf[0:], rows), (buf[1:n + 1, 8:], rows), (buf.flatten()[rows - wide + 8:], rows), (q, wide)]
    for o, ld in bad:
        with pytest.raises(kf.KoifishError, match="over"):
            s.attend(ctx, 0.1, q=q, ldq=rows, out=o, ldo=ld)
    ref, tol = s.expect(0.1, 0)
    s.attend(ctx, 0.1, q=q, ldq=rows, out=buf[1:n + 1, wide:], ldo=rows)
    torch.cuda.synchronize()
    assert torch.all((buf[1:n + 1, wide:2 * wide].double() - ref).abs() <= tol) and torch.equal(buf[1:n + 1, :wide], s.q)
    r = kf.Rotation(At(torch.ones(32, device="cuda", dtype=torch.float64)), 64, pos=At(i32([0] * n)))
    for o, ld in bad[1:]:
        with pytest.raises(kf.KoifishError, match="over|in place"):
            kf.rope_axes(ctx, r, At(q), n, 4, 64, ldx=rows, out=At(o), ldo=ld)
        with pytest.raises(kf.KoifishError, match="over|in place"):
            kf.paged_append(ctx, s.desc, None, At(q), At(q[:, wide:]), At(q[:, wide + 128:]), n, 4, ldq=rows, ldk=rows, ldv=rows, out=At(o), ldo=ld)
    for o in (q[:, wide:], q[:, wide + 200:]):  # over the keys, over the values
        with pytest.raises(kf.KoifishError, match="over"):
            kf.paged_append(ctx, s.desc, None, At(q), At(q[:, wide:]), At(q[:, wide + 128:]), n, 4, ldq=rows, ldk=rows, ldv=rows, out=At(o), ldo=rows)
    panel = torch.zeros(n, 3 * wide, device="cuda")
    with pytest.raises(kf.KoifishError, match="over"):  # bf16 queries over a float panel's
        kf.paged_append(ctx, s.desc, None, At(panel), At(panel[:, wide:]), At(panel[:, wide + 128:]), n, 4, ldq=3 * wide, ldk=3 * wide, ldv=3 * wide, out=At(panel[:, 8:]), ldo=6 * wide,
                        src_f32=True)
    for o in (q, q[:, 2 * wide:]):
        kf.rope_axes(ctx, r, At(q), n, 4, 64, ldx=rows, out=At(o), ldo=rows)
        kf.paged_append(ctx, s.desc, None, At(q), At(q[:, wide:]), At(q[:, wide + 128:]), n, 4, ldq=rows, ldk=rows, ldv=rows, out=At(o), ldo=rows)
    torch.cuda.synchronize()
    assert torch.equal(q[:, :wide], s.q) and torch.equal(q[:, 2 * wide:], s.q)


def test_timed_calls_on_another_stream():
    """The calls of perf/operators.py go to the stream that is current, for a state of another stream as well, and give the same bits there."""
    import importlib.util
    import os
    spec = importlib.util.spec_from_file_location("timed_operators", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True
    case = [c for c in ops.listed() if c["name"] == "append_decode"][0]
    first, side = ops.prepare(case, 1), torch.cuda.Stream()
    want = [t.clone() for t in ops.run(first)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for s in (first, ops.prepare(case, 1)):
            got = ops.run(s)
            c = s["handles"]["ctx"]
            assert c.lib.kf_ctx_stream(c.h) == side.cuda_stream
            side.synchronize()
            assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(want, got))
    ops.run(first)
    assert first["handles"]["ctx"].lib.kf_ctx_stream(first["handles"]["ctx"].h) == 1
    torch.cuda.synchronize()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_seq,chunk", [(1100, 0), (1100, 90), (2500, 3), (8192, 40)])
def test_attention_of_many_sequences(ctx, hd, n_seq, chunk):
    """More than 1024 sequences, most of them idle or with one token, in both kernels: a run begins behind many that it has no part in."""
    r = np.random.RandomState(n_seq + chunk)
    new = (r.rand(n_seq) < min(1.0, 400 / n_seq)).astype(int)
    length = new + r.randint(0, 30, n_seq)
    new[0], length[0], new[-1], length[-1] = 1, 200, 1, 333
    if chunk:
        for i in (5, n_seq // 2, n_seq - 2):
            new[i], length[i] = chunk, chunk + 100
    Step(new, length, 4, 2, hd, 16, seed=chunk, pad=1).check(ctx)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("window", [5, 70, 300])
def test_chunks_hidden_values(ctx, hd, page, window):
    """Infinities and NaN in keys and values before the first row's window, in pages that are still there, and behind the last position."""
    new, length = [3, 150, 1, 60], [500, 640, 777, 64]
    s = Step(new, length, 8, 2, hd, page, seed=window + page)
    for i, n in enumerate(length):
        for j in range(max(0, n - new[i] + 1 - window)):
            e, m = int(s.table[i, j // page]), j % page
            s.k[e, m], s.v[e, m] = float("inf") if j % 2 else float("nan"), float("nan") if j % 3 else float("-inf")
    s.check(ctx, window=window)
    s.check(ctx, window=window, max_q=2)


def test_append_far_pages(ctx):
    """Rows that lie more than 2^32 elements into the pool."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 20 GB")
    kv, hd, page, n_pages = 2, 64, 16, 40
    stride = (1 << 27) + 8
    pool = torch.zeros(n_pages * stride, device="cuda", dtype=torch.bfloat16)
    s = Step([1, 30], [300, 200], 4, kv, hd, page, seed=16)
    s.table[s.table == s.n_pages - 1], s.table[0, 18] = s.table[0, 18], s.n_pages - 1  # the page that the first sequence's token falls into is the last
    s.d[0].copy_(i32(np.where(s.table > 2 ** 31 - 1, 0, s.table)))
    assert (s.n_pages - 1) * stride > 1 << 32
    far = [pool[off:off + (s.n_pages - 1) * stride + page * kv * hd].as_strided((s.n_pages, page, kv, hd), (stride, kv * hd, hd, 1)) for off in (0, page * kv * hd)]
    desc = kf.PagedKV(At(far[0]), At(far[1]), s.n_pages, page, kv, hd, At(s.d[0]), s.cols, 2, At(s.d[1]), At(s.d[2]), page_stride=stride)
    k, v = (torch.randn(s.rows, kv * hd, device="cuda").bfloat16() for _ in "kv")
    kf.paged_append(ctx, desc, None, At(s.q), At(k), At(v), s.rows, 4, out=At(s.q))
    torch.cuda.synchronize()
    for i, n in enumerate(s.new):
        for j in range(n):
            t = s.length[i] - n + j
            e, m = int(s.table[i, t // page]), t % page
            assert torch.equal(far[0][e, m].flatten(), k[s.start[i] + j]) and torch.equal(far[1][e, m].flatten(), v[s.start[i] + j])
