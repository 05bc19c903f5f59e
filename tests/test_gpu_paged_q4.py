"""GPU tests of the paged cache in 4 bits: quantising append, reading back, attention with a window and first positions, and runs of them together.
Results are compared with the definitions in 64 bits; bytes of the pool are looked up by the documented places, one entry at a time."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import koifish_b200 as kf
from test_gpu_paged import HALF16, NORM, TURN, At, gen, i32, normed, turned

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = kf.Context(0, stream=torch.cuda.current_stream().cuda_stream or 1)
    yield c
    c.close()


def places(kv, hd, page, value):
    """Bytes of a page: codes [page, kv, hd] (the even entries' in the lower half of a byte), steps and zeros [page, kv, groups]."""
    p, h, d, j = (torch.arange(n, device="cuda") for n in (page, kv, hd, hd // 32))
    p, h = p[:, None, None], h[:, None]
    G, unit = hd // 32, 10 * hd
    at, r = (h * (page // 8) + p // 8) * unit, p % 8
    if value:
        at = at + 4 * hd + 32 * G
        code = at + (d % 32 // 4) * (hd // 2) + (r // 2) * (hd // 8) + (r % 2) * (hd // 16) + (d // 64) * 4 + (d // 32 % 2) * 2 + d % 4 // 2
        return code, at + 4 * hd + 2 * (r * G + j), at + 4 * hd + 16 * G + 2 * (j * 8 + r)
    code = at + r * (hd // 2) + (d % 32 // 8) * (4 * G) + (d // 32) * 4 + d % 8 // 2
    return code, at + 4 * hd + 2 * (r * G + j), at + 4 * hd + 16 * G + 2 * (r * G + j)


def write(pages, kv, hd, page, value, e, r, codes, step, zero):
    """codes [n, kv, hd], step and zero [n, kv, groups] of rows r of pages e."""
    at, s, z = (x[r] for x in places(kv, hd, page, value))
    c = codes.to(torch.uint8)
    pages[e[:, None, None], at[..., ::2]] = c[..., ::2] | c[..., 1::2] << 4
    for where, x in ((s, step), (z, zero)):
        b = x.bfloat16().contiguous().view(torch.uint8).unflatten(-1, (-1, 2))
        pages[e[:, None, None], where], pages[e[:, None, None], where + 1] = b[..., 0], b[..., 1]


def read(pages, kv, hd, page, value, e, r):
    """codes, steps and zeros in 64 bits."""
    at, s, z = (x[r] for x in places(kv, hd, page, value))
    e = e[:, None, None]
    b = pages[e, at]
    codes = torch.where(torch.arange(hd, device="cuda") % 2 == 1, b >> 4, b & 15).double()
    f = [((pages[e, w].int() | pages[e, w + 1].int() << 8) << 16).view(torch.float32).double() for w in (s, z)]
    return codes, f[0], f[1]


def wide(x):
    return x.repeat_interleave(32, -1)


class Step:
    """A step of sequences with `new` tokens and `length` positions over pages in random order, one of `layers` that lie side by side.  What belongs to no sequence is not a number:
    steps and zeros of rows that nobody has and of rows behind a sequence's last position, and padding rows of the panel."""

    def __init__(self, new, length, heads, kv, hd, page, seed=0, layers=1, pad=0, drop=None, cols=0, extra=0):
        g = gen(seed)
        self.new, self.length, self.heads, self.kv, self.hd, self.page = list(new), list(length), heads, kv, hd, page
        held = [-(-n // page) for n in length]
        self.n_pages = sum(held) + 3
        self.cols = max(cols, max(held) + 1)
        order = torch.randperm(self.n_pages, generator=g, device="cuda").cpu().numpy()
        table, at = np.full((len(held), self.cols), 2 ** 31 - 1, dtype=np.int64), 0  # behind the last page: must not be followed
        valid = np.zeros((self.n_pages, page), dtype=bool)
        for i, n in enumerate(held):
            table[i, :n] = order[at:at + n]
            for j in range(n):
                valid[order[at + j], :min(page, length[i] - j * page)] = True
            at += n
        for i, j, e in drop or []:
            table[i, j] = e
        self.table = table
        self.rows = sum(new) + pad + extra
        start = np.concatenate([[0], np.cumsum(new)]) + extra
        self.bytes = kf.PagedQ4.page_bytes(page, kv, hd)
        assert self.bytes == page * kv * hd * 5 // 4
        self.pool = torch.full((self.n_pages, layers, self.bytes), 0xff, device="cuda", dtype=torch.uint8)
        self.pages = self.pool[:, layers // 2]
        e, r = (torch.from_numpy(x).cuda() for x in np.nonzero(valid))
        self.k, self.v, self.ks, self.vs = (torch.zeros(self.n_pages, page, kv, hd, device="cuda", dtype=torch.float64) for _ in range(4))
        rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
        for value, x, size in ((0, self.k, self.ks), (1, self.v, self.vs)):
            for a in range(0, len(e), 1 << 15):
                n = len(e[a:a + (1 << 15)])
                codes = (rnd(n, kv, hd) * 3.5 + 7.5).round().clamp(0, 15)
                step, zero = (0.3 * torch.exp(0.4 * rnd(n, kv, hd // 32))).bfloat16(), (7.5 + rnd(n, kv, hd // 32)).bfloat16()
                self.put(value, e[a:a + (1 << 15)], r[a:a + (1 << 15)], codes, step, zero)
        self.start = start.tolist()
        self.q = torch.full((self.rows, heads * hd), float("nan"), device="cuda", dtype=torch.bfloat16)
        a, b = self.start[0], self.start[-1]
        self.q[a:b] = (rnd(b - a, heads * hd) * 1.3).bfloat16()
        self.d = [i32(np.where(table > 2 ** 31 - 1, 0, table)), i32(start), i32(length)]
        self.desc = self.describe()

    def put(self, value, e, r, codes, step, zero):
        write(self.pages, self.kv, self.hd, self.page, value, e, r, codes, step, zero)
        (self.v if value else self.k)[e, r] = wide(step.double()) * (codes.double() - wide(zero.double()))
        (self.vs if value else self.ks)[e, r] = wide(step.double().abs()) * (codes.double() + wide(zero.double().abs()))

    def describe(self, **kw):
        d = dict(pool=At(self.pages), n_pages=self.n_pages, page_size=self.page, n_kv=self.kv, head_dim=self.hd, table=At(self.d[0]), table_cols=self.cols, n_seq=len(self.new),
                 q_start=At(self.d[1]), lens=At(self.d[2]), page_stride=self.pages.stride(0))
        d.update(kw)
        return kf.PagedQ4(**d)

    def flat(self, i, pool):
        """rows of sequence i, and which of them are there"""
        n = self.length[i]
        pages = self.table[i, :-(-n // self.page)]
        ok = torch.tensor([0 <= int(e) < self.n_pages for e in pages for _ in range(self.page)], device="cuda", dtype=torch.bool)[:n]
        idx = torch.tensor([int(e) if 0 <= int(e) < self.n_pages else 0 for e in pages], device="cuda", dtype=torch.long)
        return pool[idx].reshape(-1, self.kv, self.hd)[:n], ok

    def expect(self, scale, window, first=0, many=False, q=None):
        """(result, bound) of attention.  The bound counts
          - the result's rounding, half a step of it;
          - the rounding of weight times step to bf16, which both the codes' and the zeros' product take: at most half a step of the weighted mean of |v|;
          - fp32 errors of a score: hd + 32 roundings or truncations (2^-23) of sums whose terms add up to size = |q| . step (code + |zero|), and of its exponential, 2^-20; they
            change a weight by as much, in numerator and denominator;
          - fp32 errors of the sums of values, 2^-18 of the weighted mean of step (code + |zero|);
          - in the kernel for many rows (many) keys and values are rounded to bf16, half a step of each: of a score half a step of |q| . |k|, of the sum half a step of mean |v|."""
        q = self.q if q is None else q
        out = torch.full((self.rows, self.heads * self.hd), float("nan"), device="cuda", dtype=torch.float64)
        tol = torch.zeros_like(out)
        group = self.heads // self.kv
        for i, n in enumerate(self.new):
            if n == 0:
                continue
            a, e, hd = self.start[i], self.length[i], self.hd
            (k, ok), (v, _), (ks, _), (vs, _) = (self.flat(i, x) for x in (self.k, self.v, self.ks, self.vs))
            p = torch.arange(e - n, e, device="cuda")[:, None]
            j = torch.arange(e, device="cuda")[None]
            sees = (j <= p) & ok[None]
            if window > 0:
                sees = sees & ((j > p - window) | (j < first))
            hidden = ~sees.any(0)[:, None, None]
            k, v, ks, vs = (x.masked_fill(hidden, 0.0) for x in (k, v, ks, vs))
            for h in range(self.heads):
                qh, g = q[a:a + n, h * hd:(h + 1) * hd].double(), h // group
                s = (scale * (qh @ k[:, g].T)).masked_fill(~sees, -math.inf)
                top = s.amax(1, keepdim=True) if e else torch.full((n, 1), -math.inf, dtype=torch.float64, device="cuda")
                w = torch.exp(s - torch.where(torch.isinf(top), 0.0, top)).masked_fill(~sees, 0.0)
                tot = w.sum(1, keepdim=True)
                w = w / torch.where(tot == 0, 1.0, tot)
                r, mean, size = w @ v[:, g], w @ v[:, g].abs(), w @ vs[:, g]
                biggest = lambda x: (scale * (qh.abs() @ x[:, g].abs().T)).masked_fill(~sees, 0.0).amax(1, keepdim=True) if e else 0.0  # noqa: E731
                delta = (hd + 32) * 2.0 ** -23 * biggest(ks) + 2.0 ** -20
                if many:
                    delta = torch.expm1(delta + HALF16 * biggest(k))
                out[a:a + n, h * hd:(h + 1) * hd] = r
                tol[a:a + n, h * hd:(h + 1) * hd] = 1.01 * (HALF16 * r.abs() + ((2 if many else 1) * HALF16 + 2 * delta) * mean + 2.0 ** -18 * size) + 1e-30
        return out, tol

    def attend(self, ctx, scale, window=0, first=0, max_q=None, q=None, ldq=0, ldo=0, out=None, desc=None):
        out = torch.full((self.rows, ldo or self.heads * self.hd), 7.0, device="cuda", dtype=torch.bfloat16) if out is None else out
        kf.paged_attention_q4(ctx, desc or self.desc, At(self.q if q is None else q), self.rows, self.heads, max_q=max(self.new) if max_q is None else max_q, scale=scale, window=window,
                              first=first, ldq=ldq, ldo=ldo, out=At(out))
        return out

    def check(self, ctx, window=0, first=0, scale=None, **kw):
        scale = self.hd ** -0.5 if scale is None else scale
        out = self.attend(ctx, scale, window, first, **kw)
        ctx.sync()
        many = max(kw.get("max_q") or max(self.new), 1) * (self.heads // self.kv) > 16
        ref, tol = self.expect(scale, window, first, many)
        a, b = self.start[0], self.start[-1]
        got = out[:, :self.heads * self.hd].double()
        assert torch.all(out[:a] == 7) and torch.all(out[b:] == 7) and torch.all(out[:, self.heads * self.hd:] == 7), "padding was written"
        err = (got[a:b] - ref[a:b]).abs()
        bad = ~(err <= tol[a:b])
        assert not bad.any(), "%d of %d off, worst %g" % (int(bad.sum()), bad.numel(), float((err / tol[a:b]).nan_to_num(1e9).max()))
        # the bound is of the worst case; errors of many weights are independent, and the whole is nearer: the roundings above are 0.29 of a step (2^-7) each on the mean
        if float(ref[a:b].norm()) > 0:
            assert float(err.norm() / ref[a:b].norm()) < 0.0085 * (2 if many else 1) * max(1.0, scale * self.hd ** 0.5)
        return out


# ---------------------------------------------------------------------------------------------------------------- attention, single tokens and few rows
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group,kv", [(1, 1), (4, 2), (5, 3), (8, 8), (11, 2), (16, 1)])
@pytest.mark.parametrize("page", [8, 24, 64, 160])
def test_single_tokens(ctx, hd, group, kv, page):
    """One token each: lengths of one, on and around page and tile ends, a sequence without new tokens, one without any position."""
    length = [1, 2, page - 1, page, page + 1, 63, 64, 65, 0, 129, 700, 1000]
    new = [1] * 12
    new[8], new[10] = 0, 0
    Step(new, length, group * kv, kv, hd, page, seed=page + hd, layers=3 if page == 24 else 1, pad=3).check(ctx)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_seq,length", [(1, 5000), (1, 40000), (3, 9001), (40, 300), (300, 37)])
def test_single_tokens_runs(ctx, hd, n_seq, length):
    """Runs that end inside sequences, sequences over many runs, many sequences in a run, more than 32 of them."""
    r = np.random.RandomState(n_seq)
    lens = [length] if n_seq == 1 else r.randint(1, length, n_seq).tolist()
    Step([1] * n_seq, lens, 8, 2, hd, 16, seed=n_seq).check(ctx)


@pytest.mark.parametrize("first", [0, 1, 4, 60, 64, 130])
@pytest.mark.parametrize("window", [1, 7, 64, 100, 2 ** 31 - 1])
def test_single_tokens_window(ctx, window, first):
    """Window and first positions apart, in one tile, side by side and over one another; pages that neither needs given back, with entries of every kind."""
    length = [1, 64, 65, 128, 200, 333, 1024]
    drop = [(i, j, [-1, -7, 10 ** 6, 2 ** 31 - 1][j % 4]) for i, n in enumerate(length) for j in range(-(-n // 16)) if (j + 1) * 16 <= n - window and j * 16 >= first]
    Step([1] * 7, length, 8, 2, 128, 16, seed=window % 1000, drop=drop).check(ctx, window=window, first=first)


@pytest.mark.parametrize("first", [0, 5, 10 ** 9])
def test_first_positions_without_a_window(ctx, first):
    """Without a window everything is visible, whatever the first positions are; with all of them first, too."""
    s = Step([1, 3], [300, 100], 8, 2, 64, 16, seed=2)
    s.check(ctx, first=first)
    if first > 300:
        s.check(ctx, window=1, first=first)


def test_single_tokens_missing_pages(ctx):
    """Pages that are not there inside what a row would see, all of them in one sequence (zeros), the last one in another, and one among the first positions."""
    drop = [(0, 2, -1), (0, 3, 99999), (1, 0, -1), (1, 1, -1), (1, 2, -1), (2, 18, -1), (3, 0, -5), (4, 0, -1)]
    s = Step([1, 1, 1, 1, 1], [100, 48, 300, 17, 500], 8, 2, 64, 16, seed=5, drop=drop)
    out = s.check(ctx)
    assert torch.all(out[1] == 0)
    s.check(ctx, window=40, first=20)


def test_beyond_the_table(ctx):
    """A length above what the table holds: positions behind it are not there, those in front are seen, and where a window lies behind it only the first positions are."""
    s = Step([4, 1, 1], [100, 64, 400], 4, 2, 128, 16, seed=14)
    s.desc = s.describe(table=At(i32(s.table[:, :6])), table_cols=6)
    s.table = s.table.copy()
    s.table[0, 6] = -1
    s.table[2, 6:] = -1
    s.check(ctx)
    s.check(ctx, window=30, first=7)
    out = s.check(ctx, window=30)
    assert torch.all(out[5] == 0)


def test_single_tokens_scales(ctx):
    """Weights on one position, and on all alike."""
    for scale in (8.0, 1e-6):
        Step([1, 1], [500, 77], 8, 2, 128, 16, seed=3).check(ctx, scale=scale)


@pytest.mark.parametrize("size", [2.0 ** -40, 2.0 ** -20, 2.0 ** 20, 2.0 ** 40])
@pytest.mark.parametrize("max_q", [1, 40])
def test_sizes_of_values(ctx, size, max_q):
    """Steps from very small to very large, of keys against queries of the inverse size, and of values."""
    s = Step([1, 3], [300, 77], 8, 2, 128, 16, seed=3)
    held = [(i, torch.arange(n, device="cuda")) for i, n in enumerate(s.length)]
    for i, t in held:
        e, r = torch.from_numpy(s.table[i]).cuda()[t // 16], t % 16
        for value, f in ((0, size), (1, 1 / size)):
            codes, step, zero = read(s.pages, s.kv, s.hd, 16, value, e, r)
            s.put(value, e, r, codes, (step * f).bfloat16(), zero.bfloat16())
    s.q = (s.q.float() / size).bfloat16()
    s.check(ctx, max_q=max_q)


def test_zeros_far_from_the_codes(ctx):
    """Groups whose values lie far from 0: zeros of hundreds of steps."""
    s = Step([1, 2], [200, 60], 8, 2, 128, 16, seed=4)
    for i, n in enumerate(s.length):
        t = torch.arange(n, device="cuda")
        e, r = torch.from_numpy(s.table[i]).cuda()[t // 16], t % 16
        for value in (0, 1):
            codes, step, zero = read(s.pages, s.kv, s.hd, 16, value, e, r)
            far = torch.where(torch.arange(s.hd // 32, device="cuda") % 2 == 1, -600.0, 900.0).expand_as(zero) + 8 * (zero - 7)
            s.put(value, e, r, codes, (step / 16).bfloat16(), far.bfloat16())
    s.check(ctx)


@pytest.mark.parametrize("new,length", [([1, 1, 1], [70, 5, 640]), ([1, 50, 3], [70, 55, 640])])
def test_rows_and_strides(ctx, new, length):
    """Queries inside wider rows, results in wider rows and at any element, rows in front of the first sequence, pages of more entries than the table says."""
    s = Step(new, length, 8, 2, 128, 32, seed=8, extra=2, pad=1, cols=40)
    wider = torch.zeros(s.rows, 8 * 128 + 64, device="cuda", dtype=torch.bfloat16)
    wider[:, 64:] = s.q
    buf = torch.full((s.rows * (8 * 128 + 5) + 1,), 7.0, device="cuda", dtype=torch.bfloat16)
    out = buf[1:].view(s.rows, 8 * 128 + 5)
    s.check(ctx, q=wider[:, 64:], ldq=8 * 128 + 64, ldo=8 * 128 + 5, out=out)
    assert buf[0] == 7


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q", [2, 3, 4, 7])
def test_drafts(ctx, hd, q):
    """A few tokens each, 10 to 35 rows a kv head: two columns of rows, and the step from one kernel to the other."""
    r = np.random.RandomState(q)
    new = [q] * 9 + [1, 0, q - 1]
    Step(new, [n + int(r.choice([0, 1, 100, 127, 128, 600, 1300])) for n in new], 15, 3, hd, 24, seed=q, pad=1).check(ctx)


@pytest.mark.parametrize("max_q", [1, 40])
def test_hidden_values(ctx, max_q):
    """Steps and zeros that are not numbers in positions that no row sees, between the first ones and the window and inside their tiles."""
    s = Step([1, 1], [90, 161], 8, 2, 128, 64, seed=9)
    for i, n in ((0, 90), (1, 161)):
        t = torch.arange(3, n - 50, device="cuda")
        e, r = torch.from_numpy(s.table[i]).cuda()[t // 64], t % 64
        for value in (0, 1):
            codes, step, zero = read(s.pages, s.kv, s.hd, 64, value, e, r)
            write(s.pages, s.kv, s.hd, 64, value, e, r, codes, torch.full_like(step, float("inf")), torch.full_like(zero, float("nan")))
    s.check(ctx, window=50, first=3, max_q=max_q)


def test_a_value_that_is_not_finite(ctx):
    """A visible group of NaN makes the results of its sequence's rows NaN and nobody else's."""
    s = Step([1, 1, 1], [90, 61, 20], 8, 2, 128, 16, seed=9)
    e = torch.tensor([int(s.table[1, 2])], device="cuda")
    for value in (0, 1):
        codes, step, zero = read(s.pages, s.kv, s.hd, 16, value, e, torch.tensor([3], device="cuda"))
        write(s.pages, s.kv, s.hd, 16, value, e, torch.tensor([3], device="cuda"), codes * 0, torch.full_like(step, float("nan")), zero * 0)
    out = s.attend(ctx, 0.1)
    ctx.sync()
    ref, tol = s.expect(0.1, 0)
    assert torch.all(torch.isnan(out[1]))
    assert torch.all((out.double() - ref).abs()[[0, 2]] <= tol[[0, 2]])


# ---------------------------------------------------------------------------------------------------------------- several tokens a sequence
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group,kv", [(1, 2), (4, 2), (5, 1), (7, 2), (8, 1), (17, 2), (64, 1)])
@pytest.mark.parametrize("new,past", [([2, 3, 1], [0, 62, 300]), ([5, 17, 0, 64], [1000, 3, 9, 0]), ([130, 1, 257], [0, 40, 511])])
def test_chunks(ctx, hd, group, kv, new, past):
    """Chunks on and around block and tile ends beside single tokens and an idle sequence."""
    Step(new, [a + b for a, b in zip(new, past)], group * kv, kv, hd, 16, seed=sum(new) + group, pad=2).check(ctx)


@pytest.mark.parametrize("max_q", [0, 1, 2, 3, 100000])
def test_hint(ctx, max_q):
    """max_q is a hint: results hold whatever it says."""
    Step([1, 40, 3, 0, 200], [9, 50, 400, 5, 1000], 8, 2, 128, 16, seed=21).check(ctx, max_q=max_q)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("first", [0, 3, 64, 200])
@pytest.mark.parametrize("window", [1, 33, 128, 500])
def test_chunks_window(ctx, hd, window, first):
    new, length = [3, 150, 1, 300, 40], [40, 150, 700, 900, 640]
    drop = [(i, j, -1) for i, n in enumerate(length) for j in range(-(-n // 8)) if (j + 1) * 8 <= n - new[i] + 1 - window and j * 8 >= first]
    s = Step(new, length, 8, 2, hd, 8, seed=window, drop=drop, layers=2)
    s.check(ctx, window=window, first=first)
    s.check(ctx, window=window, first=first, max_q=2)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group,kv,window,first", [(7, 4, 0, 0), (7, 4, 300, 0), (4, 2, 100, 70), (12, 2, 0, 0)])
@pytest.mark.parametrize("seed", [0, 1])
def test_mixed_runs(ctx, hd, group, kv, window, first, seed):
    """Steps with several blocks in a run: blocks of one row tile and of two, of one tile of positions and of many, in every order."""
    r = np.random.RandomState(seed)
    new = [1, 1, 1, 90, 1, 0, 30, 1, 40, 1] + [int(r.choice([1, 1, 2, 20, 75])) for _ in range(50)]
    length = [n + int(r.choice([0, 60, 200, r.randint(0, 900)])) for n in new]
    Step(new, length, group * kv, kv, hd, 16, seed=seed).check(ctx, window=window, first=first)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,first", [(0, 0), (700, 5)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_long_mixed_runs(ctx, hd, window, first, seed):
    """Many tiles a thread block: blocks with one and with two row tiles and single tokens, whose tiles are worth one or two units, so that runs begin and end inside tiles."""
    r = np.random.RandomState(100 * hd + seed)
    new = [int(x) for x in r.choice([1, 1, 2, 5, 20, 33, 70, 150], 14)] + [0, 1]
    length = [n + int(r.randint(0, 7000)) for n in new]
    s = Step(new, length, 8 * (4 if seed else 7), 8, hd, 64, seed=seed, pad=1)
    assert sum(-(-n // 128) for n in length) * 8 > 4 * 148 and 8 * 4 * 2 > 16
    s.check(ctx, window=window, first=first, max_q=150)


def test_chunks_before_the_first_position(ctx):
    """More new tokens than positions: the first rows stand before position 0 and see nothing."""
    s = Step([20, 40], [8, 33], 4, 1, 128, 8, seed=4)
    for window, first in ((0, 0), (5, 2)):
        out = s.attend(ctx, 0.1, window=window, first=first)
        ctx.sync()
        assert torch.all(out[:12] == 0) and torch.all(out[20:27] == 0)
        t = Step([8, 33], [8, 33], 4, 1, 128, 8, seed=4)
        t.k, t.v, t.ks, t.vs, t.table = s.k, s.v, s.ks, s.vs, s.table
        ref, tol = t.expect(0.1, window, first, many=True, q=torch.cat([s.q[12:20], s.q[27:60]]))
        got = torch.cat([out[12:20], out[27:60]]).double()
        assert torch.all((got - ref).abs() <= tol)


def test_chunks_missing_pages(ctx):
    s = Step([100, 9], [400, 9], 8, 2, 128, 24, seed=6, drop=[(0, 0, -1), (0, 7, -2), (0, 14, 5000), (1, 0, -1)])
    out = s.check(ctx)
    assert torch.all(out[100:109] == 0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_seq,chunk", [(1100, 0), (2500, 30), (8192, 40)])
def test_attention_of_many_sequences(ctx, hd, n_seq, chunk):
    """More than 1024 sequences, most of them idle or with one token: a run begins behind many that it has no part in."""
    r = np.random.RandomState(n_seq + chunk)
    new = (r.rand(n_seq) < min(1.0, 400 / n_seq)).astype(int)
    length = new + r.randint(0, 30, n_seq)
    new[0], length[0], new[-1], length[-1] = 1, 200, 1, 333
    if chunk:
        for i in (5, n_seq // 2, n_seq - 2):
            new[i], length[i] = chunk, chunk + 100
    Step(new, length, 4, 2, hd, 16, seed=chunk, pad=1).check(ctx)


def test_shared_pages(ctx):
    """Sequences that share the pages of a prefix, and a page that stands twice in a table."""
    s = Step([1, 1, 1], [130, 150, 90], 8, 2, 128, 16, seed=7)
    s.table[1, :8] = s.table[0, :8]
    s.table[2, 3] = s.table[2, 1]
    s.d[0].copy_(i32(np.where(s.table > 2 ** 31 - 1, 0, s.table)))
    s.check(ctx)


@pytest.mark.parametrize("new", [[1, 30], [1, 2]])
def test_far_pages(ctx, new):
    """Pages that lie more than 2^32 bytes apart from the first."""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 12 GB")
    s = Step(new, [300, 200], 16, 8, 128, 16, seed=15)
    stride = (1 << 28) + 16
    assert s.n_pages * stride > 1 << 33
    pool = torch.empty((s.n_pages - 1) * stride + s.bytes, device="cuda", dtype=torch.uint8)
    far = pool.as_strided((s.n_pages, s.bytes), (stride, 1))
    far.copy_(s.pages)
    s.pages = far
    s.desc = s.describe()
    s.check(ctx)
    back = [torch.zeros(s.rows, 8 * 128, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    kf.paged_read_q4(ctx, s.desc, s.rows, k_out=At(back[0]), v_out=At(back[1]))
    torch.cuda.synchronize()
    for i, n in enumerate(s.new):
        for x, b in ((s.k, back[0]), (s.v, back[1])):
            want = s.flat(i, x)[0][s.length[i] - n:].flatten(1)
            assert torch.equal(b[s.start[i]:s.start[i] + n], want.float().bfloat16())
    k = torch.randn(s.rows, 8 * 128, device="cuda").bfloat16()
    kf.paged_append_q4(ctx, s.desc, None, At(s.q), At(k), At(k), s.rows, 16, out=At(s.q))
    kf.paged_read_q4(ctx, s.desc, s.rows, k_out=At(back[0]), v_out=At(back[1]))
    torch.cuda.synchronize()
    want = stands_for(k.float().view(-1, 8, 128)).flatten(1).bfloat16()
    assert torch.equal(back[0], want) and torch.equal(back[1], want)


def test_same_bits(ctx):
    """Pieces are merged in order: the same call gives the same bits, whatever ran before."""
    for new, length in (([1, 1, 60, 5], [3000, 700, 900, 5000]), ([1, 1, 2, 1], [3000, 700, 900, 5000])):
        s = Step(new, length, 8, 2, 128, 16, seed=31)
        other = Step([130] * 20, [400] * 20, 64, 1, 128, 16, seed=3)
        loud = other.q * 50
        a = s.attend(ctx, 0.1)
        for i in range(5):
            if i > 1:
                other.attend(ctx, 0.1, q=loud)
            b = s.attend(ctx, 0.1)
            ctx.sync()
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("group,kv", [(5, 8), (7, 4), (12, 3), (17, 3)])
@pytest.mark.parametrize("hd", [64, 128])
def test_same_bits_whatever_ran_before(ctx, group, kv, hd):
    """Rows of a row tile that are nobody's hold what the call before left in shared memory, here queries fifty times as large: no result depends on them."""
    for new in ([138, 1, 77], [1, 1, 1]):
        s = Step(new, [2231, 900, 1500], group * kv, kv, hd, 16, seed=group)
        other = Step([130] * 20, [400] * 20, 64, 1, hd, 16, seed=3)
        loud = other.q * 50
        a = s.attend(ctx, hd ** -0.5)
        for _ in range(4):
            other.attend(ctx, hd ** -0.5, q=loud)
            b = s.attend(ctx, hd ** -0.5)
            ctx.sync()
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("window,first", [(5, 0), (70, 3), (300, 40)])
@pytest.mark.parametrize("max_q", [150, 2])
def test_chunks_hidden_values(ctx, hd, page, window, first, max_q):
    """Steps and zeros that are not finite behind the first positions and before the first row's window, in pages that are still there, and behind the last position."""
    new, length = [3, 150, 1, 60], [500, 640, 777, 64]
    s = Step(new, length, 8, 2, hd, page, seed=window + page)
    for i, n in enumerate(length):
        t = torch.arange(first, max(first, n - new[i] + 1 - window), device="cuda")
        if len(t) == 0:
            continue
        e, r = torch.from_numpy(s.table[i]).cuda()[t // page], t % page
        for value in (0, 1):
            codes, step, zero = read(s.pages, s.kv, s.hd, page, value, e, r)
            nan = (t % 2 == 0)[:, None, None].expand_as(step)
            write(s.pages, s.kv, s.hd, page, value, e, r, codes, torch.where(nan, float("nan"), torch.full_like(step, float("inf"))), torch.where(nan, zero, torch.full_like(zero, float("-inf"))))
    s.check(ctx, window=window, first=first, max_q=max_q)


# ---------------------------------------------------------------------------------------------------------------- append and read
def quantised(x):
    """x [.., hd] fp32 -> codes [.., hd], step, zero [.., groups] by the definition, in fp32 on the CPU (true divisions)."""
    x = x.float().cpu().unflatten(-1, (-1, 32))
    lo, hi = x.amin(-1), x.amax(-1)
    step = torch.maximum((hi - lo) / 15, x.abs().amax(-1) / 2048)
    step = ((step.view(torch.int32) + 0xffff) & -0x10000).view(torch.float32)
    some = torch.where(step > 0, step, 1.0)
    zero = torch.where(step > 0, -lo / some, 0.0).bfloat16().float()
    codes = (x / some[..., None] + zero[..., None]).round().clamp(0, 15).flatten(-2)
    return codes.cuda(), step.cuda(), zero.cuda()


def stands_for(x):
    c, s, z = quantised(x)
    return wide(s) * (c - wide(z))


def append_and_check(ctx, src, hd, heads, kv, rot, layout, axes, norm, off, new, length):
    g = gen(hd + rot + axes)
    s = Step(new, length, heads, kv, hd, 24, seed=1, extra=1, pad=2, layers=1 + off)
    ld = (heads + 2 * kv) * hd + 8 + off
    panel = torch.randn(s.rows, ld, generator=g, device="cuda").to(src)
    q, k, v = (panel[:, off + a * hd:off + b * hd] for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    freq = 1e4 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) / max(1, rot // 2))
    axis = torch.arange(rot // 2, device="cuda", dtype=torch.int32) % axes
    pos = torch.randint(-3, 200000, (axes, s.rows + 3), generator=g, device="cuda", dtype=torch.int32) if axes > 1 else None
    wq, wk = ((1 + 0.3 * torch.randn(hd, generator=g, device="cuda")).bfloat16() for _ in "qk") if norm else (None, None)
    amp = 1.25 if axes == 2 else 1.0
    r = kf.Rotation(At(freq), rot, layout=layout, amp=amp, n_axes=axes, pair_axis=At(axis) if axes > 1 else None, pos=At(pos) if axes > 1 else None, pos_stride=s.rows + 3 if axes > 1 else 0)
    out = torch.full((s.rows, heads * hd + off), 7.0, device="cuda", dtype=torch.bfloat16)
    before = s.pool.clone()
    kf.paged_append_q4(ctx, s.desc, r, At(q), At(k), At(v), s.rows, heads, q_norm=At(wq) if norm else None, k_norm=At(wk) if norm else None, eps=1e-5, ldq=ld, ldk=ld, ldv=ld,
                       out=At(out), ldo=heads * hd + off, src_f32=src == torch.float32)
    torch.cuda.synchronize()
    a, b = s.start[0], s.start[-1]
    assert torch.all(out[:a] == 7) and torch.all(out[b:] == 7) and torch.all(out[:, heads * hd:] == 7)
    mine = before[:, (1 + off) // 2]
    for i, n in enumerate(new):
        if n == 0:
            continue
        lo, hi = s.start[i], s.start[i + 1]
        place = torch.arange(length[i] - n, length[i], device="cuda")
        p = [place] if pos is None else [pos[x, lo:hi] for x in range(axes)]
        e, row = torch.from_numpy(s.table[i]).cuda()[place // 24], place % 24
        for x, w, h, kind in ((q, wq, heads, "q"), (k, wk, kv, "k")):
            y, size = turned(normed(x[lo:hi].double().reshape(n, h, hd), w, 1e-5), freq, axis if axes > 1 else axis * 0, p, layout, amp)
            err = (TURN + NORM) * amp * size  # of the finished row, fp32
            if kind == "q":
                got = out[lo:hi, :heads * hd].reshape(n, h, hd)
                assert torch.all((got.double() - y).abs() <= 1.01 * (HALF16 * y.abs() + err) + 1e-30), (kind, i)
                continue
            codes, step, zero = read(s.pages, kv, hd, 24, 0, e, row)
            # the step is the definition's, one bf16 up or down where the rows' own errors carry it over (2^-7); a code is off by half a step, by the zero's rounding (a step of
            # bf16 of it is at most |zero| / 128, half of that) and by the row's error
            yg = y.unflatten(-1, (-1, 32))
            want = torch.maximum((yg.amax(-1) - yg.amin(-1)) / 15, yg.abs().amax(-1) / 2048)
            slack = 2 * err.unflatten(-1, (-1, 32)).amax(-1) / 15
            assert torch.all(step >= want * (1 - 2 ** -22) - slack) and torch.all(step <= (want + slack) * (1 + 2 ** -7 + 2 ** -22))
            got = wide(step) * (codes - wide(zero))
            tol = wide(step) * (0.5 + wide(zero.abs()) / 256 + 2 ** -20) * (1 + 2 ** -20) + 2 * err
            assert torch.all((got - y).abs() <= tol), (kind, i, float(((got - y).abs() / tol).max()))
            if not norm and rot == 0:
                c, st, z = quantised(x[lo:hi].reshape(n, h, hd))
                assert torch.equal(codes, c.double()) and torch.equal(step, st.double()) and torch.equal(zero, z.double())
            write(mine, kv, hd, 24, 0, e, row, codes, step, zero)
        c, st, z = quantised(v[lo:hi].reshape(n, kv, hd))
        codes, step, zero = read(s.pages, kv, hd, 24, 1, e, row)
        assert torch.equal(codes, c.double()) and torch.equal(step, st.double()) and torch.equal(zero, z.double())
        write(mine, kv, hd, 24, 1, e, row, codes, step, zero)
    assert torch.equal(before, s.pool), "something else was written"


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,heads,kv,rot,layout,axes,norm", [
    (128, 8, 2, 128, 1, 1, True), (128, 5, 5, 64, 1, 3, False), (128, 32, 8, 128, 0, 3, True), (64, 7, 1, 64, 1, 1, True), (64, 4, 2, 6, 0, 2, False),
    (128, 3, 1, 40, 1, 2, True), (64, 16, 4, 0, 1, 1, True), (64, 3, 3, 0, 1, 1, False), (128, 6, 3, 0, 0, 1, False), (128, 4, 2, 96, 1, 1, True)])
@pytest.mark.parametrize("off", [0, 1])
def test_append(ctx, src, hd, heads, kv, rot, layout, axes, norm, off):
    """Every layout and type, rows at 16 bytes and at any element (off), tokens on page ends, a sequence without new tokens, padding on both sides; every byte of the pool that
    belongs to no new token stays as it was."""
    append_and_check(ctx, src, hd, heads, kv, rot, layout, axes, norm, off, [1, 40, 0, 7, 1], [1, 100, 30, 24, 300])


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,heads,kv,rot,layout,axes,norm", [(128, 3, 1, 128, 1, 3, True), (64, 20, 5, 32, 0, 1, False), (128, 65, 8, 128, 0, 1, True), (64, 2, 2, 64, 1, 2, False)])
@pytest.mark.parametrize("off", [0, 1])
def test_append_panels(ctx, src, hd, heads, kv, rot, layout, axes, norm, off):
    """Panels of so many tokens that a block takes four: sequences that end inside one, padding on both sides, heads that take one turn of a block and several."""
    append_and_check(ctx, src, hd, heads, kv, rot, layout, axes, norm, off, [1501, 1, 0, 1202, 3, 1], [1501, 700, 5, 1300, 24, 1])


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
def test_append_kinds_of_groups(ctx, src):
    """Groups of zeros, of one value, of values far from 0 with a small range, of very small and very large ones, with ties, and with entries that are not finite: what comes
    back is the definition's, and of the last NaN."""
    r = np.random.RandomState(0)
    rows = [np.zeros(32), np.full(32, 3.7), np.full(32, -1e-30), 100 + 0.5 * r.rand(32), -7 - r.rand(32), 1e-20 * r.randn(32), 1e14 * r.randn(32), np.arange(32) % 16 * 0.25 + 0.125,
            (np.arange(32) - 16) * 0.5, np.r_[np.zeros(31), 5.0], np.r_[np.full(31, 2.0 ** -20), 1.0], np.r_[np.full(31, -3.0), 0.0]]
    bad = [np.r_[r.randn(31), np.nan], np.r_[np.inf, r.randn(31)], np.r_[r.randn(16), -np.inf, r.randn(15)], np.r_[3e38, -3e38, np.zeros(30)]]
    x = torch.tensor(np.stack(rows + bad), dtype=torch.float32).to(src).cuda()
    n = len(rows) + len(bad)
    k = x.view(n // 4, 128).contiguous()
    s = Step([n // 4], [50], 1, 1, 128, 16, seed=1)
    kf.paged_append_q4(ctx, s.desc, None, At(s.q if src == torch.bfloat16 else s.q.float()), At(k), At(k), n // 4, 1, out=At(torch.zeros_like(s.q)), src_f32=src == torch.float32)
    back = [torch.zeros(n // 4, 128, device="cuda") for _ in "kv"]
    kf.paged_read_q4(ctx, s.desc, n // 4, k_out=At(back[0]), v_out=At(back[1]), out_f32=True)
    torch.cuda.synchronize()
    want = stands_for(x)
    for b in back:
        b = b.view(n, 32)
        assert torch.equal(b[:len(rows)], want[:len(rows)]) and torch.all(torch.isnan(b[len(rows):]))
    c, st, z = quantised(x[:len(rows)])
    assert torch.all((want[:len(rows)].double() - x[:len(rows)].double()).abs() <= wide(st).double() * (0.5 + wide(z.abs()).double() / 256 + 2 ** -20))


def test_append_many_sequences(ctx):
    """Finding a token's sequence among up to 8192, most of them without new tokens, and reading the rows back."""
    r = np.random.RandomState(0)
    for n_seq in (33, 1025, 8192):
        new = (r.rand(n_seq) < 0.02).astype(int) * r.randint(1, 4, n_seq)
        new[-1], new[0] = 2, 1
        length = new + r.randint(0, 9, n_seq)
        s = Step(new, length, 1, 1, 64, 8, seed=n_seq)
        k, v = (torch.randn(s.rows, 64, device="cuda").bfloat16() for _ in "kv")
        kf.paged_append_q4(ctx, s.desc, None, At(s.q), At(k), At(v), s.rows, 1, out=At(s.q))
        back = [torch.zeros(s.rows, 64, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
        kf.paged_read_q4(ctx, s.desc, s.rows, k_out=At(back[0]), v_out=At(back[1]))
        torch.cuda.synchronize()
        assert torch.equal(back[0], stands_for(k).bfloat16()) and torch.equal(back[1], stands_for(v).bfloat16())


def test_append_missing_pages(ctx):
    """Nothing is written for a token whose page is not there or that lies outside the table, its query is finished all the same, and its rows read as zeros."""
    s = Step([6, 3, 2, 4], [30, 3, 2, 2], 2, 1, 64, 8, seed=2, drop=[(0, 3, -1), (1, 0, 10 ** 8)])
    s.d[2][2] = 8 * s.cols + 1  # the third sequence's second token is behind the table; the last one's first two stand before position 0
    before = s.pool.clone()
    k = torch.randn(s.rows, 64, device="cuda").bfloat16()
    out = torch.zeros_like(s.q)
    kf.paged_append_q4(ctx, s.desc, None, At(s.q), At(k), At(k), s.rows, 2, out=At(out))
    back = torch.full((s.rows, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    kf.paged_read_q4(ctx, s.desc, s.rows, v_out=At(back))
    torch.cuda.synchronize()
    assert torch.equal(out, s.q)
    there = [13, 14]
    assert torch.all(back[[i for i in range(15) if i not in there]] == 0) and torch.equal(back[there], stands_for(k[there]).bfloat16())
    e = int(s.table[3, 0])
    before[e], s.pool[e] = 0, 0
    assert torch.equal(before, s.pool)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,kv,page", [(64, 1, 8), (64, 3, 40), (128, 8, 16), (128, 5, 64), (128, 1, 24)])
@pytest.mark.parametrize("off", [0, 1, 4])
def test_read(ctx, t, hd, kv, page, off):
    """Whole sequences and parts of them, in rows at any element and side by side, with padding on both sides that stays as it is."""
    new, length = [1, 33, 0, 100, 7, page], [1, 33, 20, 321, 500, page]
    s = Step(new, length, kv, kv, hd, page, seed=hd + page, extra=2, pad=5, layers=2)
    ld = 2 * kv * hd + 2 * off
    buf = torch.full((s.rows, ld), 7.0, device="cuda", dtype=t)
    kf.paged_read_q4(ctx, s.desc, s.rows, k_out=At(buf[:, off:]), v_out=At(buf[:, off + kv * hd:]), ldk=ld, ldv=ld, out_f32=t == torch.float32)
    torch.cuda.synchronize()
    want = torch.full_like(buf, 7.0)
    for i, n in enumerate(new):
        for x, at in ((s.k, off), (s.v, off + kv * hd)):
            want[s.start[i]:s.start[i] + n, at:at + kv * hd] = s.flat(i, x)[0][length[i] - n:].flatten(1).float().to(t)  # step (code - zero) is exact in fp32 but for one rounding
    # the product step * (code - zero): code - zero has at most 12 bits here, the step 8, so 32 bits hold it
    assert torch.equal(buf, want)
    for only in "kv":
        one = torch.full((s.rows, kv * hd), 7.0, device="cuda", dtype=t)
        kf.paged_read_q4(ctx, s.desc, s.rows, **{only + "_out": At(one)}, out_f32=t == torch.float32)
        torch.cuda.synchronize()
        at = off + (kv * hd if only == "v" else 0)
        assert torch.equal(one, want[:, at:at + kv * hd])


def test_read_long(ctx):
    """More rows than a block takes, by far, and a sequence read from its middle."""
    s = Step([9000, 3001], [9000, 5000], 8, 8, 128, 32, seed=3)
    back = [torch.zeros(s.rows, 8 * 128, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    kf.paged_read_q4(ctx, s.desc, s.rows, k_out=At(back[0]), v_out=At(back[1]))
    torch.cuda.synchronize()
    for i, n in enumerate(s.new):
        for x, b in ((s.k, back[0]), (s.v, back[1])):
            assert torch.equal(b[s.start[i]:s.start[i] + n], s.flat(i, x)[0][s.length[i] - n:].flatten(1).float().bfloat16())


# ---------------------------------------------------------------------------------------------------------------- together
def serve(ctx, heads, kv, hd, page, chunks, window=0, first=0, seed=0, graph=False):
    """Sequences fed in steps of `chunks` (a list of steps, each a list of new tokens per sequence): append, attention and reading back.  Attention is compared with attention over
    everything in 64 bits, with the keys and values that the cache says it holds; these with what went in."""
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
    pool = torch.full((n_pages, kf.PagedQ4.page_bytes(page, kv, hd)), 0xff, device="cuda", dtype=torch.uint8)
    freq = 1e4 ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) / (hd // 2))
    wq, wk = ((1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).bfloat16() for _ in "qk")
    ld = (heads + 2 * kv) * hd
    most = max(int(np.sum(c)) for c in chunks)
    panel, qbuf, out = (torch.zeros(most, w, device="cuda", dtype=torch.bfloat16) for w in (ld, heads * hd, heads * hd))
    back = [torch.zeros(most, kv * hd, device="cuda") for _ in "kv"]
    start, lens = i32([0] * (n_seq + 1)), i32([0] * n_seq)
    desc = kf.PagedQ4(At(pool), n_pages, page, kv, hd, At(table), max(held), n_seq, At(start), At(lens))
    rot = kf.Rotation(At(freq), hd)
    max_q = max(max(c) for c in chunks)
    many = max_q * (heads // kv) > 16

    def step():
        kf.paged_append_q4(ctx, desc, rot, At(panel), At(panel[:, heads * hd:]), At(panel[:, (heads + kv) * hd:]), most, heads, At(wq), At(wk), ldq=ld, ldk=ld, ldv=ld, out=At(qbuf))
        kf.paged_attention_q4(ctx, desc, At(qbuf), most, heads, max_q=max_q, window=window, first=first, out=At(out))
        kf.paged_read_q4(ctx, desc, most, k_out=At(back[0]), v_out=At(back[1]), out_f32=True)

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
        panel[:n] = torch.randn(n, ld, generator=g, device="cuda").bfloat16()
        start.copy_(i32(np.concatenate([[0], np.cumsum(c)])))
        lens.copy_(i32(past + c))
        out.fill_(7.0)
        torch.cuda.synchronize()
        if graph:
            ctx.check(ctx.lib.kf_graph_launch(ctx.h, h), "launch")
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
            k, size = turned(normed(x[:, heads * hd:(heads + kv) * hd].reshape(m, kv, hd), wk, 1e-6), freq, torch.zeros(hd // 2, dtype=torch.int32), [place], 1, 1.0)
            kb, vb = (b[row:row + m].view(m, kv, hd) for b in back)
            # a group's step is at most its range / 15 and a bf16 step of that, its zero under 16
            kg = k.unflatten(-1, (-1, 32))
            tol = wide((kg.amax(-1) - kg.amin(-1).clamp(max=0)).clamp(min=0) / 15 * 0.6) + (TURN + NORM) * 4 * size
            assert torch.all((kb.double() - k).abs() <= tol)
            assert torch.equal(vb, stands_for(x[:, (heads + kv) * hd:].reshape(m, kv, hd)))
            keys[i].append(kb.double()), vals[i].append(vb.double())
            q = qbuf[row:row + m].double().view(m, heads, hd)
            kk, vv = torch.cat(keys[i]), torch.cat(vals[i])
            j = torch.arange(len(kk), device="cuda")[None]
            sees = j <= place[:, None]
            if window:
                sees = sees & ((j > place[:, None] - window) | (j < first))
            for hh in range(heads):
                s = (q[:, hh] @ kk[:, hh // (heads // kv)].T) * hd ** -0.5
                size = (q[:, hh].abs() @ kk[:, hh // (heads // kv)].abs().T) * hd ** -0.5
                w = torch.softmax(s.masked_fill(~sees, -math.inf), 1)
                v = vv[:, hh // (heads // kv)]
                r, mean = w @ v, w @ v.abs()
                # as in Step.expect; step (code + |zero|) is under 16 steps + 16, of keys and values whose groups' ranges are 15 steps: bounded by 40 steps, so by 40 / 7 of the
                # largest |x| of a group, here by 8 times the mean size
                delta = torch.expm1(((HALF16 if many else 0) + 8 * (hd + 32) * 2.0 ** -23) * size.masked_fill(~sees, 0.0).amax(1, keepdim=True)) + 2.0 ** -19
                err = (out[row:row + m, hh * hd:(hh + 1) * hd].double() - r).abs()
                assert torch.all(err <= 1.01 * (HALF16 * r.abs() + ((2 if many else 1) * HALF16 + 2 * delta) * mean) + 2.0 ** -15 * mean.amax()), (c, i, hh)
                assert float(err.norm() / r.norm()) < 0.02
            row += m
        past = past + np.asarray(c)
    if h:
        ctx.check(ctx.lib.kf_graph_destroy(h), "destroy")


@pytest.mark.parametrize("heads,kv,hd,page,window,first", [(8, 2, 128, 16, 0, 0), (4, 4, 64, 24, 0, 0), (10, 2, 128, 16, 50, 4), (8, 1, 64, 8, 90, 20)])
def test_serving(ctx, heads, kv, hd, page, window, first):
    """A prompt in chunks beside decoding sequences, drafts, idle slots."""
    serve(ctx, heads, kv, hd, page, [[70, 1, 5], [130, 1, 0], [1, 1, 300], [1, 0, 1], [4, 5, 3], [1, 1, 1]], window, first)


def test_serving_single_tokens(ctx):
    """Decoding from the first token on, in the kernel for few rows."""
    serve(ctx, 8, 2, 128, 8, [[1, 1, 0]] * 3 + [[1, 2, 1]] * 20, window=9, first=2)


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
    h = C.c_void_p()
    c.check(c.lib.kf_graph_begin(c.h), "begin")
    with pytest.raises(kf.KoifishError, match="before graph capture"):
        a.attend(c, 0.1, out=outs[0])
    c.check(c.lib.kf_graph_end(c.h, C.byref(h)), "end")
    c.check(c.lib.kf_graph_destroy(h), "destroy")
    for s, o in zip((b, a), reversed(outs)):
        s.attend(c, 0.1, out=o)
    graphs = []
    for s, o in zip((a, b), outs):
        h = C.c_void_p()
        c.check(c.lib.kf_graph_begin(c.h), "begin")
        s.attend(c, 0.1, out=o)
        c.check(c.lib.kf_graph_end(c.h, C.byref(h)), "end")
        graphs.append(h)
    c.sync()
    for o in outs:
        o.fill_(7.0)
    torch.cuda.synchronize()
    for h in graphs * 2 + graphs[::-1]:
        c.check(c.lib.kf_graph_launch(c.h, h), "launch")
    c.sync()
    for s, o, many in zip((a, b), outs, (False, True)):
        ref, tol = s.expect(0.1, 0, many=many)
        assert torch.all((o.double() - ref).abs() <= tol)
    for h in graphs:
        c.check(c.lib.kf_graph_destroy(h), "destroy")
    c.close()


def test_two_streams():
    """Two contexts on two streams at once, each with its own workspace."""
    a, b = Step([1] * 8, [900] * 8, 8, 2, 128, 16, seed=62), Step([1, 40], [5000, 400], 8, 2, 64, 16, seed=63)
    torch.cuda.synchronize()
    cs = [kf.Context(0), kf.Context(0)]
    outs = [torch.zeros(s.rows, s.heads * s.hd, device="cuda", dtype=torch.bfloat16) for s in (a, b)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, c, o in zip((a, b), cs, outs):
            s.attend(c, 0.1, out=o)
    for s, c, o, many in zip((a, b), cs, outs, (False, True)):
        c.sync()
        ref, tol = s.expect(0.1, 0, many=many)
        assert torch.all((o.double() - ref).abs() <= tol)
        c.close()


def test_against_the_bf16_cache(ctx):
    """The same step over a bf16 cache that holds what the 4-bit one stands for: both near 64 bits."""
    s = Step([1, 1, 1], [512, 100, 333], 16, 4, 128, 16, seed=40)
    kp, vp = (torch.nan_to_num(x).bfloat16() for x in (s.k, s.v))
    desc = kf.PagedKV(At(kp), At(vp), s.n_pages, 16, 4, 128, At(s.d[0]), s.cols, 3, At(s.d[1]), At(s.d[2]))
    out = torch.zeros(3, 16 * 128, device="cuda", dtype=torch.bfloat16)
    kf.paged_attention(ctx, desc, At(s.q), 3, 16, max_q=1, out=At(out))
    got = s.attend(ctx, 128 ** -0.5)
    ctx.sync()
    ref, _ = s.expect(128 ** -0.5, 0)
    assert float((got.double() - ref).norm() / ref.norm()) < 1.1 * float((out.double() - ref).norm() / ref.norm())


# ---------------------------------------------------------------------------------------------------------------- limits
def test_nothing_to_do(ctx):
    """No rows at all, and rows that all are padding."""
    s = Step([1], [5], 2, 1, 64, 8, seed=1)
    out = torch.full((4, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(4, 128, device="cuda", dtype=torch.bfloat16)
    before = s.pool.clone()
    for M in (0, 4):
        kf.paged_attention_q4(ctx, s.desc, At(q), M, 2, max_q=1, out=At(out))
        kf.paged_append_q4(ctx, s.desc, None, At(q), At(q), At(q), M, 2, out=At(out))
        kf.paged_read_q4(ctx, s.desc, M, k_out=At(out))
        s.d[1][:] = 0
    torch.cuda.synchronize()
    assert torch.all(out == 7) and torch.equal(before, s.pool)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cta", [0, 70])
@pytest.mark.parametrize("chunk,fresh", [(256, False), (256, True), (2, False), (2, True)])
def test_wait_that_runs_out_among_many_pieces(hd, cta, chunk, fresh):
    """A thread block that loads nothing and whose run is longer than the queue of pieces: what the merge reads of it says that nothing goes on, whatever the workspace held.  The
    error is told, rows of nobody stay as they are, and the next call is right."""
    c = kf.Context(0, stream=torch.cuda.current_stream().cuda_stream or 1)
    r = np.random.RandomState(hd)
    length = r.randint(20, 121, 200).tolist() + [400]
    s = Step([1] * 200 + [chunk], length, 32, 8, hd, 16, seed=hd, extra=2, pad=3)
    other = Step([130] * 20, [400] * 20, 64, 1, 192 - hd, 16, seed=3)
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
def test_wait_that_runs_out_is_reported(new):
    """A thread block that loads nothing: the call ends, the next synchronisation says so, and the context works afterwards."""
    c = kf.Context(0, stream=torch.cuda.current_stream().cuda_stream or 1)
    s = Step(new, [400, 300], 8, 2, 128, 16, seed=50)
    s.check(c)
    for told_by in ("sync", "call"):
        c.set_int("attn_wait_us", 20000), c.set_int("attn_drop", 1)
        s.attend(c, 0.1)
        c.set_int("attn_drop", 0), c.set_int("attn_wait_us", 0)
        assert [c.get_int(k) for k in ("attn_tc_error", "attn_gqa_error", "attn_paged_error")] == [0, 0, 1]  # waits for the stream
        with pytest.raises(kf.KoifishError, match="wait ran out in the paged attention kernel"):
            c.sync() if told_by == "sync" else s.attend(c, 0.1)
        c.sync()
        s.check(c)
    c.close()


def test_results_over_their_sources(ctx):
    """A result that lies over a part of what it is made of, or keys over values, is refused."""
    s = Step([1, 3, 1], [30, 20, 9], 4, 2, 64, 16, seed=70)
    n = s.rows
    buf = torch.zeros(n + 4, 3 * 256, device="cuda", dtype=torch.bfloat16)
    buf[1:n + 1, :256] = s.q
    q, rows = buf[1:n + 1], buf.stride(0)
    for o, ld in [(q, rows), (buf[2:], rows), (buf[0:], rows), (q[:, 8:], rows), (buf.flatten()[rows - 256 + 8:], rows), (q, 256)]:
        with pytest.raises(kf.KoifishError, match="over"):
            s.attend(ctx, 0.1, q=q, ldq=rows, out=o, ldo=ld)
    for o in (q[:, 256:], q[:, 256 + 200:]):
        with pytest.raises(kf.KoifishError, match="over"):
            kf.paged_append_q4(ctx, s.desc, None, At(q), At(q[:, 256:]), At(q[:, 256 + 128:]), n, 4, ldq=rows, ldk=rows, ldv=rows, out=At(o), ldo=rows)
    with pytest.raises(kf.KoifishError, match="over"):
        kf.paged_read_q4(ctx, s.desc, n, k_out=At(q), v_out=At(q[:, 100:]), ldk=rows, ldv=rows)
    kf.paged_append_q4(ctx, s.desc, None, At(q), At(q[:, 256:]), At(q[:, 256 + 128:]), n, 4, ldq=rows, ldk=rows, ldv=rows, out=At(q), ldo=rows)  # in place
    torch.cuda.synchronize()
    assert torch.equal(q[:, :256], s.q)


def test_timed_calls_on_another_stream():
    """The calls of perf/more_operators.py go to the stream that is current, for a state of another stream as well, and give the same bits there."""
    import importlib.util
    import os
    spec = importlib.util.spec_from_file_location("more_timed_operators", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "more_operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True
    for name in ("append_decode", "attn_one", "read_short"):
        case = [c for c in ops.listed() if c["name"] == name][0]
        first, side = ops.prepare(case, 1), torch.cuda.Stream()
        flat = lambda x: [t.clone().view(torch.uint8) for t in (x if isinstance(x, tuple) else (x,))]  # noqa: E731
        want = flat(ops.run(first))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for s in (first, ops.prepare(case, 1)):
                got = flat(ops.run(s))
                c = s["handles"]["ctx"]
                assert c.lib.kf_ctx_stream(c.h) == side.cuda_stream
                side.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(want, got))
        torch.cuda.synchronize()


# ---------------------------------------------------------------------------------------------------------------- the ends of what is allowed, in every kernel
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads", [8, 96])
def test_long_sums_of_large_values(ctx, hd, heads):
    """Values just below 2^50 whose zeros are some 2000 steps away, over a long sequence whose scores grow by less than what sums are rescaled for: weights of up to 2^7.75, 4096 of them
    a warp.  Sequences that share their pages, more of them than there are teams of thread blocks, so that one block has a whole one."""
    n, kv = 16384, 8
    s = Step([1], [n], heads, kv, hd, 64, seed=heads)
    n_seq = 60
    t = torch.arange(n, device="cuda")
    e, r = torch.from_numpy(s.table[0]).cuda()[t // 64], t % 64
    codes, step, zero = read(s.pages, kv, hd, 64, 0, e, r)
    codes[:] = 0
    codes[128:, :, 0] = 5
    s.put(0, e, r, codes, torch.ones_like(step).bfloat16(), torch.zeros_like(zero).bfloat16())
    codes, step, zero = read(s.pages, kv, hd, 64, 1, e, r)
    s.put(1, e, r, codes, torch.full_like(step, 2.0 ** 39).bfloat16(), torch.full_like(zero, -2000.0).bfloat16())
    assert float(s.v.abs().max()) < 2.0 ** 50
    s.new, s.length, s.rows, s.table = [1] * n_seq, [n] * n_seq, n_seq, np.repeat(s.table, n_seq, 0)
    s.start = list(range(n_seq + 1))
    s.q = torch.zeros(n_seq, heads * hd, device="cuda", dtype=torch.bfloat16)
    s.q[:, ::hd] = 1
    s.d = [i32(np.where(s.table > 2 ** 31 - 1, 0, s.table)), i32(s.start), i32(s.length)]
    s.desc = s.describe()
    s.check(ctx, scale=7.75 / (5 * math.log2(math.e)))


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
def test_append_of_the_largest_ranges(ctx, src):
    """A group comes back within its bound as long as its range is a number of 32 bits; where the range is none it comes back as NaN, like one with an entry that is not finite."""
    r = np.random.RandomState(1)
    x = np.stack([1.69e38 * (2 * r.rand(32) - 1), np.r_[-1.69e38, 1.69e38, np.zeros(30)], 1e38 * (1 + 2 * r.rand(32)), np.r_[1.8e38, -1.8e38, np.zeros(30)]])
    x = torch.tensor(x, dtype=torch.float32).to(src).cuda()
    k = x.view(1, 128)
    s = Step([1], [50], 1, 1, 128, 16, seed=1)
    kf.paged_append_q4(ctx, s.desc, None, At(s.q if src == torch.bfloat16 else s.q.float()), At(k), At(k), 1, 1, out=At(torch.zeros_like(s.q)), src_f32=src == torch.float32)
    back = [torch.zeros(1, 128, device="cuda") for _ in "kv"]
    kf.paged_read_q4(ctx, s.desc, 1, k_out=At(back[0]), v_out=At(back[1]), out_f32=True)
    torch.cuda.synchronize()
    c, st, z = quantised(x[:3])
    for b in back:
        b = b.view(4, 32)
        assert torch.all((b[:3].double() - x[:3].double()).abs() <= wide(st).double() * (0.5 + wide(z.abs()).double() / 256 + 2 ** -20))
        assert torch.all(torch.isnan(b[3]))


# heads of a kv head and new tokens of three sequences: 8, 12, 16 and 96 rows of a sequence and kv head
ROWS = [(4, [1, 2, 1]), (6, [2, 1, 2]), (16, [1, 1, 1]), (24, [1, 4, 2])]


def regroup(s, value, change):
    """Steps and zeros of all cached rows of a Step by change(step, zero)."""
    for i, n in enumerate(s.length):
        t = torch.arange(n, device="cuda")
        e, r = torch.from_numpy(s.table[i]).cuda()[t // s.page], t % s.page
        codes, step, zero = read(s.pages, s.kv, s.hd, s.page, value, e, r)
        s.put(value, e, r, codes, *(x.bfloat16() for x in change(step, zero)))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group,new", ROWS)
def test_zeros_far_from_the_codes_in_every_kernel(ctx, hd, group, new):
    """Zeros of hundreds of steps of both signs, a group beside the next."""
    s = Step(new, [200, 60, 333], 2 * group, 2, hd, 16, seed=group + hd)
    far = lambda step, zero: (step / 16, torch.where(torch.arange(hd // 32, device="cuda") % 2 == 1, -600.0, 900.0).expand_as(zero) + 8 * (zero - 7))  # noqa: E731
    regroup(s, 0, far), regroup(s, 1, far)
    s.check(ctx)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("key,value", [(-45, -58), (-40, 40), (-20, -20), (20, 44), (44, -40)])
@pytest.mark.parametrize("group,new", ROWS)
def test_sizes_of_values_in_every_kernel(ctx, hd, key, value, group, new):
    """Steps from very small to very large, of keys against queries of the inverse size, and of values: entries of 2^-60 .. 2^50."""
    s = Step(new, [300, 77, 130], 2 * group, 2, hd, 16, seed=group + hd)
    regroup(s, 0, lambda step, zero: (step * 2.0 ** key, zero)), regroup(s, 1, lambda step, zero: (step * 2.0 ** value, zero))
    s.q = (s.q.float() * 2.0 ** -key).bfloat16()
    assert max(float(x.abs().max()) for x in (s.k, s.v, torch.nan_to_num(s.q.float()))) < 2.0 ** 50
    s.check(ctx)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("max_q", [None, 0, 40])
@pytest.mark.parametrize("group,new", ROWS)
def test_how_near_the_result_is(ctx, hd, group, new, max_q):
    """The roundings' errors are independent, so on the whole their squares add up.  Half a step of bf16 at most is 2^-8 / sqrt(3) = 2.26e-3 in the mean square where a number's bits are 1.0 ..,
    and 1 / sqrt(E m^2) of that, 1.5e-3 .. 1.7e-3, over numbers of all sizes.  Few rows: the result and weight times step, 2.3e-3.  Many rows: the result, weights and values, 1.7e-3 each, and
    keys, which change a score by 1.6e-3 of scale * sqrt(sum q^2 k^2) = 1.3 * 1.2 here, 2.5e-3: 3.9e-3.  Half as much again is allowed."""
    s = Step(new, [700, 1000, 333], 2 * group, 2, hd, 16, seed=group + hd)
    rows = max(max(new) if max_q is None else max_q, 1) * group
    out = s.attend(ctx, hd ** -0.5, max_q=max_q)
    ctx.sync()
    ref, _ = s.expect(hd ** -0.5, 0)
    assert float((out.double() - ref).norm() / ref.norm()) < (6e-3 if rows > 16 else 3.5e-3)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_seq,active,kv,past,few", [(33, 33, 2, 200, True), (40, 40, 4, 100, True), (1100, 60, 2, 250, True), (8192, 70, 2, 300, True), (200, 200, 4, 250, False), (8192, 300, 3, 300, False)])
@pytest.mark.parametrize("window,first", [(0, 0), (60, 5)])
def test_few_tiles_of_many_sequences(ctx, hd, n_seq, active, kv, past, few, window, first):
    """More than 32 sequences with up to four tiles a thread block and with more: chunks of one and of two row tiles, drafts, single tokens, idle slots between them."""
    r = np.random.RandomState(n_seq + active)
    new = np.zeros(n_seq, dtype=int)
    at = np.sort(r.choice(n_seq, active, replace=False))
    new[at] = r.choice([1, 1, 1, 5, 20, 33, 90], active)
    new[at[0]] = new[at[-1]] = 90
    length = new + r.randint(0, past if n_seq < 1000 else 30, n_seq)
    length[at] = new[at] + r.randint(0, past, active)
    tiles = sum(-(-(e - n + min(n, b + 64)) // 128) for n, e in zip(new.tolist(), length.tolist()) for b in range(0, n, 64)) * kv  # 64 tokens of 4 heads are two row tiles
    assert (tiles <= 4 * torch.cuda.get_device_properties(0).multi_processor_count) == few
    Step(new, length, 4 * kv, kv, hd, 16, seed=active, pad=1).check(ctx, window=window, first=first)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [[1, 1, 2], [1, 40, 3]])
def test_more_kv_heads_than_thread_blocks(ctx, hd, new):
    """300 kv heads: one team of thread blocks in the kernel for few rows, runs of several heads of a sequence in the other."""
    Step(new, [200, 77, 140], 300, 300, hd, 16, seed=hd).check(ctx)
    Step(new, [200, 77, 140], 900, 300, hd, 8, seed=hd + 1).check(ctx, window=50, first=3, max_q=40)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("max_q", [2, 3, 40])
def test_a_query_that_is_not_finite(ctx, hd, max_q):
    """It makes the result of its own row and head NaN and nobody else's."""
    s = Step([3, 1, 2], [90, 61, 20], 8, 2, hd, 16, seed=9)
    bad = torch.zeros(6, 8, device="cuda", dtype=torch.bool)
    for row, head in ((1, 2), (3, 7), (5, 0)):
        s.q[row, head * hd + 5 * row] = float("nan")
        bad[row, head] = True
    out = s.attend(ctx, hd ** -0.5, max_q=max_q)
    ctx.sync()
    ref, tol = s.expect(hd ** -0.5, 0, many=max_q * 4 > 16)
    off = (out.double() - ref).abs().view(6, 8, hd)
    assert torch.all(torch.isnan(off[bad])) and torch.all(off[~bad] <= tol.view(6, 8, hd)[~bad])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("max_q", [1, 2, 4])
def test_the_nearer_kernel_by_choice(ctx, hd, max_q):
    """With max_q for at most 16 rows of a sequence and kv head, drafts and chunks have the error of single tokens."""
    s = Step([1, 30, 5], [700, 1000, 333], 8, 2, hd, 16, seed=hd)
    out = s.attend(ctx, hd ** -0.5, max_q=max_q)
    ctx.sync()
    ref, _ = s.expect(hd ** -0.5, 0)
    assert float((out.double() - ref).norm() / ref.norm()) < 3.5e-3
