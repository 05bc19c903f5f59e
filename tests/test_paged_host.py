"""Host tests of the paged cache's entry points: refusals, and the arithmetic of blocks and tiles against a count of every position.  No device."""
import ctypes as C

import numpy as np
import pytest

import koifish_b200 as kf
from koifish_b200 import _lib as L

BAD = L.KF_ERR_BAD_ARG


@pytest.fixture(scope="module")
def lib():
    return kf.load()


def cache(**kw):
    d = dict(k_dev=1024, v_dev=2048, page_stride=0, n_pages=10, page_size=16, n_kv=2, head_dim=128, table_dev=64, table_cols=4, n_seq=3, q_start_dev=128, len_dev=192)
    d.update(kw)
    return L.PagedKVDesc(**d)


def rotation(**kw):
    d = dict(inv_freq_dev=64, rot_dims=128, layout=1, amp=1.0, n_axes=1, axis_dev=None, pos_dev=None, pos_stride=0)
    d.update(kw)
    return L.RotationDesc(**d)


BAD_CACHES = [dict(k_dev=None), dict(v_dev=None), dict(table_dev=None), dict(q_start_dev=None), dict(len_dev=None), dict(head_dim=96), dict(head_dim=0), dict(n_kv=0), dict(n_kv=1025),
              dict(n_pages=0), dict(page_size=0), dict(page_size=12), dict(page_size=-8), dict(table_cols=0), dict(table_cols=1 << 28), dict(n_seq=0), dict(n_seq=8193),
              dict(page_stride=4096 + 4), dict(page_stride=16 * 2 * 128 - 8), dict(k_dev=1026), dict(v_dev=2056)]


def attention(lib, c, out=4096, ldo=1024, q=8192, ldq=1024, M=5, n_head=8, scale=0.1, max_q=1):
    lib.kf_paged_attention_args.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_float, C.c_int]
    return lib.kf_paged_attention_args(C.byref(c) if c is not None else None, out, ldo, q, ldq, M, n_head, scale, max_q)


def append(lib, c, r, q_out=4096, ldqo=1024, q=8192, ldq=1024, k=16384, ldk=256, v=32768, ldv=256, src_f32=0, M=5, n_head=8):
    lib.kf_paged_append_args.argtypes = [C.c_void_p, C.c_void_p] + [C.c_void_p, C.c_int] * 4 + [C.c_int] * 3
    return lib.kf_paged_append_args(C.byref(c) if c is not None else None, C.byref(r) if r is not None else None, q_out, ldqo, q, ldq, k, ldk, v, ldv, src_f32, M, n_head)


def rope(lib, r, out=4096, ldo=1024, x=8192, ldx=1024, f32=0, M=5, n_head=8, hd=128):
    lib.kf_rope_axes_args.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p] + [C.c_int] * 5
    return lib.kf_rope_axes_args(C.byref(r) if r is not None else None, out, ldo, x, ldx, f32, M, n_head, hd)


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_caches_that_are_refused(lib, bad):
    assert attention(lib, cache()) == 0 and append(lib, cache(), rotation()) == 0
    assert attention(lib, cache(**bad)) == BAD
    assert append(lib, cache(**bad), None) == BAD


@pytest.mark.parametrize("bad", [dict(out=None), dict(q=None), dict(ldq=1016), dict(ldo=1023), dict(q=8200), dict(ldq=1028), dict(M=-1), dict(n_head=0), dict(n_head=7), dict(n_head=130),
                                 dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(max_q=-1), dict(out=8192), dict(M=2 ** 30)])
def test_attention_refusals(lib, bad):
    assert attention(lib, cache(), **bad) == BAD


def test_attention_limits(lib):
    assert attention(lib, None) == BAD
    assert attention(lib, cache(n_kv=1, n_seq=8192), n_head=64, ldq=64 * 128, ldo=64 * 128, M=0, max_q=0) == 0
    assert attention(lib, cache(page_stride=2 * 16 * 2 * 128, page_size=16), out=4097) == 0
    assert lib.kf_paged_attention(None, None, None, 0, None, 0, 0, 0, 1.0, 0, 0) == BAD


@pytest.mark.parametrize("bad", [dict(q_out=None), dict(q=None), dict(k=None), dict(v=None), dict(ldq=1023), dict(ldqo=1000), dict(ldk=255), dict(ldv=128), dict(src_f32=2), dict(M=-1),
                                 dict(n_head=0), dict(q_out=8192, src_f32=1), dict(q_out=8192, ldqo=2048)])
def test_append_refusals(lib, bad):
    assert append(lib, cache(), None, **bad) == BAD


@pytest.mark.parametrize("bad", [dict(rot_dims=-2), dict(rot_dims=7), dict(rot_dims=130), dict(layout=2), dict(layout=-1), dict(n_axes=0), dict(n_axes=9), dict(inv_freq_dev=None),
                                 dict(pos_stride=4, pos_dev=64)])
def test_rotations_that_are_refused(lib, bad):
    assert append(lib, cache(), rotation(**bad)) == BAD
    assert rope(lib, rotation(**dict(dict(pos_dev=64), **bad))) == BAD


def test_append_in_place(lib):
    assert append(lib, cache(), rotation(), q_out=8192) == 0
    assert append(lib, None, rotation()) == BAD
    assert lib.kf_paged_append(None, None, None, None, 0, None, 0, None, 0, None, 0, 0, 0, 0, None, None, 0.0) == BAD


@pytest.mark.parametrize("bad", [dict(out=None), dict(x=None), dict(ldx=1000), dict(ldo=1000), dict(f32=3), dict(M=-1), dict(n_head=0), dict(hd=257), dict(hd=1), dict(out=8192, ldo=2048)])
def test_rope_refusals(lib, bad):
    assert rope(lib, rotation(pos_dev=64)) == 0
    assert rope(lib, rotation(pos_dev=64), **bad) == BAD


def test_rope_needs_positions(lib):
    assert rope(lib, rotation()) == BAD and rope(lib, None) == BAD
    assert lib.kf_rope_axes(None, None, None, 0, None, 0, 0, 0, 0, 0) == BAD


def test_blocks(lib):
    """First and last position that the rows of a block see, and the tiles they touch, against a count of every (row, position) -- so that no look-up goes behind the last visible
    position or the table."""
    r = np.random.RandomState(0)
    got = (C.c_int * 3)()
    for _ in range(4000):
        tile, tb = int(r.choice([64, 128])), int(r.choice([1, 2, 3, 16, 36, 50, 256]))
        n, len_ = int(r.randint(1, 400)), int(r.choice([0, r.randint(0, 80), r.randint(0, 700)]))
        cap = int(r.choice([8, 64, 200, 800]))
        window = int(r.choice([0, 1, 5, 64, 300, 2 ** 31 - 1]))
        for b in range(-(-n // tb)):
            tiles = lib.kf_paged_attention_block(tile, cap, tb, window, n, len_, b, got)
            seen = set()
            for tok in range(b * tb, min(n, (b + 1) * tb)):
                p = len_ - n + tok
                seen |= set(range(max(0, p - window + 1) if window else 0, min(p + 1, cap)))
            if not seen:
                assert tiles == 1 and list(got) == [0, 0, 0]
                continue
            assert (got[0], got[1]) == (min(seen), max(seen) + 1) and got[1] <= cap
            assert got[2] == min(seen) // tile and tiles == max(seen) // tile - min(seen) // tile + 1


def test_page_of_a_position(lib):
    """The division by a page size as the kernels do it, up to the largest position."""
    r = np.random.RandomState(1)
    for page in [8, 16, 24, 40, 48, 56, 64, 120, 128, 136, 1000, 4096, 65528, 1 << 20, (1 << 20) + 8, (1 << 30) - 8, 1 << 30]:
        near = [k * page + d for k in [0, 1, 2, 3, (2 ** 31 - 1) // page] for d in (-1, 0, 1)]
        for p in near + r.randint(0, 2 ** 31 - 1, 200).tolist():
            if 0 <= p < 2 ** 31:
                assert lib.kf_paged_page_of(page, p) == p // page


@pytest.mark.parametrize("page", [(1 << 30) + 8, (1 << 30) + (1 << 29), 2 ** 31 - 264])
def test_largest_pages(lib, page):
    """Pages of more than 2^30 positions: accepted as one column of a table, and divided by."""
    assert attention(lib, cache(page_size=page, table_cols=1, n_kv=1), n_head=8) == 0 and append(lib, cache(page_size=page, table_cols=1), None) == 0
    assert attention(lib, cache(page_size=page, table_cols=2)) == BAD
    for p in [0, 1, 7, page // 2, page - 1, page, page + 1, 2 ** 31 - 1]:
        assert lib.kf_paged_page_of(page, p) == p // page


def test_rows_that_overlap(lib):
    """Panels in one buffer, side by side, interleaved and shifted, against a count of every byte."""
    lib.kf_rows_overlap.argtypes = [C.c_void_p, C.c_size_t, C.c_size_t] * 2 + [C.c_int]
    r = np.random.RandomState(2)
    base, seen = 1 << 20, [0, 0]
    for _ in range(6000):
        M, aw, bw = int(r.randint(1, 7)), int(r.randint(1, 9)), int(r.randint(1, 9))
        ap = aw + int(r.choice([0, 1, 5, 20]))
        bp = ap if r.rand() < 0.6 and bw <= ap else bw + int(r.choice([0, 2, 17]))
        d = int(r.randint(-60, 61))
        a, b = ({x for i in range(M) for x in range(at + i * p, at + i * p + w)} for at, p, w in ((0, ap, aw), (d, bp, bw)))
        assert lib.kf_rows_overlap(base, ap, aw, base + d, bp, bw, M) == int(bool(a & b)), (M, ap, aw, d, bp, bw)
        seen[bool(a & b)] += 1
    assert min(seen) > 1000
    assert lib.kf_rows_overlap(base, 8, 8, base, 8, 8, 0) == 0
    far = 1 << 40  # offsets of more than 32 bits
    assert lib.kf_rows_overlap(far, 1 << 20, 64, far + (1 << 34) + 32, 1 << 20, 64, 20000) == 1 and lib.kf_rows_overlap(far, 1 << 20, 64, far + (1 << 34) + 64, 1 << 20, 64, 20000) == 0


class Recorder:
    """Stands in for a context: remembers the arguments of the library's calls."""

    def __init__(self):
        self.h, self.lib, self.calls = None, self, []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


class Buf:
    def __init__(self, ptr):
        self.ptr = ptr


@pytest.mark.parametrize("same", [True, False])  # the panel's own object, or another one at its address
def test_in_place_rows_from_python(same):
    """In place, the rows of the result are those of the panel unless they are given."""
    c, q, b = Recorder(), Buf(4096), Buf(64)
    o = q if same else Buf(4096)
    kv = kf.PagedKV(b, b, 4, 16, 2, 128, b, 4, 1, b, b)
    rot = kf.Rotation(b, 128, pos=b)
    kf.paged_append(c, kv, rot, q, Buf(8192), Buf(9216), 3, 8, ldq=1536, ldk=1536, ldv=1536, out=o)
    kf.paged_append(c, kv, rot, q, Buf(8192), Buf(9216), 3, 8, ldq=1536, ldk=1536, ldv=1536, out=Buf(1 << 20))
    kf.paged_append(c, kv, rot, q, Buf(8192), Buf(9216), 3, 8, out=o)
    kf.rope_axes(c, rot, q, 3, 8, 128, ldx=1536, out=o)
    kf.rope_axes(c, rot, q, 3, 8, 128, ldx=1536, out=Buf(1 << 20))
    assert [a[4 if name == "kf_paged_append" else 3] for name, a in c.calls] == [1536, 1024, 1024, 1536, 1024]
