"""Host tests of the 4-bit paged cache's entry points: refusals, page sizes, and the arithmetic of blocks with first positions against a count of every position.  No device."""
import ctypes as C

import numpy as np
import pytest

import koifish_b200 as kf
from koifish_b200 import _lib as L
from test_paged_host import Buf, Recorder, rotation

BAD = L.KF_ERR_BAD_ARG


@pytest.fixture(scope="module")
def lib():
    return kf.load()


def cache(**kw):
    d = dict(pool_dev=1024, page_stride=0, n_pages=10, page_size=16, n_kv=2, head_dim=128, table_dev=64, table_cols=4, n_seq=3, q_start_dev=128, len_dev=192)
    d.update(kw)
    return L.PagedQ4Desc(**d)


PAGE = 16 * 2 * 160
BAD_CACHES = [dict(pool_dev=None), dict(table_dev=None), dict(q_start_dev=None), dict(len_dev=None), dict(head_dim=96), dict(head_dim=0), dict(n_kv=0), dict(n_kv=1025), dict(n_pages=0),
              dict(page_size=0), dict(page_size=12), dict(page_size=-8), dict(table_cols=0), dict(table_cols=1 << 28), dict(n_seq=0), dict(n_seq=8193), dict(page_stride=PAGE + 8),
              dict(page_stride=PAGE - 16), dict(page_stride=1 << 63), dict(pool_dev=1032)]


def attention(lib, c, out=4096, ldo=1024, q=1 << 20, ldq=1024, M=5, n_head=8, scale=0.1, first=0, max_q=1):
    lib.kf_paged_attention_q4_args.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_float, C.c_int, C.c_int]
    return lib.kf_paged_attention_q4_args(C.byref(c) if c is not None else None, out, ldo, q, ldq, M, n_head, scale, first, max_q)


def append(lib, c, r, q_out=4096, ldqo=1024, q=8192, ldq=1024, k=16384, ldk=256, v=32768, ldv=256, src_f32=0, M=5, n_head=8):
    lib.kf_paged_append_q4_args.argtypes = [C.c_void_p, C.c_void_p] + [C.c_void_p, C.c_int] * 4 + [C.c_int] * 3
    return lib.kf_paged_append_q4_args(C.byref(c) if c is not None else None, C.byref(r) if r is not None else None, q_out, ldqo, q, ldq, k, ldk, v, ldv, src_f32, M, n_head)


def read(lib, c, k=4096, ldk=256, v=1 << 20, ldv=256, f32=0, M=5):
    lib.kf_paged_read_q4_args.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_int, C.c_int]
    return lib.kf_paged_read_q4_args(C.byref(c) if c is not None else None, k, ldk, v, ldv, f32, M)


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_caches_that_are_refused(lib, bad):
    assert attention(lib, cache()) == 0 and append(lib, cache(), rotation()) == 0 and read(lib, cache()) == 0
    assert attention(lib, cache(**bad)) == BAD and append(lib, cache(**bad), None) == BAD and read(lib, cache(**bad)) == BAD


@pytest.mark.parametrize("bad", [dict(out=None), dict(q=None), dict(ldq=1016), dict(ldo=1023), dict(q=8200), dict(ldq=1028), dict(M=-1), dict(n_head=0), dict(n_head=7), dict(n_head=130),
                                 dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(scale=2.0 ** 21), dict(max_q=-1), dict(first=-1), dict(out=1 << 20),
                                 dict(M=2 ** 30), dict(out=4097), dict(out=(1 << 20) + 16)])
def test_attention_refusals(lib, bad):
    assert attention(lib, cache(), **bad) == BAD


@pytest.mark.parametrize("bad", [dict(q_out=None), dict(q=None), dict(k=None), dict(v=None), dict(ldq=1023), dict(ldqo=1000), dict(ldk=255), dict(ldv=128), dict(src_f32=2), dict(M=-1),
                                 dict(n_head=0), dict(q_out=8192, src_f32=1), dict(q_out=8192, ldqo=2048)])
def test_append_refusals(lib, bad):
    assert append(lib, cache(), None, **bad) == BAD


@pytest.mark.parametrize("bad", [dict(rot_dims=-2), dict(rot_dims=7), dict(rot_dims=130), dict(layout=2), dict(n_axes=0), dict(n_axes=9), dict(inv_freq_dev=None), dict(pos_stride=4, pos_dev=64)])
def test_rotations_that_are_refused(lib, bad):
    assert append(lib, cache(), rotation(**bad)) == BAD


@pytest.mark.parametrize("bad", [dict(k=None, v=None), dict(ldk=255), dict(ldv=0), dict(f32=2), dict(f32=-1), dict(M=-1), dict(k=4097), dict(v=4098, f32=1), dict(v=4096), dict(v=4096 + 256), dict(k=(1 << 20) + 1536)])
def test_read_refusals(lib, bad):
    assert read(lib, cache(), **bad) == BAD


def test_read_limits(lib):
    assert read(lib, cache(), k=None) == 0 and read(lib, cache(), v=None, ldv=0) == 0 and read(lib, cache(), M=0) == 0
    assert read(lib, cache(), k=4096, v=4096 + 512, ldk=512, ldv=512) == 0 and read(lib, cache(), k=4096, v=4096 + 510, ldk=512, ldv=512) == BAD
    assert read(lib, None) == BAD and attention(lib, None) == BAD and append(lib, None, None) == BAD
    assert attention(lib, cache(n_kv=1, n_seq=8192), n_head=64, ldq=64 * 128, ldo=64 * 128, M=0, max_q=0, first=2 ** 31 - 1) == 0
    assert lib.kf_paged_attention_q4(None, None, None, 0, None, 0, 0, 0, 1.0, 0, 0, 0) == BAD
    assert lib.kf_paged_read_q4(None, None, None, 0, None, 0, 0, 0) == BAD
    assert lib.kf_paged_append_q4(None, None, None, None, 0, None, 0, None, 0, None, 0, 0, 0, 0, None, None, 0.0) == BAD


def test_page_bytes(lib):
    assert kf.PagedQ4.page_bytes(16, 8, 128) == 16 * 8 * 160 and kf.PagedQ4.page_bytes(8, 1, 64) == 8 * 80
    assert kf.PagedQ4.page_bytes(1 << 20, 1024, 128) == (1 << 30) * 160
    assert [kf.PagedQ4.page_bytes(*a) for a in ((12, 1, 64), (0, 1, 64), (8, 0, 64), (8, 1, 96), (-8, 1, 64))] == [0] * 5


def test_blocks_with_first_positions(lib):
    """Positions that the rows of a block see and the tiles they touch, in order, against a count of every (row, position)."""
    r = np.random.RandomState(0)
    got = (C.c_int * 4)()
    kinds = set()
    for _ in range(6000):
        tile, tb = int(r.choice([64, 96, 128])), int(r.choice([1, 2, 3, 16, 36, 50, 256]))
        n, len_ = int(r.randint(1, 400)), int(r.choice([0, r.randint(0, 80), r.randint(0, 900)]))
        cap = int(r.choice([8, 64, 200, 1000]))
        window, first = int(r.choice([0, 1, 5, 64, 300, 2 ** 31 - 1])), int(r.choice([0, 1, 4, 64, 100, 2 ** 31 - 1]))
        for b in range(-(-n // tb)):
            tiles = lib.kf_paged_attention_block_first(tile, cap, tb, window, first, n, len_, b, got)
            lo, hi, kt0, ns = got
            seen = set()
            for tok in range(b * tb, min(n, (b + 1) * tb)):
                p = len_ - n + tok
                seen |= set(j for j in range(max(0, min(p + 1, cap))) if not window or j > p - window or j < first)
            if not seen:
                assert tiles == 1 and list(got) == [0, 0, 0, 0]
                continue
            listed = [t if t >= kt0 else t - kt0 + ns for t in range(kt0 - ns, kt0 - ns + tiles)]
            assert listed == sorted(set(j // tile for j in seen))
            fs = first if lo > 0 else 0
            assert seen == set(j for j in range(hi) if j >= lo or j < fs)
            kinds.add((ns > 0, lo > 0, first > 0))
    assert len(kinds) >= 5


def test_calls_from_python():
    """Rows are dense unless their distances are given; in place, the rows of the result are those of the panel."""
    c, q, b = Recorder(), Buf(4096), Buf(64)
    kv = kf.PagedQ4(b, 4, 16, 2, 128, b, 4, 1, b, b)
    rot = kf.Rotation(b, 128, pos=b)
    kf.paged_append_q4(c, kv, rot, q, Buf(8192), Buf(9216), 3, 8, ldq=1536, ldk=1536, ldv=1536, out=q)
    kf.paged_append_q4(c, kv, rot, q, Buf(8192), Buf(9216), 3, 8, out=Buf(1 << 20))
    kf.paged_read_q4(c, kv, 3, k_out=b)
    kf.paged_read_q4(c, kv, 3, v_out=b, ldv=300, out_f32=True)
    kf.paged_attention_q4(c, kv, q, 3, 8, max_q=2, window=10, first=4, out=b)
    names = [n for n, _ in c.calls]
    assert names == ["kf_paged_append_q4"] * 2 + ["kf_paged_read_q4"] * 2 + ["kf_paged_attention_q4"]
    assert [a[4] for _, a in c.calls[:2]] == [1536, 1024]
    assert c.calls[2][1][2:] == (64, 256, None, 256, 0, 3) and c.calls[3][1][2:] == (None, 256, 64, 300, 1, 3)
    assert c.calls[4][1][2:] == (64, 1024, 4096, 1024, 3, 8, 128 ** -0.5, 10, 4, 2)
