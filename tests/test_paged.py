"""The arithmetic of the paged cache on what its tables say, compiled for the host, and the refusals of the 8-bit serving operators that need no GPU."""
import ctypes as C
import subprocess

import numpy as np
import pytest

import serve8 as S
import tile_share
from blok_amd.lib import KxFp8Args, KxPagedCache, KxPagedConfig, KxPagedRows, kx


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    exe = tile_share.build(tmp_path_factory.mktemp("paged"), "paged_place")

    def ask(lines):
        out = subprocess.run([exe], input="\n".join(lines), capture_output=True, text=True, timeout=60, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return ask


def test_rows_stay_inside_whatever_the_tables_hold(ask):
    big = 2 ** 31 - 1
    values = [-big - 1, -1, 0, 1, 5, 63, 64, 65, 1000, big]
    cases = [(a, b, p, t, cap) for a in values for b in values for p in values for t in (0, 5, 64, 1000) for cap in (64, 1024, big - 63)]
    for (a, b, p, t, cap), (first, n, pos, fault, units) in zip(cases, ask(["r %d %d %d %d %d" % c for c in cases])):
        assert 0 <= first and 0 <= n and first + n <= max(t, first)
        good_rows = 0 <= a <= b <= t
        good = good_rows and (a == b or 0 <= p <= cap - (b - a))
        assert fault == (0 if good else 2 if good_rows else 4)
        if good:
            assert (first, n) == (a, b - a)
        if n:
            assert pos == p and 0 <= pos and pos + n <= cap and units == (pos + n - 1) // 64 - pos // 64 + 1
        else:
            assert units == 0


def test_pages_outside_the_cache_are_seen(ask):
    cases = [(i, n) for i in (-2 ** 31, -1, 0, 1, 6, 7, 8, 2 ** 31 - 1) for n in (1, 7)]
    assert [a for a, in ask(["g %d %d" % c for c in cases])] == [int(0 <= i < n) for i, n in cases]


def test_places_of_values(ask):
    got = ask(["p %d" % t for t in range(64)])
    assert [token for _, token in got] == S.ORDER
    assert all(S.ORDER[place] == t for t, (place, _) in enumerate(got))


def test_exponents_of_scales(ask):
    xs = [0.0, 2.0 ** -149, 2.0 ** -126, 1e-35, 448 * 2.0 ** -101, 448 * 2.0 ** -100, 449 * 2.0 ** -100, 1.0, 1.75, np.nextafter(np.float32(1.75), np.float32(2)), 447.9, 448.0, 448.1, 3.4e38]
    xs += list(np.random.default_rng(0).standard_normal(200) ** 9)
    xs = [float(np.float32(abs(x))) for x in xs]
    assert [e for e, _ in ask(["e " + x.hex() for x in xs])] == list(S.exponent(xs))
    assert all(a == b for a, b in ask(["e " + x.hex() for x in xs]))


def test_widths(ask):
    cases = [(1, 1), (64, 64), (64, 65), (65, 1), (128, 128), (129, 64), (192, 128), (192, 129), (193, 1), (256, 256), (257, 1), (1, 257)]
    want = [(64, 64), (64, 64), (128, 128), (128, 128), (128, 128), (192, 128), (192, 128), (256, 256), (256, 256), (256, 256), (0, 0), (0, 0)]
    assert ask(["w %d %d" % c for c in cases]) == want


GOOD = dict(heads=4, kv_heads=2, dim=64, vdim=64, page=64, block=32, rot=64, pairs=0, size=0, scale=0.125, base=10000.0)


@pytest.mark.parametrize("bad", [dict(heads=0), dict(heads=3), dict(kv_heads=0), dict(kv_heads=-1), dict(dim=0), dict(dim=257), dict(vdim=0), dict(vdim=257), dict(page=0), dict(page=32), dict(page=96),
                                 dict(block=8), dict(block=128), dict(block=48), dict(rot=-2), dict(rot=3), dict(rot=66), dict(pairs=2), dict(size=-1), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(base=0.0), dict(base=-1.0), dict(base=float("nan"))])
def test_paged_create_refuses(bad):
    lib, h = kx(), C.c_void_p(5)
    assert lib.kx_paged_create(C.byref(KxPagedConfig(**{**GOOD, **bad})), None, 0, 1, 1, C.byref(h)) != 0
    assert h.value is None and b"kx_paged_create" in lib.kx_last_error()


def test_paged_create_refuses_sizes_and_null():
    lib, h, c = kx(), C.c_void_p(), KxPagedConfig(**GOOD)
    for batch, tokens in ((0, 1), (1, 0), (-1, 1), (1, -1), (1, 2 ** 31 - 1), (2 ** 31 - 1, 1)):
        assert lib.kx_paged_create(C.byref(c), None, 0, batch, tokens, C.byref(h)) != 0
    assert lib.kx_paged_create(None, None, 0, 1, 1, C.byref(h)) != 0 and lib.kx_paged_create(C.byref(c), None, 0, 1, 1, None) != 0
    freq = np.array([1.0, np.inf] * 16)
    assert lib.kx_paged_create(C.byref(c), freq.ctypes.data, 0, 1, 1, C.byref(h)) != 0 and b"frequency 1" in lib.kx_last_error()


def test_calls_without_a_handle_are_refused():
    lib, c, r, n = kx(), KxPagedCache(), KxPagedRows(), C.c_int32()
    assert lib.kx_paged_append(None, C.byref(c), C.byref(r), None, 0, 0, 0, None) != 0
    assert lib.kx_paged_attend(None, C.byref(c), C.byref(r), None, 0, 0, None, 0, None) != 0
    assert lib.kx_paged_read(None, C.byref(c), C.byref(r), None, 0, None, 0, None) != 0
    assert lib.kx_paged_faults(None, C.byref(n), None) != 0
    assert lib.kx_paged_destroy(None) == 0 and lib.kx_fp8_destroy(None) == 0
    assert lib.kx_fp8_run(None, C.byref(KxFp8Args()), None) != 0
    h = C.c_void_p()
    for tokens, cols in ((0, 1), (1, 0), (-1, 1), (1, -1), (2 ** 31 - 1, 1), (1, 2 ** 17 + 1), (1, 2 ** 31 - 1)):
        assert lib.kx_fp8_create(tokens, cols, C.byref(h)) != 0
    assert lib.kx_fp8_create(1, 1, None) != 0


def test_plain_codes():
    """The plain form's own rounding: every code is itself, and what lies between two goes to the nearer, ties to the even one."""
    v = S.VALUES[:127]
    assert (S.rounded(v) == v).all() and (S.codes(v) == np.arange(127)).all() and (S.codes(-v) == np.arange(127) + 128).all()
    mid = (v[:-1] + v[1:]) / 2
    assert (S.codes(S.rounded(mid)) == np.where(np.arange(126) % 2, np.arange(126) + 1, np.arange(126))).all()
    assert (S.rounded(np.nextafter(mid, 1e9)) == v[1:]).all() and (S.rounded(np.nextafter(mid, -1e9)) == v[:-1]).all()
