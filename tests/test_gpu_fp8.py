"""Products with 8-bit matrices (kx_fp8_run) on the GPU against the plain form in 64 bits, element by element."""
import ctypes as C

import numpy as np
import pytest

import serve8 as S
from blok_amd.lib import DevBuf, KxFp8Args, check
from kxt import say

pytestmark = pytest.mark.gpu


def handle(lib, tokens, cols):
    h = C.c_void_p()
    check(lib.kx_fp8_create(tokens, cols, C.byref(h)))
    return h


def rows_of(rng, tokens, cols, x_f32):
    x = (rng.standard_normal((tokens, cols)) * np.exp(rng.standard_normal((tokens, 1)))).astype(np.float32)
    if not x_f32:
        x = ((x.view(np.uint32) >> 16) << 16).view(np.float32)
    return x


def near(got, q, w, out_f32):
    y = q @ w.T
    over = np.abs(got - y) / S.product_tolerance(q, w, y, out_f32)
    print(f"  off by {over.max():.3f} of the tolerance", flush=True)
    assert (over <= 1).all(), f"{(over > 1).sum()} of {over.size}, {over.max():.2f} times the tolerance at {np.unravel_index(over.argmax(), over.shape)}"


@pytest.mark.parametrize("x_f32,out_f32", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 128), (17, 127), (200, 300), (130, 1100), (64, 2048)])
def test_products(kxlib, rows, cols, x_f32, out_f32):
    rng = np.random.default_rng(rows * 1000 + cols)
    c, s, w = S.matrix(rng, rows, cols, ld=-(-cols // 128) * 128 + 128)
    h = handle(kxlib, 300, cols + 200)
    for tokens in (1, 2, 5, 16, 17, 33, 64, 65, 129, 300):
        say(f"product {tokens} x {rows} x {cols} x_f32={x_f32} out_f32={out_f32}")
        x = rows_of(rng, tokens, cols, x_f32)
        near(S.product(kxlib, h, c, s, x, cols, out_f32, x_f32), S.row_codes(x), w, out_f32)
    check(kxlib.kx_fp8_destroy(h))


@pytest.mark.parametrize("tokens,rows,cols", [(512, 640, 1024), (513, 385, 900), (1000, 257, 4000)])
@pytest.mark.parametrize("out_f32", [False, True])
def test_large_products(kxlib, tokens, rows, cols, out_f32):
    say(f"large {tokens} x {rows} x {cols} out_f32={out_f32}")
    rng = np.random.default_rng(tokens)
    c, s, w = S.matrix(rng, rows, cols)
    h = handle(kxlib, tokens, cols)
    x = rows_of(rng, tokens, cols, False)
    near(S.product(kxlib, h, c, s, x, cols, out_f32, False), S.row_codes(x), w, out_f32)
    check(kxlib.kx_fp8_destroy(h))


@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 7, 20, 40, 70])
def test_long_rows_and_many_rows(kxlib, tokens):
    """More blocks of columns than lie in LDS at once, shares of rows that begin inside a band of 128, and parts of the columns."""
    rng = np.random.default_rng(tokens)
    for rows, cols in ((24, 33000), (130, 9000), (8300, 500), (33000, 130)):
        say(f"long {tokens} x {rows} x {cols}")
        c, s, w = S.matrix(rng, rows, cols)
        h = handle(kxlib, tokens, cols)
        x = rows_of(rng, tokens, cols, False)
        for out_f32 in (False, True):
            near(S.product(kxlib, h, c, s, x, cols, out_f32, False), S.row_codes(x), w, out_f32)
        check(kxlib.kx_fp8_destroy(h))


def test_rows_of_every_size(kxlib):
    """Magnitudes from the smallest to the largest float, blocks of zeros, and what is not finite."""
    rng = np.random.default_rng(9)
    c, s, w = S.matrix(rng, 40, 640)
    s[:] = 1.0
    w = S.VALUES[c].astype(np.float64)
    h = handle(kxlib, 64, 640)
    x = rows_of(rng, 40, 640, True)
    x[1, :128] = 0.0
    x[2] *= np.float32(1e-30)
    x[3] *= np.float32(1e-37)
    x[4] = 0.0
    x[5, 128:256] *= np.float32(1e20)
    x[6, 5], x[7, 200], x[8, 639] = np.nan, np.inf, -np.inf
    x[9, 0] = 448.0
    x[10, 0] = np.nextafter(np.float32(448.0), np.float32(1e9))
    for tokens in (12, 40):
        for out_f32 in (True, False):
            say(f"sizes {tokens} out_f32={out_f32}")
            got = S.product(kxlib, h, c, s, x[:tokens], 640, out_f32, True)
            bad = np.zeros(tokens, bool)
            bad[6:9] = True
            assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
            near(got[~bad], S.row_codes(x[:tokens][~bad]), w, out_f32)
    check(kxlib.kx_fp8_destroy(h))


def test_nan_of_the_matrix_reaches_its_row_alone(kxlib):
    say("NaN in the matrix")
    rng = np.random.default_rng(10)
    c, s, w = S.matrix(rng, 70, 256)
    c[33, 100] = 0x7f
    h = handle(kxlib, 64, 256)
    for tokens in (3, 64):
        x = rows_of(rng, tokens, 256, False)
        got = S.product(kxlib, h, c, s, x, 256, False, False)
        assert np.isnan(got[:, 33]).all() and np.isfinite(np.delete(got, 33, 1)).all()
    check(kxlib.kx_fp8_destroy(h))


def test_rows_behind_the_last_token_stay(kxlib):
    say("rows behind")
    rng = np.random.default_rng(11)
    c, s, w = S.matrix(rng, 50, 256)
    h = handle(kxlib, 300, 256)
    for out_f32 in (False, True):
        for tokens, more in ((1, 3), (20, 20), (260, 7)):
            x = rows_of(rng, tokens + more, 256, False)
            got = S.product(kxlib, h, c, s, x, 256, out_f32, False, tokens=tokens)
            near(got, S.row_codes(x[:tokens]), w, out_f32)
    check(kxlib.kx_fp8_destroy(h))


def test_refusals(kxlib):
    say("refusals")
    h, d = handle(kxlib, 4, 200), DevBuf(1 << 20)
    good = dict(x_f32=0, out_f32=0, tokens=4, rows=10, cols=200, ld=256, x_ld=200, out_ld=10, d_w=d.ptr, d_w_scale=d.ptr, d_x=d.ptr, d_out=d.ptr)
    for bad in (dict(tokens=-1), dict(tokens=5), dict(rows=0), dict(rows=-1), dict(cols=0), dict(cols=257), dict(ld=200), dict(ld=128), dict(ld=320 + 1), dict(x_ld=199), dict(out_ld=9), dict(d_w=None),
                dict(d_w_scale=None), dict(d_x=None), dict(d_out=None), dict(d_w=d.ptr + 8), dict(d_w_scale=d.ptr + 2), dict(d_x=d.ptr + 1), dict(d_out=d.ptr + 1), dict(x_f32=1, d_x=d.ptr + 2),
                dict(out_f32=1, d_out=d.ptr + 2)):
        assert kxlib.kx_fp8_run(h, C.byref(KxFp8Args(**{**good, **bad})), None) != 0, bad
        assert b"kx_fp8_run" in kxlib.kx_last_error()
    assert kxlib.kx_fp8_run(h, C.byref(KxFp8Args(**{**good, "tokens": 0})), None) == 0
    check(kxlib.kx_fp8_destroy(h))
