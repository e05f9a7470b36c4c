"""Forms of the 8-bit serving operators that a call takes by sizes and strides alone: results whose rows are whole pieces, and parts that the last workgroup in adds up, in both forms of the hand-over."""
import ctypes as C
import os

import numpy as np
import pytest

import serve8 as S
from blok_amd.lib import DevBuf, KxFp8Args, KxPagedConfig, check, load_library
from kxt import say
from test_gpu_fp8 import handle, rows_of
from test_gpu_fp8 import near as product_near
from test_gpu_serve8_weights import attend, expect, near

pytestmark = pytest.mark.gpu

FORMATS = pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])


@pytest.fixture(scope="module")
def strict(pytestconfig):
    """The library whose workgroups hand over in the form of the memory model."""
    return load_library(os.path.join(str(pytestconfig.rootpath), "blok_amd", "libkx_strict.so"))


@FORMATS
@pytest.mark.parametrize("dim,vdim", [(64, 64), (80, 80), (96, 96), (128, 128), (192, 128), (256, 256), (64, 60)])
def test_results_in_whole_pieces(kxlib, dim, vdim, f32):
    """Rows of results that begin at multiples of four elements and rows that do not hold the same bits, from one part and from several; nothing beside them is written."""
    say(f"pieces of {dim} / {vdim} f32={f32}")
    lens = [700, 1, 65]
    p = S.Paged(kxlib, heads=6, kv=2, dim=dim, vdim=vdim, rot=dim // 2, block=64, batch=3, f32=f32, tokens=1000, pages=20)
    p.append(lens, [0] * 3)
    for new in ([1, 1, 1], [6, 0, 9], [60, 1, 30]):
        pos, q = [n - m for n, m in zip(lens, new)], p.queries(sum(new))
        want = expect(p, new, pos, q)
        for longest in (1, 700):
            held = [attend(p, new, pos, q, longest, pad=pad) for pad in (0, 4, 3)]
            near(held[0], want, f"{new} longest {longest}")
            for other in held[1:]:
                np.testing.assert_array_equal(other, held[0])
    p.close()


@FORMATS
@pytest.mark.parametrize("heads,kv,new", [(8, 1, [1, 1]), (8, 1, [5, 5]), (4, 2, [39, 35])], ids=str)
def test_parts_of_an_attention_in_both_forms_of_handing_over(kxlib, strict, heads, kv, new, f32):
    """Few columns, several blocks of them, and columns that waves have for themselves: the same bits again and again."""
    say(f"attention of {new} rows, {heads} heads, f32={f32}")
    lens = [4000, 900]
    p = S.Paged(kxlib, heads=heads, kv=kv, dim=128, vdim=128, block=64, batch=2, f32=f32, tokens=5000, pages=80)
    p.append(lens, [0, 0])
    pos, q = [n - m for n, m in zip(lens, new)], p.queries(sum(new))
    first = attend(p, new, pos, q)
    near(first, expect(p, new, pos, q))
    for lib in (None, strict, None, strict, strict):
        np.testing.assert_array_equal(attend(p, new, pos, q, lib=lib), first)
    p.close()


@pytest.mark.parametrize("out_f32", [False, True])
@pytest.mark.parametrize("tokens,rows,cols", [(40, 24, 33000), (20, 130, 24000), (64, 70, 9000), (70, 300, 9000), (333, 300, 4000)])
def test_parts_of_a_product_in_both_forms_of_handing_over(kxlib, strict, tokens, rows, cols, out_f32):
    """Parts of the columns, of up to 64 tokens and of tiles: the same bits again and again."""
    say(f"product {tokens} x {rows} x {cols} out_f32={out_f32}")
    rng = np.random.default_rng(tokens)
    c, s, w = S.matrix(rng, rows, cols)
    h, x = handle(kxlib, tokens, cols), rows_of(rng, tokens, cols, False)
    first = S.product(kxlib, h, c, s, x, cols, out_f32, False)
    product_near(first, S.row_codes(x), w, out_f32)
    for lib in (kxlib, strict, kxlib, strict, strict):
        np.testing.assert_array_equal(S.product(lib, h, c, s, x, cols, out_f32, False), first)
    check(kxlib.kx_fp8_destroy(h))


def test_products_of_too_many_rows_are_refused(kxlib):
    """Shares of the rows are worked out in 32 bits, which 2^26 rows and 256 workgroups pass."""
    say("too many rows")
    h, d = handle(kxlib, 4, 128), DevBuf(1 << 20)
    for rows in ((1 << 25) + 1, 1 << 26, 2 ** 31 - 1):
        for tokens in (0, 1, 4):
            a = KxFp8Args(x_f32=0, out_f32=0, tokens=tokens, rows=rows, cols=128, ld=128, x_ld=128, out_ld=rows, d_w=d.ptr, d_w_scale=d.ptr, d_x=d.ptr, d_out=d.ptr)
            assert kxlib.kx_fp8_run(h, C.byref(a), None) != 0 and b"kx_fp8_run: rows" in kxlib.kx_last_error()
    check(kxlib.kx_fp8_destroy(h))


def test_products_whose_scales_do_not_fit_beside_a_share(kxlib):
    """As many rows as there may be: the scales of a workgroup's rows are more than its LDS holds, so that the product is worked out in blocks of rows.  Some rows are looked at."""
    say("scales beside a share")
    tokens, rows, cols, ld = 5, 1 << 25, 1100, 1152
    rng = np.random.default_rng(12)
    d, at = DevBuf(rows * ld), [0, 1 << 24, rows - 128]              # 39 GB, of which these three bands of 128 rows are set
    scales = np.full((rows // 128, 9), np.nan, np.float32)
    w = []
    for a in at:
        c, s, x = S.matrix(rng, 128, cols)
        check(kxlib.kx_h2d(d.ptr + a * ld, c.ctypes.data, c.nbytes))
        scales[a // 128] = s
        w.append(x)
    x, ds = rows_of(rng, tokens, cols, True), DevBuf.from_numpy(scales)
    dx, out, h = DevBuf.from_numpy(x), DevBuf(tokens * rows * 4), handle(kxlib, tokens, cols)
    a = KxFp8Args(x_f32=1, out_f32=1, tokens=tokens, rows=rows, cols=cols, ld=ld, x_ld=cols, out_ld=rows, d_w=d.ptr, d_w_scale=ds.ptr, d_x=dx.ptr, d_out=out.ptr)
    check(kxlib.kx_fp8_run(h, C.byref(a), None))
    check(kxlib.kx_sync(None))
    for first, m in zip(at, w):
        got = np.stack([out.to_numpy(np.float32, (128,), (t * rows + first) * 4) for t in range(tokens)])
        product_near(got.astype(np.float64), S.row_codes(x), m, True)
    check(kxlib.kx_fp8_destroy(h))


@FORMATS
def test_caches_of_more_than_four_gigabytes(kxlib, f32):
    """Pages whose places, and places of scales, pass 32 bits; what the memory held before is of no account."""
    say(f"large cache f32={f32}")
    pages, page, kv, dim = 36, 1 << 20, 2, 64
    p = S.Paged(kxlib, heads=4, kv=kv, dim=dim, vdim=dim, rot=dim, block=16, batch=3, f32=f32, tokens=800)
    check(kxlib.kx_paged_destroy(p.h))
    p.page, p.pages, p.h = page, pages, C.c_void_p()
    cfg = KxPagedConfig(4, kv, dim, dim, page, 16, dim, 0, 0, p.scale, 10000.0)
    check(kxlib.kx_paged_create(C.byref(cfg), None, int(f32), 3, 800, C.byref(p.h)))
    p.dk, p.dv = DevBuf(pages * kv * page * dim), DevBuf(pages * kv * page * dim)      # 4.8 GB each
    p.dks, p.dvs = DevBuf(pages * kv * page // 16 * 4), DevBuf(pages * kv * page // 16 * 4)
    p.free = [0, 17, pages - 1]
    lens = [300, 65, 120]
    p.append(lens, [0] * 3)
    for b, (k, v) in enumerate(p.read(lens, [0] * 3)):
        np.testing.assert_array_equal(k, p.k[b])
        np.testing.assert_array_equal(v, p.v[b])
    for new in ([1, 1, 1], [70, 3, 90]):
        pos, q = [n - m for n, m in zip(lens, new)], p.queries(sum(new))
        near(attend(p, new, pos, q), expect(p, new, pos, q))
    assert p.faults() == 0
    p.close()
