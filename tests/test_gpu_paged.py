"""The paged 8-bit cache on the GPU against plain forms in 64 bits: what appending leaves, and attention over it, element by element."""
import ctypes as C

import numpy as np
import pytest

import serve8 as S
from blok_amd.lib import DevBuf, KxPagedRows, check, load_library
from kxt import say

pytestmark = pytest.mark.gpu


def same(p, n, pos):
    for b, (k, v) in enumerate(p.read(n, pos)):
        if n[b]:
            np.testing.assert_array_equal(k, p.k[b][pos[b]:pos[b] + n[b]])
            np.testing.assert_array_equal(v, p.v[b][pos[b]:pos[b] + n[b]])


def near(got, want):
    y, tol = want
    assert got.shape == y.shape
    over = np.abs(got - y) / np.maximum(tol, 1e-300)
    print(f"  off by {np.nanmax(over):.3f} of the tolerance", flush=True)
    assert (over <= 1).all(), f"{(over > 1).sum()} of {over.size} off, {over.max():.3f} times the tolerance, at {np.unravel_index(over.argmax(), over.shape)}"


SHAPES = [dict(dim=128, vdim=128, rot=128), dict(dim=64, vdim=64, rot=32, pairs=1), dict(dim=80, vdim=72, rot=80, block=16), dict(dim=33, vdim=7, rot=32, pairs=1, block=64),
          dict(dim=192, vdim=128, rot=64, page=128, block=64), dict(dim=256, vdim=256, rot=0, block=16), dict(dim=130, vdim=1, rot=2, page=192)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s.values())))
def test_append_leaves_the_plain_cache(kxlib, shape):
    say(f"append {shape}")
    p = S.Paged(kxlib, heads=3, kv=3, batch=4, **shape)
    for new in ([70, 1, 0, 64], [1, 63, 5, 1], [1, 1, 1, 1], [130, 2, 60, 0]):
        pos = [len(k) for k in p.k]
        p.append(new, pos, tokens=sum(new) + 3)
        n = [len(k) for k in p.k]
        same(p, n, [0] * 4)
    assert p.faults() == 0
    p.close()


@pytest.mark.parametrize("block", [16, 32, 64])
def test_tokens_one_by_one_and_scales_that_grow(kxlib, block):
    say(f"one by one, blocks of {block}")
    p = S.Paged(kxlib, heads=2, kv=2, dim=64, vdim=64, block=block, batch=2)
    for i in range(80):   # magnitudes from 1e-6 to 1e6 in an order that makes scales grow in the middle of blocks, by a little and by a lot
        sigma = 10.0 ** (((i * 7) % 13) - 6)
        p.append([1, 1], [i, i], sigma=sigma)
        if i % 16 in (3, 15) or i > 75:
            same(p, [i + 1, i + 1], [0, 0])
    p.close()


def test_append_in_pieces_is_append_at_once_where_scales_do_not_grow(kxlib):
    say("pieces")
    k = np.random.default_rng(3).uniform(-1, 1, (150, 2, 64)).astype(np.float32)
    k[0:150:16] = np.sign(k[0:150:16])   # the first token of every block has the largest magnitude
    held = []
    for cuts in ([150], [1, 1, 14, 30, 2, 64, 38], [64, 64, 22]):
        p = S.Paged(kxlib, heads=2, kv=2, dim=64, vdim=64, block=16)
        at = 0
        for c in cuts:
            p.append([c], [at], k=k[at:at + c], v=k[at:at + c])
            at += c
        same(p, [150], [0])
        held.append(p.read([150], [0])[0])
        p.close()
    for k1, v1 in held[1:]:
        np.testing.assert_array_equal(k1, held[0][0])
        np.testing.assert_array_equal(v1, held[0][1])


def test_going_back_writes_over_what_was_there(kxlib):
    say("back")
    p = S.Paged(kxlib, heads=2, kv=1, dim=64, vdim=64, block=32, batch=1)
    p.append([100], [0])
    p.append([7], [90])      # a drafted tail was rejected
    p.append([1], [64], sigma=100.0)
    same(p, [65], [0])
    p.append([40], [65])
    same(p, [105], [0])
    p.close()


def test_large_small_and_not_finite(kxlib):
    say("not finite")
    p = S.Paged(kxlib, heads=1, kv=1, dim=64, vdim=64, block=16, batch=1)
    x = np.random.default_rng(5).standard_normal((64, 1, 64)).astype(np.float32)
    x[0] = 0.0
    x[16:32] *= np.float32(1e-38)
    x[32:48] *= np.float32(1e37)
    x[50, 0, 3], x[51, 0, 4], x[52, 0, 5] = np.nan, np.inf, -np.inf
    x[53] = -0.0
    p.append([64], [0], k=x, v=x[::-1].copy())
    k, v = p.read([64], [0])[0]
    np.testing.assert_array_equal(k, p.k[0])
    np.testing.assert_array_equal(v, p.v[0])
    assert np.isnan(k[50, 0, 3]) and np.isnan(k[51, 0, 4]) and np.isnan(k[52, 0, 5]) and np.isfinite(k[49]).all()
    p.close()


def test_far_positions_turn_exactly(kxlib):
    say("far positions")
    freq = np.concatenate(([1.0, 3.0, 0.1], 10.0 ** -np.arange(29.0)))
    p = S.Paged(kxlib, heads=1, kv=1, dim=64, vdim=64, rot=64, page=1 << 20, block=64, pages=3, freq=freq)
    p.of[0] = [2, 0]
    pos = (1 << 20) - 30     # across the end of a page
    p.k[0], p.v[0] = np.zeros((pos, 1, 64)), np.zeros((pos, 1, 64))
    p.ke[0, pos // 64 * 64] = p.ve[0, pos // 64 * 64] = np.array([-7])
    start = 2 * (1 << 20) + pos // 64 * 64   # the block that is kept: zeros at scale 2^-7
    check(kxlib.kx_dev_memset(p.dk.ptr + start * 64, 0, 64 * 64, None))
    check(kxlib.kx_dev_memset(p.dv.ptr + start * 64, 0, 64 * 64, None))
    for d in (p.dks, p.dvs):
        check(kxlib.kx_h2d(d.ptr + start // 64 * 4, np.array([2.0 ** -7], np.float32).ctypes.data, 4))
    p.append([60], [pos])
    same(p, [60], [pos])
    p.close()


def run_attend(kxlib, f32, heads, kv, lens, new, seed=1, sigma=2.0, **more):
    p = S.Paged(kxlib, heads=heads, kv=kv, batch=len(lens), tokens=max(sum(lens), 1), f32=f32, pages=sum(-(-n // more.get("page", 64)) for n in lens) + 2, seed=seed, **more)
    p.append(lens, [0] * len(lens))
    pos = [n - m for n, m in zip(lens, new)]
    q = p.queries(sum(new) + 2, sigma)
    near(p.attend(new, pos, q, tokens=sum(new) + 2), p.expect(new, pos, q))
    assert p.faults() == 0
    return p, q, pos


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s.values())))
def test_attend_shapes(kxlib, shape, f32):
    """Every width, one token and several, at lengths around the groups of 64."""
    say(f"attend {shape} f32={f32}")
    p, _, _ = run_attend(kxlib, f32, 6, 3, [1, 64, 65, 200, 127], [1, 1, 1, 1, 1], **shape)
    p.close()
    p, _, _ = run_attend(kxlib, f32, 6, 3, [3, 64, 130, 200, 70], [3, 0, 9, 17, 70], **shape)
    p.close()


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (16, 1), (17, 1), (40, 2), (64, 1), (8, 8)])
def test_attend_groups_of_heads(kxlib, heads, kv, f32):
    say(f"heads {heads} of {kv} f32={f32}")
    p, _, _ = run_attend(kxlib, f32, heads, kv, [90, 5, 150], [1, 1, 1], dim=64, vdim=64, rot=64)
    p.close()
    p, _, _ = run_attend(kxlib, f32, heads, kv, [90, 5, 150], [4, 2, 40], dim=64, vdim=64, rot=64)
    p.close()


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [1, 2, 63, 64, 65, 100, 1000])
def test_attend_windows(kxlib, size, f32):
    say(f"window {size} f32={f32}")
    p, _, _ = run_attend(kxlib, f32, 4, 2, [1, 64, 129, 300], [1, 1, 1, 1], size=size, dim=64, vdim=64)
    p.close()
    p, _, _ = run_attend(kxlib, f32, 4, 2, [10, 64, 129, 300], [10, 3, 0, 150], size=size, dim=64, vdim=64)
    p.close()


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
def test_attend_long_in_parts(kxlib, f32):
    """Positions split between workgroups, for one token and for many; what `longest` says changes who does the work and nothing else that matters."""
    say(f"parts f32={f32}")
    p, q, pos = run_attend(kxlib, f32, 8, 1, [5000, 333], [1, 1], dim=128, vdim=128, rot=128, block=64)
    want = p.expect([1, 1], pos, q)
    for longest in (1, 64, 700, 2 ** 31 - 1):
        near(p.attend([1, 1], pos, q, longest=longest), want)
    p.close()
    p, q, pos = run_attend(kxlib, f32, 2, 1, [2500], [70], dim=64, vdim=64, rot=64, block=64)
    near(p.attend([70], pos, q, longest=1), p.expect([70], pos, q))
    p.close()


def test_attend_gives_the_same_bits_again_and_in_the_other_form_of_handing_over(kxlib, pytestconfig):
    say("same bits")
    import os
    strict = load_library(os.path.join(str(pytestconfig.rootpath), "blok_amd", "libkx_strict.so"))
    p, q, pos = run_attend(kxlib, False, 8, 1, [4000, 900], [1, 1], dim=128, vdim=128, block=64)
    first = p.attend([1, 1], pos, q)
    for _ in range(5):
        np.testing.assert_array_equal(p.attend([1, 1], pos, q), first)
    for _ in range(3):
        np.testing.assert_array_equal(p.attend([1, 1], pos, q, lib=strict), first)
    p.close()


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
def test_attend_keys_queries_and_values_of_very_different_sizes(kxlib, f32):
    say(f"sizes f32={f32}")
    p = S.Paged(kxlib, heads=2, kv=1, dim=64, vdim=64, block=16, f32=f32, tokens=512)
    r = np.random.default_rng(2)
    v = r.standard_normal((200, 1, 64)) * 10.0 ** r.integers(-12, 12, 200 // 8).repeat(8)[:, None, None]
    k = r.standard_normal((200, 1, 64)) * np.where(np.arange(200) // 16 % 3 == 1, 1e-6, 1.0)[:, None, None]
    p.append([200], [0], k=k.astype(np.float32), v=v.astype(np.float32))
    for sigma in (1e-30, 1e-3, 1.0, 3.0):
        q = p.queries(5, sigma)
        near(p.attend([5], [195], q), p.expect([5], [195], q))
    p.close()


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
def test_what_is_masked_does_not_matter(kxlib, f32):
    """NaN in a position that a row does not see leaves the row alone; a row that sees a NaN value has NaN in that dimension, one that sees a NaN key is NaN."""
    say(f"masked NaN f32={f32}")
    p = S.Paged(kxlib, heads=4, kv=2, dim=64, vdim=64, block=16, f32=f32, tokens=512, size=100)
    r = np.random.default_rng(4)
    k, v = r.standard_normal((180, 2, 64)).astype(np.float32), r.standard_normal((180, 2, 64)).astype(np.float32)
    v[170, 1, 7] = np.inf
    k[175, 0, 3] = np.nan
    p.append([180], [0], k=k, v=v)
    q = p.queries(150)
    got = p.attend([150], [30], q)                            # positions 30 .. 179
    clean = p.k[0], p.v[0]
    p.k[0], p.v[0] = np.nan_to_num(clean[0]), np.nan_to_num(clean[1])
    y, tol = p.expect([150], [30], q)
    at = 30 + np.arange(150)
    bad = np.zeros(y.shape, bool)
    bad[np.ix_(at >= 170, [2, 3], [7])] = True
    bad[np.ix_(at >= 175, [0, 1])] = True
    assert (np.isnan(got) == bad).all()
    assert (np.abs(got - y)[~bad] <= tol[~bad]).all()
    # of a window, what lies before it
    v[40] = np.nan
    k[40] = np.nan
    p.append([180], [0], k=k, v=v)
    p.k[0], p.v[0] = np.nan_to_num(p.k[0]), np.nan_to_num(p.v[0])
    q = p.queries(3)
    got = p.attend([3], [145], q)
    y, tol = p.expect([3], [145], q)
    assert (np.abs(got - y) <= tol).all()
    p.close()


def test_a_row_without_positions_is_zero_and_bad_tables_are_reported(kxlib):
    """What the tables hold was checked on the host (rows_of, page_ok): rows and pages outside are left out, and said."""
    say("bad tables")
    p = S.Paged(kxlib, heads=4, kv=2, dim=64, vdim=64, block=16, batch=3, tokens=512)
    p.append([100, 100, 100], [0, 0, 0])
    q = p.queries(3)
    t = p.table()
    t[0] = [-1, 64]                                            # outside
    t[1, 1] = 2 ** 31 - 1
    got = p.attend([1, 1, 1], [99, 99, 99], q, table=t)
    assert p.faults() == 1 and p.faults() == 0
    assert (got[0] == 0).all()
    y, tol = p.expect([1, 1, 1], [99, 99, 99], q)
    assert (np.abs(got[2] - y[2]) <= tol[2]).all()
    # the first page alone
    p.k[1], p.v[1] = p.k[1][:64], p.v[1][:64]
    only = S.Paged.expect(p, [0, 1, 0], [0, 63, 0], q[1:])     # no turning: a query is the same at every position
    assert (np.abs(got[1] - only[0][0]) <= only[1][0]).all()
    # positions outside the table, and rows outside the call
    got = p.attend([1, 1, 1], [128, -1, 99], q)
    assert p.faults() == 2
    out = DevBuf.from_numpy(np.full((3, 4 * 64), 0x5a5a, np.uint16))
    dq = DevBuf.from_numpy(q)
    start = DevBuf.from_numpy(np.array([0, 5, 1, 2], np.int32))
    pos = DevBuf.from_numpy(np.array([0, 0, 99], np.int32))
    c = p.cache(p.table())
    check(kxlib.kx_paged_attend(p.h, C.byref(c), C.byref(KxPagedRows(start.ptr, pos.ptr, 3, 3, 100)), dq.ptr, q.shape[1], 2, out.ptr, 256, None))
    assert p.faults() == 4
    y = out.to_numpy(np.uint16, (3, 256))
    assert (y[0] == 0x5a5a).all() and (y[2] == 0x5a5a).all() and not (y[1] == 0x5a5a).any()
    # rows for pages that are not there are dropped, the others stay as they were
    before = [x.to_numpy(np.uint8, (x.nbytes,)) for x in (p.dk, p.dv, p.dks, p.dvs)]
    t = np.full_like(p.table(), 64)
    t[:, 1] = -5
    d = DevBuf.from_numpy(np.ones((3, 2 * 128), np.float32))
    c, r = p.cache(t), p.rows([1, 1, 1], [100, 30, 64])
    check(kxlib.kx_paged_append(p.h, C.byref(c), C.byref(r), d.ptr, 256, 0, 128, None))
    assert p.faults() == 1
    for x, y in zip((p.dk, p.dv, p.dks, p.dvs), before):
        np.testing.assert_array_equal(x.to_numpy(np.uint8, (x.nbytes,)), y)
    p.close()


def test_many_sequences(kxlib):
    """More sequences than a wave has lanes, some without rows."""
    say("many sequences")
    r = np.random.default_rng(8)
    lens = [int(n) for n in r.integers(1, 90, 150)]
    new = [int(min(n, m)) for n, m in zip(lens, r.integers(0, 3, 150))]
    p, _, _ = run_attend(kxlib, False, 2, 1, lens, new, dim=64, vdim=64, rot=64, pairs=1)
    p.append([1] * 150, lens, tokens=155)
    same(p, [n + 1 for n in lens], [0] * 150)
    p.close()


def test_refusals(kxlib):
    say("refusals")
    p = S.Paged(kxlib, heads=4, kv=2, dim=64, vdim=64, block=16, batch=2, tokens=8)
    p.append([4, 4], [0, 0])
    t = p.table()
    d = DevBuf(1 << 16)

    def calls(c=None, r=None, ld=256, off=0, out=d.ptr, out_ld=256, proj=d.ptr, which="aer"):
        c, r = c or p.cache(t), r or p.rows([1, 1], [4, 4])
        rc = []
        if "a" in which:
            rc.append(kxlib.kx_paged_append(p.h, C.byref(c), C.byref(r), proj, ld, off, min(off + 128, ld - 128), None))
        if "e" in which:
            rc.append(kxlib.kx_paged_attend(p.h, C.byref(c), C.byref(r), proj, ld, off, out, out_ld, None))
        if "r" in which:
            rc.append(kxlib.kx_paged_read(p.h, C.byref(c), C.byref(r), out, out_ld, out, out_ld, None))
        return rc
    for f, v in (("d_k", None), ("d_v", None), ("d_k_scale", None), ("d_v_scale", None), ("d_table", None), ("d_k", d.ptr + 8), ("d_v", d.ptr + 1), ("d_k_scale", d.ptr + 2), ("pages", 0), ("pages", -1),
                 ("table_ld", 0), ("table_ld", -3), ("table_ld", 2 ** 31 - 1)):
        c = p.cache(t)
        setattr(c, f, v)
        assert all(calls(c=c)), f
    for f, v in (("d_start", None), ("d_pos", None), ("batch", 0), ("batch", 3), ("batch", -1), ("tokens", -1), ("longest", 0), ("longest", -1)):
        r = p.rows([1, 1], [4, 4])
        setattr(r, f, v)
        assert all(calls(r=r)), f
    r = p.rows([1, 1], [4, 4])
    r.tokens = 9
    assert all(calls(r=r, which="ae"))
    assert all(calls(ld=255, which="e")) and all(calls(ld=127, which="a")) and all(calls(off=-1, which="ae")) and all(calls(off=1, which="e"))
    assert all(calls(out_ld=255, which="e")) and all(calls(out_ld=127, which="r")) and all(calls(out=None, which="er")) and all(calls(out=d.ptr + 1, which="er"))
    assert all(calls(proj=None, which="ae")) and all(calls(proj=d.ptr + 2, which="ae"))
    r.tokens = 0
    assert not any(calls(r=r))
    assert p.faults() == 0
    p.close()
