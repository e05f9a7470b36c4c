"""Attention over the paged cache where few positions outweigh many, where the sizes of a query's elements or of blocks of values lie far apart, and where a query is not finite, element by element
against the form in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import serve8 as S
from blok_amd.lib import DevBuf, check
from kxt import say

pytestmark = pytest.mark.gpu

FORMATS = pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])


def expect(p, new, pos, proj):
    """The attention in 64 bits, and how far a result may be off, element by element, by the roundings alone.

    An element of a query is rounded to f16, 2^-11 of it (for float results to the sum of two, 2^-22), and never better than 2^-25 beside a largest one of 2^14 or more: 2^-39 of that.  A
    score is a 32-bit sum of dim products, turned and scaled in 32 bits.  With S the largest sum of |q_d k_d| scale, K that of |k_d| scale times the largest |q_d| and B the largest
    exponent of a block of values, its exponent of two is off by d = (h + (dim + 8) 2^-24) S + 2^-39 K + (2 S + B) 2^-23 at most, and the weight by expm1(d).  For bf16 results
    a weight is rounded to f16 in turn, 2^-11 of it or 2^-25 beside a largest w_t 2^b_t of 2^11 or more: 2^-36 of that; for float results to the sum of three bf16, which hold a float.  Sums of n terms
    add (2 n + 64) 2^-24, and a result's own rounding is 2^-8 for bf16 and 2^-24 for float."""
    h, hw, last, least = (2.0 ** -22, 2.0 ** -24, 2.0 ** -24, 0.0) if p.f32 else (2.0 ** -11, 2.0 ** -11, 2.0 ** -8, 2.0 ** -36)
    g, ys, tols, at, scale = p.heads // p.kv, [], [], 0, float(p.scale)
    for b in range(p.batch):
        if not new[b]:
            continue
        at_pos = pos[b] + np.arange(new[b])
        q = S.turned(proj[at:at + new[b], 2:2 + p.heads * p.dim].reshape(-1, p.heads, p.dim), at_pos, p.rot, p.pairs, p.freq)
        at += new[b]
        n = at_pos[-1] + 1
        j = np.arange(n)
        hide = (j > at_pos[:, None]) | (at_pos[:, None] - j >= (p.size or n))
        y, tol = np.zeros((new[b], p.heads, p.vdim)), np.zeros((new[b], p.heads, p.vdim))
        for head in range(p.heads):
            k, v = p.k[b][:n, head // g], p.v[b][:n, head // g]
            e = np.array([p.ve[b, lo][head // g] for lo in j // p.block * p.block])
            unit = np.ldexp(1.0, e)
            s = q[:, head] @ k.T * scale
            s[hide] = -np.inf
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            y[:, head] = w @ v
            most = (np.abs(q[:, head]) @ np.abs(k).T * abs(scale)).max(1)
            d = (h + (p.dim + 8) * 2.0 ** -24) * most + 2.0 ** -39 * np.abs(q[:, head]).max(1) * np.abs(k).sum(1).max() * abs(scale) + (2 * most + np.abs(e).max()) * 2.0 ** -23
            rounds = (hw + np.expm1(2 * d) + (2 * n + 64) * 2.0 ** -24)[:, None]
            small = least * (w * unit).max(1)[:, None] * ((~hide).astype(float) @ (np.abs(v) / unit[:, None]))
            tol[:, head] = 1.01 * (last * np.abs(y[:, head]) + rounds * (w @ np.abs(v)) + small)
        ys.append(y)
        tols.append(tol)
    return np.concatenate(ys), np.concatenate(tols)


def attend(p, new, pos, proj, longest=None, lib=None, pad=3):
    """As Paged.attend, with rows of results of `pad` more elements, which stay as they were."""
    n, width = sum(new), p.heads * p.vdim + pad
    fill = np.full((n + 2, width), 0x5a5a5a5a, np.uint32) if p.f32 else np.full((n + 2, width), 0x5a5a, np.uint16)
    o, d = DevBuf.from_numpy(fill), DevBuf.from_numpy(proj)
    check((lib or p.lib).kx_paged_attend(p.h, C.byref(p.cache(p.table())), C.byref(p.rows(new, pos, n + 2, longest)), d.ptr, proj.shape[1], 2, o.ptr, width, None))
    check(p.lib.kx_sync(None))
    y = o.to_numpy(fill.dtype, fill.shape)
    assert (y[:, width - pad:] == fill[0, 0]).all() and (y[n:] == fill[0, 0]).all()
    y = np.ascontiguousarray(y[:n, :width - pad])
    return (y.view(np.float32).astype(np.float64) if p.f32 else S.bf16(y)).reshape(n, p.heads, p.vdim)


def near(got, want, what=""):
    over = np.abs(got - want[0]) / np.maximum(want[1], 1e-300)
    print(f"  {what} off by {np.nanmax(over):.3f} of the tolerance", flush=True)
    assert (over <= 1).all(), f"{what}: {(~(over <= 1)).sum()} of {over.size} off, {np.nanmax(over):.3f} times the tolerance, at {np.unravel_index(np.nanargmax(over), over.shape)}"


# rows that the waves of a workgroup share, one and several blocks of them, and rows that each wave has for itself
ROWS = [(1, 2), (5, 8), (80, 2)]


@FORMATS
@pytest.mark.parametrize("rows,heads", ROWS)
@pytest.mark.parametrize("bits", [14, 20, 26])
def test_many_positions_far_below_one(kxlib, rows, heads, bits, f32):
    """The first position has a weight of 2^bits times any other's and values of zero, so that all of the result comes from the others."""
    say(f"{rows} rows of {heads} heads, {bits} bits, f32={f32}")
    n = 3000
    p = S.Paged(kxlib, heads=heads, kv=1, dim=64, vdim=64, block=16, f32=f32, tokens=n, pages=50)
    r = np.random.default_rng(bits)
    k, v = 0.1 * r.standard_normal((n, 1, 64)).astype(np.float32), (1 + 0.3 * r.standard_normal((n, 1, 64))).astype(np.float32)
    k[:, 0, 0] = 0.0
    k[0], v[0] = 0.0, 0.0
    k[0, 0, 0] = 16.0
    p.append([n], [0], k=k, v=v)
    q = p.queries(rows, 0.5)
    q[:, 2:2 + heads * 64:64] = bits * np.log(2.0) / (16 * p.scale)
    for longest in (1, n):   # all positions by one workgroup, and in parts
        near(attend(p, [rows], [n - rows], q, longest), expect(p, [rows], [n - rows], q), f"longest {longest}")
    assert p.faults() == 0
    p.close()


@FORMATS
@pytest.mark.parametrize("rows,heads", ROWS)
@pytest.mark.parametrize("bits", [20, 24])
def test_queries_with_one_large_element(kxlib, rows, heads, bits, f32):
    """An element of a query that meets keys of zero and is 2^bits times as large as the others takes nothing from these."""
    say(f"{rows} rows of {heads} heads, an element of 2^{bits}, f32={f32}")
    n = 400
    p = S.Paged(kxlib, heads=heads, kv=1, dim=64, vdim=64, block=32, f32=f32, tokens=n, pages=8)
    k = np.random.default_rng(bits).standard_normal((n, 1, 64)).astype(np.float32)
    k[:, 0, 5] = 0.0
    p.append([n], [0], k=k, v=k[::-1].copy())
    q = p.queries(rows, 1.0)
    q[:, 2 + 5:2 + heads * 64:64] = 2.0 ** bits
    near(attend(p, [rows], [n - rows], q), expect(p, [rows], [n - rows], q))
    p.close()


@FORMATS
@pytest.mark.parametrize("rows,heads", ROWS)
@pytest.mark.parametrize("large", [1.0, 1e14, 1e30])
@pytest.mark.parametrize("first", [False, True])
def test_values_of_zero_beside_large_ones(kxlib, rows, heads, large, first, f32):
    """Positions whose values are zero, in blocks whose scale is the least there is, have their share of the weights whatever the others' values are."""
    say(f"{rows} rows of {heads} heads, values of {large}, zeros first={first}, f32={f32}")
    n = 700
    p = S.Paged(kxlib, heads=heads, kv=1, dim=64, vdim=64, block=64, f32=f32, tokens=n, pages=12)
    r = np.random.default_rng(3)
    k, v = r.standard_normal((n, 1, 64)).astype(np.float32), (large * (1 + 0.3 * r.standard_normal((n, 1, 64)))).astype(np.float32)
    v[:320] = 0.0
    if not first:
        v = v[::-1].copy()
        v[n - 320 // 64 * 64 + 60:] = 0.0
    p.append([n], [0], k=k, v=v)
    q = p.queries(rows, 0.3)
    for longest in (1, n):
        near(attend(p, [rows], [n - rows], q, longest), expect(p, [rows], [n - rows], q), f"longest {longest}")
    p.close()


@FORMATS
@pytest.mark.parametrize("n", [1, 200])
def test_queries_that_are_not_finite(kxlib, n, f32):
    """The scores of such a query are infinite or not numbers, whatever the sign, and so is the softmax of them; the other heads and rows are as they would be."""
    for rows in (1, 5, 80):
        if rows > n:
            continue
        say(f"not finite, {rows} of {n} rows, f32={f32}")
        p = S.Paged(kxlib, heads=4, kv=2, dim=64, vdim=64, block=16, f32=f32, tokens=n + 2, pages=8)
        k = np.random.default_rng(6).uniform(1, 2, (n, 2, 64)).astype(np.float32)
        p.append([n], [0], k=k, v=k[::-1].copy())
        q = p.queries(rows, 0.5)
        want = expect(p, [rows], [n - rows], q)
        bad = np.zeros((rows, 4), bool)
        for i, x in enumerate((-np.inf, np.inf, np.nan)):
            row, head = (i * 2) % rows, i
            q[row, 2 + head * 64 + 9 * i] = x
            bad[row, head] = True
        got = attend(p, [rows], [n - rows], q)
        assert np.isnan(got[bad]).all()
        near(got[~bad], (want[0][~bad], want[1][~bad]))
        p.close()


@FORMATS
@pytest.mark.parametrize("rows,heads", ROWS)
def test_values_far_below_the_largest_of_their_block(kxlib, rows, heads, f32):
    """The largest value of each block is one that no row has a weight for, and all others are codes from 2^-9, the smallest there is, to 2^-4: subnormal numbers of every format that they go through."""
    say(f"{rows} rows of {heads} heads, small codes, f32={f32}")
    n = 700
    p = S.Paged(kxlib, heads=heads, kv=1, dim=64, vdim=64, block=16, f32=f32, tokens=n, pages=12)
    r = np.random.default_rng(11)
    k, v = (0.1 * r.standard_normal((n, 1, 64))).astype(np.float32), np.ldexp(1.0, r.integers(-9, -3, (n, 1, 64))).astype(np.float32)
    k[:, 0, 0] = 16.0
    k[::16], v[::16] = 0.0, 448.0
    p.append([n], [0], k=k, v=v)
    assert (p.v[0][1:16] == v[1:16]).all()
    q = p.queries(rows, 0.5)
    q[:, 2:2 + heads * 64:64] = 120 * np.log(2.0) / (16 * p.scale)      # 2^-120 of the others' weights
    want = expect(p, [rows], [n - rows], q)
    assert (want[0] < 0.05).all()
    for longest in (1, n):
        near(attend(p, [rows], [n - rows], q, longest), want, f"longest {longest}")
    p.close()
