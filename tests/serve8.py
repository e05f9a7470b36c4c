"""Plain forms in 64 bits of the 8-bit serving operators (blok_amd/csrc/kx_paged.h, kx_fp8.h), and a paged cache to call them with."""
import ctypes as C

import numpy as np

from blok_amd.lib import DevBuf, KxFp8Args, KxPagedCache, KxPagedConfig, KxPagedRows, check

LEAST, MOST = -100, 448.0
WIDTHS = ((64, 64), (128, 128), (192, 128), (256, 256))


def _table():
    c = np.arange(256)
    e, f = c >> 3 & 15, c & 7
    x = np.where(e > 0, np.ldexp(8.0 + f, e - 10), np.ldexp(f * 1.0, -9))
    x = np.where((c & 127) == 127, np.nan, x)
    return np.where(c > 127, -x, x)


VALUES = _table()                                              # what the 256 codes stand for
ORDER = [32 * h + 16 * r + 4 * q + j for q in range(4) for h in range(2) for r in range(2) for j in range(4)]   # token of each place of 64


def exponent(most):
    """The least e >= -100 with most <= 448 * 2^e, element by element."""
    m, e = np.frexp(np.asarray(most, np.float64))
    return np.maximum(np.where(m > 0, e - 9 + (m > 0.875), LEAST), LEAST).astype(int)


def rounded(x):
    """The nearest 8-bit elements to numbers of at most 448, ties to even; NaN for what is not finite."""
    x = np.where(np.isfinite(x), x, np.nan)
    step = np.frexp(np.maximum(np.abs(np.nan_to_num(x)), 2.0 ** -6))[1] - 4
    return np.ldexp(np.rint(np.ldexp(x, -step)), step)


def most_of(x, axis):
    return np.max(np.where(np.isfinite(x), np.abs(x), 0.0), axis=axis, initial=0.0)


def codes(x):
    """Codes of 8-bit elements."""
    c = np.full(x.shape, 0x7f, np.uint8)
    order = np.argsort(VALUES[:127])
    ok = np.isfinite(x)
    c[ok] = order[np.searchsorted(VALUES[:127][order], np.abs(x[ok]))]
    return np.where(np.signbit(x) & ok, c | 0x80, c).astype(np.uint8)


def turned(x, pos, rot, pairs, freq):
    """x [n][heads][dim] at positions pos [n], the first rot dimensions turned in pairs."""
    x = np.array(x, np.float64)
    if rot:
        a = np.asarray(pos, np.float64)[:, None, None] * freq
        c, s = np.cos(a), np.sin(a)
        i, j = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
        u, v = x[..., i].copy(), x[..., j].copy()
        x[..., i], x[..., j] = u * c - v * s, u * s + v * c
    return x


def bf16(a):
    """bf16 bits -> float64"""
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Paged:
    """A cache of numpy values beside the device's: k, v [sequence][position][kv][...] as the operators are to hold them."""

    def __init__(self, lib, heads=4, kv=2, dim=128, vdim=128, page=64, block=32, rot=0, pairs=0, size=0, f32=False, batch=1, tokens=512, pages=64, scale=None, base=10000.0, freq=None,
                 seed=0):
        self.lib, self.heads, self.kv, self.dim, self.vdim, self.page, self.block, self.rot, self.pairs, self.size, self.f32 = lib, heads, kv, dim, vdim, page, block, rot, pairs, size, f32
        self.scale = np.float32(dim ** -0.5 if scale is None else scale)
        self.batch, self.pages = batch, pages
        self.freq = base ** (-2.0 * np.arange(rot // 2) / max(rot, 1)) if freq is None else np.asarray(freq, np.float64)
        self.dp, self.vp = next(w for w in WIDTHS if dim <= w[0] and vdim <= w[1])
        self.h = C.c_void_p()
        cfg = KxPagedConfig(heads, kv, dim, vdim, page, block, rot, pairs, size, self.scale, base)
        check(lib.kx_paged_create(C.byref(cfg), None if freq is None else self.freq.ctypes.data, int(f32), batch, tokens, C.byref(self.h)))
        self.rng = np.random.default_rng(seed)
        # whatever the memory held before: NaN codes, and scales of every kind
        self.dk = DevBuf.from_numpy(np.full((pages, kv, page, self.dp), 0x7f, np.uint8))
        self.dv = DevBuf.from_numpy(np.full((pages, kv, page // 64, self.vp, 64), 0xff, np.uint8))
        junk = np.array([np.nan, np.inf, 0.0, -1.0, 1e30], np.float32)
        self.dks, self.dvs = (DevBuf.from_numpy(np.resize(junk, (pages, kv, page // block)).astype(np.float32)) for _ in range(2))
        self.free = list(self.rng.permutation(pages))
        self.of = [[] for _ in range(batch)]
        self.k, self.v = ([np.zeros((0, kv, d)) for _ in range(batch)] for d in (dim, vdim))
        self.ke, self.ve = ({}, {})                              # exponents by (sequence, block)
        self.keep = []

    def close(self):
        check(self.lib.kx_paged_destroy(self.h))

    def table(self, ld=None):
        ld = max(ld or 0, max(len(p) for p in self.of), 1)
        t = np.full((self.batch, ld), -1, np.int32)
        for b, p in enumerate(self.of):
            t[b, :len(p)] = p
        return t

    def cache(self, table):
        d = DevBuf.from_numpy(table)
        self.keep.append(d)
        return KxPagedCache(self.dk.ptr, self.dv.ptr, self.dks.ptr, self.dvs.ptr, d.ptr, self.pages, table.shape[1])

    def rows(self, new, pos, tokens=None, longest=None):
        start = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        ds, dp = DevBuf.from_numpy(start), DevBuf.from_numpy(np.asarray(pos, np.int32))
        self.keep += [ds, dp]
        return KxPagedRows(ds.ptr, dp.ptr, len(new), int(start[-1]) if tokens is None else tokens, longest or max(1, max(p + n for p, n in zip(pos, new))))

    def reserve(self, b, n):
        while len(self.of[b]) * self.page < n:
            self.of[b].append(int(self.free.pop()))

    def _hold(self, b, pos, k, v):
        """What appending turned keys and values at pos leaves in the plain cache."""
        for held, exps, x in ((self.k, self.ke, k), (self.v, self.ve, v)):
            held[b] = np.concatenate((held[b][:pos], np.asarray(x, np.float64)))
            n = pos + len(x)
            for lo in range(pos // self.block * self.block, n, self.block):
                part = held[b][lo:min(lo + self.block, n)]
                new = part[max(pos - lo, 0):]
                e = exponent(most_of(new, (0, 2)))
                if lo < pos:
                    e = np.maximum(e, exps[b, lo])
                exps[b, lo] = e
                s = np.ldexp(1.0, e)[:, None]
                held[b][lo:min(lo + self.block, n)] = rounded(part / s) * s

    def append(self, new, pos, sigma=1.0, k=None, v=None, tokens=None, stream=None, lib=None, ld_more=3):
        """new[b] rows at pos[b] of every sequence, on the device and in the plain cache; returns the projections."""
        n = sum(new)
        for b in range(self.batch):
            self.reserve(b, pos[b] + new[b])
        kd, vd = self.kv * self.dim, self.kv * self.vdim
        proj = (sigma * self.rng.standard_normal((max(n, tokens or 0, 1), kd + vd + ld_more))).astype(np.float32)
        if k is not None:
            proj[:n, 1:1 + kd] = k.reshape(n, kd)
        if v is not None:
            proj[:n, 1 + kd:1 + kd + vd] = v.reshape(n, vd)
        if tokens:
            proj[n:] = np.nan
        at = 0
        for b in range(self.batch):
            r = proj[at:at + new[b]].astype(np.float64)
            at += new[b]
            if new[b]:
                with np.errstate(invalid="ignore"):
                    x = turned(r[:, 1:1 + kd].reshape(-1, self.kv, self.dim), pos[b] + np.arange(new[b]), self.rot, self.pairs, self.freq)
                self._hold(b, pos[b], x, r[:, 1 + kd:1 + kd + vd].reshape(-1, self.kv, self.vdim))
        d = DevBuf.from_numpy(proj)
        self.keep.append(d)
        check((lib or self.lib).kx_paged_append(self.h, C.byref(self.cache(self.table())), C.byref(self.rows(new, pos, tokens)), d.ptr, proj.shape[1], 1, 1 + kd, stream))
        return proj

    def read(self, n, pos):
        """[(k, v)] of n[b] positions from pos[b] on, as float64"""
        t, kd, vd = max(sum(n), 1), self.kv * self.dim + 1, self.kv * self.vdim + 2
        ok, ov = (DevBuf.from_numpy(np.full((t, w), 0x1234, np.uint16)) for w in (kd, vd))
        check(self.lib.kx_paged_read(self.h, C.byref(self.cache(self.table())), C.byref(self.rows(n, pos)), ok.ptr, kd, ov.ptr, vd, None))
        check(self.lib.kx_sync(None))
        k, v = ok.to_numpy(np.uint16, (t, kd)), ov.to_numpy(np.uint16, (t, vd))
        assert (k[:, -1] == 0x1234).all() and (v[:, -2:] == 0x1234).all()
        k, v = bf16(k[:, :-1]).reshape(t, self.kv, self.dim), bf16(v[:, :-2]).reshape(t, self.kv, self.vdim)
        cut = np.cumsum([0] + list(n))
        return [(k[a:b], v[a:b]) for a, b in zip(cut, cut[1:])]

    def queries(self, n, sigma=2.0):
        return (sigma * self.rng.standard_normal((n, self.heads * self.dim + 5))).astype(np.float32)

    def attend(self, new, pos, proj, tokens=None, longest=None, table=None, lib=None, stream=None, out=None):
        """[tokens][heads][vdim] as float64; rows behind the last sequence are checked to be as they were."""
        n, width = sum(new), self.heads * self.vdim + 3
        t = max(n if tokens is None else tokens, 1)
        fill = np.full((t, width), 0x5a5a5a5a, np.uint32) if self.f32 else np.full((t, width), 0x5a5a, np.uint16)
        o, d = DevBuf.from_numpy(fill), DevBuf.from_numpy(proj)
        check((lib or self.lib).kx_paged_attend(self.h, C.byref(self.cache(self.table() if table is None else table)), C.byref(self.rows(new, pos, tokens, longest)), d.ptr, proj.shape[1], 2,
                                                o.ptr, width, stream))
        check(self.lib.kx_sync(stream))
        y = o.to_numpy(fill.dtype, fill.shape)
        assert (y[:, -3:] == fill[0, 0]).all() and (y[n:] == fill[0, 0]).all()
        y = y[:n, :-3]
        return (np.ascontiguousarray(y).view(np.float32).astype(np.float64) if self.f32 else bf16(y)).reshape(n, self.heads, self.vdim)

    def expect(self, new, pos, proj):
        """The attention in 64 bits, and how far a result may be off, element by element.

        A query is divided by a power of two and rounded to f16, 2^-11 of each element (in the 32-bit format to two of them, 2^-22), but never better than half of
        the smallest step, 2^-25, where the largest element is 1/2 or more: 2^-24 of the largest.  Scores and sums are 32-bit.  With S the largest sum of |q_d k_d| scale, and
        K that of |k_d| scale times the largest |q_d|, a score is off by d = (h + (dim + 8) 2^-24) S + 2^-24 K at most.  A weight is off by d of itself and rounded to f16, h of
        itself or, where it is small, 2^-25 of the largest one times its block's scale; the denominator is off by d, and n terms add n 2^-24 to each sum.  The result's own
        rounding is 2^-8 for bf16, 2^-24 for float."""
        h, last = (2.0 ** -22, 2.0 ** -24) if self.f32 else (2.0 ** -11, 2.0 ** -8)
        g, ys, tols, at = self.heads // self.kv, [], [], 0
        for b in range(self.batch):
            if not new[b]:
                continue
            p = pos[b] + np.arange(new[b])
            q = turned(proj[at:at + new[b], 2:2 + self.heads * self.dim].reshape(-1, self.heads, self.dim), p, self.rot, self.pairs, self.freq)
            at += new[b]
            j = np.arange(p[-1] + 1)
            y, tol = np.zeros((new[b], self.heads, self.vdim)), np.zeros((new[b], self.heads, self.vdim))
            blocks = j // self.block * self.block
            for head in range(self.heads):
                k, v = self.k[b][:p[-1] + 1, head // g], self.v[b][:p[-1] + 1, head // g]
                unit = np.ldexp(1.0, np.array([self.ve[b, lo][head // g] for lo in blocks]))   # scale of a token's values
                for i in range(new[b]):
                    see = slice(max(0, p[i] - self.size + 1) if self.size else 0, p[i] + 1)
                    s = (k[see] @ q[i, head]) * float(self.scale)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    y[i, head] = w @ v[see]
                    most, size = (np.max(np.abs(k[see]) @ x) * abs(float(self.scale)) for x in (np.abs(q[i, head]), np.full(self.dim, np.abs(q[i, head]).max())))
                    n = see.stop - see.start
                    d = (h + (self.dim + 8) * 2.0 ** -24) * most + 2.0 ** -24 * size
                    a = w @ np.abs(v[see])
                    small = n * 2.0 ** -25 * np.max(w * unit[see]) * 448.0
                    tol[i, head] = 1.01 * (last * np.abs(y[i, head]) + a * (h + np.expm1(2 * d) + (2 * n + 64) * 2.0 ** -24) + small)
            ys.append(y)
            tols.append(tol)
        return np.concatenate(ys), np.concatenate(tols)

    def faults(self):
        b = C.c_int32(-1)
        check(self.lib.kx_paged_faults(self.h, C.byref(b), None))
        return b.value


# ---- products -----------------------------------------------------------------------------------------------------
def matrix(rng, rows, cols, ld=None, sigma=1.0):
    """Codes [rows][ld], scales, and the matrix that they stand for."""
    nb = -(-cols // 128)
    c = np.zeros((rows, ld or nb * 128), np.uint8)
    x = rounded(np.clip(sigma * 60 * rng.standard_normal((rows, cols)), -MOST, MOST))
    c[:, :cols] = codes(x)
    s = np.exp(rng.standard_normal((-(-rows // 128), nb))).astype(np.float32) * np.float32(0.01)
    w = x * s.astype(np.float64).repeat(128, 0)[:rows].repeat(128, 1)[:, :cols]
    return c, s, w


def row_codes(x):
    """What rows are rounded to: [tokens][cols] in 64 bits."""
    t, cols = x.shape
    y = np.zeros((t, -(-cols // 128) * 128))
    y[:, :cols] = x
    y = y.reshape(t, -1, 128)
    s = np.ldexp(1.0, exponent(most_of(y, 2)))[..., None]
    return (rounded(y / s) * s).reshape(t, -1)[:, :cols]


def product(lib, h, c, s, x, cols, out_f32, x_f32, tokens=None, stream=None):
    """x [tokens][cols] float32 (bf16 values where not x_f32) through kx_fp8_run; float64."""
    t, rows = x.shape[0] if tokens is None else tokens, c.shape[0]
    xp = np.full((x.shape[0], cols + 5), np.nan, np.float32)
    xp[:, :cols] = x
    dx = DevBuf.from_numpy(xp if x_f32 else (xp.view(np.uint32) >> 16).astype(np.uint16))
    fill = np.full((x.shape[0], rows + 3), 0x5a5a5a5a, np.uint32) if out_f32 else np.full((x.shape[0], rows + 3), 0x5a5a, np.uint16)
    dc, ds, do = DevBuf.from_numpy(c), DevBuf.from_numpy(s), DevBuf.from_numpy(fill)
    a = KxFp8Args(x_f32, out_f32, t, rows, cols, c.shape[1], cols + 5, rows + 3, dc.ptr, ds.ptr, dx.ptr, do.ptr)
    check(lib.kx_fp8_run(h, C.byref(a), stream))
    check(lib.kx_sync(stream))
    y = do.to_numpy(fill.dtype, fill.shape)
    assert (y[:, rows:] == fill[0, 0]).all() and (y[t:] == fill[0, 0]).all()
    y = np.ascontiguousarray(y[:t, :rows])
    return y.view(np.float32).astype(np.float64) if out_f32 else bf16(y)


def product_tolerance(q, w, y, out_f32):
    """Float results are sums of exact products in 32 bits: (cols + 8) 2^-24 of the sum of their magnitudes.  For bf16 results the matrix cores add 8-bit products with fewer bits: a block of
    128 came out 1.5e-5 of its root mean square off at most (normal codes of three magnitudes, 16384 sums each), for which 2^-14 of the magnitudes' sum is 20 times as
    much; the rounding of the result is 2^-8."""
    a = np.abs(q) @ np.abs(w).T
    return 1.01 * ((q.shape[1] + 8) * 2.0 ** -24 * a + (0 if out_f32 else 2.0 ** -14 * a + 2.0 ** -8 * np.abs(y))) + 1e-300
