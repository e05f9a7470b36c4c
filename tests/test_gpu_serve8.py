"""The 8-bit serving operators as a layer uses them, one behind the other on a stream: projections of 8-bit matrices, their rows appended to a paged cache, attention over it and
the projection of its result.  Prompts, decoded and drafted tokens, on streams of their own and replayed as a graph; every result against the plain form in 64 bits of what it was
computed from."""
import ctypes as C

import numpy as np
import pytest

import serve8 as S
from blok_amd.lib import DevBuf, KxFp8Args, KxPagedCache, KxPagedRows, check
from kxt import say

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, VDIM, HIDDEN = 8, 2, 64, 48, 200
ROWS = HEADS * DIM + KV * (DIM + VDIM)


class Hip:
    """Streams and graphs of the runtime that the library is linked with."""

    def __init__(self, lib):
        self.lib, p = lib, C.c_void_p
        for name, args in (("hipStreamCreate", [C.POINTER(p)]), ("hipStreamDestroy", [p]), ("hipStreamBeginCapture", [p, C.c_int]), ("hipStreamEndCapture", [p, C.POINTER(p)]),
                           ("hipGraphInstantiate", [C.POINTER(p), p, p, p, C.c_size_t]), ("hipGraphLaunch", [p, p]), ("hipGraphExecDestroy", [p]), ("hipGraphDestroy", [p])):
            f = getattr(lib, name)
            f.argtypes, f.restype = args, C.c_int
            setattr(self, name, lambda *a, f=f, name=name: self._ok(name, f(*a)))

    @staticmethod
    def _ok(name, rc):
        assert rc == 0, f"{name}: {rc}"

    def stream(self):
        s = C.c_void_p()
        self.hipStreamCreate(C.byref(s))
        return s

    def capture(self, stream, calls):
        graph, ready = C.c_void_p(), C.c_void_p()
        self.hipStreamBeginCapture(stream, 1)
        try:
            calls()
        finally:
            self.hipStreamEndCapture(stream, C.byref(graph))
        self.hipGraphInstantiate(C.byref(ready), graph, None, None, 0)
        self.hipGraphDestroy(graph)
        return ready


class Layer:
    """A layer with buffers for `tokens` rows of `batch` sequences that stay where they are; `pages` pages in the table of each."""

    def __init__(self, lib, batch, tokens, pages, seed):
        self.lib, self.batch, self.tokens, self.pages = lib, batch, tokens, pages
        self.p = S.Paged(lib, heads=HEADS, kv=KV, dim=DIM, vdim=VDIM, rot=32, block=32, batch=batch, tokens=tokens, pages=batch * pages, seed=seed)
        self.rng = np.random.default_rng(seed + 100)
        self.c1, self.s1, self.w1 = S.matrix(self.rng, ROWS, HIDDEN)
        self.c2, self.s2, self.w2 = S.matrix(self.rng, HIDDEN, HEADS * VDIM)
        self.h1, self.h2 = C.c_void_p(), C.c_void_p()
        check(lib.kx_fp8_create(tokens, HIDDEN, C.byref(self.h1)))
        check(lib.kx_fp8_create(tokens, HEADS * VDIM, C.byref(self.h2)))
        self.d = {n: DevBuf.from_numpy(a) for n, a in dict(c1=self.c1, s1=self.s1, c2=self.c2, s2=self.s2, x=np.zeros((tokens, HIDDEN), np.float32),
                                                           proj=np.zeros((tokens, ROWS + 2), np.float32), mid=np.zeros((tokens, HEADS * VDIM), np.uint16),
                                                           out=np.zeros((tokens, HIDDEN), np.float32), start=np.zeros(batch + 1, np.int32), pos=np.zeros(batch, np.int32),
                                                           table=np.full((batch, pages), -1, np.int32)).items()}

    def put(self, new, pos):
        """Inputs of a step into the buffers."""
        self.new, self.pos, n = new, pos, sum(new)
        for b in range(self.batch):
            self.p.reserve(b, pos[b] + new[b])
        self.x = np.full((self.tokens, HIDDEN), np.nan, np.float32)   # rows behind the last sequence are of no account
        self.x[:n] = self.rng.standard_normal((n, HIDDEN))
        self.d["x"].upload(self.x)
        self.d["start"].upload(np.concatenate(([0], np.cumsum(new))).astype(np.int32))
        self.d["pos"].upload(np.asarray(pos, np.int32))
        self.d["table"].upload(self.p.table(self.pages))
        for name, bits in (("mid", 16), ("out", 32)):
            self.d[name].upload(np.full(self.d[name].nbytes // (bits // 8), 0x5a5a, np.uint16 if bits == 16 else np.uint32))

    def run(self, stream, tokens=None):
        d, t, lib = {n: b.ptr for n, b in self.d.items()}, self.tokens if tokens is None else tokens, self.lib
        cache = KxPagedCache(self.p.dk.ptr, self.p.dv.ptr, self.p.dks.ptr, self.p.dvs.ptr, d["table"], self.p.pages, self.pages)
        rows = KxPagedRows(d["start"], d["pos"], self.batch, t, self.pages * 64)
        first = KxFp8Args(True, True, t, ROWS, HIDDEN, self.c1.shape[1], HIDDEN, ROWS + 2, d["c1"], d["s1"], d["x"], d["proj"] + 8)
        check(lib.kx_fp8_run(self.h1, C.byref(first), stream))
        check(lib.kx_paged_append(self.p.h, C.byref(cache), C.byref(rows), d["proj"], ROWS + 2, 2 + HEADS * DIM, 2 + HEADS * DIM + KV * DIM, stream))
        check(lib.kx_paged_attend(self.p.h, C.byref(cache), C.byref(rows), d["proj"], ROWS + 2, 2, d["mid"], HEADS * VDIM, stream))
        second = KxFp8Args(False, True, t, HIDDEN, HEADS * VDIM, self.c2.shape[1], HEADS * VDIM, HIDDEN, d["c2"], d["s2"], d["mid"], d["out"])
        check(lib.kx_fp8_run(self.h2, C.byref(second), stream))

    def verify(self, stream):
        """Each operator's result from its own inputs, as the device had them."""
        check(self.lib.kx_sync(stream))
        n, x = sum(self.new), S.row_codes(self.x[:sum(self.new)].astype(np.float64))
        proj, mid = self.d["proj"].to_numpy(np.float32, (self.tokens, ROWS + 2)), self.d["mid"].to_numpy(np.uint16, (self.tokens, HEADS * VDIM))
        out = self.d["out"].to_numpy(np.float32, (self.tokens, HIDDEN))
        assert (mid[n:] == 0x5a5a).all()
        y = x @ self.w1.T
        self.close_to("projection", proj[:n, 2:], y, S.product_tolerance(x, self.w1, y, True))
        at, kd = 0, 2 + HEADS * DIM
        for b in range(self.batch):
            r = proj[at:at + self.new[b]].astype(np.float64)
            at += self.new[b]
            if self.new[b]:
                k = S.turned(r[:, kd:kd + KV * DIM].reshape(-1, KV, DIM), self.pos[b] + np.arange(self.new[b]), self.p.rot, self.p.pairs, self.p.freq)
                self.p._hold(b, self.pos[b], k, r[:, kd + KV * DIM:].reshape(-1, KV, VDIM))
        for b, (k, v) in enumerate(self.p.read([len(k) for k in self.p.k], [0] * self.batch)):
            np.testing.assert_array_equal(k, self.p.k[b])
            np.testing.assert_array_equal(v, self.p.v[b])
        y, tol = self.p.expect(self.new, self.pos, proj[:n])
        self.close_to("attention", S.bf16(mid[:n]).reshape(y.shape), y, tol)
        z = S.row_codes(S.bf16(mid[:n]))
        y = z @ self.w2.T
        self.close_to("result", out[:n], y, S.product_tolerance(z, self.w2, y, True))
        assert self.p.faults() == 0

    @staticmethod
    def close_to(what, got, want, tol):
        over = np.abs(got - want) / np.maximum(tol, 1e-300)
        print(f"  {what} off by {over.max():.3f} of the tolerance", flush=True)
        assert (over <= 1).all(), f"{what}: {(over > 1).sum()} of {over.size}, {over.max():.3f} times the tolerance"

    def close(self):
        self.p.close()
        for h in (self.h1, self.h2):
            check(self.lib.kx_fp8_destroy(h))


STEPS = [[70, 33, 0], [1, 1, 5], [1, 1, 1], [4, 0, 4], [1, 1, 1], [1, 64, 1]]


def test_prompts_decoding_and_drafts(kxlib):
    """Steps of their own sizes, the inputs of each as the one before left the cache; a rejected draft is written over."""
    hip = Hip(kxlib)
    st, layer = hip.stream(), Layer(kxlib, 3, 160, 4, seed=1)
    pos = [0, 0, 0]
    for i, new in enumerate(STEPS):
        say(f"step {i} of {new} at {pos}")
        layer.put(new, pos)
        layer.run(st, tokens=sum(new) + i % 3)   # padded batches, too
        layer.verify(st)
        pos = [p + n for p, n in zip(pos, new)]
        if i == 3:   # of the four drafted tokens one was right
            pos = [p - 3 if n == 4 else p for p, n in zip(pos, new)]
    hip.hipStreamDestroy(st)
    layer.close()


def test_a_captured_step_follows_tables_and_lengths(kxlib):
    """One graph for every step of up to 8 rows: lengths, positions and pages are read when it runs.  Eager calls and synchronizations lie between its replays."""
    hip = Hip(kxlib)
    st, layer = hip.stream(), Layer(kxlib, 3, 8, 4, seed=2)
    layer.put([2, 0, 5], [0, 0, 0])
    layer.run(st)
    layer.verify(st)
    say("capture")
    ready = hip.capture(st, lambda: layer.run(st))
    pos = [2, 0, 5]
    for i, new in enumerate([[1, 1, 1], [2, 3, 3], [0, 8, 0], [1, 1, 1], [1, 0, 1], [2, 2, 4], [1, 1, 1]]):
        say(f"replay {i} of {new} at {pos}")
        layer.put(new, pos)
        hip.hipGraphLaunch(ready, st)
        layer.verify(st)   # reads the cache back with calls outside the graph
        pos = [p + n for p, n in zip(pos, new)]
        if i == 3:
            say("eager")
            layer.put([1, 2, 1], pos)
            layer.run(None)
            layer.verify(None)
            pos = [p + n for p, n in zip(pos, [1, 2, 1])]
    hip.hipGraphExecDestroy(ready)
    hip.hipStreamDestroy(st)
    layer.close()


def test_two_handles_on_two_streams(kxlib):
    hip = Hip(kxlib)
    layers = [Layer(kxlib, 2, 40, 4, seed=s) for s in (3, 4)]
    streams = [hip.stream() for _ in layers]
    pos = [[0, 0], [0, 0]]
    for new in ([30, 3], [1, 1], [1, 30], [1, 1]):
        say(f"two layers, {new}")
        for layer, p in zip(layers, pos):
            layer.put(new, list(p))
        for layer, st in zip(layers, streams):
            layer.run(st, tokens=sum(new))
        for layer, st in zip(layers, streams):
            layer.verify(st)
        pos = [[a + b for a, b in zip(p, new)] for p in pos]
    for layer, st in zip(layers, streams):
        hip.hipStreamDestroy(st)
        layer.close()


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("lens", [[1], [700, 64, 65]], ids=str)
def test_tables_for_caches_beyond_the_last_level(kxlib, f32, lens):
    """What `longest` allows, and not what is there, says that positions are read past the caches."""
    say(f"wide tables {lens} f32={f32}")
    p = S.Paged(kxlib, heads=4, kv=2, dim=128, vdim=100, block=64, batch=len(lens), f32=f32, tokens=sum(lens), seed=7)
    p.append(lens, [0] * len(lens))
    pos, q = [n - 1 for n in lens], p.queries(len(lens))
    got = p.attend([1] * len(lens), pos, q, longest=2 ** 31 - 1, table=p.table(8192))   # 524288 positions of 512 bytes
    y, tol = p.expect([1] * len(lens), pos, q)
    Layer.close_to("attention", got, y, tol)
    assert p.faults() == 0
    p.close()


@pytest.mark.parametrize("shape", [dict(dim=64, vdim=64, rot=64), dict(dim=128, vdim=128, rot=64, pairs=1, block=64), dict(dim=250, vdim=250, rot=250, block=16)], ids=lambda s: str(s["dim"]))
@pytest.mark.parametrize("at", [0, 1, 15, 16, 31, 47, 60, 63])
def test_rows_that_begin_and_end_inside_a_group(kxlib, shape, at):
    """Every place of the first new row among 64, few rows and many, scales that grow and scales that stay."""
    say(f"{shape} from {at}")
    p = S.Paged(kxlib, heads=2, kv=2, batch=6, pages=40, **shape)
    if at:
        p.append([at] * 6, [0] * 6)
    for sigma, new in ((1.0, [1, 2, 4, 5, 17, 64 - at]), (8.0, [1, 2, 4, 5, 17, 70]), (0.1, [4, 4, 60, 1, 3, 2])):
        p.append(new, [len(k) for k in p.k], sigma=sigma)
        for b, (k, v) in enumerate(p.read([len(k) for k in p.k], [0] * 6)):
            np.testing.assert_array_equal(k, p.k[b])
            np.testing.assert_array_equal(v, p.v[b])
    assert p.faults() == 0
    p.close()


def test_rows_read_into_aligned_pieces(kxlib):
    """Results whose rows are whole pieces of 16 bytes, and results whose rows are not, hold the same; nothing beside them is written."""
    say("aligned")
    p = S.Paged(kxlib, heads=2, kv=2, dim=64, vdim=40, block=16, batch=2)
    p.append([100, 3], [0, 0])
    n, pos = [77, 2], [20, 1]
    held = p.read(n, pos)   # rows of 129 and 82
    for k_ld, v_ld in ((128, 80), (136, 96), (132, 88)):
        ok, ov = (DevBuf.from_numpy(np.full((79, ld), 0x1234, np.uint16)) for ld in (k_ld, v_ld))
        check(kxlib.kx_paged_read(p.h, C.byref(p.cache(p.table())), C.byref(p.rows(n, pos)), ok.ptr, k_ld, ov.ptr, v_ld, None))
        check(kxlib.kx_sync(None))
        k, v = ok.to_numpy(np.uint16, (79, k_ld)), ov.to_numpy(np.uint16, (79, v_ld))
        assert (k[:, 128:] == 0x1234).all() and (v[:, 80:] == 0x1234).all()
        np.testing.assert_array_equal(S.bf16(k[:, :128]).reshape(79, 2, 64), np.concatenate([h[0] for h in held]))
        np.testing.assert_array_equal(S.bf16(v[:, :80]).reshape(79, 2, 40), np.concatenate([h[1] for h in held]))
    p.close()


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [dict(dim=64, vdim=64, rot=64), dict(dim=128, vdim=100, rot=64, block=64), dict(dim=192, vdim=128, size=700), dict(dim=200, vdim=256, block=16)], ids=lambda s: str(s["dim"]))
def test_many_rows_behind_many_positions(kxlib, f32, shape):
    """Columns that waves have for themselves, their positions split between workgroups; the same bits again."""
    say(f"many rows {shape} f32={f32}")
    p = S.Paged(kxlib, heads=4, kv=1, batch=2, f32=f32, tokens=2700, pages=60, seed=8, **shape)
    lens, new = [2600, 100], [39, 35]
    p.append(lens, [0, 0])
    pos, q = [n - m for n, m in zip(lens, new)], p.queries(sum(new))
    got = p.attend(new, pos, q)
    y, tol = p.expect(new, pos, q)
    Layer.close_to("attention", got, y, tol)
    for _ in range(3):
        np.testing.assert_array_equal(p.attend(new, pos, q), got)
    assert p.faults() == 0
    p.close()
