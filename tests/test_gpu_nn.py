"""GPU tests (-m gpu) of the operators of a transformer on ciphertexts (include/acehip.h: acehip_linear_i8, acehip_rope*, acehip_linattn_*) against their
formulas in whole numbers of any length: results are canonical residues, so every comparison is for equality, and every word of a result's memory
that the call does not own has to stay as it was."""
import ctypes as C
import itertools

import numpy as np
import pytest

import ace_compiler_amd as A

pytestmark = pytest.mark.gpu

SETS = {  # name: N, L, q0, sf, dnum
    "n16": (16, 10, 60, 59, 3),       # 59- and 60-bit primes: sums are brought back to a residue every few terms
    "n32": (32, 5, 33, 30, 0),        # primes below 2^32
    "n64": (64, 7, 60, 51, 3),
    "n1024": (1024, 5, 60, 55, 2),
    "n2048": (2048, 4, 51, 50, 2),
}
_open = {}


@pytest.fixture(scope="module")
def contexts():
    yield lambda name: _open.setdefault(name, A.AceHip(*SETS[name]))
    for rt in _open.values():
        rt.close()
    _open.clear()


class Block:
    """A matrix of ciphertexts [heads][rows][cols][comps] in device memory of its own: the axes nested in `order` (outermost first), each polynomial
    `level` + K limbs and `pad` words; filled with values that are no residues outside the limbs of the call."""

    def __init__(self, rt, shape, level, limbs, order="hrcp", pad=0, data=None, seed=0, base_pad=0):
        self.rt, self.shape, self.limbs = rt, tuple(shape), limbs
        words = (level + rt.K) * rt.N + pad
        strides, s = {}, words
        for ax in reversed(order):
            strides[ax] = s
            s *= max(1, shape["hrcp".index(ax)])
        self.strides = [strides[ax] for ax in "hrcp"]
        self.base = base_pad
        self.host = np.full(s + base_pad + 5, 0xDEADBEEFDEADBEEF, dtype=np.uint64)
        if data is None:
            rng = np.random.default_rng(seed)
            data = np.stack([rng.integers(0, p, size=(*shape, rt.N), dtype=np.uint64) for p in self.primes(level)], axis=-2)
        if data is not False:
            self.put(self.host, data)
        self.buf = rt.to_device(self.host)
        self.mat = rt.mat(self.buf.ptr + 8 * base_pad, *self.strides)
        self.level = level

    def primes(self, level):
        return [self.rt.primes[p if p < level else self.rt.L + p - level] for p in self.limbs]

    def spots(self, words):
        N = self.rt.N
        for ix in itertools.product(*map(range, self.shape)):
            at = self.base + sum(i * s for i, s in zip(ix, self.strides))
            for k, p in enumerate(self.limbs):
                yield ix, k, words[at + p * N: at + (p + 1) * N]

    def put(self, words, data):
        for ix, k, w in self.spots(words):
            if data[ix][k] is not None:
                w[:] = np.asarray(data[ix][k], dtype=np.uint64)

    def values(self):
        """residues as Python integers, [h][r][c][p][limb][N]"""
        got = np.zeros((*self.shape, len(self.limbs), self.rt.N), dtype=object)
        for ix, k, w in self.spots(self.host):
            got[ix][k] = w.astype(object)
        return got

    def q(self):
        return np.array(self.primes(self.level), dtype=object)[:, None]

    def check(self, want, written=None):
        """the memory holds `want` (where written) and nothing else has changed"""
        expect = self.host.copy()
        for ix, k, w in self.spots(expect):
            if written is None or written(ix):
                w[:] = want[ix][k].astype(np.uint64)
        got = self.buf.download()
        bad = np.flatnonzero(got != expect)
        assert bad.size == 0, "%d words differ, first at %d: %x for %x" % (bad.size, bad[0], got[bad[0]], expect[bad[0]])

    def free(self):
        self.buf.free()


def extreme(rt, shape, level, limbs, kind):
    """all residues q - 1, or 0 and q - 1 in turn"""
    p = np.array([rt.primes[x if x < level else rt.L + x - level] for x in limbs], dtype=np.uint64)[:, None]
    d = np.broadcast_to(p - np.uint64(1), (*shape, len(limbs), rt.N)).copy()
    if kind == "alternate":
        d[..., ::2] = 0
    return d


def dev(rt, arr):
    return rt.to_device(np.ascontiguousarray(arr))


# ---- linear layers ---------------------------------------------------------------------------------------------------------------------
def linear_case(rt, level, limbs, rows, n_in, n_out, n_comp, mul=False, tok=False, order="hrcp", pad=0, kind=None, ld=None, w_off=0, seed=1, weights=None, tok_stride=None):
    rng = np.random.default_rng(seed)
    shape = (1, rows, n_in, n_comp)
    x = Block(rt, shape, level, limbs, order, pad, data=extreme(rt, shape, level, limbs, kind) if kind else None, seed=seed)
    y = Block(rt, (1, rows, n_out, n_comp), level, limbs, order, pad, data=False)
    ld = ld or n_in
    w = rng.integers(-128, 128, size=(n_out, ld)).astype(np.int8) if weights is None else np.full((n_out, ld), weights, np.int8)
    dw = dev(rt, np.concatenate([np.zeros(w_off, np.int8), w.ravel(), np.zeros(1, np.int8)]))
    m = rng.integers(-(1 << 62), 1 << 62, size=n_out) if mul else None
    if mul:
        m[:3] = [-(1 << 63), (1 << 63) - 1, 0][: len(m)]
    dm = dev(rt, m) if mul else None
    t = Block(rt, (1, rows, 1, 1), level, limbs, seed=seed + 7) if tok else None
    shared = tok and tok_stride == 0
    rt.linear_i8(y.mat, x.mat, dw.ptr + w_off, ld, rows, n_in, n_out, n_comp, level, pos0=limbs[0], n_limbs=len(limbs), d_mul=dm.ptr if mul else None,
                 d_tok=t.buf.ptr if tok else None, tok_stride=(0 if shared else t.strides[1]) if tok else 0)
    v = x.values()[0]                                                   # [r][i][p][limb][N]
    want = np.tensordot(w[:, :n_in].astype(object), v, (1, 1)).swapaxes(0, 1) if n_in else np.zeros((rows, n_out, n_comp, len(limbs), rt.N), dtype=object)
    if mul:
        want = want * np.array([int(a) for a in m], dtype=object)[:, None, None, None]
    if tok:
        tv = t.values()[0, :, 0, 0]
        want = want * (tv[:1] if shared else tv)[:, None, None]
    y.check(want[None] % y.q())
    for b in filter(None, (x, y, t, dw, dm)):
        b.free()


@pytest.mark.parametrize("name,level,limbs", [("n16", 5, [0, 1, 2, 3, 4]), ("n16", 4, [3, 4, 5]), ("n32", 4, [0, 1, 2, 3, 4]), ("n64", 3, [0, 1, 2]), ("n64", 7, [6, 7, 8]), ("n1024", 2, [0, 1]),
                                              ("n2048", 2, [0, 1])])
@pytest.mark.parametrize("n_in,n_out", [(1, 1), (5, 3), (64, 16), (65, 33), (130, 70)])
def test_linear_shapes(contexts, name, level, limbs, n_in, n_out):
    rt = contexts(name)
    if rt.N >= 1024 and n_in > 65:
        n_in, n_out = 67, 35
    linear_case(rt, level, limbs, 1, n_in, n_out, 2)


@pytest.mark.parametrize("n_in,n_out", [(1, 300), (300, 1), (257, 129), (63, 257), (128, 128), (192, 65), (65, 200), (70, 32), (64, 385)])
@pytest.mark.parametrize("mul,tok", [(True, False), (False, True), (True, True)])
def test_linear_tiles_and_scales(contexts, n_in, n_out, mul, tok):
    linear_case(contexts("n64"), 2, [0, 1], 2, n_in, n_out, 1, mul, tok)


@pytest.mark.parametrize("order", ["hrcp", "hcrp", "hpcr", "prch"])
@pytest.mark.parametrize("pad", [0, 3])
def test_linear_layouts(contexts, order, pad):
    linear_case(contexts("n64"), 3, [1, 2], 3, 20, 9, 3, True, True, order, pad)
    linear_case(contexts("n1024"), 1, [0], 2, 20, 9, 2, True, True, order, pad, tok_stride=0)


@pytest.mark.parametrize("ld,w_off", [(70, 0), (71, 1), (80, 16), (77, 3)])
def test_linear_weights_of_any_alignment(contexts, ld, w_off):
    linear_case(contexts("n64"), 2, [0, 1], 1, 70, 40, 2, ld=ld, w_off=w_off)


@pytest.mark.parametrize("name", ["n16", "n32", "n64", "n1024"])
@pytest.mark.parametrize("weights", [-128, 127])
@pytest.mark.parametrize("kind", ["top", "alternate"])
def test_linear_extremes(contexts, name, weights, kind):
    rt = contexts(name)
    n_in = 600 if rt.N < 1024 else 96
    linear_case(rt, 2, [0, 1, 2], 1, n_in, 2, 1, weights=weights, kind=kind)


def test_linear_longest_sum(contexts):
    """ACEHIP_LINEAR_MAX_IN inputs of q - 1 by -128: the column stride is zero, so that one polynomial stands for all"""
    rt = contexts("n16")
    x = Block(rt, (1, 1, 1, 1), 2, [0, 1], data=extreme(rt, (1, 1, 1, 1), 2, [0, 1], "top"))
    x.mat.col_stride = 0
    for wv in (-128, 127):
        y = Block(rt, (1, 1, 17, 1), 2, [0, 1], data=False)
        w = dev(rt, np.full((17, 65536), wv, np.int8))
        rt.linear_i8(y.mat, x.mat, w.ptr, 65536, 1, 65536, 17, 1, 2)
        y.check(np.broadcast_to(65536 * wv * x.values() % x.q(), (1, 1, 17, 1, 2, rt.N)))
        w.free()
        y.free()
    x.free()


def mul_mod(a, b, q):
    """a * b mod q for uint64 a, b < q < 2^61: quotient from a product in 64 bits of mantissa, at most one off"""
    f = np.floor(a.astype(np.longdouble) * b.astype(np.longdouble) / q.astype(np.longdouble)).astype(np.uint64)
    r = (a * b - f * q).astype(np.int64)
    q = q.astype(np.int64)
    r = np.where(r < 0, r + q, r)
    return np.where(r >= q, r - q, r).astype(np.uint64)


@pytest.mark.parametrize("n_in,n_out,rows,n_comp", [(65, 257, 1, 2), (40, 300, 1, 2), (129, 144, 3, 1), (192, 260, 1, 3), (3, 33, 5, 3), (65, 250, 1, 2), (40, 96, 2, 2), (70, 20, 3, 2)])
def test_linear_many_column_blocks(contexts, n_in, n_out, rows, n_comp):
    """large enough a ring that a workgroup takes several column blocks, across polynomials and rows"""
    rt = _open.setdefault("n16384", A.AceHip(16384, 2, 60, 50, 1))
    level, limbs, N = 2, [0, 1, 2], rt.N
    q = np.array([rt.primes[i] for i in range(3)], dtype=np.uint64)[:, None]
    rng = np.random.default_rng(n_in)
    x = np.stack([rng.integers(0, p[0], size=(rows, n_in, n_comp, N), dtype=np.uint64) for p in q], axis=-2)   # [row][i][comp][limb][N]
    w, m = rng.integers(-128, 128, size=(n_out, n_in)).astype(np.int8), rng.integers(-(1 << 62), 1 << 62, size=n_out)
    tok = np.stack([rng.integers(0, p[0], size=(rows, N), dtype=np.uint64) for p in q], axis=-2)
    dx, dw, dm, dt, dy = dev(rt, x), dev(rt, w), dev(rt, m), dev(rt, tok), dev(rt, np.full((rows, n_out, n_comp, 3, N), 7, np.uint64))
    strides = lambda n: dict(row=n * n_comp * 3 * N, col=n_comp * 3 * N, comp=3 * N)
    rt.linear_i8(rt.mat(dy.ptr, **strides(n_out)), rt.mat(dx.ptr, **strides(n_in)), dw.ptr, n_in, rows, n_in, n_out, n_comp, level, n_limbs=3, d_mul=dm.ptr, d_tok=dt.ptr,
                 tok_stride=3 * N)
    some = np.unique(np.concatenate([[0, n_out - 1], rng.integers(0, n_out, size=14)]))   # outputs that are compared
    got = dy.download((rows, n_out, n_comp, 3, N))[:, some]
    w, m, n_out = w[some], m[some], len(some)
    flat = x.transpose(1, 0, 2, 3, 4).reshape(n_in, -1)
    parts = [(w.astype(np.float64) @ (flat >> np.uint64(s) & np.uint64((1 << 20) - 1)).astype(np.float64)).astype(np.int64) for s in (0, 20, 40)]   # exact: below 2^38
    parts = [p.reshape(n_out, rows, n_comp, 3, N) for p in parts]
    qi = q.astype(np.int64)
    y = np.zeros_like(parts[0], dtype=np.uint64)
    for p in parts[::-1]:
        y = ((mul_mod(y, np.broadcast_to(np.uint64(1 << 20), y.shape), q) + (p % qi).astype(np.uint64)) % q).astype(np.uint64)
    factor = np.array([[int(a) % int(b) for b in q[:, 0]] for a in m], dtype=np.uint64)
    y = mul_mod(mul_mod(y, np.broadcast_to(factor[:, None, None, :, None], y.shape), q), np.broadcast_to(tok[None, :, None], y.shape), q)
    assert np.array_equal(got, y.transpose(1, 0, 2, 3, 4))
    for d in (dx, dw, dm, dt, dy):
        d.free()


@pytest.mark.parametrize("apart", [(1 << 22) + 64, (1 << 24) - 192 - 64, 1 << 24])
def test_linear_far_inputs(contexts, apart):
    """ciphertexts 32 and 128 MiB apart"""
    linear_case(contexts("n64"), 3, [0, 1, 2], 1, 3, 2, 1, True, pad=apart)


@pytest.mark.parametrize("same", ["row", "col", "comp", "all"])
@pytest.mark.parametrize("n_in,n_out", [(5, 3), (70, 40)])
def test_linear_shared_inputs(contexts, same, n_in, n_out):
    """strides of zero: one row, one input or one polynomial for all"""
    rt = contexts("n64")
    level, limbs, rows, comps = 3, [0, 1, 2], 2, 2
    shape = dict(row=rows, col=n_in, comp=comps)
    shape = {k: 1 if same in (k, "all") else n for k, n in shape.items()}
    x = Block(rt, (1, *shape.values()), level, limbs)
    strides = {k: 0 if shape[k] == 1 else s for k, s in zip(shape, x.strides[1:])}
    y = Block(rt, (1, rows, n_out, comps), level, limbs, data=False)
    w = np.random.default_rng(8).integers(-128, 128, size=(n_out, n_in)).astype(np.int8)
    dw = dev(rt, w)
    rt.linear_i8(y.mat, rt.mat(x.buf.ptr, **strides), dw.ptr, n_in, rows, n_in, n_out, comps, level)
    v = np.broadcast_to(x.values()[0], (rows, n_in, comps, len(limbs), rt.N))
    y.check(np.tensordot(w.astype(object), v, (1, 1)).swapaxes(0, 1)[None] % y.q())
    for b in (x, y, dw):
        b.free()


@pytest.mark.parametrize("n_out", [512, 600, 1030])
def test_linear_weights_in_parts(contexts, n_out):
    """as many packed weights as the workspace holds (512 outputs), or more"""
    rt = contexts("n64")
    assert 32 * 1024 <= rt.lib.acehip_workspace_words(rt.h) * 8 < 38 * 1024
    linear_case(rt, 2, [0, 1], 12, 3, n_out, 3, mul=True)


def test_linear_empty_sum_is_zero(contexts):
    linear_case(contexts("n64"), 2, [0, 1], 1, 0, 5, 2, True, True)


# ---- rotary positions ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n_pos,n_pairs,n_axes", [(1, 1, 1), (3, 300, 3), (1000, 17, 2), (257, 8, 8)])
def test_rope_messages(contexts, n_pos, n_pairs, n_axes):
    rt = contexts("n64")
    rng = np.random.default_rng(n_pos)
    pos = np.concatenate([rng.integers(0, 1 << 21, size=(n_axes, n_pos)).astype(np.float64), np.zeros((n_axes, 2))], axis=1)
    freq, axis = [float(10000.0 ** (-i / n_pairs)) for i in range(n_pairs)], [int(a) for a in rng.integers(0, n_axes, n_pairs)]
    stride = n_pos + 3
    d_pos, d_cos, d_sin = dev(rt, pos), dev(rt, np.full(n_pairs * stride, 7.0)), dev(rt, np.full(n_pairs * stride, 7.0))
    rt.rope_messages(d_cos.ptr, d_sin.ptr, stride, d_pos.ptr, n_pos + 2, n_pos, freq, axis, n_axes)
    angle = (pos[axis, :n_pos] * np.array(freq)[:, None]).astype(np.longdouble)
    for d, f in ((d_cos, np.cos), (d_sin, np.sin)):
        got = d.download((n_pairs, stride))
        assert np.all(got[:, n_pos:] == 7.0)
        # the device's double sine and cosine are within 2 units in the last place; one is at most 2^-53 for values up to 1
        assert np.max(np.abs(got[:, :n_pos] - f(angle).astype(np.float64))) <= 2 * 2.0**-53 + 2.0**-54
    for d in (d_pos, d_cos, d_sin):
        d.free()


def rope_case(rt, level, limbs, heads, rows, dim, n_comp, interleaved=False, order="hrcp", pad=0, in_place=False, shared_rows=False, kind=None, seed=3):
    shape = (heads, rows, dim, n_comp)
    x = Block(rt, shape, level, limbs, order, pad, seed=seed, data=extreme(rt, shape, level, limbs, kind) if kind else None)
    y = x if in_place else Block(rt, shape, level, limbs, order, pad, data=False)
    tabs = [Block(rt, (1, rows, dim // 2, 1), level, limbs, seed=seed + 1 + t, data=extreme(rt, (1, rows, dim // 2, 1), level, limbs, kind) if kind else None) for t in (0, 1)]
    rt.rope(y.mat, x.mat, tabs[0].buf.ptr, tabs[1].buf.ptr, tabs[0].strides[2], 0 if shared_rows else tabs[0].strides[1], heads, rows, dim, n_comp, level, pos0=limbs[0],
            n_limbs=len(limbs), interleaved=interleaved)
    v = x.values()
    c, s = (t.values()[:, :, :, 0] for t in tabs)
    if shared_rows:
        c, s = c[:, :1], s[:, :1]
    want = np.zeros_like(v)
    for i in range(dim // 2):
        f0, f1 = (2 * i, 2 * i + 1) if interleaved else (i, i + dim // 2)
        ci, si = c[:, :, i, None], s[:, :, i, None]
        want[:, :, f0] = v[:, :, f0] * ci - v[:, :, f1] * si
        want[:, :, f1] = v[:, :, f0] * si + v[:, :, f1] * ci
    y.check(want % y.q())
    for b in {x, y, *tabs}:
        b.free()


@pytest.mark.parametrize("name,level,limbs", [("n16", 4, [0, 1, 2, 3]), ("n16", 3, [2, 3, 4]), ("n32", 3, [0, 1, 2, 3]), ("n64", 3, [1, 2]), ("n1024", 2, [0, 1, 2]), ("n2048", 1, [0])])
@pytest.mark.parametrize("heads,rows,dim,n_comp", [(1, 1, 2, 1), (2, 3, 6, 2), (5, 1, 10, 2), (3, 2, 4, 3), (11, 1, 2, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(contexts, name, level, limbs, heads, rows, dim, n_comp, interleaved):
    rope_case(contexts(name), level, limbs, heads, rows, dim, n_comp, interleaved)


@pytest.mark.parametrize("order,pad", [("hrcp", 1), ("rchp", 0), ("pcrh", 5)])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("shared_rows", [False, True])
def test_rope_layouts(contexts, order, pad, in_place, shared_rows):
    rope_case(contexts("n64"), 3, [0, 1, 2], 2, 3, 8, 2, order=order, pad=pad, in_place=in_place, shared_rows=shared_rows)


@pytest.mark.parametrize("name", ["n16", "n32", "n64", "n2048"])
@pytest.mark.parametrize("kind", ["top", "alternate"])
def test_rope_extremes(contexts, name, kind):
    rope_case(contexts(name), 2, [0, 1, 2], 1, 1, 4, 2, kind=kind)


@pytest.mark.parametrize("dim", [12, 6, 2])
def test_rope_in_large_launches(dim):
    """a ring of 16384: one workgroup for all heads of a pair, or several"""
    rt = _open.setdefault("n16384", A.AceHip(16384, 2, 60, 50, 1))
    heads, comps, N = 3, 2, rt.N
    q = np.array([rt.primes[i] for i in range(3)], dtype=np.uint64)[:, None]
    rng = np.random.default_rng(dim)
    draw = lambda *shape: np.stack([rng.integers(0, p[0], size=(*shape, N), dtype=np.uint64) for p in q], axis=-2)
    x, c, s = draw(heads, dim, comps), draw(dim // 2, 1), draw(dim // 2, 1)
    dx, dc, ds, dy = (dev(rt, v) for v in (x, c, s, np.full_like(x, 7)))
    strides = dict(head=dim * comps * 3 * N, col=comps * 3 * N, comp=3 * N)
    rt.rope(rt.mat(dy.ptr, **strides), rt.mat(dx.ptr, **strides), dc.ptr, ds.ptr, 3 * N, 0, heads, 1, dim, comps, 2, n_limbs=3)
    x0, x1 = x[:, :dim // 2], x[:, dim // 2:]
    full = lambda v: np.broadcast_to(v, x0.shape)
    y0 = (mul_mod(x0, full(c), q) + q - mul_mod(x1, full(s), q)) % q
    y1 = (mul_mod(x0, full(s), q) + mul_mod(x1, full(c), q)) % q
    assert np.array_equal(dy.download(x.shape), np.concatenate([y0, y1], axis=1))
    for d in (dx, dc, ds, dy):
        d.free()


# ---- linear attention ------------------------------------------------------------------------------------------------------------------
def pair(a, b):
    """product of two ciphertexts [2][limb][N] before relinearisation"""
    return np.stack([a[0] * b[0], a[0] * b[1] + a[1] * b[0], a[1] * b[1]])


def factors(rng, *shape):
    f = rng.integers(-(1 << 62), 1 << 62, size=shape)
    f.ravel()[:2] = [-(1 << 63), (1 << 63) - 1][: f.size]
    return f, np.vectorize(int, otypes=[object])(f) if f.size else f.astype(object)


class Attn:
    """operands of the three calls for one set of sizes"""

    Block = Block

    def __init__(self, rt, level, limbs, H, kv, nq, nk, dk, dv, orders=("hrcp",) * 6, pad=0, kind=None, seed=5, factor=True):
        self.rt, self.level, self.limbs, self.sizes = rt, level, limbs, (H, kv, nq, nk, dk, dv)
        self.n = rt.N
        rng = np.random.default_rng(seed)
        b = iter(range(100))

        def block(*shape, order):
            return self.Block(rt, shape, level, limbs, order, pad, seed=seed + next(b), data=extreme(rt, shape, level, limbs, kind) if kind else None)

        self.q = block(H, nq, dk, 2, order=orders[0])
        self.k = block(kv, nk, dk, 2, order=orders[1])
        self.v = block(kv, nk, dv, 2, order=orders[2])
        self.S = block(H, dk, dv, 2, order=orders[3])
        self.p = block(H, nq, nk, 2, order=orders[4])
        self.order = orders[5]
        self.pad = pad
        self.din, self.din_i = factors(rng, H, nq)
        self.dec, self.dec_i = factors(rng, H, nk)
        self.keep, self.keep_i = factors(rng, H)
        self.dd = [dev(rt, f) if f.size else None for f in (self.din, self.dec, self.keep)]

    def result(self, *shape):
        return self.Block(self.rt, (*shape, 3), self.level, self.limbs, self.order, self.pad, data=False)

    def range(self):
        return dict(pos0=self.limbs[0], n_limbs=len(self.limbs))

    def ptr(self, i, on=True):
        return self.dd[i].ptr if on and self.dd[i] else None

    def scores(self, causal=True):
        H, kv, nq, nk, dk, dv = self.sizes
        y = self.result(H, nq, nk)
        self.rt.linattn_scores(y.mat, self.q.mat, self.k.mat, H, kv, nq, nk, dk, self.level, causal=causal, **self.range())
        q, k = self.q.values(), self.k.values()
        want = np.zeros((H, nq, nk, 3, len(self.limbs), self.n), dtype=object)
        for h, t, s in itertools.product(range(H), range(nq), range(nk)):
            want[h, t, s] = sum((pair(q[h, t, a], k[h * kv // H, s, a]) for a in range(dk)), want[h, t, s]) % y.q()
        y.check(want, (lambda ix: ix[2] <= ix[1] + nk - nq) if causal else None)
        y.free()

    def out(self, state=True, chunk=True, causal=True, factor=True):
        H, kv, nq, nk, dk, dv = self.sizes
        y = self.result(H, nq, dv)
        dec = factor and causal
        self.rt.linattn_out(y.mat, self.q.mat if state else None, self.S.mat if state else None, self.p.mat if chunk else None, self.v.mat if chunk else None, H, kv, nq, nk,
                            dk, dv, self.level, d_in=self.ptr(0, factor), d_decay=self.ptr(1, dec), causal=causal, **self.range())
        q, S, p, v = self.q.values(), self.S.values(), self.p.values(), self.v.values()
        want = np.zeros((H, nq, dv, 3, len(self.limbs), self.n), dtype=object)
        for h, t, b in itertools.product(range(H), range(nq), range(dv)):
            r = want[h, t, b]
            if state:
                r = r + (self.din_i[h, t] if factor else 1) * sum((pair(q[h, t, a], S[h, a, b]) for a in range(dk)), r)
            if chunk:
                for s in range(nk):
                    d = t + nk - nq - s
                    if d >= 0 or not causal:
                        r = r + (self.dec_i[h, d] if dec else 1) * pair(p[h, t, s], v[h * kv // H, s, b])
            want[h, t, b] = r % y.q()
        y.check(want)
        y.free()

    def state(self, kept=True, factor=True, in_place=False):
        H, kv, nq, nk, dk, dv = self.sizes
        y = self.result(H, dk, dv)
        S = self.S
        if in_place:
            S = self.Block(self.rt, (H, dk, dv, 3), self.level, self.limbs, self.order, self.pad, seed=99)
            y.free()
            y = S
        self.rt.linattn_state(y.mat, S.mat if kept else None, self.k.mat, self.v.mat, H, kv, nk, dk, dv, self.level, d_keep=self.ptr(2, factor), d_decay=self.ptr(1, factor),
                              **self.range())
        Sv, k, v = S.values(), self.k.values(), self.v.values()
        want = np.zeros((H, dk, dv, 3, len(self.limbs), self.n), dtype=object)
        for h, a, b in itertools.product(range(H), range(dk), range(dv)):
            r = want[h, a, b].copy()
            for s in range(nk):
                r = r + (self.dec_i[h, nk - 1 - s] if factor else 1) * pair(k[h * kv // H, s, a], v[h * kv // H, s, b])
            if kept:
                r[:2] = r[:2] + (self.keep_i[h] if factor else 1) * Sv[h, a, b, :2]
            want[h, a, b] = r % y.q()
        y.check(want)
        y.free()

    def free(self):
        for b in (self.q, self.k, self.v, self.S, self.p, *filter(None, self.dd)):
            b.free()


SIZES = [  # heads, kv heads, queries, keys, dk, dv
    (1, 1, 1, 1, 1, 1), (2, 1, 1, 1, 5, 3), (2, 2, 4, 4, 4, 4), (4, 2, 3, 3, 5, 7), (3, 1, 5, 5, 2, 9), (1, 1, 2, 6, 3, 4), (2, 1, 6, 2, 3, 5), (1, 1, 9, 9, 1, 1), (6, 3, 1, 4, 8, 8),
]


@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("name,level,limbs", [("n16", 4, [0, 1, 2, 3]), ("n32", 3, [0, 1, 2, 3]), ("n64", 5, [3, 4, 5])])
def test_linear_attention(contexts, name, level, limbs, sizes):
    a = Attn(contexts(name), level, limbs, *sizes)
    a.scores()
    a.scores(causal=False)
    a.out()
    a.out(causal=False)
    a.out(state=False)
    a.out(chunk=False)
    a.out(factor=False)
    a.state()
    a.state(kept=False)
    a.state(factor=False)
    a.state(in_place=True)
    a.free()


@pytest.mark.parametrize("name,level,limbs", [("n1024", 2, [0, 1, 2]), ("n2048", 2, [0, 1])])
@pytest.mark.parametrize("sizes", [(2, 1, 3, 3, 4, 5), (1, 1, 1, 1, 9, 6)], ids=str)
def test_linear_attention_larger_rings(contexts, name, level, limbs, sizes):
    a = Attn(contexts(name), level, limbs, *sizes)
    a.scores()
    a.out()
    a.state()
    a.free()


@pytest.mark.parametrize("name", ["n16", "n32", "n64", "n2048"])
@pytest.mark.parametrize("kind", ["top", "alternate"])
@pytest.mark.parametrize("factor", [False, True])
def test_linear_attention_extremes(contexts, name, kind, factor):
    """long sums of products of q - 1"""
    rt = contexts(name)
    limbs = [0, 1, 2]
    n = 70 if rt.N <= 64 else 9
    a = Attn(rt, 2, limbs, 1, 1, 2, n, n, 2, kind=kind)
    a.scores()
    a.out(factor=factor)
    a.state(factor=factor)
    a.free()


class Sampled(Block):
    """of a large ring, compared at some coefficients"""

    AT = np.array([0, 1, 62, 63, 64, 255, 256, 4097, 9999, 16382, 16383])

    def values(self):
        got = np.zeros((*self.shape, len(self.limbs), len(self.AT)), dtype=object)
        for ix, k, w in self.spots(self.host):
            got[ix][k] = w[self.AT].astype(object)
        return got

    def check(self, want, written=None):
        got = self.buf.download()
        for (ix, k, w), (_, _, before) in zip(self.spots(got), self.spots(self.host)):
            if written is None or written(ix):
                assert np.array_equal(w[self.AT], want[ix][k].astype(np.uint64)), (ix, k)
                w[:] = before
        assert np.array_equal(got, self.host)


class LargeAttn(Attn):
    Block = Sampled

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.n = len(self.Block.AT)


class Sampled1024(Sampled):
    AT = np.array([0, 1, 63, 64, 500, 1023])


class MiddleAttn(LargeAttn):
    Block = Sampled1024


@pytest.mark.parametrize("sizes,kind", [((2, 1, 1, 1, 5, 18), None), ((2, 1, 3, 4, 3, 9), None), ((2, 1, 9, 9, 10, 6), None), ((1, 1, 5, 66, 2, 5), None), ((1, 1, 6, 17, 33, 5), "top"),
                                        ((1, 1, 1, 20, 33, 17), "top"), ((1, 1, 4, 9, 20, 4), "alternate"), ((2, 2, 13, 6, 9, 4), None)], ids=str)
def test_linear_attention_in_large_launches(sizes, kind):
    """a launch that fills the card (a ring of 16384): rows, small and large sets of results, sums over many terms"""
    rt = _open.setdefault("n16384", A.AceHip(16384, 2, 60, 50, 1))
    a = LargeAttn(rt, 2, [0, 1, 2], *sizes, kind=kind)
    a.scores()
    a.scores(causal=False)
    a.out()
    a.out(causal=False)
    a.out(state=False, factor=False)
    a.state()
    a.state(factor=False)
    a.state(in_place=True)
    a.free()


@pytest.mark.parametrize("name,args", [("n1024_60", (1024, 2, 60, 59, 1)), ("n1024_56", (1024, 2, 60, 56, 1)), ("n1024", SETS["n1024"])])
@pytest.mark.parametrize("sizes,kind", [((1, 1, 9, 9, 20, 10), None), ((2, 1, 7, 10, 13, 11), "top"), ((3, 1, 1, 70, 66, 15), None), ((1, 1, 2, 33, 40, 3), "top"), ((2, 1, 1, 1, 17, 31), None)],
                         ids=str)
def test_linear_attention_in_middle_launches(name, args, sizes, kind):
    """launches that do not fill the card: sums cut over the waves of a workgroup, small tiles"""
    rt = _open.setdefault(name, A.AceHip(*args))
    a = MiddleAttn(rt, 2, [0, 1], *sizes, kind=kind)
    a.scores()
    a.scores(causal=False)
    a.out()
    a.out(causal=False)
    a.out(state=False, factor=False)
    a.state()
    a.state(kept=False)
    a.state(in_place=True)
    a.free()


@pytest.mark.parametrize("kind", [None, "top"])
@pytest.mark.parametrize("sizes", [(1, 1, 5, 40, 17, 5), (1, 1, 2, 70, 40, 3)], ids=str)
def test_linear_attention_long_sums_at_56_bits(sizes, kind):
    """factors staged without their last reduction, sums that carry in between, row factors at the end of a sum or at its terms"""
    for name, cls in (("n16384_56", LargeAttn), ("n1024_56", Attn)):
        rt = _open.setdefault(name, A.AceHip(16384 if cls is LargeAttn else 1024, 2, 60, 56, 1))
        a = cls(rt, 2, [0, 1], *(sizes if cls is LargeAttn else (1, 1, 2, 40, 17, 2)), kind=kind)
        a.out()
        a.out(causal=False)
        a.state()
        a.free()


@pytest.mark.parametrize("orders", [("rhcp",) * 6, ("pcrh",) * 6, ("rhcp", "cprh", "rhcp", "hcrp", "hprc", "hrpc")], ids=str)
@pytest.mark.parametrize("pad", [0, 1])
def test_linear_attention_layouts(contexts, orders, pad):
    a = Attn(contexts("n64"), 3, [1, 2], 4, 2, 3, 4, 3, 5, orders=orders, pad=pad)
    a.scores()
    a.out()
    a.state()
    a.state(in_place=True)
    a.free()


def test_linear_attention_empty_sums(contexts):
    """no keys, no features, rows that see nothing: zeros, and the state as it was kept"""
    rt = contexts("n64")
    a = Attn(rt, 2, [0, 1], 2, 1, 3, 1, 2, 2)
    H, kv, nq, nk, dk, dv = a.sizes
    zero = lambda y: np.zeros((*y.shape, 2, rt.N), dtype=object)
    y = a.result(H, nq, nk)
    rt.linattn_scores(y.mat, a.q.mat, a.k.mat, H, kv, nq, nk, 0, 2, causal=False)
    y.check(zero(y))
    y.free()
    y = a.result(H, nq, dv)
    rt.linattn_out(y.mat, None, None, None, None, H, kv, nq, nk, dk, dv, 2)
    y.check(zero(y))
    rt.linattn_out(y.mat, a.q.mat, a.S.mat, a.p.mat, a.v.mat, H, kv, nq, 0, 0, dv, 2)
    y.check(zero(y))
    y.free()
    y = a.result(H, dk, dv)
    rt.linattn_state(y.mat, a.S.mat, a.k.mat, a.v.mat, H, kv, 0, dk, dv, 2, d_keep=a.ptr(2))
    want = zero(y)
    want[:, :, :, :2] = a.S.values() * a.keep_i[:, None, None, None, None, None] % y.q()
    y.check(want)
    y.free()
    a.free()


# ---- contexts, streams, graphs, replicas -----------------------------------------------------------------------------------------------


def hip():
    lib = C.CDLL("libamdhip64.so")
    lib.hipStreamCreateWithFlags.argtypes = [C.POINTER(C.c_void_p), C.c_uint]
    lib.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    lib.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    lib.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
    lib.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    lib.hipStreamSynchronize.argtypes = lib.hipGraphDestroy.argtypes = lib.hipGraphExecDestroy.argtypes = lib.hipStreamDestroy.argtypes = [C.c_void_p]
    return lib


def ok(rc):
    assert rc == 0, rc


def test_captured_and_replayed(contexts):
    """a chunk's calls in one graph on a stream of its own, replayed on new inputs in the same memory, other work of the library in between"""
    rt = contexts("n64")
    lib = hip()
    H, kv, nq, nk, dk, dv, level = 2, 1, 3, 3, 4, 5, 2
    a = Attn(rt, level, [0, 1], H, kv, nq, nk, dk, dv, factor=True)
    w = np.arange(-20, 20, dtype=np.int8)[: dk * dk].reshape(dk, dk)
    dw = dev(rt, w)
    lin, p3, o3, s3 = (Block(rt, s, level, [0, 1], data=False) for s in ((H, nq, dk, 2), (H, nq, nk, 3), (H, nq, dv, 3), (H, dk, dv, 3)))
    st, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    ok(lib.hipStreamCreateWithFlags(C.byref(st), 1))

    def calls(stream):
        for h in range(H):
            lm, qm = (rt.mat(b.buf.ptr + 8 * h * b.strides[0], 0, *b.strides[1:]) for b in (lin, a.q))
            rt.linear_i8(lm, qm, dw.ptr, dk, nq, dk, dk, 2, level, stream=stream)
        rt.linattn_scores(p3.mat, lin.mat, a.k.mat, H, kv, nq, nk, dk, level, causal=False, stream=stream)
        rt.linattn_out(o3.mat, lin.mat, a.S.mat, a.p.mat, a.v.mat, H, kv, nq, nk, dk, dv, level, d_in=a.ptr(0), d_decay=a.ptr(1), stream=stream)
        rt.linattn_state(s3.mat, a.S.mat, a.k.mat, a.v.mat, H, kv, nk, dk, dv, level, d_keep=a.ptr(2), d_decay=a.ptr(1), stream=stream)

    ok(lib.hipStreamBeginCapture(st, 1))  # thread-local
    calls(st)
    ok(lib.hipStreamEndCapture(st, C.byref(graph)))
    ok(lib.hipGraphInstantiate(C.byref(run), graph, None, None, 0))
    rng = np.random.default_rng(1)
    for _ in range(4):
        for b in (a.q, a.k, a.v, a.S, a.p):
            b.put(b.host, np.stack([rng.integers(0, p, size=(*b.shape, rt.N), dtype=np.uint64) for p in b.primes(level)], axis=-2))
            b.buf.upload(b.host)
        rt.sync()
        ok(lib.hipGraphLaunch(run, st))
        ok(lib.hipStreamSynchronize(st))
        got = [b.buf.download() for b in (lin, p3, o3, s3)]
        for b in (lin, p3, o3, s3):
            b.buf.upload(b.host)
        calls(None)
        rt.sync()
        for b, g in zip((lin, p3, o3, s3), got):
            assert np.array_equal(b.buf.download(), g) and not np.array_equal(g, b.host)
    a.out()
    a.state()
    ok(lib.hipGraphExecDestroy(run))
    ok(lib.hipGraphDestroy(graph))
    ok(lib.hipStreamDestroy(st))
    for b in (a, lin, p3, o3, s3, dw):
        b.free()



def test_replicas(contexts):
    """operands in the arena follow the selected replicas, weights and plaintexts outside it are shared; a result outside the arena is refused"""
    N, L = 64, 4
    rt = A.AceHip(N, L, 60, 50, 2)
    level, n_rep, dim = 3, 3, 4
    poly = level * N
    words = 1 << 16
    ws = int(rt.lib.acehip_workspace_words(rt.h))
    total = words + ws + 64 * N
    base = rt.buf(total * n_rep)
    cfg = A.binding.ArenaCfg(base.ptr, total * 8, total * 8, n_rep, base.ptr + 8 * words, base.ptr + 8 * (words + ws), 64)
    rt.check(rt.lib.acehip_ctx_set_arena(rt.h, C.byref(cfg)))
    rng = np.random.default_rng(2)
    x = np.stack([np.stack([rng.integers(0, rt.primes[p], size=(n_rep, dim, 2, N), dtype=np.uint64) for p in range(level)], axis=-2)])[0]   # [rep][i][comp][limb][N]
    host = np.zeros((n_rep, total), np.uint64)
    host[:, : dim * 2 * poly] = x.reshape(n_rep, -1)
    base.upload(host)
    xm = rt.mat(base.ptr, 0, 0, 2 * poly, poly)
    y_at, z_at = 8192, 16384
    ym = rt.mat(base.ptr + 8 * y_at, 0, 0, 2 * poly, poly)
    zm = rt.mat(base.ptr + 8 * z_at, dim * dim * 3 * poly, dim * 3 * poly, 3 * poly, poly)
    w = rng.integers(-128, 128, size=(dim, dim)).astype(np.int8)
    dw = dev(rt, w)
    tab = Block(rt, (1, 1, dim // 2, 1), level, list(range(level)), seed=4)
    rt.check(rt.lib.acehip_ctx_select(rt.h, 1, 2))
    rt.linear_i8(ym, xm, dw.ptr, dim, 1, dim, dim, 2, level)
    rt.rope(ym, ym, tab.buf.ptr, tab.buf.ptr, tab.strides[2], 0, 1, 1, dim, 2, level)
    rt.linattn_scores(zm, rt.mat(base.ptr + 8 * y_at, 0, 2 * poly, 0, poly), rt.mat(base.ptr, 0, 2 * poly, 0, poly), 1, 1, dim, dim, 1, level, causal=False)
    out = rt.buf(dim * 2 * poly)
    with pytest.raises(A.AceHipError, match="outside the arena"):
        rt.linear_i8(rt.mat(out.ptr, 0, 0, 2 * poly, poly), xm, dw.ptr, dim, 1, dim, dim, 2, level)
    edge = rt.mat(base.ptr + 8 * (total - poly), 0, 0, 2 * poly, poly)
    with pytest.raises(A.AceHipError, match="end of the arena"):
        rt.linear_i8(edge, xm, dw.ptr, dim, 1, dim, dim, 2, level)
    with pytest.raises(A.AceHipError, match="end of the arena"):
        rt.linear_i8(ym, edge, dw.ptr, dim, 1, dim, dim, 2, level)
    rt.check(rt.lib.acehip_ctx_select(rt.h, 0, 1))
    rt.linear_i8(rt.mat(out.ptr, 0, 0, 2 * poly, poly), xm, dw.ptr, dim, 1, dim, dim, 2, level)
    rt.sync()
    q = np.array(rt.primes[:level], dtype=object)[:, None]
    xo, t = x.astype(object), tab.values()[0, 0, :, 0]
    lin = np.stack([np.tensordot(w.astype(object), xo[r], (1, 0)) for r in range(n_rep)]) % q
    rot = lin.copy()
    for i in range(dim // 2):
        f1 = i + dim // 2
        rot[:, i], rot[:, f1] = (lin[:, i] - lin[:, f1]) * t[i] % q, (lin[:, i] + lin[:, f1]) * t[i] % q
    got = base.download((n_rep, total))
    for r in range(n_rep):
        y = got[r, y_at: y_at + dim * 2 * poly].reshape(dim, 2, level, N)
        z = got[r, z_at: z_at + dim * dim * 3 * poly].reshape(dim, dim, 3, level, N)
        if r == 0:
            assert not y.any() and not z.any()
            continue
        assert np.array_equal(y, rot[r].astype(np.uint64))
        for i, j in itertools.product(range(dim), range(dim)):
            assert np.array_equal(z[i, j], (pair(rot[r, i], xo[r, j]) % q).astype(np.uint64))
    assert np.array_equal(out.download((dim, 2, level, N)), lin[0].astype(np.uint64))
    for b in (base, out, dw, tab):
        b.free()
    rt.close()


def test_sharded_context_computes_its_limbs(contexts):
    """simulated ranks: replica h of the arena gets the limbs of rank h and no others"""
    N, L, world, level, dim = 64, 4, 2, 4, 4
    rt = A.AceHip(N, L, 60, 50, 2)
    poly = level * N
    words = 1 << 15
    ws = int(rt.lib.acehip_workspace_words(rt.h))
    total = words + ws + 64 * N
    base = rt.buf(total * world)
    cfg = A.binding.ArenaCfg(base.ptr, total * 8, total * 8, world, base.ptr + 8 * words, base.ptr + 8 * (words + ws), 64)
    rt.check(rt.lib.acehip_ctx_set_arena(rt.h, C.byref(cfg)))
    rt.check(rt.lib.acehip_ctx_shard_sim(rt.h, world))
    rng = np.random.default_rng(3)
    x = np.stack([rng.integers(0, rt.primes[p], size=(dim, 2, N), dtype=np.uint64) for p in range(level)], axis=-2)
    host = np.zeros((world, total), np.uint64)
    host[:, : x.size] = x.reshape(-1)
    base.upload(host)
    w = rng.integers(-128, 128, size=(dim, dim)).astype(np.int8)
    dw = dev(rt, w)
    y_at, z_at = 8192, 16384
    rt.linear_i8(rt.mat(base.ptr + 8 * y_at, 0, 0, 2 * poly, poly), rt.mat(base.ptr, 0, 0, 2 * poly, poly), dw.ptr, dim, 1, dim, dim, 2, level)
    rt.linattn_state(rt.mat(base.ptr + 8 * z_at, 0, 0, 3 * poly, poly), None, rt.mat(base.ptr, 0, 0, 0, poly), rt.mat(base.ptr, 0, 0, 2 * poly, poly), 1, 1, 1, 1, dim, level)
    rt.sync()
    q = np.array(rt.primes[:level], dtype=object)[:, None]
    lin = np.tensordot(w.astype(object), x.astype(object), (1, 0)) % q
    got = base.download((world, total))
    for r in range(world):
        y = got[r, y_at: y_at + dim * 2 * poly].reshape(dim, 2, level, N)
        z = got[r, z_at: z_at + dim * 3 * poly].reshape(dim, 3, level, N)
        for l in range(level):
            if l % world == r:
                assert np.array_equal(y[:, :, l], lin[:, :, l].astype(np.uint64))
                for j in range(dim):
                    assert np.array_equal(z[j, :, l], (pair(x[0].astype(object), x[j].astype(object)) % q)[:, l].astype(np.uint64))
            else:
                assert not y[:, :, l].any() and not z[:, :, l].any()
    for b in (base, dw):
        b.free()
    rt.close()


# ---- used together: a layer on encrypted data ------------------------------------------------------------------------------------------
class Client:
    """A CKKS user on top of the C ABI: secret and relinearisation key, encryption, decryption and decoding in whole numbers on the host
    (transforms on the device)."""

    def __init__(self, rt, seed):
        self.rt, self.rng = rt, np.random.default_rng(seed)
        self.N, self.q = rt.N, np.array(rt.primes, dtype=object)[:, None]
        self.full = list(range(rt.L + rt.K))
        self.s = self.ntt(self.rng.integers(-1, 2, self.N).astype(object), self.full)
        s2 = self.s * self.s % self.q
        P = int(np.prod(self.q[rt.L:, 0]))
        key = []
        for d in range(rt.dnum):
            a = self.uniform(self.full)
            own = np.array([[P % int(self.q[i, 0]) if i < rt.L and i // rt.alpha == d else 0] for i in self.full], dtype=object)
            key += [(self.noise(self.full) - a * self.s + own * s2) % self.q, a]
        self.key = dev(rt, np.stack(key).astype(np.uint64))
        j = np.array([pow(5, int(k), 2 * self.N) for k in range(self.N // 2)])
        self.decode_matrix = np.exp(1j * np.pi * (j[:, None] * np.arange(self.N)[None] % (2 * self.N)) / self.N)

    def ntt(self, coefficients, limbs):
        return self.rt.ntt((coefficients[None] % self.q[limbs]).astype(np.uint64), self.rt.L, pos0=limbs[0]).astype(object)

    def uniform(self, limbs):
        return np.stack([self.rng.integers(0, int(self.q[i, 0]), self.N, dtype=np.uint64) for i in limbs]).astype(object)

    def noise(self, limbs):
        return self.ntt(np.rint(self.rng.normal(0, 3.2, self.N)).astype(np.int64).astype(object), limbs)

    def encrypt(self, message, level):
        limbs = list(range(level))
        m = self.rt.encode(np.asarray(message, dtype=np.float64), level)[0].astype(object)
        a = self.uniform(limbs)
        return np.stack([(m + self.noise(limbs) - a * self.s[:level]) % self.q[:level], a]).astype(np.uint64)

    def decrypt(self, ct, scale):
        """ct: [2][level][N]"""
        m = (ct[0, :1].astype(object) + ct[1, :1].astype(object) * self.s[:1]) % self.q[:1]
        c = self.rt.ntt(m.astype(np.uint64), self.rt.L, inverse=True)[0].astype(object)
        c = np.where(c > self.q[0] // 2, c - self.q[0], c).astype(np.float64) / scale
        return (self.decode_matrix @ c).real


class Cts:
    """device array of ciphertexts [heads][rows][cols][comps], limbs of `level`, with their scale"""

    def __init__(self, rt, shape, level, scale, data=None):
        self.rt, self.shape, self.level, self.scale = rt, shape, level, scale
        self.poly = level * rt.N
        self.buf = rt.to_device(data) if data is not None else rt.buf(int(np.prod(shape)) * self.poly)

    def strides(self):
        h, r, c, p = self.shape
        return dict(head=r * c * p * self.poly, row=c * p * self.poly, col=p * self.poly, comp=self.poly)

    def mat(self, **other):
        return self.rt.mat(self.buf.ptr, **{**self.strides(), **other})

    def at(self, i, p):
        return self.buf.ptr + 8 * self.poly * (i * self.shape[3] + p)

    def finish(self, client, times):
        """relinearised where there are three polynomials, then rescaled `times` times"""
        rt, lib, N = self.rt, self.rt.lib, self.rt.N
        n = int(np.prod(self.shape[:3]))
        out = Cts(rt, (*self.shape[:3], 2), self.level - times, self.scale / float(np.prod([float(rt.primes[self.level - 1 - t]) for t in range(times)])))
        t = [rt.buf(self.poly) for _ in range(6)]
        for i in range(n):
            c = [self.at(i, 0), self.at(i, 1)]
            if self.shape[3] == 3:
                rt.check(lib.acehip_key_switch(rt.h, t[0].ptr, t[1].ptr, self.at(i, 2), client.key.ptr, self.level, None))
                for p in (0, 1):
                    rt.check(lib.acehip_modadd(rt.h, t[p].ptr, t[p].ptr, c[p], self.level, 0, self.level, None))
                c = [t[0].ptr, t[1].ptr]
            for k in range(times):
                to = [out.at(i, 0), out.at(i, 1)] if k == times - 1 else [t[2 + 2 * (k % 2)].ptr, t[3 + 2 * (k % 2)].ptr]
                rt.check(lib.acehip_rescale2(rt.h, to[0], to[1], c[0], c[1], self.level - k, None))
                c = to
        rt.sync()
        for b in (*t, self.buf):
            b.free()
        return out

    def values(self, client):
        d = self.buf.download((*self.shape, self.level, self.rt.N))
        return np.array([[[client.decrypt(d[h, r, c], self.scale) for c in range(self.shape[2])] for r in range(self.shape[1])] for h in range(self.shape[0])])


def test_layer_on_encrypted_data():
    """Projections with int8 weights, rotary positions with two axes, causal linear attention over a chunk of two tokens, its state, a third token in
    the recurrent form, output projection -- against the same layer in double precision on the messages.  A scale of 2^51 leaves errors of
    2^-51 times noise (about 2^6 fresh, 2^12 from a key switch or a rescale in every slot) times values and weights of a few units through six levels:
    below 2^-30; a wrong term is of the size of the values."""
    rt = A.AceHip(1024, 7, 60, 51, 3)
    cl = Client(rt, 11)
    N, slots, delta = rt.N, rt.N // 2, 2.0**51
    rng = np.random.default_rng(12)
    H, dk, dv, din, T = 2, 4, 3, 5, 3
    x = rng.uniform(-1, 1, (T, din, slots))
    assert np.max(np.abs(cl.decrypt(cl.encrypt(x[0, 0], 3), delta) - x[0, 0])) < 2.0**-35
    cx = Cts(rt, (1, T, din, 2), 7, delta, np.stack([[cl.encrypt(x[t, i], 7) for i in range(din)] for t in range(T)]))
    d_x = cx

    def project(src, w, scale, tok=None, shape=None):
        """w * scale: rows of tokens -> [token][n_out]"""
        n_out = w.shape[0]
        mul = np.rint(scale * delta).astype(np.int64)
        out = Cts(rt, shape or (1, T, n_out, 2), src.level, src.scale * delta * (delta if tok else 1))
        dw, dm = dev(rt, w), dev(rt, mul)
        rt.linear_i8(rt.mat(out.buf.ptr, row=n_out * 2 * out.poly, col=2 * out.poly, comp=out.poly), src.mat(), dw.ptr, w.shape[1], T, w.shape[1], n_out, 2, src.level,
                     d_mul=dm.ptr, d_tok=tok.ptr if tok else None, tok_stride=out.poly)
        rt.sync()
        dw.free()
        dm.free()
        return out

    wq, wk, wv = (rng.integers(-127, 128, (n, din)).astype(np.int8) for n in (H * dk, dk, dv))
    sq, sk, sv = (rng.uniform(0.002, 0.008, n) for n in (H * dk, dk, dv))
    keep_slot = rng.integers(0, 2, (T, slots)).astype(np.float64)      # tokens that are padding in some of the sequences
    mask = dev(rt, np.stack([rt.encode(keep_slot[t], 7)[0] for t in range(T)]))
    q = project(d_x, wq, sq, shape=(T, H, dk, 2)).finish(cl, 1)        # [token][head][feature]
    k = project(d_x, wk, sk, shape=(T, 1, dk, 2)).finish(cl, 1)
    v = project(d_x, wv, sv, tok=mask, shape=(T, 1, dv, 2)).finish(cl, 2)
    xq = np.einsum("ji,tis->tjs", wq * sq[:, None], x).reshape(T, H, dk, slots)
    xk, xv = np.einsum("ji,tis->tjs", wk * sk[:, None], x), np.einsum("ji,tis->tjs", wv * sv[:, None], x) * keep_slot[:, None]
    assert np.max(np.abs(v.values(cl)[:, 0] - xv)) < 2.0**-30

    # rotary positions: pair 0 by time, pair 1 by place; tables at the level of the queries, one for each token
    pos = np.stack([np.repeat(np.arange(T) + 1000.0, slots), np.tile(np.arange(slots) % 7, T).astype(np.float64)])
    freq, axis = [1.0, 0.1], [0, 1]
    d_pos, d_cos, d_sin = dev(rt, pos), rt.buf(2 * T * slots, np.float64), rt.buf(2 * T * slots, np.float64)
    rt.rope_messages(d_cos.ptr, d_sin.ptr, T * slots, d_pos.ptr, T * slots, T * slots, freq, axis, 2)
    tables = []
    for d in (d_cos, d_sin):
        t = rt.buf(T * 2 * q.poly)
        for tok, pair_i in itertools.product(range(T), range(2)):
            rt.check(rt.lib.acehip_encode(rt.h, t.at((tok * 2 + pair_i) * q.poly), None, d.at(pair_i * T * slots + tok * slots), 1, slots, 0, delta, 1, q.level, 0, None))
        tables.append(t)
    ang = (pos[axis] * np.array(freq)[:, None]).reshape(2, T, slots).transpose(1, 0, 2)

    def turn(ct, heads, val):
        rt.rope(ct.mat(head=ct.strides()["row"], row=ct.strides()["head"]), ct.mat(head=ct.strides()["row"], row=ct.strides()["head"]), tables[0].ptr, tables[1].ptr, ct.poly,
                2 * ct.poly, heads, T, dk, 2, ct.level)
        ct.scale *= delta
        a, b = val[..., :2, :], val[..., 2:, :]
        c, s = (f(ang) if val.ndim == 3 else f(ang)[:, None] for f in (np.cos, np.sin))
        return ct.finish(cl, 1), np.concatenate([a * c - b * s, a * s + b * c], axis=-2)

    q, xq = turn(q, H, xq)
    k, xk = turn(k, 1, xk)
    tokens = lambda ct, first=0: rt.mat(ct.buf.ptr + 8 * first * ct.strides()["head"], head=ct.strides()["row"], row=ct.strides()["head"], col=ct.strides()["col"], comp=ct.poly)
    assert np.max(np.abs(q.values(cl) - xq)) < 2.0**-30 and q.level == k.level == v.level == 5

    # a chunk of two tokens
    gamma = np.array([0.9, 0.75])
    decay = np.rint(gamma[:, None] ** np.arange(2) * delta).astype(np.int64)
    d_decay = dev(rt, decay)
    p = Cts(rt, (H, 2, 2, 3), 5, q.scale * k.scale, np.zeros((H, 2, 2, 3, 5, N), np.uint64))
    rt.linattn_scores(p.mat(), tokens(q), tokens(k), H, 1, 2, 2, dk, 5)
    p = p.finish(cl, 1)
    o = Cts(rt, (H, 2, dv, 3), 4, p.scale * v.scale * delta)
    rt.linattn_out(o.mat(), None, None, p.mat(), tokens(v), H, 1, 2, 2, dk, dv, 4, d_decay=d_decay.ptr)
    o = o.finish(cl, 2)
    want = np.zeros((H, T, dv, slots))
    for h, t in itertools.product(range(H), range(T)):
        for s in range(t + 1):
            want[h, t] += gamma[h] ** (t - s) * np.sum(xq[t, h] * xk[s], axis=0) * xv[s]
    assert np.max(np.abs(o.values(cl) - want[:, :2])) < 2.0**-30

    # its state, and the third token
    S = Cts(rt, (H, dk, dv, 3), 5, k.scale * v.scale * delta)
    rt.linattn_state(S.mat(), None, tokens(k), tokens(v), H, 1, 2, dk, dv, 5, d_decay=d_decay.ptr)
    S = S.finish(cl, 2)
    keep = dev(rt, np.rint(gamma * (k.scale * v.scale / S.scale)).astype(np.int64))
    S1 = Cts(rt, (H, dk, dv, 3), 3, k.scale * v.scale)
    rt.linattn_state(S1.mat(), S.mat(), tokens(k, 2), tokens(v, 2), H, 1, 1, dk, dv, 3, d_keep=keep.ptr)
    S1 = S1.finish(cl, 1)
    o1 = Cts(rt, (H, 1, dv, 3), 2, q.scale * S1.scale)
    rt.linattn_out(o1.mat(), tokens(q, 2), S1.mat(), None, None, H, 1, 1, 0, dk, dv, 2)
    o1 = o1.finish(cl, 1)
    assert o1.level == 1 and np.max(np.abs(o1.values(cl)[:, 0] - want[:, 2])) < 2.0**-30

    # output projection of the third token: heads and features as one row of inputs
    wo = rng.integers(-3, 4, (4, H * dv)).astype(np.int8)
    y, dw = Cts(rt, (1, 1, 4, 2), 1, o1.scale), dev(rt, wo)
    rt.linear_i8(y.mat(), rt.mat(o1.buf.ptr, col=2 * o1.poly, comp=o1.poly), dw.ptr, H * dv, 1, H * dv, 4, 2, 1)
    assert np.max(np.abs(y.values(cl)[0, 0] - wo @ want[:, 2].reshape(H * dv, slots))) < 2.0**-26
    rt.close()
