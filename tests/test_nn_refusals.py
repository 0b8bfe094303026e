"""CPU tests of the argument checks of the operators on ciphertexts (csrc/api_nn.cpp): on a context without a GPU a call that is refused
says so (ACEHIP_EINVAL), and one that would run says that there is no device (ACEHIP_ENODEV)."""
import ctypes as C

import pytest

import ace_compiler_amd as A

EINVAL, ENODEV = -1, -3
N, LEVEL = 64, 3
POLY = LEVEL * N  # words
BASE = 1 << 32    # addresses are never followed here


@pytest.fixture(scope="module")
def rt():
    r = A.AceHip(N, 4, 60, 50, 2, host_only=True)
    yield r
    r.close()


def mat(at, *shape):
    """contiguous [..][comp] matrix of ciphertexts: shape = (heads, rows, cols, comps) counts"""
    s, strides = POLY, []
    for n in reversed(shape):
        strides.append(s)
        s *= n
    return A.binding.Mat(BASE + at, *reversed(strides))


def ref(m):
    return None if m is None else C.byref(m)


FAR = 1 << 30  # between the operands


class Linear:
    def __init__(self):
        self.a = dict(out=mat(0, 1, 2, 5, 2), x=mat(FAR, 1, 2, 7, 2), w=BASE + 2 * FAR, ld=7, rows=2, n_in=7, n_out=5, comps=2, mul=BASE + 3 * FAR,
                      tok=BASE + 4 * FAR, ts=POLY, level=LEVEL, pos0=0, n=LEVEL)

    def call(self, rt):
        a = self.a
        return rt.lib.acehip_linear_i8(rt.h, ref(a["out"]), ref(a["x"]), a["w"], a["ld"], a["rows"], a["n_in"], a["n_out"], a["comps"], a["mul"], a["tok"],
                                       a["ts"], a["level"], a["pos0"], a["n"], None)


class Rope:
    def __init__(self):
        self.a = dict(out=mat(0, 2, 3, 8, 2), x=mat(FAR, 2, 3, 8, 2), c=BASE + 2 * FAR, s=BASE + 3 * FAR, ps=POLY, rs=4 * POLY, heads=2, rows=3, dim=8, comps=2,
                      level=LEVEL, pos0=0, n=LEVEL)

    def call(self, rt):
        a = self.a
        return rt.lib.acehip_rope(rt.h, ref(a["out"]), ref(a["x"]), a["c"], a["s"], a["ps"], a["rs"], a["heads"], a["rows"], a["dim"], a["comps"], 0,
                                  a["level"], a["pos0"], a["n"], None)


class Messages:
    def __init__(self):
        self.a = dict(cos=BASE, sin=BASE + FAR, os=10, pos=BASE + 2 * FAR, ps=10, n=10, freq=(C.c_double * 4)(1, 2, 3, 4), axis=(C.c_uint32 * 4)(0, 1, 2, 1), pairs=4,
                      axes=3)

    def call(self, rt):
        a = self.a
        return rt.lib.acehip_rope_messages(rt.h, a["cos"], a["sin"], a["os"], a["pos"], a["ps"], a["n"], a["freq"], a["axis"], a["pairs"], a["axes"], None)


class Scores:
    def __init__(self):
        self.a = dict(out=mat(0, 4, 5, 6, 3), q=mat(FAR, 4, 5, 7, 2), k=mat(2 * FAR, 2, 6, 7, 2), heads=4, kv=2, nq=5, nk=6, dim=7, level=LEVEL, pos0=0, n=LEVEL)

    def call(self, rt):
        a = self.a
        return rt.lib.acehip_linattn_scores(rt.h, ref(a["out"]), ref(a["q"]), ref(a["k"]), a["heads"], a["kv"], a["nq"], a["nk"], a["dim"], 1, a["level"],
                                            a["pos0"], a["n"], None)


class Out:
    def __init__(self):
        self.a = dict(out=mat(0, 4, 5, 3, 3), q=mat(FAR, 4, 5, 7, 2), S=mat(2 * FAR, 4, 7, 3, 2), p=mat(3 * FAR, 4, 5, 6, 2), v=mat(4 * FAR, 2, 6, 3, 2), heads=4, kv=2,
                      nq=5, nk=6, dk=7, dv=3, din=BASE + 5 * FAR, decay=BASE + 6 * FAR, causal=1, level=LEVEL, pos0=0, n=LEVEL)

    def call(self, rt):
        a = self.a
        return rt.lib.acehip_linattn_out(rt.h, ref(a["out"]), ref(a["q"]), ref(a["S"]), ref(a["p"]), ref(a["v"]), a["heads"], a["kv"], a["nq"], a["nk"], a["dk"],
                                         a["dv"], a["din"], a["decay"], a["causal"], a["level"], a["pos0"], a["n"], None)


class State:
    def __init__(self):
        self.a = dict(out=mat(0, 4, 7, 3, 3), S=mat(FAR, 4, 7, 3, 2), k=mat(2 * FAR, 2, 6, 7, 2), v=mat(3 * FAR, 2, 6, 3, 2), heads=4, kv=2, nk=6, dk=7, dv=3,
                      keep=BASE + 4 * FAR, decay=BASE + 5 * FAR, level=LEVEL, pos0=0, n=LEVEL)

    def call(self, rt):
        a = self.a
        return rt.lib.acehip_linattn_state(rt.h, ref(a["out"]), ref(a["S"]), ref(a["k"]), ref(a["v"]), a["heads"], a["kv"], a["nk"], a["dk"], a["dv"], a["keep"],
                                           a["decay"], a["level"], a["pos0"], a["n"], None)


ALL = [Linear, Rope, Messages, Scores, Out, State]
MATS = [c for c in ALL if c is not Messages]


def changed(cls, **new):
    c = cls()
    for k in new:
        assert k in c.a
    c.a.update(new)
    return c


@pytest.mark.parametrize("cls", ALL, ids=lambda c: c.__name__)
def test_a_good_call_only_lacks_the_device(rt, cls):
    assert cls().call(rt) == ENODEV
    assert cls().call(type("NoContext", (), {"lib": rt.lib, "h": None})) == EINVAL


@pytest.mark.parametrize("cls", MATS, ids=lambda c: c.__name__)
def test_limb_ranges(rt, cls):
    for bad in (dict(level=5, n=5), dict(pos0=1, n=LEVEL + rt.K), dict(pos0=0xFFFFFFFF, n=1), dict(n=0xFFFFFFFF), dict(pos0=LEVEL + rt.K + 1, n=0)):
        assert changed(cls, **bad).call(rt) == EINVAL, bad
        assert cls.__name__.lower() in rt.err().replace("linattn_", "").replace("linear_i8", "linear")
    for good in (dict(n=0), dict(pos0=2, n=1), dict(n=LEVEL + rt.K) if cls is not Linear else dict(n=1)):
        # (more limbs than the matrices are laid out for overlap: given strides that hold them)
        c = changed(cls, **good)
        if c.a["n"] > LEVEL:
            for m in [v for v in c.a.values() if isinstance(v, A.binding.Mat)]:
                for f in ("head_stride", "row_stride", "col_stride", "comp_stride"):
                    setattr(m, f, getattr(m, f) * 4)
        assert c.call(rt) == ENODEV, (good, rt.err())


@pytest.mark.parametrize("cls", MATS, ids=lambda c: c.__name__)
def test_matrices(rt, cls):
    names = [k for k, v in cls().a.items() if isinstance(v, A.binding.Mat)]
    for k in names:
        c = cls()
        c.a[k].data = None
        assert c.call(rt) == EINVAL and "null" in rt.err()
        c = cls()
        c.a[k].data += 4
        assert c.call(rt) == EINVAL and "aligned" in rt.err()
        c = cls()
        c.a[k].col_stride = 1 << 61
        assert c.call(rt) == EINVAL
        if k != "out":  # every operand apart from the result, polynomial by polynomial
            c = cls()
            c.a[k].data = c.a["out"].data + 8 * (POLY - 1)
            assert c.call(rt) == EINVAL and "overlaps" in rt.err(), k
            c = cls()
            c.a[k].row_stride = c.a[k].col_stride = c.a[k].head_stride = c.a[k].comp_stride = 0  # broadcast operands are fine
            assert c.call(rt) == ENODEV, rt.err()
    for f in ("row_stride", "col_stride", "comp_stride"):
        c = cls()
        setattr(c.a["out"], f, POLY - 1)
        assert c.call(rt) == EINVAL and "overlap" in rt.err(), f
        c = cls()
        setattr(c.a["out"], f, 0)
        assert c.call(rt) == EINVAL


def test_interleaved_operands_are_accepted(rt):
    """inputs and results of a linear layer side by side in one block: [row][input 0, output 0, input 1, ...], and a transposed result"""
    c = Linear()
    c.a.update(out=A.binding.Mat(BASE + 8 * POLY, 0, 100 * POLY, 4 * POLY, 2 * POLY), x=A.binding.Mat(BASE, 0, 100 * POLY, 4 * POLY, 2 * POLY))
    assert c.call(rt) == ENODEV, rt.err()
    c.a["out"].data = BASE + 8 * POLY - 8
    assert c.call(rt) == EINVAL
    c = Linear()
    c.a["out"] = A.binding.Mat(BASE, 0, POLY, 2 * POLY, 10 * POLY)  # [comp][col][row]
    assert c.call(rt) == ENODEV, rt.err()
    # strides that cross without a polynomial in common: 2 rows 3 polynomials apart, 5 columns 2 apart and so on
    c.a["out"] = A.binding.Mat(BASE, 0, 3 * POLY, 2 * POLY, 50 * POLY)
    assert c.call(rt) == ENODEV, rt.err()
    c.a["out"] = A.binding.Mat(BASE, 0, 4 * POLY, 2 * POLY, 50 * POLY)
    assert c.call(rt) == EINVAL


def test_in_place(rt):
    c = Rope()
    c.a["x"] = mat(0, 2, 3, 8, 2)
    assert c.call(rt) == ENODEV, rt.err()
    c.a["x"].data += 8 * POLY
    assert c.call(rt) == EINVAL
    c = State()
    c.a["S"] = mat(0, 4, 7, 3, 3)
    assert c.call(rt) == ENODEV, rt.err()
    c.a["S"].comp_stride *= 2
    assert c.call(rt) == EINVAL


def test_linear(rt):
    for bad in (dict(w=None), dict(ld=6), dict(n_in=65537, ld=65537), dict(mul=BASE + 4), dict(mul=BASE), dict(w=BASE + 100), dict(tok=BASE + 8), dict(tok=BASE + 3 * FAR + 1),
                dict(tok=BASE - 8 * POLY, ts=POLY)):
        assert changed(Linear, **bad).call(rt) == EINVAL, bad
    for good in (dict(mul=None, tok=None), dict(w=BASE + 2 * FAR + 3), dict(n_in=0, x=None, w=None), dict(n_out=0, out=None), dict(rows=0), dict(ts=0), dict(comps=1)):
        assert changed(Linear, **good).call(rt) == ENODEV, (good, rt.err())


def test_rope(rt):
    for bad in (dict(dim=7), dict(c=None), dict(s=None), dict(c=BASE), dict(s=BASE + 2 * FAR + 4)):
        assert changed(Rope, **bad).call(rt) == EINVAL, bad
    for good in (dict(rs=0), dict(ps=0, rs=0), dict(heads=0), dict(dim=0), dict(comps=3, out=mat(0, 2, 3, 8, 3), x=mat(FAR, 2, 3, 8, 3))):
        assert changed(Rope, **good).call(rt) == ENODEV, (good, rt.err())


def test_rope_messages(rt):
    for bad in (dict(axes=9), dict(axes=2), dict(axes=0), dict(cos=None), dict(sin=None), dict(pos=None), dict(freq=None), dict(axis=None), dict(os=9), dict(cos=BASE + 4),
                dict(sin=BASE + 8), dict(pos=BASE + 16), dict(pos=BASE + FAR - 8), dict(pairs=65536), dict(os=1 << 61), dict(n=1 << 31, os=1 << 31, cos=1 << 50, sin=1 << 51, pos=1 << 52)):
        assert changed(Messages, **bad).call(rt) == EINVAL, bad
    for good in (dict(n=0), dict(pairs=0), dict(ps=0), dict(pairs=1, os=0)):
        assert changed(Messages, **good).call(rt) == ENODEV, (good, rt.err())


def test_linear_attention(rt):
    for cls in (Scores, Out, State):
        for bad in (dict(kv=3), dict(kv=0), dict(kv=8), dict(nk=1 << 31)):
            assert changed(cls, **bad).call(rt) == EINVAL, bad
    one = A.binding.Mat(BASE + FAR, 0, 0, 0, 0)  # (strides of zero: any count of features lies in memory)
    assert changed(Scores, dim=1 << 31, q=one, k=one).call(rt) == EINVAL
    assert changed(Scores, dim=(1 << 31) - 1, q=one, k=one).call(rt) == ENODEV
    assert changed(Out, dk=1 << 31, q=one, S=one).call(rt) == EINVAL
    for bad in (dict(q=None), dict(S=None), dict(p=None), dict(v=None), dict(causal=0), dict(din=BASE + 5 * FAR + 4), dict(decay=BASE + 8)):
        assert changed(Out, **bad).call(rt) == EINVAL, bad
    for good in (dict(q=None, S=None), dict(p=None, v=None), dict(q=None, S=None, p=None, v=None), dict(causal=0, decay=None), dict(nk=0), dict(dk=0), dict(nq=0),
                 dict(din=None, decay=None)):
        assert changed(Out, **good).call(rt) == ENODEV, (good, rt.err())
    for good in (dict(S=None), dict(S=None, keep=None), dict(nk=0), dict(dk=0), dict(keep=None, decay=None), dict(heads=0, kv=0)):
        assert changed(State, **good).call(rt) == ENODEV, (good, rt.err())
    for bad in (dict(keep=BASE + 4), dict(decay=BASE)):
        assert changed(State, **bad).call(rt) == EINVAL, bad
    assert changed(Scores, dim=0).call(rt) == ENODEV
    # a launch has fewer than 2^24 workgroups along x
    big = changed(Scores, nq=1 << 16, nk=1 << 16, out=A.binding.Mat(BASE, 0, POLY << 18, 3 * POLY, POLY), q=A.binding.Mat(BASE, 0, 0, 0, 0), k=A.binding.Mat(BASE, 0, 0, 0, 0),
                  heads=1, kv=1)
    big.a["q"].data = big.a["k"].data = 4096
    assert big.call(rt) == EINVAL and "too many" in rt.err()
