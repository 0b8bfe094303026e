"""GPU tests (-m gpu) of the operators on ciphertexts at the calls that tests/test_gpu_nn.py leaves out: packed weights of every kind, large rings."""
import ctypes as C
import itertools

import numpy as np
import pytest
from test_gpu_nn import Attn, LargeAttn, Sampled, _open, contexts, dev, hip, linear_case, ok, pair  # noqa: F401  (a fixture)

import ace_compiler_amd as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_in,n_out,ld", [(3, 1025, None), (3, 1028, None), (1, 1025, None), (1, 1039, None), (7, 1026, 9), (3, 1056, None), (3, 1057, None)])
def test_linear_last_part_of_packed_weights(contexts, n_in, n_out, ld):  # noqa: F811
    """parts of 512 outputs and a last one whose weights are fewer bytes than a fragment's 16, which is up to 32 outputs, or just more"""
    rt = contexts("n64")
    assert 32 * 1024 <= rt.lib.acehip_workspace_words(rt.h) * 8 < 38 * 1024
    linear_case(rt, 2, [0, 1], 12, n_in, n_out, 3, ld=ld)


# ---- the ring of the networks ------------------------------------------------------------------------------------------------------------
class Sampled65536(Sampled):
    AT = np.array([0, 1, 63, 64, 255, 256, 4097, 32767, 32768, 65535])


class Attn65536(LargeAttn):
    Block = Sampled65536


@pytest.fixture(scope="module")
def large():
    r = A.AceHip(65536, 2, 60, 56, 1)
    yield r
    r.close()


@pytest.mark.parametrize("sizes", [(2, 1, 5, 6, 3, 4), (1, 1, 1, 20, 5, 17)], ids=str)
def test_linear_attention_in_the_largest_ring(large, sizes):
    a = Attn65536(large, 2, [0, 1, 2], *sizes)
    a.scores()
    a.out()
    a.state()
    a.state(in_place=True)
    a.free()


@pytest.mark.parametrize("n_in,n_out,mul,tok", [(5, 3, False, False), (33, 70, True, True)])
def test_linear_in_the_largest_ring(large, n_in, n_out, mul, tok):
    level, limbs = 2, [0, 1, 2]
    rng = np.random.default_rng(n_in)
    x, y, t = (Sampled65536(large, s, level, limbs, data=d, seed=n_out) for s, d in (((1, 2, n_in, 2), None), ((1, 2, n_out, 2), False), ((1, 2, 1, 1), None)))
    w, m = rng.integers(-128, 128, size=(n_out, n_in)).astype(np.int8), rng.integers(-(1 << 62), 1 << 62, size=n_out)
    dw, dm = dev(large, w), dev(large, m)
    large.linear_i8(y.mat, x.mat, dw.ptr, n_in, 2, n_in, n_out, 2, level, n_limbs=3, d_mul=dm.ptr if mul else None, d_tok=t.buf.ptr if tok else None, tok_stride=t.strides[1])
    want = np.tensordot(w.astype(object), x.values()[0], (1, 1)).swapaxes(0, 1)
    if mul:
        want = want * m.astype(object)[:, None, None, None]
    if tok:
        want = want * t.values()[0, :, :1]
    y.check(want[None] % y.q())
    for b in (x, y, t, dw, dm):
        b.free()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_in_the_largest_ring(large, interleaved):
    shape, level, limbs = (2, 3, 6, 2), 2, [0, 1, 2]
    x, y, c, s = (Sampled65536(large, n, level, limbs, data=d, seed=k) for k, (n, d) in enumerate(((shape, None), (shape, False), ((1, 3, 3, 1), None), ((1, 3, 3, 1), None))))
    large.rope(y.mat, x.mat, c.buf.ptr, s.buf.ptr, c.strides[2], c.strides[1], *shape, level, n_limbs=3, interleaved=interleaved)
    v, cv, sv = x.values(), c.values(), s.values()
    f0, f1 = (slice(0, 6, 2), slice(1, 6, 2)) if interleaved else (slice(0, 3), slice(3, 6))
    want = np.zeros_like(v)
    want[:, :, f0] = v[:, :, f0] * cv - v[:, :, f1] * sv
    want[:, :, f1] = v[:, :, f0] * sv + v[:, :, f1] * cv
    y.check(want % y.q())
    for b in (x, y, c, s):
        b.free()


def test_many_results_in_the_largest_ring(large):
    """64 x 64 scores of four heads, 26 GB of one limb"""
    H, T, N = 4, 64, large.N
    q = int(large.primes[0])
    rng = np.random.default_rng(3)
    x, k = (rng.integers(0, q, size=(T, 2, N), dtype=np.uint64) for _ in range(2))
    x = np.stack([np.roll(x, -h, axis=0) for h in range(H)])  # one feature each
    dx, dk, dy = dev(large, x), dev(large, k), large.buf(H * T * T * 3 * N)
    strides = dict(head=T * T * 3 * N, row=T * 3 * N, col=3 * N, comp=N)
    large.linattn_scores(large.mat(dy.ptr, **strides), large.mat(dx.ptr, head=T * 2 * N, row=2 * N, comp=N), large.mat(dk.ptr, row=2 * N, comp=N), H, 1, T, T, 1, 1,
                         causal=False)
    large.sync()
    got, at = np.empty(3 * N, np.uint64), Sampled65536.AT
    for h, t, s in [(0, 0, 0), (3, 63, 63), (1, 63, 0), (2, 0, 63)] + [tuple(int(v) for v in rng.integers(0, (H, T, T))) for _ in range(40)]:
        large.check(large.lib.acehip_memcpy_d2h(got.ctypes.data, dy.at(h * strides["head"] + t * strides["row"] + s * strides["col"]), got.nbytes, None))
        want = pair(x[h, t][:, at].astype(object), k[s][:, at].astype(object)) % q
        assert np.array_equal(got.reshape(3, N)[:, at], want.astype(np.uint64)), (h, t, s)
    for b in (dx, dk, dy):
        b.free()


# ---- what the mask leaves out --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name,args,cls", [("n64", None, Attn), ("n16", None, Attn), ("n32", None, Attn), ("n16384", (16384, 2, 60, 50, 1), LargeAttn)])
@pytest.mark.parametrize("sizes", [(2, 1, 5, 5, 2, 3), (1, 1, 7, 4, 13, 5), (1, 1, 3, 70, 2, 2)], ids=str)
def test_unseen_scores_hold_anything(contexts, name, args, cls, sizes):  # noqa: F811
    """p[h][t][s] of keys that query t does not see: no residues, all bits set"""
    rt = contexts(name) if args is None else _open.setdefault(name, A.AceHip(*args))
    a = cls(rt, 2, [0, 1], *sizes)
    H, kv, nq, nk, dk, dv = sizes
    for ix, _, words in a.p.spots(a.p.host):
        if ix[2] > ix[1] + nk - nq:
            words[:] = ~np.uint64(0)
    a.p.buf.upload(a.p.host)
    a.out()
    a.out(factor=False)
    a.out(state=False)
    a.free()


# ---- packed weights: where they lie, and what reads them -----------------------------------------------------------------------------------
class Arena:
    """a context whose polynomials and workspace lie in memory that the test sees, `n_rep` times; a linear layer of ROWS rows that share their inputs,
    large enough a launch for its weights to be packed"""

    N, LEVEL, ROWS, COMPS = 64, 3, 48, 2

    def __init__(self, n_rep, n_in, n_out, ld, seed=1):
        self.rt = rt = A.AceHip(self.N, 7, 60, 51, 3)
        self.poly, self.n_in, self.n_out, self.ld, self.n_rep = self.LEVEL * self.N, n_in, n_out, ld, n_rep
        self.rng = np.random.default_rng(seed)
        ws = int(rt.lib.acehip_workspace_words(rt.h))
        sizes = dict(x=n_in * self.COMPS * self.poly, y=self.ROWS * n_out * self.COMPS * self.poly, w=(n_out * ld + 64) // 8, ws=ws, scratch=64 * self.N)
        self.at, self.total = {}, 0
        for k, n in sizes.items():
            self.at[k] = (self.total, n)
            self.total += n + n % 2
        self.base = rt.buf(self.total * n_rep)
        cfg = A.binding.ArenaCfg(self.base.ptr, self.total * 8, self.total * 8, n_rep, self.ptr("ws"), self.ptr("scratch"), 64)
        rt.check(rt.lib.acehip_ctx_set_arena(rt.h, C.byref(cfg)))
        self.host = np.zeros((n_rep, self.total), np.uint64)
        self.q = np.array(rt.primes[: self.LEVEL], dtype=object)[:, None]

    def ptr(self, k):
        return self.base.ptr + 8 * self.at[k][0]

    def part(self, words, k):
        return words[:, self.at[k][0]: sum(self.at[k])]

    def fill(self):
        """new inputs; results and workspace cleared"""
        x = np.stack([self.rng.integers(0, int(p), size=(self.n_rep, self.n_in, self.COMPS, self.N), dtype=np.uint64) for p in self.q[:, 0]], axis=-2)
        self.host[:] = 0
        self.part(self.host, "x")[:] = x.reshape(self.n_rep, -1)
        self.base.upload(self.host)
        return x

    def weights(self, *lead):
        return self.rng.integers(-128, 128, size=(*lead, self.n_out, self.ld)).astype(np.int8)

    def call(self, d_w, stream=None):
        self.rt.linear_i8(self.rt.mat(self.ptr("y"), 0, self.n_out * self.COMPS * self.poly, self.COMPS * self.poly, self.poly), self.rt.mat(self.ptr("x"), 0, 0, self.COMPS * self.poly, self.poly),
                          d_w, self.ld, self.ROWS, self.n_in, self.n_out, self.COMPS, self.LEVEL, stream=stream)

    def memory(self):
        self.rt.sync()
        return self.base.download((self.n_rep, self.total))

    def want(self, w, x):
        """of one row and replica: [output][polynomial][limb][N]"""
        return (np.tensordot(w[:, : self.n_in].astype(object), x.astype(object), (1, 0)) % self.q).astype(np.uint64)

    def results(self, words):
        return self.part(words, "y").reshape(self.n_rep, self.ROWS, self.n_out, self.COMPS, self.LEVEL, self.N)

    def close(self):
        self.base.free()
        self.rt.close()


@pytest.mark.parametrize("n_in,n_out,ld,w_off", [(70, 40, 70, 0), (70, 40, 71, 1), (70, 70, 80, 16), (70, 33, 77, 3), (64, 129, 64, 5), (1, 40, 1, 1), (65, 200, 67, 2)])
def test_packed_weights_of_any_alignment(n_in, n_out, ld, w_off):
    a = Arena(1, n_in, n_out, ld)
    x, w = a.fill(), a.weights()
    dw = dev(a.rt, np.concatenate([np.zeros(w_off, np.int8), w.ravel()[: (n_out - 1) * ld + n_in]]))
    a.call(dw.ptr + w_off)
    got = a.memory()
    assert a.part(got, "ws").any()  # packed
    y = a.results(got)[0]
    assert np.array_equal(y, np.broadcast_to(a.want(w, x[0]), y.shape))
    dw.free()
    a.close()


def test_packed_weights_under_a_selection():
    """replicas 1 and 2 of three: they share packed weights, and nothing of replica 0 changes, its workspace neither; weights in the arena are each
    replica's own and are read as they lie"""
    a = Arena(3, 20, 40, 23)
    x, w, own = a.fill(), a.weights(), a.weights(3)
    dw = dev(a.rt, w)
    a.rt.check(a.rt.lib.acehip_ctx_select(a.rt.h, 1, 2))
    a.call(dw.ptr)
    got = a.memory()
    assert a.part(got, "ws").any()
    assert np.array_equal(got[0], a.host[0])
    for r in (1, 2):
        y = a.results(got)[r]
        assert np.array_equal(y, np.broadcast_to(a.want(w, x[r]), y.shape))
    x = a.fill()
    for r in range(3):
        a.part(a.host, "w")[r].view(np.int8)[: own[r].size] = own[r].ravel()
    a.base.upload(a.host)
    a.call(a.ptr("w"))
    got = a.memory()
    assert not a.part(got, "ws").any()
    assert np.array_equal(got[0], a.host[0])
    for r in (1, 2):
        y = a.results(got)[r]
        assert np.array_equal(y, np.broadcast_to(a.want(own[r], x[r]), y.shape))
    dw.free()
    a.close()


def test_packed_weights_of_simulated_ranks():
    a = Arena(2, 20, 40, 20)
    a.rt.check(a.rt.lib.acehip_ctx_shard_sim(a.rt.h, 2))
    x, w = a.fill(), a.weights()
    a.part(a.host, "x")[1] = a.part(a.host, "x")[0]
    a.base.upload(a.host)
    dw = dev(a.rt, w)
    a.call(dw.ptr)
    got = a.memory()
    assert a.part(got, "ws").any()
    want = a.want(w, x[0])
    for r, l in itertools.product(range(2), range(a.LEVEL)):
        y = a.results(got)[r, ..., l, :]
        assert np.array_equal(y, np.broadcast_to(want[..., l, :], y.shape)) if l % 2 == r else not y.any()
    dw.free()
    a.close()


def test_packed_weights_in_a_graph():
    """two layers that pack into the same workspace in one graph, replayed on new inputs and weights with eager calls in between"""
    a = Arena(1, 70, 40, 70)
    lib = hip()
    w = a.weights(2)
    dw = [dev(a.rt, v) for v in w]
    x = a.fill()
    st, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    ok(lib.hipStreamCreateWithFlags(C.byref(st), 1))
    keep = a.rt.buf(a.at["y"][1])  # the first layer's results
    ok(lib.hipStreamBeginCapture(st, 1))  # thread-local
    y = a.rt.mat(keep.ptr, 0, a.n_out * a.COMPS * a.poly, a.COMPS * a.poly, a.poly)
    a.rt.linear_i8(y, a.rt.mat(a.ptr("x"), 0, 0, a.COMPS * a.poly, a.poly), dw[0].ptr, a.ld, a.ROWS, a.n_in, a.n_out, a.COMPS, a.LEVEL, stream=st)
    a.call(dw[1].ptr, stream=st)
    ok(lib.hipStreamEndCapture(st, C.byref(graph)))
    ok(lib.hipGraphInstantiate(C.byref(run), graph, None, None, 0))
    for _ in range(4):
        x, w = a.fill(), a.weights(2)
        for d, v in zip(dw, w):
            d.upload(v.ravel())
        a.rt.sync()
        ok(lib.hipGraphLaunch(run, st))
        ok(lib.hipStreamSynchronize(st))
        got = a.memory()
        assert a.part(got, "ws").any()
        for words, v in ((keep.download((1, -1)), w[0]), (a.part(got, "y"), w[1])):
            y = words.reshape(a.ROWS, a.n_out, a.COMPS, a.LEVEL, a.N)
            assert np.array_equal(y, np.broadcast_to(a.want(v, x[0]), y.shape))
        a.call(dw[0].ptr)
        y = a.results(a.memory())[0]
        assert np.array_equal(y, np.broadcast_to(a.want(w[0], x[0]), y.shape))
    ok(lib.hipGraphExecDestroy(run))
    ok(lib.hipGraphDestroy(graph))
    ok(lib.hipStreamDestroy(st))
    for d in (*dw, keep):
        d.free()
    a.close()
