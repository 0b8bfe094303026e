"""GPU tests (-m gpu) of the operators on ciphertexts at the calls that tests/test_gpu_nn.py leaves out: packed weights of every kind, large rings."""
import numpy as np
import pytest
from test_gpu_nn import LargeAttn, Sampled, contexts, dev, linear_case, pair  # noqa: F401  (a fixture)

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
