"""CPU tests of the argument checks of the operators on ciphertexts (csrc/api_nn.cpp) at the calls that tests/test_nn_refusals.py leaves out: a call that
is refused says so (ACEHIP_EINVAL), one that would run says that there is no device (ACEHIP_ENODEV)."""
import pytest
from test_nn_refusals import BASE, EINVAL, FAR, Linear, Out, Rope, Scores, State, changed, rt  # noqa: F401  (a fixture)

import ace_compiler_amd as A

Mat = A.binding.Mat


# counts whose product passes 64 bits, as 0 or as a small number: not empty, and not to be listed
PAST = [(1 << 30, 1 << 30, 16), (1 << 22, 1 << 22, 1 << 20), (242243305, 197908, 384773)]


@pytest.mark.parametrize("n", PAST, ids=str)
def test_counts_past_64_bits(rt, n):  # noqa: F811
    out, one = Mat(BASE, 1 << 20, 3 << 10, 1 << 10, 1), Mat(BASE - FAR, 0, 0, 0, 0)
    calls = [changed(Linear, out=out, x=one, rows=n[0], n_out=n[1], comps=n[2], ts=0, mul=None), changed(Rope, out=out, x=one, rows=n[0], dim=n[1], heads=n[2], rs=0, ps=0),
             changed(Rope, out=out, x=one, rows=8, dim=8, heads=n[0], comps=n[1], rs=0, ps=0),
             changed(Scores, out=out, q=one, k=one, nq=n[0], nk=n[1], heads=n[2], kv=n[2]),
             changed(Out, out=out, q=one, S=one, p=one, v=one, nq=n[0], dv=n[1], heads=n[2], kv=n[2], din=None, decay=None),
             changed(State, out=out, S=one, k=one, v=one, dk=n[0], dv=n[1], heads=n[2], kv=n[2], keep=None, decay=None)]
    for c in calls:
        if isinstance(c, Linear):
            c.a["w"] = 1
        assert c.call(rt) == EINVAL, c
        assert "too many" in rt.err() or "overlap" in rt.err(), rt.err()


@pytest.mark.parametrize("n_out", [(1 << 32) - 7, (1 << 32) - 1, 1 << 31])
def test_linear_outputs_near_32_bits(rt, n_out):  # noqa: F811
    c = changed(Linear, out=Mat(1 << 45, 0, 0, 192, 0), rows=1, comps=1, n_out=n_out, ld=7, w=1 << 61, mul=None, tok=None)
    assert c.call(rt) == EINVAL and "too many" in rt.err()
