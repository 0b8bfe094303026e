"""GPU tests (-m gpu) of the operators on ciphertexts at the calls that tests/test_gpu_nn.py leaves out: packed weights of every kind, large rings."""
import pytest
from test_gpu_nn import contexts, linear_case  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_in,n_out,ld", [(3, 1025, None), (3, 1028, None), (1, 1025, None), (1, 1039, None), (7, 1026, 9), (3, 1056, None), (3, 1057, None)])
def test_linear_last_part_of_packed_weights(contexts, n_in, n_out, ld):  # noqa: F811
    """parts of 512 outputs and a last one whose weights are fewer bytes than a fragment's 16, which is up to 32 outputs, or just more"""
    rt = contexts("n64")
    assert 32 * 1024 <= rt.lib.acehip_workspace_words(rt.h) * 8 < 38 * 1024
    linear_case(rt, 2, [0, 1], 12, n_in, n_out, 3, ld=ld)
