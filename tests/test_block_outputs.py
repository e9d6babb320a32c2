"""Outputs of the layer norm and the recurrence that begin at one place are refused before any launch (no GPU needed):
one of the two would be lost."""
import pytest

F32, BF16 = 2, 6
A, B, C, D, E, G = (4096 * i for i in range(1, 7))  # addresses that no call reads


@pytest.fixture(scope="module")
def L():
    import lc_parallel_primitive_amd as lcpp

    return lcpp.lib()


def test_sum_over_out(L):
    assert L.lcpp_layer_norm_add_forward(BF16, F32, A, 64, B, 64, 0.1, 1, 2, None, None, None, 1e-5, C, 64, C, 64, None, None, 4,
                                         64, None) == -1


def test_statistics_over_each_other(L):
    assert L.lcpp_layer_norm_forward(BF16, F32, A, 64, None, None, 1e-5, B, 64, C, C, 4, 64, None) == -1
    assert L.lcpp_layer_norm_add_forward(BF16, F32, A, 64, B, 64, 0.1, 1, 2, None, None, None, 1e-5, C, 64, D, 64, E, E, 4, 64,
                                         None) == -1


def test_gradients_over_each_other(L):
    assert L.lcpp_layer_norm_backward(BF16, F32, A, 1 << 30, B, 64, C, 64, None, D, E, G, 64, B, B, 4, 64, None) == -1
    # the residual's gradient and the branch's differ by the dropout
    assert L.lcpp_layer_norm_add_backward(BF16, F32, A, 1 << 30, B, 64, None, 0, C, 64, None, D, E, 0.5, 1, 2, None, G, 64, G, 64,
                                          None, None, 4, 64, None) == -1
    assert L.lcpp_recurrence_backward(F32, 0, A, 1 << 40, B, 64, 32000, C, 64, 32000, D, E, 64, 32000, G, 64, 32000, G, 64, 32000,
                                      None, None, 3, 500, 64, None, None, 0, None) == -1


def test_nothing_to_write_is_no_conflict(L):
    assert L.lcpp_layer_norm_add_forward(BF16, F32, A, 64, B, 64, 0.1, 1, 2, None, None, None, 1e-5, C, 64, C, 64, E, E, 0, 64,
                                         None) == 0
    assert L.lcpp_layer_norm_backward(BF16, F32, A, 1 << 30, B, 64, C, 64, None, D, E, G, 64, None, None, 4, 0, None) == 0
