"""Size queries of the recurrence: host arithmetic, no GPU."""
import ctypes

import pytest

BF16, F32, P = 6, 2, 4096


@pytest.fixture(scope="module")
def L():
    import lc_parallel_primitive_amd as lcpp

    return lcpp.lib()


def query(L, *sizes):
    b = ctypes.c_size_t(77)
    return L.lcpp_recurrence_temp_bytes(*sizes, ctypes.byref(b)), b.value


def forward(L, t, temp_bytes, n, length, c):
    """The call's status with too little temp storage, or its refusal of the shape: nothing is launched."""
    return L.lcpp_recurrence_forward(t, 2, P, temp_bytes, P, c, c * length, P, c, c * length, P, c, c * length, None, None, None,
                                     n, length, c, None, None, 0, None)


def test_sizes_that_only_two_byte_types_allow(L):
    """512 x 131072 x 1024: 2^22 tiles of 128 channels, which a launch holds, and 2^23 of 64 channels, which none does."""
    rc, b = query(L, 512, 131072, 1024)
    assert rc == 0 and b == 256 + 512 * 1024 * 1024 * 8
    assert forward(L, BF16, b - 1, 512, 131072, 1024) == -2  # the call takes the shape and wants that many bytes
    assert forward(L, F32, b, 512, 131072, 1024) == -1


def test_a_refused_query_writes_nothing(L):
    assert query(L, 1024, 131072, 1024) == (-1, 77)
    assert query(L, 1, 1 << 31, 1) == (-1, 77)
    assert L.lcpp_recurrence_temp_bytes(1, 1, 1, None) == -1


@pytest.mark.parametrize("n,length,c", [(1, 129, 1), (3, 777, 1000), (7, 129, 64), (2, 300, 65), (1, 65536, 2048), (1, 128, 9)])
def test_the_size_is_enough_for_every_type_and_needed_by_one(L, n, length, c):
    rc, b = query(L, n, length, c)
    assert rc == 0
    if length <= 128:
        assert b == 0
    else:
        assert -2 in (forward(L, BF16, b - 1, n, length, c), forward(L, F32, b - 1, n, length, c))
