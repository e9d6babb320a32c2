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
    need = 256 + 512 * 1024 * 1024 * 8
    assert rc == 0 and need <= b <= need * 1.01  # (packed sequences, which the size is for too, need some more)
    assert forward(L, BF16, need - 1, 512, 131072, 1024) == -2  # the call takes the shape and wants that many bytes
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


def packed_query(L, n, longest, c, rows):
    b, r = ctypes.c_size_t(77), ctypes.c_uint64(77)
    rc = L.lcpp_recurrence_packed_temp_bytes(n, longest, c, rows, ctypes.byref(b))
    assert L.lcpp_recurrence_packed_checkpoint_rows(n, longest, rows, ctypes.byref(r)) == 0
    return rc, b.value, r.value


def packed_forward(L, t, temp_bytes, n, longest, c, rows):
    return L.lcpp_recurrence_forward(t, 2, P, temp_bytes, P, c, 0, P, c, 0, P, c, 0, None, None, None, n, longest, c, P, P, rows,
                                     None)


def test_packed_sizes_go_by_the_rows(L):
    """256 documents of 262144 rows in all: no more than 262144 / 128 + 256 tiles, however long the longest."""
    for longest in (32768, 262144, 1 << 30):
        rc, b, saved = packed_query(L, 256, longest, 2048, 262144)
        assert rc == 0 and b < 40 << 20 and saved == 2048 + 256
        assert packed_forward(L, BF16, b - 1, 256, longest, 2048, 262144) == -2 or \
            packed_forward(L, F32, b - 1, 256, longest, 2048, 262144) == -2
    # short ones of nearly one length need no more than max_length each
    rc, b, saved = packed_query(L, 100, 200, 64, 19000)
    assert rc == 0 and saved == 100 * 2
    assert packed_query(L, 100, 200, 64, 9000)[2] == 9000 // 128 + 100
    assert packed_query(L, 100, 129, 64, 1 << 30)[2] == 200
    assert packed_query(L, 100, 128, 64, 12800) == (0, 0, 100)
    assert packed_query(L, 3, 500, 64, 0) == (0, 0, 3)


@pytest.mark.parametrize("n,longest,rows", [(1023, 65536, 262144), (2000, 65536, 1 << 20), (1000, 100000, 200000)])
def test_many_documents_with_a_long_one_are_taken(L, n, longest, rows):
    rc, b, _ = packed_query(L, n, longest, 2048, rows)
    assert rc == 0 and 0 < b <= 256 + (rows // 128 + n) * (2048 * 8 + 32) + 512
    for t in (BF16, F32):
        assert packed_forward(L, t, 256, n, longest, 2048, rows) == -2  # wants temp storage, does not refuse the sizes


def test_the_size_without_rows_serves_packed_calls(L):
    for n, longest, c in ((1, 129, 1), (1, 40000, 64), (24, 5000, 1536), (300, 70000, 65), (5, 100000, 1)):
        rc, b = query(L, n, longest, c)
        for rows in (longest, n * longest, 1 << 40):
            prc, pb, saved = packed_query(L, n, longest, c, rows)
            assert rc == prc == 0 and pb <= b and saved <= n * -(-longest // 128)


def test_packed_refusals(L):
    b, r = ctypes.c_size_t(77), ctypes.c_uint64(77)
    assert L.lcpp_recurrence_packed_temp_bytes(1 << 20, 1 << 20, 2048, 1 << 40, ctypes.byref(b)) == -1 and b.value == 77
    assert L.lcpp_recurrence_packed_temp_bytes(1, 1 << 31, 1, 1, ctypes.byref(b)) == -1
    assert L.lcpp_recurrence_packed_temp_bytes(1, 1, 1, 1, None) == -1
    assert L.lcpp_recurrence_packed_checkpoint_rows(1, 1 << 31, 1, ctypes.byref(r)) == -1 and r.value == 77
    assert L.lcpp_recurrence_packed_checkpoint_rows(1, 1, 1, None) == -1
    assert packed_forward(L, BF16, 1 << 40, 1 << 20, 1 << 20, 2048, 1 << 40) == -1
