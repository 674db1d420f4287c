"""Calls of the paged attention that are refused on the host (CPU): results over
the queries in rows of another stride would land in other streams' queries."""
import pytest

from conftest import load_xe


class At:
    def __init__(self, ptr):
        self.ptr = ptr


@pytest.fixture(scope="module")
def xe():
    return load_xe()


@pytest.fixture
def kv(xe):
    return xe.PagedKV(At(0x1000), At(0x2000), At(0x3000), 8, 2, 16, 64, 3, 4)


def attn(xe, kv, ldq, ldo, out=0x4000, hq=4):
    assert xe.lib().xe_paged_attn_dev(None, kv, 0x4000, ldq, 0x5000, hq, 1.0, 0, out, ldo) == -1
    return xe.last_error()


@pytest.mark.parametrize("ldq,ldo", [(512, 0), (0, 512), (512, 256), (256, 260), (512, 516)])
def test_out_over_q_in_rows_of_another_stride(xe, kv, ldq, ldo):
    assert "row stride" in attn(xe, kv, ldq, ldo)
    assert attn(xe, kv, ldq, ldo, out=0x9000) == "null ctx"  # elsewhere any stride will do


@pytest.mark.parametrize("ldq,ldo", [(0, 0), (256, 0), (0, 256), (512, 512)])
def test_out_over_q_in_its_own_rows(xe, kv, ldq, ldo):
    assert attn(xe, kv, ldq, ldo) == "null ctx"


def test_one_row_has_no_stride(xe, kv):
    kv.batch = 1
    assert attn(xe, kv, 512, 0) == "null ctx"
