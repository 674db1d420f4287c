"""Calls over a paged cache that are refused on the host (CPU): results over the
queries in rows of another stride would land in other streams' queries; tables
and rows beyond what one launch counts."""
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


@pytest.mark.parametrize("batch,hkv,hq,positions,fits", [
    (64, 12, 12, 1 << 24, True), (64, 12, 12, 1 << 26, False), (64, 12, 12, 1 << 30, False),
    (1, 1, 16, 1 << 30, True), (31, 1, 16, 1 << 30, True), (32, 1, 16, 1 << 30, False), (16, 1, 17, 1 << 30, False),
    (15, 1, 17, 1 << 30, True), (4096, 1, 1, 1 << 23, False), (4096, 1, 1, (1 << 23) - 16, True)])
def test_most_keys_in_a_table(xe, kv, batch, hkv, hq, positions, fits):
    """batch * hkv * blocks of 16 query heads * positions below 2^35."""
    kv.batch, kv.hkv, kv.max_pages = batch, hkv, positions // 16
    kv.page_stride = 0
    assert (batch * hkv * -(-hq // hkv // 16) * positions < 2 ** 35) == fits
    said = attn(xe, kv, 0, 0, hq=hq)
    assert (said == "null ctx") == fits
    assert fits or "more keys" in said


@pytest.mark.parametrize("n_rows,fits", [(((1 << 35) - 2049) // 512, True), (((1 << 35) - 2048) // 512, False), (1 << 30, False)])
def test_most_rows_of_an_append(xe, kv, n_rows, fits):
    rows = xe.PagedRows(n_rows, 4, q=0x4000, k=0x5000, v=0x6000, ldq=256, ldkv=128, q_out=0x7000, ldqo=256, pos=0x8000, start=0x9000)
    assert (n_rows * (4 + 2 * 2) * 64 < 2 ** 35 - 2048) == fits
    assert xe.lib().xe_paged_append_dev(None, kv, rows) == -1
    assert (xe.last_error() == "null ctx") == fits
