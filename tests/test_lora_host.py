"""CPU tests of what zmi_lora_direct refuses about its operands' places in memory.  Every call here is refused before anything
touches an address."""
import random

import pytest

from zendnn_amd import capi
from tests.test_cabi_host import fake_pointers
from tests.test_router_lora_host import ADDR, lora

ROW = 32 * 2   # bytes of a row of `lora()`: 32 bf16 columns


@fake_pointers
@pytest.mark.parametrize("T,off,ld_base,ld_dst,overlap", [
    # (base stands `off` bytes behind dst)
    (4, 2, 32, 32, True), (4, -2, 32, 32, True), (4, ROW, 32, 32, True), (4, 3 * ROW, 32, 32, True), (4, 4 * ROW, 32, 32, False),
    (4, -4 * ROW, 32, 32, False), (4, -4 * ROW + 2, 32, 32, True), (4, 3 * ROW + ROW - 2, 32, 32, True),
    (1, ROW - 2, 32, 99, True), (1, ROW, 32, 32, False), (1, -ROW, 1 << 62, 1 << 61, False), (2, -ROW, 1 << 62, 1 << 61, False),
    # columns of one buffer beside each other, and columns that meet
    (4, ROW, 64, 64, False), (4, -ROW, 64, 64, False), (4, ROW - 2, 64, 64, True), (4, ROW + 2, 64, 64, True), (4, ROW + 2, 65, 65, False),
    (4, 2 * ROW + ROW, 64, 64, False), (4, 3 * 2 * ROW + ROW - 2, 64, 64, True), (4, 4 * 2 * ROW - ROW + 2, 64, 64, False),
    (4, 4 * 2 * ROW - ROW, 64, 64, False), (4, 4 * 2 * ROW, 64, 64, False),
    # other strides: rows between the other one's rows, and rows that meet one
    (2, ROW, 32 * 5, 32 * 3, False), (2, ROW, 32 * 2, 32 * 3, True), (4, ROW, 32 * 4, 32 * 2, False), (4, ROW, 32 * 3, 32 * 2, True),
    (3, ROW, 32, 32 * 4, False), (4, ROW, 32, 32 * 4, True), (4, 64 * ROW, 32, 64, False)])
def test_a_base_that_meets_dst_in_part_is_refused(T, off, ld_base, ld_dst, overlap):
    st, err = lora(T=T, dst=ADDR + 0x4000, base=ADDR + 0x4000 + off, ld_base=ld_base, ld_dst=ld_dst)
    assert st == capi.FAILURE
    assert ("overlap" if overlap else "64 KiB") in err, err


@fake_pointers
def test_overlap_goes_by_bytes_and_by_all_columns():
    at = ADDR + 0x4000
    two = dict(N=(32, 32), dst=at, ld_dst=64, ld_base=64)
    st, err = lora(base=at + 2 * 64 * 4 - 2, T=4, **two)      # (inside the last two rows)
    assert st == capi.FAILURE and "overlap" in err
    st, err = lora(base=at + 2 * 64 * 4, T=4, **two)
    assert st == capi.FAILURE and "64 KiB" in err
    st, err = lora(base=at + 2 * 64 * 4, T=4, dt_dst=capi.DT_F32, **two)
    assert st == capi.FAILURE and "overlap" in err


@fake_pointers
def test_overlap_of_random_layouts_against_the_rows_themselves():
    rng = random.Random(1)
    met = 0
    for _ in range(2000):
        T, cols = rng.randint(1, 6), 32
        ld_b, ld_d = rng.randint(cols, 3 * cols), rng.randint(cols, 3 * cols)
        if rng.random() < 0.5:
            ld_b = ld_d
        off = rng.randint(-8 * cols, 8 * cols)
        if off == 0:
            continue
        rows_b = [(off + i * ld_b, off + i * ld_b + cols) for i in range(T)]
        rows_d = [(i * ld_d, i * ld_d + cols) for i in range(T)]
        overlap = any(a < d and c < b for a, b in rows_b for c, d in rows_d)
        met += overlap
        st, err = lora(T=T, dst=ADDR + 0x4000, base=ADDR + 0x4000 + 2 * off, ld_base=ld_b, ld_dst=ld_d)
        assert st == capi.FAILURE and ("overlap" if overlap else "64 KiB") in err, (T, ld_b, ld_d, off, err)
    assert 200 < met < 1900

