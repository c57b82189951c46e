"""The operators where values, indices or lengths are at the edge of what they may be, on the GPU: the
cases of tests/test_cpu_operator_kernels.py again."""
import numpy as np
import pytest

from paged_cases import HEADS, HUGE_FAR, LOST_BLOCKS, ODD_KEYS, ODD_QUERIES, ODD_VALUES, PRECISION, SMALL_ROOM, LostBlocks, OddKey, OddQuery, OddValue, Precision, SmallRoom, falling_starts, huge_far_values, huge_values
from sanic_amd import ir
from test_gpu_operators import Batch, bind, read, words

pytestmark = pytest.mark.gpu


def attention(dev, t):
    p = t.program()
    bufs = bind(dev, p, t.values())
    exe = dev.prepare(p)
    exe.execute_static(bufs)
    return read(p, bufs, "o"), exe.stage_kernel(0)


@pytest.mark.parametrize("case", ODD_VALUES)
def test_a_value_not_finite_in_the_past(dev, case):
    odd = OddValue(**ODD_VALUES[case])
    odd.check(*attention(dev, odd.batch))


@pytest.mark.parametrize("case", ODD_KEYS)
def test_a_key_of_minus_infinity_has_no_weight(dev, case):
    odd = OddKey(**ODD_KEYS[case])
    odd.check(*attention(dev, odd.batch))


@pytest.mark.parametrize("case", ODD_QUERIES)
def test_a_nan_in_a_query_is_in_its_row(dev, case):
    odd = OddQuery(**ODD_QUERIES[case])
    odd.check(*attention(dev, odd.batch))


@pytest.mark.parametrize("case", LOST_BLOCKS)
def test_lost_blocks_have_no_slots(dev, case):
    t = LostBlocks(**LOST_BLOCKS[case])
    p = t.program()
    bufs = bind(dev, p, t.values())
    dev.prepare(p).execute_static(bufs)
    assert words(p, bufs, "plan.slots").tolist() == t.slots()


@pytest.mark.parametrize("HD,dq", [(64, ir.BF16), (128, ir.F16), (24, ir.F32)])
def test_starts_that_fall_leave_nothing_behind(dev, HD, dq):
    """Nothing is written, and the next call (its arrivals are counted in the same words) is right."""
    t, starts = falling_starts(HD, dq)
    p = t.program()
    bufs = bind(dev, p, t.values())
    exe = dev.prepare(p)
    for _ in range(2):
        bufs["starts"].upload_array(np.asarray(starts, np.uint32))
        bufs["o"].upload(b"\xa5" * p.by_name["o"].nbytes)
        exe.execute_static(bufs)
        assert bufs["o"].download() == b"\xa5" * p.by_name["o"].nbytes
        bufs["starts"].upload_array(np.asarray(t.starts, np.uint32))
        exe.execute_static(bufs)
        t.check(read(p, bufs, "o"), exe.stage_kernel(0))


@pytest.mark.parametrize("case", PRECISION)
def test_bits_of_the_weights(dev, case):
    t = Precision(**PRECISION[case])
    t.check(*attention(dev, t.batch))


@pytest.mark.parametrize("HD", HEADS)
def test_every_head_size(dev, HD):
    for do in (ir.BF16, ir.F32):
        t = Batch(past=[190, 99], new=[1, 30], NKV=1, rep=2, HD=HD, BS=16, do=do)
        t.check(*attention(dev, t))


@pytest.mark.parametrize("case", SMALL_ROOM)
def test_little_room_for_partials(dev, case):
    t = SmallRoom(**SMALL_ROOM[case])
    p = t.program()
    bufs = bind(dev, p, {**t.values(), "ballast.in": np.zeros(p.by_name["ballast.in"].shape)})
    exe = dev.prepare(p)
    for _ in range(2):
        exe.execute_static(bufs)
        t.check(read(p, bufs, "o"), exe.stage_kernel(0))


@pytest.mark.parametrize("new,HD", [(1, 64), (5, 128), (12, 64)])
def test_values_near_the_end_of_the_range(dev, new, HD):
    t = huge_values(new, HD)
    t.check(*attention(dev, t))


@pytest.mark.parametrize("case", HUGE_FAR)
def test_huge_values_without_weight(dev, case):
    t = huge_far_values(**HUGE_FAR[case])
    t.check(*attention(dev, t))
