"""The sum form with decays above 1, whose product passes fp32 where no state does: cut in chunks and walked through, against the steps in
64 bits. Tolerances are those of test_gated_scan_gpu; where a state is 0 they are 0."""
import pytest
import torch

from test_gated_scan_gpu import check, inputs

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def growing(T, D, dtype, rate, length, at):
    """Decays of e^rate for `length` steps from `at` on; nothing comes in before their end, and nothing of what follows is asked for."""
    x, gate, _, _, dy, _ = inputs((T, 1, D), dtype, 'sum')
    gate[at:at + length] = rate
    x[:at + length] = 0
    dy[at:] = 0
    return x, gate, dy


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('T, D, rate, length, at', [(400, 256, 1.0, 200, 100), (400, 33, 3.0, 60, 7), (500, 5, 88.0, 150, 3), (300, 8, 0.5, 290, 10)])
def test_where_there_is_no_state(T, D, rate, length, at, dtype):
    x, gate, dy = growing(T, D, dtype, rate, length, at)
    check(x, gate, None, None, dy, None, 'sum')
    check(x, gate, torch.zeros(1, D, device='cuda'), None, dy, torch.zeros(1, D, device='cuda'), 'sum')
    reset = torch.zeros(T, 1, dtype=torch.bool, device='cuda')
    reset[at + length // 2] = True
    check(x, gate, None, reset, dy, None, 'sum')


@pytest.mark.parametrize('T, D, rate, length, at', [(2400, 256, 1.0, 1200, 96), (4000, 6, 0.25, 3000, 500)])
def test_long_ones(T, D, rate, length, at):
    x, gate, dy = growing(T, D, torch.bfloat16, rate, length, at)
    check(x, gate, None, None, dy, None, 'sum')


def test_walked_through():
    """As many sequences as have a thread a channel: the same values."""
    x, gate, dy = growing(400, 256, torch.float32, 1.0, 200, 100)
    many = lambda t: t.expand(400, 400, 256)
    check(many(x), many(gate), None, None, many(dy), None, 'sum')


@pytest.mark.parametrize('T, D', [(700, 4), (700, 33), (1500, 64)])
def test_small_states_grow_and_fall(T, D):
    """e^150 up and down again: from 1e-30 to 1e35. Joining chunks as products in fp32 makes infinities of it."""
    x, gate, h0, _, dy, dlast = inputs((T, 1, D), torch.float32, 'sum')
    gate[200:350], gate[350:500] = 1, -1
    small = [t * 1e-30 for t in (x, h0, dy, dlast)]
    check(small[0], gate, small[1], None, small[2], small[3], 'sum')
    gate[200:350], gate[350:500] = 0.9, -0.9
    reset = torch.zeros(T, 1, dtype=torch.bool, device='cuda')
    reset[100] = True
    check(small[0], gate, small[1], reset, small[2], small[3], 'sum')


def test_far_powers():
    """Rises and falls of e^30000 and more with no state in them: the power of 2 that goes with the product, far past fp32's and fp64's."""
    T, D = 1200, 16
    x, gate, _, _, dy, _ = inputs((T, 1, D), torch.float32, 'sum')
    gate[100:600], gate[600:1100], gate[150:1000:7] = 80, -85, 0.1
    x[:1100], dy[100:] = 0, 0
    check(x, gate, None, None, dy, None, 'sum')
    gate[100:1100] = gate[100:1100].flip(0)
    check(x, gate, None, None, dy, None, 'sum')


def test_the_work_buffer_of_a_growing_one():
    """The products' powers lie behind the maps: nothing behind the buffer's stated size is written."""
    from d1._lib import check as ok, library, stream_of
    T, D = 8192, 48
    x, gate, dy = growing(T, D, torch.float32, 1.0, 200, 100)
    lib, at = library(), lambda t: t.data_ptr()
    size = lib.d1_gated_scan_work_bytes(T, 1, D)
    work = torch.full((size + 4096,), 171, dtype=torch.uint8, device='cuda')
    y, last = torch.empty_like(x), torch.empty(D, device='cuda')
    for form in (0, 1):
        ok(lib.d1_gated_scan(at(x), D, D, at(gate), D, D, 0, form, T, 1, D, None, None, 0, 0, at(y), at(last), at(work), stream_of(x)))
        assert (work[size:] == 171).all() and not y.isnan().any()
