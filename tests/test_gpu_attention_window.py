"""A window, or a bound on the new tokens, beyond 32 bits is no limit."""
import pytest

from test_gpu_paged_attention import Problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [[1, 1], [70, 5]])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 3, 2 ** 63])
def test_a_window_beyond_32_bits_is_none(new, window):
    import mars_b200 as mb
    import torch
    p = Problem(torch, [300, 40], new, 4, 2, 64, 16, "bfloat16")
    want = p.run(mb)
    got = p.run(mb, window=window)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(mb.MarsError) as e:
        p.run(mb, window=-1)
    assert e.value.status == mb.MARS_ERR_INVALID


def test_a_bound_beyond_32_bits_is_none():
    import mars_b200 as mb
    import torch
    p = Problem(torch, [300, 40], [70, 5], 4, 2, 64, 16, "bfloat16")
    want = p.run(mb)
    got = p.run(mb, max_new=2 ** 32 + 1)                   # the low bits would say 1: the other kernel
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
