"""Tensors that lie on another device than the call are refused before any
pointer is taken (without a GPU, on stand-ins that say where they lie)."""
import pytest


class Elsewhere:
    """What the checks ask of a tensor, of one that lies on another GPU (or on the host: -1)."""

    def __init__(self, dtype, shape, device):
        self.dtype, self.shape, self._device = dtype, shape, device
        self.is_cuda = device >= 0

    def get_device(self):
        return self._device

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 256


@pytest.mark.parametrize("device", [1, -1])
def test_a_tensor_of_another_device_is_refused(device):
    import torch
    from mars_b200 import kv
    i32, f32 = torch.int32, torch.float32
    here = dict(positions=Elsewhere(i32, (3, 2), 0), freq=Elsewhere(f32, (4,), 0), axis=Elsewhere(i32, (4,), 0))
    table = kv._table(3, **here, interleaved=False, device=0)
    assert (table.rot_dim, table.n_axes, table.freq, table.axis) == (8, 2, 256, 256)
    for name, t in here.items():
        with pytest.raises(ValueError, match=name):
            kv._table(3, **dict(here, **{name: Elsewhere(t.dtype, t.shape, device)}), interleaved=False, device=0)
    # every tensor of the context's calls; the last of each has its own check and comes first here
    ctx = kv.KvContext.__new__(kv.KvContext)
    ctx.handle, ctx.device = None, 0
    ints = lambda shape, d=0: Elsewhere(i32, shape, d)
    shapes = dict(kv_lens=(2,), finished=(2,), tables=(2, 5), free_pages=(9,), free_count=(1,))
    for name in shapes:
        with pytest.raises(ValueError, match=name):
            ctx.release(**{n: ints(s, device if n == name else 0) for n, s in shapes.items()}, page_size=8)
    with pytest.raises(ValueError, match="status"):
        ctx.release(**{n: ints(s) for n, s in shapes.items()}, page_size=8, status=ints((1,), device))
    shapes["new_lens"] = shapes.pop("finished")
    for name in shapes:
        with pytest.raises(ValueError, match=name):
            ctx.plan(**{n: ints(s, device if n == name else 0) for n, s in shapes.items()}, page_size=8, max_tokens=1)
    for name in ("decay", "x"):
        with pytest.raises(ValueError, match=name):
            kv._floats(name, Elsewhere(f32, (4,), device), 0, 4)
    assert kv._floats("decay", Elsewhere(f32, (4,), 0), 0, 4) == 256
