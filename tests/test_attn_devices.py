"""Cache, batch, rows and workspace on the host or on devices of their own: refused before a pointer of theirs is passed
on. No GPU: where a device is needed, a stand-in says that it is on one and points nowhere."""
import pytest
import torch

import attn_oracle as ao
import q3q4


class OnDevice:
    """What the calls ask of a tensor, on device 0."""

    is_cuda, dtype, device = True, torch.float32, "cuda:0"

    def __init__(self, rows, width, dtype=torch.float32, contiguous=True, index=0):
        self.shape, self.dtype, self.index, self.whole = (rows, width), dtype, index, contiguous

    def stride(self):
        return (self.shape[1] * (1 if self.whole else 2), 1)

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return self.whole

    def numel(self):
        return self.shape[0] * self.shape[1]

    def element_size(self):
        return 4

    def data_ptr(self):
        return 0


def ints(*s, device="cpu"):
    return torch.zeros(s, dtype=torch.int32, device=device)


def cache_and_batch(cache_device=None, batch_device=None):
    c = q3q4.KVCache(ao.F16, 1, 16, 1, 64, data=torch.empty(4096, dtype=torch.uint8))
    b = q3q4.KVBatch(ints(3), ints(2), ints(2, 4), 2, 1, 16)
    if cache_device is not None:
        c.device = cache_device
    if batch_device is not None:
        b.device = batch_device
    return c, b


CALLS = {"write": q3q4.kv_write, "read": q3q4.kv_read,
         "attention": lambda c, b, x, y: q3q4.attention(c, b, x, y, 0.1)}


@pytest.mark.parametrize("what", CALLS)
@pytest.mark.parametrize("cache_device,batch_device", [(None, None), (0, None), (None, 0), (0, 1)])
def test_cache_and_batch_have_to_be_on_one_device(what, cache_device, batch_device):
    c, b = cache_and_batch(cache_device, batch_device)
    with pytest.raises(q3q4.Q3Q4Error, match="cache's data and the batch's tensors must be device tensors on one"):
        CALLS[what](c, b, OnDevice(2, 64), OnDevice(2, 64))


@pytest.mark.parametrize("what", CALLS)
@pytest.mark.parametrize("x,y", [(torch.zeros(2, 64), OnDevice(2, 64)), (OnDevice(2, 64), torch.zeros(2, 64)),
                                 (OnDevice(2, 64, index=1), OnDevice(2, 64))], ids=["first", "second", "other"])
def test_rows_have_to_be_on_the_cache_s_device(what, x, y):
    c, b = cache_and_batch(0, 0)
    with pytest.raises(q3q4.Q3Q4Error, match="cache's device"):
        CALLS[what](c, b, x, y)


@pytest.mark.parametrize("workspace", [torch.zeros(64), OnDevice(8, 64, index=1), OnDevice(8, 64, contiguous=False)],
                         ids=["host", "other", "strided"])
def test_the_workspace_has_to_be_whole_and_on_the_cache_s_device(workspace):
    c, b = cache_and_batch(0, 0)
    with pytest.raises(q3q4.Q3Q4Error, match="workspace must be a contiguous tensor on the cache's device"):
        q3q4.attention(c, b, OnDevice(2, 64), OnDevice(2, 64), 0.1, workspace=workspace)


@pytest.mark.parametrize("at", [0, 1, 2])
def test_a_batch_is_on_one_device(at):
    t = [ints(3), ints(2), ints(2, 4)]
    t[at] = ints(*t[at].shape, device="meta")
    with pytest.raises(q3q4.Q3Q4Error, match="one device"):
        q3q4.KVBatch(*t, 2, 1, 16)


@pytest.mark.parametrize("shape", [(), (64,), (1, 2, 64)])
def test_attention_of_rows_that_are_not_2d_is_refused(shape):
    c, b = cache_and_batch(0, 0)
    q = OnDevice(2, 64)
    q.shape, q.stride = shape, lambda: (1,) * len(shape)
    with pytest.raises(q3q4.Q3Q4Error, match="2-d"):
        q3q4.attention(c, b, q, q, 0.1)
