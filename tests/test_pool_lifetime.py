"""When the memory of a cache pool goes: with the last view of it, at once."""
import gc
import weakref

import pytest
import torch

from cyb_b200 import qeng


class Library:
    def __init__(self):
        self.freed = 0

    def qeng_kv_pool_data(self, h):
        return 4096

    def qeng_kv_pool_free(self, ctx, h):
        self.freed += 1
        return 0


class Owner:
    h, device = 1, 0


@pytest.fixture
def collector_off():
    gc.collect()
    gc.disable()
    yield
    gc.enable()


def test_a_pool_goes_with_its_last_view(monkeypatch, collector_off):
    """No GPU: a stand-in for torch's view that holds, as torch does, the object it was made from."""
    lib = Library()
    monkeypatch.setattr(qeng, "_lib", lib)

    class View:
        def __init__(self, obj):
            self.obj = obj

        def view(self, *shape):
            assert shape == (3, 2, 2, 16, 128)
            return self

    monkeypatch.setattr(torch, "as_tensor", lambda obj, device: View(obj))
    pool = qeng.KVPool(Owner, 7, 3, 2, 128)
    view, other = pool.tensor(), pool.tensor()
    info = view.obj.__cuda_array_interface__
    assert info["data"] == (4096, False) and info["shape"] == (3 * 2 * 2 * 16 * 128,) and info["typestr"] == "<f2"
    alive = weakref.ref(pool)
    del pool, other
    assert lib.freed == 0
    del view
    freed = lib.freed
    if alive() is not None:
        alive().h = None  # nothing for the real library to free later
    assert freed == 1


@pytest.mark.gpu
def test_a_view_of_the_device_keeps_its_pool_no_longer_than_it_lives(ctx, collector_off):
    pool = ctx.kv_pool(3, 1)
    view, alive = pool.tensor()[1:], weakref.ref(pool)
    view.fill_(2)
    del pool
    assert alive() is not None and bool((view == 2).all())
    del view
    assert alive() is None


@pytest.mark.gpu
def test_a_pool_may_be_freed_while_a_stream_is_captured(ctx):
    """As a collector may do at any allocation: the capture stays valid, and the memory is given back."""
    before = torch.cuda.mem_get_info()[0]
    pool, kept = ctx.kv_pool(4096, 8), ctx.kv_pool(2, 1)
    assert torch.cuda.mem_get_info()[0] <= before - 4096 * 8 * 8192
    x = torch.arange(3 * 128, device="cuda", dtype=torch.float32).view(1, 384) / 128
    pos, slots, q = (torch.zeros(1, dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.float16))
    q = q.expand(128).contiguous().view(1, 1, 128)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.rope_append(kept, x, pos, slots, 1e4, out=q)
        del pool
        ctx.rope_append(kept, x, pos, slots, 1e4, out=q)
    assert torch.cuda.mem_get_info()[0] > before - 4096 * 8 * 8192
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(q.view(-1), x[0, :128].half())
    kept.free()
    ctx.device_status()
