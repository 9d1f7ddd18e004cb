"""More of what the Python binding of the serving calls refuses before the library is called; no GPU."""
import os
import subprocess
import sys

import pytest
import torch

from test_serve_args import CALLS, OnDevice, attn, attn_args, ctx, dev, lib  # noqa: F401


@pytest.mark.parametrize("heads", [4, 32])
@pytest.mark.parametrize("dims", [8, 64, 256])
def test_heads_of_another_size_than_the_pools_are_refused(lib, ctx, heads, dims):  # noqa: F811
    """In rows that are wide enough for as many heads of 128, so that the library would take them for such."""
    a = attn_args()
    for name, dtype in (("q", torch.float16), ("out", torch.float32)):
        a[name] = dev(5, heads * max(dims, 128), dtype=dtype)[:, :heads * dims].unflatten(1, (heads, dims))
    with pytest.raises(AssertionError):
        attn(ctx, a)
    assert not lib.calls


class Elsewhere(OnDevice):
    def get_device(self):
        return 1


@pytest.mark.parametrize("call,args,name", [(c, a, n) for c, a in CALLS for n in a()])
def test_a_tensor_of_another_device_is_refused(lib, ctx, call, args, name):  # noqa: F811
    a = args()
    a[name] = a[name].as_subclass(Elsewhere)
    with pytest.raises(AssertionError):
        call(ctx, a)
    assert not lib.calls


@pytest.mark.parametrize("call,args", CALLS)
def test_all_of_another_device_are_refused(lib, ctx, call, args):  # noqa: F811
    a = {name: t.as_subclass(Elsewhere) for name, t in args().items()}
    with pytest.raises(AssertionError):
        call(ctx, a)
    assert not lib.calls
    ctx.device = 1
    call(ctx, a)
    assert len(lib.calls) == 1


WITHOUT_ASSERTIONS = """
import sys
sys.path[:0] = [%r, %r]
from cyb_b200 import qeng
from test_serve_args import CALLS, Library
import torch
lib = qeng._lib = Library()
qeng._cur_stream = lambda: None
ctx = qeng.Context.__new__(qeng.Context)
ctx.h, ctx.device = None, 0
passed = []
for call, args in CALLS:
    for name in args():
        for change in (lambda t: t.as_subclass(torch.Tensor), lambda t: t[:1]):
            a = args()
            a[name] = change(a[name])
            try:
                call(ctx, a)
            except AssertionError:
                continue
            passed.append(name)
ctx.h = None
print(sys.flags.optimize, lib.calls, passed)
"""


def test_refusals_do_not_go_with_assertions():
    """python -O: tensors of the host, and tensors with too few entries."""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-O", "-c", WITHOUT_ASSERTIONS % (os.path.dirname(here), here)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    # one entry or row is enough of a ring, of a table whose rows are named, and of the one group's pages
    assert r.stdout.split("\n")[0] == "1 ['qeng_kv_plan', 'qeng_attn_shared', 'qeng_attn_shared'] ['ring', 'table', 'pages']", r.stdout
