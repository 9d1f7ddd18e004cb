"""More of what the Python binding of the serving calls refuses before the library is called; no GPU."""
import pytest
import torch

from test_serve_args import attn, attn_args, ctx, dev, lib  # noqa: F401


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
