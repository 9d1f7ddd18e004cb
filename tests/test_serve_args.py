"""What the Python binding of the serving calls refuses before the library is called; no GPU: tensors that say they are on one, and
a library that must not be reached."""
import pytest
import torch

from cyb_b200 import qeng


class OnDevice(torch.Tensor):
    is_cuda = True


def dev(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append(name) or 0


class Pool:
    h, pages, kv_heads, hd = None, 8, 2, 128


@pytest.fixture
def lib(monkeypatch):
    lib = Library()
    monkeypatch.setattr(qeng, "_lib", lib)
    monkeypatch.setattr(qeng, "_cur_stream", lambda: None)
    return lib


@pytest.fixture
def ctx():
    c = qeng.Context.__new__(qeng.Context)
    c.h, c.device = None, 0
    return c


def plan_args():
    return dict(lens=dev(3), add=dev(3), keep=dev(3), table=dev(3, 4), ring=dev(8), ends=dev(2, dtype=torch.int64), starts=dev(4), slots=dev(8), pos=dev(8),
                seen=dev(8), rows=dev(8), lens_out=dev(3), ends_out=dev(2, dtype=torch.int64))


def plan(ctx, a):
    out = qeng.KVPlan(a["starts"], a["slots"], a["pos"], a["seen"], a["rows"], a["lens_out"], a["ends_out"])
    ctx.kv_plan(Pool, a["lens"], a["add"], a["table"], a["ring"], a["ends"], 8, keep=a["keep"], out=out)


def append_args():
    f16, f32 = torch.float16, torch.float32
    return dict(qkv=dev(5, 8 * 128, dtype=f32), pos=dev(5), slots=dev(5), q_gain=dev(128, dtype=f32), k_gain=dev(128, dtype=f32), out=dev(5, 4, 128, dtype=f16))


def append(ctx, a):
    ctx.rope_append(Pool, a["qkv"], a["pos"], a["slots"], 1e4, q_gain=a["q_gain"], k_gain=a["k_gain"], out=a["out"])


def attn_args():
    f16, f32 = torch.float16, torch.float32
    return dict(q=dev(5, 4, 128, dtype=f16), table=dev(5, 4), lens=dev(5), first=dev(2), pages=dev(1), rows=dev(5), out=dev(5, 4, 128, dtype=f32))


def attn(ctx, a):
    ctx.attn_shared(Pool, a["q"], a["table"], a["lens"], a["first"], a["pages"], rows=a["rows"], out=a["out"])


CALLS = [(plan, plan_args), (append, append_args), (attn, attn_args)]


@pytest.mark.parametrize("call,args", CALLS)
def test_good_arguments_reach_the_library(lib, ctx, call, args):
    call(ctx, args())
    assert len(lib.calls) == 1


@pytest.mark.parametrize("call,args,name", [(c, a, n) for c, a in CALLS for n in a()])
def test_a_tensor_of_the_host_is_refused(lib, ctx, call, args, name):
    a = args()
    a[name] = a[name].as_subclass(torch.Tensor)
    with pytest.raises(AssertionError):
        call(ctx, a)
    assert not lib.calls


@pytest.mark.parametrize("call,args,name", [(c, a, n) for c, a in CALLS for n in a()])
def test_a_tensor_of_another_type_is_refused(lib, ctx, call, args, name):
    a = args()
    a[name] = a[name].to(torch.int16).as_subclass(OnDevice)
    with pytest.raises((AssertionError, KeyError)):
        call(ctx, a)
    assert not lib.calls


def test_a_plan_with_a_tensor_replaced_is_looked_at_again(lib, ctx):
    a = plan_args()
    out = qeng.KVPlan(a["starts"], a["slots"], a["pos"], a["seen"], a["rows"], a["lens_out"], a["ends_out"])
    assert out._replace(lens=a["lens"]).lens is a["lens"]
    with pytest.raises(AssertionError):
        out._replace(lens=a["lens"].as_subclass(torch.Tensor))
    with pytest.raises(AssertionError):
        ctx.kv_plan(Pool, a["lens"], a["add"], a["table"], a["ring"], a["ends"], 8, out=tuple(out))
    assert not lib.calls


@pytest.mark.parametrize("name", ["starts", "slots", "pos", "seen", "rows", "lens_out", "ends_out"])
def test_a_broadcast_result_of_the_plan_is_refused(lib, ctx, name):
    a = plan_args()
    a[name] = a[name][:1].expand(a[name].numel()).as_subclass(OnDevice)
    with pytest.raises(AssertionError):
        plan(ctx, a)
    assert not lib.calls
