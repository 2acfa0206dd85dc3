"""Calls of the token-sequence operators at their edges that need no GPU: what
tracers and dispatch modes see of them, and refusals."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from uplift_b200 import _native, ops, tokens


def qkv(T=4, S=4, Hq=2, Hk=1, D=16, dt=torch.float32):
    return torch.randn(T, Hq, D).to(dt), torch.randn(S, Hk, D).to(dt), torch.randn(S, Hk, D).to(dt)


def cu(*n):
    return torch.tensor(n, dtype=torch.int32)


def attention(q, k, v):
    return ops.packed_attention(q, k, v, cu(0, 4))


def rotated(q, k, v):
    return ops.norm_rotate(q, k, None, None, torch.ones(4, 8), torch.ones(4, 8))


CALLS = {"packed_attention": attention, "norm_rotate": rotated}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("train", [False, True])
def test_a_traced_call_is_recorded(name, train):
    """make_fx records the operator (and with gradients its backward), not memory that nobody fills."""
    def f(*args):
        args = [t.detach().requires_grad_(train) for t in args]
        out = CALLS[name](*args)
        out = out if isinstance(out, tuple) else (out,)
        return (*out, *torch.autograd.grad([o.sum() for o in out], args[:2])) if train else out

    args = qkv()
    graph = make_fx(f, tracing_mode="fake")(*args).graph
    called = [str(n.target) for n in graph.nodes if n.op == "call_function"]
    assert f"uplift_b200.{name}.default" in called
    assert (f"uplift_b200.{name}_backward.default" in called) == train
    assert not any("empty" in n for n in called)


@pytest.mark.parametrize("name", CALLS)
def test_dispatch_modes_see_the_call(name):
    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with FakeTensorMode():
        args = qkv(dt=torch.bfloat16)
        with Log():
            CALLS[name](*args)
    assert f"uplift_b200.{name}.default" in seen


@pytest.mark.parametrize("name", CALLS)
def test_tensor_subclasses_are_handed_to_the_operator(name):
    """Fake tensors outside of their mode: shapes and types, no launch."""
    mode = FakeTensorMode()
    args = [mode.from_tensor(t) for t in qkv(dt=torch.float16)]
    extra = [mode.from_tensor(t) for t in (cu(0, 4), torch.ones(4, 8))]
    if name == "packed_attention":
        out = ops.packed_attention(*args, extra[0])
        assert out.shape == args[0].shape and out.dtype == torch.float16
    else:
        a, b = ops.norm_rotate(args[0], args[1], None, None, extra[1], extra[1])
        assert a.shape == args[0].shape and b.shape == args[1].shape


def test_functionalized_calls_are_recorded():
    def f(q, k, v):
        return attention(q, k, v) + 1
    graph = make_fx(torch.func.functionalize(f), tracing_mode="fake")(*qkv()).graph
    assert any("uplift_b200.packed_attention" in str(n.target) for n in graph.nodes)


# ----------------------------------------------------------------- refusals
def test_heads_without_channels_and_single_numbers_are_refused():
    """Also with the default scale, D ** -0.5."""
    q, k, v = qkv()
    for bad in ((q[..., :0], k[..., :0], v[..., :0]), (q.sum(), k, v), (q.sum(), k.sum(), v.sum()), (q, k.sum(), v)):
        for kw in ({}, {"cu_k": cu(0, 4)}, {"scale": 0.5}):
            with pytest.raises(ValueError):
                ops.packed_attention(*bad, cu(0, 4), **kw)
        with pytest.raises(ValueError):
            ops.norm_rotate(bad[0], bad[1], None, None, torch.ones(4, 8), torch.ones(4, 8))


def test_more_sequences_than_the_kernels_count_are_refused():
    q, k, v = qkv()
    many = cu(0).expand(1 << 31)
    with pytest.raises(ValueError, match="at most"):
        ops.packed_attention(q, k, v, many)
    lib = _native.load(build_if_missing=True)
    rows = [16, 128, 64] * 9
    for B in ((1 << 31) - 1, (1 << 31) - 65536):
        args = tokens._PA_ARGS.pack(tokens._PA_ARGS.size, *rows, 16, 16, 16, 16, 0, 16, 1 << 40, 40, 4, B, 2, 1, 64,
                                    0.125, 1, _native.BF16, 0)
        assert lib.uplift_tok_attention_forward(args, None) == _native.ERR_SHAPE
        assert lib.uplift_tok_attention_backward(args, None) == _native.ERR_SHAPE


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("which", [0, 1])
def test_forward_mode_derivatives_are_refused(name, which):
    """Tangents would be left out of the result without an error."""
    from torch.autograd import forward_ad
    with FakeTensorMode(), forward_ad.dual_level():
        args = list(qkv())
        CALLS[name](*args)  # no tangents: as ever
        args[which] = forward_ad.make_dual(args[which], torch.randn(args[which].shape))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[name](*args)
    args = qkv()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda *a: CALLS[name](*a), args, tuple(torch.ones_like(a) for a in args))
