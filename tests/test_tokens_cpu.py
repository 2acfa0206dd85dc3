"""Refusals of the token-sequence operators, and their 64-bit restatements
against differences: no GPU."""
import pytest
import torch

import tokens_reference as R
from uplift_b200 import _native, ops, tokens


@pytest.fixture(scope="module")
def lib():
    return _native.load(build_if_missing=True)


def _attn_args(kw):
    a = dict(q=16, k=16, v=16, out=16, lo=0, dout=16, dq=16, dk=16, dv=16, st=(128, 64), lse=16, delta=16, cu=16, ws=0,
             ws_bytes=0, B=1, T=40, S=4, Hq=2, Hk=1, D=64, scale=0.125, causal=1, dtype=_native.BF16,
             size=tokens._PA_ARGS.size)
    a.update(kw)
    rows = [x for n in ("q", "k", "v", "out", "lo", "dout", "dq", "dk", "dv") for x in (a[n], *a["st"])]
    return tokens._PA_ARGS.pack(a["size"], *rows, a["lse"], a["delta"], a["cu"], a["cu"], 0, a["ws"], a["ws_bytes"],
                                a["T"], a["S"], a["B"], a["Hq"], a["Hk"], a["D"], a["scale"], a["causal"], a["dtype"],
                                0)


def _attn(lib, **kw):
    return lib.uplift_tok_attention_forward(_attn_args(kw), None)


def _attn_bwd(lib, **kw):
    return lib.uplift_tok_attention_backward(_attn_args(kw), None)


def _nr_args(kw):
    a = dict(q=16, k=16, qo=16, ko=16, dq=16, dk=16, st=(128, 64), wt=0, cos=16, pos=0, dw=0, partial=0, T=4, P=8,
             Hq=2, Hk=1, D=64, R=64, eps=1e-6, dtype=1, size=tokens._NR_ARGS.size)
    a.update(kw)
    rows = [x for n in ("q", "k", "qo", "ko", "dq", "dk") for x in (a[n], *a["st"])]
    return tokens._NR_ARGS.pack(a["size"], *rows, 0, 0, a["cos"], a["cos"], a["pos"], a["dw"], a["partial"], a["T"],
                                a["P"], a["Hq"], a["Hk"], a["D"], a["R"], a["eps"], 0, a["wt"], 0, a["dtype"], 0)


def _nr(lib, **kw):
    return lib.uplift_tok_norm_rotate(_nr_args(kw), None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=5), "ERR_ARG"), (dict(Hq=3, Hk=2), "ERR_SHAPE"), (dict(Hk=0), "ERR_SHAPE"), (dict(D=0), "ERR_SHAPE"),
    (dict(D=136), "ERR_SHAPE"), (dict(D=60), "ERR_SHAPE"), (dict(B=-1), "ERR_SHAPE"), (dict(T=-1), "ERR_SHAPE"),
    (dict(T=1 << 31), "ERR_SHAPE"), (dict(S=1 << 31), "ERR_SHAPE"), (dict(scale=0.0), "ERR_ARG"),
    (dict(scale=-1.0), "ERR_ARG"), (dict(scale=float("nan")), "ERR_ARG"), (dict(scale=float("inf")), "ERR_ARG"),
    (dict(q=0), "ERR_ARG"), (dict(out=0), "ERR_ARG"), (dict(cu=0), "ERR_ARG"), (dict(q=8), "ERR_LAYOUT"),
    (dict(lo=8), "ERR_LAYOUT"),
    (dict(st=(132, 64)), "ERR_LAYOUT"), (dict(st=(128, 4)), "ERR_LAYOUT"), (dict(st=(0, 64)), "ERR_LAYOUT"),
    (dict(size=8), "ERR_ARG"),
])
def test_attention_entry_refuses(lib, kw, code):
    assert _attn(lib, **kw) == getattr(_native, code)
    assert lib.uplift_la_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=-1), "ERR_ARG"), (dict(lse=0), "ERR_ARG"), (dict(delta=0), "ERR_ARG"),
    (dict(dout=0), "ERR_ARG"), (dict(out=0), "ERR_ARG"), (dict(v=24), "ERR_LAYOUT"),
    (dict(D=129), "ERR_SHAPE"), (dict(Hq=5, Hk=2), "ERR_SHAPE"), (dict(cu=0), "ERR_ARG"),
    # more items than a 32-bit counter holds: one per sequence, 128 rows and head
    (dict(B=1 << 26, T=1 << 26, Hq=32, Hk=1), "ERR_SHAPE"), (dict(B=1 << 26, S=1 << 26, Hq=32, Hk=32), "ERR_SHAPE"),
])
def test_attention_backward_entry_refuses(lib, kw, code):
    assert _attn_bwd(lib, **kw) == getattr(_native, code)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=9), "ERR_ARG"), (dict(wt=9), "ERR_ARG"), (dict(D=257), "ERR_SHAPE"), (dict(D=0), "ERR_SHAPE"),
    (dict(R=63), "ERR_SHAPE"), (dict(R=66), "ERR_SHAPE"), (dict(R=-2), "ERR_SHAPE"), (dict(P=3), "ERR_SHAPE"),
    (dict(Hq=0), "ERR_SHAPE"), (dict(T=-1), "ERR_SHAPE"), (dict(eps=-1.0), "ERR_ARG"),
    (dict(eps=float("nan")), "ERR_ARG"), (dict(q=0), "ERR_ARG"), (dict(cos=0), "ERR_ARG"),
    (dict(size=8), "ERR_ARG"),
])
def test_norm_rotate_entry_refuses(lib, kw, code):
    assert _nr(lib, **kw) == getattr(_native, code)
    assert lib.uplift_tok_norm_rotate_backward(_nr_args(kw), None) == getattr(_native, code)


def test_no_arguments_at_all(lib):
    for name in ("norm_rotate", "norm_rotate_backward", "attention_forward", "attention_backward"):
        assert getattr(lib, "uplift_tok_" + name)(None, None) == _native.ERR_ARG


def test_backward_and_step_workspaces(lib):
    assert lib.uplift_tok_norm_rotate_backward(_nr_args(dict(dw=16)), None) == _native.ERR_ARG
    assert lib.uplift_tok_norm_rotate_backward(_nr_args(dict(dq=0)), None) == _native.ERR_ARG
    need = lib.uplift_tok_attention_workspace(4, 4, 100, 8, 2, 64, _native.BF16)
    assert need > 0 and lib.uplift_tok_attention_workspace(4, 4, 100, 8, 2, 64, _native.F32) == 0
    assert lib.uplift_tok_attention_workspace(4000, 4000, 100, 8, 2, 64, _native.BF16) == 0  # a chunk per token
    step = dict(B=4, T=4, S=100, Hq=8, Hk=2, st=(512, 64))
    assert _attn(lib, **step) == _native.ERR_ARG
    assert _attn(lib, ws=16, ws_bytes=need - 1, **step) == _native.ERR_ARG
    assert _attn(lib, ws=24, ws_bytes=need, **step) == _native.ERR_ARG


def test_empty_calls_touch_no_device(lib):
    assert _attn(lib, T=0) == _native.OK
    assert _attn_bwd(lib, T=0, S=0) == _native.OK
    assert _attn_bwd(lib, T=0, S=0, B=0, cu=0) == _native.OK
    assert _nr(lib, T=0) == _native.OK
    assert lib.uplift_tok_norm_rotate_partial_floats(64) > 0


def _qkv(T=4, S=4, Hq=2, Hk=1, D=16, dt=torch.float32):
    return torch.randn(T, Hq, D).to(dt), torch.randn(S, Hk, D).to(dt), torch.randn(S, Hk, D).to(dt)


def _cu(*n):
    return torch.tensor(n, dtype=torch.int32)


def test_packed_attention_refuses():
    q, k, v = _qkv()
    cu = _cu(0, 4)
    for bad in (dict(q=q.double()), dict(k=k.half()), dict(v=v[:3]), dict(q=q[..., :8]), dict(q=q[0]),
                dict(cu_q=cu.long()), dict(cu_k=_cu(0, 2, 4)), dict(cu_q=cu[None]), dict(used_k=_cu(1, 2)),
                dict(used_k=torch.tensor([4.0])), dict(scale=0.0), dict(scale=float("inf")),
                dict(q=torch.randn(4, 3, 16), k=torch.randn(4, 2, 16), v=torch.randn(4, 2, 16)),
                dict(q=torch.randn(4, 2, 136), k=torch.randn(4, 1, 136), v=torch.randn(4, 1, 136)),
                dict(q=q.bfloat16()[..., :12], k=k.bfloat16()[..., :12], v=v.bfloat16()[..., :12]),
                dict(cu_q=_cu(), cu_k=_cu()), dict(k=k[:, :0], v=v[:, :0])):
        args = dict(q=q, k=k, v=v, cu_q=cu, cu_k=cu)
        args.update(bad)
        with pytest.raises(ValueError):
            ops.packed_attention(**args)
    with pytest.raises(ValueError, match="pass cu_k"):
        ops.packed_attention(q, k[:3], v[:3], cu)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.packed_attention(q, k, v, cu)


def test_norm_rotate_refuses():
    q, k, _ = _qkv()
    cos = torch.ones(8, 8)
    w = torch.ones(16)
    ok = dict(q=q, k=k, q_weight=w, k_weight=w, cos=cos, sin=cos)
    for bad in (dict(q=q.double()), dict(k=k[:3]), dict(k=k[..., :8]), dict(q_weight=w[:8]), dict(q_weight=w.double()),
                dict(k_weight=w.half()), dict(cos=cos.half()), dict(sin=cos[:4]), dict(cos=cos[:3], sin=cos[:3]),
                dict(cos=torch.ones(8, 9), sin=torch.ones(8, 9)), dict(positions=torch.zeros(3, dtype=torch.int32)),
                dict(positions=torch.zeros(4)), dict(cos=cos.clone().requires_grad_()),
                dict(q=torch.randn(4, 1, 264), k=torch.randn(4, 1, 264), q_weight=None, k_weight=None)):
        args = dict(ok)
        args.update(bad)
        with pytest.raises(ValueError):
            ops.norm_rotate(**args)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.norm_rotate(**ok)


def test_operators_are_traced_under_fake_tensors():
    """The custom ops have fake kernels with the outputs' shapes and types."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k, v = _qkv(dt=torch.bfloat16)
        out, lse, lo = torch.ops.uplift_b200.packed_attention(q, k, v, _cu(0, 4), _cu(0, 4), None, True, 0.25, True, True)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (2, 4) and lse.dtype == torch.float32
        assert lo.shape == q.shape and lo.dtype == q.dtype
        a, b = torch.ops.uplift_b200.norm_rotate(q, k, None, None, torch.ones(4, 8), torch.ones(4, 8), None, 1e-6, False)
        assert a.shape == q.shape and b.shape == k.shape


# ---------------------------------------- the restatements against differences
def _difference(f, x, d, h=1e-5):
    return (f(x + h * d) - f(x - h * d)) / (2 * h)


@pytest.mark.parametrize("causal", [True, False])
def test_reference_attention_gradients_are_differences(causal):
    torch.manual_seed(0)
    q, k, v = (t.double() for t in _qkv(T=7, S=9, Hq=4, Hk=2, D=8))
    cu_q, cu_k, used = _cu(0, 5, 7), _cu(0, 3, 9), torch.tensor([3, 5], dtype=torch.int32)
    g = torch.randn_like(q)
    r = R.attention(q, k, v, cu_q, cu_k, used, causal, 0.3, g)
    for n, i in (("dq", 0), ("dk", 1), ("dv", 2)):
        d = torch.randn_like((q, k, v)[i])

        def f(x):
            args = [q, k, v]
            args[i] = x
            return (R.attention(*args, cu_q, cu_k, used, causal, 0.3)["out"] * g).sum()

        # central differences with h = 1e-5: h^2 times third derivatives (order 1 here), 1e-16 / h of cancellation
        assert abs(_difference(f, (q, k, v)[i], d) - (r[n] * d).sum()) < 1e-8


@pytest.mark.parametrize("interleaved", [True, False])
def test_reference_norm_rotate_gradients_are_differences(interleaved):
    torch.manual_seed(0)
    x, w, g = torch.randn(5, 2, 8).double(), torch.randn(8).double(), torch.randn(5, 2, 8).double()
    ang = torch.randn(6, 3).double()
    pos = torch.tensor([3, -1, 0, 5, 2])
    args = (ang.cos(), ang.sin(), pos, 1e-3, interleaved)
    _, dx, dw = R.norm_rotate(x, w, *args, g=g)
    d = torch.randn_like(x)
    assert abs(_difference(lambda t: (R.norm_rotate(t, w, *args) * g).sum(), x, d) - (dx * d).sum()) < 1e-8
    e = torch.randn_like(w)
    assert abs(_difference(lambda t: (R.norm_rotate(x, t, *args) * g).sum(), w, e) - (dw * e).sum()) < 1e-8
