"""The token-sequence operators where masks, types and forms meet: what a
masked row may not reach in the gradients, gradients of any size, and the weight
gradients of the forms that take several heads at a time."""
import json
import math

import pytest
import torch

import tokens_reference as R
from uplift_b200 import _native, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _lib(cuda_lib):
    yield
    assert _native.device_status(clear=True) == 0  # no bounded wait ran out


def starts(lens, first=0):
    return torch.tensor([first] + [first + sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32, device=DEV)


def rand(gen, *shape, dt=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(DEV).to(dt)


def qkv(gen, T, S, Hq, Hk, D, dt, scale=1.3):
    return rand(gen, T, Hq, D, dt=dt, scale=scale), rand(gen, S, Hk, D, dt=dt, scale=scale), rand(gen, S, Hk, D, dt=dt)


def attention_and_gradients(q, k, v, g, *args, **kw):
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out = ops.packed_attention(*leaves, *args, **kw)
    return (out.detach(), *torch.autograd.grad(out, leaves, g))


# ------------------------------------------------- gradients behind the mask
KINDS = [(BF16, 128), (F16, 64), (BF16, 80), (F32, 64)]


@pytest.mark.parametrize("dt,D", KINDS)
@pytest.mark.parametrize("Hq,Hk", [(2, 1), (3, 3), (4, 2)])
@pytest.mark.parametrize("n_q,n_k", [(300, 300), (130, 333), (333, 130)])
@pytest.mark.parametrize("at", [1, 63, 64, 100, 128])
def test_later_keys_do_not_reach_gradients_of_earlier_queries(dt, D, Hq, Hk, n_q, n_k, at):
    """Causal: NaN and infinities in keys and values from `at` on leave dq of the queries that see none of them as it
    was (zero for those that see no key), and make that of the others NaN."""
    gen = torch.Generator().manual_seed(51)
    q, k, v = qkv(gen, n_q + 20, n_k + 20, Hq, Hk, D, dt)
    g = rand(gen, *q.shape, dt=dt)
    cu = starts([n_q, 20]), starts([n_k, 20])
    out, dq, _, _ = attention_and_gradients(q, k, v, g, *cu)
    k[at:n_k], v[at + 1:n_k] = math.nan, math.inf
    got, got_dq, _, _ = attention_and_gradients(q, k, v, g, *cu)
    hidden = torch.arange(n_q + 20, device=DEV) + n_k - n_q < at  # the last key that they see is before `at`
    hidden[n_q:] = True  # the other sequence
    assert torch.equal(got[hidden], out[hidden])
    assert torch.equal(got_dq[hidden], dq[hidden])
    assert bool(got_dq[~hidden].isnan().all())
    if n_q > n_k:
        assert not got_dq[:n_q - n_k].any()


@pytest.mark.parametrize("dt,D", KINDS)
@pytest.mark.parametrize("Hq,Hk", [(2, 1), (3, 3), (4, 2)])
@pytest.mark.parametrize("n_q,n_k", [(300, 300), (130, 333), (333, 130)])
@pytest.mark.parametrize("end", [1, 64, 100, 128])
def test_earlier_queries_do_not_reach_gradients_of_later_keys(dt, D, Hq, Hk, n_q, n_k, end):
    """Causal: NaN in the first `end` queries and infinities in their outputs' gradients leave dk and dv of the keys
    that none of them sees as they were."""
    gen = torch.Generator().manual_seed(53)
    q, k, v = qkv(gen, n_q + 20, n_k + 20, Hq, Hk, D, dt)
    g = rand(gen, *q.shape, dt=dt)
    cu = starts([n_q, 20]), starts([n_k, 20])
    _, _, dk, dv = attention_and_gradients(q, k, v, g, *cu)
    q[:end:2], g[:end] = math.nan, math.inf
    _, _, got_dk, got_dv = attention_and_gradients(q, k, v, g, *cu)
    hidden = torch.arange(n_k + 20, device=DEV) > end - 1 + n_k - n_q
    hidden[n_k:] = True
    assert torch.equal(got_dk[hidden], dk[hidden]) and torch.equal(got_dv[hidden], dv[hidden])
    assert not bool(got_dk[~hidden].isfinite().any()) and not bool(got_dv[~hidden].isfinite().any())


@pytest.mark.parametrize("dt,D", KINDS)
@pytest.mark.parametrize("row", [0, 70, 127, 128, 200, 299])
def test_an_infinite_gradient_reaches_the_keys_that_its_query_sees(dt, D, row):
    """One infinity in the outputs' gradient: its channel of dv is infinite for the keys that the query sees, and the
    other channels are as they were; dk is not finite there."""
    gen = torch.Generator().manual_seed(55)
    q, k, v = qkv(gen, 300, 300, 4, 2, D, dt, scale=0.3)
    g = rand(gen, *q.shape, dt=dt)
    cu = starts([300])
    _, _, dk, dv = attention_and_gradients(q, k, v, g, cu)
    g[row, 1, 5] = -math.inf
    _, dq, got_dk, got_dv = attention_and_gradients(q, k, v, g, cu)
    assert bool((got_dv[:row + 1, 0, 5] == -math.inf).all()) and not bool(got_dk[:row + 1, 0].isfinite().any())
    got_dv[:row + 1, 0, 5] = dv[:row + 1, 0, 5]
    got_dk[:row + 1, 0] = dk[:row + 1, 0]
    assert torch.equal(got_dv, dv) and torch.equal(got_dk, dk)
    assert dq.isfinite().all(-1).sum() == 300 * 4 - 1


# ------------------------------------------------- maxima that grow all along
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("Hq,Hk", [(4, 2), (3, 3)])
@pytest.mark.parametrize("causal", [True, False])
def test_maxima_that_grow_in_every_tile(dt, D, Hq, Hk, causal):
    """Scores that rise by about 9 powers of two per 64 keys for some rows, less for others: sums are rescaled in
    every key tile, and each run gives the same bits."""
    gen = torch.Generator().manual_seed(63)
    n = 1500
    q, k, v = qkv(gen, n, n, Hq, Hk, D, dt, scale=0.5)
    rise = torch.arange(n, device=DEV)[:, None] * (9 * math.log(2) / 64 / 16)
    q[:, :, 0] = torch.randint(4, 18, (n, Hq), generator=gen).to(DEV)
    k[:, :, 0] = rise.to(dt)
    run = [ops.packed_attention(q, k, v, starts([n]), causal=causal, scale=1.0, return_lse=True) for _ in range(10)]
    assert all(torch.equal(a, b) for r in run[1:] for a, b in zip(r, run[0]))
    ref = R.attention(q, k, v, starts([n]), starts([n]), None, causal, 1.0, None, dt)
    R.check(run[0][0], ref["out"], ref["out_tol"], "out")
    R.check(run[0][1], ref["lse"], ref["lse_tol"], "lse")


# --------------------------------------- values shared by two query tiles
@pytest.mark.parametrize("dt,D", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("Hq,Hk", [(3, 3), (3, 1), (2, 1)])
@pytest.mark.parametrize("key", [0, 70, 127, 150])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_an_infinite_value_of_no_weight_gives_one_result(dt, D, Hq, Hk, key, bad):
    """A value that is not finite, with a weight that rounds to zero for the rows from 128 on: wherever the row of
    tiles takes it from, every run gives the same bits, rows that do not see it are as they were, and the others of
    its item are not finite in its channel alone."""
    gen = torch.Generator().manual_seed(65)
    n = 300
    q, k, v = qkv(gen, n, n, Hq, Hk, D, dt, scale=0.5)
    q[:, :, 0], k[:, :, 0] = 0, 0
    q[128:, :, 0], k[key, :, 0] = 30, -40  # a score of -1200 D^-1/2: exp of it is below 2^-150
    clean = ops.packed_attention(q, k, v, starts([n]))
    v[key, 0, 3] = bad
    first = ops.packed_attention(q, k, v, starts([n]))
    for _ in range(40):
        again = ops.packed_attention(q, k, v, starts([n]))
        assert torch.equal(again.view(torch.int16), first.view(torch.int16))
    heads = Hq // Hk
    assert torch.equal(first[:key], clean[:key]) and torch.equal(first[:, heads:], clean[:, heads:])
    item = 256 if heads % 2 else 128
    seen = first[key:item, :heads, 3]
    assert bool((seen == bad).all()) if bad == math.inf else bool(seen.isnan().all())
    first[key:, :heads, 3] = clean[key:, :heads, 3]
    assert torch.equal(first, clean)


# ------------------------------------------------------------------ tracers
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("tracer", ["make_fx", "jit"])
def test_a_trace_computes_what_the_call_does(dt, tracer):
    """A recorded call (with its gradients, where the tracer takes them), run on other inputs."""
    from torch.fx.experimental.proxy_tensor import make_fx
    gen = torch.Generator().manual_seed(67)
    one, two = (qkv(gen, 90, 90, 4, 2, 64, dt) for _ in range(2))
    g = rand(gen, 90, 4, 64, dt=dt)
    cu, ang = starts([30, 60]), rand(gen, 90, 32)
    cos, sin, w = ang.cos(), ang.sin(), 1 + rand(gen, 64, scale=0.2).to(dt)

    def f(q, k, v):
        a, b = ops.norm_rotate(q, k, w, w, cos, sin)
        return ops.packed_attention(a, b, v, cu)

    def step(q, k, v):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(f(*leaves), leaves, g)

    if tracer == "make_fx":
        assert torch.equal(make_fx(f)(*one)(*two), f(*two))
        assert all(torch.equal(a, b) for a, b in zip(make_fx(step)(*one)(*two), step(*two)))
    else:
        assert torch.equal(torch.jit.trace(f, one, check_trace=False)(*two), f(*two))


# --------------------------------------------------------- gradients in fp16
def test_large_gradients_in_fp16():
    """dO of some 10^4: P (dP - delta) exceeds the largest fp16 value (9 10^4), the gradients do not."""
    gen = torch.Generator().manual_seed(57)
    n_q, n_k = [4, 3, 5, 2, 130], [2, 3, 8, 1, 4]
    q, k, v = qkv(gen, sum(n_q), sum(n_k), 4, 2, 64, F16, scale=0.3)
    v = 2 * v
    g = rand(gen, *q.shape, scale=8000.0).clamp(-6e4, 6e4).to(F16)
    g[-130:] *= 2.0 ** -6
    ref = R.attention(q, k, v, starts(n_q), starts(n_k), None, False, None, g, F16)
    most = max(ref[n].abs().max().item() for n in ("dq", "dk", "dv"))
    assert most < 6e4  # all of them are fp16 values
    _, *grads = attention_and_gradients(q, k, v, g, starts(n_q), starts(n_k), causal=False)
    for n, d in zip(("dq", "dk", "dv"), grads):
        R.check(d, ref[n], ref[n + "_tol"], n)


@pytest.mark.parametrize("causal", [True, False])
def test_small_gradients_in_fp16(causal):
    """dO of some 2^-19 on a thousand keys: score gradients of 10^-9, below the smallest fp16 value, times keys of
    some hundred.  dS may be off by u of itself and, among the subnormals, by 2^-25 where the largest |dO|
    is brought to 2^-5 .. 2^-4; P by 2^-33."""
    gen = torch.Generator().manual_seed(59)
    n, D, u = 1000, 64, 2.0 ** -11
    q, k, v = rand(gen, n, 2, D, dt=F16, scale=0.01), rand(gen, n, 2, D, dt=F16, scale=100.0), rand(gen, n, 2, D, dt=F16)
    g = rand(gen, n, 2, D, scale=2.0 ** -19).to(F16)
    _, dq, _, dv = attention_and_gradients(q, k, v, g, starts([n]), causal=causal)
    scale = D ** -0.5
    seen = torch.ones(n, n, dtype=torch.bool, device=DEV)
    seen = seen.tril() if causal else seen
    for h in range(2):
        qs, ks, vs, gs = (t[:, h].double() for t in (q, k, v, g))
        p = (qs @ ks.T * scale).masked_fill(~seen, -math.inf).softmax(1)
        dp = gs @ vs.T
        ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
        # scores, exponentials and sums in fp32: as in tokens_reference
        c = 2 * (scale * (D + 4) * 2 * R.F32 * (qs.abs() @ ks.abs().T).max() + 2.0 ** -20) + 2 * n * R.F32
        size = (gs.abs() @ vs.abs().T + (p @ (gs.abs() @ vs.abs().T).T).diagonal()[:, None]) * p * scale
        # delta: that of out and what its rounding left, u^2 of it, and of the weights' rounding
        e = (u + 2 * c) * ds.abs() + (2 * u + c + 2 * (D + 8) * R.F32) * size + 2.0 ** -20 * g.double().abs().max() * scale * seen
        want = ds @ ks
        R.check(dq[:, h], want, u * want.abs() + 2.0 ** -25 + (e + 2 * n * R.F32 * ds.abs()) @ ks.abs(), f"dq {h}")
        want = p.T @ gs
        tol = ((u + c + 2 * n * R.F32) * p + 2.0 ** -33 * seen).T @ gs.abs()
        R.check(dv[:, h], want, u * want.abs() + 2.0 ** -25 + tol, f"dv {h}")



def test_padding_does_not_set_the_size_of_gradients_in_fp16():
    """Rows of no sequence hold the largest fp16 values; the gradients of the others are as without them."""
    gen = torch.Generator().manual_seed(60)
    q, k, v = qkv(gen, 400, 400, 2, 1, 64, F16)
    g = rand(gen, 400, 2, 64, scale=2.0 ** -18).to(F16)
    cu = starts([150, 180], 20)
    _, *clean = attention_and_gradients(q, k, v, g, cu)
    g[:20], g[350:] = 65504.0, -65504.0
    _, *grads = attention_and_gradients(q, k, v, g, cu)
    assert all(torch.equal(a, b) for a, b in zip(grads, clean))


def test_many_equal_weights_in_fp16():
    """200,000 keys of equal weight, 5 10^-6: each key's dv is that times dO, off by the weight's rounding (2^-33 at
    most, and u), a few steps of fp32 and its own rounding."""
    gen = torch.Generator().manual_seed(62)
    n, u = 200_000, 2.0 ** -11
    q, k, v = rand(gen, 1, 2, 64, dt=F16), torch.zeros(n, 1, 64, dtype=F16, device=DEV), rand(gen, n, 1, 64, dt=F16)
    g = rand(gen, 1, 2, 64, scale=20000.0).clamp(-6e4, 6e4).to(F16)
    _, _, _, dv = attention_and_gradients(q, k, v, g, starts([1]), starts([n]))
    want = g.double().sum(1) / n
    tol = (g.double().abs() * (u / n + 2.0 ** -33 + 2.0 ** -18 / n)).sum(1) + u * want.abs() + 2.0 ** -25
    R.check(dv[:, 0], want.expand(n, 64), tol.expand(n, 64), "dv")


# ------------------------------------------------------- a limit on the CTAs
@pytest.mark.parametrize("dt", [BF16, F16])
def test_a_limit_on_the_ctas_holds_and_changes_no_result(dt, tmp_path):
    """uplift_la_set_max_ctas: no more CTAs of these kernels at a time, in prompts, gradients and steps."""
    gen = torch.Generator().manual_seed(69)
    q, k, v = qkv(gen, 900, 900, 8, 2, 64, dt)
    g, cu = rand(gen, 900, 8, 64, dt=dt), starts([500, 300, 100])
    one, room = starts([1] * 3), starts([300] * 3)

    def run():
        return (*attention_and_gradients(q, k, v, g, cu), ops.packed_attention(q[:3], k, v, one, room))

    full = run()
    try:
        for n in (37, 1):
            _native.set_max_ctas(n)
            assert all(torch.equal(a, b) for a, b in zip(full, run()))
            with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
                run()
                torch.cuda.synchronize()
            prof.export_chrome_trace(str(tmp_path / "trace.json"))
            events = json.loads((tmp_path / "trace.json").read_text())["traceEvents"]
            ran = [(e["ts"], e["ts"] + e["dur"], e["args"]["grid"], e["name"]) for e in events
                   if e.get("cat") == "kernel" and any(s in e["name"] for s in ("attention_kernel", "gradient_kernel", "chunk_kernel"))]
            assert len(ran) == 4, ran
            assert all(grid[0] * grid[1] * grid[2] <= n for _, _, grid, _ in ran), ran
            dq, dkv = sorted(e for e in ran if "gradient_kernel" in e[3])
            assert dkv[0] >= dq[1], ran
    finally:
        _native.set_max_ctas(0)


# ------------------------------------- weight gradients over all of the rows
def norm_rotate_sums(x, w, cos, sin, pos, eps, interleaved, g):
    """z, dx and dw in 64 bits, and the sums of absolute values that their errors are counted from."""
    x, g, w = x.double(), g.double(), w.double()
    half = cos.shape[1]
    a, b = R.pair_index(2 * half, interleaved)
    there = (pos >= 0)[:, None, None]
    c = torch.where(there, cos[pos.clamp(min=0).long()].double()[:, None], 1.0)
    s = torch.where(there, sin[pos.clamp(min=0).long()].double()[:, None], 0.0)

    def turned(y, c, s):
        z = y.clone()
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
        return z

    r = 1.0 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    h = x * r
    gy, ga = turned(g, c, -s), g.abs()
    ga[..., a], ga[..., b] = (g.abs()[..., i] * c.abs() + g.abs()[..., j] * s.abs() for i, j in ((a, b), (b, a)))
    gw, gwa = gy * w, ga * w.abs()
    dx = r * (gw - h * (gw * h).mean(-1, keepdim=True))
    dxa = r * (gwa + h.abs() * (gwa * h.abs()).mean(-1, keepdim=True))
    return turned(h * w, c, s), dx, (gy * h).sum((0, 1)), dxa, (ga * h.abs()).sum((0, 1))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt,wdt,T,Hq,Hk,D,rot", [
    (BF16, BF16, 3001, 10, 5, 64, 64), (F16, F32, 1203, 13, 6, 128, 64), (F32, F32, 1501, 6, 3, 128, 128),
    (BF16, F32, 1100, 8, 2, 256, 256), (F32, F32, 2003, 9, 10, 64, 32), (F16, F16, 160, 300, 7, 64, 64),
    (BF16, BF16, 130, 5, 290, 96, 96), (F32, F32, 700, 9, 5, 256, 128), (BF16, BF16, 1500, 9, 6, 36, 36)])
def test_weight_gradients_of_many_rows(dt, wdt, T, Hq, Hk, D, rot, interleaved):
    """Calls large enough for the forms that take several heads per group of lanes (and two that run a warp per row):
    every dx and the sums over all rows, with weights of their own for queries and keys."""
    gen = torch.Generator().manual_seed(61)
    P = 997
    q, k = rand(gen, T, Hq, D, dt=dt, scale=2.0), rand(gen, T, Hk, D, dt=dt, scale=2.0)
    gq, gk = rand(gen, T, Hq, D, dt=dt), rand(gen, T, Hk, D, dt=dt)
    ang = torch.randn(P, rot // 2, generator=gen, dtype=torch.float64) * 10
    cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    pos = torch.randint(-1, P, (T,), generator=gen).int().to(DEV)
    wq, wk = (1 + rand(gen, D, scale=0.3)).to(wdt), (1 + rand(gen, D, scale=0.3)).to(wdt)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    out = ops.norm_rotate(*leaves, cos, sin, pos, 1e-6, interleaved)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    u, tiny = R.u_of(dt), torch.finfo(dt).tiny * R.u_of(dt) + 1e-30
    f = 2 * (D + 16) * R.F32  # of a term, as in tokens_reference
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        z, dx, dw, dxa, dwa = norm_rotate_sums(x.detach(), w.detach(), cos, sin, pos, 1e-6, interleaved, g)
        # |z| <= |a c| + |b s|: at most sqrt 2 of the pair's length
        pair = z.abs().amax(-1, keepdim=True)
        R.check(out[i], z, u * z.abs() + 2 * f * pair + tiny, ("q", "k")[i])
        R.check(grads[i], dx, u * dx.abs() + f * dxa + tiny, ("dq", "dk")[i])
        # a lane adds at most 32 rows in 32 bits, a block its groups (64 at most); the blocks are added in 64 bits
        R.check(grads[2 + i], dw, (f + 2 * (32 + 64) * R.F32) * dwa + R.u_of(wdt) * dw.abs(), ("dwq", "dwk")[i])


# ------------------------------------------------------ waits that run out
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("Hq,Hk", [(4, 2), (3, 3)])
@pytest.mark.parametrize("part", ["forward", "backward"])
def test_a_wait_that_runs_out_is_reported_and_the_context_survives(dt, D, Hq, Hk, part):
    """The producers stop loading after a few tiles, so every role's wait runs out or is ended by another's (20 ms
    here): the launch records it, drains and ends, the next call raises, and the one after that is right."""
    lib = _native.load()
    gen = torch.Generator().manual_seed(71)
    q, k, v = qkv(gen, 1000, 1000, Hq, Hk, D, dt)
    g, cu = rand(gen, *q.shape, dt=dt), starts([700, 300])
    want = attention_and_gradients(q, k, v, g, cu)  # also registers the host's word
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.packed_attention(*leaves, cu)
    torch.cuda.synchronize()
    _native.check(lib.uplift_la_test_hook(1, 20_000_000), "test hook")
    try:
        if part == "forward":
            ops.packed_attention(q, k, v, cu)
        else:
            torch.autograd.grad(out, leaves, g)
        torch.cuda.synchronize()
    finally:
        lib.uplift_la_test_hook(0, 0)
    with pytest.raises(_native.ExpiredWaitError):
        ops.packed_attention(q, k, v, cu)
    assert _native.device_status(clear=True) == 0  # raising cleared it
    assert all(torch.equal(a, b) for a, b in zip(attention_and_gradients(q, k, v, g, cu), want))
    assert _native.host_status.value() == 0


# ------------------------------------------- prompts among single tokens
@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("Hq,Hk", [(8, 2), (3, 3), (10, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_a_prompt_among_single_tokens(dt, D, Hq, Hk, causal):
    """Few queries per sequence on average, many in one: the eight-row form walks a prompt, with gradients."""
    gen = torch.Generator().manual_seed(73)
    n_q = [1] * 30 + [300] + [1, 0, 2] * 10
    n_k = [1 + 17 * i % 400 for i in range(30)] + [450] + [3, 5, 700] * 10
    q, k, v = qkv(gen, sum(n_q), sum(n_k), Hq, Hk, D, dt)
    assert sum(n_q) <= 8 * len(n_q)
    g = rand(gen, *q.shape, dt=dt)
    ref = R.attention(q, k, v, starts(n_q), starts(n_k), None, causal, None, g, dt)
    got = attention_and_gradients(q, k, v, g, starts(n_q), starts(n_k), causal=causal)
    for n, x in zip(("out", "dq", "dk", "dv"), got):
        R.check(x, ref[n], ref[n + "_tol"], n)


# ------------------------------------------------ offsets beyond 32 bits
def test_prompts_and_gradients_beyond_32_bit_offsets():
    """Queries and keys whose element offsets are above 2^31: results and gradients of the rows alone."""
    T, D = 2_200_000, 128
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    gen = torch.Generator().manual_seed(75)
    lens, n = [130, 170], 300
    small = [rand(gen, n, 8, D, dt=BF16) for _ in range(4)]
    want = attention_and_gradients(*small, starts(lens))
    large = []
    for t in small:
        x = torch.zeros(T, 8, D, dtype=BF16, device=DEV)
        x[-n:] = t
        large.append(x)
    got = attention_and_gradients(*large, starts(lens, T - n))
    for a, b in zip(got, want):
        assert torch.equal(a[-n:], b)
        assert not a[:T - n].any()
    cos, sin = (rand(gen, T, 64) for _ in range(2))
    a, _ = ops.norm_rotate(large[0], large[1][:, :1], None, None, cos, sin)
    b, _ = ops.norm_rotate(small[0], small[1][:, :1], None, None, cos[-n:], sin[-n:])
    assert torch.equal(a[-n:], b)
    assert not a[:T - n].any()


# -------------------------------------------------- captured fp16 gradients
def test_a_captured_fp16_step_takes_gradients_of_any_size():
    """A training step in a CUDA graph: the largest dO is found anew in each replay."""
    gen = torch.Generator().manual_seed(77)
    q, k, v = qkv(gen, 400, 400, 4, 2, 64, F16)
    g, cu = rand(gen, 400, 4, 64, dt=F16), starts([150, 250])
    static = g.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention_and_gradients(q, k, v, static, cu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attention_and_gradients(q, k, v, static, cu)
    for factor in (1.0, 2.0 ** 12, 2.0 ** -14, 0.0, 1.0):
        static.copy_(g * factor)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, attention_and_gradients(q, k, v, g * factor, cu)))
