"""The token-sequence operators on the GPU against their 64-bit
restatements: lengths from zero on, masks that leave rows without keys, odd
sizes, strides, streams, graphs, compile."""
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


def run_attention(q, k, v, cu_q, cu_k, used, causal, scale=None, grads=True, gen=None):
    """Forward (and backward) through the public entry, checked against 64 bits."""
    g = rand(gen, *q.shape, dt=q.dtype) if grads else None
    ref = R.attention(q, k, v, cu_q, cu_k, used, causal, scale, g, q.dtype)
    leaves = [t.detach().requires_grad_(grads) for t in (q, k, v)]
    out, lse = ops.packed_attention(*leaves, cu_q, cu_k, used_k=used, causal=causal, scale=scale, return_lse=True)
    R.check(out, ref["out"], ref["out_tol"], "out")
    R.check(lse, ref["lse"], ref["lse_tol"], "lse")
    if grads:
        for n, d in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, g)):
            R.check(d, ref[n], ref[n + "_tol"], n)
    return out


# (queries, keys) of each sequence
PACKS = {
    "one": [(1, 1)],
    "tiny": [(3, 3), (0, 0), (1, 1), (7, 7)],
    "tile": [(64, 64), (128, 128), (65, 65)],
    "ragged": [(129, 129), (17, 17), (300, 300), (1, 1), (255, 255)],
    "more keys": [(5, 70), (130, 200), (1, 257), (40, 300)],
    "fewer keys": [(70, 5), (200, 130), (3, 0), (300, 140), (64, 64)],
    "no queries": [(0, 50), (20, 20), (0, 3)],
}
HEADS = {"mha": (3, 3), "group": (4, 2), "one key head": (5, 1)}


@pytest.mark.parametrize("pack", PACKS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt,D", [(BF16, 64), (BF16, 128), (F16, 64), (F16, 128), (BF16, 8), (BF16, 80), (F16, 104),
                                  (F32, 64), (F32, 33), (F32, 128), (F32, 100)])
def test_attention_packs(pack, causal, dt, D):
    gen = torch.Generator().manual_seed(hash((len(pack), causal, D)) & 0xffff)
    n_q, n_k = zip(*PACKS[pack])
    q, k, v = qkv(gen, sum(n_q), sum(n_k), 4, 2, D, dt)
    run_attention(q, k, v, starts(n_q), starts(n_k), None, causal, gen=gen)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dt", [BF16, F32])
def test_attention_head_layouts(heads, dt):
    gen = torch.Generator().manual_seed(1)
    Hq, Hk = HEADS[heads]
    q, k, v = qkv(gen, 230, 230, Hq, Hk, 64, dt)
    run_attention(q, k, v, starts([100, 130]), starts([100, 130]), None, True, gen=gen)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (BF16, 80), (F32, 64)])
@pytest.mark.parametrize("Hq,Hk", [(8, 2), (3, 3), (16, 1), (24, 1), (7, 1)])
def test_single_tokens(dt, D, Hq, Hk):
    """One new token per sequence on histories from none to long, in segments with room."""
    gen = torch.Generator().manual_seed(2)
    n_k = [1, 2, 0, 63, 64, 65, 700, 1300, 129]
    seg = [n + n // 8 + 1 for n in n_k]
    q, k, v = qkv(gen, len(n_k), sum(seg), Hq, Hk, D, dt)
    used = torch.tensor(n_k, dtype=torch.int32, device=DEV)
    run_attention(q, k, v, starts([1] * len(n_k)), starts(seg), used, True, grads=False, gen=gen)


@pytest.mark.parametrize("causal", [True, False])
def test_a_few_tokens_on_long_histories(causal):
    gen = torch.Generator().manual_seed(3)
    n_q, n_k = [3, 1, 0, 5, 2], [2000, 3, 9, 515, 1]
    q, k, v = qkv(gen, sum(n_q), sum(n_k), 8, 2, 64, BF16)
    run_attention(q, k, v, starts(n_q), starts(n_k), None, causal, gen=gen)


def test_a_step_of_many_sequences():
    """So many that every token's keys are one chunk (no workspace), some without keys."""
    gen = torch.Generator().manual_seed(47)
    n_q, n_k = [1 + (i % 3 == 0) for i in range(500)], [(i * 13) % 90 for i in range(500)]
    assert _native.load().uplift_tok_attention_workspace(500, sum(n_q), sum(n_k), 16, 8, 64, _native.BF16) == 0
    q, k, v = qkv(gen, sum(n_q), sum(n_k), 16, 8, 64, BF16)
    run_attention(q, k, v, starts(n_q), starts(n_k), None, True, grads=False, gen=gen)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_gradients_in_segments_with_room(dt, D, causal):
    """Rows of a key segment behind used_k, NaN here, reach nothing, and their gradients are zero."""
    gen = torch.Generator().manual_seed(31)
    n_q, n_k, seg = [40, 70, 3], [55, 130, 0], [64, 150, 9]
    q, k, v = qkv(gen, sum(n_q), sum(seg), 4, 2, D, dt)
    used = torch.tensor(n_k, dtype=torch.int32, device=DEV)
    room = torch.cat([torch.arange(s, device=DEV) >= n for s, n in zip(seg, n_k)])
    g = rand(gen, *q.shape, dt=dt)
    ref = R.attention(q, k, v, starts(n_q), starts(seg), used, causal, None, g, dt)
    k[room], v[room] = math.nan, math.inf
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.packed_attention(*leaves, starts(n_q), starts(seg), used_k=used, causal=causal)
    R.check(out, ref["out"], ref["out_tol"], "out")
    for n, d in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, g)):
        R.check(d, ref[n], ref[n + "_tol"], n)
        if n != "dq":
            assert not d[room].any()


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (BF16, 40)])
@pytest.mark.parametrize("Hq,Hk", [(3, 3), (8, 2), (6, 2), (10, 1), (24, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_a_few_tokens_per_sequence(dt, D, Hq, Hk, causal):
    """Rows of several tokens in one tile, tiles that end inside a token, edges inside the last keys."""
    gen = torch.Generator().manual_seed(33)
    n_q, n_k = [3, 1, 2, 0, 3, 1, 2, 3, 2], [300, 0, 2, 5, 1, 1025, 64, 65, 63]
    q, k, v = qkv(gen, sum(n_q), sum(n_k), Hq, Hk, D, dt)
    run_attention(q, k, v, starts(n_q), starts(n_k), None, causal, gen=gen)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("at", [0, 1, 2])
def test_later_tokens_do_not_reach_earlier_ones_of_a_step(dt, D, at):
    gen = torch.Generator().manual_seed(35)
    q, k, v = qkv(gen, 6, 205, 4, 2, D, dt)
    cu, cu_k = starts([3, 3]), starts([102, 103])
    clean = ops.packed_attention(q, k, v, cu, cu_k)
    k, v = k.clone(), v.clone()
    for end in (102, 205):
        v[end - 3 + at:end, 0, 3] = math.inf
        v[end - 3 + at, 1, 5] = math.nan
    out = ops.packed_attention(q, k, v, cu, cu_k)
    for b in range(2):
        assert torch.equal(out[3 * b:3 * b + at], clean[3 * b:3 * b + at])
        seen = out[3 * b + at:3 * b + 3]
        assert not bool(seen[:, :2, 3].isfinite().any()) and bool(seen[:, 2:, 5].isnan().all())
        assert bool(seen[:, :, 6].isfinite().all())


def test_one_token_on_a_very_long_history():
    gen = torch.Generator().manual_seed(4)
    q, k, v = qkv(gen, 1, 70001, 4, 1, 128, BF16)
    run_attention(q, k, v, starts([1]), starts([70001]), None, True, grads=False, gen=gen)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_many_sequences(dt):
    gen = torch.Generator().manual_seed(5)
    n = [(i * 7) % 23 for i in range(700)]
    q, k, v = qkv(gen, sum(n), sum(n), 2, 2, 64, dt)
    run_attention(q, k, v, starts(n), starts(n), None, True, gen=gen)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_rows_of_no_sequence(dt):
    """Rows before the first and behind the last sequence, and unused rows of key segments: zero, and NaN in them
    reaches nothing."""
    gen = torch.Generator().manual_seed(6)
    n_q, n_k, first = [20, 140], [60, 200], 9
    T, S = first + sum(n_q) + 300, first + sum(n_k) + 7
    q, k, v = qkv(gen, T, S, 4, 2, 64, dt)
    cu_q, cu_k = starts(n_q, first), starts(n_k, first)
    used = torch.tensor([41, 150], dtype=torch.int32, device=DEV)
    g = rand(gen, *q.shape, dt=dt)
    ref = R.attention(q, k, v, cu_q, cu_k, used, True, None, g, dt)
    hidden_q = torch.ones(T, dtype=torch.bool, device=DEV)
    hidden_q[first:first + sum(n_q)] = False
    hidden_k = torch.ones(S, dtype=torch.bool, device=DEV)
    hidden_k[first:first + 41] = False
    hidden_k[first + 60:first + 210] = False
    q[hidden_q], g[hidden_q] = math.nan, math.inf
    k[hidden_k], v[hidden_k] = math.inf, math.nan
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out, lse = ops.packed_attention(*leaves, cu_q, cu_k, used_k=used, return_lse=True)
    R.check(out, ref["out"], ref["out_tol"], "out")
    R.check(lse, ref["lse"], ref["lse_tol"], "lse")
    for n, d in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, g)):
        R.check(d, ref[n], ref[n + "_tol"], n)
    assert bool((out[hidden_q] == 0).all())


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("at", [0, 100, 127, 128, 200, 299])
def test_later_tokens_do_not_reach_earlier_ones(dt, D, at):
    """Causal: NaN and infinities from token `at` on leave the outputs before it as they were, and reach those
    after it."""
    gen = torch.Generator().manual_seed(7)
    q, k, v = qkv(gen, 300, 300, 2, 1, D, dt)
    cu = starts([300])
    clean = ops.packed_attention(q, k, v, cu)
    v2, k2 = v.clone(), k.clone()
    v2[at:, 0, 3] = math.inf
    v2[at, 0, 5] = math.nan
    out = ops.packed_attention(q, k, v2, cu)
    assert torch.equal(out[:at], clean[:at])
    assert bool(out[at:, :, 5].isnan().all()) and not bool(out[at:, :, 3].isfinite().any())
    assert bool(out[at:, :, 4].isfinite().all())
    k2[at:] = math.nan
    out = ops.packed_attention(q, k2, v2, cu)
    assert torch.equal(out[:at], clean[:at])
    assert bool(out[at:].isnan().all())


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_single_token_ignores_nan_behind_its_history(dt):
    gen = torch.Generator().manual_seed(8)
    q, k, v = qkv(gen, 2, 400, 8, 2, 64, dt)
    cu_q, cu_k = starts([1, 1]), starts([200, 200])
    used = torch.tensor([77, 130], dtype=torch.int32, device=DEV)
    clean = ops.packed_attention(q, k, v, cu_q, cu_k, used_k=used)
    for t in (k, v):
        t[77:200], t[330:] = math.nan, math.inf
    assert torch.equal(ops.packed_attention(q, k, v, cu_q, cu_k, used_k=used), clean)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_scores_of_any_size(dt):
    """Scores up to thousands: one key takes nearly all weight, the row maximum grows along the keys."""
    gen = torch.Generator().manual_seed(9)
    q, k, v = qkv(gen, 260, 260, 2, 2, 64, dt, scale=4.0)
    ramp = torch.linspace(0.1, 6, 260, device=DEV)[:, None, None]
    run_attention(q, (k * ramp).to(dt), v, starts([260]), starts([260]), None, True, scale=1.0, gen=gen)
    run_attention(q, (k * ramp.flip(0)).to(dt), v, starts([260]), starts([260]), None, False, scale=1.0, gen=gen)
    run_attention(q, k, v, starts([260]), starts([260]), None, False, scale=1e-6, gen=gen)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_attention_of_views(dt):
    """Queries, keys and values as views of one projection output; a shared (expanded) key head; odd alignment."""
    gen = torch.Generator().manual_seed(10)
    x = rand(gen, 150, 8, 64, dt=dt)
    cu = starts([70, 80])
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    same = ops.packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu)
    assert torch.equal(ops.packed_attention(q, k, v, cu), same)
    wide = torch.zeros(150, 8, 67, dtype=dt, device=DEV)
    wide[..., 3:] = x
    q, k, v = wide[:, :4, 3:], wide[:, 4:6, 3:], wide[:, 6:, 3:]
    assert torch.equal(ops.packed_attention(q, k, v, cu), same)
    t = x.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    assert torch.equal(ops.packed_attention(t[:, :4], t[:, 4:6], t[:, 6:], cu), same)
    last = x.permute(2, 0, 1).contiguous().permute(1, 2, 0)  # channels outermost
    assert torch.equal(ops.packed_attention(last[:, :4], last[:, 4:6], last[:, 6:], cu), same)
    # one key head shared by expanding it: the gradient of the original sums over the copies
    one = rand(gen, 150, 1, 64, dt=dt).requires_grad_(True)
    g = rand(gen, 150, 4, 64, dt=dt)
    y = ops.packed_attention(x[:, :4], one.expand(-1, 4, -1), one.expand(-1, 4, -1), cu)
    z = ops.packed_attention(x[:, :4], one, one, cu)
    assert torch.equal(y, z)
    (a,), (b,) = torch.autograd.grad(y, one, g), torch.autograd.grad(z, one, g)
    ref = R.attention(x[:, :4], one, one, cu, cu, None, True, None, g, dt)
    tol = ref["dk_tol"] + ref["dv_tol"] + 2 * R.u_of(dt) * (ref["dk"] + ref["dv"]).abs()
    R.check(b, ref["dk"] + ref["dv"], tol, "shared head")
    # the copies' gradients are rounded one by one: up to u times each copy's size, taken as 4 times the bound
    R.check(a, ref["dk"] + ref["dv"], 4 * tol + 8 * R.u_of(dt) * (ref["dk"].abs().max() + ref["dv"].abs().max()), "expanded")


def test_gradients_of_broadcast_outputs():
    """An incoming gradient that is an expanded scalar (stride 0)."""
    gen = torch.Generator().manual_seed(11)
    q, k, v = qkv(gen, 90, 90, 2, 1, 64, BF16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    cu = starts([40, 50])
    a = torch.autograd.grad(ops.packed_attention(*leaves, cu).sum(), leaves)
    b = torch.autograd.grad(ops.packed_attention(*leaves, cu), leaves, torch.ones(90, 2, 64, device=DEV, dtype=BF16))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("lens", [(300, 150, 33), (3, 1, 4)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_gradients_that_cancel(dt, lens):
    """Two equal keys, the second's value the first's with its halves exchanged, and equal halves in dO: the two
    products dO . v are the same number, dS is zero, and what is left of dq and dk is the error of rowsum(dO O).
    Were O taken as rounded, that error would be u |dO . O|; with the rounding's rest it is u u |dO . O|, plus that
    of the two sums of D products in 32 bits (2^-23 an addition in the matrix unit)."""
    gen = torch.Generator().manual_seed(23)
    D, B = 64, len(lens)
    T, u = sum(lens), torch.finfo(dt).eps / 2
    q, g = rand(gen, T, 2, D, dt=dt), rand(gen, T, 2, D // 2, dt=dt).repeat(1, 1, 2)
    k, v = rand(gen, B, 1, D, dt=dt).repeat_interleave(2, 0), rand(gen, B, 1, D, dt=dt)
    v = torch.stack([v, v.roll(D // 2, -1)], 1).reshape(2 * B, 1, D)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = ops.packed_attention(*leaves, starts(list(lens)), starts([2] * B), causal=False)
    dq, dk, _ = torch.autograd.grad(out, leaves, g)
    seq = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(lens, device=DEV))
    size = (g.abs() * v.view(B, 2, 1, D).abs().mean(1)[seq]).double().sum(-1)  # [T, 2], at least |dO| . |O|
    err = D ** -0.5 * size * (u * u + 2 * D * 2.0 ** -23)  # of dS, for the two keys together
    qmax, kmax = q.double().abs(), k.view(B, 2, 1, D)[seq, 0].double().abs()
    assert (dq.double().abs() <= err[..., None] * kmax * (1 + 4 * u)).all()
    most = torch.zeros(B, 1, D, dtype=torch.float64, device=DEV).index_add_(0, seq, (err[..., None] * qmax).sum(1, True))
    assert (dk.double().abs() <= (most * (1 + 4 * u)).repeat_interleave(2, 0)).all()


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
def test_results_do_not_change_between_runs(dt, D):
    gen = torch.Generator().manual_seed(12)
    q, k, v = qkv(gen, 1500, 1500, 8, 2, D, dt)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    cu, g = starts([1000, 500]), rand(gen, 1500, 8, D, dt=dt)

    def step():
        o = ops.packed_attention(*leaves, cu)
        return (o.detach(),) + torch.autograd.grad(o, leaves, g)

    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))


def test_row_numbers_are_clamped():
    """Starts and counts outside the tensors are cut to them (no row outside is touched)."""
    gen = torch.Generator().manual_seed(13)
    q, k, v = qkv(gen, 50, 60, 2, 1, 64, BF16)
    t = lambda *n: torch.tensor(n, dtype=torch.int32, device=DEV)  # noqa: E731
    a = ops.packed_attention(q, k, v, t(-5, 20, 1000), t(-7, 30, 4000), used_k=t(-3, 99))
    b = ops.packed_attention(q, k, v, t(0, 20, 50), t(0, 30, 60), used_k=t(0, 30))
    assert torch.equal(a, b) and bool((a[:20] == 0).all())


def test_no_sequences_and_no_rows():
    q = torch.randn(5, 2, 64, device=DEV, dtype=BF16)
    k = torch.randn(5, 1, 64, device=DEV, dtype=BF16)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert bool((ops.packed_attention(q, k, k, none) == 0).all())
    assert ops.packed_attention(q[:0], k, k, none, none).shape == (0, 2, 64)
    two = torch.zeros(2, dtype=torch.int32, device=DEV)
    out, lse = ops.packed_attention(q, k[:0], k[:0], starts([5]), two, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    leaves = [t.requires_grad_(True) for t in (q, k[:0].clone(), k[:0].clone())]
    grads = torch.autograd.grad(ops.packed_attention(*leaves, starts([5]), two).sum(), leaves)
    assert bool((grads[0] == 0).all()) and grads[1].shape == (0, 1, 64)
    leaves = [t.requires_grad_(True) for t in (q[:0].detach().clone(), k, k.detach().clone())]
    grads = torch.autograd.grad(ops.packed_attention(*leaves, two, starts([5])).sum(), leaves)
    assert bool((grads[1] == 0).all()) and bool((grads[2] == 0).all())


# ------------------------------------------------------------- norm_rotate
def tables(gen, P, R2, dev=DEV):
    ang = torch.randn(P, R2, generator=gen, dtype=torch.float64) * 10
    return ang.cos().float().to(dev), ang.sin().float().to(dev)


def run_norm_rotate(gen, T, Hq, Hk, D, rot, dt, wdt, positions, interleaved, P=None, view=False, eps=1e-6):
    P = P or max(T, 1)
    cos, sin = tables(gen, P, rot // 2)
    if view:
        x = rand(gen, T, Hq + 2 * Hk, D, dt=dt, scale=2.0)
        q, k = x[:, :Hq], x[:, Hq:Hq + Hk]
    else:
        q, k = rand(gen, T, Hq, D, dt=dt, scale=2.0), rand(gen, T, Hk, D, dt=dt, scale=2.0)
    wq = wk = None
    if wdt is not None:
        wq, wk = (1 + rand(gen, D, scale=0.3)).to(wdt), (1 + rand(gen, D, scale=0.3)).to(wdt)
    gq, gk = rand(gen, T, Hq, D, dt=dt), rand(gen, T, Hk, D, dt=dt)
    leaves = [t.detach().requires_grad_(True) for t in (q, k) + ((wq, wk) if wq is not None else ())]
    out = ops.norm_rotate(*leaves[:2], *(leaves[2:] or (None, None)), cos, sin, positions, eps, interleaved)
    plain = ops.norm_rotate(q, k, wq, wk, cos, sin, positions, eps, interleaved)
    assert all(torch.equal(a, b) for a, b in zip(out, plain))
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        z, dx, dw = R.norm_rotate(x, w, cos, sin, positions, eps, interleaved, g)
        tz, tx, tw = R.norm_rotate_bounds(x, w, cos, sin, positions, eps, interleaved, dt, g)
        R.check(out[i], z, tz, ("q", "k")[i])
        R.check(grads[i], dx, tx, ("dq", "dk")[i])
        if w is not None:
            R.check(grads[2 + i], dw, tw + R.u_of(wdt) * dw.abs(), ("dwq", "dwk")[i])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt,wdt", [(BF16, BF16), (F16, F32), (F32, F32), (BF16, F32), (F32, None)])
@pytest.mark.parametrize("D,rot", [(64, 64), (128, 128), (128, 64), (80, 80), (96, 32), (256, 256), (36, 20), (7, 6),
                                   (64, 0), (1, 0)])
def test_norm_rotate_sizes(dt, wdt, D, rot, interleaved):
    gen = torch.Generator().manual_seed(D + rot)
    run_norm_rotate(gen, 19, 5, 2, D, rot, dt, wdt, None, interleaved)


@pytest.mark.parametrize("T,Hq,Hk", [(1, 1, 1), (1, 32, 8), (3, 6, 6), (1500, 9, 3)])
@pytest.mark.parametrize("pdt", [torch.int32, torch.int64])
def test_norm_rotate_positions_and_views(T, Hq, Hk, pdt):
    gen = torch.Generator().manual_seed(T)
    pos = torch.randint(-1, 50, (T,), generator=gen).to(pdt).to(DEV)
    run_norm_rotate(gen, T, Hq, Hk, 64, 64, BF16, BF16, pos, False, P=50, view=True)
    run_norm_rotate(gen, T, Hq, Hk, 64, 32, F32, F32, pos, True, P=50, view=True)


def test_norm_rotate_many_rows():
    """Enough rows for the four-heads-per-group form, heads that do not divide by four."""
    gen = torch.Generator().manual_seed(20)
    T = 9000
    q, k = rand(gen, T, 10, 64, dt=BF16), rand(gen, T, 5, 64, dt=BF16)
    cos, sin = tables(gen, 4096, 32)
    pos = (torch.arange(T, device=DEV) % 4096).int()
    w = (1 + rand(gen, 64, scale=0.2)).bfloat16()
    qo, ko = ops.norm_rotate(q, k, w, w, cos, sin, pos)
    gq, gk = rand(gen, T, 10, 64, dt=BF16), rand(gen, T, 5, 64, dt=BF16)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, w)]
    grads = torch.autograd.grad(ops.norm_rotate(leaves[0], leaves[1], leaves[2], leaves[2], cos, sin, pos), leaves, (gq, gk))
    pick = torch.tensor([0, 1, 4095, 4096, 8999], device=DEV)
    for x, o, g, d in ((q, qo, gq, grads[0]), (k, ko, gk, grads[1])):
        args = (x[pick], w, cos, sin, pos[pick], 1e-6, False)
        z, dx, _ = R.norm_rotate(*args, g=g[pick])
        tz, tx, _ = R.norm_rotate_bounds(*args, dtype=BF16, g=g[pick])
        R.check(o[pick], z, tz, "out")
        R.check(d[pick], dx, tx, "dx")


def test_norm_rotate_unrotated_out_of_table_and_infinite():
    gen = torch.Generator().manual_seed(21)
    q, k = rand(gen, 6, 2, 64), rand(gen, 6, 1, 64)
    cos, sin = tables(gen, 4, 16)  # channels 32.. are not rotated
    pos = torch.tensor([0, -1, 3, 4, 1 << 30, -(1 << 31)], dtype=torch.int32, device=DEV)
    qo, ko = ops.norm_rotate(q, k, None, None, cos, sin, pos)
    want = R.norm_rotate(q, None, cos, sin, pos.clamp(max=3), 1e-6, False)
    assert bool(qo[3:5, :, :32].isnan().all()) and bool(ko[3:5, :, :32].isnan().all())
    ok = [0, 1, 2, 5]
    assert torch.allclose(qo[ok].double(), want[ok], rtol=1e-5, atol=1e-6)
    assert torch.allclose(qo[3:5, :, 32:].double(), want[3:5, :, 32:], rtol=1e-5, atol=1e-6)
    z = torch.zeros(2, 1, 64, device=DEV)
    a, _ = ops.norm_rotate(z, z, None, None, cos, sin)
    assert bool((a == 0).all())
    q[1, 0, 3] = math.nan  # the other heads and tokens are as they were
    again, _ = ops.norm_rotate(q, k, None, None, cos, sin, pos)
    assert bool(again[1, 0].isnan().all()) and torch.equal(again[1, 1], qo[1, 1]) and torch.equal(again[0], qo[0])


def test_norm_rotate_partial_needs_and_empty():
    gen = torch.Generator().manual_seed(22)
    q, k = rand(gen, 5, 2, 64), rand(gen, 5, 1, 64)
    cos, sin = tables(gen, 5, 32)
    w = torch.ones(64, device=DEV, requires_grad=True)
    q.requires_grad_(True)
    a, _ = ops.norm_rotate(q, k, w, None, cos, sin)  # the key output is not used
    dq, dw = torch.autograd.grad(a.sum(), (q, w))
    assert dq.shape == q.shape and dw.shape == (64,)
    e = torch.empty(0, 2, 64, device=DEV, requires_grad=True)
    a, b = ops.norm_rotate(e, e[:, :1], w, None, cos, sin)
    dw, = torch.autograd.grad(a.sum() + b.sum(), w)
    assert a.shape == (0, 2, 64) and bool((dw == 0).all())


# ------------------------------------------------------------ the two together
def chain(x, w, cos, sin, pos, cu, Hq, Hk):
    q, k = ops.norm_rotate(x[:, :Hq], x[:, Hq:Hq + Hk], w[0], w[1], cos, sin, pos)
    return ops.packed_attention(q, k, x[:, Hq + Hk:], cu)


def chain_inputs(gen, lens, Hq, Hk, D, dt):
    T = sum(lens)
    x = rand(gen, T, Hq + 2 * Hk, D, dt=dt)
    cos, sin = tables(gen, max(lens), D // 2)
    pos = torch.cat([torch.arange(n) for n in lens]).int().to(DEV)
    w = (1 + rand(gen, 2, D, scale=0.2)).to(dt)
    return x, w, cos, sin, pos, starts(lens), Hq, Hk


@pytest.mark.parametrize("dt", [BF16, F32])
def test_norm_rotate_into_attention(dt):
    """Projection output -> norm + rotation -> attention, and the gradients back to the projection output."""
    gen = torch.Generator().manual_seed(30)
    args = chain_inputs(gen, [90, 1, 170], 4, 2, 64, dt)
    x, w, cos, sin, pos, cu, Hq, Hk = args
    x.requires_grad_(True)
    w.requires_grad_(True)
    g = rand(gen, x.shape[0], Hq, 64, dt=dt)
    out = chain(*args)
    dx, dw = torch.autograd.grad(out, (x, w), g)
    # 64 bits throughout
    q64 = R.norm_rotate(x[:, :Hq], w[0], cos, sin, pos, 1e-6, False)
    k64 = R.norm_rotate(x[:, Hq:Hq + Hk], w[1], cos, sin, pos, 1e-6, False)
    ref = R.attention(q64, k64, x[:, Hq + Hk:].double(), cu, cu, None, True, None, g)
    _, dq64, dwq = R.norm_rotate(x[:, :Hq], w[0], cos, sin, pos, 1e-6, False, ref["dq"])
    _, dk64, dwk = R.norm_rotate(x[:, Hq:Hq + Hk], w[1], cos, sin, pos, 1e-6, False, ref["dk"])
    # relative 2-norm: each of about eight roundings (q, k, weights, output, score gradients, dq, dk, the result)
    # moves values by at most u, and a score of size s by 2 u s with |s| up to about 6 here
    tol = (8 + 2 * 6) * R.u_of(dt) + 1e-5

    def near(a, b, what):
        off = ((a.double() - b).norm() / b.norm()).item()
        assert off <= tol, (what, off, tol)

    near(out, ref["out"], "out")
    near(dx[:, :Hq], dq64, "dq")
    near(dx[:, Hq:Hq + Hk], dk64, "dk")
    near(dx[:, Hq + Hk:], ref["dv"], "dv")
    near(dw[0], dwq, "dwq")
    near(dw[1], dwk, "dwk")


def test_chain_in_a_graph_and_on_a_stream():
    """A training step captured into a CUDA graph, replayed on new inputs, while an eager call runs on a second
    stream; and two graphs at once."""
    gen = torch.Generator().manual_seed(31)
    a = chain_inputs(gen, [300, 20, 513], 4, 2, 128, BF16)
    b = chain_inputs(gen, [300, 20, 513], 4, 2, 128, BF16)
    g = rand(gen, 833, 4, 128, dt=BF16)

    def step(args):
        x = args[0].detach().requires_grad_(True)
        out = chain(x, *args[1:])
        return out, torch.autograd.grad(out, x, g)[0]

    want_a, want_b = step(a), step(b)
    static = [t.clone() for t in a[:4]] + list(a[4:])  # projection output, weights, cos, sin
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(static))
        graphs.append(graph)
    for args, want in ((b, want_b), (a, want_a)):
        for mine, new in zip(static[:4], args):
            mine.copy_(new)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        eager = step(static)
        torch.cuda.synchronize()
        for got in (*outs, eager):
            for x, y in zip(got, want):
                assert torch.equal(x, y)


def test_single_token_step_in_a_graph():
    """A captured step replayed while the histories grow: the counts are read on the device."""
    gen = torch.Generator().manual_seed(32)
    q, k, v = qkv(gen, 3, 3 * 600, 8, 2, 128, BF16)
    cu_q, cu_k = starts([1] * 3), starts([600] * 3)
    used = torch.tensor([1, 300, 599], dtype=torch.int32, device=DEV)
    ops.packed_attention(q, k, v, cu_q, cu_k, used_k=used)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.packed_attention(q, k, v, cu_q, cu_k, used_k=used)
    for n in ([1, 300, 599], [2, 301, 600], [0, 64, 65]):
        used.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        ref = R.attention(q, k, v, cu_q, cu_k, used, True, None, None, BF16)
        R.check(out, ref["out"], ref["out_tol"], str(n))


def test_chain_compiles_without_graph_breaks():
    gen = torch.Generator().manual_seed(33)
    args = chain_inputs(gen, [130, 70], 4, 2, 64, BF16)
    g = rand(gen, 200, 4, 64, dt=BF16)

    def f(x):
        return chain(x * 1.0, *args[1:]) + 0.0

    def grad(fn):
        x = args[0].detach().requires_grad_(True)
        o = fn(x)
        return o.detach(), torch.autograd.grad(o, x, g)[0]

    want = grad(f)
    got = grad(torch.compile(f, fullgraph=True))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_beyond_32_bit_offsets():
    """A key row whose element offset is above 2^31."""
    S, Hk, D = 2_200_000, 8, 128
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of free device memory")
    k = torch.zeros(S, Hk, D, dtype=BF16, device=DEV)
    gen = torch.Generator().manual_seed(34)
    tail = rand(gen, 200, Hk, D, dt=BF16)
    k[-200:] = tail
    q = rand(gen, 3, 8, D, dt=BF16)
    cu_k = torch.tensor([S - 200, S - 100, S - 100, S], dtype=torch.int32, device=DEV)
    got = ops.packed_attention(q, k, k, starts([1, 0, 2]), cu_k)
    small = ops.packed_attention(q, tail, tail, starts([1, 0, 2]), starts([100, 0, 100]))
    ref = R.attention(q, tail, tail, starts([1, 0, 2]), starts([100, 0, 100]), None, True, None, None, BF16)
    R.check(small, ref["out"], ref["out_tol"], "small")
    R.check(got, ref["out"], ref["out_tol"], "large")


@pytest.mark.parametrize("dt", [BF16, F32])
def test_one_tensor_in_three_places(dt):
    """q, k and v are the same leaf: its gradient is the sum of the three."""
    gen = torch.Generator().manual_seed(41)
    x, g = rand(gen, 150, 2, 64, dt=dt, scale=1.2), rand(gen, 150, 2, 64, dt=dt)
    cu = starts([70, 80])
    three = [x.clone().requires_grad_() for _ in range(3)]
    apart = torch.autograd.grad(ops.packed_attention(*three, cu), three, g)
    x.requires_grad_()
    (together,) = torch.autograd.grad(ops.packed_attention(x, x, x, cu), x, g)
    # two additions in the storage type, each off by half a step
    size = sum(d.double().abs() for d in apart)
    err = (together.double() - sum(d.double() for d in apart)).abs()
    assert (err <= 2.1 * torch.finfo(dt).eps / 2 * size).all()


def test_calls_from_several_threads_and_streams():
    """Steps, prompts and gradients at once, each thread on its stream: the results of the calls one by one."""
    import threading
    gen = torch.Generator().manual_seed(43)
    jobs = []
    for i, (lens, D, dt) in enumerate([([600, 77], 128, BF16), ([1] * 5, 64, F16), ([333], 64, F16), ([90, 200], 64, F32)]):
        q, k, v = qkv(gen, sum(lens), sum(lens), 4, 2, D, dt)
        jobs.append((q, k, v, starts(lens), rand(gen, *q.shape, dt=dt)))

    def run(q, k, v, cu, g):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.packed_attention(*leaves, cu)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]
    alone = [run(*j) for j in jobs]
    torch.cuda.synchronize()
    wrong, streams = [], [torch.cuda.Stream() for _ in jobs]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                if not all(torch.equal(a, b) for a, b in zip(run(*jobs[i]), alone[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_two_graphs_at_once():
    """Two captured steps and a captured prompt replayed together share no workspace."""
    gen = torch.Generator().manual_seed(45)
    runs = []
    for n_q, n_k in (([1, 1, 1], [900, 1, 400]), ([2, 1, 1], [700, 50, 1300]), ([300, 20], [300, 20])):
        q, k, v = qkv(gen, sum(n_q), sum(n_k), 8, 2, 64, BF16)
        cu_q, cu_k = starts(n_q), starts(n_k)
        exp = ops.packed_attention(q, k, v, cu_q, cu_k)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.packed_attention(q, k, v, cu_q, cu_k)
        runs.append((graph, torch.cuda.Stream(), out, exp, (q, k, v, cu_q, cu_k)))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, exp, _ in runs:
        assert torch.equal(out, exp)


def test_a_second_derivative_is_refused():
    q = torch.randn(20, 2, 64, device=DEV, requires_grad=True)
    out = ops.packed_attention(q, q, q, starts([20]))
    (d,) = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice"):
        d.sum().backward()
