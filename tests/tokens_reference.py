"""64-bit restatements of the token-sequence operators for the tests, and
bounds on how far a result of `dtype` may be from them.

The bounds count roundings.  u = finfo(dtype).eps / 2 is the largest relative
error of one rounding to the storage type; a result is rounded once, and in
16 bits so are the softmax weights and score gradients that the tensor cores
multiply.  What is computed in fp32 is off by at most a few steps of 2^-24
per operation of a sum; the tensor cores may drop the bits that a rounding
would keep, so twice that is counted.  Among the subnormals of a type the spacing
is finfo.tiny * eps whatever the value, so a rounding there is off by up to
s = finfo.tiny * u absolutely instead of u relatively: fp16, whose tiny is
2^-14, needs that (2^-25) for small results and small operands.
"""
import math

import torch

F32 = 2.0 ** -24


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------- norm_rotate
def pair_index(R, interleaved):
    i = torch.arange(R // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)


def rotation_matrices(cos, sin, positions, T, D, interleaved):
    """[T, D, D]: z = M y."""
    R = 2 * cos.shape[1]
    a, b = (i.to(cos.device) for i in pair_index(R, interleaved))
    M = torch.eye(D, dtype=torch.float64, device=cos.device).repeat(T, 1, 1)
    for t in range(T):
        p = t if positions is None else int(positions[t])
        if p < 0 or R == 0:
            continue
        c, s = cos[p].double(), sin[p].double()
        M[t, a, a], M[t, b, b], M[t, a, b], M[t, b, a] = c, c, -s, s
    return M


def norm_rotate(x, w, cos, sin, positions, eps, interleaved, g=None):
    """z, and with g (gradient of z) also (dx, dw)."""
    x = x.detach().double()
    T, H, D = x.shape
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    r = 1.0 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    M = rotation_matrices(cos, sin, positions, T, D, interleaved)
    z = torch.einsum("tij,thj->thi", M, x * r * w)
    if g is None:
        return z
    gy = torch.einsum("tji,thj->thi", M, g.double())
    h = x * r
    dx = r * (gy * w - h * (gy * w * h).mean(-1, keepdim=True))
    return z, dx, (gy * h).sum((0, 1))


def norm_rotate_bounds(x, w, cos, sin, positions, eps, interleaved, dtype, g):
    """How far z, dx, dw may be off: one rounding to the type, and fp32 sums of up to D (dw: rows) terms whose
    relative error is at most (terms + 8) F32 of the sum of absolute values."""
    x = x.detach().double()
    T, H, D = x.shape
    u, f = u_of(dtype), 2 * (D + 16) * F32
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    r = 1.0 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    M = rotation_matrices(cos, sin, positions, T, D, interleaved).abs()
    za = torch.einsum("tij,thj->thi", M, (x * r * w).abs())
    z, dx, dw = norm_rotate(x, w, cos, sin, positions, eps, interleaved, g)
    ga = torch.einsum("tji,thj->thi", M, g.double().abs())
    h = (x * r).abs()
    dxa = r * (ga * w.abs() + h * (ga * w.abs() * h).mean(-1, keepdim=True))
    dwa = (ga * h).sum((0, 1))
    tiny = torch.finfo(dtype).tiny * u + 1e-30  # a rounding among the subnormals
    # dw is fp32 in the kernel and rounded to the weight's type by its user
    return u * z.abs() + f * za + tiny, u * dx.abs() + f * dxa + tiny, (f + 2 * T * H * F32) * dwa + 1e-30


# -------------------------------------------------------- packed_attention
def attention(q, k, v, cu_q, cu_k, used_k=None, causal=True, scale=None, g=None, dtype=None):
    """dict with out, lse and, with g, dq, dk, dv; with dtype also a bound `*_tol` for each."""
    T, Hq, D = q.shape
    S, Hk, _ = k.shape
    scale = D ** -0.5 if scale is None else scale
    dev = q.device
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=dev)  # noqa: E731
    r = {"out": z(T, Hq, D), "lse": torch.full((Hq, T), -math.inf, dtype=torch.float64, device=dev),
         "out_tol": z(T, Hq, D), "lse_tol": z(Hq, T)}
    if g is not None:
        g = g.double()
        for n, like in (("dq", q), ("dk", k), ("dv", v)):
            r[n], r[n + "_tol"] = torch.zeros_like(like), torch.zeros_like(like)
    u = u_of(dtype) if dtype is not None else 0.0
    sub = torch.finfo(dtype).tiny * u if dtype is not None else 0.0
    half = dtype in (torch.float16, torch.bfloat16)
    u16, sub16 = (u, sub) if half else (0.0, 0.0)  # rounding of tensor-core operands
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for b in range(len(cq) - 1):
        nq, nk = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        if used_k is not None:
            nk = min(nk, int(used_k[b]))
        if nq == 0 or nk <= 0:
            continue
        i = torch.arange(nq, device=dev)[:, None]
        j = torch.arange(nk, device=dev)[None, :]
        seen = (j <= i + nk - nq) if causal else torch.ones(nq, nk, dtype=torch.bool, device=dev)
        some = seen.any(1)
        for h in range(Hq):
            hk = h // (Hq // Hk)
            qs, ks, vs = q[cq[b]:cq[b] + nq, h], k[ck[b]:ck[b] + nk, hk], v[ck[b]:ck[b] + nk, hk]
            s = (qs @ ks.T * scale).masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(s, 1)
            p = torch.where(seen, torch.exp(s - torch.where(some, lse, 0.0)[:, None]), 0.0)
            rows = slice(cq[b], cq[b] + nq)
            cols = slice(ck[b], ck[b] + nk)
            o = p @ vs
            r["out"][rows, h], r["lse"][h, rows] = o, lse
            # relative error of a weight: twice that of a score (fp32 sum of D products; the score and the
            # row's sum), of an exponential (2^-20) and of the fp32 sum over the keys
            c = 2 * (scale * (D + 4) * 2 * F32 * (qs.abs() @ ks.abs().T).max().item() + 2.0 ** -20) + 2 * nk * F32
            oa = p @ vs.abs()
            seen_d = seen.double()
            o_err = (u16 + c) * oa + sub16 * (seen_d @ vs.abs())
            r["out_tol"][rows, h] = u * o.abs() + o_err + sub + 1e-30
            r["lse_tol"][h, rows] = torch.where(some, c + 4 * F32 * lse.abs(), 0.0)
            if g is None:
                continue
            go = g[rows, h]
            dp = go @ vs.T
            delta = (go * o).sum(1, keepdim=True)
            ds = p * (dp - delta) * scale
            r["dq"][rows, h] = ds @ ks
            r["dk"][cols, hk] += ds.T @ qs
            r["dv"][cols, hk] += p.T @ go
            # delta comes from the rounded output; dp and delta are fp32 sums of D products
            d_delta = (go.abs() * (u * o.abs() + o_err + sub)).sum(1, keepdim=True)
            f = (D + 8) * 2 * F32
            ga = go.abs() @ vs.abs().T
            e = p * scale * (d_delta + f * (ga + (go * o).abs().sum(1, keepdim=True))) + (u16 + 2 * c) * ds.abs()
            e = e + sub16 * max(1.0, scale) * seen_d
            n = 2 * F32
            r["dq_tol"][rows, h] = sub + u * r["dq"][rows, h].abs() + (e + n * nk * ds.abs()) @ ks.abs() + 1e-30
            r["dk_tol"][cols, hk] += (e + n * nq * ds.abs()).T @ qs.abs()
            r["dv_tol"][cols, hk] += ((u16 + c + n * nq) * p + sub16 * seen_d).T @ go.abs()
    if g is not None:
        for m in ("dk", "dv"):  # the heads of a group: one rounding of their sum
            r[m + "_tol"] += (u + 2 * F32 * Hq) * r[m].abs() + sub + 1e-30
    return r


def check(got, ref, tol, what):
    """Elementwise |got - ref| <= tol (both -inf counts as equal)."""
    got, ref = got.detach().double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    same = (got == ref)
    bad = ~same & ~((got - ref).abs() <= tol)
    if bad.any():
        at = tuple(int(x) for x in bad.nonzero()[0])
        worst = ((got - ref).abs() / tol)[~same].max().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values are off, first at {at}: "
                             f"{got[at].item()} for {ref[at].item()} (may be off by {tol[at].item():.3g}); "
                             f"worst {worst:.3g} of its bound")
