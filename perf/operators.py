"""Cases of the token-sequence operators: `norm_rotate` (RMS norm of query and key heads with the position
rotation) and `packed_attention` (attention over packed sequences, grouped heads, causal or not), forward,
training step and the single-token form.

`run` computes them in plain torch where `own` is false, and through uplift_b200.ops where it is true;
`exact` computes them in 64 bits from the definitions.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of 16 requests: the norm and rotation between the projection and the attention
        {"name": "norm_rotate step", "op": "norm_rotate", "dtype": "bf16", "tokens": 16, "heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 128, "table": 32768, "interleaved": False, "unrotated": 0, "train": False},
        # a packed prompt batch
        {"name": "norm_rotate prompt", "op": "norm_rotate", "dtype": "bf16", "tokens": 12347, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "table": 16384, "interleaved": False, "unrotated": 0, "train": False},
        # image tokens in fp32: 8 images of 1022 px with 14 px patches (73 x 73) and a class token, 6 heads of 64
        {"name": "norm_rotate images", "op": "norm_rotate", "dtype": "fp32", "tokens": 42640, "heads": 6,
         "kv_heads": 6, "dim": 64, "rot": 64, "table": 5329, "interleaved": True, "unrotated": 8, "train": False},
        # a training step of the norm and rotation: outputs and all gradients
        {"name": "norm_rotate train", "op": "norm_rotate", "dtype": "bf16", "tokens": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "table": 8192, "interleaved": False, "unrotated": 0, "train": True},
        # one short prompt: latency
        {"name": "attention short prompt", "op": "attention", "dtype": "fp16", "batch": 1, "longest": 333,
         "shortest": 333, "context": 0, "heads": 8, "kv_heads": 8, "dim": 64, "causal": True, "lens_seed": 1,
         "train": False},
        # a serving batch of prompts of very different lengths
        {"name": "attention ragged prompts", "op": "attention", "dtype": "bf16", "batch": 16, "longest": 2011,
         "shortest": 17, "context": 0, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "lens_seed": 2,
         "train": False},
        # one long prompt
        {"name": "attention long prompt", "op": "attention", "dtype": "bf16", "batch": 1, "longest": 16384,
         "shortest": 16384, "context": 0, "heads": 16, "kv_heads": 4, "dim": 128, "causal": True, "lens_seed": 3,
         "train": False},
        # backbone attention over 8 images of 1022 px (73 x 73 patches and a class token), 6 heads of 64
        {"name": "attention images", "op": "attention", "dtype": "bf16", "batch": 8, "longest": 5330,
         "shortest": 5330, "context": 0, "heads": 6, "kv_heads": 6, "dim": 64, "causal": False, "lens_seed": 4,
         "train": False},
        # a decoding step of 4 requests: latency
        {"name": "attention step of 4", "op": "attention", "dtype": "bf16", "batch": 4, "longest": 1,
         "shortest": 1, "context": 1500, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "lens_seed": 5,
         "train": False},
        # a decoding step of 64 requests with long and short histories in segments with room to grow
        {"name": "attention step of 64", "op": "attention", "dtype": "bf16", "batch": 64, "longest": 1,
         "shortest": 1, "context": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "lens_seed": 6,
         "train": False},
        # a training step over packed documents: output and gradients
        {"name": "attention train documents", "op": "attention", "dtype": "bf16", "batch": 6, "longest": 2500,
         "shortest": 300, "context": 0, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "lens_seed": 7,
         "train": True},
        # a training step over 16 images of 448 px (32 x 32 patches and a class token), 6 heads of 64
        {"name": "attention train images", "op": "attention", "dtype": "fp16", "batch": 16, "longest": 1025,
         "shortest": 1025, "context": 0, "heads": 6, "kv_heads": 6, "dim": 64, "causal": False, "lens_seed": 8,
         "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm_rotate", "norm_rotate", "prompt", "prompt", "step", "train", "train"))
    kv = rng.choice((1, 2, 4, 6, 8))
    if kind == "norm_rotate":
        train = rng.random() < 0.4
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        dim = rng.choice((64, 80, 96, 128))
        heads = kv * rng.choice((1, 2, 4))
        most = min(40000, int((4e7 if train else 6e7) / ((heads + kv) * dim)))
        tokens = _log(rng, 1, most)
        return {"op": "norm_rotate", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv, "dim": dim,
                "rot": rng.choice((dim, dim, dim // 2)), "table": _log(rng, 64, 32768),
                "interleaved": rng.random() < 0.3, "unrotated": rng.choice((0, 0, 1)), "train": train}
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    dim = rng.choice((64, 64, 80, 96, 128, 128))
    group = rng.choice((1, 2, 4, 4, 8))
    lens_seed = rng.randrange(1 << 20)
    if kind == "step":  # single tokens, now and then a few
        context = _log(rng, 1, 12000)
        batch = _log(rng, 1, max(1, min(96, int(3e8 / (context * kv * dim)))))
        return {"op": "attention", "dtype": dtype, "batch": batch, "longest": rng.choice((1, 1, 1, 3)), "shortest": 1,
                "context": context, "heads": kv * group, "kv_heads": kv, "dim": dim, "causal": True,
                "lens_seed": lens_seed, "train": False}
    train = kind == "train"
    heads = kv * min(group, 32 // kv)
    longest = _log(rng, 2, 3000) if train else _log(rng, 1, 6000)
    batch = _log(rng, 1, max(1, min(48, int((1.0e9 if train else 2.0e9) / (heads * longest * longest)))))
    return {"op": "attention", "dtype": dtype, "batch": batch, "longest": longest,
            "shortest": rng.randint(1, longest), "context": 0 if train else rng.choice((0, 0, 0, 700)),
            "heads": heads, "kv_heads": kv, "dim": dim, "causal": rng.random() < 0.7, "lens_seed": lens_seed,
            "train": train}


def lengths(case):
    """(queries, keys, key segments) of each sequence: the segments of a history hold up to an eighth more
    rows than are used, as a cache with room for the next tokens does."""
    rng = random.Random(case["lens_seed"])
    n_q = [case["longest"]] + [_log(rng, case["shortest"], case["longest"]) for _ in range(case["batch"] - 1)]
    if not case["context"]:
        return n_q, list(n_q), None
    hist = [case["context"]] + [_log(rng, max(1, case["context"] // 16), case["context"])
                                for _ in range(case["batch"] - 1)]
    n_k = [a + b for a, b in zip(n_q, hist)]
    return n_q, n_k, [n + n // 8 + 1 for n in n_k]


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "norm_rotate":
        t = case["tokens"]
        data = t * (hq + hk) * d
        side = min(t, case["table"]) * case["rot"] * 4 + 4 * t + 2 * d * es
        if not case["train"]:
            return {"bytes": 2 * data * es + side, "flops": 10 * data}
        # forward: read x, write z; backward: read x and dz, write dx
        return {"bytes": 5 * data * es + 2 * side, "flops": 30 * data}
    n_q, n_k, _ = lengths(case)
    pairs = 0
    for a, b in zip(n_q, n_k):
        if not case["causal"]:
            pairs += a * b
        else:  # row i sees i + 1 + b - a keys (none where that is not positive)
            first = max(1, 1 + b - a)
            last = b
            pairs += (first + last) * (last - first + 1) // 2 if last >= first else 0
    q, kv = sum(n_q) * hq * d * es, sum(n_k) * hk * d * es
    if not case["train"]:
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * d * hq * pairs}
    # forward reads q, k, v, writes o; backward reads q, k, v, o, do, writes dq, dk, dv
    return {"bytes": 6 * q + 6 * kv, "flops": 14 * d * hq * pairs}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dt)

    s = {"case": case}
    if case["op"] == "norm_rotate":
        t = case["tokens"]
        qkv = rand(t, hq + 2 * hk, d, scale=1.7)  # the projection's output: queries, keys and values of a token
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hk]
        s["wq"] = (1 + 0.2 * torch.randn(d, generator=gen, device=dev)).to(dt)
        s["wk"] = (1 + 0.2 * torch.randn(d, generator=gen, device=dev)).to(dt)
        freq = 10000.0 ** (-torch.arange(case["rot"] // 2, device=dev, dtype=torch.float64) / (case["rot"] // 2))
        ang = torch.arange(case["table"], device=dev, dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        start = torch.randint(0, case["table"], (1,), generator=gen, device=dev)
        pos = (torch.arange(t, device=dev) + start) % case["table"]
        if case["unrotated"]:  # class tokens
            pos[:: max(1, t // case["unrotated"])] = -1
        s["positions"] = pos.to(torch.int32)
        if case["train"]:
            s["gq"], s["gk"] = rand(t, hq, d), rand(t, hk, d)
            for n in ("q", "k", "wq", "wk"):
                s[n].requires_grad_(True)
        return s
    n_q, n_k, seg = lengths(case)
    rows_k = sum(seg or n_k)
    s["q"], s["k"], s["v"] = rand(sum(n_q), hq, d, scale=1.2), rand(rows_k, hk, d, scale=1.2), rand(rows_k, hk, d)

    def starts(n):
        return torch.tensor([0] + n, dtype=torch.int64).cumsum(0).to(torch.int32).to(dev)

    s["cu_q"] = starts(n_q)
    s["cu_k"] = starts(seg or n_k) if seg else s["cu_q"]
    s["used_k"] = torch.tensor(n_k, dtype=torch.int32, device=dev) if seg else None
    s["max_q"], s["max_k"] = max(n_q), max(n_k)
    if case["train"]:
        s["g"] = rand(sum(n_q), hq, d)
        for n in ("q", "k", "v"):
            s[n].requires_grad_(True)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if case["op"] == "norm_rotate":
        if own:
            return _own_norm_rotate(s)
        with torch.no_grad():
            return _plain_norm_rotate(s)
    if own:
        return _own_attention(s)
    with torch.no_grad():
        return _plain_attention(s)


def _own_norm_rotate(s):
    from uplift_b200 import ops
    q, k = ops.norm_rotate(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], positions=s["positions"], eps=EPS,
                           interleaved=s["case"]["interleaved"])
    if not s["case"]["train"]:
        return q, k
    grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
    return (q.detach(), k.detach()) + grads


def _own_attention(s):
    from uplift_b200 import ops
    o = ops.packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], used_k=s["used_k"],
                             causal=s["case"]["causal"])
    if not s["case"]["train"]:
        return o
    return (o.detach(),) + torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["g"])


# ------------------------------------------------------------------ plain forms (32 bits)
def _split_pairs(x, rot, interleaved):
    return (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2:rot])


def _join_pairs(a, b, rest, interleaved):
    pair = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((pair, rest), -1)


def _plain_norm_rotate(s):
    case = s["case"]
    rot, inter = case["rot"], case["interleaved"]
    pos = s["positions"].long()
    there = (pos >= 0)[:, None, None]
    c = torch.where(there, s["cos"][pos.clamp(min=0)][:, None], 1.0)
    n = torch.where(there, s["sin"][pos.clamp(min=0)][:, None], 0.0)

    def forward(x, w):
        x = x.float()
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = _split_pairs(y, rot, inter)
        return _join_pairs(a * c - b * n, b * c + a * n, y[..., rot:], inter)

    def backward(x, w, g):
        x, g = x.float(), g.float()
        r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        a, b = _split_pairs(g, rot, inter)
        g = _join_pairs(a * c + b * n, b * c - a * n, g[..., rot:], inter)
        h = x * r
        gw = g * w.float()
        dx = r * (gw - h * (gw * h).mean(-1, keepdim=True))
        # the sum over all rows in 64 bits: it is long
        return dx, (g * h).sum((0, 1), dtype=torch.float64)

    out = [forward(s["q"], s["wq"]).to(s["q"].dtype), forward(s["k"], s["wk"]).to(s["k"].dtype)]
    if not case["train"]:
        return tuple(out)
    dq, dwq = backward(s["q"], s["wq"], s["gq"])
    dk, dwk = backward(s["k"], s["wk"], s["gk"])
    return tuple(out) + (dq.to(s["q"].dtype), dk.to(s["k"].dtype), dwq.to(s["wq"].dtype), dwk.to(s["wk"].dtype))


def _plain_attention(s):
    """Padded to the longest sequence: scores of every query with every key of its sequence in one product."""
    case = s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    g, lq, lk = hq // hk, s["max_q"], s["max_k"]
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    n_q = cu_q[1:] - cu_q[:-1]
    n_k = s["used_k"].long() if s["used_k"] is not None else cu_k[1:] - cu_k[:-1]
    iq, ik = torch.arange(lq, device=q.device), torch.arange(lk, device=q.device)
    there_q, there_k = iq < n_q[:, None], ik < n_k[:, None]
    at_q = torch.where(there_q, cu_q[:-1, None] + iq, 0)
    at_k = torch.where(there_k, cu_k[:-1, None] + ik, 0)
    batch = at_q.shape[0]

    def rows(x):  # [B, kv heads, group * queries, D]
        return x[at_q].float().view(batch, lq, hk, g, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, g * lq, d)

    def cols(x):  # [B, kv heads, keys, D]
        return x[at_k].float().transpose(1, 2)

    seen = there_k[:, None, :].expand(batch, lq, lk)
    if case["causal"]:
        seen = seen & (ik <= iq[:, None] + (n_k - n_q)[:, None, None])
    hidden = ~seen[:, None].repeat(1, 1, g, 1)  # [B, 1, group * queries, keys]
    scale = 1.0 / math.sqrt(d)
    qf, kf, vf = rows(q), cols(k), cols(v)
    p = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale).masked_fill_(hidden, -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total > 0, total, 1.0))
    o = torch.matmul(p, vf)

    def packed(x, at, there, n, heads):  # [B, L, heads, D] -> [rows, heads, D], padding into a row that is dropped
        out = torch.zeros(n + 1, heads, d, device=q.device, dtype=torch.float32)
        out[torch.where(there, at, n).flatten()] = x.reshape(-1, heads, d)
        return out[:n]

    def unrows(x):
        return packed(x.view(batch, hk, g, lq, d).permute(0, 3, 1, 2, 4), at_q, there_q, q.shape[0], hq)

    def uncols(x):
        return packed(x.transpose(1, 2), at_k, there_k, k.shape[0], hk)

    out = unrows(o).to(q.dtype)
    if not case["train"]:
        return out
    do = rows(s["g"]) * there_q[:, None, None, :, None].expand(batch, 1, g, lq, 1).reshape(batch, 1, g * lq, 1)
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, vf.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, kf), torch.matmul(ds.transpose(-1, -2), qf)
    return out, unrows(dq).to(q.dtype), uncols(dk).to(k.dtype), uncols(dv).to(v.dtype)


# ------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm_rotate":
            return _exact_norm_rotate(case, s)
        return _exact_attention(case, s)


def _exact_norm_rotate(case, s):
    """Pairs as complex numbers: the rotation is a product with cos + i sin, its transpose one with the conjugate."""
    d, half = case["dim"], case["rot"] // 2
    if case["interleaved"]:
        first = [2 * i for i in range(half)]
        second = [2 * i + 1 for i in range(half)]
    else:
        first = list(range(half))
        second = [half + i for i in range(half)]
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    unit = torch.ones_like(turn[:1])
    pos = s["positions"].long()
    turn = torch.cat((turn, unit))[torch.where(pos < 0, turn.shape[0], pos)][:, None, :]

    def rotated(y, by):
        z = torch.complex(y[..., first], y[..., second]) * by
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    outs, grads, sums = [], [], []
    for x, w, g in ((s["q"], s["wq"], s.get("gq")), (s["k"], s["wk"], s.get("gk"))):
        x, w = x.detach().double(), w.detach().double()
        size = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / d + EPS)
        outs.append(rotated(x * w / size, turn))
        if case["train"]:
            gy = rotated(g.double(), turn.conj())
            unit_x = x / size
            sums.append(torch.einsum("thd,thd->d", gy, unit_x))
            along = torch.einsum("thd,thd->th", gy * w, unit_x) / d
            grads.append((gy * w - unit_x * along[..., None]) / size)
    return tuple(outs + grads + sums)


def _exact_attention(case, s):
    n_q, n_k, seg = lengths(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    pairs = hq * sum(a * b for a, b in zip(n_q, n_k))
    if pairs * d * (14 if case["train"] else 4) > 1e14:
        return None
    dev = s["q"].device
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    o = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if case["train"] else None
    go = s["g"].double() if case["train"] else None
    row, col = 0, 0
    for a, b, c in zip(n_q, n_k, seg or n_k):
        band = torch.ones(a, b, dtype=torch.bool, device=dev)
        if case["causal"]:
            band = torch.tril(band, diagonal=b - a)
        for h in range(hq):
            i, j = (slice(row, row + a), h), (slice(col, col + b), h * hk // hq)
            logit = torch.einsum("id,jd->ij", q[i], k[j]) / d ** 0.5
            p = torch.softmax(logit.masked_fill(~band, -math.inf), dim=1).nan_to_num(0.0)
            o[i] = p @ v[j]
            if case["train"]:
                dp = go[i] @ v[j].T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / d ** 0.5
                grads[0][i] = ds @ k[j]
                grads[1][j] += ds.T @ q[i]
                grads[2][j] += p.T @ go[i]
            del logit, p
        row, col = row + a, col + c
    return o if not case["train"] else (o, *grads)
