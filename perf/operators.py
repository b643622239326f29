"""Cases of the training LayerNorm and of sequence attention: what is measured of them, their plain
forms in elementary torch operations, and their values in 64 bits.

LayerNorm: y = (x - mean) * rstd * w + b over the last dim, and its backward pass (dx, dw, db).
Sequence attention: softmax over the visible keys of cap * tanh(scale q.k / cap) - slope |distance|,
with causal, prefix, document and length masks, shared key heads, and its backward pass. The queries
are the last Nq tokens of each sequence; a query that sees no key gives zeros.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def _norm(name, rows, cols, dtype, wdtype="f32"):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "wdtype": wdtype}


def _attend(name, train, batch, heads, kv_heads, dim, nq, nk, dtype, causal=False, prefix=0, documents=0, pad=0,
            shortest=0, cap=0.0, slopes=False):
    return {"name": name, "op": "attend", "train": train, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "nq": nq, "nk": nk, "dtype": dtype, "causal": causal, "prefix": prefix,
            "documents": documents, "pad": pad, "shortest": shortest, "cap": cap, "slopes": slopes}


def listed():
    return [
        # The single track (384 channels) of a 72-token input: launches and host work.
        _norm("norm 72x384 f32", 72, 384, "f32"),
        # A pair tensor's norm at 768 tokens and 128 channels: many short rows.
        _norm("norm 589824x128 bf16", 768 * 768, 128, "bf16"),
        # A language model's hidden states, weights in the activations' type.
        _norm("norm 8192x4096 bf16", 8192, 4096, "bf16", "bf16"),
        # An odd width: no row but the first starts on 16 bytes.
        _norm("norm 5003x769 f32", 5003, 769, "f32"),
        # Training on the single track (16 heads of 24), three chains in one sequence, learned distance slopes.
        _attend("train 384 16x24 f32 chains", True, 1, 16, 16, 24, 384, 384, "f32", documents=3, pad=17, slopes=True),
        # Training the diffusion transformer's attention (16 heads of 48, 5 samples), padding, distance slopes.
        _attend("train 5x768 16x48 bf16", True, 5, 16, 16, 48, 768, 768, "bf16", documents=1, pad=77, slopes=True),
        # Training on packed sequences of many lengths, shared key heads.
        _attend("train 2x4096 16/4x128 bf16 packed", True, 2, 16, 4, 128, 4096, 4096, "bf16", causal=True, documents=5),
        # Training with a prefix that all tokens see, capped scores, a length that fits no tile.
        _attend("train 3x1111 8/2x64 bf16 prefix", True, 3, 8, 2, 64, 1111, 1111, "bf16", causal=True, prefix=300, cap=30.0),
        # A long prompt with capped scores.
        _attend("prompt 8192 16/8x128 bf16 cap", False, 1, 16, 8, 128, 8192, 8192, "bf16", causal=True, cap=50.0),
        # The next 200 tokens of sequences whose keys so far are in a cache, each with its own length.
        _attend("chunk 4x200 of 5000 32/8x128 bf16", False, 4, 32, 8, 128, 200, 5000, "bf16", causal=True, shortest=1500),
        # One token each of 16 running sequences over a long cache.
        _attend("token 16x1 of 8192 32/8x128 bf16", False, 16, 32, 8, 128, 1, 8192, "bf16", causal=True, shortest=700,
                cap=50.0),
        # One token of a short sequence: the smallest call.
        _attend("token 1x1 of 257 16x48 bf16", False, 1, 16, 16, 48, 1, 257, "bf16", causal=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.35:
        cols = _spread(rng, 16, 8192)
        if rng.random() < 0.6:
            cols = max(8, cols // 8 * 8)
        rows = _spread(rng, 1, min(600000, 33000000 // cols))
        dtype = rng.choice(["f32", "bf16"])
        c = _norm("", rows, cols, dtype, rng.choice(["f32", dtype]))
    else:
        kind = rng.choice(["train", "train", "prompt", "chunk", "token"])
        kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
        dim = rng.choice([16, 24, 32, 40, 48, 64, 72, 96, 128])
        batch = rng.randint(1, 6)
        dtype = rng.choice(["bf16", "bf16", "f32"])
        cap = rng.choice([0.0, 0.0, 20.0, 50.0])
        slopes = rng.random() < 0.3
        if kind in ("train", "prompt"):
            most = int(math.sqrt((6e7 if dtype == "f32" else 2.5e8) / (batch * kv * group)))
            n = _spread(rng, 16, max(17, min(4096 if kind == "train" else 8192, most)))
            causal = rng.random() < 0.6
            c = _attend("", kind == "train", batch, kv * group, kv, dim, n, n, dtype, causal,
                        rng.randint(1, n) if causal and rng.random() < 0.4 else 0, rng.choice([0, 0, 1, 4]),
                        0, 0, cap, slopes)
            if c["documents"]:
                c["pad"] = rng.randint(0, n // 8)
        else:
            nk = _spread(rng, 64, 8192)
            nq = 1 if kind == "token" else _spread(rng, 2, min(nk, 512))
            c = _attend("", False, batch, kv * group, kv, dim, nq, nk, dtype, True, 0, 0, 0,
                        rng.randint(max(1, nk // 8), nk), cap, slopes)
    del c["name"]
    return c


# ------------------------------------------------------------------------------ inputs

def _lengths(case):
    """Sequence lengths in the cache, spread from `shortest` to the whole of it (0: no lengths)."""
    if not case["shortest"]:
        return None
    return np.linspace(case["nk"], case["shortest"], case["batch"]).astype(np.int64)


def _documents(case):
    """Document of each token: runs of uneven lengths, the last `pad` tokens in none."""
    if not case["documents"]:
        return None
    n = case["nk"] - case["pad"]
    share = np.array([1.0 + (3 * i) % 5 for i in range(case["documents"])])
    ends = np.round(np.cumsum(share) / share.sum() * n).astype(np.int64)
    ids = np.searchsorted(ends, np.arange(n), side="right")
    return np.concatenate([ids, np.full(case["pad"], -1)]).astype(np.int32)


def _visible_pairs(case):
    """Number of (batch entry, query, key) triples that the masks leave."""
    nq, nk, total = case["nq"], case["nk"], 0
    lengths, ids = _lengths(case), _documents(case)
    for b in range(case["batch"]):
        n = nk if lengths is None else int(lengths[b])
        pos = np.arange(nq) + n - nq
        pos = pos[pos >= 0]
        low, high = np.zeros_like(pos), np.full_like(pos, n)
        if ids is not None:
            kept = ids[pos]
            pos = pos[kept >= 0]
            low = np.searchsorted(ids[: nk - case["pad"]], ids[pos], side="left")
            high = np.searchsorted(ids[: nk - case["pad"]], ids[pos], side="right")
        if case["causal"]:
            high = np.minimum(high, np.maximum(pos + 1, min(case["prefix"], n)))
        total += int(np.maximum(high - low, 0).sum())
    return total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, spread=1.0, middle=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * spread + middle).to(dtype)

    dtype = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, cols, wdtype = case["rows"], case["cols"], DTYPES[case["wdtype"]]
        s = {"x": normal((rows, cols), dtype, 1.5, 0.3).requires_grad_(),
             "w": normal((cols,), wdtype, 0.2, 1.0).requires_grad_(), "b": normal((cols,), wdtype, 0.2).requires_grad_(),
             "dy": normal((rows, cols), dtype)}
        return {"case": case, **s}
    B, H, Hk, D, nq, nk = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "nq", "nk"))
    train = case["train"]
    # Heads side by side in a token's row, as a projection leaves them; a cache is held head by head.
    q = normal((B, nq, H, D), dtype, 2.0 if case["cap"] else 1.2).transpose(1, 2)
    if case["shortest"]:
        k, v = normal((B, Hk, nk, D), dtype), normal((B, Hk, nk, D), dtype)
    else:
        k, v = normal((B, nk, Hk, D), dtype).transpose(1, 2), normal((B, nk, Hk, D), dtype).transpose(1, 2)
    s = {"q": q.requires_grad_(train), "k": k.requires_grad_(train), "v": v.requires_grad_(train)}
    lengths, ids = _lengths(case), _documents(case)
    s["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["documents"] = None if ids is None else torch.tensor(ids, device="cuda").expand(B, nk).contiguous()
    s["prefix"] = torch.full((B,), case["prefix"], dtype=torch.int32, device="cuda") if case["prefix"] else None
    s["slopes"] = None
    if case["slopes"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda").requires_grad_(train)
    if train:
        s["dout"] = normal((B, nq, H, D), dtype).transpose(1, 2)
    return {"case": case, **s}


# ------------------------------------------------------------------------------ one pass

def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return (_plain_norm if state["case"]["op"] == "norm" else _plain_attend)(state)


def _own(s):
    from xfold_cpu_amd import fastnn

    case = s["case"]
    if case["op"] == "norm":
        y = fastnn.trainable_layer_norm(s["x"], (case["cols"],), s["w"], s["b"], EPS)
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    out = fastnn.sequence_attention(s["q"], s["k"], s["v"], causal=case["causal"], prefix=s["prefix"],
                                    documents=s["documents"], lengths=s["lengths"], softcap=case["cap"] or None,
                                    slopes=s["slopes"])
    if not case["train"]:
        return {"out": out}
    leaves = [s["q"], s["k"], s["v"]] + ([s["slopes"]] if case["slopes"] else [])
    grads = torch.autograd.grad(out, leaves, s["dout"])
    return {"out": out.detach(), **dict(zip(("dq", "dk", "dv", "dslopes"), grads))}


def _plain_norm(s):
    x, w, dy = s["x"].float(), s["w"].float(), s["dy"].float()
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    h = centred * rstd
    y = h * w + s["b"].float()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return {"y": y.to(s["x"].dtype), "dx": dx.to(s["x"].dtype), "dw": (dy * h).sum(0).to(s["w"].dtype),
            "db": dy.sum(0).to(s["b"].dtype)}


def _plain_attend(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    dtype, device = q.dtype, q.device
    (B, H, nq, D), Hk, nk = q.shape, k.shape[1], k.shape[2]
    group, scale, cap = H // Hk, D ** -0.5, case["cap"]
    rows = lambda t: t.float().reshape(B, Hk, group * nq, D)                          # noqa: E731
    k32, v32 = k.float().contiguous(), v.float().contiguous()

    keys = torch.arange(nk, device=device)
    n = torch.full((B,), nk, device=device) if s["lengths"] is None else s["lengths"].long()
    pos = torch.arange(nq, device=device)[None] + (n - nq)[:, None]                   # [B, nq]
    keep = (keys[None, None] < n[:, None, None]) & (pos[:, :, None] >= 0)
    if case["causal"]:
        seen = keys[None, None] <= pos[:, :, None]
        if s["prefix"] is not None:
            seen = seen | (keys[None, None] < s["prefix"][:, None, None])
        keep = keep & seen
    if s["documents"] is not None:
        mine = torch.gather(s["documents"], 1, pos.clamp(min=0))
        keep = keep & (mine[:, :, None] == s["documents"][:, None]) & (mine >= 0)[:, :, None]
    keep = keep[:, None, None]                                                        # [B, 1, 1, nq, nk]

    q32 = rows(q)
    score = torch.matmul(q32, k32.transpose(2, 3)).mul_(scale).view(B, Hk, group, nq, nk)
    if cap:
        capped = torch.tanh(score / cap)
        score = capped * cap
    if s["slopes"] is not None:
        distance = (pos[:, :, None] - keys).abs().float()[:, None, None]
        score = score - s["slopes"].view(1, Hk, group, 1, 1) * distance
    score = score.masked_fill(~keep, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    del score
    flat = p.view(B, Hk, group * nq, nk)
    out = torch.matmul(flat, v32)
    result = {"out": out.view(B, H, nq, D).to(dtype)}
    if not case["train"]:
        return result
    dout = rows(s["dout"])
    result["dv"] = torch.matmul(flat.transpose(2, 3), dout).to(dtype)
    dp = torch.matmul(dout, v32.transpose(2, 3))
    delta = (dout * out).sum(-1, keepdim=True)
    ds = (flat * (dp - delta)).view(B, Hk, group, nq, nk)
    if s["slopes"] is not None:
        result["dslopes"] = -(ds * distance).sum(-1).double().sum((0, 3)).reshape(H).float()
    if cap:
        ds = ds * (1.0 - capped * capped)
    ds = ds.mul_(scale).view(B, Hk, group * nq, nk)
    result["dq"] = torch.matmul(ds, k32).view(B, H, nq, D).to(dtype)
    result["dk"] = torch.matmul(ds.transpose(2, 3), q32).to(dtype)
    return result


# ------------------------------------------------------------------------------ what a pass needs

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        elements = case["rows"] * case["cols"]
        wsize = 4 if case["wdtype"] == "f32" else 2
        return {"bytes": 4 * elements * size + 4 * case["cols"] * wsize, "flops": 22 * elements}
    B, H, Hk, D, nq, nk = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "nq", "nk"))
    lengths = _lengths(case)
    tokens = B * nk if lengths is None else int(lengths.sum())
    pairs = _visible_pairs(case) * H
    queries, cached = B * H * nq * D * size, tokens * Hk * D * size
    if not case["train"]:
        return {"bytes": 2 * queries + 2 * cached, "flops": 4 * D * pairs}
    return {"bytes": 4 * queries + 4 * cached, "flops": 14 * D * pairs}


# ------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(s) if case["op"] == "norm" else _exact_attend(s)


def _exact_norm(s):
    x, w, b, dy = (s[name].detach().double() for name in ("x", "w", "b", "dy"))
    count = x.shape[1]
    mu = x.sum(1) / count
    var = (x * x).sum(1) / count - mu * mu
    sigma = (var + EPS).sqrt()
    unit = (x - mu[:, None]) / sigma[:, None]
    # The derivative of the normalised row, projected off the constant and off the row itself.
    scaled = dy * w
    along = (scaled * unit).sum(1) / count
    return {"y": unit * w + b, "dx": (scaled - (scaled.sum(1) / count)[:, None] - along[:, None] * unit) / sigma[:, None],
            "dw": (unit * dy).sum(0), "db": dy.sum(0)}


def _exact_attend(s):
    case = s["case"]
    B, H, Hk, D, nq, nk = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "nq", "nk"))
    q, k, v = (s[name].detach().double() for name in ("q", "k", "v"))
    train, cap, device = case["train"], case["cap"], q.device
    lengths, ids = _lengths(case), _documents(case)
    out = torch.zeros_like(q)
    given = s["dout"].double() if train else None
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v)) if train else (None, None, None)
    dslopes = torch.zeros(H, dtype=torch.float64, device=device)
    column = torch.arange(nk, device=device)
    for b in range(B):
        n = nk if lengths is None else int(lengths[b])
        row = torch.arange(n - nq, n, device=device)
        visible = (column[None] < n) & (row[:, None] >= 0)
        if case["causal"]:
            visible &= column[None] < (row[:, None] + 1).clamp(min=case["prefix"])
        if ids is not None:
            t = torch.tensor(ids, device=device)
            of = t[row.clamp(min=0)]
            visible &= (of[:, None] == t[None]) & (of[:, None] != -1)
        gap = (row[:, None] - column[None]).abs().double()
        for h in range(H):
            kv = h * Hk // H
            raw = q[b, h] @ k[b, kv].T / math.sqrt(D)
            bent = cap * torch.tanh(raw / cap) if cap else raw
            logits = bent - float(s["slopes"][h]) * gap if case["slopes"] else bent
            weight = torch.softmax(logits.masked_fill(~visible, -math.inf), -1).masked_fill(~visible, 0.0)
            out[b, h] = weight @ v[b, kv]
            if not train:
                continue
            g = given[b, h]
            dv[b, kv] += weight.T @ g
            back = g @ v[b, kv].T
            back = weight * (back - (weight * back).sum(1, keepdim=True))
            if case["slopes"]:
                dslopes[h] -= (back * gap).sum()
            if cap:
                back = back * (1.0 - (bent / cap) ** 2)
            dq[b, h] = back @ k[b, kv] / math.sqrt(D)
            dk[b, kv] += back.T @ q[b, h] / math.sqrt(D)
    if not train:
        return {"out": out}
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, **({"dslopes": dslopes} if case["slopes"] else {})}
