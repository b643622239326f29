"""Sequence attention (fastnn.sequence_attention) against its 64-bit plain form: masks, layouts, types,
sizes around the tiles, empty rows, masked places that hold NaN, gradients, graphs and streams."""

import math

import pytest
import torch

from tests import sequence_reference as ref

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def data(device, dtype, B, H, Hk, nq, nk, D, Dv=None, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    Dv = D if Dv is None else Dv
    make = lambda *shape: (torch.randn(*shape, generator=g) * spread).to(dtype).to(device)            # noqa: E731
    return make(B, H, nq, D), make(B, Hk, nk, D), make(B, Hk, nk, Dv), make(B, H, nq, Dv)


def run(q, k, v, dout, **options):
    from xfold_cpu_amd import fastnn
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    slopes = options.get("slopes")
    leaves = [q, k, v]
    if slopes is not None:
        slopes = options["slopes"] = slopes.detach().requires_grad_()
        leaves.append(slopes)
    out = fastnn.sequence_attention(q, k, v, **options)
    grads = torch.autograd.grad(out, leaves, dout)
    return {"out": out.detach(), **dict(zip(("dq", "dk", "dv", "dslopes"), grads))}


def compare(q, k, v, dout, what, **options):
    print(f"[case] {what}", flush=True)
    got = run(q, k, v, dout, **dict(options))
    want = ref.attend(q, k, v, dout, **options)
    for name in want:
        ref.check(got[name], want[name], f"{what} {name}")
    return got


SHAPES = [  # B, H, Hk, Nq, Nk, D, Dv
    (1, 1, 1, 1, 1, 1, 1), (1, 2, 1, 1, 70, 16, 16), (2, 4, 2, 63, 63, 24, 24), (1, 3, 3, 64, 64, 33, 17),
    (1, 2, 2, 65, 65, 48, 48), (2, 6, 2, 130, 130, 64, 64), (1, 4, 1, 129, 200, 100, 72), (1, 2, 1, 200, 200, 128, 128),
    (1, 8, 2, 3, 321, 80, 96), (3, 1, 1, 17, 129, 5, 128),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_shapes(device, shape, dtype, causal):
    q, k, v, dout = data(device, dtype, *shape, seed=sum(shape))
    compare(q, k, v, dout, f"{shape} {dtype} causal={causal}", causal=causal)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_more_queries_than_keys(device, dtype):
    q, k, v, dout = data(device, dtype, 2, 2, 2, 150, 40, 32)
    compare(q, k, v, dout, "150 queries of 40 keys")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("options", ["cap", "slopes", "cap+slopes"])
def test_cap_and_distance(device, dtype, causal, options):
    q, k, v, dout = data(device, dtype, 2, 4, 2, 90, 150, 40, seed=5, spread=2.0)
    kw = {"causal": causal}
    if "cap" in options:
        kw["softcap"] = 7.0
    if "slopes" in options:
        kw["slopes"] = torch.tensor([0.5, 0.0, 0.03125, -0.01], device=device)
    compare(q, k, v, dout, f"{options} {dtype} causal={causal}", **kw)


def documents(kind, n):
    t = torch.arange(n)
    if kind == "packed":
        return torch.where(t < 10, 3, torch.where(t < 100, 0, torch.where(t < n - 9, 7, -1))).int()
    if kind == "mixed":                                    # tokens of several documents side by side
        return (t * 7 % 5 - 1).int()
    if kind == "single":
        return torch.full((n,), 2 ** 31 - 1).int()
    if kind == "none":
        return torch.full((n,), -1).int()
    return torch.where(t < n // 2, -5, 0).int()            # padding in front


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["packed", "mixed", "single", "none", "left"])
@pytest.mark.parametrize("causal,nq", [(False, 170), (True, 170), (True, 77)])
def test_documents(device, dtype, kind, causal, nq):
    q, k, v, dout = data(device, dtype, 2, 4, 2, nq, 170, 32, seed=nq)
    one = documents(kind, 170).to(device)
    both = torch.stack([one, documents("mixed", 170).to(device)])
    for docs in (one, both):
        got = compare(q, k, v, dout, f"{kind} {dtype} causal={causal} nq={nq}", causal=causal, documents=docs,
                      slopes=torch.tensor([0.1, 0.02, 0.3, 0.0], device=device))
    if kind == "none":
        assert not got["out"][0].any() and not got["dq"][0].any() and not got["dk"][0].any() and not got["dv"][0].any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_prefix(device, dtype):
    q, k, v, dout = data(device, dtype, 4, 2, 1, 140, 140, 48)
    docs = documents("packed", 140).to(device)
    for prefix in (0, 70, 1000, torch.tensor([0, 64, 139, 2 ** 31 - 1], dtype=torch.int32, device=device),
                   torch.tensor([-2 ** 31, 1, 65, 130], dtype=torch.int32, device=device)):
        compare(q, k, v, dout, f"prefix {prefix} {dtype}", causal=True, prefix=prefix)
        compare(q, k, v, dout, f"prefix {prefix} {dtype} documents", causal=True, prefix=prefix, documents=docs)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("nq", [1, 5, 100])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_lengths(device, dtype, nq, causal):
    nk = 300
    lengths = torch.tensor([nk, 0, 1, 63, 64, 65, 4, -3, nk + 9], dtype=torch.int32, device=device)
    q, k, v, dout = data(device, dtype, len(lengths), 4, 2, nq, nk, 64, seed=nq)
    for b, n in enumerate(lengths.tolist()):               # keys from the length on are not read
        k[b, :, max(n, 0):] = math.nan
        v[b, :, max(n, 0):] = math.nan
    docs = torch.arange(nk).div(50, rounding_mode="floor").int().to(device)
    slopes = torch.tensor([0.2, 0.1, 0.0, 0.01], device=device)
    compare(q, k, v, dout, f"lengths nq={nq} {dtype} causal={causal}", causal=causal, lengths=lengths)
    compare(q, k, v, dout, f"lengths nq={nq} {dtype} causal={causal} documents", causal=causal, lengths=lengths,
            documents=docs, softcap=20.0, slopes=slopes)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["padding", "future", "other document"])
def test_masked_places_hold_anything(device, dtype, value, where):
    """What no query sees, or only queries that are not looked at, changes nothing."""
    n = 150
    q, k, v, dout = data(device, dtype, 1, 4, 2, n, n, 32, seed=9)
    docs = torch.zeros(n, dtype=torch.int32)
    kw = {"causal": where == "future"}
    if where == "padding":
        docs[-30:] = -1
        kw["documents"], spoilt = docs.to(device), slice(n - 30, n)
    elif where == "other document":
        docs[40:90] = 1
        kw["documents"], spoilt = docs.to(device), slice(40, 90)
    else:
        spoilt = slice(n - 40, n)
    keep = torch.ones(n, dtype=torch.bool)
    keep[spoilt] = False
    want = run(q, k, v, torch.where(keep.to(device)[:, None], dout, torch.zeros_like(dout)), **kw)
    for t in (q, k, v, dout):
        t[:, :, spoilt] = value
    if where == "future":                                  # (gradients of the others come from the spoilt rows too)
        from xfold_cpu_amd import fastnn
        got = fastnn.sequence_attention(q, k, v, **kw)
        assert torch.equal(got[:, :, keep], want["out"][:, :, keep])
        assert torch.isnan(got[:, :, ~keep]).any()
        q2, k2, v2 = (t.clone() for t in (q, k, v))
        clean = run(q2, k2, v2, dout, **kw)
        assert torch.equal(clean["dq"][:, :, keep], want["dq"][:, :, keep])
        return
    got = run(q, k, v, dout, **kw)
    for name in ("out", "dq", "dk", "dv"):
        assert torch.equal(got[name][:, :, keep], want[name][:, :, keep]), (where, name)
    if where == "padding":
        for name in ("out", "dq", "dk", "dv"):
            assert not got[name][:, :, ~keep].any(), name
    else:
        assert torch.isnan(got["out"][:, :, ~keep]).any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_seen_infinity_in_v(device, dtype):
    q, k, v, dout = data(device, dtype, 1, 1, 1, 70, 70, 16)
    v[0, 0, 3, 5], v[0, 0, 4, 6], v[0, 0, 5, 7] = math.inf, -math.inf, math.nan
    from xfold_cpu_amd import fastnn
    out = fastnn.sequence_attention(q, k, v, causal=True)[0, 0]
    assert torch.isfinite(out[:3]).all()
    assert (out[3:, 5] == math.inf).all() and (out[4:, 6] == -math.inf).all() and torch.isnan(out[5:, 7]).all()
    rest = [d for d in range(16) if d not in (5, 6, 7)]
    assert torch.isfinite(out[:, rest]).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strides(device, dtype):
    B, H, Hk, n, D = 2, 4, 2, 75, 40
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(B, n, (H + 2 * Hk) * D, generator=g).to(dtype).to(device)
    q = fused[..., :H * D].view(B, n, H, D).transpose(1, 2)
    k = fused[..., H * D:(H + Hk) * D].view(B, n, Hk, D).transpose(1, 2)
    v = fused[..., (H + Hk) * D:].view(B, n, Hk, D).transpose(1, 2)
    dout = torch.randn(B, n, H, D, generator=g).to(dtype).to(device).transpose(1, 2)
    got = compare(q, k, v, dout, "heads side by side", causal=True)
    assert got["out"].transpose(1, 2).is_contiguous() and got["dq"].transpose(1, 2).is_contiguous()
    same = run(q.contiguous(), k.contiguous(), v.contiguous(), dout.contiguous(), causal=True)
    for name in same:
        assert torch.equal(same[name], got[name]), name
    # last dim not contiguous; broadcast batch; storage off 16 bytes; expanded gradient
    qt = q.transpose(2, 3).contiguous().transpose(2, 3)
    kx = k[:1].expand(B, Hk, n, D)
    odd = torch.zeros(v.numel() + 1, dtype=dtype, device=device)[1:].view(v.shape).copy_(v)
    ones = torch.ones((), dtype=dtype, device=device).expand(B, H, n, D)
    compare(qt, kx, odd, ones, "transposed, broadcast, off alignment", causal=True)
    compare(q[:, ::2], k[:, 1:], v[:, 1:], dout[:, ::2], "every other head", causal=False)
    compare(q[:, :, ::3], k, v, dout[:, :, ::3], "every third query", causal=True)


def test_broadcast_gradient_is_summed(device):
    q, k, v, dout = data(device, F32, 3, 2, 1, 20, 20, 8)
    from xfold_cpu_amd import fastnn
    kx = k[:1].detach().requires_grad_()
    out = fastnn.sequence_attention(q, kx.expand(3, 1, 20, 8), v)
    (got,) = torch.autograd.grad(out, [kx], dout)
    want = ref.attend(q, kx.detach().expand(3, 1, 20, 8), v, dout)["dk"]
    ref.check(got, (want[0].sum(0, keepdim=True), want[1].sum(0, keepdim=True) + 3 * ref.U32 * want[0].abs().sum(0)), "dk")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_unbatched_and_no_gradient(device, dtype):
    q, k, v, dout = data(device, dtype, 1, 2, 2, 30, 30, 16)
    from xfold_cpu_amd import fastnn
    whole = fastnn.sequence_attention(q, k, v, causal=True)
    assert not whole.requires_grad
    assert torch.equal(fastnn.sequence_attention(q[0], k[0], v[0], causal=True), whole[0])
    with torch.no_grad():
        out = fastnn.sequence_attention(q.requires_grad_(), k, v, causal=True)
    assert torch.equal(out, whole) and not out.requires_grad
    (dk,) = torch.autograd.grad(fastnn.sequence_attention(q.detach(), k.requires_grad_(), v, causal=True), [k], dout)
    assert torch.equal(dk, run(q, k, v, dout, causal=True)["dk"])


def test_only_what_is_asked_for(device):
    q, k, v, dout = data(device, BF16, 1, 4, 2, 100, 100, 32)
    slopes = torch.tensor([0.1, 0.0, 0.2, 0.3], device=device)
    from xfold_cpu_amd import fastnn
    want = run(q, k, v, dout, causal=True, slopes=slopes)
    t = {"q": q, "k": k, "v": v, "slopes": slopes}
    for name in t:
        leaf = t[name].detach().requires_grad_()
        kw = {**t, name: leaf}
        out = fastnn.sequence_attention(kw["q"], kw["k"], kw["v"], causal=True, slopes=kw["slopes"])
        (g,) = torch.autograd.grad(out, [leaf], dout)
        assert torch.equal(g, want["d" + name]), name


def test_empty(device):
    from xfold_cpu_amd import fastnn
    for shape in [(0, 2, 1, 5, 5, 8), (2, 2, 1, 0, 5, 8), (2, 2, 1, 5, 0, 8), (1, 0, 1, 5, 5, 8)]:
        q, k, v, dout = data(device, BF16, *shape)
        got = run(q, k, v, dout, slopes=torch.zeros(shape[1], device=device))
        for name in ("out", "dq", "dk", "dv", "dslopes"):
            assert not got[name].any(), (shape, name)


def test_large_scores(device):
    """Scores far beyond exp's range, and all equal."""
    q, k, v, dout = data(device, F32, 1, 1, 1, 70, 70, 16, spread=30.0)
    compare(q, k, v, dout, "large scores", causal=True)
    compare(torch.zeros_like(q), k, v, dout, "equal scores", causal=True)


def test_gradients_against_differences(device):
    """<gradient, direction> against central differences of the 64-bit plain form."""
    shape = (1, 2, 1, 40, 40, 16)
    q, k, v, dout = data(device, F32, *shape, seed=3)
    docs = documents("mixed", 40).to(device)
    slopes = torch.tensor([0.05, 0.2], device=device)
    kw = dict(causal=True, prefix=11, documents=docs, softcap=4.0)
    got = run(q, k, v, dout, slopes=slopes, **kw)
    g = torch.Generator().manual_seed(4)
    base = {"q": q.cpu().double(), "k": k.cpu().double(), "v": v.cpu().double(), "slopes": slopes.cpu().double()}
    for name in base:
        way = torch.randn(base[name].shape, generator=g, dtype=torch.float64)
        values = []
        for sign in (1, -1):
            moved = {**base, name: base[name] + sign * 1e-5 * way}
            s = moved.pop("slopes")
            out = ref.attend(moved["q"], moved["k"], moved["v"], slopes=s, **kw)["out"][0]
            values.append(float((out * dout.cpu().double()).sum()))
        want = (values[0] - values[1]) / 2e-5
        mine = float((got["d" + name].cpu().double() * way).sum())
        size = float(got["d" + name].cpu().double().norm() * way.norm())
        # differences: 1e-10 of third order, 64-bit rounding over 1e-5; the kernel: FP32 over 40-term sums.
        assert abs(mine - want) <= 1e-5 * size + 1e-8, (name, mine, want)


def test_autocast(device):
    from xfold_cpu_amd import fastnn
    q, k, v, dout = data(device, F32, 1, 2, 1, 50, 50, 24)
    low = [t.to(BF16) for t in (q, k, v, dout)]
    want = run(*low, causal=True)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    with torch.autocast("cuda", dtype=BF16):
        out = fastnn.sequence_attention(*leaves, causal=True)
    assert out.dtype == BF16 and torch.equal(out.detach(), want["out"])
    grads = torch.autograd.grad(out, leaves, low[3])
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert got.dtype == F32 and torch.equal(got, want[name].float()), name


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_same_bits_every_time_and_on_another_stream(device, dtype):
    q, k, v, dout = data(device, dtype, 2, 8, 2, 333, 333, 64)
    kw = dict(causal=True, softcap=15.0, slopes=torch.linspace(0.0, 0.3, 8, device=device),
              documents=documents("packed", 333).to(device))
    first = run(q, k, v, dout, **dict(kw))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(q, k, v, dout, **dict(kw))
    third = run(q, k, v, dout, **dict(kw))                 # both in flight
    torch.cuda.synchronize()
    for name in first:
        assert torch.equal(first[name], second[name]) and torch.equal(first[name], third[name]), name


def test_graph_replays(device):
    from tests.test_gpu_graph import capture
    q, k, v, dout = data(device, BF16, 2, 4, 2, 130, 130, 48)
    docs = documents("packed", 130).to(device)
    slopes = torch.tensor([0.1, 0.2, 0.0, 0.05], device=device)
    held = {}

    def step():
        held.update(run(q, k, v, dout, causal=True, documents=docs, slopes=slopes, softcap=9.0))
    graph = capture(step)
    captured = dict(held)
    for seed in range(3):
        new = data(device, BF16, 2, 4, 2, 130, 130, 48, seed=20 + seed)
        for old, t in zip((q, k, v, dout), new):
            old.copy_(t)
        docs.copy_(documents(("mixed", "left", "packed")[seed], 130))
        graph.replay()
        torch.cuda.synchronize()
        got = {name: t.clone() for name, t in captured.items()}
        want = run(q, k, v, dout, causal=True, documents=docs, slopes=slopes, softcap=9.0)
        for name in want:
            assert torch.equal(got[name], want[name]), (seed, name)


def test_offsets_beyond_32_bits(device):
    """A cache whose second entry and last token start past 2^31 elements."""
    far, D, n = 2 ** 31 + 64, 32, 70
    store = torch.zeros(far + 2 ** 20, dtype=BF16, device=device)
    q, k, v, dout = data(device, BF16, 2, 2, 1, n, n, D, seed=8)
    kc = store.as_strided((2, 1, n, D), (far, 0, D, 1)).copy_(k)
    compare(q, kc, v, dout, "batch stride over 2^31", causal=True)
    step = far // (n - 1) // 8 * 8 + 8
    vc = store.as_strided((1, 1, n, D), (0, 0, step, 1)).copy_(v[:1])
    compare(q[:1], k[:1], vc, dout[:1], "token stride to 2^31", causal=True)


def test_second_backward_is_refused(device):
    from xfold_cpu_amd import fastnn
    q, k, v, _ = data(device, F32, 1, 1, 1, 5, 5, 4)
    q.requires_grad_()
    (dq,) = torch.autograd.grad(fastnn.sequence_attention(q, k, v).sum(), [q], create_graph=True)
    with pytest.raises(RuntimeError):
        dq.sum().backward()


SPLIT = [  # B, H, Hk, Nq, Nk, D: few work items, so keys, heads and queries are split and joined
    (1, 2, 1, 1, 2100, 48), (2, 4, 2, 7, 1500, 128), (1, 3, 1, 40, 3000, 33), (1, 1, 1, 200, 1100, 64), (1, 4, 1, 600, 600, 24),
    (1, 2, 2, 700, 700, 96),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SPLIT, ids=lambda s: "x".join(map(str, s)))
def test_split_work(device, shape, dtype):
    B, H, Hk, nq, nk, D = shape
    q, k, v, dout = data(device, dtype, *shape, seed=nq)
    compare(q, k, v, dout, f"split {shape} {dtype}", causal=True, softcap=25.0)
    docs = documents("packed", nk).to(device)
    compare(q, k, v, dout, f"split {shape} {dtype} documents", documents=docs,
            slopes=torch.linspace(0.0, 0.02, H, device=device))
    lengths = torch.tensor([nk // 3, 0][:B], dtype=torch.int32, device=device)
    got = compare(q, k, v, dout, f"split {shape} {dtype} lengths", causal=True, lengths=lengths)
    if B > 1:
        assert not got["out"][1].any() and not got["dk"][1].any()
    # a NaN that only the last query's documents hide
    docs = torch.zeros(nk, dtype=torch.int32, device=device)
    docs[nk // 2] = 5
    want = run(q, k, v, dout, causal=True, documents=docs)
    rest = torch.arange(nk, device=device) != nk // 2
    for t in (k, v):
        t[:, :, nk // 2] = math.nan
    got = run(q, k, v, dout, causal=True, documents=docs)
    own = rest[nk - nq:]
    assert torch.equal(got["out"][:, :, own], want["out"][:, :, own]) and torch.equal(got["dq"][:, :, own], want["dq"][:, :, own])
    for name in ("dk", "dv"):
        assert torch.equal(got[name][:, :, rest], want[name][:, :, rest]), name


def test_two_calls_at_once(device):
    """Calls of two threads on streams of their own, and of one thread on two streams, with split work."""
    import threading
    cases = [data(device, BF16, 1, 4, 1, 300, 900, 64, seed=s) for s in (1, 2)]
    kw = dict(causal=True, softcap=10.0)
    want = [run(*c, **kw) for c in cases]
    torch.cuda.synchronize()
    got, streams = [None, None], [torch.cuda.Stream(), torch.cuda.Stream()]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                got[i] = run(*cases[i], **kw)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        for name in want[i]:
            assert torch.equal(got[i][name], want[i][name]), name


RAGGED = [  # H, Hk, Nq, Nk, D, lengths: the sequences share the parts by their lengths
    (8, 2, 5, 2300, 128, (2300, 17, 0, 900, 1)), (4, 1, 150, 1700, 64, (1, 1700, 64, 1100)),
    (2, 1, 1, 600, 24, tuple((37 * i) % 601 for i in range(70))), (3, 1, 40, 3000, 33, (3000, 30)),
    (2, 2, 90, 2100, 96, (0, 0, 0)),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", RAGGED, ids=lambda s: "x".join(map(str, (len(s[5]),) + s[:5])))
def test_split_sequences_of_different_lengths(device, shape, dtype):
    H, Hk, nq, nk, D, lengths = shape
    q, k, v, dout = data(device, dtype, len(lengths), H, Hk, nq, nk, D, seed=nk)
    lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
    compare(q, k, v, dout, f"lengths {shape} {dtype}", causal=True, lengths=lengths)
    compare(q, k, v, dout, f"lengths {shape} {dtype} documents", documents=documents("packed", nk).to(device), lengths=lengths)


def test_captured_call_reads_the_lengths_of_its_replay(device):
    from xfold_cpu_amd import fastnn
    q, k, v, _ = data(device, BF16, 4, 8, 2, 30, 2000, 64, seed=11)
    lengths = torch.tensor([2000, 40, 700, 0], dtype=torch.int32, device=device)
    call = lambda: fastnn.sequence_attention(q, k, v, causal=True, lengths=lengths)           # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for now in ((2000, 40, 700, 0), (1, 2000, 2000, 2000), (65, 0, 0, 1999), (2000, 2000, 2000, 2000)):
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call()), now


def test_refusals_of_the_library_are_value_errors(device):
    from xfold_cpu_amd import fastnn
    from xfold_cpu_amd.fastnn import native_hip as nh
    q, k, v, _ = data(device, F32, 1, 1, 1, 5, 5, 4)
    for leaf in (q, q.clone().requires_grad_()):
        with pytest.raises(ValueError, match="softcap too small"):
            fastnn.sequence_attention(leaf, k, v, softcap=1e-39)
        with pytest.raises(ValueError, match="eps must be nonnegative"):
            nh.autograd().trainable_layer_norm(leaf, None, None, 4, -1.0, False)
    out = fastnn.sequence_attention(q, k, v)                       # nothing is left behind
    assert torch.equal(out, fastnn.sequence_attention(q, k, v))
