"""The training LayerNorm (fastnn.trainable_layer_norm, LayerNorm in training mode) against its 64-bit plain
form: sizes around the kernels' row widths, types, strides, gradients, graphs; and a pre-norm attention
sub-block of it and sequence attention, trained as one."""

import math

import pytest
import torch

from tests import sequence_reference as ref

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-5


def data(device, dtype, wdtype, rows, C, seed=0, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g)                                                    # noqa: E731
    return ((make(rows, C) * 1.5 + mean).to(dtype).to(device), (make(C) * 0.3 + 1).to(wdtype).to(device),
            (make(C) * 0.3).to(wdtype).to(device), make(rows, C).to(dtype).to(device))


def run(x, w, b, dy, eps=EPS):
    from xfold_cpu_amd import fastnn
    leaves = {name: t.detach().requires_grad_() for name, t in (("x", x), ("w", w), ("b", b)) if t is not None}
    y = fastnn.trainable_layer_norm(leaves["x"], (x.shape[-1],), leaves.get("w"), leaves.get("b"), eps)
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    return {"y": y.detach(), **{"d" + name: g for name, g in zip(leaves, grads)}}


def compare(x, w, b, dy, what, eps=EPS):
    print(f"[case] {what}", flush=True)
    got = run(x, w, b, dy, eps)
    want = ref.norm(x, w, b, dy, eps, x.dtype)
    for name in got:
        ref.check(got[name], want[name], f"{what} {name}")
    return got


SIZES = [(1, 1), (3, 7), (5, 8), (72, 384), (40, 128), (1000, 129), (33, 256), (9, 257), (7, 512), (6, 520), (7, 769),
         (4, 1024), (5, 1032), (3, 2048), (5, 4096), (2, 4104), (3, 8191), (2, 16384), (2, 16385), (70, 20000), (20011, 16),
         (33001, 24)]


@pytest.mark.parametrize("types", [(F32, F32), (BF16, F32), (BF16, BF16)], ids=["f32", "bf16-f32", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_sizes(device, size, types):
    x, w, b, dy = data(device, *types, *size, seed=size[1])
    compare(x, w, b, dy, f"{size} {types}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_parameters_may_be_missing(device, dtype):
    x, w, b, dy = data(device, dtype, F32, 50, 96)
    compare(x, None, None, dy, "no weight, no bias")
    compare(x, w, None, dy, "no bias")
    compare(x, None, b, dy, "no weight")
    compare(x, w.to(BF16), b, dy, "weight and bias of two types")


def test_large_mean_and_constant_rows(device):
    x, w, b, dy = data(device, F32, F32, 40, 300, mean=1000.0)
    compare(x, w, b, dy, "mean 1000 times the deviation")
    compare(torch.full_like(x, 3.0), w, b, dy, "constant rows")


def test_strides_and_shapes(device):
    x, w, b, dy = data(device, BF16, F32, 60, 64)
    wide = torch.zeros(60, 200, dtype=BF16, device=device)
    wide[:, 8:72] = x
    off = torch.zeros(60, 201, dtype=BF16, device=device)
    off[:, 3:67] = dy
    compare(wide[:, 8:72], w, b, off[:, 3:67], "slices of wider rows")
    compare(x.t().contiguous().t(), w, b, dy.t().contiguous().t(), "transposed")
    compare(x[:1].expand(60, 64), w, b, dy[:1].expand(60, 64), "expanded")
    from xfold_cpu_amd import fastnn
    flat = run(x, w, b, dy)
    leaf = x.view(3, 20, 4, 16).detach().requires_grad_()
    y = fastnn.trainable_layer_norm(leaf, (4, 16), w.view(4, 16), b.view(4, 16))
    (dx,) = torch.autograd.grad(y, [leaf], dy.view(3, 20, 4, 16))
    assert torch.equal(y.detach().view(60, 64), flat["y"]) and torch.equal(dx.view(60, 64), flat["dx"])


def test_no_rows(device):
    x, w, b, dy = data(device, F32, F32, 0, 32)
    got = run(x, w, b, dy)
    assert got["y"].shape == (0, 32) and got["dx"].shape == (0, 32) and not got["dw"].any() and not got["db"].any()


@pytest.mark.parametrize("C", [128, 769, 4096])
def test_a_bad_row_leaves_the_others_alone(device, C):
    x, w, b, dy = data(device, F32, F32, 40, C)
    want = run(x, w, b, dy)
    x[7], x[9, 3] = math.nan, math.inf
    got = run(x, w, b, dy)
    keep = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(got["y"][keep], want["y"][keep]) and torch.equal(got["dx"][keep], want["dx"][keep])
    assert torch.isnan(got["y"][7]).all() and torch.equal(got["db"], want["db"])


def test_only_what_is_asked_for(device):
    from xfold_cpu_amd import fastnn
    x, w, b, dy = data(device, BF16, F32, 50, 384)
    want = run(x, w, b, dy)
    for name in ("x", "w", "b"):
        t = {"x": x, "w": w, "b": b}
        t[name] = t[name].detach().requires_grad_()
        y = fastnn.trainable_layer_norm(t["x"], 384, t["w"], t["b"])
        (g,) = torch.autograd.grad(y, [t[name]], dy)
        assert torch.equal(g, want["d" + name]), name
    y = fastnn.trainable_layer_norm(x, 384, w, b)
    assert not y.requires_grad and torch.equal(y, want["y"])


def test_gradients_against_differences(device):
    x, w, b, dy = data(device, F32, F32, 6, 40)
    got = run(x, w, b, dy)
    g = torch.Generator().manual_seed(2)
    base = {"x": x.cpu().double(), "w": w.cpu().double(), "b": b.cpu().double()}
    for name in base:
        way, values = torch.randn(base[name].shape, generator=g, dtype=torch.float64), []
        for sign in (1, -1):
            t = {**base, name: base[name] + sign * 1e-5 * way}
            d = t["x"] - t["x"].mean(1, keepdim=True)
            y = d / ((d * d).mean(1, keepdim=True) + EPS).sqrt() * t["w"] + t["b"]
            values.append(float((y * dy.cpu().double()).sum()))
        size = float(got["d" + name].cpu().double().norm() * way.norm())
        mine = float((got["d" + name].cpu().double() * way).sum())
        # differences: 1e-10 of third order, 64-bit rounding over 1e-5; the kernel: FP32 over 40-term sums.
        assert abs(mine - (values[0] - values[1]) / 2e-5) <= 1e-5 * size + 1e-8, name


def test_module_in_training_mode(device):
    from xfold_cpu_amd import fastnn
    x, w, b, dy = data(device, BF16, F32, 30, 384)
    module = fastnn.LayerNorm(384).to(device)
    with torch.no_grad():
        module.weight.copy_(w)
        module.bias.copy_(b)
    want = run(x, w, b, dy)
    leaf = x.detach().requires_grad_()
    y = module(leaf)
    y.backward(dy)
    assert torch.equal(y.detach(), want["y"]) and torch.equal(leaf.grad, want["dx"])
    assert torch.equal(module.weight.grad, want["dw"]) and torch.equal(module.bias.grad, want["db"])
    with torch.autocast("cuda", dtype=BF16):
        high = module(leaf)
    assert high.dtype == F32
    ref.check(high, ref.norm(x, w, b, dy, EPS, F32)["y"], "autocast")
    (dx,) = torch.autograd.grad(high, [leaf], dy.float())
    ref.check(dx, ref.norm(x, w, b, dy, EPS, F32)["dx"], "autocast dx")
    with torch.no_grad():
        module.eval()
        assert module(x).dtype == BF16


def test_graph_replays_and_streams(device):
    from tests.test_gpu_graph import capture
    x, w, b, dy = data(device, BF16, F32, 700, 384)
    held = {}
    graph = capture(lambda: held.update(run(x, w, b, dy)))
    captured = dict(held)
    for seed in range(3):
        new = data(device, BF16, F32, 700, 384, seed=30 + seed)
        for old, t in zip((x, w, b, dy), new):
            old.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        got = {name: t.clone() for name, t in captured.items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = run(x, w, b, dy)
        torch.cuda.synchronize()
        for name in want:
            assert torch.equal(got[name], want[name]), (seed, name)


def test_more_rows_than_a_launch(device):
    from xfold_cpu_amd import fastnn
    rows, C = (1 << 26) + 5, 2
    x = torch.empty(rows, C, dtype=BF16, device=device).copy_((torch.arange(rows, device=device) % 253)[:, None])
    x[:, 1] -= (torch.arange(rows, device=device) % 7).to(BF16)
    w, b = torch.tensor([1.5, -0.5], device=device), torch.tensor([0.25, 4.0], device=device)
    for part in (slice(0, 100), slice((1 << 26) - 50, (1 << 26) + 5)):
        leaf, some = x.detach().requires_grad_(), x[part].detach().requires_grad_()
        y, want = fastnn.trainable_layer_norm(leaf, (C,), w, b), fastnn.trainable_layer_norm(some, (C,), w, b)
        assert torch.equal(y[part], want)
        dy = torch.zeros_like(y)
        dy[part] = torch.tensor([1.0, 3.0], dtype=BF16, device=device)
        (dx,), (want,) = torch.autograd.grad(y, leaf, dy), torch.autograd.grad(want, some, dy[part])
        assert torch.equal(dx[part], want)


# ------------------------------------------------------------------------------ the operators together

class Block(torch.nn.Module):
    """x + out(attention(LayerNorm(x))), two chains in one sequence, a distance slope per head."""

    def __init__(self, norm, attention, c=96, heads=4, kv_heads=2, dim=24):
        super().__init__()
        self.norm, self.attention, self.heads, self.kv_heads, self.dim = norm, attention, heads, kv_heads, dim
        self.qkv = torch.nn.Linear(c, (heads + 2 * kv_heads) * dim, bias=False)
        self.out = torch.nn.Linear(heads * dim, c, bias=False)
        self.slopes = torch.nn.Parameter(torch.linspace(0.02, 0.3, heads))

    def forward(self, x, **masks):
        B, n, _ = x.shape
        y = self.qkv(self.norm(x)).view(B, n, self.heads + 2 * self.kv_heads, self.dim).transpose(1, 2)
        q, k, v = y.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        o = self.attention(q, k, v, slopes=self.slopes, **masks)
        return x + self.out(o.transpose(1, 2).reshape(B, n, self.heads * self.dim))


def plain_attention(q, k, v, slopes, causal, documents, softcap):
    n, group = q.shape[2], q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = softcap * torch.tanh(q @ k.transpose(2, 3) * q.shape[-1] ** -0.5 / softcap)
    t = torch.arange(n)
    s = s - slopes[:, None, None] * (t[:, None] - t).abs()
    keep = (documents[:, :, None] == documents[:, None]) & (t[:, None] >= t)
    return torch.softmax(s.masked_fill(~keep[:, None], -math.inf), -1) @ v


def test_pre_norm_attention_block(device):
    from xfold_cpu_amd import fastnn
    torch.manual_seed(0)
    mine = Block(fastnn.LayerNorm(96), fastnn.sequence_attention)
    plain = Block(torch.nn.LayerNorm(96), plain_attention).double()
    plain.load_state_dict(mine.state_dict())
    mine.to(device).train()
    x = torch.randn(2, 90, 96)
    docs = (torch.arange(90) >= 33).int().expand(2, 90).contiguous()
    dy = torch.randn(2, 90, 96)
    leaf, leaf64 = x.to(device).requires_grad_(), x.double().requires_grad_()
    out = mine(leaf, causal=True, documents=docs.to(device), softcap=12.0)
    out64 = plain(leaf64, causal=True, documents=docs, softcap=12.0)
    out.backward(dy.to(device))
    out64.backward(dy.double())
    pairs = [("out", out, out64), ("dx", leaf.grad, leaf64.grad)]
    pairs += [(name, p.grad, dict(plain.named_parameters())[name].grad) for name, p in mine.named_parameters()]
    for name, got, want in pairs:
        err = float((got.detach().cpu().double() - want.detach()).norm() / want.detach().norm())
        print(f"[block] {name}: {err:.2e}", flush=True)
        # FP32 throughout: five products in a row over at most 180 terms, each 180 * 2^-24 = 1e-5 of its
        # absolute terms at most; errors add at random, but the norms of sums are smaller than their terms'.
        assert err <= 5e-5, (name, err)


def test_checkpointed_block(device):
    """Recomputed in the backward pass, with hooks on the saved tensors: the same bits."""
    from torch.utils.checkpoint import checkpoint
    from xfold_cpu_amd import fastnn
    torch.manual_seed(1)
    block = Block(fastnn.LayerNorm(96), fastnn.sequence_attention).to(device).train()
    x = torch.randn(2, 70, 96, device=device, requires_grad=True)
    leaves = [x, *block.parameters()]
    call = lambda t: block(t, causal=True, softcap=12.0)                                              # noqa: E731
    want = torch.autograd.grad(call(x).square().sum(), leaves)
    got = torch.autograd.grad(checkpoint(call, x, use_reentrant=False).square().sum(), leaves)
    with torch.autograd.graph.save_on_cpu():
        moved = torch.autograd.grad(call(x).square().sum(), leaves)
    for w, g, m in zip(want, got, moved):
        assert torch.equal(w, g) and torch.equal(w, m)


def test_gradients_of_two_graphs_and_of_some_inputs(device):
    """One graph differentiated twice, and for one input at a time: what is not asked for is left out."""
    x, w, b, dy = data(device, BF16, F32, 300, 96)
    want = run(x, w, b, dy)
    from xfold_cpu_amd import fastnn
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = fastnn.trainable_layer_norm(leaves[0], (96,), *leaves[1:])
    for _ in range(2):
        for name, leaf in zip(("dx", "dw", "db"), leaves):
            (g,) = torch.autograd.grad(y, leaf, dy, retain_graph=True)
            assert torch.equal(g, want[name]), name
    y = fastnn.trainable_layer_norm(leaves[0], (96,), None, leaves[2])          # no weight: the bias keeps its place
    gx, gb = torch.autograd.grad(y, (leaves[0], leaves[2]), dy)
    assert torch.equal(gb, want["db"]) and gx.shape == x.shape
    (twice,) = torch.autograd.grad(fastnn.trainable_layer_norm(leaves[0], (96,)).sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        twice.sum().backward()
