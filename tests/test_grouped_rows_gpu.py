"""Operators over rows grouped by an index, on the GPU: the grouping itself, group norm with an activation, embedding
lookup with its gradient, rows sorted by expert and back.  Every operator is compared with its definition in 64 bits.

Tolerances: a result rounded to its type is off by at most eps / 2 of its value; `extra` bounds what the 32-bit
arithmetic before that rounding loses: 2^-24 of the terms' absolute values for each rounding on the longest chain."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def close(got, want, extra):
    """|got - want| <= half a unit of got's type + extra, elementwise; `want` and `extra` in 64 bits."""
    assert got.shape == want.shape
    if got.numel() == 0:
        return
    half = torch.finfo(got.dtype).eps / 2
    floor = 2.0 ** -25 if got.dtype == torch.float16 else 0.0        # half of fp16's smallest step
    bound = half * (want.abs() + extra) + extra + floor
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound.clamp(min=1e-300)).max()):.3g} bounds"


def unaligned(t):
    """The same values one element behind an aligned address."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.reshape(-1)
    return flat[1:].view(t.shape)


# ------------------------------------------------------------------------------------------------ grouping
@pytest.mark.parametrize("n", [0, 1, 33, 4096, 4097, 70001])
@pytest.mark.parametrize("groups", [1, 2, 255, 256, 300, 65535, 65536, 20_000_000])
def test_group_rows_is_a_stable_sort(n, groups):
    from torchsparse_b200.nn import functional as F

    g = torch.Generator().manual_seed(n + groups)
    keys = torch.randint(-2, min(groups, 1 << 30) + 2, (n,), generator=g)
    for dtype in (torch.int32, torch.int64):
        order, inverse, offsets = F.expert_sort(keys.to(dtype).cuda(), groups)
        inverse = inverse.view(-1)
        for a, b in zip((order, offsets), F.group_rows(keys.to(dtype).cuda(), groups)):
            assert torch.equal(a, b)
        folded = torch.where((keys < 0) | (keys >= groups), groups, keys)
        want = torch.sort(folded, stable=True)
        assert torch.equal(order.cpu().long(), want.indices)
        assert torch.equal(inverse.cpu().long()[want.indices], torch.arange(n))
        assert torch.equal(offsets.cpu().long(), torch.searchsorted(want.values, torch.arange(groups + 1)))


def test_group_rows_of_strided_extreme_and_constant_keys():
    from torchsparse_b200.nn import functional as F

    coords = torch.randint(0, 5, (9001, 4), generator=torch.Generator().manual_seed(1)).int().cuda()
    got = F.group_rows(coords[:, 0], 5)
    assert torch.equal(got.order.long(), torch.sort(coords[:, 0], stable=True).indices)
    same = F.group_rows(torch.full((9001,), 3, device="cuda"), 4)
    assert torch.equal(same.order, torch.arange(9001, device="cuda", dtype=torch.int32))
    assert same.offsets.tolist() == [0, 0, 0, 0, 9001]
    far = torch.tensor([2 ** 62, -2 ** 62, 2 ** 32, 2 ** 32 + 1, 1, -2 ** 32 + 1, 0], device="cuda")
    got = F.group_rows(far, 2)                                 # keys whose low 32 bits would be valid
    assert got.offsets.tolist() == [0, 1, 2] and got.order.tolist() == [6, 4, 0, 1, 2, 3, 5]
    one = F.group_rows(torch.zeros(1, dtype=torch.int32, device="cuda").expand(5000), 1)      # stride 0
    assert one.offsets.tolist() == [0, 5000]


# ------------------------------------------------------------------------------------------------ group norm
def norm_in_64_bits(x, cuts, order, groups, w, b, eps, act, slope, dy):
    """(y, dx, dw, db) and the sizes of the terms that the bounds need."""
    x, dy = x.double(), dy.double()
    n, c = x.shape
    w = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if b is None else b.double()
    y, dx, hat, z_all = (torch.zeros_like(x) for _ in range(4))
    dz_all, scale = torch.zeros_like(x), torch.zeros_like(x)
    term, mean_of, var_err = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    for lo, hi in zip(cuts, cuts[1:]):
        if hi <= lo:
            continue
        rows = torch.arange(lo, hi, device=x.device) if order is None else order[lo:hi].long()
        v = x[rows].view(hi - lo, groups, -1)
        mean = v.mean(dim=(0, 2), keepdim=True)
        var = ((v - mean) ** 2).mean(dim=(0, 2), keepdim=True)
        rstd = (var + eps).rsqrt()
        h = (v - mean) * rstd
        z = h.reshape(hi - lo, c) * w + b
        if act == "relu":
            a, da = z.clamp(min=0), (z > 0).double()
        elif act == "leaky_relu":
            a, da = torch.where(z > 0, z, z * slope), torch.where(z > 0, 1.0, slope).double()
        elif act == "silu":
            p = torch.sigmoid(z)
            a, da = z * p, p * (1 + z * (1 - p))
        else:
            a, da = z, torch.ones_like(z)
        dz = dy[rows] * da
        g = (dz * w).view_as(v)
        d = rstd * (g - g.mean(dim=(0, 2), keepdim=True) - h * (g * h).mean(dim=(0, 2), keepdim=True))
        y[rows], dx[rows], hat[rows], z_all[rows], dz_all[rows] = a, d.reshape(hi - lo, c), h.reshape(hi - lo, c), z, dz
        size = v.abs().amax(dim=(0, 2), keepdim=True) * rstd        # how far cancellation can magnify a rounding
        scale[rows] = size.expand_as(v).reshape(hi - lo, c)
        most = rstd * (g.abs() + g.abs().mean(dim=(0, 2), keepdim=True) + h.abs() * (g * h).abs().mean(dim=(0, 2), keepdim=True)
                       + g.abs().amax(dim=(0, 2), keepdim=True) * (1 + h.abs().amax(dim=(0, 2), keepdim=True) ** 2))
        term[rows] = most.reshape(hi - lo, c)
    return {"y": y, "dx": dx, "dw": (dz_all * hat).sum(0), "db": dz_all.sum(0), "hat": hat, "z": z_all, "dz": dz_all, "scale": scale,
            "term": term, "w": w, "b": b, "dy": dy}


def check_norm(x, cuts, groups, w, b, act=None, slope=0.01, order=None, eps=1e-5, seed=0):
    from torchsparse_b200.nn import functional as F

    g = torch.Generator(device="cuda").manual_seed(seed)
    dy = torch.randn(x.shape, generator=g, device="cuda").to(x.dtype)
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    want = norm_in_64_bits(x, cuts, order, groups, w, b, eps, act, slope, dy)
    if act in ("relu", "leaky_relu"):      # no value at the kink, where a rounding decides between two gradients
        for _ in range(8):
            near = (want["z"].abs() < 2e-3) & (want["scale"] > 0)
            if not bool(near.any()):
                break
            x = torch.where(near, x + 0.25, x)
            want = norm_in_64_bits(x, cuts, order, groups, w, b, eps, act, slope, dy)
        assert not bool(near.any())
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = F.group_norm(leaves[0], offsets, groups, leaves[1], leaves[2], eps, act, slope, order)
    assert torch.equal(y, F.group_norm(x, offsets, groups, w, b, eps, act, slope, order))      # without a graph too
    # 32 roundings of the statistics and the affine step, each magnified by |x| / sigma at most; act' is at most 1.1
    z_off = 32 * U * ((want["scale"] + want["hat"].abs() + 1) * want["w"].abs() + want["b"].abs())
    close(y, want["y"], 1.1 * z_off)
    present = [t for t in leaves if t is not None]
    got = dict(zip([k for k, t in zip(("dx", "dw", "db"), leaves) if t is not None], torch.autograd.grad(y, present, dy)))
    # dz: act'' is at most 1 / 2; sums: 256 roundings on the longest chain
    dz_off = want["dy"].abs() * (z_off * 0.5 + 8 * U)
    rel = 64 * U * (1 + want["scale"])
    close(got["dx"], want["dx"], want["term"] * (rel + 256 * U) + (want["term"].amax() if n_rows(want) else 0) * z_off.amax())
    if w is not None:
        each = (want["dz"] * want["hat"]).abs() * (rel + 256 * U) + dz_off * want["hat"].abs() + want["dz"].abs() * rel
        close(got["dw"], want["dw"], each.sum(0))
    if b is not None:
        close(got["db"], want["db"], (want["dz"].abs() * 256 * U + dz_off).sum(0))
    return y.detach(), got


def n_rows(want):
    return want["y"].shape[0]


def features(n, c, dtype, seed=0, offset=0.5, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, c, generator=g, device="cuda") * spread + offset * torch.rand(c, generator=g, device="cuda")).to(dtype)


def affine(c, dtype=torch.float32, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return ((torch.rand(c, generator=g, device="cuda") + 0.5).to(dtype),
            (torch.randn(c, generator=g, device="cuda") * 0.3).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c,groups", [(1, 1), (16, 4), (96, 8), (64, 64), (99, 9), (100, 5), (256, 32), (98, 7), (2056, 2)])
@pytest.mark.parametrize("cuts", [[0, 1], [0, 700], [0, 3, 3, 250, 251, 251, 900]])
def test_group_norm_forward_and_gradient(dtype, c, groups, cuts):
    if c // groups * min(q - p for p, q in zip(cuts, cuts[1:]) if q > p) == 1:
        pytest.skip("a group of one value: test_group_norm_of_a_single_value")
    w, b = affine(c)
    check_norm(features(cuts[-1], c, dtype), cuts, groups, w, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c,groups", [(1, 1), (16, 4), (24, 12), (96, 8), (64, 64), (99, 9), (98, 7), (256, 32), (2056, 257)])
@pytest.mark.parametrize("cuts", [[0, 9001], [0, 4500, 4501, 13001]])
def test_group_norm_of_long_samples(dtype, c, groups, cuts):
    """Samples beyond what one block holds: the rows in chunks, their sums joined."""
    w, b = affine(c)
    check_norm(features(cuts[-1], c, dtype), cuts, groups, w, b, "silu")


@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_of_one_long_sample_among_short_ones(dtype):
    """Many samples that a block holds and one that it has to read again."""
    cuts = [0, 30, 60, 9000] + [9000 + 40 * k for k in range(1, 26)]
    w, b = affine(16)
    check_norm(features(10000, 16, dtype), cuts, 2, w, b, "silu")


@pytest.mark.parametrize("act", ["relu", "leaky_relu", "silu", None])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("params", ["float", "same", "none", "weight", "bias"])
def test_group_norm_activations_and_parameters(act, dtype, params):
    c = 48
    w, b = affine(c, dtype if params == "same" else torch.float32)
    if params in ("none", "bias"):
        w = None
    if params in ("none", "weight"):
        b = None
    check_norm(features(531, c, dtype), [0, 200, 531], 6, w, b, act, 0.2)


@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_of_interleaved_rows_and_rows_of_no_sample(dtype):
    from torchsparse_b200.nn import functional as F

    n, c, samples = 20011, 32, 5
    g = torch.Generator(device="cuda").manual_seed(3)
    batch = torch.randint(-1, samples + 1, (n,), generator=g, device="cuda")
    rows = F.group_rows(batch, samples)
    w, b = affine(c)
    x = features(n, c, dtype)
    few = F.group_rows(batch[:900], samples)
    check_norm(x[:900], few.offsets.tolist(), 8, w, b, "silu", order=few.order)
    y, got = check_norm(x, rows.offsets.tolist(), 8, w, b, "silu", order=rows.order)
    outside = (batch < 0) | (batch >= samples)
    assert bool((y[outside] == 0).all()) and bool((got["dx"][outside] == 0).all())
    # rows before the first sample and behind the last
    y, got = check_norm(x, [100, 5000, 15000], 8, w, b, "silu")
    assert bool((y[:100] == 0).all()) and bool((y[15000:] == 0).all()) and bool((got["dx"][15000:] == 0).all())


def test_group_norm_of_many_small_samples_and_of_a_far_mean():
    cuts = list(range(0, 6001, 2))
    w, b = affine(24)
    check_norm(features(6000, 24, torch.float32), cuts, 3, w, b, "silu")
    check_norm(features(30000, 24, torch.float32, offset=1000.0, spread=0.1), [0, 30000], 24, w, b)
    x = features(5000, 24, torch.float32)
    x[0] = 3e4                                                   # a first row far from all others
    check_norm(x, [0, 5000], 3, w, b)


def test_group_norm_unaligned_transposed_and_constant_features():
    w, b = affine(64)
    for dtype in TYPES:
        x = features(257, 64, dtype)
        check_norm(unaligned(x), [0, 257], 8, unaligned(w), unaligned(b), "silu")
        check_norm(x.t().contiguous().t(), [0, 257], 8, w, b)
    flat = torch.full((300, 64), 2.0, device="cuda")
    y, _ = check_norm(flat, [0, 300], 8, w, b)
    assert torch.equal(y, b.expand(300, 64))


def test_group_norm_of_a_single_value_and_of_nothing():
    from torchsparse_b200.nn import functional as F

    w, b = affine(7)
    x = torch.randn(1, 7, device="cuda")
    y = F.group_norm(x, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 7, w, b)
    assert torch.equal(y, b[None])
    for n, cuts in ((0, [0]), (0, [0, 0, 0]), (5, [0]), (5, [0, 0])):
        x = torch.randn(n, 7, device="cuda", requires_grad=True)
        ws, bs = w.clone().requires_grad_(), b.clone().requires_grad_()
        y = F.group_norm(x, torch.tensor(cuts, dtype=torch.int32, device="cuda"), 7, ws, bs, activation="relu")
        assert y.shape == (n, 7) and bool((y == 0).all())
        for grad in torch.autograd.grad(y.sum(), (x, ws, bs)):
            assert bool((grad == 0).all())


def test_group_norm_keeps_nan_and_infinity_in_their_sample_and_group():
    from torchsparse_b200.nn import functional as F

    x = features(300, 16, torch.float32)
    clean = F.group_norm(x, torch.tensor([0, 100, 200, 300], dtype=torch.int32, device="cuda"), 4, activation="relu")
    x[150, 5], x[250, 0] = float("nan"), float("inf")
    y = F.group_norm(x, torch.tensor([0, 100, 200, 300], dtype=torch.int32, device="cuda"), 4, activation="relu")
    touched = torch.zeros_like(x, dtype=torch.bool)
    touched[100:200, 4:8] = touched[200:300, 0:4] = True
    assert bool(y[touched].isnan().all()) and torch.equal(y[~touched], clean[~touched])


def test_group_norm_gradient_against_differences():
    from torchsparse_b200.nn import functional as F

    cuts = torch.tensor([0, 40, 97], dtype=torch.int32, device="cuda")
    x = features(97, 12, torch.float32)
    w, b = affine(12)
    g = torch.Generator(device="cuda").manual_seed(5)
    dy, dirs = torch.randn(97, 12, generator=g, device="cuda"), [torch.randn(t.shape, generator=g, device="cuda") for t in (x, w, b)]
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(F.group_norm(leaves[0], cuts, 3, leaves[1], leaves[2], activation="silu"), leaves, dy)
    h = 2.0 ** -7
    for k in range(3):
        up, down = ([t + s * h * dirs[k] if i == k else t for i, t in enumerate((x, w, b))] for s in (1, -1))
        slope = ((F.group_norm(up[0], cuts, 3, up[1], up[2], activation="silu").double()
                  - F.group_norm(down[0], cuts, 3, down[1], down[2], activation="silu").double()) * dy).sum() / (2 * h)
        want = (grads[k].double() * dirs[k]).sum()
        # third derivatives of order 1 per unit of dy and direction: h^2 / 6 * sum |dy| |dir|^3 is below 1e-4 * sum |dy| * 6
        assert abs(float(slope - want)) < 6e-4 * float(dy.abs().sum())


@pytest.mark.parametrize("ordered", [False, True])
@pytest.mark.parametrize("act", [None, "silu", "leaky_relu"])
def test_group_norm_gradient_differentiated_again(act, ordered):
    """A gradient penalty: the first derivative under create_graph equals the kernels', the second the definition's in 64
    bits.  1e-4 of the largest value is some 800 roundings of fp32; the chain of two derivatives has below 100."""
    from torchsparse_b200.nn import functional as F

    cuts, n, c = [5, 40, 40, 97], 100, 12
    g = torch.Generator(device="cuda").manual_seed(6)
    order = torch.randperm(n, generator=g, device="cuda").int() if ordered else None
    x, dy, (w, b) = features(n, c, torch.float32), torch.randn(n, c, generator=g, device="cuda"), affine(c)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, dy)]
    y = F.group_norm(leaves[0], torch.tensor(cuts, dtype=torch.int32, device="cuda"), 3, leaves[1], leaves[2], 1e-5, act, 0.1, order)
    first = torch.autograd.grad(y, leaves[:3], leaves[3], create_graph=True)
    plain = torch.autograd.grad(y, leaves[:3], leaves[3], retain_graph=True)
    wide = [t.double().requires_grad_() for t in (x, w, b, dy)]
    parts = torch.zeros(n, c, dtype=torch.float64, device="cuda")
    for lo, hi in zip(cuts, cuts[1:]):
        rows = torch.arange(lo, hi, device="cuda") if order is None else order[lo:hi].long()
        if hi > lo:
            v = torch.nn.functional.group_norm(wide[0][rows].t()[None], 3, wide[1], wide[2], 1e-5)[0].t()
            v = {None: lambda t: t, "silu": torch.nn.functional.silu,
                 "leaky_relu": lambda t: torch.nn.functional.leaky_relu(t, 0.1)}[act](v)
            parts = parts.index_copy(0, rows, v)
    want = torch.autograd.grad(parts, wide[:3], wide[3], create_graph=True)
    for a, k, e in zip(first, plain, want):
        assert float((a - k).detach().abs().max()) < 1e-4 * float(e.detach().abs().max())
        assert float((a - e).detach().abs().max()) < 1e-4 * float(e.detach().abs().max())
    # without an activation the bias has no part in the first derivative: zeros
    second = torch.autograd.grad(sum(t.square().sum() for t in first), leaves, materialize_grads=True)
    for a, e in zip(second, torch.autograd.grad(sum(t.square().sum() for t in want), wide, materialize_grads=True)):
        assert float((a - e).abs().max()) < 1e-4 * max(float(e.abs().max()), 1.0)


def test_group_norm_beyond_32_bit_offsets():
    from torchsparse_b200.nn import functional as F

    n, c = 2_200_000, 1024                                        # 2.25e9 values
    x = torch.empty(n, c, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    cuts = [0, 1_000_000, n]
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    y = F.group_norm(x, offsets, 8)
    last = x[1_000_000:, 896:].double()
    want = (last - last.mean()) / (last.var(correction=0) + 1e-5).sqrt()
    close(y[1_000_000:, 896:], want, (want.abs() + 5) * 64 * U)


def test_group_norm_module_matches_torch_and_takes_rows():
    import torchsparse_b200 as ts
    from torchsparse_b200 import nn as spnn
    from torchsparse_b200.nn import functional as F

    g = torch.Generator().manual_seed(2)
    coords = torch.randint(0, 50, (3000, 4), generator=g).int()
    coords[:, 0] = torch.randint(0, 4, (3000,), generator=g)      # interleaved samples
    x = ts.SparseTensor(torch.randn(3000, 48, generator=g).cuda(), coords.cuda())
    for act, fn in ((None, lambda t: t), ("relu", torch.relu), ("silu", torch.nn.functional.silu)):
        m = spnn.GroupNorm(8, 48, activation=act).cuda()
        with torch.no_grad():
            m.weight.uniform_(0.5, 1.5)
            m.bias.uniform_(-0.5, 0.5)
        y = m(x)
        assert y.coords is x.coords and y._caches is x._caches and y.stride == x.stride
        assert torch.equal(m(x, F.sample_rows(x)).feats, y.feats)
        for coords_too in (x.coords.cpu(), x.coords.long(), x.coords.short()):      # wherever and whatever the coordinates are
            assert torch.equal(m(ts.SparseTensor(x.feats, coords_too)).feats, y.feats)
        for s in range(4):
            rows = x.coords[:, 0] == s
            want = fn(torch.nn.functional.group_norm(x.feats[rows].t()[None].double(), 8, m.weight.double(), m.bias.double(), m.eps))
            close(y.feats[rows].detach(), want[0].t().detach(), 64 * U * (want[0].t().detach().abs() + 2))
    plain = spnn.GroupNorm(8, 48, activation="silu").cuda().double()      # a dtype of torch's alone
    xd = ts.SparseTensor(x.feats.double(), x.coords)
    same = spnn.GroupNorm(8, 48, activation="silu").cuda()(x).feats
    close(same.detach(), plain(xd).feats.detach(), torch.full_like(xd.feats, 400 * U))


# ------------------------------------------------------------------------------------------------ embedding
def check_embedding(tokens, table, scale, padding=None, seed=0):
    from torchsparse_b200.nn import functional as F

    v, c = table.shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    dy = torch.randn(*tokens.shape, c, generator=g, device="cuda").to(table.dtype)
    leaf = table.detach().requires_grad_()
    y = F.embedding(tokens, leaf, scale, padding)
    flat = tokens.reshape(-1).long()
    inside = (flat >= 0) & (flat < v)
    scale32 = float(torch.tensor(scale, dtype=torch.float32))
    want = torch.zeros(flat.numel(), c, dtype=torch.float64, device="cuda")
    want[inside] = table.double()[flat[inside]] * scale32
    close(y.reshape(-1, c), want, want.abs() * U)
    assert torch.equal(F.embedding(tokens, table, scale, padding), y)
    (dt,) = torch.autograd.grad(y, leaf, dy)
    if padding is not None:
        inside = inside & (flat != padding % v)
    grad = dy.reshape(-1, c).double()[inside] * scale32
    total = torch.zeros(v, c, dtype=torch.float64, device="cuda").index_add_(0, flat[inside], grad)
    size = torch.zeros(v, c, dtype=torch.float64, device="cuda").index_add_(0, flat[inside], grad.abs())
    often = torch.bincount(flat[inside], minlength=v).double().clamp(max=512)[:, None]      # roundings of the longest chain
    close(dt, total, size * (often + 2) * U)
    return dt


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 300, 9000])
@pytest.mark.parametrize("v,c", [(1, 8), (3, 64), (301, 33), (5000, 100), (70000, 16), (257, 2500)])
def test_embedding_and_its_gradient(dtype, n, v, c):
    g = torch.Generator(device="cuda").manual_seed(n + v)
    tokens = torch.randint(-1, v + 1, (n,), generator=g, device="cuda")
    check_embedding(tokens, torch.randn(v, c, generator=g, device="cuda").to(dtype), 1.5, padding=v - 1 if v > 1 else None)


@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_of_one_token_and_of_runs_that_cross_every_border(dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randn(6, 72, generator=g, device="cuda").to(dtype)
    check_embedding(torch.full((20000,), 4, device="cuda", dtype=torch.int32), table, 0.01)
    for n in (63, 64, 65, 511, 4097):
        check_embedding((torch.arange(n, device="cuda") * 5 // n), table, 1.0)
    check_embedding(torch.full((50,), -1, device="cuda"), table, 1.0)
    check_embedding(torch.randint(0, 6, (3, 5, 7), generator=g, device="cuda"), table, 1.0, padding=-2)
    check_embedding(torch.zeros(0, dtype=torch.int64, device="cuda"), table, 1.0)
    check_embedding(torch.zeros(2, 0, dtype=torch.int64, device="cuda"), table, 1.0)


def test_embedding_unaligned_strided_and_empty_tables():
    from torchsparse_b200.nn import functional as F

    g = torch.Generator(device="cuda").manual_seed(4)
    for dtype in TYPES:
        table = torch.randn(50, 24, generator=g, device="cuda").to(dtype)
        tokens = torch.randint(0, 50, (999, 2), generator=g, device="cuda")
        check_embedding(tokens[:, 1], unaligned(table), 2.0)
        for c in (1, 2, 3, 5, 7, 12):                            # rows shorter than a vector of the result
            narrow = torch.randn(50, c, generator=g, device="cuda").to(dtype)
            for n in (1, 2, 3, 999):
                check_embedding(tokens[:n, 1] - 3, narrow, 2.0)
        check_embedding(tokens[:, 0], table.t().contiguous().t(), 2.0)
    empty = torch.empty(0, 24, device="cuda", requires_grad=True)
    y = F.embedding(torch.zeros(5, dtype=torch.int64, device="cuda"), empty)
    assert bool((y == 0).all()) and torch.autograd.grad(y.sum(), empty)[0].shape == (0, 24)


def test_embedding_beyond_32_bit_offsets():
    from torchsparse_b200.nn import functional as F

    n, c, v = 1_100_000, 2048, 3
    table = torch.arange(v, device="cuda", dtype=torch.float16)[:, None].expand(v, c).contiguous()
    tokens = torch.arange(n, device="cuda") % v
    y = F.embedding(tokens, table.requires_grad_())
    assert bool((y[-3:, 0] == tokens[-3:]).all()) and bool((y[:, -1] == tokens).all())
    dy = torch.full_like(y, 2.0 ** -14)
    (grad,) = torch.autograd.grad(y, table, dy)
    want = torch.bincount(tokens).double() * 2.0 ** -14             # powers of two: every partial sum is exact
    assert torch.equal(grad.double(), want.half().double()[:, None].expand(v, c))
    far = F.embedding(torch.tensor([0, n, 1_099_999, 1_099_999, -1], device="cuda"), dy.requires_grad_())      # a table of 2.25e9
    assert bool((far[[0, 2, 3]] == 2.0 ** -14).all()) and bool((far[[1, 4]] == 0).all())
    (big,) = torch.autograd.grad(far.sum(), dy)
    assert bool((big[1_099_999] == 2).all()) and bool((big[0] == 1).all()) and int(big[:, 7].count_nonzero()) == 2


def test_embedding_module_on_a_sparse_tensor():
    import torchsparse_b200 as ts
    from torchsparse_b200 import nn as spnn

    labels = torch.randint(0, 20, (500, 1), generator=torch.Generator().manual_seed(1)).cuda()
    coords = torch.zeros(500, 4, dtype=torch.int32, device="cuda")
    m = spnn.Embedding(20, 32, padding_idx=0, scale=3.0).cuda()
    y = m(ts.SparseTensor(labels, coords))
    assert y.coords is coords and torch.equal(y.feats, (m.weight * 3.0)[labels[:, 0]])
    y.feats.sum().backward()
    assert bool((m.weight.grad[0] == 0).all())
    assert torch.equal(m.weight.grad[1:, 0], 3.0 * torch.bincount(labels[:, 0], minlength=20)[1:].float())
    assert torch.equal(m(labels[:, 0]), y.feats)


# ------------------------------------------------------------------------------------------------ experts
def check_experts(choice, e, c, dtype, w_dtype=torch.float32, seed=0, shift=lambda t: t):
    from torchsparse_b200.nn import functional as F

    n, k = choice.shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda")      # noqa: E731
    x, ys, dxs, dout = (shift(make(r, c).to(dtype)) for r in (n, n * k, n * k, n))
    w = make(n, k).to(w_dtype)
    rows = F.expert_sort(choice, e)
    used = (choice >= 0) & (choice < e)
    key = torch.where(used, choice, e).reshape(-1)
    want = torch.sort(key, stable=True)
    assert torch.equal(rows.order.long(), want.indices) and rows.inverse.shape == (n, k)
    assert torch.equal(rows.inverse.reshape(-1).long()[want.indices], torch.arange(n * k, device="cuda"))
    kept = int(used.sum())
    assert int(rows.offsets[-1]) == kept and rows.offsets.shape == (e + 1,)
    xl, yl, wl = (t.detach().requires_grad_() for t in (x, ys, w))
    xs, out = F.expert_dispatch(xl, rows), F.expert_combine(yl, wl, rows)
    assert torch.equal(xs[:kept], x[want.indices[:kept] // k]) and bool((xs[kept:] == 0).all())
    mine = ys.double()[rows.inverse.long().reshape(-1)].view(n, k, c) * used[..., None]
    w64 = w.double() * used
    close(out, (mine * w64[..., None]).sum(1), (mine * w64[..., None]).abs().sum(1) * (k + 1) * U)
    dx, dys, dw = torch.autograd.grad((xs, out), (xl, yl, wl), (dxs, dout))
    back = dxs.double()[rows.inverse.long().reshape(-1)].view(n, k, c) * used[..., None]
    close(dx, back.sum(1), back.abs().sum(1) * (k + 1) * U)
    each = (w64[..., None] * dout.double()[:, None]).view(n * k, c)
    placed = torch.zeros_like(each)
    placed[rows.inverse.long().reshape(-1)] = each
    close(dys, placed, placed.abs() * U)
    products = dout.double()[:, None] * mine
    close(dw, products.sum(2), products.abs().sum(2) * (c / 32 + 16) * U)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,e", [(1, 1, 1), (1, 8, 256), (16, 2, 8), (1500, 6, 130), (4097, 1, 3), (700, 3, 70000), (90, 13, 40)])
@pytest.mark.parametrize("c", [8, 99, 200, 1024, 2600])
def test_experts_there_and_back(dtype, n, k, e, c):
    choice = torch.randint(-1, e + 1, (n, k), generator=torch.Generator(device="cuda").manual_seed(n + e), device="cuda")
    check_experts(choice, e, c, dtype)


def test_experts_with_16_bit_weights_odd_addresses_repeats_and_drops():
    g = torch.Generator(device="cuda").manual_seed(0)
    choice = torch.randint(0, 4, (333, 2), generator=g, device="cuda")
    for w_dtype in TYPES:
        check_experts(choice.int(), 4, 40, torch.bfloat16, w_dtype)
    for dtype in TYPES:
        check_experts(choice, 4, 40, dtype, shift=unaligned)
        check_experts(torch.full((50, 3), 2, device="cuda"), 4, 40, dtype)          # one expert, thrice for each row
        check_experts(torch.full((50, 3), -1, device="cuda"), 4, 40, dtype)         # every choice dropped
    check_experts(torch.randint(0, 4, (2, 333), generator=g, device="cuda").t(), 4, 40, torch.float32)      # a transposed view


def test_dropped_choices_hide_nan_of_their_rows():
    from torchsparse_b200.nn import functional as F

    rows = F.expert_sort(torch.tensor([[0, -1], [1, 2]], device="cuda"), 2)
    ys = torch.ones(4, 8, device="cuda")
    ys[2:] = float("nan")                                         # what stands behind the last expert
    ys.requires_grad_()
    w = torch.tensor([[2.0, float("inf")], [3.0, float("nan")]], device="cuda", requires_grad=True)
    out = F.expert_combine(ys, w, rows)
    assert torch.equal(out, torch.tensor([[2.0], [3.0]], device="cuda").expand(2, 8))
    dys, dw = torch.autograd.grad(out.sum(), (ys, w))
    assert bool((dys[2:] == 0).all()) and dw.tolist() == [[8.0, 0.0], [8.0, 0.0]]


def test_what_belongs_to_nothing_may_hold_anything():
    """NaN in rows of no sample, of no token and of no expert, and in their gradients, reaches nothing else."""
    from torchsparse_b200.nn import functional as F

    for n in (600, 20000):                                        # one block per sample and group, and chunks of rows
        off = torch.tensor([n // 6, n // 2, n - n // 5], dtype=torch.int32, device="cuda")
        outside = torch.ones(n, dtype=torch.bool, device="cuda")
        outside[n // 6:n - n // 5] = False
        for order in (None, torch.randperm(n, device="cuda").int()):
            x, dy = features(n, 24, torch.float32, 1), features(n, 24, torch.float32, 2)
            where = outside if order is None else torch.zeros_like(outside).index_put_((order.long(),), outside)
            w, b = (t.requires_grad_() for t in affine(24))
            results = []
            for fill in (0.0, float("nan")):
                xs = torch.where(where[:, None], fill, x).requires_grad_()
                y = F.group_norm(xs, off, 3, w, b, activation="silu", order=order)
                grads = torch.autograd.grad(y, (xs, w, b), torch.where(where[:, None], fill, dy))
                results.append([y.detach(), *grads])
            assert bool((results[1][0][where] == 0).all()) and bool((results[1][1][where] == 0).all())
            for a, c in zip(*results):
                assert torch.equal(a, c)
    table = torch.randn(5, 24, device="cuda", requires_grad=True)
    tokens = torch.tensor([0, -1, 3, 2, 7, 2], device="cuda")
    dy = torch.ones(6, 24, device="cuda")
    dy[[1, 3, 4, 5]] = float("nan")                               # no token, the padding, no token, the padding
    (dt,) = torch.autograd.grad(F.embedding(tokens, table, padding_idx=2), table, dy)
    assert dt[:, 0].tolist() == [1, 0, 0, 1, 0]
    rows = F.expert_sort(torch.tensor([[0, -1], [1, 2]], device="cuda"), 2)
    x = torch.randn(2, 24, device="cuda", requires_grad=True)
    dxs = torch.ones(4, 24, device="cuda")
    dxs[2:] = float("inf")                                        # behind the last expert
    assert bool((torch.autograd.grad(F.expert_dispatch(x, rows), x, dxs)[0] == 1).all())


def test_experts_of_no_rows():
    from torchsparse_b200.nn import functional as F

    rows = F.expert_sort(torch.zeros(0, 2, dtype=torch.int64, device="cuda"), 3)
    assert rows.offsets.tolist() == [0, 0, 0, 0]
    x, w = torch.zeros(0, 16, device="cuda", requires_grad=True), torch.zeros(0, 2, device="cuda", requires_grad=True)
    xs = F.expert_dispatch(x, rows)
    out = F.expert_combine(xs, w, rows)
    assert xs.shape == (0, 16) and out.shape == (0, 16)
    assert [t.shape for t in torch.autograd.grad(out.sum(), (x, w))] == [(0, 16), (0, 2)]


def test_expert_rows_beyond_32_bit_offsets():
    from torchsparse_b200.nn import functional as F

    n, k, c = 1_100_000, 2, 1024                                  # 2.25e9 sorted values
    choice = torch.stack([torch.arange(n, device="cuda") % 5, torch.arange(n, device="cuda") % 7], 1)
    rows = F.expert_sort(choice, 7)
    x = (torch.arange(n, device="cuda") % 1024).half()[:, None].expand(n, c).contiguous()
    xs = F.expert_dispatch(x, rows)
    assert torch.equal(xs[:, -1], x[:, 0][rows.order.long() // k])
    w = torch.full((n, k), 0.5, device="cuda")
    assert torch.equal(F.expert_combine(xs, w, rows), x)


# ------------------------------------------------------------------------------------------------ how they are used
def _training_step(state):
    """Labels -> vectors -> sparse convolution -> group norm with SiLU -> two of four experts -> loss; the gradients."""
    import torchsparse_b200 as ts
    from torchsparse_b200.nn import functional as F

    x = state["embed"](ts.SparseTensor(state["labels"], state["coords"]))
    x = state["norm"](state["conv"](x), state["samples"])
    rows = F.expert_sort(state["choice"], 4)
    xs = F.expert_dispatch(x.feats, rows)
    expert = torch.repeat_interleave(torch.arange(4, device="cuda"), (rows.offsets[1:] - rows.offsets[:-1]).long())
    ys = torch.einsum("nc,ncd->nd", xs, state["experts"][expert])
    out = F.expert_combine(ys, state["gate"], rows)
    return (out * state["dout"]).sum(), out


def _plain_step(state):
    """The same with torch's own operations around the convolution."""
    import torchsparse_b200 as ts

    x = torch.nn.functional.embedding(state["labels"], state["embed"].weight) * state["embed"].scale
    x = state["conv"](ts.SparseTensor(x, state["coords"])).feats
    parts = []
    for s in range(3):
        sample = x[state["coords"][:, 0] == s]
        parts.append(torch.nn.functional.group_norm(sample.t()[None], 4, state["norm"].weight, state["norm"].bias, 1e-5)[0].t())
    x = torch.nn.functional.silu(torch.cat(parts))
    out = 0
    for j in range(2):
        out = out + state["gate"][:, j:j + 1] * torch.einsum("nc,ncd->nd", x, state["experts"][state["choice"][:, j]])
    return (out * state["dout"]).sum(), out


def test_a_training_step_with_all_of_them_together():
    import torchsparse_b200 as ts
    from torchsparse_b200 import nn as spnn
    from torchsparse_b200.nn import functional as F

    from conftest import random_coords

    coords = torch.from_numpy(random_coords(np.random.default_rng(0), 400, (12, 12, 12), 3)).cuda()
    n, g = coords.shape[0], torch.Generator(device="cuda").manual_seed(7)
    torch.manual_seed(0)
    state = {"embed": spnn.Embedding(30, 16, scale=2.0).cuda(), "conv": spnn.Conv3d(16, 32, 3).cuda(),
             "norm": spnn.GroupNorm(4, 32, activation="silu").cuda(), "coords": coords,
             "labels": torch.randint(0, 30, (n,), generator=g, device="cuda"),
             "choice": torch.rand(n, 4, generator=g, device="cuda").topk(2, dim=1).indices,
             "gate": torch.rand(n, 2, generator=g, device="cuda").requires_grad_(),
             "experts": (torch.randn(4, 32, 32, generator=g, device="cuda") / 6).requires_grad_(),
             "dout": torch.randn(n, 32, generator=g, device="cuda")}
    state["samples"] = F.sample_rows(ts.SparseTensor(coords, coords))
    leaves = [state["embed"].weight, state["conv"].kernel, state["norm"].weight, state["norm"].bias, state["gate"], state["experts"]]
    loss, out = _training_step(state)
    plain_loss, plain_out = _plain_step(state)
    # two chains of the same fp32 operations in another order: 1e-5 is some 160 roundings of the largest value
    assert float((out - plain_out).detach().abs().max()) < 1e-5 * float(plain_out.detach().abs().max())
    for a, b in zip(torch.autograd.grad(loss, leaves), torch.autograd.grad(plain_loss, leaves)):
        assert float((a - b).norm()) < 1e-5 * float(b.norm())


def _everything(s):
    from torchsparse_b200.nn import functional as F

    x = s["x"].detach().requires_grad_()
    t = s["table"].detach().requires_grad_()
    w = s["w"].detach().requires_grad_()
    y = F.group_norm(x, s["offsets"], 4, s["gamma"], s["beta"], activation="silu") + F.embedding(s["tokens"], t, 2.0)
    rows = F.expert_sort(s["choice"], 9)
    out = F.expert_combine(F.expert_dispatch(y, rows), w, rows)
    return [out, rows.order, rows.offsets] + list(torch.autograd.grad(out, (x, t, w), s["dout"]))


def _inputs(seed, n=9001, c=40):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda")      # noqa: E731
    return {"x": make(n, c), "table": make(77, c), "w": make(n, 2), "gamma": make(c), "beta": make(c), "dout": make(n, c),
            "tokens": torch.randint(-1, 77, (n,), generator=g, device="cuda"),
            "choice": torch.randint(-1, 9, (n, 2), generator=g, device="cuda"),
            "offsets": torch.tensor([0, 1000 + seed, 1000 + seed, n], dtype=torch.int32, device="cuda")}


def test_the_same_call_gives_the_same_bits():
    s = _inputs(1)
    first = _everything(s)
    for _ in range(3):
        for a, b in zip(first, _everything(s)):
            assert torch.equal(a, b)


def test_two_captured_steps_replayed_on_new_inputs():
    """Two graphs with memory pools of their own, replayed on two streams; inputs and offsets change between replays."""
    graphs = []
    side = torch.cuda.Stream()
    for seed in (1, 2):
        s = _inputs(seed)
        with torch.cuda.stream(side):
            _everything(s)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = _everything(s)
        graphs.append((graph, s, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in (3, 5):
        for i, (graph, s, _) in enumerate(graphs):
            for k, v in _inputs(seed + i).items():
                s[k].copy_(v)
        torch.cuda.synchronize()
        for stream, (graph, _, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for i, (_, _, out) in enumerate(graphs):
            for a, b in zip(out, _everything(_inputs(seed + i))):
                assert torch.equal(a, b)


def test_calls_on_another_stream_wait_for_nothing_else():
    s = _inputs(4)
    want = _everything(s)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _everything(s)
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_calls_from_two_threads_at_once():
    """Each thread on a stream of its own, with inputs of its own."""
    import threading

    inputs, want, got = [_inputs(s, n=5000 + s) for s in (1, 2)], [], [None, None]
    want = [_everything(s) for s in inputs]
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[i] = _everything(inputs[i])
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for i in (0, 1):
        for a, b in zip(got[i], want[i]):
            assert torch.equal(a, b)


def test_an_input_changed_before_its_gradient_is_an_error():
    from torchsparse_b200.nn import functional as F

    off = torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    x, w = torch.randn(10, 8, device="cuda", requires_grad=True), torch.ones(10, 1, device="cuda", requires_grad=True)
    rows = F.expert_sort(torch.zeros(10, dtype=torch.int64, device="cuda"), 1)
    for make in (lambda: F.group_norm(x, off, 2), lambda: F.expert_combine(x, w, rows)):
        y = make()
        with torch.no_grad():
            x.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_offsets_and_positions_outside_their_range_are_cut_to_it():
    from torchsparse_b200.nn import functional as F

    x = torch.randn(10, 8, device="cuda")
    cut = F.group_norm(x, torch.tensor([0, 3, 10], dtype=torch.int32, device="cuda"), 2)
    assert torch.equal(F.group_norm(x, torch.tensor([-5, 3, 999], dtype=torch.int32, device="cuda"), 2), cut)
    big = torch.randn(9000, 8, device="cuda")
    cut = F.group_norm(big, torch.tensor([0, 3, 9000], dtype=torch.int32, device="cuda"), 2)
    assert torch.equal(F.group_norm(big, torch.tensor([-5, 3, 99999], dtype=torch.int32, device="cuda"), 2), cut)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    w = torch.ones(2, 1, device="cuda", requires_grad=True)
    for kept in (-3, 2, 10 ** 9):
        rows = F.ExpertRows(ints(0, 1), ints(-7, 10 ** 9)[:, None], ints(0, kept))
        ys = torch.ones(2, 8, device="cuda", requires_grad=True)
        out = F.expert_combine(ys, w, rows)
        assert bool((out == 0).all()) and bool((torch.autograd.grad(out.sum(), w)[0] == 0).all())
        F.expert_dispatch(ys, rows)


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    from torchsparse_b200 import nn as spnn
    from torchsparse_b200.nn import functional as F

    x, off = torch.randn(10, 8, device="cuda"), torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    w = torch.ones(8, device="cuda")
    for bad in (lambda: F.group_norm(x, off, 3), lambda: F.group_norm(x, off, 0), lambda: F.group_norm(x[None], off, 2),
                lambda: F.group_norm(x, off.long(), 2), lambda: F.group_norm(x, off[:0], 2), lambda: F.group_norm(x, off, 2, w[:7]),
                lambda: F.group_norm(x, off, 2, w, w.half()), lambda: F.group_norm(x, off, 2, activation="tanh"),
                lambda: F.group_norm(x, off, 2, order=off), lambda: F.group_rows(x[:, 0], 2), lambda: F.group_rows(off, 0),
                lambda: F.group_rows(off[None], 2), lambda: F.group_rows(off, 2 ** 31),
                lambda: F.embedding(x[:, 0], x), lambda: F.embedding(off, x[0]), lambda: F.embedding(off, x, padding_idx=10),
                lambda: F.embedding(off, x, padding_idx=-11), lambda: spnn.GroupNorm(2, 8, activation="gelu"),
                lambda: F.expert_sort(x, 2), lambda: F.expert_sort(off.view(1, 1, 2), 2), lambda: F.expert_sort(off[:, None][:, :0], 2),
                lambda: F.expert_dispatch(x[:9], F.expert_sort(torch.zeros(10, 2, dtype=torch.int64, device="cuda"), 2)),
                lambda: F.expert_combine(x, w[:, None], F.expert_sort(torch.zeros(10, dtype=torch.int64, device="cuda"), 2)),
                lambda: F.expert_combine(x, x[:, :1], F.expert_sort(torch.zeros(10, 2, dtype=torch.int64, device="cuda"), 2))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: F.group_norm(x.double(), off, 2), lambda: F.group_norm(x, off, 2, w.double()),
                lambda: F.embedding(off, x.double()), lambda: F.embedding(off, x.int()),
                lambda: F.expert_dispatch(x.double(), F.expert_sort(torch.zeros(10, dtype=torch.int64, device="cuda"), 2)),
                lambda: F.group_norm(x, off.cpu(), 2), lambda: F.embedding(off.cpu(), x)):
        with pytest.raises(RuntimeError):
            bad()
    # a second derivative is refused, not wrong
    leaf, gate = x.clone().requires_grad_(), torch.ones(10, 1, device="cuda", requires_grad=True)
    rows = F.expert_sort(torch.zeros(10, dtype=torch.int64, device="cuda"), 2)
    for make in (lambda: F.embedding(off, leaf), lambda: F.expert_dispatch(leaf, rows), lambda: F.expert_combine(leaf, gate, rows)):
        (g,) = torch.autograd.grad(make().square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once only"):
            g.sum().backward()
