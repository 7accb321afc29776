"""More of the operators over grouped rows on the GPU: cases that their first tests did not reach."""
import pytest
import torch

from test_grouped_rows_gpu import TYPES, U, affine, check_norm, features

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ group norm
@pytest.mark.parametrize("n", [900, 200_000])      # one block per sample and group, and chunks of rows
def test_an_empty_sample_without_eps_leaves_the_parameters_gradients(n):
    """An empty sample has no deviation: 1 / sqrt(0 + 0) must reach nothing."""
    from torchsparse_b200.nn import functional as F

    w, b = affine(24)
    x = features(n, 24, torch.float32)
    check_norm(x, [0, n // 3, n // 3, n], 3, w, b, "silu", eps=0.0)
    leaf = w.clone().requires_grad_()
    y = F.group_norm(x, ints([0, 0]), 3, leaf, b, eps=0.0)      # nothing but an empty sample
    assert bool((y == 0).all()) and bool((torch.autograd.grad(y.sum(), leaf)[0] == 0).all())


def test_a_group_of_one_value_is_refused_by_the_layer_wherever_it_runs():
    """As torch's layer does; F.group_norm, and the layer with rows that the caller grouped, give act(bias)."""
    import torchsparse_b200 as ts
    from torchsparse_b200 import nn as spnn
    from torchsparse_b200.nn import functional as F

    coords = torch.tensor([[0, 1, 1, 1], [0, 2, 1, 1], [1, 3, 1, 1]], dtype=torch.int32)
    x = torch.randn(3, 8, generator=torch.Generator().manual_seed(0))
    for device in ("cpu", "cuda"):
        m, s = spnn.GroupNorm(8, 8).to(device), ts.SparseTensor(x.to(device), coords.to(device))
        with pytest.raises(ValueError, match="more than 1 value"):
            m(s)
        m(ts.SparseTensor(s.feats[:2], s.coords[:2]))                     # two rows in each group
        spnn.GroupNorm(4, 8).to(device)(s)                                # two channels in each group
    y = m(s, F.sample_rows(s))
    assert torch.equal(y.feats[2], m.bias)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c,groups", [(16, 4), (24, 12), (96, 8), (64, 64), (99, 9), (98, 7), (256, 32), (2056, 257), (2057, 11)])
@pytest.mark.parametrize("ragged", [False, True])
def test_group_norm_of_long_interleaved_samples(dtype, c, groups, ragged):
    """The kernels that walk chunks of rows, through an order: groups inside a vector, across vectors and across tiles of
    columns, single 16-bit values, rows before the first sample and behind the last."""
    n = -(-(9 << 20) // (c * torch.finfo(dtype).bits // 8))      # one block serves a sample and group up to 8 MB in all
    cuts = [7, n // 3, n // 3 + 1, n // 3 + 1, n - 11] if ragged else [0, n]
    order = torch.randperm(n, generator=torch.Generator(device="cuda").manual_seed(n + c), device="cuda").int()
    w, b = affine(c)
    y, got = check_norm(features(n, c, dtype), cuts, groups, w, b, "silu", order=order)
    outside = torch.cat([order[:cuts[0]], order[cuts[-1]:]]).long()
    assert bool((y[outside] == 0).all()) and bool((got["dx"][outside] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,c,groups", [(10, 65536, 65536), (300, 4096, 4096), (700, 8192, 2), (65, 65535, 5)])
def test_group_norm_of_few_wide_rows(dtype, n, c, groups):
    w, b = affine(c)
    check_norm(features(n, c, dtype), [0, n // 2, n // 2, n], groups, w, b, "silu")


def test_group_norm_through_the_layer_on_long_interleaved_scans():
    import torchsparse_b200 as ts
    from torchsparse_b200 import nn as spnn

    n, c = 60_011, 96
    g = torch.Generator(device="cuda").manual_seed(2)
    coords = torch.randint(0, 50, (n, 4), generator=g, device="cuda").int()
    coords[:, 0] = torch.randint(0, 3, (n,), generator=g, device="cuda")
    m = spnn.GroupNorm(8, c, activation="silu").cuda()
    for dtype in TYPES:
        x = features(n, c, dtype)
        y = m(ts.SparseTensor(x, coords)).feats.detach()
        for s in range(3):
            rows = coords[:, 0] == s
            z = torch.nn.functional.group_norm(x[rows].double().t()[None], 8, m.weight.double(), m.bias.double(), m.eps)[0].t()
            want = torch.nn.functional.silu(z).detach()
            # 32 roundings of the statistics and the affine step, magnified by |x| / sigma, below 8 here; silu' is below 1.1
            bound = torch.finfo(dtype).eps / 2 * want.abs() + 1.1 * 32 * U * (8 + want.abs()) + 2.0 ** -25
            assert bool(((y[rows].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("n", [900, 100_000])      # one block per sample and group, and chunks of rows
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("far", [0.5, 30.0, 1000.0])
def test_group_norm_gradient_of_far_means_value_by_value(n, act, far):
    """dx within what its own value may be off: no share of the largest term or of the largest error elsewhere.

    z: x - mean is off by 2 roundings of |x| (the mean's and its own), rstd by 32 roundings and by what that does to the
    variance.  dz by |dy| act'' dz + 8 roundings, act'' being at most 1 / 2.  The means of g and g * xhat by the mean of
    their terms' errors and 128 roundings of their sizes."""
    from torchsparse_b200.nn import functional as F
    from test_grouped_rows_gpu import norm_in_64_bits

    c, groups, cuts = 24, 3, [0, n // 3, n]
    w, b = affine(c)
    x = features(n, c, torch.float32, seed=3, offset=far)
    dy = torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = F.group_norm(leaves[0], ints(cuts), groups, leaves[1], leaves[2], activation=act)
    (dx,) = torch.autograd.grad(y, leaves[:1], dy)
    want = norm_in_64_bits(x, cuts, None, groups, w, b, 1e-5, act, 0.01, dy)
    for lo, hi in zip(cuts, cuts[1:]):
        part = lambda t: t[lo:hi].double().view(hi - lo, groups, -1)      # noqa: E731
        mean = lambda t: t.mean(dim=(0, 2), keepdim=True)      # noqa: E731
        v, h, z, dz, e = part(x), part(want["hat"]), part(want["z"]), part(want["dz"]), part(want["dx"])
        wide_w = w.double().view(1, groups, -1)
        var = mean((v - mean(v)) ** 2)
        rstd = (var + 1e-5).rsqrt()
        d_off = 2 * U * (v.abs() + mean(v).abs())                         # of x - mean
        r_off = 32 * U + mean(2 * (v - mean(v)).abs() * d_off + d_off ** 2) / (2 * var)
        h_off = rstd * d_off + h.abs() * (r_off + 2 * U)
        z_off = h_off * wide_w.abs() + 2 * U * (z.abs() + b.double().view(1, groups, -1).abs())
        g, g_off = dz * wide_w, wide_w.abs() * part(dy).abs() * ((0.5 * z_off if act else 0) + 8 * U)
        m1_off = mean(g_off) + 128 * U * mean(g.abs())
        m2_off = mean(g_off * h.abs() + g.abs() * h_off) + 128 * U * mean((g * h).abs())
        bound = e.abs() * r_off + rstd * (g_off + m1_off + h_off * mean(g * h).abs() + h.abs() * m2_off
                                          + 8 * U * (g.abs() + mean(g).abs() + (h * mean(g * h)).abs()))
        off = (part(dx) - e).abs()
        assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.3g} bounds"


def test_a_captured_step_with_a_gradient_of_a_gradient():
    """A gradient penalty recorded into a graph and replayed on other inputs and offsets."""
    from torchsparse_b200.nn import functional as F

    def inputs(seed, n=9001, c=24):
        g = torch.Generator(device="cuda").manual_seed(seed)
        return {"x": torch.randn(n, c, generator=g, device="cuda"), "dy": torch.randn(n, c, generator=g, device="cuda"),
                "w": torch.rand(c, generator=g, device="cuda") + 0.5, "b": torch.randn(c, generator=g, device="cuda"),
                "order": torch.randperm(n, generator=g, device="cuda").int(), "offsets": ints([0, 3000 + seed, 3000 + seed, n - seed])}

    def step(s):
        leaves = [s[k].detach().requires_grad_() for k in ("x", "w", "b")]
        y = F.group_norm(leaves[0], s["offsets"], 3, leaves[1], leaves[2], activation="silu", order=s["order"])
        first = torch.autograd.grad(y, leaves, s["dy"], create_graph=True)
        return list(first) + list(torch.autograd.grad(first[0].square().sum(), leaves))

    s, side = inputs(1), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(s)
    for seed in (2, 5):
        for k, v in inputs(seed).items():
            s[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(inputs(seed))):
            assert torch.equal(a.detach(), b.detach())
