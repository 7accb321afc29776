"""What autograd, forward-mode differentiation, functional transforms and tracing see of the operators over grouped rows.

Tolerances are shares of the largest value of a result: 2e-5 is 335 roundings of fp32 (2^-24 each).  The longest chain of a
first derivative or a tangent is below 200 of them: a sum over a sample is joined piece by piece, at most 100 deep, and some
twenty steps lie before and behind each of the two sums.  A second derivative goes through that twice and takes differences
of its terms: 1e-4."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

FIRST, SECOND = 2e-5, 1e-4
ACTS = {None: lambda t: t, "relu": torch.relu, "leaky_relu": lambda t: torch.nn.functional.leaky_relu(t, 0.1),
        "silu": lambda t: t * torch.sigmoid(t)}


def definition(x, w, b, cuts, order, groups, act, eps=1e-5):
    """Sample by sample with torch's own group norm, in the type of x; zeros in rows of no sample."""
    y = torch.zeros_like(x)
    for lo, hi in zip(cuts, cuts[1:]):
        if hi > lo:
            rows = torch.arange(lo, hi, device=x.device) if order is None else order[lo:hi].long()
            z = torch.nn.functional.group_norm(x[rows].t()[None], groups, w, b, eps)[0].t()
            y = y.index_copy(0, rows, ACTS[act](z))
    return y


def near(got, want, share):
    assert got.shape == want.shape
    if got.numel():
        off = float((got.detach().double() - want.detach()).abs().max())
        assert off <= share * float(want.detach().abs().max()), f"off by {off / max(float(want.detach().abs().max()), 1e-300):.3g}"


def data(n, c, seed=0, samples=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda")      # noqa: E731
    x = make(n, c) + 0.5
    w, b = torch.rand(c, generator=g, device="cuda") + 0.5, make(c) * 0.3
    order = torch.randperm(n, generator=g, device="cuda").int() if samples is None else None
    return x, w, b, make(n, c), order, make


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ traced programs
def test_traced_operators_are_in_the_graph_and_run_on_new_inputs():
    from torchsparse_b200.nn import functional as F

    def everything(x, w, b, offsets, tokens, choice, gate, table):
        y = F.group_norm(x, offsets, 3, w, b, activation="silu") + F.embedding(tokens, table, 2.0)
        rows = F.expert_sort(choice, 4)
        return F.expert_combine(F.expert_dispatch(y, rows), gate, rows), F.group_rows(tokens, 9).order

    def inputs(seed):
        x, w, b, _, _, make = data(500, 12, seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        return (x, w, b, ints([0, 100 + seed, 500]), torch.randint(0, 9, (500,), generator=g, device="cuda"),
                torch.randint(-1, 4, (500, 2), generator=g, device="cuda"), make(500, 2), make(9, 12))

    for record in (False, True):
        with torch.set_grad_enabled(record):
            args = [t.requires_grad_() if record and t.is_floating_point() else t for t in inputs(1)]
            traced = torch.jit.trace(everything, args, check_trace=False)
        kinds = {node.kind() for node in traced.graph.nodes()}
        for name in ("group_norm", "embedding", "expert_sort", "expert_dispatch", "expert_combine", "group_rows"):
            assert f"torchsparse_b200::{name}" in kinds
        with torch.no_grad():
            for got, want in zip(traced(*inputs(2)), everything(*inputs(2))):
                assert torch.equal(got, want)


def test_a_traced_norm_layer_runs_on_new_features():
    import torchsparse_b200 as ts
    from torchsparse_b200 import nn as spnn

    m = spnn.GroupNorm(4, 16, activation="silu").cuda().requires_grad_(False)      # a function is traced, so they are constants
    coords = torch.randint(0, 9, (400, 4), generator=torch.Generator().manual_seed(0)).int().cuda()
    coords[:, 0] = torch.arange(400, device="cuda") % 3
    run = lambda x: m(ts.SparseTensor(x, coords)).feats      # noqa: E731
    with torch.no_grad():
        traced = torch.jit.trace(run, data(400, 16, 1)[0], check_trace=False)
        x = data(400, 16, 2)[0]
        assert torch.equal(traced(x), run(x))


def test_gradients_recorded_by_a_dispatch_mode():
    """A recorder below autograd sees the operators and their gradients, not what their kernels leave behind."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from torchsparse_b200.nn import functional as F

    tokens = torch.randint(-1, 9, (300,), generator=torch.Generator().manual_seed(3)).cuda()
    rows = F.expert_sort(torch.randint(-1, 4, (300, 2), generator=torch.Generator().manual_seed(4)).cuda(), 4)
    offsets = ints([0, 100, 300])

    def step(x, w, b, table, gate, dout):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, table, gate)]
        y = F.group_norm(leaves[0], offsets, 3, leaves[1], leaves[2], activation="silu") + F.embedding(tokens, leaves[3], 2.0)
        out = F.expert_combine(F.expert_dispatch(y, rows), leaves[4], rows)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, dout))

    def inputs(seed):
        x, w, b, dout, _, make = data(300, 12, seed)
        return x, w, b, make(9, 12), make(300, 2), dout

    graph = make_fx(step)(*inputs(1))
    for got, want in zip(graph(*inputs(2)), step(*inputs(2))):
        assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------ a gradient of a gradient
def test_gradient_of_a_very_long_sample_to_be_differentiated_again():
    """More rows than fp32 counts one by one, and a mean that is no zero."""
    from torchsparse_b200.nn import functional as F

    n, c = 17_000_003, 2
    x, w, b, dy, _, _ = data(n, c, 1, samples=1)
    x += 2.0
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = F.group_norm(leaves[0], ints([0, n]), 1, leaves[1], leaves[2])
    got = torch.autograd.grad(y, leaves, dy, create_graph=True)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad(definition(*wide, [0, n], None, 1, None), wide, dy.double())
    for a, e in zip(got, want):
        near(a, e, FIRST)


@pytest.mark.parametrize("ordered", [False, True])
def test_second_derivative_of_long_samples(ordered):
    from torchsparse_b200.nn import functional as F

    n, c, cuts = 4_000_003, 4, [2, 3_999_000, 3_999_000, 4_000_000]
    x, w, b, dy, order, _ = data(n, c, 2, None if ordered else 1)
    leaves = [t.requires_grad_() for t in (x, w, b, dy)]
    y = F.group_norm(leaves[0], ints(cuts), 2, leaves[1], leaves[2], activation="silu", order=order)
    first = torch.autograd.grad(y, leaves[:3], leaves[3], create_graph=True)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad(definition(*wide[:3], cuts, order, 2, "silu"), wide[:3], wide[3], create_graph=True)
    for a, e in zip(first, want):
        near(a, e, FIRST)
    second = torch.autograd.grad(first[0].square().sum(), leaves)
    for a, e in zip(second, torch.autograd.grad(want[0].square().sum(), wide)):
        near(a, e, SECOND)


def test_second_derivative_gives_the_same_bits():
    from torchsparse_b200.nn import functional as F

    x, w, b, dy, order, _ = data(300_000, 8, 3)
    runs = []
    for _ in range(4):
        leaves = [t.clone().requires_grad_() for t in (x, w, b, dy)]
        y = F.group_norm(leaves[0], ints([0, 100_000, 299_000]), 2, leaves[1], leaves[2], activation="silu", order=order)
        first = torch.autograd.grad(y, leaves[:3], leaves[3], create_graph=True)
        runs.append(list(first) + list(torch.autograd.grad(first[0].square().sum(), leaves)))
    for run in runs[1:]:
        for a, e in zip(run, runs[0]):
            assert torch.equal(a, e)


@pytest.mark.parametrize("n,cuts", [(0, [0]), (0, [0, 0, 0]), (5, [0]), (5, [2, 2])])
def test_second_derivative_of_no_rows(n, cuts):
    from torchsparse_b200.nn import functional as F

    x, w, b, dy, order, _ = data(n, 12, 4)
    for o in (None, order):
        leaves = [t.clone().requires_grad_() for t in (x, w, b, dy)]
        y = F.group_norm(leaves[0], ints(cuts), 3, leaves[1], leaves[2], activation="silu", order=o)
        first = torch.autograd.grad(y, leaves[:3], leaves[3], create_graph=True)
        assert [t.shape for t in first] == [x.shape, w.shape, b.shape] and all(bool((t == 0).all()) for t in first)
        second = torch.autograd.grad(sum(t.square().sum() for t in first), leaves, materialize_grads=True)
        assert all(bool((t == 0).all()) for t in second)


@pytest.mark.parametrize("n", [40, 70_001])
def test_second_derivative_with_an_order_that_is_no_permutation(n):
    """Wrong values, and no fault: entries that are no rows go nowhere, as in the kernels."""
    from torchsparse_b200.nn import functional as F

    x, w, b, dy, order, _ = data(n, 12, 10)
    order[::7], order[1], order[2] = n, -1, 2 ** 31 - 1
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = F.group_norm(leaves[0], ints([-5, n // 3, 2 * n]), 3, leaves[1], leaves[2], activation="silu", order=order)
    first = torch.autograd.grad(y, leaves, dy, create_graph=True)
    second = torch.autograd.grad(first[0].square().sum(), leaves)
    for t in (*first, *second):
        assert bool(t.isfinite().all())


# ------------------------------------------------------------------------------------------------ forward-mode tangents
@pytest.mark.parametrize("ordered", [False, True])
@pytest.mark.parametrize("recorded", ["off", "frozen", "trained"])
def test_tangents_of_group_norm(ordered, recorded):
    import torch.autograd.forward_ad as fwAD

    from torchsparse_b200.nn import functional as F

    cuts = [3, 5000, 5000, 9001]
    x, w, b, _, order, make = data(9010, 12, 5, None if ordered else 1)
    tangents = [make(*t.shape) for t in (x, w, b)]
    if recorded == "trained":
        w.requires_grad_()
        b.requires_grad_()
    for which in ((0,), (1, 2), (0, 1, 2)):
        with torch.set_grad_enabled(recorded != "off"), fwAD.dual_level():
            args = [fwAD.make_dual(t, d) if i in which else t for i, (t, d) in enumerate(zip((x, w, b), tangents))]
            y = F.group_norm(args[0], ints(cuts), 3, args[1], args[2], activation="silu", order=order)
            got = fwAD.unpack_dual(y).tangent
            assert got is not None
        wide = [t.detach().double() for t in (x, w, b)]
        moved = [d.double() if i in which else torch.zeros_like(d).double() for i, d in enumerate(tangents)]
        _, want = torch.func.jvp(lambda *a: definition(*a, cuts, order, 3, "silu"), tuple(wide), tuple(moved))
        near(got, want, FIRST)


def test_tangents_of_embedding_and_expert_rows():
    import torch.autograd.forward_ad as fwAD

    from torchsparse_b200.nn import functional as F

    g = torch.Generator(device="cuda").manual_seed(6)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda")      # noqa: E731
    tokens = torch.randint(-1, 9, (200,), generator=g, device="cuda")
    rows = F.expert_sort(torch.randint(-1, 4, (200, 2), generator=g, device="cuda"), 4)
    table, x, ys, gate = make(9, 16), make(200, 16), make(400, 16), make(200, 2)
    for record in (False, True):
        leaves = [t.clone().requires_grad_(record) for t in (table, x, ys, gate)]
        t_table, t_x, t_ys, t_gate = (make(*t.shape) for t in leaves)
        with fwAD.dual_level():
            dual = fwAD.make_dual
            tangent = lambda t: fwAD.unpack_dual(t).tangent      # noqa: E731
            table_, x_, ys_, gate_ = leaves
            assert torch.equal(tangent(F.embedding(tokens, dual(table_, t_table), 2.0)), F.embedding(tokens, t_table, 2.0))
            assert torch.equal(tangent(F.expert_dispatch(dual(x_, t_x), rows)), F.expert_dispatch(t_x, rows))
            by_rows, by_gate = F.expert_combine(t_ys, gate, rows), F.expert_combine(ys, t_gate, rows)
            assert torch.equal(tangent(F.expert_combine(dual(ys_, t_ys), gate_, rows)), by_rows)
            assert torch.equal(tangent(F.expert_combine(ys_, dual(gate_, t_gate), rows)), by_gate)
            both = F.expert_combine(dual(ys_, t_ys), dual(gate_, t_gate), rows)
            assert torch.equal(tangent(both), by_rows + by_gate)
            if record:      # a gradient of the values next to the tangents
                (got,) = torch.autograd.grad(fwAD.unpack_dual(both).primal.sum(), gate_)
                assert torch.equal(got, torch.autograd.grad(F.expert_combine(ys_, gate_, rows).sum(), gate_)[0])


def test_a_tangent_in_a_gradient_is_carried_or_refused():
    import torch.autograd.forward_ad as fwAD

    from torchsparse_b200.nn import functional as F

    x, w, b, dy, _, make = data(300, 12, 7)
    tokens = torch.randint(0, 9, (300,), generator=torch.Generator().manual_seed(7)).cuda()
    rows = F.expert_sort(tokens, 9)
    leaf, t_dy = x.clone().requires_grad_(), make(300, 12)
    y = F.group_norm(leaf, ints([0, 300]), 3, w, b, activation="silu")
    wide = x.double().requires_grad_()
    (want,) = torch.autograd.grad(definition(wide, w.double(), b.double(), [0, 300], None, 3, "silu"), wide, t_dy.double())
    with fwAD.dual_level():
        (dx,) = torch.autograd.grad(y, leaf, fwAD.make_dual(dy, t_dy))
        near(fwAD.unpack_dual(dx).tangent, want, FIRST)      # linear in dy
        table, gate = make(9, 12).requires_grad_(), make(300, 1).requires_grad_()
        for out in (F.embedding(tokens, table), F.expert_dispatch(leaf, rows), F.expert_combine(leaf, gate, rows)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, [t for t in (table, leaf, gate)], fwAD.make_dual(dy, t_dy), allow_unused=True)


# ------------------------------------------------------------------------------------------------ functional transforms
def _layer():
    import torchsparse_b200 as ts
    from torchsparse_b200 import nn as spnn

    m = spnn.GroupNorm(3, 12, activation="silu").cuda()
    coords = torch.randint(0, 9, (600, 4), generator=torch.Generator().manual_seed(0)).int().cuda()
    coords[:, 0] = torch.arange(600, device="cuda") % 2
    order = torch.cat([torch.arange(0, 600, 2), torch.arange(1, 600, 2)]).int().cuda()

    def run(x, w, b):
        return torch.func.functional_call(m, {"weight": w, "bias": b}, (ts.SparseTensor(x, coords),)).feats

    return run, lambda *a: definition(*a, [0, 300, 600], order, 3, "silu")


def test_functional_gradient_jvp_and_hessian_product_of_a_norm_layer():
    run, plain = _layer()
    x, w, b, dy, _, make = data(600, 12, 8)
    wide = tuple(t.double() for t in (x, w, b))
    loss = lambda f, out: lambda *a: (f(*a) * out).sum()      # noqa: E731
    got = torch.func.grad(loss(run, dy), (0, 1, 2))(x, w, b)
    want = torch.func.grad(loss(plain, dy.double()), (0, 1, 2))(*wide)
    for a, e in zip(got, want):
        near(a, e, FIRST)
    moved = tuple(make(*t.shape) for t in (x, w, b))
    near(torch.func.jvp(run, (x, w, b), moved)[1], torch.func.jvp(plain, wide, tuple(t.double() for t in moved))[1], FIRST)
    got = torch.func.jvp(torch.func.grad(loss(run, dy), (0, 1, 2)), (x, w, b), moved)[1]
    want = torch.func.jvp(torch.func.grad(loss(plain, dy.double()), (0, 1, 2)), wide, tuple(t.double() for t in moved))[1]
    for a, e in zip(got, want):
        near(a, e, SECOND)


def test_vmap_over_a_norm_layer():
    run, _ = _layer()
    x, w, b, dy, _, make = data(600, 12, 9)
    xs = make(3, 600, 12)
    assert torch.equal(torch.func.vmap(lambda t: run(t, w, b))(xs), torch.stack([run(t, w, b) for t in xs]))
    got = torch.func.vmap(torch.func.grad(lambda t: (run(t, w, b) * dy).sum()))(xs)
    for a, t in zip(got, xs):
        near(a, torch.func.grad(lambda u: (run(u, w, b) * dy).sum())(t).double(), FIRST)
