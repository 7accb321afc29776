"""What is timed of the operators over rows that an index groups, and their plain forms.

* group norm with an activation over the rows of a batch of scans, channels last (rows grouped by sample);
* embedding lookup with scaling, and its gradient (rows grouped by token);
* rows sorted by expert and back with weights, and their gradients (rows grouped by expert).

``run`` computes an operator in elementary torch operations in 32 bits, or, with ``own`` set, through the calls a
user makes of the package.  ``exact`` computes the same from the definitions in 64 bits: sample by sample, with
gradients by differentiation where ``run`` has closed formulas.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_SLOPE, _EPS = 0.01, 1e-5


def _gn(name, rows, samples, channels, groups, dtype, activation, train):
    return {"name": name, "op": "group_norm", "rows": rows, "samples": samples, "channels": channels, "groups": groups,
            "dtype": dtype, "activation": activation, "train": train}


def _emb(name, tokens, vocab, channels, dtype, train):
    return {"name": name, "op": "embedding", "tokens": tokens, "vocab": vocab, "channels": channels, "dtype": dtype,
            "train": train}


def _moe(name, rows, top, experts, channels, dtype, train):
    return {"name": name, "op": "experts", "rows": rows, "top": top, "experts": experts, "channels": channels,
            "dtype": dtype, "train": train}


def listed():
    # Where a gradient is taken the activation is smooth: at the kink of a ReLU the sign of a rounding error decides
    # between two gradients, and a difference there says nothing about either side.
    return [
        # the coarsest level of a U-Net at batch 1 when it serves one scan: latency alone
        _gn("norm_serve_small", 1217, 1, 256, 32, "f16", "relu", False),
        # the finest level of a batch of four scans, served
        _gn("norm_serve_scans", 400003, 4, 96, 8, "f16", "leaky_relu", False),
        # a training step at a middle level, groups of 12 channels
        _gn("norm_train_middle", 61441, 2, 96, 8, "bf16", "silu", True),
        # the finest level of a batch of ragged scans, a million voxels
        _gn("norm_train_large", 1000000, 8, 64, 16, "bf16", "silu", True),
        # the same in 32 bits with many small samples and no activation
        _gn("norm_train_f32", 150011, 37, 128, 32, "f32", "none", True),
        # one step of generation for a few sequences
        _emb("embed_serve_few", 7, 32768, 1024, "f16", False),
        # a class label for each voxel of a batch of scans, looked up and trained: few rows, each used very often
        _emb("embed_train_labels", 500009, 301, 64, "bf16", True),
        # a batch of token sequences over a large vocabulary
        _emb("embed_train_tokens", 32768, 100003, 2048, "bf16", True),
        # odd width, 32 bits
        _emb("embed_train_odd", 60013, 4001, 99, "f32", True),
        # a few rows routed to two experts of eight
        _moe("experts_serve_few", 16, 2, 8, 1024, "f16", False),
        # a training step, many narrow experts
        _moe("experts_train_many", 30011, 6, 130, 200, "f32", True),
        # a training step over a long batch
        _moe("experts_train_large", 131072, 2, 8, 512, "bf16", True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op, dtype, train = rng.choice(("group_norm", "embedding", "experts")), rng.choice(("f32", "f16", "bf16")), rng.random() < 0.6
    if op == "group_norm":
        channels, groups = rng.choice(((16, 4), (24, 3), (32, 8), (48, 16), (64, 8), (96, 32), (100, 5), (128, 32), (192, 16),
                                       (256, 32), (320, 32), (77, 7)))
        rows = min(_log(rng, 300, 900000), 60_000_000 // channels)
        activation = rng.choice(("none", "silu") if train else ("none", "relu", "leaky_relu", "silu"))
        c = _gn("", rows, min(rows // 20, _log(rng, 1, 40)), channels, groups, dtype, activation, train)
    elif op == "embedding":
        vocab, channels = _log(rng, 8, 150000), _log(rng, 8, 2048)
        channels = channels if rng.random() < 0.3 else -(-channels // 8) * 8
        vocab = min(vocab, 150_000_000 // channels)
        c = _emb("", min(_log(rng, 1, 500000), 30_000_000 // channels), vocab, channels, dtype, train)
    else:
        top, experts, channels = rng.randint(1, 8), _log(rng, 8, 256), _log(rng, 16, 2048)
        channels = channels if rng.random() < 0.3 else -(-channels // 8) * 8
        c = _moe("", min(_log(rng, 1, 130000), 60_000_000 // (channels * top)), top, experts, channels, dtype, train)
    del c["name"]
    return c


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "group_norm":
        n, c = case["rows"] * case["channels"], case["channels"]
        offsets = 4 * (case["samples"] + 1)
        if not case["train"]:      # x in, y out
            return {"bytes": 2 * n * size + offsets + 8 * c, "flops": 10 * n}
        return {"bytes": 4 * n * size + offsets + 16 * c, "flops": 30 * n}      # and the gradients of both
    if case["op"] == "embedding":
        n, c = case["tokens"], case["channels"]
        rows = min(n, case["vocab"])
        got = {"bytes": (rows + n) * c * size + 8 * n, "flops": n * c}
        if case["train"]:          # the gradient of every output in, that of the whole table out
            got = {"bytes": got["bytes"] + (n + case["vocab"]) * c * size, "flops": 3 * n * c}
        return got
    n, k, c = case["rows"], case["top"], case["channels"]
    index = 8 * n * k + 8 * n * k + 4 * (case["experts"] + 1)      # the choices in; order, places and offsets out
    forward = n * c * size + n * k * c * size + n * k * c * size + n * c * size + 4 * n * k
    if not case["train"]:          # x in, sorted rows out; the experts' rows in, their weighted sums out
        return {"bytes": index + forward, "flops": 2 * n * k * c}
    return {"bytes": index + 2 * forward, "flops": 7 * n * k * c}


def _generator(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    dev = torch.device("cuda")
    g, host = _generator(seed, dev), _generator(seed + 1, "cpu")
    dtype, train, c = _TYPES[case["dtype"]], case["train"], case["channels"]
    normal = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, generator=g, device=dev)  # noqa: E731
    s = {"case": case}
    if case["op"] == "group_norm":
        n, b = case["rows"], case["samples"]
        share = torch.rand(b, generator=host) + 0.3                     # scans of a batch are of unlike sizes
        cuts = [0] + [int(v) for v in (share.cumsum(0) / share.sum() * n).long().tolist()[:-1]] + [n]
        s["longest"] = max(q - p for p, q in zip(cuts, cuts[1:]))
        s["cuts"] = cuts
        s["offsets"] = torch.tensor(cuts, dtype=torch.int32, device=dev)
        s["x"] = (normal(n, c) * (0.5 + uniform(c)) + (uniform(c) - 0.5)).to(dtype)
        s["weight"], s["bias"] = 0.5 + uniform(c), 0.2 * normal(c)
        if train:
            s["dy"] = normal(n, c).to(dtype)
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_()
    elif case["op"] == "embedding":
        n, v = case["tokens"], case["vocab"]
        rank = (uniform(n).double() * math.log(v + 1)).exp().long().sub(1).clamp(0, v - 1)      # a token's share falls as 1 / rank
        s["tokens"] = torch.randperm(v, generator=g, device=dev)[rank]
        s["tokens"][uniform(n) < 0.02] = -1                              # rows without a token
        s["table"] = normal(v, c).mul(c ** -0.5).to(dtype)
        s["scale"] = c ** 0.5
        if train:
            s["dy"] = normal(n, c).to(dtype)
            s["table"].requires_grad_()
    else:
        n, k, e = case["rows"], case["top"], case["experts"]
        liking = normal(n, e) + normal(e)                                # some experts are chosen more often
        best = liking.topk(min(k, e), dim=1)
        s["weights"] = torch.softmax(best.values, dim=1)
        s["choice"] = best.indices
        s["choice"][uniform(n, min(k, e)) < 0.02] = -1                   # choices dropped for want of room
        s["x"] = normal(n, c).to(dtype)
        s["ys"] = normal(n * min(k, e), c).to(dtype)                     # what the experts made of the sorted rows
        if train:
            s["dxs"], s["dout"] = normal(n * min(k, e), c).to(dtype), normal(n, c).to(dtype)
            for name in ("x", "ys", "weights"):
                s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------ the package's operators
def _own(s):
    from torchsparse_b200.nn import functional as F

    case = s["case"]
    if case["op"] == "group_norm":
        activation = None if case["activation"] == "none" else case["activation"]
        y = F.group_norm(s["x"], s["offsets"], case["groups"], s["weight"], s["bias"], _EPS, activation, _SLOPE)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "embedding":
        y = F.embedding(s["tokens"], s["table"], s["scale"])
        if not case["train"]:
            return {"y": y}
        return {"y": y, "dtable": torch.autograd.grad(y, s["table"], s["dy"])[0]}
    rows = F.expert_sort(s["choice"], case["experts"])
    xs = F.expert_dispatch(s["x"], rows)
    out = F.expert_combine(s["ys"], s["weights"], rows)
    got = {"order": rows.order, "inverse": rows.inverse, "offsets": rows.offsets, "xs": xs, "out": out}
    if case["train"]:
        dx, dys, dw = torch.autograd.grad((xs, out), (s["x"], s["ys"], s["weights"]), (s["dxs"], s["dout"]))
        got.update(dx=dx, dys=dys, dweights=dw)
    return got


# ------------------------------------------------------------------------------------------ plain forms
def _activate(z, activation):
    if activation == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if activation == "leaky_relu":
        return torch.where(z > 0, z, _SLOPE * z)
    return z / (1 + torch.exp(-z)) if activation == "silu" else z


def _slope_of(z, activation):
    if activation == "relu":
        return (z > 0).float()
    if activation == "leaky_relu":
        return torch.where(z > 0, torch.ones_like(z), torch.full_like(z, _SLOPE))
    if activation == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_norm(s):
    case, offsets = s["case"], s["offsets"].long()
    n, c, groups = case["rows"], case["channels"], case["groups"]
    x, weight, bias = s["x"].detach().float(), s["weight"].detach(), s["bias"].detach()
    sample = torch.searchsorted(offsets[1:], torch.arange(n, device=x.device), right=True)
    place = offsets[:-1, None] + torch.arange(s["longest"], device=x.device)        # the samples side by side, padded
    inside = (place < offsets[1:, None])[..., None]
    place = place.clamp(max=n - 1)
    count = (offsets[1:] - offsets[:-1]).clamp(min=1)[:, None] * (c // groups)

    def mean(t):      # [n, groups] of every sample and group, back at its rows
        return ((t[place] * inside).sum(1) / count)[sample].repeat_interleave(c // groups, dim=1)

    part = lambda t: t.view(n, groups, -1).sum(2)  # noqa: E731
    d = x - mean(part(x))
    rstd = 1 / torch.sqrt(mean(part(d * d)) + _EPS)
    hat = d * rstd
    z = hat * weight + bias
    y = _activate(z, case["activation"]).to(s["x"].dtype)
    if not case["train"]:
        return {"y": y}
    dz = s["dy"].float() * _slope_of(z, case["activation"])
    g = dz * weight
    dx = rstd * (g - mean(part(g)) - hat * mean(part(g * hat)))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (dz * hat).sum(0), "dbias": dz.sum(0)}


def _plain_embedding(s):
    tokens, table = s["tokens"], s["table"].detach()
    inside = (tokens >= 0) & (tokens < table.shape[0])
    at = torch.where(inside, tokens, torch.zeros_like(tokens))
    factor = (inside * s["scale"]).float()[:, None]
    y = (table[at].float() * factor).to(table.dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dtable = torch.zeros(table.shape, device=table.device).index_add_(0, at, s["dy"].float() * factor)
    return {"y": y, "dtable": dtable.to(table.dtype)}


def _plain_experts(s):
    choice, e = s["choice"], s["case"]["experts"]
    n, k = choice.shape
    x, ys, weights = s["x"].detach(), s["ys"].detach(), s["weights"].detach()
    flat = choice.reshape(-1)
    key = torch.where((flat >= 0) & (flat < e), flat, torch.full_like(flat, e))
    key, order = torch.sort(key, stable=True)                            # the dropped choices come last
    offsets = torch.searchsorted(key, torch.arange(e + 1, device=key.device))
    inverse = torch.empty_like(order)
    inverse[order] = torch.arange(n * k, device=key.device)
    kept = (key < e)[:, None]
    used = ((choice >= 0) & (choice < e))[..., None]
    xs = torch.where(kept, x[order // k], torch.zeros_like(x[:1]))
    mine = torch.where(used, ys[inverse].view(n, k, -1).float(), torch.zeros((), device=x.device))      # the experts' rows of each row
    got = {"order": order.int(), "inverse": inverse.view(n, k).int(), "offsets": offsets.int(), "xs": xs,
           "out": (weights[..., None] * mine).sum(1).to(x.dtype)}
    if s["case"]["train"]:
        dout = s["dout"].float()
        dx = (s["dxs"][inverse].view(n, k, -1).float() * used).sum(1)
        dys = kept * (weights.reshape(-1)[order][:, None] * dout[order // k])
        got.update(dx=dx.to(x.dtype), dys=dys.to(ys.dtype), dweights=(dout[:, None] * mine).sum(2))
    return got


def run(state):
    if own:
        return _own(state)
    return {"group_norm": _plain_norm, "embedding": _plain_embedding, "experts": _plain_experts}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------ 64 bits
def _wide(t, grad=False):
    return t.detach().double().requires_grad_(grad)


def _exact_norm(s):
    case = s["case"]
    d = case["channels"] // case["groups"]
    train = case["train"]
    x, weight, bias = (_wide(s[name], train) for name in ("x", "weight", "bias"))
    y = []
    for first, last in zip(s["cuts"], s["cuts"][1:]):
        rows = x[first:last].reshape(last - first, case["groups"], d)
        if last > first:
            var, mean = torch.var_mean(rows, dim=(0, 2), correction=0, keepdim=True)
            rows = (rows - mean) * (var + _EPS).rsqrt()
        y.append(rows.reshape(last - first, -1) * weight + bias)
    y = torch.cat(y)
    if case["activation"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["activation"] != "none":
        y = torch.maximum(y, y * (_SLOPE if case["activation"] == "leaky_relu" else 0.0))
    if not train:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (x, weight, bias), s["dy"].double())
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def _exact_embedding(s):
    table = _wide(s["table"])
    # one more row, of zeros, for what has no token; its gradient is not asked for
    table = torch.cat([table, torch.zeros_like(table[:1])]).requires_grad_(s["case"]["train"])
    tokens = torch.where(s["tokens"] < 0, table.shape[0] - 1, s["tokens"])
    y = table.index_select(0, tokens) * s["scale"]
    if not s["case"]["train"]:
        return {"y": y}
    return {"y": y.detach(), "dtable": torch.autograd.grad(y, table, s["dy"].double())[0][:-1]}


def _exact_experts(s):
    train = s["case"]["train"]
    x, ys, weights = (_wide(s[name], train) for name in ("x", "ys", "weights"))
    choice = s["choice"].cpu().numpy()
    n, k = choice.shape
    bins = [[] for _ in range(s["case"]["experts"] + 1)]
    for i, e in enumerate(choice.reshape(-1).tolist()):
        bins[e].append(i)                                                # -1: the last list
    order = torch.tensor([i for one in bins for i in one], device=x.device)
    kept = sum(len(one) for one in bins[:-1])
    place = torch.empty_like(order)
    place[order] = torch.arange(n * k, device=x.device)
    xs = torch.cat([x[order[:kept] // k], torch.zeros_like(ys[kept:])])
    weighted = ys[:kept] * weights.reshape(-1)[order[:kept], None]
    out = torch.zeros_like(x).index_add(0, order[:kept] // k, weighted)
    got = {"order": None, "inverse": None, "offsets": None, "xs": xs.detach(), "out": out.detach()}
    if train:
        dx, dys, dw = torch.autograd.grad((xs, out), (x, ys, weights), (s["dxs"].double(), s["dout"].double()))
        got.update(dx=dx, dys=dys, dweights=dw)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"group_norm": _exact_norm, "embedding": _exact_embedding, "experts": _exact_experts}[case["op"]](s)
