"""The expert and adapter operators over the sizes they serve: cases, plain forms and exact values.

Four operators (camoe_b200/experts.py, camoe_b200/adapters.py):

* ``dispatch``: tokens sorted by the expert that each of their slots chose, and its gradient;
* ``combine``: the experts' rows back to their tokens, weighted, and its gradients;
* ``ffn``: each expert's squared-ReLU feed-forward product over its own rows, and its gradients;
* ``adapter``: a projection shared by all rows with the low-rank adapter of each row's request beside it.

``run`` computes the plain form (elementary torch operations in 32 bits, rounded once at the end) or, where
``own`` is true, makes the calls a user makes of this package.
"""
import math

import torch

own = False


# ---------------------------------------------------------------- cases

def listed():
    """The layer sizes are those of this package's workloads: width 1024 and 2048, 8 sequences of 1024 steps, eight
    experts of which each token takes two, a feed-forward four times as wide as the model."""
    return [
        # one generated token for each of 16 sequences: what counts is the launch
        dict(name="dispatch_step", op="dispatch", tokens=16, k=2, experts=8, width=1024, dtype="bf16", empty=0.0, grad=False),
        # one layer of a training step over 8 x 1024 tokens
        dict(name="dispatch_layer", op="dispatch", tokens=8192, k=2, experts=8, width=1024, dtype="bf16", empty=0.0, grad=True),
        # a long share with many small experts in 32 bits, some slots dropped by a capacity limit
        dict(name="dispatch_long", op="dispatch", tokens=32771, k=3, experts=61, width=2048, dtype="fp32", empty=0.1, grad=True),
        # one generated token
        dict(name="combine_token", op="combine", tokens=1, k=2, experts=8, width=1024, dtype="bf16", empty=0.0, grad=False),
        # the way back in the same training layer, with slots dropped
        dict(name="combine_layer", op="combine", tokens=8192, k=2, experts=8, width=1024, dtype="bf16", empty=0.05, grad=True),
        # one generated token: two experts' weights are read for one row each
        dict(name="ffn_token", op="ffn", tokens=1, k=2, experts=8, width=1024, hidden=4096, empty=0.0, grad=False),
        # one generated token for each of 64 sequences: all experts' weights for a few rows each
        dict(name="ffn_batch", op="ffn", tokens=64, k=2, experts=8, width=1024, hidden=4096, empty=0.0, grad=False),
        # a prompt of odd length through six experts of odd width
        dict(name="ffn_prompt", op="ffn", tokens=2501, k=2, experts=6, width=1000, hidden=3560, empty=0.1, grad=False),
        # the experts of the training layer: forward and all gradients
        dict(name="ffn_layer", op="ffn", tokens=8192, k=2, experts=8, width=1024, hidden=4096, empty=0.0, grad=True),
        # one generated token of a request with an adapter
        dict(name="adapter_token", op="adapter", tokens=1, width=1024, out=1024, rank=16, adapters=4, packed=False, empty=0.0),
        # one token of each of 96 requests that use 40 adapters, some none
        dict(name="adapter_batch", op="adapter", tokens=96, width=2048, out=2048, rank=32, adapters=40, packed=False, empty=0.1),
        # packed prompts of several requests, each with its adapter, through a wide projection
        dict(name="adapter_prompt", op="adapter", tokens=7001, width=1024, out=4096, rank=64, adapters=9, packed=True, empty=0.1),
    ]


def _spread(rng, low, high, step=1):
    """A multiple of `step` in [low, high], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + 1)))
    return max(low, min(high, int(v) // step * step)) if step > 1 else max(low, min(high, int(v)))


def draw(rng):
    op = rng.choice(("dispatch", "combine", "ffn", "ffn", "adapter", "adapter"))
    empty = rng.choice((0.0, 0.0, 0.1, 0.5))
    if op in ("dispatch", "combine"):
        k = rng.choice((1, 2, 2, 3, 4))
        # widths of whole heads, of whole 16-byte pieces, and odd ones
        width = _spread(rng, 64, 2048, rng.choice((64, 8, 1)))
        most = 32771 * 3 * 2048 // (k * width)
        return dict(op=op, tokens=_spread(rng, 1, min(65536, most)), k=k, experts=max(k, rng.choice((2, 6, 8, 61, 200))),
                    width=width, dtype=rng.choice(("bf16", "bf16", "fp32")), empty=empty, grad=rng.random() < 0.6)
    if op == "ffn":
        width = _spread(rng, 128, 2048, rng.choice((64, 8)))
        hidden = max(8, int(width * rng.choice((2.0, 3.5, 4.0))) // 8 * 8)
        experts, k = rng.choice((4, 6, 8, 16)), rng.choice((1, 2, 2, 3))
        most = 16384 * 1024 * 4096 // (width * hidden * k)
        return dict(op=op, tokens=_spread(rng, 1, max(1, min(8192, most))), k=k, experts=experts, width=width, hidden=hidden,
                    empty=empty, grad=rng.random() < 0.5)
    packed = rng.random() < 0.5
    return dict(op=op, tokens=_spread(rng, 257, 16384) if packed else _spread(rng, 1, 512),
                width=_spread(rng, 128, 2048, rng.choice((64, 8))), out=_spread(rng, 128, 4096, rng.choice((64, 8))),
                rank=rng.choice((8, 16, 16, 32, 64, 96, 128)), adapters=rng.choice((1, 3, 12, 64)), packed=packed, empty=empty)


# ---------------------------------------------------------------- inputs

def _routes(g, tokens, k, experts, empty):
    """[tokens, k] chosen experts, distinct for a token and unevenly popular; a share of the slots is empty (-1)."""
    popular = torch.randn(experts, generator=g, device="cuda")
    logits = torch.randn(tokens, experts, generator=g, device="cuda") + 0.5 * popular
    value, index = torch.topk(logits, k, dim=1)
    weight = torch.softmax(value, dim=1)
    if empty:
        index = torch.where(torch.rand(tokens, k, generator=g, device="cuda") < empty, -1, index)
    return index, weight


def _sorted(index, experts):
    """Slots in the order of their experts (stable): offsets [experts + 1], position [tokens, k], source [tokens k]."""
    flat = index.reshape(-1)
    used = (flat >= 0) & (flat < experts)
    key, order = torch.sort(torch.where(used, flat, experts), stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device=flat.device)).to(torch.int32)
    rank = torch.arange(flat.numel(), device=flat.device)
    position = torch.empty_like(order)
    position[order] = rank
    position = torch.where(used, position, -1).to(torch.int32).reshape(index.shape)
    source = torch.where(rank < offsets[-1], order, -1).to(torch.int32)
    return offsets, position, source


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype)

    s = dict(case)
    n, c = case["tokens"], case["width"]
    if case["op"] == "adapter":
        count = case["adapters"]
        if case["packed"]:  # each request's rows together, requests of different lengths
            cut = torch.sort(torch.randint(0, n, (count,), generator=g, device="cuda")).values
            request = torch.searchsorted(cut, torch.arange(n, device="cuda"), right=True)
            of = torch.randint(0, count, (count + 1,), generator=g, device="cuda")
            of = torch.where(torch.rand(count + 1, generator=g, device="cuda") < case["empty"], -1, of)
            adapter = of[request]
        else:
            adapter = torch.randint(0, count, (n,), generator=g, device="cuda")
            adapter = torch.where(torch.rand(n, generator=g, device="cuda") < case["empty"], -1, adapter)
        s.update(x=normal(n, c), weight=normal(case["out"], c, scale=c ** -0.5),
                 down=normal(count, case["rank"], c, scale=c ** -0.5),
                 up=normal(count, case["out"], case["rank"], scale=case["rank"] ** -0.5),
                 scale=0.5 + 1.5 * torch.rand(count, generator=g, device="cuda"), adapter=adapter.to(torch.int32))
        return s
    index, weight = _routes(g, n, case["k"], case["experts"], case["empty"])
    rows = n * case["k"]
    if case["op"] == "dispatch":
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        s.update(index=index, x=normal(n, c, dtype=dtype).requires_grad_(case["grad"]))
        if case["grad"]:
            s["dxs"] = normal(rows, c, dtype=dtype)
        return s
    s["offsets"], s["position"], s["source"] = _sorted(index, case["experts"])
    if case["op"] == "combine":
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        s.update(ys=normal(rows, c, dtype=dtype).requires_grad_(case["grad"]), weight=weight.requires_grad_(case["grad"]))
        if case["grad"]:
            s["dout"] = normal(n, c, dtype=dtype)
        return s
    e, f = case["experts"], case["hidden"]
    s.update(xs=normal(rows, c).requires_grad_(case["grad"]), w_up=normal(e, f, c, scale=c ** -0.5).requires_grad_(case["grad"]),
             w_down=normal(e, c, f, scale=f ** -0.5).requires_grad_(case["grad"]))
    if case["grad"]:
        s["dys"] = normal(rows, c)
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    from camoe_b200 import adapters, experts

    if s["op"] == "adapter":
        return {"y": adapters.adapter_linear(s["x"], s["weight"], s["down"], s["up"], s["adapter"], s["scale"])}
    if s["op"] == "dispatch":
        xs, plan = experts.expert_dispatch(s["x"], s["index"], s["experts"])
        out = {"xs": xs, "offsets": plan.offsets, "position": plan.position, "source": plan.source}
        if s["grad"]:
            out["dx"], = torch.autograd.grad(xs, (s["x"],), s["dxs"])
        return out
    if s["op"] == "combine":
        plan = experts.ExpertPlan(s["offsets"], s["position"], s["source"])
        out = {"out": experts.expert_combine(s["ys"], s["weight"], plan)}
        if s["grad"]:
            out["dys"], out["dweight"] = torch.autograd.grad(out["out"], (s["ys"], s["weight"]), s["dout"])
        return out
    out = {"ys": experts.expert_ffn(s["xs"], s["w_up"], s["w_down"], s["offsets"])}
    if s["grad"]:
        out["dxs"], out["dw_up"], out["dw_down"] = torch.autograd.grad(out["ys"], (s["xs"], s["w_up"], s["w_down"]), s["dys"])
    return out


@torch.no_grad()
def _plain(s):
    return {"dispatch": _plain_dispatch, "combine": _plain_combine, "ffn": _plain_ffn, "adapter": _plain_adapter}[s["op"]](s)


def _take(rows, at):
    """rows[at] in 32 bits, zeros where `at` is negative."""
    return torch.where((at >= 0)[..., None], rows.float()[at.clamp(min=0).long()], 0.0)


def _plain_dispatch(s):
    x, k = s["x"], s["k"]
    offsets, position, source = _sorted(s["index"], s["experts"])
    xs = _take(x, torch.where(source >= 0, source // k, -1)).to(x.dtype)
    out = {"xs": xs, "offsets": offsets, "position": position, "source": source}
    if s["grad"]:
        out["dx"] = _take(s["dxs"], position).sum(1).to(x.dtype)
    return out


def _plain_combine(s):
    ys, weight, position, source = s["ys"], s["weight"], s["position"], s["source"]
    rows = _take(ys, position)
    out = {"out": (rows * weight[..., None]).sum(1).to(ys.dtype)}
    if s["grad"]:
        dout = s["dout"].float()
        w = torch.where(source >= 0, weight.reshape(-1)[source.clamp(min=0).long()], 0.0)
        out["dys"] = (_take(dout, torch.where(source >= 0, source // s["k"], -1)) * w[:, None]).to(ys.dtype)
        out["dweight"] = torch.where(position >= 0, (rows * dout[:, None]).sum(2), 0.0)
    return out


def _padded(offsets, rows):
    """Where each group's rows stand in [groups, most rows of a group]: (at, used), both of that shape."""
    count = offsets.diff()
    lane = torch.arange(max(1, int(count.max())), device=offsets.device)
    used = lane < count[:, None]
    return torch.where(used, offsets[:-1, None] + lane, -1), used


def _unpadded(batch, at, used, rows):
    """The groups' rows in one [rows, columns] matrix, zeros in rows of no group."""
    flat = batch.new_zeros(rows + 1, batch.shape[-1])  # the last row takes what is padding
    flat[torch.where(used, at, rows).long()] = batch
    return flat[:rows]


def _plain_ffn(s):
    xs, w_up, w_down = s["xs"], s["w_up"].float(), s["w_down"].float()
    rows = xs.shape[0]
    at, used = _padded(s["offsets"], rows)
    x = _take(xs, at)
    gate = torch.relu(x @ w_up.transpose(1, 2))
    h = gate * gate
    out = {"ys": _unpadded(h @ w_down.transpose(1, 2), at, used, rows).to(xs.dtype)}
    if s["grad"]:
        dy = _take(s["dys"], at)
        dpre = (dy @ w_down) * (2.0 * gate)
        out["dxs"] = _unpadded(dpre @ w_up, at, used, rows).to(xs.dtype)
        out["dw_up"] = (dpre.transpose(1, 2) @ x).to(s["w_up"].dtype)
        out["dw_down"] = (dy.transpose(1, 2) @ h).to(s["w_down"].dtype)
    return out


def _plain_adapter(s):
    x, rows = s["x"].float(), s["x"].shape[0]
    offsets, position, source = _sorted(s["adapter"][:, None], s["adapters"])
    at, used = _padded(offsets, rows)
    at = torch.where(used, source[at.clamp(min=0).long()], -1)
    low = _take(x, at) @ s["down"].float().transpose(1, 2)
    added = (low @ s["up"].float().transpose(1, 2)) * s["scale"][:, None, None]
    return {"y": (x @ s["weight"].float().t() + _unpadded(added, at, used, rows)).to(s["x"].dtype)}


# ---------------------------------------------------------------- work and exact values

def work(case):
    n, c = case["tokens"], case["width"]
    if case["op"] == "adapter":
        m, d = case["out"], case["rank"]
        used = min(case["adapters"], max(1, round(n * (1 - case["empty"])))) if not case["packed"] else case["adapters"]
        return {"bytes": 2 * (n * c + m * c + n * m + used * d * (c + m)) + 4 * n,
                "flops": 2 * n * c * m + 2 * n * (1 - case["empty"]) * d * (c + m)}
    rows = n * case["k"]
    full = rows * (1 - case["empty"])
    if case["op"] == "ffn":
        f, e = case["hidden"], min(case["experts"], max(1, round(full)))
        passes = 3 if case["grad"] else 1
        # forward: rows in and out, both weights; backward: the rows' two inputs and one output, both weights again, both gradients
        return {"bytes": 2 * (2 * rows * c + 2 * e * c * f) + (2 * (3 * rows * c + 2 * (e + case["experts"]) * c * f) if case["grad"] else 0),
                "flops": 4 * full * c * f * passes}
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "dispatch":
        return {"bytes": size * c * (n + rows) + (size * c * (full + n) if case["grad"] else 0) + 8 * rows + 8 * rows,
                "flops": full * c if case["grad"] else 0}
    return {"bytes": size * c * (full + n) + 8 * rows + ((size * c * (n + full + rows) + 4 * rows) if case["grad"] else 0),
            "flops": 2 * full * c * (3 if case["grad"] else 1)}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    d = {key: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for key, v in s.items()}
    if case["op"] == "adapter":
        y = d["x"] @ d["weight"].t()
        for a in range(case["adapters"]):
            at = torch.nonzero(s["adapter"] == a)[:, 0]
            y[at] += d["scale"][a] * ((d["x"][at] @ d["down"][a].t()) @ d["up"][a].t())
        return {"y": y}
    if case["op"] == "dispatch":
        flat = s["index"].reshape(-1)
        groups = [torch.nonzero(flat == e)[:, 0] for e in range(case["experts"])]
        order = torch.cat(groups)
        xs = d["x"].new_zeros(flat.numel(), case["width"])
        xs[: order.numel()] = d["x"][order // case["k"]]
        out = {"xs": xs, "offsets": None, "position": None, "source": None}
        if case["grad"]:
            out["dx"] = torch.zeros_like(d["x"]).index_add_(0, order // case["k"], d["dxs"][: order.numel()])
        return out
    if case["op"] == "combine":
        used = int(s["offsets"][-1])
        at = s["source"][:used].long()
        w = d["weight"].reshape(-1)[at]
        out = {"out": d["ys"].new_zeros(case["tokens"], case["width"]).index_add_(0, at // case["k"], d["ys"][:used] * w[:, None])}
        if case["grad"]:
            out["dys"] = torch.zeros_like(d["ys"])
            out["dys"][:used] = d["dout"][at // case["k"]] * w[:, None]
            dw = d["weight"].new_zeros(d["weight"].numel())
            dw[at] = torch.einsum("rc,rc->r", d["ys"][:used], d["dout"][at // case["k"]])
            out["dweight"] = dw.reshape(d["weight"].shape)
        return out
    cut = s["offsets"].tolist()
    out = {"ys": torch.zeros_like(d["xs"])}
    if case["grad"]:
        out.update(dxs=torch.zeros_like(d["xs"]), dw_up=torch.zeros_like(d["w_up"]), dw_down=torch.zeros_like(d["w_down"]))
    for e, (i, j) in enumerate(zip(cut[:-1], cut[1:])):
        x, pre = d["xs"][i:j], d["xs"][i:j] @ d["w_up"][e].t()
        h = torch.clamp(pre, min=0) ** 2
        out["ys"][i:j] = h @ d["w_down"][e].t()
        if case["grad"]:
            dy = d["dys"][i:j]
            dpre = (dy @ d["w_down"][e]) * 2 * torch.clamp(pre, min=0)
            out["dxs"][i:j] = dpre @ d["w_up"][e]
            out["dw_up"][e], out["dw_down"][e] = dpre.t() @ x, dy.t() @ h
    return out
