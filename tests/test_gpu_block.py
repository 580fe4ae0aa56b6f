"""The expert layer, the adapters and the time mix together (camoe_b200/block.py).

The layer against the formula in 64 bits (dispatch, products and combine round
to bf16 once, twice and once: within 4 u = 4 * 2^-9 in the 2-norm; gradients one
rounding more); generation step by step against one pass over the sequence (the
same rounded activations by different kernels: 2e-2 of the largest, as for the
time mix); adapters against the weights they amount to.
"""
import pytest
import torch

from camoe_b200 import _lib, experts
from camoe_b200.adapters import AdapterSet
from camoe_b200.block import ExpertBlock
from helpers import nrel

pytestmark = pytest.mark.gpu
U = 2.0 ** -9


@pytest.fixture(autouse=True)
def _no_device_timeouts():
    before = _lib.lib().camoe_wkv7_device_errors()
    yield
    assert _lib.lib().camoe_wkv7_device_errors() == before


def block(C=128, layers=2, layer=0, seed=0, **kw):
    torch.manual_seed(seed)
    b = ExpertBlock(C, layers, layer, **kw).cuda()
    with torch.no_grad():  # away from the zero initialisation of the output projections
        b.experts.w_down.normal_(0, b.experts.w_down.shape[2] ** -0.5)
        b.att.output.weight.normal_(0, C ** -0.5)
    return b


@pytest.mark.parametrize("tokens", [3, 900])
def test_expert_layer_and_its_gradients(tokens):
    C, E, F, k = 64, 5, 160, 2
    torch.manual_seed(1)
    layer = experts.ExpertLayer(C, E, F).cuda()
    with torch.no_grad():
        for p in (layer.w_up, layer.w_down):  # values that bf16 holds, so that the cast is exact
            p.copy_(torch.randn_like(p).mul_(p.shape[2] ** -0.5).bfloat16())
    x = torch.randn(tokens, C, device="cuda").bfloat16().float().requires_grad_()
    index = torch.randint(-1, E, (tokens, k), device="cuda")
    weight = torch.rand(tokens, k, device="cuda").requires_grad_()
    dout = torch.randn(tokens, C, device="cuda").bfloat16().float()
    out = layer(x, index, weight)
    ins = (x, weight, layer.w_up, layer.w_down)
    grads = torch.autograd.grad(out, ins, dout)
    d = [t.detach().double().requires_grad_() for t in ins]
    want = torch.zeros(tokens, C, dtype=torch.float64, device="cuda")
    for j in range(k):
        for e in range(E):
            at = torch.nonzero(index[:, j] == e)[:, 0]
            y = torch.relu(d[0][at] @ d[2][e].t()) ** 2 @ d[3][e].t()
            want = want.index_add(0, at, y * d[1][at, j:j + 1])
    exact = torch.autograd.grad(want, d, dout.double())
    assert float((out.double() - want).norm()) <= 4 * U * float(want.norm())
    for name, g, e in zip(("x", "weight", "w_up", "w_down"), grads, exact):
        assert float((g.double() - e).norm()) <= 5 * U * float(e.norm()), name
    assert grads[2].dtype == torch.float32


def test_block_trains_and_generates_the_same_steps():
    B, T, C = 2, 33, 128
    b = block(C)
    x = torch.randn(B, T, C, device="cuda")
    y, v, srep = b(x)
    (y.square().sum() + srep.sum()).backward()
    for name, p in b.named_parameters():
        if name.startswith(("att.v0", "att.v1", "att.v2")):
            continue  # the first layer has no value residual
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    assert b.experts.w_up.grad.abs().sum() > 0 and b.router.weight.grad.abs().sum() > 0
    # the routes are discontinuous: keep the router's logits well apart in both passes
    with torch.no_grad():
        b.router.weight.zero_()
        b.router.weight[:, 0] = torch.arange(8, device="cuda").float()
        b.ln2.bias[0] = 5.0
        b.ln2.weight[0] = 0.0
        y, v, _ = b(x)
        state, outs = None, []
        for t0, t1 in ((0, 20), (20, 32), (32, 33)):
            o, _, state = b.forward_state(x[:, t0:t1].contiguous(), None, state)
            outs.append(o)
    assert nrel(torch.cat(outs, 1).cpu(), y.detach().cpu()) < 2e-2


def in_bf16(module):
    """(the module in fp32 with values that bf16 holds, the module in bf16)"""
    import copy
    low = copy.deepcopy(module).bfloat16()
    return copy.deepcopy(low).float(), low


@pytest.mark.parametrize("layer", [0, 1])
def test_a_time_mix_in_bf16_is_the_same_with_those_values(layer):
    """The kernels take fp32 parameters and the products bf16 ones: which of both the
    module holds is no difference, but that its gradients are rounded."""
    B, T, C = 2, 48, 128
    full, low = in_bf16(block(C, layer=layer, seed=5).att)
    x = torch.randn(B, T, C, device="cuda")
    v_first = torch.randn(B, T, C, device="cuda").bfloat16() if layer else None
    got = []
    for m in (full, low):
        xs = x.clone().requires_grad_()
        y, _, srep = m(xs, v_first)
        (y.float().square().sum() + srep.square().sum()).backward()
        got.append((y, srep, xs.grad, {n: p.grad for n, p in m.named_parameters()}))
    for a, b in zip(got[0][:3], got[1][:3]):
        assert torch.equal(a, b)
    for n, g in got[0][3].items():
        assert (g is None) == (got[1][3][n] is None), n
        if g is not None:
            assert got[1][3][n].dtype == torch.bfloat16 and torch.equal(g.bfloat16(), got[1][3][n]), n
    with torch.no_grad():
        for m in (full, low):
            y, _, srep, _ = m.forward_state(x, v_first)
            got.append((y, srep))
    assert torch.equal(got[2][0], got[3][0]) and torch.equal(got[2][1], got[3][1])


@pytest.mark.parametrize("tokens", [1, 900])
def test_an_expert_layer_in_bf16_is_the_same_with_those_values(tokens):
    full, low = in_bf16(block(64, seed=6, n_experts=5, hidden=160).experts)
    x = torch.randn(tokens, 64, device="cuda").bfloat16()
    index = torch.randint(-1, 5, (tokens, 2), device="cuda")
    weight = torch.rand(tokens, 2, device="cuda")
    dout = torch.randn(tokens, 64, device="cuda").bfloat16()
    a, b = full(x, index, weight), low(x, index, weight)
    assert torch.equal(a, b)
    for p, q in zip(torch.autograd.grad(a, (full.w_up, full.w_down), dout),
                    torch.autograd.grad(b, (low.w_up, low.w_down), dout)):
        assert q.dtype == torch.bfloat16 and torch.equal(p.bfloat16(), q)


def test_a_block_in_bf16_trains_and_generates():
    """Against the fp32 block with the same values: ln1, the router's logits, ln2 and the
    two sums round to bf16 in one of them only (2e-2 of the largest, as between the
    block's own passes); the logits are far apart."""
    B, T, C = 3, 24, 128
    b = block(C, seed=7)
    with torch.no_grad():
        b.router.weight.zero_()
        b.router.weight[:, 0] = torch.arange(8, device="cuda").float()
        b.ln2.bias[0] = 5.0
        b.ln2.weight[0] = 0.0
    full, low = in_bf16(b)
    x = torch.randn(B, T, C, device="cuda").bfloat16()
    y, _, _ = low(x)
    assert y.dtype == torch.bfloat16
    y.float().square().sum().backward()
    assert all(torch.isfinite(p.grad).all() for n, p in low.named_parameters() if p.grad is not None)
    assert low.experts.w_up.grad.abs().sum() > 0 and low.att.r_k.grad.abs().sum() > 0
    with torch.no_grad():
        assert low(x.float())[0].dtype == torch.float32
        want = full(x.float())[0]
        state, outs = None, []
        for t0, t1 in ((0, 1), (1, 20), (20, 21), (21, 24)):
            o, _, state = low.forward_state(x[:, t0:t1].contiguous(), None, state)
            outs.append(o)
    assert nrel(y.detach().float().cpu(), want.cpu()) < 2e-2
    assert nrel(torch.cat(outs, 1).float().cpu(), want.cpu()) < 2e-2


@pytest.mark.parametrize("T", [1, 300])
def test_adapters_are_the_weights_they_amount_to(T):
    B, C, L, D = 3, 128, 2, 8
    b = block(C, seed=3).att
    x = torch.randn(B, T, C, device="cuda")
    down = {n: torch.randn(L, D, C, device="cuda") * C ** -0.5 for n in ("receptance", "key", "value", "output")}
    up = {n: torch.randn(L, C, D, device="cuda") * 0.3 for n in down}
    scale = torch.tensor([0.5, 2.0], device="cuda")
    adapters = AdapterSet()
    for n in down:
        adapters.add(n, down[n], up[n], scale)
    which = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    got = b.forward_state(x, adapters=adapters, adapter=which)[0]
    plain = {n: getattr(b, n).weight.detach().clone() for n in down}
    for i, a in enumerate(which.tolist()):
        with torch.no_grad():
            for n in down:
                w = plain[n].bfloat16().float()
                if a >= 0:
                    w = w + scale[a] * (up[n][a].bfloat16().float() @ down[n][a].bfloat16().float())
                getattr(b, n).weight.copy_(w)
            want = b.forward_state(x[i:i + 1].contiguous())[0]
        # the merged weights are rounded to bf16 again: one rounding of every projection apart
        assert nrel(got[i].float().cpu(), want[0].float().cpu()) < 3e-2, i
    with pytest.raises(ValueError):
        b.forward_state(x, adapters=adapters)


@pytest.mark.parametrize("T", [1, 5])
def test_ids_of_adapters_are_taken_as_they_are(T):
    """64-bit ids whose low 32 bits are an adapter's are outside [0, L): no adapter; ids
    of another kind than whole numbers are refused."""
    B, C = 3, 128
    b = block(C, seed=8).att
    x = torch.randn(B, T, C, device="cuda")
    adapters = AdapterSet().add("key", torch.randn(2, 8, C, device="cuda"), torch.randn(2, C, 8, device="cuda"))
    run = lambda ids, dtype: b.forward_state(x, adapters=adapters, adapter=torch.tensor(ids, dtype=dtype, device="cuda"))[0]
    want = run([-1, 1, -1], torch.int32)
    assert torch.equal(run([2 ** 32, 1, -2 ** 32 + 1], torch.int64), want)
    assert torch.equal(run([-1, 1, -1], torch.int8), want)
    for dtype in (torch.float32, torch.bool):
        with pytest.raises(TypeError):
            run([0, 1, 0], dtype)


def test_the_example_runs():
    from camoe_b200 import block as module
    module.main()
