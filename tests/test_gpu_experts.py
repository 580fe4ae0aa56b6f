"""GPU numerics of the expert layer (camoe_b200/experts.py, include/camoe_experts.h)
against a plain statement of the same formulas in 64 bits.

The sort and the copies are exact, and so is the rounded sum of two rows.
Elsewhere tolerances follow from the number of roundings: one rounding to bf16
moves a value by at most 2^-8 of itself, uniformly over values by 2^-8 / sqrt(6)
in the root mean square, which is below u = 2^-9; so a tensor whose values went
through m of them is within m u of the exact one in the 2-norm; fp32 sums of n
terms are within n 2^-24 of the sum of the terms' magnitudes.
"""
import pytest
import torch

from camoe_b200 import _lib, experts

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -9


@pytest.fixture(autouse=True)
def _no_device_timeouts():
    before = _lib.lib().camoe_wkv7_device_errors()
    yield
    assert _lib.lib().camoe_wkv7_device_errors() == before


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(*shape, seed, scale=1.0, dtype=BF):
    return (scale * torch.randn(*shape, generator=gen(seed))).to(dtype).cuda()


def close(got, want, tol, name):
    """2-norm of the difference over that of the result, whole and for each row
    (a row may be off by twice the share: its error is not averaged as much)."""
    got, want = got.detach().double(), want.double()
    assert torch.isfinite(got).all(), name
    got, want = got.reshape(-1, got.shape[-1]), want.reshape(-1, want.shape[-1])
    norm = want.norm()
    assert float((got - want).norm()) <= tol * float(norm), name
    typical = norm / max(1, want.shape[0]) ** 0.5
    rows = (got - want).norm(dim=1) / torch.maximum(want.norm(dim=1), typical).clamp(min=1e-300)
    assert (rows <= 2 * tol).all(), (name, rows.tolist())


def plain_sort(index, E):
    """(offsets, position, source) by definition, on the host."""
    flat = index.cpu().reshape(-1).tolist()
    of = [[] for _ in range(E)]
    for s, e in enumerate(flat):
        if 0 <= e < E:
            of[e].append(s)
    order = [s for slots in of for s in slots]
    position, source = [-1] * len(flat), order + [-1] * (len(flat) - len(order))
    for p, s in enumerate(order):
        position[s] = p
    offsets = [sum(len(slots) for slots in of[:b]) for b in range(E + 1)]
    return offsets, position, source


def index_of(N, k, E, seed, empty=0.0, dtype=torch.int64):
    g = gen(seed)
    i = torch.randint(0, E, (N, k), generator=g)
    return torch.where(torch.rand(N, k, generator=g) < empty, -1, i).to(dtype).cuda()


SORTS = [  # N, k, E: one slot, the one-launch path's ends, chunk borders, many experts
    (1, 1, 1), (1, 2, 8), (7, 3, 5), (1024, 2, 8), (1025, 2, 8), (683, 3, 1024), (2048, 1, 3), (5000, 2, 61),
    (4096, 4, 200), (8192, 4, 8), (32769, 1, 7),
]


@pytest.mark.parametrize("N,k,E", SORTS)
@pytest.mark.parametrize("empty,dtype", [(0.0, torch.int64), (0.3, torch.int32), (1.0, torch.int64)])
def test_dispatch_is_the_stable_sort(N, k, E, empty, dtype):
    index = index_of(N, k, E, 1, empty, dtype)
    x = rnd(N, 72, seed=2)
    xs, plan = experts.expert_dispatch(x, index, E)
    offsets, position, source = plain_sort(index, E)
    assert plan.offsets.tolist() == offsets
    assert plan.position.reshape(-1).tolist() == position
    assert plan.source.tolist() == source
    want = torch.zeros_like(xs)
    used = offsets[-1]
    want[:used] = x[plan.source[:used].long() // k]
    assert torch.equal(xs, want)


@pytest.mark.parametrize("E", [1, 8, 16, 17, 200, 511, 512])
@pytest.mark.parametrize("N,k", [(2049, 1), (2048, 2), (8191, 1), (4096, 2), (2731, 3)])
def test_dispatch_where_each_block_counts_all_slots(N, k, E):
    """Up to 8192 slots of up to 16 experts are placed in one launch, in which a block
    counts the slots before its chunk and behind it with the same counters; the others
    in two.  Fresh indices each time, spread, skewed and all of one expert."""
    x = rnd(N, 8, seed=3)
    for seed in range(4):
        index = index_of(N, k, E, 200 + seed, 0.0 if seed % 2 else 0.2, torch.int32)
        if seed == 2:
            index = torch.where(index > 0, index // 16, index)
        if seed == 3:
            index.fill_(E - 1)
        offsets, position, source = plain_sort(index, E)
        xs, plan = experts.expert_dispatch(x, index, E)
        assert plan.offsets.tolist() == offsets
        assert plan.position.reshape(-1).tolist() == position
        assert plan.source.tolist() == source
        used = offsets[-1]
        assert torch.equal(xs[:used], x[plan.source[:used].long() // k]) and not xs[used:].any()


def test_values_outside_the_experts_are_unused():
    index = torch.tensor([[0, 5], [-7, 2], [2 ** 40, 3], [1, -2 ** 40]]).cuda()
    _, plan = experts.expert_dispatch(rnd(4, 8, seed=3), index, 4)
    assert plan.offsets.tolist() == [0, 1, 2, 3, 4]
    assert plan.position.tolist() == [[0, -1], [-1, 2], [-1, 3], [1, -1]]
    assert plan.source.tolist() == [0, 6, 3, 5, -1, -1, -1, -1]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("C", [1, 7, 64, 1000, 2048])
@pytest.mark.parametrize("N", [3, 1500])
def test_dispatch_and_its_gradient(N, C, dtype):
    k, E = 2, 6
    index = index_of(N, k, E, 4, 0.2)
    x = rnd(N, C, seed=5, dtype=dtype).requires_grad_()
    xs, plan = experts.expert_dispatch(x, index, E)
    used = int(plan.offsets[-1])
    assert torch.equal(xs[:used], x.detach()[plan.source[:used].long() // k])
    assert not xs[used:].any()
    g = rnd(N * k, C, seed=6, dtype=dtype)
    g[used:] = float("nan")  # rows of no slot have no part in the gradient
    dx, = torch.autograd.grad(xs, x, g)
    want = torch.zeros(N, C, dtype=torch.float64, device="cuda")
    want.index_add_(0, plan.source[:used].long() // k, g[:used].double())
    if dtype == F32:
        assert torch.allclose(dx.double(), want, rtol=2 ** -23, atol=k * 2.0 ** -24 * float(g[:used].abs().max()))
    else:
        assert torch.equal(dx, want.float().to(BF))  # two values: the fp32 sum is the rounded exact one


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,k,C", [(1, 1, 8), (1, 2, 1024), (5, 3, 33), (300, 2, 2048), (2000, 5, 200)])
def test_combine_and_its_gradients(N, k, C, dtype):
    E = 7
    index = index_of(N, k, E, 7, 0.25)
    index[0] = -1 if N > 1 else index[0]  # a token with no slot at all
    _, plan = experts.expert_dispatch(rnd(N, 8, seed=8), index, E)
    used = int(plan.offsets[-1])
    ys = rnd(N * k, C, seed=9, dtype=dtype)
    ys[used:] = float("nan")
    ys.requires_grad_()
    w = rnd(N, k, seed=10, dtype=F32).requires_grad_()
    out = experts.expert_combine(ys, w, plan)
    dout = rnd(N, C, seed=11, dtype=dtype)
    dys, dw = torch.autograd.grad(out, (ys, w), dout)
    y, wd, g = ys.detach().double()[:used], w.detach().double().reshape(-1), dout.double()
    at = plan.source[:used].long()
    want = torch.zeros(N, C, dtype=torch.float64, device="cuda").index_add_(0, at // k, y * wd[at, None])
    dyw = g[at // k] * wd[at, None]
    dww = torch.zeros(N * k, dtype=torch.float64, device="cuda")
    dww[at] = (y * g[at // k]).sum(1)
    mag = torch.zeros_like(dww)
    mag[at] = (y * g[at // k]).abs().sum(1)
    if N > 1:
        assert not out[0].any() and not dw[0].any()
    assert not dys[used:].any()
    if dtype == F32:
        size = torch.zeros_like(want).index_add_(0, at // k, (y * wd[at, None]).abs())
        assert ((out.double() - want).abs() <= (k + 1) * 2.0 ** -24 * size).all()
        assert ((dys[:used].double() - dyw).abs() <= 2.0 ** -24 * dyw.abs()).all()
    else:
        close(out, want, U * 1.001, "out")
        close(dys[:used], dyw, U * 1.001, "dys")
    assert ((dw.reshape(-1).double() - dww).abs() <= C * 2.0 ** -24 * mag).all()


def test_combine_gradients_against_differences():
    """Central differences of the fp32 forward, which is linear in each input: with
    steps of a quarter the difference is the derivative up to fp32 rounding."""
    N, k, C, E = 40, 2, 96, 5
    _, plan = experts.expert_dispatch(rnd(N, 8, seed=12), index_of(N, k, E, 13, 0.2), E)
    ys, w = (rnd(N * k, C, seed=14, dtype=F32).requires_grad_(), rnd(N, k, seed=15, dtype=F32).requires_grad_())
    dout = rnd(N, C, seed=16, dtype=F32)
    grads = torch.autograd.grad(experts.expert_combine(ys, w, plan), (ys, w), dout)
    f = lambda a, b: float((experts.expert_combine(a, b, plan).double() * dout.double()).sum())
    with torch.no_grad():
        for t, other, g, pick in ((ys, w, grads[0], 0), (w, ys, grads[1], 1)):
            v = torch.randn(t.shape, generator=gen(17)).cuda()
            hi, lo = (f(t + s * v, other) if pick == 0 else f(other, t + s * v) for s in (0.25, -0.25))
            slope = float((g.double() * v.double()).sum())
            scale = float((g.double() * v.double()).abs().sum())
            assert abs((hi - lo) / 0.5 - slope) <= 1e-5 * scale


# ---------------------------------------------------------------- the experts' products

def split(counts, unused=0):
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()
    return offsets, sum(counts) + unused


FFN = [  # counts per expert, unused rows, C, F: rows streamed (few), row tiles' borders, odd widths, empty experts
    ([1], 0, 8, 8),
    ([1, 0, 1], 0, 1024, 4096),
    ([0, 0, 0], 3, 64, 128),
    ([3, 0, 9, 17, 0, 1, 2, 33], 5, 200, 520),
    ([40, 0, 24], 0, 128, 256),
    ([127, 128, 129, 0, 1], 0, 264, 328),
    ([600, 0, 5, 63, 64, 65], 30, 320, 1000),
    ([0, 0, 700], 0, 1000, 136),
    ([257, 255, 256], 1, 512, 768),
    ([0] * 300 + [20] + [0] * 700 + [9, 0], 2, 64, 72),         # few rows among 1003 experts
    ([0] * 12 + [33000 // 30] * 30 + [0] * 3, 0, 64, 136),      # a wide grid of full tiles
    ([2600, 0, 1700], 10, 256, 264),
]


def ffn_inputs(counts, unused, C, F, seed=20):
    offsets, R = split(counts, unused)
    E = len(counts)
    xs = rnd(R, C, seed=seed)
    xs[sum(counts):] = float("nan")  # rows of no expert are not read
    return offsets, xs, rnd(E, F, C, seed=seed + 1, scale=C ** -0.5), rnd(E, C, F, seed=seed + 2, scale=F ** -0.5)


def ffn_exact(offsets, xs, w_up, w_down, dys=None):
    cut = offsets.tolist()
    x, u, d = xs.double(), w_up.double(), w_down.double()
    out = {"ys": torch.zeros_like(x), "dxs": torch.zeros_like(x), "dw_up": torch.zeros_like(u), "dw_down": torch.zeros_like(d)}
    for e, (i, j) in enumerate(zip(cut[:-1], cut[1:])):
        pre = x[i:j] @ u[e].t()
        gate = pre.clamp(min=0)
        out["ys"][i:j] = gate ** 2 @ d[e].t()
        if dys is not None:
            g = dys[i:j].double()
            dpre = (g @ d[e]) * 2 * gate
            out["dxs"][i:j] = dpre @ u[e]
            out["dw_up"][e], out["dw_down"][e] = dpre.t() @ x[i:j], g.t() @ gate ** 2
    return out


@pytest.mark.parametrize("counts,unused,C,F", FFN)
def test_ffn_and_its_gradients(counts, unused, C, F):
    offsets, xs, w_up, w_down = ffn_inputs(counts, unused, C, F)
    used = sum(counts)
    for t in (xs, w_up, w_down):
        t.requires_grad_()
    ys = experts.expert_ffn(xs, w_up, w_down, offsets)
    dys = rnd(*ys.shape, seed=23)
    dys[used:] = float("nan")
    grads = torch.autograd.grad(ys, (xs, w_up, w_down), dys)
    want = ffn_exact(offsets, xs.detach(), w_up.detach(), w_down.detach(), dys)
    assert not ys[used:].any() and not grads[0][used:].any()
    # roundings: h and ys; h (halved by the root), dpre and the result; h and the result
    for name, got, tol in (("ys", ys, 2 * U), ("dxs", grads[0], 2.5 * U), ("dw_up", grads[1], 2.5 * U),
                           ("dw_down", grads[2], 2 * U)):
        close(got[:used] if name in ("ys", "dxs") else got, want[name][:used] if name in ("ys", "dxs") else want[name],
              tol, name)
    for e, n in enumerate(counts):
        if n == 0:
            assert not grads[1][e].any() and not grads[2][e].any()


def test_ffn_gradients_against_differences():
    """Central differences of the formula in 64 bits along random directions: the
    kernels' gradient is within its rounding (2.5 u of its norm, times the share of a
    random direction that falls on one error: a 2-norm over the entries)."""
    counts, C, F = [90, 0, 70], 128, 192
    offsets, xs, w_up, w_down = ffn_inputs(counts, 0, C, F, seed=30)
    ins = [t.requires_grad_() for t in (xs, w_up, w_down)]
    dys = rnd(*xs.shape, seed=33)
    grads = torch.autograd.grad(experts.expert_ffn(*ins, offsets), ins, dys)
    f = lambda a: float((ffn_exact(offsets, *a)["ys"] * dys.double()).sum())
    for i, g in enumerate(grads):
        v = torch.randn(g.shape, generator=gen(34 + i), dtype=torch.float64).cuda()
        v /= v.norm()
        v = v + g.double() / g.double().norm()  # along the gradient too, so that the slope is not near zero
        base = [t.detach().double() for t in ins]
        hi, lo = ([b + s * v if j == i else b for j, b in enumerate(base)] for s in (1e-5, -1e-5))
        slope = float((g.double() * v).sum())
        assert abs((f(hi) - f(lo)) / 2e-5 - slope) <= 2 * 2.5 * U * float(g.double().norm())


def test_ffn_keeps_each_row_to_itself():
    """A row of infinities or NaN changes its own result alone, on both paths."""
    for counts in ([5, 3], [300, 200]):
        offsets, xs, w_up, w_down = ffn_inputs(counts, 0, 64, 128, seed=40)
        clean = experts.expert_ffn(xs, w_up, w_down, offsets)
        bad = xs.clone()
        bad[4] = float("inf")
        bad[counts[0]] = float("nan")
        got = experts.expert_ffn(bad, w_up, w_down, offsets)
        keep = torch.ones(xs.shape[0], dtype=torch.bool, device="cuda")
        keep[4] = keep[counts[0]] = False
        assert torch.equal(got[keep], clean[keep])
        assert torch.isnan(got[counts[0]]).all() and not torch.isfinite(got[4]).any()


def test_ffn_gradient_of_one_expert_ignores_the_next_ones_rows():
    """The last rows of a group share a 64-row piece with the next group's: those must
    not reach its weight gradients, infinities among them."""
    offsets, xs, w_up, w_down = ffn_inputs([70, 70], 0, 64, 128, seed=45)
    dys = rnd(*xs.shape, seed=48)
    def grads(x, g):
        ins = [t.clone().requires_grad_() for t in (x, w_up, w_down)]
        return torch.autograd.grad(experts.expert_ffn(*ins, offsets), ins, g)
    clean = grads(xs, dys)
    bad = dys.clone()
    bad[70:] = float("inf")
    got = grads(xs, bad)
    assert torch.equal(got[1][0], clean[1][0]) and torch.equal(got[2][0], clean[2][0])


def test_results_repeat_bit_for_bit_and_on_another_stream():
    offsets, xs, w_up, w_down = ffn_inputs([300, 17, 0, 211], 4, 256, 512, seed=50)
    ins = [t.requires_grad_() for t in (xs, w_up, w_down)]
    dys = rnd(*xs.shape, seed=53)
    def one():
        ys = experts.expert_ffn(*ins, offsets)
        return (ys, *torch.autograd.grad(ys, ins, dys))
    first = one()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = one()
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a[:528] if a.shape == xs.shape else a, b[:528] if b.shape == xs.shape else b)


@pytest.mark.parametrize("tokens", [6, 1500])
def test_the_operators_replay_from_a_cuda_graph(tokens):
    """Their launches overlap (programmatic dependent launches): captured and replayed
    on new inputs they give what the calls give."""
    from camoe_b200 import adapters
    C, F, E, k = 128, 256, 5, 2
    x, index = rnd(tokens, C, seed=80), index_of(tokens, k, E, 81, 0.1)
    w = rnd(tokens, k, seed=82, dtype=F32)
    w_up, w_down = rnd(E, F, C, seed=83, scale=C ** -0.5), rnd(E, C, F, seed=84, scale=F ** -0.5)
    proj, down, up = rnd(C, C, seed=85, scale=C ** -0.5), rnd(3, 8, C, seed=86, scale=C ** -0.5), rnd(3, C, 8, seed=87)
    which = (torch.arange(tokens, device="cuda") % 4 - 1).to(torch.int32)

    def run():
        y = adapters.adapter_linear(x, proj, down, up, which)
        xs, plan = experts.expert_dispatch(y, index, E)
        return experts.expert_combine(experts.expert_ffn(xs, w_up, w_down, plan.offsets), w, plan)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    x.copy_(rnd(tokens, C, seed=88))
    index.copy_(index_of(tokens, k, E, 89, 0.4))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, run())


def test_gradients_that_are_strided_or_off_alignment():
    offsets, xs, w_up, w_down = ffn_inputs([40, 20], 0, 64, 128, seed=100)
    ins = [t.requires_grad_() for t in (xs, w_up, w_down)]
    dys = rnd(60, 64, seed=103)
    odd = torch.empty(60 * 64 + 1, dtype=BF, device="cuda")[1:].view(60, 64).copy_(dys)
    want = torch.autograd.grad(experts.expert_ffn(*ins, offsets), ins, dys)
    for g in (odd, dys.t().contiguous().t()):
        got = torch.autograd.grad(experts.expert_ffn(*ins, offsets), ins, g)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = rnd(30, 64, seed=104).requires_grad_()
    index = index_of(30, 2, 4, 105, 0.1)
    a, = torch.autograd.grad(experts.expert_dispatch(x, index, 4)[0], x, dys)
    b, = torch.autograd.grad(experts.expert_dispatch(x, index, 4)[0], x, odd)
    assert torch.equal(a, b)


def test_sorts_of_different_sizes_from_two_host_threads():
    """Through the C ABI, whose calls run side by side: sorts that need different amounts
    of shared memory."""
    import threading
    lib, failed = _lib.lib(), []

    def sorts(N, E, stream):
        index = index_of(N, 1, E, 110, 0.1, torch.int32)
        offsets, position, source = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, N, N))
        need = lib.camoe_ex_dispatch_work_bytes(N, 1, E)
        work = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for _ in range(3000):
            status = lib.camoe_ex_dispatch(None, 0, index.data_ptr(), 4, None, offsets.data_ptr(), position.data_ptr(),
                                           source.data_ptr(), work.data_ptr(), need, N, 1, E, 8, stream.cuda_stream)
            if status:
                return failed.append(status)
        stream.synchronize()
        if [offsets.tolist(), position.tolist(), source.tolist()] != list(plain_sort(index, E)):
            failed.append("wrong")

    threads = [threading.Thread(target=sorts, args=(N, E, torch.cuda.Stream())) for N, E in ((9000, 1024), (9000, 800))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_empty_inputs():
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    w_up, w_down = rnd(3, 16, 8, seed=60), rnd(3, 8, 16, seed=61)
    ins = [torch.empty(0, 8, dtype=BF, device="cuda").requires_grad_(), w_up.requires_grad_(), w_down.requires_grad_()]
    ys = experts.expert_ffn(*ins, offsets)
    grads = torch.autograd.grad(ys, ins, torch.empty_like(ys))
    assert ys.shape == (0, 8) and not grads[1].any() and not grads[2].any()
    xs, plan = experts.expert_dispatch(torch.empty(0, 8, dtype=BF, device="cuda"),
                                       torch.empty(0, 2, dtype=torch.int64, device="cuda"), 3)
    assert xs.shape == (0, 8) and plan.offsets.tolist() == [0] * 4
    out = experts.expert_combine(xs, torch.empty(0, 2, device="cuda"), plan)
    assert out.shape == (0, 8)


def test_refusals():
    x, index = rnd(4, 16, seed=70), torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    xs, plan = experts.expert_dispatch(x, index, 3)
    w = torch.ones(4, 2, device="cuda")
    w_up, w_down = rnd(3, 32, 16, seed=71), rnd(3, 16, 32, seed=72)
    bad = [
        (TypeError, lambda: experts.expert_dispatch(x.half(), index, 3)),
        (TypeError, lambda: experts.expert_dispatch(x, index.float(), 3)),
        (ValueError, lambda: experts.expert_dispatch(x, index.cpu(), 3)),
        (ValueError, lambda: experts.expert_dispatch(x, index[:3], 3)),
        (ValueError, lambda: experts.expert_dispatch(x.t().contiguous().t(), index, 3)),
        (ValueError, lambda: experts.expert_dispatch(x, index, 0)),
        (ValueError, lambda: experts.expert_dispatch(x, index, 1025)),
        (ValueError, lambda: experts.expert_combine(xs[:7], w, plan)),
        (TypeError, lambda: experts.expert_combine(xs, w.to(BF), plan)),
        (ValueError, lambda: experts.expert_combine(xs, w.t(), plan)),
        (TypeError, lambda: experts.expert_ffn(xs.float(), w_up, w_down, plan.offsets)),
        (TypeError, lambda: experts.expert_ffn(xs, w_up, w_down, plan.offsets.long())),
        (ValueError, lambda: experts.expert_ffn(xs, w_up, w_up, plan.offsets)),
        (ValueError, lambda: experts.expert_ffn(xs, w_up, w_down, plan.offsets[:3])),
        (ValueError, lambda: experts.expert_ffn(xs[:, :12].contiguous(), w_up[:, :, :12].contiguous(),
                                                w_down[:, :12].contiguous(), plan.offsets)),
        (_lib.CamoeError, lambda: experts.expert_ffn(torch.empty(8 * 16 + 1, dtype=BF, device="cuda")[1:].view(8, 16),
                                                     w_up, w_down, plan.offsets)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused_not_dropped(grad):
    """Forward-mode derivatives, with and without a gradient wanted as well."""
    import torch.autograd.forward_ad as fw
    from camoe_b200 import adapters
    x, index = rnd(4, 16, seed=120), torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    xs, plan = experts.expert_dispatch(x, index, 3)
    w = torch.ones(4, 2, device="cuda")
    w_up, w_down = rnd(3, 32, 16, seed=121), rnd(3, 16, 32, seed=122)
    down, up, which = rnd(2, 8, 16, seed=123), rnd(2, 32, 8, seed=124), torch.zeros(4, dtype=torch.int32, device="cuda")
    scale = torch.ones(2, device="cuda")
    calls = [
        (lambda a: experts.expert_dispatch(a, index, 3), (x,)),
        (lambda a, b: experts.expert_combine(a, b, plan), (xs, w)),
        (lambda a, b, c: experts.expert_ffn(a, b, c, plan.offsets), (xs, w_up, w_down)),
        (lambda a, b, c, d, e: adapters.adapter_linear(a, b, c, d, which, e), (x, w_up[0], down, up, scale)),
    ]
    for call, args in calls:
        for i in range(len(args)):
            with fw.dual_level(), torch.set_grad_enabled(grad and len(args) < 5):
                dual = fw.make_dual(args[i], torch.ones_like(args[i]))
                other = [t.clone().requires_grad_(grad and len(args) < 5) for t in args]
                with pytest.raises(RuntimeError, match="forward"):
                    call(*[dual if j == i else t for j, t in enumerate(other)])


def test_second_derivatives_are_refused_not_dropped():
    """A gradient that was recorded takes part in another backward: an error, also where
    the loss reaches the inputs by another way.  Recorded and not gone through again
    it is the gradient."""
    N, k, E, C, F = 40, 2, 3, 16, 32
    index = index_of(N, k, E, 130, 0.1)
    x, ys = rnd(N, C, seed=131).requires_grad_(), rnd(N * k, C, seed=132).requires_grad_()
    w = rnd(N, k, seed=133, dtype=F32).requires_grad_()
    w_up, w_down = rnd(E, F, C, seed=134).requires_grad_(), rnd(E, C, F, seed=135).requires_grad_()
    plan = experts.expert_dispatch(x.detach(), index, E)[1]
    for call, ins in (
        (lambda: experts.expert_dispatch(x, index, E)[0], (x,)),
        (lambda: experts.expert_combine(ys, w, plan), (ys, w)),
        (lambda: experts.expert_ffn(ys, w_up, w_down, plan.offsets), (ys, w_up, w_down)),
    ):
        out = call()
        dout = torch.ones_like(out).requires_grad_()
        want = torch.autograd.grad(call(), ins, dout.detach())
        got = torch.autograd.grad(out, ins, dout, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for g in got:
            with pytest.raises(RuntimeError, match="differentiable once"):
                (g.float().square().sum() + ins[0].float().sum() + dout.float().sum()).backward(retain_graph=True)
    # a weight as the only way to what the gradient depends on
    out = experts.expert_combine(ys, w, plan)
    dys, = torch.autograd.grad(out, ys, torch.ones_like(out), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (dys.float().sum() + w.sum()).backward()
    # a gradient that depends on constants alone: nothing to refuse
    dys, = torch.autograd.grad(experts.expert_combine(ys, w.detach(), plan), ys, torch.ones_like(out), create_graph=True)
    assert not dys.requires_grad
    out = experts.expert_dispatch(x, index, E)[0]
    dx, = torch.autograd.grad(out, x, torch.ones_like(out), create_graph=True)
    assert not dx.requires_grad


def test_combine_refuses_what_its_backward_could_not_take():
    """The limits of the sort, before the forward rather than in the backward."""
    def call(N, k, E):
        plan = experts.ExpertPlan(torch.zeros(E + 1, dtype=torch.int32, device="cuda"),
                                  torch.full((N, k), -1, dtype=torch.int32, device="cuda"),
                                  torch.full((N * k,), -1, dtype=torch.int32, device="cuda"))
        ys = torch.zeros(N * k, 8, device="cuda").requires_grad_()
        return ys, experts.expert_combine(ys, torch.zeros(N, k, device="cuda"), plan)
    for N, k, E in ((4, 2, 1025), (4, 65, 8), (4, 0, 8)):
        with pytest.raises(ValueError, match="experts and 1 to 64 slots"):
            call(N, k, E)
    ys, out = call(4, 64, 1024)
    assert not torch.autograd.grad(out.sum(), ys)[0].any() and not out.any()
