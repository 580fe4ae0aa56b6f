"""GPU numerics of the adapter projection (camoe_b200/adapters.py) against the
formula in 64 bits.  A rounding to bf16 is at most 2^-8 of a value and below u =
2^-9 in the root mean square; with few rows y is rounded once, with many the
low-rank rows are rounded too: two roundings at most."""
import pytest
import torch

from camoe_b200 import _lib, adapters

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
U = 2.0 ** -9


@pytest.fixture(autouse=True)
def _no_device_timeouts():
    before = _lib.lib().camoe_wkv7_device_errors()
    yield
    assert _lib.lib().camoe_wkv7_device_errors() == before


def rnd(*shape, seed, scale=1.0, dtype=BF):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def inputs(N, C, M, D, L, seed=0):
    g = torch.Generator().manual_seed(seed)
    adapter = torch.randint(-1, L, (N,), generator=g).to(torch.int32).cuda()
    scale = (0.5 + torch.rand(L, generator=g)).cuda()
    return (rnd(N, C, seed=seed + 1), rnd(M, C, seed=seed + 2, scale=C ** -0.5),
            rnd(L, D, C, seed=seed + 3, scale=C ** -0.5), rnd(L, M, D, seed=seed + 4, scale=D ** -0.5), adapter, scale)


def exact(x, weight, down, up, adapter, scale):
    x = x.double()
    y = x @ weight.double().t()
    for a in range(down.shape[0]):
        at = torch.nonzero(adapter == a)[:, 0]
        s = 1.0 if scale is None else float(scale[a].double())
        y[at] += s * ((x[at] @ down[a].double().t()) @ up[a].double().t())
    return y


def close(got, want, tol):
    got = got.double()
    assert torch.isfinite(got).all()
    assert float((got - want).norm()) <= tol * float(want.norm())
    typical = want.norm() / max(1, want.shape[0]) ** 0.5
    assert float(((got - want).norm(dim=1) / torch.maximum(want.norm(dim=1), typical)).max()) <= 2 * tol


CASES = [  # N, C, M, D, L
    (1, 8, 8, 8, 1), (1, 1024, 1024, 16, 4), (7, 200, 72, 24, 3), (9, 64, 136, 40, 2), (33, 2048, 1000, 128, 64),
    (256, 512, 512, 256, 5), (257, 64, 64, 8, 1), (300, 1000, 520, 16, 3), (400, 128, 256, 32, 64),
    (1000, 264, 328, 96, 7), (2100, 512, 1032, 256, 2), (5000, 128, 128, 64, 40),
    (513, 64, 264, 200, 33), (700, 128, 512, 16, 1024), (3000, 96, 520, 136, 64), (520, 2048, 4096, 64, 12),
]


@pytest.mark.parametrize("N,C,M,D,L", CASES)
def test_adapter_linear(N, C, M, D, L):
    x, w, down, up, adapter, scale = inputs(N, C, M, D, L)
    close(adapters.adapter_linear(x, w, down, up, adapter, scale), exact(x, w, down, up, adapter, scale), 2 * U)
    close(adapters.adapter_linear(x, w, down, up, adapter), exact(x, w, down, up, adapter, None), 2 * U)


@pytest.mark.parametrize("lengths", [[256, 256, 256], [1, 255, 257, 0, 511, 1], [0, 0, 700], [600, 0, 0], [255, 1, 0, 768]])
@pytest.mark.parametrize("none", [0, 100])
def test_requests_that_end_on_and_beside_tile_borders(lengths, none):
    L = len(lengths)
    N = sum(lengths) + none
    x, w, down, up, _, scale = inputs(N, 128, 320, 72, L, seed=50)
    adapter = torch.cat([torch.full((n,), a) for a, n in enumerate(lengths)] + [torch.full((none,), -1)])
    adapter = adapter[torch.randperm(N, generator=torch.Generator().manual_seed(51))] if none else adapter
    adapter = adapter.to(torch.int32).cuda()
    close(adapters.adapter_linear(x, w, down, up, adapter, scale), exact(x, w, down, up, adapter, scale), 2 * U)


@pytest.mark.parametrize("N", [20, 600])
def test_rows_without_an_adapter_get_the_projection_alone(N):
    x, w, down, up, adapter, scale = inputs(N, 128, 192, 16, 3, seed=10)
    for none in (-1, 3, -2 ** 31, 2 ** 31 - 1):
        adapter[:] = none
        got = adapters.adapter_linear(x, w, down * float("nan"), up * float("nan"), adapter, scale)
        close(got, x.double() @ w.double().t(), U * 1.01)
    adapter[:] = 1  # one adapter for all, infinities in the others
    down[0], up[2] = float("inf"), float("nan")
    close(adapters.adapter_linear(x, w, down, up, adapter, scale),
          exact(x, w, down[1:2], up[1:2], adapter - 1, scale[1:2]), 2 * U)


@pytest.mark.parametrize("N", [50, 700])
def test_a_row_of_infinities_stays_by_itself(N):
    x, w, down, up, adapter, scale = inputs(N, 64, 128, 8, 4, seed=20)
    clean = adapters.adapter_linear(x, w, down, up, adapter, scale)
    bad = x.clone()
    bad[5] = float("nan")
    got = adapters.adapter_linear(bad, w, down, up, adapter, scale)
    keep = torch.arange(N, device="cuda") != 5
    assert torch.equal(got[keep], clean[keep]) and torch.isnan(got[5]).all()


@pytest.mark.parametrize("N,M,D", [(60, 192, 16), (700, 320, 72), (1800, 512, 16)])
@pytest.mark.parametrize("which", ["up", "down", "scale"])
def test_an_adapter_that_is_not_finite_reaches_its_own_rows_alone(N, M, D, which):
    """Rows of several adapters and of none share tiles; one adapter overflowed.  The
    other rows keep their bits; its own are what the formula gives."""
    x, w, down, up, adapter, scale = inputs(N, 128, M, D, 5, seed=60)
    clean = adapters.adapter_linear(x, w, down, up, adapter, scale)
    broken = {"up": up, "down": down, "scale": scale}
    bad = broken[which].clone()
    bad[2].reshape(-1)[:1] = float("inf")
    bad[2].reshape(-1)[-1:] = float("nan") if which != "scale" else float("inf")
    broken[which] = bad
    got = adapters.adapter_linear(x, w, broken["down"], broken["up"], adapter, broken["scale"])
    own = adapter == 2
    assert own.any() and torch.equal(got[~own], clean[~own])
    if which == "up":  # the first output row of up holds the infinity, the last the NaN
        assert not torch.isfinite(got[own][:, 0]).any() and torch.isnan(got[own][:, -1]).all()
        assert torch.equal(got[own][:, 1:-1], clean[own][:, 1:-1])
    else:
        assert not torch.isfinite(got[own]).any()


def test_empty_and_another_stream():
    x, w, down, up, adapter, scale = inputs(500, 128, 256, 16, 5, seed=30)
    first = adapters.adapter_linear(x, w, down, up, adapter, scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = adapters.adapter_linear(x, w, down, up, adapter, scale)
    side.synchronize()
    assert torch.equal(first, second)
    assert adapters.adapter_linear(x[:0], w, down, up, adapter[:0], scale).shape == (0, 256)


def test_refusals():
    x, w, down, up, adapter, scale = inputs(4, 64, 32, 8, 2, seed=40)
    call = adapters.adapter_linear
    for kind, args in [
        (TypeError, (x.float(), w, down, up, adapter, scale)),
        (TypeError, (x, w, down, up, adapter.long(), scale)),
        (TypeError, (x, w, down, up, adapter, scale.to(BF))),
        (ValueError, (x, w, down, up[:1], adapter, scale)),
        (ValueError, (x, w[:, :60].contiguous(), down, up, adapter, scale)),
        (ValueError, (x, w, down[:, :4].contiguous(), up[:, :, :4].contiguous(), adapter, scale)),
        (ValueError, (x, w, down, up, adapter[:3], scale)),
        (ValueError, (x.cpu(), w, down, up, adapter, scale)),
        (ValueError, (x.t().contiguous().t(), w, down, up, adapter, scale)),
        (RuntimeError, (x, w.clone().requires_grad_(), down, up, adapter, scale)),
    ]:
        with pytest.raises(kind):
            call(*args)
    with torch.no_grad():
        call(x, w.clone().requires_grad_(), down, up, adapter, scale)


def test_a_trainable_scale_is_refused_as_the_other_inputs_are():
    x, w, down, up, adapter, scale = inputs(4, 64, 32, 8, 2, seed=41)
    with pytest.raises(RuntimeError, match="no backward"):
        adapters.adapter_linear(x, w, down, up, adapter, scale.requires_grad_())
    with torch.no_grad():
        adapters.adapter_linear(x, w, down, up, adapter, scale)


def test_a_status_of_the_library_is_its_own_error():
    """A width that only the library refuses, before any launch."""
    C = (1 << 24) + 8
    x, w, down = (torch.zeros(*s, C, dtype=BF, device="cuda") for s in ((1,), (8,), (1, 8)))
    with pytest.raises(_lib.CamoeError) as e:
        adapters.adapter_linear(x, w, down, torch.zeros(1, 8, 8, dtype=BF, device="cuda"),
                                torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert e.value.status == _lib.ERR_SHAPE
