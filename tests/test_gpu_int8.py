"""GPU: the W8A8 projection against 64-bit arithmetic: the row quantiser and the product with its epilogues."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(shape, seed, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if spread:
        x *= torch.exp(spread * torch.randn(shape[0], 1, generator=g))
    return x.to(torch.bfloat16)


def _quantize(x):
    """(codes, scale) of the row rule in float64."""

    x = x.double()
    amax = x.abs().amax(1)
    codes = (x * (127 / amax.clamp_min(1e-300))[:, None]).round()
    return codes, amax / 127


@pytest.mark.parametrize(("m", "k"), [(1, 1), (3, 7), (5, 128), (64, 2048), (2, 1000), (9, 8192), (2, 20001), (7, 1025),
                                      (1, 33000)])
def test_quantize_rows(nqt, cuda, m, k):
    x = _rand((m, k), m + k, spread=3.0)
    x[m // 2, :] = 0 if m > 1 else x[m // 2, :]
    q, s = nqt.kernels.int8_quantize_rows(x.to(cuda))
    want, scale = _quantize(x)
    # one fp32 division
    assert ((s.cpu().double() - scale).abs() <= 2.0**-23 * scale).all()
    # x * f with f and the product rounded to fp32: the codes differ only where x / scale is within 127 * 2^-22 of
    # the middle between two, and then by one
    exact = x.double() / scale.clamp_min(1e-300)[:, None]
    near = ((exact - exact.floor()) - 0.5).abs() <= 127 * 2.0**-22
    diff = (q.cpu().double() - want).abs()
    assert (diff[~near] == 0).all() and (diff <= 1).all()
    assert q.stride(0) % 16 == 0 or m == 1


def test_quantize_rows_strided_and_special(nqt, cuda):
    base = _rand((6, 300), 3)
    x = base[:, 5:205]  # rows that are only 2-byte aligned
    q, s = nqt.kernels.int8_quantize_rows(x.to(cuda)[:, :])
    q2, s2 = nqt.kernels.int8_quantize_rows(base.to(cuda)[:, 5:205])
    assert torch.equal(q, q2) and torch.equal(s, s2)
    y = _rand((4, 64), 4)
    y[0, 3], y[1, 5], y[2] = float("nan"), float("inf"), 1e-40
    q, s = nqt.kernels.int8_quantize_rows(y.to(cuda))
    s = s.cpu()
    assert s[0].isnan() and s[1].isinf() and s[2] > 0 and s[3].isfinite()
    assert (q[2].cpu() == 127).all()


def _product(x, wq, ws, bias=None, gate_up=False):
    """The definition in float64 from given codes (x: (codes, scale))."""

    y = x[0] @ wq.double().t() * x[1][:, None] * ws.double()[None]
    if bias is not None:
        y = y + bias.double()
    if gate_up:
        f = y.shape[1] // 2
        y = torch.nn.functional.silu(y[:, :f]) * y[:, f:]
    return y


def _weight(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8), torch.rand(n, generator=g) * 0.01 + 1e-4


SHAPES = [(1, 1, 1), (1, 2048, 2048), (2, 17, 300), (8, 40, 129), (9, 33, 16), (16, 256, 4096), (64, 1000, 2047),
          (65, 130, 96), (127, 31, 640), (128, 4096, 128), (129, 300, 257), (300, 777, 1000), (1000, 513, 64),
          (2500, 640, 384)]


@pytest.mark.parametrize(("m", "n", "k"), SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_product_of_codes_is_exact(nqt, cuda, m, n, k, bias):
    """The integer sums are exact: what remains is fp32 scaling (three roundings) and one rounding to bf16."""

    g = torch.Generator().manual_seed(m * 7 + n)
    xq = torch.randint(-127, 128, (m, (k + 15) // 16 * 16), generator=g, dtype=torch.int8)[:, :k]
    xs = torch.rand(m, generator=g) + 0.01
    wq, ws = _weight(n, k, k)
    b = _rand((1, n), 5)[0] * 10 if bias else None
    weight = nqt.kernels.Int8Weight.from_quantized(wq.to(cuda), ws.to(cuda))
    dx = torch.empty((m, (k + 15) // 16 * 16), dtype=torch.int8, device=cuda)[:, :k]
    dx.copy_(xq)
    nqt.kernels.clear_status(cuda)
    y = nqt.kernels.linear_int8(dx, weight, None if b is None else b.to(cuda), xscale=xs.to(cuda))
    want = _product((xq.double(), xs.double()), wq, ws, b)
    size = want.abs() if b is None else want.abs() + b.double().abs()
    assert ((y.cpu().double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-21 * size).all()
    assert nqt.kernels.read_status(cuda) == 0


@pytest.mark.parametrize(("m", "f", "k"), [(1, 1, 16), (1, 6144, 2048), (3, 15, 70), (64, 16, 2048), (64, 1000, 512),
                                           (130, 17, 130), (600, 333, 257), (2000, 1024, 256)])
def test_gate_up(nqt, cuda, m, f, k):
    x = _rand((m, k), 1)
    wq, ws = _weight(2 * f, k, 2)
    xq, xs = nqt.kernels.int8_quantize_rows(x.to(cuda))
    weight = nqt.kernels.Int8Weight.from_quantized(wq.to(cuda), ws.to(cuda), gate_up=True)
    y = nqt.kernels.linear_int8(xq, weight, xscale=xs)
    gu = _product((xq.cpu().double(), xs.cpu().double()), wq, ws)
    want = torch.nn.functional.silu(gu[:, :f]) * gu[:, f:]
    # fp32 scaling moves the gate by 2^-22 of itself, the sigmoid by up to that times |g| (relative, on its small
    # side), and the fast exponential and division by 2^-21 (1 + |g|)
    rel = 2.0**-20 * (2 + gu[:, :f].abs())
    assert ((y.cpu().double() - want).abs() <= (2.0**-8 + rel) * want.abs() + 1e-30).all()
    # bf16 rows quantised on the way give the same
    assert torch.equal(nqt.kernels.linear_int8(x.to(cuda), weight), y)


@pytest.mark.parametrize(("m", "n", "k"), [(1, 300, 2048), (4, 100, 77), (8, 2048, 6144), (9, 64, 1000), (64, 512, 33),
                                           (200, 96, 1024), (1500, 64, 130)])
def test_bf16_rows_equal_quantize_then_product(nqt, cuda, m, n, k):
    x = _rand((m, k), 11, spread=2.0).to(cuda)
    weight = nqt.kernels.Int8Weight(_rand((n, k), 12).to(cuda))
    want, scale = _quantize(_rand((n, k), 12))
    assert ((weight.scale.cpu().double() - scale).abs() <= 2.0**-23 * scale).all()
    xq, xs = nqt.kernels.int8_quantize_rows(x)
    y = nqt.kernels.linear_int8(x, weight)
    assert torch.equal(y, nqt.kernels.linear_int8(xq, weight, xscale=xs))
    ref = _product((xq.cpu().double(), xs.cpu().double()), weight.q.cpu(), weight.scale.cpu())
    assert ((y.cpu().double() - ref).abs() <= (2.0**-8 + 2.0**-21) * ref.abs()).all()


def test_extreme_sums(nqt, cuda):
    """The largest int32 sums that K allows, of both signs."""

    k = 131072
    xq = torch.full((2, k), 127, dtype=torch.int8)
    xq[1] = -127
    wq = torch.full((3, k), 127, dtype=torch.int8)
    wq[1] = -127
    wq[2, ::2] = -127
    weight = nqt.kernels.Int8Weight.from_quantized(wq.to(cuda), torch.ones(3, device=cuda))
    y = nqt.kernels.linear_int8(xq.to(cuda), weight, xscale=torch.full((2,), 2.0**-20, device=cuda))
    want = _product((xq.double(), torch.full((2,), 2.0**-20).double()), wq, torch.ones(3))
    assert ((y.cpu().double() - want).abs() <= (2.0**-8 + 2.0**-22) * want.abs()).all()


def test_strided_output_and_rows(nqt, cuda):
    """Outputs in a wider, oddly aligned buffer leave its gaps alone; x rows of a packed projection."""

    for m, n, k, lead in ((5, 70, 200, 1), (200, 70, 200, 1), (140, 256, 512, 8)):
        x = _rand((m, k + 24), 21).to(cuda)[:, 8:8 + k]
        weight = nqt.kernels.Int8Weight(_rand((n, k), 22).to(cuda))
        wide = torch.full((m, n + 2 * lead + 1), 7.0, dtype=torch.bfloat16, device=cuda)
        y = nqt.kernels.linear_int8(x, weight, out=wide[:, lead:lead + n])
        assert torch.equal(y, nqt.kernels.linear_int8(x.contiguous(), weight))
        assert (wide[:, :lead] == 7).all() and (wide[:, lead + n:] == 7).all()


def test_graph_replay_and_empty(nqt, cuda):
    x = _rand((64, 512), 31).to(cuda)
    weight = nqt.kernels.Int8Weight(_rand((256, 512), 32).to(cuda), gate_up=True)
    out = torch.empty(64, 128, dtype=torch.bfloat16, device=cuda)
    nqt.kernels.linear_int8(x, weight, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nqt.kernels.linear_int8(x, weight, out=out)
    x.copy_(_rand((64, 512), 33))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, nqt.kernels.linear_int8(x, weight))
    assert nqt.kernels.linear_int8(x[:0], weight).shape == (0, 128)


def test_nan_rows_stay_their_own(nqt, cuda):
    x = _rand((70, 256), 41)
    x[3, 7] = float("nan")
    weight = nqt.kernels.Int8Weight(_rand((64, 256), 42).to(cuda))
    for rows in (5, 70):
        y = nqt.kernels.linear_int8(x[:rows].to(cuda), weight).cpu()
        assert y[3].isnan().all()
        assert y[torch.arange(rows) != 3].isfinite().all()


@pytest.mark.parametrize(("m", "n", "k"), [(9, 256, 4096), (16, 2048, 2048), (64, 2048, 6144), (64, 333, 5000),
                                           (128, 2048, 6144), (77, 100, 8192), (240, 2048, 6144), (130, 514, 4097),
                                           (512, 2048, 6144), (24, 33, 20000), (12, 1, 6000)])
@pytest.mark.parametrize("kind", ["plain", "bias", "gate_up"])
def test_long_sums_shared_by_clusters(nqt, cuda, m, n, k, kind):
    """Few tiles and a long K: the product of bf16 rows, its K shared among CTAs, next to the exact one of its codes."""

    x = _rand((m, k), 5 * m + n, spread=1.0).to(cuda)
    rows = 2 * n if kind == "gate_up" else n
    wq, ws = _weight(rows, k, m + n)
    weight = nqt.kernels.Int8Weight.from_quantized(wq.to(cuda), ws.to(cuda), gate_up=kind == "gate_up")
    bias = (torch.arange(n) % 7 - 3).to(torch.bfloat16) if kind == "bias" else None
    codes, scale = nqt.kernels.int8_quantize_rows(x)
    nqt.kernels.clear_status(cuda)
    got = nqt.kernels.linear_int8(x, weight, None if bias is None else bias.to(cuda))
    again = nqt.kernels.linear_int8(codes, weight, None if bias is None else bias.to(cuda), xscale=scale)
    assert nqt.kernels.read_status(cuda) == 0 and torch.equal(got, again)
    want = _product((codes.cpu().double(), scale.cpu().double()), wq, ws, bias, kind == "gate_up")
    # bf16's half step, and fp32: the sum's conversion, the scales' product, theirs, the bias's addition (2^-24 each, of
    # the terms); gate_up also the exponential and the quotient, some 2^-21
    size = want.abs() if bias is None else want.abs() + bias.double().abs()
    if kind == "gate_up":
        # silu's slope is under 1.1, so an error of 3 * 2^-24 |g| moves silu(g) u by as much of |g u| at most
        g, u = _product((codes.cpu().double(), scale.cpu().double()), wq, ws).split(n, dim=1)
        size = want.abs() + (g * u).abs() * 2.0**-2
    assert ((got.cpu().double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-20 * size + 1e-30).all()
