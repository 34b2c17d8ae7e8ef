"""GPU: the 8-bit paged KV cache against 64-bit arithmetic: the quantised write, reading pages back, and decode
attention (through the package's functions)."""

from __future__ import annotations

import pytest
import torch

from oracle import cache8 as oc8
from tests._cache8 import attention_tolerance, make_cache8, numbers, poison_dead_tokens

pytestmark = pytest.mark.gpu


def _to(cuda, *ts):
    return [t.to(cuda) for t in ts]


def _q(rows, hq, d, seed, strided=False):
    g = torch.Generator().manual_seed(seed)
    if strided:  # a view of a packed projection
        return torch.randn(rows, hq * d + 256, generator=g).to(torch.bfloat16)[:, :hq * d].view(rows, hq, d)
    return torch.randn(rows, hq, d, generator=g).to(torch.bfloat16)


def _close(got, want, mag):
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() - attention_tolerance(want, mag)
    assert over.max() <= 0, f"off by {over.max():.3g} above the tolerance"


# ------------------------------------------------------------------------------------------------ decode
def _decode(nqt, cuda, lens, *, kind="int8", page_size=16, hq=16, hkv=8, d=128, seed=0, strided=False, poison=True,
            sm_scale=None, spread=1.0, q_gain=1.0):
    codes, scales, indptr, indices, last = make_cache8(lens, kind=kind, page_size=page_size, hkv=hkv, d=d, seed=seed,
                                                       spread=spread)
    q = _q(len(lens), hq, d, seed + 1, strided) * q_gain
    want, mag = oc8.attention(q, numbers(codes), scales.double(), indptr, indices, last, sm_scale=sm_scale)
    if poison:
        poison_dead_tokens(codes, scales, indptr, indices, last)
    nqt.kernels.clear_status(cuda)
    ws = nqt.decode_paged8_workspace(len(lens), hq, d, cuda)
    dev = _to(cuda, q, codes, scales, indptr, indices, last)
    for _ in range(2):  # the second launch meets the workspace the first one left
        out = nqt.batch_decode_paged8(*dev, ws, sm_scale=sm_scale)
    torch.cuda.synchronize()
    assert nqt.kernels.read_status(cuda) == 0
    _close(out.cpu(), want, mag)
    return out.cpu()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("lens", [[1], [1, 15, 16, 17, 31, 32, 33], [0, 5, 0, 0, 40, 0], [0, 0], [2048, 1, 700, 64, 3, 1999],
                                  [5000]])
def test_decode_lengths(nqt, cuda, kind, lens):
    out = _decode(nqt, cuda, lens, kind=kind)
    for r, n in enumerate(lens):
        assert n or (out[r] == 0).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize(("hq", "hkv", "d"), [(16, 8, 64), (8, 8, 128), (14, 2, 64), (32, 4, 128), (6, 2, 128),
                                              (5, 1, 64), (24, 3, 128), (1, 1, 128)])
def test_decode_head_layouts(nqt, cuda, kind, hq, hkv, d):
    _decode(nqt, cuda, [77, 300, 16, 1], kind=kind, hq=hq, hkv=hkv, d=d, seed=4, strided=True)


@pytest.mark.parametrize("page_size", [32, 64, 256])
def test_decode_page_sizes(nqt, cuda, page_size):
    _decode(nqt, cuda, [5, 130, 333, 1024, 255, 257], page_size=page_size, seed=3)


def test_decode_many_rows(nqt, cuda):
    """More rows than threads of a CTA, most of them short or empty."""

    g = torch.Generator().manual_seed(9)
    _decode(nqt, cuda, torch.randint(0, 40, (700,), generator=g).tolist(), hq=4, hkv=2, d=64, seed=5)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_decode_peaked_scores_and_wide_scales(nqt, cuda, kind):
    """Scores of hundreds (the running reference moves often) and block scales over many orders of magnitude."""

    _decode(nqt, cuda, [400, 33, 1500], kind=kind, seed=6, q_gain=30.0)
    _decode(nqt, cuda, [400, 33, 1500], kind=kind, seed=7, spread=6.0, q_gain=1e-3)


def test_decode_huge_and_tiny_queries(nqt, cuda):
    """Queries far outside fp16's range."""

    for gain, scale in ((2.0**60, 2.0**-63), (2.0**-60, 2.0**57)):
        _decode(nqt, cuda, [130, 20], seed=8, q_gain=gain, sm_scale=scale)


def test_decode_zero_scales_and_zero_queries(nqt, cuda):
    codes, scales, indptr, indices, last = make_cache8([100, 40], seed=9)
    scales[indices[:3].long()] = 0.0  # blocks that stand for zeros
    q = _q(2, 16, 128, 10)
    q[1, :5] = 0
    want, mag = oc8.attention(q, numbers(codes), scales.double(), indptr, indices, last)
    ws = nqt.decode_paged8_workspace(2, 16, 128, cuda)
    out = nqt.batch_decode_paged8(*_to(cuda, q, codes, scales, indptr, indices, last), ws)
    _close(out.cpu(), want, mag)


def test_decode_output_strides_capacity_and_graph(nqt, cuda):
    """A strided output whose gaps stay untouched, a workspace for more rows, capture and replay with new lengths."""

    lens = [500, 20, 333]
    codes, scales, indptr, indices, last = make_cache8(lens, seed=11)
    q = _q(3, 16, 128, 12)
    dq, dc, ds, dp, di, dl = _to(cuda, q, codes, scales, indptr, indices, last)
    ws = nqt.decode_paged8_workspace(64, 16, 128, cuda)
    wide = torch.full((3, 16, 160), 7.0, dtype=torch.bfloat16, device=cuda)
    view = wide[:, :, 2:130]
    nqt.batch_decode_paged8(dq, dc, ds, dp, di, dl, ws, batch_capacity=64, out=view)
    want, mag = oc8.attention(q, numbers(codes), scales.double(), indptr, indices, last)
    _close(view.cpu(), want, mag)
    assert (wide[:, :, :2] == 7).all() and (wide[:, :, 130:] == 7).all()

    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(dq)
    with torch.cuda.graph(graph):
        nqt.batch_decode_paged8(dq, dc, ds, dp, di, dl, ws, batch_capacity=64, out=out)
    dl.copy_(torch.tensor([1, 2, 3], dtype=torch.int32))
    for _ in range(3):
        graph.replay()
    want, mag = oc8.attention(q, numbers(codes), scales.double(), indptr, indices, torch.tensor([1, 2, 3]))
    _close(out.cpu(), want, mag)


def test_decode_is_deterministic(nqt, cuda):
    codes, scales, indptr, indices, last = make_cache8([9000, 3, 2000], seed=13)
    dev = _to(cuda, _q(3, 16, 128, 14), codes, scales, indptr, indices, last)
    ws = nqt.decode_paged8_workspace(3, 16, 128, cuda)
    first = nqt.batch_decode_paged8(*dev, ws)
    for _ in range(20):
        assert torch.equal(nqt.batch_decode_paged8(*dev, ws), first)


def test_decode_bad_page_reports_and_reads_zeros(nqt, cuda):
    codes, scales, indptr, indices, last = make_cache8([40, 40], seed=15)
    indices[1] = codes.shape[0] + 7
    nqt.kernels.clear_status(cuda)
    ws = nqt.decode_paged8_workspace(2, 16, 128, cuda)
    out = nqt.batch_decode_paged8(*_to(cuda, _q(2, 16, 128, 16), codes, scales, indptr, indices, last), ws)
    assert nqt.kernels.read_status(cuda) & 0x1
    assert torch.isfinite(out.float()).all()
    nqt.kernels.clear_status(cuda)


def test_decode_short_wait_reports_and_recovers(nqt, cuda):
    """A launch whose pipeline waits give up reports it, and the workspace serves the next one.  The cache is far
    larger than L2 and every CTA streams hundreds of tiles, so that some copy is still in flight at a wait."""

    g = torch.Generator().manual_seed(17)
    lens = torch.randint(3000, 9000, (64,), generator=g).tolist()
    need = [-(-n // 16) for n in lens]
    codes = torch.randint(-127, 128, (sum(need), 2, 16, 8, 128), dtype=torch.int8, device=cuda)
    scales = torch.full((sum(need), 2, 1, 8), 0.01, device=cuda)
    indptr = torch.tensor([0, *torch.tensor(need).cumsum(0).tolist()], dtype=torch.int32, device=cuda)
    indices = torch.randperm(sum(need), generator=g).to(torch.int32).to(cuda)
    last = torch.tensor([n - (p - 1) * 16 for n, p in zip(lens, need, strict=True)], dtype=torch.int32, device=cuda)
    args = (_q(64, 16, 128, 18).to(cuda), codes, scales, indptr, indices, last,
            nqt.decode_paged8_workspace(64, 16, 128, cuda))
    nqt.kernels.clear_status(cuda)
    want = nqt.batch_decode_paged8(*args)
    assert nqt.kernels.read_status(cuda) == 0
    for _ in range(3):
        nqt.batch_decode_paged8(*args, short_wait=True)
    assert nqt.kernels.read_status(cuda) & 0x2
    nqt.kernels.clear_status(cuda)
    for _ in range(2):
        assert torch.equal(nqt.batch_decode_paged8(*args), want)
    assert nqt.kernels.read_status(cuda) == 0


# ------------------------------------------------------------------------------------------------ write
EPS, THETA = 1e-6, 1.0e6


def _write_case(lens, chunks, *, kind, page_size=16, hq=16, hkv=8, d=128, seed=0, gain=1.0, at=0):
    """Rows of ``lens`` tokens whose last ``chunks`` the call writes; ``at``: added to every position."""

    codes, scales, indptr, indices, last = make_cache8(lens, kind=kind, page_size=page_size, hkv=hkv, d=d, seed=seed)
    g = torch.Generator().manual_seed(seed + 50)
    pos, pages, offs = [], [], []
    for r, (n, c) in enumerate(zip(lens, chunks, strict=True)):
        for i in range(n - c, n):
            pos.append(i + at)
            pages.append(int(indices[int(indptr[r]) + i // page_size]))
            offs.append(i % page_size)
    t = len(pos)
    qkv = (torch.randn(t, (hq + 2 * hkv) * d, generator=g) * torch.exp(torch.randn(t, 1, generator=g)) * gain)
    qkv = qkv.to(torch.bfloat16)
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(torch.bfloat16) for _ in range(2))
    return codes, scales, qkv, qw, kw, torch.tensor(pos), torch.tensor(pages), torch.tensor(offs)


def _split(qkv, hq, hkv, d):
    t = qkv.shape[0]
    return (qkv[:, :hq * d].view(t, hq, d), qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d),
            qkv[:, (hq + hkv) * d:].view(t, hkv, d))


def _check_write(nqt, cuda, case, *, kind, hq=16, hkv=8, d=128):
    codes, scales, qkv, qw, kw, pos, pages, offs = case
    q, k, v = _split(qkv, hq, hkv, d)
    dc, ds = _to(cuda, codes, scales)
    dq, dk, dv = _split(qkv.to(cuda), hq, hkv, d)
    rest = _to(cuda, qw, kw, pos)
    where = _to(cuda, pages, offs)
    nqt.kernels.clear_status(cuda)
    rot = nqt.paired_qk_norm_rope_paged_cache8(dq, dk, dv, *rest, EPS, THETA, dc, ds, *where)
    torch.cuda.synchronize()
    assert nqt.kernels.read_status(cuda) == 0
    assert torch.equal(dq.cpu(), q) and torch.equal(dk.cpu(), k)

    wq = oc8.norm_rope(q, qw, pos, EPS, THETA)
    # one rounding to bf16; fp32 norm, angle and rotation are off by a few 2^-24 of the row's largest element
    assert ((rot.cpu().double() - wq).abs() <= 2.0**-8 * wq.abs() + 2.0**-19 * wq.abs().amax(-1, keepdim=True)).all()

    new = torch.stack([oc8.norm_rope(k, kw, pos, EPS, THETA), v.double()], 1)
    wc, ws = numbers(codes), scales.double()
    oc8.write(wc, ws, new, pages.tolist(), offs.tolist(), kind)
    gc, gs = numbers(dc.cpu()), ds.cpu().double()
    # scales: fp32 arithmetic on fp32 keys
    assert ((gs - ws).abs() <= 2.0**-18 * ws).all()
    # codes: equal but where x / s lies within fp32's error of the middle between two codes, one step there
    step = torch.ones_like(wc) if kind == "int8" else torch.exp2(torch.floor(torch.log2(wc.abs().clamp_min(2.0**-6))) - 3)
    assert ((gc - wc).abs() <= 2.0 * step).all()
    assert (gc != wc).double().mean() <= 1e-3
    # tokens and blocks that the call does not name keep their bits
    untouched = torch.ones(codes.shape[:3], dtype=torch.bool)
    for p, o in zip(pages.tolist(), offs.tolist(), strict=True):
        untouched[p, :, o - o % 16:o - o % 16 + 16] = False
    assert torch.equal(dc.cpu().view(torch.uint8)[untouched], codes.view(torch.uint8)[untouched])
    return dc, ds


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("lens_chunks", [([1, 16, 17, 40, 33], [1, 1, 1, 1, 1]), ([37, 300, 16, 129], [37, 45, 16, 1]),
                                         ([20, 30, 64], [3, 15, 50])])
def test_write_lengths(nqt, cuda, kind, lens_chunks):
    lens, chunks = lens_chunks
    _check_write(nqt, cuda, _write_case(lens, chunks, kind=kind), kind=kind)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize(("hq", "hkv", "d", "page_size"), [(16, 8, 64, 16), (14, 2, 64, 64), (5, 1, 128, 32),
                                                           (24, 3, 128, 256)])
def test_write_layouts(nqt, cuda, kind, hq, hkv, d, page_size):
    case = _write_case([50, 400, 7], [50, 100, 1], kind=kind, hq=hq, hkv=hkv, d=d, page_size=page_size, seed=2)
    _check_write(nqt, cuda, case, kind=kind, hq=hq, hkv=hkv, d=d)


def test_write_far_positions(nqt, cuda):
    """Angles of millions of positions keep fp32's accuracy."""

    _check_write(nqt, cuda, _write_case([20, 33], [20, 5], kind="int8", at=3_000_000, seed=3), kind="int8")


def test_write_grows_scales_step_by_step(nqt, cuda):
    """Sixteen single-token writes into one block, each larger than the last."""

    g = torch.Generator().manual_seed(4)
    for kind in ("int8", "e4m3"):
        hq, hkv, d = 2, 2, 128
        codes = torch.zeros(2, 2, 16, hkv, d, dtype=oc8.DTYPE[kind])
        scales = torch.zeros(2, 2, 1, hkv)
        wc, ws, dc, ds = numbers(codes), scales.double(), *_to(cuda, codes, scales)
        w = torch.ones(d, dtype=torch.bfloat16)
        values = []
        for i in range(16):
            q, k, v = (torch.randn(1, 2, d, generator=g).to(torch.bfloat16) for _ in range(3))
            v = (v * 1.3**i).to(torch.bfloat16)
            at = torch.tensor([i])
            page = torch.tensor([1])
            nqt.paired_qk_norm_rope_paged_cache8(*_to(cuda, q, k, v, w, w, at), EPS, THETA, dc, ds,
                                                 *_to(cuda, page, at))
            new = torch.stack([oc8.norm_rope(k, w, at, EPS, THETA), v.double()], 1)
            oc8.write(wc, ws, new, [1], [i], kind)
            values.append(v[0].double())
        assert ((ds.cpu().double() - ws).abs() <= 2.0**-18 * ws).all()
        got = oc8.values(numbers(dc.cpu()), ds.cpu().double())[1, 1]
        s = ds.cpu().double()[1, 1, 0][None, :, None]
        x = torch.stack(values)
        # rounded again only when the scale at least doubled: in all within one final step of the value
        bound = s if kind == "int8" else 2 * (2.0**-4 * x.abs() + 2.0**-10 * s)
        assert ((got - x).abs() <= bound * (1 + 1e-5)).all()


def test_write_zero_rows_and_special_values(nqt, cuda):
    """A block of zeros has scale zero and a later token sets it; NaN and infinities stay in their own codes."""

    hq, hkv, d = 2, 1, 128
    w = torch.ones(d, dtype=torch.bfloat16)
    codes, scales = torch.full((1, 2, 16, hkv, d), 5, dtype=torch.int8), torch.full((1, 2, 1, hkv), 3.0)
    dc, ds = _to(cuda, codes, scales)
    one = torch.ones(1, 1, d, dtype=torch.bfloat16)
    for i, x in enumerate([0 * one, 2 * one]):
        q = torch.zeros(1, hq, d, dtype=torch.bfloat16)
        nqt.paired_qk_norm_rope_paged_cache8(*_to(cuda, q, x, x, w, w, torch.tensor([i])), EPS, THETA, dc, ds,
                                             *_to(cuda, torch.tensor([0]), torch.tensor([i])))
        back = nqt.read_paged_cache8(dc, ds, torch.tensor([0], device=cuda)).cpu()
        assert (back[0, 1, :i + 1, 0].float() == torch.tensor([0.0, 2.0])[:i + 1, None]).all()
    x = one.clone()
    x[0, 0, 3], x[0, 0, 4], x[0, 0, 5] = float("nan"), float("inf"), -float("inf")
    nqt.paired_qk_norm_rope_paged_cache8(*_to(cuda, torch.zeros(1, hq, d, dtype=torch.bfloat16), one, x, w, w,
                                              torch.tensor([0])), EPS, THETA, dc, ds,
                                         *_to(cuda, torch.tensor([0]), torch.tensor([0])))
    assert torch.isfinite(ds).all()
    assert dc[0, 1, 0, 0, 3:6].cpu().tolist() == [0, 127, -127]


def test_write_bad_page_reports_and_writes_nothing(nqt, cuda):
    case = _write_case([20, 20], [1, 1], kind="int8", seed=6)
    codes, scales, qkv, qw, kw, pos, pages, offs = case
    pages[0], offs[1] = codes.shape[0], 16
    dc, ds = _to(cuda, codes, scales)
    nqt.kernels.clear_status(cuda)
    nqt.paired_qk_norm_rope_paged_cache8(*_split(qkv.to(cuda), 16, 8, 128), *_to(cuda, qw, kw, pos), EPS, THETA, dc,
                                         ds, *_to(cuda, pages, offs))
    assert nqt.kernels.read_status(cuda) & 0x1
    nqt.kernels.clear_status(cuda)
    assert torch.equal(dc.cpu(), codes) and torch.equal(ds.cpu(), scales)


def test_write_odd_strides(nqt, cuda):
    """Rows that are only 2-byte aligned take the narrow loads."""

    codes, scales, qkv, qw, kw, pos, pages, offs = _write_case([35, 4], [35, 4], kind="int8", seed=7)
    q, k, v = _split(qkv, 16, 8, 128)
    wide = [torch.zeros(39, t.shape[1], 131, dtype=torch.bfloat16, device=cuda) for t in (q, k, v)]
    for w, t in zip(wide, (q, k, v), strict=True):
        w[:, :, 1:129] = t.to(cuda)
    out = torch.zeros(39, 16, 131, dtype=torch.bfloat16, device=cuda)
    a, b = _to(cuda, codes, scales), _to(cuda, codes, scales)
    rest, where = _to(cuda, qw, kw, pos), _to(cuda, pages, offs)
    r1 = nqt.paired_qk_norm_rope_paged_cache8(*(w[:, :, 1:129] for w in wide), *rest, EPS, THETA, *a, *where,
                                              out=out[:, :, 1:129])
    r2 = nqt.paired_qk_norm_rope_paged_cache8(*_to(cuda, q, k, v), *rest, EPS, THETA, *b, *where)
    assert torch.equal(r1, r2) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert (out[:, :, 0] == 0).all() and (out[:, :, 129:] == 0).all()


# ------------------------------------------------------------------------------------------------ read
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize(("page_size", "hkv", "d"), [(16, 8, 128), (64, 3, 64)])
def test_read_pages(nqt, cuda, kind, page_size, hkv, d):
    codes, scales, *_ = make_cache8([70, 30], kind=kind, page_size=page_size, hkv=hkv, d=d, seed=1)
    pages = torch.tensor([3, 0, 3, codes.shape[0] - 1])
    got = nqt.read_paged_cache8(*_to(cuda, codes, scales, pages)).cpu()
    want = oc8.values(numbers(codes), scales.double())[pages]
    assert got.shape == want.shape
    # code * scale in fp32, then bf16
    assert ((got.double() - want).abs() <= (2.0**-8 + 2.0**-23) * want.abs()).all()
    nqt.kernels.clear_status(cuda)
    bad = nqt.read_paged_cache8(*_to(cuda, codes, scales, torch.tensor([1, -1])))
    assert nqt.kernels.read_status(cuda) & 0x1 and (bad[1] == 0).all()
    nqt.kernels.clear_status(cuda)
    assert nqt.read_paged_cache8(*_to(cuda, codes, scales, pages[:0])).shape[0] == 0
