"""GPU: what the 8-bit operators' contracts promise beyond single calls: one workspace for calls of every shape, exact
codes at ties, NaN scales and codes that stay visible to those who see them and to nobody else."""

from __future__ import annotations

import pytest
import torch

from oracle import cache8 as oc8
from tests._cache8 import attention_tolerance, make_cache8, numbers

pytestmark = pytest.mark.gpu

EPS, THETA = 1e-6, 1.0e6


def _q(rows, hq, d, seed):
    return torch.randn(rows, hq, d, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ workspace
def _decode_shape(cuda, rows, hi, hq, hkv, d, seed):
    lens = torch.randint(1, hi, (rows,), generator=torch.Generator().manual_seed(seed)).tolist()
    case = (_q(rows, hq, d, seed), *make_cache8(lens, hkv=hkv, d=d, seed=seed))
    return [t.to(cuda) for t in case]


@pytest.mark.parametrize("shapes", [
    [(64, 1000, 8, 8, 128), (64, 1000, 32, 4, 128)],  # head layouts
    [(300, 200, 4, 2, 64), (2048, 60, 4, 2, 64)],     # capacities
    [(1, 30000, 5, 1, 64), (40, 700, 32, 4, 128), (9, 5000, 16, 2, 64), (1500, 40, 8, 8, 64)],
])
def test_a_workspace_serves_calls_of_every_shape(nqt, cuda, shapes):
    """Calls of unlike rows, heads and head sizes take turns on one workspace, each with its default capacity, and give
    what they give on a fresh one."""

    size = max(nqt.decode_paged8_workspace(rows, hq, d, cuda).numel() for rows, _, hq, _, d in shapes)
    shared = torch.zeros(size, dtype=torch.uint8, device=cuda)
    cases = [_decode_shape(cuda, *shape, seed=i + 3) for i, shape in enumerate(shapes)]
    want = [nqt.batch_decode_paged8(*c, nqt.decode_paged8_workspace(len(c[0]), c[0].shape[1], c[0].shape[2], cuda))
            for c in cases]
    nqt.kernels.clear_status(cuda)
    for _ in range(3):
        for case, expected in zip(cases, want, strict=True):
            out = torch.full_like(expected, 7.0)
            nqt.batch_decode_paged8(*case, shared, out=out)
            assert torch.equal(out, expected)
    assert nqt.kernels.read_status(cuda) == 0


def test_a_workspace_serves_every_capacity(nqt, cuda):
    """The capacity that a call names does not matter to the next one on the workspace."""

    case = _decode_shape(cuda, 4, 9000, 4, 2, 64, 17)
    ws = nqt.decode_paged8_workspace(8192, 4, 64, cuda)
    want = nqt.batch_decode_paged8(*case, nqt.decode_paged8_workspace(4, 4, 64, cuda))
    for capacity in (None, 8192, 5, 1700, 4, 2048):
        out = torch.full_like(want, 7.0)
        nqt.batch_decode_paged8(*case, ws, batch_capacity=capacity, out=out)
        assert torch.equal(out, want)


# ------------------------------------------------------------------------------------------------ quantiser
def _tie_rows(exponent):
    """Rows whose largest value has each mantissa once, with every smaller bf16 down to 2^-10 of it: the ties of
    x * 127 / amax among them."""

    mantissa = torch.arange(128, 256).double()
    x = torch.cat([mantissa * 2.0**-e for e in range(11)])
    rows = torch.where(x[None] <= mantissa[:, None], x[None], 0.0)
    return torch.cat([rows, -rows], 1) * 2.0**exponent


@pytest.mark.parametrize("exponent", [0, -60, 100, -118, -134])
@pytest.mark.parametrize("odd", [False, True])
def test_quantize_rows_ties_to_even(nqt, cuda, exponent, odd):
    """Every code is round(x * 127 / amax), ties to even; the rows of -134 are subnormal numbers."""

    x = _tie_rows(exponent).to(torch.bfloat16)
    if odd:
        x = torch.cat([x, x[:, :1] * 0], 1)  # a length that takes the narrow loads
    exact = x.double() * 127
    # in 64 bits a tie is exact and nothing else comes near one: 8-bit significands keep quotients 2^-19 apart from it
    want = (exact / x.double().abs().amax(1, keepdim=True)).round()
    q, s = nqt.kernels.int8_quantize_rows(x.to(cuda))
    assert torch.equal(q.cpu().double(), want)
    top = x.double().abs().amax(1) / 127
    assert ((s.cpu().double() - top).abs() <= 2.0**-24 * top + 2.0**-150).all()


def test_product_of_few_tokens_quantises_ties_alike(nqt, cuda):
    """The launch for up to 8 tokens quantises by itself: every code it multiplies is the row quantiser's."""

    rows = _tie_rows(0).to(torch.bfloat16)[40:48]
    x = torch.cat([rows[:, 128:828], rows.amax(1, keepdim=True)], 1)
    k = x.shape[1]
    weight = nqt.kernels.Int8Weight.from_quantized(torch.eye(k, dtype=torch.int8, device=cuda), torch.ones(k, device=cuda))
    amax = x.double().abs().amax(1, keepdim=True)
    scale = (amax / 127).float().double()
    want = ((x.double() * 127 / amax).round() * scale).to(torch.float32).to(torch.bfloat16)
    for m in (1, 2, 3, 8):
        assert torch.equal(nqt.kernels.linear_int8(x[:m].to(cuda), weight).cpu(), want[:m])


# ------------------------------------------------------------------------------------------------ NaN scales
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("what", [0, 1])
@pytest.mark.parametrize(("hq", "hkv", "lens"), [(16, 8, [300, 77, 40]), (7, 1, [6000, 33, 1]), (4, 2, [300, 9000])])
def test_decode_shows_nan_scales(nqt, cuda, kind, what, hq, hkv, lens):
    """A NaN scale of K (0) or V (1) of a block that row 0 holds makes that row and KV head NaN, and nothing else."""

    codes, scales, indptr, indices, last = make_cache8(lens, kind=kind, hkv=hkv, seed=5)
    dev = [t.to(cuda) for t in (_q(len(lens), hq, 128, 6), codes, scales, indptr, indices, last)]
    ws = nqt.decode_paged8_workspace(len(lens), hq, 128, cuda)
    clean = nqt.batch_decode_paged8(*dev, ws)
    for block in (0, 7, (lens[0] - 1) // 16):
        bad = scales.clone()
        bad[int(indices[block]), what, 0, hkv - 1] = float("nan")
        out = nqt.batch_decode_paged8(dev[0], dev[1], bad.to(cuda), *dev[3:], ws)
        first = hq - hq // hkv
        assert out[0, first:].isnan().all()
        assert torch.equal(out[0, :first], clean[0, :first]) and torch.equal(out[1:], clean[1:])


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("what", [0, 1])
@pytest.mark.parametrize(("hq", "hkv", "copies"), [(16, 8, 30), (2, 1, 1), (7, 1, 1)])
def test_prefill_shows_nan_scales_to_those_who_see_them(nqt, cuda, kind, what, hq, hkv, copies):
    """A block with a NaN scale makes the queries NaN that see one of its keys; the others keep every bit.  Many rows
    and few: with and without keys shared by a cluster."""

    lens, chunks = [300] * copies, [200] * copies
    codes, scales, indptr, indices, last = make_cache8(lens, kind=kind, hkv=hkv, d=64, seed=7)
    qo = (200 * torch.arange(copies + 1)).to(torch.int32)
    q = _q(200 * copies, hq, 64, 8)
    dev = [t.to(cuda) for t in (q, codes, scales, qo, indptr, indices, last)]
    clean = nqt.batch_prefill_paged8(*dev)
    first = hq - hq // hkv
    for block in (0, 6, 9, 10, 18):
        bad = scales.clone()
        bad[int(indices[block]), what, 0, hkv - 1] = float("nan")
        out = nqt.batch_prefill_paged8(dev[0], dev[1], bad.to(cuda), *dev[3:])
        seen = max(0, 16 * block - 100)  # the first query that sees the block
        assert out[seen:200, first:].isnan().all()
        assert torch.equal(out[:seen], clean[:seen]) and torch.equal(out[200:], clean[200:])
        assert torch.equal(out[:, :first], clean[:, :first])


# ------------------------------------------------------------------------------------------------ launches and scratch
def test_linear_launches_as_it_says(nqt, cuda):
    """One launch or two by nqt_linear_int8_launches, in the count of launches too; one needs no scratch."""

    lib = nqt._lib.lib()
    for m, k in ((1, 64), (8, 2048), (8, 12288), (8, 12304), (5, 16384), (4, 24592), (3, 24576), (9, 64), (64, 2048)):
        g = torch.Generator().manual_seed(m + k)
        x = torch.randn(m, k, generator=g).to(torch.bfloat16).to(cuda)
        weight = nqt.kernels.Int8Weight(torch.randn(48, k, generator=g).to(torch.bfloat16).to(cuda))
        codes, scale = nqt.kernels.int8_quantize_rows(x)
        nqt._lib.reset_launch_count()
        y = nqt.kernels.linear_int8(x, weight)
        assert nqt._lib.launch_count() == lib.nqt_linear_int8_launches(m, k)
        assert torch.equal(y, nqt.kernels.linear_int8(codes, weight, xscale=scale))
        pitch = (k + 15) // 16 * 16
        out = torch.empty_like(y)
        scratch = torch.full((m * (pitch + 4),), 7, dtype=torch.uint8, device=cuda)
        one = lib.nqt_linear_int8_launches(m, k) == 1
        nqt._lib.call("nqt_linear_int8", x.data_ptr(), k, None if one else scratch.data_ptr(), pitch,
                      None if one else scratch.data_ptr() + m * pitch, weight.data.data_ptr(), weight.data.stride(0),
                      weight.data_scale.data_ptr(), None, out.data_ptr(), 48, m, 48, 48, k, 0,
                      nqt.kernels.device_status(cuda).data_ptr(), nqt._lib.stream_handle(cuda))
        assert torch.equal(out, y)


# ------------------------------------------------------------------------------------------------ special values
def _write_one(nqt, cuda, dc, ds, k, v, offset, hq=2):
    d = k.shape[-1]
    w = torch.ones(d, dtype=torch.bfloat16, device=cuda)
    q = torch.zeros(len(k), hq, d, dtype=torch.bfloat16, device=cuda)
    at = (torch.arange(len(k)) + offset).to(cuda)
    nqt.paired_qk_norm_rope_paged_cache8(q, k.to(cuda), v.to(cuda), w, w, at, EPS, THETA, dc, ds, torch.zeros_like(at), at)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
def test_write_nan_tokens(nqt, cuda, kind, d):
    """A NaN is code 0 (int8) or the NaN code (e4m3), also where the block holds nothing else: a NaN key element makes
    its whole row NaN, so the first token of a block leaves the scale 0."""

    def expect(row, nan):
        raw = row.view(torch.uint8).flatten()
        return ((raw & 0x7F) == 0x7F).all() if nan and kind == "e4m3" else (raw & 0x7F == 0).all()

    ones = torch.ones(1, 1, d, dtype=torch.bfloat16)
    dc = torch.full((1, 2, 16, 1, d), 3).to(oc8.DTYPE[kind]).to(cuda)
    ds = torch.ones(1, 2, 1, 1, device=cuda)
    bad = ones.clone()
    bad[0, 0, 5] = float("nan")
    _write_one(nqt, cuda, dc, ds, bad, ones * float("nan"), 0)
    assert (ds == 0).all() and expect(dc[0, 0, 0, 0], True) and expect(dc[0, 1, 0, 0], True)
    # a later token sets the scale; what was NaN stays so
    _write_one(nqt, cuda, dc, ds, ones, 2 * ones, 1)
    assert (ds > 0).all() and expect(dc[0, 0, 0, 0], True) and expect(dc[0, 1, 0, 0], True)
    back = nqt.read_paged_cache8(dc, ds, torch.tensor([0], device=cuda))
    assert (back[0, 1, 1, 0] == 2).all() and back[0, 0, 1].isfinite().all()
    # and a row of zeros beside a NaN row
    _write_one(nqt, cuda, dc, ds, torch.cat([0 * ones, bad]), torch.cat([0 * ones, bad * 0]), 0)
    assert (ds == 0).all() and expect(dc[0, 0, 0, 0], False) and expect(dc[0, 0, 1, 0], True)
    assert expect(dc[0, 1, 0, 0], False) and expect(dc[0, 1, 1, 0, 5:6], True) and expect(dc[0, 1, 1, 0, :5], False)


# ------------------------------------------------------------------------------------------------ infinities
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_write_infinite_keys_and_values(nqt, cuda, kind):
    """An infinite V is the largest code.  An infinite element of K makes the row's RMS infinite: it and its partner in
    the rotation become NaN, the row's other elements zero; other tokens of the block are not touched."""

    d, top = 128, oc8.TOP[kind]
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(4, 1, d, generator=g).to(torch.bfloat16) for _ in range(2))
    pair = torch.zeros(d, dtype=torch.bool)
    pair[[6, 70]] = True
    dc = [torch.zeros(1, 2, 16, 1, d, dtype=oc8.DTYPE[kind], device=cuda) for _ in range(2)]
    ds = [torch.zeros(1, 2, 1, 1, device=cuda) for _ in range(2)]
    k2 = k.clone()
    k2[2, 0, 70] = float("inf")
    _write_one(nqt, cuda, dc[0], ds[0], k2, v, 0)
    got = dc[0][0, 0, 2, 0].cpu()
    raw = got.view(torch.uint8) & 0x7F
    assert (raw[~pair] == 0).all() and (raw[pair] == (0 if kind == "int8" else 0x7F)).all()
    k2[2] = 0  # contributes nothing to the block's scale, as the infinite row does
    _write_one(nqt, cuda, dc[1], ds[1], k2, v, 0)
    others = torch.tensor([0, 1, 3])
    assert torch.equal(ds[0], ds[1])
    assert torch.equal(dc[0][0, 0].view(torch.uint8)[others.to(cuda)], dc[1][0, 0].view(torch.uint8)[others.to(cuda)])
    v[1, 0, 9], v[1, 0, 10] = float("inf"), -float("inf")
    _write_one(nqt, cuda, dc[0], ds[0], k, v, 0)
    assert numbers(dc[0].cpu())[0, 1, 1, 0, 9:11].tolist() == [top, -top] and ds[0].isfinite().all()
    # a query fares as a key does, in bf16
    q, w = torch.ones(4, 2, d, dtype=torch.bfloat16), torch.ones(d, dtype=torch.bfloat16)
    q[2, 1, 70] = float("inf")
    at = torch.arange(4)
    rot = nqt.paired_qk_norm_rope_paged_cache8(*(t.to(cuda) for t in (q, k, v, w, w, at)), EPS, THETA, dc[0], ds[0],
                                               torch.zeros_like(at).to(cuda), at.to(cuda)).cpu()
    assert rot[2, 1, pair].isnan().all() and (rot[2, 1, ~pair] == 0).all()
    rot[2, 1] = 1
    assert rot.isfinite().all()


# ------------------------------------------------------------------------------------------------ empty rows
def test_quantize_no_rows(nqt, cuda):
    q, s = nqt.kernels.int8_quantize_rows(torch.zeros(0, 40, dtype=torch.bfloat16, device=cuda))
    assert q.shape == (0, 40) and s.shape == (0,)


# ------------------------------------------------------------------------------------------------ single rows
def test_one_row_of_codes_with_any_pitch(nqt, cuda):
    """The pitch of a single row says nothing: a row cut out of a matrix of odd width is taken."""

    g = torch.Generator().manual_seed(4)
    base = torch.randint(-127, 128, (16, 101), generator=g, dtype=torch.int8)
    weight = nqt.kernels.Int8Weight.from_quantized(torch.randint(-127, 128, (20, 33), generator=g, dtype=torch.int8).to(cuda),
                                                   torch.ones(20, device=cuda))
    xs = torch.ones(1, device=cuda)
    x = base.to(cuda)[:1, :33]
    assert x.stride(0) == 101
    want = (base[0, :33].double() @ weight.q.cpu().double().t()).to(torch.float32).to(torch.bfloat16)
    assert torch.equal(nqt.kernels.linear_int8(x, weight, xscale=xs).cpu()[0], want)


# ------------------------------------------------------------------------------------------------ stricter checks
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize(("lens", "chunks"), [([1, 16, 17, 40, 33], [1, 1, 1, 1, 1]), ([37, 300, 16, 129], [37, 45, 16, 1]),
                                              ([20, 30, 64, 700], [3, 15, 50, 640])])
def test_write_each_code(nqt, cuda, kind, lens, chunks):
    """Every code that the call writes or rounds again, by itself: equal to the exact one, or one step beside it where
    the exact quotient lies within fp32's error of the middle between two codes."""

    hq, hkv, d = 16, 8, 128
    codes, scales, indptr, indices, _ = make_cache8(lens, kind=kind, hkv=hkv, d=d, seed=21)
    g = torch.Generator().manual_seed(22)
    pos = torch.cat([torch.arange(n - c, n) for n, c in zip(lens, chunks, strict=True)])
    row = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(chunks))
    pages = indices.long()[indptr.long()[row] + pos // 16]
    offs = pos % 16
    t = len(pos)
    qkv = (torch.randn(t, hq + 2 * hkv, d, generator=g) * torch.exp(torch.randn(t, 1, 1, generator=g))).to(torch.bfloat16)
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(torch.bfloat16) for _ in range(2))
    k, v = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    dq, dc, ds = qkv.to(cuda), codes.to(cuda), scales.to(cuda)
    nqt.paired_qk_norm_rope_paged_cache8(dq[:, :hq], dq[:, hq:hq + hkv], dq[:, hq + hkv:], qw.to(cuda), kw.to(cuda),
                                         pos.to(cuda), EPS, THETA, dc, ds, pages.to(cuda), offs.to(cuda))
    new = torch.stack([oc8.norm_rope(k, kw, pos, EPS, THETA), v.double()], 1)  # [t, 2, hkv, d]
    wc, ws = numbers(codes), scales.double()
    oc8.write(wc, ws, new, pages.tolist(), offs.tolist(), kind)
    gc, gs = numbers(dc.cpu()), ds.cpu().double()

    written = torch.zeros(codes.shape[:3], dtype=torch.bool)
    written[pages, :, offs] = True
    # codes that a growing scale rounded again, and all that the call left: a power of two is exact
    assert torch.equal(gc[~written], wc[~written])
    # A rotated key: 2^-20 of the two elements that it is made of (cos and sin 2^-22; the norm 2^-22 of rsqrt and as much
    # of its sum; four roundings).  The block's largest is at least half of such a pair, so the scale is off by 2^-19.  The
    # scale's division and the quotient's two roundings: 2^-22 in all, for V too.
    plain = torch.sqrt(k.double().square().mean(-1, keepdim=True) + EPS)
    plain = (k.double() / plain * kw.double()).abs()
    pair = plain + plain.roll(d // 2, -1)
    err = torch.stack([2.0**-20 * pair, torch.zeros_like(pair)], 1)
    s = ws[pages, :, offs // 16][..., None]
    x = torch.where(s > 0, new / s.clamp_min(1e-300), 0.0)
    err = err / s.clamp_min(1e-300) + x.abs() * torch.tensor([2.0**-19 + 2.0**-22, 2.0**-22]).view(1, 2, 1, 1).double()
    want, got = oc8.nearest_code(x, kind), gc[pages, :, offs]
    low, high = oc8.nearest_code(x - err, kind), oc8.nearest_code(x + err, kind)
    assert torch.equal(want, wc[pages, :, offs])
    assert ((got >= low) & (got <= high)).all()
    assert ((gs - ws).abs() <= 2.0**-19 * ws).all()


def _step(nqt, case, ws, overlap):
    q, k, v, w, pos, cache, scales, pages, offs, table = case
    rot = nqt.paired_qk_norm_rope_paged_cache8(q, k, v, w, w, pos, EPS, THETA, cache, scales, pages, offs)
    return nqt.batch_decode_paged8(rot, cache, scales, *table, ws, overlap_kv_write=overlap)


def _step_case(cuda, lens, kind, seed):
    codes, scales, indptr, indices, last = make_cache8(lens, kind=kind, seed=seed)
    qkv = _q(len(lens), 32, 128, seed + 1).to(cuda)
    pos = torch.tensor(lens) - 1
    pages = indices.long()[indptr.long()[:-1] + pos // 16]
    w = torch.ones(128, dtype=torch.bfloat16, device=cuda)
    return [qkv[:, :16], qkv[:, 16:24], qkv[:, 24:], w, pos.to(cuda), codes.to(cuda), scales.to(cuda), pages.to(cuda),
            (pos % 16).to(cuda), [t.to(cuda) for t in (indptr, indices, last)]]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_streams_at_once_each_with_its_own_cache(nqt, cuda, kind):
    """Two captured steps on two streams and eager ones on a third, each with a cache and a workspace of its own: every
    result on every round is the one that it gives alone."""

    cases = [_step_case(cuda, lens, kind, s) for s, lens in ((31, [3000, 5, 77, 640]), (33, [64, 4100]), (35, [1900, 9, 48]))]
    start = [(c[5].clone(), c[6].clone()) for c in cases]
    spaces = [nqt.decode_paged8_workspace(len(c[4]), 16, 128, cuda) for c in cases]

    def reset():
        for c, (cache, scales) in zip(cases, start, strict=True):
            c[5].copy_(cache)
            c[6].copy_(scales)
        torch.cuda.synchronize()

    want = []
    for c, ws in zip(cases, spaces, strict=True):
        reset()
        want.append(_step(nqt, c, ws, False))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c, ws in zip(cases[:2], spaces, strict=False):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(nqt, c, ws, True))
        graphs.append(graph)
    for _ in range(10):
        reset()
        for s, graph in zip(streams, graphs, strict=False):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = _step(nqt, cases[2], spaces[2], True)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])


# ------------------------------------------------------------------------------------------------ page sizes and many rows
def _close(got, want, mag):
    over = (got.cpu().double() - want).abs() - attention_tolerance(want, mag)
    assert torch.isfinite(got).all() and over.max() <= 0, f"off by {float(over.max()):.3g} above the tolerance"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("page_size", [48, 80, 112, 240])
def test_page_sizes_that_are_no_power_of_two(nqt, cuda, kind, page_size):
    lens, chunks = [700, 95, 48, 1], [150, 95, 1, 1]
    codes, scales, indptr, indices, last = make_cache8(lens, kind=kind, page_size=page_size, hkv=2, d=64, seed=page_size)
    qo = torch.tensor([0, *torch.tensor(chunks).cumsum(0).tolist()], dtype=torch.int32)
    q = _q(sum(chunks), 6, 64, 3)
    table = [t.to(cuda) for t in (indptr, indices, last)]
    dev = [t.to(cuda) for t in (codes, scales)]
    exact = (numbers(codes), scales.double(), indptr, indices, last)
    nqt.kernels.clear_status(cuda)
    _close(nqt.batch_prefill_paged8(q.to(cuda), *dev, qo.to(cuda), *table), *oc8.attention(q, *exact, qo))
    ends = (qo[1:] - 1).long()
    ws = nqt.decode_paged8_workspace(4, 6, 64, cuda)
    _close(nqt.batch_decode_paged8(q[ends].to(cuda), *dev, *table, ws), *oc8.attention(q[ends], *exact))
    # the write: block by block what it is in pages of 16
    pos = torch.cat([torch.arange(n - c, n) for n, c in zip(lens, chunks, strict=True)])
    row = torch.repeat_interleave(torch.arange(4), torch.tensor(chunks))
    pages, offs = indices.long()[indptr.long()[row] + pos // page_size], pos % page_size
    per = page_size // 16
    small = [codes.view(-1, 2, per, 16, 2, 64).transpose(1, 2).reshape(-1, 2, 16, 2, 64).contiguous().to(cuda),
             scales.transpose(1, 2).reshape(-1, 2, 1, 2).contiguous().to(cuda)]
    k, v = (_q(len(pos), 2, 64, s).to(cuda) for s in (4, 5))
    w = torch.ones(64, dtype=torch.bfloat16, device=cuda)
    for cache, page, off in ((dev, pages, offs), (small, pages * per + offs // 16, offs % 16)):
        nqt.paired_qk_norm_rope_paged_cache8(q.to(cuda), k, v, w, w, pos.to(cuda), EPS, THETA, *cache, page.to(cuda),
                                             off.to(cuda))
    big = dev[0].view(-1, 2, per, 16, 2, 64).transpose(1, 2).reshape(-1, 2, 16, 2, 64)
    assert torch.equal(big.view(torch.uint8), small[0].view(torch.uint8))
    assert torch.equal(dev[1].transpose(1, 2).reshape(-1, 2, 1, 2), small[1])
    got = [nqt.read_paged_cache8(*c, torch.arange(len(c[0]), device=cuda)) for c in (dev, small)]
    assert torch.equal(got[0].view(-1, 2, per, 16, 2, 64).transpose(1, 2).reshape(-1, 2, 16, 2, 64), got[1])
    assert nqt.kernels.read_status(cuda) == 0


def test_decode_as_many_rows_as_a_launch_takes(nqt, cuda):
    lens = torch.randint(0, 24, (8192,), generator=torch.Generator().manual_seed(1)).tolist()
    lens[77] = 3000
    codes, scales, indptr, indices, last = make_cache8(lens, hkv=1, d=64, seed=2)
    q = _q(8192, 2, 64, 3)
    dev = [t.to(cuda) for t in (q, codes, scales, indptr, indices, last)]
    ws = nqt.decode_paged8_workspace(8192, 2, 64, cuda)
    first = nqt.batch_decode_paged8(*dev, ws)
    assert torch.equal(first, nqt.batch_decode_paged8(*dev, ws))
    _close(first, *oc8.attention(q, numbers(codes), scales.double(), indptr, indices, last))
    with pytest.raises(nqt._lib.NqtError):
        nqt.batch_decode_paged8(dev[0].repeat(2, 1, 1), *dev[1:3], torch.zeros(16385, dtype=torch.int32, device=cuda),
                                dev[4], torch.ones(16384, dtype=torch.int32, device=cuda), ws)
