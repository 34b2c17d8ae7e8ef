"""GPU: the 8-bit operators where a call is allowed and easily forgotten: rows that many CTAs share among few KV heads,
pools behind 32-bit offsets, other streams, two captured graphs, a decode behind its own write."""

from __future__ import annotations

import pytest
import torch

from oracle import cache8 as oc8
from tests._cache8 import attention_tolerance, make_cache8, numbers

pytestmark = pytest.mark.gpu

EPS, THETA = 1e-6, 1.0e6


def _q(rows, hq, d, seed):
    return torch.randn(rows, hq, d, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def _close(got, want, mag):
    over = (got.cpu().double() - want).abs() - attention_tolerance(want, mag)
    assert torch.isfinite(got).all() and over.max() <= 0, f"off by {float(over.max()):.3g} above the tolerance"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize(("hq", "hkv", "d", "lens"), [(14, 2, 64, [20000, 5, 7001]), (8, 1, 128, [30000]),
                                                      (7, 1, 64, [9000, 0, 33]), (16, 2, 128, [16001, 40])])
def test_decode_rows_shared_by_many_ctas(nqt, cuda, kind, hq, hkv, d, lens):
    codes, scales, indptr, indices, last = make_cache8(lens, kind=kind, hkv=hkv, d=d, seed=len(lens) + hq)
    q = _q(len(lens), hq, d, 3)
    want, mag = oc8.attention(q, numbers(codes), scales.double(), indptr, indices, last)
    dev = [t.to(cuda) for t in (q, codes, scales, indptr, indices, last)]
    ws = nqt.decode_paged8_workspace(len(lens), hq, d, cuda)
    nqt.kernels.clear_status(cuda)
    first = nqt.batch_decode_paged8(*dev, ws)
    for _ in range(10):
        assert torch.equal(nqt.batch_decode_paged8(*dev, ws), first)
    assert nqt.kernels.read_status(cuda) == 0
    _close(first, want, mag)


def test_decode_short_wait_with_shared_heads(nqt, cuda):
    g = torch.Generator().manual_seed(17)
    pages = 40000
    codes = torch.randint(-127, 128, (pages, 2, 64, 2, 64), dtype=torch.int8, device=cuda)
    scales = torch.full((pages, 2, 4, 2), 0.01, device=cuda)
    indptr = torch.tensor([0, 15000, 15001, pages], dtype=torch.int32, device=cuda)
    indices = torch.randperm(pages, generator=g).to(torch.int32).to(cuda)
    last = torch.tensor([64, 3, 17], dtype=torch.int32, device=cuda)
    args = (_q(3, 14, 64, 18).to(cuda), codes, scales, indptr, indices, last,
            nqt.decode_paged8_workspace(3, 14, 64, cuda))
    want = nqt.batch_decode_paged8(*args)
    nqt.kernels.clear_status(cuda)
    for _ in range(3):
        nqt.batch_decode_paged8(*args, short_wait=True)
    assert nqt.kernels.read_status(cuda) & nqt._lib.NQT_DEV_TIMEOUT
    nqt.kernels.clear_status(cuda)
    for _ in range(2):
        assert torch.equal(nqt.batch_decode_paged8(*args), want)
    assert nqt.kernels.read_status(cuda) == 0


def _step(nqt, q, k, v, w, pos, cache, scales, pages, offs, table, ws, overlap):
    rot = nqt.paired_qk_norm_rope_paged_cache8(q, k, v, w, w, pos, EPS, THETA, cache, scales, pages, offs)
    return nqt.batch_decode_paged8(rot, cache, scales, *table, ws, overlap_kv_write=overlap)


def _step_inputs(cuda, lens, kind, seed):
    """A decode step of rows that have ``lens`` tokens with the new one."""

    codes, scales, indptr, indices, last = make_cache8(lens, kind=kind, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    n = len(lens)
    qkv = torch.randn(n, 32, 128, generator=g).to(torch.bfloat16).to(cuda)
    pos = torch.tensor(lens) - 1
    pages = indices.long()[indptr.long()[:-1] + pos // 16]
    w = torch.ones(128, dtype=torch.bfloat16, device=cuda)
    args = [qkv[:, :16], qkv[:, 16:24], qkv[:, 24:], w, pos.to(cuda), codes.to(cuda), scales.to(cuda), pages.to(cuda),
            (pos % 16).to(cuda), [t.to(cuda) for t in (indptr, indices, last)]]
    return args


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_decode_behind_its_own_write(nqt, cuda, kind):
    """With NQT_DECODE_OVERLAP_KV_WRITE the result is that of the two calls apart, launch after launch."""

    args = _step_inputs(cuda, [1, 16, 17, 2000, 33, 513, 48, 900], kind, 5)
    cache, scales = args[5].clone(), args[6].clone()
    ws = nqt.decode_paged8_workspace(8, 16, 128, cuda)
    want = _step(nqt, *args, ws, False)
    after = args[5].clone(), args[6].clone()
    for _ in range(30):
        args[5].copy_(cache)
        args[6].copy_(scales)
        got = _step(nqt, *args, ws, True)
        assert torch.equal(got, want)
        assert torch.equal(args[5].view(torch.uint8), after[0].view(torch.uint8)) and torch.equal(args[6], after[1])


def test_streams_and_graphs_run_apart(nqt, cuda):
    """Two captured steps with a workspace each, replayed on two streams at once, and eager calls on a third."""

    cases = [_step_inputs(cuda, lens, "int8", s) for s, lens in ((7, [3000, 5, 77, 640]), (11, [64, 4100]))]
    spaces = [nqt.decode_paged8_workspace(len(c[4]), 16, 128, cuda) for c in cases]
    weight = nqt.kernels.Int8Weight(torch.randn(512, 2048, device=cuda).to(torch.bfloat16))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def layer(c, ws, overlap):
        return nqt.kernels.linear_int8(_step(nqt, *c, ws, overlap).view(len(c[4]), 2048), weight)

    want = []
    with torch.cuda.stream(side):
        for c, ws in zip(cases, spaces, strict=True):
            want.append(layer(c, ws, False))
    side.synchronize()
    graphs, outs = [], []
    for c, ws in zip(cases, spaces, strict=True):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(layer(c, ws, True))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    third = nqt.decode_paged8_workspace(4, 16, 128, cuda)
    for _ in range(20):
        for s, graph in zip(streams, graphs, strict=True):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(side):
            eager = nqt.batch_decode_paged8(cases[0][0].contiguous(), cases[0][5], cases[0][6], *cases[0][9], third)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want, strict=True)) and torch.isfinite(eager).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_pages_behind_32_bit_offsets(nqt, cuda, kind):
    """A pool of 4.9 GB, used at its far end by the write, the page read, decode and prefill."""

    pages, n = 150_000, 45
    cache = torch.zeros(pages, 2, 16, 8, 128, dtype=oc8.DTYPE[kind], device=cuda)
    scales = torch.zeros(pages, 2, 1, 8, device=cuda)
    ids = torch.tensor([pages - 1, pages - 3, pages - 2], dtype=torch.int32)
    pos = torch.arange(n)
    where = ids.long()[pos // 16]
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(n, 32, 128, generator=g).to(torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16)
    dq = qkv.to(cuda)
    rot = nqt.paired_qk_norm_rope_paged_cache8(dq[:, :16], dq[:, 16:24], dq[:, 24:], w.to(cuda), w.to(cuda), pos.to(cuda),
                                               EPS, THETA, cache, scales, where.to(cuda), (pos % 16).to(cuda))
    got = nqt.read_paged_cache8(cache, scales, ids.long().to(cuda)).cpu().double()
    assert (nqt.read_paged_cache8(cache, scales, torch.tensor([0, 1], device=cuda)) == 0).all()
    k = oc8.norm_rope(qkv[:, 16:24], w, pos, EPS, THETA)
    new = torch.stack([k, qkv[:, 24:].double()], 1)  # [n, 2, 8, 128]
    back = got.transpose(1, 2).reshape(48, 2, 8, 128)[:n]
    # a block's scale is amax / top: half a step of it (int8), or e4m3's half step 2^-4 of the value and half the
    # smallest step 2^-10 of the scale; then bf16's 2^-8
    step = torch.stack([new[i * 16:(i + 1) * 16].abs().amax(dim=(0, 3)) for i in range(3)]) / oc8.TOP[kind]
    step = step.repeat_interleave(16, 0)[:n, :, :, None]
    bound = step * 0.5 if kind == "int8" else new.abs() * 2.0**-4 + step * 2.0**-10
    assert ((back - new).abs() <= bound * (1 + 2.0**-8) + new.abs() * 2.0**-8 + 2.0**-16).all()

    table = [torch.tensor([0, 3], dtype=torch.int32), ids, torch.tensor([n - 32], dtype=torch.int32)]
    small = [t.cpu()[pages - 4:] for t in (cache, scales)]
    args = (numbers(small[0]), small[1].double(), table[0], ids - (pages - 4), table[2])
    dt = [t.to(cuda) for t in table]
    ws = nqt.decode_paged8_workspace(1, 16, 128, cuda)
    _close(nqt.batch_decode_paged8(rot[-1:], cache, scales, *dt, ws), *oc8.attention(rot[-1:].cpu(), *args))
    qo = torch.tensor([0, n], dtype=torch.int32)
    _close(nqt.batch_prefill_paged8(rot, cache, scales, qo.to(cuda), *dt), *oc8.attention(rot.cpu(), *args, qo))


def test_products_behind_32_bit_offsets(nqt, cuda):
    """More outputs than 2^31, and the last rows of them."""

    m, n, k = 270_000, 8_000, 48
    g = torch.Generator().manual_seed(2)
    wq = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    weight = nqt.kernels.Int8Weight.from_quantized(wq.to(cuda), torch.full((n,), 0.01, device=cuda))
    x = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8).to(cuda)
    xs = torch.full((m,), 0.5, device=cuda)
    out = nqt.kernels.linear_int8(x, weight, xscale=xs)
    for rows in (slice(0, 3), slice(m - 130, m)):
        want = x[rows].cpu().double() @ wq.double().t() * (0.5 * float(torch.tensor(0.01)))
        assert ((out[rows].cpu().double() - want).abs() <= (2.0**-8 + 2.0**-21) * want.abs()).all()


def test_broadcast_queries(nqt, cuda):
    """One query for every row, or one head for all, without a copy in memory."""

    codes, scales, indptr, indices, last = make_cache8([40, 33, 90], seed=21)
    dev = [t.to(cuda) for t in (codes, scales, indptr, indices, last)]
    ws = nqt.decode_paged8_workspace(3, 16, 128, cuda)
    qo = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    for q in (_q(1, 16, 128, 22).expand(3, 16, 128), _q(3, 1, 128, 23).expand(3, 16, 128)):
        want = oc8.attention(q, numbers(codes), scales.double(), indptr, indices, last)
        base = q.to(cuda)[:1, :, :] if q.stride(0) == 0 else q.to(cuda)[:, :1]
        dq = base.expand(3, 16, 128)
        assert 0 in dq.stride()
        _close(nqt.batch_decode_paged8(dq, *dev, ws), *want)
        _close(nqt.batch_prefill_paged8(dq, *dev[:2], qo.to(cuda), *dev[2:]), *want)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 6, 7, 8])
def test_prefill_groups_over_long_keys(nqt, cuda, group):
    """Every group size, tiles with rows left over, keys beyond one stage of the rings, chunks that end inside a tile."""

    chunks, lens = [150, 1, 61], [400, 1000, 61]
    codes, scales, indptr, indices, last = make_cache8(lens, kind="e4m3", hkv=2, d=128, page_size=32, seed=group)
    q = _q(sum(chunks), 2 * group, 128, 31)
    qo = torch.tensor([0, 150, 151, 212], dtype=torch.int32)
    want = oc8.attention(q, numbers(codes), scales.double(), indptr, indices, last, qo)
    dev = [t.to(cuda) for t in (q, codes, scales, qo, indptr, indices, last)]
    first = nqt.batch_prefill_paged8(*dev)
    assert torch.equal(first, nqt.batch_prefill_paged8(*dev))
    _close(first, *want)


def test_prefill_more_work_than_the_gpu_holds_at_once(nqt, cuda):
    """Far more tiles than SMs, of very different costs: CTAs take over one another's work; rows without queries or keys
    among them.  Equal from launch to launch, with tokens behind the last chunk left as they were."""

    g = torch.Generator().manual_seed(41)
    chunks = [int(n) for n in torch.randint(0, 260, (48,), generator=g)] + [0, 3, 700, 0]
    lens = [n + int(e) for n, e in zip(chunks, torch.randint(0, 200, (52,), generator=g), strict=True)]
    lens[5], chunks[7] = 0, 0  # queries without keys, keys without queries
    codes, scales, indptr, indices, last = make_cache8(lens, kind="int8", hkv=8, d=64, seed=43)
    total = sum(chunks)
    q = _q(total + 5, 8, 64, 44)
    qo = torch.tensor([0, *torch.tensor(chunks).cumsum(0).tolist()], dtype=torch.int32)
    dev = [t.to(cuda) for t in (q, codes, scales, qo, indptr, indices, last)]
    out = torch.full((total + 5, 8, 64), 7.0, dtype=torch.bfloat16, device=cuda)
    nqt.kernels.clear_status(cuda)
    first = nqt.batch_prefill_paged8(*dev, out=out).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nqt.batch_prefill_paged8(*dev, out=out)
    for _ in range(20):
        out[:total] = 0
        graph.replay()
        assert torch.equal(out, first)
    assert nqt.kernels.read_status(cuda) == 0 and (first[total:] == 7).all()
    want, mag = oc8.attention(q[:total], numbers(codes), scales.double(), indptr, indices, last, qo)
    _close(first[:total], want, mag)


@pytest.mark.parametrize(("rows", "lo", "hi"), [(3, 0, 40), (30, 1, 600), (64, 20, 120), (64, 900, 3100), (110, 0, 90),
                                                (130, 1, 50), (255, 0, 40), (256, 1, 30)])
def test_decode_rows_cut_one_by_one_or_across(nqt, cuda, rows, lo, hi):
    """Row counts and lengths on both sides of the rules that decide how the tiles are cut."""

    lens = torch.randint(lo, hi, (rows,), generator=torch.Generator().manual_seed(rows + hi)).tolist()
    codes, scales, indptr, indices, last = make_cache8(lens, hkv=2, d=64, seed=rows)
    q = _q(rows, 4, 64, 9)
    want = oc8.attention(q, numbers(codes), scales.double(), indptr, indices, last)
    dev = [t.to(cuda) for t in (q, codes, scales, indptr, indices, last)]
    ws = nqt.decode_paged8_workspace(rows, 4, 64, cuda)
    first = nqt.batch_decode_paged8(*dev, ws)
    assert torch.equal(first, nqt.batch_decode_paged8(*dev, ws))
    _close(first, *want)
