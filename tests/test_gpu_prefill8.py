"""GPU: ragged causal prefill attention over the 8-bit paged KV cache, against 64-bit arithmetic."""

from __future__ import annotations

import pytest
import torch

from oracle import cache8 as oc8
from tests._cache8 import attention_tolerance, make_cache8, numbers, poison_dead_tokens

pytestmark = pytest.mark.gpu


def _case(lens, qlens, *, kind="int8", page_size=16, hq=16, hkv=8, d=128, seed=0, spread=1.0, q_gain=1.0):
    codes, scales, indptr, indices, last = make_cache8(lens, kind=kind, page_size=page_size, hkv=hkv, d=d, seed=seed,
                                                       spread=spread)
    qo = torch.tensor([0, *torch.tensor(qlens).cumsum(0).tolist()], dtype=torch.int32)
    q = (torch.randn(int(qo[-1]), hq, d, generator=torch.Generator().manual_seed(seed + 1)) * q_gain).to(torch.bfloat16)
    return q, codes, scales, qo, indptr, indices, last


def _check(nqt, cuda, case, *, sm_scale=None, poison=True):
    q, codes, scales, qo, indptr, indices, last = case
    want, mag = oc8.attention(q, numbers(codes), scales.double(), indptr, indices, last, qo, sm_scale)
    if poison:
        poison_dead_tokens(codes, scales, indptr, indices, last)
    nqt.kernels.clear_status(cuda)
    out = nqt.batch_prefill_paged8(*(t.to(cuda) for t in case), sm_scale=sm_scale)
    torch.cuda.synchronize()
    assert nqt.kernels.read_status(cuda) == 0
    got = out.cpu()
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() - attention_tolerance(want, mag)
    assert over.max() <= 0, f"off by {over.max():.3g} above the tolerance"
    return got


LENGTHS = [
    ([1], [1]),
    ([37, 1, 300, 128], [37, 1, 45, 128]),
    ([16, 17, 64, 65], [1, 17, 33, 2]),
    ([1024, 700], [1024, 500]),
    ([2500], [3]),
    ([129, 5, 640, 63, 64, 300, 2, 77, 90, 18, 450], [129, 5, 200, 63, 64, 300, 2, 70, 1, 18, 130]),
]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize(("lens", "qlens"), LENGTHS)
def test_prefill_lengths(nqt, cuda, kind, lens, qlens):
    _check(nqt, cuda, _case(lens, qlens, kind=kind))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize(("hq", "hkv", "d"), [(16, 8, 64), (8, 8, 128), (14, 2, 64), (32, 4, 128), (6, 2, 128),
                                              (5, 1, 64), (24, 3, 128), (1, 1, 128)])
def test_prefill_head_layouts(nqt, cuda, kind, hq, hkv, d):
    _check(nqt, cuda, _case([200, 333, 9], [200, 100, 2], kind=kind, hq=hq, hkv=hkv, d=d, seed=3))


@pytest.mark.parametrize("page_size", [32, 64, 256])
def test_prefill_page_sizes(nqt, cuda, page_size):
    _check(nqt, cuda, _case([500, 31, 257], [300, 31, 60], page_size=page_size, seed=4))


def test_prefill_keys_shared_by_a_cluster(nqt, cuda):
    """Few query tiles over long caches: one to eight CTAs share the keys of a pair of tiles."""

    _check(nqt, cuda, _case([6000], [20], hq=2, hkv=1, seed=5))
    _check(nqt, cuda, _case([3000, 40], [150, 3], hq=4, hkv=2, d=64, kind="e4m3", seed=6))
    _check(nqt, cuda, _case([4100], [333], hq=7, hkv=1, seed=7))
    _check(nqt, cuda, _case([130, 1], [130, 1], hq=2, hkv=2, seed=8))


def test_prefill_empty_rows_and_rows_without_keys(nqt, cuda):
    """Rows without queries, rows without pages, and queries that lie before the first key."""

    got = _check(nqt, cuda, _case([0, 50, 0, 20, 3], [7, 20, 0, 0, 5], hq=4, hkv=2, seed=9))
    assert (got[:7] == 0).all() and (got[27:29] == 0).all() and (got[29:] != 0).any()
    _check(nqt, cuda, _case([0, 0], [300, 1], hq=16, hkv=8, seed=10))


def test_prefill_many_rows(nqt, cuda):
    """More rows than are put in order, with empty ones among them."""

    g = torch.Generator().manual_seed(11)
    q = torch.randint(0, 4, (700,), generator=g)
    kv = q + torch.randint(0, 30, (700,), generator=g)
    _check(nqt, cuda, _case(kv.tolist(), q.tolist(), hq=2, hkv=1, d=64, seed=12))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_prefill_peaked_scores_and_wide_scales(nqt, cuda, kind):
    _check(nqt, cuda, _case([400, 900], [400, 300], kind=kind, seed=13, q_gain=30.0))
    _check(nqt, cuda, _case([400, 900], [400, 300], kind=kind, seed=14, spread=6.0, q_gain=1e-3))


def test_prefill_zero_scales(nqt, cuda):
    case = _case([300], [200], seed=15)
    case[2][case[5][2:6].long()] = 0.0
    _check(nqt, cuda, case)


def test_prefill_strides_and_leftover_tokens(nqt, cuda):
    """Strided and oddly aligned q and out; tokens behind the last row are left as they are."""

    lens, qlens = [300, 40], [150, 40]
    q, codes, scales, qo, indptr, indices, last = _case(lens, qlens, seed=16)
    want, mag = oc8.attention(q, numbers(codes), scales.double(), indptr, indices, last, qo)
    dev = [t.to(cuda) for t in (codes, scales, qo, indptr, indices, last)]
    for lead, width in ((0, 128), (8, 144), (1, 131)):
        wq = torch.zeros(200, 16, width, dtype=torch.bfloat16, device=cuda)
        wq[:190, :, lead:lead + 128] = q.to(cuda)
        wo = torch.full((200, 16, width), 7.0, dtype=torch.bfloat16, device=cuda)
        nqt.batch_prefill_paged8(wq[:, :, lead:lead + 128], *dev, out=wo[:, :, lead:lead + 128])
        got = wo[:190, :, lead:lead + 128].cpu().double()
        assert ((got - want).abs() <= attention_tolerance(want, mag)).all()
        assert (wo[190:] == 7).all() and (wo[:, :, :lead] == 7).all() and (wo[:, :, lead + 128:] == 7).all()


def test_prefill_graph_replay_is_deterministic(nqt, cuda):
    case = _case([2000, 30], [64, 30], hq=4, hkv=2, seed=17)
    dev = [t.to(cuda) for t in case]
    want = nqt.batch_prefill_paged8(*dev)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nqt.batch_prefill_paged8(*dev, out=out)
    for _ in range(10):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_prefill_bad_page_reports_and_reads_zeros(nqt, cuda):
    q, codes, scales, qo, indptr, indices, last = _case([100, 40], [100, 10], seed=18)
    indices[1] = -3
    nqt.kernels.clear_status(cuda)
    out = nqt.batch_prefill_paged8(*(t.to(cuda) for t in (q, codes, scales, qo, indptr, indices, last)))
    assert nqt.kernels.read_status(cuda) & 0x1
    assert torch.isfinite(out.float()).all()
    nqt.kernels.clear_status(cuda)
