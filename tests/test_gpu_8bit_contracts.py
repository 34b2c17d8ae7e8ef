"""GPU: what the 8-bit operators' contracts promise beyond single calls: one workspace for calls of every shape, exact
codes at ties, NaN scales and codes that stay visible to those who see them and to nobody else."""

from __future__ import annotations

import pytest
import torch

from tests._cache8 import make_cache8

pytestmark = pytest.mark.gpu


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
