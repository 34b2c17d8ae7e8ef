"""Seeded 8-bit paged caches shared by the GPU tests (CPU tensors; tests move them)."""

from __future__ import annotations

import torch

from oracle import cache8 as oc8


def numbers(codes: torch.Tensor) -> torch.Tensor:
    """Stored codes as float64 numbers."""

    return codes.to(torch.float32).double()


def make_cache8(lens, *, kind="int8", page_size=16, hkv=8, d=128, extra_pages=5, seed=0, spread=1.0):
    """A cache quantised from N(0, 1) with block magnitudes spread by e^(spread N(0, 1)); each row's pages
    scattered.  A length of zero has no page.

    Returns (codes, scales f32, indptr, indices, last_page_len)."""

    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page_size) for n in lens]
    total = sum(need) + extra_pages
    nb = page_size // oc8.BLOCK
    x = torch.randn(total, 2, nb, oc8.BLOCK, hkv, d, generator=g)
    x *= torch.exp(spread * torch.randn(total, 2, nb, 1, hkv, 1, generator=g))
    scales = x.abs().amax(dim=(3, 5)) / oc8.TOP[kind]
    x = (x / scales[:, :, :, None, :, None]).view(total, 2, page_size, hkv, d)
    codes = (x.round() if kind == "int8" else x).to(oc8.DTYPE[kind])
    perm = torch.randperm(total, generator=g).tolist()
    indptr, indices, last = [0], [], []
    for n, p in zip(lens, need, strict=True):
        indices.extend(perm[:p])
        perm = perm[p:]
        indptr.append(len(indices))
        last.append(n - (p - 1) * page_size if p else 0)
    i32 = torch.int32
    return (codes, scales, torch.tensor(indptr, dtype=i32), torch.tensor(indices, dtype=i32),
            torch.tensor(last, dtype=i32))


def poison_dead_tokens(codes, scales, indptr, indices, last):
    """What belongs to no token gets the worst codes (NaN codes for e4m3): behind each row's end and in the pages
    of nobody; scales of whole dead blocks become NaN."""

    raw = codes.view(torch.uint8)
    worst = 0x7F if codes.dtype == torch.float8_e4m3fn else 0x80
    page_size = codes.shape[2]
    used = set(indices.tolist())
    for p in range(codes.shape[0]):
        if p not in used:
            raw[p] = worst
            scales[p] = float("nan")
    for r in range(len(indptr) - 1):
        if indptr[r + 1] > indptr[r]:
            p, ll = int(indices[indptr[r + 1] - 1]), int(last[r])
            raw[p, :, ll:] = worst
            scales[p, :, -(-ll // oc8.BLOCK):] = float("nan")
    assert page_size >= oc8.BLOCK


def attention_tolerance(want, mag):
    """One rounding to bf16 (2^-8 of the value), and under the average: weights rounded to fp16 (finfo.eps / 2 =
    2^-11 each; both kernels hold them 2^8 above their value against a reference that some weight reaches, and fp16
    rounds what is under 2^-14 by up to 2^-25) with fp32 scores, exponentials and sums (2^-18)."""

    return 2.0**-8 * want.abs() + (2.0**-11 + 2.0**-18) * mag + 1e-30
