"""64-bit CPU restatement of the 8-bit paged KV cache: its codes, the write's scale rule, and attention over it.

A cache is held here as float64 numbers: ``codes`` [pages, 2, P, Hkv, D] (the number a code is, before its
scale) and ``scales`` [pages, 2, P / 16, Hkv]."""

from __future__ import annotations

import math

import torch

BLOCK = 16
TOP = {"int8": 127.0, "e4m3": 448.0}
DTYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def nearest_code(x: torch.Tensor, kind: str) -> torch.Tensor:
    """The nearest code (ties to even) as a number, saturating."""

    x = x.clamp(-TOP[kind], TOP[kind])
    if kind == "int8":
        return x.round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0**-6))) - 3)
    return (x / step).round() * step


def norm_rope(x: torch.Tensor, weight: torch.Tensor, positions: torch.Tensor, eps: float, theta: float) -> torch.Tensor:
    """RMSNorm per head then the split-half rotation, float64.  x [T, H, D]."""

    x = x.double()
    x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    h = x.shape[-1] // 2
    angle = positions.double()[:, None, None] * torch.exp(-math.log(theta) * torch.arange(h).double() / h)
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)


def groups(pages: list[int], offsets: list[int]) -> list[tuple[int, int]]:
    """(first token, count) of the runs of tokens that one write treats together: one page and block, rising
    offsets."""

    out: list[tuple[int, int]] = []
    for t in range(len(pages)):
        if t and pages[t] == pages[t - 1] and offsets[t] // BLOCK == offsets[t - 1] // BLOCK \
                and offsets[t] > offsets[t - 1]:
            out[-1] = (out[-1][0], out[-1][1] + 1)
        else:
            out.append((t, 1))
    return out


def write(codes: torch.Tensor, scales: torch.Tensor, new: torch.Tensor, pages: list[int], offsets: list[int],
          kind: str) -> None:
    """In place: the tokens ``new`` [T, 2, Hkv, D] at (page, offset), by the scale rule of the write."""

    for t, n in groups(pages, offsets):
        p, b, o = pages[t], offsets[t] // BLOCK, offsets[t] % BLOCK
        part = new[t:t + n].double()  # [n, 2, Hkv, D]
        need = part.abs().amax(dim=(0, 3)) / TOP[kind]
        old = scales[p, :, b].clone()
        if o == 0:
            to = need
        else:
            k = torch.ceil(torch.log2((need / old.clamp_min(1e-300)).clamp_min(1.0)))
            to = torch.where(old > 0, old * torch.exp2(k), need)
            block = codes[p, :, b * BLOCK:b * BLOCK + o]  # [2, o, Hkv, D]
            ratio = torch.where((to > 0) & (to != old), old / to.clamp_min(1e-300), 1.0)
            block.copy_(nearest_code(block * ratio[:, None, :, None], kind))
        scales[p, :, b] = to
        for i in range(n):
            x = part[i] / to.clamp_min(1e-300)[..., None]
            codes[p, :, offsets[t + i]] = nearest_code(torch.where(to[..., None] > 0, x, 0.0), kind)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """code * scale, [pages, 2, P, Hkv, D]."""

    return codes * scales.repeat_interleave(BLOCK, dim=2)[..., None]


def attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, indptr, indices, last, qo_indptr=None,
              sm_scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of ragged query rows (one per row without ``qo_indptr``) over the cached tokens.  Returns
    (out, err), float64 [T, Hq, D]: err is the same average of |v| plus 2^-22 of (largest visible scale of v) times
    the sum of the visible |codes|, so that 2^-11 err bounds what it costs to round every weight p c (probability
    times value scale) to 11 bits or, where it is tiny, to a multiple of 2^-32 of a weight that occurs: 2^-33 of it
    for each code, divided by a sum of probabilities that is at least that weight's."""

    tokens, hq, d = q.shape
    hkv, page_size = codes.shape[3], codes.shape[2]
    scale = d**-0.5 if sm_scale is None else sm_scale
    out, mag = torch.zeros(tokens, hq, d, dtype=torch.float64), torch.zeros(tokens, hq, d, dtype=torch.float64)
    rows = len(indptr) - 1
    for r in range(rows):
        q0, q1 = (r, r + 1) if qo_indptr is None else (int(qo_indptr[r]), int(qo_indptr[r + 1]))
        ids = indices[int(indptr[r]):int(indptr[r + 1])].long()
        if len(ids) == 0 or q1 <= q0:
            continue
        n = (len(ids) - 1) * page_size + min(max(int(last[r]), 1), page_size)
        kv = values(codes[ids], scales[ids]).transpose(0, 1).reshape(2, -1, hkv, d)[:, :n]
        raw = codes[ids][:, 1].reshape(-1, hkv, d)[:n].abs()
        top = scales[ids][:, 1].repeat_interleave(BLOCK, dim=1).reshape(-1, hkv)[:n].amax(0)
        lim = n - (q1 - q0) + torch.arange(q1 - q0)
        hidden = torch.arange(n)[None] > lim[:, None]
        for h in range(hq):
            k, v = kv[0, :, h // (hq // hkv)], kv[1, :, h // (hq // hkv)]
            s = (q[q0:q1, h].double() @ k.t() * scale).masked_fill(hidden, -math.inf)
            p = torch.nan_to_num(s.softmax(-1)) if bool((lim < 0).any()) else s.softmax(-1)
            out[q0:q1, h] = p @ v
            g = h // (hq // hkv)
            mag[q0:q1, h] = p @ v.abs() + 2.0**-22 * top[g] * ((~hidden).double() @ raw[:, g])
    return out, mag
