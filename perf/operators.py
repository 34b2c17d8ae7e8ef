"""The 8-bit serving operators as cases: attention over a paged KV cache held in 8 bits (decode and chunked
prefill), the write into that cache, and the W8A8 integer projection.

`run` computes each in plain torch (fp32, angles in 64 bits) where `own` is false, and through the package's
public functions where it is true.

The 8-bit cache of one layer is `cache` [pages, 2, P, Hkv, D] (int8 or e4m3; kind 0 = K, 1 = V) with one fp32
scale for every 16 tokens of a page and KV head, `scales` [pages, 2, P / 16, Hkv]; an element stands for
code * scale.
"""

import importlib
import math
import random

import torch

own = False

BLOCK = 16  # tokens that share a scale
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
EPS, THETA = 1e-6, 1.0e6


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one request in its first second of audio: nothing but latency
        dict(name="decode_first_frames", op="decode", cache="int8", rows=1, lo=300, hi=300, hq=16, hkv=8, d=128, page=16,
             ragged=1),
        # the talker's decode batch: 64 requests of up to 2048 frames
        dict(name="decode_talker_64", op="decode", cache="int8", rows=64, lo=64, hi=2048, hq=16, hkv=8, d=128, page=16,
             ragged=2),
        # the decode rows of a full continuous batch
        dict(name="decode_batch_240", op="decode", cache="e4m3", rows=240, lo=32, hi=4096, hq=16, hkv=8, d=128, page=16,
             ragged=3),
        # few requests with very long caches, an odd GQA group and wide pages: the work has to be split along the cache
        dict(name="decode_long_group7", op="decode", cache="e4m3", rows=5, lo=20001, hi=98765, hq=14, hkv=2, d=64,
             page=64, ragged=4),
        # first chunks of eight prompts, ragged
        dict(name="prefill_chunks", op="prefill", cache="int8", rows=8, qlo=128, qhi=1024, clo=0, chi=0, hq=16, hkv=8,
             d=128, page=16, ragged=5),
        # a late chunk of two long prompts: most keys come from the cache
        dict(name="prefill_late_chunk", op="prefill", cache="e4m3", rows=2, qlo=301, qhi=515, clo=9000, chi=16001, hq=16,
             hkv=8, d=128, page=32, ragged=6),
        # eight whole prompts at once
        dict(name="prefill_long_prompts", op="prefill", cache="int8", rows=8, qlo=2048, qhi=2048, clo=0, chi=0, hq=16,
             hkv=8, d=128, page=16, ragged=7),
        # the write of a decode step: one token for each of 64 requests, most into a block that has tokens already
        dict(name="append_decode_64", op="append", cache="int8", rows=64, qlo=1, qhi=1, clo=64, chi=2047, hq=16, hkv=8,
             d=128, page=16, ragged=8),
        # the write of a prefill: eight ragged chunks behind ragged contexts
        dict(name="append_chunks", op="append", cache="e4m3", rows=8, qlo=128, qhi=1024, clo=0, chi=333, hq=16, hkv=8,
             d=128, page=16, ragged=9),
        # the attention output projection of a single request, with a bias
        dict(name="linear_o_1", op="linear", m=1, n=2048, k=2048, bias=True, gate_up=False),
        # the talker's gate/up with SwiGLU for a decode batch
        dict(name="linear_gate_up_64", op="linear", m=64, n=12288, k=2048, bias=False, gate_up=True),
        # the down projection over a prefill batch of odd length
        dict(name="linear_down_4613", op="linear", m=4613, n=2048, k=6144, bias=False, gate_up=False),
    ]


HEADS = [(16, 8), (8, 8), (14, 2), (32, 4), (6, 2), (5, 1), (12, 4), (24, 3)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prefill", "append", "linear", "linear"])
    if op == "linear":
        while True:
            m, k = _log(rng, 1, 8192), _log(rng, 16, 8192)
            gate_up = rng.random() < 0.4
            n = 2 * _log(rng, 8, 6144) if gate_up else _log(rng, 1, 12288)
            if m * n * k <= 4613 * 2048 * 6144:
                return dict(op=op, m=m, n=n, k=k, bias=not gate_up and rng.random() < 0.5, gate_up=gate_up)
    while True:
        hq, hkv = rng.choice(HEADS)
        d, page = rng.choice([64, 128]), rng.choice([16, 16, 32, 64])
        case = dict(op=op, cache=rng.choice(["int8", "e4m3"]), hq=hq, hkv=hkv, d=d, page=page,
                    ragged=rng.randrange(1 << 30))
        if op == "decode":
            rows, hi = _log(rng, 1, 256), _log(rng, 1, 131072)
            lo = _log(rng, 1, hi) if rng.random() < 0.8 else 0  # a row may hold nothing yet
            # the plain form's time goes with the padded batch of keys, the kernel's with the real one
            if rows * hi * hkv * d <= 240 * 4096 * 8 * 128 and rows * hi * hq <= 240 * 4096 * 16:
                return dict(case, rows=rows, lo=lo, hi=hi)
            continue
        rows, qhi = _log(rng, 1, 16), _log(rng, 1, 2048)
        chi = _log(rng, 1, 16384) if rng.random() < 0.6 else 0
        qlo, clo = _log(rng, 1, qhi), rng.randint(0, chi)
        if op == "append":
            if rows * qhi * (hq + 2 * hkv) * d <= 8 * 1024 * 32 * 128 and rows * (qhi + chi) * hkv * d <= 8 * 4096 * 1024:
                return dict(case, rows=rows, qlo=qlo, qhi=qhi, clo=clo, chi=chi)
        elif rows * hq * qhi * (qhi + chi) * d <= 8 * 16 * 2048 * 2048 * 128:
            return dict(case, rows=rows, qlo=qlo, qhi=qhi, clo=clo, chi=chi)


def _lengths(case):
    """Query and key lengths of the rows: they belong to the case, the values to the seed."""
    r, rows = random.Random(case["ragged"]), case["rows"]
    if case["op"] == "decode":
        kv = [case["hi"]] + [r.randint(case["lo"], case["hi"]) for _ in range(rows - 1)]
        return [1] * rows, kv
    q = [case["qhi"]] + [r.randint(case["qlo"], case["qhi"]) for _ in range(rows - 1)]
    return q, [n + r.randint(case["clo"], case["chi"]) for n in q]


# --------------------------------------------------------------------------------------------------- inputs
def _generator(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def _normal(shape, g, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device=g.device).to(dtype)


def _filled_cache(case, pages, g):
    """A pool whose blocks were quantised from N(0, 1) keys and values with a spread of magnitudes."""
    dtype, top = CODES[case["cache"]]
    shape = (pages, 2, case["page"] // BLOCK, BLOCK, case["hkv"], case["d"])
    x = torch.randn(shape, generator=g, device=g.device)
    x *= torch.exp(0.5 * torch.randn((pages, 2, case["page"] // BLOCK, 1, case["hkv"], 1), generator=g, device=g.device))
    s = x.abs().amax(dim=(3, 5)) / top
    x /= s[:, :, :, None, :, None]
    if dtype == torch.int8:
        x = x.round_()
    return x.to(dtype).view(pages, 2, case["page"], case["hkv"], case["d"]), s


def _prepare_paged(case, seed):
    dev = torch.device("cuda")
    g = _generator(seed, dev)
    order = random.Random(case["ragged"] + seed)
    qlens, kvlens = _lengths(case)
    page = case["page"]
    need = [-(-n // page) for n in kvlens]
    total = sum(need) + 4
    ids = list(range(total))
    order.shuffle(ids)  # the requests' pages are scattered over the pool
    cache, scales = _filled_cache(case, total, g)
    indptr, last, tables, at = [0], [], [], 0
    for n, p in zip(kvlens, need):
        tables.append(ids[at:at + p])
        at += p
        indptr.append(at)
        last.append(n - (p - 1) * page if p else 1)

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s = dict(case=case, cache=cache, scales=scales, kv_indptr=i32(indptr), kv_indices=i32(ids[:at]), last=i32(last),
             kvlens=torch.tensor(kvlens, device=dev), qlens=torch.tensor(qlens, device=dev))
    # every row's page table, padded with its own first entries, for the plain form
    widest = max(max(need), 1)
    s["table"] = torch.tensor([(t + [0] * widest)[:widest] for t in tables], device=dev)
    if case["op"] == "decode":
        s["q"] = _normal((case["rows"], case["hq"], case["d"]), g)
        return s
    q0 = [0]
    for n in qlens:
        q0.append(q0[-1] + n)
    tokens = q0[-1]
    s["qo_indptr"] = i32(q0)
    # place (row, index in its chunk) of every packed token
    s["tok_row"] = torch.repeat_interleave(torch.arange(case["rows"], device=dev), s["qlens"])
    s["tok_idx"] = torch.arange(tokens, device=dev) - s["qo_indptr"].long()[s["tok_row"]]
    s["positions"] = (s["kvlens"] - s["qlens"])[s["tok_row"]] + s["tok_idx"]
    if case["op"] == "prefill":
        s["q"] = _normal((tokens, case["hq"], case["d"]), g)
        return s
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    s["qkv"] = _normal((tokens, (hq + 2 * hkv) * d), g)  # one projection's output: q, k and v are strided views
    s["qw"] = (1 + 0.1 * torch.randn(d, generator=g, device=dev)).to(torch.bfloat16)
    s["kw"] = (1 + 0.1 * torch.randn(d, generator=g, device=dev)).to(torch.bfloat16)
    s["write_pages"] = s["table"][s["tok_row"], s["positions"] // page]
    s["write_offsets"] = s["positions"] % page
    touched = []
    for t, n, kv in zip(tables, qlens, kvlens):
        touched += t[(kv - n) // page:]
    s["touched"] = torch.tensor(touched, device=dev)
    return s


def prepare(case, seed):
    if case["op"] != "linear":
        return _prepare_paged(case, seed)
    dev = torch.device("cuda")
    g = _generator(seed, dev)
    m, n, k = case["m"], case["n"], case["k"]
    x = torch.randn((m, k), generator=g, device=dev)
    x *= torch.exp(0.5 * torch.randn((1, k), generator=g, device=dev))  # channels of unlike magnitude
    w = torch.randn((n, k), generator=g, device=dev) * k ** -0.5
    ws = w.abs().amax(dim=1) / 127.0
    s = dict(case=case, x=x.to(torch.bfloat16), wq=(w / ws[:, None]).round_().to(torch.int8), ws=ws)
    s["bias"] = _normal((n,), g) if case["bias"] else None
    return s


# --------------------------------------------------------------------------------------------------- plain forms
def _codes(s, pages):
    """The codes of the given pages as fp32 numbers."""
    return s["cache"].view(torch.uint8)[pages].view(s["cache"].dtype).float()


def _row_keys(s, kind):
    """[rows, longest, Hkv, D] fp32: every row's keys (kind 0) or values (kind 1), what lies past its end as zeros."""
    c = s["case"]
    codes = s["cache"].view(torch.uint8)[:, kind][s["table"]].view(s["cache"].dtype).float()  # [rows, pages, P, Hkv, D]
    r, p = codes.shape[:2]
    codes = codes.view(r, p, c["page"] // BLOCK, BLOCK, c["hkv"], c["d"])
    x = codes * s["scales"][:, kind][s["table"]][:, :, :, None, :, None]
    x = x.reshape(r, p * c["page"], c["hkv"], c["d"])
    live = torch.arange(x.shape[1], device=x.device)[None] < s["kvlens"][:, None]
    return torch.where(live[:, :, None, None], x, 0.0), live


def _softmax(score, seen):
    """Softmax of the last axis over the places in `seen`; a row that sees nothing gives zeros."""
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(dim=-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    return e / e.sum(dim=-1, keepdim=True).clamp_min(1e-30)


def _plain_decode(s):
    c = s["case"]
    k, live = _row_keys(s, 0)
    v, _ = _row_keys(s, 1)
    q = s["q"].float().view(c["rows"], c["hkv"], c["hq"] // c["hkv"], c["d"])
    score = torch.einsum("rhgd,rthd->rhgt", q, k) * c["d"] ** -0.5
    p = _softmax(score, live[:, None, None, :])
    return torch.einsum("rhgt,rthd->rhgd", p, v).reshape(c["rows"], c["hq"], c["d"]).to(torch.bfloat16)


def _plain_prefill(s):
    c = s["case"]
    k, live = _row_keys(s, 0)
    v, _ = _row_keys(s, 1)
    rows, g = c["rows"], c["hq"] // c["hkv"]
    longest = c["qhi"]
    q = torch.zeros((rows, longest, c["hq"], c["d"]), device=k.device)
    q[s["tok_row"], s["tok_idx"]] = s["q"].float()
    q = q.view(rows, longest, c["hkv"], g, c["d"])
    score = torch.einsum("rihgd,rthd->rhgit", q, k) * c["d"] ** -0.5
    last = (s["kvlens"] - s["qlens"])[:, None] + torch.arange(longest, device=k.device)  # last key that query i sees
    seen = torch.arange(k.shape[1], device=k.device)[None, None] <= last[:, :, None]
    p = _softmax(score, (seen & live[:, None])[:, None, None])
    out = torch.einsum("rhgit,rthd->rihgd", p, v).reshape(rows, longest, c["hq"], c["d"])
    return out[s["tok_row"], s["tok_idx"]].to(torch.bfloat16)


def _split_qkv(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    t = s["qkv"].shape[0]
    return (s["qkv"][:, :hq * d].view(t, hq, d), s["qkv"][:, hq * d:(hq + hkv) * d].view(t, hkv, d),
            s["qkv"][:, (hq + hkv) * d:].view(t, hkv, d))


def _norm_rope(x, w, positions):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * w.float()
    half = x.shape[-1] // 2
    angle = positions.double()[:, None, None] * THETA ** (-torch.arange(half, device=x.device).double() / half)
    cos, sin = angle.cos().float(), angle.sin().float()
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _to_codes(x, dtype, top):
    x = x.clamp(-top, top)
    return (x.round() if dtype == torch.int8 else x).to(dtype)


def _plain_append(s):
    """The write: a block's scale is its largest magnitude / the largest code when the call writes its first token;
    else the scale stays, or is doubled until the new tokens fit, and the codes of the tokens before them follow."""
    c = s["case"]
    dtype, top = CODES[c["cache"]]
    q, k, v = _split_qkv(s)
    rot = _norm_rope(q, s["qw"], s["positions"]).to(torch.bfloat16)
    new = torch.stack([_norm_rope(k, s["kw"], s["positions"]), v.float()], dim=1)  # [T, 2, Hkv, D]
    pages, blocks = s["cache"].shape[0], c["page"] // BLOCK
    block = s["write_pages"] * blocks + s["write_offsets"] // BLOCK
    at = s["write_offsets"] % BLOCK
    need = torch.zeros((pages * blocks, 2, c["hkv"]), device=q.device)
    need = need.index_reduce(0, block, new.abs().amax(dim=-1), "amax") / top
    first = torch.full((pages * blocks,), BLOCK, device=q.device).index_reduce(0, block, at, "amin")
    fresh = first == 0
    scales = s["scales"].transpose(1, 2).reshape(pages * blocks, 2, c["hkv"])
    mant, expo = torch.frexp(need / scales.clamp_min(1e-45))
    grow = (expo - (mant == 0.5).to(expo.dtype)).clamp_min(0)
    after = torch.where(fresh[:, None, None] | (scales == 0), need, torch.ldexp(scales, grow))
    after = torch.where(need > 0, after, torch.where(fresh[:, None, None], need, scales))
    # the codes before the written ones, brought to the new scale; what lies behind stays as it is
    view = s["cache"].view(torch.uint8).view(pages, 2, blocks, BLOCK, c["hkv"], c["d"])
    p, b = s["write_pages"], s["write_offsets"] // BLOCK
    old = view[p, :, b].view(dtype).float()  # [T, 2, BLOCK, Hkv, D]
    ratio = torch.where(after > 0, scales / after.clamp_min(1e-45), 1.0)[block][:, :, None, :, None]
    before = torch.arange(BLOCK, device=q.device)[None] < first[block][:, None]
    ratio = torch.where(before[:, None, :, None, None], ratio, 1.0)
    view[p, :, b] = _to_codes(old * ratio, dtype, top).view(torch.uint8)
    mine = after[block][..., None]
    codes = _to_codes(torch.where(mine > 0, new / mine.clamp_min(1e-45), 0.0), dtype, top)
    view[p, :, b, at] = codes.view(torch.uint8)
    s["scales"].copy_(after.view(pages, blocks, 2, c["hkv"]).transpose(1, 2))
    return rot, _plain_read(s)


def _plain_read(s):
    c = s["case"]
    codes = _codes(s, s["touched"]).view(-1, 2, c["page"] // BLOCK, BLOCK, c["hkv"], c["d"])
    x = codes * s["scales"][s["touched"]][:, :, :, None, :, None]
    return x.view(-1, 2, c["page"], c["hkv"], c["d"]).to(torch.bfloat16)


def _plain_linear(s):
    c = s["case"]
    x = s["x"].float()
    xs = x.abs().amax(dim=1, keepdim=True) / 127.0
    xq = torch.where(xs > 0, x / xs.clamp_min(1e-45), 0.0).round().clamp(-127, 127)
    y = xq @ s["wq"].float().t()
    y = y * xs * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["gate_up"]:
        gate, up = y[:, :c["n"] // 2], y[:, c["n"] // 2:]
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(torch.bfloat16)


# --------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    nqt = importlib.import_module("nari-qwen3-tts_b200")
    c = s["case"]
    if c["op"] == "decode":
        if "workspace" not in s:
            s["workspace"] = nqt.decode_paged8_workspace(c["rows"], c["hq"], c["d"], s["q"].device)
        return nqt.batch_decode_paged8(s["q"], s["cache"], s["scales"], s["kv_indptr"], s["kv_indices"], s["last"],
                                       s["workspace"])
    if c["op"] == "prefill":
        return nqt.batch_prefill_paged8(s["q"], s["cache"], s["scales"], s["qo_indptr"], s["kv_indptr"],
                                        s["kv_indices"], s["last"])
    if c["op"] == "append":
        q, k, v = _split_qkv(s)
        rot = nqt.paired_qk_norm_rope_paged_cache8(q, k, v, s["qw"], s["kw"], s["positions"], EPS, THETA, s["cache"],
                                                   s["scales"], s["write_pages"], s["write_offsets"])
        return rot, nqt.read_paged_cache8(s["cache"], s["scales"], s["touched"])
    if "weight" not in s:
        s["weight"] = nqt.kernels.Int8Weight.from_quantized(s["wq"], s["ws"], gate_up=c["gate_up"])
    return nqt.kernels.linear_int8(s["x"], s["weight"], bias=s["bias"])


def run(state):
    if own:
        return _own(state)
    return {"decode": _plain_decode, "prefill": _plain_prefill, "append": _plain_append,
            "linear": _plain_linear}[state["case"]["op"]](state)


# --------------------------------------------------------------------------------------------------- work and exact values
def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        out = n // 2 if case["gate_up"] else n
        return {"bytes": 2 * m * k + n * k + 4 * n + (2 * n if case["bias"] else 0) + 2 * m * out, "flops": 2 * m * n * k}
    qlens, kvlens = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    tokens, keys = sum(qlens), sum(kvlens)
    blocks = sum(-(-n // BLOCK) for n in kvlens)
    if case["op"] == "append":
        pages = sum(-(-n // case["page"]) - (n - q) // case["page"] for q, n in zip(qlens, kvlens))
        back = pages * 2 * case["page"] * hkv * d
        return {"bytes": 2 * tokens * (2 * hq + 2 * hkv) * d + 2 * tokens * hkv * d + 24 * tokens + 3 * back,
                "flops": 12 * tokens * (hq + 2 * hkv) * d}
    pairs = sum(q * (n - q) + q * (q + 1) // 2 for q, n in zip(qlens, kvlens) if n)
    return {"bytes": 2 * keys * hkv * d + 8 * blocks * hkv + 4 * tokens * hq * d, "flops": 4 * pairs * hq * d}


def _exact_attention(case, s):
    """One row and KV head at a time, from softmax(q k^T / sqrt(d)) v."""
    qlens, kvlens = _lengths(case)
    d, g, page = case["d"], case["hq"] // case["hkv"], case["page"]
    if sum(q * n for q, n in zip(qlens, kvlens)) * case["hq"] * d > 4e11:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    q0 = 0
    for r, (nq, nk) in enumerate(zip(qlens, kvlens)):
        ids = s["kv_indices"][int(s["kv_indptr"][r]):int(s["kv_indptr"][r + 1])].long()
        for h in range(case["hkv"] if nk else 0):
            sc = s["scales"][ids][..., h].double().repeat_interleave(BLOCK, dim=2)  # [pages, 2, P]
            kv = (_codes(s, ids)[:, :, :, h].double() * sc[..., None]).transpose(0, 1)
            key, val = (t.reshape(-1, d)[:nk] for t in kv)
            for e in range(h * g, (h + 1) * g):
                for lo in range(0, nq, 512):
                    hi = min(lo + 512, nq)
                    z = s["q"][q0 + lo:q0 + hi, e].double() @ key.t() / math.sqrt(d)
                    hidden = torch.arange(nk, device=z.device)[None] > (nk - nq + torch.arange(lo, hi, device=z.device))[:, None]
                    out[q0 + lo:q0 + hi, e] = z.masked_fill(hidden, -math.inf).softmax(dim=-1) @ val
        q0 += nq
    return out


def _exact_append(case, s):
    """Token blocks one by one, from the definition of the write."""
    qlens, kvlens = _lengths(case)
    _, top = CODES[case["cache"]]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    freq = torch.exp(-math.log(THETA) * 2.0 * torch.arange(d // 2, device=x.device, dtype=torch.float64) / d)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), s["positions"].double()[:, None] * freq)
    w = torch.cat([s["qw"].double().expand(hq, d), s["kw"].double().expand(hkv, d)])
    y = x[:, :hq + hkv]
    y = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w
    z = torch.complex(y[..., :d // 2], y[..., d // 2:]) * turn[:, None]
    y = torch.cat([z.real, z.imag], dim=-1)
    new = torch.stack([y[:, hq:], x[:, hq + hkv:]], dim=1)
    nb = page // BLOCK
    codes = s["cache"].to(torch.float32).double().view(-1, 2, nb, BLOCK, hkv, d)
    scale = s["scales"].double().clone()
    t = 0
    for r, (nq, nk) in enumerate(zip(qlens, kvlens)):
        pos = nk - nq
        while pos < nk:
            n = min(BLOCK - pos % BLOCK, nk - pos)
            p, b, o = int(s["table"][r, pos // page]), pos % page // BLOCK, pos % BLOCK
            part = new[t:t + n].transpose(0, 1)  # [2, n, Hkv, D]
            fit = part.abs().amax(dim=(1, 3)) / top
            old = scale[p, :, b]
            if o == 0:
                to = fit
            else:
                to = torch.where(old > 0, old * torch.exp2(torch.ceil(torch.log2((fit / old).clamp_min(1.0)))), fit)
                was = codes[p, :, b, :o] * (old / to)[:, None, :, None]
                codes[p, :, b, :o] = _nearest(was, case["cache"], top)
            codes[p, :, b, o:o + n] = _nearest(part / to[:, None, :, None], case["cache"], top)
            scale[p, :, b] = to
            pos, t = pos + n, t + n
    back = codes * scale[:, :, :, None, :, None]
    return y[:, :hq], back.view(-1, 2, page, hkv, d)[s["touched"]]


def _nearest(x, kind, top):
    """The nearest code (ties to even) as the number that it stands for, before its scale."""
    x = x.nan_to_num(0.0).clamp(-top, top)
    if kind == "int8":
        return x.round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)  # e4m3: three mantissa bits, from 2^-6
    return (x / step).round() * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("decode", "prefill"):
        return _exact_attention(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    x = s["x"].double()
    amax = x.abs().amax(dim=1)
    codes = (x * (127.0 / amax.clamp_min(1e-300))[:, None]).round()
    out = (codes @ s["wq"].double().t()) * (amax / 127.0)[:, None] * s["ws"].double()[None]
    if s["bias"] is not None:
        out = out + s["bias"].double()
    if case["gate_up"]:
        out = torch.nn.functional.silu(out[:, :case["n"] // 2]) * out[:, case["n"] // 2:]
    return out
