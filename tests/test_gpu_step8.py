"""GPU: the 8-bit operators together, as a talker layer and a talker step use them: int8 projections around the
quantised write and the attention over the 8-bit cache, through the binding and through the captured step."""

from __future__ import annotations

from importlib import import_module

import pytest
import torch

from oracle import cache8 as oc8
from tests._cache8 import attention_tolerance, make_cache8, numbers
from tests._paged import FakeAttention

pytestmark = pytest.mark.gpu


def _binding(nqt, cuda, storage, scales, rows, tokens, hq, hkv, d, page_size, mode):
    return nqt.B200TalkerBinding(storage=storage, scales=scales, capture_batch_size=rows, token_capacity=tokens,
                                 num_qo_heads=hq, num_kv_heads=hkv, head_dim=d, page_size=page_size,
                                 total_pages=storage.shape[1], device=cuda, dtype=torch.bfloat16, mode=mode)


def _metadata(nqt, indptr, indices, last, pos, pages, offs, qo):
    return nqt.TalkerAttentionMetadata(qo_indptr=qo, paged_kv_indptr=indptr, paged_kv_indices=indices,
                                       paged_kv_last_page_len=last, position_ids=pos, write_pages=pages,
                                       write_offsets=offs, padding_pages=())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("chunks", [[1, 1, 1, 1], [30, 1, 129, 16]])
def test_layer_chain(nqt, cuda, kind, chunks):
    """x -> int8 QKV -> binding.attend (write, then decode or prefill) -> int8 O, each against 64-bit arithmetic on
    the GPU's own input to it."""

    hq, hkv, d, hidden, page_size = 16, 8, 128, 512, 16
    lens = [n + c for n, c in zip([64, 0, 300, 15], chunks, strict=True)]
    decode = max(chunks) == 1
    codes, scales, indptr, indices, last = make_cache8(lens, kind=kind, seed=1)
    g = torch.Generator().manual_seed(2)
    tokens = sum(chunks)
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16)
    w_qkv = (torch.randn((hq + 2 * hkv) * d, hidden, generator=g) * hidden**-0.5).to(torch.bfloat16)
    w_o = (torch.randn(hidden, hq * d, generator=g) * (hq * d)**-0.5).to(torch.bfloat16)
    norm = [(1 + 0.1 * torch.randn(d, generator=g)).to(torch.bfloat16) for _ in range(2)]
    pos = torch.cat([torch.arange(n - c, n) for n, c in zip(lens, chunks, strict=True)])
    row = torch.repeat_interleave(torch.arange(4), torch.tensor(chunks))
    pages = indices.long()[indptr.long()[row] + pos // page_size]
    offs = pos % page_size
    qo = torch.tensor([0, *torch.tensor(chunks).cumsum(0).tolist()], dtype=torch.int32)

    storage, dscales = codes[None].to(cuda), scales[None].to(cuda)
    qkv8, o8 = (nqt.kernels.Int8Weight(w.to(cuda)) for w in (w_qkv, w_o))
    b = _binding(nqt, cuda, storage, dscales, 4, tokens, hq, hkv, d, page_size, None)
    b.plan(_metadata(nqt, indptr, indices, last, pos, pages, offs, None if decode else qo))
    b.select_layer(0)
    attention = FakeAttention(*(w.to(cuda) for w in norm))
    nqt.kernels.clear_status(cuda)
    qkv = nqt.kernels.linear_int8(x.to(cuda), qkv8)
    q = qkv[:, :hq * d].view(tokens, hq, d)
    k = qkv[:, hq * d:(hq + hkv) * d].view(tokens, hkv, d)
    v = qkv[:, (hq + hkv) * d:].view(tokens, hkv, d)
    attn = b.attend(attention, q, k, v)
    out = nqt.kernels.linear_int8(attn.view(tokens, hq * d), o8)
    torch.cuda.synchronize()
    assert nqt.kernels.read_status(cuda) == 0

    def product(inp, weight, got):
        xq, xs = nqt.kernels.int8_quantize_rows(inp)
        want = (xq.cpu().double() @ weight.q.cpu().double().t()) * xs.cpu().double()[:, None] * weight.scale.cpu().double()
        assert ((got.cpu().double() - want).abs() <= (2.0**-8 + 2.0**-21) * want.abs()).all()

    product(x.to(cuda), qkv8, qkv)
    # the write: the oracle's cache from the GPU's qkv, one code apart at most where a value lies between two
    kc, vc, qc = k.cpu(), v.cpu(), q.cpu()
    new = torch.stack([oc8.norm_rope(kc, norm[1], pos, 1e-6, 1e6), vc.double()], 1)
    wc, ws = numbers(codes), scales.double()
    oc8.write(wc, ws, new, pages.tolist(), offs.tolist(), kind)
    gc, gs = numbers(storage[0].cpu()), dscales[0].cpu().double()
    assert ((gs - ws).abs() <= 2.0**-18 * ws).all()
    assert (gc != wc).double().mean() <= 1e-3
    # attention over the GPU's own cache, with the query rounded to bf16 as the binding passes it on
    rot = oc8.norm_rope(qc, norm[0], pos, 1e-6, 1e6)
    want, mag = oc8.attention(rot.to(torch.bfloat16), gc, gs, indptr, indices, last, None if decode else qo)
    # the GPU's query may round the other way where fp32 and 64 bits part: one bf16 step of few elements
    err = (attn.cpu().double() - want).abs()
    over = err > attention_tolerance(want, mag)
    assert over.double().mean() <= 2e-2 and (err <= attention_tolerance(want, mag) + 2.0**-7 * mag).all()
    product(attn.view(tokens, hq * d), o8, out)


def test_binding_refuses_mixed_storage(nqt, cuda):
    codes, scales, *_ = make_cache8([20])
    args = (nqt, cuda, codes[None].to(cuda))
    with pytest.raises(ValueError, match="comes with scales"):
        _binding(*args, None, 1, 1, 16, 8, 128, 16, "decode")
    with pytest.raises(ValueError, match="comes with scales"):
        _binding(nqt, cuda, codes[None].to(cuda).to(torch.bfloat16), scales[None].to(cuda), 1, 1, 16, 8, 128, 16, "decode")
    with pytest.raises(TypeError, match="float32"):
        _binding(*args, scales[None].to(cuda).double(), 1, 1, 16, 8, 128, 16, "decode")


@pytest.mark.parametrize(("kv", "gate_up", "projections"), [("int8", "int8", "int8"), ("e4m3", "fp8", "bf16"),
                                                            ("bf16", "int8", "int8")])
def test_talker_step_at_8_bits(nqt, cuda, kv, gate_up, projections):
    """The captured step equals the eager one, stays near the bf16 step, and its replays append to the cache."""

    ts = import_module("nari-qwen3-tts_b200.talker_step")
    shape = ts.TalkerShape(num_layers=2)
    contexts = [17, 300, 64, 1, 511, 33, 128, 90]
    kw = dict(shape=shape, batch=8, total_pages=512, max_pages_per_seq=64, device=cuda, seed=3)

    def build(**opts):
        step = ts.TalkerDecodeStep(**kw, **opts)
        step.admit(contexts)
        step.hidden_in.copy_(torch.randn(8, shape.hidden, generator=torch.Generator().manual_seed(4)))
        return step

    step = build(kv=kv, gate_up=gate_up, projections=projections, publish=False)
    nqt.kernels.clear_status(cuda)
    trace: list = []
    step.forward(trace)
    first = trace[-2][0].clone()
    hidden = first.float()
    step.capture(warmup=1)
    step.replay()
    torch.cuda.synchronize()
    assert nqt.kernels.read_status(cuda) == 0 and step.planner.check() == 0
    again: list = []
    step.forward(again)
    # discarded steps write the same tokens at the same places: a block's scale that grew once is large enough now
    assert torch.equal(again[-2][0], first)
    assert torch.equal(step.last_hidden, first) and torch.isfinite(hidden).all()

    plain = build(gate_up="bf16", publish=False)
    if step.scales is not None:  # the same cached keys and values, in bf16
        for layer in range(2):
            pages = torch.arange(512, device=cuda)
            plain.storage[layer] = nqt.read_paged_cache8(step.storage[layer], step.scales[layer], pages)
    else:
        plain.storage.copy_(step.storage)
    other: list = []
    plain.forward(other)
    ref = other[-2][0].float()
    # An int8 operand of n = 2048 Gaussian elements has steps of amax / 127 = 3.7 / 127 of their deviation, an rms error
    # of that / sqrt(12) = 0.0084; two operands make 0.012 of a product's norm, and the 4 products of 2 layers at most
    # sqrt(8) 0.012 = 0.034 of the state's.  An e4m3 operand's rms error is under 2^-4 / sqrt(3) = 0.036 of each
    # element, gate, up and their product under sqrt(2) * sqrt(2) * 0.036 = 0.072 of an MLP's output, which is one of
    # five parts of the state (the input, 2 attentions, 2 MLPs).
    assert ((hidden - ref).norm() / ref.norm()) < 0.1
    assert step.weight_bytes() <= plain.weight_bytes()
    assert kv == "bf16" or step.attention_bytes_per_layer() < 0.55 * plain.attention_bytes_per_layer()


def test_step_options_are_checked(nqt, cuda):
    ts = import_module("nari-qwen3-tts_b200.talker_step")
    for bad in (dict(kv="fp4"), dict(projections="fp8"), dict(gate_up="int4")):
        with pytest.raises(ValueError):
            ts.TalkerDecodeStep(shape=ts.TalkerShape(num_layers=1), batch=1, total_pages=64, device=cuda, **bad)
