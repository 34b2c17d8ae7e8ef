"""CPU: what the 8-bit operators refuse, before any launch: argument errors of the C ABI and of the package's
functions."""

from __future__ import annotations

import importlib

import pytest
import torch

ARG, UNSUPPORTED, CAPACITY = -1, -4, -3
A = 1 << 20  # an aligned address that is never read: every call here is refused first


def _lib():
    return importlib.import_module("nari-qwen3-tts_b200._lib").lib()


def _decode_args(**kw):
    a = dict(q=A, qt=2048, qh=128, cache=A, scales=A, pages=64, page=16, indptr=A, indices=A, last=A, batch=2, cap=2,
             hq=16, hkv=8, d=128, scale=0.1, code=3, out=A, ot=2048, oh=128, ws=A, nbytes=1 << 30, flags=0, status=A,
             stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize(("change", "want"), [
    (dict(q=None), ARG), (dict(cache=None), ARG), (dict(scales=None), ARG), (dict(indptr=None), ARG), (dict(ws=None), ARG),
    (dict(out=None), ARG), (dict(code=0), UNSUPPORTED), (dict(code=9), UNSUPPORTED), (dict(d=96), UNSUPPORTED),
    (dict(page=24), UNSUPPORTED), (dict(page=272), UNSUPPORTED), (dict(page=8), UNSUPPORTED), (dict(hkv=0), ARG),
    (dict(hq=12), ARG), (dict(hq=72), UNSUPPORTED), (dict(pages=0), ARG), (dict(batch=3), ARG), (dict(batch=-1), ARG),
    (dict(q=A + 2), ARG), (dict(qt=2049), ARG), (dict(oh=127), ARG), (dict(cache=A + 8), ARG), (dict(nbytes=100), CAPACITY),
    (dict(batch=9000, cap=9000), CAPACITY), (dict(flags=4), ARG), (dict(ws=A + 4), ARG), (dict(pages=1 << 30), UNSUPPORTED),
])
def test_decode_refusals(change, want):
    assert _lib().nqt_decode_attention8(*_decode_args(**change)) == want


def _prefill_args(**kw):
    a = dict(q=A, qt=2048, qh=128, cache=A, scales=A, pages=64, page=16, qo=A, indptr=A, indices=A, last=A, batch=2,
             tokens=10, hq=16, hkv=8, d=128, scale=0.1, code=4, out=A, ot=2048, oh=128, status=A, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize(("change", "want"), [
    (dict(q=None), ARG), (dict(qo=None), ARG), (dict(batch=0), ARG), (dict(tokens=-1), ARG), (dict(scale=-1.0), ARG),
    (dict(scale=float("nan")), ARG), (dict(q=A + 8), ARG), (dict(qt=2052), ARG), (dict(hq=18), ARG),
    (dict(hq=72), UNSUPPORTED), (dict(d=32), UNSUPPORTED), (dict(code=2), UNSUPPORTED), (dict(page=100), UNSUPPORTED),
])
def test_prefill_refusals(change, want):
    assert _lib().nqt_prefill_attention8(*_prefill_args(**change)) == want


def _write_args(**kw):
    a = dict(q=A, qt=4096, qh=128, k=A, kt=4096, kh=128, v=A, vt=4096, vh=128, qw=A, kw=A, pos=A, pages=A, offs=A,
             out=A, ot=2048, oh=128, cache=A, scales=A, total=64, page=16, tokens=3, hq=16, hkv=8, d=128, eps=1e-6,
             theta=1e6, code=3, status=A, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize(("change", "want"), [
    (dict(q=None), ARG), (dict(v=None), ARG), (dict(pos=None), ARG), (dict(cache=None), ARG), (dict(scales=A + 2), ARG),
    (dict(tokens=-1), ARG), (dict(theta=0.0), ARG), (dict(theta=float("nan")), ARG), (dict(d=256), UNSUPPORTED),
    (dict(code=1), UNSUPPORTED), (dict(hq=0), ARG), (dict(page=20), UNSUPPORTED),
])
def test_write_refusals(change, want):
    assert _lib().nqt_qk_norm_rope_paged_cache8(*_write_args(**change)) == want


def test_read_refusals():
    f = _lib().nqt_read_paged_cache8
    ok = [A, A, 64, 16, 8, 128, 3, A, 2, A, A, None]
    for at, bad, want in ((0, None, ARG), (7, None, ARG), (8, -1, ARG), (9, A + 8, ARG), (6, 7, UNSUPPORTED),
                          (5, 80, UNSUPPORTED)):
        args = list(ok)
        args[at] = bad
        assert f(*args) == want


def _gemm_args(**kw):
    a = dict(xq=A, ldx=64, xs=A, w=A, ldw=64, ws=A, bias=None, y=A, ldy=32, m=4, n=32, cols=32, k=64, epilogue=0,
             status=A, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize(("change", "want"), [
    (dict(xq=None), ARG), (dict(w=None), ARG), (dict(ws=None), ARG), (dict(y=None), ARG), (dict(m=-1), ARG),
    (dict(n=0, cols=0), ARG), (dict(k=0), ARG), (dict(cols=31), ARG), (dict(epilogue=3), ARG), (dict(epilogue=1), ARG),
    (dict(epilogue=2), ARG), (dict(epilogue=2, n=40, cols=20), ARG), (dict(ldx=60), ARG), (dict(ldx=48), ARG),
    (dict(xq=A + 8), ARG), (dict(w=A + 1), ARG), (dict(ldw=63), ARG), (dict(ldy=31), ARG),
    (dict(k=131073, ldx=131088, ldw=131088), UNSUPPORTED),
])
def test_gemm_refusals(change, want):
    assert _lib().nqt_gemm_int8(*_gemm_args(**change)) == want


def _cpu_case():
    q = torch.zeros(2, 16, 128, dtype=torch.bfloat16)
    cache, scales = torch.zeros(4, 2, 16, 8, 128, dtype=torch.int8), torch.ones(4, 2, 1, 8)
    i = torch.zeros(3, dtype=torch.int32)
    return q, cache, scales, i


def test_functions_refuse_wrong_arguments(nqt):
    q, cache, scales, i = _cpu_case()
    ws = torch.zeros(64, dtype=torch.uint8)
    decode = nqt.batch_decode_paged8
    with pytest.raises(TypeError, match="bf16 query"):
        decode(q.float(), cache, scales, i, i, i, ws)
    with pytest.raises(TypeError, match="int8 or float8"):
        decode(q, cache.float(), scales, i, i, i, ws)
    with pytest.raises(TypeError, match="float32"):
        decode(q, cache, scales.double(), i, i, i, ws)
    with pytest.raises(ValueError, match="scales must be"):
        decode(q, cache, scales[:3], i, i, i, ws)
    with pytest.raises(TypeError, match="int32"):
        decode(q, cache, scales, i.long(), i, i, ws)
    with pytest.raises(ValueError, match="every row"):
        decode(q, cache, scales, i[:2], i, i, ws)
    with pytest.raises(ValueError, match="1 to 8 query heads"):
        decode(torch.zeros(2, 9, 128, dtype=torch.bfloat16), cache, scales, i, i, i, ws)
    with pytest.raises(ValueError, match="output must be"):
        decode(q, cache, scales, i, i, i, ws, out=torch.zeros(2, 16, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="contiguous"):
        decode(q, torch.zeros(4, 2, 8, 16, 128, dtype=torch.int8).transpose(2, 3), scales, i, i, i, ws)
    with pytest.raises(ValueError, match="batch_capacity"):
        decode(q, cache, scales, i, i, i, ws, batch_capacity=1)
    with pytest.raises(ValueError, match="CUDA"):
        decode(q, cache, scales, i, i, i, ws)
    with pytest.raises(TypeError, match="tensors"):
        decode(q, cache, None, i, i, i, ws)

    prefill = nqt.batch_prefill_paged8
    with pytest.raises(ValueError, match="sm_scale"):
        prefill(q, cache, scales, i, i, i, i, sm_scale=-0.5)
    with pytest.raises(ValueError, match="every row"):
        prefill(q, cache, scales, i, i, i, i, batch=7)
    with pytest.raises(ValueError, match="CUDA"):
        prefill(q, cache, scales, i, i, i, i)

    w, pos = torch.ones(128, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.long)
    k = torch.zeros(2, 8, 128, dtype=torch.bfloat16)

    def write(**kw):
        a = dict(query=q, key=k, value=k, query_weight=w, key_weight=w, position_ids=pos, epsilon=1e-6, rope_theta=1e6,
                 layer_cache=cache, layer_scales=scales, write_pages=pos, write_offsets=pos)
        return nqt.paired_qk_norm_rope_paged_cache8(**{**a, **kw})

    with pytest.raises(ValueError, match="incompatible"):
        write(value=k[:, :4])
    with pytest.raises(ValueError, match="norm weights"):
        write(key_weight=w[:64])
    with pytest.raises(ValueError, match="one entry per token"):
        write(write_pages=pos[:1])
    with pytest.raises(TypeError, match="int64"):
        write(write_offsets=pos.int())
    with pytest.raises(TypeError, match="bf16"):
        write(query=q.half())
    with pytest.raises(ValueError, match="rope_theta"):
        write(rope_theta=0.0)
    with pytest.raises(ValueError, match="CUDA"):
        write()
    with pytest.raises(TypeError, match="int64"):
        nqt.read_paged_cache8(cache, scales, pos.int())
    with pytest.raises(ValueError, match="CUDA"):
        nqt.read_paged_cache8(cache, scales, pos)


def test_int8_functions_refuse_wrong_arguments(nqt):
    kn = nqt.kernels
    with pytest.raises(ValueError):
        kn.int8_quantize_rows(torch.zeros(4, 8))
    with pytest.raises(ValueError):
        kn.Int8Weight(torch.zeros(4, 8))
    with pytest.raises(ValueError):
        kn.Int8Weight.from_quantized(torch.zeros(4, 8), torch.ones(4))
    with pytest.raises(ValueError):
        kn.Int8Weight.from_quantized(torch.zeros(4, 8, dtype=torch.int8), torch.ones(3))
    with pytest.raises(TypeError):
        kn.linear_int8(torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8))
    weight = kn.Int8Weight.__new__(kn.Int8Weight)
    weight._lay_out(torch.zeros(6, 16, dtype=torch.int8), torch.ones(6), False)
    gate_up = kn.Int8Weight.__new__(kn.Int8Weight)
    gate_up._lay_out(torch.zeros(6, 16, dtype=torch.int8), torch.ones(6), True)
    x = torch.zeros(2, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="matching the weight"):
        kn.linear_int8(x[:, :8], weight)
    with pytest.raises(TypeError, match="bf16 rows"):
        kn.linear_int8(x.float(), weight)
    with pytest.raises(TypeError, match="xscale"):
        kn.linear_int8(x.to(torch.int8), weight)
    with pytest.raises(ValueError, match="belongs to int8"):
        kn.linear_int8(x, weight, xscale=torch.ones(2))
    with pytest.raises(ValueError, match="no bias"):
        kn.linear_int8(x, gate_up, torch.zeros(6, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="bias must be"):
        kn.linear_int8(x, weight, torch.zeros(5, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="output must be"):
        kn.linear_int8(x, weight, out=torch.zeros(2, 5, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA"):
        kn.linear_int8(x, weight)
    with pytest.raises(ValueError, match="even number"):
        gate_up._lay_out(torch.zeros(5, 16, dtype=torch.int8), torch.ones(5), True)


def test_gate_up_layout_interleaves_groups_of_16(nqt):
    f, k = 20, 24
    q = torch.arange(2 * f, dtype=torch.int8)[:, None].expand(2 * f, k).contiguous()
    w = nqt.kernels.Int8Weight.__new__(nqt.kernels.Int8Weight)
    w._lay_out(q, torch.arange(2 * f, dtype=torch.float32), True)
    assert w.data.shape == (64, 32) and w.cols == f
    rows = w.data[:, 0].tolist()
    assert rows[:16] == list(range(16)) and rows[16:32] == list(range(f, f + 16))
    assert rows[32:36] == list(range(16, f)) and rows[36:48] == [0] * 12
    assert rows[48:52] == list(range(f + 16, 2 * f)) and (w.data[:, k:] == 0).all()
    assert w.data_scale[:16].tolist() == list(range(16)) and w.data_scale[36:48].tolist() == [0.0] * 12


def test_oracle_codes_match_torch():
    """The oracle's e4m3 rounding is torch's, and int8 rounds half to even."""

    from oracle import cache8 as oc8

    x = torch.cat([torch.linspace(-500, 500, 20001), torch.logspace(-12, 3, 5000, base=2.0)])
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).double()
    assert torch.equal(oc8.nearest_code(x.double(), "e4m3"), want)
    assert oc8.nearest_code(torch.tensor([0.5, 1.5, -2.5, 300.0]).double(), "int8").tolist() == [0, 2, -2, 127]
