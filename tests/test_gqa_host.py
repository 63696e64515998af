"""Host side of the grouped-head cache: its C entry points refuse bad arguments before any launch (no GPU is
touched), and its sizes."""
from ctypes import addressof, c_int32

import pytest

from rsllm_b200 import _abi

BASE = 0x100000
SHAPE, INDEX, LAYER, ARG = (_abi.RKV_ERR_SHAPE_MISMATCH, _abi.RKV_ERR_INDEX_OUT_OF_RANGE, _abi.RKV_ERR_INVALID_LAYER,
                            _abi.RKV_ERR_INVALID_ARGUMENT)


def view(**kw):
    f = dict(base=BASE, n_pages=8, n_layers=2, n_kv_heads=2, head_dim=128, dtype=_abi.GQA_BF16)
    f.update(kw)
    return _abi.GqaView(*(f[k] for k, _ in _abi.GqaView._fields_))


def decode(v, layer=0, q=BASE, ts=1024, hs=128, n_seq=1, heads=8, pt=BASE, stride=4, lens=BASE, window=0, sinks=0,
           scale=0.1, ws=BASE, out=BASE, null=False):
    return _abi.load().rkv_gqa_decode(0 if null else addressof(v), layer, q, ts, hs, n_seq, heads, pt, stride, lens,
                                      window, sinks, scale, ws, out, 0, 0)


def prefill(v, layer=0, q=BASE, ts=1024, hs=128, n=1, heads=8, cu=BASE, n_seq=1, pt=BASE, stride=4, lens=BASE,
            window=0, scale=0.1, ws=BASE, out=BASE):
    return _abi.load().rkv_gqa_prefill(addressof(v), layer, q, ts, hs, n, heads, cu, n_seq, pt, stride, lens, window,
                                       0, scale, ws, out, 0, 0)


def append(v, layer=0, k=BASE, ts=256, hs=128, vv=BASE, n=1, slots=BASE, rot=None, pos=BASE, q=0, heads=0, q_out=0):
    return _abi.load().rkv_gqa_append(addressof(v), layer, k, ts, hs, vv, ts, hs, n, slots,
                                      addressof(rot) if rot is not None else 0, pos, q, 1024, 128, heads, q_out, 0, 0)


def rotary(table=BASE, rows=16, rot=128, inter=0, sections=(64,)):
    return _abi.GqaRotary(table, rows, rot, inter, len(sections), (c_int32 * 4)(*sections))


def test_sizes():
    lib = _abi.load()
    assert lib.rkv_gqa_page_bytes(8, 128) == 2 * 8 * 64 * 128 * 2
    assert lib.rkv_gqa_page_bytes(1, 64) == 16384
    assert lib.rkv_gqa_page_bytes(0, 64) == lib.rkv_gqa_page_bytes(1, 96) == -1
    v = view(n_pages=1 << 16, n_layers=3, n_kv_heads=8)
    assert lib.rkv_gqa_bytes(addressof(v)) == 3 * (1 << 16) * 262144
    assert lib.rkv_gqa_prefill_workspace_bytes(addressof(v)) >= 2 * 148 * 256 * (128 + 2) * 4
    assert lib.rkv_gqa_prefill_workspace_bytes(0) == -1
    assert lib.rkv_gqa_decode_workspace_bytes(addressof(v), -1, 32) == -1


@pytest.mark.parametrize("call", [decode, prefill, append])
def test_cache_view(call):
    assert call(view(base=0)) == ARG
    assert call(view(base=BASE + 16)) == ARG
    for name in ("n_pages", "n_layers", "n_kv_heads"):
        assert call(view(**{name: 0})) == ARG
    assert call(view(head_dim=96)) == SHAPE
    assert call(view(dtype=2)) == ARG
    assert call(view(n_pages=1 << 25)) == ARG  # slots past int32
    assert call(view(n_pages=1 << 20, n_layers=60, n_kv_heads=8)) == ARG  # rows past int32
    assert call(view(), layer=2) == LAYER
    assert call(view(), layer=-1) == LAYER
    assert _abi.last_error_info()["max"] == 2


@pytest.mark.parametrize("call", [decode, prefill])
def test_attention_arguments(call):
    v = view()
    assert call(v, heads=7) == SHAPE and call(v, heads=0) == SHAPE and call(v, heads=130) == SHAPE
    assert call(v, q=0) == ARG and call(v, q=BASE + 8) == ARG
    assert call(v, ts=1028) == SHAPE and call(v, hs=-128) == SHAPE
    assert call(v, n_seq=-1) == SHAPE
    assert call(v, stride=0) == SHAPE and call(v, stride=1 << 26) == SHAPE
    assert call(v, window=-1) == SHAPE
    for scale in (0.0, -0.5, float("nan"), float("inf")):
        assert call(v, scale=scale) == ARG
    for name in ("pt", "lens", "out"):
        assert call(v, **{name: 0}) == ARG
    assert call(v, out=BASE + 8) == ARG


def test_decode_arguments():
    assert decode(view(), null=True) == ARG
    assert decode(view(), ws=0) == ARG and decode(view(), ws=BASE + 8) == ARG
    assert decode(view(), n_seq=0, q=0, pt=0, lens=0, out=0, ws=0) == 0


def test_prefill_arguments():
    v = view()
    assert prefill(v, n=-1) == SHAPE and prefill(v, cu=0) == ARG
    assert prefill(v, ws=0) == ARG and prefill(v, ws=BASE + 8) == ARG
    assert prefill(v, n_seq=0) == SHAPE  # tokens without a sequence
    assert prefill(v, n=0, q=0, out=0) == 0


def test_append_arguments():
    v = view()
    assert append(v, n=-1) == SHAPE
    assert append(v, k=BASE + 2) == ARG and append(v, vv=0) == ARG and append(v, slots=0) == ARG
    assert append(v, ts=100) == SHAPE
    assert append(v, q=BASE, heads=8, q_out=BASE) == ARG  # q without rotary
    assert append(v, rot=rotary(), pos=0) == ARG
    assert append(v, rot=rotary(table=0)) == ARG and append(v, rot=rotary(rows=0)) == ARG
    assert append(v, rot=rotary(rot=120, sections=(60,))) == SHAPE
    assert append(v, rot=rotary(rot=144, sections=(72,))) == SHAPE
    assert append(v, rot=rotary(sections=(32, 31))) == SHAPE and append(v, rot=rotary(sections=(64, 0))) == SHAPE
    assert append(v, rot=rotary(inter=2)) == ARG
    assert append(v, rot=rotary(), q=BASE, heads=7, q_out=BASE) == SHAPE
    assert append(v, rot=rotary(), q=BASE, heads=8, q_out=0) == ARG
    assert append(v, n=0, k=0, vv=0, slots=0) == 0


def test_copy_arguments():
    lib, v = _abi.load(), view()
    assert lib.rkv_gqa_copy_pages(addressof(v), 0, BASE, 1, 0, 0) == ARG
    assert lib.rkv_gqa_copy_pages(addressof(v), BASE, BASE, -1, 0, 0) == SHAPE
    assert lib.rkv_gqa_copy_pages(addressof(v), BASE, BASE, 1 << 31, 0, 0) == SHAPE
    assert lib.rkv_gqa_copy_pages(addressof(v), 0, 0, 0, 0, 0) == 0


def test_python_layer_fails_loudly_without_cuda():
    import torch

    import rsllm_b200 as rk

    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    with pytest.raises(rk.CudaError):
        rk.GqaKvPool(4, 2, 128)
    with pytest.raises(rk.CudaError):
        rk.GqaKvPool.over(torch.zeros((1, 2, 2, 2, 64, 64), dtype=torch.bfloat16))
    with pytest.raises(rk.ShapeMismatch):
        rk.RotaryTable(torch.zeros((4, 32, 2)))
