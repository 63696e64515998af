"""GqaKvPool's own bookkeeping, without a GPU: a pool over CPU tensors whose library is a stand-in that records what
it is given."""
import threading
from ctypes import addressof

import pytest
import torch

import rsllm_b200 as rk
from rsllm_b200 import _abi, gqa

BF = torch.bfloat16


class Lib:
    """Every attention call runs ``during(name, workspace, stream)``."""

    def __init__(self, during=lambda *a: None):
        self.during = during

    def rkv_gqa_prefill_workspace_bytes(self, view):
        return 4096

    def rkv_gqa_decode_workspace_bytes(self, view, n_seq, heads):
        return 1024

    def rkv_gqa_decode(self, *a):
        self.during("decode", a[13], a[16])
        return 0

    def rkv_gqa_prefill(self, *a):
        self.during("prefill", a[15], a[18])
        return 0

    def rkv_gqa_append(self, *a):
        self.during("append", 0, a[18])
        return 0

    def rkv_gqa_copy_pages(self, *a):
        self.during("copy", 0, a[5])
        return 0


@pytest.fixture
def make(monkeypatch):
    """make(during): (pool, decode, prefill); ``make.state`` holds the current stream's handle and the current device
    (CPU tensors are on "device" -1)."""
    state = type("State", (), {"stream": 0, "device": -1})()
    monkeypatch.setattr(gqa, "_raw_stream", lambda index: state.stream)
    monkeypatch.setattr(gqa, "_current_device", lambda: state.device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)

    def build(during):
        lib = Lib(during)
        monkeypatch.setattr(gqa._abi, "load", lambda: lib)
        pool = gqa.GqaKvPool.__new__(gqa.GqaKvPool)
        pool._bind(torch.zeros((1, 4, 2, 2, 64, 64), dtype=BF), None)
        q = torch.zeros((1, 4, 64), dtype=BF)
        lens, table = torch.tensor([5], dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32)
        cu = torch.tensor([0, 1], dtype=torch.int32)
        return pool, lambda: pool.decode(0, q, table, lens), lambda: pool.prefill(0, q, cu, table, lens)

    build.state = state
    return build


def test_threads_of_one_stream_have_workspaces_of_their_own(make):
    """An attention is two launches, and two threads may queue theirs in turn: each must find its own partial results
    there.  Both threads are inside the call together."""
    inside = threading.Barrier(2, timeout=20)
    seen, errors = [], []

    def during(name, workspace, stream):
        seen.append((threading.get_ident(), workspace))
        inside.wait()

    pool, decode, prefill = make(during)

    def work():
        try:
            for call in (decode, prefill, decode, prefill):
                call()
        except Exception as e:  # a barrier that broke
            errors.append(e)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(seen) == 8
    a, b = ({w for who, w in seen if who == t.ident} for t in threads)
    assert a and b and not a & b


def test_a_thread_keeps_one_workspace_a_stream(make):
    seen = []
    pool, decode, prefill = make(lambda name, workspace, stream: seen.append((stream, workspace)))
    prefill()  # the larger one
    first = seen[0][1]
    decode(), prefill(), decode()
    assert seen == [(0, first)] * 4
    make.state.stream = 77
    decode()
    decode()
    assert seen[4] == seen[5] and seen[4][0] == 77 and seen[4][1] != first
    make.state.stream = 0
    decode()
    assert seen[6] == (0, first)


def test_calls_run_on_the_pools_device(make, monkeypatch):
    """With another device current, every call makes the pool's own current until it is back: the library launches,
    and a capture is asked about, on the current one."""
    calls = []
    pool, decode, prefill = make(lambda name, workspace, stream: calls.append((name, make.state.device)))

    class Guard:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, make.state.device = make.state.device, self.index

        def __exit__(self, *exc):
            make.state.device = self.before

    def capturing():
        calls.append(("capturing", make.state.device))
        return False

    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", capturing)
    k = torch.zeros((1, 2, 64), dtype=BF)
    one = torch.tensor([1], dtype=torch.int32)
    for current in (-1, 3):
        make.state.device = current
        calls.clear()
        decode()
        prefill()
        pool.append(0, k, k, one)
        pool.copy_pages(one, one)
        pool.apply_moves([1, 1], [2, 3])
        assert {name for name, _ in calls} == {"decode", "prefill", "append", "copy", "capturing"}
        assert all(device == -1 for _, device in calls), calls
        assert make.state.device == current
        with pytest.raises(rk.ShapeMismatch):  # and after an error
            pool.append(0, k[:, :1], k, one)
        assert make.state.device == current


def test_a_stream_of_another_device_is_refused(make):
    calls = []
    pool, *_ = make(lambda *a: calls.append(a))
    k = torch.zeros((1, 2, 64), dtype=BF)
    q = torch.zeros((1, 4, 64), dtype=BF)
    one = torch.tensor([1], dtype=torch.int32)
    table = torch.zeros((1, 2), dtype=torch.int32)
    cu = torch.tensor([0, 1], dtype=torch.int32)
    other = type("Stream", (), {"device_index": 1, "cuda_stream": 5})()
    for call in (lambda: pool.append(0, k, k, one, stream=other), lambda: pool.copy_pages(one, one, stream=other),
                 lambda: pool.decode(0, q, table, one, stream=other),
                 lambda: pool.prefill(0, q, cu, table, one, stream=other)):
        with pytest.raises(rk.InvalidArgument):
            call()
    assert not calls


def test_prefill_refuses_a_broadcast_q():
    """A stride of 0 between tokens or heads, before anything is launched; with one of them it is of no use."""
    base = 0x100000
    view = _abi.GqaView(base, 8, 2, 2, 128, _abi.GQA_BF16)

    def prefill(n, heads, ts, hs, cu=base):
        return _abi.load().rkv_gqa_prefill(addressof(view), 0, base, ts, hs, n, heads, cu, 1, base, 4, base, 0, 0, 0.1,
                                           base, base, 0, 0)

    assert prefill(2, 8, 0, 128) == _abi.RKV_ERR_SHAPE_MISMATCH
    assert prefill(2, 8, 1024, 0) == _abi.RKV_ERR_SHAPE_MISMATCH
    assert prefill(1, 8, 0, 128, cu=0) == _abi.RKV_ERR_INVALID_ARGUMENT  # refused for its offsets only
