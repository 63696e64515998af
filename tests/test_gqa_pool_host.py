"""GqaKvPool's own bookkeeping, without a GPU: a pool over CPU tensors whose library is a stand-in that records what
it is given."""
import threading

import pytest
import torch

import rsllm_b200 as rk
from rsllm_b200 import gqa

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
    """make(during): (pool, decode, prefill); ``make.stream`` is the current stream's handle."""
    state = type("State", (), {"stream": 0})()
    monkeypatch.setattr(gqa, "_raw_stream", lambda index: state.stream)
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
