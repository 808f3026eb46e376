"""CPU tests of the paged operators' host side with a stand-in for the library."""
import ctypes

import torch

import tabinfer_b200.ops as ops


class _Lib:
    """notes the streams it is given; a workspace of 100 bytes a row"""
    def __init__(self):
        self.streams, self.queries = [], 0

    def tb_ctx_set_stream(self, h, s):
        self.streams.append(s.value)

    def size(self, h, kv, T, out):
        self.queries += 1
        out._obj.value = 100 * T
        return 0


class _Ctx:
    h = None

    def check(self, rc, what):
        assert rc == 0


def test_workspace_sizes_are_bounded(monkeypatch):
    lib = _Lib()
    monkeypatch.setattr(ops, "LIB", lib)
    monkeypatch.setattr(ops, "_ws_sizes", {})
    lens, kv = torch.zeros(1, dtype=torch.int32), bytes(88)
    for T in range(1, 5000):
        ws, n = ops._workspace(_Ctx(), "size", 0, kv, lens, T)
        assert n == max(256, 100 * T + 3 & ~3) and ws.numel() * 4 == n and ws.dtype is torch.int32
        assert len(ops._ws_sizes) <= 1024
    before = lib.queries
    ops._workspace(_Ctx(), "size", 0, kv, lens, 4999)
    assert lib.queries == before                              # the last size is known


def test_current_stream_with_and_without_the_raw_handle(monkeypatch):
    lib = _Lib()
    monkeypatch.setattr(ops, "LIB", lib)
    monkeypatch.setattr(torch.cuda, "init", lambda: None)

    class Stream:
        def __init__(self, device):
            self.cuda_stream = 0 if device == 0 else 4000 + device
    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    for raw in (None, lambda device: Stream(device).cuda_stream):
        monkeypatch.setattr(ops, "_raw_stream", raw)
        for device in (0, 3):
            c = object.__new__(ops.Context)
            c.h, c.device = None, device
            c.bind_stream()
    assert lib.streams == [ops.CUDA_STREAM_LEGACY, 4003] * 2
