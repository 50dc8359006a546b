"""Attention over cache pages called from two threads: each call counts its own kernels (a stand-in for the library, no GPU)."""
import ctypes
import threading
from types import SimpleNamespace

import torch

from llmss_b200.ops import _lib
from llmss_b200.ops import cuda_impl as cu
from pages_oracle import make_batch, make_pages


def test_calls_of_two_threads_count_their_own_kernels(monkeypatch):
    batch, seen = make_batch([1, 1], [20, 30], 16, [], "cpu")
    k, v = (make_pages(seen.blocks, 2, 16, 64, torch.int8, torch.bfloat16, "cpu", seed=i) for i in range(2))
    both = threading.Barrier(2, timeout=30)

    def call(*args):
        hq = args[16]
        both.wait()                                  # inside of the library at the same time
        if hq == 4:
            ctypes.c_int.from_address(args[-2]).value = 3
            both.wait()
            both.wait()
        else:
            both.wait()
            ctypes.c_int.from_address(args[-2]).value = 1
            both.wait()
        return 0

    lib = SimpleNamespace(llmss_attn_pages_scratch_floats=lambda *a: 0, llmss_attn_pages=call)
    monkeypatch.setattr(_lib, "load", lambda *a, **kw: lib)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    monkeypatch.setattr(cu, "_stream", lambda: 0)
    counted = {}
    monkeypatch.setattr(cu, "_count", lambda n=1: counted.__setitem__(threading.get_ident(), n))
    got = {}

    def run(hq):
        q = torch.zeros(2, hq * 64, dtype=torch.bfloat16)
        cu.attention_pages(q, torch.empty_like(q), batch, k, v, hq, 2, 64, 0.1)
        got[hq] = counted[threading.get_ident()]

    threads = [threading.Thread(target=run, args=(hq,)) for hq in (4, 8)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert got == {4: 3, 8: 1}
