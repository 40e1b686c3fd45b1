"""Whose check sees a device wait that gave up: a communicator's also those of GEMMs and linear layers on its device, and nobody's reading hides it from others."""
import contextlib

import pytest
import torch

from fast_b200 import runtime
from fast_b200.ops import gemm


class _Block:
    def __init__(self, *values):
        self.values = values or (0, 0, 0, 0, 0)

    def read(self):
        return self.values

    def clear(self):
        self.values = (0, 0, 0, 0, 0)


@pytest.mark.parametrize("where", ["own", "gemm", "linear"])
def test_a_communicators_check_reads_all_blocks(where, monkeypatch):
    from fast_b200.parallel import Communicator

    failed = (1, 8, 400, 0, 0)
    blocks = {name: _Block(*(failed if name == where else ())) for name in ("own", "gemm", "linear")}
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(gemm, "_status", blocks["gemm"])
    monkeypatch.setattr(runtime, "ext", lambda: type("C", (), {"dense_status": staticmethod(lambda: blocks["linear"])}))
    comm = Communicator.__new__(Communicator)
    comm.status, comm.device, comm.broken = blocks["own"], torch.device("cuda", 0), False
    for _ in range(2):            # reading takes nothing away
        with pytest.raises(runtime.CollectiveTimeout):
            comm.check()
        if where != "own":
            with pytest.raises(runtime.CollectiveTimeout):
                gemm.check()
    assert comm.broken == (where == "own")
    gemm.reset()
    if where != "own":
        comm.check()
        gemm.check()
    monkeypatch.setattr(gemm, "_status", None)   # no GEMM of the module has run yet
    blocks["own"].clear()
    comm.check()


@pytest.mark.gpu
def test_a_linear_layers_wait_that_gave_up_is_seen_by_the_layers_check():
    """The wait is that of a probe which nothing wakes, reported where linear layers on this device report."""
    from fast_b200.models import MoELayer
    from fast_b200.parallel import Communicator

    C = runtime.ext()
    comm, other = (Communicator(heap_bytes=64 << 20, device=0) for _ in range(2))
    layer = MoELayer(comm, 512, 256, 8, 2, max_tokens=64, shared_inter=128)
    x = torch.randn(16, 512, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        layer(x)
    comm.check()
    flag = torch.zeros(1, dtype=torch.int64, device="cuda")
    C.wait_probe(flag.data_ptr(), 1, C.dense_status(), 5_000_000)   # 5 ms
    for check in (comm.check, gemm.check, other.check, comm.check):
        with pytest.raises(runtime.CollectiveTimeout):
            check()
    comm.reset()
    for check in (comm.check, gemm.check, other.check):
        check()
    with torch.no_grad():
        layer(x)
    comm.check()
