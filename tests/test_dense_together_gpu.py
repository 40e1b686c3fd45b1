"""The dense operators one behind the other, as a block uses them, under what a training program does around them: checkpointing, several threads."""
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from fast_b200.ops import fused, gemm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _block():
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(300, 512, generator=g, device="cuda").to(BF)
    w1, w2 = ((torch.randn(*s, generator=g, device="cuda") * 0.05).to(BF).requires_grad_() for s in ((1024, 512), (512, 512)))
    nw = torch.ones(512, device="cuda", dtype=BF, requires_grad=True)
    idx = torch.zeros(300, 2, device="cuda", dtype=torch.int32)

    def run(a):
        r = fused.add_rms_norm(a, nw, residual=a)
        y = fused.linear(fused.linear(r.y, w1, activation="swiglu"), w2, activation="gelu", residual=r.h)
        return y.float().sum() + 3 * fused.balance_loss(y.float()[:, :8], idx)[0]

    return x, (w1, w2, nw), run


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_block_has_the_same_gradients(reentrant):
    x, weights, run = _block()
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    want = torch.autograd.grad(run(a), [a, *weights])
    checkpoint(run, b, use_reentrant=reentrant).backward()
    assert all(torch.equal(p, q) for p, q in zip(want, [b.grad, *(w.grad for w in weights)]))
    gemm.check()


@pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream")
def test_several_threads_on_streams_of_their_own():
    x, weights, run = _block()
    want = torch.autograd.grad(run(x.clone().requires_grad_()), weights)
    torch.cuda.synchronize()
    seen = []

    def work():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(15):
                got = torch.autograd.grad(run(x.clone().requires_grad_()), weights)
                stream.synchronize()
                seen.append(all(torch.equal(p, q) for p, q in zip(got, want)))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert seen == [True] * 60
    gemm.check()
