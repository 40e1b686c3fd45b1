"""What lies behind a result in memory stays as it was, to the byte: results are made to land in front of bytes of a known value.

A block of a result's size is taken from the allocator in front of a guard, filled, and given back: the next allocation of that size gets it again (asserted), and every byte from
the result's end to the guard's end is read back afterwards. Sizes end inside tiles, boxes, words and rows of all kernels."""
import contextlib

import numpy as np
import pytest
import torch

from fast_b200 import runtime
from fast_b200.models.moe import interleave_gate_up
from fast_b200.ops import fused, gemm

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
MARK, SMALL = 0xA5, 1 << 20   # the allocator has one pool for up to 1 MiB and one for more: block, guard and both together have to be of one


def _at(size, where, held):
    """A block of `size` bytes at address `where`; what the allocator gives instead is held."""
    while True:
        t = torch.empty(size, dtype=torch.uint8, device="cuda")
        if t.data_ptr() == where:
            return t
        assert len(held) < 4096
        held.append(t)


def _bytes(ptr, size):
    from cuda.bindings import runtime as rt

    host = np.empty(size, np.uint8)
    (err,) = rt.cudaMemcpy(host.ctypes.data, ptr, size, rt.cudaMemcpyKind.cudaMemcpyDeviceToHost)
    assert int(err) == 0
    return host


@contextlib.contextmanager
def guarded(*sizes):
    """The next allocations of these many bytes land in front of guards, which are whole at the end; yields the addresses."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    held, spots = [], []
    for n in sizes:
        rounded = -(-n // 512) * 512
        behind = 4 * SMALL if rounded > SMALL else max(512, SMALL - rounded)
        assert rounded != SMALL
        region = torch.empty(rounded + behind, dtype=torch.uint8, device="cuda")
        where = region.data_ptr()
        del region
        block = _at(rounded, where, held)
        guard = _at(behind, where + rounded, held)
        block.fill_(MARK), guard.fill_(MARK)
        spots.append((where, n, rounded + behind, block, guard))
    torch.cuda.synchronize()
    guards = [s[4] for s in spots]
    spots = [s[:3] for s in spots]
    block = guard = None   # the blocks are free again
    yield [s[0] for s in spots]
    torch.cuda.synchronize()
    for where, n, end in spots:
        behind = _bytes(where + n, end - n)
        assert (behind == MARK).all(), (n, int((behind != MARK).nonzero()[0][0]))
    del guards, held


def whole(shape, seed, most=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda", dtype=torch.int8).to(BF)


def path(*a, **kw):
    return runtime.ext().dense_path(*a, **kw)


# (tokens, inputs, outputs): few tokens, one and several token tiles; tiles of 256 features, uncut, cut as a stream and in parts; tiles of up to 512 tokens
LINEAR = [(33, 128, 264, True), (1, 8, 8, True), (250, 1104, 2056, True), (333, 512, 20040, False), (1235, 1000, 2760, False), (100, 8192, 20000, False), (781, 7256, 1368, False), (8200, 8200, 3432, False)]


@pytest.mark.parametrize("act,extra", [(None, False), ("relu", True)])
@pytest.mark.parametrize("T,K,N,few", LINEAR)
def test_behind_a_linear_layer_and_what_it_keeps(T, K, N, few, act, extra):
    assert path(T, N, K, False, not extra, K % 16 == 0)["few"] == few
    x, w = whole((T, K), 1), whole((N, K), 2)
    b, r = (whole((N,), 3), whole((T, N), 4)) if extra else (None, None)
    z = x.double() @ w.double().t()
    want = (torch.relu(z + b.double()) + r.double() if extra else z).to(BF)
    del z
    with torch.no_grad(), guarded(2 * T * N) as (where,):
        y = fused.linear(x, w, bias=b, activation=act, residual=r)
        assert y.data_ptr() == where and torch.equal(y, want)
    if not extra:
        return
    del y
    lx = x.clone().requires_grad_()
    with guarded(2 * T * N, 2 * T * N) as where:              # the result and the pre-activation
        y = fused.linear(lx, w, bias=b, activation=act, residual=r)
        assert y.data_ptr() in where and torch.equal(y, want)
        torch.cuda.synchronize()
        other = where[1 - where.index(y.data_ptr())]
        assert not (_bytes(other, min(2 * T * N, 4096)) == MARK).all()      # the other one is in use too
    gemm.check()


@pytest.mark.parametrize("T,K,I,few", [(33, 128, 256, True), (250, 1032, 1024, True), (333, 512, 10368, False), (129, 7512, 2432, False), (972, 7256, 640, False)])
def test_behind_swiglu_and_what_it_keeps(T, K, I, few):
    assert path(T, 2 * I, K, True, False, True)["few"] == few
    w = interleave_gate_up(whole((1, I, K), 2, 1), whole((1, I, K), 3, 1))[0]
    x = whole((T, K), 1, 1)
    with torch.no_grad(), guarded(2 * T * I) as (where,):
        y = fused.linear(x, w, activation="swiglu")
        assert y.data_ptr() == where
    want = y
    lx = x.clone().requires_grad_()
    with guarded(2 * T * I, 8 * T * I) as where:              # gate and up, twice 16 bits each
        y = fused.linear(lx, w, activation="swiglu")
        assert y.data_ptr() == where[0] and torch.equal(y, want)
        torch.cuda.synchronize()
        kept = torch.from_numpy(_bytes(where[1], 8 * T * I)).cuda().view(torch.bfloat16).view(T, 4 * I)
        z = x.double() @ w.double().t()
        assert torch.equal(kept[:, :2 * I].double() + kept[:, 2 * I:].double(), z)      # whole numbers below 2^16
    gemm.check()


@pytest.mark.parametrize("T,K,N", [(33, 136, 264), (1235, 1000, 2760), (8000, 1000, 1032), (4280, 136, 3376), (333, 20040, 512), (8200, 3432, 8200)])
def test_behind_the_gradients_of_a_linear_layer(T, K, N):
    """Data gradient, weight gradient (its rows shared out or not), bias gradient; dz in between."""
    x, w, b, dy = whole((T, K), 1).requires_grad_(), whole((N, K), 2).requires_grad_(), whole((N,), 3).requires_grad_(), whole((T, N), 4)
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    dz = dy.double() * (z > 0)
    sizes = {"x": 2 * T * K, "weight": 2 * N * K, "bias": 2 * N}
    for name, leaf, want in (("x", x, dz @ w.detach().double()), ("weight", w, dz.t() @ x.detach().double()), ("bias", b, dz.sum(0))):
        y = fused.linear(x, w, bias=b, activation="relu")
        with guarded(sizes[name], 2 * T * N) as where:
            (g,) = torch.autograd.grad(y, leaf, dy)
            assert g.data_ptr() in where and torch.equal(g, want.to(BF)), name
        del g, y
    gemm.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,quantise", [(1, 1, False), (3, 7, False), (5, 384, True), (17, 1001, False), (7, 16384, True), (301, 264, False), (90, 9000, False), (33, 4097, False), (4, 32768, False), (3, 49152, True)])
def test_behind_the_norm_and_its_gradients(T, H, quantise, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, res, w, dy, dh = ((torch.randn(*s, generator=g, device="cuda")).to(dtype).requires_grad_(i < 3) for i, s in enumerate(((T, H), (T, H), (H,), (T, H), (T, H))))
    rows = x.element_size() * T * H
    with torch.no_grad():
        want = fused.add_rms_norm(x, w, residual=res, quantise=quantise)
    with torch.no_grad(), guarded(rows, rows, *([T * H, T * H // 32] if quantise else [])) as where:
        out = fused.add_rms_norm(x, w, residual=res, quantise=quantise)
        assert {t.data_ptr() for t in out if t is not None} == set(where)
        assert all(torch.equal(a, b) for a, b in zip(out, want) if a is not None)
    del out
    kept = fused.add_rms_norm(x, w, residual=res)
    grads = torch.autograd.grad([kept.y, kept.h], [x, w], [dy, dh], retain_graph=True)
    with guarded(rows, x.element_size() * H) as where:
        again = torch.autograd.grad([kept.y, kept.h], [x, w], [dy, dh], retain_graph=True)
        assert again[0].data_ptr() == where[0] and all(torch.equal(a, b) for a, b in zip(again, grads))


@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (61, 64, 6), (2049, 33, 4), (700, 257, 8), (20011, 8, 2)])
def test_behind_the_balance_loss(T, E, K):
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(T, E, generator=g, device="cuda").requires_grad_()
    idx = torch.randint(0, E, (T, K), generator=g, device="cuda").to(torch.int32)
    loss, counts = fused.balance_loss(logits, idx)
    one = torch.ones((), device="cuda")
    (want,) = torch.autograd.grad(loss, logits, one, retain_graph=True)
    with guarded(4 * T * E) as (where,):
        (got,) = torch.autograd.grad(loss, logits, one, retain_graph=True)
        assert got.data_ptr() == where and torch.equal(got, want)
    with guarded(4 * E, 4 * (E + 1)) as where:
        again, cnt = fused.balance_loss(logits.detach(), idx)
        assert cnt.data_ptr() in where and torch.equal(cnt, counts)
