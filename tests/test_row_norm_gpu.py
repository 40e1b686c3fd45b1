"""RMS norm with residual and e4m3 output against a plain implementation in 64 bits.

Tolerances count roundings: half a step of the type once for a value that is rounded once, and fp32 arithmetic (2^-24 an operation, a few
of them, and one more for each term that a thread adds in turn) relative to the magnitudes that are added."""
import pytest
import torch

from fast_b200 import runtime
from fast_b200.ops import fused

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0**-24


def half_step(t):
    return torch.finfo(t).eps / 2


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def plain(x, w, eps, residual=None):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)   # fp32 sum of two values, rounded to the type
    h64 = h.double()
    r = 1.0 / torch.sqrt(h64.pow(2).mean(-1, keepdim=True) + eps)
    return h, r, h64 * r * w.double()


def check_y(y, want, dtype):
    # a square root's reciprocal, a sum over the row, three products: 2^-18 relative covers 64 fp32 roundings
    err = (y.double() - want).abs()
    assert (err <= (half_step(dtype) + 64 * U) * want.abs() + 1e-37).all(), err.max().item()


@pytest.mark.parametrize("wtype", [BF, F32])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H", [(1, 1), (1, 4096), (3, 7), (5, 128), (17, 1001), (64, 1000), (33, 2048), (9, 7168), (7, 16384), (4, 32768), (3, 49152), (300, 264), (1300, 1003), (700, 8200), (160, 16383), (90, 9000), (640, 4104)])
def test_forward_and_gradients(T, H, dtype, wtype):
    x, res = rand((T, H), dtype, 1), rand((T, H), dtype, 2, 2.0)
    w = (1 + rand((H,), F32, 3, 0.2)).to(wtype)
    dy, dh = rand((T, H), dtype, 4), rand((T, H), dtype, 5)
    for residual in (None, res):
        leaves = [t.clone().requires_grad_() for t in ([x, w] if residual is None else [x, w, residual])]
        out = fused.add_rms_norm(leaves[0], leaves[1], 1e-5, residual=leaves[2] if residual is not None else None)
        h, r, y = plain(x, w, 1e-5, residual)
        assert torch.equal(out.h, h) and out.q is None and out.scales is None
        check_y(out.y, y, dtype)
        with torch.no_grad():   # the serving path gives the same bits
            again = fused.add_rms_norm(x, w, 1e-5, residual=residual)
        assert torch.equal(again.y, out.y) and torch.equal(again.h, h)
        grads = torch.autograd.grad([out.y] + [out.h] * (residual is not None), leaves, [dy] + [dh] * (residual is not None))
        hat, g = h.double() * r, dy.double() * w.double()
        s = (g * hat).mean(-1, keepdim=True)
        want = r * (g - hat * s) + (dh.double() if residual is not None else 0)
        size = r * (g.abs() + hat.abs() * (g * hat).abs().mean(-1, keepdim=True)) + (dh.double().abs() if residual is not None else 0)
        assert ((grads[0].double() - want).abs() <= half_step(dtype) * want.abs() + 64 * U * size).all()
        if residual is not None:
            assert torch.equal(grads[2], grads[0])
        p = dy.double() * hat
        assert ((grads[1].double() - p.sum(0)).abs() <= half_step(wtype) * p.sum(0).abs() + (64 + T) * U * p.abs().sum(0)).all()


def test_gradients_of_one_output_alone():
    x, res, w = rand((6, 512), BF, 1).requires_grad_(), rand((6, 512), BF, 2).requires_grad_(), rand((512,), BF, 3).requires_grad_()
    out = fused.add_rms_norm(x, w, residual=res)
    d = rand((6, 512), BF, 4)
    gx, gw, gr = torch.autograd.grad(out.h, [x, w, res], d, retain_graph=True)
    assert torch.equal(gx, d) and torch.equal(gr, d) and not gw.any()
    both = torch.autograd.grad(out.y, [x, res], d)
    assert torch.equal(both[0], both[1])
    frozen = fused.add_rms_norm(x, w.detach(), residual=res.detach())
    assert torch.autograd.grad(frozen.y, x, d)[0].shape == x.shape


def test_gradient_against_differences():
    T, H, step = 3, 96, 2.0**-7
    x, res, w = rand((T, H), F32, 1), rand((T, H), F32, 2), 1 + rand((H,), F32, 3, 0.3)
    cy, ch = rand((T, H), F32, 4).double(), rand((T, H), F32, 5).double()
    d = [rand((T, H), F32, 6), rand((H,), F32, 7), rand((T, H), F32, 8)]
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    out = fused.add_rms_norm(leaves[0], leaves[1], 1e-5, residual=leaves[2])
    grads = torch.autograd.grad([out.y, out.h], leaves, [cy.float(), ch.float()])
    for i in range(3):
        def value(sign):
            at = [t + sign * step * d[i] if j == i else t for j, t in enumerate((x, w, res))]
            o = fused.add_rms_norm(at[0], at[1], 1e-5, residual=at[2])
            return (o.y.double() * cy).sum() + (o.h.double() * ch).sum()
        slope = (value(1) - value(-1)) / (2 * step)
        want = (grads[i].double() * d[i].double()).sum()
        # third derivatives times step^2 (each row's sums are of the order of sqrt(H)) and fp32 roundings of T * H values divided by the step
        assert abs(slope - want) <= 50 * step**2 + 3 * T * H * U / step, (i, slope.item(), want.item())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H", [(1, 128), (5, 384), (40, 7168), (2, 16384), (3, 49152)])
def test_e4m3_rows_are_those_of_the_dispatch(T, H, dtype):
    C = runtime.ext()
    x, res, w = rand((T, H), dtype, 1, 4.0), rand((T, H), dtype, 2), 1 + rand((H,), F32, 3, 0.2)
    x[0, :128] = 0
    res[0, :128] = 0
    out = fused.add_rms_norm(x, w, residual=res, quantise=True)
    assert out.q.dtype == torch.uint8 and out.q.shape == (T, H) and out.scales.shape == (T, H // 128)
    if dtype == BF and H % 256 == 0 and H <= 16384:   # what the dispatch takes
        q, s = torch.empty_like(out.q), torch.empty_like(out.scales)
        C.quantise_rows(out.y, q, s, 148)
        assert torch.equal(q, out.q) and torch.equal(s, out.scales)
    y = out.y.double().view(T, -1, 128)
    back = out.q.view(torch.float8_e4m3fn).double().view(T, -1, 128) * out.scales.double().unsqueeze(-1)
    # e4m3: half a step of 2^-3 relative above its smallest normal number 2^-6, of 2^-9 absolute below; scale and quotient are rounded too
    assert ((back - y).abs() <= (2.0**-4 + 2.0**-20) * y.abs() + 2.0**-10 * out.scales.double().unsqueeze(-1)).all()
    amax = y.abs().amax(-1)
    live = amax > 1e-9
    assert (out.scales.double()[live] * 448 >= amax[live] * (1 - 2 * U)).all() and (out.scales.double()[live] * 448 <= amax[live] * (1 + 2.0**-6)).all()
    assert torch.equal(out.scales.bfloat16().float(), out.scales)
    read = fused.dequantise_rows(out.q, out.scales)
    assert ((read.double().view_as(back) - back).abs() <= half_step(BF) * back.abs()).all()
    leaf = x.clone().requires_grad_()
    trained = fused.add_rms_norm(leaf, w, residual=res, quantise=True)
    assert torch.equal(trained.q, out.q) and torch.equal(trained.scales, out.scales) and not trained.q.requires_grad and not trained.scales.requires_grad
    assert torch.autograd.grad(trained.y.float().sum(), leaf)[0].isfinite().all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_alignment_and_shapes(dtype):
    T, H = 13, 520
    w = 1 + rand((H,), F32, 3, 0.2)
    wide = rand((T, 2 * H + 3), dtype, 1)
    flat = rand((T * H + 1,), dtype, 2)
    views = [wide[:, :H], wide[:, 5:5 + H], wide[::2, :H], flat[1:].view(T, H), rand((H, T), dtype, 4).t(), rand((1, H), dtype, 5).expand(T, H), rand((3, 5, H), dtype, 6),
             rand((4, 3, 2 * H), dtype, 7)[:, :, ::2], rand((H,), dtype, 8)]
    for v in views:
        res = torch.flip(v, (0,))
        a, b = fused.add_rms_norm(v, w, residual=res), fused.add_rms_norm(v.contiguous().clone(), w, residual=res)
        assert a.y.shape == v.shape and torch.equal(a.h, b.h)
        check_y(a.y, plain(v, w, 1e-5, res)[2], dtype)
        check_y(fused.add_rms_norm(v, w).y, plain(v, w, 1e-5)[2], dtype)
        leaf = v.detach().requires_grad_()
        (g,) = torch.autograd.grad(fused.add_rms_norm(leaf, w).y, leaf, torch.ones_like(v))
        assert g.shape == v.shape and g.isfinite().all()
    q = fused.add_rms_norm(wide[:, 5:5 + 512], w[:512].contiguous(), quantise=True)
    p = fused.add_rms_norm(wide[:, 5:5 + 512].contiguous(), w[:512].contiguous(), quantise=True)
    assert ((q.y.double() - p.y.double()).abs() <= 2 * (half_step(dtype) + 64 * U) * p.y.double().abs()).all()
    assert ((fused.dequantise_rows(q.q, q.scales).double() - q.y.double()).abs() <= (2.0**-4 + 2.0**-7) * q.y.double().abs() + 2.0**-9 * q.scales.amax().item()).all()


def test_no_rows_and_rows_of_zeros_infinities_and_nan():
    w = torch.ones(256, device="cuda", dtype=BF, requires_grad=True)
    x = torch.empty(0, 256, device="cuda", dtype=BF, requires_grad=True)
    out = fused.add_rms_norm(x, w, residual=x, quantise=True)
    assert out.y.shape == (0, 256) and out.scales.shape == (0, 2)
    gx, gw = torch.autograd.grad(out.y, [x, w], torch.empty_like(x))
    assert gx.shape == (0, 256) and not gw.any()
    rows = rand((6, 256), BF, 1)
    clean = fused.add_rms_norm(rows, w.detach()).y
    rows[1], rows[3, 5], rows[4, 7] = 0, float("inf"), float("nan")
    y = fused.add_rms_norm(rows, w.detach()).y
    assert not y[1].any() and y[3].isnan().any() and y[4].isnan().all()
    assert all(torch.equal(y[i], clean[i]) for i in (0, 2, 5))


def test_offsets_past_32_bits():
    T, H = 70000, 32768   # 2.3e9 elements
    x = torch.zeros(T, H, device="cuda", dtype=BF)
    x[-3:] = rand((3, H), BF, 1)
    w = 1 + rand((H,), F32, 2, 0.1)
    out = fused.add_rms_norm(x, w, residual=x)
    check_y(out.y[-3:], plain(x[-3:], w, 1e-5, x[-3:])[2], BF)
    assert not out.y[:-3].any()
    del out
    leaf = x.requires_grad_()
    (g,) = torch.autograd.grad(fused.add_rms_norm(leaf, w).y, leaf, x.detach())
    h, r, _ = plain(x[-3:].detach(), w, 1e-5)
    hat, gw = h.double() * r, x[-3:].detach().double() * w.double()
    want = r * (gw - hat * (gw * hat).mean(-1, keepdim=True))
    size = r * (gw.abs() + hat.abs() * (gw * hat).abs().mean(-1, keepdim=True))
    assert ((g[-3:].double() - want).abs() <= half_step(BF) * want.abs() + 64 * U * size).all()


def test_other_stream_and_graph_replay():
    x, res, w = rand((50, 1024), BF, 1), rand((50, 1024), BF, 2), rand((1024,), BF, 3)
    want = fused.add_rms_norm(x, w, residual=res, quantise=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fused.add_rms_norm(x, w, residual=res, quantise=True)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph, a, b = torch.cuda.CUDAGraph(), x.clone(), res.clone()
    with torch.cuda.graph(graph):
        out = fused.add_rms_norm(a, w, residual=b, quantise=True)
    for seed in (7, 8):
        a.copy_(rand((50, 1024), BF, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, fused.add_rms_norm(a, w, residual=b, quantise=True)))


def test_training_step_captured_and_replayed():
    w = (1 + rand((768,), BF, 3, 0.1)).requires_grad_()
    x, res, dy, dh = (rand((90, 768), BF, s) for s in (1, 2, 4, 5))

    def step(a, b):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        out = fused.add_rms_norm(a, w, residual=b)
        return torch.autograd.grad([out.y, out.h], [a, w, b], [dy, dh])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, res)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step(x, res)
    for seed in (11, 12):
        x.copy_(rand((90, 768), BF, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, step(x, res)))


def test_its_backward_has_no_gradient():
    x, w = rand((3, 256), BF, 1).requires_grad_(), rand((256,), BF, 2).requires_grad_()
    g = torch.autograd.grad(fused.add_rms_norm(x, w, residual=x).y.float().sum(), [x, w], create_graph=True)
    for t in g:
        with pytest.raises(RuntimeError, match="no gradient"):
            t.float().sum().backward()
