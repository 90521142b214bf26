"""GPU tests of the windowed attention (sliding window, sink tokens, grouped k / v heads) and its
gradients against the formulas in 64 bits (window_reference.py derives the bounds)."""
from __future__ import annotations

import pytest
import torch

import mini_flash_attention as mfa
from mini_flash_attention import capi
from window_reference import check, reference, visible

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])


def randn(shape, seed, dtype=torch.float16):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


def inputs(b, h, hk, n, d, dtype, seed=7):
    return (randn((b, h, n, d), seed, dtype), randn((b, hk, n, d), seed + 1, dtype),
            randn((b, hk, n, d), seed + 2, dtype), randn((b, h, n, d), seed + 3, dtype))


# one token; a block and one more; windows of 1, one block less one, one block, more than the
# sequence; sinks inside, at and past a block's end, more than the sequence
SHAPES = [
    (1, 1, 1, 1, 1, 0), (2, 2, 1, 2, 1, 1), (1, 3, 1, 63, 16, 0), (1, 2, 2, 128, 128, 0),
    (1, 2, 1, 129, 1, 0), (1, 4, 2, 129, 127, 1), (2, 5, 1, 255, 64, 4), (1, 2, 2, 256, 128, 128),
    (1, 6, 2, 257, 129, 129), (1, 2, 1, 300, 1000, 50), (1, 2, 2, 300, 50, 1000),
    (1, 3, 3, 777, 128, 4), (2, 8, 2, 1000, 256, 130), (1, 4, 1, 1153, 200, 0),
    (1, 2, 1, 2000, 2, 300), (1, 4, 4, 2048, 512, 16),
]


@pytest.mark.parametrize("d", [32, 64, 128])
@TYPES
@pytest.mark.parametrize("b,h,hk,n,window,sinks", SHAPES)
def test_forward(b, h, hk, n, window, sinks, dtype, d):
    q, k, v, _ = inputs(b, h, hk, n, d, dtype)
    want = reference(q, k, v, window, sinks)
    out, lse = mfa.forward_window_lse(q, k, v, window, sinks)
    assert out.dtype == dtype and lse.dtype == torch.float32
    check("out", out, *want["out"])
    check("lse", lse, *want["lse"])
    assert torch.equal(out, mfa.forward_window(q, k, v, window, sinks))


@pytest.mark.parametrize("d", [32, 64, 128])
@TYPES
@pytest.mark.parametrize("b,h,hk,n,window,sinks", SHAPES)
def test_gradients(b, h, hk, n, window, sinks, dtype, d):
    q, k, v, dout = inputs(b, h, hk, n, d, dtype)
    want = reference(q, k, v, window, sinks, dout)
    out, lse = mfa.forward_window_lse(q, k, v, window, sinks)
    for name, x in zip(("dq", "dk", "dv"),
                       mfa.backward_window(q, k, v, out, lse, dout, window, sinks)):
        assert x.dtype == dtype
        check(name, x, *want[name])


# units in pieces: few heads and long reaches (every key block's unit is cut), and sink blocks
# alone cut
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("b,h,hk,n,window,sinks", [
    (1, 1, 1, 4096, 4096, 0), (1, 8, 1, 2048, 2048, 0), (1, 4, 1, 3000, 128, 200),
    (1, 16, 2, 2500, 300, 4), (2, 2, 2, 4000, 1, 1),
])
def test_gradients_in_pieces(b, h, hk, n, window, sinks, d):
    q, k, v, dout = inputs(b, h, hk, n, d, torch.bfloat16, seed=31)
    want = reference(q, k, v, window, sinks, dout)
    out, lse = mfa.forward_window_lse(q, k, v, window, sinks)
    first = mfa.backward_window(q, k, v, out, lse, dout, window, sinks)
    for name, x in zip(("dq", "dk", "dv"), first):
        check(name, x, *want[name])
    again = mfa.backward_window(q, k, v, out, lse, dout, window, sinks)
    assert all(torch.equal(x, y) for x, y in zip(first, again))


# far more units than CTAs: every buffer and ring entry is used again, with and without pieces
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("b,h,hk,n,window,sinks", [
    (16, 8, 8, 700, 130, 0), (3, 32, 8, 1100, 256, 4),
])
def test_gradients_many_units(b, h, hk, n, window, sinks, d):
    q, k, v, dout = inputs(b, h, hk, n, d, torch.float16, seed=57)
    out, lse = mfa.forward_window_lse(q, k, v, window, sinks)
    got = mfa.backward_window(q, k, v, out, lse, dout, window, sinks)
    for i in range(0, b, 2):
        part = [x[i:i + 1] for x in (q, k, v)]
        want = reference(*part, window, sinks, dout[i:i + 1])
        for name, x in zip(("dq", "dk", "dv"), got):
            check(name, x[i:i + 1], *want[name])


# what lies before and behind a gradient stays as it was (a block's rows past the last token, the
# columns past D = 32)
@pytest.mark.parametrize("layout", [capi.LAYOUT_BHND, capi.LAYOUT_BNHD], ids=["bhnd", "bnhd"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("n,window,sinks", [(1, 1, 0), (77, 10, 3), (2050, 2050, 1)])
def test_gradients_write_nothing_else(n, window, sinks, d, layout):
    b, h, hk = 2, 4, 2
    q, k, v, dout = inputs(b, h, hk, n, d, torch.float16, seed=91)
    want = reference(q, k, v, window, sinks, dout)
    turn = (lambda x: x) if layout == capi.LAYOUT_BHND else lambda x: x.transpose(1, 2).contiguous()
    x = [turn(t) for t in (q, k, v, dout)]
    room = 256 * d
    buffers = [torch.full((t.numel() + 2 * room,), 7.0, device="cuda", dtype=torch.float16)
               for t in (q, q, k, v)]
    out, dq, dk, dv = [t[room:-room] for t in buffers]
    lse = torch.empty((b, h, n), device="cuda")
    common = dict(dtype=capi.DTYPE_FP16, layout=layout,
                  stream=torch.cuda.current_stream().cuda_stream)
    capi.fwd_window(*(t.data_ptr() for t in x[:3]), out.data_ptr(), lse.data_ptr(), b, h, hk, n, d,
                    window, sinks, d ** -0.5, **common)
    capi.bwd_window(*(t.data_ptr() for t in x[:3]), out.data_ptr(), x[3].data_ptr(),
                    lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), b, h, hk, n, d,
                    window, sinks, d ** -0.5, **common)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, dq, dk, dv)):
        heads = h if name in ("out", "dq") else hk
        shape = (b, heads, n, d) if layout == capi.LAYOUT_BHND else (b, n, heads, d)
        check(name, turn(got.view(shape)), *want[name])
    for t in buffers:
        assert (t[:room] == 7).all() and (t[-room:] == 7).all()


def test_whole_window_is_causal_attention():
    q, k, v, _ = inputs(2, 4, 4, 1500, 64, torch.float16)
    want = mfa.forward(q, k, v, causal=True).double()
    got = mfa.forward_window(q, k, v, 1500)
    # the same formula, other partial sums: one rounding of the output each, and the weights'
    bound = reference(q, k, v, 1500, 0)["out"][1]
    assert ((got.double() - want).abs() <= 2 * bound).all()


def test_large_scores():
    # scores of hundreds: the running maximum moves often, weights underflow
    q, k, v, dout = inputs(1, 2, 1, 700, 64, torch.float16)
    q, k = q * 8, k * 8
    want = reference(q, k, v, 150, 3, dout)
    out, lse = mfa.forward_window_lse(q, k, v, 150, 3)
    # a score of up to about 500 is off by up to 64 products' 2^-24 relative in 32 bits, and its
    # logarithm base 2 by one more step: at most 2e-4 * 4 in the exponent
    value, bound = want["out"]
    check("out", out, value, 5 * bound)
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("d", [32, 64, 128])
def test_autograd_and_differences(d):
    q, k, v, dout = inputs(1, 4, 2, 200, d, torch.float16)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = mfa.window_attention(*leaves, 50, 2)
    grads = torch.autograd.grad(out, leaves, dout)
    want = reference(*(x.detach() for x in leaves), 50, 2, dout)
    for name, x in zip(("dq", "dk", "dv"), grads):
        check(name, x, *want[name])
    # against differences of the formula in 64 bits along a random direction
    direction = [torch.randn_like(x, dtype=torch.float64) for x in leaves]

    def loss(step):
        x, y, z = (t.detach().double() + step * w for t, w in zip(leaves, direction))
        y, z = (t.repeat_interleave(2, 1) for t in (y, z))
        s = x @ y.transpose(-1, -2) * d ** -0.5
        s = s.masked_fill(~visible(200, 50, 2, x.device), -torch.inf)
        return (torch.softmax(s, -1) @ z * dout.double()).sum()

    slope = ((loss(1e-5) - loss(-1e-5)) / 2e-5).item()
    ours = sum((g.double() * w).sum() for g, w in zip(grads, direction)).item()
    room = sum((want[m][1] * w.abs()).sum().item()
               for m, w in zip(("dq", "dk", "dv"), direction))
    assert abs(ours - slope) <= room + 1e-4 * abs(slope)


def test_broadcast_output_gradient_and_second_order():
    q, k, v, _ = inputs(1, 2, 1, 130, 64, torch.bfloat16)
    q.requires_grad_()
    out = mfa.window_attention(q, k, v, 20, 1)
    (dq,) = torch.autograd.grad(out.sum(), q, create_graph=True)  # dout has stride 0
    want = reference(q.detach(), k, v, 20, 1, torch.ones_like(q))
    check("dq", dq.detach(), *want["dq"])
    with pytest.raises(RuntimeError):
        dq.sum().backward()


def test_other_stream_and_captured_step():
    q, k, v, dout = inputs(1, 4, 2, 1000, 64, torch.float16)
    out, lse = mfa.forward_window_lse(q, k, v, 200, 4)
    want = (out, *mfa.backward_window(q, k, v, out, lse, dout, 200, 4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out2, lse2 = mfa.forward_window_lse(q, k, v, 200, 4)
        got = (out2, *mfa.backward_window(q, k, v, out2, lse2, dout, 200, 4))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # the step in two graphs, replayed on new inputs, in turn
    graphs = []
    for _ in range(2):
        buffers = [torch.zeros_like(x) for x in (q, k, v, dout)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, l = mfa.forward_window_lse(*buffers[:3], 200, 4)
            result = (o, *mfa.backward_window(*buffers[:3], o, l, buffers[3], 200, 4))
        graphs.append((graph, buffers, result))
    for seed in (7, 50):
        x = inputs(1, 4, 2, 1000, 64, torch.float16, seed=seed)
        o, l = mfa.forward_window_lse(*x[:3], 200, 4)
        want = (o, *mfa.backward_window(*x[:3], o, l, x[3], 200, 4))
        for graph, buffers, _ in graphs:
            for to, t in zip(buffers, x):
                to.copy_(t)
            graph.replay()
        for _, _, result in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, result))


@pytest.mark.parametrize("n,d", [(700, 64), (700, 128), (1300, 128), (1300, 32)])
def test_captured_autograd_step(n, d):
    # the whole step in a graph (as for any operator, no eager graph of the leaves may live then)
    q, k, v, dout = inputs(1, 4, 2, n, d, torch.float16)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    want_out = mfa.window_attention(*leaves, 100, 3)
    want = torch.autograd.grad(want_out, leaves, dout)
    want_out = want_out.detach().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mfa.window_attention(*leaves, 100, 3)
        got = torch.autograd.grad(out, leaves, dout)
    graph.replay()
    assert torch.equal(out, want_out) and all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("d", [64, 128])
def test_two_graphs_and_two_streams(d):
    """Steps of two layers captured apart and replayed together on two streams, again and again:
    each has workspaces, counters and results of its own."""
    steps = []
    for seed, (h, hk, n, window, sinks) in enumerate(((8, 2, 2500, 300, 4), (4, 4, 1000, 1000, 0))):
        q, k, v, dout = inputs(1, h, hk, n, d, torch.bfloat16, seed=20 * seed)
        out, lse, rest = mfa.forward_window_lse(q, k, v, window, sinks, rest=True)
        want = (out, lse, *mfa.backward_window(q, k, v, out, lse, dout, window, sinks, rest))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, s, r = mfa.forward_window_lse(q, k, v, window, sinks, rest=True)
            got = (o, s, *mfa.backward_window(q, k, v, o, s, dout, window, sinks, r))
        steps.append((graph, got, want, torch.cuda.Stream(), (q, k, v, dout)))
    torch.cuda.synchronize()
    for _ in range(5):
        for _, got, *_ in steps:
            for x in got:
                x.zero_()
        torch.cuda.synchronize()
        for graph, _, _, stream, _ in steps:
            with torch.cuda.stream(stream):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for _, got, want, *_ in steps:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_capi_bnhd_layout():
    b, h, hk, n, window, sinks = 2, 4, 2, 333, 70, 5
    q, k, v, dout = inputs(b, h, hk, n, 64, torch.bfloat16)
    want = reference(q, k, v, window, sinks, dout)
    t = [x.transpose(1, 2).contiguous() for x in (q, k, v, dout)]
    out, dq, dk, dv = (torch.empty_like(x) for x in (t[0], t[0], t[1], t[2]))
    lse = torch.empty((b, h, n), device="cuda", dtype=torch.float32)
    stream = torch.cuda.current_stream().cuda_stream
    common = dict(dtype=capi.DTYPE_BF16, layout=capi.LAYOUT_BNHD, stream=stream)
    ptr = [x.data_ptr() for x in t]
    capi.fwd_window(*ptr[:3], out.data_ptr(), lse.data_ptr(), b, h, hk, n, 64, window, sinks,
                    0.125, **common)
    capi.bwd_window(*ptr[:3], out.data_ptr(), ptr[3], lse.data_ptr(), dq.data_ptr(),
                    dk.data_ptr(), dv.data_ptr(), b, h, hk, n, 64, window, sinks, 0.125, **common)
    for name, x in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        check(name, x.transpose(1, 2), *want[name])
    check("lse", lse, *want["lse"])
    assert capi.device_status(torch.cuda.current_device()) == 0


# parts of a fused projection [B, N, (H + 2 Hkv) D], with one gradient for all of them
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("b,h,hk,n,window,sinks", [(2, 4, 2, 300, 70, 3), (1, 1, 1, 150, 40, 0),
                                                   (3, 6, 1, 1, 5, 0), (1, 8, 8, 2100, 2100, 0)])
def test_views_of_a_projection(b, h, hk, n, window, sinks, d):
    q, k, v, dout = inputs(b, h, hk, n, d, torch.bfloat16, seed=11)
    want = reference(q, k, v, window, sinks, dout)
    fused = torch.cat([x.transpose(1, 2).reshape(b, n, -1) for x in (q, k, v)], 2)
    fused.requires_grad_()
    parts = [x.view(b, n, -1, d).transpose(1, 2) for x in fused.split((h * d, hk * d, hk * d), 2)]
    out = mfa.window_attention(*parts, window, sinks)
    check("out", out.detach(), *want["out"])
    merged = out.transpose(1, 2)
    assert merged.is_contiguous()  # ready for the next projection
    merged.reshape(b, n, -1).backward(dout.transpose(1, 2).reshape(b, n, -1))
    grads = fused.grad.split((h * d, hk * d, hk * d), 2)
    for name, x in zip(("dq", "dk", "dv"), grads):
        check(name, x.view(b, n, -1, d).transpose(1, 2), *want[name])


@pytest.mark.parametrize("d", [32, 64, 128])
def test_mixed_layouts(d):
    """Each tensor in another layout: bit for bit the results of contiguous ones."""
    q, k, v, dout = inputs(2, 6, 3, 333, d, torch.float16, seed=5)
    out, lse = mfa.forward_window_lse(q, k, v, 100, 2)
    want = mfa.backward_window(q, k, v, out, lse, dout, 100, 2)
    room = randn((2, 7, 400, d + 8), 3)
    room[:, 2:5, 17:350, 8:] = v
    for x in (q, q.transpose(1, 2).contiguous().transpose(1, 2),
              q.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)):
        y = (x, k.transpose(1, 2).contiguous().transpose(1, 2), room[:, 2:5, 17:350, 8:])
        o, s = mfa.forward_window_lse(*y, 100, 2)
        assert torch.equal(o, out) and torch.equal(s, lse) and torch.equal(
            mfa.forward_window(*y, 100, 2), out)
        for other in (dout, dout.transpose(1, 2).contiguous().transpose(1, 2)):
            got = mfa.backward_window(*y, o, s, other, 100, 2)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            assert all(a.is_contiguous() == x.is_contiguous() for a in got)
    with pytest.raises(RuntimeError, match="lse must be contiguous"):
        mfa.backward_window(q, k, v, out, lse.transpose(0, 1).contiguous().transpose(0, 1), dout,
                            100, 2)


@pytest.mark.parametrize("d", [32, 64, 128])
@TYPES
@pytest.mark.parametrize("b,h,hk,n,window,sinks", [(2, 2, 1, 1, 1, 0), (1, 4, 2, 300, 40, 3),
                                                   (1, 3, 3, 1153, 200, 0), (2, 6, 2, 257, 257, 0)])
def test_rest_of_the_output(b, h, hk, n, window, sinks, dtype, d):
    q, k, v, dout = inputs(b, h, hk, n, d, dtype, seed=77)
    want = reference(q, k, v, window, sinks, dout)
    out, lse, rest = mfa.forward_window_lse(q, k, v, window, sinks, rest=True)
    plain = mfa.forward_window_lse(q, k, v, window, sinks)
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
    # the output's rounding is out of the bound, the rest's own in it: u |rest| <= u^2 |out| (1 + u),
    # or half of fp16's smallest step
    u = torch.finfo(dtype).eps / 2
    value, bound = want["out"]
    bound = bound - u * value.abs() + 1.01 * u * u * value.abs() + 2.0 ** -25
    assert ((out.double() + rest.double() - value).abs() <= bound).all()
    assert (rest.double().abs() <= 1.01 * u * out.double().abs() + 2.0 ** -24).all()
    turned = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    got = mfa.backward_window(q, k, v, out, lse, dout, window, sinks, rest)
    for name, x in zip(("dq", "dk", "dv"), got):
        check(name, x, *want[name])
    again = mfa.backward_window(q, k, v, out, lse, dout, window, sinks, turned(rest))
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    views = [turned(x) for x in (q, k, v)]
    same = mfa.forward_window_lse(*views, window, sinks, rest=True)
    assert all(torch.equal(x, y) for x, y in zip(same, (out, lse, rest)))
    for x in (rest[..., :16], rest.float(), rest.cpu()):
        with pytest.raises(RuntimeError, match="rest must have"):
            mfa.backward_window(q, k, v, out, lse, dout, window, sinks, x)


@TYPES
@pytest.mark.parametrize("window", [2, 3, 8])
def test_few_visible_keys(window, dtype):
    """dq and dk of rows that see few keys. Three roundings of about the same size make up their
    error: their own, that of dS and, through the row sums, that of the forward's weights; so
    it is at most 3 ** 0.5 times that of the first alone (and 1 in 100 for chance). The rounding of
    the output, were it in the row sums, would make that 2.3 at two keys."""
    q, k, v, dout = inputs(1, 4, 2, 1000, 64, dtype, seed=3)
    want = reference(q, k, v, window, 0, dout)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(mfa.window_attention(*leaves, window), leaves, dout)
    for name, x in zip(("dq", "dk"), grads):
        value = want[name][0]
        error = (x.double() - value).norm() / (value.to(dtype).double() - value).norm()
        assert error <= 3 ** 0.5 * 1.01, (name, error.item())


def test_without_gradients():
    q, k, v, _ = inputs(1, 4, 2, 150, 64, torch.float16)
    want = mfa.forward_window(q, k, v, 40, 2)
    assert torch.equal(mfa.window_attention(q, k, v, 40, 2), want)
    k.requires_grad_()
    with torch.no_grad():
        out = mfa.window_attention(q, k, v, 40, 2)
    assert torch.equal(out, want) and not out.requires_grad
    del out
    before = torch.cuda.memory_allocated()
    out = mfa.window_attention(q, k, v, 40, 2)
    assert torch.equal(out, want) and out.requires_grad
    del out
    assert torch.cuda.memory_allocated() == before


def test_autograd_unaligned_output_gradient():
    q, k, v, dout = inputs(1, 4, 2, 150, 64, torch.bfloat16)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = mfa.window_attention(*leaves, 40, 2)
    odd = torch.empty(dout.numel() + 1, device="cuda", dtype=dout.dtype)[1:].view_as(dout)
    odd.copy_(dout)
    grads = torch.autograd.grad(out, leaves, odd)
    want = reference(*(x.detach() for x in leaves), 40, 2, dout)
    for name, x in zip(("dq", "dk", "dv"), grads):
        check(name, x, *want[name])


def test_empty():
    q = torch.empty((0, 4, 100, 64), device="cuda", dtype=torch.float16)
    k = torch.empty((0, 2, 100, 64), device="cuda", dtype=torch.float16)
    assert mfa.forward_window(q, k, k, 10).shape == q.shape
    q, k = q.new_empty((1, 4, 0, 64)), q.new_empty((1, 2, 0, 64))
    out, lse = mfa.forward_window_lse(q, k, k, 10, 1)
    assert lse.shape == (1, 4, 0)
    assert [x.shape for x in mfa.backward_window(q, k, k, out, lse, out, 10, 1)] == [
        q.shape, k.shape, k.shape]


def test_refusals():
    q, k, v, dout = inputs(1, 4, 2, 100, 64, torch.float16)
    for call, match in (
            (lambda: mfa.forward_window(q, k, v, 0), "window must be at least 1"),
            (lambda: mfa.forward_window(q, k, v, 5, -1), "sinks must not be negative"),
            (lambda: mfa.forward_window(q[:, :3].contiguous(), k, v, 5), "multiple"),
            (lambda: mfa.forward_window(q, k[:, :, :50].contiguous(), v, 5), "k must have shape"),
            (lambda: mfa.forward_window(q, k, v[:, :1].contiguous(), 5), "same shape as k"),
            (lambda: mfa.forward_window(q, k.bfloat16(), v, 5), "same dtype"),
            (lambda: mfa.forward_window(q.float(), k, v, 5), "float16 or bfloat16"),
            (lambda: mfa.forward_window(q.repeat_interleave(2, 3)[..., ::2], k, v, 5),
             "q must be contiguous in D"),
            (lambda: mfa.forward_window(q, k[:, :1].expand(1, 2, 100, 64), v, 5),
             "strides of q, k and v must be positive multiples of 8"),
            (lambda: mfa.forward_window(q, k, randn((1, 2, 100, 68), 9)[..., :64], 5),
             "strides of q, k and v must be positive multiples of 8"),
            (lambda: mfa.forward_window(q, k, randn((1, 2, 100, 72), 9)[..., 4:68], 5),
             "v must be 16-byte aligned"),
            (lambda: mfa.forward_window(q, k.cpu(), v, 5), "CUDA tensor")):
        with pytest.raises(RuntimeError, match=match):
            call()
    x = randn((1, 2, 100, 48), 3)
    with pytest.raises(RuntimeError, match="D=32, D=64 and D=128"):
        mfa.forward_window(x, x, x, 5)
    with pytest.raises(RuntimeError, match="D=32, D=64 and D=128"):
        mfa.backward_window(x, x, x, x, randn((1, 2, 100), 4, torch.float32), x, 5)
