"""Group norm with an activation, forward and backward, against the formulas in
64 bits with bounds derived from the roundings (blocks_reference.py)."""

import pytest
import torch

import blocks_reference as ref
import torchbvh_amd as tb

pytestmark = pytest.mark.gpu


def _run(x, groups, weight, bias, layout, up, **how):
    given = {"dx": x.detach().requires_grad_()}
    given |= {n: t.detach().requires_grad_() for n, t in (("dw", weight), ("db", bias)) if t is not None}
    out = tb.group_norm_act(given["dx"], groups, given.get("dw"), given.get("db"), layout, **how)
    return {"out": out} | dict(zip(given, torch.autograd.grad(out, list(given.values()), up)))


def _check(sizes, C, groups, kind, wide, activation, seed, shift=0.0, spread=1.0, eps=1e-5):
    g = torch.Generator("cuda").manual_seed(seed)
    x = (torch.randn((sum(sizes), C), generator=g, device="cuda") * spread + shift).to(kind)
    up = torch.randn((sum(sizes), C), generator=g, device="cuda").to(kind)
    weight, bias = (torch.randn(C, generator=g, device="cuda").to(torch.float32 if wide else kind) for _ in range(2))
    offsets = ref.layout_lists(sizes, 1)[0]
    layout = tb.block_layout(torch.tensor(offsets, dtype=torch.int64, device="cuda"), 64)
    how = dict(activation=activation, eps=eps)
    got = _run(x, groups, weight, bias, layout, up, **how)
    again = _run(x, groups, weight, bias, layout, up, **how)
    assert all(torch.equal(got[n], again[n]) for n in got)
    ref.within(got, ref.group_norm(x, offsets, groups, weight, bias, eps, activation, up))


@pytest.mark.parametrize("kind,wide", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("sizes,C,groups,activation", [
    ([1], 1, 1, "none"), ([1], 8, 4, "silu"), ([7], 5, 1, "gelu"), ([1000], 64, 8, "silu"),
    ([300, 1, 2000], 88, 8, "gelu"), ([129], 13, 13, "relu"), ([513, 64], 256, 32, "silu"),
    ([40] * 33, 24, 3, "gelu"), ([17], 2056, 4, "none"), ([20_001], 16, 16, "silu"), ([5000], 96, 1, "relu"),
])
def test_against_64_bits(kind, wide, sizes, C, groups, activation):
    _check(sizes, C, groups, kind, wide, activation, sum(sizes) + C)


@pytest.mark.parametrize("shift,spread", [(1000.0, 1.0), (-3e4, 0.5), (0.0, 1e-4), (0.0, 1e6)])
def test_large_means_and_odd_scales(shift, spread):
    _check([3000, 100], 32, 4, torch.float32, False, "silu", 1, shift, spread)


def test_constant_channels():
    x = torch.full((100, 8), 3.25, device="cuda")
    out = tb.group_norm_act(x, 2, None, None, activation="none")
    assert not out.any()
    out = tb.group_norm_act(x, 2, None, torch.full((8,), 2.0, device="cuda"), activation="none", eps=0.125)
    assert (out == 2.0).all()


def test_batched_is_every_cloud_alone():
    x = torch.randn((5, 333, 24), device="cuda")
    w, b, up = torch.randn(24, device="cuda"), torch.randn(24, device="cuda"), torch.randn_like(x)
    got = _run(x, 3, w, b, None, up)
    packed = _run(x.reshape(-1, 24), 3, w, b, tb.block_layout((5, 333), 64), up.reshape(-1, 24))
    assert all(torch.equal(got[n].reshape(packed[n].shape), packed[n]) for n in got)
    assert torch.equal(tb.group_norm_act(x[0], 3, w, b), tb.group_norm_act(x[:1], 3, w, b)[0])


def test_optional_parameters_and_wanted_gradients():
    x, up = torch.randn((50, 12), device="cuda"), torch.randn((50, 12), device="cuda")
    ref.within(_run(x, 4, None, None, None, up),
               {n: v for n, v in ref.group_norm(x, [0, 50], 4, None, None, 1e-5, "silu", up).items() if n in ("out", "dx")})
    w = torch.randn(12, device="cuda", requires_grad=True)
    out = tb.group_norm_act(x, 4, w)
    (dw,) = torch.autograd.grad(out, w, up)
    want = _run(x, 4, w, None, None, up)
    assert torch.equal(dw, want["dw"])
    assert not tb.group_norm_act(x, 4).requires_grad


def test_strides_empty_and_special_values():
    x = torch.randn((24, 60), device="cuda").t()
    want = tb.group_norm_act(x.contiguous(), 3)
    assert torch.equal(tb.group_norm_act(x, 3), want)
    odd = torch.empty(60 * 24 + 1, device="cuda")[1:].reshape(60, 24).copy_(x)  # not on 16 bytes
    torch.testing.assert_close(tb.group_norm_act(odd, 3), want, rtol=1e-6, atol=1e-6)
    empty = torch.empty((0, 8), device="cuda", requires_grad=True)
    out = tb.group_norm_act(empty, 2)
    assert out.shape == (0, 8)
    assert torch.autograd.grad(out.sum(), empty)[0].shape == (0, 8)
    big = torch.tensor([[-200.0, 200.0, 0.0, 1.0]], device="cuda").repeat(1, 2)
    for act in ("silu", "gelu"):
        y = tb.group_norm_act(big, 1, torch.full((8,), 500.0, device="cuda"), activation=act)
        assert torch.isfinite(y).all() and y.min() > -1.0
    x = torch.randn((2, 40, 8), device="cuda")
    x[0, 3, 1] = float("nan")  # its group of its cloud
    bad = torch.isnan(tb.group_norm_act(x, 2))
    assert bad[0, :, :4].all() and not bad[0, :, 4:].any() and not bad[1].any()


def test_other_streams_and_graphs():
    x, up = torch.randn((5000, 32), device="cuda"), torch.randn((5000, 32), device="cuda")
    w, b = torch.randn(32, device="cuda"), torch.randn(32, device="cuda")
    want = _run(x, 4, w, b, None, up)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(x, 4, w, b, None, up)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = _run(x, 4, w, b, None, up)
    for i in range(4):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        want = _run(x, 4, w, b, None, up)
        assert all(torch.equal(kept[n], want[n]) for n in want), i


def test_refusals():
    x = torch.randn((6, 8), device="cuda")
    layout = tb.block_layout((1, 6), 4)
    w = torch.ones(8, device="cuda")
    for args, how, match in (((x.half(), 2), {}, "x must be float32 or bfloat16"), ((x, 3), {}, "multiple of num_groups"),
                             ((x, 0), {}, "multiple of num_groups"), ((x, 2), {"activation": "tanh"}, "activation must"),
                             ((x, 2), {"eps": -1.0}, "eps must"), ((x, 2, w[:4]), {}, "weight must have shape"),
                             ((x, 2, w.bfloat16()), {}, "weight must be float32 or of x's type"),
                             ((x.bfloat16(), 2, w, w.bfloat16()), {}, "the same type"),
                             ((x, 2, w.cpu()), {}, "weight must be on the same device"),
                             ((x, 2, w, w, layout[:3]), {}, "layout must be a BlockLayout")):
        with pytest.raises(ValueError, match=match):
            tb.group_norm_act(*args, **how)
