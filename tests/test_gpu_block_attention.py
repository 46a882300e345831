"""Attention over chosen blocks, forward and backward, against the formulas in
64 bits with bounds derived from the roundings (blocks_reference.py): types, head
layouts, channels, block sizes, choices that leave rows empty, strides, values
that must not leak, streams, graphs."""

import pytest
import torch

import blocks_reference as ref
import torchbvh_amd as tb

pytestmark = pytest.mark.gpu


def _layout(sizes, block):
    return tb.block_layout(torch.tensor(ref.layout_lists(sizes, 1)[0], dtype=torch.int64, device="cuda"), block)


def _inputs(q_sizes, k_sizes, heads, kv_heads, D, kind, axes, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(kind)

    q, up = normal(sum(q_sizes), heads, D), normal(sum(q_sizes), heads, D)
    k, v = normal(sum(k_sizes), kv_heads, D), normal(sum(k_sizes), kv_heads, D)
    bias = None
    if axes:
        reach = 6
        buckets = tb.relative_buckets(5, reach)
        cells = [torch.randint(-9, 10, (n, axes), generator=g, device="cuda", dtype=torch.int32)
                 for n in (sum(q_sizes), sum(k_sizes))]
        bias = (normal(axes, 9, heads), buckets, *cells)
    return q, k, v, up, bias


def _run(q, k, v, up, bias, selected, q_layout, k_layout, scale=None):
    given = [t.detach().requires_grad_() for t in (q, k, v)]
    table = None if bias is None else bias[0].detach().requires_grad_()
    out = tb.block_attention(*given, selected, q_layout, k_layout, scale=scale,
                             bias=None if bias is None else tb.RelativeBias(table, *bias[1:]))
    wanted = given + ([table] if bias is not None else [])
    grads = torch.autograd.grad(out, wanted, up)
    return {"out": out} | dict(zip(("dq", "dk", "dv", "dtable"), grads))


def _check(q, k, v, up, bias, selected, q_layout, k_layout, scale=None):
    got = _run(q, k, v, up, bias, selected, q_layout, k_layout, scale)
    again = _run(q, k, v, up, bias, selected, q_layout, k_layout, scale)
    assert all(torch.equal(got[n], again[n]) for n in got)  # one order of sums
    times = ref.multiplicity(selected, q_layout.starts.tolist(), k_layout.starts.tolist())
    ref.within(got, ref.attention(q, k, v, times, q.size(2)**-0.5 if scale is None else scale, bias, up))
    return got


def _choice(q_layout, k_layout, count, seed):
    """Random blocks of the group's cloud, some of them none."""
    g = torch.Generator().manual_seed(seed)
    groups = q_layout.starts.numel() - 1
    qc, kc = q_layout.clouds.tolist(), k_layout.clouds.tolist()
    out = torch.full((groups, count), -1, dtype=torch.int32)
    for c in range(len(qc) - 1):
        n = kc[c + 1] - kc[c]
        for i in range(qc[c], qc[c + 1]):
            some = torch.randperm(n, generator=g)[:count] + kc[c]
            out[i, : len(some)] = some.int()
    if count > 2:
        out[:, 1] = -1
    return out.cuda()


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes,q_block,k_block,count,heads,kv_heads,D,axes", [
    ([1], 1, 1, 1, 1, 1, 8, 0),                 # one token
    ([64], 64, 64, 1, 1, 1, 32, 0),
    ([200], 64, 64, 4, 2, 2, 16, 3),            # a last block of 8 rows
    ([130, 1, 77], 32, 64, 3, 4, 2, 24, 2),     # clouds of one row and less than a block
    ([333], 64, 32, 5, 6, 1, 40, 0),            # six heads share one
    ([257], 16, 128, 3, 3, 3, 64, 1),
    ([150], 128, 64, 3, 2, 1, 128, 3),
    ([97], 17, 19, 4, 5, 5, 48, 2),             # odd blocks
    ([300], 1, 64, 4, 8, 2, 64, 2),             # single rows
])
def test_against_64_bits(kind, sizes, q_block, k_block, count, heads, kv_heads, D, axes):
    q_layout, k_layout = _layout(sizes, q_block), _layout(sizes, k_block)
    tensors = _inputs(sizes, sizes, heads, kv_heads, D, kind, axes, sum(sizes) + D)
    _check(*tensors, _choice(q_layout, k_layout, count, D), q_layout, k_layout)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,q_block,heads,D", [(1, 1, 2, 64), (3, 8, 2, 128), (2, 64, 1, 64), (600, 1, 8, 32)])
def test_few_rows_over_many_blocks(kind, groups, q_block, heads, D):
    """Few tiles split their blocks between waves."""
    q_sizes, k_sizes = [groups * q_block], [1500]
    q_layout, k_layout = _layout(q_sizes, q_block), _layout(k_sizes, 64)
    tensors = _inputs(q_sizes, k_sizes, heads, heads, D, kind, 2, groups)
    _check(*tensors, _choice(q_layout, k_layout, 21, 3), q_layout, k_layout)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_choices_that_are_empty_repeated_or_no_block(kind):
    q_layout, k_layout = _layout([160], 16), _layout([200], 64)
    tensors = _inputs([160], [200], 2, 2, 32, kind, 2, 9)
    selected = torch.tensor([[-1, -1, -1], [0, 0, 1], [3, -1, 3], [4, 1000, -7], [2, 2, 2], [0, 1, 2], [3, 3, 3],
                             [-1, 2, -1], [2**31 - 1, -(2**31), 1], [1, 0, 3]], dtype=torch.int32, device="cuda")
    got = _check(*tensors, selected, q_layout, k_layout)
    for group in (0, 3):
        assert not got["out"][16 * group : 16 * group + 16].any()
        assert not got["dq"][16 * group : 16 * group + 16].any()


def test_no_choice_no_rows_no_keys():
    layout = _layout([40], 16)
    q, k, v, up, bias = _inputs([40], [40], 2, 2, 16, torch.float32, 1, 1)
    none = torch.empty((3, 0), dtype=torch.int32, device="cuda")
    got = _run(q, k, v, up, bias, none, layout, layout)
    assert all(not t.any() for t in got.values())
    empty = tb.block_layout((1, 0), 16)
    got = _run(q[:0], k, v, up[:0], None, none[:0], empty, layout)
    assert got["out"].shape == (0, 2, 16) and not got["dk"].any()
    got = _run(q, k[:0], v[:0], up, None, torch.zeros((3, 2), dtype=torch.int32, device="cuda"), layout, empty)
    assert not got["out"].any() and not got["dq"].any()


def test_what_is_not_chosen_does_not_leak():
    layout = _layout([256], 64)
    q, k, v, up, bias = _inputs([256], [256], 2, 2, 32, torch.bfloat16, 3, 4)
    selected = torch.tensor([[0, 2], [2, 0], [0, -1], [2, -1]], dtype=torch.int32, device="cuda")
    want = _run(q, k, v, up, bias, selected, layout, layout)
    k[64:128], v[64:128], k[192:], v[192:] = float("nan"), float("inf"), float("-inf"), float("nan")
    got = _run(q, k, v, up, bias, selected, layout, layout)
    assert all(torch.equal(got[n], want[n]) for n in got)
    # The rows after a short last block are another tensor's.
    both = torch.full((300, 2, 32), float("nan"), dtype=torch.bfloat16, device="cuda")
    both[:100] = k[128:192].repeat(2, 1, 1)[:100]
    short = tb.block_layout((1, 100), 64)
    out = tb.block_attention(q[:100], both[:100], both[:100], torch.tensor([[0, 1], [1, 0]], dtype=torch.int32, device="cuda"),
                             short, short)
    assert torch.isfinite(out).all()


def test_infinite_and_undefined_scores():
    layout = _layout([32], 16)
    q, k, v, up, _ = _inputs([32], [32], 1, 1, 8, torch.float32, 0, 5)
    q = q.abs()
    k[3] = float("-inf")   # weight zero
    selected = torch.tensor([[0, -1], [0, 1]], dtype=torch.int32, device="cuda")
    out = tb.block_attention(q, k, v, selected, layout, layout)
    rest = k.clone()
    rest[3] = 0
    s = (q[:, 0] @ rest[:, 0].T) * 8**-0.5
    s[:, 3] = float("-inf")
    s[:16, 16:] = float("-inf")
    want = torch.softmax(s.double(), 1) @ v[:, 0].double()
    torch.testing.assert_close(out[:, 0].double(), want, rtol=1e-5, atol=1e-5)
    k[:16] = float("-inf")  # no weight at all: zero, as with nothing chosen
    assert not tb.block_attention(q, k, v, selected, layout, layout)[:16].any()
    k[20] = float("nan")
    out = tb.block_attention(q, k, v, selected, layout, layout)
    assert not out[:16].any() and torch.isnan(out[16:]).all()


def test_extreme_scores():
    """Scores of thousands, cells at the ends of int32, values of one sign."""
    layout = _layout([128], 32)
    q, k, v, up, bias = _inputs([128], [128], 2, 1, 16, torch.float32, 2, 6)
    bias[2][::3], bias[3][1::3] = 2**31 - 1, -(2**31)
    _check(q * 30, k * 30, v, up, bias, _choice(layout, layout, 4, 1), layout, layout, scale=-0.7)
    _check(q, k, v.abs(), up, bias, _choice(layout, layout, 4, 1), layout, layout, scale=0.0)


@pytest.mark.parametrize("D", [1, 5, 20, 100])
def test_channels_that_are_padded(D):
    layout = _layout([70], 64)
    _check(*_inputs([70], [70], 2, 2, D, torch.float32, 1, D), _choice(layout, layout, 2, 1), layout, layout)


def test_strided_inputs_and_gradients():
    layout = _layout([140], 64)
    q, k, v, up, bias = _inputs([140], [140], 4, 4, 16, torch.bfloat16, 2, 7)
    selected = _choice(layout, layout, 2, 1)
    want = _run(q, k, v, up, bias, selected, layout, layout)
    packed = torch.stack([q, k, v], 1)                     # one projection's output
    got = _run(*packed.unbind(1), up, bias, selected, layout, layout)
    assert all(torch.equal(got[n], want[n]) for n in got)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    odd = [torch.empty((140, 4, 17), dtype=t.dtype, device="cuda")[..., 1:].copy_(t) for t in (q, k, v)]
    backwards = up.transpose(0, 2).contiguous().transpose(0, 2)
    wide = torch.stack([selected, selected], 2)[..., 0]
    for three in (turned, odd):
        got = _run(*three, backwards, bias, wide, layout, layout)
        assert all(torch.equal(got[n], want[n]) for n in got)


def test_heads_that_share_by_expansion():
    """Keys expanded over heads give the sum of the heads' gradients."""
    layout = _layout([100], 64)
    q, k, v, up, _ = _inputs([100], [100], 4, 1, 32, torch.float32, 0, 8)
    selected = _choice(layout, layout, 2, 2)
    want = _run(q, k, v, up, None, selected, layout, layout)
    k1, v1 = (t.detach().requires_grad_() for t in (k, v))
    out = tb.block_attention(q, k1.expand(-1, 4, -1), v1.expand(-1, 4, -1), selected, layout, layout)
    dk, dv = torch.autograd.grad(out, (k1, v1), up)
    # The same products, the four heads' sums added in another order.
    for got, name in ((out, "out"), (dk, "dk"), (dv, "dv")):
        torch.testing.assert_close(got, want[name], rtol=1e-5, atol=1e-5)


def test_gradients_against_differences():
    layout = _layout([96], 32)
    q, k, v, up, bias = _inputs([96], [96], 2, 2, 16, torch.float32, 2, 10)
    selected = _choice(layout, layout, 2, 3)
    got = _run(q, k, v, up, bias, selected, layout, layout)
    args = {"q": q, "k": k, "v": v, "table": bias[0]}

    def loss(a):
        out = tb.block_attention(a["q"], a["k"], a["v"], selected, layout, layout,
                                 bias=tb.RelativeBias(a["table"], *bias[1:]))
        return (out.double() * up.double()).sum().item()

    h = 2.0**-7
    for name, x in args.items():
        d = torch.sign(got["d" + name])  # a direction in which nothing cancels
        slope = (loss(args | {name: x + h * d}) - loss(args | {name: x - h * d})) / (2 * h)
        want = got["d" + name].double().abs().sum().item()
        # Differences are off by h^2 / 6 of the third derivative (unit steps in 16
        # channels and 64 keys: below 2^6 of the first) and by 2^-24 / h.
        assert abs(slope - want) < 2.0**6 * h * h * want


def test_other_streams_and_graphs():
    layout = _layout([500], 64)
    q, k, v, up, bias = _inputs([500], [500], 2, 2, 32, torch.bfloat16, 2, 11)
    selected = _choice(layout, layout, 3, 3)
    want = _run(q, k, v, up, bias, selected, layout, layout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, up, bias, selected, layout, layout)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = _run(q, k, v, up, bias, selected, layout, layout)
    for i in range(4):
        q.copy_(torch.randn_like(q)), up.copy_(torch.randn_like(up))
        graph.replay()
        torch.cuda.synchronize()
        want = _run(q, k, v, up, bias, selected, layout, layout)
        assert all(torch.equal(kept[n], want[n]) for n in want), i


def test_only_the_wanted_gradients():
    layout = _layout([64], 64)
    q, k, v, up, _ = _inputs([64], [64], 1, 1, 8, torch.float32, 0, 12)
    selected = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    assert not tb.block_attention(q, k, v, selected, layout, layout).requires_grad
    q1 = q.clone().requires_grad_()
    out = tb.block_attention(q1, k, v, selected, layout, layout)
    (dq,) = torch.autograd.grad(out, q1, up, retain_graph=True)
    assert torch.equal(dq, _run(q, k, v, up, None, selected, layout, layout)["dq"])
    (dq,) = torch.autograd.grad(out, q1, up, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), q1)  # not differentiable twice


def test_refusals():
    layout = _layout([64], 64)
    q, k, v, up, bias = _inputs([64], [64], 4, 2, 16, torch.float32, 2, 13)
    s = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    bias = tb.RelativeBias(*bias)
    cases = (
        (dict(q=q.half(), k=k.half(), v=v.half()), "q must be float32 or bfloat16"),
        (dict(k=k.bfloat16()), "k and v must have q's type"),
        (dict(k=k[:40]), "k and v must have the same shape"),
        (dict(q=q[..., :8]), "k and v must have q's channels"),
        (dict(q=torch.zeros((64, 2, 136), device="cuda")), "D must be 1 to 128"),
        (dict(q=q[:, :3]), "q's heads must be a multiple"),
        (dict(selected=s.long()), "selected must be int32"),
        (dict(selected=s.repeat(2, 1)), "selected must have shape"),
        (dict(selected=s.cpu()), "selected must be on the same device"),
        (dict(query_layout=tuple(layout)), "query_layout must be a BlockLayout"),
        (dict(bias=bias._replace(table=bias.table.bfloat16())), "bias.table must have q's type"),
        (dict(bias=bias._replace(table=bias.table[..., :3])), "bias.table must have shape"),
        (dict(bias=bias._replace(table=bias.table.repeat(1, 20, 1))), "at most 256"),
        (dict(bias=bias._replace(buckets=bias.buckets[1:])), "odd number of entries"),
        (dict(bias=bias._replace(buckets=bias.buckets.repeat(99))), "at most 4096"),
        (dict(bias=bias._replace(key_cells=bias.key_cells[1:])), "bias.key_cells must be int32"),
        (dict(bias=bias._replace(query_cells=bias.query_cells.long())), "bias.query_cells must be int32"),
    )
    whole = dict(q=q, k=k, v=v, selected=s, query_layout=layout, key_layout=layout, bias=None)
    for changed, match in cases:
        with pytest.raises(ValueError, match=match):
            tb.block_attention(**(whole | changed))
