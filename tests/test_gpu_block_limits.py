"""Where blocks, scores and caches end: rows that a last block lacks beside scores
far below and above zero, tensors of more than 2^31 elements and 2^32 bytes, a
choice replayed from a graph, the roundings of gradients in bfloat16."""

import pytest
import torch

import blocks_reference as ref
import torchbvh_amd as tb

pytestmark = pytest.mark.gpu


def _layout(sizes, block):
    return tb.block_layout(torch.tensor(ref.layout_lists(sizes, 1)[0], dtype=torch.int64, device="cuda"), block)


def _normal(seed, kind, *shape):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(kind)


def _grads(q, k, v, up, selected, q_layout, k_layout, scale=None, bias=None):
    given = [t.detach().requires_grad_() for t in (q, k, v)]
    if bias is not None:
        bias = bias._replace(table=bias.table.detach().requires_grad_())
        given.append(bias.table)
    out = tb.block_attention(given[0], given[1], given[2], selected, q_layout, k_layout, scale=scale, bias=bias)
    return {"out": out} | dict(zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, given, up)))


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("block", [64, 32, 24, 1])
@pytest.mark.parametrize("level", [-3.0, 3.0])
def test_rows_a_block_lacks_beside_scores_far_from_zero(kind, block, level):
    """Every score is about 16 * 3 * level * 3: -432 or 432."""
    q_layout, k_layout = _layout([150], block), _layout([90], 32)
    q, k = 3.0 + 0.1 * _normal(1, kind, 150, 2, 16), level + 0.1 * _normal(2, kind, 90, 1, 16)
    v, up = _normal(3, kind, 90, 1, 16), _normal(4, kind, 150, 2, 16)
    groups = q_layout.starts.numel() - 1
    selected = torch.arange(3, dtype=torch.int32, device="cuda").repeat(groups, 1)
    got = _grads(q, k, v, up, selected, q_layout, k_layout, 3.0)
    times = ref.multiplicity(selected, q_layout.starts.tolist(), k_layout.starts.tolist())
    ref.within(got, ref.attention(q, k, v, times, 3.0, None, up))


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("level", [-300.0, 300.0])
def test_rows_a_block_lacks_beside_biases_far_from_zero(kind, level):
    layout = _layout([75], 32)
    q, k, v, up = (_normal(i, kind, 75, 2, 16) for i in range(4))
    table = level + _normal(5, kind, 2, 9, 2)
    cells = torch.randint(-6, 7, (75, 2), dtype=torch.int32, device="cuda")
    bias = (table, tb.relative_buckets(5, 6), cells, cells)
    selected = torch.tensor([[0, 1], [1, 2], [2, 0]], dtype=torch.int32, device="cuda")
    got = _grads(q, k, v, up, selected, layout, layout, None, tb.RelativeBias(*bias))
    times = ref.multiplicity(selected, layout.starts.tolist(), layout.starts.tolist())
    ref.within(got, ref.attention(q, k, v, times, 0.25, bias, up))


@pytest.mark.parametrize("kind,heads", [(torch.float32, 1), (torch.bfloat16, 2)])
def test_caches_past_32_bits(kind, heads):
    """Blocks on both sides of 2^31 elements and 2^32 bytes of one cache give what
    they give in a small one."""
    D, block = 64, 64
    rows = 2**31 // (heads * D) + 5 * block + 7
    k, v = (torch.zeros((rows, heads, D), dtype=kind, device="cuda") for _ in range(2))
    layout = tb.block_layout((1, rows), block, device="cuda")
    last = layout.starts.numel() - 2
    blocks = [0, 1, 2**31 // (heads * D * block) - 1, last - 4, last - 1, last]
    if kind == torch.float32:
        blocks[1] = 2**30 // (heads * D * block)
    small = _layout([64 * 5 + 7], block)
    for i, b in enumerate(blocks):
        n = 64 if i < 5 else 7
        k[b * block : b * block + n] = _normal(i, kind, n, heads, D)
        v[b * block : b * block + n] = _normal(10 + i, kind, n, heads, D)
    where = torch.cat([torch.arange(b * block, min((b + 1) * block, rows)) for b in blocks]).cuda()
    q, up = (_normal(20 + i, kind, 40, heads, D) for i in range(2))
    asked = _layout([40], 20)
    far = torch.tensor([blocks, blocks[::-1]], dtype=torch.int32, device="cuda")
    near = torch.tensor([range(6), range(5, -1, -1)], dtype=torch.int32, device="cuda")
    got = _grads(q, k, v, up, far, asked, layout)
    times = ref.multiplicity(near, asked.starts.tolist(), small.starts.tolist())
    want = ref.attention(q, k[where], v[where], times, D**-0.5, None, up)
    ref.within({n: t[where] if n in ("dk", "dv") else t for n, t in got.items()}, want)
    for name in ("dk", "dv"):
        got[name][where] = 0
        assert not got[name].any()


def test_queries_past_32_bits():
    D, block = 64, 64
    rows = 2**31 // D + 3 * block + 9
    q = torch.zeros((rows, 1, D), dtype=torch.bfloat16, device="cuda")
    up = torch.zeros_like(q)
    q[-73:], up[-73:] = _normal(1, torch.bfloat16, 73, 1, D), _normal(2, torch.bfloat16, 73, 1, D)
    k, v = (_normal(i, torch.bfloat16, 200, 1, D) for i in (3, 4))
    layout, keys = tb.block_layout((1, rows), block, device="cuda"), _layout([200], 64)
    groups = layout.starts.numel() - 1
    selected = torch.full((groups, 3), -1, dtype=torch.int32, device="cuda")
    selected[0] = selected[-100:] = torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda")
    got = _grads(q, k, v, up, selected, layout, keys)
    first = layout.starts[-3].item()  # the last two blocks, 64 and 9 rows; the others add nothing to dk and dv
    times = ref.multiplicity(selected[-2:], [0, block, rows - first], keys.starts.tolist())
    ref.within({n: t[first:] if n in ("out", "dq") else t for n, t in got.items()},
               ref.attention(q[first:], k, v, times, D**-0.5, None, up[first:]))
    assert not got["out"][64:first - 98 * block].any()


def test_norm_past_32_bits():
    C = 64
    rows = 2**31 // C + 1000
    x = _normal(1, torch.bfloat16, rows, C)
    layout = tb.block_layout(torch.tensor([0, rows - 900, rows], device="cuda"), 64)
    up = torch.zeros_like(x)
    up[-900:] = _normal(2, torch.bfloat16, 900, C)
    given = x.requires_grad_()
    out = tb.group_norm_act(given, 8, layout=layout)
    (dx,) = torch.autograd.grad(out, given, up)
    ref.within({"out": out[-900:], "dx": dx[-900:]},
               {n: t for n, t in ref.group_norm(x[-900:].detach(), [0, 900], 8, None, None, 1e-5, "silu", up[-900:]).items()
                if n in ("out", "dx")})
    with torch.no_grad():
        # One group's statistics of the large cloud, in 64 bits, applied to its last rows.
        part = x[: rows - 900, :8].double()
        mean, var = part.mean(), part.var(unbiased=False)
        z = (part[-500:] - mean) * torch.rsqrt(var + 1e-5)
        want = z * torch.sigmoid(z)
        # One rounding to bf16; z's few roundings in 32 bits.
        assert ((out[rows - 1400 : rows - 900, :8].double() - want).abs() <= 2.0**-8 * want.abs() + 1e-5).all()


def test_choice_in_a_graph():
    points = torch.rand((3000, 3), device="cuda")
    bvh = tb.build_bvh(points)
    layout, boxes = tb.block_layout(bvh, 64), tb.block_boxes(bvh, 64)
    for n in (40, 20_000):  # a team of waves for each query, and one wave
        asked = torch.rand((n, 3), device="cuda")
        queries = tb.block_layout((1, n), 1, device="cuda")
        tb.select_blocks(asked, boxes, 9, queries, layout)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = tb.select_blocks(asked, boxes, 9, queries, layout)
        for i in range(4):
            asked.copy_(torch.rand_like(asked))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(kept, tb.select_blocks(asked, boxes, 9, queries, layout)), (n, i)


@pytest.mark.parametrize("axes", [0, 3])
def test_roundings_in_bfloat16(axes):
    """Against 64 bits, over all values: one rounding to bfloat16 is off by 2^-8 / sqrt 3
    in the mean square at most (errors even in half an ulp, at mantissa 1).  A
    gradient is rounded once itself and takes over the one rounding of its terms'
    weights or ds: sqrt 2 times that, with half as much again for terms that cancel.
    The output and a table's gradient take over none."""
    kind, layout = torch.bfloat16, _layout([700], 64)
    q, k, v, up = (_normal(i, kind, 700, 2, 32) for i in range(4))
    # Outputs much larger than their gradients' variation: delta's error would show.
    v = (v.float() + 4.0).to(kind)
    bias = None
    if axes:
        cells = torch.randint(-9, 10, (700, axes), dtype=torch.int32, device="cuda")
        bias = (_normal(9, kind, axes, 9, 2), tb.relative_buckets(5, 6), cells, cells)
    groups = layout.starts.numel() - 1
    selected = torch.stack([torch.randperm(groups, generator=torch.Generator().manual_seed(i))[:6]
                            for i in range(groups)]).int().cuda()
    got = _grads(q, k, v, up, selected, layout, layout, None, None if bias is None else tb.RelativeBias(*bias))
    times = ref.multiplicity(selected, layout.starts.tolist(), layout.starts.tolist())
    want = ref.attention(q, k, v, times, 32**-0.5, bias, up)
    one = 2.0**-8 / 3**0.5
    for name, (value, _) in want.items():
        off = ((got[name].detach().cpu().double() - value).norm() / value.norm()).item()
        assert off <= (one if name in ("out", "dtable") else 1.5 * 2**0.5 * one), (name, off)


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 1), (18, 1)])
@pytest.mark.parametrize("scale", [None, 0.0, -2.0, 1e-20])
@pytest.mark.parametrize("spread", [3, 9, 400])
def test_biases_by_products_and_by_lookups(heads, kv_heads, scale, spread):
    """bf16: cells within 16 of each other and further apart, scales that nothing is
    divided by, heads that share many tables."""
    kind, layout = torch.bfloat16, _layout([130, 50], 64)
    q, up = (_normal(i, kind, 180, heads, 16) for i in range(2))
    k, v = (_normal(i, kind, 180, kv_heads, 16) for i in (2, 3))
    cells = [torch.randint(-spread, spread + 1, (180, 3), dtype=torch.int32, device="cuda") for _ in range(2)]
    cells[0][64:128] //= 4
    bias = (_normal(5, kind, 3, 9, heads), tb.relative_buckets(5, 12), *cells)
    selected = torch.tensor([[0, 1, 2], [2, 0, -1], [1, 1, 0], [3, -1, -1]], dtype=torch.int32, device="cuda")
    got = _grads(q, k, v, up, selected, layout, layout, scale, tb.RelativeBias(*bias))
    times = ref.multiplicity(selected, layout.starts.tolist(), layout.starts.tolist())
    ref.within(got, ref.attention(q, k, v, times, 0.25 if scale is None else scale, bias, up))


@pytest.mark.parametrize("value", [float("-inf"), -1e30, 1e25])
def test_tables_that_are_not_small(value):
    """A bucket that nothing may be chosen from, and one that outweighs everything."""
    kind, layout = torch.bfloat16, _layout([128], 64)
    q, k, v, up = (_normal(i, kind, 128, 2, 32) for i in range(4))
    cells = torch.randint(-4, 5, (128, 2), dtype=torch.int32, device="cuda")
    table = _normal(5, kind, 2, 9, 2)
    table[0, 6] = value
    bias = (table, tb.relative_buckets(5, 6), cells, cells)
    selected = torch.tensor([[0, 1], [1, 0]], dtype=torch.int32, device="cuda")
    got = _grads(q, k, v, up, selected, layout, layout, None, tb.RelativeBias(*bias))
    big = torch.tensor(value, dtype=kind).double().item()
    s = torch.einsum("ihd,jhd->hij", q.cpu().double(), k.cpu().double()) * 32**-0.5
    which = bias[1].cpu()[(cells[:, None] - cells[None]).cpu().clamp(-6, 6) + 6].long()
    for axis in range(2):
        s = s + table.cpu().double()[axis][which[..., axis]].permute(2, 0, 1)
    p = torch.softmax(s, -1)
    want = torch.einsum("hij,jhd->ihd", p, v.cpu().double())
    assert abs(big) > 2.0**64
    # Where the table outweighs, scores differ by less than its own digits: any of them may win.
    if value < 0:
        assert ((got["out"].cpu().double() - want).abs() <= 2.0**-7 * 4).all()
        assert all(torch.isfinite(t).all() for t in got.values())
    else:
        assert torch.isfinite(got["out"]).all()


@pytest.mark.parametrize("axes,reach,D", [(1, 2047, 128), (3, 682, 32), (3, 682, 128)])
def test_tables_as_large_as_they_may_be(axes, reach, D):
    kind, layout = torch.bfloat16, _layout([150], 64)
    q, k, v, up = (_normal(i, kind, 150, 2, D) for i in range(4))
    cells = torch.randint(-reach, reach, (150, axes), dtype=torch.int32, device="cuda")
    cells[:70] = cells[:70] % 9
    sizes = {1: 128, 3: 43}[axes]
    bias = (_normal(5, kind, axes, 2 * sizes - 1, 2), tb.relative_buckets(sizes, reach), cells, cells)
    selected = torch.tensor([[0, 1], [2, 0], [1, 2]], dtype=torch.int32, device="cuda")
    got = _grads(q, k, v, up, selected, layout, layout, None, tb.RelativeBias(*bias))
    times = ref.multiplicity(selected, layout.starts.tolist(), layout.starts.tolist())
    ref.within(got, ref.attention(q, k, v, times, D**-0.5, bias, up))
