"""Boxes and choice of key blocks: against brute force in the same fp32 order,
over cloud sizes, block sizes, dimensions, ties and values that are not finite."""

import pytest
import torch

import blocks_reference as ref
import torchbvh_amd as tb

pytestmark = pytest.mark.gpu


def _points(sizes, dim, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.rand((sum(sizes), dim), generator=g, device="cuda")


def _offsets(sizes):
    return torch.tensor(ref.layout_lists(sizes, 1)[0], dtype=torch.int64, device="cuda")


def _choose(queries, boxes, count, query_layout, key_layout):
    """Brute force, one block of queries after the other, on the CPU."""
    queries, boxes = queries.cpu(), boxes.cpu()
    dim = queries.shape[1]
    q, k = ([t.tolist() for t in layout[:3]] for layout in (query_layout, key_layout))
    out = torch.full((len(q[1]) - 1, count), -1, dtype=torch.int32)
    for cloud in range(len(q[2]) - 1):
        first, last = k[2][cloud], k[2][cloud + 1]
        lo, hi = boxes[first:last, :dim], boxes[first:last, dim:]
        for g in range(q[2][cloud], q[2][cloud + 1]):
            rows = queries[q[1][g] : q[1][g + 1]]
            nan = torch.isnan(rows)
            least = torch.where(nan, torch.inf, rows).amin(0)
            most = torch.where(nan, -torch.inf, rows).amax(0)
            c = 0.5 * least + 0.5 * most
            d = torch.maximum(torch.maximum(lo - c, c - hi), torch.zeros(()))
            s = d[:, 0] * d[:, 0] + d[:, 1] * d[:, 1]
            if dim == 3:
                s = s + d[:, 2] * d[:, 2]
            s = torch.where(torch.isfinite(s), s, torch.inf)
            order = torch.sort(s, stable=True).indices[:count]
            order = order[torch.isfinite(s[order])]
            out[g, : len(order)] = (order + first).int()
    return out


@pytest.mark.parametrize("block", [1, 16, 64, 128])
@pytest.mark.parametrize("sizes", [[1], [63], [64], [65], [1000], [4097], [1, 700, 64, 2, 333]])
def test_boxes_are_the_tree_nodes(sizes, block):
    dim = 2 + len(sizes) % 2
    points = _points(sizes, dim, sum(sizes))
    bvh = tb.build_bvh(points, batch_offsets=_offsets(sizes)) if len(sizes) > 1 else tb.build_bvh(points)
    layout, boxes = tb.block_layout(bvh, block), tb.block_boxes(bvh, block)
    offsets, starts, clouds = ref.layout_lists(sizes, block)
    assert (layout.offsets.tolist(), layout.starts.tolist(), layout.clouds.tolist()) == (offsets, starts, clouds)
    handles = bvh._handles if len(sizes) > 1 else [bvh]
    rows = torch.cat([points[o:][h["sorted_indices"]] for o, h in zip(offsets, handles)])
    want = torch.stack([torch.cat([rows[a:b].amin(0), rows[a:b].amax(0)]) for a, b in zip(starts, starts[1:])])
    assert torch.equal(boxes, want)


def test_batched_boxes():
    points = torch.rand((3, 201, 3), device="cuda")
    bvh = tb.build_bvh(points)
    boxes = tb.block_boxes(bvh, 32)
    assert torch.equal(boxes, torch.cat([tb.block_boxes(tb.build_bvh(p), 32) for p in points]))
    assert tb.block_layout(bvh, 32).starts.numel() == boxes.size(0) + 1


@pytest.mark.parametrize("dim", [2, 3])
@pytest.mark.parametrize("sizes,q_block,count", [([1], 1, 1), ([64], 64, 4), ([1000], 64, 64), ([3000], 1, 16),
                                                 ([20_000], 16, 32), ([1, 129, 5000, 64], 64, 8),
                                                 ([300] * 70, 128, 13), ([70_001], 64, 16)])
def test_choice_matches_brute_force(dim, sizes, q_block, count):
    points = _points(sizes, dim, count)
    bvh = tb.build_bvh(points, batch_offsets=_offsets(sizes))
    keys, boxes = tb.block_layout(bvh, 16), tb.block_boxes(bvh, 16)
    if q_block == 1:
        asked = [min(n, 40) for n in sizes]
        queries = _points(asked, dim, 5) * 1.4 - 0.2
    else:
        asked, queries = sizes, points
    layout = tb.block_layout(_offsets(asked), q_block)
    got = tb.select_blocks(queries, boxes, count, layout, keys)
    assert got.dtype == torch.int32
    assert torch.equal(got.cpu(), _choose(queries, boxes, count, layout, keys))


def test_ties_go_to_the_lower_block():
    side = torch.arange(4, device="cuda", dtype=torch.float32)
    grid = torch.cartesian_prod(side, side, side)
    points = grid.repeat_interleave(16, 0).repeat(3, 1)  # every box a point, three of each
    boxes = torch.cat([points[::16], points[::16]], 1)
    keys = tb.block_layout((1, points.size(0)), 16)
    queries = torch.cat([grid, grid + 0.5])
    layout = tb.block_layout((1, queries.size(0)), 1)
    got = tb.select_blocks(queries, boxes, 50, layout, keys)
    assert torch.equal(got.cpu(), _choose(queries, boxes, 50, layout, keys))


def test_values_that_are_not_finite():
    boxes = torch.rand((200, 3), device="cuda")
    boxes = torch.cat([boxes, boxes + 0.1], 1)
    boxes[3, 1], boxes[5, 4], boxes[7, 0], boxes[9] = float("nan"), float("nan"), float("-inf"), float("inf")
    boxes[11, 3:] = float("inf")
    keys = tb.block_layout((1, 400), 2)
    queries = torch.rand((96, 3), device="cuda")
    queries[5] = float("nan")
    queries[16:32] = float("nan")
    queries[33, 1] = float("inf")
    queries[50, 2] = 3e38
    for block in (1, 16):
        layout = tb.block_layout((1, 96), block)
        got = tb.select_blocks(queries, boxes, 8, layout, keys)
        assert torch.equal(got.cpu(), _choose(queries, boxes, 8, layout, keys))


def test_empty_clouds_and_no_queries():
    keys = tb.block_layout((2, 30), 8)
    boxes = torch.rand((keys.starts.numel() - 1, 4), device="cuda")
    none = tb.block_layout((2, 0), 8)
    assert tb.select_blocks(torch.rand((0, 2), device="cuda"), boxes, 3, none, keys).shape == (0, 3)
    queries = tb.block_layout((2, 9), 8)
    got = tb.select_blocks(torch.rand((18, 2), device="cuda"), boxes[:0], 3, queries, none)
    assert got.shape == (4, 3) and (got == -1).all()


def test_refusals():
    q, boxes = torch.rand((6, 3), device="cuda"), torch.rand((2, 6), device="cuda")
    layout, other = tb.block_layout((1, 6), 4), tb.block_layout((2, 3), 4)
    for args, match in (((q.double(), boxes, 1, layout, layout), "queries must be float32"),
                        ((q, boxes.cpu(), 1, layout, layout), "boxes must be a CUDA tensor"),
                        ((q, boxes[:, :4], 1, layout, layout), "boxes must have shape"),
                        ((q, boxes[:1], 1, layout, layout), "a row for every block"),
                        ((q, boxes, 0, layout, layout), "count must be 1 to 64"),
                        ((q, boxes, 65, layout, layout), "count must be 1 to 64"),
                        ((q, boxes, 1, layout, other), "same clouds"),
                        ((q, boxes, 1, layout._replace(starts=layout.starts.int()), layout), "must be a BlockLayout"),
                        ((q, boxes, 1, layout, layout._replace(block_size=0)), "must be a BlockLayout")):
        with pytest.raises(ValueError, match=match):
            tb.select_blocks(*args)
