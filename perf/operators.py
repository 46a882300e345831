"""Performance cases of the operators around attention between points: the
choice of blocks, attention over the chosen blocks with a learned bias of the
relative position, and group norm with an activation.

Rows (points, tokens) are packed cloud after cloud in curve order and cut into
blocks of at most ``block`` rows that never straddle two clouds; ``starts``
holds each block's first row, ``clouds`` each cloud's first block and
``offsets`` each cloud's first row.  A case is a dict of plain values; ``op``
names the operator:

- ``select``: for every block of queries (one query to 64) the ``count`` blocks
  whose boxes are nearest to the centre of the queries' box, ties to the lower
  block number.
- ``attend``: attention of every block of queries over its chosen blocks, with
  or without the bias; ``train`` adds the gradients.
- ``norm``: group norm with an activation over channels-last rows; ``train``
  adds the gradients.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}

# Largest (query, key, head) count of one chunk of exact()'s arrays in 64 bits.
EXACT_CHUNK = 1 << 26


def listed():
    return [
        # A decoder asks a field at a handful of places: latency counts.
        {"name": "select_16_of_65k", "op": "select", "clouds": 1, "least": 65_536, "most": 65_536, "queries": 16,
         "query_block": 1, "block": 64, "dim": 3, "count": 16},
        # A training batch of scans of very different sizes, every patch of 64
        # points of a cloud looks for its neighbour patches.
        {"name": "select_ragged_16", "op": "select", "clouds": 16, "least": 1_000, "most": 60_013, "queries": 0,
         "query_block": 64, "block": 64, "dim": 3, "count": 16},
        # The patches of one million points.
        {"name": "select_1m", "op": "select", "clouds": 1, "least": 1_048_576, "most": 1_048_576, "queries": 0,
         "query_block": 64, "block": 64, "dim": 3, "count": 32},
        # One probe of a field of 65,536 points, the single-token call.
        {"name": "attend_1_of_65k", "op": "attend", "clouds": 1, "least": 65_536, "most": 65_536, "queries": 1,
         "query_block": 1, "block": 64, "dim": 3, "count": 16, "heads": 8, "kv_heads": 8, "channels": 64,
         "type": "bfloat16", "bias": False, "train": False},
        # Two thousand probes that share two heads of keys between eight of
        # queries, with the bias, in the library's own type.
        {"name": "attend_2k_shared", "op": "attend", "clouds": 1, "least": 50_000, "most": 50_000, "queries": 2_000,
         "query_block": 1, "block": 64, "dim": 2, "count": 8, "heads": 8, "kv_heads": 2, "channels": 32,
         "type": "float32", "bias": True, "train": False},
        # A batch of small planar clouds (the published benchmark's shape)
        # through a layer's forward pass.
        {"name": "attend_16x10k", "op": "attend", "clouds": 16, "least": 10_000, "most": 10_000, "queries": 0,
         "query_block": 64, "block": 64, "dim": 2, "count": 8, "heads": 4, "kv_heads": 4, "channels": 32,
         "type": "bfloat16", "bias": True, "train": False},
        # A training step in the library's own type, odd sizes.
        {"name": "attend_train_f32", "op": "attend", "clouds": 3, "least": 4_999, "most": 14_999, "queries": 0,
         "query_block": 64, "block": 64, "dim": 3, "count": 8, "heads": 4, "kv_heads": 4, "channels": 24,
         "type": "float32", "bias": True, "train": True},
        # A training step over scans of different sizes.
        {"name": "attend_train_ragged", "op": "attend", "clouds": 8, "least": 1_000, "most": 20_011, "queries": 0,
         "query_block": 64, "block": 64, "dim": 3, "count": 16, "heads": 8, "kv_heads": 8, "channels": 32,
         "type": "bfloat16", "bias": True, "train": True},
        # The forward pass of a wide layer over a large cloud.
        {"name": "attend_262k", "op": "attend", "clouds": 1, "least": 262_144, "most": 262_144, "queries": 0,
         "query_block": 64, "block": 64, "dim": 3, "count": 16, "heads": 8, "kv_heads": 8, "channels": 64,
         "type": "bfloat16", "bias": False, "train": False},
        # The norm of a small cloud's features.
        {"name": "norm_1k", "op": "norm", "clouds": 1, "least": 1_000, "most": 1_000, "channels": 64, "groups": 8,
         "type": "float32", "activation": "silu", "train": False},
        # A training step over scans of different sizes, odd channels.
        {"name": "norm_train_ragged", "op": "norm", "clouds": 16, "least": 1_000, "most": 60_013, "channels": 88,
         "groups": 8, "type": "bfloat16", "activation": "gelu", "train": True},
        # A training step over one million points of 256 channels.
        {"name": "norm_train_1m", "op": "norm", "clouds": 1, "least": 1_048_576, "most": 1_048_576,
         "channels": 256, "groups": 32, "type": "bfloat16", "activation": "silu", "train": True},
    ]


def _log_int(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def draw(rng):
    op = rng.choice(["select", "attend", "attend", "attend", "norm"])
    kind = rng.choice(["float32", "bfloat16"])
    clouds = rng.choice([1, 1, 2, 7, 16])
    if op == "norm":
        channels = 8 * rng.randint(2, 32)
        groups = rng.choice([g for g in (1, 2, 4, 8, 16, 32) if channels % g == 0])
        most = _log_int(rng, 500, 1_048_576 * 256 // (2 * channels * clouds))
        return {"op": op, "clouds": clouds, "least": max(1, most // rng.randint(1, 9)), "most": most,
                "channels": channels, "groups": groups, "type": kind,
                "activation": rng.choice(["none", "relu", "gelu", "silu"]), "train": rng.random() < 0.5}
    probes = rng.random() < 0.4
    case = {"op": op, "clouds": clouds, "queries": _log_int(rng, 1, 4_000) if probes else 0,
            "query_block": 1 if probes else rng.choice([32, 64]), "block": 64, "dim": rng.choice([2, 3, 3]),
            "count": rng.choice([4, 8, 13, 16, 32])}
    if op == "select":
        most = _log_int(rng, 200, 600_000 // clouds)
        return {**case, "least": max(1, most // rng.randint(1, 9)), "most": most}
    heads, share = rng.choice([(1, 1), (4, 1), (4, 4), (6, 1), (8, 1), (8, 2)])
    case |= {"heads": heads, "kv_heads": heads // share, "channels": rng.choice([16, 24, 32, 48, 64, 128]),
             "type": kind, "bias": rng.random() < 0.6, "train": rng.random() < 0.4}
    # Pairs times heads times channels below the largest listed case's.
    room = 262_144 * 1024 * 8 * 64 // (case["count"] * 64 * heads * case["channels"] * clouds)
    room //= (4 if case["train"] else 1) * (8 if kind == "float32" else 2) * (2 if case["bias"] else 1)
    if case["bias"]:
        # The plain form holds the buckets of every pair as unit vectors.
        room = min(room, 80_000_000 // (case["count"] * 64 * clouds))
    most = _log_int(rng, 100, max(101, min(room, 262_144 // clouds)))
    return {**case, "least": max(1, most // rng.randint(1, 9)), "most": most}


# ---- inputs -----------------------------------------------------------------

def _sizes(case):
    g = np.random.default_rng(case["clouds"] * 1009 + case["most"])
    return g.integers(case["least"], case["most"] + 1, size=case["clouds"]).tolist()


def _query_sizes(case):
    """Queries per cloud; a case without a number of its own asks at its points."""
    if case["queries"] == 0:
        return _sizes(case)
    n, b = case["queries"], case["clouds"]
    return [(n * (i + 1)) // b - (n * i) // b for i in range(b)]


def _layout(sizes, block):
    """(offsets, starts, clouds, block) of packed clouds of these sizes."""
    offsets = np.concatenate([[0], np.cumsum(sizes)])
    clouds = np.concatenate([[0], np.cumsum([-(-s // block) for s in sizes])])
    starts = np.concatenate([np.arange(a, b, block) for a, b in zip(offsets, offsets[1:])] + [offsets[-1:]])
    return tuple(torch.from_numpy(x.astype(np.int64)).to(DEVICE) for x in (offsets, starts, clouds)) + (block,)


def _curve(points, cloud):
    """Rows of the packed points in Morton order within each cloud."""
    dim = points.shape[1]
    bits = torch.arange(10, device=points.device)
    cells = (points.clamp(0.0, 1.0) * 1023.0).long()
    spread = (((cells[:, :, None] >> bits) & 1) << (bits * dim)).sum(-1)
    code = (spread << torch.arange(dim, device=points.device)).sum(-1)
    return torch.argsort((cloud << 30) | code, stable=True)


def _points(sizes, dim, g):
    total = sum(sizes)
    cloud = torch.repeat_interleave(torch.arange(len(sizes), device=DEVICE), torch.tensor(sizes, device=DEVICE),
                                    output_size=total)
    # Half the points in the volume, half near a sphere's surface.
    points = torch.rand((total, dim), generator=g, device=DEVICE)
    away = torch.randn((total, dim), generator=g, device=DEVICE)
    away = 0.5 + 0.4 * away / away.norm(dim=1, keepdim=True).clamp(min=1e-6)
    points = torch.where((torch.arange(total, device=DEVICE) % 2 == 0)[:, None], points, away)
    return points[_curve(points, cloud)].contiguous()


def _rows(layout):
    """(blocks, block) row numbers of a layout's blocks, clamped to the
    block's last row, and which of them are real."""
    _, starts, _, block = layout
    rows = starts[:-1, None] + torch.arange(block, device=starts.device)
    last = starts[1:, None] - 1
    return torch.minimum(rows, last), rows <= last


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    state = {"case": case}
    if case["op"] == "norm":
        kind, channels = TYPES[case["type"]], case["channels"]
        sizes = _sizes(case)
        state["layout"] = _layout(sizes, 64)
        total = sum(sizes)
        x = normal(total, channels) * (0.5 + torch.rand(channels, generator=g, device=DEVICE)) + normal(channels)
        state["x"] = x.to(kind)
        state["weight"] = 1.0 + 0.2 * normal(channels)
        state["bias"] = 0.2 * normal(channels)
        if case["train"]:
            state["grad"] = normal(total, channels).to(kind)
        return state
    sizes = _sizes(case)
    state["key_layout"] = _layout(sizes, case["block"])
    points = _points(sizes, case["dim"], g)
    if case["queries"]:
        queries = _points(_query_sizes(case), case["dim"], g)
    else:
        queries = points
    state["query_layout"] = _layout(_query_sizes(case), case["query_block"])
    rows, _ = _rows(state["key_layout"])
    boxes = torch.cat([points[rows].amin(1), points[rows].amax(1)], dim=1)
    state["queries"], state["boxes"] = queries, boxes
    if case["op"] == "select":
        return state
    kind, d = TYPES[case["type"]], case["channels"]
    state["selected"] = _select(queries, boxes, case["count"], state["query_layout"], state["key_layout"])
    state["q"] = normal(queries.shape[0], case["heads"], d).to(kind)
    state["k"] = normal(points.shape[0], case["kv_heads"], d).to(kind)
    state["v"] = normal(points.shape[0], case["kv_heads"], d).to(kind)
    if case["bias"]:
        # Cells about as wide as a patch of 16 points, distances up to 24 cells
        # in 16 buckets a side: exact up to 8, then ever coarser.
        cell = (16 / case["most"]) ** (1 / case["dim"])
        far = torch.arange(-24, 25, device=DEVICE)
        step = 8 + (8 * (far.abs().clamp(min=8) / 8.0).log() / math.log(3.0)).int().clamp(max=7)
        bucket = torch.where(far.abs() < 8, far.abs(), step)
        state["buckets"] = torch.where(far < 0, bucket + 15, bucket).int()
        state["query_cells"] = (queries / cell).int()
        state["key_cells"] = (points / cell).int()
        state["table"] = (0.5 * normal(case["dim"], 31, case["heads"])).to(kind)
    if case["train"]:
        state["grad"] = normal(queries.shape[0], case["heads"], d).to(kind)
    return state


# ---- the operators in plain tensor operations -------------------------------

def _select(queries, boxes, count, query_layout, key_layout):
    """The `count` nearest boxes of every block of queries, as int32 block
    numbers in ascending (score, number), -1 where a cloud has fewer."""
    rows, _ = _rows(query_layout)
    centre = queries[rows].amin(1) * 0.5 + queries[rows].amax(1) * 0.5
    dim = queries.shape[1]
    lo, hi = boxes[:, :dim], boxes[:, dim:]
    groups, blocks = rows.shape[0], boxes.shape[0]

    def away(a):
        c = centre[:, None, a]
        d = torch.maximum(lo[None, :, a] - c, c - hi[None, :, a]).clamp(min=0.0)
        return d * d

    score = away(0) + away(1)
    if dim == 3:
        score = score + away(2)
    group_cloud = torch.searchsorted(query_layout[2], torch.arange(groups, device=boxes.device), right=True)
    block_cloud = torch.searchsorted(key_layout[2], torch.arange(blocks, device=boxes.device), right=True)
    here = (group_cloud[:, None] == block_cloud[None, :]) & torch.isfinite(score)
    key = (score.view(torch.int32).long() << 32) | torch.arange(blocks, device=boxes.device)
    none = torch.iinfo(torch.int64).max
    key = torch.where(here, key, none)
    best = torch.topk(key, min(count, blocks), dim=1, largest=False, sorted=True).values
    chosen = torch.where(best == none, -1, best & 0xFFFFFFFF).int()
    return torch.nn.functional.pad(chosen, (0, count - chosen.shape[1]), value=-1)


def _attend(state, q, k, v, table):
    """Softmax attention of padded groups of queries over their gathered keys,
    in float32; a row without keys is zero."""
    (rows, real), (key_rows, key_real) = _rows(state["query_layout"]), _rows(state["key_layout"])
    selected = state["selected"].long()
    groups, block = rows.shape
    heads, d = q.shape[1:]
    kv, share = k.shape[1], heads // k.shape[1]
    at = key_rows[selected.clamp(min=0)].reshape(groups, -1)
    has = (key_real[selected.clamp(min=0)] & (selected >= 0)[..., None]).reshape(groups, 1, 1, 1, -1)
    keys = k[at].permute(0, 2, 3, 1).unsqueeze(2)       # (groups, kv, 1, d, keys)
    values = v[at].permute(0, 2, 1, 3).unsqueeze(2)     # (groups, kv, 1, keys, d)
    ask = q[rows].reshape(groups, block, kv, share, d).permute(0, 2, 3, 1, 4)
    logits = torch.matmul(ask, keys.contiguous()) / math.sqrt(d)
    if table is not None:
        reach = (state["buckets"].shape[0] - 1) // 2
        apart = state["query_cells"][rows][:, :, None] - state["key_cells"][at][:, None]
        bucket = state["buckets"][apart.clamp(-reach, reach) + reach].reshape(groups, -1, apart.shape[-1])

        def along(a):
            # A product with the buckets as unit vectors: its gradient is a
            # product too, summed group by group.
            unit = (bucket[..., a, None] == torch.arange(table.shape[1], device=q.device)).float()
            return torch.bmm(unit, table[a].expand(groups, -1, -1))

        bias = along(0) if table.shape[0] == 1 else along(0) + along(1)
        if table.shape[0] == 3:
            bias = bias + along(2)
        logits = logits + bias.reshape(groups, block, at.shape[1], kv, share).permute(0, 3, 4, 1, 2)
    logits = logits.masked_fill(~has, -math.inf)
    most = logits.detach().amax(-1, keepdim=True)
    weight = torch.exp(logits - most.masked_fill(torch.isinf(most), 0.0))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight / total.masked_fill(total == 0.0, 1.0), values.contiguous())
    return out.permute(0, 3, 1, 2, 4).reshape(groups, block, heads, d)[real]


def _activate(z, activation):
    if activation == "relu":
        return torch.relu(z)
    if activation == "silu":
        return z / (1.0 + torch.exp(-z))
    if activation == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _norm(x, weight, bias, offsets, groups, activation):
    """Group norm of every cloud's rows, padded to the longest cloud's."""
    counts = offsets[1:] - offsets[:-1]
    clouds, longest = counts.shape[0], int(counts.max())
    cloud = torch.repeat_interleave(torch.arange(clouds, device=x.device), counts, output_size=x.shape[0])
    slot = torch.arange(x.shape[0], device=x.device) - offsets[cloud] + cloud * longest
    wide = torch.zeros((clouds * longest, x.shape[1]), device=x.device).index_copy(0, slot, x)
    wide = wide.reshape(clouds, longest, groups, -1)
    real = (torch.arange(longest, device=x.device) < counts[:, None])[..., None, None]
    n = (counts * wide.shape[3])[:, None, None, None]
    apart = (wide - wide.sum((1, 3), keepdim=True) / n) * real
    hat = apart * torch.rsqrt((apart * apart).sum((1, 3), keepdim=True) / n + 1e-5)
    z = hat.reshape(clouds * longest, -1).index_select(0, slot) * weight + bias
    return _activate(z, activation)


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "select":
        return _select(state["queries"], state["boxes"], case["count"], state["query_layout"], state["key_layout"])
    train = case["train"]
    names = ["x", "weight", "bias"] if case["op"] == "norm" else ["q", "k", "v", "table"][: 4 if case["bias"] else 3]
    with torch.set_grad_enabled(train):
        wide = [state[n].float().requires_grad_(train) if state[n].dtype != torch.float32
                else state[n].detach().requires_grad_(train) for n in names]
        if case["op"] == "norm":
            out = _norm(*wide, state["layout"][0], case["groups"], case["activation"])
        else:
            out = _attend(state, *wide, *([None] if not case["bias"] else []))
    result = {"out": out.detach().to(state[names[0]].dtype)}
    if train:
        grads = torch.autograd.grad(out, wide, state["grad"].float())
        result |= {"d" + n: x.to(state[n].dtype) for n, x in zip(names, grads)}
    return result


# ---- the same through the library -------------------------------------------

def _run_own(state, case):
    import torchbvh_amd as tb

    def layout(name):
        return tb.BlockLayout(*state[name])

    if case["op"] == "select":
        return tb.select_blocks(state["queries"], state["boxes"], case["count"], layout("query_layout"),
                                layout("key_layout"))
    train = case["train"]
    names = ["x", "weight", "bias"] if case["op"] == "norm" else ["q", "k", "v", "table"][: 4 if case["bias"] else 3]
    with torch.set_grad_enabled(train):
        given = [state[n].detach().requires_grad_(train) for n in names]
        if case["op"] == "norm":
            out = tb.group_norm_act(given[0], case["groups"], given[1], given[2], layout("layout"),
                                    activation=case["activation"])
        else:
            bias = None
            if case["bias"]:
                bias = tb.RelativeBias(given[3], state["buckets"], state["query_cells"], state["key_cells"])
            out = tb.block_attention(*given[:3], state["selected"], layout("query_layout"), layout("key_layout"),
                                     bias=bias)
    result = {"out": out.detach()}
    if train:
        grads = torch.autograd.grad(out, given, state["grad"])
        result |= {"d" + n: x for n, x in zip(names, grads)}
    return result


# ---- what a pass cannot do without ------------------------------------------

def _pairs(case):
    """(query rows, key rows, (query, key) pairs, key rows that some query reads)."""
    sizes, asked = _sizes(case), _query_sizes(case)
    blocks = [min(case["count"], -(-s // case["block"])) for s in sizes]
    pairs = sum(n * min(b * case["block"], s) for n, b, s in zip(asked, blocks, sizes))
    groups = [-(-n // case["query_block"]) for n in asked]
    read = sum(min(s, g * b * case["block"]) for s, g, b in zip(sizes, groups, blocks))
    return sum(asked), sum(sizes), pairs, read


def work(case):
    if case["op"] == "norm":
        # x read and y written; dy read and dx written by a training step.
        size = 4 if case["type"] == "float32" else 2
        values = sum(_sizes(case)) * case["channels"]
        return {"bytes": values * size * (4 if case["train"] else 2), "flops": values * (24 if case["train"] else 10)}
    if case["op"] == "select":
        groups = sum(-(-n // case["query_block"]) for n in _query_sizes(case))
        blocks = sum(-(-s // case["block"]) for s in _sizes(case))
        dim, count = case["dim"], case["count"]
        return {"bytes": sum(_query_sizes(case)) * dim * 4 + blocks * dim * 8 + groups * count * 4,
                "flops": groups * min(count, blocks) * dim * 5}
    asked, _, pairs, read = _pairs(case)
    size = 4 if case["type"] == "float32" else 2
    d, heads, kv = case["channels"], case["heads"], case["kv_heads"]
    # Forward: q, k, v read, out written.  Training step: the gradient read, dq, dk and dv written.
    data = (2 * asked * heads + 2 * read * kv) * d * size
    if case["train"]:
        data += (2 * asked * heads + 2 * read * kv) * d * size
    return {"bytes": data, "flops": pairs * heads * d * (14 if case["train"] else 4)}


# ---- the same in 64 bits ----------------------------------------------------

def exact(case, seed):
    if case["op"] == "select":
        return None  # whole numbers only
    state = prepare(case, seed)
    return _exact_norm(state, case) if case["op"] == "norm" else _exact_attend(state, case)


def _exact_norm(state, case):
    x, w, b = (state[n].double() for n in ("x", "weight", "bias"))
    up = state["grad"].double() if case["train"] else None
    out, dx = torch.empty_like(x), torch.empty_like(x)
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    bounds = state["layout"][0].tolist()
    for lo, hi in zip(bounds, bounds[1:]):
        rows = x[lo:hi].reshape(hi - lo, case["groups"], -1)
        var, mean = torch.var_mean(rows, dim=(0, 2), unbiased=False, keepdim=True)
        hat = ((rows - mean) / torch.sqrt(var + 1e-5)).reshape(hi - lo, -1)
        z = hat * w + b
        name = case["activation"]
        if name == "relu":
            y, slope = z.clamp(min=0.0), (z > 0).double()
        elif name == "silu":
            s = torch.sigmoid(z)
            y, slope = z * s, s * (1.0 + z * (1.0 - s))
        elif name == "gelu":
            cdf = torch.special.ndtr(z)
            y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
        else:
            y, slope = z, torch.ones_like(z)
        out[lo:hi] = y
        if up is None:
            continue
        dz = up[lo:hi] * slope
        dw += (dz * hat).sum(0)
        db += dz.sum(0)
        g, h = (dz * w).reshape(rows.shape), hat.reshape(rows.shape)
        g = g - g.mean((0, 2), keepdim=True) - h * (g * h).mean((0, 2), keepdim=True)
        dx[lo:hi] = (g / torch.sqrt(var + 1e-5)).reshape(hi - lo, -1)
    return {"out": out} if up is None else {"out": out, "dx": dx, "dweight": dw, "dbias": db}


def _exact_attend(state, case):
    q, k, v = (state[n].double() for n in ("q", "k", "v"))
    up = state["grad"].double() if case["train"] else None
    heads, kv, d = case["heads"], case["kv_heads"], case["channels"]
    starts, key_starts = state["query_layout"][1], state["key_layout"][1]
    groups, block, count = starts.shape[0] - 1, case["query_block"], case["count"]
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    table = state["table"].double() if case["bias"] else None
    dtable = torch.zeros_like(table) if case["bias"] else None
    step = max(1, EXACT_CHUNK // (block * count * 64 * heads))
    for first in range(0, groups, step):
        ids = torch.arange(first, min(groups, first + step), device=DEVICE)
        rows = starts[ids, None] + torch.arange(block, device=DEVICE)
        asks = rows < starts[ids + 1, None]
        rows = torch.where(asks, rows, starts[ids, None])
        chosen = state["selected"][ids].long()
        at = key_starts[chosen.clamp(min=0), None] + torch.arange(case["block"], device=DEVICE)
        there = (at < key_starts[chosen.clamp(min=0) + 1, None]) & (chosen >= 0)[..., None]
        at = torch.where(there, at, 0).flatten(1)
        mask = asks[:, :, None] & there.flatten(1)[:, None, :]
        if case["bias"]:
            reach = (state["buckets"].shape[0] - 1) // 2
            apart = state["query_cells"][rows][:, :, None, :] - state["key_cells"][at][:, None, :, :]
            bucket = state["buckets"][apart.clamp(-reach, reach) + reach].long()
        for h in range(heads):
            c = h * kv // heads
            qs, ks, vs = q[rows, h], k[at, c], v[at, c]
            s = torch.bmm(qs, ks.transpose(1, 2).contiguous()) * d ** -0.5
            if case["bias"]:
                for a in range(case["dim"]):
                    s += table[a, :, h][bucket[..., a]]
            s = torch.where(mask, s, torch.tensor(-math.inf, dtype=s.dtype, device=DEVICE))
            lse = torch.logsumexp(s, -1, keepdim=True)
            p = torch.where(mask, torch.exp(s - lse), torch.zeros_like(s))
            o = torch.bmm(p, vs)
            out[rows[asks], h] = o[asks]
            if up is None:
                continue
            go = up[rows, h] * asks[..., None]
            dp = torch.bmm(go, vs.transpose(1, 2).contiguous())
            ds = p * (dp - (go * o).sum(-1, keepdim=True))
            dq[rows[asks], h] = (torch.bmm(ds, ks) * d ** -0.5)[asks]
            flat = at.flatten()
            dk[:, c].index_add_(0, flat, torch.bmm(ds.transpose(1, 2).contiguous(), qs).flatten(0, 1) * d ** -0.5)
            dv[:, c].index_add_(0, flat, torch.bmm(p.transpose(1, 2).contiguous(), go).flatten(0, 1))
            if case["bias"]:
                for a in range(case["dim"]):
                    dtable[a, :, h] += torch.bincount(bucket[..., a].flatten(), ds.flatten(), table.shape[1])
    if up is None:
        return {"out": out}
    result = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    return result | {"dtable": dtable} if case["bias"] else result
