"""64-bit restatements of the block operators, dense and written from the
formulas, with bounds on what fp32 accumulation and one rounding of each weight
and output to the tensors' type may differ by."""

import torch


def unit(dtype) -> float:
    """Largest relative error of one rounding."""
    return 2.0**-8 if dtype == torch.bfloat16 else 2.0**-24


def layout_lists(sizes, block):
    """(offsets, starts, clouds) of packed clouds, by counting."""
    offsets, starts, clouds = [0], [], [0]
    for n in sizes:
        starts += range(offsets[-1], offsets[-1] + n, block)
        offsets.append(offsets[-1] + n)
        clouds.append(len(starts))
    return offsets, starts + [offsets[-1]], clouds


def multiplicity(selected, q_starts, k_starts):
    """(query rows, key rows): how often row i's block chose row j's."""
    out = torch.zeros((q_starts[-1], k_starts[-1]), dtype=torch.float64)
    blocks = len(k_starts) - 1
    for g, chosen in enumerate(selected.tolist()):
        for b in chosen:
            if 0 <= b < blocks:
                out[q_starts[g] : q_starts[g + 1], k_starts[b] : k_starts[b + 1]] += 1
    return out


def attention(q, k, v, times, scale, bias=None, grad=None):
    """Outputs, gradients and bounds of attention, head by head, on the CPU.
    `bias`: (table, buckets, query_cells, key_cells).  Returns {name: (value, bound)}."""
    kind = q.dtype
    u, f = unit(kind), 2.0**-24
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    rows, heads, D = q.shape
    share = heads // k.shape[1]
    n = int(times.sum(1).max()) if times.numel() else 0
    out, out_bound = torch.zeros_like(q), torch.zeros_like(q)
    names = {"out": (out, out_bound)}
    if grad is not None:
        grad = grad.detach().cpu().double()
        for name, t in (("dq", q), ("dk", k), ("dv", v)):
            names[name] = (torch.zeros_like(t), torch.zeros_like(t))
    if bias is not None:
        table, buckets, qc, kc = (t.detach().cpu() for t in bias)
        table = table.double()
        reach = len(buckets) // 2
        which = buckets[(qc[:, None].long() - kc[None].long()).clamp(-reach, reach) + reach].long()
        if grad is not None:
            names["dtable"] = (torch.zeros_like(table), torch.zeros_like(table))
    calls = times.sum(0)
    for h in range(heads):
        c = h // share
        s = q[:, h] @ k[:, c].T * scale
        # Error of a score: D products summed, scaled, D + 1 biases added.
        size = q[:, h].abs() @ k[:, c].abs().T * abs(scale)
        if bias is not None:
            for a in range(table.shape[0]):
                s = s + table[a, :, h][which[..., a]]
                size = size + table[a, :, h][which[..., a]].abs()
        seen = torch.where(times > 0, s, -torch.inf)
        top = seen.amax(1, keepdim=True) if s.shape[1] else torch.full((rows, 1), -torch.inf, dtype=torch.float64)
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        w = times * torch.exp(torch.where(times > 0, s - top, -torch.inf))
        p = w / w.sum(1, keepdim=True).clamp(min=1e-300)
        # Relative error of a weight: the scores' (also the maximum's and the
        # sum's, in the same units), an exponential, a sum of n weights.
        err = (D + 8) * f * torch.where(times > 0, size, torch.zeros_like(size)).amax(1, keepdim=True) if n else 0.0
        rel = 4 * err + (n + 32) * f
        o = p @ v[:, c]
        out[:, h] = o
        out_bound[:, h] = u * o.abs() + (u + rel) * 1.01 * (p @ v[:, c].abs()) + 1e-37
        if grad is None:
            continue
        g = grad[:, h]
        dp = g @ v[:, c].T
        dp_size = g.abs() @ v[:, c].abs().T
        delta = (g * o).sum(1, keepdim=True)
        ds = p * (dp - delta)
        # delta is formed from the stored output.
        delta_err = (g.abs() * out_bound[:, h]).sum(1, keepdim=True) + (D + 8) * f * (g * o).abs().sum(1, keepdim=True)
        ds_err = p * ((D + 8) * f * dp_size + delta_err) + (rel + 4 * f) * p * (dp.abs() + delta.abs())
        rounded = ds_err + u * (ds.abs() + ds_err)
        m = max(n, 1) + 32
        value, bound = names["dq"]
        value[:, h] = ds @ k[:, c] * scale
        bound[:, h] = (rounded + m * f * ds.abs()) @ k[:, c].abs() * abs(scale) + u * value[:, h].abs() + 1e-37
        terms = (calls * share)[:, None] + 32
        value, bound = names["dk"]
        value[:, c] += ds.T @ q[:, h] * scale
        bound[:, c] += (rounded.T @ q[:, h].abs() + terms * f * (ds.abs().T @ q[:, h].abs())) * abs(scale)
        value, bound = names["dv"]
        value[:, c] += p.T @ g
        bound[:, c] += ((u + rel) * 1.01 * p).T @ g.abs() + terms * f * (p.T @ g.abs())
        if bias is not None:
            value, bound = names["dtable"]
            total = (times > 0).sum().item() + 32
            for a in range(table.shape[0]):
                value[a, :, h] += torch.bincount(which[..., a].flatten(), ds.flatten(), table.shape[1])
                # Sums of 64 lanes' and 192 parts' partial sums: their depth, not their length.
                slack = ds_err + min(total, 16384) * f * ds.abs()
                bound[a, :, h] += torch.bincount(which[..., a].flatten(), slack.flatten(), table.shape[1])
    for name in ("dk", "dv", "dtable"):
        if name in names:
            value, bound = names[name]
            bound += u * value.abs() + u * bound + 1e-37
    return names


def group_norm(x, offsets, groups, weight, bias, eps, activation, grad=None):
    """Outputs, gradients and bounds of group norm with an activation, cloud by
    cloud, on the CPU.  Returns {name: (value, bound)}."""
    u, f = unit(x.dtype), 2.0**-24
    x = x.detach().cpu().double()
    C = x.shape[1]
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight.detach().cpu().double()
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias.detach().cpu().double()
    grad = None if grad is None else grad.detach().cpu().double()
    out, out_bound = torch.zeros_like(x), torch.zeros_like(x)
    names = {"out": (out, out_bound)}
    if grad is not None:
        names |= {"dx": (torch.zeros_like(x), torch.zeros_like(x)), "dw": (torch.zeros_like(w), torch.zeros_like(w)),
                  "db": (torch.zeros_like(b), torch.zeros_like(b))}
    for lo, hi in zip(offsets, offsets[1:]):
        n = hi - lo
        if n == 0:
            continue
        rows = x[lo:hi].reshape(n, groups, -1)
        count = n * rows.shape[2]
        mean = rows.mean((0, 2), keepdim=True)
        var = (rows - mean).square().mean((0, 2), keepdim=True)
        rstd = 1.0 / torch.sqrt(var + eps)
        hat = ((rows - mean) * rstd).reshape(n, C)
        # Means of means: their depth is at most 8 + 9 (rows of a thread and of a
        # group of threads) + 11 (slices) joins of three roundings, on values of
        # the largest magnitude; the variance has the same depth, and a mean that
        # is off by e adds e^2 to it.
        most = rows.abs().amax((0, 2), keepdim=True)
        mean_err = 96 * f * most
        var_err = 192 * f * var + 4 * mean_err * torch.sqrt(var) + mean_err.square()
        rel = var_err / (var + eps) + 8 * f
        hat_err = (mean_err * rstd + 4 * f * most * rstd).expand_as(rows).reshape(n, C) \
            + rel.expand_as(rows).reshape(n, C) * hat.abs()
        z = hat * w + b
        z_err = hat_err * w.abs() + 4 * f * (hat * w).abs() + 4 * f * b.abs()
        # Slopes are below 1.13, their own slopes below 1.2; exponentials and the
        # error function are good to a few units in the last place of 1.
        y, s, steps = _activation(z, activation, z_err)
        out[lo:hi] = y
        out_bound[lo:hi] = u * y.abs() + 1.2 * z_err + 16 * f * (z.abs() + y.abs()) + 1e-37
        if grad is None:
            continue
        up = grad[lo:hi]
        dz = up * s
        s_err = torch.where(steps, torch.full_like(z, 1.2), 1.2 * z_err + 32 * f * (1 + z.abs()))
        dz_err = up.abs() * s_err + 2 * f * dz.abs()
        names["dw"][0].add_((dz * hat).sum(0))
        names["dw"][1].add_((dz_err * hat.abs() + dz.abs() * hat_err).sum(0) + min(n + 64, 4096) * f * (dz * hat).abs().sum(0))
        names["db"][0].add_(dz.sum(0))
        names["db"][1].add_(dz_err.sum(0) + min(n + 64, 4096) * f * dz.abs().sum(0))
        t = dz * w
        t_err = dz_err * w.abs() + 2 * f * t.abs()

        def group_mean(a):
            return a.reshape(n, groups, -1).sum((0, 2), keepdim=True).div(count).expand_as(rows).reshape(n, C)

        m, mh = group_mean(t), group_mean(t * hat)
        deep = min(count + 64, 8192) * f
        m_err = group_mean(t_err) + deep * group_mean(t.abs())
        mh_err = group_mean(t_err * hat.abs() + t.abs() * hat_err) + deep * group_mean((t * hat).abs())
        wide = rstd.expand_as(rows).reshape(n, C)
        dx = wide * (t - m - hat * mh)
        names["dx"][0][lo:hi] = dx
        names["dx"][1][lo:hi] = u * dx.abs() + wide * (1 + u) * (
            t_err + m_err + hat_err * mh.abs() + hat.abs() * mh_err + 8 * f * (t.abs() + m.abs() + (hat * mh).abs())
            + rel.expand_as(rows).reshape(n, C) * (t - m - hat * mh).abs()) + 1e-37
    if grad is not None:
        # Parameters may be fp32 beside a narrower x; the caller scales by their unit.
        for name, p in (("dw", weight), ("db", bias)):
            if p is not None:
                names[name][1].add_(unit(p.dtype) * names[name][0].abs() + 1e-37)
    return names


def _activation(z, name, z_err):
    """(value, slope, where the slope jumps within z's error)."""
    never = torch.zeros_like(z, dtype=torch.bool)
    if name == "relu":
        return z.clamp(min=0.0), (z > 0).double(), z.abs() <= z_err
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s)), never
    if name == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5, never
    return z, torch.ones_like(z), never


def within(got, want) -> None:
    """Every value inside its bound."""
    for name, (value, bound) in want.items():
        x = got[name].detach().cpu().double()
        assert x.shape == value.shape, name
        off = (x - value).abs()
        worst = (off / bound).max().item() if off.numel() else 0.0
        assert bool((off <= bound).all()), f"{name}: {worst:.3g} times its bound"
