"""Measured work of the feature operators behind the sampler: row lookup with
its gradient (``group.gather_rows``), the choice of the nearest blocks of a
cloud (``attention.select_blocks``) and attention over them with its gradient
(``attention.block_attention``).

``run`` computes a case with elementary torch operations, or, where ``own`` is
set, with the package's operators.  Sizes follow the workloads of the
repository's benchmark (10,000 points -> 1,000 samples; 122,880 -> 16,384;
32 clouds of 16,384 -> 4,096; 1,048,576 points).
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _rows(name, B, N, C, P, dtype, pattern, grad, scale):
    return {"name": name, "op": "rows", "B": B, "N": N, "C": C, "P": P, "dtype": dtype,
            "pattern": pattern, "grad": grad, "scale": scale}


def _select(name, B, N, M, block, top, ragged):
    return {"name": name, "op": "select", "B": B, "N": N, "M": M, "block": block, "top": top,
            "ragged": ragged}


def _attend(name, B, N, M, H, G, D, block, top, dtype, ragged, grad):
    return {"name": name, "op": "attend", "B": B, "N": N, "M": M, "H": H, "G": G, "D": D,
            "block": block, "top": top, "dtype": dtype, "ragged": ragged, "grad": grad}


def listed():
    return [
        # features of the 1,000 samples of a small cloud: a call's latency
        _rows("rows 10k cloud samples", 1, 10_000, 64, 1_000, "fp32", "spread", False, 1.0),
        # features of 16 neighbours of every sample, 32 clouds: bandwidth
        _rows("rows 32 clouds grouped", 32, 16_384, 64, 65_536, "bf16", "near", False, 1.0),
        # the same in training, 8 neighbours and wider features
        _rows("rows 32 clouds train", 32, 16_384, 96, 32_768, "bf16", "near", True, 1.0),
        # a learned table looked up by skewed ids with padding, scaled by sqrt(width)
        _rows("rows skewed table train", 1, 50_021, 200, 30_011, "fp32", "skewed", True,
              math.sqrt(200.0)),
        # one new centre in a LiDAR scan
        _select("select one centre", 1, 122_880, 1, 64, 16, False),
        # the batch of 32 padded clouds
        _select("select 32 clouds", 32, 16_384, 4_096, 32, 16, True),
        # all samples of a LiDAR scan
        _select("select scan", 1, 122_880, 16_384, 64, 16, False),
        # a single token of a long scan
        _attend("attend one query", 1, 122_880, 1, 8, 8, 64, 64, 16, "bf16", False, False),
        # a few tokens over a million keys, shared heads
        _attend("attend few, 1M keys", 1, 1_048_576, 16, 16, 2, 128, 128, 64, "bf16", False, False),
        # all samples of a LiDAR scan, inference
        _attend("attend scan", 1, 122_880, 16_384, 4, 4, 64, 32, 16, "fp16", False, False),
        # training, shared heads, odd lengths
        _attend("train shared heads", 2, 8_191, 1_023, 8, 2, 128, 64, 8, "bf16", True, True),
        # training on four padded clouds
        _attend("train 4 clouds", 4, 16_384, 4_096, 4, 4, 64, 32, 16, "bf16", True, True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rows", "rows", "select", "attend", "attend", "attend"])
    if op == "rows":
        B, C = log(1, 32), log(3, 256)
        N, P = log(1, 60_000), log(1, 60_000)
        most = 30_000_000  # elements of the output or of the table
        c = _rows("", B, max(1, min(N, most // (B * C))), C, max(1, min(P, most // (B * C))),
                  rng.choice(["fp32", "bf16", "fp16"]), rng.choice(["spread", "near", "skewed"]),
                  rng.random() < 0.5, rng.choice([1.0, 0.5, math.sqrt(C)]))
    elif op == "select":
        block, top = rng.choice([16, 32, 64, 128]), log(1, 64)
        B, N = log(1, 32), log(2_000, 130_000)
        M = max(1, min(log(1, 16_384), 60_000_000 // (B * (N // block + 1))))
        c = _select("", B, N, M, block, top, rng.random() < 0.5)
    else:
        grad = rng.random() < 0.5
        G, g = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 3, 8])
        D, block, top = 8 * rng.randint(2, 16), rng.choice([16, 32, 64, 128]), log(1, 24)
        B, N = log(1, 4), log(1, 123_000)
        N = max(1, min(N, (25_000_000 if grad else 60_000_000) // (B * G * D)))
        most = 1_000_000_000 if grad else 2_000_000_000  # elements of the gathered keys
        M = max(1, min(log(1, 16_384), most // (B * G * g * D * top * block),
                       20_000_000 // (B * G * g * D)))
        c = _attend("", B, N, M, G * g, G, D, block, top, rng.choice(["bf16", "fp16"]),
                    rng.random() < 0.5, grad)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cloud(B, N, g):
    """Points of B clouds in a spatially coherent order: surfaces of a box and
    clutter, ordered by the Morton code of a 10-bit grid."""
    p = torch.rand(B, N, 3, device="cuda", generator=g) * 2 - 1
    flat = torch.rand(B, N, device="cuda", generator=g) < 0.6
    p[..., 2] = torch.where(flat, p[..., 2] * 0.02 - 0.5, p[..., 2])
    cell = ((p + 1) * 512).long().clamp_(0, 1023)
    code = torch.zeros(B, N, dtype=torch.int64, device="cuda")
    for bit in range(10):
        for a in range(3):
            code |= ((cell[..., a] >> bit) & 1) << (3 * bit + a)
    return torch.gather(p, 1, code.argsort(dim=1)[..., None].expand(B, N, 3)).contiguous()


def _lengths(case, g):
    """Valid points of each padded cloud; of several ragged clouds the last is
    empty."""
    B, N = case["B"], case["N"]
    if not case["ragged"]:
        return None
    n = torch.randint(N // 2 + 1, N + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    if B > 1:
        n[-1] = 0
    return n


def _centers(points, lengths, M, g):
    B, N = points.shape[:2]
    u = torch.rand(B, M, device="cuda", generator=g)
    top = torch.full((B, 1), N, device="cuda") if lengths is None else lengths[:, None].clamp(min=1)
    pick = (u * top).long().clamp_(max=N - 1)
    at = torch.gather(points, 1, pick[..., None].expand(B, M, 3))
    return at + 0.01 * torch.randn(B, M, 3, device="cuda", generator=g)


def prepare(case, seed):
    g = _generator(seed)
    B, N = case["B"], case["N"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(_DTYPES[case["dtype"]])

    state = {"case": case}
    if case["op"] == "rows":
        C, P = case["C"], case["P"]
        u = torch.rand(B, P, device="cuda", generator=g)
        if case["pattern"] == "spread":      # samples: anywhere, few repeats
            idx = (u * N).long()
        elif case["pattern"] == "near":      # neighbours: runs around a moving centre
            at = torch.arange(P, device="cuda") // 16 * 16 * (N / max(P, 1))
            idx = (at + u * 64).long() % N
        else:                                # ids: a power law, some padding (-1)
            idx = ((N + 1) ** u - 1).long()
            idx[torch.rand(B, P, device="cuda", generator=g) < 0.1] = -1
        state["table"] = normal(B, N, C)
        state["idx"] = idx.clamp_(max=N - 1)
        if case["grad"]:
            state["dout"] = normal(B, P, C)
        return state
    points = _cloud(B, N, g)
    lengths = _lengths(case, g)
    state["lengths"] = lengths
    if case["op"] == "select":
        state["points"] = points
        state["centers"] = _centers(points, lengths, case["M"], g)
        return state
    M, H, G, D = case["M"], case["H"], case["G"], case["D"]
    state["blocks"] = _plain_select(points, _centers(points, lengths, M, g), case["block"],
                                    case["top"], lengths)[0]
    state["q"], state["k"], state["v"] = normal(B, M, H, D), normal(B, N, G, D), normal(B, N, G, D)
    if lengths is not None:                  # what lies behind a cloud's end is not data
        pad = torch.arange(N, device="cuda")[None, :] >= lengths[:, None]
        state["k"][pad] = math.nan
        state["v"][pad] = math.nan
    if case["grad"]:
        state["dout"] = normal(B, M, H, D)
    return state


# -------------------------------------------------------------- plain forms

def _plain_rows(table, idx, scale):
    B, N, C = table.shape
    flat = (idx.clamp(min=0) + N * torch.arange(B, device=idx.device)[:, None]).reshape(-1)
    out = table.reshape(B * N, C)[flat].reshape(B, -1, C).float() * scale
    return torch.where((idx >= 0)[..., None], out, 0.0).to(table.dtype)


def _plain_rows_grad(dout, idx, scale, N):
    B, P, C = dout.shape
    flat = (idx.clamp(min=0) + N * torch.arange(B, device=idx.device)[:, None]).reshape(-1)
    add = torch.where((idx >= 0)[..., None], dout.float(), 0.0).reshape(-1, C)
    grad = torch.zeros(B * N, C, device=dout.device).index_add_(0, flat, add)
    return (grad * scale).to(dout.dtype).reshape(B, N, C)


def _plain_select(points, centers, block, top, lengths):
    B, N, _ = points.shape
    M, nb = centers.shape[1], (N + block - 1) // block
    n = torch.full((B,), N, device="cuda") if lengths is None else lengths.long()
    out_of = (torch.arange(nb * block, device="cuda")[None, :] >= n[:, None])[..., None]
    pts = torch.nn.functional.pad(points, (0, 0, 0, nb * block - N))
    lo = torch.where(out_of, math.inf, pts).reshape(B, 1, nb, block, 3).amin(3)
    hi = torch.where(out_of, -math.inf, pts).reshape(B, 1, nb, block, 3).amax(3)
    c = centers[:, :, None, :]

    def square(a):
        d = torch.maximum(lo[..., a] - c[..., a], c[..., a] - hi[..., a]).clamp_(min=0.0)
        return d * d

    d2 = (square(0) + square(1)) + square(2)
    # a block without points lies behind every other one
    none = torch.arange(nb, device="cuda")[None, None, :] * block >= n[:, None, None]
    order = torch.sort(torch.where(none, math.inf, d2), dim=2, stable=True).indices[..., :top]
    missing = torch.gather(none.expand(B, M, nb), 2, order)
    d2 = torch.where(missing, math.inf, torch.gather(d2, 2, order))
    order = torch.where(missing, -1, order)
    more = (0, top - order.shape[2])
    return (torch.nn.functional.pad(order, more, value=-1),
            torch.nn.functional.pad(d2, more, value=math.inf))


def _gathered(t, key, ok):
    B, N, G, D = t.shape
    flat = key.clamp(max=N - 1) + N * torch.arange(B, device=t.device)[:, None, None]
    rows = t.reshape(B * N, G, D).float()[flat]
    return torch.where(ok[..., None, None], rows, 0.0), flat


def _plain_attend(q, k, v, blocks, block, lengths, dout):
    B, M, H, D = q.shape
    N, G = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(D)
    n = torch.full((B,), N, device="cuda") if lengths is None else lengths.long()
    key = (blocks.clamp(min=0)[..., None] * block +
           torch.arange(block, device="cuda")).reshape(B, M, -1)
    ok = (blocks >= 0).repeat_interleave(block, dim=2) & (key < n[:, None, None])
    kg, flat = _gathered(k, key, ok)
    vg, _ = _gathered(v, key, ok)
    qf = q.float().reshape(B, M, G, H // G, D)
    s = torch.einsum("bmgrd,bmtgd->bmgrt", qf, kg) * scale
    s = s.masked_fill(~ok[:, :, None, None, :], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    out = torch.einsum("bmgrt,bmtgd->bmgrd", p, vg).reshape(B, M, H, D).to(q.dtype)
    if dout is None:
        return out
    do = dout.float().reshape(B, M, G, H // G, D)
    dp = torch.einsum("bmgrd,bmtgd->bmgrt", do, vg)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    dq = torch.einsum("bmgrt,bmtgd->bmgrd", ds, kg).reshape(B, M, H, D).to(q.dtype)
    del kg, vg

    def back(w, x):
        rows = torch.einsum("bmgrt,bmgrd->bmtgd", w, x).reshape(-1, G, D)
        full = torch.zeros(B * N, G, D, device="cuda").index_add_(0, flat.reshape(-1), rows)
        return full.reshape(B, N, G, D).to(q.dtype)

    return out, dq, back(ds, qf), back(p, do)


# --------------------------------------------------------------------- run

def run(state):
    c = state["case"]
    if c["op"] == "rows":
        if own:
            from ns_fps_b200 import group
            if not c["grad"]:
                return group.gather_rows(state["table"], state["idx"], c["scale"])
            table = state["table"].detach().requires_grad_()
            out = group.gather_rows(table, state["idx"], c["scale"])
            return out.detach(), torch.autograd.grad(out, table, state["dout"])[0]
        out = _plain_rows(state["table"], state["idx"], c["scale"])
        if not c["grad"]:
            return out
        return out, _plain_rows_grad(state["dout"], state["idx"], c["scale"], c["N"])
    if c["op"] == "select":
        if own:
            from ns_fps_b200 import attention
            return attention.select_blocks(state["points"], state["centers"], c["block"],
                                           c["top"], lengths=state["lengths"])
        return _plain_select(state["points"], state["centers"], c["block"], c["top"],
                             state["lengths"])
    if own:
        from ns_fps_b200 import attention
        if not c["grad"]:
            return attention.block_attention(state["q"], state["k"], state["v"], state["blocks"],
                                             c["block"], lengths=state["lengths"])
        leaves = [state[x].detach().requires_grad_() for x in ("q", "k", "v")]
        out = attention.block_attention(*leaves, state["blocks"], c["block"],
                                        lengths=state["lengths"])
        return (out.detach(), *torch.autograd.grad(out, leaves, state["dout"]))
    return _plain_attend(state["q"], state["k"], state["v"], state["blocks"], c["block"],
                         state["lengths"], state.get("dout"))


# -------------------------------------------------------------------- work

def work(case):
    c, B, N = case, case["B"], case["N"]
    if c["op"] == "rows":
        e = 4 if c["dtype"] == "fp32" else 2
        P, C = c["P"], c["C"]
        seen = min(N, P)  # rows of the table that are read at most
        nbytes = B * (P * 8 + seen * C * e + P * C * e)
        if c["grad"]:
            nbytes += B * (P * C * e + N * C * e)
        return {"bytes": nbytes, "flops": B * P * C * (2 if c["grad"] else 1)}
    M, nb = c["M"], (N + c["block"] - 1) // c["block"]
    if c["op"] == "select":
        return {"bytes": B * (12 * N + 12 * M + 12 * M * c["top"]),
                "flops": B * (6 * N + 14 * M * nb)}
    H, G, D = c["H"], c["G"], c["D"]
    listed_ = min(c["top"], nb)
    keys = min(listed_ * c["block"], N)
    reach = min(N, M * keys)  # keys that any query reads
    nbytes = B * (2 * 2 * M * H * D + 2 * 2 * reach * G * D + 8 * M * c["top"])
    flops = 4 * B * M * H * keys * D
    if c["grad"]:  # reads dout, q, k, v, out again; writes dq, dk, dv
        nbytes += B * (2 * 4 * M * H * D + 2 * 2 * reach * G * D + 2 * 2 * N * G * D)
        flops += 10 * B * M * H * keys * D
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------- the definitions, 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    c, B, N = case, case["B"], case["N"]
    if c["op"] == "select":
        # the blocks are whole numbers by a 32-bit score: no 64-bit value
        d2 = torch.full((B, c["M"], c["top"]), math.inf, dtype=torch.float64, device="cuda")
        for b in range(B):
            n = N if s["lengths"] is None else int(s["lengths"][b])
            parts = s["points"][b, :n].double().split(c["block"])
            if n == 0:
                continue
            lo = torch.stack([p.amin(0) for p in parts])
            hi = torch.stack([p.amax(0) for p in parts])
            ctr = s["centers"][b].double()
            far = torch.zeros(c["M"], len(parts), dtype=torch.float64, device="cuda")
            for a in range(3):
                x = ctr[:, a, None]
                far += (torch.clamp(x, lo[:, a], hi[:, a]) - x) ** 2
            k = min(c["top"], len(parts))
            d2[b, :, :k] = far.sort(dim=1).values[:, :k]
        return None, d2
    if c["op"] == "rows":
        outs, grads = [], []
        for b in range(B):
            idx = s["idx"][b]
            some = idx >= 0
            out = torch.zeros(c["P"], c["C"], dtype=torch.float64, device="cuda")
            out[some] = s["table"][b].double()[idx[some]] * c["scale"]
            outs.append(out)
            if c["grad"]:
                g = torch.zeros(N, c["C"], dtype=torch.float64, device="cuda")
                g.index_add_(0, idx[some], s["dout"][b].double()[some])
                grads.append(g * c["scale"])
        return (torch.stack(outs), torch.stack(grads)) if c["grad"] else torch.stack(outs)
    M, H, G, D, bs = c["M"], c["H"], c["G"], c["D"], c["block"]
    nb, r = (N + bs - 1) // bs, c["H"] // c["G"]
    out = torch.zeros(B, M, H, D, dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(out)
    dk = torch.zeros(B, N, G, D, dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    step = max(1, min(M, 100_000_000 // max(N, 1)))
    for b in range(B):
        n = N if s["lengths"] is None else int(s["lengths"][b])
        if n == 0:
            continue
        for m in range(0, M, step):
            lists = s["blocks"][b, m:m + step]
            member = torch.zeros(lists.shape[0], nb + 1, dtype=torch.bool, device="cuda")
            member.scatter_(1, torch.where(lists < 0, nb, lists), True)
            seen = member[:, :nb].repeat_interleave(bs, dim=1)[:, :n]
            for h in range(H):
                kh, vh = s["k"][b, :n, h // r].double(), s["v"][b, :n, h // r].double()
                qh = s["q"][b, m:m + step, h].double()
                w = torch.where(seen, qh @ kh.T / math.sqrt(D), -math.inf)
                w = torch.nan_to_num(torch.softmax(w, dim=1))
                out[b, m:m + step, h] = w @ vh
                if c["grad"]:
                    oh = s["dout"][b, m:m + step, h].double()
                    dv[b, :n, h // r] += w.T @ oh
                    dw = oh @ vh.T
                    dw = w * (dw - (w * dw).sum(1, keepdim=True)) / math.sqrt(D)
                    dq[b, m:m + step, h] = dw @ kh
                    dk[b, :n, h // r] += dw.T @ qh
    return (out, dq, dk, dv) if c["grad"] else out
