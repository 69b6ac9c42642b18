"""What the attention operators of the framework are measured on: cross attention from the tokens of a frame to the tokens of its
neighbours, and the per-head norms of queries and keys with the position rotation in front of it.

`own` False computes them from elementary torch operations in 32 bits (angles in 64), `own` True calls
`mono_vifi_amd.ops.qk_norm_rope` and `mono_vifi_amd.ops.cross_attention`.  Token counts are those of feature pyramids at
640x192 and 1024x320: an image has 120 / 480 / 1,920 / 7,680 tokens at 1/32 ... 1/4 of 640x192, 1,280 / 5,120 at 1/16 and 1/8 of
1024x320, and two neighbour frames have twice as many."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS, BASE = 1e-6, 10000.0


def _rotate(name, dtype, train, B, Lq, Lk, Hq, Hk, D, axes, rot, pairs, first):
    return {"name": name, "op": "rotate", "dtype": dtype, "train": train, "B": B, "Lq": Lq, "Lk": Lk, "Hq": Hq, "Hk": Hk, "D": D,
            "axes": axes, "rot": rot, "pairs": pairs, "first": first}


def _attend(name, dtype, train, B, Lq, Lk, Hq, Hk, D, mask):
    return {"name": name, "op": "attend", "dtype": dtype, "train": train, "B": B, "Lq": Lq, "Lk": Lk, "Hq": Hq, "Hk": Hk, "D": D,
            "mask": mask}


def listed():
    return [
        # one new token of four running sequences, far along: the smallest call, latency alone
        _rotate("rotate_token_bf16", "bf16", False, 4, 1, 1, 8, 2, 64, 1, 64, "halves", 200000),
        # training step at 1/16 of 640x192, batch 12, rows and columns as the two axes
        _rotate("rotate_sixteenth_f32_train", "f32", True, 12, 480, 960, 4, 4, 64, 2, 64, "halves", 0),
        # narrow odd heads (80 channels in 8 heads) at 1/8 of 1024x320: no wide load fits them
        _rotate("rotate_narrow_f32", "f32", False, 8, 5120, 10240, 8, 8, 10, 2, 8, "neighbours", 0),
        # training step at 1/4 of 640x192: the largest, bound by memory
        _rotate("rotate_quarter_bf16_train", "bf16", True, 12, 7680, 15360, 8, 8, 64, 2, 64, "halves", 0),
        # one query token of a sequence against the states of two frames, heads shared by four: latency and bandwidth
        _attend("attend_token_bf16", "bf16", False, 4, 1, 15360, 8, 2, 64, "none"),
        # a handful of queries against a long store of states, one length per sequence
        _attend("attend_few_f32", "f32", False, 2, 5, 40001, 6, 3, 80, "lens"),
        # training step at 1/32 of 640x192: the smallest level of the pyramid
        _attend("attend_coarse_f32_train", "f32", True, 12, 120, 240, 8, 8, 64, "none"),
        # training step at 1/16 with shared heads, a padded batch and invalid pixels
        _attend("attend_sixteenth_bf16_train", "bf16", True, 12, 480, 960, 8, 2, 32, "both"),
        # training step at 1/8 of 640x192 in the trainer's default type
        _attend("attend_eighth_f32_train", "f32", True, 12, 1920, 3840, 4, 4, 32, "none"),
        # odd lengths and heads of 28 channels (224 in 8), some pixels invalid, one sequence with no states at all
        _attend("attend_odd_f32", "f32", False, 3, 333, 1281, 8, 8, 28, "empty"),
        # inference at 1/4 of 640x192: the longest sequences
        _attend("attend_quarter_bf16", "bf16", False, 2, 7680, 15360, 4, 4, 64, "none"),
        # training step at 1/16 of 1024x320 with wide heads: bound by matrix products
        _attend("attend_wide_bf16_train", "bf16", True, 4, 1280, 2560, 8, 8, 128, "none"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def draw(rng):
    dtype, train = rng.choice(["f32", "bf16"]), rng.random() < 0.5
    Hk = rng.choice([1, 2, 3, 4, 8])
    Hq = Hk * rng.choice([1, 1, 2, 4])
    if rng.random() < 0.4:
        axes, D = rng.choice([1, 2, 3]), rng.choice([10, 16, 28, 32, 48, 64, 80, 96, 128])
        rot = rng.choice([D, D // 2]) // (2 * axes) * (2 * axes)
        while True:
            B, Lq, Lk = rng.randint(1, 12), _spread(rng, 1, 7680), _spread(rng, 1, 15360)
            if B * (Lq * Hq + Lk * Hk) * D <= 12 * 23040 * 8 * 64 // 4:
                return _unnamed(_rotate("", dtype, train, B, Lq, Lk, Hq, Hk, D, axes, rot, rng.choice(["halves", "neighbours"]),
                                        rng.choice([0, 1000, 300000])))
    D, mask = rng.choice([6, 16, 28, 32, 48, 64, 80, 96, 128]), rng.choice(["none", "lens", "mask", "both", "empty"])
    while True:
        # (one state alone has no gradient to compare: softmax of it is 1 whatever the query is)
        B, Lq = rng.randint(2 if mask == "empty" else 1, 12), _spread(rng, 1, 7680)
        Lk = _spread(rng, 8 if train or mask in ("mask", "both", "empty") else 1, 40000)
        if B * Hq * Lq * Lk <= 12 * 4 * 1920 * 3840 and B * Hq * Lq * Lk * D <= 12 * 4 * 1920 * 3840 * 32:
            return _unnamed(_attend("", dtype, train, B, Lq, Lk, Hq, Hk, D, mask))


# ------------------------------------------------------------------------------------------------ inputs
def _positions(L, axes, first, device):
    """Token positions: one running index, rows and columns of a grid, or frame, row and column of two frames."""
    i = torch.arange(L, device=device)
    if axes == 1:
        return (i + first)[:, None].int()
    width = max(1, int(math.sqrt(L * 3.2 / (axes - 1))))
    if axes == 2:
        return torch.stack([i // width + first, i % width], 1).int()
    half = -(-L // 2)
    return torch.stack([i // half, i % half // width + first, i % half % width], 1).int()


def _lengths(case):
    """States that each sequence has: the same numbers for every seed, so that the work is known."""
    B, Lk, kind = case["B"], case["Lk"], case["mask"]
    if kind in ("lens", "both"):
        return [max(1, Lk - (b * Lk) // (2 * B)) for b in range(B)]
    if kind == "empty":
        return [0 if b == B - 1 else max(1, Lk - (b * Lk) // (2 * B)) for b in range(B)]
    return [Lk] * B


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = TYPES[case["dtype"]]
    B, Lq, Lk, Hq, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "Hq", "Hk", "D"))

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=dev) * std).to(t)

    s = {"case": case}
    if case["op"] == "rotate":
        q, kv = normal(B, Lq, Hq * D, std=1.5), normal(B, Lk, 2 * Hk * D, std=1.5)      # the two projections, keys and values in one
        s["q"], s["k"] = q.view(B, Lq, Hq, D), kv[..., :Hk * D].unflatten(-1, (Hk, D))
        s["wq"], s["wk"] = (1.0 + 0.2 * torch.randn(D, generator=g, device=dev) for _ in range(2))
        s["pq"], s["pk"] = (_positions(n, case["axes"], case["first"], dev) for n in (Lq, Lk))
        leaves = ("q", "k", "wq", "wk")
        if case["train"]:
            s["gq"], s["gk"] = normal(B, Lq, Hq, D), normal(B, Lk, Hk, D)
    else:
        q, kv = normal(B, Lq, Hq * D), normal(B, Lk, 2 * Hk * D)
        s["q"] = q.view(B, Lq, Hq, D)
        s["k"], s["v"] = (kv[..., i * Hk * D:(i + 1) * Hk * D].unflatten(-1, (Hk, D)) for i in range(2))
        s["lens"] = s["valid"] = None
        if case["mask"] != "none" and case["mask"] != "mask":
            s["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
        if case["mask"] in ("mask", "both", "empty"):
            s["valid"] = torch.rand(B, Lk, generator=g, device=dev) > 0.125              # pixels that left the image
        leaves = ("q", "k", "v")
        if case["train"]:
            s["go"] = normal(B, Lq, Hq, D)
    if case["train"]:
        for n in leaves:
            s[n] = s[n].detach().requires_grad_(True)
        s["leaves"] = leaves
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_norm_rope(x, w, pos, axes, rot, pairs):
    n = x.float()
    n = n * torch.rsqrt((n * n).mean(-1, keepdim=True) + EPS) * w
    if rot == 0:
        return n.to(x.dtype)
    ra = rot // axes
    freq = BASE ** (-torch.arange(0, ra, 2, device=x.device, dtype=torch.float64) / ra)
    ang = pos.double()[:, :, None] * freq                                               # [L, axes, ra / 2]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]                     # [L, 1, axes, ra / 2]
    r = n[..., :rot].unflatten(-1, (axes, ra))
    if pairs == "halves":
        a, b = r[..., :ra // 2], r[..., ra // 2:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([r.flatten(-2), n[..., rot:]], -1).to(x.dtype)


def _allowed(lens, valid, B, Lk, device):
    m = None
    if lens is not None:
        m = torch.arange(Lk, device=device) < lens[:, None]
    if valid is not None:
        m = valid if m is None else m & valid
    return m


def _plain_attention(q, k, v, lens, valid):
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = Hq // Hk
    m = _allowed(lens, valid, B, Lk, q.device)
    kf, vf = k.float(), v.float()
    if m is not None:
        kf, vf = (x.masked_fill(~m[:, :, None, None], 0.0) for x in (kf, vf))
    qf = q.float().unflatten(2, (Hk, G)).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Lq, D)
    s = torch.matmul(qf, kf.permute(0, 2, 3, 1).contiguous()) * (1.0 / math.sqrt(D))
    if m is not None:
        s = s.masked_fill(~m[:, None, None, :], -math.inf)
    top = s.detach().amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, vf.permute(0, 2, 1, 3).contiguous()) / torch.where(total == 0, torch.ones_like(total), total)
    return o.view(B, Hk, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, Hq, D).to(q.dtype)


def run(s):
    c = s["case"]
    if c["op"] == "rotate":
        if own:
            from mono_vifi_amd import ops
            out = ops.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["pq"], s["pk"], rot_dim=c["rot"], base=BASE, eps=EPS,
                                   interleaved=c["pairs"] == "neighbours")
        else:
            out = [_plain_norm_rope(s[x], s["w" + x], s["p" + x], c["axes"], c["rot"], c["pairs"]) for x in ("q", "k")]
        if c["train"]:
            return [o.detach() for o in out] + list(torch.autograd.grad(list(out), [s[n] for n in s["leaves"]], [s["gq"], s["gk"]]))
        return list(out)
    if own:
        from mono_vifi_amd import ops
        o = ops.cross_attention(s["q"], s["k"], s["v"], key_mask=s["valid"], kv_lens=s["lens"])
    else:
        o = _plain_attention(s["q"], s["k"], s["v"], s["lens"], s["valid"])
    if c["train"]:
        return [o.detach()] + list(torch.autograd.grad(o, [s[n] for n in s["leaves"]], s["go"]))
    return [o]


# ------------------------------------------------------------------------------------------------ what cannot be done without
def work(case):
    B, Lq, Lk, Hq, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotate":
        n = B * (Lq * Hq + Lk * Hk) * D
        # in and out, and the two gradients of a training step; positions and the weights with their gradients once
        return {"bytes": n * size * (4 if case["train"] else 2) + 4 * case["axes"] * (Lq + Lk) + 8 * D * (2 if case["train"] else 1),
                "flops": n * (20 if case["train"] else 7)}
    states = sum(_lengths(case))
    # q and out, k and v of the states that count; with the four gradients in a training step (those of k and v whole)
    moved = 2 * B * Lq * Hq * D + 2 * states * Hk * D
    if case["train"]:
        moved += 2 * B * Lq * Hq * D + 2 * B * Lk * Hk * D
    extra = (B * Lk if case["mask"] in ("mask", "both", "empty") else 0) + 4 * B
    # two products forward, four more backward
    return {"bytes": moved * size + extra, "flops": (12 if case["train"] else 4) * Hq * Lq * states * D}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rotate(s, case) if case["op"] == "rotate" else _exact_attend(s, case)


def _exact_rotate(s, case):
    D, axes, rot = case["D"], case["axes"], case["rot"]
    ra = rot // axes

    def turn(x, pos, sign):
        """x with each pair (a, b) as the complex number a + ib multiplied by exp(i * sign * angle)."""
        y = x.clone()
        for a in range(axes):
            for j in range(ra // 2):
                lo, hi = (a * ra + j, a * ra + j + ra // 2) if case["pairs"] == "halves" else (a * ra + 2 * j, a * ra + 2 * j + 1)
                ang = pos[:, a].double() * BASE ** (-2.0 * j / ra)
                z = torch.complex(x[..., lo], x[..., hi]) * torch.polar(torch.ones_like(ang), sign * ang)[None, :, None]
                y[..., lo], y[..., hi] = z.real, z.imag
        return y

    outs, grads, wgrads = [], [], []
    with torch.no_grad():
        for n in ("q", "k"):
            x, w, pos = s[n].double(), s["w" + n].double(), s["p" + n]
            inv = (x.square().sum(-1, keepdim=True) / D + EPS).pow(-0.5)
            outs.append(turn(x * inv * w, pos, 1.0))
            if case["train"]:
                u = turn(s["g" + n].double(), pos, -1.0)              # the gradient of the normed, weighted row
                wgrads.append((u * x * inv).sum((0, 1, 2)))
                h = u * w
                grads.append(inv * h - x * inv.pow(3) * (h * x).sum(-1, keepdim=True) / D)
    return outs + grads + wgrads


def _exact_attend(s, case):
    B, Lq, Lk, Hq, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    G, scale = Hq // Hk, 1.0 / math.sqrt(D)
    lens = _lengths(case)
    with torch.no_grad():
        q, k, v = (s[n].double() for n in ("q", "k", "v"))
        o = torch.zeros_like(q)
        go = s["go"].double() if case["train"] else None
        dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v)) if case["train"] else (None, None, None)
        for b in range(B):
            keep = torch.arange(lens[b], device=q.device)
            if s["valid"] is not None:
                keep = keep[s["valid"][b, :lens[b]]]
            if keep.numel() == 0:
                continue
            for h in range(Hq):
                kh, vh = k[b, keep, h // G], v[b, keep, h // G]
                for i in range(0, Lq, 2048):
                    r = slice(i, i + 2048)
                    p = torch.softmax(q[b, r, h] @ kh.T * scale, -1)
                    o[b, r, h] = p @ vh
                    if case["train"]:
                        dp = go[b, r, h] @ vh.T
                        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                        dq[b, r, h] = ds @ kh
                        dk[b, :, h // G].index_add_(0, keep, ds.T @ q[b, r, h])
                        dv[b, :, h // G].index_add_(0, keep, p.T @ go[b, r, h])
    return [o, dq, dk, dv] if case["train"] else [o]
