"""Cross attention and the query / key norm with position rotation against plain implementations in 64 bits.

Tolerances are derived, per element.  u = 2^-24 is the rounding of fp32; an output in bf16 is off by at most 2^-8 of itself,
and so is what the kernels hold in bf16 between two products (P and dS).  fp32 products run as six of bf16 planes cut to 8 + 8
+ 8 bits: what is left out of a product ab is below 2^-21 |ab| (two terms of 2^-7 * 2^-15, and a smaller one).  A sum of n terms
in fp32 is off by at most n u times the sum of their magnitudes.  Every bound below is the propagation of these through the
formula, evaluated in 64 bits on the same inputs."""
import ctypes as C
import math

import pytest
import torch

import mono_vifi_amd  # noqa: F401
from mono_vifi_amd import _native as nat
from mono_vifi_amd import ops

gpu = pytest.mark.gpu
U = 2.0 ** -24


# ------------------------------------------------------------------------------------------------ attention: 64-bit reference
def attention_ref(q, k, v, scale, allowed, go=None):
    """(out, bound of its error[, dq, dk, dv and their bounds]); allowed [B, Lk] bool or None.  All on q's device in 64 bits."""
    bf16 = q.dtype == torch.bfloat16
    uo = 2.0 ** -8 if bf16 else U                       # rounding of an output
    up = 2.0 ** -8 if bf16 else 2.0 ** -21              # P and dS as operands of a product
    um = 0.0 if bf16 else 2.0 ** -21                    # the other products
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = Hq // Hk
    q, k, v = (x.detach().double() for x in (q, k, v))
    if allowed is not None:
        k, v = (x.masked_fill(~allowed[:, :, None, None], 0.0) for x in (k, v))
    kh, vh = (x.permute(0, 2, 1, 3).repeat_interleave(G, 1) for x in (k, v))           # [B, Hq, Lk, D]
    qh = q.permute(0, 2, 1, 3)
    s = qh @ kh.transpose(-1, -2).contiguous() * scale
    size = qh.abs() @ kh.abs().transpose(-1, -2).contiguous() * scale                  # sum of |q||k|
    if allowed is not None:
        s = s.masked_fill(~allowed[:, None, None, :], -math.inf)
        size = size.masked_fill(~allowed[:, None, None, :], 0.0)
    if Lk == 0:
        p = torch.zeros_like(s)
    else:
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    o = p @ vh
    big = size.amax(-1, keepdim=True) if Lk else torch.zeros_like(o[..., :1])
    # a probability: scores off by (um + (D + 16) u) * size, in numerator and sum; the exponent's own rounding; the sum over Lk
    rel = 2 * (um + (D + 16) * U) * big + 8 * U * big + (Lk + 64) * U
    to = (up + rel) * (p @ vh.abs()) + uo * o.abs()
    back = lambda x: x.permute(0, 2, 1, 3)  # noqa: E731
    if go is None:
        return back(o), back(to)
    g = go.double().permute(0, 2, 1, 3)
    dp = g @ vh.transpose(-1, -2).contiguous()
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    edp = (um + (D + 16) * U) * (g.abs() @ vh.abs().transpose(-1, -2).contiguous())
    edelta = (g.abs() * to).sum(-1, keepdim=True) + (D + 16) * U * (g.abs() * o.abs()).sum(-1, keepdim=True)
    eds = ds.abs() * (up + rel) + p * (edp + edelta)
    dq = ds @ kh * scale
    tq = scale * ((eds + (Lk + 64) * U * ds.abs()) @ kh.abs()) + uo * dq.abs()
    R = Lq * G
    dsT, pT = ds.transpose(-1, -2).contiguous(), p.transpose(-1, -2).contiguous()
    fold = lambda x: x.unflatten(1, (Hk, G)).sum(2)  # noqa: E731
    dk, dv = fold(dsT @ qh) * scale, fold(pT @ g)
    tk = scale * fold((eds + (R + 64) * U * ds.abs()).transpose(-1, -2).contiguous() @ qh.abs()) + uo * dk.abs()
    tv = fold(((up + rel + (R + 64) * U) * p).transpose(-1, -2).contiguous() @ g.abs()) + uo * dv.abs()
    return [back(x) for x in (o, to, dq, tq, dk, tk, dv, tv)]


def near(got, want, tol, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not got.numel():
        return
    e = (got.double() - want).abs() - tol
    finite, over, at = bool(torch.isfinite(got).all()), float(e.max()), float(tol.flatten()[e.argmax()])
    assert finite, f"{what}: not finite"
    assert over <= 1e-30, f"{what}: error exceeds its bound by {over:.3e} (bound there {at:.3e})"


def make(seed, dtype, B, Lq, Lk, Hq, Hk, D, spread=1.0, strided=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(*shape):
        return (torch.randn(shape, generator=g, device="cuda") * spread).to(dtype)
    if strided:                                           # one projection for keys and values, heads in front of tokens for queries
        q = t(B, Hq, Lq, D + 3)[..., 1:1 + D].permute(0, 2, 1, 3)
        kv = t(B, Lk, 2, Hk, D)
        k, v = kv[:, :, 0], kv[:, :, 1]
    else:
        q, k, v = t(B, Lq, Hq, D), t(B, Lk, Hk, D), t(B, Lk, Hk, D)
    return q, k, v, t(B, Lq, Hq, D)


def check_attention(q, k, v, go, key_mask=None, kv_lens=None, scale=None, train=True):
    B, Lk = k.shape[:2]
    allowed = None
    if kv_lens is not None:
        allowed = torch.arange(Lk, device=q.device) < kv_lens[:, None]
    if key_mask is not None:
        allowed = key_mask.bool() if allowed is None else allowed & key_mask.bool()
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    ref = attention_ref(q, k, v, sc, allowed, go if train else None)
    if not train:
        out = ops.cross_attention(q, k, v, scale=scale, key_mask=key_mask, kv_lens=kv_lens)
        near(out, *ref, "out")
        return out
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = ops.cross_attention(*leaves, scale=scale, key_mask=key_mask, kv_lens=kv_lens)
    grads = torch.autograd.grad(out, leaves, go)
    near(out.detach(), *ref[:2], "out")
    for i, n in enumerate(("dq", "dk", "dv")):
        near(grads[i], ref[2 + 2 * i], ref[3 + 2 * i], n)
    if allowed is not None:
        for gr in grads[1:]:
            assert not gr[~allowed].any(), "a state that does not count has a gradient"
        empty = ~allowed.any(1)
        assert not out[empty].any() and not grads[0][empty].any()
    return out, grads


SHAPES = [  # B, Lq, Lk, Hq, Hk, D
    (1, 1, 1, 1, 1, 1), (2, 1, 7, 4, 1, 6), (1, 31, 33, 2, 2, 28), (2, 33, 64, 3, 3, 32), (2, 129, 65, 4, 2, 40),
    (1, 5, 257, 6, 3, 64), (1, 200, 130, 2, 1, 80), (1, 64, 96, 1, 1, 96), (1, 130, 161, 2, 2, 100), (1, 97, 140, 2, 1, 128),
    (3, 120, 240, 8, 8, 64)]
DTYPES = [torch.float32, torch.bfloat16]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_and_gradients(dtype, shape):
    check_attention(*make(1, dtype, *shape))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(3, 33, 150, 4, 2, 28), (4, 40, 200, 2, 2, 64), (2, 3, 2500, 4, 1, 80)], ids=str)
@pytest.mark.parametrize("kind", ["lens", "mask", "both"])
def test_masked_states_and_empty_rows(dtype, shape, kind):
    """Garbage (NaN, infinities, the type's lowest value) in states that do not count; one sequence with none at all."""
    q, k, v, go = make(2, dtype, *shape)
    B, Lk = k.shape[:2]
    g = torch.Generator(device="cuda").manual_seed(3)
    lens = mask = None
    allowed = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
    if kind in ("lens", "both"):
        lens = torch.tensor([Lk - 1 - 37 * b for b in range(B - 1)] + [0], dtype=torch.int32, device="cuda")
        allowed &= torch.arange(Lk, device="cuda") < lens[:, None]
    if kind in ("mask", "both"):
        mask = torch.rand(B, Lk, generator=g, device="cuda") > 0.4
        mask[0, :70] = False                              # a whole tile of states, and the first
        mask[B - 1] = False
        allowed &= mask
    for i, bad in enumerate((math.nan, math.inf, -math.inf, torch.finfo(dtype).min)):
        at = ~allowed & (torch.arange(Lk, device="cuda") % 4 == i)
        k[at], v[at] = bad, bad
    check_attention(q, k, v, go, mask, lens)
    check_attention(q, k, v, go, mask, lens, train=False)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 70, 90, 4, 2, 64), (1, 40, 75, 2, 2, 27), (2, 1, 300, 3, 1, 32)], ids=str)
def test_strides(dtype, shape):
    q, k, v, go = make(4, dtype, *shape, strided=True)
    check_attention(q, k, v, go)
    mask = torch.rand(k.shape[1], k.shape[0], device="cuda").t() > 0.3                  # a transposed mask
    check_attention(q, k, v, go, mask.to(torch.uint8))
    # a gradient that is expanded, and states shared by the sequences of a batch
    one = k[:1].detach().requires_grad_(True)
    out = ops.cross_attention(q, one.expand(k.shape), v)
    (gk,) = torch.autograd.grad(out, one, torch.ones((), dtype=dtype, device="cuda").expand(out.shape))
    full = check_attention(q, k[:1].expand(k.shape), v, torch.ones_like(q))[1][1]
    assert torch.equal(gk, full.sum(0, keepdim=True))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 90, 200, 4, 2, 28), (2, 40, 130, 6, 2, 64), (1, 33, 70, 4, 4, 128), (2, 3, 300, 4, 2, 100)], ids=str)
def test_packed_projections(dtype, shape):
    """Keys and values as halves of one projection (16-byte loads with strides), with a mask and lengths."""
    B, Lq, Lk, Hq, Hk, D = shape
    q, _, _, go = make(16, dtype, *shape)
    kv = make(17, dtype, B, Lk, 1, 2 * Hk, 1, D)[0]
    mask = torch.rand(B, Lk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(18)) > 0.3
    lens = torch.tensor([Lk - 5] * B, dtype=torch.int32, device="cuda")
    check_attention(q, kv[:, :, :Hk], kv[:, :, Hk:], go, mask, lens)


@gpu
@pytest.mark.parametrize("stride", [1 << 22, 1 << 25], ids=["wide", "narrow"])
def test_states_far_apart(stride):
    """States whose byte offsets pass 32 bits, within the reach of a tile's 32-bit offsets (2^22 elements a state) and beyond it."""
    Lk = (1 << 33) // (2 * stride) + 9                                       # a little over 8 GiB of bf16
    q, k0, v0, go = make(19, torch.bfloat16, 1, 40, Lk, 1, 1, 64)
    store = torch.empty(Lk * stride, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.as_strided(store, (1, Lk, 1, 64), (0, stride, 64, 1), 64 * i) for i in range(2))
    k.copy_(k0)
    v.copy_(v0)
    check_attention(q, k, v, go)
    check_attention(q[:, :1], k, v, go[:, :1])


@gpu
def test_saved_tensors_may_travel():
    """Saved-tensor hooks: what the backward unpacks lies elsewhere, with other strides."""
    q, k, v, go = make(20, torch.float32, 2, 40, 70, 4, 2, 32, strided=True)
    w = torch.linspace(0.5, 1.5, 32, device="cuda")
    pos = positions(20, 40, 1)

    def grads():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, w)]
        out = ops.cross_attention(ops.qk_norm_rope(leaves[0], None, leaves[3], q_pos=pos), leaves[1], leaves[2])
        return torch.autograd.grad(out, leaves, go)
    want = grads()
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    # (packed keys become contiguous: the same products by other loads)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 9000, 8, 2, 64), (2, 4, 5001, 4, 4, 80), (1, 9000, 3, 2, 1, 32), (1, 3000, 40, 2, 2, 128),
                                   (1, 7, 700, 4, 2, 128), (1, 16, 333, 4, 2, 100), (3, 2, 130, 2, 2, 27)], ids=str)
def test_few_queries_and_few_states(dtype, shape):
    """The axis that is split over the chip and joined: states for few queries, rows for few states."""
    check_attention(*make(5, dtype, *shape))
    B, Lk = shape[0], shape[2]
    check_attention(*make(6, dtype, *shape), kv_lens=torch.tensor([Lk // 2 + 1] * B, device="cuda"))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 600, 700, 2, 2, 27), (2, 700, 600, 2, 1, 64), (2, 300, 1300, 1, 1, 96), (2, 1500, 300, 4, 4, 40)], ids=str)
def test_a_few_parts_of_which_some_hold_nothing(dtype, shape):
    """Two to eight parts of the states and of the rows; lengths that end in the first part, at once, or nowhere."""
    q, k, v, go = make(96, dtype, *shape)
    check_attention(q, k, v, go)
    for lens in ([130, 0], [shape[2], 65]):
        check_attention(q, k, v, go, kv_lens=torch.tensor(lens, device="cuda"))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 1, 700, 16, 1, 128), (1, 17, 900, 1, 1, 96), (2, 4, 1000, 8, 2, 48), (1, 5, 333, 9, 3, 27), (1, 11, 515, 3, 1, 128),
                                   (3, 2, 257, 8, 8, 30), (1, 31, 65, 2, 2, 57), (1, 33, 65, 2, 2, 64), (2, 3, 31, 5, 1, 100), (1, 1, 1, 1, 1, 1)], ids=str)
@pytest.mark.parametrize("masked", [False, True], ids=["all", "masked"])
def test_rows_that_fill_a_product_or_not(dtype, shape, masked):
    """1 .. 33 rows against every width of the tiles: the forms for at most 16 and at most 32 rows and the next one."""
    B, _, Lk = shape[:3]
    q, k, v, _ = make(97, dtype, *shape)
    kw = {}
    if masked:
        g = torch.Generator(device="cuda").manual_seed(98)
        kw = dict(key_mask=torch.rand(B, Lk, device="cuda", generator=g) < 0.3,
                  kv_lens=torch.randint(0, Lk + 1, (B,), device="cuda", generator=g))
    check_attention(q, k, v, None, train=False, **kw)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_scores_of_any_size(dtype):
    """Running maximum: scores rise along the states, fall, and one of them outweighs all (spread 12: scores of +-1,000)."""
    q, k, v, go = make(7, dtype, 1, 50, 300, 2, 2, 32)
    ramp = torch.linspace(0.0, 4.0, 300, device="cuda").to(dtype)[None, :, None, None]
    check_attention(q, k * ramp, v, go)
    check_attention(q, k * ramp.flip(1), v, go)
    check_attention(q * 12, k * 12, v, go, train=False)
    check_attention(q, k, v, go, scale=1e-3)
    check_attention(q, k, v, go, scale=2.5)


@gpu
def test_nothing_to_do():
    for dtype in DTYPES:
        q, k, v, go = make(8, dtype, 2, 5, 0, 2, 1, 16)
        out, grads = check_attention(q, k, v, go)
        assert not out.any() and not grads[0].any()
        q, k, v, go = make(8, dtype, 2, 0, 9, 2, 1, 16)
        out, grads = check_attention(q, k, v, go)
        assert out.shape == (2, 0, 2, 16) and not grads[1].any() and not grads[2].any()
        q, k, v, go = make(8, dtype, 0, 4, 9, 2, 1, 16)
        assert ops.cross_attention(q, k, v).shape == (0, 4, 2, 16)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_nan_reaches_only_its_rows(dtype):
    """A NaN query makes its own row NaN; an infinite value of a state that counts makes that channel of every query infinite or
    NaN (in fp32 an infinity meets the empty lower planes of a probability: inf * 0), and no other."""
    q, k, v, _ = make(9, dtype, 2, 40, 70, 2, 2, 32)
    q[1, 3, 0, 5] = math.nan
    out = ops.cross_attention(q, k, v)
    bad = torch.isnan(out)
    assert bad[1, 3, 0].all() and int(bad.sum()) == 32
    q, k, v, _ = make(9, dtype, 2, 40, 70, 2, 2, 32)
    v[0, 69, 1, 7] = math.inf
    out = ops.cross_attention(q, k, v)
    assert not torch.isfinite(out[0, :, 1, 7]).any() and int((~torch.isfinite(out)).sum()) == 40


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_runs_repeat_bit_for_bit(dtype):
    for shape in ((2, 1, 3000, 4, 2, 64), (2, 200, 300, 4, 2, 32)):
        q, k, v, go = make(10, dtype, *shape)
        leaves = [x.requires_grad_(True) for x in (q, k, v)]
        runs = []
        for _ in range(3):
            out = ops.cross_attention(*leaves)
            runs.append([out.detach()] + list(torch.autograd.grad(out, leaves, go)))
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@gpu
def test_gradient_against_differences():
    """Central differences of the 64-bit formula along random directions: dq, dk, dv are the gradient of what the forward computes."""
    q, k, v, go = make(11, torch.float32, 1, 12, 20, 2, 1, 16)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    grads = torch.autograd.grad(ops.cross_attention(*leaves), leaves, go)
    g = torch.Generator(device="cuda").manual_seed(12)

    def f(args):
        s = torch.einsum("bihd,bjd->bhij", args[0], args[1][:, :, 0]) * 0.25
        return float((torch.einsum("bhij,bjd->bihd", torch.softmax(s, -1), args[2][:, :, 0]) * go.double()).sum())
    for i in range(3):
        base = [x.detach().double() for x in leaves]
        d = torch.randn(base[i].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-4
        lo, hi = list(base), list(base)
        lo[i], hi[i] = base[i] - h * d, base[i] + h * d
        want, got = (f(hi) - f(lo)) / (2 * h), float((grads[i].double() * d).sum())
        # differences: h^2 times a third derivative of order one per channel; the gradient: fp32
        assert abs(want - got) <= 1e-4 * max(1.0, float((grads[i].double().abs() * d.abs()).sum()))


@gpu
def test_only_the_gradients_that_are_asked_for():
    q, k, v, go = make(13, torch.float32, 2, 30, 50, 2, 2, 32)
    _, grads = check_attention(q, k, v, go)
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        leaves = [x.detach().requires_grad_(n) for x, n in zip((q, k, v), need)]
        out = ops.cross_attention(*leaves)
        out.backward(go)
        for x, n, want in zip(leaves, need, grads):
            assert (x.grad is not None) == n
            if n:
                assert torch.equal(x.grad, want)
    x = q.detach().requires_grad_(True)
    for out in (ops.cross_attention(x, k, v), ops.qk_norm_rope(x)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(out, x, go, create_graph=True)


@gpu
def test_changed_inputs_are_noticed_before_the_backward():
    q, k, v, go = make(14, torch.float32, 2, 30, 50, 2, 2, 32)
    lens = torch.tensor([50, 20], dtype=torch.int32, device="cuda")
    x = q.requires_grad_(True)
    out = ops.cross_attention(x, k, v, kv_lens=lens)
    lens.fill_(10)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(go)


@gpu
def test_lengths_outside_the_states_are_clamped():
    q, k, v, _ = make(15, torch.float32, 3, 20, 50, 2, 2, 32)
    for t in (torch.int32, torch.int64):
        lens = torch.tensor([-5, 50, 1 << 30], dtype=t, device="cuda")
        out = ops.cross_attention(q, k, v, kv_lens=lens)
        assert torch.equal(out[1:], ops.cross_attention(q[1:], k[1:], v[1:])) and not out[0].any()
    lens = torch.tensor([1 << 40, 3, 1 << 33], dtype=torch.int64, device="cuda")
    want = ops.cross_attention(q, k, v, kv_lens=torch.tensor([50, 3, 50], dtype=torch.int32, device="cuda"))
    assert torch.equal(ops.cross_attention(q, k, v, kv_lens=lens), want)


# ------------------------------------------------------------------------------------------------ norm and rotation
def rotate_ref(x, w, pos, axes, rot, base, eps, interleaved, dy=None):
    """(y, bound[, dx, bound, dw, bound]) in 64 bits."""
    uo = 2.0 ** -8 if x.dtype == torch.bfloat16 else U
    B, L, H, D = x.shape
    x = x.detach().double()
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    ra = rot // axes
    pairs = [(a * ra + j, a * ra + j + ra // 2) if not interleaved else (a * ra + 2 * j, a * ra + 2 * j + 1)
             for a in range(axes) for j in range(ra // 2)]
    where = [(a, j) for a in range(axes) for j in range(ra // 2)]

    def turn(t, sign, spread=False):
        y = t.clone()
        if pos is None:
            return y.abs() if spread else y
        p = pos if pos.dim() == 3 else pos[None]
        for (lo, hi), (a, j) in zip(pairs, where):
            ang = sign * p[..., a].double() * base ** (-2.0 * j / ra)
            c, s = ang.cos()[..., None], ang.sin()[..., None]
            if spread:                                    # |a| + |b|: what the errors of sine and cosine multiply
                y[..., lo] = y[..., hi] = t[..., lo].abs() + t[..., hi].abs()
            else:
                y[..., lo], y[..., hi] = t[..., lo] * c - t[..., hi] * s, t[..., lo] * s + t[..., hi] * c
        return y.abs() if spread else y
    r = ((x * x).mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r * w
    y = turn(n, 1.0)
    # sine and cosine: argument off by 2 u of at most pi / 4, polynomials by 2 u; the norm by (D / 2 + 8) u
    ty = (D + 24) * U * turn(n, 1.0, True) + uo * y.abs()
    if dy is None:
        return y, ty
    g = dy.double()
    u, au = turn(g, -1.0), turn(g, -1.0, True)
    d = (u * w * x).sum(-1, keepdim=True)
    ad = (au * w.abs() * x.abs()).sum(-1, keepdim=True)
    dx = r * w * u - x * r ** 3 / D * d
    tx = (3 * D + 48) * U * (r * w.abs() * au + x.abs() * r ** 3 / D * ad) + uo * dx.abs()
    dw = (u * x * r).sum((0, 1, 2))
    tw = (B * L * H + D + 48) * U * (au * x.abs() * r).sum((0, 1, 2))
    return y, ty, dx, tx, dw, tw


def check_rotate(q, k, wq, wk, pq, pk, rot, base=10000.0, eps=1e-6, interleaved=False, seed=0):
    axes = next((p.shape[-1] if p.dim() > 1 else 1 for p in (pq, pk) if p is not None), 1)
    sides = [("q", q, wq, pq)] + ([("k", k, wk, pk)] if k is not None else [])
    g = torch.Generator(device="cuda").manual_seed(seed)
    leaves = [None if x is None else x.detach().requires_grad_(True) for x in (q, k, wq, wk)]
    out = ops.qk_norm_rope(*leaves, pq, pk, rot_dim=rot, base=base, eps=eps, interleaved=interleaved)
    outs = [out] if k is None else list(out)
    dys = [torch.randn(o.shape, generator=g, device="cuda").to(o.dtype) for o in outs]
    live = [x for x in leaves if x is not None]
    grads = dict(zip([id(x) for x in live], torch.autograd.grad(outs, live, dys)))
    with torch.no_grad():
        again = ops.qk_norm_rope(q, k, wq, wk, pq, pk, rot_dim=rot, base=base, eps=eps, interleaved=interleaved)
    for i, (n, x, w, p) in enumerate(sides):
        p = p[:, None] if p is not None and p.dim() == 1 else p
        ref = rotate_ref(x, w, p, axes, rot, base, eps, interleaved, dys[i])
        near(outs[i].detach(), ref[0], ref[1], n)
        assert torch.equal(outs[i], again if k is None else again[i])
        near(grads[id(leaves[i])], ref[2], ref[3], "d" + n)
        if w is not None:
            assert grads[id(leaves[2 + i])].dtype == w.dtype
            near(grads[id(leaves[2 + i])], ref[4], ref[5] + (2.0 ** -8 * ref[4].abs() if w.dtype == torch.bfloat16 else 0), "dw" + n)
    return outs, grads


def rows(seed, dtype, B, L, H, D, strided=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if strided:
        return (1.5 * torch.randn(B, H, 2, L, D, generator=g, device="cuda")).to(dtype)[:, :, 1].permute(0, 2, 1, 3)
    return (1.5 * torch.randn(B, L, H, D, generator=g, device="cuda")).to(dtype)


def positions(seed, L, axes, far=1000, batch=None, dtype=torch.int32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (L, axes) if batch is None else (batch, L, axes)
    return torch.randint(-far, far, shape, generator=g, device="cuda", dtype=dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("case", [  # B, Lq, Lk, Hq, Hk, D, axes, rot
    (1, 1, 1, 1, 1, 2, 1, 2), (2, 3, 5, 4, 2, 64, 1, 64), (2, 17, 33, 8, 8, 64, 2, 64), (1, 40, 9, 3, 1, 10, 2, 8),
    (2, 11, 20, 6, 3, 96, 3, 96), (1, 7, 13, 2, 2, 128, 1, 64), (2, 30, 31, 5, 5, 27, 3, 24), (1, 9, 4, 2, 1, 80, 2, 48),
    (1, 6, 8, 1, 1, 1, 1, 0), (3, 100, 200, 9, 2, 32, 2, 32), (1, 5, 5, 3, 3, 48, 1, 0)], ids=str)
def test_norm_and_rotation(dtype, interleaved, case):
    B, Lq, Lk, Hq, Hk, D, axes, rot = case
    g = torch.Generator(device="cuda").manual_seed(21)
    wq, wk = (1 + 0.3 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    for strided in (False, True):
        q, k = rows(22, dtype, B, Lq, Hq, D, strided), rows(23, dtype, B, Lk, Hk, D, strided)
        check_rotate(q, k, wq, wk, positions(24, Lq, axes), positions(25, Lk, axes, batch=B), rot, interleaved=interleaved)
    check_rotate(q, None, wq, None, positions(24, Lq, axes, batch=B), None, rot, interleaved=interleaved)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_rotation_options(dtype):
    q, k = rows(31, dtype, 2, 12, 4, 64), rows(32, dtype, 2, 20, 2, 64)
    w = torch.linspace(0.5, 1.5, 64, device="cuda")
    check_rotate(q, k, None, None, None, None, 64)                                                    # the norm alone
    check_rotate(q, k, w, None, None, positions(33, 20, 2), 64)                                       # one side without positions
    check_rotate(q, k, None, w.to(dtype), positions(33, 12, 1), positions(34, 20, 1, dtype=torch.int64), 32, base=100.0, eps=1e-3)
    check_rotate(q[..., :50], k[..., 14:], w[:50], w[1:51], positions(33, 12, 1)[:, 0], positions(34, 20, 1)[:, 0], 50)      # unaligned
    y = ops.qk_norm_rope(q.transpose(1, 3).contiguous().transpose(1, 3), k, w, w, positions(33, 12, 2), positions(34, 20, 2))
    z = ops.qk_norm_rope(q, k, w, w, positions(33, 12, 2), positions(34, 20, 2), rot_dim=64)          # channels not adjacent: copied
    assert torch.equal(y[0], z[0]) and torch.equal(y[1], z[1])


@gpu
@pytest.mark.parametrize("far", [300_000, 2 ** 31 - 1, 2 ** 40])
def test_far_positions_keep_their_angles(far):
    """The angle of a position is exact modulo a turn: 2^-53 far is what the frequencies' own rounding leaves (64-bit floats, also
    in the reference), below an fp32 step up to 2^28 turns."""
    dtype = torch.int64 if far > 2 ** 31 else torch.int32
    q = rows(41, torch.float32, 1, 64, 2, 32)
    pos = positions(42, 64, 1, far=far, dtype=dtype)
    y = ops.qk_norm_rope(q, q_pos=pos)
    want, tol = rotate_ref(q, None, pos, 1, 32, 10000.0, 1e-6, False)
    n = q.double() * ((q.double() ** 2).mean(-1, keepdim=True) + 1e-6).rsqrt()
    near(y, want, tol + 4 * far * 2.0 ** -53 * n.abs().amax(-1, keepdim=True), "y")


@gpu
def test_zero_rows_and_empty_calls():
    for dtype in DTYPES:
        q = torch.zeros(2, 3, 2, 32, dtype=dtype, device="cuda")
        check_rotate(q, q.clone(), None, None, positions(1, 3, 1), positions(2, 3, 1), 32)
        w = torch.ones(32, device="cuda", requires_grad=True)
        x = q[:, :0].clone().requires_grad_(True)
        y = ops.qk_norm_rope(x, None, w, q_pos=positions(1, 3, 1)[:0])
        gx, gw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
        assert gx.shape == x.shape and not gw.any()
        a, b = ops.qk_norm_rope(q[:, :0], q, w, w, positions(1, 3, 1)[:0], positions(1, 3, 1))
        assert a.shape == (2, 0, 2, 32) and not b.any()


@gpu
def test_rotated_products_depend_on_the_distance_alone():
    """<R(i) q, R(j) k> is a function of i - j: what the rotation is for."""
    q, k = rows(51, torch.float32, 1, 1, 1, 64), rows(52, torch.float32, 1, 1, 1, 64)
    dots = []
    for off in (0, 5, 1234, 70000):
        p = torch.tensor([[7 + off]], dtype=torch.int32, device="cuda")
        r = torch.tensor([[2 + off]], dtype=torch.int32, device="cuda")
        a, b = ops.qk_norm_rope(q, k, q_pos=p, k_pos=r)
        dots.append(float((a.double() * b.double()).sum()))
    # two rotations of 64 channels, each off by at most (D + 24) u of a pair; |q'||k'| = 64
    assert max(dots) - min(dots) <= 2 * 2 * 88 * U * 64


# ------------------------------------------------------------------------------------------------ both, as they are used
@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_a_run_of_both(dtype):
    """Normed, rotated queries and keys into the attention, forward and backward in one graph, against autograd of the formulas in
    64 bits.  Bound: relative 2-norm, 5 roundings of the type along the chain (normed q and k, P, dS, output and gradient), and for
    fp32 a hundred of its roundings."""
    B, Lq, Lk, H, Hk, D = 2, 60, 130, 4, 2, 32
    q, kv = rows(61, dtype, B, Lq, H, D), rows(62, dtype, B, Lk, 2 * Hk, D)
    wq, wk = (1 + 0.2 * torch.randn(D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(s)) for s in (63, 64))
    pq, pk = positions(65, Lq, 2), positions(66, Lk, 2)
    lens = torch.tensor([Lk, 77], dtype=torch.int32, device="cuda")
    go = rows(67, dtype, B, Lq, H, D)
    leaves = [x.requires_grad_(True) for x in (q, kv, wq, wk)]
    a, b = ops.qk_norm_rope(leaves[0], leaves[1][:, :, :Hk], wq, wk, pq, pk)
    out = ops.cross_attention(a, b, leaves[1][:, :, Hk:], kv_lens=lens)
    got = [out] + list(torch.autograd.grad(out, leaves, go))

    ref = [x.detach().double().requires_grad_(True) for x in leaves]

    def norm_rope(x, w, pos):
        n = x * ((x * x).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        parts = []
        for ax in range(2):
            lo, hi = n[..., 16 * ax:16 * ax + 8], n[..., 16 * ax + 8:16 * ax + 16]
            ang = (pos[:, ax, None].double() * 10000.0 ** (-torch.arange(0, 16, 2, device="cuda", dtype=torch.float64) / 16))[:, None]
            parts += [lo * ang.cos() - hi * ang.sin(), lo * ang.sin() + hi * ang.cos()]
        return torch.cat(parts, -1)
    qr, kr = norm_rope(ref[0], ref[2], pq), norm_rope(ref[1][:, :, :Hk], ref[3], pk)
    kr, vr = (x.repeat_interleave(2, 2).permute(0, 2, 1, 3) for x in (kr, ref[1][:, :, Hk:]))
    s = qr.permute(0, 2, 1, 3) @ kr.transpose(-1, -2) * D ** -0.5
    s = s.masked_fill(~(torch.arange(Lk, device="cuda") < lens[:, None])[:, None, None, :], -math.inf)
    want = (torch.softmax(s, -1) @ vr).permute(0, 2, 1, 3)
    wants = [want] + list(torch.autograd.grad(want, ref, go.double()))
    tol = 5 * 2.0 ** -8 if dtype == torch.bfloat16 else 100 * U
    for g, w in zip(got, wants):
        assert float((g.double() - w).norm()) <= tol * float(w.norm())


@gpu
def test_on_another_stream():
    q, k, v, go = make(71, torch.float32, 2, 40, 3000, 4, 2, 64)
    pos = positions(72, 40, 1)
    want = check_attention(ops.qk_norm_rope(q, q_pos=pos), k, v, go)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        leaves = [x.detach().requires_grad_(True) for x in (ops.qk_norm_rope(q, q_pos=pos), k, v)]
        out = ops.cross_attention(*leaves)
        grads = torch.autograd.grad(out, leaves, go)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want[1]))


@gpu
def test_two_captured_graphs_replay():
    """Two graphs (a split and an unsplit shape, forward and backward) replayed in turn with eager calls between: every replay
    gives the eager bits, also after the inputs changed in place."""
    state = []
    for seed, shape in ((81, (1, 2, 4000, 4, 2, 64)), (82, (2, 90, 130, 4, 2, 32))):
        q, k, v, go = make(seed, torch.float32, *shape)
        state.append([x.requires_grad_(True) for x in (q, k, v)] + [go, positions(seed, shape[1], 1)])

    def step(q, k, v, go, pos):
        out = ops.cross_attention(ops.qk_norm_rope(q, q_pos=pos), k, v)
        return [out] + list(torch.autograd.grad(out, [q, k, v], go))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for st in state:
            step(*st)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for st in state:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(*st)
        graphs.append((g, outs))
    for turn in range(4):
        for (g, outs), st in zip(graphs, state):
            with torch.no_grad():
                for x in st[:3]:
                    x.mul_(0.9)
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, step(*st)):
                assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("which", ["attention", "norm"])
def test_a_captured_backward_refuses_leaves_of_a_living_eager_graph(which):
    """The eager graph's accumulation nodes sit on the default stream, which cannot join a capture: an error, before the engine gets
    there.  Without the eager graph the same capture runs and replays."""
    q, k, v, go = make(91, torch.float32, 1, 5, 40, 2, 2, 32)
    w = torch.ones(32, device="cuda")
    leaves = [x.requires_grad_(True) for x in ((q, k, v) if which == "attention" else (q, w))]

    def call():
        return ops.cross_attention(q, k, v) if which == "attention" else ops.qk_norm_rope(q, None, w)
    eager = call()
    want = [x.clone() for x in torch.autograd.grad(eager, leaves, go, retain_graph=True)]
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(g):
            torch.autograd.grad(call(), leaves, go)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(eager, leaves, go), want))
    del eager
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(call(), leaves, go)
    for _ in range(3):
        for x in got:
            x.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ the modules that use them
def layer_ref(m, x, states, xp, sp, allowed):
    """layers.CrossAttention in 64 bits from its parameters."""
    P = {n: p.detach().double().requires_grad_(True) for n, p in m.named_parameters()}
    hd, H, Hk = m.head_dim, m.num_heads, m.num_kv_heads

    def norm_rope(t, w, pos):
        n = t * ((t * t).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        axes = pos.shape[-1]
        ra = hd // (2 * axes) * 2
        out = []
        for a in range(axes):
            lo, hi = n[..., a * ra:a * ra + ra // 2], n[..., a * ra + ra // 2:(a + 1) * ra]
            ang = (pos[:, a, None].double() * m.base ** (-torch.arange(0, ra, 2, device=t.device, dtype=torch.float64) / ra))[:, None]
            out += [lo * ang.cos() - hi * ang.sin(), lo * ang.sin() + hi * ang.cos()]
        return torch.cat(out + [n[..., axes * ra:]], -1)
    q = torch.nn.functional.linear(x, P["q.weight"], P["q.bias"]).unflatten(-1, (H, hd))
    kv = torch.nn.functional.linear(states, P["kv.weight"], P["kv.bias"]).unflatten(-1, (2, Hk, hd))
    q, k = norm_rope(q, P["q_norm"], xp), norm_rope(kv[:, :, 0], P["k_norm"], sp)
    k, v = (t.repeat_interleave(H // Hk, 2).permute(0, 2, 1, 3) for t in (k, kv[:, :, 1]))
    s = (q.permute(0, 2, 1, 3) @ k.transpose(-1, -2).contiguous() * hd ** -0.5).masked_fill(~allowed[:, None, None, :], -math.inf)
    y = (torch.softmax(s, -1) @ v).permute(0, 2, 1, 3).flatten(2)
    return torch.nn.functional.linear(y, P["proj.weight"], P["proj.bias"]), P


@gpu
@pytest.mark.parametrize("autocast", [False, True], ids=["f32", "autocast"])
def test_the_layer(autocast):
    """Projections, norm, rotation and attention of layers.CrossAttention with shared heads and a padded batch, against the formulas
    in 64 bits: relative 2-norm, 8 roundings of the type in a row (3 projections, q / k, P, dS, output, gradient); for fp32, whose
    products go through the library's matrix kernels, 1e-4."""
    from mono_vifi_amd import layers
    torch.manual_seed(0)
    m = layers.CrossAttention(48, num_heads=4, num_kv_heads=2, states_dim=32).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 30, 48, device="cuda", generator=g, requires_grad=True)
    st = torch.randn(2, 60, 32, device="cuda", generator=g, requires_grad=True)
    go = torch.randn(2, 30, 48, device="cuda", generator=g)
    xp, sp = layers.token_positions(5, 6, (0,), x.device), layers.token_positions(5, 6, (-1, 1), x.device)
    assert sp.shape == (60, 3) and sp[31].tolist() == [1, 0, 1] and layers.token_positions(5, 6, (-1, 1), x.device) is sp
    lens = torch.tensor([60, 37], dtype=torch.int32, device="cuda")
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        y = m(x, st, xp, sp, kv_lens=lens)
    assert y.dtype == (torch.bfloat16 if autocast else torch.float32)
    names = [n for n, _ in m.named_parameters()]
    got = [y] + list(torch.autograd.grad(y, [x, st] + [p for _, p in m.named_parameters()], go.to(y.dtype)))
    xr, sr = x.detach().double().requires_grad_(True), st.detach().double().requires_grad_(True)
    want, P = layer_ref(m, xr, sr, xp, sp, torch.arange(60, device="cuda") < lens[:, None])
    wants = [want] + list(torch.autograd.grad(want, [xr, sr] + [P[n] for n in names], go.double()))
    tol = 8 * 2.0 ** -8 if autocast else 1e-4
    for n, a, b in zip(["y", "x", "states"] + names, got, wants):
        assert float((a.double() - b).norm()) <= tol * float(b.norm()), n


@gpu
def test_fusion_module_attends(tmp_path):
    """--fusion_attention: the same fused features at first (the output projection starts at zero), gradients in every parameter of
    the attention once it does not, checkpoint keys beside the reference's."""
    from types import SimpleNamespace
    from mono_vifi_amd.networks import FusionModule
    ch = [64, 64, 128, 256, 512]
    torch.manual_seed(0)
    plain = FusionModule(SimpleNamespace(backbone="ResNet18"), ch).cuda()
    with_attn = FusionModule(SimpleNamespace(backbone="ResNet18", fusion_attention=2), ch).cuda()
    extra = set(with_attn.state_dict()) - set(plain.state_dict())
    assert all(k.startswith("cross_frame.") for k in extra) and len(extra) == 2 * 8
    with_attn.load_state_dict(plain.state_dict(), strict=False)
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    feats = [[r(2, c, 64 >> i, 96 >> i) for i, c in zip(range(1, 6), ch)] for _ in range(3)]
    flows, mask = [3 * r(2, 2, 64, 96) for _ in range(2)], torch.rand(2, 1, 64, 96, device="cuda", generator=g)
    a, b = plain(feats, flows, mask), with_attn(feats, flows, mask)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    for m in with_attn.cross_frame:
        torch.nn.init.normal_(m.attn.proj.weight, std=0.05)
    out = with_attn(feats, flows, mask)
    assert all(torch.equal(out[i], a[i]) for i in range(3)) and not torch.equal(out[4], a[4]) and not torch.equal(out[3], a[3])
    sum(o.square().mean() for o in out).backward()
    for n, p in with_attn.cross_frame.named_parameters():
        assert torch.isfinite(p.grad).all() and float(p.grad.norm()) > 0, n


@gpu
@pytest.mark.parametrize("amp", [False, True], ids=["f32", "amp_bf16"])
def test_training_step_with_fusion_attention(tmp_path, amp):
    from test_trainer_gpu import device_batch, make_trainer
    t = make_trainer(tmp_path, fusion_attention=2, amp_bf16=amp)
    t.set_train()
    proj = t.models["fusion_module"].cross_frame[0].attn.proj.weight
    assert not proj.any()
    batch = device_batch(2, 64, 96, t.device)
    for _ in range(2):
        losses = t.optimisation_step(dict(batch))
        assert math.isfinite(float(losses["loss"]))
    assert proj.any() and all(torch.isfinite(p).all() for p in t.models["fusion_module"].parameters())


def graph_worker(*args, timeout):
    import os
    import subprocess
    import sys
    p = subprocess.run([sys.executable, os.path.join(os.path.dirname(__file__), "attention_graph_worker.py"), *args],
                       env={"MIOPEN_FIND_MODE": "FAST", **os.environ}, capture_output=True, text=True, timeout=timeout)
    assert p.returncode == 0, p.stderr[-3000:]
    return [line for line in p.stdout.splitlines() if line.startswith("RESULT ")][-1][len("RESULT "):]


@gpu
def test_the_layer_in_a_captured_graph():
    """Every replay gives the eager result, projections and their biases' sums included (same kernels: the bar only allows the
    libraries another order of a sum: fp32 sums of 12 * 960 terms)."""
    assert float(graph_worker("layer", timeout=110)) <= 12 * 960 * U


@gpu
def test_captured_training_step_with_fusion_attention(tmp_path):
    """--hip_graph with --fusion_attention follows the eager trainer (bars: tests/test_trainer_gpu.py, the same comparison without it)."""
    import json
    r = json.loads(graph_worker("step", "ResNet18", "2", "64", "96", str(tmp_path), "step", timeout=300))
    e, g = r["eager"], r["graph"]
    assert g["captured"] and all(math.isfinite(x) for row in g["losses"] for x in row)
    for i, (a, b) in enumerate(zip(g["losses"], e["losses"])):
        assert all(abs(x - y) <= (1e-4 if i < 2 else 5e-2) * abs(y) + 1e-6 for x, y in zip(a, b)), (i, a, b)
    assert g["delta_norm"] > 0.5 * e["delta_norm"] > 0 and r["resume_equal"]


@pytest.mark.parametrize("channels", [18, 36, 48, 64, 80, 128, 224, 512, 1024, 2048])
def test_heads_of_the_fusion_attention(channels):
    """Every width of a pyramid level gets heads that the attention takes (ResNet50's coarsest level has 2,048 channels)."""
    from mono_vifi_amd.networks.fusion_module import CrossFrame
    m = CrossFrame(channels).attn
    assert m.num_heads * m.head_dim == channels and 6 <= m.head_dim <= 128
    assert m.num_heads <= 8 or channels > 8 * 128


@gpu
@pytest.mark.parametrize("channels", [36, 2048])
def test_fusion_attention_of_wide_and_narrow_levels(channels):
    from mono_vifi_amd.networks.fusion_module import CrossFrame
    m = CrossFrame(channels).cuda()
    torch.nn.init.normal_(m.attn.proj.weight, std=0.02)
    f = [torch.randn(1, channels, 3, 5, device="cuda", requires_grad=True) for _ in range(4)]
    y = m(*f)
    assert y.shape == f[0].shape and not torch.equal(y, f[0])
    y.square().mean().backward()
    assert all(torch.isfinite(x.grad).all() and x.grad.any() for x in f)


def test_the_layer_refuses_heads_that_are_too_wide():
    from mono_vifi_amd import layers
    with pytest.raises(ValueError, match="at most 128"):
        layers.CrossAttention(1024, 4)


def test_the_layer_refuses_heads_that_do_not_divide():
    from mono_vifi_amd import layers
    for args in ((50, 8), (48, 4, 3)):
        with pytest.raises(ValueError, match="do not divide"):
            layers.CrossAttention(*args)
    m = layers.CrossAttention(16, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        m(torch.zeros(1, 3, 16), torch.zeros(1, 4, 16))


# ------------------------------------------------------------------------------------------------ refusals (no GPU)
def cpu(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("args,kw,match", [
    ((cpu(2, 3, 4), cpu(1, 2, 2, 4), cpu(1, 2, 2, 4)), {}, "batch, tokens, heads, channels"),
    ((cpu(1, 3, 2, 4, dtype=torch.float16),) * 3, {}, "float32 or bfloat16"),
    ((cpu(1, 3, 2, 4), cpu(1, 3, 2, 4, dtype=torch.bfloat16), cpu(1, 3, 2, 4)), {}, "queries are"),
    ((cpu(1, 3, 2, 160),) * 3, {}, "1..128 channels"),
    ((cpu(1, 3, 0, 4),) * 3, {}, "at least one head"),
    ((cpu(1, 3, 3, 4), cpu(1, 5, 2, 4), cpu(1, 5, 2, 4)), {}, "do not fit"),
    ((cpu(1, 3, 2, 4), cpu(2, 5, 2, 4), cpu(2, 5, 2, 4)), {}, "do not fit"),
    ((cpu(1, 3, 2, 4), cpu(1, 5, 2, 4), cpu(1, 6, 2, 4)), {}, "differ"),
    ((cpu(1, 3, 2, 4),) * 3, {"scale": 0.0}, "positive"),
    ((cpu(1, 3, 2, 4),) * 3, {"scale": math.nan}, "positive"),
    ((cpu(1, 3, 2, 4),) * 3, {"key_mask": torch.ones(1, 4, dtype=torch.bool)}, "key_mask"),
    ((cpu(1, 3, 2, 4),) * 3, {"key_mask": torch.ones(1, 3)}, "key_mask"),
    ((cpu(1, 3, 2, 4),) * 3, {"kv_lens": torch.ones(2, dtype=torch.int32)}, "kv_lens"),
    ((cpu(1, 3, 2, 4),) * 3, {"kv_lens": torch.ones(1)}, "kv_lens"),
    ((cpu(1, 3, 2, 4),) * 3, {}, "no CPU fallback"),
])
def test_attention_refuses(args, kw, match):
    with pytest.raises(RuntimeError, match=match):
        ops.cross_attention(*args, **kw)


X = cpu(1, 3, 2, 8)
P = torch.zeros(3, 1, dtype=torch.int32)


@pytest.mark.parametrize("args,kw,match", [
    ((cpu(3, 2, 8),), {}, "batch, tokens, heads, channels"),
    ((X, cpu(2, 3, 2, 8)), {}, "does not fit"),
    ((X, cpu(1, 3, 2, 6)), {}, "does not fit"),
    ((X, None, None, torch.ones(8)), {}, "without k"),
    ((X, None, torch.ones(7)), {}, "q_weight"),
    ((X, X, None, torch.ones(8, dtype=torch.float64)), {}, "k_weight"),
    ((X, None, None, None, P.float()), {}, "int32 or int64"),
    ((X, None, None, None, P[:2]), {}, "q_pos must be"),
    ((X, None, None, None, torch.zeros(3, 4, dtype=torch.int32)), {}, "q_pos must be"),
    ((X, None, None, None, torch.zeros(2, 3, 1, dtype=torch.int32)), {}, "q_pos must be"),
    ((X, X, None, None, P, torch.zeros(3, 2, dtype=torch.int32)), {}, "different numbers of axes"),
    ((X, None, None, None, P), {"rot_dim": 3}, "rot_dim"),
    ((X, None, None, None, P), {"rot_dim": 10}, "rot_dim"),
    ((X, None, None, None, P), {"rot_dim": -2}, "rot_dim"),
    ((X,), {"eps": -1.0}, "eps"),
    ((X,), {"base": 0.0}, "base"),
    ((X,), {}, "no CPU fallback"),
])
def test_norm_refuses(args, kw, match):
    with pytest.raises(RuntimeError, match=match):
        ops.qk_norm_rope(*args, **kw)


def test_groups_beyond_the_kernels_division_are_refused():
    """The dk / dv kernel finds a row's token by a product in fp32, exact for groups of at most 65,536 heads."""
    g, x = (torch.arange(n, dtype=torch.float64) for n in (65537, 64))
    for G in (1, 3, 7, 63, 1000, 65535, 65536):
        inv = (torch.ones(1) / G).float()
        row = torch.unique(torch.cat([g[:G][:200], g[:G][-200:]]))[:, None] + x            # g0 + row, g0 < G
        got = ((row.float() + 0.5) * inv).floor()
        assert torch.equal(got.double(), torch.floor(row / G)), G
    lib = nat.lib()
    buf = (C.c_float * 64)()
    P = C.addressof(buf) + (-C.addressof(buf)) % 16
    d = nat.AttnDesc(q=P, k=P, v=P, B=1, Lq=1, Lk=1, Hq=65537, Hk=1, D=1, dtype=nat.DTYPE_F32, scale=1.0)
    assert lib.mvf_cross_attention_fwd(C.byref(d), P, None, None, None) == 1
    assert lib.mvf_cross_attention_bwd(C.byref(d), P, P, P, P, P, P, P, None) == 1


def test_entry_points_refuse_bad_descriptors():
    """The C entry points check their arguments before the first HIP call (hipErrorInvalidValue = 1)."""
    if not __import__("os").path.exists(nat.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    lib = nat.lib()
    buf = (C.c_float * 64)()
    P = C.addressof(buf) + (-C.addressof(buf)) % 16

    def desc(**kw):
        d = dict(q=P, k=P, v=P, B=1, Lq=2, Lk=2, Hq=2, Hk=1, D=8, dtype=nat.DTYPE_F32, scale=1.0)
        return nat.AttnDesc(**{**d, **kw})

    def fwd(d, out=P):
        return lib.mvf_cross_attention_fwd(C.byref(d) if d is not None else None, out, None, None, None)
    for bad in (dict(D=0), dict(D=129), dict(Hq=3, Hk=2), dict(Hk=0), dict(Lq=-1), dict(dtype=7), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=math.nan), dict(scale=math.inf), dict(q=None), dict(k=None), dict(Lk=(1 << 30) + 1),
                dict(B=1 << 20, Hk=1 << 10, Hq=1 << 10)):
        assert fwd(desc(**bad)) == 1, bad
        assert lib.mvf_cross_attention_bwd(C.byref(desc(**bad)), P, P, P, P, P, P, P, None) == 1, bad
    assert fwd(None) == 1 and fwd(desc(), out=None) == 1 and fwd(desc(), out=P + 4) == 1
    assert fwd(desc(Lk=100000)) == 1                                     # split: needs its workspace
    assert lib.mvf_cross_attention_fwd_workspace_bytes(C.byref(desc(Lk=100000))) > 0
    assert fwd(desc(B=0)) == 0 and fwd(desc(Lq=0)) == 0                  # nothing to do
    assert lib.mvf_cross_attention_bwd(C.byref(desc()), P, None, P, P, P, P, P, None) == 1
    assert lib.mvf_cross_attention_bwd(C.byref(desc()), P, P, P, P, P, None, P, None) == 1

    freq = (C.c_uint64 * 64)()

    def norm(**kw):
        d = dict(q=P, k=P, freq=C.addressof(freq), B=1, Lq=2, Lk=2, Hq=1, Hk=1, D=8, dtype=nat.DTYPE_F32, axes=1, rot=8, eps=1e-6)
        return nat.QkNormDesc(**{**d, **kw})
    for bad in (dict(D=0), dict(D=130), dict(axes=0), dict(axes=4), dict(rot=9), dict(rot=7), dict(rot=-2), dict(freq=None), dict(dtype=3),
                dict(Hq=0), dict(Lk=-1), dict(Lq=1 << 30, Hq=2)):
        assert lib.mvf_qk_norm_rope_fwd(C.byref(norm(**bad)), P, P, None) == 1, bad
        assert lib.mvf_qk_norm_rope_bwd(C.byref(norm(**bad)), P, P, P, P, None, None, None, None) == 1, bad
    assert lib.mvf_qk_norm_rope_fwd(C.byref(norm()), None, P, None) == 1
    assert lib.mvf_qk_norm_rope_fwd(C.byref(norm()), P, P + 4, None) == 1
    assert lib.mvf_qk_norm_rope_bwd(C.byref(norm()), P, P, P, P, P, None, None, None) == 1      # weight gradients need the workspace
    assert lib.mvf_qk_norm_rope_fwd(C.byref(norm(B=0)), None, None, None) == 0
