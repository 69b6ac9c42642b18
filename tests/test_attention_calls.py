"""Calls of the token-attention operators that are not the ordinary one: tracing and forward mode, captured backwards of leaves that the
call converts, positions made in another mode, sizes at the launch limits; and how exact the fp32 products are, normwise."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.fx.experimental.proxy_tensor import make_fx

import mono_vifi_amd  # noqa: F401
from mono_vifi_amd import ops

gpu = pytest.mark.gpu


def heads(device="cpu", B=1, Lq=3, Lk=5, H=2, D=8):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(B, n, H, D, generator=g).to(device) for n in (Lq, Lk, Lk)]


def calls(device="cpu"):
    """(name, function, tensors) of both operators."""
    q, k, v = heads(device)
    w = torch.linspace(0.5, 1.5, q.shape[-1], device=device)
    return [("cross_attention", lambda q, k, v: ops.cross_attention(q, k, v), [q, k, v]),
            ("qk_norm_rope", lambda q, k, wq, wk: ops.qk_norm_rope(q, k, wq, wk)[0], [q, k, w, w.clone()])]


# ------------------------------------------------------------------------------------------------ routes past the operators
def refuses_forward_mode(device):
    for name, f, xs in calls(device):
        for i in range(len(xs)):
            for grad in (False, True):
                with fwAD.dual_level():
                    args = [x.clone().requires_grad_(grad) for x in xs]
                    args[i] = fwAD.make_dual(args[i], torch.ones_like(args[i]))
                    with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
                        f(*args)


def refuses_tracing(device):
    for name, f, xs in calls(device):
        for grad in (False, True):
            args = tuple(x.clone().requires_grad_(grad) for x in xs)
            with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
                torch.jit.trace(f, args)
            with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
                make_fx(f)(*args)


def test_forward_mode_is_refused():
    """A tangent that would be dropped: refused before the device is looked at, whichever input carries it."""
    refuses_forward_mode("cpu")


def test_tracing_is_refused():
    """A trace would hold the allocation of the output and not the kernels that fill it."""
    refuses_tracing("cpu")
    from mono_vifi_amd import layers
    m = layers.CrossAttention(16, 2)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(m, (torch.zeros(1, 3, 16), torch.zeros(1, 4, 16)), check_trace=False)


@gpu
def test_other_routes_are_refused_on_the_device():
    refuses_forward_mode("cuda")
    refuses_tracing("cuda")
    for _, f, xs in calls("cuda"):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, tuple(xs), tuple(torch.ones_like(x) for x in xs))
        with pytest.raises(RuntimeError):
            torch.vmap(f)(*(torch.stack([x, x]) for x in xs))


@gpu
def test_a_backward_under_another_route_is_refused():
    """The gradient that arrives carries a tangent, or the backward runs while a trace is recorded."""
    for name, f, xs in calls("cuda"):
        leaves = [x.requires_grad_(True) for x in xs]
        out = f(*leaves)
        go = torch.ones_like(out)
        want = torch.autograd.grad(out, leaves, go, retain_graph=True)
        with fwAD.dual_level():
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(out, leaves, fwAD.make_dual(go, go), retain_graph=True)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(lambda g: torch.autograd.grad(out, leaves, g, retain_graph=True))(go)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, go), want))


# ------------------------------------------------------------------------------------------------ checkpoints of --fusion_attention
def fusion(levels, seed):
    from types import SimpleNamespace
    from mono_vifi_amd.networks import FusionModule
    torch.manual_seed(seed)
    m = FusionModule(SimpleNamespace(backbone="ResNet18", fusion_attention=levels), [16, 16, 32, 48, 64])
    for p in m.parameters():
        torch.nn.init.normal_(p)
    return m


def load(checkpoint, model):
    from types import SimpleNamespace
    from mono_vifi_amd.trainer import Trainer
    fake = SimpleNamespace(models={"fusion_module": model}, _check_attention_levels=getattr(Trainer, "_check_attention_levels", None))
    Trainer._load_into_models(fake, {"fusion_module": checkpoint.state_dict()})


@pytest.mark.parametrize("saved,mine", [(2, 0), (2, 1), (1, 0), (5, 4)])
def test_a_checkpoint_does_not_lose_its_attention(saved, mine):
    source, model = fusion(saved, 1), fusion(mine, 2)
    before = [p.detach().clone() for p in model.parameters()]
    with pytest.raises(ValueError, match=f"--fusion_attention {saved}"):
        load(source, model)
    assert all(torch.equal(a, b) for a, b in zip(before, model.parameters()))


@pytest.mark.parametrize("saved,mine", [(0, 0), (2, 2), (0, 2), (1, 2)])
def test_a_checkpoint_loads_with_as_many_levels_or_more(saved, mine, caplog):
    """Every saved entry arrives; levels that the checkpoint lacks keep theirs, with a warning."""
    source, model = fusion(saved, 1), fusion(mine, 2)
    own = {k: v.clone() for k, v in model.state_dict().items()}
    with caplog.at_level("WARNING"):
        load(source, model)
    assert bool(caplog.records) == (saved < mine)
    given, now = source.state_dict(), model.state_dict()
    assert set(given) <= set(now) and len(now) - len(given) == 8 * (mine - saved)
    assert all(torch.equal(now[k], given[k] if k in given else own[k]) for k in now)


@gpu
def test_resume_with_fusion_attention(tmp_path):
    """A trainer with two levels resumes as one with two, parameter for parameter and with its optimizer's moments; with fewer it is
    refused."""
    from test_trainer_gpu import device_batch, make_trainer
    t = make_trainer(tmp_path, fusion_attention=2)
    t.set_train()
    t.optimisation_step(device_batch(2, 64, 96, t.device))
    t.save_model(batch_idx=1)
    again = make_trainer(tmp_path, fusion_attention=2, resume=True)
    assert len(again.parameters_to_train) == len(t.parameters_to_train)
    assert all(torch.equal(a, b) for a, b in zip(t.parameters_to_train, again.parameters_to_train))
    assert len(again.model_optimizer.state) == len(t.model_optimizer.state) > 0
    with pytest.raises(ValueError, match="--fusion_attention 2"):
        make_trainer(tmp_path, resume=True)


# ------------------------------------------------------------------------------------------------ tensors that are made once
def made_once():
    from mono_vifi_amd import consts, layers
    return [lambda d: layers.token_positions(3, 7, (-2, 5), d), lambda d: consts.const_tensor((0.125, 77.0), d)]


def test_tensors_made_under_inference_mode_can_be_saved_for_a_backward(monkeypatch):
    from mono_vifi_amd import consts
    monkeypatch.setattr(consts, "_CACHE", {})
    for make in made_once():
        with torch.inference_mode():
            first = make("cpu")
        assert make("cpu") is first and not first.is_inference()
        x = torch.ones(first.shape, requires_grad=True)
        (g,) = torch.autograd.grad((x * first).sum(), x)
        assert torch.equal(g, first.to(g.dtype))


def test_a_device_without_an_index_is_the_current_one(monkeypatch):
    """What was made for "cuda" on one GPU is not handed out on another: the key names the index."""
    from mono_vifi_amd import consts
    for make, key in zip(made_once(), (("token_positions", 3, 7, (-2, 5)), ((0.125, 77.0),))):
        monkeypatch.setattr(consts, "_CACHE", {key + ("cuda:0",) + tail: "first" for tail in ((), (torch.float32,))} |
                            {key + ("cuda:1",) + tail: "second" for tail in ((), (torch.float32,))})
        for current, want in enumerate(("first", "second")):
            monkeypatch.setattr(torch.cuda, "current_device", lambda: current)
            assert make("cuda") == make(torch.device("cuda")) == make(f"cuda:{current}") == want


def test_positions_of_frames_that_can_be_read_once():
    from mono_vifi_amd import layers
    pos = layers.token_positions(2, 2, (f for f in (-3, 4)), "cpu")
    assert pos.tolist() == [[f, r, c] for f in (-3, 4) for r in range(2) for c in range(2)]


# ------------------------------------------------------------------------------------------------ captured backwards
def captured_backward(kind):
    """(call, leaves): leaves that the operators reach behind a copy, a conversion or a view."""
    q, k, v = heads("cuda", Lq=5, Lk=40, D=32)
    w = torch.linspace(0.5, 1.5, 32, device="cuda")
    if kind == "weight in bfloat16":
        leaves = [q.bfloat16().requires_grad_(True), w.bfloat16().requires_grad_(True)]
        return lambda: ops.qk_norm_rope(leaves[0], None, leaves[1]), leaves
    if kind == "channels not adjacent":
        leaves = [x.transpose(1, 3).contiguous().transpose(1, 3).requires_grad_(True) for x in (q, k, v)]
        return lambda: ops.cross_attention(*leaves), leaves
    leaves = [q.requires_grad_(True), torch.cat([k, v], 2).requires_grad_(True)]
    return lambda: ops.cross_attention(leaves[0], leaves[1][:, :, :2], leaves[1][:, :, 2:]), leaves


@gpu
@pytest.mark.parametrize("kind", ["weight in bfloat16", "channels not adjacent", "packed projection"])
def test_a_captured_backward_finds_the_leaves_of_a_living_eager_graph(kind):
    """As for leaves that are the operators' own inputs: an error, and without the eager graph the same capture runs and replays."""
    call, leaves = captured_backward(kind)
    eager = call()
    go = torch.ones_like(eager)
    want = [x.clone() for x in torch.autograd.grad(eager, leaves, go, retain_graph=True)]
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
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


@gpu
def test_a_captured_backward_looks_only_at_leaves_that_it_reaches():
    """An eager graph of a leaf whose gradient is not asked for does not stand in the way."""
    q, k, v = (x.requires_grad_(True) for x in heads("cuda"))
    eager = q * 2                                          # keeps q's accumulation node on the default stream
    go = torch.ones_like(q)
    want = torch.autograd.grad(ops.cross_attention(q.detach(), k, v), [k, v], go)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(ops.cross_attention(q, k, v), [k, v], go)
    for _ in range(3):
        for x in got:
            x.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert eager.requires_grad


# ------------------------------------------------------------------------------------------------ the build
def make(*args):
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mono-vifi_amd", "csrc")
    return subprocess.run(["make", "-n", "-C", csrc, "PYTHON=/nonexistent/python", *args], capture_output=True, text=True, timeout=60)


@pytest.mark.parametrize("target", [(), ("all",), ("fast",), ("clean",)], ids=str)
def test_the_c_library_is_built_without_python(target):
    r = make(*target)
    assert r.returncode == 0 and "/nonexistent" not in r.stdout + r.stderr and "mvf_torch" not in r.stdout
    assert "/nonexistent" in make("torch").stdout                   # (the target that does need it)


@pytest.mark.parametrize("what,change", [("ABI 17", lambda mp, nat: mp.setattr(nat, "ABI_VERSION", 99)),
                                         ("torch 2", lambda mp, nat: mp.setattr(torch, "__version__", "1.0.0+other"))])
def test_an_extension_of_another_build_is_not_loaded(monkeypatch, what, change):
    from mono_vifi_amd import _native as nat
    nat.lib()
    monkeypatch.setattr(nat, "_torch_ops", None)
    change(monkeypatch, nat)
    with pytest.raises(nat.NativeLibraryError, match=f"built for .*{what}.*run "):
        nat.torch_ops()
    monkeypatch.undo()
    monkeypatch.setattr(nat, "_torch_ops", None)
    monkeypatch.setattr(torch, "__version__", torch.__version__.split("+")[0] + "a0+git1234567")      # (the header knows the three numbers)
    assert nat.torch_ops() is not None


# ------------------------------------------------------------------------------------------------ sizes at the limits of a launch
def c_call(cls, **kw):
    """A descriptor over a little host memory: what is refused is refused before anything is launched."""
    import ctypes as C
    buf = (C.c_uint64 * 64)()
    P = C.addressof(buf) + (-C.addressof(buf)) % 16
    fields = dict(q=P, k=P, B=1, Lq=1, Lk=1, Hq=1, Hk=1, D=8)
    fields.update({"v": P, "scale": 1.0} if cls.__name__ == "AttnDesc" else {"freq": C.addressof(buf), "axes": 1, "eps": 1e-6})
    return cls(**{**fields, **kw}), P, buf


# a launch takes at most 2^32 - 1 threads.  Per sequence and head of states: fp32, at most 16 rows: 512 threads (256 at more than 96 channels), 32 rows: 256;
# bf16: 256; the backward's two kernels: 256 per 128 rows and per 128 states
@pytest.mark.parametrize("kw,most", [
    (dict(dtype=0), (1 << 23) - 1), (dict(dtype=0, D=128), (1 << 24) - 1), (dict(dtype=0, Lq=32), (1 << 24) - 1), (dict(dtype=1), (1 << 24) - 1),
    (dict(dtype=0, Lq=129), (1 << 23) - 1), (dict(dtype=1, Lk=257), ((1 << 24) - 1) // 3)])
def test_attention_sizes_at_the_limit_of_a_launch(kw, most):
    import ctypes as C
    from mono_vifi_amd import _native as nat
    lib = nat.lib()
    for heads_ in (1, 8):
        inside, P, keep = c_call(nat.AttnDesc, **kw, B=most // heads_, Hq=heads_, Hk=heads_)
        assert lib.mvf_cross_attention_bwd_workspace_bytes(C.byref(inside)) > 0
        beyond, P, keep = c_call(nat.AttnDesc, **kw, B=most // heads_ + 1, Hq=heads_, Hk=heads_)
        assert lib.mvf_cross_attention_bwd_workspace_bytes(C.byref(beyond)) == 0
        assert lib.mvf_cross_attention_fwd(C.byref(beyond), P, None, P, None) == 1
        assert lib.mvf_cross_attention_bwd(C.byref(beyond), P, P, P, P, P, P, P, None) == 1


def test_the_rest_of_the_output_has_to_be_aligned():
    import ctypes as C
    from mono_vifi_amd import _native as nat
    d, P, keep = c_call(nat.AttnDesc, dtype=1)
    d.out_low = P + 4
    assert nat.lib().mvf_cross_attention_fwd(C.byref(d), P, None, P, None) == 1
    assert nat.lib().mvf_cross_attention_bwd(C.byref(d), P, P, P, P, P, P, P, None) == 1


# a workgroup of 256 threads takes 256 rows of one pair of channels, 64 of 4 lanes, 4 of 64
@pytest.mark.parametrize("kw,rows", [(dict(D=2, rot=2), 256), (dict(D=32, rot=32), 64), (dict(D=128, rot=126, axes=3), 4)])
def test_norm_sizes_at_the_limit_of_a_launch(kw, rows):
    import ctypes as C
    from mono_vifi_amd import _native as nat
    lib = nat.lib()
    most = min(((1 << 24) - 1) * rows, (1 << 30) - 1)
    inside, P, keep = c_call(nat.QkNormDesc, **kw, k=None, Lq=most)
    assert lib.mvf_qk_norm_rope_bwd_workspace_floats(C.byref(inside)) > 0
    beyond, P, keep = c_call(nat.QkNormDesc, **kw, k=None, Lq=most + 1)
    assert lib.mvf_qk_norm_rope_bwd_workspace_floats(C.byref(beyond)) == 0
    assert lib.mvf_qk_norm_rope_fwd(C.byref(beyond), P, None, None) == 1
    assert lib.mvf_qk_norm_rope_bwd(C.byref(beyond), P, None, P, None, None, None, None, None) == 1


# ------------------------------------------------------------------------------------------------ how exact the fp32 products are
# An fp32 value is three planes of bf16 (8 + 8 + 8 bits, cut), a product the six plane products of order <= 2.  Worst-case bounds of sums leave
# room for a whole missing term; a relative 2-norm does not.  With all six, what is left out and the fp32 roundings of P and dS come to
# 2e-7 of an output or gradient (the emulation below, exact sums).  The kernels' sums round about 6 D / 16 times per product and once per
# tile of states, at random: sqrt(48 + 40) 2^-24 = 6e-7 of the result, twice that where two such sums follow each other.  So 2e-6; any one term
# missing in any one product is 5e-6 or more in what depends on it.
BAR = 2e-6
TERMS = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)]
PRODUCTS = ["S", "PV", "dP", "dSK", "S of dk, dv", "PtG", "dStQ"]


def planes(x):
    out, x = [], x.float()
    for _ in range(3):
        cut = (x.contiguous().view(torch.int32) & -65536).view(torch.float32)
        out.append(cut.double())
        x = x - cut
    return out


def by_heads(q, k, v):
    G = q.shape[2] // k.shape[2]
    return [q.permute(0, 2, 1, 3)] + [x.permute(0, 2, 1, 3).repeat_interleave(G, 1) for x in (k, v)]


def emulated(q, k, v, go, missing=(None, None)):
    """[out, dq, dk, dv] of the three-plane products with exact sums; missing: (product, term of it that is left out)."""
    def mm(name, a, b):
        A, B = planes(a), planes(b)
        return sum(A[i] @ B[j] for i, j in TERMS if (name, (i, j)) != missing)
    t = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    fold = lambda x: x.unflatten(1, (k.shape[2], -1)).sum(2).permute(0, 2, 1, 3)  # noqa: E731
    scale = q.shape[-1] ** -0.5
    c = torch.tensor(scale / 0.6931471805599453, dtype=torch.float32)
    qh, kh, vh = by_heads(q, k, v)
    gh = go.permute(0, 2, 1, 3)
    s = mm("S", qh * c, t(kh))
    m = s.amax(-1, keepdim=True)
    p = torch.exp2(s - m).float()
    total = p.double().sum(-1, keepdim=True)
    o = mm("PV", p, vh) / total
    lse = m + total.log2()
    delta = (gh.double() * o.float().double()).sum(-1, keepdim=True)
    dp = mm("dP", gh, t(vh))
    dq = mm("dSK", torch.exp2(s - lse) * (dp - delta), kh) * scale
    p = torch.exp2(mm("S of dk, dv", qh, t(kh * c)) - lse)
    return [o.permute(0, 2, 1, 3), dq.permute(0, 2, 1, 3), fold(mm("dStQ", t(p * (dp - delta)), qh)) * scale, fold(mm("PtG", t(p), gh))]


def defined(q, k, v, go):
    xs = [x.detach().double().requires_grad_(True) for x in (q, k, v)]
    qh, kh, vh = by_heads(*xs)
    p = torch.softmax(qh @ kh.transpose(-1, -2).contiguous() * q.shape[-1] ** -0.5, -1)
    o = (p @ vh).permute(0, 2, 1, 3)
    return [o.detach()] + list(torch.autograd.grad(o, xs, go.double()))


def deviations(got, want):
    return [float((a.double() - b).norm() / b.norm()) for a, b in zip(got, want)]


def normal(seed, B, Lq, Lk, Hq, Hk, D, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, n, h, D, generator=g).to(device) for n, h in ((Lq, Hq), (Lk, Hk), (Lk, Hk), (Lq, Hq))]


@pytest.mark.parametrize("shape", [(1, 130, 200, 2, 1, 32), (1, 70, 200, 2, 2, 28), (1, 20, 600, 1, 1, 128), (2, 3, 2500, 4, 1, 80)], ids=str)
def test_the_bar_notices_a_missing_term(shape):
    xs = normal(1, *shape)
    want = defined(*xs)
    assert max(deviations(emulated(*xs), want)) <= BAR / 8
    depend = {"S": (0, 1), "PV": (0,), "dP": (1, 2), "dSK": (1,), "S of dk, dv": (2, 3), "PtG": (3,), "dStQ": (2,)}
    for name in PRODUCTS:
        for term in TERMS[1:]:
            e = deviations(emulated(*xs, (name, term)), want)
            assert max(e[i] for i in depend[name]) >= 2.5 * BAR, (name, term, e)


FORMS = [(1, 130, 200, 2, 1), (2, 600, 700, 2, 2), (1, 8, 600, 2, 1), (2, 3, 2500, 4, 1), (1, 20, 600, 1, 1), (1, 31, 40, 1, 1)]


@gpu
@pytest.mark.parametrize("D", [28, 32, 57, 64, 80, 96, 100, 128])
@pytest.mark.parametrize("form", FORMS, ids=["rows", "rows in parts", "16 rows", "16 rows in parts", "32 rows in parts", "32 rows"])
def test_fp32_products_keep_all_their_terms(form, D):
    q, k, v, go = normal(2, *form, D, device="cuda")
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = ops.cross_attention(*leaves)
    e = deviations([out.detach()] + list(torch.autograd.grad(out, leaves, go)), defined(q, k, v, go))
    assert max(e) <= BAR, e


@gpu
def test_the_layer_in_a_captured_graph_stays_with_the_eager_one():
    """The replays of the captured layer against eager calls: the operators' bits are equal, the libraries may sum in another order: twice
    the random walk of the longest sum, 12 * 960 terms."""
    from test_attention import graph_worker
    assert float(graph_worker("layer", timeout=110)) <= 2 * (12 * 960) ** 0.5 * 2.0 ** -24


# ------------------------------------------------------------------------------------------------ far positions
def sines(pos, n, base):
    """Sine and cosine of pos * base^(-2 j / n), j < n / 2, from 60 digits."""
    import decimal
    import math
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        pi = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
        out = []
        for p in pos:
            row = []
            for j in range(n // 2):
                turns = decimal.Decimal(p) * (decimal.Decimal(-2 * j) / n * decimal.Decimal(base).ln()).exp() / (2 * pi)
                a = float((turns - turns.to_integral_value(decimal.ROUND_FLOOR)) * 2 * pi)
                row.append((math.sin(a), math.cos(a)))
            out.append(row)
    return torch.tensor(out, dtype=torch.float64)                    # [L, n / 2, 2]


def test_sines_of_near_positions_are_those_of_64_bits():
    pos = [-70, 0, 1, 999]
    ang = torch.tensor(pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, 16, 2, dtype=torch.float64) / 16)
    # (an angle in 64 bits: the frequency and the product round, 2^-52 of up to 1,000)
    assert (sines(pos, 16, 10000) - torch.stack([ang.sin(), ang.cos()], -1)).abs().max() <= 1000 * 2.0 ** -52


@gpu
@pytest.mark.parametrize("base", [10000, 100])
@pytest.mark.parametrize("bits", [20, 31, 37, 40, 48, 62])
def test_far_positions_are_off_by_their_frequencies_rounding_alone(bits, base):
    """|pos| * 2^-64 of a turn, and the fp32 roundings of the norm and the rotation, (D + 24) 2^-24 of the pair (tests/test_attention.py)."""
    import math
    import random
    D, rng = 32, random.Random(bits)
    pos = [(1 << bits) - 1, 1 - (1 << bits), (1 << (bits - 1)) + 1] + [rng.randrange(-(1 << bits), 1 << bits) for _ in range(13)]
    x = torch.randn(1, len(pos), 1, D, generator=torch.Generator().manual_seed(bits))
    got = ops.qk_norm_rope(x.cuda(), q_pos=torch.tensor(pos, device="cuda"), base=float(base), eps=0.0)[0, :, 0].double().cpu()
    n = x[0, :, 0].double()
    n = n / (n * n).mean(-1, keepdim=True).sqrt()
    a, b = n[:, :D // 2], n[:, D // 2:]
    s, c = sines(pos, D, base).unbind(-1)
    want = torch.cat([a * c - b * s, a * s + b * c], -1)
    off = 2 * math.pi * torch.tensor([abs(p) for p in pos], dtype=torch.float64)[:, None] * 2.0 ** -64
    size = (a.abs() + b.abs()).repeat(1, 2)
    assert ((got - want).abs() <= size * ((D + 24) * 2.0 ** -24 + off) + 2.0 ** -24 * want.abs()).all()
    # and at far positions the bound itself says something: not more than a hundredth of a radian up to 2^48
    assert bits > 48 or float(off.max()) < 1e-2


# ------------------------------------------------------------------------------------------------ bfloat16: how far beyond the result's own rounding
# 1 is the error that rounding the exact result makes (relative 2-norm).  P and dS in two planes (2^-16 of a term) and delta from the output
# and its rest add a hundredth of that; P or dS in one plane are terms rounded to as many bits as the result, independently: sqrt(2), and a few
# percent where the terms cancel by chance.
def beyond_rounding(got, want):
    return [float((a.double() - b).norm() / (b.bfloat16().double() - b).norm()) for a, b in zip(got, want)]


def bf16_call(B, Lq, Lk, Hq, Hk, D, spread=1.0):
    q, k, v, go = (x.bfloat16() for x in normal(3, B, Lq, Lk, Hq, Hk, D, device="cuda"))
    q = (q * spread).bfloat16()
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = ops.cross_attention(*leaves)
    got = [out.detach()] + list(torch.autograd.grad(out, leaves, go))
    with torch.no_grad():
        alone = ops.cross_attention(*leaves)
    want = defined(q, k, v, go)
    return beyond_rounding(got, want), beyond_rounding([alone], want[:1])[0]


@gpu
@pytest.mark.parametrize("spread", [1.0, 4.0])
@pytest.mark.parametrize("D", [6, 16, 28, 64, 80, 128])
@pytest.mark.parametrize("form", [(4, 100, 8, 3, 3), (4, 100, 40, 4, 2), (10, 281, 72, 3, 3), (2, 600, 700, 2, 2), (2, 3, 2500, 4, 1), (3, 20, 600, 1, 1), (8, 4, 30, 8, 2)], ids=str)
def test_bf16_gradients_of_few_states_and_narrow_heads(form, D, spread):
    """Small calls: no precision is lost beyond the rounding of the results, also where a query attends to few states."""
    got, alone = bf16_call(*form, D, spread=spread)
    assert max(got) <= 1.05 and alone <= 1.05, (got, alone)


@gpu
@pytest.mark.parametrize("D,Lq,Lk", [(6, 3000, 4000), (12, 2000, 4000), (16, 4000, 2000), (32, 2000, 2100), (64, 1300, 1100), (96, 1200, 1000), (128, 1000, 1300)])
@pytest.mark.parametrize("spread", [1.0, 4.0])
def test_bf16_gradients_of_larger_calls(D, Lq, Lk, spread):
    """The output of a training step and dq in two planes, the others in one."""
    got, alone = bf16_call(2, Lq, Lk, 2, 2, D, spread=spread)
    assert 4 * 4 * Lq * Lk * D > 1e9                                  # (where one plane begins)
    bars = [1.05, 1.05, 1.5, 1.5]
    assert all(a <= b for a, b in zip(got, bars)) and alone <= 1.5, (got, alone)


@gpu
@pytest.mark.parametrize("form", [(2, 40, 70, 2, 2, 32), (1, 3, 300, 4, 2, 64), (1, 20, 300, 1, 1, 80), (1, 2, 5000, 2, 1, 64), (2, 600, 700, 2, 2, 28)], ids=str)
def test_bf16_infinities_that_count_come_out_as_infinities(form):
    """Every probability is positive: an infinite value of a state is infinite in that channel of every query that reads it, and nothing else
    changes."""
    q, k, v, _ = (x.bfloat16() for x in normal(4, *form, device="cuda"))
    D, group = form[-1], form[3] // form[4]
    for grad in (False, True):
        clean = ops.cross_attention(q.detach().requires_grad_(grad), k, v)
        for value in (float("inf"), float("-inf")):
            w = v.clone()
            w[0, form[2] // 2, 0, D - 3] = value
            out = ops.cross_attention(q.detach().requires_grad_(grad), k, w)
            assert (out[0, :, :group, D - 3] == value).all()
            rest = torch.ones_like(out, dtype=torch.bool)
            rest[0, :, :group, D - 3] = False
            assert torch.equal(out[rest], clean[rest])


# ------------------------------------------------------------------------------------------------ fp32: scores of a trained network's size
def plain_fp32(q, k, v, go):
    """[out, dq, dk, dv] from elementary operations in fp32, probabilities normalised before the products."""
    xs = [x.detach().requires_grad_(True) for x in (q, k, v)]
    qh, kh, vh = by_heads(*xs)
    s = qh @ kh.transpose(-1, -2).contiguous() * q.shape[-1] ** -0.5
    e = torch.exp(s - s.detach().amax(-1, keepdim=True))
    out = ((e / e.sum(-1, keepdim=True)) @ vh.contiguous()).permute(0, 2, 1, 3)
    return [out.detach()] + list(torch.autograd.grad(out, xs, go))


@gpu
@pytest.mark.parametrize("spread", [1.0, 4.0, 10.0, 30.0])
@pytest.mark.parametrize("form", [(2, 300, 400, 4, 2, 64), (2, 300, 40, 3, 3, 6), (2, 200, 3000, 2, 2, 32), (2, 5, 3000, 4, 2, 64), (1, 600, 700, 2, 2, 128),
                                  (2, 20, 900, 1, 1, 96), (2, 90, 130, 2, 2, 57)], ids=str)
def test_fp32_gradients_at_large_scores(form, spread):
    """Scores up to 150: no further off than three times the plain form in fp32, or 1e-6.  Both round the scores, each in its order (2^-24 of
    150, 8e-6 of a probability), and normalise what they got, so that the roundings of a row's largest scores cancel; three times for the
    random choice of the rows that weigh most.  Kernels that rounded a score apart in the forward and the backward are up to 10 times off."""
    q, k, v, go = normal(5, *form, device="cuda")
    q = q * spread
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = ops.cross_attention(*leaves)
    want = defined(q, k, v, go)
    got = deviations([out.detach()] + list(torch.autograd.grad(out, leaves, go)), want)
    plain = deviations(plain_fp32(q, k, v, go), want)
    assert all(a <= max(1e-6, 3 * b) for a, b in zip(got, plain)), (got, plain)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("form", [(2, 130, 200, 2, 1, 32), (1, 3, 900, 4, 2, 64), (2, 600, 700, 2, 2, 28)], ids=str)
def test_the_c_entry_points_without_their_optional_tensors(form, dtype):
    """lse alone, as one number per row: the same gradients but for its rounding (2^-24 of scores below 16) and, in bf16, that of the output in
    delta; with the optional tensors, the bits of the torch function."""
    import ctypes as C
    from mono_vifi_amd import _native as nat
    lib, (B, Lq, Lk, Hq, Hk, D) = nat.lib(), form
    q, k, v, go = (x.to(dtype) for x in normal(6, *form, device="cuda"))
    stream = torch.cuda.current_stream().cuda_stream

    def call(optional):
        d = nat.AttnDesc(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_stride=q.stride()[:3], k_stride=k.stride()[:3], v_stride=v.stride()[:3],
                         B=B, Lq=Lq, Lk=Lk, Hq=Hq, Hk=Hk, D=D, dtype=nat.DTYPE_F32 if dtype == torch.float32 else nat.DTYPE_BF16, scale=D ** -0.5)
        rest, lse = torch.empty_like(q), torch.empty(2, B, Lq, Hq, device="cuda")
        if optional:
            d.out_low, d.inv_sum = rest.data_ptr(), lse[1].data_ptr()
        out, gq, gk, gv = torch.empty_like(q), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        for size, entry, args in ((lib.mvf_cross_attention_fwd_workspace_bytes, lib.mvf_cross_attention_fwd, (out, lse)),
                                  (lib.mvf_cross_attention_bwd_workspace_bytes, lib.mvf_cross_attention_bwd, (out, lse, go, gq, gk, gv))):
            ws = torch.empty(size(C.byref(d)) + 16, dtype=torch.uint8, device="cuda")
            assert entry(C.byref(d), *(x.data_ptr() for x in args), ws.data_ptr(), stream) == 0
        return [out, gq, gk, gv]
    want = defined(q, k, v, go)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    o = ops.cross_attention(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(call(True), [o] + list(torch.autograd.grad(o, leaves, go))))
    assert max(deviations(call(False), want)) <= (BAR if dtype == torch.float32 else 3 * 2.0 ** -8)
