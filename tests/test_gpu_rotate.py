"""rotate_heads on the GPU against its definition in 64 bits (oracle/rotate_oracle.py).

Tolerances, derived before the first run. An output is rounded once (eps / 2 of its type). Before that, relative to the length of its pair: the mean of squares has
16 additions in a lane, 3 across lanes and 2 products, half of which reach its root (11 * 2**-24), root, weight and the turn's products and sum add 6 * 2**-24, sine and cosine
2**-21 (16-bit types: the hardware's, documented at 2**-21.4 and 2**-21.2) or 2**-23: below 2**-19 altogether. In the backward a sum of products has the same
length, and enters in full: below 2**-18. Sums over rows (the weights' gradients) have chains of at most 600 additions here: 2**-14 of the sum of magnitudes covers them with
the above."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import rotate_oracle as ro

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}   # a rounding, relative


def strided(t, layout):
    """The values of a (B, H, T, D) tensor in another memory order."""
    if layout == "bthd":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "odd":   # rows that are not 16-byte aligned
        wide = torch.zeros((*t.shape[:3], t.shape[3] + 3), dtype=t.dtype, device=t.device)
        wide[..., 1:-2] = t
        return wide[..., 1:-2]
    if layout == "dlast":   # head dim not the fastest
        return t.transpose(2, 3).contiguous().transpose(2, 3)
    return t.contiguous()


def wide(t):
    return t.detach().double().cpu().numpy()


def assert_within(got, want, bound, name):
    got, bad = wide(got), np.isnan(want)
    assert np.array_equal(np.isnan(got), bad), f"{name}: NaN elsewhere"
    err = np.abs(got - want)[~bad]
    over = err > bound[~bad]
    assert not over.any(), f"{name}: {over.sum()} of {err.size} beyond, worst {np.max(err / np.maximum(bound[~bad], 1e-300)):.2f} of the bound"


CASES = [
    # D, R, Hq, Hk, B, T, type, weights' type, layout, sections, interleaved, which weights
    (64, 64, 4, 2, 2, 70, "bf16", "bf16", "bhtd", None, False, "qk"),
    (128, 128, 5, 1, 1, 33, "f16", "f32", "bthd", None, True, "qk"),
    (128, 64, 2, 2, 3, 17, "f32", "f32", "bhtd", (8, 12, 12), False, "qk"),
    (16, 16, 1, 1, 2, 300, "bf16", "f32", "bthd", None, False, "k"),
    (32, 16, 3, 3, 1, 129, "f16", "f16", "odd", (3, 5), True, "qk"),
    (48, 48, 7, 1, 2, 5, "f32", "bf16", "odd", None, False, "qk"),
    (80, 80, 12, 4, 2, 41, "f32", "f32", "bthd", (8, 16, 16), False, "qk"),
    (96, 32, 2, 0, 1, 1, "bf16", "bf16", "bhtd", None, False, "q"),
    (112, 112, 3, 3, 5, 9, "f16", "f16", "dlast", (0, 56, 0), False, "q"),
    (128, 128, 32, 8, 64, 1, "bf16", "bf16", "bthd", None, False, ""),
    (64, 32, 2, 1, 1, 1000, "f32", "f32", "bhtd", None, True, ""),
]


def make(case, seed=0):
    D, R, Hq, Hk, B, T, dtype, wtype, layout, sections, interleaved, which = case
    rng = np.random.default_rng(seed)
    tensor = lambda x, t: torch.tensor(x).to(DT[t]).to(DEV)  # noqa: E731
    q = strided(tensor(rng.standard_normal((B, Hq, T, D)) * np.exp(rng.standard_normal((B, Hq, T, 1))), dtype), layout)
    k = strided(tensor(rng.standard_normal((B, Hk, T, D)), dtype), layout) if Hk else None
    w = {name: tensor(1 + 0.3 * rng.standard_normal(D), wtype) if name in which else None for name in "qk"}
    pos = rng.integers(-3, 5000, (len(sections or (1,)), B, T))
    return q, k, w, pos


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"d{c[0]}r{c[1]}-{c[6]}-{c[8]}")
@pytest.mark.parametrize("out_layout", ["contiguous", "input"])
def test_outputs_and_gradients(case, out_layout):
    from kerneldev_b200 import Rotation, rotate_heads
    D, R, Hq, Hk, B, T, dtype, wtype, layout, sections, interleaved, which = case
    q, k, w, pos = make(case)
    rotation, rot = Rotation(D, R, sections=sections, interleaved=interleaved, device=DEV), ro.rotation(D, R, sections=sections, interleaved=interleaved)
    leaves = [t.requires_grad_() for t in (q, k, w["q"], w["k"]) if t is not None]
    positions = torch.tensor(pos, device=DEV, dtype=torch.int64 if D % 32 else torch.int32)
    out = rotate_heads(q, k, rotation, positions if sections else positions[0], q_weight=w["q"], k_weight=w["k"], out_layout=out_layout)
    rng = np.random.default_rng(5)
    pairs = [(n, x, y) for n, x, y in (("q", q, out[0]), ("k", k, out[1])) if x is not None]
    assert (out[1] is None) == (k is None)
    grads = [torch.tensor(rng.standard_normal(y.shape)).to(DT[dtype]).to(DEV) for _, _, y in pairs]
    got = dict(zip((id(t) for t in leaves), torch.autograd.grad([y for _, _, y in pairs], leaves, [strided(g, layout) for g in grads])))
    for (name, x, y), g in zip(pairs, grads):
        weight = None if w[name] is None else wide(w[name])
        want, size = ro.forward(rot, wide(x), pos, weight)
        assert y.dtype == x.dtype and y.shape == x.shape
        if out_layout == "contiguous":
            assert y.is_contiguous()
        elif layout != "odd":
            assert y.stride() == x.stride()
        assert_within(y, want, size * 2.0 ** -19 + np.abs(want) * HALF[dtype] + 1e-7 * (dtype == "f16"), name)
        dx, dw, big, sums = ro.backward(rot, wide(x), wide(g), pos, weight)
        assert got[id(x)].dtype == x.dtype
        assert_within(got[id(x)], dx, big * 2.0 ** -18 + np.abs(dx) * HALF[dtype] + 1e-7 * (dtype == "f16"), "d" + name)
        if dw is not None:
            assert got[id(w[name])].dtype == w[name].dtype
            assert_within(got[id(w[name])], dw, sums * 2.0 ** -14 + np.abs(dw) * HALF[wtype] + 1e-7 * (wtype == "f16"), "d" + name + "_weight")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_far_and_negative_positions(dtype):
    """Angles of positions up to the ends of 32 and beyond of 40 bits: whole turns are left out before anything is rounded."""
    from kerneldev_b200 import Rotation, rotate_heads
    far = [0, 1, -1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7]
    rng = np.random.default_rng(2)
    x = torch.tensor(rng.standard_normal((1, 2, len(far), 64))).to(DT[dtype]).to(DEV)
    rot, rotation = ro.rotation(64), Rotation(64, device=DEV)
    want, size = ro.forward(rot, wide(x), np.array([[far]]))
    # a step is off by 2^-65 turns at most: 2^-34 at 2^31; the angle is cut to 32 bits
    bound = size * (2.0 ** -19 + 2.0 ** -28) + np.abs(want) * HALF[dtype]
    for kind in (torch.int32, torch.int64):
        assert_within(rotate_heads(x, None, rotation, torch.tensor([far], dtype=kind, device=DEV))[0], want, bound, str(kind))
    very = torch.tensor([[2 ** 40 + 3] * len(far)], device=DEV)
    want, size = ro.forward(rot, wide(x), np.array([[[2 ** 40 + 3] * len(far)]]))
    assert_within(rotate_heads(x, None, rotation, very)[0], want, size * (2.0 ** -19 + 2.0 ** -21) + np.abs(want) * HALF[dtype], "2^40")   # 2^40 * 2^-65 turns, and the oracle's 64 bits


def test_positions_by_offsets_by_default_and_for_all_sequences():
    from kerneldev_b200 import Rotation, rotate_heads
    x = torch.randn((3, 2, 5, 32), device=DEV)
    rotation = Rotation(32, device=DEV)
    at = torch.arange(5, device=DEV)
    same = lambda a, b: torch.equal(a[0], b[0])  # noqa: E731
    plain = rotate_heads(x, None, rotation)
    assert same(plain, rotate_heads(x, None, rotation, at[None]))
    assert same(plain, rotate_heads(x, None, rotation, at[None].expand(3, 5).int()))
    assert same(plain, rotate_heads(x, None, rotation, at[None, None].expand(1, 3, 5)))
    assert same(plain, rotate_heads(x, None, rotation, offsets=torch.zeros(3, dtype=torch.int32, device=DEV)))
    off = torch.tensor([7, 0, -4, 9, 9, 9], dtype=torch.int32, device=DEV)
    assert same(rotate_heads(x, None, rotation, off[:3, None] + at), rotate_heads(x, None, rotation, offsets=off[:3]))
    assert same(rotate_heads(x, None, rotation, off[::2, None] + at), rotate_heads(x, None, rotation, offsets=off[::2]))
    # an explicit table of the default's frequencies
    freq = torch.tensor([10000.0 ** (-2.0 * i / 32) for i in range(16)], dtype=torch.float64)
    assert same(plain, rotate_heads(x, None, Rotation(32, frequencies=freq, device=DEV)))


@pytest.mark.parametrize("shape", [(0, 2, 3, 16), (2, 2, 0, 16)])
def test_nothing_to_turn(shape):
    from kerneldev_b200 import Rotation, rotate_heads
    x, w = torch.zeros(shape, device=DEV, requires_grad=True), torch.ones(16, device=DEV, requires_grad=True)
    q, k = rotate_heads(x, x, Rotation(16, device=DEV), q_weight=w)
    assert q.shape == k.shape == shape
    dx, dw = torch.autograd.grad((q.sum() + k.sum()), (x, w))
    assert dx.shape == shape and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_special_rows(dtype):
    """Zeros, infinities and NaN stay in their rows; those of elements that do not turn, in their elements."""
    from kerneldev_b200 import Rotation, rotate_heads
    x = torch.randn((1, 1, 8, 64), device=DEV).to(DT[dtype])
    x[0, 0, 1] = 0
    x[0, 0, 2, 3] = float("nan")
    x[0, 0, 4, 40] = float("inf")
    rotation, w = Rotation(64, 32, device=DEV), torch.ones(64, device=DEV, dtype=DT[dtype])
    y = rotate_heads(x, None, rotation)[0][0, 0]
    bad = torch.zeros((8, 64), dtype=torch.bool, device=DEV)
    bad[2, 3] = bad[2, 19] = bad[4, 40] = True
    assert torch.equal(~torch.isfinite(y), bad) and torch.equal(y[1], torch.zeros_like(y[1]))
    y = rotate_heads(x, None, rotation, q_weight=w)[0][0, 0]
    assert torch.isfinite(y[[0, 1, 3, 5, 6, 7]]).all() and torch.equal(y[1], torch.zeros_like(y[1])) and torch.isnan(y[2]).all()


def test_gradients_that_are_missing_expanded_or_of_another_layout():
    from kerneldev_b200 import Rotation, rotate_heads
    rotation = Rotation(32, device=DEV)
    q, k = (torch.randn((2, 3, 7, 32), device=DEV, requires_grad=True) for _ in range(2))
    w = torch.randn(32, device=DEV, requires_grad=True)
    a, b = rotate_heads(q, k, rotation, q_weight=w, k_weight=w)
    only = torch.autograd.grad(a.sum(), (q, k, w), retain_graph=True)   # k's output has no gradient, q's is one number for all
    assert torch.equal(only[1], torch.zeros_like(k))
    both = torch.autograd.grad((a, b), (q, k, w), (torch.ones_like(a), torch.zeros_like(b)), retain_graph=True)
    for x, y in zip(only, both):
        assert torch.equal(x, y)
    with torch.autograd.graph.save_on_cpu():
        c, d = rotate_heads(q, k, rotation, q_weight=w, k_weight=w)
    for x, y in zip(torch.autograd.grad((c, d), (q, k, w), (torch.ones_like(a), torch.zeros_like(b))), both):
        assert torch.equal(x, y)
    x = torch.randn((1, 1, 1, 32), device=DEV).expand(2, 3, 7, 32).requires_grad_()   # one row for all: its memory is read once a row
    assert torch.equal(rotate_heads(x, None, rotation, out_layout="input")[0], rotate_heads(x.detach().contiguous(), None, rotation)[0])


def test_gradients_of_weights_do_not_vary():
    from kerneldev_b200 import Rotation, rotate_heads
    rotation = Rotation(128, device=DEV)
    q, k = (torch.randn((4, h, 700, 128), device=DEV).bfloat16() for h in (16, 4))
    w = torch.ones(128, device=DEV, requires_grad=True)
    first = None
    for _ in range(5):
        a, b = rotate_heads(q, k, rotation, q_weight=w, k_weight=w)
        g, = torch.autograd.grad((a, b), w, (q, k))
        first = g if first is None else first
        assert torch.equal(g, first)


def test_refusals():
    from kerneldev_b200 import Rotation, rotate_heads
    r, r3 = Rotation(32, device=DEV), Rotation(32, sections=(4, 6, 6), device=DEV)
    x, i = torch.zeros((2, 3, 4, 32), device=DEV), lambda *s: torch.zeros(s, dtype=torch.int64, device=DEV)  # noqa: E731
    w = torch.ones(32, device=DEV)

    def refused(kind, text, *args, **more):
        with pytest.raises(kind, match=text):
            rotate_heads(*args, **more)

    refused(ValueError, "batch, heads", x[0], None, r)
    refused(RuntimeError, "no CPU path", x.cpu(), None, r)
    refused(RuntimeError, "no CPU path", x, x.cpu(), r)
    refused(ValueError, "dtype", x.double(), None, r)
    refused(ValueError, "dtype", x, x.half(), r)
    refused(ValueError, "head_dim", x[..., :16], None, r)
    refused(ValueError, "batch and time", x, x[:1], r)
    refused(ValueError, "batch and time", x, x[:, :, :2], r)
    refused(ValueError, "heads", x[:, :0], None, r)
    refused(ValueError, "exclude", x, None, r, i(2, 4), offsets=i(2).int())
    refused(ValueError, "int64 or int32", x, None, r, i(2, 4).float())
    refused(ValueError, "positions must", x, None, r, i(3, 4))
    refused(ValueError, "positions must", x, None, r, i(2, 5))
    refused(ValueError, "positions must", x, None, r, i(2, 2, 4))
    refused(ValueError, "axes", x, None, r3, i(2, 4))
    refused(ValueError, "needs positions", x, None, r3)
    refused(ValueError, "needs positions", x, None, r3, offsets=i(2).int())
    refused(ValueError, "positions must live", x, None, r, i(2, 4).cpu())
    refused(ValueError, "offsets must", x, None, r, offsets=i(2))
    refused(ValueError, "offsets must", x, None, r, offsets=i(3).int())
    refused(ValueError, "offsets must live", x, None, r, offsets=i(2).int().cpu())
    refused(ValueError, "weights must have", x, None, r, q_weight=w[:16])
    refused(ValueError, "weights must share", x, x, r, q_weight=w, k_weight=w.half())
    refused(ValueError, "weights must live", x, None, r, q_weight=w.cpu())
    refused(ValueError, "k is not", x, None, r, k_weight=w)
    for eps in (-1e-6, float("nan"), float("inf")):
        refused(ValueError, "eps", x, None, r, eps=eps)
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        refused(NotImplementedError, "forward mode", fwad.make_dual(x, x), None, r)


def test_other_streams_and_captured_steps():
    """A step captured once serves every later token: offsets are read at replay. The rotation is let go of by the caller, and replaced in memory."""
    from kerneldev_b200 import Rotation, rotate_heads
    side = torch.cuda.Stream()
    q, k, off = torch.randn((3, 4, 1, 64), device=DEV).bfloat16(), torch.randn((3, 2, 1, 64), device=DEV).bfloat16(), torch.tensor([5, 0, 9], dtype=torch.int32, device=DEV)
    w = torch.randn(64, device=DEV)
    keep = Rotation(64, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):
        rotation = Rotation(64, device=DEV)
        with torch.cuda.stream(side):
            rotate_heads(q, k, rotation, offsets=off, q_weight=w)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = rotate_heads(q, k, rotation, offsets=off, q_weight=w)
        graphs.append((g, out))
        del rotation
    junk = [torch.full((32,), 0x7FFF7FFF, dtype=torch.int64, device=DEV) for _ in range(100)]
    for step in range(3):
        off += step
        q.normal_()
        for g, out in graphs:
            g.replay()
        want = rotate_heads(q, k, keep, offsets=off, q_weight=w)
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    del junk


def test_captured_training_step():
    from kerneldev_b200 import Rotation, rotate_heads
    rotation = Rotation(64, device=DEV)
    q, k = (torch.randn((2, h, 50, 64), device=DEV).half().requires_grad_() for h in (4, 2))
    w = torch.ones(64, device=DEV, requires_grad=True)

    def step():
        a, b = rotate_heads(q, k, rotation, q_weight=w, k_weight=w)
        return (a, b, *torch.autograd.grad((a, b), (q, k, w), (a.detach() * 2, b.detach())))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = step()
    with torch.no_grad():
        q.normal_()
        w.normal_()
    g.replay()
    for x, y in zip(out, step()):
        assert torch.equal(x, y)


def test_captured_backward_beside_an_eager_graph_of_the_same_leaves_is_refused():
    """Not by the end of the process, which is what torch's engine would do. (In a process of its own, for that reason.)"""
    code = """
import torch
from kerneldev_b200 import Rotation, rotate_heads
rotation = Rotation(32, device="cuda")
q, w = torch.randn((1, 2, 4, 32), device="cuda", requires_grad=True), torch.ones(32, device="cuda", requires_grad=True)
eager, _ = rotate_heads(q, None, rotation, q_weight=w)
g = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(g):
        y, _ = rotate_heads(q, None, rotation, q_weight=w)
        y.sum().backward()
except RuntimeError as e:
    print("refused:", "cannot be captured" in str(e))
torch.cuda.synchronize()
eager.sum().backward()
print("alive:", torch.isfinite(q.grad).all().item())
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "refused: True" in r.stdout and "alive: True" in r.stdout, r.stdout + r.stderr


def test_captured_backward_for_named_leaves_beside_an_eager_graph_is_refused():
    """backward(inputs=...) adds to the leaves that it names: refused too, where one of those belongs to the eager graph, and captured where none does. (In a process of its own, as above.)"""
    code = """
import torch
from kerneldev_b200 import Rotation, rotate_heads
rotation = Rotation(32, device="cuda")
q, w = torch.randn((1, 2, 4, 32), device="cuda", requires_grad=True), torch.ones(32, device="cuda", requires_grad=True)
fresh = torch.ones(32, device="cuda", requires_grad=True)
eager, _ = rotate_heads(q, None, rotation, q_weight=w)
g = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(g):
        y, _ = rotate_heads(q, None, rotation, q_weight=fresh)
        y.sum().backward(inputs=[q])
except RuntimeError as e:
    print("refused:", "cannot be captured" in str(e))
torch.cuda.synchronize()
fresh = torch.ones(32, device="cuda", requires_grad=True)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y, _ = rotate_heads(q, None, rotation, q_weight=fresh)
    y.sum().backward(inputs=[fresh])
g.replay()
torch.cuda.synchronize()
eager.sum().backward()
print("alive:", torch.equal(fresh.grad, w.grad) and torch.isfinite(q.grad).all().item())
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "refused: True" in r.stdout and "alive: True" in r.stdout, r.stdout + r.stderr


def test_rotation_then_attention_trains_as_the_definition_says():
    """rotate_heads and flash_attention together: causal attention of turned and normalised heads, and the gradients of everything ahead of it."""
    from kerneldev_b200 import Rotation, flash_attention, rotate_heads
    torch.manual_seed(0)
    B, H, T, D = 1, 2, 150, 64
    rotation = Rotation(D, base=500.0, device=DEV)
    q, k, v = (torch.randn((B, T, H, D), device=DEV).half().transpose(1, 2).requires_grad_() for _ in range(3))
    w = (1 + 0.2 * torch.randn(D, device=DEV)).requires_grad_()
    a, b = rotate_heads(q, k, rotation, q_weight=w, k_weight=w, out_layout="input")
    o = flash_attention(a, b, v, causal=True, out_layout="input")
    do = torch.randn_like(o)
    got = torch.autograd.grad(o, (q, k, v, w), do)
    # the same in 64 bits
    q6, k6, v6 = (x.detach().double().cpu().requires_grad_() for x in (q, k, v))
    w6 = w.detach().double().cpu().requires_grad_()
    angle = torch.tensor(ro.angles(ro.rotation(D, base=500.0), np.arange(T)[None, None]))[:, None]

    def turned(x):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w6
        e, f = y[..., :D // 2], y[..., D // 2:]
        return torch.cat((e * angle.cos() - f * angle.sin(), f * angle.cos() + e * angle.sin()), -1)

    s = turned(q6) @ turned(k6).transpose(2, 3) / D ** 0.5
    p = s.masked_fill(~torch.ones((T, T), dtype=torch.bool).tril(), -np.inf).softmax(-1)
    want_o = p @ v6
    want = torch.autograd.grad(want_o, (q6, k6, v6, w6), do.double().cpu())
    # operands, probabilities and their gradients are halves: the operator's own tolerance, and for the weight's gradient, a sum over 300 rows, that of each
    assert float((o.double().cpu() - want_o).abs().max()) < 2e-2
    for name, x, y in zip("qkvw", got, want):
        err = (x.double().cpu() - y).abs()
        assert bool((err <= 2e-2 * (300 if name == "w" else 1) + 1e-2 * y.abs()).all()), name
        assert float(err.norm() / y.norm()) < 1e-2, name


def test_offsets_beyond_32_bits():
    """Heads 2**32 elements apart."""
    from kerneldev_b200 import Rotation, rotate_heads
    free, _ = torch.cuda.mem_get_info()
    if free < 2 ** 34 + 2 ** 30:
        pytest.skip("needs 17 GB")
    memory = torch.empty(2 ** 32 + 4096, dtype=torch.bfloat16, device=DEV)
    x, grad = [memory.as_strided((1, 2, 3, 64), (2 ** 32, 2 ** 32, 64, 1), at).normal_() for at in (0, 2048)]
    w = torch.ones(64, device=DEV, requires_grad=True)
    rotation = Rotation(64, device=DEV)
    y, _ = rotate_heads(x, None, rotation, q_weight=w)
    z, _ = rotate_heads(x.contiguous(), None, rotation, q_weight=w)
    assert torch.equal(y, z)
    assert torch.equal(torch.autograd.grad(y, w, grad)[0], torch.autograd.grad(z, w, grad.contiguous())[0])


def test_two_calls_at_once_on_two_threads():
    """Each with a stream and leaves of its own."""
    import threading
    from kerneldev_b200 import Rotation, rotate_heads
    rotation = Rotation(64, device=DEV)
    work, errors = [], []
    for i in range(2):
        q = torch.randn((2, 4, 300 + i, 64), device=DEV).bfloat16().requires_grad_()
        w = torch.randn(64, device=DEV, requires_grad=True)
        y, _ = rotate_heads(q, None, rotation, q_weight=w)
        work.append((q, w, y.detach(), torch.autograd.grad(y, (q, w), y.detach())))
    torch.cuda.synchronize()

    def go(q, w, y, grads):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    z, _ = rotate_heads(q, None, rotation, q_weight=w)
                    got = torch.autograd.grad(z, (q, w), y)
                torch.cuda.current_stream().synchronize()
                assert torch.equal(z, y) and all(torch.equal(a, b) for a, b in zip(got, grads))
        except BaseException as e:   # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=go, args=x) for x in work]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors


def test_second_derivatives_have_no_history():
    """As those of flash_attention: with create_graph the gradients are plain tensors."""
    from kerneldev_b200 import Rotation, rotate_heads
    q = torch.randn((1, 1, 3, 16), device=DEV, requires_grad=True)
    y, _ = rotate_heads(q, None, Rotation(16, device=DEV))
    g, = torch.autograd.grad(y.square().sum(), q, create_graph=True)
    assert not g.requires_grad
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):   # what a backward reads again may not change
        w = torch.ones(16, device=DEV, requires_grad=True)
        pos = torch.zeros((1, 3), dtype=torch.int32, device=DEV)
        y, _ = rotate_heads(q, None, Rotation(16, device=DEV), pos, q_weight=w)
        pos += 1
        torch.autograd.grad(y.sum(), q)
