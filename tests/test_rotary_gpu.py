"""Rotary positions (csrc/rotary.hip) against the rotation in 64 bits.

An output is m (a cos - b sin): cos and sin carry 2^-24 of the reduced turn (half a step of fp32 times pi, under 2^-22 of the angle's unit) and sincospif's own
2 units; with the three roundings of the products that is under 2^-20 (|a| + |b|) m, before the one rounding to the tensors' type."""
import math

import pytest
import torch

from seq_util import DTYPES, close, rounded

pytestmark = pytest.mark.gpu


def _reference(x, pos, plan, inverse=False):
    x = x.detach().double().cpu()
    w = torch.tensor(plan.frequencies, dtype=torch.float64)
    ang = pos.double().cpu()[..., None, None] * w * (-1.0 if inverse else 1.0)
    c, s = ang.cos() * plan.gain, ang.sin() * plan.gain
    n, out, err = w.numel(), x.clone(), torch.zeros_like(x)
    lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if plan.interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., lo], x[..., hi]
    out[..., lo], out[..., hi] = a * c - b * s, b * c + a * s
    err[..., lo] = err[..., hi] = (a.abs() + b.abs()) * plan.gain * 2.0 ** -20
    return out, err


def _check(got, x, pos, plan, what, inverse=False):
    ref, err = _reference(x, pos, plan, inverse)
    # the reference's own angle: p w in 64 bits is off by 2^-53 of itself
    far = float(pos.abs().max()) * 2.0 ** -52
    close(got, ref, rounded(ref, got.dtype, err * (1.0 + far * 2.0 ** 20)), what)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,T,H,Hk,D,rd", [(2, 5, 3, 1, 64, 64), (1, 1, 4, 4, 128, 64), (3, 37, 2, 2, 96, 96), (2, 130, 1, 1, 62, 62), (1, 70, 5, 3, 10, 6),
                                           (4, 9, 2, 1, 7, 2), (1, 3, 1, 1, 2, 2), (2, 2100, 2, 1, 40, 20), (1, 5, 2, 1, 8192, 8192), (1, 4, 300, 7, 16, 16)])
def test_forward_and_gradient(dt, inter, B, T, H, Hk, D, rd):
    from xva_trainer_amd import seq_ops as S
    torch.manual_seed(B * T + D)
    plan = S.RotaryPlan(rd, interleaved=inter)
    q = torch.randn(B, T, H, D, device="cuda").to(DTYPES[dt]).requires_grad_(True)
    k = torch.randn(B, T, Hk, D, device="cuda").to(DTYPES[dt]).requires_grad_(True)
    pos = torch.randint(0, 5000, (B, T), device="cuda")
    qo, ko = S.rotary(plan, q, k, positions=pos)
    _check(qo, q, pos, plan, "q"), _check(ko, k, pos, plan, "k")
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    _check(gq, dq, pos, plan, "dq", True), _check(gk, dk, pos, plan, "dk", True)


@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 16.0)])
@pytest.mark.parametrize("first", [0, 100003, 2 ** 31 - 40, 2 ** 40 + 12345, -77])
def test_far_positions_and_scalings(scaling, factor, first):
    from xva_trainer_amd import seq_ops as S
    torch.manual_seed(3)
    plan = S.RotaryPlan(64, scaling=scaling, factor=factor)
    q = torch.randn(1, 33, 2, 64, device="cuda")
    pos = torch.arange(first, first + 33, device="cuda")
    _check(S.rotary(plan, q, positions=pos), q, pos[None], plan, "q")


def test_the_gradient_by_differences():
    from xva_trainer_amd import seq_ops as S
    torch.manual_seed(4)
    plan = S.RotaryPlan(6, interleaved=True, scaling="yarn", factor=2.0)
    q, g = torch.randn(1, 4, 1, 8, device="cuda", requires_grad=True), torch.randn(1, 4, 1, 8, device="cuda")
    grad, = torch.autograd.grad(S.rotary(plan, q), q, g)
    step = torch.randn_like(q)
    with torch.no_grad():                       # the map is linear: a difference of any size is exact but for roundings of 2^-20 of the values
        diff = (S.rotary(plan, q + step) - S.rotary(plan, q - step)).double() / 2
    assert abs((diff * g).sum().item() - (grad * step).double().sum().item()) < 64 * 8 * 2.0 ** -20


@pytest.mark.parametrize("shape", [(7,), (1, 7), (3, 1), (1,), (3, 7)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_positions_of_any_shape(shape, dtype):
    from xva_trainer_amd import seq_ops as S
    plan = S.RotaryPlan(16)
    q = torch.randn(3, 7, 2, 16, device="cuda")
    pos = torch.randint(0, 999, shape, device="cuda", dtype=dtype)
    _check(S.rotary(plan, q, positions=pos), q, pos.expand(3, 7) if pos.dim() == 2 else pos.expand(7)[None].expand(3, 7), plan, "q")
    _check(S.rotary(plan, q), q, torch.arange(7)[None].expand(3, 7), plan, "default")


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_strided_views_and_in_place(dt):
    """q and k as slices of one projection, with odd offsets (narrow accesses); in place nothing else of the projection changes."""
    from xva_trainer_amd import seq_ops as S
    torch.manual_seed(5)
    for start, D, rd in ((0, 64, 64), (0, 64, 32), (1, 62, 30), (3, 33, 8)):
        plan = S.RotaryPlan(rd)
        whole = torch.randn(2, 19, 5 * D + 8, device="cuda").to(DTYPES[dt])
        before = whole.clone()
        q = whole[:, :, start:start + 3 * D].unflatten(2, (3, D))
        k = whole[:, :, start + 3 * D:start + 4 * D].unflatten(2, (1, D))
        pos = torch.randint(0, 300, (2, 19), device="cuda")
        qo, ko = S.rotary(plan, q, k, positions=pos)
        _check(qo, q, pos, plan, "q"), _check(ko, k, pos, plan, "k")
        tr = q.transpose(1, 2).contiguous().transpose(1, 2)                 # heads outside rows
        assert torch.equal(S.rotary(plan, tr, positions=pos), qo)
        S.rotary(plan, q, k, positions=pos, inplace=True)
        assert torch.equal(q, qo) and torch.equal(k, ko)
        rest = torch.ones_like(whole, dtype=torch.bool)
        rest[:, :, start:start + 4 * D] = False
        assert torch.equal(whole[rest], before[rest])


def test_empty_and_graph_and_stream():
    from xva_trainer_amd import seq_ops as S
    plan = S.RotaryPlan(32)
    assert S.rotary(plan, torch.zeros(0, 5, 2, 32, device="cuda")).shape == (0, 5, 2, 32)
    assert S.rotary(plan, torch.zeros(2, 0, 2, 32, device="cuda")).shape == (2, 0, 2, 32)
    q, k = torch.randn(4, 1, 8, 32, device="cuda"), torch.randn(4, 1, 2, 32, device="cuda")
    pos = torch.randint(0, 100, (4, 1), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        S.rotary(plan, q, k, positions=pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = S.rotary(plan, q, k, positions=pos)
    for turn in range(4):
        q.normal_(), k.normal_(), pos.random_(0, 1000)
        graph.replay()
        eager = S.rotary(plan, q, k, positions=pos)
        torch.cuda.synchronize()
        assert torch.equal(qo, eager[0]) and torch.equal(ko, eager[1]), turn


def test_in_place_refuses_shared_memory_and_tells_autograd():
    from xva_trainer_amd import seq_ops as S
    plan = S.RotaryPlan(32)
    q = torch.randn(2, 3, 4, 32, device="cuda")
    for bad in (lambda: S.rotary(plan, q, q, inplace=True), lambda: S.rotary(plan, q[:1].expand(2, 3, 4, 32), inplace=True),
                lambda: S.rotary(plan, q, q[:, :, :1].expand(2, 3, 2, 32), inplace=True)):
        with pytest.raises(S.XvaError):
            bad()
    with torch.no_grad():
        one, two = S.rotary(plan, q, q)                                  # read only, the same tensor may come twice
    assert torch.equal(one, two)
    w = torch.ones(32, device="cuda", requires_grad=True)
    y = (q * w).sum()                                                    # saves q
    S.rotary(plan, q, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals():
    from xva_trainer_amd import seq_ops as S
    plan = S.RotaryPlan(32)
    q = torch.zeros(2, 3, 2, 32, device="cuda")
    for bad in (lambda: S.rotary(plan, q[0]), lambda: S.rotary(plan, q, q.half()), lambda: S.rotary(plan, q[..., :16]), lambda: S.rotary(plan, q.double()),
                lambda: S.rotary(plan, q, positions=torch.zeros(3, 3, device="cuda", dtype=torch.int64)),
                lambda: S.rotary(plan, q, positions=torch.zeros(2, 3, device="cuda")), lambda: S.rotary(plan, q, positions=torch.zeros(2, 3, dtype=torch.int64)),
                lambda: S.rotary(plan, q.clone().requires_grad_(True), inplace=True), lambda: S.rotary(plan, q.cpu()), lambda: S.rotary(plan, q, q[:1])):
        with pytest.raises(S.XvaError):
            bad()
    assert math.isclose(S.RotaryPlan(8, gain=2.0).gain, 2.0)


def test_in_place_refuses_views_that_overlap():
    """Views that are not dense: heads of one projection that lie on each other, and windows over it."""
    from xva_trainer_amd import seq_ops as S
    plan = S.RotaryPlan(32)
    whole = torch.randn(2, 5, 8 * 32 + 3, device="cuda")
    heads = lambda a, n: whole[..., a:a + n * 32].unflatten(-1, (n, 32))
    for bad in (lambda: S.rotary(plan, heads(0, 5), heads(4 * 32, 2), inplace=True), lambda: S.rotary(plan, heads(0, 4), heads(4 * 32 - 1, 2), inplace=True),
                lambda: S.rotary(plan, whole.as_strided((2, 5, 4, 32), (1295, 259, 31, 1)), inplace=True)):
        with pytest.raises(S.XvaError, match="inplace"):
            bad()
    # each head's query beside its key, heads outside rows, and different projections
    pairs = whole[..., :256].unflatten(-1, (4, 2, 32))
    want = S.rotary(plan, pairs[..., 0, :], pairs[..., 1, :])
    got = S.rotary(plan, pairs[..., 0, :], pairs[..., 1, :], inplace=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    cache = torch.randn(2, 6, 50, 32, device="cuda").transpose(1, 2)
    want = S.rotary(plan, cache[:, 7:12, :4], cache[:, 7:12, 4:])
    got = S.rotary(plan, cache[:, 7:12, :4], cache[:, 7:12, 4:], inplace=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 3.0), ("yarn", 16.0)])
@pytest.mark.parametrize("first", [2 ** 31 - 40, 2 ** 40 + 12345, -2 ** 42 - 77, 2 ** 44])
def test_positions_that_a_double_cannot_turn(scaling, factor, first):
    """Angles by integers: position times the frequency in 60 digits, modulo a turn.  Allowed beside fp32's own 2^-20 (|a| + |b|): p times half a unit of the table,
    p 2^-65 turns, 2^-18 radians at 2^44 - where a frequency in double would be off by 2^-12 of a turn."""
    from decimal import Decimal as D, getcontext, localcontext

    from xva_trainer_amd import seq_ops as S
    torch.manual_seed(6)
    rd = 64
    plan = S.RotaryPlan(rd, scaling=scaling, factor=factor)
    q = torch.randn(1, 9, 2, rd, device="cuda")
    pos = torch.arange(first, first + 9, device="cuda")
    with localcontext():
        getcontext().prec = 80
        pi, ang = D("3.14159265358979323846264338327950288419716939937510582097494459230781640628620900"), []
        for p in pos.tolist():
            row = []
            for i in range(rd // 2):
                f = D(10000) ** (D(-2 * i) / D(rd))
                if scaling == "linear":
                    f = f / D(factor)
                elif scaling == "yarn":
                    pair = lambda turns: rd * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
                    low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rd - 1)
                    ramp = min(max(D(i - low) / D(max(high - low, 1e-3)), D(0)), D(1))
                    f = f * (1 - ramp) + f / D(factor) * ramp
                turn = D(p) * f / (2 * pi)
                row.append(float((turn - turn.to_integral_value()) * 2 * pi))
            ang.append(row)
    ang = torch.tensor(ang, dtype=torch.float64)[None, :, None]
    x, n = q.double().cpu(), rd // 2
    a, b = x[..., :n], x[..., n:]
    c, s = ang.cos() * plan.gain, ang.sin() * plan.gain
    ref = torch.cat((a * c - b * s, b * c + a * s), -1)
    size = (a.abs() + b.abs()) * plan.gain
    err = torch.cat((size, size), -1) * (2.0 ** -20 + abs(first) * 2.0 ** -65 * 2 * math.pi * 1.01)
    close(S.rotary(plan, q, positions=pos), ref, rounded(ref, q.dtype, err), "q")
