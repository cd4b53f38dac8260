"""The gated linear recurrence (csrc/recurrence.hip) against a loop in 64 bits, gradients by the formulas in 64 bits.

fp32 errors: f and 1 - f carry 2^-21 relative (exp of an argument rounded at |gate| 2^-24, one reciprocal); a state is a sum of terms f..f u, each a product of up
to t factors, but |error| obeys e_t <= f e_{t-1} + 2^-21 (2 |h_t| + |u_t|), the same recurrence: it is run on the magnitudes (`e` below) with 2^-19 to cover the
regrouping of the products."""
import pytest
import torch

from seq_util import DTYPES, close, lengths, rounded

pytestmark = pytest.mark.gpu
E = 2.0 ** -19


def _reference(x, gate, h0, dh, dlast, lens, reverse, gain):
    x, gate, h0, dh, dlast = (t.detach().double().cpu() for t in (x, gate, h0, dh, dlast))
    B, T, C = x.shape
    f, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    k = keep if gain == "convex" else torch.ones_like(f)
    live = (torch.arange(T)[None] < lens.cpu()[:, None]).double()[..., None] if lens is not None else torch.ones(B, T, 1, dtype=torch.float64)
    zero = torch.zeros_like(x)
    x, dh = torch.where(live > 0, x, zero), torch.where(live > 0, dh, zero)
    f, k, keep = torch.where(live > 0, f, torch.ones_like(f)), torch.where(live > 0, k, zero), torch.where(live > 0, keep, zero)
    order = list(range(T))[::-1] if reverse else list(range(T))
    h, e = h0, E * h0.abs()
    hs, before, es, eb = zero.clone(), zero.clone(), zero.clone(), zero.clone()
    for t in order:
        before[:, t], eb[:, t] = h, e
        u = k[:, t] * x[:, t]
        h, e = f[:, t] * h + u, f[:, t] * (e + E * h.abs()) + E * u.abs()
        hs[:, t], es[:, t] = h, e
    g, ge = dlast.clone(), E * dlast.abs()
    tot, tote = zero.clone(), zero.clone()
    for t in order[::-1]:
        g, ge = g + dh[:, t], ge + E * dh[:, t].abs()
        tot[:, t], tote[:, t] = g, ge
        g, ge = f[:, t] * g, f[:, t] * (ge + E * g.abs())
    pull, pulle = (before - x, eb + 2.0 ** -23 * (before.abs() + x.abs())) if gain == "convex" else (before, eb)
    s = f * keep
    outs = (hs * live, h, tot * k, tot * pull * s, g)
    errs = (es * live, e, tote * k + E * (tot * k).abs(), (tote * pull.abs() + tot.abs() * pulle + E * (tot * pull).abs()) * s, ge)
    return outs, errs


def _run(x, gate, h0, dh, dlast, lens=None, reverse=False, gain="convex"):
    from xva_trainer_amd import seq_ops as S
    x, gate = x.detach().requires_grad_(True), gate.detach().requires_grad_(True)
    h0 = h0.detach().requires_grad_(True)
    h, last = S.gated_recurrence(x, gate, h0, lens=lens, reverse=reverse, gain=gain)
    got = (h.detach(), last.detach()) + torch.autograd.grad((h, last), (x, gate, h0), (dh, dlast))
    ref, err = _reference(x, gate, h0, dh, dlast, lens, reverse, gain)
    for name, o, r, e in zip(("h", "last", "dx", "dgate", "dh0"), got, ref, err):
        close(o, r, rounded(r, o.dtype, e + 1e-37), name)
    with torch.no_grad():
        again = S.gated_recurrence(x, gate, h0, lens=lens, reverse=reverse, gain=gain)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
    return got


def _data(B, T, C, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000 + B * 77 + T * 13 + C)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return n(B, T, C).to(DTYPES[dt]), (2 + 1.5 * n(B, T, C)).to(DTYPES[dt]), n(B, C), n(B, T, C).to(DTYPES[dt]), n(B, C)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("ragged", [None, "some", "empty"])
@pytest.mark.parametrize("B,T,C", [(1, 1, 1), (64, 1, 128), (3, 7, 5), (2, 8, 64), (2, 9, 130), (4, 127, 33), (3, 128, 2), (2, 129, 256), (3, 860, 48), (1, 3000, 7),
                                   (2, 2500, 128), (5, 1, 2048),
                                   # rows of 32 bytes: one tile, several, an odd width
                                   (16, 200, 128), (32, 1300, 65), (9, 1100, 448)])
def test_shapes(dt, reverse, ragged, B, T, C):
    lens = lengths(B, T, ragged)
    got = _run(*_data(B, T, C, dt), lens=lens.cuda() if lens is not None else None, reverse=reverse, gain="unit" if C % 2 else "convex")
    if lens is not None:
        dead = torch.arange(T)[None] >= lens[:, None]
        assert all((got[i].cpu()[dead] == 0).all() for i in (0, 2, 3))


@pytest.mark.parametrize("gain", ["convex", "unit"])
@pytest.mark.parametrize("B,T,C", [(2, 300, 64), (1, 5000, 16)])
def test_gates_at_their_ends(gain, B, T, C):
    """Gates that keep or drop everything, among them ones whose exponential leaves fp32."""
    x, gate, h0, dh, dlast = _data(B, T, C, "fp32", seed=2)
    ends = torch.tensor([-3e38, -200.0, -100.0, -30.0, 0.0, 12.0, 100.0, 3e38], device="cuda")
    gate = torch.where(torch.rand_like(gate) < 0.2, ends[torch.randint(0, 8, gate.shape, device="cuda")], gate - 2)
    _run(x, gate, h0, dh, dlast, gain=gain)


def test_not_numbers_stay():
    from xva_trainer_amd import seq_ops as S
    x, gate, h0, _, _ = _data(1, 40, 4, "fp32", seed=3)
    gate[0, 10, 1] = float("nan")
    x[0, 20, 2] = float("inf")
    h, last = S.gated_recurrence(x, gate, h0)
    assert torch.isnan(h[0, 10:, 1]).all() and torch.isfinite(h[0, :10]).all() and torch.isfinite(h[0, :, 0]).all()
    assert torch.isinf(h[0, 20, 2]) and torch.isnan(last[0, 1])


@pytest.mark.parametrize("reverse", [False, True])
def test_steps_continue_a_sequence(reverse):
    """One token at a time, the last state handed on, is the whole sequence at once; so are two halves."""
    from xva_trainer_amd import seq_ops as S
    x, gate, h0, _, _ = _data(3, 40, 24, "fp32", seed=4)
    whole, last = S.gated_recurrence(x, gate, h0, reverse=reverse)
    state, outs = h0, [None] * 40
    for t in (range(39, -1, -1) if reverse else range(40)):
        outs[t], state = S.gated_recurrence(x[:, t:t + 1], gate[:, t:t + 1], state, reverse=reverse)
    steps = torch.cat(outs, 1)
    # both are within the reference's error of each other
    (ref, rl, *_), (e, el, *_) = _reference(x, gate, h0, torch.zeros_like(x), torch.zeros_like(h0), None, reverse, "convex")
    close(steps, ref, rounded(ref, torch.float32, e), "steps")
    close(state, rl, rounded(rl, torch.float32, el), "last")
    close(whole, ref, rounded(ref, torch.float32, e), "whole")


@pytest.mark.parametrize("T", [1, 30, 700])
def test_what_lies_behind_an_item_is_not_read(T):
    from xva_trainer_amd import seq_ops as S
    for reverse in (False, True):
        x, gate, h0, dh, dlast = _data(4, T, 40, "bf16", seed=5)
        lens = torch.tensor([T, T // 2, 0, min(1, T)], dtype=torch.int32)
        dead = (torch.arange(T)[None] >= lens[:, None]).cuda()[..., None]
        outs = []
        for fill in (0.0, float("nan"), float("inf")):
            a, b = (t.masked_fill(dead, fill).requires_grad_(True) for t in (x, gate))
            h, last = S.gated_recurrence(a, b, h0, lens=lens.cuda(), reverse=reverse)
            outs.append((h, last) + torch.autograd.grad((h, last), (a, b), (dh.masked_fill(dead, fill), dlast)))
        for other in outs[1:]:
            assert all(torch.equal(p, q) for p, q in zip(outs[0], other))
        assert torch.equal(outs[0][1][2], h0[2])                     # an empty item hands its state on


def test_no_first_state_and_parts_of_the_gradient():
    from xva_trainer_amd import seq_ops as S
    x, gate, h0, dh, dlast = _data(2, 300, 32, "fp32", seed=6)
    x.requires_grad_(True), gate.requires_grad_(True)
    h, last = S.gated_recurrence(x, gate)
    a = torch.autograd.grad((h, last), (x, gate), (dh, dlast), retain_graph=True)
    b = torch.autograd.grad(h, (x, gate), dh, retain_graph=True)
    c = torch.autograd.grad(last, (x, gate), dlast)
    for p, q, r in zip(a, b, c):                                     # linear in the gradients: three roundings of sums of the same terms
        assert (p - q - r).abs().max().item() < 2.0 ** -17 * (q.abs().max() + r.abs().max()).item()
    z, zl = S.gated_recurrence(x, gate, torch.zeros_like(h0))
    assert torch.equal(z, h) and torch.equal(zl, last)


def test_the_gradient_by_differences():
    from xva_trainer_amd import seq_ops as S
    x, gate, h0, dh, dlast = _data(1, 200, 8, "fp32", seed=7)
    gate.requires_grad_(True)
    h, last = S.gated_recurrence(x, gate, h0)
    grad, = torch.autograd.grad((h, last), gate, (dh, dlast))
    step = torch.randn_like(gate)
    d = 2.0 ** -7
    with torch.no_grad():
        def f(s):
            o, l = S.gated_recurrence(x, gate + s * d * step, h0)
            return (o.double() * dh).sum() + (l.double() * dlast).sum()
        diff = ((f(1) - f(-1)) / (2 * d)).item()
    size = (grad.abs() * step.abs()).sum().item() + dh.abs().sum().item()
    assert abs(diff - (grad.double() * step).sum().item()) < size * (16 * d * d + 2.0 ** -20 / d)


def test_views_and_odd_addresses():
    store = torch.randn(3, 50, 200, device="cuda").bfloat16()
    _, _, h0, _, dl = _data(3, 50, 64, "bf16")
    for x, gate in ((store[:, :, :64], store[:, :, 64:128]), (store[:, :, 1:65], store[:, :, 66:130]), (store[:, 5:40], store[:, 4:39]),
                    (store[:, ::2, :64], store[:, 1::2, :64]), (store.transpose(0, 1)[:3, :, :10], store.transpose(0, 1)[3:6, :, 20:30]),
                    (store.transpose(1, 2)[:, :64, :32], store.transpose(1, 2)[:, 64:128, :32])):
        B, T, C = x.shape
        n = torch.randn(B, C, device="cuda")
        _run(x, gate, n, torch.randn(B, T, C, device="cuda").bfloat16(), n.flip(0))
    # a gradient that comes with strides of its own
    from xva_trainer_amd import seq_ops as S
    x, gate = (torch.randn(2, 30, 6, device="cuda", requires_grad=True) for _ in range(2))
    h, _ = S.gated_recurrence(x, gate)
    g1, = torch.autograd.grad(h.sum(), x, retain_graph=True)
    g2, = torch.autograd.grad(h, x, torch.ones_like(h))
    assert torch.equal(g1, g2)


def test_empty_graph_and_repeats():
    from xva_trainer_amd import seq_ops as S
    for shape in ((0, 4, 8), (3, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        h0 = torch.randn(shape[0], 8, device="cuda", requires_grad=True)
        h, last = S.gated_recurrence(x, x.detach(), h0)
        assert h.shape == shape and torch.equal(last, h0)
        g, = torch.autograd.grad(last.sum(), h0)
        assert (g == 1).all()
    for B, T in ((4, 1), (1, 4000)):
        x, gate, h0, dh, dlast = _data(B, T, 32, "bf16", seed=8)
        x.requires_grad_(True), gate.requires_grad_(True), h0.requires_grad_(True)
        def step():
            h, last = S.gated_recurrence(x, gate, h0)
            return (h.detach(), last.detach()) + torch.autograd.grad((h, last), (x, gate, h0), (dh, dlast))
        assert all(torch.equal(p, q) for p, q in zip(step(), step()))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for turn in range(4):
            with torch.no_grad():
                x.normal_(), h0.normal_(), dh.normal_()
            graph.replay()
            eager = step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, eager)), turn


def test_refusals():
    from xva_trainer_amd import seq_ops as S
    x = torch.zeros(2, 3, 8, device="cuda")
    for bad in (lambda: S.gated_recurrence(x, x[:, :2]), lambda: S.gated_recurrence(x, x.half()), lambda: S.gated_recurrence(x.double(), x.double()),
                lambda: S.gated_recurrence(x[0], x[0]), lambda: S.gated_recurrence(x, x, torch.zeros(2, 7, device="cuda")), lambda: S.gated_recurrence(x, x, gain="half"),
                lambda: S.gated_recurrence(x, x, lens=torch.tensor([1], device="cuda")), lambda: S.gated_recurrence(x, x, lens=torch.tensor([1, 2])),
                lambda: S.gated_recurrence(x.cpu(), x.cpu()), lambda: S.gated_recurrence(x, x, torch.zeros(2, 8))):
        with pytest.raises(S.XvaError):
            bad()
