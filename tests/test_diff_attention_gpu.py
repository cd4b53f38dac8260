"""Differential attention (csrc/diff_attention.hip) against the formulas in 64 bits.

Roundings, u half a step of the 16-bit type (2^-8 bf16, 2^-11 fp16): each softmax weight is rounded once before it meets V, so an output is off by u (P_1 + |lam| P_2) |V|;
the maps' own outputs, from which D comes, by that and one more rounding; each dS = P o (dP - D) by u of itself and P times D's error; P_1 - lam P_2 by u of itself;
every result by u of itself.  fp32 work (scores, exponentials, sums): E of the magnitudes that meet."""
import math

import pytest
import torch

from seq_util import DTYPES, HALF, TINY, close, lengths

pytestmark = pytest.mark.gpu
E = 2.0 ** -15      # scores of size |q| |k| sqrt(d) ~ 20 carry 20 x 2^-22 absolute into the exponent, with the roundings of the exponential and of the sums


def _reference(q, k, v, lam, dout, ql, kl, causal, scale):
    q, k, v, lam, dout = (t.detach().double().cpu() for t in (q, k, v, lam, dout))
    u, tiny = HALF[_reference.dtype], TINY[_reference.dtype]
    B, Tq, H, _, d = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    out, dq, dk, dv, dl = torch.zeros_like(dout), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(lam)
    eo, eq, ek, ev, el = (torch.zeros_like(t) for t in (out, dq, dk, dv, dl))
    for b in range(B):
        nq, nk = (Tq if ql is None else int(ql[b])), (Tk if kl is None else int(kl[b]))
        if nq == 0 or nk == 0:
            continue
        see = torch.ones(nq, nk, dtype=torch.bool)
        if causal:
            see = torch.arange(nk)[None] <= torch.arange(nq)[:, None] + nk - nq
        for h in range(H):
            hk = h // (H // Hk)
            V, g = v[b, :nk, hk], dout[b, :nq, h]
            P = []
            for m in range(2):
                s = (q[b, :nq, h, m] @ k[b, :nk, hk, m].T * scale).masked_fill(~see, -math.inf)
                P.append(torch.nan_to_num(torch.softmax(s, -1), nan=0.0))
            l, la = lam[h], lam[h].abs()
            both, size = P[0] - l * P[1], P[0] + la * P[1]
            out[b, :nq, h] = both @ V
            eo[b, :nq, h] = (u + E) * (size @ V.abs()) + tiny * (1 + la) * (see.double() @ V.abs())
            dP = g @ V.T
            dl[h] -= (P[1] * dP).sum()
            el[h] += E * (P[1] * (g.abs() @ V.abs().T)).sum()
            dv[b, :nk, hk] += both.T @ g
            ev[b, :nk, hk] += (u * both.abs() + E * size + tiny).T @ g.abs()
            for m, c in ((0, torch.ones(())), (1, -l)):
                D = (P[m] * dP).sum(-1, keepdim=True)
                gv = g.abs() @ V.abs().T
                eD = ((2 * u + E) * (P[m] * gv).sum(-1, keepdim=True)) + 2 * tiny * g.abs().sum(-1, keepdim=True) * (1 + V.abs().max() * see.sum(-1, keepdim=True))
                dS = c * P[m] * (dP - D)
                eS = c.abs() * P[m] * (eD + E * (gv + D.abs() + gv.mul(P[m]).sum(-1, keepdim=True))) + u * dS.abs() + tiny * (see.double())
                dq[b, :nq, h, m] = scale * dS @ k[b, :nk, hk, m]
                eq[b, :nq, h, m] = scale * eS @ k[b, :nk, hk, m].abs()
                dk[b, :nk, hk, m] += scale * dS.T @ q[b, :nq, h, m]
                ek[b, :nk, hk, m] += scale * eS.T @ q[b, :nq, h, m].abs()
    refs, errs = (out, dq, dk, dv), (eo, eq, ek, ev)
    return refs + (dl,), tuple(u * (r.abs() + e) + tiny + 1.01 * e for r, e in zip(refs, errs)) + (el + E * dl.abs(),)


def _data(B, Tq, Tk, H, Hk, d, dt, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000 + B * 77 + Tq * 13 + Tk * 7 + d)
    n = lambda *s: (torch.randn(*s, device="cuda", generator=g) * size).to(DTYPES[dt])
    return n(B, Tq, H, 2, d), n(B, Tk, Hk, 2, d), n(B, Tk, Hk, 2 * d), 0.5 + 0.2 * torch.randn(H, device="cuda", generator=g), n(B, Tq, H, 2 * d)


def _run(q, k, v, lam, dout, ql=None, kl=None, causal=False, scale=None):
    from xva_trainer_amd import seq_ops as S
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    cuda = lambda t: t.cuda() if t is not None else None
    out = S.differential_attention(*leaves, causal=causal, scale=scale, q_lens=cuda(ql), k_lens=cuda(kl))
    got = (out.detach(),) + torch.autograd.grad(out, leaves, dout)
    _reference.dtype = q.dtype
    ref, err = _reference(q, k, v, lam, dout, ql, kl, causal, scale or q.shape[-1] ** -0.5)
    for name, o, r, e in zip(("out", "dq", "dk", "dv", "dlam"), got, ref, err):
        close(o, r, e, name)
    with torch.no_grad():                        # the call without a gradient may take another path: the same bounds
        alone = S.differential_attention(q, k, v, lam, causal=causal, scale=scale, q_lens=cuda(ql), k_lens=cuda(kl))
    close(alone, ref[0], err[0], "out, no gradient")
    return got


SHAPES = [(1, 1, 1, 1, 1, 8), (2, 5, 5, 2, 1, 16), (1, 64, 64, 1, 1, 32), (2, 65, 65, 2, 2, 64), (1, 130, 130, 4, 2, 48), (2, 150, 150, 2, 2, 32), (1, 33, 200, 3, 1, 24),
          (1, 200, 33, 2, 1, 40), (3, 17, 129, 4, 1, 56), (1, 300, 300, 1, 1, 64), (2, 1, 700, 4, 2, 64), (1, 3, 513, 8, 1, 16), (4, 1, 9, 2, 2, 32)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ragged", [None, "some", "empty"])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,d", SHAPES)
def test_shapes(dt, causal, ragged, B, Tq, Tk, H, Hk, d):
    kl = lengths(B, Tk, ragged)
    ql = lengths(B, Tq, ragged) if Tq == Tk or ragged == "empty" else None
    got = _run(*_data(B, Tq, Tk, H, Hk, d, dt), ql=ql, kl=kl, causal=causal)
    if ql is not None:
        dead = torch.arange(Tq)[None] >= ql[:, None]
        assert (got[0].cpu()[dead] == 0).all() and (got[1].cpu()[dead] == 0).all()
    if kl is not None:
        dead = torch.arange(Tk)[None] >= kl[:, None]
        assert (got[2].cpu()[dead] == 0).all() and (got[3].cpu()[dead] == 0).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Tq,Tk", [(1, 5000), (4, 3001), (700, 700)])
def test_long_rows(causal, Tq, Tk):
    _run(*_data(2, Tq, Tk, 4, 2, 64, "bf16", seed=1), causal=causal, kl=torch.tensor([Tk, Tk // 3], dtype=torch.int32))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ragged", [None, "some", "empty"])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,d", [(2, 700, 300, 4, 2, 40), (1, 1300, 130, 2, 1, 64), (3, 400, 700, 1, 1, 8), (1, 2050, 64, 3, 1, 24), (2, 90, 1000, 8, 2, 48)])
def test_key_blocks_in_pieces(causal, ragged, B, Tq, Tk, H, Hk, d):
    """Few key blocks, many query tiles: dK and dV are summed over several workgroups."""
    _run(*_data(B, Tq, Tk, H, Hk, d, "bf16", seed=5), ql=lengths(B, Tq, ragged), kl=lengths(B, Tk, ragged), causal=causal)


@pytest.mark.parametrize("Tq,Tk", [(200, 900), (300, 100), (4, 900), (1, 40)])
@pytest.mark.parametrize("causal", [False, True])
def test_a_query_that_is_no_number_stays_one(Tq, Tk, causal):
    from xva_trainer_amd import seq_ops as S
    q, k, v, lam, dout = _data(1, Tq, Tk, 2, 1, 32, "bf16", seed=7)
    with torch.no_grad():
        clean = S.differential_attention(q, k, v, lam, causal=causal)
        q[0, Tq - 1, 1] = float("nan")
        out = S.differential_attention(q, k, v, lam, causal=causal)
    assert out[0, Tq - 1, 1].isnan().all()
    out[0, Tq - 1, 1] = clean[0, Tq - 1, 1]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", [[600, 0, 17, 600, 300], [1] * 4 + [530] * 3, [520] * 66, list(range(64))])
def test_items_of_any_lengths_in_any_order(causal, lens):
    """Long ragged batches start their longest items first: ties, empty items, more items than are ranked."""
    T, kl = max(max(lens), 513), torch.tensor(lens, dtype=torch.int32)
    _run(*_data(len(lens), T, T, 1, 1, 8, "bf16", seed=8), ql=kl, kl=kl, causal=causal)
    _run(*_data(len(lens), 70, T, 2, 1, 16, "bf16", seed=9), kl=kl, causal=causal)


@pytest.mark.parametrize("Tq,Tk,causal", [(200, 200, True), (1, 90, False), (4, 900, True), (700, 130, False), (90, 2000, False)])
@pytest.mark.parametrize("lam_type", [torch.bfloat16, torch.float16, torch.float64])
def test_numbers_of_any_type(Tq, Tk, causal, lam_type):
    """lam and its gradient in their own type: the results are those of the same numbers in fp32, the gradient is that one rounded once."""
    from xva_trainer_amd import seq_ops as S
    q, k, v, lam, dout = _data(2, Tq, Tk, 4, 2, 32, "bf16", seed=10)
    lam = lam.to(lam_type)
    out = {}
    for number in (lam, lam.float()):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, number)]
        y = S.differential_attention(*leaves, causal=causal)
        with torch.no_grad():
            out[number.dtype] = (y, S.differential_attention(*leaves, causal=causal)) + torch.autograd.grad(y, leaves, dout)
    mine, want = out[lam_type], out[torch.float32]
    assert mine[-1].dtype == lam_type and torch.equal(mine[-1], want[-1].to(lam_type))
    assert all(torch.equal(p, r) for p, r in zip(mine[:-1], want[:-1]))


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_numbers_of_a_head_of_any_sign(dt):
    q, k, v, lam, dout = _data(2, 200, 200, 6, 3, 32, dt, seed=6)
    lam.copy_(torch.tensor([0.0, -0.7, 1.5, -0.0, 1e-3, -3.0]))
    _run(q, k, v, lam, dout, causal=True)


@pytest.mark.parametrize("size,scale", [(4.0, None), (1.0, 2.0), (0.05, None)])
def test_sharp_and_flat_rows(size, scale):
    """Scores of hundreds (one key takes all), and of nothing (all keys alike)."""
    global E
    keep, E = E, E * max(1.0, size * size * (scale or 64 ** -0.5) * 8)      # scores grow by that much over the standard ones, and their fp32 error with them
    try:
        _run(*_data(1, 150, 150, 2, 1, 64, "bf16", seed=2, size=size), scale=scale, causal=True)
    finally:
        E = keep


def test_a_lone_key_gives_its_value_and_no_score_gradient():
    q, k, v, lam, dout = _data(3, 1, 1, 2, 2, 32, "bf16", seed=3)
    got = _run(q, k, v, lam, dout)
    ref = (v.double() * (1 - lam.double())[None, None, :, None])
    assert (got[0].double() - ref).abs().max() <= 2.0 ** -8 * ref.abs().max()
    # exact zeros but for the fp32 difference of two sums of the same 64 products, times keys of size 4
    assert max(got[1].abs().max().item(), got[2].abs().max().item()) < 64 * 16 * 2.0 ** -22 * 4


@pytest.mark.parametrize("Tq,Tk", [(70, 70), (1, 200), (90, 40)])
@pytest.mark.parametrize("causal", [False, True])
def test_what_lies_behind_an_item_is_not_read(Tq, Tk, causal):
    from xva_trainer_amd import seq_ops as S
    q, k, v, lam, dout = _data(4, Tq, Tk, 2, 1, 48, "bf16", seed=4)
    kl = torch.tensor([Tk, Tk // 2, 0, 1], dtype=torch.int32)
    ql = torch.tensor([Tq, max(1, Tq // 2), Tq, 0], dtype=torch.int32)
    dq_, dk_ = (torch.arange(Tq)[None] >= ql[:, None]).cuda(), (torch.arange(Tk)[None] >= kl[:, None]).cuda()
    outs = []
    for fill in (0.0, float("nan"), float("inf")):
        leaves = [q.masked_fill(dq_[..., None, None, None], fill), k.masked_fill(dk_[..., None, None, None], fill), v.masked_fill(dk_[..., None, None], fill), lam.clone()]
        leaves = [t.requires_grad_(True) for t in leaves]
        out = S.differential_attention(*leaves, causal=causal, q_lens=ql.cuda(), k_lens=kl.cuda())
        with torch.no_grad():
            alone = S.differential_attention(*leaves, causal=causal, q_lens=ql.cuda(), k_lens=kl.cuda())
        outs.append((out.detach(), alone) + torch.autograd.grad(out, leaves, dout.masked_fill(dq_[..., None, None], fill)))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_views_of_a_projection_and_of_a_cache():
    """q, k, v as slices of one projection; keys as the head of a longer cache; addresses and strides that the kernel needs copied."""
    H, Hk, d = 4, 2, 32
    whole = torch.randn(2, 90, H * 2 * d + Hk * 4 * d + 3, device="cuda").bfloat16()
    lam, dout = torch.rand(H, device="cuda"), torch.randn(2, 90, H, 2 * d, device="cuda").bfloat16()
    for at in (0, 1, 3):
        w = whole[..., at:at + H * 2 * d + Hk * 4 * d]
        q, k, v = w.split((H * 2 * d, Hk * 2 * d, Hk * 2 * d), -1)
        _run(q.unflatten(-1, (H, 2, d)), k.unflatten(-1, (Hk, 2, d)), v.unflatten(-1, (Hk, 2 * d)), lam, dout)
    cache = torch.randn(2, Hk, 300, 2, d, device="cuda").bfloat16().transpose(1, 2)
    vals = torch.randn(2, Hk, 300, 2 * d, device="cuda").bfloat16().transpose(1, 2)
    q = torch.randn(2, 1, H, 2, d, device="cuda").bfloat16()
    _run(q, cache[:, :200], vals[:, :200], lam, dout[:, :1], kl=torch.tensor([200, 31], dtype=torch.int32), causal=True)
    _run(q.expand(2, 70, H, 2, d), cache, vals, lam.bfloat16().float(), dout[:, :70].transpose(2, 3).contiguous().transpose(2, 3))


def test_lam_of_other_types_and_signs():
    from xva_trainer_amd import seq_ops as S
    q, k, v, _, dout = _data(2, 40, 40, 4, 4, 16, "fp16", seed=5)
    for lam in (torch.zeros(4, device="cuda"), torch.tensor([-1.0, 2.0, 0.0, 1.0], device="cuda")):
        _run(q, k, v, lam, dout)
    lam = torch.tensor([0.1, 0.9, 0.3, 0.5], device="cuda").half().requires_grad_(True)
    out = S.differential_attention(q, k, v, lam)
    g, = torch.autograd.grad(out, lam, dout)
    assert g.dtype == torch.float16
    lam32 = lam.detach().float().requires_grad_(True)
    g32, = torch.autograd.grad(S.differential_attention(q, k, v, lam32), lam32, dout)
    assert torch.equal(g, g32.half())


def test_the_gradient_by_differences():
    """Against differences of the loss itself; outputs carry u of the weights' sums, so the step is large and the bound follows it."""
    from xva_trainer_amd import seq_ops as S
    q, k, v, lam, dout = _data(1, 48, 48, 2, 1, 32, "fp16", seed=6)
    lam.requires_grad_(True)
    vv = v.clone().requires_grad_(True)
    out = S.differential_attention(q, k, vv, lam, causal=True)
    gv, gl = torch.autograd.grad(out, (vv, lam), dout)
    step = torch.randn_like(lam)
    with torch.no_grad():                                            # linear in lam and in v
        f = lambda l, x: (S.differential_attention(q, k, x, l, causal=True).double() * dout.double()).sum()
        by_lam = (f(lam + step, v) - f(lam - step, v)) / 2
        by_v = (f(lam, v + v) - f(lam, v - v)) / 2
    noise = 2.0 ** -10 * (1 + lam.abs().max().item() + step.abs().max().item()) * dout.double().abs().sum().item() * v.abs().max().item()
    n = dout.numel() ** 0.5 / dout.numel()                           # of independent roundings, ten deviations
    assert abs(by_lam.item() - (gl * step).sum().item()) < 10 * n * noise
    assert abs(by_v.item() - (gv.double() * v.double()).sum().item()) < 10 * n * noise


def test_repeats_graph_and_streams():
    from xva_trainer_amd import seq_ops as S
    for Tq, Tk in ((200, 200), (1, 900), (700, 1500)):
        q, k, v, lam, dout = _data(2, Tq, Tk, 4, 2, 64, "bf16", seed=7)
        leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
        kl = torch.tensor([Tk, Tk // 2], device="cuda", dtype=torch.int32)
        def step():
            out = S.differential_attention(*leaves, k_lens=kl)
            with torch.no_grad():
                alone = S.differential_attention(*leaves, k_lens=kl)
            return (out.detach(), alone) + torch.autograd.grad(out, leaves, dout)
        assert all(torch.equal(a, b) for a, b in zip(step(), step()))
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
                q.normal_(), k.normal_(), dout.normal_(), kl.random_(1, Tk + 1)
            graph.replay()
            eager = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, eager)), turn


def test_two_calls_at_once():
    """Passes on two streams that cut their blocks into pieces: each has its own workspace."""
    from xva_trainer_amd import seq_ops as S
    sets = [[t.requires_grad_(True) for t in _data(1, 600, 1400, 2, 1, 48, "bf16", seed=s)] for s in (11, 12)]
    def step(t):
        out = S.differential_attention(*t[:4], causal=True)
        return (out.detach(),) + torch.autograd.grad(out, t[:4], t[4].detach())
    want = [step(t) for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for turn in range(3):
        got = []
        for t, s in zip(sets, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step(t))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w)), turn


def test_empty():
    from xva_trainer_amd import seq_ops as S
    for B, Tq, Tk in ((0, 3, 3), (2, 0, 3), (2, 3, 0)):
        q, k, v, lam, dout = _data(B, Tq, Tk, 2, 1, 16, "bf16")
        leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
        out = S.differential_attention(*leaves)
        assert out.shape == (B, Tq, 2, 32) and (out == 0).all()
        assert all((g == 0).all() for g in torch.autograd.grad(out, leaves, dout))


def test_refusals():
    from xva_trainer_amd import seq_ops as S
    q, k, v, lam, _ = _data(2, 3, 4, 4, 2, 16, "bf16")
    for bad in (lambda: S.differential_attention(q.float(), k.float(), v.float(), lam), lambda: S.differential_attention(q, k.half(), v, lam),
                lambda: S.differential_attention(q, k, v[:, :3], lam), lambda: S.differential_attention(q[:, :, :3], k, v, lam[:3]),
                lambda: S.differential_attention(q, k, v, lam[:3]), lambda: S.differential_attention(q[..., :12], k[..., :12], v[..., :24], lam),
                lambda: S.differential_attention(q, k, v, lam.long()), lambda: S.differential_attention(q, k, v, lam, scale=0.0),
                lambda: S.differential_attention(q, k, v, lam, scale=float("nan")), lambda: S.differential_attention(q, k, v, lam, k_lens=torch.tensor([1, 2])),
                lambda: S.differential_attention(q, k, v, lam, q_lens=torch.tensor([1, 2, 3], device="cuda")), lambda: S.differential_attention(q.cpu(), k, v, lam),
                lambda: S.differential_attention(q[:, :, :, 0], k, v, lam), lambda: S.differential_attention(torch.zeros(1, 2, 1, 2, 72, device="cuda").half(),
                                                                                                          torch.zeros(1, 2, 1, 2, 72, device="cuda").half(),
                                                                                                          torch.zeros(1, 2, 1, 144, device="cuda").half(), lam[:1])):
        with pytest.raises(S.XvaError):
            bad()


@pytest.mark.parametrize("Tq", [1, 40])
@pytest.mark.parametrize("width", [2048, 2053, 2049])
def test_one_row_of_a_projection_of_any_width(Tq, width):
    """Dimensions of 1 may have any stride; torch calls such a slice contiguous and copies nothing."""
    H, d, T = 16, 64, 70
    whole = torch.randn(2, T, width, device="cuda").bfloat16()
    q = whole[..., :H * 2 * d].unflatten(-1, (H, 2, d))[:1, :Tq]
    k, v = whole[1:, ..., :2 * d].unflatten(-1, (1, 2, d))[:, :T if Tq > 1 else 1], whole[:1, :T if Tq > 1 else 1, 64:64 + 2 * d].unflatten(-1, (1, 2 * d))
    dout = torch.randn(1, T, width, device="cuda").bfloat16()[:, :Tq, :H * 2 * d].unflatten(-1, (H, 2 * d))
    _run(q, k, v, torch.rand(H, device="cuda"), dout, causal=True)


def _norm_bounds(q, k, v, lam, dout, causal):
    """Gradients in 64 bits, and how far the norm of each one's error may be: roundings are independent, so a sum of products that are each off by u of themselves is off
    by u of its norm or so.  P_1 - lam P_2 or dS as an operand, the maps' outputs behind D, the result itself: 4 u bounds them, fp32's own E beside them.  Besides, each
    element of the result is off by 2^-25, and each weight that meets dO in dV."""
    u, tiny = HALF[q.dtype], TINY[q.dtype]
    q, k, v, lam, dout = (t.detach().double() for t in (q, k, v, lam, dout))
    q, k, v, lam = (t.requires_grad_(True) for t in (q, k, v, lam))
    share, n = q.shape[2] // k.shape[2], q.shape[1]
    s = torch.matmul(q.permute(0, 2, 3, 1, 4), k.permute(0, 2, 3, 4, 1).repeat_interleave(share, 1).contiguous()) * q.shape[-1] ** -0.5
    if causal:
        s = s.masked_fill(torch.ones(n, k.shape[1], dtype=torch.bool, device=q.device).triu(1 + k.shape[1] - n), -math.inf)
    p = torch.softmax(s, -1)
    out = torch.matmul(p[:, :, 0] - lam[:, None, None] * p[:, :, 1], v.permute(0, 2, 1, 3).repeat_interleave(share, 1).contiguous()).permute(0, 2, 1, 3)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    bound = lambda g, more=0.0: (4 * u + E) * g.norm().item() + tiny * g.numel() ** 0.5 + more
    parts = {"dq_1": grads[0][..., 0, :], "dq_2": grads[0][..., 1, :], "dk_1": grads[1][..., 0, :], "dk_2": grads[1][..., 1, :], "dv": grads[2]}
    return {m: (g, bound(g, tiny * (k.shape[1] * dout.square().sum().item()) ** 0.5 if m == "dv" else 0.0)) for m, g in parts.items()}


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("lam_size", [0.5, 0.01, 1e-4, 30.0])
@pytest.mark.parametrize("dout_size,H,Hk,T,d,causal", [(1.0, 2, 1, 860, 48, False), (1e-3, 4, 2, 860, 48, False), (1e-4, 1, 1, 4096, 48, False), (1e-3, 2, 2, 700, 64, True),
                                                       (1e-3, 2, 1, 300, 32, True), (1e-3, 4, 1, 90, 16, False)])
def test_gradients_of_any_size(dt, lam_size, dout_size, H, Hk, T, d, causal):
    """The loss of a training step is a mean, so dO is small; lam may be: no part of the gradient sinks into fp16's subnormal numbers on the way, judged by the norm of
    its error (values are large enough that the results themselves do not)."""
    from xva_trainer_amd import seq_ops as S
    q, k, v, lam, dout = _data(2, T, T, H, Hk, d, dt, seed=13)
    q, k, v = (t * 4 if t is v else t for t in (q, k, v))
    lam = lam_size * (1 + 0.2 * torch.randn(H, device="cuda"))
    dout = (dout.float() * dout_size).to(q.dtype)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    got = torch.autograd.grad(S.differential_attention(*leaves, causal=causal), leaves[:3], dout)
    got = {"dq_1": got[0][..., 0, :], "dq_2": got[0][..., 1, :], "dk_1": got[1][..., 0, :], "dk_2": got[1][..., 1, :], "dv": got[2]}
    for name, (ref, bound) in _norm_bounds(q, k, v, lam, dout, causal).items():
        off = (got[name].double() - ref).norm().item()
        assert off <= bound, "%s off by %.3g of %.3g, %.3g allowed" % (name, off, ref.norm().item(), bound)


def test_gradients_beyond_the_type_on_the_way():
    """dO . v of a quarter of a million, more than fp16 holds, on the way to gradients of a few hundred; items of very different size in one batch."""
    from xva_trainer_amd import seq_ops as S
    q, k, v, lam, dout = _data(2, 300, 300, 2, 1, 48, "fp16", seed=14)
    q, k, v, dout = q * 0.05, k * 0.05, v * 4, dout * 5000
    dout[1] *= 1e-7
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    got = torch.autograd.grad(S.differential_attention(*leaves, causal=True), leaves[:3], dout)
    assert all(g.isfinite().all() for g in got)
    for b in range(2):
        mine = {"dq_1": got[0][b:b + 1, ..., 0, :], "dq_2": got[0][b:b + 1, ..., 1, :], "dk_1": got[1][b:b + 1, ..., 0, :], "dk_2": got[1][b:b + 1, ..., 1, :], "dv": got[2][b:b + 1]}
        for name, (ref, bound) in _norm_bounds(q[b:b + 1], k[b:b + 1], v[b:b + 1], lam, dout[b:b + 1], True).items():
            off = (mine[name].double() - ref).norm().item()
            assert off <= bound, "%s of item %d off by %.3g of %.3g, %.3g allowed" % (name, b, off, ref.norm().item(), bound)


def test_empty_in_fp16():
    from xva_trainer_amd import seq_ops as S
    for B, Tq, Tk in ((0, 3, 3), (2, 0, 3), (2, 3, 0)):
        q, k, v, lam, dout = _data(B, Tq, Tk, 2, 1, 16, "fp16")
        leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
        out = S.differential_attention(*leaves)
        assert out.shape == (B, Tq, 2, 32) and (out == 0).all()
        assert all((g == 0).all() for g in torch.autograd.grad(out, leaves, dout))


@pytest.mark.parametrize("causal", [False, True])
def test_what_lies_behind_an_item_is_not_read_in_fp16(causal):
    """The gradient's range is that of live rows; and an item whose gradient is not finite leaves the others theirs."""
    from xva_trainer_amd import seq_ops as S
    q, k, v, lam, dout = _data(4, 90, 90, 2, 1, 48, "fp16", seed=16)
    dout = dout * 1e-3
    kl = torch.tensor([90, 45, 0, 1], dtype=torch.int32)
    dead = (torch.arange(90)[None] >= kl[:, None]).cuda()
    outs = []
    for fill in (0.0, float("nan"), float("inf")):
        leaves = [t.masked_fill(dead.view(4, 90, *[1] * (t.dim() - 2)), fill).requires_grad_(True) for t in (q, k, v)] + [lam.clone().requires_grad_(True)]
        out = S.differential_attention(*leaves, causal=causal, q_lens=kl.cuda(), k_lens=kl.cuda())
        outs.append((out.detach(),) + torch.autograd.grad(out, leaves, dout.masked_fill(dead[..., None, None], fill)))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))
    for bad in (float("nan"), float("inf")):
        g = dout.clone()
        g[0, 3, 1, 5] = bad
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        got = torch.autograd.grad(S.differential_attention(*leaves, lam, causal=causal), leaves, g)
        want = torch.autograd.grad(S.differential_attention(*leaves, lam, causal=causal), leaves, dout)
        assert all(torch.equal(a[1:], b[1:]) for a, b in zip(got, want)) and all((~a[0].isfinite()).any() for a in got)


def test_graph_of_gradients_of_any_size():
    """Captured fp16 passes: the powers of two follow the data of each replay; two passes at once have their own."""
    from xva_trainer_amd import seq_ops as S
    for T in (150, 700):
        q, k, v, lam, dout = _data(2, T, T, 4, 2, 48, "fp16", seed=17)
        leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
        lens = torch.tensor([T, T // 2], device="cuda", dtype=torch.int32)
        def step():
            out = S.differential_attention(*leaves, q_lens=lens, k_lens=lens)
            return (out.detach(),) + torch.autograd.grad(out, leaves, dout)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for turn, (size, number) in enumerate(((1.0, 0.5), (1e-3, 1e-3), (2000.0, 4.0), (1e-2, 0.0), (1.0, -0.5))):
            with torch.no_grad():
                q.normal_(), k.normal_(), v.normal_(), dout.copy_(torch.randn_like(dout, dtype=torch.float32) * size), lam.fill_(number), lens.random_(1, T + 1)
            graph.replay()
            eager = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, eager)), turn
        two, streams = [], [torch.cuda.Stream() for _ in range(2)]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                two.append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for got in two for a, b in zip(got, eager))


@pytest.mark.parametrize("size", [1e-3, 1.0, 5000.0])
@pytest.mark.parametrize("d,causal", [(16, False), (32, True), (48, False), (64, True)])
def test_gradients_of_any_size_where_blocks_are_whole(size, d, causal):
    """Enough key blocks that none is cut into pieces: the factors are undone where a block's own sums are rounded."""
    from xva_trainer_amd import seq_ops as S
    q, k, v, lam, dout = _data(24, 200, 200, 4, 4, d, "fp16", seed=18)
    q, k, v, dout = q * 0.05, k * 0.05, v * 4, (dout.float() * size).half()
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    got = torch.autograd.grad(S.differential_attention(*leaves, causal=causal), leaves[:3], dout)
    got = {"dq_1": got[0][..., 0, :], "dq_2": got[0][..., 1, :], "dk_1": got[1][..., 0, :], "dk_2": got[1][..., 1, :], "dv": got[2]}
    for name, (ref, bound) in _norm_bounds(q, k, v, lam, dout, causal).items():
        off = (got[name].double() - ref).norm().item()
        assert off <= bound, "%s off by %.3g of %.3g, %.3g allowed" % (name, off, ref.norm().item(), bound)
