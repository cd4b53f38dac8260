"""Group normalisation with an activation (csrc/group_norm.hip) against the formulas in 64 bits, with gradients by autograd in 64 bits.

fp32 errors: xh carries a few roundings of x - mu (|x - mu| + |mu| 2^-24 at worst, times r) and of r (the mean of n squares: under 2^-20 relative for pairwise and
short sums); every later step multiplies or adds a handful of values of the sizes below.  2^-18 of those sizes covers them with room; sums over rows of N random
products add at most N 2^-24 of the sum of magnitudes."""
import pytest
import torch

from seq_util import DTYPES, close, lengths, rounded

pytestmark = pytest.mark.gpu
ACTS = ["none", "relu", "lrelu", "tanh", "silu", "gelu"]
E = 2.0 ** -18


def _act(z, act, slope):
    return {"none": lambda: z, "relu": lambda: z.relu(), "lrelu": lambda: torch.where(z > 0, z, slope * z), "tanh": lambda: z.tanh(),
            "silu": lambda: z * torch.sigmoid(z), "gelu": lambda: 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))}[act]()


def _reference(x, w, b, dy, lens, G, eps, act, slope):
    """Outputs and gradients in 64 bits on the CPU, and the sizes that their errors scale with."""
    x, dy = x.detach().double().cpu().requires_grad_(True), dy.detach().double().cpu()
    B, T, C = x.shape
    w = (w.detach().double().cpu() if w is not None else torch.ones(C, dtype=torch.float64)).requires_grad_(True)
    b = (b.detach().double().cpu() if b is not None else torch.zeros(C, dtype=torch.float64)).requires_grad_(True)
    live = torch.ones(B, T, 1, dtype=torch.float64)
    if lens is not None:
        live = (torch.arange(T)[None] < lens.cpu()[:, None]).double()[:, :, None]
    xs = torch.where(live > 0, x, torch.zeros_like(x)).view(B, T, G, C // G)
    n = (live.sum((1, 2)) * (C // G)).clamp_min(1).view(B, 1, 1, 1)
    mu = xs.sum((1, 3), keepdim=True) / n
    off = (xs - mu) * live[..., None]
    r = (off.square().sum((1, 3), keepdim=True) / n + eps).rsqrt()
    z = (off * r).reshape(B, T, C) * w + b
    y = _act(z, act, slope) * live
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.where(live > 0, dy, torch.zeros_like(dy)))
    with torch.no_grad():
        # an error of x - mu of 2^-24 (|x| + |mu|), times r
        xh = (off * r).reshape(B, T, C)
        exh = (E * (1 + xh.abs()) + 2.0 ** -23 * ((xs.abs() + mu.abs()) * r).reshape(B, T, C)) * live
        ez = exh * w.abs() + E * (xh * w).abs() + E * b.abs()
        g = torch.where(live > 0, dy, torch.zeros_like(dy)).abs()
        ey = 1.2 * ez + E * y.abs()
        wg = (g * w.abs() * 1.2)
        mean = lambda t: ((t.view(B, T, G, C // G)).sum((1, 3), keepdim=True) / n).expand(B, T, G, C // G).reshape(B, T, C)
        # every term of dx moves by the error of xh (activations' slopes change by at most 1.2 of it) and by E of itself
        m_x, big = mean(wg * xh.abs()), (1 + xh.abs())
        ex = (r.expand(B, T, G, C // G).reshape(B, T, C) *
              ((E + ez * 1.5) * wg + mean((E + ez * 1.5) * wg) + big * mean((E * (1 + xh.abs()) + exh + ez * 1.5 * xh.abs()) * wg) + exh * m_x + E * big * m_x)) * live
        N = float(B * T)
        ew = ((E + N * 2.0 ** -24) * (wg / w.abs().clamp_min(1e-3) * big) + (exh + 1.5 * ez * xh.abs()) * g * 1.2).sum((0, 1))
        eb = ((E + N * 2.0 ** -24 + 1.5 * ez) * g * 1.2).sum((0, 1))
    return (y.detach(), dx, dw, db), (ey, ex, ew, eb)


def _run(x, w, b, dy, lens, G, eps=1e-5, act="none", slope=0.1, kink=False):
    from xva_trainer_amd import seq_ops as S
    x = x.detach().requires_grad_(True)
    ps = [p for p in (w, b) if p is not None]
    for p in ps:
        p.requires_grad_(True)
    y = S.group_norm_act(x, G, w, b, lens=lens, eps=eps, act=act, slope=slope)
    got = torch.autograd.grad(y, [x] + ps, dy)
    ref, err = _reference(x, w, b, dy, lens, G, eps, act, slope)
    close(y, ref[0], rounded(ref[0], x.dtype, err[0]), "y")
    if not kink:
        close(got[0], ref[1], rounded(ref[1], x.dtype, err[1]), "dx")
        for i, p in enumerate(ps):
            which = 2 if p is w else 3
            close(got[1 + i], ref[which], rounded(ref[which], p.dtype, err[which]), ("dw", "db")[which - 2])
    with torch.no_grad():
        assert torch.equal(S.group_norm_act(x, G, w, b, lens=lens, eps=eps, act=act, slope=slope), y)
    return y, got


def _data(B, T, C, dt, seed=0, mean=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000 + B * 77 + T * 13 + C)
    x = (torch.randn(B, T, C, device="cuda", generator=g) + mean).to(DTYPES[dt])
    dy = torch.randn(B, T, C, device="cuda", generator=g).to(DTYPES[dt])
    w = 1 + 0.1 * torch.randn(C, device="cuda", generator=g)
    return x, w, 0.1 * torch.randn(C, device="cuda", generator=g), dy


SHAPES = [(1, 1, 16, 1), (300, 1, 512, 8), (5, 1, 1024, 2), (3, 2, 48, 3), (2, 860, 384, 16), (1, 1, 8, 2), (3, 65, 40, 5), (2, 33, 31, 1), (4, 300, 21, 3),
          (1, 2000, 32, 4), (2, 9, 1023, 1), (1, 40, 2048, 32), (2, 700, 8, 8), (7, 3, 136, 8), (600, 5, 72, 8), (1, 5000, 16, 1), (2, 17, 2048, 2048), (1, 1, 1023, 3),
          # vectors of two, one to eight of them to a lane; groups of two values to the workgroup; many chunks, few channels; more items than one join takes
          (5, 7, 432, 8), (3, 9, 432, 8), (2, 60, 432, 8), (3, 1, 150, 3), (2, 2500, 150, 3), (3, 388, 8, 8), (1, 20011, 16, 4), (1, 9000, 150, 3), (1100, 20, 32, 1),
          (1100, 3, 2, 1), (1030, 21, 33, 1), (2, 70, 4088, 2)]


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("ragged", [None, "some", "empty"])
@pytest.mark.parametrize("B,T,C,G", SHAPES)
def test_shapes(dt, ragged, B, T, C, G):
    x, w, b, dy = _data(B, T, C, dt)
    lens = lengths(B, T, ragged)
    y, got = _run(x, w, b, dy, lens.cuda() if lens is not None else None, G, act="silu" if C % 3 else "none")
    if lens is not None:
        dead = torch.arange(T)[None] >= lens[:, None]
        assert (y.cpu()[dead] == 0).all() and (got[0].cpu()[dead] == 0).all()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("B,T,C,G", [(40, 1, 64, 4), (3, 200, 64, 4)])
def test_activations(act, B, T, C, G):
    """relu and lrelu: z must not lie on the kink within its error, so their inputs are moved away from it."""
    x, w, b, dy = _data(B, T, C, "fp32", seed=7)
    if act in ("relu", "lrelu"):
        w = torch.ones_like(w)
        x = torch.where(x > 0.3, x + 0.5, x - 0.5)
        b = torch.zeros_like(b) + 0.05
    _run(x, w, b, dy, None, G, act=act)


@pytest.mark.parametrize("B,T", [(30, 1), (2, 500)])
def test_without_weight_and_bias_and_with_16_bit_ones(B, T):
    x, w, b, dy = _data(B, T, 64, "bf16", seed=2)
    _run(x, None, None, dy, None, 8)
    _run(x, w, None, dy, None, 8)
    _run(x, w.bfloat16(), b.bfloat16(), dy, None, 8)


@pytest.mark.parametrize("B,T,C", [(20, 1, 128), (2, 900, 64)])
def test_a_mean_far_from_zero(B, T, C):
    """A mean of a thousand deviations: the error allowed is that of x - mu alone (see `_reference`), so a variance from E[x^2] - mu^2 would fail."""
    x, w, b, dy = _data(B, T, C, "fp32", seed=3, mean=1000.0)
    _run(x, w, b, dy, None, 4)


def test_constant_groups():
    """No deviation at all: xh is 0, r is eps^-1/2."""
    from xva_trainer_amd import seq_ops as S
    for B, T in ((3, 1), (2, 400)):
        x = torch.full((B, T, 32), 2.0, device="cuda")
        b = torch.randn(32, device="cuda")
        assert torch.equal(S.group_norm_act(x, 4, None, b), b.expand(B, T, 32))


@pytest.mark.parametrize("T,C,G", [(1, 64, 4), (3, 24, 2), (300, 64, 4), (90, 33, 3)])
def test_what_lies_behind_an_item_is_not_read(T, C, G):
    from xva_trainer_amd import seq_ops as S
    x, w, b, dy = _data(4, T, C, "bf16", seed=4)
    lens = torch.tensor([T, T // 2, 0, min(1, T)], dtype=torch.int32)
    dead = (torch.arange(T)[None] >= lens[:, None]).cuda()
    outs = []
    for fill in (0.0, float("nan"), float("inf")):
        xf, gf = x.masked_fill(dead[..., None], fill).requires_grad_(True), dy.masked_fill(dead[..., None], fill)
        w.requires_grad_(True)
        y = S.group_norm_act(xf, G, w, b, lens=lens.cuda(), act="silu")
        outs.append((y.detach(),) + torch.autograd.grad(y, (xf, w), gf))
    for other in outs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(outs[0], other))


def test_views_strides_and_flat_rows():
    from xva_trainer_amd import seq_ops as S
    store = torch.randn(3, 40, 100, device="cuda").bfloat16()
    for view in (store[:, 1:-1, :64], store[:, ::2, 8:72], store[:, :, 3:67], store.transpose(0, 1)[..., :32], store[1:2].expand(3, 40, 100)[..., :96],
                 store.transpose(1, 2)[:, :64, :32], store[:, :, 2:66], store[:, :1, 2:66], store[:, :, 6:14]):
        G = 4
        dy = torch.randn(view.shape, device="cuda").bfloat16()
        _run(view, None, None, dy, None, G)
    rows = torch.randn(50, 96, device="cuda")
    assert torch.equal(S.group_norm_act(rows, 6), S.group_norm_act(rows[:, None], 6)[:, 0])


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_many_channels_at_any_address(dt):
    """2048 channels need vectors: an input or a gradient that lies between two of them is taken all the same."""
    from xva_trainer_amd import seq_ops as S
    x, w, b, dy = _data(2, 300, 2048, dt, seed=8)
    odd = lambda t: torch.cat([t[..., :1], t, t[..., :2]], -1)[..., 1:2049]
    x.requires_grad_(True), w.requires_grad_(True)
    y = S.group_norm_act(x, 4, w, b, act="silu")
    want = torch.autograd.grad(y, (x, w), dy)
    x2 = odd(x.detach()).requires_grad_(True)
    y2 = S.group_norm_act(x2, 4, w, b, act="silu")
    assert torch.equal(y, y2)
    for got in (torch.autograd.grad(y2, (x2, w), odd(dy), retain_graph=True), torch.autograd.grad(y2, (x2, w), dy)):
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    flat = torch.zeros(x.numel() + 1, device="cuda", dtype=x.dtype)[1:].view(x.shape).copy_(x.detach())      # contiguous, at an odd address
    with torch.no_grad():
        assert torch.equal(S.group_norm_act(flat, 4, w, b, act="silu"), y)


def test_repeats_bit_for_bit():
    x, w, b, dy = _data(3, 1500, 96, "bf16", seed=5)
    y1, g1 = _run(x, w, b, dy, None, 8, act="gelu")
    y2, g2 = _run(x, w, b, dy, None, 8, act="gelu")
    assert torch.equal(y1, y2) and all(torch.equal(p, q) for p, q in zip(g1, g2))


def test_the_gradient_by_differences():
    from xva_trainer_amd import seq_ops as S
    for B, T in ((4, 1), (2, 300)):
        x, w, b, dy = _data(B, T, 32, "fp32", seed=6)
        x.requires_grad_(True)
        grad, = torch.autograd.grad(S.group_norm_act(x, 4, w, b, act="gelu"), x, dy)
        step = torch.randn_like(x)
        h = 2.0 ** -7
        with torch.no_grad():
            f = lambda s: (S.group_norm_act(x + s * h * step, 4, w, b, act="gelu").double() * dy).sum()
            diff = ((f(1) - f(-1)) / (2 * h)).item()
        exact = (grad.double() * step).sum().item()
        # third differences of a smooth function of values of size 1: h^2 of the sum of magnitudes; fp32 outputs: 2^-20 / h of it
        size = (grad.abs() * step.abs()).sum().item() + dy.abs().sum().item()
        assert abs(diff - exact) < size * (h * h + 2.0 ** -20 / h)


def test_empty_graph_and_stream():
    from xva_trainer_amd import seq_ops as S
    w = torch.ones(32, device="cuda", requires_grad=True)
    for shape in ((0, 4, 32), (3, 0, 32)):
        y = S.group_norm_act(torch.zeros(shape, device="cuda", requires_grad=True), 4, w)
        assert y.shape == shape
        assert (torch.autograd.grad(y.sum(), w)[0] == 0).all()
    del y                                        # (an eager graph of a leaf must not live while a backward pass of that leaf is captured: torch ties the two streams)
    for B, T in ((6, 1), (2, 700), (1100, 20), (1, 6000)):
        x, dy = torch.randn(B, T, 32, device="cuda", requires_grad=True), torch.randn(B, T, 32, device="cuda")
        def step():
            y = S.group_norm_act(x, 4, w, act="silu")
            return (y.detach(),) + torch.autograd.grad(y, (x, w), dy)
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
                x.normal_(), dy.normal_()
            graph.replay()
            eager = step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, eager)), turn


def test_refusals():
    from xva_trainer_amd import seq_ops as S
    x = torch.zeros(2, 3, 32, device="cuda")
    for bad in (lambda: S.group_norm_act(x, 5), lambda: S.group_norm_act(x, 0), lambda: S.group_norm_act(x.double(), 4), lambda: S.group_norm_act(x, 4, act="elu"),
                lambda: S.group_norm_act(x, 4, torch.ones(31, device="cuda")), lambda: S.group_norm_act(x, 4, torch.ones(32)), lambda: S.group_norm_act(x[None], 4),
                lambda: S.group_norm_act(x, 4, lens=torch.tensor([1, 2, 3], device="cuda")), lambda: S.group_norm_act(x, 4, lens=torch.tensor([1, 2])),
                lambda: S.group_norm_act(x, 4, lens=torch.tensor([1.0, 2.0], device="cuda")), lambda: S.group_norm_act(x[0], 4, lens=torch.tensor([1, 2], device="cuda")),
                lambda: S.group_norm_act(x, 4, eps=-1.0), lambda: S.group_norm_act(x.cpu(), 4),
                lambda: S.group_norm_act(torch.zeros(1, 300, 16384, device="cuda"), 2), lambda: S.group_norm_act(torch.zeros(1, 600, 4096, device="cuda"), 4096)):
        with pytest.raises(S.XvaError):
            bad()


@pytest.mark.parametrize("shape,G", [((0, 5000, 32), 1), ((0, 300, 64), 4), ((0, 500, 33), 1), ((0, 600, 4096), 4096), ((3, 0, 32), 4)])
def test_no_items_or_rows_in_any_form(shape, G):
    from xva_trainer_amd import seq_ops as S
    x, w, b = torch.zeros(shape, device="cuda", requires_grad=True), torch.ones(shape[2], device="cuda", requires_grad=True), torch.ones(shape[2], device="cuda", requires_grad=True)
    y = S.group_norm_act(x, G, w, b, act="silu")
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == dx.shape == shape and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("B,T,C,G", [(2, 300, 2048, 4), (300, 1, 512, 8), (2, 860, 384, 16), (2, 2500, 32, 4), (2, 60, 430, 5)])
def test_weights_at_any_address(dt, B, T, C, G):
    """Slices of a flat parameter buffer: the same results and gradients, whatever their address."""
    from xva_trainer_amd import seq_ops as S
    x, w, b, dy = _data(B, T, C, dt, seed=9)
    flat = torch.zeros(2 * C + 3, device="cuda")
    outs = []
    for at in (None, 1, 2, 3):
        ws = [t.clone() if at is None else flat[at + i * C:at + (i + 1) * C].copy_(t) for i, t in enumerate((w, b))]
        leaves = [t.detach().requires_grad_(True) for t in [x] + ws]
        y = S.group_norm_act(leaves[0], G, leaves[1], leaves[2], act="silu")
        outs.append((y.detach(),) + torch.autograd.grad(y, leaves, dy))
    for other in outs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(outs[0], other))


@pytest.mark.parametrize("size", [1.0, 1e-1, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("B,T,C,G", [(40, 1, 64, 4), (3, 200, 64, 4), (2, 2500, 32, 4)])
def test_tanh_of_small_weights(size, B, T, C, G):
    """z carries the weights' size, and so do the errors allowed (`_reference`): a tanh that is off by a share of 1 would not do."""
    from xva_trainer_amd import seq_ops as S
    x, w, b, dy = _data(B, T, C, "fp32", seed=10)
    w, b = (t * size for t in (w, b))
    x.requires_grad_(True)
    y = S.group_norm_act(x, G, w, b, act="tanh")
    dx, = torch.autograd.grad(y, x, dy)
    ref, err = _reference(x, w, b, dy, None, G, 1e-5, "tanh", 0.0)
    close(y, ref[0], rounded(ref[0], x.dtype, err[0]), "y")
    close(dx, ref[1], rounded(ref[1], x.dtype, err[1]), "dx")


def test_tanh_far_out():
    """Slopes of saturated values, where 1 - tanh^2 would have nothing left: 4 e / (1 + e)^2 with e = exp(-2 |z|).  The exponential's argument, up to 40, is off by
    1.5 x 2^-24 of itself (the product with log2 e and that constant), e and the reciprocals by some units: under 40 x 1.5 x 2^-24 + 8 x 2^-24 < 2^-17 of the slope."""
    from xva_trainer_amd import seq_ops as S
    x = torch.tensor([1.0, -1.0], device="cuda").repeat(32)[None].requires_grad_(True)
    b = torch.linspace(-20, 20, 64, device="cuda").requires_grad_(True)
    y = S.group_norm_act(x, 1, torch.zeros(64, device="cuda"), b, eps=0.0, act="tanh")
    db, = torch.autograd.grad(y, b, torch.ones_like(y))
    z = b.detach().double().cpu()
    close(y.detach()[0], z.tanh(), 2.0 ** -22 * z.tanh().abs(), "y")
    close(db, z.cosh() ** -2, 2.0 ** -17 * z.cosh() ** -2, "slope")


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("B,T", [(1, 300), (1, 1), (5, 1)])
def test_one_row_or_item_at_any_stride(dt, B, T):
    """The stride of a dimension of 1 says nothing: the same results as of a copy, also where 2048 channels in one group of long rows need vectors."""
    from xva_trainer_amd import seq_ops as S
    whole = torch.randn(B * 301 * 2051 + 8, device="cuda").to(DTYPES[dt])
    for sb, st in ((301 * 2051, 2048), (2048, 2051), (2051 * 8, 3)):
        x = whole.as_strided((B, T, 2048), (sb if B == 1 else 2048 * T, st if T == 1 else 2048, 1)).requires_grad_(True)
        want = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
        dy = torch.randn(B, T, 2048, device="cuda").to(DTYPES[dt])
        for G in (2, 32):
            y, z = S.group_norm_act(x, G, act="gelu"), S.group_norm_act(want, G, act="gelu")
            assert torch.equal(y, z) and torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(z, want, dy)[0])
