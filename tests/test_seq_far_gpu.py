"""The sequence operators on tensors that lie far apart in memory: offsets beyond 2^31 elements and 2^32 bytes, between items, rows, heads and maps, give the results
of contiguous copies bit for bit (the plans depend on sizes and alignment alone, which are the same; the recurrence apart, see there)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
FAR = 2 ** 31 + 2 ** 20        # elements; multiples of 64


@pytest.fixture(scope="module")
def store():
    yield torch.empty(3 * 2 ** 31, device="cuda", dtype=torch.bfloat16)
    torch.cuda.empty_cache()


def _spread(store, t, strides, at=0):
    """A view of `store` with t's values."""
    view = store.as_strided(t.shape, strides + (1,), at)
    return view.copy_(t)


def _same(call, near, far, grads):
    out = []
    for ts in (near, far):
        leaves = [t.detach().requires_grad_(True) for t in ts]
        y = call(*leaves)
        ys = list(y) if isinstance(y, (tuple, list)) else [y]
        with torch.no_grad():
            alone = call(*leaves)
        out.append([v.detach() for v in ys] + (list(alone) if isinstance(alone, (tuple, list)) else [alone]) + list(torch.autograd.grad(ys, leaves, grads)))
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("strides", [(FAR, 128, 64), (128, FAR, 64), (256, 512, FAR)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(store, strides, interleaved):
    from xva_trainer_amd import seq_ops as S
    plan = S.RotaryPlan(64, interleaved=interleaved)
    q = torch.randn(2, 2, 2, 64, device="cuda").bfloat16()
    k = torch.randn(2, 2, 2, 64, device="cuda").bfloat16()
    _same(lambda a, b: S.rotary(plan, a, b), [q, k], [_spread(store, q, strides), _spread(store, k, strides, 2 ** 30 + 64)], [torch.randn_like(q), torch.randn_like(k)])
    want = S.rotary(plan, q)
    far = _spread(store, q, strides)
    S.rotary(plan, far, inplace=True)
    assert torch.equal(far, want)


# (items, rows, heads, maps): rows and maps up to 2^24 - 8 elements apart, items and heads anywhere
@pytest.mark.parametrize("strides", [(FAR, 512, 256, 64), (2 ** 17, 512, FAR, 64), (64, 2 ** 24 - 1024, 2 ** 10, 2 ** 9), (2 ** 10, 2 ** 11, 2 ** 23, 2 ** 24 - 8)])
@pytest.mark.parametrize("Tq", [1, 140])
@pytest.mark.parametrize("causal", [False, True])
def test_differential_attention(store, strides, Tq, causal):
    from xva_trainer_amd import seq_ops as S
    B, Tk, H, d = 2, 150, 2, 32
    n = lambda *s: torch.randn(*s, device="cuda").bfloat16()
    q, k, v, dout, lam = n(B, Tq, H, 2, d), n(B, Tk, H, 2, d), n(B, Tk, H, 2 * d), n(B, Tq, H, 2 * d), torch.rand(H, device="cuda")
    # (v's rows hold 2 d columns where k's hold a map's d: the four tensors at distances that keep them apart)
    far = [_spread(store, q, strides), _spread(store, k, strides, 2 ** 14 * 3), _spread(store, v, strides[:3], 2 ** 14 * 7)]
    call = lambda q_, k_, v_, l: S.differential_attention(q_, k_, v_, l, causal=causal)
    near = [q, k, v]
    for i, t in enumerate(far):                                      # one at a time: views of one store may lie on each other
        _spread(store, near[i], t.stride()[:-1], t.storage_offset())
        _same(call, near + [lam], [t if j == i else near[j] for j in range(3)] + [lam], [dout])
    g = _spread(store, dout, strides[:3])
    leaves = [t.detach().requires_grad_(True) for t in near + [lam]]
    y = call(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, g, retain_graph=True), torch.autograd.grad(y, leaves, dout)))


@pytest.mark.parametrize("T,strides", [(700, (FAR, 64)), (1, (FAR, 64)), (5, (64, 2 ** 29)), (90, (64, 2 ** 25 + 64)), (600, (128, 2 ** 22))])
@pytest.mark.parametrize("reverse", [False, True])
def test_gated_recurrence(store, T, strides, reverse):
    """Against 64 bits: where rows lie too far apart for 32-bit offsets in a tile, other code runs (the same formulas, other fused products)."""
    from test_recurrence_gpu import _data, _run
    x, gate, h0, dh, dlast = _data(2, T, 64, "bf16", seed=15)
    _run(_spread(store, x, strides), gate, h0, dh, dlast, reverse=reverse)
    _run(x, _spread(store, gate, strides), h0, dh, dlast, reverse=reverse)
    _run(x, gate, h0, _spread(store, dh, strides), dlast, reverse=reverse)


@pytest.mark.parametrize("T,G,strides", [(1, 8, (FAR, 64)), (40, 8, (FAR, 64)), (300, 8, (64, 2 ** 23)), (3000, 2, (FAR, 64)), (3000, 2, (64, 2 ** 20)), (5, 8, (64, 2 ** 29))])
def test_group_norm(store, T, G, strides):
    from xva_trainer_amd import seq_ops as S
    x, w, b = torch.randn(2, T, 64, device="cuda").bfloat16(), torch.rand(64, device="cuda"), torch.rand(64, device="cuda")
    dy = torch.randn_like(x)
    call = lambda *a: S.group_norm_act(a[0], G, a[1], a[2], act="silu")
    _same(call, [x, w, b], [_spread(store, x, strides), w, b], [dy])
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = call(*leaves)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, dy, retain_graph=True), torch.autograd.grad(y, leaves, _spread(store, dy, strides))))
