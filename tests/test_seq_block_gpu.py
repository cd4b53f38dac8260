"""The sequence operators one after the other, as a block of an acoustic model uses them: group norm + silu -> q / k / v -> rotary positions -> differential attention ->
each head's norm -> gate and input -> gated recurrence; ragged, with the gradient of every input and weight, against the same block in 64 bits."""
import math

import pytest
import torch

from seq_util import lengths

pytestmark = pytest.mark.gpu


def _block(S, x, p, lens, H, Hk, d, plan, wide):
    """`wide` computes the products; S the operators (the package's, or `Plain` below)."""
    B, T, C = x.shape
    h = S.group_norm_act(x, 8, p["w1"], p["b1"], lens=lens, act="silu")
    q, k, v = wide(h, p["qkv"]).split((H * 2 * d, Hk * 2 * d, Hk * 2 * d), -1)
    q, k = S.rotary(plan, q.unflatten(-1, (2 * H, d)), k.unflatten(-1, (2 * Hk, d)))
    o = S.differential_attention(q.unflatten(2, (H, 2)), k.unflatten(2, (Hk, 2)), v.unflatten(-1, (Hk, 2 * d)), p["lam"], causal=True, q_lens=lens, k_lens=lens)
    o = S.group_norm_act(o.reshape(B * T, H * 2 * d), H, p["w2"], None)
    u, gate = wide(o.view(B, T, -1), p["ug"]).chunk(2, -1)
    y, last = S.gated_recurrence(u, gate + 1, p["h0"], lens=lens)
    return y, last


class Plain:
    @staticmethod
    def group_norm_act(x, G, w, b, lens=None, act="none"):
        flat = x.dim() == 2
        x = x[:, None] if flat else x
        B, T, C = x.shape
        live = torch.ones(B, T, 1, 1, dtype=x.dtype) if lens is None else (torch.arange(T)[None] < lens[:, None])[..., None, None].to(x.dtype)
        g = x.view(B, T, G, -1)
        n = live.sum((1, 3), keepdim=True).clamp_min(1) * (C // G)
        mu = (g * live).sum((1, 3), keepdim=True) / n
        var = ((g - mu).square() * live).sum((1, 3), keepdim=True) / n
        z = ((g - mu) * (var + 1e-5).rsqrt()).reshape(B, T, C) * w + (b if b is not None else 0)
        y = (z * torch.sigmoid(z) if act == "silu" else z) * live[..., 0]
        return y[:, 0] if flat else y

    @staticmethod
    def rotary(plan, q, k):
        def turn(x):
            ang = torch.arange(x.shape[1], dtype=x.dtype)[:, None, None] * torch.tensor(plan.frequencies, dtype=x.dtype)
            n = len(plan.frequencies)
            a, b, rest = x[..., :n], x[..., n:2 * n], x[..., 2 * n:]
            return torch.cat((a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), rest), -1)
        return turn(q), turn(k)

    @staticmethod
    def differential_attention(q, k, v, lam, causal, q_lens, k_lens):
        T, share = q.shape[1], q.shape[2] // k.shape[2]
        see = torch.arange(T)[None] <= torch.arange(T)[:, None]
        see = see[None] & (torch.arange(T)[None, :, None] < q_lens[:, None, None])          # (causal: keys behind the length are behind every live query)
        k, v = k.repeat_interleave(share, 2), v.repeat_interleave(share, 2)
        s = torch.einsum("bihmd,bjhmd->bhmij", q, k) * q.shape[-1] ** -0.5
        p = torch.nan_to_num(torch.softmax(s.masked_fill(~see[:, None, None], -math.inf), -1), nan=0.0)
        return torch.einsum("bhij,bjhe->bihe", p[:, :, 0] - lam[:, None, None] * p[:, :, 1], v)

    @staticmethod
    def gated_recurrence(x, gate, h, lens):
        f, out = torch.sigmoid(gate), []
        for t in range(x.shape[1]):
            live = (t < lens)[:, None]
            h = torch.where(live, f[:, t] * h + (1 - f[:, t]) * x[:, t], h)
            out.append(h * live)
        return torch.stack(out, 1), h


@pytest.mark.parametrize("dt,tol", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_block_forward_and_gradient(dt, tol):
    """Norm of the difference over the norm of the result.  Each of the ~12 tensors between input and output is rounded once, u = half a step; a tensor of
    independent roundings is off by at most u of its norm, and they pass through maps whose gains are a few at most (a norm over 64 values, differences of
    softmax maps with lam < 1): 40 u bounds forward and gradients."""
    from xva_trainer_amd import seq_ops as S
    torch.manual_seed(11)
    B, T, C, H, Hk, d = 3, 70, 64, 4, 2, 16
    lens = lengths(B, T, "some")
    p = {"w1": 1 + 0.1 * torch.randn(C), "b1": 0.1 * torch.randn(C), "qkv": torch.randn(H * 2 * d + Hk * 4 * d, C) * C ** -0.5, "lam": 0.2 + 0.1 * torch.rand(H),
         "w2": 1 + 0.1 * torch.randn(H * 2 * d), "ug": torch.randn(2 * C, H * 2 * d) * (H * 2 * d) ** -0.5, "h0": torch.randn(B, C)}
    p = {n: (t.to(dt).float() if n in ("qkv", "ug") else t) for n, t in p.items()}
    x, dy, dl = torch.randn(B, T, C).to(dt), torch.randn(B, T, C).to(dt), torch.randn(B, C)
    plan = S.RotaryPlan(16)
    mine = {n: (t.to(dt) if n in ("qkv", "ug") else t).cuda().requires_grad_(True) for n, t in p.items()}
    xm = x.cuda().requires_grad_(True)
    outs = _block(S, xm, mine, lens.cuda(), H, Hk, d, plan, lambda a, w: (a.float() @ w.float().T).to(dt))
    got = [o.detach() for o in outs] + list(torch.autograd.grad(outs, [xm] + list(mine.values()), (dy.cuda(), dl.cuda())))
    ref64 = {n: t.double().requires_grad_(True) for n, t in p.items()}
    x64 = x.double().requires_grad_(True)
    outs64 = _block(Plain, x64, ref64, lens.long(), H, Hk, d, plan, lambda a, w: a @ w.T)
    ref = [o.detach() for o in outs64] + list(torch.autograd.grad(outs64, [x64] + list(ref64.values()), (dy.double(), dl.double())))
    for name, a, b in zip(["y", "last", "dx"] + ["d" + n for n in p], got, ref):
        rel = ((a.double().cpu() - b).norm() / b.norm()).item()
        assert rel < 40 * tol, (name, rel)


def _calls(S):
    """name -> (call, leaves): each operator, small."""
    plan = S.RotaryPlan(8)
    n = lambda *s: torch.randn(*s, device="cuda").requires_grad_(True)
    half = lambda *s: torch.randn(*s, device="cuda").half().requires_grad_(True)
    return {"rotary": (lambda q, k: S.rotary(plan, q, k)[0], [n(2, 3, 2, 8), n(2, 3, 1, 8)]),
            "differential_attention": (S.differential_attention, [half(2, 5, 2, 2, 8), half(2, 5, 1, 2, 8), half(2, 5, 1, 16), n(2)]),
            "gated_recurrence": (lambda x, g, h: S.gated_recurrence(x, g, h)[0], [n(2, 5, 4), n(2, 5, 4), n(2, 4)]),
            "group_norm_act": (lambda x, w, b: S.group_norm_act(x, 2, w, b, act="silu"), [n(2, 5, 8), n(8), n(8)])}


@pytest.mark.parametrize("op", ["differential_attention", "gated_recurrence", "group_norm_act"])
def test_a_second_derivative_says_that_there_is_none(op):
    """A gradient penalty added to another loss must not lose its own gradient without a word; the first gradient is the usual one."""
    from xva_trainer_amd import seq_ops as S
    call, leaves = _calls(S)[op]
    want = torch.autograd.grad(call(*leaves).float().sum(), leaves)
    y = call(*leaves).float().sum()
    got = torch.autograd.grad(y, leaves, create_graph=True)
    assert all(torch.equal(a, b.detach()) for a, b in zip(want, got))
    for g in got:
        with pytest.raises(RuntimeError, match="differentiate twice"):
            (y + g.float().square().sum()).backward(retain_graph=True)


def test_a_rotation_of_a_constant_gradient_is_a_constant():
    """The rotation's gradient does not depend on what is rotated: its second derivative is nothing, unless the incoming gradient is a variable."""
    from xva_trainer_amd import seq_ops as S
    call, (q, k) = _calls(S)["rotary"]
    y = call(q, k)
    g, = torch.autograd.grad(y.sum(), q, create_graph=True)
    want, = torch.autograd.grad(y.sum(), q, retain_graph=True)
    got, = torch.autograd.grad(y.sum() + g.square().sum(), q)
    assert torch.equal(got, want)
    y = call(q, k)
    g, = torch.autograd.grad(y.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()


@pytest.mark.parametrize("op", ["rotary", "differential_attention", "gated_recurrence", "group_norm_act"])
def test_a_tangent_of_the_incoming_gradient_is_refused(op):
    import torch.autograd.forward_ad as fwd
    from xva_trainer_amd import seq_ops as S
    call, leaves = _calls(S)[op]
    y = call(*leaves)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, leaves[0], fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize("dt,tol", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_a_captured_step_of_a_serving_loop(dt, tol):
    """One frame of each stream: rotary positions in place, the frame's key and value into the cache, attention over it, each head's norm, the recurrence's step with its
    state carried on; captured once, replayed frame by frame.  Every frame against the same calls made eagerly (bit for bit, also the caches and the state), and all
    frames against one pass over the whole sequence, which takes other kernels: each of its five tensors is rounded the same way from sums that differ in fp32 alone,
    so a value differs where a rounding flips, by one step 2 u of itself; 10 u of the norm bounds five of them."""
    from xva_trainer_amd import seq_ops as S
    torch.manual_seed(12)
    B, T, H, Hk, d, C = 3, 40, 4, 2, 32, 64
    plan = S.RotaryPlan(d)
    q, k, v = (torch.randn(B, T, n, w, device="cuda").to(dt) for n, w in ((2 * H, d), (2 * Hk, d), (Hk, 2 * d)))
    lam, weight = torch.rand(H, device="cuda"), 1 + 0.1 * torch.randn(H * 2 * d, device="cuda")
    mix = (torch.randn(2 * C, H * 2 * d, device="cuda") * (H * 2 * d) ** -0.5).to(dt)

    class Stream:
        def __init__(self):
            z = lambda *s: torch.zeros(*s, device="cuda", dtype=dt)
            self.q, self.k, self.v, self.pos = z(B, 1, 2 * H, d), z(B, 1, 2 * Hk, d), z(B, 1, Hk, 2 * d), torch.zeros(1, device="cuda", dtype=torch.int64)
            self.keys, self.values, self.lens = z(B, T, Hk, 2, d), z(B, T, Hk, 2 * d), torch.zeros(B, device="cuda", dtype=torch.int32)
            self.state, self.y = torch.zeros(B, C, device="cuda"), z(B, 1, C)

        def feed(self, t):
            self.q.copy_(q[:, t:t + 1]), self.k.copy_(k[:, t:t + 1]), self.v.copy_(v[:, t:t + 1]), self.pos.fill_(t)

        def step(self):
            S.rotary(plan, self.q, self.k, positions=self.pos, inplace=True)
            self.keys.index_copy_(1, self.pos, self.k.unflatten(2, (Hk, 2)))
            self.values.index_copy_(1, self.pos, self.v)
            self.lens.copy_((self.pos + 1).expand(B))
            o = S.differential_attention(self.q.unflatten(2, (H, 2)), self.keys, self.values, lam, causal=True, k_lens=self.lens)
            o = S.group_norm_act(o.view(B, H * 2 * d), H, weight)
            u, gate = (o @ mix.T).view(B, 1, 2 * C).chunk(2, -1)
            h, last = S.gated_recurrence(u, gate, self.state)
            self.state.copy_(last), self.y.copy_(h)

    with torch.no_grad():
        warm, eager, captured = Stream(), Stream(), Stream()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            warm.feed(0), warm.step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.step()
        ys = []
        for t in range(T):
            captured.feed(t), eager.feed(t)
            graph.replay()
            eager.step()
            torch.cuda.synchronize()
            for name in ("q", "k", "keys", "values", "lens", "state", "y"):
                assert torch.equal(getattr(captured, name), getattr(eager, name)), (t, name)
            ys.append(captured.y.clone())
        qr, kr = S.rotary(plan, q, k)
        o = S.differential_attention(qr.unflatten(2, (H, 2)), kr.unflatten(2, (Hk, 2)), v, lam, causal=True)
        o = S.group_norm_act(o.reshape(B * T, H * 2 * d), H, weight)
        u, gate = (o @ mix.T).view(B, T, 2 * C).chunk(2, -1)
        whole, last = S.gated_recurrence(u, gate)
        ys = torch.cat(ys, 1)
        for a, b in ((ys, whole), (captured.state, last)):
            assert (a.double() - b.double()).norm().item() < 10 * tol * b.double().norm().item()


def test_lengths_of_64_bits():
    """Lengths beyond an item's rows mean all of them, those below zero none, also where 32 bits would take them for others."""
    from xva_trainer_amd import seq_ops as S
    T = 9
    long = torch.tensor([2 ** 63 - 1, 2 ** 32, 2 ** 32 + 3, 2 ** 31, -2 ** 40, 5, -2 ** 32 + 4], device="cuda")
    short = torch.tensor([T, T, T, T, 0, 5, 0], device="cuda", dtype=torch.int32)
    B = long.numel()
    x, g = torch.randn(B, T, 8, device="cuda"), torch.randn(B, T, 8, device="cuda")
    q, k, v = (torch.randn(B, T, 2, *s, device="cuda").bfloat16() for s in ((2, 8), (2, 8), (16,)))
    for call in (lambda l: S.group_norm_act(x, 2, lens=l), lambda l: S.gated_recurrence(x, g, lens=l)[0],
                 lambda l: S.differential_attention(q, k, v, torch.ones(2, device="cuda") * 0.3, q_lens=l, k_lens=l)):
        assert torch.equal(call(long), call(short))


def test_an_argument_without_memory_is_not_taken_for_one_left_out():
    """A weight, bias, first state, length or position that is a wrapper has no address, as one that was not given."""
    from test_seq_ops_cpu import Bare
    from xva_trainer_amd import seq_ops as S
    x, n = torch.randn(2, 5, 8, device="cuda"), torch.ones(8, device="cuda")
    lens, plan = torch.tensor([5, 2], device="cuda", dtype=torch.int32), S.RotaryPlan(8)
    q, k, v = (torch.randn(2, 5, 1, *s, device="cuda").half() for s in ((2, 8), (2, 8), (16,)))
    for call in (lambda: S.group_norm_act(x, 2, Bare(n)), lambda: S.group_norm_act(x, 2, n, Bare(n)), lambda: S.group_norm_act(x, 2, lens=Bare(lens)),
                 lambda: S.gated_recurrence(x, x, Bare(torch.zeros(2, 8))), lambda: S.gated_recurrence(x, x, lens=Bare(lens)),
                 lambda: S.rotary(plan, x[:, :, None], positions=Bare(torch.zeros(5, dtype=torch.int64))),
                 lambda: S.differential_attention(q, k, v, n[:1], q_lens=Bare(lens)), lambda: S.differential_attention(q, k, v, n[:1], k_lens=Bare(lens))):
        with pytest.raises(S.XvaError, match="without memory"):
            call()


def test_inference_mode():
    """Serving loops run in it: the same results, in place too, on its own tensors and on others."""
    from xva_trainer_amd import seq_ops as S
    torch.manual_seed(3)
    plan = S.RotaryPlan(8)
    made = lambda *s: torch.randn(*s, device="cuda")
    outside = [made(2, 5, 2, 8), made(2, 5, 2, 2, 8).half(), made(2, 5, 1, 2, 8).half(), made(2, 5, 1, 16).half(), made(2), made(2, 5, 8), made(2, 5, 8)]
    def calls(q, dq, dk, dv, lam, x, g):
        return [S.rotary(plan, q), S.differential_attention(dq, dk, dv, lam), S.gated_recurrence(x, g)[0], S.group_norm_act(x, 2, g[0, 0], act="gelu"), S.rotary(plan, q, inplace=True)]
    with torch.no_grad():
        want = calls(*[t.clone() for t in outside])
    with torch.inference_mode():
        for ts in ([t.clone() for t in outside], outside):
            assert all(torch.equal(a, b) for a, b in zip(calls(*ts), want))
