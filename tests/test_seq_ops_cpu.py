"""The sequence operators without a GPU: plans, the C structs' layout, refusals at the C entry points and of host tensors."""
import ctypes as C
import math
import os
import subprocess

import pytest
import torch

from seq_util import DiffAttentionArgs, GroupNormArgs, RecurrenceArgs, RotaryArgs, entry, i64
from xva_trainer_amd import _lib, seq_ops as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_plan_frequencies_as_turns():
    for kw in ({}, {"scaling": "linear", "factor": 4.0}, {"scaling": "ntk", "factor": 8.0}, {"scaling": "yarn", "factor": 16.0}):
        plan = S.RotaryPlan(64, device="cpu", **kw)
        for f, t in zip(plan.frequencies, plan.turns.tolist()):
            assert abs((t % 2 ** 64) / 2.0 ** 64 - f / (2 * math.pi)) <= 2.0 ** -52
    base = S.RotaryPlan(64, device="cpu").frequencies
    assert base[0] == 1.0 and math.isclose(base[16], 10000.0 ** -0.5)
    ntk = S.RotaryPlan(64, device="cpu", scaling="ntk", factor=8.0).frequencies
    assert ntk[0] == 1.0 and math.isclose(ntk[31], base[31] / 8.0)
    yarn = S.RotaryPlan(64, device="cpu", scaling="yarn", factor=16.0)
    assert yarn.frequencies[0] == base[0] and math.isclose(yarn.frequencies[31], base[31] / 16.0) and math.isclose(yarn.gain, 0.1 * math.log(16.0) + 1.0)
    assert all(a >= b for a, b in zip(yarn.frequencies, yarn.frequencies[1:]))


@pytest.mark.parametrize("bad", [dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, base=1.0),
                                 dict(rotary_dim=8, factor=0.5)])
def test_plan_refusals(bad):
    with pytest.raises(S.XvaError):
        S.RotaryPlan(device="cpu", **bad)


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 2, 8)
    for call in (lambda: S.rotary(S.RotaryPlan(8, device="cpu"), x), lambda: S.gated_recurrence(x[0], x[0]), lambda: S.group_norm_act(x[0], 2),
                 lambda: S.differential_attention(x[:, :, None].bfloat16(), x[:, :, None].bfloat16(), torch.zeros(1, 2, 1, 16).bfloat16(), torch.zeros(1))):
        with pytest.raises(S.XvaError, match="device tensors"):
            call()


STRUCTS = {"xva_rotary_args": RotaryArgs, "xva_group_norm_args": GroupNormArgs, "xva_recurrence_args": RecurrenceArgs,
           "xva_diff_attention_args": DiffAttentionArgs}


def test_structs_match_the_header(tmp_path):
    """Size and every field's offset, as a C compiler lays the header out (arrays by their elements)."""
    lines = []
    for name, t in STRUCTS.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        fields = [f for f, _ in t._fields_]
        for f in fields:
            base = f.rstrip("0123456789")
            array = base in ("q_stride", "k_stride", "v_stride", "q_out_stride", "k_out_stride", "pos_stride", "x_stride", "dy_stride", "out_stride", "dout_stride",
                             "gate_stride", "h_stride", "dh_stride", "dx_stride", "dgate_stride")
            at = "offsetof(%s, %s)" % (name, base if array else f)
            lines.append('printf("%%zu\\n", %s + %s * sizeof(int64_t));' % (at, f[len(base):] if array else "0"))
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "xva_hip.h"\nint main(void) {\n%s\nreturn 0; }\n' % "\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    said = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    mine = []
    for t in STRUCTS.values():
        mine.append(C.sizeof(t))
        mine += [getattr(t, f).offset for f, _ in t._fields_]
    assert said == mine


A = 1 << 20        # an address for arguments that are refused before anything reads them


def _diff(**kw):
    base = dict(q=A, k=A, v=A, lam=A, out=A, dtype=1, B=1, Tq=4, Tk=4, H=2, Hk=1, d=16, causal=0, scale=0.25)
    return DiffAttentionArgs(**{**base, **kw})


@pytest.mark.parametrize("bad,says", [(dict(q=None), "null"), (dict(dtype=0), "dtype"), (dict(d=12), "head width"), (dict(d=72), "head width"), (dict(Hk=0), "Hk"),
                                      (dict(H=3, Hk=2), "Hk"), (dict(B=-1), "B -1"), (dict(scale=0.0), "scale"), (dict(q=A + 2), "aligned"),
                                      (dict(k_stride1=4), "strides"), (dict(out=None), "null"), (dict(lse=A), "null"), (dict(Tq=1 << 30), "Tq")])
def test_diff_attention_refuses(bad, says):
    assert entry("xva_diff_attention_fwd")(C.byref(_diff(**bad)), None, 0, None) < 0
    assert says in _lib.lib.xva_last_error().decode()


def test_diff_attention_backward_refuses_a_small_workspace():
    a = _diff(dout=A, maps=A, lse=A, dq=A, dk=A, dv=A, dlam=A)
    need = entry("xva_diff_attention_workspace_bytes", i64)(C.byref(a), 1)
    assert need > 0
    assert entry("xva_diff_attention_bwd")(C.byref(a), A, need - 1, None) == -3
    assert entry("xva_diff_attention_bwd")(C.byref(a), None, need, None) == -3
    assert entry("xva_diff_attention_bwd")(C.byref(_diff()), A, need, None) < 0


@pytest.mark.parametrize("bad,says", [(dict(q=None), "null"), (dict(turns=None), "null"), (dict(dtype=3), "dtype"), (dict(rd=3), "rotary width"), (dict(rd=34), "rotary width"),
                                      (dict(D=9000), "rotary width"), (dict(k=None), "null keys"), (dict(q_out=A), "in place"), (dict(q_out=A, k_out=A), "other strides"),
                                      (dict(B=1 << 20, T=1 << 12), "tokens"), (dict(H=0), "H 0")])
def test_rotary_refuses(bad, says):
    base = dict(q=A, k=A, q_out=2 * A, k_out=2 * A, turns=A, dtype=0, B=1, T=2, H=2, Hk=1, D=32, rd=32, gain=1.0, q_stride0=64)
    assert entry("xva_rotary")(C.byref(RotaryArgs(**{**base, **bad})), None) < 0
    assert says in _lib.lib.xva_last_error().decode()


@pytest.mark.parametrize("bad,says", [(dict(x=None), "null"), (dict(mean=None), "null"), (dict(dtype=-1), "dtype"), (dict(G=5), "groups"), (dict(G=0), "groups"),
                                      (dict(act=9), "activation"), (dict(eps=-1.0), "eps"), (dict(T=500, C=16384, G=2), "vectors"), (dict(T=600, C=4096, G=4096), "2048 groups"),
                                      (dict(T=3500, C=16384, G=4096, dtype=2), "2048 groups"),     # (the forward alone could: its backward could not)
                                      (dict(T=500, C=1025, G=1), "vectors")])
def test_group_norm_refuses(bad, says):
    base = dict(x=A, out=A, mean=A, rstd=A, dtype=1, B=2, T=3, C=32, G=4, act=0, eps=1e-5)
    assert entry("xva_group_norm_act_fwd")(C.byref(GroupNormArgs(**{**base, **bad})), None, 0, None) < 0
    assert says in _lib.lib.xva_last_error().decode()


def test_group_norm_refuses_a_small_workspace():
    a = GroupNormArgs(x=A, dy=A, out=A, mean=A, rstd=A, dtype=1, B=2, T=3000, C=32, G=4, act=0, eps=1e-5)
    for bwd, call in ((0, entry("xva_group_norm_act_fwd")), (1, entry("xva_group_norm_act_bwd"))):
        need = entry("xva_group_norm_workspace_bytes", i64)(C.byref(a), bwd)
        assert need > 0 and call(C.byref(a), A, need - 1, None) == -3


@pytest.mark.parametrize("bad,says", [(dict(x=None), "null"), (dict(last=None), "null"), (dict(dtype=5), "dtype"), (dict(C=0), "C 0"), (dict(T=-1), "T -1"),
                                      (dict(B=1 << 20, C=1 << 12), "B ")])
def test_recurrence_refuses(bad, says):
    base = dict(x=A, gate=A, h=A, last=A, dtype=0, B=2, T=3, C=8)
    assert entry("xva_recurrence_fwd")(C.byref(RecurrenceArgs(**{**base, **bad})), None, 0, None) < 0
    assert says in _lib.lib.xva_last_error().decode()


def test_recurrence_refuses_a_small_workspace():
    need = entry("xva_recurrence_workspace_bytes", i64)(1, 30000, 64)
    assert need > 0
    assert entry("xva_recurrence_fwd")(C.byref(RecurrenceArgs(x=A, gate=A, h=A, last=A, dtype=0, B=1, T=30000, C=64)), A, need - 1, None) == -3
    assert entry("xva_recurrence_bwd")(C.byref(RecurrenceArgs(x=A, gate=A, dtype=0, B=1, T=30000, C=64)), A, need, None) < 0


@pytest.mark.parametrize("T,channels,G", [(1, 64, 4), (300, 64, 4), (5000, 32, 1), (500, 33, 1), (500, 1025, 1)])
@pytest.mark.parametrize("B,T0", [(0, None), (3, 0)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_group_norm_without_items_or_rows(T, channels, G, B, T0, dtype):
    """At the shapes of all three forms: no workspace and nothing launched (dweight and dbias, which would be zeroed, are not asked for)."""
    a = GroupNormArgs(dtype=dtype, B=B, T=T if T0 is None else T0, C=channels, G=G, act=0, eps=1e-5)
    for bwd, call in ((0, entry("xva_group_norm_act_fwd")), (1, entry("xva_group_norm_act_bwd"))):
        assert entry("xva_group_norm_workspace_bytes", i64)(C.byref(a), bwd) == 0
        assert call(C.byref(a), None, 0, None) == 0


@pytest.mark.parametrize("T", [1, 200, 3000])
def test_group_norm_refuses_a_null_workspace(T):
    a = GroupNormArgs(x=A, dy=A, out=A, mean=A, rstd=A, dtype=1, B=2, T=T, C=32, G=4, act=0, eps=1e-5)
    for bwd, call in ((0, entry("xva_group_norm_act_fwd")), (1, entry("xva_group_norm_act_bwd"))):
        need = entry("xva_group_norm_workspace_bytes", i64)(C.byref(a), bwd)
        if need > 0:
            assert call(C.byref(a), None, need, None) == -3


@pytest.mark.parametrize("dtype", [0, 1])
def test_group_norm_takes_weights_at_any_address(dtype):
    """2048 channels need vectors of x; the weights' address does not take them away (the call gets as far as its workspace)."""
    for at in (dict(weight=A + 4), dict(bias=A + 4), dict(weight=A + 8, bias=A + 12)):
        a = GroupNormArgs(x=A, dy=A, out=A, mean=A, rstd=A, dtype=dtype, B=2, T=300, C=2048, G=4, act=0, eps=1e-5, x_stride0=300 * 2048, x_stride1=2048, out_stride0=300 * 2048,
                          out_stride1=2048, dy_stride0=300 * 2048, dy_stride1=2048, **at)
        assert entry("xva_group_norm_act_fwd")(C.byref(a), None, 0, None) == -3
        assert entry("xva_group_norm_act_bwd")(C.byref(a), None, 0, None) == -3


def _every_call():
    """Each operator on host tensors; (x, others): the call takes a tensor like x in x's place."""
    plan, x, lam = S.RotaryPlan(8, device="cpu"), torch.zeros(1, 2, 2, 8), torch.zeros(2)
    half = torch.zeros(1, 2, 2, 2, 8).half()
    return {"rotary q": (x, lambda t: S.rotary(plan, t)), "rotary k": (x, lambda t: S.rotary(plan, x, t)),
            "attention q": (half, lambda t: S.differential_attention(t, half, half[:, :, :, 0].repeat(1, 1, 1, 2), lam)),
            "attention lam": (lam, lambda t: S.differential_attention(half, half, half[:, :, :, 0].repeat(1, 1, 1, 2), t)),
            "recurrence gate": (x[0], lambda t: S.gated_recurrence(x[0], t)), "recurrence h0": (x[0, 0], lambda t: S.gated_recurrence(x[0], x[0], t)),
            "norm x": (x[0], lambda t: S.group_norm_act(t, 2)), "norm bias": (x[0, 0, 0], lambda t: S.group_norm_act(x[0], 2, None, t))}


@pytest.mark.parametrize("which", list(_every_call()))
def test_forward_mode_and_tracing_are_refused(which):
    """A tangent would be dropped and a trace would hold no launch, both without a word (refused before the device is looked at)."""
    import torch.autograd.forward_ad as fwd
    x, call = _every_call()[which]
    with fwd.dual_level():
        with pytest.raises(S.XvaError, match="forward-mode"):
            call(fwd.make_dual(x, torch.ones_like(x)))
    with pytest.raises(S.XvaError, match="device tensors"):
        call(x)
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(call, (x,), check_trace=False)


def test_views_that_share_elements_are_told_apart_from_those_that_do_not():
    """Every answer against the elements themselves; views as slices of projections have them, and any strides.  "Not known" (2) is refused like a meeting: it may
    only be said of strides that no slice has."""
    import random

    from xva_trainer_amd import _seq_torch
    rng, store = random.Random(5), torch.zeros(4000)
    places = lambda t: [torch.arange(t.shape[3])[None] + (torch.cartesian_prod(*[torch.arange(n) for n in t.shape[:3]]) * torch.tensor(t.stride()[:3])).sum(1, keepdim=True)
                        + t.storage_offset()][0]
    said = {0: 0, 1: 0, 2: 0}
    for turn in range(3000):
        shape = [rng.randint(1, 4) for _ in range(3)] + [rng.randint(2, 6)]
        if turn % 2:                                                    # slices of one projection, in either order of heads and rows
            heads, width = rng.randint(1, 5), shape[3] + rng.choice([0, 0, 1, 3])
            whole = store[:shape[0] * shape[1] * heads * width].view(shape[0], shape[1], heads, width)
            cut = lambda: (lambda a, d: whole[:, :, a:rng.randint(a + 1, heads), d:d + shape[3]])(rng.randint(0, heads - 1), rng.randint(0, width - shape[3]))
            q, k = cut(), cut()
            if rng.random() < 0.3:
                q, k = q.transpose(1, 2), k.transpose(1, 2)
            k = k[:, :q.shape[1]]
            q = q[:, :k.shape[1]]
        else:
            view = lambda n: store.as_strided(shape[:2] + [n, shape[3]], [rng.choice([0, 1, 5, 7, 24, 60, 100]) for _ in range(3)] + [1], rng.randint(0, 60))
            q, k = view(shape[2]), view(rng.randint(1, 4))
        at = [places(t).flatten() for t in (q, k)]
        for t, a in zip((q, k), at):
            own = _seq_torch.overlap(t, None)
            said[own] += 1
            # (elements of a head never meet: a place that comes twice belongs to two heads)
            assert own == (1 if a.unique().numel() < a.numel() else 0), (t.shape, t.stride())
        both = _seq_torch.overlap(q, k)
        said[both] += 1
        assert both == int(torch.isin(at[0], at[1]).any()), (q.shape, q.stride(), q.storage_offset(), k.shape, k.stride(), k.storage_offset())
    assert said[0] > 500 and said[1] > 500 and said[2] == 0
    whole = torch.zeros(64, 512, 24, 128)                                # sizes of a model
    assert _seq_torch.overlap(whole[:, :, :16], whole[:, :, 16:]) == 0 and _seq_torch.overlap(whole[:, :, :17], whole[:, :, 16:]) == 1
    assert _seq_torch.overlap(whole[..., :64], whole[..., 64:]) == 0 and _seq_torch.overlap(whole, torch.zeros(64, 512, 2, 128)) == 0
    assert _seq_torch.overlap(whole.transpose(1, 2)[:, :16], whole.transpose(1, 2)[:, 16:20]) == 0


@pytest.mark.parametrize("kw", [{}, {"base": 500000.0}, {"scaling": "linear", "factor": 3.0}, {"scaling": "ntk", "factor": 8.0}, {"scaling": "yarn", "factor": 16.0}])
@pytest.mark.parametrize("rd", [2, 6, 64, 254])
def test_turns_to_half_a_unit(kw, rd):
    """The table against the definition in 80 digits, each power by itself: half a unit of 2^-64 of a turn (and a billionth of one for the digits)."""
    from decimal import Decimal as D, getcontext, localcontext
    plan = S.RotaryPlan(rd, device="cpu", **kw)
    with localcontext():
        getcontext().prec = 80
        pi = D("3.141592653589793238462643383279502884197169399375105820974944592307816406286208998628034825")
        base, factor, scaling = D(kw.get("base", 10000.0)), D(kw.get("factor", 1.0)), kw.get("scaling", "none")
        if scaling == "ntk" and rd > 2:
            base = base * factor ** (D(rd) / D(rd - 2))
        for i, t in enumerate(plan.turns.tolist()):
            f = base ** (D(-2 * i) / D(rd))
            if scaling == "linear":
                f = f / factor
            elif scaling == "yarn":
                pair = lambda turns: rd * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
                low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rd - 1)
                ramp = min(max(D(i - low) / D(max(high - low, 1e-3)), D(0)), D(1))
                f = f * (1 - ramp) + f / factor * ramp
            assert abs(D(t % 2 ** 64) - f / (2 * pi) * 2 ** 64) <= D(1) / 2 + D(10) ** -9, i


@pytest.mark.parametrize("T", [1 << 30, (1 << 31) - 300, (1 << 31) - 1])
@pytest.mark.parametrize("channels", [1, 32])
def test_group_norm_refuses_rows_that_int32_cannot_step_over(T, channels):
    a = GroupNormArgs(x=A, dy=A, out=A, mean=A, rstd=A, dtype=1, B=1, T=T, C=channels, G=1, act=0, eps=1e-5)
    for bwd, call in ((0, entry("xva_group_norm_act_fwd")), (1, entry("xva_group_norm_act_bwd"))):
        assert entry("xva_group_norm_workspace_bytes", i64)(C.byref(a), bwd) == -1
        assert call(C.byref(a), None, 0, None) == -1 and "T %d" % T in _lib.lib.xva_last_error().decode()


@pytest.mark.parametrize("dtype,channels", [(0, 1 << 29), (1, 1 << 30), (2, (1 << 31) - 1)])
def test_recurrence_refuses_rows_of_two_gigabytes(dtype, channels):
    """Offsets within a row are 32 bits (h null: a call that gets past this is refused for that)."""
    a = RecurrenceArgs(x=A, gate=A, h=None, last=A, dtype=dtype, B=1, T=1, C=channels)
    assert entry("xva_recurrence_fwd")(C.byref(a), None, 0, None) == -1
    assert "2^31 bytes" in _lib.lib.xva_last_error().decode()
    assert entry("xva_recurrence_fwd")(C.byref(RecurrenceArgs(x=A, gate=A, h=None, last=A, dtype=dtype, B=1, T=1, C=channels // 2)), None, 0, None) == -1
    assert "null" in _lib.lib.xva_last_error().decode()


def test_launches_that_the_runtime_would_cut_are_refused():
    """2^32 threads or more along a dimension run as that number modulo 2^32, without an error: refused before anything is launched (workspaces null, so that a call that
    gets past the check is refused too, with another code)."""
    said = lambda: _lib.lib.xva_last_error().decode()
    rotary = RotaryArgs(q=A, q_out=2 * A, turns=A, dtype=1, B=1 << 14, T=1 << 14, H=1, D=2, rd=2, gain=1.0)
    assert entry("xva_rotary")(C.byref(rotary), None) == -1 and "tokens" in said()
    for T, B in ((1, 1 << 26), (5000, 1 << 23)):                       # a wave to an item, eight waves
        a = RecurrenceArgs(x=A, gate=A, h=A, last=A, states=A, dh=A, dx=A, dgate=A, dtype=1, B=B, T=T, C=1)
        assert entry("xva_recurrence_fwd")(C.byref(a), None, 0, None) == -1 and "too many items" in said()
        assert entry("xva_recurrence_bwd")(C.byref(a), None, 0, None) == -1 and "too many items" in said()
    for T, channels in ((600, 1), (1100, 8)):
        a = GroupNormArgs(x=A, dy=A, out=A, mean=A, rstd=A, dtype=1, B=(1 << 24), T=T, C=channels, G=1, act=0, eps=1e-5, x_stride0=T * channels, x_stride1=channels,
                          out_stride0=T * channels, out_stride1=channels, dy_stride0=T * channels, dy_stride1=channels)
        assert entry("xva_group_norm_act_bwd")(C.byref(a), None, 0, None) == -1 and "items" in said()
    fwd, bwd = entry("xva_diff_attention_fwd"), entry("xva_diff_attention_bwd")
    one = dict(H=1, Hk=1, d=8)
    for kw in (dict(B=1 << 24, Tq=1, Tk=1), dict(B=1 << 20, Tq=1 << 10, Tk=1), dict(B=1 << 20, Tq=1, Tk=1 << 10)):
        assert fwd(C.byref(_diff(**one, **kw)), None, 0, None) == -1 and "too many" in said()
    back = dict(dout=A, maps=A, lse=A, dq=A, dk=A, dv=A, dlam=A)
    for kw in (dict(B=1 << 20, Tq=256, Tk=1), dict(B=1 << 20, Tq=1, Tk=256)):
        assert bwd(C.byref(_diff(**one, **back, **kw)), None, 0, None) == -1 and "too many" in said()
    assert bwd(C.byref(_diff(**one, **back, B=1 << 20, Tq=1, Tk=1)), None, 0, None) == -3


class Bare(torch.Tensor):
    """A wrapper without memory of its own that says it is on a GPU."""
    @staticmethod
    def __new__(cls, like):
        return torch.Tensor._make_wrapper_subclass(cls, like.shape, dtype=like.dtype, device=torch.device("cuda:0"))

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError("%s reached" % func)


def test_tensors_without_memory_are_refused():
    plan = S.RotaryPlan(8, device="cpu")
    plan.turns = Bare(plan.turns)
    x, half = Bare(torch.zeros(1, 2, 2, 8)), Bare(torch.zeros(1, 2, 2, 2, 8).half())
    for call in (lambda: S.rotary(plan, x), lambda: S.gated_recurrence(Bare(torch.zeros(1, 2, 8)), Bare(torch.zeros(1, 2, 8))), lambda: S.group_norm_act(Bare(torch.zeros(1, 2, 8)), 2),
                 lambda: S.differential_attention(half, half, Bare(torch.zeros(1, 2, 2, 16).half()), Bare(torch.zeros(2)))):
        with pytest.raises(S.XvaError, match="without memory"):
            call()
