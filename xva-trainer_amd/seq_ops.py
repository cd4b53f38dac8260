"""Sequence operators on time-major device tensors: rotary positions, differential attention, a gated linear recurrence and group normalisation with an
activation (csrc/rotary.hip, diff_attention.hip, recurrence.hip, group_norm.hip; C ABI in include/xva_hip.h).

  RotaryPlan(rotary_dim, ...), rotary(plan, q, k)                 positions turned into the heads of queries and keys
  differential_attention(q, k, v, lam, ...)                       (softmax(q1 k1^T) - lam softmax(q2 k2^T)) v, shared key heads, ragged, causal
  gated_recurrence(x, gate, h0, ...)                              h_t = f_t h_{t-1} + (1 - f_t) x_t, f = sigmoid(gate)
  group_norm_act(x, groups, weight, bias, ...)                    act(group_norm(x)), channels last

The reference has none of these (its text encoder is `RelativePositionMultiHeadAttention`, python/xvapitch/glow_tts.py:173-292, its norms are layer norms,
:34-56); they are what a changed acoustic model is built from.  Tensors are fp32, bf16 or fp16 (attention: bf16 / fp16) with any strides over all but the last
dimension; one that is not contiguous in the last, or not aligned as a kernel needs it, is copied first.  Ragged batches give `lens` (B,) int32: rows at or
behind an item's length are not read, and are zero in the results.  Everything is differentiable through torch.autograd, launches on torch's current stream of
the tensors' device, does not synchronise and can be captured into a graph (a backward pass, as with every torch operator, only while no eager graph of the same
leaves lives: torch would tie the capture to the eager graph's stream).  There is no CPU fallback."""
import ctypes as C
import math

import torch

from . import _lib

lib = _lib.lib
i32, i64, f32, vp = C.c_int32, C.c_int64, C.c_float, C.c_void_p
XvaError = _lib.XvaError


def _fields(*spec):
    """[(name, type)] of a C struct; "name[n]" stands for n fields name0 .. (the layout of an array)."""
    out = []
    for names, t in spec:
        for n in names.split():
            if n.endswith("]"):
                n, count = n[:-1].split("[")
                out += [("%s%d" % (n, e), t) for e in range(int(count))]
            else:
                out.append((n, t))
    return out


class _RotaryArgs(C.Structure):
    _fields_ = _fields(("q k q_out k_out", vp), ("q_stride[3] k_stride[3] q_out_stride[3] k_out_stride[3]", i64), ("turns positions", vp), ("pos_stride[2]", i64),
                       ("positions64 dtype B T H Hk D rd interleaved inverse", i32), ("gain", f32))


class _GroupNormArgs(C.Structure):
    _fields_ = _fields(("x dy out", vp), ("x_stride[2] dy_stride[2] out_stride[2]", i64), ("weight bias mean rstd dweight dbias lens", vp),
                       ("dtype B T C G act", i32), ("eps slope", f32))


class _RecurrenceArgs(C.Structure):
    _fields_ = _fields(("x gate h h0 last states dh dlast dx dgate dh0 lens", vp),
                       ("x_stride[2] gate_stride[2] h_stride[2] dh_stride[2] dx_stride[2] dgate_stride[2]", i64), ("dtype B T C reverse unit_gain", i32))


class _DiffAttentionArgs(C.Structure):
    _fields_ = _fields(("q k v lam out maps lse dout dq dk dv dlam q_lens k_lens", vp), ("q_stride[4] k_stride[4] v_stride[3] out_stride[3] dout_stride[3]", i64),
                       ("dtype B Tq Tk H Hk d causal", i32), ("scale", f32))


lib.xva_rotary.argtypes = [C.POINTER(_RotaryArgs), vp]
for _n, _t in (("group_norm_act", _GroupNormArgs), ("recurrence", _RecurrenceArgs), ("diff_attention", _DiffAttentionArgs)):
    for _d in ("fwd", "bwd"):
        _f = getattr(lib, "xva_%s_%s" % (_n, _d))
        _f.restype, _f.argtypes = i32, [C.POINTER(_t), vp, i64, vp]
lib.xva_group_norm_workspace_bytes.restype, lib.xva_group_norm_workspace_bytes.argtypes = i64, [C.POINTER(_GroupNormArgs), i32]
lib.xva_diff_attention_workspace_bytes.restype, lib.xva_diff_attention_workspace_bytes.argtypes = i64, [C.POINTER(_DiffAttentionArgs), i32]
lib.xva_recurrence_workspace_bytes.restype, lib.xva_recurrence_workspace_bytes.argtypes = i64, [i32, i32, i32]
lib.xva_recurrence_state_floats.restype, lib.xva_recurrence_state_floats.argtypes = i64, [i32, i32, i32]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {"none": 0, "relu": 1, "lrelu": 2, "tanh": 3, "silu": 4, "gelu": 5}


def _refuse(cond, msg, *args):
    if cond:
        raise XvaError(msg % args)


def _device(first, *others):
    """All on one GPU; entered as the current device where it is not (launches and allocations go there)."""
    _refuse(not first.is_cuda, "libxvahip ops need device tensors; got a %s tensor (no CPU fallback exists)", first.device)
    for t in others:
        _refuse(t is not None and t.device != first.device, "tensors on %s and %s", first.device, t.device if t is not None else None)
    return first.device


class _on:
    """`with _on(device)`: torch.cuda.device, but free where the device is the current one."""
    __slots__ = ("guard",)

    def __init__(self, device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)


def _run(rc, what):
    if rc != 0:
        _lib.check(rc, what)


def _p(t):
    return t.data_ptr() if t is not None else None


def _lens(lens, B, device, what="lens"):
    if lens is None:
        return None
    _refuse(lens.dim() != 1 or lens.shape[0] != B, "%s: %s, expected (%d,)", what, tuple(lens.shape), B)
    _refuse(lens.dtype not in (torch.int32, torch.int64), "%s: int32 or int64, got %s", what, lens.dtype)
    _refuse(lens.device != device, "%s on %s, the tensors on %s", what, lens.device, device)
    return lens.to(torch.int32).contiguous()


def _rows(t):
    """`t` with a contiguous last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------------------------------------------------------ rotary ----
class RotaryPlan:
    """Frequencies of rotary positions, kept on a device.

    rotary_dim   how many of a head's first elements turn (even); the rest pass
    base         pair i of n = rotary_dim / 2 turns by base^(-i / n) radians per position
    interleaved  pairs are elements (2 i, 2 i + 1); otherwise (i, i + n)
    scaling      for contexts `factor` times longer than the model was trained on:
                 "none"; "linear": positions divided by the factor; "ntk": the base raised to base * factor^(d / (d - 2)), which leaves the fastest pair
                 alone and divides the slowest by the factor; "yarn": pairs that make more than `beta_fast` turns over `original_length` positions are left
                 alone, those under `beta_slow` divided by the factor, a ramp between, and cosines and sines times 0.1 ln(factor) + 1 (or `gain`)."""

    def __init__(self, rotary_dim, base=10000.0, interleaved=False, scaling="none", factor=1.0, original_length=4096, beta_fast=32.0, beta_slow=1.0, gain=None,
                 device="cuda"):
        _refuse(rotary_dim < 2 or rotary_dim % 2, "rotary_dim %d: an even number of elements", rotary_dim)
        _refuse(scaling not in ("none", "linear", "ntk", "yarn"), "scaling %r: none, linear, ntk or yarn", scaling)
        _refuse(not (base > 1.0 and factor >= 1.0 and original_length >= 1), "base %g, factor %g, original_length %d", base, factor, original_length)
        n = rotary_dim // 2
        self.rotary_dim, self.interleaved, self.gain = rotary_dim, bool(interleaved), 1.0
        if scaling == "ntk" and rotary_dim > 2:
            base = base * factor ** (rotary_dim / (rotary_dim - 2.0))
        freq = [base ** (-2.0 * i / rotary_dim) for i in range(n)]
        if scaling == "linear":
            freq = [f / factor for f in freq]
        elif scaling == "yarn":
            def pair_of(turns):
                return rotary_dim * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
            low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
            for i in range(n):
                ramp = min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0)
                freq[i] = freq[i] * (1.0 - ramp) + freq[i] / factor * ramp
            self.gain = 0.1 * math.log(factor) + 1.0
        if gain is not None:
            self.gain = float(gain)
        self.frequencies = freq
        # fractions of a turn per position as 64-bit fixed point (two's complement: the upper half reads as negative)
        fixed = [int(round(f / (2.0 * math.pi) * 2.0 ** 64)) % 2 ** 64 for f in freq]
        self.turns = torch.tensor([v - 2 ** 64 if v >= 2 ** 63 else v for v in fixed], dtype=torch.int64).to(device)

    def to(self, device):
        self.turns = self.turns.to(device)
        return self


def _rotary_launch(plan, q, k, pos, inverse, inplace):
    B, T, H, D = q.shape
    q = _rows(q)
    qo = q if inplace else torch.empty((B, T, H, D), device=q.device, dtype=q.dtype)
    if k is not None:
        k = _rows(k)
        ko = k if inplace else torch.empty(k.shape, device=q.device, dtype=q.dtype)
        ks, kos, Hk = k.stride(), ko.stride(), k.shape[2]
    else:
        ko, ks, kos, Hk = None, (0, 0, 0), (0, 0, 0), 0
    qs, qos = q.stride(), qo.stride()
    pb, pt = (0, 0) if pos is None else (pos.stride() if pos.dim() == 2 else (0, pos.stride(0)))
    if pos is not None:
        pb, pt = (0 if pos.dim() == 2 and pos.shape[0] == 1 else pb), (0 if pos.shape[-1] == 1 else pt)
    a = _RotaryArgs(q.data_ptr(), _p(k), qo.data_ptr(), _p(ko), qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], qos[0], qos[1], qos[2], kos[0], kos[1], kos[2],
                    plan.turns.data_ptr(), _p(pos), pb, pt, int(pos is not None and pos.dtype == torch.int64), _DTYPES[q.dtype], B, T, H, Hk, D, plan.rotary_dim,
                    int(plan.interleaved), int(inverse), plan.gain)
    _run(lib.xva_rotary(C.byref(a), _lib.raw_stream(q.device)), "xva_rotary")
    return qo, ko


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, plan):
        ctx.plan, ctx.pos = plan, pos
        qo, ko = _rotary_launch(plan, q, k, pos, False, False)
        return (qo, ko) if k is not None else qo

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        with _on(dq.device):
            gq, gk = _rotary_launch(ctx.plan, dq, dk, ctx.pos, True, False)
        return gq, gk, None, None


def rotary(plan, q, k=None, positions=None, inplace=False):
    """Turns q (B, T, H, D) and, if given, k (B, T, Hk, D) by their positions: (B, T) or (T,), a dimension of 1 standing for all, int32 or int64;
    None: 0 .. T - 1.  Returns q', or (q', k').  inplace: writes over q and k (no gradient)."""
    dev = _device(q, k, positions, plan.turns)
    _refuse(q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3])), "q %s, k %s: (B, T, heads, D)",
            tuple(q.shape), tuple(k.shape) if k is not None else None)
    _refuse(q.dtype not in _DTYPES or (k is not None and k.dtype != q.dtype), "q is %s, k %s", q.dtype, k.dtype if k is not None else None)
    _refuse(plan.rotary_dim > q.shape[3], "rotary_dim %d of heads of %d", plan.rotary_dim, q.shape[3])
    if positions is not None:
        _refuse(positions.dtype not in (torch.int32, torch.int64), "positions: int32 or int64, got %s", positions.dtype)
        _refuse(positions.dim() not in (1, 2) or positions.shape[-1] not in (1, q.shape[1]) or (positions.dim() == 2 and positions.shape[0] not in (1, q.shape[0])),
                "positions %s of (%d, %d) rows", tuple(positions.shape), q.shape[0], q.shape[1])
    grad = _needs_grad(q, k)
    _refuse(inplace and (grad or q.stride(-1) != 1 or (k is not None and k.stride(-1) != 1)), "inplace: no gradient, and a contiguous last dimension")
    with _on(dev):
        if grad:
            return _Rotary.apply(q, k, positions, plan)
        qo, ko = _rotary_launch(plan, q, k, positions, False, inplace)
    return (qo, ko) if k is not None else qo


# -------------------------------------------------------------------------------------------------------- differential attention ----
def _wide(t):
    """`t` as the attention kernels read it: 16-byte rows, 64 of them and their maps within 32-bit offsets."""
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0 and not any(s % 8 for s in st[:-1]) and st[1] < 1 << 24 and st[3] < 1 << 24:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _diff_args(q, k, v, lam, out, maps, lse, dout, dq, dk, dv, dlam, ql, kl, causal, scale):
    B, Tq, H, _, d = q.shape
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), out.stride() if out is not None else (0, 0, 0)
    gs = dout.stride() if dout is not None else (0, 0, 0)
    return _DiffAttentionArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), _p(out), _p(maps), _p(lse), _p(dout), _p(dq), _p(dk), _p(dv), _p(dlam),
                              _p(ql), _p(kl), qs[0], qs[1], qs[2], qs[3], ks[0], ks[1], ks[2], ks[3], vs[0], vs[1], vs[2], os[0], os[1], os[2], gs[0], gs[1], gs[2],
                              _DTYPES[q.dtype], B, Tq, k.shape[1], H, k.shape[2], d, int(causal), scale)


def _workspace(n, device):
    return torch.empty(n, device=device, dtype=torch.uint8) if n else None


def _diff_forward(q, k, v, lam, ql, kl, causal, scale, train):
    B, Tq, H, _, d = q.shape
    out = torch.empty((B, Tq, H, 2 * d), device=q.device, dtype=q.dtype)
    maps = torch.empty((2, B, Tq, H, 2 * d), device=q.device, dtype=q.dtype) if train else None
    lse = torch.empty((2, B, H, Tq), device=q.device, dtype=torch.float32) if train else None
    a = _diff_args(q, k, v, lam, out, maps, lse, None, None, None, None, None, ql, kl, causal, scale)
    n = lib.xva_diff_attention_workspace_bytes(C.byref(a), 0)
    ws = _workspace(n, q.device)
    _run(lib.xva_diff_attention_fwd(C.byref(a), _p(ws), n, _lib.raw_stream(q.device)), "xva_diff_attention_fwd")
    return out, maps, lse


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, ql, kl, causal, scale):
        out, maps, lse = _diff_forward(q, k, v, lam, ql, kl, causal, scale, True)
        ctx.save_for_backward(q, k, v, lam, maps, lse, ql, kl)
        ctx.how = (causal, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, lam, maps, lse, ql, kl = ctx.saved_tensors
        with _on(q.device):
            dout = _wide(dout.to(q.dtype))
            dq, dk, dv = (torch.empty(t.shape, device=q.device, dtype=q.dtype) for t in (q, k, v))
            dlam = torch.empty_like(lam)
            if q.numel() == 0:
                for t in (dk, dv, dlam):
                    t.zero_()
            else:
                a = _diff_args(q, k, v, lam, None, maps, lse, dout, dq, dk, dv, dlam, ql, kl, *ctx.how)
                n = lib.xva_diff_attention_workspace_bytes(C.byref(a), 1)
                ws = _workspace(n, q.device)
                _run(lib.xva_diff_attention_bwd(C.byref(a), _p(ws), n, _lib.raw_stream(q.device)), "xva_diff_attention_bwd")
        return dq, dk, dv, dlam, None, None, None, None


def differential_attention(q, k, v, lam, scale=None, causal=False, q_lens=None, k_lens=None):
    """(softmax(scale q_1 k_1^T) - lam softmax(scale q_2 k_2^T)) v, head by head; bf16 or fp16.

    q (B, Tq, H, 2, d): two queries a head; k (B, Tk, Hk, 2, d); v (B, Tk, Hk, 2 d); d a multiple of 8, 64 at most; query head h reads key head
    h // (H / Hk).  lam (H,): any float type, differentiable.  scale: d^-1/2 unless given.  q_lens / k_lens (B,): live queries and keys; causal: query i sees
    keys j <= i + k_len - q_len (the last query sees all).  Returns (B, Tq, H, 2 d); a row that sees no key is zero.  With Tq = 1 and no gradient this is the
    step of a serving loop: k and v may be slices of a longer cache."""
    dev = _device(q, k, v, lam, q_lens, k_lens)
    _refuse(q.dim() != 5 or k.dim() != 5 or v.dim() != 4 or q.shape[3] != 2 or k.shape[3] != 2, "q %s (B, Tq, H, 2, d), k %s (B, Tk, Hk, 2, d), v %s (B, Tk, Hk, 2 d)",
            tuple(q.shape), tuple(k.shape), tuple(v.shape))
    B, Tq, H, _, d = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    _refuse(k.shape[0] != B or k.shape[4] != d or tuple(v.shape) != (B, Tk, Hk, 2 * d), "q %s, k %s, v %s do not belong together", tuple(q.shape), tuple(k.shape),
            tuple(v.shape))
    _refuse(Hk < 1 or H % Hk, "%d query heads on %d key heads", H, Hk)
    _refuse(d % 8 or d < 8 or d > 64, "head width %d: a multiple of 8 up to 64", d)
    _refuse(q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype, "q, k, v are %s, %s, %s: one of bf16, fp16", q.dtype, k.dtype,
            v.dtype)
    _refuse(tuple(lam.shape) != (H,) or not lam.is_floating_point(), "lam %s %s: (%d,), a float type", tuple(lam.shape), lam.dtype, H)
    scale = d ** -0.5 if scale is None else float(scale)
    _refuse(not scale > 0.0, "scale %g", scale)
    with _on(dev):
        ql, kl = _lens(q_lens, B, dev, "q_lens"), _lens(k_lens, B, dev, "k_lens")
        q, k, v, lam = _wide(q), _wide(k), _wide(v), lam.float().contiguous()
        if _needs_grad(q, k, v, lam):
            return _DiffAttention.apply(q, k, v, lam, ql, kl, bool(causal), scale)
        return _diff_forward(q, k, v, lam, ql, kl, causal, scale, False)[0]


# ------------------------------------------------------------------------------------------------------------- gated recurrence ----
def _recurrence_launch(x, gate, h0, lens, reverse, unit, train):
    B, T, Cn = x.shape
    h = torch.empty((B, T, Cn), device=x.device, dtype=x.dtype)
    last = torch.empty((B, Cn), device=x.device, dtype=torch.float32)
    states = torch.empty(lib.xva_recurrence_state_floats(B, T, Cn), device=x.device, dtype=torch.float32) if train else None
    n = lib.xva_recurrence_workspace_bytes(B, T, Cn)
    ws = _workspace(n, x.device)
    xs, gs, hs = x.stride(), gate.stride(), h.stride()
    a = _RecurrenceArgs(x.data_ptr(), gate.data_ptr(), h.data_ptr(), _p(h0), last.data_ptr(), _p(states), None, None, None, None, None, _p(lens),
                        xs[0], xs[1], gs[0], gs[1], hs[0], hs[1], 0, 0, 0, 0, 0, 0, _DTYPES[x.dtype], B, T, Cn, reverse, unit)
    _run(lib.xva_recurrence_fwd(C.byref(a), _p(ws), n, _lib.raw_stream(x.device)), "xva_recurrence_fwd")
    return h, last, states


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, lens, reverse, unit):
        h, last, states = _recurrence_launch(x, gate, h0, lens, reverse, unit, True)
        ctx.save_for_backward(x, gate, states, lens)
        ctx.how = (reverse, unit, h0 is not None)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast):
        x, gate, states, lens = ctx.saved_tensors
        reverse, unit, with_h0 = ctx.how
        B, T, Cn = x.shape
        with _on(x.device):
            dh = torch.zeros((1, 1, Cn), device=x.device, dtype=x.dtype).expand(B, T, Cn) if dh is None else _rows(dh.to(x.dtype))
            dlast = dlast.float().contiguous() if dlast is not None else None
            dx, dg = (torch.empty((B, T, Cn), device=x.device, dtype=x.dtype) for _ in range(2))
            dh0 = torch.empty((B, Cn), device=x.device, dtype=torch.float32) if with_h0 else None
            n = lib.xva_recurrence_workspace_bytes(B, T, Cn)
            ws = _workspace(n, x.device)
            xs, gs, ds, os = x.stride(), gate.stride(), dh.stride(), dx.stride()
            a = _RecurrenceArgs(x.data_ptr(), gate.data_ptr(), None, None, None, states.data_ptr(), dh.data_ptr(), _p(dlast), dx.data_ptr(), dg.data_ptr(), _p(dh0),
                                _p(lens), xs[0], xs[1], gs[0], gs[1], 0, 0, ds[0], ds[1], os[0], os[1], os[0], os[1], _DTYPES[x.dtype], B, T, Cn, reverse, unit)
            _run(lib.xva_recurrence_bwd(C.byref(a), _p(ws), n, _lib.raw_stream(x.device)), "xva_recurrence_bwd")
        return dx, dg, dh0, None, None, None


def gated_recurrence(x, gate, h0=None, lens=None, reverse=False, gain="convex"):
    """h_t = f_t h_{t-1} + (1 - f_t) x_t with f = sigmoid(gate), each channel by itself; gain "unit": + x_t.

    x, gate (B, T, C) of one type; h0 (B, C): the state before the first step (None: zeros); reverse: from an item's last live row to its first.  Returns
    (h (B, T, C), last (B, C) fp32): the states, and the one behind the last step, which is the next call's h0.  States are fp32 throughout; h is rounded once."""
    dev = _device(x, gate, h0, lens)
    _refuse(x.dim() != 3 or gate.shape != x.shape, "x %s, gate %s: (B, T, C)", tuple(x.shape), tuple(gate.shape))
    _refuse(x.dtype not in _DTYPES or gate.dtype != x.dtype, "x is %s, gate %s", x.dtype, gate.dtype)
    _refuse(gain not in ("convex", "unit"), "gain %r: convex or unit", gain)
    B, T, Cn = x.shape
    _refuse(Cn < 1, "x %s: no channels", tuple(x.shape))
    _refuse(h0 is not None and (tuple(h0.shape) != (B, Cn) or not h0.is_floating_point()), "h0 %s: (%d, %d), a float type",
            tuple(h0.shape) if h0 is not None else None, B, Cn)
    with _on(dev):
        lens = _lens(lens, B, dev)
        x, gate = _rows(x), _rows(gate)
        h0 = h0.float().contiguous() if h0 is not None else None
        if _needs_grad(x, gate, h0):
            return _Recurrence.apply(x, gate, h0, lens, int(bool(reverse)), int(gain == "unit"))
        return _recurrence_launch(x, gate, h0, lens, int(bool(reverse)), int(gain == "unit"), False)[:2]


# ------------------------------------------------------------------------------------------------------------------ group norm ----
def _norm_args(x, dy, out, weight, bias, mean, rstd, dw, db, lens, groups, act, eps, slope):
    B, T, Cn = x.shape
    xs, os, gs = x.stride(), out.stride(), dy.stride() if dy is not None else (0, 0)
    return _GroupNormArgs(x.data_ptr(), _p(dy), out.data_ptr(), xs[0], xs[1], gs[0], gs[1], os[0], os[1], _p(weight), _p(bias), mean.data_ptr(), rstd.data_ptr(),
                          _p(dw), _p(db), _p(lens), _DTYPES[x.dtype], B, T, Cn, groups, act, eps, slope)


def _norm_forward(x, weight, bias, lens, groups, act, eps, slope):
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    stats = torch.empty((2, x.shape[0], groups), device=x.device, dtype=torch.float32)
    a = _norm_args(x, None, y, weight, bias, stats[0], stats[1], None, None, lens, groups, act, eps, slope)
    n = lib.xva_group_norm_workspace_bytes(C.byref(a), 0)
    ws = _workspace(n, x.device)
    _run(lib.xva_group_norm_act_fwd(C.byref(a), _p(ws), n, _lib.raw_stream(x.device)), "xva_group_norm_act_fwd")
    return y, stats


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, lens, groups, act, eps, slope):
        y, stats = _norm_forward(x, weight, bias, lens, groups, act, eps, slope)
        ctx.save_for_backward(x, weight, bias, lens, stats)
        ctx.how = (groups, act, eps, slope)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, lens, stats = ctx.saved_tensors
        with _on(x.device):
            dy = _rows(dy.to(x.dtype))
            dx = torch.empty(x.shape, device=x.device, dtype=x.dtype)
            dw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[1] else None
            db = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[2] else None
            a = _norm_args(x, dy, dx, weight, bias, stats[0], stats[1], dw, db, lens, *ctx.how)
            n = lib.xva_group_norm_workspace_bytes(C.byref(a), 1)
            ws = _workspace(n, x.device)
            _run(lib.xva_group_norm_act_bwd(C.byref(a), _p(ws), n, _lib.raw_stream(x.device)), "xva_group_norm_act_bwd")
        return dx, dw, db, None, None, None, None, None


def group_norm_act(x, groups, weight=None, bias=None, lens=None, eps=1e-5, act="none", slope=0.01):
    """act(weight * xh + bias), xh = x normalised over an item's live rows and each of `groups` equal groups of channels; x (B, T, C), or (B, C): one row each,
    so that attention heads as groups are normalised by themselves.  weight, bias (C,): any float type (None: 1, 0).  act: none, relu, lrelu (`slope`), tanh,
    silu, gelu (erf)."""
    flat = x.dim() == 2
    _refuse(x.dim() not in (2, 3) or (flat and lens is not None), "x %s: (B, T, C), or (B, C) without lens", tuple(x.shape))
    dev = _device(x, weight, bias, lens)
    _refuse(x.dtype not in _DTYPES, "x is %s", x.dtype)
    _refuse(act not in _ACTS, "act %r: one of %s", act, ", ".join(_ACTS))
    Cn = x.shape[-1]
    _refuse(groups < 1 or Cn < 1 or Cn % groups, "%d channels in %d groups", Cn, groups)
    _refuse(not eps >= 0.0, "eps %g", eps)
    for name, t in (("weight", weight), ("bias", bias)):
        _refuse(t is not None and (tuple(t.shape) != (Cn,) or not t.is_floating_point()), "%s %s: (%d,), a float type", name, tuple(t.shape) if t is not None else None, Cn)
    with _on(dev):
        x = _rows(x.unsqueeze(1) if flat else x)
        lens = _lens(lens, x.shape[0], dev)
        weight = weight.float().contiguous() if weight is not None else None
        bias = bias.float().contiguous() if bias is not None else None
        if _needs_grad(x, weight, bias):
            y = _GroupNormAct.apply(x, weight, bias, lens, groups, _ACTS[act], float(eps), float(slope))
        else:
            y = _norm_forward(x, weight, bias, lens, groups, _ACTS[act], float(eps), float(slope))[0]
    return y.squeeze(1) if flat else y
