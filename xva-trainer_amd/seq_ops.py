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
import functools
import math
import struct

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


def _packer(t):
    """The struct's bytes from its fields in order: one C call, where filling a ctypes structure of 40 fields takes longer than a small kernel."""
    return struct.Struct("@" + "".join({vp: "P", i64: "q", i32: "i", f32: "f"}[f[1]] for f in t._fields_) + "0q").pack


_rotary_args, _norm_args, _recurrence_args, _diff_args = (_packer(t) for t in (_RotaryArgs, _GroupNormArgs, _RecurrenceArgs, _DiffAttentionArgs))

lib.xva_rotary.restype, lib.xva_rotary.argtypes = i32, [vp, vp]
for _n in ("group_norm_act", "recurrence", "diff_attention"):
    for _d in ("fwd", "bwd"):
        _f = getattr(lib, "xva_%s_%s" % (_n, _d))
        _f.restype, _f.argtypes = i32, [vp, vp, i64, vp]
lib.xva_group_norm_workspace_bytes.restype, lib.xva_group_norm_workspace_bytes.argtypes = i64, [vp, i32]
lib.xva_diff_attention_workspace_bytes.restype, lib.xva_diff_attention_workspace_bytes.argtypes = i64, [vp, i32]
lib.xva_recurrence_workspace_bytes.restype, lib.xva_recurrence_workspace_bytes.argtypes = i64, [i32, i32, i32]
lib.xva_recurrence_state_floats.restype, lib.xva_recurrence_state_floats.argtypes = i64, [i32, i32, i32]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {"none": 0, "relu": 1, "lrelu": 2, "tanh": 3, "silu": 4, "gelu": 5}
_HOW_MANY = 4096        # sizes of workspaces that are remembered, by shape


def _fail(msg, *args):
    raise XvaError(msg % args)


def _device(first, *others):
    """All on one GPU."""
    dev = first.device
    if dev.type != "cuda":
        _fail("libxvahip ops need device tensors; got a %s tensor (no CPU fallback exists)", dev)
    for t in others:
        if t is not None and t.device != dev:
            _fail("tensors on %s and %s", dev, t.device)
    return dev


def _here(fn):
    """Calls `fn` with its first argument's device as the current one (launches and allocations go there)."""
    @functools.wraps(fn)
    def call(t, *args):
        if t.device.index == torch.cuda.current_device():
            return fn(t, *args)
        with torch.cuda.device(t.device):
            return fn(t, *args)
    return call


def _p(t):
    return t.data_ptr() if t is not None else 0


def _lens(lens, B, device, what="lens"):
    if lens is None:
        return None
    if lens.dim() != 1 or lens.shape[0] != B:
        _fail("%s: %s, expected (%d,)", what, tuple(lens.shape), B)
    if lens.device != device:
        _fail("%s on %s, the tensors on %s", what, lens.device, device)
    if lens.dtype != torch.int32:
        if lens.dtype != torch.int64:
            _fail("%s: int32 or int64, got %s", what, lens.dtype)
        lens = lens.to(torch.int32)
    return lens.contiguous()


def _float(t):
    """fp32 and contiguous."""
    return t.float().contiguous() if t is not None and (t.dtype != torch.float32 or not t.is_contiguous()) else t


def _rows(t):
    """`t` with a contiguous last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _needs_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _workspace(n, device):
    return torch.empty(n, device=device, dtype=torch.uint8) if n else None


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
        if rotary_dim < 2 or rotary_dim % 2:
            _fail("rotary_dim %d: an even number of elements", rotary_dim)
        if scaling not in ("none", "linear", "ntk", "yarn"):
            _fail("scaling %r: none, linear, ntk or yarn", scaling)
        if not (1.0 < base < math.inf and 1.0 <= factor < math.inf and original_length >= 1 and beta_fast > beta_slow > 0.0):
            _fail("base %g, factor %g, original_length %d, beta_fast %g, beta_slow %g", base, factor, original_length, beta_fast, beta_slow)
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


@_here
def _rotary_launch(q, k, plan, pos, inverse, inplace):
    B, T, H, D = q.shape
    dtype, dev = q.dtype, q.device
    q = _rows(q)
    qo = q if inplace else torch.empty((B, T, H, D), device=dev, dtype=dtype)
    if k is not None:
        k = _rows(k)
        Hk = k.shape[2]
        ko = k if inplace else torch.empty((B, T, Hk, D), device=dev, dtype=dtype)
        ks, kos, kp, kop = k.stride(), ko.stride(), k.data_ptr(), ko.data_ptr()
    else:
        ko, ks, kos, kp, kop, Hk = None, (0, 0, 0), (0, 0, 0), 0, 0, 0
    qs, qos = q.stride(), qo.stride()
    pb = pt = pp = wide = 0
    if pos is not None:
        pp, wide = pos.data_ptr(), int(pos.dtype == torch.int64)
        if pos.dim() == 2 and pos.shape[0] > 1:
            pb = pos.stride(0)
        if pos.shape[-1] > 1:
            pt = pos.stride(-1)
    a = _rotary_args(q.data_ptr(), kp, qo.data_ptr(), kop, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], qos[0], qos[1], qos[2], kos[0], kos[1], kos[2],
                     plan.turns.data_ptr(), pp, pb, pt, wide, _DTYPES[dtype], B, T, H, Hk, D, plan.rotary_dim, plan.interleaved, inverse, plan.gain)
    rc = lib.xva_rotary(a, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "xva_rotary")
    return qo, ko


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, plan):
        ctx.plan, ctx.pos = plan, pos
        qo, ko = _rotary_launch(q, k, plan, pos, False, False)
        return (qo, ko) if k is not None else qo

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        gq, gk = _rotary_launch(dq, dk, ctx.plan, ctx.pos, True, False)
        return gq, gk, None, None


def rotary(plan, q, k=None, positions=None, inplace=False):
    """Turns q (B, T, H, D) and, if given, k (B, T, Hk, D) by their positions: (B, T) or (T,), a dimension of 1 standing for all, int32 or int64;
    None: 0 .. T - 1.  Returns q', or (q', k').  inplace: writes over q and k (no gradient)."""
    _device(q, k, positions, plan.turns)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != shape[:2] or k.shape[3] != shape[3])):
        _fail("q %s, k %s: (B, T, heads, D)", tuple(shape), tuple(k.shape) if k is not None else None)
    if dtype not in _DTYPES or (k is not None and k.dtype != dtype):
        _fail("q is %s, k %s", dtype, k.dtype if k is not None else None)
    if plan.rotary_dim > shape[3]:
        _fail("rotary_dim %d of heads of %d", plan.rotary_dim, shape[3])
    if positions is not None:
        ps = positions.shape
        if positions.dtype != torch.int64 and positions.dtype != torch.int32:
            _fail("positions: int32 or int64, got %s", positions.dtype)
        if len(ps) not in (1, 2) or ps[-1] not in (1, shape[1]) or (len(ps) == 2 and ps[0] not in (1, shape[0])):
            _fail("positions %s of (%d, %d) rows", tuple(ps), shape[0], shape[1])
    if _needs_grad(q, k):
        if inplace:
            _fail("inplace: no gradient")
        return _Rotary.apply(q, k, positions, plan)
    if inplace and (q.stride(-1) != 1 or (k is not None and k.stride(-1) != 1)):
        _fail("inplace: a contiguous last dimension")
    qo, ko = _rotary_launch(q, k, plan, positions, False, inplace)
    return (qo, ko) if k is not None else qo


# -------------------------------------------------------------------------------------------------------- differential attention ----
def _wide(t):
    """`t` as the attention kernels read it: 16-byte rows, 64 of them and their maps within 32-bit offsets."""
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0 and not any(s % 8 for s in st[:-1]) and st[1] < 1 << 24 and st[3] < 1 << 24:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


@functools.lru_cache(_HOW_MANY)
def _diff_sizes(B, Tq, Tk, H, Hk, d, train, bwd):
    a = _DiffAttentionArgs(B=B, Tq=Tq, Tk=Tk, H=H, Hk=Hk, d=d, maps=1 if train else None)
    return lib.xva_diff_attention_workspace_bytes(C.byref(a), bwd)


@_here
def _diff_forward(q, k, v, lam, ql, kl, causal, scale, train):
    B, Tq, H, _, d = q.shape
    Tk, Hk, dev, dtype = k.shape[1], k.shape[2], q.device, q.dtype
    out = torch.empty((B, Tq, H, 2 * d), device=dev, dtype=dtype)
    maps = torch.empty((2, B, Tq, H, 2 * d), device=dev, dtype=dtype) if train else None
    lse = torch.empty((2, B, H, Tq), device=dev, dtype=torch.float32) if train else None
    n = _diff_sizes(B, Tq, Tk, H, Hk, d, train, 0)
    ws = _workspace(n, dev)
    a = _diff_args(q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), out.data_ptr(), _p(maps), _p(lse), 0, 0, 0, 0, 0, _p(ql), _p(kl),
                   *q.stride()[:4], *k.stride()[:4], *v.stride()[:3], *out.stride()[:3], 0, 0, 0, _DTYPES[dtype], B, Tq, Tk, H, Hk, d, causal, scale)
    rc = lib.xva_diff_attention_fwd(a, _p(ws), n, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "xva_diff_attention_fwd")
    return out, maps, lse


@_here
def _diff_backward(q, k, v, lam, maps, lse, ql, kl, causal, scale, dout):
    B, Tq, H, _, d = q.shape
    Tk, Hk, dev, dtype = k.shape[1], k.shape[2], q.device, q.dtype
    dout = _wide(dout if dout.dtype == dtype else dout.to(dtype))
    dq = torch.empty((B, Tq, H, 2, d), device=dev, dtype=dtype)
    dk = torch.empty((B, Tk, Hk, 2, d), device=dev, dtype=dtype)
    dv = torch.empty((B, Tk, Hk, 2 * d), device=dev, dtype=dtype)
    dlam = torch.empty((H,), device=dev, dtype=torch.float32)
    if B == 0 or Tq == 0:
        for t in (dk, dv, dlam):
            t.zero_()
        return dq, dk, dv, dlam
    n = _diff_sizes(B, Tq, Tk, H, Hk, d, True, 1)
    ws = _workspace(n, dev)
    a = _diff_args(q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), 0, maps.data_ptr(), lse.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                   dv.data_ptr(), dlam.data_ptr(), _p(ql), _p(kl), *q.stride()[:4], *k.stride()[:4], *v.stride()[:3], 0, 0, 0, *dout.stride()[:3], _DTYPES[dtype],
                   B, Tq, Tk, H, Hk, d, causal, scale)
    rc = lib.xva_diff_attention_bwd(a, _p(ws), n, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "xva_diff_attention_bwd")
    return dq, dk, dv, dlam


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
        return _diff_backward(*ctx.saved_tensors, *ctx.how, dout) + (None, None, None, None)


def differential_attention(q, k, v, lam, scale=None, causal=False, q_lens=None, k_lens=None):
    """(softmax(scale q_1 k_1^T) - lam softmax(scale q_2 k_2^T)) v, head by head; bf16 or fp16.

    q (B, Tq, H, 2, d): two queries a head; k (B, Tk, Hk, 2, d); v (B, Tk, Hk, 2 d); d a multiple of 8, 64 at most; query head h reads key head
    h // (H / Hk).  lam (H,): any float type, differentiable.  scale: d^-1/2 unless given.  q_lens / k_lens (B,): live queries and keys; causal: query i sees
    keys j <= i + k_len - q_len (the last query sees all).  Returns (B, Tq, H, 2 d); a row that sees no key is zero.  With Tq = 1 and no gradient this is the
    step of a serving loop: k and v may be slices of a longer cache."""
    dev = _device(q, k, v, lam, q_lens, k_lens)
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != 5 or len(ks) != 5 or len(vs) != 4 or qs[3] != 2 or ks[3] != 2:
        _fail("q %s (B, Tq, H, 2, d), k %s (B, Tk, Hk, 2, d), v %s (B, Tk, Hk, 2 d)", tuple(qs), tuple(ks), tuple(vs))
    B, _, H, _, d = qs
    Hk = ks[2]
    if ks[0] != B or ks[4] != d or vs != (B, ks[1], Hk, 2 * d):
        _fail("q %s, k %s, v %s do not belong together", tuple(qs), tuple(ks), tuple(vs))
    if Hk < 1 or H < 1 or H % Hk:
        _fail("%d query heads on %d key heads", H, Hk)
    if d % 8 or d < 8 or d > 64:
        _fail("head width %d: a multiple of 8 up to 64", d)
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        _fail("q, k, v are %s, %s, %s: one of bf16, fp16", q.dtype, k.dtype, v.dtype)
    if lam.shape != (H,) or not lam.is_floating_point():
        _fail("lam %s %s: (%d,), a float type", tuple(lam.shape), lam.dtype, H)
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        _fail("scale %g", scale)
    ql, kl = _lens(q_lens, B, dev, "q_lens"), _lens(k_lens, B, dev, "k_lens")
    q, k, v, lam = _wide(q), _wide(k), _wide(v), _float(lam)
    if _needs_grad(q, k, v, lam):
        return _DiffAttention.apply(q, k, v, lam, ql, kl, bool(causal), scale)
    return _diff_forward(q, k, v, lam, ql, kl, bool(causal), scale, False)[0]


# ------------------------------------------------------------------------------------------------------------- gated recurrence ----
@functools.lru_cache(_HOW_MANY)
def _recurrence_sizes(B, T, Cn):
    return lib.xva_recurrence_workspace_bytes(B, T, Cn), lib.xva_recurrence_state_floats(B, T, Cn)


@_here
def _recurrence_forward(x, gate, h0, lens, reverse, unit, train):
    B, T, Cn = x.shape
    dev, dtype = x.device, x.dtype
    n, states = _recurrence_sizes(B, T, Cn)
    h = torch.empty((B, T, Cn), device=dev, dtype=dtype)
    last = torch.empty((B, Cn), device=dev, dtype=torch.float32)
    states = torch.empty(states, device=dev, dtype=torch.float32) if train else None
    ws = _workspace(n, dev)
    a = _recurrence_args(x.data_ptr(), gate.data_ptr(), h.data_ptr(), _p(h0), last.data_ptr(), _p(states), 0, 0, 0, 0, 0, _p(lens),
                         *x.stride()[:2], *gate.stride()[:2], T * Cn, Cn, 0, 0, 0, 0, 0, 0, _DTYPES[dtype], B, T, Cn, reverse, unit)
    rc = lib.xva_recurrence_fwd(a, _p(ws), n, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "xva_recurrence_fwd")
    return h, last, states


@_here
def _recurrence_backward(x, gate, states, lens, reverse, unit, with_h0, dh, dlast):
    B, T, Cn = x.shape
    dev, dtype = x.device, x.dtype
    if dh is None:
        dh = torch.zeros((1, 1, Cn), device=dev, dtype=dtype).expand(B, T, Cn)
    else:
        dh = _rows(dh if dh.dtype == dtype else dh.to(dtype))
    dlast = _float(dlast)
    dx = torch.empty((B, T, Cn), device=dev, dtype=dtype)
    dg = torch.empty((B, T, Cn), device=dev, dtype=dtype)
    dh0 = torch.empty((B, Cn), device=dev, dtype=torch.float32) if with_h0 else None
    n = _recurrence_sizes(B, T, Cn)[0]
    ws = _workspace(n, dev)
    a = _recurrence_args(x.data_ptr(), gate.data_ptr(), 0, 0, 0, states.data_ptr(), dh.data_ptr(), _p(dlast), dx.data_ptr(), dg.data_ptr(), _p(dh0), _p(lens),
                         *x.stride()[:2], *gate.stride()[:2], 0, 0, *dh.stride()[:2], T * Cn, Cn, T * Cn, Cn, _DTYPES[dtype], B, T, Cn, reverse, unit)
    rc = lib.xva_recurrence_bwd(a, _p(ws), n, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "xva_recurrence_bwd")
    return dx, dg, dh0


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, lens, reverse, unit):
        h, last, states = _recurrence_forward(x, gate, h0, lens, reverse, unit, True)
        ctx.save_for_backward(x, gate, states, lens)
        ctx.how = (reverse, unit, h0 is not None)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast):
        return _recurrence_backward(*ctx.saved_tensors, *ctx.how, dh, dlast) + (None, None, None)


def gated_recurrence(x, gate, h0=None, lens=None, reverse=False, gain="convex"):
    """h_t = f_t h_{t-1} + (1 - f_t) x_t with f = sigmoid(gate), each channel by itself; gain "unit": + x_t.

    x, gate (B, T, C) of one type; h0 (B, C): the state before the first step (None: zeros); reverse: from an item's last live row to its first.  Returns
    (h (B, T, C), last (B, C) fp32): the states, and the one behind the last step, which is the next call's h0.  States are fp32 throughout; h is rounded once."""
    dev = _device(x, gate, h0, lens)
    shape = x.shape
    if len(shape) != 3 or gate.shape != shape:
        _fail("x %s, gate %s: (B, T, C)", tuple(shape), tuple(gate.shape))
    if x.dtype not in _DTYPES or gate.dtype != x.dtype:
        _fail("x is %s, gate %s", x.dtype, gate.dtype)
    if gain not in ("convex", "unit"):
        _fail("gain %r: convex or unit", gain)
    B, _, Cn = shape
    if Cn < 1:
        _fail("x %s: no channels", tuple(shape))
    if h0 is not None and (h0.shape != (B, Cn) or not h0.is_floating_point()):
        _fail("h0 %s: (%d, %d), a float type", tuple(h0.shape), B, Cn)
    lens = _lens(lens, B, dev)
    x, gate, h0 = _rows(x), _rows(gate), _float(h0)
    if _needs_grad(x, gate, h0):
        return _Recurrence.apply(x, gate, h0, lens, bool(reverse), gain == "unit")
    return _recurrence_forward(x, gate, h0, lens, bool(reverse), gain == "unit", False)[:2]


# ------------------------------------------------------------------------------------------------------------------ group norm ----
@functools.lru_cache(_HOW_MANY)
def _norm_size(dtype, B, T, Cn, groups, bwd):
    return lib.xva_group_norm_workspace_bytes(C.byref(_GroupNormArgs(dtype=dtype, B=B, T=T, C=Cn, G=groups)), bwd)


@_here
def _norm_forward(x, weight, bias, lens, groups, act, eps, slope):
    B, T, Cn = x.shape
    dev, dt = x.device, _DTYPES[x.dtype]
    y = torch.empty((B, T, Cn), device=dev, dtype=x.dtype)
    stats = torch.empty((2, B, groups), device=dev, dtype=torch.float32)
    mean = stats.data_ptr()
    n = _norm_size(dt, B, T, Cn, groups, 0)
    ws = _workspace(n, dev)
    a = _norm_args(x.data_ptr(), 0, y.data_ptr(), *x.stride()[:2], 0, 0, T * Cn, Cn, _p(weight), _p(bias), mean, mean + 4 * B * groups, 0, 0, _p(lens),
                   dt, B, T, Cn, groups, act, eps, slope)
    rc = lib.xva_group_norm_act_fwd(a, _p(ws), n, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "xva_group_norm_act_fwd")
    return y, stats


@_here
def _norm_backward(x, weight, bias, lens, stats, groups, act, eps, slope, dy, want_w, want_b):
    B, T, Cn = x.shape
    dev, dt = x.device, _DTYPES[x.dtype]
    dy = _rows(dy if dy.dtype == x.dtype else dy.to(x.dtype))
    dx = torch.empty((B, T, Cn), device=dev, dtype=x.dtype)
    dw = torch.empty((Cn,), device=dev, dtype=torch.float32) if want_w else None
    db = torch.empty((Cn,), device=dev, dtype=torch.float32) if want_b else None
    mean = stats.data_ptr()
    n = _norm_size(dt, B, T, Cn, groups, 1)
    ws = _workspace(n, dev)
    a = _norm_args(x.data_ptr(), dy.data_ptr(), dx.data_ptr(), *x.stride()[:2], *dy.stride()[:2], T * Cn, Cn, _p(weight), _p(bias), mean, mean + 4 * B * groups,
                   _p(dw), _p(db), _p(lens), dt, B, T, Cn, groups, act, eps, slope)
    rc = lib.xva_group_norm_act_bwd(a, _p(ws), n, _lib.raw_stream(dev))
    if rc:
        _lib.check(rc, "xva_group_norm_act_bwd")
    return dx, dw, db


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
        need = ctx.needs_input_grad
        return _norm_backward(*ctx.saved_tensors, *ctx.how, dy, need[1], need[2]) + (None, None, None, None, None)


def group_norm_act(x, groups, weight=None, bias=None, lens=None, eps=1e-5, act="none", slope=0.01):
    """act(weight * xh + bias), xh = x normalised over an item's live rows and each of `groups` equal groups of channels; x (B, T, C), or (B, C): one row each,
    so that attention heads as groups are normalised by themselves.  weight, bias (C,): any float type (None: 1, 0).  act: none, relu, lrelu (`slope`), tanh,
    silu, gelu (erf)."""
    shape = x.shape
    flat = len(shape) == 2
    if len(shape) not in (2, 3) or (flat and lens is not None):
        _fail("x %s: (B, T, C), or (B, C) without lens", tuple(shape))
    dev = _device(x, weight, bias, lens)
    if x.dtype not in _DTYPES:
        _fail("x is %s", x.dtype)
    if act not in _ACTS:
        _fail("act %r: one of %s", act, ", ".join(_ACTS))
    Cn = shape[-1]
    if groups < 1 or Cn < 1 or Cn % groups:
        _fail("%d channels in %d groups", Cn, groups)
    if not 0.0 <= eps < math.inf:
        _fail("eps %g", eps)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (Cn,) or not t.is_floating_point()):
            _fail("%s %s: (%d,), a float type", name, tuple(t.shape), Cn)
    x = _rows(x.unsqueeze(1) if flat else x)
    lens, weight, bias = _lens(lens, shape[0], dev), _float(weight), _float(bias)
    if _needs_grad(x, weight, bias):
        y = _GroupNormAct.apply(x, weight, bias, lens, groups, _ACTS[act], eps, slope)
    else:
        y = _norm_forward(x, weight, bias, lens, groups, _ACTS[act], eps, slope)[0]
    return y.squeeze(1) if flat else y
