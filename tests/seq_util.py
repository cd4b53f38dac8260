"""Shared by the tests of the sequence operators (xva_trainer_amd.seq_ops): types, roundings, comparisons."""
import ctypes as C

import torch

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# (a rounding is off by half a step at most)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# fp16 below 2^-14 is spaced 2^-24 apart: half a step of it, where a value may be as small
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def close(got, ref, bound, what=""):
    """|got - ref| <= bound, element by element; `ref` and `bound` in 64 bits on the CPU."""
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), "%s: not finite" % what
    over = (got - ref).abs() - bound
    assert over.max().item() <= 0.0 if over.numel() else True, "%s: off by %.3g where %.3g is allowed" % (
        what, (got - ref).abs().flatten()[over.argmax()].item(), (bound + torch.zeros_like(ref)).flatten()[over.argmax()].item())


def rounded(ref, dtype, fp32_error):
    """Bound of a value that is computed in fp32 with an absolute error of `fp32_error`, then rounded once to `dtype`."""
    return HALF[dtype] * (ref.abs() + fp32_error) + TINY[dtype] + fp32_error


def lengths(B, T, kind):
    if kind is None:
        return None
    if kind == "empty":                       # the first item has nothing, the last one row
        return torch.tensor([0] + [max(1, T - 3 * i) for i in range(1, B - 1)] + [min(1, T)], dtype=torch.int32)[:B]
    return torch.tensor([max(0, T - (i * 37) % (T // 2 + 1)) for i in range(B)], dtype=torch.int32)


# ---- the C structs of include/xva_hip.h, for calls of the C ABI itself
i32, i64, f32, vp = C.c_int32, C.c_int64, C.c_float, C.c_void_p


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


class RotaryArgs(C.Structure):
    _fields_ = _fields(("q k q_out k_out", vp), ("q_stride[3] k_stride[3] q_out_stride[3] k_out_stride[3]", i64), ("turns positions", vp), ("pos_stride[2]", i64),
                       ("positions64 dtype B T H Hk D rd interleaved inverse", i32), ("gain", f32))


class GroupNormArgs(C.Structure):
    _fields_ = _fields(("x dy out", vp), ("x_stride[2] dy_stride[2] out_stride[2]", i64), ("weight bias mean rstd dweight dbias lens", vp),
                       ("dtype B T C G act", i32), ("eps slope", f32))


class RecurrenceArgs(C.Structure):
    _fields_ = _fields(("x gate h h0 last states dh dlast dx dgate dh0 lens", vp),
                       ("x_stride[2] gate_stride[2] h_stride[2] dh_stride[2] dx_stride[2] dgate_stride[2]", i64), ("dtype B T C reverse unit_gain", i32))


class DiffAttentionArgs(C.Structure):
    _fields_ = _fields(("q k v lam out maps lse dout dq dk dv dlam q_lens k_lens", vp), ("q_stride[4] k_stride[4] v_stride[3] out_stride[3] dout_stride[3]", i64),
                       ("dtype B Tq Tk H Hk d causal lam_dtype", i32), ("scale", f32))


def entry(name, restype=i32):
    """An entry point of the library, with argument types that take the structs above by reference."""
    from xva_trainer_amd import _lib
    f = getattr(_lib.lib, name)
    f.restype = restype
    f.argtypes = [i32, i32, i32] if name.startswith("xva_recurrence_") and restype == i64 else [vp, vp] if name == "xva_rotary" else [vp, i32] if restype == i64 else [vp, vp, i64, vp]
    return f
