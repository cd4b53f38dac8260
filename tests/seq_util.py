"""Shared by the tests of the sequence operators (xva_trainer_amd.seq_ops): types, roundings, comparisons."""
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
