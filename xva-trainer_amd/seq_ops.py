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
leaves lives: torch would tie the capture to the eager graph's stream).  There are no second derivatives (they raise), no forward mode and no torch.jit.trace
(both refused).  There is no CPU fallback."""
import ctypes as C
import decimal
import math
from decimal import Decimal

import torch

from . import _lib

try:
    from . import _seq_torch
except ImportError as e:
    raise _lib.XvaError("_seq_torch is not built (%s). Run `python -c 'import __graft_entry__ as g; g.build()'`" % e)

XvaError = _lib.XvaError
_ENTRIES = ("xva_last_error", "xva_rotary", "xva_group_norm_workspace_bytes", "xva_group_norm_act_fwd", "xva_group_norm_act_bwd", "xva_recurrence_workspace_bytes",
            "xva_recurrence_state_floats", "xva_recurrence_fwd", "xva_recurrence_bwd", "xva_diff_attention_workspace_bytes", "xva_diff_attention_fwd",
            "xva_diff_attention_bwd")
_seq_torch.bind({n: C.cast(getattr(_lib.lib, n), C.c_void_p).value for n in _ENTRIES}, XvaError)

_PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628621")


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
            raise XvaError("rotary_dim %d: an even number of elements" % (rotary_dim))
        if scaling not in ("none", "linear", "ntk", "yarn"):
            raise XvaError("scaling %r: none, linear, ntk or yarn" % (scaling))
        if not (1.0 < base < math.inf and 1.0 <= factor < math.inf and original_length >= 1 and beta_fast > beta_slow > 0.0):
            raise XvaError("base %g, factor %g, original_length %d, beta_fast %g, beta_slow %g" % (base, factor, original_length, beta_fast, beta_slow))
        n = rotary_dim // 2
        self.rotary_dim, self.interleaved, self.gain = rotary_dim, bool(interleaved), 1.0
        # In 60 digits: a double's 53 bits of a frequency leave 2^-56 of a turn for every position, which is 1e-4 radians at 2^40
        with decimal.localcontext(decimal.Context(prec=60, Emin=-10 ** 6, Emax=10 ** 6)):
            by, longer = Decimal(float(base)), Decimal(float(factor))
            if scaling == "ntk" and rotary_dim > 2:
                by = by * (longer.ln() * rotary_dim / (rotary_dim - 2)).exp()
            ratio, freq = (by.ln() * -2 / rotary_dim).exp(), [Decimal(1)]
            while len(freq) < n:
                freq.append(freq[-1] * ratio)
            if scaling == "linear":
                freq = [f / longer for f in freq]
            elif scaling == "yarn":
                def pair_of(turns):
                    return rotary_dim * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
                low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
                for i in range(n):
                    ramp = min(max(Decimal(i - low) / Decimal(max(high - low, 1e-3)), Decimal(0)), Decimal(1))
                    freq[i] = freq[i] * (1 - ramp) + freq[i] / longer * ramp
                self.gain = 0.1 * math.log(factor) + 1.0
            # fractions of a turn per position as 64-bit fixed point, to half a unit (two's complement: the upper half reads as negative)
            fixed = [int((f / (2 * _PI) * 2 ** 64).to_integral_value()) % 2 ** 64 for f in freq]
        self.frequencies = [float(f) for f in freq]
        if gain is not None:
            self.gain = float(gain)
        self.turns = torch.tensor([v - 2 ** 64 if v >= 2 ** 63 else v for v in fixed], dtype=torch.int64).to(device)

    def to(self, device):
        self.turns = self.turns.to(device)
        return self


def rotary(plan, q, k=None, positions=None, inplace=False):
    """Turns q (B, T, H, D) and, if given, k (B, T, Hk, D) by their positions: (B, T) or (T,), a dimension of 1 standing for all, int32 or int64;
    None: 0 .. T - 1.  Returns q', or (q', k').  inplace: writes over q and k (no gradient; heads that lie on each other, or may, are refused)."""
    out = _seq_torch.rotary(plan.turns, plan.rotary_dim, plan.interleaved, plan.gain, q, k, positions, inplace)
    return out[0] if k is None else (out[0], out[1])


def differential_attention(q, k, v, lam, scale=None, causal=False, q_lens=None, k_lens=None):
    """(softmax(scale q_1 k_1^T) - lam softmax(scale q_2 k_2^T)) v, head by head; bf16 or fp16.

    q (B, Tq, H, 2, d): two queries a head; k (B, Tk, Hk, 2, d); v (B, Tk, Hk, 2 d); d a multiple of 8, 64 at most; query head h reads key head
    h // (H / Hk).  lam (H,): any float type, differentiable.  scale: d^-1/2 unless given.  q_lens / k_lens (B,): live queries and keys; causal: query i sees
    keys j <= i + k_len - q_len (the last query sees all).  Returns (B, Tq, H, 2 d); a row that sees no key is zero.  Rows behind k_len and q_len are not read; a
    value that is not finite in a live row may reach every query of its item, also one that `causal` hides it from (its weight is zero, its product is not a
    number).  With Tq = 1 and no gradient this is the step of a serving loop: k and v may be slices of a longer cache."""
    return _seq_torch.differential_attention(q, k, v, lam, scale, causal, q_lens, k_lens)


def gated_recurrence(x, gate, h0=None, lens=None, reverse=False, gain="convex"):
    """h_t = f_t h_{t-1} + (1 - f_t) x_t with f = sigmoid(gate), each channel by itself; gain "unit": + x_t.

    x, gate (B, T, C) of one type; h0 (B, C): the state before the first step (None: zeros); reverse: from an item's last live row to its first.  Returns
    (h (B, T, C), last (B, C) fp32): the states, and the one behind the last step, which is the next call's h0.  States are fp32 throughout; h is rounded once."""
    return _seq_torch.gated_recurrence(x, gate, h0, lens, reverse, gain)


def group_norm_act(x, groups, weight=None, bias=None, lens=None, eps=1e-5, act="none", slope=0.01):
    """act(weight * xh + bias), xh = x normalised over an item's live rows and each of `groups` equal groups of channels; x (B, T, C), or (B, C): one row each,
    so that attention heads as groups are normalised by themselves.  weight, bias (C,): any float type (None: 1, 0).  act: none, relu, lrelu (`slope`), tanh,
    silu, gelu (erf)."""
    return _seq_torch.group_norm_act(x, groups, weight, bias, lens, eps, act, slope)
