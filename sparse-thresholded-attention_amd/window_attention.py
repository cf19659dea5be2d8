"""Causal attention over packed sequences with a sliding window and first keys that stay visible (sinks), on the
gfx950 kernels of libsta_hip.so, for training and prompts.

    window_attention        differentiable
    window_attention_grad   its gradients on their own

A training step of a layer with a window, sequences of different lengths packed into one tensor:

    q, k = norm_rotary(q, k, q_weight, k_weight, positions, inv_freq)       # paged_cache.py
    out = window_attention(q, k, v, window=4096, sinks=4, starts=starts)    # (T, H, D)
    out.backward(dout)

The form for new tokens of cached sequences is paged_attention(..., window=, sinks=) of paged_cache.py.

Both launch on the current stream of the tensors' device, allocate their results and their workspace from torch's
allocator, and neither synchronise nor keep anything between calls, so a HIP graph can capture them (a captured
training step calls window_attention_grad itself).  Gradients have one order of sums: a call repeated gives the same
bits.  There is no fallback: a CPU tensor, an unsupported shape or a missing library raises.
"""
import inspect

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

import _sta_native as native


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(q, k, v, window, sinks, starts, k_starts, sm_scale):
        return native.window_attention(q, k, v, window, sinks, starts, k_starts, sm_scale, want_rest=True)

    @staticmethod
    def setup_context(ctx, inputs, output):
        q, k, v, *ctx.how, starts, k_starts, ctx.sm_scale = inputs
        out, lse, rest = output
        ctx.mark_non_differentiable(*(x for x in (lse, rest) if x is not None))
        ctx.save_for_backward(q, k, v, out, lse, rest, starts, k_starts)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, *_):
        *tensors, starts, k_starts = ctx.saved_tensors
        return (*native.window_attention_grad(dout, *tensors, *ctx.how, starts, k_starts, ctx.sm_scale),
                None, None, None, None, None)


# apply() asks for it in every call: formed anew it would take 20 us of them
_WindowAttention.forward.__signature__ = inspect.signature(_WindowAttention.forward)


def window_attention(q, k, v, window=None, sinks=0, starts=None, k_starts=None, sm_scale=None, want_lse=False,
                     want_rest=False):
    """Attention of q (T, H, D) over k, v (S, Hkv, D), H a multiple of Hkv, D 64 or 128, in one dtype of bf16, fp16
    and fp32; returns out like q, with want_lse also the log-sum-exp of the scaled scores (T, H) fp32, with want_rest
    also what rounding out to a 16-bit type left (None for fp32), both for window_attention_grad and without gradients.

    starts (B + 1,) int32 or int64, ascending: sequence b has the rows starts[b] .. starts[b + 1] - 1 of q, and of k
    and v the rows k_starts[b] .. k_starts[b + 1] - 1 (default: starts, with S = T).  Without starts all rows are one
    sequence.  The last row of a sequence stands at its last key: row i of nq is at position p = nk - nq + i and sees
    the keys j <= p with j > p - window or j < sinks.  window None: every j <= p.  A row that sees no key, or none
    with a score above -inf, gets zeros and -inf, and so do rows outside all sequences, whatever they hold.
    sm_scale: default D ** -0.5.  Scores, softmax and sums are fp32; 16-bit types round the probabilities (and
    the gradients of the scores) once to the type for the second product, the probabilities to twice its bits where
    rows see at most some 1000 keys.  The bits of out do not depend on whether a gradient is wanted.
    What a row does not see reaches neither its out nor its dq, infinities and NaN included, and a key that holds such
    reaches dk and dv of those keys alone that one of the rows which see it sees too; a row of q or of the
    gradient that holds such makes dk and dv of its sequence's keys so, whether it sees them or not.  Such values make a
    call many times slower: 32 rows at a time go over their keys one by one (8192 tokens of 32 heads, every row
    seeing a NaN: 30 ms in place of 0.7, the gradient 53 in place of 2.6; with a window of 1024 1.7 and 3.6 ms).

    Differentiable once, in q, k and v; forward-mode tangents are refused and transforms of torch.func raise.  T and S
    up to 2^28, token strides up to 2^29 bytes."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(x).tangent is not None for x in (q, k, v)):
        raise RuntimeError("window_attention has no forward-mode derivative")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse, rest = _WindowAttention.apply(q, k, v, window, sinks, starts, k_starts, sm_scale)
    else:
        out, lse, rest = native.window_attention(q, k, v, window, sinks, starts, k_starts, sm_scale, want_rest)
    results = (out,) + ((lse.t(),) if want_lse else ()) + ((rest,) if want_rest else ())
    return results if len(results) > 1 else out


def window_attention_grad(dout, q, k, v, out, lse, rest=None, window=None, sinks=0, starts=None, k_starts=None, sm_scale=None):
    """The gradients (dq, dk, dv) from dout (T, H, D) and what window_attention(..., want_lse=True, want_rest=True)
    returned for the same arguments, without an autograd graph.  Without rest, dq and dk of 16-bit types err by
    1.5 to 1.6 times what rounding them costs, with it by up to 1.48.  Inputs with forward-mode tangents are refused."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(x).tangent is not None
                                              for x in (dout, q, k, v, out)):
        raise RuntimeError("window_attention_grad keeps no graph and no forward-mode tangents")
    return native.window_attention_grad(dout, q, k, v, out, lse.t(), rest, window, sinks, starts, k_starts,
                                        sm_scale)
