"""A paged key-value cache and the operators around it, on the gfx950 kernels of libsta_hip.so.

The reference's decode keeps one contiguous cache of one sequence; these entry points serve a batch
of sequences whose keys lie in pages, and a cache held at a budget of keys:

    rotary            rotary positions with one or several axes (time, height, width), differentiable
    rotary_grad       the rotation's gradient on its own
    norm_rotary       each head's row divided by its root mean square, then rotated, in one pass; differentiable
    norm_rotary_grad  its gradients on their own
    cache_append      new keys and values into the pages
    paged_attention   a few new tokens of every sequence over its cached keys (dense: no threshold), all of
                      them or the latest of a window and the first few (sinks)
    prefix_attention  the same for sequences that begin with the same keys, which are read once for all
    cache_evict       drop the keys of least accumulated attention weight

A decoding step of a batch, held at `budget` keys a head:

    cache = PagedCache.empty(pages, 16, kv_heads, 128)
    q, k = rotary(q, k, seen, inv_freq)                                 # (B, heads, D)
    lens = cache_append(cache, k, v, table, lens, seen=seen)
    out = paged_attention(q, cache, table, lens, accumulate=True)
    lens = cache_evict(cache, table, lens, budget)

All of them launch on the current stream of the tensors' device, allocate their results and their
workspace from torch's allocator, and neither synchronise nor keep anything between calls, so a HIP
graph can capture them (a captured training step calls rotary_grad and norm_rotary_grad itself).  rotary
takes part in automatic differentiation, in both modes, and norm_rotary in reverse mode, once; the others keep
neither gradients nor tangents.  There is no fallback: a CPU tensor, an unsupported shape or a missing library raises.
"""
import inspect

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

import _sta_native as native
from _sta_native import PagedCache  # noqa: F401


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(q, k, positions, inv_freq, sections, pos_scale, rope_scale, inverse):
        return native.rotary(q, k, positions, inv_freq, sections, pos_scale, rope_scale, inverse)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, _, positions, inv_freq, *ctx.how, ctx.inverse = inputs
        ctx.save_for_backward(positions, inv_freq)
        ctx.save_for_forward(positions, inv_freq)

    # linear in q and k: the gradient is the rotation the other way, the tangent the rotation of theirs; both are
    # differentiable themselves
    @staticmethod
    def backward(ctx, dq, dk):
        return (*_Rotary.apply(dq, dk, *ctx.saved_tensors, *ctx.how, not ctx.inverse),
                None, None, None, None, None, None)

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        return _Rotary.apply(tq, tk, *ctx.saved_tensors, *ctx.how, ctx.inverse)


def rotary(q, k, positions, inv_freq, sections=None, pos_scale=1.0, rope_scale=1.0):
    """Rotate q (T, H, D) and k (T, Hkv, D), or q alone (k None), to their positions; returns both, in
    their dtype.

    positions (T,) or (axes, T): int32, int64 or float32.  inv_freq (R / 2,): pair (i, R / 2 + i) of a
    row turns by positions[axis of i] * pos_scale * inv_freq[i], the angle formed in 64 bits from the
    scale and the frequency in 32, and is scaled by rope_scale; elements from R on are copied.
    sections: how many frequencies each axis owns, in order (default: all of them one axis).  D a
    multiple of 8 up to 512, R / 2 a multiple of 8, T below 2^31.  Gradients and forward-mode tangents
    pass through q and k, not through positions or frequencies."""
    if torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad) \
            or forward_ad._current_level >= 0:               # a level in which a tensor may carry a tangent
        return _Rotary.apply(q, k, positions, inv_freq, sections, pos_scale, rope_scale, False)
    return native.rotary(q, k, positions, inv_freq, sections, pos_scale, rope_scale)


def rotary_grad(dq, dk, positions, inv_freq, sections=None, pos_scale=1.0, rope_scale=1.0):
    """The gradients of rotary's inputs from those of its outputs, without an autograd graph: the
    rotation the other way round, with the same scale.  Inputs with forward-mode tangents are refused."""
    if forward_ad._current_level >= 0 and any(x is not None and forward_ad.unpack_dual(x).tangent is not None
                                              for x in (dq, dk)):
        raise RuntimeError("rotary_grad keeps no graph and no forward-mode tangents: differentiate rotary")
    return native.rotary(dq, dk, positions, inv_freq, sections, pos_scale, rope_scale, inverse=True)


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(q, k, q_weight, k_weight, positions, inv_freq, sections, eps, pos_scale, rope_scale):
        return native.norm_rotary(q, k, q_weight, k_weight, positions, inv_freq, sections, eps, pos_scale, rope_scale)

    @staticmethod
    def setup_context(ctx, inputs, output):
        *tensors, ctx.sections, ctx.eps, ctx.pos_scale, ctx.rope_scale = inputs
        ctx.save_for_backward(*tensors)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        want = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        return (*native.norm_rotary_grad(dq, dk, *ctx.saved_tensors, ctx.sections, ctx.eps, ctx.pos_scale,
                                         ctx.rope_scale, want), None, None, None, None, None, None)


# apply() asks for it in every call: formed anew it would take 20 us of them
_NormRotary.forward.__signature__ = inspect.signature(_NormRotary.forward)


def norm_rotary(q, k, q_weight, k_weight, positions, inv_freq, sections=None, eps=1e-6, pos_scale=1.0, rope_scale=1.0):
    """Norm each head's row of q (T, H, D) and k (T, Hkv, D), or of q alone (k and k_weight None), and rotate it as
    rotary does; returns both, in their dtype.

    y = R(x / sqrt(mean(x^2) + eps) * weight), the mean over all D elements of a head's row.  q_weight and k_weight:
    (D,), shared by the heads, of one dtype of their own (bf16, fp16, fp32), or None for ones.  In fp32, rounded once
    at the end; positions, inv_freq, sections and scales as in rotary.  eps is at least 0.  Differentiable once, in q, k
    and the weights; forward-mode tangents are refused."""
    tensors = [x for x in (q, k, q_weight, k_weight) if x is not None]
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise RuntimeError("norm_rotary has no forward-mode derivative")
    if torch.is_grad_enabled() and any(x.requires_grad for x in tensors):
        return _NormRotary.apply(q, k, q_weight, k_weight, positions, inv_freq, sections, eps, pos_scale, rope_scale)
    return native.norm_rotary(q, k, q_weight, k_weight, positions, inv_freq, sections, eps, pos_scale, rope_scale)


def norm_rotary_grad(dq, dk, q, k, q_weight, k_weight, positions, inv_freq, sections=None, eps=1e-6, pos_scale=1.0,
                     rope_scale=1.0):
    """The gradients (dq, dk, dq_weight, dk_weight) of norm_rotary's inputs from those of its outputs, without an
    autograd graph; None where the input is None.  The weights' are summed over tokens and heads in one order: a
    call repeated gives the same bits.  Inputs with forward-mode tangents are refused."""
    if forward_ad._current_level >= 0 and any(x is not None and forward_ad.unpack_dual(x).tangent is not None
                                              for x in (dq, dk, q, k, q_weight, k_weight)):
        raise RuntimeError("norm_rotary_grad keeps no graph and no forward-mode tangents")
    return native.norm_rotary_grad(dq, dk, q, k, q_weight, k_weight, positions, inv_freq, sections, eps, pos_scale,
                                   rope_scale)


def cache_append(cache, k, v, table, lens, starts=None, seen=None):
    """Write new keys and values k, v (T, Hkv, D) behind the sequences' cached ones; returns the new
    lengths (B,) int32 (lens itself is not changed).

    table (B, pages of a sequence) int32, -1 where there is no page; lens (B,) int32 (64-bit numbers of
    either are clamped to 32).  Without starts
    every sequence gets one row (T = B); with starts (B + 1,) int32 the rows starts[b] ..
    starts[b + 1] - 1 are sequence b's, as far as k has them, and rows outside all of them are not
    read.  seen (B,): how many tokens the sequence has had before these, the first new key's cache.pos
    (default: its slot, right while nothing has been evicted).  New keys start with weight 0."""
    return native.cache_append(cache, k, v, table, lens, starts, seen)


def paged_attention(q, cache, table, lens, sm_scale=None, accumulate=False, want_lse=False, max_len=None, window=None,
                    sinks=0):
    """Attention of the last token, or the last Q tokens, of every sequence over its cached keys (their
    own among them): q (B, H, D) or (B, H, Q, D), query i of Q sees the first len - (Q - 1 - i) keys.
    Returns out like q; with want_lse also the log-sum-exp of the scaled scores, (B, H[, Q]) fp32.
    A query that sees no key gets zeros and -inf.

    window: of those keys a query, at position p, sees j > p - window and j < sinks only (default: all).
    Pages that no query of a sequence sees may be gone from its table (-1).  Slots count as positions, so
    not after an eviction, and accumulate does not go with it.

    accumulate: add every key's probability, summed over the queries and the heads of its kv head, to
    cache.weight; a page of such a call stands in one place of one sequence's table.  max_len: a bound
    on lens known to the host, at least 1 (default: the table's); lengths past it count as max_len.  It sizes the
    workspace of accumulate, 4 bytes a query row and key for fp32 and below 64 rows (queries times heads
    of a kv head).  Meant for a few new tokens: the last Q - 1 keys (with a window as many in front of it)
    are taken row by row."""
    return native.paged_attention(q, cache, table, lens, sm_scale, accumulate, want_lse, max_len, window, sinks)


def prefix_attention(q, cache, prefix, prefix_len, table, lens, sm_scale=None, want_lse=False, max_len=None):
    """paged_attention for sequences that begin with the same keys: every query sees the prefix_len keys
    (a number, at least 1) in the pages of prefix (pages,) int32, which all sequences share, and then its
    sequence's own: the keys of table and lens, which count these alone, as in paged_attention; lens may be 0.
    The prefix's keys are read once for all sequences.  B * H * Q up to 2^22."""
    return native.prefix_attention(q, cache, prefix, prefix_len, table, lens, sm_scale, want_lse, max_len)


def cache_evict(cache, table, lens, budget, n_global=32, n_local=32, dst_table=None, max_len=None):
    """Keep min(len, budget) keys of each kv head: the sequence's first n_global tokens and its latest
    n_local, then the keys of largest accumulated weight, the lower slot first among equals.  Returns
    the new lengths (B,) int32 (lens itself is not changed).

    In place (dst_table None) the kept keys in slots from budget on move into the dropped ones' slots, so
    that the keys of a sequence are no longer in the order of their tokens; cache.pos says which they
    are; a page stands in one place of one sequence's table, and a kept key whose new slot has no page is
    lost.  With dst_table (B, pages) the kept keys
    are copied, in order, to that table's pages, others than the source's, which may be shared and stay
    as they are.  Keys without a page rank last; one that is kept all the same leaves its slot of
    dst_table unwritten."""
    return native.cache_evict(cache, table, lens, budget, n_global, n_local, dst_table, max_len)
