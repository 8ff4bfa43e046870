"""Operators over a paged KV cache held in 8 bits, as workload steps.

A cache of ``P`` pages for ``H`` key heads of size ``D`` is two code tensors ``[P, H, page, D]``
(``DType.I8`` or ``DType.F8E4M3``) and two scale tensors ``[P, H]`` (F32): a stored number is its code
times the scale of its page and head.  A request's tokens lie in the pages that its row of the page
table names, ``page`` tokens each.  A serving step of requests with new tokens, packed one behind the
other into rows, is

* ``paged_plan``       pages for the new tokens, where each row goes, where each request starts;
* ``paged_norm_rotate`` norms of the rows' queries and keys, and their rotation by position;
* ``paged_store``      the rows' keys and values into the cache;
* ``paged_attention``  the rows' queries over their requests' tokens;
* ``paged_prefix_attention`` the same where requests share a prefix, which is read once for all of them.

Each call returns a ``Workload`` that compiles by itself, stands in ``sequential`` beside others, or,
called inside a ``@workload``, is added to the loop around it; operands are tensors or views of them
indexed by constants and loop variables (``K[layer]``).  Loops around an operator run on the host, in
order.  A compiled program may be captured into a HIP graph after a run with the same bindings; run it
once more before it is captured again, since every captured run keeps its workspace.

Wrong types, shapes and attributes raise ``CompileError`` from ``compile()``, wrong strides or devices
``RuntimeError`` from ``execute()``, as does a written operand of which a byte is another operand's or its own
again (keys and values may lie between each other's rows); lengths, slots and page numbers are read on the device, and
``synchronize()`` raises ``ExecutionError`` for the ones out of range.  The cycle model has no tasks here.
"""

from __future__ import annotations

import math
from typing import Any, Optional

from pto_wsp.types import Tensor
from pto_wsp.workload import Workload

__all__ = ["paged_plan", "paged_norm_rotate", "paged_store", "paged_attention", "paged_prefix_attention"]


def _operator(op: str, tensors: dict, attrs: dict) -> Workload:
    from pto_wsp.primitives import _builder_add

    for name, t in tensors.items():
        if not isinstance(t, Tensor):
            raise TypeError(f"{op}: {name} must be a Tensor (got {type(t).__name__})")
    w = Workload("operator", op=op, tensors=tensors, attrs=attrs)
    _builder_add(w, needs_frame=False)
    return w


def paged_plan(*, lengths: Tensor, counts: Tensor, page_table: Tensor, free_pages: Tensor, used: Tensor,
               new_lengths: Tensor, new_used: Tensor, starts: Tensor, slots: Tensor, page_size: int) -> Workload:
    """Pages and rows for the new tokens of ``B`` requests.  Every tensor is I32.

    ``lengths[B]`` tokens are cached, ``counts[B]`` are added (0: none).  ``page_table[B, W]`` names the
    pages of the cached tokens; the pages that a request lacks are appended to its row, taken in order of
    requests from ``free_pages[F]``, whose first ``used[1]`` entries are gone.  Writes

    * ``new_lengths[B]`` = lengths + counts and ``new_used[1]`` (each may be where it comes from, with the same stride);
    * ``starts[B + 1]``: request b has the rows ``starts[b] .. starts[b + 1] - 1``;
    * ``slots[T]``: page * page_size + offset of each row's token, -1 behind the last row.

    Where a length or count is negative, or the page table, the free pages or the ``T`` rows do not
    suffice, ``synchronize()`` raises and nothing has been written.  Steps behind it in the same run take
    ``starts`` and ``slots`` as they were: a plan that may run out of pages is synchronized before the
    rows are stored.
    """
    return _operator("paged_plan", {"lengths": lengths, "counts": counts, "page_table": page_table, "free_pages": free_pages,
                                    "used": used, "new_lengths": new_lengths, "new_used": new_used, "starts": starts,
                                    "slots": slots}, {"page_size": int(page_size)})


def paged_norm_rotate(*, q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, lengths: Tensor, starts: Tensor, q_out: Tensor, k_out: Tensor,
                      q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None, offsets: Optional[Tensor] = None,
                      eps: float = 1e-6, interleaved: bool = False) -> Workload:
    """Norm and rotation of rows ``q [T, Hq, D]`` and ``k [T, Hk, D]`` (BF16, F16 or F32) in one pass.

    Each head becomes ``x / sqrt(mean(x^2) + eps) * weight`` where its ``q_weight[D]`` or ``k_weight[D]`` (any of
    the types) is given.  Then the first ``R = 2 * cos.shape[1]`` of its dims are rotated: pair i, which is dims
    ``i`` and ``i + R / 2`` or, ``interleaved``, ``2 i`` and ``2 i + 1``, becomes ``(a c - b s, b c + a s)`` with
    ``c, s = cos[p][i], sin[p][i]`` (``[positions, R / 2]``, F32).  Request b holds ``lengths[B]`` tokens, its rows
    ``starts[b] .. starts[b + 1] - 1`` are its last ones; a token's position p is its place among them, plus
    ``offsets[b]`` (the tokens of a shared prefix, say).  D is a multiple of 16 up to 256.

    All is computed in float32 (heads whose squares add up to more than it holds become 0) and rounded once, into
    ``q_out`` and ``k_out`` (as q and k, and each may be where it comes from, with the same strides).  Rows of no
    request are left alone; positions outside the tables, and rows of a request beyond its ``lengths[b]`` tokens, raise
    from ``synchronize()`` and are left out; starts that go down, or lie beyond the rows, raise too.
    """
    tensors: dict[str, Any] = {"q": q, "k": k, "cos": cos, "sin": sin, "lengths": lengths, "starts": starts, "q_out": q_out, "k_out": k_out}
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight), ("offsets", offsets)):
        if t is not None:
            tensors[name] = t
    return _operator("paged_norm_rotate", tensors, {"eps": float(eps), "interleaved": int(interleaved)})


def paged_store(*, k: Tensor, v: Tensor, slots: Tensor, k_cache: Tensor, v_cache: Tensor, k_scale: Tensor,
                v_scale: Tensor) -> Workload:
    """Rows ``k, v [T, H, D]`` (BF16, F16 or F32) into the cache at ``slots[T]`` (I32; below 0: not stored).

    Neighbouring rows of one page go into it together; a page is named by one such run of rows.  With the
    tokens ahead of the run's first one kept, the scale of a page and head becomes the largest of its old
    value (if tokens are kept), ``max |x| / top`` over the run's finite numbers (top: 127 or 448) and
    2^-126; kept tokens are coded anew where it grows.  A code is ``x * (1 / scale)`` rounded to nearest
    (even on ties) within +-top; scale, reciprocal and product are float32.  Infinities are stored as
    +-top, a NaN as the e4m3 NaN or 0.  Tokens of the page behind the run count as not stored.
    """
    return _operator("paged_store", {"k": k, "v": v, "slots": slots, "k_cache": k_cache, "v_cache": v_cache,
                                     "k_scale": k_scale, "v_scale": v_scale}, {})


def paged_attention(*, q: Tensor, k_cache: Tensor, v_cache: Tensor, k_scale: Tensor, v_scale: Tensor, page_table: Tensor,
                    lengths: Tensor, starts: Tensor, out: Tensor, scale: Optional[float] = None, window: int = 0,
                    lse: Optional[Tensor] = None) -> Workload:
    """Causal attention of rows ``q [T, G * H, D]`` (BF16, F16 or F32) over an 8-bit paged cache.

    Query head ``h`` reads key head ``h // G``.  Request b holds ``lengths[B]`` tokens, the new ones
    among them; its rows ``starts[b] .. starts[b + 1] - 1`` are its last tokens, one or many.  A row at
    position p attends to the positions 0 .. p, or to the last ``window`` of those.  ``out`` (as q) is
    softmax(scale * q k^T) v, 0 for a row without positions; ``lse [T, G * H]`` (F32) the logarithm of the
    softmax's sum, -inf there.  ``scale`` defaults to 1 / sqrt(D) and may be negative; scales of the cache
    are not.  Rows behind the last request, and what lies in the cache beyond a request's tokens, are left
    alone.

    Scores, maxima and sums are float32.  A weight is held to 2^-16 of itself for 16-bit queries and to 2^-24
    for F32 ones.  In prompts of BF16 queries (requests of more than 64 rows a key head, in calls of more than
    8192 query rows; head size up to 128, pages of a multiple of 16 tokens) weights, values and their scales
    are f16, each off by at most 2^-11, an eighth of the output's own rounding.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if isinstance(q, Tensor) and q.shape and q.shape[-1] > 0 else 1.0
    tensors: dict[str, Any] = {"q": q, "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale,
                               "page_table": page_table, "lengths": lengths, "starts": starts, "out": out}
    if lse is not None:
        tensors["lse"] = lse
    return _operator("paged_attention", tensors, {"window": int(window), "scale": float(scale)})


def paged_prefix_attention(*, q: Tensor, k_cache: Tensor, v_cache: Tensor, k_scale: Tensor, v_scale: Tensor, prefix_table: Tensor,
                           prefix_lengths: Tensor, members: Tensor, page_table: Tensor, lengths: Tensor, starts: Tensor, out: Tensor,
                           scale: Optional[float] = None, lse: Optional[Tensor] = None) -> Workload:
    """``paged_attention`` of requests in groups, each behind a prefix of its own that the group shares.

    Group s is the requests ``members[s] .. members[s + 1] - 1`` (``members[S + 1]``, ascending); requests ahead of
    the first group and behind the last one have no prefix.  Its prefix is ``prefix_lengths[S]`` tokens (0: none)
    in the pages of ``prefix_table[S, W]``, of the same cache.  ``lengths[B]``, ``page_table[B, W]`` and
    ``starts[B + 1]`` are of the requests' own tokens, as in ``paged_attention``, and a row attends to its group's
    whole prefix and to the positions 0 .. p of its own: one softmax over both.  ``out`` and ``lse`` are as there.

    A group's rows go over its prefix together, so that its pages are read once and not once a request.  Sums,
    maxima and the results of both parts are float32; weights are held as there, and in groups of more than 64
    rows a key head as in prompts there, in calls of any size.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if isinstance(q, Tensor) and q.shape and q.shape[-1] > 0 else 1.0
    tensors: dict[str, Any] = {"q": q, "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale, "page_table": page_table,
                               "lengths": lengths, "starts": starts, "prefix_table": prefix_table, "prefix_lengths": prefix_lengths,
                               "members": members, "out": out}
    if lse is not None:
        tensors["lse"] = lse
    return _operator("paged_prefix_attention", tensors, {"scale": float(scale)})
