"""Matrix products of 8-bit floating point with a scale for each block of 128, as workload steps.

A matrix is held as e4m3 codes (``DType.F8E4M3``) and float32 scales: a number is its code times the scale of its
block.  Activations have blocks of 1 row by 128 columns, weights of 128 by 128; the last ones may be cut short.

* ``block_quantize``  numbers into codes and scales;
* ``block_matmul``    the product of activations and weights.

Each call returns a ``Workload`` as the operators over a paged cache do (``pto_wsp.paged``): it compiles by itself,
stands in ``sequential`` beside others, or is added to the loop around it, and raises as they do.
"""

from __future__ import annotations

from pto_wsp.paged import _operator
from pto_wsp.types import Tensor
from pto_wsp.workload import Workload

__all__ = ["block_quantize", "block_matmul"]


def block_quantize(*, x: Tensor, codes: Tensor, scales: Tensor, rows: int = 1) -> Workload:
    """``x [M, K]`` (BF16, F16 or F32) as ``codes [M, K]`` (F8E4M3) and ``scales [ceil(M / rows), ceil(K / 128)]`` (F32).

    Blocks have ``rows`` rows, 1 (activations) or 128 (weights), and 128 columns.  A block's scale is the larger of
    ``max |x| / 448`` over its finite numbers and 2^-126; a code is ``x * (1 / scale)`` rounded to nearest (even on
    ties) within +-448; scale, reciprocal and product are float32.  Infinities become +-448, a NaN the e4m3 NaN.
    """
    return _operator("block_quantize", {"x": x, "codes": codes, "scales": scales}, {"rows": int(rows)})


def block_matmul(*, a: Tensor, a_scale: Tensor, b: Tensor, b_scale: Tensor, out: Tensor) -> Workload:
    """``out [M, N]`` (BF16, F16 or F32) = activations ``a [M, K]`` times the transpose of weights ``b [N, K]``.

    ``a_scale [M, ceil(K / 128)]`` and ``b_scale [ceil(N / 128), ceil(K / 128)]`` are the scales of their codes:
    ``out[m, n]`` is the sum over blocks j of ``a_scale[m, j] * b_scale[n // 128, j]`` times the sum of the block's
    products of codes.  Sums are float32, rounded once at the end.  For BF16 and F16 results the matrix instruction
    cuts each product at 2^-13 of the largest of the eight that it adds at once, which costs 1.5e-5 of a typical
    result; for F32 results products are exact.  Scales may be any, also such that their product lies beyond float32
    where the result does not.  Rows of a and b may lie at any distance; where a row's codes, its distance and K are
    multiples of 16 bytes they are loaded straight into shared memory.
    """
    return _operator("block_matmul", {"a": a, "a_scale": a_scale, "b": b, "b_scale": b_scale, "out": out}, {})
