"""Operands of the paged operators that share memory, on the CPU (launches are recorded instead of run)."""

import ctypes

import numpy as np
import pytest

import hip_stub
from pto_wsp import DType, Tensor
from test_paged_host import E4M3, I32, T, attend, cache, plan, store


def tensor(x, dtype):
    return Tensor(data=x, shape=x.shape, dtype=dtype)


class Pool:
    """Views of one allocation."""

    def __init__(self, dtype, n):
        self.x = np.zeros(n, dtype)

    def view(self, kind, first, shape, strides):
        assert first + sum((n - 1) * s for n, s in zip(shape, strides)) < len(self.x)
        return tensor(np.lib.stride_tricks.as_strided(self.x[first:], shape, [s * self.x.itemsize for s in strides]), kind)

    def run(self, workload):
        with hip_stub.program(workload) as once:
            hip_stub._lib.stub_allocation(ctypes.c_void_p(self.x.ctypes.data), ctypes.c_uint64(self.x.nbytes))
            try:
                return once()
            finally:
                hip_stub._lib.stub_allocation(None, ctypes.c_uint64(0))


def rows(pool, first, step=8 * 64):
    return pool.view(DType.BF16, first, (5, 8, 64), (step, 64, 1))


def codes(pool, first, strides, shape=(6, 2, 16, 64)):
    return pool.view(E4M3, first, shape, strides)


@pytest.mark.parametrize("first,step,ok", [
    (0, 512, False), (512, 512, False), (4 * 512, 512, False), (4 * 512 + 511, 512, False), (5 * 512, 512, True),
    (2 * 512, 1024, False),  # other strides, a row in common
])
def test_rows_of_one_buffer(first, step, ok):
    pool = Pool(np.uint16, 16 * 512)
    w = attend(q=rows(pool, 0), out=rows(pool, first, step))
    if ok:
        assert pool.run(w)
        return
    with pytest.raises(RuntimeError, match="out is written and lies where q does"):
        pool.run(w)


def test_rows_between_each_other():
    """[q | out] rows, and out a byte's worth into q's."""
    pool = Pool(np.uint16, 5 * 1024)
    assert pool.run(attend(q=rows(pool, 0, 1024), out=rows(pool, 512, 1024)))
    with pytest.raises(RuntimeError, match="out is written and lies where q does"):
        pool.run(attend(q=rows(pool, 0, 1024), out=rows(pool, 511, 1024)))


def test_fused_caches():
    """Keys and values of a token beside each other, of a page, of a head; then a token, a page or 16 bytes too near."""
    pool = Pool(np.uint8, 1 << 17)
    for strides, other in (((4096, 64, 256, 1), 128), ((4096, 1024, 64, 1), 2048), ((4096, 2048, 128, 1), 64), ((4096, 2048, 64, 1), 1024)):
        assert pool.run(store(c=cache(k_cache=codes(pool, 0, strides), v_cache=codes(pool, other, strides))))
    for strides, other in (((4096, 64, 256, 1), 64), ((4096, 1024, 64, 1), 2048 - 64), ((4096, 2048, 128, 1), 48), ((2048, 1024, 64, 1), 2048)):
        with pytest.raises(RuntimeError, match="_cache is written and lies where ._cache does"):
            pool.run(store(c=cache(k_cache=codes(pool, 0, strides), v_cache=codes(pool, other, strides))))


def test_an_operand_upon_itself():
    pool = Pool(np.uint8, 1 << 17)
    for strides in ((1024, 1024, 64, 1), (2048, 1024, 32, 1), (2048, 512, 64, 1)):
        with pytest.raises(RuntimeError, match="k_cache is written and has elements that share memory"):
            pool.run(store(c=cache(k_cache=codes(pool, 0, strides))))
    assert pool.run(attend(c=cache(k_cache=codes(pool, 0, (1024, 1024, 64, 1)))))  # read only
    pool.run(store(c=cache(k_cache=codes(pool, 0, (1024, 6 * 1024, 64, 1)))))  # heads ahead of pages


def test_random_views():
    """Against every element's address."""
    rng = np.random.default_rng(0)
    pool, seen = Pool(np.int32, 400), [0, 0]

    def draw(shape):
        s = rng.choice([1, 2, 3, 4, 5, 6, 8, 12, 24], len(shape))
        return int(rng.integers(0, 60)), [int(x) for x in s]

    def elements(first, shape, strides):
        return (first + sum(np.arange(n).reshape([-1 if i == d else 1 for i in range(len(shape))]) * s for d, (n, s) in enumerate(zip(shape, strides)))).ravel()

    for _ in range(200):
        (a, sa), (b, sb) = draw((4, 5)), draw((4,))
        table, lengths = pool.view(I32, a, (4, 5), sa), pool.view(I32, b, (4,), sb)
        ea, eb = elements(a, (4, 5), sa), elements(b, (4,), sb)
        bad = len(set(ea)) < len(ea) or bool(set(ea) & set(eb))
        seen[bad] += 1
        w = plan(batch=4, width=5, page_table=table, lengths=lengths)
        if bad:
            with pytest.raises(RuntimeError, match="share memory|lies where"):
                pool.run(w)
        else:
            pool.run(w)
    assert min(seen) > 20


def test_plans_in_place():
    pool = Pool(np.int32, 64)
    here = pool.view(I32, 8, (4,), (2,))
    assert pool.run(plan(lengths=here, new_lengths=here))
    assert pool.run(plan(lengths=here, new_lengths=pool.view(I32, 8, (4,), (2,))))
    for first, step in ((8, 1), (10, 2), (6, 4)):
        with pytest.raises(RuntimeError, match="new_lengths is written and lies where lengths does"):
            pool.run(plan(lengths=here, new_lengths=pool.view(I32, first, (4,), (step,))))
    assert pool.run(plan(batch=1, lengths=pool.view(I32, 8, (1,), (2,)), new_lengths=pool.view(I32, 8, (1,), (1,))))
    with pytest.raises(RuntimeError, match="new_used is written and lies where lengths does"):
        pool.run(plan(lengths=here, new_used=pool.view(I32, 14, (1,), (1,))))


def test_strides_alone_are_not_memory():
    """Two large views over small buffers of their own: what lies there is not known."""
    with hip_stub.program(attend(rows=4000, q=T(DType.BF16, 4000, 8, 64), out=T(DType.BF16, 4000, 8, 64))) as once:
        assert once()
