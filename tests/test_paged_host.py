"""Host side of the paged operators, on the CPU: what compile() refuses, and the launches of a run
(recorded by hip_stub, so operands may be views of any size over a small buffer)."""

import numpy as np
import pytest

import hip_stub
import paged_ref as R
from pto_wsp import CompileError, Dense, DenseDyn, DType, P, Tensor, paged_attention, paged_plan, paged_store, sequential, workload

NP = {DType.I32: np.int32, DType.F32: np.float32, DType.F16: np.float16, DType.BF16: np.uint16, DType.I8: np.int8, DType.F8E4M3: np.uint8}


def T(dtype, *shape):
    """A tensor of any size; its first elements alone are backed by memory."""
    return Tensor(data=np.lib.stride_tricks.as_strided(np.zeros(4096, NP[dtype]), shape, _strides(shape, NP[dtype])), shape=shape, dtype=dtype)


def _strides(shape, dtype):
    out, at = [], np.dtype(dtype).itemsize
    for n in reversed(shape):
        out.append(at)
        at *= max(n, 1)
    return tuple(reversed(out))


I32, F32, BF16, E4M3 = DType.I32, DType.F32, DType.BF16, DType.F8E4M3


def plan(batch=4, width=8, rows=7, page=16, **other):
    t = dict(lengths=T(I32, batch), counts=T(I32, batch), page_table=T(I32, batch, width), free_pages=T(I32, 9), used=T(I32, 1),
             new_lengths=T(I32, batch), new_used=T(I32, 1), starts=T(I32, batch + 1), slots=T(I32, rows), page_size=page)
    return paged_plan(**dict(t, **other))


def cache(code=E4M3, pages=6, heads=2, page=16, D=64, **other):
    t = {x + "_cache": T(code, pages, heads, page, D) for x in "kv"} | {x + "_scale": T(F32, pages, heads) for x in "kv"}
    return dict(t, **other)


def store(rows=5, heads=2, D=64, dt=BF16, c=None, **other):
    return paged_store(**dict(dict(k=T(dt, rows, heads, D), v=T(dt, rows, heads, D), slots=T(I32, rows)) | (c or cache(heads=heads, D=D)), **other))


def attend(rows=5, heads=2, G=4, D=64, batch=3, dt=BF16, c=None, **other):
    t = dict(q=T(dt, rows, heads * G, D), out=T(dt, rows, heads * G, D), page_table=T(I32, batch, 4), lengths=T(I32, batch), starts=T(I32, batch + 1))
    return paged_attention(**dict(t | (c or cache(heads=heads, D=D)), **other))


@pytest.mark.parametrize("make,match", [
    (lambda: plan(counts=T(I32, 5)), "counts has the shape"),
    (lambda: plan(starts=T(I32, 4)), "starts has the shape"),
    (lambda: plan(page_table=T(I32, 3, 8)), "3 rows for 4 requests"),
    (lambda: plan(lengths=T(DType.I8, 4)), "unsupported type i8"),
    (lambda: plan(used=T(I32, 2)), "used has the shape"),
    (lambda: plan(page=0), "pages of 0 tokens"),
    (lambda: plan(page=5000), "pages of 5000 tokens"),
    (lambda: plan(slots=T(I32, 7, 1)), "rank 1 is needed"),
    (lambda: store(v=T(BF16, 5, 2, 32)), "v has the shape"),
    (lambda: store(v=T(DType.F16, 5, 2, 64)), "k and v differ in type"),
    (lambda: store(slots=T(I32, 4)), "slots has the shape"),
    (lambda: store(c=cache(BF16)), "unsupported type bf16"),
    (lambda: store(c=cache(v_cache=T(DType.I8, 6, 2, 16, 64))), "differ in type"),
    (lambda: store(c=cache(k_scale=T(F32, 6, 1))), "k_scale has the shape"),
    (lambda: store(c=cache(v_scale=T(BF16, 6, 2))), "unsupported type bf16"),
    (lambda: store(heads=3), None),
    (lambda: store(D=72), "head size 72"),
    (lambda: store(D=272), "head size 272"),
    (lambda: store(c=cache(pages=0)), "a cache of 0 pages"),
    (lambda: store(dt=I32), "unsupported type i32"),
    (lambda: attend(c=cache(D=32)), "q has the head size 64"),
    (lambda: attend(c=cache(heads=3)), "8 query heads for 3 key heads"),
    (lambda: attend(out=T(F32, 5, 8, 64)), "q and out differ in type"),
    (lambda: attend(out=T(BF16, 4, 8, 64)), "out has the shape"),
    (lambda: attend(lse=T(F32, 5, 2)), "lse has the shape"),
    (lambda: attend(starts=T(I32, 3)), "starts has the shape"),
    (lambda: attend(page_table=T(I32, 2, 4)), "2 rows for 3 requests"),
    (lambda: attend(page_table=T(I32, 3, 1 << 28)), "2\\^31 tokens"),
    (lambda: attend(window=-1), "a negative window"),
    (lambda: attend(dt=F32, window=9, c=cache(page=8)), "multiple of 16 tokens"),
    (lambda: attend(dt=F32, window=9, c=cache(page=16)), None),
    (lambda: attend(dt=F32, c=cache(page=8)), None),
    (lambda: attend(scale=float("inf")), "non-finite"),
    (lambda: attend(q=T(BF16, 5, 8)), "rank 3 is needed"),
])
def test_refusals(make, match):
    w = make()
    if match is None:
        with hip_stub.program(w):
            return
    with pytest.raises(CompileError, match=match):
        w.compile(target="hip_gfx950")


def test_operands_are_tensors():
    with pytest.raises(TypeError, match="q must be a Tensor"):
        attend(q=np.zeros((5, 8, 64)))
    with pytest.raises(TypeError):
        paged_store(k=T(BF16, 1, 2, 64))


def test_indexed_by_host_values_only():
    counts, index = T(I32, 3, 4), T(I32, 3)

    @workload
    def wl():
        for i in P.seq(Dense[3](), name="i"):
            plan(counts=counts[index[i]])

    with pytest.raises(CompileError, match="not indexed by a tensor"):
        wl().compile(target="hip_gfx950")


def test_index_outside_its_tensor():
    counts, n = T(I32, 3, 4), DenseDyn(0)

    @workload
    def wl():
        for i in P(n, names=["i"]):
            plan(counts=counts[i])

    with hip_stub.program(wl()) as once:
        once.prog.set_axis_sizes({"i": 3})
        assert len(once()) == 3
        once.prog.set_axis_sizes({"i": 4})
        with pytest.raises(RuntimeError, match="index 3 of counts is outside its tensor"):
            once()


def _entries(launches):
    return [x.entry.replace("ptowsp_paged_", "") for x in launches]


def test_launches_of_a_plan():
    for batch, rows, want in ((4096, 6144, ["plan"]), (4097, 4, ["plan_sums", "plan_rows"]), (1, 6145, ["plan_sums", "plan_rows"]), (5000, 0, ["plan_sums"])):
        with hip_stub.program(plan(batch, 8, rows)) as once:
            launches = once()
            assert _entries(launches) == want
            if len(launches) == 2:
                assert launches[1].blocks == -(-rows // 1024)


def test_launches_of_attention():
    """The kernel for prompts only where a request may have more than 64 rows a key head, of a call of more than 8192."""
    few, prompts = ["attention", "attention_join"], ["attention_units", "attention_prompts", "attention_finish"]
    for rows, batch, G, want in ((1024, 3, 4, few), (1025, 3, 4, prompts), (1040, 1025, 4, few), (1041, 1025, 4, prompts), (64, 1, 64, few), (65, 1, 64, prompts)):
        with hip_stub.program(attend(rows=rows, batch=batch, G=G)) as once:
            assert _entries(once()) == want


def test_empty_calls_launch_nothing():
    for w in (store(rows=0), attend(rows=0), attend(batch=0, page_table=T(I32, 0, 4))):
        with hip_stub.program(w) as once:
            assert once() == []


def test_operands_at_execute():
    """Strides and overlaps, known when a run binds its tensors."""
    k = T(E4M3, 6, 2, 16, 64)
    k.data = np.zeros((6, 2, 16, 128), np.uint8)[..., ::2]
    q = T(BF16, 5, 8, 64)
    wide = T(BF16, 5, 8, 64)
    wide.data = np.zeros((64, 8, 5), np.uint16).transpose(2, 1, 0)
    odd = T(E4M3, 6, 2, 16, 64)
    odd.data = np.zeros((6, 2, 16, 72), np.uint8)[..., :64]
    far = T(E4M3, 6, 2, 16, 64)
    far.data = np.lib.stride_tricks.as_strided(np.zeros(64, np.uint8), (6, 2, 16, 64), (64, 64, 1 << 27, 1))
    apart = T(E4M3, 2, 2, 16, 64)
    apart.data = np.lib.stride_tricks.as_strided(np.zeros(64, np.uint8), (2, 2, 16, 64), (1 << 32, 1024, 64, 1))
    two = cache(pages=2, k_cache=apart)
    sparse = T(F32, 6, 2)
    sparse.data = np.lib.stride_tricks.as_strided(np.zeros(64, np.float32), (6, 2), (1 << 34, 4))
    for w, match in ((attend(c=two), "pages lie too far apart"), (store(c=two), "pages lie too far apart"),
                     (attend(v_scale=sparse), "pages lie too far apart"),
                     (attend(k_cache=k), "must have stride 1"), (attend(q=q, out=q), "lies where q does"), (attend(q=wide), "must have stride 1"),
                     (attend(k_cache=odd), "multiples of 16"), (store(k_cache=odd), "multiples of 16"), (attend(v_cache=far), "too far apart")):
        with hip_stub.program(w) as once:
            with pytest.raises(RuntimeError, match=match):
                once()


def test_captured_runs_keep_their_workspace():
    with hip_stub.program(sequential(plan(5000), attend(batch=5000, rows=5000, page_table=T(I32, 5000, 4)))) as once:
        with pytest.raises(RuntimeError):  # nothing has been allocated yet
            once(capture=True)
        assert len(once()) == 4
        assert len(once(capture=True)) == 4
        with pytest.raises(RuntimeError, match="captured after a run"):
            once(capture=True)
        once()
        once(capture=True)


def test_loops_over_layers():
    c = {x: T(t.dtype, 3, *t.shape) for x, t in cache().items()}
    q, out = T(BF16, 3, 5, 8, 64), T(BF16, 3, 5, 8, 64)

    @workload
    def wl():
        plan()
        for i in P.seq(Dense[3](), name="i"):
            attend(q=q[i], out=out[i], c={x: t[i] for x, t in c.items()})

    with hip_stub.program(wl()) as once:
        assert _entries(once())[0] == "plan" and sum(e.startswith("attention") for e in _entries(once())) >= 3
        assert once.prog.stats.task_count == 0 and once.prog.stats.total_cycles == 0


def test_tiles_of_f8_are_refused():
    from pto_wsp import In, Out, Tile, kernel, pto

    @kernel
    def copy(x: In[Tile[4, 4, E4M3]], y: Out[Tile[4, 4, E4M3]]):
        pto.store(y, x)

    a, b = T(E4M3, 4, 4), T(E4M3, 4, 4)

    @workload
    def wl():
        copy(x=a, y=b)

    with pytest.raises(CompileError, match="f8e4m3"):
        wl().compile(target="hip_gfx950")


def test_reference_codes():
    """The tests' own codes against torch's conversion, over every code, its neighbours and the ties between them."""
    import torch

    v = R.E4M3
    mids = (v[1:] + v[:-1]) / 2
    y = np.concatenate([v, mids, np.nextafter(mids, 0), np.nextafter(mids, 999), [448.0, 449.0, 1e9]]).astype(np.float32).astype(np.float64)
    y = np.concatenate([y, -y])
    want = torch.from_numpy(np.clip(y, -448, 448).astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(R.encode(y, "e4m3"), want)
    assert np.array_equal(R.decode(np.arange(256), "e4m3")[:127], torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())
