"""Embedding lookup and its gradient against 64-bit sums.  Tolerances: a sum of c float32 terms added one by one is
off by at most (c - 1) * 2^-24 times the sum of the terms' sizes (twice that to first order covers the levels of
partial sums), the product with the scale adds 2^-24, and the rounding to the element type half a step."""
import ctypes

import numpy as np
import pytest
import torch

from featgraph_amd import _lib, nd, placeholder
from featgraph_amd.module import EmbeddingLookupGradhip, EmbeddingLookuphip

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -25}


def _normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(TYPES[dtype]).cuda()


def _ids(n, V, kind, seed, itype="int32"):
    rng = np.random.default_rng(seed)
    if kind == "power":
        ids = np.minimum((rng.random(n) ** 3 * V).astype(np.int64), V - 1)
    elif kind == "one":
        ids = np.full(n, V // 2, dtype=np.int64)
    elif kind == "two":
        ids = np.where(np.arange(n) < n // 3, V - 1, 0).astype(np.int64)
    elif kind == "distinct":
        ids = rng.permutation(V)[:n].astype(np.int64)
    elif kind == "padding":
        ids = np.full(n, -1, dtype=np.int64)
    else:
        ids = rng.integers(0, V, n)
        ids[rng.random(n) < 0.2] = -1
        if n:
            ids[rng.integers(0, n, max(1, n // 50))] = V       # one past the last row
            ids[0] = V - 1
    return torch.from_numpy(ids).to(getattr(torch, itype)).cuda()


def _want_grad(ids, dout, V, scale):
    i = ids.reshape(-1).long()
    ok = (i >= 0) & (i < V)
    D = dout.shape[-1]
    d = dout.reshape(-1, D)[ok].double() * scale
    want = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_put_((i[ok],), d, accumulate=True)
    size = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_put_((i[ok],), d.abs(), accumulate=True)
    count = torch.zeros(V, dtype=torch.float64, device="cuda").index_put_((i[ok],), torch.ones_like(i[ok], dtype=torch.float64), accumulate=True)
    return want, size, count


def _check_grad(got, want, size, count, dtype, extra=0.0):
    tol = 2 * (count[:, None] + 2) * 2.0 ** -24 * size + HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -8) + TINY[dtype] + extra
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (7, 5, 3), (61, 4096, 64), (257, 100, 100), (1000, 333, 30), (5, 9, 1030),
                                   (3, 4, 4099)])
@pytest.mark.parametrize("itype", ["int32", "int64"])
def test_lookup(dtype, n, V, D, itype):
    table, ids = _normal((V, D), dtype, 1), _ids(n, V, "mixed", 2, itype)
    scale = 1.7
    m = EmbeddingLookuphip(scale)
    m.build([placeholder((V, D), dtype), placeholder((n,), itype)])
    m.out_tvm.tensor.fill_(9)
    got = m.run([table, ids]).tensor
    ok = (ids >= 0) & (ids < V)
    want = torch.zeros(n, D, dtype=torch.float64, device="cuda")
    want[ok] = table[ids[ok].long()].double() * float(torch.tensor(scale, dtype=torch.float32))
    # the product of two float32 values is exact in float64; it is rounded to float32 (2^-24) and to the element type
    # (half a step), or at once to the element type where the device has such a multiplication, as it does for float16
    tol = want.abs() * (2.0 ** -24 * (dtype != "float32") + HALF_STEP[dtype]) * (1 + 2.0 ** -20) + TINY[dtype]
    assert got.dtype == TYPES[dtype] and got.shape == (n, D)
    assert bool(((got.double() - want).abs() <= tol).all()) and not got[~ok].any()


@pytest.mark.gpu
def test_lookup_of_a_matrix_of_ids_and_of_none():
    table = _normal((50, 24), "float32", 3)
    ids = _ids(35, 50, "mixed", 4, "int64").reshape(5, 7)
    m = EmbeddingLookuphip()
    m.build([placeholder((50, 24)), placeholder((5, 7), "int64")])
    got = m.run([nd.array(table), nd.array(ids)])
    assert got.shape == (5, 7, 24)
    ok = (ids >= 0) & (ids < 50)
    assert torch.equal(got.tensor[ok], table[ids[ok]]) and not got.tensor[~ok].any()
    none = EmbeddingLookuphip()
    none.build([placeholder((50, 24)), placeholder((0,), "int32")])
    assert none.run([table, ids.reshape(-1)[:0].int()]).shape == (0, 24)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,V,D,kind", [(1, 1, 1, "mixed"), (1, 7, 5, "padding"), (16, 3, 8, "one"), (17, 40, 33, "mixed"),
                                        (333, 4096, 100, "power"), (2000, 70, 64, "mixed"), (8192, 5000, 12, "power"),
                                        (8193, 5000, 12, "power"), (9000, 9, 130, "mixed"), (20000, 3, 40, "two"),
                                        (70001, 50, 6, "one"), (30000, 4097, 520, "power"), (50000, 5000000, 4, "distinct"),
                                        (12345, 1, 7, "mixed"), (9999, 77, 5, "padding")])
def test_gradient(dtype, n, V, D, kind):
    if V > 2000000 and dtype != "float32":
        D = 2
    itype = "int64" if n % 2 else "int32"
    ids, dout = _ids(n, V, kind, n + 1, itype), _normal((n, D), dtype, n + 2, 0.5)
    m = EmbeddingLookupGradhip(0.75)
    m.build([placeholder((V, D), dtype), placeholder((n,), itype)])
    got = m.run([ids, dout]).tensor
    want, size, count = _want_grad(ids, dout, V, 0.75)
    _check_grad(got, want, size, count, dtype)
    assert not got[count == 0].any()
    got = got.clone()
    m.out_tvm.tensor.fill_(float("nan"))                      # every row is written, and the same bits come again
    assert torch.equal(m.run([ids, dout]).tensor, got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,V,D,kind", [(40, 300, 20, "mixed"), (20000, 1000, 24, "power"), (9000, 4, 16, "one")])
def test_gradient_added_to_the_callers(dtype, n, V, D, kind):
    ids, dout, grad = _ids(n, V, kind, 5), _normal((n, D), dtype, 6, 0.1), _normal((V, D), dtype, 7)
    m = EmbeddingLookupGradhip(2.0)
    m.build([placeholder((V, D), dtype), placeholder((n,), "int32")])
    want, size, count = _want_grad(ids, dout, V, 2.0)
    before = grad.clone()
    out = m.run([ids, dout, grad])
    assert out.tensor.data_ptr() == grad.data_ptr()
    _check_grad(grad, want + before.double(), size + before.double().abs(), count, dtype)
    assert torch.equal(grad[count == 0], before[count == 0])  # rows that no id names keep their bits


@pytest.mark.gpu
def test_padding_rows_may_hold_anything():
    n, V, D = 500, 60, 48
    ids = _ids(n, V, "mixed", 8)
    dout = _normal((n, D), "float32", 9)
    m = EmbeddingLookupGradhip()
    m.build([placeholder((V, D)), placeholder((n,), "int32")])
    want = m.run([ids, dout]).tensor.clone()
    pad = (ids < 0) | (ids >= V)
    dout[pad] = float("nan")
    assert torch.equal(m.run([ids, dout]).tensor, want)


@pytest.mark.gpu
def test_operands_off_their_alignment():
    n, V, D = 300, 64, 32
    for dtype in TYPES:
        flat, ids = _normal((V * D + 1,), dtype, 10), _ids(n, V, "mixed", 11)
        table = flat[1:].view(V, D)                            # contiguous, one element behind a 16-byte border
        m = EmbeddingLookuphip(1.0)
        m.build([placeholder((V, D), dtype), placeholder((n,), "int32")])
        got = m.run([table, ids]).tensor
        ok = (ids >= 0) & (ids < V)
        assert torch.equal(got[ok], table[ids[ok].long()])
        dflat = _normal((n * D + 1,), dtype, 12)
        g = EmbeddingLookupGradhip(1.0)
        g.build([placeholder((V, D), dtype), placeholder((n,), "int32")])
        want = g.run([ids, dflat[1:].view(n, D).clone()]).tensor.clone()
        assert torch.equal(g.run([ids, dflat[1:].view(n, D)]).tensor, want)


@pytest.mark.gpu
def test_gradient_is_the_lookups_adjoint():
    """<lookup(T), C> is linear in T: its derivative along E is <lookup(E), C> = <E, grad(C)>."""
    n, V, D = 700, 90, 20
    ids, C, E = _ids(n, V, "mixed", 13), _normal((n, D), "float32", 14), _normal((V, D), "float32", 15)
    f, g = EmbeddingLookuphip(1.5), EmbeddingLookupGradhip(1.5)
    ph = [placeholder((V, D)), placeholder((n,), "int32")]
    f.build(ph), g.build(ph)
    left = (f.run([E, ids]).tensor.double() * C.double()).sum()
    right = (g.run([ids, C]).tensor.double() * E.double()).sum()
    size = (f.out_tvm.tensor.double() * C.double()).abs().sum()
    assert abs(float(left - right)) <= 60 * 2.0 ** -24 * float(size)   # at most about 25 terms a row, both sides rounded


@pytest.mark.gpu
def test_replay_from_a_graph_and_on_another_stream():
    n, V, D = 9000, 500, 32
    ids, dout, table = _ids(n, V, "power", 16), _normal((n, D), "bfloat16", 17), _normal((V, D), "bfloat16", 18)
    ph = [placeholder((V, D), "bfloat16"), placeholder((n,), "int32")]
    f, g = EmbeddingLookuphip(0.5), EmbeddingLookupGradhip(0.5)
    f.build(ph), g.build(ph)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f.run([table, ids]), g.run([ids, dout])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f.run([table, ids]), g.run([ids, dout])
    for step in range(3):
        ids.copy_(_ids(n, V, "mixed", 20 + step))
        dout.copy_(_normal((n, D), "bfloat16", 30 + step))
        graph.replay()
        torch.cuda.synchronize()
        a, b = f.out_tvm.tensor.clone(), g.out_tvm.tensor.clone()
        assert torch.equal(a, f.run([table, ids]).tensor) and torch.equal(b, g.run([ids, dout]).tensor)


@pytest.mark.gpu
def test_refusals():
    ph = [placeholder((10, 4)), placeholder((6,), "int32")]
    table, ids, dout = _normal((10, 4), "float32", 1), _ids(6, 10, "mixed", 1), _normal((6, 4), "float32", 2)
    m = EmbeddingLookuphip()
    with pytest.raises(RuntimeError):
        m.run([table, ids])
    for bad in ([placeholder((10, 4), "float64"), ph[1]], [ph[0], placeholder((6,), "float32")]):
        with pytest.raises(TypeError):
            m.build(bad)
    for bad in ([placeholder((10,)), ph[1]], [placeholder((0, 4)), ph[1]], [placeholder((2 ** 31, 4)), ph[1]], ph[:1]):
        with pytest.raises(ValueError):
            m.build(bad)
    m.build(ph)
    for bad in ([table[:9], ids], [table, ids[:5]], [table.cpu(), ids], [table], [table.t().contiguous().t(), ids]):
        with pytest.raises(ValueError):
            m.run(bad)
    for bad in ([table.half(), ids], [table, ids.long()]):
        with pytest.raises(TypeError):
            m.run(bad)
    g = EmbeddingLookupGradhip()
    g.build(ph)
    with pytest.raises(ValueError):
        g.run([ids, dout, table[:5]])
    whole = _normal((16, 4), "float32", 3)
    with pytest.raises(ValueError):
        g.run([ids, whole[8:14], whole[:10]])                  # the gradient overlaps what is added to it
    with pytest.raises(ValueError):
        same = EmbeddingLookuphip()
        same.build([placeholder((6, 4)), placeholder((6,), "int32")])
        same.run([same.out_tvm, ids])


def test_bad_arguments_of_the_entry_points_without_a_device():
    L = _lib.lib()
    need = ctypes.c_int64(0)
    assert L.fg_embedding_lookup(0, 4, 1, 8, 8, 8, 1.0, 0, 0, None) == -1
    assert L.fg_embedding_lookup(2 ** 31, 4, 1, 8, 8, 8, 1.0, 0, 0, None) == -1
    assert L.fg_embedding_lookup(4, 0, 1, 8, 8, 8, 1.0, 0, 0, None) == -1
    assert L.fg_embedding_lookup(4, 4, -1, 8, 8, 8, 1.0, 0, 0, None) == -1
    assert L.fg_embedding_lookup(4, 4, 1, 8, 8, 8, 1.0, 3, 0, None) == -1       # no such element type
    assert L.fg_embedding_lookup(4, 4, 1, 8, 8, 8, 1.0, 0, 2, None) == -1       # no such index type
    assert L.fg_embedding_lookup(4, 4, 1, None, 8, 8, 1.0, 0, 0, None) == -1
    assert L.fg_embedding_lookup(4, 4, 0, None, None, None, 1.0, 0, 0, None) == 0
    assert L.fg_embedding_grad_workspace(4, 4, 100, None) == -1
    assert L.fg_embedding_grad_workspace(4, 4, 100, ctypes.byref(need)) == 0 and need.value > 0
    small, big = need.value, ctypes.c_int64(0)
    assert L.fg_embedding_grad_workspace(4, 4, 100000, ctypes.byref(big)) == 0 and big.value > small
    assert L.fg_embedding_grad(4, 4, 100, 8, 8, 8, 1.0, 0, 0, 0, 256, small - 1, None) == -1
    assert b"workspace" in L.fg_last_error()
    assert L.fg_embedding_grad(4, 4, 100, 8, 8, 8, 1.0, 0, 0, 0, 264, small, None) == -1   # not at a multiple of 256
    assert L.fg_embedding_grad(4, 4, 100, 8, None, 8, 1.0, 0, 0, 0, 256, small, None) == -1
    assert L.fg_embedding_grad(4, 4, 0, None, None, None, 1.0, 1, 0, 0, None, 0, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("V,D", [(40000, 3), (40000, 8), (9001, 5), (700, 33), (700, 32), (63, 1), (1, 7)])
@pytest.mark.parametrize("offset", [0, 1])
def test_absent_rows_become_zeros_and_nothing_beside_them(dtype, V, D, offset):
    """Rows that no id names, alone, in pairs and in long ranges, of a gradient that begins `offset` elements past an
    aligned address, between guards.  Every id is named once, so each sum is one element and the result exact."""
    L = _lib.lib()
    t = getattr(torch, dtype)
    patterns = [torch.tensor([V // 2]), torch.arange(0, V, 2), torch.arange(0, V, 3), torch.arange(max(1, V - 70)),
                torch.tensor([0, V - 1][:V]), torch.arange(V)]
    for pattern in patterns:
        ids = pattern.to("cuda", torch.int32)
        n = ids.numel()
        dout = torch.arange(1, n * D + 1, device="cuda").remainder(97).add(1).to(t).reshape(n, D)
        buf = torch.full((offset + V * D + 24,), float("nan"), device="cuda", dtype=t)
        need = ctypes.c_int64(0)
        assert L.fg_embedding_grad_workspace(V, D, n, ctypes.byref(need)) == 0
        space = torch.empty(need.value, dtype=torch.uint8, device="cuda")
        grad = buf[offset:offset + V * D]
        assert L.fg_embedding_grad(V, D, n, ids.data_ptr(), dout.data_ptr(), grad.data_ptr(), 1.0, 0,
                                   {"float32": 0, "float16": 2}[dtype], 0, space.data_ptr(), need.value,
                                   torch.cuda.current_stream().cuda_stream) == 0
        want = torch.zeros(V, D, device="cuda", dtype=t)
        want[ids.long()] = dout
        assert torch.equal(grad.reshape(V, D), want)
        assert buf[:offset].isnan().all() and buf[offset + V * D:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("n", [12287, 12288, 12289, 12353])
@pytest.mark.parametrize("V", [1, 500, 70000])
def test_gradient_around_the_border_of_the_two_sorts(n, V, index):
    """Whole numbers below 2^24 in every sum, so that float32 holds each exactly whatever the order."""
    rng = np.random.default_rng(n + V)
    ids = rng.integers(-1, V, n)
    dout = rng.integers(-8, 9, (n, 3)).astype(np.float32)
    g = EmbeddingLookupGradhip()
    g.build([placeholder((V, 3)), placeholder((n,), index)])
    got = g.run([torch.from_numpy(ids).to("cuda", getattr(torch, index)), torch.from_numpy(dout).cuda()]).asnumpy()
    want = np.zeros((V, 3), np.float64)
    np.add.at(want, ids[ids >= 0], dout[ids >= 0])
    assert np.array_equal(got, want.astype(np.float32))


@pytest.mark.gpu
def test_more_ids_than_one_launch_has_threads_for():
    """2^28 rows of 33 float16 take 16 threads each, 2^32 together, which is more than a launch may have."""
    n, V, D = 2 ** 28 + 5, 7, 33
    ids = torch.arange(n, dtype=torch.int32, device="cuda") % 9 - 1            # -1, 0 .. 6 and 7: padding on both sides
    table = _normal((V, D), "float16", 1)
    m = EmbeddingLookuphip(0.5)
    m.build([placeholder((V, D), "float16"), placeholder((n,), "int32")])
    m.out_tvm.tensor.fill_(float("nan"))
    out = m.run([table, ids]).tensor
    rows = torch.zeros(V + 2, D, dtype=torch.float16, device="cuda")
    rows[1:V + 1] = table * 0.5                                                 # exact: no value is below 2^-13
    assert float(table.abs().min()) >= 2.0 ** -13
    step = 9 << 20
    want = rows.repeat(step // 9, 1)
    for at in range(0, n, step):
        assert torch.equal(out[at:at + step], want[:min(step, n - at)])
