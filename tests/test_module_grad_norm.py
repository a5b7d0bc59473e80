"""Global norm and clipping against 64-bit sums.  The squares of float32 values are exact in float64 and their sum is
off by at most (terms) * 2^-53 of itself, so the float32 norm is off by half a step, 2^-24 (plus that); the coefficient
is rounded to float32 once, the product once to float32 and once to the element type."""
import ctypes

import pytest
import torch

from featgraph_amd import _lib, placeholder
from featgraph_amd.module import ClipGradNormhip, GradNormhip

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}

LISTS = [
    [((1,), "float32")],
    [((3, 5), "bfloat16"), ((7,), "float32"), ((), "float16")],
    [((64, 64), "float32")] * 6,
    [((4097,), "float32"), ((0,), "float32"), ((8193,), "bfloat16"), ((0, 3), "float16"), ((123457,), "float16")],
    [((1000003,), "float32"), ((17,), "float32"), ((300, 300), "bfloat16")],
    [((11 + i,), list(TYPES)[i % 3]) for i in range(97)],
    [((5000 + i,), list(TYPES)[i % 3]) for i in range(260)],
    [((3000001,), "bfloat16"), ((2000003,), "float16"), ((5,), "float32")],
]


def _make(spec, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale * 3.0 ** -(i % 4)).to(TYPES[d]).cuda() for i, (s, d) in enumerate(spec)]


def _norm(tensors):
    return sum(float((t.double() ** 2).sum()) for t in tensors) ** 0.5


def _check(got, grads, c):
    for y, x in zip(got, grads):
        want = x.double() * c
        tol = want.abs() * (3 * 2.0 ** -24 + HALF_STEP[x.dtype]) + TINY[x.dtype]
        assert y.dtype == x.dtype and y.shape == x.shape and bool(((y.double() - want).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("spec", LISTS, ids=[str(i) for i in range(len(LISTS))])
def test_norm_and_clip(spec):
    grads = _make(spec, 1)
    ph = [placeholder(s, d) for s, d in spec]
    want = _norm(grads)
    norm = GradNormhip()
    norm.build(ph)
    assert abs(float(norm.run(grads).tensor) - want) <= 1.01 * 2.0 ** -24 * want
    for max_norm in (want / 3, want * 2):
        m = ClipGradNormhip(max_norm)
        m.build(ph)
        got_norm, clipped = m.run(grads)
        assert got_norm.shape == () and abs(float(got_norm.tensor) - want) <= 1.01 * 2.0 ** -24 * want
        c = min(1.0, max_norm / (want + 1e-6))
        _check([y.tensor for y in clipped], grads, c)
        if c == 1.0:
            assert all(torch.equal(y.tensor, x) for y, x in zip(clipped, grads))
        first = [y.tensor.clone() for y in clipped]
        assert all(torch.equal(a, y.tensor) for a, y in zip(first, m.run(grads)[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("spec", LISTS[1:], ids=[str(i) for i in range(1, len(LISTS))])
def test_in_place(spec):
    grads = _make(spec, 2)
    kept = [g.clone() for g in grads]
    want = _norm(grads)
    m = ClipGradNormhip(want / 2)
    m.build([placeholder(s, d) for s, d in spec], {"in_place": True})
    _, out = m.run(grads)
    assert all(o.tensor.data_ptr() == g.data_ptr() for o, g in zip(out, grads))
    _check(grads, kept, 0.5 * want / (want + 1e-6))
    still = [g.clone() for g in grads]
    n = ClipGradNormhip(want)                                   # below the limit now: nothing changes
    n.build([placeholder(s, d) for s, d in spec], {"in_place": True})
    n.run(grads)
    assert all(torch.equal(a, b) for a, b in zip(still, grads))


@pytest.mark.gpu
def test_values_whose_squares_leave_float32():
    big = torch.full((5000,), 2.0 ** 100, device="cuda")
    small = torch.full((300,), 2.0 ** -100, device="cuda")
    m = ClipGradNormhip(1.0)
    m.build([placeholder((5000,)), placeholder((300,))])
    norm, (a, b) = m.run([big, small])
    want = 5000 ** 0.5 * 2.0 ** 100
    assert abs(float(norm.tensor) - want) <= 1.01 * 2.0 ** -24 * want
    _check([a.tensor], [big], 1.0 / want)
    s = GradNormhip()
    s.build([placeholder((300,))])
    want = 300 ** 0.5 * 2.0 ** -100
    assert abs(float(s.run([small]).tensor) - want) <= 1.01 * 2.0 ** -24 * want


@pytest.mark.gpu
def test_norms_that_are_no_number_zero_or_infinite():
    ph = [placeholder((40,)), placeholder((20000,))]
    m = ClipGradNormhip(1.0)
    m.build(ph)
    x, y = torch.ones(40, device="cuda"), torch.ones(20000, device="cuda")
    x[3] = float("nan")
    norm, out = m.run([x, y])
    assert torch.isnan(norm.tensor) and all(bool(torch.isnan(o.tensor).all()) for o in out)
    x[3] = float("inf")
    norm, out = m.run([x, y])
    assert float(norm.tensor) == float("inf") and not out[1].tensor.any() and bool(torch.isnan(out[0].tensor[3]))
    norm, out = m.run([torch.zeros_like(x), torch.zeros_like(y)])
    assert float(norm.tensor) == 0.0 and not any(o.tensor.any() for o in out)
    none = ClipGradNormhip(1.0)
    none.build([])
    assert float(none.run([])[0].tensor) == 0.0
    empty = ClipGradNormhip(1.0)
    empty.build([placeholder((0,))])
    assert float(empty.run([x[:0]])[0].tensor) == 0.0


@pytest.mark.gpu
def test_tensors_off_their_alignment():
    flat = _make([((30001,), "float32"), ((30001,), "bfloat16")], 3)
    views = [f[1:] for f in flat]
    m = ClipGradNormhip(1.0)
    m.build([placeholder((30000,)), placeholder((30000,), "bfloat16")])
    norm, out = m.run(views)
    want = _norm(views)
    assert abs(float(norm.tensor) - want) <= 1.01 * 2.0 ** -24 * want
    _check([o.tensor for o in out], views, 1.0 / (want + 1e-6))
    before = [f[0].clone() for f in flat]
    place = ClipGradNormhip(1.0)
    place.build([placeholder((30000,)), placeholder((30000,), "bfloat16")], {"in_place": True})
    place.run(views)
    assert all(torch.equal(v, o.tensor) for v, o in zip(views, out)) and all(bool(f[0] == b) for f, b in zip(flat, before))


@pytest.mark.gpu
@pytest.mark.parametrize("spec", [LISTS[2], LISTS[6]], ids=["one launch", "many"])
def test_replay_from_a_graph(spec):
    grads = _make(spec, 4)
    m = ClipGradNormhip(1.0)
    m.build([placeholder(s, d) for s, d in spec])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.run(grads)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.run(grads)
    for step in range(3):
        for g, new in zip(grads, _make(spec, 5 + step)):
            g.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        norm, out = m._norm.tensor.clone(), [o.tensor.clone() for o in m._clipped]
        again, eager = m.run(grads)
        assert torch.equal(norm, again.tensor) and all(torch.equal(a, b.tensor) for a, b in zip(out, eager))


@pytest.mark.gpu
def test_refusals():
    x = torch.ones(64, device="cuda")
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            ClipGradNormhip(bad)
    m = ClipGradNormhip(1.0)
    with pytest.raises(RuntimeError):
        m.run([x])
    with pytest.raises(TypeError):
        m.build([placeholder((64,), "float64")])
    with pytest.raises(TypeError):
        m.build([placeholder((64,))], {"inplace": True})
    m.build([placeholder((64,))])
    for bad in ([x[:63]], [x, x], [x.cpu()], [torch.ones(128, device="cuda")[::2]], [m._clipped[0]]):
        with pytest.raises(ValueError):
            m.run(bad)
    with pytest.raises(TypeError):
        m.run([x.half()])
    two = ClipGradNormhip(1.0)
    two.build([placeholder((40,)), placeholder((40,))], {"in_place": True})
    with pytest.raises(ValueError):
        two.run([x[:40], x[24:]])
    two.run([x[:24].repeat(2)[:40], x[:40]])


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
def test_the_norm_is_no_gradient_of_the_same_call(in_place):
    m = ClipGradNormhip(1.0)
    m.build([placeholder((1,)), placeholder((8,))], {"in_place": in_place})
    x = torch.ones(8, device="cuda")
    norm, _ = m.run([torch.ones(1, device="cuda"), x])
    assert float(norm.tensor) == 3.0
    with pytest.raises(ValueError):
        m.run([norm.tensor.reshape(1), x])


def test_bad_arguments_of_the_entry_points_without_a_device():
    L = _lib.lib()
    need = ctypes.c_int64(0)
    assert L.fg_grad_norm_workspace(None) == -1
    assert L.fg_grad_norm_workspace(ctypes.byref(need)) == 0 and need.value > 0
    t = (_lib.Tensor * 1)()
    t[0].n, t[0].dtype, t[0].data, t[0].out = 4, 0, 16, 16
    assert L.fg_grad_norm(-1, t, 16, 256, need.value, None) == -1
    assert L.fg_grad_norm(1, None, 16, 256, need.value, None) == -1
    assert L.fg_grad_norm(1, t, None, 256, need.value, None) == -1
    assert L.fg_grad_norm(1, t, 16, 256, need.value - 1, None) == -1
    assert L.fg_grad_norm(1, t, 16, 264, need.value, None) == -1
    assert L.fg_grad_clip(1, t, -1.0, 0.0, 16, 256, need.value, None) == -1
    assert L.fg_grad_clip(1, t, float("nan"), 0.0, 16, 256, need.value, None) == -1
    t[0].dtype = 3
    assert L.fg_grad_norm(1, t, 16, 256, need.value, None) == -1
    t[0].dtype, t[0].out = 0, None
    assert L.fg_grad_clip(1, t, 1.0, 0.0, 16, 256, need.value, None) == -1
    t[0].n = -1
    assert L.fg_grad_norm(1, t, 16, 256, need.value, None) == -1
