"""Linear softmax cross entropy and its gradients against the formulas in 64 bits.

Tolerances.  A sum of K float32 terms on the device differs from the exact one by K roundings, each at most half a
step (2^-24) of a partial sum, which A = the sum of the terms' sizes bounds; roundings are of random sign, and six
standard deviations of K of them are 6 * sqrt(K / 3) * 2^-24 * A < 4 * sqrt(K) * 2^-24 * A.  sums(K) below is that with
room for the few roundings of partial joins; float32 operands, split into two float16 parts (each element to 2^-23 of
itself), add 3 K products and leave out one of 2^-24 A at most.  A logit off by d moves exp by a factor 1 + d, lse by at most the largest d of its
row, and G by |dloss| p (d + d_lse); exp2 of a product rounds its argument (|l - lse| 2^-23).  bfloat16 operands round G
to bfloat16 (half a step, 2^-8), and the results are rounded to their type (half a step)."""
import ctypes
import math

import pytest
import torch

from featgraph_amd import _lib, placeholder
from featgraph_amd.module import LinearCrossEntropyGradhip, LinearCrossEntropyhip

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}
TINY = 2.0 ** -126


def _operands(dtype, N, V, D, seed, spread=1.5, itype="int32", ignored=0.1):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(N, D, generator=g).to(TYPES[dtype]).cuda()
    w = (torch.randn(V, D, generator=g) * (spread / math.sqrt(D))).to(TYPES[dtype]).cuda()
    y = torch.randint(0, V, (N,), generator=g)
    if N:
        y[0] = V - 1
    if N > 3:
        y[torch.rand(N, generator=g) < ignored] = -1
        y[2] = V                                             # one past the last class: ignored as well
        y[1] = 0
    dl = (0.5 + torch.rand(N, generator=g)).cuda() / max(N, 1)
    return h, w, y.to(getattr(torch, itype)).cuda(), dl


def _sums(K, dtype):
    return (8 + 4 * math.sqrt(K * (3 if dtype == "float32" else 1)) + (5 if dtype == "float32" else 0)) * 2.0 ** -24


def _reference(h, w, y, dl, dtype, loss, lse, dh, dw):
    """Checks the four results against 64 bits."""
    N, D = h.shape
    V = w.shape[0]
    H, W = h.double(), w.double()
    logits, size = H @ W.T, H.abs() @ W.abs().T
    d = (_sums(D, dtype) * size).amax(1)                      # of every logit of the row
    want = torch.logsumexp(logits, 1)
    far = (logits - want[:, None]).abs().amax(1)
    d_lse = d + (far * 2.0 ** -23 + 2.0 ** -21) + _sums(V, "bfloat16") + 2.0 ** -23 * want.abs()
    assert bool(((lse.double() - want).abs() <= d_lse).all())
    ok = (y >= 0) & (y < V)
    n = torch.arange(N, device="cuda")[ok]
    at = y[ok].long()
    want_loss = torch.zeros_like(want)
    want_loss[ok] = want[ok] - logits[n, at]
    tol = d_lse + d + 2.0 ** -23 * want_loss.abs()
    assert bool(((loss.double() - want_loss).abs() <= tol).all()) and not loss[~ok].any()
    if dh is None:
        return
    p = torch.exp(logits - want[:, None])
    f = torch.where(ok, dl.double(), 0.0)[:, None]
    G = p * f
    G[n, at] -= dl.double()[ok]
    off = f * (p * (d + d_lse + far * 2.0 ** -23 + 2.0 ** -21)[:, None] + 2.0 ** -22 * (p + 0.0))
    off[n, at] += 2.0 ** -22 * dl.double()[ok]
    rounding = 2.0 ** -8 if dtype == "bfloat16" else 2 * 2.0 ** -23      # of both factors, where those are split
    floor = 2.0 ** -50 if dtype == "float32" else 0.0
    off = off + floor * f
    for got, a, b, K, e in ((dh, G, W, V, off), (dw, G.T, H, N, off.T)):
        exact = a @ b
        tol = (e + (rounding + _sums(K, dtype)) * a.abs()) @ b.abs() + floor * (a.abs() @ b.abs().amax().expand(b.shape)) + HALF_STEP[dtype] * exact.abs() * 1.01 + TINY
        assert bool(((got.double() - exact).abs() <= tol).all())
    assert not dh[~ok].any()


def _run(h, w, y, dl, dtype, itype="int32"):
    ph = [placeholder(tuple(h.shape), dtype), placeholder(tuple(w.shape), dtype), placeholder(tuple(y.shape), itype)]
    f, g = LinearCrossEntropyhip(), LinearCrossEntropyGradhip()
    f.build(ph), g.build(ph)
    loss, lse = f.run([h, w, y])
    g._dhidden.tensor.fill_(float("nan")), g._dweight.tensor.fill_(float("nan"))
    dh, dw = g.run([h, w, y, lse, dl])
    return loss.tensor, lse.tensor, dh.tensor, dw.tensor


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (5, 3, 2), (64, 41, 64), (127, 255, 100), (33, 300, 64), (300, 70, 130),
                                   (257, 1025, 192), (70, 5000, 72), (1000, 41, 256), (20, 30001, 40), (1, 4096, 64),
                                   (2049, 513, 24), (9, 1, 5), (20, 50, 600), (17, 40, 1100)])
def test_loss_and_gradients(dtype, N, V, D):
    itype = "int64" if N % 2 else "int32"
    h, w, y, dl = _operands(dtype, N, V, D, N + V + D, itype=itype)
    loss, lse, dh, dw = _run(h, w, y, dl, dtype, itype)
    assert loss.dtype == lse.dtype == torch.float32 and dh.dtype == dw.dtype == TYPES[dtype]
    _reference(h, w, y, dl, dtype, loss, lse, dh, dw)


@pytest.fixture
def config():
    yield _lib.config_set
    _lib.config_set("ce.tile", 0)
    _lib.config_set("ce.piece_rows", 0)
    _lib.config_set("ce.native", -1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tile", [1, 2, 3, 4])
@pytest.mark.parametrize("N,V,D,piece", [(300, 700, 192, 0), (300, 700, 192, 256), (65, 1300, 70, 512), (600, 257, 128, 256)])
def test_every_tile_and_pieces_of_the_vocabulary(config, dtype, tile, N, V, D, piece):
    config("ce.tile", tile)
    config("ce.piece_rows", piece)
    h, w, y, dl = _operands(dtype, N, V, D, tile + N)
    first = _run(h, w, y, dl, dtype)
    _reference(h, w, y, dl, dtype, *first)
    assert all(torch.equal(a, b) for a, b in zip(first, _run(h, w, y, dl, dtype)))      # the same bits again


@pytest.mark.gpu
@pytest.mark.parametrize("native", [0, 1])
@pytest.mark.parametrize("tile", [1, 2, 3, 4])
@pytest.mark.parametrize("N,V,D", [(70, 600, 1), (33, 300, 30), (257, 100, 33), (40, 1500, 64), (300, 41, 127), (5, 2000, 447)])
def test_float32_as_copies_and_as_it_is(config, native, tile, N, V, D):
    """Rows of every length modulo 16 bytes and 32 elements; rows of NaN between the others reach nothing but themselves."""
    config("ce.native", native)
    config("ce.tile", tile)
    h, w, y, dl = _operands("float32", N, V, D, tile + D, ignored=0.3)
    ph = [placeholder((N, D)), placeholder((V, D)), placeholder((N,), "int32")]
    f = LinearCrossEntropyhip()
    f.build(ph)
    loss, lse = (x.tensor.clone() for x in f.run([h, w, y]))
    _reference(h, w, y, dl, "float32", loss, lse, None, None)
    bad = (y < 0) | (y >= V)
    h[bad] = float("nan")
    loss2, lse2 = f.run([h, w, y])
    assert torch.equal(loss2.tensor, loss) and torch.equal(lse2.tensor[~bad], lse[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_steep_and_flat_logits(dtype):
    h, w, y, dl = _operands(dtype, 130, 500, 64, 3, spread=200.0)      # logits of hundreds: the softmax is a maximum
    _reference(h, w, y, dl, dtype, *_run(h, w, y, dl, dtype))
    h.zero_()                                                          # all logits 0: lse = log V, G = 1 / V
    loss, lse, dh, dw = _run(h, w, y, dl, dtype)
    assert bool(((lse.double() - math.log(500)).abs() <= 2.0 ** -20).all())
    _reference(h, w, y, dl, dtype, loss, lse, dh, dw)


@pytest.mark.gpu
def test_the_smallest_and_largest_values():
    """float32 operands near the ends of the range: leading parts that would round to infinity are cut instead.  The
    weights are powers of two, so that every part of every product is a normal number."""
    h = torch.zeros(4, 8, device="cuda")
    w = torch.zeros(5, 8, device="cuda")
    h[0, 0], w[1, 0] = 3.4e38, 2.0 ** -125
    h[1, 1], w[2, 1] = 1.2345678 * 2.0 ** -100, 2.0 ** 102
    h[2, 2], w[3, 2] = -torch.finfo(torch.float32).max, 2.0 ** -126
    y = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    loss, lse, _, _ = _run(h, w, y, torch.ones(4, device="cuda"), "float32")
    logits = h.double() @ w.double().T
    want = torch.logsumexp(logits, 1)
    tol = 40 * 2.0 ** -24 * (logits.abs().amax(1) + 4)                  # a dozen roundings of values up to the logit, exp, log
    assert bool(((lse.double() - want).abs() <= tol).all())
    at = logits[torch.arange(4, device="cuda"), y.long()]
    assert bool(((loss.double() - (want - at)).abs() <= 2 * tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_ignored_rows_may_hold_anything(dtype):
    h, w, y, dl = _operands(dtype, 200, 333, 96, 5, ignored=0.4)
    bad = (y < 0) | (y >= 333)
    ph = [placeholder((200, 96), dtype), placeholder((333, 96), dtype), placeholder((200,), "int32")]
    f, g = LinearCrossEntropyhip(), LinearCrossEntropyGradhip()
    f.build(ph), g.build(ph)
    loss, lse = (x.tensor.clone() for x in f.run([h, w, y]))
    dh, dw = (x.tensor.clone() for x in g.run([h, w, y, lse, dl]))
    h[bad] = float("nan")
    dl[bad] = float("inf")
    loss2, lse2 = f.run([h, w, y])
    assert torch.equal(loss2.tensor, loss) and torch.equal(lse2.tensor[~bad], lse[~bad])
    dh2, dw2 = g.run([h, w, y, lse2, dl])
    assert torch.equal(dh2.tensor, dh) and torch.equal(dw2.tensor, dw) and not dh2.tensor[bad].any()
    y.fill_(-1)                                                        # nothing left
    assert not f.run([h, w, y])[0].tensor.any()
    dh3, dw3 = g.run([h, w, y, lse2, dl])
    assert not dh3.tensor.any() and not dw3.tensor.any()


@pytest.mark.gpu
def test_gradient_against_differences():
    """(L(x + e u) - L(x - e u)) / 2e for the summed loss L along a direction u.  Along it every logit moves linearly
    (in h) with slope s; the third derivative of lse is at most 2 * max |s|^3 (a third cumulant of a variable within
    [-max, max] is below 2 max^3), so the difference is off by e^2 / 6 of that, plus the losses' own error over e."""
    N, V, D = 64, 300, 48
    h, w, y, dl = _operands("float32", N, V, D, 7)
    ph = [placeholder((N, D)), placeholder((V, D)), placeholder((N,), "int32")]
    f, g = LinearCrossEntropyhip(), LinearCrossEntropyGradhip()
    f.build(ph), g.build(ph)
    ok = (y >= 0) & (y < V)
    _, lse = f.run([h, w, y])
    dh, dw = (x.tensor.double().clone() for x in g.run([h, w, y, lse, dl]))
    gen = torch.Generator().manual_seed(8)
    loss_error = 4 * float((_sums(D, "float32") * (h.double().abs() @ w.double().abs().T)).max()) + 2.0 ** -18
    for which in (0, 1):
        u = torch.randn(*(h, w)[which].shape, generator=gen).cuda() / math.sqrt(D)
        slopes = (u.double() @ w.double().T) if which == 0 else (h.double() @ u.double().T)
        e = 1.0 / 64
        sides = []
        for sign in (1, -1):
            x = [h, w]
            x[which] = x[which] + sign * e * u
            sides.append((f.run([x[0], x[1], y])[0].tensor.double() * dl.double())[ok].sum())
            real = (x[which] - (h, w)[which]).double()
            sides[-1] = (sides[-1], real)
        step = (sides[0][1] - sides[1][1])                              # what the sums in float32 really moved by
        want = float((step * (dh, dw)[which]).sum())
        got = float(sides[0][0] - sides[1][0])
        total = float(dl[ok].sum())
        bound = total * (2 * loss_error + e ** 3 / 3 * 2 * float(slopes.abs().max()) ** 3)
        assert abs(got - want) <= bound and abs(want) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_operands_off_their_alignment(dtype):
    N, V, D = 70, 200, 128
    h, w, y, dl = _operands(dtype, N, V, D, 9)
    fh, fw = torch.zeros(N * D + 1, dtype=h.dtype, device="cuda"), torch.zeros(V * D + 1, dtype=h.dtype, device="cuda")
    fh[1:], fw[1:] = h.reshape(-1), w.reshape(-1)
    _reference(h, w, y, dl, dtype, *_run(fh[1:].view(N, D), fw[1:].view(V, D), y, dl, dtype))


@pytest.mark.gpu
def test_no_rows():
    h, w, y, dl = _operands("bfloat16", 0, 50, 16, 10)
    loss, lse, dh, dw = _run(h, w, y, dl, "bfloat16")
    assert loss.shape == lse.shape == (0,) and dh.shape == (0, 16) and not dw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_replay_from_a_graph(config, dtype):
    N, V, D = 200, 900, 80
    config("ce.piece_rows", 512)
    h, w, y, dl = _operands(dtype, N, V, D, 11)
    ph = [placeholder((N, D), dtype), placeholder((V, D), dtype), placeholder((N,), "int32")]
    f, g = LinearCrossEntropyhip(), LinearCrossEntropyGradhip()
    f.build(ph), g.build(ph)

    def step():
        loss, lse = f.run([h, w, y])
        return (loss, lse) + tuple(g.run([h, w, y, lse, dl]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        for x, new in zip((h, w, y, dl), _operands(dtype, N, V, D, 20 + k)):
            x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.tensor.clone() for o in out]
        assert all(torch.equal(a, b.tensor) for a, b in zip(got, step()))
        _reference(h, w, y, dl, dtype, *got)


@pytest.mark.gpu
def test_refusals():
    ph = [placeholder((6, 8)), placeholder((10, 8)), placeholder((6,), "int32")]
    m = LinearCrossEntropyhip()
    h, w, y, dl = _operands("float32", 6, 10, 8, 12)
    with pytest.raises(RuntimeError):
        m.run([h, w, y])
    for bad in ([placeholder((6, 8), "float16"), placeholder((10, 8), "float16"), ph[2]],
                [ph[0], placeholder((10, 8), "bfloat16"), ph[2]], [ph[0], ph[1], placeholder((6,), "float32")]):
        with pytest.raises(TypeError):
            m.build(bad)
    for bad in ([ph[0], placeholder((10, 9)), ph[2]], [ph[0], ph[1], placeholder((5,), "int32")], ph[:2],
                [ph[0], placeholder((0, 8)), ph[2]], [placeholder((2 ** 23, 8)), ph[1], placeholder((2 ** 23,), "int32")]):
        with pytest.raises(ValueError):
            m.build(bad)
    m.build(ph)
    for bad in ([h[:5], w, y], [h, w[:9], y], [h, w], [h.cpu(), w, y], [h, w.t().contiguous().t(), y]):
        with pytest.raises(ValueError):
            m.run(bad)
    for bad in ([h.bfloat16(), w, y], [h, w, y.long()]):
        with pytest.raises(TypeError):
            m.run(bad)
    g = LinearCrossEntropyGradhip()
    g.build(ph)
    _, lse = m.run([h, w, y])
    with pytest.raises(ValueError):
        g.run([h, w, y, lse])
    with pytest.raises(ValueError):
        g.run([g._dhidden, w, y, lse, dl])                              # an output as an operand
    with pytest.raises(TypeError):
        g.run([h, w, y, lse.tensor.double(), dl])


def test_bad_arguments_of_the_entry_points_without_a_device():
    L = _lib.lib()
    need = ctypes.c_int64(0)
    for sizes in ((-1, 4, 4), (4, 0, 4), (4, 4, 0), (2 ** 23, 4, 4), (4, 2 ** 31, 4), (4, 4, 2 ** 17)):
        assert L.fg_linear_ce_workspace(*sizes, 0, ctypes.byref(need)) == -1
        assert L.fg_linear_ce(*sizes, 16, 16, 16, 16, 16, 0, 0, 256, 1 << 40, None) == -1
        assert L.fg_linear_ce_grad(*sizes, 16, 16, 16, 16, 16, 16, 16, 0, 0, 256, 1 << 40, None) == -1
    assert L.fg_linear_ce_workspace(4, 4, 4, 2, ctypes.byref(need)) == -4               # float16
    assert L.fg_linear_ce_workspace(4, 4, 4, 0, None) == -1
    assert L.fg_linear_ce_workspace(4, 4, 4, 0, ctypes.byref(need)) == 0 and need.value > 0
    assert L.fg_linear_ce(4, 4, 4, 16, 16, 16, 16, 16, 0, 2, 256, need.value, None) == -1        # no such index type
    assert L.fg_linear_ce(4, 4, 4, 16, None, 16, 16, 16, 0, 0, 256, need.value, None) == -1
    assert L.fg_linear_ce(4, 4, 4, 16, 16, 16, 16, 16, 0, 0, 256, 16, None) == -1                # workspace too small
    assert b"workspace" in L.fg_last_error()
    assert L.fg_linear_ce(0, 4, 4, None, None, None, None, None, 0, 0, None, 0, None) == 0
    assert L.fg_linear_ce_grad_workspace(4, 4, 4, 0, ctypes.byref(need)) == 0
    assert L.fg_linear_ce_grad(4, 4, 4, 16, 16, 16, 16, None, 16, 16, 0, 0, 256, need.value, None) == -1
    assert L.fg_linear_ce_grad(4, 4, 4, 16, 16, 16, 16, 16, 16, 16, 0, 0, 264, need.value, None) == -1


@pytest.mark.parametrize("dtype", [0, 1])
def test_pieces_stay_within_32_bit_offsets(dtype):
    """The kernels reach 2^22 vocabulary rows of a piece with 32-bit offsets: a larger wish gives pieces of that size."""
    L = _lib.lib()
    sizes = []
    try:
        for rows in (2 ** 22, 2 ** 22 + 1, 2 ** 30, 2 ** 31 - 1):
            _lib.config_set("ce.piece_rows", rows)
            need = ctypes.c_int64(0)
            assert L.fg_linear_ce_grad_workspace(64, 2 ** 24, 64, dtype, ctypes.byref(need)) == 0
            sizes.append(need.value)
    finally:
        _lib.config_set("ce.piece_rows", 0)
    assert len(set(sizes)) == 1, sizes


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [128, 67, 100])
@pytest.mark.parametrize("tile,piece", [(0, 0), (1, 256), (2, 256), (3, 512), (4, 256)])
def test_ignored_rows_in_every_path(dtype, D, tile, piece):
    """Operands read in place, padded and with rows of odd length; one piece and several; infinities beside NaN."""
    N, V = 150, 700
    h, w, y, dl = _operands(dtype, N, V, D, 11, ignored=0.3)
    bad = (y < 0) | (y >= V)
    try:
        _lib.config_set("ce.tile", tile)
        _lib.config_set("ce.piece_rows", piece)
        ph = [placeholder((N, D), dtype), placeholder((V, D), dtype), placeholder((N,), "int32")]
        f, g = LinearCrossEntropyhip(), LinearCrossEntropyGradhip()
        f.build(ph), g.build(ph)
        _, lse = (x.tensor.clone() for x in f.run([h, w, y]))
        dh, dw = (x.tensor.clone() for x in g.run([h, w, y, lse, dl]))
        assert bool(bad.any()) and dh.isfinite().all() and dw.isfinite().all()
        h[bad] = float("nan")
        h[bad, ::2] = float("inf")
        lse[bad], dl[bad] = float("nan"), float("-inf")
        loss2, _ = f.run([h, w, y])
        assert not loss2.tensor[bad].any() and loss2.tensor.isfinite().all()
        dh2, dw2 = g.run([h, w, y, lse, dl])
        assert torch.equal(dh2.tensor, dh) and torch.equal(dw2.tensor, dw) and not dh2.tensor[bad].any()
        w[5] = float("inf")                             # a class that spoils every row it meets, but not the ignored ones
        assert not g.run([h, w, y, lse, dl])[0].tensor[bad].any()
    finally:
        _lib.config_set("ce.tile", 0)
        _lib.config_set("ce.piece_rows", 0)


# One range of the vocabulary per workgroup, and as many ranges as there are tiles: the sums of exponentials are long.
LONG_RANGES = [("bfloat16", tile, 0, -1, 65536) for tile in (0, 1, 2, 3, 4)] + \
              [("float32", tile, 0, native, 65536) for tile in (1, 2, 3, 4) for native in (0, 1)] + \
              [(dtype, 0, 256, -1, 40) for dtype in TYPES]


@pytest.mark.gpu
@pytest.mark.parametrize("place", ["flat", "first", "last"])
@pytest.mark.parametrize("dtype,tile,piece,native,N", LONG_RANGES)
def test_sums_over_a_long_vocabulary(config, dtype, tile, piece, native, N, place):
    """232,965 classes of one logit c (whose exponential is no power of two), and the same with one class 17.75 above the
    others, whose term alone is larger than 2^24 of theirs: lse = c + log(V) and c + log(V - 1 + e^17.75).

    Sixteen terms are added one by one and four such sums together (18 roundings), the running sum is two floats that are
    put together once, halves of a wave and four waves make four more, exp2 is off by a step (2 halves), its argument by
    the rounding of log2(e) (1.4e-8 |l| log2(e), with |l| below 19 less than 5 halves) and its own (|argument| at most 1
    for the terms that count): below 32 * 2^-24 together.  The result is rounded to float32."""
    V, peak = 232965, 17.75
    config("ce.tile", tile)
    config("ce.piece_rows", piece)
    config("ce.native", native)
    h = torch.ones(N, 2, dtype=TYPES[dtype], device="cuda")
    h[:, 0] = 0.296875 + (torch.arange(N, device="cuda") % 8) / 16.0
    w = torch.zeros(V, 2, dtype=TYPES[dtype], device="cuda")
    w[:, 0] = 1.0
    at = V - 1 if place == "last" else 0
    w[at, 1] = 0.0 if place == "flat" else peak
    y = torch.full((N,), at, dtype=torch.int32, device="cuda")
    f = LinearCrossEntropyhip()
    f.build([placeholder((N, 2), dtype), placeholder((V, 2), dtype), placeholder((N,), "int32")])
    loss, lse = (x.tensor for x in f.run([h, w, y]))
    c = h[:, 0].double()
    top = math.exp(float(w[at, 1]))
    want = c + math.log(V - 1 + top)
    want_loss = torch.full_like(want, math.log(V - 1 + top) - float(w[at, 1]))
    tol = 32 * 2.0 ** -24 + 1.01 * 2.0 ** -24 * want
    assert bool(((lse.double() - want).abs() <= tol).all())
    assert bool(((loss.double() - want_loss).abs() <= tol + 2.0 ** -24 * want_loss).all())

    # the label's gradient, p - 1, of a few rows with the lse of all: p is off by p times the errors of lse, the logit's
    # and exp2's (16 * 2^-24), G and the result are rounded to the type or to two parts
    some = torch.arange(0, N, max(1, N // 40), device="cuda")
    g = LinearCrossEntropyGradhip()
    g.build([placeholder((some.numel(), 2), dtype), placeholder((V, 2), dtype), placeholder((some.numel(),), "int32")])
    dl = torch.ones(some.numel(), device="cuda")
    dh = g.run([h[some].contiguous(), w, y[some].contiguous(), lse[some].contiguous(), dl])[0].tensor
    exact = float(w[at, 1]) * (top / (V - 1 + top) - 1)
    off = float(w[at, 1]) * (tol[some] + 16 * 2.0 ** -24) + 4 * HALF_STEP[dtype] * abs(exact)
    assert bool(((dh[:, 1].double() - exact).abs() <= off).all())


@pytest.mark.parametrize("N,V,D", [(232965, 65536, 64), (65536, 232965, 128), (2 ** 22, 65536, 64), (2449029, 232965, 128)])
def test_workspace_of_the_loss_holds_what_the_kernels_write(N, V, D):
    """Beside the padded copies of operands off their alignment there are a reference and a sum for every row and range of
    the vocabulary.  With this many rows every workgroup slot of the device is busy several times over with a few ranges."""
    need = ctypes.c_int64(0)
    assert _lib.lib().fg_linear_ce_workspace(N, V, D, 1, ctypes.byref(need)) == 0
    copies = 2 * (N + V) * D + 2 * 256 * D                    # the piece of the vocabulary is a multiple of 256 rows
    assert need.value <= copies + 32 * 8 * N + 4096, (need.value - copies) / (8 * N)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tile,piece", [(0, 0), (1, 256), (2, 512), (3, 768), (4, 256)])
@pytest.mark.parametrize("N,V,D", [(5, 3000, 16), (300, 1025, 64), (2000, 70, 33), (1, 1, 1), (64, 20000, 128), (9000, 1300, 64)])
def test_nothing_is_written_behind_the_workspace(config, dtype, tile, piece, N, V, D):
    config("ce.tile", tile)
    config("ce.piece_rows", piece)
    h, w, y, dl = _operands(dtype, N, V, D, N + V)
    ph = [placeholder((N, D), dtype), placeholder((V, D), dtype), placeholder((N,), "int32")]
    f, g = LinearCrossEntropyhip(), LinearCrossEntropyGradhip()
    f.build(ph), g.build(ph)
    for m in (f, g):
        need, behind = m._space.numel(), 1 << 20
        m._space = torch.full((need + behind,), 0x5a, dtype=torch.uint8, device="cuda")
        if m is f:
            _, lse = m.run([h, w, y])
        else:
            m.run([h, w, y, lse, dl])
        assert bool((m._space[need:] == 0x5a).all())


@pytest.mark.gpu
@pytest.mark.parametrize("native", [0, 1])
@pytest.mark.parametrize("N,V,D", [(200, 300, 64), (37, 2001, 90), (1500, 41, 33)])
def test_float32_of_very_different_sizes(config, native, N, V, D):
    """The bound that the header states, where it is reached: features and row weights over ten decades, probabilities
    down to 1e-20.  An element x of a row or matrix whose largest is m is kept to 2^-23 |x| + 2^-50 m (two float16 parts
    with the largest at 2^14 or above: the second part is off by half of 2^-24 there, 2^-11 smaller), G / dloss to
    2^-23 of itself and 2^-50; products of two second parts, at most 2^-22, are within what _sums allows.

    Sums: a matrix instruction aligns eight products at a time by the sum of their factors' exponents and cuts each at 2^-24
    of the largest, where a factor below float16's normal numbers counts as the smallest of them, 2^-14, which is 2^-28
    of the largest element at 2^14: 16384 * 2^-23 with 7.476e-4 * 0.01299 beside it loses 5.86e-8 = 0.98 * 2^-24 *
    (2^14 * 2^-14), with 2^-5 * 2^-4 in place of the first 2^-33.  So the sums' error is that of the factors' sizes
    raised to at least 2^-28 of the largest, 8 * 2^-24 of each group's largest product and so of the whole sum of sizes,
    beside _sums for the accumulations."""
    config("ce.native", native)
    h, w, y, dl = _operands("float32", N, V, D, N + D, spread=40.0)
    h *= 10.0 ** -(torch.arange(D, device="cuda") % 11)
    w *= 10.0 ** (torch.arange(D, device="cuda") % 11 / 2)
    dl *= 10.0 ** -(torch.arange(N, device="cuda") % 9)
    h[1, :], w[1, :] = h[1, :] * 1e-6, w[1, :] * 1e-6
    loss, lse, dh, dw = _run(h, w, y, dl, "float32")
    H, W, dl = h.double(), w.double(), dl.double()
    ok = (y >= 0) & (y < V)
    n, at = torch.arange(N, device="cuda")[ok], y[ok].long()
    kept, floor = 2.0 ** -23, 2.0 ** -50

    def largest(x):
        return x.abs().amax(1, keepdim=True)

    def raised(x, most):
        return torch.maximum(x.abs(), 2.0 ** -28 * most)

    def sums(K):
        return _sums(K, "float32") + 8 * 2.0 ** -24

    logits = H @ W.T
    d = sums(D) * (raised(H, largest(H)) @ raised(W, largest(W)).T)
    d += floor * (largest(H) * W.abs().sum(1) + H.abs().sum(1)[:, None] * largest(W).T)
    want = torch.logsumexp(logits, 1)
    far = (logits - want[:, None]).abs().amax(1)
    d_lse = d.amax(1) + (far * 2.0 ** -23 + 2.0 ** -21) + _sums(V, "bfloat16") + 2.0 ** -23 * want.abs()
    assert bool(((lse.double() - want).abs() <= d_lse).all())
    want_loss = torch.zeros_like(want)
    want_loss[ok] = want[ok] - logits[n, at]
    assert bool(((loss.double() - want_loss).abs() <= d_lse + d.amax(1) + 2.0 ** -23 * want_loss.abs()).all())
    p = torch.exp(logits - want[:, None])
    e = p * (d + (d_lse + far * 2.0 ** -23 + 2.0 ** -21)[:, None]) + 2.0 ** -22 * p
    e[n, at] += 2.0 ** -22
    P = p.clone()
    P[n, at] -= 1.0
    e += kept * P.abs() + floor
    P[~ok], e[~ok] = 0.0, 0.0
    F = torch.where(ok, dl, 0.0)[:, None] * H
    assert float(p[ok].min()) < 2.0 ** -50 and float(F[ok].abs().max() / F[ok].abs().amin()) > 2.0 ** 30
    for got, a, ea, b, K, f in ((dw, P.T, e.T, F, N, torch.ones(V, 1, device="cuda")), (dh, P, e, W, V, torch.where(ok, dl, 0.0)[:, None])):
        eb = 1.5 * kept * b.abs() + floor * b.abs().max()      # a product with dloss is rounded as well
        exact = f * (a @ b)
        rounding = sums(K) * (raised(a, torch.ones_like(a)) @ raised(b, b.abs().max()))
        tol = f * (ea @ (b.abs() + eb) + a.abs() @ eb + rounding) + 2 * HALF_STEP["float32"] * exact.abs() + TINY
        assert bool(((got.double() - exact).abs() <= tol).all())
