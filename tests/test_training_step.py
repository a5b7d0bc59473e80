"""The training operators together, as a step on learned vertex embeddings uses them: the rows of a mini-batch's vertices
are looked up, aggregated over a graph, and scored against all vertices (the table is the scorer too); the gradients go
back the same way, both contributions to the table's gradient are added, and all gradients are clipped by their norm."""
import numpy as np
import pytest
import scipy.sparse
import torch

from featgraph_amd import _lib, placeholder
from featgraph_amd.module import (ClipGradNormhip, EmbeddingLookupGradhip, EmbeddingLookuphip, LinearCrossEntropyGradhip,
                                  LinearCrossEntropyhip, VanillaSpMMGradhip, VanillaSpMMhip)

pytestmark = pytest.mark.gpu


class Step:
    """One training step over a batch of `n` looked-up vertices, `rows` of which (the graph's destinations) are scored."""

    def __init__(self, adj, V, D, max_norm):
        rows, n = adj.shape
        self.lookup, self.lookup_grad = EmbeddingLookuphip(0.5), EmbeddingLookupGradhip(0.5)
        self.spmm, self.spmm_grad = VanillaSpMMhip(adj), VanillaSpMMGradhip(adj)
        self.loss, self.loss_grad = LinearCrossEntropyhip(), LinearCrossEntropyGradhip()
        self.clip = ClipGradNormhip(max_norm)
        table, ids, label = placeholder((V, D)), placeholder((n,), "int64"), placeholder((rows,), "int64")
        for m in (self.lookup, self.lookup_grad):
            m.build([table, ids])
        self.spmm.build([placeholder((n, D))], {}, {})
        self.spmm_grad.build([placeholder((n, D))], {}, {})
        for m in (self.loss, self.loss_grad):
            m.build([placeholder((rows, D)), table, label])
        self.clip.build([table])

    def run(self, table, ids, label, dloss):
        looked_up = self.lookup.run([table, ids])
        hidden = self.spmm.run([looked_up])
        loss, lse = self.loss.run([hidden, table, label])
        dhidden, dtable = self.loss_grad.run([hidden, table, label, lse, dloss])
        got = self.spmm_grad.run([looked_up, dhidden])
        dlooked_up = got[0] if isinstance(got, tuple) else got
        self.lookup_grad.run([ids, dlooked_up, dtable])          # the table's other gradient, added in place
        norm, (clipped,) = self.clip.run([dtable])
        return loss.tensor, norm.tensor, clipped.tensor


def _case(seed, n=300, rows=120, V=500, D=48):
    rng = np.random.default_rng(seed)
    adj = scipy.sparse.random(rows, n, density=0.05, format="csr", random_state=rng, dtype=np.float32)
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(V, D, generator=g).cuda()
    ids = torch.randint(-1, V, (n,), generator=g).cuda()
    label = torch.randint(-1, V, (rows,), generator=g).cuda()
    dloss = ((0.5 + torch.rand(rows, generator=g)) / rows).cuda()
    return adj, table, ids, label, dloss


def _reference(adj, table, ids, label, dloss, max_norm):
    t = table.double().requires_grad_(True)
    looked_up = torch.where((ids >= 0)[:, None], t[ids.clamp(min=0)] * 0.5, 0.0)
    hidden = torch.from_numpy(adj.toarray()).cuda().double() @ looked_up
    logits = hidden @ t.T
    ok = label >= 0
    loss = torch.where(ok, torch.logsumexp(logits, 1) - logits.gather(1, label.clamp(min=0)[:, None])[:, 0], 0.0)
    (loss * dloss.double() * ok).sum().backward()
    norm = t.grad.norm()
    return loss.detach(), norm, t.grad * min(1.0, max_norm / (float(norm) + 1e-6))


def test_a_step_matches_double_precision():
    """Each operator's own error is bounded in its own tests; together, sums of at most a few hundred float32 terms, the
    two-norm of the result's error stays below a hundred roundings (100 * 2^-24) of the largest intermediate's, whose
    logits of size |l| <= 30 scale the relative error of the probabilities."""
    adj, table, ids, label, dloss = _case(1)
    want = _reference(adj, table, ids, label, dloss, 0.05)
    got = Step(adj, 500, 48, 0.05).run(table, ids, label, dloss)
    for x, y in zip(got, want):
        assert float((x.double() - y).norm()) <= 30 * 100 * 2.0 ** -24 * float(y.norm())


def test_a_step_replays_from_a_graph():
    adj, table, ids, label, dloss = _case(2)
    step = Step(adj, 500, 48, 0.05)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step.run(table, ids, label, dloss)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step.run(table, ids, label, dloss)
    for k in range(3):
        _, t, i, y, d = _case(10 + k)
        for old, new in zip((table, ids, label, dloss), (t, i, y, d)):
            old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step.run(table, ids, label, dloss)))


def test_offsets_beyond_32_bits():
    """A table of 9.3 GB (2.3G elements), and probabilities of more than 4 GB, which are taken in pieces."""
    V, D = 9_000_001, 258
    table = torch.empty(V, D, device="cuda")
    table[-300:] = torch.arange(300 * D, device="cuda", dtype=torch.float32).reshape(300, D)
    ids = torch.arange(V - 300, V, device="cuda")
    ids[7] = -1
    f = EmbeddingLookuphip(2.0)
    f.build([placeholder((V, D)), placeholder((300,), "int64")])
    got = f.run([table, ids]).tensor
    want = table[-300:] * 2
    want[7] = 0
    assert torch.equal(got, want)
    del table
    g = EmbeddingLookupGradhip(2.0)
    g.build([placeholder((V, D)), placeholder((300,), "int64")])
    grad = g.run([ids, got]).tensor
    assert torch.equal(grad[-300:], want * 2) and not grad[:-300].any()
    del f, g, got, grad, want
    torch.cuda.empty_cache()

    N, V, D = 40001, 60013, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    h = torch.randn(N, D, generator=gen, device="cuda").bfloat16()
    w = (torch.randn(V, D, generator=gen, device="cuda") / 8).bfloat16()
    y = torch.randint(0, V, (N,), generator=gen, device="cuda", dtype=torch.int32)
    dl = torch.full((N,), 1.0 / N, device="cuda")
    ph = [placeholder((N, D), "bfloat16"), placeholder((V, D), "bfloat16"), placeholder((N,), "int32")]
    loss, grad = LinearCrossEntropyhip(), LinearCrossEntropyGradhip()
    loss.build(ph), grad.build(ph)
    _, lse = loss.run([h, w, y])
    dh, dw = grad.run([h, w, y, lse, dl])
    some_n, some_v = torch.arange(0, N, 3999, device="cuda"), torch.arange(0, V, 5999, device="cuda")
    H, W, L = h.double(), w.double(), lse.tensor.double()
    assert bool(((torch.logsumexp(H[some_n] @ W.T, 1) - L[some_n]).abs() <= 2.0 ** -18).all())   # 64-term logits below 8
    for rows, cols, got, other in ((some_n, None, dh.tensor[some_n], W), (None, some_v, dw.tensor[some_v], H)):
        a = H if rows is None else H[rows]
        b = W if cols is None else W[cols]
        p = torch.exp(a @ b.T - (L if rows is None else L[rows])[:, None])
        at = y.long() if rows is None else y[rows].long()
        names = torch.arange(V, device="cuda") if cols is None else cols
        p -= (at[:, None] == names[None, :]).double()
        p /= N
        p = p if cols is None else p.T
        want = p @ other
        # G rounded to bfloat16 (2^-8), the result too, and the float32 sums (see the cross entropy's own tests)
        tol = (2.0 ** -8 + (16 + 4 * 250) * 2.0 ** -24) * (p.abs() @ other.abs()) + 2.0 ** -8 * want.abs()
        assert bool(((got.double() - want).abs() <= tol * 1.01 + 1e-30).all())


def test_two_runs_on_two_streams():
    """Two modules at once on two streams do not disturb each other."""
    adj, table, ids, label, dloss = _case(4)
    a, b = Step(adj, 500, 48, 0.05), Step(adj, 500, 48, 0.05)
    want = [x.clone() for x in a.run(table, ids, label, dloss)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        outs = []
        for s, step in zip(streams, (a, b)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(step.run(table, ids, label, dloss))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for out in outs for x, y in zip(out, want))


def test_config_keys_of_the_products():
    assert _lib.config_get("ce.tile") == 0 and _lib.config_get("ce.piece_rows") == 0


def test_build_leaves_nothing_to_do_on_its_stream():
    """Modules built while their stream is busy, and run at once on another one: nothing that build() enqueued may
    arrive later and write into the results."""
    V, n, D = 300, 70, 40
    g = torch.Generator().manual_seed(5)
    table, dout = torch.randn(V, D, generator=g).cuda(), torch.randn(n, D, generator=g).cuda()
    ids = torch.randint(0, V, (n,), generator=g).cuda()
    hidden, dloss = torch.randn(n, D, generator=g).cuda(), torch.rand(n, generator=g).cuda() + 0.5
    ph = [placeholder((V, D)), placeholder((n,), "int64")]
    triple = [placeholder((n, D))] + ph

    def build():
        m = (EmbeddingLookuphip(2.0), EmbeddingLookupGradhip(2.0), LinearCrossEntropyhip(), LinearCrossEntropyGradhip(), ClipGradNormhip(0.5))
        for x, p in zip(m, (ph, ph, triple, triple, [placeholder((V, D)), placeholder((n, D))])):
            x.build(p)
        return m

    def run(m):
        rows, grad = m[0].run([table, ids]), m[1].run([ids, dout])
        loss, lse = m[2].run([hidden, table, ids])
        dh, dw = m[3].run([hidden, table, ids, lse, dloss])
        norm, clipped = m[4].run([table, dout])
        return [x.tensor for x in (rows, grad, loss, lse, dh, dw, norm, *clipped)]

    first = build()
    want = [x.clone() for x in run(first)]
    a = torch.randn(8192, 8192, device="cuda")
    b = torch.empty_like(a)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(6):                      # some 40 ms of work
        torch.mm(a, a, out=b)
    m = build()
    with torch.cuda.stream(side):
        got = run(m)
    side.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
