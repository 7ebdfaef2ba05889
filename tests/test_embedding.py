"""Embedding lookup and its gradient against the definition in 64 bits.

Tolerances.  Lookup: one fp32 product and one rounding, |err| <= |y| (2^-24 + eps/2) and half the smallest subnormal of the
result's type.  Gradient: a sum of c terms in fp32 in any order is off by at most c 2^-24 sum|g|, the factor and the result's
rounding as above."""
import ctypes
import threading

import pytest
import torch

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}
U = 2.0 ** -24
NO_PADDING = -(1 << 63)


def _within(got, ref, extra, dtype):
    bound = ref.abs() * (2 * U + torch.finfo(dtype).eps / 2) * (1 + 1e-6) + extra * 1.01 + TINY[dtype]
    bad = ~((got.double() - ref).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - ref).abs() - bound)[bad].max()))


def _grad_ref(g, ids, rows, scale, padding=None):
    """(sums, sums of magnitudes times counts times 2^-24) in 64 bits."""
    ids = ids.reshape(-1).long()
    g = g.reshape(-1, g.shape[-1]).double()
    keep = (ids >= 0) & (ids < rows)
    if padding is not None:
        keep &= ids != padding
    ids, g = ids[keep], g[keep]
    ref = torch.zeros(rows, g.shape[1], dtype=torch.float64, device=g.device).index_add_(0, ids, g) * scale
    mag = torch.zeros_like(ref).index_add_(0, ids, g.abs()) * abs(scale)
    count = torch.bincount(ids, minlength=rows)[:, None]
    return ref, mag * count * U


def _randn(*shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def _ids(n, rows, seed=0, dtype=torch.int64, skew=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    u = torch.rand(n, generator=g, device="cuda")
    return ((u ** 6 if skew else u) * rows).long().clamp(max=rows - 1).to(dtype)


# ---- without a GPU ------------------------------------------------------------------------------

def test_entries_refuse_bad_arguments_before_any_launch():
    from trspmm import _lib
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    a = (ctypes.addressof(buf) + 255) & ~255
    sz = ctypes.c_size_t()

    def look(table=a, tt=0, rows=4, ts=8, ids=a, n=2, F=8, out=a, ot=0, os=8):
        return lib.trs_embedding(table, tt, rows, ts, ids, 1, n, F, 1.0, NO_PADDING, out, ot, os, None)
    assert look(n=0) == 0
    for bad in (dict(table=None), dict(ids=None), dict(out=None), dict(rows=0), dict(n=-1), dict(F=0), dict(tt=3), dict(ot=-1),
                dict(ts=7), dict(os=7)):
        assert look(**bad) == -1, bad
    assert look(table=a + 2) == -1 and look(out=a + 1, ot=1) == -1 and look(ids=a + 4) == -1   # not on element boundaries
    for big in (dict(rows=1 << 31), dict(n=1 << 31), dict(F=(1 << 20) + 1, ts=1 << 21, os=1 << 21), dict(ts=1 << 31), dict(os=1 << 31)):
        assert look(**big) == -10, big
    assert lib.trs_embedding_grad_workspace_bytes(10, 4, 8, None) == -1
    assert lib.trs_embedding_grad_workspace_bytes(10, 0, 8, ctypes.byref(sz)) == -1
    assert lib.trs_embedding_grad_workspace_bytes(0, 4, 8, ctypes.byref(sz)) == 0 and sz.value == 0
    assert lib.trs_embedding_grad_workspace_bytes(1 << 20, 1 << 20, 128, ctypes.byref(sz)) == 0 and sz.value > 16 << 20

    def grad(g=a, gt=0, gs=8, ids=a, n=2, rows=4, F=8, out=a, ot=0, os=8, acc=0, ws=a, wb=0):
        return lib.trs_embedding_grad(g, gt, gs, ids, 1, n, rows, F, 1.0, NO_PADDING, out, ot, os, acc, ws, wb, None)
    for bad in (dict(g=None), dict(ids=None), dict(out=None), dict(rows=0), dict(n=-1), dict(F=0), dict(gt=3), dict(ot=3), dict(gs=7),
                dict(os=7)):
        assert grad(**bad) == -1, bad
    assert grad(g=a + 2) == -1 and grad(out=a + 1, ot=2) == -1 and grad(ids=a + 4) == -1
    assert grad(wb=100) == -7 and grad(ws=None, wb=1 << 30) == -7 and grad(ws=a + 8, wb=1 << 30) == -7
    assert grad(n=1 << 31) == -10
    assert grad(n=0, acc=1) == 0


def test_python_entries_refuse_cpu_tensors():
    from trspmm import embedding, embedding_grad
    ids = torch.tensor([0, 1])
    with pytest.raises(ValueError):
        embedding(torch.ones(2, 4), ids)
    with pytest.raises(ValueError):
        embedding_grad(torch.ones(2, 4), ids, 2)


# ---- lookup -----------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("table", [F32, F16, BF16])
@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("F", [1, 2, 7, 12, 47, 64, 96, 100, 256, 520])
def test_lookup_types_and_widths(table, out, F):
    from trspmm import embedding
    W, ids = _randn(301, F, dtype=table), _ids(1003, 301, seed=F)
    got = embedding(W, ids, scale=0.7, out_dtype=out)
    assert got.dtype is out and got.shape == (1003, F)
    _within(got, W.double()[ids] * torch.tensor(0.7, dtype=F32).double().item(), 0.0, out)
    if table is out:
        assert torch.equal(embedding(W, ids), W[ids])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [0, 1, 3, 4, 5, 31, 257])
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_lookup_lengths_shapes_padding_and_ids_outside(n, idt):
    from trspmm import embedding
    W = _randn(17, 40, dtype=F16)
    ids = _ids(n, 17, seed=n, dtype=idt)
    if n > 4:
        ids[1], ids[2], ids[3], ids[4] = -1, 17, torch.iinfo(idt).max, torch.iinfo(idt).min
    got = embedding(W, ids, padding_id=5)
    inside = (ids >= 0) & (ids < 17)
    ref = W[ids.clamp(0, 16).long()]
    ref[ids == 5] = 0
    ref[~inside] = float("nan")
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0))
    got = embedding(W, ids, padding_id=-1)     # a padding id outside the table
    ref = torch.where((ids == -1)[:, None], torch.zeros_like(ref), W[ids.clamp(0, 16).long()])
    ref[~inside & (ids != -1)] = float("nan")
    assert torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0))
    if n == 4:
        assert torch.equal(embedding(W, ids.view(2, 2)), W[ids.long()].view(2, 2, 40))
        assert embedding(W, ids[0]).shape == (40,)


@pytest.mark.gpu
@pytest.mark.parametrize("offset,width,F", [(0, 64, 48), (1, 65, 48), (2, 50, 47), (4, 72, 64), (8, 80, 64)])
def test_lookup_strided_rows(offset, width, F):
    from trspmm import embedding
    big = _randn(50, width, dtype=BF16)
    W = big[:, offset:offset + F]
    dst = torch.full((99, width), 3.0, dtype=BF16, device="cuda")
    ids = _ids(99, 50)
    got = embedding(W, ids, out=dst[:, offset:offset + F])
    assert got.data_ptr() == dst[:, offset:].data_ptr() and torch.equal(got, W[ids])
    rest = torch.ones(width, dtype=torch.bool, device="cuda")
    rest[offset:offset + F] = False
    assert bool((dst[:, rest] == 3.0).all())


@pytest.mark.gpu
def test_lookup_far_rows():
    """Offsets past 2^31 elements in the table and in the result."""
    from trspmm import embedding
    rows, F = 35_000_000, 64
    W = torch.zeros(rows, F, dtype=F16, device="cuda")
    W[-1], W[33554432 + 5] = 2.0, 3.0
    ids = torch.full((rows,), 1, dtype=torch.int32, device="cuda")
    ids[-1], ids[-2] = rows - 1, 33554432 + 5
    got = embedding(W, ids)
    assert bool((got[-1] == 2).all()) and bool((got[-2] == 3).all()) and float(got[:-2].abs().max()) == 0


@pytest.mark.gpu
def test_refusals():
    from trspmm import embedding, embedding_grad
    W, ids = _randn(8, 16, dtype=F16), _ids(6, 8)
    with pytest.raises(TypeError):
        embedding(W.double(), ids)
    with pytest.raises(TypeError):
        embedding(W, ids.short())
    with pytest.raises(TypeError):
        embedding(W, ids, out_dtype=torch.float64)
    for call in (lambda: embedding(W, ids.cpu()), lambda: embedding(W.t(), ids), lambda: embedding(W[:1].expand(8, 16), ids),
                 lambda: embedding(W, torch.stack([ids, ids], 1)[:, 0]), lambda: embedding(W[0], ids), lambda: embedding(W[:0], ids),
                 lambda: embedding(W, ids, out=W[:6]), lambda: embedding(W, ids, out=torch.empty(5, 16, dtype=F16, device="cuda")),
                 lambda: embedding(W.requires_grad_(), ids, out=torch.empty(6, 16, dtype=F16, device="cuda")),
                 lambda: embedding_grad(W.detach()[:6], ids, 0), lambda: embedding_grad(W.detach(), ids, 8),
                 lambda: embedding_grad(W.detach()[:6], ids, 8, accumulate=True),
                 lambda: embedding_grad(W.detach()[:1].expand(6, 16), ids, 8),
                 lambda: embedding_grad(W.detach()[:6], ids, 8, out=W.detach()),
                 lambda: embedding_grad(W.detach()[:6], ids, 8, out=torch.empty(7, 16, dtype=F16, device="cuda"))):
        with pytest.raises(ValueError):
            call()


# ---- gradient ------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("gt", [F32, F16, BF16])
@pytest.mark.parametrize("ot", [F32, F16, BF16])
@pytest.mark.parametrize("F", [1, 7, 12, 47, 64, 100, 264])
def test_grad_types_and_widths(gt, ot, F):
    from trspmm import embedding_grad
    ids, g = _ids(2100, 333, seed=F, skew=True), _randn(2100, F, dtype=gt, seed=1)
    got = embedding_grad(g, ids, 333, scale=0.75, out_dtype=ot)
    ref, extra = _grad_ref(g, ids, 333, 0.75)
    _within(got, ref, extra, ot)
    assert torch.equal(got, embedding_grad(g, ids, 333, scale=0.75, out_dtype=ot))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 2047, 2048, 70001, (1 << 22) + 3])
@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, 4096, 4097, 20000, 70001])
def test_grad_sizes(rows, n):
    """One, two and three passes of the sort; lengths around its tiles and the summed blocks."""
    from trspmm import embedding_grad
    ids, g = _ids(n, rows, seed=n, skew=rows > 100), _randn(n, 8, seed=2)
    got = embedding_grad(g, ids, rows)
    ref, extra = _grad_ref(g, ids, rows, 1.0)
    _within(got, ref, extra, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 300, 70001, (1 << 20), (1 << 22) + 3, (1 << 24) + 1])
@pytest.mark.parametrize("n", [(1 << 19) - 1, 1 << 19, 600_011])
def test_grad_of_many_ids(rows, n):
    """One to four passes of narrow digits, and the last length that takes wide ones."""
    from trspmm import embedding_grad
    ids, g = _ids(n, rows, seed=n, skew=rows > 1000), _randn(n, 4, seed=2)
    ref, extra = _grad_ref(g, ids, rows, 1.0)
    _within(embedding_grad(g, ids, rows), ref, extra, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("pattern", ["one row", "two rows", "sorted", "reversed", "runs", "last row"])
@pytest.mark.parametrize("n", [300, 9000, 600_011])
def test_grad_popular_rows(pattern, n):
    """Rows with a block's, a span's and many spans' worth of positions, with ragged ends on both sides."""
    from trspmm import embedding_grad
    rows = 5000
    i = torch.arange(n, device="cuda")
    ids = {"one row": i * 0 + 77, "two rows": (i >= n // 3).long() * 4999, "sorted": i * rows // n, "reversed": rows - 1 - i * rows // n,
           "runs": torch.where(i % 7 < 5, 1234, (i * 31) % rows), "last row": i * 0 + rows - 1}[pattern]
    g = _randn(n, 40, dtype=F16, seed=3)
    got = embedding_grad(g, ids, rows, out_dtype=F32)
    ref, extra = _grad_ref(g, ids, rows, 1.0)
    _within(got, ref, extra, F32)
    # one and the same order of the sum whatever the other rows hold
    other = torch.cat([ids, (i[:100] * 13) % 3000 + 1500])
    if pattern == "one row":
        again = embedding_grad(torch.cat([g, torch.zeros_like(g[:100])]), other, rows, out_dtype=F32)
        assert torch.equal(again[77], got[77])


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [1, 3, 1000])
@pytest.mark.parametrize("F,dtype", [(40, F16), (3, F32), (300, BF16)])
def test_grad_rows_of_every_length_side_by_side(gap, F, dtype):
    """Rows of a few positions, of as many as make a row popular, of blocks and spans, next to each other and apart."""
    from trspmm import embedding_grad
    lengths = torch.tensor([0, 1, 2, 7, 8, 9, 22, 23, 24, 25, 26, 47, 63, 64, 65, 0, 127, 128, 129, 24, 24, 500, 511, 512, 513, 1, 1025, 23] * 3,
                           device="cuda")
    ids = torch.repeat_interleave(torch.arange(lengths.numel(), device="cuda") * gap, lengths)
    rows = lengths.numel() * gap + 5
    for order in (torch.arange(ids.numel(), device="cuda"), torch.randperm(ids.numel(), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")):
        g = _randn(ids.numel(), F, dtype=dtype, seed=7)
        got = embedding_grad(g, ids[order], rows, out_dtype=F32)
        ref, extra = _grad_ref(g, ids[order], rows, 1.0)
        _within(got, ref, extra, F32)
        out = torch.ones(rows, F, device="cuda")
        embedding_grad(g, ids[order], rows, out=out, accumulate=True)
        _within(out, ref + 1.0, extra + 4 * U, F32)
        assert bool((out[got.abs().sum(1) == 0] == 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_grad_padding_ids_outside_and_nothing_left(idt):
    from trspmm import embedding_grad
    ids = _ids(3000, 50, dtype=idt)
    ids[::7], ids[1::9], ids[2::11] = -1, 50, torch.iinfo(idt).max
    g = _randn(3000, 24, dtype=BF16)
    g[ids == -1] = float("nan")
    g[ids == 3] = float("inf")
    got = embedding_grad(g, ids, 50, padding_id=3, out_dtype=F32)
    ok = (ids >= 0) & (ids < 50) & (ids != 3)
    ref, extra = _grad_ref(g[ok], ids[ok], 50, 1.0)
    _within(got, ref, extra, F32)
    assert float(got[3].abs().max()) == 0
    empty = embedding_grad(g, torch.full_like(ids, 50), 50)
    assert float(empty.float().abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("ot", [F32, F16])
def test_grad_accumulates_and_leaves_other_rows(ot):
    from trspmm import embedding_grad
    wide = _randn(400, 100, dtype=ot, seed=5)
    before = wide.clone()
    out = wide[:, 3:43]
    ids, g = _ids(500, 200, skew=True), _randn(500, 40, dtype=ot, seed=6)
    got = embedding_grad(g, ids, 400, out=out, accumulate=True)
    assert got is out
    named = torch.bincount(ids, minlength=400) > 0
    ref, extra = _grad_ref(g, ids, 400, 1.0)
    ref = ref + before[:, 3:43].double()
    extra = extra + before[:, 3:43].abs().double() * 2 * U
    _within(out, ref, extra, ot)
    assert torch.equal(out[~named], before[:, 3:43][~named])
    rest = torch.ones(100, dtype=torch.bool, device="cuda")
    rest[3:43] = False
    assert torch.equal(wide[:, rest], before[:, rest])
    same = wide.clone()
    embedding_grad(g[:0], ids[:0], 400, out=out, accumulate=True)
    assert torch.equal(wide, same)


@pytest.mark.gpu
def test_grad_far_rows():
    """Offsets past 2^31 elements in the gradient and in the table's gradient."""
    from trspmm import embedding_grad
    rows, F = 35_000_000, 64
    g = torch.zeros(rows, F, dtype=F16, device="cuda")
    g[-1], g[-2], g[0] = 2.0, 3.0, 1.0
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ids[-1], ids[-2] = rows - 1, 33554432 + 5
    got = embedding_grad(g, ids, rows)
    assert bool((got[-1] == 2).all()) and bool((got[33554432 + 5] == 3).all()) and bool((got[0] == 1).all())
    assert float(got[1:33554432].abs().max()) == 0


# ---- through autograd, streams, graphs, threads ---------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,F", [(F32, 20), (F16, 64), (BF16, 33)])
def test_autograd_gradient_is_the_formula_and_the_differences(dtype, F):
    from trspmm import embedding
    W = _randn(40, F, dtype=dtype).requires_grad_()
    ids = _ids(300, 40, skew=True).view(30, 10)
    G = _randn(30, 10, F, dtype=dtype, seed=9)
    y = embedding(W, ids, scale=1.5, padding_id=2)
    y.backward(G)
    ref, extra = _grad_ref(G, ids, 40, 1.5, padding=2)
    assert W.grad.dtype is dtype
    _within(W.grad, ref, extra, dtype)
    if dtype is F32:   # the lookup is linear in the table: a difference is the derivative up to its roundings
        with torch.no_grad():
            d = _randn(40, F, seed=11)
            lhs = ((embedding(W + d, ids, 1.5, 2).double() - embedding(W, ids, 1.5, 2).double()) * G.double()).sum()
            rhs = (W.grad.double() * ((W + d).double() - W.double())).sum()
        mag = (G.double().abs() * 1.5 * (W[ids].double().abs() + (W + d)[ids].double().abs())).sum()
        assert abs(float(lhs - rhs)) <= 310 * U * float(mag)
    embedding(W, ids).sum().backward()     # an expanded gradient
    mixed = embedding(W, ids, out_dtype=F16)
    g, = torch.autograd.grad(mixed, W, torch.ones_like(mixed))
    assert g.dtype is dtype and g.shape == W.shape


@pytest.mark.gpu
def test_another_stream_and_a_replayed_graph():
    from trspmm import embedding, embedding_grad
    W, ids, g = _randn(3000, 64, dtype=F16), _ids(9000, 3000, skew=True), _randn(9000, 64, dtype=F16, seed=1)
    want, want_g = embedding(W, ids), embedding_grad(g, ids, 3000)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a, b = embedding(W, ids), embedding_grad(g, ids, 3000)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, want) and torch.equal(b, want_g)
    graphs = []
    for _ in range(2):   # two graphs, replayed at once: neither may use the other's workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a, b = embedding(W, ids), embedding_grad(g, ids, 3000)
        graphs.append((graph, a, b, torch.cuda.Stream()))
    ids2 = _ids(9000, 3000, seed=5)
    ids.copy_(ids2)
    want, want_g = embedding(W, ids), embedding_grad(g, ids, 3000)
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, _a, _b, st in graphs:
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _graph, a, b, _st in graphs:
        assert torch.equal(a, want) and torch.equal(b, want_g)


@pytest.mark.gpu
def test_calls_from_several_threads():
    from trspmm import embedding_grad
    cases = [(_ids(5000 + k, 700 + 300 * k, seed=k, skew=True), _randn(5000 + k, 32, seed=k), 700 + 300 * k) for k in range(4)]
    want = [embedding_grad(g, i, r) for i, g, r in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                i, g, r = cases[k]
                got = embedding_grad(g, i, r)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[k]):
                    wrong.append(k)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("table,out", [(F16, F16), (F32, F16), (BF16, F32)])
def test_forward_mode_is_refused(table, out):
    """A tangent is not dropped in silence, whichever operand has it."""
    import torch.autograd.forward_ad as fw
    from trspmm import embedding, embedding_grad
    W, ids, g = _randn(8, 16, dtype=table), _ids(6, 8), _randn(6, 16, dtype=table)
    plain = embedding(W, ids, out_dtype=out)
    with fw.dual_level():
        dual, dual_g = fw.make_dual(W, torch.ones_like(W)), fw.make_dual(g, torch.ones_like(g))
        dual_out = fw.make_dual(torch.zeros_like(plain), torch.ones_like(plain))
        for call in (lambda: embedding(dual, ids, out_dtype=out), lambda: embedding(dual, ids, out=torch.empty_like(plain)),
                     lambda: embedding(W, ids, out=dual_out), lambda: embedding_grad(dual_g, ids, 8),
                     lambda: embedding_grad(dual_g, ids, 8, out=torch.empty_like(W)), lambda: embedding_grad(g, ids, 8, out=dual)):
            with pytest.raises(RuntimeError):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError):
                call()
        leaf = W.clone().requires_grad_()
        y = embedding(leaf, ids)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, leaf, dual_g)
        assert torch.equal(embedding(W, ids, out_dtype=out), plain)   # no tangent: as outside the level
    assert torch.equal(embedding(W, ids, out_dtype=out), plain)


@pytest.mark.gpu
def test_results_written_in_place_are_noticed_by_autograd():
    """out= changes a tensor that a graph may have kept: its backward pass raises as after any change in place."""
    from trspmm import embedding, embedding_grad
    W, ids = _randn(8, 16), _ids(6, 8)
    for write in (lambda t: embedding(W, ids, out=t), lambda t: embedding(W, ids, out=t[:, :]),
                  lambda t: embedding_grad(_randn(9, 16), _ids(9, 6), 6, out=t),
                  lambda t: embedding_grad(_randn(9, 16), _ids(9, 6), 6, out=t, accumulate=True)):
        w = torch.ones(6, 16, device="cuda", requires_grad=True)
        kept = torch.ones(6, 16, device="cuda")
        y = w * kept
        write(kept)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    leaf = torch.ones(6, 16, device="cuda", requires_grad=True)
    for out in (leaf, leaf * 2):   # what autograd follows is not overwritten behind its back
        for call in (lambda: embedding(W, ids, out=out), lambda: embedding_grad(_randn(9, 16), _ids(9, 6), 6, out=out)):
            with pytest.raises(ValueError):
                call()
            with torch.no_grad():
                assert call() is out
    with torch.inference_mode():
        assert torch.equal(embedding(W, ids, out=torch.empty(6, 16, device="cuda")), W[ids])


@pytest.mark.gpu
def test_ids_that_64_bits_do_not_hold_are_refused():
    """They do not come back as other ids."""
    from trspmm import embedding, embedding_grad
    W, ids = _randn(8, 16, dtype=F16), _ids(6, 8)
    for bad in (1 << 64, (1 << 64) + 3, 1 << 63, -(1 << 63), -(1 << 64) + 1):
        for call in (lambda: embedding(W, ids, padding_id=bad), lambda: embedding_grad(W[:6], ids, 8, padding_id=bad)):
            with pytest.raises(ValueError):
                call()
    for far in ((1 << 63) - 1, 1 - (1 << 63)):
        assert torch.equal(embedding(W, ids, padding_id=far), W[ids])
