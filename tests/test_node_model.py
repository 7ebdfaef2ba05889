"""The operators as a node model uses them: a looked-up table of features, products with the graph, log probabilities of
labels - trained, classified, and the parts of ShardedGCN2 that call them."""
import pytest
import torch

from trspmm import graphs

pytestmark = pytest.mark.gpu


def _graph(scale=9, seed=4):
    rp, col, val = graphs.rmat_graph(scale, 8, seed=seed)
    n = rp.numel() - 1
    rows = torch.repeat_interleave(torch.arange(n), (rp[1:] - rp[:-1]).long())
    A = torch.sparse_coo_tensor(torch.stack([rows, col.long()]), val.half().double(), (n, n)).to_dense().cuda()
    return rp.cuda(), col.cuda(), val.cuda(), n, A


def _close(got, ref, bar):
    """Largest difference over the largest magnitude."""
    err = float((got.detach().double() - ref).abs().max() / ref.abs().max())
    assert err <= bar, err


@pytest.mark.parametrize("table_dtype", [torch.float32, torch.float16])
def test_training_step_of_a_node_classifier(table_dtype):
    """Gradients of the table and both weights against fp64 autograd through the same expression.

    Between the table and the loss lie six roundings to fp16 forward and as many backward, each at most 2^-11 of the value;
    sums of rounded values with signs lose up to the ratio of their magnitudes to the result, which is below 4 for
    these seeds' entries of largest magnitude: 12 * 4 * 2^-11 = 2.4e-2."""
    from trspmm import DifferentiableSpmm, class_logprobs, embedding
    rp, col, val, n, A = _graph()
    val = val / 4
    A = A / 4
    V, F0, F1, C = 100, 48, 32, 7
    g = torch.Generator(device="cuda").manual_seed(0)
    table = torch.randn(V, F0, generator=g, device="cuda").to(table_dtype).requires_grad_()
    W1 = (torch.randn(F0, F1, generator=g, device="cuda") * 0.1).half().requires_grad_()
    W2 = (torch.randn(F1, C, generator=g, device="cuda") * 0.1).half().requires_grad_()
    ids = torch.randint(0, V, (n,), generator=g, device="cuda")
    labels = torch.randint(0, C, (n,), generator=g, device="cuda")
    labels[::3] = -1
    op = DifferentiableSpmm(rp, col, val, n)
    count = int((labels >= 0).sum())

    x = embedding(table, ids, scale=0.5, padding_id=3, out_dtype=torch.float16)
    h = torch.relu(op(x @ W1))
    out = class_logprobs(op(h @ W2), labels, ignore_id=-1, top=2)
    loss = -out.logprobs.sum() - 0.1 * out.entropy.sum()
    loss.backward()

    t64, a64, b64 = [p.detach().double().requires_grad_() for p in (table, W1, W2)]
    x64 = 0.5 * t64[ids] * (ids != 3)[:, None]
    z = A @ (torch.relu(A @ (x64 @ a64)) @ b64)
    lp = torch.log_softmax(z, 1)
    H = -(lp.exp() * lp).sum(1)
    lab = lp.gather(1, labels.clamp(min=0)[:, None])[:, 0] * (labels >= 0)
    want = -lab.sum() - 0.1 * H.sum()
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 5e-3 * count
    for got, ref in ((table, t64), (W1, a64), (W2, b64)):
        assert got.grad.dtype is got.dtype
        _close(got.grad, ref.grad, 2.4e-2)
    assert float(table.grad[3].abs().max()) == 0
    assert torch.equal(out.top_ids[:, 0].long(), op(h @ W2).max(1).indices)


@pytest.mark.parametrize("V", [60, 3000])   # a table shorter and one longer than the graph has nodes
@pytest.mark.parametrize("gather", ["h1", "z2", "gemm_bcast"])
def test_gcn_with_looked_up_features_and_classes(V, gather):
    from trspmm import ShardedGCN2, class_logprobs, embedding
    rp, col, val, n, _ = _graph(11)
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randn(V, 64, generator=g, device="cuda").half()
    W1, W2 = [(torch.randn(a, b, generator=g, device="cuda") * 0.1).half() for a, b in ((64, 64), (64, 32))]
    ids = torch.randint(0, V, (n,), generator=g, device="cuda").to(torch.int32)
    model = ShardedGCN2(rp, col, val)
    plain = model.forward(embedding(table, ids), W1, W2, gather=gather)
    got = model.forward(table, W1, W2, gather=gather, ids=ids)
    # a row of the product is the same row whether looked up before it or behind it, up to the library's order of its sum (one fp16
    # rounding of the first product, carried through two layers)
    _close(got, plain.double(), 1e-2)
    labels = torch.randint(0, 32, (n,), generator=g, device="cuda")
    r = model.classify(table, W1, W2, labels, top=3, gather=gather, ids=ids)
    want = class_logprobs(got, labels, top=3)
    assert torch.equal(r.top_ids, want.top_ids) and torch.equal(r.logprobs, want.logprobs) and torch.equal(r.entropy, want.entropy)
    assert model.classify(embedding(table, ids), W1, W2, gather=gather).top_ids.shape == (n, 1)
    with pytest.raises(ValueError):
        model.forward(table, W1, W2, ids=ids[:-1])


def test_first_order_gradients_under_create_graph_and_no_second_order():
    from trspmm import class_logprobs, embedding
    W = torch.randn(10, 8, device="cuda", requires_grad=True)
    ids = torch.arange(10, device="cuda")
    r = class_logprobs(embedding(W, ids), ids % 8)
    g, = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), W, create_graph=True)
    want, = torch.autograd.grad(class_logprobs(embedding(W, ids), ids % 8).logprobs.sum(), W)
    assert g.shape == want.shape
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), W)


@pytest.mark.parametrize("top", [0, 3])
def test_entropy_alone_without_targets(top):
    """Outputs that are None beside one that has a gradient."""
    from trspmm import class_logprobs, class_logprobs_grad
    x = torch.randn(20, 33, device="cuda", requires_grad=True)
    r = class_logprobs(x, top=top)
    assert r.logprobs is None and (r.top_ids is None) == (top == 0)
    r.entropy.sum().backward()
    lp = torch.log_softmax(x.detach().double(), 1)
    H = -(lp.exp() * lp).sum(1, keepdim=True)
    want = -lp.exp() * (lp + H)
    # p, log p and H are off by a few 2^-24 of magnitudes up to 10
    assert float((x.grad.double() - want).abs().max()) <= 64 * 2.0 ** -24
    with torch.no_grad():
        again = class_logprobs_grad(x, None, class_logprobs(x, top=top), g_entropy=torch.ones(20, device="cuda"))
    assert torch.equal(again, x.grad)


def test_a_whole_step_captured_and_replayed():
    """Lookup, log probabilities and both gradients in one graph, replayed on new ids and labels."""
    from trspmm import class_logprobs, embedding
    g = torch.Generator(device="cuda").manual_seed(0)
    table = torch.randn(5000, 47, generator=g, device="cuda").half().requires_grad_()
    ids = torch.randint(0, 5000, (6000,), generator=g, device="cuda")
    labels = torch.randint(0, 47, (6000,), generator=g, device="cuda")

    def step():
        r = class_logprobs(embedding(table, ids, scale=0.5), labels, top=2)
        return (r.logprobs, r.top_ids, *torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), table))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    ids.copy_(torch.randint(0, 50, (6000,), generator=g, device="cuda"))
    labels.copy_(torch.randint(0, 47, (6000,), generator=g, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_classify_refuses_labels_of_another_graph():
    """Labels are all nodes': a longer list is another graph's, and its first part not this one's."""
    from trspmm import ShardedGCN2
    rp, col, val, n, _ = _graph()
    model = ShardedGCN2(rp, col, val)
    X, W1, W2 = [torch.zeros(*s, dtype=torch.float16, device="cuda") for s in ((n, 16), (16, 16), (16, 8))]
    for bad in (n + 1, n - 1, 2 * n):
        with pytest.raises(ValueError):
            model.classify(X, W1, W2, torch.zeros(bad, dtype=torch.int64, device="cuda"))


def test_create_graph_gives_the_same_first_order_gradients():
    """Every upstream gradient arrives, in its place, through the form that runs under create_graph."""
    from trspmm import class_logprobs, embedding
    g = torch.Generator(device="cuda").manual_seed(0)
    W = torch.randn(40, 24, generator=g, device="cuda", requires_grad=True)
    ids = torch.randint(0, 40, (90,), generator=g, device="cuda")
    a, b, c = [torch.randn(*s, generator=g, device="cuda") for s in ((90,), (90,), (90, 3))]

    def grad(create_graph):
        r = class_logprobs(embedding(W, ids, scale=0.5, padding_id=3), ids % 24, top=3, scale=1.5, ignore_id=5)
        loss = (r.logprobs * a).sum() + (r.entropy * b).sum() + (r.top_logprobs * c).sum()
        return torch.autograd.grad(loss, W, create_graph=create_graph)[0]
    assert torch.equal(grad(True).detach(), grad(False))
