"""Log probabilities, entropy, alternatives and their gradient against the definition in 64 bits.

Tolerances, with U = 2^-24, z = scale (x - max x) and E the mean under p.  A difference, the factor and the exponent's argument each
round once (a few U |z|), the exponential is off by 2^-22, a sum over C terms kept by 32 to 1024 threads by at most (C / 32 + 64) U, a
rescaling by (4 |climb| + 8) U where the climb ends at 104 (e^-104 is 0 in fp32).  So log S is off by U (4 E|z| + C / 32 + 128 + 4 R)
with R = min(range of z, 104), a log probability by that and 4 U |z_target|, the entropy by that, by U 4 E z^2 and E|z| times the
relative error of the sums."""
import ctypes

import pytest
import torch

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TINY = {F32: 2.0 ** -126, F16: 2.0 ** -24, BF16: 2.0 ** -126}
U = 2.0 ** -24
NEG = float("-inf")


def _scores(n, C, dtype=F32, seed=0, spread=2.0, width=None, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * C)
    x = (torch.randn(n, C, generator=g, device="cuda") * spread).to(dtype)
    if width is None:
        return x
    big = torch.full((n, width), 99.0, dtype=dtype, device="cuda")
    big[:, offset:offset + C] = x
    return big[:, offset:offset + C]


class Ref:
    """The operator in 64 bits, with the tolerances of what fp32 makes of it."""

    def __init__(self, x, targets=None, top=0, mask=None, scale=1.0, ignore=None):
        n, C = x.shape
        self.x, self.scale, self.t, self.ignore = x, scale, targets, ignore
        raw = x.detach().double()
        may = torch.ones_like(raw, dtype=torch.bool) if mask is None else mask.expand(n, C).clone()
        may &= raw != NEG
        raw = raw.masked_fill(~may, NEG)
        self.may, self.none = may, ~may.any(1)
        self.broken = (torch.isnan(raw) | (raw == float("inf"))).any(1)
        ok = ~self.none & ~self.broken
        m = raw.max(1).values
        z = scale * (raw - torch.where(ok, m, 0.0)[:, None])
        z = torch.where(may & ok[:, None], z, NEG)
        log_S = torch.where(ok, torch.logsumexp(torch.where(ok[:, None], z, 0.0), 1), 0.0)
        self.logp = z - log_S[:, None]
        self.p = torch.exp(self.logp)
        zf, lf = z.masked_fill(z == NEG, 0.0), self.logp.masked_fill(z == NEG, 0.0)
        self.lf = lf
        self.H = -(self.p * lf).sum(1)
        Ez, Ez2 = (self.p * zf.abs()).sum(1), (self.p * zf ** 2).sum(1)
        R = (-zf).max(1).values.clamp(max=104.0)
        self.err_S = U * (4 * Ez + C / 32 + 128 + 4 * R)
        self.err_H = self.err_S * (1 + Ez) + 4 * U * Ez2 + 4 * U * self.H.abs()
        self.zf = zf
        nan = torch.full((n,), float("nan"), dtype=torch.float64, device=x.device)
        self.entropy = torch.where(self.broken, nan, self.H)
        if targets is not None:
            t = targets.long()
            inside = (t >= 0) & (t < C)
            rows = torch.arange(n, device=x.device)
            tc = t.clamp(0, C - 1)
            lp = torch.where(inside & ~self.broken, self.logp[rows, tc], nan)
            self.counts = inside
            if ignore is not None:
                lp = torch.where(t == ignore, 0.0, lp)
                self.counts = inside & (t != ignore)
            self.logprobs, self.err_lp = lp, self.err_S + 4 * U * zf[rows, tc].abs()
        if top:
            order = torch.sort(torch.where(torch.isnan(raw), NEG, raw), dim=1, descending=True, stable=True).indices[:, :top]
            order = torch.nn.functional.pad(order, (0, top - order.shape[1]), value=-1)
            at = self.logp.gather(1, order.clamp(min=0)).masked_fill(order < 0, NEG)
            gone = (order < 0) | ~may.gather(1, order.clamp(min=0)) | self.broken[:, None]
            self.top_ids = order.masked_fill(gone, -1).to(torch.int32)
            self.top = at.masked_fill(gone, NEG).masked_fill(self.broken[:, None], float("nan"))
            self.err_top = self.err_S[:, None] + 4 * U * zf.gather(1, order.clamp(min=0)).abs()

    def grad(self, g_lp=None, g_h=None, g_top=None):
        """(gradient, tolerance without the rounding to the result's type)"""
        n, C = self.x.shape
        own = torch.zeros_like(self.p)
        rows = torch.arange(n, device=own.device)
        if g_lp is not None:
            own.index_put_((rows, self.t.long().clamp(0, C - 1)), g_lp.double() * self.counts, accumulate=True)
        if g_top is not None:
            for k in range(g_top.shape[1]):
                i = self.top_ids[:, k].long()
                own.index_put_((rows, i.clamp(min=0)), g_top[:, k].double() * (i >= 0), accumulate=True)
        b = torch.zeros(n, dtype=torch.float64, device=own.device) if g_h is None else g_h.double()
        A = own.sum(1)
        mag = own.abs().sum(1)
        w = A[:, None] + b[:, None] * (self.lf + self.H[:, None])
        dx = self.scale * (own - self.p * w)
        rel = self.err_S[:, None] + U * (4 * self.zf.abs() + 16)
        err_w = 8 * U * mag[:, None] + b.abs()[:, None] * (self.err_H + self.err_S + 4 * U * (self.H.abs() + 40))[:, None] \
            + 4 * U * b.abs()[:, None] * self.zf.abs().clamp(max=140)
        err = self.scale * (self.p * (w.abs() * rel + err_w) + 4 * U * own.abs() + 2.0 ** -126 * (mag + 200 * b.abs())[:, None])
        zero = (A == 0) & (b == 0) if g_lp is None and g_top is None else (mag == 0) & (b == 0)
        dx = torch.where(self.broken[:, None] & ~zero[:, None], float("nan"), dx)
        dx = torch.where(self.may & ~self.none[:, None], dx, 0.0)
        return dx, err

    def check(self, r, grad=None, weights=None):
        def same(got, ref, err, what):
            got = got.double()
            assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
            inf = torch.isinf(ref)
            assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], ref[inf]), what
            fine = torch.isfinite(ref)
            off = (got - ref).abs()[fine] - err[fine]
            assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()))
        same(r.entropy, self.entropy, self.err_H, "entropy")
        if self.t is not None:
            same(r.logprobs, self.logprobs, self.err_lp, "logprobs")
        else:
            assert r.logprobs is None
        if hasattr(self, "top_ids"):
            assert torch.equal(r.top_ids, self.top_ids)
            same(r.top_logprobs, self.top, self.err_top, "top")
        else:
            assert r.top_ids is None and r.top_logprobs is None
        if grad is not None:
            ref, err = self.grad(*weights)
            dt = grad.dtype
            assert dt is self.x.dtype and grad.shape == self.x.shape
            big = ref.abs() > torch.finfo(dt).max
            assert not bool(big.any())
            same(grad, ref, err * 1.01 + ref.abs() * (torch.finfo(dt).eps / 2) * (1 + 1e-6) + TINY[dt], "grad")


def _run(x, top=0, mask=None, scale=1.0, ignore=None, seed=5, targets=None, entropy=True):
    """Forward and gradient of a call with all weights, checked."""
    from trspmm import class_logprobs
    n, C = x.shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    if targets is None:
        targets = torch.randint(0, C, (n,), generator=g, device="cuda")
    w = [torch.randn(n, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda") if entropy else None,
         torch.randn(n, top, generator=g, device="cuda") if top else None]
    leaf = x.detach().requires_grad_()
    r = class_logprobs(leaf, targets, top=top, mask=mask, scale=scale, ignore_id=ignore)
    outs = [(o, k) for o, k in zip((r.logprobs, r.entropy, r.top_logprobs), w) if k is not None]
    grad, = torch.autograd.grad([o for o, _ in outs], leaf, [k for _, k in outs])
    ref = Ref(x, targets, top, mask, scale, ignore)
    ref.check(r, grad, w)
    return r, grad, ref


# ---- without a GPU ----------------------------------------------------------------------------------

def test_entries_refuse_bad_arguments_before_any_launch():
    from trspmm import _lib
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    a = (ctypes.addressof(buf) + 255) & ~255
    no = -(1 << 63)

    def fwd(x=a, ty=0, n=2, C=4, st=4, t=a, mask=None, ms=0, scale=1.0, top=0, lp=a, h=a, tl=None, ti=None, stats=a):
        return lib.trs_logprobs(x, ty, n, C, st, t, 1, no, mask, ms, scale, top, lp, h, tl, ti, stats, None)
    assert fwd(n=0) == 0
    for bad in (dict(x=None), dict(x=a + 2), dict(ty=3), dict(ty=-1), dict(n=-1), dict(C=0), dict(st=3), dict(t=None), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(top=-1), dict(top=1), dict(top=1, tl=a),
                dict(mask=a, ms=3), dict(stats=a + 4), dict(ty=1, x=a + 1), dict(t=a + 4), dict(lp=a + 2), dict(scale=3e38)):
        assert fwd(**bad) == -1, bad
    for big in (dict(n=1 << 31), dict(C=(1 << 30) + 1, st=1 << 31), dict(top=33, tl=a, ti=a)):
        assert fwd(**big) == -10, big

    def bwd(x=a, ty=0, n=2, C=4, st=4, t=a, top=0, ti=None, stats=a, h=a, gl=a, gh=None, gt=None, dx=a, ds=4):
        return lib.trs_logprobs_grad(x, ty, n, C, st, t, 1, no, None, 0, 1.0, top, ti, stats, h, gl, gh, gt, dx, ds, None)
    assert bwd(n=0) == 0
    for bad in (dict(x=None), dict(stats=None), dict(stats=a + 4), dict(dx=None), dict(dx=a + 1), dict(ds=3), dict(t=None), dict(gh=a, h=None),
                dict(gt=a), dict(gt=a, top=2), dict(gt=a, ti=a), dict(C=0)):
        assert bwd(**bad) == -1, bad


def test_python_entries_refuse_cpu_tensors():
    from trspmm import class_logprobs
    with pytest.raises(ValueError):
        class_logprobs(torch.ones(2, 4), torch.tensor([0, 1]))


# ---- sizes, types, layouts ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("C", [1, 2, 3, 7, 8, 9, 16, 31, 47, 64, 65, 100, 121, 128, 250, 255, 500, 505, 506, 1000, 1017, 1025, 2047, 2049, 4100, 16385])
def test_classes_and_types(C, dtype):
    x = _scores(37 if C > 300 else 301, C, dtype)
    _run(x, top=min(5, C))
    _run(x[:1], top=0, scale=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,C", [(1, 50021), (2, 131072), (1, 262147), (3, 70001), (150, 33000), (1, 1_000_003)])
def test_long_rows(n, C, dtype):
    _run(_scores(n, C, dtype, spread=3.0), top=8, scale=1.25)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [1, 2, 8, 31, 32])
@pytest.mark.parametrize("C", [4, 40, 300, 3000, 40000])
def test_numbers_of_alternatives(top, C):
    for dtype in (F32, F16):
        _run(_scores(9, C, dtype), top=top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("width,offset,C", [(64, 0, 47), (65, 3, 47), (1001, 1, 1000), (3001, 2, 2990), (50030, 5, 50021), (9000, 8, 8192)])
def test_rows_apart_and_on_any_boundary(width, offset, C, dtype):
    x = _scores(11, C, dtype, width=width, offset=offset)
    _run(x, top=3)
    from trspmm import class_logprobs, class_logprobs_grad
    # a strided result: nothing between its rows is written
    t = torch.zeros(11, dtype=torch.int32, device="cuda")
    r = class_logprobs(x, t)
    dst = torch.full((11, width), 7.0, dtype=dtype, device="cuda")
    g = torch.ones(11, device="cuda")
    got = class_logprobs_grad(x, t, r, g, out=dst[:, offset:offset + C])
    want = class_logprobs_grad(x.contiguous(), t, r, g)
    assert torch.equal(got, want)
    rest = torch.ones(width, dtype=torch.bool, device="cuda")
    rest[offset:offset + C] = False
    assert bool((dst[:, rest] == 7.0).all())


@pytest.mark.gpu
def test_far_rows():
    """Offsets past 2^31 elements."""
    from trspmm import class_logprobs, class_logprobs_grad
    n, C = 35_000, 65_536
    x = torch.zeros(n, C, dtype=F16, device="cuda")
    x[-1, 65_000] = 9.0
    t = torch.full((n,), 65_000, dtype=torch.int64, device="cuda")
    r = class_logprobs(x, t, top=2)
    assert torch.allclose(r.logprobs[:-1], torch.full((n - 1,), -11.090354888959125, device="cuda"), rtol=1e-6)
    assert r.top_ids[-1].tolist() == [65_000, 0] and r.top_ids[-2].tolist() == [0, 1]
    d = class_logprobs_grad(x, t, r, torch.ones(n, device="cuda"))
    ref, _ = Ref(x[-1:], t[-1:]).grad(torch.ones(1, device="cuda"))
    assert torch.allclose(d[-1:].double(), ref, rtol=2e-3, atol=1e-6)
    assert float(d[-2].float().max()) == 1.0


# ---- values -------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("C", [5, 47, 600, 5000, 66000])
@pytest.mark.parametrize("kind", ["equal", "ascending", "descending", "lowest", "one above", "zeros of both signs", "few values", "one part",
                                  "large", "half -inf"])
def test_values(kind, C, dtype):
    i = torch.arange(C, device="cuda", dtype=F32)
    low = torch.finfo(dtype).min
    x = {"equal": i * 0 + 3.5, "ascending": i / C * 8, "descending": -i / C * 8, "lowest": i * 0 + low,
         "one above": torch.where(i == C // 2, 50.0, -50.0), "zeros of both signs": torch.where(i % 2 == 0, -0.0, 0.0),
         "few values": (i * 7919) % 5, "large": 3e4 + 16 * ((i * 31) % 3), "half -inf": torch.where(i % 2 == 0, NEG, (i * 31) % 17),
         # the largest scores all in places that one thread of a strided loop has
         "one part": torch.where(i % 4096 < 8, 5 + (i * 31 % 1009) / 1009, -5.0)}[kind]
    x = x.to(dtype).expand(4, C).contiguous()
    if kind == "lowest":
        x[1, C // 3] = 0.0
        if C > 5:
            x[2, C // 4:] = NEG
    # (the entropy of scores 1e38 apart has no gradient in fp32: log p of the far ones is -1e38)
    _run(x, top=7, entropy=kind != "lowest")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("C", [5, 47, 600, 5000, 66000])
def test_masks_and_rows_with_nothing_left(C, dtype):
    g = torch.Generator(device="cuda").manual_seed(C)
    n = 23
    x = _scores(n, C, dtype)
    keep = torch.rand(n, C, generator=g, device="cuda") < 0.6
    keep[3] = False
    keep[4] = False
    keep[4, C - 1] = True
    keep[5] = False
    keep[5, 0] = True
    x = torch.where(keep, x, torch.tensor([float("nan"), float("inf"), NEG, torch.finfo(dtype).min], device="cuda")[
        torch.randint(0, 4, (n, C), generator=g, device="cuda")].to(dtype))
    x[6] = NEG
    r, grad, ref = _run(x, top=4, mask=keep)
    assert bool(ref.none[3]) and bool(ref.none[6]) and float(r.entropy[3]) == 0 and r.top_ids[3].tolist() == [-1] * 4
    assert float(grad[~keep].float().abs().max()) == 0 and float(grad[6].float().abs().max()) == 0
    _run(x, top=0, mask=keep, scale=2.0)
    # rows of the mask apart, and off any boundary
    wide = torch.zeros(n, C + 3, dtype=torch.bool, device="cuda")
    wide[:, 1:C + 1] = keep
    r2, grad2, _ = _run(x, top=4, mask=wide[:, 1:C + 1])
    assert torch.equal(grad, grad2) and torch.equal(r.entropy, r2.entropy)
    cls = keep[7]
    y = torch.where(cls, _scores(n, C, dtype, seed=3), torch.full((), float("nan"), dtype=dtype, device="cuda"))
    _run(y, top=4, mask=cls)
    _run(y, top=4, mask=cls & False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("C", [6, 47, 600, 5000, 66000])
def test_nan_and_infinite_scores(C, dtype):
    x = _scores(8, C, dtype)
    x[1, C - 1], x[2, 0], x[3, C // 2], x[4, 3] = float("nan"), float("inf"), NEG, float("nan")
    t = torch.tensor([0, 1, 2, C // 2, 5, 0, 1, C - 1], device="cuda")
    r, grad, _ = _run(x, top=3, targets=t)
    for k in (1, 2, 4):
        assert r.top_ids[k].tolist() == [-1] * 3 and bool(torch.isnan(r.entropy[k]))
    assert float(r.logprobs[3]) == NEG and float(grad[3, C // 2]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
@pytest.mark.parametrize("C", [7, 47, 3000, 40000])
def test_targets_ignored_outside_and_none(C, idt):
    from trspmm import class_logprobs, class_logprobs_grad
    x = _scores(10, C, F16)
    t = torch.tensor([0, -100, C, -1, C - 1, torch.iinfo(idt).max, torch.iinfo(idt).min, 1, 2, -100], device="cuda").to(idt)
    r, grad, _ = _run(x, top=2, targets=t, ignore=-100)
    assert float(r.logprobs[1]) == 0 and bool(torch.isnan(r.logprobs[2]))
    leaf = x.clone().requires_grad_()
    r = class_logprobs(leaf, t, ignore_id=-100)
    d, = torch.autograd.grad(r.logprobs, leaf, torch.ones(10, device="cuda"))
    for k in (1, 2, 3, 5, 6, 9):
        assert float(d[k].float().abs().max()) == 0
    _run(x, targets=t, ignore=0)
    assert class_logprobs(x).logprobs is None
    Ref(x, None, 3).check(class_logprobs(x, top=3))
    empty = class_logprobs(x[:0], t[:0], top=2)
    assert empty.logprobs.shape == (0,) and empty.top_ids.shape == (0, 2)
    assert class_logprobs_grad(x[:0], t[:0], empty, empty.logprobs).shape == (0, C)
    with pytest.raises(ValueError):
        class_logprobs_grad(x, None, class_logprobs(x), torch.ones(10, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("C", [5, 300, 5000])
def test_gradient_against_differences(C):
    """fp64 differences of the definition along a direction, against the kernel's fp32 gradient."""
    from trspmm import class_logprobs
    x = _scores(6, C, F32).requires_grad_()
    t = torch.arange(6, device="cuda") % C
    r = class_logprobs(x, t, top=2, scale=0.7)
    w = [_scores(6, 1, seed=k)[:, 0] for k in (1, 2)] + [_scores(6, 2, seed=3)]
    g, = torch.autograd.grad((r.logprobs, r.entropy, r.top_logprobs), x, w)
    d = _scores(6, C, seed=9).double()
    h = 1e-5

    def value(y):
        z = 0.7 * y
        lp = torch.log_softmax(z, 1)
        H = -(lp.exp() * lp).sum(1)
        return (lp.gather(1, t[:, None])[:, 0] * w[0].double() + H * w[1].double() + (lp.gather(1, r.top_ids.long()) * w[2].double()).sum(1))
    diff = (value(x.detach().double() + h * d) - value(x.detach().double() - h * d)) / (2 * h)
    _, err = Ref(x.detach(), t, 2, None, 0.7).grad(*w)
    tol = (err * d.abs()).sum(1) + (g.double() * d).abs().sum(1) * U + 1e-8 * (1 + d.abs().max() ** 3) * 40
    assert bool(((g.double() * d).sum(1) - diff).abs().le(tol).all())


@pytest.mark.gpu
def test_refusals():
    from trspmm import class_logprobs, class_logprobs_grad
    x, t = _scores(4, 10, F16), torch.zeros(4, dtype=torch.int64, device="cuda")
    r = class_logprobs(x, t, top=2)
    one = torch.ones(4, device="cuda")
    for call in (lambda: class_logprobs(x.double(), t), lambda: class_logprobs(x, t.float()), lambda: class_logprobs(x, t, mask=t)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: class_logprobs(x[0], t), lambda: class_logprobs(x[:, :0], t), lambda: class_logprobs(x.t(), t),
                 lambda: class_logprobs(x[:1].expand(4, 10), t), lambda: class_logprobs(x, t[:3]), lambda: class_logprobs(x, t.cpu()),
                 lambda: class_logprobs(x, t, top=33), lambda: class_logprobs(x, t, top=-1), lambda: class_logprobs(x, t, scale=0.0),
                 lambda: class_logprobs(x, t, scale=float("nan")), lambda: class_logprobs(x, t, mask=torch.ones(9, dtype=torch.bool, device="cuda")),
                 lambda: class_logprobs(x, t, mask=torch.ones(3, 10, dtype=torch.bool, device="cuda")),
                 lambda: class_logprobs(x, t, mask=torch.ones(4, 10, dtype=torch.bool)),
                 lambda: class_logprobs_grad(x, t, r, one.half()), lambda: class_logprobs_grad(x, t, r, one[:3]),
                 lambda: class_logprobs_grad(x, t, r, one, out=x), lambda: class_logprobs_grad(x, t, r, one, out=x.float()),
                 lambda: class_logprobs_grad(x, t, r, g_top_logprobs=torch.ones(4, 3, device="cuda")),
                 lambda: class_logprobs_grad(x, t, class_logprobs(x, t), g_top_logprobs=torch.ones(4, 2, device="cuda"))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("n,C", [(500, 47), (3, 70001), (40, 3001)])
def test_streams_graphs_and_repeats(n, C):
    from trspmm import class_logprobs, class_logprobs_grad
    x, t = _scores(n, C, F16), torch.arange(n, device="cuda") % C
    g = torch.ones(n, device="cuda")

    def both():
        r = class_logprobs(x, t, top=4)
        return (*r, class_logprobs_grad(x, t, r, g, g, torch.ones(n, 4, device="cuda")))
    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    x.copy_(_scores(n, C, F16, seed=8))
    want = both()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.gpu
@pytest.mark.parametrize("C", [6, 47, 600, 5000, 66000])
def test_rows_without_a_distribution_are_nan_wherever_they_lie(C):
    """A NaN beside scores of -inf: the gradient is NaN in every place that is not masked, whichever alignment the row has."""
    from trspmm import class_logprobs, class_logprobs_grad
    for offset in (0, 1, 3):
        x = _scores(5, C, F16, width=C + 8, offset=offset)
        x[:, 1::2] = NEG
        x[:, C - 2] = float("nan")
        r = class_logprobs(x)
        assert bool(torch.isnan(r.entropy).all())
        keep = torch.arange(C, device="cuda") % 4 != 3
        for mask in (None, keep):
            d = class_logprobs_grad(x, None, class_logprobs(x, mask=mask), g_entropy=torch.ones(5, device="cuda"), mask=mask)
            broken = mask is None or bool(keep[C - 2])
            if mask is None:
                assert bool(torch.isnan(d).all())
            elif broken:
                assert bool(torch.isnan(d[:, keep]).all()) and float(d[:, ~keep].float().abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("C", [5, 47, 200, 500, 1000, 5000])
def test_fp32_scores_that_differ_in_their_last_bits(C):
    """The order of alternatives goes by all bits of a score, whatever part of them a comparison starts with."""
    from trspmm import class_logprobs
    i = torch.arange(C, device="cuda")
    x = torch.stack([1.0 + ((i * 7919) % 61).float() * 2.0 ** -23, 1.0 + (i % 61).float() * 2.0 ** -23, -1.0 - (i % 61).float() * 2.0 ** -23,
                     torch.where(i % 2 == 0, 1.0, 1.0 + 2.0 ** -23), (i % 3).float() * 2.0 ** -126])
    for top in (1, 4, 32):
        Ref(x, None, top).check(class_logprobs(x, top=top))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("C", [4, 7, 47, 255, 600, 1025, 5000, 66000])
@pytest.mark.parametrize("layout", ["plain", "apart", "masked"])
def test_weights_of_a_row_that_cancel(C, dtype, layout):
    """Margins: the weights of a row's target and alternatives add up to 0 (small whole numbers: exactly), and are not 0."""
    from trspmm import class_logprobs, class_logprobs_grad
    n = 30
    x = _scores(n, C, dtype, width=C + 3 if layout == "apart" else None, offset=1 if layout == "apart" else 0)
    g = torch.Generator(device="cuda").manual_seed(C)
    mask = None
    if layout == "masked":
        mask = torch.rand(n, C, generator=g, device="cuda") < 0.7
        mask[7], mask[8] = False, False
        mask[8, C - 1] = True
        x = torch.where(mask, x, float("nan"))
    targets = torch.randint(0, C, (n,), generator=g, device="cuda")
    best = Ref(x, targets, 2, mask).top_ids.long()
    targets[10:15], targets[15:20] = best[10:15, 0].clamp(min=0), best[15:20, 1].clamp(min=0)   # the target is an alternative too
    kinds = torch.tensor([[0, 1, -1, 0], [1, -1, 0, 0], [2, -1, -1, 0], [-3, 1, 1, 1], [1, 0, 0, -1]], dtype=F32, device="cuda")
    w = kinds.repeat(n // 5, 1)
    w[29] = 0
    g_lp, g_top = w[:, 0].contiguous(), w[:, 1:].contiguous()
    some = torch.where(torch.arange(n, device="cuda") % 3 == 0, 0.5, 0.0)
    for g_h in (None, some):
        leaf = x.detach().requires_grad_()
        r = class_logprobs(leaf, targets, top=3, mask=mask, scale=1.25)
        outs = (r.logprobs, r.top_logprobs) if g_h is None else (r.logprobs, r.top_logprobs, r.entropy)
        grad, = torch.autograd.grad(outs, leaf, (g_lp, g_top) if g_h is None else (g_lp, g_top, g_h))
        Ref(x, targets, 3, mask, 1.25).check(r, grad, (g_lp, g_h, g_top))
        assert torch.equal(grad, class_logprobs_grad(x, targets, r, g_lp, g_h, g_top, mask, 1.25))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("C", [6, 47, 600, 5000, 66000])
def test_alternatives_alone_of_rows_without_a_distribution(C, dtype):
    """Where the forward call gave NaN, so does the gradient of its alternatives - in every place that is not masked, and unless all
    weights are 0."""
    from trspmm import class_logprobs
    x = _scores(7, C, dtype)
    x[1, C - 1], x[2, 0], x[3, C // 2], x[4, 3], x[5, 2] = float("nan"), float("inf"), float("nan"), float("inf"), float("nan")
    keep = torch.ones(7, C, dtype=torch.bool, device="cuda")
    keep[:, 1] = False
    keep[5, 2] = False   # its NaN is masked
    keep[6] = False
    w = torch.tensor([[1, 2], [1, 2], [1, -1], [0, 3], [0, 0], [1, 2], [1, 2]], dtype=F32, device="cuda")
    for mask in (None, keep):
        broken = [1, 2, 3] + ([5] if mask is None else [])
        leaf = x.clone().requires_grad_()
        r = class_logprobs(leaf, top=2, mask=mask)
        d, = torch.autograd.grad(r.top_logprobs, leaf, w)
        for k in range(7):
            may = torch.ones_like(keep[k]) if mask is None else mask[k]
            assert bool((torch.isnan(d[k]) == (may & (k in broken))).all()), (k, mask is None)
            assert k in broken or k in (0, 5) or (k == 6 and mask is None) or float(d[k].float().abs().max()) == 0


@pytest.mark.gpu
def test_forward_mode_is_refused():
    """A tangent is not dropped in silence, whichever operand has it."""
    import torch.autograd.forward_ad as fw
    from trspmm import class_logprobs, class_logprobs_grad
    x, t, one = _scores(4, 10, F32), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.ones(4, device="cuda")
    r = class_logprobs(x, t, top=2)
    two = torch.ones(4, 2, device="cuda")
    with fw.dual_level():
        def dual(v):
            return fw.make_dual(v.clone(), torch.ones_like(v))
        for call in (lambda: class_logprobs(dual(x), t), lambda: class_logprobs(dual(x), top=1),
                     lambda: class_logprobs_grad(dual(x), t, r, one), lambda: class_logprobs_grad(x, t, r, dual(one)),
                     lambda: class_logprobs_grad(x, t, r, g_entropy=dual(one)), lambda: class_logprobs_grad(x, t, r, g_top_logprobs=dual(two)),
                     lambda: class_logprobs_grad(x, t, r._replace(stats=dual(r.stats)), one),
                     lambda: class_logprobs_grad(x, t, r._replace(entropy=dual(r.entropy)), g_entropy=one),
                     lambda: class_logprobs_grad(x, t, r, one, out=dual(x))):
            with pytest.raises(RuntimeError):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError):
                call()
        leaf = x.clone().requires_grad_()
        y = class_logprobs(leaf, t)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y.logprobs, leaf, dual(one))
        assert torch.equal(class_logprobs(x, t).logprobs, r.logprobs)


@pytest.mark.gpu
def test_a_gradient_written_in_place_is_noticed_by_autograd():
    """out= changes a tensor that a graph may have kept: its backward pass raises as after any change in place."""
    from trspmm import class_logprobs, class_logprobs_grad
    x, t = _scores(4, 10, F32), torch.zeros(4, dtype=torch.int64, device="cuda")
    w = torch.ones(4, 10, device="cuda", requires_grad=True)
    kept = torch.ones(4, 10, device="cuda")
    y = w * kept
    class_logprobs_grad(x, t, class_logprobs(x, t), torch.ones(4, device="cuda"), out=kept)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(ValueError):
        class_logprobs_grad(x, t, class_logprobs(x, t), torch.ones(4, device="cuda"), out=w)


@pytest.mark.gpu
def test_ids_that_64_bits_do_not_hold_are_refused():
    """They do not come back as other classes."""
    from trspmm import class_logprobs, class_logprobs_grad
    x, t, one = _scores(4, 10, F32), torch.tensor([0, 3, 2, 0], device="cuda"), torch.ones(4, device="cuda")
    r = class_logprobs(x, t)
    for bad in (1 << 64, (1 << 64) + 3, 1 << 63, -(1 << 63), -(1 << 64) + 1):
        for call in (lambda: class_logprobs(x, t, ignore_id=bad), lambda: class_logprobs_grad(x, t, r, one, ignore_id=bad)):
            with pytest.raises(ValueError):
                call()
    for far in ((1 << 63) - 1, 1 - (1 << 63)):
        assert torch.equal(class_logprobs(x, t, ignore_id=far).logprobs, r.logprobs)


@pytest.mark.gpu
def test_a_gradient_over_what_the_call_reads_is_refused():
    """Rows are written while others still read their weights."""
    from trspmm import class_logprobs, class_logprobs_grad
    x, one = _scores(4, 10, F32), torch.ones(4, device="cuda")
    t, mask = torch.tensor([0, 3, 2, 0], device="cuda"), torch.ones(4, 10, dtype=torch.bool, device="cuda")
    r = class_logprobs(x, t, top=2, mask=mask)
    two = torch.ones(4, 2, device="cuda")

    def into(**what):   # all arguments apart from the one that lies in the result's memory
        out = torch.zeros(4, 10, device="cuda")
        a = dict(t=t, g=one, h=one, k=two, mask=mask, entropy=r.entropy, top_ids=r.top_ids, stats=r.stats)
        for name in what:
            v = a[name]
            place = out.view(-1).view(v.dtype)[2:2 + v.numel()].view(v.shape)
            a[name] = place.copy_(v)
        return class_logprobs_grad(x, a["t"], r._replace(entropy=a["entropy"], top_ids=a["top_ids"], stats=a["stats"]), a["g"], a["h"], a["k"],
                                   a["mask"], out=out)
    assert torch.equal(into(), class_logprobs_grad(x, t, r, one, one, two, mask))
    for name in ("t", "g", "h", "k", "mask", "entropy", "top_ids", "stats"):
        with pytest.raises(ValueError):
            into(**{name: True})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("C", [3, 17, 20, 47, 100, 200, 300, 480, 900])
@pytest.mark.parametrize("layout", ["plain", "apart", "masked"])
def test_many_short_rows(C, dtype, layout):
    """So many rows that a group of lanes does several of them one after the other, the last group fewer."""
    from trspmm import class_logprobs, class_logprobs_grad
    pieces = (C + 16 // dtype.itemsize - 1 + 16 // dtype.itemsize - 1) * dtype.itemsize // 16
    n = (606_208 if pieces * 16 // dtype.itemsize <= 128 else 303_104 if pieces * 16 // dtype.itemsize <= 256 else 151_552) + 3
    g = torch.Generator(device="cuda").manual_seed(C)
    x = _scores(n, C, dtype, width=C + 3 if layout == "apart" else None, offset=1 if layout == "apart" else 0)
    mask = None
    if layout == "masked":
        mask = torch.rand(n, C, generator=g, device="cuda") < 0.7
        mask[5::11] = False
    t = torch.randint(0, C, (n,), generator=g, device="cuda")
    t[::7] = -1
    top = min(C, 4)
    w = [torch.randn(n, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda"), torch.randn(n, top, generator=g, device="cuda")]
    r = class_logprobs(x, t, top=top, mask=mask, scale=0.75, ignore_id=-1)
    d = class_logprobs_grad(x, t, r, *w, mask=mask, scale=0.75, ignore_id=-1)
    pick = torch.cat([torch.arange(2000), torch.arange(n - 2000, n), torch.randint(0, n, (2000,))]).cuda()
    part = type(r)(*[v[pick] for v in r])
    Ref(x[pick], t[pick], top, None if mask is None else mask[pick], 0.75, -1).check(part, d[pick], [v[pick] for v in w])
    # the other rows: the same bits as by calls of few rows, in which a group has one
    for a in range(0, n, 100_000):
        b = min(a + 100_000, n)
        m = None if mask is None else mask[a:b]
        few = class_logprobs(x[a:b], t[a:b], top=top, mask=m, scale=0.75, ignore_id=-1)
        assert all(torch.equal(p.view(torch.int32), q[a:b].view(torch.int32)) for p, q in zip(few, r))
        again = class_logprobs_grad(x[a:b], t[a:b], few, *[v[a:b] for v in w], mask=m, scale=0.75, ignore_id=-1)
        assert torch.equal(again.view(torch.int16), d[a:b].view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n,C", [(4739, 1100), (4739, 2000), (2371, 6000), (1187, 30_000), (600, 70_001)])
def test_many_long_rows(n, C, dtype):
    """So many rows that each has few threads, down to one warp; values that crowd the alternatives' lists."""
    from trspmm import class_logprobs, class_logprobs_grad
    i = torch.arange(C, device="cuda")
    vec = 16 // dtype.itemsize
    g = torch.Generator(device="cuda").manual_seed(C)
    for kind in ("random", "equal", "few values", "one lane", "one lane, equal", "masked", "apart"):
        x = _scores(n, C, dtype, width=C + 5 if kind == "apart" else None, offset=3 if kind == "apart" else 0)
        mask = None
        lane = i // vec % 32 == 5   # places that one thread of a warp has
        if kind == "equal":
            x.fill_(2.5)
        elif kind == "few values":
            x.copy_(((i * 7919) % 5).to(dtype))
        elif kind == "one lane":
            x[:, lane] += 20
        elif kind == "one lane, equal":
            x[:, lane] = 20
        elif kind == "masked":
            mask = torch.rand(n, C, generator=g, device="cuda") < 0.7
            mask[3::5] = False
        t = torch.randint(0, C, (n,), generator=g, device="cuda")
        t[::7] = -1
        w = [torch.randn(n, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda"), torch.randn(n, 9, generator=g, device="cuda")]
        r = class_logprobs(x, t, top=9, mask=mask, ignore_id=-1)
        d = class_logprobs_grad(x, t, r, *w, mask=mask, ignore_id=-1)
        for pick in (torch.arange(100, device="cuda"), torch.arange(n - 100, n, device="cuda")):
            part = type(r)(*[v[pick] for v in r])
            Ref(x[pick], t[pick], 9, None if mask is None else mask[pick], 1.0, -1).check(part, d[pick], [v[pick] for v in w])
