"""Linear cross entropy and its first and second gradients against their
formulas in float64, element by element (bounds: tests/_ops_util.py)."""
import pytest
import torch

from tests._ops_util import lce_ref, within
from testtimeideas_amd.ttt_e2e import linear_cross_entropy

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _inputs(n, d, v, dtype, seed, masked=False, ignored=False):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    w = (rn(v, d) * 2 / d ** 0.5).to(dtype)
    t = torch.randint(0, v, (n,), generator=g)
    x = (rn(n, d) + w[t].float()).to(dtype)
    wt = torch.ones(n)
    if masked:
        wt = (torch.rand(n, generator=g) < 0.7).float() * (0.5 + torch.rand(n, generator=g))
    if ignored:
        t[torch.rand(n, generator=g) < 0.3] = -100
    return dict(x=x, w=w, t=t, mask=wt if masked else None, a=rn(n, d).to(dtype), b=(rn(v, d) / n ** 0.5).to(dtype))


def _weights(s):
    wt = torch.ones(len(s["t"])) if s["mask"] is None else s["mask"]
    return torch.where(s["t"] == -100, 0.0, wt).double()


def _run(s, names=("a", "b"), reduction="mean", up=None, up_grad=True):
    """up_grad: the incoming gradient asks for its own (another way to form h)."""
    x, w = s["x"].cuda().requires_grad_(), s["w"].cuda().requires_grad_()
    mask = None if s["mask"] is None else s["mask"].cuda()
    loss = linear_cross_entropy(x, w, s["t"].cuda(), mask, reduction=reduction)
    up = (torch.ones_like(loss) if up is None else up.cuda()).requires_grad_(up_grad)
    first = torch.autograd.grad(loss, (x, w), up, create_graph=True)
    pairs = [(f, s[k].cuda()) for f, k in zip(first, ("a", "b")) if k in names]
    second = torch.autograd.grad([p[0] for p in pairs], (x, w, up) if up_grad else (x, w), [p[1] for p in pairs])
    loss_name, up_name = ("rows", "gup") if reduction == "none" else ("loss", "gloss")
    return dict(zip((loss_name, "dx", "dw", "gx", "gw", up_name), (loss, *first, *second)))


def _check(s, got, names=("a", "b"), reduction="mean", up=1.0):
    wt = _weights(s)
    inv = 1 / max(float(wt.sum()), 1.0) if reduction == "mean" else 1.0
    d = {k: s[k].double() for k in ("x", "w", "a", "b")}
    ref, bound = lce_ref(d["x"], d["w"], s["t"], wt, up, inv, s["x"].dtype, *(d[k] if k in names else None
                                                                              for k in ("a", "b")))
    for k, v in got.items():
        within(k, v, ref[k], bound[k])


SIZES = [(1, 1, 1), (1, 512, 4096), (1, 64, 1000), (2, 3, 5), (7, 24, 33), (65, 40, 130), (128, 64, 128),
         (129, 72, 257), (300, 200, 1003), (257, 131, 511), (1024, 384, 512), (1000, 64, 4099), (33, 1032, 600)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,d,v", SIZES)
def test_values_and_both_gradients(n, d, v, dtype):
    s = _inputs(n, d, v, dtype, seed=n + d + v)
    _check(s, _run(s))
    _check(s, _run(s, up_grad=False))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions_masks_and_ignored_rows(reduction, dtype):
    s = _inputs(200, 80, 300, dtype, seed=1, masked=True, ignored=True)
    up = torch.rand(200, generator=torch.Generator().manual_seed(2)) if reduction == "none" else torch.tensor(0.7)
    got = _run(s, reduction=reduction, up=up)
    _check(s, got, reduction=reduction, up=up.double())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("names", [("a",), ("b",)])
def test_one_cotangent(names, dtype):
    """The second gradient through dx or dw alone (the other may not exist)."""
    s = _inputs(150, 64, 260, dtype, seed=3, masked=True)
    x, w = s["x"].cuda().requires_grad_(), s["w"].cuda().requires_grad_()
    loss = linear_cross_entropy(x, w, s["t"].cuda(), s["mask"].cuda())
    wrt, k = ((x,), "a") if names == ("a",) else ((w,), "b")
    first = torch.autograd.grad(loss, wrt, create_graph=True)
    gx, gw = torch.autograd.grad(first, (x, w), [s[k].cuda()])
    _check(s, dict(gx=gx, gw=gw, **{"dx" if k == "a" else "dw": first[0]}), names=names)


def test_second_gradient_of_one_operand():
    s = _inputs(70, 48, 90, torch.float32, seed=4)
    both = _run(s)
    for k, other in (("x", "w"), ("w", "x")):
        t = {j: s[j].cuda() for j in ("x", "w")}
        t[k].requires_grad_()
        first, = torch.autograd.grad(linear_cross_entropy(t["x"], t["w"], s["t"].cuda()), (t[k],), create_graph=True)
        assert torch.equal(first, both["d" + k])
        got, = torch.autograd.grad(first, (t[k],), s["a" if k == "x" else "b"].cuda())
        _check(s, {"g" + k: got}, names=("a",) if k == "x" else ("b",))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_pieces_of_the_vocabulary(dtype):
    """Enough rows times vocabulary that the gradients run in several pieces,
    the last one short."""
    s = _inputs(8200, 24, 33001, dtype, seed=5, ignored=True)
    _check(s, _run(s))
    _check(s, _run(s, up_grad=False))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [70001, 300001], ids=["one", "merged"])
def test_large_vocabulary_of_few_rows(vocab, dtype):
    """More vocabulary than a piece has, and more of its tiles' statistics than
    are kept before they are merged."""
    s = _inputs(3, 16, vocab, dtype, seed=6)
    _check(s, _run(s))


@pytest.mark.parametrize("n", [1, 2, 5, 31, 32, 33, 63, 64, 65, 129])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_rows_of_the_joins(n, reduction):
    """Each way in which a row's parts are read, and its last workgroup."""
    s = _inputs(n, 40, 3000, torch.bfloat16, seed=60 + n, masked=n > 2)
    up = torch.ones(n) if reduction == "none" else torch.tensor(1.0)
    _check(s, _run(s, reduction=reduction, up=up), reduction=reduction, up=up.double())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_that_do_not_count_may_hold_anything(dtype):
    s = _inputs(140, 64, 200, dtype, seed=7, masked=True, ignored=True)
    dead = _weights(s) == 0
    clean = [_run(s, up_grad=u) for u in (True, False)]
    s["x"][dead] = float("nan")
    s["x"][dead.nonzero()[0]] = float("inf")
    s["a"][dead] = float("nan")
    for u in (True, False):
        got = _run(s, up_grad=u)
        for k in got:
            assert torch.equal(got[k], clean[1 - u][k]), k
        assert not got["dx"][dead.cuda()].any() and not got["gx"][dead.cuda()].any()


@pytest.mark.parametrize("how", ["ignored", "masked"])
def test_no_row_counts(how):
    s = _inputs(30, 32, 50, torch.bfloat16, seed=8)
    if how == "ignored":
        s["t"][:] = -100
    else:
        s["mask"] = torch.zeros(30)
    got = _run(s)
    assert all(not v.any() for v in got.values())


def test_no_rows():
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    w = torch.randn(20, 16, device="cuda", requires_grad=True)
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    for reduction in ("none", "sum", "mean"):
        loss = linear_cross_entropy(x, w, t, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss), create_graph=True)
        gw, = torch.autograd.grad(dw, (w,), torch.ones_like(dw))
        assert dx.shape == (0, 16) and not dw.any() and not gw.any() and not loss.any()


def test_ignore_index_inside_the_vocabulary():
    s = _inputs(60, 32, 40, torch.float32, seed=9)
    got = linear_cross_entropy(s["x"].cuda(), s["w"].cuda(), s["t"].cuda(), ignore_index=int(s["t"][0]),
                               reduction="none")
    ref = linear_cross_entropy(s["x"].cuda(), s["w"].cuda(), s["t"].cuda(), reduction="none")
    same = s["t"] == s["t"][0]
    assert torch.equal(got, ref.masked_fill(same.cuda(), 0.0))


@pytest.mark.parametrize("bad", [-1, 40, 2 ** 32 + 3, -2 ** 40])
def test_a_target_outside_the_vocabulary_is_nan(bad):
    s = _inputs(10, 32, 40, torch.bfloat16, seed=10)
    s["t"][4] = bad
    x, w = s["x"].cuda().requires_grad_(), s["w"].cuda().requires_grad_()
    rows = linear_cross_entropy(x, w, s["t"].cuda(), reduction="none")
    assert rows[4].isnan() and not rows[[0, 1, 2, 3, 5, 6, 7, 8, 9]].isnan().any()
    dx, dw = torch.autograd.grad(rows.sum(), (x, w))
    assert dx[4].isnan().all() and not dx[:4].isnan().any() and dw.isnan().all()
    assert linear_cross_entropy(x, w, s["t"].cuda()).isnan()


def test_large_logits():
    """Logits of some hundreds: the running maximum keeps them finite."""
    s = _inputs(64, 96, 300, torch.float32, seed=11)
    s["x"] *= 60.0
    _check(s, _run(s))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_upstream_of_any_size(dtype):
    """fp16 holds the pieces scaled: neither a large nor a tiny upstream gradient loses them."""
    s = _inputs(90, 64, 120, dtype, seed=12)
    for up in (2.0 ** 10, 2.0 ** -10):
        _check(s, _run(s, up=torch.tensor(up)), up=up)


def test_strides_and_leading_shape():
    g = torch.Generator().manual_seed(13)
    base = torch.randn(6, 10, 96, generator=g).cuda().bfloat16()
    w = torch.randn(70, 100, generator=g).cuda().bfloat16()
    for v, ww in ((base[..., 8:72], w[:, :64]), (base.transpose(0, 1)[..., :64], w[:, 1:65]),
                  (base[:, :1, :64].expand(6, 10, 64), w[:, 36:]), (base[..., 3:30], w[::2, 5:32]),
                  (base[2, 3, :40], w[:, :40])):
        t = torch.randint(0, ww.shape[0], v.shape[:-1], generator=g).cuda()
        outs = []
        for x, h in ((v, ww), (v.clone(memory_format=torch.contiguous_format),
                               ww.clone(memory_format=torch.contiguous_format))):
            x, h = x.detach().requires_grad_(), h.detach().requires_grad_()
            loss = linear_cross_entropy(x, h, t, reduction="none")
            assert loss.shape == t.shape and loss.dtype == torch.float32
            dx, dw = torch.autograd.grad(loss.sum(), (x, h), create_graph=True)
            outs.append((loss, dx, dw, *torch.autograd.grad((dx.float().square().sum() + dw.float().square().sum()),
                                                            (x, h))))
        assert all(torch.equal(p, q) for p, q in zip(*outs))


def test_python_refusals_on_the_gpu():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(16, 8, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    bad = [(ValueError, (x, w[:, :7], t), {}), (ValueError, (x, w.half(), t), {}), (TypeError, (x, w, t.int()), {}),
           (ValueError, (x, w, t[:3]), {}), (ValueError, (x, w, t.cpu()), {}), (ValueError, (x, w, t), {"reduction": "max"}),
           (ValueError, (x, w, t, torch.ones(3, device="cuda")), {}), (ValueError, (x, w.cpu(), t), {}),
           (TypeError, (x.double(), w.double(), t), {}), (ValueError, (x, w[:0], t), {}),
           (TypeError, (x, w, t, torch.ones(4, device="cuda", dtype=torch.complex64)), {})]
    for err, args, kw in bad:
        with pytest.raises(err):
            linear_cross_entropy(*args, **kw)
    with pytest.raises(RuntimeError, match="2\\^16"):
        linear_cross_entropy(torch.zeros(1, 65544, device="cuda"), torch.zeros(2, 65544, device="cuda"), t[:1])


def test_repeats_bitwise():
    s = _inputs(700, 120, 900, torch.bfloat16, seed=14, masked=True)
    for u in (True, False):
        one, two = _run(s, up_grad=u), _run(s, up_grad=u)
        assert all(torch.equal(one[k], two[k]) for k in one)


def test_no_upstream_gradient():
    """Upstream 0: gradients 0, but the gradient of the upstream itself is not."""
    s = _inputs(50, 64, 80, torch.bfloat16, seed=20)
    got = _run(s, up=torch.tensor(0.0))
    _check(s, {k: got[k] for k in ("loss", "gloss")}, up=0.0)
    assert not any(got[k].any() for k in ("dx", "dw", "gx", "gw")) and got["gloss"] != 0


def test_third_derivative_raises():
    s = _inputs(8, 16, 20, torch.float32, seed=15)
    x, w = s["x"].cuda().requires_grad_(), s["w"].cuda().requires_grad_()
    dx, = torch.autograd.grad(linear_cross_entropy(x, w, s["t"].cuda()), (x,), create_graph=True)
    gx, = torch.autograd.grad(dx.square().sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        torch.autograd.grad(gx.sum(), (x,))


def test_gradient_against_differences():
    """Both gradients against central differences, step 2^-7: off by its
    square times the third differences (of the order of the sums of
    magnitudes here), and by the rounding of the differences."""
    s = _inputs(6, 20, 15, torch.float32, seed=16)
    w, t, a = s["w"].cuda(), s["t"].cuda(), s["a"].cuda()
    v = torch.randn(6, 20, generator=torch.Generator().manual_seed(17)).cuda()
    h = 2.0 ** -7

    def slope(x):
        x = x.detach().requires_grad_()
        loss = linear_cross_entropy(x, w, t, reduction="sum")
        dx, = torch.autograd.grad(loss, (x,), create_graph=True)
        return loss, (dx * a).sum(), dx, x

    x0 = s["x"].cuda()
    loss, f, dx, x = slope(x0)
    gx, = torch.autograd.grad(f, (x,))
    up, down = slope(x0 + h * v), slope(x0 - h * v)
    reach = float((v.abs() @ w.abs().t()).max()) ** 3 * 6
    assert abs(float((dx * v).sum() - (up[0] - down[0]) / (2 * h))) <= h * h * reach + 2.0 ** -20 / h * float(loss.abs() + 1)
    reach *= float((a.abs() @ w.abs().t()).max())
    assert abs(float((gx * v).sum() - (up[1] - down[1]) / (2 * h))) <= h * h * reach + 2.0 ** -20 / h * float(f.abs() + 1)


def test_graph_replays():
    s = _inputs(260, 64, 700, torch.bfloat16, seed=18, masked=True)
    x, w, t, mask, a, b = (s[k].cuda() for k in ("x", "w", "t", "mask", "a", "b"))
    x.requires_grad_(), w.requires_grad_()

    def step():
        loss = linear_cross_entropy(x, w, t, mask)
        first = torch.autograd.grad(loss, (x, w), create_graph=True)
        return [loss, *first, *torch.autograd.grad(first, (x, w), (a, b))]

    with torch.autograd.set_multithreading_enabled(False):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        ref = [r.detach().clone() for r in step()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for _ in range(3):
            for o in out:
                o.detach().fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, r) for o, r in zip(out, ref))
            step()
            torch.cuda.synchronize()


def test_another_stream():
    s = _inputs(300, 64, 500, torch.float16, seed=19)
    ref = _run(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _run(s)
    side.synchronize()
    assert all(torch.equal(got[k], ref[k]) for k in ref)


def test_nan_stays_in_its_row():
    s = _inputs(70, 64, 300, torch.bfloat16, seed=30)
    bad = dict(s, x=s["x"].clone())
    bad["x"][5, 3] = float("nan")
    keep = torch.arange(70) != 5
    for u in (True, False):
        clean, got = (_run(t, reduction="none", up=torch.ones(70), names=("a",), up_grad=u) for t in (s, bad))
        for k in ("rows", "dx", "gx"):
            assert torch.equal(got[k][keep.cuda()], clean[k][keep.cuda()]), k
            assert got[k][5].isnan().all(), k


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_one_tensor_as_both_operands(dtype):
    """hidden and weight the same leaf: its gradients are the two operands' sums."""
    s = _inputs(60, 48, 60, dtype, seed=31)
    s["x"] = s["w"].clone()
    apart = _run(s, up_grad=False)
    t = s["w"].cuda().requires_grad_()
    loss = linear_cross_entropy(t, t, s["t"].cuda())
    dt, = torch.autograd.grad(loss, (t,), create_graph=True)
    within("dt", dt, (apart["dx"].double() + apart["dw"].double()).cpu(),
           torch.finfo(dtype).eps / 2 * (apart["dx"].double() + apart["dw"].double()).abs().cpu() + 1e-30)
    # one cotangent serves both: gx and gw of a = b
    s["b"] = s["a"]
    apart = _run(s, up_grad=False)
    gt, = torch.autograd.grad(dt, (t,), s["a"].cuda())
    want = apart["gx"].double() + apart["gw"].double()
    within("gt", gt, want.cpu(), torch.finfo(dtype).eps / 2 * want.abs().cpu() + 1e-30)


def test_offsets_past_32_bits():
    """A head of more than 2^31 values, zero but for its first and last rows:
    against the formulas with the zero rows counted."""
    n, d, v, k = 4, 4096, 600000, 3
    g = torch.Generator().manual_seed(32)
    ends = (torch.randn(2 * k, d, generator=g) * 2 / d ** 0.5).bfloat16()
    x = torch.randn(n, d, generator=g).bfloat16()
    rows = torch.tensor([0, 1, 2, v - 3, v - 2, v - 1, v // 2])  # the ends and one row of zeros
    at = torch.tensor([4, 5, 0, 6])  # the targets' places among them
    w = torch.zeros(v, d, dtype=torch.bfloat16, device="cuda")
    w[:k], w[-k:] = ends[:k].cuda(), ends[k:].cuda()
    w.requires_grad_()
    xd = x.cuda().requires_grad_()
    loss = linear_cross_entropy(xd, w, rows[at].cuda())
    dx, dw = torch.autograd.grad(loss, (xd, w))

    x, we = x.double(), torch.cat([ends.double(), torch.zeros(1, d).double()])
    z = x @ we.T
    lse = torch.log(z[:, :-1].exp().sum(1) + (v - 2 * k))
    grad = (z - lse[:, None]).exp()
    grad[torch.arange(n), at] -= 1
    grad /= n
    # products of d terms in fp32 make z, whose error is p's relative one; G and the results are rounded to bf16
    ez = d * 2.0 ** -24 * (x.abs() @ we.abs().T).max().item()
    unit = 2.0 ** -8
    within("loss", loss, (lse - z[torch.arange(n), at]).mean(), torch.tensor(2 * ez + 1e-5))
    within("dx", dx, grad @ we, (2 * unit + 2 * ez) * (grad.abs() @ we.abs()) + 1e-30)
    within("dw", dw[rows.cuda()], grad.T @ x, (2 * unit + 2 * ez) * (grad.abs().T @ x.abs()) + 1e-30)
    # the zero rows in between all have the same gradient
    other = (-lse).exp() / n
    for j in (k, 524288, 599000):
        within(f"dw[{j}]", dw[j], other @ x, (2 * unit + 2 * ez) * (other.abs() @ x.abs()) + 1e-30)


def test_fp32_errors_have_no_common_sign():
    """Sums over many rows would gather one.  The rows' errors are independent,
    so their mean is within four deviations, 4 / sqrt(rows) of their root mean
    square."""
    n = 8000
    s = _inputs(n, 100, 1700, torch.float32, seed=40)
    got = _run(s, names=("a",), up_grad=False)
    d = {k: s[k].double().cuda() for k in ("x", "w", "a")}
    p = torch.softmax(d["x"] @ d["w"].T, 1)
    u = d["a"] @ d["w"].T
    h = p * (u - (p * u).sum(1, keepdim=True))
    g = p.clone()
    g[torch.arange(n), s["t"].cuda()] -= 1
    ref = dict(dx=g @ d["w"] / n, gx=h @ d["w"] / n)
    for k, want in ref.items():
        err = got[k].double() - want
        assert err.mean().abs() < 4 / n ** 0.5 * err.square().mean().sqrt(), k
