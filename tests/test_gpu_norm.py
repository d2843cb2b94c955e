"""Layer norm and its first and second gradients against their formulas in
float64, element by element (bounds: tests/_ops_util.py)."""
import pytest
import torch

from tests._ops_util import norm_bound, norm_ref, within
from testtimeideas_amd.ttt_e2e import LayerNorm, layer_norm

pytestmark = pytest.mark.gpu
EPS = 1e-5


def _inputs(n, d, dtype, seed, pdtype=None, offset=0.0):
    g = torch.Generator().manual_seed(seed)

    def randn(*shape, add=0.0, dt=dtype):
        return (torch.randn(shape, generator=g) + add).to(dt)

    pd = pdtype or dtype
    return dict(x=randn(n, d, add=offset), w=randn(d, add=1.0, dt=pd), b=randn(d, dt=pd), dy=randn(n, d),
                a=randn(n, d), cw=randn(d, dt=pd), cb=randn(d, dt=pd))


def _run(s, eps=EPS, names=("a", "cw", "cb")):
    x, w, b, dy = (s[k].cuda().requires_grad_() for k in ("x", "w", "b", "dy"))
    y = layer_norm(x, w, b, eps)
    first = torch.autograd.grad(y, (x, w, b), dy, create_graph=True)
    pairs = [(f, s[k].cuda()) for f, k in zip(first, ("a", "cw", "cb")) if k in names]
    second = torch.autograd.grad([p[0] for p in pairs], (x, w, dy), [p[1] for p in pairs])
    return dict(zip(("y", "dx", "dw", "db", "gx", "gw", "gdy"), (y, *first, *second)))


def _check(s, got, eps=EPS, names=("a", "cw", "cb")):
    dt = {"dw": s["w"].dtype, "db": s["w"].dtype, "gw": s["w"].dtype}
    d = {k: v.double() for k, v in s.items()}
    ref, mag = norm_ref(d["x"], d["w"], d["b"], eps, d["dy"], *(d[k] if k in names else None for k in ("a", "cw", "cb")))
    for k, v in got.items():
        within(k, v, ref[k], norm_bound(ref[k], mag[k], dt.get(k, s["x"].dtype)))


SIZES = [(1, 1), (1, 512), (3, 7), (5, 64), (130, 384), (1000, 65), (257, 1003), (64, 1024), (33, 1032), (40, 2048),
         (9, 3001), (6, 4096), (3, 8200), (2, 16384)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("n,d", SIZES)
def test_values_and_both_gradients(n, d, dtype):
    s = _inputs(n, d, dtype, seed=n + d)
    _check(s, _run(s))


def test_longest_rows():
    s = _inputs(2, 32768, torch.bfloat16, seed=1)
    _check(s, _run(s))


def test_many_rows_share_workgroups():
    s = _inputs(9001, 40, torch.float32, seed=2)
    _check(s, _run(s))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_fp32_parameters(dtype):
    s = _inputs(70, 200, dtype, seed=3, pdtype=torch.float32)
    got = _run(s)
    assert got["y"].dtype == dtype and got["dw"].dtype == torch.float32
    _check(s, got)


@pytest.mark.parametrize("names", [("a",), ("cw",), ("cb",), ("cw", "cb"), ("a", "cb")])
def test_some_cotangents(names):
    """A second gradient through some of dx, dw, db alone."""
    s = _inputs(33, 100, torch.float32, seed=4)
    x, w, b, dy = (s[k].cuda().requires_grad_() for k in ("x", "w", "b", "dy"))
    y = layer_norm(x, w, b, EPS)
    first = dict(zip(("a", "cw", "cb"), torch.autograd.grad(y, (x, w, b), dy, create_graph=True)))
    got = torch.autograd.grad([first[k] for k in names], (x, w, dy), [s[k].cuda() for k in names])
    _check(s, dict(zip(("gx", "gw", "gdy"), got)), names=names)


def test_first_gradients_one_at_a_time():
    s = _inputs(50, 130, torch.bfloat16, seed=5)
    for k, name in (("x", "dx"), ("w", "dw"), ("b", "db")):
        t = {j: s[j].cuda() for j in ("x", "w", "b")}
        t[k].requires_grad_()
        g, = torch.autograd.grad(layer_norm(t["x"], t["w"], t["b"]), (t[k],), s["dy"].cuda())
        _check(s, {name: g})


def test_no_parameters():
    s = _inputs(20, 96, torch.float32, seed=6)
    x, dy = s["x"].cuda().requires_grad_(), s["dy"].cuda().requires_grad_()
    y = layer_norm(x)
    dx, = torch.autograd.grad(y, (x,), dy, create_graph=True)
    gx, gdy = torch.autograd.grad(dx, (x, dy), s["a"].cuda())
    s = dict(s, w=torch.ones(96), b=torch.zeros(96))
    _check(s, dict(y=y, dx=dx, gx=gx, gdy=gdy), names=("a",))


def test_rows_far_from_zero():
    """A common offset of 300 costs x - mean what its own rounding costs, and no more."""
    s = _inputs(40, 500, torch.float32, seed=7, offset=300.0)
    _check(s, _run(s))


def test_constant_rows():
    """Variance 0: eps alone holds the scale."""
    s = _inputs(6, 48, torch.float32, seed=8)
    s["x"][2] = 3.0
    s["x"][4] = 0.0
    _check(s, _run(s))


def test_strides_and_leading_shape():
    """Transposed, sliced and expanded operands give what their copies give."""
    base = torch.randn(6, 5, 80, generator=torch.Generator().manual_seed(9)).cuda()
    w, b = torch.randn(40).cuda(), torch.randn(40).cuda()
    views = [base[..., 7:47], base.transpose(0, 1)[..., :40], base[:, :1, 3:43].expand(6, 5, 40),
             base[:, :, ::2], base[1:, 2, 1:41]]
    for v in views:
        x = v.detach().requires_grad_()
        c = v.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
        dy = torch.randn(v.shape, device="cuda").transpose(0, 1).contiguous().transpose(0, 1)
        gx = torch.autograd.grad(layer_norm(x, w, b), (x,), dy)[0]
        gc = torch.autograd.grad(layer_norm(c, w, b), (c,), dy.contiguous())[0]
        assert torch.equal(layer_norm(x, w, b), layer_norm(c, w, b))
        assert torch.equal(gx, gc)


def test_no_rows():
    x = torch.empty(0, 32, device="cuda", requires_grad=True)
    w, b = torch.ones(32, device="cuda", requires_grad=True), torch.zeros(32, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y), create_graph=True)
    assert y.shape == dx.shape == (0, 32) and not dw.any() and not db.any()


def test_nan_stays_in_its_row():
    s = _inputs(10, 300, torch.bfloat16, seed=10)
    clean = layer_norm(s["x"].cuda(), s["w"].cuda(), s["b"].cuda())
    s["x"][3, 7] = float("nan")
    s["x"][5, 0] = float("inf")
    y = layer_norm(s["x"].cuda(), s["w"].cuda(), s["b"].cuda())
    keep = [i for i in range(10) if i not in (3, 5)]
    assert torch.equal(y[keep], clean[keep]) and y[3].isnan().all() and y[5].isnan().all()


def test_repeats_bitwise():
    s = _inputs(3000, 320, torch.float32, seed=11)
    one, two = _run(s), _run(s)
    assert all(torch.equal(one[k], two[k]) for k in one)


def test_third_derivative_raises():
    s = _inputs(4, 16, torch.float32, seed=12)
    x, w, b = (s[k].cuda().requires_grad_() for k in ("x", "w", "b"))
    dx, = torch.autograd.grad(layer_norm(x, w, b).square().sum(), (x,), create_graph=True)
    gx, = torch.autograd.grad(dx.square().sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        torch.autograd.grad(gx.sum(), (x,))


def test_gradient_against_differences():
    """The second gradient against central differences of the first, both in
    float32: step 2^-7, whose own error is of the order of its square."""
    s = _inputs(5, 24, torch.float32, seed=13)
    w, b, dy, a = (s[k].cuda() for k in ("w", "b", "dy", "a"))
    v = torch.randn(5, 24, generator=torch.Generator().manual_seed(14)).cuda()

    def slope(x):
        x = x.detach().requires_grad_()
        return (torch.autograd.grad(layer_norm(x, w, b), (x,), dy, create_graph=True)[0] * a).sum(), x

    f, x = slope(s["x"].cuda())
    got = (torch.autograd.grad(f, (x,))[0] * v).sum()
    h = 2.0 ** -7
    diff = (slope(s["x"].cuda() + h * v)[0] - slope(s["x"].cuda() - h * v)[0]) / (2 * h)
    # third derivatives of a row are of the order of its sums: h^2 of them, and 2^-24 / h of the rounding
    scale = float((a.abs() * dy.abs() * w.abs()).sum() * v.abs().max() ** 3)
    assert abs(float(got - diff)) <= (h * h + 2.0 ** -20 / h) * scale


def test_module_matches_its_function_and_torch_state():
    m = LayerNorm(64).cuda()
    ref = torch.nn.LayerNorm(64)
    m.load_state_dict(ref.state_dict())
    x = torch.randn(3, 4, 64, device="cuda")
    assert torch.equal(m(x), layer_norm(x, m.weight, m.bias, m.eps))
    assert list(m.state_dict()) == list(ref.state_dict())


def test_graph_replays():
    """Forward, backward and the second gradient captured in a HIP graph;
    every replay against the eager result, with eager work in between."""
    s = _inputs(300, 200, torch.bfloat16, seed=15)
    t = {k: v.cuda() for k, v in s.items()}
    for k in ("x", "w", "b", "dy"):
        t[k].requires_grad_()

    def step():
        y = layer_norm(t["x"], t["w"], t["b"])
        first = torch.autograd.grad(y, (t["x"], t["w"], t["b"]), t["dy"], create_graph=True)
        return [y, *first, *torch.autograd.grad(first, (t["x"], t["w"], t["dy"]), (t["a"], t["cw"], t["cb"]))]

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
    s = _inputs(500, 256, torch.float32, seed=16)
    ref = _run(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _run(s)
    side.synchronize()
    assert all(torch.equal(got[k], ref[k]) for k in ref)


def test_offsets_past_32_bits():
    """More than 2^31 values: the last rows against the formulas."""
    n, d = 66000, 32768
    s = _inputs(3, d, torch.bfloat16, seed=21)
    x = torch.zeros(n, d, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros_like(x)
    x[-3:], dy[-3:] = s["x"].cuda(), s["dy"].cuda()
    x.requires_grad_()
    y = layer_norm(x, s["w"].cuda(), s["b"].cuda(), EPS)
    dx, = torch.autograd.grad(y, (x,), dy)
    _check(s, {"y": y[-3:], "dx": dx[-3:]})
    # a row of zeros: the bias, and no gradient
    assert torch.equal(y[0].cpu(), s["b"]) and not dx[:-3].any()
