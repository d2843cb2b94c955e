"""The operators at the model's tail as they are used: layer norm into the
cross entropy of the head, both derivatives through the two together; the
model's meta step with them (``ModelConfig.fused_tail``) against the same
model in float64 on the CPU; and their calls captured in HIP graphs beside
others of the same leaves.

Tolerances.  Losses relative 1e-5 and meta-gradients relative Frobenius 1e-3
in fp32, as for the model without them.  The chain in 16 bits: each of the
five tensors between input and output (the norm's y, the loss' dX and H, the
norm's dy and gx) is rounded by at most u of its values, and G once more, so
the relative Frobenius error is at most 6 u / sqrt(3) where the errors of many
values are independent, doubled for the sums in which terms cancel.
"""
import copy

import pytest
import torch

from oracle import math_path
from tests._ops_util import unit
from tests._util import rel_fro
from testtimeideas_amd.ttt_e2e import attention as attn_mod
from testtimeideas_amd.ttt_e2e import layer_norm, linear_cross_entropy
from ttt_e2e import data, meta
from ttt_e2e.model import ModelConfig, TTTModel

pytestmark = pytest.mark.gpu


def _inputs(n, d, v, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    head = rn(v, d) * 2 / d ** 0.5
    t = torch.randint(0, v, (n,), generator=g)
    t[torch.rand(n, generator=g) < 0.1] = -100
    x = rn(n, d) + torch.where((t >= 0)[:, None], head[t.clamp(min=0)], 0.0)
    mask = (torch.rand(n, generator=g) < 0.75).float()
    return dict(x=x.to(dtype), w=(1 + 0.1 * rn(d)).to(dtype), b=(0.1 * rn(d)).to(dtype), head=head.to(dtype), t=t,
                mask=mask, a=rn(n, d).to(dtype))


def _chain(s):
    leaves = [s[k].cuda().requires_grad_() for k in ("x", "w", "b", "head")]
    y = layer_norm(*leaves[:3])
    loss = linear_cross_entropy(y, leaves[3], s["t"].cuda(), s["mask"].cuda())
    dx, = torch.autograd.grad(loss, leaves[:1], create_graph=True)
    return [loss, dx, *torch.autograd.grad(dx, leaves, s["a"].cuda())]


def _chain_ref(s):
    leaves = [s[k].double().requires_grad_() for k in ("x", "w", "b", "head")]
    y = torch.nn.functional.layer_norm(leaves[0], (leaves[0].size(1),), leaves[1], leaves[2], 1e-5)
    nll = torch.nn.functional.cross_entropy(y @ leaves[3].t(), s["t"], reduction="none", ignore_index=-100)
    w = s["mask"].double() * (s["t"] != -100)
    loss = (nll * w).sum() / w.sum().clamp_min(1.0)
    dx, = torch.autograd.grad(loss, leaves[:1], create_graph=True)
    return [loss, dx, *torch.autograd.grad(dx, leaves, s["a"].double())]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("n,d,v", [(1, 64, 100), (300, 96, 1000), (1025, 40, 333)])
def test_norm_into_loss_twice_differentiated(n, d, v, dtype):
    s = _inputs(n, d, v, dtype, seed=n)
    if n == 1:  # the one row counts
        s["t"][:], s["mask"][:] = 7, 1.0
    tol = 1e-4 if dtype == torch.float32 else 2 * 6 * unit(dtype) / 3 ** 0.5
    for name, got, ref in zip(("loss", "dx", "gx", "gw", "gb", "ghead"), _chain(s), _chain_ref(s)):
        assert rel_fro(got, ref) <= tol, f"{name}: {rel_fro(got, ref):.2e} > {tol:.2e}"


def _oracle_windowed(q, k, v, window, local=True, scale=None, bwd_mode=None):
    return math_path.window_chunks_attention(q, k, v, window if window is not None else q.size(-2))


@pytest.mark.parametrize("param_filter", ["mlp_fast", "mlp_fast,suffix_blocks.0.ln,ln_f,head"])
def test_meta_step_with_the_fused_tail(param_filter, monkeypatch):
    """The second filter adapts the norms and the head too, so their gradients
    are differentiated."""
    t = 128
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=64, max_seq_len=t, window_size=64, d_model=64, n_heads=2, n_layers=2, d_ff=128,
                      suffix_layers=1, dual_mlp=True, fused_tail=True)
    gpu = TTTModel(cfg).cuda()
    cpu_cfg = copy.copy(cfg)
    cpu_cfg.fused_tail = False
    cpu = TTTModel(cpu_cfg)
    cpu.load_state_dict(gpu.state_dict())
    cpu = cpu.double()
    g = torch.Generator().manual_seed(5)
    bt = data.generate_kv_batch(2, (t * 3) // 4, t // 4, cfg.vocab_size, num_keys=16, device="cpu", pad_to=t,
                                far_frac=0.5, generator=g)
    kw = dict(inner_lr=0.1, inner_steps=2, param_filter=param_filter, chunk_size=64)
    inner_g, outer_g = meta.meta_step(gpu, bt.input_ids.cuda(), bt.targets.cuda(), bt.inner_mask.cuda(),
                                      bt.outer_mask.cuda(), **kw)
    outer_g.backward()
    monkeypatch.setattr(attn_mod, "windowed_attention", _oracle_windowed)
    inner_c, outer_c = meta.meta_step(cpu, bt.input_ids, bt.targets, bt.inner_mask.double(), bt.outer_mask.double(),
                                      **kw)
    outer_c.backward()
    assert abs(inner_g.item() - inner_c.item()) <= 1e-5 * abs(inner_c.item())
    assert abs(outer_g.item() - outer_c.item()) <= 1e-5 * abs(outer_c.item())
    ref = dict(cpu.named_parameters())
    top = max(float(p.grad.norm()) for p in ref.values() if p.grad is not None)
    for name, p in gpu.named_parameters():
        r = ref[name].grad
        assert (p.grad is None) == (r is None), name
        if r is not None:
            err = float((p.grad.double().cpu() - r).norm())
            assert err <= 1e-3 * max(float(r.norm()), 1e-4 * top), f"{name}: {err:.3e} of {float(r.norm()):.3e}"


def test_fused_tail_refusals():
    m = TTTModel(ModelConfig(vocab_size=16, max_seq_len=8, window_size=None, d_model=16, n_heads=1, n_layers=1,
                             d_ff=16)).cuda()
    ids = torch.zeros(1, 8, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="fused_tail"):
        m(ids, targets=ids)


def _captured(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


def _steps():
    s1, s2 = _inputs(200, 64, 500, torch.bfloat16, 1), _inputs(90, 64, 3000, torch.bfloat16, 2)
    dev = [{k: v.cuda() for k, v in s.items()} for s in (s1, s2)]
    for s in dev:
        for k in ("x", "w", "b", "head"):
            s[k].requires_grad_()

    def step_of(s):
        def step():
            y = layer_norm(s["x"], s["w"], s["b"])
            loss = linear_cross_entropy(y, s["head"], s["t"], s["mask"])
            first = torch.autograd.grad(loss, (s["x"], s["head"]), create_graph=True)
            return [loss, *first, *torch.autograd.grad(first, (s["x"], s["w"], s["head"]),
                                                       (s["a"], torch.ones_like(s["head"])))]
        return step

    return dev, [step_of(s) for s in dev]


def test_two_captured_steps():
    """Two graphs replayed in turn, with eager steps in between: none disturbs
    another's workspace."""
    _, steps = _steps()
    with torch.autograd.set_multithreading_enabled(False):
        refs = [[r.detach().clone() for r in step()] for step in steps]
        graphs = [_captured(step) for step in steps]
        for turn in range(3):
            for (graph, out), ref in zip(graphs, refs):
                for o in out:
                    o.detach().fill_(3.0)
                graph.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(o, r) for o, r in zip(out, ref))
            for step, ref in zip(steps, refs):
                assert all(torch.equal(o, r) for o, r in zip(step(), ref))


def test_capture_beside_a_living_eager_graph_is_refused():
    """Its end would end the process; the eager graph itself goes on."""
    (s, _), (step, _) = _steps()
    with torch.autograd.set_multithreading_enabled(False):
        ref = [r.detach().clone() for r in step()]
        live = linear_cross_entropy(layer_norm(s["x"], s["w"], s["b"]), s["head"], s["t"], s["mask"])
        with pytest.raises(RuntimeError, match="cannot be captured while a graph of the same leaf"):
            _captured(step)
        torch.cuda.synchronize()
        got = torch.autograd.grad(live, (s["x"], s["head"]))
        assert all(torch.equal(a, b) for a, b in zip(got, ref[1:3]))
        del live, got
        graph, out = _captured(step)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, r) for o, r in zip(out, ref))


def test_two_streams_at_once():
    """The same call on two streams at once: each has its own workspace."""
    s = {k: v.cuda() for k, v in _inputs(700, 128, 4000, torch.float16, 3).items()}
    x, head = s["x"].requires_grad_(), s["head"].requires_grad_()

    def call():
        return torch.autograd.grad(linear_cross_entropy(x, head, s["t"], s["mask"]), (x, head))

    ref = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, ref))
