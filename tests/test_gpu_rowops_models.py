"""
The row-wise MLP operators where models reach them: `MLP(fused=True)` (honn/utils.py), the layer families built from it, a captured training
step over batch slots, captured and replayed on their own, and next to each other in one program.

Tolerances: two f32 evaluations of the same network differ by the f32 error of each, bounded per block by (K + 128) 2^-24 of the absolute sums and
amplified by the norms' 1 / sigma; 2e-5 of a tensor's largest value covers the three blocks here (measured against 64 bits: below 2e-6).
"""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

KEY = "X___X___1___A___0"


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def near(a, b, tol, what):
    s = float(b.abs().max()) + 1e-12
    assert float((a.double() - b.double()).abs().max()) <= tol * s, (what, float((a.double() - b.double()).abs().max()) / s)


@pytest.mark.parametrize("norm", ["ln", "none"])
@pytest.mark.parametrize("act", ["silu", "ELU", "relu"])
def test_fused_mlp_equals_the_stock_modules(dev, norm, act):
    from pygho_amd.honn.utils import MLP
    torch.manual_seed(0)
    for hid, out, layers, tail, dp in ((96, 96, 3, True, 0.0), (128, 1, 2, False, 0.0), (40, 72, 1, True, 0.0), (64, 64, 2, True, 0.3)):
        stock = MLP(hid, out, layers, tail, dp=dp, norm=norm, act=act).to(dev)
        fused = MLP(hid, out, layers, tail, dp=dp, norm=norm, act=act, fused=True).to(dev)
        with torch.no_grad():
            for p in stock.parameters():
                p.add_(0.1 * torch.randn_like(p))
        fused.load_state_dict(stock.state_dict())
        stock.eval() if dp else None
        fused.eval() if dp else None
        for shape in ((517, hid), (3, 7, 5, hid)):
            x = torch.randn(shape, device=dev)
            res = torch.randn(shape[:-1] + (out,), device=dev)
            got, want = [], []
            for m, o in ((fused, got), (stock, want)):
                xx, rr = x.clone().requires_grad_(True), res.clone().requires_grad_(True)
                y = m(xx, residual=rr)
                gy = torch.cos(torch.arange(y.numel(), device=dev, dtype=torch.float32)).reshape(y.shape)
                o.append(y.detach())
                if act != "relu":                              # (relu's slope jumps where two correct sums may fall on either side)
                    o += list(torch.autograd.grad(y, [xx, rr, *m.parameters()], gy))
            for k, (a, b) in enumerate(zip(got, want)):
                near(a, b, 2e-5, (norm, act, hid, out, shape, k))


def test_fused_mlp_with_active_dropout(dev):
    """dropout between the norm and the activation: the block stops in front of it; the same draws give the same result"""
    from pygho_amd.honn.utils import MLP
    torch.manual_seed(1)
    stock = MLP(64, 64, 2, True, dp=0.5, norm="ln", act="silu").to(dev)
    fused = MLP(64, 64, 2, True, dp=0.5, norm="ln", act="silu", fused=True).to(dev)
    fused.load_state_dict(stock.state_dict())
    x = torch.randn(300, 64, device=dev)
    out = []
    for m in (stock, fused):
        torch.manual_seed(7)
        out.append(m(x, residual=x))
    near(out[1].detach(), out[0].detach(), 2e-5, "dropout")


@pytest.mark.parametrize("norm", ["ln", "none"])
def test_fused_mlp_under_autocast(dev, norm):
    """16-bit compute, f32 master parameters: the block's output in the autocast dtype, gradients in f32.  Against f32: every tensor is rounded at
    most once per block on its way (input, output, dz: 3 blocks x 3 roundings of 2^-8, each relative to its value, random in sign)"""
    from pygho_amd import _ops
    from pygho_amd.honn.utils import MLP
    torch.manual_seed(2)
    fused = MLP(128, 128, 3, True, norm=norm, act="silu", fused=True).to(dev)
    x = torch.randn(9000, 128, device=dev)
    for dt, step in ((torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)):
        ref = []
        for use in (False, True):
            _ops.ensure_cast_arena(fused, dt)
            xx = x.clone().requires_grad_(True)
            with torch.autocast("cuda", dtype=dt, enabled=use):
                y = fused(xx)
            assert y.dtype == (dt if use else torch.float32)
            g = torch.autograd.grad(y, [xx, *fused.parameters()], torch.ones_like(y) * 0.01)
            assert all(t.dtype == torch.float32 for t in g)
            ref.append([y.detach().float(), *g])
        for k, (a, b) in enumerate(zip(ref[1], ref[0])):
            assert float((a - b).norm()) <= 9 * step * float(b.norm()) + 1e-6, (norm, dt, k, float((a - b).norm() / b.norm()))


@pytest.mark.parametrize("conv", ["NGNN", "SSWL", "GNNAK", "SUN", "PPGN"])
def test_layer_families_on_fused_mlps(dev, conv):
    """the example models with LayerNorm MLPs, fused against stock, f32: predictions and parameter gradients"""
    from pygho_amd import synth
    from pygho_amd.honn.SpOperator import parse_precomputekey
    from pygho_amd.models import SpModel
    torch.manual_seed(5)
    stock = SpModel(conv, num_layer=2, hiddim=32, mlp={"norm": "ln", "act": "silu", "dp": 0.0}, outlayer=2).to(dev)
    fused = SpModel(conv, num_layer=2, hiddim=32, mlp={"norm": "ln", "act": "silu", "dp": 0.0, "fused": True}, outlayer=2).to(dev)
    fused.load_state_dict(stock.state_dict())
    hb = synth.make_batch(6, "zinc", seed=17, keys=tuple(parse_precomputekey(stock)))
    dd = synth.to_datadict(hb, dev)
    w = torch.randn(hb.num_graphs, 1, device=dev)
    got = []
    for m in (stock, fused):
        y = m(dict(dd))
        m.zero_grad()
        (y * w).sum().backward()
        got.append((y.detach(), {k: p.grad for k, p in m.named_parameters() if p.grad is not None}))
    near(got[1][0], got[0][0], 2e-4, conv)
    assert got[0][1].keys() == got[1][1].keys()
    for k in got[0][1]:
        near(got[1][1][k], got[0][1][k], 2e-3, (conv, k))


def test_captured_slot_step_with_fused_layer_norm_mlps(dev):
    """ONE captured training step over a batch slot (rows counted on the device) serves different batches with the eager step's bits: losses,
    and every parameter after the optimizer's steps -- eager work and synchronisations between the replays"""
    from pygho_amd import synth
    from pygho_amd.collate import DeviceGraphStore
    from pygho_amd.graphs import SlotStep
    from pygho_amd.ngnn import SpModel
    rng = np.random.default_rng(5)
    store = DeviceGraphStore([synth.make_graph(rng, "zinc", 3, (KEY,)) for _ in range(128)], dev)

    def stepper(m):
        opt = torch.optim.AdamW(m.parameters(), lr=1e-3, capturable=True)

        def step(batch):
            opt.zero_grad(set_to_none=True)
            with torch.autocast("cuda", dtype=torch.bfloat16):
                pred = m(batch)
            loss = torch.nn.functional.l1_loss(batch["y"].unsqueeze(-1), pred.float())
            loss.backward()
            opt.step()
            return loss.detach()
        return step
    for hidden in (128, 64):
        torch.manual_seed(0)
        model = SpModel(1, 2, hidden, mlp={"norm": "ln", "act": "silu", "dp": 0.0, "fused": True}, act_dtype=torch.bfloat16).to(dev)
        ref = copy.deepcopy(model)
        ids = [np.random.default_rng(10 + k).permutation(128)[:48] for k in range(6)]
        eager = stepper(ref)
        for _ in range(3):
            eager(store.collate(ids[0]))
        want = [eager(store.collate(i)).clone() for i in ids[1:]]
        ss = SlotStep(store, 48, stepper(model), warmup_ids=ids[0], warmup=3)
        got = []
        for i in ids[1:]:
            got.append(ss.run(i).clone())
            torch.cuda.synchronize()
            torch.randn(1000, device=dev).sum()
        assert ss.replays == 5 and all(torch.equal(a, b) for a, b in zip(got, want)), [(float(a), float(b)) for a, b in zip(got, want)]
        for (k, p), q in zip(model.named_parameters(), ref.parameters()):
            assert torch.equal(p, q), (hidden, k)


def test_operators_together_captured_and_replayed(dev):
    """norm -> linear -> block in a row, forward and backward, captured once and replayed on new values; two graphs of the same call, and eager calls
    on another stream in between, do not disturb each other (workspaces belong to a call)"""
    from pygho_amd import _ops
    torch.manual_seed(3)
    for dtype, n in ((torch.bfloat16, 128), (torch.float32, 72), (torch.float16, 520)):
        m, k = 1500, 96
        par = [torch.randn(s, device=dev).div_(4).to(dtype) for s in ((k,), (k,), (n, k), (n,), (n, n), (n,), (n,), (n,))]
        gy = torch.randn(m, n, device=dev).to(dtype)

        def run(x, p):
            leaves = [t.detach().requires_grad_(True) for t in (x, *p)]
            x1 = _ops.layer_norm_act(leaves[0], leaves[1], leaves[2], act="silu")
            x2 = _ops.linear_act(x1, leaves[3], leaves[4], "elu")
            y = _ops.linear_norm_act(x2, leaves[5], leaves[6], leaves[7], leaves[8], act="silu", residual=x2)
            return [y.detach(), *torch.autograd.grad(y, leaves, gy)]
        static = [torch.randn(m, k, device=dev).to(dtype) for _ in range(2)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for s in static:
                run(s, par)
        torch.cuda.current_stream().wait_stream(side)
        graphs, outs = [], []
        for s in static:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(run(s, par))
            graphs.append(g)
        for _ in range(4):
            new = [torch.randn(m, k, device=dev).to(dtype) for _ in range(2)]
            for s, v in zip(static, new):
                s.copy_(v)
            for g in graphs:
                g.replay()
            with torch.cuda.stream(side):
                run(new[0] * 2, par)
            torch.cuda.synchronize()
            for o, v in zip(outs, new):
                want = run(v, par)
                assert all(torch.equal(a, b) for a, b in zip(o, want)), (dtype, n)


def test_operators_on_two_streams_at_once(dev):
    from pygho_amd import _ops
    torch.manual_seed(4)
    x = [torch.randn(20000, 128, device=dev).bfloat16() for _ in range(2)]
    w, b = torch.randn(128, 128, device=dev).div_(8).bfloat16(), torch.randn(128, device=dev).bfloat16()
    gy = torch.randn(20000, 128, device=dev).bfloat16()

    def run(t):
        t = t.detach().requires_grad_(True)
        ww, bb = w.detach().requires_grad_(True), b.detach().requires_grad_(True)
        y = _ops.linear_norm_act(t, ww, bb, bb, bb, act="silu")
        return torch.autograd.grad(y, (t, ww, bb), gy)
    want = [run(t) for t in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, t in zip(streams, x):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run(t))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b2) for g, u in zip(got, want) for a, b2 in zip(g, u))


def test_an_operator_runs_twice_in_one_graph_of_gradients(dev):
    """shared parameters and a shared input: gradients add up; a parameter changed in place between forward and backward is refused by autograd"""
    from pygho_amd import _ops
    torch.manual_seed(6)
    x = torch.randn(200, 64, device=dev, requires_grad=True)
    w = (torch.randn(64, 64, device=dev) / 8).requires_grad_(True)
    b = torch.randn(64, device=dev, requires_grad=True)
    y = _ops.linear_act(_ops.linear_act(x, w, b, "silu", residual=x), w, b, "silu", residual=x)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    x6, w6, b6 = (t.detach().double().requires_grad_(True) for t in (x, w, b))
    f = torch.nn.functional
    h = f.silu(x6 @ w6.t() + b6) + x6
    want = torch.autograd.grad((f.silu(h @ w6.t() + b6) + x6).sum(), (x6, w6, b6))
    for a, c, name in zip((gx, gw, gb), want, "xwb"):
        near(a, c, 2e-5, name)
    y = _ops.linear_act(x, w, b, "silu")
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)
