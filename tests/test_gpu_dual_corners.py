"""
The one-pass backward's table-gradient form (csrc/seg_dual.hip) with messages that are not finite: an infinity or NaN belongs to the table rows that its
messages look up, the others are the sums of their own messages.
"""
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_message_that_is_not_finite_stays_in_its_table_rows(dev, dtype, bad):
    from pygho_amd import _ops, synth
    from pygho_amd.collate import DeviceGraphStore
    rng = np.random.default_rng(5)
    store = DeviceGraphStore([synth.make_graph(rng, "zinc", 3, (KEY,)) for _ in range(60)], dev)
    dd = store.collate(np.arange(60))
    acd = dd[KEY + "___acd"]
    nt, ne, d = dd["X"].nnz, dd["A"].nnz, 128
    plan = _ops.message_plan(acd, nt, nt, ne)
    look = dd["A"].values[acd[2]]
    look_fwd, look_byc = plan.lookup(_ops.flat_index(dd["A"].values))
    gen = torch.Generator(device=dev).manual_seed(1)
    g, h = (torch.randint(1, 4, (nt, d), generator=gen, device=dev).to(dtype) for _ in range(2))       # integers: sums below 2^24 are exact
    table = torch.randn(16, d, generator=gen, device=dev).to(dtype)
    clean = _ops.dual_backward_tg(plan, g, h, table, look_fwd, look_byc)[1]
    want = torch.zeros(16, d, dtype=torch.float64, device=dev).index_add_(0, look, g.double()[acd[0]] * h.double()[acd[1]])
    assert float(want.max()) < 2 ** 24 and torch.equal(clean.double(), want)
    # a row of g whose messages all look up one table row, in the middle of the batch
    rows = [int(a) for a in acd[0].unique()[nt // 2:nt // 2 + 400] if look[acd[0] == a].unique().numel() == 1]
    a = rows[0]
    hit = int(look[acd[0] == a][0])
    g[a, 5] = bad
    got = _ops.dual_backward_tg(plan, g, h, table, look_fwd, look_byc)[1].double()
    keep = torch.ones(16, d, dtype=torch.bool, device=dev)
    keep[hit, 5] = False
    assert torch.equal(got[keep], want[keep]) and not bool(torch.isfinite(got[hit, 5]))
