"""The residual norm's entry points with results over their inputs, as the header allows: the same bits as with arrays apart."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _device(cuda):
    yield


def rand(*shape, dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("norm,post", [("rms", True), ("layer", True), ("rms", False)])
@pytest.mark.parametrize("xt,ft", [(F32, BF), (BF, BF), (BF, F32)])
@pytest.mark.parametrize("rows,width,groups", [(3000, 64, 1500), (700, 1000, 1), (900, 4096, 300), (40, 16384, 1), (500, 75, 500), (30, 8201, 1)])
def test_results_over_inputs(rows, width, groups, xt, ft, norm, post):
    from b200 import _lib as L
    from b200 import ops

    x, f, ds, dh = (rand(rows, width, dtype=t, seed=i) for i, t in enumerate((xt, ft, xt, ft)))
    w = {"gamma": rand(width, seed=5), "gate": rand(groups, width, seed=6)}
    if post:
        w["post_gamma"] = rand(width, seed=7)
    d = L.ResidualNorm()
    d.rows, d.cols, d.groups, d.kind, d.post, d.scale, d.eps = rows, width, groups, int(norm == "layer"), int(post), 0.5, 1e-5
    d.x_dtype, d.f_dtype, d.weight_dtype, d.gate_dtype = ops.code(x), ops.code(f), L.F32, L.F32
    for name, t in w.items():
        setattr(d, name, t.data_ptr())

    def forward(x, f, total, normed):
        L.call("b200_residual_norm_forward", d, x.data_ptr(), f.data_ptr(), total.data_ptr(), normed.data_ptr(), ops.stream_ptr())
        return total, normed

    def gradient(ds, dh, x, f, dx, df):
        made = {n: torch.empty_like(t) for n, t in w.items()}
        g = L.ResidualNormGrads()
        for name, t in made.items():
            setattr(g, "d" + name, t.data_ptr())
        n = L.lib().b200_residual_norm_grad_workspace_bytes(d)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        L.call("b200_residual_norm_grad", d, ds.data_ptr(), dh.data_ptr(), x.data_ptr(), f.data_ptr(), dx.data_ptr(), df.data_ptr(), g, ws.data_ptr(), n,
               ops.stream_ptr())
        return dx, df, *made.values()

    want = forward(x, f, torch.empty_like(x), torch.empty_like(f))
    for over_x, over_f in ((True, True), (True, False), (False, True)):
        a, b = x.clone(), f.clone()
        got = forward(a, b, a if over_x else torch.empty_like(x), b if over_f else torch.empty_like(f))
        assert all(torch.equal(s, t) for s, t in zip(got, want)), (over_x, over_f)
    want = gradient(ds, dh, x, f, torch.empty_like(x), torch.empty_like(f))
    for over_x in ("ds", "x", None):
        for over_f in ("dh", "f", None):
            own = {"ds": ds.clone(), "dh": dh.clone(), "x": x.clone(), "f": f.clone()}
            got = gradient(*own.values(), own[over_x] if over_x else torch.empty_like(x), own[over_f] if over_f else torch.empty_like(f))
            assert all(torch.equal(s, t) for s, t in zip(got, want)), (over_x, over_f)
