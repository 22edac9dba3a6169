"""Attention over the contiguous cache where scores are so large that their products are rounded to whole powers of two and coarser."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qc():
    import cherryq_b200
    return cherryq_b200.load_quant_cuda()


@pytest.mark.parametrize("big", [1000.0, 3000.0, 30000.0])
@pytest.mark.parametrize("D,H,KV", [(64, 8, 2), (128, 8, 2), (128, 4, 4), (128, 8, 1), (64, 3, 3)])
@pytest.mark.parametrize("T", [1, 40, 300, 2000])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores(qc, big, D, H, KV, T, sign):
    """One key far above the others gives its value, two equal ones their mean.  (The other scores are 0, or twice as far below: their weights
    vanish, however scores are rounded.  A weight is kept in two halves of 11 bits, and a few sums in 32 bits come to it.)"""
    g = torch.Generator(device="cuda").manual_seed(D + T)
    k = torch.full((1, T, KV, D), 0.0 if sign > 0 else -2 * big, dtype=torch.half, device="cuda")
    v = torch.randn(1, T, KV, D, device="cuda", generator=g).half()
    for first, second in ((0, 0), (T - 1, T - 1), (T // 2, T // 2), (T // 3, T - 1)):
        q = (big * (1 + 0.3 * torch.rand(1, H, D, device="cuda", generator=g))).half()
        row = (sign * big * (0.5 + 0.3 * torch.rand(KV, D, device="cuda", generator=g))).half()
        keys = k.clone()
        keys[0, first] = keys[0, second] = row
        want = (v[0, first].double() + v[0, second].double()) / 2
        want = want[:, None].expand(KV, H // KV, D).reshape(H, D)
        out = qc.attn_decode(q, keys, v, torch.tensor([T - 1], device="cuda")).view(H, D).double()
        tol = torch.finfo(torch.half).eps / 2 * want.abs() + (2.0 ** -21 + 8 * 2.0 ** -24) * float(v.abs().max())
        assert bool(((out - want).abs() <= tol).all()), (first, second)
