"""The weight update where a moment leaves fp32, and at the ends of the documented ranges."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


@pytest.mark.parametrize("which,value", [("exp_avg_sq", 1e30), ("both", float("inf")), ("both", float("nan"))])
@pytest.mark.parametrize("shift", [0, 1])
def test_moments_that_are_not_finite_in_8_bits(api, which, value, shift):
    """All states of the block are NaN, as the next step's weights then are: none goes on as if nothing had been; the blocks
    beside it are as ever."""
    import torch
    n = 256 * 5 + 40
    p, g = [torch.randn(n + shift, device="cuda")[shift:] for _ in range(2)]
    g[256 * 2 + 7] = value
    g[256 * 2 + 8] = 0
    opt = api.AdamW([p], [g], state_bits=8)
    opt.step(0.01)
    torch.cuda.synchronize()
    block = torch.zeros(n, dtype=torch.bool, device="cuda")
    block[512:768] = True
    for k in ("exp_avg", "exp_avg_sq"):
        held = opt.state[k][0].float() * opt.state[k + "_scale"][0].repeat_interleave(256)[:n]
        bad = torch.isnan(held)
        assert torch.equal(bad, block if which == "both" or k == which else torch.zeros_like(block))
    g.zero_()
    opt.step(0.01)
    assert torch.equal(torch.isnan(p), block)
