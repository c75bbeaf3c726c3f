"""Plans of the weight update that are dropped while another stream still runs them."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


@pytest.mark.parametrize("bits", [32, 8])
def test_plans_dropped_while_a_stream_runs_them(api, bits):
    import torch
    heavy = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    torch.manual_seed(0)
    p0, g = [torch.randn(200000, device="cuda") for _ in range(2)]
    sizes = {(int(api.lib().ob200_grad_norm_workspace_bytes()),), (800000,), (200000,), (3128,)}

    def steps(p, stream, drop):
        norm, opt = api.GradNorm([g]), api.AdamW([p], [g], state_bits=bits)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            if drop:
                for _ in range(20):
                    torch.mm(heavy, heavy)       # milliseconds ahead of the plans' kernels
            out = []
            for _ in range(2):
                out.append(norm.run(1.0).clone())
                opt.step(0.01, grad_scale=norm.clip)
        if drop:
            del norm, opt
            # memory of their sizes, written by a stream that waits for nothing
            junk = [torch.full(s, 255, dtype=torch.uint8, device="cuda") for s in sizes for _ in range(8)]
            del junk
        torch.cuda.synchronize()
        return out
    a, b = p0.clone(), p0.clone()
    want, side = steps(a, torch.cuda.current_stream(), False), torch.cuda.Stream()
    for _ in range(3):
        b.copy_(p0)
        got = steps(b, side, True)
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(a, b)
