"""The weight update: gradient norm and AdamW against 64 bits, 8-bit states code by code, tensor sizes around the blocks and
chunks, many tensors, strides off alignment, steps that are left out, device-side step counts under graph replay."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ODD = [1, 3, 255, 256, 257, 0, 1000, 2047, 2048, 2049, 5000, 64, 36864]


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


def dtype_of(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def views(sizes, dtype, shift, fill=0.0):
    """Tensors laid one behind the other, each starting `shift` elements off a 64-byte line; the whole buffer too."""
    import torch
    starts, at = [], 0
    for k in sizes:
        starts.append(at + shift)
        at += (k + shift + 63) // 64 * 64
    flat = torch.full((at + 64,), fill, device="cuda").to(dtype)
    return [flat[s:s + k] for s, k in zip(starts, sizes)], flat


def bits_of(t):
    import torch
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("repeat", [1, 5, 45])
def test_grad_norm(api, dt, shift, repeat):
    import torch
    torch.manual_seed(shift + repeat)
    gs, _ = views(ODD * repeat, dtype_of(dt), shift, fill=3.0)
    for i, g in enumerate(gs):
        g.copy_(torch.randn(g.shape, device="cuda") * 10.0 ** (i % 4 - 2))
    plan = api.GradNorm(gs)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    out = plan.run(1.0).clone()
    # a square and at most 8 * (chunks of a CTA) <= 64 additions a thread in fp32, the rest in fp64; half of it under the root
    assert abs(float(out[0]) - want) <= 66 * 2.0 ** -24 * want
    assert abs(float(out[1]) - 1.0 / float(out[0])) <= 2 * 2.0 ** -24 / want
    for _ in range(3):
        assert torch.equal(plan.run(1.0), out)
    assert float(plan.run(1e9)[1]) == 1.0 and float(plan.run()[1]) == 1.0
    gs[-1][5] = float("inf")
    out = plan.run(1.0)
    assert math.isinf(float(out[0])) and math.isnan(float(out[1]))


def test_grad_norm_of_zeros_and_of_nothing(api):
    import torch
    plan = api.GradNorm([torch.zeros(5, device="cuda"), torch.zeros(0, device="cuda")])
    assert plan.run(1.0).tolist() == [0.0, 1.0]
    assert api.GradNorm([torch.zeros(0, device="cuda")]).run(1.0).tolist() == [0.0, 1.0]


def test_grad_norm_large(api):
    import torch
    g = torch.empty(300_000_001, dtype=torch.bfloat16, device="cuda")[1:]
    g.fill_(2.0)
    g[-1] = 3.0
    got = float(api.GradNorm([g]).run(1.0)[0])
    # the squares are whole numbers and a thread's sum of them stays below 2^24: exact but for the last rounding
    want = math.sqrt(4.0 * (g.numel() - 1) + 9.0)
    assert abs(got - want) <= 2.0 ** -23 * want


def make(api, sizes, p_dt, g_dt, bits, shift, seed=0, decay=None, eps=1e-8):
    import torch
    torch.manual_seed(seed)
    ps, pflat = views(sizes, dtype_of(p_dt), shift, 5.0)
    gs, _ = views(sizes, dtype_of(g_dt), shift)
    for i, (p, g) in enumerate(zip(ps, gs)):
        p.copy_(torch.randn(p.shape, device="cuda") * 0.1)
        g.copy_(torch.randn(g.shape, device="cuda") * 10.0 ** (i % 5 - 3))
    held = torch.float32 if bits == 32 else torch.uint8
    ms, mflat = views(sizes, held, shift, 9)
    vs, vflat = views(sizes, held, shift, 9)
    state = {}
    for t in ms + vs:
        t.zero_()
    if bits == 8:
        ms, vs = [t.view(torch.float8_e4m3fn) for t in ms], [t.view(torch.float8_e4m3fn) for t in vs]
        for k in ("exp_avg_scale", "exp_avg_sq_scale"):
            state[k] = [torch.zeros((k_ + 255) // 256, device="cuda") for k_ in sizes]
    state.update(exp_avg=ms, exp_avg_sq=vs)
    decay = [0.1 if i % 2 else 0.0 for i in range(len(sizes))] if decay is None else decay
    return api.AdamW(ps, gs, state_bits=bits, weight_decay=decay, state=state, eps=eps), pflat, mflat, vflat


def set_moments(opt):
    """Moments as some steps would leave them (fp32 states)."""
    import torch
    for i in range(len(opt.params)):
        g = opt.grads[i].float()
        opt.state["exp_avg"][i].copy_(g * 0.5 + 0.3 * g.roll(1))
        opt.state["exp_avg_sq"][i].copy_(g.square() * torch.rand_like(g) + 0.01 * g.square().roll(2))


@pytest.mark.parametrize("p_dt,g_dt", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f16"), ("f16", "f16")])
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_adamw_32(api, p_dt, g_dt, shift):
    import torch
    opt, pflat, mflat, vflat = make(api, ODD, p_dt, g_dt, 32, shift)
    set_moments(opt)
    lr, step, scale = 0.01, 7, torch.tensor([0.5], device="cuda")
    old = [(p.double(), g.double() * 0.5, m.double(), v.double()) for p, g, m, v in
           zip(opt.params, opt.grads, opt.state["exp_avg"], opt.state["exp_avg_sq"])]
    outside = [bits_of(f).clone() for f in (pflat, mflat, vflat)]
    opt.step(lr, step=step, grad_scale=scale)
    torch.cuda.synchronize()
    u = 2.0 ** -24
    half = torch.finfo(dtype_of(p_dt)).eps / 2
    for i, (p, g, m, v) in enumerate(old):
        wd = 0.1 if i % 2 else 0.0
        m1, v1 = 0.9 * m + (1 - 0.9) * g, 0.999 * v + (1 - 0.999) * g * g
        # two products and their sum, the coefficients rounded too: 5 half steps of the terms (7 of v's, which has a square)
        assert ((opt.state["exp_avg"][i].double() - m1).abs() <= 5 * u * (0.9 * m.abs() + 0.1 * g.abs())).all()
        assert ((opt.state["exp_avg_sq"][i].double() - v1).abs() <= 7 * u * v1).all()
        move = lr / (1 - 0.9 ** step) * m1 / ((v1 / (1 - 0.999 ** step)).sqrt() + 1e-8)
        size = lr / (1 - 0.9 ** step) * (0.9 * m.abs() + 0.1 * g.abs()) / ((v1 / (1 - 0.999 ** step)).sqrt() + 1e-8)
        want = p * (1 - lr * wd) - move
        # the moments' 5 and 7 / 2, root, denominator, rate and quotient 10; the weight's factor and product 4; the result 1
        tol = u * (20 * size + 5 * p.abs()) + (half * want.abs() if half > u else u * want.abs()) + torch.finfo(dtype_of(p_dt)).smallest_normal * 2 * half
        assert ((opt.params[i].double() - want).abs() <= tol).all(), (i, float(((opt.params[i].double() - want).abs() / tol).max()))
    # what lies between the tensors is not touched
    for f, before, ts in ((pflat, outside[0], opt.params), (mflat, outside[1], opt.state["exp_avg"]), (vflat, outside[2], opt.state["exp_avg_sq"])):
        same = bits_of(f) == before
        at = 0
        mask = torch.ones(f.numel(), dtype=torch.bool, device="cuda")
        for t in ts:
            start = (t.data_ptr() - f.data_ptr()) // f.element_size()
            mask[start:start + t.numel()] = False
        assert same[mask].all()


def quantise(x, root):
    """One tensor's values -> e4m3 codes (uint8) and scales, with the operations the header names, each rounded to fp32."""
    import torch
    n = x.numel()
    b = torch.zeros((n + 255) // 256 * 256, device="cuda")
    b[:n] = x
    b = b.view(-1, 256)
    top = b.abs().amax(1, keepdim=True).clamp_min(2.0 ** -110)
    q = b * (top.reciprocal() * 448.0)
    if root:
        q = torch.where((b > 0) & (q < 2.0 ** -9), torch.full_like(q, 2.0 ** -9), q)
    return q.to(torch.float8_e4m3fn).view(torch.uint8).reshape(-1)[:n], (top * float(np.float32(1.0) / np.float32(448.0))).view(-1)


def dequantise(q, scale):
    import torch
    s = scale.repeat_interleave(256)[:q.numel()]
    return q.view(torch.float8_e4m3fn).float() * s


@pytest.mark.parametrize("p_dt,g_dt", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_adamw_8_codes_are_exact(api, p_dt, g_dt, shift):
    """Three steps: codes and scales equal those of the same fp32 operations, and the weights follow the unrounded moments."""
    import torch
    opt, pflat, mflat, vflat = make(api, ODD, p_dt, g_dt, 8, shift)
    lr = 0.01
    n = len(ODD)
    st = {k: [t.clone() for t in v] for k, v in opt.state.items()}
    for step in (1, 2, 3):
        for i, g in enumerate(opt.grads):
            g.copy_(torch.randn(g.shape, device="cuda") * 10.0 ** (i % 5 - 3) * torch.rand_like(g.float()).square())
            g[::7] = 0
        ps = [p.clone() for p in opt.params]
        opt.step(lr)
        torch.cuda.synchronize()
        assert opt.steps == step
        for i in range(n):
            if not ODD[i]:
                continue
            g = opt.grads[i].float()
            m = dequantise(st["exp_avg"][i], st["exp_avg_scale"][i])
            v = dequantise(st["exp_avg_sq"][i], st["exp_avg_sq_scale"][i]).square()
            m = m * 0.9 + g * (1.0 - 0.9)
            v = v * 0.999 + (g * g) * (1.0 - 0.999)
            mq, msc = quantise(m, False)
            vq, vsc = quantise(v.sqrt(), True)
            assert torch.equal(opt.state["exp_avg_scale"][i], msc) and torch.equal(opt.state["exp_avg_sq_scale"][i], vsc), i
            assert torch.equal(opt.state["exp_avg"][i].view(torch.uint8), mq), i
            assert torch.equal(opt.state["exp_avg_sq"][i].view(torch.uint8), vq), i
            wd = 0.1 if i % 2 else 0.0
            size = lr / (1 - 0.9 ** step) * m.double().abs() / ((v.double() / (1 - 0.999 ** step)).sqrt() + 1e-8)
            want = ps[i].double() * (1 - lr * wd) - size * m.double().sign()
            half = torch.finfo(dtype_of(p_dt)).eps / 2
            tol = 2.0 ** -24 * (12 * size + 5 * ps[i].double().abs()) + half * want.abs() + torch.finfo(dtype_of(p_dt)).smallest_normal * 2 * half
            assert ((opt.params[i].double() - want).abs() <= tol).all(), i
            st["exp_avg"][i].view(torch.uint8).copy_(mq)
            st["exp_avg_sq"][i].view(torch.uint8).copy_(vq)
            st["exp_avg_scale"][i].copy_(msc)
            st["exp_avg_sq_scale"][i].copy_(vsc)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(api, bits):
    """More tensors than one launch takes, in a shuffled order of memory: the same as one after the other."""
    import torch
    sizes = (ODD * 90)[:1100]
    a, *_ = make(api, sizes, "f32", "f32", bits, 0, seed=3, decay=0.05)
    order = np.random.default_rng(0).permutation(len(sizes))
    pick = lambda ts: [ts[j] for j in order]  # noqa: E731
    p2 = [p.clone() for p in a.params]
    st2 = {k: [t.clone() for t in v] for k, v in a.state.items()}
    b = api.AdamW(pick(a.params), pick(a.grads), state_bits=bits, weight_decay=0.05, state={k: pick(v) for k, v in a.state.items()})
    b.step(0.01, step=1)
    for i in range(0, len(sizes), 37):
        one = api.AdamW([p2[i]], [a.grads[i]], state_bits=bits, weight_decay=0.05, state={k: [v[i]] for k, v in st2.items()})
        one.step(0.01, step=1)
        assert torch.equal(p2[i], a.params[i])
        for k in st2:
            assert torch.equal(bits_of(st2[k][i]), bits_of(a.state[k][i]))


@pytest.mark.parametrize("bits", [32, 8])
def test_step_left_out_when_the_scale_is_not_finite(api, bits):
    import torch
    opt, pflat, mflat, vflat = make(api, ODD, "f32", "f32", bits, 0)
    before = [bits_of(f).clone() for f in (pflat, mflat, vflat)]
    opt.grads[6][3] = float("nan")
    norm = api.GradNorm(opt.grads)
    norm.run(1.0)
    opt.step(0.01, grad_scale=norm.clip)
    torch.cuda.synchronize()
    for f, b in zip((pflat, mflat, vflat), before):
        assert torch.equal(bits_of(f), b)


def test_zero_gradients_and_a_block_of_zeros(api):
    """A block that never saw a gradient stays at zero and its weights stay finite; tiny gradients do not overflow the scale."""
    import torch
    p = torch.ones(600, device="cuda")
    g = torch.zeros(600, device="cuda")
    g[300] = 1e-38
    g[599] = 1e-30
    opt = api.AdamW([p], [g], state_bits=8, weight_decay=0.0)
    for _ in range(3):
        opt.step(0.01)
    torch.cuda.synchronize()
    assert torch.isfinite(p).all() and (p[:256] == 1).all()
    assert not opt.state["exp_avg"][0].float()[:256].any() and not opt.state["exp_avg_sq"][0].float()[:256].any()
    assert torch.isfinite(opt.state["exp_avg_scale"][0]).all()


def test_captured_training_step(api):
    """Loss -> gradient -> norm -> update captured once and replayed with the step count and the rate on the device; an eager
    run of the same calls gives the same weights."""
    import torch
    torch.manual_seed(0)
    x = torch.randn(64, 32, device="cuda")
    t = torch.rand(64, 225, device="cuda")
    w0 = torch.randn(225, 32, device="cuda") * 0.1

    def build():
        s = {"w": w0.clone(), "g": torch.zeros_like(w0), "lr": torch.tensor(0.01, device="cuda"),
             "step": torch.zeros(1, dtype=torch.int32, device="cuda"), "z": torch.empty(64, 225, device="cuda"),
             "out": (torch.empty(64, device="cuda"), torch.empty(64, 225, device="cuda"), None)}
        s["norm"] = api.GradNorm([s["g"]])
        s["opt"] = api.AdamW([s["w"]], [s["g"]], state_bits=8)
        return s

    def one(s):
        s["step"].add_(1)
        torch.mm(x, s["w"].t(), out=s["z"])
        api.policy_loss_search(s["z"], t, out=s["out"])
        torch.mm(s["out"][1].t(), x, out=s["g"])
        s["norm"].run(0.5)
        s["opt"].step(s["lr"], step=s["step"], grad_scale=s["norm"].clip)

    a, b = build(), build()
    one(b)                                          # warm up, then from the start again
    b2 = build()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one(b2)
    b2["step"].zero_()
    for k in range(4):
        lr = 0.01 / (k + 1)
        a["lr"].fill_(lr)
        b2["lr"].fill_(lr)
        one(a)
        graph.replay()
    torch.cuda.synchronize()
    assert int(b2["step"]) == 4 and torch.equal(a["w"], b2["w"]) and not torch.equal(a["w"], w0)
    # and the host's step count and rate give what the device's give, to the rounding of the two factors
    h = build()
    for k in range(4):
        torch.mm(x, h["w"].t(), out=h["z"])
        api.policy_loss_search(h["z"], t, out=h["out"])
        torch.mm(h["out"][1].t(), x, out=h["g"])
        h["norm"].run(0.5)
        h["opt"].step(0.01 / (k + 1), grad_scale=h["norm"].clip)
    assert torch.allclose(h["w"], a["w"], rtol=0, atol=4 * 0.01 * 2.0 ** -20)


@pytest.mark.parametrize("bits", [32, 8])
def test_device_step_below_one_changes_nothing(api, bits):
    import torch
    opt, pflat, mflat, vflat = make(api, ODD, "f32", "f32", bits, 0)
    before = [bits_of(f).clone() for f in (pflat, mflat, vflat)]
    step = torch.zeros(1, dtype=torch.int32, device="cuda")
    for k in (0, -3):
        step.fill_(k)
        opt.step(0.01, step=step)
        assert all(torch.equal(bits_of(f), b) for f, b in zip((pflat, mflat, vflat), before))
    step.fill_(1)
    opt.step(0.01, step=step)
    assert not torch.equal(bits_of(pflat), before[0])


def test_plans_on_two_streams_and_in_two_graphs(api):
    """Plans of their own at the same time, and one plan in two graphs and without one: each norm is the one it gives alone."""
    import torch
    torch.manual_seed(1)
    lists = [[torch.randn(n + k, device="cuda") for n in (300000, 5, 70000) * 20] for k in (0, 1)]
    plans = [api.GradNorm(gs) for gs in lists]
    want = [p.run(1.0).clone() for p in plans]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in plans], [[], []]
    for _ in range(20):
        for s, p, out in zip(streams, plans, got):
            with torch.cuda.stream(s):
                out.append(p.run(1.0).clone())
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for out, w in zip(got, want) for x in out)
    graphs = []
    for limit in (1.0, 2.0):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            plans[0].run(limit)
    for i in (0, 1, 1, 0):
        graphs[i].replay()
        twice = plans[0].out.clone()
        assert torch.equal(twice[:1], want[0][:1]) and abs(float(twice[1] / want[0][1]) - (1 + i)) <= 2.0 ** -22
        assert torch.equal(plans[0].run(1.0), want[0])


FIRST = """
import torch
from omoknuni_small_b200 import capi
n = 6
z = {A: torch.randn(n, A, device="cuda") for A in (225, 4672, 40000, 300007)}
t = {A: torch.rand(n, A, device="cuda") for A in z}
act, one = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.ones(n, device="cuda")
p, g = [torch.ones(5000, device="cuda") for _ in range(2)]
norm, opt = capi.GradNorm([g]), capi.AdamW([p], [g], state_bits=8)
count = torch.zeros(1, dtype=torch.int32, device="cuda")
def calls():
    out = [x for A in z for x in capi.policy_loss_search(z[A], t[A])]
    out += [x for A in z for x in capi.policy_loss_clipped(z[A], act, -one, one, ref_logits=t[A], kl_coef=0.1)]
    norm.run(1.0)
    count.add_(1)
    opt.step(0.01, step=count, grad_scale=norm.clip)
    return out
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls()
graph.replay()
torch.cuda.synchronize()
w = p.clone()
assert float(norm.out[0]) > 1 and not (w == 1).any()
assert all(torch.equal(a, b) for a, b in zip(got, calls()))
"""


def test_first_call_of_a_process_is_captured(api):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_plans_are_made_outside_captures_and_run_on_any_stream(api):
    import torch
    p, g = [torch.ones(70000, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.add_(0)
        with pytest.raises(api.Error):
            api.GradNorm([g])
        with pytest.raises(api.Error):
            api.AdamW([p], [g])
    side = torch.cuda.Stream()
    big = torch.empty(1 << 28, device="cuda")
    for k in range(3):
        big.fill_(k)                                # keeps the stream of the plans busy
        norm, opt = api.GradNorm([g]), api.AdamW([p], [g], state_bits=8)
        with torch.cuda.stream(side):
            got = norm.run(1.0)
            opt.step(0.0, grad_scale=norm.clip)
        side.synchronize()
        assert abs(float(got[0]) - math.sqrt(70000.0)) <= 2.0 ** -20 * 265 and float(opt.state["exp_avg"][0].float().min()) == 448
        assert float(p.min()) == 1 == float(p.max())
