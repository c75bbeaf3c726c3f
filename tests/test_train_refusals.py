"""What the training operators refuse, and what their Python mirror refuses, without a device: arguments are checked first."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def api(lib):
    from omoknuni_small_b200 import capi
    return capi


def rows(api, **kw):
    base = dict(logits=0x10000, legal_bits=None, row_weight=None, grad=0x900000, loss=None, stats=None, logits_pitch=225, grad_pitch=225,
                n=8, n_actions=225, mask_words=0, dtype=api.DTYPE_F32)
    base.update(kw)
    return api.PolicyRows(**base)


def search(api, r, target=0x2000000, pitch=225, kind=0):
    return api.lib().ob200_launch_policy_loss_search(C.byref(r) if r is not None else None, target, pitch, kind, 0.0, None)


def clipped(api, r, act=0x3000000, old=0x3001000, adv=0x3002000, ref=None, pitch=0, lo=0.2, hi=0.2, kl=0.0):
    return api.lib().ob200_launch_policy_loss_clipped(C.byref(r) if r is not None else None, act, old, adv, ref, pitch, lo, hi, kl, 0.0, None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(grad=None), dict(n=-1), dict(n_actions=0), dict(logits_pitch=224), dict(grad_pitch=0), dict(dtype=7), dict(dtype=-1),
    dict(logits=0x10002), dict(grad=0x900001), dict(legal_bits=0x5000, mask_words=7), dict(legal_bits=0x5001, mask_words=8),
    dict(stats=0x5008), dict(row_weight=0x5002), dict(loss=0x5002),
    dict(grad=0x10000, grad_pitch=226),            # in place with another pitch
    dict(grad=0x10000 + 4), dict(grad=0x10000 + 8 * 225 * 4 - 4),      # overlaps
    dict(grad=0x10000 + 400, logits_pitch=450, grad_pitch=450),        # columns of one buffer that meet
])
def test_policy_rows_refused(api, bad):
    assert search(api, rows(api, **bad)) == api.ERR_INVALID
    assert clipped(api, rows(api, **bad)) == api.ERR_INVALID
    assert api.lib().ob200_last_error()


def test_policy_losses_refused(api):
    r = rows(api)
    assert search(api, rows(api, n_actions=(1 << 30) + 1, logits_pitch=1 << 31, grad_pitch=1 << 31)) == 7
    assert search(api, rows(api, logits_pitch=(1 << 31) + 1)) == api.ERR_INVALID
    assert search(api, None) == clipped(api, None) == api.ERR_INVALID
    assert search(api, r, target=None) == search(api, r, target=0x2000002) == search(api, r, pitch=224) == search(api, r, kind=2) == api.ERR_INVALID
    assert search(api, r, target=0x900000 + 64) == api.ERR_INVALID
    for kw in (dict(act=None), dict(old=None), dict(adv=0x3002001), dict(lo=-0.1), dict(hi=float("nan")), dict(kl=0.1),
               dict(ref=0x4000000, pitch=100, kl=0.1), dict(ref=0x4000002, pitch=225), dict(ref=0x900000, pitch=225)):
        assert clipped(api, r, **kw) == api.ERR_INVALID, kw


def test_allowed_placements_reach_the_device_check(api):
    """In place, and logits and gradient as columns of one buffer, are no argument errors."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a device: the pointers are made up")
    no_device = 2
    assert search(api, rows(api, grad=0x10000)) == no_device
    assert search(api, rows(api, grad=0x10000 + 900, logits_pitch=450, grad_pitch=450)) == no_device
    assert clipped(api, rows(api), ref=0x4000000, pitch=225, kl=0.1) == no_device
    assert search(api, rows(api, n=0, logits=None, grad=None), target=None) == no_device


def tensors(api, k=2, **kw):
    t = (api.TrainTensor * k)()
    for i in range(k):
        at = 0x100000 * (i + 1)
        t[i] = api.TrainTensor(at, at + 0x10000, at + 0x20000, at + 0x30000, at + 0x40000, at + 0x50000, 1000, 0.0)
    for name, v in kw.items():
        setattr(t[k - 1], name, v)
    return t


def config(api, **kw):
    base = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=1, param_dtype=api.DTYPE_F32, grad_dtype=api.DTYPE_F32, state_bits=32)
    base.update(kw)
    return api.AdamWConfig(**base)


def test_adamw_refused(api):
    L = api.lib()

    def call(t, c, n=2):
        return L.ob200_launch_adamw(t, n, C.byref(c) if c is not None else None, None)
    assert call(tensors(api), None) == call(None, config(api)) == call(tensors(api), config(api), -1) == api.ERR_INVALID
    for kw in (dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(numel=-1), dict(param=0x200002),
               dict(grad=0x210001), dict(exp_avg=0x220002), dict(exp_avg_sq=0x220000),
               dict(param=0x100000), dict(param=0x100000 + 3996), dict(exp_avg=0x120000 - 4), dict(exp_avg_sq=0x130000)):
        assert call(tensors(api, **kw), config(api)) == api.ERR_INVALID, kw
    assert call(tensors(api, numel=1 << 43), config(api)) == 7
    for kw in (dict(exp_avg_scale=None), dict(exp_avg_sq_scale=None), dict(exp_avg_scale=0x240002)):
        assert call(tensors(api, **kw), config(api, state_bits=8)) == api.ERR_INVALID, kw
    for kw in (dict(step=0), dict(param_dtype=3), dict(grad_dtype=-1), dict(state_bits=16), dict(beta1=1.0), dict(beta2=-0.1),
               dict(eps=float("nan")), dict(grad_scale=0x5002), dict(step_device=0x5001), dict(lr_device=0x5003)):
        assert call(tensors(api), config(api, **kw)) == api.ERR_INVALID, kw


def test_grad_norm_refused(api):
    L = api.lib()

    def call(t, n=2, dtype=2, most=1.0, ws=0x7000, out=0x8000):
        return L.ob200_launch_grad_norm(t, n, dtype, most, ws, out, None)
    t = tensors(api)
    assert call(None) == call(t, -1) == call(t, dtype=5) == call(t, most=0.0) == call(t, most=float("nan")) == api.ERR_INVALID
    assert call(t, ws=None) == call(t, ws=0x7004) == call(t, out=None) == call(t, out=0x8002) == api.ERR_INVALID
    assert call(tensors(api, grad=None)) == call(tensors(api, grad=0x210002)) == call(tensors(api, numel=-5)) == api.ERR_INVALID
    assert L.ob200_grad_norm_workspace_bytes() > 0


def test_python_mirror_refuses(api):
    import torch
    z = torch.zeros(4, 9)
    with pytest.raises(api.Error, match="CUDA device"):
        api.policy_loss_search(z, torch.zeros(4, 9))
    for args, kw in (((z[0], z), {}), ((z.double(), z), {}), ((z, torch.zeros(4, 8)), {}), ((z, z.double()), {}),
                     ((z.t(), torch.zeros(9, 4)), {}), ((z, z), dict(row_weight=torch.zeros(3))),
                     ((z, z), dict(legal_bits=torch.zeros(4, 1))), ((z, z), dict(row_weight=torch.zeros(8)[::2]))):
        with pytest.raises(api.Error) as e:
            api.policy_loss_search(*args, **kw)
        assert e.value.code == api.ERR_INVALID
    with pytest.raises(api.Error):
        api.policy_loss_clipped(z, torch.zeros(4), torch.zeros(4), torch.zeros(4))
    for make in (lambda: api.GradNorm([]), lambda: api.GradNorm([z, z.bfloat16()]), lambda: api.GradNorm([z.t()]), lambda: api.GradNorm([z]),
                 lambda: api.AdamW([z], []), lambda: api.AdamW([z], [z], state_bits=4), lambda: api.AdamW([z], [z]),
                 lambda: api.AdamW([z], [z], weight_decay=[0.1, 0.2]), lambda: api.AdamW([z, z.half()], [z, z])):
        with pytest.raises(api.Error):
            make()
