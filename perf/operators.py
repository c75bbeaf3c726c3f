"""Performance cases of the training operators: what a learner calls between the search's visit counts and the next weights.

  policy_loss_search   cross entropy of a policy with the search's visit distribution over the legal moves, and its gradient
  policy_loss_clipped  clipped-ratio policy loss with a KL term against a reference policy, and its gradient
  grad_norm            2-norm of all gradients of a network and the factor that clips it
  adamw                AdamW over all tensors of a network, states in 32 or 8 bits

  listed()          the named cases
  draw(rng)         one more case of the same ranges
  prepare(case, s)  what a learner holds before the call
  run(state)        one pass: in elementary torch operations, or (own = True) through the library's entry points
  work(case)        bytes and floating-point operations the pass cannot do without
  exact(case, s)    the same outputs from the definition in 64 bits
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
LOSS_SCALE = {"f32": 1.0, "bf16": 1.0, "f16": 1024.0}      # fp16 gradients of a mean over many rows need one
BLOCK = 256                        # elements that share a scale of an 8-bit state
E4M3_MAX = 448.0
E4M3_LEAST = 2.0 ** -9             # smallest positive e4m3 value
SCALE_FLOOR = 2.0 ** -110          # block maxima below this are taken as this
CLIP, KL, ENTROPY = 0.2, 0.1, 0.01
LR, BETA1, BETA2, EPS, STEP, MAX_NORM = 1e-3, 0.9, 0.999, 1e-8, 100, 1.0


# ---- the cases ------------------------------------------------------------------
def _rows(kind, n, actions, dtype, mask=True, **kw):
    return dict(kw, kind=kind, n=n, actions=actions, dtype=dtype, mask=mask)


def _net(kind, filters, blocks, planes, board, policy, head, dtype="f32", **kw):
    return dict(kw, kind=kind, filters=filters, blocks=blocks, planes=planes, board=board, policy=policy, head=head, dtype=dtype)


def listed():
    return [
        # the positions of one short game, Gomoku: the launch itself counts
        _rows("clipped", 8, 225, "f32", ref=True, name="clipped_gomoku_8"),
        # a learner's batch of chess positions, 16-bit logits
        _rows("clipped", 2048, 4672, "bf16", ref=True, name="clipped_chess_2048"),
        # few positions with a very large action space
        _rows("clipped", 37, 65536, "f16", ref=True, mask=False, name="clipped_37x65536"),
        # a whole shard over a wide action space: memory bandwidth
        _rows("clipped", 4096, 32768, "bf16", ref=True, mask=False, name="clipped_4096x32768"),
        # a learner's batch from self-play records: visit counts as the search returns them
        _rows("search", 512, 225, "f32", target="visits", name="search_gomoku_512"),
        # a replay shard, Go 19x19 with pass, 16-bit logits, visit distributions
        _rows("search", 65536, 362, "bf16", target="pi", name="search_go_65536"),
        # a replay shard of chess positions
        _rows("search", 8192, 4672, "f32", target="pi", name="search_chess_8192"),
        # gradients of the 64-filter Gomoku network with the reference's 32-channel heads
        _net("norm", 64, 10, 17, 15, 225, 32, name="norm_gomoku"),
        # 16-bit gradients of the 256-filter network
        _net("norm", 256, 20, 119, 8, 4672, 2, dtype="bf16", name="norm_256x20"),
        # the weight update of the Gomoku network, clipped to norm 1
        _net("adamw", 64, 10, 17, 15, 225, 32, bits=32, clip=True, name="adamw_gomoku"),
        # the 256-filter network, states in 8 bits, clipped
        _net("adamw", 256, 20, 119, 8, 4672, 2, bits=8, clip=True, name="adamw_256x20_8bit"),
        # 1,024 filters, 20 layers: far larger than the caches, 16-bit weights, states in 32 bits
        _net("adamw", 1024, 10, 119, 8, 4672, 2, dtype="bf16", bits=32, clip=False, name="adamw_1024x10_bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["clipped", "clipped", "search", "search", "norm", "adamw", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind in ("clipped", "search"):
        actions = rng.choice([225, 362, 4672, _log_int(rng, 2, 1024), _log_int(rng, 256, 65536), _log_int(rng, 256, 65536)])
        n = _log_int(rng, 1, min(65536, (1 << 26) // actions))
        case = _rows(kind, n, actions, dtype, mask=rng.random() < 0.7)
        case["pad"] = rng.choice([0, 0, 0, 1, 7, 8])            # columns between rows that belong to somebody else
        if kind == "clipped":
            case["ref"] = rng.random() < 0.8
        else:
            case["target"] = rng.choice(["visits", "pi"])
        return case
    board = rng.choice([8, 9, 15, 19])
    case = _net(kind, rng.choice([64, 128, 256, rng.randint(8, 448)]), rng.randint(0, 20), rng.choice([3, 17, 19, 119]), board,
                rng.choice([board * board, board * board + 1, 4672]), rng.choice([1, 2, 32]), dtype)
    case["shift"] = rng.choice([0, 0, 1, 3])                    # elements by which all tensors are off their alignment
    if kind == "adamw":
        case["bits"] = rng.choice([32, 8])
        case["clip"] = rng.random() < 0.5
    return case


# ---- inputs of the policy losses ------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    return g


def _pack_bits(legal):
    n, A = legal.shape
    words = (A + 31) // 32
    padded = torch.zeros((n, words * 32), dtype=torch.int64, device=legal.device)
    padded[:, :A] = legal
    w = (padded.view(n, words, 32) << torch.arange(32, device=legal.device)).sum(2)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _pitched(x, pad):
    """The same values in rows `pad` elements further apart."""
    if not pad:
        return x.contiguous()
    wide = torch.zeros((x.shape[0], x.shape[1] + pad), dtype=x.dtype, device=x.device)
    wide[:, :x.shape[1]] = x
    return wide[:, :x.shape[1]]


def _prepare_rows(case, seed):
    g = _gen(seed)
    n, A, dt, pad = case["n"], case["actions"], DTYPES[case["dtype"]], case.get("pad", 0)
    s = {"case": case}
    z = torch.randn((n, A), generator=g, device=DEVICE).mul_(2.0)
    s["logits"] = _pitched(z.to(dt), pad)
    legal = None
    if case["mask"]:
        # 30 to 100 % of the moves are legal, in some rows a single one, in some (finished games) none
        share = torch.rand((n, 1), generator=g, device=DEVICE).mul_(0.7).add_(0.3)
        legal = torch.rand((n, A), generator=g, device=DEVICE) < share
        odd = torch.rand(n, generator=g, device=DEVICE)
        legal[odd < 0.03] = False
        legal[odd < 0.02, 0] = True
        s["legal_bits"] = _pack_bits(legal)
    else:
        s["legal_bits"] = None
    # rows that fill up a batch have weight 0
    w = torch.rand(n, generator=g, device=DEVICE).add_(0.5).mul_(LOSS_SCALE[case["dtype"]] / n)
    s["weight"] = torch.where(torch.rand(n, generator=g, device=DEVICE) < 0.02, torch.zeros_like(w), w)
    s["weight"][0] = LOSS_SCALE[case["dtype"]] / n
    zf = s["logits"].float()
    if legal is not None:
        zf = zf.masked_fill(~legal, -math.inf)
    if case["kind"] == "clipped":
        if case["ref"]:
            s["ref"] = _pitched((z + torch.randn((n, A), generator=g, device=DEVICE).mul_(0.4)).to(dt), pad)
        else:
            s["ref"] = None
        key = torch.rand((n, A), generator=g, device=DEVICE)
        if legal is not None:
            key.masked_fill_(~legal, -1.0)
        s["action"] = key.argmax(1).to(torch.int32)
        lse = torch.logsumexp(zf.double(), 1)
        logp = zf.double().gather(1, s["action"].long()[:, None])[:, 0] - lse
        d = torch.randn(n, generator=g, device=DEVICE, dtype=torch.float64).mul_(0.25)
        # the gradient jumps where the ratio crosses the border: no row stands within a thousandth of it, where the
        # rounding of 32 bits would decide
        for border in (math.log1p(-CLIP), math.log1p(CLIP)):
            d = torch.where((d - border).abs() < 1e-3, torch.full_like(d, border + 2e-3), d)
        old = (logp - d).nan_to_num(0.0, 0.0, 0.0)
        s["old_logp"] = old.float()
        s["advantage"] = torch.randn(n, generator=g, device=DEVICE)
    else:
        # a sharpened, noisy version of the policy, as a search of 800 simulations leaves it
        t = torch.softmax(zf + torch.randn((n, A), generator=g, device=DEVICE), 1).nan_to_num(0.0)
        s["target"] = _pitched((t * 800.0).round().to(torch.int32) if case["target"] == "visits" else t, pad)
    s["grad"] = _pitched(torch.zeros((n, A), dtype=dt, device=DEVICE), pad)
    s["loss"] = torch.zeros(n, dtype=torch.float32, device=DEVICE)
    s["stats"] = torch.zeros((n, 4), dtype=torch.float32, device=DEVICE)
    return s


# ---- the policy losses in plain form --------------------------------------------------------
def _legal(s):
    n, A = s["logits"].shape
    if s["legal_bits"] is None:
        return torch.ones((n, A), dtype=torch.bool, device=s["logits"].device)
    at = torch.arange(A, device=s["logits"].device)
    return ((s["legal_bits"][:, at >> 5] >> (at & 31).to(torch.int32)) & 1).bool()


def _log_softmax(z):
    """log of the softmax over the last axis of z, -inf in places that are out; rows without any place: all -inf."""
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    d = z - m
    return d - torch.log(torch.exp(d).sum(1, keepdim=True))


def _clipped(s, f):
    """The definition, computed in the type f: loss, gradient, (log-probability of the action, ratio, KL, entropy)."""
    legal = _legal(s)
    logp = _log_softmax(s["logits"].to(f).masked_fill(~legal, -math.inf))
    a = s["action"].long()[:, None]
    live = (s["weight"] != 0) & legal.gather(1, a)[:, 0]
    p = torch.where(live[:, None] & legal, torch.exp(logp), 0.0)
    logp = torch.where(p > 0, logp, 0.0)
    la = logp.gather(1, a)[:, 0]
    adv = s["advantage"].to(f)
    ratio = torch.exp(la - s["old_logp"].to(f))
    free, held = ratio * adv, ratio.clamp(1.0 - CLIP, 1.0 + CLIP) * adv
    c = torch.where(free <= held, -free, 0.0)
    H = -(p * logp).sum(1)
    loss = -torch.minimum(free, held) - ENTROPY * H
    grad = -c[:, None] * p
    grad.scatter_add_(1, a, c[:, None])
    grad = grad + ENTROPY * p * (logp + H[:, None])
    kl = torch.zeros_like(H)
    if s["ref"] is not None:
        x = torch.where(p > 0, logp - _log_softmax(s["ref"].to(f).masked_fill(~legal, -math.inf)), 0.0)
        kl = (p * x).sum(1)
        loss = loss + KL * kl
        grad = grad + KL * p * (x - kl[:, None])
    w = s["weight"].to(f)
    loss, grad = torch.where(live, w * loss, 0.0), torch.where(live[:, None], w[:, None] * grad, 0.0)
    stats = torch.where(live[:, None], torch.stack([la, ratio, kl, H], 1), 0.0)
    return loss, grad, stats


def _search(s, f):
    """The definition, computed in the type f: loss, gradient, (cross entropy, entropy, sum of the target, log of the sum)."""
    legal = _legal(s)
    z = s["logits"].to(f).masked_fill(~legal, -math.inf)
    t = s["target"].to(f).masked_fill(~legal, 0.0)
    total = t.sum(1)
    live = (s["weight"] != 0) & (total > 0)
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    lse = m[:, 0] + torch.log(torch.exp(z - m).sum(1))
    lse = torch.where(live, lse, 0.0)
    logp = torch.where(legal, z - lse[:, None], 0.0)
    p = torch.where(legal, torch.exp(logp), 0.0)
    pi = t / torch.where(live, total, 1.0)[:, None]
    ce = -(pi * logp).sum(1)
    H = -(p * logp).sum(1)
    w = s["weight"].to(f)
    loss = torch.where(live, w * (ce - ENTROPY * H), 0.0)
    grad = torch.where(live[:, None], w[:, None] * (p - pi + ENTROPY * p * (logp + H[:, None])), 0.0)
    stats = torch.where(live[:, None], torch.stack([ce, H, total, lse], 1), 0.0)
    return loss, grad, stats


# ---- inputs of the weight update ---------------------------------------------------------------
def _tensors(case):
    """(elements, weight decay) of each trained tensor of the residual network: convolutions, their BatchNorm factors and
    offsets, the two heads.  Only matrices and filters decay."""
    F, S2, hc = case["filters"], case["board"] * case["board"], case["head"]
    conv = [(case["planes"] * F * 9, 1e-2), (F, 0.0), (F, 0.0)] + 2 * case["blocks"] * [(F * F * 9, 1e-2), (F, 0.0), (F, 0.0)]
    heads = 2 * [(F * hc, 1e-2), (hc, 0.0), (hc, 0.0)]
    fc = [(case["policy"] * hc * S2, 1e-2), (case["policy"], 0.0), (256 * hc * S2, 1e-2), (256, 0.0), (256, 1e-2), (1, 0.0)]
    return conv + heads + fc


def _slots(case):
    """Elements each tensor takes in a flat buffer: whole blocks."""
    return [(k + BLOCK - 1) // BLOCK * BLOCK for k, _ in _tensors(case)]


def _flat(case, dtype):
    """A zeroed flat buffer of whole blocks, `shift` elements off its allocation."""
    shift = case.get("shift", 0)
    return torch.zeros(sum(_slots(case)) + shift, dtype=dtype, device=DEVICE)[shift:]


def _views(case, flat):
    out, at = [], 0
    for (k, _), slot in zip(_tensors(case), _slots(case)):
        out.append(flat[at:at + k])
        at += slot
    return out


def _prepare_net(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    sizes, slots = [k for k, _ in _tensors(case)], _slots(case)
    total = sum(slots)
    at = torch.arange(total, device=DEVICE)
    starts = torch.tensor([0] + slots, device=DEVICE).cumsum(0)
    which = torch.repeat_interleave(torch.arange(len(sizes), device=DEVICE), torch.tensor(slots, device=DEVICE))
    real = at - starts[which] < torch.tensor(sizes, device=DEVICE)[which]        # False in the gaps between tensors
    # gradients of one tensor differ in size from another's by orders of magnitude
    size = torch.exp(torch.rand(len(sizes), generator=g, device=DEVICE) * 5.0 - 10.0)[which] * real
    del at, which
    s["g"] = _flat(case, dt)
    s["g"].copy_(torch.randn(total, generator=g, device=DEVICE) * size)
    if case["kind"] == "adamw":
        s["p"] = _flat(case, dt)
        s["p"].copy_(torch.randn(total, generator=g, device=DEVICE) * 0.05 * real)
        m = torch.randn(total, generator=g, device=DEVICE) * size * 0.3
        v = (torch.randn(total, generator=g, device=DEVICE).square() + 0.1) * size.square()
        if case["bits"] == 32:
            s["m"], s["v"] = _flat(case, torch.float32), _flat(case, torch.float32)
            s["m"].copy_(m)
            s["v"].copy_(v)
        else:
            s["m"], s["v"] = _flat(case, torch.float8_e4m3fn), _flat(case, torch.float8_e4m3fn)
            for key, (q, scale) in (("m", _quantise(m)), ("v", _quantise_root(v.sqrt()))):
                s[key].copy_(q)
                s[key + "_scale"] = scale
        s["decay"] = torch.repeat_interleave(torch.tensor([d for _, d in _tensors(case)], device=DEVICE),
                                             torch.tensor(slots, device=DEVICE) // BLOCK)
    s["norm"] = torch.zeros(2, dtype=torch.float32, device=DEVICE)
    if own:
        from omoknuni_small_b200 import capi
        grads = _views(case, s["g"])
        s["norm_plan"] = capi.GradNorm(grads, out=s["norm"])
        if case["kind"] == "adamw":
            state = {"exp_avg": _views(case, s["m"]), "exp_avg_sq": _views(case, s["v"])}
            if case["bits"] == 8:
                at = 0
                for key in ("exp_avg_scale", "exp_avg_sq_scale"):
                    state[key] = []
                for slot in slots:
                    state["exp_avg_scale"].append(s["m_scale"][at:at + slot // BLOCK])
                    state["exp_avg_sq_scale"].append(s["v_scale"][at:at + slot // BLOCK])
                    at += slot // BLOCK
            s["plan"] = capi.AdamW(_views(case, s["p"]), grads, state_bits=case["bits"], betas=(BETA1, BETA2), eps=EPS,
                                   weight_decay=[d for _, d in _tensors(case)], state=state)
    return s


# ---- the weight update in plain form -----------------------------------------------------------------
def _quantise(x):
    """Blocks of 256 values -> e4m3 codes and the scale of each block, its largest magnitude over 448."""
    b = x.view(-1, BLOCK)
    top = b.abs().amax(1, keepdim=True).clamp_min(SCALE_FLOOR)
    return (b * (E4M3_MAX / top)).to(torch.float8_e4m3fn).view(-1), (top / E4M3_MAX).view(-1)


def _quantise_root(r):
    """The same for the root of the second moment: what is not zero does not become zero."""
    b = r.view(-1, BLOCK)
    top = b.amax(1, keepdim=True).clamp_min(SCALE_FLOOR)
    x = b * (E4M3_MAX / top)
    return torch.where(b > 0, x.clamp_min(E4M3_LEAST), x).to(torch.float8_e4m3fn).view(-1), (top / E4M3_MAX).view(-1)


def _norm(s):
    # a sum of up to 10^8 squares: in 64 bits
    total = s["g"].double().square().sum().sqrt()
    return total, torch.where(total > MAX_NORM, MAX_NORM / total, torch.ones_like(total))


def _update(s, f, clip):
    """One step in the type f from the states as they are held: new weights, first moment, second moment (its root in 8 bits)."""
    bits, blocks = s["case"]["bits"], (-1, BLOCK)
    g = s["g"].to(f).view(blocks)
    if clip is not None:
        g = g * clip.to(f)
    if bits == 32:
        m, v = s["m"].to(f).view(blocks), s["v"].to(f).view(blocks)
    else:
        m = s["m"].to(f).view(blocks) * s["m_scale"].to(f)[:, None]
        v = (s["v"].to(f).view(blocks) * s["v_scale"].to(f)[:, None]).square()
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    r = v.sqrt()
    p = s["p"].to(f).view(blocks) * (1.0 - LR * s["decay"].to(f)[:, None])
    p = p - (LR / (1.0 - BETA1 ** STEP)) * m / (r / math.sqrt(1.0 - BETA2 ** STEP) + EPS)
    return p.view(-1), m.view(-1), (v if bits == 32 else r).view(-1)


# ---- the interface -----------------------------------------------------------------------------------
def prepare(case, seed):
    return _prepare_rows(case, seed) if case["kind"] in ("clipped", "search") else _prepare_net(case, seed)


def _run_own(s):
    from omoknuni_small_b200 import capi
    case = s["case"]
    kind = case["kind"]
    if kind == "clipped":
        return capi.policy_loss_clipped(s["logits"], s["action"], s["old_logp"], s["advantage"], legal_bits=s["legal_bits"],
                                        ref_logits=s["ref"], row_weight=s["weight"], clip_low=CLIP, clip_high=CLIP,
                                        kl_coef=KL if s["ref"] is not None else 0.0, entropy_coef=ENTROPY,
                                        out=(s["loss"], s["grad"], s["stats"]))
    if kind == "search":
        return capi.policy_loss_search(s["logits"], s["target"], legal_bits=s["legal_bits"], row_weight=s["weight"],
                                       entropy_coef=ENTROPY, out=(s["loss"], s["grad"], s["stats"]))
    if kind == "norm":
        return s["norm_plan"].run(MAX_NORM)
    if case["clip"]:
        s["norm_plan"].run(MAX_NORM)
    s["plan"].step(LR, step=STEP, grad_scale=s["norm_plan"].clip if case["clip"] else None)
    return _net_outputs(s)


def _net_outputs(s):
    out = {k: s[k] for k in ("p", "m", "v")}
    if s["case"]["bits"] == 8:
        out.update(m_scale=s["m_scale"], v_scale=s["v_scale"])
    if s["case"]["clip"]:
        out["norm"] = s["norm"]
    return out


def run(state):
    s = state
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind in ("clipped", "search"):
        loss, grad, stats = (_clipped if kind == "clipped" else _search)(s, torch.float32)
        s["loss"].copy_(loss)
        s["grad"].copy_(grad)
        s["stats"].copy_(stats)
        return s["loss"], s["grad"], s["stats"]
    clip = None
    if kind == "norm" or s["case"]["clip"]:
        total, clip = _norm(s)
        s["norm"][0] = total
        s["norm"][1] = clip
        if kind == "norm":
            return s["norm"]
        clip = s["norm"][1]
    p, m, v = _update(s, torch.float32, clip)
    s["p"].copy_(p)
    if s["case"]["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        q, scale = _quantise(m)
        s["m"].copy_(q)
        s["m_scale"].copy_(scale)
        q, scale = _quantise_root(v)
        s["v"].copy_(q)
        s["v_scale"].copy_(scale)
    return _net_outputs(s)


def work(case):
    kind, e = case["kind"], BYTES[case["dtype"]]
    if kind in ("clipped", "search"):
        n, A = case["n"], case["actions"]
        second = e if kind == "clipped" and case["ref"] else 4 if kind == "search" else 0
        mask = n * ((A + 31) // 32) * 4 if case["mask"] else 0
        return {"bytes": n * A * (2 * e + second) + mask + n * (4 + 16 + 16), "flops": n * A * (14 if second else 10)}
    total = sum(k for k, _ in _tensors(case))
    if kind == "norm":
        return {"bytes": total * e + 8, "flops": 2 * total}
    # gradient, weight twice, two states twice; the scales of 8-bit states
    states = 16 if case["bits"] == 32 else 4 + 16.0 / BLOCK
    return {"bytes": total * (3 * e + states), "flops": total * (17 if case["clip"] else 14)}


# ---- the outputs in 64 bits, from the definitions --------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm" or (kind == "adamw" and case["clip"]):
        norm = torch.linalg.vector_norm(s["g"].double())
        factor = min(1.0, MAX_NORM / float(norm))
        both = torch.tensor([float(norm), factor], dtype=torch.float64, device=DEVICE)
        if kind == "norm":
            return both
    if kind == "adamw":
        return _exact_update(s, both if case["clip"] else None)
    n, A = s["logits"].shape
    loss = torch.zeros(n, dtype=torch.float64, device=DEVICE)
    grad = torch.zeros((n, A), dtype=torch.float64, device=DEVICE)
    stats = torch.zeros((n, 4), dtype=torch.float64, device=DEVICE)
    step = max(1, (1 << 25) // A)
    for lo in range(0, n, step):
        sl = slice(lo, min(n, lo + step))
        logits = s["logits"][sl].double()
        legal = torch.ones_like(logits, dtype=torch.bool)
        if s["legal_bits"] is not None:
            words = s["legal_bits"][sl].long() & 0xFFFFFFFF
            legal = ((words[:, :, None] >> torch.arange(32, device=DEVICE)) & 1).bool().reshape(len(words), -1)[:, :A]
        masked = torch.where(legal, logits, -math.inf)
        rows = legal.any(1) & (s["weight"][sl] != 0)
        weight = s["weight"][sl].double()
        # only rows that count; autograd gives the gradient
        part = (_exact_clipped if kind == "clipped" else _exact_search)(s, sl, masked, legal, rows, weight)
        if part is not None:
            keep, l, d, st = part
            at = lo + keep
            loss[at], grad[at], stats[at] = l, d, st
    return loss, grad, stats


def _exact_clipped(s, sl, masked, legal, rows, weight):
    keep = rows.nonzero()[:, 0]
    if not len(keep):
        return None
    z = masked[keep].requires_grad_(True)
    lp = torch.log_softmax(z, 1)
    act = s["action"][sl].long()[keep]
    la = lp[torch.arange(len(keep), device=DEVICE), act]
    zero = torch.zeros((), dtype=torch.float64, device=DEVICE)
    safe = torch.where(legal[keep], lp, zero)
    prob = torch.where(legal[keep], safe.exp(), zero)
    entropy = -(prob * safe).sum(1)
    ratio = (la - s["old_logp"][sl].double()[keep]).exp()
    adv = s["advantage"][sl].double()[keep]
    gain = torch.where(adv >= 0, torch.clamp(ratio, max=1.0 + CLIP), torch.clamp(ratio, min=1.0 - CLIP)) * adv
    kl = torch.zeros_like(entropy)
    total = -gain - ENTROPY * entropy
    if s["ref"] is not None:
        lq = torch.log_softmax(torch.where(legal[keep], s["ref"][sl].double()[keep], -math.inf), 1)
        kl = (prob * (safe - torch.where(legal[keep], lq, zero))).sum(1)
        total = total + KL * kl
    total = total * weight[keep]
    d, = torch.autograd.grad(total.sum(), z)
    return keep, total.detach(), torch.where(legal[keep], d, zero), torch.stack([la, ratio, kl, entropy], 1).detach()


def _exact_search(s, sl, masked, legal, rows, weight):
    t = torch.where(legal, s["target"][sl].double(), torch.zeros((), dtype=torch.float64, device=DEVICE))
    keep = (rows & (t.sum(1) > 0)).nonzero()[:, 0]
    if not len(keep):
        return None
    t = t[keep]
    z = masked[keep].requires_grad_(True)
    zero = torch.zeros((), dtype=torch.float64, device=DEVICE)
    safe = torch.where(legal[keep], torch.log_softmax(z, 1), zero)
    prob = torch.where(legal[keep], safe.exp(), zero)
    entropy = -(prob * safe).sum(1)
    ce = -(t * safe).sum(1) / t.sum(1)
    total = (ce - ENTROPY * entropy) * weight[keep]
    d, = torch.autograd.grad(total.sum(), z)
    lse = torch.logsumexp(masked[keep], 1)
    return keep, total.detach(), torch.where(legal[keep], d, zero), torch.stack([ce, entropy, t.sum(1), lse], 1).detach()


def _exact_update(s, norm):
    """States in 8 bits have no 64-bit value: a value between two codes may fall to either."""
    case = s["case"]
    g = s["g"].double()
    if norm is not None:
        g = g * norm[1]
    per_block = torch.arange(len(g), device=DEVICE) // BLOCK
    m, v = s["m"].double(), s["v"].double()
    if case["bits"] == 8:
        m = m * s["m_scale"].double()[per_block]
        v = (v * s["v_scale"].double()[per_block]) ** 2
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g ** 2, v, BETA2)
    rate = m / (1.0 - BETA1 ** STEP) / (torch.sqrt(v / (1.0 - BETA2 ** STEP)) + EPS) + s["decay"].double()[per_block] * s["p"].double()
    out = {"p": s["p"].double() - LR * rate, "m": m if case["bits"] == 32 else None, "v": v if case["bits"] == 32 else None}
    if case["bits"] == 8:
        tops = m.view(-1, BLOCK).abs().amax(1), v.view(-1, BLOCK).amax(1).sqrt()
        out["m_scale"], out["v_scale"] = (torch.clamp(top, min=SCALE_FLOOR) / E4M3_MAX for top in tops)
    if norm is not None:
        out["norm"] = norm
    return out
