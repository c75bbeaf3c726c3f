"""Learning from self-play: the heads of a Gomoku network fitted to the records of selfplay.SelfPlay.

Takes the place of one optimiser step of the reference's learner (alphazero_train.py,
python/alphazero/alphazero_trainer.py: cross entropy with the search's policy plus squared error of the value, Adam) for
the two heads; the tower stays as it is and runs on the handle's own kernels.  A step is: positions -> planes -> tower
(capi.encode_gomoku, Net.tower_copy_device), heads forward (PyTorch), loss and its gradient over the legal moves
(capi.policy_loss_search / policy_loss_clipped), heads backward (PyTorch), norm of the gradients and the weight update
(capi.GradNorm, capi.AdamW).  weights() gives the whole network under the reference's names, for a new handle
(capi.Net(...).load) and for checkpoint.write_flat.
"""
import numpy as np

from . import capi

BN_EPS = 1e-5
HEADS = ("policy_conv", "policy_bn", "policy_fc", "value_conv", "value_bn", "value_fc1", "value_fc2")
FROZEN = ("running_mean", "running_var")


def positions_of(record):
    """(moves so far, policy, outcome for the side to move) for every recorded ply of a game."""
    opening = list(record.get("opening", ()))
    moves, winner = opening + list(record["moves"]), int(record["winner"])
    for i, pi in enumerate(record["policies"]):
        ply = len(opening) + i
        side = 1 if ply % 2 == 0 else 2
        yield moves[:ply], pi, 0.0 if winner == 0 else 1.0 if winner == side else -1.0


def batch_of(positions, board_size):
    """Host arrays of a batch: history [n, 16] int16 (most recent move first), n_hist and to_move [n] uint8, legal_bits
    [n, words] int32 (the empty cells), target [n, cells] float32, outcome [n] float32."""
    n, A = len(positions), board_size * board_size
    history, n_hist, to_move = np.full((n, 16), -1, np.int16), np.zeros(n, np.uint8), np.zeros(n, np.uint8)
    empty = np.zeros((n, (A + 31) // 32 * 32), np.uint8)
    empty[:, :A] = 1
    target, outcome = np.zeros((n, A), np.float32), np.zeros(n, np.float32)
    for i, (moves, pi, z) in enumerate(positions):
        recent = moves[::-1][:16]
        history[i, :len(recent)], n_hist[i], to_move[i] = recent, len(recent), 1 + len(moves) % 2
        empty[i, moves] = 0
        target[i], outcome[i] = pi, z
    bits = np.packbits(empty, axis=1, bitorder="little").view(np.int32).reshape(n, -1)
    return dict(history=history, n_hist=n_hist, to_move=to_move, legal_bits=np.ascontiguousarray(bits), target=target, outcome=outcome)


def check_positions(device, history, n_hist, to_move, outcome=None):
    """Refuses what the encoder would read out of its bounds or as something else."""
    import torch
    n = history.shape[0] if history.dim() else 0
    for t, what, shape, dtype in ((history, "history", (n, 16), torch.int16), (n_hist, "n_hist", (n,), torch.uint8), (to_move, "to_move", (n,), torch.uint8),
                                  (outcome, "outcome", (n,), None)):
        if t is not None and (tuple(t.shape) != shape or t.device != device or dtype not in (None, t.dtype) or (dtype and not t.is_contiguous())):
            raise capi.Error(capi.ERR_INVALID, f"HeadLearner: {what} is {shape} of {dtype or 'numbers'} on {device}, got {tuple(t.shape)} of "
                                               f"{t.dtype} on {t.device}")


class HeadLearner:
    """One optimiser over the heads of `net` (a finalised capi.Net for Gomoku) whose tensors are `weights`.  Steps run on
    PyTorch's current stream and return without waiting; the handle may answer and search between them.  A loss
    kernel that gave up on a wait makes its step's losses NaN and the step is left out; fit() and weights() report that, and a
    tower's, until capi.device_error_code() or a call of the handle has cleared the code.

    state_bits: AdamW states in 32 or 8 bits.  max_norm: the gradients' norm is clipped to it.  value_coef: factor of the
    squared error of the value.  The heads as they are at the start are the reference of the KL term of step_clipped."""

    def __init__(self, net, weights, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-4, state_bits=32, max_norm=1.0, value_coef=1.0,
                 entropy_coef=0.0):
        import torch
        self.torch, self.net, self.S, self.F = torch, net, net.board_size, net.cfg.filters
        if "policy_fc.weight" not in weights:
            raise capi.Error(capi.ERR_INVALID, "HeadLearner: the network's policy head is not the fully connected one")
        self.device = torch.device("cuda", net.cfg.device)
        self.all = {k: np.array(v, np.float32) for k, v in weights.items()}
        names = [k for k in weights if k.split(".")[0] in HEADS]
        self.fixed = {k: torch.from_numpy(self.all[k]).to(self.device) for k in names if k.endswith(FROZEN)}
        names = [k for k in names if not k.endswith(FROZEN)]
        # one buffer for the gradients, so that one call clears them
        sizes = [(self.all[k].size + 63) // 64 * 64 for k in names]
        self.flat_grad = torch.zeros(sum(sizes), device=self.device)
        self.params, at = {}, 0
        for k, size in zip(names, sizes):
            p = torch.from_numpy(self.all[k]).to(self.device).requires_grad_(True)
            p.grad = self.flat_grad[at:at + p.numel()].view(p.shape)
            self.params[k] = p
            at += size
        self.reference = {k: p.detach().clone() for k, p in self.params.items()}
        plain = [p.detach() for p in self.params.values()]
        grads = [p.grad for p in self.params.values()]
        self.norm = capi.GradNorm(grads)
        decay = [weight_decay if p.dim() > 1 else 0.0 for p in plain]          # filters and matrices only
        self.opt = capi.AdamW(plain, grads, state_bits=state_bits, betas=betas, eps=eps, weight_decay=decay)
        self.max_norm, self.value_coef, self.entropy_coef = max_norm, value_coef, entropy_coef

    def features(self, history, n_hist, to_move):
        """Tower output [n, filters, S, S] float32 of positions given as device arrays (capi.encode_gomoku)."""
        check_positions(self.device, history, n_hist, to_move)
        torch, S, n = self.torch, self.S, history.shape[0]
        channels = self.net.input_tensor_channels()
        if n > self.net.cfg.max_batch:
            raise capi.Error(capi.ERR_INVALID, f"HeadLearner: {n} positions, the handle takes {self.net.cfg.max_batch}")
        with torch.cuda.device(self.device):
            planes = capi.encode_gomoku(history, n_hist, to_move, S, self.net.cfg.input_channels, channels, self.net.tower_dtype)
            raw = self.net.tower_copy_device(planes, n)      # the handle's own memory belongs to its next call
            t = raw.view(torch.float16 if self.net.tower_dtype == capi.DTYPE_F16 else torch.bfloat16)
            G, GP = capi.GUARD, S + 1
            x = t.as_strided((n, self.F, S, S), (GP * GP * self.F, 1, GP * self.F, self.F), G * self.F)
            return x.float()

    def heads(self, x, params=None):
        """(logits [n, A], value [n]) of tower outputs, BatchNorm with its stored statistics."""
        f, p = self.torch.nn.functional, self.params if params is None else params

        cells = x.permute(0, 2, 3, 1)              # as the tower writes it

        def branch(name):
            # a matrix product in fp32: PyTorch's convolutions would round their operands to TF32
            y = f.linear(cells, p[name + "_conv.weight"][:, :, 0, 0])
            scale = p[name + "_bn.weight"] * self.torch.rsqrt(self.fixed[name + "_bn.running_var"] + BN_EPS)
            y = (y - self.fixed[name + "_bn.running_mean"]) * scale + p[name + "_bn.bias"]
            return f.relu(y).permute(0, 3, 1, 2).flatten(1)
        logits = f.linear(branch("policy"), p["policy_fc.weight"], p["policy_fc.bias"])
        v = f.relu(f.linear(branch("value"), p["value_fc1.weight"], p["value_fc1.bias"]))
        return logits, self.torch.tanh(f.linear(v, p["value_fc2.weight"], p["value_fc2.bias"])).flatten()

    def _backward(self, logits, grad, value, outcome, weight):
        """Gradients of both heads into the flat buffer; the value's loss, row by row."""
        torch = self.torch
        # a row of weight 0 may hold anything as its outcome
        off = torch.where(weight != 0, value.detach() - outcome, 0.0)
        self.flat_grad.zero_()
        torch.autograd.backward([logits, value], [grad, 2.0 * self.value_coef * weight * off])
        return self.value_coef * weight * off * off

    def _update(self, lr):
        norm = self.norm.run(self.max_norm)
        self.opt.step(lr, grad_scale=self.norm.clip)
        return norm.clone()                        # the next step writes the plan's own again

    def _weight(self, n, row_weight):
        torch = self.torch
        return torch.full((n,), 1.0 / n, device=self.device) if row_weight is None else row_weight

    def step_search(self, history, n_hist, to_move, target, outcome, legal_bits=None, row_weight=None, lr=1e-3):
        """One step towards the search's policies (`target`: visit counts int32, or float32) and the games' outcomes.
        Device arrays; row_weight [n] (default 1 / n), 0 for rows that fill up a batch.  Returns (loss of the policy rows
        [n], loss of the value rows [n], statistics of the policy rows [n, 4], (norm, factor)), all on the device."""
        check_positions(self.device, history, n_hist, to_move, outcome)
        w = self._weight(history.shape[0], row_weight)
        with self.torch.cuda.device(self.device):
            logits, value = self.heads(self.features(history, n_hist, to_move))
            loss, grad, stats = capi.policy_loss_search(logits.detach(), target, legal_bits, w, self.entropy_coef)
            value_loss = self._backward(logits, grad, value, outcome, w)
            norm = self._update(lr)
        return loss, value_loss, stats, norm

    def step_clipped(self, history, n_hist, to_move, action, old_logp, advantage, outcome, legal_bits=None, row_weight=None, clip=0.2,
                     kl_coef=0.0, lr=1e-3):
        """One step of the clipped-ratio objective on moves that were played: `old_logp` is the log-probability with which
        each was drawn; kl_coef holds the policy to that of the heads the learner started with.  Returns as step_search."""
        check_positions(self.device, history, n_hist, to_move, outcome)
        w = self._weight(history.shape[0], row_weight)
        with self.torch.cuda.device(self.device):
            x = self.features(history, n_hist, to_move)
            logits, value = self.heads(x)
            ref = None
            if kl_coef:
                with self.torch.no_grad():
                    ref = self.heads(x, self.reference)[0]
            loss, grad, stats = capi.policy_loss_clipped(logits.detach(), action, old_logp, advantage, legal_bits, ref, w, clip, clip, kl_coef,
                                                         self.entropy_coef)
            value_loss = self._backward(logits, grad, value, outcome, w)
            norm = self._update(lr)
        return loss, value_loss, stats, norm

    def fit(self, records, steps, batch=512, lr=1e-3, seed=0):
        """`steps` steps of step_search on positions drawn from self-play records.  Returns the mean losses [steps, 2]."""
        torch, rng = self.torch, np.random.default_rng(seed)
        pool = [p for r in records for p in positions_of(r) if sum(p[1]) > 0]
        if not pool:
            raise capi.Error(capi.ERR_INVALID, "HeadLearner.fit: the records hold no position with a policy")
        batch, seen = min(batch, self.net.cfg.max_batch), []
        for _ in range(steps):
            b = batch_of([pool[i] for i in rng.integers(0, len(pool), batch)], self.S)
            b = {k: torch.from_numpy(v).to(self.device) for k, v in b.items()}
            loss, value_loss, _, _ = self.step_search(b["history"], b["n_hist"], b["to_move"], b["target"], b["outcome"], b["legal_bits"], lr=lr)
            seen.append(torch.stack([loss.sum(), value_loss.sum()]))
        losses = torch.stack(seen).cpu().numpy() if seen else np.zeros((0, 2), np.float32)
        self._reported()
        return losses

    def weights(self):
        """Every tensor of the network under the reference's names, the heads as they are now (numpy float32)."""
        out = dict(self.all)
        out.update({k: p.detach().cpu().numpy().copy() for k, p in self.params.items()})
        self._reported()
        return out

    def _reported(self):
        """Raises what a kernel that gave up on a wait has left on the device; steps it had a part in were left out.  A search
        or an answer under way may have to read it too, so it stays."""
        with self.torch.cuda.device(self.device):
            code = capi.device_error_code(clear=False)
        if code:
            raise capi.Error(capi.ERR_TIMEOUT, f"HeadLearner: a kernel gave up on a bounded wait (code {code})")
