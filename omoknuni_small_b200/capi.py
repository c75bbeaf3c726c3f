"""ctypes bindings of libomoknuni_b200.so — the Python host-side mirror of the
C ABI in include/omoknuni_b200.h.  Used by the tests and by bench.py.

Loading fails loudly when the library has not been built; there is no
fallback implementation.
"""
import ctypes as C
import os
import threading

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libomoknuni_b200.so")

OUT_PROBS, OUT_LOGITS = 0, 1
GUARD = 32
RULES_FREESTYLE, RULES_OMOK, RULES_RENJU = 0, 1, 2
DTYPE_BF16, DTYPE_F16 = 0, 1     # storage type of board tensors and packed tower weights
DTYPE_F32 = 2                    # policy rows, gradients and weights of the training operators
TARGET_VISITS, TARGET_PROBS = 0, 1
ERR_INVALID, ERR_TIMEOUT = 1, 6


class Error(RuntimeError):
    def __init__(self, code, text):
        super().__init__(f"omoknuni_b200 error {code}: {text}")
        self.code = code


class TreeView(C.Structure):
    _fields_ = [("N", C.c_void_p), ("W", C.c_void_p), ("P", C.c_void_p), ("VL", C.c_void_p),
                ("legal_bits", C.c_void_p), ("node_visits", C.c_void_p), ("child_node", C.c_void_p),
                ("n_nodes", C.c_int32), ("n_children", C.c_int32), ("pitch", C.c_int32), ("mask_words", C.c_int32)]


POLICY_FC, POLICY_CONV_PLANES = 0, 1


class NetConfig(C.Structure):
    _fields_ = [(k, C.c_int32) for k in ("board_size", "input_channels", "filters", "blocks", "policy_size",
                                          "policy_head_ch", "value_head_ch", "value_hidden", "max_batch", "device",
                                          "policy_kind", "tower_dtype")]


def widening_seed(seed, runs_before):
    """The 64-bit value that, with a node's id and a move, ranks the moves of a node under progressive widening
    during the (runs_before + 1)-th ob200_search_run of a handle created with `seed`."""
    m = (1 << 64) - 1
    z = (seed + 0x632BE59BD9B4E019 * (runs_before + 1)) & m
    z ^= z >> 31
    z = (z * 0xD6E8FEB86659FD93) & m
    z ^= z >> 32
    return z


class SearchConfig(C.Structure):
    _fields_ = [("n_trees", C.c_int32), ("sims_per_move", C.c_int32), ("leaf_batch", C.c_int32), ("max_depth", C.c_int32),
                ("c_puct", C.c_float), ("virtual_loss", C.c_int32), ("dirichlet_alpha", C.c_float),
                ("dirichlet_epsilon", C.c_float), ("value_sign", C.c_int32), ("use_transposition_table", C.c_int32),
                ("seed", C.c_uint64), ("max_children", C.c_int32), ("use_progressive_widening", C.c_int32),
                ("progressive_widening_c", C.c_float), ("progressive_widening_k", C.c_float), ("rules", C.c_int32)]


class SearchStats(C.Structure):
    _fields_ = [("simulations", C.c_int64), ("evaluations", C.c_int64), ("nodes", C.c_int64),
                ("terminal_leaves", C.c_int64), ("device_ms", C.c_double), ("wall_ms", C.c_double)]


class PolicyRows(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("legal_bits", C.c_void_p), ("row_weight", C.c_void_p), ("grad", C.c_void_p),
                ("loss", C.c_void_p), ("stats", C.c_void_p), ("logits_pitch", C.c_int64), ("grad_pitch", C.c_int64),
                ("n", C.c_int32), ("n_actions", C.c_int32), ("mask_words", C.c_int32), ("dtype", C.c_int32)]


class TrainTensor(C.Structure):
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("exp_avg", C.c_void_p), ("exp_avg_sq", C.c_void_p),
                ("exp_avg_scale", C.c_void_p), ("exp_avg_sq_scale", C.c_void_p), ("numel", C.c_int64), ("weight_decay", C.c_float)]


class AdamWConfig(C.Structure):
    _fields_ = [("lr", C.c_double), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double), ("step", C.c_int32),
                ("param_dtype", C.c_int32), ("grad_dtype", C.c_int32), ("state_bits", C.c_int32), ("grad_scale", C.c_void_p),
                ("lr_device", C.c_void_p), ("step_device", C.c_void_p)]


class Counters(C.Structure):
    _fields_ = [(k, C.c_uint64) for k in ("evals", "batches", "selections", "backups", "kernel_launches")]


# name -> (restype, argtypes); every symbol the header declares
SIGNATURES = {
    "ob200_last_error": (C.c_char_p, []),
    "ob200_version": (C.c_int, []),
    "ob200_device_count": (C.c_int, []),
    "ob200_tree_pitch": (C.c_int32, [C.c_int32]),
    "ob200_tree_mask_words": (C.c_int32, [C.c_int32]),
    "ob200_launch_puct_select": (C.c_int, [C.POINTER(TreeView), C.c_void_p, C.c_int32, C.c_float, C.c_int32, C.c_int32,
                                           C.c_void_p, C.c_void_p]),
    "ob200_launch_vl_apply": (C.c_int, [C.POINTER(TreeView), C.c_void_p, C.c_void_p, C.c_int32, C.c_int32, C.c_void_p]),
    "ob200_launch_vl_revert": (C.c_int, [C.POINTER(TreeView), C.c_void_p, C.c_void_p, C.c_int32, C.c_int32, C.c_void_p]),
    "ob200_launch_backup": (C.c_int, [C.POINTER(TreeView), C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_int32,
                                      C.c_int32, C.c_void_p]),
    "ob200_launch_set_priors": (C.c_int, [C.POINTER(TreeView), C.c_void_p, C.c_int32, C.c_void_p, C.c_int32, C.c_void_p,
                                          C.c_void_p]),
    "ob200_launch_traverse": (C.c_int, [C.POINTER(TreeView), C.c_void_p, C.c_int32, C.c_int32, C.c_float, C.c_int32,
                                        C.c_int32, C.c_void_p, C.c_void_p, C.c_void_p]),
    "ob200_tree_create": (C.c_int, [C.c_int32, C.c_int32, C.c_int32, C.POINTER(C.c_void_p)]),
    "ob200_tree_destroy": (None, [C.c_void_p]),
    "ob200_tree_view_of": (C.c_int, [C.c_void_p, C.POINTER(TreeView)]),
    "ob200_tree_node_count": (C.c_int32, [C.c_void_p]),
    "ob200_tree_clear": (C.c_int, [C.c_void_p]),
    "ob200_tree_add_nodes": (C.c_int, [C.c_void_p, C.c_int32, C.c_void_p, C.c_int32, C.POINTER(C.c_int32)]),
    "ob200_tree_link": (C.c_int, [C.c_void_p, C.c_int32, C.c_void_p, C.c_void_p, C.c_void_p]),
    "ob200_tree_select": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_float, C.c_int32, C.c_int32, C.c_void_p]),
    "ob200_tree_virtual_loss": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_int32]),
    "ob200_tree_backup": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_int32, C.c_int32]),
    "ob200_tree_set_priors": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_void_p, C.c_int32]),
    "ob200_tree_read": (C.c_int, [C.c_void_p, C.c_int32, C.c_int32, C.c_int32, C.c_void_p]),
    "ob200_tree_write": (C.c_int, [C.c_void_p, C.c_int32, C.c_int32, C.c_int32, C.c_void_p]),
    "ob200_board_tensor_positions": (C.c_int64, [C.c_int32, C.c_int32]),
    "ob200_board_tensor_bytes": (C.c_int64, [C.c_int32, C.c_int32, C.c_int32]),
    "ob200_launch_encode_gomoku": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_int32, C.c_int32,
                                             C.c_int32, C.c_void_p, C.c_void_p]),
    "ob200_launch_encode_gomoku_dt": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_int32, C.c_int32,
                                                C.c_int32, C.c_int32, C.c_void_p, C.c_void_p]),
    "ob200_launch_encode_go": (C.c_int, [C.c_void_p] * 4 + [C.c_int32] * 3 + [C.c_void_p, C.c_void_p]),
    "ob200_launch_encode_gomoku3": (C.c_int, [C.c_void_p, C.c_void_p] + [C.c_int32] * 3 + [C.c_void_p, C.c_void_p]),
    "ob200_launch_gomoku_attack_defense": (C.c_int, [C.c_void_p, C.c_void_p] + [C.c_int32] * 3 + [C.c_void_p] * 3),
    "ob200_launch_encode_chess": (C.c_int, [C.c_void_p] * 3 + [C.c_int32] * 2 + [C.c_void_p, C.c_void_p]),
    "ob200_launch_planes_to_board_tensor": (C.c_int, [C.c_void_p, C.c_int32, C.c_int32, C.c_int32, C.c_int32, C.c_void_p,
                                                      C.c_void_p]),
    "ob200_launch_planes_to_board_tensor_dt": (C.c_int, [C.c_void_p, C.c_int32, C.c_int32, C.c_int32, C.c_int32, C.c_int32,
                                                         C.c_void_p, C.c_void_p]),
    "ob200_launch_conv3x3_dt": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_int32,
                                          C.c_int32, C.c_int32, C.c_int32, C.c_int32, C.c_void_p]),
    "ob200_pack_conv3x3_weights_dt": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_int32, C.c_int32, C.c_int32,
                                                C.c_void_p]),
    "ob200_launch_conv3x3": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_int32,
                                       C.c_int32, C.c_int32, C.c_int32, C.c_void_p]),
    "ob200_packed_conv3x3_bytes": (C.c_int64, [C.c_int32, C.c_int32]),
    "ob200_pack_conv3x3_weights": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_int32, C.c_int32, C.c_void_p]),
    "ob200_net_create": (C.c_int, [C.POINTER(NetConfig), C.POINTER(C.c_void_p)]),
    "ob200_net_destroy": (None, [C.c_void_p]),
    "ob200_net_set_tensor": (C.c_int, [C.c_void_p, C.c_char_p, C.c_void_p, C.c_int64]),
    "ob200_net_finalize": (C.c_int, [C.c_void_p]),
    "ob200_net_infer_planes": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_int32, C.c_void_p, C.c_void_p, C.c_int32]),
    "ob200_net_infer_gomoku": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_void_p,
                                         C.c_void_p, C.c_int32]),
    "ob200_net_submit_gomoku": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_void_p,
                                          C.c_void_p, C.c_int32, C.POINTER(C.c_int32)]),
    "ob200_net_wait": (C.c_int, [C.c_void_p, C.c_int32]),
    "ob200_net_forward_device": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_void_p, C.c_void_p, C.c_int32,
                                           C.c_void_p]),
    "ob200_net_forward_gomoku_device": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_void_p,
                                                  C.c_void_p, C.c_int32, C.c_void_p]),
    "ob200_debug_bounded_wait": (C.c_int, [C.c_int32, C.c_void_p]),
    "ob200_net_debug_tower_output": (C.c_void_p, [C.c_void_p]),
    "ob200_net_debug_tower_path": (C.c_int32, [C.c_void_p]),
    "ob200_net_tower_device": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_void_p]),
    "ob200_net_tower_copy_device": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_void_p, C.c_void_p]),
    "ob200_net_input_tensor_channels": (C.c_int32, [C.c_void_p]),
    "ob200_net_value_head_noalloc": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_void_p, C.c_void_p]),
    "ob200_value_head_noalloc_capacity": (C.c_int64, []),
    "ob200_device_error_code": (C.c_int, [C.POINTER(C.c_int32)]),
    "ob200_device_error_peek": (C.c_int, [C.POINTER(C.c_int32)]),
    "ob200_search_create": (C.c_int, [C.c_void_p, C.POINTER(SearchConfig), C.POINTER(C.c_void_p)]),
    "ob200_search_destroy": (None, [C.c_void_p]),
    "ob200_search_run": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_float, C.c_void_p, C.c_void_p,
                                   C.POINTER(SearchStats)]),
    "ob200_search_debug_tree": (C.c_int, [C.c_void_p, C.POINTER(TreeView), C.POINTER(C.c_int32)]),
    "ob200_search_debug_hooks": (C.c_int, [C.c_void_p, C.c_float, C.c_int32]),
    "ob200_search_debug_phases": (C.c_int, [C.c_void_p, C.c_int32, C.c_void_p]),
    "ob200_search_debug_record": (C.c_int, [C.c_void_p, C.POINTER(C.c_void_p), C.POINTER(C.c_void_p), C.POINTER(C.c_void_p)]),
    "ob200_copy_to_host": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int64]),
    "ob200_launch_policy_loss_search": (C.c_int, [C.POINTER(PolicyRows), C.c_void_p, C.c_int64, C.c_int32, C.c_float, C.c_void_p]),
    "ob200_launch_policy_loss_clipped": (C.c_int, [C.POINTER(PolicyRows), C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                                   C.c_int64, C.c_float, C.c_float, C.c_float, C.c_float, C.c_void_p]),
    "ob200_debug_policy_waits": (None, [C.c_int32]),
    "ob200_grad_norm_workspace_bytes": (C.c_int64, []),
    "ob200_launch_grad_norm": (C.c_int, [C.POINTER(TrainTensor), C.c_int32, C.c_int32, C.c_float, C.c_void_p, C.c_void_p,
                                         C.c_void_p]),
    "ob200_launch_adamw": (C.c_int, [C.POINTER(TrainTensor), C.c_int32, C.POINTER(AdamWConfig), C.c_void_p]),
    "ob200_get_counters": (C.c_int, [C.POINTER(Counters)]),
    "ob200_reset_counters": (None, []),
}

_lib = None


def lib():
    """The loaded library.  Raises when it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise Error(-1, f"{LIB_PATH} is missing: run `python -m omoknuni_small_b200.build` (there is no fallback)")
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _lib = L
    return _lib


def check(rc):
    if rc != 0:
        raise Error(rc, lib().ob200_last_error().decode())


def counters():
    c = Counters()
    check(lib().ob200_get_counters(C.byref(c)))
    return {k: getattr(c, k) for k, _ in Counters._fields_}


def device_error_code(clear=True):
    v = C.c_int32(0)
    check((lib().ob200_device_error_code if clear else lib().ob200_device_error_peek)(C.byref(v)))
    return v.value


def _ptr(t):
    """Device pointer of a torch tensor (or None)."""
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


class DeviceTree:
    """Edge statistics on the device (torch tensors own the memory) + the view
    struct the launchers take.  `tree` is a dict as synth.make_selection_tree
    returns; an optional 'child_node' [n_nodes, pitch] int32 enables descent."""

    def __init__(self, tree, device="cuda:0"):
        import torch
        self.torch = torch
        self.n_nodes, self.pitch = tree["N"].shape
        self.n_children = int(tree["n_children"])
        self.t = {k: torch.from_numpy(np.ascontiguousarray(tree[k])).to(device)
                  for k in ("N", "W", "P", "VL", "node_visits") if k in tree}
        self.t["legal_bits"] = torch.from_numpy(np.ascontiguousarray(tree["legal_bits"]).view(np.int32)).to(device)
        if tree.get("child_node") is not None:
            self.t["child_node"] = torch.from_numpy(np.ascontiguousarray(tree["child_node"])).to(device)
        self.mask_words = tree["legal_bits"].shape[1]
        self.device = device
        self.view = TreeView(self.t["N"].data_ptr(), self.t["W"].data_ptr(), self.t["P"].data_ptr(),
                             self.t["VL"].data_ptr(), self.t["legal_bits"].data_ptr(),
                             self.t["node_visits"].data_ptr(),
                             self.t["child_node"].data_ptr() if "child_node" in self.t else None,
                             self.n_nodes, self.n_children, self.pitch, self.mask_words)

    def host(self, key):
        return self.t[key].cpu().numpy()

    def select(self, node_ids=None, c_puct=1.5, vl_value=3, apply_vl=True, out=None):
        torch = self.torch
        n = self.n_nodes if node_ids is None else node_ids.numel()
        if out is None:
            out = torch.empty(n, dtype=torch.int32, device=self.device)
        check(lib().ob200_launch_puct_select(C.byref(self.view), _ptr(node_ids), n, c_puct, vl_value, int(apply_vl),
                                             _ptr(out), _stream()))
        return out

    def vl_apply(self, sel, vl_value=3, node_ids=None):
        check(lib().ob200_launch_vl_apply(C.byref(self.view), _ptr(node_ids), _ptr(sel), sel.numel(), vl_value, _stream()))

    def vl_revert(self, sel, vl_value=3, node_ids=None):
        check(lib().ob200_launch_vl_revert(C.byref(self.view), _ptr(node_ids), _ptr(sel), sel.numel(), vl_value, _stream()))

    def backup(self, paths, path_len, leaf_values, vl_value=3):
        n, max_depth, _ = paths.shape
        check(lib().ob200_launch_backup(C.byref(self.view), _ptr(paths), _ptr(path_len), _ptr(leaf_values), n, max_depth,
                                        vl_value, _stream()))

    def set_priors(self, node_ids, policy, slot_action=None):
        check(lib().ob200_launch_set_priors(C.byref(self.view), _ptr(node_ids), policy.shape[0], _ptr(policy),
                                            policy.shape[1], _ptr(slot_action), _stream()))

    def traverse(self, roots, sims_per_tree, c_puct=1.5, vl_value=3, max_depth=64):
        torch = self.torch
        n = roots.numel() * sims_per_tree
        paths = torch.zeros((n, max_depth, 2), dtype=torch.int32, device=self.device)
        plen = torch.zeros(n, dtype=torch.int32, device=self.device)
        check(lib().ob200_launch_traverse(C.byref(self.view), _ptr(roots), roots.numel(), sims_per_tree, c_puct, vl_value,
                                          max_depth, _ptr(paths), _ptr(plen), _stream()))
        return paths, plen


# ---- board tensors -------------------------------------------------------------
def board_positions(board_size, B):
    return int(lib().ob200_board_tensor_positions(board_size, B))


def board_tensor_to_planes(bt_u16, board_size, B, channels, dtype=DTYPE_BF16):
    """16-bit NHWC board tensor (numpy uint16 view, flat, `channels` rounded up to 8
    per position) -> fp32 planes [B, channels, S, S] plus a flag telling whether
    every padding / guard element is zero.  Host-side helper for tests."""
    S, GP = board_size, board_size + 1
    slots = GP * GP
    PT = board_positions(S, B)
    Cp = (channels + 7) // 8 * 8
    a = np.asarray(bt_u16).reshape(-1)[: PT * Cp].reshape(PT, Cp)
    f = a.view(np.float16).astype(np.float32) if dtype == DTYPE_F16 else (a.astype(np.uint32) << 16).view(np.float32)
    body = f[GUARD:GUARD + B * slots].reshape(B, GP, GP, Cp)
    planes = body[:, :S, :S, :channels].transpose(0, 3, 1, 2)
    pad_zero = (not f[:GUARD].any() and not f[GUARD + B * slots:].any()
                and not body[:, S, :, :].any() and not body[:, :, S, :].any())
    return np.ascontiguousarray(planes), bool(pad_zero)


def planes_to_board_tensor_host(planes, out_channels, dtype=DTYPE_BF16):
    """fp32 planes [B, C, S, S] -> 16-bit NHWC board tensor as a flat numpy uint16
    array (round to nearest even), the host-side twin of the device conversion."""
    B, Cc, S, _ = planes.shape
    GP = S + 1
    PT = board_positions(S, B)
    full = np.zeros((B, GP, GP, out_channels), np.float32)
    full[:, :S, :S, :Cc] = planes.transpose(0, 2, 3, 1)
    u = full.view(np.uint32)
    r = full.astype(np.float16).view(np.uint16) if dtype == DTYPE_F16 else ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    out = np.zeros((PT, out_channels), np.uint16)
    out[GUARD:GUARD + B * GP * GP] = r.reshape(B * GP * GP, out_channels)
    return out.reshape(-1)


def encode_gomoku(history, n_hist, to_move, board_size=15, planes=19, out_channels=64, dtype=DTYPE_BF16, out=None):
    """Device tensors in (int16 [B,16], uint8 [B], uint8 [B]) -> board tensor
    (torch int16 tensor holding the bf16 / fp16 bits; `out`: a tensor of that size to write into)."""
    import torch
    B = history.shape[0]
    nbytes = int(lib().ob200_board_tensor_bytes(board_size, B, out_channels))
    if out is None:
        out = torch.empty(nbytes // 2, dtype=torch.int16, device=history.device)
    assert out.numel() * out.element_size() == nbytes
    check(lib().ob200_launch_encode_gomoku_dt(_ptr(history), _ptr(n_hist), _ptr(to_move), B, board_size, planes,
                                              out_channels, dtype, _ptr(out), _stream()))
    return out


def encode_go(stones, ko_point, to_move, legal_bits, board_size, out_channels=64):
    """Device tensors in (int8 [B,S*S], int32 [B], uint8 [B], int32 [B,ceil(S*S/32)] bit masks)
    -> bf16 board tensor (int16 view) with the reference's 10 Go planes."""
    import torch
    B = stones.shape[0]
    nbytes = int(lib().ob200_board_tensor_bytes(board_size, B, out_channels))
    out = torch.empty(nbytes // 2, dtype=torch.int16, device=stones.device)
    check(lib().ob200_launch_encode_go(_ptr(stones), _ptr(ko_point), _ptr(to_move), _ptr(legal_bits), B, board_size,
                                       out_channels, _ptr(out), _stream()))
    return out


def encode_gomoku3(stones, to_move, board_size, out_channels=64):
    """Device tensors in (int8 [B,S*S], uint8 [B]) -> bf16 board tensor with the 3-plane representation."""
    import torch
    B = stones.shape[0]
    nbytes = int(lib().ob200_board_tensor_bytes(board_size, B, out_channels))
    out = torch.empty(nbytes // 2, dtype=torch.int16, device=stones.device)
    check(lib().ob200_launch_encode_gomoku3(_ptr(stones), _ptr(to_move), B, board_size, out_channels, _ptr(out), _stream()))
    return out


def gomoku_attack_defense(stones, to_move, board_size, stone_placed=False):
    """Device tensors in (int8 [B,S*S], uint8 [B]) -> (attack, defense) fp32 [B,S*S] each."""
    import torch
    B = stones.shape[0]
    att = torch.empty((B, board_size * board_size), dtype=torch.float32, device=stones.device)
    dfn = torch.empty_like(att)
    check(lib().ob200_launch_gomoku_attack_defense(_ptr(stones), _ptr(to_move), B, board_size, int(stone_placed), _ptr(att),
                                                   _ptr(dfn), _stream()))
    return att, dfn


def encode_chess(pieces, meta, legal_to, out_channels=64):
    """Device tensors in (int8 [B,64], int32 [B,6], int32 [B,2] bit masks) -> bf16 board tensor
    (int16 view, board_size 8) with the reference's 20 chess planes."""
    import torch
    B = pieces.shape[0]
    nbytes = int(lib().ob200_board_tensor_bytes(8, B, out_channels))
    out = torch.empty(nbytes // 2, dtype=torch.int16, device=pieces.device)
    check(lib().ob200_launch_encode_chess(_ptr(pieces), _ptr(meta), _ptr(legal_to), B, out_channels, _ptr(out), _stream()))
    return out


def planes_to_board_tensor(planes, out_channels, dtype=DTYPE_BF16):
    import torch
    B, Cc, S, _ = planes.shape
    nbytes = int(lib().ob200_board_tensor_bytes(S, B, out_channels))
    out = torch.empty(nbytes // 2, dtype=torch.int16, device=planes.device)
    check(lib().ob200_launch_planes_to_board_tensor_dt(_ptr(planes), B, Cc, S, out_channels, dtype, _ptr(out), _stream()))
    return out


def pack_conv3x3(w_oihw, scale, cin=64, dtype=DTYPE_BF16):
    """fp32 [cout, cin_real, 3, 3] (+ per-output-channel scale or None) -> packed
    bf16 / fp16 image as numpy uint16."""
    w = np.ascontiguousarray(w_oihw, np.float32)
    cout, cin_real = w.shape[:2]
    out = np.empty(int(lib().ob200_packed_conv3x3_bytes(cin, cout)) // 2, np.uint16)
    sc = None if scale is None else np.ascontiguousarray(scale, np.float32)
    check(lib().ob200_pack_conv3x3_weights_dt(w.ctypes.data_as(C.c_void_p), None if sc is None else sc.ctypes.data_as(C.c_void_p),
                                              cout, cin_real, cin, dtype, out.ctypes.data_as(C.c_void_p)))
    return out


def conv3x3(x_bt, packed_w, bias, residual_bt, B, board_size, cin=64, cout=64, relu=True, out=None, dtype=DTYPE_BF16):
    """One conv layer on device board tensors (torch int16 tensors with bf16 / fp16 bits)."""
    import torch
    if out is None:
        nbytes = int(lib().ob200_board_tensor_bytes(board_size, B, cout))
        out = torch.zeros(nbytes // 2, dtype=torch.int16, device=x_bt.device)
    check(lib().ob200_launch_conv3x3_dt(_ptr(x_bt), _ptr(packed_w), _ptr(bias), _ptr(residual_bt), _ptr(out), B, board_size,
                                        cin, cout, int(relu), dtype, _stream()))
    return out


# ---- network handle ------------------------------------------------------------
class Net:
    """The residual policy/value network on one GPU (host-side mirror of the
    reference's ResNetModel: constructor arguments in the same order, weights
    under the same names, inference on host buffers)."""

    def __init__(self, input_channels, board_size, blocks, filters, policy_size, policy_head_ch=32, value_head_ch=32,
                 value_hidden=256, max_batch=1024, device=0, policy_kind=POLICY_FC, tower_dtype=DTYPE_BF16):
        self.cfg = NetConfig(board_size, input_channels, filters, blocks, policy_size or board_size * board_size,
                             policy_head_ch, value_head_ch, value_hidden, max_batch, device, policy_kind, tower_dtype)
        self.tower_dtype = tower_dtype
        self.h = C.c_void_p()
        check(lib().ob200_net_create(C.byref(self.cfg), C.byref(self.h)))
        self.policy_size = self.cfg.policy_size
        self.board_size = board_size

    def load(self, weights):
        """weights: dict name -> numpy array under the reference's parameter names."""
        for name, arr in weights.items():
            a = np.ascontiguousarray(arr, np.float32)
            check(lib().ob200_net_set_tensor(self.h, name.encode(), a.ctypes.data_as(C.c_void_p), a.size))
        check(lib().ob200_net_finalize(self.h))
        return self

    def infer_planes(self, planes, out_kind=OUT_PROBS):
        x = np.ascontiguousarray(planes, np.float32)
        B, Cc = x.shape[:2]
        pol = np.empty((B, self.policy_size), np.float32)
        val = np.empty(B, np.float32)
        check(lib().ob200_net_infer_planes(self.h, x.ctypes.data_as(C.c_void_p), B, Cc, pol.ctypes.data_as(C.c_void_p),
                                           val.ctypes.data_as(C.c_void_p), out_kind))
        return pol, val

    def infer_gomoku(self, history, n_hist, to_move, out_kind=OUT_PROBS, out=None):
        """out: optional (policy [B, A] float32, value [B] float32) numpy arrays to fill; arrays in
        page-locked memory are written by the copy engine directly (small results go through the handle's own)."""
        h = np.ascontiguousarray(history, np.int16)
        nh = np.ascontiguousarray(n_hist, np.uint8)
        tm = np.ascontiguousarray(to_move, np.uint8)
        B = h.shape[0]
        if out is not None:
            pol, val = out
            assert pol.dtype == np.float32 and val.dtype == np.float32 and pol.flags.c_contiguous and val.flags.c_contiguous
            assert pol.shape == (B, self.policy_size) and val.shape == (B,)
        else:
            pol = np.empty((B, self.policy_size), np.float32)
            val = np.empty(B, np.float32)
        check(lib().ob200_net_infer_gomoku(self.h, h.ctypes.data_as(C.c_void_p), nh.ctypes.data_as(C.c_void_p),
                                           tm.ctypes.data_as(C.c_void_p), B, pol.ctypes.data_as(C.c_void_p),
                                           val.ctypes.data_as(C.c_void_p), out_kind))
        return pol, val

    def submit_gomoku(self, history, n_hist, to_move, out, out_kind=OUT_PROBS):
        """Asynchronous infer_gomoku: enqueues the call and returns a ticket for wait().  The arrays (C-contiguous
        int16 / uint8 / uint8 inputs, float32 outputs in `out`) must stay alive and untouched until then; at most two
        calls may be pending."""
        pol, val = out
        B = history.shape[0]
        assert history.dtype == np.int16 and n_hist.dtype == np.uint8 and to_move.dtype == np.uint8
        assert pol.dtype == np.float32 and val.dtype == np.float32 and pol.shape == (B, self.policy_size) and val.shape == (B,)
        ticket = C.c_int32(-1)
        check(lib().ob200_net_submit_gomoku(self.h, history.ctypes.data_as(C.c_void_p), n_hist.ctypes.data_as(C.c_void_p),
                                            to_move.ctypes.data_as(C.c_void_p), B, pol.ctypes.data_as(C.c_void_p),
                                            val.ctypes.data_as(C.c_void_p), out_kind, C.byref(ticket)))
        return ticket.value

    def wait(self, ticket):
        check(lib().ob200_net_wait(self.h, ticket))

    def input_tensor_channels(self):
        return int(lib().ob200_net_input_tensor_channels(self.h))

    def forward_device(self, input_bt, B, policy_out, value_out, out_kind=OUT_PROBS):
        check(lib().ob200_net_forward_device(self.h, _ptr(input_bt), B, _ptr(policy_out), _ptr(value_out), out_kind,
                                             _stream()))

    def forward_gomoku_device(self, history, n_hist, to_move, policy_out, value_out, out_kind=OUT_PROBS):
        """encode -> tower -> heads on device move histories (torch tensors: int16 [B,16], uint8 [B], uint8 [B])."""
        check(lib().ob200_net_forward_gomoku_device(self.h, _ptr(history), _ptr(n_hist), _ptr(to_move), history.shape[0],
                                                    _ptr(policy_out), _ptr(value_out), out_kind, _stream()))

    def tower_device(self, input_bt, B):
        """The residual tower alone on a device input tensor (asynchronous)."""
        check(lib().ob200_net_tower_device(self.h, _ptr(input_bt), B, _stream()))

    def tower_copy_device(self, input_bt, B, out=None):
        """The same into memory of the caller's, ordered with the handle's own calls and searches whatever the current stream
        is.  Returns the board tensor (int16 holding the 16-bit values; `out`: a tensor of that size to write into)."""
        import torch
        nbytes = int(lib().ob200_board_tensor_bytes(self.board_size, B, self.cfg.filters))
        if out is None:
            out = torch.empty(nbytes // 2, dtype=torch.int16, device=torch.device("cuda", self.cfg.device))
        assert out.is_contiguous() and out.numel() * out.element_size() == nbytes
        check(lib().ob200_net_tower_copy_device(self.h, _ptr(input_bt), B, _ptr(out), _stream()))
        return out

    def tower_output_ptr(self):
        return lib().ob200_net_debug_tower_output(self.h)

    def tower_path(self):
        """0 launch per layer, 1 one cooperative launch, 2 boards resident in shared memory (last forward)."""
        return int(lib().ob200_net_debug_tower_path(self.h))

    def value_head_noalloc(self, tower_ptr, B, value_out):
        """Value head from a tower output already on the device, using only the
        library's built-in scratch array (no allocation anywhere)."""
        check(lib().ob200_net_value_head_noalloc(self.h, C.c_void_p(tower_ptr), B, _ptr(value_out), _stream()))

    def close(self):
        if self.h:
            lib().ob200_net_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- leaf-parallel search ---------------------------------------------------------
class Search:
    """Leaf-parallel MCTS over a group of Gomoku games on one GPU (host-side mirror of
    MCTSEngine::search for many games at once)."""

    def __init__(self, net, n_trees=64, sims_per_move=800, leaf_batch=1024, max_depth=64, c_puct=1.5, virtual_loss=3,
                 dirichlet_alpha=0.3, dirichlet_epsilon=0.25, value_sign=1, transposition_table=False, seed=0,
                 max_children=0, progressive_widening=None, rules=0):
        """progressive_widening: None (off, as the reference's shipped configuration) or (c, k) of MCTSSettings.
        rules: RULES_FREESTYLE or RULES_OMOK."""
        self.net = net                       # keep the network alive
        pw = progressive_widening
        self.cfg = SearchConfig(n_trees, sims_per_move, leaf_batch, max_depth, c_puct, virtual_loss, dirichlet_alpha,
                                dirichlet_epsilon, value_sign, int(transposition_table), seed, max_children,
                                int(pw is not None), pw[0] if pw else 0.0, pw[1] if pw else 0.0, rules)
        self.h = C.c_void_p()
        check(lib().ob200_search_create(net.h, C.byref(self.cfg), C.byref(self.h)))

    def run(self, move_lists, temperature=1.0):
        """move_lists: one sequence of actions per tree.  Returns (pi [T,225], visits [T,225], stats dict)."""
        T = self.cfg.n_trees
        assert len(move_lists) == T
        stride = max(1, max(len(m) for m in move_lists))
        moves = np.full((T, stride), -1, np.int16)
        n = np.zeros(T, np.int32)
        for t, m in enumerate(move_lists):
            moves[t, :len(m)] = m
            n[t] = len(m)
        pi = np.zeros((T, 225), np.float32)
        visits = np.zeros((T, 225), np.int32)
        st = SearchStats()
        check(lib().ob200_search_run(self.h, moves.ctypes.data_as(C.c_void_p), n.ctypes.data_as(C.c_void_p), stride,
                                     temperature, pi.ctypes.data_as(C.c_void_p), visits.ctypes.data_as(C.c_void_p),
                                     C.byref(st)))
        return pi, visits, {k: getattr(st, k) for k, _ in SearchStats._fields_}

    def debug_hooks(self, value_quantum=0.0, record_rounds=0):
        """Test hooks: round network values to multiples of 1 / value_quantum; keep the network outputs of the
        root evaluation and of the first `record_rounds` rounds of each run."""
        check(lib().ob200_search_debug_hooks(self.h, value_quantum, record_rounds))
        self._rec_rounds = record_rounds

    def phase_timing(self, enable=True):
        """Switches per-phase event timing of the following runs on or off; returns the sums (ms) of the last timed run
        as a dict: descent, leaf_positions, network, expansion, backup."""
        out = (C.c_double * 5)()
        check(lib().ob200_search_debug_phases(self.h, int(enable), out))
        return dict(zip(("descent", "leaf_positions", "network", "expansion", "backup"), [float(v) for v in out]))

    def record(self):
        """(policy [R + 1, L, 225], value [R + 1, L], noise [T, 228]) of the last run, as numpy arrays."""
        pp, vp, nz = C.c_void_p(), C.c_void_p(), C.c_void_p()
        check(lib().ob200_search_debug_record(self.h, C.byref(pp), C.byref(vp), C.byref(nz)))
        R, L, T = self._rec_rounds, self.cfg.leaf_batch, self.cfg.n_trees

        def pull(ptr, shape):
            a = np.empty(shape, np.float32)
            check(lib().ob200_copy_to_host(a.ctypes.data_as(C.c_void_p), ptr, a.nbytes))
            return a
        return pull(pp, (R + 1, L, 225)), pull(vp, (R + 1, L)), pull(nz, (T, 228))

    def tree(self):
        """Host copies of the search's tree arrays (for tests): dict of numpy arrays + nodes used."""
        v = TreeView()
        used = C.c_int32(0)
        check(lib().ob200_search_debug_tree(self.h, C.byref(v), C.byref(used)))
        n, pitch, mw = used.value, v.pitch, v.mask_words

        def pull(ptr, count, dtype):
            a = np.empty(count, dtype)
            check(lib().ob200_copy_to_host(a.ctypes.data_as(C.c_void_p), C.c_void_p(ptr), a.nbytes))
            return a
        return {"N": pull(v.N, n * pitch, np.int32).reshape(n, pitch), "W": pull(v.W, n * pitch, np.float32).reshape(n, pitch),
                "P": pull(v.P, n * pitch, np.float32).reshape(n, pitch), "VL": pull(v.VL, n * pitch, np.int32).reshape(n, pitch),
                "child_node": pull(v.child_node, n * pitch, np.int32).reshape(n, pitch),
                "legal_bits": pull(v.legal_bits, n * mw, np.uint32).reshape(n, mw),
                "node_visits": pull(v.node_visits, n, np.int32), "n_children": v.n_children, "nodes": n}

    def close(self):
        if self.h:
            lib().ob200_search_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- training operators ---------------------------------------------------------------
def _refuse(text, *args):
    raise Error(ERR_INVALID, text % args if args else text)


def _require(ok, text, *args):
    if not ok:
        _refuse(text, *args)


_TRAIN_TYPES = {}


def _train_dtype(dtype, what):
    if not _TRAIN_TYPES:
        import torch
        _TRAIN_TYPES.update({torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16})
    kind = _TRAIN_TYPES.get(dtype)
    if kind is None:
        _refuse("%s: float32, bfloat16 or float16 is wanted, got %s", what, dtype)
    return kind


def _launch_on(device, fn, *args):
    """fn(*args, stream) with the tensors' device as the current one, on its current stream, which is returned."""
    import torch
    if device.type != "cuda":
        _refuse("the tensors are not on a CUDA device (there is no CPU path)")
    raw, index = torch._C._cuda_getCurrentRawStream, device.index      # what torch.cuda.current_stream() wraps, a tenth of its time
    stream = raw(index)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc != 0:
        check(rc)
    return stream


def _pitch(t, what, n, A, device, dtype):
    """Pitch of a matrix of n rows of A adjacent elements of dtype."""
    if t.dtype != dtype or t.device != device or t.shape != (n, A):
        _refuse("%s: a matrix (%d, %d) of %s on the logits' device is wanted, got %s of %s on %s", what, n, A, dtype, tuple(t.shape), t.dtype, t.device)
    step, one = t.stride()
    if one != 1 and A != 1:
        _refuse("%s: the elements of a row have to be adjacent", what)
    return step if n > 1 else max(step, A)


def _vector(t, what, n, device, dtype):
    if t is None:
        return None
    if t.dtype != dtype or t.device != device or t.shape != (n,) or not t.is_contiguous():
        _refuse("%s: %d adjacent values of %s on the logits' device are wanted", what, n, dtype)
    return t.data_ptr()


def _policy_rows(torch, logits, legal_bits, row_weight, out):
    """The struct of both losses, and (loss, grad, stats)."""
    if logits.dim() != 2 or not logits.shape[1]:
        _refuse("logits: a matrix of rows is wanted, got shape %s", tuple(logits.shape))
    n, A = logits.shape
    f32, dtype, dev = torch.float32, logits.dtype, logits.device
    kind = _train_dtype(dtype, "logits")
    if out is None:
        out = (torch.empty(n, dtype=f32, device=dev), torch.empty((n, A), dtype=dtype, device=dev), torch.empty((n, 4), dtype=f32, device=dev))
    loss, grad, stats = out
    bits, words = None, 0
    if legal_bits is not None:
        if legal_bits.dim() != 2 or legal_bits.shape[0] != n or legal_bits.dtype != torch.int32 or legal_bits.device != dev or not legal_bits.is_contiguous():
            _refuse("legal_bits: a contiguous int32 matrix [%d, words] on the logits' device is wanted", n)
        bits, words = legal_bits.data_ptr(), legal_bits.shape[1]
    if stats is not None and (stats.dtype != f32 or stats.device != dev or stats.shape != (n, 4) or not stats.is_contiguous()):
        _refuse("stats: a contiguous float32 matrix [%d, 4] on the logits' device is wanted", n)
    return PolicyRows(logits.data_ptr(), bits, _vector(row_weight, "row_weight", n, dev, f32), grad.data_ptr(), _vector(loss, "loss", n, dev, f32),
                      None if stats is None else stats.data_ptr(), _pitch(logits, "logits", n, A, dev, dtype), _pitch(grad, "grad", n, A, dev, dtype),
                      n, A, words, kind), out


def policy_loss_search(logits, target, legal_bits=None, row_weight=None, entropy_coef=0.0, out=None):
    """Cross entropy of the policy with the search's visit distribution, row by row, and its gradient
    (ob200_launch_policy_loss_search).  logits [n, A] float32 / bfloat16 / float16, target [n, A] int32 visit counts or
    float32, legal_bits [n, words] int32 bit masks as DeviceTree holds them, row_weight [n] float32: the factor of each
    row's loss, 0 for rows that only fill up a batch.  Returns (loss [n] float32, grad [n, A] of the logits' type,
    stats [n, 4] float32: cross entropy, entropy, sum of the target, log-sum-exp); `out`: the three to write into (loss and
    stats may be None, grad may be the logits).  With logits from autograd: torch.autograd.backward(logits, grad)."""
    import torch
    rows, out = _policy_rows(torch, logits, legal_bits, row_weight, out)
    visits = target.dtype == torch.int32
    pitch = _pitch(target, "target", rows.n, rows.n_actions, logits.device, torch.int32 if visits else torch.float32)
    _launch_on(logits.device, lib().ob200_launch_policy_loss_search, rows, target.data_ptr(), pitch,
               TARGET_VISITS if visits else TARGET_PROBS, entropy_coef)
    return out


def policy_loss_clipped(logits, action, old_logp, advantage, legal_bits=None, ref_logits=None, row_weight=None, clip_low=0.2,
                        clip_high=0.2, kl_coef=0.0, entropy_coef=0.0, out=None):
    """Clipped-ratio policy loss with a KL term against a reference policy, row by row, and its gradient
    (ob200_launch_policy_loss_clipped).  action [n] int32, old_logp and advantage [n] float32, ref_logits [n, A] of the
    logits' type or None; the rest as policy_loss_search.  stats: log-probability of the action, ratio, KL, entropy."""
    import torch
    rows, out = _policy_rows(torch, logits, legal_bits, row_weight, out)
    dev, n, ref, ref_pitch = logits.device, rows.n, None, 0
    if ref_logits is not None:
        ref, ref_pitch = ref_logits.data_ptr(), _pitch(ref_logits, "ref_logits", n, rows.n_actions, dev, logits.dtype)
    act, old, adv = (_vector(action, "action", n, dev, torch.int32), _vector(old_logp, "old_logp", n, dev, torch.float32),
                     _vector(advantage, "advantage", n, dev, torch.float32))
    _launch_on(dev, lib().ob200_launch_policy_loss_clipped, rows, act, old, adv, ref, ref_pitch, clip_low, clip_high, kl_coef, entropy_coef)
    return out


def _same_kind(tensors, what):
    """The OB200_DTYPE_* and device that all tensors of a list share; each has to be contiguous."""
    first = tensors[0]
    for i, t in enumerate(tensors):
        _require(t.dtype == first.dtype and t.device == first.device, "%s %d: type or device differs from the first one's", what, i)
        _require(t.is_contiguous(), "%s %d is not contiguous", what, i)
    return _train_dtype(first.dtype, what), first.device


def _cleared(make, device, what):
    """make() - zeroed tensors that a plan keeps - done when this returns, so that the plan may run on any stream."""
    import torch
    with torch.cuda.device(device):
        _require(not torch.cuda.is_current_stream_capturing(), "%s: a plan is made before a graph is captured, not in it", what)
        made = make()
        torch.cuda.current_stream().synchronize()
    return made


class _Plan:
    """What keeps memory of its own for calls on any stream: `_own`, allocated on the stream `_home`."""

    def _keep(self, tensors):
        import torch
        self._own, self._home, self._seen = tensors, torch._C._cuda_getCurrentRawStream(self.device.index), set()

    def _ran_on(self, stream):
        """Tells the allocator of another stream, so that dropping the plan does not hand its memory out while that still runs."""
        if stream == self._home or stream in self._seen:
            return
        import torch
        self._seen.add(stream)
        current = torch.cuda.current_stream(self.device)
        for t in self._own:
            t.record_stream(current)


class GradNorm(_Plan):
    """2-norm over a fixed list of gradients and the factor that clips it (ob200_launch_grad_norm).  run(max_norm) fills
    and returns `out` (float32 [2] on the device: norm, factor); `clip` is the factor as AdamW.step takes it.  The plan
    keeps the gradients and its workspace: one plan per stream that runs at the same time.  It may be dropped while a call
    runs; a graph that captured one needs the plan as long as it is replayed."""

    def __init__(self, grads, out=None):
        import torch
        self.grads = list(grads)
        _require(len(self.grads) > 0, "GradNorm: no gradients")
        self.dtype, self.device = _same_kind(self.grads, "grad")
        _require(self.device.type == "cuda", "the tensors are not on a CUDA device (there is no CPU path)")
        count = int(lib().ob200_grad_norm_workspace_bytes()) // 8
        self.out, self.workspace = _cleared(lambda: (torch.zeros(2, dtype=torch.float32, device=self.device) if out is None else out,
                                                     torch.zeros(count, dtype=torch.float64, device=self.device)), self.device, "GradNorm")
        _require(self.out.dtype == torch.float32 and self.out.device == self.device and tuple(self.out.shape) == (2,)
                 and self.out.is_contiguous(), "GradNorm: out is float32 [2] on the gradients' device")
        self.clip = self.out[1:]
        self._keep([self.workspace] + ([self.out] if out is None else []))
        self.table = (TrainTensor * len(self.grads))()
        for e, g in zip(self.table, self.grads):
            e.grad, e.numel = g.data_ptr(), g.numel()

    def run(self, max_norm=float("inf")):
        self._ran_on(_launch_on(self.device, lib().ob200_launch_grad_norm, self.table, len(self.table), self.dtype, max_norm,
                                self.workspace.data_ptr(), self.out.data_ptr()))
        return self.out


class AdamW(_Plan):
    """AdamW over a fixed list of weights and gradients, one launch a step (ob200_launch_adamw).

    params, grads: contiguous tensors of one float type each on one device; the gradients' buffers are kept, so whatever
    fills them has to write in place.  state_bits: 32, or 8 (e4m3 codes with a float32 scale per 256 elements).
    weight_decay: a number, or one per tensor.  state: {"exp_avg": [...], "exp_avg_sq": [...]} and for 8 bits
    {"exp_avg_scale": [...], "exp_avg_sq_scale": [...]} to go on from, zeros otherwise; it is `self.state`, updated in
    place.  `self.steps` is the count of the last step that was counted on the host.  Steps from several threads are launched one
    after the other."""

    BLOCK = 256

    def __init__(self, params, grads, state_bits=32, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state=None):
        import torch
        self.params, self.grads = list(params), list(grads)
        n = len(self.params)
        _require(n > 0 and len(self.grads) == n, "AdamW: as many gradients as params are wanted, at least one")
        _require(state_bits in (8, 32), "AdamW: state_bits is 8 or 32")
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * n
        _require(len(decay) == n, "AdamW: a weight decay for each param is wanted")
        p_dtype, self.device = _same_kind(self.params, "param")
        g_dtype, g_device = _same_kind(self.grads, "grad")
        _require(self.device.type == "cuda", "the tensors are not on a CUDA device (there is no CPU path)")
        _require(g_device == self.device, "AdamW: params and gradients are on different devices")
        for i, (p, g) in enumerate(zip(self.params, self.grads)):
            _require(p.numel() == g.numel(), "AdamW: param %d has %d elements, its gradient %d", i, p.numel(), g.numel())
        held = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        keys = {"exp_avg": (held, 1), "exp_avg_sq": (held, 1)}
        if state_bits == 8:
            keys.update(exp_avg_scale=(torch.float32, self.BLOCK), exp_avg_sq_scale=(torch.float32, self.BLOCK))

        def size(p, per):
            return (p.numel() + per - 1) // per
        given = state is not None
        if not given:
            state = _cleared(lambda: {k: [torch.zeros(size(p, per), dtype=torch.uint8 if dt == torch.float8_e4m3fn else dt, device=self.device).view(dt)
                                          for p in self.params] for k, (dt, per) in keys.items()}, self.device, "AdamW")
        self.state = {k: list(state[k]) if k in state else None for k in keys}
        for k, (dt, per) in keys.items():
            _require(self.state[k] is not None and len(self.state[k]) == n, "AdamW: state %s: a tensor for each param is wanted", k)
            for i, (t, p) in enumerate(zip(self.state[k], self.params)):
                _require(t.dtype == dt and t.device == self.device and t.is_contiguous() and t.numel() == size(p, per),
                         "AdamW: state %s %d: %d contiguous values of %s are wanted", k, i, size(p, per), dt)
        self.table = (TrainTensor * n)()
        for i, e in enumerate(self.table):
            e.param, e.grad, e.numel, e.weight_decay = self.params[i].data_ptr(), self.grads[i].data_ptr(), self.params[i].numel(), decay[i]
            for k in keys:
                setattr(e, k, self.state[k][i].data_ptr())
        self._lock = threading.Lock()        # cfg and steps are a step's own while it is launched
        self.cfg = AdamWConfig(beta1=betas[0], beta2=betas[1], eps=eps, param_dtype=p_dtype, grad_dtype=g_dtype, state_bits=state_bits)
        self._keep([] if given else [t for ts in self.state.values() for t in ts])
        self.steps = 0

    def _scalar(self, t, what, dtype):
        if t.dtype != dtype or t.device != self.device or t.numel() != 1:
            _refuse("AdamW: %s is one %s on the weights' device", what, dtype)
        return t.data_ptr()

    def step(self, lr, step=None, grad_scale=None):
        """One step.  lr: a number, or a float32 scalar on the device; step: 1 for the first one (default: counted here), or an
        int32 scalar on the device - for captured graphs, nothing is changed while it is below 1; grad_scale: a float32 scalar on the device that multiplies every
        gradient (GradNorm.clip); when it is not finite weights and states stay as they are, while the count goes on."""
        import torch
        with self._lock:
            c = self.cfg
            c.grad_scale = None if grad_scale is None else self._scalar(grad_scale, "grad_scale", torch.float32)
            if isinstance(lr, torch.Tensor):
                c.lr, c.lr_device = 0.0, self._scalar(lr, "lr", torch.float32)
            else:
                c.lr, c.lr_device = lr, None
            if isinstance(step, torch.Tensor):
                c.step, c.step_device = 0, self._scalar(step, "step", torch.int32)
            else:
                c.step, c.step_device = self.steps + 1 if step is None else step, None
            self._ran_on(_launch_on(self.device, lib().ob200_launch_adamw, self.table, len(self.table), c))
            if c.step:
                self.steps = c.step
