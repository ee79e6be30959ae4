"""What the entry of the attention over a paged cache plans for a call, asked of the built extension without a GPU: nothing is launched."""
import ctypes

import torch  # noqa: F401  (its libraries are what the extension links)

from archscale_b200.ops import backend


class View(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "ks", "vs")] \
        + [(n, ctypes.c_int64) for n in ("k_page", "k_group", "k_slot", "v_page", "v_group", "v_slot", "ks_page", "ks_group", "ks_slot", "vs_page", "vs_group", "vs_slot")] \
        + [(n, ctypes.c_void_p) for n in ("table", "lengths", "new_lengths")] + [("table_row", ctypes.c_int64)] \
        + [(n, ctypes.c_int) for n in ("pages", "groups", "page_size", "dim", "type", "table_cols")] + [("status", ctypes.c_void_p)]


class Query(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "out", "lse", "sink", "lam", "w")] + [(n, ctypes.c_int64) for n in ("q_batch", "q_token", "q_head")] \
        + [(n, ctypes.c_float) for n in ("scale", "gain", "eps")] \
        + [(n, ctypes.c_int) for n in ("B", "T", "H", "type", "window", "diff", "sink_type", "lam_type", "w_type")]


def workspace(B, T, H, G, D, S, cols, window=-1, diff=False, e4m3=False, sms=148):
    """Bytes of the workspace: 0 where an item lies in one CTA or one cluster, or where the kernel of one query row per CTA takes the call."""
    pages = max(1, B * cols)
    c = View(1 << 20, 1 << 20, 1 << 20, 1 << 20, *(2 * (G * S * D, S * D, D)), *(2 * (G * S, S, 1)), 1 << 20, 1 << 20, None, cols, pages, G, S, D, 2 if e4m3 else 1, cols, None)
    a = Query(1 << 20, 1 << 20, None, None, None, None, T * H * D, H * D, D, 0.1, 1.0, 1e-5, B, T, H, 1, window, int(diff), 0, 0, 0)
    f = ctypes.CDLL(backend.extension_path()).b200_paged_attention_workspace
    f.restype, f.argtypes = ctypes.c_int64, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int]
    return f(ctypes.byref(c), ctypes.byref(a), sms)
