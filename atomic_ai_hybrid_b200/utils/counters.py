"""Counts launches of this package's CUDA kernels (the ``gpu_launches`` figure of
``bench.py``).  Every call into the extension is counted with the number of
kernels that binding launches (1 unless listed in ``MULTI``, as a number or as a function of
the call's arguments)."""
from __future__ import annotations


def _scan_kernels(a, k):
    from ..ops._ext import ext
    # selective_scan(x, dt, A, B, C, conv_w, conv_b, conv_state, state, tokens a row, cu_seqlens, ...)
    return ext()._mod.selective_scan_kernels(a[0], a[8], a[9], a[10])


def _attention_kernels(a, k):
    """``cached_attention(q, k, v, k_cache, .., tokens a row [8], cu_seqlens, slots, prefix, seen, mass, ..)``: the new rows, the row
    kernel and the join; the tile kernel where a sequence or a run may have more than eight query rows, with a join of its
    own where there is no prefix; what rows gather."""
    q, cache, cu, prefix, mass = a[0], a[3], a[9], a[11], a[13]
    if q.shape[0] == 0 or (cu is not None and cu.numel() == 1):
        return 0
    group = q.shape[1] // (cache.shape[1] * cache.shape[3])
    tiles = prefix is not None or cu is not None or a[8] * group > 8
    return 3 + tiles + (tiles and prefix is None) + (0 if mass is None else 1 + tiles)


class LaunchCounter:
    MULTI = {"gdn_fwd": 2, "gdn_fwd_train": 2, "gdn_bwd": 4, "gdn_bwd_saved": 2, "ssd_fwd": 2, "ssd_fwd_train": 2,
             "ssd_bwd": 4, "moe_fwd": 7, "moe_bwd": 8, "ce_online_fwd": 2, "add_rmsnorm_bwd": 2,
             "norm_gate_bwd": 2, "selective_scan": _scan_kernels,
             "cached_attention": _attention_kernels,
             # three GEMMs per row chunk: ce_online_bwd(h, W, labels, lse, ls, g, dW_acc, chunk_rows)
             "ce_online_bwd": lambda a, k: 3 * -(-a[0].shape[0] // a[7])}

    def __init__(self):
        self.count = 0
        self.on = False

    def reset(self):
        self.count = 0

    def enable(self):
        self.on = True

    def disable(self):
        self.on = False

    def add(self, name: str, args=(), kwargs=None):
        if self.on:
            n = self.MULTI.get(name, 1)
            self.count += n(args, kwargs or {}) if callable(n) else n


launch_counter = LaunchCounter()
