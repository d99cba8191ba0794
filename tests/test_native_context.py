"""The native context that an engine and its clones share (CPU: insmos_ctx_create / _destroy are host code, here the library's own or stand-ins)."""
import gc
import threading
import time

import pytest
import torch

from insmos_amd import _lib
from insmos_amd.engine import Engine


class _Library:
    """Context calls that note when they run; `create` takes a while without the interpreter's lock, as the foreign call may."""

    def __init__(self, real=None, wait=0.02):
        self.real, self.wait, self.made, self.gone = real, wait, [], []

    def insmos_ctx_create(self, cfg, names, layers, n, out):
        time.sleep(self.wait)
        if self.real is not None:
            rc = self.real.insmos_ctx_create(cfg, names, layers, n, out)
        else:
            rc, out._obj.value = 0, 1 + len(self.made)
        self.made.append(out._obj.value)
        return rc

    def insmos_ctx_destroy(self, handle):
        self.gone.append(handle.value)
        return self.real.insmos_ctx_destroy(handle) if self.real is not None else 0


def _engine(lib):
    e = object.__new__(Engine)
    e.lib, e._split_owner, e._ctx_box = lib, False, [None]
    e.w0_const = e.b0_const = e.nbr_bev = torch.zeros(16)
    e.vs, e.dt, e.range, e.tvs = [0.1] * 3, 0.1, [0.0] * 6, [0.1] * 3
    e.score_thresh = e.nms_thresh = e.out_factor = 1.0
    e.shape = {lvl: [1, 1, 1] for lvl in (1, 2, 3, 4, 5)}
    for name in ("in_ch", "ncls", "max_voxels", "max_points", "bevD", "bevH", "bevW", "nbev", "n_bev_layers", "up_ch", "head_ld", "pre_max", "post_max",
                 "quirk_exact"):
        setattr(e, name, 3)

    class Layer:
        w = b = torch.zeros(16)
        K, cin, cout = 27, 16, 16

    e.L = {f"layer{i}": Layer() for i in range(40)}
    return e


@pytest.mark.parametrize("real", [False, True])
def test_clones_that_start_together_share_one_context(real):
    """The launch sets of the first forward of a model start on threads of their own, at the same time.  All get the same context, and none is
    destroyed while a thread runs on it (two were built in every other first forward of two threads, and the first one freed under the thread that
    had been handed it: its layer table, and with it the addresses that kernels are given)."""
    lib = _Library(_lib.load() if real else None)
    e = _engine(lib)
    engines = [e] + [e.clone_shared() for _ in range(3)]
    bar, got, gone_in_use = threading.Barrier(len(engines)), [None] * len(engines), []

    def first_forward(i):
        bar.wait()
        ctx = engines[i]._native_ctx()
        got[i] = ctx.handle.value
        time.sleep(0.05)     # the forward call: it holds no lock
        if ctx.handle.value in lib.gone:
            gone_in_use.append(i)

    threads = [threading.Thread(target=first_forward, args=(i,)) for i in range(len(engines))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(lib.made) == 1 and set(got) == set(lib.made)
    assert not lib.gone and not gone_in_use
    del e, engines
    gc.collect()
    assert lib.gone == lib.made      # and with its last engine it goes


def test_a_context_outlives_a_change_of_weights_under_a_running_call():
    """_load_weights() gives an engine a new box; who runs on the old context keeps it until done."""
    lib = _Library()
    e = _engine(lib)
    ctx = e._native_ctx()
    e._ctx_box = [None]              # (what _load_weights() does)
    e._native_ctx()
    assert len(lib.made) == 2 and not lib.gone
    del ctx
    gc.collect()
    assert lib.gone == lib.made[:1]
