"""Sweeps of different sizes from several host threads at once, each on a stream
and with a workspace of its own: none takes the other's shared-memory limit for
its launch."""
import ctypes as C
import threading

import pytest
import torch

import cases
from stadeb200 import _lib
from stadeb200 import kernels as K

pytestmark = pytest.mark.gpu

# two sizes of a kernel each that want different amounts of shared memory, both
# past the 48 KB that need no limit set
SIZES = {"affine": [(64, 100, 60), (64, 150, 100)],       # n_s, n_o, n_i
         "logits": [(256, 64, 1024, 10), (256, 64, 2048, 10)],       # n_s, n_i, n_h, n_o
         "head": [(64, 5, 1000, 16), (64, 5, 3000, 16)],
         "hv": [(64, 20, 300, 10), (64, 20, 512, 10)]}


def _call(op, size):
    """(C function, arguments, workspace bytes, arrays)"""
    L = _lib.lib()
    if op == "affine":
        st, _ = cases.affine_state(*size)
        names, fn, need = cases.AFFINE_ARGS, L.stade_affine_ls_b_f64, K.affine_ls_b_workspace(*size)
    elif op == "hv":
        st, _ = cases.mlp_hv_state(*size)
        names, fn, need = cases.MLP_ARGS, L.stade_mlp2_ce_hv_f64, K.mlp2_ce_hv_workspace(*size)
    else:
        st, _ = cases.mlp_state(*size)
        names, fn, need = cases.MLP_ARGS, L.stade_mlp2_ce_b_f32, K.mlp2_ce_b_workspace(*size)
    dev = {k: torch.from_numpy(v).cuda() for k, v in st.items() if hasattr(v, "dtype")}
    args = [dev[a].data_ptr() for a in names] + list(size)
    if op == "hv":
        args += [dev[a].data_ptr() for a in cases.MLP_TAN]
    return fn, args, need, dev


@pytest.mark.parametrize("op", list(SIZES))
def test_host_threads(op):
    L, failed, ready = _lib.lib(), [], threading.Barrier(4)

    def work(k):
        torch.cuda.set_device(0)
        s = torch.cuda.Stream()
        fn, args, need, _dev = _call(op, SIZES[op][k])
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        o = _lib.make_opts(s.cuda_stream, ws.data_ptr(), need, 0)
        torch.cuda.synchronize()
        ready.wait()
        codes = {fn(*args, C.byref(o)) for _ in range(1500)}
        s.synchronize()
        if codes != {_lib.STADE_OK}:
            failed.append((k, codes, L.stade_last_error()))

    threads = [threading.Thread(target=work, args=(k % 2,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert L.stade_device_error() == 0
