"""Loader for the sm_100a extension ``nexttransformer_b200._C``.

CUDA tensors always go through these kernels.  If the library is missing on a machine with a
GPU, every op raises instead of silently running a slower PyTorch path; CPU tensors use the
plain-PyTorch restatement of each op (the oracle the kernels are tested against).
"""
import importlib

import torch

_lib = None
_err = None


def ext():
    """Return the compiled extension module or raise with build instructions."""
    global _lib, _err
    if _lib is None and _err is None:
        try:
            _lib = importlib.import_module("nexttransformer_b200._C")
        except ImportError as e:  # pragma: no cover - depends on the build
            _err = e
    if _lib is None:
        raise RuntimeError("nexttransformer_b200._C is not built; run `python -m nexttransformer_b200.build` "
                           f"({_err})")
    return _lib


def available():
    try:
        ext()
        return True
    except RuntimeError:
        return False


def check_errors():
    """Raise for what the kernels launched so far, on any stream of the current device, have recorded: bounded waits that
    gave up (see csrc/common.cuh), and positions, page numbers and slots that the serving operators refused.  Reading
    clears the record, so everything in it is told at once."""
    if torch.cuda.is_initialized():
        torch.cuda.synchronize()  # the words are read on the default stream, which waits for no other
    g, gw, a, aw, d, dw, sp, sw = ext().read_errors()
    p, pw, ds, dsw = ext().read_serving_errors()
    said = []
    if g or a or d or sp:
        said.append(f"device pipeline wait expired: gemm code {g} at {gw:#x}, attention code {a} at {aw:#x}, "
                    f"delta scan code {d} at {dw:#x}, sparse attention code {sp} at {sw:#x}")
    if p:
        what = {1: "a position lies behind the row's page table", 2: "a page number lies outside the cache",
                3: "a position lies behind the rotary table"}
        said.append(f"paged cache: {what.get(p, f'code {p}')} (row {pw})")
    if ds == 1:
        said.append(f"delta_recurrent: device pipeline wait expired ({dsw:#x})")
    elif ds:
        said.append(f"delta_recurrent: slot outside the states (row {dsw})")
    if said:
        raise RuntimeError("; ".join(said))
