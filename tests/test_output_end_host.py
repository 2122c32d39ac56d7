"""CPU tests of the entry points for rows of logits and layer norm: what can be refused without a device, and that the header, the binding
and the documentation name the same arguments."""
import ctypes
import inspect
import os
import re

import pytest

import motifcl_b200 as mb

ENTRIES = ["layernorm", "layernorm_backward", "token_logprobs", "token_logprobs_backward", "distillation_loss", "distillation_loss_backward"]


def _parameters(name):
    text = open(mb._lib.HEADER_PATH).read()
    args = re.search(r"int mcl_cuda_%s\(([^)]*)\);" % name, text).group(1)
    return [a.strip() for a in args.split(",")]


@pytest.mark.parametrize("name", ENTRIES)
def test_binding_matches_the_header(name):
    kinds = {"size_t": ctypes.c_size_t, "float": ctypes.c_float}
    want = [ctypes.c_void_p if "*" in p else kinds[p.split()[0]] for p in _parameters(name)]
    assert getattr(mb.lib(), "mcl_cuda_" + name).argtypes == want


@pytest.mark.parametrize("name", ENTRIES)
def test_a_null_context_is_refused(name):
    f = getattr(mb.lib(), "mcl_cuda_" + name)
    assert f(*[None if t is ctypes.c_void_p else 1 for t in f.argtypes]) == 1
    assert mb.lib().mcl_cuda_last_error(None) == b"context is NULL"


def test_the_longest_list_is_the_kernels():
    csrc = os.path.join(os.path.dirname(mb._lib.HEADER_PATH), os.pardir, "motifcl_b200", "csrc")
    header = re.search(r"#define MCL_CUDA_LIST_MAX (\d+)", open(mb._lib.HEADER_PATH).read()).group(1)
    assert re.search(r"kVocabListMax = (\d+);", open(os.path.join(csrc, "kernels.h")).read()).group(1) == header


@pytest.mark.parametrize("name", ENTRIES)
def test_tensors_of_another_type_are_refused(name):
    """Ids as torch makes them (int64), logits of 16 bits, ids in the place of logits: an address says none of that to the C call."""
    torch = pytest.importorskip("torch")
    args = {n: torch.zeros(4) for n in inspect.signature(getattr(mb.Context, name)).parameters}
    sizes = {"rows", "cols", "n_top", "n_teacher", "eps", "temperature", "row_stride"}
    for n in list(args):
        if n in sizes:
            args[n] = 1
        elif n in ("tokens", "top_ids", "teacher_ids"):
            args[n] = torch.zeros(4, dtype=torch.int32)
    ctx = object.__new__(mb.Context)
    ctx._lib, ctx._ctx = mb.lib(), None
    args.pop("self")
    with pytest.raises(mb.MotifclCudaError, match="context is NULL"):       # as far as the C call
        getattr(ctx, name)(**args)
    for n in args:
        if n in sizes:
            continue
        ids = args[n].dtype == torch.int32
        for wrong in (torch.int64, torch.int16, torch.float32, torch.float64) if ids else (torch.bfloat16, torch.float16, torch.float64, torch.int32):
            with pytest.raises(mb.MotifclCudaError, match="must be int32" if ids else "float32 tensor is needed") as e:
                getattr(ctx, name)(**{**args, n: args[n].to(wrong)})
            assert e.value.code == 1
