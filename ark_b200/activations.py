"""Activation operators beside the optimizer step: 8-bit activation
checkpoints and the backward that reads them, and the norm and rotary
positions of queries and keys.

They produce what the step consumes: `weight_grad` writes (or adds) a
projection's gradient straight into its range of the FP16 gradient buffer
(`Optimizer.weight_grad` finds the range by the tensor's name), and the gains'
gradients of `qk_norm_rope_backward` go the same way.

Every function is asynchronous on torch's current stream of the tensors'
device, allocates what it returns (and workspaces) from torch's allocator, and
may be captured into a CUDA graph.  A tensor made on another stream has to be
ordered before the call, as for torch's own operators.  Everything goes
through libark_cuda.so, by way of the binding ark_b200/lib/_ark_torch.so
(ark_b200/csrc/ark_torch.cpp); there is no autograd node and no fallback.
"""
from __future__ import annotations

import importlib.util
import os

import torch  # noqa: F401  (its libraries have to be loaded before the binding)

from . import _lib

_lib.lib()     # the binding links it; missing or of another version, this says so


def _binding():
    # by its file: importing the directory `lib` as a submodule would put a module in the
    # place of the package's function lib()
    path = os.path.join(os.path.dirname(_lib.LIB_PATH), "_ark_torch.so")
    spec = importlib.util.spec_from_file_location("ark_b200._ark_torch", path)
    try:
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    except ImportError as e:
        raise RuntimeError("ark_b200/lib/_ark_torch.so is missing or was built for another torch: build it "
                           "with `make -C ark_b200/csrc all torch` (or __graft_entry__.build()); ark_b200 "
                           "has no fallback") from e
    return module


_ark_torch = _binding()

Act8, RopePlan = _ark_torch.Act8, _ark_torch.RopePlan
act8_pack, act8_unpack, weight_grad = _ark_torch.act8_pack, _ark_torch.act8_unpack, _ark_torch.weight_grad
swiglu, swiglu_backward = _ark_torch.swiglu, _ark_torch.swiglu_backward
rope, qk_norm_rope = _ark_torch.rope, _ark_torch.qk_norm_rope
qk_norm_rope_backward = _ark_torch.qk_norm_rope_backward
