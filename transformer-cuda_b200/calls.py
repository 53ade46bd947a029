"""Loader of lib/_b200calls.so (binding/calls.cpp): the tensor calls that are made once per layer and token, checked and
launched in a few microseconds. There is no fallback: a missing library raises."""
import importlib.util
import os

from . import lib as _lib

HERE = os.path.dirname(os.path.abspath(__file__))
SO_PATH = os.path.join(HERE, "lib", "_b200calls.so")
_module = None


def load():
    global _module
    if _module is None:
        if not os.path.exists(SO_PATH):
            raise _lib.B200AttnError(_lib.ERR_CUDA, f"{SO_PATH} is missing; build it with `python -c \"import __graft_entry__ as e; e.build()\"` "
                                                    "(needs nvcc and g++). There is no CPU or PyTorch fallback.")
        import torch  # noqa: F401  (its libraries have to be in the process first)

        from .loss_ops import B200LossError
        spec = importlib.util.spec_from_file_location("_b200calls", SO_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.set_errors(_lib.B200AttnError, B200LossError)
        _module = module
    return _module
