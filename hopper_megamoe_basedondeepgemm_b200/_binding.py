"""The compiled binding of the operators around the layer (csrc/mm_block_binding.cpp), loaded at their first call. There is no fallback: a missing one is an error."""
import importlib.machinery
import importlib.util
import os

import torch

from .build import BINDING_PATH, binding_fits


class _Binding:
    """Its functions as attributes; the first one asked for loads it."""

    def __getattr__(self, name):
        if not os.path.exists(BINDING_PATH):
            raise RuntimeError(f'{BINDING_PATH} is missing: build it with `python -m hopper_megamoe_basedondeepgemm_b200.build` '
                               '(nvcc, sm_100a; g++). There is no CPU or eager fallback for these operators.')
        if not binding_fits(os.path.dirname(torch.__file__)):
            raise RuntimeError(f'{BINDING_PATH} was built with another torch or Python than this one (torch {torch.__version__}): '
                               'build it again with `python -m hopper_megamoe_basedondeepgemm_b200.build`')
        loader = importlib.machinery.ExtensionFileLoader('mm_block_binding', BINDING_PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_file_location('mm_block_binding', BINDING_PATH, loader=loader))
        loader.exec_module(module)
        self.__dict__.update({k: v for k, v in vars(module).items() if not k.startswith('_')})
        return self.__dict__[name]


binding = _Binding()
