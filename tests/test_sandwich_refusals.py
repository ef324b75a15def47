"""A refusal of the norms around a block at the C entry, on the CPU."""

import ctypes


def test_residual_out_without_a_branch(pkg):
    from importlib import import_module

    lib, p = import_module("vllm-omni-neuron_b200._lib").load(), ctypes.c_void_p(256)
    norm = lambda x, r: lib.vomni_sandwich_norm(x, p, None, None, None, None, 8, 12, 8, 0, 1e-6, 1, 0, r, p, None)
    assert norm(None, p) == 1  # it would stay unwritten
    assert norm(None, None) == 2 and norm(p, p) == 2  # on to the next check: a width of 12
