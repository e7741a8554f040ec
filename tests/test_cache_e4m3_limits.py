"""The 8-bit cache's entry points at the limits of what they take, on a machine without a GPU."""
import ctypes

import pytest
import torch

from sonicboom_b200 import abi, ops


@pytest.mark.parametrize("name", list(abi.RECORDS))
def test_a_packed_record_is_as_long_as_its_struct(name):
    """An entry point copies the whole struct, the padding behind its last member too."""
    of = {"p": ctypes.c_void_p, "z": ctypes.c_size_t, "i": ctypes.c_int, "f": ctypes.c_float}
    struct = type(name, (ctypes.Structure,), {"_fields_": [(f"m{i}", of[c]) for i, c in enumerate(abi.RECORDS[name])]})
    assert len(abi.pack[name](*[0] * len(abi.RECORDS[name]))) == abi.RECORD_STRUCTS[name].size == ctypes.sizeof(struct)
