"""Stores of 16 bytes through a buffer descriptor have no scalar offset.

The compiler leaves two wait states between a store of more than 8 bytes and an instruction that writes the registers it reads from, but
none where the store's offset is a scalar register; on gfx950 such registers have been written too early (tests/test_stage_of_pairs_gpu.py).
A source that passes 0 for the scalar offset leaves the wait states to the compiler."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "linear_cross_entropy_loss_amd", "csrc")


def _arguments(text, start):
    """The arguments of the call whose opening bracket is at `start`."""
    depth, args, last = 0, [], start + 1
    for i in range(start, len(text)):
        c = text[i]
        if c in "([{":
            depth += 1
        elif c in ")]}":
            depth -= 1
            if depth == 0:
                return args + [text[last:i].strip()]
        elif c == "," and depth == 1:
            args.append(text[last:i].strip())
            last = i + 1
    raise ValueError("no end")


@pytest.mark.parametrize("name", sorted(n for n in os.listdir(CSRC) if n.endswith((".hip", ".h"))))
def test_wide_buffer_stores_have_no_scalar_offset(name):
    text = open(os.path.join(CSRC, name)).read()
    for call in re.finditer(r"__builtin_amdgcn_(?:raw|struct)_buffer_store_(b96|b128)\(", text):
        args = _arguments(text, call.end() - 1)
        assert args[3] == "0", (name, text[:call.start()].count("\n") + 1, args)
    assert "llvm.amdgcn.raw.buffer.store" not in text and not re.search(r"buffer_store_dwordx[34]", text)
