"""What check_errors says of each bit of the context's error word (csrc/common.cuh), which the context's other operators set
as well: each by its name, a wait that gave up as TimeoutError."""
import os
import re

import pytest
import torch

from agxforge.kernels import kv4
from agxforge_b200 import _native as N

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "agxforge_b200", "csrc")


@pytest.fixture
def word(monkeypatch):
    class Lib:
        value = 0

        def agxc_ctx_error_word(self, ctx, p):
            p._obj.value, self.value = self.value, 0
            return 0

    lib = Lib()
    monkeypatch.setattr(N, "lib", lambda: lib)
    monkeypatch.setattr(N, "context", lambda device=0: None)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda d=None: None)
    return lib


@pytest.mark.parametrize("bits,kind,texts,absent", [
    (1, TimeoutError, ["a bounded device wait gave up"], ["out of range"]),
    (2, RuntimeError, ["token"], ["out of range", "wait"]),
    (4, RuntimeError, ["a position, slot, length or page was out of range"], ["wait"]),
    (5, TimeoutError, ["a bounded device wait gave up", "out of range"], []),
    (8, TimeoutError, ["grid barrier"], ["out of range"]),
    (1 << 20, RuntimeError, ["0x100000"], ["out of range"]),
])
def test_each_bit_by_its_name(word, bits, kind, texts, absent):
    word.value = bits
    with pytest.raises(kind) as e:
        kv4.check_errors()
    assert all(t in str(e.value) for t in texts + ["error word 0x%x" % bits]), str(e.value)
    assert not any(t in str(e.value) for t in absent), str(e.value)
    kv4.check_errors()                                    # read and cleared


def test_every_bit_of_the_library_has_a_name():
    text = open(os.path.join(CSRC, "common.cuh")).read()
    bits = [1 << int(b) for b in re.findall(r"constexpr unsigned kErr\w+ = 1u << (\d+);", text)]
    assert sorted(bits) == sorted(N.ERRORS)
