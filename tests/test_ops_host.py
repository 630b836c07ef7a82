"""What the operators' Python side refuses before it calls the library: tensors that a kernel could not reach, arrays too small."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from pega_omni_b200.ops import Ops, OpsError


class Tensor:
    """A tensor's metadata on a device of one's choice."""

    def __init__(self, *shape, dtype=torch.int32, device=0, pinned=False):
        self._t, self._device, self._pinned = torch.empty(*shape, dtype=dtype), device, pinned

    def get_device(self):
        return self._device

    def is_pinned(self):
        return self._pinned

    @property
    def device(self):
        return torch.device("cpu" if self._device < 0 else f"cuda:{self._device}")

    def __getattr__(self, name):
        return getattr(self._t, name)


class Library:
    """Counts calls instead of making them."""
    calls = 0

    def __getattr__(self, name):
        def call(*args):
            self.calls += 1
            return 0
        return call


@pytest.fixture
def ops():
    o = Ops.__new__(Ops)
    o._lib, o._h, o._device = Library(), None, 0
    return o


HQ, HK, D = 4, 2, 64


def arguments(name):
    ints = lambda *s: Tensor(*s)  # noqa: E731
    rows = lambda n, heads: Tensor(n, heads * D, dtype=torch.bfloat16)  # noqa: E731
    gain = lambda: Tensor(D, dtype=torch.bfloat16)  # noqa: E731
    cache = [Tensor(9, HK, 2, 16, D, dtype=torch.uint8), Tensor(9, HK, 2, dtype=torch.float32)]
    return {
        "kv_tables": [ints(3), ints(3), ints(3, 4), ints(20), ints(1), ints(3), ints(1), ints(4), ints(12), ints(4), ints(7), ints(7), ints(7), ints(1)],
        "qk_norm_rope": [rows(5, HQ + HK), gain(), gain(), ints(5), HQ, HK, D, 1e-6, 1e4, rows(5, HQ + HK)],
        "packed_attend": [rows(5, HQ), rows(5, HK), rows(5, HK), ints(3), HQ, HK, D, 0.1, rows(5, HQ)],
        "kv8_append": [rows(5, HK), rows(5, HK), ints(5), *cache],
        "kv8_attend": [rows(5, HQ), *cache, ints(5), ints(6), ints(9), HQ, 0.1, rows(5, HQ), ints(5)],
    }[name]


NAMES = ["kv_tables", "qk_norm_rope", "packed_attend", "kv8_append", "kv8_attend"]


@pytest.mark.parametrize("name", NAMES)
def test_tensors_of_the_device_are_taken(ops, name):
    getattr(ops, name)(*arguments(name))
    assert ops._lib.calls == 1


@pytest.mark.parametrize("where", [-1, 1])
@pytest.mark.parametrize("name", NAMES)
def test_tensors_elsewhere_are_refused(ops, name, where):
    """On the host, or on another device: one of a call's tensors after the other."""
    for i, a in enumerate(arguments(name)):
        if isinstance(a, Tensor):
            args = arguments(name)
            args[i]._device = where
            with pytest.raises(OpsError, match="cpu" if where < 0 else "cuda:1"):
                getattr(ops, name)(*args)
    assert ops._lib.calls == 0


@pytest.mark.parametrize("name", NAMES)
def test_pinned_host_memory(ops, name):
    """Words that the host reads or writes may lie there; rows, gains and pages may not."""
    for i, a in enumerate(arguments(name)):
        if isinstance(a, Tensor):
            args = arguments(name)
            args[i]._device, args[i]._pinned = -1, True
            if a.dtype is torch.int32:
                getattr(ops, name)(*args)
            else:
                with pytest.raises(OpsError, match="cpu"):
                    getattr(ops, name)(*args)


@pytest.mark.parametrize("which", [4, 6, 13])
def test_a_word_for_counts_and_status(ops, which):
    args = arguments("kv_tables")
    args[which] = Tensor(0)
    with pytest.raises(OpsError, match="a word"):
        ops.kv_tables(*args)
    assert ops._lib.calls == 0


def test_torch_is_not_needed_to_import_them():
    code = "import sys; sys.modules['torch'] = None; import pega_omni_b200.ops as o; assert o.Ops and o.gemm_noalloc"
    subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], check=True, timeout=60)
