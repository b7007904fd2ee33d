"""gave_up_waits: the bounded waits that gave up, as the host reads them."""
import contextlib
import ctypes

import pytest
import torch

import bevfusion_triton_b200
from bevfusion_triton_b200 import _lib


class Library:
    """Two error words, and a call that may fail."""

    def __init__(self, spconv=0, attention=0, status=0):
        self.words, self.status = [spconv, attention], status

    def _read(self, n, count, reset):
        ctypes.cast(count, ctypes.POINTER(ctypes.c_uint64)).contents.value = self.words[n]
        if reset:
            self.words[n] = 0
        return self.status

    def bfb_spconv_timeouts(self, count, reset):
        return self._read(0, count, reset)

    def bfb_attention_timeouts(self, count, reset):
        return self._read(1, count, reset)


@pytest.fixture
def library(monkeypatch):
    def use(**words):
        lib, seen = Library(**words), []
        monkeypatch.setattr(_lib, 'load_native', lambda: lib)
        monkeypatch.setattr(torch.cuda, 'device', lambda d: seen.append(d) or contextlib.nullcontext())
        monkeypatch.setattr(torch.cuda, 'synchronize', lambda: seen.append('synchronize'))
        return lib, seen
    return use


def test_sums_both_and_resets(library):
    lib, seen = library(spconv=2, attention=3)
    assert bevfusion_triton_b200.gave_up_waits() == 5 and lib.words == [2, 3]
    assert bevfusion_triton_b200.gave_up_waits('cuda:1', reset=True) == 5 and lib.words == [0, 0]
    assert bevfusion_triton_b200.gave_up_waits() == 0
    assert seen == [None, 'synchronize', 'cuda:1', 'synchronize', None, 'synchronize']


def test_a_failing_read_is_an_error(library):
    library(status=-5)
    with pytest.raises(RuntimeError, match='status -5'):
        bevfusion_triton_b200.gave_up_waits()


@pytest.mark.gpu
def test_none_gave_up(cuda):
    assert bevfusion_triton_b200.gave_up_waits() == 0
    assert bevfusion_triton_b200.gave_up_waits(0, reset=True) == 0
