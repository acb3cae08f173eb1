"""A kernel's wait that gives up reaches the caller as an error (the status word faked: no device needed)."""
import contextlib

import pytest
import torch

from compressai_b200 import _lib
from compressai_b200 import attention as A


class Fake:
    """The library with a status word of our own."""

    def __init__(self, lib, word):
        self.lib, self.word = lib, word

    def vq2_attention_status(self, reset):
        word, self.word = self.word, _lib.VQ2_OK if reset else self.word
        return word

    def __getattr__(self, name):
        return getattr(self.lib, name)


def test_check_status(monkeypatch):
    monkeypatch.setattr(torch.cuda, "device", contextlib.nullcontext)
    fake = Fake(_lib.load(), _lib.VQ2_ERR_TIMEOUT)
    monkeypatch.setattr(_lib, "load", lambda: fake)
    with pytest.raises(_lib.VQ2Error, match="vq2_paged_attention"):
        A.check_status()
    A.check_status()   # told once
    fake.word = _lib.VQ2_ERR_LAUNCH
    with pytest.raises(_lib.VQ2Error):
        A.check_status()
