"""One process drives one GPU: the kernels' error word lies there, and calls for another GPU are refused or run the plain statements."""

import re
from pathlib import Path

import pytest
import torch

from torchure_b200 import ops

CSRC = Path(__file__).resolve().parent.parent / "torchure_b200" / "csrc"


@pytest.mark.skipif(ops.ext() is None, reason="the CUDA extension is not built")
def test_calls_for_another_gpu_are_refused():
    ops.ext().check_one_gpu(0, 0)
    ops.ext().check_one_gpu(3, 3)
    for home, now in ((0, 1), (5, 0)):
        with pytest.raises(ValueError, match=f"cuda:{home}.*cuda:{now}"):
            ops.ext().check_one_gpu(home, now)


def test_kernels_get_the_error_word_through_the_check():
    """The unchecked word goes to the host's own readers only; every binding that launches takes it with its operands' device current."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "bindings.cpp").read_text())
    assert len(re.findall(r"\berror_word\(\)", text)) == 3          # its definition, the check, the reader in Python
    assert "check_one_gpu(t.get_device(), at::cuda::current_device())" in text
    assert "Tensor attn_err_word() { return err_word(); }" in text
    for path in CSRC.glob("*_bindings.cpp"):
        if path.name != "comm_bindings.cpp":          # (the collectives have a word of their own)
            assert not re.search(r"torch::zeros\(\{4\}", path.read_text()), path.name


def test_available_asks_the_current_gpu(monkeypatch):
    """A machine with a GPU that runs the kernels and one that does not: the answer is the current one's, whichever was asked first."""
    now, kinds = [0], [(10, 0), (9, 0)]
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 2)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda device=None: kinds[now[0] if device is None else device])
    monkeypatch.setattr(ops, "ext", lambda: object())
    monkeypatch.setattr(ops, "_EVERY_GPU", False)
    for device in (1, 0, 1, 0):
        now[0] = device
        assert ops.available() == (device == 0)
    kinds[1] = (10, 0)          # two of a kind: asked once
    for device in (1, 0):
        now[0] = device
        assert ops.available()
    monkeypatch.setattr(torch.cuda, "get_device_capability", None)
    assert ops.available()
    ops.force_fallback(True)
    try:
        assert not ops.available()
    finally:
        ops.force_fallback(False)
