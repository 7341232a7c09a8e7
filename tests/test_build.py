"""The build's own logic. Nothing is compiled."""
import sys

from ridge_amd import build as B


def test_without_torch_only_its_extension_is_left_out(monkeypatch, capsys):
    ran = []
    monkeypatch.setattr(B, "_run", lambda cmd, capture=False: ran.append(cmd) or "")
    monkeypatch.setattr(B.os, "replace", lambda a, b: None)
    monkeypatch.setitem(sys.modules, "torch", None)   # import torch raises ImportError
    assert B.build_int8().endswith("libridge_int8.so")
    assert len(ran) == len(B.INT8_SRCS) + 1 and not any("int8_binding" in word for cmd in ran for word in cmd)
    assert "no torch" in capsys.readouterr().out
