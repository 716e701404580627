"""Options of the decode command that concern its context, without a GPU."""
import torch

from cudalab_amd import decode


def test_context_options(monkeypatch, capsys):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    assert decode.main(["--context", "-1"]) == 2
    assert "--context" in capsys.readouterr().err
    assert decode.main(["--context", "100", "--cache-bits", "4"]) == 1
    assert "no GPU visible" in capsys.readouterr().err
