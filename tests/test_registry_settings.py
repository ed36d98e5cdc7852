"""Settings that a model's decoder does not have are refused by name, in Python and on the command line."""

import json

import pytest

from quantibbler_b200 import registry
from quantibbler_b200.gpu import GpuContext


@pytest.fixture(params=["Virudra", "Vogizen"])
def layered(request, tmp_path):
    """A folder that the registry takes for a layered model (nothing but its kind is read before a refusal)."""
    (tmp_path / "config.json").write_text(json.dumps({"architecture": request.param}))
    return tmp_path


@pytest.mark.parametrize("setting", [{"kv_dtype": "int8"}, {"max_prefix": 5}, {"layers": []}])
def test_a_layered_model_refuses_what_it_has_not(layered, setting):
    with pytest.raises(registry.UnknownSetting, match=f"has no setting '{next(iter(setting))}'; known: max_batch"):
        registry.load_decoder(None, layered, serving="float32", **setting)


def test_the_factorized_decoder_refuses_what_it_has_not(tmp_path):
    with pytest.raises(registry.UnknownSetting, match="factorized decoder has no setting 'vector_rows'"):
        registry.load_decoder(None, tmp_path, vector_rows=3)


@pytest.mark.parametrize("argv,named", [(["generate", "--kv-dtype", "int8"], "kv_dtype"),
                                        (["score", "--continuation", "4"], "max_prefix")])
def test_the_command_line_ends_with_the_reason(layered, monkeypatch, capsys, argv, named):
    from quantibbler_b200.__main__ import main
    monkeypatch.setattr(GpuContext, "init", classmethod(lambda cls: None))
    with pytest.raises(SystemExit) as end:
        main([argv[0], "--model", str(layered), "--prompt", "1,2", *argv[1:]])
    assert end.value.code == 2 and f"has no setting '{named}'" in capsys.readouterr().err
