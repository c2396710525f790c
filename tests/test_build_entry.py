"""The build entry point without a reference source."""

import pytest


def test_a_reference_source_that_is_named_must_exist(tmp_path, monkeypatch, capsys):
    """A wrong ``LRB_REFERENCE_SRC`` is an error; without the variable a missing source is
    reported and the build goes on."""
    import __graft_entry__ as entry

    monkeypatch.setattr(entry, "ROOT", str(tmp_path))
    monkeypatch.setenv("LRB_REFERENCE_SRC", str(tmp_path / "nowhere"))
    with pytest.raises(RuntimeError, match="nowhere"):
        entry.install_reference()
    monkeypatch.delenv("LRB_REFERENCE_SRC")
    monkeypatch.setattr(entry, "DEFAULT_REFERENCE_SRC", str(tmp_path / "missing"))
    entry.install_reference()
    assert "not installed" in capsys.readouterr().out
