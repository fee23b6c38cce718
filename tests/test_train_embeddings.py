"""The arguments of python -m tcc_amd.train_embeddings, on the host, and its
documented command lines on the device."""
import pytest

SMALL = ["--graphs", "6", "--nodes", "300", "--mean-rows", "20", "--dim", "16", "--hidden", "32", "--steps", "2"]


@pytest.mark.parametrize("bad", [["--distill", "4", "--classes", "3"], ["--distill", "65", "--classes", "100"], ["--distill", "-1"],
                                 ["--distill", "2", "--temperature", "0"], ["--distill", "2", "--temperature", "nan"],
                                 ["--classes", "0"], ["--blocks", "1"], ["--norm", "layer", "--blocks", "-1"]])
def test_usage_errors_come_before_any_training(bad, monkeypatch, capsys):
    from tcc_amd import gcn, train_embeddings

    monkeypatch.setattr(train_embeddings, "batch_of_graphs", lambda *a, **k: pytest.fail("something was begun"))
    monkeypatch.setattr(gcn, "EmbeddingGCN", lambda *a, **k: pytest.fail("something was begun"))
    with pytest.raises(SystemExit) as e:
        train_embeddings.main([*SMALL, *bad])
    assert e.value.code == 2 and "error:" in capsys.readouterr().err


@pytest.mark.parametrize("bad", [dict(distill=3, classes=2), dict(distill=65, classes=100), dict(distill=-1), dict(classes=0),
                                 dict(distill=1, temperature=0.0), dict(blocks=1)])
def test_values_that_no_call_takes_come_before_any_training(bad, monkeypatch):
    from tcc_amd import gcn, train_embeddings

    monkeypatch.setattr(train_embeddings, "batch_of_graphs", lambda *a, **k: pytest.fail("something was begun"))
    monkeypatch.setattr(gcn, "EmbeddingGCN", lambda *a, **k: pytest.fail("something was begun"))
    with pytest.raises(ValueError):
        train_embeddings.train(**bad)


@pytest.mark.gpu
@pytest.mark.parametrize("flags,lines", [([], 2), (["--norm", "layer", "--blocks", "2"], 2), (["--distill", "4"], 4),
                                         (["--norm", "layer", "--blocks", "2", "--distill", "4"], 4),
                                         (["--distill", "2", "--classes", "2"], 4)])
def test_documented_commands(gpu, capsys, flags, lines):
    from tcc_amd import train_embeddings

    assert train_embeddings.main([*SMALL, *flags]) == 0
    out = capsys.readouterr().out.splitlines()
    assert len(out) == lines and out[0].startswith("step 0: loss ")
    assert lines == 2 or out[2].startswith("student: step 0: loss ")
