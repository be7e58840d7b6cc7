"""Options of the benchmark that a run would not honour are refused before anything is built or timed (no GPU)."""
import pytest

from tensorline_b200 import benchmark


@pytest.fixture
def runs(monkeypatch):
    started = []
    for name in ("run_ours", "run_design", "run_reference"):
        monkeypatch.setattr(benchmark, name, lambda a, name=name: started.append((name, a)) or 0)
    return started


@pytest.mark.parametrize("argv", [["--quantize-head"], ["--design", "vutesun", "--weight-bits", "4"], ["--impl", "reference", "--weight-bits", "4"],
                                  ["--design", "fimolix", "--weight-bits", "4", "--quantize-head"], ["--impl", "reference", "--quantize-head"]])
def test_refused(runs, argv, capsys):
    with pytest.raises(SystemExit) as e:
        benchmark.main(argv)
    assert e.value.code == 2 and not runs and "--weight-bits" in capsys.readouterr().err


@pytest.mark.parametrize("argv,run", [([], "run_ours"), (["--weight-bits", "4"], "run_ours"), (["--weight-bits", "4", "--quantize-head"], "run_ours"),
                                      (["--design", "vutesun"], "run_design"), (["--impl", "reference"], "run_reference")])
def test_taken(runs, argv, run):
    assert benchmark.main(argv) == 0 and [name for name, _ in runs] == [run]


def test_the_weights_are_named_with_the_precision(runs):
    for argv, named in (([], "bf16"), (["--weight-bits", "4"], "bf16, weights of 4 bits"), (["--weight-bits", "4", "--quantize-head"], "bf16, weights and output head of 4 bits")):
        benchmark.main(argv)
        assert benchmark.precision(runs[-1][1]) == named
