"""What the benchmark command's --window cannot take is refused before anything is measured."""

import pytest

import benchmark_attention as bench_mod


@pytest.mark.parametrize("argv,message", [
    (["--window", "0"], "--window must be"),
    (["--window", "-5"], "--window must be"),
    (["--window", "8", "--sinks", "-1"], "--sinks"),
    (["--window", "8", "--d", "129"], "--d and --dv"),
    (["--window", "8", "--dv", "256"], "--d and --dv"),
    (["--window", "8", "--scale", "inf"], "finite --scale"),
    (["--window", "8", "--dtype", "float64"], "float32, bfloat16 and float16"),
])
def test_window_is_checked_first(monkeypatch, capsys, argv, message):
    monkeypatch.setattr(bench_mod, "run_one", lambda *a: pytest.fail("a row was measured"))
    with pytest.raises(SystemExit) as e:
        bench_mod.main(argv)
    assert e.value.code == 2 and message in capsys.readouterr().err


@pytest.mark.parametrize("argv", [["--d", "256"], ["--sinks", "-1"], ["--dtype", "float64"], ["--window", "8", "--d", "128"]])
def test_other_arguments_are_taken(monkeypatch, argv):
    seen = []
    monkeypatch.setattr(bench_mod, "run_one", lambda args, n: seen.append(n) or {})
    monkeypatch.setattr(bench_mod, "print_table", lambda rows: None)
    bench_mod.main(argv)
    assert seen == [256, 512, 1024]
