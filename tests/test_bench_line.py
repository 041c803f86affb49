"""bench.py prints one line on standard output, short enough to be read back
from the end of a log, with the other configs on standard error."""
import json


def test_one_short_line(monkeypatch, capsys):
    import bench
    line = {"metric": "m", "value": 1.0, "config": {}}
    monkeypatch.setattr(bench, "gpu_arm", lambda a: dict(line))
    monkeypatch.setattr(bench, "run_suite", lambda a: {"config1": {"text": "x" * 30000}})
    monkeypatch.setattr(bench, "finish_ranks", lambda: None)
    monkeypatch.setattr(bench.sys, "argv", ["bench.py"])
    assert bench.main() == 0
    out, err = capsys.readouterr()
    assert [json.loads(x) for x in out.splitlines()] == [line]
    assert list(json.loads(err)["configs"]) == ["config1"]
