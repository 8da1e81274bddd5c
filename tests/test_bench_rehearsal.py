"""bench.py's rehearsal of its ranks on a busy host."""
import json
import types

import bench


def test_a_stretched_sleep_does_not_decide_a_rehearsal(monkeypatch, capsys):
  """The first sleeps of a region are stretched tenfold, as under load: the time is that of an undisturbed region."""
  clock, stretched = [0.0], [7]

  def sleep(seconds):
    clock[0] += seconds * (10 if stretched[0] > 0 else 1)
    stretched[0] -= 1
  monkeypatch.setattr(bench, "time", types.SimpleNamespace(sleep=sleep, perf_counter=lambda: clock[0]))
  bench.rehearse(types.SimpleNamespace(steps=5, warmup=0, lines_per_gpu=4, frames=10), 1, 0)
  assert abs(json.loads(capsys.readouterr().out)["ms_per_step"] - 2.0) < 1e-6
