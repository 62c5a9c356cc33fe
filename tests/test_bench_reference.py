"""bench.py's reference arm times the reference's own code or says that it cannot."""
import json
import types

import bench
import oracle


def test_the_restatement_is_not_passed_off_as_the_reference(monkeypatch, capsys):
    monkeypatch.setattr(oracle.RefBlock, "available", classmethod(lambda cls: False))
    monkeypatch.setattr(bench, "ref_decode", lambda *a: {"value": 1.0, "ms_per_step": 1.0, "cores": 1, "kind": "port",
                                                         "sample": "", "cpu": ""})
    bench.run_reference(types.SimpleNamespace(gpus=1, steps=1, warmup=3), 0)
    line = json.loads(capsys.readouterr().out)
    assert line["impl"] == "reference" and "not built" in line["unavailable"] and "value" not in line


def test_the_reference_s_own_block_is_timed(monkeypatch, capsys):
    monkeypatch.setattr(oracle.RefBlock, "available", classmethod(lambda cls: True))
    monkeypatch.setattr(bench, "ref_decode", lambda *a: {"value": 2.0, "ms_per_step": 1.0, "cores": 1, "kind": "reference",
                                                         "sample": "", "cpu": ""})
    bench.run_reference(types.SimpleNamespace(gpus=1, steps=1, warmup=3), 0)
    line = json.loads(capsys.readouterr().out)
    assert line["value"] == 2.0 and "unavailable" not in line
