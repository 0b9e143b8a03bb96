"""The line that bench.py prints: whole in the last few KB of the output."""
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_long_line_keeps_its_values_and_moves_its_reports():
    sys.path.insert(0, ROOT)
    import bench
    leg = {"value": 46.3, "unit": "it/s", "ms_per_step": 21.6, "roofline": {"kernel": "x" * 2000}, "kernel_families": {str(i): {"ms": 1.0} for i in range(100)}}
    out = {"metric": "m", "value": 193.8, "unit": "it/s", "variants_summary": {"sdxl": {"value": 46.3}}, "config": {"workload": "w" * 300}, "roofline": {"kernel": "y" * 2000},
           "kernel_families": {str(i): {"ms": 1.0, "launches": 3} for i in range(60)}, "variants": {"sdxl": leg, "bs8": leg, "batch_invariant": leg}, "steps": 20}
    line, details = bench.contract_line(dict(out))
    assert len(json.dumps(line)) <= 6000 and set(details) == {"variants"}
    assert {**line, **details} == out
    wide = dict(out, kernel_families={str(i): {"ms": 1.0, "launches": 3} for i in range(300)})
    line, details = bench.contract_line(dict(wide))
    assert len(json.dumps(line)) <= 6000 and {**line, **details} == wide and set(details) == {"variants", "kernel_families"}
    short = {"metric": "m", "value": 1.0, "variants": {}, "kernel_families": {}}
    assert bench.contract_line(short) == (short, {})
