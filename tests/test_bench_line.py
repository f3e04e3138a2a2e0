"""bench.py's result line: the contract's keys, the headline's numbers as measured, and a length that
an output cut to its last 8000 characters still holds."""
import importlib.util
import json
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def bench():
    spec = importlib.util.spec_from_file_location("bench", os.path.join(ROOT, "bench.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def entry(**more):
    return dict({"bound": "mfma", "us": 72.8712345678901, "mean_us": 73.4861234567, "launches_per_step": 2.0,
                 "tflops_f32_equivalent": 221.0312345678, "kernel": "a kernel's name, and how its tiles are cut " * 2,
                 "achieved": 663.0812345678, "peak": 2500.0, "unit": "TFLOP/s", "frac": 0.2652312345678,
                 "max_norm_err_vs_cpu": 3.99951234567e-07, "tokens_checked": 8}, **more)


def a_report(points):
    legs = {"config": "a configuration and what it is", "flops_per_step": 16106127360.0}
    return {
        "metric": "GB/s", "value": 6615.688652137211, "unit": "GB/s", "n_gpus": 1, "steps": 20, "warmup": 5,
        "ms_per_step": 0.09619079999999999, "higher_is_better": True, "scaling": "weak", "vs_baseline": None, "dtype": "f32",
        "data": "synthetic", "config": {"workload": "w" * 150, "weights_bytes": 633233408},
        "roofline": {"bound": "hbm", "achieved": 6815.2812345, "peak": 8000.0, "unit": "GB/s", "frac": 0.851912345, "traffic": 644.75e6,
                     "traffic_source": "s" * 230, "kernel": "k",
                     "gemm_m512": dict(legs, **{f"leg {i}": entry() for i in range(6)},
                                       one_commit_per_product={"us": 1.0, "products": [entry() for _ in range(7)]}),
                     "gemma": dict(legs, **{f"leg {i}": entry() for i in range(4)}),
                     "sweep_2b": dict(legs, points=[dict(entry(), M=8, path="int8 activations, fused tail", tflops=1.23456789,
                                                         frac_hbm=0.123456789, frac_mfma=None) for _ in range(points)])},
        "cpu_baseline": {"value": 2.5369404, "unit": "GB/s", "cores": 1, "kind": "port", "sample": "s" * 100,
                         "per_config": {f"config{i}": {"sample": "s" * 200, "gflops": 4.73921234567} for i in (2, 3, 4)}},
    }


@pytest.mark.parametrize("points", [26, 40, 400])
def test_the_line_is_whole_in_its_last_8000_characters(bench, points):
    report = a_report(points)
    text = bench.result_line(report)
    assert len(text) <= bench.LINE_BYTES < 8000 and "\n" not in text
    line = json.loads(text)
    for k in ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling", "vs_baseline",
              "dtype", "data"):
        assert line[k] == report[k], k
    assert line["config"] == report["config"]
    for k in ("bound", "peak", "unit", "traffic", "traffic_source", "kernel"):
        assert line["roofline"][k] == report["roofline"][k], k
    assert abs(line["roofline"]["achieved"] - report["roofline"]["achieved"]) <= 0.05
    assert line["cpu_baseline"]["cores"] == 1
    if points == 26:  # (as many as the sweep reports)
        assert line["roofline"]["gemm_m512"]["leg 0"]["frac"] == 0.26523
        assert len(line["roofline"]["sweep_2b"]["points"]) == 27
        assert line["roofline"]["sweep_2b"]["points"][1][:2] == [8, "int8 activations, fused tail"]
        assert set(line["cpu_baseline"]["per_config"]) == {"config2", "config3", "config4"}


def test_a_report_without_the_other_configurations(bench):
    report = a_report(1)
    for k in ("gemm_m512", "gemma", "sweep_2b"):
        del report["roofline"][k]
    del report["cpu_baseline"]
    line = json.loads(bench.result_line(report))
    assert set(line) == set(report) and set(line["roofline"]) == set(report["roofline"])
