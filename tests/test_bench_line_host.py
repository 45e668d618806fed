"""The benchmark's JSON line: short enough to be read whole from the last 8000 characters of a
log, with every key that its reader looks for and the legs' times."""

from __future__ import annotations

import json

CLOCKS = {f"{what}_{n}": 2000.0 for what in ("gfx_mhz", "mem_mhz", "power_w") for n in ("min", "mean", "max")} | {
    "quotable": True, "spread_frac": 0.01}
CHECK = {"ok": True, "max_abs_err": 1e-4, "cosine": 0.9999999, "units": 256, "what": "a leg " * 20}


def _leg(us):
    return {"us_per_step": us, "split_kernel_us": us, "cache_bytes": 1 << 30, "clocks": CLOCKS,
            "step_us_per_replay": [us] * 3}


def _record():
    rows = [{"ctx": c, "method": m, "hot_us": 5.5, "cold_us": 6.5, "cold_gbps": 1.0, "warmup": {"hot_replays": 500}}
            for c in (512, 2048, 8192, 16384) for m in ("fused4", "fused2", "fp16", "nosplit", "torch", "other")]
    return {
        "metric": "us", "value": 200.1, "unit": "us/decode step", "n_gpus": 1, "steps": 20, "warmup": 5,
        "ms_per_step": 0.2, "higher_is_better": False, "scaling": "weak", "vs_baseline": None, "dtype": "int4",
        "data": "synthetic", "config": {"workload": "w" * 140, "batch": 32}, "roofline": {"frac": 0.83},
        "cpu_baseline": {"value": 1.0, "cores": 16, "config1_reference_cpu_step": {"sample": "s" * 300}},
        "check": {"llama": CHECK, "qwen": {str(i): [CHECK, CHECK] for i in range(60)}}, "check_ok": True,
        "warmup_replays": 25, "warmup_s": 0.5, "clocks": CLOCKS,
        "detail": {"fused4": _leg(200.1), "fp16": _leg(613.0), "paged4": {"page32": _leg(206.0)},
                   "channel_keys": {"k2v2": _leg(152.0)}, "quant_effect_4b": 3.0,
                   "qwen2.5-1.5b": {"rows": rows, "effects": {"512": {str(i): 1.0 for i in range(200)}}},
                   "qwen2.5-1.5b_e2e_decode": {"batch": 16, "ctx": {"8192": {
                       "stock": {"eager_us": 9.0}, "tkv": {"eager_us": 8.0, "graph_us": 7.0}, "speedup": 2.0}}}}}


def test_the_line_is_short_and_complete():
    import bench

    record = _record()
    assert len(json.dumps(record)) > 20000
    line = bench.short_line(record)
    assert len(json.dumps(line)) < 4096 and json.loads(json.dumps(line)) == line
    for key in ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling",
                "vs_baseline", "dtype", "data", "config", "roofline", "check_ok", "warmup_replays", "warmup_s"):
        assert line[key] == record[key]
    assert line["checks"] == {"records": 121, "failed": 0} and line["cpu_baseline"] == {"value": 1.0, "cores": 16}
    assert line["legs"] == {"fused4": 200.1, "fp16": 613.0, "paged4_page32": 206.0, "channel_keys_k2v2": 152.0}
    assert line["qwen2.5-1.5b_hot_cold"]["512"]["fused4"] == [5.5, 6.5]
    assert line["qwen2.5-1.5b_e2e"] == {"8192": {"stock": 9.0, "tkv": 7.0}}
    assert record == _record()


def test_a_failed_check_shows_and_a_quick_run_has_a_line():
    import bench

    record = _record()
    record["check"]["llama"] = dict(CHECK, ok=False)
    assert bench.short_line(record)["checks"] == {"records": 121, "failed": 1}
    quick = dict(_record(), cpu_baseline=None, check=None, check_ok=None, clocks=None, detail={"fused4": _leg(1.0)})
    line = bench.short_line(quick)
    assert line["legs"] == {"fused4": 1.0} and line["checks"] is None and "clocks" not in line
