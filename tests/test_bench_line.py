"""The line that bench.py prints: its keys, and that it is short enough for a log that holds the last 16 KB."""
import json
import math

import bench


def _line():
    """As long as a default run's: long numbers and texts in every place, eleven workloads more."""
    x = 12345.678901234567
    entry = dict(fwd_us=x, bwd_us=x, eager_ms_per_step=x, eager_calling_thread_ms_per_step=x, peak_transient_bytes=207915984,
                 state_history_bytes=10737418240)

    def parts():
        dom = {"pass": "bwd", "index": 2, "us": x, "bytes": 103956480, "pass_us": x, "pass_frac": x, "n_kernels_in_pass": 4}
        return dict(roofline=dict(bound="hbm", achieved=x, peak=8000.0, unit="GB/s", traffic=x, frac=x, kernel=dom),
                    mfma=dict(util=x, achieved=x, peak=157.3, unit="TFLOP/s", dtype="f32", frac=x, util_grbm=x, flops_per_launch=x,
                              mops_per_mfma_inst=x, valu_insts=x, mfma_insts=x, formula="f" * 240),
                    cpu_baseline=dict(value=x, unit="tokens/s", cores=16, kind="port", sample="s" * 110, method="m" * 140),
                    kernels=[{"pass": p, "index": i, "us": 123.456} for p in ("fwd", "bwd") for i in range(4)], **entry)

    also = {f"workload_{i}_dh128": dict(workload="w" * 70, config=dict(B=3, L=512, H=12, Dh=128, N=64, seg=32, arithmetic="a" * 140),
                                        tokens_per_s=x, ms_per_step=x, **parts()) for i in range(11)}
    decode = {f"decode_{i}": dict(config=dict(kind="ssd", B=3, H=12, Dh=64, N=16), us_per_token=x, eager_us_per_token=x,
                                  tokens_per_s=x, bytes_per_token=42518080,
                                  roofline=dict(bound="hbm", achieved=x, peak=8000.0, unit="GB/s", frac=x)) for i in range(5)}
    return dict(metric=bench.METRIC, value=x, unit="tokens/s", n_gpus=1, steps=20, warmup=5, ms_per_step=x / 1e6,
                higher_is_better=True, scaling="weak", vs_baseline=None, dtype="bf16-in/f32-accum", data="synthetic",
                config=dict(workload="ssd_scan fwd+bwd", B=3, L=512, arithmetic="a" * 160), also=also, decode=decode, **parts())


def test_line_is_kept_whole():
    line = _line()
    before = json.dumps(line)
    text = json.dumps(bench.compact(line), separators=(",", ":"))
    assert len(before) > 16000 and len(text) < 15500
    assert json.dumps(line) == before
    got = json.loads(text)
    for k in ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling", "vs_baseline",
              "dtype", "data", "config"):
        assert got[k] == line[k], k
    assert got.keys() == line.keys() | {"notes"} and got["also"].keys() == line["also"].keys()
    for a, b in zip(got["also"].values(), line["also"].values()):
        assert a.keys() == b.keys() and math.isclose(a["tokens_per_s"], b["tokens_per_s"], rel_tol=1e-5)
        assert sum(a["kernels"]["fwd"] + a["kernels"]["bwd"]) == sum(k["us"] for k in b["kernels"])
    assert got["notes"] == {"mfma_f32": "f" * 240, "cpu_baseline": "m" * 140, "arithmetic_also_f32_or_dense": "a" * 140}


def test_line_without_the_optional_parts():
    line = _line()
    line.update(also={}, decode={}, mfma=None, cpu_baseline=None)
    got = bench.compact(line)
    assert got["notes"] == {} and got["mfma"] is None and got["value"] == line["value"]
