"""The line that bench.py prints stays short enough to be read from the end of a log."""
import json

import bench


def test_details_leave_the_line_and_one_figure_per_group_stays():
    groups = {"row_program_with_a_long_name_%d_16384x4096" % i: {"ms": 0.08325, "GB/s": 6449.3, "frac_of_peak": 0.9848, "elements_per_s": 806156642085.8854,
                                                                 "kernels": ["softmax_row_f32_g256_v4_r1"], "bytes": 536870912, "note": "n" * 60}
              for i in range(70)}
    groups["execute"] = {"us_per_run": 3.085, "note": "host clock"}
    line = {"metric": "m", "value": 6307.92, "e2e": {"value": 75.725}, "config": {"strong_scaling": {"world": 1}}, "groups": groups,
            "strong_scaling_detail": {"c1": {"t1_us": 1.893}}}
    short, detail = bench.split_detail(line)
    assert len(json.dumps(line)) > 16000 and len(json.dumps(short)) < 5000
    assert {k: short[k] for k in ("metric", "value", "e2e", "config")} == {k: line[k] for k in ("metric", "value", "e2e", "config")}
    assert short["groups"]["execute"] == 3.085 and all(v == 0.9848 for n, v in short["groups"].items() if n != "execute")
    assert detail == {"groups": groups, "strong_scaling_detail": line["strong_scaling_detail"]} and line["groups"] is groups
    assert bench.split_detail({"value": 1}) == ({"value": 1}, {})
