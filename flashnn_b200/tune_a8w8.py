"""Offline tuning of the A8W8 shape -> tile plan (the static counterpart of the reference's autotune cache,
flashnn/triton_kernels/triton_utils.py:84-151).

    python -m flashnn_b200.tune_a8w8 --measure > points.jsonl     # on a B200: times every pair-tile width per shape
    python -m flashnn_b200.tune_a8w8 --fit points.jsonl           # anywhere: writes csrc/a8w8_plan.h

The planner in csrc/a8w8_kernels.cuh predicts the time of a launch as waves x tile width x a per-width cost of one
output column (narrow tiles re-read the A rows for fewer columns).  `--fit` derives those per-width costs from the
measured points: for every shape, time(width) / time(256) divided by the same ratio of waves x width, then the
median over shapes.  The header it writes holds the constants and, as a comment, the measured table they came from.
"""
import argparse
import json
import os
import statistics
import sys

WIDTHS = [256, 224, 192, 160, 128]
SHAPES = [(4096, 57344, 8192), (4096, 28672, 8192), (4096, 14336, 8192), (4096, 7168, 8192), (4096, 8192, 28672),
          (4096, 4096, 28672), (4096, 2048, 28672), (4096, 1024, 28672), (8192, 8192, 8192), (4096, 11008, 4096),
          (1024, 8192, 8192), (764, 8192, 8192)]
HERE = os.path.dirname(os.path.abspath(__file__))


def waves(m, n, width, pairs=74):
    tiles = ((m + 255) // 256) * ((n + width - 1) // width)
    return (tiles + pairs - 1) // pairs


def measure():
    import torch
    from . import DynamicQuantize  # noqa: F401  (loads the library)
    from . import GemmA8W8, _lib
    from . import workloads as W
    dev = torch.device("cuda", 0)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device=dev)
    op = GemmA8W8(torch.bfloat16)
    for m, n, k in SHAPES:
        a, b = W.rand_int8((m, k), 0).to(dev), W.rand_int8((n, k), 1).to(dev)
        row, col = W.rand_uniform((m,), 2, 0.005, 0.02).to(dev), W.rand_uniform((n,), 3, 0.001, 0.01).to(dev)
        for width in WIDTHS:
            _lib.set_option(_lib.OPT_A8W8_PAIR_TILE, width)
            try:
                ts = []
                for i in range(13):
                    flush.zero_()
                    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                    e0.record()
                    op(a, b, row, col)
                    e1.record()
                    torch.cuda.synchronize()
                    if i >= 3:
                        ts.append(e0.elapsed_time(e1))
            finally:
                _lib.set_option(_lib.OPT_A8W8_PAIR_TILE, 0)
            print(json.dumps({"m": m, "n": n, "k": k, "tile": width, "ms": round(statistics.median(ts), 5)}), flush=True)


def fit(path, out):
    pts = {}
    for ln in open(path):
        ln = ln[ln.index("{"):] if "{" in ln else ""
        if not ln:
            continue
        d = json.loads(ln)
        tile = d.get("tile")
        if tile is None or tile == 0:
            continue
        pts[(d["m"], d["n"], d["k"], tile)] = d["ms"]
    shapes = sorted({k[:3] for k in pts})
    cost = {256: 1.0}
    for w in WIDTHS[1:]:
        ratios = []
        for (m, n, k) in shapes:
            if (m, n, k, w) in pts and (m, n, k, 256) in pts and m * n >= 4096 * 7168:  # large shapes: many waves
                ratios.append(pts[(m, n, k, w)] / pts[(m, n, k, 256)] * (waves(m, n, 256) * 256) / (waves(m, n, w) * w))
        cost[w] = round(statistics.median(ratios), 3)
    lines = ["// Generated by `python -m flashnn_b200.tune_a8w8 --fit` from points measured on a B200 with",
             "// `python -m flashnn_b200.tune_a8w8 --measure`.  Do not edit by hand: re-measure and re-fit.",
             "//",
             "// Time of a CTA-pair launch ~ waves x tile width x kPairColumnCost[width]; a single-CTA launch costs",
             "// kSingleCtaPenalty per column on top of its own waves x width.  plan_a8w8() picks the cheapest.",
             "#pragma once", "", "namespace fnn {", "",
             "constexpr int kPairWidths[] = {" + ", ".join(str(w) for w in WIDTHS) + "};",
             "constexpr double kPairColumnCost[] = {" + ", ".join(f"{cost[w]:.3f}" for w in WIDTHS) + "};",
             "constexpr double kSingleCtaPenalty = 1.35;", "",
             "// Measured points (ms per launch, L2 flushed; * = the planner's choice):",
             "//        M      N      K " + " ".join(f"{w:>8d}" for w in WIDTHS)]
    sys.path.insert(0, os.path.dirname(HERE))
    for (m, n, k) in shapes:
        best = min(WIDTHS, key=lambda w: (waves(m, n, w) * w * cost[w], -w))
        cells = []
        for w in WIDTHS:
            v = pts.get((m, n, k, w))
            cells.append(("%7.4f" % v if v is not None else "      -") + ("*" if w == best else " "))
        lines.append(f"//   {m:6d} {n:6d} {k:6d} " + " ".join(cells))
    lines += ["", "}  // namespace fnn", ""]
    with open(out, "w") as f:
        f.write("\n".join(lines))
    print("wrote", out, cost)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--measure", action="store_true")
    ap.add_argument("--fit", metavar="POINTS")
    ap.add_argument("--out", default=os.path.join(HERE, "csrc", "a8w8_plan.h"))
    a = ap.parse_args()
    if a.measure:
        measure()
    elif a.fit:
        fit(a.fit, a.out)
    else:
        ap.error("give --measure or --fit POINTS")
