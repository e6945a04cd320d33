#!/usr/bin/env python3
"""Runs timed cases of the 8-bit K/V cache (perf/operators.py) a few times, for a profiler, or prints drawn ones.

    rocprofv3 --kernel-trace --stats --output-format csv -d OUT -- python3 tools/kv8_cases.py run all 20
    rocprofv3 --pmc SQ_WAVE_CYCLES SQ_WAIT_ANY ... --output-format csv -d OUT -- python3 tools/kv8_cases.py run NAME[,NAME] 3
    python3 tools/kv8_cases.py times OUT        launches by kernel and grid, median and shortest duration (of a kernel trace)
    python3 tools/kv8_cases.py counters OUT     means per launch by kernel (of a counter run)
    python3 tools/kv8_cases.py drawn SEED N     the sizes of N drawn cases
"""
import collections
import csv
import glob
import os
import random
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "perf")]


def rows(folder, what):
    for f in glob.glob(os.path.join(folder, "**", f"*{what}.csv"), recursive=True):
        with open(f) as g:
            yield from (r for r in csv.DictReader(g) if "kv8" in r["Kernel_Name"])


def kernel(r):
    return r["Kernel_Name"].split("(")[0].split("::")[-1]


def run(names, passes):
    import torch

    import operators as ops
    ops.own = True
    for case in ops.listed():
        if names == ["all"] or case["name"] in names:
            states = [ops.prepare(case, seed) for seed in range(3)]        # three in turn: no pass finds its own input in a cache
            torch.cuda.synchronize()
            for i in range(passes):
                ops.run(states[i % 3])
            torch.cuda.synchronize()
            print(case["name"], flush=True)
            del states


def times(folder):
    d = collections.defaultdict(list)
    for r in rows(folder, "kernel_trace"):
        d[kernel(r), "threads " + " x ".join(r[f"Grid_Size_{c}"] for c in "XYZ")].append(int(r["End_Timestamp"]) - int(r["Start_Timestamp"]))
    for (name, grid), v in d.items():
        v.sort()
        print(f"{name} {grid}: {len(v)} launches, median {v[len(v) // 2] / 1e3:.2f} us, shortest {v[0] / 1e3:.2f}")


def counters(folder):
    d = collections.defaultdict(list)
    for r in rows(folder, "counter_collection"):
        d[kernel(r), r["Counter_Name"]].append(float(r["Counter_Value"]))
    for (name, counter), v in sorted(d.items()):
        print(f"{name} {counter} {sum(v) / len(v):.4g} ({len(v)} launches)")


def drawn(seed, n):
    import operators as ops
    rng = random.Random(seed)
    for i in range(n):
        print(f"drawn {i}", ops.draw(rng))


if __name__ == "__main__":
    what, args = sys.argv[1], sys.argv[2:]
    if what == "run":
        run(args[0].split(","), int(args[1]))
    elif what == "drawn":
        drawn(int(args[0]), int(args[1]))
    else:
        {"times": times, "counters": counters}[what](args[0])
