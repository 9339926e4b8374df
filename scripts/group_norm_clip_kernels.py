"""Kernel times and counters of group norm and gradient clipping on the cases of perf/operators.py (on an MI355X):
    rocprofv3 --kernel-trace -f csv -d DIR -o t -- python3 scripts/group_norm_clip_kernels.py run
    rocprofv3 --pmc FETCH_SIZE -f csv -d DIR -o f -- python3 scripts/group_norm_clip_kernels.py run last_block_train,clip_large_mixed,norm_large_bf16
    python3 scripts/group_norm_clip_kernels.py times DIR/t_kernel_trace.csv
    python3 scripts/group_norm_clip_kernels.py counters DIR/*_counter_collection.csv"""
import collections
import csv
import os
import re
import statistics
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
OURS = re.compile(r"(k_gn_\w+?|k_grad_\w+?)(IDF16|If|ILb|E|<|\()")


def run(names):
    import torch
    from perf import operators as ops
    ops.own = True
    for case in ops.listed():
        if names and case["name"] not in names:
            continue
        st = ops.prepare(case, 1)
        for _ in range(13):
            ops.run(st)
        torch.cuda.synchronize()
    print("done", flush=True)


def times(path):
    """medians of the last ten of thirteen calls; the inputs' random numbers separate the cases"""
    from perf import operators as ops
    cases, now = [], []
    for r in sorted(csv.DictReader(open(path)), key=lambda r: int(r["Start_Timestamp"])):
        name = r["Kernel_Name"]
        m = OURS.search(name)
        if m:
            kind = "" if "k_grad" in m.group(1) else "bf16" if "IDF16b" in name else "f16" if "IDF16_" in name else "f32"
            now.append(((m.group(1), kind, r["Grid_Size_X"]), (int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3))
        elif now and ("normal" in name or "distribution" in name):
            cases.append(now)
            now = []
    cases.append(now)
    for case, launches in zip(ops.listed(), cases):
        by = collections.OrderedDict()
        for k, t in launches:
            by.setdefault(k, []).append(t)
        total = sum(statistics.median(v[3:]) * (len(v) / 13) for v in by.values())
        print("%s: sum %.1f us" % (case["name"], total))
        for k, v in by.items():
            print("   %-18s %-5s grid %8s  n %d  median %7.1f us" % (*k, len(v), statistics.median(v[3:])))


def counters(paths):
    by = collections.OrderedDict()
    for path in paths:
        for r in csv.DictReader(open(path)):
            m = OURS.search(r["Kernel_Name"])
            if m:
                by.setdefault((m.group(1), r["Grid_Size"]), collections.OrderedDict()).setdefault(r["Counter_Name"], []).append(float(r["Counter_Value"]))
    for k, v in by.items():
        print("%-18s grid %8s " % k, " ".join("%s=%.4g" % (c, statistics.median(x)) for c, x in v.items()))


if __name__ == "__main__":
    if sys.argv[1] == "run":
        run(sys.argv[2].split(",") if len(sys.argv) > 2 else None)
    elif sys.argv[1] == "times":
        times(sys.argv[2])
    else:
        counters(sys.argv[2:])
