"""profiles/f8_kernels.json from the raw output of profiles/collect_f8.sh: summarize_f8.py <folder>"""
import csv
import glob
import json
import os
import re
import sys

src = sys.argv[1]
short = lambda n: re.sub(r"^void ", "", n).split("(")[0].replace("ssmi::", "")  # noqa: E731
out = {}
for folder in sorted(glob.glob(os.path.join(src, "stats_*/"))):
    name = os.path.basename(os.path.dirname(folder))[6:]
    for f in glob.glob(folder + "**/*kernel_stats.csv", recursive=True):
        for r in csv.DictReader(open(f)):
            if "ssmi::f8_" in r["Name"]:
                out.setdefault(name, {})[short(r["Name"])] = {"launches": int(r["Calls"]), "us": round(float(r["AverageNs"]) / 1e3, 2), "min_us": round(float(r["MinNs"]) / 1e3, 2)}
for folder in sorted(glob.glob(os.path.join(src, "pmc_*/"))):
    name = re.sub(r"_(FETCH_SIZE|WRITE_SIZE|SQ_\w+)$", "", os.path.basename(os.path.dirname(folder))[4:])
    sums = {}
    for f in glob.glob(folder + "**/*counter_collection.csv", recursive=True):
        for r in csv.DictReader(open(f)):
            if "ssmi::f8_" in r["Kernel_Name"]:
                s = sums.setdefault((short(r["Kernel_Name"]), r["Counter_Name"]), [0.0, set()])
                s[0] += float(r["Counter_Value"])
                s[1].add(r["Dispatch_Id"])
    for (kernel, counter), (total, launches) in sums.items():
        out.setdefault(name, {}).setdefault(kernel, {})[counter] = round(total / len(launches), 1)
for kernels in out.values():
    for v in kernels.values():
        if v.get("GRBM_GUI_ACTIVE") and "SQ_VALU_MFMA_BUSY_CYCLES" in v:
            # (GRBM counts per XCD, SQ per SIMD: 8 XCDs, 1024 SIMDs)
            v["matrix_pipe_busy"] = round(v["SQ_VALU_MFMA_BUSY_CYCLES"] / (v["GRBM_GUI_ACTIVE"] / 8 * 1024), 3)
            if v.get("us", 0) > 100:   # (shorter ones are not alone in the counted time)
                v["clock_GHz"] = round(v["GRBM_GUI_ACTIVE"] / 8 / v["us"] / 1e3, 2)
        if "FETCH_SIZE" in v:
            v["read_GB"] = round(v["FETCH_SIZE"] * 2048 / 1e9, 3)   # (KiB; half of a wide coalesced read is counted)
json.dump({"command": "rocprofv3 --kernel-trace --stats / --pmc (a run each) -- python3 tools/prof_f8.py ...: profiles/collect_f8.sh",
           "note": "us per launch; counters per launch, collected apart from the times (a profiled clock may differ)", "runs": out},
          open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "f8_kernels.json"), "w"), indent=1)
