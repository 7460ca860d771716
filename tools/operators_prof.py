"""GPU: the timed cases of perf/operators.py, and the forms of those operators that the general engine calls in precision 'mx4', as a workload for
rocprofv3 -- and the table of what it collected, per case and kernel (input generators left out):

    rocprofv3 --kernel-trace --output-format csv -d DIR -o r -- python3 tools/operators_prof.py run
    rocprofv3 --pmc COUNTERS --output-format csv -d DIR -o r -- python3 tools/operators_prof.py run      (one directory per set of counters)
    python3 tools/operators_prof.py table DIR [DIR ..] > profiles/operators/kernel_times.csv
    python3 tools/operators_prof.py graph                    (us a call inside a replayed HIP graph of 20 of them, no profiler)

A case is introduced by three launches of a block norm one element wide, which nothing else here makes."""
import collections
import csv
import glob
import importlib.util
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))
PASSES, WARM = 12, 2                                                         # of a case; the first ones are not counted
MARK = "block_norm_rows_kernel<16, 1, false, true>"


def cases():
    """-> [(name, function that prepares the case and returns the call)]"""
    import torch
    from uit_mobile_amd import mx4, norms                                    # (neither touches a GPU before a call: the table needs the names only)
    spec = importlib.util.spec_from_file_location("operators", ROOT / "perf" / "operators.py")
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True

    def timed(case):
        state = ops.prepare(case, 1)
        return lambda: ops.run(state)

    def engine(which):
        """64 ten-second clips of the default UITBase (248 tokens each): one product or norm of a block"""
        M, D = 64 * 248, 768
        g = torch.Generator(device="cuda").manual_seed(1)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")
        affine = (1 + 0.2 * rand(D), 0.1 * rand(D))
        if which == "first norm":
            r = rand(M, D)
            return lambda: norms.block_norm(None, r, pre=affine, out_dtype="mx4")
        if which == "norm":
            y, r = rand(M, D), rand(M, D)
            return lambda: norms.block_norm(y, r, pre=affine, out_dtype="mx4", inplace=True)
        N, K, raw, act, out = {"qkv": (3 * D, D, False, None, torch.float32), "proj": (D, D, True, None, torch.float32),
                               "fc1": (4 * D, D, False, "gelu", "mx4"), "fc2": (D, 4 * D, False, None, torch.float32)}[which]
        w, b, x = mx4.quantize(rand(N, K) * K ** -0.5), 0.1 * rand(N), rand(M, K)
        x = x if raw else mx4.quantize(x)
        return lambda: mx4.linear(x, w, bias=b, act=act, out_dtype=out)
    return ([(c["name"], (lambda c=c: timed(c))) for c in ops.listed()]
            + [(f"engine, 64 clips: {w}", (lambda w=w: engine(w))) for w in ("first norm", "qkv", "proj", "norm", "fc1", "fc2")])


def run():
    import torch
    from uit_mobile_amd import norms
    one, affine = torch.zeros(1, 1, device="cuda"), (None, None)
    with torch.no_grad():
        for name, prepare in cases():
            call = prepare()
            torch.cuda.synchronize()
            for _ in range(3):
                norms.block_norm(None, one, pre=affine)
            for _ in range(PASSES):
                call()
            torch.cuda.synchronize()
            print(name, flush=True)


def graph():
    import torch
    with torch.no_grad():
        for name, prepare in cases():
            call = prepare()
            call()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                for _ in range(20):
                    call()
            e, best = [torch.cuda.Event(enable_timing=True) for _ in range(2)], float("inf")
            for _ in range(12):
                e[0].record()
                g.replay()
                e[1].record()
                torch.cuda.synchronize()
                best = min(best, e[0].elapsed_time(e[1]) * 1e3 / 20)
            print(f"{name}: {best:.2f} us", flush=True)


def short(name):
    """mx4_rows_kernel<1, 8, __bf16, false>; the tools' demanglers do not know __bf16 and lose what follows it"""
    if name.startswith("_Z"):
        name = subprocess.run(["c++filt", name.replace("DF16b", "u6__bf16").replace("DF16_", "u5__f16")], capture_output=True, text=True).stdout.strip()
    return name.split("(")[0].replace("void ", "").replace("uitk::", "").replace("bool _Accum, bool, E", "__bf16, ..")


def table(dirs):
    names = [name for name, _ in cases()]
    out = collections.defaultdict(lambda: collections.defaultdict(list))     # (case, kernel) -> column -> values
    for d in dirs:
        for f in glob.glob(f"{d}/**/*_kernel_trace.csv", recursive=True) + glob.glob(f"{d}/**/*_counter_collection.csv", recursive=True):
            rows = list(csv.DictReader(open(f)))
            counters = "Counter_Name" in rows[0]
            launches = collections.defaultdict(dict)
            for r in rows:
                e = launches[int(r["Dispatch_Id"])]
                e["name"], e["us"] = r["Kernel_Name"], (int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3
                if counters:
                    e[r["Counter_Name"]] = float(r["Counter_Value"])
            at, marks, per = -1, 0, collections.Counter()
            for _, e in sorted(launches.items()):
                if MARK in e["name"]:
                    marks += 1
                    if marks == 3:
                        at, marks, per = at + 1, 0, collections.Counter()
                    continue
                if at < 0 or not any(k in e["name"] for k in ("mx4_", "block_norm")):
                    continue
                per[e["name"]] += 1
                if marks or not WARM < per[e["name"]] <= PASSES:             # (what comes behind the last pass prepares the next case)
                    continue
                for k, v in e.items():
                    if k != "name" and (k != "us" or not counters):
                        out[(names[at], short(e["name"]))][k].append(v)
    cols = ["us"] + sorted({k for v in out.values() for k in v} - {"us"})
    w = csv.writer(sys.stdout, lineterminator="\n")
    w.writerow(["case", "kernel"] + ["us mean", "us min"] + cols[1:])
    for (case, kernel), v in out.items():
        us = v.get("us", [])
        w.writerow([case, kernel, "%.2f" % (sum(us) / len(us)) if us else "", "%.2f" % min(us) if us else ""] + ["%.4g" % (sum(v[c]) / len(v[c])) if c in v else "" for c in cols[1:]])


if __name__ == "__main__":
    {"run": run, "graph": graph}[sys.argv[1]]() if sys.argv[1] != "table" else table(sys.argv[2:])
