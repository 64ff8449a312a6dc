#!/usr/bin/env python3
"""The records of profiles/gradient_ops/: the gradient operators' kernels over
the cases of perf/operators.py, and forms that these cases leave out.

    python tools/gradient_ops.py passes [NAME,NAME]     18 passes of every case over three
                                                        states in turn, to be profiled
    python tools/gradient_ops.py calls > calls.csv      us a pass of every case, whole calls: in the
                                                        plain form, and here
    python tools/gradient_ops.py forms > forms.csv      us a call: clipping in place, feedback
                                                        in place, stacks of payloads off the
                                                        128-byte lines, making the object
    python tools/gradient_ops.py summary DIR OUT        DIR/{time,fetch,write}: rocprofv3 output
                                                        of `passes` (kernel trace; FETCH_SIZE;
                                                        WRITE_SIZE) -> OUT/kernel_times.csv,
                                                        OUT/hbm_bytes.csv

FETCH_SIZE reports half of the bytes of a wide streaming read on gfx950 and is
doubled; it counts what the Infinity Cache serves too.
"""
import collections
import csv
import glob
import os
import statistics
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "perf")]
PASSES, STATES = 18, 3


def cases(names=None):
    import operators
    operators.own = True
    return operators, [c for c in operators.listed() if not names or c["name"] in names]


def passes(names):
    import torch
    operators, todo = cases(names)
    for c in todo:
        states = [operators.prepare(c, i) for i in range(STATES)]
        for i in range(PASSES):
            operators.run(states[i % STATES])
        torch.cuda.synchronize()
        print(c["name"], flush=True)
        del states
        torch.cuda.empty_cache()


def per_call(fn, sets, rounds=7):
    """us a call, the sets in turn: median of seven groups of `rounds` of them."""
    import torch
    reps = rounds * len(sets)
    for i in range(reps):
        fn(sets[i % len(sets)])
    groups = []
    for _ in range(7):
        e0, e1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        e0.record()
        for i in range(reps):
            fn(sets[i % len(sets)])
        e1.record()
        torch.cuda.synchronize()
        groups.append(e0.elapsed_time(e1) / reps * 1e3)
    return statistics.median(groups)


def calls():
    import torch
    operators, todo = cases()
    print("case,plain_us,us", flush=True)
    for c in todo:
        states = [operators.prepare(c, i) for i in range(STATES)]
        operators.own = False
        plain = per_call(operators.run, states, 1)
        operators.own = True
        here = per_call(operators.run, states)
        print("%s,%.1f,%.1f" % (c["name"], plain, here), flush=True)
        del states
        torch.cuda.empty_cache()


def forms():
    import torch

    import gloo_amd
    from gloo_amd import mx
    operators, _ = cases()

    def report(name, us):
        print('"%s",%.1f' % (name, us), flush=True)
        torch.cuda.empty_cache()

    def tensors(numel, count, dtype, seed):
        gen = torch.Generator("cuda").manual_seed(seed)
        flat = torch.randn(numel, device="cuda", generator=gen).mul_(0.02).to(dtype)
        return flat, list(flat.split(operators._split(numel, count)))

    print("form,us", flush=True)
    for mib, count in ((16, 148), (256, 148), (1024, 291)):
        sets = []
        for i in range(STATES):
            flat, grads = tensors(mib << 18, count, torch.float32, i)
            sets.append((gloo_amd.Gradients(grads), flat,
                         torch.full((), 9.0, dtype=torch.float64, device="cuda")))
        size = "f32 %d MiB" % mib
        report("norm " + size, per_call(lambda s: s[0].norm(), sets))
        report("clip in place, nothing to clip, " + size,
               per_call(lambda s: s[0].clip_norm(float("inf")), sets))
        limits = {id(s): float(s[0].norm()) for s in sets}

        def clipped(s):  # by a limit that falls a little every time
            limits[id(s)] *= 0.9995
            s[0].clip_norm(limits[id(s)])
        report("clip in place, clipped, " + size, per_call(clipped, sets))
        report("clip in place by a given power sum, " + size,
               per_call(lambda s: s[0].clip_norm(2.999, power_sum=s[2]), sets))
        del sets
    for n, dtype in ((64 << 20, torch.bfloat16), (256 << 20, torch.float32)):
        sets = []
        for i in range(STATES):
            x = tensors(n, 1, dtype, i)[0]
            sets.append((x, torch.zeros(n, device="cuda"),
                         torch.empty(mx.payload_bytes(n), dtype=torch.uint8, device="cuda")))
        report("quantise, feedback in place, %s %d Mi" % (str(dtype)[6:], n >> 20),
               per_call(lambda s: mx.quantize(s[0], s[2], residual=s[1], residual_out=s[1]), sets))
        del sets, x
    for k, n, dtype in ((8, 256 << 20, torch.float32), (8, 128 << 20, torch.bfloat16),
                        (4, 128 << 20, None)):
        x = tensors(n, 1, torch.float32, 7)[0]
        one = mx.quantize(x)
        for extra, how in ((0, "128-byte lines"), (16, "16 bytes more each")):
            sets = []
            for i in range(STATES):
                stack = torch.empty(k, one.numel() + extra, dtype=torch.uint8, device="cuda")
                stack[:, :one.numel()] = one
                out = torch.empty_like(one) if dtype is None else \
                    torch.empty(n, dtype=dtype, device="cuda")
                sets.append((out, list(stack)))
            fn = (lambda s: mx.requantize_n(s[0], s[1], n, scale=1 / k)) if dtype is None else \
                (lambda s: mx.reduce_n(s[0], s[1], scale=1 / k))
            report("fold of %d into %s, %d Mi, rows at %s" % (
                k, "a payload" if dtype is None else str(dtype)[6:], n >> 20, how),
                per_call(fn, sets))
            del sets, stack, out
        del x, one
    for count in (24, 148, 291):
        grads = [torch.zeros(4096, device="cuda") for _ in range(count)]
        torch.cuda.synchronize()
        made, closed = [], []
        for _ in range(50):
            t0 = time.perf_counter()
            g = gloo_amd.Gradients(grads)
            t1 = time.perf_counter()
            g.close()
            made.append(t1 - t0)
            closed.append(time.perf_counter() - t1)
        report("making a Gradients of %d tensors (host)" % count, statistics.median(made) * 1e6)
        report("closing it, the device idle (host)", statistics.median(closed) * 1e6)


def kernel_name(mangled):
    return mangled.split("(anonymous namespace)::", 1)[1].replace(
        "glx::(anonymous namespace)::", "").split("(")[0]


def launches(path, pattern, value):
    """{(case, kernel): values} of profiled passes, the kernels of a case in the
    order of their launches."""
    with open(os.path.join(path, "passes.txt")) as f:
        names = [line.strip() for line in f if line.strip() in {c["name"] for c in cases()[1]}]
    files = glob.glob(os.path.join(path, "**", "*" + pattern), recursive=True)
    assert len(files) == 1, files
    with open(files[0]) as f:
        rows = [r for r in csv.DictReader(f) if "glx::" in r["Kernel_Name"]]
    rows.sort(key=lambda r: int(r["Dispatch_Id"]))
    out, at = collections.OrderedDict(), 0
    for c in names:
        # one kernel a pass, or two that differ
        k = 1 if kernel_name(rows[at]["Kernel_Name"]) == kernel_name(rows[at + 1]["Kernel_Name"]) \
            else 2
        for j in range(k):
            part = rows[at + j:at + PASSES * k:k]
            kernels = {kernel_name(r["Kernel_Name"]) for r in part}
            assert len(part) == PASSES and len(kernels) == 1, (c, kernels)
            out[c, kernels.pop()] = [value(r) for r in part]
        at += PASSES * k
    assert at == len(rows), (at, len(rows))
    return out


def summary(src, out):
    def us(r):
        return (int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3

    def kib(times):
        return lambda r: float(r["Counter_Value"]) * 1024 * times
    t = launches(os.path.join(src, "time"), "kernel_trace.csv", us)
    with open(os.path.join(out, "kernel_times.csv"), "w") as f:
        f.write("case,kernel,launches,median_us,min_us\n")
        for (c, k), v in t.items():
            f.write('%s,"%s",%d,%.2f,%.2f\n' % (c, k, len(v), statistics.median(v), min(v)))
    fetched = launches(os.path.join(src, "fetch"), "counter_collection.csv", kib(2))
    written = launches(os.path.join(src, "write"), "counter_collection.csv", kib(1))
    with open(os.path.join(out, "hbm_bytes.csv"), "w") as f:
        f.write("case,kernel,fetched_bytes,written_bytes\n")
        for (c, k), v in fetched.items():
            f.write('%s,"%s",%.0f,%.0f\n' % (c, k, statistics.median(v),
                                             statistics.median(written[c, k])))


if __name__ == "__main__":
    what, args = sys.argv[1], sys.argv[2:]
    if what == "passes":
        passes(args[0].split(",") if args else None)
    else:
        {"calls": calls, "forms": forms, "summary": summary}[what](*args)
