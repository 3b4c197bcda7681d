"""Times and calls of the workloads in perf/operators.py, on one GPU.

    python scripts/operators.py times [--draw N] [--only NAME,NAME]   plain form and kernels, in turn: us a pass (median of 5 runs), distance from 64 bits
    python scripts/operators.py extra                                 what the workloads leave out: dx and dw apart, few rows a group, the group look-up, the norm
                                                                      alone, offsets on the host, the one-use clip, a training step
    python scripts/operators.py run [--calls N] [--only NAME,NAME]    N passes of each on the kernels, for a profiler
    python scripts/operators.py counters FILE                         rocprofv3's counter_collection.csv of such a run -> the mean of each counter by kernel

The files operators_*.txt and operators_*.csv under profiles/ are what it printed, or what rocprofv3 wrote beside it."""
from __future__ import annotations

import argparse
import importlib
import random
import sys
import time
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))


def passes(call, runs=5, target=0.02):
    """us a call, the median of `runs` runs of about `target` seconds, after warming up"""
    import torch
    for _ in range(3):
        call()
    torch.cuda.synchronize()
    start = time.perf_counter()
    call()
    torch.cuda.synchronize()
    n = max(3, min(500, int(target / (time.perf_counter() - start))))
    found = []
    for _ in range(runs):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            call()
        b.record()
        b.synchronize()
        found.append(a.elapsed_time(b) * 1000 / n)
    return sorted(found)[runs // 2]


def flat(out):
    import torch
    if isinstance(out, dict):
        out = list(out.values())
    if isinstance(out, (list, tuple)):
        return [t for o in out for t in flat(o)]
    return [out.double().reshape(-1) if isinstance(out, torch.Tensor) else torch.tensor([float(out)], dtype=torch.float64, device="cuda")]


def distance(out, exact):
    """The largest over the outputs of |out - exact| / |exact|"""
    return max(float((a - b.to(a.device)).norm() / b.norm()) if float(b.norm()) else float(a.norm()) for a, b in zip(flat(out), flat(exact)) if a.numel())


def cases(o, args):
    chosen = [c for c in o.listed() if not args.only or c["name"] in args.only.split(",")]
    rng = random.Random(1)
    return chosen + [dict(o.draw(rng), name=f"drawn {i}") for i in range(args.draw)]


def times(o, args):
    import torch
    print(f"{'case':24s} {'plain us':>10s} {'here us':>10s} {'ratio':>7s}   distance from 64 bits: plain, here")
    for case in cases(o, args):
        us, off = [], []
        exact = o.exact(case, 1)
        for own in (False, True):
            o.own = own
            state = o.prepare(case, 1)
            us.append(passes(lambda: o.run(state)))
            off.append(distance(o.run(state), exact) if exact is not None else float("nan"))
            del state
            torch.cuda.empty_cache()
        print(f"{case['name']:24s} {us[0]:10.2f} {us[1]:10.2f} {us[0] / us[1]:7.2f}   {off[0]:.1e} {off[1]:.1e}", flush=True)


def run(o, args):
    import torch
    o.own = True
    for case in cases(o, args):
        state = o.prepare(case, 1)
        for _ in range(args.calls):
            o.run(state)
        torch.cuda.synchronize()
        print(case["name"], flush=True)
        del state


def extra(o, args):
    import numpy as np
    import torch as t
    grouped, gradients = (importlib.import_module(f"3deecelltracker_amd.{m}") for m in ("grouped", "gradients"))
    types = {"fp32": t.float32, "bf16": t.bfloat16, "fp16": t.float16}
    say = lambda what, us, more="": print(f"{what:72s} {us:10.2f} us  {more}", flush=True)

    def operands(rows, groups, k, n, kind):
        off = t.tensor([rows * i // groups for i in range(groups + 1)], dtype=t.int32, device="cuda")
        return (t.randn(rows, k, device="cuda").to(types[kind]), t.randn(groups, k, n, device="cuda").to(types[kind]), t.randn(rows, n, device="cuda").to(types[kind]), off)
    for rows, groups, k, n, kind in ((8192, 8, 1024, 1024, "fp32"), (64, 64, 2048, 1024, "bf16"), (64, 64, 2048, 256, "fp32"), (3001, 7, 776, 1112, "fp16"), (128, 1, 512, 1, "fp32")):
        x, w, dy, off = operands(rows, groups, k, n, kind)
        flop, size = 2.0 * rows * k * n, x.element_size()
        us = passes(lambda: grouped.product(x, w, off))
        say(f"product {rows} x {k} x {n} {kind}, {groups} groups", us, f"{flop / us * 1e-6:.1f} TFLOP/s, {size * (rows * (k + n) + min(groups, rows) * k * n) / us * 1e-6:.2f} TB/s")
    for rows, groups, k, n, kind in ((2048, 2, 512, 512, "fp32"), (256, 2, 512, 512, "fp32"), (2048, 1, 61, 512, "fp32"), (256, 1, 61, 512, "fp32"), (1024, 1, 512, 1, "fp32"),
                                     (128, 1, 512, 1, "fp32"), (16384, 16, 2048, 1536, "bf16"), (64, 64, 2048, 1024, "bf16"), (300, 40, 128, 1000, "fp32"), (32768, 1, 512, 512, "fp32")):
        x, w, dy, off = operands(rows, groups, k, n, kind)
        us = [passes(lambda kw=kw: grouped.product_grad(dy, x, w, off, **kw)) for kw in ({}, dict(need_w=False), dict(need_x=False))]
        say(f"gradients {rows} x {k} x {n} {kind}, {groups} groups", us[0], f"dx alone {us[1]:.2f}, dw alone {us[2]:.2f}")
    for groups in (64, 1024, 8192, 65536):
        x, w, dy, off = operands(65536, groups, 64, 64, "bf16")
        say(f"product 65536 x 64 x 64 bf16 with one block, {groups} groups", passes(lambda: grouped.product(x, w[:1].expand(groups, 64, 64), off)), "(the look-up of a tile's group)")
    x, w, dy, off = operands(600, 3, 64, 64, "fp32")
    host = off.tolist()
    say("product 600 x 64 x 64 fp32, offsets on the device", passes(lambda: grouped.product(x, w, off)))
    say("the same, offsets on the host", passes(lambda: grouped.product(x, w, host)))
    large = [t.randn(12_500_000, device="cuda").to(t.bfloat16) for _ in range(24)]
    us = passes(gradients.GradientSet(large).norm)
    say("norm of 24 tensors, 300 M bf16 values", us, f"{2 * 300e6 / us * 1e-6:.2f} TB/s")
    ffn = importlib.import_module("3deecelltracker_amd.ffn")
    synth = importlib.import_module("3deecelltracker_amd.synth")
    model = ffn.FFN().set_weights_dict(synth.make_ffn_weights(seed=1))
    model.compile(global_clipnorm=1.0)
    grads = list(model._training.g.values())
    for g in grads:
        g.normal_()
    out = [t.empty_like(g) for g in grads]
    say("clip of the matching network's gradients, a set kept", passes(lambda s=gradients.GradientSet(grads, out=out): s.clip(1.0)))
    say("the same list used once", passes(lambda: gradients.clip_by_global_norm(grads, 1.0, out=out)))
    for rows in (128, 1024):
        rng = np.random.default_rng(rows)
        x, y = t.from_numpy(rng.normal(size=(rows, 122)).astype(np.float32)).cuda(), t.from_numpy((rng.uniform(size=rows) < 0.5).astype(np.float32)).cuda()
        say(f"FFN.train_on_batch, {rows} pairs on the device", passes(lambda: model.train_on_batch(x, y)))


def counters(o, args):
    import csv
    found = {}
    for row in csv.DictReader(open(args.file, newline="")):
        name = row["Kernel_Name"]
        if any(k in name for k in ("product_kernel", "dw_kernel", "grad_kernel", "join_kernel", "norm_kernel", "clip_kernel")):
            found.setdefault(name, {}).setdefault(row["Counter_Name"], []).append(float(row["Counter_Value"]))
    columns = sorted({c for v in found.values() for c in v})
    out = csv.writer(sys.stdout, lineterminator="\n")
    out.writerow(["kernel", "calls", *columns])
    for name, v in found.items():
        out.writerow([name, max(len(x) for x in v.values()), *(round(sum(v[c]) / len(v[c])) for c in columns)])


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("what", choices=["times", "extra", "run", "counters"])
    p.add_argument("file", nargs="?")
    p.add_argument("--draw", type=int, default=0)
    p.add_argument("--only", default="")
    p.add_argument("--calls", type=int, default=23)
    args = p.parse_args()
    o = importlib.import_module("perf.operators") if args.what != "counters" else None
    {"counters": counters, "times": times, "extra": extra, "run": run}[args.what](o, args)


if __name__ == "__main__":
    main()
