#!/usr/bin/env python3
"""The scoring head's operators, kernel by kernel.

    rocprofv3 --kernel-trace --output-format csv -d DIR -- python3 profiles/scoring_head.py
    python3 profiles/scoring_head.py summary DIR/.../*_kernel_trace.csv > profiles/scoring_head_kernel_stats.csv

    rocprofv3 --pmc SQ_BUSY_CU_CYCLES ... --kernel-trace --output-format csv -d DIR -- python3 profiles/scoring_head.py
    python3 profiles/scoring_head.py counters DIR/.../*_counter_collection.csv > profiles/scoring_head_pmc.json

    python3 profiles/scoring_head.py rates > profiles/scoring_head_rates.json

The first runs every case REPEATS times on inputs that lie in memory; the second
writes, per case and kernel, the number of launches a call, the median time and what
the case's bytes and operations make of it; the third the means of the counters that
were collected, per kernel; the fourth what a large copy, fill and library product reach on the same card."""
import csv
import json
import os
import re
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
REPEATS, WARM = 12, 4


def product(m, n, k, fmt, out):
    size, width = {"float32": 4, "bfloat16": 2}[out], {"mxfp4": 17 / 32, "mxfp8": 33 / 32}[fmt]
    return (f"product {m} x {n} x {k} {'8' if fmt == 'mxfp8' else '4'} x 4 bits to {'fp32' if size == 4 else 'bf16'}", "matmul", (m, n, k, fmt, out),
            n * k * 17 / 32 + m * k * width + m * n * size, 2 * m * n * k)


# name, operator, sizes, bytes a call has to move, operations of its products
CASES = [
    ("quantize 34 x 4096 fp32 to 8 bits", "quantize", (34, 4096, "float32", "mxfp8"), 34 * 4096 * (4 + 1 + 1 / 32), 0),
    ("quantize 1M x 1024 bf16 to 4 bits", "quantize", (1_000_000, 1024, "bfloat16", "mxfp4"), 1_000_000 * 1024 * (2 + 0.5 + 1 / 32), 0),
    ("read back 1M x 1024 4 bits to bf16", "dequantize", (1_000_000, 1024, "bfloat16", "mxfp4"), 1_000_000 * 1024 * (2 + 0.5 + 1 / 32), 0),
    ("read back 4032 x 4096 4 bits to fp32", "dequantize", (4032, 4096, "float32", "mxfp4"), 4032 * 4096 * (4 + 0.5 + 1 / 32), 0),
    ("read back 1M x 1000 8 bits to bf16", "dequantize", (1_000_000, 1000, "bfloat16", "mxfp8"), 1_000_000 * (2000 + 1024 + 32), 0),
    ("norm 1 x 4096 bf16 + residual to 8 bits", "norm", (1, 4096, "bfloat16"), 4096 * (6 + 2 + 1 + 1 / 32), 0),
    ("norm 8192 x 4096 bf16 + residual to 8 bits", "norm", (8192, 4096, "bfloat16"), 8192 * 4096 * (6 + 1 + 1 / 32), 0),
    *(product(*sizes) for sizes in (
        (1, 131072, 4096, "mxfp8", "float32"), (1, 4_000_000, 768, "mxfp8", "float32"),
        (32, 131072, 4096, "mxfp8", "float32"), (64, 131072, 4096, "mxfp8", "float32"), (250, 131072, 4096, "mxfp8", "float32"),     # a re-ranking batch
        (300, 4032, 4096, "mxfp8", "float32"), (512, 4032, 4096, "mxfp8", "float32"), (1024, 4032, 4096, "mxfp8", "float32"),
        (256, 16384, 4096, "mxfp8", "float32"), (512, 16384, 4096, "mxfp8", "float32"),
        (64, 131072, 4096, "mxfp4", "float32"), (511, 100_003, 768, "mxfp4", "float32"), (1024, 4032, 4096, "mxfp4", "float32"),
        (2048, 131072, 4096, "mxfp8", "float32"), (2048, 131072, 4096, "mxfp8", "bfloat16"), (2048, 131072, 4096, "mxfp4", "bfloat16"))),
    ("log probabilities 1 x 131072 fp32 top 20", "logprobs", (1, 131072, "float32", 20), 131072 * 4, 0),
    ("log probabilities 63 x 50257 fp16 top 5", "logprobs", (63, 50257, "float16", 5), 63 * 50257 * 2, 0),
    ("log probabilities 2048 x 131072 bf16 top 1", "logprobs", (2048, 131072, "bfloat16", 1), 2048 * 131072 * 2, 0),
    ("log probabilities 250 x 131072 fp32", "logprobs", (250, 131072, "float32", 0), 250 * 131072 * 4, 0),
]


def call(op, sizes):
    import torch

    from medical_rag_amd import scoring
    rows = lambda n, d, dtype: torch.randn(n, d, device="cuda", dtype=getattr(torch, dtype))  # noqa: E731
    if op == "quantize":
        x = rows(*sizes[:3])
        return lambda: scoring.mx_quantize(x, sizes[3])
    if op == "dequantize":
        q = scoring.mx_quantize(rows(*sizes[:3]), sizes[3])
        return lambda: scoring.mx_dequantize(q, getattr(torch, sizes[2]))
    if op == "norm":
        x, residual, weight = rows(*sizes), rows(*sizes), rows(1, *sizes[1:])[0]
        return lambda: scoring.rms_norm_mx(x, weight, residual=residual)
    if op == "matmul":
        m, n, k, fmt, out = sizes
        a, b = scoring.mx_quantize(rows(m, k, "bfloat16"), fmt), scoring.mx_quantize(rows(n, k, "bfloat16"))
        return lambda: scoring.mx_matmul(a, b, getattr(torch, out))
    logits = rows(*sizes[:3])
    tokens = torch.randint(0, sizes[1], (sizes[0],), device="cuda")
    return lambda: scoring.token_logprobs(logits, tokens, sizes[3])


def run():
    import torch
    mark = torch.zeros(1, dtype=torch.int16, device="cuda")
    for name, op, sizes, _, _ in CASES:
        f = call(op, sizes)
        for i in range(WARM + REPEATS):
            if i == WARM:
                torch.cuda.synchronize()
                mark += 1               # a kernel of torch's own between the cases' setup and their calls
            f()
        torch.cuda.synchronize()
        print(name, flush=True)


def summary(path):
    launches = sorted(csv.DictReader(open(path)), key=lambda r: int(r["Start_Timestamp"]))
    ours = ("mx_", "rms_norm_mx", "turn_scales", "token_logprobs")
    runs, inside = [], False
    for r in launches:
        name = r["Kernel_Name"]
        if any(o in name for o in ours):
            if inside:
                runs[-1].append((name, (int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3, r["Grid_Size_X"], r["Workgroup_Size_X"]))
        elif "short" in name and "add" in name.lower():
            runs.append([])
            inside = True
        else:
            inside = False
    assert len(runs) == len(CASES), (len(runs), len(CASES))
    out = csv.writer(sys.stdout)
    out.writerow(["case", "kernel", "launches_a_call", "threads", "median_us", "gb_per_s", "tflop_per_s"])
    for (name, _, _, size, flops), calls in zip(CASES, runs):
        for kernel in dict.fromkeys(c[0] for c in calls):
            mine = [c for c in calls if c[0] == kernel]
            us = sorted(c[1] for c in mine)[len(mine) // 2]
            main = "join" not in kernel and "turn" not in kernel
            short = re.search(r"(mx|rms_norm|turn_scales|token_logprobs)\w*_kernel", kernel).group(0)
            out.writerow([name, short, f"{len(mine) / REPEATS:g}", f"{mine[0][2]}", f"{us:.2f}", f"{size / us / 1e3:.0f}" if main else "",
                          f"{flops / us / 1e6:.0f}" if main and flops else ""])


def counters(path):
    out = {}
    for r in csv.DictReader(open(path)):
        kernel = re.search(r"(mx|rms_norm|turn_scales|token_logprobs)\w*_kernel(<[^>]*>|I\w*E(?=Ev))?", r["Kernel_Name"])
        if kernel:
            of = out.setdefault(f"{kernel.group(0)}, {r['Grid_Size']} threads", {})
            of.setdefault(r["Counter_Name"], {})[r["Dispatch_Id"]] = float(r["Counter_Value"])
    print(json.dumps({k: {c: round(sum(d.values()) / len(d)) for c, d in v.items()} for k, v in out.items()}, indent=1))


def rates():
    import torch

    def median_us(f):
        times = []
        for i in range(WARM + REPEATS):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            f()
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end) * 1e3)
        return sorted(times[WARM:])[REPEATS // 2]
    a, b = (torch.zeros(1 << 28, device="cuda") for _ in range(2))     # 1 GiB each
    x, y = (torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    print(json.dumps({"copy 1 GiB, TB/s read and written": round(2 * 2 ** 30 / median_us(lambda: b.copy_(a)) / 1e6, 2),
                      "fill 1 GiB, TB/s": round(2 ** 30 / median_us(lambda: b.fill_(1.0)) / 1e6, 2),
                      "library product of two 8192 x 8192 bf16, PFLOP/s": round(2 * 8192 ** 3 / median_us(lambda: x @ y) / 1e9, 2)}, indent=1))


if __name__ == "__main__":
    modes = {"summary": summary, "counters": counters, "rates": rates}
    modes[sys.argv[1]](*sys.argv[2:]) if len(sys.argv) > 1 else run()
