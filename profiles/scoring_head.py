#!/usr/bin/env python3
"""The scoring head's operators, kernel by kernel.

    rocprofv3 --kernel-trace --output-format csv -d DIR -- python3 profiles/scoring_head.py
    python3 profiles/scoring_head.py summary DIR/.../*_kernel_trace.csv > profiles/scoring_head_kernel_stats.csv

    rocprofv3 --pmc SQ_BUSY_CU_CYCLES ... --kernel-trace --output-format csv -d DIR -- python3 profiles/scoring_head.py
    python3 profiles/scoring_head.py counters DIR/.../*_counter_collection.csv > profiles/scoring_head_pmc.json

The first runs every case REPEATS times on inputs that lie in memory; the second
writes, per case and kernel, the number of launches a call, the median time and what
the case's bytes and operations make of it; the third the means of the counters that
were collected, per kernel."""
import csv
import json
import os
import re
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
REPEATS, WARM = 12, 4

# name, operator, sizes, bytes a call has to move, operations of its products
CASES = [
    ("quantize 34 x 4096 fp32 to 8 bits", "quantize", (34, 4096, "float32", "mxfp8"), 34 * 4096 * (4 + 1 + 1 / 32), 0),
    ("quantize 1M x 1024 bf16 to 4 bits", "quantize", (1_000_000, 1024, "bfloat16", "mxfp4"), 1_000_000 * 1024 * (2 + 0.5 + 1 / 32), 0),
    ("read back 1M x 1024 4 bits to bf16", "dequantize", (1_000_000, 1024, "bfloat16", "mxfp4"), 1_000_000 * 1024 * (2 + 0.5 + 1 / 32), 0),
    ("read back 4032 x 4096 4 bits to fp32", "dequantize", (4032, 4096, "float32", "mxfp4"), 4032 * 4096 * (4 + 0.5 + 1 / 32), 0),
    ("read back 1M x 1000 8 bits to bf16", "dequantize", (1_000_000, 1000, "bfloat16", "mxfp8"), 1_000_000 * (2000 + 1024 + 32), 0),
    ("norm 1 x 4096 bf16 + residual to 8 bits", "norm", (1, 4096, "bfloat16"), 4096 * (6 + 2 + 1 + 1 / 32), 0),
    ("norm 8192 x 4096 bf16 + residual to 8 bits", "norm", (8192, 4096, "bfloat16"), 8192 * 4096 * (6 + 1 + 1 / 32), 0),
    ("product 1 x 131072 x 4096 8 x 4 bits to fp32", "matmul", (1, 131072, 4096, "mxfp8", "float32"), 131072 * (4096 * 17 / 32 + 4), 2 * 131072 * 4096),
    ("product 64 x 131072 x 4096 8 x 4 bits to fp32", "matmul", (64, 131072, 4096, "mxfp8", "float32"), 131072 * (4096 * 17 / 32 + 256), 2 * 64 * 131072 * 4096),
    ("product 511 x 100003 x 768 4 x 4 bits to fp32", "matmul", (511, 100_003, 768, "mxfp4", "float32"), 100_003 * (768 * 17 / 32 + 511 * 4), 2 * 511 * 100_003 * 768),
    ("product 2048 x 131072 x 4096 8 x 4 bits to fp32", "matmul", (2048, 131072, 4096, "mxfp8", "float32"), 131072 * (4096 * 17 / 32 + 8192), 2 * 2048 * 131072 * 4096),
    ("product 2048 x 131072 x 4096 8 x 4 bits to bf16", "matmul", (2048, 131072, 4096, "mxfp8", "bfloat16"), 131072 * (4096 * 17 / 32 + 4096), 2 * 2048 * 131072 * 4096),
    ("product 2048 x 131072 x 4096 4 x 4 bits to bf16", "matmul", (2048, 131072, 4096, "mxfp4", "bfloat16"), 131072 * (4096 * 17 / 32 + 4096), 2 * 2048 * 131072 * 4096),
    ("log probabilities 1 x 131072 fp32 top 20", "logprobs", (1, 131072, "float32", 20), 131072 * 4, 0),
    ("log probabilities 63 x 50257 fp16 top 5", "logprobs", (63, 50257, "float16", 5), 63 * 50257 * 2, 0),
    ("log probabilities 2048 x 131072 bf16 top 1", "logprobs", (2048, 131072, "bfloat16", 1), 2048 * 131072 * 2, 0),
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


if __name__ == "__main__":
    {"summary": summary, "counters": counters}[sys.argv[1]](sys.argv[2]) if len(sys.argv) > 1 else run()
