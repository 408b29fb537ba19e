"""Runs one hot-path kernel a few times on device-resident inputs - the command to put under a profiler.

    python -m accera_b200.profile_cases gemm_bf16 [--m 8192 --n 8192 --k 8192] [--compute tensor_2sm] [--iters 3] [--beta 1.0]
    python -m accera_b200.profile_cases reduce_mean [--rows 8192 --cols 4096]
    python -m accera_b200.profile_cases gather [--table-rows 32000 --cols 4096 --indices 16384]
    python -m accera_b200.profile_cases matmul_relu_f32 [--m 512 --n 512 --k 512]
    python -m accera_b200.profile_cases range [--elements 134217728]
    python -m accera_b200.profile_cases gemm_f16 | gemm_s8 | gemm_tf32 [--m --n --k]      (row-major A, column-major B)
    python -m accera_b200.profile_cases reduce_cols [--rows 4096 --cols 8192]              (mean over the first axis)
    python -m accera_b200.profile_cases gather_elem [--table-rows 4096 --cols 32000 --indices 16384]   (gather along axis 1)
    python -m accera_b200.profile_cases gemm_fp8 [--m --n --k] [--column-scales]           (e4m3, one scale per 128 along K)
    python -m accera_b200.profile_cases quantize_fp8 [--rows 8192 --cols 8192] [--across] [--tiles] [--dtype f32]
    python -m accera_b200.profile_cases embedding | embedding_grad [--table-rows 32000 --cols 4096 --indices 16384] [--dtype f16]

Sizes default to cases whose inputs exceed the 126 MB L2 while holding well under a
few GB on the device, so that a multi-pass profiler capture stays short.
"""
from __future__ import annotations

import argparse

import torch

from . import runtime as rt


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("case", choices=["gemm_bf16", "gemm_f16", "gemm_s8", "gemm_tf32", "reduce_mean", "reduce_cols", "gather", "gather_elem",
                                     "matmul_relu_f32", "range", "gemm_fp8", "quantize_fp8", "embedding", "embedding_grad"])
    ap.add_argument("--elements", type=int, default=1 << 27)
    ap.add_argument("--m", type=int, default=None)
    ap.add_argument("--n", type=int, default=None)
    ap.add_argument("--k", type=int, default=None)
    ap.add_argument("--rows", type=int, default=8192)
    ap.add_argument("--cols", type=int, default=4096)
    ap.add_argument("--table-rows", type=int, default=32000)
    ap.add_argument("--indices", type=int, default=16384)
    ap.add_argument("--compute", default="tensor_2sm")
    ap.add_argument("--iters", type=int, default=3)
    ap.add_argument("--beta", type=float, default=1.0, help="GEMM cases: C <- A @ B + beta * C")
    ap.add_argument("--a-col-major", action="store_true", help="gemm_bf16 / gemm_f16: A stored column-major (M contiguous)")
    ap.add_argument("--b-row-major", action="store_true", help="gemm_bf16 / gemm_f16: B stored row-major (N contiguous)")
    ap.add_argument("--column-scales", action="store_true", help="gemm_fp8: a scale per column of B (the weight gradient) instead of per 128")
    ap.add_argument("--across", action="store_true", help="quantize_fp8: groups down the columns, transposed result")
    ap.add_argument("--tiles", action="store_true", help="quantize_fp8: a scale per 128 x 128 instead of per 1 x 128")
    ap.add_argument("--dtype", choices=["f32", "f16", "bf16"], default="bf16", help="quantize_fp8: type of x; embedding: of table and rows")
    ap.add_argument("--block-major-scales", action="store_true", help="gemm_fp8: a block's scales of all rows and columns side by side")
    ap.add_argument("--option", action="append", default=[], metavar="NAME=VALUE",
                    help="a launch override for this run, e.g. gemm.group_n=16 (see accb_set_option)")
    a = ap.parse_args()
    for item in a.option:
        name, _, value = item.partition("=")
        rt.set_option(name, int(value))
    dev = torch.device("cuda:0")
    torch.manual_seed(0)
    dtype = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[a.dtype]
    if a.case == "gemm_fp8":
        m, n, k = a.m or 8192, a.n or 8192, a.k or 8192
        A = torch.randn(m, k, device=dev).to(torch.float8_e4m3fn)
        B = torch.randn(n, k, device=dev).to(torch.float8_e4m3fn).t()
        blocks = -(-k // rt.FP8_BLOCK)
        sa = torch.rand(m, blocks, device=dev) + 0.5
        sb = (torch.rand(n if a.column_scales else -(-n // rt.FP8_BLOCK), blocks, device=dev) + 0.5).t()
        if a.block_major_scales:
            sa, sb = sa.t().contiguous().t(), sb.contiguous()
        C = torch.zeros(m, n, device=dev, dtype=torch.float32 if a.column_scales else torch.bfloat16)
        for _ in range(a.iters):
            rt.gemm_fp8(A, B, C, sa, sb, beta=0.0)
    elif a.case == "quantize_fp8":
        x = torch.randn(a.rows, a.cols if a.cols != 4096 else 8192, device=dev).to(dtype)
        x = x.t() if a.across else x
        q = torch.empty(x.shape, device=dev, dtype=torch.float8_e4m3fn)
        s = torch.empty(-(-x.shape[0] // rt.FP8_BLOCK) if a.tiles else x.shape[0], -(-x.shape[1] // rt.FP8_BLOCK), device=dev)
        for _ in range(a.iters):
            rt.quantize_fp8(x, q, s)
    elif a.case.startswith("embedding"):
        T = (torch.randn(a.table_rows, a.cols, device=dev) * 0.02).to(dtype)
        u = torch.rand(a.indices, device=dev, dtype=torch.float64)          # word frequencies fall like one over the rank
        ids = (float(a.table_rows) ** u - 1).long().clamp_(0, a.table_rows - 1)
        rows = torch.empty(a.indices, a.cols, device=dev, dtype=dtype)
        grad = torch.empty(a.table_rows, a.cols, device=dev)
        for _ in range(a.iters):
            rt.embedding(T, ids, rows, scale=64.0)
            if a.case == "embedding_grad":
                rt.embedding_grad(rows, ids, grad, scale=64.0)
    elif a.case.startswith("gemm_"):
        m, n, k = a.m or 8192, a.n or 8192, a.k or 8192
        if a.case == "gemm_s8":
            A = torch.randint(-128, 128, (m, k), device=dev, dtype=torch.int8)
            B = torch.randint(-128, 128, (n, k), device=dev, dtype=torch.int8).t()
            C = torch.zeros(m, n, device=dev, dtype=torch.int32)
        elif a.case == "gemm_tf32":
            A = torch.randn(m, k, device=dev)
            B = (torch.randn(n, k, device=dev) / k ** 0.5).t()
            C = torch.zeros(m, n, device=dev)
        else:
            dt = torch.bfloat16 if a.case == "gemm_bf16" else torch.float16
            A = torch.randn(k, m, device=dev).to(dt).t() if a.a_col_major else torch.randn(m, k, device=dev).to(dt)
            B = (torch.randn(k, n, device=dev) / k ** 0.5).to(dt) if a.b_row_major else (torch.randn(n, k, device=dev) / k ** 0.5).to(dt).t()
            C = torch.zeros(m, n, device=dev, dtype=dt if a.case == "gemm_bf16" else torch.float32)
        for _ in range(a.iters):
            rt.gemm(A, B, C, beta=a.beta, relu=a.case != "gemm_s8", compute=a.compute)
    elif a.case == "matmul_relu_f32":
        m, n, k = a.m or 512, a.n or 512, a.k or 512
        A = torch.rand(m, k, device=dev); B = torch.rand(k, n, device=dev); C = torch.zeros(m, n, device=dev)
        for _ in range(a.iters):
            rt.gemm(A, B, C, relu=True, compute="simt")
    elif a.case == "range":
        out = torch.empty(a.elements, device=dev)
        for _ in range(a.iters):
            rt.range_f32(out, 0.0, 0.001)
    elif a.case == "reduce_cols":
        x = torch.randn(1, a.rows, a.cols, device=dev)
        y = torch.empty(a.cols, device=dev)
        for _ in range(a.iters):
            rt.reduce_mean_rank3(x, y, [1])
    elif a.case == "gather_elem":
        T = torch.randn(a.table_rows, a.cols, device=dev) * 0.02
        idx = torch.randint(0, a.cols, (a.indices, 1), device=dev)
        out = torch.empty(a.table_rows, a.indices, 1, device=dev)
        for _ in range(a.iters):
            rt.gather_rank2(T, idx, out, 1)
    elif a.case == "reduce_mean":
        x = torch.randn(1, a.rows, a.cols, device=dev)
        y = torch.empty(a.rows, device=dev)
        for _ in range(a.iters):
            rt.reduce_mean_rank3(x, y, [2])
    else:
        T = torch.randn(a.table_rows, a.cols, device=dev) * 0.02
        idx = torch.randint(0, a.table_rows, (a.indices, 1), device=dev)
        out = torch.empty(a.indices, 1, a.cols, device=dev)
        for _ in range(a.iters):
            rt.gather_rank2(T, idx, out, 0)
    rt.synchronize()
    torch.cuda.synchronize()
    print(f"{a.case}: {a.iters} launches done, {rt.launch_count()} kernels launched by the library")


if __name__ == "__main__":
    main()
