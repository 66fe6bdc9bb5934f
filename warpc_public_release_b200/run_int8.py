"""Quantise, multiply in 8 bits, check and time -- run_tma's contract for the 8-bit operators.

    python -m warpc_public_release_b200.run_int8 M N K [repeat] [--norm] [--out bf16|fp16|fp32]

A (M x K, a row a token) and Bt (N x K, a row a channel) are run_tma's fp16 inputs (uniform[-1, 1] unless WARPC_INPUTS names another
family).  Bt goes to 8 bits once, A in front of every product: by its rows' largest values, or with --norm through the
root-mean-square norm of A plus a residual.  The first pass is checked against the definitions in 64 bits on up to 64 tokens --
8-bit values and the stored sum for equality, scales and products within their roundings -- then `repeat` passes of each operator
run back to back between two CUDA events:

    quantise_rows MxK  ms  GB/s
    int8_KERNEL MxNxK grid=G  MATCH|MISMATCH bad=x/y  ms  TFLOP/s

Returns True when the check passed.  (The reference has no counterpart; the checker is numpy, as in its own harness.)
"""
import os
import sys

import numpy as np

from . import int8
from .run_tma import make_inputs

EPS = 1e-5
KERNEL_NAMES = {v: k for k, v in int8.KERNELS.items()}


def quantise64(t):
    """The definition in 64 bits: q and the largest magnitude of each row."""
    a = np.abs(t).max(axis=1)
    return np.rint(t * 127 / np.where(a > 0, a, 1)[:, None]).astype(np.int8), a


def run(m, n, k, repeat=30, norm=False, out="bf16", stream=None):
    stream = stream or sys.stdout
    import torch
    if not torch.cuda.is_available():
        raise RuntimeError("run_int8: no CUDA device (this library has no CPU path)")
    if "WARPC_INPUTS" in os.environ:
        a, bt, _ = make_inputs(m, n, k)
    else:
        rng = np.random.default_rng(1)
        a, bt = (rng.uniform(-1.0, 1.0, size=(rows, k)).astype(np.float16) for rows in (m, n))
    ld = -(-k // 16) * 16
    kind = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[out]
    da, db = torch.from_numpy(a).cuda(), torch.from_numpy(bt).cuda()
    r, h, w = torch.flip(da, (0,)).contiguous(), torch.empty_like(da), (1 + 0.25 * db[0]).contiguous()
    qa, qb = (torch.zeros((rows, ld), dtype=torch.int8, device="cuda") for rows in (m, n))
    sa, sb = torch.empty(m, device="cuda"), torch.empty(n, device="cuda")
    c = torch.full((m, n), float("nan"), dtype=kind, device="cuda")
    int8.quantise_rows(n, k, db.data_ptr(), qb.data_ptr(), sb.data_ptr(), dtype="fp16", ldq=ld)
    plan = int8.Int8Plan(n, k, qb.data_ptr(), sb.data_ptr(), out=out, ldb=ld)

    def rows():
        if norm:
            int8.norm_quantise_rows(m, k, da.data_ptr(), w.data_ptr(), EPS, qa.data_ptr(), sa.data_ptr(), dR=r.data_ptr(), dH=h.data_ptr(), dtype="fp16",
                                    ldq=ld)
        else:
            int8.quantise_rows(m, k, da.data_ptr(), qa.data_ptr(), sa.data_ptr(), dtype="fp16", ldq=ld)

    def product():
        plan.launch(m, qa.data_ptr(), sa.data_ptr(), c.data_ptr(), lda=ld)

    rows()
    product()
    plan.status()
    # the definitions, on the first tokens
    some = min(m, 64)
    t = a[:some].astype(np.float64)
    bad = 0
    if norm:
        s = (a[:some].astype(np.float32) + r[:some].cpu().numpy().astype(np.float32)).astype(np.float16)
        bad += int(np.count_nonzero(h[:some].cpu().numpy() != s))
        t = s.astype(np.float64) * w.cpu().numpy().astype(np.float64)
        root = np.sqrt((s.astype(np.float64) ** 2).mean(axis=1) + EPS)
    q, top = quantise64(t)
    scale = top / 127 / (root if norm else 1.0)
    bad += int(np.count_nonzero(qa[:some, :k].cpu().numpy() != q))
    bad += int(np.count_nonzero(~(np.abs(sa[:some].cpu().numpy() - scale) <= 1e-5 * scale)))
    q_b, top_b = quantise64(bt.astype(np.float64))
    bad += int(np.count_nonzero(qb[:, :k].cpu().numpy() != q_b))
    ref = (q.astype(np.float64) @ q_b.astype(np.float64).T) * sa[:some].cpu().numpy().astype(np.float64)[:, None] * (top_b / 127)
    half = torch.finfo(kind).eps / 2
    bad += int(np.count_nonzero(~(np.abs(c[:some].double().cpu().numpy() - ref) <= (half * 1.001 + 4 * 2.0 ** -24) * np.abs(ref) + 1e-7)))
    print("first pass done, %d wrong" % bad, file=sys.stderr, flush=True)

    def timed(f):
        f()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(repeat):
            f()
        end.record()
        torch.cuda.synchronize()
        return begin.elapsed_time(end) / repeat

    ms = timed(rows)
    moved = m * k * (7 if norm else 3) + 4 * m
    print("%s %dx%d  %.4f ms  %.0f GB/s" % ("norm_quantise_rows" if norm else "quantise_rows", m, k, ms, moved / ms / 1e6), file=stream)
    ms = timed(product)
    plan.status()
    info = int8.int8_choose(m, n, k)
    name = "int8_%s_%dx%d" % (KERNEL_NAMES[info.kernel], info.tile_m, info.tile_n) + ("_split%d" % info.split if info.split > 1 else "")
    print("%-28s %dx%dx%d grid=%d  %s bad=%d/%d  %.4f ms  %.1f TFLOP/s" % (name, m, n, k, info.grid, "MATCH" if bad == 0 else "MISMATCH", bad, some * n, ms,
                                                                        2.0 * m * n * k / ms / 1e9), file=stream)
    plan.close()
    return bad == 0


def main(argv=None):
    args = list(sys.argv[1:] if argv is None else argv)
    norm = "--norm" in args
    args = [x for x in args if x != "--norm"]
    out = "bf16"
    if "--out" in args:
        i = args.index("--out")
        out = args[i + 1] if i + 1 < len(args) else ""
        del args[i:i + 2]
    try:
        m, n, k = (int(x) for x in args[:3])
        repeat = int(args[3]) if len(args) > 3 else 30
    except ValueError:
        m = 0
    if m <= 0 or n <= 0 or k <= 0 or repeat <= 0 or len(args) > 4 or out not in ("bf16", "fp16", "fp32"):
        print(__doc__, file=sys.stderr)
        return 2
    return 0 if run(m, n, k, repeat, norm, out) else 1


if __name__ == "__main__":
    sys.exit(main())
