#!/usr/bin/env python3
"""Benchmark of the llsa hot path on one MI355X.

    python bench.py [--gpus 1] [--steps K] [--warmup W] [--workload c3|c2|c5|n65536|c4|c5_l3|fwd_sweep] [--no-extras]

A step is one forward + backward of the operator on one batch of synthetic input that is
already resident in HBM.  The default workload is the configuration the headline metric is
quoted on: llsa_l2, B=2, H=6, N=16384 (128x128 Z-ordered), D=64, bf16, topk 16/16, 2-D RoPE
applied in-kernel, smooth-field inputs, dO ~ N(0,1).

One JSON line is printed:
  value        effective TFLOP/s = 14*B*H*N*D*n_kv / step time (algorithmic FLOPs: forward 4, backward 10)
  ms_per_step  forward + backward wall time per step (K steps between two synchronisations; before the W warm-up
               steps the step runs untimed for a quarter of a second so that clocks and caches have settled)
  step_event_times  median and 20 % / 80 % quantiles of per-step HIP-event times (>= 50 steps), the statistics
               the reference's harness reports
  roofline     the slowest MFMA kernel of the step, timed with HIP events on the launch stream in a
               second pass that runs the same kernels stage by stage; `traffic` = its HBM-side bytes per
               launch as the committed rocprofv3 summary named in `traffic_source` holds them, null
               where that summary was taken with other kernels
  roofline_hbm the pooling pyramid (the q, k, v launch) against the HBM peak, on its algorithmic bytes
  cpu_baseline the CPU oracle (plain PyTorch restatement) on the host cores, same workload in fp32, and
               under `c1` benchmark configuration 1 (llsa_l1 forward, fp32, N = 1024), median of 10
  kernels      per-stage times of that second pass (ms), with the achieved rate of each (TFLOP/s on
               algorithmic FLOPs for the attention kernels, GB/s on algorithmic bytes for the others)
  dense_sdpa   F.scaled_dot_product_attention forward+backward on the same shapes, same GPU
  other_workloads  (default workload only) the two other sizes the target names, 20 steps each: llsa_l2 against
               dense SDPA at B=1, H=6, N=65536, and llsa_l2 at B=1, H=6, N=262144

--workload c4 times something else, one training step of the operator's caller (a pixel DiT-S with
llsa_l2 in its 12 attention layers, batch 8 of 3x128x128, bf16 autocast, AdamW), and prints a line
of its own kind: ms per step, images/s and the share of the step spent in the operator.  With --fused-layers
the layer norms, linear layers and feed-forward blocks around the attention are this package's operators too.
"""
from __future__ import annotations

import argparse
import json
import math
import os
import sys
import time

ROOT = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, ROOT)

PEAK_BF16_TFLOPS = 2500.0      # MI355X dense bf16 MFMA
PEAK_HBM_GBS = 8000.0          # MI355X HBM3E

# HBM-side bytes per launch (L2 <-> fabric, reads + writes) come from the rocprofv3 --pmc FETCH_SIZE / WRITE_SIZE
# summaries under profiles/ (each counter scaled by what it reads for a 256 MiB elementwise copy; the files say how):
# the table of the workload is parsed at run time, so the figure printed is the one the committed profile holds.
# A profile counts only while the kernels it was taken with are the tree's: its "kernel sources" line is compared with theirs.
TRAFFIC_KERNELS = {"attn_fwd": "attn_fwd_kernel", "bwd_dq": "attn_dq_kernel", "bwd_dkv": "attn_kside_kernel",
                   "bwd_pooled_groups": "attn_kside_group_kernel", "bwd_dpkv_dense": "attn_kside_dense_kernel",
                   "pool_pyramid": "pool_pyramid_kernel", "topk_sparse": "topk_sparse_kernel", "topk_cascade": "topk_sparse_kernel",
                   "topk_dense": "topk_dense_kernel"}


def measured_traffic(workload):
    """{stage: bytes per launch} and the file they were read from ({} and the reason where there is no such measurement)."""
    from llsa_amd.build import kernel_sources_digest
    path = os.path.join(ROOT, "profiles", f"step_kernels_{workload}_hbm_traffic.txt")
    if not os.path.exists(path):
        return {}, None
    rel = os.path.relpath(path, ROOT)
    if f"kernel sources: {kernel_sources_digest()}\n" not in open(path).read():
        return {}, f"none: {rel} was taken with other kernels"
    rows = {}
    for line in open(path):
        parts = line.split()
        if len(parts) >= 7 and parts[0].startswith("llsa::"):
            try:
                rows.setdefault(parts[0], (float(parts[-3]) + float(parts[-2])) * 1e6)       # read_MB + write_MB; a kernel's first row is its largest dispatch shape
            except ValueError:
                pass
    out = {}
    for stage, kern in TRAFFIC_KERNELS.items():
        for name, val in rows.items():
            if name.split("<")[0] == "llsa::" + kern or name.startswith("llsa::" + kern + "<"):
                out.setdefault(stage, val)
    return out, rel


WORKLOADS = {
    # name: (op, B, H, N, topk1, topk2, rope)
    "c2": ("l1", 4, 6, 4096, 16, 0, False),
    "c3": ("l2", 2, 6, 16384, 16, 16, True),
    "c5": ("l2", 1, 6, 262144, 16, 16, True),
    "n65536": ("l2", 1, 6, 65536, 16, 16, True),
    "c5_l3": ("l3", 1, 6, 262144, 16, 16, True),      # three pooled levels (topk 16/16/16), no counterpart in the reference
}


def n_kv(op, N, t1, t2):
    if op == "l3":
        return 16 * t1 + 16 * t2 + 16 * t2 + N // 4096
    return 16 * t1 + N // 16 if op == "l1" else 16 * t1 + 16 * t2 + N // 256


def make_inputs(B, H, N, D, dev):
    import torch
    from llsa_amd.utils.synth import smooth_field
    q = smooth_field(1, B, H, N, D).to(dev)
    k = smooth_field(2, B, H, N, D).to(dev)
    v = smooth_field(3, B, H, N, D).to(dev)
    do = torch.randn(B, H, N, D, generator=torch.Generator().manual_seed(4)).bfloat16().to(dev)
    return q, k, v, do


def timed(fn, iters, torch):
    """Average ms of fn() over iters calls, HIP events on the current stream."""
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(iters):
        fn()
    e1.record()
    e1.synchronize()
    return e0.elapsed_time(e1) / iters


def stage_profile(op, q, k, v, do, t1, t2, freq, iters, torch):
    """Runs the kernels of one forward + backward one stage at a time, the same launches the
    fused operator makes, and times each stage with events on the launch stream."""
    from llsa_amd.kernel.hip import _attention as A
    from llsa_amd._lib import current_lib as _cur
    from llsa_amd.kernel.hip.indices_transpose import transpose_indices_levels
    from llsa_amd.kernel.hip.mean_pool import PoolSpec, pool_pyramid
    from llsa_amd.kernel.hip.topk import compute_topk_indices_sparse, gen_sparse_indices
    # (queued behind ten passes over half a gigabyte, so that stages of a few microseconds are timed back to back on the GPU
    # and not at the rate Python issues them)
    filler = torch.empty(1 << 27, device=q.device, dtype=torch.float32)

    def stage_time(fn, iters, torch):
        for _ in range(10):
            filler.mul_(1.0)
        return timed(fn, iters, torch)

    B, H, N, D = q.shape
    l2 = op == "l2"
    rope = freq is not None
    res = {}

    def pyramid():
        return pool_pyramid([PoolSpec(q, y1=True, y2=l2, xr=True, rope=rope),
                             PoolSpec(k, y1=True, y2=l2, xr=True, y1r=True, rope=rope, y2r=l2),
                             PoolSpec(v, y1=True, y2=l2, xr=True, y1r=True, y1t=True, y2r=l2, y2t=l2)], freq)

    oq, ok, ov = pyramid()
    res["pool_pyramid"] = stage_time(pyramid, iters, torch)
    pq, pk, pv = oq["y1"], ok["y1"], ov["y1"]
    tiles = dict(qr=oq["xr"], kr=ok["xr"], vr=ov["xr"], pkr=ok["y1r"], pvr=ov["y1r"], pvt=ov["y1t"])
    if l2:
        pq2, pk2, pv2 = oq["y2"], ok["y2"], ov["y2"]
        tiles.update(pk2r=ok["y2r"], pv2r=ov["y2r"], pv2t=ov["y2t"])
        from llsa_amd._lib import current_lib
        n2 = N // 256
        if n2 <= current_lib().topk_cascade_max_parents() and (n2 <= 64 or B * H * n2 < 2048):      # the operator's rule: both in one launch
            from llsa_amd.kernel.hip.topk import topk_cascade
            pidx, idx = topk_cascade(pq2, pk2, pq, pk, t1, t2)
            res["topk_cascade"] = stage_time(lambda: topk_cascade(pq2, pk2, pq, pk, t1, t2), iters, torch)
        else:
            pidx = gen_sparse_indices(pq2, pk2, t2)
            res["topk_dense"] = stage_time(lambda: gen_sparse_indices(pq2, pk2, t2), iters, torch)
            idx = compute_topk_indices_sparse(pq, pk, pidx, t1, t2)
            res["topk_sparse"] = stage_time(lambda: compute_topk_indices_sparse(pq, pk, pidx, t1, t2), iters, torch)
        kw = dict(pk2=pk2, pv2=pv2, p_indices=pidx, token_weight_2=256.0)
        cgw = 16.0
    else:
        pidx = None
        idx = gen_sparse_indices(pq, pk, t1)
        res["topk_dense"] = stage_time(lambda: gen_sparse_indices(pq, pk, t1), iters, torch)
        kw = {}
        cgw = 1.0
    o, lse = A.attn_fwd(q, k, v, pk, pv, idx, 16.0, tiles=tiles, **kw)
    res["attn_fwd"] = stage_time(lambda: A.attn_fwd(q, k, v, pk, pv, idx, 16.0, tiles=tiles, **kw), iters, torch)

    chunk = _cur().fine_chunk_for(B, H, N, t1)

    def transposes():          # all levels with one call, as the operator does it
        r = transpose_indices_levels([idx, pidx] if l2 else [idx], chunk)
        return r[0] + r[1] if l2 else r[0]

    csr = transposes()
    res["transpose_indices"] = stage_time(transposes, iters, torch)
    bkw = dict(kw, tiles=tiles, csr=csr, chunk=chunk)
    # as the fused operator calls it: pooled gradients folded into dk / dv by the fine pass
    run = lambda st: A.attn_bwd(do, q, k, v, pk, pv, o, lse, idx, 16.0, cgw, stages=st, freq_dq=freq, fold_pooled=True,
                                freq_dk=freq, **bkw)
    run(0)
    NO_REDUCE = 32
    # l2 at this size: the dense coarsest level rides on the group-major pass of the pooled levels (stage bits 8 | 16)
    merged = l2 and (N // 4096) <= 8
    stages = [("bwd_dq", 2), ("bwd_dkv", 4 | NO_REDUCE)]
    if l2:
        stages.append(("bwd_pooled_groups", (8 | 16 | NO_REDUCE) if merged else (8 | NO_REDUCE)))
    if not merged:
        stages.append(("bwd_dpkv_dense", 16 | NO_REDUCE))
    for name, st in stages:
        # a stage run alone reads whatever workspace the allocator hands back (the block the complete call
        # above filled with delta and the dO tiles); only its duration is used
        res[name] = stage_time(lambda: run(st), iters, torch)
    # the K-side passes with the launches that add up their partial sums, in one piece (no difference of timings)
    res["bwd_kside_all_with_reductions"] = stage_time(lambda: run(4 | 8 | 16), iters, torch)
    return res


def other_workloads(dev):
    """The two other sizes the target names, 20 steps each after 10 untimed ones (HIP events on the launch stream; three
    after one for the dense comparison, whose step is 54 ms):
    llsa_l2 forward + backward against dense F.scaled_dot_product_attention at B=1, H=6, N=65536 (the sparse-vs-dense
    comparison), and llsa_l2 at the largest configuration, B=1, H=6, N=262144.  Same generator, seeds and in-kernel
    RoPE as the headline workload; the reference's harness sweeps the same three sizes (test_kernel.py:27-53)."""
    import torch
    import torch.nn.functional as F
    import llsa_amd
    from llsa_amd.utils.rope_table import rope_table
    res = {}
    for name in ("n65536", "c5"):
        op, B, H, N, t1, t2, rope = WORKLOADS[name]
        q, k, v, do = make_inputs(B, H, N, 64, dev)
        freq = rope_table(math.isqrt(N), dtype=torch.bfloat16).to(dev)
        q.requires_grad_(True), k.requires_grad_(True), v.requires_grad_(True)

        def step():
            q.grad = k.grad = v.grad = None
            llsa_amd.llsa_l2(q, k, v, t1, t2, 16, rope=freq).backward(do)

        def dense():
            q.grad = k.grad = v.grad = None
            F.scaled_dot_product_attention(q, k, v).backward(do)

        n_warm, n_timed = 10, 20           # (the first steps at a new shape are slower: allocator, clocks)
        for _ in range(n_warm):
            step()
        ms = timed(step, n_timed, torch)
        flops = 14.0 * B * H * N * 64 * n_kv(op, N, t1, t2)
        e = {"workload": f"llsa_l2 fwd+bwd B={B} H={H} N={N} D=64 topk={t1}/{t2} rope=in-kernel", "steps": n_timed, "ms_per_step": ms,
             "tflops": flops / (ms * 1e-3) / 1e12}
        if name == "n65536":
            try:
                dense()
                ms_d = timed(dense, 3, torch)
                e["dense_sdpa_ms_per_step"] = ms_d
                e["speedup_llsa_over_dense"] = ms_d / ms
            except Exception as ex:                 # noqa: BLE001
                e["dense_sdpa_error"] = str(ex)[:200]
        res[name] = e
        del q, k, v, do, freq
        torch.cuda.empty_cache()
    return res


def cpu_baseline(op, B, H, N, D, t1, t2, rope):
    """The CPU oracle (plain PyTorch restatement of the reference's algorithm), forward + backward in
    fp32 on the host cores, on the same synthetic inputs."""
    import torch
    from llsa_amd.utils.synth import smooth_field
    from oracle import llsa_oracle as O
    # whole workload when it is small enough for ~20 s of CPU time, else one (b,h) slice; the
    # oracle is run slice by slice to bound its memory
    Bs, Hs = (B, H) if N <= 16384 else (1, 1)
    q, k, v = (smooth_field(s, Bs, Hs, N, D).float() for s in (1, 2, 3))
    do = torch.randn(Bs, Hs, N, D, generator=torch.Generator().manual_seed(4))
    if rope:
        freq = O.rope_table(math.isqrt(N), dtype=torch.float32)
    reps, t_best, t0_all = 0, float("inf"), time.time()
    while reps < 3 and (time.time() - t0_all) < 20.0:
        t0 = time.time()
        for b in range(Bs):
            for h in range(Hs):
                qs, ks, vs, ds = (t[b:b + 1, h:h + 1] for t in (q, k, v, do))
                qr, kr = (O.rope_apply(qs, freq), O.rope_apply(ks, freq)) if rope else (qs, ks)
                if op == "l2":
                    o, ctx = O.llsa_l2_fwd(qr, kr, vs, t1, t2)
                    dq, dk, dv, _ = O.llsa_l2_bwd(ds, ctx)
                else:
                    o, ctx = O.llsa_l1_fwd(qr, kr, vs, t1)
                    dq, dk, dv, _ = O.llsa_l1_bwd(ds, ctx)
                if rope:
                    dq, dk = O.rope_apply_bwd(dq, freq), O.rope_apply_bwd(dk, freq)
        t_best = min(t_best, time.time() - t0)
        reps += 1
    flops = 14.0 * Bs * Hs * N * D * n_kv(op, N, t1, t2)
    return {"value": flops / t_best / 1e12, "unit": "TFLOP/s", "cores": torch.get_num_threads(), "kind": "port",
            "sample": f"oracle llsa_{op} fwd+bwd fp32, B={Bs} H={Hs} N={N} (best of {reps}), {t_best * 1e3:.0f} ms",
            "ms": t_best * 1e3, "c1": cpu_baseline_c1()}


def cpu_baseline_c1():
    """Benchmark configuration 1, the reference's own CPU-runnable case: llsa_l1 forward in fp32, B=1, H=6, N=1024
    (32 x 32 tokens in Z-order), D=64, block_size 16, topk 8, q, k, v ~ N(0,1) from seed 0; median of 10 runs of the
    oracle on the host cores.  (Of the reference only gen_sparse_indices, topk.py:6-9, is plain PyTorch; the oracle
    restates the rest of the path.)"""
    import torch
    from oracle import llsa_oracle as O
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 6, 1024, 64, generator=g) for _ in range(3))
    O.llsa_l1_fwd(q, k, v, 8, 16)
    times = []
    for _ in range(10):
        t0 = time.perf_counter()
        O.llsa_l1_fwd(q, k, v, 8, 16)
        times.append((time.perf_counter() - t0) * 1e3)
    times.sort()
    med = 0.5 * (times[4] + times[5])
    flops = 4.0 * 6 * 1024 * 64 * n_kv("l1", 1024, 8, 0)
    return {"workload": "c1: llsa_l1 forward fp32 B=1 H=6 N=1024 D=64 topk=8, N(0,1) seed 0", "ms_median_of_10": med,
            "ms_min": times[0], "gflops": flops / (med * 1e-3) / 1e9, "cores": torch.get_num_threads(), "kind": "port"}


def bench_dit(args):
    """One flow-matching training step of llsa_amd.caller.PixelDiT (DiT-S: 12 layers, hidden 384, 6 heads
    of 64, qk RMS norm, 2-D RoPE, llsa_l2 topk 16/16) on 8 synthetic 3x128x128 images."""
    import torch
    import llsa_amd
    from llsa_amd._lib import get_lib
    from llsa_amd.caller import FlowMatchingStep, PixelDiT
    from llsa_amd.utils.synth import smooth_field
    get_lib()
    assert torch.cuda.is_available(), "bench.py needs the GPU"
    dev = torch.device("cuda:0")
    B, side, layers, H, D, t1, t2 = 8, 128, 12, 6, 64, 16, 16
    N = side * side
    torch.manual_seed(0)
    model = PixelDiT(num_layers=layers, num_attention_heads=H, attention_head_dim=D, sample_size=side, sparse_topk=(t2, t1),
                     fused_prologue=not args.unfused, fused_layers=args.fused_layers).to(dev)
    step = FlowMatchingStep(model)
    # images: smooth fields in raster order scaled into [-1, 1]; timesteps uniform in [0, 1000); noise N(0,1)
    f = smooth_field(7, B, 1, N, 3, dtype=torch.float32, mix=(1.0, 0.0), zorder=False).reshape(B, side, side, 3).permute(0, 3, 1, 2)
    images = (f / f.abs().amax()).contiguous().to(dev)
    g = torch.Generator().manual_seed(8)
    noise = torch.randn(B, 3, side, side, generator=g).to(dev)
    tsteps = torch.randint(0, 1000, (B,), generator=g).to(dev)

    def time_fn(fn, warmup, steps):
        for _ in range(warmup):
            fn()
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for _ in range(steps):
            fn()
        torch.cuda.synchronize()
        return (time.perf_counter() - t0) * 1e3 / steps

    losses = []
    ms = time_fn(lambda: losses.append(step(images, noise, tsteps)), args.warmup, args.steps)
    losses = [float(l) for l in losses]
    # the operator alone at the shape one layer gives it: (B, N, H, D) memory, qk norm and RoPE inside
    x = (torch.randn(B, N, 3 * H * D, generator=torch.Generator().manual_seed(9)).bfloat16().to(dev))
    q, k, v = (x[..., i * H * D:(i + 1) * H * D].reshape(B, N, H, D).transpose(1, 2).requires_grad_(True) for i in range(3))
    do = torch.randn(B, N, H, D, generator=torch.Generator().manual_seed(10)).bfloat16().to(dev).transpose(1, 2)
    gq = torch.ones(D, device=dev, requires_grad=True)
    gk = torch.ones(D, device=dev, requires_grad=True)

    def op_step():
        q.grad = k.grad = v.grad = gq.grad = gk.grad = None
        llsa_amd.llsa_l2(q, k, v, t1, t2, 16, rope=model.freq, qk_norm=(gq, gk, 1e-5)).backward(do)

    ms_op = time_fn(op_step, 5, 20)
    nparams = sum(p.numel() for p in model.parameters())
    attn_flops = 14.0 * B * H * N * D * n_kv("l2", N, t1, t2) * layers
    linear_flops = 6.0 * B * N * (nparams - 12 * (256 * 384 + 384 + 384 * 384 + 384 + 384 * 6 * 384 + 6 * 384))
    print(json.dumps({
        "metric": "pixel DiT-S training step with llsa_l2 in every attention layer, ms per step", "value": ms, "unit": "ms",
        "n_gpus": 1, "steps": args.steps, "warmup": args.warmup, "ms_per_step": ms, "higher_is_better": False,
        "scaling": "weak", "vs_baseline": None, "dtype": "bf16", "data": "synthetic",
        "config": {"workload": f"c4: DiT-S {layers} layers hidden {H * D} heads {H}x{D}, batch {B} of 3x{side}x{side} (N={N} tokens, "
                               f"Z-order), llsa_l2 topk {t1}/{t2}, qk RMS norm + RoPE "
                               + ("composed before the operator" if args.unfused else "inside the operator")
                               + (", norms, linear layers and feed-forward blocks by llsa_amd" if args.fused_layers else "")
                               + ", bf16 autocast, AdamW, grad-norm clip 1.0",
                   "parameters": nparams},
        "images_per_s": B / (ms * 1e-3),
        "operator": {"ms_fwd_bwd_one_layer": ms_op, "ms_all_layers": ms_op * layers, "share_of_step": ms_op * layers / ms,
                     "tflops": attn_flops / layers / (ms_op * 1e-3) / 1e12},
        "algorithmic_tflop_per_step": {"attention": attn_flops / 1e12, "linear_layers": linear_flops / 1e12},
        "loss_first_last": [losses[0], losses[-1]],
    }))


def bench_fwd_sweep(args):
    """The reference's own harness restated (test_kernel.py:27-58): forward only, B=2, H=4, D=64, bf16 N(0,1)
    inputs, default topk 8, N = 128^2, 256^2, 512^2; median and 20 % / 80 % quantiles of the time of one call,
    the L2 flushed before every call as triton.testing.do_bench does.  llsa_l3 is added where N allows it."""
    import torch
    import llsa_amd
    from llsa_amd._lib import get_lib
    get_lib()
    assert torch.cuda.is_available(), "bench.py needs the GPU"
    dev = torch.device("cuda:0")
    B, H, D, topk = 2, 4, 64, 8
    flush = torch.empty(256 << 20, dtype=torch.int8, device=dev)
    rows = []
    for size in (128, 256, 512):
        N = size * size
        g = torch.Generator().manual_seed(size)
        q, k, v = (torch.randn(B, H, N, D, generator=g).bfloat16().to(dev) for _ in range(3))
        ops = {"l1": lambda: llsa_amd.llsa_l1(q, k, v, topk, 16), "l2": lambda: llsa_amd.llsa_l2(q, k, v, topk, topk, 16)}
        if N % 262144 == 0:
            ops["l3"] = lambda: llsa_amd.llsa_l3(q, k, v, topk, topk, topk, 16)
        for name, fn in ops.items():
            with torch.no_grad():
                for _ in range(max(3, args.warmup)):
                    fn()
                times = []
                for _ in range(max(10, args.steps)):
                    flush.zero_()
                    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                    e0.record()
                    fn()
                    e1.record()
                    e1.synchronize()
                    times.append(e0.elapsed_time(e1))
            t = torch.tensor(times)
            rows.append({"op": "llsa_" + name, "size": size, "N": N, "ms_median": t.median().item(),
                         "ms_p20": t.quantile(0.2).item(), "ms_p80": t.quantile(0.8).item()})
    print(json.dumps({
        "metric": "forward-only time of one call, the reference's test_kernel.py harness", "unit": "ms", "n_gpus": 1,
        "steps": max(10, args.steps), "warmup": max(3, args.warmup), "higher_is_better": False, "vs_baseline": None,
        "dtype": "bf16", "data": "synthetic",
        "config": {"workload": f"fwd_sweep: B={B} H={H} D={D} topk={topk} block_size=16, N(0,1) inputs, no RoPE, L2 flushed before every call"},
        "value": next(r["ms_median"] for r in rows if r["op"] == "llsa_l2" and r["size"] == 128), "rows": rows}))


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--warmup", type=int, default=10)
    ap.add_argument("--workload", default="c3", choices=sorted(WORKLOADS) + ["c4", "fwd_sweep"])
    ap.add_argument("--no-extras", action="store_true", help="skip stage profile, CPU baseline and dense SDPA")
    ap.add_argument("--unfused", action="store_true", help="use the reference's composition (separate pools, autograd adds)")
    ap.add_argument("--fused-layers", action="store_true", help="c4: layer norms, linear layers and feed-forward blocks by this package's operators")
    ap.add_argument("--calibrate", action="store_true",
                    help="after the timed region also launch a plain elementwise copy of 256 MiB (fp32, read 256 MiB + "
                         "write 256 MiB) five times, so that a counter profile of this command holds a kernel of known "
                         "HBM traffic to scale FETCH_SIZE / WRITE_SIZE by")
    args = ap.parse_args()
    if args.gpus != 1:
        print("bench.py: this build runs on one GPU only (one MI355X per box); --gpus must be 1", file=sys.stderr)
        sys.exit(2)
    if args.workload == "c4":
        return bench_dit(args)
    if args.workload == "fwd_sweep":
        return bench_fwd_sweep(args)

    import torch
    import llsa_amd
    from llsa_amd._lib import get_lib
    from llsa_amd.build import kernel_sources_digest
    from llsa_amd.utils.rope_table import rope_table
    get_lib()
    assert torch.cuda.is_available(), "bench.py needs the GPU"
    dev = torch.device("cuda:0")
    op, B, H, N, t1, t2, rope = WORKLOADS[args.workload]
    D = 64
    q, k, v, do = make_inputs(B, H, N, D, dev)
    freq = rope_table(math.isqrt(N), dtype=torch.bfloat16).to(dev) if rope else None
    q.requires_grad_(True), k.requires_grad_(True), v.requires_grad_(True)

    def fwd(q_, k_, v_):
        if args.unfused:
            qq, kk = (llsa_amd.my_rope_fn(q_, freq), llsa_amd.my_rope_fn(k_, freq)) if rope else (q_, k_)
            return llsa_amd.llsa_l2_unfused(qq, kk, v_, t1, t2, 16) if op == "l2" else llsa_amd.llsa_l1_unfused(qq, kk, v_, t1, 16)
        if op == "l3":
            return llsa_amd.llsa_l3(q_, k_, v_, t1, t2, t2, 16, rope=freq)
        return llsa_amd.llsa_l2(q_, k_, v_, t1, t2, 16, rope=freq) if op == "l2" else llsa_amd.llsa_l1(q_, k_, v_, t1, 16, rope=freq)

    def eager_step():
        q.grad = k.grad = v.grad = None
        fwd(q, k, v).backward(do)

    def time_steps(step):
        # A cold process gives the GPU a few milliseconds of work before the timed region (W steps of 0.4 ms); its
        # clocks and caches take some tens of milliseconds of load to settle, so the step runs untimed for a quarter
        # of a second first.  The W warm-up steps and the K timed steps follow as asked for.
        t_end = time.perf_counter() + 0.25
        while time.perf_counter() < t_end:
            for _ in range(10):
                step()
            torch.cuda.synchronize()
        for _ in range(args.warmup):
            step()
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for _ in range(args.steps):
            step()
        torch.cuda.synchronize()
        return (time.perf_counter() - t0) * 1e3 / args.steps

    # `value` is the step as a user's training loop issues it: one operator call and its backward, about ten launches.
    ms = time_steps(eager_step)

    def step_quantiles(step, n):
        """Per-step times from HIP events on the launch stream (every step is fenced by two events; the lists that run
        on the second stream are joined back before the step's last kernel): median and 20 % / 80 % quantiles, the
        statistics the reference's harness reports (test_kernel.py:45-51)."""
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(n + 1)]
        ev[0].record()
        for i in range(n):
            step()
            ev[i + 1].record()
        ev[n].synchronize()
        t = torch.tensor([ev[i].elapsed_time(ev[i + 1]) for i in range(n)], dtype=torch.float64)
        return {"n": n, "ms_median": t.median().item(), "ms_p20": t.quantile(0.2).item(), "ms_p80": t.quantile(0.8).item(),
                "ms_mean": t.mean().item()}

    quant = step_quantiles(eager_step, max(50, args.steps))

    if args.calibrate:
        src = torch.ones(64 * 1024 * 1024, device=dev, dtype=torch.float32)
        dst = torch.empty_like(src)
        for _ in range(5):
            torch.mul(src, 1.0, out=dst)
        torch.cuda.synchronize()
        del src, dst

    nkv = n_kv(op, N, t1, t2)
    unit_flops = B * H * N * D * nkv                    # one "GEMM unit": 2 * this = one product
    flops = 14.0 * unit_flops
    out = {
        "metric": f"llsa_{op} fwd+bwd effective TFLOP/s at N={N}, D={D}, bf16",
        "value": flops / (ms * 1e-3) / 1e12, "unit": "TFLOP/s", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup,
        "ms_per_step": ms, "higher_is_better": True, "scaling": "weak", "vs_baseline": None, "dtype": "bf16",
        "data": "synthetic",
        "config": {"workload": f"{args.workload}: llsa_{op} fwd+bwd B={B} H={H} N={N} D={D} block_size=16 topk={t1}"
                               + (f"/{t2}" if op == "l2" else f"/{t2}/{t2}" if op == "l3" else "") + (" rope=in-kernel" if rope else "")
                               + (" (unfused composition)" if args.unfused else ""),
                   "n_kv_per_query": nkv, "algorithmic_gflop": flops / 1e9},
        "frac_of_bf16_mfma_peak": flops / (ms * 1e-3) / 1e12 / PEAK_BF16_TFLOPS,
        "step_event_times": quant, "kernel_sources": kernel_sources_digest(),
    }

    if not args.no_extras and op != "l3":      # (the stage profile and the CPU baseline know one and two levels)
        prof_iters = max(5, min(args.steps, 20))
        with torch.no_grad():
            st = stage_profile(op, q.detach(), k.detach(), v.detach(), do, t1, t2, freq, prof_iters, torch)
        alg = {"attn_fwd": 4.0 * unit_flops, "bwd_dq": 6.0 * unit_flops, "bwd_dkv": 4.0 * B * H * N * D * 16 * t1}
        n_dense = N // 256 if op == "l2" else N // 16
        if op == "l2":
            merged = "bwd_dpkv_dense" not in st
            alg["bwd_pooled_groups"] = 4.0 * B * H * N * D * (16 * t2 + (n_dense if merged else 0))
        if "bwd_dpkv_dense" in st:
            alg["bwd_dpkv_dense"] = 4.0 * B * H * N * D * n_dense
        # algorithmic bytes of the bandwidth-bound kernels: inputs read once, results written once (bf16 = 2 B, indices 4 B)
        el = 2 * B * H * N * D
        BH, n1, n2 = B * H, N // 16, N // 256
        hbm = {"pool_pyramid": 3 * el * (1 + 1 / 16 + (1 / 256 if op == "l2" else 0))}
        # (the pooling kernel also writes the operand tiles the attention kernels read; those bytes
        # are layout work of this implementation and are not counted as algorithmic)
        if op == "l2":
            hbm["topk_dense"] = BH * (2 * n2 * D * 2 + n2 * t2 * 4)
            hbm["topk_sparse"] = BH * (2 * n1 * D * 2 + n2 * t2 * 4 + n1 * t1 * 4)
            hbm["topk_cascade"] = hbm["topk_dense"] + hbm["topk_sparse"]      # (both selections in one launch)
            hbm["transpose_indices"] = BH * ((n1 * t1 * 4) * 2 + (n1 + 1) * 4 + (n2 * t2 * 4) * 3 + (n2 + 1) * 4)
        else:
            hbm["topk_dense"] = BH * (2 * n1 * D * 2 + n1 * t1 * 4)
            hbm["transpose_indices"] = BH * ((n1 * t1 * 4) * 2 + (n1 + 1) * 4)
        traffic, traffic_src = measured_traffic(args.workload)
        kernels = {}
        for name, t in st.items():
            e = {"ms": t}
            if name in alg:
                e["tflops"] = alg[name] / (t * 1e-3) / 1e12
                e["frac_mfma_peak"] = e["tflops"] / PEAK_BF16_TFLOPS
            if name in hbm:
                e["algorithmic_mb"] = hbm[name] / 1e6
                e["gbs"] = hbm[name] / (t * 1e-3) / 1e9
                e["frac_hbm_peak"] = e["gbs"] / PEAK_HBM_GBS
            if name in traffic:
                e["hbm_traffic_mb"] = traffic[name] / 1e6
            kernels[name] = e
        out["kernels"] = kernels
        out["stage_sum_ms"] = sum(t for n_, t in st.items() if n_ != "bwd_kside_all_with_reductions")
        dom = max(alg, key=lambda n: st[n])
        out["roofline"] = {"kernel": dom, "bound": "mfma", "achieved": kernels[dom]["tflops"], "peak": PEAK_BF16_TFLOPS,
                           "unit": "TFLOP/s", "frac": kernels[dom]["frac_mfma_peak"],
                           "traffic": traffic.get(dom), "traffic_source": traffic_src,
                           "avg_launch_ms": st[dom], "algorithmic_gflop_per_launch": alg[dom] / 1e9}
        out["roofline_hbm"] = {"kernel": "pool_pyramid (the q, k, v launch)", "bound": "hbm", "achieved": kernels["pool_pyramid"]["gbs"],
                               "peak": PEAK_HBM_GBS, "unit": "GB/s", "frac": kernels["pool_pyramid"]["frac_hbm_peak"],
                               "traffic": traffic.get("pool_pyramid"), "traffic_source": traffic_src}
        # dense attention on the same GPU
        try:
            import torch.nn.functional as F
            qd, kd, vd = (t.detach().clone().requires_grad_(True) for t in (q, k, v))

            def dense():
                qd.grad = kd.grad = vd.grad = None
                F.scaled_dot_product_attention(qd, kd, vd).backward(do)

            for _ in range(2):
                dense()
            torch.cuda.synchronize()
            n_d = 3 if N > 16384 else 10
            t_d = timed(dense, n_d, torch)
            out["dense_sdpa"] = {"ms_per_step": t_d, "speedup_llsa_over_dense": t_d / ms,
                                 "dense_tflops": 14.0 * B * H * N * D * N / (t_d * 1e-3) / 1e12}
        except Exception as e:                      # dense attention may not fit at the largest sizes
            out["dense_sdpa"] = {"error": str(e)[:200]}
        if args.workload == "c3":
            del qd, kd, vd
            out["other_workloads"] = other_workloads(dev)
        out["cpu_baseline"] = cpu_baseline(op, B, H, N, D, t1, t2, rope)
    print(json.dumps(out))


if __name__ == "__main__":
    main()
