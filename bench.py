#!/usr/bin/env python
"""bench.py -- the poly-attention hot path on one MI355X.

Workload: order-2 causal poly attention, B=4, N=4096, heads=16,
dim_head=64, bf16.  The inputs of the timed op are the module's own q1/q2/q3/v3: a
PolyAttention(dim=1024, heads=16, dim_head=64, causal=True) with random-init bf16 weights
(seed 0) applied to x ~ N(0,1) [4, 4096, 1024] (seed 1), i.e. the projections and q/k
RMSNorms of the reference module.  One step = the fused core forward (both passes) +
backward (all four input gradients) for upstream grad ~ N(0,1) (seed 2).

Printed: ONE JSON line with the headline metric (core TFLOP/s over the algorithmic flops of
the step), the live per-kernel roofline of the dominant kernel (HIP events on its launch
stream), the CPU oracle baseline timed on this host, the full module step time, and, as
extra fields, the other GPU configs of BASELINE.json: config 5 (GQA decode step, GB/s
against 8 TB/s), config 3 (PolyViT forward, images/s and the attention core's share) and
config 4 (order-3 causal decode loop through a PolyLM-style stack, tokens/s).

    python bench.py [--gpus 1] [--steps K] [--warmup W] [--no-cpu] [--no-decode]
                    [--no-module] [--no-vit] [--no-lm]
"""

from __future__ import annotations

import argparse
import json
import os
import re
import platform
import subprocess
import sys
import time

ROOT = os.path.dirname(os.path.abspath(__file__))
for _p in (os.path.join(ROOT, "poly-attention_amd"), ROOT):
    if _p not in sys.path:
        sys.path.insert(0, _p)

import torch  # noqa: E402

METRIC = "poly-attn fwd+bwd TFLOP/s (%MFMA peak) N=4096 h16 d64 bf16; decode GB/s"
PEAK_BF16_TFLOPS = 2500.0   # MI355X dense bf16 MFMA (published)
PEAK_FP32_TFLOPS = 157.3    # MI355X fp32 (published)
PEAK_HBM_GBS = 8000.0       # MI355X HBM3E (published)

B, N, DIM, H, DH = 4, 4096, 1024, 16, 64


def log(*a):
    print(*a, file=sys.stderr, flush=True)


# ---------------------------------------------------------------------------------------
# algorithmic work


def core_flops_fwd(b, h, nq, nk, d, causal):
    """4 * Nq * Nk * d per (batch, head) and attention level; causal x 1/2."""
    return 4.0 * nq * nk * d * b * h * (0.5 if causal else 1.0)


def step_flops():
    # two levels (pass 1 at kv_heads = 16, pass 2 at 16 heads), forward 4 N^2 d, backward 10 N^2 d
    fwd = 2 * core_flops_fwd(B, H, N, N, DH, True)
    return fwd, fwd * 10.0 / 4.0


# per kernel family: (bound, peak, work per launch for this workload, unit)
def kernel_work(name):
    per_level_fwd = core_flops_fwd(B, H, N, N, DH, True)
    table = {
        "mfma_fwd": ("mfma", PEAK_BF16_TFLOPS, per_level_fwd, "TFLOP/s"),
        # dK/dV kernel: S, dP, dV, dK = 4 GEMMs; dQ kernel: S, dP, dQ = 3 GEMMs
        "mfma_bwd_dkv": ("mfma", PEAK_BF16_TFLOPS, per_level_fwd * 2.0, "TFLOP/s"),
        "mfma_bwd_dq": ("mfma", PEAK_BF16_TFLOPS, per_level_fwd * 1.5, "TFLOP/s"),
        "simt_bwd_dkv": ("mfma", PEAK_FP32_TFLOPS, per_level_fwd * 2.0, "TFLOP/s"),
        "simt_bwd_dq": ("mfma", PEAK_FP32_TFLOPS, per_level_fwd * 1.5, "TFLOP/s"),
        # preprocess: reads O and dO (bf16) and lse, writes three fp32 rows (bytes)
        "bwd_pre": ("hbm", PEAK_HBM_GBS, B * H * N * (2 * DH * 2 + 4 + 12), "GB/s"),
    }
    return table.get(name)


TRAFFIC_PROFILE = os.path.join(ROOT, "profiles", "pmc_hbm_traffic_config2_config5.md")


def measured_traffic(family):
    """HBM bytes per launch of a kernel family from the committed rocprofv3 FETCH_SIZE /
    WRITE_SIZE summary (calibrated against a plain copy in the same runs), or None."""
    try:
        with open(TRAFFIC_PROFILE) as f:
            for line in f:
                cells = [c.strip() for c in line.strip().strip("|").split("|")]
                if len(cells) == 7 and cells[0] == family:
                    return int(float(cells[6]))
    except OSError:
        pass
    return None


KERNEL_PROFILE = os.path.join(ROOT, "profiles", "bench_config2_and_decode_kernel_stats.md")


def rocprof_avg_ms(family):
    """The average launch duration of a kernel family in the committed rocprofv3 --stats
    summary of this workload (calls-weighted over its instantiations), or None."""
    calls = total = 0.0
    try:
        with open(KERNEL_PROFILE) as f:
            for line in f:
                cells = [c.strip().strip("`") for c in line.strip().strip("|").split("|")]
                # mangled names: _ZN2pa<len>k_<family>[_dma]I<template arguments>
                m = re.match(r"_ZN2pa\d+k_(\w+?)(_dma)?I", cells[0]) if len(cells) == 6 else None
                if m and m.group(1) == family:
                    calls += float(cells[1])
                    total += float(cells[1]) * float(cells[2])
    except (OSError, ValueError):
        return None
    return total / calls / 1e3 if calls else None


def achieved_rate(work, avg_ms, unit):
    return work / (avg_ms / 1e3) / (1e12 if unit == "TFLOP/s" else 1e9)


# ---------------------------------------------------------------------------------------
# config 2: fused fwd + bwd


def make_config2(dev):
    from poly_attention import PolyAttention

    torch.manual_seed(0)
    m = PolyAttention(dim=DIM, heads=H, dim_head=DH, causal=True).to(dev, torch.bfloat16)
    g = torch.Generator(device="cpu").manual_seed(1)
    x = torch.randn(B, N, DIM, generator=g).to(dev, torch.bfloat16)
    with torch.no_grad():
        q1 = m.split_q(m.to_q(x))[0]
        q2 = m.split_kv1(m.to_kvs[0](x))[0]
        q3, v3 = m.split_kv(m.to_kvs[1](x))
        q1, q2, q3 = (norm(q) for norm, q in zip(m.q_norms, (q1, q2, q3)))
    qs = [t.contiguous().requires_grad_() for t in (q1, q2, q3, v3)]
    g2 = torch.Generator(device="cpu").manual_seed(2)
    dout = torch.randn(B, H, N, DH, generator=g2).to(dev, torch.bfloat16)
    dx = torch.randn(B, N, DIM, generator=g2).to(dev, torch.bfloat16)
    return m, x, qs, dout, dx


def core_step(qs, dout):
    from poly_attention.flash_poly_attention import flash_poly_attention

    for t in qs:
        t.grad = None
    out = flash_poly_attention(*qs, is_causal=True)
    out.backward(dout)


def module_step(m, x, dx):
    m.zero_grad(set_to_none=True)
    xr = x.detach().requires_grad_()
    out = m(xr)
    out.backward(dx)


def masked_core_bench(qs, dout, steps, warmup):
    """Config 2's core step with the op's mask (a key mask of both passes,
    flash_poly_attention.py:109-112 of the reference) as padding: batch rows keep N, 7N/8, 3N/4
    and N/2 keys.  right_pad masks the trailing keys; left_pad the leading ones, so the first
    causal rows of the padded batch rows are fully masked in both passes (the backward's
    fix-up path).  Same nominal work as the unmasked step."""
    from poly_attention import _lib
    from poly_attention.flash_poly_attention import flash_poly_attention

    lengths = (N, N - N // 8, N - N // 4, N // 2)
    masks = {"right_pad": torch.ones(B, N, dtype=torch.bool),
             "left_pad": torch.ones(B, N, dtype=torch.bool)}
    for b, keep in enumerate(lengths):
        masks["right_pad"][b, keep:] = False
        masks["left_pad"][b, :N - keep] = False
    res = {"kept_keys_per_batch_row": list(lengths)}
    for name, mask in masks.items():
        mk = mask.to(dout.device)

        def step():
            for t in qs:
                t.grad = None
            out = flash_poly_attention(*qs, mask=mk, is_causal=True)
            out.backward(dout)

        ms = time_steps(step, steps, warmup)
        with _lib.KernelProfile() as prof:
            for _ in range(3):
                step()
        res[name] = {"ms_per_step": round(ms, 4),
                     "kernels": {k: {"launches_per_step": n // 3, "avg_ms": round(t / n, 4)}
                                 for k, (n, t) in prof.times.items()}}
    return res


def time_steps(fn, steps, warmup):
    for _ in range(warmup):
        fn()
    torch.cuda.synchronize()
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(steps):
        fn()
    stop.record()
    torch.cuda.synchronize()
    return start.elapsed_time(stop) / steps


# ---------------------------------------------------------------------------------------
# config 5: GQA decode step


def decode_bench(dev, steps, warmup):
    from poly_attention import _lib, _ops

    Bd, Hq, G, n_old, d = 32, 32, 8, 8192, 128
    n = n_old + 1
    g = torch.Generator(device="cpu").manual_seed(3)

    def rnd(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float32).to(dev, torch.bfloat16)

    q2c, q3c, v3c = rnd(Bd, G, n, d), rnd(Bd, G, n, d), rnd(Bd, G, n, d)
    msg = rnd(Bd, Hq, n, d)
    lse = (torch.log(torch.arange(1, n + 1, dtype=torch.float32))
           + torch.randn(Bd, Hq, n, generator=g)).to(dev)
    q1 = rnd(Bd, Hq, 1, d)
    q2n = q2c[:, :, -1:].contiguous()

    def step():
        _ops.poly_decode_step([q1, q2n], [q2c, q3c], [v3c], [msg], [lse], kv_heads=G, heads=Hq,
                              softclamp=None, scale=d ** -0.5)

    ms = time_steps(step, steps, warmup)
    # every cached tensor read once in its stored dtype (order 2: q2, q3, v3 at kv heads;
    # msg (bf16) and lse (fp32) at query heads)
    bytes_step = Bd * n * ((2 * 2 - 1) * G * d * 2 + (2 - 1) * Hq * (d * 2 + 4))
    with _lib.KernelProfile() as prof:
        for _ in range(steps):
            step()
    part = prof.times.get("dec_partial", (0, 0.0))
    part_bytes = Bd * n_old * (3 * G * d * 2 + Hq * (d * 2 + 4))
    part_ms = part[1] / max(part[0], 1)
    del q2c, q3c, v3c, msg, lse
    torch.cuda.empty_cache()
    return {
        "workload": "order-2 GQA decode step, Hq=32 Hkv=8 d=128 B=32, 8192 cached + 1 new, bf16 cache, fp32 lse",
        "ms_per_step": round(ms, 4),
        "GB_per_s": round(bytes_step / ms / 1e6, 1),
        "frac_hbm_peak": round(bytes_step / ms / 1e6 / PEAK_HBM_GBS, 4),
        "bytes_per_step": bytes_step,
        "tokens_per_s": round(Bd / (ms / 1e3), 1),
        "kernel": {"name": "dec_partial", "avg_ms": round(part_ms, 4),
                   "GB_per_s": round(part_bytes / part_ms / 1e6, 1) if part_ms else None,
                   "algorithmic_bytes": part_bytes, "traffic": measured_traffic("dec_partial")},
    }


# ---------------------------------------------------------------------------------------
# config 3: PolyViT forward (poly_vit.py:56-95 with BASELINE configs[2]'s sizes)


def _linear_flops(model, run):
    """2 * rows * in * out summed over every nn.Linear call made by ``run()``."""
    total = [0]

    def hook(mod, inp, out):
        total[0] += 2 * (inp[0].numel() // mod.in_features) * mod.in_features * mod.out_features

    hs = [mod.register_forward_hook(hook) for mod in model.modules()
          if isinstance(mod, torch.nn.Linear)]
    try:
        run()
    finally:
        for h in hs:
            h.remove()
    return total[0]


def make_vit(dev, dtype, batch):
    from poly_attention import PolyViT

    torch.manual_seed(0)
    m = PolyViT(image_size=256, patch_size=32, num_classes=1000, dim=1024, depth=6, heads=16,
                mlp_dim=2048, order=2).to(dev, dtype).eval()
    g = torch.Generator(device="cpu").manual_seed(1)
    img = torch.randn(batch, 3, 256, 256, generator=g).to(dev, dtype)
    return m, img


def config1_bench(dev, steps, warmup, cpu):
    """PolyAttention(dim=512, heads=8, dim_head=64, causal=False) fp32
    forward on x ~ N(0,1) (1, 1024, 512), random init (seed 0) -- the reference's
    CPU-runnable case.  GPU: the module forward (fp32 passes on v_mfma_f32_32x32x2_f32), and
    a training step of the same module with a key padding mask; CPU: the oracle's eager module
    forward (the reference's CPU path restated) at the same shape, median of 5."""
    from poly_attention import PolyAttention, _lib

    torch.manual_seed(0)
    m = PolyAttention(dim=512, heads=8, dim_head=64, causal=False)
    params = {k: v.detach().clone() for k, v in m.state_dict().items()}
    x = torch.randn(1, 1024, 512, generator=torch.Generator().manual_seed(1))
    md, xd = m.to(dev), x.to(dev)
    with torch.no_grad():
        ms = time_steps(lambda: md(xd), steps, warmup)
        with _lib.KernelProfile() as prof:
            for _ in range(5):
                md(xd)
    # the fp32 pass: the key-split kernel at this grid (the plain one on other shapes)
    n_l, tot = prof.times.get("mfma_fwd_f32_split", prof.times.get("mfma_fwd_f32", (0, 0.0)))
    core_flops = 2 * core_flops_fwd(1, 8, 1024, 1024, 64, False)  # two passes per forward
    res = {"workload": "PolyAttention(512, h8, d64, non-causal) fp32 forward, x (1, 1024, 512)",
           "ms_per_forward": round(ms, 4),
           "pass_kernel_avg_ms": round(tot / n_l, 4) if n_l else None,
           "core_gflop_per_forward": round(core_flops / 1e9, 3)}
    if n_l:
        tf = core_flops / 2 / (tot / n_l / 1e3) / 1e12
        res["pass_tflops"] = round(tf, 2)
        res["pass_frac_fp32_peak"] = round(tf / PEAK_FP32_TFLOPS, 4)
    # the same module trained in fp32 with a key padding mask (the last quarter of the keys
    # masked): masked passes on the fp32 MFMA kernels, forward and backward (the key term and
    # the fully-masked-row fix-ups around them)
    mask = torch.ones(1, 1024, dtype=torch.bool, device=dev)
    mask[:, 768:] = False
    xg = xd.clone().requires_grad_()
    gy = torch.randn(1, 1024, 512, generator=torch.Generator().manual_seed(2)).to(dev)

    def masked_step():
        xg.grad = None
        md.zero_grad(set_to_none=True)
        md(xg, mask=mask).backward(gy)

    res["masked_train_ms_per_step"] = round(time_steps(masked_step, steps, warmup), 4)
    with _lib.KernelProfile() as mprof:
        for _ in range(3):
            masked_step()
    res["masked_train_kernels"] = {k: {"launches_per_step": n // 3, "avg_ms": round(t / n, 4)}
                                   for k, (n, t) in mprof.times.items()}
    if cpu:
        import oracle.poly_oracle as O

        torch.set_num_threads(cpu_threads()[0])
        cfg = dict(heads=8, dim_head=64, causal=False)
        with torch.no_grad():
            O.order2_forward(params, cfg, x)
            t = []
            for _ in range(5):
                t0 = time.perf_counter()
                O.order2_forward(params, cfg, x)
                t.append((time.perf_counter() - t0) * 1e3)
        # this config's CPU baseline: the oracle's restatement of the reference's CPU path
        res["cpu_baseline"] = {"ms_per_forward": round(sorted(t)[len(t) // 2], 3),
                               "kind": "port", "cores": torch.get_num_threads()}
    return res


def vit_bench(dev, steps, warmup, cpu):
    """Config 3 forward, eagerly (one Python call per step; at batch 64 the host issues the
    launches no faster than the GPU runs them) and replayed from a HIP graph captured once
    (fixed shapes: the inference deployment), checked equal to the eager output."""
    batch = 64
    m, img = make_vit(dev, torch.bfloat16, batch)
    with torch.no_grad():
        proj_flops = _linear_flops(m, lambda: m(img))
        eager_ms = time_steps(lambda: m(img), steps, warmup)
        ref = m(img)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                m(img)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(img)
        graph.replay()
        torch.cuda.synchronize()
        graph_diff = (out.float() - ref.float()).abs().max().item()
        assert graph_diff <= 2e-2 * max(1.0, ref.float().abs().max().item()), \
            f"graph replay differs from the eager forward by {graph_diff}"
        ms = time_steps(graph.replay, steps, warmup)
        with _lib().KernelProfile() as prof:
            for _ in range(steps):
                m(img)
    npatch = (256 // 32) ** 2
    core_flops = 6 * 2 * core_flops_fwd(batch, 16, npatch, npatch, 64, False)
    core_ms = sum(t for _, t in prof.times.values()) / steps
    res = {
        "workload": "PolyViT fwd (image 256, patch 32, dim 1024, depth 6, heads 16, mlp 2048, "
                    "order 2, 1000 classes), batch 64 bf16, inference (BASELINE configs[2])",
        "ms_per_step": round(ms, 4),
        "images_per_s": round(batch / (ms / 1e3), 1),
        "mode": "forward captured once into a HIP graph, replayed per step",
        "eager_ms_per_step": round(eager_ms, 4),
        "eager_images_per_s": round(batch / (eager_ms / 1e3), 1),
        "graph_vs_eager_max_abs_diff": graph_diff,
        "flops_per_step": proj_flops + core_flops,
        "TFLOP_per_s": round((proj_flops + core_flops) / (ms / 1e3) / 1e12, 2),
        "core_flops_per_step": core_flops,
        "core_ms_per_step": round(core_ms, 4),
        "core_share_of_time": round(core_ms / ms, 4),
        "kernels": {k: {"launches": n // steps, "avg_ms": round(t / n, 4)}
                    for k, (n, t) in prof.times.items()},
    }
    del m, img, graph, out, ref
    torch.cuda.empty_cache()
    if cpu:
        threads = cpu_threads()[0]
        torch.set_num_threads(threads)
        cb = 8
        mc, imgc = make_vit(torch.device("cpu"), torch.float32, cb)
        with torch.no_grad():
            mc(imgc)
            times = []
            for _ in range(3):
                t0 = time.perf_counter()
                mc(imgc)
                times.append(time.perf_counter() - t0)
        med = sorted(times)[1]
        res["cpu_baseline"] = {
            "value": round(cb / med, 2), "unit": "images/s", "cores": threads, "kind": "port",
            "sample": f"the same PolyViT in fp32 on this host (eager attention, the reference's "
                      f"CPU path), batch {cb}, median of 3 after 1 warm-up, {med * 1e3:.0f} ms each"}
    return res


# ---------------------------------------------------------------------------------------
# config 4: order-3 causal decode with the KV cache, through a PolyLM-style stack
# (train_enwik8.py:112-177: token embedding, external RoPE, [RMSNorm -> NPolyAttention ->
# residual, RMSNorm -> FeedForward -> residual] x depth, RMSNorm, logits)


class _Block(torch.nn.Module):
    """train_enwik8.py:112-127 with order 3 (NPolyAttention) and x-transformers' default
    FeedForward(dim): Linear(dim, 4 dim) -> GELU -> Linear(4 dim, dim)."""

    def __init__(self, dim, heads, dim_head, order):
        super().__init__()
        from poly_attention import NPolyAttention

        self.attn = NPolyAttention(dim, order=order, heads=heads, dim_head=dim_head, causal=True)
        self.norm1 = torch.nn.RMSNorm(dim)
        self.norm2 = torch.nn.RMSNorm(dim)
        self.ffn = torch.nn.Sequential(torch.nn.Linear(dim, 4 * dim), torch.nn.GELU(),
                                       torch.nn.Linear(4 * dim, dim))

    def forward(self, x, rotary_pos_emb=None, cache=None, parents=None):
        attn_out, new_cache = self.attn(self.norm1(x), rotary_pos_emb=rotary_pos_emb,
                                        cache=cache, return_cache=True, parents=parents)
        if x.is_cuda:
            # decode-sized inputs: the residual add, the norm, the GELU and the second residual
            # add ride in the projections' launches (pa_linear_small), rounded as the separate
            # ops; larger ones take the same torch ops
            from poly_attention import _ops

            h, x = _ops.linear(self.ffn[0], x, x_add=attn_out, norm=self.norm2, gelu=True,
                               return_sum=True)
            return _ops.linear(self.ffn[2], h, residual=x), new_cache
        x = x + attn_out
        return x + self.ffn(self.norm2(x)), new_cache


class _PolyLM(torch.nn.Module):
    """train_enwik8.py:129-177 (inference branch)."""

    def __init__(self, num_tokens=256, dim=1024, depth=8, heads=16, dim_head=64, order=3):
        super().__init__()
        from poly_attention.rotary import RotaryEmbedding

        self.token_emb = torch.nn.Embedding(num_tokens, dim)
        self.rotary_emb = RotaryEmbedding(dim_head)
        self.layers = torch.nn.ModuleList([_Block(dim, heads, dim_head, order)
                                           for _ in range(depth)])
        self.norm = torch.nn.RMSNorm(dim)
        self.to_logits = torch.nn.Linear(dim, num_tokens, bias=False)

    def forward(self, x, cache=None, pos=None, parents=None):
        """``pos``: the positions as a device tensor (a captured step has no host count);
        ``parents``: the tree of a drafted step's tokens (DraftCaches)."""
        seq_len = x.shape[1]
        past = 0 if cache is None else cache[1]
        layer_caches = [None] * len(self.layers) if cache is None else cache[0]
        if pos is None:
            pos = torch.arange(seq_len, device=x.device) + past
        rot = self.rotary_emb(pos)
        x = self.token_emb(x)
        new = []
        for layer, lc in zip(self.layers, layer_caches):
            x, nc = layer(x, rotary_pos_emb=rot, cache=lc, parents=parents)
            new.append(nc)
        if x.is_cuda:
            from poly_attention import _ops

            logits = _ops.linear(self.to_logits, x, norm=self.norm)
        else:
            logits = self.to_logits(self.norm(x))
        return logits, (new, None if past is None else past + seq_len)


def _greedy(lm, prompt, steps):
    """Prefill ``prompt`` with return_cache, then ``steps`` greedy single-token steps
    (train_enwik8.py:85-108 with argmax in place of the gumbel top-k sample)."""
    logits, cache = lm(prompt)
    tok = logits[:, -1].argmax(-1, keepdim=True)
    out = [tok]
    for _ in range(steps - 1):
        logits, cache = lm(tok, cache)
        tok = logits[:, -1].argmax(-1, keepdim=True)
        out.append(tok)
    return torch.cat(out, dim=1)


def _flip_margins(logits, tok_eager, tok_graph):
    """At the first step where the eager and the graph paths pick different greedy tokens: per
    differing batch row, the eager logits' top-2 margin, their gap between the two picked
    tokens, and that gap in units of one bf16 rounding of the logit (2^-8 |logit|)."""
    rows = (tok_eager != tok_graph).nonzero().flatten().tolist()
    out = []
    for r in rows:
        lg = logits[r].float()
        top = lg.topk(2).values
        te, tg = int(tok_eager[r]), int(tok_graph[r])
        gap = float(lg[te] - lg[tg])
        out.append({"row": r, "eager_token": te, "graph_token": tg,
                    "eager_top2_margin": round(float(top[0] - top[1]), 6),
                    "eager_gap_between_picks": round(gap, 6),
                    "gap_in_bf16_roundings": round(gap / (2.0 ** -8 * float(lg[te].abs())), 3)})
    return out


def make_lm(dev, depth=8, heads=16, dh=64, dim=1024, batch=8, prefill=2048):
    """Config 4's stack (random-init bf16 weights, seed 0) and its uniform random prompt."""
    torch.manual_seed(0)
    lm = _PolyLM(dim=dim, depth=depth, heads=heads, dim_head=dh).to(dev, torch.bfloat16).eval()
    g = torch.Generator(device="cpu").manual_seed(1)
    prompt = torch.randint(0, 256, (batch, prefill), generator=g).to(dev)
    return lm, prompt


def decode_two_ways(lm, prompt, steps, warm=2, eager=True, more=16, profile=True):
    """The config-4 decode two ways: (1) the reference's calling pattern, one eager module call
    per token with the growing cache tuples (skipped with ``eager=False``); (2) the same steps
    on StaticCaches, one decode step (all layers, logits, argmax) captured into a HIP graph and
    replayed per token.  Returns the tokens of both (the prefill's pick first), the eager
    logits behind each token, the wall times and (``profile``) the per-launch kernel times of
    ``more`` further eager StaticCache steps."""
    from poly_attention import StaticCache

    dev = prompt.device
    batch, prefill = prompt.shape
    out = {}
    with torch.no_grad():
        _greedy(lm, prompt[:, :256], 8)  # warm-up (allocator, kernels)
        torch.cuda.synchronize()
        # (1) eager steps, tuple caches
        t0 = time.perf_counter()
        logits, cache = lm(prompt)
        tok = logits[:, -1].argmax(-1, keepdim=True)
        torch.cuda.synchronize()
        t1 = time.perf_counter()
        toks_eager = [tok]
        logits_eager = [logits[:, -1]]  # the logits behind each greedy token (device)
        for _ in range(steps if eager else 0):
            logits, cache = lm(tok, cache)
            tok = logits[:, -1].argmax(-1, keepdim=True)
            toks_eager.append(tok)
            logits_eager.append(logits[:, -1])
        torch.cuda.synchronize()
        t2 = time.perf_counter()
        out["toks_eager"] = torch.cat(toks_eager, dim=1)
        out["logits_eager"] = logits_eager
        del cache, logits
        # (2) StaticCache + one captured step per token
        logits, (lcs, _) = lm(prompt)
        tok = logits[:, -1].argmax(-1, keepdim=True)
        # one step counter shared by the layers' caches, advanced once per token
        counter = StaticCache.make_counter(lcs[0])
        scs = [StaticCache(c, capacity=prefill + steps + more + 1, counter=counter) for c in lcs]
        del lcs, logits
        tok_buf = tok.clone()
        pos_buf = torch.full((1,), prefill, dtype=torch.int64, device=dev)
        rec = torch.zeros(batch, steps + more + 1, dtype=torch.int64, device=dev)
        rec[:, :1] = tok

        def step():
            lg, _ = lm(tok_buf, (scs, None), pos=pos_buf)
            nxt = lg[:, -1].argmax(-1, keepdim=True)
            tok_buf.copy_(nxt)
            StaticCache.advance_counter(counter)
            pos_buf.add_(1)
            rec.index_copy_(1, pos_buf - prefill, nxt)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(warm):  # real decode steps, run eagerly before the capture
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        torch.cuda.synchronize()
        t3 = time.perf_counter()
        for _ in range(steps - warm):
            graph.replay()
        torch.cuda.synchronize()
        t4 = time.perf_counter()
        assert scs[0].seq_len() == prefill + steps
        scs[0].check_overflow()
        out["toks_graph"] = rec[:, :steps + 1].clone()
        out["times"] = (t0, t1, t2, t3, t4)
        if profile:
            # kernel times of a few more steps (events per launch, eager steps: host gaps count)
            with _lib().KernelProfile() as prof:
                for _ in range(more):
                    step()
                torch.cuda.synchronize()
            out["prof"] = prof
        del scs, graph
    return out


def decode_order3_bench(dev, cpu, steps=512, prefill=2048, batch=8, warm=2, eager=True):
    """Config 4 timed two ways (``decode_two_ways``); the graph replays are the figure."""
    depth, heads, dh, dim = 8, 16, 64, 1024
    more = 16
    lm, prompt = make_lm(dev, depth, heads, dh, dim, batch, prefill)
    runs = decode_two_ways(lm, prompt, steps, warm, eager, more)
    t0, t1, t2, t3, t4 = runs["times"]
    prof = runs["prof"]
    # greedy tokens of random-init weights sit on near-ties: a last-bit difference
    # (summation order of the split-K chunks, fused vs separate roundings) can flip one
    # argmax, after which the sequences diverge; report where the first flip happens and the
    # eager logits' margins there
    first_flip = None
    flip = None
    if eager:
        toks_eager, rec = runs["toks_eager"], runs["toks_graph"]
        diff = (rec != toks_eager).any(dim=0).nonzero()
        first_flip = int(diff[0].item()) if diff.numel() else steps + 1
        if first_flip <= steps:
            flip = _flip_margins(runs["logits_eager"][first_flip], toks_eager[:, first_flip],
                                 rec[:, first_flip])
    eager_s, graph_s = t2 - t1, t4 - t3
    graph_steps = steps - warm
    # cache bytes per step and layer (order 3, kv heads = heads): every cached tensor read
    # once -- (2*order-1) q/v tensors (bf16) + (order-1) msg (bf16) and lse (fp32)
    per_tok = (2 * 3 - 1) * heads * dh * 2 + (3 - 1) * heads * (dh * 2 + 4)
    weight_bytes = 2 * sum(p.numel() for n, p in lm.named_parameters()
                           if not n.startswith("token_emb") and not n.endswith("freqs"))

    def step_bytes(s):  # decode step s (0-based) attends over prefill + s + 1 positions
        return batch * depth * per_tok * (prefill + s + 1) + weight_bytes

    eager_bytes = sum(step_bytes(s) for s in range(steps))
    graph_bytes = sum(step_bytes(s) for s in range(warm, steps))
    kern = {k: {"launches": n // more, "avg_ms": round(t / n, 4)}
            for k, (n, t) in prof.times.items()}
    res = {
        "workload": f"order-3 causal decode, PolyLM-style stack depth {depth}, dim {dim}, heads "
                    f"{heads}, dim_head {dh}, batch {batch}, prefill {prefill} tokens, {steps} "
                    f"greedy steps, bf16 weights and cache, fp32 lse (BASELINE configs[3])",
        "prefill_ms": round((t1 - t0) * 1e3, 2),
        "ms_per_step": round(graph_s * 1e3 / graph_steps, 4),
        "tokens_per_s": round(batch * graph_steps / graph_s, 1),
        "GB_per_s": round(graph_bytes / graph_s / 1e9, 1),
        "frac_hbm_peak": round(graph_bytes / graph_s / 1e9 / PEAK_HBM_GBS, 4),
        "mode": f"StaticCache + one HIP graph per token ({warm} eager warm-up steps, "
                f"{graph_steps} replays timed)",
        "eager_tuple_cache": None if not eager else {
            "ms_per_step": round(eager_s * 1e3 / steps, 4),
            "tokens_per_s": round(batch * steps / eager_s, 1),
            "GB_per_s": round(eager_bytes / eager_s / 1e9, 1)},
        "greedy_tokens_identical_to_eager_until": first_flip,
        "first_flip": flip,
        "cache_GB_per_step_mean": round((eager_bytes - steps * weight_bytes) / steps / 1e9, 4),
        "weight_GB_per_step": round(weight_bytes / 1e9, 4),
        "kernels_timer": "HIP events around each launch over 16 eager StaticCache steps "
                         "(host gaps between launches count; rocprofv3 kernel traces in "
                         "profiles/ give the kernels' own durations)",
        "kernels": kern,
    }
    del lm, runs
    torch.cuda.empty_cache()
    if cpu:
        threads = cpu_threads()[0]
        torch.set_num_threads(threads)
        torch.manual_seed(0)
        lmc = _PolyLM(dim=dim, depth=depth, heads=heads, dim_head=dh).eval()
        cb, cprefill, csteps = 1, 512, 8
        with torch.no_grad():
            logits, cache = lmc(prompt[:cb, :cprefill].cpu())
            tok = logits[:, -1].argmax(-1, keepdim=True)
            t0 = time.perf_counter()
            for _ in range(csteps):
                logits, cache = lmc(tok, cache)
                tok = logits[:, -1].argmax(-1, keepdim=True)
            dt = time.perf_counter() - t0
        res["cpu_baseline"] = {
            "value": round(cb * csteps / dt, 2), "unit": "tokens/s", "cores": threads,
            "kind": "port",
            "sample": f"the same stack in fp32 on this host (eager cached steps, the reference's "
                      f"CPU path), batch {cb}, prefill {cprefill}, {csteps} steps, "
                      f"{dt / csteps * 1e3:.0f} ms per step"}
    return res


def drafted_decode_bench(dev, drafts, steps=256, prefill=2048, batch=8, warm=2):
    """Config 4's stack with ``drafts`` tokens a row and step: the last decided one and drafts that
    follow it, each the token that last followed the one before in its row (prompt and output).
    One step -- drafting, the model, verification (greedy), commit -- is one HIP graph."""
    from poly_attention import DraftCache, commit_drafts, verify_drafts

    lm, prompt = make_lm(dev, batch=batch, prefill=prefill)
    with torch.no_grad():
        logits, (layer_caches, n) = lm(prompt)
        counts = torch.full((batch,), n, dtype=torch.int32, device=dev)
        caches = [DraftCache(c, n + (steps + warm) * drafts, max_drafts=drafts, counts=counts)
                  for c in layer_caches]
        del layer_caches
        last = logits[:, -1].argmax(-1)
        follow = torch.zeros(batch, 256, dtype=torch.int64, device=dev)
        follow.scatter_(1, prompt[:, :-1], prompt[:, 1:])
        tokens = torch.zeros(batch, drafts, dtype=torch.int64, device=dev)
        slot = torch.arange(drafts, device=dev)

        def step():
            tokens[:, 0] = last
            for t in range(1, drafts):
                tokens[:, t:t + 1] = follow.gather(1, tokens[:, t - 1:t])
            lg, _ = lm(tokens, (caches, None), pos=caches[0].positions(drafts))
            path, kept, token = verify_drafts(lg, tokens)
            commit_drafts(caches, path, kept)
            after = torch.where(slot + 1 == kept[:, None], token[:, None], tokens.roll(-1, 1))
            follow.scatter_(1, tokens, torch.where(slot < kept[:, None], after, follow.gather(1, tokens)))
            last.copy_(token)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(warm):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        torch.cuda.synchronize()
        before = counts.sum().item()
        t0 = time.perf_counter()
        for _ in range(steps):
            graph.replay()
        torch.cuda.synchronize()
        seconds = time.perf_counter() - t0
        for c in caches:
            c.check_overflow()
        kept = counts.sum().item() - before
    return {"workload": f"order-3 drafted decode, config 4's stack, batch {batch}, prefill {prefill}, {drafts} tokens "
                        f"per row and step, {steps} greedy steps",
            "ms_per_step": round(seconds / steps * 1e3, 4), "tokens_per_s": round(kept / seconds, 1),
            "kept_per_row_and_step": round(kept / steps / batch, 3),
            "mode": "DraftCache + one HIP graph per step"}


def _lib():
    from poly_attention import _lib as lib

    return lib


# ---------------------------------------------------------------------------------------
# CPU baseline: the oracle (the reference's eager math) on this host's cores


def cpu_threads():
    """Threads for the CPU baseline: the CPUs this process may run on, capped by
    OMP_NUM_THREADS when set.  A GPU box of this pool gives each GPU a share of the host (16
    CPUs, with OMP_NUM_THREADS=16 exported) while os.cpu_count() reports the whole host; more
    threads than the share only oversubscribe it.  Returns (threads, os.cpu_count(), usable)."""
    total = os.cpu_count() or 1
    try:
        usable = len(os.sched_getaffinity(0))
    except (AttributeError, OSError):
        usable = total
    threads = usable
    omp = os.environ.get("OMP_NUM_THREADS", "")
    if omp.isdigit() and int(omp) > 0:
        threads = min(threads, int(omp))
    return max(1, threads), total, usable


def cpu_model() -> str:
    """The host CPU's model name (lscpu, else /proc/cpuinfo)."""
    names = []
    try:
        out = subprocess.run(["lscpu"], capture_output=True, text=True, timeout=10).stdout
        names += [ln.split(":", 1)[1].strip() for ln in out.splitlines()
                  if ln.startswith("Model name")]
    except Exception:  # noqa: BLE001
        pass
    try:
        with open("/proc/cpuinfo") as f:
            names += [ln.split(":", 1)[1].strip() for ln in f if ln.startswith("model name")][:1]
    except OSError:
        pass
    names = [n for n in names if n]
    return max(names, key=len) if names else (platform.processor() or "unknown")


def cpu_identity() -> dict:
    """CPU family / model / stepping and clock from /proc/cpuinfo: on hosts whose model name
    is only "AMD EPYC" (virtualised), these identify the generation (family 25 = Zen 3 / 4,
    26 = Zen 5)."""
    info = {}
    try:
        with open("/proc/cpuinfo") as f:
            for ln in f:
                if not ln.strip():
                    break  # the first processor's block
                k, _, v = ln.partition(":")
                k = k.strip()
                if k in ("cpu family", "model", "stepping", "cpu MHz", "cache size"):
                    info[k.replace(" ", "_")] = v.strip()
    except OSError:
        pass
    return info


def cpu_baseline(max_seconds=20.0):
    import oracle.poly_oracle as O

    threads, total, usable = cpu_threads()
    torch.set_num_threads(threads)
    hs = 2
    g = torch.Generator().manual_seed(4)
    ts = [torch.randn(1, hs, N, DH, generator=g).requires_grad_() for _ in range(4)]
    dout = torch.randn(1, hs, N, DH, generator=g)

    def step():
        for t in ts:
            t.grad = None
        out, _, _ = O.reference_poly_attention(ts[0], ts[1], ts[1], ts[2], ts[3], causal=True)
        out.backward(dout)

    step()  # warm-up
    times = []
    t_end = time.perf_counter() + max_seconds
    while len(times) < 2 or (time.perf_counter() < t_end and len(times) < 10):
        t0 = time.perf_counter()
        step()
        times.append(time.perf_counter() - t0)
    times.sort()
    med = times[len(times) // 2]
    fwd, bwd = step_flops()
    flops_sample = (fwd + bwd) / (B * H) * hs
    cpu_name = cpu_model()
    return {
        "value": round(flops_sample / med / 1e12, 5),
        "unit": "TFLOP/s",
        "cores": threads,
        "host_cpus": total,
        "usable_cpus": usable,
        "cpu_model": cpu_name,
        "cpu_identity": cpu_identity(),
        "threads_reason": "torch threads = CPUs this process may use, capped by OMP_NUM_THREADS "
                          "(the box's per-GPU CPU share)",
        "kind": "port",
        "sample": f"oracle reference_poly_attention fp32 causal fwd+bwd, B=1 heads={hs} N={N} d={DH} "
                  f"(1/{B * H // hs} of the step), median of {len(times)} after 1 warm-up, "
                  f"{med * 1e3:.0f} ms each; cpu: {cpu_name}",
        "ms_per_step_scaled": round(med * (B * H / hs) * 1e3, 1),
    }


# ---------------------------------------------------------------------------------------


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=30)
    # after an idle spell the GPU's clock takes ~15 config-2 steps (~20 ms) to come up: the
    # first steps run up to 20% slower (1.60 falling to 1.32 ms), so the default warmup
    # covers that ramp
    ap.add_argument("--warmup", type=int, default=25)
    ap.add_argument("--no-cpu", action="store_true")
    ap.add_argument("--no-decode", action="store_true")
    ap.add_argument("--no-module", action="store_true")
    ap.add_argument("--no-masked", action="store_true", help="skip the masked config-2 steps")
    ap.add_argument("--no-vit", action="store_true", help="skip config 3 (PolyViT forward)")
    ap.add_argument("--no-lm", action="store_true", help="skip config 4 (order-3 decode loop)")
    ap.add_argument("--lm-steps", type=int, default=512, help="config 4: greedy decode steps")
    ap.add_argument("--lm-drafts", type=int, default=0,
                    help="config 4 with this many drafted tokens per row and step, beside it (0: off)")
    ap.add_argument("--lm-no-eager", action="store_true",
                    help="config 4: skip the eager tuple-cache loop (profiling runs)")
    ap.add_argument("--calib-copy", action="store_true",
                    help="also run one plain 256 MiB device copy (the reference kernel for scaling "
                         "rocprofv3 FETCH_SIZE / WRITE_SIZE readings)")
    args = ap.parse_args()

    if args.gpus != 1:
        print(f"bench.py measures one GPU: every box of this build has a single MI355X; "
              f"--gpus {args.gpus} is not supported (run with --gpus 1)", file=sys.stderr)
        sys.exit(2)
    if int(os.environ.get("WORLD_SIZE", "1")) > 1:
        print("bench.py runs a single process on one GPU", file=sys.stderr)
        sys.exit(2)

    from poly_attention import _lib

    assert torch.cuda.is_available(), "bench.py needs the GPU"
    _lib.load()
    dev = torch.device("cuda:0")

    m, x, qs, dout, dx = make_config2(dev)
    log(f"[bench] config 2 ready on {torch.cuda.get_device_name(0)}; timing {args.steps} steps")
    ms = time_steps(lambda: core_step(qs, dout), args.steps, args.warmup)
    fwd_f, bwd_f = step_flops()
    tflops = (fwd_f + bwd_f) / (ms / 1e3) / 1e12
    log(f"[bench] core fwd+bwd {ms:.3f} ms/step, {tflops:.1f} TFLOP/s")

    # live per-kernel timing of the same workload (events on the launch stream)
    with _lib.KernelProfile() as prof:
        for _ in range(args.steps):
            core_step(qs, dout)
    kernels = {k: {"launches": n, "avg_ms": round(t / n, 4)} for k, (n, t) in prof.times.items()}
    dominant = max(prof.times.items(), key=lambda kv: kv[1][1])[0]
    n_l, tot = prof.times[dominant]
    bound, peak, work, unit = kernel_work(dominant)
    avg_ms = tot / n_l
    achieved = achieved_rate(work, avg_ms, unit)
    roofline = {"bound": bound, "kernel": dominant, "achieved": round(achieved, 2),
                "peak": peak, "unit": unit, "frac": round(achieved / peak, 4),
                "traffic": measured_traffic(dominant), "avg_ms": round(avg_ms, 4),
                "timer": "HIP events around each launch of the kernel on its own stream "
                         "(libpolyattn pa_profile_start/stop), over a second timed region of "
                         "the same workload"}
    rp = rocprof_avg_ms(dominant)
    if rp:
        # the same figure from the committed rocprofv3 --kernel-trace --stats summary
        roofline["rocprof_avg_ms"] = round(rp, 4)
        roofline["rocprof_frac"] = round(achieved_rate(work, rp, unit) / peak, 4)
    log(f"[bench] kernels: {kernels}")
    # the shader clock under matrix-core load right after the timed steps (libpolyattn
    # pa_measure_clock): tells a slower-clocked box apart from a code change
    gpu_clock = {"ghz": round(_lib.measure_clock(dev), 3),
                 "how": "s_memtime cycles per 100 MHz s_memrealtime tick over a ~50 us all-CU "
                        "MFMA probe run right after the timed steps (libpolyattn "
                        "pa_measure_clock); the bf16 peak of 2.5 PFLOP/s assumes 2.4 GHz"}
    log(f"[bench] gpu clock under MFMA load {gpu_clock['ghz']} GHz")

    module_ms = module_epi_ms = None
    module_kernels = None
    if not args.no_module:
        module_ms = time_steps(lambda: module_step(m, x, dx), max(3, args.steps // 2), 2)
        log(f"[bench] module fwd+bwd {module_ms:.3f} ms/step")
        with _lib.KernelProfile() as mprof:
            for _ in range(3):
                module_step(m, x, dx)
        # the per-head q/k RMSNorms: x read + y written (fwd); x, dy read + dx written (bwd)
        norm_elems = B * H * N * DH
        module_kernels = {}
        for k, (n_l, t) in mprof.times.items():
            rec = {"launches_per_step": n_l // 3, "avg_ms": round(t / n_l, 4)}
            moved = {"rms_fwd": 2 * norm_elems * 2 + B * H * N * 4,
                     "rms_bwd": 3 * norm_elems * 2 + B * H * N * 4}.get(k)
            if moved:
                rec["GB_per_s"] = round(moved / (t / n_l / 1e3) / 1e9, 1)
            module_kernels[k] = rec
        log(f"[bench] module kernels {module_kernels}")
        # the same module with the root-value / gate epilogue (fused into pass 2)
        from poly_attention import PolyAttention

        torch.manual_seed(0)
        me = PolyAttention(dim=DIM, heads=H, dim_head=DH, causal=True, multiply_root_value=True,
                           attn_gate=True).to(dev, torch.bfloat16)
        module_epi_ms = time_steps(lambda: module_step(me, x, dx), max(3, args.steps // 2), 2)
        log(f"[bench] module with root value + gate fwd+bwd {module_epi_ms:.3f} ms/step")
        del me
    masked = None
    if not args.no_masked:
        masked = masked_core_bench(qs, dout, max(3, args.steps // 2), 2)
        log(f"[bench] masked core steps {masked}")
    del qs, dout
    torch.cuda.empty_cache()

    if args.calib_copy:
        src = torch.empty(256 << 20, dtype=torch.uint8, device=dev)
        dst = torch.empty_like(src)
        dst.copy_(src)
        torch.cuda.synchronize()
        del src, dst

    config1 = config1_bench(dev, max(5, args.steps), args.warmup, cpu=not args.no_cpu)
    log(f"[bench] config 1 {config1}")

    decode = None
    if not args.no_decode:
        decode = decode_bench(dev, args.steps, args.warmup)
        log(f"[bench] decode {decode}")

    vit = None
    if not args.no_vit:
        vit = vit_bench(dev, args.steps, args.warmup, cpu=not args.no_cpu)
        log(f"[bench] config 3 {vit}")

    lm = None
    if not args.no_lm:
        lm = decode_order3_bench(dev, cpu=not args.no_cpu, steps=args.lm_steps,
                                 eager=not args.lm_no_eager)
        log(f"[bench] config 4 {lm}")
        if args.lm_drafts:
            lm["drafted"] = drafted_decode_bench(dev, args.lm_drafts)
            log(f"[bench] config 4 drafted {lm['drafted']}")

    cpu = None
    if not args.no_cpu:
        cpu = cpu_baseline()
        log(f"[bench] cpu {cpu}")

    line = {
        "metric": METRIC,
        "value": round(tflops, 2),
        "unit": "TFLOP/s",
        "n_gpus": 1,
        "steps": args.steps,
        "warmup": args.warmup,
        "ms_per_step": round(ms, 4),
        "higher_is_better": True,
        "scaling": "weak",
        "vs_baseline": None,
        "dtype": "bf16",
        "data": "synthetic: x~N(0,1), random-init projections (seed 0), upstream grad~N(0,1)",
        "config": {
            "workload": "order-2 causal poly-attention core fwd+bwd (flash_poly_attention) on the "
                        "q1/q2/q3/v3 of PolyAttention(dim=1024, heads=16, dim_head=64, causal) "
                        "applied to x [4, 4096, 1024] bf16 (BASELINE configs[1])",
            "batch": B, "seq_len": N, "heads": H, "dim_head": DH, "order": 2, "causal": True,
        },
        "frac_mfma_peak": round(tflops / PEAK_BF16_TFLOPS, 4),
        "tokens_per_s": round(B * N / (ms / 1e3), 1),
        "flops_per_step": fwd_f + bwd_f,
        "roofline": roofline,
        "gpu_clock": gpu_clock,
        "kernels": kernels,
        "masked_core": masked,
        "module_ms_per_step": round(module_ms, 4) if module_ms else None,
        "module_root_value_gate_ms_per_step": round(module_epi_ms, 4) if module_epi_ms else None,
        "module_kernels": module_kernels,
        "cpu_baseline": cpu,
        "config1": config1,
        "decode": decode,
        "vit": vit,
        "decode_order3": lm,
    }
    print(json.dumps(line), flush=True)


if __name__ == "__main__":
    main()
