"""Benchmark of the MI355X token sampler (one ns_sample launch per step).

    python bench.py [--gpus 1] [--steps K] [--warmup W] [--cpu-rows R] [--config C]

Workload: the decode-heavy batch -- 256 sampled rows x vocab 128256, logits
stored as bfloat16 (N(0, 3^2)) and upcast in the kernel, temperature 1.0,
top_k 50, top_p 0.95, repetition penalty 1.1 over 2048 Zipf-distributed
history ids per row, one uniform per row.  A step is one ``ns_sample`` call
over the whole batch with every input already resident in device memory.

The timed loop rotates ROTATE independent input sets (logits, histories and
uniforms) so that the working set (> 512 MB) exceeds the 256 MB Infinity
Cache and the rate measured is the HBM rate.  Kernel time is taken with HIP
events on the stream the kernel is launched on.

Prints one JSON line: rows/s (whole job), the roofline of the sampling
kernel against MI355X's 8 TB/s HBM peak, and the CPU baseline (the reference
sampler's op sequence restated on torch CPU, timed on this host).

``--config C`` times another of the five workloads instead (0: B=8 fp32; 1: B=64
mixed parameters; 3: B=128 x 256000 fp32, top-p 0.99; 4: 320 of 4096 rows through
sample indices); its input sets are copies of the workload's own logits rolled
along the vocabulary, so every set keeps the workload's value distribution.
"""
from __future__ import annotations

import argparse
import ctypes
import importlib
import json
import os
import sys
import time

import numpy as np

ROOT = os.path.dirname(os.path.abspath(__file__))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
PKG = "nanoserve---custom-llm-inference-engine_amd"

HBM_PEAK_GBS = 8000.0
MFMA_BF16_PEAK_TFLOPS = 2500.0   # dense bf16
ROTATE = 8
# rocprofv3 FETCH_SIZE + WRITE_SIZE summary of this workload (copy-calibrated HBM bytes per launch)
PMC_SUMMARY = os.path.join(ROOT, "profiles", "topk_kernel_decode_b256_v128256_bf16_pmc.md")
CSRC = os.path.join(ROOT, PKG, "csrc")
WORKLOAD_CFG = 2
METRIC = "sampled rows/sec at B=256, V=128256 fp32; achieved HBM GB/s vs peak"


def _pkg(sub=""):
    return importlib.import_module(PKG + ("." + sub if sub else ""))


def build_sets(w, dev, n_sets, roll=False):
    """Device inputs for ``n_sets`` independent calls over workload ``w`` (sets after the
    first: fresh N(0, 3^2) logits, or with ``roll`` the workload's own rolled along the
    vocabulary)."""
    import torch

    S = _pkg("sampler")
    C = _pkg("config")
    params = [C.SamplingParams(temperature=float(w.temperature[i]), top_k=int(w.top_k[i]), top_p=float(w.top_p[i]),
                               repetition_penalty=float(w.repetition_penalty[i])) for i in range(w.batch)]
    sets = []
    for s in range(n_sets):
        if s == 0:
            logits = w.device_logits(dev)
        elif roll:
            logits = torch.roll(w.device_logits(dev, rotate=s), shifts=7919 * s, dims=1).contiguous()
        else:
            g = torch.Generator(device=dev)
            g.manual_seed(5150 + s)
            x = torch.randn((w.batch, w.vocab), generator=g, device=dev, dtype=torch.float32).mul_(3.0)
            logits = x.to(torch.bfloat16) if w.bf16_bits is not None else x
            del x
        hist = w.histories if s == 0 else [np.roll(h, s) for h in w.histories]
        packed = S.PackedRows(params, hist, w.vocab)
        d = packed.to_device(dev)
        rng = np.random.default_rng(900 + s)
        u = w.uniforms if s == 0 else rng.random(w.batch, dtype=np.float32)
        ut = torch.from_numpy(np.asarray(u, dtype=np.float32)).to(dev)
        out = torch.empty(w.batch, dtype=torch.int64, device=dev)
        sidx = None if w.sample_indices is None else torch.from_numpy(w.sample_indices).to(dev)
        sets.append(dict(logits=logits, d=d, max_hist=packed.max_hist, u=ut, out=out, sidx=sidx,
                         kinds=packed.row_kinds))
    torch.cuda.synchronize()
    return sets


def make_args(L, st, ws):
    import torch

    logits = st["logits"]
    d = st["d"]
    a = L.NsSampleArgs()
    a.logits = logits.data_ptr()
    a.dtype = L.NS_DTYPE_BF16 if logits.dtype == torch.bfloat16 else L.NS_DTYPE_F32
    a.n_sample = int(st["out"].shape[0])
    a.n_rows_total = int(logits.shape[0])
    a.vocab = int(logits.shape[1])
    a.row_stride = int(logits.stride(0))
    a.sample_idx = 0 if st["sidx"] is None else st["sidx"].data_ptr()
    a.temperature = d["temperature"].data_ptr()
    a.top_k = d["top_k"].data_ptr()
    a.top_p = d["top_p"].data_ptr()
    a.rep_penalty = d["rep_penalty"].data_ptr()
    a.hist_offsets = 0 if d["hist_offsets"] is None else d["hist_offsets"].data_ptr()
    a.hist_ids = 0 if d["hist_ids"] is None else d["hist_ids"].data_ptr()
    a.max_hist = int(st["max_hist"])
    a.uniforms = st["u"].data_ptr()
    a.out_ids = st["out"].data_ptr()
    a.out_probs = 0
    a.out_info = 0
    a.workspace = ws.data_ptr()
    a.workspace_bytes = ws.numel()
    a.row_kinds = st["kinds"]
    return a


def lm_head_handoff(L, lib, dev, w, st, stream, iters=50):
    """The step's logits producer in front of the sampler: a random-init lm_head (2048 x V
    bf16, the decode batch's hidden size) as a plain library GEMM, its bf16 output handed to
    ns_sample directly, against the reference's handoff (engine.py:235-236: ``.float()``,
    then the sampler on fp32).  Returns microseconds per step for the GEMM alone and for
    each handoff."""
    import torch

    H = 2048
    g = torch.Generator(device=dev)
    g.manual_seed(4242)
    hidden = torch.randn((w.batch, H), generator=g, device=dev, dtype=torch.float32).to(torch.bfloat16)
    # the lm_head weight stored (H, V): a plain row-major right operand, no transposed view
    weight = (torch.randn((H, w.vocab), generator=g, device=dev, dtype=torch.float32) * (3.0 / H ** 0.5)
              ).to(torch.bfloat16)
    lbf = torch.empty((w.batch, w.vocab), dtype=torch.bfloat16, device=dev)
    lf32 = torch.empty((w.batch, w.vocab), dtype=torch.float32, device=dev)
    # both workspaces stay referenced here: the cached one may be regrown for the fp32 call
    ws_bf = L.workspace_for(dev, w.batch, w.vocab, L.NS_DTYPE_BF16)
    ws32 = L.workspace_for(dev, w.batch, w.vocab, L.NS_DTYPE_F32)
    a_bf = make_args(L, dict(st, logits=lbf), ws_bf)
    a_f32 = make_args(L, dict(st, logits=lf32), ws32)
    sh = ctypes.c_void_p(int(stream.cuda_stream))

    w_vh = weight.t().contiguous()   # the (V, H) lm_head layout ns_lm_head_bf16 reads

    def gemm():
        torch.mm(hidden, weight, out=lbf)

    packed = L.PackedLmHead(w_vh)     # one-time pack, as at model load

    def native_gemm():
        L.lm_head_bf16(hidden, w_vh, out=lbf, stream=stream)

    def packed_gemm():
        L.lm_head_bf16(hidden, packed, out=lbf, stream=stream)

    def reference_gemm():
        # the reference's call on the (V, H) embedding layout (llama.py:141)
        torch.nn.functional.linear(hidden, w_vh)

    def native_step():
        packed_gemm()   # the native producer with the weight packed once at model load
        if lib.ns_sample(ctypes.byref(a_bf), sh) != 0:
            raise RuntimeError(f"ns_sample failed: {L.last_error()}")

    def bf16_step():
        gemm()
        if lib.ns_sample(ctypes.byref(a_bf), sh) != 0:
            raise RuntimeError(f"ns_sample failed: {L.last_error()}")

    def f32_step():
        gemm()
        lf32.copy_(lbf)
        if lib.ns_sample(ctypes.byref(a_f32), sh) != 0:
            raise RuntimeError(f"ns_sample failed: {L.last_error()}")

    res = {}
    for name, fn in (("gemm", gemm), ("bf16_handoff", bf16_step), ("f32_handoff", f32_step),
                     ("native_gemm", native_gemm), ("native_handoff", native_step), ("packed_gemm", packed_gemm),
                     ("reference_gemm", reference_gemm)):
        for _ in range(5):
            fn()
        torch.cuda.synchronize()
        e0 = torch.cuda.Event(enable_timing=True)
        e1 = torch.cuda.Event(enable_timing=True)
        e0.record(stream)
        for _ in range(iters):
            fn()
        e1.record(stream)
        torch.cuda.synchronize()
        res[name] = e0.elapsed_time(e1) / iters * 1e3
    gemm_bytes = weight.numel() * 2 + hidden.numel() * 2 + lbf.numel() * 2
    gemm_flop = 2.0 * w.batch * w.vocab * H
    out = {"lm_head_gemm_us": res["gemm"], "lm_head_gemm_hbm_gbs": gemm_bytes / (res["gemm"] * 1e-6) / 1e9,
           "lm_head_bf16_handoff_us": res["bf16_handoff"], "lm_head_f32_handoff_us": res["f32_handoff"],
           "lm_head_native_gemm_us": res["native_gemm"],
           "lm_head_native_hbm_frac": gemm_bytes / (res["native_gemm"] * 1e-6) / 1e9 / HBM_PEAK_GBS,
           "lm_head_native_mfma_frac": gemm_flop / (res["native_gemm"] * 1e-6) / 1e12 / MFMA_BF16_PEAK_TFLOPS,
           "lm_head_native_handoff_us": res["native_handoff"], "lm_head_packed_gemm_us": res["packed_gemm"],
           "lm_head_reference_layout_gemm_us": res["reference_gemm"]}
    del hidden, weight, w_vh, packed, lbf, lf32, ws_bf, ws32
    return out


def engine_step_legs(sampler, w, dh, reqs, kw, logits, steps=200):
    """The engine's sampling step with its host work (engine.py:238-254): the next step's
    SamplingParams list built and packed (``Sampler.pack``), device histories appended in the
    kernel.  Synchronous: sample, read the ids (``.tolist()``), then the host work of the next
    step.  Pipelined: sample with ``async_ids``, do the next step's host work while the GPU
    samples and the ids travel, then read them.  Returns milliseconds per step for each."""
    C = _pkg("config")

    def host_work():
        params = [C.SamplingParams(temperature=float(w.temperature[i]), top_k=int(w.top_k[i]),
                                   top_p=float(w.top_p[i]), repetition_penalty=float(w.repetition_penalty[i]))
                  for i in range(w.batch)]
        return sampler.pack(params, None, w.vocab, device_histories=dh, history_requests=reqs)

    def run(pipelined):
        packed = host_work()
        for _ in range(5):
            sampler.sample(logits, packed, None, device_histories=dh, **kw).tolist()
        t0 = time.perf_counter()
        for _ in range(steps):
            if pipelined:
                h = sampler.sample(logits, packed, None, device_histories=dh, async_ids=True, **kw)
                packed = host_work()
                h.tolist()
            else:
                sampler.sample(logits, packed, None, device_histories=dh, **kw).tolist()
                packed = host_work()
        return (time.perf_counter() - t0) / steps * 1e3

    return run(False), run(True)


def lm_head_sweep(L, dev, batches=(256, 128, 64, 16, 1), iters=20):
    """The logits producer alone over decode batch sizes: hidden (B, 2048) bf16 times a
    random-init (128256, 2048) bf16 lm_head, through ns_lm_head_bf16 on the weight as
    stored, on the packed weight, and through the library GEMM on the reference's layout
    (F.linear, llama.py:141) and on a transposed copy.  One JSON line per batch size."""
    import torch
    import torch.nn.functional as F

    H, V = 2048, 128256
    g = torch.Generator(device=dev)
    g.manual_seed(4243)
    hid = torch.randn((max(batches), H), generator=g, device=dev, dtype=torch.float32).to(torch.bfloat16)
    w = (torch.randn((V, H), generator=g, device=dev, dtype=torch.float32) * (3.0 / H ** 0.5)).to(torch.bfloat16)
    w_hv = w.t().contiguous()
    pw = L.PackedLmHead(w)
    out = torch.empty((max(batches), V), dtype=torch.bfloat16, device=dev)

    def timed(fn):
        for _ in range(3):
            fn()
        torch.cuda.synchronize()
        e0 = torch.cuda.Event(enable_timing=True)
        e1 = torch.cuda.Event(enable_timing=True)
        e0.record()
        for _ in range(iters):
            fn()
        e1.record()
        torch.cuda.synchronize()
        return e0.elapsed_time(e1) / iters * 1e3

    for m in batches:
        h, o = hid[:m], out[:m]
        r = {"batch": m, "native_us": timed(lambda: L.lm_head_bf16(h, w, out=o)),
             "packed_us": timed(lambda: L.lm_head_bf16(h, pw, out=o)),
             "library_reference_layout_us": timed(lambda: F.linear(h, w)),
             "library_transposed_copy_us": timed(lambda: torch.mm(h, w_hv))}
        nbytes = V * H * 2 + m * H * 2 + m * V * 2
        r["packed_hbm_frac"] = nbytes / (r["packed_us"] * 1e-6) / 1e9 / HBM_PEAK_GBS
        r["packed_mfma_frac"] = 2.0 * m * V * H / (r["packed_us"] * 1e-6) / 1e12 / MFMA_BF16_PEAK_TFLOPS
        print(json.dumps({"lm_head_sweep": r}), flush=True)


def kernel_source_hash():
    """sha256 (first 16 hex digits) over the sampler's kernel sources, in name order."""
    import hashlib

    h = hashlib.sha256()
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".hip", ".h")) and name not in (
                "ns_probe.hip", "ns_paged_attention.hip", "ns_pa_window.h", "ns_kv_cache.hip"):
            with open(os.path.join(CSRC, name), "rb") as f:
                h.update(name.encode() + b"\0" + f.read())
    return h.hexdigest()[:16]


def measured_traffic():
    """HBM bytes per launch from the committed rocprofv3 counter summary -- only when the
    summary was taken on the kernel sources present now (its ``source_sha16`` line), else None."""
    vals = {}
    try:
        with open(PMC_SUMMARY) as f:
            for line in f:
                if ":" in line and line.split(":", 1)[0] in ("traffic_bytes_per_launch", "source_sha16"):
                    k, v = line.split(":", 1)
                    vals[k] = v.strip()
    except OSError:
        return None
    if vals.get("source_sha16") != kernel_source_hash() or "traffic_bytes_per_launch" not in vals:
        return None
    return int(vals["traffic_bytes_per_launch"])


# stamp slots of the top-k kernel, in the order a row passes them
STAMP_SLOTS = (("entry", 0), ("wave0_streamed", 1), ("last_wave_streamed", 2), ("last_wave_bound", 7),
               ("bound_barrier", 3), ("wave0_staged", 8), ("wave0_listed", 9), ("list_barrier", 4),
               ("order_barrier", 5), ("wave0_cut", 10), ("drawn", 6))
NS_STAMPS = 16


def phase_stamps(L, dev, w, sets, ws, stream, reps=20, calls=20):
    """Where the top-k kernel's time goes, from its phase stamps: libns_sampling_stamps.so is
    the sampler built with NS_PHASE_STAMPS, whose top-k kernel stores the shader clock
    (s_memtime) of each workgroup at the points STAMP_SLOTS names: entry; wave 0 and the last
    wave done streaming and reducing their share of the row; the last wave's bound; the bound's
    barrier; wave 0's chunks staged and candidates listed; the list's barrier; the ordering's
    barrier; wave 0's top-k cut; the id drawn.  ``reps`` times: ``calls`` back-to-back calls
    over the rotating input sets, then the last call's stamps (every workgroup's, in steady
    state) are read.  Returns, per point, the median clocks since entry over all rows and
    repetitions, and the same in microseconds at the clock rate that makes the median
    workgroup's span equal the per-call time measured by events in the same run."""
    import torch

    so = os.path.join(ROOT, PKG, "libns_sampling_stamps.so")
    lib = ctypes.CDLL(so)
    lib.ns_sample.restype = ctypes.c_int
    lib.ns_phase_stamps_set.restype = ctypes.c_int
    buf = torch.zeros(w.batch * NS_STAMPS, dtype=torch.int64, device=dev)
    if lib.ns_phase_stamps_set(ctypes.c_void_p(buf.data_ptr())) != 0:
        raise RuntimeError("ns_phase_stamps_set failed")
    cargs = [make_args(L, st, ws) for st in sets]
    sh = ctypes.c_void_p(int(stream.cuda_stream))
    rows = []
    e0 = torch.cuda.Event(enable_timing=True)
    e1 = torch.cuda.Event(enable_timing=True)
    t_ms = 0.0
    for r in range(reps):
        torch.cuda.synchronize()
        e0.record(stream)
        for i in range(calls):
            if lib.ns_sample(ctypes.byref(cargs[(r * calls + i) % ROTATE]), sh) != 0:
                raise RuntimeError("stamped ns_sample failed")
        e1.record(stream)
        torch.cuda.synchronize()
        t_ms += e0.elapsed_time(e1)
        rows.append(buf.view(w.batch, NS_STAMPS).cpu().numpy().astype(np.int64))
    lib.ns_phase_stamps_set(ctypes.c_void_p(0))
    st = np.concatenate(rows)
    t0 = st[:, 0]
    us_per_call = t_ms / (reps * calls) * 1e3
    span = float(np.median(st[:, 6] - t0))
    per_us = span / us_per_call
    out = {"stamped_kernel_us": us_per_call, "median_workgroup_span_clocks": span, "clocks_per_us": per_us}
    prev = STAMP_SLOTS[0]
    for name, slot in STAMP_SLOTS[1:]:
        out[f"{name}_after_entry_us"] = float(np.median(st[:, slot] - t0)) / per_us
        out[f"{prev[0]}->{name}_us"] = float(np.median(st[:, slot] - st[:, prev[1]])) / per_us
        prev = (name, slot)
    return out


def cpu_model():
    try:
        with open("/proc/cpuinfo") as f:
            for line in f:
                if line.startswith("model name"):
                    return line.split(":", 1)[1].strip()
    except OSError:
        pass
    return None


def read_floor(L, sets, stream, iters=200):
    """Time of a kernel that only streams the input sets' logits rows, in the sampler's
    layout and cache policy (libns_probe.so): the floor of a one-pass kernel over the same
    bytes, measured on this GPU.  Returns microseconds per call, or None when the rows do not
    fit the probe (more than 256 KiB per row, or sample indices)."""
    import torch

    so = os.path.join(ROOT, PKG, "libns_probe.so")
    lg = sets[0]["logits"]
    row_bytes = lg.shape[1] * lg.element_size()
    if not os.path.exists(so) or sets[0]["sidx"] is not None or row_bytes % 16 or row_bytes > 16 * 1024 * 16:
        return None
    lib = ctypes.CDLL(so)
    lib.ns_probe_read_rows.restype = ctypes.c_int
    lib.ns_probe_read_rows.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int32,
                                       ctypes.c_void_p, ctypes.c_void_p]
    out = torch.empty(lg.shape[0] * 16, dtype=torch.int32, device=lg.device)   # one word per wave
    sh = ctypes.c_void_p(int(stream.cuda_stream))

    def call(i):
        x = sets[i % len(sets)]["logits"]
        if lib.ns_probe_read_rows(x.data_ptr(), x.stride(0) * x.element_size(), row_bytes, x.shape[0],
                                  out.data_ptr(), sh) != 0:
            raise RuntimeError("ns_probe_read_rows refused its arguments")

    for i in range(20):
        call(i)
    torch.cuda.synchronize()
    e0 = torch.cuda.Event(enable_timing=True)
    e1 = torch.cuda.Event(enable_timing=True)
    e0.record(stream)
    for i in range(iters):
        call(i)
    e1.record(stream)
    torch.cuda.synchronize()
    return e0.elapsed_time(e1) / iters * 1e3


def cpu_baseline(w, rows: int, reps: int):
    """The reference sampler's op sequence on torch CPU over ``rows`` rows of the workload."""
    import torch

    from oracle import sampler_oracle as O  # the CPU restatement of sampler.py:28-89

    cores = len(os.sched_getaffinity(0))
    torch.set_num_threads(cores)
    rows = min(rows, w.batch)
    x = torch.from_numpy(np.ascontiguousarray(w.rows[:rows]))
    args = (w.temperature[:rows], w.top_k[:rows], w.top_p[:rows], w.repetition_penalty[:rows],
            [list(map(int, h)) for h in w.histories[:rows]])
    gen = torch.Generator()
    gen.manual_seed(0)
    O.reference_restatement_multinomial(x[:1], *(a[:1] for a in args), generator=gen)  # warm
    times = []
    for _ in range(reps):
        t0 = time.perf_counter()
        O.reference_restatement_multinomial(x, *args, generator=gen)
        times.append(time.perf_counter() - t0)
    med = float(np.median(times))
    return {"value": rows / med, "unit": "rows/s", "cores": cores, "kind": "port", "cpu_model": cpu_model(),
            "sample": f"{rows} rows of the same workload (fp32 logits, the reference's .float() input), "
                      f"median of {reps} runs of {med:.3f} s; torch {torch.__version__} CPU"}


def small_batch_leg(L, lib, dev, stream, steps=400, cpu_reps=20):
    """The reference's CPU-runnable case (B=8 x V=128256 fp32, t=0.8 top_k=50 top_p=0.9,
    penalty 1.1 over 64 ids): ns_sample's kernel time on it, and the CPU sampler on the same rows."""
    import torch

    w = _pkg("workloads").make_workload(0)
    sets = build_sets(w, dev, ROTATE, roll=True)
    ws = L.workspace_for(dev, w.batch, w.vocab, L.NS_DTYPE_F32)
    cargs = [make_args(L, st, ws) for st in sets]
    sh = ctypes.c_void_p(int(stream.cuda_stream))
    for i in range(40):
        if lib.ns_sample(ctypes.byref(cargs[i % ROTATE]), sh) != 0:
            raise RuntimeError(f"ns_sample failed: {L.last_error()}")
    torch.cuda.synchronize()
    e0 = torch.cuda.Event(enable_timing=True)
    e1 = torch.cuda.Event(enable_timing=True)
    e0.record(stream)
    for i in range(steps):
        lib.ns_sample(ctypes.byref(cargs[i % ROTATE]), sh)
    e1.record(stream)
    torch.cuda.synchronize()
    us = e0.elapsed_time(e1) / steps * 1e3
    cpu = cpu_baseline(w, w.batch, cpu_reps) if cpu_reps > 0 else None
    return {"small_batch_b8_kernel_us": us, "small_batch_b8_rows_per_s": w.batch / (us * 1e-6),
            "small_batch_b8_hbm_frac": _pkg("workloads").algorithmic_bytes(w) / (us * 1e-6) / 1e9 / HBM_PEAK_GBS,
            "small_batch_b8_cpu_baseline": cpu}


def copy_reference(dev, mb):
    """4 plain device copies of ``mb`` MiB: a known-size reference for HBM byte counters."""
    import torch

    n = mb * (1 << 20) // 4
    src = torch.ones(n, dtype=torch.float32, device=dev)
    dst = torch.empty_like(src)
    for _ in range(4):
        dst.copy_(src)
    torch.cuda.synchronize()
    del src, dst


def paged_attention_leg(dev, stream, steps=200, seqs=64, ctx=2048):
    """Paged attention at a decode step of Llama-3.2-3B's layout (24 query heads, 8 KV heads, head_dim
    128, block_size 16, bf16): ``seqs`` rows of ``ctx`` positions each, physical blocks shuffled, two
    caches alternated so consecutive calls do not hit the previous call's KV in the last-level cache.
    Algorithmic bytes: every visible key and value row once (seqs * ctx * 8 heads * 128 * 2 B * 2)
    plus the query read and the output write."""
    import torch

    A = _pkg("paged_attention")
    hq, hkv, d, bs = 24, 8, 128, 16
    nblk = seqs * ctx // bs
    g = torch.Generator(device=dev)
    g.manual_seed(7)
    caches = [(torch.randn(nblk, bs, hkv, d, device=dev, generator=g, dtype=torch.bfloat16),
               torch.randn(nblk, bs, hkv, d, device=dev, generator=g, dtype=torch.bfloat16)) for _ in range(2)]
    bt = torch.randperm(nblk, device=dev, generator=g).to(torch.int32).view(seqs, ctx // bs)
    q = torch.randn(seqs, hq, d, device=dev, generator=g, dtype=torch.bfloat16)
    sl = torch.full((seqs,), ctx, dtype=torch.int32, device=dev)
    ql = torch.ones(seqs, dtype=torch.int32, device=dev)
    qsl = torch.arange(seqs + 1, dtype=torch.int32, device=dev)
    out = torch.empty_like(q)
    ws = torch.empty(max(A.workspace_bytes(seqs, hq, hkv, d, ctx), 1), dtype=torch.uint8, device=dev)
    cnt = torch.zeros(seqs * hkv, dtype=torch.int32, device=dev)

    def call(i):
        k, v = caches[i % 2]
        A.paged_attention_hip(q, k, v, bt, sl, qsl, ql, d ** -0.5, bs, max_seq_len=ctx, max_query_len=1, out=out,
                              workspace=ws, counters=cnt, stream=stream.cuda_stream)

    for i in range(20):
        call(i)
    torch.cuda.synchronize()
    e0 = torch.cuda.Event(enable_timing=True)
    e1 = torch.cuda.Event(enable_timing=True)
    e0.record(stream)
    for i in range(steps):
        call(i)
    e1.record(stream)
    torch.cuda.synchronize()
    us = e0.elapsed_time(e1) / steps * 1e3
    nbytes = seqs * ctx * hkv * d * 2 * 2 + 2 * q.numel() * 2
    gbs = nbytes / (us * 1e-6) / 1e9
    del caches
    return {"paged_attention_decode_b%d_ctx%d_us" % (seqs, ctx): us,
            "paged_attention_decode_algorithmic_bytes": nbytes,
            "paged_attention_decode_hbm_gbs": gbs,
            "paged_attention_decode_hbm_frac": gbs / HBM_PEAK_GBS,
            "paged_attention_decode_tokens_per_s": seqs / (us * 1e-6)}


def paged_attention_prefill_leg(dev, stream, steps=50, chunk=512, ends=(2048, 4096, 6144, 8192)):
    """A chunked-prefill step at Llama-3.2-3B's layout (24 query heads, 8 KV heads, head_dim 128,
    block_size 16, bf16): one 512-token chunk (the reference's chunked_prefill_size, config.py:53)
    ending at each of ``ends`` positions, physical blocks shuffled, two caches alternated.  Timed
    on the query-tile MFMA kernel (the plan made once, as an engine makes it once per step for all
    its layers) and on the per-token kernel for the same batch.  Roofline: MFMA bf16; algorithmic
    flops 4 * head_dim per (query token, query head, visible position) (the two products; the
    kernel's second, low-part product of P is not counted)."""
    import torch

    A = _pkg("paged_attention")
    hq, hkv, d, bs = 24, 8, 128, 16
    seqs = len(ends)
    per = [e // bs for e in ends]
    nblk = sum(per)
    g = torch.Generator(device=dev)
    g.manual_seed(11)
    caches = [(torch.randn(nblk, bs, hkv, d, device=dev, generator=g, dtype=torch.bfloat16),
               torch.randn(nblk, bs, hkv, d, device=dev, generator=g, dtype=torch.bfloat16)) for _ in range(2)]
    perm = torch.randperm(nblk, device=dev, generator=g).to(torch.int32)
    bt = torch.zeros((seqs, max(per)), dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(per):
        bt[s, :n] = perm[at:at + n]
        at += n
    total_q = chunk * seqs
    q = torch.randn(total_q, hq, d, device=dev, generator=g, dtype=torch.bfloat16)
    sl = torch.tensor(list(ends), dtype=torch.int32, device=dev)
    ql = torch.full((seqs,), chunk, dtype=torch.int32, device=dev)
    qsl = torch.arange(0, total_q + 1, chunk, dtype=torch.int32, device=dev)
    out = torch.empty_like(q)
    plan = A.PagedAttentionPlan(sl, qsl, ql, hq, hkv, dev)
    res = {}
    for name, kw in (("tiles", dict(plan=plan)), ("per_token", dict(max_query_len=1))):
        ws, cnt = None, None

        def call(i):
            k, v = caches[i % 2]
            return A.paged_attention_hip(q, k, v, bt, sl, qsl, ql, d ** -0.5, bs, max_seq_len=max(ends), out=out,
                                         workspace=ws, counters=cnt, stream=stream.cuda_stream, **kw)

        for i in range(3):
            call(i)
        torch.cuda.synchronize()
        n = steps if name == "tiles" else max(3, steps // 10)
        e0 = torch.cuda.Event(enable_timing=True)
        e1 = torch.cuda.Event(enable_timing=True)
        e0.record(stream)
        for i in range(n):
            call(i)
        e1.record(stream)
        torch.cuda.synchronize()
        res[name] = e0.elapsed_time(e1) / n * 1e3
    visible = sum(sum(e - chunk + i + 1 for i in range(chunk)) for e in ends)
    flops = 4.0 * d * hq * visible
    kv_bytes = sum(ends) * hkv * d * 2 * 2
    del caches
    tf = flops / (res["tiles"] * 1e-6) / 1e12
    return {"paged_attention_prefill_workload": f"{seqs} chunks of {chunk} tokens ending at {list(ends)} positions, "
                                                f"24/8 heads, head_dim 128, bf16",
            "paged_attention_prefill_tiles_us": res["tiles"], "paged_attention_prefill_per_token_us": res["per_token"],
            "paged_attention_prefill_algorithmic_flops": flops, "paged_attention_prefill_tflops": tf,
            "paged_attention_prefill_mfma_frac": tf / MFMA_BF16_PEAK_TFLOPS,
            "paged_attention_prefill_kv_bytes": kv_bytes,
            "paged_attention_prefill_tokens_per_s": total_q / (res["tiles"] * 1e-6)}


def paged_attention_cpu_baseline(seqs=64, ctx=2048, reps=3):
    """The reference's SDPA backend (paged_attention_torch.py:31-100: per sequence, gather the KV
    through the block table, repeat the KV heads, scaled_dot_product_attention) restated in torch on
    the host CPU, on the same decode step as the GPU leg (bf16, shuffled blocks). Median of ``reps``."""
    import torch
    import torch.nn.functional as F

    hq, hkv, d, bs = 24, 8, 128, 16
    g = torch.Generator()
    g.manual_seed(7)
    nblk = seqs * ctx // bs
    k_cache = torch.randn(nblk, bs, hkv, d, generator=g).to(torch.bfloat16)
    v_cache = torch.randn(nblk, bs, hkv, d, generator=g).to(torch.bfloat16)
    bt = torch.randperm(nblk, generator=g).to(torch.int32).view(seqs, ctx // bs)
    q = torch.randn(seqs, hq, d, generator=g).to(torch.bfloat16)

    def step():
        out = torch.empty_like(q)
        for i in range(seqs):
            k = k_cache.index_select(0, bt[i]).reshape(-1, hkv, d).repeat_interleave(hq // hkv, dim=1)
            v = v_cache.index_select(0, bt[i]).reshape(-1, hkv, d).repeat_interleave(hq // hkv, dim=1)
            a = F.scaled_dot_product_attention(q[i:i + 1].transpose(0, 1).unsqueeze(0), k.transpose(0, 1).unsqueeze(0),
                                               v.transpose(0, 1).unsqueeze(0), scale=d ** -0.5)
            out[i] = a.squeeze(0).transpose(0, 1)[0]
        return out

    step()
    times = []
    for _ in range(reps):
        t0 = time.perf_counter()
        step()
        times.append(time.perf_counter() - t0)
    sec = sorted(times)[len(times) // 2]
    return {"value": seqs / sec, "unit": "decode rows/s", "cores": torch.get_num_threads(), "kind": "port",
            "cpu_model": cpu_model(),
            "sample": f"the full {seqs} x {ctx} bf16 decode step through the SDPA backend restated in torch "
                      f"(paged_attention_torch.py:31-100), median of {reps} runs of {sec:.3f} s; torch {torch.__version__} CPU"}


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=400)
    ap.add_argument("--warmup", type=int, default=40)
    ap.add_argument("--cpu-rows", type=int, default=256, help="rows in the CPU-baseline sample (0 = skip)")
    ap.add_argument("--cpu-reps", type=int, default=3)
    ap.add_argument("--config", type=int, default=WORKLOAD_CFG, choices=range(5),
                    help="workload to time (default: the decode batch the metric is quoted on)")
    ap.add_argument("--copy-mb", type=int, default=0,
                    help="after the timed loop, run 4 plain device copies of this many MiB (a known-size "
                         "reference for HBM byte counters under rocprofv3 --pmc)")
    ap.add_argument("--lm-head-sweep", action="store_true",
                    help="time only the logits producer (lm_head GEMM) over decode batch sizes and exit")
    ap.add_argument("--paged-attention", action="store_true",
                    help="time only the paged-attention decode leg (64 rows x 2048 positions) and exit")
    ap.add_argument("--phase-stamps", action="store_true",
                    help="print where the top-k kernel's time goes (the stamps library) and exit")
    args = ap.parse_args(argv)
    if args.gpus != 1 or int(os.environ.get("WORLD_SIZE", "1")) != 1:
        print("bench.py measures one GPU: the sampler's rows are independent and this build runs on a single "
              "MI355X; --gpus above 1 is not supported", file=sys.stderr)
        return 2

    import torch

    if not torch.cuda.is_available():
        print("bench.py needs a GPU", file=sys.stderr)
        return 2
    W = _pkg("workloads")
    L = _pkg("_lib")
    lib = L.load()
    dev = torch.device("cuda:0")
    torch.cuda.set_device(dev)
    if args.lm_head_sweep:
        lm_head_sweep(L, dev)
        if args.copy_mb > 0:
            copy_reference(dev, args.copy_mb)
        return 0
    if args.paged_attention:
        st = torch.cuda.current_stream(dev)
        line = {}
        for seqs, ctx in ((64, 2048), (8, 8192), (256, 1024)):
            r = paged_attention_leg(dev, st, steps=args.steps, seqs=seqs, ctx=ctx)
            print(f"[bench] paged attention decode {seqs}x{ctx}: {r}", file=sys.stderr, flush=True)
            line.update({k.replace("paged_attention_decode_", f"paged_attention_decode_b{seqs}_ctx{ctx}_")
                         if not k.startswith(f"paged_attention_decode_b{seqs}_ctx{ctx}") else k: v
                         for k, v in r.items()})
        line.update(paged_attention_prefill_leg(dev, st, steps=max(10, args.steps // 8)))
        print(json.dumps(line), flush=True)
        if args.copy_mb > 0:
            copy_reference(dev, args.copy_mb)
        return 0

    w = W.make_workload(args.config)
    sets = build_sets(w, dev, ROTATE, roll=args.config != WORKLOAD_CFG)
    ws = L.workspace_for(dev, w.batch, w.vocab, L.NS_DTYPE_BF16 if w.bf16_bits is not None else L.NS_DTYPE_F32)
    cargs = [make_args(L, st, ws) for st in sets]
    stream = torch.cuda.current_stream(dev)
    sh = ctypes.c_void_p(int(stream.cuda_stream))
    bytes_per_call = W.algorithmic_bytes(w)
    if args.phase_stamps:
        print(json.dumps({"phase_stamps": phase_stamps(L, dev, w, sets, ws, stream), "config": args.config}),
              flush=True)
        return 0

    def step(i):
        rc = lib.ns_sample(ctypes.byref(cargs[i % ROTATE]), sh)
        if rc != 0:
            raise RuntimeError(f"ns_sample failed ({rc}): {L.last_error()}")

    for i in range(args.warmup):
        step(i)
    torch.cuda.synchronize()
    ev0 = torch.cuda.Event(enable_timing=True)
    ev1 = torch.cuda.Event(enable_timing=True)
    t0 = time.perf_counter()
    ev0.record(stream)
    for i in range(args.steps):
        step(i)
    ev1.record(stream)
    torch.cuda.synchronize()
    wall = time.perf_counter() - t0
    gpu_ms = ev0.elapsed_time(ev1)
    ms_per_step = gpu_ms / args.steps
    rows_per_s = w.batch / (ms_per_step * 1e-3)
    achieved = bytes_per_call / (ms_per_step * 1e-3) / 1e9

    # wrapper-inclusive rate (Sampler.sample: host packing and the host-to-device copy of params/histories)
    S = _pkg()
    C = _pkg("config")
    params = [C.SamplingParams(temperature=float(w.temperature[i]), top_k=int(w.top_k[i]), top_p=float(w.top_p[i]),
                               repetition_penalty=float(w.repetition_penalty[i])) for i in range(w.batch)]
    hist_lists = [list(map(int, h)) for h in w.histories]
    sampler = S.Sampler(dev)
    kw = dict(uniforms=sets[0]["u"], sample_indices=sets[0]["sidx"])
    for _ in range(3):
        sampler.sample(sets[0]["logits"], params, hist_lists, **kw)
    torch.cuda.synchronize()
    nwrap = 10
    t1 = time.perf_counter()
    for _ in range(nwrap):
        ids = sampler.sample(sets[0]["logits"], params, hist_lists, **kw)
    ids.tolist()
    wrap_ms = (time.perf_counter() - t1) / nwrap * 1e3
    # the same calls with the histories kept on the device (copied once per request, each
    # sampled token appended in place): the per-step host work is the parameters only
    dh = S.DeviceHistories(dev, w.batch, capacity=_pkg("_lib").NS_LDS_HISTORY)
    for i, h in enumerate(hist_lists):
        dh.open(i, h)
    reqs = list(range(w.batch))
    for _ in range(3):
        sampler.sample(sets[0]["logits"], params, None, device_histories=dh, history_requests=reqs, **kw)
    torch.cuda.synchronize()
    t1 = time.perf_counter()
    for _ in range(nwrap):
        ids = sampler.sample(sets[0]["logits"], params, None, device_histories=dh, history_requests=reqs, **kw)
    ids.tolist()
    wrap_dev_ms = (time.perf_counter() - t1) / nwrap * 1e3
    step_sync_ms, step_pipe_ms = engine_step_legs(sampler, w, dh, reqs, kw, sets[0]["logits"])
    del dh
    producer = lm_head_handoff(L, lib, dev, w, sets[0], stream) if args.config == WORKLOAD_CFG else {}
    floor_us = read_floor(L, sets, stream)
    floor = {} if floor_us is None else {
        "read_floor_us": floor_us, "read_floor_frac_of_peak": bytes_per_call / (floor_us * 1e-6) / 1e9 / HBM_PEAK_GBS,
        "kernel_over_read_floor": ms_per_step * 1e3 / floor_us}

    if args.copy_mb > 0:
        copy_reference(dev, args.copy_mb)

    cpu = cpu_baseline(w, args.cpu_rows, args.cpu_reps) if args.cpu_rows > 0 else None
    small = small_batch_leg(L, lib, dev, stream, cpu_reps=20 if args.cpu_rows > 0 else 0) \
        if args.config == WORKLOAD_CFG else {}
    attention = paged_attention_leg(dev, stream) if args.config == WORKLOAD_CFG else {}
    if attention:
        attention.update(paged_attention_prefill_leg(dev, stream))
    if attention and args.cpu_rows > 0:
        attention["paged_attention_cpu_baseline"] = paged_attention_cpu_baseline()
    if args.config != WORKLOAD_CFG:
        desc = {0: "batch B=8 x V=128256 fp32, t=0.8 top_k=50 top_p=0.9 penalty=1.1, 64 history ids/row",
                1: "batch B=64 x V=128256 fp32, mixed per-row parameters (greedy and sampled), 512 Zipf ids/row",
                3: "batch B=128 x V=256000 fp32 heavy-tailed logits, t=1.2 top_p=0.99, no penalty",
                4: "320 sampled rows of a 4096 x 128256 fp32 flat tensor (sample indices), mixed parameters, "
                   "histories U[1,4096]"}[args.config]
        nb = f"B={w.batch}, V={w.vocab} {w.dtype}"
        line = {"metric": f"sampled rows/sec at {nb}; achieved HBM GB/s vs peak", "value": rows_per_s,
                "unit": "rows/s", "n_gpus": 1, "steps": args.steps, "warmup": args.warmup,
                "ms_per_step": ms_per_step, "higher_is_better": True, "scaling": "weak", "vs_baseline": None,
                "dtype": "f32", "data": "synthetic (the workload's seeded logits, rolled per input set)",
                "config": {"workload": desc, "batch": w.batch, "vocab": w.vocab, "rotating_input_sets": ROTATE,
                           "parallelism": "single GPU"},
                "roofline": {"bound": "hbm", "achieved": achieved, "peak": HBM_PEAK_GBS, "unit": "GB/s",
                             "frac": achieved / HBM_PEAK_GBS, "traffic": None},
                "cpu_baseline": cpu,
                "extra": {"algorithmic_bytes_per_call": bytes_per_call, "kernel_us": ms_per_step * 1e3,
                          "wall_s": wall, "wrapper_inclusive_ms": wrap_ms,
                          "wrapper_inclusive_ms_device_histories": wrap_dev_ms,
                          "engine_step_sync_ids_ms": step_sync_ms, "engine_step_async_ids_ms": step_pipe_ms,
                          **floor}}
        print(json.dumps(line), flush=True)
        return 0
    line = {
        "metric": METRIC,
        "value": rows_per_s,
        "unit": "rows/s",
        "n_gpus": 1,
        "steps": args.steps,
        "warmup": args.warmup,
        "ms_per_step": ms_per_step,
        "higher_is_better": True,
        "scaling": "weak",
        "vs_baseline": None,
        "dtype": "f32",
        "data": "synthetic (seeded N(0,3^2) logits rounded to bf16, Zipf histories)",
        "config": {"workload": "decode batch B=256 x V=128256, bf16 logits upcast to f32 in-kernel, "
                               "t=1.0 top_k=50 top_p=0.95 penalty=1.1, 2048 history ids/row",
                   "batch": w.batch, "vocab": w.vocab, "history": 2048, "rotating_input_sets": ROTATE,
                   "parallelism": "single GPU"},
        "roofline": {"bound": "hbm", "achieved": achieved, "peak": HBM_PEAK_GBS, "unit": "GB/s",
                     "frac": achieved / HBM_PEAK_GBS, "traffic": measured_traffic()},
        "cpu_baseline": cpu,
        "extra": {"algorithmic_bytes_per_call": bytes_per_call, "kernel_us": ms_per_step * 1e3,
                  "wall_s": wall, "wrapper_inclusive_ms": wrap_ms,
                  "wrapper_inclusive_rows_per_s": w.batch / (wrap_ms * 1e-3),
                  "wrapper_inclusive_ms_device_histories": wrap_dev_ms,
                  "wrapper_inclusive_rows_per_s_device_histories": w.batch / (wrap_dev_ms * 1e-3),
                  "engine_step_sync_ids_ms": step_sync_ms, "engine_step_async_ids_ms": step_pipe_ms,
                  "kernel_source_sha16": kernel_source_hash(), **floor, **small, **producer, **attention},
    }
    print(json.dumps(line), flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
