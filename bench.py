#!/usr/bin/env python3
"""bench.py -- headline benchmark of the MI355X-native qMRI hot path.

    python bench.py --gpus N --steps K --warmup W
    (N > 1: launched by the driver through torch.distributed.run, one rank per GPU)

Metric: voxel-fits/sec, 8-echo mono-exponential T2 fit of a 512x512x160 volume
(configs[1]: "T2 monoexponential fit, 512x512x160 x 8 echoes, fp32, 1 MI355X") + UNet2D slices/sec.

A "step" is one pass of the hot path over one synthetic volume per GPU: ONE launch of the fused
kernel (LM fit + MonoExponentialFit post-processing) on (8, 41 943 040) fp32 samples already
resident in HBM, writing fp32 (a, tc) + r2 -- i.e. `MonoExponentialFit().fit(x, y)` with the
reference's defaults (tc0 = 30 -> p0 = (1, -1/30), bounds (0, 100), r2 >= 0.9, 1 decimal).  `value` is that rate at
every N (weak scaling: one volume per GPU per step, no data-path collective), so the per-N values are comparable.
Reported beside it in the same JSON line:

  "parity"       what the TIMED kernel wrote, checked after the timed loop against the oracle's C restatement on the
                 SURVEY 8(d) sample (first 20 000 tissue + 1 000 background voxels) -- the oracle is the checker here,
                 never inside a timed region;
  "runs"         the f64-output variant (56 B/voxel, what the drop-in API returns), the scan-class recipe
                 (tc0 = "polyfit", 3 decimals) and BASELINE configs[2] (T1rho ROI);
  "unet2d"       UNet2D slices/s at 384x384x160: `value` = the mode that meets the 1e-3 logit bar,
                 the plain-bf16 mode beside it;
  "cfg5"         BASELINE configs[4]: 8 volumes per GPU (64 at N = 8), fit + 512x512 UNet segmentation per volume,
                 sharded by dosma_amd.dist.run_batch, UNet weights made on rank 0 and broadcast once (RCCL);
  "roofline"     algorithmic HBM bytes (44 B/voxel = 8 x 4 B in + 12 B out) / kernel
                 time measured with HIP events on the launch stream, vs the 8 TB/s HBM3E peak;
  "cpu_baseline" the reference's own call pattern (one scipy.optimize.curve_fit per voxel, serial and under
                 multiprocessing.Pool, dosma/core/fitting.py:855-868, 1026-1073) timed on this
                 host's cores on a bounded sample of the same volume (N = 1 runs only).
"""
import argparse
import ctypes
import hashlib
import json
import os
import sys
import time
from functools import partial

import numpy as np

ROOT = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, ROOT)

SHAPE = (512, 512, 160)
E = 8
TE = np.arange(1, E + 1) * 10.0  # ms
BYTES_PER_VOXEL = 4 * E + 4 * 3  # fp32 echoes in, fp32 (a, tc, r2) out -- SURVEY.md section 8(d)
BYTES_PER_VOXEL_F64 = 4 * E + 8 * 3  # float64 outputs like the reference returns (56 B)
HBM_PEAK_GBS = 8000.0            # MI355X_MICROARCH.md: HBM3E 8.0 TB/s spec
P0_A = (1.0, -1 / 30.0)


def make_volume(torch, device, seed):
    """70 % tissue S0~U(300,1500), T2~U(15,80) ms, SNR 50; 30 % exact zeros."""
    n = SHAPE[0] * SHAPE[1] * SHAPE[2]
    gen = torch.Generator(device=device).manual_seed(seed)
    s0 = torch.rand(n, device=device, generator=gen) * 1200 + 300
    t2 = torch.rand(n, device=device, generator=gen) * 65 + 15
    te = torch.tensor(TE, device=device, dtype=torch.float32)
    y = s0[None, :] * torch.exp(-te[:, None] / t2[None, :])
    y += (900.0 / 50.0) * torch.randn(y.shape, device=device, generator=gen)
    bg = torch.rand(n, device=device, generator=gen) < 0.3
    y[:, bg] = 0
    return y.contiguous()


def make_args(L, y, popt, r2, stream, recipe, out_dtype=None):
    a = L.default_args()
    n = y.shape[1]
    a.y, a.y_dtype, a.E, a.N, a.ld = y.data_ptr(), L.QMRI_F32, E, n, n
    a.x = TE.ctypes.data_as(ctypes.POINTER(ctypes.c_double))
    a.popt, a.r2, a.out_dtype = popt.data_ptr(), r2.data_ptr(), (L.QMRI_F32 if out_dtype is None else out_dtype)
    a.stream = stream
    bounds = ((-np.inf, np.inf), (0.0, 100.0))
    if recipe == "A":  # MonoExponentialFit() defaults
        a.init, a.a0, a.b0 = L.INIT_SCALAR, P0_A[0], P0_A[1]
        L.set_post(a, inv_abs_b=True, bounds=bounds, r2_threshold=0.9, nan_to_num=0.0, decimals=1)
    else:              # scan classes: tc0="polyfit", decimal_precision=3
        a.init = L.INIT_LOGLIN
        L.set_post(a, inv_abs_b=True, bounds=bounds, r2_threshold=0.9, nan_to_num=0.0, decimals=3)
    return a


def parity_sample(L, torch, y, popt, r2):
    """What the timed kernel wrote vs the oracle (SURVEY.md 8(d) cfg2 parity sample).  `popt` / `r2` are the output
    buffers of the LAST TIMED LAUNCH (recipe A, fp32): post-processed (a, tc) and r2 of every voxel."""
    from oracle import fit_oracle as fo  # the checker (never inside a timed region)

    nz = (y != 0).any(dim=0)
    idx = torch.cat([torch.nonzero(nz)[:20000, 0], torch.nonzero(~nz)[:1000, 0]])
    ys = y[:, idx].cpu().numpy().astype(np.float64)
    got_p = popt[idx].cpu().numpy().astype(np.float64)
    got_r = r2[idx].cpu().numpy().astype(np.float64)
    _, ref_r, ref_p = fo.monoexp_fit_arrays(TE, ys, bounds=(0, 100), tc0=30.0, r2_threshold=0.9, decimal_precision=None)
    same_zero = (got_p == 0) == (ref_p == 0)
    both = (ref_p != 0) & (got_p != 0)
    with np.errstate(all="ignore"):
        rel = np.abs(got_p[both] / ref_p[both] - 1)
    # MINPACK's own trajectory: an extra UNTIMED launch of the same kernel on the sample with the raw outputs and the
    # per-voxel stop code / evaluation count, against the C restatement run with full_output
    raw = L.monoexp_fit_host(TE, ys.astype(np.float32), p0=P0_A, want_info=True)
    cp, cr, cinfo, cnfev = fo.curve_fit_c(TE, ys.astype(np.float32), P0_A, full_output=True)
    ok = ~np.isnan(cp[:, 0])
    with np.errstate(all="ignore"):
        raw_rel = np.abs(raw["popt"][ok] / cp[ok] - 1)
    return {
        "n": int(idx.numel()), "sample": "first 20000 tissue + first 1000 background voxels of the timed volume",
        "timed_outputs": {"max_rel": float(rel.max()) if rel.size else 0.0,
                          "zero_pattern_equal_frac": float(same_zero.mean()),
                          "r2_max_abs": float(np.abs(got_r - ref_r).max()),
                          "what": "popt (a, tc) and r2 written by the last timed launch (fp32) vs "
                                  "oracle.fit_oracle.monoexp_fit_arrays (float64)"},
        "max_rel": float(np.nanmax(raw_rel)) if raw_rel.size else 0.0,
        "nfev_equal_frac": float((raw["nfev"] == cnfev).mean()),
        "info_class_equal_frac": float((((raw["info"] >= 1) & (raw["info"] <= 4)) == ((cinfo >= 1) & (cinfo <= 4))).mean()),
        "failed_equal": bool(np.array_equal(np.isnan(raw["popt"][:, 0]), ~ok)),
        "tolerance": "north_star: popt / r2 within 1e-4 relative of scipy.optimize.curve_fit",
    }


def bench_t1rho_roi(L, lib, torch, device, local_rank, args):
    """BASELINE.json configs[2] (a parity-test configuration, reported for information): CubeQuant T1rho, 4 spin-lock
    times, 384 x 384 x 120 int16 volumes, cartilage-mask ROI (~2 % of the voxels), tc0="polyfit", bounds (0, 500),
    3 decimals.  Device-resident, kernel time from HIP events."""
    shape = (384, 384, 120)
    n = shape[0] * shape[1] * shape[2]
    tsl = np.array([1.0, 10.0, 30.0, 60.0])
    gen = torch.Generator(device=device).manual_seed(384)
    s0 = torch.rand(n, device=device, generator=gen) * 2200 + 800
    t1r = torch.rand(n, device=device, generator=gen) * 45 + 25
    t = torch.tensor(tsl, device=device, dtype=torch.float32)
    y = s0[None, :] * torch.exp(-t[:, None] / t1r[None, :]) + 20.0 * torch.randn((4, n), device=device, generator=gen)
    y = y.round().clamp(-32768, 32767).to(torch.int16).contiguous()
    mask = torch.zeros(shape, dtype=torch.uint8, device=device)
    mask[150:230, 120:260, 40:70] = (torch.rand((80, 140, 30), device=device, generator=gen) < 0.85).to(torch.uint8)
    mask = mask.reshape(-1).contiguous()
    roi = int(mask.sum().item())
    popt = torch.empty((n, 2), dtype=torch.float32, device=device)
    r2 = torch.empty(n, dtype=torch.float32, device=device)
    tc = torch.empty(n, dtype=torch.float32, device=device)
    stream = torch.cuda.current_stream(device)
    a = L.default_args()
    a.y, a.y_dtype, a.E, a.N, a.ld = y.data_ptr(), L.QMRI_I16, 4, n, n
    a.x = tsl.ctypes.data_as(ctypes.POINTER(ctypes.c_double))
    a.mask = mask.data_ptr()
    a.popt, a.r2, a.tc, a.out_dtype = popt.data_ptr(), r2.data_ptr(), tc.data_ptr(), L.QMRI_F32
    a.stream = stream.cuda_stream
    a.device = local_rank
    a.init = L.INIT_LOGLIN
    L.set_post(a, inv_abs_b=True, bounds=((-np.inf, np.inf), (0.0, 500.0)), r2_threshold=0.9, nan_to_num=0.0, decimals=3)
    for _ in range(max(args.warmup, 1)):
        L.check(lib.qmri_monoexp_fit_device(ctypes.byref(a), None))
    ev0 = torch.cuda.Event(enable_timing=True)
    ev1 = torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize(device)
    ev0.record(stream)
    for _ in range(args.steps):
        L.check(lib.qmri_monoexp_fit_device(ctypes.byref(a), None))
    ev1.record(stream)
    torch.cuda.synchronize(device)
    ms = ev0.elapsed_time(ev1) / args.steps
    return {"config": "T1rho (CubeQuant recipe), 4 spin-lock times, 384x384x120 int16, ROI mask only (BASELINE configs[2])",
            "volume_voxels": n, "roi_voxels": roi, "kernel_ms": ms,
            "roi_voxel_fits_per_s": roi / (ms * 1e-3), "volume_voxels_per_s": n / (ms * 1e-3),
            "hbm_gb_per_s": (n * (1 + 3 * 4) + roi * 4 * 2) / (ms * 1e-3) / 1e9,
            "kernel": lib.qmri_monoexp_kernel_name(ctypes.byref(a)).decode()}


def _ref_style_voxel(y_i, x, p0, ftol, maxfev, eps):
    """One voxel the way the reference's `_curve_fit` treats it (dosma/core/fitting.py:1026-1073): skip rule,
    scipy.optimize.curve_fit(func, x, y, p0, ftol, maxfev), r2, RuntimeError -> NaN / 0.  Module level so that
    `partial(...)` of it pickles ONCE per chunk like the reference's `partial(_curve_fit, ...)` (:844-853)."""
    from oracle import fit_oracle as fo

    return fo._one_voxel_scipy((fo.monoexponential, x, y_i, p0, ftol, maxfev, eps, 2, False))


def effective_cores():
    """What the lease really delivers: the cgroup CPU quota (cpu.max, v2; cfs quota, v1) next to the affinity count.
    (256 visible cores, ~10 cores' worth of throughput.)"""
    quota = None
    try:
        q, p = open("/sys/fs/cgroup/cpu.max").read().split()[:2]
        if q != "max":
            quota = float(q) / float(p)
    except (OSError, ValueError):
        try:
            q = float(open("/sys/fs/cgroup/cpu/cpu.cfs_quota_us").read())
            p = float(open("/sys/fs/cgroup/cpu/cpu.cfs_period_us").read())
            if q > 0:
                quota = q / p
        except (OSError, ValueError):
            pass
    return quota


def _scaling_ladder(fitter, y_T, cores):
    """voxel-fits/s of the reference's call pattern with 1, 2, 4, ... workers on a fixed 40 000-voxel slice: where the
    curve flattens is the number of cores the host actually gives this process."""
    import multiprocessing as mp

    m = min(len(y_T), 40000)
    ladder = {}
    w = 1
    while w <= cores:
        with mp.Pool(w) as pool:
            pool.map(fitter, y_T[: w * 4], chunksize=4)
            t = time.perf_counter()
            pool.map(fitter, y_T[:m], chunksize=max(50, min(1000, m // (4 * w))))
            ladder[w] = m / (time.perf_counter() - t)
        if w >= 4 and ladder[w] < 1.15 * ladder[w // 2] and ladder[w // 2] < 1.15 * ladder[w // 4]:
            break   # flat twice in a row: more workers only add processes
        w *= 2
    if cores not in ladder:  # the reference's own default for "all cores" (num_workers = os.cpu_count()), for the record
        with mp.Pool(cores) as pool:
            pool.map(fitter, y_T[: cores * 4], chunksize=4)
            t = time.perf_counter()
            pool.map(fitter, y_T[:m], chunksize=max(50, min(1000, m // (4 * cores))))
            ladder[cores] = m / (time.perf_counter() - t)
    return ladder


def cpu_baseline(y_dev, cores_cap=None):
    """The reference's per-voxel scipy loop (fitting.py:855-868) on a bounded sample of the bench volume, timed on
    this host: serial (num_workers = 0), Pool(1) (num_workers = 1) and Pool(all cores) with
    chunksize 1000 -- rows of y_T mapped through ONE partial, exactly the reference's `p.map(fitter, y_T, chunksize)`."""
    import multiprocessing as mp

    import scipy

    from oracle import fit_oracle as fo  # the checker, used here only as the timed CPU baseline

    try:
        cores = len(os.sched_getaffinity(0))
    except AttributeError:
        cores = os.cpu_count() or 1
    if cores_cap:
        cores = min(cores, cores_cap)
    n = int(min(y_dev.shape[1], 6000 * cores, 800_000))
    ys = y_dev[:, :n].cpu().numpy()
    y_T = np.ascontiguousarray(ys.T)  # (N, E): one row per voxel, like the reference's y.T (:833)
    fitter = partial(_ref_style_voxel, x=TE, p0=P0_A, ftol=fo.FTOL, maxfev=fo.MAXFEV, eps=fo.R2_EPS)
    # serial (num_workers = 0) and one worker (num_workers = 1) on a small slice
    m1 = min(n, 12000)
    t = time.perf_counter()
    for i in range(m1):
        fitter(y_T[i])
    dt_serial = time.perf_counter() - t
    with mp.Pool(1) as pool:
        pool.map(fitter, y_T[:64], chunksize=8)
        t = time.perf_counter()
        pool.map(fitter, y_T[:m1], chunksize=1000)
        dt_one = time.perf_counter() - t
    # how many cores does the host really give this process?  cgroup quota if there is one, else where the worker
    # ladder of the same call pattern flattens (throughput with all workers / throughput with one)
    ladder = _scaling_ladder(fitter, y_T, cores)
    quota = effective_cores()
    scale = max(ladder.values()) / ladder[1]
    if quota:
        eff, eff_how = min(float(cores), quota), "cgroup cpu.max quota"
    else:
        eff, eff_how = min(float(cores), max(1.0, scale)), "all-worker / one-worker throughput of the reference's call pattern"
    # the baseline is the host's BEST -- the ladder's best rung (Pool(256) on a 16-core quota cost it 25 %),
    # timed on the whole sample
    # (the ladder's slice is short and its chunks small: its two best rungs are both timed on the whole sample, the faster one is `value`)
    full = {}
    for w in sorted(ladder, key=ladder.get, reverse=True)[:2]:
        with mp.Pool(w) as pool:
            pool.map(fitter, y_T[: w * 4], chunksize=4)  # start the workers
            t = time.perf_counter()
            pool.map(fitter, y_T, chunksize=1000)
            full[w] = time.perf_counter() - t
    best_w = min(full, key=full.get)
    dt = full[best_w]
    # single-thread C restatement of MINPACK on a slice, for scale
    m = min(n, 200_000)
    t = time.perf_counter()
    fo.curve_fit_c(TE, ys[:, :m], P0_A, threads=1)
    dt_c = time.perf_counter() - t
    # the same C restatement on every core (threads inside the library): the best this host can do with the algorithm
    fo.curve_fit_c(TE, ys[:, : min(n, 4 * cores)], P0_A, threads=cores)  # start the threads
    t = time.perf_counter()
    fo.curve_fit_c(TE, ys, P0_A, threads=cores)
    dt_call = time.perf_counter() - t
    return {
        "value": n / dt, "unit": "voxel-fits/s", "cores": best_w, "kind": "port",
        "sample": (f"first {n} voxels of the bench volume (70% tissue / 30% zero background): one "
                   f"scipy.optimize.curve_fit per voxel, rows of y.T through multiprocessing.Pool({best_w}).map("
                   f"partial(fitter), chunksize=1000) (the reference's call pattern, fitting.py:860-868) with the number "
                   f"of workers that was fastest on this host (worker_ladder_voxel_fits_per_s; {cores} cores visible), scipy "
                   f"{scipy.__version__}, {dt:.1f} s wall, pool start-up excluded"),
        "workers": best_w,
        "visible_cores": cores,
        "full_sample_voxel_fits_per_s_by_workers": {str(w): n / t for w, t in full.items()},
        "effective_cores": eff,
        "effective_cores_how": eff_how,
        "per_core": n / dt / eff,
        "per_worker": n / dt / best_w,
        "worker_ladder_voxel_fits_per_s": {str(k): v for k, v in ladder.items()},
        "cgroup_cpu_quota_cores": quota,
        "num_workers_0_serial": m1 / dt_serial,
        "num_workers_1": m1 / dt_one,
        "serial_sample": f"first {m1} voxels",
        "c_restatement_1thread": m / dt_c,
        "c_restatement_all_cores": n / dt_call,
    }


def bench_dess(L, lib, torch, device, local_rank, world, args, barrier):
    """qDESS analytic T2 map: one fused streaming pass over two fp32 echo volumes of
    384x384x160 -> fp64 map (the reference's dtype).  HBM-bound: 2 x 4 B in + 8 B out per voxel."""
    n = 384 * 384 * 160
    gen = torch.Generator(device=device).manual_seed(11 + local_rank)
    e1 = torch.rand(n, device=device, generator=gen) * 780 + 20
    e2 = e1 * (torch.rand(n, device=device, generator=gen) * 0.88 + 0.02)
    t2 = torch.empty(n, device=device, dtype=torch.float64)
    a = L.QmriDessArgs()
    a.echo1, a.echo2, a.dtype, a.out_dtype, a.N = e1.data_ptr(), e2.data_ptr(), L.QMRI_F32, L.QMRI_F64, n
    a.c0, a.k, a.c1 = -27.864, 0.0434, 3.9e-3
    a.use_bounds, a.lo, a.hi, a.use_nan_to_num, a.nan_value, a.decimals = 1, 0.0, 100.0, 1, 0.0, 1
    a.t2, a.device = t2.data_ptr(), local_rank
    stream = torch.cuda.current_stream(device)
    a.stream = stream.cuda_stream
    for _ in range(3):
        L.check(lib.qmri_dess_t2_device(ctypes.byref(a)))
    ev0, ev1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    barrier()
    ev0.record(stream)
    reps = 20
    for _ in range(reps):
        L.check(lib.qmri_dess_t2_device(ctypes.byref(a)))
    ev1.record(stream)
    barrier()
    ms = ev0.elapsed_time(ev1) / reps
    gbs = 16.0 * n / (ms * 1e-3) / 1e9
    # the same kernel on a batch of 8 volumes in ONE launch (3 GB of traffic): long enough to leave launch ramp and tail behind
    nb = 8 * n
    e1b = e1.repeat(8)
    e2b = e2.repeat(8)
    t2b = torch.empty(nb, device=device, dtype=torch.float64)
    b = L.QmriDessArgs()
    ctypes.memmove(ctypes.byref(b), ctypes.byref(a), ctypes.sizeof(a))
    b.echo1, b.echo2, b.t2, b.N = e1b.data_ptr(), e2b.data_ptr(), t2b.data_ptr(), nb
    for _ in range(2):
        L.check(lib.qmri_dess_t2_device(ctypes.byref(b)))
    barrier()
    ev0.record(stream)
    for _ in range(10):
        L.check(lib.qmri_dess_t2_device(ctypes.byref(b)))
    ev1.record(stream)
    barrier()
    msb = ev0.elapsed_time(ev1) / 10
    gbsb = 16.0 * nb / (msb * 1e-3) / 1e9
    same = bool(torch.equal(t2b[:n], t2) and torch.equal(t2b[7 * n:], t2))
    del e1b, e2b, t2b
    return {"metric": "qDESS analytic T2 map, 384x384x160, fp32 echoes -> fp64 map", "voxels_per_s": n / (ms * 1e-3),
            "kernel_ms": ms, "roofline": {"bound": "hbm", "achieved": gbs, "peak": HBM_PEAK_GBS, "unit": "GB/s",
                                          "frac": gbs / HBM_PEAK_GBS, "algorithmic_bytes_per_voxel": 16},
            "batch8": {"what": "8 volumes in one launch (3.0 GB algorithmic)", "kernel_ms": msb, "voxels_per_s": nb / (msb * 1e-3),
                       "roofline": {"bound": "hbm", "achieved": gbsb, "peak": HBM_PEAK_GBS, "unit": "GB/s",
                                    "frac": gbsb / HBM_PEAK_GBS},
                       "outputs_equal_single_volume": same}}


UNET_HW = 384
UNET_SLICES = 160
UNET_GFLOP_PER_SLICE = 70.79   # 35.39 GMAC per 384x384 slice
MFMA_BF16_PEAK_TFLOPS = 2500.0  # MI355X_MICROARCH.md: dense bf16 / fp16 MFMA peak
UNET_PARITY_MODE = "fp16x3"      # the precision mode whose logits meet north_star's 1e-3 (tests/test_unet_gpu.py)


def _mfma_ceiling():
    """What v_mfma_f32_32x32x16_f16 sustains on THIS part on N(0,1) operands with nothing else in the loop (data-dependent
    power sets the clock): a constant read from the committed stdout of scripts/probes/mfma_peak.hip (profiles/r0*_mfma_peak.txt,
    newest tag), not re-measured by this run.  `peak` of the roofline stays the 2.5 PF of MI355X_MICROARCH.md."""
    import glob
    import re
    for path in sorted(glob.glob(os.path.join(ROOT, "profiles", "r0*_mfma_peak.txt")), key=os.path.basename, reverse=True):
        try:
            vals = [float(m.group(1)) for line in open(path) if line.startswith("N(0,1)")
                    for m in [re.search(r"=\s*([0-9.]+) TFLOP/s", line)] if m]
        except OSError:
            continue
        if vals:
            return {"tflops": max(vals), "source": os.path.relpath(path, ROOT),
                    "what": "scripts/probes/mfma_peak.hip, N(0,1) fp16 operands, best of 1 / 2 waves per SIMD"}
    return None


UNET_REF_SCLK_GHZ = 1.82  # the clock round 5's 1.38 kW forward held (profiles/r05_power.txt): the reference point of value_at_ref_clock


class GpuSampler:
    """Shader clock and board power of one GPU, sampled in a side thread while a timed loop runs (the MFMA
    legs run against the 1.4 kW cap and boxes differ by +-3 % in the clock they hold; without the clock in the line two rounds'
    numbers cannot be compared).  Reads the amdgpu hwmon files of the device's PCI function (freq1_input = sclk in Hz,
    power1_average / power1_input in microwatts: what rocm-smi prints) every few ms; where the box exposes no hwmon node it
    falls back to polling `rocm-smi --showpower --showclocks` (the logic of scripts/power_sample.sh; ~3 samples per second).
    Never raises: a box without either yields {"samples": 0}."""

    def __init__(self, torch, dev_index, period_s=0.004):
        import glob
        import threading

        self.period, self.rows, self._stop, self._thr, self.dev_index = period_s, [], threading.Event(), None, dev_index
        self.how, self.f_clk, self.f_pow = None, None, None
        cands = []
        try:
            pr = torch.cuda.get_device_properties(dev_index)
            bdf = f"{pr.pci_domain_id:04x}:{pr.pci_bus_id:02x}:{pr.pci_device_id:02x}.0"
            cands = sorted(glob.glob(f"/sys/bus/pci/devices/{bdf}/hwmon/hwmon*"))
        except Exception:
            pass
        if not cands:  # no PCI address from torch: the dev_index-th amdgpu hwmon node in PCI order
            nodes = []
            for h in glob.glob("/sys/class/drm/card*/device/hwmon/hwmon*"):
                try:
                    if open(os.path.join(h, "name")).read().strip() == "amdgpu":
                        nodes.append((os.path.realpath(os.path.join(h, "..", "..")), h))
                except OSError:
                    pass
            nodes.sort()
            if dev_index < len(nodes):
                cands = [nodes[dev_index][1]]
        for h in cands:
            clk = os.path.join(h, "freq1_input")
            pw = next((os.path.join(h, f) for f in ("power1_average", "power1_input") if os.path.exists(os.path.join(h, f))), None)
            self.f_pow = self.f_pow or pw  # (a node without the clock's file still has the power's)
            if os.path.exists(clk) and self._read(clk) is not None:
                self.how, self.f_clk, self.f_pow = f"hwmon ({os.path.basename(clk)}, {os.path.basename(pw) if pw else 'no power file'})", clk, pw
                break
        if self.how is None:
            import shutil

            self.smi = shutil.which("rocm-smi") or "/opt/rocm/bin/rocm-smi"
            if os.path.exists(self.smi):
                self.how = "rocm-smi --showpower --showclocks (polled)"
                if self.f_pow:
                    self.how += f", hwmon {os.path.basename(self.f_pow)}"

    @staticmethod
    def _read(path):
        try:
            with open(path) as f:
                return float(f.read().strip())
        except (OSError, ValueError):
            return None

    def _poll_smi(self):
        import re
        import subprocess

        try:
            txt = subprocess.run([self.smi, "-d", str(self.dev_index), "--showpower", "--showclocks"], stdout=subprocess.PIPE,
                                 stderr=subprocess.DEVNULL, text=True, timeout=5).stdout
        except Exception:
            return None, None
        c = re.search(r"sclk clock level:\s*\w+:\s*\((\d+)Mhz\)", txt)
        w = re.search(r"Power \(W\):\s*([\d.]+)", txt)
        return (float(c.group(1)) * 1e6 if c else None), (float(w.group(1)) * 1e6 if w else None)

    def _run(self):
        while not self._stop.is_set():
            if self.f_clk:
                c, w = self._read(self.f_clk), (self._read(self.f_pow) if self.f_pow else None)
                self._stop.wait(self.period)
            else:
                c, w = self._poll_smi()
                w = w or (self._read(self.f_pow) if self.f_pow else None)
            self.rows.append((time.perf_counter(), c, w))

    def __enter__(self):
        import threading

        if self.how is not None:
            self.rows, self._stop = [], threading.Event()
            self._thr = threading.Thread(target=self._run, daemon=True)
            self._thr.start()
        return self

    def __exit__(self, *exc):
        if self._thr is not None:
            self._stop.set()
            self._thr.join(timeout=10)
            self._thr = None
        return False

    def summary(self, t0=None, t1=None):
        """Means over the samples taken in [t0, t1] (time.perf_counter values; the whole run when omitted)."""
        rows = [r for r in self.rows if (t0 is None or r[0] >= t0) and (t1 is None or r[0] <= t1)]
        clk = [r[1] for r in rows if r[1]]
        pw = [r[2] for r in rows if r[2]]
        return {"samples": len(rows), "how": self.how,
                "sclk_ghz_mean": (sum(clk) / len(clk) / 1e9) if clk else None,
                "sclk_ghz_min": (min(clk) / 1e9) if clk else None, "sclk_ghz_max": (max(clk) / 1e9) if clk else None,
                "power_w_mean": (sum(pw) / len(pw) / 1e6) if pw else None, "power_w_max": (max(pw) / 1e6) if pw else None}


def bench_unet(L, torch, dist, device, local_rank, world, args, barrier, red_device):
    """UNet2D slices/s (IWOAIOAIUnet2DNormalized, 384x384x160, MFMA conv).

    A step = one whole volume (160 sagittal slices incl. whole-volume whitening) per GPU through the
    network, input resident in HBM, logits + masks written to HBM.  `value` is the PARITY mode (logits within 1e-3 of
    the fp64 restatement: three 16-bit MFMAs per product); the plain-bf16 mode (one MFMA per product, logits within
    ~0.25) is reported beside it.  Random He-initialised weights of the reference architecture (the trained .h5 is
    not distributed; throughput does not depend on the values) and random-normal input (not zeros: DVFS,
    cdna_hip_programming.md rule 25)."""
    from dosma_amd.models import weights as W

    eng = L.Unet2dEngine(W.to_abi_order(W.random_weights(seed=0)), UNET_HW, UNET_HW,
                         max_batch=args.unet_batch, precision="bf16", device=local_rank)
    gen = torch.Generator(device=device).manual_seed(7 + local_rank)
    x = torch.randn((UNET_SLICES, UNET_HW, UNET_HW), device=device, generator=gen) * 150 + 300
    logits = torch.empty((UNET_SLICES, UNET_HW, UNET_HW, 4), device=device)
    mask = torch.empty((UNET_SLICES, UNET_HW, UNET_HW, 4), device=device, dtype=torch.uint8)
    stream = torch.cuda.current_stream(device)
    steps = max(2, args.steps // 4)
    res, clocks = {}, {}
    sampler = GpuSampler(torch, local_rank)
    rank_zero_extras = (not dist.is_initialized()) or dist.get_rank() == 0
    for prec in ("bf16", UNET_PARITY_MODE):
        eng.set_precision(prec)
        for _ in range(max(1, args.warmup // 2)):
            eng.forward_device(x.data_ptr(), UNET_SLICES, logits.data_ptr(), mask.data_ptr(), whiten=True,
                               stream=stream.cuda_stream)
        barrier()
        with sampler:
            t0 = time.perf_counter()
            for _ in range(steps):
                eng.forward_device(x.data_ptr(), UNET_SLICES, logits.data_ptr(), mask.data_ptr(), whiten=True,
                                   stream=stream.cuda_stream)
            barrier()
            t1 = time.perf_counter()
        el = t1 - t0
        if dist.is_initialized():
            t = torch.tensor([el], device=red_device, dtype=torch.float64)
            dist.all_reduce(t, op=dist.ReduceOp.MAX)
            el = t[0].item()
        res[prec] = UNET_SLICES * world * steps / el
        clocks[prec] = sampler.summary(t0, t1)
    # the timed loop is a fraction of a second; under a power cap the clock keeps settling for longer than that.  The same
    # forward for ~2 s more (outside `value`), sampled: the steady-state rate and the clock / power it is held at -- the pair that
    # makes two boxes' (two rounds') numbers comparable
    eng.set_precision(UNET_PARITY_MODE)
    sustained = None
    if rank_zero_extras:
        n_sus = max(steps, int(2.0 / max(1e-3, UNET_SLICES * world / res[UNET_PARITY_MODE])))
        torch.cuda.synchronize(device)
        with sampler:
            t0 = time.perf_counter()
            for _ in range(n_sus):
                eng.forward_device(x.data_ptr(), UNET_SLICES, logits.data_ptr(), mask.data_ptr(), whiten=True,
                                   stream=stream.cuda_stream)
            torch.cuda.synchronize(device)
            t1 = time.perf_counter()
        sustained = {"steps": n_sus, "seconds": t1 - t0, "slices_per_s_this_rank": UNET_SLICES * n_sus / (t1 - t0),
                     **sampler.summary(t0 + 0.25 * (t1 - t0), t1)}
    eng.close()
    ck = clocks[UNET_PARITY_MODE]
    # (the clock read during the fraction-of-a-second timed loop is a lagging average that still carries the previous mode's
    # clock -- first run of round 6: 1.94 GHz in the timed loop, 1.82 GHz sustained, the same slices/s in both -- so the
    # reference-clock figure uses the sustained leg's clock)
    sclk_ref = (sustained or {}).get("sclk_ghz_mean") or ck.get("sclk_ghz_mean")
    ref_clock = (res[UNET_PARITY_MODE] * UNET_REF_SCLK_GHZ / sclk_ref) if sclk_ref else None
    tf = res[UNET_PARITY_MODE] / world * UNET_GFLOP_PER_SLICE / 1e3
    tf16 = res["bf16"] / world * UNET_GFLOP_PER_SLICE / 1e3
    return {
        "metric": "UNet2D slices/sec (IWOAIOAIUnet2DNormalized, 384x384x160, MFMA conv)",
        "value": res[UNET_PARITY_MODE], "unit": "slices/s", "steps": steps, "batch": args.unet_batch,
        "precision": f"{UNET_PARITY_MODE}: 16-bit hi + lo operand parts, hi*hi + hi*lo + lo*hi on MFMA (3 per product), "
                     "fp32 accumulate -- the mode whose logits are within 1e-3 of the fp64 restatement "
                     "(tests/test_unet_gpu.py); the plain-bf16 mode (1 MFMA per product, logits within ~0.25) is "
                     "`slices_per_s_bf16`",
        "slices_per_s_bf16": res["bf16"],
        "value_at_ref_clock": ref_clock,
        "value_at_ref_clock_note": f"value x {UNET_REF_SCLK_GHZ} GHz / sclk_ghz_mean of the sustained leg (rank 0's GPU), as VERDICT r5 asked.  CAVEAT, measured "
                                   "in round 6 on three boxes at the same 1.37 kW: reported sclk 1.806 / 1.825 / 1.959 GHz, sustained 5417 / 5430 / 5500 slices/s -- the "
                                   "rate does NOT follow the reported clock one to one (+8.5 % clock, +1.5 % rate), so this field over-corrects; read `value` with "
                                   "`sustained.sclk_ghz_mean` / `power_w_mean` beside it and trust only same-box alternating A/Bs below +-2 % (README: comparing rounds)",
        "sustained": sustained,
        "data": "synthetic (random He weights of the reference architecture, random-normal input)",
        "roofline": {"bound": "mfma", "achieved": tf, "peak": MFMA_BF16_PEAK_TFLOPS, "unit": "TFLOP/s",
                     "frac": tf / MFMA_BF16_PEAK_TFLOPS, "gflop_per_slice": UNET_GFLOP_PER_SLICE,
                     "sclk_ghz_mean": sclk_ref, "power_w_mean": (sustained or {}).get("power_w_mean") or ck.get("power_w_mean"),
                     "clock_samples": ck, "bf16_mode_clock_samples": clocks.get("bf16"),
                     "mfma_issued_frac": 3 * tf / MFMA_BF16_PEAK_TFLOPS,
                     "mfma_ceiling_measured": _mfma_ceiling(),
                     "frac_of_measured_ceiling": (3 * tf / _mfma_ceiling()["tflops"]) if _mfma_ceiling() else None,
                     "note": "achieved = ALGORITHMIC flops (70.79 GFLOP per slice); the parity mode issues 3 MFMAs per "
                             "product, so the matrix pipes are busy 3x that fraction (mfma_issued_frac)",
                     "bf16_mode": {"achieved": tf16, "frac": tf16 / MFMA_BF16_PEAK_TFLOPS},
                     **_unet_traffic()},
    }


UNET_SOURCES = ("unet_s3.hip", "unet_c4.hip", "unet_d4.hip", "unet_c4_common.h", "unet_enc0.hip", "unet_kernels.hip", "unet_rw.hip", "unet_engine.hip", "qmri_internal.h")


def _source_sha1(files):
    h = hashlib.sha1()
    for f in files:
        with open(os.path.join(ROOT, "dosma_amd", "csrc", f), "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()


def _unet_source_sha1():
    return _source_sha1(UNET_SOURCES)


def unet_algorithmic_bytes(hw=UNET_HW, slices=UNET_SLICES, nf=(32, 64, 128, 256, 512, 1024)):
    """Layer-by-layer minimum HBM bytes of one forward in the parity mode AS BUILT (4 B per activation value = fp16 hi +
    lo; first block, pooling and classifier fused): every feature map that crosses a kernel boundary is written once and
    read once.  (25.4 GB written + 25.5 GB read = 50.9 GB per 160 slices of 384 x 384.)"""
    px = [float(hw * hw) / 4 ** l for l in range(len(nf))]
    wr = rd = 0.0
    rd += px[0] * 4                                  # the whitened input image (fp32)
    for l, c in enumerate(nf):                       # encoder
        if l > 0:
            rd += px[l] * nf[l - 1] * 4              # conv1 reads the pooled tensor
            wr += px[l] * c * 4                      # conv1 -> conv2 (level 0: conv1 lives in LDS only)
            rd += px[l] * c * 4
        wr += px[l] * c * 4                          # conv2 (+ BN): the skip tensor (deepest level: the bottom tensor)
        if l < len(nf) - 1:
            wr += px[l + 1] * c * 4                  # pooled output (fused into conv2's epilogue ...
            if (hw >> l) <= 48:
                rd += px[l] * c * 4                  # ... except on the flattened narrow levels: a separate pooling kernel)
    for l in range(len(nf) - 2, -1, -1):             # decoder
        c = nf[l]
        rd += px[l + 1] * nf[l + 1] * 4              # transposed convolution reads the level below
        wr += px[l] * c * 4                          # ... and writes its half of the concat buffer
        rd += px[l] * 2 * c * 4                      # conv1 reads [up | skip]
        wr += px[l] * c * 4                          # conv1 -> conv2
        rd += px[l] * c * 4
        if l > 0:
            wr += px[l] * c * 4                      # conv2 (+ BN) -> next transposed convolution
    wr += px[0] * (4 * 4 + 4)                        # logits (fp32 x 4) + mask bytes of the fused classifier
    return slices * (wr + rd), slices * wr, slices * rd


def _unet_traffic():
    """HBM bytes of one 160-slice forward in the parity mode: a constant from the newest rocprofv3 --pmc collection
    (scripts/collect_profile.sh -> profiles/<tag>_unet_counters.json), not re-measured by this run; `stale` says whether
    the UNet kernel sources have changed since it was collected."""
    import glob
    alg, alg_w, alg_r = unet_algorithmic_bytes()
    base = {"algorithmic_bytes": alg, "algorithmic_bytes_written": alg_w, "algorithmic_bytes_read": alg_r,
            "algorithmic_bytes_note": "layer-by-layer minimum as built (4 B per activation value, first block / pooling / "
                                      "classifier fused): every feature map crossing a kernel boundary written once, read once"}
    # newest first BY TAG (r04c > r03g: file times do not survive a checkout); a file whose recorded source hash matches
    # the current sources wins over a newer tag that does not
    paths = sorted(glob.glob(os.path.join(ROOT, "profiles", "r0*_unet_counters.json")),
                   key=lambda q: os.path.basename(q), reverse=True)
    cur = _unet_source_sha1()

    def _sha_of(q):
        try:
            return json.load(open(q)).get("kernel_source_sha1")
        except (OSError, ValueError):
            return None
    paths.sort(key=lambda q: _sha_of(q) != cur)  # stable: matching files first, tag order kept inside each group
    for path in paths:
        try:
            pj = json.load(open(path))
        except (OSError, ValueError):
            continue
        hbm = pj.get("hbm")
        if hbm:
            sha = pj.get("kernel_source_sha1")
            return {"traffic": hbm["bytes_per_forward"], "traffic_over_algorithmic": hbm["bytes_per_forward"] / alg, **base,
                    "traffic_source": {"file": os.path.relpath(path, ROOT), "per": "160-slice forward (one step of this leg)",
                                       "kind": "constant from a rocprofv3 --pmc collection (FETCH_SIZE doubled per the gfx950 "
                                               "correction + WRITE_SIZE), not re-measured by this run",
                                       "kernel_source_sha1": sha,
                                       "stale": (sha != _unet_source_sha1()) if sha else None}}
    return {"traffic": None, **base}


def bench_cfg5(L, lib, torch, qd, device, local_rank, rank, world, args, vol0):
    """BASELINE.json configs[4] / SURVEY 8(d) cfg5: a batch of knee volumes (512x512x160 x 8 echoes), 8 per GPU
    (64 at N = 8), per volume the mono-exponential fit + the UNet2D segmentation of one 512x512x160 channel, sharded on
    the batch axis by dosma_amd.dist.run_batch (volume v -> rank v mod world, no collective on the data path).
    The UNet weights are created on rank 0 only and reach the other ranks through ONE broadcast (RCCL over xGMI).
    Host feed: the volumes are generated on-device from seeds and are resident in HBM before the clock starts
    (86 GB of fp32 input at N = 8 would otherwise come over PCIe); the host-fed rate of ONE volume per rank through the
    host entry -- all ranks at once, so host memory bandwidth is shared like in a real N-GPU run -- is `host_feed`."""
    from dosma_amd.models import weights as W

    per_gpu = args.cfg5_volumes_per_gpu
    n_vol = per_gpu * world
    n = vol0.shape[1]
    H = W_ = 512
    S = 160
    # ---- weights: rank 0's values everywhere ----
    t0 = time.perf_counter()
    wts = W.random_weights(seed=0 if rank == 0 else 1000 + rank)  # other ranks: same shapes, different values
    t_make = time.perf_counter() - t0
    t0 = time.perf_counter()
    wts = qd.broadcast_weights(wts, src=0)
    t_bcast = time.perf_counter() - t0
    checksum = float(sum(float(np.asarray(v, dtype=np.float64).sum()) for v in wts.values()))
    import zlib

    crc = 0
    for k in sorted(wts):  # every byte of every tensor, in name order (a CRC-32 is exact in a float64)
        crc = zlib.crc32(np.ascontiguousarray(wts[k]).tobytes(), crc)
    gathered = qd.allgather_scalars([checksum, float(crc)])
    sums, crcs = gathered[:, 0], gathered[:, 1]
    wbytes = int(sum(np.asarray(v).size for v in wts.values()) * 4)
    eng = L.Unet2dEngine(W.to_abi_order(wts), H, W_, max_batch=args.cfg5_unet_batch, precision=UNET_PARITY_MODE,
                         device=local_rank)
    stream = torch.cuda.current_stream(device)
    popt = torch.empty((n, 2), dtype=torch.float32, device=device)
    r2 = torch.empty(n, dtype=torch.float32, device=device)
    mask = torch.empty((S, H, W_, 4), device=device, dtype=torch.uint8)
    vols = {}

    def setup(mine):
        for v in mine:  # resident in HBM before the timed region (on-device generation from the volume's seed)
            vols[v] = vol0 if v == rank else make_volume(torch, device, 20260928 + v)
        torch.cuda.synchronize(device)

    def per_volume(v):
        y = vols[v]
        t = time.perf_counter()
        a = make_args(L, y, popt, r2, stream.cuda_stream, "A")
        a.device = local_rank
        L.check(lib.qmri_monoexp_fit_device(ctypes.byref(a), None))
        torch.cuda.synchronize(device)
        t_fit = time.perf_counter() - t
        t = time.perf_counter()
        # one 512 x 512 x 160 channel of the volume (echo 1), as 160 slices of 512 x 512 (the flat echo row
        # reinterpreted: synthetic voxels carry no geometry), whole-volume whitening like IWOAIOAIUnet2DNormalized
        eng.forward_device(y[0].data_ptr(), S, None, mask.data_ptr(), whiten=True, stream=stream.cuda_stream)
        torch.cuda.synchronize(device)
        t_seg = time.perf_counter() - t
        fitted = float((popt[:, 1] > 0).sum().item())
        return {"fit_s": t_fit, "seg_s": t_seg, "voxels": float(n), "slices": float(S), "t2_nonzero": fitted,
                "mask_voxels": float(mask[..., 0].sum().item()), "owner_rank": float(rank), "volume_index": float(v)}

    # The same batch with the two pipes overlapped: the fit is fp64 VALU at three waves per SIMD, the network
    # MFMA at one -- independent calls in the reference (qdess.py:64-103 segmentation, cube_quant.py:139-185 fit).  Volume v + 1's fit
    # is launched on a second stream (its own result buffers) before volume v's segmentation is; no collective, per rank.
    side = torch.cuda.Stream(device)
    popt2 = torch.empty((n, 2), dtype=torch.float32, device=device)
    r22 = torch.empty(n, dtype=torch.float32, device=device)

    def overlapped(mine):
        res = {}
        bufs = [(popt, r2), (popt2, r22)]
        done = [torch.cuda.Event(), torch.cuda.Event()]

        def launch_fit(i):
            a = make_args(L, vols[mine[i]], bufs[i & 1][0], bufs[i & 1][1], side.cuda_stream, "A")
            a.device = local_rank
            L.check(lib.qmri_monoexp_fit_device(ctypes.byref(a), None))
            done[i & 1].record(side)

        if mine:
            launch_fit(0)
        for i, v in enumerate(mine):
            t = time.perf_counter()
            if i + 1 < len(mine):
                launch_fit(i + 1)  # (its buffers: read two volumes ago, by the .item() below)
            eng.forward_device(vols[v][0].data_ptr(), S, None, mask.data_ptr(), whiten=True, stream=stream.cuda_stream)
            done[i & 1].synchronize()
            torch.cuda.synchronize(device) if i + 1 == len(mine) else None
            res[v] = {"fit_s": float("nan"), "seg_s": float("nan"), "voxels": float(n), "slices": float(S),
                      "t2_nonzero": float((bufs[i & 1][0][:, 1] > 0).sum().item()),
                      "mask_voxels": float(mask[..., 0].sum().item()), "owner_rank": float(rank), "volume_index": float(v),
                      "wall_s": time.perf_counter() - t}
        return res

    # warm-up (kernel module load, workspace allocation) on this rank's own volume, then the batch
    setup([rank])
    per_volume(rank)
    out = qd.run_batch(n_vol, per_volume, setup=setup)
    summ = out.pop("summary")
    ovl = qd.run_batch(n_vol, per_volume, setup=setup, pipelined=overlapped)
    osumm = ovl.pop("summary")
    same = bool(np.array_equal(osumm["t2_nonzero"], summ["t2_nonzero"]) and np.array_equal(osumm["mask_voxels"], summ["mask_voxels"]))
    out["two_streams"] = {
        "what": "the same batch with volume v + 1's fit launched on a second HIP stream before volume v's segmentation "
                "(fp64 VALU kernel beside the MFMA kernels); reported beside cfg5's headline, which is always back to back",
        "wall_s": ovl["wall_s"], "volumes_per_s": ovl["volumes_per_s"], "speedup_vs_back_to_back": out["wall_s"] / ovl["wall_s"],
        "same_results": same, "back_to_back_wall_s": out["wall_s"], "back_to_back_volumes_per_s": out["volumes_per_s"],
        # the per-volume scalars both schedules are compared on (fitted voxels with tc > 0, voxels of the first class mask)
        "t2_nonzero": {"back_to_back": summ["t2_nonzero"].tolist(), "two_streams": osumm["t2_nonzero"].tolist()},
        "mask_voxels": {"back_to_back": summ["mask_voxels"].tolist(), "two_streams": osumm["mask_voxels"].tolist()},
    }
    # the headline (wall_s / volumes_per_s / the rates below) is ALWAYS the back-to-back schedule -- one fixed schedule
    # from run to run and box to box; the two-stream schedule is reported beside it under fixed keys and never replaces it
    out["schedule"] = "back_to_back"
    out.update({
        "config": f"{n_vol} volumes of 512x512x160 x 8 echoes: mono-exponential fit (MonoExponentialFit defaults) + UNet2D "
                  f"segmentation at 512x512 ({UNET_PARITY_MODE}) per volume, {per_gpu} volumes per GPU, fit and segmentation back to back "
                  f"on one stream (BASELINE configs[4])",
        "voxel_fits_per_s": float(np.nansum(summ["voxels"])) / out["wall_s"],
        "slices_per_s": float(np.nansum(summ["slices"])) / out["wall_s"],
        "fit_s_per_volume": float(np.nanmean(summ["fit_s"])), "seg_s_per_volume": float(np.nanmean(summ["seg_s"])),
        "unet_gflop_per_slice_512": UNET_GFLOP_PER_SLICE * (512 / 384) ** 2,
        "host_feed_note": "inputs generated on-device from per-volume seeds, resident in HBM before the clock starts",
        # which rank ran which volume (gathered after the clock): every index 0 .. n_vol - 1 owned by exactly one rank
        "volume_owner": [None if np.isnan(r) else int(r) for r in summ["owner_rank"]],
        "every_volume_once": bool(np.array_equal(summ["volume_index"], np.arange(n_vol)) and sum(out["per_rank"]) == n_vol
                                  and all((not np.isnan(r)) and int(r) == v % world for v, r in enumerate(summ["owner_rank"]))),
        "weights_broadcast": {"bytes": wbytes, "seconds": t_bcast, "make_seconds_rank0": t_make,
                              "identical_on_all_ranks": bool(np.all(sums == sums[0]) and np.all(crcs == crcs[0])),
                              "crc32_per_rank": [int(c) for c in crcs],
                              "collective": "one torch.distributed.broadcast of the packed fp32 weights (RCCL) from rank 0"},
    })
    eng.close()
    # ---- host-fed rate: one volume per rank through the host entry (pageable numpy in, numpy out), all ranks at once
    y_host = [vol0[e].cpu().numpy() for e in range(E)]

    def host_fed(rows):
        walls, per_rank = [], None
        for _ in range(2):  # first call: the result blocks are allocated (page-locked); second: served from the free list
            qd.barrier()
            t0 = time.perf_counter()
            res = L.monoexp_fit_host(TE, rows, p0=P0_A, want_tc=True, want_popt=False,
                                     post=dict(inv_abs_b=True, bounds=((-np.inf, np.inf), (0.0, 100.0)), r2_threshold=0.9,
                                               nan_to_num=0.0, decimals=1), device=local_rank)
            mine = time.perf_counter() - t0
            qd.barrier()
            walls.append(qd.allreduce_max(time.perf_counter() - t0))
            per_rank = qd.allgather_scalars([mine])[:, 0]
            del res
        return walls, per_rank

    walls, per_rank = host_fed(y_host)
    # the dtype scanners produce: DICOM pixel data is int16 / uint16, and the reference keeps the volumes' dtype up to scipy
    # (fitting.py:194-196); the ABI takes it as it is (converted on load in the kernel) at half the upload of float32
    y_host16 = [np.clip(np.rint(v), -32768, 32767).astype(np.int16) for v in y_host]
    walls16, per_rank16 = host_fed(y_host16)
    del y_host16
    # host <-> device copy bandwidth per rank, every rank copying at the same time: what bounds the host-fed rate of an
    # N-GPU node (each rank moves 1.34 GB up + 0.67 GB down per volume through ONE host memory system)
    up_host = np.concatenate([v.reshape(-1) for v in y_host])           # 1.34 GB pageable
    down_dev = torch.empty(2 * n, dtype=torch.float64, device=device)   # 0.67 GB
    down_host = np.empty(2 * n, dtype=np.float64)
    down_host[:] = 0                                                    # pages resident: measure the copy, not the zero-fill
    up_dev = torch.empty(up_host.size, dtype=torch.float32, device=device)
    copy_bw = {}
    for name, fn, nbytes in (("h2d", lambda: up_dev.copy_(torch.from_numpy(up_host)), up_host.nbytes),
                             ("d2h", lambda: torch.from_numpy(down_host).copy_(down_dev), down_host.nbytes)):
        fn()
        torch.cuda.synchronize(device)
        qd.barrier()
        t0 = time.perf_counter()
        fn()
        torch.cuda.synchronize(device)
        mine = time.perf_counter() - t0
        secs = qd.allgather_scalars([mine])[:, 0]
        copy_bw[name] = {"bytes_per_rank": int(nbytes), "gb_per_s_per_rank": (nbytes / secs / 1e9).tolist(),
                         "gb_per_s_all_ranks": float(nbytes * world / secs.max() / 1e9)}
    del up_dev, down_dev, up_host, down_host
    host_bytes = 4 * E * n + 16 * n   # per volume and rank through the host entry: samples up, tc + r2 (float64) down
    out["host_feed"] = {
        "what": "qmri_monoexp_fit_host on one 512x512x160x8 float32 volume per rank (1.34 GB of pageable numpy up, tc + r2 "
                "float64 = 0.67 GB down into result arrays from dosma_amd/_hostpool.py: page-locked blocks recycled when the "
                "caller drops a result), every rank at the same time; wall_s = the steady state (second call), "
                "first_call_wall_s includes allocating the blocks",
        "seconds_per_rank": per_rank.tolist(), "wall_s": walls[1], "first_call_wall_s": walls[0],
        "voxel_fits_per_s": n * world / walls[1],
        "host_bytes_per_rank": host_bytes,
        "host_traffic_gb_per_s_all_ranks": host_bytes * world / walls[1] / 1e9,
        "int16": {"what": "the same volume rounded to int16 (what DICOM holds; configs[2]'s dtype): 0.67 GB up instead of 1.34",
                  "seconds_per_rank": per_rank16.tolist(), "wall_s": walls16[1], "first_call_wall_s": walls16[0],
                  "voxel_fits_per_s": n * world / walls16[1],
                  "host_bytes_per_rank": 2 * E * n + 16 * n,
                  "host_traffic_gb_per_s_all_ranks": (2 * E * n + 16 * n) * world / walls16[1] / 1e9},
        "copy_bandwidth": copy_bw,
        "copy_bandwidth_note": "pageable numpy <-> device copies of the same sizes, all ranks at once (resident pages): "
                               "gb_per_s_all_ranks is the node-level host traffic these copies sustain at this N -- the "
                               "ceiling of the host-fed rate; the device-resident headline does not depend on it",
    }
    return out


def _launch_ranks(n: int) -> int:
    """Re-run this command as n ranks under `python -m torch.distributed.run --nnodes=1 --nproc-per-node n` (what the
    driver's own multi-GPU command line is) and return the launcher's exit code.  stdout / stderr are inherited: the
    single JSON line rank 0 prints is this process's output."""
    import socket
    import subprocess

    with socket.socket(socket.AF_INET, socket.SOCK_STREAM) as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    env = dict(os.environ)
    env.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")  # dmabuf IPC only on these hosts (RCCL needs it)
    env.setdefault("OMP_NUM_THREADS", "1")
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={n}",
           "--master-addr", "127.0.0.1", "--master-port", str(port), os.path.abspath(__file__)] + sys.argv[1:]
    return subprocess.call(cmd, env=env)


def _kernel_source_sha1():
    return _source_sha1(("monoexp_lm.hip", "fp64_fast.h", "qmri_internal.h"))


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--recipes", default="B,A", help="which recipes to time (A = headline, last)")
    ap.add_argument("--no-unet", action="store_true", help="skip the UNet2D slices/s leg")
    ap.add_argument("--no-cfg5", action="store_true", help="skip the BASELINE configs[4] batch (8 volumes per GPU: fit + seg)")
    ap.add_argument("--no-parity", action="store_true", help="skip the post-run parity sample")
    ap.add_argument("--unet-batch", type=int, default=160,
                    help="slices per pass through the network (default: the whole 160-slice volume)")
    ap.add_argument("--cfg5-volumes-per-gpu", type=int, default=8)
    ap.add_argument("--cfg5-unet-batch", type=int, default=160)
    ap.add_argument("--force-dist", action="store_true",
                    help="create the torch.distributed group also for ONE rank (the RCCL calls of an N-GPU run on a 1-GPU box); "
                         "implied when launched by torch.distributed.run")
    ap.add_argument("--print-kernel-hash", action="store_true")
    ap.add_argument("--print-unet-hash", action="store_true")
    args = ap.parse_args()
    if args.print_kernel_hash:
        print(_kernel_source_sha1())
        return
    if args.print_unet_hash:
        print(_unet_source_sha1())
        return

    from dosma_amd import _lib as L

    lib = L.load()
    import torch
    import torch.distributed as dist

    from dosma_amd import dist as qd

    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local_rank = int(os.environ.get("LOCAL_RANK", "0"))
    if world != args.gpus:
        if "WORLD_SIZE" not in os.environ and args.gpus > 1:
            # plain `python bench.py --gpus N`: become the launcher -- N ranks of this very command under
            # torch.distributed.run (one per GPU, rendezvous on 127.0.0.1 at a free port); rank 0's JSON line is the
            # children's stdout, the exit code is the launcher's
            raise SystemExit(_launch_ranks(args.gpus))
        raise SystemExit(f"--gpus {args.gpus} but WORLD_SIZE={world}: launch one rank per GPU "
                         f"(python bench.py --gpus N launches them itself)")
    # QMRI_BENCH_BACKEND=gloo lets the N > 1 code path be exercised on a box with fewer GPUs than ranks
    # (ranks then share devices); the real runs use nccl (= RCCL over xGMI), one rank per GPU.
    backend = os.environ.get("QMRI_BENCH_BACKEND", "nccl")
    ndev = torch.cuda.device_count()
    dev_index = local_rank if backend == "nccl" else local_rank % max(ndev, 1)
    torch.cuda.set_device(dev_index)
    device = torch.device("cuda", dev_index)
    red_device = device if backend == "nccl" else torch.device("cpu")
    # the process group exists whenever torch.distributed.run launched us (any N, one included) or --force-dist is given:
    # every `dist.` call below then goes through RCCL exactly as it will at N = 8
    use_dist = world > 1 or args.force_dist or qd.launched_by_torchrun()
    if use_dist:
        os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
        os.environ.setdefault("MASTER_PORT", "29500")
        if backend == "nccl":
            dist.init_process_group("nccl", rank=rank, world_size=world, device_id=device)
        else:
            dist.init_process_group(backend, rank=rank, world_size=world)
    local_rank = dev_index
    L.set_default_device(local_rank)

    y = make_volume(torch, device, 20260928 + rank)
    n = y.shape[1]
    popt = torch.empty((n, 2), dtype=torch.float32, device=device)
    r2 = torch.empty(n, dtype=torch.float32, device=device)
    stream = torch.cuda.current_stream(device)

    def barrier():
        torch.cuda.synchronize(device)
        if use_dist:
            dist.barrier()
        torch.cuda.synchronize(device)

    fit_sampler = GpuSampler(torch, local_rank)

    def timed_fit(a):
        for _ in range(args.warmup):
            L.check(lib.qmri_monoexp_fit_device(ctypes.byref(a), None))
        ev0 = torch.cuda.Event(enable_timing=True)
        ev1 = torch.cuda.Event(enable_timing=True)
        barrier()
        with fit_sampler:
            t0 = time.perf_counter()
            ev0.record(stream)
            for _ in range(args.steps):
                L.check(lib.qmri_monoexp_fit_device(ctypes.byref(a), None))
            ev1.record(stream)
            barrier()
            t1 = time.perf_counter()
        elapsed = t1 - t0
        clocks = fit_sampler.summary(t0, t1)
        kernel_ms = ev0.elapsed_time(ev1) / args.steps  # HIP events on the launch stream
        if use_dist:
            t = torch.tensor([elapsed, kernel_ms], device=red_device, dtype=torch.float64)
            dist.all_reduce(t, op=dist.ReduceOp.MAX)
            elapsed, kernel_ms = t[0].item(), t[1].item()
        return dict(elapsed=elapsed, kernel_ms=kernel_ms, kernel=lib.qmri_monoexp_kernel_name(ctypes.byref(a)).decode(), clocks=clocks)

    results = {}
    # float64 outputs (what the drop-in API returns: 56 B/voxel) first, the headline (fp32 outputs) last so that the
    # parity check below reads the headline's own output buffers
    popt64 = torch.empty((n, 2), dtype=torch.float64, device=device)
    r264 = torch.empty(n, dtype=torch.float64, device=device)
    a64 = make_args(L, y, popt64, r264, stream.cuda_stream, "A", out_dtype=L.QMRI_F64)
    a64.device = local_rank
    results["A_f64"] = timed_fit(a64)
    del popt64, r264
    for recipe in args.recipes.split(","):  # A last: it is the headline
        a = make_args(L, y, popt, r2, stream.cuda_stream, recipe)
        a.device = local_rank
        results[recipe] = timed_fit(a)

    parity = None
    if rank == 0 and not args.no_parity and args.recipes.split(",")[-1] == "A":
        parity = parity_sample(L, torch, y, popt, r2)

    roi_run = bench_t1rho_roi(L, lib, torch, device, local_rank, args) if rank == 0 else None
    dess = bench_dess(L, lib, torch, device, local_rank, world, args, barrier) if rank == 0 or world > 1 else None
    unet = None
    if not args.no_unet:
        unet = bench_unet(L, torch, dist, device, local_rank, world, args, barrier, red_device)
    cfg5 = None
    if not args.no_cfg5:
        cfg5 = bench_cfg5(L, lib, torch, qd, device, local_rank, rank, world, args, y)

    if rank == 0:
        ra = results["A"]
        total_voxels = n * world * args.steps
        value = total_voxels / ra["elapsed"]
        achieved = BYTES_PER_VOXEL * n / (ra["kernel_ms"] * 1e-3) / 1e9
        # HBM traffic and VALU lane-instructions per launch are rocprofv3 PMC results (separate passes: gpurun refuses
        # counters + tracing in one run), collected by scripts/collect_profile.sh and reduced by
        # scripts/summarize_profile.py into profiles/<round>_hbm_traffic.json together with the hash of the kernel
        # sources they were measured on; a kernel edit makes them "stale" here instead of silently wrong
        traffic = valu_lane_instr = None
        traffic_src = None
        import glob
        for prof in sorted(glob.glob(os.path.join(ROOT, "profiles", "r0*_hbm_traffic.json")), reverse=True):
            name = os.path.basename(prof)
            if os.path.exists(prof):
                with open(prof) as f:
                    pj = json.load(f)
                traffic = pj.get("hbm_bytes_per_launch")
                valu_lane_instr = pj.get("valu_lane_instr_per_launch")
                sha = pj.get("kernel_source_sha1")
                traffic_src = {"file": f"profiles/{name}", "counters": pj.get("source"),
                               "kind": "constant from a rocprofv3 --pmc collection (not re-measured by this run)",
                               "stale": (sha != _kernel_source_sha1()) if sha else None, "pmc": pj.get("pmc")}
                break
        # the bound that actually binds: vector-ALU issue.  Peak = 256 CUs x 4 SIMDs x 16 lanes/clk x 2.4 GHz lane-
        # instructions/s (an fp64 FMA on every lane every clock = the 78.6 TFLOP/s vector fp64 figure); achieved = the
        # kernel's active lane-instructions per launch (rocprofv3 PMC, SQ_INSTS_VALU x lanes active per instruction)
        # over the launch duration measured here
        valu_peak = 256 * 4 * 16 * 2.4e9
        valu_rate = valu_lane_instr / (ra["kernel_ms"] * 1e-3) if valu_lane_instr else None
        solved = int((y != 0).any(dim=0).sum().item())
        out = {
            "metric": "voxel-fits/sec (8-echo monoexp, 512x512x160) [+ UNet2D slices/sec under \"unet2d\"]",
            "value": value,
            "unit": "voxel-fits/s",
            # `value` counts every voxel of the volume, including the ~30 % all-zero background the reference's skip
            # rule (fitting.py:1065-1067) retires without a solve; this is the rate over the voxels that ran the solver
            "solved_voxel_fits_per_s": value * solved / n,
            "n_gpus": world,
            "process_group": ({"backend": dist.get_backend(), "world_size": dist.get_world_size(),
                               "collectives_on": str(red_device)} if use_dist else None),
            "steps": args.steps,
            "warmup": args.warmup,
            "ms_per_step": ra["elapsed"] / args.steps * 1e3,
            "higher_is_better": True,
            "scaling": "weak",
            "vs_baseline": None,
            "dtype": "f64",
            "data": "synthetic",
            "config": {
                "workload": "T2 monoexponential fit, 512x512x160 x 8 echoes, fp32 samples "
                            "(BASELINE.json configs[1]); MonoExponentialFit() defaults; "
                            "one volume per GPU per step",
                "voxels_per_gpu_per_step": n,
                "solved_voxels_per_gpu_per_step": solved,
                "echoes": E,
                "parallelism": f"volumes sharded over {world} GPU(s), no data-path collective",
                "kernel": ra["kernel"],
            },
            "roofline": {
                "bound": "hbm",
                "achieved": achieved,
                "peak": HBM_PEAK_GBS,
                "unit": "GB/s",
                "frac": achieved / HBM_PEAK_GBS,
                "traffic": traffic,
                "traffic_source": traffic_src,
                "algorithmic_bytes_per_voxel": BYTES_PER_VOXEL,
                "sclk_ghz_mean": ra["clocks"].get("sclk_ghz_mean"), "power_w_mean": ra["clocks"].get("power_w_mean"),
                "clock_samples": ra["clocks"],
                "kernel_ms": ra["kernel_ms"],
                "note": "the kernel is fp64-VALU bound, not HBM bound: MINPACK's early-stopped trajectory is ~20 LM rounds "
                        "per voxel (53 charged model evaluations) of ~1000 fp64 VALU instructions each (lmpar, model "
                        "evaluation, ratio tests, forward-difference Jacobian + QR); see `valu` and DESIGN.md 3.1",
                "valu": {"lane_instr_per_launch": valu_lane_instr, "lane_instr_per_s": valu_rate,
                         "peak_lane_instr_per_s": valu_peak,
                         "frac_of_valu_peak": (valu_rate / valu_peak) if valu_rate else None,
                         "source": traffic_src},
            },
            "runs": {
                "A_defaults_fixed_p0": {"voxel_fits_per_s": n * world * args.steps / ra["elapsed"],
                                        "kernel_ms": ra["kernel_ms"]},
                "A_f64_outputs": {"voxel_fits_per_s": n * world * args.steps / results["A_f64"]["elapsed"],
                                  "kernel_ms": results["A_f64"]["kernel_ms"],
                                  "algorithmic_bytes_per_voxel": BYTES_PER_VOXEL_F64,
                                  "hbm_gb_per_s": BYTES_PER_VOXEL_F64 * n / (results["A_f64"]["kernel_ms"] * 1e-3) / 1e9,
                                  "note": "float64 (popt, r2) like the reference returns -- what the drop-in API uses"},
            },
        }
        if parity is not None:
            out["parity"] = parity
        if unet is not None:
            out["unet2d"] = unet
        if dess is not None:
            out["dess_t2"] = dess
        if cfg5 is not None:
            out["cfg5"] = cfg5
        if roi_run is not None:
            out["runs"]["cfg2_t1rho_roi"] = roi_run
        if "B" in results:
            out["runs"]["B_polyfit_init"] = {
                "voxel_fits_per_s": n * world * args.steps / results["B"]["elapsed"],
                "kernel_ms": results["B"]["kernel_ms"]}
        if world == 1 and not args.no_cpu_baseline:
            out["cpu_baseline"] = cpu_baseline(y)
        print(json.dumps(out))
    if use_dist:
        dist.barrier()
        dist.destroy_process_group()


if __name__ == "__main__":
    main()
