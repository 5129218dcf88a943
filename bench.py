#!/usr/bin/env python
"""Headline benchmark: images/sec of one full GAN training iteration (G+D fwd+bwd + both Adam steps) at
128x128 COCO-layout, per-GPU batch 32, bf16 MFMA operands (the reference loop
train_context_app_v2.py:148-189 with the VGG term omitted -- its weights cannot be downloaded here).

    python bench.py --gpus N --steps K --warmup W          (N > 1: launched by torch.distributed.run)

At N = 1 the iteration is captured once as a HIP graph and replayed (GanTrainer.capture); --no-graph runs eagerly.
Every timed step is the same thing (a replay, or an eager iteration); the latents z are drawn per iteration as the
reference does. The roofline leg's instrumented eager iteration runs behind the timed region.

Prints ONE JSON line on rank 0, including
  roofline     -- the implicit-GEMM conv kernel (forward + data-gradient launches): algorithmic FLOPs
                  (2*M*N*K of the unpadded layer shapes) / launch time measured with HIP events on the
                  launching stream (one eager iteration directly behind the timed region), against the 2.5 PFLOP/s dense
                  bf16 MFMA peak;
  cpu_baseline -- the oracle (pure-PyTorch restatement of the reference, oracle/model.py) timed on this
                  host's cores on a bounded sample (batch 4) of the same workload;
  f32_mode     -- the same iteration with exact-f32 operands (the mode that meets the L-inf < 1e-3 image bar), secondary.
"""
import argparse
import json
import os
import subprocess
import sys
import time

import torch

ROOT = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, ROOT)


def cpu_baseline(netG, netD, size, batch=32):
    """The oracle's training iteration on the host CPU (all cores), the SAME workload as the GPU line: one warm-up iteration at batch 4
    (thread pools, allocator), then ONE timed iteration at the line's own batch (batch 32 at 128x128: ~20 s on the GPU box's host).
    Returns images/sec."""
    from oracle import model as O
    from layout2img_amd.synthetic import make_batch
    threads = min(os.cpu_count() or 1, 32)  # (more threads than this slow the oracle down)
    torch.set_num_threads(threads)
    sd_g = O.make_trainable({k: v.detach().float().cpu() for k, v in netG.state_dict().items()})
    sd_d = O.make_trainable({k: v.detach().float().cpu() for k, v in netD.state_dict().items()})
    tr = O.OracleTrainer(sd_g, sd_d)
    tr.step(*make_batch(4, size, "coco", seed=98, device="cpu"))  # warm-up
    real, label, bbox, z, z_im = make_batch(batch, size, "coco", seed=99, device="cpu")
    t0 = time.time()
    tr.step(real, label, bbox, z, z_im)
    dt = time.time() - t0
    return dict(value=batch / dt, unit="images/sec", cores=threads, kind="port", batch=batch,
                sample=f"1 training iteration at batch {batch} (after a batch-4 warm-up), {size}x{size}, fp32, oracle/model.py OracleTrainer (VGG term omitted)")


TRAFFIC_FILE = "r06_conv_traffic.json"   # PMC passes of this round (tools/perf/traffic2.sh); absent -> roofline.traffic is null


RESULT_CHANGING_ENV = ("L2I_CONV_NOEPI", "L2I_WGRAD_NOEPI")   # ablation switches (results are wrong; -DL2I_ABLATIONS builds only)


def l2i_env():
    """Every L2I_* variable of this process: tuning / A-B switches change what is measured, so they are part of the line."""
    return {k: v for k, v in sorted(os.environ.items()) if k.startswith("L2I_")}


def refuse_wrong_result_switches():
    bad = [k for k in RESULT_CHANGING_ENV if os.environ.get(k, "0") not in ("", "0")]
    if "L2I_ABLATIONS" in os.environ.get("L2I_EXTRA_FLAGS", ""):
        bad.append("L2I_EXTRA_FLAGS=-DL2I_ABLATIONS")
    if bad:
        raise SystemExit("bench.py: refusing to print a headline with results-changing switches set: " + ", ".join(bad))


def g_forward_figures(netG, args, z, bbox, z_im, label, op_dtype):
    import torch
    from layout2img_amd.sampling import sample
    out = {}
    flop_img = 26.35e9 if (args.size == 128 and args.layout == "coco") else None
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                netG(z, bbox, z_im=z_im, y=label)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        fwd = lambda: netG(z, bbox, z_im=z_im, y=label)
        mode = "eager"
        if not args.no_graph:   # (a failed capture is not recoverable in-process: with --no-graph nothing is captured at all)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                netG(z, bbox, z_im=z_im, y=label)
            fwd, mode = graph.replay, "HIP graph replay"
        for _ in range(3):
            fwd()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        n = 30
        a.record()
        for _ in range(n):
            fwd()
        b.record()
        torch.cuda.synchronize()
        ms = a.elapsed_time(b) / n
        out.update(images_per_sec=round(args.batch / ms * 1e3, 1), ms=round(ms, 3), launch=mode)
        if flop_img:
            tf = flop_img * args.batch / (ms * 1e-3) / 1e12
            peak = 2500.0 if op_dtype == torch.bfloat16 else 157.3
            out.update(tflops=round(tf, 1), frac_of_mfma_peak=round(tf / peak, 4), gflop_per_image=26.35)
        # batch-1 sampling (eval mode, truncated latents drawn inside): the replayed graph of sampling.GraphSampler over the arena's
        # cached eval-mode packs (wall time per call, host side included); the eager call beside it
        lab1, box1 = label[:1], bbox[:1]
        for _ in range(3):
            sample(netG, lab1, box1)
        torch.cuda.synchronize()
        t1 = time.perf_counter()
        for _ in range(10):
            sample(netG, lab1, box1)
        torch.cuda.synchronize()
        out["sample_batch1_eager_ms"] = round((time.perf_counter() - t1) / 10 * 1e3, 3)
        out["sample_batch1_ms"] = out["sample_batch1_eager_ms"]
        if not args.no_graph:
            from layout2img_amd.sampling import GraphSampler
            gs = GraphSampler(netG)
            for _ in range(3):
                gs(lab1, box1)
            torch.cuda.synchronize()
            t1 = time.perf_counter()
            for _ in range(20):
                gs(lab1, box1)
            torch.cuda.synchronize()
            out["sample_batch1_ms"] = round((time.perf_counter() - t1) / 20 * 1e3, 3)
            out["sample_batch1_launch"] = "HIP graph replay (sampling.GraphSampler), cached eval-mode weight packs"
        # the same forward at larger batches (what a sampling service would run): at b = 32 most launches are a fraction of one
        # round of workgroups; these say what the kernels do once a launch fills the chip
        if args.g_batch_sweep and flop_img and op_dtype == torch.bfloat16:
            from layout2img_amd.synthetic import make_batch
            sweep = {}
            for bs in (128, 256):
                _, lab_b, box_b, z_b, zim_b = make_batch(bs, args.size, args.layout, seed=4321, device=z.device)
                zim_b = zim_b if z_im is not None else None
                for _ in range(2):
                    netG(z_b, box_b, z_im=zim_b, y=lab_b)
                torch.cuda.synchronize()
                fwd_b, mode_b = (lambda: netG(z_b, box_b, z_im=zim_b, y=lab_b)), "eager"
                if not args.no_graph:
                    gb = torch.cuda.CUDAGraph()
                    side.wait_stream(torch.cuda.current_stream())
                    with torch.cuda.graph(gb, stream=side):
                        netG(z_b, box_b, z_im=zim_b, y=lab_b)
                    fwd_b, mode_b = gb.replay, "HIP graph replay"
                for _ in range(2):
                    fwd_b()
                a.record()
                for _ in range(10):
                    fwd_b()
                b.record()
                torch.cuda.synchronize()
                ms_b = a.elapsed_time(b) / 10
                tf_b = flop_img * bs / (ms_b * 1e-3) / 1e12
                sweep[str(bs)] = {"ms": round(ms_b, 3), "images_per_sec": round(bs / ms_b * 1e3, 1), "tflops": round(tf_b, 1),
                                  "frac_of_mfma_peak": round(tf_b / 2500.0, 4), "launch": mode_b}
                del fwd_b
            out["batch_sweep"] = sweep
        if op_dtype == torch.bfloat16 and args.size == 128 and args.layout == "coco":
            out["precision_modes"] = precision_mode_figures(netG, args, z, bbox, z_im, label, ms)
    return out


def precision_mode_figures(netG, args, z, bbox, z_im, label, ms_bf16):
    """The generator forward (same weights, same inputs, eval mode) in the two modes that meet the north star's image bar
    L_inf < 1e-3 -- exact-f32 MFMA operands, and "bf16x3" (bf16 operands carried as hi + lo, three MFMA products per pair) --
    timed eagerly, with each mode's measured L_inf against the exact-f32 mode's image (which is within 9.4e-6 of the reference,
    tests/test_gpu_00_models.py). Secondary figures: never `value`."""
    import layout2img_amd as L
    dev = z.device
    nets = {}
    for name, dt in (("f32", torch.float32), ("bf16x3", "bf16x3")):
        g = L.ResnetGenerator128_context(num_classes=184)
        g.load_state_dict({k: v.detach().cpu().clone() for k, v in netG.state_dict().items()})
        nets[name] = g.finalize(dev, dt).eval()
    was_training = netG.training
    netG.eval()
    imgs, res = {}, {}
    with torch.no_grad():
        for name, g in (("bf16", netG), ("f32", nets["f32"]), ("bf16x3", nets["bf16x3"])):
            for _ in range(2):
                img = g(z, bbox, z_im=z_im, y=label)
            torch.cuda.synchronize()
            t0, n = time.perf_counter(), 5
            for _ in range(n):
                img = g(z, bbox, z_im=z_im, y=label)
            torch.cuda.synchronize()
            imgs[name] = img
            res[name] = dict(ms=round((time.perf_counter() - t0) / n * 1e3, 3), launch="eager, eval mode")
    netG.train(was_training)
    for name in ("bf16", "bf16x3"):
        res[name]["image_linf_vs_f32_mode"] = float((imgs[name] - imgs["f32"]).abs().max())
    res["f32"]["image_linf_vs_reference"] = "9.4e-6 (tests/test_gpu_00_models.py::test_generator_coco_vs_reference[f32])"
    res["bar"] = 1e-3
    return res


def f32_mode_figures(args, dev, real, label, bbox, steps=4):
    """images/s of the same iteration with exact-f32 MFMA operands (157.3 TFLOP/s peak), fresh networks, eager."""
    import layout2img_amd as L
    torch.manual_seed(4321)
    g = L.ResnetGenerator128_context(num_classes=184).finalize(dev, torch.float32)
    d = L.CombineDiscriminator128_app(num_classes=184).finalize(dev, torch.float32)
    g.train(), d.train()
    tr = L.GanTrainer(g, d)
    for _ in range(2):
        tr.step(real, label, bbox, None, None)
    tr.flush()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(steps):
        tr.step(real, label, bbox, None, None)
    tr.flush()
    torch.cuda.synchronize()
    dt = time.perf_counter() - t0
    return dict(images_per_sec=round(args.batch * steps / dt, 1), ms_per_step=round(1e3 * dt / steps, 2), steps=steps, launch="eager",
                dtype="f32", image_linf_vs_reference="9.4e-6 (tests/test_gpu_00_models.py, bar 1e-3)")


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--batch", type=int, default=32, help="per-GPU batch")
    ap.add_argument("--size", type=int, default=128)
    ap.add_argument("--dtype", default="bf16", choices=["bf16", "f32"])
    ap.add_argument("--layout", default="coco", choices=["coco", "vg"],
                    help="coco: BASELINE config 3/4 (o = 8, 184 classes, ResnetGenerator128_context); "
                         "vg: config 5 (o = 31, 179 classes, context_aware_generator)")
    ap.add_argument("--vgg", action="store_true", help="add the VGG19 perceptual term to the G loss (random-init VGG weights; "
                    "not part of the headline metric, which omits it on both sides)")
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--no-kernel-timer", action="store_true")
    ap.add_argument("--no-g-forward", action="store_true", help="skip the secondary generator-forward measurement (profiling runs)")
    ap.add_argument("--g-batch-sweep", action="store_true",
                    help="also time the generator forward at batch 128 / 256 (g_forward.batch_sweep); off by default so that the default "
                         "command's kernel statistics hold the batch-32 launches only")
    ap.add_argument("--no-f32-mode", action="store_true", help="skip the secondary exact-f32 operand-mode measurement")
    ap.add_argument("--graph-iters", type=int, default=4,
                    help="iterations per graph replay (N = 1 GPU): a second graph of this many consecutive iterations carries the timed steps "
                         "(steps %% n run on the one-iteration graph); 1 = one iteration per replay")
    ap.add_argument("--no-graph", action="store_true", help="run every iteration eagerly (default: replay a captured HIP graph at N=1)")
    args = ap.parse_args()
    refuse_wrong_result_switches()

    if args.gpus > 1 and "WORLD_SIZE" not in os.environ:
        # `python bench.py --gpus N` without a launcher: re-launch this script as N ranks (one process per GPU) under
        # torch.distributed.run on this node and pass the ranks' output through (rank 0 prints the JSON line).
        import socket
        with socket.socket() as sk:
            sk.bind(("127.0.0.1", 0))
            port = sk.getsockname()[1]
        cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={args.gpus}",
               "--master-addr", "127.0.0.1", "--master-port", str(port), os.path.abspath(__file__)] + sys.argv[1:]
        raise SystemExit(subprocess.call(cmd))

    import torch.distributed as dist
    import layout2img_amd as L
    from layout2img_amd import ops, parallel
    from layout2img_amd.synthetic import make_batch

    rank, world, local = parallel.init_from_env()
    if world != args.gpus:
        raise SystemExit(f"--gpus {args.gpus} but WORLD_SIZE={world}: launch with torch.distributed.run --nproc-per-node {args.gpus}")
    torch.cuda.set_device(local)
    dev = torch.device("cuda", local)
    op_dtype = torch.bfloat16 if args.dtype == "bf16" else torch.float32

    torch.manual_seed(1234)
    if args.size == 64:   # BASELINE configs 1-2 (not the headline metric)
        netG = L.ResnetGenerator64_context(num_classes=184).finalize(dev, op_dtype)
        netD = L.CombineDiscriminator64(num_classes=184).finalize(dev, op_dtype)
    elif args.layout == "vg":   # BASELINE config 5 (not the headline metric)
        netG = L.context_aware_generator(num_classes=179).finalize(dev, op_dtype)
        netD = L.CombineDiscriminator128_app(num_classes=179).finalize(dev, op_dtype)
    else:
        netG = L.ResnetGenerator128_context(num_classes=184).finalize(dev, op_dtype)
        netD = L.CombineDiscriminator128_app(num_classes=184).finalize(dev, op_dtype)
    netG.train(), netD.train()
    if "L2I_CONV_CFG" in os.environ:   # tuning hook (tools/perf): force a conv tile configuration
        from layout2img_amd import _lib
        _lib.call("l2i_set_conv_config", int(os.environ["L2I_CONV_CFG"]))
    vgg = L.VGGLoss().finalize(dev, op_dtype) if args.vgg else None
    trainer = L.GanTrainer(netG, netD, vgg=vgg)
    real, label, bbox, z, z_im = make_batch(args.batch, args.size, args.layout, seed=1234 + rank, device=dev)
    # real ROIs / ROI slots of this batch (read once, outside the timed region): launches over the ROI heads are limited to
    # the real ROIs by a device-side count, and the roofline leg credits them with the work on those rows only
    ops.LIVE_IMAGE_FRACTION = float((label != 0).sum()) / label.numel()

    def sync():
        torch.cuda.synchronize()
        if world > 1:
            dist.barrier()
        torch.cuda.synchronize()

    # The iteration is ~800 launches and costs the host nearly as long as the GPU: at N = 1 the whole iteration (both
    # forwards, both backwards, both Adam steps, and the draw of the latents z, which the reference draws per iteration --
    # train_context_app_v2.py:165) is captured once as a HIP graph and replayed. Every timed step is a replay; the roofline
    # leg's HIP-event-instrumented eager iteration runs AFTER the clock is read (round 3 ran it as the last timed step and
    # under-reported the steady state by ~8 % at --steps 20).
    graphed = False
    if (world == 1 or os.environ.get("L2I_DDP_GRAPH", "0") == "1") and not args.no_graph:   # (N > 1: opt-in, see GanTrainer.capture)
        try:
            graphed = trainer.capture(real, label, bbox, None)
        except Exception as e:
            # A capture that was invalidated leaves the HIP runtime and torch's generator in a sticky error state (probed:
            # tools/parity/capture_failure_probe.py -- every later launch in the process fails), so "stay on the eager path" has
            # to mean a fresh process: re-run this command with --no-graph (one GPU; a rank of a multi-process job cannot), as a child whose
            # exit code becomes this process's (a process that holds the GPU is not replaced; its own teardown is skipped, the runtime being unusable).
            print(f"[bench] graph capture unavailable ({type(e).__name__}: {str(e)[:200]}); re-running eagerly (--no-graph)", file=sys.stderr, flush=True)
            if world > 1:
                raise
            os._exit(subprocess.call([sys.executable, os.path.abspath(__file__)] + sys.argv[1:] + ["--no-graph"]))
    # n iterations per replay: the ~0.3 ms a graph launch costs on top of its kernels is paid once per n iterations (GanTrainer.capture_multi)
    n_multi = args.graph_iters if (graphed and world == 1 and args.graph_iters > 1) else 1
    if n_multi > 1:
        try:
            if not trainer.capture_multi([(real, label, bbox, None)] * n_multi):
                n_multi = 1
        except Exception as e:   # (sticky, as above: a fresh process with one iteration per replay)
            print(f"[bench] multi-iteration capture unavailable ({type(e).__name__}: {str(e)[:200]}); re-running with --graph-iters 1", file=sys.stderr, flush=True)
            os._exit(subprocess.call([sys.executable, os.path.abspath(__file__)] + sys.argv[1:] + ["--graph-iters", "1"]))
    step = (lambda: trainer.step_graphed(real, label, bbox, None)) if graphed else (lambda: trainer.step(real, label, bbox, None, None))
    multi = [(real, label, bbox, None)] * n_multi

    def run_steps(k):   # EXACTLY k iterations: k // n replays of the n-iteration graph, the rest on the one-iteration graph / eagerly
        for _ in range(k // n_multi if n_multi > 1 else 0):
            trainer.step_graphed_multi(multi)
        for _ in range(k % n_multi if n_multi > 1 else k):
            step()
    run_steps(args.warmup)
    sync()
    t0 = time.perf_counter()
    run_steps(args.steps)
    trainer.flush()   # (data parallel: the last iteration's deferred generator all-reduce + Adam belong to the timed region)
    torch.cuda.synchronize()
    local = time.perf_counter() - t0   # this rank's own K steps, before the closing barrier: a straggler shows up in the spread below
    sync()
    elapsed = time.perf_counter() - t0
    t = torch.tensor([elapsed], device=dev, dtype=torch.float64)
    rank_ms = None
    if world > 1:
        dist.all_reduce(t, op=dist.ReduceOp.MAX)
        lo = torch.tensor([local], device=dev, dtype=torch.float64)
        hi = lo.clone()
        dist.all_reduce(lo, op=dist.ReduceOp.MIN)
        dist.all_reduce(hi, op=dist.ReduceOp.MAX)
        rank_ms = {"min": round(1e3 * float(lo) / args.steps, 3), "max": round(1e3 * float(hi) / args.steps, 3),
                   "note": "per-rank ms per step up to the rank's own device synchronisation, before the closing barrier"}
    elapsed = float(t)
    if not args.no_kernel_timer:
        # roofline leg: ONE eager iteration on one stream with HIP events on every conv / weight-gradient dispatch, right behind
        # the timed region (same process, same batch, same weights' shapes); a first eager iteration warms the allocator.
        # (data parallel: every rank runs the two iterations -- they carry collectives -- rank 0 instruments its own)
        ov, trainer.overlap = trainer.overlap, False   # one stream: a launch is timed while it owns the GPU
        trainer.step(real, label, bbox, None, None)
        trainer.flush()
        torch.cuda.synchronize()
        if rank == 0:
            ops.TIMER = ops.KernelTimer()
        trainer.step(real, label, bbox, None, None)
        trainer.flush()
        torch.cuda.synchronize()
        trainer.overlap = ov
    comm = None
    from layout2img_amd import parallel as _par
    if _par.active():
        # the collectives of ONE eager iteration (every rank runs it; they are collectives): how many, how many gradient bytes,
        # and for how long the issuing stream was held up by them (HIP events around every blocking collective / every wait)
        _par.CommStats.start()
        trainer.step(real, label, bbox, None, None)
        trainer.flush()
        comm = _par.CommStats.stop()
        comm["measured"] = "one eager iteration behind the timed region; exposed = stream time between HIP events around each blocking collective and each wait for an asynchronous one"
        comm["grad_groups"] = {"G": netG.arena.grad_groups["n"], "D": netD.arena.grad_groups["n"]} if trainer.g_opt.chunked else None
    if world > 1:
        dist.barrier()

    if rank == 0:
        roof = None
        if ops.TIMER is not None:
            s = ops.TIMER.summary()["conv_igemm"]
            peak = 2500.0 if op_dtype == torch.bfloat16 else 157.3
            ach = s["work"] / (s["ms"] * 1e-3) / 1e12
            # HBM bytes per launch from the PMC counters cannot be collected inside this process: they come from separate
            # rocprofv3 --pmc passes of this same command (tools/perf/traffic2.sh), committed under profiles/ with the commit
            # they were taken at; labelled as not measured in this run. null when no file of THIS round exists.
            traffic, traffic_src = None, None
            tpath = os.path.join(ROOT, "profiles", TRAFFIC_FILE)
            if op_dtype == torch.bfloat16 and args.size == 128 and args.layout == "coco" and not args.vgg and os.path.exists(tpath):
                tj = json.load(open(tpath))
                traffic = round(tj["conv(fwd+dgrad)"]["traffic_bytes_per_launch"])
                traffic_src = {"file": "profiles/" + TRAFFIC_FILE, "measured_in_run": False, "commit": tj.get("commit"),
                               "method": "rocprofv3 --pmc FETCH_SIZE x2, WRITE_SIZE; separate passes"}
            roof = dict(bound="mfma", kernel="l2i_conv2d_fwd launches (conv_halo2/3_kernel + conv_igemm_kernel), forward and data-gradient",
                        timing="HIP events attached to each dispatch (hipExtLaunchKernelGGL) on the launching stream, over one eager "
                               "iteration run directly behind the timed region (same process and batch; the timed steps are graph replays)",
                        achieved=round(ach, 2), peak=peak, unit="TFLOP/s", frac=round(ach / peak, 4), traffic=traffic,
                        traffic_unit="HBM bytes per launch", traffic_source=traffic_src,
                        algorithmic_bytes_per_launch=round(s["bytes"] / s["launches"]),
                        launches_per_step=s["launches"], kernels_per_step=s["kernels"], timed_steps=1, live_roi_fraction=round(ops.LIVE_IMAGE_FRACTION, 4),
                        avg_launch_us=round(1e3 * s["ms"] / s["launches"], 2),
                        gflop_per_launch=round(s["work"] / s["launches"] / 1e9, 3))
            w = ops.TIMER.summary().get("conv_wgrad")
            if w and w["launches"]:
                roof["wgrad_tflops"] = round(w["work"] / (w["ms"] * 1e-3) / 1e12, 2)
                roof["wgrad_frac"] = round(w["work"] / (w["ms"] * 1e-3) / 1e12 / peak, 4)
                roof["wgrad_launches_per_step"] = w["launches"]
            ops.TIMER.close()
            ops.TIMER = None
        # the eager iteration (python + autograd enqueue every launch): what layout2img_amd.train falls back to when it cannot
        # replay a graph (data parallel), measured OUTSIDE the timed region on a few iterations (kernel timer closed)
        eager = None
        if world == 1 and graphed:
            for _ in range(2):
                trainer.step(real, label, bbox, None, None)
            trainer.flush(); sync()
            te, ne = time.perf_counter(), 5
            for _ in range(ne):
                trainer.step(real, label, bbox, None, None)
            trainer.flush(); sync()
            te = time.perf_counter() - te
            eager = dict(images_per_sec=round(args.batch * ne / te, 1), ms_per_step=round(1e3 * te / ne, 3), steps=ne)
        # secondary figures of SURVEY section 8d: the generator forward alone (train-mode statistics, no autograd tape),
        # replayed as its own HIP graph, against the MFMA roofline (26.35 GFLOP per image), and the batch-1
        # sampling latency (test_context_app_v2.py:68-77)
        g_fwd = None
        if world == 1 and not args.no_g_forward:
            g_fwd = g_forward_figures(netG, args, z, bbox, z_im, label, op_dtype)
        # the exact-f32 operand mode (the mode that meets the north star's L-inf < 1e-3 image bar: 9.4e-6 measured) on the same
        # workload, timed eagerly on a few iterations: a secondary figure, never `value`
        f32_mode = None
        if world == 1 and args.dtype == "bf16" and not args.no_f32_mode and args.size == 128 and args.layout == "coco" and not args.vgg:
            f32_mode = f32_mode_figures(args, dev, real, label, bbox)
        cpu = None
        if not args.no_cpu_baseline and world == 1 and args.size == 128 and args.layout == "coco":
            cpu = cpu_baseline(netG, netD, args.size, args.batch)
        out = {
            "metric": f"images/sec (G+D fwd+bwd) at {args.size}x{args.size} {'COCO' if args.layout == 'coco' else 'VG'}-layout",
            "value": round(args.batch * world * args.steps / elapsed, 2),
            "unit": "images/sec",
            "n_gpus": world, "steps": args.steps, "warmup": args.warmup,
            "ms_per_step": round(1e3 * elapsed / args.steps, 3),
            "higher_is_better": True, "scaling": "weak", "vs_baseline": None,
            "dtype": args.dtype, "data": "synthetic",
            "config": {"workload": f"{args.size}x{args.size}, batch {args.batch}/GPU, "
                                   + ("COCO-stuff layouts (8 slots, 3-8 objects), ResnetGenerator128_context" if args.layout == "coco"
                                      else "VG layouts (31 slots, 3-30 objects), context_aware_generator")
                                   + " + CombineDiscriminator128_app, full D-step + G-step with Adam, "
                                   + ("VGG19 perceptual term included (random-init VGG)" if args.vgg else "VGG loss term omitted")
                                   + ", random-init weights",
                       "global_batch": args.batch * world, "parallelism": f"dp{world}",
                       "launch": ("HIP graph replay of the whole iteration incl. the draw of z (every timed step)" if graphed else "eager"),
                       "iterations_per_replay": n_multi},
            "roofline": roof, "env": l2i_env(), "comm": comm, "rank_ms_per_step": rank_ms,
            "cpu_baseline": cpu, "g_forward": g_fwd, "eager": eager, "f32_mode": f32_mode,
            "g_forward_images_per_sec": None if g_fwd is None else g_fwd["images_per_sec"],
        }
    if dist.is_initialized():   # (world > 1, or the forced one-rank group of L2I_FORCE_COLLECTIVES=1)
        dist.barrier()
        dist.destroy_process_group()
    if rank == 0:
        # RCCL writes its version banner to the C-level stdout, which is block-buffered when piped and would otherwise come out AFTER
        # this line at exit: flush the C streams first so that the JSON line is the LAST line of rank 0's stdout
        try:
            import ctypes
            ctypes.CDLL(None).fflush(None)
        except Exception:
            pass
        print(json.dumps(out), flush=True)


if __name__ == "__main__":
    main()
