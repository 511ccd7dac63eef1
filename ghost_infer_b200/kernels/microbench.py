"""Times one kernel at one shape with CUDA events and relates it to the roofline.

    python -m ghost_infer_b200.kernels.microbench --kernel gemm_stream --m 8 --n 28672 --k 4096
    python -m ghost_infer_b200.kernels.microbench --kernel attn_decode --batch 8 --context 2048

Kernels: gemm_stream, gemm_skinny (decode products), gemm_tc (prefill product), attn_decode, attn_prefill (mma.sync),
attn_prefill_t5 (tcgen05), attn_latent_decode, attn_latent_prefill (attention over one shared latent row per position:
--heads, --rank, --rot-dim),
linear_state, mamba2_scan (the token-by-token recurrences: --batch, --context, --heads, --kv-heads, --head-dim, --v-dim,
--delta), attn_tree (trees of --nodes drafted tokens behind --context positions), beam_select (--batch sequences of --beams beams over
--n tokens, --width candidates), rmsnorm, rope, sample.  Operands rotate through enough different buffers to exceed the L2 cache, so a bytes
figure is a DRAM figure.  The same command under `ncu --clock-control none -k regex:<kernel> -c 3` profiles exactly these launches.
The reference times whole runs only (`bench`, src/main.rs:1241-1285) and, per operation, wall-clock buckets
(src/profile.rs:7-46); per-kernel device timing is what a roofline needs.
"""
from __future__ import annotations

import argparse
import json
import os

import torch

from . import ops

L2_BYTES = 126 << 20


def _peaks():
    root = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    try:
        with open(os.path.join(root, "MEASURED_PEAKS.json")) as f:
            p = json.load(f)
        return float(p["hbm_gbs"]), float(p["bf16_tflops"]), "measured"
    except Exception:
        return 6650.0, 1590.0, "fallback"


def _time(fn, n_rot, iters, warmup):
    for i in range(warmup):
        fn(i % n_rot)
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    for i in range(iters):
        fn(i % n_rot)
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) * 1e3 / iters      # microseconds


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--kernel", required=True)
    ap.add_argument("--m", type=int, default=8)
    ap.add_argument("--n", type=int, default=4096)
    ap.add_argument("--k", type=int, default=4096)
    ap.add_argument("--mode", default="store", choices=["store", "accum", "swiglu", "f32"])
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--context", type=int, default=2048)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--head-dim", type=int, default=128)
    ap.add_argument("--rank", type=int, default=512, help="attn_latent_*: numbers of the latent (the values' width)")
    ap.add_argument("--rot-dim", type=int, default=64, help="attn_latent_*: numbers of the rotated key part behind the latent")
    ap.add_argument("--v-dim", type=int, default=0, help="linear_state, mamba2_scan: columns of a head's state (default: --head-dim)")
    ap.add_argument("--delta", type=int, default=0, help="linear_state: 1 = the gated delta rule (--kv-heads query/key heads), 0 = a constant decay")
    ap.add_argument("--splits", type=int, default=0)
    ap.add_argument("--own-tiles", type=int, default=0, help="attn_decode: slices of that many tiles of each sequence's own span")
    ap.add_argument("--tile-keys", type=int, default=0, help="attn_decode: 16 or 32 keys per tile (default: the engine's)")
    ap.add_argument("--merge-inside", type=int, default=-1, help="attn_decode: 1 = slices merged by the last block, 0 = by a second kernel")
    ap.add_argument("--tail", type=int, default=1, help="gemm_tc: 0 = full-width tiles only, 1 = narrower tiles in an unfilled last round")
    ap.add_argument("--stages", type=int, default=0, help="attn_decode: depth of each warp's ring of tiles (2 to 4)")
    ap.add_argument("--keys-on-rows", type=int, default=-1, help="attn_decode: warps per block of the kernel with the keys on the tile's rows (0: the other kernel; default: the engine's choice)")
    ap.add_argument("--shortest", type=int, default=0, help="attn_decode: lengths uniform in [shortest, context] instead of all equal")
    ap.add_argument("--nodes", type=int, default=64, help="attn_tree: nodes of every tree, each below any one before it")
    ap.add_argument("--beams", type=int, default=8)
    ap.add_argument("--width", type=int, default=0, help="beam_select: candidates of a sequence (default: twice the beams)")
    ap.add_argument("--iters", type=int, default=20)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--pdl", action="store_true")
    args = ap.parse_args()
    dev = "cuda:0"
    ops.set_pdl(args.pdl)
    if args.keys_on_rows >= 0:
        ops.TUNE["attn_keys_on_rows"] = args.keys_on_rows > 0
        if args.keys_on_rows > 0:
            ops.TUNE["attn_kr_warps"] = args.keys_on_rows
            if args.stages:
                ops.TUNE["attn_kr_stages"] = args.stages
    hbm, tflops, src = _peaks()
    bf = torch.bfloat16
    mode = {"store": ops.SKINNY_STORE_BF16, "accum": ops.SKINNY_ACCUM_F32, "swiglu": ops.SKINNY_SWIGLU, "f32": ops.SKINNY_STORE_F32}[args.mode]
    out = {"kernel": args.kernel, "peaks": src}
    if args.kernel in ("gemm_stream", "gemm_skinny", "gemm_tc"):
        M, N, K = args.m, args.n, args.k
        ops.gemm_tc_tail_tiles(bool(args.tail))
        n_rot = max(2, L2_BYTES * 2 // (N * K * 2) + 1)
        ws = [torch.randn(N, K, device=dev, dtype=bf) * 0.02 for _ in range(n_rot)]
        x = torch.randn(M, K, device=dev, dtype=bf)
        cols = N // 2 if args.mode == "swiglu" else N
        o = torch.zeros(M, cols, device=dev, dtype=bf if args.mode in ("store", "swiglu") else torch.float32)
        fn = {"gemm_stream": ops.gemm_stream, "gemm_skinny": ops.gemm_skinny, "gemm_tc": ops.gemm_tc}[args.kernel]
        us = _time(lambda i: fn(x, ws[i], mode, o), n_rot, args.iters, args.warmup)
        flops, nbytes = 2.0 * M * N * K, N * K * 2 + M * K * 2 + o.numel() * o.element_size()
        out.update(shape=[M, N, K], mode=args.mode, tail=args.tail, us=round(us, 2), tflops=round(flops / us / 1e6, 1),
                   gbs=round(nbytes / us / 1e3, 1), frac_hbm=round(nbytes / us / 1e3 / hbm, 3),
                   frac_tensor=round(flops / us / 1e6 / tflops, 3))
    elif args.kernel in ("attn_decode", "attn_prefill", "attn_prefill_t5"):
        B, S, H, KV, hd = args.batch, args.context, args.heads, args.kv_heads, args.head_dim
        pages_per = (S + 63) // 64
        n_sets = max(2, L2_BYTES * 2 // (B * pages_per * KV * 64 * hd * 2 * 2) + 1) if args.kernel == "attn_decode" else 1
        kc = torch.randn(n_sets * B * pages_per + 1, KV, 64, hd, device=dev, dtype=bf)
        vc = torch.randn_like(kc)
        tables = [(torch.arange(B * pages_per, dtype=torch.int32, device=dev).reshape(B, pages_per) + 1 + s * B * pages_per) for s in range(n_sets)]
        slots = torch.arange(B, dtype=torch.int32, device=dev)
        scale = hd ** -0.5
        if args.kernel == "attn_decode":
            q = torch.randn(B, (H + 2 * KV) * hd, device=dev, dtype=bf)
            lens = torch.full((B,), S, dtype=torch.int32, device=dev)
            if args.shortest:
                lens = torch.randint(args.shortest, S + 1, (B,), generator=torch.Generator().manual_seed(0)).to(torch.int32).to(dev)
            # the engine's choice (StepContext.decode_splits): one wave of as many blocks as an SM holds, slices of at least 128 keys
            sms = torch.cuda.get_device_properties(0).multi_processor_count
            per_sm = ops.attn_decode_blocks_per_sm(hd, True)
            splits, own = ops.attn_decode_plan(B, S, sms, H, KV, hd, None, bf, lens.tolist())
            if args.splits or args.own_tiles:
                splits, own = args.splits or 1, args.own_tiles
            tile = args.tile_keys or int(ops.TUNE["attn_tile_keys"])
            if own:
                splits = max(splits, (S + own * tile - 1) // (own * tile))
            inside = None if args.merge_inside < 0 else bool(args.merge_inside)
            o = torch.empty(B, H * hd, device=dev, dtype=bf)
            po = torch.empty(B * H * splits * hd, device=dev)
            pml = torch.empty(B * H * splits * 2, device=dev)
            us = _time(lambda i: ops.attn_decode_tc(q, kc, vc, tables[i], slots, lens, B, H, KV, hd, scale, None, splits, o, po, pml,
                                                    tile_keys=tile, own_tiles=own, merge_inside=inside, stages=args.stages or None),
                       n_sets, args.iters, args.warmup)
            nbytes = int(lens.sum()) * KV * hd * 2 * 2
            out.update(shape=[B, S, H, KV, hd], shortest=args.shortest, splits=splits, own_tiles=own, tile_keys=tile,
                       merge_inside=inside, stages=args.stages, keys_on_rows=int(ops.TUNE["attn_kr_warps"]) if ops.TUNE["attn_keys_on_rows"] else 0,
                       us=round(us, 2), gbs=round(nbytes / us / 1e3, 1), frac_hbm=round(nbytes / us / 1e3 / hbm, 3))
        else:
            q = torch.randn(B * S, (H + 2 * KV) * hd, device=dev, dtype=bf)
            cu = (torch.arange(B + 1, dtype=torch.int32, device=dev) * S)
            pos0 = torch.zeros(B, dtype=torch.int32, device=dev)
            o = torch.empty(B * S, H * hd, device=dev, dtype=bf)
            fn = ops.attn_prefill_t5 if args.kernel == "attn_prefill_t5" else ops.attn_prefill_tc
            us = _time(lambda i: fn(q, kc, vc, tables[0], cu, slots, pos0, B, S, H, KV, hd, scale, None, o),
                       1, args.iters, args.warmup)
            flops = 2.0 * B * H * hd * S * (S + 1)
            out.update(shape=[B, S, H, KV, hd], us=round(us, 2), tflops=round(flops / us / 1e6, 1),
                       frac_tensor=round(flops / us / 1e6 / tflops, 3))
    elif args.kernel in ("attn_latent_decode", "attn_latent_prefill"):
        from types import SimpleNamespace
        from ..cache.sequence_cache import LayerMemory
        B, S, H, r, dr = args.batch, args.context, args.heads, args.rank, args.rot_dim
        dk = r + dr
        pages_per = (S + 63) // 64
        decode = args.kernel == "attn_latent_decode"
        n_sets = max(2, L2_BYTES * 2 // (B * pages_per * 64 * dk * 2) + 1) if decode else 1
        kc = torch.randn(n_sets * B * pages_per + 1, 1, 64, dk, device=dev, dtype=bf) * 0.5
        tables = [(torch.arange(B * pages_per, dtype=torch.int32, device=dev).reshape(B, pages_per) + 1 + s * B * pages_per) for s in range(n_sets)]
        mems = [LayerMemory(kc, None, t, None, True, None) for t in tables]
        slots = torch.arange(B, dtype=torch.int32, device=dev)
        sms = torch.cuda.get_device_properties(0).multi_processor_count
        scale = dk ** -0.5
        if decode:
            step = SimpleNamespace(n_seqs=B, n_tokens=B, max_q_len=1, max_kv_len=S, is_decode=True, seq_slots=slots,
                                   seq_lens=torch.full((B,), S, dtype=torch.int32, device=dev), sm_count=sms)
            qa = torch.randn(B, H * dk, device=dev, dtype=bf) * 0.5
            o = torch.empty(B, H * r, device=dev, dtype=bf)
            plan = ops.attn_latent_decode_plan(B, S, sms, H, r, dr, bf)
            if args.splits:
                plan = (plan[0], args.splits, 0)
            us = _time(lambda i: ops.attention_latent(qa, mems[i], step, H, r, dr, scale, o, plan=plan), n_sets, args.iters, args.warmup)
            nbytes = B * S * dk * 2
            out.update(shape=[B, S, H, r, dr], plan=list(plan), us=round(us, 2), gbs=round(nbytes / us / 1e3, 1),
                       frac_hbm=round(nbytes / us / 1e3 / hbm, 3))
        else:
            step = SimpleNamespace(n_seqs=B, n_tokens=B * S, max_q_len=S, max_kv_len=S, is_decode=False, seq_slots=slots,
                                   cu_seqlens=torch.arange(B + 1, dtype=torch.int32, device=dev) * S,
                                   seq_pos0=torch.zeros(B, dtype=torch.int32, device=dev), sm_count=sms)
            qa = torch.randn(B * S, H * dk, device=dev, dtype=bf) * 0.5
            o = torch.empty(B * S, H * r, device=dev, dtype=bf)
            us = _time(lambda i: ops.attention_latent(qa, mems[0], step, H, r, dr, scale, o), 1, args.iters, args.warmup)
            flops = 2.0 * B * H * (dk + r) * S * (S + 1) / 2
            out.update(shape=[B, S, H, r, dr], us=round(us, 2), tflops=round(flops / us / 1e6, 1),
                       frac_tensor=round(flops / us / 1e6 / tflops, 3))
    elif args.kernel in ("linear_state", "mamba2_scan"):
        # the token-by-token recurrences: --batch sequences of --context tokens each (--context 1: a decode step), --heads
        # heads of a --head-dim x --v-dim state (mamba2_scan: --v-dim columns per head, --head-dim rows of state)
        from types import SimpleNamespace
        B, S, H, K = args.batch, args.context, args.heads, args.head_dim
        V = args.v_dim or K
        n = B * S
        step = SimpleNamespace(n_seqs=B, cu_seqlens=torch.arange(B + 1, dtype=torch.int32, device=dev) * S,
                               seq_slots=torch.arange(B, dtype=torch.int32, device=dev))
        passes = 2      # a state entry is decayed and written, then read out
        if args.kernel == "linear_state":
            G = args.kv_heads if args.delta else H
            rows = torch.randn(n, 2 * G * K + H * V + 2 * H, device=dev, dtype=bf)
            q, k, v = rows[:, :G * K], rows[:, G * K:2 * G * K], rows[:, 2 * G * K:2 * G * K + H * V]
            state = torch.zeros(B + 1, H * K * V, device=dev)
            if args.delta:
                passes = 3
                a_log, dt_bias = torch.zeros(H, device=dev), torch.zeros(H, device=dev)
                fn = lambda i: ops.linear_state(q, k, v, state, step, H, G, K, V, a_log, decay_in=rows[:, -H:], dt_bias=dt_bias,
                                                beta_in=rows[:, -2 * H:-H], unit_norm=True, q_scale=K ** -0.5, delta=True)
            else:
                decay = torch.full((H,), 0.99, device=dev)
                fn = lambda i: ops.linear_state(q, k, v, state, step, H, H, K, V, decay, in_act=True)
        else:
            G, taps = args.kv_heads, 4
            inner, channels = H * V, H * V + 2 * G * K
            xbc = torch.randn(n, channels, device=dev, dtype=bf)
            proj = torch.randn(n, 2 * inner + 2 * G * K + H, device=dev, dtype=bf)
            consts = [torch.zeros(H, device=dev) for _ in range(3)]
            state = torch.zeros(B + 1, H * K * V + (taps - 1) * channels, device=dev)
            fn = lambda i: ops.mamba2_scan(xbc, proj, consts[0], consts[1], consts[2], state, step, H, V, K, G, taps)
        us = _time(fn, 1, args.iters, args.warmup)
        # 32-bit multiply-adds: one per state entry and pass; the peak is 128 lanes per SM at the clock's maximum
        props = torch.cuda.get_device_properties(0)
        fma, peak = float(passes) * n * H * K * V, props.multi_processor_count * 128 * props.clock_rate * 1e3
        nbytes = 2.0 * B * H * K * V * 4 + n * H * V * 4
        out.update(shape=[B, S, H, G, K, V], delta=int(args.delta), us=round(us, 2), ns_per_token=round(us * 1e3 / S, 1),
                   gfma_per_s=round(fma / us / 1e3, 1), frac_fp32=round(fma / us * 1e6 / peak, 3),
                   gbs=round(nbytes / us / 1e3, 1), frac_hbm=round(nbytes / us / 1e3 / hbm, 3))
    elif args.kernel == "attn_tree":
        B, S, H, KV, hd, n = args.batch, args.context, args.heads, args.kv_heads, args.head_dim, args.nodes
        import numpy as np
        from ..engine.step import tree_facts
        pages_per = (S + n + 63) // 64
        n_sets = max(2, L2_BYTES * 2 // (B * pages_per * KV * 64 * hd * 2 * 2) + 1)
        kc = torch.randn(n_sets * B * pages_per + 1, KV, 64, hd, device=dev, dtype=bf)
        vc = torch.randn_like(kc)
        tables = [(torch.arange(B * pages_per, dtype=torch.int32, device=dev).reshape(B, pages_per) + 1 + s * B * pages_per) for s in range(n_sets)]
        draw = torch.Generator().manual_seed(0)
        parents = [[-1] + [int(torch.randint(i, (1,), generator=draw)) for i in range(1, n)] for _ in range(B)]
        masks = torch.from_numpy(np.concatenate([tree_facts(p, (n + 31) // 32)[0] for p in parents]).view(np.int32)).to(dev)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
        cu, slots, pos0 = i32([n * b for b in range(B + 1)]), i32(list(range(B))), i32([S] * B)
        q, o = torch.randn(B * n, H * hd, device=dev, dtype=bf), torch.empty(B * n, H * hd, device=dev, dtype=bf)
        us = _time(lambda i: ops.attention_tree(q, kc, vc, tables[i], cu, slots, pos0, masks, B, n, S + n, H, KV, hd, hd ** -0.5, o),
                   n_sets, args.iters, args.warmup)
        nbytes, flops = B * (S + n) * KV * hd * 2 * 2 + 2 * B * n * H * hd * 2, 4.0 * B * n * (S + n) * H * hd
        out.update(shape=[B, n, S, H, KV, hd], us=round(us, 2), gbs=round(nbytes / us / 1e3, 1), frac_hbm=round(nbytes / us / 1e3 / hbm, 3),
                   tflops=round(flops / us / 1e6, 1), frac_tensor=round(flops / us / 1e6 / tflops, 3))
    elif args.kernel == "beam_select":
        rows, width = args.batch * args.beams, args.width or 2 * args.beams
        n_sets = max(2, L2_BYTES * 2 // (rows * args.n * 4) + 1)
        logits = [torch.randn(rows, args.n, device=dev) for _ in range(n_sets)]
        scores = -torch.rand(args.batch, args.beams, device=dev)
        us = _time(lambda i: ops.beam_select(logits[i], scores, width), n_sets, args.iters, args.warmup)
        nbytes = rows * args.n * 4
        out.update(shape=[args.batch, args.beams, args.n], width=width, us=round(us, 2), gbs=round(nbytes / us / 1e3, 1),
                   frac_hbm=round(nbytes / us / 1e3 / hbm, 3))
    elif args.kernel == "rmsnorm":
        x = torch.randn(args.m, args.k, device=dev)
        w = torch.ones(args.k, device=dev, dtype=bf)
        us = _time(lambda i: ops.rmsnorm(x, w, 1e-5, bf), 1, args.iters, args.warmup)
        out.update(shape=[args.m, args.k], us=round(us, 2))
    elif args.kernel == "sample":
        logits = torch.randn(args.m, args.n, device=dev)
        state = torch.arange(1, args.m + 1, dtype=torch.int64, device=dev)
        us_g = _time(lambda i: ops.sample(logits, 0.0, 0, 1.0), 1, args.iters, args.warmup)
        us_s = _time(lambda i: ops.sample(logits, 0.7, 40, 0.9, state), 1, args.iters, args.warmup)
        us_t = _time(lambda i: ops.sample(logits, 0.7, 0, 1.0, state), 1, args.iters, args.warmup)
        us_p = _time(lambda i: ops.sample(logits, 0.7, 0, 0.9, state), 1, args.iters, args.warmup)
        out.update(shape=[args.m, args.n], us_greedy=round(us_g, 2), us_top_k_top_p=round(us_s, 2), us_temperature=round(us_t, 2),
                   us_top_p=round(us_p, 2))
    else:
        ap.error(f"unknown kernel {args.kernel}")
    print(json.dumps(out))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
