"""Attention over the 8-bit KV cache beside the bf16 one, one layer at a time.

    python -m helexa_b200.bench.kv8_bench [--heads 32 8 128] [--batch 1 8] [--context 2048 8192 32768 131072]

Decode: us a step and GB/s of cache read (a few caches in turn, so that together they exceed L2).
Prefill: us and TFLOP/s of a causal prompt (the 8-bit side includes its append).
"""
from __future__ import annotations

import argparse

import torch

from .. import ops
from ..ops.kv8 import KV8


def _time(fns, iters: int) -> float:
    for f in fns:
        f()
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    for i in range(iters):
        fns[i % len(fns)]()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) * 1e3 / iters


def decode(Hq: int, Hkv: int, D: int, B: int, L: int, kv: str, iters: int = 60) -> tuple[float, float]:
    C, dev, bf = ops.C, "cuda", torch.bfloat16
    cache_bytes = 2 * B * Hkv * L * D * (2 if kv == "bf16" else 1)
    sets = max(1, min(8, -(-(400 << 20) // cache_bytes)))
    proj = torch.randn(B, (Hq + 2 * Hkv) * D, device=dev).to(bf)
    inv = torch.ones(D // 2, device=dev)
    slots = torch.arange(B, dtype=torch.int32, device=dev)
    pos = torch.full((B,), L - 1, dtype=torch.int32, device=dev)
    out = torch.empty(B, Hq * D, dtype=bf, device=dev)
    fns = []
    for _ in range(sets):
        if kv == "bf16":
            sms = torch.cuda.get_device_properties(0).multi_processor_count
            ns = max(8, min(256, (sms // (B * Hkv) + 7) // 8 * 8))  # as the model chooses it
            kc, vc = (torch.randn(B, Hkv, L, D, device=dev).to(bf) for _ in range(2))
            po, pm = torch.empty(B, Hq, ns, D, device=dev), torch.empty(B, Hq, ns, 2, device=dev)
            cnt = torch.zeros(B, Hkv, dtype=torch.int32, device=dev)
            fns.append(lambda kc=kc, vc=vc, po=po, pm=pm, cnt=cnt: C.attn_decode(
                proj, None, None, inv, kc, vc, slots, pos, po, pm, cnt, out, Hq, Hkv, D, D, False, 1e-6))
        else:
            c, ws = KV8.alloc(B, Hkv, L, D, kv, dev), C.kv8_workspace(B, Hq, Hkv, D)
            for b in range(B):
                k, v = torch.randn(2, L, Hkv, D, device=dev).to(bf)
                C.kv8_append(k, v, *c, b, 0)
            fns.append(lambda c=c, ws=ws: C.attn_decode_kv8(proj, None, None, inv, *c, slots, pos, ws, out, Hq, D,
                                                            False, 1e-6))
    us = _time(fns, iters)
    return us, cache_bytes / us / 1e3


def prefill(Hq: int, Hkv: int, D: int, T: int, kv: str, iters: int = 10) -> tuple[float, float]:
    C, dev, bf = ops.C, "cuda", torch.bfloat16
    q = torch.randn(T, Hq * D, device=dev).to(bf)
    k, v = torch.randn(2, Hkv, T, D, device=dev).to(bf)
    o, err = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device=dev)
    if kv == "bf16":
        fn = lambda: C.attn_prefill_tc(q, k, v, o, Hq, 0, D ** -0.5, None, 0, err)  # noqa: E731
    else:
        c = KV8.alloc(1, Hkv, T, D, kv, dev)

        def fn():
            C.kv8_append(k.transpose(0, 1), v.transpose(0, 1), *c, 0, 0)
            C.attn_prefill_kv8(q, *c, 0, 0, o, Hq, D ** -0.5, None, 0, err)
    us = _time([fn], iters)
    return us, 2 * Hq * D * T * (T + 1) / us / 1e6


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--heads", type=int, nargs=3, default=[32, 8, 128], metavar=("HQ", "HKV", "D"))
    ap.add_argument("--batch", type=int, nargs="+", default=[1, 8])
    ap.add_argument("--context", type=int, nargs="+", default=[2048, 8192, 32768, 131072])
    ap.add_argument("--prompt", type=int, nargs="+", default=[1024, 4096, 8192])
    a = ap.parse_args()
    for B in a.batch:
        for L in a.context:
            if B * L * a.heads[1] * a.heads[2] * 4 > 20 << 30:
                continue
            row = {kv: decode(*a.heads, B, L, kv) for kv in ("bf16", "int8", "fp8")}
            print(f"decode  batch {B} context {L}: " + ", ".join(f"{k} {u:.1f} us ({g:.0f} GB/s)"
                                                                 for k, (u, g) in row.items()), flush=True)
    for T in a.prompt:
        row = {kv: prefill(*a.heads, T, kv) for kv in ("bf16", "int8", "fp8")}
        print(f"prefill {T} tokens: " + ", ".join(f"{k} {u:.0f} us ({g:.0f} TFLOP/s)" for k, (u, g) in row.items()),
              flush=True)


if __name__ == "__main__":
    main()
