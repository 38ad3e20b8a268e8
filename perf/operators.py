"""Measured cases of the 8-bit KV cache: quantising as it is written, reading it back, and
attention over it (one token a sequence, and the tokens of a prompt).

The cache of one layer is six tensors. Tokens are held in blocks of 32. A complete block
has 8-bit codes and one f32 scale for each kv head; the sequence's last block is also kept
in bf16 (its "tail"), and is read from there until it is complete:

  kc  [S, Hkv, NB, D/64, 32 keys, 64 dims]   codes of K (int8 or float8_e4m3fn)
  vc  [S, Hkv, NB, D/64, 64 dims, 32 keys]   codes of V, keys innermost
  ks, vs  f32 [S, Hkv, NB]                   scales: value = code * scale
  kt  bf16 [S, Hkv, D/64, 32, 64]            the last block, laid out like kc
  vt  bf16 [S, Hkv, D/64, 64, 32]            the last block, laid out like vc

scale = max|x| / M over a block and head (M = 127 for int8, 448 for float8_e4m3fn) and
code = round(x * (M / max|x|)), ties to even.
"""
import math
import random

import torch

own = False

BLK = 32
TOP = {"int8": 127.0, "fp8": 448.0}
DTYPE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
EPS = 1e-6


def listed():
    return [
        # a prompt chunk's K / V of an 8B dense model (32 / 8 heads of 128) entering an empty slot
        {"name": "append_chunk_8k", "op": "append", "fmt": "int8", "T": 8192, "p0": 0, "Hkv": 8, "D": 128},
        # the few tokens of a follow-up message behind a restored prefix, gated-attention heads (2 of 256)
        {"name": "append_short_odd", "op": "append", "fmt": "fp8", "T": 37, "p0": 1003, "Hkv": 2, "D": 256},
        # a 32K prefix read back as bf16 (leaving the 8-bit cache, or a check of it)
        {"name": "read_prefix_32k", "op": "read", "fmt": "fp8", "L": 32785, "start": 0, "Hkv": 8, "D": 128},
        # the end of a short conversation, from the middle of a block
        {"name": "read_short", "op": "read", "fmt": "int8", "L": 777, "start": 33, "Hkv": 2, "D": 64},
        # the smallest step: one new conversation, small heads, an odd number of query heads per kv head
        {"name": "decode_small_g3", "op": "decode", "fmt": "int8", "B": 1, "L": 96, "Hq": 6, "Hkv": 2, "D": 64,
         "rot": 0, "gated": False},
        # one chat at the 8K context of the benchmark: 16 / 2 heads of 256, quarter rotary, output gate
        {"name": "decode_gated_8k", "op": "decode", "fmt": "fp8", "B": 1, "L": 8192, "Hq": 16, "Hkv": 2, "D": 256,
         "rot": 64, "gated": True},
        # a full continuous batch of conversations of many lengths, 32 / 8 heads of 128
        {"name": "decode_batch8_16k", "op": "decode", "fmt": "int8", "B": 8, "L": 16384, "Hq": 32, "Hkv": 8, "D": 128,
         "rot": 128, "gated": False},
        # four long documents, 16 query heads on each kv head (64 / 4 heads of 128)
        {"name": "decode_g16_40k", "op": "decode", "fmt": "fp8", "B": 4, "L": 40901, "Hq": 64, "Hkv": 4, "D": 128,
         "rot": 128, "gated": False},
        # a whole 4K prompt of an 8B dense model
        {"name": "prefill_4k", "op": "prefill", "fmt": "int8", "T": 4096, "p0": 0, "Hq": 32, "Hkv": 8, "D": 128,
         "gated": False},
        # the second 8K chunk of a long prompt, gated attention
        {"name": "prefill_gated_chunk", "op": "prefill", "fmt": "fp8", "T": 8192, "p0": 8192, "Hq": 16, "Hkv": 2,
         "D": 256, "gated": True},
        # a short follow-up turn behind a 30K prefix
        {"name": "prefill_turn_30k", "op": "prefill", "fmt": "int8", "T": 61, "p0": 30007, "Hq": 32, "Hkv": 8,
         "D": 128, "gated": False},
        # an odd prompt behind a short prefix, 64 / 8 heads
        {"name": "prefill_odd", "op": "prefill", "fmt": "fp8", "T": 1537, "p0": 13, "Hq": 64, "Hkv": 8, "D": 128,
         "gated": False},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "prefill", "prefill"])
    fmt = rng.choice(["int8", "fp8"])
    D = rng.choice([64, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8] if D < 256 else [1, 2])
    if op == "append":
        return {"op": op, "fmt": fmt, "T": _spread(rng, 1, 8192), "p0": rng.choice([0, _spread(rng, 1, 8192)]),
                "Hkv": Hkv, "D": D}
    if op == "read":
        L = _spread(rng, 1, 32785)
        return {"op": op, "fmt": fmt, "L": L, "start": rng.choice([0, rng.randrange(L)]), "Hkv": Hkv, "D": D}
    G = rng.choice([1, 2, 3, 4, 7, 8, 16] if D < 256 else [1, 2, 5, 8])
    if op == "decode":
        B = rng.choice([1, 1, 2, 3, 4, 8])
        return {"op": op, "fmt": fmt, "B": B, "L": _spread(rng, 1, 40901 if B <= 4 else 16384), "Hq": Hkv * G,
                "Hkv": Hkv, "D": D, "rot": rng.choice([0, D // 4, D]), "gated": rng.choice([False, True])}
    Hq = min(Hkv * G, 64)
    T = _spread(rng, 1, 4096)
    most = 16 * 8192 * 16384  # queries x keys x heads of the largest listed prompt
    p0 = rng.choice([0, _spread(rng, 1, 30007)])
    p0 = max(0, min(p0, most // (T * Hq) - T))
    return {"op": op, "fmt": fmt, "T": T, "p0": p0, "Hq": Hq, "Hkv": Hkv, "D": D,
            "gated": rng.choice([False, True])}


def _lens(case):
    """Tokens in each sequence of a decode batch, the new one included: the longest has L, the others
    are spread below it. An int8 step that completes a block rounds the rotated key to whole codes, which
    need not agree in their last place between two ways of rotating it; those lengths are left to the
    int8 cases without rotation, and to float8 codes."""
    r = random.Random(case["B"] * 1000003 + case["L"])
    lens = [case["L"]] + [r.randint(max(1, case["L"] // 8), case["L"]) for _ in range(case["B"] - 1)]
    if case["fmt"] == "int8" and case["rot"]:
        lens = [n - 1 if n % BLK == 0 else n for n in lens]
    return lens


def _pools(g, S, Hkv, nb, D, fmt):
    """Caches as earlier tokens left them: normal values, a little apart from block to block."""
    n = D // 64
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731

    def codes(*s):
        x = (rnd(*s) * (TOP[fmt] / 4)).clamp_(-TOP[fmt], TOP[fmt])
        return (x.round_() if fmt == "int8" else x).to(DTYPE[fmt])
    scale = lambda: (4 / TOP[fmt]) * torch.exp(0.3 * rnd(S, Hkv, nb))  # noqa: E731
    return {"kc": codes(S, Hkv, nb, n, BLK, 64), "vc": codes(S, Hkv, nb, n, 64, BLK), "ks": scale(), "vs": scale(),
            "kt": rnd(S, Hkv, n, BLK, 64).bfloat16(), "vt": rnd(S, Hkv, n, 64, BLK).bfloat16()}


CACHE = ("kc", "vc", "ks", "vs", "kt", "vt")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    D, Hkv, op = case["D"], case["Hkv"], case["op"]
    st = {"case": dict(case)}
    if op == "append":
        T, p0 = case["T"], case["p0"]
        st.update(_pools(g, 2, Hkv, (p0 + T) // BLK + 2, D, case["fmt"]))
        st["slot"] = 1
        # rotated keys, a head after another, and values still in the rows of a [q | k | v] projection
        st["k"] = rnd(Hkv, T, D).bfloat16().transpose(0, 1)
        st["v"] = rnd(T, 6 * Hkv * D).bfloat16()[:, 5 * Hkv * D:].view(T, Hkv, D)
    elif op == "read":
        L = case["L"]
        st.update(_pools(g, 2, Hkv, L // BLK + 2, D, case["fmt"]))
        st["slot"] = 1
        st["k_out"] = torch.empty(Hkv, L - case["start"], D, dtype=torch.bfloat16, device="cuda")
        st["v_out"] = torch.empty_like(st["k_out"])
    elif op == "decode":
        B, Hq, rot = case["B"], case["Hq"], case["rot"]
        lens = _lens(case)
        st.update(_pools(g, B + 1, Hkv, max(lens) // BLK + 1, D, case["fmt"]))
        order = torch.randperm(B + 1, generator=g, device="cuda")[:B]
        st["slots"] = order.to(torch.int32)
        st["pos"] = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
        st["pos"][order] = torch.tensor(lens, dtype=torch.int32, device="cuda") - 1
        qw = 2 * D if case["gated"] else D
        st["proj"] = rnd(B, Hq * qw + 2 * Hkv * D).bfloat16()
        norm = bool(rot)  # models that rotate here normalise here too
        st["q_norm"] = (1.0 + 0.5 * torch.rand(D, generator=g, device="cuda")) if norm else None
        st["k_norm"] = (0.75 + 0.5 * torch.rand(D, generator=g, device="cuda")) if norm else None
        st["inv_freq"] = 1e6 ** (-torch.arange(0, max(rot, 2), 2, device="cuda").float() / max(rot, 2))
        st["out"] = torch.empty(B, Hq * D, dtype=torch.bfloat16, device="cuda")
    else:
        T, p0, Hq = case["T"], case["p0"], case["Hq"]
        st.update(_pools(g, 2, Hkv, (p0 + T) // BLK + 1, D, case["fmt"]))
        st["slot"] = 1
        st["q"] = (1.5 * rnd(T, Hq * D)).bfloat16()
        # the gate's rows lie beside the query's in the projection, a head after another
        st["gate"] = rnd(T, Hq * 2 * D).bfloat16()[:, D:] if case["gated"] else None
        st["out"] = torch.empty(T, Hq * D, dtype=torch.bfloat16, device="cuda")
        st["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return st


# ---- the plain forms ----------------------------------------------------------------------


def _quantise(x, fmt):
    """Codes and scales of x [..., rows, cols] in 32 bits, one scale over the last three axes."""
    m = x.float().abs().amax((-3, -2, -1))
    top = torch.full_like(m, TOP[fmt])
    y = x.float() * torch.where(m > 0, top / m, torch.zeros_like(m))[..., None, None, None]
    return (y.round() if fmt == "int8" else y).to(DTYPE[fmt]), m / top


def _keys(c):
    """[..., NB, D/64, 32, 64] (K's layout) -> [..., NB * 32, D]"""
    c = c.transpose(-3, -2)
    return c.reshape(*c.shape[:-4], c.shape[-4] * BLK, c.shape[-2] * 64)


def _values(c):
    """[..., NB, D/64, 64, 32] (V's layout) -> [..., NB * 32, D]"""
    c = c.permute(*range(c.dim() - 3), -1, -3, -2)
    return c.reshape(*c.shape[:-4], c.shape[-4] * BLK, c.shape[-2] * 64)


def _to_keys(x):
    """[..., n * 32, D] -> [..., n, D/64, 32, 64]"""
    return x.reshape(*x.shape[:-2], -1, BLK, x.shape[-1] // 64, 64).transpose(-3, -2)


def _to_values(x):
    """[..., n * 32, D] -> [..., n, D/64, 64, 32]"""
    x = x.reshape(*x.shape[:-2], -1, BLK, x.shape[-1] // 64, 64)
    return x.permute(*range(x.dim() - 3), -2, -1, -3)


def _append(st):
    c, s = st["case"], st["slot"]
    p0, L = c["p0"], c["p0"] + c["T"]
    b0, r0, last = p0 // BLK, p0 % BLK, (L - 1) // BLK
    k = torch.cat([_keys(st["kt"][s, :, None])[:, :r0], st["k"].transpose(0, 1)], 1)  # from the first touched block on
    v = torch.cat([_values(st["vt"][s, :, None])[:, :r0], st["v"].transpose(0, 1)], 1)
    n = L // BLK - b0
    if n:
        st["kc"][s, :, b0:b0 + n], st["ks"][s, :, b0:b0 + n] = _quantise(_to_keys(k[:, :n * BLK]), c["fmt"])
        st["vc"][s, :, b0:b0 + n], st["vs"][s, :, b0:b0 + n] = _quantise(_to_values(v[:, :n * BLK]), c["fmt"])
    rows = L - last * BLK
    kl, vl = k[:, (last - b0) * BLK:], v[:, (last - b0) * BLK:]
    st["kt"][s, :, :, :rows] = kl.reshape(kl.shape[0], rows, -1, 64).transpose(1, 2)
    st["vt"][s, :, :, :, :rows] = vl.reshape(vl.shape[0], rows, -1, 64).permute(0, 2, 3, 1)
    return {x: st[x] for x in CACHE}


def _dequantised(st, at, nb):
    """K and V of the first nb blocks of slots `at`, in 32 bits: [..., NB * 32, D]."""
    fmt = DTYPE[st["case"]["fmt"]]
    k, v = (st[x].view(torch.uint8)[at][..., :nb, :, :, :].view(fmt).float() for x in ("kc", "vc"))
    k *= st["ks"][at][..., :nb, None, None, None]
    v *= st["vs"][at][..., :nb, None, None, None]
    return _keys(k), _values(v)


def _read(st):
    c, s, L = st["case"], st["slot"], st["case"]["L"]
    k, v = _dequantised(st, s, L // BLK)
    r = L % BLK
    k = torch.cat([k, _keys(st["kt"][s, :, None]).float()[:, :r]], 1)[:, c["start"]:]
    v = torch.cat([v, _values(st["vt"][s, :, None]).float()[:, :r]], 1)[:, c["start"]:]
    return {"k": k.bfloat16(), "v": v.bfloat16()}


def _softmax(s):
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _rotated(x, pos, inv_freq, rot):
    """Rotate-half rotary embedding of the first `rot` dims of x [B, H, D]."""
    if not rot:
        return x
    a = pos.to(inv_freq.dtype)[:, None, None] * inv_freq[None, None, :]
    a = torch.cat([a, a], -1)
    y = x[..., :rot]
    turned = torch.cat([-y[..., rot // 2:], y[..., :rot // 2]], -1)
    return torch.cat([y * torch.cos(a) + turned * torch.sin(a), x[..., rot:]], -1)


def _split(st, x):
    """(q, gate, k, v) of the rows of a projection, [B, heads, D] each."""
    c = st["case"]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    qw = 2 * D if c["gated"] else D
    q = x[:, :Hq * qw].view(B, Hq, qw)
    kv = x[:, Hq * qw:].view(B, 2, Hkv, D)
    return q[..., :D], (q[..., D:] if c["gated"] else None), kv[:, 0], kv[:, 1]


def _decode(st):
    c = st["case"]
    Hkv, D = c["Hkv"], c["D"]
    at = st["slots"].long()
    pos = st["pos"][at].long()
    L, row, blk = pos + 1, pos % BLK, pos // BLK
    q, gate, k, v = _split(st, st["proj"].float())
    q = _rotated(_normed(q, st["q_norm"]), pos, st["inv_freq"], c["rot"])
    k = _rotated(_normed(k, st["k_norm"]), pos, st["inv_freq"], c["rot"])
    # the token enters its sequence's last block; a block that it completes gets its codes
    st["kt"][at, :, :, row] = k.bfloat16().view(-1, Hkv, D // 64, 64)
    st["vt"][at, :, :, :, row] = v.bfloat16().view(-1, Hkv, D // 64, 64)
    whole = (L % BLK == 0)[:, None]
    for_k, sk = _quantise(st["kt"][at], c["fmt"])
    for_v, sv = _quantise(st["vt"][at], c["fmt"])
    here = whole[..., None, None, None]
    kc, vc = st["kc"].view(torch.uint8), st["vc"].view(torch.uint8)  # codes as bytes: float8 has no where()
    kc[at, :, blk] = torch.where(here, for_k.view(torch.uint8), kc[at, :, blk])
    vc[at, :, blk] = torch.where(here, for_v.view(torch.uint8), vc[at, :, blk])
    st["ks"][at, :, blk] = torch.where(whole, sk, st["ks"][at, :, blk])
    st["vs"][at, :, blk] = torch.where(whole, sv, st["vs"][at, :, blk])
    nb = st["ks"].shape[2]
    kd, vd = _dequantised(st, at, nb)
    kd = torch.cat([kd, _keys(st["kt"][at, :, None]).float()], 2)
    vd = torch.cat([vd, _values(st["vt"][at, :, None]).float()], 2)
    j = torch.arange((nb + 1) * BLK, device="cuda")
    inside = torch.where(j < nb * BLK, j < (L // BLK * BLK)[:, None], j - nb * BLK < (L % BLK)[:, None])
    s = torch.matmul(q.reshape(-1, Hkv, c["Hq"] // Hkv, D), kd.transpose(-1, -2)) * D ** -0.5
    p = _softmax(s.masked_fill(~inside[:, None, None], -math.inf))
    o = torch.matmul(p, vd).reshape(-1, c["Hq"], D)
    if gate is not None:
        o = o / (1 + torch.exp(-gate))
    return {"out": o.reshape(len(at), -1).bfloat16(), **{x: st[x] for x in CACHE}}


def _prefill(st):
    c, slot = st["case"], st["slot"]
    T, p0, Hq, Hkv, D = c["T"], c["p0"], c["Hq"], c["Hkv"], c["D"]
    L = p0 + T
    k, v = _dequantised(st, slot, L // BLK)
    r = L % BLK
    k = torch.cat([k, _keys(st["kt"][slot, :, None]).float()[:, :r]], 1)
    v = torch.cat([v, _values(st["vt"][slot, :, None]).float()[:, :r]], 1)
    q = st["q"].float().view(T, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3)
    s = torch.matmul(q, k[:, None].transpose(-1, -2)) * D ** -0.5
    later = torch.arange(L, device="cuda") > torch.arange(p0, L, device="cuda")[:, None]
    o = torch.matmul(_softmax(s.masked_fill_(later, -math.inf)), v[:, None]).permute(2, 0, 1, 3).reshape(T, Hq, D)
    if st["gate"] is not None:
        gate = st["gate"].as_strided((T, Hq, D), (st["gate"].stride(0), 2 * D, 1)).float()
        o = o / (1 + torch.exp(-gate))
    return {"out": o.reshape(T, Hq * D).bfloat16()}


# ---- the framework's operators ------------------------------------------------------------


def _run_own(st):
    from helexa_b200 import ops
    C = ops.C
    c = st["case"]
    cache = [st[x] for x in CACHE]
    if c["op"] == "append":
        C.kv8_append(st["k"], st["v"], *cache, st["slot"], c["p0"])
        return {x: st[x] for x in CACHE}
    if c["op"] == "read":
        C.kv8_read(*cache, st["slot"], c["L"], c["start"], st["k_out"], st["v_out"])
        return {"k": st["k_out"], "v": st["v_out"]}
    if c["op"] == "decode":
        if "ws" not in st:  # made once for a batch size, as a serving loop keeps its buffers
            st["ws"] = C.kv8_workspace(c["B"], c["Hq"], c["Hkv"], c["D"])
        C.attn_decode_kv8(st["proj"], st["q_norm"], st["k_norm"], st["inv_freq"], *cache, st["slots"], st["pos"],
                          st["ws"], st["out"], c["Hq"], c["rot"], c["gated"], EPS)
        return {"out": st["out"], **{x: st[x] for x in CACHE}}
    C.attn_prefill_kv8(st["q"], *cache, st["slot"], c["p0"], st["out"], c["Hq"], c["D"] ** -0.5, st["gate"],
                       2 * c["D"], st["err"])
    return {"out": st["out"]}


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append, "read": _read, "decode": _decode, "prefill": _prefill}[state["case"]["op"]](state)


def work(case):
    D, Hkv, op = case["D"], case["Hkv"], case["op"]
    token = 2 * Hkv * D  # K and V values of one token
    if op == "append":
        T, p0 = case["T"], case["p0"]
        n = (p0 + T) // BLK - p0 // BLK  # blocks completed
        kept = p0 % BLK if n else 0      # tail rows that enter the first of them
        left = (p0 + T - 1) % BLK + 1
        return {"bytes": token * (2 * T + 2 * kept + BLK * n + 2 * min(left, T)) + 8 * Hkv * n, "flops": 2 * token * T}
    if op == "read":
        n = case["L"] - case["start"]
        tail = min(n, case["L"] % BLK)
        return {"bytes": token * ((n - tail) + 2 * tail + 2 * n) + 8 * Hkv * ((n - tail) / BLK), "flops": token * n}
    Hq = case["Hq"]
    if op == "decode":
        lens = _lens(case)
        seen = sum((n // BLK) * (BLK * token + 8 * Hkv) + 2 * (n % BLK) * token for n in lens)
        row = 2 * ((2 if case["gated"] else 1) * Hq * D + token) + 2 * token + 2 * Hq * D
        return {"bytes": seen + case["B"] * row, "flops": 4 * Hq * D * sum(lens)}
    T, p0 = case["T"], case["p0"]
    pairs = T * p0 + T * (T + 1) // 2
    rows = 2 * T * Hq * D * (3 if case["gated"] else 2)
    return {"bytes": (p0 + T) * token + rows, "flops": 4 * Hq * D * pairs}


# ---- from the definition, in 64 bits ------------------------------------------------------


def _exact_block(codes, scales, tail, L, keys):
    """[Hkv, L, D] in 64 bits of one slot's codes [Hkv, NB, D/64, a, b], scales and tail."""
    order = (0, 1, 3, 2, 4) if keys else (0, 1, 4, 2, 3)
    H, n, D = codes.shape[0], L // BLK, 64 * codes.shape[2]
    x = (codes[:, :n].double() * scales[:, :n].double()[..., None, None, None]).permute(*order).reshape(H, n * BLK, D)
    t = tail.double()[:, None].permute(*order).reshape(H, BLK, D)
    return torch.cat([x, t[:, :L - n * BLK]], 1)


def _exact_attention(q, k, v, first):
    """q [Hq, T, D] at positions first.., k and v [Hkv, L, D], all 64-bit: a kv head at a time."""
    Hkv, L, D = k.shape
    out, G = [], q.shape[0] // Hkv
    j = torch.arange(L, device=q.device)
    for h in range(q.shape[0]):
        rows = []
        for t in range(0, q.shape[1], 2048):
            s = q[h, t:t + 2048] @ k[h // G].T / math.sqrt(D)
            s.masked_fill_(j > first + t + torch.arange(len(s), device=q.device)[:, None], -math.inf)
            rows.append(torch.softmax(s, -1) @ v[h // G])
        out.append(torch.cat(rows))
    return torch.stack(out)


def exact(case, seed):
    st = prepare(case, seed)
    op, D, Hkv = case["op"], case["D"], case["Hkv"]
    if op == "append":  # the scales; codes are whole by definition, and the tail is a copy
        s, p0, T = st["slot"], case["p0"], case["T"]
        b0, n = p0 // BLK, (p0 + T) // BLK - p0 // BLK
        got = {}
        for x, y, t, keys in (("k", "ks", "kt", True), ("v", "vs", "vt", False)):
            old = _exact_block(st[x + "c"][s], st[y][s], st[t][s], p0 % BLK, keys)
            rows = torch.cat([old, st[x].double().transpose(0, 1)], 1)[:, :n * BLK]
            scales = st[y].double()
            scales[s, :, b0:b0 + n] = rows.reshape(Hkv, n, BLK * D).abs().amax(-1) / TOP[case["fmt"]] if n else 0
            got[y] = scales
        return {"kc": None, "vc": None, "ks": got["ks"], "vs": got["vs"], "kt": None, "vt": None}
    if op == "read":
        s, L = st["slot"], case["L"]
        return {x: _exact_block(st[x + "c"][s], st[x + "s"][s], st[x + "t"][s], L, x == "k")[:, case["start"]:]
                for x in ("k", "v")}
    if op == "prefill":
        s, T, p0, Hq = st["slot"], case["T"], case["p0"], case["Hq"]
        k, v = (_exact_block(st[x + "c"][s], st[x + "s"][s], st[x + "t"][s], p0 + T, x == "k") for x in ("k", "v"))
        o = _exact_attention(st["q"].double().view(T, Hq, D).transpose(0, 1), k, v, p0).transpose(0, 1)
        if st["gate"] is not None:
            o = o * torch.sigmoid(torch.stack([st["gate"][:, h * 2 * D:h * 2 * D + D] for h in range(Hq)], 1).double())
        return {"out": o.reshape(T, Hq * D)}
    q, gate, k, v = _split(st, st["proj"].double())
    out, rot = [], case["rot"]
    for b, L in enumerate(_lens(case)):
        s, r = int(st["slots"][b]), (L - 1) % BLK

        def head(x, w):
            if w is not None:
                x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
            if rot:
                a, h = (L - 1) * st["inv_freq"].double(), rot // 2
                lo, hi = x[..., :h], x[..., h:rot]
                x = torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin(), x[..., rot:]], -1)
            return x
        # the cache holds the token in bf16
        st["kt"][s, :, :, r] = head(k[b], st["k_norm"]).bfloat16().view(Hkv, -1, 64)
        st["vt"][s, :, :, :, r] = v[b].bfloat16().view(Hkv, -1, 64)
        if r == BLK - 1:
            for x in ("k", "v"):
                t = st[x + "t"][s].double()
                m = t.abs().amax((1, 2, 3), keepdim=True)
                y = t * (TOP[case["fmt"]] / m)
                st[x + "c"][s, :, L // BLK - 1] = (y.round() if case["fmt"] == "int8" else y.float()).to(DTYPE[case["fmt"]])
                st[x + "s"][s, :, L // BLK - 1] = (m / TOP[case["fmt"]]).view(-1).float()
        ks, vs = (_exact_block(st[x + "c"][s], st[x + "s"][s], st[x + "t"][s], L, x == "k") for x in ("k", "v"))
        o = _exact_attention(head(q[b], st["q_norm"])[:, None], ks, vs, L - 1)[:, 0]
        out.append((o * torch.sigmoid(gate[b]) if gate is not None else o).reshape(-1))
    return {"out": torch.stack(out), "kc": None, "vc": None, "ks": st["ks"].double(), "vs": st["vs"].double(),
            "kt": None, "vt": None}
