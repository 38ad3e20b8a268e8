"""The 8-bit KV cache (append, read back, decode and prefill attention) against plain 64-bit
implementations, at the lengths, offsets, strides and head layouts where it can go wrong.

Tolerances. Outputs are bf16: half a unit in the last place is 2^-9 of a value. The attention
kernels may round q and the probabilities to 11 bits or more and sum in f32, which stays
below 2^-10 of the largest |v| a row mixes; `ATOL` leaves twice that, `RTOL` twice a bf16
rounding.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BLK = 32
TOP = {"int8": 127.0, "fp8": 448.0}
DTYPE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
RTOL, ATOL = 2.0 ** -8, 2.0 ** -9


def _C():
    from helexa_b200 import ops
    return ops.C


def _alloc(S, H, nb, D, fmt, fill=None):
    """An empty cache: codes and tails hold `fill` bytes (what nobody wrote must not matter)."""
    n = D // 64
    def bytes_(*s):
        return torch.full(s, 0x7f if fill is None else fill, dtype=torch.uint8, device="cuda")
    kc = bytes_(S, H, nb, n, BLK, 64).view(DTYPE[fmt])
    vc = bytes_(S, H, nb, n, 64, BLK).view(DTYPE[fmt])
    ks = torch.full((S, H, nb), float("nan"), device="cuda")
    kt = torch.full((S, H, n, BLK, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    vt = torch.full((S, H, n, 64, BLK), float("nan"), dtype=torch.bfloat16, device="cuda")
    return [kc, vc, ks, ks.clone(), kt, vt]


def _quant(x, fmt):
    """Codes (as f64) and scale of one block [32, D], by the definition, in f32 like the cache."""
    f = x.float()
    m = torch.where(f.isfinite(), f.abs(), torch.zeros_like(f)).max()
    if m < 1e-30:
        return torch.zeros_like(f).double(), torch.zeros((), device=x.device)
    y = f * (torch.full_like(m, TOP[fmt]) / m)
    y = torch.where(y.isnan(), torch.zeros_like(y), y.clamp(-TOP[fmt], TOP[fmt]))
    c = y.round().double() if fmt == "int8" else y.to(torch.float8_e4m3fn).double()
    return c, m / torch.full_like(m, TOP[fmt])


def _model(rows, fmt):
    """What a sequence of bf16 rows [L, H, D] reads as: f64 [H, L, D] and the codes' scales [H, nb]."""
    L, H, D = rows.shape
    out = rows.double().transpose(0, 1).clone()
    scales = torch.zeros(H, L // BLK, device=rows.device)
    codes = torch.zeros(H, L // BLK * BLK, D, dtype=torch.float64, device=rows.device)
    for h in range(H):
        for b in range(L // BLK):
            c, s = _quant(rows[b * BLK:(b + 1) * BLK, h], fmt)
            codes[h, b * BLK:(b + 1) * BLK] = c
            scales[h, b] = s
            out[h, b * BLK:(b + 1) * BLK] = c * s.double()
    return out, codes, scales


def _code_rows(kc, slot, nb, keys):
    c = kc[slot, :, :nb].float().double()
    c = c.permute(0, 1, 3, 2, 4) if keys else c.permute(0, 1, 4, 2, 3)
    return c.reshape(c.shape[0], nb * BLK, kc.shape[3] * 64)


def _attend(q, k, v, first, scale):
    """q [T, Hq, D] f64 at positions first..; k, v [H, L, D] f64."""
    T, Hq, D = q.shape
    G = Hq // k.shape[0]
    kr, vr = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    s = torch.einsum("thd,hld->htl", q, kr) * scale
    j = torch.arange(k.shape[1], device=q.device)
    s = s.masked_fill(j[None, None] > first + torch.arange(T, device=q.device)[None, :, None], -math.inf)
    return torch.einsum("htl,hld->thd", torch.softmax(s, -1), vr)


def _check(got, want, vmax):
    err = (got.double() - want).abs()
    assert bool((err <= RTOL * want.abs() + ATOL * vmax).all()), float((err - RTOL * want.abs()).max())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("D,H", [(64, 3), (128, 2), (256, 1)])
@pytest.mark.parametrize("parts", [[1], [31], [32], [33], [64], [5, 27, 1], [40, 1, 90], [31, 1, 1, 200], [0, 7, 0]])
def test_append_and_read(fmt, D, H, parts):
    """Codes and scales bit for bit, however the tokens arrive; then every row read back."""
    C = _C()
    torch.manual_seed(sum(parts) + D)
    L, S, slot = sum(parts), 3, 1
    nb = L // BLK + 1
    cache = _alloc(S, H, nb, D, fmt)
    before = [t.clone() for t in cache]
    k = torch.randn(L, H, D, device="cuda").bfloat16()
    wide = torch.randn(L, 3 * H * D, device="cuda").bfloat16()  # v: a column slice of a projection
    v = wide[:, H * D:2 * H * D].view(L, H, D)
    kh = k.transpose(0, 1).contiguous().transpose(0, 1)         # k: head-major rows
    p = 0
    for n in parts:
        C.kv8_append(kh[p:p + n], v[p:p + n], *cache, slot, p)
        p += n
    full = L // BLK
    for x, rows, code, scale, keys in (("k", k, 0, 2, True), ("v", v, 1, 3, False)):
        want, codes, scales = _model(rows, fmt)
        assert torch.equal(_code_rows(cache[code], slot, full, keys), codes), x
        assert torch.equal(cache[scale][slot, :, :full], scales), x
        for start in {0, min(L - 1, 3), L - 1}:
            ko = torch.full((H, L - start, D), float("nan"), dtype=torch.bfloat16, device="cuda")
            vo = ko.clone()
            C.kv8_read(*cache, slot, L, start, ko, vo)
            got = ko if keys else vo
            assert torch.equal(got, want.float()[:, start:].bfloat16()), (x, start)
    for t, old in zip(cache, before):  # other slots, and blocks past the sequence, are untouched
        assert torch.equal(t[0].view(torch.uint8), old[0].view(torch.uint8))
        assert torch.equal(t[2].view(torch.uint8), old[2].view(torch.uint8))
    assert torch.equal(cache[0][slot, :, full:].view(torch.uint8), before[0][slot, :, full:].view(torch.uint8))
    assert torch.equal(cache[1][slot, :, full:].view(torch.uint8), before[1][slot, :, full:].view(torch.uint8))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_append_unaligned_rows(fmt):
    """Rows that start on odd elements, with an odd row stride."""
    C = _C()
    torch.manual_seed(3)
    T, H, D = 70, 2, 128
    cache, ref = _alloc(1, H, 4, D, fmt), _alloc(1, H, 4, D, fmt)
    k = torch.randn(T, H * D + 3, device="cuda").bfloat16()[:, 1:1 + H * D].unflatten(1, (H, D))
    v = torch.randn(T, H * D + 5, device="cuda").bfloat16()[:, 3:3 + H * D].unflatten(1, (H, D))
    C.kv8_append(k, v, *cache, 0, 5)
    C.kv8_append(k.contiguous(), v.contiguous(), *ref, 0, 5)
    for a, b in zip(cache, ref):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_append_special_values(fmt):
    """Zero blocks, values at the ends of bf16's range, ties, infinities and NaN."""
    C = _C()
    torch.manual_seed(4)
    H, D = 1, 64
    k = torch.randn(5 * BLK, H, D, device="cuda").bfloat16()
    k[:BLK] = 0
    k[BLK:2 * BLK] *= 2.0 ** 120
    k[2 * BLK:3 * BLK] *= 2.0 ** -90
    k[3 * BLK, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0], device="cuda")
    k[4 * BLK:, 0] = torch.linspace(-1, 1, 64, device="cuda").bfloat16()  # max / 2 is a tie for int8
    k[4 * BLK, 0, 5] = 0.5
    v = (k * 1e-38).bfloat16()  # below the smallest maximum that counts
    cache = _alloc(1, H, 5, D, fmt)
    C.kv8_append(k, v, *cache, 0, 0)
    for rows, code, scale, keys in ((k, 0, 2, True), (v, 1, 3, False)):
        _, codes, scales = _model(rows, fmt)
        assert torch.equal(_code_rows(cache[code], 0, 5, keys), codes)
        assert torch.equal(cache[scale][0], scales)


def _filled(S, H, D, fmt, lens, extra=1, seed=0):
    """A cache whose slot s holds lens[s] random tokens; returns it with the rows' bf16 originals."""
    C = _C()
    g = torch.Generator(device="cuda").manual_seed(seed)
    nb = max(lens) // BLK + extra
    cache = _alloc(S, H, nb, D, fmt)
    rows = []
    for s, L in enumerate(lens):
        k = torch.randn(L, H, D, generator=g, device="cuda").bfloat16()
        v = torch.randn(L, H, D, generator=g, device="cuda").bfloat16()
        if L:
            C.kv8_append(k, v, *cache, s, 0)
        rows.append((k, v))
    return cache, rows


def _norm_rope64(x, w, pos, inv_freq, rot, eps):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if rot:
        a, h = (torch.tensor(float(pos)) .cuda() * inv_freq).double(), rot // 2  # the angle is an f32 product
        lo, hi = x[..., :h], x[..., h:rot]
        x = torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin(), x[..., rot:]], -1)
    return x


DECODE = [
    # D, Hkv, G, gated, rot, lengths of the slots before the new token
    (64, 2, 3, False, 0, [0, 5]),
    (64, 1, 1, True, 64, [31, 32, 63]),
    (128, 8, 4, False, 128, [700, 1]),
    (128, 4, 16, False, 128, [1500, 31, 95]),
    (128, 1, 7, True, 32, [33]),
    (128, 2, 8, False, 0, [4095, 0, 64, 1000, 31, 62, 2000, 17]),
    (256, 2, 8, True, 64, [1900, 700]),
    (256, 1, 5, False, 256, [30, 31, 0]),
    (256, 1, 16, True, 64, [330, 31]),
    # more pairs than CTAs: each takes several units; and one long sequence among empty ones
    (64, 8, 2, False, 64, [(i * 37) % 90 for i in range(48)]),
    (128, 2, 4, False, 128, [0] * 9 + [6001] + [1] * 30),
]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("D,H,G,gated,rot,lens", DECODE)
def test_attn_decode_kv8(fmt, D, H, G, gated, rot, lens):
    """One step for a ragged batch on permuted slots; twice, since a step may be repeated."""
    C = _C()
    torch.manual_seed(D + G)
    B, Hq, eps = len(lens), H * G, 1e-6
    cache, rows = _filled(B + 1, H, D, fmt, lens + [50], seed=G)
    order = torch.randperm(B)
    slots = order.to(torch.int32).cuda()
    pos = torch.tensor(lens + [50], dtype=torch.int32, device="cuda")
    qw = 2 * D if gated else D
    proj = torch.randn(B, Hq * qw + 2 * H * D + 8, device="cuda").bfloat16()
    qn = torch.rand(D, device="cuda") + 0.5 if rot else None
    kn = torch.rand(D, device="cuda") + 0.5 if rot else None
    delta = torch.randint(-3, 4, (B + 1,), dtype=torch.int32, device="cuda").clamp_(min=0) if rot else None
    inv = 1e6 ** (-torch.arange(0, max(rot, 2), 2, device="cuda").float() / max(rot, 2))
    ws = C.kv8_workspace(B, Hq, H, D)
    out = torch.full((B, Hq * D), float("nan"), dtype=torch.bfloat16, device="cuda")
    for _ in range(2):
        C.attn_decode_kv8(proj, qn, kn, inv, *cache, slots, pos, ws, out, Hq, rot, gated, eps, delta)
    assert int(ws[0]) == 0
    for b in range(B):
        s = int(order[b])
        p = lens[s]
        x = proj[b]
        rp = p + (int(delta[s]) if rot else 0)
        q = _norm_rope64(x[:Hq * qw].view(Hq, qw)[:, :D], qn, rp, inv, rot, eps)
        k = _norm_rope64(x[Hq * qw:Hq * qw + H * D].view(H, D), kn, rp, inv, rot, eps)
        v = x[Hq * qw + H * D:Hq * qw + 2 * H * D].view(H, D)
        # the new row as the cache holds it: the nearest bf16, or its neighbour
        kt = cache[4][s].permute(0, 2, 1, 3).reshape(H, BLK, D)[:, p % BLK]
        assert bool(((kt.double() - k).abs() <= 2.0 ** -8 * k.abs() + 1e-5).all())
        assert torch.equal(cache[5][s].permute(0, 3, 1, 2).reshape(H, BLK, D)[:, p % BLK], v)
        kk = torch.cat([rows[s][0], kt[None]])
        vv = torch.cat([rows[s][1], v[None]])
        kr, kcodes, kscales = _model(kk, fmt)
        vr, vcodes, vscales = _model(vv, fmt)
        n = (p + 1) // BLK
        assert torch.equal(_code_rows(cache[0], s, n, True), kcodes)
        assert torch.equal(_code_rows(cache[1], s, n, False), vcodes)
        assert torch.equal(cache[2][s, :, :n], kscales) and torch.equal(cache[3][s, :, :n], vscales)
        o = _attend(q[None], kr, vr, p, D ** -0.5)[0]
        if gated:
            o = o * torch.sigmoid(x[:Hq * qw].view(Hq, qw)[:, D:].double())
        _check(out[b].view(Hq, D), o, float(vr.abs().max()))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_decode_steps_equal_one_append(fmt):
    """Seventy single-token steps leave the cache that one append of the same rows leaves."""
    C = _C()
    torch.manual_seed(9)
    H, G, D, n = 2, 4, 128, 70
    Hq = H * G
    cache, ref = _alloc(1, H, 3, D, fmt), _alloc(1, H, 3, D, fmt)
    proj = torch.randn(n, 1, Hq * D + 2 * H * D, device="cuda").bfloat16()
    inv, pos = torch.ones(1, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws, out = C.kv8_workspace(1, Hq, H, D), torch.empty(1, Hq * D, dtype=torch.bfloat16, device="cuda")
    for t in range(n):
        pos.fill_(t)
        C.attn_decode_kv8(proj[t], None, None, inv, *cache, slots, pos, ws, out, Hq, 0, False, 1e-6)
    kv = proj[:, 0, Hq * D:].view(n, 2, H, D)
    C.kv8_append(kv[:, 0], kv[:, 1], *ref, 0, 0)
    for a, b in zip(cache[:4], ref[:4]):
        assert torch.equal(a[:, :, :2].view(torch.uint8), b[:, :, :2].view(torch.uint8))
    r = n % BLK
    assert torch.equal(cache[4][..., :r, :], ref[4][..., :r, :]) and torch.equal(cache[5][..., :r], ref[5][..., :r])


PREFILL = [
    # T, p0, D, Hq, Hkv, gated
    (1, 0, 64, 4, 2, False),
    (1, 100, 64, 4, 2, True),
    (5, 3, 128, 7, 1, False),
    (31, 1, 256, 8, 1, True),
    (33, 31, 128, 8, 8, False),
    (64, 0, 128, 4, 4, False),
    (70, 33, 64, 3, 1, False),
    (127, 129, 256, 5, 1, False),
    (200, 0, 256, 16, 2, True),
    (300, 64, 128, 16, 1, True),
    (513, 700, 64, 8, 2, False),
    (1030, 7, 128, 8, 2, False),
    (9, 3000, 128, 32, 8, False),
    (3, 2500, 256, 4, 1, True),     # keys split over CTAs at head dim 256
    (1, 5000, 64, 2, 2, False),
    (40, 4100, 128, 8, 1, True),    # split, two row tiles
]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("T,p0,D,Hq,H,gated", PREFILL)
def test_attn_prefill_kv8(fmt, T, p0, D, Hq, H, gated):
    C = _C()
    torch.manual_seed(T + p0)
    cache, rows = _filled(2, H, D, fmt, [40, p0 + T], seed=T)
    q = 1.5 * torch.randn(T, Hq * D + 8, device="cuda")
    q = q.bfloat16()[:, :Hq * D]
    gate = torch.randn(T, Hq * 2 * D, device="cuda").bfloat16()[:, D:] if gated else None
    out = torch.full((T, Hq * D + 16), float("nan"), dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    C.attn_prefill_kv8(q, *cache, 1, p0, out[:, :Hq * D], Hq, D ** -0.5, gate, 2 * D, err)
    assert int(err) == 0
    kr, vr = _model(rows[1][0], fmt)[0], _model(rows[1][1], fmt)[0]
    o = _attend(q.double().view(T, Hq, D), kr, vr, p0, D ** -0.5)
    if gated:
        o = o * torch.sigmoid(torch.stack([gate[:, 2 * D * h:2 * D * h + D] for h in range(Hq)], 1).double())
    _check(out[:, :Hq * D].view(T, Hq, D), o, float(vr.abs().max()))
    assert bool(out[:, Hq * D:].isnan().all())


@pytest.mark.parametrize("D,gated", [(64, True), (128, False), (256, True)])
def test_unaligned_operands_give_the_same_bits(D, gated):
    """Projections, queries, gates and outputs that start on odd elements or have odd row strides."""
    C = _C()
    torch.manual_seed(D)
    H, G, B = 2, 4, 2
    Hq, qw = H * G, 2 * D if gated else D
    inv = 1e4 ** (-torch.arange(0, D, 2, device="cuda").float() / D)
    wide = torch.randn(B, Hq * qw + 2 * H * D + 7, device="cuda").bfloat16()
    outs = []
    for proj in (wide[:, 3:3 + Hq * qw + 2 * H * D], wide[:, 3:3 + Hq * qw + 2 * H * D].contiguous()):
        cache, _ = _filled(B, H, D, "int8", [300, 63], seed=5)
        pos = torch.tensor([300, 63], dtype=torch.int32, device="cuda")
        out = torch.empty(B, Hq * D, dtype=torch.bfloat16, device="cuda")
        C.attn_decode_kv8(proj, None, None, inv, *cache, torch.arange(B, dtype=torch.int32, device="cuda"), pos,
                          C.kv8_workspace(B, Hq, H, D), out, Hq, D, gated, 1e-6)
        outs.append([out, *cache])
    for x, y in zip(*outs):
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
    T = 37
    cache, _ = _filled(1, H, D, "fp8", [T + 100], seed=6)
    q = torch.randn(T, Hq * D + 5, device="cuda").bfloat16()[:, 1:1 + Hq * D]
    gate = torch.randn(T, Hq * 2 * D + 3, device="cuda").bfloat16()[:, 3:] if gated else None
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    a = torch.empty(T, Hq * D + 9, dtype=torch.bfloat16, device="cuda")[:, 5:5 + Hq * D]
    b = torch.empty(T, Hq * D, dtype=torch.bfloat16, device="cuda")
    C.attn_prefill_kv8(q, *cache, 0, 100, a, Hq, D ** -0.5, gate, 2 * D, err)
    C.attn_prefill_kv8(q.contiguous(), *cache, 0, 100, b, Hq, D ** -0.5, gate.contiguous() if gated else None, 2 * D, err)
    assert int(err) == 0 and torch.equal(a, b)


def test_offsets_past_32_bits():
    """The second slot of a cache whose slots are 4.6 GB each, and positions at its far end."""
    C = _C()
    torch.manual_seed(2)
    H, D, nb = 1, 128, 1_100_000
    cache = [torch.zeros(2, H, nb, 2, BLK, 64, dtype=torch.int8, device="cuda"),
             torch.zeros(2, H, nb, 2, 64, BLK, dtype=torch.int8, device="cuda"),
             torch.zeros(2, H, nb, device="cuda"), torch.zeros(2, H, nb, device="cuda"),
             torch.zeros(2, H, 2, BLK, 64, dtype=torch.bfloat16, device="cuda"),
             torch.zeros(2, H, 2, 64, BLK, dtype=torch.bfloat16, device="cuda")]
    k, v = torch.randn(2, 70, H, D, device="cuda").bfloat16()
    q = torch.randn(5, 4 * D, device="cuda").bfloat16()
    ko, vo = torch.empty(2, H, 70, D, dtype=torch.bfloat16, device="cuda")
    for p0 in (0, nb * BLK - 96):
        C.kv8_append(k, v, *cache, 1, p0)
        C.kv8_read(*cache, 1, p0 + 70, p0, ko, vo)
        kr, vr = _model(k, "int8")[0], _model(v, "int8")[0]
        assert torch.equal(ko, kr.float().bfloat16()) and torch.equal(vo, vr.float().bfloat16())
        if p0:
            continue
        out, err = torch.empty(5, 4 * D, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        C.attn_prefill_kv8(q, *cache, 1, 65, out, 4, D ** -0.5, None, 0, err)
        _check(out.view(5, 4, D), _attend(q.double().view(5, 4, D), kr, vr, 65, D ** -0.5), float(vr.abs().max()))
        proj = torch.cat([q[:1], k[69:70].view(1, D), v[69:70].view(1, D)], 1)
        o = torch.empty(1, 4 * D, dtype=torch.bfloat16, device="cuda")
        C.attn_decode_kv8(proj, None, None, torch.ones(1, device="cuda"), *cache,
                          torch.ones(1, dtype=torch.int32, device="cuda"), torch.tensor([0, 69], dtype=torch.int32, device="cuda"),
                          C.kv8_workspace(1, 4, H, D), o, 4, 0, False, 1e-6)
        _check(o.view(4, D), _attend(q[:1].double().view(1, 4, D), kr, vr, 69, D ** -0.5)[0], float(vr.abs().max()))
    assert not cache[0][0].any()


def test_workspace_serves_every_batch_it_was_made_for():
    """One scratch for 48 sequences, then one, then 48: counters and partials keep apart."""
    C = _C()
    H, G, D = 2, 2, 64
    lens = [700 + 40 * i for i in range(48)]
    cache, rows = _filled(48, H, D, "int8", lens, extra=2)
    pos = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = C.kv8_workspace(48, H * G, H, D)
    proj = torch.randn(48, (H * G + 2 * H) * D, device="cuda").bfloat16()
    inv = torch.ones(1, device="cuda")

    def step(at, ws):
        out = torch.empty(len(at), H * G * D, dtype=torch.bfloat16, device="cuda")
        C.attn_decode_kv8(proj[at], None, None, inv, *cache, torch.tensor(at, dtype=torch.int32, device="cuda"), pos, ws,
                          out, H * G, 0, False, 1e-6)
        return out
    for at in (list(range(48)), [5], [47, 3], list(range(48)), [0]):
        assert torch.equal(step(at, ws), step(at, C.kv8_workspace(len(at), H * G, H, D))), at
    assert int(ws[0]) == 0


def test_decode_extreme_values():
    """Keys and values near bf16's ends, and a query whose norm is large: the scales carry them."""
    C = _C()
    torch.manual_seed(12)
    H, D, L = 1, 128, 130
    for fmt in ("int8", "fp8"):
        for kmul, vmul, qmul in ((2.0 ** -60, 2.0 ** 90, 2.0 ** 60), (2.0 ** 40, 2.0 ** -40, 2.0 ** -40)):
            cache = _alloc(1, H, 5, D, fmt)
            k = (torch.randn(L, H, D, device="cuda") * kmul).bfloat16()
            v = (torch.randn(L, H, D, device="cuda") * vmul).bfloat16()
            C.kv8_append(k[:-1], v[:-1], *cache, 0, 0)
            q = (torch.randn(1, D, device="cuda") * qmul).bfloat16()
            proj = torch.cat([q, k[-1], v[-1]], 1)
            out = torch.empty(1, D, dtype=torch.bfloat16, device="cuda")
            pos = torch.full((1,), L - 1, dtype=torch.int32, device="cuda")
            C.attn_decode_kv8(proj, None, None, torch.ones(1, device="cuda"), *cache, torch.zeros_like(pos), pos,
                              C.kv8_workspace(1, 1, H, D), out, 1, 0, False, 1e-6)
            kr, vr = _model(k, fmt)[0], _model(v, fmt)[0]
            want = _attend(q.double()[None].view(1, 1, D), kr, vr, L - 1, D ** -0.5)[0]
            _check(out, want, float(vr.abs().max()))
            o2 = torch.empty(1, D, dtype=torch.bfloat16, device="cuda")
            err = torch.zeros(1, dtype=torch.int32, device="cuda")
            C.kv8_append(k[-1:], v[-1:], *cache, 0, L - 1)
            C.attn_prefill_kv8(q, *cache, 0, L - 1, o2, 1, D ** -0.5, None, 0, err)
            _check(o2, want, float(vr.abs().max()))


def test_decode_refuses_positions_outside():
    """A slot or position outside the cache touches nothing: zero row, error word; others go on."""
    C = _C()
    torch.manual_seed(1)
    H, D = 1, 64
    cache, rows = _filled(2, H, D, "int8", [20, 20])
    before = [t.clone() for t in cache]
    proj = torch.randn(3, 3 * D, device="cuda").bfloat16()
    out = torch.full((3, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    ws = C.kv8_workspace(3, 1, H, D)
    slots = torch.tensor([5, 1, 0], dtype=torch.int32, device="cuda")
    pos = torch.tensor([20, 10 ** 6], dtype=torch.int32, device="cuda")
    C.attn_decode_kv8(proj, None, None, torch.ones(1, device="cuda"), *cache, slots, pos, ws, out, 1, 0, False, 1e-6)
    assert int(ws[0]) == 6001
    assert bool((out[:2] == 0).all()) and bool(out[2].isfinite().all()) and bool((out[2] != 0).any())
    for t, old in zip(cache, before):
        assert torch.equal(t[1].view(torch.uint8), old[1].view(torch.uint8))


def test_refusals():
    C = _C()
    H, D = 2, 128
    cache = _alloc(2, H, 4, D, "int8")
    k = torch.zeros(4, H, D, dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def bad(fn, *a):
        with pytest.raises(RuntimeError):
            fn(*a)
    bad(C.kv8_append, k, k, *cache, 2, 0)                      # slot
    bad(C.kv8_append, k, k, *cache, -1, 0)
    bad(C.kv8_append, k, k, *cache, 0, 125)                    # past the cache
    bad(C.kv8_append, k, k, *cache, 0, -1)
    bad(C.kv8_append, k.float(), k, *cache, 0, 0)              # type
    bad(C.kv8_append, k[:, :1], k[:, :1], *cache, 0, 0)        # heads
    bad(C.kv8_append, k, k[:2], *cache, 0, 0)                  # lengths differ
    bad(C.kv8_append, k.cpu(), k, *cache, 0, 0)                # device
    bad(C.kv8_append, k, k, cache[1], cache[0], *cache[2:], 0, 0)          # layouts swapped
    bad(C.kv8_append, k, k, cache[0], cache[1].view(torch.float8_e4m3fn), *cache[2:], 0, 0)
    o = torch.empty(H, 4, D, dtype=torch.bfloat16, device="cuda")
    bad(C.kv8_read, *cache, 0, 3, 0, o, o)                     # more rows than tokens
    bad(C.kv8_read, *cache, 0, 129, 0, o, o)
    bad(C.kv8_read, *cache, 0, 100, -1, o, o)
    bad(C.kv8_read, *cache, 0, 100, 0, o, o[:, :, :64])
    q, out = torch.zeros(4, 4 * D, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 4 * D, dtype=torch.bfloat16, device="cuda")
    bad(C.attn_prefill_kv8, q, *cache, 0, 0, out, 3, 1.0, None, 0, err)    # 3 heads over 2
    bad(C.attn_prefill_kv8, q, *cache, 0, 125, out, 4, 1.0, None, 0, err)
    bad(C.attn_prefill_kv8, q, *cache, 0, 0, out[:3], 4, 1.0, None, 0, err)
    bad(C.attn_prefill_kv8, q, *cache, 0, 0, out, 4, 1.0, out, 2 * D, err)  # gate too narrow
    ws = C.kv8_workspace(2, 4, H, D)
    slots = torch.zeros(2, dtype=torch.int32, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    proj = torch.zeros(2, 8 * D, dtype=torch.bfloat16, device="cuda")
    inv = torch.ones(64, device="cuda")
    o2 = torch.zeros(2, 4 * D, dtype=torch.bfloat16, device="cuda")
    ok = (proj, None, None, inv, *cache, slots, pos, ws, o2, 4, 128, False, 1e-6)
    C.attn_decode_kv8(*ok)

    def but(i, x):
        a = list(ok)
        a[i] = x
        bad(C.attn_decode_kv8, *a)
    but(0, proj[:, :7 * D])
    but(0, proj[:1])
    but(1, torch.ones(64, device="cuda"))
    but(3, inv[:10])
    but(10, slots.long())
    but(11, pos[:1])
    but(12, torch.zeros(1, dtype=torch.int32, device="cuda"))
    but(13, o2[:, :D])
    but(14, 3)
    but(15, 129)
    but(15, 130)
    bad(C.kv8_workspace, 0, 4, 2, 128)
    bad(C.kv8_workspace, 257, 4, 2, 128)
    big = torch.zeros(3, 8 * D, dtype=torch.bfloat16, device="cuda")
    bad(C.attn_decode_kv8, big, None, None, inv, *cache, torch.zeros(3, dtype=torch.int32, device="cuda"), pos, ws[:-1],
        torch.zeros(3, 4 * D, dtype=torch.bfloat16, device="cuda"), 4, 128, False, 1e-6)
    bad(C.kv8_workspace, 1, 3, 2, 128)
    bad(C.kv8_workspace, 1, 4, 2, 96)
    C.kv8_append(k[:0], k[:0], *cache, 0, 0)                   # nothing to do
    C.attn_prefill_kv8(q[:0], *cache, 0, 0, out[:0], 4, 1.0, None, 0, err)


def test_other_stream():
    """Operators run on the caller's stream: tensors made on a side stream, used there."""
    C = _C()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        cache, rows = _filled(1, 2, 64, "int8", [100])
        o = torch.empty(2, 100, 64, dtype=torch.bfloat16, device="cuda")
        v = torch.empty_like(o)
        C.kv8_read(*cache, 0, 100, 0, o, v)
    s.synchronize()
    assert torch.equal(o, _model(rows[0][0], "int8")[0].float().bfloat16())
