"""Token runs and shared prefixes over the paged KV cache: append, run (prefill)
attention and shared-prefix decode against plain 64-bit implementations.

Bounds on an attention output o = sum p v / sum p, elementwise, with
A = sum p |v| / sum p and S = max_j sum_i |q_i k_ij| / 16 of the row:
  f32   q and p enter the tensor cores as f16 hi + lo (2^-22 relative each) and
        products accumulate in chains of at most 32 steps per score (2^-23 of S a
        step, truncated) and (positions / 8 + 64) steps per output:
        |ds| <= 2^-17 S, |do| <= 2 |ds| A + (n / 8 + 64) 2^-23 A.
  f16   besides that, p is rounded to f16 once (2^-11 A) and the result once
        (2^-11 |o|).
  f16 over q8_0 planes: K and V values d * q are rounded to f16 too:
        |ds| += 2^-11 S, |do| += 2^-11 A.
The sigmoid gate (at most 1) multiplies all of it, with 2^-22 |o| of its own.
"""
import ctypes as C
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from qwowl35_b200 import _lib

ROOT = Path(__file__).resolve().parent.parent
H, KV, D, CH = 16, 4, 256, 256
Q8ROW = 272
EPS = 1e-6


# ---- a cache and its plain reading -------------------------------------------------------

class Cache:
    """Shuffled chunks of two layers (the second is the one in use); everything unwritten is NaN (q8_0: NaN scales)."""

    def __init__(self, lengths, q8, seed, max_chunks=None):
        self.q8 = q8
        self.plane = KV * CH * (Q8ROW if q8 else 2 * D)
        self.k_off, self.v_off = 2 * self.plane, 3 * self.plane
        counts = [-(-n // CH) for n in lengths]
        g = torch.Generator().manual_seed(seed)
        perm = torch.randperm(max(1, sum(counts)), generator=g)
        self.raw = torch.zeros(max(1, sum(counts)), 4, self.plane, dtype=torch.uint8, device="cuda")
        if q8:
            self.raw.view(-1, 34)[:, :2] = torch.tensor([0, 0x7e], dtype=torch.uint8, device="cuda")
        else:
            self.raw.view(torch.float16).fill_(float("nan"))
        self.ids = torch.full((len(lengths), max_chunks or max(1, max(counts))), -1, dtype=torch.int64)
        at = 0
        for i, c in enumerate(counts):
            self.ids[i, :c] = perm[at:at + c]
            at += c

    def ptrs(self):
        """The chunk table; entries that no chunk backs are 0."""
        t = self.raw.data_ptr() + self.ids * 4 * self.plane
        return torch.where(self.ids >= 0, t, torch.zeros_like(t)).cuda()

    def rows(self):
        """The layer's planes as [chunk, K or V, head, position, row]: f16 values, or q8_0 bytes [8, 34]."""
        part = self.raw[:, 2:]
        if self.q8:
            return part.view(-1, 2, KV, CH, 8, 34)
        return part.view(torch.float16).view(-1, 2, KV, CH, D)

    def values(self):
        """What the planes stand for, in 64 bits."""
        r = self.rows()
        if self.q8:
            return (r[..., 2:].view(torch.int8).double() * r[..., :2].view(torch.float16).double()).flatten(-2)
        return r.double()

    def fill(self, lengths, seed, scale=1.0):
        """Random rows at positions [0, lengths[i]) of every sequence."""
        g = torch.Generator("cuda").manual_seed(seed)
        rows = self.rows()
        for i, n in enumerate(lengths):
            for c in range(-(-n // CH)):
                m = min(CH, n - c * CH)
                part = rows[int(self.ids[i, c])][:, :, :m]
                if self.q8:
                    part[..., 2:] = torch.randint(-127, 128, part.shape[:-1] + (32,), dtype=torch.int8, device="cuda",
                                                  generator=g).view(torch.uint8)
                    d = (0.5 + torch.rand(part.shape[:-1] + (1,), device="cuda", generator=g)) * scale * 1.7 / 127
                    part[..., :2] = d.half().view(torch.uint8)
                else:
                    part.copy_(torch.randn(part.shape, device="cuda", generator=g) * scale)
        return self

    def sequence(self, i, n):
        """K, V [head, n, dim] of sequence i in 64 bits."""
        v = self.values()[self.ids[i, :-(-n // CH)].cuda()] if n else self.values()[:0]
        kv = v.permute(1, 2, 0, 3, 4).reshape(2, KV, -1, D)[:, :, :n]
        return kv[0], kv[1]


def attend(q, gate, k, v, length, window=0, sink=0):
    """One row: q, gate [16, 256] -> (o, A, S) of the formulas above, 64 bits."""
    q = q.double().view(KV, H // KV, D)
    j = torch.arange(k.shape[1], device="cuda")
    keep = j < length
    few = min(sink, max(length, 0))
    if window > 0 and few + window < length:
        keep &= (j < few) | (j >= length - window)
    sig = torch.sigmoid(gate.double()) if gate is not None else torch.ones(H, D, device="cuda", dtype=torch.float64)
    if not bool(keep.any()):
        z = torch.zeros(H, D, dtype=torch.float64, device="cuda")
        return z, z, torch.zeros(H, 1, dtype=torch.float64, device="cuda")
    k, v = k[:, keep], v[:, keep]
    s = q @ k.transpose(1, 2) / math.sqrt(D)
    p = torch.softmax(s, -1)
    big = (q.abs() @ k.abs().transpose(1, 2)).amax(-1) / math.sqrt(D)
    return (p @ v).view(H, D) * sig, (p @ v.abs()).view(H, D) * sig, big.view(H, 1)


def bound(o, a, s, n, half, q8):
    ds = 2.0 ** -17 * s
    extra = (n / 8 + 64) * 2.0 ** -23 * a + 2.0 ** -22 * o.abs()
    if half:
        extra = extra + 2.0 ** -11 * a + 2.0 ** -11 * o.abs() + 2.0 ** -24
        if q8:
            ds = ds + 2.0 ** -11 * s
            extra = extra + 2.0 ** -11 * a
    return torch.expm1(2 * ds) * a + extra + 1e-30


def check_rows(out, rows, half, q8):
    """rows: [(row of out, o, A, S, context length)]."""
    worst = 0.0
    for r, o, a, s, n in rows:
        y = out[r].double().view(H, D)
        assert torch.isfinite(y).all(), r
        worst = max(worst, float(((y - o).abs() / bound(o, a, s, max(n, 0), half, q8)).max()))
    assert worst <= 1.0, worst


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def some(n, seed, kind, scale=1.5):
    g = torch.Generator("cuda").manual_seed(seed)
    return (scale * torch.randn(n, H, D, device="cuda", generator=g)).to(kind)


# ---- append -----------------------------------------------------------------------------

def append_reference(qkv, qw, kw, freq, pos, axis):
    """q, gate [n, 16, 256], k, v [n, 4, 256] in 64 bits; pos [axes, n], axis [32]."""
    x = qkv[:, :10240].double()
    n = x.shape[0]
    ang = torch.stack([pos[a].double() * freq[i].double() for i, a in enumerate(axis)], 1)[:, None]
    c, s = ang.cos(), ang.sin()

    def head(y, w):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
        lo, hi = y[..., :32].clone(), y[..., 32:64].clone()
        y[..., :32], y[..., 32:64] = lo * c - hi * s, lo * s + hi * c
        return y

    full = x[:, :8192].view(n, H, 2, D)
    kv = x[:, 8192:].view(n, 2, KV, D)
    return head(full[:, :, 0].clone(), qw), full[:, :, 1], head(kv[:, 0].clone(), kw), kv[:, 1]


def axes_of(sections, interleaved):
    if interleaved and len(sections) == 3:
        return [i % 3 if i % 3 and i < 3 * sections[i % 3] else 0 for i in range(32)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


FREQ = (1e7 ** (-torch.arange(32, dtype=torch.float64) / 32)).float()


def near(y, ref, kind, norm):
    """f32: 2^-20 of the row's scale `norm` (a 256-term sum, rsqrt and the turn: some 16 roundings of 2^-24); f16: that and half a step."""
    tol = 2.0 ** -20 * norm + (2.0 ** -11 * ref.abs() + 2.0 ** -24 if kind == torch.float16 else 0)
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("sections,interleaved", [((32,), True), ((11, 11, 10), True), ((11, 11, 10), False), ((20, 12), False),
                                                  ((32, 0, 0), True)])
def test_append_matches_the_formulas(half, q8, sections, interleaved):
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    # tokens of three rows in mixed order, chunk borders and the far end of the table, one padding token
    where = [(0, 0), (2, 255), (2, 256), (1, 511), (0, 1), (-1, 7), (2, 257), (1, 300), (0, 767)]
    c = Cache([768, 512, 300], q8, 3)
    n = len(where)
    g = torch.Generator("cuda").manual_seed(11)
    wide = torch.randn(n, 10400, device="cuda", generator=g) * 3
    qkv = wide[:, 4:10300] if half else wide[:, 3:10300]  # strided rows, also off a 16-byte border
    qw, kw = (1 + 0.2 * torch.randn(256, device="cuda", generator=g) for _ in range(2))
    pos = torch.randint(0, 262144, (len(sections), n), generator=torch.Generator().manual_seed(4)).int().cuda()
    pos[:, 0] = 262143
    seq, at = ints(*[w[0] for w in where]), ints(*[w[1] for w in where])
    before = c.raw.clone()
    q0 = torch.full((n, H, D), 7.0, dtype=kind, device="cuda")
    q, gate = ops.attn_append(qkv, qw, kw, FREQ.cuda(), pos, sections, seq, at, c.ptrs(), c.k_off, c.v_off, eps=EPS,
                              interleaved=interleaved, dtype=kind, kv_q8=q8, q=q0, gate=q0.clone())
    rq, rg, rk, rv = append_reference(qkv, qw, kw, FREQ.cuda(), pos, axes_of(sections, interleaved))
    real = [t for t in range(n) if where[t][0] >= 0]
    near(q[real], rq[real], kind, rq.abs().amax(-1, keepdim=True)[real])
    assert torch.equal(gate[real], rg[real].to(kind))
    assert bool((q[5] == 7).all()) and bool((gate[5] == 7).all())
    touched = torch.zeros(c.raw.shape[:2] + (KV, CH), dtype=torch.bool)
    rows = c.rows()
    for t in real:
        s, p = where[t]
        chunk = int(c.ids[s, p // CH])
        touched[chunk, 2:, :, p % CH] = True
        k, v = rows[chunk, 0, :, p % CH], rows[chunk, 1, :, p % CH]
        if q8:
            for got, ref in ((k, rk[t]), (v, rv[t])):
                blocks = ref.view(KV, 8, 32)
                d = blocks.abs().amax(-1, keepdim=True) / 127
                value = got[..., 2:].view(torch.int8).double() * got[..., :2].view(torch.float16).double()
                # half a step of d, the stored d's own rounding on up to 127 steps, and the f32 work before it
                assert bool(((value - blocks).abs() <= d * (0.5 + 127 * 2.0 ** -11 + 0.01)).all())
        else:
            near(k, rk[t], torch.float16, rk[t].abs().amax(-1, keepdim=True))
            assert torch.equal(v, rv[t].half())
    same = (c.raw.view(*c.raw.shape[:2], KV, CH, -1) == before.view(*c.raw.shape[:2], KV, CH, -1)).all(-1).cpu()
    assert bool(same[~touched].all())


@pytest.mark.gpu
@pytest.mark.parametrize("half,q8", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("n,off", [(148, 0), (591, 0), (1500, 0), (1500, 1)])
def test_append_of_many_tokens(half, q8, n, off):
    """One to eleven tokens an SM, a padding token among every 37; off: rows that no 16-byte copy can fetch."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    c = Cache([n], q8, 3)
    g = torch.Generator("cuda").manual_seed(n + off)
    qkv = torch.randn(n, 10240 + 8, device="cuda", generator=g)[:, off:10240 + off]
    qw, kw = (1 + 0.2 * torch.randn(256, device="cuda", generator=g) for _ in range(2))
    pos = torch.randint(0, 262144, (3, n), generator=torch.Generator().manual_seed(n)).int().cuda()
    t = torch.arange(n, device="cuda")
    pad = t % 37 == 5
    seq = torch.where(pad, -1, 0).int()
    at = ((t * 7919) % n).int()
    q0 = torch.full((n, H, D), 7.0, dtype=kind, device="cuda")
    before = c.rows().clone()
    q, gate = ops.attn_append(qkv, qw, kw, FREQ.cuda(), pos, (11, 11, 10), seq, at, c.ptrs(), c.k_off, c.v_off, eps=EPS, dtype=kind,
                              kv_q8=q8, q=q0, gate=q0.clone())
    rq, rg, rk, rv = append_reference(qkv, qw, kw, FREQ.cuda(), pos, axes_of((11, 11, 10), True))
    near(q[~pad], rq[~pad], kind, rq.abs().amax(-1, keepdim=True)[~pad])
    assert torch.equal(gate[~pad], rg[~pad].to(kind))
    assert bool((q[pad] == 7).all()) and bool((gate[pad] == 7).all())
    chunk, p = c.ids[0].cuda()[at.long() // CH], at.long() % CH
    k, v = c.rows()[chunk, 0, :, p], c.rows()[chunk, 1, :, p]
    old = before[chunk, :, :, p]
    assert torch.equal(torch.stack([k, v], 1)[pad].view(torch.uint8), old[pad].view(torch.uint8))
    if q8:
        for got, ref in ((k, rk), (v, rv)):
            blocks = ref.view(n, KV, 8, 32)[~pad]
            d = blocks.abs().amax(-1, keepdim=True) / 127
            value = (got[..., 2:].view(torch.int8).double() * got[..., :2].view(torch.float16).double())[~pad]
            assert bool(((value - blocks).abs() <= d * (0.5 + 127 * 2.0 ** -11 + 0.01)).all())
    else:
        near(k[~pad], rk[~pad], torch.float16, rk.abs().amax(-1, keepdim=True)[~pad])
        assert torch.equal(v[~pad], rv[~pad].half())
    assert _lib.lib().qw35_cuda_device_error() == 0


@pytest.mark.gpu
def test_append_agrees_with_the_single_token_preprocess():
    """One axis and near positions (where the f32 angle is exact enough): the same cache rows, q and gate."""
    from qwowl35_b200 import ops
    lens = [5, 260]
    g = torch.Generator("cuda").manual_seed(2)
    qkv = torch.randn(2, 10240, device="cuda", generator=g)
    w = 1 + 0.1 * torch.randn(2, 256, device="cuda", generator=g)
    a, b = Cache(lens, False, 1), Cache(lens, False, 1)
    pos = ints(4, 259)
    f = FREQ.cuda()
    q1, g1 = ops.attn_preprocess(qkv, w[0].contiguous(), w[1].contiguous(), f, pos, a.ptrs(), a.k_off, a.v_off)
    q2, g2 = ops.attn_append(qkv, w[0].contiguous(), w[1].contiguous(), f, pos[None].contiguous(), (32,), ints(0, 1), pos, b.ptrs(),
                             b.k_off, b.v_off)
    # the f32 angle of position 259 is off by at most 259 * 2^-24 rad
    assert float((q1 - q2).abs().max()) <= 2.0 ** -15 * float(q2.abs().max()) and torch.equal(g1, g2)
    ka, kb = a.rows().float(), b.rows().float()
    assert torch.equal(ka.isnan(), kb.isnan())
    assert bool(((ka - kb).nan_to_num().abs() <= 2.0 ** -10 * kb.nan_to_num().abs() + 2.0 ** -13).all())


# ---- run attention -----------------------------------------------------------------------

RUNS = [
    [(0, 1)],
    [(4095, 1)],
    [(0, 300)],
    [(255, 2), (1024, 7), (3000, 33), (0, 0), (100, 32)],
    [(0, 31), (0, 32), (0, 33), (127, 1), (128, 1), (129, 64)],
    [(700, 161), (9000, 5)],
]
CUTS = [(0, 0), (1, 0), (200, 4), (128, 300), (2 ** 31 - 1, 2 ** 31 - 1)]


def prefill_case(runs, half, q8, window, sink, gate=True, seed=0, splits=None):
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    lens = [c + r for c, r in runs]
    cache = Cache(lens, q8, seed + 1).fill(lens, seed + 2)
    n = sum(r for _, r in runs)
    q, gt = some(n + 3, seed + 3, kind), some(n + 3, seed + 4, kind, 1.0)
    off = [0]
    for _, r in runs:
        off.append(off[-1] + r)
    out = torch.full((n + 3, H * D), 5.0, dtype=kind, device="cuda")
    ops.gqa_prefill(q, gt if gate else None, ints(*off), ints(*lens), max(r for _, r in runs), max(lens), cache.ptrs(),
                    cache.k_off, cache.v_off, window=window, sink=sink, out=out, kv_q8=q8)
    assert bool((out[n:] == 5).all())  # rows behind the last run
    rows = []
    for i, (c, r) in enumerate(runs):
        k, v = cache.sequence(i, lens[i])
        picks = sorted({0, 1, 30, 31, 32, 63, 64, r // 2, r - 2, r - 1} & set(range(r)))
        for t in picks:
            x = off[i] + t
            rows.append((x, *attend(q[x], gt[x] if gate else None, k, v, c + t + 1, window, sink), c + t + 1))
    check_rows(out, rows, half, q8)
    assert _lib.lib().qw35_cuda_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("runs", RUNS)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q8", [False, True])
def test_prefill_matches_the_formula(runs, half, q8):
    prefill_case(runs, half, q8, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sink", CUTS)
@pytest.mark.parametrize("half,q8", [(True, False), (False, True)])
def test_prefill_window_and_sink(window, sink, half, q8):
    prefill_case([(300, 70), (0, 600), (2000, 3)], half, q8, window, sink)


@pytest.mark.gpu
def test_prefill_without_gate():
    prefill_case([(100, 40)], True, False, 0, 0, gate=False)


@pytest.mark.gpu
def test_prefill_long_context():
    prefill_case([(40000, 64)], False, False, 0, 0, seed=9)
    prefill_case([(70001, 1), (3, 2)], True, True, 0, 0, seed=10)


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
def test_prefill_rows_before_the_context_attend_nothing(half):
    """A run longer than its context length: its first rows see no position and come out zero."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    cache = Cache([40], False, 5).fill([40], 6)
    q, gt = some(50, 1, kind), some(50, 2, kind)
    out = ops.gqa_prefill(q, gt, ints(0, 50), ints(40), 50, 40, cache.ptrs(), cache.k_off, cache.v_off)
    assert bool((out[:10] == 0).all())
    k, v = cache.sequence(0, 40)
    check_rows(out, [(r, *attend(q[r], gt[r], k, v, r - 9), r - 9) for r in range(10, 50, 3)], half, False)


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("scale", [1e-3, 8.0])
def test_prefill_flat_and_peaked_scores(half, scale):
    """Scores near zero (every position counts alike) and scores of hundreds (one position counts)."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    cache = Cache([900], False, 5).fill([900], 6)
    q, gt = some(70, 1, kind, scale), some(70, 2, kind)
    out = ops.gqa_prefill(q, gt, ints(0, 70), ints(900), 70, 900, cache.ptrs(), cache.k_off, cache.v_off)
    k, v = cache.sequence(0, 900)
    check_rows(out, [(r, *attend(q[r], gt[r], k, v, 831 + r), 831 + r) for r in range(0, 70, 7)], half, False)


def poison(cache, i, positions, value, planes=(0, 1)):
    """Writes `value` into a few dims of K and V (q8_0: as a block's d) at positions of sequence i."""
    rows = cache.rows()
    for n, pos in enumerate(positions):
        part = rows[int(cache.ids[i, pos // CH])]
        for plane in planes:
            for head in range(KV):
                if cache.q8:
                    part[plane, head, pos % CH, (3 * n + head) % 8, :2] = torch.tensor([value], dtype=torch.float16).view(torch.uint8).cuda()
                else:
                    part[plane, head, pos % CH, (37 * n + 5 * head) % D] = value


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("inf"), float("nan"), -float("inf")])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q8", [False, True])
def test_prefill_keeps_what_a_row_does_not_attend_from_it(value, half, q8):
    """Infinities and NaNs at later tokens of the run and outside the window reach only the rows that attend them."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    for ctx, rows, at, window, sink in ((300, 40, (320, 339), 0, 0), (0, 300, (150, 151, 290), 0, 0), (900, 200, (1, 40, 500, 1050), 120, 3),
                                          (900, 200, (40, 500, 1050), 120, 3)):
        n = ctx + rows
        cache = Cache([n], q8, 5).fill([n], 6)
        poison(cache, 0, at, value)
        q, gt = some(rows, 1, kind), some(rows, 2, kind, 1.0)
        for r0 in (0, rows - 3):  # as one run, and its last rows alone (split along the positions)
            out = ops.gqa_prefill(q[r0:], gt[r0:], ints(0, rows - r0), ints(n), rows - r0, n, cache.ptrs(), cache.k_off, cache.v_off,
                                  window=window, sink=sink, kv_q8=q8)
            k, v = cache.sequence(0, n)
            clean, hit = [], []
            for r in sorted({r0, r0 + 1, r0 + 2, *range(r0, rows, 7), *(p - ctx + d for p in at for d in (-1, 0, 1) if r0 <= p - ctx + d < rows)}):
                length = ctx + r + 1
                few = min(sink, length)
                seen = [p for p in at if p < length and (window <= 0 or few + window >= length or p < few or p >= length - window)]
                (hit if seen else clean).append(r)
                if not seen:
                    o, a, s = attend(q[r], gt[r], k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0), length, window, sink)
                    check_rows(out, [(r - r0, o, a, s, length)], half, q8)
            assert clean or r0 or 1 in at  # (position 1 is a sink: every row attends it)
            for r in hit:
                assert not torch.isfinite(out[r - r0]).all()
    assert _lib.lib().qw35_cuda_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("half,q8", [(False, False), (True, False), (False, True)])
def test_shared_keeps_what_a_sequence_does_not_attend_from_it(half, q8):
    """A sequence that ends inside the prefix, and windows that leave some of it out, beside others that see it all."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    lens, shared = [700, 130, 900, 333], 640
    for at, window in (((400, 639), 0), ((10, 200), 300)):
        cache = Cache([900] * 4, q8, 5).fill([900] * 4, 6)
        poison(cache, 0, at, float("nan"))
        cache.ids[1:, :shared // CH] = cache.ids[0, :shared // CH]
        rows = cache.rows()
        for j in range(1, 4):
            rows[int(cache.ids[j, 2])][:, :, :128] = rows[int(cache.ids[0, 2])][:, :, :128]
        q, gt = some(4, 1, kind), some(4, 2, kind, 1.0)
        out = ops.gqa_decode_shared(q, gt, ints(*lens), ints(0, 4), ints(shared), shared, 260, cache.ptrs(), cache.k_off, cache.v_off,
                                    window=window, kv_q8=q8)
        for i, length in enumerate(lens):
            seen = [p for p in at if p < length and (window <= 0 or p >= length - window)]
            if seen:
                assert not torch.isfinite(out[i]).all()
            else:
                k, v = cache.sequence(i, length)
                check_rows(out, [(i, *attend(q[i], gt[i], k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0), length, window), length)], half, q8)


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("ctx,rows", [(4000, 5), (300, 200), (9000, 70)])
def test_prefill_nan_queries_and_keys_come_out(half, q8, ctx, rows):
    """A NaN in a head's q makes that head's row NaN and no other; keys that are NaN over whole parts make every row NaN."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    n = ctx + rows
    cache = Cache([n], q8, 5).fill([n], 6)
    q, gt = some(rows, 1, kind), some(rows, 2, kind, 1.0)
    r, h = rows // 2, 5
    args = (gt, ints(0, rows), ints(n), rows, n, cache.ptrs(), cache.k_off, cache.v_off)
    q[r, h, 77] = float("nan")
    out = ops.gqa_prefill(q, *args, kv_q8=q8).view(rows, H, D)
    bad = out.isnan()
    assert bool(bad[r, h].all()) and int(bad.sum()) == D
    q[r, h, 77] = 0.5
    part = cache.rows()[int(cache.ids[0, 0]), 0]
    if q8:
        part[..., :2] = torch.tensor([0, 0x7e], dtype=torch.uint8, device="cuda")
    else:
        part.fill_(float("nan"))
    assert bool(ops.gqa_prefill(q, *args, kv_q8=q8).isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("half,q8", [(False, False), (True, False), (False, True)])
def test_shared_nan_queries_come_out(half, q8):
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    cache = Cache([900] * 4, q8, 5).fill([900] * 4, 6)
    cache.ids[1:, :2] = cache.ids[0, :2]
    q, gt = some(4, 1, kind), some(4, 2, kind, 1.0)
    q[2, 9, 0] = float("nan")
    out = ops.gqa_decode_shared(q, gt, ints(900, 600, 700, 513), ints(0, 4), ints(512), 512, 388, cache.ptrs(), cache.k_off, cache.v_off,
                                kv_q8=q8).view(4, H, D)
    assert bool(out[2, 9].isnan().all()) and int(out.isnan().sum()) == D


# ---- shared prefixes -----------------------------------------------------------------------

def shared_case(groups, half, q8, window=0, sink=0, gate=True, seed=0, max_own=None):
    """groups: [(shared length, [own lengths])]; an own length may be negative (the sequence ends inside the prefix)."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    lens = [max(0, s + o) for s, own in groups for o in own]
    pre = [s for s, own in groups for _ in own]
    cache = Cache([max(n, s) for n, s in zip(lens, pre)], q8, seed + 1)
    cache.fill([max(n, s) for n, s in zip(lens, pre)], seed + 2)
    at, off = 0, [0]
    rows = cache.rows()
    for s, own in groups:  # the prefix's whole chunks are one, its last part a copy
        for j in range(at + 1, at + len(own)):
            cache.ids[j, :s // CH] = cache.ids[at, :s // CH]
            if s % CH:
                rows[int(cache.ids[j, s // CH])][:, :, :s % CH] = rows[int(cache.ids[at, s // CH])][:, :, :s % CH]
        at += len(own)
        off.append(at)
    n = len(lens)
    q, gt = some(n, seed + 3, kind), some(n, seed + 4, kind, 1.0)
    own_most = max(1, max(a - b for a, b in zip(lens, pre))) if max_own is None else max_own
    args = (q, gt if gate else None, ints(*lens), ints(*off), ints(*[s for s, _ in groups]), max(s for s, _ in groups), own_most,
            cache.ptrs(), cache.k_off, cache.v_off)
    out = ops.gqa_decode_shared(*args, window=window, sink=sink, kv_q8=q8)
    ref = []
    for i, length in enumerate(lens):
        k, v = cache.sequence(i, length)
        ref.append((i, *attend(q[i], gt[i] if gate else None, k, v, length, window, sink), length))
    check_rows(out, ref, half, q8)
    assert _lib.lib().qw35_cuda_device_error() == 0
    return cache, args, out, ref


GROUPS = [
    [(700, [3, 40])],
    [(256, [1] * 33)],
    [(1, [0])],
    [(0, [17, 300])],
    [(513, [0, 1, 255, 256, 600]), (0, [5]), (4096, [9]), (129, list(range(1, 70)))],
    [(1000, [-999, -1000, -500, -1, 20])],
    [(20000, [30, 1])],
]


@pytest.mark.gpu
@pytest.mark.parametrize("groups", GROUPS)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q8", [False, True])
def test_shared_matches_the_formula(groups, half, q8):
    shared_case(groups, half, q8)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sink", CUTS)
@pytest.mark.parametrize("half,q8", [(False, False), (True, True)])
def test_shared_window_and_sink(window, sink, half, q8):
    shared_case([(500, [1, 30, 190, 260]), (260, [3, -200])], half, q8, window, sink)


@pytest.mark.gpu
def test_shared_without_gate_and_with_generous_bounds():
    shared_case([(300, [4, 5])], False, False, gate=False, max_own=512)


@pytest.mark.gpu
def test_shared_agrees_with_gqa_decode():
    from qwowl35_b200 import ops
    cache, args, out, ref = shared_case([(777, [12, 90, 1]), (2048, [400])], False, False, seed=20)
    q, gate, seq_len = args[:3]
    plain = ops.gqa_decode(q, gate, seq_len, int(seq_len.max()), args[7], cache.k_off, cache.v_off)
    check_rows(plain, ref, False, False)
    check_rows(out, ref, False, False)


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
def test_shared_leaves_sequences_of_no_group(half):
    """Sequences before the first group, between groups and behind the last keep what out held."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    cache = Cache([300] * 8, False, 2).fill([300] * 8, 3)
    q, gt = some(8, 1, kind), some(8, 2, kind)
    out = torch.full((8, H * D), 5.0, dtype=kind, device="cuda")
    ops.gqa_decode_shared(q, gt, ints(*[280] * 8), ints(1, 1, 3), ints(64, 128), 128, 216, cache.ptrs(), cache.k_off, cache.v_off,
                          out=out)
    # (groups [1, 1) and [1, 3); the second reads its 128 shared positions through table row 1)
    assert bool((out[0] == 5).all()) and bool((out[3:] == 5).all())
    ref = []
    for i in (1, 2):
        (k, v), (k1, v1) = cache.sequence(i, 280), cache.sequence(1, 280)
        k, v = torch.cat([k1[:, :128], k[:, 128:]], 1), torch.cat([v1[:, :128], v[:, 128:]], 1)
        ref.append((i, *attend(q[i], gt[i], k, v, 280), 280))
    check_rows(out, ref, half, False)


@pytest.mark.gpu
def test_bounds_below_the_lengths_still_attend_everything():
    """max_len, max_shared and max_own size the split, not the work."""
    from qwowl35_b200 import ops
    cache = Cache([3000, 3000], False, 2).fill([3000, 3000], 3)
    q, gt = some(20, 1, torch.float32), some(20, 2, torch.float32)
    out = ops.gqa_prefill(q, gt, ints(0, 20), ints(3000), 20, 200, cache.ptrs()[:1].contiguous(), cache.k_off, cache.v_off)
    k, v = cache.sequence(0, 3000)
    check_rows(out, [(r, *attend(q[r], gt[r], k, v, 2981 + r), 2981 + r) for r in (0, 7, 19)], False, False)
    cache.ids[1, :8] = cache.ids[0, :8]
    out = ops.gqa_decode_shared(q[:2], gt[:2], ints(3000, 2900), ints(0, 2), ints(2048), 100, 50, cache.ptrs(), cache.k_off,
                                cache.v_off)
    ref = []
    for i, n in enumerate((3000, 2900)):
        k, v = cache.sequence(i, n)
        ref.append((i, *attend(q[i], gt[i], k, v, n), n))
    check_rows(out, ref, False, False)


@pytest.mark.gpu
@pytest.mark.parametrize("off,lens", [((-64, 32), (500,)), ((0, 90), (500,)), ((20, 10, 40), (500, 500)), ((0, 40), (-7,)), ((0, 0), (9,))])
def test_offsets_that_make_no_sense_are_skipped(off, lens):
    """Runs outside the rows, backwards or empty, and lengths below zero: nothing is read or written out of range."""
    from qwowl35_b200 import ops
    cache = Cache([512] * len(lens), False, 2).fill([512] * len(lens), 3)
    q = some(40, 1, torch.float16)
    for gate in (None, q):
        out = ops.gqa_prefill(q, gate, ints(*off), ints(*lens), 40, 512, cache.ptrs(), cache.k_off, cache.v_off)
    tables = cache.ptrs()[[0] * 40].contiguous()
    ops.gqa_decode_shared(q, q, ints(*[500] * 40), ints(*off), ints(*lens), 500, 100, tables, cache.k_off, cache.v_off, out=out)
    torch.cuda.synchronize()
    assert _lib.lib().qw35_cuda_device_error() == 0


@pytest.mark.gpu
def test_more_runs_than_a_warp_and_one_row_each():
    """70 single-token runs and 45 groups: the searches go beyond one warp's width."""
    from qwowl35_b200 import ops
    lens = [1 + (i * 29) % 300 for i in range(70)]
    cache = Cache(lens, True, 2).fill(lens, 3)
    q, gt = some(70, 1, torch.float32), some(70, 2, torch.float32)
    table = cache.ptrs()
    out = ops.gqa_prefill(q, gt, ints(*range(71)), ints(*lens), 1, max(lens), table, cache.k_off, cache.v_off, kv_q8=True)
    ref = []
    for i, n in enumerate(lens):
        k, v = cache.sequence(i, n)
        ref.append((i, *attend(q[i], gt[i], k, v, n), n))
    check_rows(out, ref, False, True)
    out = ops.gqa_decode_shared(q, gt, ints(*lens), ints(*range(71)), ints(*[n // 2 for n in lens]), 150, 151, table, cache.k_off,
                                cache.v_off, kv_q8=True)
    check_rows(out, ref, False, True)


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
def test_out_may_be_the_gate(half):
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    cache = Cache([700], False, 2).fill([700], 3)
    for rows in (5, 700):
        q, gt = some(rows, 1, kind), some(rows, 2, kind)
        args = (ints(0, rows), ints(700), rows, 700, cache.ptrs(), cache.k_off, cache.v_off)
        want = ops.gqa_prefill(q, gt, *args)
        got = ops.gqa_prefill(q, gt, *args, out=gt)
        assert torch.equal(got.view(want.shape), want)


# ---- together, captured, on several streams ---------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("half,q8", [(False, False), (True, False), (False, True)])
def test_append_prefill_fork_and_shared_decode_together(half, q8):
    """Two prompts enter the cache and attend; three continuations of the first then decode over its prefix."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    runs = [(0, 300), (0, 45)]
    cache = Cache([600, 300, 600, 600], q8, 31)
    cache.ids[2, 0] = cache.ids[3, 0] = cache.ids[0, 0]  # the whole chunk of the prompt is shared
    g = torch.Generator("cuda").manual_seed(8)
    qw, kw = (1 + 0.2 * torch.randn(256, device="cuda", generator=g) for _ in range(2))
    qkv = torch.randn(345, 10240, device="cuda", generator=g)
    pos = torch.cat([torch.arange(300), torch.arange(45)]).int().cuda()
    seq = torch.cat([torch.zeros(300), torch.ones(45)]).int().cuda()
    table, f = cache.ptrs(), FREQ.cuda()
    q, gate = ops.attn_append(qkv, qw, kw, f, pos[None].repeat(3, 1), (11, 11, 10), seq, pos, table, cache.k_off, cache.v_off,
                              dtype=kind, kv_q8=q8)
    out = ops.gqa_prefill(q, gate, ints(0, 300, 345), ints(300, 45), 300, 300, table, cache.k_off, cache.v_off, kv_q8=q8)
    rows = []
    for i, (_, r) in enumerate(runs):
        k, v = cache.sequence(i, r)
        rows += [(300 * i + t, *attend(q[300 * i + t], gate[300 * i + t], k, v, t + 1), t + 1) for t in (0, 1, 31, 32, 44, r - 1)]
    check_rows(out, rows, half, q8)
    # fork: sequences 2 and 3 continue sequence 0 with their own copy of its last chunk
    raw = cache.raw
    for j in (2, 3):
        raw[int(cache.ids[j, 1])] = raw[int(cache.ids[0, 1])]
    order = [0, 2, 3]
    tables = table[order].contiguous()
    step = torch.randn(3, 10240, device="cuda", generator=g)
    at = ints(300, 300, 300)
    q, gate = ops.attn_append(step, qw, kw, f, at[None].contiguous(), (32,), ints(0, 1, 2), at, tables, cache.k_off, cache.v_off,
                              dtype=kind, kv_q8=q8)
    out = ops.gqa_decode_shared(q, gate, at + 1, ints(0, 3), ints(300), 300, 1, tables, cache.k_off, cache.v_off, kv_q8=q8)
    rows = []
    for r, i in enumerate(order):
        k, v = cache.sequence(i, 301)
        rows.append((r, *attend(q[r], gate[r], k, v, 301), 301))
    check_rows(out, rows, half, q8)


@pytest.mark.gpu
def test_captured_calls_replay_over_other_lengths():
    """One graph of both attentions, captured with upper bounds, replayed after the lengths on the device changed."""
    from qwowl35_b200 import ops
    cache = Cache([1500] * 4, False, 2).fill([1500] * 4, 3)
    cache.ids[3, :2] = cache.ids[2, :2]
    table = cache.ptrs()
    q, gt = some(40, 1, torch.float32), some(40, 2, torch.float32)
    off, lens = ints(0, 10, 40), ints(700, 800)
    soff, slen, shared = ints(0, 2), ints(600, 520), ints(512)
    out1, out2 = torch.zeros(40, 4096, device="cuda"), torch.zeros(2, 4096, device="cuda")
    ws1, ws2 = ops.gqa_prefill_workspace(40, 2, 40, 1500), ops.gqa_decode_shared_workspace(2, 1, 512, 900)

    def both():
        ops.gqa_prefill(q, gt, off, lens, 40, 1500, table, cache.k_off, cache.v_off, ws=ws1, out=out1)
        ops.gqa_decode_shared(q[:2], gt[:2], slen, soff, shared, 512, 900, table[2:], cache.k_off, cache.v_off, ws=ws2, out=out2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for cut, n0, n1, s0, s1, sh in ((10, 700, 800, 600, 520, 512), (37, 1500, 3, 1400, 1, 500), (1, 20, 1499, 0, 512, 0)):
        off.copy_(ints(0, cut, 40))
        lens.copy_(ints(n0, n1))
        slen.copy_(ints(s0, s1))
        shared.copy_(ints(sh))
        graph.replay()
        rows = []
        for i, (a, b, n) in enumerate(((0, cut, n0), (cut, 40, n1))):
            k, v = cache.sequence(i, n)
            rows += [(r, *attend(q[r], gt[r], k, v, n - (b - r) + 1), n - (b - r) + 1) for r in range(a, b, 3)]
        check_rows(out1, rows, False, False)
        rows = []
        for i, n in enumerate((s0, s1)):
            k, v = cache.sequence(2 + i, n)
            rows.append((i, *attend(q[i], gt[i], k, v, n), n))
        check_rows(out2, rows, False, False)


@pytest.mark.gpu
def test_two_streams_with_their_own_workspaces():
    from qwowl35_b200 import ops
    cache = Cache([3000, 2500], False, 2).fill([3000, 2500], 3)
    q, gt = some(128, 1, torch.float16), some(128, 2, torch.float16)
    want = [ops.gqa_prefill(q[64 * i:64 * i + 64], gt[64 * i:64 * i + 64], ints(0, 64), ints(n), 64, n, cache.ptrs()[i:i + 1].contiguous(),
                            cache.k_off, cache.v_off) for i, n in enumerate((3000, 2500))]
    tables = [cache.ptrs()[i:i + 1].contiguous() for i in range(2)]
    off, lens = ints(0, 64), [ints(3000), ints(2500)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, n in enumerate((3000, 2500)):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.gqa_prefill(q[64 * i:64 * i + 64], gt[64 * i:64 * i + 64], off, lens[i], 64, n, tables[i],
                                              cache.k_off, cache.v_off))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, want[i])  # no atomics: the same bits every time


# ---- refusals (no GPU work) -----------------------------------------------------------------

def _append_args(**over):
    a = dict(n=4, qkv=16, stride=10240, qw=16, kw=16, freq=16, pos=16, axes=3, sec=(11, 11, 10), inter=1, seq=16, at=16, n_seq=2,
             table=16, chunks=4, k=0, v=1 << 19, kv=0, q=16, gate=16, dtype=0)
    a.update(over)
    sec = (C.c_int32 * len(a["sec"]))(*a["sec"]) if a["sec"] is not None else None
    return (a["n"], a["qkv"], a["stride"], a["qw"], a["kw"], a["freq"], a["pos"], a["axes"], sec, a["inter"], a["seq"], a["at"],
            a["n_seq"], a["table"], a["chunks"], a["k"], a["v"], a["kv"], a["q"], a["gate"], a["dtype"], 1e-6, None)


@pytest.mark.parametrize("over,message", [
    (dict(qkv=None), "invalid append"), (dict(table=None), "invalid append"), (dict(seq=None), "invalid append"),
    (dict(sec=None), "invalid append"), (dict(stride=10239), "invalid append"), (dict(n_seq=0), "invalid append"),
    (dict(chunks=0), "invalid append"), (dict(k=8), "invalid append"), (dict(kv=2), "invalid append"), (dict(dtype=2), "invalid append"),
    (dict(q=20), "invalid append"), (dict(axes=0), "rotary sections"), (dict(axes=4, sec=(8, 8, 8, 8)), "rotary sections"),
    (dict(sec=(11, 11, 11)), "rotary sections"), (dict(sec=(33, -1, 0)), "rotary sections"),
    (dict(sec=(1 << 31 - 1, 1 << 31 - 1, 34)), "rotary sections"), (dict(axes=2, sec=(20, 12)), "rotary sections"),
])
def test_append_refuses(over, message):
    with pytest.raises(_lib.Qw35Error, match=message):
        _lib.call("qw35_cuda_attn_append", *_append_args(**over))


def test_calls_without_rows_do_nothing():
    _lib.call("qw35_cuda_attn_append", *_append_args(n=0))
    _lib.call("qw35_cuda_gqa_prefill", *_prefill_args(n=0))
    _lib.call("qw35_cuda_gqa_decode_shared", *_shared_args(n=0))


@pytest.mark.parametrize("sizes", [(0, 0, 0, 0), (0, 1, 1, 1), (4, 0, 1, 5), (4, 1, 0, 5), (4, 1, 1, 0), (4, 1, 5, 5),
                                   (4, 1, 2 ** 32 - 1, 5), (4, 1, 2 ** 31, 5)])
def test_prefill_sizes_without_work_need_no_workspace(sizes):
    assert _lib.lib().qw35_cuda_gqa_prefill_workspace_bytes(*sizes) == 0


@pytest.mark.parametrize("sizes", [(0, 0, 0, 0), (0, 1, 1, 1), (4, 0, 1, 5), (4, 1, 0, 0), (65536, 1, 1, 5)])
def test_shared_sizes_without_work_need_no_workspace(sizes):
    assert _lib.lib().qw35_cuda_gqa_decode_shared_workspace_bytes(*sizes) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
def test_wrappers_take_batches_without_rows(half):
    from qwowl35_b200 import ops
    cache = Cache([40], False, 5).fill([40], 6)
    kind = torch.float16 if half else torch.float32
    q, one = some(0, 1, kind), some(1, 1, kind)
    at = (cache.ptrs(), cache.k_off, cache.v_off)
    assert ops.gqa_prefill(q, q, ints(0, 0), ints(40), 0, 40, *at).shape == (0, H * D)
    assert ops.gqa_prefill(q, None, ints(0), ints(), 0, 0, *at).shape == (0, H * D)
    assert ops.gqa_decode_shared(q, q, ints(), ints(0, 0), ints(8), 8, 32, *at).shape == (0, H * D)
    out = torch.full((1, H * D), 5.0, dtype=kind, device="cuda")  # a row of no group
    ops.gqa_decode_shared(one, one, ints(40), ints(0), ints(), 0, 0, *at, out=out)
    ops.gqa_prefill(one, one, ints(0), ints(), 0, 0, *at, out=out)
    assert bool((out == 5).all()) and _lib.lib().qw35_cuda_device_error() == 0


def _prefill_args(**over):
    a = dict(n=4, q=16, gate=None, dtype=0, runs=1, off=16, len=16, max_run=4, max_len=100, table=16, chunks=1, k=0, v=1 << 19, kv=0,
             window=0, sink=0, out=16, ws=16, bytes=1 << 40)
    a.update(over)
    return tuple(a.values()) + (None,)


def _shared_args(**over):
    a = dict(n=4, q=16, gate=None, dtype=0, len=16, groups=1, off=16, shared=16, max_shared=100, max_own=100, table=16, chunks=1,
             k=0, v=1 << 19, kv=0, window=0, sink=0, out=16, ws=16, bytes=1 << 40)
    a.update(over)
    return tuple(a.values()) + (None,)


@pytest.mark.parametrize("over", [dict(q=None), dict(q=8), dict(gate=8), dict(out=None), dict(off=None), dict(len=None), dict(dtype=2),
                                  dict(table=None), dict(chunks=0), dict(max_len=257), dict(k=8), dict(v=8), dict(kv=2), dict(ws=None),
                                  dict(n=1 << 25)])
def test_prefill_refuses(over):
    with pytest.raises(_lib.Qw35Error, match="invalid prefill"):
        _lib.call("qw35_cuda_gqa_prefill", *_prefill_args(**over))


@pytest.mark.parametrize("over", [dict(max_run=0), dict(max_run=5), dict(max_len=0)])
def test_prefill_refuses_bounds(over):
    with pytest.raises(_lib.Qw35Error, match="invalid prefill"):
        _lib.call("qw35_cuda_gqa_prefill", *_prefill_args(**over))


@pytest.mark.parametrize("over", [dict(q=None), dict(q=8), dict(gate=8), dict(out=None), dict(off=None), dict(len=None), dict(dtype=2),
                                  dict(shared=None), dict(table=None), dict(chunks=0), dict(max_own=257), dict(max_shared=257), dict(k=8), dict(kv=2),
                                  dict(max_shared=0, max_own=0), dict(n=65536), dict(max_shared=1 << 30, max_own=1 << 30)])
def test_shared_refuses(over):
    with pytest.raises(_lib.Qw35Error, match="invalid shared-prefix"):
        _lib.call("qw35_cuda_gqa_decode_shared", *_shared_args(**over))


def test_small_workspaces_are_refused():
    need = _lib.lib().qw35_cuda_gqa_prefill_workspace_bytes(4, 1, 4, 100)
    assert need > 0
    with pytest.raises(_lib.Qw35Error, match="workspace too small"):
        _lib.call("qw35_cuda_gqa_prefill", *_prefill_args(bytes=need - 1))
    need = _lib.lib().qw35_cuda_gqa_decode_shared_workspace_bytes(4, 1, 100, 100)
    assert need > 0
    with pytest.raises(_lib.Qw35Error, match="workspace too small"):
        _lib.call("qw35_cuda_gqa_decode_shared", *_shared_args(bytes=need - 1))


@pytest.mark.gpu
def test_wrappers_refuse_tensors_of_another_kind():
    from qwowl35_b200 import ops
    cache = Cache([40], False, 5).fill([40], 6)
    q = some(4, 1, torch.float32)
    good = (q, q, ints(0, 4), ints(40), 4, 40, cache.ptrs(), cache.k_off, cache.v_off)
    ops.gqa_prefill(*good)
    for at, bad in ((0, q.double()), (1, q.half()), (2, ints(0, 4).long()), (2, ints(0, 4, 4)), (6, cache.ptrs().float())):
        with pytest.raises(TypeError):
            ops.gqa_prefill(*good[:at], bad, *good[at + 1:])
    with pytest.raises(ValueError):
        ops.gqa_prefill(*good[:2], ints(0, 2, 4), ints(40, 40), *good[4:])


@pytest.mark.gpu
def test_wrappers_refuse_workspaces_elsewhere():
    from qwowl35_b200 import ops
    cache = Cache([40], False, 5).fill([40], 6)
    q = some(4, 1, torch.float32)
    at = (cache.ptrs(), cache.k_off, cache.v_off)
    n = max(ops.gqa_prefill_workspace(4, 1, 4, 40).numel(), ops.gqa_decode_shared_workspace(1, 1, 8, 32).numel())
    bad = [torch.empty(n, dtype=torch.uint8), torch.empty(n, dtype=torch.float32, device="cuda"),
           torch.empty(2 * n, dtype=torch.uint8, device="cuda")[::2]]
    if torch.cuda.device_count() > 1:
        bad.append(torch.empty(n, dtype=torch.uint8, device="cuda:1"))
    for ws in bad:
        with pytest.raises(TypeError, match="workspace"):
            ops.gqa_prefill(q, q, ints(0, 4), ints(40), 4, 40, *at, ws=ws)
        with pytest.raises(TypeError, match="workspace"):
            ops.gqa_decode_shared(q[:1], q[:1], ints(40), ints(0, 1), ints(8), 8, 32, *at, ws=ws)


@pytest.mark.gpu
def test_append_refuses_rows_too_far_apart():
    """The C call takes the stride in 32 bits: 2^32 + 10240 must not become 10240."""
    from qwowl35_b200 import ops
    cache = Cache([40], False, 5)
    qkv = torch.empty(2 ** 32 + 2 * 10240, device="cuda").as_strided((2, 10240), (2 ** 32 + 10240, 1))
    w = torch.ones(256, device="cuda")
    with pytest.raises(TypeError, match="apart"):
        ops.attn_append(qkv, w, w, FREQ.cuda(), ints(0, 1)[None], (32,), ints(0, 0), ints(0, 1), cache.ptrs(), cache.k_off, cache.v_off)


def test_wrappers_refuse_host_tensors():
    from qwowl35_b200 import ops
    t, i = torch.zeros(1, 10240), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError, match="device tensor"):
        ops.attn_append(t, t, t, t, i, (32,), i, i, i, 0, 0)
    with pytest.raises(TypeError, match="device tensor"):
        ops.gqa_prefill(t, None, i, i, 1, 1, i, 0, 0)
    with pytest.raises(TypeError, match="device tensor"):
        ops.gqa_decode_shared(t, None, i, i, i, 1, 1, i, 0, 0)


@pytest.mark.gpu
def test_tensors_on_another_device_than_the_current_one():
    """The calls run on their tensors' device and leave the current one as it was."""
    from qwowl35_b200 import ops
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    cache = Cache([700], False, 2).fill([700], 3)
    q, gt = some(5, 1, torch.float16), some(5, 2, torch.float16)
    want = ops.gqa_prefill(q, gt, ints(0, 5), ints(700), 5, 700, cache.ptrs(), cache.k_off, cache.v_off)
    raw = cache.raw.to("cuda:1")
    table = torch.where(cache.ids >= 0, raw.data_ptr() + cache.ids * 4 * cache.plane, 0).to("cuda:1")
    got = ops.gqa_prefill(q.to("cuda:1"), gt.to("cuda:1"), ints(0, 5).to("cuda:1"), ints(700).to("cuda:1"), 5, 700, table, cache.k_off,
                          cache.v_off)
    assert torch.cuda.current_device() == 0 and torch.equal(got.cpu(), want.cpu())
    with pytest.raises(TypeError):
        ops.gqa_prefill(q, gt.to("cuda:1"), ints(0, 5), ints(700), 5, 700, cache.ptrs(), cache.k_off, cache.v_off)


# ---- gates, and values that are not finite --------------------------------------------------------------

GATES = [float("nan"), float("inf"), float("-inf"), 0.0, -0.5, 3.0, -5.0, 12.0, -12.0, 20.0, -20.0, 60.0, -60.0, -80.0, -86.0, 86.0, -88.0,
         88.0, -104.0, 104.0, -300.0, 300.0, -60000.0, 60000.0]


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shared", [False, True])
def test_gates_of_every_size(half, shared):
    """One attended position: the output is its value times the gate's sigmoid, to 2^-20 (an exponential and a quotient of
    2^-22 each, four roundings of 2^-24) and nothing below the smallest normal number; NaN gates come out as NaN."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    n = 40
    cache = Cache([1] * n, False, 5).fill([1] * n, 6)
    q = some(n, 1, kind)
    g = torch.Generator("cuda").manual_seed(3)
    gate = (torch.rand(n, H, D, device="cuda", generator=g) * 220 - 110).to(kind)
    gate[::2] = torch.tensor(GATES, device="cuda").to(kind).repeat(H * D)[:H * D].view(H, D)
    at = (cache.ptrs(), cache.k_off, cache.v_off)
    if shared:  # (parts are joined)
        out = ops.gqa_decode_shared(q, gate, ints(*[1] * n), ints(*range(n + 1)), ints(*[i % 2 for i in range(n)]), 1, 1, *at)
    else:
        out = ops.gqa_prefill(q, gate, ints(*range(n + 1)), ints(*[1] * n), 1, 1, *at)
    v = torch.stack([cache.sequence(i, 1)[1][:, 0] for i in range(n)]).repeat_interleave(H // KV, 1)
    want, got = v * torch.sigmoid(gate.double()), out.view(n, H, D).double()
    nan = gate.isnan()
    assert bool(got[nan].isnan().all()) and bool(torch.isfinite(got[~nan]).all())
    tol = (2.0 ** -20 + (2.0 ** -11 if half else 0)) * want.abs() + 2.0 ** -126 * v.abs() + (2.0 ** -25 if half else 2.0 ** -149)
    err = ((got - want).abs() / tol)[~nan]
    assert float(err.max()) <= 1.0, float(err.max())
    assert bool((got[gate == float("-inf")] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("half,q8", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("ctx,rows", [(300, 20), (4000, 5), (9000, 70)])
def test_prefill_nan_and_infinite_gates(half, q8, ctx, rows):
    """In one piece, joined, and on CTA pairs: a gate's NaN stays at its own value."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    n = ctx + rows
    cache = Cache([n], q8, 5).fill([n], 6)
    q, gt = some(rows, 1, kind), some(rows, 2, kind, 1.0)
    args = (ints(0, rows), ints(n), rows, n, cache.ptrs(), cache.k_off, cache.v_off)
    want = ops.gqa_prefill(q, gt, *args, kv_q8=q8).view(rows, H, D)
    bare = ops.gqa_prefill(q, None, *args, kv_q8=q8).view(rows, H, D)
    gt[1::3, 3, 7::11] = float("nan")
    gt[::2, 9, 5::13] = float("inf")
    gt[::2, 15, 2::3] = -float("inf")
    got = ops.gqa_prefill(q, gt, *args, kv_q8=q8).view(rows, H, D)
    assert torch.equal(got.isnan(), gt.isnan())
    assert torch.equal(got[gt == float("inf")], bare[gt == float("inf")]) and bool((got[gt == -float("inf")] == 0).all())
    same = torch.isfinite(gt)
    assert torch.equal(got[same], want[same])


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("ctx,rows,top,at", [(4095, 1, 4000, 700), (4095, 1, 700, 4000), (300, 40, 0, 320), (9000, 70, 8999, 100)])
def test_prefill_attended_nans_come_out_whatever_their_weight(half, value, ctx, rows, top, at):
    """One key outweighs the rest by e^200 and more; a value that is not finite still reaches the rows that attend it."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    n = ctx + rows
    cache = Cache([n], False, 5).fill([n], 6)
    q, gt = some(rows, 1, kind), some(rows, 2, kind, 1.0)
    q[:] = q[:1, :1]
    planes = cache.rows()
    planes[int(cache.ids[0, top // CH]), 0, :, top % CH] = (8 * q[0, 0]).half()
    planes[int(cache.ids[0, at // CH]), 1, :, at % CH, 33] = value
    out = ops.gqa_prefill(q, gt, ints(0, rows), ints(n), rows, n, cache.ptrs(), cache.k_off, cache.v_off).view(rows, H, D)
    sees = torch.tensor([ctx + r >= at for r in range(rows)], device="cuda")
    assert not bool(torch.isfinite(out[sees][..., 33]).any())
    out[..., 33][sees] = 0
    assert bool(torch.isfinite(out).all())


@pytest.mark.gpu
def test_prefill_nan_values_of_infinitely_low_scores_come_out():
    """A part of which every score is -infinity (f16: 0 times an infinity does not come up) still has its values."""
    from qwowl35_b200 import ops
    n = 4096
    cache = Cache([n], False, 5).fill([n], 6)
    q = some(1, 1, torch.float16)
    q[..., 0] = 1.0
    planes = cache.rows()
    chunk = int(cache.ids[0, 2])
    planes[chunk, 0, :, :128, 0] = -float("inf")
    args = (None, ints(0, 1), ints(n), 1, n, cache.ptrs(), cache.k_off, cache.v_off)
    assert bool(torch.isfinite(ops.gqa_prefill(q, *args)).all())
    planes[chunk, 1, :, 77, 33] = float("nan")
    bad = torch.zeros(H, D, dtype=torch.bool, device="cuda")
    bad[:, 33] = True
    assert torch.equal(ops.gqa_prefill(q, *args).view(H, D).isnan(), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("half,q8", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("seqs,n,rows", [(1, 1100, 5), (1, 1100, 1100), (40, 700, 3)])  # joined; pairs; single CTAs
def test_prefill_missing_chunks_are_zeros(half, q8, seqs, n, rows):
    """Also in units that a value that is not finite sends to the CUDA cores."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    cache = Cache([n] * seqs, q8, 5).fill([n] * seqs, 6)
    cache.rows()[cache.ids[:, 1].cuda()] = 0
    table = cache.ptrs()
    table[:, 1] = 0
    q, gt = some(rows * seqs, 1, kind), some(rows * seqs, 2, kind, 1.0)
    off = ints(*range(0, rows * seqs + 1, rows))
    kv = [cache.sequence(i, n - 1) for i in range(seqs)]
    for poisoned in (False, True):
        if poisoned:
            for i in range(seqs):
                poison(cache, i, (n - 1,), float("nan"), planes=(1,))
        out = ops.gqa_prefill(q, gt, off, ints(*[n] * seqs), rows, n, table, cache.k_off, cache.v_off, kv_q8=q8)
        ref = [(i * rows + r, *attend(q[i * rows + r], gt[i * rows + r], *kv[i], n - rows + r + 1), n - rows + r + 1)
               for i in range(0, seqs, 13) for r in sorted({0, 1, rows // 2, rows - 2})]
        check_rows(out, ref, half, q8)
        assert not poisoned or not bool(torch.isfinite(out[rows - 1::rows]).all(1).any())


# ---- sizes at the limits --------------------------------------------------------------------------------

@pytest.mark.parametrize("sizes", [(61731, 51426, 484746496, 505329920), (65535, 1, 1 << 29, 1 << 29), (65535, 65535, 1 << 29, 0),
                                   (65535, 65535, 1 << 29, 1 << 29)])
def test_shared_workspace_of_the_largest_sizes(sizes):
    """More work than 32 bits hold, a share at a time: a part for the prefix and one for the tail.  (In a process of its own: a
    division by zero would end it.)"""
    code = "from qwowl35_b200 import _lib; print(_lib.lib().qw35_cuda_gqa_decode_shared_workspace_bytes(*%r))" % (sizes,)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0, r.returncode
    assert int(r.stdout) == sizes[0] * 16 * 2 * (8 + 1024)


@pytest.mark.gpu
@pytest.mark.parametrize("half,q8", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("n", [5, 1000])
def test_append_nans_come_out(half, q8, n):
    """A NaN or an infinity of a token's q, gate, k or v is one in what is written of it (q8_0: in its block), and nowhere else."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    g = torch.Generator("cuda").manual_seed(n)
    qkv = torch.randn(n, 10240, device="cuda", generator=g)
    w, pos = torch.ones(256, device="cuda"), torch.arange(n, device="cuda").int()
    nan, inf = float("nan"), float("inf")
    qkv[1, 3 * 512 + 100], qkv[2, 5 * 512 + 256 + 7] = nan, nan                          # q head 3, gate 5
    qkv[1, 8192 + 256 + 200], qkv[3, 8192 + 1024 + 512 + 77] = nan, nan                  # k head 1, v head 2
    qkv[2, 8192 + 768 + 200], qkv[4, 8192 + 1024 + 30], qkv[4, 8192 + 1024 + 255] = inf, inf, -inf  # k head 3, v head 0
    cache = Cache([n], q8, 3).fill([n], 4)
    q, gate = ops.attn_append(qkv, w, w, FREQ.cuda(), pos[None].contiguous(), (32,), torch.zeros_like(pos), pos, cache.ptrs(), cache.k_off,
                              cache.v_off, dtype=kind, kv_q8=q8)
    bad = torch.zeros(n, H, D, dtype=torch.bool, device="cuda")
    bad[1, 3] = True
    assert torch.equal(~torch.isfinite(q), bad)
    bad[:] = False
    bad[2, 5, 7] = True
    assert torch.equal(~torch.isfinite(gate), bad)
    k, v = cache.sequence(0, n)
    bad = torch.zeros(2, KV, n, D, dtype=torch.bool, device="cuda")
    wide = slice(192, 224) if q8 else slice(200, 201)
    bad[0, 1, 1] = True
    bad[0, 3, 2, wide] = True
    bad[1, 2, 3, slice(64, 96) if q8 else slice(77, 78)] = True
    bad[1, 0, 4, slice(0, 32) if q8 else slice(30, 31)] = True
    bad[1, 0, 4, slice(224, 256) if q8 else slice(255, 256)] = True
    assert torch.equal(~torch.isfinite(torch.stack([k, v])), bad)


@pytest.mark.gpu
def test_prefill_bound_of_rows_may_exceed_them():
    from qwowl35_b200 import ops
    cache = Cache([300], False, 5).fill([300], 6)
    q, gt = some(40, 1, torch.float16), some(40, 2, torch.float16)
    at = (cache.ptrs(), cache.k_off, cache.v_off)
    want = ops.gqa_prefill(q, gt, ints(0, 40), ints(300), 40, 300, *at)
    ws = ops.gqa_prefill_workspace(40, 1, 64, 300)
    for kw in ({}, {"ws": ws}):
        assert torch.equal(ops.gqa_prefill(q, gt, ints(0, 40), ints(300), 64, 300, *at, **kw), want)


# ---- long contexts --------------------------------------------------------------------------------------

LONG = [(False, False, 32768), (False, True, 32768), (True, False, 140000), (True, True, 140000)]


@pytest.mark.gpu
@pytest.mark.parametrize("half,q8,n", LONG)
@pytest.mark.parametrize("runs,rows", [(1, 1300), (40, 3), (16, 1)])  # pairs and single CTAs in one piece; joined from two
def test_prefill_over_long_contexts_stays_exact(half, q8, n, runs, rows):
    """In the 2-norm of a head's row.  O sums at most 2,048 positions in a chain of truncated steps (2^-23 each, 16 positions and
    operand half; q8_0 three), f16 65,536 in steps of half; the rest as over short contexts."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    cache = Cache([n], q8, 5).fill([n], 6)
    q, gt = some(runs * rows, 1, kind), some(runs * rows, 2, kind, 1.0)
    table = cache.ptrs().expand(runs, -1).contiguous()
    for poisoned in (False, True):
        if poisoned:  # (the last row of each run attends it)
            poison(cache, 0, (n - 1,), float("nan"), planes=(1,))
        out = ops.gqa_prefill(q, gt, ints(*range(0, runs * rows + 1, rows)), ints(*[n] * runs), rows, n, table, cache.k_off, cache.v_off,
                              kv_q8=q8)
        k, v = cache.sequence(0, n)
        chain = 65536 / 16 * 2.0 ** -23 + (2.0 ** -10 if q8 else 2.0 ** -11) if half else 2048 / 16 * (3 if q8 else 2) * 2.0 ** -23
        for r in sorted({0, rows // 2, max(rows - 2, 0), (runs // 2) * rows}):
            if poisoned and r % rows == rows - 1:
                assert not bool(torch.isfinite(out[r]).all())
                continue
            see = n - rows + r % rows + 1
            o = attend(q[r], gt[r], k[:, :see], v[:, :see], see)[0]
            err = float(((out[r].double().view(H, D) - o).norm(dim=-1) / o.norm(dim=-1)).max())
            assert err <= 2.0 ** -18 + chain, (r, err)
    assert _lib.lib().qw35_cuda_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("half,q8,n", LONG)
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("runs,rows", [(1, 1300), (40, 3)])
def test_prefill_scores_that_climb_and_fall_over_a_long_context(half, q8, n, up, runs, rows):
    """The maximum grows from tile to tile, over what was put away too; or every later position counts for less."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    cache = Cache([n], q8, 5).fill([n], 6, 0.25)
    q, gt = some(runs * rows, 1, kind, 0.3), some(runs * rows, 2, kind, 1.0)
    q[..., 7] = 3.0
    ramp = torch.arange(n, device="cuda", dtype=torch.float32) / n * (1.0 if up else -1.0)
    rows_k = cache.rows()
    for c in range(-(-n // CH)):
        part, m = rows_k[int(cache.ids[0, c])], min(CH, n - c * CH)
        if q8:  # (block 0: dim 7's code at its largest, d so that d * 127 is the ramp's value)
            part[0, :, :m, 0, 2:] = 0
            part[0, :, :m, 0, 2 + 7] = 127
            d = (ramp[c * CH:c * CH + m] * 200 / 127).half()
            part[0, :, :m, 0, :2] = d.view(torch.uint8).view(m, 2)
        else:
            part[0, :, :m, 7] = (ramp[c * CH:c * CH + m] * 200).half()
    table = cache.ptrs().expand(runs, -1).contiguous()
    out = ops.gqa_prefill(q, gt, ints(*range(0, runs * rows + 1, rows)), ints(*[n] * runs), rows, n, table, cache.k_off, cache.v_off, kv_q8=q8)
    k, v = cache.sequence(0, n)
    ref = []
    for r in sorted({0, rows // 2, rows - 1, (runs // 2) * rows}):
        see = n - rows + r % rows + 1
        ref.append((r, *attend(q[r], gt[r], k[:, :see], v[:, :see], see), see))
    check_rows(out, ref, half, q8)
    assert _lib.lib().qw35_cuda_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("half,q8", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("window,sink", [(0, 0), (1000, 5)])
def test_shared_over_long_prefixes(half, q8, window, sink):
    """Forty pairs of sequences behind one long prefix: parts long enough to put O away; with a window, a sequence that ends early
    attends nothing of most of its part."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    shared, groups = 30000, 40
    cache = Cache([shared + 100, shared + 100], q8, 5).fill([shared + 100] * 2, 6)
    cache.ids[1, :shared // CH] = cache.ids[0, :shared // CH]
    planes = cache.rows()
    planes[int(cache.ids[1, shared // CH])][:, :, :shared % CH] = planes[int(cache.ids[0, shared // CH])][:, :, :shared % CH]
    lens = [5000, shared + 77] * groups
    q, gt = some(2 * groups, 1, kind), some(2 * groups, 2, kind, 1.0)
    out = ops.gqa_decode_shared(q, gt, ints(*lens), ints(*range(0, 2 * groups + 1, 2)), ints(*[shared] * groups), shared, 100,
                                cache.ptrs().repeat(groups, 1), cache.k_off, cache.v_off, window=window, sink=sink, kv_q8=q8)
    ref = []
    for r in (0, 1, 40, 79):
        k, v = cache.sequence(r % 2, lens[r])
        ref.append((r, *attend(q[r], gt[r], k, v, lens[r], window, sink), lens[r]))
    check_rows(out, ref, half, q8)
    assert _lib.lib().qw35_cuda_device_error() == 0


# ---- more of runs: pairs, repeats, precision ---------------------------------------------------------------

def wants_pairs(ctx, rows):
    """The rule by which one run goes to CTA pairs: more than a tile of rows, and two row tiles x 128 positions an SM."""
    return rows > 32 and ((rows - 1) // 32 + 1) * KV * -(-(ctx + rows) // 128) > 2 * 148


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("half,q8", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("ctx,rows,window,sink", [(2000, 200, 0, 0), (9000, 70, 0, 0), (3000, 300, 120, 3)])
@pytest.mark.parametrize("dim", [5, 250])
def test_prefill_on_pairs_keeps_what_a_row_does_not_attend_from_it(value, half, q8, ctx, rows, window, sink, dim):
    """A value in either half of the dims, at positions that some rows of either CTA of a pair do not attend."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    assert wants_pairs(ctx, rows)
    n = ctx + rows
    q, gt = some(rows, 1, kind), some(rows, 2, kind, 1.0)
    for at in (ctx + 10, ctx + 45, ctx + rows - 1):
        cache = Cache([n], q8, 5).fill([n], 6)
        part = cache.rows()[int(cache.ids[0, at // CH]), 1, :, at % CH]
        if q8:
            part[:, dim // 32, :2] = torch.tensor([value], dtype=torch.float16).view(torch.uint8).cuda()
        else:
            part[:, dim] = value
        out = ops.gqa_prefill(q, gt, ints(0, rows), ints(n), rows, n, cache.ptrs(), cache.k_off, cache.v_off, window=window, sink=sink, kv_q8=q8)
        k, v = cache.sequence(0, n)
        wide = ~torch.isfinite(v[0, at])
        k, v = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
        for r in range(0, rows):
            length = ctx + r + 1
            hit = at < length and (window <= 0 or at >= length - window)
            y = out[r].view(H, D)
            assert torch.equal(~torch.isfinite(y), (wide & hit).expand(H, D)), (r, at)
            if r % 9 == 0 or abs(r - (at - ctx)) < 2:
                o, a, s = attend(q[r], gt[r], k, v, length, window, sink)
                err = ((y.double() - o).abs() / bound(o, a, s, length, half, q8))[:, ~wide]
                assert float(err.max()) <= 1.0, (r, at)
    assert _lib.lib().qw35_cuda_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("half,q8", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("ctx,rows", [(4095, 1), (2000, 200), (0, 1500), (0, 5000)])
def test_prefill_repeats_itself(half, q8, ctx, rows):
    """The same bits every time; 5,000 positions leave TMEM in pieces (f32)."""
    from qwowl35_b200 import ops
    kind = torch.float16 if half else torch.float32
    n = ctx + rows
    cache = Cache([n], q8, 5).fill([n], 6)
    q, gt = some(rows, 1, kind), some(rows, 2, kind, 1.0)
    args = (q, gt, ints(0, rows), ints(n), rows, n, cache.ptrs(), cache.k_off, cache.v_off)
    want = ops.gqa_prefill(*args, kv_q8=q8)
    for _ in range(20):
        assert torch.equal(ops.gqa_prefill(*args, kv_q8=q8), want)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("ctx,rows,part", [(0, 300, 300), (4095, 1, 128), (3000, 33, 128), (0, 1100, 1100), (32704, 64, 1920)])
def test_prefill_f32_is_finer_than_f16_operands(q8, ctx, rows, part):
    """In the 2-norm of a head's row.  An operand whose lo half were left out would be off by up to 2^-12 of itself, 2^-13 rms.
    What is there: scores, 2^-18 (48 truncated steps of |s| <= 5, half of 2^-23 each, of which softmax passes on the differences);
    o, 2^-23 a step of 16 positions and operand half (two, q8_0 three)."""
    from qwowl35_b200 import ops
    n = ctx + rows
    cache = Cache([n], q8, 5).fill([n], 6)
    q, gt = some(rows, 1, torch.float32), some(rows, 2, torch.float32, 1.0)
    out = ops.gqa_prefill(q, gt, ints(0, rows), ints(n), rows, n, cache.ptrs(), cache.k_off, cache.v_off, kv_q8=q8)
    k, v = cache.sequence(0, n)
    tol = 2.0 ** -18 + part / 16 * (3 if q8 else 2) * 2.0 ** -23
    assert tol < 2.0 ** -14
    for r in sorted({rows // 3, rows // 2, rows - 1}):
        o = attend(q[r], gt[r], k, v, ctx + r + 1)[0]
        err = (out[r].double().view(H, D) - o).norm(dim=-1) / o.norm(dim=-1)
        assert float(err.max()) <= tol, (r, float(err.max()), tol)
        # the bound tells: the plain form with q rounded to f16 is beyond it
        half_q = attend(q[r].half(), gt[r], k, v, ctx + r + 1)[0]
        assert float(((half_q - o).norm(dim=-1) / o.norm(dim=-1)).max()) > 2 * tol


def test_append_refuses_sections_that_sum_to_32_by_wrapping():
    """2^31 - 1 twice and 34 are 32 in 32 bits."""
    with pytest.raises(_lib.Qw35Error, match="rotary sections"):
        _lib.call("qw35_cuda_attn_append", *_append_args(sec=((1 << 31) - 1, (1 << 31) - 1, 34)))


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("ctx,rows,part", [(0, 2000, 2000), (4095, 1, 128)])
def test_prefill_f32_is_not_short_of_itself(q8, ctx, rows, part):
    """A truncating adder leaves a sum of N steps short by 0 to N 2^-23 of it, some N / 2 steps of 0.72 x 2^-24, which is added
    back: over many heads' rows, what is missing along the exact output is under a third of that (and 2^-21 of scores and gate)."""
    from qwowl35_b200 import ops
    n = ctx + rows
    cache = Cache([n], q8, 5).fill([n], 6)
    q, gt = some(rows, 1, torch.float32), some(rows, 2, torch.float32, 1.0)
    out = ops.gqa_prefill(q, gt, ints(0, rows), ints(n), rows, n, cache.ptrs(), cache.k_off, cache.v_off, kv_q8=q8)
    k, v = cache.sequence(0, n)
    short = []
    for r in range(max(0, rows - 120), rows, 7):
        o = attend(q[r], gt[r], k, v, ctx + r + 1)[0]
        short.append((((out[r].double().view(H, D) - o) * o).sum(-1) / (o * o).sum(-1)).mean())
    steps = part / 16 * (3 if q8 else 2)
    short = float(torch.stack(short).mean())
    assert abs(short) <= 0.72 * 2.0 ** -24 * steps / 2 / 3 + 2.0 ** -21, (short, 0.72 * 2.0 ** -24 * steps / 2)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("where,value,scale", [(None, 0, 12.0), (0, 32.0, 1.5), (0, 48.0, 1.5), (0, 64.0, 1.5), (0, 100.0, 1.5), (-1, 40.0, 1.5)])
def test_prefill_f32_of_rows_that_lean_on_one_position(q8, where, value, scale):
    """The first or the last position, or each row's own, outweighs the rest by e^8 to e^25.  How much of a sum is cut depends on
    when it grew and on what still reaches its last place: what is added back follows that, and leaves at most 0.6 of the half
    of all steps (0.72 x 2^-24 each) that rows without such a position lose, beside 2^-20 of the scores."""
    from qwowl35_b200 import ops
    n = 2000
    cache = Cache([n], q8, 5).fill([n], 6)
    q, gt = some(n, 1, torch.float32, scale), some(n, 2, torch.float32, 1.0)
    if where is not None:
        q[..., 3] = 4.0
        pos = where % n
        part = cache.rows()[int(cache.ids[0, pos // CH]), 0, :, pos % CH]
        if q8:
            part[:, 0, 2:] = 0
            part[:, 0, 2 + 3] = 127
            part[:, 0, :2] = torch.tensor([value / 127], dtype=torch.float16).view(torch.uint8).cuda()
        else:
            part[:, 3] = value
    out = ops.gqa_prefill(q, gt, ints(0, n), ints(n), n, n, cache.ptrs(), cache.k_off, cache.v_off, kv_q8=q8)
    k, v = cache.sequence(0, n)
    errs = []
    for r in range(n - 30, n, 3) if where != -1 else (n - 1,):
        o = attend(q[r], gt[r], k, v, r + 1)[0]
        errs.append(float((out[r].double().view(H, D) - o).norm() / o.norm()))
    err = sum(errs) / len(errs)
    assert err <= 0.6 * 0.72 * 2.0 ** -24 * n / 16 * (3 if q8 else 2) / 2 + 2.0 ** -20, err


@pytest.mark.gpu
def test_captured_long_prompts_replay_on_two_streams():
    """O of 5,000 positions leaves TMEM twice: the same bits in every replay, beside another graph with its own workspace, and right
    for the lengths that stand in device memory."""
    from qwowl35_b200 import ops
    n, rows = 5000, 400
    cache = Cache([n, n], False, 5).fill([n, n], 6)
    q, gt = some(rows, 1, torch.float32), some(rows, 2, torch.float32, 1.0)
    table = cache.ptrs()
    lens = [ints(n), ints(n)]
    off, outs = ints(0, rows), [torch.zeros(rows, H * D, device="cuda") for _ in range(2)]
    ws = [ops.gqa_prefill_workspace(rows, 1, rows, n) for _ in range(2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    tables = [table[i:i + 1].contiguous() for i in range(2)]
    call = lambda i: ops.gqa_prefill(q, gt, off, lens[i], rows, n, tables[i], cache.k_off, cache.v_off, ws=ws[i], out=outs[i])  # noqa: E731
    want = [call(i).clone() for i in range(2)]
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            call(i)
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], want[i]) for i in range(2))
    lens[1].copy_(ints(2100))
    graphs[1].replay()
    k, v = cache.sequence(1, 2100)
    ref = [(r, *attend(q[r], gt[r], k, v, 2100 - rows + r + 1), 2100 - rows + r + 1) for r in (0, 63, 64, 347, 348, 349, rows - 1)]
    check_rows(outs[1], ref, False, False)
    assert _lib.lib().qw35_cuda_device_error() == 0
